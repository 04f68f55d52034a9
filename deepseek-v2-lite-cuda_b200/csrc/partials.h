// Plain C++ (no CUDA): used by the kernels that join the attention's partials, and by a host test.
#pragma once

#if defined(__CUDACC__)
#define DS_HOST_DEVICE __host__ __device__
#else
#define DS_HOST_DEVICE
#endif

namespace ds {

// A row's partials are `count` of the `parts` that the workspace has, from `first` on.  An attention
// CTA whose load did not arrive in time leaves rows behind it without an entry, and what the joining
// kernels then read there is whatever the workspace held: false for all that lies outside.
DS_HOST_DEVICE inline bool partials_exist(int first, int count, int parts) {
  return first >= 0 && count >= 0 && count <= parts && first <= parts - count;
}

}  // namespace ds
