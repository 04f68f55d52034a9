// Matrix product in 8-bit integers with one scale per token and one per output channel
// (W8A8), and the row quantisation that feeds it.  No reference counterpart (additive).
//
// Quantisation of a row x (bf16, K values), a = max |x|:
//   q_k = rint(127 x_k / a), ties to even;  s = a / 127  (x_k stands as q_k s)
// a = 0 gives q = 0, s = 0; a row holding an infinity or a NaN gives q = 0, s = NaN, so its
// whole output row is NaN and no other row is touched.  The quotient is exact to its side of
// every border: 127 x has 15 significant bits, so fmaf(-n, a, 127 x) is the exact remainder
// of a candidate n, which decides the neighbour and the ties (x = a/2 is one: 63.5).
// Product: out_mn = bf16((sum_k q_mk w_nk) * (s_m * ws_n)); the sum is exact in 32 bits
// (K <= 131072), so no split or order of it changes the result.
#include <cmath>

#include "kernels.cuh"
#include "ptx.cuh"

namespace ds {
namespace i8 {
namespace {

constexpr int kMaxK = 131072;

// rint(127 x / a) for finite |x| <= a, a > 0; r ~ 127 / a, both scaled alike.
__device__ __forceinline__ int quant1(float x, float a, float r) {
  const float x127 = x * 127.f;  // exact: 8 + 7 significant bits
  float n = rintf(x * r);
  const float e = fmaf(-n, a, x127);  // exact: |n| <= 128 has 8 bits, a has 8
  const float e2 = 2.f * fabsf(e);
  const float step = copysignf(1.f, e);
  const bool odd = (static_cast<int>(n) & 1) != 0;
  if (e2 > a || (e2 == a && odd)) n += step;
  return static_cast<int>(n);
}

// One warp per row when rows are short, one block otherwise (rows of 16-byte vectors).
__global__ void __launch_bounds__(256)
    quantize_kernel(const uint4* __restrict__ x, int64_t ld8, int rows, int k8,
                    uint2* __restrict__ q, float* __restrict__ scale) {
  __shared__ float red[8];
  const int row = blockIdx.x;
  const uint4* src = x + static_cast<int64_t>(row) * ld8;
  float a = 0.f;
  bool bad = false;
  for (int c = threadIdx.x; c < k8; c += 256) {
    const uint4 v = __ldg(src + c);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lo = __uint_as_float(w[i] << 16), hi = __uint_as_float(w[i] & 0xFFFF0000u);
      bad |= !(fabsf(lo) <= 3.4e38f) || !(fabsf(hi) <= 3.4e38f);
      a = fmaxf(a, fmaxf(fabsf(lo), fabsf(hi)));
    }
  }
  if (bad) a = INFINITY;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, d));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) a = fmaxf(a, red[i]);
  const bool finite = a <= 3.4e38f;
  if (threadIdx.x == 0) scale[row] = finite ? a / 127.f : __uint_as_float(0x7FC00000u);
  // subnormal and tiny rows are scaled up by a power of two, so that 127 / a stays finite,
  // huge ones down, so that 127 x does
  const float up = a < 1e-30f ? 1.2676506e30f : a > 1e30f ? 7.8886091e-31f : 1.f;  // 2^100, 2^-100
  const float au = a * up;
  const float r = finite && au > 0.f ? 127.f / au : 0.f;
  uint2* dst = q + static_cast<int64_t>(row) * k8;
  for (int c = threadIdx.x; c < k8; c += 256) {
    uint32_t o[2] = {0u, 0u};
    if (r != 0.f) {
      const uint4 v = __ldg(src + c);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int lo = quant1(__uint_as_float(w[i] << 16) * up, au, r);
        const int hi = quant1(__uint_as_float(w[i] & 0xFFFF0000u) * up, au, r);
        o[i >> 1] |= ((lo & 0xFF) | ((hi & 0xFF) << 8)) << (16 * (i & 1));
      }
    }
    dst[c] = make_uint2(o[0], o[1]);
  }
}

// out[m, n] = bf16(acc * (sa[m] * sw[n])).  64 x 64 outputs a block, 4 x 4 a thread, 64
// bytes of K at a time through shared memory, __dp4a.
__global__ void __launch_bounds__(256)
    gemm_dp4a_kernel(const int8_t* __restrict__ a, const float* __restrict__ sa,
                     const int8_t* __restrict__ w, const float* __restrict__ sw,
                     __nv_bfloat16* __restrict__ out, int M, int N, int K) {
  __shared__ int ta[64][17], tw[64][17];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  int acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 64) {
    const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 16;
    int4 va = make_int4(0, 0, 0, 0), vw = va;
    if (k0 + c < K) {
      if (m0 + r < M)
        va = *reinterpret_cast<const int4*>(a + static_cast<int64_t>(m0 + r) * K + k0 + c);
      if (n0 + r < N)
        vw = *reinterpret_cast<const int4*>(w + static_cast<int64_t>(n0 + r) * K + k0 + c);
    }
    __syncthreads();
    ta[r][c / 4] = va.x; ta[r][c / 4 + 1] = va.y; ta[r][c / 4 + 2] = va.z; ta[r][c / 4 + 3] = va.w;
    tw[r][c / 4] = vw.x; tw[r][c / 4 + 1] = vw.y; tw[r][c / 4 + 2] = vw.z; tw[r][c / 4 + 3] = vw.w;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      int x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = ta[ty + 16 * i][k];
        y[i] = tw[tx + 16 * i][k];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(x[i], y[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int m = m0 + ty + 16 * i;
    if (m >= M) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx + 16 * j;
      if (n < N)
        out[static_cast<int64_t>(m) * N + n] =
            __float2bfloat16_rn(static_cast<float>(acc[i][j]) * (__ldg(sa + m) * __ldg(sw + n)));
    }
  }
}

int check_shape(int64_t M, int N, int K) {
  DS_REQUIRE(M >= 0 && M < (1LL << 31) && N >= 0 && K > 0, "int8_linear: bad shape");
  DS_REQUIRE(K % 16 == 0 && K <= kMaxK, "int8_linear: K=%d must be a multiple of 16, at most %d",
             K, kMaxK);
  DS_REQUIRE(N % 8 == 0, "int8_linear: N=%d must be a multiple of 8", N);
  return DS_OK;
}

}  // namespace

int launch_quantize(const void* x, int64_t ld, int64_t rows, int K, void* q, float* scale,
                    cudaStream_t s) {
  if (rows == 0) return DS_OK;
  quantize_kernel<<<static_cast<unsigned>(rows), 256, 0, s>>>(
      static_cast<const uint4*>(x), ld / 8, static_cast<int>(rows), K / 8, static_cast<uint2*>(q),
      scale);
  DS_LAUNCH_CHECK("quantize_kernel");
  return DS_OK;
}

int launch_gemm(const void* a, const float* sa, const void* w, const float* sw, void* out,
                int64_t M, int N, int K, cudaStream_t s) {
  if (M == 0 || N == 0) return DS_OK;
  const int64_t my = (M + 63) / 64;
  DS_REQUIRE(my <= 65535, "int8_linear: too many rows");
  gemm_dp4a_kernel<<<dim3((N + 63) / 64, static_cast<unsigned>(my)), 256, 0, s>>>(
      static_cast<const int8_t*>(a), sa, static_cast<const int8_t*>(w), sw,
      static_cast<__nv_bfloat16*>(out), static_cast<int>(M), N, K);
  DS_LAUNCH_CHECK("gemm_dp4a_kernel");
  return DS_OK;
}

size_t linear_workspace(int64_t M, int K) {
  return align_up(static_cast<size_t>(M) * K, 256) + align_up(static_cast<size_t>(M) * 4, 256);
}

int launch_linear(const void* x, int64_t ld, const void* w, const float* sw, void* out, int64_t M,
                  int N, int K, void* workspace, size_t ws_bytes, cudaStream_t s) {
  Carve c(workspace, ws_bytes);
  int8_t* q = c.take<int8_t>(static_cast<size_t>(M) * K);
  float* sa = c.take<float>(static_cast<size_t>(M));
  if (!c.ok()) return fail(DS_ERR_WORKSPACE, "int8_linear: workspace needs %zu bytes", c.used);
  DS_TRY(launch_quantize(x, ld, M, K, q, sa, s));
  return launch_gemm(q, sa, w, sw, out, M, N, K, s);
}

}  // namespace i8
}  // namespace ds

extern "C" {

int ds_int8_quantize(const void* x_bf16, int64_t row_stride, int rows, int cols, void* q_int8,
                     float* scale, void* stream) {
  DS_REQUIRE(rows >= 0 && cols > 0 && cols % 16 == 0, "int8_quantize: cols=%d must be a positive multiple of 16", cols);
  if (rows == 0) return DS_OK;
  DS_REQUIRE(x_bf16 && q_int8 && scale, "int8_quantize: null pointer");
  DS_REQUIRE(row_stride >= cols && row_stride % 8 == 0 && ds::aligned16(x_bf16) &&
                 ds::aligned16(q_int8),
             "int8_quantize: rows must start on 16-byte boundaries");
  return ds::i8::launch_quantize(x_bf16, row_stride, rows, cols, q_int8, scale,
                                 static_cast<cudaStream_t>(stream));
}

size_t ds_int8_linear_workspace_size(int rows, int out_features, int in_features) {
  (void)out_features;
  if (rows <= 0 || in_features <= 0) return 0;
  return ds::i8::linear_workspace(rows, in_features);
}

int ds_int8_linear(const void* x_bf16, int64_t row_stride, const void* w_int8,
                   const float* w_scale, void* out_bf16, int rows, int out_features,
                   int in_features, void* workspace, size_t workspace_bytes, void* stream) {
  DS_TRY(ds::i8::check_shape(rows, out_features, in_features));
  if (rows == 0 || out_features == 0) return DS_OK;
  DS_REQUIRE(x_bf16 && w_int8 && w_scale && out_bf16 && workspace, "int8_linear: null pointer");
  DS_REQUIRE(row_stride >= in_features && row_stride % 8 == 0 && ds::aligned16(x_bf16) &&
                 ds::aligned16(w_int8) && ds::aligned16(out_bf16) && ds::aligned16(workspace),
             "int8_linear: x rows, w, out and workspace must be 16-byte aligned");
  return ds::i8::launch_linear(x_bf16, row_stride, w_int8, w_scale, out_bf16, rows, out_features,
                               in_features, workspace, workspace_bytes,
                               static_cast<cudaStream_t>(stream));
}

}  // extern "C"
