// Matrix product in 8-bit integers with one scale per token and one per output channel
// (W8A8), and the row quantisation that feeds it.  No reference counterpart (additive).
//
// Quantisation of a row x (bf16, K values), a = max |x|:
//   q_k = rint(127 x_k / a), ties to even;  s = a / 127  (x_k stands as q_k s)
// a = 0 gives q = 0, s = 0; a row holding an infinity or a NaN gives q = 0, s = NaN, so its
// whole output row is NaN and no other row is touched.  Every quotient goes to its own side: with
// 127 / a = rh + rl to twice f32's bits, fmaf(x, rh, x rl) is 127 x / a rounded once, so a tie (x
// = a / 2 is one: 63.5) stays one, and no other quotient of two 8-bit significands is nearer to
// a tie than 2^-15 of itself.
// Product: out_mn = bf16((sum_k q_mk w_nk) * (s_m * ws_n)); the sum is exact in 32 bits
// (K <= 131072), so no split or order of it changes the result.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "kernels.cuh"
#include "ptx.cuh"

namespace ds {
namespace i8 {
namespace {

constexpr int kMaxK = 131072;

// The larger magnitudes of eight bf16 values, two to a word, as bit patterns: those of finite
// values order as the values do, infinities and NaN lie above them.
__device__ __forceinline__ uint32_t abs_max8(const uint4& v, uint32_t a) {
  a = __vmaxu2(a, __vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu));
  return __vmaxu2(a, __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
}

struct RowScale {
  float up, rh, rl;  // quotient = x up (rh + rl); all 0 for an empty or non-finite row
};
__device__ __forceinline__ RowScale row_scale(float a, bool finite) {
  RowScale s;
  // subnormal and tiny rows are scaled up by a power of two, so that 127 / a stays finite,
  // huge ones down, so that its lower part does not vanish
  s.up = a < 1e-30f ? 0x1p100f : a > 1e30f ? 0x1p-100f : 1.f;
  const float au = a * s.up;
  const bool some = finite && au > 0.f;
  s.rh = some ? 127.f / au : 0.f;
  s.rl = some ? fmaf(-s.rh, au, 127.f) / au : 0.f;
  return s;
}
// rint into the low byte: adding 1.5 * 2^23 rounds to a whole number, ties to even.
__device__ __forceinline__ uint32_t quant1(float x, const RowScale& s) {
  return __float_as_uint(fmaf(x, s.rh, x * s.rl) + 12582912.f);
}
__device__ __forceinline__ uint2 quant8(const uint4& v, const RowScale& s) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float lo = __uint_as_float(w[i] << 16), hi = __uint_as_float(w[i] & 0xFFFF0000u);
    if (s.up != 1.f) {
      lo *= s.up;
      hi *= s.up;
    }
    h[i] = __byte_perm(quant1(lo, s), quant1(hi, s), 0x0040);
  }
  const bool some = s.rh != 0.f;  // (a non-finite row's products are not numbers)
  return make_uint2(some ? __byte_perm(h[0], h[1], 0x5410) : 0u,
                    some ? __byte_perm(h[2], h[3], 0x5410) : 0u);
}

// TPR threads a row (a warp, or the block of 256); a row of at most TPR * V 16-byte vectors
// stays in registers between the maximum and the quotients, a longer one is read twice.  Bound by its
// bytes: 16384 x 2048 takes 17.8 us, 5.7 TB/s.
template <int TPR, int V>
__global__ void __launch_bounds__(256)
    quantize_kernel(const uint4* x, int64_t ld8, int rows, int k8,
                    uint2* q, float* scale) {
  __shared__ uint32_t red[8];
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int row = TPR == 32 ? static_cast<int>(blockIdx.x) * 8 + (threadIdx.x >> 5)
                            : static_cast<int>(blockIdx.x);
  if (TPR == 32 && row >= rows) return;
  const int t = TPR == 32 ? threadIdx.x & 31 : threadIdx.x;
  const uint4* src = x + static_cast<int64_t>(row) * ld8;
  uint2* dst = q + static_cast<int64_t>(row) * k8;
  uint4 v[V];
#pragma unroll
  for (int i = 0; i < V; ++i)
    v[i] = t + i * TPR < k8 ? src[t + i * TPR] : make_uint4(0, 0, 0, 0);
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) m2 = abs_max8(v[i], m2);
  for (int c = t + V * TPR; c < k8; c += TPR) m2 = abs_max8(src[c], m2);
  uint32_t m = max(m2 & 0xFFFFu, m2 >> 16);
  m = __reduce_max_sync(0xffffffffu, m);
  if (TPR > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, red[i]);
  }
  const bool finite = m < 0x7F80u;
  const float a = __uint_as_float(m << 16);
  if (t == 0) scale[row] = finite ? a / 127.f : __uint_as_float(0x7FC00000u);
  const RowScale s = row_scale(a, finite);
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (t + i * TPR < k8) dst[t + i * TPR] = quant8(v[i], s);
  for (int c = t + V * TPR; c < k8; c += TPR) dst[c] = quant8(src[c], s);
}

// ---- the product ----------------------------------------------------------------------------
// tcgen05.mma kind::i8 (K = 32 an instruction, 32-bit integer accumulators in TMEM), operands
// by TMA in k-blocks of 128 bytes, 128-byte swizzle.  Every wait is bounded.
constexpr int kBK = 128;
constexpr uint32_t kTileBytes = 128 * kBK;  // 128 rows of a k-block
constexpr long long kTimeoutCycles = 4000000000LL;

// Instruction descriptor, kind::i8: signed 8-bit A and B (K-major), 32-bit integer D.
__host__ __device__ constexpr uint32_t idesc_i8(int M, int N) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Few rows: the weights are the M operand, so a tile is 128 output channels x NT rows of x and
// the kernel streams the weights once, whatever the rows (bound: the weights' bytes).  To have
// enough CTAs streaming, a cluster of `splits` CTAs shares a tile, each with a part of K; the
// partial sums are integers and meet through distributed shared memory, exactly.  The weight
// loads of the first stages go out before the kernel waits for the quantised rows (programmatic
// dependent launch behind quantize_kernel).
constexpr int kFewThreads = 128;
// QUANT: up to four rows of x, rows * K <= kQuantHere: every CTA takes the maxima of whole rows
// itself and quantises its part of K straight into the operand's shared-memory layout; no first
// kernel, whose launch costs more than reading x once per CTA (1 x 2048 x 9792: 6.8 us against 7.7
// and a second launch on the host).
constexpr int kQuantHere = 16384;   // values of x
constexpr int kQuantRows = 4;
constexpr int kQuantBlocks = 16;    // k-blocks of a CTA (2 KB of operand each)
template <int NT>
struct FewTile {
  static constexpr int stages = NT <= 16 ? 6 : NT <= 32 ? 5 : NT <= 64 ? 4 : 3;  // two CTAs an SM
  static constexpr uint32_t stage = kTileBytes + NT * kBK;
  static constexpr uint32_t tmem_cols = NT < 32 ? 32 : NT;
  static constexpr size_t smem = 1024 + stages * stage + 256;
  static constexpr int quant_stages = 5;
  static constexpr size_t smem_quant(int k_blocks) {
    return 1024 + quant_stages * kTileBytes + static_cast<size_t>(k_blocks) * NT * kBK + 256 + NT * 32;
  }
  // [splits][ceil(NT / splits)][128] sums, splits <= 8
  static_assert((NT + 7) * 128 * 4 <= stages * stage, "the sums reuse the ring");
};
struct FewParams {
  const uint4* x;  // QUANT: the rows, ld8 vectors apart
  int64_t ld8;
  int k8;
  const float* sa;
  const float* sw;
  __nv_bfloat16* out;
  int M, N, k_blocks, splits, kb_per_split;
  int* status;
};

template <int NT, bool QUANT>
__global__ void __launch_bounds__(kFewThreads)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                    const FewParams p) {
  using T = FewTile<NT>;
  constexpr int kFewStages = QUANT ? T::quant_stages : T::stages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t s0 = ptx::smem_u32(smem);
  // a stage's weights, then its rows of x; QUANT: all stages' weights, then all rows of x
  constexpr uint32_t kStage = QUANT ? kTileBytes : T::stage;
  uint8_t* tail = smem + kFewStages * kStage + (QUANT ? p.kb_per_split * NT * kBK : 0);
  float* row_scale_s = reinterpret_cast<float*>(tail + 256);  // QUANT
  const uint32_t full0 = ptx::smem_u32(tail), empty0 = full0 + 8 * kFewStages;
  const uint32_t done = empty0 + 8 * kFewStages;
  uint32_t* holder = reinterpret_cast<uint32_t*>(tail + 8 * (2 * kFewStages + 1));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(holder + 1);
  volatile int* never_flag = abort_flag + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.splits;
  const int n0 = static_cast<int>(blockIdx.x) / p.splits * 128;
  const int m0 = static_cast<int>(blockIdx.y) * NT;
  const int kb0 = rank * p.kb_per_split;
  const int nkb = min(p.k_blocks, kb0 + p.kb_per_split) - kb0;  // >= 1: no split is empty
  if (threadIdx.x == 0) {
    for (int i = 0; i < kFewStages; ++i) {
      ptx::mbar_init(full0 + 8 * i, 1);
      ptx::mbar_init(empty0 + 8 * i, 1);
    }
    ptx::mbar_init(done, 1);
    *abort_flag = 0;
    *never_flag = 0;
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(holder), T::tmem_cols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *holder;
  const int pre = min(nkb, kFewStages);
  // (not QUANT: quantize_kernel lets this one in once all before it is complete, so the weights
  // may be read at once, and the quantised rows after the wait)
  if (QUANT) ptx::pdl_wait();
  if (warp == 0 && lane == 0) {
    for (int i = 0; i < pre; ++i) {
      ptx::mbar_arrive_expect_tx(full0 + 8 * i, kStage);
      ptx::tma_load_2d(s0 + i * kStage, &tmW, full0 + 8 * i, (kb0 + i) * kBK, n0);
    }
    if (!QUANT) {
      ptx::pdl_wait();
      for (int i = 0; i < pre; ++i)
        ptx::tma_load_2d(s0 + i * kStage + kTileBytes, &tmX, full0 + 8 * i, (kb0 + i) * kBK, m0);
    }
  }
  __syncwarp();
  if (QUANT) {
    // the rows' maxima over all of K, then this CTA's part of them, 16 bytes of operand a thread
    // and step, in the 128-byte swizzle; rows behind the last, and k behind K, are zeros
    uint8_t* xs = smem + kFewStages * kStage;
    uint32_t* part_max = reinterpret_cast<uint32_t*>(tail + 256 + NT * 16);  // [4][NT]
    RowScale* scales = reinterpret_cast<RowScale*>(tail + 256 + NT * 4);     // [NT]
    {
      const int tpr = p.M == 1 ? kFewThreads : p.M == 2 ? 64 : 32;  // threads a row: whole warps
      const int r = threadIdx.x / tpr;
      uint32_t m2 = 0;
      if (r < p.M) {
        const uint4* src = p.x + static_cast<int64_t>(r) * p.ld8;
#pragma unroll 8
        for (int c = threadIdx.x % tpr; c < p.k8; c += tpr) m2 = abs_max8(src[c], m2);
      }
      const uint32_t m = __reduce_max_sync(0xffffffffu, max(m2 & 0xFFFFu, m2 >> 16));
      if (lane < kQuantRows) part_max[warp * NT + lane] = lane == r ? m : 0u;
    }
    __syncthreads();
    if (threadIdx.x < p.M) {
      const int r = threadIdx.x;
      const uint32_t m = max(max(part_max[r], part_max[NT + r]),
                             max(part_max[2 * NT + r], part_max[3 * NT + r]));
      const bool finite = m < 0x7F80u;
      const float a = __uint_as_float(m << 16);
      row_scale_s[r] = finite ? a / 127.f : __uint_as_float(0x7FC00000u);
      scales[r] = row_scale(a, finite);
    }
    __syncthreads();
    const int per_row = nkb * 8;
#pragma unroll 2
    for (int i = threadIdx.x; i < NT * per_row; i += kFewThreads) {
      const int r = i / per_row, c = i - r * per_row;
      const int k = kb0 * 16 + 2 * c;  // in vectors of 8 values
      uint2 lo = make_uint2(0u, 0u), hi = lo;
      if (r < p.M && k < p.k8) {  // (K is a multiple of 16: both vectors or none)
        const uint4* src = p.x + static_cast<int64_t>(r) * p.ld8 + k;
        const RowScale rs = scales[r];
        lo = quant8(src[0], rs);
        hi = quant8(src[1], rs);
      }
      *reinterpret_cast<uint4*>(xs + (c >> 3) * (NT * kBK) + r * kBK + (((c & 7) ^ (r & 7)) << 4)) =
          make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    ptx::fence_async_shared();  // written by threads, read by the MMAs
    __syncthreads();
  }
  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int issued = pre;
      for (int i = pre; ok && i < nkb; ++i) {
        const int st = i % kFewStages;
        ok = ptx::mbar_wait(empty0 + 8 * st, (i / kFewStages - 1) & 1, abort_flag, p.status,
                            kTimeoutCycles, DS_ERR_TIMEOUT);
        if (!ok) break;
        ptx::mbar_arrive_expect_tx(full0 + 8 * st, kStage);
        ptx::tma_load_2d(s0 + st * kStage, &tmW, full0 + 8 * st, (kb0 + i) * kBK, n0);
        if (!QUANT)
          ptx::tma_load_2d(s0 + st * kStage + kTileBytes, &tmX, full0 + 8 * st, (kb0 + i) * kBK, m0);
        issued = i + 1;
      }
      // every load has landed before this CTA goes on: the last fill of each stage
      for (int i = max(0, issued - kFewStages); i < issued; ++i)
        ptx::mbar_wait(full0 + 8 * (i % kFewStages), (i / kFewStages) & 1, never_flag, p.status,
                       kTimeoutCycles, DS_ERR_TIMEOUT);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_i8(128, NT);
      for (int i = 0; i < nkb; ++i) {
        const int st = i % kFewStages;
        if (!ptx::mbar_wait(full0 + 8 * st, (i / kFewStages) & 1, abort_flag, p.status,
                            kTimeoutCycles, DS_ERR_TIMEOUT))
          break;
        ptx::tc_fence_after();
        const uint32_t a = s0 + st * kStage;
        const uint32_t b = QUANT ? s0 + kFewStages * kStage + i * (NT * kBK) : a + kTileBytes;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_i8(tmem, ptx::sw128_kmajor_desc(a + 32u * k), ptx::sw128_kmajor_desc(b + 32u * k),
                  idesc, i != 0 || k != 0);
        ptx::umma_commit(empty0 + 8 * st);
      }
      ptx::umma_commit(done);
    }
  }
  __syncwarp();
  int ok = 1;
  if (lane == 0)
    ok = ptx::mbar_wait(done, 0, never_flag, p.status, kTimeoutCycles, DS_ERR_TIMEOUT) &&
         !*abort_flag;
  ok = __syncthreads_and(__shfl_sync(0xffffffffu, ok, 0));
  ptx::tc_fence_after();
  // D (lane = channel, column = row of x): each CTA finishes `per` of the rows and takes the
  // others' sums for them into its ring, [CTA][row][128 channels].  Stores travel without a
  // reply, so one barrier pays for all of them (remote loads in the sum cost 2-5 us).
  __syncwarp();
  if (p.splits > 1) ptx::cluster_sync();  // every CTA's ring is free
  const uint32_t tb = tmem + (static_cast<uint32_t>(warp * 32) << 16);
  const int mrows = min(NT, p.M - m0);
  const int per = (mrows + p.splits - 1) / p.splits;
  int owner = 0, in_owner = 0;
  uint32_t to = (p.splits > 1 ? ptx::mapa_shared(s0, 0) : s0) + (rank * per * 128 + threadIdx.x) * 4;
#pragma unroll 1
  for (int c = 0; c < NT; c += 32) {
    if (c >= mrows) break;
    uint32_t v[32];
    ptx::tmem_ld32(tb + c, v);
    ptx::tmem_wait_ld(v);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (i >= NT || c + i >= mrows) break;
      asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to), "r"(v[i]) : "memory");
      to += 128 * 4;
      if (++in_owner == per && p.splits > 1) {
        in_owner = 0;
        to = ptx::mapa_shared(s0, min(++owner, p.splits - 1)) + (rank * per * 128 + threadIdx.x) * 4;
      }
    }
  }
  ptx::tc_fence_before();
  __syncwarp();
  if (p.splits > 1) ptx::cluster_sync();  // all sums have arrived; no remote access follows
  else __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, T::tmem_cols);
  }
  if (!QUANT) ptx::pdl_wait();  // the rows' scales
  ptx::pdl_launch_dependents();
  if (!ok) return;
  // 16 threads a row, 8 channels each
  const int r0 = rank * per, rn = min(mrows, r0 + per) - r0;
  const int n = n0 + (threadIdx.x & 15) * 8;
  if (n >= p.N) return;  // (N is a multiple of 8)
  float sw[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) sw[j] = p.sw[n + j];
  for (int r = threadIdx.x >> 4; r < rn; r += kFewThreads / 16) {
    const float sa = QUANT ? row_scale_s[r0 + r] : p.sa[m0 + r0 + r];
    const int4* src = reinterpret_cast<const int4*>(smem) + r * 32 + (threadIdx.x & 15) * 2;
    int4 x = src[0], y = src[1];
    for (int k = 1; k < p.splits; ++k) {
      const int4 u = src[k * per * 32], v = src[k * per * 32 + 1];
      x.x += u.x; x.y += u.y; x.z += u.z; x.w += u.w;
      y.x += v.x; y.y += v.y; y.z += v.z; y.w += v.w;
    }
    const uint4 o = make_uint4(
        pack2(static_cast<float>(x.x) * (sa * sw[0]), static_cast<float>(x.y) * (sa * sw[1])),
        pack2(static_cast<float>(x.z) * (sa * sw[2]), static_cast<float>(x.w) * (sa * sw[3])),
        pack2(static_cast<float>(y.x) * (sa * sw[4]), static_cast<float>(y.y) * (sa * sw[5])),
        pack2(static_cast<float>(y.z) * (sa * sw[6]), static_cast<float>(y.w) * (sa * sw[7])));
    *reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(m0 + r0 + r) * p.N + n) = o;
  }
}

// Many rows: tiles of 256 rows x 256 channels by pairs of CTAs (cta_group::2), persistent over
// the tiles, as grouped_gemm_kernel's pair mode: each CTA loads its own 128 rows and its half of
// the channels (32 KB a k-block, 6 stages), two accumulators of 256 columns let the epilogue of
// a tile run under the products of the next.  A last tile of fewer channels runs narrower MMAs.
// Bound by the tensor cores: 16384 x 2048 x 3648 takes 88 us, 2.8 Pop/s (twice the bf16 burst rate:
// 73 us).
constexpr int kManyStages = 6;
constexpr int kManyThreads = 192;
constexpr uint32_t kSlabBytes = 32 * 128;
constexpr size_t kManySmem = 1024 + kManyStages * 2 * kTileBytes + 4 * kSlabBytes + 256 + 2 * 256 * 4;
struct ManyParams {
  const float* sa;
  const float* sw;
  int M, N, k_blocks, n_tiles, tiles;
  int* status;
};

__global__ void __launch_bounds__(kManyThreads, 1)
    many_rows_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                     const __grid_constant__ CUtensorMap tmO, const ManyParams p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t sX = ptx::smem_u32(smem), sW = sX + kManyStages * kTileBytes;
  const uint32_t sOut = sW + kManyStages * kTileBytes;
  uint8_t* tail = smem + kManyStages * 2 * kTileBytes + 4 * kSlabBytes;
  float* sw = reinterpret_cast<float*>(tail + 256);  // [2][256] channel scales of a tile
  const uint32_t full0 = ptx::smem_u32(tail), empty0 = full0 + 8 * kManyStages;
  const uint32_t tfull0 = empty0 + 8 * kManyStages, tempty0 = tfull0 + 16, drain = tempty0 + 16;
  uint32_t* holder = reinterpret_cast<uint32_t*>(tail + 8 * (2 * kManyStages + 5));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(holder + 1);
  volatile int* never_flag = abort_flag + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const int unit = blockIdx.x >> 1, units = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kManyStages; ++i) {
      ptx::mbar_init(full0 + 8 * i, 1);
      ptx::mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(tfull0 + 8 * i, 1);
      ptx::mbar_init(tempty0 + 8 * i, 8);
    }
    ptx::mbar_init(drain, 1);
    *abort_flag = 0;
    *never_flag = 0;
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(ptx::smem_u32(holder), 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  ptx::tc_fence_before();
  __syncwarp();
  ptx::cluster_sync();  // both CTAs' barriers are set up before either signals the other's
  ptx::tc_fence_after();
  const uint32_t tmem = *holder;
  if (warp == 0) {
    if (lane == 0) {
      int st = 0;
      uint32_t phase = 0, used = 0, phases = 0;
      bool ok = true;
      for (int t = unit; ok && t < p.tiles; t += units) {
        const int m0 = t / p.n_tiles * 256 + rank * 128, n0 = t % p.n_tiles * 256;
        const int half = (min(256, p.N - n0) + 31) / 32 * 16;  // channels of this CTA's half
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!ptx::mbar_wait(empty0 + 8 * st, phase ^ 1u, abort_flag, p.status, kTimeoutCycles,
                              DS_ERR_TIMEOUT)) {
            ok = false;
            break;
          }
          // the leader's barrier counts both CTAs' bytes
          const uint32_t lead = ptx::mapa_shared(full0 + 8 * st, 0);
          if (rank == 0) ptx::mbar_arrive_expect_tx(full0 + 8 * st, 4 * kTileBytes);
          ptx::tma_load_2d_pair(sX + st * kTileBytes, &tmX, lead, kb * kBK, m0);
          ptx::tma_load_2d_pair(sW + st * kTileBytes, &tmW, lead, kb * kBK, n0 + rank * half);
          used |= 1u << st;
          phases = (phases & ~(1u << st)) | (phase << st);
          if (++st == kManyStages) {
            st = 0;
            phase ^= 1u;
          }
        }
      }
      // every load has landed before the CTA may exit (the peer sees the leader's stages as
      // consumed by the MMAs)
      for (int i = 0; i < kManyStages; ++i)
        if (used & (1u << i))
          ptx::mbar_wait((rank != 0 ? empty0 : full0) + 8 * i, (phases >> i) & 1u, never_flag,
                         p.status, kTimeoutCycles, DS_ERR_TIMEOUT);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int st = 0, acc = 0;
      uint32_t phase = 0, aphase = 0;
      bool ok = true;
      for (int t = unit; ok && t < p.tiles; t += units) {
        if (!ptx::mbar_wait(tempty0 + 8 * acc, aphase ^ 1u, abort_flag, p.status, kTimeoutCycles,
                            DS_ERR_TIMEOUT))
          break;
        ptx::tc_fence_after();
        const int n0 = t % p.n_tiles * 256;
        const uint32_t idesc = idesc_i8(256, (min(256, p.N - n0) + 31) / 32 * 32);
        const uint32_t d = tmem + acc * 256;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!ptx::mbar_wait(full0 + 8 * st, phase, abort_flag, p.status, kTimeoutCycles,
                              DS_ERR_TIMEOUT)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
          const uint32_t a = sX + st * kTileBytes, b = sW + st * kTileBytes;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_i8_pair(d, ptx::sw128_kmajor_desc(a + 32u * k),
                         ptx::sw128_kmajor_desc(b + 32u * k), idesc, kb != 0 || k != 0);
          ptx::umma_commit_pair(empty0 + 8 * st);  // the stage is free in both CTAs
          ptx::umma_commit_pair(ptx::mapa_shared(empty0 + 8 * st, 1));
          if (++st == kManyStages) {
            st = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        ptx::umma_commit_pair(tfull0 + 8 * acc);
        ptx::umma_commit_pair(ptx::mapa_shared(tfull0 + 8 * acc, 1));
        if (++acc == 2) {
          acc = 0;
          aphase ^= 1u;
        }
      }
      ptx::umma_commit_pair(drain);  // no MMA may still write when TMEM is released
      ptx::mbar_wait(drain, 0, never_flag, p.status, kTimeoutCycles, DS_ERR_TIMEOUT);
    }
  } else {
    const int q = warp & 3, r = q * 32 + lane;  // TMEM lane quarter of this warp
    const int et = threadIdx.x - 64;
    const uint32_t slab = sOut + (warp - 2) * kSlabBytes;
    int acc = 0;
    uint32_t aphase = 0;
    for (int t = unit; t < p.tiles; t += units) {
      const int m0 = t / p.n_tiles * 256 + rank * 128, n0 = t % p.n_tiles * 256;
      const int cols = min(256, p.N - n0);
      float* swt = sw + acc * 256;
      swt[et] = n0 + et < p.N ? p.sw[n0 + et] : 0.f;
      swt[et + 128] = n0 + et + 128 < p.N ? p.sw[n0 + et + 128] : 0.f;
      const float sa = m0 + r < p.M ? p.sa[m0 + r] : 0.f;
      __syncwarp();
      ptx::named_bar_sync(1, 128);
      int ok = 1;
      if (lane == 0)
        ok = ptx::mbar_wait(tfull0 + 8 * acc, aphase, abort_flag, p.status, kTimeoutCycles,
                            DS_ERR_TIMEOUT);
      // (all four epilogue warps leave together: the named barrier above counts them)
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (ok) {
        ptx::tc_fence_after();
        const uint32_t tb = tmem + acc * 256 + (static_cast<uint32_t>(q * 32) << 16);
#pragma unroll 1
        for (int c = 0; c < 256; c += 64) {
          if (c >= cols || m0 + q * 32 >= p.M) break;
          uint32_t a[32], b[32];
          ptx::tmem_ld32(tb + c, a);
          ptx::tmem_ld32(tb + c + 32, b);
          ptx::tmem_wait_ld2(a, b);
          uint32_t w[32];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 f = *reinterpret_cast<const float2*>(swt + c + 2 * i);
            const float2 g = *reinterpret_cast<const float2*>(swt + c + 32 + 2 * i);
            w[i] = pack2(static_cast<float>(static_cast<int>(a[2 * i])) * (sa * f.x),
                         static_cast<float>(static_cast<int>(a[2 * i + 1])) * (sa * f.y));
            w[16 + i] = pack2(static_cast<float>(static_cast<int>(b[2 * i])) * (sa * g.x),
                              static_cast<float>(static_cast<int>(b[2 * i + 1])) * (sa * g.y));
          }
          if (lane == 0) ptx::bulk_wait_read0();  // the slab's last store has read it
          __syncwarp();
          // 128-byte rows, 16-byte chunks swizzled as the output's tensor map expects
          const uint32_t row = slab + lane * 128u;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                             row + ((static_cast<uint32_t>(j) ^ (lane & 7u)) << 4)),
                         "r"(w[4 * j]), "r"(w[4 * j + 1]), "r"(w[4 * j + 2]), "r"(w[4 * j + 3])
                         : "memory");
          ptx::fence_async_shared();
          __syncwarp();
          if (lane == 0) {  // rows and channels outside the output are not stored
            ptx::tma_store_2d(&tmO, slab, n0 + c, m0 + q * 32);
            ptx::bulk_commit();
          }
        }
        ptx::tc_fence_before();
      }
      __syncwarp();
      if (lane == 0 && ok) {
        if (rank != 0) ptx::mbar_arrive_remote(ptx::mapa_shared(tempty0 + 8 * acc, 0));
        else ptx::mbar_arrive(tempty0 + 8 * acc);
      }
      if (++acc == 2) {
        acc = 0;
        aphase ^= 1u;
      }
    }
    if (lane == 0) ptx::bulk_wait0();
  }
  __syncwarp();
  ptx::tc_fence_before();
  ptx::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem, 512);
  }
}

// ---- host side ------------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;

int tmap(CUtensorMap* m, const void* ptr, CUtensorMapDataType type, int bytes, int64_t rows,
         int64_t cols, uint32_t box_cols, uint32_t box_rows) {
  std::call_once(g_encode_once, [] {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  if (g_encode == nullptr) return fail(DS_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * bytes};
  cuuint32_t box[2] = {box_cols, box_rows};
  cuuint32_t estr[2] = {1u, 1u};
  const CUresult r = g_encode(m, type, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(DS_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return DS_OK;
}

bool g_attr_set[64] = {};
std::mutex g_attr_mutex;
int g_pairs[64] = {};  // co-resident CTA pairs of the many-rows kernel

template <int NT>
int few_attr() {
  DS_CUDA(cudaFuncSetAttribute(few_rows_kernel<NT, false>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(FewTile<NT>::smem)));
  if (NT == 16)
    DS_CUDA(cudaFuncSetAttribute(few_rows_kernel<16, true>,
                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 static_cast<int>(FewTile<16>::smem_quant(kQuantBlocks))));
  return DS_OK;
}

int set_attrs(const DeviceInfo& di) {
  std::lock_guard<std::mutex> lock(g_attr_mutex);
  if (g_attr_set[di.device]) return DS_OK;
  DS_TRY(few_attr<16>());
  DS_TRY(few_attr<32>());
  DS_TRY(few_attr<64>());
  DS_TRY(few_attr<128>());
  DS_CUDA(cudaFuncSetAttribute(many_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>(kManySmem)));
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(2 * (di.num_sms / 2));
  cfg.blockDim = dim3(kManyThreads);
  cfg.dynamicSmemBytes = kManySmem;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  DS_CUDA(cudaOccupancyMaxActiveClusters(&n, many_rows_kernel, &cfg));
  g_pairs[di.device] = n;
  g_attr_set[di.device] = true;
  return DS_OK;
}

// K in parts: enough CTAs for the SMs to stream (up to 1.6 a SM; two fit), two k-blocks each or more (the
// last part may have fewer, and none is empty), clusters of at most 8: of 1 to 4 or 6 to 8 as it comes out.
void few_splits(int64_t tiles, int k_blocks, int num_sms, int* splits, int* per) {
  int n = 1;
  while (n < 8 && tiles * n * 10 <= num_sms * 8 && k_blocks >= 4 * n) n *= 2;
  *per = (k_blocks + n - 1) / n;
  *splits = (k_blocks + *per - 1) / *per;
}

// Which kernel takes more than 64 rows: an estimate of both, in hundredths of a microsecond, from
// their times at 65 to 1024 rows of nine weights (256 x 2048 to 9792 x 8192).  A pair takes 0.36 us
// for 256 x 256 x 128 products, the tensor cores' rate, and does not split K; a CTA of the other
// kernel takes 0.27 us for 128 x 128 x 128 beside a second one, splits K over a cluster when
// there are few tiles, and writes its transposed tile more slowly.  Few / many rows' kernel:
// 128 x 2048 x 9792 15.0 / 13.2 us, 256 x 1424 x 2840 13.1 / 11.4, 512 x 8192 x 2048 23.2 / 30.7,
// 192 x 8192 x 9792 37.0 / 30.1, 333 x 8192 x 9792 39.2 / 52.9, 1024 x 2048 x 9792 47.7 / 27.4.
bool many_rows_faster(int M, int N, int K, int num_sms, int pairs) {
  if (pairs < 1) return false;
  const int64_t kb = (K + kBK - 1) / kBK, n128 = (N + 127) / 128, m128 = (M + 127) / 128;
  if (m128 > 65535) return true;  // the other kernel's grid ends there
  const int64_t tiles = n128 * m128, pair_tiles = ((N + 255) / 256) * static_cast<int64_t>((M + 255) / 256);
  int splits = 1, per = static_cast<int>(kb);
  few_splits(tiles, static_cast<int>(kb), num_sms, &splits, &per);
  const int64_t few = 600 + 270 * std::min(M, 128) / 128 + (splits > 1 ? 50 : 0) +
                      27 * ((tiles * splits + num_sms - 1) / num_sms) * per;
  return 570 + 36 * ((pair_tiles + pairs - 1) / pairs) * kb <= few;
}

// x: the rows to quantise (QUANT) or null; a, sa: the quantised rows.
template <int NT, bool QUANT>
int launch_few(const void* x, int64_t ld, const void* a, const float* sa, const void* w,
               const float* sw, void* out, int M, int N, int K, const DeviceInfo& di,
               cudaStream_t s) {
  CUtensorMap tmW, tmX;
  DS_TRY(tmap(&tmW, w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, N, K, kBK, 128));
  if (QUANT) tmX = tmW;
  else DS_TRY(tmap(&tmX, a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, M, K, kBK, NT));
  FewParams p{};
  p.x = static_cast<const uint4*>(x);
  p.ld8 = ld / 8;
  p.k8 = K / 8;
  p.sa = sa;
  p.sw = sw;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.M = M;
  p.N = N;
  p.k_blocks = (K + kBK - 1) / kBK;
  const int tiles = (N + 127) / 128, mt = (M + NT - 1) / NT;
  few_splits(static_cast<int64_t>(tiles) * mt, p.k_blocks, di.num_sms, &p.splits, &p.kb_per_split);
  p.status = device_status_ptr();
  if (p.status == nullptr) return fail(DS_ERR_CUDA, "device status word unavailable");
  DS_CUDA(launch_chained(few_rows_kernel<NT, QUANT>, dim3(tiles * p.splits, mt), dim3(kFewThreads),
                         QUANT ? FewTile<NT>::smem_quant(p.kb_per_split) : FewTile<NT>::smem, s,
                         p.splits, tmW, tmX, p));
  return DS_OK;
}

int launch_many(const void* a, const float* sa, const void* w, const float* sw, void* out, int M,
                int N, int K, const DeviceInfo& di, cudaStream_t s) {
  CUtensorMap tmX, tmW, tmO;
  DS_TRY(tmap(&tmX, a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, M, K, kBK, 128));
  DS_TRY(tmap(&tmW, w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, N, K, kBK, 128));
  DS_TRY(tmap(&tmO, out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, M, N, 64, 32));
  ManyParams p{};
  p.sa = sa;
  p.sw = sw;
  p.M = M;
  p.N = N;
  p.k_blocks = (K + kBK - 1) / kBK;
  p.n_tiles = (N + 255) / 256;
  const int64_t tiles = static_cast<int64_t>(p.n_tiles) * ((M + 255) / 256);
  DS_REQUIRE(tiles < (1LL << 31), "int8_linear: too many tiles");
  p.tiles = static_cast<int>(tiles);
  p.status = device_status_ptr();
  if (p.status == nullptr) return fail(DS_ERR_CUDA, "device status word unavailable");
  DS_CUDA(launch_chained(many_rows_kernel, dim3(2 * std::min(p.tiles, g_pairs[di.device])),
                         dim3(kManyThreads), kManySmem, s, 2, tmX, tmW, tmO, p));
  return DS_OK;
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
  const uint4* src = static_cast<const uint4*>(x);
  uint2* dst = static_cast<uint2*>(q);
  const int k8 = K / 8, n = static_cast<int>(rows);
  const unsigned r = static_cast<unsigned>(rows), r8 = static_cast<unsigned>((rows + 7) / 8);
  if (rows >= 1024 && k8 <= 256) {  // a warp a row once there are rows enough to fill the SMs
    if (k8 <= 128) DS_CUDA(launch_chained(quantize_kernel<32, 4>, dim3(r8), dim3(256), 0, s, 1, src, ld / 8, n, k8,
                           dst, scale));
    else DS_CUDA(launch_chained(quantize_kernel<32, 8>, dim3(r8), dim3(256), 0, s, 1, src, ld / 8, n, k8,
                           dst, scale));
  } else if (k8 <= 256) {
    DS_CUDA(launch_chained(quantize_kernel<256, 1>, dim3(r), dim3(256), 0, s, 1, src, ld / 8, n, k8,
                           dst, scale));
  } else {
    DS_CUDA(launch_chained(quantize_kernel<256, 4>, dim3(r), dim3(256), 0, s, 1, src, ld / 8, n, k8,
                           dst, scale));
  }
  DS_LAUNCH_CHECK("quantize_kernel");
  return DS_OK;
}

int launch_gemm(const void* a, const float* sa, const void* w, const float* sw, void* out,
                int64_t M64, int N, int K, cudaStream_t s) {
  if (M64 == 0 || N == 0) return DS_OK;
  const int M = static_cast<int>(M64);
  DeviceInfo di;
  DS_TRY(device_info(&di));
  DS_TRY(set_attrs(di));
  int st;
  if (M <= 16) st = launch_few<16, false>(nullptr, 0, a, sa, w, sw, out, M, N, K, di, s);
  else if (M <= 32) st = launch_few<32, false>(nullptr, 0, a, sa, w, sw, out, M, N, K, di, s);
  else if (M <= 64) st = launch_few<64, false>(nullptr, 0, a, sa, w, sw, out, M, N, K, di, s);
  else if (!many_rows_faster(M, N, K, di.num_sms, g_pairs[di.device]))
    st = launch_few<128, false>(nullptr, 0, a, sa, w, sw, out, M, N, K, di, s);
  else st = launch_many(a, sa, w, sw, out, M, N, K, di, s);
  DS_TRY(st);
  DS_LAUNCH_CHECK("int8 product");
  return DS_OK;
}

// Rows that the product's kernel quantises itself, whatever the number of splits.
bool quantized_inside(int64_t M, int K) {
  return M <= kQuantRows && M * K <= kQuantHere && K <= kQuantBlocks * kBK;
}

size_t linear_workspace(int64_t M, int K) {
  if (quantized_inside(M, K)) return 0;
  return align_up(static_cast<size_t>(M) * K, 256) + align_up(static_cast<size_t>(M) * 4, 256);
}

int launch_linear(const void* x, int64_t ld, const void* w, const float* sw, void* out, int64_t M,
                  int N, int K, void* workspace, size_t ws_bytes, cudaStream_t s) {
  if (M <= kQuantRows && M * K <= kQuantHere && N > 0) {
    DeviceInfo di;
    DS_TRY(device_info(&di));
    DS_TRY(set_attrs(di));
    int splits, per;
    few_splits((N + 127) / 128, (K + kBK - 1) / kBK, di.num_sms, &splits, &per);
    if (per <= kQuantBlocks)
      return launch_few<16, true>(x, ld, nullptr, nullptr, w, sw, out, static_cast<int>(M), N, K,
                                  di, s);
  }
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
  DS_REQUIRE(x_bf16 && w_int8 && w_scale && out_bf16 &&
                 (workspace || ds::i8::linear_workspace(rows, in_features) == 0),
             "int8_linear: null pointer");
  DS_REQUIRE(row_stride >= in_features && row_stride % 8 == 0 && ds::aligned16(x_bf16) &&
                 ds::aligned16(w_int8) && ds::aligned16(out_bf16) && ds::aligned16(workspace),
             "int8_linear: x rows, w, out and workspace must be 16-byte aligned");
  return ds::i8::launch_linear(x_bf16, row_stride, w_int8, w_scale, out_bf16, rows, out_features,
                               in_features, workspace, workspace_bytes,
                               static_cast<cudaStream_t>(stream));
}

}  // extern "C"
