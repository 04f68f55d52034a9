// The latent KV cache held in 4 bits (additive; the bf16 cache it stands beside is that of
// src/kernels/mla_cache.py:29-219): filling it, reading it back, one decode step's attention
// over it, and eviction from it by accumulated attention weight.
//
// Per sequence and slot: 576 codes of 4 bits (512 of the raw latent, 64 of k_pe rotated at its
// position; value = (code - 8) * scale, dimension d in the low (even d) or high (odd d) half
// of byte d/2), one bf16 scale per group (four of 128 latent dimensions, one for k_pe; laid
// out [batch, 5, slots] so that neighbouring slots' scales are neighbours), rstd =
// rsqrt(mean(latent^2) + eps) of the latent before quantisation (f32), the position (int32)
// and the accumulated attention weight (f32): 310 bytes against 1156.
//   scale_g = bf16(max_g |v| / 7);  code = 8 + clamp(rint(v / scale_g), -7, 7), ties to even
// Symmetric 15-level codes: the tensor cores then take code - 8, an exact bf16, and a group's
// scale multiplies one probability instead of 128 values.  A group holding an infinity or a
// NaN gets scale NaN.  state[0..batch) holds the sequences' lengths in slots,
// state[batch..2 batch) their next positions (tokens seen, evicted ones included).
#include <cmath>

#include "kernels.cuh"
#include "ptx.cuh"

namespace ds {
namespace c4 {
namespace {

constexpr int kLatent = 512;
constexpr int kRope = 64;
constexpr int kQCols = kLatent + kRope;
constexpr int kRowBytes = kQCols / 2;  // 288
constexpr int kGroups = 5;
constexpr int kMaxHeads = 128;

struct Cache {
  uint8_t* codes;         // [batch, slots, 288]
  __nv_bfloat16* scales;  // [batch, 5, slots]
  float* rstd;            // [batch, slots]
  int32_t* pos;           // [batch, slots]
  float* mass;            // [batch, slots]
  int32_t* state;         // [2, batch]
  int batch, slots;
};

// 8 + clamp(rint(v / sigma), -7, 7) for bf16 v and sigma > 0; r ~ 1 / sigma.  v - n sigma is
// exact in f32 (8 and 4 + 8 significant bits of nearby size), so it decides borders and ties.
__device__ __forceinline__ uint32_t code1(float v, float sigma, float r) {
  float n = rintf(v * r);
  n = fminf(fmaxf(n, -8.f), 8.f);
  const float e = fmaf(-n, sigma, v);
  const float e2 = 2.f * fabsf(e);
  const bool odd = (static_cast<int>(n) & 1) != 0;
  if (e2 > sigma || (e2 == sigma && odd)) n += copysignf(1.f, e);
  n = fminf(fmaxf(n, -7.f), 7.f);
  return static_cast<uint32_t>(static_cast<int>(n) + 8);
}

// The bf16 scale of a group with largest magnitude a (a NaN or infinity inside: NaN).
__device__ __forceinline__ __nv_bfloat16 group_scale(float a) {
  return a <= 3.4e38f ? __float2bfloat16_rn(a / 7.f) : __ushort_as_bfloat16(0x7FC0);
}
__device__ __forceinline__ float abs_or_inf(float x) {
  return fabsf(x) <= 3.4e38f ? fabsf(x) : INFINITY;
}
// The scale as the quotients use it: 0 (all codes 8) for an empty or non-finite group; a group
// whose scale underflows to 0 reads back as zeros.
__device__ __forceinline__ float usable(__nv_bfloat16 sc) {
  const float s = __bfloat162float(sc);
  return s > 0.f ? s : 0.f;  // false for NaN
}

// One warp quantises one token into (b, slot): lane l holds latent dimensions 16 l .. 16 l +
// 15 (a group of 128 = 8 lanes) and the rotation pair l of k_pe.
__device__ __forceinline__ void put_token(const Cache& c, int b, int slot, int position,
                                          const __nv_bfloat16* lat, const __nv_bfloat16* kpe,
                                          const __nv_bfloat16* cos_t, const __nv_bfloat16* sin_t,
                                          int table_rows, float eps) {
  const int lane = threadIdx.x & 31;
  const uint4* l4 = reinterpret_cast<const uint4*>(lat) + 2 * lane;
  const uint4 a0 = l4[0], a1 = l4[1];
  const __nv_bfloat162 kp = reinterpret_cast<const __nv_bfloat162*>(kpe)[lane];
  const uint32_t w[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
  float v[16];
  float amax = 0.f, ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    amax = fmaxf(amax, fmaxf(abs_or_inf(v[2 * i]), abs_or_inf(v[2 * i + 1])));
    ss = fmaf(v[2 * i], v[2 * i], fmaf(v[2 * i + 1], v[2 * i + 1], ss));
  }
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
  const __nv_bfloat16 sc = group_scale(amax);
  const float sg = usable(sc);
  // a subnormal scale's reciprocal would overflow: scale both by 2^64
  const float up = sg < 1e-30f ? 1.8446744e19f : 1.f;
  const float r = sg > 0.f ? 1.f / (sg * up) : 0.f;
  uint2 packed = make_uint2(0u, 0u);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const uint32_t n = r > 0.f ? code1(v[i] * up, sg * up, r) : 8u;
    if (i < 8) packed.x |= n << (4 * i);
    else packed.y |= n << (4 * (i - 8));
  }
  // k_pe at its position: the interleave -> half RoPE of src/reference/mla.py:176-206
  const int prow = min(position, table_rows - 1);
  const __nv_bfloat16* cr = cos_t + static_cast<int64_t>(prow) * kRope;
  const __nv_bfloat16* sr = sin_t + static_cast<int64_t>(prow) * kRope;
  const float xa = __low2float(kp), xb = __high2float(kp);
  // both products are exact in f32, so the sums round once, contracted or not
  const float r0 = __bfloat162float(__float2bfloat16_rn(xa * __bfloat162float(cr[lane]) -
                                                        xb * __bfloat162float(sr[lane])));
  const float r1 = __bfloat162float(__float2bfloat16_rn(xb * __bfloat162float(cr[32 + lane]) +
                                                        xa * __bfloat162float(sr[32 + lane])));
  float ka = fmaxf(abs_or_inf(r0), abs_or_inf(r1));
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) ka = fmaxf(ka, __shfl_xor_sync(0xffffffffu, ka, d));
  const __nv_bfloat16 ksc = group_scale(ka);
  const float kg = usable(ksc);
  const float kup = kg < 1e-30f ? 1.8446744e19f : 1.f;
  const float kr = kg > 0.f ? 1.f / (kg * kup) : 0.f;
  const uint32_t c0 = kr > 0.f ? code1(r0 * kup, kg * kup, kr) : 8u;
  const uint32_t c1 = kr > 0.f ? code1(r1 * kup, kg * kup, kr) : 8u;
  const uint32_t n0 = __shfl_down_sync(0xffffffffu, c0, 1);
  const uint32_t n1 = __shfl_down_sync(0xffffffffu, c1, 1);
  const int64_t row = static_cast<int64_t>(b) * c.slots + slot;
  uint8_t* dst = c.codes + row * kRowBytes;
  reinterpret_cast<uint2*>(dst)[lane] = packed;
  if ((lane & 1) == 0) {  // byte d/2 of dimensions d = lane, lane + 1 (and 32 above)
    dst[kLatent / 2 + lane / 2] = static_cast<uint8_t>(c0 | (n0 << 4));
    dst[kLatent / 2 + 16 + lane / 2] = static_cast<uint8_t>(c1 | (n1 << 4));
  }
  __nv_bfloat16* sd = c.scales + static_cast<int64_t>(b) * kGroups * c.slots + slot;
  if ((lane & 7) == 0) sd[static_cast<int64_t>(lane >> 3) * c.slots] = sc;
  if (lane == 0) {
    sd[static_cast<int64_t>(4) * c.slots] = ksc;
    c.rstd[row] = rsqrtf(ss / kLatent + eps);
    c.pos[row] = position;
    c.mass[row] = 0.f;
  }
}

// n_new tokens of each sequence (new_lens[b] of them when given) behind its last slot; a warp
// per token.  `advance`: one block holds all of a sequence's tokens and moves its length on.
__global__ void __launch_bounds__(256)
    append_kernel(Cache c, const __nv_bfloat16* __restrict__ lat, int64_t lat_ld,
                  const __nv_bfloat16* __restrict__ kpe, int64_t kpe_ld, int64_t src_bstride,
                  int n_new, const int32_t* __restrict__ new_lens,
                  const __nv_bfloat16* __restrict__ cos_t, const __nv_bfloat16* __restrict__ sin_t,
                  int table_rows, float eps, int advance) {
  const int b = blockIdx.y;
  const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int len = c.state[b], next = c.state[c.batch + b];
  const int n = new_lens != nullptr ? min(n_new, __ldg(new_lens + b)) : n_new;
  if (i < n && len >= 0 && len + i < c.slots) {
    const int64_t src = static_cast<int64_t>(b) * src_bstride + i;
    put_token(c, b, len + i, next + i, lat + src * lat_ld, kpe + src * kpe_ld, cos_t, sin_t,
              table_rows, eps);
  }
  if (advance) {
    __syncthreads();  // every warp has read the length
    if (threadIdx.x == 0) {
      const int add = max(0, min(n, c.slots - len));
      c.state[b] = len + add;
      c.state[c.batch + b] = next + add;
    }
  }
}

__global__ void advance_kernel(Cache c, int n_new, const int32_t* __restrict__ new_lens) {
  const int b = blockIdx.x * blockDim.x + threadIdx.x;
  if (b >= c.batch) return;
  const int n = new_lens != nullptr ? min(n_new, __ldg(new_lens + b)) : n_new;
  const int add = max(0, min(n, c.slots - c.state[b]));
  c.state[b] += add;
  c.state[c.batch + b] += add;
}

// Eight codes of one word -> eight bf16 values code * scale (rounded once).
__device__ __forceinline__ uint4 values8(uint32_t w, float s) {
  uint4 o;
  uint32_t* u = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = static_cast<float>(static_cast<int>((w >> (8 * i)) & 15u) - 8) * s;
    const float hi = static_cast<float>(static_cast<int>((w >> (8 * i + 4)) & 15u) - 8) * s;
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    u[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return o;
}

// Slots 0 .. n-1 of every sequence as bf16 values, zeros from its length on; a warp per slot.
__global__ void __launch_bounds__(256)
    get_kernel(Cache c, int n, uint4* __restrict__ lat, uint4* __restrict__ kpe) {
  const int lane = threadIdx.x & 31;
  const int64_t i = blockIdx.x * static_cast<int64_t>(8) + (threadIdx.x >> 5);
  if (i >= static_cast<int64_t>(c.batch) * n) return;
  const int b = static_cast<int>(i / n), t = static_cast<int>(i - static_cast<int64_t>(b) * n);
  uint4 v0 = make_uint4(0, 0, 0, 0), v1 = v0, v2 = v0;
  if (t < c.state[b]) {
    const int64_t row = static_cast<int64_t>(b) * c.slots + t;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(c.codes + row * kRowBytes);
    const __nv_bfloat16* s = c.scales + static_cast<int64_t>(b) * kGroups * c.slots + t;
    v0 = values8(w[lane], __bfloat162float(s[static_cast<int64_t>(lane >> 4) * c.slots]));
    v1 = values8(w[32 + lane], __bfloat162float(s[static_cast<int64_t>(2 + (lane >> 4)) * c.slots]));
    if (lane < 8)
      v2 = values8(w[64 + lane], __bfloat162float(s[static_cast<int64_t>(4) * c.slots]));
  }
  lat[i * 64 + lane] = v0;
  lat[i * 64 + 32 + lane] = v1;
  if (lane < 8) kpe[i * 8 + lane] = v2;
}

// ---- attention ------------------------------------------------------------------------------
// Partials of (sequence, split): o f32 [batch][nsplit][heads][512], then maximum (log2 domain)
// and sum f32 [batch][nsplit][2][heads].  With scores set, s * log2(e) of every slot goes to
// scores [batch][heads][slots].
struct AttnParams {
  Cache c;
  const __nv_bfloat16* q;  // [batch, heads, 576]
  int heads, nsplit, split_tokens;
  float scale_log2;
  float* part_o;
  float* part_ml;
  float* scores;
};

__global__ void __launch_bounds__(256) attend4_kernel(const AttnParams p) {
  const Cache& c = p.c;
  __shared__ float so[8][kLatent];
  __shared__ float sm[8], sl[8];
  const int bh = blockIdx.x, b = bh / p.heads, h = bh - b * p.heads;
  const int split = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int len = min(c.state[b], c.slots);
  const int t0 = split * p.split_tokens, t1 = min(len, t0 + p.split_tokens);
  const __nv_bfloat16* q = p.q + static_cast<int64_t>(bh) * kQCols;
  float ql[16], qr[2], o[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    ql[i] = __bfloat162float(q[16 * lane + i]) * p.scale_log2;
    o[i] = 0.f;
  }
  qr[0] = __bfloat162float(q[kLatent + 2 * lane]) * p.scale_log2;
  qr[1] = __bfloat162float(q[kLatent + 2 * lane + 1]) * p.scale_log2;
  float m = -INFINITY, l = 0.f;
  const __nv_bfloat16* sc = c.scales + static_cast<int64_t>(b) * kGroups * c.slots;
  for (int t = t0 + warp; t < t1; t += 8) {
    const int64_t row = static_cast<int64_t>(b) * c.slots + t;
    const uint2 w = *reinterpret_cast<const uint2*>(c.codes + row * kRowBytes + 8 * lane);
    const uint32_t wr = c.codes[row * kRowBytes + kLatent / 2 + lane];
    const float sg = __bfloat162float(sc[static_cast<int64_t>(lane >> 3) * c.slots + t]) *
                     c.rstd[row];
    const float sr = __bfloat162float(sc[static_cast<int64_t>(4) * c.slots + t]);
    float v[16], dot = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t x = ((i < 8 ? w.x : w.y) >> (4 * (i & 7))) & 15u;
      v[i] = static_cast<float>(static_cast<int>(x) - 8) * sg;
      dot = fmaf(v[i], ql[i], dot);
    }
    dot += sr * (static_cast<float>(static_cast<int>(wr & 15u) - 8) * qr[0] +
                 static_cast<float>(static_cast<int>(wr >> 4) - 8) * qr[1]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if (p.scores != nullptr && lane == 0)
      p.scores[static_cast<int64_t>(bh) * c.slots + t] = dot;
    const float mn = fmaxf(m, dot);
    const float ref = mn == -INFINITY ? 0.f : mn;  // a NaN score stays one
    const float f = exp2f(m - ref);
    const float pr = exp2f(dot - ref);
    l = l * f + pr;
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = fmaf(pr, v[i], o[i] * f);
    m = mn;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) so[warp][16 * lane + i] = o[i];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  float M = -INFINITY, L = 0.f, f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) M = fmaxf(M, sm[i]);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = exp2f(sm[i] - (M == -INFINITY ? 0.f : M));
    L += sl[i] * f[i];
  }
  const int64_t part = static_cast<int64_t>(b) * p.nsplit + split;
  for (int d = threadIdx.x; d < kLatent; d += 256) {
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a += so[i][d] * f[i];
    p.part_o[(part * p.heads + h) * kLatent + d] = a;
  }
  if (threadIdx.x == 0) {
    p.part_ml[(part * 2) * p.heads + h] = M;
    p.part_ml[(part * 2 + 1) * p.heads + h] = L;
  }
}

// Merge the splits of each (sequence, head); lse[b, h] = M + log2 L for the weights.
__global__ void __launch_bounds__(128)
    merge_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, int nsplit,
                 int heads, __nv_bfloat16* __restrict__ out, float* __restrict__ lse) {
  const int64_t b = blockIdx.x / heads;
  const int h = blockIdx.x - static_cast<int>(b) * heads;
  float M = -INFINITY;
  for (int s = 0; s < nsplit; ++s)
    M = fmaxf(M, __ldg(part_ml + (b * nsplit + s) * 2 * heads + h));
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < nsplit; ++s) {
    const float* ml = part_ml + (b * nsplit + s) * 2 * heads;
    const float ls = __ldg(ml + heads + h);
    if (ls == 0.f) continue;
    const float w = ptx::ex2(__ldg(ml + h) - ref);
    L = fmaf(w, ls, L);
    const float* po = part_o + ((b * nsplit + s) * heads + h) * kLatent;
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = fmaf(w, __ldg(po + k * 128 + threadIdx.x), acc[k]);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;  // no slot: zeros
  __nv_bfloat16* o = out + (b * heads + h) * kLatent;
#pragma unroll
  for (int k = 0; k < 4; ++k) o[k * 128 + threadIdx.x] = __float2bfloat16_rn(acc[k] * inv);
  if (lse != nullptr && threadIdx.x == 0) lse[b * heads + h] = M + log2f(L);
}

// mass[b, t] = decay * mass[b, t] + sum_h 2^(s_h(t) - lse_h) (decay 0: not read), t < length.
__global__ void __launch_bounds__(256)
    mass_kernel(Cache c, const float* __restrict__ scores, const float* __restrict__ lse,
                int heads, float decay) {
  __shared__ float sl[kMaxHeads];
  const int b = blockIdx.y;
  const int t = blockIdx.x * 256 + threadIdx.x;
  const int len = min(c.state[b], c.slots);
  if (blockIdx.x * 256 >= len) return;
  for (int h = threadIdx.x; h < heads; h += 256) sl[h] = lse[static_cast<int64_t>(b) * heads + h];
  __syncthreads();
  if (t >= len) return;
  const float* s = scores + static_cast<int64_t>(b) * heads * c.slots + t;
  float a = 0.f;
  for (int h = 0; h < heads; ++h) a += ptx::ex2(__ldg(s + static_cast<int64_t>(h) * c.slots) - sl[h]);
  float* m = c.mass + static_cast<int64_t>(b) * c.slots + t;
  *m = decay != 0.f ? fmaf(decay, *m, a) : a;
}

// ---- eviction -------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t evict_key(float mass, int pos, int newest_from) {
  if (pos >= newest_from) return 0xFFFFFFFFu;  // protected: above +inf
  if (isnan(mass)) return 0u;                  // below -inf
  const uint32_t u = __float_as_uint(mass + 0.f);  // -0 counts as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Exclusive prefix of `flag` over the block in thread order; total in *total.
__device__ __forceinline__ int block_rank(bool flag, int* warp_sum, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned m = __ballot_sync(0xffffffffu, flag);
  if (lane == 0) warp_sum[warp] = __popc(m);
  __syncthreads();
  int base = 0, all = 0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) {
    if (i < warp) base += warp_sum[i];
    all += warp_sum[i];
  }
  __syncthreads();
  *total = all;
  return base + __popc(m & ((1u << lane) - 1u));
}

// One block per sequence: the budget-th largest key by four 8-bit radix passes, ties to the
// lowest slots, then src_of[b, j] = the slot whose row result slot j takes: itself where slot
// j < budget stays, else the next survivor from behind the budget, both in ascending order.
__global__ void __launch_bounds__(1024)
    evict_plan_kernel(Cache c, int32_t* __restrict__ dst_state, int budget, int recent,
                      int32_t* __restrict__ src_of, int32_t* __restrict__ holes) {
  __shared__ int hist[256];
  __shared__ int warp_sum[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int b = blockIdx.x;
  const int len = min(max(c.state[b], 0), c.slots), next = c.state[c.batch + b];
  const float* mass = c.mass + static_cast<int64_t>(b) * c.slots;
  const int32_t* pos = c.pos + static_cast<int64_t>(b) * c.slots;
  int32_t* src = src_of + static_cast<int64_t>(b) * budget;
  int32_t* hole = holes + static_cast<int64_t>(b) * budget;
  const int kept_n = min(len, budget);
  for (int j = threadIdx.x; j < kept_n; j += blockDim.x) src[j] = j;
  if (len > budget) {
    const int from = next - recent;
    uint32_t prefix = 0, mask = 0;
    int need = budget;  // how many of the keys with this prefix are kept
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += blockDim.x) hist[i] = 0;
      __syncthreads();
      for (int t = threadIdx.x; t < len; t += blockDim.x) {
        const uint32_t k = evict_key(mass[t], pos[t], from);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        int left = need, d = 255;
        while (d > 0 && hist[d] < left) left -= hist[d--];
        s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
        s_need = left;
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
      mask |= 255u << shift;
    }
    // keys above `prefix` stay, and the first `need` slots of those equal to it
    int eq = 0, nh = 0, ns = 0;
    const int tiles = (len + 1023) / 1024;
    for (int pass = 0; pass < 2; ++pass) {
      eq = 0;
      for (int tile = 0; tile < tiles; ++tile) {
        const int t = tile * 1024 + threadIdx.x;
        const bool in = t < len;
        const uint32_t k = in ? evict_key(mass[t], pos[t], from) : 0u;
        const bool tie = in && k == prefix;
        int tot;
        const int r = eq + block_rank(tie, warp_sum, &tot);
        eq += tot;
        const bool keep = in && (k > prefix || (tie && r < need));
        if (pass == 0) {
          const bool h = in && t < budget && !keep;
          const int hr = nh + block_rank(h, warp_sum, &tot);
          nh += tot;
          if (h) hole[hr] = t;
        } else {
          const bool sv = keep && t >= budget;
          const int sr = ns + block_rank(sv, warp_sum, &tot);
          ns += tot;
          if (sv) src[hole[sr]] = t;
        }
      }
      __syncthreads();  // the holes are written before survivors are paired with them
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    dst_state[b] = kept_n;
    dst_state[c.batch + b] = next;
  }
}

// Result slot j of sequence b takes row src_of[b, j] (a warp per row; in place, rows that
// stay are skipped: sources are at or behind the budget and targets before it, so no row
// is both).
__global__ void __launch_bounds__(256)
    evict_move_kernel(Cache s, Cache d, int budget, const int32_t* __restrict__ src_of,
                      int in_place) {
  const int b = blockIdx.y;
  const int j = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (j >= d.state[b]) return;
  const int t = src_of[static_cast<int64_t>(b) * budget + j];
  if (in_place && t == j) return;
  const int64_t sr = static_cast<int64_t>(b) * s.slots + t;
  const int64_t dr = static_cast<int64_t>(b) * d.slots + j;
  if (lane < kRowBytes / 16)
    reinterpret_cast<uint4*>(d.codes + dr * kRowBytes)[lane] =
        reinterpret_cast<const uint4*>(s.codes + sr * kRowBytes)[lane];
  if (lane >= 18 && lane < 23) {
    const int64_t g = lane - 18;
    d.scales[(static_cast<int64_t>(b) * kGroups + g) * d.slots + j] =
        s.scales[(static_cast<int64_t>(b) * kGroups + g) * s.slots + t];
  }
  if (lane == 23) d.rstd[dr] = s.rstd[sr];
  if (lane == 24) d.pos[dr] = s.pos[sr];
  if (lane == 25) d.mass[dr] = s.mass[sr];
}

Cache cache_of(void* codes, void* scales, float* rstd, int32_t* pos, float* mass, int32_t* state,
               int batch, int slots) {
  Cache c{};
  c.codes = static_cast<uint8_t*>(codes);
  c.scales = static_cast<__nv_bfloat16*>(scales);
  c.rstd = rstd;
  c.pos = pos;
  c.mass = mass;
  c.state = state;
  c.batch = batch;
  c.slots = slots;
  return c;
}

int check_cache(const Cache& c, const char* op) {
  DS_REQUIRE(c.batch >= 0 && c.batch <= 65535 && c.slots > 0 && c.slots % 64 == 0,
             "%s: batch must be at most 65535 and slots a positive multiple of 64", op);
  if (c.batch == 0) return DS_OK;
  DS_REQUIRE(c.codes && c.scales && c.rstd && c.pos && c.mass && c.state, "%s: null pointer", op);
  DS_REQUIRE(aligned16(c.codes) && aligned16(c.scales) && aligned16(c.rstd),
             "%s: the cache arrays must be 16-byte aligned", op);
  return DS_OK;
}

int split_count(int batch, int heads, int max_len, int num_sms, int* tokens) {
  (void)batch;
  (void)heads;
  (void)num_sms;
  *tokens = 1024;
  const int n = (max_len + *tokens - 1) / *tokens;
  return n < 1 ? 1 : n;
}

struct AttnBuffers {
  float* part_o;
  float* part_ml;
  float* scores;
  float* lse;
};

void carve_attn(Carve& w, AttnBuffers* b, int batch, int heads, int slots, int nsplit,
                bool mass) {
  b->part_o = w.take<float>(static_cast<size_t>(batch) * nsplit * heads * kLatent);
  b->part_ml = w.take<float>(static_cast<size_t>(batch) * nsplit * 2 * heads);
  b->scores = mass ? w.take<float>(static_cast<size_t>(batch) * heads * slots) : nullptr;
  b->lse = mass ? w.take<float>(static_cast<size_t>(batch) * heads) : nullptr;
}

int launch_append(const Cache& c, const void* lat, int64_t lat_ld, const void* kpe,
                  int64_t kpe_ld, int64_t src_bstride, int n_new, const int32_t* new_lens,
                  const void* cos_t, const void* sin_t, int table_rows, float eps,
                  cudaStream_t s) {
  if (c.batch == 0 || n_new == 0) return DS_OK;
  const int gx = (n_new + 7) / 8;
  append_kernel<<<dim3(gx, c.batch), 256, 0, s>>>(
      c, static_cast<const __nv_bfloat16*>(lat), lat_ld, static_cast<const __nv_bfloat16*>(kpe),
      kpe_ld, src_bstride, n_new, new_lens, static_cast<const __nv_bfloat16*>(cos_t),
      static_cast<const __nv_bfloat16*>(sin_t), table_rows, eps, gx == 1 ? 1 : 0);
  DS_LAUNCH_CHECK("append_kernel");
  if (gx > 1) {
    advance_kernel<<<(c.batch + 255) / 256, 256, 0, s>>>(c, n_new, new_lens);
    DS_LAUNCH_CHECK("advance_kernel");
  }
  return DS_OK;
}

int launch_attention(const Cache& c, const void* q, int heads, int max_len, float softmax_scale,
                     int accumulate, float decay, void* out, void* workspace, size_t ws_bytes,
                     cudaStream_t s) {
  if (c.batch == 0) return DS_OK;
  DeviceInfo di;
  DS_TRY(device_info(&di));
  AttnParams p{};
  p.nsplit = split_count(c.batch, heads, max_len, di.num_sms, &p.split_tokens);
  Carve w(workspace, ws_bytes);
  AttnBuffers b{};
  carve_attn(w, &b, c.batch, heads, c.slots, p.nsplit, accumulate != 0);
  if (!w.ok())
    return fail(DS_ERR_WORKSPACE, "mla_decode_attention4: workspace needs %zu bytes", w.used);
  p.c = c;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.heads = heads;
  p.scale_log2 = static_cast<float>(static_cast<double>(softmax_scale) * 1.4426950408889634);
  p.part_o = b.part_o;
  p.part_ml = b.part_ml;
  p.scores = b.scores;
  attend4_kernel<<<dim3(c.batch * heads, p.nsplit), 256, 0, s>>>(p);
  DS_LAUNCH_CHECK("attend4_kernel");
  merge_kernel<<<c.batch * heads, 128, 0, s>>>(b.part_o, b.part_ml, p.nsplit, heads,
                                               static_cast<__nv_bfloat16*>(out), b.lse);
  DS_LAUNCH_CHECK("merge_kernel");
  if (accumulate && max_len > 0) {
    mass_kernel<<<dim3((max_len + 255) / 256, c.batch), 256, 0, s>>>(c, b.scores, b.lse, heads,
                                                                     decay);
    DS_LAUNCH_CHECK("mass_kernel");
  }
  return DS_OK;
}

}  // namespace
}  // namespace c4
}  // namespace ds

// ---- C ABI ------------------------------------------------------------------------------------
extern "C" {

int ds_mla_cache4_append(const void* latent_bf16, int64_t latent_ld, const void* kpe_bf16,
                         int64_t kpe_ld, int64_t src_rows_per_seq, int new_tokens,
                         const int32_t* new_lens, const void* cos_bf16, const void* sin_bf16,
                         int table_rows, float eps, void* codes, void* scales_bf16, float* rstd,
                         int32_t* pos, float* mass, int32_t* state, int batch, int slots,
                         void* stream) {
  const ds::c4::Cache c =
      ds::c4::cache_of(codes, scales_bf16, rstd, pos, mass, state, batch, slots);
  DS_TRY(ds::c4::check_cache(c, "mla_cache4_append"));
  DS_REQUIRE(new_tokens >= 0 && table_rows > 0, "mla_cache4_append: bad shape");
  DS_REQUIRE(new_tokens <= slots, "mla_cache4_append: cache overflow");
  if (batch == 0 || new_tokens == 0) return DS_OK;
  DS_REQUIRE(latent_bf16 && kpe_bf16 && cos_bf16 && sin_bf16, "mla_cache4_append: null pointer");
  DS_REQUIRE(latent_ld % 8 == 0 && kpe_ld % 8 == 0 && ds::aligned16(latent_bf16) &&
                 ds::aligned16(kpe_bf16),
             "mla_cache4_append: rows must start on 16-byte boundaries");
  return ds::c4::launch_append(c, latent_bf16, latent_ld, kpe_bf16, kpe_ld, src_rows_per_seq,
                               new_tokens, new_lens, cos_bf16, sin_bf16, table_rows, eps,
                               static_cast<cudaStream_t>(stream));
}

int ds_mla_cache4_get(const void* codes, const void* scales_bf16, const int32_t* state, int batch,
                      int slots, int seq_len, void* latent_out_bf16, void* kpe_out_bf16,
                      void* stream) {
  DS_REQUIRE(batch >= 0 && seq_len >= 0 && seq_len <= slots && slots > 0 && slots % 64 == 0,
             "mla_cache4_get: bad shape");
  const int64_t rows = static_cast<int64_t>(batch) * seq_len;
  if (rows == 0) return DS_OK;
  DS_REQUIRE(codes && scales_bf16 && state && latent_out_bf16 && kpe_out_bf16,
             "mla_cache4_get: null pointer");
  DS_REQUIRE(ds::aligned16(codes) && ds::aligned16(latent_out_bf16) && ds::aligned16(kpe_out_bf16),
             "mla_cache4_get: 16-byte aligned pointers");
  DS_REQUIRE((rows + 7) / 8 < (1LL << 31), "mla_cache4_get: too many rows");
  const ds::c4::Cache c = ds::c4::cache_of(const_cast<void*>(codes), const_cast<void*>(scales_bf16),
                                           nullptr, nullptr, nullptr,
                                           const_cast<int32_t*>(state), batch, slots);
  ds::c4::get_kernel<<<static_cast<unsigned>((rows + 7) / 8), 256, 0,
                       static_cast<cudaStream_t>(stream)>>>(
      c, seq_len, static_cast<uint4*>(latent_out_bf16), static_cast<uint4*>(kpe_out_bf16));
  DS_LAUNCH_CHECK("get_kernel");
  return DS_OK;
}

size_t ds_mla_decode_attention4_workspace_size(int batch, int heads, int slots, int max_len,
                                               int accumulate) {
  if (batch <= 0 || heads <= 0 || max_len < 0) return 0;
  ds::DeviceInfo di;
  if (ds::device_info(&di) != DS_OK) return 0;
  int tokens;
  const int ns = ds::c4::split_count(batch, heads, max_len, di.num_sms, &tokens);
  ds::Carve w(nullptr, 0);
  ds::c4::AttnBuffers b{};
  ds::c4::carve_attn(w, &b, batch, heads, slots, ns, accumulate != 0);
  return ds::align_up(w.used, 256);
}

int ds_mla_decode_attention4(const void* q_bf16, int heads, const void* codes,
                             const void* scales_bf16, const float* rstd, float* mass,
                             const int32_t* state, int batch, int slots, int max_len,
                             float softmax_scale, int accumulate, float mass_decay,
                             void* out_bf16, void* workspace, size_t workspace_bytes,
                             void* stream) {
  const ds::c4::Cache c = ds::c4::cache_of(
      const_cast<void*>(codes), const_cast<void*>(scales_bf16), const_cast<float*>(rstd),
      const_cast<int32_t*>(state), mass, const_cast<int32_t*>(state), batch, slots);
  DS_REQUIRE(heads >= 1 && heads <= ds::c4::kMaxHeads,
             "mla_decode_attention4: heads=%d outside [1, %d]", heads, ds::c4::kMaxHeads);
  DS_TRY(ds::c4::check_cache(c, "mla_decode_attention4"));
  DS_REQUIRE(max_len >= 0 && max_len <= slots, "mla_decode_attention4: max_len outside the cache");
  if (batch == 0) return DS_OK;
  DS_REQUIRE(q_bf16 && out_bf16 && workspace, "mla_decode_attention4: null pointer");
  DS_REQUIRE(ds::aligned16(q_bf16) && ds::aligned16(out_bf16) && ds::aligned16(workspace),
             "mla_decode_attention4: q, out and workspace must be 16-byte aligned");
  return ds::c4::launch_attention(c, q_bf16, heads, max_len, softmax_scale, accumulate, mass_decay,
                                  out_bf16, workspace, workspace_bytes,
                                  static_cast<cudaStream_t>(stream));
}

size_t ds_mla_cache4_evict_workspace_size(int batch, int budget) {
  if (batch <= 0 || budget <= 0) return 0;
  return 2 * ds::align_up(static_cast<size_t>(batch) * budget * 4, 256);
}

int ds_mla_cache4_evict(void* codes, void* scales_bf16, float* rstd, int32_t* pos, float* mass,
                        int32_t* state, int batch, int slots, int budget, int recent,
                        void* dst_codes, void* dst_scales_bf16, float* dst_rstd, int32_t* dst_pos,
                        float* dst_mass, int32_t* dst_state, int dst_slots, void* workspace,
                        size_t workspace_bytes, void* stream) {
  const ds::c4::Cache s =
      ds::c4::cache_of(codes, scales_bf16, rstd, pos, mass, state, batch, slots);
  const ds::c4::Cache d = ds::c4::cache_of(dst_codes, dst_scales_bf16, dst_rstd, dst_pos,
                                           dst_mass, dst_state, batch, dst_slots);
  DS_TRY(ds::c4::check_cache(s, "mla_cache4_evict"));
  DS_TRY(ds::c4::check_cache(d, "mla_cache4_evict"));
  DS_REQUIRE(budget >= 1 && budget <= dst_slots, "mla_cache4_evict: budget outside the cache");
  DS_REQUIRE(recent >= 0 && recent <= budget, "mla_cache4_evict: recent must be in [0, budget]");
  if (batch == 0) return DS_OK;
  const bool in_place = dst_codes == codes;
  DS_REQUIRE(in_place ? (dst_scales_bf16 == scales_bf16 && dst_rstd == rstd && dst_pos == pos &&
                         dst_mass == mass && dst_state == state && dst_slots == slots)
                      : (dst_scales_bf16 != scales_bf16 && dst_rstd != rstd && dst_pos != pos &&
                         dst_mass != mass && dst_state != state),
             "mla_cache4_evict: the result must be the cache itself or share nothing with it");
  ds::Carve w(workspace, workspace_bytes);
  int32_t* src_of = w.take<int32_t>(static_cast<size_t>(batch) * budget);
  int32_t* holes = w.take<int32_t>(static_cast<size_t>(batch) * budget);
  if (!w.ok())
    return ds::fail(DS_ERR_WORKSPACE, "mla_cache4_evict: workspace needs %zu bytes", w.used);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ds::c4::evict_plan_kernel<<<batch, 1024, 0, st>>>(s, dst_state, budget, recent, src_of, holes);
  DS_LAUNCH_CHECK("evict_plan_kernel");
  ds::c4::evict_move_kernel<<<dim3((budget + 7) / 8, batch), 256, 0, st>>>(s, d, budget, src_of,
                                                                           in_place ? 1 : 0);
  DS_LAUNCH_CHECK("evict_move_kernel");
  return DS_OK;
}

}  // extern "C"
