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
// NaN gets scale NaN.  state[0..batch) holds the sequences' lengths in slots, state[batch..2
// batch) their next positions (tokens seen, evicted ones included), the third row counters that
// are zero between calls.
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "kernels.cuh"
#include "partials.h"
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
  int32_t* state;         // [3, batch]
  int batch, slots;
};

// Codes 8 + clamp(rint(v / sigma), -7, 7) of bf16 values.  With 1 / sigma = rh + rl to twice
// f32's bits, fmaf(v, rh, v rl) is v / sigma rounded once: a tie stays a tie, and no other quotient
// of two 8-bit significands comes near one.  Adding 1.5 * 2^23 + 8 rounds (ties to even) into
// the low bits.  The clamp is for scales that lost bits to underflow: otherwise |v| / sigma is at
// most 7 (1 + 2^-8).
struct Quant {
  float up, rh, rl;  // 0 where all codes are 8: an empty or non-finite group
};
__device__ __forceinline__ Quant quant_of(float sigma) {
  Quant q;
  q.up = sigma < 1e-30f ? 0x1p64f : 1.f;  // a subnormal scale's reciprocal would overflow
  const float s = sigma * q.up;
  q.rh = s > 0.f ? 1.f / s : 0.f;
  q.rl = s > 0.f ? fmaf(-q.rh, s, 1.f) * q.rh : 0.f;
  return q;
}
constexpr float kRound8 = 12582920.f;          // 1.5 * 2^23 + 8
constexpr uint32_t kRoundBits = 0x4B400000u;   // its bits, less 8
template <bool TINY>
__device__ __forceinline__ uint32_t code_bits(float v, const Quant& q) {  // kRoundBits + code
  if (TINY) v *= q.up;
  float t = fmaf(v, q.rh, v * q.rl);
  if (TINY) t = fminf(fmaxf(t, -7.f), 7.f);
  return __float_as_uint(t + kRound8);
}
// Eight codes, the first in the low nibble: one shifted addition each; what kRoundBits adds is
// known, and taken off at the end.
template <bool TINY>
__device__ __forceinline__ uint32_t codes8(const float* v, const Quant& q) {
  uint32_t w = 0, off = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w += code_bits<TINY>(v[i], q) << (4 * i);
    off += kRoundBits << (4 * i);
  }
  return q.rh == 0.f ? 0x88888888u : w - off;
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

// The RoPE tables' row of a position, which stands in an array that the caller may write.
__device__ __forceinline__ int table_row(int position, int rows) {
  return min(max(position, 0), rows - 1);
}

// One warp quantises one token into (b, slot): lane l holds latent dimensions 16 l .. 16 l +
// 15 (a group of 128 = 8 lanes) and the rotation pair l of k_pe.
struct Token {
  uint4 a0, a1;
  __nv_bfloat162 kp;
};
__device__ __forceinline__ Token load_token(const __nv_bfloat16* lat, const __nv_bfloat16* kpe) {
  const int lane = threadIdx.x & 31;
  Token t;
  t.a0 = *(reinterpret_cast<const uint4*>(lat) + 2 * lane);
  t.a1 = *(reinterpret_cast<const uint4*>(lat) + 2 * lane + 1);
  t.kp = *(reinterpret_cast<const __nv_bfloat162*>(kpe) + lane);
  return t;
}
__device__ __forceinline__ void put_token(const Cache& c, int b, int slot, int position,
                                          const Token& tok, const __nv_bfloat16* cos_t,
                                          const __nv_bfloat16* sin_t, int table_rows, float eps) {
  const int lane = threadIdx.x & 31;
  const uint4 a0 = tok.a0, a1 = tok.a1;
  const __nv_bfloat162 kp = tok.kp;
  const uint32_t w[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
  float v[16];
  float ss = 0.f;
  uint32_t m2 = 0;  // the largest magnitudes as bit patterns, two to a word
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    ss = fmaf(v[2 * i], v[2 * i], fmaf(v[2 * i + 1], v[2 * i + 1], ss));
    m2 = __vmaxu2(m2, w[i] & 0x7FFF7FFFu);
  }
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) m2 = __vmaxu2(m2, __shfl_xor_sync(0xffffffffu, m2, d));
  const float amax = __uint_as_float(max(m2 & 0xFFFFu, m2 >> 16) << 16);  // (NaN, inf: not finite)
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
  const __nv_bfloat16 sc = group_scale(amax);
  const Quant qs = quant_of(usable(sc));
  uint2 packed;
  if (__any_sync(0xffffffffu, qs.up != 1.f))  // (rare)
    packed = make_uint2(codes8<true>(v, qs), codes8<true>(v + 8, qs));
  else
    packed = make_uint2(codes8<false>(v, qs), codes8<false>(v + 8, qs));
  // k_pe at its position: the interleave -> half RoPE of src/reference/mla.py:176-206
  const int prow = table_row(position, table_rows);
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
  const Quant kq = quant_of(usable(ksc));
  const uint32_t c0 = kq.rh == 0.f ? 8u : code_bits<true>(r0, kq) - kRoundBits;
  const uint32_t c1 = kq.rh == 0.f ? 8u : code_bits<true>(r1, kq) - kRoundBits;
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

// n_new tokens of each sequence (new_lens[b] of them when given) behind its last slot; a warp takes
// TPW tokens, the next one's loads under the work on the last.  The block that finishes last of a
// sequence moves its length on: by then every other one has read it (state's third row counts them,
// and is zero between calls).  A block has 32 tokens of a prompt: the blocks meet at that counter, one
// address a sequence, and with 8 tokens a block their arrivals took longer than the tokens (4 x 4096: 22
// us).  By 32 warps, or, from 8192 tokens on, by 8 warps of four tokens each: 4 x 4096 tokens 12.7 and
// 10.1 us, 1 x 4096 3.4 and 5.4.
constexpr int kManyTokens = 8192;
template <int TPW>
__global__ void __launch_bounds__(TPW == 1 ? 1024 : 256)
    append_kernel(Cache c, const __nv_bfloat16* lat, int64_t lat_ld,
                  const __nv_bfloat16* kpe, int64_t kpe_ld, int64_t src_bstride,
                  int n_new, const int32_t* new_lens,
                  const __nv_bfloat16* cos_t, const __nv_bfloat16* sin_t,
                  int table_rows, float eps) {
  const int b = blockIdx.y;
  const int warps = blockDim.x >> 5;
  const int i0 = blockIdx.x * warps * TPW + (threadIdx.x >> 5);
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int64_t src0 = static_cast<int64_t>(b) * src_bstride;
  Token tok{};
  if (i0 < n_new) tok = load_token(lat + (src0 + i0) * lat_ld, kpe + (src0 + i0) * kpe_ld);
  const int len = c.state[b], next = c.state[c.batch + b];
  const int n = new_lens != nullptr ? min(n_new, new_lens[b]) : n_new;
#pragma unroll 1
  for (int k = 0; k < TPW; ++k) {
    const int i = i0 + warps * k;
    if (i >= n || len < 0 || len + i >= c.slots) break;
    const Token now = tok;
    if (k + 1 < TPW && i + warps < n)
      tok = load_token(lat + (src0 + i + warps) * lat_ld, kpe + (src0 + i + warps) * kpe_ld);
    put_token(c, b, len + i, next + i, now, cos_t, sin_t, table_rows, eps);
  }
  __syncthreads();  // every warp has read the length
  if (threadIdx.x == 0 &&
      (gridDim.x == 1 ||
       atomicAdd(c.state + 2 * c.batch + b, 1) == static_cast<int>(gridDim.x) - 1)) {
    const int add = max(0, min(n, c.slots - len));
    c.state[b] = len + add;
    c.state[c.batch + b] = next + add;
    c.state[2 * c.batch + b] = 0;
  }
}

// Lengths, positions and counters to 0 (a kernel like the others: a memset node would end the
// overlap of what lies before it with what lies behind).
__global__ void __launch_bounds__(256) reset_kernel(int32_t* state, int n) {
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  for (int i = threadIdx.x; i < n; i += 256) state[i] = 0;
}

// What a decode step does between its projection and the attention, a block a sequence: warp 0
// appends the new token (latent and k_pe of the projection's row) and moves the length on, the
// others copy the heads' absorbed queries and rotate their q_pe at the token's position.
__global__ void __launch_bounds__(288)
    decode4_prepare_kernel(Cache c, const __nv_bfloat16* proj, int ld, int heads,
                           const __nv_bfloat16* cos_t,
                           const __nv_bfloat16* sin_t, int table_rows, float eps,
                           __nv_bfloat16* q) {
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const __nv_bfloat16* row = proj + static_cast<int64_t>(b) * ld;
  const int len = c.state[b], next = c.state[c.batch + b];
  if (warp == 0) {
    const __nv_bfloat16* lat = row + heads * kQCols;
    const Token tok = load_token(lat, lat + kLatent);
    if (len >= 0 && len < c.slots)
      put_token(c, b, len, next, tok, cos_t, sin_t, table_rows, eps);
  } else {
    const int prow = table_row(next, table_rows);
    const __nv_bfloat16* cr = cos_t + static_cast<int64_t>(prow) * kRope;
    const __nv_bfloat16* sr = sin_t + static_cast<int64_t>(prow) * kRope;
    for (int h = warp - 1; h < heads; h += 8) {
      __nv_bfloat16* dst = q + (static_cast<int64_t>(b) * heads + h) * kQCols;
      const uint4* s4 = reinterpret_cast<const uint4*>(row + h * kLatent) + 2 * lane;
      reinterpret_cast<uint4*>(dst)[2 * lane] = s4[0];
      reinterpret_cast<uint4*>(dst)[2 * lane + 1] = s4[1];
      const __nv_bfloat162 x =
          reinterpret_cast<const __nv_bfloat162*>(row + heads * kLatent + h * kRope)[lane];
      const float xa = __low2float(x), xb = __high2float(x);
      dst[kLatent + lane] = __float2bfloat16_rn(xa * __bfloat162float(cr[lane]) -
                                                xb * __bfloat162float(sr[lane]));
      dst[kLatent + 32 + lane] = __float2bfloat16_rn(xb * __bfloat162float(cr[32 + lane]) +
                                                     xa * __bfloat162float(sr[32 + lane]));
    }
  }
  __syncthreads();  // every warp has read the position
  if (threadIdx.x == 0 && len < c.slots) {
    c.state[b] = len + 1;
    c.state[c.batch + b] = next + 1;
  }
}

// Eight codes of one word -> eight bf16 values (code - 8) * scale, rounded once: 128 + code is a
// bf16 pair under a mask, 136 off it is exact, and the product rounds.
__device__ __forceinline__ uint4 values8(uint32_t w, uint32_t scale2) {
  uint32_t p[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // nibbles j and j + 4
    const uint32_t x = ((w >> (4 * j)) & 0x000F000Fu) | 0x43004300u;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(p[j]) : "r"(x), "r"(0x43084308u));
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(p[j]) : "r"(p[j]), "r"(scale2));
  }
  return make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410),
                    __byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x7632));
}

// Slots 0 .. n-1 of every sequence as bf16 values, zeros from its length on; four slots a warp,
// so that their loads are in flight together.
constexpr int kGetSlots = 4;
__global__ void __launch_bounds__(256)
    get_kernel(Cache c, int n, uint4* lat, uint4* kpe) {
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.y;
  const int t0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * kGetSlots;
  if (t0 >= n) return;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int len = c.state[b];
  const int64_t row0 = static_cast<int64_t>(b) * c.slots + t0;
  const unsigned short* sc = reinterpret_cast<const unsigned short*>(c.scales) +
                             static_cast<int64_t>(b) * kGroups * c.slots + t0;
  uint32_t w[kGetSlots][3], s[kGetSlots][3];
#pragma unroll
  for (int k = 0; k < kGetSlots; ++k) {  // (slots are a multiple of 64: all four exist)
    const uint32_t* src = reinterpret_cast<const uint32_t*>(c.codes + (row0 + k) * kRowBytes);
    w[k][0] = src[lane];
    w[k][1] = src[32 + lane];
    w[k][2] = lane < 8 ? src[64 + lane] : 0u;
    s[k][0] = *(sc + static_cast<int64_t>(lane >> 4) * c.slots + k);
    s[k][1] = *(sc + static_cast<int64_t>(2 + (lane >> 4)) * c.slots + k);
    s[k][2] = *(sc + static_cast<int64_t>(4) * c.slots + k);
  }
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int k = 0; k < kGetSlots; ++k) {
    if (t0 + k >= n) break;
    const bool in = t0 + k < len;
    const int64_t o = static_cast<int64_t>(b) * n + t0 + k;
    lat[o * 64 + lane] = in ? values8(w[k][0], s[k][0] * 0x00010001u) : zero;
    lat[o * 64 + 32 + lane] = in ? values8(w[k][1], s[k][1] * 0x00010001u) : zero;
    if (lane < 8) kpe[o * 8 + lane] = in ? values8(w[k][2], s[k][2] * 0x00010001u) : zero;
  }
}

// ---- attention ------------------------------------------------------------------------------
// One query token per sequence over its slots, 16 heads (an MMA's M) at a time.
//
// Work is cut into segments of one (sequence, head tile): up to `per` consecutive chunks of 128
// slots, `per` the smallest number for which there are no more segments than CTAs (two an SM), so
// whatever the lengths the CTAs are about equally long; every block works that out from the
// lengths on the device.  A segment that is all of its sequence writes the output; the others
// leave partials, which merge_kernel joins.  (Equal ranges of chunks that cross sequences balance
// better still, but most CTAs then set up two segments: 64 x 2048 slots took 43 us against 36.8.)
//
// Products run on mma.sync m16n8k16 (f16, f32 accumulators) with the 16 heads as M.  A pair of CTAs
// takes 8900 cycles for two chunks, 35 a slot and SM: S 3850, P V 3300, maxima, exponentials and
// barriers 1100, waiting 350; the MMAs alone would take 18 a slot, with the conversion of their
// operands' codes 29 (the two add up: eight warps a CTA took 115 us against 96 for 32 x 16384 slots).
// tcgen05 on codes unpacked to bytes, with q in three and P in four 8-bit digits, takes 12.8 a slot
// for its MMAs but fills the SM's shared memory, which starves the copies and the softmax beside
// it: 166 us.
// Here the codes go from shared memory to the fragments:
//   * a nibble c in bits 0-3 of a half, under the exponent of 1024, is 1024 + c; in bits 4-7, under
//     that of 64, 64 + c.  One AND-OR and one subtraction (1032, 72) make two operands code - 8,
//     exactly, and one shift by 8 a word serves its other four codes: 9 instructions for 8
//     codes.  (The nibble as it stands is the f16 subnormal c 2^-24 and would need no subtraction
//     but the products then lose about ten bits when the tensor core aligns them; an offset left
//     in the operands costs f32 bits of every sum.)
//   * a group's scale multiplies the accumulator of its 128 dimensions (S) or the probability
//     (O; warp w has the dimensions of group w), never the 128 values.
//   * any bijection of an MMA's K index and of its N index serves, if both operands use it: K of
//     S is the order in which a word's nibbles come out, and slot T(c, m) = (c ^ 2(m&1)) + 4m of
//     16 sits at the m-th column pair of thread c, so that S fragments are P fragments after one
//     16-byte store and every shared load is free of bank conflicts (288 bytes a row = 8 banks
//     modulo 32: four slots that differ modulo 4 meet all banks).
// q is scaled by a power of two per head, P by one per group and CTA, into f16's range (2^29 of
// normal numbers below the largest), so P carries 11 bits where bf16 would carry 8.
// The running maximum of a head is raised, and O rescaled, only when it grows by more than 2^4.
constexpr int kChunk = 128;
constexpr int kAttnThreads = 128;
constexpr int kStages = 2;       // chunks of codes in shared memory
constexpr int kCtasPerSm = 2;
constexpr int kPLd = 144;  // floats; 16 modulo 32: conflict-free 16-byte rows
constexpr uint32_t kStageBytes = kChunk * kRowBytes;                 // 36,864
constexpr uint32_t kQLd = 2 * kQCols * 2 + 64;  // two heads; 64 modulo 128: conflict-free
constexpr uint32_t kQBytes = 8 * kQLd;                               // 18,944
constexpr uint32_t kPBytes = 16 * kPLd * 4;                          // 9,216
constexpr uint32_t kFacBytes = kGroups * kChunk * 4;                 // 2,560, twice
constexpr uint32_t kOffQ = kStages * kStageBytes;
constexpr uint32_t kOffP = kOffQ + kQBytes;
constexpr uint32_t kOffFac = kOffP + kPBytes;
constexpr uint32_t kOffSmall = kOffFac + 2 * kFacBytes;
struct AttnSmall {  // behind the tiles
  unsigned long long bar[kStages];
  float row[16];            // accumulator -> log2 of a weight
  float wmax[4][16];
  float wsum[4][16];
  alignas(16) int scan[16];
  int abort_flag;
  int never_flag;
};
constexpr size_t kAttnSmem = kOffSmall + sizeof(AttnSmall);
constexpr long long kTimeoutCycles = 4000000000LL;

struct AttnParams {
  Cache c;
  const __nv_bfloat16* q;  // [batch, heads, 576]
  __nv_bfloat16* out;      // [batch, heads * 512]
  int heads, tiles;        // head tiles of 16
  int max_chunks;          // of any sequence, as the host knows it
  float scale_log2;
  float* part_o;           // [segment][4 warps][16 (row half, k, j / 4)][32 lanes][4 j]: see its store
  float* part_ml;          // [segment][2][16]: maximum (log2), sum
  int2* where;             // [batch, tiles]: a row's first segment, and how many
  float* lse;              // [batch, tiles * 16]: of whole segments, then of all
  float* scores;           // [batch, tiles, max_chunks, 16, 128] (slots in fragment order) or null
  int ctas;
  int* status;
};

__device__ __forceinline__ int chunks_of(const Cache& c, int b, int max_chunks) {
  const int len = min(max(c.state[b], 0), c.slots);
  return min((len + kChunk - 1) / kChunk, max_chunks);
}
// Position of slot t (0..15) of a 16-slot group in fragment order, and back.
__device__ __forceinline__ int frag_pos(int t) {
  const int m = (t >> 2) & 3;
  return (t & ~15) | (((t & 3) ^ (2 * (m & 1))) * 4 + m);
}
__device__ __forceinline__ int frag_slot(int pos) {
  const int m = pos & 3, c = (pos >> 2) & 3;
  return (pos & ~15) | ((c ^ (2 * (m & 1))) + 4 * m);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The eight codes of a word, less 8, as four f16 pairs: pair j = nibbles j and j + 4.
struct Masks {  // constants kept in registers, so that the AND-OR is one instruction
  uint32_t m0, e0, s0, m1, e1, s1;
};
__device__ __forceinline__ Masks masks() {
  Masks k;
  asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(k.m0));
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(k.e0));  // 1024
  asm volatile("mov.b32 %0, 0xE408E408;" : "=r"(k.s0));  // -1032
  asm volatile("mov.b32 %0, 0x00F000F0;" : "=r"(k.m1));
  asm volatile("mov.b32 %0, 0x54005400;" : "=r"(k.e1));  // 64
  asm volatile("mov.b32 %0, 0xD480D480;" : "=r"(k.s1));  // -72
  return k;
}
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t m, uint32_t e) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(m), "r"(e));
  return r;
}
__device__ __forceinline__ uint32_t add_f16x2(uint32_t x, uint32_t y) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(y));
  return r;
}
__device__ __forceinline__ void codes_f16(uint32_t w, const Masks& k, uint32_t (&o)[4]) {
  const uint32_t v = w >> 8;
  o[0] = add_f16x2(and_or(w, k.m0, k.e0), k.s0);
  o[1] = add_f16x2(and_or(w, k.m1, k.e1), k.s1);
  o[2] = add_f16x2(and_or(v, k.m0, k.e0), k.s0);
  o[3] = add_f16x2(and_or(v, k.m1, k.e1), k.s1);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Sums of u and v over the block (kAttnThreads threads); `red`: 8 words that no earlier call in
// flight uses (callers alternate between two).
__device__ __forceinline__ int2 block_add(int u, int v, int* red) {
  u = __reduce_add_sync(0xffffffffu, u);
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) {
    red[threadIdx.x >> 5] = u;
    red[4 + (threadIdx.x >> 5)] = v;
  }
  __syncthreads();
  const int4 x = *reinterpret_cast<const int4*>(red), y = *reinterpret_cast<const int4*>(red + 4);
  return make_int2((x.x + x.y) + (x.z + x.w), (y.x + y.y) + (y.z + y.w));
}
// The segments' plan, the same in every block: chunks a segment, and the segments in all.
// Segments are numbered sequence by sequence, head tile by head tile.  (Chunks fit 32 bits: one
// is 36 KB of cache.)
struct Plan {
  int per, segments;
};
__device__ __forceinline__ Plan plan_segments(const AttnParams& p, int* red) {
  // up to 128 sequences stay in registers, one a thread
  const int mine = static_cast<int>(threadIdx.x) < p.c.batch ? chunks_of(p.c, threadIdx.x, p.max_chunks) : 0;
  int n = mine, some = mine > 0 ? 1 : 0;
  for (int b = threadIdx.x + kAttnThreads; b < p.c.batch; b += kAttnThreads) {
    const int k = chunks_of(p.c, b, p.max_chunks);
    n += k;
    some += k > 0 ? 1 : 0;
  }
  const int2 sum = block_add(n, some, red);
  const int total = sum.x * p.tiles, rows = sum.y * p.tiles;  // rows: not empty
  Plan w;
  if (rows >= p.ctas) {  // a segment each
    w.per = p.max_chunks;
    w.segments = rows;
    return w;
  }
  // a row of n chunks has at most n / per + 1 segments, so total / (ctas - rows) chunks fit
  int lo = max(1, (total + p.ctas - 1) / p.ctas);
  int hi = max(lo, min(p.max_chunks, (total + p.ctas - rows - 1) / (p.ctas - rows)));
  for (int turn = 1;; ++turn) {
    w.per = (lo + hi) >> 1;
    n = (mine + w.per - 1) / w.per;
    for (int b = threadIdx.x + kAttnThreads; b < p.c.batch; b += kAttnThreads)
      n += (chunks_of(p.c, b, p.max_chunks) + w.per - 1) / w.per;
    w.segments = block_add(n, 0, red + 8 * (turn & 1)).x * p.tiles;
    if (lo == hi) return w;
    if (w.segments <= p.ctas) hi = w.per;
    else lo = w.per + 1;
  }
}

// The scales of slot t0 + threadIdx.x as they multiply the accumulators: scale * rstd for the
// latent groups; 0 outside the segment, whatever the memory there holds.  The loads are without
// condition (the last slot's behind it), wait for nothing and stay where they are written, ahead of
// S: as plain ones they were moved behind it, and 64 x 2048 slots took 33.2 us against 30.4, 32 x 16384
// 95.3 against 96.4.
struct Factors {
  unsigned short s[kGroups];
  float rstd;
  bool in;
};
__device__ __forceinline__ Factors load_factors(const Cache& c, int b, int t, int t_end) {
  Factors f;
  f.in = t < t_end;
  t = min(t, c.slots - 1);
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
    f.s[g] = __ldcg(reinterpret_cast<const unsigned short*>(c.scales) +
                    (static_cast<int64_t>(b) * kGroups + g) * c.slots + t);
  f.rstd = __ldcg(c.rstd + static_cast<int64_t>(b) * c.slots + t);
  return f;
}
__device__ __forceinline__ void store_factors(float* fac, const Factors& f) {
  const int pos = frag_pos(threadIdx.x);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const float x = __uint_as_float(static_cast<uint32_t>(f.s[g]) << 16);
    fac[g * kChunk + pos] = f.in ? (g < 4 ? x * f.rstd : x) : 0.f;
  }
}

__global__ void __launch_bounds__(kAttnThreads, kCtasPerSm) attend4_kernel(const AttnParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  const Cache& c = p.c;
  AttnSmall& sm = *reinterpret_cast<AttnSmall*>(smem + kOffSmall);
  const uint32_t s0 = ptx::smem_u32(smem);
  const uint32_t bar0 = ptx::smem_u32(sm.bar);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, cc = lane & 3;  // fragment row (or column) and column pair
  if (threadIdx.x == 0) {
    ptx::mbar_init(bar0, 1);
    ptx::mbar_init(bar0 + 8, 1);
    sm.abort_flag = 0;
    sm.never_flag = 0;
    ptx::fence_barrier_init();
  }
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const Plan plan = plan_segments(p, sm.scan);
  const Masks km = masks();
  uint32_t it = 0;  // chunks taken so far: stage it & 1, phase (it >> 1) & 1
  for (int index = blockIdx.x; index < plan.segments; index += gridDim.x) {
    // the sequence of segment `index`: 32 sequences at a time, every warp alike
    int b = 0, before = 0;
    for (int base = 0;; base += 32) {
      const int n = base + lane < c.batch
                        ? (chunks_of(c, base + lane, p.max_chunks) + plan.per - 1) / plan.per * p.tiles
                        : 0;
      int incl = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + incl > index);
      if (hit != 0u) {
        const int l = __ffs(hit) - 1;
        b = base + l;
        before += __shfl_sync(0xffffffffu, incl - n, l);
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
      if (base + 32 >= c.batch) return;  // not reached: index < segments
    }
    const int nch = chunks_of(c, b, p.max_chunks);
    const int nseg = (nch + plan.per - 1) / plan.per;
    const int tile = (index - before) / nseg;
    const int c0 = (index - before - tile * nseg) * plan.per;
    const int seg = min(plan.per, nch - c0);
    const bool whole = nseg == 1;
    if (c0 == 0 && threadIdx.x == 0) p.where[b * p.tiles + tile] = make_int2(index, nseg);
    const int len = min(c.state[b], c.slots);
    const int nh = min(16, p.heads - tile * 16);
    const uint8_t* codes = c.codes + static_cast<int64_t>(b) * c.slots * kRowBytes;
    // The last chunk may reach past the slots: copy the rows that exist.  The second chunk is asked
    // for when the first has arrived: side by side, all CTAs first products would wait for both
    // (64 x 2048 slots: 34.0 us against 30.5).
    auto load_chunk = [&](int i, uint32_t at) {
      const int t0 = (c0 + i) * kChunk;
      const uint32_t bytes = static_cast<uint32_t>(min(kChunk, c.slots - t0)) * kRowBytes;
      const uint32_t bar = bar0 + 8 * (at & 1);
      ptx::mbar_arrive_expect_tx(bar, bytes);
      ptx::bulk_load_1d(s0 + (at & 1) * kStageBytes, codes + static_cast<int64_t>(t0) * kRowBytes,
                        bytes, bar);
    };
    __syncthreads();  // the last segment is done with the tiles (and the barriers are set up)
    if (threadIdx.x == 0) {
      load_chunk(0, it);
    }
    Factors nf = load_factors(c, b, c0 * kChunk + threadIdx.x, len);
    // Q as f16 fragments: warp w makes the heads r and r + 8 of rows r = 2w, 2w + 1, whose words
    // lie side by side as an MMA takes them.  Lane l holds dimensions 16 l .. (and 2 of q_pe);
    // k-step s of a quad of 64 dimensions takes pairs j = 2 (s & 1), + 1 of word s / 2.
    uint32_t qw[4][9];  // heads 2w, 2w + 8, 2w + 1, 2w + 9: all on their way before the first is used
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = warp * 2 + (i >> 1) + 8 * (i & 1);
      const __nv_bfloat16* q =
          p.q + (static_cast<int64_t>(b) * p.heads + tile * 16 + (h < nh ? h : 0)) * kQCols;
      const uint4 x0 = *(reinterpret_cast<const uint4*>(q) + 2 * lane);
      const uint4 x1 = *(reinterpret_cast<const uint4*>(q) + 2 * lane + 1);
      qw[i][0] = x0.x, qw[i][1] = x0.y, qw[i][2] = x0.z, qw[i][3] = x0.w;
      qw[i][4] = x1.x, qw[i][5] = x1.y, qw[i][6] = x1.z, qw[i][7] = x1.w;
      qw[i][8] = *(reinterpret_cast<const uint32_t*>(q + kLatent) + lane);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = warp * 2 + i;
      uint32_t f[2][8], fr[2][2];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const int h = r + 8 * hh;
        const uint32_t(&w)[9] = qw[2 * i + hh];
        // the largest magnitude, as a bf16's bits (infinities and NaN order above)
        uint32_t m2 = 0;
#pragma unroll
        for (int j = 0; j < 9; ++j) m2 = __vmaxu2(m2, w[j] & 0x7FFF7FFFu);
        const uint32_t m = __reduce_max_sync(0xffffffffu, max(m2 & 0xFFFFu, m2 >> 16));
        // its exponent to 2^14, by two factors: their product may pass 2^127
        const int e = m == 0 || m >= 0x7F80u ? 0 : 14 + 127 - max(static_cast<int>(m >> 7), 1);
        const float fa = __int_as_float((127 + e / 2) << 23);
        const float fb = h < nh ? __int_as_float((127 + e - e / 2) << 23) : 0.f;
        float v[18];
#pragma unroll
        for (int j = 0; j < 9; ++j) {
          v[2 * j] = __uint_as_float(w[j] << 16) * fa * fb;
          v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u) * fa * fb;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int n = (j & 3) + 8 * (j >> 2);
          f[hh][j] = pack_f16(v[n], v[n + 4]);
        }
        // q_pe dimensions 2 l and 2 l + 1; their partners are two lanes up
        fr[hh][0] = pack_f16(v[16], __shfl_down_sync(0xffffffffu, v[16], 2));
        fr[hh][1] = pack_f16(v[17], __shfl_down_sync(0xffffffffu, v[17], 2));
        if (lane == 0)
          sm.row[h] = p.scale_log2 * __int_as_float((127 - e / 2) << 23) *
                      __int_as_float((127 - (e - e / 2)) << 23);
      }
      uint8_t* row = smem + kOffQ + r * kQLd;
#pragma unroll
      for (int s = 0; s < 4; ++s)
        *reinterpret_cast<uint4*>(row + (lane >> 2) * 256 + s * 64 + (lane & 3) * 16) =
            make_uint4(f[0][2 * s], f[1][2 * s], f[0][2 * s + 1], f[1][2 * s + 1]);
      if ((lane & 2) == 0)
        *reinterpret_cast<uint4*>(row + 8 * 256 + ((lane & 4) >> 1 | (lane & 1)) * 64 +
                                  (lane >> 3) * 16) =
            make_uint4(fr[0][0], fr[1][0], fr[0][1], fr[1][1]);
    }
    store_factors(reinterpret_cast<float*>(smem + kOffFac) + (it & 1) * (kFacBytes / 4), nf);
    __syncthreads();

    float o[16][4];
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[j][k] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float pmax = 0.f, pscale = 1.f;  // of this warp's group: largest factor seen, power of two
    const float row0 = sm.row[g], row1 = sm.row[g + 8];
    for (int i = 0; i < seg; ++i, ++it) {
      const int t0 = (c0 + i) * kChunk;
      const bool ok = ptx::mbar_wait(bar0 + 8 * (it & 1), (it >> 1) & 1, &sm.abort_flag, p.status,
                                     kTimeoutCycles, DS_ERR_TIMEOUT);
      if (threadIdx.x == 0 && i == 0 && seg > 1) load_chunk(1, it + 1);
      const uint8_t* st = smem + (it & 1) * kStageBytes;
      float* fac = reinterpret_cast<float*>(smem + kOffFac + (it & 1) * kFacBytes);
      const bool more = i + 1 < seg;
      if (more) nf = load_factors(c, b, t0 + kChunk + threadIdx.x, len);
      // ---- S: this warp's 32 slots (four blocks of 8 columns) against 16 heads
      float sc[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[k][j] = 0.f;
      {
        // column n = g of block k: slot T(g / 2, g & 1 | 2 (k & 1)) of 16-slot group 2 warp + k / 2
        const int te = (((g >> 1) ^ (2 * (g & 1))) + 4 * (g & 1)) + warp * 32;
        const uint8_t* base = st + te * kRowBytes + cc * 8;
        const uint8_t* q0 = smem + kOffQ + g * kQLd + cc * 16;
        const float* fac0 = fac + warp * 32 + 4 * cc;
#pragma unroll 1
        for (int gr = 0; gr < kGroups; ++gr) {
          float acc[4][4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[k][j] = 0.f;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            if (half == 1 && gr == 4) break;  // 64 dimensions of k_pe
            const int qd = 2 * gr + half;
            uint4 a[4];
            uint2 x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const uint2*>(base + (k * 8) * kRowBytes + qd * 32);
#pragma unroll
            for (int s = 0; s < 4; ++s) a[s] = *reinterpret_cast<const uint4*>(q0 + qd * 256 + s * 64);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              uint32_t v[4], w[4];
              codes_f16(x[k].x, km, v);
              mma_f16(acc[k], a[0].x, a[0].y, a[0].z, a[0].w, v[0], v[1]);
              mma_f16(acc[k], a[1].x, a[1].y, a[1].z, a[1].w, v[2], v[3]);
              codes_f16(x[k].y, km, w);
              mma_f16(acc[k], a[2].x, a[2].y, a[2].z, a[2].w, w[0], w[1]);
              mma_f16(acc[k], a[3].x, a[3].y, a[3].z, a[3].w, w[2], w[3]);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // the group is complete: times its slots' factors
            const float2 f = *reinterpret_cast<const float2*>(fac0 + gr * kChunk + (k >> 1) * 16 + 2 * (k & 1));
            sc[k][0] = fmaf(acc[k][0], f.x, sc[k][0]);
            sc[k][1] = fmaf(acc[k][1], f.y, sc[k][1]);
            sc[k][2] = fmaf(acc[k][2], f.x, sc[k][2]);
            sc[k][3] = fmaf(acc[k][3], f.y, sc[k][3]);
          }
        }
      }
      // column pair cc of block k: slots T(cc, 2 (k & 1)) and T(cc, 2 (k & 1) + 1)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        sc[k][0] *= row0;
        sc[k][1] *= row0;
        sc[k][2] *= row1;
        sc[k][3] *= row1;
      }
      if (t0 + kChunk > len) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (t0 + warp * 32 + k * 8 + (cc ^ (2 * j)) + 4 * j >= len)
              sc[k][j] = sc[k][2 + j] = -INFINITY;
      }
      float mx0 = sc[0][0], mx1 = sc[0][2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        mx0 = fmaxf(mx0, fmaxf(sc[k][0], sc[k][1]));
        mx1 = fmaxf(mx1, fmaxf(sc[k][2], sc[k][3]));
      }
      mx0 = fmaxf(mx0, -INFINITY);  // (all NaN: a maximum must not be one)
      mx1 = fmaxf(mx1, -INFINITY);
      if (p.scores != nullptr) {
        float* dst = p.scores +
                     ((static_cast<int64_t>(b) * p.tiles + tile) * p.max_chunks + c0 + i) * 16 * kChunk +
                     warp * 32 + 4 * cc;
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          *reinterpret_cast<float4*>(dst + g * kChunk + 8 * k) =
              make_float4(sc[k][0], sc[k][1], sc[k + 1][0], sc[k + 1][1]);
          *reinterpret_cast<float4*>(dst + (g + 8) * kChunk + 8 * k) =
              make_float4(sc[k][2], sc[k][3], sc[k + 1][2], sc[k + 1][3]);
        }
      }
#pragma unroll
      for (int d = 2; d > 0; d >>= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, d));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, d));
      }
      if (cc == 0) {
        sm.wmax[warp][g] = mx0;
        sm.wmax[warp][g + 8] = mx1;
      }
      // barrier A: the maxima are there; every warp is done with the last chunk's P and codes
      if (!__syncthreads_and(ok)) {  // a load did not arrive in time: wait (bounded) and leave
        if (threadIdx.x == 0) {
          ptx::mbar_wait(bar0 + 8 * (it & 1), (it >> 1) & 1, &sm.never_flag, p.status,
                         kTimeoutCycles, DS_ERR_TIMEOUT);
          if (more && i == 0)  // (later chunks are asked for behind this barrier)
            ptx::mbar_wait(bar0 + 8 * ((it + 1) & 1), ((it + 1) >> 1) & 1, &sm.never_flag, p.status,
                           kTimeoutCycles, DS_ERR_TIMEOUT);
        }
        return;
      }
      if (threadIdx.x == 0 && i >= 1 && more) load_chunk(i + 1, it + 1);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        mx0 = fmaxf(mx0, sm.wmax[w][g]);
        mx1 = fmaxf(mx1, sm.wmax[w][g + 8]);
      }
      const float n0 = mx0 > m0 + 4.f ? mx0 : m0, n1 = mx1 > m1 + 4.f ? mx1 : m1;
      if (__any_sync(0xffffffffu, n0 != m0 || n1 != m1)) {
        const float f0 = ptx::ex2(m0 - (n0 == -INFINITY ? 0.f : n0));
        const float f1 = ptx::ex2(m1 - (n1 == -INFINITY ? 0.f : n1));
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          o[j][0] *= f0;
          o[j][1] *= f0;
          o[j][2] *= f1;
          o[j][3] *= f1;
        }
        l0 *= f0;
        l1 *= f1;
        m0 = n0;
        m1 = n1;
      }
      const float r0 = m0 == -INFINITY ? 0.f : m0, r1 = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        float4 a, bb;
        a.x = ptx::ex2(sc[k][0] - r0);
        a.y = ptx::ex2(sc[k][1] - r0);
        a.z = ptx::ex2(sc[k + 1][0] - r0);
        a.w = ptx::ex2(sc[k + 1][1] - r0);
        bb.x = ptx::ex2(sc[k][2] - r1);
        bb.y = ptx::ex2(sc[k][3] - r1);
        bb.z = ptx::ex2(sc[k + 1][2] - r1);
        bb.w = ptx::ex2(sc[k + 1][3] - r1);
        l0 += (a.x + a.y) + (a.z + a.w);
        l1 += (bb.x + bb.y) + (bb.z + bb.w);
        float* dst = reinterpret_cast<float*>(smem + kOffP) + warp * 32 + 8 * k + 4 * cc;
        *reinterpret_cast<float4*>(dst + g * kPLd) = a;
        *reinterpret_cast<float4*>(dst + (g + 8) * kPLd) = bb;
      }
      if (more)
        store_factors(reinterpret_cast<float*>(smem + kOffFac) + ((it + 1) & 1) * (kFacBytes / 4), nf);
      __syncthreads();  // barrier B: P and the next chunk's factors are there
      // ---- O += P V over the 128 dimensions of group `warp`
      {
        float* fw = fac + warp * kChunk;
        const float4 fl = reinterpret_cast<const float4*>(fw)[lane];
        float fm = fmaxf(fmaxf(fl.x, fl.y), fmaxf(fl.z, fl.w));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) fm = fmaxf(fm, __shfl_xor_sync(0xffffffffu, fm, d));
        if (fm > 16.f * pmax && fm <= 3.4e38f) {  // (warp-uniform) largest factor to [2^6, 2^7)
          const float ns = ldexpf(1.f, max(-100, min(100, 6 - ilogbf(fm))));
          if (pmax > 0.f) {
            const float f = ns / pscale;  // powers of two
#pragma unroll
            for (int j = 0; j < 16; ++j)
#pragma unroll
              for (int k = 0; k < 4; ++k) o[j][k] *= f;
          }
          pscale = ns;
          pmax = fm;
        }
        // this group's factors, scaled, back in place: no other warp reads them any more
        __syncwarp();
        reinterpret_cast<float4*>(fw)[lane] =
            make_float4(fl.x * pscale, fl.y * pscale, fl.z * pscale, fl.w * pscale);
        __syncwarp();
        // B: slots T(cc, 0..3) of the 16, dimensions 128 warp + 16 g + 0..15
        const uint8_t* v0 = st + cc * kRowBytes + warp * 64 + g * 8;
        const uint8_t* v1 = st + ((cc ^ 2) + 4) * kRowBytes + warp * 64 + g * 8;
        const float* pr = reinterpret_cast<const float*>(smem + kOffP) + g * kPLd + 4 * cc;
#pragma unroll 2
        for (int kk = 0; kk < 8; ++kk) {
          const float4 p0 = *reinterpret_cast<const float4*>(pr + kk * 16);
          const float4 p1 = *reinterpret_cast<const float4*>(pr + 8 * kPLd + kk * 16);
          const float4 f = *reinterpret_cast<const float4*>(fw + kk * 16 + 4 * cc);
          const uint2 x0 = *reinterpret_cast<const uint2*>(v0 + (kk * 16) * kRowBytes);
          const uint2 x1 = *reinterpret_cast<const uint2*>(v1 + (kk * 16) * kRowBytes);
          const uint2 x2 = *reinterpret_cast<const uint2*>(v0 + (kk * 16 + 8) * kRowBytes);
          const uint2 x3 = *reinterpret_cast<const uint2*>(v1 + (kk * 16 + 8) * kRowBytes);
          const uint32_t a0 = pack_f16(p0.x * f.x, p0.y * f.y), a1 = pack_f16(p1.x * f.x, p1.y * f.y);
          const uint32_t a2 = pack_f16(p0.z * f.z, p0.w * f.w), a3 = pack_f16(p1.z * f.z, p1.w * f.w);
#pragma unroll
          for (int wi = 0; wi < 2; ++wi) {
            const uint32_t y0 = wi ? x0.y : x0.x, y1 = wi ? x1.y : x1.x;
            const uint32_t y2 = wi ? x2.y : x2.x, y3 = wi ? x3.y : x3.x;
#pragma unroll
            for (int up = 0; up < 2; ++up) {
              uint32_t b0[4], b1[4];
              codes_f16(__byte_perm(y0, y1, up ? 0x7632 : 0x5410), km, b0);
              codes_f16(__byte_perm(y2, y3, up ? 0x7632 : 0x5410), km, b1);
#pragma unroll
              for (int j = 0; j < 4; ++j)
                mma_f16(o[8 * wi + 4 * up + j], a0, a1, a2, a3, b0[j], b1[j]);
            }
          }
        }
      }
    }
    // ---- the segment's result
#pragma unroll
    for (int d = 2; d > 0; d >>= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, d);
      l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    if (cc == 0) {
      sm.wsum[warp][g] = l0;
      sm.wsum[warp][g + 8] = l1;
    }
    __syncthreads();
    l0 = (sm.wsum[0][g] + sm.wsum[1][g]) + (sm.wsum[2][g] + sm.wsum[3][g]);
    l1 = (sm.wsum[0][g + 8] + sm.wsum[1][g + 8]) + (sm.wsum[2][g + 8] + sm.wsum[3][g + 8]);
    const float unit = 1.f / pscale;
    float f0 = unit, f1 = unit;
    if (whole) {
      f0 = l0 == 0.f ? 0.f : unit / l0;
      f1 = l1 == 0.f ? 0.f : unit / l1;
    }
    if (warp == 0 && cc == 0) {
      if (whole) {
        if (p.lse != nullptr) {
          float* lse = p.lse + (static_cast<int64_t>(b) * p.tiles + tile) * 16;
          lse[g] = m0 + log2f(l0);
          lse[g + 8] = m1 + log2f(l1);
        }
      } else {
        float* ml = p.part_ml + static_cast<int64_t>(index) * 32;
        ml[g] = m0;
        ml[g + 8] = m1;
        ml[16 + g] = l0;
        ml[16 + g + 8] = l1;
      }
    }
    // block j holds dimensions 128 warp + 16 (2 cc) + j and 16 (2 cc + 1) + j
    if (whole) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int h = g + 8 * r;
        const float f = r ? f1 : f0;
        if (h >= nh) continue;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          __nv_bfloat16* dst = p.out + (static_cast<int64_t>(b) * p.heads + tile * 16 + h) * kLatent +
                               128 * warp + 16 * (2 * cc + k);
#pragma unroll
          for (int j = 0; j < 16; j += 8) {
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const __nv_bfloat162 v = __floats2bfloat162_rn(o[j + 2 * x][2 * r + k] * f,
                                                             o[j + 2 * x + 1][2 * r + k] * f);
              w[x] = *reinterpret_cast<const uint32_t*>(&v);
            }
            *reinterpret_cast<uint4*>(dst + j) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
    } else {
      // in the order of the fragments, a warp's 512 bytes side by side (by rows, every store
      // would touch 32 lines: 2000 cycles a segment)
      float4* dst = reinterpret_cast<float4*>(p.part_o) +
                    (static_cast<int64_t>(index) * 4 + warp) * 16 * 32 + lane;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int j = 0; j < 16; j += 4) {
            const float f = r ? f1 : f0;
            dst[(r * 8 + k * 4 + j / 4) * 32] =
                make_float4(o[j][2 * r + k] * f, o[j + 1][2 * r + k] * f, o[j + 2][2 * r + k] * f,
                            o[j + 3][2 * r + k] * f);
          }
    }
  }
}

// A row's first partial and how many it has (1: none, the attention wrote the output); none for a sequence
// without slots, nor where the attention gave up (the status word says so) before it wrote the entry.
__device__ __forceinline__ int2 partials_of(const AttnParams& p, int b, int tile) {
  if (chunks_of(p.c, b, p.max_chunks) == 0) return make_int2(0, 0);
  const int2 w = __ldcg(p.where + b * p.tiles + tile);
  if (w.y == 1 || partials_exist(w.x, w.y, p.ctas)) return w;
  return make_int2(0, 0);
}

// Joins the partials of a (sequence, head tile), up to `most` of them: four blocks each, four heads
// a block, a warp a head (warps of heads that a last tile does not have leave at once, without the wait: its
// first block has a head and waits); lse (log2 of the weights' sum) where it is wanted; zeros for a sequence
// without slots.  (48 registers and no shared memory: two blocks fit beside two CTAs of the attention and
// are there when it ends.  With 64 registers, one, 64 x 2048 slots took 31.7 us against 30.2.)
__global__ void __launch_bounds__(kAttnThreads) merge_kernel(const AttnParams p, int most) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.y, tile = blockIdx.x >> 2, r = (blockIdx.x & 3) * 4 + warp;
  const int h = tile * 16 + r;
  if (h >= p.heads) return;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int2 w = partials_of(p, b, tile);
  if (w.y == 1 || w.y > most) return;  // written by the attention kernel; merge_wide_kernel's
  __nv_bfloat16* o = p.out + (static_cast<int64_t>(b) * p.heads + h) * kLatent;
  const float* ml = p.part_ml + static_cast<int64_t>(w.x) * 32 + r;
  // lane = (k, j / 4, cc): dimensions 128 w + 16 (2 cc + k) + j .. of row r, for the four w
  const int cc = lane & 3, jk = lane >> 2;
  const float4* po = reinterpret_cast<const float4*>(p.part_o) +
                     (static_cast<int64_t>(w.x) * 64 + (r >> 3) * 8 + jk) * 32 + (r & 7) * 4 + cc;
  float M = -INFINITY, L = 0.f;
  float a[16];  // four dimensions of each w
#pragma unroll
  for (int k = 0; k < 16; ++k) a[k] = 0.f;
  for (int i0 = 0; i0 < w.y; i0 += 32) {  // 32 partials at a time: lane i has the i-th's weight
    const bool in = i0 + lane < w.y;
    const float m = in ? __ldcg(ml + (i0 + lane) * 32) : -INFINITY;
    float l = in ? __ldcg(ml + (i0 + lane) * 32 + 16) : 0.f;
    float mx = fmaxf(m, M);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float ref = mx == -INFINITY ? 0.f : mx;
    const float keep = ptx::ex2(M - ref);
    const float f = in ? ptx::ex2(m - ref) : 0.f;
    l *= f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    L = fmaf(L, keep, l);
    M = mx;
#pragma unroll
    for (int k = 0; k < 16; ++k) a[k] *= keep;
#pragma unroll 4
    for (int i = 0; i < min(32, w.y - i0); ++i) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      const float4* src = po + static_cast<int64_t>(i0 + i) * (16 * kLatent / 4);  // (64 rows of 32)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float4 v = __ldcg(src + 16 * 32 * k);
        a[4 * k] = fmaf(fi, v.x, a[4 * k]);
        a[4 * k + 1] = fmaf(fi, v.y, a[4 * k + 1]);
        a[4 * k + 2] = fmaf(fi, v.z, a[4 * k + 2]);
        a[4 * k + 3] = fmaf(fi, v.w, a[4 * k + 3]);
      }
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a[4 * k] * inv, a[4 * k + 1] * inv);
    const __nv_bfloat162 y = __floats2bfloat162_rn(a[4 * k + 2] * inv, a[4 * k + 3] * inv);
    *reinterpret_cast<uint2*>(o + 128 * k + 16 * (2 * cc + (jk >> 2)) + 4 * (jk & 3)) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  }
  if (p.lse != nullptr && lane == 0)
    p.lse[(static_cast<int64_t>(b) * p.tiles + tile) * 16 + r] = M + log2f(L);
}

// The same for many partials, `least` or more (or none): a block a head and D-th of its dimensions, W
// warps that take the partials in turn.  A long sequence alone has one of every CTA: 1 x 32768 slots
// took 90 us with a warp a head, 24 with <8, 1>, 18.5 with <16, 4> (16 blocks of <16, 1> read 0.5 MB
// each, an SM's 4 us: 23).
constexpr int kWideRows = 48, kWiderRows = 4, kMergeMost = 32;
template <int W, int D>
__global__ void __launch_bounds__(32 * W) merge_wide_kernel(const AttnParams p, int least) {
  constexpr int kW = 4 / D;  // of the four w of merge_kernel
  __shared__ float4 sum[W][kLatent / 4 / D];
  __shared__ float2 ml_of[W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.y, tile = blockIdx.x >> 4, r = blockIdx.x & 15;
  if (tile * 16 + r >= p.heads) return;  // (head 0 has blocks)
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int2 w = partials_of(p, b, tile);
  if (w.y == 1 || w.y < least) return;
  const float* ml = p.part_ml + static_cast<int64_t>(w.x) * 32 + r;
  const int cc = lane & 3, jk = lane >> 2;  // as in merge_kernel
  const float4* po = reinterpret_cast<const float4*>(p.part_o) +
                     (static_cast<int64_t>(w.x) * 64 + (r >> 3) * 8 + jk) * 32 + (r & 7) * 4 + cc +
                     16 * 32 * kW * static_cast<int>(blockIdx.z);
  const int used = min(w.y, W);
  if (warp < used) {
    float M = -INFINITY, L = 0.f;
    float a[4 * kW];
#pragma unroll
    for (int k = 0; k < 4 * kW; ++k) a[k] = 0.f;
    const int n = (w.y - warp + W - 1) / W;  // partials warp, warp + 8, ..
    for (int i0 = 0; i0 < n; i0 += 32) {
      const bool in = i0 + lane < n;
      const int64_t at = static_cast<int64_t>(i0 + lane) * W + warp;
      const float m = in ? __ldcg(ml + at * 32) : -INFINITY;
      float l = in ? __ldcg(ml + at * 32 + 16) : 0.f;
      float mx = fmaxf(m, M);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const float ref = mx == -INFINITY ? 0.f : mx;
      const float keep = ptx::ex2(M - ref);
      const float f = in ? ptx::ex2(m - ref) : 0.f;
      l *= f;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
      L = fmaf(L, keep, l);
      M = mx;
#pragma unroll
      for (int k = 0; k < 4 * kW; ++k) a[k] *= keep;
#pragma unroll (4 * D > 8 ? 8 : 4 * D)
      for (int i = 0; i < min(32, n - i0); ++i) {
        const float fi = __shfl_sync(0xffffffffu, f, i);
        const float4* src = po + (static_cast<int64_t>(i0 + i) * W + warp) * (16 * kLatent / 4);
#pragma unroll
        for (int k = 0; k < kW; ++k) {
          const float4 v = __ldcg(src + 16 * 32 * k);
          a[4 * k] = fmaf(fi, v.x, a[4 * k]);
          a[4 * k + 1] = fmaf(fi, v.y, a[4 * k + 1]);
          a[4 * k + 2] = fmaf(fi, v.z, a[4 * k + 2]);
          a[4 * k + 3] = fmaf(fi, v.w, a[4 * k + 3]);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kW; ++k)
      sum[warp][32 * k + lane] = make_float4(a[4 * k], a[4 * k + 1], a[4 * k + 2], a[4 * k + 3]);
    if (lane == 0) ml_of[warp] = make_float2(M, L);
  }
  __syncthreads();
  if (warp >= kW) return;
  // warp k: the lane's four dimensions of the block's k-th w
  float M = -INFINITY, L = 0.f;
  for (int k = 0; k < used; ++k) M = fmaxf(M, ml_of[k].x);
  const float ref = M == -INFINITY ? 0.f : M;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < used; ++k) {
    const float f = ptx::ex2(ml_of[k].x - ref);
    const float4 v = sum[k][threadIdx.x];
    L = fmaf(f, ml_of[k].y, L);
    o.x = fmaf(f, v.x, o.x);
    o.y = fmaf(f, v.y, o.y);
    o.z = fmaf(f, v.z, o.z);
    o.w = fmaf(f, v.w, o.w);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const __nv_bfloat162 x = __floats2bfloat162_rn(o.x * inv, o.y * inv);
  const __nv_bfloat162 y = __floats2bfloat162_rn(o.z * inv, o.w * inv);
  __nv_bfloat16* dst = p.out + (static_cast<int64_t>(b) * p.heads + tile * 16 + r) * kLatent;
  *reinterpret_cast<uint2*>(dst + 128 * (kW * blockIdx.z + warp) + 16 * (2 * cc + (jk >> 2)) + 4 * (jk & 3)) =
      make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
  if (p.lse != nullptr && threadIdx.x == 0 && blockIdx.z == 0)
    p.lse[(static_cast<int64_t>(b) * p.tiles + tile) * 16 + r] = M + log2f(L);
}

// mass[t] = decay mass[t] + sum_h 2^(s_h(t) - lse_h); one chunk of one sequence a block.
__global__ void __launch_bounds__(kChunk) mass_kernel(const AttnParams p, float decay) {
  __shared__ float slse[kMaxHeads];
  const int tid = threadIdx.x, b = blockIdx.y, chunk = blockIdx.x;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int len = min(p.c.state[b], p.c.slots);
  if (chunk * kChunk >= len) return;
  if (tid < p.heads) slse[tid] = __ldcg(p.lse + static_cast<int64_t>(b) * p.tiles * 16 + tid);
  __syncthreads();
  const int t = chunk * kChunk + frag_slot(tid);
  float a = 0.f;
  for (int tile = 0; tile < p.tiles; ++tile) {
    const float* s = p.scores +
                     ((static_cast<int64_t>(b) * p.tiles + tile) * p.max_chunks + chunk) * 16 * kChunk + tid;
    if (p.heads >= 16 * tile + 16) {
      float v[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) v[r] = __ldcg(s + r * kChunk);
#pragma unroll
      for (int r = 0; r < 16; ++r) a += ptx::ex2(v[r] - slse[tile * 16 + r]);
    } else {
      for (int r = 0; r < p.heads - 16 * tile; ++r)
        a += ptx::ex2(__ldcg(s + r * kChunk) - slse[tile * 16 + r]);
    }
  }
  if (t >= len) return;
  float* m = p.c.mass + static_cast<int64_t>(b) * p.c.slots + t;
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

// Result slots j0 .. j0 + 3 of sequence b take the rows t of lanes 0 .. 3 (of lanes 4 .. 7 and so
// on again; -1: none): a warp's work, all loads before the stores.  Lanes: 18 16-byte pieces of codes a row, and for the small fields one
// (field, row) each.  In place, rows that stay are skipped: sources lie at or behind the budget
// and targets before it, so no row is both.
constexpr int kMoveRows = 4;
__device__ __forceinline__ void move_rows(const Cache& s, const Cache& d, int b, int j0, int t,
                                          bool in_place) {
  const int lane = threadIdx.x & 31;
  const int mine = lane & 3;
  if (in_place && t == j0 + mine) t = -1;
  uint4 v[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int i = lane + 32 * k, row = i / 18;
    const int tr = __shfl_sync(0xffffffffu, t, row & 3);
    if (row < kMoveRows && tr >= 0)
      v[k] = __ldcg(reinterpret_cast<const uint4*>(
                        s.codes + (static_cast<int64_t>(b) * s.slots + tr) * kRowBytes) + i % 18);
  }
  const int f = lane >> 2;  // field: 0-4 scales, 5 rstd, 6 position, 7 mass
  const int64_t ss = static_cast<int64_t>(b) * s.slots + t, ds = static_cast<int64_t>(b) * d.slots + j0 + mine;
  const int64_t gs = (static_cast<int64_t>(b) * kGroups + f) * s.slots + t;
  const int64_t gd = (static_cast<int64_t>(b) * kGroups + f) * d.slots + j0 + mine;
  __nv_bfloat16 g = __float2bfloat16_rn(0.f);
  uint32_t w = 0u;
  if (t >= 0) {
    if (f < 5) g = s.scales[gs];
    else w = __ldcg((f == 5   ? reinterpret_cast<const uint32_t*>(s.rstd)
                     : f == 6 ? reinterpret_cast<const uint32_t*>(s.pos)
                              : reinterpret_cast<const uint32_t*>(s.mass)) + ss);
  }
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const int i = lane + 32 * k, row = i / 18;
    const int tr = __shfl_sync(0xffffffffu, t, row & 3);
    if (row < kMoveRows && tr >= 0)
      reinterpret_cast<uint4*>(d.codes + (static_cast<int64_t>(b) * d.slots + j0 + row) * kRowBytes)[i % 18] = v[k];
  }
  if (t >= 0) {
    if (f < 5) d.scales[gd] = g;
    else (f == 5   ? reinterpret_cast<uint32_t*>(d.rstd)
          : f == 6 ? reinterpret_cast<uint32_t*>(d.pos)
                   : reinterpret_cast<uint32_t*>(d.mass))[ds] = w;
  }
}

// Exclusive prefix of v over the block's threads (1024); `red`: 32 words that no earlier call in
// flight uses.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += y;
  }
  if (lane == 31) red[warp] = incl;
  __syncthreads();
  const uint32_t before = __reduce_add_sync(0xffffffffu, lane < warp ? red[lane] : 0u);
  return before + incl - v;
}

// One round of the search: a1, a2, a3 keys are at or above v + 1, 2, 3 << shift; the largest of
// the four bounds that `want` keys reach becomes v, and the range what lies up to the next.
__device__ __forceinline__ void narrow(int want, int shift, int a1, int a2, int a3, uint32_t* v,
                                       int* in_range, int* over_end) {
  if (a3 >= want) {
    *v |= 3u << shift;
    *in_range = a3 - *over_end;
  } else if (a2 >= want) {
    *v |= 2u << shift;
    *in_range = a2 - a3;
    *over_end = a3;
  } else if (a1 >= want) {
    *v |= 1u << shift;
    *in_range = a1 - a2;
    *over_end = a2;
  } else {
    *in_range += *over_end - a1;
    *over_end = a1;
  }
}
// The same among n <= kFewKeys keys of a list, by the block's first four warps, four keys a lane;
// returns the value with v's bits completed.
constexpr int kFewKeys = 512;
__device__ __forceinline__ uint32_t find_in_list(const uint32_t* list, int n, int want, int shift,
                                                 uint32_t v, uint32_t (*part)[4]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t k[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) k[i] = threadIdx.x + 128 * i < n ? list[threadIdx.x + 128 * i] : 0u;
#pragma unroll 1
  for (int round = 0; shift >= 0; shift -= 2, ++round) {
    const uint32_t c1 = v | (1u << shift), c2 = v | (2u << shift), c3 = v | (3u << shift);
    uint32_t x = 0;  // three counts of 10 bits
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x += (k[i] >= c1 ? 1u : 0u) + (k[i] >= c2 ? 1u << 10 : 0u) + (k[i] >= c3 ? 1u << 20 : 0u);
    x = __reduce_add_sync(0xffffffffu, x);
    if (lane == 0) part[round & 1][warp] = x;
    __syncwarp();
    ptx::named_bar_sync(1, 128);
    const uint4 y = *reinterpret_cast<const uint4*>(part[round & 1]);
    x = (y.x + y.y) + (y.z + y.w);
    if (static_cast<int>(x >> 20) >= want) v = c3;
    else if (static_cast<int>((x >> 10) & 1023u) >= want) v = c2;
    else if (static_cast<int>(x & 1023u) >= want) v = c1;
  }
  return v;
}

// One block per sequence: which slots stay, and src_of[b, j] = the slot whose row result slot j
// takes: itself where slot j < budget stays, else the next survivor from behind the budget,
// both in ascending order.  Up to 1024 * IPT slots, whose keys stay in registers (thread i has
// slots IPT i ..).  The budget-th largest key is found two bits a round, by counting the keys at
// or above three candidates: no histogram, whose atomics collide when weights are alike (four
// passes of 8 bits took 23 us for 333 slots and 68 us for 8192).  A round of the whole block
// takes 450 cycles and 100 a key of a thread, so once kFewKeys or fewer keys share the bits found
// so far, they go to shared memory and four warps find the rest (one warp took 500 a round, and
// counting the keys before each key, n^2 comparisons, 10800 for 333).
// `rows_here` (budget <= kRowsHere): the block moves the rows itself.
constexpr int kRowsHere = 256;
constexpr int kSharedPlan = 2048;  // budgets whose lists fit shared memory
template <int IPT>
__global__ void __launch_bounds__(1024)
    evict_plan_kernel(Cache c, Cache dst, int budget, int recent, int32_t* src_of,
                      int32_t* holes, int rows_here, int in_place) {
  __shared__ uint32_t red[6][32];
  __shared__ uint32_t list[kFewKeys];
  __shared__ int32_t src_s[kSharedPlan], hole_s[kSharedPlan];
  __shared__ uint32_t found;
  __shared__ __align__(16) uint32_t part[2][4];
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int b = blockIdx.x, lane = threadIdx.x & 31;
  const int t0 = threadIdx.x * IPT;
  // weights and positions are on their way while the lengths are read
  const float* mass = c.mass + static_cast<int64_t>(b) * c.slots;
  const int32_t* pos = c.pos + static_cast<int64_t>(b) * c.slots;
  float m[IPT];
  int ps[IPT];
  if (IPT >= 4) {
#pragma unroll
    for (int i = 0; i < IPT; i += 4)
      if (t0 + i < c.slots) {  // (slots are a multiple of 64)
        *reinterpret_cast<float4*>(m + i) = *reinterpret_cast<const float4*>(mass + t0 + i);
        *reinterpret_cast<int4*>(ps + i) = *reinterpret_cast<const int4*>(pos + t0 + i);
      }
  } else if (t0 < c.slots) {
    m[0] = mass[t0];
    ps[0] = pos[t0];
  }
  const int len = min(max(c.state[b], 0), c.slots), next = c.state[c.batch + b];
  int32_t* const out = src_of + static_cast<int64_t>(b) * budget;
  const bool shared = budget <= kSharedPlan;
  int32_t* src = shared ? src_s : out;
  int32_t* hole = shared ? hole_s : holes + static_cast<int64_t>(b) * budget;
  const int kept_n = min(len, budget);
  if (len > budget) {
    const int from = next - recent;
    uint32_t key[IPT];
#pragma unroll
    for (int i = 0; i < IPT; ++i)  // slots behind the last: 0, below every candidate
      key[i] = t0 + i < len ? evict_key(m[i], ps[i], from) : 0u;
    // the largest v with at least `budget` keys >= v
    uint32_t v = 0;
    int in_range = len;  // keys in [v, v + 2^(shift + 2)) before a round ...
    int over_end = 0;    // ... and at or above its end
    int shift = 30;
#pragma unroll 1
    for (int round = 0; shift >= 0 && in_range > kFewKeys; shift -= 2, ++round) {
      uint32_t n12 = 0, n3 = 0;
      const uint32_t c1 = v | (1u << shift), c2 = v | (2u << shift), c3 = v | (3u << shift);
#pragma unroll
      for (int i = 0; i < IPT; ++i) {
        n12 += (key[i] >= c1 ? 1u : 0u) + (key[i] >= c2 ? 0x10000u : 0u);
        n3 += key[i] >= c3 ? 1u : 0u;
      }
      // (a block has at most 8192 keys: two counts to a word)
      const uint32_t w12 = __reduce_add_sync(0xffffffffu, n12);
      const uint32_t w3 = __reduce_add_sync(0xffffffffu, n3);
      uint32_t* r = red[2 * (round & 1)];
      if (lane == 0) {
        r[threadIdx.x >> 5] = w12;
        r[32 + (threadIdx.x >> 5)] = w3;
      }
      __syncthreads();
      const uint32_t s12 = __reduce_add_sync(0xffffffffu, r[lane]);
      const int a1 = static_cast<int>(s12 & 0xFFFFu), a2 = static_cast<int>(s12 >> 16);
      const int a3 = static_cast<int>(__reduce_add_sync(0xffffffffu, r[32 + lane]));
      narrow(budget, shift, a1, a2, a3, &v, &in_range, &over_end);
    }
    if (shift >= 0) {  // the rest by four warps: the keys in range, the others counted
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < IPT; ++i)
        mine += t0 + i < len && (shift == 30 || (key[i] >> (shift + 2)) == (v >> (shift + 2))) ? 1u : 0u;
      uint32_t at = block_prefix(mine, red[4]);
#pragma unroll
      for (int i = 0; i < IPT; ++i)
        if (t0 + i < len && (shift == 30 || (key[i] >> (shift + 2)) == (v >> (shift + 2))))
          list[at++] = key[i];
      __syncthreads();
      if (threadIdx.x < 128) {
        const uint32_t f = find_in_list(list, in_range, budget - over_end, shift, v, part);
        if (threadIdx.x == 0) found = f;
      }
      __syncthreads();
      v = found;
    }
    uint32_t above = 0, ties = 0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      above += key[i] > v ? 1u : 0u;
      ties += key[i] == v && t0 + i < len ? 1u : 0u;
    }
    // ties that stay: the first ones (both counts are at most 8192)
    const uint32_t packed = above | (ties << 16);
    const uint32_t before_t = block_prefix(packed, red[5]);
    uint32_t rank = before_t >> 16;
    // the last warp's last thread ends the prefix: the block's total of `above`
    if (threadIdx.x == 1023) list[0] = (before_t + packed) & 0xFFFFu;
    __syncthreads();
    const uint32_t need = budget - list[0];
    uint32_t keep = 0, n_hole = 0, n_late = 0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const int t = t0 + i;
      bool k = key[i] > v;
      if (key[i] == v && t < len) k = rank++ < need;
      if (k) keep |= 1u << i;
      n_hole += t < budget && !k ? 1u : 0u;
      n_late += t >= budget && k ? 1u : 0u;
    }
    const uint32_t before = block_prefix(n_hole | (n_late << 16), red[4]);
    uint32_t h = before & 0xFFFFu, l = before >> 16;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const int t = t0 + i;
      if (t >= budget) continue;
      if (keep >> i & 1u) src[t] = t;
      else hole[h++] = t;
    }
    __syncthreads();  // the holes are written before survivors are paired with them
#pragma unroll
    for (int i = 0; i < IPT; ++i)
      if (t0 + i >= budget && (keep >> i & 1u)) src[hole[l++]] = t0 + i;
  } else {
    for (int j = threadIdx.x; j < kept_n; j += 1024) src[j] = j;
  }
  __syncthreads();
  if (rows_here)
    for (int j = (threadIdx.x >> 5) * kMoveRows; j < kept_n; j += 32 * kMoveRows) {
      const int k = j + (lane & 3);
      move_rows(c, dst, b, j, k < kept_n ? src_s[k] : -1, in_place != 0);
    }
  else if (shared)
    for (int j = threadIdx.x; j < kept_n; j += 1024) out[j] = src_s[j];
  if (threadIdx.x == 0) {
    dst.state[b] = kept_n;
    dst.state[c.batch + b] = next;
  }
}

// Sums of three counts over the cluster's blocks, and over those before this one: each block's go to
// all (`x`: [2][8] entries; calls alternate between the two, and the barrier of the one between them
// says that everyone has read the last).
struct ClusterSum {
  int all[3], before[3];
};
__device__ __forceinline__ ClusterSum cluster_sum(int u, int v, int w, int4 (*x)[8], int turn) {
  const uint32_t rank = ptx::cluster_ctarank();
  uint32_t size;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  if (threadIdx.x < size) {
    const uint32_t to = ptx::mapa_shared(ptx::smem_u32(&x[turn & 1][rank]), threadIdx.x);
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(u), "r"(v), "r"(w), "r"(0)
                 : "memory");
  }
  __syncwarp();  // the barrier is `.aligned`: a warp's lanes have to reach it together
  ptx::cluster_sync();
  ClusterSum s = {};
  for (uint32_t k = 0; k < size; ++k) {
    const int4 y = x[turn & 1][k];
    const int z[3] = {y.x, y.y, y.z};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      s.all[i] += z[i];
      if (k < rank) s.before[i] += z[i];
    }
  }
  return s;
}

// The plan of more slots by a cluster of blocks a sequence, 1024 * IPT slots each: as above, with the
// counts of every round summed over the cluster, the last keys found by its first block, and the lists in
// global memory.  (8 x 32768 slots to 4096: 29.5 us against 53 with 32 keys a thread in one block; 2 x
// 100000 to 4096: 67 against 635 with histograms.)
template <int IPT>
__global__ void __launch_bounds__(1024)
    evict_plan_cluster_kernel(Cache c, Cache dst, int budget, int recent, int32_t* src_of, int32_t* holes) {
  __shared__ uint32_t red[4][32];
  __shared__ uint32_t list[kFewKeys];
  __shared__ uint32_t found;
  __shared__ __align__(16) uint32_t part[2][4];
  __shared__ __align__(16) int4 counts[2][8];
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  uint32_t blocks;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
  const int b = blockIdx.x / blocks, lane = threadIdx.x & 31;
  const int t0 = (rank * 1024 + threadIdx.x) * IPT;
  const float* mass = c.mass + static_cast<int64_t>(b) * c.slots;
  const int32_t* pos = c.pos + static_cast<int64_t>(b) * c.slots;
  float m[IPT];
  int ps[IPT];
#pragma unroll
  for (int i = 0; i < IPT; i += 4)
    if (t0 + i < c.slots) {  // (slots are a multiple of 64)
      *reinterpret_cast<float4*>(m + i) = *reinterpret_cast<const float4*>(mass + t0 + i);
      *reinterpret_cast<int4*>(ps + i) = *reinterpret_cast<const int4*>(pos + t0 + i);
    }
  const int len = min(max(c.state[b], 0), c.slots), next = c.state[c.batch + b];
  __syncwarp();  // (some lanes may have had slots to load)
  ptx::cluster_sync();  // all blocks have started, and have read the length
  int32_t* const src = src_of + static_cast<int64_t>(b) * budget;
  int32_t* const hole = holes + static_cast<int64_t>(b) * budget;
  const int kept_n = min(len, budget);
  if (len > budget) {  // (the same for all of the cluster)
    const int from = next - recent;
    uint32_t key[IPT];
#pragma unroll
    for (int i = 0; i < IPT; ++i) key[i] = t0 + i < len ? evict_key(m[i], ps[i], from) : 0u;
    uint32_t v = 0;
    int in_range = len, over_end = 0, shift = 30, turn = 0;
#pragma unroll 1
    for (; shift >= 0 && in_range > kFewKeys; shift -= 2, ++turn) {
      uint32_t n12 = 0, n3 = 0;
      const uint32_t c1 = v | (1u << shift), c2 = v | (2u << shift), c3 = v | (3u << shift);
#pragma unroll
      for (int i = 0; i < IPT; ++i) {
        n12 += (key[i] >= c1 ? 1u : 0u) + (key[i] >= c2 ? 0x10000u : 0u);
        n3 += key[i] >= c3 ? 1u : 0u;
      }
      // (a block has at most 32768 keys: two counts to a word)
      const uint32_t w12 = __reduce_add_sync(0xffffffffu, n12);
      const uint32_t w3 = __reduce_add_sync(0xffffffffu, n3);
      if (lane == 0) {
        red[0][threadIdx.x >> 5] = w12;
        red[1][threadIdx.x >> 5] = w3;
      }
      __syncthreads();
      const uint32_t s12 = __reduce_add_sync(0xffffffffu, red[0][lane]);
      const uint32_t s3 = __reduce_add_sync(0xffffffffu, red[1][lane]);
      const ClusterSum s = cluster_sum(s12 & 0xFFFFu, s12 >> 16, s3, counts, turn);
      narrow(budget, shift, s.all[0], s.all[1], s.all[2], &v, &in_range, &over_end);
    }
    if (shift >= 0) {  // the rest by four warps of the first block
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < IPT; ++i)
        mine += t0 + i < len && (shift == 30 || (key[i] >> (shift + 2)) == (v >> (shift + 2))) ? 1u : 0u;
      uint32_t at = block_prefix(mine, red[2]);
      if (threadIdx.x == 1023) red[3][0] = at + mine;
      __syncthreads();
      at += cluster_sum(red[3][0], 0, 0, counts, turn++).before[0];
      const uint32_t first = ptx::mapa_shared(ptx::smem_u32(list), 0);
#pragma unroll
      for (int i = 0; i < IPT; ++i)
        if (t0 + i < len && (shift == 30 || (key[i] >> (shift + 2)) == (v >> (shift + 2)))) {
          asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(first + 4 * at), "r"(key[i]) : "memory");
          ++at;
        }
      __syncwarp();
      ptx::cluster_sync();
      if (rank == 0 && threadIdx.x < 128) {
        const uint32_t f = find_in_list(list, in_range, budget - over_end, shift, v, part);
        if (threadIdx.x < blocks)
          asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(ptx::mapa_shared(ptx::smem_u32(&found), threadIdx.x)),
                       "r"(f)
                       : "memory");
      }
      __syncwarp();
      ptx::cluster_sync();
      v = found;
    }
    uint32_t above = 0, ties = 0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      above += key[i] > v ? 1u : 0u;
      ties += key[i] == v && t0 + i < len ? 1u : 0u;
    }
    __syncthreads();  // (the words of `red` are free)
    const uint32_t packed = above | (ties << 16);
    const uint32_t before_t = block_prefix(packed, red[0]);
    if (threadIdx.x == 1023) red[3][1] = before_t + packed;
    __syncthreads();
    const ClusterSum kept = cluster_sum(red[3][1] & 0xFFFFu, red[3][1] >> 16, 0, counts, turn++);
    // ties that stay: the first ones
    int rank_t = static_cast<int>(before_t >> 16) + kept.before[1];
    const int need = budget - kept.all[0];
    uint32_t keep = 0, n_hole = 0, n_late = 0;
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const int t = t0 + i;
      bool k = key[i] > v;
      if (key[i] == v && t < len) k = rank_t++ < need;
      if (k) keep |= 1u << i;
      n_hole += t < budget && !k ? 1u : 0u;
      n_late += t >= budget && k ? 1u : 0u;
    }
    const uint32_t moved = n_hole | (n_late << 16);
    const uint32_t before = block_prefix(moved, red[1]);
    if (threadIdx.x == 1023) red[3][2] = before + moved;
    __syncthreads();
    const ClusterSum gone = cluster_sum(red[3][2] & 0xFFFFu, red[3][2] >> 16, 0, counts, turn++);
    int h = static_cast<int>(before & 0xFFFFu) + gone.before[0];
    int l = static_cast<int>(before >> 16) + gone.before[1];
#pragma unroll
    for (int i = 0; i < IPT; ++i) {
      const int t = t0 + i;
      if (t >= budget) continue;
      if (keep >> i & 1u) src[t] = t;
      else hole[h++] = t;
    }
    __syncwarp();
    ptx::cluster_sync();  // the holes are written before survivors are paired with them
#pragma unroll
    for (int i = 0; i < IPT; ++i)
      if (t0 + i >= budget && (keep >> i & 1u)) src[__ldcg(hole + l++)] = t0 + i;
  } else {
    for (int j = rank * 1024 + threadIdx.x; j < kept_n; j += 1024 * static_cast<int>(blocks)) src[j] = j;
  }
  if (rank == 0 && threadIdx.x == 0) {
    dst.state[b] = kept_n;
    dst.state[c.batch + b] = next;
  }
}

// The same for any number of slots: the keys are made again for each pass, four of which build
// histograms of 8 bits, and slots are ranked tile by tile.
__global__ void __launch_bounds__(1024)
    evict_plan_long_kernel(Cache c, Cache dst, int budget, int recent,
                      int32_t* src_of, int32_t* holes) {
  __shared__ int hist[256];
  __shared__ int warp_sum[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
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
    dst.state[b] = kept_n;
    dst.state[c.batch + b] = next;
  }
}

// The rows of a plan.
__global__ void __launch_bounds__(256)
    evict_move_kernel(Cache s, Cache d, int budget, const int32_t* src_of,
                      int in_place) {
  ptx::pdl_wait();
  ptx::pdl_launch_dependents();
  const int b = blockIdx.y;
  const int j = (blockIdx.x * 8 + (threadIdx.x >> 5)) * kMoveRows;
  const int n = __ldcg(d.state + b);
  if (j >= n) return;
  const int k = j + (threadIdx.x & 3);
  move_rows(s, d, b, j, k < n ? __ldcg(src_of + static_cast<int64_t>(b) * budget + k) : -1,
            in_place != 0);
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

struct AttnBuffers {
  int2* where;
  float* part_o;
  float* part_ml;
  float* scores;
  float* lse;
};

// CTAs of the attention kernel: as many as run at once, no more than there can be chunks.
int attn_ctas(int batch, int tiles, int max_chunks, int num_sms) {
  const int64_t units = static_cast<int64_t>(batch) * tiles * max_chunks;
  const int most = kCtasPerSm * num_sms;
  return static_cast<int>(units < most ? (units < 1 ? 1 : units) : most);
}

void carve_attn(Carve& w, AttnBuffers* b, int batch, int heads, int max_len, int num_sms,
                bool mass) {
  const int tiles = (heads + 15) / 16, chunks = (max_len + kChunk - 1) / kChunk;
  // a partial segment shares its (sequence, head tile) with another one, so there are no more
  // than CTAs; with more sequences than CTAs every segment is whole, and numbered further
  const size_t parts = std::max<size_t>(attn_ctas(batch, tiles, chunks, num_sms), 1);
  b->where = w.take<int2>(static_cast<size_t>(batch) * tiles);
  b->part_o = w.take<float>(parts * 16 * kLatent);
  b->part_ml = w.take<float>(parts * 32);
  b->lse = mass ? w.take<float>(static_cast<size_t>(batch) * tiles * 16) : nullptr;
  b->scores =
      mass ? w.take<float>(static_cast<size_t>(batch) * tiles * chunks * 16 * kChunk) : nullptr;
}

bool g_attr_set[64] = {};
std::mutex g_attr_mutex;

int launch_append(const Cache& c, const void* lat, int64_t lat_ld, const void* kpe,
                  int64_t kpe_ld, int64_t src_bstride, int n_new, const int32_t* new_lens,
                  const void* cos_t, const void* sin_t, int table_rows, float eps,
                  cudaStream_t s) {
  if (c.batch == 0 || n_new == 0) return DS_OK;
  const int tokens = n_new <= 64 ? 8 : 32;  // of a block
  const bool many = tokens == 32 && static_cast<int64_t>(c.batch) * n_new >= kManyTokens;
  DS_CUDA(launch_chained(
      many ? append_kernel<4> : append_kernel<1>, dim3((n_new + tokens - 1) / tokens, c.batch),
      dim3(many ? 256 : 32 * tokens), 0, s, 1, c, static_cast<const __nv_bfloat16*>(lat), lat_ld,
      static_cast<const __nv_bfloat16*>(kpe), kpe_ld, src_bstride, n_new, new_lens,
      static_cast<const __nv_bfloat16*>(cos_t), static_cast<const __nv_bfloat16*>(sin_t), table_rows,
      eps));
  DS_LAUNCH_CHECK("append_kernel");
  return DS_OK;
}

int launch_evict(const Cache& s, const Cache& d, int budget, int recent, bool in_place,
                 int32_t* src_of, int32_t* holes, cudaStream_t st) {
  // One block a sequence up to 8192 slots, whatever the batch: clusters of two or more (four keys a thread)
  // meet over the SMs in every round and need the second launch, 8192 slots to 256: 17.6 us against 14.5
  // (1 sequence), 18.7 against 14.7 (32), 31.2 against 19.2 (148); 2048 slots to 1024: 16.6 against 12.2,
  // 20.4 against 15.6, 41.0 against 30.7.
  // Few rows: the planning block moves them (no second launch); many: all SMs do.
  const bool one = s.slots <= 8192, here = one && budget <= kRowsHere;
  if (one) {
    DS_CUDA(launch_chained(s.slots <= 1024 ? evict_plan_kernel<1> : evict_plan_kernel<8>, dim3(s.batch),
                           dim3(1024), 0, st, 1, s, d, budget, recent, src_of, holes, here ? 1 : 0,
                           in_place ? 1 : 0));
  } else if (s.slots <= 262144) {
    const int ipt = s.slots <= 65536 ? 8 : 32;
    int blocks = 2;
    while (blocks * ipt * 1024 < s.slots) blocks *= 2;
    DS_CUDA(launch_chained(ipt == 8 ? evict_plan_cluster_kernel<8> : evict_plan_cluster_kernel<32>,
                           dim3(s.batch * blocks), dim3(1024), 0, st, blocks, s, d, budget, recent, src_of,
                           holes));
  } else {
    DS_CUDA(launch_chained(evict_plan_long_kernel, dim3(s.batch), dim3(1024), 0, st, 1, s, d,
                           budget, recent, src_of, holes));
  }
  DS_LAUNCH_CHECK("evict_plan_kernel");
  if (here) return DS_OK;
  DS_CUDA(launch_chained(evict_move_kernel,
                         dim3((budget + 8 * kMoveRows - 1) / (8 * kMoveRows), s.batch), dim3(256),
                         0, st, 1, s, d, budget, static_cast<const int32_t*>(src_of),
                         in_place ? 1 : 0));
  DS_LAUNCH_CHECK("evict_move_kernel");
  return DS_OK;
}

int launch_attention(const Cache& c, const void* q, int heads, int max_len, float softmax_scale,
                     int accumulate, float decay, void* out, void* workspace, size_t ws_bytes,
                     cudaStream_t s) {
  if (c.batch == 0) return DS_OK;
  DeviceInfo di;
  DS_TRY(device_info(&di));
  AttnParams p{};
  p.c = c;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.heads = heads;
  p.tiles = (heads + 15) / 16;
  p.max_chunks = (max_len + kChunk - 1) / kChunk;
  p.scale_log2 = static_cast<float>(static_cast<double>(softmax_scale) * 1.4426950408889634);
  Carve w(workspace, ws_bytes);
  AttnBuffers b{};
  carve_attn(w, &b, c.batch, heads, max_len, di.num_sms, accumulate != 0);
  if (!w.ok())
    return fail(DS_ERR_WORKSPACE, "mla_decode_attention4: workspace needs %zu bytes", w.used);
  p.where = b.where;
  p.part_o = b.part_o;
  p.part_ml = b.part_ml;
  p.scores = b.scores;
  p.lse = b.lse;
  p.status = device_status_ptr();
  if (p.status == nullptr) return fail(DS_ERR_CUDA, "device status word unavailable");
  {
    std::lock_guard<std::mutex> lock(g_attr_mutex);
    if (!g_attr_set[di.device]) {
      DS_CUDA(cudaFuncSetAttribute(attend4_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   static_cast<int>(kAttnSmem)));
      g_attr_set[di.device] = true;
    }
  }
  p.ctas = attn_ctas(c.batch, p.tiles, p.max_chunks, di.num_sms);
  if (max_len > 0) {
    DS_CUDA(launch_chained(attend4_kernel, dim3(p.ctas), dim3(kAttnThreads), kAttnSmem, s, 1, p));
    DS_LAUNCH_CHECK("attend4_kernel");
  }
  // the kernel for many partials takes all of few rows, and of many rows those that have more than
  // kMergeMost all the same
  const int64_t rows = static_cast<int64_t>(c.batch) * p.tiles;
  const bool few = rows <= kWideRows;
  if (!few)
    DS_CUDA(launch_chained(merge_kernel, dim3(p.tiles * 4, c.batch), dim3(kAttnThreads), 0, s, 1, p, kMergeMost));
  if (rows <= kWiderRows)
    DS_CUDA(launch_chained(merge_wide_kernel<16, 4>, dim3(p.tiles * 16, c.batch, 4), dim3(512), 0, s, 1, p, 0));
  else if (few || std::min(p.max_chunks, p.ctas) > kMergeMost)
    DS_CUDA(launch_chained(merge_wide_kernel<8, 1>, dim3(p.tiles * 16, c.batch), dim3(256), 0, s, 1, p,
                           few ? 0 : kMergeMost + 1));
  DS_LAUNCH_CHECK("merge_kernel");
  if (accumulate && max_len > 0) {
    DS_CUDA(launch_chained(mass_kernel, dim3(p.max_chunks, c.batch), dim3(kChunk), 0, s, 1, p, decay));
    DS_LAUNCH_CHECK("mass_kernel");
  }
  return DS_OK;
}

// A decode step's buffers in its workspace.
struct StepBuffers {
  __nv_bfloat16* proj;  // [batch, heads * 576 + 576]
  __nv_bfloat16* q;     // [batch, heads, 576]
  __nv_bfloat16* olat;  // [batch, heads * 512]
  uint8_t* linear;
  size_t linear_bytes;
  uint8_t* attn;
  size_t attn_bytes;
};
void carve_step(Carve& w, StepBuffers* s, int batch, int heads, int hidden, int max_len,
                int num_sms, bool mass) {
  Carve a(nullptr, 0);
  AttnBuffers ab{};
  carve_attn(a, &ab, batch, heads, max_len, num_sms, mass);
  s->attn_bytes = align_up(a.used, 256);
  s->linear_bytes = std::max(i8::linear_workspace(batch, hidden),
                             i8::linear_workspace(batch, heads * kLatent));
  s->proj = w.take<__nv_bfloat16>(static_cast<size_t>(batch) * (heads + 1) * kQCols);
  s->q = w.take<__nv_bfloat16>(static_cast<size_t>(batch) * heads * kQCols);
  s->olat = w.take<__nv_bfloat16>(static_cast<size_t>(batch) * heads * kLatent);
  s->linear = w.take<uint8_t>(s->linear_bytes);
  s->attn = w.take<uint8_t>(s->attn_bytes);
}

}  // namespace
}  // namespace c4
}  // namespace ds

// ---- C ABI ------------------------------------------------------------------------------------
extern "C" {

int ds_mla_cache4_reset(int32_t* state, int batch, void* stream) {
  DS_REQUIRE(batch >= 0 && batch <= 65535, "mla_cache4_reset: batch must be at most 65535");
  if (batch == 0) return DS_OK;
  DS_REQUIRE(state != nullptr, "mla_cache4_reset: null pointer");
  DS_CUDA(ds::launch_chained(ds::c4::reset_kernel, dim3(1), dim3(256), 0,
                             static_cast<cudaStream_t>(stream), 1, state, 3 * batch));
  DS_LAUNCH_CHECK("reset_kernel");
  return DS_OK;
}

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
  DS_REQUIRE(ds::aligned2(cos_bf16) && ds::aligned2(sin_bf16),
             "mla_cache4_append: misaligned RoPE tables");
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
  DS_REQUIRE(ds::aligned16(codes) && ds::aligned16(scales_bf16) &&
                 ds::aligned16(latent_out_bf16) && ds::aligned16(kpe_out_bf16),
             "mla_cache4_get: codes, scales and outputs must be 16-byte aligned");
  DS_REQUIRE(batch <= 65535, "mla_cache4_get: batch must be at most 65535");
  const ds::c4::Cache c = ds::c4::cache_of(const_cast<void*>(codes), const_cast<void*>(scales_bf16),
                                           nullptr, nullptr, nullptr,
                                           const_cast<int32_t*>(state), batch, slots);
  const int per_block = 8 * ds::c4::kGetSlots;
  DS_CUDA(ds::launch_chained(ds::c4::get_kernel,
                             dim3((seq_len + per_block - 1) / per_block, batch), dim3(256), 0,
                             static_cast<cudaStream_t>(stream), 1, c, seq_len,
                             static_cast<uint4*>(latent_out_bf16),
                             static_cast<uint4*>(kpe_out_bf16)));
  DS_LAUNCH_CHECK("get_kernel");
  return DS_OK;
}

size_t ds_mla_decode_attention4_workspace_size(int batch, int heads, int slots, int max_len,
                                               int accumulate) {
  (void)slots;
  if (batch <= 0 || heads <= 0 || max_len < 0) return 0;
  ds::DeviceInfo di;
  if (ds::device_info(&di) != DS_OK) return 0;
  ds::Carve w(nullptr, 0);
  ds::c4::AttnBuffers b{};
  ds::c4::carve_attn(w, &b, batch, heads, max_len, di.num_sms, accumulate != 0);
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

size_t ds_mla_decode4_workspace_size(int batch, int heads, int hidden, int max_len,
                                     int accumulate) {
  if (batch <= 0 || heads <= 0 || hidden <= 0 || max_len < 0) return 0;
  ds::DeviceInfo di;
  if (ds::device_info(&di) != DS_OK) return 0;
  ds::Carve w(nullptr, 0);
  ds::c4::StepBuffers s{};
  ds::c4::carve_step(w, &s, batch, heads, hidden, max_len, di.num_sms, accumulate != 0);
  return ds::align_up(w.used, 256);
}

int ds_mla_decode4_step(const void* x_bf16, const void* w_dec_int8, const float* w_dec_scale,
                        const void* w_out_int8, const float* w_out_scale, const void* cos_bf16,
                        const void* sin_bf16, int table_rows, int hidden, int heads, float eps,
                        float softmax_scale, int accumulate, float mass_decay, void* codes,
                        void* scales_bf16, float* rstd, int32_t* pos, float* mass, int32_t* state,
                        int batch, int slots, int max_len, void* out_bf16, void* workspace,
                        size_t workspace_bytes, void* stream) {
  using namespace ds::c4;
  const Cache c = cache_of(codes, scales_bf16, rstd, pos, mass, state, batch, slots);
  DS_REQUIRE(heads >= 1 && heads <= kMaxHeads, "mla_decode4_step: heads=%d outside [1, %d]", heads,
             kMaxHeads);
  DS_REQUIRE(hidden > 0 && hidden % 16 == 0, "mla_decode4_step: hidden=%d must be a multiple of 16",
             hidden);
  DS_TRY(check_cache(c, "mla_decode4_step"));
  DS_REQUIRE(max_len >= 1 && max_len <= slots, "mla_decode4_step: max_len outside the cache");
  DS_REQUIRE(table_rows > 0, "mla_decode4_step: empty RoPE tables");
  if (batch == 0) return DS_OK;
  DS_REQUIRE(x_bf16 && w_dec_int8 && w_dec_scale && w_out_int8 && w_out_scale && cos_bf16 &&
                 sin_bf16 && out_bf16 && workspace,
             "mla_decode4_step: null pointer");
  DS_REQUIRE(ds::aligned16(x_bf16) && ds::aligned16(w_dec_int8) && ds::aligned16(w_out_int8) &&
                 ds::aligned16(out_bf16) && ds::aligned16(workspace),
             "mla_decode4_step: x, weights, out and workspace must be 16-byte aligned");
  DS_REQUIRE(ds::aligned2(cos_bf16) && ds::aligned2(sin_bf16),
             "mla_decode4_step: misaligned RoPE tables");
  ds::DeviceInfo di;
  DS_TRY(ds::device_info(&di));
  ds::Carve w(workspace, workspace_bytes);
  StepBuffers b{};
  carve_step(w, &b, batch, heads, hidden, max_len, di.num_sms, accumulate != 0);
  if (!w.ok())
    return ds::fail(DS_ERR_WORKSPACE, "mla_decode4_step: workspace needs %zu bytes", w.used);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int cols = (heads + 1) * kQCols;
  DS_TRY(ds::i8::launch_linear(x_bf16, hidden, w_dec_int8, w_dec_scale, b.proj, batch, cols, hidden,
                               b.linear, b.linear_bytes, s));
  DS_CUDA(ds::launch_chained(
      decode4_prepare_kernel, dim3(batch), dim3(288), 0, s, 1, c,
      static_cast<const __nv_bfloat16*>(b.proj), cols, heads,
      static_cast<const __nv_bfloat16*>(cos_bf16), static_cast<const __nv_bfloat16*>(sin_bf16),
      table_rows, eps, b.q));
  DS_LAUNCH_CHECK("decode4_prepare_kernel");
  DS_TRY(launch_attention(c, b.q, heads, max_len, softmax_scale, accumulate, mass_decay, b.olat,
                          b.attn, b.attn_bytes, s));
  return ds::i8::launch_linear(b.olat, heads * kLatent, w_out_int8, w_out_scale, out_bf16, batch,
                               hidden, heads * kLatent, b.linear, b.linear_bytes, s);
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
  // weights and positions of more than 1024 slots are read four at a time
  DS_REQUIRE(ds::aligned16(mass) && ds::aligned16(pos),
             "mla_cache4_evict: the cache's mass and pos must be 16-byte aligned");
  const bool in_place = dst_codes == codes;
  DS_REQUIRE(in_place ? (dst_scales_bf16 == scales_bf16 && dst_rstd == rstd && dst_pos == pos &&
                         dst_mass == mass && dst_state == state && dst_slots == slots)
                      : (dst_scales_bf16 != scales_bf16 && dst_rstd != rstd && dst_pos != pos &&
                         dst_mass != mass && dst_state != state),
             "mla_cache4_evict: the result must be the cache itself or share nothing with it");
  DS_REQUIRE(ds::aligned16(workspace), "mla_cache4_evict: workspace must be 16-byte aligned");
  ds::Carve w(workspace, workspace_bytes);
  int32_t* src_of = w.take<int32_t>(static_cast<size_t>(batch) * budget);
  int32_t* holes = w.take<int32_t>(static_cast<size_t>(batch) * budget);
  if (!w.ok())
    return ds::fail(DS_ERR_WORKSPACE, "mla_cache4_evict: workspace needs %zu bytes", w.used);
  return ds::c4::launch_evict(s, d, budget, recent, in_place, src_of, holes,
                              static_cast<cudaStream_t>(stream));
}

}  // extern "C"
