// The 8-bit key/value cache (gfx950 / CDNA4): its write, its read-back and the
// attention rows over it.
//
// One layer's cache holds e4m3 codes with a power-of-two scale for each block
// of 64 tokens, kv head and tensor; value = code * scale.
//   k       [B, Hkv, cap, D]            a token's row is D bytes
//   v       [B, Hkv, cap / 64, D, 64]   a block's tokens for one column together;
//                                       token 16 t + 4 g + r (t, g, r in 0..3)
//                                       at place 16 g + 4 t + r
//   scales  [B, Hkv, cap / 64] fp32     2^e, e in [E_MIN, E_MAX]
//
// Why powers of two: e4m3 is a floating format, so a finer scale would gain no
// relative precision, while with 2^e every value code * scale is exact in bf16,
// and a block's codes move to a larger scale (when a later token of the block
// needs one) without a second rounding, apart from those that become subnormal.
//
// Why this place order of the values: the attention rows form S^T = K Q^T and
// O^T = V^T P^T with 16x16x32 MFMAs. A lane (column c = lane % 16, group g =
// lane / 16) then holds the probabilities of tokens 16 t + 4 g + r of its row c,
// which is the second product's right operand as it stands, if the left operand
// V^T holds the same tokens in the same lane: 16 consecutive bytes of a column
// of the cache. Neither product needs LDS or a transpose.
#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "capi_common.h"
#include "delta_attn.h"
#include "device_common.h"

namespace da {
namespace {

constexpr int KB = 64;               // tokens per block
constexpr int MAX_CAP = 1 << 30;     // tokens of a sequence (row numbers and limits stay inside 32 bits)
constexpr int E_MIN = -117;          // 2^-9 * 2^-117 (the smallest code's value) is a normal float
constexpr int E_MAX = 120;           // 448 * 2^120 reaches the largest bf16

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Half;   // 16-bit element: bits of infinity, largest value
template <> struct Half<__bf16> {
  static constexpr uint32_t inf = 0x7f80;
  static constexpr float max = 3.3895313892515355e38f;
};
template <> struct Half<_Float16> {
  static constexpr uint32_t inf = 0x7c00;
  static constexpr float max = 65504.f;
};

// Token of place p of a block's values, and the other way round.
__host__ __device__ constexpr int token_of(int p) { return (p % 16 / 4) * 16 + (p / 16) * 4 + p % 4; }

__host__ __device__ constexpr int place_of(int i) { return (i % 16 / 4) * 16 + (i / 16) * 4 + i % 4; }

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The smallest e with amax <= 448 * 2^e, in [E_MIN, E_MAX]: 448 = 1.75 * 2^8.
__device__ __forceinline__ int block_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return min(max(e, E_MIN), E_MAX);
}

// Exponent of a stored scale (any bits give one in range).
__device__ __forceinline__ int scale_exponent(float s) {
  return min(max((int)((__float_as_uint(s) >> 23) & 0xff) - 127, E_MIN), E_MAX);
}

// Four codes times f, rounded to codes again.
__device__ __forceinline__ uint32_t move4(uint32_t w, float f) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a.x * f, a.y * f, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(b.x * f, b.y * f, r, true);
}

// The largest of the lanes' values.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  auto step = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});   // row_shr 1, 2, 4, 8
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});   // across the rows of 16
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return __builtin_amdgcn_readlane(x, 63);
}

// Byte i of the result is 0xff where bit i of `bits` is set.
__device__ __forceinline__ uint32_t byte_mask(uint32_t bits) {
  return ((bits & 1) * 0xffu) | ((bits >> 1 & 1) * 0xff00u) | ((bits >> 2 & 1) * 0xff0000u) |
         ((bits >> 3 & 1) * 0xff000000u);
}

struct Cache {
  uint8_t *k, *v;
  float *ks, *vs;
  int64_t k_b, k_h, v_b, v_h, ks_b, ks_h, vs_b, vs_h;   // batch and head strides
  int cap;
};

// Writes and reads deal groups of G workgroups beside each other to the XCDs in
// turn (workgroup x runs on XCD x % 8), so that the XCDs work beside each other
// too; a last, incomplete round stays in launch order.
template <int G>
__device__ __forceinline__ uint32_t dealt() {
  const uint32_t x = blockIdx.x, first = x / (8 * G) * (8 * G);
  return first + 8 * G <= gridDim.x ? first + x % 8 * G + x / 8 % G : x;
}

// The (sequence, block, head, tensor) of a workgroup or wave.
struct Units {
  FastDiv inner, per_seq;      // of a block or of a head's tensor, of a sequence
  uint32_t n, heads;
};

// Writes: heads innermost (a token's heads lie together in the input). A prompt
// of 131072 tokens takes 143 us in groups of 16, 166 of 8, 168 in launch order,
// 149 with an eighth of the write to each XCD; 32 x 4000 tokens of 8 heads of 128
// 118, 117, 111 and 118 us.
template <int PER_WG>
__device__ __forceinline__ bool write_unit(const Units& u, int& b, int& j, int& h, bool& is_v) {
  const uint32_t i = dealt<16>() * PER_WG + (PER_WG > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0);
  if (i >= u.n) return false;
  b = fdiv(i, u.per_seq);
  const uint32_t rest = i - b * u.per_seq.d;
  j = fdiv(rest, u.inner);
  const uint32_t w = rest - j * u.inner.d;
  is_v = w >= u.heads;
  h = w - (is_v ? u.heads : 0);
  return true;
}

// Reads: a head's blocks innermost (both sides are contiguous along them), each
// of W waves. 131072 rows of 8 heads of 256 take 267 us in groups of 8, 276 of 4,
// 257 of 16, 270 in launch order; 32 x 200 14.7, 15.3, 15.1 and 19.3, 32 x 4000
// of 128 132, 132, 140 and 132.
template <int W>
__device__ __forceinline__ bool read_unit(const Units& u, int& b, int& j, int& h, bool& is_v, int& part) {
  const uint32_t k = dealt<8>() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64), i = k / W;
  part = k % W;
  if (i >= u.n) return false;
  b = fdiv(i, u.per_seq);
  const uint32_t rest = i - b * u.per_seq.d;
  const uint32_t w = fdiv(rest, u.inner);
  j = rest - w * u.inner.d;
  h = w >> 1;
  is_v = w & 1;
  return true;
}

// ---------------------------------------------------------------------------
// write: a workgroup of D / 32 waves per block, head and tensor. A lane holds 8
// columns of 4 tokens of consecutive places, so that keys (8 bytes of a row) and
// values (4 bytes of a column) are both packed inside the lane; only the block's
// largest magnitude crosses lanes, and waves through LDS.
//
// Memory bounds long writes (5.6 TB/s), one block's chain of loads, maximum and
// stores short ones: the more waves share a block, the shorter. One wave for all
// of it (D / 8 tokens a lane) took 8.1 us for a block of 8 heads of 128 and 14.5
// of 256 (3.7 and 4.3 so), 8 tokens a lane 5.7 and 6.2; 32 x 2000 tokens of 8
// heads of 256 take 109 us so, 154 and 127.
constexpr int TPL = 4;                         // tokens per lane

struct WriteArgs {
  Cache c;
  const void *k, *v;
  int64_t kx_b, kx_s, kx_h, vx_b, vx_s, vx_h;
  const int64_t* pos_dev;
  int64_t pos;
  const int* counts;
  int pos_step, counts_step;   // 1: an entry per sequence, 0: one for all
  int S;
  Units units;
};

template <int D> struct Shape {
  static constexpr int W = D / 8 / TPL;        // waves of a block
  static constexpr int PER_WG = W == 1 ? 4 : 1;   // blocks of a writing workgroup
  static constexpr int THREADS = 64 * W * PER_WG;
};

template <typename T, int D>
__global__ __launch_bounds__(Shape<D>::THREADS) void kv8_write_kernel(WriteArgs a) {
  using E = Elt<T>;
  constexpr int DG = D / 8, W = Shape<D>::W;   // lanes across a row, waves of the block
  __shared__ uint32_t s_top[2][W];
  __shared__ int s_e;
  int b, j, h;
  bool is_v;
  if (!write_unit<Shape<D>::PER_WG>(a.units, b, j, h, is_v)) return;
  const int lane = threadIdx.x % 64, wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int64_t pos = a.pos_dev ? a.pos_dev[(int64_t)b * a.pos_step] : a.pos;
  const int count = a.counts ? min(max(a.counts[(int64_t)b * a.counts_step], 0), a.S) : a.S;
  if (pos < 0 || pos > (int64_t)a.c.cap - count) return;
  const int blk = (int)(pos / KB) + j;
  const int base = blk * KB;
  const int r0 = max((int)pos - base, 0), r1 = min((int)pos + count - base, KB);   // its new rows
  if (r1 <= r0) return;
  const bool full = r0 == 0 && r1 == KB;

  // Keys: the waves share out the tokens. Values: the columns, so that runs of 64
  // bytes are stored whole (by tokens a block of 8 heads of 256 takes 6.4 us, not
  // 4.3, 32 x 2000 tokens 158, not 115).
  const int dg = is_v ? wave * TPL + lane % TPL : lane % DG;
  const int p0 = (is_v ? lane / TPL : (wave * 64 + lane) / DG) * TPL;
  const T* src = is_v ? (const T*)a.v + b * a.vx_b + h * a.vx_h : (const T*)a.k + b * a.kx_b + h * a.kx_h;
  const int64_t step = is_v ? a.vx_s : a.kx_s;
  src += (int64_t)(base - (int)pos) * step + dg * 8;
  float* scale = (is_v ? a.c.vs + b * a.c.vs_b + h * a.c.vs_h : a.c.ks + b * a.c.ks_b + h * a.c.ks_h) + blk;
  u32x4 x[TPL];
  uint32_t fresh = 0, older = 0;               // bit i: token i of this lane is new, or holds an earlier token
#pragma unroll
  for (int i = 0; i < TPL; ++i) {
    const int r = token_of(p0 + i);
    // non-temporal where the loads are whole lines, else ordinary (32 x 2000 tokens
    // of 8 heads of 32: 14.7 us, 23.0 non-temporal)
    const T* at = src + (int64_t)min(max(r, r0), r1 - 1) * step;
    x[i] = (is_v ? TPL : DG) * 16 < 128 ? *(const u32x4*)at : ld_nt4(at);
    fresh |= (uint32_t)(r >= r0 && r < r1) << i;
    older |= (uint32_t)(r < r0) << i;
  }
  const float before = r0 > 0 && wave == 0 ? *scale : 0.f;
  uint32_t was[8];                             // a part block's other tokens share its values' words
  uint8_t* vdst = a.c.v + b * a.c.v_b + h * a.c.v_h + (int64_t)blk * KB * D + dg * 8 * KB + p0;
  if (is_v && !full) {
#pragma unroll
    for (int n = 0; n < 8; ++n) was[n] = *(const uint32_t*)(vdst + n * KB);
  }
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < TPL; ++i) {
#pragma unroll
    for (int w = 0; w < 4; ++w)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[i][w] & 0x7fff7fffu));
  }
  // the largest of all the waves'
  auto joined = [&](uint32_t x, int i) __attribute__((always_inline)) {
    x = wave_max(x);
    if constexpr (W > 1) {
      if (lane == 0) s_top[i][wave] = x;
      if (i == 0 && wave == 0 && lane == 0) s_e = scale_exponent(before);
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W; ++w) x = max(x, s_top[i][w]);
    }
    return x;
  };
  uint32_t top = joined(max((uint32_t)m.x, (uint32_t)m.y), 0);
  const bool odd = top >= Half<T>::inf;        // infinities or NaN among them
  if (odd) {
    top = 0;
#pragma unroll
    for (int i = 0; i < TPL; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t lo = x[i][w] & 0x7fffu, hi = x[i][w] >> 16 & 0x7fffu;
        top = max(top, max(lo < Half<T>::inf ? lo : 0u, hi < Half<T>::inf ? hi : 0u));
      }
    top = joined(top, 1);
  }
  int e = block_exponent(E::lo(top));
  bool grown = false;
  float f = 1.f;
  if (r0 > 0) {
    const int eo = W > 1 ? s_e : scale_exponent(before);
    grown = e > eo;
    if (grown) f = pow2(eo) * pow2(-e);        // (0 where that is below the floats: so are the values)
    e = max(e, eo);
  }
  const float inv = pow2(-e);
  if (wave == 0 && lane == 0) *scale = pow2(e);
  // a finite value is at most 448 after the scale; the others become NaN
  auto val = [&](uint32_t w, bool hi) __attribute__((always_inline)) {
    const float y = (hi ? E::hi(w) : E::lo(w)) * inv;
    return odd && !(fabsf(y) < 512.f) ? __builtin_nanf("") : y;
  };
  if (!is_v) {
    uint8_t* dst = a.c.k + b * a.c.k_b + h * a.c.k_h + (int64_t)base * D + dg * 8;
#pragma unroll
    for (int i = 0; i < TPL; ++i) {
      u32x2 w;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(val(x[i][2 * n], false), val(x[i][2 * n], true), 0, false);
        w[n] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(val(x[i][2 * n + 1], false), val(x[i][2 * n + 1], true), c, true);
      }
      u32x2* row = (u32x2*)(dst + token_of(p0 + i) * D);
      if (full || (fresh >> i & 1)) {
        *row = w;
      } else if (grown && (older >> i & 1)) {
        const u32x2 o = *row;
        *row = (u32x2){move4(o[0], f), move4(o[1], f)};
      }
    }
  } else {
    const uint32_t nm = byte_mask(fresh), om = grown ? byte_mask(older) : 0;
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(val(x[0][n / 2], n & 1), val(x[1][n / 2], n & 1), 0, false);
      uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(val(x[2][n / 2], n & 1), val(x[3][n / 2], n & 1), c, true);
      if (!full) w = (w & nm) | (move4(was[n], f) & om) | (was[n] & ~(nm | om));
      *(uint32_t*)(vdst + n * KB) = w;
    }
  }
}

// A few tokens per sequence (a decode step's one, drafted ones): one wave per
// sequence, block, head and tensor, a lane 8 columns of NP tokens. The block's
// other tokens are touched only where the new ones need a larger scale than
// theirs, and the tokens' loads wait for nothing. 4 tokens of 32 sequences of 8
// heads of 256 take 5.1 us (by the kernel above 8.8), 8 of 128 4.8 (5.9), 16 of 64
// 3.8 (4.5). With four passes 8 tokens of 256 take 7.1 (8.9), but those of a single
// sequence 6.2 (4.3): two at most.
// ONE: a single token, which every lane group then holds (2.8 us, 3.0 without).
template <typename T, int D, int NP, bool ONE>
__global__ __launch_bounds__(256) void kv8_append_kernel(WriteArgs a) {
  using E = Elt<T>;
  constexpr int DG = D / 8, AT_ONCE = 64 / DG;  // lanes across a token, tokens side by side
  int b, j, h;
  bool is_v;
  if (!write_unit<4>(a.units, b, j, h, is_v)) return;
  const int lane = threadIdx.x % 64, dg = lane % DG, t0 = lane / DG;
  const T* src = is_v ? (const T*)a.v + b * a.vx_b + h * a.vx_h : (const T*)a.k + b * a.kx_b + h * a.kx_h;
  const int64_t step = is_v ? a.vx_s : a.kx_s;
  u32x4 x[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int t = i * AT_ONCE + t0;
    x[i] = *(const u32x4*)(ONE ? src + dg * 8 : src + min(t, a.S - 1) * step + dg * 8);
  }
  const int64_t pos = a.pos_dev ? a.pos_dev[(int64_t)b * a.pos_step] : a.pos;
  const int S = ONE ? 1 : a.S, count = a.counts ? min(max(a.counts[(int64_t)b * a.counts_step], 0), S) : S;
  if (pos < 0 || pos > (int64_t)a.c.cap - count) return;
  if (ONE) j = 0;                              // (its only block)
  const int blk = (int)(pos / KB) + j, r0 = j == 0 ? (int)(pos % KB) : 0;   // the first new row's
  const int lo = j == 0 ? 0 : blk * KB - (int)pos, hi = min(count, (blk + 1) * KB - (int)pos);
  if (ONE ? count < 1 : hi <= lo) return;      // tokens lo .. hi - 1 are this block's
  auto mine = [&](int i) __attribute__((always_inline)) {
    const int t = i * AT_ONCE + t0;
    return ONE || (t >= lo && t < hi);         // (one token: every lane group holds it)
  };
  float* scale = (is_v ? a.c.vs + b * a.c.vs_b + h * a.c.vs_h : a.c.ks + b * a.c.ks_b + h * a.c.ks_h) + blk;
  const float before = *scale;

  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < NP; ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, mine(i) ? x[i][w] & 0x7fff7fffu : 0u));
  uint32_t top = wave_max(max((uint32_t)m.x, (uint32_t)m.y));
  const bool odd = top >= Half<T>::inf;        // infinities or NaN among them
  if (odd) {
    top = 0;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t y = mine(i) ? x[i][w] : 0u, even = y & 0x7fffu, next = y >> 16 & 0x7fffu;
        top = max(top, max(even < Half<T>::inf ? even : 0u, next < Half<T>::inf ? next : 0u));
      }
    top = wave_max(top);
  }
  int e = block_exponent(E::lo(top));
  uint8_t* block = is_v ? a.c.v + b * a.c.v_b + h * a.c.v_h + (int64_t)blk * KB * D
                        : a.c.k + b * a.c.k_b + h * a.c.k_h + (int64_t)blk * KB * D;
  if (r0 > 0) {
    const int eo = scale_exponent(before);
    if (e > eo) {                              // the earlier tokens' codes move to the new scale
      const float f = pow2(eo) * pow2(-e);
      if (!is_v) {
        for (int i = lane; i < r0 * D / 16; i += 64) {
          u32x4* c = (u32x4*)block + i;
          const u32x4 w = *c;
          *c = (u32x4){move4(w[0], f), move4(w[1], f), move4(w[2], f), move4(w[3], f)};
        }
      } else {
        for (int i = lane; i < KB * D / 16; i += 64) {
          u32x4* c = (u32x4*)block + i;
          u32x4 w = *c;
#pragma unroll
          for (int t = 0; t < 4; ++t) {        // tokens 16 t + 4 (i % 4) + 0 .. 3
            const int n = min(max(r0 - 16 * t - 4 * (i % 4), 0), 4);
            const uint32_t om = n == 4 ? 0xffffffffu : (1u << 8 * n) - 1;
            w[t] = (move4(w[t], f) & om) | (w[t] & ~om);
          }
          *c = w;
        }
        __threadfence_block();                 // the new tokens' bytes below lie in these words
      }
    }
    e = max(e, eo);
  }
  const float inv = pow2(-e);
  if (lane == 0) *scale = pow2(e);
  auto val = [&](uint32_t w, bool hi) __attribute__((always_inline)) {
    const float y = (hi ? E::hi(w) : E::lo(w)) * inv;
    return odd && !(fabsf(y) < 512.f) ? __builtin_nanf("") : y;
  };
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    if (ONE ? t0 > 0 : !mine(i)) continue;
    const int r = ONE ? r0 : r0 + i * AT_ONCE + t0 - lo;
    u32x2 c;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int lo2 = __builtin_amdgcn_cvt_pk_fp8_f32(val(x[i][2 * n], false), val(x[i][2 * n], true), 0, false);
      c[n] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(val(x[i][2 * n + 1], false), val(x[i][2 * n + 1], true), lo2, true);
    }
    if (!is_v) {
      *(u32x2*)(block + r * D + dg * 8) = c;
    } else {
      uint8_t* dst = block + dg * 8 * KB + place_of(r);
#pragma unroll
      for (int n = 0; n < 8; ++n) dst[n * KB] = (uint8_t)(c[n / 4] >> 8 * (n % 4));
    }
  }
}

// ---------------------------------------------------------------------------
// read: the write's lanes the other way round, without a maximum to share: D / 32
// waves a block, each by itself, with non-temporal stores (131072 rows: 144 us,
// 174 with ordinary ones, by one wave a block). A wave of the values covers 64
// columns of half the tokens, so that its stores are whole lines of 128 bytes:
// 131072 rows of 8 heads of 128 take 133 us so, 149 with half lines, 143 with
// twice as long ones; one wave a block took 144, and 500 rows 5.7 us (3.3 so).
struct ReadArgs {
  Cache c;
  void *k, *v;
  int64_t ko_b, ko_h, ko_s, vo_b, vo_h, vo_s;
  const int* n_keys;
  int n_step;
  int start, n;
  Units units;
};

template <typename T, int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(ReadArgs a) {
  using E = Elt<T>;
  constexpr int DG = D / 8, W = Shape<D>::W;
  constexpr int AC = DG < 8 ? DG : 8, CG = DG / AC;   // lanes across the values' columns, waves across them
  int b, j, h, part;
  bool is_v;
  if (!read_unit<W>(a.units, b, j, h, is_v, part)) return;
  const int lane = threadIdx.x % 64;
  const int blk = a.start / KB + j;
  const int live = a.n_keys ? a.n_keys[(int64_t)b * a.n_step] : a.c.cap;
  const int dg = is_v ? part % CG * AC + lane % AC : lane % DG;
  const int p0 = (is_v ? part / CG * (64 / AC) + lane / AC : (part * 64 + lane) / DG) * TPL;
  const float s = (is_v ? a.c.vs + b * a.c.vs_b + h * a.c.vs_h : a.c.ks + b * a.c.ks_b + h * a.c.ks_h)[blk];
  const bool sat = 448.f * s > Half<T>::max;   // (also where the product is infinite)
  auto fix = [&](float y) __attribute__((always_inline)) {
    return sat && y == y ? fminf(fmaxf(y, -Half<T>::max), Half<T>::max) : y;
  };
  T* dst = is_v ? (T*)a.v + b * a.vo_b + h * a.vo_h : (T*)a.k + b * a.ko_b + h * a.ko_h;
  const int64_t step = is_v ? a.vo_s : a.ko_s;
  auto put = [&](int r, u32x4 w) __attribute__((always_inline)) {
    const int row = blk * KB + r;
    if (row < a.start || row >= a.start + a.n) return;
    if (row >= live) w = (u32x4){0, 0, 0, 0};
    st_nt4(dst + (int64_t)(row - a.start) * step + dg * 8, w);
  };
  if (!is_v) {
    const uint8_t* src = a.c.k + b * a.c.k_b + h * a.c.k_h + (int64_t)blk * KB * D + dg * 8;
    u32x2 x[TPL];
#pragma unroll
    for (int i = 0; i < TPL; ++i) x[i] = *(const u32x2*)(src + token_of(p0 + i) * D);
#pragma unroll
    for (int i = 0; i < TPL; ++i) {
      u32x4 o;
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(x[i][n], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(x[i][n], true);
        o[2 * n] = E::pack2(fix(lo.x * s), fix(lo.y * s));
        o[2 * n + 1] = E::pack2(fix(hi.x * s), fix(hi.y * s));
      }
      put(token_of(p0 + i), o);
    }
  } else {
    const uint8_t* src = a.c.v + b * a.c.v_b + h * a.c.v_h + (int64_t)blk * KB * D + dg * 8 * KB + p0;
    uint32_t x[8];
#pragma unroll
    for (int n = 0; n < 8; ++n) x[n] = *(const uint32_t*)(src + n * KB);
    float y[4][8];
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(x[n], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(x[n], true);
      y[0][n] = fix(lo.x * s);
      y[1][n] = fix(lo.y * s);
      y[2][n] = fix(hi.x * s);
      y[3][n] = fix(hi.y * s);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      put(token_of(p0 + r), (u32x4){E::pack2(y[r][0], y[r][1]), E::pack2(y[r][2], y[r][3]),
                                    E::pack2(y[r][4], y[r][5]), E::pack2(y[r][6], y[r][7])});
  }
}

// ---------------------------------------------------------------------------
// attention rows at the end of each sequence's cache
struct RowsArgs {
  Cache c;
  const void* q;
  int64_t q_b, q_h, q_s;
  void* o;
  int64_t o_b, o_h, o_s;
  const void* add;
  int64_t add_b, add_h, add_s;
  const int* n_dev;         // key counts on the device (entry b * n_step), or NULL: `n`
  int n_step, n;
  int B, Hkv, G, s;         // G query heads per kv head, s rows at the end of each sequence
  int n_rt, rows;           // row tiles of `rows` rows (flattened row i * G + head) per sequence and kv head
  int window, sink;
  float scale2;             // 2 |sm_scale| log2(e), above zero: references and differences are halves
  uint32_t flip;            // the sign bits of Q where sm_scale is negative
  int alike;                // every sequence splits alike: one count for all, or
  int whole;                // above zero: no list is split, and none has more blocks
  int most;                 // splits at most, where the sequences split alike
  int slots;                // workgroups that are resident together
  FastDiv round;            // blocks that they take at most: slots * CHUNK
  FastDiv units, tiles, heads;   // Hkv * n_rt, n_rt, G
  float* part;              // per item: rows x D sums, then rows references, rows weights
  int64_t pitch;            // floats per item
};

// Probabilities are held relative to a row reference (half a score q k, not yet
// times sm_scale: half the difference of two finite scores is finite) that may lag
// its maximum by up to LAG (log2), times 2^BIAS: at most 2^14, inside fp16, and
// fp16 ends 2^-32 below the reference.
constexpr float NO_KEYS = -FLT_MAX / 2;        // the reference of a row without keys yet: half the lowest score
constexpr float LAG = 6.f, BIAS = 8.f;

// The blocks that a sequence's rows see: those of the sinks, then [lo, hi).
struct Blocks {
  int first, lo, n;         // sink blocks, first block after them, all together
  __device__ __forceinline__ int at(int i) const { return i < first ? i : lo + i - first; }
};

__device__ __forceinline__ int keys_of(const RowsArgs& a, int b) {
  const int n = a.n_dev ? a.n_dev[(int64_t)b * a.n_step] : a.n;
  return min(max(n, 0), a.c.cap);
}

__device__ __forceinline__ Blocks blocks_of(const RowsArgs& a, int n) {
  Blocks l;
  l.lo = a.window > 0 ? max(n - a.s - a.window + 1, 0) / KB : 0;
  l.first = a.window > 0 ? min((a.sink + KB - 1) / KB, l.lo) : 0;
  l.n = l.first + (n + KB - 1) / KB - l.lo;
  return l;
}

constexpr int WAVES = 4;
// Waves per SIMD of the rows kernel: what the registers of a block's codes, the
// sums and MT tiles of probabilities leave room for.
__host__ __device__ constexpr int rows_waves(int D, int mt) {
  return D * mt <= 64 ? (mt == 1 ? 4 : 3) : D * mt <= 128 ? 2 : 1;
}
constexpr int CHUNK = 64;                    // blocks of an item at most, where there are many

// Lists stay whole, an item each, where no list's own chain of blocks (a
// workgroup takes D * 3.7 ns a block beside 5 us of start and end) is longer than
// a split's second launch and join, or where there are so many lists that their
// blocks keep memory busy together. One row each, 12 blocks of 128 columns in 8
// lists 7.4 us whole and 7.6 split, 16 9.4 and 8.0; 32 blocks, all full / of 1 to
// 32, in 128 lists 21 / 19 and 18 / 15, in 256 25 / 21 and 29 / 22, in 512 43 / 31
// and 46 / 35; six rows each in 384 lists of 24 blocks of 64 columns 17 / 13 and 28
// / 31. Four row tiles take twice as long a block: 8 blocks 17 and 17, 12 20 and 17.
__host__ __device__ constexpr bool stays_whole(int64_t blocks, int64_t lists, int D, int mt) {
  const int64_t few = mt < 4 ? 1280 : 1024;
  return blocks <= WAVES || (blocks <= CHUNK && blocks * D <= (few > 16 * lists ? few : 16 * lists));
}

// Splits: every item takes `chunk` blocks of one (sequence, kv head, row tile).
// There are as many items as workgroups are resident together, or some rounds of
// them where an item would exceed CHUNK blocks (eight sequences of 98K-131K keys
// take 283 us at 64 blocks, 304 at 24, 320 at 16, 371 at 8); sequences of
// different lengths give items of one size. An item's place is found by each
// wave for itself: the sequences' item counts, summed over 64 lanes.
// `blocks`: all sequences', kv heads' and row tiles' together (below 2^31).
__host__ __device__ __forceinline__ int item_budget(int blocks, int slots, const FastDiv& round) {
  return slots * (int)(fdiv(blocks + round.d - 1, round));
}

// Within a sequence the items lie by kv head, split, row tile: the tiles of one
// split, which read the same codes, are next to each other.
struct Place {
  int b, head, tile, split, n_split, chunk;
  int slot;                 // the item, or a tile's first one (the others n_rt apart)
};

// Inclusive sum over the lanes up to this one.
__device__ __forceinline__ int scan64(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);    // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);   // row 0's total to row 1, 2's to 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);   // rows 0 and 1's to rows 2 and 3
  return x;
}

// locate() among sequences of different lengths, 64 at a time with one to a
// lane; the counts of the first KEPT rounds stay in registers.
template <bool ITEM, int KEPT>
__device__ __forceinline__ bool among(const RowsArgs& a, int i, Place& p, int& rest, int& first) {
  const int lane = threadIdx.x % 64, units = a.units.d, nu = KEPT == 1 ? 1 : (a.B + 63) / 64;
  auto load = [&](int u) __attribute__((always_inline)) {
    const int b = u * 64 + lane;
    return b < a.B ? blocks_of(a, keys_of(a, b)).n : -1;
  };
  int kept[KEPT];
#pragma unroll
  for (int u = 0; u < KEPT; ++u) kept[u] = u < nu ? load(u) : -1;
  auto blocks = [&](int u) __attribute__((always_inline)) {   // -1 past the last sequence
    if constexpr (KEPT == 1) return kept[0];
    else return u == 0 ? kept[0] : u == 1 ? kept[1] : u == 2 ? kept[2] : u == 3 ? kept[3] : load(u);
  };
  auto items = [&](int u) __attribute__((always_inline)) {
    const int n = blocks(u);
    return n < 0 ? 0 : max((n + p.chunk - 1) / p.chunk, 1);
  };
  int total = 0;
  for (int u = 0; u < nu; ++u) total += __builtin_amdgcn_readlane(scan64(max(blocks(u), 0)), 63);
  const int budget = item_budget(total * units, a.slots, a.round);
  p.chunk = max((total * units + budget - 1) / max(budget, 1), WAVES);
  // the sequences' last items are short: longer ones, until all fit the budget
  for (int tries = 0; tries < 4 && a.B * units < budget; ++tries) {
    int all = 0;
    for (int u = 0; u < nu; ++u) all += __builtin_amdgcn_readlane(scan64(items(u)), 63) * units;
    if (all <= budget) break;
    p.chunk += max((p.chunk * (all - budget)) / budget, 1);
  }
  first = 0;
  for (int u = 0, have = i; u < nu; ++u) {
    const int mine = items(u), upto = scan64(mine);
    const uint64_t past = __ballot(mine > 0 && (ITEM ? upto : lane + 1) * units > have);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      p.n_split = __builtin_amdgcn_readlane(mine, l);
      const int before = (__builtin_amdgcn_readlane(upto, l) - p.n_split) * units;
      p.b = u * 64 + l;
      first += before;
      rest = have - (ITEM ? before : l * units);
      return true;
    }
    const int here = __builtin_amdgcn_readlane(upto, 63) * units;
    first += here;
    have -= ITEM ? here : 64 * units;
  }
  return false;
}

// The splits of every sequence where they split alike.
__device__ __forceinline__ void split_alike(const RowsArgs& a, Place& p) {
  if (a.whole > 0) {
    p.chunk = a.whole;
    p.n_split = 1;
  } else {
    const int n = blocks_of(a, __builtin_amdgcn_readfirstlane(keys_of(a, 0))).n, pairs = a.B * (int)a.units.d;
    const int splits = max(item_budget(n * pairs, a.slots, a.round) / pairs, 1);
    p.chunk = max((n + splits - 1) / splits, WAVES);
    p.n_split = max((n + p.chunk - 1) / p.chunk, 1);
  }
}

// Tile, head and split of the `rest`th item (ITEM false: pair of head and tile)
// of a sequence whose items have slots from `first` on, `room` a pair.
template <bool ITEM>
__device__ __forceinline__ void place(const RowsArgs& a, Place& p, int rest, int first, int room) {
  const int group = fdiv(rest, a.tiles);            // (kv head, split), or the kv head
  p.tile = rest - group * a.n_rt;
  p.head = ITEM ? group / p.n_split : group;
  p.split = ITEM ? group - p.head * p.n_split : 0;
  p.slot = first + (p.head * room + p.split) * a.n_rt + p.tile;
}

// Where the sequences split alike, a pair's slots depend on no count.
__device__ __forceinline__ bool place_alike(const RowsArgs& a, int i, Place& p) {
  const int units = a.units.d;
  p.b = a.B == 1 ? 0 : fdiv(i, a.units);
  if (p.b >= a.B || i - p.b * units >= units) return false;
  place<false>(a, p, i - p.b * units, p.b * units * a.most, a.most);
  return true;
}

// The place of item `i`, or (ITEM false, sequences of different lengths) of
// (sequence, kv head, row tile) `i`; false past the last.
template <bool ITEM>
__device__ __forceinline__ bool locate(const RowsArgs& a, int i, Place& p) {
  int rest, first;          // `i` and the first item, within the sequence
  if (ITEM && a.alike) {
    split_alike(a, p);
    const int units = a.units.d, per_seq = units * p.n_split;
    p.b = a.B == 1 ? 0 : i / per_seq;
    rest = i - p.b * per_seq;
    if (p.b >= a.B || rest >= per_seq) return false;
    place<ITEM>(a, p, rest, p.b * units * a.most, a.most);
    return true;
  }
  // (a separate copy for up to 64 sequences, one to a lane)
  if (!(a.B <= 64 ? among<ITEM, 1>(a, i, p, rest, first) : among<ITEM, 4>(a, i, p, rest, first))) return false;
  place<ITEM>(a, p, rest, first, p.n_split);
  return true;
}

// What a row's sums are divided by: a row without keys (standing before the
// sequence's start) is zero; one whose every score is -inf has no weight either,
// and no softmax: NaN.
__device__ __forceinline__ float inverse(float weight, int row) { return row < 0 ? 0.f : 1.f / weight; }

__device__ __forceinline__ float group_max(float x) {   // over the four lanes of one row
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// 16x16x32 products of one type, and eight codes as its left operand. SCALED:
// the conversion applies the block's scale, exactly (bf16 has float's range:
// scores then overflow only where they would anyway; half of it where a code may
// reach 256 * 2^120, past both types' largest); fp16 takes the codes alone.
template <typename T> struct Dot;
template <> struct Dot<__bf16> {
  static constexpr bool SCALED = true;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u32x4 codes(uint32_t lo, uint32_t hi, float scale) {
    return (u32x4){__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
  }
};
template <> struct Dot<_Float16> {
  static constexpr bool SCALED = false;
  static __device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ u32x4 codes(uint32_t lo, uint32_t hi, float = 1.f) {
    return (u32x4){__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true))};
  }
};

// Stores a finished row's four columns: rnd(o), or rnd(rnd(o) + add).
template <typename T>
__device__ __forceinline__ void store4(const RowsArgs& a, int b, int h, int i, int d, f32x4 o) {
  using E = Elt<T>;
  u32x2 w = {E::pack2(o[0], o[1]), E::pack2(o[2], o[3])};
  if (a.add) {
    const u32x2 x = *(const u32x2*)((const T*)a.add + b * a.add_b + h * a.add_h + i * a.add_s + d);
    w = (u32x2){E::pack2(E::lo(w[0]) + E::lo(x[0]), E::hi(w[0]) + E::hi(x[0])),
                E::pack2(E::lo(w[1]) + E::lo(x[1]), E::hi(w[1]) + E::hi(x[1]))};
  }
  *(u32x2*)((T*)a.o + b * a.o_b + h * a.o_h + i * a.o_s + d) = w;
}

// One item: its waves take its blocks in turn and are joined through LDS. A block
// is one pass of S^T = K Q^T, the probabilities with a running reference, O^T =
// V^T P^T; a block's codes go straight to registers, the next block's keys loaded
// when the first product has read this one's, its values after the second.
//
// What bounds it: memory, where there is enough of it (a dense row of 32 / 8 heads
// over 131072 keys 44.2 us, 6.1 TB/s with the first loads; eight sequences of that
// length 6.65 TB/s); else a launch (1.9 us) and the loads that wait for each other
// (arguments, count, codes: 5.2 us for a single block). Registers, not MFMA or
// conversions, limit the waves (203 at head_dim 128 and one row tile).
//
// MT: 16-row tiles per wave. The P V product is formed in fp16 whatever Q's
// type: the codes are exact in it, and its 11 bits keep the probabilities'
// rounding below that of a bf16 result (bf16 probabilities would add as much
// again to the result's own rounding error). Each tile's weights are summed by an
// MFMA with ones, from the same rounded probabilities.
template <typename T, int D, int MT>
__global__ __launch_bounds__(64 * WAVES, rows_waves(D, MT)) void kv8_rows_kernel(RowsArgs a) {
  constexpr int KS = D / 32;                 // steps of the Q K product
  constexpr int KW = D >= 64 ? D / 64 : 1;   // loads of a key's row per lane
  constexpr int DT = D / 16;
  using P = Dot<_Float16>;
  Place p;
  // The row tiles of one split run on one XCD (workgroup x runs on XCD x % 8):
  // its L2 holds the codes that they share.
  int item = blockIdx.x;
  if (a.n_rt > 1) {
    const int q = item / 8, k = fdiv(q, a.tiles);
    item = (k * 8 + item % 8) * a.n_rt + q - k * a.n_rt;
  }
  if (!locate<true>(a, item, p)) return;
  // (all of it is the wave's: scalar registers)
  p.b = __builtin_amdgcn_readfirstlane(p.b);
  p.head = __builtin_amdgcn_readfirstlane(p.head);
  p.tile = __builtin_amdgcn_readfirstlane(p.tile);
  p.split = __builtin_amdgcn_readfirstlane(p.split);
  p.chunk = __builtin_amdgcn_readfirstlane(p.chunk);
  p.n_split = __builtin_amdgcn_readfirstlane(p.n_split);
  p.slot = __builtin_amdgcn_readfirstlane(p.slot);
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int c = lane % 16, g = lane / 16;
  const int b = p.b, hk = p.head, m0 = p.tile * a.rows;
  const int n = __builtin_amdgcn_readfirstlane(keys_of(a, b));
  const Blocks list = blocks_of(a, n);
  const int n_rows = min(a.rows, a.s * a.G - m0);

  // Q as the product's right operand, its columns in the order of the keys'
  // loads: step 2 w + u holds columns 64 w + 16 g + 8 u .. + 7
  u32x4 qf[MT][KS];
  int lim[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    // (columns behind the last row repeat it; nothing is made of them)
    const int m = m0 + min(mt * 16 + c, n_rows - 1);
    const int i = fdiv(m, a.heads);
    lim[mt] = n - a.s + i;
    const T* src = (const T*)a.q + b * a.q_b + (int64_t)(hk * a.G + m - i * a.G) * a.q_h + i * a.q_s;
#pragma unroll
    for (int k = 0; k < KS; ++k)
      qf[mt][k] = *(const u32x4*)(src + (D >= 64 ? k / 2 * 64 + g * 16 + k % 2 * 8 : g * 8)) ^ a.flip;
  }
  const uint8_t* kc = a.c.k + b * a.c.k_b + hk * a.c.k_h;
  const uint8_t* vc = a.c.v + b * a.c.v_b + hk * a.c.v_h;
  const float* ksc = a.c.ks + b * a.c.ks_b + hk * a.c.ks_h;
  const float* vsc = a.c.vs + b * a.c.vs_b + hk * a.c.vs_h;

  f32x4 acc[MT][DT], sum[MT];
  float ref[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    ref[mt] = NO_KEYS;
    sum[mt] = (f32x4){0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[mt][t] = (f32x4){0, 0, 0, 0};
  }
  const uint32_t one = 0x3c003c00u;
  const u32x4 ones = {one, one, one, one};
  // rows m0 / G .. of the tile: the first's and the last's limits
  const int lim_lo = n - a.s + (int)fdiv(m0, a.heads), lim_hi = n - a.s + (int)fdiv(m0 + n_rows - 1, a.heads);

  // this wave's blocks of the list: one in WAVES, up to the tile's last key
  int end = min((p.split + 1) * p.chunk, list.n);
  end = min(end, lim_hi < 0 ? 0 : list.first + lim_hi / KB + 1 - list.lo);
  int x = p.split * p.chunk + wave;
  u32x4 kf[4][KW], vf[DT];
  float sk, sv;
  // A block's loads; none are made (zeros) where there is no block. Non-temporal:
  // a decode step's other layers and weights pass between two reads of a cache.
  // Caches of 2 GB together, 4 to 268 MB a call: 9.3 -> 8.5 to 54.2 -> 48.0 us; a
  // single cache of 34 to 268 MB read again and again: up to 5 % slower. (The
  // most rows a wave holds may be one of several row tiles, which share codes.)
  constexpr int STREAM = MT == (D == 256 ? 2 : 4) ? 0 : 2;
  const uint32_t k_off = c * D + g * (D >= 64 ? 16 : 8), v_off = c * KB + g * 16;
  auto load_k = [&](int blk, bool any) __attribute__((always_inline)) {
    const auto r = make_rsrc(kc + (int64_t)blk * (KB * D), any ? KB * D : 0);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        if constexpr (D >= 64) {
          kf[t][w] = __builtin_amdgcn_raw_buffer_load_b128(r, k_off, t * 16 * D + w * 64, STREAM);
        } else {
          const u32x2 y = __builtin_amdgcn_raw_buffer_load_b64(r, k_off, t * 16 * D, STREAM);
          kf[t][w] = (u32x4){y[0], y[1], 0, 0};
        }
      }
    sk = ksc[blk];
  };
  auto load_v = [&](int blk, bool any) __attribute__((always_inline)) {
    const auto r = make_rsrc(vc + (int64_t)blk * (KB * D), any ? KB * D : 0);
#pragma unroll
    for (int t = 0; t < DT; ++t) vf[t] = __builtin_amdgcn_raw_buffer_load_b128(r, v_off, t * 16 * KB, STREAM);
    sv = vsc[blk];
  };
  int blk = x < end ? list.at(x) : 0;
  load_k(blk, x < end);
  __builtin_amdgcn_sched_barrier(0);          // (the keys are waited for first)
  load_v(blk, x < end);
  while (x < end) {
    const int key0 = blk * KB;
    x += WAVES;
    const bool more = x < end;
    blk = more ? list.at(x) : 0;
    // every row sees every key of the block?
    const bool whole = key0 + KB - 1 <= lim_lo &&
        (a.window == 0 || key0 > lim_hi - a.window || key0 + KB <= a.sink);
    // bit 4 t + r: the row sees token 16 t + 4 g + r of the block
    auto seen = [&](int mt) __attribute__((always_inline)) {
      const int hi = lim[mt] - key0 - g * 4, lo = a.window > 0 ? hi - a.window : -1, sink = a.sink - key0 - g * 4;
      uint32_t bits = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int at = e / 4 * 16 + e % 4;
        bits |= (uint32_t)(at <= hi && (at > lo || at < sink)) << e;
      }
      return bits;
    };
    // s holds the scores, or (the largest scale) half of them: s * half is half a score
    const bool far = Dot<T>::SCALED && sk > pow2(E_MAX - 1);
    const float by = far ? pow2(E_MAX - 1) : sk, half = far ? 1.f : 0.5f;
    f32x4 s[MT][4];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const u32x4 af = Dot<T>::codes(kf[t][k / 2][k % 2 * 2], kf[t][k / 2][k % 2 * 2 + 1], by);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          s[mt][t] = Dot<T>::mfma(af, qf[mt][k], k == 0 ? (f32x4){0, 0, 0, 0} : s[mt][t]);
      }
      __builtin_amdgcn_sched_barrier(0);      // (the conversions stay beside their products: fewer registers)
    }
    const float unit = sk;
    load_k(blk, more);                        // the keys' registers are free from here on
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (!Dot<T>::SCALED) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[mt][e / 4][e % 4] *= unit;
    }
    if (!whole) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const uint32_t bits = seen(mt);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[mt][e / 4][e % 4] = bits >> e & 1 ? s[mt][e / 4][e % 4] : -INFINITY;
      }
    }
    u32x4 pf[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float top = s[mt][0][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, s[mt][e / 4][e % 4]);
      top = group_max(top);
      if (__any(fmaf(top, half, -ref[mt]) * a.scale2 > LAG)) {
        const float to = fmaxf(ref[mt], top * half);
        const float alpha = fast_exp2((ref[mt] - to) * a.scale2);
        ref[mt] = to;
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[mt][r] *= alpha;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[mt][t][r] *= alpha;
      }
      auto weight = [&](float y) __attribute__((always_inline)) {
        return fast_exp2(fmaf(fmaf(y, half, -ref[mt]), a.scale2, BIAS));
      };
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int t = 2 * u + w / 2, r = w % 2 * 2;
          pf[mt][u][w] = Elt<_Float16>::pack2(weight(s[mt][t][r]), weight(s[mt][t][r + 1]));
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (!whole) {
      // A NaN code of a token that a row does not see (behind the last key,
      // outside the row's window) must not reach it through 0 * NaN: the code
      // is taken as zero, and the rows that do see one get theirs from a
      // product of the codes' and the rows' marks.
      auto nans = [&](uint32_t w) __attribute__((always_inline)) {      // bit 0 of its NaN bytes
        return ((w & 0x7f7f7f7fu) + 0x01010101u) >> 7 & 0x01010101u;
      };
      uint32_t bad = 0;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int w = 0; w < 4; ++w) bad |= nans(vf[t][w]);
      if (__any(bad != 0)) {
        u32x4 mark[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const uint32_t bits = seen(mt);
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            const uint32_t two = bits >> 2 * w & 3;
            mark[mt][w / 4][w % 4] = (two & 1) * 0x3c00u | (two >> 1) * 0x3c000000u;
          }
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          uint32_t hit[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            hit[w] = nans(vf[t][w]);
            vf[t][w] &= ~(hit[w] * 0xffu);
            hit[w] *= 0x38u;                                            // the code of 1
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            f32x4 hits = P::mfma(P::codes(hit[0], hit[1]), mark[mt][0], (f32x4){0, 0, 0, 0});
            hits = P::mfma(P::codes(hit[2], hit[3]), mark[mt][1], hits);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[mt][t][r] = hits[r] > 0.f ? __builtin_nanf("") : acc[mt][t][r];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int u = 0; u < 2; ++u) sum[mt] = P::mfma(ones, pf[mt][u], sum[mt]);
#pragma unroll
    for (int t = 0; t < DT; ++t) {
      const u32x4 v0 = P::codes(vf[t][0], vf[t][1]), v1 = P::codes(vf[t][2], vf[t][3]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        f32x4 y = P::mfma(v0, pf[mt][0], (f32x4){0, 0, 0, 0});
        y = P::mfma(v1, pf[mt][1], y);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[mt][t][r] = fmaf(y[r], sv, acc[mt][t][r]);
      }
      if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    load_v(blk, more);
    __builtin_amdgcn_sched_barrier(0);
  }

  // join the waves, one 16-row tile after the other
  constexpr int LD = D + 4;                    // row pitch: the 16 rows of a column spread over the banks
  __shared__ float s_o[WAVES][16][LD];
  __shared__ float s_m[WAVES][16], s_l[WAVES][16];
  float* part = a.part + (int64_t)p.slot * a.pitch;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (mt > 0) __syncthreads();
#pragma unroll
    for (int t = 0; t < DT; ++t) *(f32x4*)&s_o[wave][c][t * 16 + g * 4] = acc[mt][t];
    if (g == 0) {
      s_m[wave][c] = ref[mt];
      s_l[wave][c] = sum[mt][0];
    }
    __syncthreads();
    for (int task = threadIdx.x; task < 16 * (D / 4); task += 64 * WAVES) {
      const int r = task / (D / 4), d = task % (D / 4) * 4, row = mt * 16 + r;
      if (row >= n_rows) break;
      float M = s_m[0][r];
#pragma unroll
      for (int w = 1; w < WAVES; ++w) M = fmaxf(M, s_m[w][r]);
      float L = 0.f;
      f32x4 o = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        const float k = fast_exp2((s_m[w][r] - M) * a.scale2);
        const f32x4 y = *(const f32x4*)&s_o[w][r][d];
        L = fmaf(s_l[w][r], k, L);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(y[e], k, o[e]);
      }
      if (p.n_split == 1) {
        const int m = m0 + row, i = fdiv(m, a.heads);
        const float inv = inverse(L, n - a.s + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] *= inv;
        store4<T>(a, b, hk * a.G + m - i * a.G, i, d, o);
      } else {
        *(f32x4*)(part + row * D + d) = o;
        if (d == 0) {
          part[a.rows * D + row] = M;
          part[a.rows * (D + 1) + row] = L;
        }
      }
    }
  }
}

// Joins the items of one (sequence, kv head, row tile): a workgroup per row, some
// items side by side and four loads of each in flight. Launch and dependent loads
// (arguments, count, partials; where the sequences split alike the first partials
// do not wait for the count): 3.5 us for 32 rows of 9 items, 4.9 for 32 of 64.
template <typename T, int D, int THREADS>
__global__ __launch_bounds__(THREADS) void kv8_join_kernel(RowsArgs a) {
  constexpr int CT = D / 4, SG = THREADS / CT; // threads across a row, items taken side by side
  __shared__ float s_w[SG][2];
  __shared__ f32x4 s_o[SG][CT];
  const int row = blockIdx.y;
  Place p;
  if (a.alike) {
    if (!place_alike(a, blockIdx.x, p)) return;
  } else {
    if (!locate<false>(a, blockIdx.x, p)) return;
  }
  const int room = a.alike ? a.most : p.n_split;    // slots of this pair
  const int hk = p.head, m = p.tile * a.rows + row;
  if (m >= a.s * a.G) return;
  const int qi = fdiv(m, a.heads);
  const int t = threadIdx.x % CT, sg = threadIdx.x / CT;
  const float* part = a.part + (int64_t)p.slot * a.pitch;
  const int64_t pitch = a.pitch * a.n_rt;
  const int n = keys_of(a, p.b);
  float M = NO_KEYS, L = 0.f;
  f32x4 o = {0, 0, 0, 0};
  constexpr int U = 4;                         // items whose loads are in flight together
  for (int i0 = sg; ; i0 += U * SG) {
    float mi[U], li[U];
    f32x4 y[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {              // (past the last item: not used)
      const float* src = part + min(i0 + u * SG, room - 1) * pitch;
      mi[u] = src[a.rows * D + row];
      li[u] = src[a.rows * (D + 1) + row];
      y[u] = *(const f32x4*)(src + row * D + t * 4);
    }
    if (i0 == sg) {                            // the first loads wait for no count
      if (a.alike) split_alike(a, p);
      if (p.n_split == 1) return;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * SG >= p.n_split) break;
      const float to = fmaxf(M, mi[u]);
      const float k0 = fast_exp2((M - to) * a.scale2), k1 = fast_exp2((mi[u] - to) * a.scale2);
      M = to;
      L = L * k0 + li[u] * k1;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = o[e] * k0 + y[u][e] * k1;
    }
    if (i0 + U * SG >= p.n_split) break;
  }
  s_o[sg][t] = o;
  if (t == 0) {
    s_w[sg][0] = M;
    s_w[sg][1] = L;
  }
  __syncthreads();
  if (sg > 0) return;
  const int used = min(SG, p.n_split);
  for (int i = 1; i < used; ++i) M = fmaxf(M, s_w[i][0]);
  L = 0.f;
  o = (f32x4){0, 0, 0, 0};
#pragma unroll 4
  for (int i = 0; i < used; ++i) {
    const float k = fast_exp2((s_w[i][0] - M) * a.scale2);
    const f32x4 y = s_o[i][t];
    L = fmaf(s_w[i][1], k, L);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(y[e], k, o[e]);
  }
  const float inv = inverse(L, n - a.s + qi);
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] *= inv;
  store4<T>(a, p.b, hk * a.G + m - qi * a.G, qi, t * 4, o);
}

// ---------------------------------------------------------------------------
// host side

// Row tiles: as many 16-row tiles per wave as the rows fill, up to what the
// registers hold.
struct RowsPlan {
  int mt, rows, n_rt;
  int64_t pairs, items;     // (sequence, kv head, row tile) triples; item slots
  int64_t grid;             // workgroups: several row tiles in multiples of 8 of them, as they are dealt to the XCDs
  int64_t pitch;            // floats of an item's partial sums (a multiple of 4)
  int slots, whole, most;
  FastDiv round;
  size_t bytes;
};

// False for more (sequence, kv head, row tile) triples, or rows, than a launch takes.
bool plan_rows(RowsPlan& p, int B, int Hkv, int G, int s, int D, int64_t max_keys, int window, int sink) {
  constexpr int64_t MAX_PAIRS = 0x7fffff;
  p = RowsPlan{};
  const int64_t m = (int64_t)G * s;
  if (m > 1 << 28 || (int64_t)B * Hkv > MAX_PAIRS) return false;   // (the products below stay inside 64 bits)
  p.mt = m <= 16 ? 1 : m <= 32 || D == 256 ? 2 : 4;
  p.rows = (int)(m < 16 * p.mt ? m : 16 * p.mt);
  const int64_t rt = (m + 16 * p.mt - 1) / (16 * p.mt);
  p.n_rt = (int)rt;
  p.pairs = (int64_t)B * Hkv * rt;
  if (p.pairs > MAX_PAIRS) return false;
  int64_t blocks = (max_keys + KB - 1) / KB;
  if (window > 0) {
    const int64_t near = ((int64_t)window + s + 2 * KB - 2) / KB + ((int64_t)sink + KB - 1) / KB;
    if (near < blocks) blocks = near;
  }
  p.slots = 256 * 4 * rows_waves(D, p.mt) / WAVES;
  p.round = make_fastdiv(p.slots * CHUNK);
  p.items = p.pairs;
  p.whole = 0;
  p.most = 1;
  if (stays_whole(blocks, p.pairs, D, p.mt)) {
    p.whole = (int)(blocks > 1 ? blocks : 1);
  } else {
    // an upper bound of the items, whatever the lengths: the budget of the longest
    // ones and one short item a pair, but no more than items of WAVES blocks
    const int64_t most = (blocks + WAVES - 1) / WAVES;
    p.most = (int)most;
    p.items *= most;
    if (blocks * p.pairs < 0x7fffffff - p.slots * CHUNK) {
      const int64_t budget = item_budget((int)(blocks * p.pairs), p.slots, p.round), each = budget / p.pairs;
      if (each < most) p.most = (int)(each > 1 ? each : 1);
      if (budget + p.pairs < p.items) p.items = budget + p.pairs;
    }
  }
  const int64_t group = p.n_rt > 1 ? 8 * (int64_t)p.n_rt : 1;
  p.grid = (p.items + group - 1) / group * group;
  p.pitch = (int64_t)p.rows * D + (2 * p.rows + 3) / 4 * 4;
  p.bytes = p.whole > 0 ? 0 : (size_t)(p.items * p.pitch) * sizeof(float);
  return true;
}

int take_cache(Cache& c, const da_kv8_cache& x, int dtype) {
  if (dtype != DA_BF16 && dtype != DA_FP16) return DA_ERR_DTYPE;
  if (!head_dim_ok(x.D)) return DA_ERR_HEAD_DIM;
  if (x.B < 0 || x.Hkv < 1 || x.cap < KB || x.cap > MAX_CAP || x.cap % KB != 0) return DA_ERR_INVALID_ARG;
  if (x.B > 0 && (!x.k || !x.v || !x.k_scale || !x.v_scale)) return DA_ERR_INVALID_ARG;
  if (!aligned16(x.k) || !aligned16(x.v) || ((uintptr_t)x.k_scale & 3) || ((uintptr_t)x.v_scale & 3) ||
      x.k_str[0] % 16 || x.k_str[1] % 16 || x.v_str[0] % 16 || x.v_str[1] % 16)
    return DA_ERR_ALIGNMENT;
  c = Cache{(uint8_t*)x.k, (uint8_t*)x.v, x.k_scale, x.v_scale, x.k_str[0], x.k_str[1], x.v_str[0], x.v_str[1],
            x.k_scale_str[0], x.k_scale_str[1], x.v_scale_str[0], x.v_scale_str[1], x.cap};
  return DA_OK;
}

template <typename T, int D>
void launch_rows(const RowsArgs& a, const RowsPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)p.grid), block(64 * WAVES);
  if (p.mt == 1) {
    hipLaunchKernelGGL((kv8_rows_kernel<T, D, 1>), grid, block, 0, st, a);
  } else if (p.mt == 2) {
    hipLaunchKernelGGL((kv8_rows_kernel<T, D, 2>), grid, block, 0, st, a);
  } else if constexpr (D < 256) {
    hipLaunchKernelGGL((kv8_rows_kernel<T, D, 4>), grid, block, 0, st, a);
  }
  if (p.bytes > 0) {
    const dim3 rows((unsigned)p.pairs, (unsigned)p.rows);
    // Wide workgroups where few rows have many items each: 32 rows of 64 items take
    // 5.2 us (5.6 with 256 threads), 16 rows of 32 at head_dim 256 4.5 (5.2), but 768
    // rows of 16 7.7 (4.4).
    if (p.items > 16 * p.pairs && p.pairs * p.rows <= 256) hipLaunchKernelGGL((kv8_join_kernel<T, D, 1024>), rows, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((kv8_join_kernel<T, D, 256>), rows, dim3(256), 0, st, a);
  }
}

template <typename T> struct Tag { using type = T; };

// f(Tag<element>, std::integral_constant<int, head dim>)
template <typename F>
void by_type(int dtype, int D, F&& f) {
  auto dims = [&](auto t) {
    if (D == 32) f(t, std::integral_constant<int, 32>{});
    else if (D == 64) f(t, std::integral_constant<int, 64>{});
    else if (D == 128) f(t, std::integral_constant<int, 128>{});
    else f(t, std::integral_constant<int, 256>{});
  };
  if (dtype == DA_BF16) dims(Tag<__bf16>{});
  else dims(Tag<_Float16>{});
}

// Blocks of a write or read, of D / 32 waves each.
bool units_for(Units& u, int B, int n_blk, int Hkv, int D, bool read) {
  const int64_t per_seq = (int64_t)n_blk * 2 * Hkv, most = 0x3ffff00 / (D / 32);   // (threads of a grid: below 2^32)
  if (per_seq > most || per_seq * B > most) return false;
  const int64_t n = per_seq * B;
  u = Units{make_fastdiv(read ? n_blk : 2 * Hkv), make_fastdiv(n_blk * 2 * Hkv), (uint32_t)n, (uint32_t)Hkv};
  return true;
}

// Results [B, H, rows, D] by their strides: false where some share their place
// (a stride of zero over more than one entry), which leaves none of them right.
bool apart(const int64_t str[3], int B, int H, int rows) {
  return (B <= 1 || str[0]) && (H <= 1 || str[1]) && (rows <= 1 || str[2]);
}

int launched() { return hipGetLastError() == hipSuccess ? DA_OK : DA_ERR_LAUNCH; }

}  // namespace
}  // namespace da

using namespace da;

extern "C" int da_kv8_write(const da_kv8_write_args* x, void* stream) {
  if (!x) return DA_ERR_INVALID_ARG;
  WriteArgs a{};
  const int rc = take_cache(a.c, x->cache, x->dtype);
  if (rc != DA_OK) return rc;
  const int B = x->cache.B, Hkv = x->cache.Hkv, cap = x->cache.cap, S = x->S;
  if (S < 0 || (!x->pos_dev && (x->pos < 0 || x->pos > cap - (int64_t)S))) return DA_ERR_INVALID_ARG;
  if (S == 0 || B == 0) return DA_OK;
  if (!x->k || !x->v) return DA_ERR_INVALID_ARG;
  // a cache that repeats itself over sequences or heads has no one value to write
  const da_kv8_cache& c = x->cache;
  if ((B > 1 && (!c.k_str[0] || !c.v_str[0] || !c.k_scale_str[0] || !c.v_scale_str[0])) ||
      (Hkv > 1 && (!c.k_str[1] || !c.v_str[1] || !c.k_scale_str[1] || !c.v_scale_str[1])))
    return DA_ERR_INVALID_ARG;
  if (!aligned16(x->k) || !aligned16(x->v) || !strides8(x->k_str) || !strides8(x->v_str) ||
      ((uintptr_t)x->pos_dev & 7) || ((uintptr_t)x->counts_dev & 3))
    return DA_ERR_ALIGNMENT;
  a.k = x->k;
  a.v = x->v;
  a.kx_b = x->k_str[0], a.kx_s = x->k_str[1], a.kx_h = x->k_str[2];
  a.vx_b = x->v_str[0], a.vx_s = x->v_str[1], a.vx_h = x->v_str[2];
  a.pos_dev = x->pos_dev;
  a.pos = x->pos;
  a.counts = x->counts_dev;
  a.pos_step = x->pos_per_seq ? 1 : 0;
  a.counts_step = x->counts_per_seq ? 1 : 0;
  a.S = S;
  // Blocks that S tokens touch, from a known row or from any: no more than the
  // capacity's, however far a padded length passes it (a block's first row, up to
  // twice the capacity, then fits 32 bits).
  const int from_any = (int)(((int64_t)S + KB - 2) / KB + 1);
  const int n_blk = x->pos_dev ? (from_any < cap / KB ? from_any : cap / KB) : (int)((x->pos + S + KB - 1) / KB - x->pos / KB);
  if (!units_for(a.units, B, n_blk, Hkv, x->cache.D, false)) return DA_ERR_INVALID_ARG;
  (void)hipGetLastError();
  by_type(x->dtype, x->cache.D, [&](auto t, auto d) {
    using E = typename decltype(t)::type;
    constexpr int DIM = decltype(d)::value, AT_ONCE = 512 / DIM;
    const auto grid = [&](int per_wg) { return dim3((a.units.n + per_wg - 1) / per_wg); };
    if (S == 1) hipLaunchKernelGGL((kv8_append_kernel<E, DIM, 1, true>), grid(4), dim3(256), 0, (hipStream_t)stream, a);
    else if (S <= AT_ONCE) hipLaunchKernelGGL((kv8_append_kernel<E, DIM, 1, false>), grid(4), dim3(256), 0, (hipStream_t)stream, a);
    else if (S <= 2 * AT_ONCE) hipLaunchKernelGGL((kv8_append_kernel<E, DIM, 2, false>), grid(4), dim3(256), 0, (hipStream_t)stream, a);
    else hipLaunchKernelGGL((kv8_write_kernel<E, DIM>), grid(Shape<DIM>::PER_WG), dim3(Shape<DIM>::THREADS), 0, (hipStream_t)stream, a);
  });
  return launched();
}

extern "C" int da_kv8_read(const da_kv8_read_args* x, void* stream) {
  if (!x) return DA_ERR_INVALID_ARG;
  ReadArgs a{};
  const int rc = take_cache(a.c, x->cache, x->dtype);
  if (rc != DA_OK) return rc;
  const int B = x->cache.B, start = x->start, n = x->n;
  if (start < 0 || n < 0 || (int64_t)start + n > x->cache.cap) return DA_ERR_INVALID_ARG;
  if (n == 0 || B == 0) return DA_OK;
  if (!x->k || !x->v || !apart(x->k_str, B, x->cache.Hkv, n) || !apart(x->v_str, B, x->cache.Hkv, n))
    return DA_ERR_INVALID_ARG;
  if (!aligned16(x->k) || !aligned16(x->v) || !strides8(x->k_str) || !strides8(x->v_str) ||
      ((uintptr_t)x->n_keys_dev & 3))
    return DA_ERR_ALIGNMENT;
  a.k = x->k;
  a.v = x->v;
  a.ko_b = x->k_str[0], a.ko_h = x->k_str[1], a.ko_s = x->k_str[2];
  a.vo_b = x->v_str[0], a.vo_h = x->v_str[1], a.vo_s = x->v_str[2];
  a.n_keys = x->n_keys_dev;
  a.n_step = x->n_keys_per_seq ? 1 : 0;
  a.start = start, a.n = n;
  const int n_blk = (int)(((int64_t)start + n + KB - 1) / KB - start / KB);
  if (!units_for(a.units, B, n_blk, x->cache.Hkv, x->cache.D, true)) return DA_ERR_INVALID_ARG;
  (void)hipGetLastError();
  by_type(x->dtype, x->cache.D, [&](auto t, auto d) {
    constexpr int DIM = decltype(d)::value, W = Shape<DIM>::W;
    hipLaunchKernelGGL((kv8_read_kernel<typename decltype(t)::type, DIM>), dim3((a.units.n * W + 3) / 4), dim3(256), 0,
                       (hipStream_t)stream, a);
  });
  return launched();
}

extern "C" size_t da_kv8_attn_workspace_bytes(int B, int Hq, int Hkv, int s, int D, int max_keys,
                                              int window, int sink) {
  if (B < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv != 0 || s < 1 || !head_dim_ok(D) || max_keys < 0 ||
      window < 0 || sink < 0)
    return 0;
  RowsPlan p;
  return plan_rows(p, B, Hkv, Hq / Hkv, s, D, max_keys, window, sink) ? p.bytes : 0;
}

extern "C" int da_kv8_attn_fwd(const da_kv8_attn_args* x, void* stream) {
  if (!x) return DA_ERR_INVALID_ARG;
  RowsArgs a{};
  const int rc = take_cache(a.c, x->cache, x->dtype);
  if (rc != DA_OK) return rc;
  const int B = x->cache.B, Hkv = x->cache.Hkv, cap = x->cache.cap, Hq = x->Hq, s = x->s;
  if (Hq < 1 || Hq % Hkv != 0 || s < 0 || x->window < 0 || x->sink < 0) return DA_ERR_INVALID_ARG;
  if (!x->n_keys_dev && (x->n_keys < 0 || x->n_keys > cap)) return DA_ERR_INVALID_ARG;
  if (!(fabsf(x->sm_scale) <= FLT_MAX)) return DA_ERR_INVALID_ARG;
  if (s == 0 || B == 0) return DA_OK;
  if (!x->q || !x->out || !apart(x->o_str, B, Hq, s)) return DA_ERR_INVALID_ARG;
  if (!aligned16(x->q) || !aligned16(x->out) || !strides8(x->q_str) || !strides8(x->o_str) ||
      ((uintptr_t)x->n_keys_dev & 3) || (x->addend && (!aligned16(x->addend) || !strides8(x->add_str))))
    return DA_ERR_ALIGNMENT;
  // (a window or sinks past the capacity are every key)
  a.window = x->window < cap ? x->window : cap;
  a.sink = x->sink < cap ? x->sink : cap;
  RowsPlan p;
  if (!plan_rows(p, B, Hkv, Hq / Hkv, s, x->cache.D, x->n_keys_dev ? cap : x->n_keys, a.window, a.sink) ||
      p.items * 256 > 0x7fffffffll || p.grid * (64 * WAVES) > 0xffffffffll || p.pairs * (cap / KB) > 0x70000000ll)
    return DA_ERR_INVALID_ARG;
  if (p.bytes > 0 && (!x->workspace || x->workspace_bytes < (int64_t)p.bytes)) return DA_ERR_WORKSPACE;
  if (!aligned16(x->workspace)) return DA_ERR_ALIGNMENT;
  a.q = x->q;
  a.q_b = x->q_str[0], a.q_h = x->q_str[1], a.q_s = x->q_str[2];
  a.o = x->out;
  a.o_b = x->o_str[0], a.o_h = x->o_str[1], a.o_s = x->o_str[2];
  a.add = x->addend;
  a.add_b = x->add_str[0], a.add_h = x->add_str[1], a.add_s = x->add_str[2];
  a.n_dev = x->n_keys_dev;
  a.n_step = x->n_keys_per_seq ? 1 : 0;
  a.n = x->n_keys;
  a.B = B, a.Hkv = Hkv, a.G = Hq / Hkv, a.s = s;
  a.n_rt = p.n_rt, a.rows = p.rows;
  // (a scale of zero, which weighs every key alike, as the smallest one: it moves
  // no weight by more than 2^-20, and a masked score's -inf stays -inf)
  a.scale2 = fminf(fmaxf(fabsf(x->sm_scale) * (2 * 1.4426950408889634f), FLT_TRUE_MIN), FLT_MAX);
  a.flip = x->sm_scale < 0.f ? 0x80008000u : 0;
  a.whole = p.whole;
  a.most = p.most;
  a.alike = p.whole > 0 || B == 1 || !a.n_dev || a.n_step == 0;
  a.slots = p.slots;
  a.round = p.round;
  a.units = make_fastdiv(Hkv * p.n_rt);
  a.tiles = make_fastdiv(p.n_rt);
  a.heads = make_fastdiv(a.G);
  a.part = (float*)x->workspace;
  a.pitch = p.pitch;
  (void)hipGetLastError();
  by_type(x->dtype, x->cache.D, [&](auto t, auto d) {
    launch_rows<typename decltype(t)::type, decltype(d)::value>(a, p, (hipStream_t)stream);
  });
  return launched();
}
