// Attention rows of a batch whose sequences share prefixes (gfx950 / CDNA4):
// sequence b of B reads the keys of prefix b / (B / P) and keys of its own.
//
//   o = softmax(scale q [Kp; K]^T) [Vp; V]
//
// A softmax over two key sets is the join of the softmaxes over each: with the
// rows' references m, sums l = sum 2^(x - m) and products a = sum 2^(x - m) v of
// each set, o = sum a 2^(m - M) / sum l 2^(m - M). So the prefix is one matrix
// product over the rows of all sequences that share it (n s G rows for n
// sequences of s rows and G query heads a kv head), read once, and each
// sequence's own keys are another over its s G rows.
//
// What bounds it: up to some 128 rows a kv head the keys' bytes (16 sequences of 32 / 8
// heads of 128 over 131072 keys 108 us in all, 5.4 TB/s; one sequence alone takes 90), past
// that the matrix products and the exponentials beside them (128 sequences over 65536 keys
// 178 us, 775 TFLOP/s; 16 of 128 rows each over 32768 keys 1050), and for few keys two
// launches (10.5 us for 2711) or one (5.7 to 7.2 us up to 256). The rows of a batch over whole caches, each with a copy of the prefix,
// take 50 us where 16 share 4096 keys in 15, and 324 where 4 share 131072 in 92.
#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "capi_common.h"
#include "delta_attn.h"
#include "device_common.h"

namespace da {
namespace {

constexpr int BN = 64;                       // keys per tile
constexpr int WAVES = 4;
constexpr int MAX_KEYS = 1 << 30;
constexpr float NO_KEYS = -FLT_MAX;          // the reference of a row that has seen no score yet
// A row's reference may lag its largest score by LAG (log2); fp16 probabilities
// are held times 2^BIAS, so that they are at most 2^14 and end 2^-32 below it.
// (With LAG 0 128 sequences over 65536 keys take 193 us for 187.)
constexpr float LAG = 6.f;
template <typename T> constexpr float BIAS = std::is_same_v<T, _Float16> ? 8.f : 0.f;

struct PrefixArgs {
  const void *q, *kp, *vp, *k, *v;
  void* o;
  int64_t q_b, q_h, q_s, o_b, o_h, o_s;
  int64_t kp_b, kp_h, vp_b, vp_h, k_b, k_h, v_b, v_h;
  uint32_t kp_s, vp_s, k_s, v_s;            // bytes from key to key
  const int *np_dev, *n_dev;                // key counts on the device, or NULL: np, n
  int np_step, n_step, np, n, Np, cap;      // (counts are clamped to Np and cap)
  int B, P, per, Hkv, G, s;                 // per = B / P sequences a prefix
  int rows;                                 // B * s * G: rows of a kv head
  int p_rows, p_rt, o_rows, o_rt;           // rows of a prefix's sequences and of a sequence, their row tiles
  int p_splits, o_splits, p_chunk, o_chunk; // splits of the keys, tiles of each
  int p_items, p_grid;                      // items of the prefixes; their workgroups, before those of the sequences' own
  FastDiv heads, rows_s, f_prt, f_psp, f_ort, f_osp, f_hkv, f_rows, f_per;   // G, s, p_rt, p_splits, o_rt, o_splits, Hkv, rows, per
  float scale2;                             // |sm_scale| log2(e), above zero
  uint32_t flip;                            // the sign bits of Q where sm_scale is negative
  float *part, *part_m, *part_l;            // [Hkv, splits, rows, D], [Hkv, splits, rows] twice
};

// Loads that are not kept in the caches: where no other row tile reads a split's keys (one
// row tile a split: 16 sequences over 131072 keys 124 -> 108 us, 3 x 5 over 20011 66 -> 57).
// Where tiles share them they cost the sharing: 128 sequences over 65536 keys 193 -> 216 us.
// The sequences' own keys come by ordinary loads (by these 57 -> 59 us).
__device__ __forceinline__ void dma16_nt(u32x4 r, uint32_t lds, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
               :: "s"(lds), "v"(voff), "s"(r) : "memory");
}
template <typename T> struct Mma;
template <> struct Mma<__bf16> {
  static constexpr uint32_t inf = 0x7f80, one = 0x3f80;
  static __device__ __forceinline__ f32x4 dot(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Mma<_Float16> {
  static constexpr uint32_t inf = 0x7c00, one = 0x3c00;
  static __device__ __forceinline__ f32x4 dot(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// A K or V tile in LDS: rows of D elements, their 16-byte chunks permuted by the
// row (chunk ^ swz(row)), so that the 16 rows that a fragment read takes the same
// chunk of lie in different banks.
template <int D> struct Tile {
  static constexpr int RB = 2 * D, CH = D / 8, BYTES = BN * RB;
  static constexpr int DMAS = BYTES / (1024 * WAVES);     // 1024-byte loads of a wave
  static __device__ __forceinline__ int swz(int row) { return (RB >= 256 ? row : row / (256 / RB)) & (CH < 16 ? CH - 1 : 15); }
};

__device__ __forceinline__ float group_max(float x) {      // over the four lanes of a row
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float group_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return sum32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Two elements' marks: the element one where f(element without sign, sign) holds.
template <typename T, typename F>
__device__ __forceinline__ uint32_t marks(uint32_t w, F&& f) {
  constexpr uint32_t one = Mma<T>::one;
  return (f(w & 0x7fffu, w >> 15 & 1) ? one : 0u) | (f(w >> 16 & 0x7fffu, w >> 31) ? one << 16 : 0u);
}

__device__ __forceinline__ int prefix_keys(const PrefixArgs& a, int p) {
  return min(max(a.np_dev ? a.np_dev[(int64_t)p * a.np_step] : a.np, 0), a.Np);
}
__device__ __forceinline__ int own_keys(const PrefixArgs& a, int b) {
  return min(max(a.n_dev ? a.n_dev[(int64_t)b * a.n_step] : a.n, 0), a.cap);
}

// Waves of a SIMD: what the accumulators and two tiles of scores leave room for.
__host__ __device__ constexpr int waves_of(int D, int mt) { return D == 256 ? 1 : D == 128 ? 2 : D * mt == 128 ? 3 : 4; }

// A wave's 16 MT rows (row c = lane % 16 of each): their queries and what they have
// gathered. ref: scaled, in log2.
template <typename T, int D, int MT>
struct Rows {
  u32x4 q[MT][D / 32];
  f32x4 acc[MT][D / 16];
  float ref[MT], sum[MT];
  int own[MT];                               // the row's place among its sequence's s rows
  // the rows from row0 on of kv head hk, n_rows of the workgroup
  __device__ __forceinline__ Rows(const PrefixArgs& a, int hk, int row0, int n_rows) {
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), c = lane % 16, g = lane / 16;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = row0 + min(wave * 16 * MT + mt * 16 + c, n_rows - 1);   // (past the last: it again)
      const int x = fdiv(r, a.heads), b = fdiv(x, a.rows_s), i = x - b * a.s;
      own[mt] = i;
      const T* src = (const T*)a.q + b * a.q_b + (int64_t)(hk * a.G + r - x * a.G) * a.q_h + i * a.q_s;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) q[mt][k] = *(const u32x4*)(src + 32 * k + 8 * g) ^ a.flip;
      ref[mt] = NO_KEYS;
      sum[mt] = 0.f;
#pragma unroll
      for (int t = 0; t < D / 16; ++t) acc[mt][t] = (f32x4){0, 0, 0, 0};
    }
  }
};

// A head's keys and values, and the bytes from key to key.
struct Keys {
  const char *k, *v;
  uint32_t k_s, v_s;
  int n;
};
template <bool OWN>
__device__ __forceinline__ Keys keys_of(const PrefixArgs& a, int list, int hk) {
  Keys x;
  x.k = (const char*)(OWN ? a.k : a.kp) + 2 * (OWN ? list * a.k_b + hk * a.k_h : list * a.kp_b + hk * a.kp_h);
  x.v = (const char*)(OWN ? a.v : a.vp) + 2 * (OWN ? list * a.v_b + hk * a.v_h : list * a.vp_b + hk * a.vp_h);
  x.k_s = OWN ? a.k_s : a.kp_s;
  x.v_s = OWN ? a.v_s : a.vp_s;
  x.n = __builtin_amdgcn_readfirstlane(OWN ? own_keys(a, list) : prefix_keys(a, list));
  return x;
}

// The rows against the keys of [key0, stop), in tiles that all waves load into LDS
// together, the next one while this one is computed. row0, n_rows: the workgroup's.
// S^T = K Q^T leaves a lane (row c = lane % 16, group g = lane / 16) the keys 16 t
// + 4 g + r of its row, which is the right operand of O^T = V^T P^T as it stands;
// V^T comes from transposed LDS reads of the same keys. Probabilities are rounded to the
// inputs' type for that product, half a step of which is within the result's own, and
// summed as rounded, so that a row's weights add up to one.
// -> the number of tiles
template <typename T, int D, int MT, bool OWN, bool STREAM>
__device__ __forceinline__ int walk(const PrefixArgs& a, Rows<T, D, MT>& rows, const Keys& keys, int key0, int stop, int row0,
                                    int n_rows, bool active, char (&smem)[2][2][Tile<D>::BYTES]) {
  using E = Elt<T>;
  using M = Mma<T>;
  using TL = Tile<D>;
  constexpr int KS = D / 32, DT = D / 16, KG = BN / 16;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int c = lane % 16, g = lane / 16;
  const char *kb = keys.k, *vb = keys.v;
  const uint32_t k_s = keys.k_s, v_s = keys.v_s;
  const int n_keys = keys.n;
  auto &acc = rows.acc;
  auto &ref = rows.ref, &sum = rows.sum;
  auto &qf = rows.q;

  // each row's last key
  const int lim0 = OWN ? n_keys - a.s : n_keys - 1;
  int lim[MT], lim_lo = lim0, lim_hi = lim0;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) lim[mt] = OWN ? lim0 + rows.own[mt] : lim0;
  if (OWN) {                                 // of the whole row tile (which may be a single row's heads)
    const int u = fdiv(row0, a.heads), w = fdiv(row0 + n_rows - 1, a.heads);
    lim_lo += u - (int)fdiv(u, a.rows_s) * a.s;
    lim_hi += w - (int)fdiv(w, a.rows_s) * a.s;
  }
  const int end = min(min(stop, n_keys), lim_hi + 1);
  const int nt = end > key0 ? (end - key0 + BN - 1) / BN : 0;

  // loads: lane i of load j of a wave fills chunk i of the wave's 1024 bytes
  uint32_t koff[TL::DMAS], voff[TL::DMAS];
#pragma unroll
  for (int j = 0; j < TL::DMAS; ++j) {
    const int at = (j * WAVES + wave) * 64 + lane, row = at / TL::CH, ch = (at % TL::CH) ^ TL::swz(row);
    koff[j] = row * k_s + ch * 16;
    voff[j] = row * v_s + ch * 16;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(DA_LDS char*)&smem[0][0][0];
  auto issue = [&](bool values, int t) __attribute__((always_inline)) {
    const int first = key0 + t * BN;
    const uint32_t step = values ? v_s : k_s;
    const int64_t left = (int64_t)(lim_hi - first) * step + TL::RB;   // what lies behind the last key seen reads as zero
    const u32x4 r = rsrc_words((values ? vb : kb) + (int64_t)first * step, left >> 32 ? 0xffffffffu : (uint32_t)left);
    const uint32_t st = lds0 + (t % 2 * 2 + values) * TL::BYTES + wave * 1024;
#pragma unroll
    for (int j = 0; j < TL::DMAS; ++j) {
      if (STREAM) dma16_nt(r, st + j * WAVES * 1024, values ? voff[j] : koff[j]);
      else dma16_untracked(r, st + j * WAVES * 1024, values ? voff[j] : koff[j]);
    }
  };
  int kread[KS], vread[DT];
#pragma unroll
  for (int k = 0; k < KS; ++k) kread[k] = c * TL::RB + ((4 * k + g) ^ TL::swz(c)) * 16;
#pragma unroll
  for (int t = 0; t < DT; ++t) {
    const int row = 4 * g + c / 4;
    vread[t] = row * TL::RB + ((2 * t + c % 4 / 2) ^ TL::swz(row)) * 16 + c % 2 * 8;
  }

  // scores of tile t (raw), with -inf where a row does not see the key
  auto scores = [&](int t, f32x4 (&s)[MT][KG]) __attribute__((always_inline)) {
    const DA_LDS char* ks = (const DA_LDS char*)&smem[t % 2][0][0];
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int i = 0; i < KG; ++i) {
        const u32x4 ka = *(const DA_LDS u32x4*)(ks + kread[k] + 16 * i * TL::RB);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt][i] = M::dot(ka, qf[mt][k], k == 0 ? (f32x4){0, 0, 0, 0} : s[mt][i]);
      }
  };
  // the references move where a row's largest score passes its own by LAG
  auto follow = [&](int t, f32x4 (&s)[MT][KG]) __attribute__((always_inline)) {
    const int first = key0 + t * BN;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if (first + BN - 1 > lim_lo) {
        const int hi = lim[mt] - first - 4 * g;
#pragma unroll
        for (int e = 0; e < 4 * KG; ++e) s[mt][e / 4][e % 4] = e / 4 * 16 + e % 4 <= hi ? s[mt][e / 4][e % 4] : -INFINITY;
      }
      // (IEEE maximum: it needs no quieting of its operands, and a NaN moves no
      // reference but reaches the row's sum)
      float top = s[mt][0][0];
#pragma unroll
      for (int e = 1; e < 4 * KG; ++e) top = __builtin_elementwise_maximum(top, s[mt][e / 4][e % 4]);
      top = group_max(top) * a.scale2;
      if (__any(top - ref[mt] > LAG)) {
        const float to = fmaxf(ref[mt], top), alpha = fast_exp2(ref[mt] - to);
        ref[mt] = to;
        sum[mt] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[mt][d][r] *= alpha;
      }
    }
  };

  // Step t: the scores of tile t + 1 are formed beside the probabilities of tile t,
  // then its products with the values. K(t + 2) and V(t + 1) are on their way: into
  // the places of K(t) and V(t - 1), which step t - 1 read last.
  f32x4 s[MT][KG];
  if (nt > 0) {
    issue(false, 0);
    issue(true, 0);
    if (nt > 1) issue(false, 1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    if (active) {
      scores(0, s);
      follow(0, s);
    }
  }
  for (int t = 0; t < nt; ++t) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    if (t + 2 < nt) issue(false, t + 2);
    if (t + 1 < nt) issue(true, t + 1);
    if (!active) continue;
    const DA_LDS char* vs = (const DA_LDS char*)&smem[t % 2][1][0];
    const int first = key0 + t * BN;
    const bool whole = first + BN - 1 <= lim_lo;
    u32x4 pf[MT][KG / 2];
    f32x4 next[MT][KG];
    // A wave with products to issue goes before one that masks, compares or waits: 128
    // sequences over 65536 keys 190 -> 179 us, 1536 rows over 30011 of 64 127 -> 121. (From the
    // scores to the probabilities alone 183 and 122, throughout the step 187 and 124.)
    __builtin_amdgcn_s_setprio(1);
    scores(t + 1, next);                     // (behind the last tile: of what lies there, not used)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const float off = BIAS<T> - ref[mt];
#pragma unroll
      for (int u = 0; u < KG / 2; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int i = 2 * u + w / 2, r = w % 2 * 2;
          auto weight = [&](float y) __attribute__((always_inline)) { return fast_exp2(fmaf(y, a.scale2, off)); };
          pf[mt][u][w] = E::pack2(weight(s[mt][i][r]), weight(s[mt][i][r + 1]));
          sum[mt] = E::add_pair(pf[mt][u][w], sum[mt]);   // (the rounded ones: as the product has them)
        }
    }
    auto values = [&](int u, int d) __attribute__((always_inline)) -> u32x4 {
      const u32x2 v0 = read_tr16(vs + vread[d] + 32 * u * TL::RB), v1 = read_tr16(vs + vread[d] + (32 * u + 16) * TL::RB);
      return (u32x4){v0[0], v0[1], v1[0], v1[1]};
    };
    // An infinity or NaN among the values of a key that one of the rows does not see
    // must not reach it through 0 * inf (keys that none of them sees are loaded as zero).
    bool odd = false;
    if (OWN && !whole && lim_lo < lim_hi) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int u = 0; u < KG / 2; ++u) {
          const u32x4 va = values(u, d);
#pragma unroll
          for (int w = 0; w < 4; ++w)
            odd |= (va[w] & M::inf) == M::inf || (va[w] >> 16 & M::inf) == M::inf;
        }
      odd = __any(odd);
    }
    if (OWN && odd) {
      // taken as zero, and given to the rows that see them from products of the
      // values' and the rows' marks
#pragma unroll
      for (int u = 0; u < KG / 2; ++u) {
        u32x4 sees[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int at = first + 32 * u + w / 2 * 16 + 4 * g + w % 2 * 2;
            sees[mt][w] = (at <= lim[mt] ? M::one : 0u) | (at + 1 <= lim[mt] ? M::one << 16 : 0u);
          }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          u32x4 va = values(u, d), up, down, none;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            up[w] = marks<T>(va[w], [](uint32_t x, uint32_t neg) { return x == M::inf && !neg; });
            down[w] = marks<T>(va[w], [](uint32_t x, uint32_t neg) { return x == M::inf && neg; });
            none[w] = marks<T>(va[w], [](uint32_t x, uint32_t) { return x > M::inf; });
            va[w] &= ((va[w] & M::inf) == M::inf ? 0u : 0xffffu) | ((va[w] >> 16 & M::inf) == M::inf ? 0u : 0xffff0000u);
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            const f32x4 zero = {0, 0, 0, 0};
            const f32x4 a = M::dot(up, sees[mt], zero), b = M::dot(down, sees[mt], zero), c = M::dot(none, sees[mt], zero);
            acc[mt][d] = M::dot(va, pf[mt][u], acc[mt][d]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              if (a[r] > 0.f) acc[mt][d][r] += INFINITY;
              if (b[r] > 0.f) acc[mt][d][r] -= INFINITY;
              if (c[r] > 0.f) acc[mt][d][r] = __builtin_nanf("");
            }
          }
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < KG / 2; ++u)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          const u32x4 va = values(u, d);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) acc[mt][d] = M::dot(va, pf[mt][u], acc[mt][d]);
        }
    }
    __builtin_amdgcn_s_setprio(0);
    if (t + 1 < nt) follow(t + 1, next);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < KG; ++i) s[mt][i] = next[mt][i];
  }
  return nt;
}

// Writes a kv head's row, four columns from `col` on for each f(col, sums) that `each`
// calls. A row without keys is zero; one whose every score is -inf has no softmax: NaN.
template <typename T, int D, typename F>
__device__ __forceinline__ void put_row(const PrefixArgs& a, int hk, int row, float l, F&& each) {
  using E = Elt<T>;
  const int y = fdiv(row, a.heads), b = fdiv(y, a.rows_s), i = y - b * a.s;
  const bool none = prefix_keys(a, fdiv(b, a.f_per)) == 0 && own_keys(a, b) - a.s + i < 0;
  const float inv = none ? 0.f : 1.f / l;
  T* dst = (T*)a.o + b * a.o_b + (int64_t)(hk * a.G + row - y * a.G) * a.o_h + i * a.o_s;
  each([&](int col, const f32x4& o) __attribute__((always_inline)) {
    *(u32x2*)(dst + col) = (u32x2){E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv)};
  });
}

// One item: a row tile of 16 MT rows a wave against a split's keys.
template <typename T, int D, int MT, bool OWN, bool STREAM>
__device__ __forceinline__ void rows_item(const PrefixArgs& a, int item, char (&smem)[2][2][Tile<D>::BYTES]) {
  constexpr int BM = 16 * MT * WAVES;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int c = lane % 16, g = lane / 16;

  // the item: (prefix or sequence, kv head, split, row tile), the row tiles of a
  // split beside each other
  const int x0 = fdiv(item, OWN ? a.f_ort : a.f_prt), tile = item - x0 * (OWN ? a.o_rt : a.p_rt);
  const int y0 = fdiv(x0, OWN ? a.f_osp : a.f_psp), part = x0 - y0 * (OWN ? a.o_splits : a.p_splits);
  const int list = fdiv(y0, a.f_hkv), hk = y0 - list * a.Hkv;        // list: the prefix or the sequence
  const int n_rows = min(BM, (OWN ? a.o_rows : a.p_rows) - tile * BM);
  const int row0 = list * (OWN ? a.o_rows : a.p_rows) + tile * BM;    // of the kv head's rows
  const int chunk = OWN ? a.o_chunk : a.p_chunk, split = OWN ? part + a.p_splits : part, key0 = part * chunk * BN;
  const bool active = wave * 16 * MT < n_rows;
  const Keys keys = keys_of<OWN>(a, list, hk);
  Rows<T, D, MT> rows(a, hk, row0, n_rows);
  const int nt = walk<T, D, MT, OWN, STREAM>(a, rows, keys, key0, key0 + chunk * BN, row0, n_rows, active, smem);

  if (!active) return;
  const int64_t slot = ((int64_t)hk * (a.p_splits + a.o_splits) + split) * a.rows;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = wave * 16 * MT + mt * 16 + c;
    const float l = group_sum(rows.sum[mt]);
    if (r >= n_rows) continue;
    const int64_t at = slot + row0 + r;
    if (g == 0) {
      a.part_m[at] = rows.ref[mt];
      a.part_l[at] = l;
    }
    if (nt == 0) continue;                   // (nothing reads the sums of a split without keys)
#pragma unroll
    for (int d = 0; d < D / 16; ++d) *(f32x4*)(a.part + at * D + 16 * d + 4 * g) = rows.acc[mt][d];
  }
}

template <typename T, int D, int MT>
__global__ __launch_bounds__(64 * WAVES, waves_of(D, MT)) void prefix_rows_kernel(PrefixArgs a) {
  __shared__ __align__(1024) char smem[2][2][Tile<D>::BYTES];
  int item = blockIdx.x;
  if (item >= a.p_grid) {
    rows_item<T, D, 1, true, false>(a, item - a.p_grid, smem);
  } else if (a.p_rt > 1) {
    // The row tiles of one split run on one XCD (workgroup x runs on XCD x % 8):
    // its L2 holds the keys that they share.
    const int q = item / 8, k = fdiv(q, a.f_prt);
    item = (k * 8 + item % 8) * a.p_rt + q - k * a.p_rt;
    if (item < a.p_items) rows_item<T, D, MT, false, false>(a, item, smem);
  } else {
    rows_item<T, D, MT, false, true>(a, item, smem);
  }
}

// Short keys: a row tile of a sequence against its prefix and its own keys, and its
// output, in one launch without partial sums.
template <typename T, int D>
__global__ __launch_bounds__(64 * WAVES, waves_of(D, 1)) void prefix_whole_kernel(PrefixArgs a) {
  __shared__ __align__(1024) char smem[2][2][Tile<D>::BYTES];
  constexpr int BM = 16 * WAVES;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int c = lane % 16, g = lane / 16;
  const int y0 = fdiv(blockIdx.x, a.f_ort), tile = blockIdx.x - y0 * a.o_rt;
  const int b = fdiv(y0, a.f_hkv), hk = y0 - b * a.Hkv;
  const int n_rows = min(BM, a.o_rows - tile * BM), row0 = b * a.o_rows + tile * BM;
  const bool active = wave * 16 < n_rows;
  const Keys prefix = keys_of<false>(a, fdiv(b, a.f_per), hk), own = keys_of<true>(a, b, hk);
  Rows<T, D, 1> rows(a, hk, row0, n_rows);
  walk<T, D, 1, false, false>(a, rows, prefix, 0, prefix.n, row0, n_rows, active, smem);
  lds_barrier();                             // (the last tiles are read)
  walk<T, D, 1, true, false>(a, rows, own, 0, own.n, row0, n_rows, active, smem);
  const int r = wave * 16 + c;
  const float l = group_sum(rows.sum[0]);
  if (r >= n_rows) return;
  put_row<T, D>(a, hk, row0 + r, l, [&](auto&& at) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < D / 16; ++d) at(16 * d + 4 * g, rows.acc[0][d]);
  });
}

// Joins a row's splits: groups of D / 4 threads, `side` (a power of two) of them a
// row, take splits side by side, four loads of each in flight, and are joined
// through LDS. One group a row, as first built, walked the splits one after another:
// 148 us in place of 119 for 16 sequences over 131072 keys, 76 for 48 at 40009 of 256. It
// takes 4 to 10 us now: its launch, and the partial sums' way through memory.
template <typename T, int D>
__global__ __launch_bounds__(256) void prefix_join_kernel(PrefixArgs a, int side) {
  constexpr int CT = D / 4, GROUPS = 256 / CT, U = 4;
  __shared__ f32x4 s_o[GROUPS][CT];
  __shared__ float s_m[GROUPS], s_l[GROUPS];
  const int t = threadIdx.x % CT, group = threadIdx.x / CT, sg = group & (side - 1);
  const int x = blockIdx.x * (GROUPS / side) + group / side;
  const bool live = x < a.rows * a.Hkv;
  const int hk = live ? fdiv(x, a.f_rows) : 0, row = live ? x - hk * a.rows : 0;
  const int splits = a.p_splits + a.o_splits;
  const int64_t at = (int64_t)hk * splits * a.rows + row;
  float m = NO_KEYS, l = 0.f;
  f32x4 o = {0, 0, 0, 0};
  for (int j0 = sg; j0 < splits; j0 += U * side) {
    float mj[U], lj[U];
    f32x4 z[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {              // (past the last: it again, without weight)
      const int64_t i = at + (int64_t)min(j0 + u * side, splits - 1) * a.rows;
      mj[u] = a.part_m[i];
      lj[u] = a.part_l[i];
      z[u] = *(const f32x4*)(a.part + i * D + 4 * t);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (lj[u] == 0.f || j0 + u * side >= splits) continue;   // (a split without keys holds no sums)
      const float to = fmaxf(m, mj[u]), k0 = fast_exp2(m - to), k1 = fast_exp2(mj[u] - to);
      m = to;
      l = l * k0 + lj[u] * k1;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = o[e] * k0 + z[u][e] * k1;
    }
  }
  if (side > 1) {
    s_o[group][t] = o;
    if (t == 0) {
      s_m[group] = m;
      s_l[group] = l;
    }
    __syncthreads();
    if (sg > 0) return;
    for (int i = 1; i < side; ++i) m = fmaxf(m, s_m[group + i]);
    l = 0.f;
    o = (f32x4){0, 0, 0, 0};
#pragma unroll 4
    for (int i = 0; i < side; ++i) {
      const float k = fast_exp2(s_m[group + i] - m);
      const f32x4 z = s_o[group + i][t];
      l = fmaf(s_l[group + i], k, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(z[e], k, o[e]);
    }
  }
  if (!live) return;
  put_row<T, D>(a, hk, row, l, [&](auto&& at) __attribute__((always_inline)) { at(4 * t, o); });
}

// ---------------------------------------------------------------------------
// host side

struct Plan {
  int mt, p_rt, o_rt, p_splits, o_splits, p_chunk, o_chunk;
  int64_t p_items, p_grid, grid, rows;
  bool whole;                                // one launch without splits
  size_t bytes;
};

bool plan_for(Plan& p, int B, int P, int Hkv, int G, int s, int D, int64_t Np, int64_t cap) {
  constexpr int64_t MOST = 1 << 22;          // items and row tiles of a launch
  p = Plan{};
  const int64_t own = (int64_t)s * G;
  if (own > MOST || (int64_t)B * Hkv > MOST || own * B > MOST) return false;
  p.rows = own * B;
  const int64_t p_rows = p.rows / P;
  // 16 rows a wave, 32 where a prefix has more than a workgroup of those: the keys are
  // read from LDS once for both. By 16 / 32: 4 rows over 2711 keys 10.4 / 11.0 us, 16 over
  // 40009 at head_dim 256 37.8 / 55.7; 512 rows over 65536 keys 208 / 187, 1536 over 30011
  // at head_dim 64 146 / 125. (64 rows, as far as registers allow, 220 and 260.)
  p.mt = p_rows <= 64 ? 1 : 2;
  const int bm = 16 * p.mt * WAVES;
  const int64_t p_rt = Np > 0 ? (p_rows + bm - 1) / bm : 0, o_rt = cap > 0 ? (own + 16 * WAVES - 1) / (16 * WAVES) : 0;
  const int64_t p_tiles = (Np + BN - 1) / BN, o_tiles = (cap + BN - 1) / BN;
  const int64_t p_lists = P * Hkv * p_rt, o_lists = (int64_t)B * Hkv * o_rt;
  if (p_lists > MOST || o_lists > MOST) return false;
  // Short keys take one launch: 4.1 us and 0.78 a tile (5 and 1.27 at head_dim 256), where
  // two take 9 and more with the sums that they pass on. By one launch / two: 4 sequences of
  // 8 x 4 heads of 128 with 2, 4, 8 tiles 5.7 / 9.3, 7.2 / 8.4, 10.2 / 9.6 us; 64 of 8 x 8
  // with 8, 12, 16 11.1 / 17.9, 14.2 / 18.3, 17.3 / 19.2; 8 of 20 rows of 64 with 12, 16
  // 13.7 / 15.1, 16.9 / 17.4; 16 of 4 x 2 heads of 256 with 2, 4, 8 7.7 / 9.1, 10.2 / 10.1,
  // 15.6 / 11.7.
  const int64_t sums = (p.rows * Hkv * D) >> 16, most = 6 + (sums < 8 ? sums : 8);
  p.whole = p_tiles + o_tiles <= (D == 256 ? most / 2 : most);
  if (p.whole) {
    p.o_rt = (int)((own + 16 * WAVES - 1) / (16 * WAVES));
    p.grid = (int64_t)B * Hkv * p.o_rt;
    p.p_rt = p.p_chunk = p.o_chunk = 1;
    return p.grid <= MOST;
  }
  const int64_t slots = 256 * waves_of(D, p.mt);
  // Tiles of an item: the count whose items end first, on a model of a launch. An
  // item takes its tiles and START more; the prefixes' items start first, the
  // sequences' own in the places beside or behind them; a split costs its partial
  // sums' way to memory and back. (Against one round of equal items: 3 prefixes of 5
  // sequences with 3008 keys of their own each 82 -> 72 us, 512 at head_dim 256 42 -> 37.
  // Spreading the own items among the prefixes' in launch order: 128 sequences over 65536
  // keys 186 -> 211 us, 16 over 131072 108 -> 116.)
  constexpr double START = 1.5;
  const int64_t least = (p_lists * p_tiles + o_lists * o_tiles + slots - 1) / slots;
  double best = 0;
  for (int64_t c = least < 2 ? 2 : least; c <= least + 40; ++c) {
    const int64_t ps = p_rt > 0 ? (p_tiles + c - 1) / c : 0, os = o_rt > 0 ? (o_tiles + c - 1) / c : 0;
    const int64_t pc = ps > 0 ? (p_tiles + ps - 1) / ps : 0, oc = os > 0 ? (o_tiles + os - 1) / os : 0;
    const int64_t pi = p_lists * ps, oi = o_lists * os, rounds = pi / slots, rest = pi % slots, room = slots - rest;
    const double tp = START + pc, to = START + oc;
    const double beside = rest > 0 ? tp : 0, own_beside = (double)((oi + room - 1) / room) * to;
    const double with = rounds * tp + (beside > own_beside ? beside : own_beside);
    const double behind = rounds * tp + beside + (double)((oi + slots - 1) / slots) * to;
    const double t = (with < behind ? with : behind) + (double)(p.rows * Hkv * (ps + os)) / (32 * slots);
    if (best == 0 || t < best) {
      best = t;
      p.p_splits = (int)ps, p.o_splits = (int)os;
      p.p_chunk = (int)(pc > 0 ? pc : 1), p.o_chunk = (int)(oc > 0 ? oc : 1);
    }
    if (c >= p_tiles && c >= o_tiles) break;
  }
  p.p_rt = (int)(p_rt > 0 ? p_rt : 1);
  p.o_rt = (int)(o_rt > 0 ? o_rt : 1);
  p.p_items = p_lists * p.p_splits;
  const int64_t deal = p.p_rt > 1 ? 8 * (int64_t)p.p_rt : 1;
  p.p_grid = (p.p_items + deal - 1) / deal * deal;
  p.grid = p.p_grid + o_lists * p.o_splits;
  if (p.grid > MOST || p.rows * Hkv > MOST * 4) return false;
  p.bytes = (size_t)(p.rows * Hkv * (p.p_splits + p.o_splits)) * (D + 2) * sizeof(float);
  return true;
}

template <typename T, int D>
void launch(const PrefixArgs& a, const Plan& p, hipStream_t st) {
  const dim3 block(64 * WAVES);
  if (p.whole) {
    hipLaunchKernelGGL((prefix_whole_kernel<T, D>), dim3((unsigned)p.grid), block, 0, st, a);
    return;
  }
  if (p.grid > 0) {
    const dim3 grid((unsigned)p.grid);
    if (p.mt == 1) hipLaunchKernelGGL((prefix_rows_kernel<T, D, 1>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((prefix_rows_kernel<T, D, 2>), grid, block, 0, st, a);
  }
  // four splits a group at once, as long as a workgroup has groups
  constexpr int GROUPS = 256 / (D / 4);
  int side = 1;
  while (side < GROUPS && 4 * side < p.p_splits + p.o_splits) side *= 2;
  const int per = GROUPS / side;
  hipLaunchKernelGGL((prefix_join_kernel<T, D>), dim3((unsigned)((p.rows * a.Hkv + per - 1) / per)), dim3(256), 0, st, a, side);
}

template <typename T>
void by_dim(int D, const PrefixArgs& a, const Plan& p, hipStream_t st) {
  if (D == 32) launch<T, 32>(a, p, st);
  else if (D == 64) launch<T, 64>(a, p, st);
  else if (D == 128) launch<T, 128>(a, p, st);
  else launch<T, 256>(a, p, st);
}

// Bytes from key to key: at most 2^25 (a tile's offsets stay inside 32 bits), and a key's
// own at least, also where there is one key: the places of a tile behind the last key lie
// behind that key's end, where loads give zero.
bool key_stride(uint32_t& to, int64_t elements, int keys, int D) {
  if (keys > 1 && (elements < D || elements > 1 << 24)) return false;
  to = (uint32_t)(2 * (keys > 1 ? elements : D));
  return true;
}

}  // namespace
}  // namespace da

using namespace da;

extern "C" size_t da_prefix_attn_workspace_bytes(int B, int P, int Hq, int Hkv, int s, int D, int max_prefix,
                                                 int max_keys) {
  if (B < 1 || P < 1 || B % P != 0 || Hq < 1 || Hkv < 1 || Hq % Hkv != 0 || s < 1 || !head_dim_ok(D) ||
      max_prefix < 0 || max_prefix > MAX_KEYS || max_keys < 0 || max_keys > MAX_KEYS)
    return 0;
  Plan p;
  return plan_for(p, B, P, Hkv, Hq / Hkv, s, D, max_prefix, max_keys) ? p.bytes : 0;
}

extern "C" int da_prefix_attn_fwd(const da_prefix_attn_args* x, void* stream) {
  if (!x) return DA_ERR_INVALID_ARG;
  if (x->dtype != DA_BF16 && x->dtype != DA_FP16) return DA_ERR_DTYPE;
  if (!head_dim_ok(x->D)) return DA_ERR_HEAD_DIM;
  const int B = x->B, P = x->P, Hkv = x->Hkv, Hq = x->Hq, s = x->s, Np = x->max_prefix, cap = x->max_keys;
  if (B < 0 || P < 1 || B % P != 0 || Hkv < 1 || Hq < 1 || Hq % Hkv != 0 || s < 0 || Np < 0 || Np > MAX_KEYS ||
      cap < 0 || cap > MAX_KEYS)
    return DA_ERR_INVALID_ARG;
  if ((!x->n_prefix_dev && (x->n_prefix < 0 || x->n_prefix > Np)) || (!x->n_keys_dev && (x->n_keys < 0 || x->n_keys > cap)))
    return DA_ERR_INVALID_ARG;
  if (!(fabsf(x->sm_scale) <= FLT_MAX)) return DA_ERR_INVALID_ARG;
  if (B == 0 || s == 0) return DA_OK;
  if (!x->q || !x->out || (Np > 0 && (!x->k_prefix || !x->v_prefix)) || (cap > 0 && (!x->k || !x->v)))
    return DA_ERR_INVALID_ARG;
  if ((B > 1 && !x->o_str[0]) || (Hq > 1 && !x->o_str[1]) || (s > 1 && !x->o_str[2])) return DA_ERR_INVALID_ARG;
  if (!aligned16(x->q) || !aligned16(x->out) || !aligned16(x->k_prefix) || !aligned16(x->v_prefix) || !aligned16(x->k) ||
      !aligned16(x->v) || !strides8(x->q_str) || !strides8(x->o_str) || !strides8(x->kp_str) || !strides8(x->vp_str) ||
      !strides8(x->k_str) || !strides8(x->v_str) || ((uintptr_t)x->n_prefix_dev & 3) || ((uintptr_t)x->n_keys_dev & 3))
    return DA_ERR_ALIGNMENT;
  PrefixArgs a{};
  if (!key_stride(a.kp_s, x->kp_str[2], Np, x->D) || !key_stride(a.vp_s, x->vp_str[2], Np, x->D) ||
      !key_stride(a.k_s, x->k_str[2], cap, x->D) || !key_stride(a.v_s, x->v_str[2], cap, x->D))
    return DA_ERR_INVALID_ARG;
  const int G = Hq / Hkv;
  Plan p;
  if (!plan_for(p, B, P, Hkv, G, s, x->D, Np, cap)) return DA_ERR_INVALID_ARG;
  if (p.bytes > 0 && (!x->workspace || x->workspace_bytes < (int64_t)p.bytes)) return DA_ERR_WORKSPACE;
  if (!aligned16(x->workspace)) return DA_ERR_ALIGNMENT;
  a.q = x->q, a.kp = x->k_prefix, a.vp = x->v_prefix, a.k = x->k, a.v = x->v, a.o = x->out;
  a.q_b = x->q_str[0], a.q_h = x->q_str[1], a.q_s = x->q_str[2];
  a.o_b = x->o_str[0], a.o_h = x->o_str[1], a.o_s = x->o_str[2];
  a.kp_b = x->kp_str[0], a.kp_h = x->kp_str[1], a.vp_b = x->vp_str[0], a.vp_h = x->vp_str[1];
  a.k_b = x->k_str[0], a.k_h = x->k_str[1], a.v_b = x->v_str[0], a.v_h = x->v_str[1];
  a.np_dev = x->n_prefix_dev, a.n_dev = x->n_keys_dev;
  a.np_step = x->n_prefix_per ? 1 : 0, a.n_step = x->n_keys_per_seq ? 1 : 0;
  a.np = x->n_prefix, a.n = x->n_keys, a.Np = Np, a.cap = cap;
  a.B = B, a.P = P, a.per = B / P, a.Hkv = Hkv, a.G = G, a.s = s;
  a.rows = (int)p.rows;
  a.p_rows = a.rows / P, a.o_rows = s * G;
  a.p_rt = p.p_rt, a.o_rt = p.o_rt;
  a.p_splits = p.p_splits, a.o_splits = p.o_splits, a.p_chunk = p.p_chunk, a.o_chunk = p.o_chunk;
  a.p_items = (int)p.p_items, a.p_grid = (int)p.p_grid;
  a.heads = make_fastdiv(G), a.rows_s = make_fastdiv(s);
  a.f_prt = make_fastdiv(p.p_rt), a.f_ort = make_fastdiv(p.o_rt);
  a.f_psp = make_fastdiv(p.p_splits > 0 ? p.p_splits : 1), a.f_osp = make_fastdiv(p.o_splits > 0 ? p.o_splits : 1);
  a.f_hkv = make_fastdiv(Hkv), a.f_rows = make_fastdiv(a.rows), a.f_per = make_fastdiv(a.per);
  // (a scale of zero, which weighs every key alike, as the smallest one: a masked
  // score's -inf stays -inf)
  a.scale2 = fminf(fmaxf(fabsf(x->sm_scale) * 1.4426950408889634f, FLT_TRUE_MIN), FLT_MAX);
  a.flip = x->sm_scale < 0.f ? 0x80008000u : 0;
  a.part = (float*)x->workspace;
  a.part_m = a.part + p.rows * Hkv * (p.p_splits + p.o_splits) * x->D;
  a.part_l = a.part_m + p.rows * Hkv * (p.p_splits + p.o_splits);
  (void)hipGetLastError();
  if (x->dtype == DA_BF16) by_dim<__bf16>(x->D, a, p, (hipStream_t)stream);
  else by_dim<_Float16>(x->D, a, p, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? DA_OK : DA_ERR_LAUNCH;
}
