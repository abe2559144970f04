// The next tokens of a batch, drawn from its logits by given random numbers
// (gfx950 / CDNA4).
//
// A row's candidates (logits above -inf that are numbers) are ordered by logit,
// largest first, equal ones by index. With x the logits, m the largest and T the
// temperature, a token weighs w = exp((x - m) / T). What is kept of the order:
//   top_k   the first k
//   top_p   of those the shortest run whose weight reaches p times theirs
//   min_p   of those the tokens with x >= m + T ln(min_p)
// (always the first one), and the token drawn is the first by index at which the
// sum of the kept weights passes u times their total.
//
// A token differs if a border of these sums falls on the other side of p or u
// times a total than it does in exact arithmetic: with 131072 borders a sum that
// is off by 2^-24 would draw other tokens in one row of a hundred. So a weight is
// a 64-bit integer, in units of 2^-45 of the largest one (fewer bits past 2^17
// tokens, so that a row's total fits 63), rounded from a 64-bit exponential.
// Integer sums have no order: a row's token does not depend on how the row is
// split over workgroups, and the products u * total and p * total are exact.
//
// Long rows are split over workgroups ("parts") and take two or three launches:
//   top     each part's largest and smallest candidate, and the largest of each of
//           the row's groups of lanes
//   gather  top_k: the k-th largest of a row's group maxima is no larger than its
//           k-th logit, so the tokens from there on hold the first k and few more:
//           they are gathered in a list. top_p: the weights' histogram over the
//           logits
//   sums    (rows without a list) the kept weight of every tile of 64 vectors;
//           with top_p the tokens of the one bin at which the histogram reaches p
//           are gathered in a list, those of larger logits are kept
// The part that is through last ends its row: the last token kept, from the list;
// the tile at which the sum passes u times the total, and the token in it. Where
// rows fill most CUs, or are short, one workgroup takes a row through the same
// passes in one launch; rows up to a list's length are their own list.
//
// What bounds it. A few rows: the launches and each one's dependent steps (loads of
// what the launch before left, a barrier or two, the last part's join): one row of
// 32000 bfloat16 tokens 12.6 us in two launches, one of 128256 with top_p 20.6 in
// three (4.5 + 5.9 + 11.3 traced). Many rows: a token's weight, 29 instructions of
// the vector ALU (two thirds of them in 64 bits) for 2 bytes read; 192 rows of 100003
// tokens with top_p weigh each token twice: 75 us, 0.5 TB/s. Rows with top_k alone
// weigh no more than their lists: 256 rows of 128256 tokens 38 us, 1.7 TB/s.
#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "capi_common.h"
#include "delta_attn.h"
#include "device_common.h"

namespace da {
namespace {

typedef unsigned __int128 u128;
typedef unsigned long long ull;

constexpr int MAX_V = 1 << 24;               // tokens of a vocabulary
constexpr int MAX_B = 0x3fffff;              // rows (four parts each: threads of a grid below 2^32)
constexpr uint32_t KEY_NONE = 0x007fffffu;   // -inf's key: candidates lie above it
constexpr int PART = 512;                    // threads of a part
constexpr int LIST = 3584;                   // tokens of a row's list (LDS for two workgroups a CU)
constexpr int BINS = 768;                    // of a part's histogram
constexpr int GROUPS = 2048;                 // group maxima of a row (four a thread of a part)
constexpr int SLOTS = 1024;                  // tile sums in LDS

struct Part {
  uint64_t first;                            // the first place in the order, 0: no candidate
  uint32_t low, pad;                         // the smallest candidate's key turned round, 0: no candidate
};

struct SampleArgs {
  const void* x;
  int64_t x_b;
  const float* u;
  const float *t_dev, *p_dev, *m_dev;       // settings of the rows, or NULL: one for all
  const int* k_dev;
  int t_step, k_step, p_step, m_step;       // 1: an entry per row, 0: one for all
  float t, p, m;
  int k;
  int64_t* token;
  float* logp;
  int B, V, bits;                           // weights in units of 2^-bits
  int parts, tiles, k_list;                 // parts of a row, tiles of a part, the largest top_k with a list
  FastDiv f_parts;
  int runs, sums;                           // whether rows may take a histogram, and whether the sums are launched
  int lanes;                                // of a group
  // workspace, by row
  Part* part;                               // [parts]
  uint32_t* maxima;                         // [GROUPS]
  uint32_t* count;                          // tokens gathered (also past the list's end)
  uint32_t* ended;                          // parts that are through
  uint64_t* hist;                           // [BINS]
  uint64_t* list;                           // [LIST] places
  uint64_t* tile;                           // [parts * tiles] kept weight
};

// A number's place in the order of floats (-0 beside 0); NaN last.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0u : (int)b < 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// A token's place in the order: larger is earlier, 0 is no candidate. The key's bits
// that the type uses, above the index turned round.
template <typename T>
struct Order {
  // low bits of a key that are alike in all of the type's numbers of one sign
  static constexpr int SPARE = sizeof(T) == 4 ? 0 : std::is_same_v<T, __bf16> ? 16 : 13;
  int bits;                                 // of an index
  __device__ __forceinline__ explicit Order(int V) : bits(V > 1 ? 32 - __clz(V - 1) : 1) {}
  __device__ __forceinline__ uint32_t turned(int i) const { return ~(uint32_t)i & ((1u << bits) - 1); }
  __device__ __forceinline__ uint64_t place(uint32_t key, int i) const {
    return key > KEY_NONE ? (uint64_t)(key >> SPARE) << bits | turned(i) : 0;
  }
  __device__ __forceinline__ int index(uint64_t place) const { return (int)turned((int)place); }
  __device__ __forceinline__ float logit(uint64_t place) const {
    const uint32_t k = (uint32_t)(place >> bits) << SPARE;
    return of_key(k >> 31 ? k : k | ((1u << SPARE) - 1));
  }
};

// Weights in units of 2^-bits (bits <= 45) of one that is 1: 2^(d * per) for d <= 0, the
// fraction's power by the polynomial of degree 10 that meets 2^f at the Chebyshev nodes
// of [-1/2, 1/2] (2^-51 of it, rounding included; the series takes two terms more), the
// whole one by the exponent. Whole numbers come from what 2^52 leaves of a sum: of the
// exponent, with the unit's `bits` above it, and of the weight, which is rounded so.
// (RAW is that 2^52 of the weight, for the sums to take off together.) A tile's weights
// are bound by these instructions: with the exponent and the units put in apart, and the
// weight's 2^52 taken off one by one, 33 for 29 (192 rows of temperature alone 48 us for
// 46). By count, tables of powers in LDS would save less than their gathers cost.
constexpr double WHOLE_OF = 6755399441055744.0;   // 1.5 * 2^52
constexpr uint64_t RAW = 0x4330000000000000ull;
__device__ __forceinline__ uint64_t raw_weight(double d, double per, double whole_of) {
  const double whole = fma(d, per, whole_of), f = fma(d, per, whole_of - whole);
  double p = 7.072585949269223e-09;
  constexpr double c[] = {1.0208690299958306e-07, 1.321544258792169e-06, 1.5252657260200837e-05, 0.0001540353044173605,
                          0.0013333558230164974, 0.009618129107606888, 0.05550410866444772, 0.24022650695910097,
                          0.69314718055995, 1.0};
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    double k = c[i];
    asm("" : "+s"(k));                      // (a scalar operand: else each term copies it first)
    p = fma(p, f, k);
  }
  const uint64_t w = (uint64_t)__double_as_longlong(p);
  uint32_t hi = (uint32_t)(w >> 32) + ((uint32_t)__double_as_longlong(whole) << 20);
  asm("" : "+v"(hi));                       // (32 bits of it: else the sum takes 64)
  const double scaled = __longlong_as_double((long long)((uint64_t)hi << 32 | (uint32_t)w));
  return (uint64_t)__double_as_longlong(scaled + 4503599627370496.0);
}

// What a row asks for.
struct Setting {
  float t, p, m;
  int k;
  bool greedy, cut, list, run;              // cut: top_k takes some away; list: by a list; run: top_p takes some away
};
__device__ __forceinline__ Setting setting_of(const SampleArgs& a, int b) {
  Setting s;
  s.t = a.t_dev ? a.t_dev[b * a.t_step] : a.t;
  s.k = a.k_dev ? a.k_dev[b * a.k_step] : a.k;
  s.p = a.p_dev ? a.p_dev[b * a.p_step] : a.p;
  s.m = a.m_dev ? a.m_dev[b * a.m_step] : a.m;
  s.greedy = !(s.t > 0.f) || s.m > 1.f;     // (a min_p above 1 leaves the first token alone)
  s.cut = s.k > 0 && s.k < a.V;
  s.list = !s.greedy && s.cut && s.k <= a.k_list;
  s.run = s.p < 1.f;
  return s;
}

// The weights of a row with a candidate, and the bins of its histogram: linear in
// the logit, from the largest to where weights vanish or the smallest candidate.
struct Scale {
  double top, per, none, whole_of;          // none: a distance from the top of no weight
  float topf, half, step, bar;              // half of the top; bins a half; bar: min_p's, the smallest float at or above it
  bool inf;                                 // an infinite largest logit: the tokens at it share the row
  __device__ __forceinline__ Scale(const SampleArgs& a, const Setting& s, float most, uint32_t least) {
    topf = most;
    inf = topf == INFINITY;
    per = fmax(1.44269504088896340736 / (double)s.t, 0x1p-300);   // (an infinite temperature: all weigh 1)
    none = -200.0 / per;
    whole_of = WHOLE_OF + a.bits;
    bar = -INFINITY;
    if (s.m > 0.f) {
      double y = s.m < 1.f ? (double)topf + (double)s.t * log((double)s.m) : (double)topf;
      if (y != y) y = topf;                 // (an infinite logit at an infinite temperature)
      bar = (float)y;
      if ((double)bar < y) bar = of_key(key_of(bar) + 1);
    }
    bar = inf ? 0.f : fmaxf(bar, -FLT_MAX);   // (candidates alone pass it)
    if (inf) topf = 0.f;
    top = topf;
    const double far = a.bits + 2, all = (top - (inf ? 0.0 : (double)of_key(least))) * per;
    const double range = all < far ? all : far;
    half = 0.5f * topf;
    step = range > 0.0 ? (float)fmin(2 * BINS * (1.0 - 1.0 / 1024) / range * per, (double)FLT_MAX) : 0.f;
  }
  // logits as the rest takes them, and the bar
  __device__ __forceinline__ float at(float y) const { return !inf ? y : y == INFINITY ? 0.f : -INFINITY; }
  __device__ __forceinline__ uint64_t raw(float z) const { return raw_weight(fmax((double)z - top, none), per, whole_of); }
  __device__ __forceinline__ uint64_t weight(float z) const { return raw(z) - RAW; }
  // Its whole part is the bin; BINS: no weight. (Half the distance: the type's largest and
  // lowest numbers are further apart than a float.)
  __device__ __forceinline__ float bin(float z) const { return fminf(fmaf(z, -0.5f, half) * step, (float)BINS); }
  // The smallest logit of the bins before `end` (1 to BINS), found by a wave: each lane
  // tries one of 64 keys of what is left. (Borders as logits cost the sums one comparison
  // a token, bins four instructions.)
  __device__ __forceinline__ float low_end(int end) const {
    uint32_t lo = KEY_NONE + 1, hi = key_of(topf);   // (the bins are of falling logits, the top in the first)
    while (lo < hi) {
      const uint32_t stride = (hi - lo) / 64 + 1, off = (threadIdx.x % 64) * stride;
      const uint64_t in = __ballot(bin(of_key(off < hi - lo ? lo + off : hi)) < (float)end);   // (from some lane on)
      const uint32_t n = in ? __ffsll((long long)in) - 1 : 64;
      if (n < 64 && n * stride < hi - lo) hi = lo + n * stride;
      if (n > 0) lo += (n - 1) * stride + 1;
    }
    return of_key(hi);
  }
  template <int E>
  __device__ __forceinline__ void at(const float (&y)[E], float (&z)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) z[e] = y[e];
    if (inf) {
#pragma unroll
      for (int e = 0; e < E; ++e) z[e] = at(y[e]);
    }
  }
  // All of a vector's, whatever becomes of them: their chains of 64-bit operations
  // run beside each other.
  template <int E>
  __device__ __forceinline__ void raws(const float (&z)[E], uint64_t (&w)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = raw(z[e]);
#pragma unroll
    for (int e = 0; e < E; ++e) asm("" : "+v"(w[e]));
  }
};

// A row as 16-byte vectors from the aligned address at or before its start; what
// lies outside the row counts as -inf.
template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const u32x4* base;
  int shift, V, n_vec;
  __device__ __forceinline__ Row(const SampleArgs& a, int b) {
    const T* p = (const T*)a.x + (int64_t)b * a.x_b;
    shift = (int)((uintptr_t)p & 15) / sizeof(T);
    base = (const u32x4*)(p - shift);
    V = a.V;
    n_vec = (V + shift + E - 1) / E;
  }
  __device__ __forceinline__ int index(int v, int e) const { return v * E + e - shift; }
  __device__ __forceinline__ u32x4 load(int v) const { return base[min(v, n_vec - 1)]; }
  __device__ __forceinline__ void unpack(u32x4 w, int v, float (&y)[E]) const {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (sizeof(T) == 4) y[e] = __uint_as_float(w[e]);
      else y[e] = e % 2 ? Elt<T>::hi(w[e / 2]) : Elt<T>::lo(w[e / 2]);
    }
    if (v == 0 || v >= n_vec - 1) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = index(v, e);
        y[e] = i >= 0 && i < V && v < n_vec ? y[e] : -INFINITY;
      }
    }
  }
  // f(logit, index) of each of the vector's candidates and others
  template <typename F>
  __device__ __forceinline__ void each(int v, F&& f) const {
    float y[E];
    unpack(load(v), v, y);
#pragma unroll
    for (int e = 0; e < E; ++e) f(y[e], index(v, e));
  }
};

// This lane's vectors of `tiles` tiles from tile0 on, wave w of W every W-th tile, U
// loads ahead: those of the first vectors are made here. None is made past the wave's
// own tiles (64 mixed rows of 151936 tokens 52 -> 47 us).
template <typename T, int W, int U>
struct Sweep {
  using R = Row<T>;
  static constexpr int WAVES = W;
  const R& row;
  int first, n;
  u32x4 w[U];
  __device__ __forceinline__ Sweep(const R& r, int tile0, int tiles) : row(r) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    first = tile0 + wave;
    n = min(tiles - wave, (r.n_vec + 63) / 64 - first);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u * W < n) w[u] = row.load(vector(u * W));
  }
  __device__ __forceinline__ int vector(int j) const { return (first + j) * 64 + (int)(threadIdx.x % 64); }
  template <typename F>
  __device__ __forceinline__ void run(F&& f) {   // f(vector, logits)
    for (int j = 0; j < n; j += U * W) {
      u32x4 now[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        now[u] = w[u];
        if (j + (U + u) * W < n) w[u] = row.load(vector(j + (U + u) * W));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j + u * W >= n) break;
        float y[R::E];
        row.unpack(now[u], vector(j + u * W), y);
        f(vector(j + u * W), y);
      }
    }
  }
};

// op over the lanes up to this one, with 0 beside them.
template <typename F>
__device__ __forceinline__ uint64_t lanes_upto(uint64_t x, F&& op) {
  auto step = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
    constexpr int C = decltype(ctrl)::value, R = decltype(rows)::value;
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, C, R, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), C, R, 0xf, false);
    x = op(x, (uint64_t)hi << 32 | lo);
  };
  using std::integral_constant;
  step(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});   // row_shr 1, 2, 4, 8
  step(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  step(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});   // across the rows of 16
  step(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return x;
}
struct Most {
  __device__ __forceinline__ uint64_t operator()(uint64_t p, uint64_t q) const { return p > q ? p : q; }
};
struct Plus {
  __device__ __forceinline__ uint64_t operator()(uint64_t p, uint64_t q) const { return p + q; }
};
__device__ __forceinline__ uint64_t scan64(uint64_t x) { return lanes_upto(x, Plus()); }
__device__ __forceinline__ uint64_t last_lane(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(x >> 32), 63) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((uint32_t)x, 63);
}
template <typename F>
__device__ __forceinline__ uint64_t wave_all(uint64_t x, F&& op) { return last_lane(lanes_upto(x, op)); }

// op over the workgroup's N threads (0 beside them). s: N / 64 words.
template <int N, typename F>
__device__ __forceinline__ uint64_t block_all(uint64_t v, uint64_t* s, F&& op) {
  v = lanes_upto(v, op);
  __syncthreads();
  if (threadIdx.x % 64 == 63) s[threadIdx.x / 64] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < N / 64; ++w) v = op(v, s[w]);
  return v;
}

// Sums of the threads before this one; `total` of all.
template <int N>
__device__ __forceinline__ uint64_t block_before(uint64_t v, uint64_t* s, uint64_t& total) {
  const uint64_t upto = scan64(v);
  __syncthreads();
  if (threadIdx.x % 64 == 63) s[threadIdx.x / 64] = upto;
  __syncthreads();
  uint64_t before = upto - v;
  total = 0;
#pragma unroll
  for (int w = 0; w < N / 64; ++w) {
    if (w < (int)threadIdx.x / 64) before += s[w];
    total += s[w];
  }
  return before;
}

// ceil or floor of f * total for 0 <= f < 1, exactly.
__device__ __forceinline__ uint64_t part_of(float f, uint64_t total, bool up) {
  const uint32_t b = __float_as_uint(f);
  if (f != f || (int)b <= 0) return 0;
  const int e = b >> 23;                    // f = mant * 2^(e - 150)
  const uint32_t mant = e ? (b & 0x7fffff) | 0x800000 : b & 0x7fffff;
  const int shift = 150 - (e ? e : 1);
  if (shift > 120) return up && total ? 1 : 0;
  if (shift < 24) return total;             // (1 and above)
  const u128 y = (u128)mant * total;
  return (uint64_t)((y + (up ? ((u128)1 << shift) - 1 : 0)) >> shift);
}

// ---------------------------------------------------------------------------
// The passes over a row, or a part of one.

// This thread's largest number, the vector that held it first, and (want) its
// smallest candidate. group: the largest of its G groups of vectors (G tiles take turns).
template <int G, typename S>
__device__ __forceinline__ void ends_of(S& sweep, bool want, float& most, int& at, float& least, float (&group)[G]) {
  constexpr int E = S::R::E;
  most = -INFINITY, least = INFINITY, at = 0;
#pragma unroll
  for (int g = 0; g < G; ++g) group[g] = -INFINITY;
  sweep.run([&](int v, const float (&y)[E]) __attribute__((always_inline)) {
    float top = y[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, y[e]);   // (a NaN gives way)
    if (want) {
#pragma unroll
      for (int e = 0; e < E; ++e) least = fminf(least, y[e] > -INFINITY ? y[e] : INFINITY);
    }
    if (top > most) {
      most = top;
      at = v;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) group[g] = fmaxf(group[g], v / (64 * S::WAVES) % G == g ? top : -INFINITY);
  });
}
// Its first place and its smallest candidate's key turned round (0: no candidate).
template <typename T>
__device__ __forceinline__ void ends_of(const Row<T>& row, const Order<T>& ord, float most, int at, float least,
                                        uint64_t& first, uint32_t& low) {
  const uint32_t key = key_of(most);
  first = 0;
  if (key > KEY_NONE)
    row.each(at, [&](float y, int i) __attribute__((always_inline)) {
      if (first == 0 && key_of(y) == key) first = ord.place(key, i);
    });
  low = least < INFINITY ? ~key_of(least) : key > KEY_NONE ? ~key : 0u;
}

// A number that fewer than k of the groups' maxima's first 16 bits pass: the
// largest one of 16 bits that is no larger than the k-th largest maximum, two bits at a
// time, by the counts of maxima that reach it, the workgroup's together. (By one wave for
// all maxima, a bit at a time without barriers, top_k 700 took 25 us for 21.) key: the
// thread's maxima. s: 24 words.
template <int N>
__device__ __forceinline__ float list_bar(const uint32_t (&key)[GROUPS / N], int k, uint32_t* s) {
  const int lane = threadIdx.x % 64;
  if (threadIdx.x < 24) s[threadIdx.x] = 0;
  __syncthreads();
  uint32_t low = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) {
    const int bit = 14 - 2 * r;
    int n[3] = {};
#pragma unroll
    for (int j = 0; j < 3; ++j)
#pragma unroll
      for (int i = 0; i < GROUPS / N; ++i) n[j] += __popcll(__ballot(key[i] >> 16 >= (low | (j + 1) << bit)));
    if (lane < 3) atomicAdd(&s[3 * r + lane], (uint32_t)(lane == 0 ? n[0] : lane == 1 ? n[1] : n[2]));
    __syncthreads();
    low |= ((s[3 * r] >= (uint32_t)k) + (s[3 * r + 1] >= (uint32_t)k) + (s[3 * r + 2] >= (uint32_t)k)) << bit;
  }
  return of_key(max(low << 16, KEY_NONE + 1));
}

// The places of the logits from `bar` on; n counts them (also past the list's end).
template <typename S, typename O>
__device__ __forceinline__ void gather_into(S& sweep, const O& ord, float bar, uint64_t* list, uint32_t* n) {
  constexpr int E = S::R::E;
  sweep.run([&](int v, const float (&y)[E]) __attribute__((always_inline)) {
    float top = y[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, y[e]);
    if (!(top >= bar)) return;              // (most vectors)
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (y[e] >= bar) {
        const uint32_t at = atomicAdd(n, 1u);
        if (at < LIST) list[at] = ord.place(key_of(y[e]), sweep.row.index(v, e));
      }
  });
}

// The weights' histogram. (Its additions in LDS take a fifth of a flat row's time, 18 of
// 96 us for 192 rows; in 32 bits, or with the waves' priorities apart, they take as long.)
template <typename S>
__device__ __forceinline__ void hist_into(S& sweep, const Scale& sc, uint64_t* hist) {
  constexpr int E = S::R::E;
  sweep.run([&](int, const float (&y)[E]) __attribute__((always_inline)) {
    float z[E];
    uint64_t w[E];
    sc.at(y, z);
    sc.raws(z, w);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float at = sc.bin(z[e]);
      if (at < (float)BINS) atomicAdd((ull*)&hist[(int)at], (ull)(w[e] - RAW));
    }
  });
}

// The bin of a row's last place kept: what lies above it is kept whole.
struct Border {
  float low, above;                         // its smallest logit, and the smallest above it
  // (none: the row is kept whole)
  __device__ __forceinline__ Border() : low(-INFINITY), above(-INFINITY) {}
  // (two waves find an end each. s: two words)
  __device__ __forceinline__ Border(const Scale& sc, int bin, uint64_t* s) {
    const int wave = threadIdx.x / 64;
    float* ends = (float*)s;
    __syncthreads();
    if (wave < 2) {
      const float end = wave == 0 ? sc.low_end(bin + 1) : bin > 0 ? sc.low_end(bin) : INFINITY;
      if (threadIdx.x % 64 == 0) ends[wave] = end;
    }
    __syncthreads();
    low = ends[0], above = ends[1];
  }
};

// put(tile, kept weight) of what lies above the border; the border's go to the list.
template <typename S, typename O, typename P>
__device__ __forceinline__ void sums_into(S& sweep, const O& ord, const Scale& sc, const Border& border, uint64_t* list,
                                          uint32_t* n, P&& put) {
  constexpr int E = S::R::E;
  const float from = fmaxf(border.above, sc.bar);
  sweep.run([&](int v, const float (&y)[E]) __attribute__((always_inline)) {
    float z[E], most;
    sc.at(y, z);
    most = z[0];
#pragma unroll
    for (int e = 1; e < E; ++e) most = fmaxf(most, z[e]);
    uint64_t sum = 0;
    if (__any(most >= from)) {
      float kept[E];
      uint64_t w[E];
#pragma unroll
      for (int e = 0; e < E; ++e) kept[e] = z[e] >= from ? z[e] : -INFINITY;
      sc.raws(kept, w);
#pragma unroll
      for (int e = 0; e < E; ++e) sum += w[e];
      sum = last_lane(scan64(sum - E * RAW));
    }
    if (threadIdx.x % 64 == 0) put(v / 64, sum);
    if (border.low < border.above && most >= border.low) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (z[e] >= border.low && z[e] < border.above) {
          const uint32_t i = atomicAdd(n, 1u);
          if (i < LIST) list[i] = ord.place(key_of(y[e]), sweep.row.index(v, e));
        }
    }
  });
}

// The bin at which a row's histogram reaches p times its total, the weight of
// those before it and what is to be reached.
template <int N>
__device__ __forceinline__ int border_bin(const uint64_t* hist, float p, uint64_t* s, uint64_t& before, uint64_t& goal) {
  constexpr int PER = BINS / 256;           // bins of a thread
  static_assert(BINS % 256 == 0 && N >= 256, "256 threads hold the bins");
  uint64_t sum[PER] = {}, mine = 0, total;
  if (threadIdx.x < 256) {
    const uint64_t* h = hist + threadIdx.x * PER;
#pragma unroll
    for (int e = 0; e < PER; ++e) sum[e] = h[e];
#pragma unroll
    for (int e = 0; e < PER; ++e) mine += sum[e];
  }
  uint64_t upto = block_before<N>(mine, s, total);
  goal = part_of(p, total, true);
  if (goal < 1) goal = 1;
  __syncthreads();
  if (upto < goal && upto + mine >= goal) {
    int e = 0;
#pragma unroll
    for (int i = 0; i < PER - 1; ++i)
      if (e == i && upto + sum[i] < goal) {
        upto += sum[i];
        e = i + 1;
      }
    s[0] = threadIdx.x * PER + e;
    s[1] = upto;
  }
  __syncthreads();
  before = s[1];
  return (int)s[0];
}

// Values with a measure: narrows [lo, hi] (lo >= 1) towards the largest value at which
// the measure, summed from the largest value down, reaches `goal` (then the rest of
// it), until no more than `few` values are left or one place. -> how many are left, 0
// if none reaches it. Nine or ten bits of the range at a time, by histograms of N bins.
// each(f) calls f(value, measure) for the thread's values. s: reach_words(N).
constexpr int reach_words(int N) { return 3 * N + 64; }
template <int N, typename F>
__device__ __forceinline__ uint32_t narrow(F&& each, uint64_t& lo, uint64_t& hi, uint64_t& goal, uint32_t few, uint64_t* s) {
  constexpr int LOG = N == 1024 ? 10 : 9;
  static_assert(N == 1 << LOG, "a bin a thread");
  const int tid = threadIdx.x, wave = tid / 64;
  uint64_t* s_scan = s + 3 * N;
  __syncthreads();
  s[tid] = 0;
  ((uint32_t*)(s + 2 * N))[tid] = 0;
  if (tid < 3) s_scan[32 + 4 * tid] = 0;    // (the third: reach's count)
  __syncthreads();
  for (int pass = 0; ; ++pass) {
    // the two passes' places take turns: what one leaves is cleared by the next
    uint64_t *bin = s + pass % 2 * N, *sums = s_scan + pass % 2 * 16, *found = s_scan + 32 + pass % 2 * 4;
    uint32_t* cnt = (uint32_t*)(s + 2 * N) + pass % 2 * N;
    const int bits = 64 - __clzll((long long)((hi - lo) | 1)), shift = bits > LOG ? bits - LOG : 0;
    each([&](uint64_t x, uint64_t measure) __attribute__((always_inline)) {
      if (x >= lo && x <= hi) {
        const int at = (int)((x - lo) >> shift);
        atomicAdd((ull*)&bin[at], (ull)measure);
        atomicAdd(&cnt[at], 1u);
      }
    });
    __syncthreads();
    const uint64_t mine = bin[N - 1 - tid], upto = scan64(mine);
    const uint32_t many = cnt[N - 1 - tid];
    if (tid % 64 == 63) sums[wave] = upto;
    s[(pass + 1) % 2 * N + tid] = 0;
    ((uint32_t*)(s + 2 * N))[(pass + 1) % 2 * N + tid] = 0;
    __syncthreads();
    uint64_t before = upto - mine;
#pragma unroll
    for (int w = 0; w < N / 64; ++w) before += w < wave ? sums[w] : 0;
    if (before < goal && before + mine >= goal) {
      found[0] = N - tid;                   // the bin and 1
      found[1] = before;
      found[2] = many;
    }
    if (tid == 0) s_scan[32 + (pass + 1) % 2 * 4] = 0;
    __syncthreads();
    if (found[0] == 0) return 0;
    goal -= found[1];
    lo += (found[0] - 1) << shift;
    if ((hi - lo) >> shift) hi = lo + ((uint64_t)1 << shift) - 1;
    if (shift == 0 || found[2] <= few) return (uint32_t)found[2];
  }
}

// The largest of n values from [lo, hi] at which the measure, summed from the largest
// down, reaches `goal`; 0 if none does. Each wave ends by itself what a lane a value is
// left of.
template <int N, typename V, typename M>
__device__ __forceinline__ uint64_t reach(int n, V&& value, M&& measure, uint64_t lo, uint64_t hi, uint64_t goal, uint64_t* s) {
  const uint32_t left = narrow<N>([&](auto&& f) __attribute__((always_inline)) {
    for (int i = threadIdx.x; i < n; i += N) f(value(i), measure(i));
  }, lo, hi, goal, 64, s);
  if (left == 0 || lo == hi) return left ? lo : 0;
  uint32_t* count = (uint32_t*)(s + 3 * N + 40);
  for (int i = threadIdx.x; i < n; i += N) {
    const uint64_t x = value(i);
    if (x >= lo && x <= hi) {
      const uint32_t at = atomicAdd(count, 1u);
      s[at] = x;                              // (the first histogram's place: 64 of them and their measures)
      s[64 + at] = measure(i);
    }
  }
  __syncthreads();
  const uint32_t lane = threadIdx.x % 64;
  const uint64_t mine = lane < left ? s[lane] : 0, weight = lane < left ? s[64 + lane] : 0;
  uint64_t before = 0;
  for (uint32_t j = 0; j < left; ++j) before += s[j] > mine ? s[64 + j] : 0;
  const uint64_t at = __ballot(lane < left && before < goal && before + weight >= goal);
  return at ? s[__ffsll((long long)at) - 1] : 0;
}

// A row's first place and smallest candidate's key, from its parts'.
__device__ __forceinline__ void row_ends(const SampleArgs& a, int b, uint64_t& first, uint32_t& least) {
  const Part* p = a.part + (int64_t)b * a.parts;
  uint32_t low = 0;
  first = 0;
  for (int i = threadIdx.x % 64; i < a.parts; i += 64) {
    first = p[i].first > first ? p[i].first : first;
    low = max(low, p[i].low);
  }
  first = wave_all(first, Most());
  least = ~(uint32_t)wave_all(low, Most());
}

// A short list's n <= FEW values by pairs, N / FEW threads a value: how many are larger
// than this thread's, and their weight. One pass and no barrier for each border, where
// histograms take one or two with three barriers each: 8 rows with top_k 50 19.4 -> 16.0
// us. (Up to 256 values it is slower: top_k 150 17 -> 23 us.)
constexpr int FEW = 128;
template <int N, typename V>
__device__ __forceinline__ void above(int n, V&& value, const uint64_t* w, uint64_t mine, uint32_t& many, uint64_t& weight) {
  constexpr int Q = N / FEW;
  many = 0, weight = 0;
#pragma unroll 4
  for (int j = threadIdx.x % Q; j < n; j += Q) {
    const bool larger = value(j) > mine;
    many += larger;
    weight += larger ? w[j] : 0;
  }
#pragma unroll
  for (int d = 1; d < Q; d *= 2) {
    many += __shfl_xor((int)many, d);
    weight += (uint64_t)__shfl_xor((long long)weight, d);
  }
}

// ---------------------------------------------------------------------------
// The end of a row: a workgroup draws its token.
enum { SHORT, PARTS, WHOLE };               // a short row, one whose parts are through, a long one by a single workgroup
__host__ __device__ constexpr int threads_of(int mode) { return mode == WHOLE ? 1024 : mode == PARTS ? PART : 512; }

template <int MODE>
struct Room {
  static constexpr int N = threads_of(MODE);
  uint64_t list[LIST], w[LIST], slot[MODE == SHORT ? 1 : SLOTS], scan[reach_words(N)], found[2];
  uint64_t hist[MODE == WHOLE ? BINS : 1];
  uint32_t count[MODE == SHORT ? 1 : 24], n, at;
};

// A word for a workgroup of the same launch, or of one.
template <typename W>
__device__ __forceinline__ void put(W* p, W w) { __hip_atomic_store(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename W>
__device__ __forceinline__ W got(const W* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// A row without a candidate, and one of its first token alone.
__device__ __forceinline__ void put_first(const SampleArgs& a, int b, uint64_t first, int index) {
  if (threadIdx.x > 0) return;
  a.token[b] = first ? index : 0;
  a.logp[b] = first ? 0.f : __builtin_nanf("");
}

// What is known of a row: its border, if the kept weight of the tiles was summed, with
// what the border's bin is to reach. n_cand: the tokens of its list.
template <int MODE, typename T>
__device__ __forceinline__ void finish(const SampleArgs& a, int b, const Setting& s, const Row<T>& row, const Order<T>& ord,
                                       uint64_t first, const Scale& sc, Border border, uint64_t goal, uint32_t n_cand,
                                       Room<MODE>& m) {
  using R = Row<T>;
  constexpr int N = threads_of(MODE);
  const int tid = threadIdx.x, lane = tid % 64;
  const int tiles = (row.n_vec + 63) / 64, per = (tiles + SLOTS - 1) / SLOTS;   // tiles of a slot
  const float u = a.u[b];
  // (loads that may turn out to be of nothing, made before it is known)
  const uint64_t *sums = a.tile + (int64_t)b * a.parts * a.tiles, *listed = a.list + (int64_t)b * LIST;
  uint64_t early_sum = 0, early_place = 0;
  if constexpr (MODE == PARTS) {
    early_sum = got(sums + min(tid, a.parts * a.tiles - 1));
    early_place = got(listed + tid);
  }
  auto weight = [&](uint64_t place) __attribute__((always_inline)) { return sc.weight(sc.at(ord.logit(place))); };
  auto drawn = [&](float y, int i, uint64_t total) __attribute__((always_inline)) {
    const double d = ((double)sc.at(y) - sc.top) / (double)s.t;
    a.token[b] = i;
    a.logp[b] = (float)(d - log(ldexp((double)total, -a.bits)));
  };
  auto aim_of = [&](uint64_t total) __attribute__((always_inline)) {
    const uint64_t aim = part_of(u, total, false);
    return aim < total ? aim : total - 1;
  };

  // a list that holds all that is kept?
  const bool whole = MODE == SHORT || (s.list && n_cand <= LIST);
  if (whole) {
    const int n = MODE == SHORT ? a.V : (int)n_cand;
    uint64_t most_off = 0;
    for (int i = tid; i < n; i += N) {
      const uint64_t place = MODE != PARTS ? m.list[i] : i == tid ? early_place : got(listed + i);
      if constexpr (MODE == PARTS) m.list[i] = place;
      m.w[i] = place ? weight(place) : 0;
      most_off = ~place > most_off && place ? ~place : most_off;
    }
    if (n <= FEW) {
      constexpr int Q = N / FEW;
      __syncthreads();
      const int i = tid / Q;
      const uint64_t place = i < n ? m.list[i] : 0, w = i < n ? m.w[i] : 0;
      uint32_t rank;
      uint64_t sum;
      above<N>(n, [&](int j) { return m.list[j]; }, m.w, place, rank, sum);
      bool kept = place && (!s.cut || rank < (uint32_t)s.k);
      if (s.run) {
        const uint64_t goal = part_of(s.p, block_all<N>(tid % Q == 0 && kept ? w : 0, m.scan, Plus()), true);
        kept = kept && (sum < goal || rank == 0);
      }
      kept = kept && sc.at(ord.logit(place)) >= sc.bar;
      const uint64_t total = block_all<N>(tid % Q == 0 && kept ? w : 0, m.scan, Plus()), aim = aim_of(total);
      if (tid % Q == 0 && i < n) m.w[i] = kept ? w : 0;
      __syncthreads();
      auto turned = [&](uint64_t place) { return ord.turned(ord.index(place)); };   // (the first index is the largest)
      above<N>(n, [&](int j) { return turned(m.list[j]); }, m.w, turned(place), rank, sum);
      if (tid % Q == 0 && kept && sum <= aim && sum + w > aim) drawn(ord.logit(place), ord.index(place), total);
      return;
    }
    const uint64_t least_place = ~block_all<N>(most_off, m.scan, Most());
    auto place = [&](int i) __attribute__((always_inline)) { return m.list[i]; };
    auto total_of = [&](auto&& kept) __attribute__((always_inline)) {
      uint64_t sum = 0;
      for (int i = tid; i < n; i += N) sum += kept(i) ? m.w[i] : 0;
      return block_all<N>(sum, m.scan, Plus());
    };
    uint64_t last = 1;                      // the last place kept
    if (s.cut) {
      const uint64_t at = reach<N>(n, place, [](int) { return (uint64_t)1; }, least_place, first, s.k, m.scan);
      if (at) last = at;                    // (0: there are fewer)
    }
    if (s.run) {
      const uint64_t goal = part_of(s.p, total_of([&](int i) { return m.list[i] >= last; }), true);
      last = goal <= 1 ? first : reach<N>(n, place, [&](int i) { return m.w[i]; }, last > 1 ? last : least_place, first, goal, m.scan);
    }
    auto kept = [&](int i) __attribute__((always_inline)) { return m.list[i] >= last && sc.at(ord.logit(m.list[i])) >= sc.bar; };
    const uint64_t total = total_of(kept), aim = aim_of(total);
    // by index: the first one is the largest number
    auto turned = [&](int i) __attribute__((always_inline)) { return kept(i) ? (uint64_t)ord.turned(ord.index(m.list[i])) + 1 : 0; };
    const uint64_t at = reach<N>(n, turned, [&](int i) { return m.w[i]; }, 1, (uint64_t)ord.turned(0) + 1, aim + 1, m.scan);
    for (int i = tid; i < n; i += N)
      if (turned(i) == at) drawn(ord.logit(m.list[i]), ord.index(m.list[i]), total);
    return;
  }
  if constexpr (MODE != SHORT) {

  uint64_t last = 1;                        // the last place kept
  const bool ready = !s.cut && (!s.run || n_cand <= LIST);   // by the passes before
  if (MODE == PARTS || !ready) {
    for (int i = tid; i < SLOTS; i += N) m.slot[i] = 0;
    __syncthreads();
  }
  if (ready) {
    if (s.run) {
      const int n = (int)n_cand;
      uint64_t least_off = 0, most = 0;
      for (int i = tid; i < n; i += N) {
        const uint64_t place = MODE != PARTS ? m.list[i] : i == tid ? early_place : got(listed + i);
        if constexpr (MODE == PARTS) m.list[i] = place;
        m.w[i] = weight(place);
        least_off = ~place > least_off ? ~place : least_off;
        most = place > most ? place : most;
      }
      if (n <= FEW) {
        constexpr int Q = N / FEW;
        if (tid == 0) m.found[0] = 0;
        __syncthreads();
        const int i = tid / Q;
        const uint64_t place = i < n ? m.list[i] : 0, w = i < n ? m.w[i] : 0;
        uint32_t rank;
        uint64_t sum;
        above<N>(n, [&](int j) { return m.list[j]; }, m.w, place, rank, sum);
        if (tid % Q == 0 && sum < goal && sum + w >= goal) m.found[0] = place;
        __syncthreads();
        last = m.found[0];
      } else {
        least_off = block_all<N>(least_off, m.scan, Most());
        most = block_all<N>(most, m.scan, Most());
        last = reach<N>(n, [&](int i) { return m.list[i]; }, [&](int i) { return m.w[i]; }, ~least_off, most, goal, m.scan);
      }
      for (int i = tid; i < n; i += N)
        if (m.list[i] >= last && sc.at(ord.logit(m.list[i])) >= sc.bar)
          atomicAdd((ull*)&m.slot[(ord.index(m.list[i]) + row.shift) / R::E / 64 / per], (ull)m.w[i]);
    }
    if constexpr (MODE == PARTS) {
      for (int i = tid; i < tiles; i += N) {
        const uint64_t w = i == tid ? early_sum : got(sums + i);
        if (w) atomicAdd((ull*)&m.slot[i / per], (ull)w);
      }
    }
    __syncthreads();
  } else {
    // What the lists do not hold (a top_k past k_list, more than LIST tokens at a
    // border): the border place by passes over the whole row, until a list holds what
    // is left.
    auto over = [&](auto&& f) {
      for (int v = tid; v < row.n_vec; v += N) row.each(v, f);
    };
    auto far = [&](auto&& measure, uint64_t goal) {   // 0: nothing reaches it
      uint64_t lo = last, hi = first;
      const uint32_t left = narrow<N>([&](auto&& f) {
        over([&](float y, int i) __attribute__((always_inline)) {
          const uint64_t place = ord.place(key_of(y), i);
          if (place >= lo && place <= hi) f(place, measure(y));
        });
      }, lo, hi, goal, LIST, m.scan);
      if (left == 0 || lo == hi) return left ? lo : 0;
      if (tid == 0) m.n = 0;
      __syncthreads();
      over([&](float y, int i) __attribute__((always_inline)) {
        const uint64_t place = ord.place(key_of(y), i);
        if (place >= lo && place <= hi) {
          const uint32_t at = atomicAdd(&m.n, 1u);
          if (at < LIST) {
            m.list[at] = place;
            m.w[at] = measure(y);
          }
        }
      });
      __syncthreads();
      return reach<N>((int)left, [&](int i) { return m.list[i]; }, [&](int i) { return m.w[i]; }, lo, hi, goal, m.scan);
    };
    auto mass = [&](float y) __attribute__((always_inline)) { return sc.weight(sc.at(y)); };
    if (s.cut) {
      const uint64_t at = far([](float) { return (uint64_t)1; }, s.k);
      if (at) last = at;
    }
    if (s.run) {
      uint64_t sum = 0;
      over([&](float y, int i) __attribute__((always_inline)) {
        if (ord.place(key_of(y), i) >= last) sum += mass(y);
      });
      sum = block_all<N>(sum, m.scan, Plus());
      const uint64_t goal = part_of(s.p, sum, true);
      last = goal <= 1 ? first : far(mass, goal);
    }
    border.above = INFINITY;                // (by place alone)
    for (int i = tid; i < SLOTS; i += N) m.slot[i] = 0;
    __syncthreads();
    for (int v = tid; v < tiles * 64; v += N) {
      uint64_t sum = 0;
      if (v < row.n_vec)
        row.each(v, [&](float y, int i) __attribute__((always_inline)) {
          if (ord.place(key_of(y), i) >= last && sc.at(y) >= sc.bar) sum += mass(y);
        });
      sum = __any(sum != 0) ? last_lane(scan64(sum)) : 0;
      if (lane == 0 && sum) atomicAdd((ull*)&m.slot[v / 64 / per], (ull)sum);
    }
    __syncthreads();
  }

  // the slot at which the sum passes the aim, then the tile and the token
  constexpr int PER = SLOTS / N;
  uint64_t mine = 0, total;
#pragma unroll
  for (int e = 0; e < PER; ++e) mine += m.slot[tid * PER + e];
  uint64_t upto_slot = block_before<N>(mine, m.scan, total);
  const uint64_t aim = aim_of(total);
  if (upto_slot <= aim && upto_slot + mine > aim) {
    int e = 0;
    while (upto_slot + m.slot[tid * PER + e] <= aim) upto_slot += m.slot[tid * PER + e++];
    m.found[0] = tid * PER + e;
    m.found[1] = upto_slot;
  }
  __syncthreads();
  if (tid >= 64) return;
  uint64_t sum_before = m.found[1];
  for (int t = (int)m.found[0] * per; t < tiles; ++t) {
    const int v = t * 64 + lane;
    float y[R::E];
    uint64_t w[R::E], sum = 0;
    row.unpack(row.load(v), v, y);
#pragma unroll
    for (int e = 0; e < R::E; ++e) {
      const float z = sc.at(y[e]);
      const bool in = z >= border.above || ord.place(key_of(y[e]), row.index(v, e)) >= last;
      w[e] = in && z >= sc.bar ? sc.weight(z) : 0;
      sum += w[e];
    }
    const uint64_t upto = scan64(sum);
    if (sum_before + last_lane(upto) > aim) {
      uint64_t sofar = sum_before + upto - sum;
      if (sofar <= aim && sofar + sum > aim) {
#pragma unroll
        for (int e = 0; e < R::E; ++e) {
          if (sofar <= aim && sofar + w[e] > aim) drawn(y[e], row.index(v, e), total);
          sofar += w[e];
        }
      }
      return;
    }
    sum_before += last_lane(upto);
  }

  }
}


// A row by one workgroup.
template <typename T, int MODE>
__global__ __launch_bounds__(threads_of(MODE)) void sample_row_kernel(SampleArgs a) {
  constexpr int N = threads_of(MODE);
  __shared__ __align__(16) Room<MODE> m;
  const int b = blockIdx.x, tid = threadIdx.x;
  const Setting s = setting_of(a, b);
  const Row<T> row(a, b);
  const Order<T> ord(a.V);
  const int tiles = (row.n_vec + 63) / 64, per = (tiles + SLOTS - 1) / SLOTS;   // tiles of a slot
  uint64_t first;
  uint32_t least = KEY_NONE + 1, maxima[MODE == WHOLE ? GROUPS / N : 1];
  if constexpr (MODE == PARTS) {
    row_ends(a, b, first, least);
  } else if constexpr (MODE == WHOLE) {
    Sweep<T, N / 64, 4> sweep(row, 0, tiles);
    float most, low;
    int at;
    uint32_t turned;
    float group[GROUPS / N];
    ends_of(sweep, a.runs, most, at, low, group);
#pragma unroll
    for (int g = 0; g < GROUPS / N; ++g) maxima[g] = key_of(group[g]);
    ends_of(row, ord, most, at, low, first, turned);
    first = block_all<N>(first, m.scan, Most());
    least = ~(uint32_t)block_all<N>(turned, m.scan, Most());
  } else {
    first = 0;
    for (int v = tid; v < row.n_vec; v += N)
      row.each(v, [&](float y, int i) __attribute__((always_inline)) {
        const uint64_t place = ord.place(key_of(y), i);
        if (i >= 0 && i < a.V) m.list[i] = place;
        first = place > first ? place : first;
      });
    first = block_all<N>(first, m.scan, Most());
  }
  if (first == 0 || s.greedy) {
    put_first(a, b, first, ord.index(first));
    return;
  }
  const Scale sc(a, s, ord.logit(first), least);
  Border border;
  uint64_t before = 0, goal = 0;
  uint32_t n_cand = 0;
  if constexpr (MODE == WHOLE) {
    if (tid == 0) m.n = 0;
    for (int i = tid; i < SLOTS; i += N) m.slot[i] = 0;
    for (int i = tid; i < BINS; i += N) m.hist[i] = 0;
    __syncthreads();
    if (s.list) {
      Sweep<T, N / 64, 4> sweep(row, 0, tiles);
      const float bar = list_bar<N>(maxima, s.k, m.count);
      gather_into(sweep, ord, bar, m.list, &m.n);
    } else if (!s.cut) {
      if (s.run) {
        Sweep<T, N / 64, 2> sweep(row, 0, tiles);
        hist_into(sweep, sc, m.hist);
        __syncthreads();
        border = Border(sc, border_bin<N>(m.hist, s.p, m.scan, before, goal), m.scan + 2);
      }
      Sweep<T, N / 64, 2> sweep(row, 0, tiles);
      sums_into(sweep, ord, sc, border, m.list, &m.n, [&](int tile, uint64_t w) __attribute__((always_inline)) {
        if (w) atomicAdd((ull*)&m.slot[tile / per], (ull)w);
      });
    }
    __syncthreads();
    n_cand = m.n;
  }
  finish<MODE>(a, b, s, row, ord, first, sc, border, goal - before, n_cand, m);
}

// ---------------------------------------------------------------------------
// A row's parts, a launch a pass.

template <typename T>
__global__ __launch_bounds__(PART) void sample_top_kernel(SampleArgs a) {
  __shared__ uint64_t s_first[PART / 64];
  __shared__ uint32_t s_low[PART / 64];
  const int b = fdiv(blockIdx.x, a.f_parts), part = blockIdx.x - b * a.parts, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  if (part == 0 && threadIdx.x == 0) a.count[b] = a.ended[b] = 0;
  if (a.runs)
    for (int i = part * PART + threadIdx.x; i < BINS; i += a.parts * PART) a.hist[(int64_t)b * BINS + i] = 0;
  const Row<T> row(a, b);
  const Order<T> ord(a.V);
  Sweep<T, PART / 64, 4> sweep(row, part * a.tiles, a.tiles);
  float most, least;
  int at;
  float group[1];
  ends_of(sweep, a.runs, most, at, least, group);
  uint32_t g = key_of(group[0]), low;
  for (int d = 1; d < a.lanes; d *= 2) g = max(g, (uint32_t)__shfl_xor((int)g, d));
  if (threadIdx.x % a.lanes == 0) a.maxima[(int64_t)b * GROUPS + (part * PART + threadIdx.x) / a.lanes] = g;
  uint64_t first;
  ends_of(row, ord, most, at, least, first, low);
  first = wave_all(first, Most());
  low = (uint32_t)wave_all(low, Most());
  if (lane == 0) {
    s_first[wave] = first;
    s_low[wave] = low;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < PART / 64; ++w) {
      first = s_first[w] > first ? s_first[w] : first;
      low = max(low, s_low[w]);
    }
    a.part[(int64_t)b * a.parts + part] = Part{first, low, 0};
  }
}

// Appends the places that the part holds to the row's list.
__device__ __forceinline__ void append(const SampleArgs& a, int b, Room<PARTS>& m) {
  __syncthreads();
  const uint32_t n = m.n;
  if (threadIdx.x == 0 && n > 0) m.at = atomicAdd(a.count + b, n);
  __syncthreads();
  if (n == 0 || n > LIST) return;
  for (uint32_t i = threadIdx.x; i < n; i += PART)
    if (m.at + i < LIST) put(a.list + (int64_t)b * LIST + m.at + i, m.list[i]);
}

// Whether all of a row's parts are through, for the last of them. What they tell it is
// put() and got(), at the device's scope: each wave waits until its words are out before
// its part counts as through, and what the last one reads comes after. Nobody waits for
// another part. (One launch less: 1 us of a single row. With fences in place of the words'
// scope, which write back and drop a whole L2 in each workgroup, 8 rows take twice as long.)
__device__ __forceinline__ bool last_part(const SampleArgs& a, int b, Room<PARTS>& m) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) m.at = atomicAdd(a.ended + b, 1u);
  __syncthreads();
  return (int)m.at == a.parts - 1;
}

// top_k's lists, and top_p's histograms. Where no sums follow (all rows have a list), the
// last part of a row ends it.
template <typename T>
__global__ __launch_bounds__(PART) void sample_gather_kernel(SampleArgs a) {
  __shared__ __align__(16) Room<PARTS> m;
  const int b = fdiv(blockIdx.x, a.f_parts), part = blockIdx.x - b * a.parts;
  const Setting s = setting_of(a, b);
  if (a.sums && !(s.cut ? s.list : s.run && !s.greedy)) return;
  const Row<T> row(a, b);
  const Order<T> ord(a.V);
  if (s.list) {
    Sweep<T, PART / 64, 4> sweep(row, part * a.tiles, a.tiles);
    const u32x4 mx = *(const u32x4*)(a.maxima + (int64_t)b * GROUPS + threadIdx.x * 4);
    const uint32_t key[] = {mx[0], mx[1], mx[2], mx[3]};
    if (threadIdx.x == 0) m.n = 0;
    const float bar = list_bar<PART>(key, s.k, m.count);
    gather_into(sweep, ord, bar, m.list, &m.n);
    append(a, b, m);
    if (a.sums || !last_part(a, b, m)) return;
  } else if (!a.sums && part > 0) {
    return;                                 // (a greedy row)
  }
  uint64_t first;
  uint32_t least;
  row_ends(a, b, first, least);
  if (first == 0 || s.greedy) {
    if (!a.sums) put_first(a, b, first, ord.index(first));
    return;
  }
  const Scale sc(a, s, ord.logit(first), least);
  if (!a.sums) {
    finish<PARTS>(a, b, s, row, ord, first, sc, Border(), 0, got(a.count + b), m);
    return;
  }
  for (int i = threadIdx.x; i < BINS; i += PART) m.w[i] = 0;
  __syncthreads();
  Sweep<T, PART / 64, 2> sweep(row, part * a.tiles, a.tiles);
  hist_into(sweep, sc, m.w);
  __syncthreads();
  ull* to = (ull*)a.hist + (int64_t)b * BINS;
  for (int i = threadIdx.x; i < BINS; i += PART)
    if (m.w[i]) atomicAdd(to + i, (ull)m.w[i]);
}

// The kept weight of the tiles; the last part of a row ends it.
template <typename T>
__global__ __launch_bounds__(PART) void sample_sums_kernel(SampleArgs a) {
  __shared__ __align__(16) Room<PARTS> m;
  const int b = fdiv(blockIdx.x, a.f_parts), part = blockIdx.x - b * a.parts;
  const Setting s = setting_of(a, b);
  const bool alone = s.greedy || s.cut;     // ended by one part, without sums
  if (alone && part > 0) return;
  const Row<T> row(a, b);
  const Order<T> ord(a.V);
  Sweep<T, PART / 64, 2> sweep(row, part * a.tiles, a.tiles);
  uint64_t first;
  uint32_t least;
  row_ends(a, b, first, least);
  if (first == 0 || s.greedy) {
    if (part == 0) put_first(a, b, first, ord.index(first));
    return;
  }
  const Scale sc(a, s, ord.logit(first), least);
  uint64_t before = 0, goal = 0;
  Border border;
  if (alone) {
    finish<PARTS>(a, b, s, row, ord, first, sc, border, 0, got(a.count + b), m);
    return;
  }
  if (s.run) border = Border(sc, border_bin<PART>(a.hist + (int64_t)b * BINS, s.p, m.scan, before, goal), m.scan + 2);
  if (threadIdx.x == 0) m.n = 0;
  __syncthreads();
  uint64_t* sums = a.tile + (int64_t)b * a.parts * a.tiles;
  sums_into(sweep, ord, sc, border, m.list, &m.n, [&](int tile, uint64_t w) __attribute__((always_inline)) { put(sums + tile, w); });
  if (s.run) append(a, b, m);
  if (last_part(a, b, m)) finish<PARTS>(a, b, s, row, ord, first, sc, border, goal - before, got(a.count + b), m);
}

// ---------------------------------------------------------------------------
// host side

struct Plan {
  int parts, tiles, lanes;                  // parts 0: a workgroup a row, one launch
  size_t part, maxima, count, ended, hist, list, tile, bytes;   // offsets
};

// A workgroup takes a whole row where there are rows for most CUs, or short ones. By
// workgroups / parts, us, bfloat16:
//                     temperature  top_k 50  top_p 0.9  a flat nucleus
//   128256 x 128         42 / 32    21 / 23    74 / 50      88 / 63
//   128256 x 192         45 / 49    24 / 43    78 / 72      90 / 98
//   32000 x 96           18 / 17    15 / 20    31 / 31      36 / 34
//   16000 x 16           14 / 12    14 / 16    22 / 22      23 / 23
//   8192 x 1             11 / 12    13 / 15    18 / 21      19 / 21
// (One rule for all settings: a nucleus of 192 rows is 8 % faster by parts. Past 256 rows
// there is a second round of workgroups: 257 rows with top_p 0.9 165 us, 256 90, 512 177.)
bool by_rows(int B, int V) { return B >= 160 || V <= 8192 || (B >= 64 && V <= 32768); }

void plan_for(Plan& p, int B, int V, int dtype, bool differ) {
  p = Plan{};
  if (by_rows(B, V)) return;
  const int E = dtype == DA_FP32 ? 4 : 8;
  const int64_t tiles = ((int64_t)V + 2 * E - 1) / E / 64 + 1;   // whatever the row's alignment
  // parts: 4 at least; then a workgroup a CU, of 8 tiles (one of each wave) at least.
  // Rows that ask for different things differ in work: two a CU spread it. 64 such rows of
  // 151936 bfloat16 tokens, 8 / 4 parts: 47 / 56 us, 48 rows 44 / 54; of rows that are alike
  // 64 with top_k 50 take 21.2 / 18.9, 32 of them 20.5 (16 parts) / 17.3 (8).
  int64_t parts = 4;
  while (parts < 32 && tiles >= parts * 2 * 8 && parts * 2 * B <= (differ && parts < 16 ? 512 : 256)) parts *= 2;
  p.tiles = (int)(((tiles + parts - 1) / parts + 7) / 8 * 8);
  p.parts = (int)parts;
  p.lanes = p.parts * PART / GROUPS;
  size_t at = 0;
  auto room = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes * B + 255) / 256 * 256;
    return here;
  };
  p.part = room(sizeof(Part) * p.parts);
  p.maxima = room(sizeof(uint32_t) * GROUPS);
  p.count = room(sizeof(uint32_t));
  p.ended = room(sizeof(uint32_t));
  p.hist = room(sizeof(uint64_t) * BINS);
  p.list = room(sizeof(uint64_t) * LIST);
  p.tile = room(sizeof(uint64_t) * p.parts * p.tiles);
  p.bytes = at;
}

template <typename T>
void launch(SampleArgs& a, hipStream_t st) {
  if (a.V <= LIST) {
    hipLaunchKernelGGL((sample_row_kernel<T, SHORT>), dim3(a.B), dim3(threads_of(SHORT)), 0, st, a);
    return;
  }
  // (what no row can ask for is not launched)
  const bool t_on = a.t_dev || a.t > 0.f, k_on = a.k_dev || (a.k > 0 && a.k < a.V);
  const bool k_all = !a.k_dev && a.k > 0 && a.k < a.V, k_list = a.k_dev || (k_on && a.k <= a.k_list);
  const bool p_on = a.p_dev || a.p < 1.f;
  a.runs = t_on && p_on && !k_all;
  if (a.parts == 0) {
    hipLaunchKernelGGL((sample_row_kernel<T, WHOLE>), dim3(a.B), dim3(threads_of(WHOLE)), 0, st, a);
    return;
  }
  const dim3 grid(a.parts * a.B);
  a.sums = t_on && !k_all;
  const bool gather = t_on && (k_list || a.runs);
  hipLaunchKernelGGL((sample_top_kernel<T>), grid, dim3(PART), 0, st, a);
  if (gather) hipLaunchKernelGGL((sample_gather_kernel<T>), grid, dim3(PART), 0, st, a);
  if (a.sums) hipLaunchKernelGGL((sample_sums_kernel<T>), grid, dim3(PART), 0, st, a);
  // (all greedy, or a top_k past the lists)
  if (!gather && !a.sums) hipLaunchKernelGGL((sample_row_kernel<T, PARTS>), dim3(a.B), dim3(PART), 0, st, a);
}

}  // namespace
}  // namespace da

using namespace da;

extern "C" size_t da_sample_workspace_bytes(int B, int V, int dtype) {
  if (B < 1 || B > MAX_B || V < 1 || V > MAX_V || (dtype != DA_BF16 && dtype != DA_FP16 && dtype != DA_FP32)) return 0;
  Plan p;
  plan_for(p, B, V, dtype, false);
  const size_t bytes = p.bytes;
  plan_for(p, B, V, dtype, true);
  return p.bytes > bytes ? p.bytes : bytes;
}

extern "C" int da_sample(const da_sample_args* x, void* stream) {
  if (!x) return DA_ERR_INVALID_ARG;
  if (x->dtype != DA_BF16 && x->dtype != DA_FP16 && x->dtype != DA_FP32) return DA_ERR_DTYPE;
  if (x->B < 0 || x->B > MAX_B || x->V < 1 || x->V > MAX_V) return DA_ERR_INVALID_ARG;
  if (x->B == 0) return DA_OK;
  if (!x->logits || !x->u || !x->tokens || !x->logprobs) return DA_ERR_INVALID_ARG;
  if (((uintptr_t)x->logits & (x->dtype == DA_FP32 ? 3 : 1)) || ((uintptr_t)x->u & 3) || ((uintptr_t)x->tokens & 7) ||
      ((uintptr_t)x->logprobs & 3) || ((uintptr_t)x->temperature_dev & 3) || ((uintptr_t)x->top_k_dev & 3) ||
      ((uintptr_t)x->top_p_dev & 3) || ((uintptr_t)x->min_p_dev & 3))
    return DA_ERR_ALIGNMENT;
  Plan p;
  const bool differ = (x->temperature_dev && x->temperature_per_row) || (x->top_k_dev && x->top_k_per_row) ||
                      (x->top_p_dev && x->top_p_per_row) || (x->min_p_dev && x->min_p_per_row);
  plan_for(p, x->B, x->V, x->dtype, differ);
  if (p.bytes > 0 && (!x->workspace || x->workspace_bytes < (int64_t)p.bytes)) return DA_ERR_WORKSPACE;
  if (!aligned16(x->workspace)) return DA_ERR_ALIGNMENT;
  SampleArgs a{};
  a.x = x->logits;
  a.x_b = x->row_stride;
  a.u = x->u;
  a.t_dev = x->temperature_dev, a.k_dev = x->top_k_dev, a.p_dev = x->top_p_dev, a.m_dev = x->min_p_dev;
  a.t_step = x->temperature_per_row ? 1 : 0, a.k_step = x->top_k_per_row ? 1 : 0;
  a.p_step = x->top_p_per_row ? 1 : 0, a.m_step = x->min_p_per_row ? 1 : 0;
  a.t = x->temperature, a.k = x->top_k, a.p = x->top_p, a.m = x->min_p;
  a.token = x->tokens;
  a.logp = x->logprobs;
  a.B = x->B, a.V = x->V;
  a.bits = 62;
  while (1 << (62 - a.bits) < x->V) --a.bits;
  if (a.bits > 45) a.bits = 45;
  a.parts = p.parts, a.tiles = p.tiles;
  a.f_parts = make_fastdiv(p.parts > 0 ? p.parts : 1);
  a.lanes = p.lanes;
  a.k_list = GROUPS / 4 * 3;
  char* ws = (char*)x->workspace;
  a.part = (Part*)(ws + p.part);
  a.maxima = (uint32_t*)(ws + p.maxima);
  a.count = (uint32_t*)(ws + p.count);
  a.ended = (uint32_t*)(ws + p.ended);
  a.hist = (uint64_t*)(ws + p.hist);
  a.list = (uint64_t*)(ws + p.list);
  a.tile = (uint64_t*)(ws + p.tile);
  (void)hipGetLastError();
  hipStream_t st = (hipStream_t)stream;
  if (x->dtype == DA_BF16) launch<__bf16>(a, st);
  else if (x->dtype == DA_FP16) launch<_Float16>(a, st);
  else launch<float>(a, st);
  return hipGetLastError() == hipSuccess ? DA_OK : DA_ERR_LAUNCH;
}
