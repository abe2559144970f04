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
// split over threads, and the products u * total and p * total are exact.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "capi_common.h"
#include "delta_attn.h"
#include "device_common.h"

namespace da {
namespace {

typedef unsigned __int128 u128;

constexpr int MAX_V = 1 << 24;               // tokens of a vocabulary
constexpr int MAX_B = 0x3fffff;              // rows (threads of a grid: below 2^32)
constexpr uint32_t KEY_NONE = 0x007fffffu;   // -inf's key: candidates lie above it

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
};

// A number's place in the order of floats (-0 beside 0); NaN last.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0u : (int)b < 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// A token's place in the order: larger is earlier. 0: no candidate.
__device__ __forceinline__ uint64_t place_of(uint32_t key, int i) {
  return key > KEY_NONE ? (uint64_t)key << 32 | (uint32_t)~i : 0;
}
__device__ __forceinline__ int index_of(uint64_t place) { return (int)~(uint32_t)place; }

// 2^t for t <= 0 in units of 2^-bits: the fraction's power by its series to the
// 13th term (2^-52 of it), the whole one by the exponent.
__device__ __forceinline__ uint64_t weight_of(double t, int bits) {
  t = fmax(t, -200.0);                      // (2^-200 of the largest: none)
  const double n = rint(t), f = (t - n) * 0.693147180559945309417;
  double p = 1.0 / 479001600;
  constexpr double c[] = {1.0 / 39916800, 1.0 / 3628800, 1.0 / 362880, 1.0 / 40320, 1.0 / 5040, 1.0 / 720,
                          1.0 / 120, 1.0 / 24, 1.0 / 6, 0.5, 1.0, 1.0};
#pragma unroll
  for (int i = 0; i < 12; ++i) p = fma(p, f, c[i]);
  return (uint64_t)rint(ldexp(p, (int)n + bits));
}

template <typename T> struct Logit;
template <> struct Logit<__bf16> {
  static __device__ __forceinline__ float at(const void* p, int i) { return Elt<__bf16>::lo(((const uint16_t*)p)[i]); }
};
template <> struct Logit<_Float16> {
  static __device__ __forceinline__ float at(const void* p, int i) { return (float)((const _Float16*)p)[i]; }
};
template <> struct Logit<float> {
  static __device__ __forceinline__ float at(const void* p, int i) { return ((const float*)p)[i]; }
};

constexpr int THREADS = 1024;
constexpr int BINS = 2048;

template <typename F>
__device__ __forceinline__ uint64_t block_reduce(uint64_t v, uint64_t* s, F&& f) {
  for (int d = 32; d > 0; d /= 2) v = f(v, __shfl_xor(v, d));
  __syncthreads();
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
  __syncthreads();
  v = s[0];
  for (int w = 1; w < THREADS / 64; ++w) v = f(v, s[w]);
  return v;
}

// ceil or floor of f * total for 0 <= f < 1, exactly.
__device__ __forceinline__ uint64_t part_of(float f, uint64_t total, bool up) {
  const uint32_t b = __float_as_uint(f);
  if (f != f || (int)b <= 0) return 0;
  const int e = b >> 23;                    // f = mant * 2^(e - 150)
  const uint32_t mant = e ? (b & 0x7fffff) | 0x800000 : b & 0x7fffff;
  const int shift = 150 - (e ? e : 1);      // 24 at least
  if (shift > 120) return up && total ? 1 : 0;
  const u128 y = (u128)mant * total;
  return (uint64_t)((y + (up ? ((u128)1 << shift) - 1 : 0)) >> shift);
}

template <typename T>
__global__ __launch_bounds__(THREADS) void sample_kernel(SampleArgs a) {
  __shared__ uint64_t s_red[THREADS / 64], s_bin[BINS], s_found[3];
  const int b = blockIdx.x, tid = threadIdx.x;
  const T* x = (const T*)a.x + (int64_t)b * a.x_b;
  const auto most = [](uint64_t p, uint64_t q) { return p > q ? p : q; };
  const auto plus = [](uint64_t p, uint64_t q) { return p + q; };

  uint64_t first = 0;
  for (int i = tid; i < a.V; i += THREADS) first = most(first, place_of(key_of(Logit<T>::at(x, i)), i));
  first = block_reduce(first, s_red, most);
  if (first == 0) {
    if (tid == 0) {
      a.token[b] = 0;
      a.logp[b] = __builtin_nanf("");
    }
    return;
  }
  const float temp = a.t_dev ? a.t_dev[b * a.t_step] : a.t;
  if (!(temp > 0.f)) {
    if (tid == 0) {
      a.token[b] = index_of(first);
      a.logp[b] = 0.f;
    }
    return;
  }
  const int k = a.k_dev ? a.k_dev[b * a.k_step] : a.k;
  const float p = a.p_dev ? a.p_dev[b * a.p_step] : a.p, m = a.m_dev ? a.m_dev[b * a.m_step] : a.m;
  const double top = of_key(first >> 32), per = 1.44269504088896340736 / (double)temp;
  auto weight = [&](float y) __attribute__((always_inline)) -> uint64_t {
    // (an infinite one: the tokens at it share the row)
    return weight_of((double)y == top ? 0.0 : ((double)y - top) * per, a.bits);
  };
  uint64_t last = 1;                        // the last place kept
  // The first place in the order at which the measure, summed, reaches `goal`
  // (0: none does), eleven bits of the place at a time.
  auto reach = [&](auto&& measure, uint64_t goal) {
    uint64_t prefix = 0, before = 0;
    for (int low = 55; low >= 0; low -= 11) {
      for (int i = tid; i < BINS; i += THREADS) s_bin[i] = 0;
      __syncthreads();
      for (int i = tid; i < a.V; i += THREADS) {
        const float y = Logit<T>::at(x, i);
        const uint64_t place = place_of(key_of(y), i);
        if (place < last || (low < 55 && place >> (low + 11) != prefix)) continue;
        const uint64_t w = measure(y);
        if (w) atomicAdd((unsigned long long*)&s_bin[place >> low & (BINS - 1)], (unsigned long long)w);
      }
      __syncthreads();
      if (tid == 0) {
        uint64_t sum = before;
        int i = BINS - 1;
        for (; i > 0 && sum + s_bin[i] < goal; --i) sum += s_bin[i];
        s_found[0] = prefix << 11 | i;
        s_found[1] = sum;
        s_found[2] = sum + s_bin[i];
      }
      __syncthreads();
      prefix = s_found[0];
      before = s_found[1];
      if (s_found[2] < goal) return (uint64_t)0;
    }
    return prefix;
  };
  if (k > 0 && k < a.V) {
    const uint64_t at = reach([](float) { return (uint64_t)1; }, k);
    if (at) last = at;
  }
  if (p < 1.f) {
    uint64_t sum = 0;
    for (int i = tid; i < a.V; i += THREADS) {
      const float y = Logit<T>::at(x, i);
      if (place_of(key_of(y), i) >= last) sum += weight(y);
    }
    sum = block_reduce(sum, s_red, plus);
    const uint64_t goal = part_of(p, sum, true);
    const uint64_t at = goal <= 1 ? first : reach(weight, goal);
    if (at) last = at;
  }
  const double bar = m > 0.f ? top + (double)temp * log((double)m) : -INFINITY;
  auto kept = [&](float y, int i) __attribute__((always_inline)) -> uint64_t {
    const uint64_t place = place_of(key_of(y), i);
    return place >= last && ((double)y >= bar || place == first) ? weight(y) : 0;
  };
  // a stretch of the row for each thread, then the stretch's own tokens
  const int len = (a.V + THREADS - 1) / THREADS, from = tid * len, to = min(from + len, a.V);
  uint64_t sum = 0;
  for (int i = from; i < to; ++i) sum += kept(Logit<T>::at(x, i), i);
  __syncthreads();
  s_bin[tid] = sum;
  __syncthreads();
  uint64_t before = 0, total = 0;
  for (int t = 0; t < THREADS; ++t) {
    if (t == tid) before = total;
    total += s_bin[t];
  }
  const uint64_t goal = part_of(a.u[b], total, false);
  const uint64_t aim = goal < total ? goal : total - 1;
  if (before > aim || before + sum <= aim) return;
  for (int i = from; i < to; ++i) {
    const float y = Logit<T>::at(x, i);
    before += kept(y, i);
    if (before > aim) {
      a.token[b] = i;
      const double d = (double)y == top ? 0.0 : ((double)y - top) / (double)temp;
      a.logp[b] = (float)(d - log(ldexp((double)total, -a.bits)));
      return;
    }
  }
}

}  // namespace
}  // namespace da

using namespace da;

extern "C" size_t da_sample_workspace_bytes(int, int, int) { return 0; }

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
  (void)hipGetLastError();
  const dim3 grid(x->B), block(THREADS);
  hipStream_t st = (hipStream_t)stream;
  if (x->dtype == DA_BF16) hipLaunchKernelGGL((sample_kernel<__bf16>), grid, block, 0, st, a);
  else if (x->dtype == DA_FP16) hipLaunchKernelGGL((sample_kernel<_Float16>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((sample_kernel<float>), grid, block, 0, st, a);
  return hipGetLastError() == hipSuccess ? DA_OK : DA_ERR_LAUNCH;
}
