/*
 * gq_sample_rows.hip — the next token of every row of a batch from random
 * numbers given, each row with its own temperature, top-k, top-p and min-p
 * (gfx950).
 *
 * A row's tokens in descending order of their logits (equal ones: lowest index
 * first) are x_0 >= x_1 >= ..; w_i = e^((x_i - x_0) / T).  Top-k keeps the
 * first k, top-p the shortest prefix of those with a sum of w of at least p of
 * theirs, min-p those of them with w >= min_p.  The token is the first in index
 * order at which the running sum of w over the kept ones passes rnd times
 * their whole sum.
 *
 * Nothing is sorted.  The two borders are found by selection: a histogram of
 * counts and sums over 2048 bins of (x_0 - x) / T, the bin that holds the
 * border, and then eleven bits at a time of the key (logit, index) within it,
 * until a bin holds one token.  A w is held as a whole number of 2^-S, S such
 * that a row's sum fits 63 bits (45 at 128256 tokens): sums are then exact in any
 * order, so atomics may add them and the same call gives the same token, and a
 * w's own error of 2^-46 moves no draw that another order of a float64 sum
 * would not.
 */
#include <algorithm>
#include <cmath>

#include "gq_device.h"
#include "gq_internal.h"

namespace {

constexpr int kT = 1024, kW = kT / GQ_WAVE, kBins = 2048, kMaxVocab = 1 << 20;

struct SampArgs {
  const float *x;
  const float *temperature, *top_p, *min_p, *rnd;
  const int32_t *top_k;
  int32_t *tokens;
  float *logprobs;
  int vocab;
  long long stride;
  int S; /* w is held in units of 2^-S */
};

/* order of the logits as an unsigned integer, -0 as +0; 0 for what is never
 * picked (-infinity, NaN) */
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v == 0.f ? 0.f : v);
  return v > -INFINITY ? ((u & 0x80000000u) ? ~u : (u | 0x80000000u)) : 0u;
}
/* (logit, index): a larger one comes first */
__device__ __forceinline__ uint64_t comp_of(float v, int i) {
  return (uint64_t)key_of(v) << 32 | (uint32_t)~i;
}

struct Shared {
  double tab[64]; /* 2^(i / 64) */
  unsigned long long mass[kBins];
  uint32_t cnt[kBins];
  unsigned long long wsum[kW];
  float wmax[kW];
  int widx[kW];
  int at;
  unsigned long long before, in;
  uint32_t n;
};

/* e^t, t <= 0, to about 2^-52: t = (k + f) ln 2 / 64, 2^(k / 64) from the
 * table, e^r of the rest (|r| < 0.0055) by its series to r^5 / 120 (the next
 * term is below 2^-54) */
__device__ __forceinline__ double exp_neg(double t, const double *tab) {
  if (!(t > -60.0)) return 0.0;
  const double k = __builtin_rint(t * 92.332482616893656877); /* 64 / ln 2 */
  /* ln 2 / 64 in two parts, the first of 33 bits, so that k times it is exact */
  double r = __builtin_fma(-k, 0x1.62e42fefp-7, t);
  r = __builtin_fma(-k, 0x1.473de6af278edp-40, r);
  double p = __builtin_fma(r, 1.0 / 120, 1.0 / 24);
  p = __builtin_fma(r, p, 1.0 / 6);
  p = __builtin_fma(r, p, 0.5);
  p = __builtin_fma(r * r, p, r);
  const int n = (int)k;
  const double s = tab[n & 63];
  return __builtin_ldexp(__builtin_fma(s, p, s), n >> 6);
}

struct Row {
  const float *x;
  float top, T;
  double two_S;
  const double *tab;
  __device__ double w(float v) const {
    return v == top ? 1.0 : key_of(v) ? exp_neg(((double)v - (double)top) / (double)T, tab) : 0.0;
  }
  /* in units of 2^-S, nearest even: added to 2^52 a double's low bits are it */
  __device__ unsigned long long mass(double w) const {
    return __builtin_bit_cast(unsigned long long, __builtin_fma(w, two_S, 0x1p52)) & 0xfffffffffffffull;
  }
};

/* The first bin at which the running sum, `base` included, reaches the target
 * (or the last bin, if none does): its number to sh.at, the sum before it to
 * sh.before, its own to sh.in, its count to sh.n.  By count, or by mass. */
template <bool COUNT>
__device__ void find_bin(Shared &sh, unsigned long long base, double target) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const unsigned long long a = COUNT ? sh.cnt[2 * tid] : sh.mass[2 * tid];
  const unsigned long long b = COUNT ? sh.cnt[2 * tid + 1] : sh.mass[2 * tid + 1];
  unsigned long long s = a + b;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long u = __shfl_up(s, o, 64);
    if (lane >= o) s += u;
  }
  if (lane == 63) sh.wsum[wave] = s;
  __syncthreads();
  unsigned long long off = base;
  for (int w = 0; w < wave; w++) off += sh.wsum[w];
  const unsigned long long c0 = off + s - a - b, c1 = c0 + a, c2 = c1 + b;
  const bool last = tid == kT - 1;
  if (!((double)c0 >= target) || tid == 0) {
    if ((double)c1 >= target) sh.at = 2 * tid, sh.before = c0, sh.in = a, sh.n = sh.cnt[2 * tid];
    else if ((double)c2 >= target || last) sh.at = 2 * tid + 1, sh.before = c1, sh.in = b, sh.n = sh.cnt[2 * tid + 1];
  }
  __syncthreads();
}

__global__ __launch_bounds__(kT) void sample_rows_kernel(SampArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocab;
  const long long rowi = blockIdx.x;
  const float *x = a.x + rowi * a.stride;
  const float T = a.temperature ? a.temperature[rowi] : 1.f;
  if (tid < 64) sh.tab[tid] = exp2((double)tid / 64);
  /* the largest logit, the lowest index of it */
  float top = -INFINITY;
  int ti = -1;
  for (int i = tid; i < V; i += kT) {
    const float v = x[i];
    if (v > top) top = v, ti = i;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const float v = __shfl_xor(top, o, 64);
    const int j = __shfl_xor(ti, o, 64);
    if (v > top || (v == top && (unsigned)j < (unsigned)ti)) top = v, ti = j;
  }
  if (lane == 0) sh.wmax[wave] = top, sh.widx[wave] = ti;
  __syncthreads();
  for (int w = 0; w < kW; w++) {
    const float v = sh.wmax[w];
    if (v > top || (v == top && (unsigned)sh.widx[w] < (unsigned)ti)) top = v, ti = sh.widx[w];
  }
  if (!(T > 0.f) || ti < 0) { /* greedy, or nothing to pick */
    if (tid == 0) {
      a.tokens[rowi] = ti;
      if (a.logprobs) a.logprobs[rowi] = ti < 0 ? -INFINITY : 0.f;
    }
    return;
  }
  const Row row{x, top, T, __builtin_ldexp(1.0, a.S), sh.tab};
  int k = a.top_k ? a.top_k[rowi] : 0;
  float top_p = a.top_p ? a.top_p[rowi] : 1.f;
  float min_p = a.min_p ? a.min_p[rowi] : 0.f;
  min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
  if (top_p <= 0.f) k = 1, top_p = 1.f;
  const bool by_k = k > 0 && k < V, by_p = top_p < 1.f;
  /* bins: the last holds what weighs nothing in units of 2^-S */
  const float scale = (float)((kBins - 1) / ((a.S + 1.5) * 0.6931471805599453)) / T;
  auto bin_of = [&](float v) {
    return v == top ? 0 : (int)fminf((top - v) * scale, (float)(kBins - 1));
  };
  uint64_t cut = 0; /* tokens with a smaller (logit, index) are left out */
  if (by_k || by_p) {
    for (int i = tid; i < kBins; i += kT) sh.cnt[i] = 0, sh.mass[i] = 0;
    __syncthreads();
    for (int i = tid; i < V; i += kT) {
      const float v = x[i];
      if (!key_of(v)) continue;
      const int b = bin_of(v);
      atomicAdd(&sh.cnt[b], 1u);
      if (b < kBins - 1) atomicAdd(&sh.mass[b], row.mass(row.w(v)));
    }
    __syncthreads();
    unsigned long long whole = 0; /* mass of what top-k keeps */
    for (int pass = 0; pass < 2; pass++) {
      if (pass == 0 ? !by_k : !by_p) {
        if (pass == 0) { /* every token */
          unsigned long long s = sh.mass[2 * tid] + sh.mass[2 * tid + 1];
#pragma unroll
          for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
          if (lane == 0) sh.wsum[wave] = s;
          __syncthreads();
          for (int w = 0; w < kW; w++) whole += sh.wsum[w];
          __syncthreads();
        }
        continue;
      }
      if (pass == 1 && by_k) { /* the histogram of the tokens again */
        for (int i = tid; i < kBins; i += kT) sh.cnt[i] = 0, sh.mass[i] = 0;
        __syncthreads();
        for (int i = tid; i < V; i += kT) {
          const float v = x[i];
          if (!key_of(v) || comp_of(v, i) < cut) continue;
          const int b = bin_of(v);
          atomicAdd(&sh.cnt[b], 1u);
          if (b < kBins - 1) atomicAdd(&sh.mass[b], row.mass(row.w(v)));
        }
        __syncthreads();
      }
      const double target = pass == 0 ? (double)k : (double)top_p * (double)whole;
      unsigned long long base = 0, above = 0; /* tokens (pass 0) and mass before the border's bin */
      if (pass == 0) {
        find_bin<true>(sh, 0, target);
        const int at = sh.at;
        unsigned long long s = 0;
        for (int i = tid; i < at; i += kT) s += sh.mass[i];
#pragma unroll
        for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
        if (lane == 0) sh.wsum[wave] = s;
        __syncthreads();
        for (int w = 0; w < kW; w++) above += sh.wsum[w];
      } else {
        find_bin<false>(sh, 0, target);
      }
      const int bin = sh.at;
      base = sh.before;
      uint32_t n = sh.n;
      unsigned long long in = sh.mass[bin];
      __syncthreads();
      if (bin == kBins - 1) { /* the rest weighs nothing */
        if (pass == 0) whole = above + in;
        continue;
      }
      /* eleven bits of (logit, index) at a time */
      uint64_t prefix = 0;
      int shift = 64;
      while (n > 1 && shift > 0) {
        const int bits = min(11, shift), low = (1 << bits) - 1;
        shift -= bits;
        for (int i = tid; i < kBins; i += kT) sh.cnt[i] = 0, sh.mass[i] = 0;
        __syncthreads();
        for (int i = tid; i < V; i += kT) {
          const float v = x[i];
          if (!key_of(v) || bin_of(v) != bin) continue;
          const uint64_t c = comp_of(v, i);
          if (c < cut || (shift + bits < 64 && c >> (shift + bits) != prefix)) continue;
          const int d = low - ((int)(c >> shift) & low); /* the largest first */
          atomicAdd(&sh.cnt[d], 1u);
          atomicAdd(&sh.mass[d], row.mass(row.w(v)));
        }
        __syncthreads();
        if (pass == 0) find_bin<true>(sh, base, target);
        else find_bin<false>(sh, base, target);
        const int at = sh.at;
        if (pass == 0) {
          unsigned long long s = 0;
          for (int i = tid; i < at; i += kT) s += sh.mass[i];
#pragma unroll
          for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
          if (lane == 0) sh.wsum[wave] = s;
          __syncthreads();
          for (int w = 0; w < kW; w++) above += sh.wsum[w];
        }
        base = sh.before, n = sh.n, in = sh.mass[at];
        prefix = prefix << bits | (uint64_t)(low - at);
        __syncthreads();
      }
      if (pass == 0) whole = above + in;
      /* the border's token, the only one left */
      if (shift == 0) {
        cut = prefix;
      } else {
        for (int i = tid; i < V; i += kT) {
          const float v = x[i];
          const uint64_t c = comp_of(v, i);
          if (key_of(v) && bin_of(v) == bin && c >= cut && (shift == 64 || c >> shift == prefix)) sh.before = c;
        }
        __syncthreads();
        cut = sh.before;
        __syncthreads();
      }
    }
  }
  /* the draw: each wave's slice of the tokens, then 64 at a time within it */
  const int per = (V + kW - 1) / kW, lo = min(V, wave * per), hi = min(V, lo + per);
  auto kept = [&](int i) -> unsigned long long {
    const float v = x[i];
    if (comp_of(v, i) < cut) return 0;
    const double w = row.w(v);
    return w >= (double)min_p ? row.mass(w) : 0ull;
  };
  unsigned long long s = 0;
  for (int i = lo + lane; i < hi; i += GQ_WAVE) s += kept(i);
#pragma unroll
  for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) sh.wsum[wave] = s;
  __syncthreads();
  unsigned long long whole = 0, before = 0;
  int slice = -1, last = 0;
  unsigned long long at = 0;
  for (int w = 0; w < kW; w++) whole += sh.wsum[w];
  const double target = (double)a.rnd[rowi] * (double)whole;
  for (int w = 0; w < kW; w++) {
    if (sh.wsum[w]) {
      last = w;
      if (slice < 0 && (double)(before + sh.wsum[w]) > target) slice = w, at = before;
    }
    before += sh.wsum[w];
  }
  const bool none = slice < 0; /* rnd 1 or more, or not a number: the last one */
  if (none) slice = last;
  if (wave != slice) return;
  int token = -1;
  for (int b = lo; b < hi && (none || token < 0); b += GQ_WAVE) {
    const int i = b + lane;
    const unsigned long long m = i < hi ? kept(i) : 0ull;
    unsigned long long c = m;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const unsigned long long u = __shfl_up(c, o, 64);
      if (lane >= o) c += u;
    }
    const uint64_t hit = __ballot(m && (none || (double)(at + c) > target));
    if (hit) token = b + (none ? 63 - __builtin_clzll(hit) : __builtin_ctzll(hit));
    at += __shfl(c, 63, 64);
  }
  if (lane == 0) {
    a.tokens[rowi] = token;
    if (a.logprobs)
      a.logprobs[rowi] = (float)(x[token] == top ? -log((double)whole / row.two_S)
                                                  : ((double)x[token] - (double)top) / (double)T - log((double)whole / row.two_S));
  }
}

} // namespace

extern "C" int gq_hip_sample_rows_dev(gq_ctx *c, const float *logits, int rows, int vocab, int row_stride,
                                      const float *temperature, const int32_t *top_k, const float *top_p,
                                      const float *min_p, const float *rnd, int32_t *tokens, float *logprobs) {
  if (!c) return -1;
  if (rows < 0 || vocab < 1 || vocab > kMaxVocab) return gq_ctx_fail(c, -1, "sample_rows: rows, or a vocabulary past 2^20");
  if (!rows) return 0;
  if (!logits || !rnd || !tokens) return gq_ctx_fail(c, -1, "sample_rows: NULL logits, rnd or tokens");
  if (row_stride < vocab) return gq_ctx_fail(c, -1, "sample_rows: rows overlap");
  for (const void *p : {(const void *)logits, (const void *)temperature, (const void *)top_k, (const void *)top_p,
                        (const void *)min_p, (const void *)rnd, (const void *)tokens, (const void *)logprobs})
    if ((uintptr_t)p & 3) return gq_ctx_fail(c, -1, "sample_rows: a pointer is not 4-byte aligned");
  const GqCtxInfo ci = gq_ctx_info(c);
  GqDeviceGuard guard(ci.dev);
  int bits = 0;
  while ((1 << bits) < vocab) bits++;
  const SampArgs a{logits, temperature, top_p, min_p, rnd, top_k, tokens, logprobs, vocab, row_stride, std::min(51, 62 - bits)};
  hipLaunchKernelGGL(sample_rows_kernel, dim3(rows), dim3(kT), 0, ci.stream, a);
  return hipGetLastError() == hipSuccess ? 0 : gq_ctx_fail(c, -4, "sample_rows launch");
}
