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
 * counts and sums over bins of (x_0 - x) / T, the bin that holds the border,
 * and then eleven bits at a time of (logit, index) within it, until a bin holds
 * one token.  A w is held as a whole number of 2^-S, S such that a row's sum
 * fits 63 bits (45 at 128256 tokens): sums are then exact in any order, so
 * atomics may add them, the same call gives the same token, and neither
 * depends on how many workgroups share a row.
 *
 * Four launches: the largest logit of every 4096 tokens; the histograms of a
 * row's parts; the border of top-k (or else top-p) and a list of the tokens in
 * its bin; one workgroup a row for the rest, which reads one part of it again
 * for the draw.  The middle two are shared by as many workgroups as fill the
 * chip, since one alone reads a row of 128256 in 10 us.
 *
 * At 128256 tokens (kernel times): 128 rows with filters of their own 11 us for
 * the largest logits (65.7 MB at 5.8 TB/s, what a copy reaches), 27 for the
 * histograms (bound by the 64-bit LDS atomics, one a token: 60 cycles a wave
 * of them; with half the vector instructions it took 25 instead of 27), 18 for
 * the lists (65.7 MB again) and 24 for the rest, 80 us together; one row 4, 7, 9 and 19
 * us, bound by the memory latencies and barriers one after the other.
 */
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gq_device.h"
#include "gq_internal.h"

namespace {

constexpr int kT = 1024, kW = kT / GQ_WAVE;
constexpr int kMaxVocab = 1 << 20;
constexpr int kTopT = 256, kTop = 4096;        /* threads and tokens of a workgroup of the first launch */
constexpr int kBins = 512, kLast = kBins - 2;  /* a part's histogram; min_p moves what it leaves out one bin on */
constexpr int kFine = 2048;                    /* bins of eleven bits */
constexpr int kChunks = 16;
constexpr int kShare = 512;                    /* tokens of the border's bin that a wave can list */
constexpr int kList = kW * kShare;
constexpr int kRows = 512;                     /* rows a launch: 43 MB of workspace at most */

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct Part { /* what a part of a row leaves for the last launch */
  unsigned long long mass[kBins]; /* of bins 0 .. this one */
  uint32_t cnt[kBins];            /* tokens of them */
  unsigned long long kept; /* mass of what min_p keeps, for rows without top-k and top-p */
  int pass;                /* the last bin that min_p keeps */
  int pad;
};

struct Border { /* of a row, by the third launch */
  unsigned long long mass[kBins]; /* of bins 0 .. this one of the whole row */
  unsigned long long base, ahead; /* before the border's bin: the count (top-k) or mass, and the mass */
  int bin, from; /* bins from .. bin are listed */
  int pass;
  int pad;
};

struct SampArgs {
  const float *x;
  const float *temperature, *top_p, *min_p, *rnd;
  const int32_t *top_k;
  int32_t *tokens;
  float *logprobs;
  uint64_t *tops;
  Part *parts;
  Border *borders;
  uint64_t *lists; /* [row][lister][kList] */
  int *counts;     /* [row][lister]: -1, if they did not fit */
  int vocab, n_tops, chunks, chunk; /* chunk: tokens a part, a multiple of 4 */
  int listers;                      /* workgroups a row of the third launch */
  long long stride;
  int S; /* w is held in units of 2^-S */
};

/* order of the logits as an unsigned integer, -0 as +0; 0 for what is never
 * picked (-infinity, NaN) */
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v == 0.f ? 0.f : v);
  return v > -INFINITY ? ((u & 0x80000000u) ? ~u : (u | 0x80000000u)) : 0u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __builtin_bit_cast(float, (key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}
/* (logit, index): a larger one comes first */
__device__ __forceinline__ uint64_t comp_of(float v, int i) {
  return (uint64_t)key_of(v) << 32 | (uint32_t)~i;
}

template <class T, class F>
__device__ __forceinline__ T wave_reduce(T v, F f) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = f(v, (T)__shfl_xor(v, o, 64));
  return v;
}
/* running sums over the lanes: within rows of 16 by row_shr 1, 2, 4 and 8, then
 * row 0's and 2's last to the row behind, then the second row's to the last two */
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long dpp_add(unsigned long long v) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
  return v + ((unsigned long long)(uint32_t)hi << 32 | (uint32_t)lo);
}
__device__ __forceinline__ unsigned long long wave_scan(unsigned long long v) {
  v = dpp_add<0x111, 0xf>(v), v = dpp_add<0x112, 0xf>(v), v = dpp_add<0x114, 0xf>(v), v = dpp_add<0x118, 0xf>(v);
  return dpp_add<0x143, 0xc>(dpp_add<0x142, 0xa>(v));
}
__device__ __forceinline__ unsigned long long last_lane(unsigned long long v) {
  return (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ unsigned long long wave_sum(unsigned long long v) { return last_lane(wave_scan(v)); }

/* use(f(v, i)) for the tokens i of [lo, hi) in some order: four neighbours a
 * thread at a time, U such loads in flight, their f side by side; lo is a
 * multiple of 4 */
template <int U, class F, class G>
__device__ __forceinline__ void tokens(const float *x, int lo, int hi, int threads, int tid, F f, G use) {
  int i = lo + 4 * tid;
  for (; i + 4 * (U - 1) * threads + 3 < hi; i += 4 * U * threads) {
    f32x4u v[U];
#pragma unroll
    for (int u = 0; u < U; u++) v[u] = *(const f32x4u *)(x + i + 4 * u * threads);
    decltype(f(0.f, 0)) r[4 * U];
#pragma unroll
    for (int u = 0; u < 4 * U; u++) r[u] = f(v[u / 4][u & 3], i + 4 * (u / 4) * threads + (u & 3));
#pragma unroll
    for (int u = 0; u < 4 * U; u++) use(r[u]);
  }
  for (; i < hi; i += 4 * threads) {
    if (i + 3 < hi) {
      const f32x4u v = *(const f32x4u *)(x + i);
#pragma unroll
      for (int e = 0; e < 4; e++) use(f(v[e], i + e));
    } else {
      for (int e = i; e < hi; e++) use(f(x[e], e));
    }
  }
}
template <int U, class F>
__device__ __forceinline__ void tokens(const float *x, int lo, int hi, int threads, int tid, F f) {
  struct None {};
  tokens<U>(x, lo, hi, threads, tid, [&](float v, int i) { return f(v, i), None{}; }, [](None) {});
}

/* 2^(S + i / 64) to tab, by the first wave */
__device__ __forceinline__ void table(double *tab, int S) {
  if (threadIdx.x < 64) tab[threadIdx.x] = __builtin_ldexp(exp2((double)threadIdx.x / 64), S);
}
/* a b + c with c in scalar registers: the compiler copies it to others first */
__device__ __forceinline__ double fma_s(double a, double b, double c) {
  double d;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "s"(c));
  return d;
}

/* a row's parameters: read before its largest logit is waited for */
struct Params {
  float T, p, min_p;
  int k;
  __device__ Params(const SampArgs &a, long long r)
      : T(a.temperature ? a.temperature[r] : 1.f), p(a.top_p ? a.top_p[r] : 1.f), min_p(a.min_p ? a.min_p[r] : 0.f),
        k(a.top_k ? a.top_k[r] : 0) {}
};
/* and what follows from them */
struct Row {
  float top, T, min_p, scale;
  int k;
  bool inf, by_k, by_p;
  float p;
  double c;   /* e^((v - top) / T) = 2^((v - top) c / 64) */
  double low; /* min_p keeps (v - top) c from here on */
  const double *tab;

  __device__ Row(const SampArgs &a, const Params &q, uint64_t first, const double *t) : T(q.T), k(q.k), p(q.p), tab(t) {
    min_p = q.min_p > 0.f ? fminf(q.min_p, 1.f) : 0.f;
    if (p <= 0.f) k = 1, p = 1.f;
    by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
    top = value_of((uint32_t)(first >> 32));
    inf = top == INFINITY; /* such a row's infinities weigh 1, the others nothing */
    if (inf) top = 0.f;
    c = 92.332482616893656877 / (double)T; /* 64 / ln 2 */
    low = min_p > 0.f ? 64.0 * log2((double)min_p) : -INFINITY;
    /* the last bin takes what weighs nothing in units of 2^-S */
    scale = fminf((float)(kLast / ((a.S + 1.5) * 0.6931471805599453)) / T, 3e38f);
  }
  __device__ float see(float v) const { return inf ? (v == INFINITY ? 0.f : -INFINITY) : v; }
  __device__ double y(float v) const { return ((double)v - (double)top) * c; }
  __device__ bool passes(float v) const { return y(v) >= low; }
  /* bins in descending order of the logits, none of which mixes what min_p
   * keeps with what it does not: that goes one bin on */
  __device__ int bin0(float v) const { return (int)fminf((top - v) * scale, (float)kLast); }
  __device__ int bin(float v) const { return bin0(v) + (min_p > 0.f && !passes(v)); }
  /* logits between which all of bins b0 .. b1 lie, and some others: the bin's
   * arithmetic is off by 2^-22 of (top - v) and of top at most */
  __device__ void bounds(int b0, int b1, float &lo, float &hi) const {
    const float d1 = (float)(b1 + 1) / scale, d0 = (float)(b0 - 1) / scale, more = 1e-6f * fabsf(top) + 1e-43f;
    hi = top;
    lo = b1 < kLast && d1 < 1e38f ? fmaxf(top - d1 * 1.000001f - more, -3.402823466e38f) : -3.402823466e38f;
    if (b0 > 1 && d0 < 1e38f) hi = fminf(top - d0 * 0.999999f + more, top);
  }
  /* e^((v - top) / T) in units of 2^-S, nearest even.  2^((k + f) / 64): 2^(k /
   * 64) from the table, e^(f ln 2 / 64) by its series to the fifth power (the
   * next term is below 2^-54), and 2^52 added: the low bits are the number. */
  __device__ unsigned long long mass(float v) const {
    const double t = fmax(y(v), -4096.0), n = t + 0x1.8p52, f = t - (n - 0x1.8p52); /* 2^-64 is nothing */
    double s = fma_s(f, 0x1.5d87fe78a6731p-40 /* (ln 2 / 64)^5 / 120 */, 0x1.3b2ab6fba4e77p-31);
    s = fma_s(f, s, 0x1.c6b08d704a0c0p-23);
    s = fma_s(f, s, 0x1.ebfbdff82c58fp-15);
    s = fma_s(f, s, 0x1.62e42fefa39efp-7);
    const int i = (int)__builtin_bit_cast(uint64_t, n);
    const uint64_t e = __builtin_bit_cast(uint64_t, tab[i & 63]);
    const double b = __builtin_bit_cast(double, e + ((uint64_t)(uint32_t)((i >> 6) << 20) << 32));
    return __builtin_bit_cast(unsigned long long, __builtin_fma(b * f, s, b) + 0x1p52) & 0xfffffffffffffull;
  }
};

/* the largest (logit, index) of every kTop tokens */
__global__ __launch_bounds__(kTopT) void tops_kernel(SampArgs a) {
  __shared__ uint64_t sh[kTopT / GQ_WAVE];
  const int tid = threadIdx.x, lo = blockIdx.x * kTop, hi = min(a.vocab, lo + kTop);
  const long long row = blockIdx.y;
  float top = -INFINITY;
  int at = -1;
  tokens<kTop / kTopT / 4>(a.x + row * a.stride, lo, hi, kTopT, tid, [&](float v, int i) {
    if (v > top) top = v, at = i;
  });
  const auto larger = [](uint64_t p, uint64_t q) { return p > q ? p : q; };
  const uint64_t w = wave_reduce(at < 0 ? 0 : comp_of(top, at), larger);
  if ((tid & 63) == 0) sh[tid >> 6] = w;
  __syncthreads();
  if (tid == 0) {
    uint64_t m = sh[0];
    for (int i = 1; i < kTopT / GQ_WAVE; i++) m = larger(m, sh[i]);
    a.tops[row * a.n_tops + blockIdx.x] = m;
  }
}

/* the row's largest, to every thread; *to is LDS */
__device__ __forceinline__ uint64_t first_of(const SampArgs &a, long long row, uint64_t *to) {
  if (threadIdx.x < GQ_WAVE) {
    uint64_t m = 0;
    for (int i = threadIdx.x; i < a.n_tops; i += GQ_WAVE) m = max(m, a.tops[row * a.n_tops + i]);
    m = wave_reduce(m, [](uint64_t p, uint64_t q) { return p > q ? p : q; });
    if (threadIdx.x == 0) *to = m;
  }
  __syncthreads();
  return *to;
}

/* the histogram of a part of a row, or only the sum of what it keeps */
__global__ __launch_bounds__(kT, 8) void parts_kernel(SampArgs a) {
  __shared__ double tab[64];
  __shared__ uint64_t first;
  __shared__ unsigned long long mass[kBins], kept;
  __shared__ uint32_t cnt[kBins];
  __shared__ int pass;
  __shared__ unsigned long long wm[kBins / GQ_WAVE];
  __shared__ uint32_t wc[kBins / GQ_WAVE];
  const int tid = threadIdx.x;
  const long long r = blockIdx.y;
  table(tab, a.S);
  for (int i = tid; i < kBins; i += kT) mass[i] = 0, cnt[i] = 0;
  if (tid == 0) kept = 0, pass = -1;
  const Params q(a, r);
  const uint64_t f = first_of(a, r, &first);
  const Row row(a, q, f, tab);
  if (!f || !(row.T > 0.f)) return;
  const int lo = min(a.vocab, (int)blockIdx.x * a.chunk), hi = min(a.vocab, lo + a.chunk);
  const float *x = a.x + r * a.stride;
  Part &to = a.parts[r * a.chunks + blockIdx.x];
  if (!row.by_k && !row.by_p) {
    unsigned long long s = 0;
    tokens<2>(x, lo, hi, kT, tid, [&](float v, int) {
      v = row.see(v);
      const unsigned long long m = row.mass(v);
      s += row.passes(v) ? m : 0;
    });
    s = wave_sum(s);
    if ((tid & 63) == 0) atomicAdd(&kept, s);
    __syncthreads();
    if (tid == 0) to.kept = kept;
    return;
  }
  int last = -1;
  struct Token {
    unsigned long long m;
    int b;
  };
  const auto fill = [&](auto min_p, auto count) {
    tokens<1>(
        x, lo, hi, kT, tid,
        [&](float v, int) {
          v = row.see(v);
          const bool in = !min_p || row.passes(v);
          const int b = row.bin0(v) + !in;
          if (min_p) last = max(last, in ? b : -1);
          return Token{row.mass(v), v > -INFINITY ? b : -1};
        },
        [&](Token t) {
          if (t.b < 0) return;
          atomicAdd(&mass[t.b], t.m);
          if (count) atomicAdd(&cnt[t.b], 1u);
        });
  };
  constexpr std::true_type yes;
  constexpr std::false_type no;
  if (row.min_p > 0.f) row.by_k ? fill(yes, yes) : fill(yes, no);
  else row.by_k ? fill(no, yes) : fill(no, no);
  if (last >= 0) atomicMax(&pass, last);
  __syncthreads();
  unsigned long long m = 0, n = 0;
  if (tid < kBins) {
    m = wave_scan(mass[tid]), n = wave_scan(cnt[tid]);
    if ((tid & 63) == 63) wm[tid >> 6] = m, wc[tid >> 6] = (uint32_t)n;
  }
  __syncthreads();
  if (tid < kBins) {
#pragma unroll
    for (int w = 0; w < kBins / GQ_WAVE - 1; w++)
      if (w < tid >> 6) m += wm[w], n += wc[w];
    to.mass[tid] = m, to.cnt[tid] = (uint32_t)n;
  }
  if (tid == 0) to.pass = pass;
}

struct Shared {
  double tab[64];
  unsigned long long mass[kFine];
  uint32_t cnt[kFine];
  uint64_t list[kList];
  unsigned long long wsum[kW], chunk[kChunks];
  uint64_t first;
  unsigned long long before, in;
  int at, last;
  uint32_t n;
};

__device__ unsigned long long block_sum(Shared &sh, unsigned long long s) {
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sh.wsum[threadIdx.x >> 6] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int w = 0; w < kW; w++) s += sh.wsum[w];
  __syncthreads();
  return s;
}

/* The first bin at which the running sum, `base` included, reaches the target
 * (or the last bin, if none does): its number to sh.at, the sum before it to
 * sh.before, its own mass to sh.in, its count to sh.n.  By count, or by mass. */
__device__ void find_bin(Shared &sh, bool count, unsigned long long base, double target) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const unsigned long long a = count ? sh.cnt[2 * tid] : sh.mass[2 * tid];
  const unsigned long long b = count ? sh.cnt[2 * tid + 1] : sh.mass[2 * tid + 1];
  const unsigned long long s = wave_scan(a + b);
  if (lane == 63) sh.wsum[wave] = s;
  __syncthreads();
  unsigned long long off = base;
#pragma unroll
  for (int w = 0; w < kW - 1; w++) off += w < wave ? sh.wsum[w] : 0;
  const unsigned long long c0 = off + s - a - b, c1 = c0 + a, c2 = c1 + b;
  if (!((double)c0 >= target) || tid == 0) {
    const int at = (double)c1 >= target ? 2 * tid : (double)c2 >= target || tid == kT - 1 ? 2 * tid + 1 : -1;
    if (at >= 0) sh.at = at, sh.before = at & 1 ? c1 : c0, sh.in = sh.mass[at], sh.n = sh.cnt[at];
  }
  __syncthreads();
}

/* tokens i .. i + 3, those before `to` */
__device__ __forceinline__ f32x4u four(const float *x, int i, int to) {
  if (i + 3 < to) return *(const f32x4u *)(x + i);
  f32x4u v;
#pragma unroll
  for (int e = 0; e < 4; e++) v[e] = i + e < to ? x[i + e] : -INFINITY;
  return v;
}

/* The tokens lo .. hi - 1 (lo a multiple of 4) of bins b0 .. b1, and a few of
 * the next ones, to each wave's own share of a list; returns how many a wave
 * has, of which the first kShare are listed.  Two compares a token: what a
 * workgroup reads bounds it (10 us for 513 KB by one of them). */
template <int U>
__device__ __forceinline__ int list_tokens(const Row &row, const float *x, int lo, int hi, int b0, int b1, uint64_t *list) {
  constexpr int D = 4 * kT;
  float vlo, vhi;
  row.bounds(b0, b1, vlo, vhi);
  int n = 0;
  for (int b = lo; b < hi; b += U * D) {
    const int i = b + 4 * threadIdx.x;
    f32x4u v[U];
    if (b + U * D <= hi) {
#pragma unroll
      for (int u = 0; u < U; u++) v[u] = *(const f32x4u *)(x + i + u * D);
    } else {
#pragma unroll
      for (int u = 0; u < U; u++) v[u] = four(x, i + u * D, hi);
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
      uint64_t hit[4], any = 0;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if (row.inf) v[u][e] = row.see(v[u][e]);
        hit[e] = __ballot(v[u][e] >= vlo && v[u][e] <= vhi), any |= hit[e];
      }
      if (any)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int j = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(hit[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit[e], 0));
          if (v[u][e] >= vlo && v[u][e] <= vhi && j < kShare) list[j] = comp_of(v[u][e], i + u * D + e);
          n += __builtin_popcountll(hit[e]);
        }
    }
  }
  return n;
}

/* a row's border of top-k, or else of top-p: its bin, and the tokens of it
 * among the parts that a workgroup looks through */
__global__ __launch_bounds__(kT) void list_kernel(SampArgs a) {
  __shared__ struct {
    unsigned long long mass[kBins];
    uint32_t cnt[kBins];
    uint64_t list[kList], first;
    int at, n[kW];
  } sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long r = blockIdx.y;
  const Part *parts = a.parts + r * a.chunks;
  const Params q(a, r);
  const uint64_t first = first_of(a, r, &sh.first);
  const Row row(a, q, first, nullptr);
  if (!first || !(row.T > 0.f) || !(row.by_k || row.by_p)) return;
  /* the histogram of the whole row */
  unsigned long long m0 = 0;
  uint32_t c0 = 0;
  const int end = a.chunks - 1;
  if (tid < kBins) {
    unsigned long long m[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; c++) m[c] = parts[min(c, end)].mass[tid];
#pragma unroll
    for (int c = 0; c < kChunks; c++) m0 += c <= end ? m[c] : 0;
  } else if (row.by_k) {
    uint32_t m[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; c++) m[c] = parts[min(c, end)].cnt[tid - kBins];
#pragma unroll
    for (int c = 0; c < kChunks; c++) c0 += c <= end ? m[c] : 0;
  }
  static_assert(kT == 2 * kBins, "sums and counts are each half of the threads'");
  if (tid < kBins) sh.mass[tid] = m0;
  else sh.cnt[tid - kBins] = c0;
  if (tid == 0) sh.at = kBins;
  __syncthreads();
  const double target = row.by_k ? (double)row.k : (double)row.p * (double)sh.mass[kBins - 1];
  if (tid < kBins) {
    const unsigned long long upto = row.by_k ? sh.cnt[tid] : sh.mass[tid];
    const unsigned long long before = tid == 0 ? 0 : row.by_k ? sh.cnt[tid - 1] : sh.mass[tid - 1];
    if ((double)upto >= target && (tid == 0 || !((double)before >= target))) sh.at = tid;
  }
  __syncthreads();
  /* a bin of mass 0: what is left weighs nothing.  With top-p to come, the
   * bins before top-k's border too, if they fit: top-p's is among them */
  int bin = sh.at;
  if (bin < kBins && sh.mass[bin] == (bin ? sh.mass[bin - 1] : 0)) bin = kBins;
  const unsigned long long ahead = bin ? sh.mass[bin - 1] : 0;
  const unsigned long long base = !row.by_k ? ahead : bin && bin < kBins ? sh.cnt[bin - 1] : 0;
  const int from = bin < kBins && row.by_k && row.by_p && sh.cnt[bin] <= kList / 2 ? 0 : bin;
  Border &to = a.borders[r];
  if (blockIdx.x == 0) {
    if (tid < kBins) to.mass[tid] = m0;
    if (wave == 0) {
      int pass = row.min_p > 0.f && lane < a.chunks ? parts[lane].pass : -1;
      pass = wave_reduce(pass, [](int p, int q) { return max(p, q); });
      if (lane == 0) to.base = base, to.ahead = ahead, to.bin = bin, to.from = from, to.pass = pass;
    }
  }
  int n = 0;
  const int per = (a.chunks + a.listers - 1) / a.listers * a.chunk;
  const int lo = min(a.vocab, (int)blockIdx.x * per), hi = min(a.vocab, lo + per);
  if (bin < kBins) n = list_tokens<8>(row, a.x + r * a.stride, lo, hi, from, bin, sh.list + wave * kShare);
  if (lane == 0) sh.n[wave] = n;
  __syncthreads();
  int at = 0, all = 0;
  bool fits = true;
#pragma unroll
  for (int w = 0; w < kW; w++) {
    const int m = sh.n[w];
    at += w < wave ? m : 0, all += m, fits = fits && m <= kShare;
  }
  const long long l = r * a.listers + blockIdx.x;
  if (tid == 0) a.counts[l] = fits ? all : -1;
  if (fits)
    for (int j = lane; j < n; j += GQ_WAVE) a.lists[l * kList + at + j] = sh.list[wave * kShare + j];
}

__global__ __launch_bounds__(kT) void draw_kernel(SampArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocab;
  const long long r = blockIdx.x;
  const float *x = a.x + r * a.stride;
  const Part *parts = a.parts + r * a.chunks;
  table(sh.tab, a.S);
  const Params q(a, r);
  const uint64_t first = first_of(a, r, &sh.first);
  const Row row(a, q, first, sh.tab);
  if (!first || !(row.T > 0.f)) { /* nothing to pick, or greedy */
    if (tid == 0) {
      a.tokens[r] = first ? (int)~(uint32_t)first : -1;
      if (a.logprobs) a.logprobs[r] = first ? 0.f : -INFINITY;
    }
    return;
  }
  int border = kBins, pass = row.min_p > 0.f ? -1 : kBins;
  uint64_t cut = 0; /* tokens with a smaller (logit, index) are left out */
  /* the tokens of bins b0 .. b1 (and a few of the next ones), if they fit LDS:
   * every wave's own share of them */
  int b0 = 1, b1 = 0, n = 0;
  bool listed = false;
  const uint64_t *list = sh.list;
  const auto gather = [&](int bin) {
    b0 = b1 = bin, list = sh.list + wave * kShare;
    n = list_tokens<2>(row, x, 0, V, bin, bin, sh.list + wave * kShare);
    if (tid == 0) sh.n = 0;
    __syncthreads();
    if (lane == 0 && n > kShare) sh.n = 1;
    __syncthreads();
    listed = !sh.n;
    __syncthreads();
  };
  /* f(v, comp) for the tokens of a bin with comp >= cut */
  const auto each = [&](int bin, auto f) {
    if (listed) {
      for (int j = lane; j < n; j += GQ_WAVE) {
        const uint64_t c = list[j];
        const float v = value_of((uint32_t)(c >> 32));
        if (c >= cut && row.bin(v) == bin) f(v, c);
      }
    } else {
      float vlo, vhi;
      row.bounds(bin, bin, vlo, vhi);
      tokens<1>(x, 0, V, kT, tid, [&](float v, int i) {
        v = row.see(v);
        if (!(v >= vlo && v <= vhi)) return;
        const uint64_t c = comp_of(v, i);
        if (c >= cut && row.bin(v) == bin) f(v, c);
      });
    }
  };
  if (row.by_k || row.by_p) {
    const Border &bd = a.borders[r];
    const unsigned long long upto = tid < kBins ? bd.mass[tid] : 0; /* of bins 0 .. tid */
    unsigned long long whole = bd.mass[kBins - 1];                  /* mass of what top-k keeps */
    if (row.min_p > 0.f) pass = bd.pass;
    { /* the third launch's lists, one behind the other */
      const int m = lane < a.listers ? a.counts[r * a.listers + lane] : 0;
      listed = !__ballot(m < 0);
      int sum = listed ? m : 0;
#pragma unroll
      for (int o = 1; o < kChunks; o <<= 1) {
        const int u = __shfl_up(sum, o, 64);
        if (lane >= o) sum += u;
      }
      const int all = __builtin_amdgcn_readlane(sum, kChunks - 1);
      listed = listed && all <= kList;
      if (listed) {
        const int l = wave % a.listers, by = kW / a.listers, k = __builtin_amdgcn_readlane(m, l);
        const int from = l ? __builtin_amdgcn_readlane(sum, l - 1) : 0;
        if (wave / a.listers < by)
          for (int j = wave / a.listers * GQ_WAVE + lane; j < k; j += by * GQ_WAVE)
            sh.list[from + j] = a.lists[(r * a.listers + l) * kList + j];
        const int share = (all + kW - 1) / kW, at = min(all, wave * share);
        list = sh.list + at, n = min(all - at, share);
        b0 = bd.from, b1 = bd.bin;
      }
      __syncthreads();
    }
    for (int by = row.by_k ? 0 : 1; by < (row.by_p ? 2 : 1); by++) {
      const bool count = by == 0;
      const double target = count ? (double)row.k : (double)row.p * (double)whole;
      int bin = bd.bin;
      unsigned long long base = bd.base; /* count or mass before the border's bin */
      if (!count && row.by_k) { /* the histogram of what top-k keeps */
        if (tid < kBins) sh.mass[tid] = tid < border ? upto : whole;
        if (tid == 0) sh.at = kBins - 1;
        __syncthreads();
        if (tid < kBins && (double)sh.mass[tid] >= target && (tid == 0 || !((double)sh.mass[tid - 1] >= target))) sh.at = tid;
        __syncthreads();
        bin = sh.at, base = bin ? sh.mass[bin - 1] : 0;
      }
      unsigned long long above = bd.ahead, in = 0; /* mass before it; of the border itself */
      if (count && bin == kBins) { /* what is left weighs nothing */
        whole = above;
        continue;
      }
      if (!listed || bin < b0 || bin > b1) gather(bin);
      /* eleven bits of (logit, index) at a time, after those that all share */
      float vlo, vhi;
      row.bounds(bin, bin, vlo, vhi);
      const uint32_t klo = key_of(vlo), khi = key_of(vhi);
      int shift = klo == khi ? 32 : 64 - __builtin_clz(klo ^ khi);
      uint64_t prefix = shift < 64 ? ((uint64_t)klo << 32) >> shift : 0;
      uint32_t left = 2;
      while (left > 1 && shift > 0) {
        const int bits = min(11, shift), mask = (1 << bits) - 1;
        shift -= bits;
        __syncthreads();
        for (int i = tid; i < kFine; i += kT) sh.cnt[i] = 0, sh.mass[i] = 0;
        __syncthreads();
        each(bin, [&](float v, uint64_t c) {
          if (shift + bits < 64 && c >> (shift + bits) != prefix) return;
          const int d = mask - ((int)(c >> shift) & mask); /* the largest first */
          atomicAdd(&sh.cnt[d], 1u);
          atomicAdd(&sh.mass[d], row.mass(v));
        });
        __syncthreads();
        find_bin(sh, count, base, target);
        const int at = sh.at;
        if (count) {
          unsigned long long s = 0;
          for (int i = tid; i < at; i += kT) s += sh.mass[i];
          above += block_sum(sh, s);
        }
        base = sh.before, left = sh.n, in = sh.in;
        prefix = prefix << bits | (uint64_t)(mask - at);
      }
      if (count) whole = above + in;
      /* the border's token, the only one left */
      uint64_t token = prefix;
      if (shift) {
        __syncthreads();
        each(bin, [&](float, uint64_t c) {
          if (c >> shift == prefix) sh.first = c;
        });
        __syncthreads();
        token = sh.first;
      }
      cut = token;
      border = bin;
      __syncthreads();
    }
  }
  /* the kept mass of every part */
  if (tid < a.chunks) {
    const int end = min(border, pass + 1);
    sh.chunk[tid] = !(row.by_k || row.by_p) ? parts[tid].kept : end ? parts[tid].mass[end - 1] : 0;
  }
  __syncthreads();
  if (border <= pass && border < kBins) {
    each(border, [&](float v, uint64_t c) { atomicAdd(&sh.chunk[(int)(~(uint32_t)c) / a.chunk], row.mass(v)); });
    __syncthreads();
  }
  unsigned long long whole = 0, before = 0;
  for (int c = 0; c < a.chunks; c++) whole += sh.chunk[c];
  const double target = (double)a.rnd[r] * (double)whole;
  int slice = -1, last = 0;
  for (int c = 0; c < a.chunks && slice < 0; c++) {
    if (!sh.chunk[c]) continue;
    last = c;
    if ((double)(before + sh.chunk[c]) > target) slice = c;
    else before += sh.chunk[c];
  }
  const bool none = slice < 0; /* rnd 1 or more, or not a number: the last one */
  if (none) slice = last;
  /* within the part: groups of 256 tokens (more, if there were more than kT of them) */
  const int lo = slice * a.chunk, hi = min(V, lo + a.chunk);
  const int size = 256 * ((hi - lo + 256 * kT - 1) / (256 * kT));
  const auto kept = [&](float v, int i) -> unsigned long long {
    v = row.see(v);
    const unsigned long long m = row.mass(v); /* 0 for what is never picked */
    return comp_of(v, i) >= cut && row.passes(v) ? m : 0;
  };
  sh.mass[tid] = 0;
  __syncthreads();
  constexpr int G = 2; /* groups that a wave reads at once */
  for (int g = wave; lo + g * size < hi; g += G * kW) {
    unsigned long long s[G] = {};
    for (int at = 4 * lane; at < size; at += 256) {
      f32x4u v[G];
#pragma unroll
      for (int u = 0; u < G; u++) v[u] = four(x, lo + (g + u * kW) * size + at, hi);
#pragma unroll
      for (int u = 0; u < G; u++)
#pragma unroll
        for (int e = 0; e < 4; e++) s[u] += kept(v[u][e], lo + (g + u * kW) * size + at + e);
    }
#pragma unroll
    for (int u = 0; u < G; u++) {
      const unsigned long long t = wave_sum(s[u]);
      if (lane == 0 && t) sh.mass[g + u * kW] = t;
    }
  }
  if (tid == 0) sh.at = kT, sh.last = 0;
  __syncthreads();
  const unsigned long long own = sh.mass[tid], sum = wave_scan(own);
  if (lane == 63) sh.wsum[wave] = sum;
  __syncthreads();
  unsigned long long at = before + sum;
#pragma unroll
  for (int w = 0; w < kW - 1; w++) at += w < wave ? sh.wsum[w] : 0;
  const uint64_t over = __ballot(own && (double)at > target), any = __ballot(own != 0);
  if (lane == 0) {
    if (over) atomicMin(&sh.at, tid + __builtin_ctzll(over));
    if (any) atomicMax(&sh.last, tid + 63 - __builtin_clzll(any));
  }
  __syncthreads();
  const int group = none ? sh.last : sh.at;
  if (tid == group) sh.before = at - own;
  __syncthreads();
  if (wave) return;
  at = sh.before;
  const int from = lo + group * size, to = min(hi, from + size);
  int token = -1;
  for (int b = from; b < to && (none || token < 0); b += 256) {
    const int i = b + 4 * lane;
    const f32x4u v = four(x, i, to);
    unsigned long long m[4], s = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) m[e] = kept(v[e], i + e), s += m[e];
    const unsigned long long c = wave_scan(s);
    unsigned long long run = at + c - s;
    int mine = -1;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      run += m[e];
      if (m[e] && (none || ((double)run > target && mine < 0))) mine = i + e;
    }
    const uint64_t hit = __ballot(mine >= 0);
    if (hit) token = __builtin_amdgcn_readlane(mine, none ? 63 - __builtin_clzll(hit) : __builtin_ctzll(hit));
    at += last_lane(c);
  }
  if (lane == 0) {
    a.tokens[r] = token;
    if (a.logprobs) {
      const double all = log((double)whole * __builtin_ldexp(1.0, -a.S));
      const float v = row.see(x[token]);
      a.logprobs[r] = (float)(v == row.top ? -all : ((double)v - (double)row.top) / (double)row.T - all);
    }
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
  SampArgs a{};
  a.vocab = vocab, a.stride = row_stride, a.S = std::min(51, 62 - bits);
  a.n_tops = (vocab + kTop - 1) / kTop;
  const int batch = std::min(rows, kRows);
  /* parts: enough workgroups for the chip, each with 4096 tokens or more */
  const int most = std::min(kChunks, (vocab + 4095) / 4096);
  a.chunks = std::max(1, std::min(most, 1024 / batch));
  a.chunk = ((vocab + a.chunks - 1) / a.chunks + 3) / 4 * 4;
  a.listers = std::max(1, std::min(a.chunks, 256 / batch));
  const size_t lists = (size_t)batch * a.listers;
  const size_t sizes[] = {sizeof(Part) * batch * a.chunks, sizeof(Border) * batch, sizeof(uint64_t) * batch * a.n_tops,
                          sizeof(uint64_t) * kList * lists, sizeof(int) * lists};
  size_t bytes = 0;
  for (size_t n : sizes) bytes += n;
  char *ws = (char *)gq_ctx_paged_ws(c, bytes);
  if (!ws) return gq_ctx_fail(c, -4, "sample_rows: workspace");
  a.parts = (Part *)ws, ws += sizes[0];
  a.borders = (Border *)ws, ws += sizes[1];
  a.tops = (uint64_t *)ws, ws += sizes[2];
  a.lists = (uint64_t *)ws, ws += sizes[3];
  a.counts = (int *)ws;
  for (int r = 0; r < rows; r += batch) {
    const int n = std::min(batch, rows - r);
    a.x = logits + (long long)r * row_stride;
    a.temperature = temperature ? temperature + r : nullptr;
    a.top_k = top_k ? top_k + r : nullptr;
    a.top_p = top_p ? top_p + r : nullptr;
    a.min_p = min_p ? min_p + r : nullptr;
    a.rnd = rnd + r, a.tokens = tokens + r;
    a.logprobs = logprobs ? logprobs + r : nullptr;
    hipLaunchKernelGGL(tops_kernel, dim3(a.n_tops, n), dim3(kTopT), 0, ci.stream, a);
    hipLaunchKernelGGL(parts_kernel, dim3(a.chunks, n), dim3(kT), 0, ci.stream, a);
    hipLaunchKernelGGL(list_kernel, dim3(a.listers, n), dim3(kT), 0, ci.stream, a);
    hipLaunchKernelGGL(draw_kernel, dim3(n), dim3(kT), 0, ci.stream, a);
  }
  return hipGetLastError() == hipSuccess ? 0 : gq_ctx_fail(c, -4, "sample_rows launch");
}
