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
 * Three launches: the largest logit of every 4096 tokens; the histograms of
 * `chunks` parts of each row; one workgroup a row for the borders and the draw,
 * which reads the row once more for the border's bin (tokens between two
 * logits: a compare each) and one part of it for the draw.
 */
#include <algorithm>
#include <cmath>

#include "gq_device.h"
#include "gq_internal.h"

namespace {

constexpr int kT = 1024, kW = kT / GQ_WAVE;
constexpr int kMaxVocab = 1 << 20;
constexpr int kTopT = 256, kTop = 4096;        /* threads and tokens of a workgroup of the first launch */
constexpr int kBins = 512, kLast = kBins - 2;  /* a part's histogram; min_p moves what it leaves out one bin on */
constexpr int kFine = 2048;                    /* bins of eleven bits */
constexpr int kChunks = 16;
constexpr int kList = 8192;                    /* tokens of the border's bin that fit LDS */
constexpr int kRows = 4096;                    /* rows a launch: 28 MB of workspace at most */

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

struct Part { /* what a part of a row leaves for the last launch */
  unsigned long long mass[kBins];
  uint32_t cnt[kBins];
  unsigned long long kept; /* mass of what min_p keeps, for rows without top-k and top-p */
  int pass;                /* the last bin that min_p keeps */
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
  int vocab, n_tops, chunks, chunk; /* chunk: tokens a part, a multiple of 4 */
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
__device__ __forceinline__ unsigned long long wave_sum(unsigned long long v) {
  return wave_reduce(v, [](unsigned long long a, unsigned long long b) { return a + b; });
}
__device__ __forceinline__ unsigned long long wave_scan(unsigned long long v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned long long u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

/* f(v, i) for the tokens i of [lo, hi) in some order: four neighbours a thread
 * at a time, U such loads in flight; lo is a multiple of 4 */
template <int U, class F>
__device__ __forceinline__ void tokens(const float *x, int lo, int hi, int threads, int tid, F f) {
  int i = lo + 4 * tid;
  for (; i + 4 * (U - 1) * threads + 3 < hi; i += 4 * U * threads) {
    f32x4u v[U];
#pragma unroll
    for (int u = 0; u < U; u++) v[u] = *(const f32x4u *)(x + i + 4 * u * threads);
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
      for (int e = 0; e < 4; e++) f(v[u][e], i + 4 * u * threads + e);
  }
  for (; i < hi; i += 4 * threads) {
    if (i + 3 < hi) {
      const f32x4u v = *(const f32x4u *)(x + i);
#pragma unroll
      for (int e = 0; e < 4; e++) f(v[e], i + e);
    } else {
      for (int e = i; e < hi; e++) f(x[e], e);
    }
  }
}

/* 2^(i / 64) to tab, by the first wave */
__device__ __forceinline__ void table(double *tab) {
  if (threadIdx.x < 64) tab[threadIdx.x] = exp2((double)threadIdx.x / 64);
}

/* a row's parameters and what follows from them alone */
struct Row {
  float top, T, min_p, scale;
  int k, S;
  bool inf, by_k, by_p;
  float p;
  double c;   /* e^((v - top) / T) = 2^((v - top) c / 64) */
  double low; /* min_p keeps (v - top) c from here on */
  const double *tab;

  __device__ Row(const SampArgs &a, long long r, uint64_t first, const double *t) : tab(t) {
    T = a.temperature ? a.temperature[r] : 1.f;
    k = a.top_k ? a.top_k[r] : 0;
    p = a.top_p ? a.top_p[r] : 1.f;
    min_p = a.min_p ? a.min_p[r] : 0.f;
    min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
    if (p <= 0.f) k = 1, p = 1.f;
    by_k = k > 0 && k < a.vocab, by_p = p < 1.f;
    top = value_of((uint32_t)(first >> 32));
    inf = top == INFINITY; /* such a row's infinities weigh 1, the others nothing */
    if (inf) top = 0.f;
    S = a.S;
    c = 92.332482616893656877 / (double)T; /* 64 / ln 2 */
    low = min_p > 0.f ? 64.0 * log2((double)min_p) : -INFINITY;
    /* the last bin takes what weighs nothing in units of 2^-S */
    scale = (float)(kLast / ((a.S + 1.5) * 0.6931471805599453)) / T;
  }
  __device__ float see(float v) const { return inf ? (v == INFINITY ? 0.f : -INFINITY) : v; }
  __device__ double y(float v) const { return ((double)v - (double)top) * c; }
  __device__ bool passes(float v) const { return y(v) >= low; }
  /* bins in descending order of the logits, none of which mixes what min_p
   * keeps with what it does not: that goes one bin on */
  __device__ int bin(float v) const {
    const int b = v == top ? 0 : (int)fminf((top - v) * scale, (float)kLast);
    return min_p > 0.f && !passes(v) ? b + 1 : b;
  }
  /* e^((v - top) / T) in units of 2^-S, nearest even.  2^((k + f) / 64): 2^(k /
   * 64) from the table, e^(f ln 2 / 64) by its series to the fifth power (the
   * next term is below 2^-54), and 2^52 added: the low bits are the number. */
  __device__ unsigned long long mass(float v) const {
    const double t = fmax(y(v), -4096.0); /* 2^-64 is nothing */
    const double n = __builtin_rint(t), f = t - n;
    double s = __builtin_fma(f, 0x1.5d87fe78a6731p-40 /* (ln 2 / 64)^5 / 120 */, 0x1.3b2ab6fba4e77p-31);
    s = __builtin_fma(f, s, 0x1.c6b08d704a0c0p-23);
    s = __builtin_fma(f, s, 0x1.ebfbdff82c58fp-15);
    s = __builtin_fma(f, s, 0x1.62e42fefa39efp-7);
    const int i = (int)n;
    const double b = tab[i & 63];
    s = __builtin_ldexp(__builtin_fma(b * f, s, b), (i >> 6) + S);
    return __builtin_bit_cast(unsigned long long, s + 0x1p52) & 0xfffffffffffffull;
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
__global__ __launch_bounds__(kT) void parts_kernel(SampArgs a) {
  __shared__ double tab[64];
  __shared__ uint64_t first;
  __shared__ unsigned long long mass[kBins], kept;
  __shared__ uint32_t cnt[kBins];
  __shared__ int pass;
  const int tid = threadIdx.x;
  const long long r = blockIdx.y;
  table(tab);
  for (int i = tid; i < kBins; i += kT) mass[i] = 0, cnt[i] = 0;
  if (tid == 0) kept = 0, pass = -1;
  const uint64_t f = first_of(a, r, &first);
  const Row row(a, r, f, tab);
  if (!f || !(row.T > 0.f)) return;
  const int lo = min(a.vocab, (int)blockIdx.x * a.chunk), hi = min(a.vocab, lo + a.chunk);
  const float *x = a.x + r * a.stride;
  Part &to = a.parts[r * a.chunks + blockIdx.x];
  if (!row.by_k && !row.by_p) {
    unsigned long long s = 0;
    tokens<2>(x, lo, hi, kT, tid, [&](float v, int) {
      v = row.see(v);
      if (row.min_p == 0.f || row.passes(v)) s += row.mass(v);
    });
    s = wave_sum(s);
    if ((tid & 63) == 0) atomicAdd(&kept, s);
    __syncthreads();
    if (tid == 0) to.kept = kept;
    return;
  }
  int last = -1;
  tokens<2>(x, lo, hi, kT, tid, [&](float v, int) {
    v = row.see(v);
    if (!(v > -INFINITY)) return;
    const int b = row.bin(v);
    if (row.min_p > 0.f && b > last && row.passes(v)) last = b;
    atomicAdd(&mass[b], row.mass(v));
    if (row.by_k) atomicAdd(&cnt[b], 1u);
  });
  if (last >= 0) atomicMax(&pass, last);
  __syncthreads();
  for (int i = tid; i < kBins; i += kT) to.mass[i] = mass[i], to.cnt[i] = cnt[i];
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
  for (int w = 0; w < wave; w++) off += sh.wsum[w];
  const unsigned long long c0 = off + s - a - b, c1 = c0 + a, c2 = c1 + b;
  if (!((double)c0 >= target) || tid == 0) {
    const int at = (double)c1 >= target ? 2 * tid : (double)c2 >= target || tid == kT - 1 ? 2 * tid + 1 : -1;
    if (at >= 0) sh.at = at, sh.before = at & 1 ? c1 : c0, sh.in = sh.mass[at], sh.n = sh.cnt[at];
  }
  __syncthreads();
}

__global__ __launch_bounds__(kT) void draw_kernel(SampArgs a) {
  __shared__ Shared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocab;
  const long long r = blockIdx.x;
  const float *x = a.x + r * a.stride;
  const Part *parts = a.parts + r * a.chunks;
  table(sh.tab);
  const uint64_t first = first_of(a, r, &sh.first);
  const Row row(a, r, first, sh.tab);
  if (!first || !(row.T > 0.f)) { /* nothing to pick, or greedy */
    if (tid == 0) {
      a.tokens[r] = first ? (int)~(uint32_t)first : -1;
      if (a.logprobs) a.logprobs[r] = first ? 0.f : -INFINITY;
    }
    return;
  }
  int border = kBins, pass = row.min_p > 0.f ? -1 : kBins;
  uint64_t cut = 0; /* tokens with a smaller (logit, index) are left out */
  /* the listed logits: keys klo .. khi */
  uint32_t klo = 1, khi = 0, n = 0;
  bool listed = false;
  /* the lowest key of bins 0 .. b: a search of 64 keys at a time */
  const auto lowest = [&](int b) {
    uint32_t lo = key_of(-3.402823466e38f), hi = key_of(row.top);
    while (lo < hi) {
      const uint32_t step = (hi - lo) / 64 + 1;
      const uint64_t u = (uint64_t)lo + (uint64_t)lane * step;
      const uint64_t in = __ballot(u >= hi || row.bin(value_of((uint32_t)u)) <= b);
      const int f = in ? __builtin_ctzll(in) : 64;
      const uint64_t up = (uint64_t)lo + (uint64_t)f * step;
      if (f) lo = lo + (uint32_t)(f - 1) * step + 1;
      hi = f == 0 ? lo : (uint32_t)min(up, (uint64_t)hi);
    }
    return hi;
  };
  /* the tokens of bins b0 .. b1 to the list, if they fit */
  const auto gather = [&](int b0, int b1) {
    khi = b0 ? lowest(b0 - 1) - 1 : key_of(row.top), klo = lowest(b1);
    const float vlo = value_of(klo), vhi = value_of(khi);
    __syncthreads();
    if (tid == 0) sh.n = 0;
    __syncthreads();
    const auto put = [&](float v, int i) {
      v = row.see(v);
      if (v >= vlo && v <= vhi) {
        const uint32_t j = atomicAdd(&sh.n, 1u);
        if (j < (uint32_t)kList) sh.list[j] = comp_of(v, i);
      }
    };
    tokens<4>(x, 0, V, kT, tid, put);
    __syncthreads();
    n = sh.n, listed = n <= (uint32_t)kList;
    __syncthreads();
  };
  /* f(comp) for the kept ones of the listed tokens with c0 <= comp <= c1 */
  const auto each = [&](uint64_t c0, uint64_t c1, auto f) {
    if (listed) {
      for (uint32_t j = tid; j < n; j += kT) {
        const uint64_t c = sh.list[j];
        if (c >= c0 && c <= c1) f(c);
      }
    } else {
      tokens<1>(x, 0, V, kT, tid, [&](float v, int i) {
        v = row.see(v);
        const uint64_t c = comp_of(v, i);
        if (v > -INFINITY && c >= c0 && c <= c1) f(c);
      });
    }
  };
  if (row.by_k || row.by_p) {
    /* bin t of the whole row is thread t's */
    unsigned long long m0 = 0, c0 = 0;
    if (tid < kBins) {
      for (int c = 0; c < a.chunks; c++) m0 += parts[c].mass[tid];
      if (row.by_k)
        for (int c = 0; c < a.chunks; c++) c0 += parts[c].cnt[tid];
    }
    if (row.min_p > 0.f)
      for (int c = 0; c < a.chunks; c++) pass = max(pass, parts[c].pass);
    for (int i = tid; i < kFine; i += kT) sh.mass[i] = i < kBins ? m0 : 0, sh.cnt[i] = i < kBins ? (uint32_t)c0 : 0;
    __syncthreads();
    unsigned long long whole = 0; /* mass of what top-k keeps */
    for (int by = 0; by < 2; by++) {
      const bool count = by == 0;
      if (count ? !row.by_k : !row.by_p) {
        if (count) whole = block_sum(sh, m0);
        continue;
      }
      const double target = count ? (double)row.k : (double)row.p * (double)whole;
      find_bin(sh, count, 0, target);
      const int bin = sh.at;
      unsigned long long base = sh.before, in = sh.in; /* count or mass before the border's bin, its own mass */
      const uint32_t below = sh.n;
      const unsigned long long ahead = count ? block_sum(sh, tid < bin ? m0 : 0) : 0;
      unsigned long long above = ahead; /* mass before it */
      if (in == 0) { /* what is left weighs nothing */
        whole = above;
        continue;
      }
      /* the bins before it too, if they fit: top-p looks among them next */
      const uint32_t lo = lowest(bin), hi = bin ? lowest(bin - 1) - 1 : key_of(row.top);
      if (!listed || lo < klo || hi > khi) gather(count && row.by_p && base + below <= (uint64_t)kList ? 0 : bin, bin);
      const uint64_t lo64 = max(cut, (uint64_t)lo << 32), hi64 = (uint64_t)hi << 32 | 0xffffffffu;
      /* eleven bits of (logit, index) at a time, after those that all share */
      int shift = lo == hi ? 32 : 64 - __builtin_clz(lo ^ hi);
      uint64_t prefix = shift < 64 ? lo64 >> shift : 0;
      uint32_t left = 2;
      while (left > 1 && shift > 0) {
        const int bits = min(11, shift), mask = (1 << bits) - 1;
        shift -= bits;
        __syncthreads();
        for (int i = tid; i < kFine; i += kT) sh.cnt[i] = 0, sh.mass[i] = 0;
        __syncthreads();
        each(lo64, hi64, [&](uint64_t c) {
          if (shift + bits < 64 && c >> (shift + bits) != prefix) return;
          const int d = mask - ((int)(c >> shift) & mask); /* the largest first */
          atomicAdd(&sh.cnt[d], 1u);
          atomicAdd(&sh.mass[d], row.mass(value_of((uint32_t)(c >> 32))));
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
      cut = prefix;
      if (shift) {
        __syncthreads();
        each(lo64, hi64, [&](uint64_t c) {
          if (c >> shift == prefix) sh.first = c;
        });
        __syncthreads();
        cut = sh.first;
      }
      border = bin;
      __syncthreads();
      if (count && row.by_p) { /* the histogram of what top-k keeps */
        for (int i = tid; i < kFine; i += kT) sh.mass[i] = i < bin ? m0 : i == bin ? whole - ahead : 0;
        __syncthreads();
      }
    }
  }
  /* the kept mass of every part */
  unsigned long long part = 0;
  if (wave < a.chunks) {
    if (row.by_k || row.by_p) {
      const int end = min(border, pass + 1);
      for (int b = lane; b < end; b += GQ_WAVE) part += parts[wave].mass[b];
      part = wave_sum(part);
    } else {
      part = parts[wave].kept;
    }
  }
  if (lane == 0 && wave < kChunks) sh.chunk[wave] = part;
  __syncthreads();
  if (border <= pass && border < kBins) {
    const uint64_t hi64 = (uint64_t)(border ? lowest(border - 1) - 1 : key_of(row.top)) << 32 | 0xffffffffu;
    each(cut, hi64, [&](uint64_t c) {
      atomicAdd(&sh.chunk[(int)(~(uint32_t)c) / a.chunk], row.mass(value_of((uint32_t)(c >> 32))));
    });
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
    return v > -INFINITY && comp_of(v, i) >= cut && (row.min_p == 0.f || row.passes(v)) ? row.mass(v) : 0ull;
  };
  for (int g = wave; g < kT; g += kW) {
    const int from = lo + g * size;
    unsigned long long s = 0;
    if (from < hi) {
      tokens<1>(x, from, min(hi, from + size), GQ_WAVE, lane, [&](float v, int i) { s += kept(v, i); });
      s = wave_sum(s);
    }
    if (lane == 0) sh.mass[g] = s;
  }
  if (tid == 0) sh.at = kT, sh.last = 0;
  __syncthreads();
  const unsigned long long own = sh.mass[tid], sum = wave_scan(own);
  if (lane == 63) sh.wsum[wave] = sum;
  __syncthreads();
  unsigned long long at = before + sum;
  for (int w = 0; w < wave; w++) at += sh.wsum[w];
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
  for (int b = from; b < to && (none || token < 0); b += GQ_WAVE) {
    const int i = b + lane;
    const unsigned long long m = i < to ? kept(x[i], i) : 0ull, c = wave_scan(m);
    const uint64_t hit = __ballot(m && (none || (double)(at + c) > target));
    if (hit) token = b + (none ? 63 - __builtin_clzll(hit) : __builtin_ctzll(hit));
    at += __shfl(c, 63, 64);
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
  a.chunks = std::max(1, std::min(most, 512 / batch));
  a.chunk = ((vocab + a.chunks - 1) / a.chunks + 3) / 4 * 4;
  const size_t parts = sizeof(Part) * batch * a.chunks, tops = sizeof(uint64_t) * batch * a.n_tops;
  char *ws = (char *)gq_ctx_paged_ws(c, parts + tops);
  if (!ws) return gq_ctx_fail(c, -4, "sample_rows: workspace");
  a.parts = (Part *)ws, a.tops = (uint64_t *)(ws + parts);
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
    hipLaunchKernelGGL(draw_kernel, dim3(n), dim3(kT), 0, ci.stream, a);
  }
  return hipGetLastError() == hipSuccess ? 0 : gq_ctx_fail(c, -4, "sample_rows launch");
}
