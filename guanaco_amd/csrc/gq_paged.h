/*
 * gq_paged.h — what the kernels over the paged K/V cache share
 * (gq_paged.hip, gq_paged_prompt.hip).
 */
#ifndef GQ_PAGED_H
#define GQ_PAGED_H

#include "gq_device.h"
#include "gq_internal.h"

typedef float gq_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 gq_bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 gq_bf16x8 __attribute__((ext_vector_type(8)));

/* gq_pages and gq_batch as the kernels take them */
struct PgdPages {
  uint8_t *k, *v;
  float *ks, *vs;
  int n_pages, lg, n_kv; /* 1 << lg positions a page */
};
struct PgdBatch {
  const int32_t *table, *pos, *first;
  int n_seqs, stride, n_tokens, max_len;
};

constexpr int pgd_bytes(int dtype) { return dtype == GQ_F32 ? 4 : dtype == GQ_BF16 ? 2 : 1; }

/* The sequence of packed row t (uniform in the wave, all lanes active): the
 * last s with first[s] <= t, so that the row lies before first[s + 1]; n_seqs
 * where it belongs to none.  64 sequences a step. */
__device__ __forceinline__ int pgd_seq_of(const PgdBatch &b, int t) {
  if (!b.first) return t < b.n_seqs ? t : b.n_seqs;
  const int lane = threadIdx.x & 63;
  for (int s0 = 0; s0 < b.n_seqs; s0 += GQ_WAVE) {
    const int s = s0 + lane;
    const uint64_t after = __ballot(s < b.n_seqs && gld<int>(b.first + min(s, b.n_seqs - 1) + 1) > t);
    if (after) return s0 + __builtin_ctzll(after);
  }
  return b.n_seqs;
}

/* Positions before the call's tokens.  None from max_len on exists, so that a
 * larger number says no more than max_len; the sum with a token's number, 0 to
 * n_tokens - 1, then stays within 31 bits (max_len and n_tokens are 2^30 at
 * most).  With n_tokens itself it need not: pgd_len. */
__device__ __forceinline__ int pgd_before(const PgdBatch &b, int pos) { return min(pos, b.max_len); }
/* positions that exist once n tokens follow `before` ones (< 0: an idle slot) */
__host__ __device__ __forceinline__ int pgd_len(int before, int n, int max_len) {
  return before < 0 ? 0 : before < max_len - n ? before + n : max_len;
}

/* (row of the first new token, their number) of a sequence, s uniform in the
 * wave; none where the rows are not in the packed arrays */
__device__ __forceinline__ int2 pgd_rows(const PgdBatch &b, int s) {
  if (!b.first) return make_int2(s, s < b.n_tokens ? 1 : 0);
  const int r0 = gq_sld<int>(b.first + s), r1 = gq_sld<int>(b.first + s + 1);
  return r0 < 0 || r1 > b.n_tokens || r1 <= r0 ? make_int2(0, 0) : make_int2(r0, r1 - r0);
}

/* Page of position p of sequence s; -1: it does not exist. */
__device__ __forceinline__ int pgd_page(const PgdPages &c, const PgdBatch &b, int s, int p) {
  const int i = p >> c.lg;
  if (p < 0 || p >= b.max_len || i >= b.stride) return -1;
  const int page = gld<int>(b.table + (size_t)s * b.stride + i);
  return (unsigned)page < (unsigned)c.n_pages ? page : -1;
}
/* The same through the scalar cache, s and p uniform in the wave. */
__device__ __forceinline__ int pgd_page_u(const PgdPages &c, const PgdBatch &b, int s, int p) {
  const int i = p >> c.lg;
  if (p < 0 || p >= b.max_len || i >= b.stride) return -1;
  const int page = gq_sld<int>(b.table + (size_t)s * b.stride + i);
  return (unsigned)page < (unsigned)c.n_pages ? page : -1;
}
/* row of (page, head, slot) in a pool */
__device__ __forceinline__ size_t pgd_row(const PgdPages &c, int page, int head, int slot) {
  return (((size_t)page * c.n_kv + head) << c.lg) + slot;
}

/* two floats to bf16, nearest even */
__device__ __forceinline__ uint32_t pgd_pack(float x, float y) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2){x, y}, gq_bf16x2));
}
__device__ __forceinline__ float pgd_lo(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float pgd_hi(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }

/* eight consecutive values of GQ_F32 or GQ_BF16, and back */
template <int T>
__device__ __forceinline__ void pgd_load8(const void *base, size_t at, float (&x)[8]) {
  if constexpr (T == GQ_F32) {
    const float4 a = gld<float4>((const float *)base + at), b = gld<float4>((const float *)base + at + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 w = gld<uint4>((const uint16_t *)base + at);
    x[0] = pgd_lo(w.x), x[1] = pgd_hi(w.x), x[2] = pgd_lo(w.y), x[3] = pgd_hi(w.y);
    x[4] = pgd_lo(w.z), x[5] = pgd_hi(w.z), x[6] = pgd_lo(w.w), x[7] = pgd_hi(w.w);
  }
}
template <int T>
__device__ __forceinline__ void pgd_store8(void *base, size_t at, const float (&x)[8]) {
  if constexpr (T == GQ_F32) {
    gst<float4>((float *)base + at, make_float4(x[0], x[1], x[2], x[3]));
    gst<float4>((float *)base + at + 4, make_float4(x[4], x[5], x[6], x[7]));
  } else {
    gst<uint4>((uint16_t *)base + at, make_uint4(pgd_pack(x[0], x[1]), pgd_pack(x[2], x[3]), pgd_pack(x[4], x[5]), pgd_pack(x[6], x[7])));
  }
}

/* stores past the caches (the `nt` policy): whole lines that no wave reads again */
template <class T>
__device__ __forceinline__ void gst_nt(void *p, T v) {
  typedef typename gq_native<sizeof(T)>::type N;
  __builtin_nontemporal_store(__builtin_bit_cast(N, v), (GQ_GLOBAL N *)p);
}

/* byte i of a dword as a signed integer */
__device__ __forceinline__ float i8f(uint32_t w, int i) { return (float)(int8_t)(w >> (8 * i)); }

/* x = hi + mid + lo exactly, bf16 each, for pairs */
__device__ __forceinline__ void split3(float x, float y, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
  hi = pgd_pack(x, y);
  x -= pgd_lo(hi), y -= pgd_hi(hi);
  mid = pgd_pack(x, y);
  x -= pgd_lo(mid), y -= pgd_hi(mid);
  lo = pgd_pack(x, y);
}
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], gq_bf16x8 (&out)[N]) {
  uint4 p[3];
  split3(x[0], x[1], p[0].x, p[1].x, p[2].x);
  split3(x[2], x[3], p[0].y, p[1].y, p[2].y);
  split3(x[4], x[5], p[0].z, p[1].z, p[2].z);
  split3(x[6], x[7], p[0].w, p[1].w, p[2].w);
#pragma unroll
  for (int i = 0; i < N; i++) out[i] = __builtin_bit_cast(gq_bf16x8, p[i]);
}

/* eight int8 codes as bf16, exactly */
__device__ __forceinline__ gq_bf16x8 codes8(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(gq_bf16x8, make_uint4(pgd_pack(i8f(a, 0), i8f(a, 1)), pgd_pack(i8f(a, 2), i8f(a, 3)),
                                                  pgd_pack(i8f(b, 0), i8f(b, 1)), pgd_pack(i8f(b, 2), i8f(b, 3))));
}

/* HIP counts a launch's threads in 32 bits */
inline bool pgd_launchable(long long blocks, int threads) { return blocks * threads < (1ll << 32); }

/* An output that an infinity or NaN of V has reached is NaN, whatever the order
 * and the parts that its weight came in made of it: infinity here, NaN there. */
__device__ __forceinline__ float pgd_finite(float y) { return __builtin_fmaf(y, 0.f, y); }

constexpr int kMaxG = 16; /* query heads per KV head */

/* attention of new tokens over the cache */
struct AttArgs {
  PgdPages c;
  PgdBatch b;
  const void *q;
  void *out;
  float *part_o, *part_ml; /* [row][head][nch][hd] and [..][2] */
  int n_heads, G, qs, os;
  int nch, chunk; /* at most nch parts, of at most `chunk` keys (decode: a multiple of 128) or blocks of 64 keys */
  float scale;    /* log2(e) / sqrt(head_dim) */
};

/* What a workgroup of the prompt kernel has in LDS: blocks of 64 keys, 32 RG
 * query rows, a wave with 64 / KH keys of every block. */
constexpr int kKeys = 64;
template <int CT, int XT, int HD, int RG, int KH>
struct PromptLds {
  /* bf16 planes of Q or P and of K or V */
  static constexpr int NX = XT == GQ_F32 ? 3 : 1, NK = CT != GQ_F32 ? 1 : NX == 3 ? 3 : 2;
  static constexpr int NB = NK < 3 ? 2 : 1;       /* blocks */
  static constexpr bool CODES = CT == GQ_I8_ROWS; /* the scales apart */
  static constexpr int KPL = kKeys * HD * 2;      /* bytes of one plane */
  static constexpr int QLO = NB * 2 * NK * KPL;   /* the third plane of Q; the others are in registers */
  static constexpr int SCL = QLO + (NX == 3 ? RG * (HD / 16) * 1024 : 0);
  static constexpr int USED = SCL + (CODES ? (4 + NB) * kKeys * 4 : 0); /* scales: four blocks of K's, NB of V's */
  /* the halves' exchange at the end, from 0 on: (m, l, O) of a lane */
  static constexpr int EXCHANGE = KH == 2 ? RG * 64 * 4 * (HD / 32 * 16 + 2) : 0;
  /* a flag per wave, read when other waves have begun the exchange: behind it */
  static constexpr int ODD = USED > EXCHANGE ? USED : EXCHANGE;
  static constexpr int BYTES = ODD + 32;
  static_assert(ODD % 16 == 0 && BYTES <= 160 * 1024, "flags are read 16 bytes at a time; LDS of a CU");
};

/* gq_paged_prompt.hip: every new token's attention.  The shape of its launch:
 * rows of a tile, blocks of 64 keys a part, at most so many parts (more than
 * one: part_o and part_ml hold n_tokens rows), workgroups (0: too many). */
struct PromptShape {
  int rows, span, parts;
  unsigned blocks;
};
PromptShape gq_paged_prompt_shape(const AttArgs &a, int cache, int xtype, int head_dim, int n_cu);
int gq_launch_paged_prompt(const AttArgs &a, int cache, int xtype, int head_dim, const PromptShape &f, hipStream_t s);

#endif
