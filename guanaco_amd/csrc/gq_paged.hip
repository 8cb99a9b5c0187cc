/*
 * gq_paged.hip — a K/V cache in pages that many sequences share: rows appended
 * and read back, and attention over them (gfx950).
 *
 * append: a row of head_dim values (a query head, or K or V of a KV head) is
 * HD / 8 lanes of eight values, so that every load and store is 16 bytes a lane
 * and the row's largest magnitude, for int8, is a DPP reduction.  Rotation is
 * the framework's: fl(fl(x0 c) - fl(x1 s)), fl(fl(x0 s) + fl(x1 c)).
 *
 * attention: see the kernels.
 */
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gq_paged.h"

namespace {

constexpr int kThreads = 256;

/* ------------------------------------------------------- append and read */
struct AppendArgs {
  PgdPages c;
  PgdBatch b;
  const void *q, *k, *v;
  void *q_out;
  const float *rope;
  int n_heads, qs, qos, ks, vs, nq; /* nq: query rows a token, 0 without q */
};

/* maximum over a row's HD / 8 lanes */
template <int HD>
__device__ __forceinline__ float row_max(float m) {
  m = fmaxf(m, gq_dpp<0x141>(m)); /* row_half_mirror: within 8 */
  m = fmaxf(m, gq_dpp<0x4e>(m));
  m = fmaxf(m, gq_dpp<0xb1>(m));
  if (HD == 128) m = fmaxf(m, gq_dpp<0x140>(m)); /* row_mirror: the other eight */
  return m;
}

/* round(y / d) to nearest even as if the quotient were exact: the candidate
 * from the rounded one is off by one at most, and the sign of y - (c +- 1/2) d,
 * which one fused operation gives exactly, says so. */
__device__ __forceinline__ int quant(float y, float d) {
  float c = __builtin_rintf(y / d);
  const float up = __builtin_fmaf(-(c + 0.5f), d, y), dn = __builtin_fmaf(-(c - 0.5f), d, y);
  const bool odd = ((int)c & 1) != 0;
  if (up > 0.f || (up == 0.f && odd)) c += 1.f;
  else if (dn < 0.f || (dn == 0.f && odd)) c -= 1.f;
  return (int)fminf(fmaxf(c, -127.f), 127.f);
}

/* Where the rows of a wave are: U times RPW of the `per` rows of each packed
 * token, one of them this lane's.  Rows are counted in tiles of 16 tokens, token
 * after token for one head and then the next head: a wave's rows are neighbours
 * in a page, their scales too.  Memory bounds both kernels on long batches: 8122
 * tokens of 32 + 16 bf16 rows appended in 49 us (4.3 TB/s of reads and writes),
 * 32000 int8 rows of 8 heads read as fp32 in 49 (6.7 TB/s, four fifths of it
 * writes).  32 tokens of as many sequences take 5.7 and 4.1, trips to memory in
 * turn: the ends of 64 sequences, from the tile's first token's to a row's own one
 * by one (up to 16), then its position, its page and its rows.  Rows read are
 * stored past the caches (83 us if not).  Rows appended are not, since attention
 * reads them next: the append would take 44 us, reading 33 MB of them back 17
 * instead of 14. */
constexpr int kRowTile = 16;
template <int U>
struct Rows {
  int t[U], j[U];     /* token and which of its rows; t -1: none */
  int p[U], page[U];  /* position and page, -1: it does not exist */
};
template <int U, int RPW>
__device__ __forceinline__ bool find_rows(const PgdPages &c, const PgdBatch &b, int per, int sub_row, Rows<U> &o) {
  static_assert(kRowTile % (U * RPW) == 0, "a wave's rows are of one head's tile");
  const uint32_t w0 = (blockIdx.x * (uint32_t)(kThreads / GQ_WAVE) + (threadIdx.x >> 6)) * (uint32_t)(U * RPW);
  const uint32_t t0 = w0 / (uint32_t)(kRowTile * per) * kRowTile;
  if (t0 >= (uint32_t)b.n_tokens) return false; /* uniform in the wave */
  const int s0 = pgd_seq_of(b, __builtin_amdgcn_readfirstlane((int)t0));
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t r = w0 - t0 * per + u * RPW + sub_row;
    const int t = (int)(t0 + r % kRowTile);
    int s = s0, r1 = t + 1; /* the sequence's end */
    o.j[u] = (int)(r / kRowTile);
    if (t < b.n_tokens) {
      if (!b.first) s = t;
      else
        while (s < b.n_seqs && (r1 = gld<int>(b.first + s + 1)) <= t) s++;
    }
    const bool in = t < b.n_tokens && s < b.n_seqs;
    const int sc = in ? s : 0;
    const int r0 = b.first ? gld<int>(b.first + sc) : t, p0 = pgd_before(b, gld<int>(b.pos + sc));
    o.t[u] = in && r0 >= 0 && t >= r0 && r1 <= b.n_tokens ? t : -1; /* as pgd_rows has it */
    o.p[u] = o.t[u] < 0 || p0 < 0 ? -1 : p0 + (t - r0);
    o.page[u] = o.t[u] < 0 || o.p[u] < 0 ? -1 : pgd_page(c, b, sc, o.p[u]);
  }
  return true;
}

/* A lane's eight values of a row: dims 8 sub .. + 7, or with SPLIT 4 sub .. + 3
 * of either half, which makes every access of fp32 rows whole lines. */
template <int T, bool SPLIT, int HD>
__device__ __forceinline__ void load_row(const void *base, size_t at, int sub, float (&x)[8]) {
  if constexpr (!SPLIT) {
    pgd_load8<T>(base, at + 8 * sub, x);
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const size_t p = at + i * (HD / 2) + 4 * sub;
      if constexpr (T == GQ_F32) {
        const float4 w = gld<float4>((const float *)base + p);
        x[4 * i] = w.x, x[4 * i + 1] = w.y, x[4 * i + 2] = w.z, x[4 * i + 3] = w.w;
      } else {
        const uint2 w = gld<uint2>((const uint16_t *)base + p);
        x[4 * i] = pgd_lo(w.x), x[4 * i + 1] = pgd_hi(w.x), x[4 * i + 2] = pgd_lo(w.y), x[4 * i + 3] = pgd_hi(w.y);
      }
    }
  }
}
/* AWAY: past the caches */
template <int T, bool SPLIT, int HD, bool AWAY>
__device__ __forceinline__ void store_row(void *base, size_t at, int sub, const float (&x)[8]) {
  const auto put = [](auto *p, auto v) {
    if constexpr (AWAY) gst_nt(p, v);
    else gst(p, v);
  };
  if constexpr (!SPLIT) {
    static_assert(T == GQ_BF16, "fp32 rows are split");
    put((uint16_t *)base + at + 8 * sub, make_uint4(pgd_pack(x[0], x[1]), pgd_pack(x[2], x[3]), pgd_pack(x[4], x[5]), pgd_pack(x[6], x[7])));
  } else {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const size_t p = at + i * (HD / 2) + 4 * sub;
      if constexpr (T == GQ_F32) put((float *)base + p, make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]));
      else put((uint16_t *)base + p, make_uint2(pgd_pack(x[4 * i], x[4 * i + 1]), pgd_pack(x[4 * i + 2], x[4 * i + 3])));
    }
  }
}

template <int CT, int XT, int HD, bool WIDE>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a) {
#pragma clang fp contract(off)
  constexpr int LPR = HD / 8, RPW = GQ_WAVE / LPR; /* lanes a row, rows a wave */
  constexpr int U = WIDE ? kRowTile / RPW : 1;
  constexpr bool SPLIT = CT != GQ_BF16 || XT != GQ_BF16;
  const int sub = threadIdx.x % LPR;
  Rows<U> o;
  if (!find_rows<U, RPW>(a.c, a.b, a.nq + 2 * a.c.n_kv, (threadIdx.x & 63) / LPR, o)) return;
  float xs[U][8];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int t = o.t[u], j = o.j[u];
    if (t < 0) continue; /* the page may still be on its way */
    if (j < a.nq) load_row<XT, SPLIT, HD>(a.q, (size_t)t * a.qs + (size_t)j * HD, sub, xs[u]);
    else if (j < a.nq + a.c.n_kv) load_row<XT, SPLIT, HD>(a.k, (size_t)t * a.ks + (size_t)(j - a.nq) * HD, sub, xs[u]);
    else load_row<XT, SPLIT, HD>(a.v, (size_t)t * a.vs + (size_t)(j - a.nq - a.c.n_kv) * HD, sub, xs[u]);
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    if (o.page[u] < 0) continue;
    const int t = o.t[u], j = o.j[u], p = o.p[u];
    const bool isq = j < a.nq, isk = !isq && j < a.nq + a.c.n_kv;
    const int h = isq ? j : isk ? j - a.nq : j - a.nq - a.c.n_kv;
    float(&x)[8] = xs[u];
    if (a.rope && (isq || isk)) {
      const float *cs = a.rope + (size_t)p * HD + (SPLIT ? 4 : 8) * sub;
      const float4 c0 = gld<float4>(cs), c1 = gld<float4>(cs + (SPLIT ? HD / 2 : 4));
      const float c[4] = {c0.x, c0.z, c1.x, c1.z}, n[4] = {c0.y, c0.w, c1.y, c1.w};
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float e = x[2 * i], d = x[2 * i + 1];
        x[2 * i] = e * c[i] - d * n[i];
        x[2 * i + 1] = e * n[i] + d * c[i];
      }
    }
    if (isq) {
      store_row<XT, SPLIT, HD, false>(a.q_out, (size_t)t * a.qos + (size_t)h * HD, sub, x);
      continue;
    }
    const size_t row = pgd_row(a.c, o.page[u], h, p & ((1 << a.c.lg) - 1));
    uint8_t *pool = isk ? a.c.k : a.c.v;
    if constexpr (CT != GQ_I8_ROWS) {
      store_row<CT, SPLIT, HD, false>(pool, row * HD, sub, x);
    } else {
      float m = 0.f;
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 8; i++) m = fmaxf(m, __builtin_fabsf(x[i])), bad |= !(__builtin_fabsf(x[i]) < INFINITY);
      m = row_max<HD>(bad ? INFINITY : m);
      const bool lost = m == INFINITY;
      const float d = lost ? __builtin_nanf("") : m / 127.0f;
      int c[8];
#pragma unroll
      for (int i = 0; i < 8; i++) c[i] = lost || !(d > 0.f) ? 0 : quant(x[i], d);
      uint2 w;
      w.x = (uint32_t)(c[0] & 255) | (uint32_t)(c[1] & 255) << 8 | (uint32_t)(c[2] & 255) << 16 | (uint32_t)c[3] << 24;
      w.y = (uint32_t)(c[4] & 255) | (uint32_t)(c[5] & 255) << 8 | (uint32_t)(c[6] & 255) << 16 | (uint32_t)c[7] << 24;
      gst<uint32_t>(pool + row * HD + 4 * sub, w.x);
      gst<uint32_t>(pool + row * HD + HD / 2 + 4 * sub, w.y);
      if (sub == 0) gst<float>((isk ? a.c.ks : a.c.vs) + row, d);
    }
  }
}

struct ReadArgs {
  PgdPages c;
  PgdBatch b;
  void *k, *v;
  int ks, vs;
};


template <int CT, int XT, int HD, bool WIDE>
__global__ __launch_bounds__(kThreads) void read_kernel(ReadArgs a) {
  constexpr int LPR = HD / 8, RPW = GQ_WAVE / LPR;
  constexpr int U = WIDE ? kRowTile / RPW : 1;
  constexpr bool SPLIT = CT != GQ_BF16 || XT != GQ_BF16;
  const int sub = threadIdx.x % LPR;
  Rows<U> o;
  if (!find_rows<U, RPW>(a.c, a.b, 2 * a.c.n_kv, (threadIdx.x & 63) / LPR, o)) return;
  float x[U][8];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const bool isk = o.j[u] < a.c.n_kv;
    if (o.page[u] < 0) {
#pragma unroll
      for (int i = 0; i < 8; i++) x[u][i] = 0.f;
      continue;
    }
    const size_t row = pgd_row(a.c, o.page[u], isk ? o.j[u] : o.j[u] - a.c.n_kv, o.p[u] & ((1 << a.c.lg) - 1));
    const uint8_t *pool = isk ? a.c.k : a.c.v;
    if constexpr (CT != GQ_I8_ROWS) {
      load_row<CT, SPLIT, HD>(pool, row * HD, sub, x[u]);
    } else {
      const uint2 w = make_uint2(gld<uint32_t>(pool + row * HD + 4 * sub), gld<uint32_t>(pool + row * HD + HD / 2 + 4 * sub));
      const float d = gld<float>((isk ? a.c.ks : a.c.vs) + row);
#pragma unroll
      for (int i = 0; i < 4; i++) x[u][i] = i8f(w.x, i) * d, x[u][4 + i] = i8f(w.y, i) * d;
    }
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    if (o.t[u] < 0) continue;
    const bool isk = o.j[u] < a.c.n_kv;
    store_row<XT, SPLIT, HD, true>(isk ? a.k : a.v, (size_t)o.t[u] * (isk ? a.ks : a.vs) + (size_t)(isk ? o.j[u] : o.j[u] - a.c.n_kv) * HD, sub, x[u]);
  }
}

/* -------------------------------------------------------------- attention */
/* The row of sequence s's last new token and the positions it sees; false: no
 * token. */
__device__ __forceinline__ bool decode_row(const AttArgs &a, int s, int &row, int &len) {
  const int2 rn = pgd_rows(a.b, s);
  if (rn.y < 1) return false;
  row = rn.x + rn.y - 1;
  len = pgd_len(gq_sld<int>(a.b.pos + s), rn.y, a.b.max_len);
  return true;
}


/* Attention of one query token (its G heads of KV head g) over the keys of one
 * part, by four waves that take 32 (fp32 caches: 16) keys each in turn, every
 * one with an online softmax of its own, joined through LDS at the end.  The
 * matrix instructions do both products with the heads as columns:
 *   S^T = K Q^T   A = K rows straight from memory: lane (c, j) = (lane % 16,
 *                 lane / 16) holds key c, and the dims are dealt to the lane
 *                 groups j so that each reads 16 bytes at a time; B = the
 *                 queries, as exact sums of bf16 parts (three for fp32).  The
 *                 lane gets head c's scores of keys 4 j + r, r < 4.
 *   O^T += V^T P^T  B = the probabilities straight from that layout (in three
 *                 bf16 parts for fp32 results, two for bf16 ones); A = V rows
 *                 4 j + r, dims VD c .. VD c + VD - 1 as they lie in memory,
 *                 transposed four by four within the lane (v_perm): tile t's
 *                 row c is dim VD c + t.  The lane holds head c's outputs of
 *                 dims VD (4 j + r) + t, so the softmax's rescale stays in the
 *                 lane.
 * int8 codes are exact in bf16; K's scale multiplies the score, V's the
 * probability.  fp32 caches use the fp32 matrix instructions, which need no
 * transposition (one key a step).  Keys that do not exist are masked, and V's
 * rows there are zeroed: what stale memory holds cannot reach a sum.
 *
 * The cache's bytes bound it: 64 sequences of up to 8192 positions (bf16, 32
 * heads over 8 of 128, 998 MB) 175 us with the merge, 5.7 TB/s where a copy
 * reaches 5.2; one of 131072 (int8, 277 MB) 51 us.  One of 301 takes 7.2 us: a
 * launch, the trips to its row, page and keys, and five steps of 64 fp32 keys a
 * workgroup, each waiting for loads of the one before.  Eight waves a workgroup
 * were slower (64 sequences 250 us for 207 then). */
template <int CT, int XT, int HD>
__global__ __launch_bounds__(kThreads) void decode_kernel(AttArgs a) {
  constexpr int NW = kThreads / GQ_WAVE;
  constexpr int TK = CT == GQ_F32 ? 1 : 2;   /* 16-key tiles a step */
  constexpr int KL = HD * pgd_bytes(CT) / 64; /* 16-byte loads of a K row per lane */
  constexpr int VD = HD / 16;                /* dims of a V row per lane */
  constexpr int VW = VD * pgd_bytes(CT) / 4; /* dwords of them */
  constexpr int NQ = XT == GQ_F32 ? 3 : 1, NP = XT == GQ_F32 ? 3 : 2;
  __shared__ float sm[NW][kMaxG], sl[NW][kMaxG];
  __shared__ float so[NW][kMaxG][HD + 4];
  const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int bid = blockIdx.x;
  const int g = bid % a.c.n_kv;
  bid /= a.c.n_kv;
  /* Workgroups go round the chip's engines in turn: with parts in the same order
   * for every sequence, the ones that shorter sequences lack leave the same
   * engines idle (128 sequences to 2000: 146 us, 111 with the order turned; 64 to
   * 8192: 185, 175). */
  const int item = bid / a.nch, part = (int)(((unsigned)bid + item + item / 2) % (unsigned)a.nch);
  /* sequence, row and length */
  const int s = item;
  int row, len;
  if (!decode_row(a, s, row, len)) return;
  const int parts = max(1, (len + a.chunk - 1) / a.chunk);
  if (part >= parts) return;
  const int k1 = min(len, (part + 1) * a.chunk);
  const int ps = 1 << a.c.lg;

  /* queries: head c of this KV head's group, zero past it */
  const size_t qat = (size_t)row * a.qs + (size_t)(g * a.G + min(c, a.G - 1)) * HD;
  constexpr int NS = CT == GQ_F32 ? HD / 16 : HD / 32; /* slices of 4 (fp32) or 8 dims per lane */
  gq_bf16x8 qp[CT == GQ_F32 ? 1 : NS][NQ];
  float qf[CT == GQ_F32 ? NS : 1][4];
#pragma unroll
  for (int i = 0; i < NS; i++) {
    if constexpr (CT == GQ_F32) {
      float x[8];
      /* dims 16 i + 4 j .. + 3 */
      const size_t at = qat + 16 * i + 4 * j;
      if constexpr (XT == GQ_F32) {
        const float4 u = gld<float4>((const float *)a.q + at);
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
      } else {
        const uint2 u = gld<uint2>((const uint16_t *)a.q + at);
        x[0] = pgd_lo(u.x), x[1] = pgd_hi(u.x), x[2] = pgd_lo(u.y), x[3] = pgd_hi(u.y);
      }
#pragma unroll
      for (int e = 0; e < 4; e++) qf[i][e] = c < a.G ? x[e] : 0.f;
    } else {
      /* bf16: dims 32 i + 8 j .. + 7; int8: 64 (i / 2) + 16 j + 8 (i % 2) */
      const int d = CT == GQ_BF16 ? 32 * i + 8 * j : 64 * (i >> 1) + 16 * j + 8 * (i & 1);
      float x[8];
      pgd_load8<XT>(a.q, qat + d, x);
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = c < a.G ? x[e] : 0.f;
      split8<NQ>(x, qp[i]);
    }
  }

  uint4 kr[TK][KL];
  uint32_t vr[TK][4][VW];
  float4 kd[TK], vd[TK];
  int lim[TK], nlim[TK]; /* keys of the tile that exist; of the next step's */
  size_t base[TK];       /* the first row in the pool of the tile loaded last */
  auto find = [&](int kb) {
#pragma unroll
    for (int u = 0; u < TK; u++) {
      const int kt = kb + 16 * u, page = kt < k1 ? pgd_page_u(a.c, a.b, s, kt) : -1;
      nlim[u] = page < 0 ? 0 : min(16, k1 - kt);
      base[u] = pgd_row(a.c, max(page, 0), g, kt & (ps - 1)); /* of none: any row there is, masked */
    }
  };
  auto loadk = [&]() {
#pragma unroll
    for (int u = 0; u < TK; u++) {
      const uint8_t *kp = a.c.k + (base[u] + c) * (size_t)(HD * pgd_bytes(CT)) + 16 * j;
#pragma unroll
      for (int i = 0; i < KL; i++) kr[u][i] = gld_nt<uint4>(kp + 64 * i);
      if constexpr (CT == GQ_I8_ROWS) kd[u] = gld<float4>(a.c.ks + base[u] + 4 * j);
    }
  };
  auto loadv = [&]() {
#pragma unroll
    for (int u = 0; u < TK; u++) {
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const uint8_t *vp = a.c.v + (base[u] + 4 * j + r) * (size_t)(HD * pgd_bytes(CT)) + VW * 4 * c;
        if constexpr (VW == 1) {
          vr[u][r][0] = gld_nt<uint32_t>(vp);
        } else if constexpr (VW == 2) {
          const uint2 w = gld_nt<uint2>(vp);
          vr[u][r][0] = w.x, vr[u][r][1] = w.y;
        } else {
#pragma unroll
          for (int i = 0; i < VW / 4; i++) {
            const uint4 w = gld_nt<uint4>(vp + 16 * i);
            vr[u][r][4 * i] = w.x, vr[u][r][4 * i + 1] = w.y, vr[u][r][4 * i + 2] = w.z, vr[u][r][4 * i + 3] = w.w;
          }
        }
      }
      if constexpr (CT == GQ_I8_ROWS) vd[u] = gld<float4>(a.c.vs + base[u] + 4 * j);
    }
  };

  float m = -INFINITY, l = 0.f; /* l: this lane's keys only */
  gq_f32x4 o[VD];
#pragma unroll
  for (int t = 0; t < VD; t++) o[t] = gq_f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int STEP = 16 * TK * NW;
  /* One set of registers: the next step's K loads once the scores have read K,
   * its V once the products have read V.  The last step is one of its own:
   * loads under a condition in the loop leave registers undefined behind it,
   * and the compiler has then put other values over V still to be read. */
  auto step = [&](int kb, auto MORE) {
    constexpr bool more = decltype(MORE)::value;
#pragma unroll
    for (int u = 0; u < TK; u++) lim[u] = nlim[u];
    if constexpr (more) find(kb + STEP);
    float4 kdu[TK], vdu[TK];
#pragma unroll
    for (int u = 0; u < TK; u++) kdu[u] = kd[u], vdu[u] = vd[u];
    float p[TK][4], mb = -INFINITY;
#pragma unroll
    for (int u = 0; u < TK; u++) {
      gq_f32x4 st = gq_f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (CT == GQ_F32) {
        gq_f32x4 s1 = st;
#pragma unroll
        for (int i = 0; i < NS; i++) {
          const float kf[4] = {__builtin_bit_cast(float, kr[u][i].x), __builtin_bit_cast(float, kr[u][i].y),
                               __builtin_bit_cast(float, kr[u][i].z), __builtin_bit_cast(float, kr[u][i].w)};
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            st = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[i][e], st, 0, 0, 0);
            s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e + 1], qf[i][e + 1], s1, 0, 0, 0);
          }
        }
        st += s1;
      } else {
#pragma unroll
        for (int n = NQ - 1; n >= 0; n--)
#pragma unroll
          for (int i = 0; i < NS; i++) {
            gq_bf16x8 kk;
            if constexpr (CT == GQ_BF16) kk = __builtin_bit_cast(gq_bf16x8, kr[u][i]);
            else if (i & 1) kk = codes8(kr[u][i >> 1].z, kr[u][i >> 1].w);
            else kk = codes8(kr[u][i >> 1].x, kr[u][i >> 1].y);
            st = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, qp[i][n], st, 0, 0, 0);
          }
      }
      if constexpr (CT == GQ_I8_ROWS) st[0] *= kdu[u].x, st[1] *= kdu[u].y, st[2] *= kdu[u].z, st[3] *= kdu[u].w;
#pragma unroll
      for (int r = 0; r < 4; r++) {
        p[u][r] = 4 * j + r < lim[u] ? st[r] * a.scale : -INFINITY;
        mb = fmaxf(mb, p[u][r]);
      }
    }
    if constexpr (more) loadk();
    mb = fmaxf(mb, __shfl_xor(mb, 16, 64));
    mb = fmaxf(mb, __shfl_xor(mb, 32, 64));
    const float mn = fmaxf(m, mb), ms = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - ms);
    m = mn;
    float lb = 0.f;
#pragma unroll
    for (int u = 0; u < TK; u++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        p[u][r] = __builtin_amdgcn_exp2f(p[u][r] - ms);
        lb += p[u][r];
      }
    l = __builtin_fmaf(l, alpha, lb);
#pragma unroll
    for (int t = 0; t < VD; t++) o[t] *= alpha;
    /* rows that do not exist: their weight is 0, but 0 * NaN is not */
#pragma unroll
    for (int u = 0; u < TK; u++) {
      if (lim[u] < 16) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const bool there = 4 * j + r < lim[u];
#pragma unroll
          for (int i = 0; i < VW; i++) vr[u][r][i] = there ? vr[u][r][i] : 0u;
        }
        if constexpr (CT == GQ_I8_ROWS) {
          vdu[u].x = 4 * j < lim[u] ? vdu[u].x : 0.f, vdu[u].y = 4 * j + 1 < lim[u] ? vdu[u].y : 0.f;
          vdu[u].z = 4 * j + 2 < lim[u] ? vdu[u].z : 0.f, vdu[u].w = 4 * j + 3 < lim[u] ? vdu[u].w : 0.f;
        }
      }
    }
    if constexpr (CT == GQ_F32) {
#pragma unroll
      for (int r = 0; r < 4; r++)
#pragma unroll
        for (int t = 0; t < VD; t++)
          o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vr[0][r][t]), p[0][r], o[t], 0, 0, 0);
    } else {
      float x[8];
#pragma unroll
      for (int u = 0; u < TK; u++) {
        if constexpr (CT == GQ_I8_ROWS) p[u][0] *= vdu[u].x, p[u][1] *= vdu[u].y, p[u][2] *= vdu[u].z, p[u][3] *= vdu[u].w;
#pragma unroll
        for (int r = 0; r < 4; r++) x[4 * u + r] = p[u][r];
      }
      gq_bf16x8 pp[NP];
      split8<NP>(x, pp);
#pragma unroll
      for (int t = 0; t < VD; t++) {
        uint32_t w[4];
#pragma unroll
        for (int u = 0; u < TK; u++)
#pragma unroll
          for (int r = 0; r < 4; r += 2) {
            if constexpr (CT == GQ_BF16)
              w[2 * u + r / 2] = __builtin_amdgcn_perm(vr[u][r + 1][t / 2], vr[u][r][t / 2], t & 1 ? 0x07060302u : 0x05040100u);
            else
              w[2 * u + r / 2] = pgd_pack(i8f(vr[u][r][t / 4], t & 3), i8f(vr[u][r + 1][t / 4], t & 3));
          }
        const gq_bf16x8 vv = __builtin_bit_cast(gq_bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
#pragma unroll
        for (int n = NP - 1; n >= 0; n--) o[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, pp[n], o[t], 0, 0, 0);
      }
    }
    if constexpr (more) loadv();
  };
  int kb = part * a.chunk + 16 * TK * wave;
  if (kb < k1) {
    find(kb), loadk(), loadv();
    for (; kb + STEP < k1; kb += STEP) step(kb, std::true_type{});
    step(kb, std::false_type{});
  }
  /* the waves' results: head c, dims VD (4 j + r) + t */
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (j == 0) sm[wave][c] = m, sl[wave][c] = l;
#pragma unroll
  for (int r = 0; r < 4; r++)
#pragma unroll
    for (int t = 0; t < VD; t++) so[wave][c][VD * (4 * j + r) + t] = o[t][r];
  __syncthreads();
  for (int i = threadIdx.x; i < a.G * HD; i += kThreads) {
    const int h = i / HD, d = i % HD;
    float M = sm[0][h];
#pragma unroll
    for (int w = 1; w < NW; w++) M = fmaxf(M, sm[w][h]);
    const float ms = M == -INFINITY ? 0.f : M;
    float L = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w++) {
      const float e = __builtin_amdgcn_exp2f(sm[w][h] - ms);
      L = __builtin_fmaf(sl[w][h], e, L);
      y = __builtin_fmaf(so[w][h][d], e, y);
    }
    const int qh = g * a.G + h;
    if (parts == 1) {
      y = pgd_finite(L == 0.f ? y * 0.f : y / L); /* nothing seen: zeros */
      const size_t at = (size_t)row * a.os + (size_t)qh * HD + d;
      if constexpr (XT == GQ_F32) gst<float>((float *)a.out + at, y);
      else gst<uint16_t>((uint16_t *)a.out + at, (uint16_t)pgd_pack(y, y));
    } else {
      const size_t at = ((size_t)item * a.n_heads + qh) * a.nch + part;
      gst<float>(a.part_o + at * HD + d, y);
      if (d == 0) gst<float>(a.part_ml + 2 * at, M), gst<float>(a.part_ml + 2 * at + 1, L);
    }
  }
}

/* The parts of a token's keys: out = sum_c o_c 2^(m_c - M) / sum_c l_c 2^(m_c -
 * M), a workgroup per 32 dims of a head, eight lanes of four dims for each of
 * 32 parts at a time. */
template <int XT, int HD>
__global__ __launch_bounds__(kThreads) void merge_kernel(AttArgs a) {
  __shared__ float sacc[32][33], sL[32], sM[kThreads / GQ_WAVE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, sub = tid & 7, cg = tid >> 3;
  const int dg = blockIdx.x % (HD / 32), item = blockIdx.x / (HD / 32), s = item / a.n_heads, h = item % a.n_heads;
  int row, len;
  if (!decode_row(a, s, row, len)) return;
  const int parts = (len + a.chunk - 1) / a.chunk;
  if (parts <= 1) return; /* its one part has written the result */
  const size_t at = (size_t)item * a.nch;
  const float *ml = a.part_ml + 2 * at, *po = a.part_o + at * HD + 32 * dg + 4 * sub;
  float M = -INFINITY;
  for (int c = tid; c < parts; c += kThreads) M = fmaxf(M, gld<float>(ml + 2 * c));
  M = gq_wave_max(M);
  if (lane == 0) sM[wave] = M;
  __syncthreads();
  M = fmaxf(fmaxf(sM[0], sM[1]), fmaxf(sM[2], sM[3]));
  const float ms = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int c = cg; c < parts; c += 32) {
    const float2 e = gld<float2>(ml + 2 * c);
    const float4 o = gld<float4>(po + (size_t)c * HD);
    const float w = __builtin_amdgcn_exp2f(e.x - ms);
    L = __builtin_fmaf(e.y, w, L);
    y.x = __builtin_fmaf(o.x, w, y.x), y.y = __builtin_fmaf(o.y, w, y.y);
    y.z = __builtin_fmaf(o.z, w, y.z), y.w = __builtin_fmaf(o.w, w, y.w);
  }
  if (sub == 0) sL[cg] = L;
  sacc[cg][4 * sub] = y.x, sacc[cg][4 * sub + 1] = y.y, sacc[cg][4 * sub + 2] = y.z, sacc[cg][4 * sub + 3] = y.w;
  __syncthreads();
  if (tid < 32) {
    float t = 0.f, l = 0.f;
#pragma unroll 8
    for (int i = 0; i < 32; i++) t += sacc[i][tid], l += sL[i];
    t = pgd_finite(l == 0.f ? t * 0.f : t / l);
    const size_t o = (size_t)row * a.os + (size_t)h * HD + 32 * dg + tid;
    if constexpr (XT == GQ_F32) gst<float>((float *)a.out + o, t);
    else gst<uint16_t>((uint16_t *)a.out + o, (uint16_t)pgd_pack(t, t));
  }
}

/* Keys a part of a decode launch, a multiple of 128.  256 KB of K and V make a
 * part long enough that its share of the merge does not show (64 sequences of
 * up to 8192 positions, bf16, 8 KV heads: 187 us with 512 keys, 197 with 1024 and
 * 209 where the rule stopped at 4096 parts; one of 131072, int8: 55 with 1024,
 * 62 with 512, 96 with 256), shorter ones where they would leave less than two
 * workgroups a CU (one sequence of 4096, bf16: 10.9 with 128 keys, 15.3 with
 * 512).  One part, without the merge's launch of 3 us, where a sequence is
 * short (one of 256, bf16: 6.6 against 9.3; of 512: 11.1 against 9.9), or where
 * the sequences alone fill the chip (64 of 500: 20 against 32; 32 of 1000,
 * int8: 19.6 against 21.8).
 * At most 64 workgroups a CU, since the bound may be far above most lengths:
 * every part costs a workgroup and workspace for its results, 34 MB then at four
 * heads per KV head.  fp32 queries over bf16, 32 heads over 8 of 128, bound
 * 131072: 128 sequences of 1000 104 us (343 without a limit, 116 at 128 a CU, 100
 * at 32), one of 131072 among them 186 (414, 188, 286); 128 of up to 16384 742
 * (791, 791, 727). */
int decode_chunk(const gq_batch *b, const gq_pages *p, int n_cu) {
  const int row = 2 * p->head_dim * pgd_bytes(p->dtype), by = 256 * 1024 / row;
  const long long heads = (long long)b->n_seqs * p->n_kv_heads;
  const int whole = std::max(1, (b->max_len + 127) / 128) * 128;
  if (b->max_len <= std::min(384, 192 * 1024 / row) || (heads >= n_cu && b->max_len <= by)) return whole;
  const long long even = (heads * b->max_len / (2 * n_cu) + 127) / 128 * 128;
  const long long most = std::max(1ll, 64ll * n_cu / heads), least = ((b->max_len + most - 1) / most + 127) / 128 * 128;
  return (int)std::min<long long>(std::max(std::min<long long>(by, std::max<long long>(even, 128)), least), whole);
}

/* ------------------------------------------------------------ entry points */
bool aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }

/* 0, or -1 / -5 with the message set */
int check_cache(gq_ctx *c, const gq_pages *p, const gq_batch *b, int xtype) {
  if (!c) return -1;
  if (!p || !b) return gq_ctx_fail(c, -1, "paged: NULL pages or batch");
  if (p->dtype != GQ_F32 && p->dtype != GQ_BF16 && p->dtype != GQ_I8_ROWS) return gq_ctx_fail(c, -1, "paged: cache dtype");
  if (xtype != GQ_F32 && xtype != GQ_BF16) return gq_ctx_fail(c, -1, "paged: xtype is GQ_F32 or GQ_BF16");
  if (!p->k || !p->v || !aligned(p->k) || !aligned(p->v)) return gq_ctx_fail(c, -1, "paged: K and V pools are not there, or not 16-byte aligned");
  if (p->dtype == GQ_I8_ROWS && (!p->k_scale || !p->v_scale || !aligned(p->k_scale) || !aligned(p->v_scale)))
    return gq_ctx_fail(c, -1, "paged: an int8 cache needs its scales, 16-byte aligned");
  if (p->head_dim != 64 && p->head_dim != 128) return gq_ctx_fail(c, -1, "paged: head_dim is 64 or 128");
  if (p->n_kv_heads < 1 || p->n_pages < 1) return gq_ctx_fail(c, -1, "paged: no KV heads or no pages");
  if (p->page_size < 16 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)))
    return gq_ctx_fail(c, -1, "paged: page_size is a power of two from 16 to 1024");
  if (b->n_seqs < 0 || b->n_tokens < 0) return gq_ctx_fail(c, -1, "paged: negative size of the batch");
  if (b->n_seqs && (!b->table || !b->pos || b->table_stride < 1 || b->max_len < 0)) return gq_ctx_fail(c, -1, "paged: incomplete batch");
  if (b->n_seqs && (((uintptr_t)b->table | (uintptr_t)b->pos | (uintptr_t)b->first) & 3))
    return gq_ctx_fail(c, -1, "paged: table, pos or first is not 4-byte aligned");
  if (b->max_len > (1 << 30) || b->n_tokens > (1 << 30) || b->n_seqs > (1 << 30))
    return gq_ctx_fail(c, -1, "paged: max_len, n_tokens or n_seqs passes 2^30");
  if (!b->first && b->n_tokens < b->n_seqs) return gq_ctx_fail(c, -1, "paged: fewer rows than sequences");
  if (b->n_seqs && (long long)b->max_len > (long long)b->table_stride * p->page_size)
    return gq_ctx_fail(c, -5, "paged: max_len passes the page table");
  return 0;
}
/* rows of `width` values at a stride */
bool row_ok(const void *p, int stride, long long width) { return p && aligned(p) && stride >= width && stride % 8 == 0; }

PgdPages pages_of(const gq_pages *p) {
  return PgdPages{(uint8_t *)p->k, (uint8_t *)p->v, p->k_scale, p->v_scale, p->n_pages, __builtin_ctz((unsigned)p->page_size), p->n_kv_heads};
}
PgdBatch batch_of(const gq_batch *b) {
  return PgdBatch{b->table, b->pos, b->first, b->n_seqs, b->table_stride, b->n_tokens, b->max_len};
}

/* f<CT, XT, HD>() of run-time types */
template <class F>
void dispatch(int ct, int xt, int hd, F f) {
  auto h = [&](auto CT, auto XT) {
    if (hd == 64) f(CT, XT, std::integral_constant<int, 64>{});
    else f(CT, XT, std::integral_constant<int, 128>{});
  };
  auto x = [&](auto CT) {
    if (xt == GQ_F32) h(CT, std::integral_constant<int, GQ_F32>{});
    else h(CT, std::integral_constant<int, GQ_BF16>{});
  };
  if (ct == GQ_F32) x(std::integral_constant<int, GQ_F32>{});
  else if (ct == GQ_BF16) x(std::integral_constant<int, GQ_BF16>{});
  else x(std::integral_constant<int, GQ_I8_ROWS>{});
}

/* A whole tile a wave (WIDE), its loads under way together, where that leaves
 * two waves a SIMD; below, a load each and more waves.  8122 tokens of 48 rows
 * with their read: 63 us against 72. */
bool wide_rows(long long rows) { return rows >= 32768; }
/* their workgroups; 0: more than a launch takes */
unsigned row_blocks(long long tokens, int each, int hd, bool wide) {
  const long long rows = (tokens + kRowTile - 1) / kRowTile * kRowTile * each;
  const long long per = wide ? kThreads / GQ_WAVE * kRowTile : kThreads / (hd / 8), blocks = (rows + per - 1) / per;
  return pgd_launchable(blocks, kThreads) ? (unsigned)blocks : 0u;
}

/* the arguments of an attention over the cache: 0, a status, or 1 for nothing
 * to do */
int att_args(gq_ctx *c, const gq_pages *p, const gq_batch *b, int xtype, int n_heads, const void *q, int q_stride,
             void *out, int out_stride, AttArgs &a) {
  if (int rc = check_cache(c, p, b, xtype)) return rc;
  if (n_heads < 1 || n_heads % p->n_kv_heads || n_heads / p->n_kv_heads > kMaxG)
    return gq_ctx_fail(c, -1, "paged attention: 1 to 16 query heads per KV head");
  if (!b->n_seqs || !b->n_tokens) return 1;
  const long long width = (long long)n_heads * p->head_dim;
  if (!row_ok(q, q_stride, width) || !row_ok(out, out_stride, width))
    return gq_ctx_fail(c, -1, "paged attention: rows of q and out (16-byte aligned, strides of 8 elements and no overlap)");
  a = AttArgs{};
  a.c = pages_of(p), a.b = batch_of(b), a.q = q, a.out = out, a.n_heads = n_heads, a.G = n_heads / p->n_kv_heads;
  a.qs = q_stride, a.os = out_stride, a.scale = (float)(1.4426950408889634 / std::sqrt((double)p->head_dim));
  return 0;
}

} // namespace

extern "C" int gq_hip_paged_append_dev(gq_ctx *c, const gq_pages *p, const gq_batch *b, int xtype, int n_heads,
                                       const void *q, int q_stride, void *q_out, int q_out_stride, const void *k,
                                       int k_stride, const void *v, int v_stride, const float *rope, int n_rope) {
  if (int rc = check_cache(c, p, b, xtype)) return rc;
  if (q && n_heads < 1) return gq_ctx_fail(c, -1, "paged append: n_heads");
  if (!b->n_seqs || !b->n_tokens) return 0;
  const long long kvw = (long long)p->n_kv_heads * p->head_dim, qw = (long long)n_heads * p->head_dim;
  if (!row_ok(k, k_stride, kvw) || !row_ok(v, v_stride, kvw) ||
      (q && (!row_ok(q, q_stride, qw) || !row_ok(q_out, q_out_stride, qw))))
    return gq_ctx_fail(c, -1, "paged append: rows of q, k and v (16-byte aligned, strides of 8 elements and no overlap)");
  if (rope && !aligned(rope)) return gq_ctx_fail(c, -1, "paged append: rope is not 16-byte aligned");
  if (rope && n_rope < b->max_len) return gq_ctx_fail(c, -5, "paged append: max_len passes the rope table");
  const GqCtxInfo ci = gq_ctx_info(c);
  GqDeviceGuard guard(ci.dev);
  AppendArgs a{pages_of(p), batch_of(b), q, k, v, q_out, rope, n_heads, q_stride, q_out_stride, k_stride, v_stride, q ? n_heads : 0};
  const int each = a.nq + 2 * p->n_kv_heads;
  const bool wide = wide_rows((long long)b->n_tokens * each);
  const unsigned blocks = row_blocks(b->n_tokens, each, p->head_dim, wide);
  if (!blocks) return gq_ctx_fail(c, -1, "paged append: the batch passes a launch");
  dispatch(p->dtype, xtype, p->head_dim, [&](auto CT, auto XT, auto HD) {
    if (wide) hipLaunchKernelGGL((append_kernel<CT(), XT(), HD(), true>), dim3(blocks), dim3(kThreads), 0, ci.stream, a);
    else hipLaunchKernelGGL((append_kernel<CT(), XT(), HD(), false>), dim3(blocks), dim3(kThreads), 0, ci.stream, a);
  });
  return hipGetLastError() == hipSuccess ? 0 : gq_ctx_fail(c, -4, "paged append launch");
}

extern "C" int gq_hip_paged_read_dev(gq_ctx *c, const gq_pages *p, const gq_batch *b, int xtype, void *k, int k_stride,
                                     void *v, int v_stride) {
  if (int rc = check_cache(c, p, b, xtype)) return rc;
  if (!b->n_seqs || !b->n_tokens) return 0;
  const long long kvw = (long long)p->n_kv_heads * p->head_dim;
  if (!row_ok(k, k_stride, kvw) || !row_ok(v, v_stride, kvw))
    return gq_ctx_fail(c, -1, "paged read: rows of k and v (16-byte aligned, strides of 8 elements and no overlap)");
  const GqCtxInfo ci = gq_ctx_info(c);
  GqDeviceGuard guard(ci.dev);
  ReadArgs a{pages_of(p), batch_of(b), k, v, k_stride, v_stride};
  const int each = 2 * p->n_kv_heads;
  const bool wide = wide_rows((long long)b->n_tokens * each);
  const unsigned blocks = row_blocks(b->n_tokens, each, p->head_dim, wide);
  if (!blocks) return gq_ctx_fail(c, -1, "paged read: the batch passes a launch");
  dispatch(p->dtype, xtype, p->head_dim, [&](auto CT, auto XT, auto HD) {
    if (wide) hipLaunchKernelGGL((read_kernel<CT(), XT(), HD(), true>), dim3(blocks), dim3(kThreads), 0, ci.stream, a);
    else hipLaunchKernelGGL((read_kernel<CT(), XT(), HD(), false>), dim3(blocks), dim3(kThreads), 0, ci.stream, a);
  });
  return hipGetLastError() == hipSuccess ? 0 : gq_ctx_fail(c, -4, "paged read launch");
}

extern "C" int gq_hip_paged_decode_dev(gq_ctx *c, const gq_pages *p, const gq_batch *b, int xtype, int n_heads,
                                       const void *q, int q_stride, void *out, int out_stride) {
  AttArgs a;
  if (int rc = att_args(c, p, b, xtype, n_heads, q, q_stride, out, out_stride, a)) return rc > 0 ? 0 : rc;
  const GqCtxInfo ci = gq_ctx_info(c);
  GqDeviceGuard guard(ci.dev);
  a.chunk = decode_chunk(b, p, ci.n_cu);
  a.nch = std::max(1, (b->max_len + a.chunk - 1) / a.chunk);
  const long long blocks = (long long)b->n_seqs * p->n_kv_heads * a.nch, rows = (long long)b->n_seqs * n_heads;
  if (!pgd_launchable(blocks, kThreads) || (a.nch > 1 && !pgd_launchable(rows * (p->head_dim / 32), kThreads)))
    return gq_ctx_fail(c, -1, "paged decode: the batch passes a launch");
  if (a.nch > 1) {
    a.part_o = (float *)gq_ctx_paged_ws(c, sizeof(float) * rows * a.nch * (p->head_dim + 2));
    if (!a.part_o) return -4;
    a.part_ml = a.part_o + rows * a.nch * p->head_dim;
  }
  dispatch(p->dtype, xtype, p->head_dim, [&](auto CT, auto XT, auto HD) {
    hipLaunchKernelGGL((decode_kernel<CT(), XT(), HD()>), dim3((unsigned)blocks), dim3(kThreads), 0, ci.stream, a);
    if (a.nch > 1)
      hipLaunchKernelGGL((merge_kernel<XT(), HD()>), dim3((unsigned)(rows * (HD() / 32))), dim3(kThreads), 0, ci.stream, a);
  });
  return hipGetLastError() == hipSuccess ? 0 : gq_ctx_fail(c, -4, "paged decode launch");
}

extern "C" int gq_hip_paged_prompt_dev(gq_ctx *c, const gq_pages *p, const gq_batch *b, int xtype, int n_heads,
                                       const void *q, int q_stride, void *out, int out_stride) {
  AttArgs a;
  if (int rc = att_args(c, p, b, xtype, n_heads, q, q_stride, out, out_stride, a)) return rc > 0 ? 0 : rc;
  const GqCtxInfo ci = gq_ctx_info(c);
  GqDeviceGuard guard(ci.dev);
  const PromptShape f = gq_paged_prompt_shape(a, p->dtype, xtype, p->head_dim, ci.n_cu);
  if (!f.blocks) return gq_ctx_fail(c, -1, "paged prompt: the batch passes a launch");
  a.nch = f.parts, a.chunk = f.span;
  if (a.nch > 1) {
    const size_t rows = (size_t)b->n_tokens * n_heads * a.nch;
    a.part_o = (float *)gq_ctx_paged_ws(c, sizeof(float) * rows * (p->head_dim + 2));
    if (!a.part_o) return -4;
    a.part_ml = a.part_o + rows * p->head_dim;
  }
  return gq_launch_paged_prompt(a, p->dtype, xtype, p->head_dim, f, ci.stream) ? gq_ctx_fail(c, -4, "paged prompt launch") : 0;
}
