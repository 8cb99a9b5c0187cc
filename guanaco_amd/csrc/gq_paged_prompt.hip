/*
 * gq_paged_prompt.hip — causal attention of packed prompts over the paged K/V
 * cache on the bf16 matrix cores (gfx950).
 */
#include <algorithm>
#include <type_traits>

#include <utility>

#include "gq_paged.h"

namespace {

typedef float gq_f32x16 __attribute__((ext_vector_type(16)));

constexpr int kPThreads = 512;

/* A tile of query rows: up to tpt new tokens of a sequence, from its t0-th on,
 * packed from row `row` on; p0 positions are before the sequence's first. */
struct Tile {
  int s, row, t0, n, p0; /* n 0: there is none */
};
/* The id-th tile: of 64 sequences at a time the longest first, and of each its
 * last one first, so that what runs longest starts first (uniform in the wave). */
__device__ __forceinline__ Tile find_tile(const PgdBatch &b, int tpt, int id) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < b.n_seqs; s0 += GQ_WAVE) {
    const int q = s0 + lane, qc = min(q, b.n_seqs - 1), cnt = min(GQ_WAVE, b.n_seqs - s0);
    int r0 = qc, r1 = qc + 1;
    if (b.first) r0 = gld<int>(b.first + qc), r1 = gld<int>(b.first + qc + 1);
    int p0 = pgd_before(b, gld<int>(b.pos + qc));
    const bool in = q < b.n_seqs && r0 >= 0 && r1 <= b.n_tokens && r1 > r0;
    if (!in) r0 = r1 = 0;
    int sq = q;
    if (cnt > 1) { /* lane i: the i-th longest */
      const int len = in ? pgd_len(p0, r1 - r0, b.max_len) : -1;
      int rank = 0;
      for (int i = 0; i < cnt; i++) {
        const int u = __builtin_amdgcn_readlane(len, i);
        rank += u > len || (u == len && i < lane);
      }
      const int to = 4 * (lane < cnt ? rank : lane);
      sq = __builtin_amdgcn_ds_permute(to, sq), p0 = __builtin_amdgcn_ds_permute(to, p0);
      r0 = __builtin_amdgcn_ds_permute(to, r0), r1 = __builtin_amdgcn_ds_permute(to, r1);
    }
    const int own = (r1 - r0 + tpt - 1) / tpt;
    int c = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(c, o, 64);
      if (lane >= o) c += u;
    }
    const uint64_t hit = __ballot(before + c > id);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int t0 = (before + __builtin_amdgcn_readlane(c, l) - 1 - id) * tpt;
      r0 = __builtin_amdgcn_readlane(r0, l), r1 = __builtin_amdgcn_readlane(r1, l);
      return Tile{__builtin_amdgcn_readlane(sq, l), r0 + t0, t0, min(tpt, r1 - r0 - t0), __builtin_amdgcn_readlane(p0, l)};
    }
    before += __builtin_amdgcn_readlane(c, 63);
  }
  return Tile{0, 0, 0, 0, 0};
}

/* Blocks of 64 keys that a tile sees, and the parts that they come in: of at
 * most a.chunk, evenly. */
__device__ __forceinline__ int2 tile_blocks(const AttArgs &a, int p0, int last) {
  const int pmax = p0 < 0 ? -1 : min(p0 + last, a.b.max_len - 1), n = max(0, (pmax + kKeys) / kKeys);
  return make_int2(n, max(1, (n + a.chunk - 1) / a.chunk));
}

/* lanes 32 .. 63 of a against lanes 0 .. 31 of b */
__device__ __forceinline__ void swap_halves(float &a, float &b) {
  const auto w = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
  const uint32_t x = w[0], y = w[1]; /* a bit cast of w[1] itself would read w[0] */
  a = __builtin_bit_cast(float, x), b = __builtin_bit_cast(float, y);
}
/* lane J's value of the lane's row of 16, an operand's modifier */
template <int J>
__device__ __forceinline__ float of_row(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + J, 0xf, 0xf, true));
}
/* f(0) .. f(N - 1) of compile-time numbers */
template <class F, int... I>
__device__ __forceinline__ void each_of(F f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void each_of(F f) {
  each_of(f, std::make_integer_sequence<int, N>{});
}

/* the larger of a lane's value and that of the lane 32 away */
__device__ __forceinline__ float max_halves(float v) {
  float w = v;
  swap_halves(v, w);
  return fmaxf(v, w);
}

__device__ __forceinline__ void pin(gq_bf16x8 &v, float &f) {
  uint4 w = __builtin_bit_cast(uint4, v);
  asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w), "+v"(f));
  v = __builtin_bit_cast(gq_bf16x8, w);
}

/* Causal attention, flash-attention style.  A workgroup of eight waves takes 32
 * RG query rows = floor(32 RG / G) tokens x the G query heads of KV head g, and
 * streams their sequence's keys in blocks of 64: wave (rg, kh) rows 32 rg .. +
 * 31, and with KH = 2 keys 32 kh .. + 31 of every block, the two halves joined
 * at the end.
 *   S^T = K Q^T    A = K [key][dim] from LDS, B = the queries, in registers
 *                  for the whole kernel; lane (r, h) = (lane % 32, lane / 32)
 *                  gets row r's scores of keys 8 a + 4 h + c (a, c < 4)
 *   O^T += V^T P^T B = the probabilities straight from that layout: the 16
 *                  keys of a step are taken in the order in which a lane holds
 *                  them, and V lies in LDS as [dim][key] in the same order
 *                  (four keys by four dims transposed in registers on the
 *                  way); lane (r, h) holds row r's outputs, so the softmax's
 *                  rescale and the division stay in the lane.
 * The blocks are loaded a block ahead into registers, turned into bf16 and put
 * into LDS, octets (16 bytes) XOR-swizzled by the row.  fp32 queries keep fp32
 * accuracy: bf16 values and int8 codes are exact there (the scales multiply
 * scores and probabilities), and an fp32 operand is split into three bf16
 * numbers that sum to it, of whose products those not below 2^-24 are kept:
 * three over a bf16 or int8 cache, six over an fp32 one.  bf16 queries take
 * probabilities rounded to bf16, like the results, and are exact themselves: one
 * product, or two over an fp32 cache, whose values are two bf16 numbers there
 * (2^-17).  With its values and int8 ones rounded to one, results are 0.0039 off
 * in the mean for 0.0021, most of it by K.
 *
 * Keys that do not exist are masked, and their V zeros in LDS, so that what stale
 * memory holds cannot reach a sum.  So are infinities and NaN of V in the blocks that
 * only some rows see whole (a masked probability of 0 times them is no 0): those
 * that see them get them at the end.  The check costs 1 to 3%.
 *
 * Vector work bounds it: of a block's 1.8 us alone (2.4 with the chip full; bf16,
 * head_dim 128, 256 rows) the MFMAs take 0.85, about 246 vector instructions a
 * wave the most of it, and a workgroup begins and ends in 6.5.  7073 tokens of
 * four bf16 prompts 215 us (168 GFLOP, 0.78 PFLOP/s), one of 16384 0.99 PFLOP/s;
 * 1119 tokens at 3058 to 7500 over int8 195 us; 1567 fp32 ones over bf16 146.
 *
 * The blocks of a tile come in parts of at most a.chunk, a workgroup each, where
 * the tiles alone would leave CUs idle; prompt_merge_kernel joins them. */
template <int CT, int XT, int HD, int RG, int KH>
__global__ __launch_bounds__(kPThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void prompt_kernel(AttArgs a) {
  static_assert(RG * KH * GQ_WAVE == kPThreads, "eight waves");
  typedef PromptLds<CT, XT, HD, RG, KH> Lds;
  constexpr int NX = Lds::NX, NK = Lds::NK;
  constexpr int NP = NX * NK == 9 ? 6 : NX * NK; /* partial products */
  /* their planes of K or V and of Q or P, the small ones first */
  constexpr int kA[4][6] = {{0}, {1, 0}, {0, 0, 0}, {1, 2, 0, 1, 0, 0}}, kB[4][6] = {{0}, {0, 0}, {2, 1, 0}, {1, 0, 2, 0, 1, 0}};
  constexpr int W = NP == 6 ? 3 : NP - 1;
  constexpr int NB = Lds::NB;
  constexpr bool PIPE = NP == 1;
  constexpr bool CODES = Lds::CODES;
  constexpr int EB = pgd_bytes(CT);
  constexpr int NO = HD / 8;                 /* octets of a K row */
  constexpr int NSL = HD / 16, ND = HD / 32; /* dim slices of S^T, dim tiles of O^T */
  constexpr int KT = 2 / KH;                 /* 32-key tiles of a wave's */
  constexpr int KPL = Lds::KPL;
  constexpr int KI = kKeys * NO / kPThreads; /* K octets a thread */
  constexpr int KPP = kPThreads / NO;        /* keys a pass of them */
  constexpr int KW = 2 * EB, VW = EB;
  constexpr int VTH = 16 * HD / 4;           /* threads with four keys x four dims of V */
  constexpr int NQ = NX == 3 ? 2 : 1;        /* planes of Q in registers; the third in LDS */
  constexpr int QLO = Lds::QLO, SCL = Lds::SCL, ODD = Lds::ODD;
  __shared__ __attribute__((aligned(16))) uint8_t smem_[Lds::BYTES];
  GQ_LDS uint8_t *smem = (GQ_LDS uint8_t *)smem_;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 31, h = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), rg = wv / KH, kh = wv % KH;
  const int G = a.G, tpt = 32 * RG / G;
  int bid = blockIdx.x;
  const int g = bid % a.c.n_kv;
  bid /= a.c.n_kv;
  /* Parts last: workgroups go round the chip's engines in turn, and with a tile's
   * parts side by side the ones that it has fewer than another tile leave the
   * same engines idle each time (7073 tokens in 2 parts: 312 us). */
  const int tiles = gridDim.x / (unsigned)(a.c.n_kv * a.nch), part = bid / tiles;
  const Tile tl = find_tile(a.b, tpt, bid % tiles);
  if (!tl.n) return;
  const int s = tl.s;
  /* position that a row of the tile sees last; none of an idle sequence */
  auto sees = [&](int row) { return tl.p0 < 0 ? -1 : min(tl.p0 + tl.t0 + min(row / G, tl.n - 1), a.b.max_len - 1); };
  const int2 bp = tile_blocks(a, tl.p0, tl.t0 + tl.n - 1);
  if (part >= bp.y) return;
  const int b0 = (int)((long long)bp.x * part / bp.y), b1 = (int)((long long)bp.x * (part + 1) / bp.y); /* this part's blocks */
  const int pmax = sees(32 * RG - 1);
  const int row = 32 * rg + r, tok = min(row / G, tl.n - 1), qh = g * G + row % G;
  const bool live = row < tpt * G && row / G < tl.n;
  const int cpos = sees(row), wlo = sees(32 * rg), whi = sees(32 * rg + 31);

  /* this row's query: dims 16 i + 8 h .. + 7 */
  gq_bf16x8 q[NSL][NQ];
  const uint32_t qlo = (uint32_t)(QLO + (rg * 64 + lane) * 16);
  auto query = [&] {
    const size_t at = (size_t)(tl.row + tok) * a.qs + (size_t)qh * HD + 8 * h;
#pragma unroll
    for (int i = 0; i < NSL; i++) {
      if constexpr (NX == 3) {
        float x[8];
        pgd_load8<XT>(a.q, at + 16 * i, x);
        gq_bf16x8 p[3];
        split8<3>(x, p);
        q[i][0] = p[0], q[i][1] = p[1];
        if (kh == 0) lst<gq_bf16x8>(smem, qlo + RG * 1024 * i, p[2]);
      } else {
        q[i][0] = gld<gq_bf16x8>((const uint16_t *)a.q + at + 16 * i);
      }
    }
  };

  /* staging: K octet ko of keys kk, kk + KPP ..; V dims 4 vd .. + 3 of keys 4
   * va .. + 3; a wave's keys are of one 16-key group each time, and so of one
   * page. */
  const int ko = tid % NO, kk = tid / NO, vd = tid % (HD / 4), va = tid / (HD / 4);
  const bool vtask = VTH == kPThreads || tid < VTH;
  uint32_t kr[KI][KW], vr[4][VW]; /* raw dwords */
  float sc = 0.f;                     /* int8: the scale of key `lane`, K's in wave 0 and V's in wave 1 */
  const int ps = (1 << a.c.lg) - 1;
  uint32_t koff[KI]; /* within a page's rows for the head, from the block's first slot */
#pragma unroll
  for (int i = 0; i < KI; i++) koff[i] = (uint32_t)((((kk + KPP * i) & ps) * HD + 8 * ko) * EB);
  const uint32_t voff = (uint32_t)((((4 * va) & ps) * HD + 4 * vd) * EB);
  /* Pages of 64 groups of 16 keys at a time, lane i: group i of blocks 16 n .. 16
   * n + 15, -1 where it does not exist; those of block b's 16 and the next 16. */
  const int32_t *table = a.b.table + (size_t)s * a.b.stride;
  auto lookup = [&](int n) {
    const int p = 16 * (64 * n + lane), page = gld<int>(table + min(p >> a.c.lg, a.b.stride - 1));
    return p <= pmax && (unsigned)page < (unsigned)a.c.n_pages ? page : -1;
  };
  int pg0 = -1, pg1 = -1, pgn = 0;
  auto pages = [&](int b) { return (b >> 4) == pgn ? pg0 : pg1; };
  auto exists = [&](int b) { return (int)(__ballot(pages(b) >= 0) >> (4 * (b & 15))) & 15; }; /* bit i: group i of b */
  /* the row of block b's first slot in the page of a key's group (uniform) */
  auto rows = [&](int b, int key) {
    const int page = __builtin_amdgcn_readlane(pages(b), __builtin_amdgcn_readfirstlane(4 * (b & 15) + (key >> 4)));
    return pgd_row(a.c, max(page, 0), g, (b * kKeys) & ps);
  };
  auto loadk = [&](int b, uint32_t (&kr)[KI][KW]) {
#pragma unroll
    for (int i = 0; i < KI; i++) {
      const size_t at = rows(b, kk + KPP * i);
      const uint8_t *kp = a.c.k + at * (size_t)(HD * EB);
      if constexpr (EB == 1) {
        const uint2 w = gld<uint2>(kp + koff[i]);
        kr[i][0] = w.x, kr[i][1] = w.y;
      } else {
#pragma unroll
        for (int e = 0; e < EB / 2; e++) {
          const uint4 w = gld<uint4>(kp + koff[i] + 16 * e);
          kr[i][4 * e] = w.x, kr[i][4 * e + 1] = w.y, kr[i][4 * e + 2] = w.z, kr[i][4 * e + 3] = w.w;
        }
      }
    }
  };
  auto loadv = [&](int b, uint32_t (&vr)[4][VW]) {
    if (vtask) {
      const size_t at = rows(b, 4 * va);
      const uint8_t *vp = a.c.v + at * (size_t)(HD * EB);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        if constexpr (EB == 1) {
          vr[i][0] = gld<uint32_t>(vp + voff + i * HD);
        } else if constexpr (EB == 2) {
          const uint2 w = gld<uint2>(vp + voff + i * HD * 2);
          vr[i][0] = w.x, vr[i][1] = w.y;
        } else {
          const uint4 w = gld<uint4>(vp + voff + i * HD * 4);
          vr[i][0] = w.x, vr[i][1] = w.y, vr[i][2] = w.z, vr[i][3] = w.w;
        }
      }
    }
  };
  auto loads = [&](int b, int w, float &sc) {
    if constexpr (CODES) {
      if (wv == w) {
        const int page = __shfl(pages(b), 4 * (b & 15) + (lane >> 4), 64);
        const float d = gld<float>((w ? a.c.vs : a.c.ks) + pgd_row(a.c, max(page, 0), g, ((b * kKeys) & ps) + (lane & ps)));
        sc = page >= 0 && b * kKeys + lane <= pmax ? d : 0.f;
      }
    }
  };
  /* blocks that not all of the tile's rows see whole */
  const int pmin = sees(0);
  uint32_t odd = 0; /* this wave has zeroed some */
  auto partial = [&](int b) { return b * kKeys + kKeys - 1 > pmin; };
  /* the loaded K or V of block b into buffer buf; V's rows that do not exist are
   * zeros (K's scores are masked), and so are in a partial block the values that
   * are no numbers: times a masked probability they would reach rows that do not
   * see them.  Those that do get them at the end. */
  auto stagek = [&](int b, int buf, uint32_t (&kr)[KI][KW], float sc) {
    const uint32_t kb = (uint32_t)(buf * 2 * NK * KPL);
#pragma unroll
    for (int i = 0; i < KI; i++) {
      const int key = kk + KPP * i;
      const uint32_t at = kb + (uint32_t)(key * HD * 2 + ((ko ^ (key & (NO - 1))) << 4));
      if constexpr (CT == GQ_BF16) {
        lst<uint4>(smem, at, make_uint4(kr[i][0], kr[i][1], kr[i][2], kr[i][3]));
      } else if constexpr (CODES) {
        lst<gq_bf16x8>(smem, at, codes8(kr[i][0], kr[i][1]));
      } else {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __builtin_bit_cast(float, kr[i][e]);
        gq_bf16x8 p[NK];
        split8<NK>(x, p);
#pragma unroll
        for (int n = 0; n < NK; n++) lst<gq_bf16x8>(smem, at + n * KPL, p[n]);
      }
    }
    if constexpr (CODES) {
      if (wv == 0) lst<float>(smem, SCL + ((b & 3) * kKeys + lane) * 4, sc * a.scale);
    }
  };
  auto stagev = [&](int b, int buf, uint32_t (&vr)[4][VW], float sc) {
    const uint32_t vb = (uint32_t)((buf * 2 + 1) * NK * KPL);
    const int ok = exists(b);
    if (ok != 15 || b * kKeys + kKeys - 1 > pmax) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const bool there = (ok >> (va >> 2 & 3) & 1) && b * kKeys + 4 * va + i <= pmax;
#pragma unroll
        for (int e = 0; e < VW; e++) vr[i][e] = there ? vr[i][e] : 0u;
      }
    }
    if (partial(b)) {
      /* added to an exponent of ones, one in its last place carries; fp32 values
       * that are to be bf16: from those on that round to an infinity */
      constexpr uint32_t ex = CT == GQ_BF16 ? 0x7f807f80u : 0x7fffffffu, top = CT == GQ_BF16 ? 0x80008000u : 0x80000000u;
      constexpr uint32_t one = CT == GQ_BF16 ? 0x00800080u : CT == GQ_F32 ? 0x00808000u : 0x00800000u;
      uint32_t bad = 0;
      if constexpr (CODES) {
        bad = wv == 1 ? (__builtin_bit_cast(uint32_t, sc) & ex) + one : 0u;
      } else if (vtask) {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
          for (int e = 0; e < VW; e++) bad |= (vr[i][e] & ex) + one;
      }
      if (__ballot((bad & top) != 0)) {
        odd = 1;
        if constexpr (CODES) {
          sc = bad & top ? 0.f : sc;
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < VW; e++) {
              const uint32_t c = ((vr[i][e] & ex) + one) & top;
              vr[i][e] &= ~(CT == GQ_BF16 ? (c >> 15) * 0xffffu : c ? ~0u : 0u);
            }
        }
      }
    }
    if (vtask) {
      const int oct = 4 * (va >> 3) + 2 * (va >> 2 & 1) + (va & 1), half = va >> 1 & 1;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int dim = 4 * vd + j;
        const uint32_t at = vb + (uint32_t)(dim * kKeys * 2 + ((oct ^ ((dim ^ (dim >> 3)) & 7)) << 4) + 8 * half);
        if constexpr (CT == GQ_BF16) {
          const uint32_t sel = j & 1 ? 0x07060302u : 0x05040100u;
          lst<uint2>(smem, at, make_uint2(__builtin_amdgcn_perm(vr[1][j / 2], vr[0][j / 2], sel),
                                          __builtin_amdgcn_perm(vr[3][j / 2], vr[2][j / 2], sel)));
        } else if constexpr (CT == GQ_I8_ROWS) {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; i++) x[i] = i8f(vr[i][0], j);
          lst<uint2>(smem, at, make_uint2(pgd_pack(x[0], x[1]), pgd_pack(x[2], x[3])));
        } else {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; i++) x[i] = __builtin_bit_cast(float, vr[i][j]);
          uint2 p[3];
          split3(x[0], x[1], p[0].x, p[1].x, p[2].x);
          split3(x[2], x[3], p[0].y, p[1].y, p[2].y);
#pragma unroll
          for (int n = 0; n < NK; n++) lst<uint2>(smem, at + n * KPL, p[n]);
        }
      }
    }
    if constexpr (CODES) {
      if (wv == 1) lst<float>(smem, SCL + ((4 + buf) * kKeys + lane) * 4, sc);
    }
  };

  float m = -INFINITY, l = 0.f; /* l: this lane's keys only */
  gq_f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) o[d] = gq_f32x16{};
  /* operand addresses within a block: K row 32 kt + r, octet 2 i + h; V row 32 d
   * + r, octet 4 kt + 2 t + h */
  const uint32_t kbase = (uint32_t)((32 * kh + r) * HD * 2 + ((h ^ (r & (NO - 1))) << 4));
  const uint32_t vbase = (uint32_t)(NK * KPL + r * kKeys * 2 + (((4 * kh + h) ^ ((r ^ (r >> 3)) & 7)) << 4));

  /* the scores of a block whose K is in buffer buf: keys 32 t + 8 (e / 4) + 4 h +
   * e % 4 of the wave's */
  auto scores = [&](int buf, gq_f32x16 (&st)[KT]) {
    const uint32_t at = (uint32_t)(buf * 2 * NK * KPL);
#pragma unroll
    for (int t = 0; t < KT; t++) st[t] = gq_f32x16{};
#pragma unroll
    for (int i = 0; i < NSL; i++) {
      gq_bf16x8 qv[NX];
      qv[0] = q[i][0];
      if constexpr (NX == 3) qv[1] = q[i][1], qv[2] = lld<gq_bf16x8>(smem, qlo + RG * 1024 * i);
#pragma unroll
      for (int t = 0; t < KT; t++) {
        gq_bf16x8 kv[NK];
#pragma unroll
        for (int n = 0; n < NK; n++) kv[n] = lld<gq_bf16x8>(smem, at + (kbase ^ (32 * i)) + 32 * t * HD * 2 + n * KPL);
#pragma unroll
        for (int u = 0; u < NP; u++) st[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kv[kA[W][u]], qv[kB[W][u]], st[t], 0, 0, 0);
      }
    }
  };
  /* int8: scores 4 c .. + 3 times K's scales (ring b & 3), in units of log 2, or
   * the probabilities times V's (ring 4 + buffer).  Lane j of each row of 16
   * holds the scale of the lanes' score j, where LDS would return all 16 to every
   * lane: 4 chunks of up to 512 tokens at up to 7500 260 us by 16-byte reads, 229
   * so. */
  struct Scales {
    float d[KT];
  };
  auto scales = [&](int ring) {
    Scales s{};
    if constexpr (CODES)
#pragma unroll
      for (int t = 0; t < KT; t++)
        s.d[t] = lld<float>(smem, SCL + (ring * kKeys + 32 * (kh + t) + 8 * (lane >> 2 & 3) + 4 * h + (lane & 3)) * 4);
    return s;
  };
  auto times = [&](const Scales &s, gq_f32x16 (&st)[KT], auto c) {
    if constexpr (CODES)
      each_of<4>([&](auto i) {
        constexpr int e = 4 * (c() % 4) + i();
        st[c() / 4][e] *= of_row<e>(s.d[c() / 4]);
      });
  };
  /* keys that do not exist or lie past the row's position: -infinity */
  auto mask = [&](int b, gq_f32x16 (&st)[KT]) {
    const int key0 = b * kKeys + 32 * kh, ok = exists(b);
#pragma unroll
    for (int t = 0; t < KT; t++) {
      if (ok != 15 || key0 + 32 * t + 31 > wlo) {
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int k = 32 * t + 8 * (e >> 2) + 4 * h + (e & 3);
          st[t][e] = key0 + k <= cpos && (ok >> ((32 * kh + k) >> 4) & 1) ? st[t][e] : -INFINITY;
        }
      }
    }
  };
  gq_bf16x8 pr[2 * KT][NX];
  float alpha;
  bool rescale;
  /* the probabilities of masked scores, with V's scales for int8 */
  auto softmax = [&](int buf, gq_f32x16 (&st)[KT]) {
    const Scales dv = scales(4 + buf);
    float mb = -INFINITY;
#pragma unroll
    for (int t = 0; t < KT; t++)
#pragma unroll
      for (int e = 0; e < 16; e++) mb = fmaxf(mb, st[t][e]);
    mb = max_halves(mb);
    if constexpr (!CODES) mb *= a.scale;
    const float mn = fmaxf(m, mb), ms = mn == -INFINITY ? 0.f : mn;
    alpha = __builtin_amdgcn_exp2f(m - ms);
    rescale = __ballot(mn > m) != 0; /* some row's maximum has risen (alpha is 1 in the others) */
    m = mn;
    l *= alpha;
#pragma unroll
    for (int t = 0; t < KT; t++) {
#pragma unroll
      for (int e = 0; e < 16; e++) {
        st[t][e] = __builtin_amdgcn_exp2f(CODES ? st[t][e] - ms : __builtin_fmaf(st[t][e], a.scale, -ms));
        l += st[t][e];
      }
      each_of<4 * KT>([&](auto c) {
        if (c() / 4 == t) times(dv, st, c);
      });
#pragma unroll
      for (int u = 0; u < 2; u++) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = st[t][8 * u + e];
        split8<NX>(x, pr[2 * t + u]);
      }
    }
  };
  auto output = [&](int buf) {
    const uint32_t at = (uint32_t)(buf * 2 * NK * KPL);
    /* fp32 results: the block's P V in accumulators of its own, so that O takes
     * one rounding a block and not one a product */
    constexpr bool OWN = NX == 3;
    if (!OWN && rescale) {
#pragma unroll
      for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] *= alpha;
    }
#pragma unroll
    for (int d = 0; d < ND; d++) {
      gq_f32x16 pv = OWN ? gq_f32x16{} : o[d];
#pragma unroll
      for (int t = 0; t < 2 * KT; t++) {
        gq_bf16x8 vv[NK];
#pragma unroll
        for (int n = 0; n < NK; n++)
          vv[n] = lld<gq_bf16x8>(smem, at + (vbase ^ (((4 * d & 7) ^ (2 * t)) << 4)) + n * KPL + 32 * d * kKeys * 2);
#pragma unroll
        for (int u = 0; u < NP; u++) pv = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vv[kA[W][u]], pr[t][kB[W][u]], pv, 0, 0, 0);
      }
      if constexpr (OWN) {
#pragma unroll
        for (int e = 0; e < 16; e++) o[d][e] = __builtin_fmaf(o[d][e], alpha, pv[e]);
      } else {
        o[d] = pv;
      }
    }
  };

  /* Loads past the end take the last block again: under a condition they would
   * leave registers undefined (decode_kernel). */
  const int bl = b1 - 1;
  auto turn = [&](int b) { /* pages for the blocks from b on */
    if ((b & 15) == 0) pg0 = pg1, pgn = b >> 4, pg1 = lookup(pgn + 1);
  };
  if (b0 < b1) pgn = b0 >> 4, pg0 = lookup(pgn), pg1 = lookup(pgn + 1);
  if constexpr (PIPE) {
    /* Block b + 1's scores and b's softmax together: a wave's matrix instructions
     * run under its own vector ones.  K is a block further ahead than V. */
    if (b0 < b1) {
      gq_f32x16 sa[KT], sb[KT];
      {
        uint32_t k0[KI][KW], k1[KI][KW], v0[4][VW];
        float c0 = 0.f, c1 = 0.f;
        const int n1 = min(b0 + 1, bl), n2 = min(b0 + 2, bl);
        loadk(b0, k0), loads(b0, 0, c0), loadv(b0, v0), loads(b0, 1, c0);
        loadk(n1, k1), loads(n1, 0, c1), loadv(n1, vr), loads(n1, 1, sc);
        loadk(n2, kr), loads(n2, 0, sc);
        query();
        stagek(b0, b0 & 1, k0, c0), stagev(b0, b0 & 1, v0, c0);
        stagek(n1, (b0 + 1) & 1, k1, c1);
      }
      __syncthreads();
      scores(b0 & 1, sa);
      const Scales dk = scales(b0 & 3);
      each_of<4 * KT>([&](auto c) { times(dk, sa, c); });
      __syncthreads(); /* K of block 0 has been read */
      /* before it K of b and b + 1 and V of b are in LDS, K of b + 2 and V of b + 1
       * in registers.  Written in the order in which it is to run: four LDS
       * operands ahead of the matrix instructions, a piece of the softmax after
       * each (the compiler's own order waits for every operand). */
      auto body = [&](int b, gq_f32x16 (&cur)[KT], gq_f32x16 (&next)[KT]) {
        constexpr int N = KT * NSL, J = 4 * KT, N2 = 2 * KT * ND, A = 4; /* A operands ahead */
        mask(b, cur);
        const Scales dv = scales(4 + (b & 1));
        const uint32_t kat = (uint32_t)(((b + 1) & 1) * 2 * KPL) + kbase, vat = (uint32_t)((b & 1) * 2 * KPL) + vbase;
        auto kop = [&](int i) { return lld<gq_bf16x8>(smem, (kat ^ (32 * (i / KT))) + 32 * (i % KT) * HD * 2); };
        auto vop = [&](int i) {
          return lld<gq_bf16x8>(smem, (vat ^ (((4 * (i % ND) & 7) ^ (2 * (i / ND))) << 4)) + 32 * (i % ND) * kKeys * 2);
        };
        gq_bf16x8 w[A];
#pragma unroll
        for (int i = 0; i < A; i++) w[i] = kop(i);
        float ms = 0.f;
        each_of<N>([&](auto I) {
          constexpr int i = I;
          __builtin_amdgcn_sched_barrier(0);
          next[i % KT] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[i % A], q[i / KT][0], i < KT ? gq_f32x16{} : next[i % KT], 0, 0, 0);
          if (i + A < N) w[i % A] = kop(i + A);
          if (i == 0) {
            float mb = -INFINITY;
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
              for (int e = 0; e < 16; e++) mb = fmaxf(mb, cur[t][e]);
            mb = max_halves(mb);
            if constexpr (!CODES) mb *= a.scale;
            const float mn = fmaxf(m, mb);
            ms = mn == -INFINITY ? 0.f : mn;
            alpha = __builtin_amdgcn_exp2f(m - ms);
            rescale = __ballot(mn > m) != 0;
            m = mn, l *= alpha;
          }
          each_of<J>([&](auto c) { /* scores 4 c .. + 3 */
            if constexpr (i == 0 || c() < (i - 1) * J / (N - 1) || c() >= i * J / (N - 1)) return;
            constexpr int t = c() / 4, e0 = 4 * (c() % 4);
#pragma unroll
            for (int e = e0; e < e0 + 4; e++) {
              cur[t][e] = __builtin_amdgcn_exp2f(CODES ? cur[t][e] - ms : __builtin_fmaf(cur[t][e], a.scale, -ms));
              l += cur[t][e];
            }
            times(dv, cur, c);
            if (c & 1) {
              float x[8];
#pragma unroll
              for (int e = 0; e < 8; e++) x[e] = cur[t][e0 - 4 + e];
              split8<1>(x, pr[c / 2]);
              pin(pr[c / 2][0], l); /* here and not where they are used */
            }
          });
        });
        __builtin_amdgcn_sched_barrier(0);
        stagek(min(b + 2, bl), b & 1, kr, sc), stagev(min(b + 1, bl), (b + 1) & 1, vr, sc);
        loadk(min(b + 3, bl), kr), loads(min(b + 3, bl), 0, sc);
        loadv(min(b + 2, bl), vr), loads(min(b + 2, bl), 1, sc);
        if (rescale) {
#pragma unroll
          for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) o[d][e] *= alpha;
        }
        const Scales dk = scales((b + 1) & 3);
#pragma unroll
        for (int i = 0; i < A; i++) w[i] = vop(i);
        each_of<N2>([&](auto I) {
          constexpr int i = I;
          __builtin_amdgcn_sched_barrier(0);
          o[i % ND] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w[i % A], pr[i / ND][0], o[i % ND], 0, 0, 0);
          if (i + A < N2) w[i % A] = vop(i + A);
          each_of<J>([&](auto c) {
            if constexpr (c() >= i * J / N2 && c() < (i + 1) * J / N2) times(dk, next, c);
          });
        });
        __builtin_amdgcn_sched_barrier(0);
        turn(b + 1);
        __syncthreads();
      };
      for (int b = b0;;) {
        body(b, sa, sb);
        if (++b >= b1) break;
        body(b, sb, sa);
        if (++b >= b1) break;
      }
    }
  } else {
    auto compute = [&](int b, int buf) {
      if (b * kKeys + 32 * kh > whi) return; /* none of this wave's rows sees any (uniform) */
      gq_f32x16 st[KT];
      scores(buf, st);
      const Scales dk = scales(b & 3);
      each_of<4 * KT>([&](auto c) { times(dk, st, c); });
      mask(b, st);
      softmax(buf, st);
      output(buf);
    };
    auto load = [&](int b) { loadk(b, kr), loads(b, 0, sc), loadv(b, vr), loads(b, 1, sc); };
    auto stage = [&](int b, int buf) { stagek(b, buf, kr, sc), stagev(b, buf, vr, sc); };
    if (b0 < b1) {
      load(b0);
      query();
      if constexpr (NB == 2) {
        stage(b0, b0 & 1);
        load(min(b0 + 1, bl));
        __syncthreads();
        for (int b = b0; b < b1; b++) {
          stage(min(b + 1, bl), (b + 1) & 1); /* last read before the barrier below */
          load(min(b + 2, bl));
          compute(b, b & 1);
          turn(b + 1);
          __syncthreads();
        }
      } else {
        for (int b = b0; b < b1; b++) {
          __syncthreads(); /* the planes are free */
          stage(b, 0);
          __syncthreads();
          load(min(b + 1, bl));
          compute(b, 0);
          turn(b + 1);
        }
        __syncthreads();
      }
    }
  }
  /* The values of partial blocks that are no numbers, to the outputs of the rows
   * that see them, which they make NaN (pgd_finite). */
  if (lane == 0) lst<uint32_t>(smem, ODD + 4 * wv, odd);
  __syncthreads();
  {
    const uint4 f = lld<uint4>(smem, ODD), f1 = lld<uint4>(smem, ODD + 16);
    odd = (uint32_t)__builtin_amdgcn_readfirstlane((int)(f.x | f.y | f.z | f.w | f1.x | f1.y | f1.z | f1.w));
  }
  for (int u = max(b0, (pmin + 1) / kKeys) * kKeys; odd && u < min(b1 * kKeys, pmax + 1); u++) { /* partial blocks */
    const int page = (KH == 1 || (u >> 5 & 1) == kh) ? pgd_page_u(a.c, a.b, s, u) : -1;
    if (page < 0) continue;
    const size_t at = pgd_row(a.c, page, g, u & ps);
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const size_t i = at * HD + 32 * d + 8 * (e >> 2) + 4 * h + (e & 3);
        float x;
        if constexpr (CT == GQ_F32) x = gld<float>((const float *)a.c.v + i);
        else if constexpr (CT == GQ_BF16) x = pgd_lo(gld<uint16_t>((const uint16_t *)a.c.v + i));
        else x = (float)*(const GQ_GLOBAL int8_t *)(a.c.v + i) * gld<float>(a.c.vs + at);
        if constexpr (CT == GQ_F32) x = pgd_lo(pgd_pack(x, x));
        if (u <= cpos && (__builtin_bit_cast(uint32_t, x) & 0x7f800000u) == 0x7f800000u) o[d][e] += x;
        __builtin_amdgcn_sched_barrier(0); /* one load at a time: no registers beside the outputs */
      }
  }
  l += __shfl_xor(l, 32, 64);
  if constexpr (KH == 2) { /* kh = 1 hands (m, l, O) to kh = 0; slower waves may still read the flags */
    GQ_LDS float *x = (GQ_LDS float *)smem + rg * 64 * (ND * 16 + 2);
    if (kh == 1) {
      x[lane] = m, x[64 + lane] = l;
#pragma unroll
      for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) x[64 * (2 + 16 * d + e) + lane] = o[d][e];
    }
    __syncthreads();
    if (kh == 1) return;
    const float m1 = x[lane], mt = fmaxf(m, m1), ms = mt == -INFINITY ? 0.f : mt;
    const float s0 = __builtin_amdgcn_exp2f(m - ms), s1 = __builtin_amdgcn_exp2f(m1 - ms);
    l = l * s0 + x[64 + lane] * s1, m = mt;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int e = 0; e < 16; e++) o[d][e] = o[d][e] * s0 + x[64 * (2 + 16 * d + e) + lane] * s1;
  }
  /* Lanes (r, 0) and (r, 1) trade halves of two runs of eight dims, so that each
   * has one whole: dims 32 d + 16 c + 8 h .. + 7. */
  const bool whole = bp.y == 1;
  const float inv = !whole ? 1.0f : l == 0.f ? 0.f : 1.0f / l; /* nothing seen: zeros */
  const size_t at = (size_t)(tl.row + tok) * a.os + (size_t)qh * HD;
  const size_t pat = ((size_t)(tl.row + tok) * a.n_heads + qh) * a.nch + part;
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int c = 0; c < 2; c++) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 4; e++) {
        y[e] = o[d][8 * c + e] * inv, y[4 + e] = o[d][8 * c + 4 + e] * inv;
        if (whole) y[e] = pgd_finite(y[e]), y[4 + e] = pgd_finite(y[4 + e]);
        swap_halves(y[e], y[4 + e]);
      }
      const int dim = 32 * d + 16 * c + 8 * h;
      if (live) {
        if (whole) pgd_store8<XT>(a.out, at + dim, y);
        else pgd_store8<GQ_F32>(a.part_o, pat * HD + dim, y);
      }
    }
  if (live && !whole && h == 0) gst<float2>(a.part_ml + 2 * pat, make_float2(m, l));
}

/* The parts of a row's keys, a workgroup per token: out = sum_c o_c 2^(m_c - M) /
 * sum_c l_c 2^(m_c - M), four dims of a head a thread. */
template <int XT, int HD>
__global__ __launch_bounds__(kPThreads) void prompt_merge_kernel(AttArgs a, int tpt) {
  const int row = blockIdx.x, s = __builtin_amdgcn_readfirstlane(pgd_seq_of(a.b, row));
  if (s >= a.b.n_seqs) return;
  const int2 rn = pgd_rows(a.b, s);
  if (row < rn.x || row >= rn.x + rn.y) return;
  const int parts = tile_blocks(a, pgd_before(a.b, gq_sld<int>(a.b.pos + s)), min((row - rn.x) / tpt * tpt + tpt, rn.y) - 1).y;
  if (parts <= 1) return; /* its one part has written the result */
  for (int i = threadIdx.x; i < a.n_heads * (HD / 4); i += kPThreads) {
    const int qh = i / (HD / 4), dim = 4 * (i % (HD / 4));
    const size_t at = ((size_t)row * a.n_heads + qh) * a.nch;
    float M = -INFINITY;
    for (int c = 0; c < parts; c++) M = fmaxf(M, gld<float>(a.part_ml + 2 * (at + c)));
    const float ms = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int c = 0; c < parts; c++) {
      const float2 ml = gld<float2>(a.part_ml + 2 * (at + c));
      const float4 o = gld<float4>(a.part_o + (at + c) * HD + dim);
      const float w = __builtin_amdgcn_exp2f(ml.x - ms);
      L = __builtin_fmaf(ml.y, w, L);
      y.x = __builtin_fmaf(o.x, w, y.x), y.y = __builtin_fmaf(o.y, w, y.y);
      y.z = __builtin_fmaf(o.z, w, y.z), y.w = __builtin_fmaf(o.w, w, y.w);
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    y.x = pgd_finite(y.x * inv), y.y = pgd_finite(y.y * inv), y.z = pgd_finite(y.z * inv), y.w = pgd_finite(y.w * inv);
    const size_t o = (size_t)row * a.os + (size_t)qh * HD + dim;
    if constexpr (XT == GQ_F32) gst<float4>((float *)a.out + o, y);
    else gst<uint2>((uint16_t *)a.out + o, make_uint2(pgd_pack(y.x, y.y), pgd_pack(y.z, y.w)));
  }
}

template <int CT, int XT, int HD, int RG>
int launch(const AttArgs &a, unsigned blocks, int tpt, hipStream_t s) {
  hipLaunchKernelGGL((prompt_kernel<CT, XT, HD, RG, 8 / RG>), dim3(blocks), dim3(kPThreads), 0, s, a);
  if (a.nch > 1) hipLaunchKernelGGL((prompt_merge_kernel<XT, HD>), dim3(a.b.n_tokens), dim3(kPThreads), 0, s, a, tpt);
  return hipGetLastError() == hipSuccess ? 0 : -4;
}

template <int CT, int XT>
int launch_hd(const AttArgs &a, int hd, const PromptShape &f, hipStream_t s) {
  const int tpt = f.rows / a.G;
  if constexpr (XT == GQ_BF16)
    if (f.rows == 256) return hd == 64 ? launch<CT, XT, 64, 8>(a, f.blocks, tpt, s) : launch<CT, XT, 128, 8>(a, f.blocks, tpt, s);
  return hd == 64 ? launch<CT, XT, 64, 4>(a, f.blocks, tpt, s) : launch<CT, XT, 128, 4>(a, f.blocks, tpt, s);
}

/* bytes of n parts' results, and their bound, which costs no time that shows: a
 * bf16 prompt of 64000 tokens (32 heads over 8 of 128) took 2.1 GB for 32.9 ms,
 * and takes 32.9 without */
size_t prompt_results(const AttArgs &a, int head_dim, int n) {
  return sizeof(float) * a.b.n_tokens * a.n_heads * n * (head_dim + 2);
}
constexpr size_t kResults = (size_t)512 << 20;

} // namespace

/* The launch: rows of a tile (256, or 128 where those leave CUs idle; fp32
 * queries always 128) and parts of a tile's keys, whichever should take least.
 * Microseconds: a workgroup, `fix` and `tau` a block of 64 keys; more of them
 * than CUs, their sum and a quarter of the longest for what the last ones leave
 * idle; parts, their merge.  Of the lengths the host knows the longest and the
 * number of new tokens alone, and takes the sequences for equally long.
 *
 * tau: one tile of 64 tokens over 8192 positions (32 heads over 8).  The other
 * constants were fitted to launches timed with every choice (1 to 8 sequences, 1
 * to 2000 new tokens at 0 to 8000, head groups of 1 to 8): over 170 others the
 * rule's choices take 3% more than the best ones together, 5% more for the worst
 * in ten; one part and 256 rows always, up to five times as long.
 */
PromptShape gq_paged_prompt_shape(const AttArgs &a, int cache, int xtype, int head_dim, int n_cu) {
  const bool f = xtype == GQ_F32, wide = head_dim > 64;
  const int t = cache == GQ_F32 ? 0 : cache == GQ_BF16 ? 1 : 2;
  constexpr double kTau[2][3][3] = {{{1.95, 1.32, 1.69}, {1.34, 0.97, 1.31}, {2.42, 1.53, 1.80}},  /* head_dim 64: bf16 queries in 256 and 128 rows, fp32 */
                                    {{3.10, 1.77, 2.28}, {2.29, 1.31, 1.55}, {5.66, 3.49, 3.61}}}; /* 128 */
  const double fix = (f ? 5.0 : 10.0) * (wide ? 1.0 : 0.3);
  const int seqs = std::min(a.b.n_seqs, a.b.n_tokens), each = (a.b.n_tokens + seqs - 1) / seqs;
  const int nblk = std::max(1, (a.b.max_len + kKeys - 1) / kKeys);
  const double mean = std::min((double)nblk, (std::max(0, a.b.max_len - each) + 0.5 * each) / kKeys + 1);
  PromptShape best{};
  double us = 1e30;
  for (int rows = f ? 128 : 256; rows >= 128; rows /= 2) {
    const int tpt = rows / a.G;
    const double w = (double)seqs * ((each + tpt - 1) / tpt) * a.c.n_kv, tau = kTau[wide][f ? 2 : rows == 128][t];
    const int most = pgd_launchable(a.b.n_tokens, kPThreads) ? std::min(16, nblk) : 1; /* the merge's launch */
    for (int k = 1; k <= most; k++) {
      const int span = (nblk + k - 1) / k, n = (nblk + span - 1) / span;
      if (n > 1 && prompt_results(a, head_dim, n) > kResults) break;
      const double parts = std::max(1.0, mean / span), longest = fix + tau * span;
      const double load = w * (parts * fix + tau * mean) / n_cu;
      double c = w * parts <= n_cu ? longest : std::max(longest, load + longest / 4);
      if (k > 1) c += 4 + 2e-6 * a.b.n_tokens * a.n_heads * head_dim * k;
      if (c < us) us = c, best.rows = rows, best.span = span, best.parts = n;
    }
  }
  const long long tiles = a.b.n_tokens / (best.rows / a.G) + seqs, blocks = tiles * a.c.n_kv * best.parts;
  best.blocks = pgd_launchable(blocks, kPThreads) ? (unsigned)blocks : 0u;
  return best;
}

int gq_launch_paged_prompt(const AttArgs &a, int cache, int xtype, int head_dim, const PromptShape &f, hipStream_t s) {
  const bool x = xtype == GQ_F32;
  if (cache == GQ_F32) return x ? launch_hd<GQ_F32, GQ_F32>(a, head_dim, f, s) : launch_hd<GQ_F32, GQ_BF16>(a, head_dim, f, s);
  if (cache == GQ_BF16) return x ? launch_hd<GQ_BF16, GQ_F32>(a, head_dim, f, s) : launch_hd<GQ_BF16, GQ_BF16>(a, head_dim, f, s);
  return x ? launch_hd<GQ_I8_ROWS, GQ_F32>(a, head_dim, f, s) : launch_hd<GQ_I8_ROWS, GQ_BF16>(a, head_dim, f, s);
}
