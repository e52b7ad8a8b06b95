// Single-token GQA attention on MFMA over a paged cache, bf16 or e4m3, with
// the work split over long sequences and prefixes that many rows share
// computed once for all of them (MI355X, gfx950).
//
//   out[b, h] = sum_j softmax_j(scale * q[b, h] . K_j) V_j,   j < seq_lens[b]
//
// A softmax over a union of token ranges joins from each range's
// (m = max s, l = sum exp(s - m), o = sum exp(s - m) V): with M = max m,
// out = sum exp(m - M) o / sum exp(m - M) l.  m, l, o are held in fp32 and s
// in units of log2, so that the exponential is one v_exp_f32.
//
// Everything is computed transposed, so that softmax stays inside a lane:
//   S^T = K Q^T  (A = K rows as they lie in the cache, B = Q rows),
//   O^T = V^T P^T (A = V^T through the LDS transposing read, B = P).
// C of the first product holds, for ONE query row per lane, the tokens
// g*4 + reg of each tile (g = the lane's group of 16, or of 32); B of the
// second wants 8 tokens a lane.  A sum over tokens may take them in any order,
// so B's slots m = 0..7 are read as {4 tokens of one half, 4 of the other}
// and V^T is read in the same order: P never leaves its registers.
//
// The matrix instruction takes bf16, so each weight of P goes through it as two
// terms: its upper bits, and what they leave out, rounded, which loses at most
// 2^-15 of it (one term alone would lose 2^-8, as much as the output's own
// rounding).  The sum l is the terms', so that the weights sum to 1.  Among own
// tokens the second term costs nothing (256 rows of 700 tokens 49 us either
// way), in the shared pass its products and splits take 512 rows with 3 prefixes
// of 8192 tokens from 134 to 156 us, 256 rows of 2048 from 64 to 67.
//
// e4m3 rows become bf16 on the way in (scale times code is exact in bf16), so
// both caches share one arithmetic.

#include "common.h"
#include "fp8.h"

#define HD 128
#define KVPAGE 64
#define MAXG 16        // query heads of one KV head: one MFMA column block
#define MAXGROUPS 64   // prefix groups of one call: one wave finds a tile's
#define MAXB 65535     // rows of one call
#define TILE 128       // query rows of one block in the shared pass
// Blocks of a launch's own tokens, two a CU.  Cold, e4m3, 32/8 heads: 8 rows of
// 32768 tokens 161 us at 256, 159 at 512, 165 at 1024; 64 rows of 1000 tokens
// 52.9, 52.2, 56.4.
#define ROOM 512
// Blocks of its prefixes, one a CU, beside which one of own tokens runs.  512
// rows in 3 groups of 8192 tokens (300 of their own, e4m3): 186 us at 192, 156
// at 256, 163 at 384, 172 at 512; 256 rows of 2048 tokens (300, bf16): 64.7,
// 67.2, 71.7, 77.4.
#define PRE_ROOM 256
// Pages of a prefix's piece, at least, and of a split where the row fills its
// table.  One row of 777 tokens in 13 pages 9.0 us at 1, 8.3 at 2, 9.2 at 4; 4
// rows of 1024 shared tokens 15.0, 14.2, 16.5.  The number of splits follows from
// the table's width, so that a short row in a wide table is cut finer, down to
// half pages.  The same bound on the device, for the row's length, takes one row
// of 100 tokens in 129 pages from 9.2 to 9.5 us and 32 of them from 9.5 to 8.7:
// not taken.  (3.3 of that is the join; in 2 pages, unsplit, 5.5 and 5.7.)
#define LEAST 2
// Splits of a row and pieces of a tile's prefix, at most: both together are
// joined by one wave.  One row of 32768 tokens 57 us at 8, 35 at 16, 33 at 32.
#define MAXPARTS 32
#define SLACK 8.f      // log2 by which a weight may pass 1

using f32x4 = __attribute__((ext_vector_type(4))) float;
using f32x16 = __attribute__((ext_vector_type(16))) float;
using bf16x8v = __attribute__((ext_vector_type(8))) __bf16;
using s16x4 = __attribute__((ext_vector_type(4))) short;
using s16x8 = __attribute__((ext_vector_type(8))) short;
using u32x4 = __attribute__((ext_vector_type(4))) unsigned;

#define MFMA16(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0)
#define MFMA32(a, b, c) __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0)

// The order of a block's instructions, by kind.
#define SCHED(kind, n) __builtin_amdgcn_sched_group_barrier(kind, n, 0)
#define MFMA 0x8
#define DS_READ 0x100

// Row pitch of V in LDS, in halfwords: 288 B = 72 banks, so that the 4-token
// blocks of a transposing read fall on banks 8 apart.
#define V_PITCH 144
// Row pitch of K: 272 B, 16 B reads of 16 rows cover all banks.
#define K_PITCH 136
// Of V in the shared kernel, whose reads take 32 dims of 4 tokens: 320 B, the
// tokens fall 16 banks apart.
#define V_PITCH32 160

namespace {

// 4 tokens x 16 dims of 16 lanes, transposed: lane i gets dim i's 4 tokens.
__device__ __forceinline__ s16x4 read_tr(const __hip_bfloat16* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) s16x4*)(p));
}

__device__ __forceinline__ bf16x8v join(s16x4 a, s16x4 b) {
  const s16x8 r = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  return __builtin_bit_cast(bf16x8v, r);
}

// 16 codes of one row -> two vectors of 8 bf16.
__device__ __forceinline__ void widen(const u32x4 c, const float s, u32x4& lo,
                                      u32x4& hi) {
  lo = (u32x4){e4m3_to_bf16x2<false>(c[0], s), e4m3_to_bf16x2<true>(c[0], s),
               e4m3_to_bf16x2<false>(c[1], s), e4m3_to_bf16x2<true>(c[1], s)};
  hi = (u32x4){e4m3_to_bf16x2<false>(c[2], s), e4m3_to_bf16x2<true>(c[2], s),
               e4m3_to_bf16x2<false>(c[3], s), e4m3_to_bf16x2<true>(c[3], s)};
}

__device__ __forceinline__ float exp2_fast(const float x) {
  return __builtin_amdgcn_exp2f(x);
}

// l + the sum of 8 bf16, two a dot product with ones, each sum in fp32.
__device__ __forceinline__ float add8(const bf16x8v p, float l) {
  using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
  const bf16x2 ones = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    l = __builtin_amdgcn_fdot2_f32_bf16((bf16x2){p[2 * j], p[2 * j + 1]}, ones,
                                        l, false);
  return l;
}

// Weights (0 and up) as two bf16 terms each: the first is the number next below
// cut to bf16, so that both are above 0 where the weight is, and an infinite
// value of V stays one (0 times it would be NaN).
struct Terms {
  u32x4 hi, lo;
};
__device__ __forceinline__ void split2(const float p, const float q, Terms& t,
                                       const int at) {
  using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
  const unsigned u =
      __builtin_elementwise_sub_sat(__float_as_uint(p), 1u) & 0xffff0000u;
  const unsigned v =
      __builtin_elementwise_sub_sat(__float_as_uint(q), 1u) & 0xffff0000u;
  t.hi[at] = __builtin_amdgcn_perm(v, u, 0x07060302);
  t.lo[at] = __builtin_bit_cast(
      unsigned,
      (bf16x2){(__bf16)(p - __uint_as_float(u)),
               (__bf16)(q - __uint_as_float(v))});
}

struct Paged {
  const void* kcache;        // [P, hkv, 64, 128] bf16 or e4m3
  const void* vcache;
  const uint8_t* kscale;     // [P, hkv, 64] or null
  const uint8_t* vscale;
  const __hip_bfloat16* q;   // [B, hq, 128], rows q_stride apart
  const int32_t* page_table;  // [B, max_pages]
  const int32_t* seq_lens;    // [B]
  const int32_t* group;       // [B] or null: prefix group, < 0 for none
  const int32_t* group_lens;  // [ngroups] tokens of each group's prefix
  float* part_o;              // [B * hq, nsplit, 128]
  float* part_ml;             // [B * hq, nsplit, 2]
  float* pre_o;               // [pieces, hkv, 128, 128]
  float* pre_ml;              // [pieces, hkv, 128, 2]
  int4* pre_at;               // [B] where a row's are: first piece, pieces, row
  int32_t* pre_has;           // [B] whether a row has any
  int64_t q_stride;
  int B, hq, hkv, G, max_pages, num_pages, ngroups;
  int nsplit;           // of each row's own tokens
  int npre;             // blocks of a KV head in the shared pass
  float scale_log2;     // |scale| * log2(e), above 0
  unsigned flip;        // sign bits for the queries where scale < 0
};

__device__ __forceinline__ int row_len(const Paged& a, const int b) {
  return min(max(a.seq_lens[b], 0), a.max_pages * KVPAGE);
}

// Tokens of row b that its group's shared pass covers: the prefix, or nothing
// of a row that ends inside it (a weight of 0 would not keep out what a token
// past the row's end holds, if that is not finite).
__device__ __forceinline__ int prefix_len(const Paged& a, const int b,
                                          const int n) {
  if (a.group == nullptr) return 0;
  const int g = a.group[b];
  const int p = (g >= 0 && g < a.ngroups) ? max(a.group_lens[g], 0) : 0;
  return p <= n ? p : 0;
}

// A row's first partial result of the prefix, for the first head of kvh; the
// next piece's is hkv * TILE rows on.
__device__ __forceinline__ int64_t prefix_row(const Paged& a, const int4 at,
                                              const int kvh) {
  return ((int64_t)at.x * a.hkv + kvh) * TILE + at.z * a.G;
}

// 8 query values, their signs turned where the scale is negative: the scale's
// own factor is then positive, and the largest score is the largest product.
__device__ __forceinline__ bf16x8v load_q(const Paged& a,
                                          const __hip_bfloat16* src) {
  return __builtin_bit_cast(bf16x8v,
                            *reinterpret_cast<const u32x4*>(src) ^ a.flip);
}

// Weights that join up to 64 partial results, one a lane: exp2(m - M) where
// the lane's l is not 0 (its o is not read otherwise), and their sum of l.
__device__ __forceinline__ float join_weight(const float m, const float l,
                                             float& M, float& L) {
  M = wave_max(m);
  const float mu = (M == -INFINITY) ? 0.f : M;
  const float w = (l == 0.f) ? 0.f : exp2_fast(m - mu);
  L = wave_sum(l == 0.f ? 0.f : w * l);
  return w;
}

}  // namespace

// ------------------------------------------------------------ each row's own
//
// One block = (row, KV head, split): NW waves take the split's half pages in
// turn.  A wave reads K straight into A fragments (a lane's 16 B of one token;
// the Q fragments take the dims in the same order) and turns V in its own LDS
// rows, so that the loop has no block barrier.  Half pages, because 122
// registers and 9 KB a wave let 4 blocks share a CU: what hides the loads'
// latency is other waves (whole pages: 2 blocks, 55.9 us where this takes 49;
// the next half page's loads under this one's products gained nothing).  Page
// ids come 64 at a time, one a lane.
//
// Bound: the bytes of the cache, in random panels of 4 KB (bf16: 8 KB) halves.
// e4m3, 256 rows of 700 tokens, again and again / with other memory read between:
// 71 / 126 us, a kernel that loads their pages and does nothing else 61 / 123; 8
// rows of 32768 tokens 102 / 160, the loads 92 / 156.  Measured on changing
// inputs, 32/8 heads: 256 rows of up to 700 tokens 49 us, 4.2 TB/s; 8 rows of up
// to 32768 tokens (64/8 heads) 93 us, 5.0 TB/s; one row of 777 tokens 9.6 us, of
// which the join is 3.3.  The matrix instructions run mostly empty (2G of 16
// columns) and still take a tenth of the vector instructions that dot products
// would.
#define UNIT 32  // tokens of one step

#define NW 4  // waves of a block

struct OwnLds {
  __hip_bfloat16 v[NW][UNIT * V_PITCH];
  float ml[NW][MAXG][2];
};

template <bool FP8, bool WIDE>
__device__ __forceinline__ void own_tokens(const Paged& a,
                                           __hip_bfloat16* __restrict__ out,
                                           const int kvh, const int b,
                                           const int split, OwnLds& L) {
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int lane = threadIdx.x % WAVE;
  const int l16 = lane & 15, g4 = lane >> 4;
  const int32_t* table = a.page_table + (int64_t)b * a.max_pages;
  // the first page ids of a row's start, before its length is known (256 rows
  // of 2048 + 300 tokens 66.8 -> 64.4 us)
  int ids = a.max_pages > 0
                ? table[min((wid + lane * NW) / (KVPAGE / UNIT),
                            a.max_pages - 1)]
                : -1;
  const int n = row_len(a, b);
  const int first = prefix_len(a, b, n);
  const int unit0 = first / UNIT;
  const int nunits = (n + UNIT - 1) / UNIT - unit0;
  const int each = (max(nunits, 0) + a.nsplit - 1) / a.nsplit;
  const int ubegin = unit0 + split * each + wid;
  const int uend = unit0 + min(nunits, (split + 1) * each);
  const int steps = uend > ubegin ? (uend - ubegin + NW - 1) / NW : 0;

  // Columns: G query heads, and where 2G fit into 16, the same heads again,
  // for their weights' second terms: the instructions are the same.
  const int cols = WIDE ? a.G : 2 * a.G;
  const bool second = !WIDE && l16 >= a.G;

  // fragment c of lane group g4 holds dims 32c + 8*g4 .. of a bf16 row, or of
  // an e4m3 row (whose 16 B are 16 dims) 64*(c/2) + 16*g4 + 8*(c%2) ..
  bf16x8v qf[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int d = FP8 ? (c / 2) * 64 + g4 * 16 + (c % 2) * 8 : c * 32 + g4 * 8;
    const u32x4 none = {0, 0, 0, 0};
    qf[c] = __builtin_bit_cast(bf16x8v, none);
    if (l16 < cols)
      qf[c] = load_q(a, a.q + b * a.q_stride +
                            (kvh * a.G + l16 - (second ? a.G : 0)) * HD + d);
  }

  float m = -INFINITY, l = 0.f;
  f32x4 o[8];
#pragma unroll
  for (int d = 0; d < 8; ++d) o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};

  __hip_bfloat16* vt = L.v[wid];
  const __hip_bfloat16* vt_read =
      vt + (g4 * 4 + (l16 >> 2)) * V_PITCH + (l16 & 3) * 4;

  constexpr int ROWB = FP8 ? HD : 2 * HD;  // bytes of a cache row
  constexpr int KLD = FP8 ? 2 : 4;    // 16 B loads of a lane, a 16-token tile
  constexpr int VROW = FP8 ? 8 : 16;  // lanes of one row of V
  constexpr int VLD = UNIT * VROW / WAVE;
  const int koff = l16 * ROWB + g4 * 16, voff = lane * 16;

  for (int i = 0; i < steps; ++i) {
    const int u = ubegin + i * NW;
    if (i % WAVE == 0 && (i > 0 || ubegin != wid)) {
      const int mine = u + lane * NW;
      ids = mine < uend ? table[mine / (KVPAGE / UNIT)] : -1;
    }
    const int page = __builtin_amdgcn_readlane(ids, i % WAVE);
    if (page < 0 || page >= a.num_pages) continue;  // no such page: no tokens
    const int tok0 = u * UNIT;
    const int64_t panel = ((int64_t)page * a.hkv + kvh) * KVPAGE +
                          (u % (KVPAGE / UNIT)) * UNIT;
    const bool whole = tok0 >= first && tok0 + UNIT <= n;

    u32x4 kr[2][KLD], vr[VLD];
    unsigned char ks[2], vs[VLD];
    const char* kp = (const char*)a.kcache + panel * ROWB;
    const char* vp = (const char*)a.vcache + panel * ROWB;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int c = 0; c < KLD; ++c)
        kr[t][c] = *reinterpret_cast<const u32x4*>(kp + t * 16 * ROWB + c * 64 +
                                                   koff);
      if (FP8) ks[t] = (a.kscale + panel)[t * 16 + l16];
    }
#pragma unroll
    for (int j = 0; j < VLD; ++j) {
      vr[j] = *reinterpret_cast<const u32x4*>(vp + j * WAVE * 16 + voff);
      if (FP8) vs[j] = (a.vscale + panel)[j * (WAVE / VROW) + lane / VROW];
    }

    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      u32x4 kf[4];
      if constexpr (FP8) {
        const float sc = e8m0_scale(ks[t]);
        widen(kr[t][0], sc, kf[0], kf[1]);
        widen(kr[t][1], sc, kf[2], kf[3]);
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) kf[c] = kr[t][c];
      }
      s[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 4; ++c)
        s[t] = MFMA16(__builtin_bit_cast(bf16x8v, kf[c]), qf[c], s[t]);
    }
    if (!whole) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int tok = tok0 + t * 16 + g4 * 4 + r;
          if (tok < first || tok >= n) s[t][r] = -INFINITY;
        }
    }
    float mt = s[0][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mt = fmaxf(mt, s[j / 4][j % 4]);
    mt = fmaxf(mt, __shfl_xor(mt, 16, WAVE));
    mt = fmaxf(mt, __shfl_xor(mt, 32, WAVE));
    const float mn = fmaxf(m, mt * a.scale_log2);
    const float mu = (mn == -INFINITY) ? 0.f : mn;  // nothing seen yet
    if (__any(mn > m)) {  // a factor of 1 otherwise
      const float keep = exp2_fast(m - mu);
      l *= keep;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d] *= keep;
    }
    m = mn;
    Terms p2;
#pragma unroll
    for (int j = 0; j < 8; j += 2)
      split2(exp2_fast(fmaf(s[j / 4][j % 4], a.scale_log2, -mu)),
             exp2_fast(fmaf(s[j / 4][j % 4 + 1], a.scale_log2, -mu)), p2,
             j / 2);
    if constexpr (!WIDE) p2.hi = second ? p2.lo : p2.hi;
    const bf16x8v pf = __builtin_bit_cast(bf16x8v, p2.hi);
    const bf16x8v pl = __builtin_bit_cast(bf16x8v, p2.lo);
    l = add8(pf, l);
    if constexpr (WIDE) l = add8(pl, l);

    // V to LDS as bf16; rows outside the sequence as zeros (weight 0 times
    // whatever a recycled page holds may be NaN)
#pragma unroll
    for (int j = 0; j < VLD; ++j) {
      const int row = j * (WAVE / VROW) + lane / VROW;
      const bool gone =
          !whole && (tok0 + row < first || tok0 + row >= n);
      __hip_bfloat16* dst = vt + row * V_PITCH;
      if constexpr (FP8) {
        u32x4 lo, hi;
        if (gone) vr[j] = (u32x4){0, 0, 0, 0};
        widen(vr[j], gone ? 1.f : e8m0_scale(vs[j]), lo, hi);
        dst += (lane % VROW) * 16;
        reinterpret_cast<u32x4*>(dst)[0] = lo;
        reinterpret_cast<u32x4*>(dst)[1] = hi;
      } else {
        if (gone) vr[j] = (u32x4){0, 0, 0, 0};
        reinterpret_cast<u32x4*>(dst + (lane % VROW) * 8)[0] = vr[j];
      }
    }
    // one wave's LDS operations run in order: only the compiler has to be told
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const bf16x8v v = join(read_tr(vt_read + d * 16),
                             read_tr(vt_read + d * 16 + 16 * V_PITCH));
      o[d] = MFMA16(v, pf, o[d]);
      if constexpr (WIDE) o[d] = MFMA16(v, pl, o[d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }

  l += __shfl_xor(l, 16, WAVE);
  l += __shfl_xor(l, 32, WAVE);

  // ---- join the waves: O rows over the V rows, now free.  The whole row
  // where nothing else is joined to it, else a partial result
  const bool whole_row = a.nsplit == 1 && first == 0;
  if (a.npre > 0 && kvh == 0 && split == 0 && threadIdx.x == 0)
    a.pre_has[b] = first > 0;
  __syncthreads();
  float* o_lds = reinterpret_cast<float*>(&L.v[0][0]);  // [NW][16][128]
  float* w_lds = o_lds + NW * MAXG * HD;                 // [16][NW]
  static_assert((NW * MAXG * HD + MAXG * NW) * 4 <= sizeof(L.v),
                "O and the weights fit V's rows");
  if (l16 < cols) {
#pragma unroll
    for (int d = 0; d < 8; ++d)
      *reinterpret_cast<f32x4*>(
          &o_lds[(wid * MAXG + l16) * HD + d * 16 + g4 * 4]) = o[d];
    if (g4 == 0) {
      L.ml[wid][l16][0] = m;
      L.ml[wid][l16][1] = l;
    }
  }
  __syncthreads();
  for (int g = wid; g < a.G; g += NW) {
    const int64_t row = (int64_t)b * a.hq + kvh * a.G + g;
    float mk = -INFINITY, lk = 0.f, M, S;
    if (lane < NW) {
      mk = L.ml[lane][g][0];
      lk = L.ml[lane][g][1];
      if constexpr (!WIDE) lk += L.ml[lane][a.G + g][1];
    }
    const float w = join_weight(mk, lk, M, S);
    // no weight at all (an empty row): zeros
    if (lane < NW)
      w_lds[g * NW + lane] = !whole_row ? w : S == 0.f ? 0.f : w / S;
    if (!whole_row && lane == 0)
      reinterpret_cast<float2*>(a.part_ml)[row * a.nsplit + split] =
          make_float2(M, S);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.G * (HD / 2); i += NW * WAVE) {
    const int g = i / (HD / 2), d = i % (HD / 2) * 2;
    const int64_t row = (int64_t)b * a.hq + kvh * a.G + g;
    float2 acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const float w = w_lds[g * NW + k];
      float2 x =
          *reinterpret_cast<const float2*>(&o_lds[(k * MAXG + g) * HD + d]);
      if constexpr (!WIDE) {
        const float2 y = *reinterpret_cast<const float2*>(
            &o_lds[(k * MAXG + a.G + g) * HD + d]);
        x.x += y.x;
        x.y += y.y;
      }
      acc.x = fmaf(w, x.x, acc.x);
      acc.y = fmaf(w, x.y, acc.y);
    }
    if (whole_row) {
      __hip_bfloat16* dst = out + row * HD + d;
      dst[0] = f2bf(acc.x);
      dst[1] = f2bf(acc.y);
    } else {
      *reinterpret_cast<float2*>(
          a.part_o + (row * a.nsplit + split) * HD + d) = acc;
    }
  }
}

// Joins the partial slots of one (row, head): a wave each, 2 dims a lane.  The
// first AHEAD o's of the row's own splits are read before their weights are
// known: room for 32 where there are many (one row of 4096 tokens 12.2 us, with
// room for 8 17.7), for 8 where there are not, and many rows take the registers.
template <int AHEAD>
__global__ __launch_bounds__(4 * WAVE) void paged_join_kernel(
    const Paged a, __hip_bfloat16* __restrict__ out) {
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int64_t row = (int64_t)blockIdx.x * 4 + wid;
  if (row >= (int64_t)a.B * a.hq) return;
  const int lane = threadIdx.x % WAVE;
  const int b = (int)(row / a.hq);  // one a wave: its branches are uniform
  int4 at = make_int4(0, 0, 0, 0);
  if (a.npre > 0) {
    at = a.pre_at[b];  // not written where the row has none
    if (a.pre_has[b] == 0) at.y = 0;
  }
  const int joined = at.y;
  if (a.nsplit == 1 && joined == 0) return;  // written whole
  const int own = a.nsplit;  // up to 32, as of prefixes
  // what is not written (an empty range) weighs nothing
  constexpr int PRE_AHEAD = 8;
  const float2* part =
      reinterpret_cast<const float2*>(a.part_o + row * own * HD) + lane;
  float2 x[AHEAD], y[PRE_AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (k < own) x[k] = part[k * (HD / 2)];
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < own)
    ml = reinterpret_cast<const float2*>(a.part_ml)[row * own + lane];
  const int head = (int)(row - (int64_t)b * a.hq);
  const int64_t first = prefix_row(a, at, head / a.G) + head % a.G;
  const int64_t step = (int64_t)a.hkv * TILE * (HD / 2);
  const float2* pre =
      reinterpret_cast<const float2*>(a.pre_o + first * HD) + lane;
#pragma unroll
  for (int k = 0; k < PRE_AHEAD; ++k)
    if (k < joined) y[k] = pre[k * step];
  if (lane >= own && lane - own < joined)
    ml = reinterpret_cast<const float2*>(
        a.pre_ml)[first + (int64_t)(lane - own) * a.hkv * TILE];
  float M, L;
  const float w = join_weight(ml.x, ml.y, M, L);
  float2 acc = make_float2(0.f, 0.f);
  const auto add = [&](const int k, const float2 o)
      __attribute__((always_inline)) {
    const float wk =
        __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), k));
    acc.x = wk == 0.f ? acc.x : fmaf(wk, o.x, acc.x);
    acc.y = wk == 0.f ? acc.y : fmaf(wk, o.y, acc.y);
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (k < own) add(k, x[k]);
#pragma unroll
  for (int k = 0; k < PRE_AHEAD; ++k)
    if (k < joined) add(own + k, y[k]);
#pragma unroll 8
  for (int k = PRE_AHEAD; k < joined; ++k) add(own + k, pre[k * step]);
  const float inv = (L == 0.f) ? 0.f : 1.f / L;
  __hip_bfloat16* dst = out + row * HD + lane * 2;
  dst[0] = f2bf(L == 0.f ? 0.f : acc.x * inv);
  dst[1] = f2bf(L == 0.f ? 0.f : acc.y * inv);
}

// -------------------------------------------------------- the shared prefix
//
// A tile is up to 128 query rows (b, g) of one group's members, in batch order;
// its work is its prefix's pages.  A KV head's blocks take equal runs of all
// its tiles' pages, one after the other, as the groups are on the device: a
// block may end one tile and begin the next, each such piece leaves a partial
// result, and no block idles for the number of rows or groups.  4 waves own 32
// rows each; pages of K and V pass through LDS, double-buffered, the next
// page's loads in flight under this page's products.  Bound: the matrix
// instructions and, at 32 rows a wave, LDS reads at the same rate (each 1 KB
// fragment feeds one 32x32x16 product of 32 cycles, four SIMDs to 128 B a
// cycle; V's feed two, a weight's terms).  Measured without own tokens, with the
// join: 512 rows (32/8 heads) in 3 groups of 8192 e4m3 tokens 147 us (125 with
// one term a weight), 470 TFLOP/s without the second terms' products; 256 rows
// of 2048 bf16 tokens 38 us.  With own tokens, of a CU's busy cycles the matrix
// units work 31 %, the vector units 44 %, LDS 33 %: one wave a SIMD alternates
// between exponentials and products.  blockIdx.x % hkv is the KV head, so that
// with 8 of them each XCD's L2 holds one head's prefixes for every tile.
struct PrefixLds {
  // two pages of K, then two of V
  __hip_bfloat16 pages[2 * KVPAGE * (K_PITCH + V_PITCH32)];
  unsigned long long longest;  // length of a tile's row << 32 | row
  int2 all_work;  // pages of all tiles, of the longest prefix
  // of each group: rows, prefix, its pages, tiles before it, work before and
  // up to its end
  int counts[MAXGROUPS], len[MAXGROUPS], pages_of[MAXGROUPS], tile0[MAXGROUPS],
      work0[MAXGROUPS], work1[MAXGROUPS];
  int tile_rows[TILE];
  int tile_count;
};

template <bool FP8>
__device__ __forceinline__ void prefix_pieces(const Paged& a, const int kvh,
                                              const int block, PrefixLds& L) {
  __hip_bfloat16* const k_lds = L.pages;
  __hip_bfloat16* const v_lds = L.pages + 2 * KVPAGE * K_PITCH;
  const int tid = threadIdx.x;
  const int wid = __builtin_amdgcn_readfirstlane(tid / WAVE);
  const int lane = tid % WAVE;
  const int r32 = lane & 31, h = lane >> 5;
  const int per_tile = TILE / a.G;

  // ---- the groups' tiles and work, one group a lane
  if (tid < MAXGROUPS) L.counts[tid] = 0;
  __syncthreads();
  const int len = lane < a.ngroups ? max(a.group_lens[lane], 0) : 0;
  const int first = tid < a.B ? a.group[tid] : -1;
  for (int b = tid; b < a.B; b += 4 * WAVE) {
    const int g = b == tid ? first : a.group[b];
    if (g >= 0 && g < a.ngroups) atomicAdd(&L.counts[g], 1);
  }
  __syncthreads();
  if (wid == 0) {
    // (any int32 may be a length: no sum that passes 2^31)
    const int pages = min(len / KVPAGE + (len % KVPAGE != 0), a.max_pages);
    const int tiles = (L.counts[lane] + per_tile - 1) / per_tile;
    int tiles_to = tiles, work = tiles * pages;
    int most = tiles > 0 ? pages : 0;
#pragma unroll
    for (int off = 1; off < WAVE; off <<= 1) {
      const int x = __shfl_up(tiles_to, off, WAVE);
      const int y = __shfl_up(work, off, WAVE);
      if (lane >= off) {
        tiles_to += x;
        work += y;
      }
      most = max(most, __shfl_xor(most, off, WAVE));
    }
    L.len[lane] = len;
    L.pages_of[lane] = pages;
    L.tile0[lane] = tiles_to - tiles;
    L.work0[lane] = work - tiles * pages;
    L.work1[lane] = work;
    if (lane == WAVE - 1) L.all_work = make_int2(work, most);
  }
  __syncthreads();
  const int work = __builtin_amdgcn_readfirstlane(L.all_work.x);
  // a tile ends in up to one piece more than its pages fill
  const int each =
      max(max((work + a.npre - 1) / a.npre, LEAST),
          (__builtin_amdgcn_readfirstlane(L.all_work.y) + MAXPARTS - 2) /
              (MAXPARTS - 1));
  const int work_end = min(work, (block + 1) * each);
  int at = block * each;
  while (at < work_end) {
    // ---- this piece's group, tile, pages and rows: each row's group goes to
    // LDS (a byte, in what the pages take later), one wave walks the members
    const int grp = __ffsll((long long)__ballot(at < L.work1[lane])) - 1;
    const int pages = __builtin_amdgcn_readfirstlane(L.pages_of[grp]);
    const int into = at - __builtin_amdgcn_readfirstlane(L.work0[grp]);
    const int tile = into / pages;  // of the group's
    const int pbegin = into % pages;
    const int piece =
        block + tile + __builtin_amdgcn_readfirstlane(L.tile0[grp]);
    const int taken = min(pages - pbegin, work_end - at);
    const int tile_end = at - pbegin + pages;  // in the head's work
    at += taken;

    unsigned char* groups = reinterpret_cast<unsigned char*>(L.pages);
    static_assert(MAXB <= sizeof(L.pages), "a byte a row");
    __syncthreads();  // nothing reads the last piece's pages or rows
    for (int b = tid; b < a.B; b += 4 * WAVE)
      groups[b] = (b == tid ? first : a.group[b]) == grp;
    if (tid == 0) L.longest = 0;
    __syncthreads();
    if (wid == 0) {
      const int skip = tile * per_tile;
      int seen = 0;
      for (int b0 = 0; b0 < a.B && seen < skip + per_tile; b0 += WAVE) {
        const bool in = b0 + lane < a.B && groups[b0 + lane];
        const unsigned long long bal = __ballot(in);
        const int rank = seen + __popcll(bal & ((1ull << lane) - 1)) - skip;
        if (in && rank >= 0 && rank < per_tile) L.tile_rows[rank] = b0 + lane;
        seen += __popcll(bal);
      }
      if (lane == 0) L.tile_count = min(seen - skip, per_tile);
    }
    __syncthreads();
    const int nrows = L.tile_count * a.G;
    if (pbegin == 0 && kvh == 0 && tid < L.tile_count)
      a.pre_at[L.tile_rows[tid]] =
          make_int4(piece, (tile_end - 1) / each - block + 1, tid, 0);

    // ---- this wave's 32 query rows: one a lane, halves h of the MFMA's K
    const int i = wid * 32 + r32;
    const bool live = i < nrows;
    const int b = L.tile_rows[live ? i / a.G : 0];
    const int head = kvh * a.G + (live ? i % a.G : 0);
    const bool wave_live = wid * 32 < nrows;
    bf16x8v qf[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      qf[k] = load_q(a, a.q + b * a.q_stride + head * HD + k * 16 + h * 8);
    // (a lane without a row computes row 0 again and writes nothing)
    if (live)
      atomicMax(&L.longest,
                (unsigned long long)row_len(a, b) << 32 | (unsigned)b);
    __syncthreads();
    // the longest row's pages (a shorter one's table may end before), none if
    // it ends inside the prefix
    const int glen = __builtin_amdgcn_readfirstlane(L.len[grp]);
    const int32_t* table =
        a.page_table + (int64_t)(unsigned)L.longest * a.max_pages;
    const int pend = glen <= (int)(L.longest >> 32) ? pbegin + taken : pbegin;

    float m = -INFINITY, l = 0.f;
    f32x16 o[4];
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.f;

    constexpr int LD = FP8 ? 2 : 4;     // 16 B loads of a thread, a page
    constexpr int ROW = FP8 ? 8 : 16;   // threads of one row
    u32x4 kr[LD], vr[LD];
    unsigned char ks[LD], vs[LD];
    const int trow = tid / ROW, tcol = tid % ROW;

    // page ids 64 at a time, one a lane: no load waits for another
    int ids = 0;
    auto fetch = [&](int pi) {
      if ((pi - pbegin) % WAVE == 0)
        ids = pi + lane < pend ? table[pi + lane] : -1;
      const int page = __builtin_amdgcn_readlane(ids, (pi - pbegin) % WAVE);
      const bool ok = page >= 0 && page < a.num_pages;
      const int64_t panel = ((int64_t)(ok ? page : 0) * a.hkv + kvh) * KVPAGE;
      const char* kp = (const char*)a.kcache + panel * (FP8 ? HD : 2 * HD);
      const char* vp = (const char*)a.vcache + panel * (FP8 ? HD : 2 * HD);
#pragma unroll
      for (int j = 0; j < LD; ++j) {
        kr[j] = *reinterpret_cast<const u32x4*>(kp + (j * 4 * WAVE + tid) * 16);
        vr[j] = *reinterpret_cast<const u32x4*>(vp + (j * 4 * WAVE + tid) * 16);
        if (FP8) {
          const int64_t at = panel + j * (4 * WAVE / ROW) + trow;
          ks[j] = a.kscale[at];
          vs[j] = a.vscale[at];
        }
      }
      return ok;
    };
    auto stage = [&](int buf, int pi) {
      const bool whole = (pi + 1) * KVPAGE <= glen;
#pragma unroll
      for (int j = 0; j < LD; ++j) {
        const int row = j * (4 * WAVE / ROW) + trow;
        // beyond the prefix: zeros (NaN there times weight 0)
        if (!whole && pi * KVPAGE + row >= glen) {
          vr[j] = (u32x4){0, 0, 0, 0};
          if (FP8) vs[j] = 127;
        }
        __hip_bfloat16* kd = &k_lds[(buf * KVPAGE + row) * K_PITCH];
        __hip_bfloat16* vd = &v_lds[(buf * KVPAGE + row) * V_PITCH32];
        if constexpr (FP8) {
          u32x4 lo, hi;
          widen(kr[j], e8m0_scale(ks[j]), lo, hi);
          reinterpret_cast<u32x4*>(kd + tcol * 16)[0] = lo;
          reinterpret_cast<u32x4*>(kd + tcol * 16)[1] = hi;
          widen(vr[j], e8m0_scale(vs[j]), lo, hi);
          reinterpret_cast<u32x4*>(vd + tcol * 16)[0] = lo;
          reinterpret_cast<u32x4*>(vd + tcol * 16)[1] = hi;
        } else {
          reinterpret_cast<u32x4*>(kd + tcol * 8)[0] = kr[j];
          reinterpret_cast<u32x4*>(vd + tcol * 8)[0] = vr[j];
        }
      }
    };

    bool ok = false;
    if (pbegin < pend) {
      ok = fetch(pbegin);
      stage(0, pbegin);
    }
    for (int pi = pbegin; pi < pend; ++pi) {
      __syncthreads();  // this page is staged; the other buffer is free
      const int buf = (pi - pbegin) & 1;
      const bool cur = ok;
      if (pi + 1 < pend) ok = fetch(pi + 1);
      if (wave_live && cur) {
        const __hip_bfloat16* kt =
            &k_lds[(buf * KVPAGE + r32) * K_PITCH + h * 8];
        const __hip_bfloat16* vt =
            &v_lds[(buf * KVPAGE + 4 * h + ((lane & 15) >> 2)) * V_PITCH32 +
                   ((lane >> 4) & 1) * 16 + (lane & 3) * 4];
        f32x16 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            s[t] = MFMA32(*reinterpret_cast<const bf16x8v*>(
                              kt + t * 32 * K_PITCH + k * 16),
                          qf[k], s[t]);
        // six fragments ahead of the products (the compiler's own order has
        // two, each product waits for LDS: 27.4 us against 25.7 for the
        // prefixes of 256 rows with 2048 shared tokens, bf16)
        SCHED(DS_READ, 6);
#pragma unroll
        for (int k = 0; k < 10; ++k) {
          SCHED(MFMA, 1);
          SCHED(DS_READ, 1);
        }
        SCHED(MFMA, 6);
        if ((pi + 1) * KVPAGE > glen) {
          // the prefix's tokens of the page, from this lane's first one
          const int left = glen - pi * KVPAGE - 4 * h;
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (t * 32 + 8 * (r / 4) + r % 4 >= left)
                s[t][r] = -INFINITY;
        }
        float mt = s[0][0];
#pragma unroll
        for (int j = 1; j < 32; ++j) mt = fmaxf(mt, s[j / 16][j % 16]);
        mt = fmaxf(mt, __shfl_xor(mt, 32, WAVE));
        const float mn = mt * a.scale_log2;
        if (__any(mn > m + SLACK)) {
          const float mu = fmaxf(m, mn);
          const float keep = exp2_fast(m - (mu == -INFINITY ? 0.f : mu));
          m = mu;
          l *= keep;
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d] *= keep;
        }
        const float mu = (m == -INFINITY) ? 0.f : m;
        bf16x8v pf[4], pl[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          Terms p2;
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const f32x16& x = s[u / 2];
            const int r = u % 2 * 8 + j;
            split2(exp2_fast(fmaf(x[r], a.scale_log2, -mu)),
                   exp2_fast(fmaf(x[r + 1], a.scale_log2, -mu)), p2, j / 2);
          }
          pf[u] = __builtin_bit_cast(bf16x8v, p2.hi);
          pl[u] = __builtin_bit_cast(bf16x8v, p2.lo);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) l = add8(pl[u], add8(pf[u], l));
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int d = 0; d < 4; ++d) {
            const __hip_bfloat16* p = vt + u * 16 * V_PITCH32 + d * 32;
            const bf16x8v v = join(read_tr(p), read_tr(p + 8 * V_PITCH32));
            o[d] = MFMA32(v, pf[u], o[d]);
            o[d] = MFMA32(v, pl[u], o[d]);
          }
        SCHED(DS_READ, 8);
#pragma unroll
        for (int k = 0; k < 12; ++k) {
          SCHED(MFMA, 2);
          SCHED(DS_READ, 2);
        }
        SCHED(MFMA, 8);
      }
      if (pi + 1 < pend) stage(buf ^ 1, pi + 1);
    }

    l += __shfl_xor(l, 32, WAVE);
    if (live) {
      const int64_t slot =
          prefix_row(a, make_int4(piece, 0, i / a.G, 0), kvh) + i % a.G;
      if (h == 0) reinterpret_cast<float2*>(a.pre_ml)[slot] = make_float2(m, l);
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *reinterpret_cast<f32x4*>(
              &a.pre_o[slot * HD + d * 32 + r * 8 + h * 4]) =
              (f32x4){o[d][r * 4], o[d][r * 4 + 1], o[d][r * 4 + 2],
                      o[d][r * 4 + 3]};
    }
  }
}

// Both in one launch: a KV head's first npre blocks are the prefixes', bound by
// products, the others its rows' own tokens, bound by bytes, and each covers
// the other's waits: with one term a weight 512 rows in 3 groups of 8192 + 300
// tokens took 134 us where the two one after the other took 142, 256 rows of
// 2048 + 300 67 / 71, 4 rows of 1024 + 90 13.1 / 18.0.  Two blocks a CU cost the
// own tokens nothing (256 rows of 700, cold: 125.1 us at four, 126.5 at two).
template <bool FP8, bool WIDE>
__global__ __launch_bounds__(NW * WAVE, 2) void paged_shared_kernel(
    const Paged a, __hip_bfloat16* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) union {
    PrefixLds prefix;
    OwnLds own;
  } L;
  const int kvh = blockIdx.x % a.hkv, i = blockIdx.x / a.hkv;
  if (i < a.npre)
    prefix_pieces<FP8>(a, kvh, i, L.prefix);
  else
    own_tokens<FP8, WIDE>(a, out, kvh, (i - a.npre) / a.nsplit,
                    (i - a.npre) % a.nsplit, L.own);
}

template <bool FP8, bool WIDE>
__global__ __launch_bounds__(NW * WAVE, 4) void paged_decode_kernel(
    const Paged a, __hip_bfloat16* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) OwnLds L;
  own_tokens<FP8, WIDE>(a, out, blockIdx.x, blockIdx.y, blockIdx.z, L);
}

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <cmath>

namespace {

// Fills the arguments both entry points share, after checking them.
Paged paged_args(const torch::Tensor& out, const torch::Tensor& q,
                 const torch::Tensor& kcache, const torch::Tensor& vcache,
                 const torch::Tensor& page_table,
                 const torch::Tensor& seq_lens, double scale) {
  const auto dev = q.device();
  TORCH_CHECK(q.scalar_type() == torch::kBFloat16 && q.dim() == 3 &&
                  q.size(2) == HD,
              "q must be bf16 [B, hq, 128]");
  const int64_t B = q.size(0), hq = q.size(1), hkv = kcache.size(1);
  TORCH_CHECK(B == 0 || (q.stride(2) == 1 && (hq == 1 || q.stride(1) == HD)),
              "q heads must be contiguous");
  TORCH_CHECK((B <= 1 || q.stride(0) % 8 == 0) &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              "q rows must start on 16 bytes");
  TORCH_CHECK(out.device() == dev && out.scalar_type() == torch::kBFloat16 &&
                  out.sizes() == q.sizes() && out.is_contiguous(),
              "out must be contiguous bf16 of q's shape");
  TORCH_CHECK(hq % hkv == 0 && hq / hkv >= 1 && hq / hkv <= MAXG,
              "hq must be a multiple of hkv, up to 16 times it");
  TORCH_CHECK(kcache.size(0) > 0 && kcache.size(0) <= INT32_MAX,
              "the cache has no pages");
  TORCH_CHECK(page_table.device() == dev &&
                  page_table.scalar_type() == torch::kInt32 &&
                  page_table.dim() == 2 && page_table.size(0) == B &&
                  page_table.is_contiguous(),
              "page_table must be a contiguous int32 [B, max_pages]");
  TORCH_CHECK(page_table.size(1) <= (1 << 24), "page_table is too wide");
  TORCH_CHECK(seq_lens.device() == dev &&
                  seq_lens.scalar_type() == torch::kInt32 &&
                  seq_lens.dim() == 1 && seq_lens.size(0) == B &&
                  seq_lens.is_contiguous(),
              "seq_lens must be a contiguous int32 [B]");
  TORCH_CHECK(B <= MAXB, "too many rows");
  Paged a{};
  a.kcache = kcache.data_ptr();
  a.vcache = vcache.data_ptr();
  a.q = (const __hip_bfloat16*)q.data_ptr();
  a.page_table = (const int32_t*)page_table.data_ptr();
  a.seq_lens = (const int32_t*)seq_lens.data_ptr();
  a.q_stride = B > 1 ? q.stride(0) : 0;
  a.B = (int)B;
  a.hq = (int)hq;
  a.hkv = (int)hkv;
  a.G = (int)(hq / hkv);
  a.max_pages = (int)page_table.size(1);
  a.num_pages = (int)kcache.size(0);
  // above 0, so that a masked score stays -inf: at a scale of 0 every weight
  // comes out as 2^(1e-37 * score) = 1
  a.scale_log2 =
      std::max((float)(std::fabs(scale) * 1.4426950408889634), 1e-37f);
  a.flip = scale < 0 ? 0x80008000u : 0u;
  return a;
}

// Splits of one row's pages so that `blocks` of them make ROOM, by the table's
// width (the lengths themselves are on the device).
int splits_for(int64_t blocks, int pages) {
  const int64_t want = ROOM / std::max<int64_t>(blocks, 1);
  return (int)std::max<int64_t>(
      1, std::min<int64_t>({want, (pages + LEAST - 1) / LEAST, MAXPARTS}));
}

template <bool FP8, bool WIDE>
void launch(const Paged& a, torch::Tensor& out, hipStream_t s) {
  auto* o = (__hip_bfloat16*)out.data_ptr();
  if (a.npre > 0) {
    const int64_t blocks = (int64_t)a.hkv * (a.npre + a.B * a.nsplit);
    TORCH_CHECK(blocks < (1 << 24), "too many rows and heads");
    hipLaunchKernelGGL((paged_shared_kernel<FP8, WIDE>), dim3((unsigned)blocks),
                       dim3(NW * WAVE), 0, s, a, o);
  } else {
    hipLaunchKernelGGL((paged_decode_kernel<FP8, WIDE>), dim3(a.hkv, a.B, a.nsplit),
                       dim3(NW * WAVE), 0, s, a, o);
  }
  const dim3 joins((unsigned)(((int64_t)a.B * a.hq + 3) / 4));
  if (a.nsplit > 8)
    hipLaunchKernelGGL((paged_join_kernel<MAXPARTS>), joins, dim3(4 * WAVE), 0,
                       s, a, o);
  else if (a.npre > 0 || a.nsplit > 1)
    hipLaunchKernelGGL((paged_join_kernel<8>), joins, dim3(4 * WAVE), 0, s, a,
                       o);
}

template <bool FP8>
void launch(const Paged& a, torch::Tensor& out) {
  hipStream_t s = at::hip::getCurrentHIPStream().stream();
  if (2 * a.G > MAXG)
    launch<FP8, true>(a, out, s);
  else
    launch<FP8, false>(a, out, s);
}

// The partial results, pieces of them the prefixes': of this call alone (the
// allocator orders their reuse on the stream, and a captured graph keeps its).
torch::Tensor partials(Paged& a, const torch::Tensor& q, int64_t pieces) {
  const int64_t own =
      a.nsplit > 1 || pieces > 0 ? (int64_t)a.B * a.hq * a.nsplit : 0;
  const int64_t pre = pieces * a.hkv * TILE;
  if (own + pre == 0) return torch::Tensor();
  const int64_t at = pieces > 0 ? (int64_t)a.B * 6 : 0;  // whole 8 B
  auto work = torch::empty({(own + pre) * (HD + 2) + at},
                           q.options().dtype(torch::kFloat32));
  a.part_o = (float*)work.data_ptr();
  a.pre_o = a.part_o + own * HD;
  a.pre_at = (int4*)(a.pre_o + pre * HD);
  a.pre_has = (int32_t*)(a.pre_at + a.B);
  a.part_ml = (float*)a.pre_at + at;
  a.pre_ml = a.part_ml + own * 2;
  return work;
}

}  // namespace

void attn_decode_fp8(torch::Tensor out, torch::Tensor q, torch::Tensor kcache,
                     torch::Tensor vcache, torch::Tensor kscale,
                     torch::Tensor vscale, torch::Tensor page_table,
                     torch::Tensor seq_lens, double scale) {
  const auto dev = q.device();
  check_fp8_cache(kcache, vcache, kscale, vscale, dev);
  Paged a = paged_args(out, q, kcache, vcache, page_table, seq_lens, scale);
  if (a.B == 0) return;
  a.kscale = (const uint8_t*)kscale.data_ptr();
  a.vscale = (const uint8_t*)vscale.data_ptr();
  c10::DeviceGuard guard(dev);
  a.nsplit = splits_for((int64_t)a.B * a.hkv, a.max_pages);
  const auto work = partials(a, q, 0);
  launch<true>(a, out);
  HIP_CHECK_LAST();
}

void attn_decode_shared(torch::Tensor out, torch::Tensor q,
                        torch::Tensor kcache, torch::Tensor vcache,
                        torch::Tensor page_table, torch::Tensor seq_lens,
                        torch::Tensor group, torch::Tensor group_lens,
                        double scale, c10::optional<torch::Tensor> kscale,
                        c10::optional<torch::Tensor> vscale) {
  const auto dev = q.device();
  TORCH_CHECK(kscale.has_value() == vscale.has_value(),
              "kscale and vscale come together");
  const bool fp8 = kscale.has_value();
  if (fp8) {
    check_fp8_cache(kcache, vcache, *kscale, *vscale, dev);
  } else {
    for (const auto* c : {&kcache, &vcache}) {
      TORCH_CHECK(c->device() == dev, "the cache is on another device");
      TORCH_CHECK(c->scalar_type() == torch::kBFloat16,
                  "a cache without scales must be bf16");
      TORCH_CHECK(c->dim() == 4 && c->size(2) == KVPAGE && c->size(3) == HD &&
                      c->size(1) > 0 && c->is_contiguous() &&
                      c->sizes() == kcache.sizes(),
                  "the caches must be contiguous [P, Hkv, 64, 128]");
      TORCH_CHECK(reinterpret_cast<uintptr_t>(c->data_ptr()) % 16 == 0,
                  "the caches must start on 16 bytes");
    }
  }
  Paged a = paged_args(out, q, kcache, vcache, page_table, seq_lens, scale);
  TORCH_CHECK(group.device() == dev && group.scalar_type() == torch::kInt32 &&
                  group.dim() == 1 && group.size(0) == a.B &&
                  group.is_contiguous(),
              "group must be a contiguous int32 [B]");
  TORCH_CHECK(group_lens.device() == dev &&
                  group_lens.scalar_type() == torch::kInt32 &&
                  group_lens.dim() == 1 && group_lens.is_contiguous(),
              "group_lens must be a contiguous int32 [groups]");
  TORCH_CHECK(group_lens.size(0) <= MAXGROUPS, "at most 64 prefix groups");
  if (a.B == 0) return;
  if (fp8) {
    a.kscale = (const uint8_t*)kscale->data_ptr();
    a.vscale = (const uint8_t*)vscale->data_ptr();
  }
  a.ngroups = (int)group_lens.size(0);
  c10::DeviceGuard guard(dev);
  a.nsplit = splits_for((int64_t)a.B * a.hkv, a.max_pages);
  // each group may leave one tile part full; no more tiles than rows
  const int per_tile = TILE / a.G;
  const int64_t tiles =
      std::min<int64_t>(a.B, (a.B + per_tile - 1) / per_tile + a.ngroups);
  TORCH_CHECK(tiles * a.max_pages <= 1 << 30, "the page table is too large");
  if (a.ngroups > 0 && a.max_pages > 0) {
    a.group = (const int32_t*)group.data_ptr();
    a.group_lens = (const int32_t*)group_lens.data_ptr();
    a.npre = (int)std::max<int64_t>(
        1, std::min<int64_t>(PRE_ROOM / a.hkv,
                             tiles * ((a.max_pages + LEAST - 1) / LEAST)));
  }
  const auto work = partials(a, q, a.npre > 0 ? a.npre + tiles : 0);
  if (fp8)
    launch<true>(a, out);
  else
    launch<false>(a, out);
  HIP_CHECK_LAST();
}
