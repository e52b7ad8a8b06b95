// Token draws under temperature, top-k, top-p and min-p from one given random
// number a row (MI355X, gfx950).
//
// With the candidates (every entry but NaN and -inf) in order of falling
// logit, ties by lowest index, m the largest logit and w = exp((x - m) / T):
//   n_k = top_k                       (all candidates where it is 0 or less)
//   n_p = #{r : sum of w before r < top_p * sum of the first n_k}
//   n_m = #{r : w_r >= min_p}
//   N = max(1, min(n_k, n_p, n_m)),  Z = sum of the first N,
//   the token is the first r whose sum up to and with it passes u * Z.
// All three filters keep a prefix of that order, so that no row is sorted: a
// histogram in the order of the values gives counts and weights before every
// bin, and each question (which rank, which sum) is a search in it.
//
// A token is an integer: it has to come out the same however the sums are
// taken, and with 128256 candidates a 32-bit sum moves some border past u in
// about every hundredth row.  Weights and sums are held in 64 bits.
//
// bf16 logits have few distinct values: bins are the values themselves, the
// counts are exact, and a row takes one exponential for each DISTINCT value
// (about 1500) instead of one for each of 128256 entries.  fp32 logits take
// linear bins of (m - x), with weights summed as 64-bit fixed point (integer
// sums do not depend on the order of the atomics) in steps of 2^-51 of the
// largest weight up to 4096 entries, 2^-48 at 32000, 2^-46 at 128256 and 2^-43
// at 2^20, each weight rounded to half a step; the bin that holds a border is
// resolved by ranking its members, whose weights are floating 64-bit ones.
//
// Rows that fit neither take a bisection over the keys, general and slow: 69
// passes over the row in memory with an exponential an entry, 137 under a top-p,
// 2.8 and 5.6 ms for 128256 bf16 entries, 1.9 and 3.4 ms for as many equal fp32
// ones, 0.3 and 0.5 ms for 12000.  They are, bf16: a magnitude of 2^23 or more
// (or below 2^-41, but 0) among values that count, over 4096 distinct values;
// fp32: an infinity, a range beyond the type's, over 2048 entries in the bin of a
// border (equal logits; 128256 random ones take 80 to 110 us by bins).
//
// One block of 1024 threads is one row; it reads the row once and holds it in
// registers (128256 bf16 are 64 registers a thread).  Bound: the histogram, one
// LDS add an entry: 13 to 18 cycles an instruction of 64 lanes (LDS itself is
// busy for 8, half of them bank conflicts), up to 37000 of the 62000 cycles of a
// bf16 row of 128256; then the row's bytes.  Measured: one bf16 row of 128256 24
// to 28 us whatever its filters (the later its rank, the longer), 11 us at
// temperature 0; 512 of them 68 us (1.9 TB/s; a CU takes two, one after the
// other, the histograms 31 us of it), 64 fp32 rows of 32000 45 us (64-bit
// exponentials and two histograms); rows that are not drawn 2.3 us for 1 and 2.4
// for 512, as any launch.  Sorting the 512 rows with library calls takes 11.7 ms.

#include "common.h"

namespace {

using u32x4 = __attribute__((ext_vector_type(4))) unsigned;

constexpr int BLOCK = 1024;
constexpr int NWAVES = BLOCK / WAVE;
constexpr int MAXCHUNKS = 257;  // of 4096 fp32 entries: up to 2^20
constexpr int MAXV = 1 << 20;

// bf16: magnitudes [2^-41, 2^23) are 64 octaves of 128 values, each sign
constexpr int BINS16 = 16384;
constexpr int LO16 = 86 << 7, HI16 = 150 << 7;
constexpr float FAR_VALUE = -8388608.f;  // -2^23
constexpr int DISTINCT = 4096;
constexpr int LISTED = BLOCK;  // equal values ranked one a thread
// fp32
constexpr int BINS32 = 8192;
constexpr int MEMBERS = 2048;

// 2^(j / 64), rounded to 64 bits.
__constant__ const double POW2_64TH[64] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0,
};

struct Args {
  int32_t* out;
  int32_t* kept;  // or null
  const void* logits;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int V;
  // steps of 1 in the fixed point of fp32 rows: the finest whose V weights sum
  // to 2^63 or less, 2^51 at most (a weight fits a double's 52 bits)
  double steps, step;  // and 1 / steps
};

// What every path is asked: the row's filters.
struct Row {
  float m;        // largest logit
  double inv_T;  // of a temperature > 0
  int k;          // top_k or V
  const double* pow2;  // POW2_64TH in LDS
};

// The token: an index, or (token < 0) the nth of the `ties` entries of value x.
struct Answer {
  int token, kept, nth, ties;
  float x;
};

// Ascending with the value; NaN and -0 are dealt with before.
__device__ __forceinline__ unsigned key_of(const float x) {
  const unsigned u = __float_as_uint(x);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(const unsigned key) {
  return __uint_as_float((key >> 31) ? (key & 0x7fffffffu) : ~key);
}

__device__ __forceinline__ bool candidate(const float x) {
  return x > -INFINITY;  // false for NaN
}

// exp(z) for z <= 0, to a few units of the last bit: z = n ln2 / 64 + y with
// |y| <= ln2 / 128, exp(y) by its series up to y^5 (the next term is below
// 2^-54), 2^(n / 64) from the table (in LDS).  A dozen operations and seven
// constants; the general exp() keeps twice as many registers busy.
__device__ __forceinline__ double exp_neg(double z, const double* pow2) {
  z = fmax(z, -800.0);
  const double n = rint(z * 0x1.71547652b82fep+6);
  double y = fma(n, -0x1.62e42fc000000p-7, z);
  y = fma(n, -0x1.7d1cf79abc9e4p-34, y);
  double p = fma(y, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(y, p, 1.0 / 6.0);
  p = fma(y, p, 0.5);
  p = fma(y, p, 1.0);
  p = fma(y, p, 1.0);
  const int i = (int)n;
  return ldexp(p * pow2[i & 63], i >> 6);
}

__device__ __forceinline__ double weight(const float x, const Row& r) {
  return x == r.m ? 1.0
                  : exp_neg(((double)x - (double)r.m) * r.inv_T, r.pow2);
}

// ---- wave- and block-wide sums and scans over DPP lane moves (a few cycles a
// step where a swap through LDS takes a hundred); `lds` holds NWAVES values

template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned moved(const unsigned x) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf,
                                               false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long moved(
    const unsigned long long x) {
  return ((unsigned long long)moved<CTRL, ROWS>((unsigned)(x >> 32)) << 32) |
         moved<CTRL, ROWS>((unsigned)x);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double moved(const double x) {
  return __longlong_as_double((long long)moved<CTRL, ROWS>(
      (unsigned long long)__double_as_longlong(x)));
}
__device__ __forceinline__ unsigned lane_of(const unsigned x, const int l) {
  return (unsigned)__builtin_amdgcn_readlane((int)x, l);
}
__device__ __forceinline__ unsigned long long lane_of(
    const unsigned long long x, const int l) {
  return ((unsigned long long)lane_of((unsigned)(x >> 32), l) << 32) |
         lane_of((unsigned)x, l);
}
__device__ __forceinline__ double lane_of(const double x, const int l) {
  return __longlong_as_double((long long)lane_of(
      (unsigned long long)__double_as_longlong(x), l));
}

// Sums up to and with each lane, within rows of 16 lanes or the whole wave.
template <typename S>
__device__ __forceinline__ S row_scan(S x) {
  x += moved<0x111, 0xf>(x);  // from 1, 2, 4, 8 lanes below
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  return x;
}
template <typename S>
__device__ __forceinline__ S wave_scan(S x) {
  x = row_scan(x);
  x += moved<0x142, 0xa>(x);  // lane 15 of each row to the next
  x += moved<0x143, 0xc>(x);  // lane 31 to the upper half
  return x;
}

template <typename S>
__device__ __forceinline__ S block_scan(const S x, S* lds, S* total) {
  const int lane = threadIdx.x % WAVE;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const S incl = wave_scan(x);
  __syncthreads();  // the last user of lds is done
  if (lane == WAVE - 1) lds[wid] = incl;
  __syncthreads();
  const S waves = row_scan(lds[lane % NWAVES]);
  *total = lane_of(waves, NWAVES - 1);
  const S before = wid > 0 ? lane_of(waves, max(wid - 1, 0)) : (S)0;
  // and the lane below's sum (not incl - x: no rounding where S is a double)
  return before + moved<0x138, 0xf>(incl);
}

template <typename S>
__device__ __forceinline__ S block_total(const S x, S* lds) {
  const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
  const S incl = wave_scan(x);
  __syncthreads();
  if (lane == WAVE - 1) lds[wid] = incl;
  __syncthreads();
  return lane_of(row_scan(lds[lane % NWAVES]), NWAVES - 1);
}

__device__ __forceinline__ float block_largest(float x, float* lds) {
  const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
  x = wave_max(x);
  __syncthreads();
  if (lane == 0) lds[wid] = x;
  __syncthreads();
  x = lds[lane % NWAVES];
#pragma unroll
  for (int off = NWAVES / 2; off > 0; off >>= 1)
    x = fmaxf(x, __shfl_xor(x, off, WAVE));
  return x;
}

// One entry a thread at a time, read again in every pass.
template <typename T>
struct Plain {
  const T* row;
  int V;
  __device__ __forceinline__ float at(const int i) const {
    if constexpr (sizeof(T) == 4)
      return row[i] + 0.f;
    else
      return bf2f(row[i]) + 0.f;
  }
};

// A row in chunks of BLOCK x 16 B: chunk c of thread t is the PER entries from
// (c * BLOCK + t) * PER - lead on, so that every load is aligned whatever the
// row's start; the first NC chunks stay in registers.  Entries outside the
// row read as NaN, which is no candidate.
template <typename T, int NC>
struct Entries {
  static constexpr int PER = 16 / sizeof(T);
  const T* row;
  int V, lead, chunks;
  u32x4 held[NC];

  __device__ __forceinline__ int first_of(const int c) const {
    return (c * BLOCK + (int)threadIdx.x) * PER - lead;
  }
  __device__ __forceinline__ u32x4 load(const int c) const {
    const int i = first_of(c);
    if (i >= 0 && i + PER <= V)
      return *reinterpret_cast<const u32x4*>(row + i);
    u32x4 v = {~0u, ~0u, ~0u, ~0u};  // NaN in either type
    if constexpr (sizeof(T) == 4) {
      const unsigned* src = reinterpret_cast<const unsigned*>(row);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j >= 0 && i + j < V) v[j] = src[i + j];
    } else {
      const unsigned short* src = reinterpret_cast<const unsigned short*>(row);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j >= 0 && i + j < V)
          v[j / 2] = (j & 1)
                         ? (v[j / 2] & 0xffffu) | ((unsigned)src[i + j] << 16)
                         : (v[j / 2] & 0xffff0000u) | src[i + j];
    }
    return v;
  }
  __device__ __forceinline__ void open(const T* r, const int v) {
    row = r;
    V = v;
    lead = (int)((reinterpret_cast<uintptr_t>(r) % 16) / sizeof(T));
    chunks = (V + lead + BLOCK * PER - 1) / (BLOCK * PER);
#pragma unroll
    for (int c = 0; c < NC; ++c)
      held[c] = c < chunks ? load(c) : (u32x4){~0u, ~0u, ~0u, ~0u};
  }
  // f(chunk, its 16 bytes)
  template <typename F>
  __device__ __forceinline__ void each_chunk(F f) const {
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (c < chunks) f(c, held[c]);
#pragma unroll 1
    for (int c = NC; c < chunks; ++c) f(c, load(c));
  }
  static __device__ __forceinline__ float get(const u32x4 v, const int j) {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(v[j]);
    else
      return __uint_as_float((j & 1) ? (v[j / 2] & 0xffff0000u)
                                     : (v[j / 2] << 16));
  }
  // whether an entry is x
  static __device__ __forceinline__ bool has(const u32x4 v, const float x) {
    if constexpr (sizeof(T) == 4) {
      return get(v, 0) == x || get(v, 1) == x || get(v, 2) == x ||
             get(v, 3) == x;
    } else {
      using u16x2 = __attribute__((ext_vector_type(2))) unsigned short;
      const unsigned code = __float_as_uint(x) >> 16;
      const unsigned keep = code ? ~0u : 0x7fff7fffu;  // both zeros
      u16x2 least = {0xffff, 0xffff};
#pragma unroll
      for (int q = 0; q < 4; ++q)
        least = __builtin_elementwise_min(
            least, __builtin_bit_cast(
                       u16x2, (v[q] ^ (code | code << 16)) & keep));
      return least[0] == 0 || least[1] == 0;
    }
  }
  // each_chunk with TURN instances of f's code: the held chunks pass through
  // the first TURN places and end where they were (a move a register and turn).
  template <int TURN, typename F>
  __device__ __forceinline__ void each_chunk_in_turn(F f) {
    static_assert(NC % TURN == 0, "whole turns");
#pragma unroll 1
    for (int c = 0; c < NC; c += TURN) {
      u32x4 now[TURN];
#pragma unroll
      for (int k = 0; k < TURN; ++k) now[k] = held[k];
#pragma unroll
      for (int k = 0; k + TURN < NC; ++k) held[k] = held[k + TURN];
#pragma unroll
      for (int k = 0; k < TURN; ++k) held[NC - TURN + k] = now[k];
#pragma unroll
      for (int k = 0; k < TURN; ++k) f(c + k, now[k]);
    }
#pragma unroll 1
    for (int c = NC; c < chunks; ++c) f(c, load(c));
  }
  // f(index, value) of every candidate, -0 as +0, one after the other
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    static_assert(PER == 4, "one word an entry");
    each_chunk_in_turn<1>([&](const int c, u32x4 v) {
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float x = get(v, j) + 0.f;
        if (candidate(x)) f(first_of(c) + j, x);
      }
    });
  }
};

struct Shared {
  double pow2[64];
  double T, top_p, min_p, u;  // in LDS: read where they are asked for
  double red_d[NWAVES];
  unsigned long long red_u[NWAVES];
  unsigned red_n[NWAVES];
  float red_f[NWAVES];
  int flag, hit, at;
  unsigned members;
  double hit_before, hit_w;
  int per_chunk[MAXCHUNKS];
};

// The j-th of the n entries, in order of index, whose value is x.  A few are
// listed as they are met and ranked; of many, the chunks are counted first.
template <typename E>
__device__ __forceinline__ int nth_of_value(const E& e, const float x,
                                            const int j, const int n,
                                            int* list, Shared& s) {
  if (threadIdx.x == 0) s.members = 0;
  for (int i = threadIdx.x; i < e.chunks; i += BLOCK) s.per_chunk[i] = 0;
  __syncthreads();
  if (n <= LISTED) {
    e.each_chunk([&](const int c, const u32x4 v) {
      if (!e.has(v, x)) return;
#pragma unroll
      for (int q = 0; q < E::PER; ++q)
        if (E::get(v, q) == x)
          list[atomicAdd(&s.members, 1u)] = e.first_of(c) + q;
    });
    __syncthreads();
    if (threadIdx.x < (unsigned)n) {
      const int mine = list[threadIdx.x];
      int rank = 0;
      for (int q = 0; q < n; ++q) rank += list[q] < mine;
      if (rank == j) s.at = mine;
    }
    __syncthreads();
    return s.at;
  }
  e.each_chunk([&](const int c, const u32x4 v) {
    int here = 0;
#pragma unroll
    for (int q = 0; q < E::PER; ++q) here += E::get(v, q) == x;
    if (here) atomicAdd(&s.per_chunk[c], here);
  });
  __syncthreads();
  int chunk = 0, left = j;
  while (chunk < e.chunks - 1 && left >= s.per_chunk[chunk])
    left -= s.per_chunk[chunk++];
  const u32x4 v = e.load(chunk);
  unsigned here = 0, all;
#pragma unroll
  for (int q = 0; q < E::PER; ++q) here += E::get(v, q) == x;
  int before = (int)block_scan<unsigned>(here, s.red_n, &all);
  if (left >= before && left < before + (int)here) {
#pragma unroll
    for (int q = 0; q < E::PER; ++q)
      if (E::get(v, q) == x && before++ == left) s.at = e.first_of(chunk) + q;
  }
  __syncthreads();
  return s.at;
}

// How many of n equal weights w, the first after `before`, come before the
// sum reaches `goal`: #{j : before + j w < goal} (or <=, with `upto`).
__device__ __forceinline__ int within(const double goal, const double before,
                                      const double w, const int n,
                                      const bool upto) {
  if (n <= 0 || w <= 0.0) return n;
  const double j = (goal - before) / w;
  const double c = upto ? floor(j) : ceil(j);
  return c <= 0.0 ? 0 : c >= (double)n ? n : (int)c;
}

// ------------------------------------------------- the general, slow search

// Count and weight of the candidates with a key above (or from) t, and the
// count of those that weigh min_p or more.
template <typename T>
__device__ __forceinline__ void above(const Plain<T>& e, const Row& r,
                                      const unsigned t, const bool from,
                                      long long& n, double& w, long long& nm,
                                      Shared& s) {
  unsigned long long cnt = 0, cm = 0;
  double sum = 0.0;
#pragma unroll 1
  for (int i = threadIdx.x; i < e.V; i += BLOCK) {
    const float x = e.at(i);
    const unsigned key = key_of(x);
    if (candidate(x) && (key > t || (from && key == t))) {
      const double wi = weight(x, r);
      ++cnt;
      cm += wi >= s.min_p;
      sum += wi;
    }
  }
  n = (long long)block_total<unsigned long long>(cnt, s.red_u);
  nm = (long long)block_total<unsigned long long>(cm, s.red_u);
  w = block_total<double>(sum, s.red_d);
}

// The four questions of a row, each by bisection for the largest key t with
// count(key >= t) >= rank, weight(key >= t) >= goal, or > goal.  All passes
// are one instance of the loop over the row: it keeps few registers.
template <typename T>
__device__ __forceinline__ Answer general(const Plain<T>& e, const Row& r,
                                          Shared& s) {
  long long all = 0, nm = 0, N = 0;
  double Z = 0.0;
  unsigned t = 0;
  int nth = 0;
  bool by_count = true;
#pragma unroll 1
  for (int step = -1; step < 4;) {
    if (step == 2) N = max(1ll, min(N, nm));
    if (step >= 0 && step < 2 && !(s.top_p < 1.0)) {
      ++step;
      continue;
    }
    const double goal = step == 1 ? s.top_p * Z : s.u * Z;
    if (step == 1 && !(goal > 0.0)) {
      N = 0;
      ++step;
      by_count = true;
      continue;
    }
    long long cnt = 0;
    double before = 0.0;
    int ties = 0;
    t = 0;
    // passes 0..31 bisect, 32 takes what lies above t, 33 that and t itself
#pragma unroll 1
    for (int pass = step < 0 ? 33 : 0; pass < 34; ++pass) {
      const unsigned key = pass < 32 ? t | (1u << (31 - pass)) : t;
      long long n, m;
      double w;
      above(e, r, key, pass != 32, n, w, m, s);
      if (pass < 32) {
        if (by_count ? n >= N : step == 1 ? w >= goal : w > goal) t = key;
      } else if (pass == 32) {
        cnt = n;
        before = w;
      } else {
        ties = (int)(n - cnt);
        all = n;
        if (step < 0) nm = m;
      }
    }
    const double wt = weight(value_of(t), r);
    if (step < 0) {
      N = min((long long)r.k, all);
    } else if (step == 3 && !by_count && cnt >= N) {
      // rounding keeps every sum short of the draw: the last rank kept
      by_count = true;
      continue;
    } else if ((step & 1) == 0) {
      Z = before + (double)(N - cnt) * wt;
    } else if (step == 1) {
      N = min(N, cnt + within(goal, before, wt, ties, false));
    } else {
      nth = (int)min((long long)within(goal, before, wt, ties - 1, true),
                     N - 1 - cnt);
    }
    ++step;
    by_count = (step & 1) == 0;
  }
  // the nth entry, in order of index, whose key is t
  int left = nth, token = 0;
#pragma unroll 1
  for (int i0 = 0; i0 < e.V && left >= 0; i0 += BLOCK) {
    const int i = i0 + threadIdx.x;
    const bool is = i < e.V && candidate(e.at(i)) && key_of(e.at(i)) == t;
    unsigned long long here;
    const int rank = (int)block_scan<unsigned long long>(is, s.red_u, &here);
    if (is && rank == left) s.at = i;
    __syncthreads();
    if (left < (int)here) token = s.at;
    left -= (int)here;
  }
  return {token, (int)N, 0, 0, 0.f};
}

// --------------------------------------------------- bf16: bins are values

struct Lds16 {
  union {
    unsigned counts[BINS16];
    struct {  // once the list is made
      double w[DISTINCT];
      int ties[LISTED];
    };
  };
  double before_w[DISTINCT + 1];
  int before_n[DISTINCT + 1];
  unsigned short code[DISTINCT];
  unsigned places[BINS16 / WAVE];  // what each 64 places hold
  uint2 before[BINS16 / WAVE];     // and what lies before them
  Shared s;
  unsigned zeros, far;
};

// Counts the row's values into their bins as its loads arrive: bin =
// magnitude - LO16, the negative ones 8192 further; as a byte address it is
// (offset * 4) | sign, in both halves of a word at once.  Words with a value
// outside the bins are left for a second, rolled loop: written out for every
// word they would not fit the instruction cache.
template <int NC>
__device__ __forceinline__ void count_values(
    const Entries<__hip_bfloat16, NC>& e, Lds16& L) {
  using u16x2 = __attribute__((ext_vector_type(2))) unsigned short;
  const auto offsets = [](const unsigned w) __attribute__((always_inline)) {
    return __builtin_bit_cast(u16x2, w & 0x7fff7fffu) -
           (u16x2){(unsigned short)LO16, (unsigned short)LO16};
  };
  const auto outside = [](const u16x2 off) __attribute__((always_inline)) {
    return (__builtin_bit_cast(unsigned, off) & 0xe000e000u) != 0;
  };
  unsigned odd = 0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const unsigned w = e.held[c][q];
      const u16x2 off = offsets(w);
      if (outside(off)) {
        odd |= 1u << c;
      } else {
        const unsigned at =
            __builtin_bit_cast(unsigned, (u16x2)(off << (u16x2){2, 2})) |
            (w & 0x80008000u);
        char* base = reinterpret_cast<char*>(L.counts);
        atomicAdd(reinterpret_cast<unsigned*>(base + (at & 0xffffu)), 1u);
        atomicAdd(reinterpret_cast<unsigned*>(base + (at >> 16)), 1u);
      }
    }
  }
#pragma unroll 1
  for (int c = 0; c < e.chunks; ++c) {
    const bool all = c >= NC;
    if (!all && !((odd >> c) & 1)) continue;
    const u32x4 v = e.load(c);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (!all && !outside(offsets(v[q]))) continue;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const unsigned u = (v[q] >> (16 * hf)) & 0xffffu;
        const unsigned a = u & 0x7fffu;
        if (a >= (unsigned)LO16 && a < (unsigned)HI16)
          atomicAdd(&L.counts[(a - LO16) + ((u >> 15) << 13)], 1u);
        else if (a == 0)
          atomicAdd(&L.zeros, 1u);
        else if (a < (unsigned)LO16)
          L.s.flag = 1;  // magnitudes below 2^-41
        else if (u > 0x8000u && a < 0x7f80u)
          atomicAdd(&L.far, 1u);  // finite, -2^23 or less
      }
    }
  }
}

// The list's last entry i for which ok(i), which holds for a prefix of it (0
// if for none).  Two rounds of 64 probes, the same in every wave.
template <typename F>
__device__ __forceinline__ int last_entry(const int entries, F ok) {
  static_assert(DISTINCT <= 64 * 64, "two rounds");
  const int lane = threadIdx.x % WAVE;
  const int step = (entries + 63) / 64;
  int i = lane * step;
  unsigned long long yes = __ballot(i < entries && ok(i));
  if (yes == 0) return 0;
  const int base = (63 - __clzll((long long)yes)) * step;
  i = base + lane;
  yes = __ballot(lane < step && i < entries && ok(i));
  return base + 63 - __clzll((long long)yes);
}

// Both row functions say false where the general search has to take the row.
template <int NC>
__device__ __forceinline__ bool bf16_row(const Entries<__hip_bfloat16, NC>& e,
                                        const Row& r, Lds16& L, Answer& ans) {
  Shared& s = L.s;
  const int tid = threadIdx.x;
  const int lane = tid % WAVE, wid = tid / WAVE;
  // far values have to weigh nothing: exp(-746) is 0 in 64 bits
  if (s.flag || r.m >= -FAR_VALUE ||
      (L.far && (double)r.m - (double)FAR_VALUE < 746.0 * s.T))
    return false;

  // ---- the list of distinct values, falling.  Place p is the positive
  // values from the largest down, then (from BINS16 / 2, after the zeros) the
  // negative ones.  A wave takes 64 places at a time, so that the few hundred
  // neighbours that hold nearly all values are shared among the waves.
  constexpr int ROUNDS = BINS16 / BLOCK;
  const auto bin_at = [](const int p) __attribute__((always_inline)) {
    return p < BINS16 / 2 ? BINS16 / 2 - 1 - p : p;
  };
  // how many values (up to 2^20) and, from bit 21 on, how many distinct
  constexpr unsigned ONE = 1u << 21;
  unsigned c[ROUNDS], incl[ROUNDS];
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) c[k] = L.counts[bin_at(k * BLOCK + tid)];
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    incl[k] = c[k] ? c[k] + ONE : 0u;
    if (__any(c[k] != 0)) incl[k] = wave_scan(incl[k]);
    if (lane == WAVE - 1) L.places[k * NWAVES + wid] = incl[k];
  }
  __syncthreads();
  // what lies before each group of 64 places: 4 groups a lane, the same in
  // every wave
  constexpr int GROUPS = BINS16 / WAVE / WAVE;
  static_assert(GROUPS == 4, "one 16 B read a lane");
  const u32x4 g = reinterpret_cast<const u32x4*>(L.places)[lane];
  unsigned gn = 0, gd = 0;
#pragma unroll
  for (int q = 0; q < GROUPS; ++q) {
    gn += g[q] & (ONE - 1);
    gd += g[q] >> 21;
  }
  const unsigned zeros = L.zeros;
  const unsigned un = wave_scan(gn), ud = wave_scan(gd);
  const int entries = (int)lane_of(ud, WAVE - 1) + (zeros != 0);
  const int listed = (int)(lane_of(un, WAVE - 1) + zeros);
  if (entries > DISTINCT) return false;
  if (wid == 0) {
    unsigned n = un - gn, d = ud - gd;
    if (lane >= 32) {  // the negative places follow the zeros
      n += zeros;
      d += zeros != 0;
    }
#pragma unroll
    for (int q = 0; q < GROUPS; ++q) {
      L.before[lane * GROUPS + q] = make_uint2(n, d);
      n += g[q] & (ONE - 1);
      d += g[q] >> 21;
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ROUNDS; ++k) {
    if (c[k]) {
      const uint2 base = L.before[k * NWAVES + wid];
      const int p = k * BLOCK + tid;
      const unsigned at = base.y + (incl[k] >> 21) - 1;
      L.before_n[at] = (int)(base.x + (incl[k] & (ONE - 1)) - c[k]);
      L.code[at] = (unsigned short)(p < BINS16 / 2
                                        ? LO16 + BINS16 / 2 - 1 - p
                                        : 0x8000 | (LO16 + p - BINS16 / 2));
    }
  }
  if (zeros && tid == 0) {  // after lane 31's groups, the positive ones
    const int at = (int)lane_of(ud, 31);
    L.code[at] = 0;
    L.before_n[at] = (int)lane_of(un, 31);
  }
  if (tid == 0) L.before_n[entries] = listed;
  __syncthreads();  // counts are done with: w takes their place

  double mine[DISTINCT / BLOCK], sum = 0.0;
#pragma unroll
  for (int j = 0; j < DISTINCT / BLOCK; ++j) mine[j] = 0.0;
  const int per = (entries + BLOCK - 1) / BLOCK;
#pragma unroll
  for (int j = 0; j < DISTINCT / BLOCK; ++j) {
    const int i = tid * per + j;
    if (j < per && i < entries) {
      const double w =
          weight(__uint_as_float((unsigned)L.code[i] << 16) + 0.f, r);
      L.w[i] = w;
      mine[j] = w * (double)(L.before_n[i + 1] - L.before_n[i]);
      sum += mine[j];
    }
  }
  double w_all;
  double upto = block_scan<double>(sum, s.red_d, &w_all);
#pragma unroll
  for (int j = 0; j < DISTINCT / BLOCK; ++j) {
    const int i = tid * per + j;
    if (j < per && i < entries) {
      L.before_w[i] = upto;
      upto += mine[j];
    }
  }
  if (tid == 0) L.before_w[entries] = w_all;
  __syncthreads();

  const auto sum_first = [&](const int n) __attribute__((always_inline)) {
    if (n >= listed) return w_all;
    const int i =
        last_entry(entries, [&](int i) { return L.before_n[i] < n; });
    return L.before_w[i] + (double)(n - L.before_n[i]) * L.w[i];
  };
  const int all = listed + (int)L.far;
  int N = min(r.k, all);
  double Z = sum_first(N);
  if (s.top_p < 1.0) {
    const double goal = s.top_p * Z;
    int np = 0;
    if (goal > 0.0) {
      const int i =
          last_entry(entries, [&](int i) { return L.before_w[i] < goal; });
      np = L.before_n[i] + within(goal, L.before_w[i], L.w[i],
                                  L.before_n[i + 1] - L.before_n[i], false);
    }
    N = min(N, np);
  }
  if (!(s.min_p <= 0.0)) {
    const int i =
        last_entry(entries, [&](int i) { return L.w[i] >= s.min_p; });
    N = min(N, L.w[i] >= s.min_p ? L.before_n[i + 1] : 0);
  }
  N = max(N, 1);
  const double goal = s.u * sum_first(N);
  const int i =
      last_entry(entries, [&](int i) { return L.before_w[i] <= goal; });
  int j = within(goal, L.before_w[i], L.w[i],
                 L.before_n[i + 1] - L.before_n[i] - 1, true);
  j = max(0, min(j, N - 1 - L.before_n[i]));
  const float x = __uint_as_float((unsigned)L.code[i] << 16) + 0.f;
  ans = {-1, N, j, L.before_n[i + 1] - L.before_n[i], x};
  return true;
}

// ----------------------------------------------------- fp32: linear bins

struct Lds32 {
  unsigned long long w[BINS32];
  unsigned n[BINS32];
  unsigned key[MEMBERS];
  int index[MEMBERS];
  unsigned sorted_key[MEMBERS];
  int sorted_index[MEMBERS];
  Shared s;
};

template <int NC>
__device__ __forceinline__ bool fp32_row(Entries<float, NC>& e, const Row& r,
                                        const Args& a, Lds32& L, Answer& ans) {
  constexpr int PT = BINS32 / BLOCK;  // bins of a thread, in order
  Shared& s = L.s;
  const int tid = threadIdx.x;
  if (r.m == INFINITY) return false;
  // values that weigh nothing (exp(-746) is 0 in 64 bits) are counted alone;
  // the bins cover the others
  const float cut = __double2float_rd((double)r.m - 746.0 * s.T);
  float low = r.m;
  e.each_chunk([&](int, const u32x4 v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = e.get(v, j);
      low = x >= cut && candidate(x) ? fminf(low, x) : low;
    }
  });
  low = -block_largest(-low, s.red_f);
  const float span = r.m - low;
  if (!(span < INFINITY)) return false;
  const float by = span > 0.f ? (float)BINS32 / span : 0.f;
  if (!(by < INFINITY)) return false;
  // monotone in x: a subtraction and a product, each rounded
  const auto bin_of = [&](const float x) __attribute__((always_inline)) {
    return min(BINS32 - 1, (int)((r.m - x) * by));
  };
  unsigned long long nm = 0, far = 0;
  e.each([&](int, const float x) {
    if (x < low) {
      ++far;
      nm += 0.0 >= s.min_p;
      return;
    }
    const double w = weight(x, r);
    const int b = bin_of(x);
    // the sum with 2^52 has the rounded integer for its mantissa
    atomicAdd(&L.w[b], (unsigned long long)__double_as_longlong(
                           fma(w, a.steps, 0x1p52)) &
                           ((1ull << 52) - 1));
    atomicAdd(&L.n[b], 1u);
    nm += w >= s.min_p;
  });
  far = block_total<unsigned long long>(far, s.red_u);
  nm = block_total<unsigned long long>(nm, s.red_u);
  __syncthreads();

  unsigned long long tw = 0, tn = 0, w_fix, listed;
  unsigned long long binw[PT];
  unsigned binn[PT];
#pragma unroll
  for (int j = 0; j < PT; ++j) {
    binw[j] = L.w[tid * PT + j];
    binn[j] = L.n[tid * PT + j];
    tw += binw[j];
    tn += binn[j];
  }
  const unsigned long long bw = block_scan<unsigned long long>(tw, s.red_u,
                                                               &w_fix);
  const unsigned long long bn = block_scan<unsigned long long>(tn, s.red_u,
                                                               &listed);
  const double w_all = (double)w_fix * a.step;

  // ---- four questions, each to one bin: the sum of the first n_k, the rank
  // of the top-p border, the sum of the first N, the rank of the draw
  const long long all = (long long)(listed + far);
  long long N = min((long long)r.k, all);
  double Z = w_all;
  int bin = -1, members = 0, before_n = 0, token = 0;
  double before_w = 0.0;
#pragma unroll 1
  for (int step = 0; step < 4; ++step) {
    if (step == 2) N = max(1ll, min(N, (long long)nm));
    if (step < 2 && !(s.top_p < 1.0)) continue;
    bool by_count = (step & 1) == 0;
    if (by_count && N >= (long long)listed) {
      Z = w_all;
      continue;
    }
    const double goal = step == 1 ? s.top_p * Z : s.u * Z;
    if (step == 1 && !(goal > 0.0)) {
      N = 0;
      continue;
    }
    bool found = false;
    const long long rank = min(N, (long long)listed);
#pragma unroll 1
    for (int again = 0; again < 2; ++again) {
      __syncthreads();
      if (tid == 0) s.hit = -1;
      __syncthreads();
      unsigned long long cw = bw, cn = bn;
#pragma unroll
      for (int j = 0; j < PT; ++j) {
        const unsigned n = binn[j];
        const unsigned long long ew = cw + binw[j], en = cn + n;
        const double d0 = (double)cw * a.step;
        const double d1 = (double)ew * a.step;
        if (n != 0 &&
            (by_count    ? ((long long)cn < rank && (long long)en >= rank)
             : step == 1 ? (d0 < goal && d1 >= goal)
                         : (d0 <= goal && d1 > goal))) {
          s.hit = tid * PT + j;
          s.at = (int)cn;
          s.hit_before = d0;
        }
        cw = ew;
        cn = en;
      }
      __syncthreads();
      found = s.hit >= 0;
      // the draw's two sums agree to the last bits only: the last rank kept
      // at most
      if (step != 3 || by_count || (found && s.at < N)) break;
      by_count = true;
    }
    if (!found) {  // (step 1: rounding keeps the whole sum short of the goal)
      N = min(N, (long long)listed);
      continue;
    }
    if (s.hit != bin) {
      bin = s.hit;
      before_n = s.at;
      before_w = s.hit_before;
      members = (int)L.n[bin];
      if (members > MEMBERS) return false;
      if (tid == 0) s.members = 0;
      __syncthreads();
      e.template each_chunk_in_turn<2>([&](const int c, const u32x4 v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = e.get(v, j) + 0.f;
          if (x >= low && bin_of(x) == bin) {
            const unsigned p = atomicAdd(&s.members, 1u);
            L.key[p] = key_of(x);
            L.index[p] = e.first_of(c) + j;
          }
        }
      });
      __syncthreads();
      for (int p = tid; p < members; p += BLOCK) {
        const unsigned key = L.key[p];
        const int i = L.index[p];
        int rank_in = 0;
#pragma unroll 4
        for (int q = 0; q < members; ++q) {
          const unsigned k2 = L.key[q];
          rank_in += k2 > key || (k2 == key && L.index[q] < i);
        }
        L.sorted_key[rank_in] = key;
        L.sorted_index[rank_in] = i;
      }
      __syncthreads();
    }
    // the bin's ranks that come before the goal, and their sum up to rank N
    const int upto =
        (step & 1) ? members : (int)min((long long)members, N - before_n);
    double mine[MEMBERS / BLOCK], t = 0.0, sum;
    const int per = (members + BLOCK - 1) / BLOCK;
#pragma unroll
    for (int j = 0; j < MEMBERS / BLOCK; ++j) {
      const int p = tid * per + j;
      mine[j] = (j < per && p < upto) ? weight(value_of(L.sorted_key[p]), r)
                                      : 0.0;
      t += mine[j];
    }
    double b = before_w + block_scan<double>(t, s.red_d, &sum);
    unsigned long long n = 0;
#pragma unroll
    for (int j = 0; j < MEMBERS / BLOCK; ++j) {
      if (j < per && tid * per + j < upto)
        n += step == 1 ? b < goal : b + mine[j] <= goal;
      b += mine[j];
    }
    n = block_total<unsigned long long>(n, s.red_u);
    if ((step & 1) == 0) Z = before_w + sum;
    if (step == 1) N = min(N, before_n + (long long)n);
    if (step == 3)
      token = L.sorted_index[(int)min((long long)min((int)n, members - 1),
                                      N - 1 - before_n)];
  }
  ans = {token, (int)N, 0, 0, 0.f};
  return true;
}

// A value that is the same in all lanes, kept in scalar registers.
__device__ __forceinline__ double uniform_of(const double x) {
  const long long u = __double_as_longlong(x);
  const int lo = __builtin_amdgcn_readfirstlane((int)(u & 0xffffffffll));
  const int hi = __builtin_amdgcn_readfirstlane((int)(u >> 32));
  return __longlong_as_double(((long long)hi << 32) | (unsigned)lo);
}

// What is the row's filters' apart from its logits; false: not asked for.
__device__ __forceinline__ bool open_row(const Args& a, const int b, Row& r,
                                         Shared& s) {
  // all at once: one latency, not one behind the other
  const float u = a.uniform[b], t = a.temperature[b], p = a.top_p[b],
              q = a.min_p[b];
  const int k = a.top_k[b];
  if (u < 0.f) return false;
  const double T = uniform_of((double)t);
  r.inv_T = uniform_of(1.0 / T);
  r.k = (k > 0 && k < a.V) ? k : a.V;
  if (threadIdx.x == 0) {  // seen after the first block-wide step
    s.T = T;
    s.top_p = (double)p;
    s.min_p = (double)q;
    s.u = fmin((double)u, 1.0 - 0x1p-53);  // [0, 1); NaN too
  }
  r.pow2 = s.pow2;
  if (threadIdx.x < 64) s.pow2[threadIdx.x] = POW2_64TH[threadIdx.x];
  return true;
}

__device__ __forceinline__ void answer(const Args& a, const int b,
                                       const int token, const int kept) {
  if (threadIdx.x == 0) {
    a.out[b] = token;
    if (a.kept) a.kept[b] = kept;
  }
}

template <typename T>
struct LdsOf;
template <>
struct LdsOf<__hip_bfloat16> {
  using type = Lds16;
};
template <>
struct LdsOf<float> {
  using type = Lds32;
};

__device__ __forceinline__ void clear(Lds16& L) {
  for (int i = threadIdx.x; i < BINS16 / 4; i += BLOCK)
    reinterpret_cast<u32x4*>(L.counts)[i] = (u32x4){0, 0, 0, 0};
  if (threadIdx.x == 0) L.zeros = L.far = L.s.flag = 0;
}
__device__ __forceinline__ void clear(Lds32& L) {
  for (int i = threadIdx.x; i < BINS32 / 2; i += BLOCK)
    reinterpret_cast<u32x4*>(L.w)[i] = (u32x4){0, 0, 0, 0};
  for (int i = threadIdx.x; i < BINS32 / 4; i += BLOCK)
    reinterpret_cast<u32x4*>(L.n)[i] = (u32x4){0, 0, 0, 0};
}
__device__ __forceinline__ int* ties_of(Lds16& L) { return L.ties; }
__device__ __forceinline__ int* ties_of(Lds32& L) { return L.index; }

// A barrier that waits for LDS alone: the row's loads stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <typename T, int NC>
__global__ __launch_bounds__(BLOCK) void sample_filtered_kernel(const Args a) {
  __shared__ __attribute__((aligned(16))) typename LdsOf<T>::type L;
  const int b = blockIdx.x;
  Row r;
  if (!open_row(a, b, r, L.s)) return;  // out and kept stay as they were
  const T* row = reinterpret_cast<const T*>(a.logits) + (int64_t)b * a.V;
  Entries<T, NC> e;
  e.open(row, a.V);  // under the loads' flight:
  const bool warm = (double)a.temperature[b] > 0.0;
  clear(L);
  lds_barrier();
  if constexpr (sizeof(T) == 2)
    if (warm) count_values(e, L);
  float m = -INFINITY;
  e.each_chunk([&](int, const u32x4 v) {
#pragma unroll
    for (int j = 0; j < e.PER; ++j) m = fmaxf(m, e.get(v, j));  // not a NaN
  });
  r.m = __uint_as_float(__builtin_amdgcn_readfirstlane(
      __float_as_uint(block_largest(m, L.s.red_f) + 0.f)));
  Answer ans{0, 1, 0, 0, 0.f};  // no candidate: token 0
  bool done = true;             // the same in all threads
  if (r.m > -INFINITY) {
    ans = {-1, 1, 0, 1 << 30, r.m};  // T <= 0: the first of the largest
    if (warm) {
      if constexpr (sizeof(T) == 2)
        done = bf16_row(e, r, L, ans);
      else
        done = fp32_row(e, r, a, L, ans);
    }
  }
  // (known to be uniform, neither branch keeps the other's registers)
  if (!__builtin_amdgcn_readfirstlane(done)) {
    __syncthreads();
    ans = general(Plain<T>{row, a.V}, r, L.s);
  } else if (__builtin_amdgcn_readfirstlane(ans.token) < 0) {
    ans.token = nth_of_value(e, ans.x, ans.nth, ans.ties, ties_of(L), L.s);
  }
  answer(a, b, ans.token, ans.kept);
}

}  // namespace

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <cmath>

void sample_filtered(torch::Tensor out, torch::Tensor logits,
                     torch::Tensor temperature, torch::Tensor top_k,
                     torch::Tensor top_p, torch::Tensor min_p,
                     torch::Tensor uniform,
                     c10::optional<torch::Tensor> kept) {
  const auto dev = logits.device();
  TORCH_CHECK(logits.dim() == 2 && logits.is_contiguous() &&
                  (logits.scalar_type() == torch::kBFloat16 ||
                   logits.scalar_type() == torch::kFloat32),
              "logits must be a contiguous bf16 or f32 [B, V]");
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V >= 1 && V <= MAXV, "V must be from 1 to 2^20");
  const auto row = [&](const torch::Tensor& t, const char* name,
                       torch::ScalarType type) {
    TORCH_CHECK(t.device() == dev, name, " is on another device");
    TORCH_CHECK(t.scalar_type() == type && t.dim() == 1 && t.size(0) == B &&
                    t.is_contiguous(),
                name, " must be a contiguous ", type, " [B]");
  };
  row(out, "out", torch::kInt32);
  row(temperature, "temperature", torch::kFloat32);
  row(top_k, "top_k", torch::kInt32);
  row(top_p, "top_p", torch::kFloat32);
  row(min_p, "min_p", torch::kFloat32);
  row(uniform, "uniform", torch::kFloat32);
  if (kept.has_value()) row(*kept, "kept", torch::kInt32);
  if (B == 0) return;
  c10::DeviceGuard guard(dev);
  hipStream_t s = at::hip::getCurrentHIPStream().stream();
  int bits = 51;
  while (V > 1ll << (63 - bits)) --bits;
  const Args a{(int32_t*)out.data_ptr(),
               kept.has_value() ? (int32_t*)kept->data_ptr() : nullptr,
               logits.data_ptr(),
               (const float*)temperature.data_ptr(),
               (const int32_t*)top_k.data_ptr(),
               (const float*)top_p.data_ptr(),
               (const float*)min_p.data_ptr(),
               (const float*)uniform.data_ptr(),
               (int)V,
               std::ldexp(1.0, bits),
               std::ldexp(1.0, -bits)};
  // what a row has beyond the registers' 64 KB (bf16, short rows), 128 KB (f32)
  // or 256 KB is read again; 64 KB keep the instructions few: 256 rows of 8192
  // take 11.8 us against 14.9 with room for 256 KB, of 32000 19.8 against 23.3
  const dim3 grid((unsigned)B), block(BLOCK);
#define LAUNCH(T, NC)                                                         \
  hipLaunchKernelGGL((sample_filtered_kernel<T, NC>), grid, block, 0, s, a)
  if (logits.scalar_type() == torch::kFloat32)
    LAUNCH(float, 8);
  else if (V * 2 <= 65536 - 16)
    LAUNCH(__hip_bfloat16, 4);
  else
    LAUNCH(__hip_bfloat16, 16);
#undef LAUNCH
  HIP_CHECK_LAST();
}
