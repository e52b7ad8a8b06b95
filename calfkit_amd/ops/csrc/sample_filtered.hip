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
// sums do not depend on the order of the atomics), and the bin that holds a
// border is resolved by ranking its members.  Rows that fit neither (values
// beyond 2^23, more distinct values than the list holds, a bin with too many
// members) take a bisection over the keys, slow and general.
//
// Bound: the row's bytes and the LDS histogram (one add an entry).  One block
// of 1024 threads is one row; it reads the row once and holds it in registers
// (128256 bf16 are 64 registers a thread).

#include "common.h"

namespace {

using u32x4 = __attribute__((ext_vector_type(4))) unsigned;

constexpr int BLOCK = 1024;
constexpr int NWAVES = BLOCK / WAVE;
constexpr int MAXCHUNKS = 512;  // 16 B loads of a thread: up to 2^20 entries
constexpr int MAXV = 1 << 20;

// bf16: magnitudes [2^-41, 2^23) are 64 octaves of 128 values, each sign
constexpr int BINS16 = 16384;
constexpr int LO16 = 86 << 7, HI16 = 150 << 7;
constexpr float FAR_VALUE = -8388608.f;  // -2^23
constexpr int DISTINCT = 4096;
// fp32
constexpr int BINS32 = 8192;
constexpr int MEMBERS = 2048;
constexpr double FIXED = 8796093022208.0;  // 2^43: 2^20 entries sum below 2^63

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
};

// What every path is asked: the row's filters.
struct Row {
  float m;        // largest logit
  double T;       // temperature > 0
  int k;          // top_k or V
  double top_p;   // >= 1: off
  double min_p;
  double u;
};

// The token: an index, or (token < 0) the nth of the entries of value x.
struct Answer {
  int token, kept, nth;
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

__device__ __forceinline__ double weight(const float x, const Row& r) {
  return x == r.m ? 1.0 : exp(((double)x - (double)r.m) / r.T);
}

// ---- block-wide sums and scans; `lds` holds NWAVES + 1 values
template <typename S>
__device__ __forceinline__ S block_scan(S x, S* lds, S* total) {
  const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
  S incl = x;
#pragma unroll
  for (int off = 1; off < WAVE; off <<= 1) {
    const S y = __shfl_up(incl, off, WAVE);
    if (lane >= off) incl += y;
  }
  __syncthreads();  // the last user of lds is done
  if (lane == WAVE - 1) lds[wid] = incl;
  __syncthreads();
  S before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < NWAVES; ++w) {
    const S y = lds[w];
    if (w < wid) before += y;
    all += y;
  }
  *total = all;
  return before + incl - x;
}

template <typename S>
__device__ __forceinline__ S block_total(S x, S* lds) {
  const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off, WAVE);
  __syncthreads();
  if (lane == 0) lds[wid] = x;
  __syncthreads();
  S all = 0;
#pragma unroll
  for (int w = 0; w < NWAVES; ++w) all += lds[w];
  return all;
}

__device__ __forceinline__ float block_largest(float x, float* lds) {
  const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
  x = wave_max(x);
  __syncthreads();
  if (lane == 0) lds[wid] = x;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NWAVES; ++w) x = fmaxf(x, lds[w]);
  return x;
}

// One row in chunks of BLOCK x 16 B: chunk c of thread t is the entries from
// (c * BLOCK + t) * PER - lead on, so that every load is aligned whatever the
// row's start; the first NC chunks stay in registers.  Entries outside the
// row read as NaN, which is no candidate.
template <typename T, int NC>
struct Entries {
  static constexpr int PER = 16 / sizeof(T);
  const T* row;
  int V, lead, chunks;
  u32x4 held[NC > 0 ? NC : 1];

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
          v[j / 2] = (j & 1) ? (v[j / 2] & 0xffffu) | ((unsigned)src[i + j] << 16)
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
    for (int c = NC; c < chunks; ++c) f(c, load(c));
  }
  static __device__ __forceinline__ float get(const u32x4 v, const int j) {
    if constexpr (sizeof(T) == 4)
      return __uint_as_float(v[j]);
    else
      return __uint_as_float((j & 1) ? (v[j / 2] & 0xffff0000u)
                                     : (v[j / 2] << 16));
  }
  // f(index, value) of every candidate, -0 as +0
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    each_chunk([&](const int c, const u32x4 v) {
      const int i = first_of(c);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float x = get(v, j) + 0.f;
        if (candidate(x)) f(i + j, x);
      }
    });
  }
};

struct Shared {
  double red_d[NWAVES + 1];
  unsigned long long red_u[NWAVES + 1];
  float red_f[NWAVES];
  int flag, hit, at;
  unsigned members;
  double hit_before, hit_w;
  int per_chunk[MAXCHUNKS];
};

// The j-th entry, in order of index, whose value is x.
template <typename E>
__device__ __forceinline__ int nth_of_value(const E& e, const float x, const int j,
                            Shared& s) {
  for (int i = threadIdx.x; i < e.chunks; i += BLOCK) s.per_chunk[i] = 0;
  __syncthreads();
  e.each_chunk([&](const int c, const u32x4 v) {
    int n = 0;
#pragma unroll
    for (int q = 0; q < E::PER; ++q) n += E::get(v, q) == x;
    if (n) atomicAdd(&s.per_chunk[c], n);
  });
  __syncthreads();
  int chunk = 0, left = j;
  while (chunk < e.chunks - 1 && left >= s.per_chunk[chunk])
    left -= s.per_chunk[chunk++];
  const u32x4 v = e.load(chunk);
  int n = 0;
#pragma unroll
  for (int q = 0; q < E::PER; ++q) n += E::get(v, q) == x;
  unsigned long long all;
  int before = (int)block_scan<unsigned long long>(n, s.red_u, &all);
  if (left >= before && left < before + n) {
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

// Count and weight of the candidates with a key above (or from) t.
template <typename E>
__device__ __forceinline__ void above(const E& e, const Row& r, const unsigned t,
                      const bool from, long long& n, double& w, Shared& s,
                      const bool weigh) {
  unsigned long long cnt = 0;
  double sum = 0.0;
  e.each([&](int, const float x) {
    const unsigned key = key_of(x);
    if (key > t || (from && key == t)) {
      ++cnt;
      if (weigh) sum += weight(x, r);
    }
  });
  n = (long long)block_total<unsigned long long>(cnt, s.red_u);
  w = weigh ? block_total<double>(sum, s.red_d) : 0.0;
}

// The largest key t with  count(key >= t) >= rank  or  weight(key >= t) > goal
template <typename E>
__device__ __forceinline__ unsigned bisect(const E& e, const Row& r, const bool by_count,
                           const long long rank, const double goal,
                           const bool reach, Shared& s) {
  unsigned t = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const unsigned up = t | (1u << bit);
    long long n;
    double w;
    above(e, r, up, true, n, w, s, !by_count);
    if (by_count ? n >= rank : (reach ? w >= goal : w > goal)) t = up;
  }
  return t;
}

template <typename E>
__device__ __forceinline__ double sum_of_first(const E& e, const Row& r, const long long n,
                               Shared& s) {
  const unsigned t = bisect(e, r, true, n, 0.0, false, s);
  long long cnt;
  double w;
  above(e, r, t, false, cnt, w, s, true);
  return w + (double)(n - cnt) * weight(value_of(t), r);
}

// A call of its own: its registers are not the fast paths'.
template <typename T>
__device__ __noinline__ Answer general(const T* row, const int V, const Row& r, Shared& s) {
  Entries<T, 0> e;  // read again in every pass
  e.open(row, V);
  long long all;
  double w_all;
  above(e, r, 0u, true, all, w_all, s, true);
  long long n = min((long long)r.k, all);
  if (r.top_p < 1.0) {
    const double goal =
        r.top_p * (n == all ? w_all : sum_of_first(e, r, n, s));
    long long np = 0;
    if (goal > 0.0) {
      // the key in which the sum reaches the goal (the last of all where
      // rounding keeps it short): ranks above it lie before the goal
      const unsigned t = bisect(e, r, false, 0, goal, true, s);
      long long upto, cnt;
      double w, before;
      above(e, r, t, true, upto, w, s, false);
      above(e, r, t, false, cnt, before, s, true);
      np = cnt + within(goal, before, weight(value_of(t), r),
                        (int)(upto - cnt), false);
    }
    n = min(n, np);
  }
  unsigned long long cm = 0;
  e.each([&](int, const float x) { cm += weight(x, r) >= r.min_p; });
  n = min(n, (long long)block_total<unsigned long long>(cm, s.red_u));
  n = max(n, 1ll);
  const double goal = r.u * sum_of_first(e, r, n, s);
  unsigned t = bisect(e, r, false, 0, goal, false, s);
  long long upto, cnt;
  double w, before;
  above(e, r, t, false, cnt, before, s, true);
  if (cnt >= n) {  // rounding kept every sum short: the last rank kept
    t = bisect(e, r, true, n, 0.0, false, s);
    above(e, r, t, false, cnt, before, s, true);
  }
  above(e, r, t, true, upto, w, s, false);
  int j = within(goal, before, weight(value_of(t), r), (int)(upto - cnt) - 1,
                 true);
  j = (int)min((long long)j, n - 1 - cnt);
  return {nth_of_value(e, value_of(t), j, s), (int)n, 0, 0.f};
}

// --------------------------------------------------- bf16: bins are values

struct Lds16 {
  union {
    unsigned counts[BINS16];
    double w[DISTINCT];  // of the list, once it is made
  };
  double before_w[DISTINCT + 1];
  int before_n[DISTINCT + 1];
  unsigned short code[DISTINCT];
  Shared s;
  unsigned zeros, far;
};

// The list's last entry i for which ok(i), which holds for a prefix of it.
template <typename F>
__device__ __forceinline__ int last_entry(const int entries, Shared& s, F ok) {
  __syncthreads();
  if (threadIdx.x == 0) s.hit = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < entries; i += BLOCK)
    if (ok(i) && (i + 1 == entries || !ok(i + 1))) atomicMax(&s.hit, i);
  __syncthreads();
  return s.hit;
}

// Both row functions say false where the general search has to take the row.
template <int NC>
__device__ __forceinline__ bool bf16_row(const Entries<__hip_bfloat16, NC>& e,
                                        const Row& r, Lds16& L, Answer& ans) {
  Shared& s = L.s;
  const int tid = threadIdx.x;
  for (int i = tid; i < BINS16 / 4; i += BLOCK)
    reinterpret_cast<uint4*>(L.counts)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) L.zeros = L.far = s.flag = 0;
  __syncthreads();

  // bin = magnitude - LO16, the negative ones 8192 further: as a byte
  // address it is (offset * 4) | sign, in both halves of a word at once
  e.each_chunk([&](int, const u32x4 v) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      using u16x2 = __attribute__((ext_vector_type(2))) unsigned short;
      const unsigned mag = v[q] & 0x7fff7fffu;
      const u16x2 off = __builtin_bit_cast(u16x2, mag) -
                        (u16x2){(unsigned short)LO16, (unsigned short)LO16};
      const unsigned offs = __builtin_bit_cast(unsigned, off);
      if ((offs & 0xe000e000u) == 0) {
        const u16x2 by4 = off << (u16x2){2, 2};
        const unsigned at =
            __builtin_bit_cast(unsigned, by4) | (v[q] & 0x80008000u);
        char* base = reinterpret_cast<char*>(L.counts);
        atomicAdd(reinterpret_cast<unsigned*>(base + (at & 0xffffu)), 1u);
        atomicAdd(reinterpret_cast<unsigned*>(base + (at >> 16)), 1u);
      } else {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const unsigned u = (v[q] >> (16 * hf)) & 0xffffu;
          const unsigned a = u & 0x7fffu;
          if (a >= (unsigned)LO16 && a < (unsigned)HI16)
            atomicAdd(&L.counts[(a - LO16) + ((u >> 15) << 13)], 1u);
          else if (a == 0)
            atomicAdd(&L.zeros, 1u);
          else if (a < (unsigned)LO16)
            s.flag = 1;  // magnitudes below 2^-41
          else if (u > 0x8000u && a < 0x7f80u)
            atomicAdd(&L.far, 1u);  // finite, -2^23 or less
        }
      }
    }
  });
  __syncthreads();
  // far values have to weigh nothing: exp(-746) is 0 in 64 bits
  if (s.flag || r.m >= -FAR_VALUE ||
      (L.far && (double)r.m - (double)FAR_VALUE < 746.0 * r.T))
    return false;

  // ---- the list of distinct values, falling: thread t looks at places
  // 16 t .., the positive values from the largest down, zero, the negative
  const auto count_at = [&](const int p) __attribute__((always_inline)) {
    return L.counts[p < BINS16 / 2 ? BINS16 / 2 - 1 - p : p];
  };
  unsigned n = 0, distinct = 0;
  const bool mid = tid == BLOCK / 2;  // the zeros come right before it
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const unsigned c = count_at(tid * 16 + j);
    n += c;
    distinct += c != 0;
  }
  if (mid && L.zeros) {
    n += L.zeros;
    ++distinct;
  }
  unsigned long long total;
  const unsigned long long pre = block_scan<unsigned long long>(
      ((unsigned long long)distinct << 32) | n, s.red_u, &total);
  const int entries = (int)(total >> 32);
  const int listed = (int)(total & 0xffffffffu);
  if (entries > DISTINCT) return false;
  int at = (int)(pre >> 32);
  int seen = (int)(pre & 0xffffffffu);
  if (mid && L.zeros) {
    L.code[at] = 0;
    L.before_n[at++] = seen;
    seen += L.zeros;
  }
#pragma unroll 4
  for (int j = 0; j < 16; ++j) {
    const int p = tid * 16 + j;
    const unsigned c = count_at(p);
    if (c == 0) continue;
    L.code[at] = (unsigned short)(
        p < BINS16 / 2 ? LO16 + BINS16 / 2 - 1 - p
                       : (0x8000 | (LO16 + p - BINS16 / 2)));
    L.before_n[at++] = seen;
    seen += c;
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
        last_entry(entries, s, [&](int i) { return L.before_n[i] < n; });
    return L.before_w[i] + (double)(n - L.before_n[i]) * L.w[i];
  };
  const int all = listed + (int)L.far;
  int N = min(r.k, all);
  double Z = sum_first(N);
  if (r.top_p < 1.0) {
    const double goal = r.top_p * Z;
    int np = 0;
    if (goal > 0.0) {
      const int i =
          last_entry(entries, s, [&](int i) { return L.before_w[i] < goal; });
      np = L.before_n[i] + within(goal, L.before_w[i], L.w[i],
                                  L.before_n[i + 1] - L.before_n[i], false);
    }
    N = min(N, np);
  }
  if (!(r.min_p <= 0.0)) {
    const int i =
        last_entry(entries, s, [&](int i) { return L.w[i] >= r.min_p; });
    N = min(N, L.w[i] >= r.min_p ? L.before_n[i + 1] : 0);
  }
  N = max(N, 1);
  const double goal = r.u * sum_first(N);
  const int i =
      last_entry(entries, s, [&](int i) { return L.before_w[i] <= goal; });
  int j = within(goal, L.before_w[i], L.w[i],
                 L.before_n[i + 1] - L.before_n[i] - 1, true);
  j = max(0, min(j, N - 1 - L.before_n[i]));
  const float x = __uint_as_float((unsigned)L.code[i] << 16) + 0.f;
  ans = {-1, N, j, x};
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
__device__ __forceinline__ bool fp32_row(const Entries<float, NC>& e,
                                        const Row& r, Lds32& L, Answer& ans) {
  constexpr int PT = BINS32 / BLOCK;  // bins of a thread, in order
  Shared& s = L.s;
  const int tid = threadIdx.x;
  for (int i = tid; i < BINS32; i += BLOCK) {
    L.w[i] = 0;
    L.n[i] = 0;
  }
  if (r.m == INFINITY) return false;
  // values that weigh nothing (exp(-746) is 0 in 64 bits) are counted alone;
  // the bins cover the others
  const double reach = 746.0 * r.T;
  float low = r.m;
  e.each([&](int, const float x) {
    if ((double)r.m - (double)x <= reach) low = fminf(low, x);
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
  const double inv = 1.0 / r.T;
  unsigned long long nm = 0, far = 0;
  e.each([&](int, const float x) {
    if (x < low) {
      ++far;
      nm += 0.0 >= r.min_p;
      return;
    }
    const double w = x == r.m ? 1.0 : exp(((double)x - (double)r.m) * inv);
    const int b = bin_of(x);
    atomicAdd(&L.w[b], (unsigned long long)(w * FIXED + 0.5));
    atomicAdd(&L.n[b], 1u);
    nm += w >= r.min_p;
  });
  far = block_total<unsigned long long>(far, s.red_u);
  nm = block_total<unsigned long long>(nm, s.red_u);
  __syncthreads();

  unsigned long long tw = 0, tn = 0, w_fix, listed;
#pragma unroll
  for (int j = 0; j < PT; ++j) {
    tw += L.w[tid * PT + j];
    tn += L.n[tid * PT + j];
  }
  const unsigned long long bw = block_scan<unsigned long long>(tw, s.red_u,
                                                               &w_fix);
  const unsigned long long bn = block_scan<unsigned long long>(tn, s.red_u,
                                                               &listed);
  const double w_all = (double)w_fix * (1.0 / FIXED);

  // ---- the bin with a rank or a sum, and its members in order
  int bin = -1, members = 0, before_n = 0;
  double before_w = 0.0;
  // (first bin whose count up to its end reaches `rank`, or whose sum does)
  const auto open = [&](const bool by_count, const long long rank,
                        const double goal, const bool pass) __attribute__((always_inline)) {
    __syncthreads();
    if (tid == 0) s.hit = -1;
    __syncthreads();
    unsigned long long cw = bw, cn = bn;
#pragma unroll
    for (int j = 0; j < PT; ++j) {
      const int b = tid * PT + j;
      const unsigned long long ew = cw + L.w[b], en = cn + L.n[b];
      const double d0 = (double)cw * (1.0 / FIXED);
      const double d1 = (double)ew * (1.0 / FIXED);
      const bool here =
          L.n[b] != 0 &&
          (by_count ? ((long long)cn < rank && (long long)en >= rank)
           : pass   ? (d0 <= goal && d1 > goal)
                    : (d0 < goal && d1 >= goal));
      if (here) {
        s.hit = b;
        s.at = (int)cn;
        s.hit_before = d0;
      }
      cw = ew;
      cn = en;
    }
    __syncthreads();
    if (s.hit < 0 || s.hit == bin) return s.hit >= 0;
    bin = s.hit;
    before_n = s.at;
    before_w = s.hit_before;
    members = (int)L.n[bin];
    if (members > MEMBERS) return true;  // the caller looks
    if (tid == 0) s.members = 0;
    __syncthreads();
    e.each([&](const int i, const float x) {
      if (x >= low && bin_of(x) == bin) {
        const unsigned p = atomicAdd(&s.members, 1u);
        L.key[p] = key_of(x);
        L.index[p] = i;
      }
    });
    __syncthreads();
    for (int p = tid; p < members; p += BLOCK) {
      const unsigned key = L.key[p];
      const int i = L.index[p];
      int rank_in = 0;
      for (int q = 0; q < members; ++q) {
        const unsigned k2 = L.key[q];
        rank_in += k2 > key || (k2 == key && L.index[q] < i);
      }
      L.sorted_key[rank_in] = key;
      L.sorted_index[rank_in] = i;
    }
    __syncthreads();
    return true;
  };
  // walks the open bin: ranks in it whose sum before (or with) them does not
  // pass the goal, at most `upto` ranks; the sum of those
  const auto walk = [&](const int upto, const double goal, const bool with,
                        double& sum) __attribute__((always_inline)) {
    const int per = (members + BLOCK - 1) / BLOCK;
    double mine[MEMBERS / BLOCK], t = 0.0, all;
#pragma unroll
    for (int j = 0; j < MEMBERS / BLOCK; ++j) {
      const int p = tid * per + j;
      mine[j] = 0.0;
      if (j < per && p < members && p < upto)
        mine[j] = weight(value_of(L.sorted_key[p]), r);
      t += mine[j];
    }
    double b = before_w + block_scan<double>(t, s.red_d, &all);
    unsigned long long n = 0;
#pragma unroll
    for (int j = 0; j < MEMBERS / BLOCK; ++j) {
      const int p = tid * per + j;
      if (j < per && p < members && p < upto)
        n += with ? (b + mine[j] <= goal) : (b < goal);
      b += mine[j];
    }
    sum = before_w + all;
    return (int)block_total<unsigned long long>(n, s.red_u);
  };
  const auto sum_first = [&](const long long n, double& Z) __attribute__((always_inline)) {
    if (n >= (long long)listed) {
      Z = w_all;
      return true;
    }
    open(true, n, 0.0, false);
    if (members > MEMBERS) return false;
    walk((int)(n - before_n), 0.0, false, Z);
    return true;
  };

  const long long all = (long long)(listed + far);
  long long N = min((long long)r.k, all);
  double Z;
  if (r.top_p < 1.0) {
    if (!sum_first(N, Z)) return false;
    const double goal = r.top_p * Z;
    long long np = 0;
    if (goal > 0.0) {
      if (open(false, 0, goal, false)) {
        if (members > MEMBERS) return false;
        double sum;
        np = before_n + walk(members, goal, false, sum);
      } else {
        np = (long long)listed;
      }
    }
    N = min(N, np);
  }
  N = max(1ll, min(N, (long long)nm));
  if (!sum_first(N, Z)) return false;
  const double goal = r.u * Z;
  // (the two sums agree to the last bits only: the last rank kept at most)
  if (!open(false, 0, goal, true) || before_n >= N) open(true, N, 0.0, false);
  if (members > MEMBERS) return false;
  double sum;
  int j = walk(members, goal, true, sum);
  j = (int)min((long long)min(j, members - 1), N - 1 - before_n);
  ans = {L.sorted_index[j], (int)N, 0, 0.f};
  return true;
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

template <typename T, int NC>
__global__ __launch_bounds__(BLOCK) void sample_filtered_kernel(const Args a) {
  __shared__ __attribute__((aligned(16))) typename LdsOf<T>::type L;
  const int b = blockIdx.x;
  const float u = a.uniform[b];
  if (u < 0.f) return;  // the row is not asked for: it stays as it was
  Entries<T, NC> e;
  e.open(reinterpret_cast<const T*>(a.logits) + (int64_t)b * a.V, a.V);
  Row r;
  float m = -INFINITY;
  e.each([&](int, const float x) { m = fmaxf(m, x); });
  r.m = block_largest(m, L.s.red_f);
  const float T_ = a.temperature[b];
  const int k = a.top_k[b];
  r.T = (double)T_;
  r.k = (k > 0 && k < a.V) ? k : a.V;
  r.top_p = (double)a.top_p[b];
  r.min_p = (double)a.min_p[b];
  r.u = fmin((double)u, 1.0 - 0x1p-53);  // [0, 1); NaN too
  Answer ans{0, 1, 0, 0.f};
  bool done = true;  // the same in all threads
  if (r.m == -INFINITY) {
    // no candidate: token 0
  } else if (!(T_ > 0.f)) {
    ans = {-1, 1, 0, r.m};
  } else {
    if constexpr (sizeof(T) == 2)
      done = bf16_row(e, r, L, ans);
    else
      done = fp32_row(e, r, L, ans);
  }
  // (known to be uniform, the call keeps no register of the other branch)
  if (!__builtin_amdgcn_readfirstlane(done)) {
    __syncthreads();
    ans = general(reinterpret_cast<const T*>(a.logits) + (int64_t)b * a.V, a.V,
                  r, L.s);
  } else if (__builtin_amdgcn_readfirstlane(ans.token) < 0) {
    ans.token = nth_of_value(e, ans.x, ans.nth, L.s);
  }
  if (threadIdx.x == 0) {
    a.out[b] = ans.token;
    if (a.kept) a.kept[b] = ans.kept;
  }
}

}  // namespace

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

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
  const Args a{(int32_t*)out.data_ptr(),
               kept.has_value() ? (int32_t*)kept->data_ptr() : nullptr,
               logits.data_ptr(),
               (const float*)temperature.data_ptr(),
               (const int32_t*)top_k.data_ptr(),
               (const float*)top_p.data_ptr(),
               (const float*)min_p.data_ptr(),
               (const float*)uniform.data_ptr(),
               (int)V};
#define LAUNCH(T, NC)                                                       \
  hipLaunchKernelGGL((sample_filtered_kernel<T, NC>), dim3((unsigned)B),    \
                     dim3(BLOCK), 0, s, a)
  // bf16 rows of up to 64 KB or 256 KB stay in registers (beyond, the rest is
  // read again); fp32 rows are read from L2 in every pass
  if (logits.scalar_type() == torch::kFloat32)
    LAUNCH(float, 0);
  else if (V * 2 <= 65536 - 16)
    LAUNCH(__hip_bfloat16, 4);
  else
    LAUNCH(__hip_bfloat16, 16);
#undef LAUNCH
  HIP_CHECK_LAST();
}
