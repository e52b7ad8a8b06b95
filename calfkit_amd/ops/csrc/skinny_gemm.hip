// Skinny-M decode GEMM for MI355X (gfx950): out[M,N] = x[M,K] @ W^T,
// W stored [N,K] row-major (nn.Linear layout), M = decode batch (<= 64).
//
// Regime: weight-streaming bound — every decode step reads every weight
// byte exactly once (16 GB for llama-8B), so the kernel's one job is to
// stream W at the HBM ceiling while the MFMA work rides along.  hipBLASLt's
// heuristic tiles ran these shapes at ~20% of the stream bound
// (profiles/r01_bench_llama8b_kernelstats.md) — this kernel exists to fix
// that, per the CDNA guide's sampling-regime GEMM recipe (decomposition
// first: (N/64)*SPLITK blocks ~ 1-2x CU count; operands as direct
// 16 B/lane fragment loads, W rows contiguous because the layout is [N,K]).
//
// Decomposition:
//   grid = (N/64, SPLITK); 4 waves per block; each wave owns 1/4 of the
//   block's K-slice (in-block split-K), accumulating the full 64x64
//   (M-pad x BN) tile in MFMA accumulators; waves reduce through LDS; the
//   block writes ONE fp32 slab [Mp, 64] to workspace[sk].
//   A separate tiny epilogue kernel (reduce_slabs*) sums the SPLITK slabs
//   and casts to bf16 — optionally fusing SiLU·mul (the MLP gate) so the
//   hand-written path covers the whole SiLU-MLP chain.
//
// Fragments (mfma_f32_16x16x32_bf16, maps verified in tests):
//   A[i][k]: lane i=l&15, k=(l>>4)*8+m  -> x row i, 16 B contiguous  (L2)
//   B[k][j]: lane j=l&15, k=(l>>4)*8+m  -> W^T row n0+j, 16 B contiguous
//   C[r][c]: lane c=l&15, r=(l>>4)*4+reg

#include "common.h"

using f32x4 = __attribute__((ext_vector_type(4))) float;
using bf16x8v = __attribute__((ext_vector_type(8))) __bf16;

#define MFMA16(a, b, c) __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0)

#define BN 64      // output columns per block
#define SGWAVES 4  // waves per block (in-block K split)

// MT: padded M (16, 32 or 64).  x is [M,K]; rows >= M read row M-1 (the
// result rows >= M are discarded by the epilogue).  KU: k-unroll depth per
// wave iteration (more independent loads in flight).  W loads are
// NONTEMPORAL: every weight byte is read exactly once per step — keeping it
// out of L2 leaves the cache to x and the KV pages.
template <int MT, int KU, bool NT>
__global__ __launch_bounds__(SGWAVES * WAVE) void skinny_gemm_kernel(
    float* __restrict__ work,            // [SPLITK, Mp, N] fp32 slabs
    __hip_bfloat16* __restrict__ out,    // [M, N] direct target (splitk==1)
    const __hip_bfloat16* __restrict__ x, // [M, K]
    const __hip_bfloat16* __restrict__ w, // [N, K]  (W^T of the math)
    const int M, const int N, const int K, const int splitk,
    const int direct) {  // 1: write bf16 straight to out (needs splitk==1)
  constexpr int MTILES = MT / 16;
  const int n0 = blockIdx.x * BN;
  const int sk = blockIdx.y;
  const int wid = threadIdx.x / WAVE;
  const int lane = threadIdx.x % WAVE;
  const int l16 = lane & 15;
  const int l4 = lane >> 4;

  // this block's K-slice, then this wave's quarter of it (32-aligned)
  const int k_block = (K / splitk);
  const int k_begin = sk * k_block + wid * (k_block / SGWAVES);
  const int k_end = k_begin + k_block / SGWAVES;

  f32x4 acc[MTILES][BN / 16];
#pragma unroll
  for (int mi = 0; mi < MTILES; ++mi)
#pragma unroll
    for (int ni = 0; ni < BN / 16; ++ni)
      acc[mi][ni] = (f32x4){0.f, 0.f, 0.f, 0.f};

  // A row per m-tile for this lane; clamp to the real M
  int arow[MTILES];
#pragma unroll
  for (int mi = 0; mi < MTILES; ++mi)
    arow[mi] = min(mi * 16 + l16, M - 1);
  const int wrow = n0 + l16;  // W^T row for this lane's B fragments

  for (int k = k_begin; k < k_end; k += KU) {
    // KU/32 k-steps unrolled: all A/B fragment loads of the span issue
    // before the MFMAs consume them (the compiler schedules the waits)
    bf16x8v a[KU / 32][MTILES], b[KU / 32][BN / 16];
#pragma unroll
    for (int kk = 0; kk < KU; kk += 32) {
#pragma unroll
      for (int mi = 0; mi < MTILES; ++mi)
        a[kk / 32][mi] = *reinterpret_cast<const bf16x8v*>(
            x + (int64_t)arow[mi] * K + k + kk + l4 * 8);
#pragma unroll
      for (int ni = 0; ni < BN / 16; ++ni) {
        const bf16x8v* src = reinterpret_cast<const bf16x8v*>(
            w + (int64_t)(wrow + ni * 16) * K + k + kk + l4 * 8);
        b[kk / 32][ni] = NT ? __builtin_nontemporal_load(src) : *src;
      }
    }
#pragma unroll
    for (int kk = 0; kk < KU; kk += 32)
#pragma unroll
      for (int ni = 0; ni < BN / 16; ++ni)
#pragma unroll
        for (int mi = 0; mi < MTILES; ++mi)
          acc[mi][ni] = MFMA16(a[kk / 32][mi], b[kk / 32][ni], acc[mi][ni]);
  }

  // ---- cross-wave reduce through LDS, then one fp32 slab write
  __shared__ float red[SGWAVES][MT][BN];
#pragma unroll
  for (int mi = 0; mi < MTILES; ++mi)
#pragma unroll
    for (int ni = 0; ni < BN / 16; ++ni)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        red[wid][mi * 16 + l4 * 4 + r][ni * 16 + l16] = acc[mi][ni][r];
  __syncthreads();

  if (direct) {
    // single-slice: write bf16 straight to the output, no slab round trip
    for (int i = threadIdx.x; i < MT * BN; i += SGWAVES * WAVE) {
      const int r = i / BN, c = i % BN;
      if (r >= M) continue;
      float v = red[0][r][c];
#pragma unroll
      for (int wv = 1; wv < SGWAVES; ++wv) v += red[wv][r][c];
      out[(int64_t)r * N + n0 + c] = f2bf(v);
    }
    return;
  }
  // 256 threads cover MT*BN outputs (MT=64: 16 each)
  float* slab = work + ((int64_t)sk * MT + 0) * N + n0;
  for (int i = threadIdx.x; i < MT * BN; i += SGWAVES * WAVE) {
    const int r = i / BN, c = i % BN;
    float v = red[0][r][c];
#pragma unroll
    for (int wv = 1; wv < SGWAVES; ++wv) v += red[wv][r][c];
    slab[(int64_t)r * N + c] = v;
  }
}

// ---- epilogue: sum SPLITK slabs -> bf16 (plain projection)
__global__ void reduce_slabs_kernel(__hip_bfloat16* __restrict__ out,  // [M,N]
                                    const float* __restrict__ work,
                                    const int M, const int N, const int Mp,
                                    const int splitk) {
  const int64_t total = (int64_t)M * N;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int r = i / N, c = i % N;
    float v = 0.f;
    for (int sk = 0; sk < splitk; ++sk)
      v += work[((int64_t)sk * Mp + r) * N + c];
    out[i] = f2bf(v);
  }
}

// ---- epilogue: gate/up slabs -> silu(gate)*up bf16 (the fused SiLU-MLP)
// work holds [splitk, Mp, 2F] with row layout [gate | up]; out is [M, F].
__global__ void reduce_slabs_silu_kernel(__hip_bfloat16* __restrict__ out,
                                         const float* __restrict__ work,
                                         const int M, const int F, const int Mp,
                                         const int splitk) {
  const int64_t total = (int64_t)M * F;
  const int64_t N = 2 * (int64_t)F;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int r = i / F, c = i % F;
    float g = 0.f, u = 0.f;
    for (int sk = 0; sk < splitk; ++sk) {
      const float* row = work + ((int64_t)sk * Mp + r) * N;
      g += row[c];
      u += row[F + c];
    }
    const float s = g / (1.f + __expf(-g));
    out[i] = f2bf(s * u);
  }
}

// ---- M=128/256 path: the guide's sampling-regime projection GEMM.
// 8 waves split the M rows; the shared W tile streams through LDS exactly
// ONCE per block (glds double-buffered, XOR-swizzled for conflict-free
// ds_read_b128 B-fragments) — the r14 version read W straight from global
// and paid 8x re-reads (0.2-0.4x of hipBLASLt); this is the fix.
// x stays as direct per-wave fragment loads (L2-resident).
template <int MT>
__global__ __launch_bounds__(8 * WAVE) void skinny_gemm_m_kernel(
    float* __restrict__ work,             // [SPLITK, Mp, N] fp32 slabs
    __hip_bfloat16* __restrict__ out,     // [M, N] direct target (direct=1)
    const __hip_bfloat16* __restrict__ x, // [M, K]
    const __hip_bfloat16* __restrict__ w, // [N, K]
    const int M, const int N, const int K, const int splitk,
    const int direct) {
  constexpr int MTILES = MT / 16 / 8;     // m-tiles per wave (8 waves)
  constexpr int KC = 64;                  // k-chunk depth
  const int n0 = blockIdx.x * BN;
  const int sk = blockIdx.y;
  const int tid = threadIdx.x;
  const int wid = tid / WAVE;
  const int lane = tid % WAVE;
  const int l16 = lane & 15;
  const int l4 = lane >> 4;

  const int k_begin = sk * (K / splitk);
  const int k_end = k_begin + K / splitk;

  // one __shared__ object only (guide §5 trap 4a): [2 bufs][64 rows][128 B]
  __shared__ __hip_bfloat16 wbuf[2][BN * KC];

  f32x4 acc[MTILES][BN / 16];
#pragma unroll
  for (int mi = 0; mi < MTILES; ++mi)
#pragma unroll
    for (int ni = 0; ni < BN / 16; ++ni)
      acc[mi][ni] = (f32x4){0.f, 0.f, 0.f, 0.f};

  int arow[MTILES];
#pragma unroll
  for (int mi = 0; mi < MTILES; ++mi)
    arow[mi] = min((wid * MTILES + mi) * 16 + l16, M - 1);

  // staging geometry: thread t loads 16 B of row r = t/8; the 16B-chunk it
  // fetches is XOR-swizzled (rule 21: swizzle the SOURCE, LDS dest linear)
  const int srow = tid / 8;
  const int schunk = (tid % 8) ^ (srow & 7);

  auto stage = [&](int buf, int k0) {
    const __hip_bfloat16* src =
        w + (int64_t)(n0 + srow) * K + k0 + schunk * 8;
    __builtin_amdgcn_global_load_lds(
        reinterpret_cast<const unsigned int*>(src),
        reinterpret_cast<unsigned int*>(
            &wbuf[buf][(wid * 8) * KC]),  // wave-uniform base; +lane*16 by HW
        16, 0, 0);
  };

  stage(0, k_begin);
  __syncthreads();

  int cur = 0;
  for (int k = k_begin; k < k_end; k += KC) {
    if (k + KC < k_end) stage(cur ^ 1, k + KC);

    // compute chunk cur: 2 k-steps of 32; B-frags from swizzled LDS
#pragma unroll
    for (int kk = 0; kk < KC; kk += 32) {
      bf16x8v a[MTILES];
#pragma unroll
      for (int mi = 0; mi < MTILES; ++mi)
        a[mi] = *reinterpret_cast<const bf16x8v*>(
            x + (int64_t)arow[mi] * K + k + kk + l4 * 8);
#pragma unroll
      for (int ni = 0; ni < BN / 16; ++ni) {
        const int row = ni * 16 + l16;
        const int chunk = ((kk / 8) + l4) ^ (row & 7);
        const bf16x8v b = *reinterpret_cast<const bf16x8v*>(
            &wbuf[cur][row * KC + chunk * 8]);
#pragma unroll
        for (int mi = 0; mi < MTILES; ++mi)
          acc[mi][ni] = MFMA16(a[mi], b, acc[mi][ni]);
      }
    }
    __syncthreads();  // drains the in-flight glds too (2-phase structure)
    cur ^= 1;
  }

  // epilogue: each wave owns its rows outright — no cross-wave reduce
#pragma unroll
  for (int mi = 0; mi < MTILES; ++mi) {
#pragma unroll
    for (int ni = 0; ni < BN / 16; ++ni) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = (wid * MTILES + mi) * 16 + l4 * 4 + r;
        const int col = n0 + ni * 16 + l16;
        if (direct) {
          if (row < M) out[(int64_t)row * N + col] = f2bf(acc[mi][ni][r]);
        } else {
          work[((int64_t)sk * MT + row) * N + col] = acc[mi][ni][r];
        }
      }
    }
  }
}

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <cstdlib>

// variant knobs (benchmarks/gemm_micro.py sweeps them; defaults are the
// winners of the within-probe A/B recorded in profiles/)
static int env_int(const char* name, int dflt) {
  const char* v = getenv(name);
  return v ? atoi(v) : dflt;
}

static void launch_skinny(torch::Tensor work, torch::Tensor out,
                          torch::Tensor x, torch::Tensor w,
                          int64_t splitk, int Mp, hipStream_t s,
                          int direct) {
  const int M = x.size(0), K = x.size(1), N = w.size(0);
  dim3 grid(N / BN, splitk), block(SGWAVES * WAVE);
  const int wave_k = Mp > 64 ? (K / splitk) : (K / splitk) / SGWAVES;
  const int ku_pref = env_int("CALF_SKGEMM_KU", 64);
  const int nt = env_int("CALF_SKGEMM_NT", 0);
  int ku = ku_pref;
  while (ku > 32 && wave_k % ku != 0) ku /= 2;
  if (wave_k % ku != 0) ku = 32;
  if (!env_int("CALF_SKGEMM_DIRECT", 1)) direct = 0;
#define L(MT, KU, NTV)                                                     \
  hipLaunchKernelGGL((skinny_gemm_kernel<MT, KU, NTV>), grid, block, 0, s, \
                     (float*)work.data_ptr(),                              \
                     (__hip_bfloat16*)out.data_ptr(),                      \
                     (const __hip_bfloat16*)x.data_ptr(),                  \
                     (const __hip_bfloat16*)w.data_ptr(), M, N, K,         \
                     (int)splitk, direct)
#define LN(MT, KU)                                                         \
  do {                                                                     \
    if (nt) L(MT, KU, true);                                               \
    else L(MT, KU, false);                                                 \
  } while (0)
#define LM(MT)                                                             \
  do {                                                                     \
    if (ku == 128) LN(MT, 128);                                            \
    else if (ku == 64) LN(MT, 64);                                         \
    else LN(MT, 32);                                                       \
  } while (0)
#define LMBIG(MT)                                                          \
  hipLaunchKernelGGL((skinny_gemm_m_kernel<MT>), grid, dim3(8 * WAVE),     \
                     0, s, (float*)work.data_ptr(),                        \
                     (__hip_bfloat16*)out.data_ptr(),                      \
                     (const __hip_bfloat16*)x.data_ptr(),                  \
                     (const __hip_bfloat16*)w.data_ptr(), M, N, K,         \
                     (int)splitk, direct)
  switch (Mp) {
    case 16: LM(16); break;
    case 32: LM(32); break;
    case 64: LM(64); break;
    case 128: LMBIG(128); break;
    case 256: LMBIG(256); break;
    default: TORCH_CHECK(false, "skinny_gemm: bad M pad ", Mp);
  }
#undef LMBIG
#undef LM
#undef LN
#undef L
}

static int pad_m(int M) {
  if (M <= 16) return 16;
  if (M <= 32) return 32;
  if (M <= 64) return 64;
  if (M <= 128) return 128;
  return 256;
}

// Each wave's (M <= 64) or block's slice of K has to be whole k-steps: the
// kernels read whole steps, past the rows' ends otherwise.
static void check_split(int64_t K, int64_t splitk, int Mp) {
  const int64_t part = Mp > 64 ? splitk * 64 : splitk * SGWAVES * 32;
  TORCH_CHECK(splitk >= 1 && K % part == 0, "K must split evenly: K=", K,
              " splitk=", splitk);
}

void skinny_gemm(torch::Tensor out, torch::Tensor x, torch::Tensor w,
                 torch::Tensor work, int64_t splitk) {
  // out[M,N] = x[M,K] @ w[N,K]^T ; work: fp32 scratch >= splitk*Mp*N
  TORCH_CHECK(x.is_contiguous() && w.is_contiguous() && out.is_contiguous());
  TORCH_CHECK(x.scalar_type() == torch::kBFloat16);
  const int M = x.size(0), K = x.size(1), N = w.size(0);
  const int Mp = pad_m(M);
  TORCH_CHECK(M <= 256, "skinny_gemm is for decode batches <= 256");
  TORCH_CHECK(N % BN == 0, "N must be a multiple of 64");
  TORCH_CHECK(K % (64 * splitk * SGWAVES) == 0 || K % (32 * splitk * SGWAVES) == 0,
              "K must split evenly: K=", K, " splitk=", splitk);
  TORCH_CHECK(splitk == 1 || work.numel() >= splitk * (int64_t)Mp * N,
              "workspace too small");
  hipStream_t s = at::hip::getCurrentHIPStream().stream();
  launch_skinny(work, out, x, w, splitk, Mp, s, splitk == 1 ? 1 : 0);
  if (splitk > 1) {
    const int64_t total = (int64_t)M * N;
    const int blocks = (int)std::min<int64_t>((total + 255) / 256, 2048);
    hipLaunchKernelGGL(reduce_slabs_kernel, dim3(blocks), dim3(256), 0, s,
                       (__hip_bfloat16*)out.data_ptr(),
                       (const float*)work.data_ptr(), M, N, Mp, (int)splitk);
  }
  HIP_CHECK_LAST();
}

void skinny_gemm_slabs(torch::Tensor x, torch::Tensor w, torch::Tensor work,
                       int64_t splitk) {
  // slab-only launch: the consumer kernel fuses the split-K reduce
  const int M = x.size(0), N = w.size(0);
  const int Mp = pad_m(M);
  check_split(x.size(1), splitk, Mp);
  TORCH_CHECK(work.numel() >= splitk * (int64_t)Mp * N, "workspace too small");
  hipStream_t s = at::hip::getCurrentHIPStream().stream();
  auto dummy_out = work;  // unused when direct=0
  launch_skinny(work, x /*placeholder bf16 tensor, unused*/, x, w, splitk, Mp,
                s, /*direct=*/0);
  HIP_CHECK_LAST();
}

void skinny_gemm_silu(torch::Tensor out, torch::Tensor x, torch::Tensor w,
                      torch::Tensor work, int64_t splitk) {
  // fused SiLU-MLP front half: out[M,F] = silu(x@Wg^T) * (x@Wu^T) where
  // w is [2F, K] = [gate rows | up rows]
  TORCH_CHECK(x.is_contiguous() && w.is_contiguous() && out.is_contiguous());
  const int M = x.size(0), K = x.size(1), N = w.size(0);
  const int F = N / 2;
  const int Mp = pad_m(M);
  check_split(K, splitk, Mp);
  TORCH_CHECK(out.size(1) == F);
  TORCH_CHECK(work.numel() >= splitk * (int64_t)Mp * N, "workspace too small");
  hipStream_t s = at::hip::getCurrentHIPStream().stream();
  // the silu epilogue mixes gate and up columns, so it always reads slabs
  launch_skinny(work, out, x, w, splitk, Mp, s, /*direct=*/0);
  const int64_t total = (int64_t)M * F;
  const int blocks = (int)std::min<int64_t>((total + 255) / 256, 2048);
  hipLaunchKernelGGL(reduce_slabs_silu_kernel, dim3(blocks), dim3(256), 0, s,
                     (__hip_bfloat16*)out.data_ptr(),
                     (const float*)work.data_ptr(), M, F, Mp, (int)splitk);
  HIP_CHECK_LAST();
}
