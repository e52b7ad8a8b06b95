// e4m3 KV cache for MI355X (gfx950): quantise as the cache is written, and
// read rows back.
//
// One row = the 128 values of one (token, KV head).  Its scale is a power of
// two, 2^e, held as the byte e + 127:
//   a = largest finite |r_i|,  e = least integer with a * 2^-e <= 448
//   (448 = e4m3fn's largest value),  c_i = e4m3fn(r_i * 2^-e), half to even.
// A power of two costs no precision (e4m3 is a floating type: only the few
// values 2^-15 below the row's largest meet its subnormals), makes r_i * 2^-e
// and the read-back c_i * 2^e exact, so that the bytes are a function of the
// row alone, and takes one byte where a float scale takes four.  NaN and
// infinities are stored as NaN (e4m3fn has no infinity) and do not enter a.
//
// Layout: codes [P, Hkv, 64, 128] as the bf16 cache, scales [P, Hkv, 64], so
// that one (page, head) panel of scales is one 64 B line.
//
// Bound: bytes.  A row is 8 lanes x (8 low + 8 high) values: both halves of
// the rotation pair (i, i + 64) sit in one lane as one 16 B load each, the
// largest value takes three lane swaps, and a wave handles 8 rows.  Measured,
// rotate and write then read back, 32/8 heads: 12288 tokens 72.4 us, 4.96 TB/s,
// the rate of a large copy (4.94); 512 tokens 8.0 us and one token 4.6 us on
// the GPU, 4.6 us a call on the host.  From split-K slabs, again and again: 4
// slabs of 1, 8 and 64 tokens 3.5, 3.7 and 4.0 us, 2 of 512 tokens 5.8 (into the
// bf16 cache 2.8, 2.8, 3.2, 8.0); kv_write_fp8 of 1, 512 and 12288 tokens 2.5,
// 3.1 and 15.1 us.

#include "common.h"
#include "fp8.h"

#define HD 128
#define KVPAGE 64
#define ROW_LANES 8

// x (16 values of a row's lane: low 8 then high 8) -> codes of the low 8 and
// the high 8; returns the scale byte, the same in all 8 lanes of the row.
__device__ __forceinline__ int quantise_row(const float (&x)[16], uint2& lo,
                                            uint2& hi) {
  float a = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float m = fabsf(x[j]);
    a = (m < INFINITY) ? fmaxf(a, m) : a;  // false for NaN too
  }
#pragma unroll
  for (int off = 1; off < ROW_LANES; off <<= 1)
    a = fmaxf(a, __shfl_xor(a, off, WAVE));
  const int e = e4m3_row_exponent(a);
  float y[16];
#pragma unroll
  for (int j = 0; j < 16; ++j)
    y[j] = (fabsf(x[j]) < INFINITY) ? ldexpf(x[j], -e) : NAN;
  lo = make_uint2(pack_e4m3(y[0], y[1], y[2], y[3]),
                  pack_e4m3(y[4], y[5], y[6], y[7]));
  hi = make_uint2(pack_e4m3(y[8], y[9], y[10], y[11]),
                  pack_e4m3(y[12], y[13], y[14], y[15]));
  return e + 127;
}

__device__ __forceinline__ void store_row(uint8_t* codes, uint8_t* scales,
                                          const int64_t row, const int l8,
                                          const float (&x)[16]) {
  uint2 lo, hi;
  const int byte = quantise_row(x, lo, hi);
  uint8_t* c = codes + row * HD;
  *reinterpret_cast<uint2*>(c + l8 * 8) = lo;
  *reinterpret_cast<uint2*>(c + HD / 2 + l8 * 8) = hi;
  if (l8 == 0) scales[row] = (uint8_t)byte;
}

__device__ __forceinline__ void unpack8(const bf16x8& v, float* x) {
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = bf2f(v.v[j]);
}

__device__ __forceinline__ bf16x8 pack8(const float* x) {
  bf16x8 v;
#pragma unroll
  for (int j = 0; j < 8; ++j) v.v[j] = f2bf(x[j]);
  return v;
}

// --------------------------------------------------------- rope + write

// Job = (token, head) of the packed row: heads [0, hq) are queries (rotated),
// [hq, hq + hkv) keys (rotated, then quantised), the rest values (quantised).
//
// SLAB: the row is the sum of splitk fp32 slabs (the projection's split-K
// reduce rides here) and is written whole into qkv.  Otherwise the rotated
// heads go back in place, or, with q_out, the queries go there and qkv stays
// as it was.  The rotated values are rounded to bf16 before they are
// quantised: the cache holds the packed row's own values in fewer bits, the
// ones a prefill's attention reads.
template <bool SLAB>
__global__ __launch_bounds__(256) void rope_qkv_write_fp8_kernel(
    __hip_bfloat16* __restrict__ qkv,  // [T, (hq + 2 hkv) * 128]
    __hip_bfloat16* __restrict__ q_out,  // [T, hq, 128] or null
    const float* __restrict__ work,      // SLAB: [splitk, Mp, W]
    uint8_t* __restrict__ kcache, uint8_t* __restrict__ vcache,
    uint8_t* __restrict__ kscale, uint8_t* __restrict__ vscale,
    const float* __restrict__ cos_sin, const int32_t* __restrict__ positions,
    const int32_t* __restrict__ slots, const int64_t T, const int hq,
    const int hkv, const int max_pos, const int64_t nslots, const int Mp,
    const int splitk) {
// the rotation rounds each product, as the formula's separate operations do
#pragma clang fp contract(off)
  const int heads = hq + 2 * hkv;
  const int64_t job =
      ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / ROW_LANES;
  if (job >= T * heads) return;  // whole rows leave: lane swaps stay inside
  const int l8 = threadIdx.x % ROW_LANES;
  const int64_t token = job / heads;
  const int head = (int)(job - token * heads);
  const int64_t W = (int64_t)heads * HD;
  __hip_bfloat16* base = qkv + token * W + head * HD;

  float x[16];
  if constexpr (SLAB) {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = 0.f;
    for (int sk = 0; sk < splitk; ++sk) {
      const float* s = work + ((int64_t)sk * Mp + token) * W + head * HD;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] += s[l8 * 8 + j];
        x[8 + j] += s[HD / 2 + l8 * 8 + j];
      }
    }
  } else {
    unpack8(reinterpret_cast<const bf16x8*>(base)[l8], x);
    unpack8(reinterpret_cast<const bf16x8*>(base + HD / 2)[l8], x + 8);
  }
  if (head < hq + hkv) {
    const int pos = min(max(positions[token], 0), max_pos - 1);
    const float* cs = cos_sin + (int64_t)pos * HD + l8 * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float c = cs[j], sn = cs[HD / 2 + j];
      const float r0 = x[j] * c - x[8 + j] * sn;
      const float r1 = x[8 + j] * c + x[j] * sn;
      x[j] = r0;
      x[8 + j] = r1;
    }
  }
  const bf16x8 lo = pack8(x), hi = pack8(x + 8);
  __hip_bfloat16* dst = nullptr;
  if (SLAB || (q_out == nullptr && head < hq + hkv)) dst = base;
  if (q_out != nullptr && head < hq) dst = q_out + (token * hq + head) * HD;
  if (dst != nullptr) {
    reinterpret_cast<bf16x8*>(dst)[l8] = lo;
    reinterpret_cast<bf16x8*>(dst + HD / 2)[l8] = hi;
  }
  if (head < hq) return;
  const int64_t slot = slots[token];
  if (slot < 0 || slot >= nslots) return;  // padding
  const bool is_k = head < hq + hkv;
  const int h = is_k ? head - hq : head - hq - hkv;
  unpack8(lo, x);
  unpack8(hi, x + 8);
  store_row(is_k ? kcache : vcache, is_k ? kscale : vscale,
            (slot / KVPAGE * hkv + h) * KVPAGE + slot % KVPAGE, l8, x);
}

// ------------------------------------------------------- write and read

__global__ __launch_bounds__(256) void kv_write_fp8_kernel(
    uint8_t* __restrict__ kcache, uint8_t* __restrict__ vcache,
    uint8_t* __restrict__ kscale, uint8_t* __restrict__ vscale,
    const __hip_bfloat16* __restrict__ k, const __hip_bfloat16* __restrict__ v,
    const int32_t* __restrict__ slots, const int64_t T, const int hkv,
    const int64_t kstride, const int64_t vstride, const int64_t nslots) {
  const int64_t job =
      ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / ROW_LANES;
  if (job >= T * 2 * hkv) return;
  const int l8 = threadIdx.x % ROW_LANES;
  const int64_t token = job / (2 * hkv);
  const int head = (int)(job - token * 2 * hkv);
  const int64_t slot = slots[token];
  if (slot < 0 || slot >= nslots) return;
  const bool is_k = head < hkv;
  const int h = is_k ? head : head - hkv;
  const __hip_bfloat16* src =
      (is_k ? k + token * kstride : v + token * vstride) + h * HD;
  float x[16];
  unpack8(reinterpret_cast<const bf16x8*>(src)[l8], x);
  unpack8(reinterpret_cast<const bf16x8*>(src + HD / 2)[l8], x + 8);
  store_row(is_k ? kcache : vcache, is_k ? kscale : vscale,
            (slot / KVPAGE * hkv + h) * KVPAGE + slot % KVPAGE, l8, x);
}

// A row's 128 codes are 8 lanes x 16 B in, 2 x 16 B out.
__global__ __launch_bounds__(256) void kv_read_fp8_kernel(
    __hip_bfloat16* __restrict__ k, __hip_bfloat16* __restrict__ v,
    const uint8_t* __restrict__ kcache, const uint8_t* __restrict__ vcache,
    const uint8_t* __restrict__ kscale, const uint8_t* __restrict__ vscale,
    const int32_t* __restrict__ slots, const int64_t T, const int hkv,
    const int64_t kstride, const int64_t vstride, const int64_t nslots) {
  const int64_t job =
      ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / ROW_LANES;
  if (job >= T * 2 * hkv) return;
  const int l8 = threadIdx.x % ROW_LANES;
  const int64_t token = job / (2 * hkv);
  const int head = (int)(job - token * 2 * hkv);
  const int64_t slot = slots[token];
  if (slot < 0 || slot >= nslots) return;  // the row stays as it was
  const bool is_k = head < hkv;
  const int h = is_k ? head : head - hkv;
  const int64_t row = (slot / KVPAGE * hkv + h) * KVPAGE + slot % KVPAGE;
  const uint4 c =
      reinterpret_cast<const uint4*>((is_k ? kcache : vcache) + row * HD)[l8];
  const float s = e8m0_scale((is_k ? kscale : vscale)[row]);
  uint4* dst = reinterpret_cast<uint4*>(
      (is_k ? k + token * kstride : v + token * vstride) + h * HD);
  dst[l8 * 2] = make_uint4(e4m3_to_bf16x2<false>(c.x, s),
                           e4m3_to_bf16x2<true>(c.x, s),
                           e4m3_to_bf16x2<false>(c.y, s),
                           e4m3_to_bf16x2<true>(c.y, s));
  dst[l8 * 2 + 1] = make_uint4(e4m3_to_bf16x2<false>(c.z, s),
                               e4m3_to_bf16x2<true>(c.z, s),
                               e4m3_to_bf16x2<false>(c.w, s),
                               e4m3_to_bf16x2<true>(c.w, s));
}

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

namespace {

void check_rows(const torch::Tensor& t, const char* name, int64_t T,
                int64_t hkv, const torch::Device dev) {
  TORCH_CHECK(t.device() == dev, name, " is on another device");
  TORCH_CHECK(t.scalar_type() == torch::kBFloat16, name, " must be bf16");
  TORCH_CHECK(t.dim() == 3 && t.size(0) == T && t.size(1) == hkv &&
                  t.size(2) == HD,
              name, " must be [T, Hkv, 128]");
  TORCH_CHECK(T == 0 || (t.stride(2) == 1 && (hkv == 1 || t.stride(1) == HD)),
              name, " heads must be contiguous");
  TORCH_CHECK(T <= 1 || t.stride(0) % 8 == 0, name,
              " rows must start on 16 bytes");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name,
              " must start on 16 bytes");
}

void check_index(const torch::Tensor& t, const char* name, int64_t T,
                 const torch::Device dev) {
  TORCH_CHECK(t.device() == dev, name, " is on another device");
  TORCH_CHECK(t.scalar_type() == torch::kInt32, name, " must be int32");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == T && t.is_contiguous(), name,
              " must be a contiguous [T]");
}

unsigned blocks_for(int64_t jobs) {
  const int64_t n = (jobs * ROW_LANES + 255) / 256;
  TORCH_CHECK(n <= 0x7fffffff, "too many rows for one launch");
  return (unsigned)n;
}

void launch_rope(torch::Tensor& qkv, const torch::Tensor* work,
                 torch::Tensor& kcache, torch::Tensor& vcache,
                 torch::Tensor& kscale, torch::Tensor& vscale,
                 torch::Tensor& cos_sin, torch::Tensor& positions,
                 torch::Tensor& slots, int64_t hq, int64_t hkv,
                 const c10::optional<torch::Tensor>& q_out, int64_t Mp,
                 int64_t splitk) {
  const auto dev = qkv.device();
  check_fp8_cache(kcache, vcache, kscale, vscale, dev);
  const int64_t T = qkv.size(0);
  TORCH_CHECK(hq > 0 && hkv == kcache.size(1),
              "hkv does not match the cache");
  TORCH_CHECK(qkv.scalar_type() == torch::kBFloat16 && qkv.dim() == 2 &&
                  qkv.is_contiguous() && qkv.size(1) == (hq + 2 * hkv) * HD,
              "qkv must be a contiguous bf16 [T, (hq + 2 hkv) * 128]");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0,
              "qkv must start on 16 bytes");
  TORCH_CHECK(cos_sin.device() == dev &&
                  cos_sin.scalar_type() == torch::kFloat32 &&
                  cos_sin.dim() == 2 && cos_sin.size(1) == HD &&
                  cos_sin.size(0) > 0 && cos_sin.is_contiguous(),
              "cos_sin must be a contiguous f32 [max_pos, 128]");
  check_index(positions, "positions", T, dev);
  check_index(slots, "slots", T, dev);
  void* qo = nullptr;
  if (q_out.has_value()) {
    TORCH_CHECK(q_out->device() == dev &&
                    q_out->scalar_type() == torch::kBFloat16 &&
                    q_out->dim() == 3 && q_out->size(0) == T &&
                    q_out->size(1) == hq && q_out->size(2) == HD &&
                    q_out->is_contiguous(),
                "q_out must be a contiguous bf16 [T, hq, 128]");
    TORCH_CHECK(reinterpret_cast<uintptr_t>(q_out->data_ptr()) % 16 == 0,
                "q_out must start on 16 bytes");
    qo = q_out->data_ptr();
  }
  if (work != nullptr) {
    TORCH_CHECK(work->device() == dev &&
                    work->scalar_type() == torch::kFloat32 &&
                    work->is_contiguous(),
                "work must be contiguous f32");
    TORCH_CHECK(splitk >= 1 && Mp >= T &&
                    work->numel() >= splitk * Mp * qkv.size(1),
                "work is too small for its slabs");
  }
  if (T == 0) return;
  c10::DeviceGuard guard(dev);
  hipStream_t s = at::hip::getCurrentHIPStream().stream();
#define LAUNCH(SLAB)                                                         \
  hipLaunchKernelGGL((rope_qkv_write_fp8_kernel<SLAB>),                      \
                     dim3(blocks_for(T * (hq + 2 * hkv))), dim3(256), 0, s,  \
                     (__hip_bfloat16*)qkv.data_ptr(), (__hip_bfloat16*)qo,   \
                     SLAB ? (const float*)work->data_ptr() : nullptr,        \
                     (uint8_t*)kcache.data_ptr(),                            \
                     (uint8_t*)vcache.data_ptr(),                            \
                     (uint8_t*)kscale.data_ptr(),                            \
                     (uint8_t*)vscale.data_ptr(),                            \
                     (const float*)cos_sin.data_ptr(),                       \
                     (const int32_t*)positions.data_ptr(),                   \
                     (const int32_t*)slots.data_ptr(), T, (int)hq, (int)hkv, \
                     (int)cos_sin.size(0), kcache.size(0) * KVPAGE, (int)Mp, \
                     (int)splitk)
  if (work != nullptr)
    LAUNCH(true);
  else
    LAUNCH(false);
#undef LAUNCH
  HIP_CHECK_LAST();
}

}  // namespace

void rope_qkv_write_fp8(torch::Tensor qkv, torch::Tensor kcache,
                        torch::Tensor vcache, torch::Tensor kscale,
                        torch::Tensor vscale, torch::Tensor cos_sin,
                        torch::Tensor positions, torch::Tensor slots,
                        int64_t hq, int64_t hkv,
                        c10::optional<torch::Tensor> q_out) {
  launch_rope(qkv, nullptr, kcache, vcache, kscale, vscale, cos_sin,
              positions, slots, hq, hkv, q_out, 0, 0);
}

void rope_qkv_write_slab_fp8(torch::Tensor qkv, torch::Tensor work,
                             torch::Tensor kcache, torch::Tensor vcache,
                             torch::Tensor kscale, torch::Tensor vscale,
                             torch::Tensor cos_sin, torch::Tensor positions,
                             torch::Tensor slots, int64_t hq, int64_t hkv,
                             int64_t Mp, int64_t splitk) {
  launch_rope(qkv, &work, kcache, vcache, kscale, vscale, cos_sin, positions,
              slots, hq, hkv, c10::nullopt, Mp, splitk);
}

void kv_write_fp8(torch::Tensor kcache, torch::Tensor vcache,
                  torch::Tensor kscale, torch::Tensor vscale, torch::Tensor k,
                  torch::Tensor v, torch::Tensor slots) {
  const auto dev = k.device();
  check_fp8_cache(kcache, vcache, kscale, vscale, dev);
  const int64_t T = k.size(0), hkv = kcache.size(1);
  check_rows(k, "k", T, hkv, dev);
  check_rows(v, "v", T, hkv, dev);
  check_index(slots, "slots", T, dev);
  if (T == 0) return;
  c10::DeviceGuard guard(dev);
  hipLaunchKernelGGL(
      kv_write_fp8_kernel, dim3(blocks_for(T * 2 * hkv)), dim3(256), 0,
      at::hip::getCurrentHIPStream().stream(), (uint8_t*)kcache.data_ptr(),
      (uint8_t*)vcache.data_ptr(), (uint8_t*)kscale.data_ptr(),
      (uint8_t*)vscale.data_ptr(), (const __hip_bfloat16*)k.data_ptr(),
      (const __hip_bfloat16*)v.data_ptr(), (const int32_t*)slots.data_ptr(),
      T, (int)hkv, k.stride(0), v.stride(0), kcache.size(0) * KVPAGE);
  HIP_CHECK_LAST();
}

void kv_read_fp8(torch::Tensor k, torch::Tensor v, torch::Tensor kcache,
                 torch::Tensor vcache, torch::Tensor kscale,
                 torch::Tensor vscale, torch::Tensor slots) {
  const auto dev = k.device();
  check_fp8_cache(kcache, vcache, kscale, vscale, dev);
  const int64_t T = slots.size(0), hkv = kcache.size(1);
  check_rows(k, "k", T, hkv, dev);
  check_rows(v, "v", T, hkv, dev);
  check_index(slots, "slots", T, dev);
  if (T == 0) return;
  c10::DeviceGuard guard(dev);
  hipLaunchKernelGGL(
      kv_read_fp8_kernel, dim3(blocks_for(T * 2 * hkv)), dim3(256), 0,
      at::hip::getCurrentHIPStream().stream(), (__hip_bfloat16*)k.data_ptr(),
      (__hip_bfloat16*)v.data_ptr(), (const uint8_t*)kcache.data_ptr(),
      (const uint8_t*)vcache.data_ptr(), (const uint8_t*)kscale.data_ptr(),
      (const uint8_t*)vscale.data_ptr(), (const int32_t*)slots.data_ptr(), T,
      (int)hkv, k.stride(0), v.stride(0), kcache.size(0) * KVPAGE);
  HIP_CHECK_LAST();
}
