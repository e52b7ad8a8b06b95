// Python bindings for the calfkit_amd CDNA4 kernel set (gfx950 only).

#include <torch/extension.h>

void rmsnorm(torch::Tensor out, torch::Tensor inp, torch::Tensor weight, double eps);
void fused_add_rmsnorm(torch::Tensor hidden, torch::Tensor residual,
                       torch::Tensor weight, double eps);
void silu_mul(torch::Tensor out, torch::Tensor gateup);
void rope_qk(torch::Tensor q, torch::Tensor k, torch::Tensor cos_sin,
             torch::Tensor positions);
void rope_qkv_write(torch::Tensor qkv, torch::Tensor kcache,
                    torch::Tensor vcache, torch::Tensor cos_sin,
                    torch::Tensor positions, torch::Tensor slots,
                    int64_t hq, int64_t hkv);
void rope_qkv_write_slab(torch::Tensor qkv, torch::Tensor work,
                         torch::Tensor kcache, torch::Tensor vcache,
                         torch::Tensor cos_sin, torch::Tensor positions,
                         torch::Tensor slots, int64_t hq, int64_t hkv,
                         int64_t Mp, int64_t splitk);
void fused_add_rmsnorm_slab(torch::Tensor hidden, torch::Tensor residual,
                            torch::Tensor work, torch::Tensor weight,
                            double eps, int64_t Mp, int64_t splitk);
void skinny_gemm_slabs(torch::Tensor x, torch::Tensor w, torch::Tensor work,
                       int64_t splitk);
void kv_write(torch::Tensor kcache, torch::Tensor vcache, torch::Tensor k,
              torch::Tensor v, torch::Tensor slots);
void attn_decode(torch::Tensor out, torch::Tensor q, torch::Tensor kcache,
                 torch::Tensor vcache, torch::Tensor page_table,
                 torch::Tensor seq_lens, double scale);
void attn_prefill(torch::Tensor out, torch::Tensor q, torch::Tensor k,
                  torch::Tensor v, double scale, int64_t past_len);
void attn_prefill_varlen(torch::Tensor out, torch::Tensor q, torch::Tensor k,
                         torch::Tensor v, torch::Tensor block_map,
                         torch::Tensor q_starts, torch::Tensor kv_starts,
                         torch::Tensor past_lens, double scale);
void rope_qkv_write_fp8(torch::Tensor qkv, torch::Tensor kcache,
                        torch::Tensor vcache, torch::Tensor kscale,
                        torch::Tensor vscale, torch::Tensor cos_sin,
                        torch::Tensor positions, torch::Tensor slots,
                        int64_t hq, int64_t hkv,
                        c10::optional<torch::Tensor> q_out);
void rope_qkv_write_slab_fp8(torch::Tensor qkv, torch::Tensor work,
                             torch::Tensor kcache, torch::Tensor vcache,
                             torch::Tensor kscale, torch::Tensor vscale,
                             torch::Tensor cos_sin, torch::Tensor positions,
                             torch::Tensor slots, int64_t hq, int64_t hkv,
                             int64_t Mp, int64_t splitk);
void kv_write_fp8(torch::Tensor kcache, torch::Tensor vcache,
                  torch::Tensor kscale, torch::Tensor vscale, torch::Tensor k,
                  torch::Tensor v, torch::Tensor slots);
void kv_read_fp8(torch::Tensor k, torch::Tensor v, torch::Tensor kcache,
                 torch::Tensor vcache, torch::Tensor kscale,
                 torch::Tensor vscale, torch::Tensor slots);
void attn_decode_fp8(torch::Tensor out, torch::Tensor q, torch::Tensor kcache,
                     torch::Tensor vcache, torch::Tensor kscale,
                     torch::Tensor vscale, torch::Tensor page_table,
                     torch::Tensor seq_lens, double scale);
void attn_decode_shared(torch::Tensor out, torch::Tensor q,
                        torch::Tensor kcache, torch::Tensor vcache,
                        torch::Tensor page_table, torch::Tensor seq_lens,
                        torch::Tensor group, torch::Tensor group_lens,
                        double scale, c10::optional<torch::Tensor> kscale,
                        c10::optional<torch::Tensor> vscale);
void sample(torch::Tensor out, torch::Tensor logits, torch::Tensor temperature,
            torch::Tensor seed_step, torch::Tensor topk, torch::Tensor cand,
            torch::Tensor row_seeds);
void sample_filtered(torch::Tensor out, torch::Tensor logits,
                     torch::Tensor temperature, torch::Tensor top_k,
                     torch::Tensor top_p, torch::Tensor min_p,
                     torch::Tensor uniform,
                     c10::optional<torch::Tensor> kept);
void skinny_gemm(torch::Tensor out, torch::Tensor x, torch::Tensor w,
                 torch::Tensor work, int64_t splitk);
void skinny_gemm_silu(torch::Tensor out, torch::Tensor x, torch::Tensor w,
                      torch::Tensor work, int64_t splitk);
void moe_gateup_silu(torch::Tensor act, torch::Tensor x, torch::Tensor w,
                     torch::Tensor tok, torch::Tensor off, torch::Tensor work);
void moe_down(torch::Tensor y, torch::Tensor act, torch::Tensor w,
              torch::Tensor off, torch::Tensor scale);
void moe_route(torch::Tensor tok, torch::Tensor off, torch::Tensor scale,
               torch::Tensor inv, torch::Tensor logits, int64_t topk);
void moe_combine(torch::Tensor out, torch::Tensor y, torch::Tensor inv,
                 int64_t topk);
std::vector<std::tuple<int64_t, double>> hipblaslt_algo_bench(
    torch::Tensor out, torch::Tensor x, torch::Tensor w, int64_t iters,
    int64_t max_algos);
void hipblaslt_gemm_indexed(torch::Tensor out, torch::Tensor x,
                            torch::Tensor w, int64_t algo_index,
                            torch::Tensor workspace);
void tile_gemm(torch::Tensor out, torch::Tensor x, torch::Tensor w,
               torch::Tensor work, int64_t bn, int64_t splitk);
void grammar_bias(torch::Tensor logits, torch::Tensor prev,
                  torch::Tensor gstate, torch::Tensor trigger,
                  torch::Tensor names, torch::Tensor pos,
                  torch::Tensor ncalls);
void tile_gemm_small(torch::Tensor out, torch::Tensor x, torch::Tensor w);
void tile_gemm_slabs(torch::Tensor x, torch::Tensor w, torch::Tensor work,
                     int64_t bn, int64_t splitk);

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("rmsnorm", &rmsnorm, "RMSNorm (bf16)");
  m.def("fused_add_rmsnorm", &fused_add_rmsnorm,
        "residual += hidden; hidden = rmsnorm(residual)");
  m.def("silu_mul", &silu_mul, "silu(gate) * up from packed [T,2F]");
  m.def("rope_qk", &rope_qk, "in-place neox RoPE on Q and K");
  m.def("rope_qkv_write", &rope_qkv_write,
        "fused QKV epilogue: in-place RoPE + paged-cache K/V scatter");
  m.def("rope_qkv_write_slab", &rope_qkv_write_slab,
        "split-K reduce + RoPE + cache scatter in one launch");
  m.def("fused_add_rmsnorm_slab", &fused_add_rmsnorm_slab,
        "split-K reduce + residual add + RMSNorm in one launch");
  m.def("skinny_gemm_slabs", &skinny_gemm_slabs,
        "skinny GEMM, slabs only (consumer fuses the reduce)");
  m.def("kv_write", &kv_write, "scatter K/V rows into the paged cache");
  m.def("attn_decode", &attn_decode, "paged GQA decode attention");
  m.def("attn_prefill", &attn_prefill, "causal GQA prefill attention (MFMA)");
  m.def("attn_prefill_varlen", &attn_prefill_varlen,
        "packed varlen causal GQA prefill attention (MFMA)");
  m.def("rope_qkv_write_fp8", &rope_qkv_write_fp8,
        "fused QKV epilogue: RoPE + e4m3 quantised paged-cache write");
  m.def("rope_qkv_write_slab_fp8", &rope_qkv_write_slab_fp8,
        "split-K reduce + RoPE + e4m3 quantised cache write in one launch");
  m.def("kv_write_fp8", &kv_write_fp8,
        "quantise K/V rows into the e4m3 paged cache");
  m.def("kv_read_fp8", &kv_read_fp8,
        "read rows of the e4m3 paged cache back as bf16");
  m.def("attn_decode_fp8", &attn_decode_fp8,
        "paged GQA decode attention over the e4m3 cache");
  m.def("attn_decode_shared", &attn_decode_shared,
        "paged GQA decode attention, shared prefixes computed once");
  m.def("sample", &sample, "Gumbel-max token sampling");
  m.def("sample_filtered", &sample_filtered,
        "temperature, top-k, top-p and min-p draw from given random numbers");
  m.def("skinny_gemm", &skinny_gemm,
        "decode projection GEMM: out = x @ w^T, w stored [N,K]");
  m.def("skinny_gemm_silu", &skinny_gemm_silu,
        "fused SiLU-MLP gate: out = silu(x@Wg^T) * (x@Wu^T)");
  m.def("moe_gateup_silu", &moe_gateup_silu,
        "grouped MoE gate-up: act[r] = silu/mul of x[tok[r]] @ W[e(r)]^T");
  m.def("moe_down", &moe_down,
        "grouped MoE down: y[r] = scale[r] * act[r] @ W[e(r)]^T");
  m.def("moe_route", &moe_route,
        "fused router: softmax -> top-K -> renorm -> stable expert buckets");
  m.def("moe_combine", &moe_combine,
        "out[t] = sum_j y[inv[t*K+j]] (deterministic scatter-combine)");
  m.def("hipblaslt_algo_bench", &hipblaslt_algo_bench,
        "time every supported hipBLASLt algo for out = x @ w^T");
  m.def("hipblaslt_gemm_indexed", &hipblaslt_gemm_indexed,
        "run out = x @ w^T with a searched hipBLASLt algo index");
  m.def("tile_gemm", &tile_gemm,
        "tiled MFMA GEMM for serving batches (M 65..512+), split-K reduce");
  m.def("tile_gemm_small", &tile_gemm_small,
        "64x128-tile MFMA GEMM, natural fill for M=384/512 projections");
  m.def("tile_gemm_slabs", &tile_gemm_slabs,
        "tiled MFMA GEMM, fp32 slabs only (consumer fuses the reduce)");
  m.def("grammar_bias", &grammar_bias,
        "tool-call grammar constrained-sampling bias (in-place on logits)");
}
