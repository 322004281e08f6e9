// Gated expert products of a mixture of experts: the first half of an expert's feed-forward network, activation and gate
// included (epilogue.cuh).  The main loops are those of the fused-MoE A8W8 GEMM (a8w8_kernels.cuh).
#include "a8w8_kernels.cuh"

namespace fnn {
namespace {

template <typename OutT>
int dispatch_moe_gated(const int8_t* a_sorted, int64_t EM, const int8_t* b, int64_t E, const A8W8Params& p, const FusedEpilogue<true>& fx,
                       cudaStream_t st) {
  // the rule of the plain expert products on the accumulator columns: the widest tile that still gives every SM work
  const int sms = sm_count();
  const int64_t cols = 2 * int64_t(p.N);
  if (p.block_m % 256 == 0 && (EM / 256) * ((cols + 255) / 256) >= sms / 2) return launch_moe_pair<OutT, 8>(a_sorted, EM, b, E, p, st, fx);
  // Small blocks: with more than one block for many experts, runs of an expert's blocks make a tile, so that its weights are
  // read once (64 tokens, two of eight experts each, 28672 x 4096 weights an expert, blocks of 16: 191 us with a tile per block,
  // 155 us; 512 tokens 652 -> 186 us).  The distribution over the experts is on the device, so the rule goes by the mean.
  // The list of runs lies in shared memory and ends at kMaxRuns blocks; a longer slot list has a tile per block, whose weights are read
  // again for each: 8132 tokens (1024 blocks of 16) 1446 us, 8140 tokens (1025) 11881; blocks of 64 or 256 take 1773 and 1546.
  const int64_t mean = p.num_valid / E;
  const int64_t used = p.num_valid < E ? p.num_valid : E;
  if (p.block_m <= 64 && fx.blocks <= kMaxRuns && mean * 5 >= p.block_m * 3) {
    const int rows = (mean > 48 || p.block_m > 32) ? kBM : 64;
    const int64_t runs = used * ((mean + rows - 1) / rows);
    if (runs * ((cols + 255) / 256) >= sms) return launch_moe_runs<OutT, 256>(a_sorted, EM, b, E, p, rows, st, fx);
    if (runs * ((cols + 127) / 128) >= sms) return launch_moe_runs<OutT, 128>(a_sorted, EM, b, E, p, rows, st, fx);
    return launch_moe_runs<OutT, 64>(a_sorted, EM, b, E, p, rows, st, fx);
  }
  const int64_t tiles_m = EM / p.tile_rows;
  if (tiles_m * ((cols + 255) / 256) >= sms) return launch_moe_rows<OutT, 256>(a_sorted, EM, b, E, p, st, fx);
  if (tiles_m * ((cols + 127) / 128) >= sms) return launch_moe_rows<OutT, 128>(a_sorted, EM, b, E, p, st, fx);
  return launch_moe_rows<OutT, 64>(a_sorted, EM, b, E, p, st, fx);
}

}  // namespace
}  // namespace fnn

extern "C" int fnn_fused_moe_a8w8_gated(const int8_t* a, int64_t lda, const int8_t* b, int64_t E, int64_t N, int64_t K,
                                        const void* alpha_row, int row_dtype, const void* alpha_col, int col_dtype, const void* bias,
                                        int bias_dtype, int activation, const int32_t* sorted_token_ids, int64_t EM,
                                        const int32_t* expert_ids, const int32_t* num_tokens_post_padded, int64_t num_valid_tokens,
                                        int top_k, int block_m, void* out, int out_dtype, int64_t ldo, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  using namespace fnn;
  if (E <= 0 || N < 0 || K <= 0 || EM < 0 || lda < K || ldo < N || num_valid_tokens < 0 || top_k <= 0 || block_m <= 0)
    return fail(FNN_ERR_SHAPE, "fused_moe_a8w8_gated: E=%lld N=%lld K=%lld EM=%lld lda=%lld ldo=%lld top_k=%d block_m=%d", (long long)E,
                (long long)N, (long long)K, (long long)EM, (long long)lda, (long long)ldo, top_k, block_m);
  if (N > INT32_MAX / 2 || E > INT32_MAX || 2 * E * N > INT32_MAX || K > INT32_MAX || EM > INT32_MAX || num_valid_tokens > INT32_MAX)
    return fail(FNN_ERR_SHAPE, "fused_moe_a8w8_gated: sizes must be below 2^31 (all experts' weight rows together included)");
  if (EM % block_m != 0) return fail(FNN_ERR_SHAPE, "fused_moe_a8w8_gated: %lld sorted slots are not a multiple of block_m=%d", (long long)EM, block_m);
  if (block_m > kBM && block_m % kBM != 0)
    return fail(FNN_ERR_UNSUPPORTED, "fused_moe_a8w8_gated: block_m must be at most %d or a multiple of it (got %d)", kBM, block_m);
  if (out_dtype != FNN_F16 && out_dtype != FNN_BF16) return fail(FNN_ERR_DTYPE, "fused_moe_a8w8_gated: output must be f16 or bf16");
  if (row_dtype < FNN_F16 || row_dtype > FNN_F32 || col_dtype < FNN_F16 || col_dtype > FNN_F32)
    return fail(FNN_ERR_DTYPE, "fused_moe_a8w8_gated: scales must be f16, bf16 or f32");
  if (bias && (bias_dtype < FNN_F16 || bias_dtype > FNN_F32)) return fail(FNN_ERR_DTYPE, "fused_moe_a8w8_gated: the bias must be f16, bf16 or f32");
  if (activation < FNN_ACT_NONE || activation > FNN_ACT_GELU_TANH)
    return fail(FNN_ERR_UNSUPPORTED, "fused_moe_a8w8_gated: unknown activation code %d", activation);
  if (EM == 0 || N == 0 || num_valid_tokens == 0) return FNN_OK;
  if (!a || !b || !alpha_row || !alpha_col || !sorted_token_ids || !expert_ids || !num_tokens_post_padded || !out)
    return fail(FNN_ERR_NULL_POINTER, "fused_moe_a8w8_gated: null tensor pointer");
  if (K % 16 != 0 || reinterpret_cast<uintptr_t>(a) % 16 != 0 || lda % 16 != 0 || reinterpret_cast<uintptr_t>(b) % 16 != 0)
    return fail(FNN_ERR_ALIGNMENT, "fused_moe_a8w8_gated: K and lda must be multiples of 16 and the operands 16-byte aligned");
  const size_t need = fnn_fused_moe_a8w8_workspace_bytes(EM, K);
  if (!workspace || workspace_bytes < need) return fail(FNN_ERR_WORKSPACE, "fused_moe_a8w8_gated: needs %zu bytes of workspace, got %zu", need, workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return fail(FNN_ERR_ALIGNMENT, "fused_moe_a8w8_gated: workspace must be 256-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int8_t* a_sorted = static_cast<int8_t*>(workspace);
  moe_gather_rows_kernel<<<unsigned((EM + 7) / 8), 256, 0, st>>>(a, lda, sorted_token_ids, num_tokens_post_padded, int(num_valid_tokens),
                                                                 top_k, a_sorted, int(K), int(EM));
  if (int e = check_cuda(cudaGetLastError(), "fused moe gather launch")) return e;
  A8W8Params p{};
  p.alpha_row = alpha_row; p.alpha_col = alpha_col; p.out = out; p.acc_out = nullptr;
  p.ldo = ldo; p.ldacc = 0; p.row_dtype = row_dtype; p.col_dtype = col_dtype;
  p.M = int(num_valid_tokens); p.N = int(N); p.K = int(K);
  p.status = device_status_word();
  p.wait_ns = kWaitLimitNs; p.skip_kb = -1;
  p.sorted_ids = sorted_token_ids; p.expert_ids = expert_ids; p.num_post_padded = num_tokens_post_padded;
  p.topk_w = nullptr; p.topk_w_dtype = FNN_F32; p.top_k = top_k; p.block_m = block_m;
  p.tile_rows = block_m < kBM ? block_m : kBM; p.num_valid = int(num_valid_tokens); p.mul_w = 0;
  p.col_stride_e = 2 * N;
  FusedEpilogue<true> fx;
  fx.bias = bias; fx.residual = nullptr; fx.ldr = 0; fx.bias_dtype = bias_dtype; fx.act = activation; fx.rows = int(2 * N); fx.experts = int(E); fx.blocks = int(EM / block_m);
  if (out_dtype == FNN_F16) return dispatch_moe_gated<__half>(a_sorted, EM, b, E, p, fx, st);
  return dispatch_moe_gated<__nv_bfloat16>(a_sorted, EM, b, E, p, fx, st);
}
