// Entry points of the A8W8 GEMM and of the fused-MoE A8W8 GEMM: argument checks and the choice of kernel and tile.  The
// kernels are in a8w8_kernels.cuh.
#include "a8w8_kernels.cuh"
#include "weight_only.cuh"

namespace fnn {
namespace {

template <typename OutT>
int dispatch(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, const A8W8Params& p, cudaStream_t st,
             void* workspace, size_t workspace_bytes) {
  const bool tma_ok = p.K > 0 && (reinterpret_cast<uintptr_t>(a) % 16 == 0) && (reinterpret_cast<uintptr_t>(b) % 16 == 0) &&
                      (lda % 16 == 0) && (ldb % 16 == 0);
  if (!tma_ok) {
    const int64_t total = int64_t(p.M) * p.N;
    a8w8_generic_kernel<OutT><<<unsigned((total + 255) / 256), 256, 0, st>>>(a, lda, b, ldb, p);
    return check_cuda(cudaGetLastError(), "a8w8 generic launch");
  }
  // Up to 8 tokens: the weight stream is all that matters, and the per-lane streaming kernel of the weight-only
  // decode path moves it faster than tile copies do: 6-10 % on wide matrices, and 2-3x on narrow, long ones
  // (N = 1024 .. 4096 at K = 28672: 57 us -> 16 .. 33 us), where 64-column tiles leave most SMs without work while
  // the streaming kernel has a CTA per 16 channels.  It declines shapes it does not cover (K not a multiple of its
  // block, activations that do not fit its shared memory).
  if (p.M <= 8 && p.N >= 512 && opt_test_stall_us() == 0) {
    const int r = gemv_a8w8_imma(a, lda, b, ldb, p.alpha_row, p.row_dtype, p.alpha_col, p.col_dtype, p.out,
                                 std::is_same<OutT, __half>::value ? FNN_F16 : FNN_BF16, p.ldo, p.M, p.N, p.K, p.acc_out,
                                 p.ldacc, st);
    if (r >= 0) return r;
  }
  // the K-balanced mode needs scratch: without it (or with a misaligned one) the best whole-tile plan runs instead
  const bool ws_ok = workspace && workspace_bytes >= sk_workspace_bytes(sm_count()) && reinterpret_cast<uintptr_t>(workspace) % 256 == 0;
  A8W8Plan plan = opt_test_stall_us() != 0 ? A8W8Plan{false, 64, 0.0}
                                           : plan_a8w8(p.M, p.N, p.K, sm_count(), ws_ok ? opt_a8w8_balanced() : 2);
  if (const int forced = opt_a8w8_pair_tile()) {  // tuning hook: a given pair-tile width wherever the pair kernel can run
    if (p.M > kBM) plan = A8W8Plan{true, forced, 0.0};
  }
  if (plan.balanced) return launch_pair<OutT, 256, true>(a, lda, b, ldb, p, st, workspace);
  if (plan.pair && opt_a8w8_epilogue_warps() != 4) {
    // Eight epilogue warps per CTA (one output staging buffer each, so the operand ring keeps its depth).  With short K
    // a tile's MMAs take less time than four warps need to write it out: measured four -> eight warps, K = 1664
    // 2037 -> 3003 TOPS, 2048 2051 -> 2766, 3328 3273 -> 3344, 4096 3322 -> 3370, 8192 the same.
    switch (plan.bn) {
      case 256: return launch_pair<OutT, 256, false, 8>(a, lda, b, ldb, p, st);
      case 224: return launch_pair<OutT, 224, false, 8>(a, lda, b, ldb, p, st);
      case 192: return launch_pair<OutT, 192, false, 8>(a, lda, b, ldb, p, st);
      case 160: return launch_pair<OutT, 160, false, 8>(a, lda, b, ldb, p, st);
      default: return launch_pair<OutT, 128, false, 8>(a, lda, b, ldb, p, st);
    }
  }
  if (plan.pair) {
    switch (plan.bn) {
      case 256: return launch_pair<OutT, 256>(a, lda, b, ldb, p, st);
      case 224: return launch_pair<OutT, 224>(a, lda, b, ldb, p, st);
      case 192: return launch_pair<OutT, 192>(a, lda, b, ldb, p, st);
      case 160: return launch_pair<OutT, 160>(a, lda, b, ldb, p, st);
      default: return launch_pair<OutT, 128>(a, lda, b, ldb, p, st);
    }
  }
  if (plan.bn == 256) return launch_umma_rows<OutT, 256>(a, lda, b, ldb, p, st);
  if (plan.bn == 128) return launch_umma_rows<OutT, 128>(a, lda, b, ldb, p, st);
  return launch_umma_rows<OutT, 64>(a, lda, b, ldb, p, st);
}

template <typename OutT>
int dispatch_moe(const int8_t* a_sorted, int64_t EM, const int8_t* b, int64_t E, const A8W8Params& p, cudaStream_t st) {
  // the widest tile that still gives every SM work; small problems stream the expert weights with 64-wide tiles
  const int sms = sm_count();
  // blocks of 256 slots with enough tiles for every CTA pair: the CTA-pair kernel (a third less operand traffic per MMA)
  if (p.block_m % 256 == 0 && (EM / 256) * ((p.N + 255) / 256) >= sms / 2)
    return launch_moe_pair<OutT>(a_sorted, EM, b, E, p, st);
  const int64_t tiles_m = EM / p.tile_rows;
  if (tiles_m * ((p.N + 255) / 256) >= sms) return launch_moe_rows<OutT, 256>(a_sorted, EM, b, E, p, st);
  if (tiles_m * ((p.N + 127) / 128) >= sms) return launch_moe_rows<OutT, 128>(a_sorted, EM, b, E, p, st);
  return launch_moe_rows<OutT, 64>(a_sorted, EM, b, E, p, st);
}

}  // namespace
}  // namespace fnn

extern "C" size_t fnn_fused_moe_a8w8_workspace_bytes(int64_t EM, int64_t K) {
  if (EM <= 0 || K <= 0) return 0;
  return (size_t(EM) * size_t(K) + 255) / 256 * 256;  // the expert-sorted copy of the token rows
}

extern "C" int fnn_fused_moe_a8w8(const int8_t* a, int64_t lda, const int8_t* b, int64_t E, int64_t N, int64_t K,
                                  const void* alpha_row, int row_dtype, const void* alpha_col, int col_dtype,
                                  const void* topk_weights, int topk_dtype, const int32_t* sorted_token_ids, int64_t EM,
                                  const int32_t* expert_ids, const int32_t* num_tokens_post_padded,
                                  int64_t num_valid_tokens, int top_k, int block_m, int mul_routed_weight, void* out,
                                  int out_dtype, int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fnn;
  if (E <= 0 || N < 0 || K <= 0 || EM < 0 || lda < K || ldo < N || num_valid_tokens < 0 || top_k <= 0 || block_m <= 0)
    return fail(FNN_ERR_SHAPE, "fused_moe_a8w8: E=%lld N=%lld K=%lld EM=%lld lda=%lld ldo=%lld top_k=%d block_m=%d", (long long)E,
                (long long)N, (long long)K, (long long)EM, (long long)lda, (long long)ldo, top_k, block_m);
  if (E * N > INT32_MAX || K > INT32_MAX || EM > INT32_MAX || num_valid_tokens > INT32_MAX)
    return fail(FNN_ERR_SHAPE, "fused_moe_a8w8: sizes must be below 2^31");
  if (EM % block_m != 0) return fail(FNN_ERR_SHAPE, "fused_moe_a8w8: %lld sorted slots are not a multiple of block_m=%d", (long long)EM, block_m);
  if (block_m > kBM && block_m % kBM != 0)
    return fail(FNN_ERR_UNSUPPORTED, "fused_moe_a8w8: block_m must be at most %d or a multiple of it (got %d)", kBM, block_m);
  if (out_dtype != FNN_F16 && out_dtype != FNN_BF16) return fail(FNN_ERR_DTYPE, "fused_moe_a8w8: output must be f16 or bf16");
  if (row_dtype < FNN_F16 || row_dtype > FNN_F32 || col_dtype < FNN_F16 || col_dtype > FNN_F32)
    return fail(FNN_ERR_DTYPE, "fused_moe_a8w8: scales must be f16, bf16 or f32");
  if (mul_routed_weight && (topk_dtype < FNN_F16 || topk_dtype > FNN_F32)) return fail(FNN_ERR_DTYPE, "fused_moe_a8w8: routing weights must be f16, bf16 or f32");
  if (EM == 0 || N == 0 || num_valid_tokens == 0) return FNN_OK;
  if (!a || !b || !alpha_row || !alpha_col || !sorted_token_ids || !expert_ids || !num_tokens_post_padded || !out ||
      (mul_routed_weight && !topk_weights))
    return fail(FNN_ERR_NULL_POINTER, "fused_moe_a8w8: null tensor pointer");
  if (K % 16 != 0 || reinterpret_cast<uintptr_t>(a) % 16 != 0 || lda % 16 != 0 || reinterpret_cast<uintptr_t>(b) % 16 != 0)
    return fail(FNN_ERR_ALIGNMENT, "fused_moe_a8w8: K and lda must be multiples of 16 and the operands 16-byte aligned");
  const size_t need = fnn_fused_moe_a8w8_workspace_bytes(EM, K);
  if (!workspace || workspace_bytes < need) return fail(FNN_ERR_WORKSPACE, "fused_moe_a8w8: needs %zu bytes of workspace, got %zu", need, workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return fail(FNN_ERR_ALIGNMENT, "fused_moe_a8w8: workspace must be 256-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int8_t* a_sorted = static_cast<int8_t*>(workspace);
  moe_gather_rows_kernel<<<unsigned((EM + 7) / 8), 256, 0, st>>>(a, lda, sorted_token_ids, num_tokens_post_padded,
                                                                 int(num_valid_tokens), top_k, a_sorted, int(K), int(EM));
  if (int e = check_cuda(cudaGetLastError(), "fused moe gather launch")) return e;
  A8W8Params p{};
  p.alpha_row = alpha_row; p.alpha_col = alpha_col; p.out = out; p.acc_out = nullptr;
  p.ldo = ldo; p.ldacc = 0; p.row_dtype = row_dtype; p.col_dtype = col_dtype;
  p.M = int(num_valid_tokens); p.N = int(N); p.K = int(K);
  p.status = device_status_word();
  p.wait_ns = kWaitLimitNs; p.skip_kb = -1;
  p.sorted_ids = sorted_token_ids; p.expert_ids = expert_ids; p.num_post_padded = num_tokens_post_padded;
  p.topk_w = topk_weights; p.topk_w_dtype = topk_dtype; p.top_k = top_k; p.block_m = block_m;
  p.tile_rows = block_m < kBM ? block_m : kBM; p.num_valid = int(num_valid_tokens); p.mul_w = mul_routed_weight ? 1 : 0;
  p.col_stride_e = N;
  if (out_dtype == FNN_F16) return dispatch_moe<__half>(a_sorted, EM, b, E, p, st);
  return dispatch_moe<__nv_bfloat16>(a_sorted, EM, b, E, p, st);
}

extern "C" size_t fnn_gemm_a8w8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  using namespace fnn;
  if (M <= 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return 0;
  if (opt_test_stall_us() != 0 || opt_a8w8_pair_tile() != 0) return 0;
  return plan_a8w8(int(M), int(N), int(K), sm_count(), opt_a8w8_balanced()).balanced ? sk_workspace_bytes(sm_count()) : 0;
}

extern "C" int fnn_gemm_a8w8_plan(int64_t M, int64_t N, int64_t K, int* kernel, int* tile_n) {
  using namespace fnn;
  if (!kernel || !tile_n) return fail(FNN_ERR_NULL_POINTER, "gemm_a8w8_plan: null output pointer");
  if (M <= 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX) return fail(FNN_ERR_SHAPE, "gemm_a8w8_plan: M, N, K must be positive");
  if (M <= 8 && N >= 512 && N % 16 == 0 && K % 4096 == 0) {  // the streaming decode kernel takes these when its own shape rules hold
    *kernel = 2;
    *tile_n = 16;
    return FNN_OK;
  }
  const A8W8Plan plan = plan_a8w8(int(M), int(N), int(K > INT32_MAX ? INT32_MAX : K), sm_count(), opt_a8w8_balanced());
  *kernel = plan.balanced ? 3 : plan.pair ? 1 : 0;
  *tile_n = plan.bn;
  return FNN_OK;
}

extern "C" int fnn_gemm_a8w8(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, const void* alpha_row,
                             int row_dtype, const void* alpha_col, int col_dtype, void* out, int out_dtype,
                             int64_t ldo, int64_t M, int64_t N, int64_t K, int32_t* acc_out, int64_t ldacc,
                             void* workspace, size_t workspace_bytes, void* stream) {
  using namespace fnn;
  if (M < 0 || N < 0 || K < 0 || lda < K || ldb < K || ldo < N || (acc_out && ldacc < N))
    return fail(FNN_ERR_SHAPE, "gemm_a8w8: M=%lld N=%lld K=%lld lda=%lld ldb=%lld ldo=%lld", (long long)M,
                (long long)N, (long long)K, (long long)lda, (long long)ldb, (long long)ldo);
  if (M > INT32_MAX || N > INT32_MAX || K > INT32_MAX) return fail(FNN_ERR_SHAPE, "gemm_a8w8: sizes must be below 2^31");
  if (out_dtype != FNN_F16 && out_dtype != FNN_BF16) return fail(FNN_ERR_DTYPE, "gemm_a8w8: output must be f16 or bf16 (got dtype code %d)", out_dtype);
  if (row_dtype < FNN_F16 || row_dtype > FNN_F32 || col_dtype < FNN_F16 || col_dtype > FNN_F32)
    return fail(FNN_ERR_DTYPE, "gemm_a8w8: scales must be f16, bf16 or f32 (got dtype codes %d, %d)", row_dtype, col_dtype);
  if (M == 0 || N == 0) return FNN_OK;
  if (!a || !b || !alpha_row || !alpha_col || !out) return fail(FNN_ERR_NULL_POINTER, "gemm_a8w8: null tensor pointer");
  A8W8Params p{};
  p.alpha_row = alpha_row; p.alpha_col = alpha_col; p.out = out; p.acc_out = acc_out;
  p.ldo = ldo; p.ldacc = ldacc; p.row_dtype = row_dtype; p.col_dtype = col_dtype;
  p.M = int(M); p.N = int(N); p.K = int(K);
  p.status = device_status_word();
  p.wait_ns = kWaitLimitNs; p.skip_kb = -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_dtype == FNN_F16) return dispatch<__half>(a, lda, b, ldb, p, st, workspace, workspace_bytes);
  return dispatch<__nv_bfloat16>(a, lda, b, ldb, p, st, workspace, workspace_bytes);
}
