// A8W8 GEMM with bias, activation, gate and residual in its epilogue (epilogue.cuh): argument checks and the choice of
// kernel and tile.  The main loops are those of the plain A8W8 GEMM (a8w8_kernels.cuh, gemv_w4_imma.cu).
#include "a8w8_kernels.cuh"
#include "weight_only.cuh"

namespace fnn {
namespace {

// Operands the TMA path cannot address, and K == 0: one thread per output element.
template <typename OutT, class FX>
__global__ void a8w8_fused_generic_kernel(const int8_t* __restrict__ a, int64_t lda, const int8_t* __restrict__ b, int64_t ldb,
                                          const A8W8Params p, const FX fx) {
  const int64_t idx = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (idx >= int64_t(p.M) * p.N) return;
  const int m = int(idx / p.N), n = int(idx % p.N);
  const int8_t* ar = a + m * lda;
  const bool same16 = (p.row_dtype == p.col_dtype) && (p.row_dtype != FNN_F32);
  const float rs = load_as_f32(p.alpha_row, p.row_dtype, m);
  auto scaled = [&](int64_t row) {
    const int8_t* br = b + row * ldb;
    int acc = 0;
    for (int k = 0; k < p.K; ++k) acc += int(ar[k]) * int(br[k]);
    float s = __fmul_rn(rs, load_as_f32(p.alpha_col, p.col_dtype, row));
    if (same16) s = round_through(s, p.row_dtype);
    float v = __fmul_rn(float(acc), s);
    if (fx.bias) v += load_as_f32(fx.bias, fx.bias_dtype, row);
    return v;
  };
  float v = activate_one(scaled(n), fx.act);
  if (FX::kGated) v *= scaled(int64_t(p.N) + n);
  if (fx.residual) v += to_f32(reinterpret_cast<const OutT*>(fx.residual)[m * fx.ldr + n]);
  reinterpret_cast<OutT*>(p.out)[m * p.ldo + n] = from_f32<OutT>(v);
}

template <typename OutT, class FX>
int dispatch_fused(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, const A8W8Params& p, const FX& fx, cudaStream_t st) {
  const bool tma_ok = p.K > 0 && (reinterpret_cast<uintptr_t>(a) % 16 == 0) && (reinterpret_cast<uintptr_t>(b) % 16 == 0) &&
                      (lda % 16 == 0) && (ldb % 16 == 0);
  if (!tma_ok) {
    const int64_t total = int64_t(p.M) * p.N;
    a8w8_fused_generic_kernel<OutT, FX><<<unsigned((total + 255) / 256), 256, 0, st>>>(a, lda, b, ldb, p, fx);
    return check_cuda(cudaGetLastError(), "a8w8 fused generic launch");
  }
  // up to 8 tokens: the streaming kernel, by the plain GEMM's rule (512 weight rows or more)
  if (p.M <= 8 && fx.rows >= 512) {
    const int r = gemv_a8w8_imma_fused(a, lda, b, ldb, p.alpha_row, p.row_dtype, p.alpha_col, p.col_dtype, p.out,
                                       std::is_same<OutT, __half>::value ? FNN_F16 : FNN_BF16, p.ldo, p.M, p.N, p.K, fx, st);
    if (r >= 0) return r;
  }
  const A8W8Plan plan = plan_a8w8(p.M, p.N, sm_count(), FX::kGated);
  if (plan.pair) {
    switch (plan.bn) {
      case 256: return launch_pair<OutT, 256, false, 8>(a, lda, b, ldb, p, st, nullptr, fx);
      case 192: return launch_pair<OutT, 192, false, 8>(a, lda, b, ldb, p, st, nullptr, fx);
      case 128: return launch_pair<OutT, 128, false, 8>(a, lda, b, ldb, p, st, nullptr, fx);
      default: break;
    }
    if constexpr (!FX::kGated) {
      if (plan.bn == 224) return launch_pair<OutT, 224, false, 8>(a, lda, b, ldb, p, st, nullptr, fx);
      return launch_pair<OutT, 160, false, 8>(a, lda, b, ldb, p, st, nullptr, fx);
    }
  }
  if (plan.bn == 256) return launch_umma_rows<OutT, 256>(a, lda, b, ldb, p, st, fx);
  if (plan.bn == 128) return launch_umma_rows<OutT, 128>(a, lda, b, ldb, p, st, fx);
  return launch_umma_rows<OutT, 64>(a, lda, b, ldb, p, st, fx);
}

template <bool GATED>
int run_fused(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, const A8W8Params& p, const void* bias, int bias_dtype, int act,
              const void* residual, int64_t ldr, int out_dtype, cudaStream_t st) {
  FusedEpilogue<GATED> fx;
  fx.bias = bias; fx.residual = residual; fx.ldr = ldr; fx.bias_dtype = bias_dtype; fx.act = act;
  fx.rows = GATED ? 2 * p.N : p.N; fx.experts = fx.blocks = 0;
  if (out_dtype == FNN_F16) return dispatch_fused<__half>(a, lda, b, ldb, p, fx, st);
  return dispatch_fused<__nv_bfloat16>(a, lda, b, ldb, p, fx, st);
}

}  // namespace
}  // namespace fnn

extern "C" int fnn_gemm_a8w8_epilogue(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, const void* alpha_row, int row_dtype,
                                      const void* alpha_col, int col_dtype, const void* bias, int bias_dtype, int activation, int gated,
                                      const void* residual, int64_t ldr, void* out, int out_dtype, int64_t ldo, int64_t M, int64_t N,
                                      int64_t K, void* stream) {
  using namespace fnn;
  if (M < 0 || N < 0 || K < 0 || lda < K || ldb < K || ldo < N || (residual && ldr < 0))
    return fail(FNN_ERR_SHAPE, "gemm_a8w8_epilogue: M=%lld N=%lld K=%lld lda=%lld ldb=%lld ldo=%lld ldr=%lld", (long long)M, (long long)N,
                (long long)K, (long long)lda, (long long)ldb, (long long)ldo, (long long)ldr);
  if (M > INT32_MAX || N > INT32_MAX / 2 || K > INT32_MAX) return fail(FNN_ERR_SHAPE, "gemm_a8w8_epilogue: sizes must be below 2^31 (weight rows included)");
  if (out_dtype != FNN_F16 && out_dtype != FNN_BF16) return fail(FNN_ERR_DTYPE, "gemm_a8w8_epilogue: output must be f16 or bf16 (got dtype code %d)", out_dtype);
  if (row_dtype < FNN_F16 || row_dtype > FNN_F32 || col_dtype < FNN_F16 || col_dtype > FNN_F32)
    return fail(FNN_ERR_DTYPE, "gemm_a8w8_epilogue: scales must be f16, bf16 or f32 (got dtype codes %d, %d)", row_dtype, col_dtype);
  if (bias && (bias_dtype < FNN_F16 || bias_dtype > FNN_F32))
    return fail(FNN_ERR_DTYPE, "gemm_a8w8_epilogue: the bias must be f16, bf16 or f32 (got dtype code %d)", bias_dtype);
  if (activation < FNN_ACT_NONE || activation > FNN_ACT_GELU_TANH)
    return fail(FNN_ERR_UNSUPPORTED, "gemm_a8w8_epilogue: unknown activation code %d", activation);
  if (M == 0 || N == 0) return FNN_OK;
  if ((K > 0 && (!a || !b)) || !alpha_row || !alpha_col || !out) return fail(FNN_ERR_NULL_POINTER, "gemm_a8w8_epilogue: null tensor pointer");
  A8W8Params p{};
  p.alpha_row = alpha_row; p.alpha_col = alpha_col; p.out = out; p.acc_out = nullptr;
  p.ldo = ldo; p.ldacc = 0; p.row_dtype = row_dtype; p.col_dtype = col_dtype;
  p.M = int(M); p.N = int(N); p.K = int(K);
  p.status = device_status_word();
  p.wait_ns = kWaitLimitNs; p.skip_kb = -1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (gated) return run_fused<true>(a, lda, b, ldb, p, bias, bias_dtype, activation, residual, ldr, out_dtype, st);
  return run_fused<false>(a, lda, b, ldb, p, bias, bias_dtype, activation, residual, ldr, out_dtype, st);
}
