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
    if (fx.bias) v = __fadd_rn(v, load_as_f32(fx.bias, fx.bias_dtype, row));
    return v;
  };
  float v = activate_one(scaled(n), fx.act);
  if (FX::kGated) v = __fmul_rn(v, scaled(int64_t(p.N) + n));
  if (fx.residual) v = __fadd_rn(v, to_f32(reinterpret_cast<const OutT*>(fx.residual)[m * fx.ldr + n]));
  reinterpret_cast<OutT*>(p.out)[m * p.ldo + n] = from_f32<OutT>(v);
}

// ---------------------------------------------------------------------------
// Few tiles, long K: a cluster of CTAs shares the K blocks of one 128 x 64 tile (accumulator columns).  Every CTA leaves its int32
// sums in its shared memory; after a cluster barrier all of them take a share of the outputs, add the CTAs' sums (exact in any order)
// through distributed shared memory and finish them, four columns a thread.  One tile per cluster, so there is nothing to
// overlap and the epilogue can be scalar code, which is also little code: such a launch fetches every instruction once.
// Latency bounds it: of 9 us for 16 x 4096 x 4096 the weights take 3.
// ---------------------------------------------------------------------------
constexpr int kSplitBN = 64;
constexpr uint64_t kDrainNs = 2000000ull;  // for copies that are in flight when a wait has run out
constexpr int kSplitPitch = kSplitBN + 4;  // words of a row of sums: 16-byte accesses of eight neighbouring rows hit different banks

__device__ __forceinline__ int4 ld_cluster_int4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

template <typename OutT, int AROWS, int STAGES, class FX>
__global__ void __launch_bounds__(kThreads, 1)
a8w8_split_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const A8W8Params p, const FX fx,
                  const int splits) {
  using L = SmemLayout<kSplitBN, STAGES, AROWS>;
  constexpr int OW = FX::kGated ? kSplitBN / 2 : kSplitBN;  // output columns of a tile
  static_assert(kBM * kSplitPitch * 4 <= STAGES * L::kStageBytes, "the sums lie where the operands were");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
  uint64_t* full_bar = bars;
  uint64_t* empty_bar = bars + STAGES;
  uint64_t* tmem_full_bar = bars + 2 * STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kTmemSlotOff);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kAbortOff);
  int* sums = reinterpret_cast<int*>(smem);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(cluster_ctarank());
  const int nb = int(blockIdx.x) / splits;
  const int kb0 = int(int64_t(p.k_blocks) * rank / splits), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / splits);
  const int n0 = nb * OW, rows = p.M;  // (at most 128)

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    mbar_init(tmem_full_bar, 1);
    mbar_fence_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kSplitBN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    const bool leader = elect_one();
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      const int i = kb - kb0, stage = i % STAGES;
      ok = mbar_wait_bounded(&empty_bar[stage], uint32_t((i / STAGES) & 1) ^ 1, abort_flag, p.wait_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (leader) report(p.status, abort_flag, DEV_TIMEOUT_PRODUCER);
        break;
      }
      if (leader && !(i == p.skip_kb && rank == 0)) {  // (test hook: one K block's loads left out)
        uint8_t* sa = smem + stage * L::kStageBytes;
        mbar_expect_tx(&full_bar[stage], L::kStageBytes);
        tma_load_2d(sa + L::kABytes, &tmap_b, &full_bar[stage], kb * kBK, n0);
        if (FX::kGated) tma_load_2d(sa + L::kABytes + OW * kBK, &tmap_b, &full_bar[stage], kb * kBK, n0 + p.N);
        tma_load_2d(sa, &tmap_a, &full_bar[stage], kb * kBK, 0);
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    const bool leader = elect_one();
    constexpr uint32_t idesc = umma_idesc(/*s32*/ 2, /*signed 8-bit*/ 1, kBM, kSplitBN);
    int done = 0;
    for (int kb = kb0; kb < kb1; ++kb, ++done) {
      const int stage = done % STAGES;
      bool ok = mbar_wait_bounded(&full_bar[stage], uint32_t((done / STAGES) & 1), abort_flag, p.wait_ns);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        if (leader) report(p.status, abort_flag, DEV_TIMEOUT_MMA);
        break;
      }
      tc_fence_after();
      if (leader) {
        const uint32_t sa = smem_u32(smem + stage * L::kStageBytes);
        const uint32_t sb = sa + L::kABytes;
#pragma unroll
        for (int k = 0; k < kBK / kUmmaK; ++k)
          umma_i8(tmem_base, umma_desc_k_sw128(sa + k * kUmmaK), umma_desc_k_sw128(sb + k * kUmmaK), idesc, (done | k) != 0 ? 1u : 0u);
        tc_commit(&empty_bar[stage]);
      }
      __syncwarp();
    }
    // also after an abort: nothing is freed before the MMAs issued have completed
    if (leader) {
      tc_commit(tmem_full_bar);
      int none = 0;
      if (!mbar_wait_bounded(tmem_full_bar, 0, &none, p.wait_ns)) report(p.status, abort_flag, DEV_TIMEOUT_DRAIN);
      // (and, after an abort, before the copies issued have landed)
      if (*abort_flag != 0)
        for (int i = done; i < kb1 - kb0 && i < done + STAGES; ++i) mbar_wait_bounded(&full_bar[i % STAGES], uint32_t((i / STAGES) & 1), &none, kDrainNs);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3;
    bool ok = mbar_wait_bounded(tmem_full_bar, 0, abort_flag, p.wait_ns);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) {
      if (lane == 0) report(p.status, abort_flag, DEV_TIMEOUT_EPILOGUE);
    } else if (quarter * 32 < rows) {
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < kSplitBN / 32; ++c) {
        uint32_t r[32];
        tmem_ld_32x32(tmem_base + (uint32_t(quarter * 32) << 16) + c * 32, r);
        tc_wait_ld();
        if (quarter * 32 + lane < rows) {
          int4* dst = reinterpret_cast<int4*>(sums + (quarter * 32 + lane) * kSplitPitch + c * 32);
#pragma unroll
          for (int j = 0; j < 8; ++j) dst[j] = make_int4(int(r[4 * j]), int(r[4 * j + 1]), int(r[4 * j + 2]), int(r[4 * j + 3]));
        }
      }
      tc_fence_before();
    }
  }

  // a thread's outputs: four columns of a row at a time; what its first ones need from global memory is on its way during the barrier
  // (an absent bias or residual is -0, which leaves every number as it is, a zero's sign included)
  struct Item {
    float rs, cs[4], bs[4], cu[4], bu[4], res[4];
  };
  constexpr int kQuads = OW / 4;
  const bool same16 = (p.row_dtype == p.col_dtype) && (p.row_dtype != FNN_F32);
  const int items = rows * kQuads, stride = splits * kThreads;
  auto fetch = [&](int i, Item& t) {
    const int row = i / kQuads, col = n0 + (i % kQuads) * 4;
    t.rs = load_as_f32(p.alpha_row, p.row_dtype, row);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool on = col + j < p.N;
      t.cs[j] = on ? load_as_f32(p.alpha_col, p.col_dtype, col + j) : 0.f;
      t.bs[j] = (on && fx.bias) ? load_as_f32(fx.bias, fx.bias_dtype, col + j) : -0.f;
      if (FX::kGated) {
        t.cu[j] = on ? load_as_f32(p.alpha_col, p.col_dtype, int64_t(p.N) + col + j) : 0.f;
        t.bu[j] = (on && fx.bias) ? load_as_f32(fx.bias, fx.bias_dtype, int64_t(p.N) + col + j) : -0.f;
      }
      t.res[j] = (on && fx.residual) ? to_f32(reinterpret_cast<const OutT*>(fx.residual)[int64_t(row) * fx.ldr + col + j]) : -0.f;
    }
  };
  int i = rank * kThreads + int(threadIdx.x);
  Item item;
  if (i < items) fetch(i, item);
  __syncthreads();
  cluster_sync_all();
  const uint32_t sums_addr = smem_u32(sums);
  while (i < items) {
    const int r = i / kQuads, c = (i % kQuads) * 4;
    int4 a = make_int4(0, 0, 0, 0), b = a;
    for (int q = 0; q < splits; ++q) {
      const uint32_t at = map_to_cta(sums_addr + (r * kSplitPitch + c) * 4, uint32_t(q));
      const int4 t = ld_cluster_int4(at);
      a.x += t.x; a.y += t.y; a.z += t.z; a.w += t.w;
      if (FX::kGated) {
        const int4 u = ld_cluster_int4(at + OW * 4);
        b.x += u.x; b.y += u.y; b.z += u.z; b.w += u.w;
      }
    }
    const int acc[4] = {a.x, a.y, a.z, a.w}, up[4] = {b.x, b.y, b.z, b.w};
    auto scaled = [&](int sum, float cs, float bias) {
      float s = __fmul_rn(item.rs, cs);
      if (same16) s = round_through(s, p.row_dtype);
      return __fadd_rn(__fmul_rn(float(sum), s), bias);
    };
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = scaled(acc[j], item.cs[j], item.bs[j]);
    activate_n(v, fx.act);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (FX::kGated) v[j] = __fmul_rn(v[j], scaled(up[j], item.cu[j], item.bu[j]));
      v[j] = __fadd_rn(v[j], item.res[j]);
    }
    OutT* out = reinterpret_cast<OutT*>(p.out) + int64_t(r) * p.ldo + n0 + c;
    if (n0 + c + 4 <= p.N && (reinterpret_cast<uintptr_t>(out) & 7) == 0) {
      *reinterpret_cast<uint2*>(out) = make_uint2(pack2<OutT>(v[0], v[1]), pack2<OutT>(v[2], v[3]));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n0 + c + j < p.N) out[j] = from_f32<OutT>(v[j]);
    }
    i += stride;
    if (i < items) fetch(i, item);
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // nobody leaves while another CTA may still read its sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kSplitBN);
  }
}

template <typename OutT, int AROWS, class FX>
int launch_split(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, A8W8Params p, const FX& fx, int splits, cudaStream_t st) {
  constexpr int kFit = 210 * 1024 / ((AROWS + kSplitBN) * kBK);
  constexpr int STAGES = kFit < 12 ? kFit : 12;
  using L = SmemLayout<kSplitBN, STAGES, AROWS>;
  static_assert(L::kDynamicBytes <= 227 * 1024, "shared memory budget");
  constexpr int OW = FX::kGated ? kSplitBN / 2 : kSplitBN;
  auto kern = a8w8_split_kernel<OutT, AROWS, STAGES, FX>;
  static std::once_flag once[64];
  static cudaError_t attr_err[64];  // per device, so that a failure is reported on every call and not only the first
  int dev = 0;
  cudaGetDevice(&dev);
  dev &= 63;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynamicBytes);
  });
  if (attr_err[dev] != cudaSuccess) return check_cuda(attr_err[dev], "cudaFuncSetAttribute(a8w8 split)");
  CUtensorMap ta, tb;
  if (int e = make_tmap_i8(&ta, a, p.M, p.K, lda, AROWS)) return e;
  if (int e = make_tmap_i8(&tb, b, fx.rows, p.K, ldb, OW)) return e;
  p.tiles_n = (p.N + OW - 1) / OW;
  p.k_blocks = (p.K + kBK - 1) / kBK;
  if (const int stall_us = opt_test_stall_us()) {  // test hook: make one wait of every cluster's first CTA run out quickly
    p.wait_ns = 1000ull * unsigned(stall_us);
    p.skip_kb = 1;  // (a CTA has four K blocks or more)
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(p.tiles_n * splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = L::kDynamicBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(splits);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, ta, tb, p, fx, splits), "a8w8 split-K launch");
}

// CTAs that share a tile of at most 128 tokens (1: no sharing): as many as leave every one an SM and four K blocks, where that gains.
// Measured, in us: a K block takes a CTA 0.25, the barrier 1.5, a thread's four columns in the joint epilogue 1.  16 x 4096 x 4096
// 12.2 -> 9.0, 2 x 68 x 17696 36 -> 8.7, 128 x 2048 x 8192 20 -> 12.6, 64 x 2048 x 28672 55 -> 22; 64 x 1024 x 1024 7.3 -> 9.0 and 300 x 1024 x 1024
// 7.9 -> 13.3, which this rule leaves alone.
inline int split_of(int M, int rows, int K, int sms) {
  if (M > kBM) return 1;
  const int64_t tiles = (rows + kSplitBN - 1) / kSplitBN;
  const int k_blocks = (K + kBK - 1) / kBK;
  for (int s = 8; s > 1; s /= 2)
    if (tiles * s <= sms && k_blocks >= 4 * s) return k_blocks * (s - 1) * 0.25 > M * (kSplitBN / 4.0) / kThreads + 1.5 * s ? s : 1;
  return 1;
}

template <typename OutT, int EPI, class FX>
int launch_pair_width(int bn, const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, const A8W8Params& p, const FX& fx, cudaStream_t st) {
  if (bn == 256) return launch_pair<OutT, 256, false, EPI>(a, lda, b, ldb, p, st, nullptr, fx);
  if (bn == 192) return launch_pair<OutT, 192, false, EPI>(a, lda, b, ldb, p, st, nullptr, fx);
  if constexpr (!FX::kGated) {
    if (bn == 224) return launch_pair<OutT, 224, false, EPI>(a, lda, b, ldb, p, st, nullptr, fx);
    if (bn == 160) return launch_pair<OutT, 160, false, EPI>(a, lda, b, ldb, p, st, nullptr, fx);
  }
  return launch_pair<OutT, 128, false, EPI>(a, lda, b, ldb, p, st, nullptr, fx);
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
  if (const int splits = split_of(p.M, fx.rows, p.K, sm_count()); splits > 1) {
    if (p.M <= 16) return launch_split<OutT, 16>(a, lda, b, ldb, p, fx, splits, st);
    if (p.M <= 64) return launch_split<OutT, 64>(a, lda, b, ldb, p, fx, splits, st);
    return launch_split<OutT, 128>(a, lda, b, ldb, p, fx, splits, st);
  }
  const A8W8Plan plan = plan_a8w8(p.M, p.N, sm_count(), FX::kGated);
  // With K up to 2048 a tile waits for its epilogue, and 16 warps finish it sooner than 8 (two against four per scheduler, chunks of
  // 16 columns): 4096 x 8192 x 1024, none 38 -> 34 us, silu 53 -> 48, bias + gelu + residual 79 -> 73 (66 with the present gelu); at 2048
  // silu 57 -> 53; from 4096 on the MMAs hide either, and the expert products, which scatter rows, take 5 % longer with 16.  No pipe
  // bounds what is left: with silu at K = 1024 the tensor pipe is busy 37 % of the time and that of conversions, exponentials and
  // reciprocals (three slots an element) 39 %; the warps wait for one another's results and for TMEM.
  if (plan.pair) return p.K <= 2048 ? launch_pair_width<OutT, 16>(plan.bn, a, lda, b, ldb, p, fx, st) : launch_pair_width<OutT, 8>(plan.bn, a, lda, b, ldb, p, fx, st);
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
