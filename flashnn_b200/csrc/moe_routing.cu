// The two ends of a mixture-of-experts layer: from router logits to the expert-sorted slot list that the expert products
// read, and from their [M, top_k, N] output back to [M, N].
#include <cooperative_groups.h>

#include <mutex>

#include "common.cuh"
#include "quantise.cuh"

namespace cg = cooperative_groups;

namespace fnn {
namespace {

// ---------------------------------------------------------------------------
// Routing: scores, balancing bias, group-limited choice, top-k, renormalised weights
// ---------------------------------------------------------------------------
// One warp per token, the row in registers: lane l holds experts l * PER .. l * PER + PER - 1, so that lane order is expert
// order and the lowest lane among equals holds the lowest expert.
//
// Which experts are chosen, and in what order, is defined in 64 bits.  Where the keys are the logits themselves (no bias,
// no sum over a group: both scores grow with the logit) comparing them is exact.  Elsewhere the row is done in fp32 first,
// with a bound on how far a key can be off; only where two keys that decide something are nearer than that (a row in some
// hundreds) is the row done again in 64 bits.
struct RouteParams {
  const void* logits;
  const float* bias;  // nullptr or [E]
  float* weights;     // [M, top_k]
  int32_t* ids;       // [M, top_k]
  int64_t ldl;
  int M, E, top_k, groups, topk_groups, group_size;
  int softmax, renormalize, summed;  // summed: a group's score is the sum of its two largest keys, else its largest
  float scale;
};

// order-preserving map of keys to unsigned integers; a NaN ranks with -infinity, 0 is left for "not there"
__device__ __forceinline__ uint32_t ordered(float v) {
  v = v != v ? __int_as_float(0xff800000) : v + 0.f;  // (-0 -> +0)
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long ordered(double v) {
  v = v != v ? __longlong_as_double(0xfff0000000000000ll) : v + 0.0;
  const unsigned long long b = __double_as_longlong(v);
  return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ double from_ordered(unsigned long long o) {
  return __longlong_as_double((o >> 63) ? o & 0x7fffffffffffffffull : ~o);
}
template <typename F> struct Ord { using type = uint32_t; };
template <> struct Ord<double> { using type = unsigned long long; };

__device__ __forceinline__ uint32_t warp_max(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  return v;
}
template <typename F> __device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

// One row in arithmetic F.  Lane i < top_k receives the i-th choice and its score; returns false where fp32 does not decide.
template <typename F, int PER>
__device__ bool route_row(const float (&x)[PER], int lane, const RouteParams& p, int& id, F& score) {
  using O = typename Ord<F>::type;
  constexpr bool kExact = sizeof(F) == 8;
  const F inf = F(__int_as_float(0x7f800000));
  const int e0 = lane * PER;
  const bool by_logit = p.bias == nullptr && !p.summed;
  // scores
  F s[PER];
  F widest = F(0);  // largest |key| or score of the row
  if (p.softmax) {
    O top_o = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (e0 + j < p.E) top_o = max(top_o, ordered(F(x[j])));
    F top = from_ordered(warp_max(top_o));
    if (top == inf || top == -inf) top = F(0);
    F total = F(0);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      s[j] = e0 + j < p.E ? exp_of(F(x[j]) - top) : F(0);
      total += s[j];
    }
    total = warp_sum(total);
    if (total == F(0)) total = F(1);
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] /= total;
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) s[j] = F(1) / (F(1) + exp_of(-F(x[j])));
  }
  // keys
  O key[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    F k = F(x[j]);
    if (!by_logit) {
      k = s[j];
      if (p.bias && e0 + j < p.E) k += F(__ldg(p.bias + e0 + j));
    }
    key[j] = e0 + j < p.E ? ordered(k) : O(0);
    if (!kExact && !by_logit && e0 + j < p.E) {
      const F a = fmaxf(fabsf(k), s[j]);
      if (a < inf) widest = fmaxf(widest, a);
    }
  }
  // How far an fp32 key can be off.  The sigmoid is within 4 roundings (2^-24 of its value each).  The softmax's argument x - max
  // is rounded by 2^-24 of up to 104 (beyond that the result is 0), its sum by one rounding per addition (at most
  // 37 in a row); its exponential and the division take 4 more: below 2^-16 of the value.  Adding the bias rounds once more.
  F tol = F(0);
  if (!kExact && !by_logit) tol = from_ordered(warp_max(ordered(widest))) * (p.softmax ? F(1.6e-5f) : F(5e-7f)) + F(1e-37f);
  bool sure = true;

  if (p.groups > 1) {
    // lane g < groups: the score of group g
    O mine = 0;
    for (int g = 0; g < p.groups; ++g) {
      const int lo = g * p.group_size, hi = lo + p.group_size;
      O best = 0;
      int at = -1;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (e0 + j >= lo && e0 + j < hi && key[j] > best) { best = key[j]; at = j; }
      const O first = warp_max(best);
      O value = first;
      if (p.summed && p.group_size > 1) {
        const int src = __ffs(__ballot_sync(0xffffffffu, best == first)) - 1;
        O second = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (e0 + j >= lo && e0 + j < hi && !(lane == src && j == at) && key[j] > second) second = key[j];
        value = ordered(from_ordered(first) + from_ordered(warp_max(second)));
      }
      if (lane == g) mine = value;
    }
    // its rank: groups with a larger score, or an equal one and a lower index
    int rank = 0;
    for (int g = 0; g < p.groups; ++g) {
      const O other = __shfl_sync(0xffffffffu, mine, g);
      rank += (other > mine || (other == mine && g < lane)) ? 1 : 0;
    }
    const bool in = lane < p.groups && rank < p.topk_groups;
    const uint32_t chosen = __ballot_sync(0xffffffffu, in);
    if (!kExact && !by_logit && p.topk_groups < p.groups) {
      const O worst_in = ~warp_max(in ? ~mine : O(0));
      const O best_out = warp_max((lane < p.groups && !in) ? mine : O(0));
      const F gap = from_ordered(worst_in) - from_ordered(best_out);
      if (!(gap > F(4) * tol)) sure = false;  // (two keys each; also where both are infinite)
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (e0 + j < p.E && !((chosen >> ((e0 + j) / p.group_size)) & 1u)) key[j] = 0;
  }

  // the top_k largest keys in order
  O last = 0;
  const int rounds = (!kExact && !by_logit) ? p.top_k + 1 : p.top_k;  // one more shows how near the first one left out is
  for (int i = 0; i < rounds; ++i) {
    O best = 0;
    int at = 0;
    F sc = F(0);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (key[j] > best) { best = key[j]; at = j; sc = s[j]; }
    const O m = warp_max(best);
    if (m == 0) break;  // (only the extra round can find nothing)
    if (!kExact && !by_logit && i > 0 && !(from_ordered(last) - from_ordered(m) > F(2) * tol)) sure = false;
    last = m;
    if (i == p.top_k) break;
    const int src = __ffs(__ballot_sync(0xffffffffu, best == m)) - 1;
    const int expert = __shfl_sync(0xffffffffu, e0 + at, src);
    const F value = __shfl_sync(0xffffffffu, sc, src);
    if (lane == i) { id = expert; score = value; }
    if (lane == src) {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (j == at) key[j] = 0;
    }
  }
  if (p.renormalize) {
    F total = warp_sum(lane < p.top_k ? score : F(0));
    if (!kExact && total < F(1e-30f)) sure = false;  // (scores that fp32 cannot hold)
    if (total == F(0)) total = F(1);
    score /= total;
  }
  score *= F(p.scale);
  return sure;
}

constexpr int kRouteWarps = 8;

template <typename T, int PER>
__global__ void __launch_bounds__(kRouteWarps * 32) moe_route_kernel(const RouteParams p) {
  const int row = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (row >= p.M) return;
  const int lane = threadIdx.x & 31;
  const T* src = reinterpret_cast<const T*>(p.logits) + row * p.ldl;
  float x[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) x[j] = lane * PER + j < p.E ? to_f32(src[lane * PER + j]) : 0.f;
  int id = 0;
  float score = 0.f;
  if (!route_row<float, PER>(x, lane, p, id, score)) {  // (the whole warp agrees)
    double exact = 0.0;
    route_row<double, PER>(x, lane, p, id, exact);
    score = float(exact);
  }
  if (lane < p.top_k) {
    const int64_t at = int64_t(row) * p.top_k + lane;
    p.weights[at] = score;
    p.ids[at] = id;
  }
}

template <typename T>
int launch_route(const RouteParams& p, cudaStream_t st) {
  const unsigned grid = unsigned((p.M + kRouteWarps - 1) / kRouteWarps);
  const int per = (p.E + 31) / 32;
  if (per <= 1) moe_route_kernel<T, 1><<<grid, kRouteWarps * 32, 0, st>>>(p);
  else if (per <= 2) moe_route_kernel<T, 2><<<grid, kRouteWarps * 32, 0, st>>>(p);
  else if (per <= 4) moe_route_kernel<T, 4><<<grid, kRouteWarps * 32, 0, st>>>(p);
  else if (per <= 8) moe_route_kernel<T, 8><<<grid, kRouteWarps * 32, 0, st>>>(p);
  else if (per <= 16) moe_route_kernel<T, 16><<<grid, kRouteWarps * 32, 0, st>>>(p);
  else moe_route_kernel<T, 32><<<grid, kRouteWarps * 32, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "moe_route launch");
}

// ---------------------------------------------------------------------------
// Expert sort: a stable counting sort of the flat (token, choice) indices by expert, every expert's slots padded to whole
// blocks
// ---------------------------------------------------------------------------
// One cluster does it in one launch.  Its warps take consecutive pieces of the list.  Pass 1 counts each warp's experts in
// shared memory; prefix sums over a CTA's warps, over the cluster's CTAs (through distributed shared memory) and over the
// experts' padded sizes give every warp its first slot of every expert; pass 2 hands the slots out in list order (a match
// over the warp ranks equal experts).  No atomics decide an order: the list is the same every time.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortMaxExperts = 1024;  // one thread per expert in the prefix sums

struct SortParams {
  const int32_t* ids;
  int32_t* sorted;
  int32_t* experts;
  int32_t* num_post_padded;
  int choices, E, bm, first, slots;
};

__global__ void __launch_bounds__(kSortThreads) moe_sort_kernel(const SortParams p) {
  extern __shared__ int32_t cnt[];            // [kSortWarps][E]: counts, then the warp's next slot within the expert
  int32_t* total = cnt + kSortWarps * p.E;    // [E] this CTA's counts
  int32_t* begin = total + p.E;               // [E] first slot of the expert
  int32_t* count = begin + p.E;               // [E] slots in use of the expert
  __shared__ int32_t scan[kSortWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = int(cluster.block_rank()), ctas = int(cluster.num_blocks());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gw = rank * kSortWarps + warp, warps = ctas * kSortWarps;
  const int piece = ((p.choices + warps - 1) / warps + 31) / 32 * 32;
  const int64_t lo64 = int64_t(gw) * piece;
  const int lo = int(lo64 < p.choices ? lo64 : p.choices);
  const int hi = int(lo64 + piece < p.choices ? lo64 + piece : p.choices);
  int32_t* mine = cnt + warp * p.E;

  for (int i = threadIdx.x; i < kSortWarps * p.E; i += kSortThreads) cnt[i] = 0;
  __syncthreads();
  for (int i = lo + lane; i < hi; i += 32) {
    const unsigned e = unsigned(p.ids[i]) - unsigned(p.first);
    if (e < unsigned(p.E)) atomicAdd(mine + e, 1);
  }
  __syncthreads();
  const int e = threadIdx.x;
  if (e < p.E) {
    int run = 0;
    for (int w = 0; w < kSortWarps; ++w) {
      const int t = cnt[w * p.E + e];
      cnt[w * p.E + e] = run;
      run += t;
    }
    total[e] = run;
  }
  cluster.sync();
  int before = 0, all = 0;
  if (e < p.E) {
    for (int c = 0; c < ctas; ++c) {
      const int t = cluster.map_shared_rank(total, c)[e];
      if (c < rank) before += t;
      all += t;
    }
  }
  const int padded = (all + p.bm - 1) / p.bm * p.bm;
  int sum = padded;  // inclusive prefix over the experts
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += t;
  }
  if (lane == 31) scan[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int t = scan[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    scan[lane] = t;
  }
  __syncthreads();
  const int in_use = scan[kSortWarps - 1];
  const int start = sum - padded + (warp > 0 ? scan[warp - 1] : 0);
  if (e < p.E) {
    begin[e] = start;
    count[e] = all;
    for (int w = 0; w < kSortWarps; ++w) cnt[w * p.E + e] += start + before;
  }
  if (rank == 0 && threadIdx.x == 0) *p.num_post_padded = in_use;
  __syncthreads();

  for (int i0 = lo; i0 < hi; i0 += 32) {
    const int i = i0 + lane;
    unsigned ex = i < hi ? unsigned(p.ids[i]) - unsigned(p.first) : 0xffffffffu;
    if (ex >= unsigned(p.E)) ex = 0xffffffffu;
    const uint32_t same = __match_any_sync(0xffffffffu, ex);
    const bool here = ex != 0xffffffffu;
    const int base = here ? mine[ex] : 0;
    const int ahead = __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (here && ahead == 0) mine[ex] = base + __popc(same);
    __syncwarp();
    if (here) p.sorted[base + ahead] = i;
  }
  // padding slots and the blocks' experts
  for (int x = gw; x < p.E; x += warps) {
    const int b = begin[x], n = count[x], end = b + (n + p.bm - 1) / p.bm * p.bm;
    for (int s = b + n + lane; s < end; s += 32) p.sorted[s] = p.choices;
    for (int k = b / p.bm + lane; k < end / p.bm; k += 32) p.experts[k] = x;
  }
  for (int s = in_use + rank * kSortThreads + threadIdx.x; s < p.slots; s += ctas * kSortThreads) p.sorted[s] = p.choices;
  for (int k = in_use / p.bm + rank * kSortThreads + threadIdx.x; k < p.slots / p.bm; k += ctas * kSortThreads) p.experts[k] = 0;
  cluster.sync();  // nobody leaves while another CTA may still read its counts
}

// ---------------------------------------------------------------------------
// Sum over a token's choices
// ---------------------------------------------------------------------------
struct CombineParams {
  const void* c;
  const float* w;      // nullptr or [M, top_k]
  const int32_t* ids;  // nullptr or [M, top_k]
  const void* residual;
  void* out;
  int64_t ldc_m, ldc_k, ldr, ldo;
  int M, N, top_k, E, first;
};

// VEC: columns of a thread, 8 (16-byte accesses) or 1
template <typename T, int VEC>
__global__ void __launch_bounds__(256) moe_combine_kernel(const CombineParams p) {
  const int64_t m = blockIdx.x;
  const int n = (blockIdx.y * 256 + threadIdx.x) * VEC;
  if (n >= p.N) return;
  float acc[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) acc[j] = 0.f;
  auto add = [&](const T* src, float w) {
    if constexpr (VEC == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(src);
      const uint32_t a[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[2 * j] = fmaf(w, lo_of<T>(a[j]), acc[2 * j]);
        acc[2 * j + 1] = fmaf(w, hi_of<T>(a[j]), acc[2 * j + 1]);
      }
    } else {
      acc[0] = fmaf(w, to_f32(*src), acc[0]);
    }
  };
  const T* c = reinterpret_cast<const T*>(p.c) + m * p.ldc_m + n;
  for (int k = 0; k < p.top_k; ++k) {
    if (p.ids && unsigned(__ldg(p.ids + m * p.top_k + k)) - unsigned(p.first) >= unsigned(p.E)) continue;
    add(c + k * p.ldc_k, p.w ? __ldg(p.w + m * p.top_k + k) : 1.f);
  }
  if (p.residual) add(reinterpret_cast<const T*>(p.residual) + m * p.ldr + n, 1.f);
  T* out = reinterpret_cast<T*>(p.out) + m * p.ldo + n;
  if constexpr (VEC == 8)
    *reinterpret_cast<uint4*>(out) = make_uint4(pack2<T>(acc[0], acc[1]), pack2<T>(acc[2], acc[3]), pack2<T>(acc[4], acc[5]), pack2<T>(acc[6], acc[7]));
  else
    *out = from_f32<T>(acc[0]);
}

template <typename T> int launch_combine(const CombineParams& p, cudaStream_t st) {
  auto aligned = [](const void* q, int64_t ld) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 8 == 0; };
  const bool vec = p.N % 8 == 0 && aligned(p.c, p.ldc_m) && p.ldc_k % 8 == 0 && aligned(p.out, p.ldo) &&
                   (!p.residual || aligned(p.residual, p.ldr));
  const int per = 256 * (vec ? 8 : 1);
  const int64_t chunks = (int64_t(p.N) + per - 1) / per;
  if (chunks > 65535) return fail(FNN_ERR_UNSUPPORTED, "moe_combine: rows of %d columns are too long", p.N);
  const dim3 grid(unsigned(p.M), unsigned(chunks));
  if (vec) moe_combine_kernel<T, 8><<<grid, 256, 0, st>>>(p);
  else moe_combine_kernel<T, 1><<<grid, 256, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "moe_combine launch");
}

}  // namespace
}  // namespace fnn

extern "C" int fnn_moe_route(const void* logits, int logits_dtype, int64_t ldl, int64_t M, int64_t E, const float* bias, int scoring,
                             int renormalize, int num_groups, int topk_groups, int group_score, float scale, int top_k,
                             float* topk_weights, int32_t* topk_ids, void* stream) {
  using namespace fnn;
  if (M < 0 || E <= 0 || ldl < E || top_k <= 0 || num_groups <= 0 || topk_groups <= 0)
    return fail(FNN_ERR_SHAPE, "moe_route: M=%lld E=%lld ldl=%lld top_k=%d num_groups=%d topk_groups=%d", (long long)M, (long long)E,
                (long long)ldl, top_k, num_groups, topk_groups);
  if (M > INT32_MAX) return fail(FNN_ERR_SHAPE, "moe_route: M must be below 2^31");
  if (E > 1024 || top_k > 32 || num_groups > 32)
    return fail(FNN_ERR_UNSUPPORTED, "moe_route: at most 1024 experts, 32 choices and 32 groups (got %lld, %d, %d)", (long long)E, top_k, num_groups);
  if (E % num_groups != 0 || topk_groups > num_groups)
    return fail(FNN_ERR_SHAPE, "moe_route: %lld experts in %d groups, %d of them chosen", (long long)E, num_groups, topk_groups);
  if (top_k > topk_groups * (E / num_groups))
    return fail(FNN_ERR_SHAPE, "moe_route: top_k=%d of the %lld experts that the chosen groups have", top_k, (long long)(topk_groups * (E / num_groups)));
  if (logits_dtype < FNN_F16 || logits_dtype > FNN_F32) return fail(FNN_ERR_DTYPE, "moe_route: logits must be f16, bf16 or f32");
  if (scoring != FNN_SCORE_SOFTMAX && scoring != FNN_SCORE_SIGMOID) return fail(FNN_ERR_UNSUPPORTED, "moe_route: unknown scoring code %d", scoring);
  if (group_score != FNN_GROUP_MAX && group_score != FNN_GROUP_TOP2) return fail(FNN_ERR_UNSUPPORTED, "moe_route: unknown group score code %d", group_score);
  if (M == 0) return FNN_OK;
  if (!logits || !topk_weights || !topk_ids) return fail(FNN_ERR_NULL_POINTER, "moe_route: null tensor pointer");
  RouteParams p{};
  p.logits = logits; p.bias = bias; p.weights = topk_weights; p.ids = topk_ids; p.ldl = ldl;
  p.M = int(M); p.E = int(E); p.top_k = top_k; p.groups = num_groups; p.topk_groups = topk_groups; p.group_size = int(E / num_groups);
  p.softmax = scoring == FNN_SCORE_SOFTMAX; p.renormalize = renormalize != 0;
  p.summed = num_groups > 1 && group_score == FNN_GROUP_TOP2; p.scale = scale;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (logits_dtype == FNN_F16) return launch_route<__half>(p, st);
  if (logits_dtype == FNN_BF16) return launch_route<__nv_bfloat16>(p, st);
  return launch_route<float>(p, st);
}

extern "C" int64_t fnn_moe_sort_slots(int64_t num_choices, int64_t E, int block_m) {
  if (num_choices <= 0 || E <= 0 || block_m <= 0) return 0;
  const int64_t used = num_choices < E ? num_choices : E;
  return (used + (num_choices - used) / block_m) * block_m;
}

extern "C" int fnn_moe_sort(const int32_t* topk_ids, int64_t num_choices, int64_t E, int64_t first_expert, int block_m,
                            int32_t* sorted_token_ids, int64_t EM, int32_t* expert_ids, int32_t* num_tokens_post_padded, void* stream) {
  using namespace fnn;
  if (num_choices < 0 || E <= 0 || block_m <= 0 || EM < 0)
    return fail(FNN_ERR_SHAPE, "moe_sort: num_choices=%lld E=%lld block_m=%d EM=%lld", (long long)num_choices, (long long)E, block_m, (long long)EM);
  if (E > kSortMaxExperts) return fail(FNN_ERR_UNSUPPORTED, "moe_sort: at most %d experts (got %lld)", kSortMaxExperts, (long long)E);
  if (first_expert < INT32_MIN || first_expert > INT32_MAX) return fail(FNN_ERR_SHAPE, "moe_sort: first_expert must fit 32 bits");
  const int64_t need = fnn_moe_sort_slots(num_choices, E, block_m);
  if (num_choices > INT32_MAX / 2 || need > INT32_MAX / 2) return fail(FNN_ERR_SHAPE, "moe_sort: %lld choices need %lld slots: too many", (long long)num_choices, (long long)need);
  if (EM != need) return fail(FNN_ERR_SHAPE, "moe_sort: the slot list has %lld entries, fnn_moe_sort_slots says %lld", (long long)EM, (long long)need);
  if (!num_tokens_post_padded || (num_choices > 0 && (!topk_ids || !sorted_token_ids || !expert_ids)))
    return fail(FNN_ERR_NULL_POINTER, "moe_sort: null tensor pointer");
  SortParams p{topk_ids, sorted_token_ids, expert_ids, num_tokens_post_padded, int(num_choices), int(E), block_m, int(first_expert), int(EM)};
  const size_t smem = size_t(kSortWarps + 3) * size_t(E) * sizeof(int32_t);
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  cudaGetDevice(&dev);
  dev &= 63;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(moe_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kSortWarps + 3) * kSortMaxExperts * 4);
  });
  if (attr_err[dev] != cudaSuccess) return check_cuda(attr_err[dev], "cudaFuncSetAttribute(moe_sort)");
  cudaLaunchConfig_t cfg = {};
  const unsigned ctas = num_choices > 4096 ? 8u : 1u;
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, moe_sort_kernel, p), "moe_sort launch");
}

extern "C" int fnn_moe_combine(const void* c, int dtype, int64_t ldc_m, int64_t ldc_k, int64_t M, int64_t top_k, int64_t N,
                               const float* topk_weights, const int32_t* topk_ids, int64_t E, int64_t first_expert,
                               const void* residual, int64_t ldr, void* out, int64_t ldo, void* stream) {
  using namespace fnn;
  if (M < 0 || N < 0 || top_k < 0 || ldc_m < 0 || ldc_k < 0 || ldo < N || (residual && ldr < 0) || (topk_ids && E <= 0))
    return fail(FNN_ERR_SHAPE, "moe_combine: M=%lld top_k=%lld N=%lld ldc_m=%lld ldc_k=%lld ldr=%lld ldo=%lld E=%lld", (long long)M,
                (long long)top_k, (long long)N, (long long)ldc_m, (long long)ldc_k, (long long)ldr, (long long)ldo, (long long)E);
  if (M > INT32_MAX || N > INT32_MAX || top_k > INT32_MAX) return fail(FNN_ERR_SHAPE, "moe_combine: sizes must be below 2^31");
  if (topk_ids && (E > INT32_MAX || first_expert < INT32_MIN || first_expert > INT32_MAX))
    return fail(FNN_ERR_SHAPE, "moe_combine: E and first_expert must fit 32 bits");
  if (dtype != FNN_F16 && dtype != FNN_BF16) return fail(FNN_ERR_DTYPE, "moe_combine: the expert outputs must be f16 or bf16 (got dtype code %d)", dtype);
  if (M == 0 || N == 0) return FNN_OK;
  if (!out || (top_k > 0 && !c)) return fail(FNN_ERR_NULL_POINTER, "moe_combine: null tensor pointer");
  CombineParams p{};
  p.c = c; p.w = topk_weights; p.ids = topk_ids; p.residual = residual; p.out = out;
  p.ldc_m = ldc_m; p.ldc_k = ldc_k; p.ldr = ldr; p.ldo = ldo;
  p.M = int(M); p.N = int(N); p.top_k = int(top_k); p.E = int(E); p.first = int(first_expert);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FNN_F16 ? launch_combine<__half>(p, st) : launch_combine<__nv_bfloat16>(p, st);
}
