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
  int wide, wide_bias, slow_groups;  // set by the launch: lanes read whole words; groups that are not a power of two of lanes
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
  const uint32_t hi = __reduce_max_sync(0xffffffffu, uint32_t(v >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, uint32_t(v >> 32) == hi ? uint32_t(v) : 0u);
  return (static_cast<unsigned long long>(hi) << 32) | lo;
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

// A lane's PER logits, experts lane * PER .. lane * PER + PER - 1; absent ones read as 0.
template <typename T, int PER>
__device__ __forceinline__ void load_logits(const RouteParams& p, int64_t row, int lane, bool wide, float (&x)[PER]) {
  const T* src = reinterpret_cast<const T*>(p.logits) + row * p.ldl + lane * PER;
  constexpr int kWord = 16 / int(sizeof(T)) < PER ? 16 / int(sizeof(T)) : PER;  // logits per load
  if (wide) {
#pragma unroll
    for (int w = 0; w < PER / kWord; ++w) {
      struct alignas(kWord * sizeof(T)) Word { T v[kWord]; };
      Word u{};
      if (lane * PER + w * kWord < p.E) u = *reinterpret_cast<const Word*>(src + w * kWord);
#pragma unroll
      for (int j = 0; j < kWord; ++j) x[w * kWord + j] = to_f32(u.v[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = lane * PER + j < p.E ? to_f32(src[j]) : 0.f;
  }
}

__device__ __forceinline__ void write_choice(const RouteParams& p, int64_t row, int lane, int id, float score) {
  if (lane < p.top_k) {
    p.weights[row * p.top_k + lane] = score;
    p.ids[row * p.top_k + lane] = id;
  }
}

// Any row: round by round, in fp32 where that decides, else in 64 bits.  Kept out of line so that the registers of the
// 64-bit form are not the fast kernel's.
template <typename T, int PER>
__device__ __noinline__ void route_slowly(const RouteParams& p, int64_t row, int lane, bool try_fp32) {
  float x[PER];
  load_logits<T, PER>(p, row, lane, false, x);
  int id = 0;
  float score = 0.f;
  if (!try_fp32 || !route_row<float, PER>(x, lane, p, id, score)) {  // (the whole warp agrees)
    double exact = 0.0;
    route_row<double, PER>(x, lane, p, id, exact);
    score = float(exact);
  }
  write_choice(p, row, lane, id, score);
}

__device__ __forceinline__ float rcp_f32(float v) {  // within 1 unit in the last place
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_max_f32(float v) {  // (skips NaNs)
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The usual row.  A NaN marks what is not there (maxima skip it, comparisons with it are false).
//
// The top_k-th largest of the 32 lanes' largest keys is no larger than the top_k-th largest key, so the keys that are not
// below it (by more than the tolerance) hold all that can be chosen; they are few, 12 or so for 8 of 256.  They move to one per lane, each
// counts those before it, and that is its place.  Against top_k rounds of a maximum over the row this is a third of the
// instructions, and instructions are what bounds it (a row of 256 fp32 logits is 1 KB of reads).
// Rows with more than 32 such keys, with group shapes that are not whole powers of two of lanes, or that fp32 does not decide
// go round by round.
template <typename T, int PER>
__global__ void __launch_bounds__(kRouteWarps * 32, 4) moe_route_kernel(const __grid_constant__ RouteParams p) {
  __shared__ float2 s_key[kRouteWarps][33];  // key and logit of the candidates, then of the choices in order
  __shared__ int s_id[kRouteWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * kRouteWarps + warp;
  if (row >= p.M) return;
  if (p.slow_groups) return route_slowly<T, PER>(p, row, lane, true);
  const float inf = __int_as_float(0x7f800000), nan = __int_as_float(0x7fffffff);
  const int e0 = lane * PER;
  const bool by_logit = p.bias == nullptr && !p.summed;
  float x[PER];
  load_logits<T, PER>(p, row, lane, p.wide, x);

  // keys
  float key[PER];
  float top = 0.f, share = 1.f;  // softmax: score = exp(x - top) * share
  if (p.softmax) {
    top = -inf;
#pragma unroll
    for (int j = 0; j < PER; ++j) top = fmaxf(top, e0 + j < p.E ? x[j] : -inf);
    top = warp_max_f32(top);
    if (top == inf || top == -inf) top = 0.f;
    float total = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      key[j] = __expf(x[j] - top);
      total += e0 + j < p.E ? key[j] : 0.f;
    }
    total = warp_sum(total);
    share = total == 0.f ? 1.f : rcp_f32(total);
  }
  if (by_logit) {
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = x[j];
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = p.softmax ? key[j] * share : rcp_f32(1.f + __expf(-x[j]));
    if (p.bias) {
      if (PER >= 4 && p.wide_bias) {
        if (e0 < p.E) {
#pragma unroll
          for (int j = 0; j < PER; j += 4) {
            const float4 b = __ldg(reinterpret_cast<const float4*>(p.bias + e0 + j));
            key[j] += b.x;
            if (PER >= 4) { key[j + 1 < PER ? j + 1 : 0] += b.y; key[j + 2 < PER ? j + 2 : 0] += b.z; key[j + 3 < PER ? j + 3 : 0] += b.w; }
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (e0 + j < p.E) key[j] += __ldg(p.bias + e0 + j);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) key[j] = e0 + j < p.E ? fmaxf(key[j], -inf) : nan;  // (a NaN key ranks with -infinity)
  // How far a key can be off: `off` plus `rel` of its size.  The hardware exponential adds as much to the softmax as the
  // argument's rounding does (route_row): 260 * 2^-24 of a score, which is at most `share`, the best one's.  A sigmoid p of x is off
  // by p (1 - p) (|x| + 4) + 4 p roundings of 2^-24, at most 5.4 of them.
  const float off = by_logit ? 0.f : (p.softmax ? 1.6e-5f * share : 1e-6f) + 1e-37f;
  const float rel = by_logit ? 0.f : 2.4e-7f;
  bool sure = true;

  bool in = e0 < p.E;
  if (p.groups > 1) {
    const int lanes = p.group_size / PER, g = lane / lanes;  // (whole groups of lanes, checked on the host)
    float a = -inf, b = -inf;  // the group's two largest keys
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      b = fmaxf(b, fminf(a, key[j]));
      a = fmaxf(a, key[j]);
    }
    for (int o = 1; o < lanes; o <<= 1) {
      const float a2 = __shfl_xor_sync(0xffffffffu, a, o), b2 = __shfl_xor_sync(0xffffffffu, b, o);
      b = fmaxf(fminf(a, a2), fmaxf(b, b2));
      a = fmaxf(a, a2);
    }
    const bool two = p.summed && p.group_size > 1;
    const float value = two ? fmaxf(a + b, -inf) : a;
    int rank = 0;
    for (int h = 0; h < p.groups; ++h) {
      const float other = __shfl_sync(0xffffffffu, value, h * lanes);
      rank += (other > value || (other == value && h < g)) ? 1 : 0;
    }
    const bool chosen = rank < p.topk_groups;
    if (!by_logit && p.topk_groups < p.groups) {
      const float slack = 2.f * off + rel * (fabsf(a) + (two ? fabsf(b) : 0.f) + fabsf(value));
      const float worst_in = -warp_max_f32(in && chosen ? slack - value : -inf);  // what the worst in and the best out can be
      const float best_out = warp_max_f32(in && !chosen ? value + slack : -inf);
      if (!(worst_in > best_out)) sure = false;
    }
    in = in && chosen;
  }

  // a bound from below on the top_k-th largest key
  float lane_top = nan;
  if (in) {
#pragma unroll
    for (int j = 0; j < PER; ++j) lane_top = fmaxf(lane_top, key[j]);
  }
  float floor_key = -inf;
  for (int i = 0; i < p.top_k; ++i) {
    const float m = warp_max_f32(lane_top);
    floor_key = m;
    if (m != m) break;  // fewer lanes than choices: every key that is there
    const uint32_t at = __ballot_sync(0xffffffffu, lane_top == m);
    if (lane == __ffs(at) - 1) lane_top = nan;
  }
  if (!by_logit) floor_key -= 2.1f * (off + rel * fabsf(floor_key));
  if (floor_key != floor_key) floor_key = -inf;  // (also -infinity less its own size)
  // the keys that are not below it, one per lane
  uint32_t picked = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) picked |= (in && key[j] >= floor_key) ? 1u << j : 0u;
  const int mine = __popc(picked);
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += t;
  }
  const int count = __shfl_sync(0xffffffffu, upto, 31);
  if (count > 32) return route_slowly<T, PER>(p, row, lane, true);
  int at = upto - mine;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if ((picked >> j) & 1u) {
      s_key[warp][at] = make_float2(key[j], x[j]);
      s_id[warp][at] = e0 + j;
      ++at;
    }
  }
  __syncwarp();
  const float2 kx = lane < count ? s_key[warp][lane] : make_float2(0.f, 0.f);
  const int id = lane < count ? s_id[warp][lane] : 0;
  const float k = kx.x;
  int rank = 0;  // list order is expert order: equal keys keep it
  for (int t = 0; t < count; ++t) {
    const float other = __shfl_sync(0xffffffffu, k, t);
    rank += (other > k || (other == k && t < lane)) ? 1 : 0;
  }
  __syncwarp();
  if (lane < count) {
    s_key[warp][rank] = kx;
    s_id[warp][rank] = id;
  }
  __syncwarp();
  const bool chosen = lane < p.top_k;
  const int best = chosen ? s_id[warp][lane] : 0;
  const float2 bx = chosen ? s_key[warp][lane] : make_float2(0.f, 0.f);
  if (!by_logit && chosen && lane + 1 < count) {
    const float next = s_key[warp][lane + 1].x;
    if (!(bx.x - next > 2.f * off + rel * (fabsf(bx.x) + fabsf(next)))) sure = false;
  }
  // the scores of the chosen alone, with the exponential that is right to two units in the last place
  float sc = p.softmax ? expf(bx.y - top) * share : __fdividef(1.f, 1.f + expf(-bx.y));
  if (p.renormalize) {
    float total = warp_sum(chosen ? sc : 0.f);
    if (total < 1e-30f) sure = false;  // scores that fp32 cannot hold
    sc = __fdiv_rn(sc, total);
  }
  if (!__all_sync(0xffffffffu, sure)) return route_slowly<T, PER>(p, row, lane, false);
  write_choice(p, row, lane, best, sc * p.scale);
}

template <typename T, int PER>
int launch_route_per(RouteParams p, cudaStream_t st) {
  const unsigned grid = unsigned((int64_t(p.M) + kRouteWarps - 1) / kRouteWarps);
  // lanes read whole words where every row starts on one and a lane has all of its experts or none
  const int word = PER * int(sizeof(T)) < 16 ? PER * int(sizeof(T)) : 16;
  p.wide = p.E % PER == 0 && reinterpret_cast<uintptr_t>(p.logits) % word == 0 && (p.ldl * int64_t(sizeof(T))) % word == 0;
  p.wide_bias = p.E % PER == 0 && reinterpret_cast<uintptr_t>(p.bias) % 16 == 0;
  const int lanes = p.group_size / PER;
  p.slow_groups = p.groups > 1 && (p.group_size % PER != 0 || (lanes & (lanes - 1)) != 0);
  moe_route_kernel<T, PER><<<grid, kRouteWarps * 32, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "moe_route launch");
}

template <typename T>
int launch_route(const RouteParams& p, cudaStream_t st) {
  const int per = (p.E + 31) / 32;
  if (per <= 1) return launch_route_per<T, 1>(p, st);
  if (per <= 2) return launch_route_per<T, 2>(p, st);
  if (per <= 4) return launch_route_per<T, 4>(p, st);
  if (per <= 8) return launch_route_per<T, 8>(p, st);
  if (per <= 16) return launch_route_per<T, 16>(p, st);
  return launch_route_per<T, 32>(p, st);
}

// ---------------------------------------------------------------------------
// Expert sort: a stable counting sort of the flat (token, choice) indices by expert, every expert's slots padded to whole
// blocks
// ---------------------------------------------------------------------------
// One cluster does it in one launch.  Its warps take consecutive pieces of the list.  Pass 1 counts each warp's experts in
// shared memory; prefix sums over a CTA's warps, over the cluster's CTAs (through distributed shared memory) and over the
// experts' padded sizes give every warp its first slot of every expert; pass 2 hands the slots out in list order.  A vote
// per bit of the expert ranks equal ones within a warp: match.any takes about 100 cycles for 32 different values, and with it the
// list of 131072 choices took 25 us, ... with votes.  No atomics decide an order: the list is the same every time.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kHeld = 16;
constexpr unsigned kNoExpert = 0xffffffffu;
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
  int32_t* base = count + p.E;                // [E] first slot of the expert that is this CTA's
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

  // experts of the piece's first kHeld steps stay in registers between the passes (all of it up to 131072 choices on eight CTAs)
  auto expert_of = [&](int i) {
    const unsigned x = i < hi ? unsigned(__ldg(p.ids + i)) - unsigned(p.first) : kNoExpert;
    return x < unsigned(p.E) ? x : kNoExpert;
  };
  unsigned held[kHeld];
#pragma unroll
  for (int s = 0; s < kHeld; ++s) held[s] = expert_of(lo + s * 32 + lane);
  for (int i = threadIdx.x; i < kSortWarps * p.E; i += kSortThreads) cnt[i] = 0;
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kHeld; ++s)
    if (held[s] != kNoExpert) atomicAdd(mine + held[s], 1);
  for (int i = lo + kHeld * 32 + lane; i < hi; i += 32) {
    const unsigned x = expert_of(i);
    if (x != kNoExpert) atomicAdd(mine + x, 1);
  }
  __syncthreads();
  const int e = threadIdx.x;
  if (e < p.E) {
    int t[kSortWarps];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) t[w] = cnt[w * p.E + e];
    int run = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      cnt[w * p.E + e] = run;
      run += t[w];
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
    base[e] = start + before;
  }
  if (rank == 0 && threadIdx.x == 0) *p.num_post_padded = in_use;
  __syncthreads();

  const int bits = 32 - __clz(p.E - 1 > 0 ? p.E - 1 : 0);
  auto hand_out = [&](unsigned x, int i) {
    const bool here = x != kNoExpert;
    uint32_t same = __ballot_sync(0xffffffffu, here);
    for (int b = 0; b < bits; ++b) {
      const uint32_t one = __ballot_sync(0xffffffffu, (x >> b) & 1u);
      same &= ((x >> b) & 1u) ? one : ~one;
    }
    const int ahead = __popc(same & ((1u << lane) - 1u));
    int next = 0;
    if (here) next = mine[x];
    __syncwarp();
    if (here && ahead == 0) mine[x] = next + __popc(same);
    __syncwarp();
    if (here) p.sorted[base[x] + next + ahead] = i;
  };
#pragma unroll
  for (int s = 0; s < kHeld; ++s)
    if (lo + s * 32 < hi) hand_out(held[s], lo + s * 32 + lane);
  for (int i = lo + kHeld * 32; i < hi; i += 32) hand_out(expert_of(i + lane), i + lane);
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
  const size_t smem = size_t(kSortWarps + 4) * size_t(E) * sizeof(int32_t);
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  int dev = 0;
  cudaGetDevice(&dev);
  dev &= 63;
  std::call_once(once[dev], [&] {
    attr_err[dev] = cudaFuncSetAttribute(moe_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kSortWarps + 4) * kSortMaxExperts * 4);
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
