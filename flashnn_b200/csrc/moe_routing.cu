// The two ends of a mixture-of-experts layer: from router logits to the expert-sorted slot list that the expert products
// read, and from their [M, top_k, N] output back to [M, N].
#include <cooperative_groups.h>

#include <mutex>
#include <type_traits>
#include <utility>

#include "common.cuh"
#include "quantise.cuh"

namespace cg = cooperative_groups;

namespace fnn {
namespace {

// ---------------------------------------------------------------------------
// Routing: scores, balancing bias, group-limited choice, top-k, renormalised weights
// ---------------------------------------------------------------------------
// General form, one warp per token, the row in registers: lane l holds experts l * PER .. l * PER + PER - 1, so that lane order is
// expert order and the lowest lane among equals holds the lowest expert.  Every lane sorts its keys (an odd-even merge network of
// minima and maxima, without the experts' numbers), and top_k rounds take the largest of the 32 heads; the lane it came from
// moves on to its next key.  A choice's expert is found afterwards, as the place of its value among that lane's unsorted keys.
// Instructions bound the kernel (a row of 256 fp32 logits is 1 KB of reads).
//
// Which experts are chosen, and in what order, is defined in 64 bits.  Where the keys are the logits themselves (no bias,
// no sum over a group: both scores grow with the logit) comparing them is exact.  Elsewhere the row is done in fp32 first,
// with a bound on how far a key can be off; only where two keys that decide something are nearer than that (a row in some
// hundreds) is the row done again in 64 bits, after the warp's others, so that the registers of the 64-bit form are not the
// usual row's.
struct RouteParams {
  const void* logits;
  const float* bias;  // nullptr or [E]
  float* weights;     // [M, top_k]
  int32_t* ids;       // [M, top_k]
  int64_t ldl;
  int M, E, top_k, groups, topk_groups, group_size;
  int softmax, renormalize, summed;  // summed: a group's score is the sum of its two largest keys, else its largest
  float scale;
  int wide;        // lanes read whole words (set by the launch)
  int whole_lanes; // a group is a power of two of lanes with all of their experts (set by the launch)
  int used;        // experts of a lane in the kernel with several tokens per warp, and whether its 64-bit form reads whole words
  int wide_64;
};

// maxima and minima that skip a NaN, which marks what is not there
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float smaller(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ double larger(double a, double b) { return fmax(a, b); }
__device__ __forceinline__ double smaller(double a, double b) { return fmin(a, b); }
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ double warp_max(double v) {
  // order-preserving map to unsigned integers, 0 for a NaN; the upper words' maximum, then the lower words' among those
  v += 0.0;  // (-0 -> +0)
  unsigned long long o = __double_as_longlong(v);
  o = v != v ? 0ull : (o >> 63) ? ~o : o | 0x8000000000000000ull;
  const uint32_t hi = __reduce_max_sync(0xffffffffu, uint32_t(o >> 32));
  const uint32_t lo = __reduce_max_sync(0xffffffffu, uint32_t(o >> 32) == hi ? uint32_t(o) : 0u);
  o = (static_cast<unsigned long long>(hi) << 32) | lo;
  if (o == 0ull) return __longlong_as_double(0x7fffffffffffffffll);
  return __longlong_as_double((o >> 63) ? o & 0x7fffffffffffffffull : ~o);
}
template <typename F> __device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// e^v of the keys: in fp32 by the hardware's 2^v, within (|v| + 4) roundings of 2^-24, 0 where that is subnormal
__device__ __forceinline__ float key_exp(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ double key_exp(double v) { return exp(v); }
__device__ __forceinline__ float reciprocal(float v) {  // within 1 unit in the last place
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ double reciprocal(double v) { return 1.0 / v; }
__device__ __forceinline__ float full_exp(float v) { return expf(v); }
__device__ __forceinline__ double full_exp(double v) { return exp(v); }

// odd-even merge network: with runs of P sorted, partners K apart within runs of 2 P
template <int P, int K, int I, typename F, int N> __device__ __forceinline__ void compare_exchange(F (&v)[N]) {
  if constexpr (I + K < N && I >= K % P && ((I - K % P) / K) % 2 == 0 && I / (2 * P) == (I + K) / (2 * P)) {
    const F a = larger(v[I], v[I + K]), b = smaller(v[I], v[I + K]);
    v[I] = a;
    v[I + K] = b;
  }
}
template <int P, int K, typename F, int N, int... I>
__device__ __forceinline__ void merge_step(F (&v)[N], std::integer_sequence<int, I...>) {
  (compare_exchange<P, K, I>(v), ...);
}
template <int P, int K, typename F, int N> __device__ __forceinline__ void merge_runs(F (&v)[N]) {
  merge_step<P, K>(v, std::make_integer_sequence<int, N>());
  if constexpr (K > 1) merge_runs<P, K / 2>(v);
}
template <int P = 1, typename F, int N> __device__ __forceinline__ void sort_descending(F (&v)[N]) {
  if constexpr (P < N) {
    merge_runs<P, P>(v);
    sort_descending<2 * P>(v);
  }
}

// sorts a bitonic sequence
template <int K, typename F, int N, int... I>
__device__ __forceinline__ void bitonic_step(F (&v)[N], std::integer_sequence<int, I...>) {
  auto one = [&](auto index) {
    constexpr int i = decltype(index)::value;
    if constexpr ((i & K) == 0) {
      const F a = larger(v[i], v[i + K]), b = smaller(v[i], v[i + K]);
      v[i] = a;
      v[i + K] = b;
    }
  };
  (one(std::integral_constant<int, I>()), ...);
}
template <int K, typename F, int N> __device__ __forceinline__ void merge_bitonic(F (&v)[N]) {
  if constexpr (K >= 1) {
    bitonic_step<K>(v, std::make_integer_sequence<int, N>());
    merge_bitonic<K / 2>(v);
  }
}

// A lane's PER logits; absent ones read as 0.
template <typename T> __device__ __forceinline__ void load_word(const T* src, bool on, float (&x)[4]) {
  if constexpr (sizeof(T) == 4) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on) v = *reinterpret_cast<const float4*>(src);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
  } else {
    uint2 v = make_uint2(0u, 0u);
    if (on) v = *reinterpret_cast<const uint2*>(src);
    x[0] = lo_of<T>(v.x); x[1] = hi_of<T>(v.x); x[2] = lo_of<T>(v.y); x[3] = hi_of<T>(v.y);
  }
}
template <typename T, int PER>
__device__ __forceinline__ void load_logits(const RouteParams& p, int64_t row, int lane, bool wide, float (&x)[PER]) {
  const T* src = reinterpret_cast<const T*>(p.logits) + row * p.ldl + lane * PER;
  if (PER >= 4 && wide) {
    const bool on = lane * PER < p.E;
#pragma unroll
    for (int w = 0; w < PER; w += 4) {
      float v[4];
      load_word(src + w, on, v);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w + j < PER) x[w + j] = v[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = lane * PER + j < p.E ? to_f32(src[j]) : 0.f;
  }
}

// One row in arithmetic F; writes the choices, or returns false where fp32 does not decide.  s_bias: the biases in shared memory, 0
// behind the last; s_keys: this warp's [PER][32] words of shared memory.
template <typename F, typename T, int PER>
__device__ __forceinline__ bool route_row(const RouteParams& p, const float (&x)[PER], int64_t row, int lane, const float* s_bias, F* s_keys) {
  constexpr bool kExact = sizeof(F) == 8;
  constexpr uint32_t kAll = 0xffffffffu;
  const F inf = F(__int_as_float(0x7f800000)), nan = F(__int_as_float(0x7fffffff));
  const int e0 = lane * PER;
  const bool by_logit = p.bias == nullptr && !p.summed;
  const bool check = !kExact && !by_logit;
  // the lane's experts that can be chosen, one bit each
  const int present = min(max(p.E - e0, 0), PER);
  uint32_t real = present == 32 ? kAll : (1u << present) - 1u;

  // keys
  F key[PER];
  F top = F(0), share = F(1);  // softmax: score = exp(x - top) * share
  if (p.softmax) {
    top = -inf;
#pragma unroll
    for (int j = 0; j < PER; ++j) top = larger(top, j < present ? F(x[j]) : -inf);
    top = warp_max(top);
    if (top == inf || top == -inf) top = F(0);
    F total = F(0);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      key[j] = key_exp(F(x[j]) - top);
      total += j < present ? key[j] : F(0);
    }
    total = warp_sum(total);
    share = total == F(0) ? F(1) : reciprocal(total);
    if (!by_logit) {
#pragma unroll
      for (int j = 0; j < PER; ++j) key[j] = kExact ? key[j] / (total == F(0) ? F(1) : total) : key[j] * share;
    }
  } else if (!by_logit) {
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = reciprocal(F(1) + key_exp(-F(x[j])));
  }
  if (by_logit) {
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = F(x[j]);
  } else if (p.bias) {
    if constexpr (PER >= 4) {
#pragma unroll
      for (int j = 0; j < PER; j += 4) {
        const float4 b = *reinterpret_cast<const float4*>(s_bias + e0 + j);
        key[j] += F(b.x); key[j + 1] += F(b.y); key[j + 2] += F(b.z); key[j + 3] += F(b.w);
      }
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) key[j] += F(s_bias[e0 + j]);
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) key[j] = j < present ? larger(key[j], -inf) : -inf;  // (a NaN key ranks with -infinity)
  // How far an fp32 key can be off: `off` plus `rel` of its size.  A softmax score's argument is rounded by 2^-24 of up to 104
  // (beyond that it is 0), the hardware exponential adds as much and the sum one rounding per addition (37 in a row): at most
  // 2 * 104 + 50 roundings of 2^-24 of the score, which is at most `share`, the best one's.  A sigmoid q of x is off by
  // q (1 - q) (|x| + 4) + 4 q such roundings, at most 5.4.
  const F off = check ? (p.softmax ? F(1.6e-5f) * share : F(3.4e-7f)) + F(1e-37f) : F(0);
  const F rel = check ? F(1.2e-7f) : F(0);
  bool sure = true;

  if (p.groups > 1) {
    const bool two = p.summed && p.group_size > 1;
    F a = -inf, b = -inf;  // the two largest keys: of this lane's group, or (below) of group `lane`
    int g, lanes = 1;      // group h's are in lane h * lanes
    if (p.whole_lanes) {
      lanes = p.group_size / PER;
      g = lane / lanes;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        b = larger(b, smaller(a, key[j]));
        a = larger(a, key[j]);
      }
      for (int o = 1; o < lanes; o <<= 1) {
        const F a2 = __shfl_xor_sync(kAll, a, o), b2 = __shfl_xor_sync(kAll, b, o);
        b = larger(smaller(a, a2), larger(b, b2));
        a = larger(a, a2);
      }
    } else {
      g = lane;
      for (int h = 0; h < p.groups; ++h) {
        const int lo = h * p.group_size - e0, hi = lo + p.group_size;
        F a1 = -inf, b1 = -inf;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
          const F v = j >= lo && j < hi ? key[j] : -inf;
          b1 = larger(b1, smaller(a1, v));
          a1 = larger(a1, v);
        }
        const F first = warp_max(a1);
        const int src = __ffs(__ballot_sync(kAll, a1 == first)) - 1;
        const F second = warp_max(lane == src ? b1 : a1);
        if (lane == h) { a = first; b = second; }
      }
    }
    const F value = two ? larger(a + b, -inf) : a;
    int rank = 0;
#pragma unroll 4
    for (int h = 0; h < p.groups; ++h) {
      const F other = __shfl_sync(kAll, value, h * lanes);
      rank += (other > value || (other == value && h < g)) ? 1 : 0;
    }
    const bool valid = g < p.groups, chosen = rank < p.topk_groups;
    if (check && p.topk_groups < p.groups) {
      const F slack = F(2) * off + rel * (fabsf(a) + (two ? fabsf(b) : F(0)) + fabsf(value));
      const F worst_in = -warp_max(valid && chosen ? slack - value : -inf);  // what the worst in and the best out can be
      const F best_out = warp_max(valid && !chosen ? value + slack : -inf);
      if (!(worst_in > best_out)) sure = false;
    }
    if (p.whole_lanes) {
      if (!chosen) real = 0;
    } else {
      const uint32_t in = __ballot_sync(kAll, valid && chosen);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (j < present && !((in >> ((e0 + j) / p.group_size)) & 1u)) {
          real &= ~(1u << j);
          key[j] = -inf;
        }
    }
  }

  // rounds
  F sorted[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) sorted[j] = key[j];
  sort_descending(sorted);
  const int mine = __popc(real);  // what cannot be chosen has sunk to the end
  F* list = s_keys + lane;  // [PER][32]
#pragma unroll
  for (int j = 0; j < PER; ++j) list[j * 32] = sorted[j];
  F head = mine > 0 ? sorted[0] : nan;
  int at = 0;
  F value = F(0);         // of this lane's choice (lane top_k: of the first one left out, which shows how near it is)
  int from = 0;           // the lane it came from
  F last = F(0);
  bool repeated = false;  // two choices have the same key
  bool extra = false;     // there is one left out
  const int rounds = check ? p.top_k + 1 : p.top_k;
  for (int i = 0; i < rounds; ++i) {
    const F m = warp_max(head);
    if (m != m) break;  // (only the extra round can find nothing)
    extra = i == p.top_k;
    const int src = __ffs(__ballot_sync(kAll, head == m)) - 1;
    repeated |= i > 0 && m == last;
    last = m;
    value = lane == i ? m : value;
    from = lane == i ? src : from;
    at += lane == src ? 1 : 0;
    const F next = list[min(at, PER - 1) * 32];
    head = lane != src ? head : at < mine ? next : nan;
  }
  if (check) {
    const F next = __shfl_down_sync(kAll, value, 1);
    if (lane < p.top_k && (extra || lane + 1 < p.top_k) && !(value - next > F(2) * off + rel * (fabsf(value) + fabsf(next)))) sure = false;
    if (!__all_sync(kAll, sure)) return false;
  }

  // the choice's expert: the first of that lane's experts with this key that no choice before it took
  uint32_t equal = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) equal |= __shfl_sync(kAll, key[j], from) == value ? 1u << j : 0u;
  equal &= __shfl_sync(kAll, real, from);
  if (repeated) {
    for (int i = 0; i + 1 < p.top_k; ++i) {
      const F v = __shfl_sync(kAll, value, i);
      const int src = __shfl_sync(kAll, from, i);
      if (i < lane && v == value && src == from) equal &= equal - 1u;
    }
  }
  const bool chosen = lane < p.top_k;
  const int id = from * PER + (chosen ? __ffs(equal) - 1 : 0);
  // the chosen ones' scores, with the full exponential
  F score = F(0);
  if (chosen) {
    const F v = F(to_f32(reinterpret_cast<const T*>(p.logits)[row * p.ldl + id]));
    score = p.softmax ? full_exp(v - top) * share : F(1) / (F(1) + full_exp(-v));
  }
  if (p.renormalize) {
    F total = warp_sum(score);
    if (!kExact && total < F(1e-30f)) return false;  // scores that fp32 cannot hold
    score /= total == F(0) ? F(1) : total;
  }
  if (chosen) {
    p.weights[row * p.top_k + lane] = float(score * F(p.scale));
    p.ids[row * p.top_k + lane] = id;
  }
  return true;
}

template <typename T, int PER>
__device__ __noinline__ void route_row_64(const RouteParams& p, int64_t row, int lane, const float* s_bias, double* s_keys) {
  float x[PER];
  load_logits<T, PER>(p, row, lane, p.wide_64 != 0, x);
  route_row<double, T, PER>(p, x, row, lane, s_bias, s_keys);
}

constexpr int kPutOff = 8;  // rows a warp puts off before it goes through them in 64 bits

// Warps take rows in turn and load the next row's logits before they work on this one's.
template <typename T, int PER, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 24 / WARPS) moe_route_kernel(const __grid_constant__ RouteParams p) {
  __shared__ double s_keys[WARPS][32 * PER];  // (the fp32 rows use half)
  __shared__ float4 s_bias4[PER * 8];
  __shared__ int64_t s_put_off[WARPS][kPutOff];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* s_bias = reinterpret_cast<float*>(s_bias4);
  if (p.bias) {
    for (int e = threadIdx.x; e < 32 * PER; e += WARPS * 32) s_bias[e] = e < p.E ? __ldg(p.bias + e) : 0.f;
    __syncthreads();
  }
  const int64_t step = int64_t(gridDim.x) * WARPS;
  int64_t row = int64_t(blockIdx.x) * WARPS + warp;
  while (row < p.M) {
    int put_off = 0;
    float x[PER];
    load_logits<T, PER>(p, row, lane, p.wide != 0, x);
    while (true) {
      const int64_t next = row + step;
      float ahead[PER];
      if (next < p.M) load_logits<T, PER>(p, next, lane, p.wide != 0, ahead);
      if (!route_row<float, T, PER>(p, x, row, lane, s_bias, reinterpret_cast<float*>(s_keys[warp]))) s_put_off[warp][put_off++] = row;
      row = next;
      if (row >= p.M || put_off == kPutOff) break;
#pragma unroll
      for (int j = 0; j < PER; ++j) x[j] = ahead[j];
    }
    __syncwarp();
    for (int i = 0; i < put_off; ++i) route_row_64<T, PER>(p, s_put_off[warp][i], lane, s_bias, s_keys[warp]);
    __syncwarp();
  }
}

// The usual shapes: top_k <= 16.  W lanes per token (several tokens per warp), lane s of them with experts s * used .. s * used + used - 1, used <= PER, in
// registers, so that a group is whole lanes.  What the one-warp kernel spends on its rounds (37 instructions each) goes into networks of minima and maxima that
// need no expert numbers: a lane sorts its keys eight (or 16) at a time and merges them into its eight largest, a butterfly merges the lanes',
// and the top_k-th of the result is all that is kept.  The keys that are not below it, less the tolerance, are the candidates,
// top_k of them and rarely more; in a list, in expert order, each counts those before it, and that is its place.
// 16384 tokens x 256 experts in groups, fp32 logits: one warp per token 980 instructions a row and 28 us, this kernel 460 and 17 us.
// Where fp32 does not decide, the two comparisons that can be in doubt (between groups, between candidates) are made in 64
// bits here, in little code: the whole row in 64 bits costs a launch 8 us, most of it fetching instructions that no other row has run.
// A row with more candidates than the list holds, or too few keys above -infinity, goes to the general form.
template <typename F, int N> __device__ __forceinline__ void merge_largest(F (&a)[N], const F (&b)[N]) {  // both sorted; a becomes the N largest
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = larger(a[i], b[N - 1 - i]);  // (a bitonic sequence)
  merge_bitonic<N / 2>(a);
}

// LIST: largest keys that a lane keeps, 8 or 16, at least top_k; the list of candidates holds twice as many.
template <typename T, int PER, int W, int LIST, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, (LIST == 8 ? 28 : 20) / WARPS) moe_route_lists_kernel(const __grid_constant__ RouteParams p) {
  static_assert(LIST <= W, "a lane for every choice");
  constexpr uint32_t kAll = 0xffffffffu;
  constexpr int kListCap = 2 * LIST;
  constexpr int kRows = 32 / W;  // tokens a warp works on
  __shared__ double s_keys[WARPS][W * PER <= 256 ? 256 : W * PER];  // for the rows that were put off (one warp per row: 32 lanes)
  __shared__ float4 s_bias4[W * PER / 4], s_lane_bias4[W * PER / 4];  // by expert, and by lane (PER words each)
  __shared__ alignas(16) float s_key[WARPS][kRows][kListCap];
  __shared__ float s_x[WARPS][kRows][kListCap];
  __shared__ int s_id[WARPS][kRows][kListCap];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % W, mine = lane / W;
  float *s_bias = reinterpret_cast<float*>(s_bias4), *s_lane_bias = reinterpret_cast<float*>(s_lane_bias4);
  if (p.bias) {
    for (int i = threadIdx.x; i < W * PER; i += WARPS * 32) {
      const int e = i / PER * p.used + i % PER;
      s_bias[i] = i < p.E ? __ldg(p.bias + i) : 0.f;
      s_lane_bias[i] = i % PER < p.used && e < p.E ? __ldg(p.bias + e) : 0.f;
    }
    __syncthreads();
  }
  const float inf = __int_as_float(0x7f800000);
  const int64_t row = (int64_t(blockIdx.x) * WARPS + warp) * kRows + mine;
  const bool live = row < p.M;
  const int e0 = sub * p.used;
  const bool by_logit = p.bias == nullptr && !p.summed;
  const int present = min(max(p.E - e0, 0), p.used);

  float key[PER];
  const T* src = reinterpret_cast<const T*>(p.logits) + (live ? row : 0) * p.ldl;
  {
    if (p.wide) {
#pragma unroll
      for (int w = 0; w < PER; w += 4) {
        float v[4];
        load_word(src + e0 + w, w < present, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) key[w + j] = v[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) key[j] = j < present ? to_f32(src[e0 + j]) : 0.f;
    }
  }
  auto across_max = [&](float v) {
#pragma unroll
    for (int o = 1; o < W; o <<= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
    return v;
  };
  auto across_sum = [&](float v) {
#pragma unroll
    for (int o = 1; o < W; o <<= 1) v += __shfl_xor_sync(kAll, v, o);
    return v;
  };
  // logits -> keys, the same arithmetic as route_row<float>
  float top = 0.f, share = 1.f;
  auto key_of = [&](float x, int e) {
    if (by_logit) return x;
    float k = p.softmax ? key_exp(x - top) * share : reciprocal(1.f + key_exp(-x));
    if (p.bias) k += s_bias[e];
    return k;
  };
  if (p.softmax) {
    top = -inf;
#pragma unroll
    for (int j = 0; j < PER; ++j) top = fmaxf(top, j < present ? key[j] : -inf);
    top = across_max(top);
    if (top == inf || top == -inf) top = 0.f;
    float total = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) total += j < present ? key_exp(key[j] - top) : 0.f;
    total = across_sum(total);
    share = total == 0.f ? 1.f : reciprocal(total);
  }
  if (!by_logit) {
    if (p.softmax) {
#pragma unroll
      for (int j = 0; j < PER; ++j) key[j] = key_exp(key[j] - top) * share;
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) key[j] = reciprocal(1.f + key_exp(-key[j]));
    }
    if (p.bias) {
#pragma unroll
      for (int j = 0; j < PER; j += 4) {
        const float4 b = *reinterpret_cast<const float4*>(s_lane_bias + sub * PER + j);
        key[j] += b.x; key[j + 1] += b.y; key[j + 2] += b.z; key[j + 3] += b.w;
      }
    }
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) key[j] = fmaxf(key[j], -inf);  // (a NaN key ranks with -infinity)
  if (present < PER) {
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = j < present ? key[j] : -inf;
  }
  const bool check = !by_logit;
  const float off = check ? (p.softmax ? 1.6e-5f * share : 3.4e-7f) + 1e-37f : 0.f;  // how far a key can be off, see route_row
  const float rel = check ? 1.2e-7f : 0.f;
  bool in = present > 0;
  // the same in 64 bits, where fp32 does not decide
  double total_64 = 0.0;
  auto need_total_64 = [&]() {
    if (!p.softmax || total_64 != 0.0) return;
#pragma unroll 2
    for (int j = 0; j < PER; ++j) total_64 += j < present ? exp(double(to_f32(src[e0 + j])) - double(top)) : 0.0;
#pragma unroll
    for (int o = 1; o < W; o <<= 1) total_64 += __shfl_xor_sync(kAll, total_64, o);
    if (total_64 == 0.0) total_64 = 1.0;
  };
  auto score_64 = [&](float v) {
    const double z = exp(p.softmax ? double(v) - double(top) : -double(v));
    return p.softmax ? z / total_64 : 1.0 / (1.0 + z);
  };

  if (p.groups > 1) {
    // (groups are whole lanes, a power of two of them: checked on the host)
    const int lanes = p.group_size / p.used, g = sub / lanes;
    const bool two = p.summed && p.group_size > 1;
    float a = -inf, b = -inf;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      b = fmaxf(b, fminf(a, key[j]));
      a = fmaxf(a, key[j]);
    }
    for (int o = 1; o < lanes; o <<= 1) {
      const float a2 = __shfl_xor_sync(kAll, a, o), b2 = __shfl_xor_sync(kAll, b, o);
      b = fmaxf(fminf(a, a2), fmaxf(b, b2));
      a = fmaxf(a, a2);
    }
    const float value = two ? fmaxf(a + b, -inf) : a;
    auto rank_of = [&](auto v) {
      int rank = 0;
#pragma unroll 4
      for (int h = 0; h < p.groups; ++h) {
        const auto other = __shfl_sync(kAll, v, mine * W + h * lanes);
        rank += (other > v || (other == v && h < g)) ? 1 : 0;
      }
      return rank;
    };
    bool chosen = rank_of(value) < p.topk_groups;
    if (check && p.topk_groups < p.groups) {
      const float slack = 2.f * off + rel * (fabsf(a) + (two ? fabsf(b) : 0.f) + fabsf(value));
      const float worst_in = -across_max(in && chosen ? slack - value : -inf);  // what the worst in and the best out can be
      const float best_out = across_max(in && !chosen ? value + slack : -inf);
      if (__any_sync(kAll, live && !(worst_in > best_out))) {
        need_total_64();
        const float near = (two ? b : a) - 2.1f * (off + rel * fabsf(two ? b : a));  // keys that can be among the group's two largest
        uint32_t maybe = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) maybe |= (j < present && !(key[j] < near)) ? 1u << j : 0u;
        double a64 = -double(inf), b64 = -double(inf);
        for (; __any_sync(kAll, maybe != 0); maybe &= maybe - 1u) {
          if (maybe != 0) {
            const int e = e0 + __ffs(maybe) - 1;
            double v = score_64(to_f32(src[e]));
            if (p.bias) v += double(s_bias[e]);
            if (v > a64) { b64 = a64; a64 = v; }
            else if (v > b64) b64 = v;
          }
        }
        for (int o = 1; o < lanes; o <<= 1) {
          const double a2 = __shfl_xor_sync(kAll, a64, o), b2 = __shfl_xor_sync(kAll, b64, o);
          const double lesser = a2 > a64 ? a64 : a2;
          b64 = b2 > b64 ? b2 : b64;
          b64 = lesser > b64 ? lesser : b64;
          a64 = a2 > a64 ? a2 : a64;
        }
        chosen = rank_of(two ? larger(a64 + b64, -double(inf)) : a64) < p.topk_groups;
      }
    }
    in = in && chosen;
  }

  // the top_k-th largest key
  constexpr int kRun = PER < LIST ? PER : LIST;  // keys sorted at a time
  float best[LIST];
  {
    float run[kRun];
#pragma unroll
    for (int j = 0; j < kRun; ++j) run[j] = key[j];
    sort_descending(run);
#pragma unroll
    for (int j = 0; j < LIST; ++j) best[j] = j < kRun && in ? run[j < kRun ? j : 0] : -inf;
  }
  if constexpr (PER > LIST) {
#pragma unroll
    for (int c = LIST; c < PER; c += LIST) {
      float run[LIST];
#pragma unroll
      for (int j = 0; j < LIST; ++j) run[j] = in ? key[c + j] : -inf;
      sort_descending(run);
      merge_largest(best, run);
    }
  }
#pragma unroll
  for (int o = 1; o < W; o <<= 1) {
    float other[LIST];
#pragma unroll
    for (int j = 0; j < LIST; ++j) other[j] = __shfl_xor_sync(kAll, best[j], o);
    merge_largest(best, other);
  }
  float least = best[0];
#pragma unroll
  for (int j = 1; j < LIST; ++j) least = j < p.top_k ? best[j] : least;
  if (check) least -= 2.1f * (off + rel * fabsf(least));
  bool odd = !(least > -inf);  // fewer keys than choices above -infinity: the general form knows what is there

  // candidates, in expert order
  uint32_t picked = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) picked |= key[j] >= least ? 1u << j : 0u;
  if (!in || !live) picked = 0;
  int upto = __popc(picked);
#pragma unroll
  for (int o = 1; o < W; o <<= 1) {
    const int t = __shfl_up_sync(kAll, upto, o);
    if (sub >= o) upto += t;
  }
  const int count = __shfl_sync(kAll, upto, mine * W + W - 1);
  int at = upto - __popc(picked);
  if (count > kListCap) odd = true;
  if (odd) picked = 0;
  while (__any_sync(kAll, picked != 0)) {
    if (picked != 0) {
      const int j = __ffs(picked) - 1;
      picked &= picked - 1u;
      const float x = to_f32(src[e0 + j]);
      s_key[warp][mine][at] = fmaxf(key_of(x, e0 + j), -inf);
      s_x[warp][mine][at] = x;
      s_id[warp][mine][at] = e0 + j;
      ++at;
    }
  }
  __syncwarp();
  // every lane counts those before its candidates sub and sub + LIST; then lane s holds choice s
  const int listed = odd ? 0 : count;
  float cx[2], ck[2];
  int place[2], cid[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int t = sub + LIST * c;
    const bool on = sub < LIST && t < listed;
    ck[c] = on ? s_key[warp][mine][t] : 0.f;
    cx[c] = on ? s_x[warp][mine][t] : 0.f;
    cid[c] = on ? s_id[warp][mine][t] : 0;
    place[c] = on ? 0 : kListCap;
  }
  const bool more = __any_sync(kAll, listed > LIST);
#pragma unroll 2
  for (int t = 0; t < (more ? kListCap : LIST); ++t) {
    const float other = t < listed ? s_key[warp][mine][t] : -inf;
#pragma unroll
    for (int c = 0; c < 2; ++c) place[c] += (other > ck[c] || (other == ck[c] && t < sub + LIST * c && t < listed)) ? 1 : 0;
  }
  bool chosen = false;
  float k = 0.f, x = 0.f;
  auto in_order = [&]() {
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      if (place[c] < kListCap) {
        s_key[warp][mine][place[c]] = ck[c];
        s_x[warp][mine][place[c]] = cx[c];
        s_id[warp][mine][place[c]] = cid[c];
      }
    }
    __syncwarp();
    chosen = sub < p.top_k && sub < listed;
    k = chosen ? s_key[warp][mine][sub] : 0.f;
    x = chosen ? s_x[warp][mine][sub] : 0.f;
  };
  in_order();
  if (check) {
    const float next = chosen && sub + 1 < listed ? s_key[warp][mine][sub + 1] : -inf;
    if (__any_sync(kAll, live && chosen && sub + 1 < listed && !(k - next > 2.f * off + rel * (fabsf(k) + fabsf(next))))) {
      need_total_64();
      double k64[2];
#pragma unroll 1
      for (int c = 0; c < 2; ++c) {
        const double v = score_64(c == 0 ? cx[0] : cx[1]) + (p.bias ? double(s_bias[c == 0 ? cid[0] : cid[1]]) : 0.0);
        if (c == 0) k64[0] = larger(v, -double(inf));
        else k64[1] = larger(v, -double(inf));
        if (!more) break;
      }
      if (!more) k64[1] = 0.0;
      place[0] = sub < LIST && sub < listed ? 0 : kListCap;
      place[1] = sub < LIST && sub + LIST < listed ? 0 : kListCap;
#pragma unroll 1
      for (int t = 0; t < kListCap; ++t) {
        const double other = __shfl_sync(kAll, t < LIST ? k64[0] : k64[1], mine * W + t % LIST);
        if (t < listed) {
#pragma unroll
          for (int c = 0; c < 2; ++c) place[c] += (other > k64[c] || (other == k64[c] && t < sub + LIST * c)) ? 1 : 0;
        }
      }
      in_order();
    }
  }
  float score = 0.f;
  if (chosen) score = p.softmax ? expf(x - top) * share : __fdividef(1.f, 1.f + expf(-x));
  if (p.renormalize) {
    const float total = across_sum(score);
    if (__any_sync(kAll, live && !odd && total < 1e-30f)) {  // scores that fp32 cannot hold
      need_total_64();
      const double exact = chosen ? score_64(x) : 0.0;
      double sum = exact;
#pragma unroll
      for (int o = 1; o < W; o <<= 1) sum += __shfl_xor_sync(kAll, sum, o);
      score = float(exact / (sum == 0.0 ? 1.0 : sum));
    } else {
      score = __fdividef(score, total);
    }
  }
  if (chosen && live) {
    p.weights[row * p.top_k + sub] = score * p.scale;
    p.ids[row * p.top_k + sub] = s_id[warp][mine][sub];
  }
  const uint32_t again = __ballot_sync(kAll, odd && live);
#pragma unroll 1
  for (int r = 0; r < kRows; ++r) {
    if ((again >> (r * W)) & 1u) {
      __syncwarp();
      route_row_64<T, (W * PER + 31) / 32>(p, (int64_t(blockIdx.x) * WARPS + warp) * kRows + r, lane, s_bias, s_keys[warp]);
    }
  }
}

// Experts of a lane (at most per), so that a group is a power of two of whole lanes and all fit in w of them; 0 if there is no such number.
inline int lane_experts(const RouteParams& p, int per, int w) {
  if (p.groups == 1) return p.E <= per * w ? per : 0;
  for (int lanes = 1; p.groups * lanes <= w; lanes *= 2)
    if (p.group_size % lanes == 0 && p.group_size / lanes <= per) return p.group_size / lanes;
  return 0;
}

template <typename T, int PER, int W, int LIST>
bool launch_route_lists(RouteParams p, cudaStream_t st, int& status) {
  constexpr int kWarps = 4, kPer64 = (W * PER + 31) / 32;
  const int64_t rows = kWarps * (32 / W);
  p.used = lane_experts(p, PER, W);
  if (p.used == 0) return false;
  p.wide = p.E % 4 == 0 && p.used % 4 == 0 && reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && (p.ldl * int64_t(sizeof(T))) % 16 == 0;
  const int lanes = p.group_size / kPer64;  // (of the 64-bit form)
  p.whole_lanes = p.group_size % kPer64 == 0 && (lanes & (lanes - 1)) == 0;
  p.wide_64 = p.wide && p.E % kPer64 == 0;
  moe_route_lists_kernel<T, PER, W, LIST, kWarps><<<unsigned((p.M + rows - 1) / rows), kWarps * 32, 0, st>>>(p);
  status = check_cuda(cudaGetLastError(), "moe_route launch");
  return true;
}

template <typename T, int PER>
int launch_route_per(RouteParams p, cudaStream_t st) {
  constexpr int kWarps = PER >= 32 ? 4 : 8;
  // lanes read whole words where every row starts on one and a lane has all of its experts or none
  const bool full = p.E % PER == 0;
  const int word = PER * int(sizeof(T)) < 16 ? PER * int(sizeof(T)) : 16;
  p.wide = full && reinterpret_cast<uintptr_t>(p.logits) % word == 0 && (p.ldl * int64_t(sizeof(T))) % word == 0;
  p.wide_64 = p.wide;
  const int lanes = p.group_size / PER;
  p.whole_lanes = p.group_size % PER == 0 && (lanes & (lanes - 1)) == 0;
  const int64_t blocks = (int64_t(p.M) + kWarps - 1) / kWarps, resident = int64_t(sm_count()) * (24 / kWarps);
  moe_route_kernel<T, PER, kWarps><<<unsigned(blocks < resident ? blocks : resident), kWarps * 32, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "moe_route launch");
}

template <typename T>
int launch_route(const RouteParams& p, cudaStream_t st) {
  // up to 32 experts a lane of the one-warp form has one key, which costs a launch of few rows less: 1 x 8 2.7 us against 3.0, but
  // 4096 x 8 4.4 against 3.6, 16384 x 8 9.1 against 6.1, 16384 x 32 10.6 against 6.3
  const bool wide_enough = p.E > 32 || p.M >= 2048;
  int status = FNN_OK;
  if (wide_enough && p.top_k <= 8 &&
      (launch_route_lists<T, 8, 8, 8>(p, st, status) || launch_route_lists<T, 16, 8, 8>(p, st, status) ||
       launch_route_lists<T, 32, 8, 8>(p, st, status) || launch_route_lists<T, 32, 16, 8>(p, st, status)))
    return status;
  if (wide_enough && p.top_k > 8 && p.top_k <= 16 &&
      (launch_route_lists<T, 8, 16, 16>(p, st, status) || launch_route_lists<T, 16, 16, 16>(p, st, status) ||
       launch_route_lists<T, 32, 16, 16>(p, st, status)))
    return status;
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
// experts' padded sizes give every warp its first slot of every expert; pass 2 hands the slots out in list order, equal experts
// within a warp ranked by a vote per bit of the expert (match.any takes about 100 cycles for 32 different values: 131072 choices 25 us with it, 17 with
// votes, eight CTAs each).  No atomics decide an order: the list is the same every time.
constexpr int kSortThreads = 1024;  // most
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
  extern __shared__ int32_t cnt[];            // [cta_warps][E]: counts, then the warp's next slot within the expert
  const int threads = int(blockDim.x), cta_warps = threads >> 5;  // (at least one thread per expert)
  int32_t* total = cnt + cta_warps * p.E;     // [E] this CTA's counts
  int32_t* begin = total + p.E;               // [E] first slot of the expert
  int32_t* count = begin + p.E;               // [E] slots in use of the expert
  int32_t* base = count + p.E;                // [E] first slot of the expert that is this CTA's
  __shared__ int32_t scan[kSortWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = int(cluster.block_rank()), ctas = int(cluster.num_blocks());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gw = rank * cta_warps + warp, warps = ctas * cta_warps;
  const int piece = ((p.choices + warps - 1) / warps + 31) / 32 * 32;
  const int64_t lo64 = int64_t(gw) * piece;
  const int lo = int(lo64 < p.choices ? lo64 : p.choices);
  const int hi = int(lo64 + piece < p.choices ? lo64 + piece : p.choices);
  int32_t* mine = cnt + warp * p.E;

  // experts of the piece's first kHeld steps stay in registers between the passes (all of it up to 131072 choices)
  auto expert_of = [&](int i) {
    const unsigned x = i < hi ? unsigned(__ldg(p.ids + i)) - unsigned(p.first) : kNoExpert;
    return x < unsigned(p.E) ? x : kNoExpert;
  };
  unsigned held[kHeld];
#pragma unroll
  for (int s = 0; s < kHeld; ++s) held[s] = expert_of(lo + s * 32 + lane);
  for (int i = threadIdx.x; i < cta_warps * p.E; i += threads) cnt[i] = 0;
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
    int run = 0;
    for (int w0 = 0; w0 < cta_warps; w0 += 8) {
      int t[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) t[w] = w0 + w < cta_warps ? cnt[(w0 + w) * p.E + e] : 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        if (w0 + w < cta_warps) cnt[(w0 + w) * p.E + e] = run;
        run += t[w];
      }
    }
    total[e] = run;
  }
  if (ctas > 1) cluster.sync();
  int before = 0, all = 0;
  if (e < p.E) {
    for (int c = 0; c < ctas; ++c) {
      const int t = ctas > 1 ? cluster.map_shared_rank(total, c)[e] : total[e];
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
    int t = lane < cta_warps ? scan[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) t += u;
    }
    scan[lane] = t;
  }
  __syncthreads();
  const int in_use = scan[cta_warps - 1];
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
  for (int s = in_use + rank * threads + threadIdx.x; s < p.slots; s += ctas * threads) p.sorted[s] = p.choices;
  for (int k = in_use / p.bm + rank * threads + threadIdx.x; k < p.slots / p.bm; k += ctas * threads) p.experts[k] = 0;
  if (ctas > 1) cluster.sync();  // nobody leaves while another CTA may still read its counts
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

// VEC: columns of an access, 8, 2 or 1, as N and the alignments allow; GROUPS: accesses of a thread and row, 256 * VEC
// columns apart, so that narrow accesses have as many bytes in flight.
template <typename T, int VEC> struct CombineWord { using type = T; };
template <typename T> struct CombineWord<T, 8> { using type = uint4; };
template <typename T> struct CombineWord<T, 2> { using type = uint32_t; };

template <typename T, int VEC, int GROUPS>
__global__ void __launch_bounds__(256) moe_combine_kernel(const CombineParams p) {
  const int64_t m = blockIdx.x;
  const int n = blockIdx.y * (256 * GROUPS * VEC) + threadIdx.x * VEC;
  if (n >= p.N) return;
  float acc[GROUPS][VEC];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[g][j] = 0.f;
  using Word = typename CombineWord<T, VEC>::type;
  auto add = [&](int g, const Word& v, float w) {
    if constexpr (VEC == 8) {
      const uint32_t a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[g][2 * j] = fmaf(w, lo_of<T>(a[j]), acc[g][2 * j]);
        acc[g][2 * j + 1] = fmaf(w, hi_of<T>(a[j]), acc[g][2 * j + 1]);
      }
    } else if constexpr (VEC == 2) {
      acc[g][0] = fmaf(w, lo_of<T>(v), acc[g][0]);
      acc[g][1] = fmaf(w, hi_of<T>(v), acc[g][1]);
    } else {
      acc[g][0] = fmaf(w, to_f32(v), acc[g][0]);
    }
  };
  auto there = [&](int g) { return n + g * 256 * VEC < p.N; };
  // Two choices' rows at a time, their loads in flight together; a choice that is not here is neither read nor added.  One at a time
  // / two / four / eight: 4096 tokens x 8 choices (an eighth of them gone) x 4096 55 / 50 / 52 / 61 us, 16384 x 2 x 4096 93 / 86 / 114 / 182.  The reads
  // bound it: 50 us are 6.7 TB/s.
  constexpr int kAhead = 2;
  const T* c = reinterpret_cast<const T*>(p.c) + m * p.ldc_m + n;
  for (int k0 = 0; k0 < p.top_k; k0 += kAhead) {
    Word v[kAhead][GROUPS];
    bool on[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int k = k0 + i;
      on[i] = k < p.top_k && !(p.ids && unsigned(__ldg(p.ids + m * p.top_k + k)) - unsigned(p.first) >= unsigned(p.E));
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        if (on[i] && there(g)) v[i][g] = *reinterpret_cast<const Word*>(c + k * p.ldc_k + g * 256 * VEC);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (!on[i]) continue;
      const float w = p.w ? __ldg(p.w + m * p.top_k + k0 + i) : 1.f;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g)
        if (there(g)) add(g, v[i][g], w);
    }
  }
  T* out = reinterpret_cast<T*>(p.out) + m * p.ldo + n;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    if (!there(g)) continue;
    if (p.residual) add(g, *reinterpret_cast<const Word*>(reinterpret_cast<const T*>(p.residual) + m * p.ldr + n + g * 256 * VEC), 1.f);
    if constexpr (VEC == 8)
      *reinterpret_cast<uint4*>(out) = make_uint4(pack2<T>(acc[g][0], acc[g][1]), pack2<T>(acc[g][2], acc[g][3]), pack2<T>(acc[g][4], acc[g][5]), pack2<T>(acc[g][6], acc[g][7]));
    else if constexpr (VEC == 2)
      *reinterpret_cast<uint32_t*>(out + g * 512) = pack2<T>(acc[g][0], acc[g][1]);
    else
      out[g * 256] = from_f32<T>(acc[g][0]);
  }
}

template <typename T, int VEC, int GROUPS> int launch_combine_as(const CombineParams& p, cudaStream_t st) {
  const int64_t chunks = (int64_t(p.N) + 256 * VEC * GROUPS - 1) / (256 * VEC * GROUPS);
  if (chunks > 65535) return fail(FNN_ERR_UNSUPPORTED, "moe_combine: rows of %d columns are too long", p.N);
  moe_combine_kernel<T, VEC, GROUPS><<<dim3(unsigned(p.M), unsigned(chunks)), 256, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "moe_combine launch");
}
template <typename T> int launch_combine(const CombineParams& p, cudaStream_t st) {
  // whether every access of `cols` columns is aligned
  auto fits = [&](int cols) {
    auto ok = [&](const void* q, int64_t ld) { return reinterpret_cast<uintptr_t>(q) % (cols * sizeof(T)) == 0 && ld % cols == 0; };
    return p.N % cols == 0 && ok(p.c, p.ldc_m) && p.ldc_k % cols == 0 && ok(p.out, p.ldo) && (!p.residual || ok(p.residual, p.ldr));
  };
  if (fits(8)) return launch_combine_as<T, 8, 1>(p, st);
  // Narrow accesses, two or four to a thread: four where the row is longer than two cover.  1 / 2 / 4 accesses, us: 4096 x 8 x
  // 1001 53 / 35 / 27, x 4097 212 / 133 / 98, x 4098 (2 columns an access; 1 column in the first figure) 212 / 81 / 67;
  // but 4096 x 8 x 1002 53 / 22 / 25, 16384 x 3 x 333 49 / 40 / 45.
  if (fits(2)) return p.N > 2 * 256 * 2 ? launch_combine_as<T, 2, 4>(p, st) : launch_combine_as<T, 2, 2>(p, st);
  return p.N > 2 * 256 ? launch_combine_as<T, 1, 4>(p, st) : launch_combine_as<T, 1, 2>(p, st);
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
  // (the kernel compares unsigned differences: a range that passes 2^31 would take in the numbers it wraps to)
  if (first_expert < INT32_MIN || first_expert > INT32_MAX || first_expert + E > int64_t(INT32_MAX) + 1)
    return fail(FNN_ERR_SHAPE, "moe_sort: expert numbers must fit 32 bits");
  const int64_t need = fnn_moe_sort_slots(num_choices, E, block_m);
  if (num_choices > INT32_MAX / 2 || need > INT32_MAX / 2) return fail(FNN_ERR_SHAPE, "moe_sort: %lld choices need %lld slots: too many", (long long)num_choices, (long long)need);
  if (EM != need) return fail(FNN_ERR_SHAPE, "moe_sort: the slot list has %lld entries, fnn_moe_sort_slots says %lld", (long long)EM, (long long)need);
  if (!num_tokens_post_padded || (num_choices > 0 && (!topk_ids || !sorted_token_ids || !expert_ids)))
    return fail(FNN_ERR_NULL_POINTER, "moe_sort: null tensor pointer");
  SortParams p{topk_ids, sorted_token_ids, expert_ids, num_tokens_post_padded, int(num_choices), int(E), block_m, int(first_expert), int(EM)};
  // 16 CTAs are more than every device promises a cluster (a partition may not hold them): asked once for the largest launch
  static std::once_flag once[64];
  static cudaError_t attr_err[64];
  static unsigned most_ctas[64];
  int dev = 0;
  cudaGetDevice(&dev);
  dev &= 63;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  std::call_once(once[dev], [&] {
    constexpr int kMostBytes = (kSortWarps + 4) * kSortMaxExperts * 4;
    attr_err[dev] = cudaFuncSetAttribute(moe_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostBytes);
    if (attr_err[dev] == cudaSuccess) attr_err[dev] = cudaFuncSetAttribute(moe_sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(kSortThreads);
    cfg.dynamicSmemBytes = kMostBytes;
    attr[0].val.clusterDim.x = 16;
    int clusters = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&clusters, moe_sort_kernel, &cfg);
    if (e != cudaSuccess) (void)cudaGetLastError();
    most_ctas[dev] = e == cudaSuccess && clusters > 0 ? 16u : 8u;
  });
  if (attr_err[dev] != cudaSuccess) return check_cuda(attr_err[dev], "cudaFuncSetAttribute(moe_sort)");
  // One CTA where a launch is all there is to it, else as many as a cluster holds: they write the slots, padding included, and 16 SMs
  // write them faster than one.  Measured, one CTA / a cluster: 64 tokens x 2 of 8 experts (240 slots) 4.4 / 5.4 us, 512 x 2 of 8
  // in blocks of 128 (1920) 5.3 / 5.6, 2048 x 2 of 8 (4992) 7.9 / 5.8, 64 x 8 of 256 (32768) 18 / 6.7.  A cluster of 8: 131072
  // choices 16.8 us, of 16: 12.1.  Warps cost barriers, and pay where their steps (32 choices each) are many: 512 / 1024
  // threads a CTA, 16384 choices 7.4 / 8.7 us, 131072 12.1 / 12.7, 262144 22.9 / 17.8.
  const unsigned ctas = need > 2048 ? most_ctas[dev] : 1u;
  unsigned threads = ctas == 1 ? 256u : num_choices > 131072 ? unsigned(kSortThreads) : 512u;
  if (int64_t(threads) < E) threads = unsigned((E + 31) / 32 * 32);
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = size_t(threads / 32 + 4) * size_t(E) * sizeof(int32_t);
  cfg.stream = static_cast<cudaStream_t>(stream);
  attr[0].val.clusterDim.x = ctas;
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
  if (topk_ids && (E > INT32_MAX || first_expert < INT32_MIN || first_expert > INT32_MAX || first_expert + E > int64_t(INT32_MAX) + 1))
    return fail(FNN_ERR_SHAPE, "moe_combine: expert numbers must fit 32 bits");
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
