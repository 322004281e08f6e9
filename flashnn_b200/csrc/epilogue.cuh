// What an A8W8 product does with its scaled sums before their one rounding to the output type: bias, activation, gate
// and residual, all in fp32.
//
//   plain   out = T(act(v[n]) + r[m, n])                with v = fl32(acc * s) + bias
//   gated   out = T(act(v[n]) * v[N + n] + r[m, n])     the weight has 2 N rows: the N rows inside the activation, then
//                                                       the N rows that its value multiplies
//
// Bias, gate and residual are each rounded (__fadd_rn, __fmul_rn are never contracted), so that all kernels give the same bits.
// The gate needs the sums of weight rows n and N + n in one thread, so a gated tile of BN accumulator columns takes
// BN / 2 rows from each half of the weight: the two halves meet in the accumulator, and the output, half as wide as the
// product, is all that leaves the chip.
#pragma once
#include "common.cuh"
#include "quantise.cuh"

namespace fnn {

// kernels without an epilogue of this kind
struct NoEpilogue {
  static constexpr bool kOn = false, kGated = false;
};
template <bool GATED> struct FusedEpilogue {
  static constexpr bool kOn = true, kGated = GATED;
  const void* bias;      // nullptr or [rows] (fused MoE: [E, rows])
  const void* residual;  // nullptr or [M, N] in the output's dtype
  int64_t ldr;
  int bias_dtype, act;   // act: fnn_activation
  int rows;              // weight rows (of one expert): N, or 2 N with a gate
  int experts, blocks;   // fused MoE: slots of a block whose expert is not one of `experts` write nothing; blocks of the slot list
};

// The hardware's 2^v and reciprocal as they are (subnormal results flushed to 0): one instruction each, where __expf and
// __fdividef add the scaling that keeps subnormals.  With K short the epilogue is what a tile waits for, and these are its longest part.
__device__ __forceinline__ float exp2_ftz(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_ftz(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 1 / (1 + e^-v): within (8 + 1.25 |v|) roundings of 2^-24, relative (the product with log2 e and its constant 1.22 |v|, the exponential 4,
// the sum 1, the reciprocal 2), far below the half step (2^-8, 2^-11) of the 16-bit output.  e^-v of a very negative v is infinite
// and its reciprocal 0 (from v = -87.3 on); a NaN stays one.
__device__ __forceinline__ float sigmoid_f32(float v) { return rcp_ftz(1.f + exp2_ftz(-1.4426950408889634f * v)); }
// v Phi(v).  Phi(v) = erfc(-v / sqrt 2) / 2, and for x = |v| / sqrt 2 the tail erfc(x) / 2 = t P(t) e^(-x^2) with t = 1 / (1 + 0.7 x):
// t P(t) is a fit of e^(x^2) erfc(x) / 2 on [0, 9.5] (ten coefficients, least relative error by reweighted least squares: 1e-7), so
// the negative tail, which is v times this, has its error relative to itself: within (20 + 2 v^2) roundings of 2^-24, the
// exponential's argument included (1.1e-5 at v = -9; the half step of fp16 is 4.9e-4).  A fit of least absolute error is 0.05 %
// off at v = -4 and 1 % at -8.  Results are 0 where e^(-v^2 / 2) is below the normal range (v < -13.2).
// The polynomial runs on pairs of values, two multiply-adds an instruction.
__device__ __forceinline__ void gelu_pair(float& a, float& b) {
  constexpr float kFit[10] = {0.197489366f,  0.196793377f, 0.157398701f,  -0.00448890822f, 0.178573206f,
                              -0.715528607f, 0.884957016f, -0.544626772f, 0.171032086f,    -0.0215994157f};
  constexpr float kSlope = 0.7f * 0.70710678118654752f, kExp = -0.72134752044448170f;
  const float ta = rcp_ftz(fmaf(kSlope, fabsf(a), 1.f)), tb = rcp_ftz(fmaf(kSlope, fabsf(b), 1.f));
  const uint64_t t = pack_f32x2(ta, tb);
  uint64_t poly = pack_f32x2(kFit[9], kFit[9]);
#pragma unroll
  for (int i = 8; i >= 0; --i) poly = ffma2_rn(t, poly, pack_f32x2(kFit[i], kFit[i]));
  float pa, pb;
  unpack_f32x2(poly, pa, pb);
  const float tail_a = __fmul_rn(ta * pa, exp2_ftz(kExp * (a * a))), tail_b = __fmul_rn(tb * pb, exp2_ftz(kExp * (b * b)));
  a *= a > 0.f ? 1.f - tail_a : tail_a;
  b *= b > 0.f ? 1.f - tail_b : tail_b;
}

template <int ACT> __device__ __forceinline__ float activate(float v) {
  if (ACT == FNN_ACT_RELU) return v < 0.f ? 0.f : v;  // (keeps a NaN)
  if (ACT == FNN_ACT_SIGMOID) return sigmoid_f32(v);
  if (ACT == FNN_ACT_SILU) return v * sigmoid_f32(v);
  // v / 2 (1 + tanh(t)) = v sigmoid(2 t)
  if (ACT == FNN_ACT_GELU_TANH) return v * sigmoid_f32(1.5957691216057308f * fmaf(0.044715f * v, v * v, v));
  return v;
}
template <int ACT, int N> __device__ __forceinline__ void activate_all(float (&v)[N]) {
  if constexpr (ACT == FNN_ACT_GELU) {
    float none = 0.f;
#pragma unroll
    for (int j = 0; j < N; j += 2) gelu_pair(v[j], j + 1 < N ? v[j + 1 < N ? j + 1 : j] : none);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = activate<ACT>(v[j]);
  }
}
// the activation is a launch argument: one uniform branch for a thread's N values
template <int N> __device__ __forceinline__ void activate_n(float (&v)[N], int act) {
  switch (act) {
    case FNN_ACT_RELU: activate_all<FNN_ACT_RELU>(v); break;
    case FNN_ACT_SIGMOID: activate_all<FNN_ACT_SIGMOID>(v); break;
    case FNN_ACT_SILU: activate_all<FNN_ACT_SILU>(v); break;
    case FNN_ACT_GELU: activate_all<FNN_ACT_GELU>(v); break;
    case FNN_ACT_GELU_TANH: activate_all<FNN_ACT_GELU_TANH>(v); break;
    default: break;
  }
}
__device__ __forceinline__ float activate_one(float v, int act) {
  float a[1] = {v};
  activate_n(a, act);
  return a[0];
}

// 2 H consecutive residual values of one row as packed pairs; zeros outside the matrix
template <typename T, int H, class FX>
__device__ __forceinline__ void load_residual(const FX& fx, int row, int col0, int M, int N, bool vec_ok, uint32_t (&r)[H]) {
  if (row >= M || col0 >= N) {
#pragma unroll
    for (int j = 0; j < H; ++j) r[j] = 0u;
    return;
  }
  const T* src = reinterpret_cast<const T*>(fx.residual) + int64_t(row) * fx.ldr + col0;
  if (vec_ok && col0 + 2 * H <= N) {
#pragma unroll
    for (int j = 0; j < H; j += 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(src + 2 * j);
      r[j] = u.x; r[j + 1] = u.y; r[j + 2] = u.z; r[j + 3] = u.w;
    }
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
    for (int j = 0; j < H; ++j) {
      const uint32_t lo = col0 + 2 * j < N ? h[2 * j] : 0u, hi = col0 + 2 * j + 1 < N ? h[2 * j + 1] : 0u;
      r[j] = lo | (hi << 16);
    }
  }
}
template <typename T, int H> __device__ __forceinline__ void add_residual(const uint32_t (&r)[H], float (&v)[2 * H]) {
#pragma unroll
  for (int j = 0; j < H; ++j) {
    v[2 * j] = __fadd_rn(v[2 * j], lo_of<T>(r[j]));
    v[2 * j + 1] = __fadd_rn(v[2 * j + 1], hi_of<T>(r[j]));
  }
}
template <int N> __device__ __forceinline__ void add_bias(const float* b, float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 4) {
    const float4 t = *reinterpret_cast<const float4*>(b + j);
    v[j] = __fadd_rn(v[j], t.x); v[j + 1] = __fadd_rn(v[j + 1], t.y);
    v[j + 2] = __fadd_rn(v[j + 2], t.z); v[j + 3] = __fadd_rn(v[j + 3], t.w);
  }
}

}  // namespace fnn
