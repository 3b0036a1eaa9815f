// Helpers of the vocabulary-row kernels (token log probabilities, distillation):
// addressing of logit rows, conversions, the order of values, block reductions.
#pragma once

#include "common.cuh"

#include <math_constants.h>

namespace dwarf {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Row r of logits [outer, inner, vocab] with two row strides.
__device__ __forceinline__ int64_t row_offset(int64_t r, int64_t inner, int64_t so, int64_t si) {
  const int64_t o = r / inner;
  return o * so + (r - o * inner) * si;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// A whole number that orders floats: -inf < finite < +inf < NaN, -0 with +0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xff800001u;  // above +inf, below all ones
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// (value, lowest id first) as one whole number: the larger is the better entry.
__device__ __forceinline__ uint64_t entry_key(float v, uint32_t id) {
  return ((uint64_t)order_key(v) << 32) | (uint32_t)~id;
}
__device__ __forceinline__ uint32_t entry_id(uint64_t key) { return ~(uint32_t)key; }

// Sums (and maxima) over a block in a fixed order; every thread gets the result.
// `scratch` holds one value per warp; a barrier at each end makes it reusable.
template <int kThreads, typename V, typename F>
__device__ __forceinline__ V block_reduce(V v, V* scratch, F f) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  V t = scratch[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) t = f(t, scratch[i]);
  return t;
}

struct AddOp {
  template <typename V>
  __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct MaxOp {
  __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
  __device__ __forceinline__ uint64_t operator()(uint64_t a, uint64_t b) const { return a > b ? a : b; }
};

// Host checks shared by the entry points: sizes, strides and the scale of a logit tensor.
inline int check_logits(const void* logits, int32_t dtype, int64_t outer, int64_t inner, int64_t vocab, int64_t so,
                        int64_t si, float inv_temperature) {
  if (outer < 0 || inner < 0 || vocab < 1 || vocab > DWARF_VOCAB_MAX) return DWARF_ERR_SHAPE;
  if (outer > 0 && inner > 0x7fffffffll / outer) return DWARF_ERR_SHAPE;
  if (so < 0 || si < 0) return DWARF_ERR_STRIDE;
  if (dtype != DWARF_F32 && dtype != DWARF_BF16 && dtype != DWARF_F16) return DWARF_ERR_DTYPE;
  const float c2 = inv_temperature * kLog2e;
  if (!(c2 > 0.0f) || c2 > 3.0e38f) return DWARF_ERR_VALUE;
  if (outer * inner > 0 && logits == nullptr) return DWARF_ERR_NULL;
  const uintptr_t mask = dtype == DWARF_F32 ? 3 : 1;
  if (reinterpret_cast<uintptr_t>(logits) & mask) return DWARF_ERR_ALIGN;
  return DWARF_OK;
}

}  // namespace dwarf
