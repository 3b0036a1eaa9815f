// Helpers of the vocabulary-row kernels (token log probabilities, distillation):
// addressing of logit rows, conversions and packed operations, the order of values, a CTA's
// part of a row, clusters, and the rules that split rows over CTAs.
//
// A row is read as 16-byte vectors from its first boundary on; a thread has eight of them in
// flight. All sums are fp32, relative to a running maximum of each warp, and joined in a
// fixed order (the same bits every time, for one split of the rows).
#pragma once

#include "common.cuh"

#include <math_constants.h>

namespace dwarf {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kRowThreads = 128;    // threads of a CTA, or of each CTA of a cluster, for a row
constexpr int kVectors = 8;         // 16-byte vectors of a row that a thread has in flight
constexpr int kMaxCluster = 8;

// Row r of logits [outer, inner, vocab] with two row strides.
__device__ __forceinline__ int64_t row_offset(int64_t r, int64_t inner, int64_t so, int64_t si) {
  const uint32_t o = (uint32_t)r / (uint32_t)inner;  // fewer than 2^28 rows
  return o * so + (int64_t)((uint32_t)r - o * (uint32_t)inner) * si;
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

// The sum over a block, in a fixed order, for every thread. `scratch`: one value per warp.
template <int kThreads>
__device__ __forceinline__ float block_sum(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = scratch[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) t += scratch[i];
  return t;
}

// Pairs of fp32: one issue slot for two elements.
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// 16 bytes of a row: kVec elements.
template <typename T>
struct Vec16;

template <>
struct Vec16<float> {
  static constexpr int kVec = 4;
  static constexpr uint32_t kMinusInf = 0xff800000u;
  __device__ __forceinline__ static void unpack(const uint4& v, float2 (&x)[2]) {
    x[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    x[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  __device__ __forceinline__ static uint4 pack(const float2 (&x)[2]) {
    return make_uint4(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x),
                      __float_as_uint(x[1].y));
  }
  // A running maximum of elements by place (NaN is passed over), its largest, and whether one reaches `bound`.
  using Max = float;
  __device__ __forceinline__ static Max max_of(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  __device__ __forceinline__ static Max join(Max a, Max b) { return fmaxf(a, b); }
  __device__ __forceinline__ static Max none() { return -CUDART_INF_F; }
  __device__ __forceinline__ static float largest(Max a) { return a; }
  using Narrow = __nv_bfloat16;  // 16 bits that are no lower than the largest, and no higher
  __device__ __forceinline__ static Narrow narrow(Max a) { return __float2bfloat16_ru(a); }
  __device__ __forceinline__ static Narrow narrow_down(Max a) { return __float2bfloat16_rd(a); }
  // The elements of at least `bound` (the nearest lower value of the type) as bits; the element of a bit; its value.
  __device__ __forceinline__ static uint32_t reach(const uint4& v, float bound) {
    return (uint32_t)(__uint_as_float(v.x) >= bound) | (uint32_t)(__uint_as_float(v.y) >= bound) << 1 |
           (uint32_t)(__uint_as_float(v.z) >= bound) << 2 | (uint32_t)(__uint_as_float(v.w) >= bound) << 3;
  }
  __device__ __forceinline__ static int element(int bit) { return bit; }
  __device__ __forceinline__ static float value(const uint4& v, int e) {
    return __uint_as_float(e & 2 ? (e & 1 ? v.w : v.z) : (e & 1 ? v.y : v.x));
  }
  // v without the elements of a mask (bit e: element e): -inf in their places.
  __device__ __forceinline__ static uint4 drop(const uint4& v, uint32_t mask) {
    return make_uint4(mask & 1u ? kMinusInf : v.x, mask & 2u ? kMinusInf : v.y, mask & 4u ? kMinusInf : v.z,
                      mask & 8u ? kMinusInf : v.w);
  }
  // Elements no lower than `low`.
  using Low = float;
  __device__ __forceinline__ static Low low_of(float v) { return v; }
  __device__ __forceinline__ static float low_value(Low low) { return low; }
  __device__ __forceinline__ static uint4 clamp(const uint4& v, Low low) {
    return make_uint4(max_nan(v.x, low), max_nan(v.y, low), max_nan(v.z, low), max_nan(v.w, low));
  }
  __device__ __forceinline__ static uint32_t max_nan(uint32_t a, float b) {
    uint32_t r;
    asm("max.NaN.f32 %0, %1, %2;" : "=r"(r) : "r"(a), "f"(b));
    return r;
  }
};

template <>
struct Vec16<__nv_bfloat16> {
  static constexpr int kVec = 8;
  static constexpr uint32_t kMinusInf = 0xff80ff80u;
  __device__ __forceinline__ static void unpack(const uint4& v, float2 (&x)[4]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  __device__ __forceinline__ static uint4 pack(const float2 (&x)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[i].x, x[i].y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  using Max = __nv_bfloat162;
  using Narrow = __nv_bfloat16;
  __device__ __forceinline__ static Narrow narrow(Max a) { return __hmax(__low2bfloat16(a), __high2bfloat16(a)); }
  __device__ __forceinline__ static Narrow narrow_down(Max a) { return narrow(a); }
  __device__ __forceinline__ static Max max_of(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    return __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  }
  __device__ __forceinline__ static Max join(Max a, Max b) { return __hmax2(a, b); }
  __device__ __forceinline__ static Max none() {
    const uint32_t w = kMinusInf;
    return *reinterpret_cast<const Max*>(&w);
  }
  __device__ __forceinline__ static float largest(Max a) {
    const float2 f = __bfloat1622float2(a);
    return fmaxf(f.x, f.y);
  }
  __device__ __forceinline__ static uint32_t reach(const uint4& v, float bound) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 b = __bfloat162bfloat162(__float2bfloat16_rd(bound));
    return (__hge2_mask(h[0], b) & 0x00010001u) | (__hge2_mask(h[1], b) & 0x00020002u) |
           (__hge2_mask(h[2], b) & 0x00040004u) | (__hge2_mask(h[3], b) & 0x00080008u);
  }
  // Adds the places' numbers of elements above g to c (exact up to 256).
  __device__ __forceinline__ static __nv_bfloat162 above(const uint4& v, __nv_bfloat16 g, __nv_bfloat162 c) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 b = __bfloat162bfloat162(g);
    c = __hadd2(c, __hgt2(h[0], b));
    c = __hadd2(c, __hgt2(h[1], b));
    c = __hadd2(c, __hgt2(h[2], b));
    return __hadd2(c, __hgt2(h[3], b));
  }
  __device__ __forceinline__ static int total(__nv_bfloat162 c) {
    const float2 f = __bfloat1622float2(c);
    return (int)(f.x + f.y);
  }
  __device__ __forceinline__ static int element(int bit) { return 2 * (bit & 15) + (bit >> 4); }
  __device__ __forceinline__ static float value(const uint4& v, int e) {
    const uint32_t w = e & 4 ? (e & 2 ? v.w : v.z) : (e & 2 ? v.y : v.x);
    return to_f32(__ushort_as_bfloat16((unsigned short)(e & 1 ? w >> 16 : w & 0xffffu)));
  }
  __device__ __forceinline__ static uint32_t drop2(uint32_t w, uint32_t mask) {
    const uint32_t gone = (mask & 1u ? 0x0000ffffu : 0u) | (mask & 2u ? 0xffff0000u : 0u);
    return (w & ~gone) | (kMinusInf & gone);
  }
  __device__ __forceinline__ static uint4 drop(const uint4& v, uint32_t mask) {
    return make_uint4(drop2(v.x, mask), drop2(v.y, mask >> 2), drop2(v.z, mask >> 4), drop2(v.w, mask >> 6));
  }
  using Low = __nv_bfloat162;
  __device__ __forceinline__ static Low low_of(float v) { return __float2bfloat162_rn(v); }
  __device__ __forceinline__ static float low_value(Low low) { return __low2float(low); }
  __device__ __forceinline__ static uint4 clamp(const uint4& v, Low low) {
    uint4 r;
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    __nv_bfloat162* o = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __hmax2_nan(h[i], low);
    return r;
  }
};

template <>
struct Vec16<__half> {
  static constexpr int kVec = 8;
  static constexpr uint32_t kMinusInf = 0xfc00fc00u;
  __device__ __forceinline__ static void unpack(const uint4& v, float2 (&x)[4]) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __half22float2(h[i]);
  }
  __device__ __forceinline__ static uint4 pack(const float2 (&x)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(x[i].x, x[i].y);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  using Max = __half2;
  using Narrow = __half;
  __device__ __forceinline__ static Narrow narrow(Max a) { return __hmax(__low2half(a), __high2half(a)); }
  __device__ __forceinline__ static Narrow narrow_down(Max a) { return narrow(a); }
  __device__ __forceinline__ static Max max_of(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    return __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  }
  __device__ __forceinline__ static Max join(Max a, Max b) { return __hmax2(a, b); }
  __device__ __forceinline__ static Max none() {
    const uint32_t w = kMinusInf;
    return *reinterpret_cast<const Max*>(&w);
  }
  __device__ __forceinline__ static float largest(Max a) {
    const float2 f = __half22float2(a);
    return fmaxf(f.x, f.y);
  }
  __device__ __forceinline__ static uint32_t reach(const uint4& v, float bound) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 b = __half2half2(__float2half_rd(bound));
    return (__hge2_mask(h[0], b) & 0x00010001u) | (__hge2_mask(h[1], b) & 0x00020002u) |
           (__hge2_mask(h[2], b) & 0x00040004u) | (__hge2_mask(h[3], b) & 0x00080008u);
  }
  // Adds the places' numbers of elements above g to c (exact up to 256).
  __device__ __forceinline__ static __half2 above(const uint4& v, __half g, __half2 c) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 b = __half2half2(g);
    c = __hadd2(c, __hgt2(h[0], b));
    c = __hadd2(c, __hgt2(h[1], b));
    c = __hadd2(c, __hgt2(h[2], b));
    return __hadd2(c, __hgt2(h[3], b));
  }
  __device__ __forceinline__ static int total(__half2 c) {
    const float2 f = __half22float2(c);
    return (int)(f.x + f.y);
  }
  __device__ __forceinline__ static int element(int bit) { return 2 * (bit & 15) + (bit >> 4); }
  __device__ __forceinline__ static float value(const uint4& v, int e) {
    const uint32_t w = e & 4 ? (e & 2 ? v.w : v.z) : (e & 2 ? v.y : v.x);
    return to_f32(__ushort_as_half((unsigned short)(e & 1 ? w >> 16 : w & 0xffffu)));
  }
  __device__ __forceinline__ static uint32_t drop2(uint32_t w, uint32_t mask) {
    const uint32_t gone = (mask & 1u ? 0x0000ffffu : 0u) | (mask & 2u ? 0xffff0000u : 0u);
    return (w & ~gone) | (kMinusInf & gone);
  }
  __device__ __forceinline__ static uint4 drop(const uint4& v, uint32_t mask) {
    return make_uint4(drop2(v.x, mask), drop2(v.y, mask >> 2), drop2(v.z, mask >> 4), drop2(v.w, mask >> 6));
  }
  using Low = __half2;
  __device__ __forceinline__ static Low low_of(float v) { return __float2half2_rn(v); }
  __device__ __forceinline__ static float low_value(Low low) { return __low2float(low); }
  __device__ __forceinline__ static uint4 clamp(const uint4& v, Low low) {
    uint4 r;
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    __half2* o = reinterpret_cast<__half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __hmax2_nan(h[i], low);
    return r;
  }
};

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// L2 keeps lines read under the first policy while it can, and gives up those read under the second.
__device__ __forceinline__ uint64_t policy_keep() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint64_t policy_leave() {
  uint64_t p;
  asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ uint4 ld_stream(const void* p, uint64_t policy) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p), "l"(policy));
  return v;
}
// Asks L2 for `bytes` (a multiple of 16) from a 16-byte boundary.
__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes, uint64_t policy) {
  asm volatile("cp.async.bulk.prefetch.L2.global.L2::cache_hint [%0], %1, %2;" ::"l"(p), "r"(bytes), "l"(policy)
               : "memory");
}

__device__ __forceinline__ void prefetch_l2(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

__device__ __forceinline__ void st_stream(void* p, const uint4& v) {
  asm volatile("st.global.cs.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

// A row as aligned 16-byte vectors. Places u count from the 16-byte boundary at or
// before the row's first element: element id lies at u = id + lead, vector j holds
// places [j kVec, (j + 1) kVec). Only the first and the last vector may hold places
// outside the row; they are read element by element, the places outside as -inf.
template <typename T>
struct RowVectors {
  static constexpr int kVec = Vec16<T>::kVec;
  const T* base;  // the boundary (not read before the row)
  int lead;       // elements between the boundary and the row
  int end;        // lead + vocab
  __device__ __forceinline__ RowVectors(const T* row, int vocab) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row);
    lead = (int)((at & 15) / sizeof(T));
    base = row - lead;
    end = lead + vocab;
  }
  __device__ __forceinline__ int count() const { return (end + kVec - 1) / kVec; }
  __device__ __forceinline__ bool whole(int j) const { return j * kVec >= lead && (j + 1) * kVec <= end; }
  __device__ __forceinline__ uint4 load(int j) const {
    if (whole(j)) return ld_stream(base + (int64_t)j * kVec);
    // the nearest element of the row for a place outside it, so that no load waits for a branch
    uint4 v;
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int i = 0; i < kVec; ++i) e[i] = base[min(max(j * kVec + i, lead), end - 1)];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int u = j * kVec + i;
      if (u < lead || u >= end) e[i] = from_f32<T>(-CUDART_INF_F);
    }
    return v;
  }
};

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Largest value over a warp, through the integers that order floats.
__device__ __forceinline__ float warp_max(float v) {
  int k = __float_as_int(v);
  k ^= (k >> 31) & 0x7fffffff;
  k = __reduce_max_sync(0xffffffffu, k);
  k ^= (k >> 31) & 0x7fffffff;
  return __int_as_float(k);
}

template <typename V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The CTAs of a cluster share one row.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The shared-memory address of the same variable in CTA `rank` of the cluster, for st.shared::cluster.
__device__ __forceinline__ uint32_t cluster_address(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// Launch with `cluster` CTAs for each row.
template <typename... Params, typename... Args>
int launch_rows(void (*kernel)(Params...), int64_t rows, int cluster, int threads, size_t smem, cudaStream_t stream,
                Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) return launch_status();
  return launch_status();
}

// A CTA's part of a row: its whole vectors, a tile of kVectors vectors for each thread at
// a time, and the up to 2 (kVec - 1) elements at the row's ends that fill no vector, one for each of
// a warp's first 16 lanes. (Ends inside the tiles' loops made the odd vocabulary of 32003 take
// 228 us where 32768 took 155: 6000 rows, distillation with gradient.)
template <typename T, int kThreads = kRowThreads>
struct Part {
  static constexpr int kVec = Vec16<T>::kVec;
  RowVectors<T> row;
  int j0, j1;  // the part's vectors
  int w0, w1;  // those of them that are whole

  __device__ __forceinline__ Part(const T* x, int vocab, int rank, int cluster) : row(x, vocab) {
    const int n = row.count(), per = ceil_div(n, cluster);
    j0 = min(rank * per, n);
    j1 = min(j0 + per, n);
    w0 = max(j0, row.lead > 0 ? 1 : 0);
    w1 = max(w0, min(j1, row.end / kVec));
  }
  __device__ __forceinline__ int size() const { return w1 - w0; }
  // Whether the tile that starts `at` vectors into the part, or its step i, has a vector for every thread.
  __device__ __forceinline__ bool full(int at) const { return at + kVectors * kThreads <= size(); }
  __device__ __forceinline__ bool full(int at, int i) const { return at + (i + 1) * kThreads <= size(); }
  // Vectors at, at + threads, ...; past the part -inf.
  __device__ __forceinline__ void load(int at, uint4 (&v)[kVectors]) const {
    load_by(at, v, [](const uint4* p) { return ld_stream(p); });
  }
  __device__ __forceinline__ void load(int at, uint4 (&v)[kVectors], uint64_t policy) const {
    load_by(at, v, [policy](const uint4* p) { return ld_stream(p, policy); });
  }
  template <typename F>
  __device__ __forceinline__ void load_by(int at, uint4 (&v)[kVectors], F ld) const {
    const uint4* p = reinterpret_cast<const uint4*>(row.base) + (w0 + at + (int)threadIdx.x);
    if (full(at)) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) v[i] = ld(p + i * kThreads);
      return;
    }
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      v[i] = make_uint4(Vec16<T>::kMinusInf, Vec16<T>::kMinusInf, Vec16<T>::kMinusInf, Vec16<T>::kMinusInf);
      if (at + i * kThreads + (int)threadIdx.x < size()) v[i] = ld(p + i * kThreads);
    }
  }
  // Whether the row has ends; the id of the element of them that a lane has, or -1.
  __device__ __forceinline__ bool ends() const { return row.lead > 0 || row.end % kVec > 0; }
  __device__ __forceinline__ int end_id(int lane) const {
    const int tail = max(row.end / kVec, row.lead > 0 ? 1 : 0);
    const int j = lane < 8 ? 0 : tail, u = lane < 8 ? row.lead + lane : tail * kVec + lane - 8;
    const int last = lane < 8 ? (row.lead > 0 ? min(kVec, row.end) : 0) : lane < 16 ? row.end : 0;
    return u < last && j >= j0 && j < j1 ? u - row.lead : -1;
  }
  // Asks L2 for the part's whole vectors under a policy, or for the first `most` of them; by one thread.
  __device__ __forceinline__ void prefetch_kept(uint64_t policy) const {
    if (size() > 0) prefetch_l2(reinterpret_cast<const uint4*>(row.base) + w0, (uint32_t)size() * 16u, policy);
  }
  __device__ __forceinline__ void prefetch_first(int most) const {
    if (size() > 0) prefetch_l2(reinterpret_cast<const uint4*>(row.base) + w0, (uint32_t)min(size(), most) * 16u);
  }
  __device__ __forceinline__ bool holds(int id) const {
    const int j = (id + row.lead) / kVec;
    return j >= j0 && j < j1;
  }
  // f(value, id) for the elements of vector j that are in the row.
  template <typename F>
  __device__ __forceinline__ void elements(const uint4& w, int j, F f) const {
    float2 x[kVec / 2];
    Vec16<T>::unpack(w, x);
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      const int u = j * kVec + e;
      if (u >= row.lead && u < row.end) f(e & 1 ? x[e / 2].y : x[e / 2].x, u - row.lead);
    }
  }
  // f(vector, j, whether j is in the part), one step of the whole block after the other, in
  // rising j, the row's ends included, while f says (the same for all threads) to go on.
  template <typename F>
  __device__ __forceinline__ void walk(F f) const {
    for (int first = j0; first < j1; first += kThreads) {
      const int j = first + threadIdx.x;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (j < j1) w = row.load(j);
      if (!f(w, j, j < j1)) break;
    }
  }
};

// Where the values of a row's vectors go: whole vectors at once where the output row lies
// on the same 16-byte boundaries as the logits, else (a slice of an odd vocabulary) by element:
// 8 x 512 rows of logits[:, :-1] at 32003 bf16 take 392 us (log probability and gradient), the same
// rows contiguous 144.
template <typename T>
struct RowStore {
  static constexpr int kVec = Vec16<T>::kVec;
  T* out;
  int lead;
  bool same;
  __device__ __forceinline__ RowStore(T* o, const RowVectors<T>& r) : out(o), lead(r.lead) {
    same = (reinterpret_cast<uintptr_t>(o) & 15) == r.lead * sizeof(T);
  }
  // f of each vector of a tile of `part`, stored.
  template <int kThreads, typename F>
  __device__ __forceinline__ void tile(const Part<T, kThreads>& part, int at, const uint4 (&v)[kVectors], F f) const {
    T* o = out + ((int64_t)(part.w0 + at + (int)threadIdx.x) * kVec - lead);
    if (same && part.full(at)) {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) st_stream(o + i * kThreads * kVec, f(v[i]));
      return;
    }
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      if (at + i * kThreads + (int)threadIdx.x >= part.size()) break;
      const uint4 w = f(v[i]);
      if (same) {
        st_stream(o + i * kThreads * kVec, w);
      } else {
        const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
        for (int h = 0; h < kVec; ++h) o[i * kThreads * kVec + h] = e[h];
      }
    }
  }
  // Zeros in the part.
  template <int kThreads>
  __device__ __forceinline__ void zero(const Part<T, kThreads>& part) const {
    const uint4 v[kVectors] = {};
    for (int at = 0; at < part.size(); at += kVectors * kThreads) tile(part, at, v, [](const uint4& w) { return w; });
    const int id = threadIdx.x < 32 ? part.end_id(threadIdx.x) : -1;
    if (id >= 0) out[id] = from_f32<T>(0.0f);
  }
};

// How many CTAs share a row: more than one only while the rows alone leave SMs with
// fewer than four CTAs and each part keeps a vector for every thread (148 rows of 32768 bf16:
// 12.3 us with one CTA each, 11.1 with four; 1000 rows: 22.1 with one, 23.3 with two),
// or where a part would have over `most` vectors.
inline int cluster_for(int64_t rows, int vectors, int most) {
  int c = 1;
  while (c < kMaxCluster && vectors > c * most) c *= 2;
  while (c < kMaxCluster && rows * c * 2 <= 4 * kNumSMs && vectors >= c * 2 * kRowThreads) c *= 2;
  return c;
}

// The same where the CTAs of a row need nothing of each other.
inline int parts_for(int64_t rows, int vectors) {
  int c = 1;
  while (rows * c * 2 <= 8 * kNumSMs && vectors >= c * 2 * kRowThreads) c *= 2;
  return c;
}

// A warp for each row, where rows of at most `most` vectors fill more than two waves of
// 128-thread CTAs: a short row's steps wait for one another (memory, barriers, searches), and
// four times as many rows are then in flight. 32768 rows of 2048 bf16, five alternatives: 156 us
// with 128 threads, 58 with a warp; 16384 rows of 16384: 118 and 98; of 32768: 190 and 201.
inline bool warp_rows(int64_t rows, int vectors, int most) { return vectors <= most && rows > 18 * kNumSMs; }

// Host check of a pointer to elements of a logit type.
inline int check_elements(const void* p, int32_t dtype) {
  return reinterpret_cast<uintptr_t>(p) & (dtype == DWARF_F32 ? 3 : 1) ? DWARF_ERR_ALIGN : DWARF_OK;
}

// Host checks shared by the entry points: sizes, strides and the scale of a logit tensor.
inline int check_logits(const void* logits, int32_t dtype, int64_t outer, int64_t inner, int64_t vocab, int64_t so,
                        int64_t si, float inv_temperature) {
  if (outer < 0 || inner < 0 || vocab < 1 || vocab > DWARF_VOCAB_MAX) return DWARF_ERR_SHAPE;
  if (outer > 0 && inner > ((1ll << 28) - 1) / outer) return DWARF_ERR_SHAPE;
  if (so < 0 || si < 0) return DWARF_ERR_STRIDE;
  if (dtype != DWARF_F32 && dtype != DWARF_BF16 && dtype != DWARF_F16) return DWARF_ERR_DTYPE;
  const float c2 = inv_temperature * kLog2e;
  if (!(c2 > 0.0f) || c2 > 3.0e38f) return DWARF_ERR_VALUE;
  if (outer * inner > 0 && logits == nullptr) return DWARF_ERR_NULL;
  return check_elements(logits, dtype);
}

}  // namespace dwarf
