// Log probabilities of given tokens with the entropy and the best alternatives
// of each logit row, and the gradient of the logits.
//
// With c = 1/temperature, m = max x, d = c (x - m), e = exp(d), S = sum e, T = sum e d:
//   lse = c m + log S, logprob = d[target] - log S, entropy = log S - T / S.
// x - m is formed before the scale, so a row at the type's lowest value does
// not overflow; e d is taken as 0 where e is 0 (masked entries, d = -inf).
#include "vocab_row.cuh"

namespace dwarf {
namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(dwarf_token_logprobs_args a) {
  __shared__ float sf[kThreads / 32];
  __shared__ uint64_t sk[kThreads / 32];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row_offset(row, a.inner, a.so, a.si);
  const int vocab = (int)a.vocab;
  const float c2 = a.inv_temperature * kLog2e;
  float m = -CUDART_INF_F;
  for (int i = threadIdx.x; i < vocab; i += kThreads) m = fmaxf(m, to_f32(x[i]));
  m = block_reduce<kThreads>(m, sf, MaxOp());
  if (m == -CUDART_INF_F) m = 0.0f;
  float s = 0.0f, t = 0.0f;
  for (int i = threadIdx.x; i < vocab; i += kThreads) {
    const float d = (to_f32(x[i]) - m) * c2;
    const float e = ex2_approx(d);
    s += e;
    t += e * fmaxf(d, -200.0f);
  }
  s = block_reduce<kThreads>(s, sf, AddOp());
  t = block_reduce<kThreads>(t, sf, AddOp());
  const float log2s = log2f(s);  // -inf for a row without a finite logit
  if (threadIdx.x == 0) {
    a.lse[row] = s > 0.0f ? fmaf(m, a.inv_temperature, log2s * kLn2) : s == 0.0f ? -CUDART_INF_F : s;
    a.entropy[row] = s == 0.0f ? 0.0f : (log2s - t / s) * kLn2;
    if (a.stats != nullptr) reinterpret_cast<float2*>(a.stats)[row] = make_float2(m, s);
    if (a.logprob != nullptr) {
      const int64_t id = a.targets[row];
      float lp = 0.0f;
      if (id != a.ignore_index) {
        lp = CUDART_NAN_F;
        if (id >= 0 && id < vocab) lp = s == 0.0f ? -CUDART_INF_F : (to_f32(x[id]) - m) * a.inv_temperature - log2s * kLn2;
      }
      a.logprob[row] = lp;
    }
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
      const uint64_t key = entry_key(to_f32(x[i]), (uint32_t)i);
      if (key < last && key > best) best = key;
    }
    last = block_reduce<kThreads>(best, sk, MaxOp());
    if (threadIdx.x == 0) {
      const uint32_t id = entry_id(last);
      a.top_ids[row * a.top_k + k] = id;
      a.top_logprobs[row * a.top_k + k] = s == 0.0f ? -CUDART_INF_F : (to_f32(x[id]) - m) * a.inv_temperature - log2s * kLn2;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_bwd_kernel(dwarf_token_logprobs_bwd_args a) {
  __shared__ float sf[kThreads / 32];
  __shared__ int64_t s_id[DWARF_TOP_K_MAX + 1];
  __shared__ float s_g[DWARF_TOP_K_MAX + 1];
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row_offset(row, a.inner, a.so, a.si);
  T* out = static_cast<T*>(a.grad) + row * a.vocab;
  const int vocab = (int)a.vocab;
  const float c2 = a.inv_temperature * kLog2e;
  const float2 ms = reinterpret_cast<const float2*>(a.stats)[row];
  // entry 0: the target; entries 1..top_k: the alternatives
  float g_lp = a.g_logprob != nullptr ? a.g_logprob[row] : 0.0f;
  const int64_t target = a.targets != nullptr ? a.targets[row] : -1;
  if (a.targets == nullptr || target == a.ignore_index) g_lp = 0.0f;
  const bool off = g_lp != 0.0f && (target < 0 || target >= vocab);
  const int n = a.g_top != nullptr ? a.top_k + 1 : 1;
  float g = 0.0f;
  bool any = g_lp != 0.0f;
  for (int j = threadIdx.x; j < n; j += kThreads) {
    const float v = j == 0 ? g_lp : a.g_top[row * a.top_k + j - 1];
    s_id[j] = j == 0 ? (g_lp != 0.0f && !off ? target : -1) : a.top_ids[row * a.top_k + j - 1];
    s_g[j] = v;
    g += v;
    any |= v != 0.0f;
  }
  g = block_reduce<kThreads>(g, sf, AddOp());
  const float g_lse = a.g_lse != nullptr ? a.g_lse[row] : 0.0f;
  const float g_h = a.g_entropy != nullptr ? a.g_entropy[row] : 0.0f;
  any = __syncthreads_or(any) || g_lse != 0.0f || g_h != 0.0f;
  if (!any || ms.y == 0.0f) {
    for (int i = threadIdx.x; i < vocab; i += kThreads) out[i] = from_f32<T>(0.0f);
    return;
  }
  const float weight = off ? CUDART_NAN_F : g - g_lse;
  const float inv_s = 1.0f / ms.y, log2s = log2f(ms.y), h2 = a.entropy[row] * kLog2e - log2s;
  auto dense = [&](float v) {
    const float d = (v - ms.x) * c2;
    const float q = ex2_approx(d) * inv_s;
    return -q * (weight + g_h * kLn2 * (fmaxf(d, -200.0f) + h2));
  };
  for (int i = threadIdx.x; i < vocab; i += kThreads) out[i] = from_f32<T>(a.inv_temperature * dense(to_f32(x[i])));
  __syncthreads();  // the listed entries are written again, with their own terms
  for (int j = threadIdx.x; j < n; j += kThreads) {
    const int64_t id = s_id[j];
    if (id < 0 || id >= vocab) continue;
    float sum = 0.0f;
    for (int l = 0; l < n; ++l)
      if (s_id[l] == id) sum += s_g[l];
    out[id] = from_f32<T>(a.inv_temperature * (sum + dense(to_f32(x[id]))));
  }
}

template <typename F>
int with_type(int32_t dtype, F f) {
  if (dtype == DWARF_F32) return f(float());
  if (dtype == DWARF_BF16) return f(__nv_bfloat16());
  return f(__half());
}

}  // namespace
}  // namespace dwarf

extern "C" int dwarf_token_logprobs(const dwarf_token_logprobs_args* args, void* stream) {
  using namespace dwarf;
  DWARF_CHECK_VERSION(args);
  const dwarf_token_logprobs_args a = *args;
  int st = check_logits(a.logits, a.dtype, a.outer, a.inner, a.vocab, a.so, a.si, a.inv_temperature);
  if (st != DWARF_OK) return st;
  if (a.top_k < 0 || a.top_k > DWARF_TOP_K_MAX || a.top_k > a.vocab) return DWARF_ERR_SHAPE;
  const int64_t rows = a.outer * a.inner;
  if (rows == 0) return DWARF_OK;
  if (a.lse == nullptr || a.entropy == nullptr) return DWARF_ERR_NULL;
  if ((a.targets == nullptr) != (a.logprob == nullptr)) return DWARF_ERR_NULL;
  if (a.top_k > 0 && (a.top_logprobs == nullptr || a.top_ids == nullptr)) return DWARF_ERR_NULL;
  return with_type(a.dtype, [&](auto t) {
    token_logprobs_kernel<decltype(t)><<<(unsigned)rows, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return launch_status();
  });
}

extern "C" int dwarf_token_logprobs_bwd(const dwarf_token_logprobs_bwd_args* args, void* stream) {
  using namespace dwarf;
  DWARF_CHECK_VERSION(args);
  const dwarf_token_logprobs_bwd_args a = *args;
  int st = check_logits(a.logits, a.dtype, a.outer, a.inner, a.vocab, a.so, a.si, a.inv_temperature);
  if (st != DWARF_OK) return st;
  if (a.top_k < 0 || a.top_k > DWARF_TOP_K_MAX || a.top_k > a.vocab) return DWARF_ERR_SHAPE;
  const int64_t rows = a.outer * a.inner;
  if (rows == 0) return DWARF_OK;
  if (a.stats == nullptr || a.entropy == nullptr || a.grad == nullptr) return DWARF_ERR_NULL;
  if (a.g_logprob != nullptr && a.targets == nullptr) return DWARF_ERR_NULL;
  if (a.g_top != nullptr && (a.top_ids == nullptr || a.top_k < 1)) return DWARF_ERR_NULL;
  return with_type(a.dtype, [&](auto t) {
    token_logprobs_bwd_kernel<decltype(t)><<<(unsigned)rows, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return launch_status();
  });
}
