// Distillation from a teacher's top entries: per row KL(teacher || student) and
// the gradient of the student's logits.
//
// With c = 1/temperature, d = c (x - max x), S = sum exp(d) over the row and
// S_* its part over the ids that the teacher does not list:
//   loss = sum_k p_k (log p_k - d_k + log S) + p_* (log p_* - log S_* + log S)
//   grad_v = s c (exp(d_v) / S * W - [v listed] sum p - [v not listed] p_* exp(d_v) / S_*),  W = sum p + p_*.
// S_* is a sum of its own: S minus the listed entries would cancel where the
// student has learnt the list. A bit per vocabulary entry says what is listed.
#include "vocab_row.cuh"

namespace dwarf {
namespace {

constexpr int kThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kThreads) topk_distill_kernel(dwarf_topk_distill_args a) {
  extern __shared__ uint32_t listed[];  // one bit per vocabulary entry
  __shared__ float sf[kThreads / 32];
  __shared__ double sd[kThreads / 32];
  __shared__ int s_id[DWARF_TOP_K_MAX];
  __shared__ float s_p[DWARF_TOP_K_MAX];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, vocab = (int)a.vocab, k = a.k;
  float scale = a.scale * (a.grad_scale != nullptr ? *a.grad_scale : 1.0f);
  if (a.grad_rows != nullptr) {
    const float g = a.grad_rows[a.grad_rows_stride ? row : 0];
    if (a.skip_if_one && g == 1.0f) return;
    scale *= g;
  }
  const T* x = static_cast<const T*>(a.logits) + row_offset(row, a.inner, a.so, a.si);
  T* out = a.grad != nullptr ? static_cast<T*>(a.grad) + row * a.vocab : nullptr;

  int id = -1;
  float l = -CUDART_INF_F;
  if (tid < k && (a.row_mask == nullptr || a.row_mask[row])) {
    const int64_t id64 = a.teacher_ids[row * k + tid];
    id = id64 < 0 ? -1 : id64 >= vocab ? vocab : (int)id64;
    if (id >= 0) l = a.teacher_logprobs[row * k + tid];
  }
  const int used = __syncthreads_or(id >= 0);
  const bool off = __syncthreads_or(id >= vocab);
  if (!used) {
    if (tid == 0 && a.loss != nullptr) a.loss[row] = 0.0f;
    if (out != nullptr)
      for (int i = tid; i < vocab; i += kThreads) out[i] = from_f32<T>(0.0f);
    return;
  }
  for (int i = tid; i < (vocab + 31) / 32; i += kThreads) listed[i] = 0;
  if (tid < k) s_id[tid] = id;
  __syncthreads();
  if (id >= 0 && id < vocab) atomicOr(&listed[id >> 5], 1u << (id & 31));
  // teacher: log p of each slot, and the rest. 1 - sum p is formed in 64 bits: it may be far below 1.
  float rest = 0.0f;
  if (a.tail) {
    const double sum = block_reduce<kThreads>(id >= 0 ? exp((double)l) : 0.0, sd, AddOp());
    rest = (float)fmax(0.0, 1.0 - sum);
    if (sum != sum) rest = CUDART_NAN_F;
  } else {
    const float top = block_reduce<kThreads>(l, sf, MaxOp());
    const float sum = block_reduce<kThreads>(id >= 0 && top > -CUDART_INF_F ? expf(l - top) : 0.0f, sf, AddOp());
    l = l - top - logf(sum);
  }
  const float p = id >= 0 ? expf(l) : 0.0f;
  if (tid < k) s_p[tid] = p;
  const float weight = off ? CUDART_NAN_F : block_reduce<kThreads>(p, sf, AddOp()) + rest;
  __syncthreads();

  const float c2 = a.inv_temperature * kLog2e;
  float m = -CUDART_INF_F;
  for (int i = tid; i < vocab; i += kThreads) m = fmaxf(m, to_f32(x[i]));
  m = block_reduce<kThreads>(m, sf, MaxOp());
  if (m == -CUDART_INF_F) m = 0.0f;
  float s_rest = 0.0f, s_list = 0.0f;
  int n_list = 0;
  for (int i = tid; i < vocab; i += kThreads) {
    const float e = ex2_approx((to_f32(x[i]) - m) * c2);
    if ((listed[i >> 5] >> (i & 31)) & 1u) {
      s_list += e;
      ++n_list;
    } else {
      s_rest += e;
    }
  }
  s_rest = block_reduce<kThreads>(s_rest, sf, AddOp());
  s_list = block_reduce<kThreads>(s_list, sf, AddOp());
  if (block_reduce<kThreads>((float)n_list, sf, AddOp()) == (float)vocab) rest = 0.0f;  // nothing is left to be the rest
  const float total = s_rest + s_list, log2s = log2f(total);
  if (a.loss != nullptr) {
    float term = p > 0.0f ? p * (l - (to_f32(x[id < vocab ? id : 0]) - m) * a.inv_temperature + log2s * kLn2) : p;
    term = block_reduce<kThreads>(term, sf, AddOp());
    if (tid == 0) {
      if (!(rest <= 0.0f)) term += rest * (logf(rest) - (log2f(s_rest) - log2s) * kLn2);
      a.loss[row] = off ? CUDART_NAN_F : term * a.loss_scale;
    }
  }
  if (out == nullptr) return;
  const float sc = scale * a.inv_temperature;
  const float w_list = sc * weight / total;
  const float w_rest = rest > 0.0f && s_rest > 0.0f ? sc * (weight / total - rest / s_rest) : w_list;
  for (int i = tid; i < vocab; i += kThreads) out[i] = from_f32<T>(ex2_approx((to_f32(x[i]) - m) * c2) * w_rest);
  __syncthreads();  // the listed entries are written again, with their own terms
  if (id < 0 || id >= vocab) return;
  float sum = 0.0f;
  for (int j = 0; j < k; ++j)
    if (s_id[j] == id) sum += s_p[j];
  out[id] = from_f32<T>(ex2_approx((to_f32(x[id]) - m) * c2) * w_list - sc * sum);
}

__global__ void __launch_bounds__(1024) row_reduce_kernel(dwarf_row_reduce_args a) {
  __shared__ double sd[32];
  double sum = 0.0;
  for (int64_t i = threadIdx.x; i < a.rows; i += 1024) sum += a.values != nullptr ? (double)a.values[i] : (double)(a.mask[i] != 0);
  sum = block_reduce<1024>(sum, sd, AddOp());
  if (threadIdx.x != 0) return;
  if (a.values == nullptr) {
    *a.out = (float)(1.0 / fmax(1.0, sum));
  } else {
    const double scale = (a.scale != nullptr ? (double)*a.scale : 1.0) * (double)a.host_scale;
    *a.out = (float)(sum * scale);
  }
}

template <typename T>
int launch_distill(const dwarf_topk_distill_args& a, cudaStream_t stream) {
  const size_t bytes = (size_t)((a.vocab + 31) / 32) * 4;
  if (bytes > 40 * 1024) {
    if (cudaFuncSetAttribute(topk_distill_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) !=
        cudaSuccess)
      return launch_status();
  }
  topk_distill_kernel<T><<<(unsigned)(a.outer * a.inner), kThreads, bytes, stream>>>(a);
  return launch_status();
}

}  // namespace
}  // namespace dwarf

extern "C" int dwarf_topk_distill(const dwarf_topk_distill_args* args, void* stream) {
  using namespace dwarf;
  DWARF_CHECK_VERSION(args);
  const dwarf_topk_distill_args a = *args;
  int st = check_logits(a.logits, a.dtype, a.outer, a.inner, a.vocab, a.so, a.si, a.inv_temperature);
  if (st != DWARF_OK) return st;
  if (a.k < 1 || a.k > DWARF_TOP_K_MAX) return DWARF_ERR_SHAPE;
  if (a.tail != 0 && a.tail != 1) return DWARF_ERR_VALUE;
  if (a.grad_rows_stride != 0 && a.grad_rows_stride != 1) return DWARF_ERR_VALUE;
  if (a.skip_if_one && (a.grad_rows == nullptr || a.grad_rows_stride != 0 || a.loss != nullptr)) return DWARF_ERR_VALUE;
  if (a.outer * a.inner == 0) return DWARF_OK;
  if (a.teacher_ids == nullptr || a.teacher_logprobs == nullptr) return DWARF_ERR_NULL;
  if (a.loss == nullptr && a.grad == nullptr) return DWARF_ERR_NULL;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == DWARF_F32) return launch_distill<float>(a, s);
  if (a.dtype == DWARF_BF16) return launch_distill<__nv_bfloat16>(a, s);
  return launch_distill<__half>(a, s);
}

extern "C" int dwarf_row_reduce(const dwarf_row_reduce_args* args, void* stream) {
  using namespace dwarf;
  DWARF_CHECK_VERSION(args);
  const dwarf_row_reduce_args a = *args;
  if (a.rows < 0) return DWARF_ERR_SHAPE;
  if (a.out == nullptr || (a.rows > 0 && a.values == nullptr && a.mask == nullptr)) return DWARF_ERR_NULL;
  row_reduce_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return launch_status();
}
