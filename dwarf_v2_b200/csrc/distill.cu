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

static_assert(kRowThreads >= DWARF_TOP_K_MAX, "one thread for each slot of the teacher's list");

// Two passes over the row where the gradient is wanted, the second from L2 (the eight CTAs
// of an SM hold 148 * 8 rows at a time: 77 MB of bf16 at a vocabulary of 32768).
template <typename T>
__global__ void __launch_bounds__(kRowThreads, 1024 / kRowThreads)
    topk_distill_kernel(const dwarf_topk_distill_args a, int cluster) {
  using V = Vec16<T>;
  constexpr int kWarps = kRowThreads / 32;
  extern __shared__ __align__(16) uint32_t listed[];  // a bit for each place of the part
  __shared__ float s_m[kWarps], s_rest[kWarps], s_list[kWarps];
  __shared__ float s_parts[kMaxCluster][3];
  __shared__ float sf[kWarps];
  __shared__ double sd[kWarps];
  __shared__ int s_id[DWARF_TOP_K_MAX];
  __shared__ float s_p[DWARF_TOP_K_MAX];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vocab = (int)a.vocab, k = a.k;
  const int rank = cluster > 1 ? (int)cluster_rank() : 0;
  const int64_t r = blockIdx.x / (unsigned)cluster;
  float scale = a.scale * (a.grad_scale != nullptr ? *a.grad_scale : 1.0f);
  if (a.grad_rows != nullptr) {
    const float g = a.grad_rows[a.grad_rows_stride ? r : 0];
    if (a.skip_if_one && g == 1.0f) return;
    scale *= g;
  }
  if (cluster > 1) cluster_arrive();  // its CTAs have started, before one writes to another
  const T* x = static_cast<const T*>(a.logits) + row_offset(r, a.inner, a.so, a.si);
  const Part<T> part(x, vocab, rank, cluster);
  const RowStore<T> store(static_cast<T*>(a.grad) + r * a.vocab, part.row);

  // the teacher's slots, one a thread
  int id = -1;
  float l = -CUDART_INF_F;
  if (tid < k && (a.row_mask == nullptr || a.row_mask[r])) {
    const int64_t id64 = a.teacher_ids[r * k + tid];
    id = id64 < 0 ? -1 : id64 >= vocab ? vocab : (int)id64;
    if (id >= 0) l = a.teacher_logprobs[r * k + tid];
  }
  const int words = ((part.j1 - part.j0) * V::kVec + 31) / 32;
  for (int i = tid; i < words; i += kRowThreads) listed[i] = 0;
  if (tid < k) s_id[tid] = id;
  const bool used = __syncthreads_or(id >= 0);
  if (cluster > 1) cluster_wait();
  if (!used) {  // the same for the whole cluster
    if (tid == 0 && rank == 0 && a.loss != nullptr) a.loss[r] = 0.0f;
    if (a.grad != nullptr)
      for (int j = part.j0 + tid; j < part.j1; j += kRowThreads) store.zero(j);
    return;
  }
  const bool mine = id >= 0 && id < vocab && part.holds(id);
  bool again = false;  // an id that another slot has too
  if (mine) {
    const int at = id + part.row.lead - part.j0 * V::kVec;
    again = (atomicOr(&listed[at >> 5], 1u << (at & 31)) >> (at & 31)) & 1u;
  }
  const float xv = to_f32(x[id >= 0 && id < vocab ? id : 0]);
  const bool off = __syncthreads_or(id >= vocab);
  // log p of each slot, and the rest: 1 - sum p in 64 bits, for it may be far below 1
  float rest = 0.0f;
  if (a.tail) {
    const double sum = block_reduce<kRowThreads>(id >= 0 ? exp((double)l) : 0.0, sd, AddOp());
    rest = (float)fmax(0.0, 1.0 - sum);
    if (sum != sum) rest = CUDART_NAN_F;
  } else {
    const float top = block_reduce<kRowThreads>(l, sf, MaxOp());
    const float sum = block_reduce<kRowThreads>(id >= 0 && top > -CUDART_INF_F ? expf(l - top) : 0.0f, sf, AddOp());
    l = l - top - logf(sum);
  }
  const float p = id >= 0 ? expf(l) : 0.0f;
  if (tid < k) s_p[tid] = p;
  float weight = block_reduce<kRowThreads>(p, sf, AddOp());
  if (k >= vocab) {  // every id may be listed: nothing is left to be the rest
    float ones = 0.0f;
    for (int i = tid; i < words; i += kRowThreads) ones += __popc(listed[i]);
    if (block_reduce<kRowThreads>(ones, sf, AddOp()) == (float)vocab) rest = 0.0f;
  }
  weight = off ? CUDART_NAN_F : weight + rest;
  const bool repeated = __syncthreads_or(again);

  const float c2 = a.inv_temperature * kLog2e;
  const float2 cc = make_float2(c2, c2);
  float m = -CUDART_INF_F;
  float2 sum = make_float2(0.0f, 0.0f), sum_list = sum;  // the ids not listed; those listed
  for (int first = part.j0; first < part.j1; first += kVectors * kRowThreads) {
    uint4 v[kVectors];
    part.load(first, v);
    typename V::Max mv = V::max_of(v[0]);
#pragma unroll
    for (int i = 1; i < kVectors; ++i) mv = V::join(mv, V::max_of(v[i]));
    const float m_new = fmaxf(m, warp_max(V::largest(mv)));
    if (m > -CUDART_INF_F) {  // a later tile: move the sums to the new maximum
      const float f = ex2_approx((m - m_new) * c2);
      sum = mul2(sum, make_float2(f, f));
      sum_list = mul2(sum_list, make_float2(f, f));
    }
    m = m_new;
    const float s = m == -CUDART_INF_F ? 0.0f : -m;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      if (first + i * kRowThreads >= part.j1) break;
      const int at = (first - part.j0 + i * kRowThreads + tid) * V::kVec;
      uint32_t bits = 0;
      if (first + i * kRowThreads + tid < part.j1)
        bits = (reinterpret_cast<const unsigned char*>(listed)[at >> 3] >> (at & 7)) & ((1u << V::kVec) - 1u);
      float2 e[V::kVec / 2];
      V::unpack(v[i], e);
#pragma unroll
      for (int h = 0; h < V::kVec / 2; ++h) {
        const float2 d = mul2(add2(e[h], make_float2(s, s)), cc);
        e[h] = make_float2(ex2_approx(d.x), ex2_approx(d.y));
      }
      if (bits != 0) {
#pragma unroll
        for (int h = 0; h < V::kVec / 2; ++h) {
          if (bits & (1u << (2 * h))) sum_list.x += e[h].x, e[h].x = 0.0f;
          if (bits & (2u << (2 * h))) sum_list.y += e[h].y, e[h].y = 0.0f;
        }
      }
#pragma unroll
      for (int h = 0; h < V::kVec / 2; ++h) sum = add2(sum, e[h]);
    }
  }
  const float w_rest_sum = warp_sum(sum.x + sum.y), w_list_sum = warp_sum(sum_list.x + sum_list.y);
  if (lane == 0) s_m[warp] = m, s_rest[warp] = w_rest_sum, s_list[warp] = w_list_sum;
  __syncthreads();
  // every warp joins the warps' sums, then the parts' sums, in the same order
  auto join = [&](float& jm, float& jr, float& jl) {
    const float top = warp_max(jm);
    const float f = ex2_approx((jm - (top == -CUDART_INF_F ? 0.0f : top)) * c2);
    jm = top;
    jr = warp_sum(jr == 0.0f ? 0.0f : f * jr);
    jl = warp_sum(jl == 0.0f ? 0.0f : f * jl);
  };
  float s_r = lane < kWarps ? s_rest[lane] : 0.0f, s_l = lane < kWarps ? s_list[lane] : 0.0f;
  m = lane < kWarps ? s_m[lane] : -CUDART_INF_F;
  join(m, s_r, s_l);
  if (cluster > 1) {
    if (tid < 3 * cluster)
      st_cluster(cluster_address(&s_parts[rank][tid % 3], tid / 3), tid % 3 == 0 ? m : tid % 3 == 1 ? s_r : s_l);
    cluster_arrive();
    cluster_wait();
    m = lane < cluster ? s_parts[lane][0] : -CUDART_INF_F;
    s_r = lane < cluster ? s_parts[lane][1] : 0.0f;
    s_l = lane < cluster ? s_parts[lane][2] : 0.0f;
    join(m, s_r, s_l);
  }
  if (m == -CUDART_INF_F) m = 0.0f;
  const float total = s_r + s_l, ln_total = log2f(total) * kLn2;
  if (a.loss != nullptr && rank == 0) {
    float term = p > 0.0f ? p * (l - (xv - m) * a.inv_temperature + ln_total) : p;
    term = block_reduce<kRowThreads>(term, sf, AddOp());
    if (tid == 0) {
      if (!(rest <= 0.0f)) term += rest * (logf(rest) - log2f(s_r) * kLn2 + ln_total);
      a.loss[r] = off ? CUDART_NAN_F : term * a.loss_scale;
    }
  }
  if (a.grad == nullptr) return;
  const float sc = scale * a.inv_temperature;
  const float k_list = sc * weight / total;
  const float k_rest = rest > 0.0f && s_r > 0.0f ? sc * (weight / total - rest / s_r) : k_list;
  const float2 shift = make_float2(-m, -m);
  for (int first = part.j0; first < part.j1; first += kVectors * kRowThreads) {
    uint4 v[kVectors];
    part.load(first, v);
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const int j = first + i * kRowThreads + tid;
      if (j >= part.j1) break;
      float2 e[V::kVec / 2];
      V::unpack(v[i], e);
#pragma unroll
      for (int h = 0; h < V::kVec / 2; ++h) {
        const float2 d = mul2(add2(e[h], shift), cc);
        e[h] = mul2(make_float2(ex2_approx(d.x), ex2_approx(d.y)), make_float2(k_rest, k_rest));
      }
      store.put(j, V::pack(e));
    }
  }
  __syncthreads();  // the listed entries are written again, with their own terms
  if (!mine) return;
  float taken = p;
  if (repeated) {
    taken = 0.0f;
    for (int j = 0; j < k; ++j)
      if (s_id[j] == id) taken += s_p[j];
  }
  store.out[id] = from_f32<T>(ex2_approx((xv - m) * c2) * k_list - sc * taken);
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
  const int64_t rows = a.outer * a.inner;
  const int vectors = ceil_div((int)a.vocab, Vec16<T>::kVec);
  const int cluster = cluster_for(rows, vectors, 262144 / Vec16<T>::kVec);  // a bit for each place: at most 32 KB
  // a row that starts off a 16-byte boundary has one vector more
  const int bytes = (ceil_div(vectors + 1, cluster) * Vec16<T>::kVec + 31) / 32 * 4;
  return launch_rows(topk_distill_kernel<T>, rows, cluster, kRowThreads, bytes, stream, a, cluster);
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
