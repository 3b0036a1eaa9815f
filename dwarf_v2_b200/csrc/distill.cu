// Distillation from a teacher's top entries: per row KL(teacher || student) and
// the gradient of the student's logits.
//
// With c = 1/temperature, m = max x, S = sum exp(c (x - m)) over the row, and S_* = sum exp(c
// (x - m_*)) over the ids that the teacher does not list:
//   loss = sum_k p_k (log p_k - c (x_k - m) + log S) + p_* (log p_* - c (m_* - m) - log S_* + log S)
//   grad_v = s c (q_v W - [v listed] sum p - [v not listed] p_* exp(c (x_v - m_*)) / S_*),  W = sum p + p_*.
// S_* is a sum of its own: S minus the listed entries would cancel where the student has
// learnt the list. A bit per vocabulary entry says what is listed. m_* is m; where the list lies so
// far above the rest that S_* would vanish in fp32, the rest is summed once more relative to its own maximum.
#include "vocab_row.cuh"

namespace dwarf {
namespace {

// (m, sums relative to m) of a warp's lanes joined, in a fixed order; lanes without a part: m = -inf, sums 0.
__device__ __forceinline__ void warp_join(float c2, float& m, float& a, float& b) {
  const float top = warp_max(m);
  const float f = ex2_approx((m - (top == -CUDART_INF_F ? 0.0f : top)) * c2);
  m = top;
  a = warp_sum(a == 0.0f ? 0.0f : f * a);
  b = warp_sum(b == 0.0f ? 0.0f : f * b);
}

// One row, or a CTA's part of one. kKnown: the gradient from the sums that a launch with
// the loss has left in `stats`; the parts need nothing of each other. Otherwise the CTAs of a row are a cluster.
template <typename T, int NT, bool kGrad, bool kKnown>
__device__ __forceinline__ void distill_row(const dwarf_topk_distill_args& a, int parts, int rank, int64_t r) {
  using V = Vec16<T>;
  constexpr int kWarps = NT / 32, kTile = kVectors * NT;
  constexpr int kSlots = NT < DWARF_TOP_K_MAX ? DWARF_TOP_K_MAX / NT : 1;  // slots of the teacher's list for a thread
  constexpr int kListWarps = NT < DWARF_TOP_K_MAX ? kWarps : DWARF_TOP_K_MAX / 32;
  extern __shared__ __align__(16) uint32_t listed[];  // a bit for each place of the part
  __shared__ float s_m[kWarps], s_rest[kWarps], s_list[kWarps];
  __shared__ float s_top[kListWarps], s_term[kListWarps];
  __shared__ double s_sum[kListWarps];
  __shared__ float s_parts[kMaxCluster][3], s_own[kMaxCluster][2];
  __shared__ int s_id[DWARF_TOP_K_MAX];
  __shared__ float s_p[DWARF_TOP_K_MAX];
  __shared__ int s_flags, s_listed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vocab = (int)a.vocab, k = a.k;
  const int cluster = kKnown ? 1 : parts;
  if (cluster > 1) cluster_arrive();  // its CTAs have started, before one writes to another
  const T* x = static_cast<const T*>(a.logits) + row_offset(r, a.inner, a.so, a.si);
  const Part<T, NT> part(x, vocab, rank, parts);
  constexpr bool kTwice = kGrad && !kKnown;  // the row is read a second time, from L2
  const uint64_t keep = kTwice ? policy_keep() : 0;

  // the teacher's slots
  const bool counted = a.row_mask == nullptr || a.row_mask[r] != 0;
  if (kTwice && tid == 0 && counted) part.prefetch_kept(keep);
  int id[kSlots];  // -1: not used; vocab: past the vocabulary
  float l[kSlots];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    const int slot = tid + s * NT;
    id[s] = -1;
    l[s] = -CUDART_INF_F;
    if (slot < k && counted) {
      const int64_t id64 = a.teacher_ids[r * k + slot];
      l[s] = a.teacher_logprobs[r * k + slot];
      id[s] = id64 < 0 ? -1 : id64 >= vocab ? vocab : (int)id64;
      if (id[s] < 0) l[s] = -CUDART_INF_F;
    }
  }
  const int words = ((part.j1 - part.j0) * V::kVec + 31) / 32;
  if (!kKnown)
    for (int i = tid; i < words; i += NT) listed[i] = 0;
  bool any = false;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    if (tid + s * NT < k) s_id[tid + s * NT] = id[s];
    any |= id[s] >= 0;
  }
  if (tid == 0) s_flags = s_listed = 0;
  const RowStore<T> store(static_cast<T*>(a.grad) + r * a.vocab, part.row);
  const int end_id = warp == 0 ? part.end_id(lane) : -1;
  const float end = end_id >= 0 && counted ? to_f32(x[end_id]) : -CUDART_INF_F;
  const bool used = __syncthreads_or(any);
  if (cluster > 1) cluster_wait();
  if (!used) {  // the same for the whole cluster
    if (tid == 0 && rank == 0 && a.loss != nullptr) a.loss[r] = 0.0f;
    if (kGrad) store.zero(part);
    return;
  }
  float xv[kSlots];
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    if (!kKnown && id[s] >= 0 && id[s] < vocab && part.holds(id[s])) {
      const int at = id[s] + part.row.lead - part.j0 * V::kVec;
      const uint32_t bit = 1u << (at & 31);
      if (atomicOr(&listed[at >> 5], bit) & bit) atomicOr(&s_flags, 1);  // an id that another slot has too
    }
    if (id[s] >= vocab) atomicOr(&s_flags, 2);
    xv[s] = to_f32(x[id[s] >= 0 && id[s] < vocab ? id[s] : 0]);
  }
  // sum p for a teacher with a tail, in 64 bits (the rest, 1 - sum p, may be far below 1); else the
  // list's maximum and the sum relative to it
  if (warp < kListWarps) {
    if (a.tail) {
      double sum = 0.0;
#pragma unroll
      for (int s = 0; s < kSlots; ++s) sum += id[s] >= 0 ? exp((double)l[s]) : 0.0;
      sum = warp_sum(sum);
      if (lane == 0) s_sum[warp] = sum;
    } else {
      float top = l[0], sum = 0.0f;
#pragma unroll
      for (int s = 1; s < kSlots; ++s) top = fmaxf(top, l[s]);
      top = warp_max(top);
#pragma unroll
      for (int s = 0; s < kSlots; ++s) sum += l[s] > -CUDART_INF_F ? expf(l[s] - top) : l[s] == l[s] ? 0.0f : l[s];
      sum = warp_sum(sum);
      if (lane == 0) s_top[warp] = top, s_sum[warp] = sum;
    }
  }
  __syncthreads();

  const float c2 = a.inv_temperature * kLog2e;
  const float2 cc = make_float2(c2, c2);
  auto teacher_sum = [&] {
    double sum_p = 0.0;
#pragma unroll
    for (int w = 0; w < kListWarps; ++w) sum_p += s_sum[w];
    return sum_p;
  };
  float m = -CUDART_INF_F, m_rest, s_r, total, rest = 0.0f;
  if (!kKnown) {
    float s_l;
    float2 sum = make_float2(0.0f, 0.0f), sum_list = sum;
    for (int at = 0; at < part.size(); at += kTile) {
      uint4 v[kVectors];
      if (kTwice) part.load(at, v, keep); else part.load(at, v);
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
      // the bits of a thread's vectors of a tile lie NT kVec / 8 bytes apart
      const int place = part.w0 - part.j0 + at + tid;
      const unsigned char* bits = reinterpret_cast<const unsigned char*>(listed) + place * V::kVec / 8;
      const int bits_shift = V::kVec == 4 ? 4 * (place & 1) : 0;
      auto add = [&](const uint4& w, uint32_t mask) {
        float2 e[V::kVec / 2];
        V::unpack(w, e);
#pragma unroll
        for (int h = 0; h < V::kVec / 2; ++h) {
          const float2 d = mul2(add2(e[h], make_float2(s, s)), cc);
          e[h] = make_float2(ex2_approx(d.x), ex2_approx(d.y));
        }
        if (mask != 0) {
#pragma unroll
          for (int h = 0; h < V::kVec / 2; ++h) {
            if (mask & (1u << (2 * h))) sum_list.x += e[h].x, e[h].x = 0.0f;
            if (mask & (2u << (2 * h))) sum_list.y += e[h].y, e[h].y = 0.0f;
          }
        }
#pragma unroll
        for (int h = 0; h < V::kVec / 2; ++h) sum = add2(sum, e[h]);
      };
      if (at + kTile <= part.size()) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
          add(v[i], (bits[i * NT * V::kVec / 8] >> bits_shift) & ((1u << V::kVec) - 1u));
      } else {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) {
          if (at + i * NT >= part.size()) break;
          const bool in = at + i * NT + tid < part.size();  // vectors outside hold -inf
          add(v[i], in ? (bits[i * NT * V::kVec / 8] >> bits_shift) & ((1u << V::kVec) - 1u) : 0u);
        }
      }
    }
    if (warp == 0 && part.ends()) {
      const float m_new = fmaxf(m, warp_max(end)), base = m_new == -CUDART_INF_F ? 0.0f : m_new;
      const float f = ex2_approx((m - base) * c2), e = ex2_approx((end - base) * c2);
      sum = mul2(sum, make_float2(f, f));
      sum_list = mul2(sum_list, make_float2(f, f));
      const int at = end_id + part.row.lead - part.j0 * V::kVec;
      if (end_id >= 0 && ((listed[at >> 5] >> (at & 31)) & 1u)) sum_list.x += e; else sum.x += e;
      m = m_new;
    }
    s_r = warp_sum(sum.x + sum.y);
    s_l = warp_sum(sum_list.x + sum_list.y);
    if (lane == 0) s_m[warp] = m, s_rest[warp] = s_r, s_list[warp] = s_l;
    if (k >= vocab) {  // every id may be listed: nothing is left to be the rest
      for (int i = tid; i < words; i += NT) atomicAdd(&s_listed, __popc(listed[i]));
    }
    __syncthreads();
    // every warp joins the warps' sums, then the parts' sums, in the same order
    s_r = lane < kWarps ? s_rest[lane] : 0.0f;
    s_l = lane < kWarps ? s_list[lane] : 0.0f;
    m = lane < kWarps ? s_m[lane] : -CUDART_INF_F;
    warp_join(c2, m, s_r, s_l);
    if (cluster > 1) {
      if (tid < 3 * cluster)
        st_cluster(cluster_address(&s_parts[rank][tid % 3], tid / 3), tid % 3 == 0 ? m : tid % 3 == 1 ? s_r : s_l);
      cluster_arrive();
      cluster_wait();
      m = lane < cluster ? s_parts[lane][0] : -CUDART_INF_F;
      s_r = lane < cluster ? s_parts[lane][1] : 0.0f;
      s_l = lane < cluster ? s_parts[lane][2] : 0.0f;
      warp_join(c2, m, s_r, s_l);
    }
    if (m == -CUDART_INF_F) m = 0.0f;
    m_rest = m;
    total = s_r + s_l;
    if (a.tail && s_listed != vocab) {
      const double sum_p = teacher_sum();
      rest = sum_p == sum_p ? (float)fmax(0.0, 1.0 - sum_p) : CUDART_NAN_F;
    }
    // Entries below 2^-126 of the maximum count as 0. While the rest is 2^-40 or more, they are at
    // most 2^-66 of it together, and the share of each in its gradient 2^-86. Below, the rest
    // is summed again, relative to its own maximum.
    if (rest > 0.0f && s_r < 0x1p-40f) {
      m_rest = -CUDART_INF_F;
      s_r = 0.0f;
      for (int at = -NT; at < part.size(); at += NT) {  // the row's ends, then a vector a thread
        uint4 v = make_uint4(V::kMinusInf, V::kMinusInf, V::kMinusInf, V::kMinusInf);
        const int place = part.w0 - part.j0 + at + tid;
        if (at >= 0 && at + tid < part.size()) {
          v = part.row.load(part.w0 + at + tid);
          const uint32_t bits = listed[place * V::kVec / 32] >> (place * V::kVec % 32);
          v = V::drop(v, bits & ((1u << V::kVec) - 1u));
        }
        float own = V::largest(V::max_of(v));
        const int end_at = end_id + part.row.lead - part.j0 * V::kVec;
        if (at < 0 && end_id >= 0 && !((listed[end_at >> 5] >> (end_at & 31)) & 1u)) own = end;
        const float m_new = fmaxf(m_rest, warp_max(own)), base = m_new == -CUDART_INF_F ? 0.0f : m_new;
        s_r *= m_rest == -CUDART_INF_F ? 0.0f : ex2_approx((m_rest - base) * c2);
        if (at < 0) {
          s_r += ex2_approx((own - base) * c2);
        } else {
          float2 e[V::kVec / 2];
          V::unpack(v, e);
#pragma unroll
          for (int h = 0; h < V::kVec / 2; ++h)
            s_r += ex2_approx((e[h].x - base) * c2) + ex2_approx((e[h].y - base) * c2);
        }
        m_rest = m_new;
      }
      s_r = warp_sum(s_r);
      __syncthreads();  // all have read the earlier sums
      if (lane == 0) s_m[warp] = m_rest, s_rest[warp] = s_r;
      __syncthreads();
      float none = 0.0f;
      s_r = lane < kWarps ? s_rest[lane] : 0.0f;
      m_rest = lane < kWarps ? s_m[lane] : -CUDART_INF_F;
      warp_join(c2, m_rest, s_r, none);
      if (cluster > 1) {
        if (tid < 2 * cluster) st_cluster(cluster_address(&s_own[rank][tid & 1], tid >> 1), tid & 1 ? s_r : m_rest);
        cluster_arrive();
        cluster_wait();
        m_rest = lane < cluster ? s_own[lane][0] : -CUDART_INF_F;
        s_r = lane < cluster ? s_own[lane][1] : 0.0f;
        warp_join(c2, m_rest, s_r, none);
      }
      if (m_rest == -CUDART_INF_F) m_rest = m;  // nothing: the loss is inf, the entries' gradients 0
    }
  } else {
    const float4* known = reinterpret_cast<const float4*>(a.stats) + 2 * r;
    const float4 first = known[0];
    m_rest = first.x, s_r = first.y, m = first.z, total = first.w, rest = known[1].x;
  }
  // the teacher: log p of the slot, sum p + rest, the rest
  const bool off = s_flags & 2;
  float weight = 1.0f;
  if (a.tail) {
    weight = (float)(teacher_sum() + (double)rest);
  } else {
    float top = -CUDART_INF_F, all = 0.0f;
#pragma unroll
    for (int w = 0; w < kListWarps; ++w) top = fmaxf(top, s_top[w]);
#pragma unroll
    for (int w = 0; w < kListWarps; ++w) all += s_sum[w] == 0.0 ? 0.0f : (float)s_sum[w] * expf(s_top[w] - top);
    const float ln_sum = logf(all);
#pragma unroll
    for (int s = 0; s < kSlots; ++s) l[s] = l[s] - top - ln_sum;
    if (!(all > 0.0f)) weight = CUDART_NAN_F;  // no slot with a finite value
  }
  if (off) weight = CUDART_NAN_F;
  float p[kSlots], term = 0.0f;
  // A row without a finite logit (m = 0 here): log q is -inf everywhere, so the loss is inf where
  // the teacher gives anything, and the gradient 0 (NaN for a NaN teacher).
  const bool empty = total == 0.0f;
  const float ln_total = empty ? 0.0f : log2f(total) * kLn2;
#pragma unroll
  for (int s = 0; s < kSlots; ++s) {
    p[s] = id[s] >= 0 ? expf(l[s]) : 0.0f;
    term += p[s] > 0.0f ? p[s] * (l[s] - (xv[s] - m) * a.inv_temperature + ln_total) : p[s];
    if (tid + s * NT < k) s_p[tid + s * NT] = p[s];
  }
  if (a.loss != nullptr && warp < kListWarps) {
    term = warp_sum(term);
    if (lane == 0) s_term[warp] = term;
  }
  float sc = 0.0f, k_list = 0.0f;
  if (kGrad) {
    sc = a.scale * a.inv_temperature;
    if (a.grad_scale != nullptr) sc *= *a.grad_scale;
    if (a.grad_rows != nullptr) sc *= a.grad_rows[a.grad_rows_stride ? r : 0];
    k_list = empty ? 0.0f * weight : sc * weight / total;
    if (empty) sc = 0.0f;
    // of exp(c (x - m_*)): q_v W and the rest's share
    float k_rest = ex2_approx((m_rest - m) * c2) * k_list;
    if (rest > 0.0f && s_r > 0.0f) k_rest -= sc * rest / s_r;
    const float2 shift = make_float2(-m_rest, -m_rest);
    const uint64_t leave = policy_leave();
    for (int at = 0; at < part.size(); at += kTile) {
      uint4 v[kVectors];
      if (kTwice) part.load(at, v, leave); else part.load(at, v);
      store.tile(part, at, v, [&](const uint4& w) {
        float2 e[V::kVec / 2];
        V::unpack(w, e);
#pragma unroll
        for (int h = 0; h < V::kVec / 2; ++h) {
          const float2 d = mul2(add2(e[h], shift), cc);
          e[h] = mul2(make_float2(ex2_approx(d.x), ex2_approx(d.y)), make_float2(k_rest, k_rest));
        }
        return V::pack(e);
      });
    }
    if (end_id >= 0) store.out[end_id] = from_f32<T>(ex2_approx((end - m_rest) * c2) * k_rest);
  }
  __syncthreads();  // the listed entries are written again, with their own terms
  if (kGrad) {
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      if (id[s] < 0 || id[s] >= vocab || !part.holds(id[s])) continue;
      float taken = p[s];
      if (kKnown || (s_flags & 1)) {
        taken = 0.0f;
        for (int j = 0; j < k; ++j)
          if (s_id[j] == id[s]) taken += s_p[j];
      }
      store.out[id[s]] = from_f32<T>(ex2_approx((xv[s] - m) * c2) * k_list - sc * taken);
    }
  }
  if (a.loss != nullptr && rank == 0 && tid == 0) {
    term = 0.0f;
#pragma unroll
    for (int w = 0; w < kListWarps; ++w) term += s_term[w];
    if (!(rest <= 0.0f))
      term += rest * (logf(rest) - log2f(s_r) * kLn2 - (m_rest - m) * a.inv_temperature + ln_total);
    a.loss[r] = off ? CUDART_NAN_F : term * a.loss_scale;
    if (a.stats != nullptr) {
      float4* known = reinterpret_cast<float4*>(a.stats) + 2 * r;
      known[0] = make_float4(m_rest, s_r, m, total);
      known[1] = make_float4(rest, 0.0f, 0.0f, 0.0f);
    }
  }
}

// The loss, and with kGrad the gradient in the same launch: the row is then read twice, the
// second time from L2. One bulk prefetch at the start fetches the row while the teacher's list
// is read, under a policy that keeps it there, and the threads of a CTA are chosen so that the
// rows in flight are about 40 MB. 16384 rows of 32768 bf16, 64 entries: 390 us (128 threads
// without either: 534, with 475 MB read for 268; the row held in shared memory: 483; 512
// threads: 540). It ends at 512 threads: against two passes over the rows at the copy's rate the
// launch takes 1.28 times as long at 32768 bf16, 1.29 at 131072, and 1.51 at 262144 (fp32: 1.18 at
// 32768, 1.47 at 131072), where two rows on each SM are 155 MB and the second pass leaves L2.
// The loss alone: 128 threads, no prefetch, 199 us (256 threads: 249).
template <typename T, int NT, bool kGrad>
__global__ void __launch_bounds__(NT, 1024 / NT) topk_distill_kernel(const dwarf_topk_distill_args a, int cluster) {
  const int rank = cluster > 1 ? (int)cluster_rank() : 0;
  distill_row<T, NT, kGrad, false>(a, cluster, rank, blockIdx.x / (unsigned)cluster);
}

// The gradient from the sums of an earlier launch: one read and one write (368 us at 16384
// rows of 32768 bf16, 5.8 TB/s). With skip_if_one a grid of one wave, which
// costs 3 us (a CTA for each of 16384 rows: 11 us) where there is nothing to do.
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT) topk_distill_grad_kernel(const dwarf_topk_distill_args a, int parts) {
  if (a.skip_if_one && *a.grad_rows == 1.0f) return;
  const uint32_t n = (uint32_t)(a.outer * a.inner) * (uint32_t)parts;
  for (uint32_t i = blockIdx.x; i < n; i += gridDim.x) {
    distill_row<T, NT, true, true>(a, parts, (int)(i % (uint32_t)parts), i / (uint32_t)parts);
    __syncthreads();  // before the next row's list takes this one's place
  }
}

// Sums in 64 bits, in an order that the launch fixes: the same bits every time.
__global__ void __launch_bounds__(1024) row_reduce_kernel(const dwarf_row_reduce_args a) {
  __shared__ double s_sum[32];
  __shared__ int s_count[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  double sum = 0.0;
  int count = 0;
  for (int64_t i = tid; i < a.rows; i += blockDim.x) {
    if (a.values != nullptr) sum += (double)a.values[i];
    if (a.mask != nullptr) count += a.mask[i] != 0;
  }
  sum = warp_sum(sum);
  count = __reduce_add_sync(0xffffffffu, count);
  if (lane == 0) s_sum[warp] = sum, s_count[warp] = count;
  __syncthreads();
  if (warp != 0) return;
  const bool some = lane < (int)blockDim.x / 32;
  sum = warp_sum(some ? s_sum[lane] : 0.0);
  count = __reduce_add_sync(0xffffffffu, some ? s_count[lane] : 0);
  if (lane != 0) return;
  double out = a.values != nullptr ? sum * (double)a.host_scale : 1.0;
  if (a.mask != nullptr) out /= (double)max(count, 1);
  *a.out = (float)out;
}

template <typename T>
int launch_distill(const dwarf_topk_distill_args& a, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner;
  const int vectors = ceil_div((int)a.vocab, Vec16<T>::kVec);
  // 32768 rows of 4096 bf16: 226 us with 128 threads, 137 with a warp; 16384 of 4096 fp32: 111, 129
  const bool warps = warp_rows(rows, vectors, a.grad == nullptr ? 2048 : 512);
  if (a.loss == nullptr) {
    const int parts = warps ? 1 : parts_for(rows, vectors), threads = warps ? 32 : 128;
    int64_t grid = rows * parts;
    if (a.skip_if_one && grid > kNumSMs * (1024 / threads)) grid = kNumSMs * (1024 / threads);
    return launch_rows(warps ? topk_distill_grad_kernel<T, 32> : topk_distill_grad_kernel<T, 128>, grid, 1, threads, 0,
                       stream, a, parts);
  }
  const int cluster = cluster_for(rows, vectors, 262144 / Vec16<T>::kVec);  // a bit for each place: at most 32 KB
  // a row that starts off a 16-byte boundary has one vector more
  const int part = ceil_div(vectors + 1, cluster);
  const int bytes = (part * Vec16<T>::kVec + 31) / 32 * 4;
  const auto go = [&](auto kernel, int threads) {
    return launch_rows(kernel, rows, cluster, threads, bytes, stream, a, cluster);
  };
  if (a.grad == nullptr) return warps ? go(topk_distill_kernel<T, 32, false>, 32) : go(topk_distill_kernel<T, 128, false>, 128);
  if (warps) return go(topk_distill_kernel<T, 32, true>, 32);
  if (part <= 2048) return go(topk_distill_kernel<T, 128, true>, 128);
  if (part <= 4097) return go(topk_distill_kernel<T, 256, true>, 256);
  return go(topk_distill_kernel<T, 512, true>, 512);
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
  if (a.loss == nullptr && (a.grad == nullptr || a.stats == nullptr)) return DWARF_ERR_NULL;
  if (!aligned16(a.stats)) return DWARF_ERR_ALIGN;
  if ((st = check_elements(a.grad, a.dtype)) != DWARF_OK) return st;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a.dtype == DWARF_F32) return launch_distill<float>(a, s);
  if (a.dtype == DWARF_BF16) return launch_distill<__nv_bfloat16>(a, s);
  return launch_distill<__half>(a, s);
}

extern "C" int dwarf_row_reduce(const dwarf_row_reduce_args* args, void* stream) {
  using namespace dwarf;
  DWARF_CHECK_VERSION(args);
  const dwarf_row_reduce_args a = *args;
  if (a.rows < 0 || a.rows >= (1ll << 28)) return DWARF_ERR_SHAPE;
  if (a.out == nullptr || (a.rows > 0 && a.values == nullptr && a.mask == nullptr)) return DWARF_ERR_NULL;
  row_reduce_kernel<<<1, a.rows <= 4096 ? 256 : 1024, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return launch_status();
}
