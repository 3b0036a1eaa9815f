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

constexpr int kCells = 4;           // cells that the vectors of a thread's tile fall into

// What a softmax needs of a part of a row: the maximum, S and T relative to it.
struct Sums {
  float m, s, t;
};

// One Sums from those of a warp's lanes (lanes without a part: m = -inf, s = t = 0), in a fixed order.
__device__ __forceinline__ Sums warp_join(Sums p, float c2) {
  const float m = warp_max(p.m);
  const float d = fmaxf((p.m - (m == -CUDART_INF_F ? 0.0f : m)) * c2, -200.0f);
  const float f = ex2_approx(d);
  return {m, warp_sum(p.s == 0.0f ? 0.0f : f * p.s), warp_sum(p.s == 0.0f ? 0.0f : f * fmaf(d, p.s, p.t))};
}

__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

// Sorts a warp's keys, the largest in lane 0: a bitonic network of 15 steps.
__device__ __forceinline__ uint64_t warp_sort(uint64_t key) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
    for (int o = size / 2; o >= 1; o /= 2) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, key, o);
      const bool larger = ((lane & size) == 0) == ((lane & o) == 0);  // this lane keeps the larger
      if ((other > key) == larger) key = other;
    }
  }
  return key;
}

// f(key, rank) for the n keys (all unlike; none is 0): runs of 32 are sorted by a warp each,
// a key's rank in the other runs is searched. (A rank by comparison with all n keys takes
// n^2 / 32 steps: 890 for the 177 candidates of 128 entries, against about 350.) Of the whole block.
template <int NT, typename F>
__device__ __forceinline__ void for_ranked(uint64_t* keys, int n, F f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int c = 32 * warp; c < n; c += NT) {
    const uint64_t key = warp_sort(c + lane < n ? keys[c + lane] : 0);
    keys[c + lane] = key;
  }
  __syncthreads();
  for (int c = 32 * warp; c < n; c += NT) {
    const uint64_t key = keys[c + lane];
    int above = lane;
    for (int o = 0; o < n; o += 32) {
      if (o == c) continue;
      int at = o;  // entries of the run from o on that are above the key
#pragma unroll
      for (int step = 16; step >= 1; step /= 2)
        if (keys[at + step - 1] > key) at += step;
      above += at - o + (keys[at] > key);
    }
    if (key != 0) f(key, above);
  }
}

// What a search may sort and look through: three times what K = 128 with 128 threads, or K = 32 with 32, comes to.
template <int NT>
struct TopShared {
  static constexpr int kGroups = 2 * NT, kCandidates = NT == 128 ? 512 : 192, kHits = kCandidates;
  uint4 value[kGroups / 8];          // the groups' maxima in 16 bits
  int hit[kHits];                    // cells that reach the bound
  alignas(16) uint64_t candidate[kCandidates];
  uint32_t bound;
  int n, hits;
  int scan[NT / 32];
};

// A bound that K entries of the part reach: the K-th largest of the maxima of G >= 2 K
// groups of entries (K <= G suffices). With entries in random places about G ln(G / (G - K))
// reach it. It is the smallest maximum that fewer than K exceed; each thread counts for
// its own, in packed 16-bit pairs (a search bit by bit in one warp has a third of the
// instructions, but its steps wait for one another: 3400 cycles against 1200 at K = 64).
template <int NT, typename N>
__device__ __forceinline__ void bound_of_groups(const N* value, int groups, int k, uint32_t* bound) {
  using V = Vec16<N>;
  for (int t = threadIdx.x; t < groups; t += NT) {
    const N g = value[t];
    const uint32_t zero = 0;
    typename V::Max c = *reinterpret_cast<const typename V::Max*>(&zero);
#pragma unroll 4
    for (int i = 0; i < groups; i += 8) c = V::above(*reinterpret_cast<const uint4*>(value + i), g, c);
    const uint32_t key = V::total(c) < k ? order_key(to_f32(g)) : 0xffffffffu;
    const uint32_t least = __reduce_min_sync(0xffffffffu, key);
    if ((threadIdx.x & 31) == 0 && least != 0xffffffffu) atomicMin(bound, least);
  }
}

// The K best entries of the part (order: value, then lowest id) among the first n
// candidates, n >= min(K, entries of the part). `cells` holds 16 bits, no lower than the
// largest entry, for each cell: every fourth of a thread's vectors of a tile. The cells
// that reach the bound are read again (from L2) and their entries that reach it become
// candidates. Where these are more than the buffers hold (ties, or many large values in
// one group), or a NaN is in the row, the K-th value is found bit by bit over the whole
// part and its ties are taken in order.
template <typename T, int NT>
__device__ __forceinline__ int best_entries(const Part<T, NT>& part, const typename Vec16<T>::Narrow* cells, int k,
                                            bool nan, float end, int end_id, TopShared<NT>& sh) {
  using N16 = Vec16<typename Vec16<T>::Narrow>;
  constexpr int kCandidates = TopShared<NT>::kCandidates, kHits = TopShared<NT>::kHits;
  const int tid = threadIdx.x;
  uint32_t limit = sh.bound;
  if (!nan) {
    const float bound = key_value(limit);
    const int n = ceil_div(part.size(), kVectors * NT) * kCells * NT;
    for (int first = 0; first < n; first += 8 * NT) {  // eight cells a thread
      const int c = first + 8 * tid;
      uint32_t m = c < n ? N16::reach(*reinterpret_cast<const uint4*>(cells + c), bound) : 0u;
      for (; m != 0; m &= m - 1) {
        const int at = atomicAdd(&sh.hits, 1);
        if (at < kHits) sh.hit[at] = c + N16::element(__ffs(m) - 1);
      }
    }
    if (end_id >= 0 && end >= bound) sh.candidate[atomicAdd(&sh.n, 1)] = entry_key(end, (uint32_t)end_id);
    __syncthreads();
    const int hits = sh.hits;
    if (hits <= kHits) {
      constexpr int kCell = kVectors / kCells, kBatch = 2;
      const int items = hits * kCell;
      for (int first = 0; first < items; first += kBatch * NT) {
        uint4 w[kBatch];
        int at_j[kBatch], found = 0;
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {  // the loads of a batch are in flight together
          const int h = first + q * NT + tid;
          at_j[q] = part.w1;
          if (h < items) {
            const int c = sh.hit[h / kCell];  // [tile][thread][cell]
            at_j[q] = part.w0 + (c / (kCells * NT) * kVectors + h % kCell * kCells + c % kCells) * NT +
                      c / kCells % NT;
          }
          if (at_j[q] < part.w1) w[q] = ld_stream(reinterpret_cast<const uint4*>(part.row.base) + at_j[q]);
        }
        uint32_t m[kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
          m[q] = at_j[q] < part.w1 ? Vec16<T>::reach(w[q], bound) : 0u;
          found += __popc(m[q]);
        }
        if (found == 0) continue;
        int at = atomicAdd(&sh.n, found);
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
          for (; m[q] != 0; m[q] &= m[q] - 1, ++at) {
            const int e = Vec16<T>::element(__ffs(m[q]) - 1);
            if (at < kCandidates)
              sh.candidate[at] = entry_key(Vec16<T>::value(w[q], e),
                                           (uint32_t)(at_j[q] * Vec16<T>::kVec + e - part.row.lead));
          }
        }
      }
      __syncthreads();
      if (sh.n <= kCandidates) return sh.n;
    }
    __syncthreads();
  }
  // entries of the part with a key of at least `from`
  auto count = [&](uint32_t from) {
    int c = 0;
    part.walk([&](const uint4& w, int j, bool in) {
      if (in) part.elements(w, j, [&](float x, int) { c += order_key(x) >= from; });
      return true;
    });
    c = __reduce_add_sync(0xffffffffu, c);
    __syncthreads();
    if ((tid & 31) == 0) sh.scan[tid >> 5] = c;
    __syncthreads();
    c = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) c += sh.scan[i];
    return c;
  };
  if (nan || count(limit + 1) >= k) {
    limit = 0;
    for (uint32_t bit = 0x80000000u; bit != 0; bit >>= 1)
      if (count(limit | bit) >= k) limit |= bit;
  }
  __syncthreads();
  if (tid == 0) sh.n = 0;
  __syncthreads();
  part.walk([&](const uint4& w, int j, bool in) {
    if (in)
      part.elements(w, j, [&](float x, int id) {
        if (order_key(x) > limit) sh.candidate[atomicAdd(&sh.n, 1)] = entry_key(x, (uint32_t)id);  // fewer than k
      });
    return true;
  });
  __syncthreads();
  int have = sh.n;
  part.walk([&](const uint4& w, int j, bool in) {
    if (have >= k) return false;
    int c = 0;
    if (in) part.elements(w, j, [&](float x, int) { c += order_key(x) == limit; });
    int at = c;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int up = __shfl_up_sync(0xffffffffu, at, o);
      if ((tid & 31) >= o) at += up;
    }
    if ((tid & 31) == 31) sh.scan[tid >> 5] = at;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
      if (i < (tid >> 5)) at += sh.scan[i];
      total += sh.scan[i];
    }
    at += have - c;
    if (in)
      part.elements(w, j, [&](float x, int id) {
        if (order_key(x) != limit) return;
        if (at < k) sh.candidate[at] = entry_key(x, (uint32_t)id);
        ++at;
      });
    have = min(k, have + total);
    __syncthreads();
    return true;
  });
  __syncthreads();
  return have;
}

// One CTA, or a cluster of them, for a row: one pass that keeps a running maximum, S
// and T for each warp, then (kTop) the search for the alternatives. Small CTAs overlap one's
// loads with another's sums and search: 16384 rows of 32768 bf16 take 162 us without
// alternatives (6.6 TB/s; 512 threads that hold a whole row in registers: 277), 183 with 5,
// 214 with 64, 294 with 128. With alternatives what bounds it is the latency of the search's
// steps, of which the reading of the cells under a full memory pipe is the longest (at 64: bound
// 1.2 k cycles, cells 0.8 k, reading them 4 k, ranking 2.5 k of 30 k for a row).
template <typename T, int NT, bool kTop, bool kAhead>
__global__ void __launch_bounds__(NT, NT == 32 ? 32 : kTop ? 9 : 8)
    token_logprobs_kernel(const dwarf_token_logprobs_args a, int cluster, int lists_at, int64_t ahead) {
  using V = Vec16<T>;
  constexpr int kWarps = NT / 32;
  extern __shared__ __align__(16) unsigned char s_dynamic[];
  typename V::Narrow* s_cells = reinterpret_cast<typename V::Narrow*>(s_dynamic);
  uint64_t* s_lists = reinterpret_cast<uint64_t*>(s_dynamic + lists_at);  // [cluster][k], in rank 0
  __shared__ Sums s_warp[kWarps];
  __shared__ float s_parts[kMaxCluster][3];
  __shared__ Sums s_row;
  __shared__ __align__(16) unsigned char s_top[kTop ? sizeof(TopShared<NT>) : 16];
  TopShared<NT>& top = *reinterpret_cast<TopShared<NT>*>(s_top);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = cluster > 1 ? (int)cluster_rank() : 0;
  const int64_t r = blockIdx.x / (unsigned)cluster;
  const T* x = static_cast<const T*>(a.logits) + row_offset(r, a.inner, a.so, a.si);
  const int vocab = (int)a.vocab, k = a.top_k;
  const float c2 = a.inv_temperature * kLog2e;
  if (cluster > 1) cluster_arrive();  // its CTAs have started, before one writes to another

  const Part<T, NT> part(x, vocab, rank, cluster);
  const int end_id = warp == 0 ? part.end_id(lane) : -1;
  const float end = end_id >= 0 ? to_f32(x[end_id]) : -CUDART_INF_F;
  Sums sum = {-CUDART_INF_F, 0.0f, 0.0f};
  typename V::Max top0 = V::none(), top1 = V::none();  // maxima of the thread's even and odd vectors
  for (int at = 0; at < part.size(); at += kVectors * NT) {
    uint4 v[kVectors];
    part.load(at, v);
    typename V::Max mv[kCells];
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      const typename V::Max of = V::max_of(v[i]);
      mv[i % kCells] = i < kCells ? of : V::join(mv[i % kCells], of);
    }
    if (kTop) {
      __align__(8) typename V::Narrow cell[kCells];
#pragma unroll
      for (int i = 0; i < kCells; ++i) cell[i] = V::narrow(mv[i]);
      reinterpret_cast<uint2*>(s_cells)[at / kVectors + tid] = *reinterpret_cast<const uint2*>(cell);
    }
    mv[0] = V::join(mv[0], mv[2]);
    mv[1] = V::join(mv[1], mv[3]);
    if (kTop) {
      top0 = V::join(top0, mv[0]);
      top1 = V::join(top1, mv[1]);
    }
    const float mx = V::largest(V::join(mv[0], mv[1]));
    const float m = fmaxf(sum.m, warp_max(mx));
    if (sum.m > -CUDART_INF_F) {  // a later tile: move the sums to the new maximum
      const float d = fmaxf((sum.m - m) * c2, -200.0f), f = ex2_approx(d);
      sum.t = f * fmaf(d, sum.s, sum.t);
      sum.s *= f;
    }
    sum.m = m;
    float2 s = make_float2(0.0f, 0.0f), t = s;
    // Entries 2^-200 below the maximum count as 0, masked ones among them (0 (-inf) is
    // not formed). Where the row's type has room for such a bound below the maximum
    // (2^-60 at least) and |c m| is below 2^20, the bound is set in packed pairs and
    // d = c x - c m takes one fused operation; what the rounding of c m leaves out (2^-5 at
    // most) is put back into the sums. Otherwise d = c (x - m) and the bound is set in fp32:
    // from |c m| = 2^31 on the part left out can pass an exponent's range (fp32 logits of 16 at
    // temperature 1e-8), and with it every sum of the row.
    const typename V::Low low = V::low_of(m - 200.0f / c2);
    const float cm = m * c2;
    if ((m - V::low_value(low)) * c2 >= 60.0f && V::low_value(low) > -1.0e38f && fabsf(cm) < 0x1p20f) {
      const float2 shift = make_float2(-cm, -cm), cc = make_float2(c2, c2);
      auto add = [&](const uint4& w) {
        float2 e[V::kVec / 2];
        V::unpack(V::clamp(w, low), e);
#pragma unroll
        for (int h = 0; h < V::kVec / 2; ++h) {
          const float2 d = fma2(e[h], cc, shift);
          const float2 p = make_float2(ex2_approx(d.x), ex2_approx(d.y));
          s = add2(s, p);
          t = fma2(p, d, t);
        }
      };
      if (at + kVectors * NT <= part.size()) {
#pragma unroll
        for (int i = 0; i < kVectors; ++i) add(v[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kVectors; ++i)
          if (at + i * NT < part.size()) add(v[i]);
      }
      const float left = fmaf(m, c2, -cm), f = ex2_approx(-left);
      const float s1 = s.x + s.y;
      sum.s += f * s1;
      sum.t += f * fmaf(-left, s1, t.x + t.y);
      continue;
    }
    const float shift = m == -CUDART_INF_F ? 0.0f : -m;
#pragma unroll
    for (int i = 0; i < kVectors; ++i) {
      if (at + i * NT >= part.size()) break;
      float2 e[V::kVec / 2];
      V::unpack(v[i], e);
#pragma unroll
      for (int h = 0; h < V::kVec / 2; ++h) {
        float2 d = mul2(add2(e[h], make_float2(shift, shift)), make_float2(c2, c2));
        const float2 p = make_float2(ex2_approx(d.x), ex2_approx(d.y));
        d = make_float2(fmaxf(d.x, -200.0f), fmaxf(d.y, -200.0f));
        s = add2(s, p);
        t = fma2(p, d, t);
      }
    }
    sum.s += s.x + s.y;
    sum.t += t.x + t.y;
  }
  if (warp == 0 && part.ends()) {
    const float m = fmaxf(sum.m, warp_max(end)), base = m == -CUDART_INF_F ? 0.0f : m;
    const float d0 = fmaxf((sum.m - base) * c2, -200.0f), f = ex2_approx(d0);
    const float d1 = (end - base) * c2, e = ex2_approx(d1);
    sum.t = f * fmaf(d0, sum.s, sum.t) + e * fmaxf(d1, -200.0f);
    sum.s = f * sum.s + e;
    sum.m = m;
  }
  // The next wave's row begins to arrive in L2 while this one's tail runs. In few waves the
  // tails leave memory idle (2047 rows of 32768 bf16, 5 alternatives: 37.0 us without, 34.9
  // with; 4096 of fp32: 94.6, 86.5); in many the CTAs have drifted apart, and only rows
  // without a search for alternatives still gain (16384 rows: 166 without, 162 with; with 64
  // alternatives: 217 without, 228 with).
  if (kAhead && tid == 0 && r + ahead < a.outer * a.inner)
    Part<T, NT>(static_cast<const T*>(a.logits) + row_offset(r + ahead, a.inner, a.so, a.si), vocab, 0, 1).prefetch_first(2048);
  sum.s = warp_sum(sum.s);
  sum.t = warp_sum(sum.t);
  if (lane == 0) s_warp[warp] = sum;
  int groups = 0;
  if (kTop) {
    typename V::Narrow* value = reinterpret_cast<typename V::Narrow*>(top.value);
    if (2 * k > NT) {
      value[tid] = V::narrow_down(top0);
      value[NT + tid] = V::narrow_down(top1);
      groups = 2 * NT;
    } else {
      top0 = V::join(top0, top1);
      int each = 32;  // groups of a warp
      for (; each * kWarps >= 2 * max(32, 2 * k); each /= 2)
        top0 = V::join(top0, __shfl_xor_sync(0xffffffffu, top0, each / 2));
      if (lane < each) value[warp * each + lane] = V::narrow_down(top0);
      groups = each * kWarps;
    }
    if (tid == 0) top.n = top.hits = 0, top.bound = 0xffffffffu;
  }
  __syncthreads();
  if (cluster > 1) cluster_wait();
  if (!kTop && warp != kWarps - 1 && cluster == 1) return;
  Sums all = {-CUDART_INF_F, 0.0f, 0.0f};  // in the last warp: of the part, then of the row
  if (warp == kWarps - 1) {
    if (lane < kWarps) all = s_warp[lane];
    all = warp_join(all, c2);
    if (cluster > 1 && lane < 3) {
      const uint32_t to = cluster_address(&s_parts[rank][lane], 0);
      st_cluster(to, lane == 0 ? all.m : lane == 1 ? all.s : all.t);
    }
  }
  int n = 0;
  if (kTop) {
    bound_of_groups<NT>(reinterpret_cast<const typename V::Narrow*>(top.value), groups, k, &top.bound);
    __syncthreads();
    // a NaN or +inf anywhere in the part makes some warp's sum NaN
    bool nan = false;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) nan |= s_warp[w].s != s_warp[w].s;
    n = best_entries(part, s_cells, k, nan, end, end_id, top);
  }
  if (cluster > 1) {
    if (kTop) {
      auto send = [&](uint64_t key, int at) {
        if (at < k) st_cluster(cluster_address(&s_lists[rank * k + at], 0), key);
      };
      for_ranked<NT>(top.candidate, n, send);
      for (int at = n + tid; at < k; at += NT) send(0, at);
    }
    cluster_arrive();
    if (rank != 0) return;
    cluster_wait();
    if (!kTop && warp != kWarps - 1) return;
  }
  if (warp == kWarps - 1) {
    if (cluster > 1) {
      all = {-CUDART_INF_F, 0.0f, 0.0f};
      if (lane < cluster) all = {s_parts[lane][0], s_parts[lane][1], s_parts[lane][2]};
      all = warp_join(all, c2);
    }
    if (all.m == -CUDART_INF_F) all.m = 0.0f;
    const float ln_s = log2f(all.s) * kLn2;  // -inf for a row without a finite logit
    if (lane == 0) {
      a.lse[r] = all.s == 0.0f ? -CUDART_INF_F : fmaf(all.m, a.inv_temperature, ln_s);
      a.entropy[r] = all.s == 0.0f ? 0.0f : ln_s - all.t / all.s * kLn2;
      if (a.stats != nullptr) reinterpret_cast<float2*>(a.stats)[r] = make_float2(all.m, all.s);
      if (a.logprob != nullptr) {
        const int64_t id = a.targets[r];
        float lp = 0.0f;
        if (id != a.ignore_index) {
          lp = CUDART_NAN_F;
          if (id >= 0 && id < vocab)
            lp = all.s == 0.0f ? -CUDART_INF_F : (to_f32(x[id]) - all.m) * a.inv_temperature - ln_s;
        }
        a.logprob[r] = lp;
      }
      s_row = {all.m, all.s, ln_s};
    }
  }
  if (!kTop) return;
  __syncthreads();
  const Sums fin = s_row;
  auto put = [&](uint64_t key, int at) {
    a.top_ids[r * k + at] = entry_id(key);
    a.top_logprobs[r * k + at] =
        fin.s == 0.0f ? -CUDART_INF_F : (key_value((uint32_t)(key >> 32)) - fin.m) * a.inv_temperature - fin.t;
  };
  if (cluster == 1) {
    for_ranked<NT>(top.candidate, n, [&](uint64_t key, int at) {
      if (at < k) put(key, at);
    });
  } else {
    for (int c = tid; c < cluster * k; c += NT) {
      const uint64_t key = s_lists[c];
      if (key == 0) continue;  // a part with fewer than k entries
      int at = c % k;
      for (int o = 0; o < cluster; ++o) {
        if (o == c / k) continue;
        int lo = 0, hi = k;  // entries of the other part's falling list that are above this one
        while (lo < hi) {
          const int mid = (lo + hi) / 2;
          if (s_lists[o * k + mid] > key) lo = mid + 1; else hi = mid;
        }
        at += lo;
      }
      if (at < k) put(key, at);
    }
  }
}

// Bytes of the cells of a part of `vectors` vectors.
constexpr int cell_bytes(int vectors, int threads) {
  return (vectors + kVectors * threads - 1) / (kVectors * threads) * kCells * threads * 2;
}
constexpr int kMostVectors = 65536;  // of a part (cells: 64 KB)

template <typename T, int NT>
int launch_forward(const dwarf_token_logprobs_args& a, int64_t rows, int vectors, int cluster, cudaStream_t stream) {
  const int64_t wave = cluster > 1 ? rows : (NT == 32 ? 32 : a.top_k > 0 ? 9 : 8) * kNumSMs;  // rows in flight
  if (a.top_k == 0) {
    const auto kernel = token_logprobs_kernel<T, NT, false, NT != 32>;
    return launch_rows(kernel, rows, cluster, NT, 0, stream, a, cluster, 0, wave);
  }
  // a row that starts off a 16-byte boundary has one vector more
  const int lists_at = cell_bytes(ceil_div(vectors + 1, cluster), NT);
  const int bytes = lists_at + (cluster > 1 ? cluster * a.top_k * 8 : 0);
  auto kernel = token_logprobs_kernel<T, NT, true, false>;
  if (NT != 32 && rows <= 4 * wave) kernel = token_logprobs_kernel<T, NT, true, NT != 32>;
  // The limit is the kernel's, for all host threads: always the most that a call can need, so that
  // a call with less cannot lower it before another one's launch.
  constexpr int kMostBytes = cell_bytes(kMostVectors + 1, NT) + kMaxCluster * DWARF_TOP_K_MAX * 8;
  if (bytes > 32 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostBytes) != cudaSuccess)
    return launch_status();
  return launch_rows(kernel, rows, cluster, NT, bytes, stream, a, cluster, lists_at, wave);
}

template <typename T>
int launch_forward(const dwarf_token_logprobs_args& a, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner;
  const int vectors = ceil_div((int)a.vocab, Vec16<T>::kVec);
  // (a warp's 64 groups bound up to 32 alternatives)
  if (a.top_k <= 32 && warp_rows(rows, vectors, 2048)) return launch_forward<T, 32>(a, rows, vectors, 1, stream);
  return launch_forward<T, 128>(a, rows, vectors, cluster_for(rows, vectors, kMostVectors), stream);
}

// grad_v = c (sparse terms - q_v (G + gH (log q_v + H))): each CTA writes its part of the
// row, then the listed entries of that part again with their terms. One read of the
// logits, one write; q from the forward's m and S. 16384 rows of 32768 bf16: 333 us, 6.4 TB/s:
// memory bounds it.
template <typename T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT)
    token_logprobs_bwd_kernel(const dwarf_token_logprobs_bwd_args a, int parts) {
  using V = Vec16<T>;
  __shared__ float sf[NT / 32];
  __shared__ int s_id[DWARF_TOP_K_MAX + 1];
  __shared__ float s_g[DWARF_TOP_K_MAX + 1];
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x / (unsigned)parts;
  const T* x = static_cast<const T*>(a.logits) + row_offset(r, a.inner, a.so, a.si);
  const int vocab = (int)a.vocab;
  const Part<T, NT> part(x, vocab, blockIdx.x % (unsigned)parts, parts);
  const RowStore<T> store(static_cast<T*>(a.grad) + r * a.vocab, part.row);
  const float c2 = a.inv_temperature * kLog2e;
  const float2 ms = reinterpret_cast<const float2*>(a.stats)[r];
  // entry 0: the target; entries 1..top_k: the alternatives
  float g_lp = a.g_logprob != nullptr ? a.g_logprob[r] : 0.0f;
  const int64_t target = a.targets != nullptr ? a.targets[r] : -1;
  if (a.targets == nullptr || target == a.ignore_index) g_lp = 0.0f;
  const bool off = g_lp != 0.0f && (target < 0 || target >= vocab);
  const int n = a.g_top != nullptr ? a.top_k + 1 : 1;
  float g = 0.0f;
  bool any = g_lp != 0.0f;
  for (int j = tid; j < n; j += NT) {
    const float v = j == 0 ? g_lp : a.g_top[r * a.top_k + j - 1];
    s_id[j] = j == 0 ? (g_lp != 0.0f && !off ? (int)target : -1) : (int)a.top_ids[r * a.top_k + j - 1];
    s_g[j] = v;
    g += v;
    any |= v != 0.0f;
  }
  g = n > 1 ? block_sum<NT>(g, sf) : g_lp;
  const float g_lse = a.g_lse != nullptr ? a.g_lse[r] : 0.0f;
  const float g_h = a.g_entropy != nullptr ? a.g_entropy[r] : 0.0f;
  any = __syncthreads_or(any) || g_lse != 0.0f || g_h != 0.0f;
  if (!any || ms.y == 0.0f) {
    store.zero(part);
    return;
  }
  const float weight = off ? CUDART_NAN_F : g - g_lse;
  const float log2s = log2f(ms.y), h2 = a.entropy[r] * kLog2e - log2s;
  // -q c (G + gH ln2 (d + h2)) = e (A + B d)
  const float scale = -a.inv_temperature / ms.y;
  const float k_b = scale * g_h * kLn2, k_a = fmaf(k_b, h2, scale * weight);
  const float2 shift = make_float2(-ms.x, -ms.x), cc = make_float2(c2, c2);
  auto dense = [&](float2 v) {
    float2 d = mul2(add2(v, shift), cc);
    const float2 e = make_float2(ex2_approx(d.x), ex2_approx(d.y));
    d = make_float2(fmaxf(d.x, -200.0f), fmaxf(d.y, -200.0f));
    return mul2(e, fma2(make_float2(k_b, k_b), d, make_float2(k_a, k_a)));
  };
  for (int at = 0; at < part.size(); at += kVectors * NT) {
    uint4 v[kVectors];
    part.load(at, v);
    store.tile(part, at, v, [&](const uint4& w) {
      float2 e[V::kVec / 2];
      V::unpack(w, e);
#pragma unroll
      for (int h = 0; h < V::kVec / 2; ++h) e[h] = dense(e[h]);
      return V::pack(e);
    });
  }
  const int end_id = tid < 32 ? part.end_id(tid) : -1;
  if (end_id >= 0) {
    const float v = to_f32(x[end_id]);
    store.out[end_id] = from_f32<T>(dense(make_float2(v, v)).x);
  }
  __syncthreads();  // the listed entries are written again, with their own terms
  for (int j = tid; j < n; j += NT) {
    const int id = s_id[j];
    if (id < 0 || id >= vocab || !part.holds(id)) continue;
    float sum = 0.0f;
    for (int l = 0; l < n; ++l)
      if (s_id[l] == id) sum += s_g[l];
    const float v = to_f32(x[id]);
    store.out[id] = from_f32<T>(fmaf(a.inv_temperature, sum, dense(make_float2(v, v)).x));
  }
}

template <typename T>
int launch_backward(const dwarf_token_logprobs_bwd_args& a, cudaStream_t stream) {
  const int64_t rows = a.outer * a.inner;
  const int vectors = ceil_div((int)a.vocab, Vec16<T>::kVec);
  if (warp_rows(rows, vectors, 512))  // 32768 rows of 4096 bf16: 112 us with 128 threads, 90 with a warp; of 8192: 172, 176
    return launch_rows(token_logprobs_bwd_kernel<T, 32>, rows, 1, 32, 0, stream, a, 1);
  const int parts = parts_for(rows, vectors);
  return launch_rows(token_logprobs_bwd_kernel<T, 128>, rows * parts, 1, 128, 0, stream, a, parts);
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
  if (reinterpret_cast<uintptr_t>(a.stats) & 7) return DWARF_ERR_ALIGN;
  if ((a.targets == nullptr) != (a.logprob == nullptr)) return DWARF_ERR_NULL;
  if (a.top_k > 0 && (a.top_logprobs == nullptr || a.top_ids == nullptr)) return DWARF_ERR_NULL;
  return with_type(a.dtype, [&](auto t) { return launch_forward<decltype(t)>(a, static_cast<cudaStream_t>(stream)); });
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
  if ((st = check_elements(a.grad, a.dtype)) != DWARF_OK) return st;
  if (reinterpret_cast<uintptr_t>(a.stats) & 7) return DWARF_ERR_ALIGN;
  if (a.g_logprob != nullptr && a.targets == nullptr) return DWARF_ERR_NULL;
  if (a.g_top != nullptr && (a.top_ids == nullptr || a.top_k < 1)) return DWARF_ERR_NULL;
  return with_type(a.dtype, [&](auto t) { return launch_backward<decltype(t)>(a, static_cast<cudaStream_t>(stream)); });
}
