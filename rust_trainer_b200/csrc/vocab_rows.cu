// Softmax and distillation over rows of logits: a cluster of CTAs a row, which holds the row in shared memory, so that it is read once.
#include "vocab_rows.cuh"

namespace rt {

// What a warp knows of its share of a row, and sends to every CTA of the cluster.
struct SoftmaxStat {
  float m, s;
};

template <class T, class O>
__global__ void __launch_bounds__(VR_THREADS, 3) softmax_rows_kernel(const T* z, size_t ld, int vocab, ExpT ex, O* prob, size_t prob_ld, int* status) {
  extern __shared__ uint4 slots[];
  __shared__ uint64_t bars[VR_MAX_STEPS];
  __shared__ SoftmaxStat stat[VR_MAX_CLUSTER * VR_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  cluster_arrive_relaxed();
  const size_t r = cluster_id();
  const RowPart<T> part(z + r * ld, vocab, slots, bars, status);
  part.load();
  __syncthreads();
  MaxSum ms;
  for (int s = 0; s < part.n_steps; ++s) {
    float x[16];
    part.wait(s);
    part.get(s, x);
    ms.take(x, ex);
  }
  float m;
  const float warp_sum = warp_join(ms, ex, &m);
  cluster_wait();  // the other CTAs run: their shared memory may be written
  if (lane < part.size)
    st_cluster(mapa_u32(smem_u32(&stat[part.rank * VR_WARPS + warp]), lane), __float_as_uint(m), __float_as_uint(warp_sum));
  cluster_arrive();
  cluster_wait();
  const int n = part.size * VR_WARPS;
  const SoftmaxStat none{-INFINITY, 0.0f}, a = lane < n ? stat[lane] : none, b = lane + 32 < n ? stat[lane + 32] : none;
  const float sum = (float)cluster_join(a.m, a.s, b.m, b.s, ex, &m);
  // a row of -inf has no probabilities, one with a NaN or +inf no number for them
  const float inv = m == -INFINITY ? 0.0f : m < INFINITY ? 1.0f / sum : NAN, ref = m == -INFINITY ? 0.0f : m;
  O* out = prob + r * prob_ld;
  const bool aligned = vectors_aligned<O, RowPart<T>::VEC>(out, part.phase);
  for (int s = 0; s < part.n_steps; ++s) {
    float x[16];
    part.get(s, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = ex(x[i] - ref) * inv;
    put_step<O>(part, s, out, aligned, x);
  }
}

// As above, of the elements outside of the teacher's list (m, s), and the sum of those on it, relative to the largest logit listed.
struct DistillStat {
  double listed;
  float m, s;
};
// What the row's sums say to every thread: a gradient outside of the list is exp(z - ref) co, one on it e listed_to - q g, where e is
// the element's exponential relative to the largest listed.
struct DistillRow {
  double rest_sum, listed_sum, listed_to;
  float ref, co, m;
};

// The bulk of what 64 bits cost here is the latency of exp, log and division (some 500 cycles each), so that they stand where the row is
// still on its way (the teacher's probabilities, the listed elements' exponentials) or, for the loss, beside the writing of the gradients.
template <class T, class O>
__global__ void __launch_bounds__(VR_THREADS, 3) distill_rows_kernel(const T* z, size_t ld, int vocab, float t, ExpT ex, const int* index, const float* teacher,
                                                                     int k, int tail, const float* weight, float* loss, O* d, size_t d_ld,
                                                                     float* row_scale, int* status) {
  constexpr int VEC = RowPart<T>::VEC, STEP = RowPart<T>::STEP;
  extern __shared__ uint4 slots[];
  __shared__ uint64_t bars[VR_MAX_STEPS];
  __shared__ DistillStat stat[VR_MAX_CLUSTER * VR_WARPS];
  __shared__ double s_mass[VR_WARPS], s_loss[VR_WARPS][2], s_q[RT_TOP_MAX];
  __shared__ float s_top[VR_WARPS];
  __shared__ int s_index[RT_TOP_MAX];
  __shared__ DistillRow s_row;
  static_assert(RT_TOP_MAX <= VR_THREADS);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster_arrive_relaxed();
  const size_t r = cluster_id();
  const T* row = z + r * ld;
  const RowPart<T> part(row, vocab, slots, bars, status);
  part.load();
  const float w = weight ? weight[r] : 1.0f, factor = w / t, g = row_scale ? 1.0f : factor;
  int at = -1, slot = 0, elem = 0;
  bool mine = false;
  double lt = -INFINITY, q = 0.0;  // 64 bits for what is left of the mass, a difference, and for the loss
  float z_at = -INFINITY;
  if (tid < k) {
    at = index[r * k + tid];
    if (at < -1 || at >= vocab) {
      if (part.rank == 0) report_status(status, RT_ERR_BAD_INDEX);
      at = -1;
    }
    if (at >= 0) {
      const float tl = teacher[r * k + tid];
      z_at = to_f32(row[at]);
      mine = part.owner(at, &slot, &elem) == part.rank;
      lt = tl;
      q = exp(lt);
    }
    s_index[tid] = at;
  }
  // a bit for each element that is on the list, a byte a vector
  uint32_t* marks = (uint32_t*)(slots + part.n_it * VR_THREADS);
  for (int i = tid; i < part.n_it * VR_THREADS / 4; i += VR_THREADS) marks[i] = 0;
  double mass = warp_sum_f64(q);
  const float warp_top = warp_max_nan(z_at);
  if (lane == 0) s_mass[warp] = mass, s_top[warp] = warp_top;
  __syncthreads();
  mass = 0.0;
  float top = -INFINITY;  // the largest logit listed
#pragma unroll
  for (int i = 0; i < VR_WARPS; ++i) mass += s_mass[i], top = max_nan(top, s_top[i]);
  const double rest = tail ? fmax(0.0, 1.0 - mass) : 0.0;
  if (!tail && mass > 0.0 && tid < k) {
    q /= mass;
    lt -= log(mass);
  }
  if (tid < k) s_q[tid] = q;
  const double x_at = z_at > -INFINITY ? (z_at == top ? 0.0 : ((double)z_at - top) / t) : -INFINITY, e_at = at >= 0 ? exp(x_at) : 0.0;
  bool again = false;
  if (mine) {
    const uint32_t bit = 1u << ((slot & 3) * 8 + elem);
    again = (atomicOr(&marks[slot >> 2], bit) & bit) != 0;
  }
  bool first = mine;
  double q_all = q;
  if (__syncthreads_or(again) && mine) {  // an index came twice: its first entry answers for all of them
    q_all = 0.0;
    for (int j = 0; j < k; ++j)
      if (s_index[j] == at) {
        if (j < tid) first = false;
        q_all += s_q[j];
      }
  }
  O* out = d ? d + r * d_ld : nullptr;
  const bool aligned = vectors_aligned<O, VEC>(out, part.phase);
  if (row_scale && tid == 0 && part.rank == 0) row_scale[r] = factor;
  if (w == 0.0f || (!tail && mass == 0.0)) {  // nothing to learn from, whatever the logits are
    if (loss && tid == 0 && part.rank == 0) loss[r] = 0.0f;
    const float zero[16] = {};
    for (int s = 0; s < part.n_steps; ++s) {
      part.wait(s);
      if (out) put_step<O>(part, s, out, aligned, zero);
    }
    cluster_wait();
    return;
  }
  if (part.rank == 0 && loss) {  // sum q (t_j - z_j / T), the z relative to the largest
    const double a = warp_sum_f64(q > 0.0 ? q * (lt - x_at) : 0.0), b = warp_sum_f64(q);
    if (lane == 0) s_loss[warp][0] = a, s_loss[warp][1] = b;
  }
  DistillStat st;
  st.listed = warp_sum_f64(first ? e_at : 0.0);
  MaxSum ms;
  for (int s = 0; s < part.n_steps; ++s) {
    float x[16];
    part.wait(s);
    part.get(s, x);
#pragma unroll
    for (int j = 0; j < STEP; ++j) {
      const int it = s * STEP + j;
      const uint32_t byte = it < part.n_it ? ((const uint8_t*)marks)[it * VR_THREADS + tid] : 0;
      if (byte) {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (byte >> i & 1) x[j * VEC + i] = -INFINITY;
      }
    }
    ms.take(x, ex);
  }
  st.s = warp_join(ms, ex, &st.m);
  cluster_wait();  // the other CTAs run: their shared memory may be written
  if (lane < part.size) {
    const uint32_t to = mapa_u32(smem_u32(&stat[part.rank * VR_WARPS + warp]), lane);
    st_cluster(to, st.listed);
    st_cluster(to + 8, __float_as_uint(st.m), __float_as_uint(st.s));
  }
  cluster_arrive();
  cluster_wait();
  if (warp == 0) {
    const int n = part.size * VR_WARPS;
    const DistillStat none{0.0, -INFINITY, 0.0f}, a = lane < n ? stat[lane] : none, b = lane + 32 < n ? stat[lane + 32] : none;
    const double listed = warp_sum_f64(a.listed + b.listed);
    float mo;
    const double so = cluster_join(a.m, a.s, b.m, b.s, ex, &mo);
    if (lane == 0) {
      const float m = max_nan(mo, top);
      const float rest_to = mo > -INFINITY ? ex(mo - m) : 0.0f, top_to = top > -INFINITY ? ex(top - m) : 0.0f;
      const float inv = 1.0f / (float)(so * rest_to + listed * top_to);
      const bool bad = !(m < INFINITY);
      s_row.rest_sum = so;
      s_row.listed_sum = listed;
      s_row.listed_to = bad ? NAN : m > -INFINITY ? (double)(top_to * inv * g) : 0.0;
      s_row.m = mo;
      s_row.ref = mo > -INFINITY ? mo : 0.0f;
      s_row.co = bad ? NAN : so > 0.0 ? (rest_to * inv - (float)rest / (float)so) * g : 0.0f;
    }
  }
  __syncthreads();
  if (out) {
    const float ref = s_row.ref, co = s_row.co;
    for (int s = 0; s < part.n_steps; ++s) {
      float x[16];
      part.get(s, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = ex(x[i] - ref) * co;
      put_step<O>(part, s, out, aligned, x);
    }
    __syncthreads();  // what is on the list overwrites what its vector's thread wrote
    if (first) out[at] = from_f32<O>((float)(e_at * s_row.listed_to - q_all * g));
  }
  if (loss && part.rank == 0 && warp == VR_WARPS - 1) {
    // log(listed + outside), the first relative to `top`, the second to mo, and log(outside); the two logarithms side by side
    const double x = ((double)s_row.m - top) / t, so = s_row.rest_sum, listed = s_row.listed_sum;  // of the outside, in units of `top`
    const bool outside_above = !(x <= 0.0) && s_row.m > -INFINITY;
    const double shrink = outside_above ? (top > -INFINITY ? exp(-x) : 0.0) : (s_row.m > -INFINITY ? exp(x) : 0.0);
    const double sum = outside_above ? so + listed * shrink : listed + so * shrink;
    const double log_of = log(lane == 0 ? sum : lane == 1 ? so : rest);
    const double log_sum = __shfl_sync(0xffffffffu, log_of, 0), log_so = __shfl_sync(0xffffffffu, log_of, 1), log_rest = __shfl_sync(0xffffffffu, log_of, 2);
    if (lane == 0) {
      const float m = max_nan(s_row.m, top);
      double a = 0.0, of = 0.0;
      for (int i = 0; i < VR_WARPS; ++i) a += s_loss[i][0], of += s_loss[i][1];
      // log-sum relative to `top` where anything is listed that can be, else relative to mo
      const double base = outside_above ? x : 0.0;
      double l = of == 0.0 ? 0.0 : top > -INFINITY ? a + of * (log_sum + base) : INFINITY;
      if (rest > 0.0) l += so > 0.0 ? rest * (log_rest - log_so + log_sum - (outside_above ? 0.0 : x)) : INFINITY;
      loss[r] = !(m < INFINITY) ? NAN : (float)(w * l);
    }
  }
}

int launch_softmax_rows(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, void* prob, int prob_dtype, size_t prob_ld) {
  const RowShape shape = row_shape(vocab, z.dtype);
  return with_dtype(z.dtype, [&](auto* zt) {
    return with_dtype(prob_dtype, [&](auto* ot) {
      using T = std::remove_pointer_t<decltype(zt)>;
      using O = std::remove_pointer_t<decltype(ot)>;
      return launch_clusters(c, softmax_rows_kernel<T, O>, rows, shape.cluster, shape.slots * 16, (const T*)z.p, z.ld, vocab, exp_t(temperature),
                             (O*)prob, prob_ld, c->status_dev);
    });
  });
}

int launch_distill_rows(rt_ctx* c, const DistillArgs& a, size_t rows) {
  const RowShape shape = row_shape(a.vocab, a.z.dtype);
  return with_dtype(a.z.dtype, [&](auto* zt) {
    return with_dtype(a.d_dtype, [&](auto* ot) {
      using T = std::remove_pointer_t<decltype(zt)>;
      using O = std::remove_pointer_t<decltype(ot)>;
      return launch_clusters(c, distill_rows_kernel<T, O>, rows, shape.cluster, shape.slots * 17, (const T*)a.z.p, a.z.ld, a.vocab, a.temperature,
                             exp_t(a.temperature), a.index, a.teacher, a.k, a.mode == RT_DISTILL_TAIL, a.weight, a.loss, (O*)a.d, a.d_ld, a.row_scale,
                             c->status_dev);
    });
  });
}

}  // namespace rt
