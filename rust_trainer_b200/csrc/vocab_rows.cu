// Softmax and distillation over rows of logits: a cluster of CTAs a row, which holds the row in shared memory, so that it is read once.
#include "vocab_rows.cuh"

namespace rt {

// What a warp knows of its share of a row, and sends to every CTA of the cluster.
struct SoftmaxStat {
  double s;
  float m, unused;
};

template <class T, class O>
__global__ void __launch_bounds__(VR_THREADS, 3) softmax_rows_kernel(const T* z, size_t ld, int vocab, ExpT ex, O* prob, size_t prob_ld) {
  extern __shared__ uint4 slots[];
  __shared__ SoftmaxStat stat[VR_MAX_CLUSTER * VR_WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  cluster_arrive_relaxed();
  const size_t r = cluster_id();
  const RowPart<T> part(z + r * ld, vocab, slots);
  part.load();
  MaxSum ms;
  for (int s = 0; s < part.n_steps; ++s) {
    float x[16];
    part.wait(s);
    part.get(s, x);
    ms.take(x, ex);
  }
  float m;
  double sum = warp_join(ms.m, ms.s, ex, &m);
  cluster_wait();  // the other CTAs run: their shared memory may be written
  if (lane < part.size) {
    const uint32_t to = mapa_u32(smem_u32(&stat[part.rank * VR_WARPS + warp]), lane);
    st_cluster(to, sum);
    st_cluster(to + 8, __float_as_uint(m), 0u);
  }
  cluster_arrive();
  cluster_wait();
  const int n = part.size * VR_WARPS;
  const SoftmaxStat none{0.0, -INFINITY, 0.0f}, a = lane < n ? stat[lane] : none, b = lane + 32 < n ? stat[lane + 32] : none;
  const float ab = max_nan(a.m, b.m);
  sum = ab > -INFINITY ? a.s * (double)ex(a.m - ab) + b.s * (double)ex(b.m - ab) : 0.0;
  sum = warp_join(ab, sum, ex, &m);
  // a row of -inf has no probabilities, one with a NaN or +inf no number for them
  const float inv = m == -INFINITY ? 0.0f : m < INFINITY ? (float)(1.0 / sum) : NAN, ref = m == -INFINITY ? 0.0f : m;
  O* out = prob + r * prob_ld;
  const bool aligned = vectors_aligned<O, RowPart<T>::VEC>(out, part.phase);
  for (int s = 0; s < part.n_steps; ++s) {
    float x[16];
    part.get(s, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = ex(x[i] - ref) * inv;
#pragma unroll
    for (int j = 0; j < RowPart<T>::STEP; ++j) {
      const int it = s * RowPart<T>::STEP + j;
      if (it < part.n_it) put_vector<O, RowPart<T>::VEC>(out, part.column(it, threadIdx.x), vocab, aligned, x + j * RowPart<T>::VEC);
    }
  }
}

// As above, of the elements outside of the teacher's list (m, s) and of those on it (mi, si).
struct DistillStat {
  double s, si;
  float m, mi;
};
// What the row's sums say to every thread: a gradient outside of the list is exp(z - ref) co, one on it (exp(z - m) inv - q) g.
struct DistillRow {
  double inv;
  float m, ref, co;
  int bad;
};

template <class T, class O>
__global__ void __launch_bounds__(VR_THREADS, 3) distill_rows_kernel(const T* z, size_t ld, int vocab, float t, ExpT ex, const int* index, const float* teacher,
                                                                     int k, int tail, const float* weight, float* loss, O* d, size_t d_ld,
                                                                     float* row_scale, int* status) {
  constexpr int VEC = RowPart<T>::VEC, STEP = RowPart<T>::STEP;
  extern __shared__ uint4 slots[];
  __shared__ DistillStat stat[VR_MAX_CLUSTER * VR_WARPS];
  __shared__ double s_mass[VR_WARPS], s_loss[VR_WARPS][3], s_q[RT_TOP_MAX];
  __shared__ int s_index[RT_TOP_MAX];
  __shared__ DistillRow s_row;
  static_assert(RT_TOP_MAX <= VR_THREADS);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster_arrive_relaxed();
  const size_t r = cluster_id();
  const T* row = z + r * ld;
  const RowPart<T> part(row, vocab, slots);
  part.load();
  // a bit for each element that is on the list, a byte a vector
  uint32_t* marks = (uint32_t*)(slots + part.n_it * VR_THREADS);
  for (int i = tid; i < part.n_it * VR_THREADS / 4; i += VR_THREADS) marks[i] = 0;
  const float w = weight ? weight[r] : 1.0f, factor = w / t, g = row_scale ? 1.0f : factor;
  int at = -1, slot = 0, elem = 0;
  bool mine = false;
  double lt = -INFINITY;
  float z_at = -INFINITY;
  if (tid < k) {
    at = index[r * k + tid];
    if (at < -1 || at >= vocab) {
      if (part.rank == 0) report_status(status, RT_ERR_BAD_INDEX);
      at = -1;
    }
    if (at >= 0) {
      lt = teacher[r * k + tid];
      mine = part.owner(at, &slot, &elem) == part.rank;
      if (mine || part.rank == 0) z_at = to_f32(row[at]);
    }
    s_index[tid] = at;
  }
  double q = tid < k ? exp(lt) : 0.0;  // 64 bits for what is left of the mass, a difference, and for the loss
  double mass = warp_sum_f64(q);
  if (lane == 0) s_mass[warp] = mass;
  __syncthreads();
  mass = 0.0;
#pragma unroll
  for (int i = 0; i < VR_WARPS; ++i) mass += s_mass[i];
  const double rest = tail ? fmax(0.0, 1.0 - mass) : 0.0;
  if (!tail && mass > 0.0 && tid < k) {
    q /= mass;
    lt -= log(mass);
  }
  if (tid < k) s_q[tid] = q;
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
    const float zero[VEC] = {};
    cp_async_wait<0>();
    cluster_wait();
    if (out)
      for (int it = 0; it < part.n_it; ++it) put_vector<O, VEC>(out, part.column(it, tid), vocab, aligned, zero);
    return;
  }
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
  DistillStat st{0.0, 0.0, -INFINITY, -INFINITY};
  st.s = warp_join(ms.m, ms.s, ex, &st.m);
  if (__any_sync(0xffffffffu, first)) {  // few elements with most of the mass: 64 bits
    st.mi = warp_max_nan(first ? z_at : -INFINITY);
    st.si = warp_sum_f64(first && z_at > -INFINITY ? exp(((double)z_at - st.mi) / t) : 0.0);
  }
  if (part.rank == 0 && loss) {
    // sum q (t_j - z_j / T), the z relative to the warp's largest: all of them may be far from 0
    const bool on = q > 0.0;
    const float top = warp_max_nan(on ? z_at : -INFINITY);
    const double x = on ? (z_at == top ? 0.0 : ((double)z_at - top) / t) : 0.0;
    const double a = warp_sum_f64(on ? q * (lt - x) : 0.0), b = warp_sum_f64(q);
    if (lane == 0) s_loss[warp][0] = a, s_loss[warp][1] = b, s_loss[warp][2] = top;
  }
  cluster_wait();  // the other CTAs run: their shared memory may be written
  if (lane < part.size) {
    const uint32_t to = mapa_u32(smem_u32(&stat[part.rank * VR_WARPS + warp]), lane);
    st_cluster(to, st.s);
    st_cluster(to + 8, st.si);
    st_cluster(to + 16, __float_as_uint(st.m), __float_as_uint(st.mi));
  }
  cluster_arrive();
  cluster_wait();
  if (warp == 0) {
    const int n = part.size * VR_WARPS;
    const DistillStat none{0.0, 0.0, -INFINITY, -INFINITY}, a = lane < n ? stat[lane] : none, b = lane + 32 < n ? stat[lane + 32] : none;
    float mo;
    const float ab = max_nan(a.m, b.m), mi = warp_max_nan(max_nan(a.mi, b.mi));
    double so = ab > -INFINITY ? a.s * (double)ex(a.m - ab) + b.s * (double)ex(b.m - ab) : 0.0;
    so = warp_join(ab, so, ex, &mo);
    const double si = warp_sum_f64((a.si > 0.0 ? a.si * exp(((double)a.mi - mi) / t) : 0.0) + (b.si > 0.0 ? b.si * exp(((double)b.mi - mi) / t) : 0.0));
    const float m = max_nan(mo, mi);
    const double out_down = ((double)mo - m) / t, down = mo > -INFINITY ? exp(out_down) : 0.0;
    const double sum = so * down + (mi > -INFINITY ? si * exp(((double)mi - m) / t) : 0.0);
    const bool bad = !(m < INFINITY);
    if (lane == 0) {
      s_row.inv = sum > 0.0 ? 1.0 / sum : 0.0;
      s_row.m = m;
      s_row.ref = mo > -INFINITY ? mo : 0.0f;
      s_row.co = bad ? NAN : so > 0.0 ? (float)(down / sum - rest / so) * g : 0.0f;
      s_row.bad = bad;
      if (loss && part.rank == 0) {
        const double log_sum = log(sum);
        double l = 0.0;
        for (int i = 0; i < VR_WARPS; ++i) {
          const double top = s_loss[i][2], of = s_loss[i][1];
          if (of != 0.0) l += top > -INFINITY ? s_loss[i][0] + of * (log_sum - (top - m) / t) : INFINITY;
        }
        if (rest > 0.0) l += rest * (log(rest) - (so > 0.0 ? out_down + log(so) - log_sum : -INFINITY));
        loss[r] = bad ? NAN : (float)(w * l);
      }
    }
  }
  if (!out) return;
  __syncthreads();
  const float ref = s_row.ref, co = s_row.co;
  for (int s = 0; s < part.n_steps; ++s) {
    float x[16];
    part.get(s, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = ex(x[i] - ref) * co;
#pragma unroll
    for (int j = 0; j < STEP; ++j) {
      const int it = s * STEP + j;
      if (it < part.n_it) put_vector<O, VEC>(out, part.column(it, tid), vocab, aligned, x + j * VEC);
    }
  }
  __syncthreads();  // what is on the list overwrites what its vector's thread wrote
  if (first) out[at] = from_f32<O>(s_row.bad ? NAN : (float)((z_at > -INFINITY ? (double)ex(z_at - s_row.m) : 0.0) * s_row.inv - q_all) * g);
}

int launch_softmax_rows(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, void* prob, int prob_dtype, size_t prob_ld) {
  const RowShape shape = row_shape(vocab, z.dtype);
  return with_dtype(z.dtype, [&](auto* zt) {
    return with_dtype(prob_dtype, [&](auto* ot) {
      using T = std::remove_pointer_t<decltype(zt)>;
      using O = std::remove_pointer_t<decltype(ot)>;
      return launch_clusters(c, softmax_rows_kernel<T, O>, rows, shape.cluster, shape.slots * 16, (const T*)z.p, z.ld, vocab, exp_t(temperature),
                             (O*)prob, prob_ld);
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
