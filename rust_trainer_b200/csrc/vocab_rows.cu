// Softmax and distillation over rows of logits: a cluster of CTAs a row, each element read once.
#include "vocab_rows.cuh"

namespace rt {

// What a warp knows of its share of a row, and sends to every CTA of the cluster: a reference, and the sum of exponentials relative to it.
struct alignas(8) SoftmaxStat {
  float m, s;
};

template <class T, class O, int NT>
__global__ void __launch_bounds__(NT + 32, ctas_of(NT))
softmax_rows_kernel(const T* z, size_t ld, size_t rows, int vocab, ExpT ex, O* prob, size_t prob_ld, int places, int* status) {
  constexpr int WARPS = NT / 32;
  extern __shared__ uint4 slots[];
  __shared__ uint64_t bars[2 * VR_MAX_BLOCKS + 2];
  __shared__ SoftmaxStat stats[2][VR_MAX_CLUSTER * WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Exchange exchange;
  Ring<T, NT> ring(slots, bars, places, status, z, ld, rows, vocab, exchange);
  if (tid >= NT) {
    if (tid == NT) ring.copy_rows();
    return;
  }
  const int warps = ring.size * WARPS;
  for (size_t r = cluster_id(); r < rows; r += ring.row_step) {
    const RowPart<T, NT> part = ring.part(r);
    ring.wait_all(part);
    work_sync<NT>();
    float mine, m;
    const float sum = ring.template exponentials<sizeof(T) == 4>(part, ex, &mine), warp_sum = warp_join(mine, sum, ex, &m);
    fence_proxy_async_smem();  // what was written in the blocks comes before the copies that follow
    SoftmaxStat* stat = stats[exchange.turn()];
    if (tid == 0) exchange.expect(warps * sizeof(SoftmaxStat));
    if (lane < ring.size)
      send(mapa_u32(smem_u32(&stat[ring.rank * WARPS + warp]), lane), exchange.bar(lane), __float_as_uint(m), __float_as_uint(warp_sum));
    exchange.wait();
    const float row_sum = (float)warp_sum_f64(lane_join(warps, [&](int i, float* mi, float* si) { *mi = stat[i].m, *si = stat[i].s; }, ex, &m));
    // a row of -inf has no probabilities, one with a NaN or +inf no number for them
    ring.put_exponentials(part, prob + r * prob_ld, mine, m, m == -INFINITY ? 0.0f : m < INFINITY ? 1.0f / row_sum : NAN, ex);
    ring.advance(part.n_it, true);
  }
}

// As above, of the elements outside of the teacher's list (m, s); the sum of those on it, relative to the largest logit listed; and the
// teacher's mass on it.
struct alignas(16) DistillStat {
  double listed, mass;
  float m, s;
  static constexpr int SENT = 24;
};
static_assert(sizeof(DistillStat) == 32, "sent as 16 and 8 bytes, which have to be aligned");

// An element on the list leaves the row, whose sums and results are then those outside of the list: -inf in its place.  Returns whether
// another entry may have taken it before.
template <class T>
__device__ __forceinline__ bool take_out(uint4* slots, int element) {
  if constexpr (sizeof(T) == 4) {
    return atomicExch((uint32_t*)slots + element, 0xff800000u) == 0xff800000u;
  } else {
    constexpr uint32_t none = std::is_same<T, __half>::value ? 0xfc00 : 0xff80;
    uint32_t* word = (uint32_t*)slots + element / 2;
    const int shift = (element & 1) * 16;
    const uint32_t old = atomicOr(word, 0xffffu << shift) >> shift & 0xffff;  // all ones between the two operations
    atomicAnd(word, ~((0xffff ^ none) << shift));
    return old == 0xffff || old == none;
  }
}


// What 64 bits cost here is latency, of exp, log and division some 1000 cycles each: the two exponentials of an entry stand side by side,
// logarithms and divisions wait for the loss, which a warp finds while the others go on with the next row.
template <class T, class O, int NT>
__global__ void __launch_bounds__(NT + 32, ctas_of(NT))
distill_rows_kernel(const T* z, size_t ld, size_t rows, int vocab, float t, ExpT ex, const int* index, const float* teacher, int k, int tail,
                    const float* weight, float* loss, O* d, size_t d_ld, float* row_scale, int places, int* status) {
  constexpr int WARPS = NT / 32, LIST_WARPS = RT_TOP_MAX / 32;
  extern __shared__ uint4 slots[];
  __shared__ uint64_t bars[2 * VR_MAX_BLOCKS + 2];
  __shared__ DistillStat stats[2][VR_MAX_CLUSTER * WARPS];
  __shared__ double s_cross[2][LIST_WARPS], s_q[RT_TOP_MAX];
  __shared__ float s_top[LIST_WARPS];
  __shared__ int s_index[RT_TOP_MAX];
  static_assert(RT_TOP_MAX <= NT);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, list_warps = (k + 31) / 32;
  Exchange exchange;
  Ring<T, NT> ring(slots, bars, places, status, z, ld, rows, vocab, exchange);
  if (tid >= NT) {
    if (tid == NT) ring.copy_rows();
    return;
  }
  const double inv_t = 1.0 / t;
  const bool with_entries = warp < list_warps;
  const int warps = ring.size * WARPS;
  // The thread's entry of the list: its index (-1: none), the teacher's log-probability, the student's logit.
  auto entry = [&](size_t r, float* tl) {
    *tl = tid < k ? teacher[r * k + tid] : 0.0f;
    return tid < k ? index[r * k + tid] : -1;
  };
  auto logit = [&](size_t r, int* i) {
    if (*i < -1 || *i >= vocab) {
      if (ring.rank == 0) report_status(status, RT_ERR_BAD_INDEX);
      *i = -1;
    }
    return *i >= 0 ? to_f32(z[r * ld + *i]) : -INFINITY;
  };
  size_t r = cluster_id();
  float w = weight ? weight[r] : 1.0f, tl;
  int my = entry(r, &tl);
  float z_my = logit(r, &my);
  for (size_t next_r; r < rows; r = next_r) {
    next_r = r + ring.row_step;
    const bool more = next_r < rows;
    const RowPart<T, NT> part = ring.part(r);
    const float factor = w / t, g = row_scale ? 1.0f : factor;
    O* out = d ? d + r * d_ld : nullptr;
    if (row_scale && tid == 0 && ring.rank == 0) row_scale[r] = factor;
    float next_tl = 0.0f, next_w = 1.0f, next_z = -INFINITY;
    int next_my = -1;
    if (more) {
      next_my = entry(next_r, &next_tl);
      if (weight) next_w = weight[next_r];
    }
    auto no_gradient = [&] {
      if (out)
        ring.put(part, out, [](const uint4&, float* x) {
#pragma unroll
          for (int i = 0; i < RowPart<T, NT>::VEC; ++i) x[i] = 0.0f;
        });
      else
        ring.release_all(part);
      if (loss && tid == 0 && ring.rank == 0) loss[r] = 0.0f;
    };
    // the list leaves the row
    int it_my = 0, element = 0;
    bool first = my >= 0 && part.owner(my, &it_my, &element) == ring.rank, again = false;
    if (with_entries) {
      const float warp_top = warp_max_nan(z_my);
      if (lane == 0) s_top[warp] = warp_top;
      if (tid < k) s_index[tid] = my;
    }
    ring.wait_all(part);
    work_sync<NT>();
    float top = -INFINITY;  // the largest logit listed
    for (int i = 0; i < list_warps; ++i) top = max_nan(top, s_top[i]);
    if (first) again = take_out<T>(ring.block(it_my), element);
    again = work_sync_or<NT>(again);
    if (w == 0.0f) {  // nothing to learn from, whatever the logits are
      fence_proxy_async_smem();
      work_sync<NT>();
      no_gradient();
      if (more) next_z = logit(next_r, &next_my);
    } else {
      DistillStat st{0.0, 0.0, -INFINITY, 0.0f};
      double q = 0.0, e_my = 0.0;  // 64 bits for what is left of the mass, a difference, and for the loss
      double q_all = 0.0;
      if (with_entries) {
        const double x_my = z_my > -INFINITY ? (z_my == top ? 0.0 : ((double)z_my - top) * inv_t) : -INFINITY, lt = tl;
        if (my >= 0) q = exp(lt), e_my = exp(x_my);
        q_all = q;
        if (again && tid < k) s_q[tid] = q;
        double cross = q > 0.0 ? q * (lt - x_my) : 0.0;  // sum q (t_j - z_j / T), the z relative to the largest
        st.mass = q;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) st.mass += __shfl_xor_sync(0xffffffffu, st.mass, o), cross += __shfl_xor_sync(0xffffffffu, cross, o);
        if (lane == 0) s_cross[exchange.turn()][warp] = cross;
      }
      if (again) {  // an index came twice: its first entry answers for all of them
        work_sync<NT>();
        if (first) {
          q_all = 0.0;
          for (int j = 0; j < k; ++j)
            if (s_index[j] == my) {
              if (j < tid) first = false;
              q_all += s_q[j];
            }
        }
      }
      if (with_entries) st.listed = warp_sum_f64(first ? e_my : 0.0);
      float mine;
      const float sum = out ? ring.template exponentials<sizeof(T) == 4>(part, ex, &mine) : ring.template exponentials<false>(part, ex, &mine);
      st.s = warp_join(mine, sum, ex, &st.m);
      fence_proxy_async_smem();  // what was written in the blocks comes before the copies that follow
      DistillStat* stat = stats[exchange.turn()];
      const double* all_cross = s_cross[exchange.turn()];
      if (tid == 0) exchange.expect(warps * DistillStat::SENT);
      if (lane < ring.size) {
        const uint32_t to = mapa_u32(smem_u32(&stat[ring.rank * WARPS + warp]), lane), bar = exchange.bar(lane);
        const uint2 a = *(const uint2*)&st.listed, b = *(const uint2*)&st.mass;
        send(to, bar, a.x, a.y, b.x, b.y);
        send(to + 16, bar, __float_as_uint(st.m), __float_as_uint(st.s));
      }
      exchange.wait();
      if (more) next_z = logit(next_r, &next_my);
      double mass = 0.0;  // every CTA has found the same
      for (int i = 0; i < list_warps; ++i) mass += stat[i].mass;
      const bool idle = !tail && mass == 0.0;
      const double rest = tail ? fmax(0.0, 1.0 - mass) : 0.0;
      // the sums of what is outside, relative to mo, and of what is listed, relative to top: in 32 bits for the gradients
      float mo, listed = 0.0f;
      const double lane_so = lane_join(warps, [&](int i, float* mi, float* si) { *mi = stat[i].m, *si = stat[i].s, listed += (float)stat[i].listed; }, ex, &mo);
      const float m = max_nan(mo, top);
      const bool bad = !(m < INFINITY);
      if (idle) {
        no_gradient();
      } else if (out) {
        float so = (float)lane_so;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) so += __shfl_xor_sync(0xffffffffu, so, o), listed += __shfl_xor_sync(0xffffffffu, listed, o);
        // a gradient outside of the list is exp(z - mo) co, one on it e to - q by, e relative to the largest listed
        const float rest_to = mo > -INFINITY ? ex(mo - m) : 0.0f, top_to = top > -INFINITY ? ex(top - m) : 0.0f;
        const float inv = 1.0f / (so * rest_to + listed * top_to);
        const float co = bad ? NAN : so > 0.0f ? (rest_to * inv - (float)rest / so) * g : 0.0f;
        const float to = bad ? NAN : m > -INFINITY ? top_to * inv * g : 0.0f, by = tail ? g : g / (float)mass;
        ring.put_exponentials(part, out, mine, mo, co, ex);
        work_sync<NT>();  // what is on the list overwrites what its vector's thread wrote
        if (first) out[my] = from_f32<O>((float)(e_my * to - q_all * by));
      }
      if (!out && !idle) ring.release_all(part);
      if (loss && !idle && ring.rank == 0 && warp == WARPS - 1) {
        double so = lane_so, listed64 = 0.0, cross = lane < list_warps ? all_cross[lane] : 0.0;
        for (int i = lane; i < warps; i += 32) listed64 += stat[i].listed;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          so += __shfl_xor_sync(0xffffffffu, so, o);
          listed64 += __shfl_xor_sync(0xffffffffu, listed64, o);
          cross += __shfl_xor_sync(0xffffffffu, cross, o);
        }
        // log(listed + outside), the first relative to `top`, the second to mo, log(outside), log(rest) and log(mass): side by side
        const double x = ((double)mo - top) * inv_t;  // of the outside, in units of `top`
        const bool above = !(x <= 0.0) && mo > -INFINITY;
        const double shrink = above ? (top > -INFINITY ? exp(-x) : 0.0) : (mo > -INFINITY ? exp(x) : 0.0);
        const double log_of = log(lane == 0 ? (above ? so + listed64 * shrink : listed64 + so * shrink) : lane == 1 ? so : lane == 2 ? rest : mass);
        const double log_sum = __shfl_sync(0xffffffffu, log_of, 0), log_so = __shfl_sync(0xffffffffu, log_of, 1), log_rest = __shfl_sync(0xffffffffu, log_of, 2),
                     log_mass = __shfl_sync(0xffffffffu, log_of, 3);
        if (lane == 0) {
          double l = mass == 0.0 ? 0.0 : top > -INFINITY ? cross + mass * (log_sum + (above ? x : 0.0)) : INFINITY;
          if (!tail) l = l / mass - log_mass;
          if (rest > 0.0) l += so > 0.0 ? rest * (log_rest - log_so + log_sum - (above ? 0.0 : x)) : INFINITY;
          loss[r] = bad ? NAN : (float)(w * l);
        }
      }
    }
    ring.advance(part.n_it, true);
    w = next_w;
    my = next_my;
    tl = next_tl;
    z_my = next_z;
  }
}

int launch_softmax_rows(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, void* prob, int prob_dtype, size_t prob_ld) {
  const RowShape shape = row_shape(c, rows, vocab, z.dtype, 0);
  return with_dtype(z.dtype, [&](auto* zt) {
    return with_dtype(prob_dtype, [&](auto* ot) {
      return with_threads(shape.threads, [&](auto threads) {
        using T = std::remove_pointer_t<decltype(zt)>;
        using O = std::remove_pointer_t<decltype(ot)>;
        return launch_clusters(c, softmax_rows_kernel<T, O, decltype(threads)::value>, true, rows, shape.threads + 32, shape.cluster, shape.smem, (const T*)z.p, z.ld,
                               rows, vocab, exp_t(temperature), (O*)prob, prob_ld, shape.places, c->status_dev);
      });
    });
  });
}

int launch_distill_rows(rt_ctx* c, const DistillArgs& a, size_t rows) {
  const RowShape shape = row_shape(c, rows, a.vocab, a.z.dtype, 0);
  return with_dtype(a.z.dtype, [&](auto* zt) {
    return with_dtype(a.d_dtype, [&](auto* ot) {
      return with_threads(shape.threads, [&](auto threads) {
        using T = std::remove_pointer_t<decltype(zt)>;
        using O = std::remove_pointer_t<decltype(ot)>;
        return launch_clusters(c, distill_rows_kernel<T, O, decltype(threads)::value>, true, rows, shape.threads + 32, shape.cluster, shape.smem, (const T*)a.z.p,
                               a.z.ld, rows, a.vocab, a.temperature, exp_t(a.temperature), a.index, a.teacher, a.k, a.mode == RT_DISTILL_TAIL, a.weight,
                               a.loss, (O*)a.d, a.d_ld, a.row_scale, shape.places, c->status_dev);
      });
    });
  });
}

}  // namespace rt
