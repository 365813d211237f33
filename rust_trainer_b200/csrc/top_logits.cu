// The k largest logits of each row, in order, with their log-probabilities: a cluster of CTAs a row, which holds the row in shared
// memory.  Which elements can be among the k largest follows from the threads' maxima, which the pass over the exponentials
// finds anyway: if every one of W warps has j = ceil(k / W) threads with a maximum of at least x, then k elements are at least x.
// The elements from there up, a few times k of them, go to the cluster's first CTA, which ranks each by counting the larger ones.
// Only where they are too many (values that tie, masked rows) is a bound sought that leaves fewer, by bisection over values and
// indices.
#include "vocab_rows.cuh"

namespace rt {

constexpr int TOP_ROOM = 2048;  // candidates
static_assert(TOP_ROOM / VR_MAX_CLUSTER >= RT_TOP_MAX, "k elements of one CTA's share have to fit");
// An element as an integer, all different: its value's order above, the lower index in front.
constexpr int TOP_INDEX_BITS = 19;
static_assert(RT_VOCAB_MAX <= 1 << TOP_INDEX_BITS);
using TopKey = unsigned long long;
__device__ __forceinline__ TopKey top_key(float v, int c) {
  return ((TopKey)order32(v) << TOP_INDEX_BITS) | (uint32_t)((1 << TOP_INDEX_BITS) - 1 - c);
}

struct TopStat {
  double s;
  float m;
  uint32_t each, own;  // what every warp of the cluster, and every warp of this CTA, has to have for k elements
};

// the lanes' values in descending order
__device__ __forceinline__ uint32_t warp_sort(uint32_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
    for (int stride = size / 2; stride > 0; stride /= 2) {
      const uint32_t o = __shfl_xor_sync(0xffffffffu, v, stride);
      const bool keep_max = ((lane & stride) == 0) == ((lane & size) == 0 || size == 32);
      v = keep_max ? max(v, o) : min(v, o);
    }
  }
  return v;
}

template <class T>
__global__ void __launch_bounds__(VR_THREADS, 2) top_logits_kernel(const T* z, size_t ld, int vocab, float t, ExpT ex, int k, int* index, float* logp, float* lse) {
  constexpr int VEC = RowPart<T>::VEC, STEP = RowPart<T>::STEP;
  extern __shared__ uint4 slots[];
  __shared__ TopStat stat[VR_MAX_CLUSTER * VR_WARPS];
  __shared__ int s_n, s_count[2], counts[2][VR_MAX_CLUSTER];
  __shared__ double s_log_sum;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster_arrive_relaxed();
  const size_t r = cluster_id();
  const RowPart<T> part(z + r * ld, vocab, slots);
  part.load();
  TopKey* room = (TopKey*)(slots + part.n_it_most() * VR_THREADS);
  const int room_each = TOP_ROOM / part.size;
  if (tid == 0) s_n = s_count[0] = s_count[1] = 0;
  MaxSum ms;
  for (int s = 0; s < part.n_steps; ++s) {
    float x[16];
    part.wait(s);
    part.get(s, x);
    ms.take(x, ex);
  }
  const uint32_t my_top = order32(ms.m), sorted = warp_sort(my_top);
  const int warps = part.size * VR_WARPS;
  TopStat st;
  st.each = __shfl_sync(0xffffffffu, sorted, (k + warps - 1) / warps - 1);
  st.own = __shfl_sync(0xffffffffu, sorted, (k + VR_WARPS - 1) / VR_WARPS - 1);
  st.s = warp_join(ms.m, ms.s, ex, &st.m);
  cluster_wait();  // the other CTAs run: their shared memory may be written
  if (lane < part.size) {
    const uint32_t to = mapa_u32(smem_u32(&stat[part.rank * VR_WARPS + warp]), lane);
    st_cluster(to, st.s);
    st_cluster(to + 8, __float_as_uint(st.m), st.each);
    st_cluster(to + 16, (int)st.own);
  }
  cluster_arrive();
  cluster_wait();
  const TopStat none{0.0, -INFINITY, 0xffffffffu, 0xffffffffu}, a = lane < warps ? stat[lane] : none, b = lane + 32 < warps ? stat[lane + 32] : none;
  uint32_t own = a.own, own_b = b.own;  // eight neighbours are a CTA's warps
#pragma unroll
  for (int o = 1; o < VR_WARPS; o *= 2) {
    own = min(own, __shfl_xor_sync(0xffffffffu, own, o));
    own_b = min(own_b, __shfl_xor_sync(0xffffffffu, own_b, o));
  }
  const uint32_t own_max = __reduce_max_sync(0xffffffffu, max(lane < warps ? own : 0u, lane + 32 < warps ? own_b : 0u));
  const uint32_t bound = max(__reduce_min_sync(0xffffffffu, min(a.each, b.each)), own_max);
  float m;
  const float ab = max_nan(a.m, b.m);
  double sum = ab > -INFINITY ? a.s * (double)ex(a.m - ab) + b.s * (double)ex(b.m - ab) : 0.0;
  sum = warp_join(ab, sum, ex, &m);

  const uint32_t leader_room = mapa_u32(smem_u32(room), 0);
  auto push = [&](TopKey key) {
    const int p = atomicAdd(&s_n, 1);
    if (p < room_each) st_cluster(leader_room + (uint32_t)(part.rank * room_each + p) * 8, key);
  };
  // a warp takes the vectors of its threads that reach the bound one thread after the other, a vector a lane
  for (unsigned with = __ballot_sync(0xffffffffu, my_top >= bound); with; with &= with - 1) {
    const int owner = warp * 32 + __ffs(with) - 1;
    for (int it = lane; it < part.n_it; it += 32) {
      if (part.column(it, owner) >= vocab) continue;
      float x[VEC];
      RowPart<T>::unpack(slots[it * VR_THREADS + owner], x);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = part.column(it, owner) + i;
        if (order32(x[i]) >= bound && c >= 0 && c < vocab) push(top_key(x[i], c));
      }
    }
  }
  // every CTA learns how many each has: `to` is written in all of them
  auto tell = [&](int* to, int n) {
    if (tid < part.size) st_cluster(mapa_u32(smem_u32(to + part.rank), tid), n);
    cluster_arrive();
    cluster_wait();
  };
  __syncthreads();
  tell(counts[0], s_n);
  bool fits = true;
  for (int i = 0; i < part.size; ++i) fits &= counts[0][i] <= room_each;
  if (!fits) {
    // elements that are at least `key`, in all, and whether every CTA's have room
    int round = 0;
    auto count = [&](TopKey key, bool* room_for_all) {
      const int at = ++round & 1;
      int n = 0;
      for (int s = 0; s < part.n_steps; ++s) {
        float x[16];
        part.get(s, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int c = part.column(s * STEP + i / VEC, tid) + i % VEC;
          n += c >= 0 && c < vocab && s * STEP + i / VEC < part.n_it && top_key(x[i], c) >= key;
        }
      }
      n = __reduce_add_sync(0xffffffffu, n);
      if (lane == 0) atomicAdd(&s_count[at], n);
      __syncthreads();
      const int mine = s_count[at];
      tell(counts[at], mine);
      if (tid == 0) s_count[at] = 0;  // before the barrier inside the next round, which uses the other one
      n = 0;
      *room_for_all = true;
      for (int i = 0; i < part.size; ++i) {
        n += counts[at][i];
        *room_for_all &= counts[at][i] <= room_each;
      }
      return n;
    };
    // lo is reached by k elements, hi by fewer; elements are all different, so that some key between is reached by exactly k
    TopKey lo = (TopKey)bound << TOP_INDEX_BITS, hi = (TopKey)1 << (32 + TOP_INDEX_BITS);
    bool room_for_all = false;
    for (TopKey mid = min(lo + ((TopKey)1 << TOP_INDEX_BITS), hi - 1); !room_for_all; mid = lo + (hi - lo) / 2) {  // first: are the bound's ties the matter?
      const int n = count(mid, &room_for_all);
      room_for_all &= n >= k;
      if (n >= k) lo = mid;
      else hi = mid;
    }
    if (tid == 0) s_n = 0;
    __syncthreads();
    for (int s = 0; s < part.n_steps; ++s) {
      float x[16];
      part.get(s, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = part.column(s * STEP + i / VEC, tid) + i % VEC;
        if (c >= 0 && c < vocab && s * STEP + i / VEC < part.n_it && top_key(x[i], c) >= lo) push(top_key(x[i], c));
      }
    }
    __syncthreads();
    tell(counts[++round & 1], s_n);
    if (tid < part.size) counts[0][tid] = counts[round & 1][tid];
    __syncthreads();
  }
  if (part.rank != 0) return;
  const bool bad = !(m < INFINITY);
  if (tid == 0) {
    s_log_sum = log(sum);
    if (lse) lse[r] = bad ? NAN : (float)((double)m / t + s_log_sum);
  }
  __syncthreads();
  for (int l = 0; l < part.size; ++l)
    for (int i = tid; i < counts[0][l]; i += VR_THREADS) {
      const TopKey key = room[l * room_each + i];
      int rank = 0;
      for (int o = 0; o < part.size; ++o)
        for (int j = 0; j < counts[0][o]; ++j) rank += room[o * room_each + j] > key;
      if (rank >= k) continue;
      const float v = order32_value((uint32_t)(key >> TOP_INDEX_BITS));
      index[r * k + rank] = (1 << TOP_INDEX_BITS) - 1 - (int)(key & ((1 << TOP_INDEX_BITS) - 1));
      logp[r * k + rank] = bad ? NAN : v == -INFINITY ? -INFINITY : (float)(((double)v - m) / t - s_log_sum);
    }
}

int launch_top_logits(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, int k, int* index, float* logp, float* lse) {
  const RowShape shape = row_shape(vocab, z.dtype);
  return with_dtype(z.dtype, [&](auto* zt) {
    using T = std::remove_pointer_t<decltype(zt)>;
    return launch_clusters(c, top_logits_kernel<T>, rows, shape.cluster, shape.slots * 16 + TOP_ROOM * 8, (const T*)z.p, z.ld, vocab, temperature,
                           exp_t(temperature), k, index, logp, lse);
  });
}

}  // namespace rt
