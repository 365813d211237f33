// The k largest logits of each row, in order, with their log-probabilities: a cluster of CTAs a row, which holds the row in shared
// memory.  Which elements can be among the k largest follows from the threads' maxima, which the pass over the exponentials
// finds anyway: if every one of W warps has j = ceil(k / W) threads with a maximum of at least x, then k elements are at least x.
// The elements from there up, a few times k of them, go to the cluster's first CTA, which ranks each by counting the larger ones.
// Only where they are too many (values that tie, masked rows) is a bound sought that leaves fewer, by bisection over values and
// indices.
#include "vocab_rows.cuh"
#include <algorithm>

namespace rt {

constexpr int TOP_ROOM = 2048;  // candidates
// slots of the row's region at least: it takes the candidates once more when the row is no longer needed
constexpr int TOP_LEAST_SLOTS = TOP_ROOM / 2 + 1;
static_assert(TOP_ROOM / VR_MAX_CLUSTER >= RT_TOP_MAX, "k elements of one CTA's share have to fit");
// An element as an integer, all different: its value's order above, the lower index in front.
constexpr int TOP_INDEX_BITS = 19;
static_assert(RT_VOCAB_MAX <= 1 << TOP_INDEX_BITS);
using TopKey = unsigned long long;
__device__ __forceinline__ TopKey top_key(float v, int c) {
  return ((TopKey)order32(v) << TOP_INDEX_BITS) | (uint32_t)((1 << TOP_INDEX_BITS) - 1 - c);
}

struct TopStat {
  float m, s;
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
__global__ void __launch_bounds__(VR_THREADS, 2) top_logits_kernel(const T* z, size_t ld, int vocab, float t, ExpT ex, int k, int* index, float* logp, float* lse, int* status) {
  constexpr int VEC = RowPart<T>::VEC, STEP = RowPart<T>::STEP;
  extern __shared__ uint4 slots[];
  __shared__ uint64_t bars[VR_MAX_STEPS];
  __shared__ TopStat stat[VR_MAX_CLUSTER * VR_WARPS];
  __shared__ int s_n, s_count[2], counts[2][VR_MAX_CLUSTER];
  __shared__ double s_log_sum;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster_arrive_relaxed();
  const size_t r = cluster_id();
  const RowPart<T> part(z + r * ld, vocab, slots, bars, status);
  part.load();
  TopKey* room = (TopKey*)(slots + max(part.n_it_most() * VR_THREADS, TOP_LEAST_SLOTS));
  const int room_each = TOP_ROOM / part.size;
  if (tid == 0) s_n = s_count[0] = s_count[1] = 0;
  __syncthreads();
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
  st.s = warp_join(ms, ex, &st.m);
  cluster_wait();  // the other CTAs run: their shared memory may be written
  if (lane < part.size) {
    const uint32_t to = mapa_u32(smem_u32(&stat[part.rank * VR_WARPS + warp]), lane);
    st_cluster(to, __float_as_uint(st.m), __float_as_uint(st.s));
    st_cluster(to + 8, st.each, st.own);
  }
  cluster_arrive();
  cluster_wait();
  const TopStat none{-INFINITY, 0.0f, 0xffffffffu, 0xffffffffu}, a = lane < warps ? stat[lane] : none, b = lane + 32 < warps ? stat[lane + 32] : none;
  uint32_t own = a.own, own_b = b.own;  // eight neighbours are a CTA's warps
#pragma unroll
  for (int o = 1; o < VR_WARPS; o *= 2) {
    own = min(own, __shfl_xor_sync(0xffffffffu, own, o));
    own_b = min(own_b, __shfl_xor_sync(0xffffffffu, own_b, o));
  }
  const uint32_t own_max = __reduce_max_sync(0xffffffffu, max(lane < warps ? own : 0u, lane + 32 < warps ? own_b : 0u));
  const uint32_t bound = max(__reduce_min_sync(0xffffffffu, min(a.each, b.each)), own_max);
  float m;
  const double sum = cluster_join(a.m, a.s, b.m, b.s, ex, &m);

  const uint32_t leader_room = mapa_u32(smem_u32(room), 0);
  auto push = [&](TopKey key) {
    const int p = atomicAdd(&s_n, 1);
    if (p < room_each) st_cluster(leader_room + (uint32_t)(part.rank * room_each + p) * 8, key);
  };
  if (my_top >= bound) {  // a few threads of a warp, which look for their elements side by side
    const float from = order32_value(bound);
    for (int it = 0; it < part.n_it; ++it) {
      const int c0 = part.column(it, tid);
      if (c0 >= vocab) break;
      float x[VEC];
      RowPart<T>::unpack(slots[it * VR_THREADS + tid], x);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (!(x[i] < from) && c0 + i >= 0 && c0 + i < vocab) push(top_key(x[i], c0 + i));  // NaN too
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
  // The lists one behind the other in what held the row: orders, filled up with the lowest to a multiple of four, and columns.
  int n = 0;
  for (int l = 0; l < part.size; ++l) n += counts[0][l];
  const int n4 = (n + 3) / 4;
  uint32_t *order = (uint32_t*)slots, *column = order + 4 * n4;
  int before = 0;
  for (int l = 0; l < part.size; ++l) {
    const int here = counts[0][l];
    for (int i = tid; i < here; i += VR_THREADS) {
      const TopKey key = room[l * room_each + i];
      order[before + i] = (uint32_t)(key >> TOP_INDEX_BITS);
      column[before + i] = (1 << TOP_INDEX_BITS) - 1 - (uint32_t)(key & ((1 << TOP_INDEX_BITS) - 1));
    }
    before += here;
  }
  if (tid < 4 * n4 - n) order[n + tid] = 0;
  __syncthreads();
  const double log_sum = s_log_sum;
  for (int i = tid; i < n; i += VR_THREADS) {
    const uint32_t mine = order[i];
    int rank = 0, same = -1;
#pragma unroll 4
    for (int j = 0; j < n4; ++j) {
      const uint4 o = ((const uint4*)order)[j];
      rank += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
      same += (o.x == mine) + (o.y == mine) + (o.z == mine) + (o.w == mine);
    }
    if (rank >= k) continue;
    if (same > 0)
      for (int j = 0; j < n; ++j) rank += order[j] == mine && column[j] < column[i];
    if (rank >= k) continue;
    const float v = order32_value(mine);
    index[r * k + rank] = (int)column[i];
    logp[r * k + rank] = bad ? NAN : v == -INFINITY ? -INFINITY : (float)(((double)v - m) / t - log_sum);
  }
}

int launch_top_logits(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, int k, int* index, float* logp, float* lse) {
  const RowShape shape = row_shape(vocab, z.dtype);
  const size_t smem = std::max(shape.slots, (size_t)TOP_LEAST_SLOTS) * 16 + TOP_ROOM * 8;
  return with_dtype(z.dtype, [&](auto* zt) {
    using T = std::remove_pointer_t<decltype(zt)>;
    return launch_clusters(c, top_logits_kernel<T>, rows, shape.cluster, smem, (const T*)z.p, z.ld, vocab, temperature,
                           exp_t(temperature), k, index, logp, lse, c->status_dev);
  });
}

}  // namespace rt
