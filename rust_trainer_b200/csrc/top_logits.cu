// The k largest logits of each row, in order, with their log-probabilities: each element read once, by a CTA a row, or by a cluster
// where there are few rows.  While the row streams by, elements from a bound up are kept, and the bound rises: it is a value that k
// threads' maxima so far reach, so that k elements reach it.  A warp's few largest maxima are sample enough to find one that not many
// more reach; it is looked for a few times, and several times k elements are kept on the way.  In the end what reaches the
// last bound, some more than k, goes to every CTA of the cluster, and each is ranked, by the CTA that found it, by
// counting the larger ones.  Only where elements kept or left are too many (values that tie, masked rows, rows in ascending order) the row
// is read again, for a better bound by bisection over values and indices.
//
// Measured, against the bytes at the rate of a copy: 64 of 1024 x 151936 f32 138 us (floor 96, 4.5 TB/s), 32 of 4096 x 128256 bf16 358 us (163), 8 of
// one row of 151936 f32 12 to 13 us.  What bounds it is instructions and their latency: 46 % of the issue slots are taken, an exponential, a comparison
// and a share of the largest for each element, 28 % of the special-function unit; three CTAs on an SM fill each other's waits at row ends
// (sorting of the sample, exchange, ranks: some 8 us a row).  One row alone is launch, a copy's latency and those.
#include "vocab_rows.cuh"

namespace rt {

// Elements that are kept on the way, and that are ranked, at most: in proportion to what random rows need, some 12 k and 2 k (in a cluster, where each
// CTA may hold k by its own bound, 2 k each: with 256 each, 200 of 30 rows of 151936 f32 took 125 us for want of room, and 36 with one CTA a row).
struct TopRoom {
  int kept, ranked;
};
constexpr int TOP_SHORT = 128;  // entries of a list that 256 threads make: 128 of 1475 x 20000 f32 took 80 us with them, 119 with 512
static TopRoom top_room(int k, int cluster) {
  return {k <= 64 ? 1536 : k <= TOP_SHORT ? 2048 : 3584, cluster > 1 ? (k <= 64 ? 256 : k <= TOP_SHORT ? 384 : 640) * cluster : k <= TOP_SHORT ? 768 : 1024};
}
static_assert(RT_TOP_MAX <= 256, "k elements of one CTA's share have to fit");
// An element as an integer, all different: its value's order above, the lower index in front.
constexpr int TOP_INDEX_BITS = 19;
static_assert(RT_VOCAB_MAX <= 1 << TOP_INDEX_BITS);
using TopKey = unsigned long long;
__device__ __forceinline__ TopKey top_key(float v, int c) {
  return ((TopKey)order32(v) << TOP_INDEX_BITS) | (uint32_t)((1 << TOP_INDEX_BITS) - 1 - c);
}

struct alignas(16) TopStat {
  float R, s;  // the sum of the warp's exponentials is s 2^R
  float m, unused;
};

// the lanes' values in descending order
__device__ __forceinline__ uint32_t warp_sort(uint32_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
    for (int stride = size / 2; stride > 0; stride /= 2) {
      const uint32_t o = __shfl_xor_sync(0xffffffffu, v, stride);
      const bool keep_max = ((lane & stride) == 0) == ((lane & size) == 0);
      v = keep_max ? max(v, o) : min(v, o);
    }
  }
  return v;
}

// Sums of exponentials as 2^(x hi - R), hi = log2(e) / T in f32 and R an integer, so that the product and the difference are rounded once,
// together, and sums with different R meet exactly.  What hi leaves out is another temperature by 2^-26 or so: the row's log-sum-exp makes up for it,
// as far as the mass is near the row's maximum.  R is set by the first elements, and again when one is 2^60 times as large, so rarely.
// Elements that are too large or too far down for such an R (beyond 2^22 in units of T / log2(e)) have none: R = inf, or stays -inf, and a
// row where that matters, one whose own R is inf or not well above the least one, is summed again, relative to its maximum.
constexpr float TOP_MOST_R = 4194304.0f;
struct RunningSum {
  float R = -INFINITY, most = -INFINITY;  // most: elements up to here need no other R
  F2 s[2] = {0, 0};
  __device__ __forceinline__ void take(const float (&x)[16], float largest, float hi) {
    if (!(largest <= most)) {
      if (R == R) {  // a NaN stays
        const float to = largest == largest ? ceilf(largest * hi) : NAN;
        if (!(to < -TOP_MOST_R)) {
          const float by = R > -INFINITY ? ex2(R - to) : 0.0f;
          s[0] = mul2(s[0], pack2(by, by));
          s[1] = mul2(s[1], pack2(by, by));
          R = to > TOP_MOST_R ? INFINITY : to;
          most = (R + 60.0f) / hi;
        }
      }
    }
    const float r = R > -INFINITY ? -R : 0.0f;
    const F2 minus_r = R > -INFINITY ? pack2(r, r) : pack2(-INFINITY, -INFINITY), by = pack2(hi, hi);
    F2 acc[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      float a, b;
      unpack2(fma2(pack2(x[i], x[i + 1]), by, minus_r), &a, &b);
      acc[i / 2 & 1] = add2(acc[i / 2 & 1], pack2(ex2(a), ex2(b)));
    }
    s[0] = add2(s[0], acc[0]);
    s[1] = add2(s[1], acc[1]);
  }
};

// SHORT: rows of one unit, where not all threads may hold elements; what such rows need took 3 to 5 % of long ones' time.
template <class T, int NT, bool SHORT>
__global__ void __launch_bounds__(NT + 32, ctas_of(NT))
top_logits_kernel(const T* z, size_t ld, size_t rows, int vocab, float t, ExpT ex, int k, int* index, float* logp, float* lse, int places,
                  int kept_most, int room_most, int* status) {
  constexpr int STEP = sizeof(T) == 4 ? 4 : 2;
  using Ring = UnitRing<T, NT, STEP>;
  constexpr int VEC = Ring::VEC, WARPS = NT / 32, SAMPLE_LANE = ((NT == 256 ? TOP_SHORT : RT_TOP_MAX) + 2 * WARPS + 31) / 32;
  extern __shared__ uint4 slots[];
  __shared__ uint64_t bars[2 * VR_MAX_UNITS + 2];
  __shared__ TopStat stats[2][VR_MAX_CLUSTER * WARPS];
  __shared__ uint2 told[2][VR_MAX_CLUSTER];  // what every CTA told
  __shared__ uint2 met[VR_MAX_CLUSTER];  // never read: that something came is all it says
  __shared__ uint32_t sample[32 * SAMPLE_LANE];
  __shared__ double s_lse, s_sums[WARPS];
  __shared__ int s_kept, s_n, s_count[2], s_found[VR_MAX_CLUSTER];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_kept = s_n = s_count[0] = s_count[1] = 0;
  Exchange exchange;
  Ring ring(slots + (kept_most + room_most) / 2, bars, places, status, vocab);
  exchange.begin(bars + 2 * VR_MAX_UNITS, status);
  cluster_sync_all();  // nobody sends to a CTA that does not run yet
  const size_t row_step = gridDim.x / (unsigned)ring.size;
  if (tid >= NT) {
    if (tid == NT) ring.copy_rows(z, ld, rows, row_step);
    return;
  }
  const double inv_t = 1.0 / t;
  const float hi = ex.hi;
  // values of a warp in the sample: W warps send at most W + k + W of them
  const int each_of_all = min((k + WARPS - 1) / WARPS + 1, 32), warps = ring.size * WARPS;
  int holders = WARPS, each = each_of_all, sampled = WARPS * each;  // warps that hold elements of the row
  TopKey *kept = (TopKey*)slots, *room = kept + kept_most;
  const int room_each = room_most / ring.size;
  // A value that k of the threads' maxima reach, and not many more of the sample's, in every warp the same.
  auto bound_of = [&](float largest) {
    const uint32_t sorted = warp_sort(order32(largest));
    work_sync<NT>();  // the last one's sample has been read
    if (lane < each && (!SHORT || warp < holders)) sample[warp * each + lane] = sorted;
    work_sync<NT>();
    uint32_t some[SAMPLE_LANE], lo = 0xffffffffu, hi = 0;  // lo is reached by k; no value is above hi
#pragma unroll
    for (int i = 0; i < SAMPLE_LANE; ++i) {
      const bool on = i * 32 + lane < sampled;
      some[i] = on ? sample[i * 32 + lane] : 0;
      if (on) lo = min(lo, some[i]);
      hi = max(hi, some[i]);
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (SHORT && sampled < k) return order32(-INFINITY);  // too few threads hold elements
    while (hi > lo) {  // at most 32 times
      const uint32_t mid = lo + (hi - lo) / 2 + 1;
      int n = 0;
#pragma unroll
      for (int i = 0; i < SAMPLE_LANE; ++i)
        if (i * 32 < sampled) n += some[i] >= mid;
      n = __reduce_add_sync(0xffffffffu, n);
      if (n >= k) lo = mid;
      else hi = mid - 1;
      if (n >= k && n <= k + k / 8 + 2) break;
    }
    return lo;
  };
  // Two numbers of every CTA, in every one of them.
  auto tell = [&](uint32_t a, uint32_t b) {
    uint2* to = told[exchange.turn()];
    if (tid == 0) exchange.expect(ring.size * 8);
    if (tid < ring.size) send(mapa_u32(smem_u32(to + ring.rank), tid), exchange.bar(tid), a, b);
    exchange.wait();
    return (const uint2*)to;
  };
  for (size_t r = cluster_id(); r < rows; r += row_step) {
    ring.begin(z + r * ld);
    if constexpr (SHORT) {
      const int with = min(NT, ring.n_vec), whole = max(with / 32, 1);
      holders = (with + 31) / 32;
      each = min((k + whole - 1) / whole + 1, min(32, 32 * SAMPLE_LANE / holders));
      sampled = holders * each;
    }
    RunningSum sum;
    float largest = -INFINITY;  // of the thread's elements
    uint32_t bound = 0;
    float from = 0.0f;  // elements from here up are kept
    auto set_bound = [&](uint32_t b) {
      bound = b;
      from = order32_value(b);
      if (from == 0.0f) from = -1.4e-45f;  // the two zeros are equal, which the sign of a difference is not
    };
#pragma unroll 1
    for (int s = 0; s < ring.n_units; ++s) {
      uint4* const at = ring.slots + ring.place * Ring::UNIT + tid;
      row_wait(ring.full + ring.place, ring.phase, status);
      if (s == 0 || s + 1 == ring.n_units) {
        ring.complete(s, at);
        fence_proxy_async_smem();  // what it wrote comes before the copies that follow
      }
      uint4 v[STEP];
#pragma unroll
      for (int j = 0; j < STEP; ++j) v[j] = at[j * NT];
      float x[16], top;
#pragma unroll
      for (int j = 0; j < STEP; ++j) unpack_vector<T>(v[j], x + j * VEC);
      using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
      const T2* const x2 = (const T2*)v;  // 16-bit elements in pairs
      if constexpr (sizeof(T) == 4) {
        top = max_nan(x[0], x[1], x[2]);
#pragma unroll
        for (int i = 3; i < 15; i += 2) top = max_nan(top, x[i], x[i + 1]);
        top = max_nan(top, x[15]);
      } else {
        T2 m = x2[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = __hmax2_nan(m, x2[i]);
        top = max_nan(to_f32(m.x), to_f32(m.y));
      }
      sum.take(x, top, hi);
      largest = max_nan(largest, top);
      // for a bound: after 1, 4, 16 ... units (1, 2, 4, 8 ... for long lists), but not shortly before the end
      if ((s & (s + 1)) == 0 && (k > TOP_SHORT || (s + 1) % 3 == 1) && (s == 0 || (s + 1) * 4 < ring.n_units * 3)) set_bound(bound_of(largest));
      if (!(top < from)) {  // NaN too
        // a bit for each element that is not below
        uint32_t hits = 0;
        if constexpr (sizeof(T) == 4) {
          const F2 minus_from = pack2(-from, -from);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float a, b;
            unpack2(add2(pack2(x[i], x[i + 1]), minus_from), &a, &b);
            hits = __funnelshift_l(__float_as_uint(a), hits, 1);
            hits = __funnelshift_l(__float_as_uint(b), hits, 1);
          }
          hits = ~hits & 0xffff;
        } else {
          const T f = from_f32<T>(from == -1.4e-45f ? 0.0f : from);  // one of the elements, or a zero
          T2 f2;
          f2.x = f2.y = f;
#pragma unroll
          for (int i = 0; i < 8; ++i) hits |= (~__hlt2_mask(x2[i], f2) & 0x00010001u) << i;
        }
        if (SHORT && from == -INFINITY) {  // nothing is below: all of a short row, but not what lies outside of it
#pragma unroll 1
          for (int i = 0; i < 16; ++i) {
            const int c = ring.column(s, i / VEC) + i % VEC;
            if (c < 0 || c >= vocab) hits &= ~(1u << (sizeof(T) == 4 ? 15 - i : i / 2 + 16 * (i & 1)));
          }
        }
        if (*(volatile int*)&s_kept <= kept_most) {  // else there are too many already
          int p = atomicAdd(&s_kept, __popc(hits));
          for (; hits && p < kept_most; ++p, hits &= hits - 1) {
            const int bit = __ffs(hits) - 1, i = sizeof(T) == 4 ? 15 - bit : 2 * (bit & 15) + (bit >> 4), j = i / VEC, c = ring.column(s, j) + i % VEC;
            // what lies outside of the row is below every element
            kept[p] = c >= 0 && c < vocab ? top_key(to_f32(((const T*)(at + j * NT))[i % VEC]), c) : 0;
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(ring.empty + ring.place);
      ring.next();
    }
    set_bound(bound_of(largest));
    TopStat st;
    {
      float a, b;
      unpack2(add2(sum.s[0], sum.s[1]), &a, &b);
      st.R = warp_max_nan(sum.R);
      st.m = warp_max_nan(largest);
      st.s = warp_sum_f32(sum.R > -INFINITY ? (a + b) * ex2(sum.R - st.R) : 0.0f);
    }
    TopStat* stat = stats[exchange.turn()];
    uint2* to = told[exchange.turn()];
    const int n_kept = s_kept;  // all have been counted before the bound's barriers
    // (What was told may be anything once a wait has run out: no count is taken for more than there is room, and no loop goes by them alone.)
    if (tid == 0) exchange.expect(warps * sizeof(TopStat) + ring.size * 8);
    if (lane < ring.size)
      send(mapa_u32(smem_u32(&stat[ring.rank * WARPS + warp]), lane), exchange.bar(lane), __float_as_uint(st.R), __float_as_uint(st.s), __float_as_uint(st.m), 0u);
    if (tid < ring.size) send(mapa_u32(smem_u32(to + ring.rank), tid), exchange.bar(tid), bound, (uint32_t)n_kept);
    exchange.wait();
    float m = -INFINITY, R = -INFINITY;
    for (int i = lane; i < warps; i += 32) m = max_nan(m, stat[i].m), R = max_nan(R, stat[i].R);
    m = warp_max_nan(m);
    R = warp_max_nan(R);
    // (R 64 above the least one: an element that was left out is at most 2^-64 of the row's sum)
    const bool bad = !(m < INFINITY), again = !bad && m > -INFINITY && !(R >= 64.0f - TOP_MOST_R && R < INFINITY);
    if (warp == WARPS - 1 && !again) {
      double all = 0.0;
      for (int i = lane; i < warps; i += 32)
        if (stat[i].R > -INFINITY) all += (double)(stat[i].s * ex2(stat[i].R - R));
      all = warp_sum_f64(all);
      // log sum 2^(x (hi + lo)), of which R and the sum have hi
      if (lane == 0) s_lse = bad ? NAN : m == -INFINITY ? -INFINITY : log(all) + ((double)R + (double)m * ex.lo) * 0.69314718055994530942;
    }
    bool fits = true;
    for (int i = 0; i < ring.size; ++i) {  // every CTA's bound holds for the row
      fits &= to[i].y <= (uint32_t)kept_most;
      bound = max(bound, to[i].x);
    }
    // elements to be ranked: this CTA's lie in its share of the room
    TopKey* mine = room + ring.rank * room_each;
    auto push = [&](TopKey key) {
      const int p = atomicAdd(&s_n, 1);
      if (p < room_each) mine[p] = key;
    };
    if (fits) {
      for (int i = tid; i < min(n_kept, kept_most); i += NT)
        if (kept[i] >= (TopKey)bound << TOP_INDEX_BITS) push(kept[i]);
    }
    work_sync<NT>();
    const uint2* found = tell((uint32_t)s_n, 0);
    for (int i = 0; i < ring.size; ++i) fits &= found[i].x <= (uint32_t)room_each;
    // the thread's elements once more, which is rare
    auto each_element = [&](auto&& f) {
#pragma unroll 1
      for (int i = 0; i < ring.n_units * STEP; ++i) {
        const int c0 = ring.column(i / STEP, i % STEP);
        for (int c = max(c0, 0); c < min(c0 + VEC, vocab); ++c) f(to_f32(ring.row[c]), c);
      }
    };
    if (again) {
      double mine = 0.0;
      each_element([&](float v, int) { mine += ex(v - m); });
      mine = warp_sum_f64(mine);
      if (lane == 0) s_sums[warp] = mine;
      work_sync<NT>();
      double all = 0.0;  // of the CTA's elements, and of the cluster's
      for (int i = 0; i < WARPS; ++i) all += s_sums[i];
      const uint2* sums = tell(__double2loint(all), __double2hiint(all));
      all = 0.0;
      for (int i = 0; i < ring.size; ++i) all += __hiloint2double(sums[i].y, sums[i].x);
      work_sync<NT>();
      if (tid == 0) s_lse = log(all) + (double)m * inv_t;
      work_sync<NT>();
    }
    if (!fits) {
      // elements that are at least `key`, in all, and whether every CTA's have room
      int round = 0;
      auto count = [&](TopKey key, bool* room_for_all) {
        const int now = ++round & 1;
        int n = 0;
        each_element([&](float v, int c) { n += top_key(v, c) >= key; });
        n = __reduce_add_sync(0xffffffffu, n);
        if (lane == 0) atomicAdd(&s_count[now], n);
        work_sync<NT>();
        const uint2* counts = tell((uint32_t)s_count[now], 0);
        n = 0;
        *room_for_all = true;
        for (int i = 0; i < ring.size; ++i) {
          n += (int)counts[i].x;
          *room_for_all &= counts[i].x <= (uint32_t)room_each;
        }
        work_sync<NT>();
        if (tid == 0) s_count[now] = 0;  // before the barrier of the next round, which uses the other one
        return n;
      };
      // low is reached by k elements, high by fewer; elements are all different, so that some key between is reached by exactly k
      TopKey low = (TopKey)bound << TOP_INDEX_BITS, high = (TopKey)1 << (32 + TOP_INDEX_BITS);
      bool room_for_all = false;
      // the first question: are the bound's ties the matter?  (Then at most one for each bit of a key.)
      for (TopKey mid = min(low + ((TopKey)1 << TOP_INDEX_BITS), high - 1); !room_for_all && round < 64; mid = low + (high - low) / 2) {
        const int n = count(mid, &room_for_all);
        room_for_all &= n >= k;
        if (n >= k) low = mid;
        else high = mid;
      }
      if (tid == 0) s_n = 0;
      work_sync<NT>();
      each_element([&](float v, int c) {
        if (top_key(v, c) >= low) push(top_key(v, c));
      });
      work_sync<NT>();
      found = tell((uint32_t)s_n, 0);
    }
    auto n_found = [&](int i) { return (int)min(found[i].x, (uint32_t)room_each); };
    int n_mine = n_found(ring.rank);
    if (ring.size > 1) {  // everybody's to everybody
      int n = 0;
      for (int i = 0; i < ring.size; ++i) n += n_found(i);
      if (tid < ring.size) s_found[tid] = n_found(tid);  // what was told may be overwritten once this exchange is over
      work_sync<NT>();
      // A word from everybody comes with them, behind the barrier: nobody goes on to the next row, and tells of it, where `found` is still read.  A
      // CTA that has all elements of the row would wait for no others.
      if (tid == 0) exchange.expect((uint32_t)(n - n_mine + ring.size) * 8);
      if (tid < ring.size) send(mapa_u32(smem_u32(met + ring.rank), tid), exchange.bar(tid), 0u, 0u);
      for (int i = tid; i < n_mine; i += NT) {
        const uint2 key = *(const uint2*)(mine + i);
        for (int o = 0; o < ring.size; ++o)
          if (o != ring.rank) send(mapa_u32(smem_u32(mine + i), o), exchange.bar(o), key.x, key.y);
      }
      exchange.wait();
    }
    const TopKey* others_room = room;
    // Many more than k, of a short row with a long list: ranks by counting would take the square of them.  A key that k reach, and few more.
    if (SHORT && n_mine > 2 * k + 64) {
      TopKey low = 0, high = (TopKey)1 << (32 + TOP_INDEX_BITS);
      while (high - low > 1) {  // at most 51 times
        const TopKey mid = low + (high - low) / 2;
        int n = 0;
        for (int i = 0; i < n_mine; i += NT) n += work_count<NT>(i + tid < n_mine && mine[i + tid] >= mid);
        if (n >= k) low = mid;
        else high = mid;
        if (n >= k && n <= k + k / 2 + 8) break;
      }
      if (tid == 0) s_kept = 0;
      work_sync<NT>();
      for (int i = tid; i < n_mine; i += NT)
        if (mine[i] >= low) kept[atomicAdd(&s_kept, 1)] = mine[i];
      work_sync<NT>();
      n_mine = s_kept;
      mine = kept;
      others_room = kept;
    }
    const double row_lse = s_lse;
    if (lse && tid == 0 && ring.rank == 0) lse[r] = (float)row_lse;
    // a thread an element: its rank is the number of larger ones
    for (int i = tid; i < n_mine; i += NT) {
      const TopKey key = mine[i];
      int rank = 0;
      for (int o = 0; o < ring.size; ++o) {
        const int n = ring.size > 1 ? s_found[o] : n_mine;
        const TopKey* const others = others_room + o * room_each;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += others[j] > key;
      }
      if (rank >= k) continue;
      const float v = order32_value((uint32_t)(key >> TOP_INDEX_BITS));
      index[r * k + rank] = (1 << TOP_INDEX_BITS) - 1 - (int)(key & ((1 << TOP_INDEX_BITS) - 1));
      logp[r * k + rank] = bad ? NAN : v == -INFINITY ? -INFINITY : (float)(v * inv_t - row_lse);
    }
    work_sync<NT>();
    if (tid == 0) s_n = s_kept = 0;  // the next row's first bound has barriers before they count again
  }
}

int launch_top_logits(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, int k, int* index, float* logp, float* lse) {
  // Long lists want more threads, whose maxima are the sample that the bound is found in.  Three CTAs on an SM, or one; more CTAs a row where there are
  // few rows, as long as two find room on an SM: 32 of 64 rows of 151936 f32 took 36 us with one, 27 with two, 25 with four and 37 with eight; of
  // 128 rows 39, 33, 41 and 57.
  const int threads = k <= TOP_SHORT ? 256 : 512, vec = z.dtype == RT_DT_F32 ? 4 : 8, units = (vec - 1 + vocab + 16 * threads - 1) / (16 * threads);
  int size = 1;
  const size_t at_once = (threads == 256 ? 2 : 1) * (size_t)c->num_sms;
  while (size * 2 <= VR_MAX_CLUSTER && units > size && rows * size * 2 <= at_once) size *= 2;
  // A CTA that has nothing but the row's last unit finds no bound if that holds elements for few of its warps: it would keep whatever it sees, and the row would be
  // read again (32 of 16 x 8692 f32: 20.5 us so, 10.3 with half as many CTAs).
  const int warps = threads / 32, last = (vocab + vec - 1) / vec - (units - 1) * 16 * threads / vec;
  while (size > 1 && units <= size && last / 32 * std::min((k + warps - 1) / warps + 1, 32) < k) size /= 2;
  const TopRoom room = top_room(k, size);
  const size_t other = (room.kept + room.ranked) * sizeof(TopKey), unit = (size_t)threads * 16 * (z.dtype == RT_DT_F32 ? 4 : 2);
  const int places = (int)std::min(((threads != 256 ? 208 : size > 1 ? 104 : 70) * 1024 - other) / unit, (size_t)VR_MAX_UNITS);
  return with_dtype(z.dtype, [&](auto* zt) {
    return with_threads(threads, [&](auto n) {
      using T = std::remove_pointer_t<decltype(zt)>;
      constexpr int NT = decltype(n)::value;
      return launch_clusters(c, units == 1 ? top_logits_kernel<T, NT, true> : top_logits_kernel<T, NT, false>, true, rows, threads + 32, size,
                             places * unit + other, (const T*)z.p, z.ld, rows, vocab, temperature, exp_t(temperature), k, index, logp, lse, places, room.kept, room.ranked, c->status_dev);
    });
  });
}

}  // namespace rt
