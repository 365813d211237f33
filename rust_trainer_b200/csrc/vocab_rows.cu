// Softmax and distillation over rows of logits.  A row is read once: it lies in the shared memory of a cluster of CTAs until its sums have
// gone round.  In each CTA some warps sum row n + 1 while others write row n and the next ones are copied, so that memory is busy while sums
// are found and go round, and a warp or a few make each row's list ready and find its loss.
//
// Measured, against the bytes at the rate of a copy: softmax of 1536 x 128256 bf16 into f32 219 to 226 us (floor 183, 5.2 to 5.4 TB/s); gradients of
// 1024 x 151936 f32 in f16 from 64 entries 215 us (144), of 2048 x 128256 bf16 from 32 244 to 248 us (162); losses alone of 777 x 50021 f16
// 37 us (12).  (All warps at one row after the other, with the same copies ahead: 285, 264, 283 and 37 us.)  What bounds distillation is the
// chain of a row: its last unit's copy (some 4500 of the f32 row's 17300 cycles over two rows), the sums (4700), the exchange and the coefficients
// (3200), the writing (4000), and two rows are all that a cluster's shared memory holds.  A wait on a barrier costs 100 to 200 cycles in
// these loops: whoever is told of a whole row does not wait for its units (219 -> 215 us, 269 -> 244).  Tried without gain, in us for the f32 rows: units in pairs
// (286), lists that are taken out unit by unit so that sums begin behind the copy (248), entries that each wait for their own unit (233), two CTAs
// on an SM with half of the row each (420 and more), clusters that start one after the other, the factor in the exponent for 16-bit results (the same).
//
// What passes between the roles, row i of a CTA (all of them mbarriers, two or four in turn):
//   full, empty   a unit has been copied; the warps that write the row (or, for a loss alone, that sum it) give it back
//   patched       the list's warps have taken the listed elements out of the row
//   summed        the row's exponentials and references are there
//   listed        the list's entries are there, for the warp that writes their gradients (what is sent to `exchange` says nothing of them)
//   exchange      all CTAs' sums of the row, and what their lists say, have come
//   written       by the warps that write
//   done          the row has been written, its listed elements too, and its loss found; row i + 2 may take its references' and its list's places.
//                 Its sums are sent after that: whoever has seen exchange i - 2 complete knows that every CTA is done with row i - 4, whose
//                 place the sums of row i take there
#include "vocab_rows.cuh"

namespace rt {

constexpr int ROW_STEP = 2;  // vectors of a thread in a unit
struct RowBars {
  uint64_t units[2 * VR_MAX_UNITS], exchange[4], summed[2], written[2], done[2], patched[2], listed[2];
};
// What a warp knows of its share of a row, and sends to every CTA of the cluster: a reference, and the sum of exponentials relative to it.
struct alignas(8) RowStat {
  float m, s;
};
__device__ __forceinline__ void row_wait_turn(uint64_t* bars, uint32_t i, uint32_t turns_log2, int* status) {
  row_wait(bars + (i & ((1u << turns_log2) - 1)), i >> turns_log2 & 1, status);
}

// The warps that sum.  A thread's reference is the largest of its warp's first vectors: an exponential may be as large as 2^10 before it changes,
// so that it rarely does, and an exponent's rounding is small where the large ones are (with the thread's own, and up to 2^30, probabilities of f32
// rows were off by 3 to 4e-7 instead of 1.4 to 2.5e-7).  KEEP (32-bit rows): the exponentials take their elements' place, for the warps that write.
template <class T, int NT, bool KEEP>
__device__ __forceinline__ void sum_rows(UnitRing<T, NT, ROW_STEP>& ring, const T* z, size_t ld, size_t rows, size_t row_step, const ExpT& ex, RowBars& b,
                                         float (*refs)[NT], RowStat (*stats)[VR_MAX_CLUSTER * (NT / 32)], uint32_t bytes, bool listed, bool give_back) {
  using Ring = UnitRing<T, NT, ROW_STEP>;
  constexpr int VEC = Ring::VEC, WARPS = NT / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float most = 10.0f / ex.hi;
  uint32_t i = 0;
  for (size_t r = cluster_id(); r < rows; r += row_step, ++i) {
    ring.begin(z + r * ld);
    if (i >= 2) row_wait_turn(b.done, i - 2, 1, ring.status);
    if (listed) row_wait_turn(b.patched, i, 1, ring.status);
    const int first_place = ring.place;
    float ref = -INFINITY;
    F2 acc[4] = {0, 0, 0, 0};
#pragma unroll 1
    for (int u = 0; u < ring.n_units; ++u) {
      if (!listed) ring.wait();  // else the list's warps have waited
      uint4* const at = ring.unit() + tid;
      if (!listed && (u == 0 || u + 1 == ring.n_units)) ring.complete(u, at);
      const uint4 v[2] = {at[0], at[NT]};
      float top;
      if constexpr (sizeof(T) == 4) {
        top = max_nan(__uint_as_float(v[0].x), __uint_as_float(v[0].y), max_nan(__uint_as_float(v[0].z), __uint_as_float(v[0].w)));
        top = max_nan(max_nan(top, __uint_as_float(v[1].x), __uint_as_float(v[1].y)), __uint_as_float(v[1].z), __uint_as_float(v[1].w));
      } else {
        using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
        T2 m = __hmax2_nan(__hmax2_nan(*(const T2*)&v[0].x, *(const T2*)&v[0].y), __hmax2_nan(*(const T2*)&v[0].z, *(const T2*)&v[0].w));
        m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(*(const T2*)&v[1].x, *(const T2*)&v[1].y), __hmax2_nan(*(const T2*)&v[1].z, *(const T2*)&v[1].w)));
        top = max_nan(to_f32(m.x), to_f32(m.y));
      }
      if (u == 0 || (!(top <= ref + most) && ref == ref)) {  // the first ones, ones that are far larger, a NaN, which stays
        if (u == 0) top = warp_max_nan(top);
        if (ref > -INFINITY) {
          const bool far = KEEP && (ref - top) * ex.hi < -60.0f;  // in two factors, as in write_row
          const float by = ex(far ? 0.5f * (ref - top) : ref - top), then = far ? by : 1.0f;
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = mul2(mul2(acc[j], pack2(by, by)), pack2(then, then));
          if constexpr (KEEP) {
#pragma unroll 1
            for (int k = 0, place = first_place; k < u; ++k) {
#pragma unroll
              for (int j = 0; j < ROW_STEP; ++j) {
                float4* e = (float4*)(ring.slots + place * Ring::UNIT + j * NT + tid);
                *e = make_float4(e->x * by * then, e->y * by * then, e->z * by * then, e->w * by * then);
              }
              if (++place == ring.places) place = 0;
            }
          }
        }
        ref = top;
      }
      const float base = ref > -INFINITY ? -ref : 0.0f;
      const F2 minus_ref = pack2(base, base);
#pragma unroll
      for (int j = 0; j < ROW_STEP; ++j) {
        float x[VEC];
        unpack_vector<T>(v[j], x);
#pragma unroll
        for (int k = 0; k < VEC; k += 2) {
          ex.pair(pack2(x[k], x[k + 1]), minus_ref, x + k, x + k + 1);
          acc[(j * VEC + k) / 2 & 3] = add2(acc[(j * VEC + k) / 2 & 3], pack2(x[k], x[k + 1]));
        }
        if constexpr (KEEP) at[j * NT] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
      }
      if (give_back) ring.release();
      ring.next();
    }
    refs[i & 1][tid] = ref;
    fence_proxy_async_smem();  // what was written in the units comes before the copies that follow
    __syncwarp();
    if (lane == 0) mbar_arrive(b.summed + (i & 1));
    float x, y, m;
    unpack2(add2(add2(acc[0], acc[1]), add2(acc[2], acc[3])), &x, &y);
    const float s = warp_join(ref, x + y, ex, &m);
    if (i >= 2) row_wait_turn(b.exchange, i - 2, 2, ring.status);
    if (tid == 0) mbar_expect_tx(b.exchange + (i & 3), bytes);
    if (lane < ring.size)
      send(mapa_u32(smem_u32(&stats[i & 3][ring.rank * WARPS + warp]), lane), mapa_u32(smem_u32(b.exchange + (i & 3)), lane), __float_as_uint(m), __float_as_uint(s));
  }
}

// One row's results into `out`, by the warps that write: (16-bit rows) e f, e the exponentials relative to the row's reference, or (32-bit rows, whose
// exponentials are there relative to the thread's reference `mine`) those times what that makes f.  Gives the units back.
// PACED: with a wait for each unit, which the warps that sum have seen full already.  Where memory binds it spreads the stores: softmax of 1536 x
// 128256 bf16 rows, one call after the other, takes 220 us with it and 224 without; distillation of 1024 x 151936 f32 rows 219 and 215, of
// 2048 x 128256 bf16 rows 269 and 244.
template <bool PACED, class O, class T, int NT>
__device__ __forceinline__ void write_row(UnitRing<T, NT, ROW_STEP>& ring, O* out, float mine, float reference, float f, const ExpT& ex) {
  using Ring = UnitRing<T, NT, ROW_STEP>;
  constexpr int VEC = Ring::VEC;
  const bool aligned = ((uintptr_t)out - (uintptr_t)ring.align * sizeof(O)) % (VEC * sizeof(O) < 16 ? VEC * sizeof(O) : 16) == 0;
  const float ref = reference > -INFINITY ? reference : 0.0f;
  // far below the reference in two factors: what is left of an exponential of 2^10 may be 2^10 larger than what one factor can say
  float h = 1.0f;
  if (sizeof(T) == 4 && mine > -INFINITY) {
    const bool far = (mine - reference) * ex.hi < -60.0f;
    const float by = ex(far ? 0.5f * (mine - reference) : mine - reference);
    if (far) h = by;
    f *= by;
  }
  const F2 minus_ref = pack2(-ref, -ref), by = pack2(f, f), half_way = pack2(h, h);
#pragma unroll 1
  for (int u = 0; u < ring.n_units; ++u) {
    if (PACED) ring.wait();
    const uint4* const at = ring.unit() + threadIdx.x % NT;
    const uint4 v[2] = {at[0], at[NT]};
    ring.release();
    ring.next();
    const int c = ring.column(u, 0);
#pragma unroll
    for (int j = 0; j < ROW_STEP; ++j) {
      float x[VEC];
      unpack_vector<T>(v[j], x);
#pragma unroll
      for (int k = 0; k < VEC; k += 2) {
        if constexpr (sizeof(T) != 4) ex.pair(pack2(x[k], x[k + 1]), minus_ref, x + k, x + k + 1);
        F2 e = pack2(x[k], x[k + 1]);
        if constexpr (sizeof(T) == 4) e = mul2(e, half_way);
        unpack2(mul2(e, by), x + k, x + k + 1);
      }
      const int cj = c + j * NT * VEC;
      if (aligned && ((u > 0 && u + 1 < ring.n_units) || (cj >= 0 && cj + VEC <= ring.vocab))) put_vector<O, VEC>(out + cj, x);
      else put_elements<O, VEC>(out, cj, ring.vocab, x);
    }
  }
}

// The lane's part of the sum of all warps' exponentials, relative to the largest of their references.
template <int WARPS>
__device__ __forceinline__ float join_stats(const RowStat* stat, int size, const ExpT& ex, float* m) {
  constexpr int EACH = (VR_MAX_CLUSTER * WARPS + 31) / 32;
  RowStat mine[EACH];
  float top = -INFINITY, s = 0.0f;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int w = i * 32 + (threadIdx.x & 31);
    mine[i] = w < size * WARPS ? stat[w] : RowStat{-INFINITY, 0.0f};
    top = max_nan(top, mine[i].m);
  }
  *m = warp_max_nan(top);
#pragma unroll
  for (int i = 0; i < EACH; ++i) s += mine[i].m > -INFINITY ? mine[i].s * ex(mine[i].m - *m) : 0.0f;
  return s;
}
__device__ __forceinline__ float2 warp_sum_f32x2(float a, float b) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  return make_float2(a, b);
}

template <class T, class O, int NT>
__global__ void __maxnreg__(NT == 256 ? 96 : 72)
softmax_rows_kernel(const T* z, size_t ld, size_t rows, int vocab, ExpT ex, O* prob, size_t prob_ld, int places, int* status) {
  constexpr int WARPS = NT / 32;
  extern __shared__ uint4 slots[];
  __shared__ RowBars b;
  __shared__ RowStat stats[4][VR_MAX_CLUSTER * WARPS];
  __shared__ float refs[2][NT];
  const int tid = threadIdx.x;
  UnitRing<T, NT, ROW_STEP> ring(slots, b.units, places, status, vocab);
  if (tid < 4) mbar_init(b.exchange + tid, 1);
  if (tid < 2) {
    mbar_init(b.summed + tid, WARPS);
    mbar_init(b.done + tid, WARPS);
  }
  mbar_fence_init();
  cluster_sync_all();  // nobody sends to a CTA that does not run yet
  const size_t row_step = gridDim.x / (unsigned)ring.size;
  if (tid < NT) {
    sum_rows<T, NT, sizeof(T) == 4>(ring, z, ld, rows, row_step, ex, b, refs, stats, ring.size * WARPS * sizeof(RowStat), false, false);
  } else if (tid < 2 * NT) {
    uint32_t i = 0;
    for (size_t r = cluster_id(); r < rows; r += row_step, ++i) {
      ring.begin(z + r * ld);
      row_wait_turn(b.exchange, i, 2, status);
      const RowStat* stat = stats[i & 3];
      float m;
      const float sum = warp_sum_f32(join_stats<WARPS>(stat, ring.size, ex, &m));
      // a row of -inf has no probabilities, one with a NaN or +inf no number for them
      const float f = m == -INFINITY ? 0.0f : m < INFINITY ? 1.0f / sum : NAN;
      row_wait_turn(b.summed, i, 1, status);
      write_row<true>(ring, prob + r * prob_ld, refs[i & 1][tid - NT], m, f, ex);
      __syncwarp();
      if ((tid & 31) == 0) mbar_arrive(b.done + (i & 1));
    }
  } else if (tid == 2 * NT) {
    ring.copy_rows(z, ld, rows, row_step);
  }
}

// What a CTA's list says of a row: the sum of its listed elements' exponentials, relative to the largest logit listed; what the teacher has
// left (-1: the list has no mass that the student could learn from); by what its probabilities are divided, inverted; the largest logit.
struct alignas(16) ListStat {
  double listed, by;  // (64 bits: what host lists call log-probabilities may be far from 0, all of them)
  float rest, top, listed32, spread;  // spread: by what the row's gradients are multiplied, beside the factor w / T
};
// Gradients are at most the larger of 1 and the teacher's listed mass, most of those over a large vocabulary a millionth of it: times 2^15 f16 holds
// the largest, and the small ones, which all have one sign outside of the list, do not round to 0 together.
__device__ __forceinline__ float spread_of(float mass) {
  return mass <= 1.0f ? 32768.0f : mass < INFINITY ? __uint_as_float((127 + 14 + 127 - (__float_as_uint(mass) >> 23)) << 23) : 1.0f;  // 2^(14 - exponent)
}
// a list of less mass than this has none
constexpr double LEAST_MASS = 1e-300;
// what a list leaves of a teacher's mass; a NaN stays
__device__ __forceinline__ double left_of(double mass) { return mass > 1.0 ? 0.0 : 1.0 - mass; }
struct alignas(16) LossStat {  // the teacher's mass, and sum q (t_j - z_j / T), the z relative to the largest
  double mass, cross;
};
// What a row's sums make of it: a gradient outside of the list is exp(z - reference) outside, one on it e listed - q by, e relative to the largest
// listed.  (Few instructions: run once a row between loops that do not leave them in the caches, each line of them is waited for.)
struct RowGradient {
  float reference, outside, listed;
  double by;
  bool idle;
};
template <int WARPS, bool SPREADS>
__device__ __forceinline__ RowGradient row_gradient(const RowStat* stat, const ListStat* list, int size, bool idle, float factor, const ExpT& ex) {
  RowGradient g;
  float mo;
  const int lane = threadIdx.x & 31;
  const float2 sums = warp_sum_f32x2(join_stats<WARPS>(stat, size, ex, &mo), lane < size ? list[lane].listed32 : 0.0f);
  const float so = sums.x, on = sums.y, top = list[0].top, rest = list[0].rest, m = max_nan(mo, top);
  // (exponentials outside may be 2^10 times their reference's, so that what makes them the row's is said down to subnormal numbers)
  const bool far = (mo - m) * ex.hi < -60.0f;
  const float half_way = ex(far ? 0.5f * (mo - m) : mo - m);
  const float rest_to = mo > -INFINITY ? (far ? half_way * half_way : half_way) : 0.0f, top_to = top > -INFINITY ? ex(top - m) : 0.0f;
  if (SPREADS) factor *= list[0].spread;
  const float scale = m < INFINITY ? factor : NAN, inv = scale / (so * rest_to + on * top_to);
  g.reference = mo;
  g.outside = so > 0.0f ? rest_to * inv - rest / so * scale : scale * 0.0f;
  g.listed = m > -INFINITY ? top_to * inv : scale * 0.0f;
  g.by = list[0].by * factor;
  g.idle = idle || rest < 0.0f;
  return g;
}

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

// One entry a thread of the list's warps.  64 bits for what is left of the teacher's mass, a difference, and for the loss, a small difference of
// large sums; for those alone, since exp, log and division take some 1000 cycles each there.
template <class T, class O, int NT>
__global__ void __maxnreg__(72)
distill_rows_kernel(const T* z, size_t ld, size_t rows, int vocab, float t, ExpT ex, const int* index, const float* teacher, int k, int tail,
                    const float* weight, float* loss, O* d, size_t d_ld, float* row_scale, int spread, int places, int* status) {
  using Ring = UnitRing<T, NT, ROW_STEP>;
  constexpr int WARPS = NT / 32, LIST_WARPS = RT_TOP_MAX / 32, VEC = Ring::VEC;
  constexpr bool SPREADS = std::is_same<T, float>::value && std::is_same<O, __half>::value;  // what the model driver asks for; elsewhere `spread` is off
  extern __shared__ uint4 slots[];
  __shared__ RowBars b;
  __shared__ RowStat stats[4][VR_MAX_CLUSTER * WARPS];
  __shared__ ListStat lists[4][VR_MAX_CLUSTER];
  __shared__ LossStat losses[4];
  __shared__ float refs[2][NT];
  __shared__ double s_e[2][RT_TOP_MAX], s_q[2][RT_TOP_MAX], s_sums[LIST_WARPS][3];
  __shared__ int s_mine[2][RT_TOP_MAX];  // the entry's column, if it is in this CTA's units and no entry before it has it, or -1
  __shared__ float s_top[LIST_WARPS];
  __shared__ int s_index[RT_TOP_MAX];
  const int tid = threadIdx.x, lane = tid & 31, list_warps = (k + 31) / 32;
  Ring ring(slots, b.units, places, status, vocab);
  const bool finds_loss = loss && ring.rank == 0;
  if (tid < 4) mbar_init(b.exchange + tid, 1);
  if (tid < 2) {
    mbar_init(b.summed + tid, WARPS);
    mbar_init(b.written + tid, WARPS);
    mbar_init(b.done + tid, 1);
    mbar_init(b.patched + tid, list_warps);
    mbar_init(b.listed + tid, list_warps);
  }
  mbar_fence_init();
  cluster_sync_all();  // nobody sends to a CTA that does not run yet
  const size_t row_step = gridDim.x / (unsigned)ring.size;
  const int writers = d ? NT : 0, copier = NT + writers, finisher = copier + 32, lister = finisher + 32;
  if (tid < NT) {
    const uint32_t bytes = ring.size * WARPS * sizeof(RowStat) + ring.size * sizeof(ListStat) + (finds_loss ? sizeof(LossStat) : 0);
    if (d) sum_rows<T, NT, sizeof(T) == 4>(ring, z, ld, rows, row_step, ex, b, refs, stats, bytes, true, false);
    else sum_rows<T, NT, false>(ring, z, ld, rows, row_step, ex, b, refs, stats, bytes, true, true);
  } else if (tid < copier) {  // writes
    uint32_t i = 0;
    for (size_t r = cluster_id(); r < rows; r += row_step, ++i) {
      const float w = weight ? weight[r] : 1.0f, factor = row_scale ? 1.0f : w / t;
      ring.begin(z + r * ld);
      row_wait_turn(b.exchange, i, 2, status);
      const RowGradient g = row_gradient<WARPS, SPREADS>(stats[i & 3], lists[i & 3], ring.size, w == 0.0f, factor, ex);
      row_wait_turn(b.summed, i, 1, status);
      // (rows that nothing is learnt from, whatever their logits are, have zeros)
      if (!g.idle) {
        write_row<false>(ring, d + r * d_ld, refs[i & 1][tid - NT], g.reference, g.outside, ex);
      } else {
        for (int u = 0; u < ring.n_units; ++u, ring.next()) {
          const float zero[VEC] = {};
          for (int j = 0; j < ROW_STEP; ++j) put_elements<O, VEC>(d + r * d_ld, ring.column(u, j), vocab, zero);
          ring.release();
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(b.written + (i & 1));
    }
  } else if (tid < finisher) {
    if (tid == copier) ring.copy_rows(z, ld, rows, row_step);
  } else if (tid < lister) {  // finds the loss, and writes the gradients on the list over what was written there
    const double inv_t = 1.0 / t;
    uint32_t i = 0;
    for (size_t r = cluster_id(); r < rows; r += row_step, ++i) {
      const float w = weight ? weight[r] : 1.0f;
      row_wait_turn(b.exchange, i, 2, status);
      const RowStat* stat = stats[i & 3];
      const ListStat* list = lists[i & 3];
      if (finds_loss) {
        const double mass = losses[i & 3].mass, cross = losses[i & 3].cross;
        const float top = list[0].top;
        float mo;
        double so = warp_sum_f64(join_stats<WARPS>(stat, ring.size, ex, &mo)), on = 0.0;
        for (int c = 0; c < ring.size; ++c) on += list[c].listed;
        const double rest = tail ? left_of(mass) : 0.0;
        // log(on + outside), the first relative to `top`, the second to mo, log(outside), log(rest) and log(mass): side by side
        const double x = ((double)mo - top) * inv_t;  // of the outside, in units of `top`
        const bool above = !(x <= 0.0) && mo > -INFINITY;
        const double shrink = above ? (top > -INFINITY ? exp(-x) : 0.0) : (mo > -INFINITY ? exp(x) : 0.0);
        const double log_of = log(lane == 0 ? (above ? so + on * shrink : on + so * shrink) : lane == 1 ? so : lane == 2 ? rest : mass);
        const double log_sum = __shfl_sync(0xffffffffu, log_of, 0), log_so = __shfl_sync(0xffffffffu, log_of, 1), log_rest = __shfl_sync(0xffffffffu, log_of, 2),
                     log_mass = __shfl_sync(0xffffffffu, log_of, 3);
        if (lane == 0) {
          double l = mass == 0.0 ? 0.0 : top > -INFINITY ? cross + mass * (log_sum + (above ? x : 0.0)) : INFINITY;
          if (!tail) l = l / mass - log_mass;
          if (rest > 0.0) l += so > 0.0 ? rest * (log_rest - log_so + log_sum - (above ? 0.0 : x)) : INFINITY;
          loss[r] = w == 0.0f || (!tail && mass < LEAST_MASS) ? 0.0f : !(max_nan(mo, top) < INFINITY) ? NAN : (float)(w * l);
        }
      }
      if (d) {
        if (row_scale && lane == 0 && ring.rank == 0) row_scale[r] = SPREADS ? w / t / list[0].spread : w / t;
        const RowGradient g = row_gradient<WARPS, SPREADS>(stat, list, ring.size, w == 0.0f, row_scale ? 1.0f : w / t, ex);
        row_wait_turn(b.listed, i, 1, status);
        row_wait_turn(b.written, i, 1, status);
        for (int j = lane; j < k; j += 32) {
          const int c = s_mine[i & 1][j];
          if (c >= 0 && !g.idle) d[r * d_ld + c] = from_f32<O>((float)(s_e[i & 1][j] * g.listed - s_q[i & 1][j] * g.by));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(b.done + (i & 1));
    }
  } else {  // makes the lists ready, a row ahead or two
    const int me = tid - lister, warp = me >> 5, threads = list_warps * 32;
    const double inv_t = 1.0 / t;
    auto list_sync = [&] { asm volatile("bar.sync 2, %0;" ::"r"(threads) : "memory"); };
    auto list_sync_or = [&](bool v) {
      uint32_t any;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.u32 p, %1, 0;\n\t"
          "bar.red.or.pred q, 2, %2, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(any)
          : "r"((uint32_t)v), "r"(threads)
          : "memory");
      return any != 0;
    };
    // The thread's entry: its index (-1: none), the teacher's log-probability, the student's logit.
    auto entry = [&](size_t r, float* tl) {
      *tl = me < k ? teacher[r * k + me] : 0.0f;
      return me < k ? index[r * k + me] : -1;
    };
    auto logit = [&](size_t r, int* i) {
      if (*i < -1 || *i >= vocab) {
        if (ring.rank == 0) report_status(status, RT_ERR_BAD_INDEX);
        *i = -1;
      }
      return *i >= 0 ? to_f32(z[r * ld + *i]) : -INFINITY;
    };
    size_t r = cluster_id();
    float tl;
    int my = entry(r, &tl);
    float z_my = logit(r, &my);
    for (uint32_t i = 0; r < rows; ++i) {
      const size_t next_r = r + row_step;
      float next_tl = 0.0f;
      const int next_entry = next_r < rows ? entry(next_r, &next_tl) : -1;
      if (i >= 2) row_wait_turn(b.exchange, i - 2, 2, status);  // not further ahead: the barriers tell two rows apart
      ring.begin(z + r * ld);
      auto place_of = [&](int u, uint32_t* phase) {
        const int n = ring.place + u;
        *phase = ring.phase ^ (n < ring.places ? 0u : 1u);
        return n < ring.places ? n : n - ring.places;
      };
      uint32_t phase;
      const float warp_top = warp_max_nan(z_my);
      if (lane == 0) s_top[warp] = warp_top;
      s_index[me] = my;
      for (int u = warp; u < ring.n_units; u += list_warps) {
        const int p = place_of(u, &phase);
        row_wait(ring.full + p, phase, status);
      }
      list_sync();
      float top = -INFINITY;  // the largest logit listed
      for (int j = 0; j < list_warps; ++j) top = max_nan(top, s_top[j]);
      // vectors that stick out of the row, and what is behind its last one
      if (ring.n_units > 0) {
        if (me == 0 && ring.rank == 0 && ring.align) ring.complete_vector(0, 0, ring.slots + place_of(0, &phase) * Ring::UNIT);
        const int u = ring.n_units - 1, at = ring.first_vector(u), end_whole = (ring.align + vocab) / VEC;
        uint4* const unit = ring.slots + place_of(u, &phase) * Ring::UNIT;
        for (int v = max(end_whole - at, 0) + me; v < Ring::UNIT; v += threads) ring.complete_vector(u, v, unit + v);
      }
      list_sync();
      bool first = false, again = false;
      if (my >= 0) {
        const int v = (my + ring.align) / VEC;
        const unsigned unit = v / Ring::UNIT, u = unit / (unsigned)ring.size;
        first = (int)(unit - u * ring.size) == ring.rank;
        if (first) again = take_out<T>(ring.slots + place_of((int)u, &phase) * Ring::UNIT, (v % Ring::UNIT) * VEC + (my + ring.align) % VEC);
      }
      again = list_sync_or(again);
      fence_proxy_async_smem();  // what was written in the units comes before the copies that follow
      __syncwarp();
      if (lane == 0) mbar_arrive(b.patched + (i & 1));
      int next_my = next_entry;
      const float next_z = next_r < rows ? logit(next_r, &next_my) : -INFINITY;
      // the list's sums
      const double x_my = z_my > -INFINITY ? (z_my == top ? 0.0 : ((double)z_my - top) * inv_t) : -INFINITY, lt = tl;
      double q = 0.0, e = 0.0;
      if (my >= 0) q = exp(lt), e = exp(x_my);
      if (i >= 2) row_wait_turn(b.done, i - 2, 1, status);
      s_e[i & 1][me] = e;
      s_q[i & 1][me] = q;
      if (again) {  // an index came twice: its first entry answers for all of them
        list_sync();
        double q_all = q;
        if (first) {
          q_all = 0.0;
          for (int j = 0; j < k; ++j)
            if (s_index[j] == my) {
              if (j < me) first = false;
              q_all += s_q[i & 1][j];
            }
        }
        list_sync();
        s_q[i & 1][me] = q_all;
      }
      s_mine[i & 1][me] = first ? my : -1;
      __syncwarp();
      if (lane == 0) mbar_arrive(b.listed + (i & 1));
      double mass = q, cross = q > 0.0 ? q * (lt - x_my) : q, on = first ? e : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        mass += __shfl_xor_sync(0xffffffffu, mass, o);
        cross += __shfl_xor_sync(0xffffffffu, cross, o);
        on += __shfl_xor_sync(0xffffffffu, on, o);
      }
      if (lane == 0) s_sums[warp][0] = mass, s_sums[warp][1] = cross, s_sums[warp][2] = on;
      list_sync();
      if (warp == 0) {
        mass = cross = on = 0.0;
        for (int j = 0; j < list_warps; ++j) mass += s_sums[j][0], cross += s_sums[j][1], on += s_sums[j][2];
        const float rest = tail ? (float)left_of(mass) : mass < LEAST_MASS ? -1.0f : 0.0f;
        const double by = tail ? 1.0 : 1.0 / mass;
        const float times = SPREADS && spread ? spread_of(tail ? (float)mass : 1.0f) : 1.0f;
        const uint64_t* bar = b.exchange + (i & 3);
        if (lane < ring.size) {
          const uint32_t to = mapa_u32(smem_u32(&lists[i & 3][ring.rank]), lane), its_bar = mapa_u32(smem_u32(bar), lane);
          send(to, its_bar, (uint32_t)__double2loint(on), (uint32_t)__double2hiint(on), (uint32_t)__double2loint(by), (uint32_t)__double2hiint(by));
          send(to + 16, its_bar, __float_as_uint(rest), __float_as_uint(top), __float_as_uint((float)on), __float_as_uint(times));
        }
        if (finds_loss && lane == 0)
          send(mapa_u32(smem_u32(&losses[i & 3]), 0), mapa_u32(smem_u32(bar), 0), (uint32_t)__double2loint(mass), (uint32_t)__double2hiint(mass),
               (uint32_t)__double2loint(cross), (uint32_t)__double2hiint(cross));
      }
      ring.place += ring.n_units;
      if (ring.place >= ring.places) ring.place -= ring.places, ring.phase ^= 1;
      r = next_r, my = next_my, tl = next_tl, z_my = next_z;
    }
  }
}

// How rows are held.  Threads that sum, and that write: few for short rows, of which an SM then holds several (registers admit four CTAs of 64
// threads, two of 128 or one of 256).  Distillation from 32 entries, by threads and the ring's KB:
//   4096 rows of 640 f32   64 x 32: 33 us, 128 x 66: 49, 256 x 208: 94
//   4096 of 2500 f32       64 x 32: 41, 128 x 66: 55, 256 x 208: 100
//   4096 of 8000 f32       128 x 66: 68, 256 x 208: 102       2048 of them: 64 x 32: 49, 128 x 66: 41
//   4096 of 16000 f32      128 x 66: 147, 256 x 208: 109
// The CTAs of a row's cluster: as few as hold two rows, one that is summed and one that is written (longer rows have eight and are held once, at
// least); with some more waits than now 1024 rows of 151936 f32 took 246 us with six CTAs, 272 with eight and 330 with four, 2048 of 128256 bf16
// 272 with three, 287 with two and 303 with four.  More where there are so few rows that SMs would be idle.  The ring's units: all that fit, as
// far as there are rows to fill them.
struct RowShape {
  int threads, cluster, places;
  size_t smem;
};
static RowShape row_shape(const rt_ctx* c, size_t rows, int vocab, int dtype) {
  const int vec = dtype == RT_DT_F32 ? 4 : 8, vectors = (vec - 1 + vocab + vec - 1) / vec;  // at the worst alignment
  const int threads = vectors <= 768 ? 64 : vectors <= 2048 ? 128 : 256, units = (vectors + ROW_STEP * threads - 1) / (ROW_STEP * threads);
  const size_t unit = (size_t)ROW_STEP * threads * 16, room = threads == 64 ? 32 * 1024 : threads == 128 ? 66 * 1024 : VR_MOST_SMEM;
  int size = 1;
  while (size * 2 <= VR_MAX_CLUSTER && units > size && rows * size * 2 <= (size_t)c->num_sms) size *= 2;
  auto each = [&] { return (size_t)((units + size - 1) / size); };
  while (size < VR_MAX_CLUSTER && 2 * each() * unit > room) ++size;
  const size_t turns = (rows * size + c->num_sms - 1) / c->num_sms, want = each() * std::min(turns, (size_t)4);
  const size_t places = std::max(each(), std::min(std::min(room / unit, (size_t)VR_MAX_UNITS), want));
  return {threads, size, (int)places, places * unit};
}
template <class F>
static int with_row_threads(int threads, F&& f) {
  if (threads == 64) return f(std::integral_constant<int, 64>());
  if (threads == 128) return f(std::integral_constant<int, 128>());
  return f(std::integral_constant<int, 256>());
}

int launch_softmax_rows(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, void* prob, int prob_dtype, size_t prob_ld) {
  const RowShape shape = row_shape(c, rows, vocab, z.dtype);
  return with_dtype(z.dtype, [&](auto* zt) {
    return with_dtype(prob_dtype, [&](auto* ot) {
      return with_row_threads(shape.threads, [&](auto threads) {
        using T = std::remove_pointer_t<decltype(zt)>;
        using O = std::remove_pointer_t<decltype(ot)>;
        return launch_clusters(c, softmax_rows_kernel<T, O, decltype(threads)::value>, true, rows, 2 * shape.threads + 32, shape.cluster, shape.smem,
                               (const T*)z.p, z.ld, rows, vocab, exp_t(temperature), (O*)prob, prob_ld, shape.places, c->status_dev);
      });
    });
  });
}

int launch_distill_rows(rt_ctx* c, const DistillArgs& a, size_t rows) {
  const RowShape shape = row_shape(c, rows, a.vocab, a.z.dtype);
  const int all_threads = (a.d ? 2 : 1) * shape.threads + 64 + (a.k + 31) / 32 * 32;
  return with_dtype(a.z.dtype, [&](auto* zt) {
    return with_dtype(a.d_dtype, [&](auto* ot) {
      return with_row_threads(shape.threads, [&](auto threads) {
        using T = std::remove_pointer_t<decltype(zt)>;
        using O = std::remove_pointer_t<decltype(ot)>;
        return launch_clusters(c, distill_rows_kernel<T, O, decltype(threads)::value>, true, rows, all_threads, shape.cluster, shape.smem, (const T*)a.z.p,
                               a.z.ld, rows, a.vocab, a.temperature, exp_t(a.temperature), a.index, a.teacher, a.k, a.mode == RT_DISTILL_TAIL, a.weight,
                               a.loss, (O*)a.d, a.d_ld, a.row_scale, a.spread, shape.places, c->status_dev);
      });
    });
  });
}

}  // namespace rt
