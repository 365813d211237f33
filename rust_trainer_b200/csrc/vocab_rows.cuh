// What the kernels over rows of logits share: element types, the temperature, the order of values.
#pragma once
#include "ctx.h"
#include "ptx.cuh"
#include "vocab_rows.h"
#include <algorithm>
#include <math.h>
#include <type_traits>

namespace rt {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// max that lets a NaN through
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Two floats in one register pair: one instruction adds or multiplies both.
using F2 = unsigned long long;
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(F2 v, float* a, float* b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(v)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// exp(d / T) for d <= 0 as 2^(d log2(e) / T), the factor in two terms: one rounded factor would be another temperature, by the same
// 2^-25 for every element, and a divergence is a small difference of large sums.  The first term is rounded towards 0, so that the
// second is positive and d = -inf gives 0.
struct ExpT {
  float hi, lo;
  __device__ __forceinline__ float operator()(float d) const { return ex2(fmaf(d, hi, d * lo)); }
  // two at once, of x - ref: minus_ref = (-ref, -ref)
  __device__ __forceinline__ void pair(F2 x, F2 minus_ref, float* a, float* b) const {
    const F2 d = add2(x, minus_ref);
    unpack2(fma2(d, pack2(hi, hi), mul2(d, pack2(lo, lo))), a, b);
    *a = ex2(*a);
    *b = ex2(*b);
  }
};
inline ExpT exp_t(float temperature) {
  const double c = 1.4426950408889634074 / (double)temperature;
  float hi = (float)c;
  if ((double)hi >= c) hi = nextafterf(hi, 0.0f);
  return {hi, (float)(c - (double)hi)};
}

// Integers in the order of the values: NaN above all, the two zeros alike.
__device__ __forceinline__ uint32_t order32(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 becomes +0
  if (v != v) return 0xffffffffu;
  return b ^ (uint32_t)(((int32_t)b >> 31) | 0x80000000);
}
__device__ __forceinline__ float order32_value(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);  // the highest one, a NaN's, is a NaN
}

// the elements of 16 bytes
template <class T>
__device__ __forceinline__ void unpack_vector(const uint4& u, float* x) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*(const __half2*)&w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}

// ---- rows on clusters
// A row is cut into vectors of 16 aligned bytes (the first and the last may stick out of it: what is outside reads as -inf), these into
// blocks of a vector a thread, and the blocks are dealt to the cluster's CTAs in turn, so that each sees a sample of the whole row
// wherever its large values lie.  A warp beside the NT threads that work brings the blocks as bulk copies into a ring in shared memory, all
// that find room there in flight at once; every element is read from memory once.  Clusters stay for as many rows as there are, and a
// block's place takes one of the next row as soon as the last warp is done with it.  What a row costs beside its bytes (barriers, sums
// that go round the cluster, lists: some microseconds a CTA) is paid by each of its CTAs, so that clusters are as small as can be:
// three CTAs hold 151936 f32 logits.
constexpr uint32_t VR_MOST_SMEM = 212 * 1024;  // dynamic shared memory of a CTA: what the kernels' fixed arrays, 13 KB at most, leave of 227
constexpr int VR_MAX_CLUSTER = 8, VR_MAX_BLOCKS = 64;  // blocks of a ring
constexpr int SITE_VOCAB_ROW = 701;

__device__ __forceinline__ size_t cluster_id() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// 8 or 16 bytes into another CTA's shared memory, counted by a barrier there
__device__ __forceinline__ void send(uint32_t to, uint32_t bar, uint32_t a, uint32_t b) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(to), "r"(a), "r"(b), "r"(bar) : "memory");
}
__device__ __forceinline__ void send(uint32_t to, uint32_t bar, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to), "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void send(uint32_t to, uint32_t bar, double v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(to), "l"(__double_as_longlong(v)), "r"(bar) : "memory");
}
// barriers of the NT threads that work
template <int NT>
__device__ __forceinline__ void work_sync() { asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory"); }
template <int NT>
__device__ __forceinline__ bool work_sync_or(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "n"(NT)
      : "memory");
  return r != 0;
}
// Waits for a phase of a barrier, asleep for up to some microseconds at a time: a warp that polls takes instructions from those that work.
// The matmul's wait gives up when another kernel has reported anything; here an index out of range in one row must not end the
// others' waits, so that only the time limit does.
__device__ __forceinline__ uint32_t mbar_sleep(uint64_t* bar, uint32_t phase) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(phase), "r"(20000u)
      : "memory");
  return ok;
}
static __device__ __noinline__ void row_wait_slow(uint64_t* bar, uint32_t phase, int* status) {
  const long long t0 = clock64();
  while (!mbar_sleep(bar, phase)) {
    if (clock64() - t0 > MBAR_WAIT_LIMIT_CYCLES) {
      report_status(status, SITE_VOCAB_ROW);
      return;
    }
  }
}
__device__ __forceinline__ void row_wait(uint64_t* bar, uint32_t phase, int* status) {
  if (!mbar_sleep(bar, phase)) row_wait_slow(bar, phase, status);
}

// Where a row's elements are: its vectors, and the blocks of them that are this CTA's.
template <class T, int NT>
struct RowPart {
  static constexpr int VEC = 16 / (int)sizeof(T);   // elements of a vector
  static constexpr int STEP = 16 / VEC;             // blocks that give a thread 16 elements
  static constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -inf
  const T* row;
  int vocab, rank, size, phase, n_vec, n_it;  // n_it: this CTA's blocks

  __device__ __forceinline__ RowPart(const T* row_, int vocab_, int rank_, int size_) : row(row_), vocab(vocab_), rank(rank_), size(size_) {
    phase = (int)(((uintptr_t)row & 15) / sizeof(T));
    n_vec = (phase + vocab + VEC - 1) / VEC;
    n_it = (int)((unsigned)((n_vec + NT - 1) / NT - rank + size - 1) / (unsigned)size);
  }
  __device__ __forceinline__ int first_vector(int it) const { return (it * size + rank) * NT; }
  // the column of the first element of the thread's vector
  __device__ __forceinline__ int column(int it) const { return (first_vector(it) + (int)threadIdx.x) * VEC - phase; }
  // where column `c` lies: its CTA, its block there, and its place among the block's elements
  __device__ __forceinline__ int owner(int c, int* it, int* element) const {
    const int v = (c + phase) / VEC;
    const unsigned block = v / NT;
    *it = (int)(block / (unsigned)size);
    *element = (v % NT) * VEC + (c + phase) % VEC;
    return (int)(block - (unsigned)*it * size);
  }
  // whether the thread's vector of a block may not be whole: only the row's first and last vectors stick out
  __device__ __forceinline__ bool outer(int it) const { return it == 0 || it + 1 == n_it; }
  static __device__ __forceinline__ void unpack(const uint4& u, float* x) { unpack_vector<T>(u, x); }
};

// A vector's results: as a whole, where they lie on 16 bytes (8 where they are no longer), or what there is of them in a row of `vocab`.
template <class O, int VEC>
__device__ __forceinline__ void put_vector(O* to, const float* x) {
  uint32_t w[VEC * sizeof(O) / 4];
  if constexpr (sizeof(O) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      if constexpr (std::is_same<O, __half>::value) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *(const uint32_t*)&h;
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *(const uint32_t*)&h;
      }
    }
  }
  if constexpr (VEC * sizeof(O) == 8) {
    __stcs((uint2*)to, make_uint2(w[0], w[1]));
  } else {
#pragma unroll
    for (int i = 0; i < (int)(VEC * sizeof(O) / 16); ++i) __stcs((uint4*)to + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
  }
}
template <class O, int VEC>
__device__ __forceinline__ void put_elements(O* out, int c, int vocab, const float* x) {
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (c + i >= 0 && c + i < vocab) out[c + i] = from_f32<O>(x[i]);
}

// Values that go round the cluster: everybody sends to everybody, and waits until all of it has come.  Two barriers in turn (and two places for
// the values), so that what a faster CTA sends next is not counted with this: nobody is two exchanges ahead of another.
struct Exchange {
  uint64_t* bars;  // [2]
  int* status;
  uint32_t n = 0;
  __device__ __forceinline__ int turn() const { return n & 1; }
  __device__ __forceinline__ uint32_t bar(uint32_t rank) const { return mapa_u32(smem_u32(bars + turn()), rank); }
  // what is to come, by one thread of the CTA (before or after it comes)
  __device__ __forceinline__ void expect(uint32_t bytes) const { mbar_expect_tx(bars + turn(), bytes); }
  __device__ __forceinline__ void wait() {
    row_wait(bars + turn(), n >> 1 & 1, status);
    ++n;
  }
};

// A CTA's ring of blocks.  Blocks are numbered over all rows of the CTA: number n is in place n % places; `full` completes a phase with each
// copy, `empty` with the last warp that is done with it.
template <class T, int NT>
struct Ring {
  using Part = RowPart<T, NT>;
  static constexpr int VEC = Part::VEC;
  uint4* slots;           // [places][NT]
  uint64_t *full, *empty;  // [places]
  int* status;
  int places, vocab, rank, size;
  int first_it, first_place;  // the oldest block that is still needed of the row that is worked on, and its place
  uint32_t first_phase;
  const T* z;
  size_t ld, rows, row_step;

  // By all threads of the CTA, the warp that copies among them; it sets up the barriers of `exchange` too.
  __device__ __forceinline__ Ring(uint4* slots_, uint64_t* bars, int places_, int* status_, const T* z_, size_t ld_, size_t rows_, int vocab_, Exchange& exchange)
      : slots(slots_), full(bars), empty(bars + VR_MAX_BLOCKS), status(status_), places(places_), vocab(vocab_), rank((int)cluster_ctarank()),
        size((int)cluster_size()), first_it(0), first_place(0), first_phase(0), z(z_), ld(ld_), rows(rows_) {
    row_step = gridDim.x / (unsigned)size;
    exchange.bars = bars + 2 * VR_MAX_BLOCKS;
    exchange.status = status;
    for (int i = threadIdx.x; i < places; i += NT) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, NT / 32);
    }
    if (threadIdx.x < 2) mbar_init(exchange.bars + threadIdx.x, 1);
    mbar_fence_init();
    fence_proxy_async_smem();
    cluster_sync_all();  // nobody sends to a CTA that does not run yet
  }
  __device__ __forceinline__ Part part(size_t r) const { return Part(z + r * ld, vocab, rank, size); }
  // The copies of all rows, in one thread of the warp that does nothing else.
  __device__ __forceinline__ void copy_rows() const {
    int place = 0;
    uint32_t phase = 1;  // of `empty`: at first every place is
    for (size_t r = cluster_id(); r < rows; r += row_step) {
      const Part p = part(r);
      const int first_whole = p.phase ? 1 : 0, end_whole = (p.phase + vocab) / VEC;  // vectors that lie in the row
      for (int it = 0; it < p.n_it; ++it) {
        const int first = p.first_vector(it), v0 = max(first, first_whole), v1 = min(first + NT, end_whole);
        const uint32_t bytes = v1 > v0 ? (uint32_t)(v1 - v0) * 16 : 0;
        row_wait(empty + place, phase, status);
        mbar_expect_tx(full + place, bytes);
        if (bytes) bulk_load_1d(slots + place * NT + (v0 - first), p.row + (v0 * VEC - p.phase), bytes, full + place);
        if (++place == places) place = 0, phase ^= 1;
      }
    }
  }
  // n blocks of the row are done with, and perhaps the row is
  __device__ __forceinline__ void advance(int n, bool next_row_begins) {
    first_it = next_row_begins ? 0 : first_it + n;
    first_place += n;
    if (first_place >= places) first_place -= places, first_phase ^= 1;
  }
  __device__ __forceinline__ int place(int it) const {
    const int n = first_place + it - first_it;
    return n < places ? n : n - places;
  }
  __device__ __forceinline__ uint4* block(int it) const { return slots + place(it) * NT; }
  __device__ __forceinline__ void wait(int it) const {
    const int n = first_place + it - first_it;
    row_wait(full + (n < places ? n : n - places), first_phase ^ (n < places ? 0u : 1u), status);
  }
  // The warp is done with n blocks that lie side by side, and what it wrote there comes before the copies that follow (the writers' fence).
  __device__ __forceinline__ void release(const uint4* first, int n) const {
    __syncwarp();
    const int lane = threadIdx.x & 31;
    if (lane < n) mbar_arrive(empty + (int)(first - slots) / NT + lane);
  }
  // The warp is done with the row.
  __device__ __forceinline__ void release_all(const Part& p) const {
    __syncwarp();
    for (int it = threadIdx.x & 31; it < p.n_it; it += 32) mbar_arrive(empty + place(it));
  }
  // What no copy brings of a block: vectors that stick out of the row, element by element, and -inf behind the row's last one, by the
  // threads that they belong to.
  __device__ __forceinline__ void complete(const Part& p, int it) const {
    const int v = p.first_vector(it) + (int)threadIdx.x, c = v * VEC - p.phase;
    if (c >= 0 && c + VEC <= vocab) return;
    uint4* slot = block(it) + threadIdx.x;
    if (v >= p.n_vec) {
      *slot = make_uint4(Part::NONE, Part::NONE, Part::NONE, Part::NONE);
    } else {
      alignas(16) T e[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = c + i >= 0 && c + i < vocab ? p.row[c + i] : from_f32<T>(-INFINITY);
      *slot = *(const uint4*)e;
    }
  }
  // The whole row is there, for every thread behind the next barrier of the CTA: each warp waits for a few blocks.
  __device__ __forceinline__ void wait_all(const Part& p) const {
    for (int it = threadIdx.x / 32; it < p.n_it; it += NT / 32) wait(it);
    if (p.n_it > 0) complete(p, 0);
    if (p.n_it > 1) complete(p, p.n_it - 1);
  }
  // f(block, blocks, where the thread's vector of the first lies) for the one or two runs of places that hold the row.
  template <class F>
  __device__ __forceinline__ void runs(const Part& p, F&& f) const {
    const int n = min(p.n_it, places - first_place);
    f(0, n, slots + first_place * NT + threadIdx.x);
    if (n < p.n_it) f(n, p.n_it - n, slots + threadIdx.x);
  }
  static constexpr int GROUP = 4;
  // The thread's reference for exponentials, one of its elements or -inf, and the sum of its exponentials relative to it.  The reference
  // is the largest of the first vectors: an exponential may be as large as 2^60 before it changes, so that it rarely does.  KEEP
  // (32-bit rows): the exponentials take their elements' place.
  template <bool KEEP>
  __device__ __forceinline__ float exponentials(const Part& p, const ExpT& ex, float* reference) const {
    float ref = -INFINITY;
    const float most = 60.0f / ex.hi;
    F2 acc[4] = {0, 0, 0, 0};
    auto work = [&](int it, uint4* at, auto count) {
      constexpr int N = decltype(count)::value;
      uint4 v[N];
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = at[j * NT];
      float top;
      if constexpr (sizeof(T) == 4) {
        top = max_nan(__uint_as_float(v[0].x), __uint_as_float(v[0].y), max_nan(__uint_as_float(v[0].z), __uint_as_float(v[0].w)));
#pragma unroll
        for (int j = 1; j < N; ++j) top = max_nan(max_nan(top, __uint_as_float(v[j].x), __uint_as_float(v[j].y)), __uint_as_float(v[j].z), __uint_as_float(v[j].w));
      } else {
        using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
        T2 m = __hmax2_nan(__hmax2_nan(*(const T2*)&v[0].x, *(const T2*)&v[0].y), __hmax2_nan(*(const T2*)&v[0].z, *(const T2*)&v[0].w));
#pragma unroll
        for (int j = 1; j < N; ++j)
          m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(*(const T2*)&v[j].x, *(const T2*)&v[j].y), __hmax2_nan(*(const T2*)&v[j].z, *(const T2*)&v[j].w)));
        top = max_nan(to_f32(m.x), to_f32(m.y));
      }
      if (!(top <= ref + most) && ref == ref) {  // the first finite ones, ones that are far larger, a NaN, which stays
        if (ref > -INFINITY) {
          const float by = ex(ref - top);
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[j] = mul2(acc[j], pack2(by, by));
          if constexpr (KEEP) {
#pragma unroll 1
            for (int i = 0; i < it; ++i) {
              float4* e = (float4*)(block(i) + threadIdx.x);
              *e = make_float4(e->x * by, e->y * by, e->z * by, e->w * by);
            }
          }
        }
        ref = top;
      }
      const float r = ref > -INFINITY ? ref : 0.0f;
      const F2 minus_ref = pack2(-r, -r);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float x[VEC];
        Part::unpack(v[j], x);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          ex.pair(pack2(x[i], x[i + 1]), minus_ref, x + i, x + i + 1);
          acc[(j * VEC + i) / 2 & 3] = add2(acc[(j * VEC + i) / 2 & 3], pack2(x[i], x[i + 1]));
        }
        if constexpr (KEEP) at[j * NT] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
      }
    };
    runs(p, [&](int it, int n, uint4* at) {
#pragma unroll 1
      for (; n >= GROUP; n -= GROUP, it += GROUP, at += GROUP * NT) work(it, at, std::integral_constant<int, GROUP>());
#pragma unroll 1
      for (; n > 0; --n, ++it, at += NT) work(it, at, std::integral_constant<int, 1>());
    });
    *reference = ref;
    float a, b;
    unpack2(add2(add2(acc[0], acc[1]), add2(acc[2], acc[3])), &a, &b);
    return a + b;
  }
  // What f(vector, its VEC results) makes of every vector of the thread goes into the row `out`, and the blocks are released on the way.
  template <class O, class F>
  __device__ __forceinline__ void put(const Part& p, O* out, F&& f) {
    const bool aligned = ((uintptr_t)out - (uintptr_t)p.phase * sizeof(O)) % (VEC * sizeof(O) < 16 ? VEC * sizeof(O) : 16) == 0;
    const int stride = p.size * NT * VEC;  // columns from block to block
    runs(p, [&](int it, int n, const uint4* at) {
#pragma unroll 1
      for (int end = it + n; it < end; it += GROUP, at += GROUP * NT) {
        const int c = p.column(it), left = min(GROUP, end - it);
        if (aligned && left == GROUP && it > 0 && it + GROUP < p.n_it) {
          uint4 v[GROUP];
          O* to = out + c;
#pragma unroll
          for (int j = 0; j < GROUP; ++j) v[j] = at[j * NT];
#pragma unroll
          for (int j = 0; j < GROUP; ++j, to += stride) {
            float x[VEC];
            f(v[j], x);
            put_vector<O, VEC>(to, x);
          }
        } else {
#pragma unroll 1
          for (int j = 0; j < left; ++j) {
            float x[VEC];
            f(at[j * NT], x);
            const int cj = c + j * stride;
            if (aligned && cj >= 0 && cj + VEC <= vocab) put_vector<O, VEC>(out + cj, x);
            else put_elements<O, VEC>(out, cj, vocab, x);
          }
        }
        release(at, left);
      }
    });
  }
  // The results e f, e the exponentials relative to the row's reference (-inf: all are 0); `mine` is the thread's.
  template <class O>
  __device__ __forceinline__ void put_exponentials(const Part& p, O* out, float mine, float reference, float f, const ExpT& ex) {
    if constexpr (sizeof(T) == 4) {  // they are there, relative to the thread's
      const float by = mine > -INFINITY ? ex(mine - reference) * f : f;
      put(p, out, [&](const uint4& v, float* x) {
        Part::unpack(v, x);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) unpack2(mul2(pack2(x[i], x[i + 1]), pack2(by, by)), x + i, x + i + 1);
      });
    } else {
      const float ref = reference > -INFINITY ? reference : 0.0f;
      const F2 minus_ref = pack2(-ref, -ref), by = pack2(f, f);
      put(p, out, [&](const uint4& v, float* x) {
        Part::unpack(v, x);
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          ex.pair(pack2(x[i], x[i + 1]), minus_ref, x + i, x + i + 1);
          unpack2(mul2(pack2(x[i], x[i + 1]), by), x + i, x + i + 1);
        }
      });
    }
  }
};

// The warp's sum of its threads' exponentials, relative to the largest of their references.  In 32 bits: five roundings, which differ from
// warp to warp.
__device__ __forceinline__ float warp_join(float m, float s, const ExpT& ex, float* warp_m) {
  *warp_m = warp_max_nan(m);
  s = m > -INFINITY ? s * ex(m - *warp_m) : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
__device__ __forceinline__ float warp_sum_f32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The row's sum from n warps' references and sums (none: -inf, 0), as get(i, &m, &s) gives them: the lane's part of it, relative to *m.
template <class F>
__device__ __forceinline__ double lane_join(int n, F&& get, const ExpT& ex, float* m) {
  float mi[4], si[4], top = -INFINITY;  // at most 128 warps
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mi[i] = -INFINITY;
    si[i] = 0.0f;
    if (i * 32 + lane < n) get(i * 32 + lane, mi + i, si + i);
    top = max_nan(top, mi[i]);
  }
  *m = warp_max_nan(top);
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i * 32 < n && mi[i] > -INFINITY) s += (double)(si[i] * ex(mi[i] - *m));
  return s;
}

// How rows are held.  Threads that work: 256 where two CTAs with a row (or its part) each find room on an SM, else 512.  The CTAs of a row's
// cluster: as few as have room for it, more where there are so few rows that SMs would be idle.  The ring's blocks: all that fit
// beside `other` bytes, as far as there are rows to fill them.
struct RowShape {
  int threads, cluster, places;
  size_t smem;
};
inline RowShape row_shape(const rt_ctx* c, size_t rows, int vocab, int dtype, size_t other) {
  const int vec = dtype == RT_DT_F32 ? 4 : 8, vectors = (vec - 1 + vocab + vec - 1) / vec;  // at the worst alignment
  const size_t third = 68 * 1024, half = 104 * 1024, all = VR_MOST_SMEM;
  int size = 1;
  while (size * 2 <= VR_MAX_CLUSTER && vectors > 512 * size && rows * size * 2 <= (size_t)c->num_sms) size *= 2;
  auto need = [&](int threads) { return (size_t)(((vectors + threads - 1) / threads + size - 1) / size) * threads * 16 + other; };
  while (size < VR_MAX_CLUSTER && need(512) > all) ++size;
  const int threads = need(256) <= half ? 256 : 512;
  const size_t block = (size_t)threads * 16, room = need(threads) <= third ? third : need(threads) <= half ? half : all;
  const size_t turns = (rows * size + c->num_sms - 1) / c->num_sms, each = (need(threads) - other) / block;
  const size_t places = std::max(each, std::min(std::min((room - other) / block, (size_t)VR_MAX_BLOCKS), each * std::min(turns, (size_t)4)));
  return {threads, size, (int)places, places * block + other};
}
// Calls f with the number of threads that work as a constant.
template <class F>
inline int with_threads(int threads, F&& f) {
  if (threads == 256) return f(std::integral_constant<int, 256>());
  return f(std::integral_constant<int, 512>());
}
// CTAs that have to find room on an SM
constexpr int ctas_of(int threads) { return threads == 256 ? 3 : 1; }

// Clusters of `size` CTAs for `rows` rows: one each, or (`stay`) as many as run at once, which take the rows in turn, in equal shares.
template <class... KArgs, class... A>
inline int launch_clusters(rt_ctx* c, void (*kernel)(KArgs...), bool stay, size_t rows, int threads, int size, size_t smem, A&&... args) {
  if (!c->raise_smem(kernel, VR_MOST_SMEM)) return 3;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * size));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = c->stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)size;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (stay) {
    int& most = c->clusters_at_once[std::make_tuple((const void*)kernel, size, smem)];
    if (most == 0 && (cudaOccupancyMaxActiveClusters(&most, kernel, &cfg) != cudaSuccess || most < 1)) return 3;
    const size_t turns = (rows + most - 1) / most;
    cfg.gridDim = dim3((unsigned)((rows + turns - 1) / turns * size));
  }
  RT_COUNT_LAUNCH(1);
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(std::forward<A>(args))...) == cudaSuccess ? 0 : 3;
}

// Calls f with a null pointer of the element type that `dtype` names.
template <class F>
inline int with_dtype(int dtype, F&& f) {
  if (dtype == RT_DT_F32) return f((float*)nullptr);
  if (dtype == RT_DT_BF16) return f((__nv_bfloat16*)nullptr);
  return f((__half*)nullptr);
}

}  // namespace rt
