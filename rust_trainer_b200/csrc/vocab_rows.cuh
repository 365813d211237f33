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
// units of a few vectors a thread, and the units are dealt to the cluster's CTAs in turn, so that each sees a sample of the whole row
// wherever its large values lie.  A warp that does nothing else brings the units as bulk copies into a ring in shared memory, all that
// find room there in flight at once; every element is read from memory once.  Clusters stay for as many rows as there are, and a
// unit's place takes one of the next row as soon as the last warp is done with it.
constexpr uint32_t VR_MOST_SMEM = 208 * 1024;  // dynamic shared memory of a CTA: what the kernels' fixed arrays, 19 KB at most, leave of 227
constexpr int VR_MAX_CLUSTER = 8, VR_MAX_UNITS = 64;  // units of a ring
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
// barriers of some of a CTA's warps
template <int NT>
__device__ __forceinline__ void work_sync() { asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory"); }

// of how many of the threads `v` is true
template <int NT>
__device__ __forceinline__ int work_count(bool v) {
  int n;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.popc.u32 %0, 1, %2, p;\n\t}"
      : "=r"(n)
      : "r"((uint32_t)v), "n"(NT)
      : "memory");
  return n;
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
  __device__ __forceinline__ void begin(uint64_t* bars_, int* status_) {
    bars = bars_;
    status = status_;
    if (threadIdx.x < 2) mbar_init(bars + threadIdx.x, 1);
    mbar_fence_init();
  }
  __device__ __forceinline__ int turn() const { return n & 1; }
  __device__ __forceinline__ uint32_t bar(uint32_t rank) const { return mapa_u32(smem_u32(bars + turn()), rank); }
  // what is to come, by one thread of the CTA (before or after it comes)
  __device__ __forceinline__ void expect(uint32_t bytes) const { mbar_expect_tx(bars + turn(), bytes); }
  __device__ __forceinline__ void wait() {
    row_wait(bars + turn(), n >> 1 & 1, status);
    ++n;
  }
};

// A CTA's ring of units of STEP vectors of NT threads, and where one of its users is in it.  Units are numbered over all rows of the CTA: number
// n is in place n % places; `full` completes a phase with each copy, `empty` with the last of the NT / 32 warps that give it back.
template <class T, int NT, int STEP>
struct UnitRing {
  static constexpr int VEC = 16 / (int)sizeof(T), UNIT = STEP * NT;  // elements of a vector; vectors of a unit
  static constexpr uint32_t NONE = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -inf
  uint4* slots;            // [places][UNIT]
  uint64_t *full, *empty;  // [places]
  int* status;
  int places, vocab, rank, size;
  int place = 0;  // of the unit that comes next, and its phase
  uint32_t phase = 0;
  // of the row that is worked on: this CTA's units
  const T* row;
  int align, n_vec, n_units;

  // The barriers are set up by all threads of the CTA, which then meet.
  __device__ __forceinline__ UnitRing(uint4* slots_, uint64_t* bars, int places_, int* status_, int vocab_)
      : slots(slots_), full(bars), empty(bars + VR_MAX_UNITS), status(status_), places(places_), vocab(vocab_), rank((int)cluster_ctarank()),
        size((int)cluster_size()) {
    for (int i = threadIdx.x; i < places; i += NT) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, NT / 32);
    }
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  __device__ __forceinline__ void begin(const T* row_) {
    row = row_;
    align = (int)(((uintptr_t)row & 15) / sizeof(T));
    n_vec = (align + vocab + VEC - 1) / VEC;
    const int units = (n_vec + UNIT - 1) / UNIT;
    n_units = (int)((unsigned)(units - rank + size - 1) / (unsigned)size);
  }
  __device__ __forceinline__ int first_vector(int u) const { return (u * size + rank) * UNIT; }
  // the column of the first element of vector `i` of a unit
  __device__ __forceinline__ int column_of(int u, int i) const { return (first_vector(u) + i) * VEC - align; }
  __device__ __forceinline__ void next() {
    if (++place == places) place = 0, phase ^= 1;
  }
  __device__ __forceinline__ uint4* unit() const { return slots + place * UNIT; }
  __device__ __forceinline__ void wait() const { row_wait(full + place, phase, status); }
  // the warp gives the unit back; what it wrote there comes before the copies that follow by the writers' fence
  __device__ __forceinline__ void release() const {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(empty + place);
  }
  __device__ __forceinline__ void copy_rows(const T* z, size_t ld, size_t rows, size_t row_step) {
    for (size_t r = cluster_id(); r < rows; r += row_step) {
      begin(z + r * ld);
      for (int u = 0; u < n_units; ++u, next()) {
        const int first = first_vector(u), v0 = max(first, align ? 1 : 0), v1 = min(first + UNIT, (align + vocab) / VEC);  // vectors that lie in the row
        const uint32_t bytes = v1 > v0 ? (uint32_t)(v1 - v0) * 16 : 0;
        row_wait(empty + place, phase ^ 1, status);
        mbar_expect_tx(full + place, bytes);
        if (bytes) bulk_load_1d(unit() + (v0 - first), row + (v0 * VEC - align), bytes, full + place);
      }
    }
  }
  // What no copy brings of the vector `i` of a unit: one that sticks out of the row, element by element, and -inf behind the row's last one.
  __device__ __forceinline__ void complete_vector(int u, int i, uint4* slot) const {
    const int c = column_of(u, i);
    if (c >= 0 && c + VEC <= vocab) return;
    if (c >= vocab) {
      *slot = make_uint4(NONE, NONE, NONE, NONE);
    } else {
      alignas(16) T e[VEC];
#pragma unroll
      for (int k = 0; k < VEC; ++k) e[k] = c + k >= 0 && c + k < vocab ? row[c + k] : from_f32<T>(-INFINITY);
      *slot = *(const uint4*)e;
    }
  }
  // the thread's vectors of a unit, the first of which is at `at`
  __device__ __forceinline__ void complete(int u, uint4* at) const {
#pragma unroll 1
    for (int j = 0; j < STEP; ++j) complete_vector(u, j * NT + (int)threadIdx.x % NT, at + j * NT);
  }
  // the column of the first element of the thread's j-th vector of a unit
  __device__ __forceinline__ int column(int u, int j) const { return column_of(u, j * NT + (int)threadIdx.x % NT); }
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
    int& most = c->clusters_at_once[std::make_tuple((const void*)kernel, size * 1024 + threads, smem)];
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
