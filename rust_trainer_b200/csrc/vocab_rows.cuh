// What the kernels over rows of logits share: element types, the temperature, the order of values.
#pragma once
#include "ctx.h"
#include "ptx.cuh"
#include "vocab_rows.h"
#include <math.h>

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

// exp(d / T) for d <= 0 as 2^(d log2(e) / T), the factor in two terms: one rounded factor would be another temperature, by the same
// 2^-25 for every element, and a divergence is a small difference of large sums.  The first term is rounded towards 0, so that the
// second is positive and d = -inf gives 0.
struct ExpT {
  float hi, lo;
  __device__ __forceinline__ float operator()(float d) const {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(fmaf(d, hi, d * lo)));
    return r;
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

// ---- a row in the shared memory of a cluster
// A row is cut into vectors of 16 aligned bytes (the first and the last may stick out of it: what is outside reads as -inf), these into
// blocks of VR_THREADS, and the blocks are dealt to the cluster's CTAs in turn, so that each sees a sample of the whole row
// wherever its large values lie.  A CTA's blocks are bulk copies, all of them in flight at once; those of a step, 16 elements a
// thread, complete one barrier.
constexpr uint32_t VR_MOST_SMEM = 214 * 1024;  // dynamic shared memory: RT_VOCAB_MAX elements of 32 bits on eight CTAs, and what is beside them
constexpr int VR_THREADS = 256, VR_WARPS = VR_THREADS / 32, VR_MAX_CLUSTER = 8;
constexpr int VR_MAX_STEPS = 16;  // 13 are the most: RT_VOCAB_MAX elements, 16 a thread and step
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
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
// The matmul's wait gives up when another kernel has reported anything; here an index out of range in one row must not end the
// others' waits, so that only the time limit does.
static __device__ __noinline__ void row_wait_slow(uint64_t* bar, int* status) {
  const long long t0 = clock64();
  for (;;) {
    for (int i = 0; i < 256; ++i)
      if (mbar_try_wait(bar, 0)) return;
    if (clock64() - t0 > MBAR_WAIT_LIMIT_CYCLES) {
      report_status(status, SITE_VOCAB_ROW);
      return;
    }
  }
}

template <class T>
struct RowPart {
  static constexpr int VEC = 16 / (int)sizeof(T);   // elements of a vector
  static constexpr int STEP = 16 / VEC;             // vectors of a thread taken at once: 16 elements
  const T* row;
  int phase, vocab, rank, size, n_vec, n_it, n_steps;  // n_it: vectors per thread of this CTA at most
  uint4* slots;                                        // [n_it][VR_THREADS]
  uint64_t* bars;                                      // [VR_MAX_STEPS]
  int* status;

  __device__ __forceinline__ RowPart(const T* row_, int vocab_, uint4* slots_, uint64_t* bars_, int* status_)
      : row(row_), vocab(vocab_), rank((int)cluster_ctarank()), size((int)cluster_size()), slots(slots_), bars(bars_), status(status_) {
    phase = (int)(((uintptr_t)row & 15) / sizeof(T));
    n_vec = (phase + vocab + VEC - 1) / VEC;
    const int blocks = (n_vec + VR_THREADS - 1) / VR_THREADS;
    n_it = blocks > rank ? (blocks - rank - 1) / size + 1 : 0;
    n_steps = (n_it + STEP - 1) / STEP;
  }
  // slots per thread of the cluster's first CTA, which has most: where what lies behind them starts in every CTA
  __device__ __forceinline__ int n_it_most() const { return ((n_vec + VR_THREADS - 1) / VR_THREADS + size - 1) / size; }
  __device__ __forceinline__ int first_vector(int it) const { return (it * size + rank) * VR_THREADS; }
  // the column of a slot's first element
  __device__ __forceinline__ int column(int it, int thread) const { return (first_vector(it) + thread) * VEC - phase; }
  // where column `c` lies: its CTA, and the index of its vector's slot there
  __device__ __forceinline__ int owner(int c, int* slot, int* elem) const {
    const int v = (c + phase) / VEC, block = v / VR_THREADS;
    *slot = block / size * VR_THREADS + v % VR_THREADS;
    *elem = (c + phase) % VEC;
    return block % size;
  }
  // Starts the copies; a __syncthreads() has to follow before the first get().
  __device__ __forceinline__ void load() const {
    const int tid = threadIdx.x;
    if (tid < 32) {
      if (tid < n_steps) mbar_init(bars + tid, 1);
      mbar_fence_init();
      fence_proxy_async_smem();
      __syncwarp();
      const int first_whole = phase ? 1 : 0, end_whole = (phase + vocab) / VEC;  // vectors that lie in the row
      if (tid < n_steps) {
        uint32_t bytes = 0;
#pragma unroll
        for (int j = 0; j < STEP; ++j) {
          const int it = tid * STEP + j, v0 = max(first_vector(it), first_whole), v1 = min(first_vector(it) + VR_THREADS, end_whole);
          if (it < n_it && v1 > v0) bytes += (uint32_t)(v1 - v0) * 16;
        }
        mbar_expect_tx(bars + tid, bytes);
#pragma unroll
        for (int j = 0; j < STEP; ++j) {
          const int it = tid * STEP + j, v0 = max(first_vector(it), first_whole), v1 = min(first_vector(it) + VR_THREADS, end_whole);
          if (it < n_it && v1 > v0)
            bulk_load_1d(slots + it * VR_THREADS + (v0 - first_vector(it)), row + (v0 * VEC - phase), (uint32_t)(v1 - v0) * 16, bars + tid);
        }
      }
    } else if (tid == 32 || tid == 64) {  // the vectors that stick out, element by element
      const int v = tid == 32 ? 0 : n_vec - 1, c = v * VEC - phase, block = v / VR_THREADS;
      if (block % size == rank && (c < 0 || c + VEC > vocab)) {
        T* e = (T*)(slots + block / size * VR_THREADS + v % VR_THREADS);
        for (int i = 0; i < VEC; ++i) e[i] = c + i >= 0 && c + i < vocab ? row[c + i] : from_f32<T>(-INFINITY);
      }
    }
  }
  __device__ __forceinline__ void wait(int step) const {
    if (!mbar_try_wait(bars + step, 0)) row_wait_slow(bars + step, status);
  }
  // whether every thread has all of its elements in this step: only the row's last block may be short
  __device__ __forceinline__ bool whole(int step) const { return (step + 1) * STEP < n_it; }
  // the 16 elements of a step, -inf where the thread has none
  template <bool WHOLE>
  __device__ __forceinline__ void get(int step, float (&x)[16]) const {
#pragma unroll
    for (int j = 0; j < STEP; ++j) {
      const int it = step * STEP + j;
      if (WHOLE || (it < n_it && first_vector(it) + (int)threadIdx.x < n_vec)) {
        unpack(slots[it * VR_THREADS + threadIdx.x], x + j * VEC);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[j * VEC + i] = -INFINITY;
      }
    }
  }
  __device__ __forceinline__ void get(int step, float (&x)[16]) const {
    if (whole(step)) get<true>(step, x);
    else get<false>(step, x);
  }
  static __device__ __forceinline__ void unpack(const uint4& u, float* x) {
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
};

// Writes a vector's results to columns c .. of a row of `vocab`; aligned: whole vectors lie on 16 bytes (8 where they are no longer).
template <class O, int VEC>
__device__ __forceinline__ void put_vector(O* out, int c, int vocab, bool aligned, const float* x) {
  if (aligned && c >= 0 && c + VEC <= vocab) {
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
      __stcs((uint2*)(out + c), make_uint2(w[0], w[1]));
    } else {
#pragma unroll
      for (int i = 0; i < (int)(VEC * sizeof(O) / 16); ++i) __stcs((uint4*)(out + c) + i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (c + i >= 0 && c + i < vocab) out[c + i] = from_f32<O>(x[i]);
  }
}
template <class O, int VEC>
__device__ __forceinline__ bool vectors_aligned(const O* out, int phase) {
  return ((uintptr_t)out - (uintptr_t)phase * sizeof(O)) % (VEC * sizeof(O) < 16 ? VEC * sizeof(O) : 16) == 0;
}

// Writes a step's results: x[i] belongs to the element that get() gave as x[i].
template <class O, class T>
__device__ __forceinline__ void put_step(const RowPart<T>& part, int step, O* out, bool aligned, const float (&x)[16]) {
  constexpr int VEC = RowPart<T>::VEC;
#pragma unroll
  for (int j = 0; j < RowPart<T>::STEP; ++j) {
    const int it = step * RowPart<T>::STEP + j;
    if (it < part.n_it) put_vector<O, VEC>(out, part.column(it, threadIdx.x), part.vocab, aligned, x + j * VEC);
  }
}

// A running maximum, and the sum of exponentials relative to it.
struct MaxSum {
  float m = -INFINITY, s = 0.0f;
  __device__ __forceinline__ void take(const float (&x)[16], const ExpT& ex) {
    float cm = max_nan(x[0], x[1], x[2]);
#pragma unroll
    for (int i = 3; i < 15; i += 2) cm = max_nan(cm, x[i], x[i + 1]);
    cm = max_nan(cm, x[15], m);
    if (cm != m) {  // a NaN too
      s = m > -INFINITY ? s * ex(m - cm) : 0.0f;
      m = cm;
    }
    const float ref = m > -INFINITY ? m : 0.0f;
    float p[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 16; ++i) p[i & 3] += ex(x[i] - ref);
    s += (p[0] + p[1]) + (p[2] + p[3]);
  }
};
// The warp's sum of its threads' exponentials, relative to the largest of their maxima.  In 32 bits: five roundings, which differ from
// warp to warp; what comes after is in 64.
__device__ __forceinline__ float warp_join(const MaxSum& t, const ExpT& ex, float* m) {
  *m = warp_max_nan(t.m);
  float s = t.m > -INFINITY ? t.s * ex(t.m - *m) : 0.0f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}
// The row's sum from the warps' (two a lane; a lane without brings m = -inf).
__device__ __forceinline__ double cluster_join(float ma, float sa, float mb, float sb, const ExpT& ex, float* m) {
  *m = warp_max_nan(max_nan(ma, mb));
  return warp_sum_f64((ma > -INFINITY ? (double)sa * ex(ma - *m) : 0.0) + (mb > -INFINITY ? (double)sb * ex(mb - *m) : 0.0));
}

// How a row is held: the cluster's CTAs, a power of two, as few as leave a thread with VR_SLOTS vectors at most (three CTAs then
// find room on an SM), eight for all longer rows; and the slots of a CTA.
constexpr int VR_SLOTS = 17;
struct RowShape {
  int cluster;
  size_t slots;
};
inline RowShape row_shape(int vocab, int dtype) {
  const int vec = dtype == RT_DT_F32 ? 4 : 8;
  const int blocks = ((vec - 1 + vocab + vec - 1) / vec + VR_THREADS - 1) / VR_THREADS;  // at the worst alignment
  int size = 1;
  while (size < VR_MAX_CLUSTER && (blocks + size - 1) / size > VR_SLOTS) size *= 2;
  return {size, (size_t)((blocks + size - 1) / size) * VR_THREADS};
}

// `rows` clusters of `size` CTAs
template <class... KArgs, class... A>
inline int launch_clusters(rt_ctx* c, void (*kernel)(KArgs...), size_t rows, int size, size_t smem, A&&... args) {
  if (!c->raise_smem(kernel, VR_MOST_SMEM)) return 3;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * size));
  cfg.blockDim = dim3(VR_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = c->stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)size;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
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
