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
// wherever its large values lie.  A thread reads in shared memory only what it copied there itself, so that no barrier stands between
// the copies and their use; all of them are in flight at once.
constexpr uint32_t VR_MOST_SMEM = 214 * 1024;  // dynamic shared memory: RT_VOCAB_MAX elements of 32 bits on eight CTAs, and what is beside them
constexpr int VR_THREADS = 256, VR_WARPS = VR_THREADS / 32, VR_MAX_CLUSTER = 8;

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
// wait until at most n of the thread's copy groups are under way (or fewer, where n is large)
__device__ __forceinline__ void cp_async_wait_n(int n) {
  if (n <= 0) cp_async_wait<0>();
  else if (n == 1) cp_async_wait<1>();
  else if (n == 2) cp_async_wait<2>();
  else if (n == 3) cp_async_wait<3>();
  else if (n <= 5) cp_async_wait<4>();
  else cp_async_wait<6>();
}

template <class T>
struct RowPart {
  static constexpr int VEC = 16 / (int)sizeof(T);   // elements of a vector
  static constexpr int STEP = 16 / VEC;             // vectors of a thread taken at once: 16 elements
  const T* row;
  int phase, vocab, rank, size, n_vec, n_it, n_steps;  // n_it: vectors per thread of this CTA at most
  uint4* slots;                                        // [n_it][VR_THREADS]

  __device__ __forceinline__ RowPart(const T* row_, int vocab_, uint4* slots_)
      : row(row_), vocab(vocab_), rank((int)cluster_ctarank()), size((int)cluster_size()), slots(slots_) {
    phase = (int)(((uintptr_t)row & 15) / sizeof(T));
    n_vec = (phase + vocab + VEC - 1) / VEC;
    const int blocks = (n_vec + VR_THREADS - 1) / VR_THREADS;
    n_it = blocks > rank ? (blocks - rank - 1) / size + 1 : 0;
    n_steps = (n_it + STEP - 1) / STEP;
  }
  // slots per thread of the cluster's first CTA, which has most: where what lies behind them starts in every CTA
  __device__ __forceinline__ int n_it_most() const { return ((n_vec + VR_THREADS - 1) / VR_THREADS + size - 1) / size; }
  // the vector that a thread's `it`-th slot holds, and the column of its first element
  __device__ __forceinline__ int vector(int it) const { return (it * size + rank) * VR_THREADS + (int)threadIdx.x; }
  __device__ __forceinline__ int column(int it, int thread) const { return ((it * size + rank) * VR_THREADS + thread) * VEC - phase; }
  // where column `c` lies: its CTA, and the index of its vector's slot there
  __device__ __forceinline__ int owner(int c, int* slot, int* lane) const {
    const int v = (c + phase) / VEC, block = v / VR_THREADS;
    *slot = block / size * VR_THREADS + v % VR_THREADS;
    *lane = (c + phase) % VEC;
    return block % size;
  }
  __device__ __forceinline__ void load() const {
    for (int s = 0; s < n_steps; ++s) {
#pragma unroll
      for (int j = 0; j < STEP; ++j) {
        const int it = s * STEP + j, v = vector(it), c = v * VEC - phase;
        if (it >= n_it || v >= n_vec) continue;
        uint4* slot = slots + it * VR_THREADS + threadIdx.x;
        if (c >= 0 && c + VEC <= vocab) {
          cp_async_16(smem_u32(slot), row + c);
        } else {
          T* e = (T*)slot;
          for (int i = 0; i < VEC; ++i) e[i] = c + i >= 0 && c + i < vocab ? row[c + i] : from_f32<T>(-INFINITY);
        }
      }
      cp_async_commit();
    }
  }
  __device__ __forceinline__ void wait(int step) const { cp_async_wait_n(n_steps - 1 - step); }
  // the 16 elements of a step, -inf where the thread has none
  __device__ __forceinline__ void get(int step, float (&x)[16]) const {
#pragma unroll
    for (int j = 0; j < STEP; ++j) {
      const int it = step * STEP + j;
      if (it < n_it && vector(it) < n_vec) {
        unpack(slots[it * VR_THREADS + threadIdx.x], x + j * VEC);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) x[j * VEC + i] = -INFINITY;
      }
    }
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
// Sums of several threads' or warps' exponentials, each relative to its own maximum, relative to the maximum of all
// (a warp's worth; lanes that have none bring m = -inf).
__device__ __forceinline__ double warp_join(float m, double s, const ExpT& ex, float* m_all) {
  const float top = warp_max_nan(m);
  *m_all = top;
  return warp_sum_f64(m > -INFINITY ? s * (double)ex(m - top) : 0.0);
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
