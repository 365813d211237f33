// Softmax and distillation over rows of logits: one CTA per row, the row read once for its maximum, once for its sums and
// once for what is written.
#include "vocab_rows.cuh"

namespace rt {

static constexpr int VR_THREADS = 512;

template <class T, class Op>
__device__ T block_reduce(T v, T none, Op op, T* sh /* 33 */) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) sh[w] = v;
  __syncthreads();
  if (w == 0) {
    v = lane < (int)(blockDim.x >> 5) ? sh[lane] : none;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane == 0) sh[32] = v;
  }
  __syncthreads();
  return sh[32];
}
struct MaxNan { __device__ float operator()(float a, float b) const { return max_nan(a, b); } };
struct AddD { __device__ double operator()(double a, double b) const { return a + b; } };

template <class T, class O>
__global__ void __launch_bounds__(VR_THREADS) softmax_rows_kernel(const T* z, size_t ld, int vocab, float t, O* prob, size_t prob_ld) {
  __shared__ float shf[33];
  __shared__ double shd[33];
  const T* row = z + blockIdx.x * ld;
  O* out = prob + blockIdx.x * prob_ld;
  const Temperature temp(t);
  float m = -INFINITY;
  for (int i = threadIdx.x; i < vocab; i += VR_THREADS) m = max_nan(m, to_f32(row[i]));
  m = block_reduce(m, -INFINITY, MaxNan(), shf);
  double s = 0.0;
  if (m > -INFINITY)
    for (int i = threadIdx.x; i < vocab; i += VR_THREADS) s += expf(temp(to_f32(row[i]) - m));
  s = block_reduce(s, 0.0, AddD(), shd);
  // a row of -inf has no probabilities, one with a NaN or +inf no number for them
  const float inv = m == -INFINITY ? 0.0f : m < INFINITY ? (float)(1.0 / s) : NAN;
  if (m == -INFINITY) m = 0.0f;
  for (int i = threadIdx.x; i < vocab; i += VR_THREADS) out[i] = from_f32<O>(expf(temp(to_f32(row[i]) - m)) * inv);
}

template <class T, class O>
__global__ void __launch_bounds__(VR_THREADS) distill_rows_kernel(const T* z, size_t ld, int vocab, float t, const int* index, const float* teacher,
                                                                  int k, int tail, const float* weight, float* loss, O* d, size_t d_ld,
                                                                  float* row_scale, int* status) {
  extern __shared__ uint32_t in_list[];  // a bit for each index
  __shared__ float shf[33];
  __shared__ double shd[33];
  __shared__ int s_index[RT_TOP_MAX];
  __shared__ double s_q[RT_TOP_MAX];
  const size_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const T* row = z + r * ld;
  O* out = d ? d + r * d_ld : nullptr;
  const Temperature temp(t);
  const float w = weight ? weight[r] : 1.0f;
  const float factor = w / t, g = row_scale ? 1.0f : factor;
  if (row_scale && tid == 0) row_scale[r] = factor;
  // the list: probabilities, and for each index its first entry with all of its probability
  for (int i = tid; i < (vocab + 31) / 32; i += VR_THREADS) in_list[i] = 0;
  int at = -1;
  double lt = -INFINITY;
  if (tid < k) {
    at = index[r * k + tid];
    if (at < -1 || at >= vocab) {
      report_status(status, RT_ERR_BAD_INDEX);
      at = -1;
    }
    if (at >= 0) lt = teacher[r * k + tid];
    s_index[tid] = at;
  }
  double q = exp(lt);
  const double mass = block_reduce(q, 0.0, AddD(), shd);
  const double rest = tail ? fmax(0.0, 1.0 - mass) : 0.0;
  if (!tail && mass > 0.0) {
    q /= mass;
    lt -= log(mass);
  }
  if (tid < k) s_q[tid] = q;
  __syncthreads();
  if (w == 0.0f || (!tail && mass == 0.0)) {  // nothing to learn from
    if (loss && tid == 0) loss[r] = 0.0f;
    if (out)
      for (int i = tid; i < vocab; i += VR_THREADS) out[i] = from_f32<O>(0.0f);
    return;
  }
  bool first = at >= 0;
  double q_all = 0.0;
  if (at >= 0) {
    for (int j = 0; j < k; ++j)
      if (s_index[j] == at) {
        if (j < tid) first = false;
        q_all += s_q[j];
      }
    if (first) atomicOr(&in_list[at >> 5], 1u << (at & 31));
  }
  __syncthreads();
  auto listed = [&](int i) { return (in_list[i >> 5] >> (i & 31)) & 1u; };
  // maximum and sum inside and outside of the list; the latter relative to their own maximum, which may be far below
  const float z_at = at >= 0 ? to_f32(row[at]) : -INFINITY;
  float mo = -INFINITY;
  for (int i = tid; i < vocab; i += VR_THREADS)
    if (!listed(i)) mo = max_nan(mo, to_f32(row[i]));
  mo = block_reduce(mo, -INFINITY, MaxNan(), shf);
  const float mi = block_reduce(z_at, -INFINITY, MaxNan(), shf), m = max_nan(mo, mi);
  const bool bad = !(m < INFINITY);
  double so = 0.0;
  if (mo > -INFINITY)
    for (int i = tid; i < vocab; i += VR_THREADS)
      if (!listed(i)) so += expf(temp(to_f32(row[i]) - mo));
  so = block_reduce(so, 0.0, AddD(), shd);
  const double x_at = z_at > -INFINITY ? ((double)z_at - m) / t : -INFINITY;
  const double si = block_reduce(first ? exp(x_at) : 0.0, 0.0, AddD(), shd);
  const double down = mo > -INFINITY ? exp(((double)mo - m) / t) : 0.0;  // of what is outside, relative to the row's maximum
  const double s = si + so * down, log_s = log(s);
  double l = q > 0.0 ? q * (lt - (s > 0.0 ? x_at - log_s : -INFINITY)) : 0.0;
  l = block_reduce(l, 0.0, AddD(), shd);
  if (loss && tid == 0) {
    if (rest > 0.0) l += rest * (log(rest) - (so > 0.0 ? ((double)mo - m) / t + log(so) - log_s : -INFINITY));
    loss[r] = bad ? NAN : (float)(w * l);
  }
  if (!out) return;
  const float co = bad ? NAN : so > 0.0 ? (float)(down / s - rest / so) * g : 0.0f;
  const float ref = mo > -INFINITY ? mo : 0.0f;
  for (int i = tid; i < vocab; i += VR_THREADS)
    if (!listed(i)) out[i] = from_f32<O>(expf(temp(to_f32(row[i]) - ref)) * co);
  if (first) out[at] = from_f32<O>(bad ? NAN : (float)((s > 0.0 ? exp(x_at) / s : 0.0) - q_all) * g);
}

int launch_softmax_rows(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, void* prob, int prob_dtype, size_t prob_ld) {
  return with_dtype(z.dtype, [&](auto* zt) {
    return with_dtype(prob_dtype, [&](auto* ot) {
      using T = std::remove_pointer_t<decltype(zt)>;
      using O = std::remove_pointer_t<decltype(ot)>;
      softmax_rows_kernel<T, O><<<(unsigned)rows, VR_THREADS, 0, c->stream>>>((const T*)z.p, z.ld, vocab, temperature, (O*)prob, prob_ld);
      RT_COUNT_LAUNCH(1);
      return cudaGetLastError() == cudaSuccess ? 0 : 3;
    });
  });
}

int launch_distill_rows(rt_ctx* c, const DistillArgs& a, size_t rows) {
  return with_dtype(a.z.dtype, [&](auto* zt) {
    return with_dtype(a.d_dtype, [&](auto* ot) {
      using T = std::remove_pointer_t<decltype(zt)>;
      using O = std::remove_pointer_t<decltype(ot)>;
      auto* kernel = distill_rows_kernel<T, O>;
      if (!c->raise_smem(kernel, RT_VOCAB_MAX / 8)) return 3;
      kernel<<<(unsigned)rows, VR_THREADS, ((size_t)a.vocab + 31) / 32 * 4, c->stream>>>(
          (const T*)a.z.p, a.z.ld, a.vocab, a.temperature, a.index, a.teacher, a.k, a.mode == RT_DISTILL_TAIL, a.weight, a.loss, (O*)a.d, a.d_ld,
          a.row_scale, c->status_dev);
      RT_COUNT_LAUNCH(1);
      return cudaGetLastError() == cudaSuccess ? 0 : 3;
    });
  });
}

}  // namespace rt
