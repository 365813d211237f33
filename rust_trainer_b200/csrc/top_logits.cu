// The k largest logits of each row: one CTA per row, which finds the largest value below the last one found k times over.
#include "vocab_rows.cuh"

namespace rt {

static constexpr int TOP_THREADS = 512;

template <class T>
__global__ void __launch_bounds__(TOP_THREADS) top_logits_kernel(const T* z, size_t ld, int vocab, float t, int k, int* index, float* logp, float* lse) {
  __shared__ unsigned long long s_best[16];
  __shared__ double s_sum[16];
  __shared__ unsigned long long s_found[RT_TOP_MAX];
  const size_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const T* row = z + r * ld;
  unsigned long long last = ~0ull;
  for (int j = 0; j < k; ++j) {
    unsigned long long best = 0;
    for (int i = tid; i < vocab; i += TOP_THREADS) {
      const unsigned long long key = ((unsigned long long)order32(to_f32(row[i])) << 32) | (uint32_t)(0x7fffffff - i);
      if (key < last && key > best) best = key;
    }
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if ((tid & 31) == 0) s_best[tid >> 5] = best;
    __syncthreads();
    for (int w = 0; w < TOP_THREADS / 32; ++w) best = max(best, s_best[w]);
    last = best;
    if (tid == 0) s_found[j] = best;
  }
  __syncthreads();
  const Temperature temp(t);
  const float m = order32_value((uint32_t)(s_found[0] >> 32));
  double s = 0.0;
  if (m > -INFINITY)
    for (int i = tid; i < vocab; i += TOP_THREADS) s += expf(temp(to_f32(row[i]) - m));
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((tid & 31) == 0) s_sum[tid >> 5] = s;
  __syncthreads();
  s = 0.0;
  for (int w = 0; w < TOP_THREADS / 32; ++w) s += s_sum[w];
  const bool bad = !(m < INFINITY);
  if (lse && tid == 0) lse[r] = bad ? NAN : (float)((double)m / t + log(s));
  if (tid < k) {
    const float v = order32_value((uint32_t)(s_found[tid] >> 32));
    index[r * k + tid] = 0x7fffffff - (int)(uint32_t)s_found[tid];
    logp[r * k + tid] = bad ? NAN : v == -INFINITY ? -INFINITY : (float)(((double)v - m) / t - log(s));
  }
}

int launch_top_logits(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, int k, int* index, float* logp, float* lse) {
  return with_dtype(z.dtype, [&](auto* zt) {
    using T = std::remove_pointer_t<decltype(zt)>;
    top_logits_kernel<T><<<(unsigned)rows, TOP_THREADS, 0, c->stream>>>((const T*)z.p, z.ld, vocab, temperature, k, index, logp, lse);
    RT_COUNT_LAUNCH(1);
    return cudaGetLastError() == cudaSuccess ? 0 : 3;
  });
}

}  // namespace rt
