// Verification of drafted tokens: one CTA per sequence.
#include "vocab_rows.cuh"

namespace rt {

static constexpr int VD_THREADS = 512, VD_WARPS = VD_THREADS / 32;

__device__ __forceinline__ double mass_of(double v) { return v > 0.0 && v < (double)INFINITY ? v : 0.0; }

template <class T>
__global__ void __launch_bounds__(VD_THREADS) verify_draft_kernel(const T* P, size_t ld_p, const T* Q, size_t ld_q, int vocab, const int* tok,
                                                                  const int* offsets, int n_seq, int n_draft, const float* u_accept,
                                                                  const float* u_sample, int* accepted, int* token, int* status) {
  __shared__ int s_first, s_bad;
  __shared__ double s_mass[VD_WARPS];
  __shared__ int s_token;
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int a = offsets[s], e = offsets[s + 1];
  if (tid == 0) { s_first = 0x7fffffff; s_bad = 0; s_token = -1; }
  __syncthreads();
  bool bad = a < 0 || e < a || e > n_draft || (s == 0 && a != 0) || (s == n_seq - 1 && e != n_draft);
  if (!bad)
    for (int i = a + tid; i < e; i += VD_THREADS) {
      const int d = tok[i];
      if (d < 0 || d >= vocab) { s_bad = 1; continue; }
      const double p = to_f32(P[(size_t)(i + s) * ld_p + d]), q = Q ? to_f32(Q[(size_t)i * ld_q + d]) : 1.0;
      if (!((double)u_accept[i] * q < p)) atomicMin(&s_first, i);
    }
  __syncthreads();
  bad |= s_bad != 0;
  if (bad) {
    if (tid == 0) {
      report_status(status, RT_ERR_BAD_INDEX);
      accepted[s] = 0;
      token[s] = -1;
    }
    return;
  }
  const int at = min(s_first, e);
  const T* p = P + (size_t)(at + s) * ld_p;
  const T* q = Q && at < e ? Q + (size_t)at * ld_q : nullptr;
  int without = !Q && at < e ? tok[at] : -1;
  // each warp a contiguous piece, so that a running sum over the pieces finds the one that holds the token
  const int per = (vocab + VD_WARPS - 1) / VD_WARPS, lo = warp * per, hi = min(vocab, lo + per);
  auto left = [&](int i) {
    const double x = to_f32(p[i]);
    return i == without ? 0.0 : mass_of(q ? x - (double)to_f32(q[i]) : x);
  };
  double before = 0.0, total = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    double m = 0.0;
    for (int i = lo + lane; i < hi; i += 32) m += left(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    if (lane == 0) s_mass[warp] = m;
    __syncthreads();
    before = total = 0.0;
    for (int w = 0; w < VD_WARPS; ++w) {
      if (w == warp) before = total;
      total += s_mass[w];
    }
    __syncthreads();
    if (total > 0.0) break;
    q = nullptr;  // nothing is left: the target's own probabilities
    without = -1;
  }
  if (tid == 0) accepted[s] = at - a;
  if (total > 0.0) {
    const float u = u_sample[s];
    const double want = u < 0.0f ? 0.0 : (double)u * total, after = warp + 1 < VD_WARPS ? before + s_mass[warp] : total;
    // the piece whose running sum is the first to exceed `want`, and the last piece with mass where none does
    const bool mine = s_mass[warp] > 0.0 && (after > want || after == total) && !(before > want);
    if (mine) {
      double run = before;
      int found = -1, last = -1;
      for (int i0 = lo; i0 < hi && found < 0; i0 += 32) {
        const int i = i0 + lane;
        const double v = i < hi ? left(i) : 0.0;
        double x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        const unsigned with = __ballot_sync(0xffffffffu, v > 0.0), over = __ballot_sync(0xffffffffu, v > 0.0 && run + x > want);
        if (over) found = i0 + __ffs(over) - 1;
        if (with) last = i0 + 31 - __clz(with);
        run += __shfl_sync(0xffffffffu, x, 31);
      }
      if (lane == 0) atomicMax(&s_token, found >= 0 ? found : last);
    }
  }
  __syncthreads();
  if (tid == 0) token[s] = s_token;
}

int launch_verify_draft(rt_ctx* c, const VerifyArgs& a) {
  return with_dtype(a.p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    verify_draft_kernel<T><<<(unsigned)a.n_seq, VD_THREADS, 0, c->stream>>>((const T*)a.p.p, a.p.ld, (const T*)a.q.p, a.q.ld, a.vocab, a.tok, a.offsets,
                                                                            a.n_seq, a.n_draft, a.u_accept, a.u_sample, a.accepted, a.token, c->status_dev);
    RT_COUNT_LAUNCH(1);
    return cudaGetLastError() == cudaSuccess ? 0 : 3;
  });
}

}  // namespace rt
