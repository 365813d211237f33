// Verification of drafted tokens: a cluster of CTAs a sequence.  Every CTA finds the first draft that does not stand (the draws are few);
// then each warp sums a contiguous piece of the row that the next token is drawn from, the warps' sums go to all CTAs, and the warp whose
// piece holds the token looks for it there, in the eighth of the piece that its own sums point to.  The row is read once.
#include "vocab_rows.cuh"

namespace rt {

constexpr int VD_EIGHTHS = 8;

__device__ __forceinline__ double mass_of(double v) { return v > 0.0 && v < (double)INFINITY ? v : 0.0; }

// The mass that a row leaves: max(p - q, 0), or p, or p without an index.  Vectors of 16 aligned bytes of p's row.
template <class T>
struct Left {
  static constexpr int VEC = 16 / (int)sizeof(T);
  const T *p, *q;
  int without, vocab, phase, n_vec;
  bool same_phase;
  __device__ __forceinline__ Left(const T* p_, const T* q_, int without_, int vocab_) : p(p_), q(q_), without(without_), vocab(vocab_) {
    phase = (int)(((uintptr_t)p & 15) / sizeof(T));
    same_phase = (((uintptr_t)p ^ (uintptr_t)q) & 15) == 0;
    n_vec = (phase + vocab + VEC - 1) / VEC;
  }
  __device__ __forceinline__ int column(int v) const { return v * VEC - phase; }
  __device__ __forceinline__ void get(int v, double (&x)[VEC]) const {
    const int c = column(v);
    float a[VEC], b[VEC];
    if (c >= 0 && c + VEC <= vocab) {
      RowPart<T>::unpack(__ldg((const uint4*)(p + c)), a);
      if (q && same_phase) RowPart<T>::unpack(__ldg((const uint4*)(q + c)), b);
      else if (q) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) b[i] = to_f32(q[c + i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const bool in = c + i >= 0 && c + i < vocab;
        a[i] = in ? to_f32(p[c + i]) : 0.0f;
        b[i] = in && q ? to_f32(q[c + i]) : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = c + i == without ? 0.0 : mass_of(q ? (double)a[i] - (double)b[i] : (double)a[i]);
  }
};

template <class T>
__global__ void __launch_bounds__(VR_THREADS) verify_draft_kernel(const T* P, size_t ld_p, const T* Q, size_t ld_q, int vocab, const int* tok,
                                                                  const int* offsets, int n_seq, int n_draft, const float* u_accept,
                                                                  const float* u_sample, int* accepted, int* token, int* status) {
  constexpr int VEC = Left<T>::VEC;
  __shared__ int s_first, s_bad;
  __shared__ double mass[2][VR_MAX_CLUSTER * VR_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster_ctarank(), size = (int)cluster_size();
  const int s = (int)cluster_id();
  cluster_arrive_relaxed();
  const int a = offsets[s], e = offsets[s + 1];
  const float u = u_sample[s];
  if (tid == 0) s_first = 0x7fffffff, s_bad = 0;
  __syncthreads();
  bool bad = a < 0 || e < a || e > n_draft || (s == 0 && a != 0) || (s == n_seq - 1 && e != n_draft);
  if (!bad)
    for (int i = a + tid; i < e; i += VR_THREADS) {
      const int d = tok[i];
      if (d < 0 || d >= vocab) { s_bad = 1; continue; }
      const double p = to_f32(P[(size_t)(i + s) * ld_p + d]), q = Q ? to_f32(Q[(size_t)i * ld_q + d]) : 1.0;
      if (!((double)u_accept[i] * q < p)) atomicMin(&s_first, i);
    }
  __syncthreads();
  bad |= s_bad != 0;
  cluster_wait();  // the other CTAs run: their shared memory may be written
  if (bad) {  // every CTA of the cluster sees the same
    if (tid == 0 && rank == 0) {
      report_status(status, RT_ERR_BAD_INDEX);
      accepted[s] = 0;
      token[s] = -1;
    }
    return;
  }
  const int at = min(s_first, e);
  if (tid == 0 && rank == 0) accepted[s] = at - a;
  const int pieces = size * VR_WARPS, piece = rank * VR_WARPS + warp;
  const T* p_row = P + (size_t)(at + s) * ld_p;
  Left<T> left(p_row, Q && at < e ? Q + (size_t)at * ld_q : nullptr, !Q && at < e ? tok[at] : -1, vocab);
  // vectors of an eighth of a piece, in rounds of a warp
  const int rounds = (left.n_vec + 32 * VD_EIGHTHS * pieces - 1) / (32 * VD_EIGHTHS * pieces), eighth = rounds * 32, lo = piece * eighth * VD_EIGHTHS;
  double sums[VD_EIGHTHS], total = 0.0, before = 0.0, mine = 0.0;
  const double* masses = nullptr;
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int j = 0; j < VD_EIGHTHS; ++j) sums[j] = 0.0;
    for (int t = 0; t < rounds; ++t) {
#pragma unroll
      for (int j = 0; j < VD_EIGHTHS; ++j) {
        const int v = lo + j * eighth + t * 32 + lane;
        if (v >= left.n_vec) continue;
        double x[VEC];
        left.get(v, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sums[j] += x[i];
      }
    }
#pragma unroll
    for (int j = 0; j < VD_EIGHTHS; ++j) sums[j] = warp_sum_f64(sums[j]);
    mine = 0.0;
#pragma unroll
    for (int j = 0; j < VD_EIGHTHS; ++j) mine += sums[j];
    if (lane < size) st_cluster(mapa_u32(smem_u32(&mass[pass][piece]), lane), mine);
    cluster_arrive();
    cluster_wait();
    total = before = 0.0;
    masses = mass[pass];
    for (int i = 0; i < pieces; ++i) {
      if (i == piece) before = total;
      total += masses[i];
    }
    if (total > 0.0) break;
    left = Left<T>(p_row, nullptr, -1, vocab);  // nothing is left: the target's own probabilities
  }
  if (!(total > 0.0)) {
    if (tid == 0 && rank == 0) token[s] = -1;
    return;
  }
  // The piece whose running sum is the first to exceed `want`; the last one with mass where none does.
  const double want = u < 0.0f ? 0.0 : (double)u * total;
  const bool none = !(total > want);
  bool here = mine > 0.0 && !(before > want) && before + mine > want;
  if (none) {
    here = mine > 0.0;
    for (int i = piece + 1; i < pieces; ++i) here &= !(masses[i] > 0.0);
  }
  if (!here) return;
  double run = before;
  int first = -1, last = -1;
#pragma unroll
  for (int j = 0; j < VD_EIGHTHS; ++j) {  // the eighth, by the same rule
    if (sums[j] > 0.0) {
      last = j;
      if (first < 0 && run + sums[j] > want) first = j;
      else if (first < 0) run += sums[j];
    }
  }
  if (first < 0) {
    first = last;
    run = before;
#pragma unroll
    for (int j = 0; j < VD_EIGHTHS; ++j)
      if (j < last) run += sums[j];
  }
  int found = -1, at_last = -1;
  for (int t = 0; t < rounds && found < 0; ++t) {
    const int v = lo + first * eighth + t * 32 + lane;
    double x[VEC] = {}, sum = 0.0;
    if (v < left.n_vec) left.get(v, x);
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += x[i];
    double up = sum;  // with the lanes in front
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const double y = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += y;
    }
    const unsigned over = __ballot_sync(0xffffffffu, sum > 0.0 && run + up > want), with = __ballot_sync(0xffffffffu, sum > 0.0);
    int hit = -1, end = -1;
    double part = run + (up - sum);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      part += x[i];
      if (x[i] > 0.0) {
        end = left.column(v) + i;
        if (hit < 0 && part > want) hit = end;
      }
    }
    if (hit < 0) hit = end;
    if (over) found = __shfl_sync(0xffffffffu, hit, __ffs(over) - 1);
    if (with) at_last = __shfl_sync(0xffffffffu, end, 31 - __clz(with));
    run += __shfl_sync(0xffffffffu, up, 31);
  }
  if (lane == 0) token[s] = found >= 0 ? found : at_last;
}

int launch_verify_draft(rt_ctx* c, const VerifyArgs& a) {
  const int size = a.vocab >= 8192 ? 8 : a.vocab >= 2048 ? 2 : 1;
  return with_dtype(a.p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_clusters(c, verify_draft_kernel<T>, a.n_seq, size, 0, (const T*)a.p.p, a.p.ld, (const T*)a.q.p, a.q.ld, a.vocab, a.tok, a.offsets,
                           a.n_seq, a.n_draft, a.u_accept, a.u_sample, a.accepted, a.token, c->status_dev);
  });
}

}  // namespace rt
