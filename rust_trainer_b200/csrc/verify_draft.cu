// Verification of drafted tokens: a cluster of CTAs a sequence.  Every CTA finds the first draft that does not stand (the draws are few);
// then each warp sums a contiguous piece of the row that the next token is drawn from, the warps' sums go to all CTAs, and the warp whose
// piece holds the token looks for it there, in the eighth of the piece that its own sums point to.  The row is read once.
//
// Measured: one sequence with four drafts over 151936 f32 12 to 13 us, 96 with up to eight over 128256 bf16 26.5 us (floor 5.7), 32 with up to three
// certain ones over 151936 f32 17 to 22 us (3).  What bounds it: dependent loads (offsets, tokens, their probabilities, the row, the piece once
// more), and for many sequences the arithmetic of exact sums: 62 % of the issue slots of SMs that work, 42 % of all.  512 threads took 42 us for the
// 32; sums of two floats on packed pairs took more registers and the same time.
#include "vocab_rows.cuh"

namespace rt {

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_cluster(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

constexpr int VD_THREADS = 256, VD_WARPS = VD_THREADS / 32, VD_EIGHTHS = 8;

__device__ __forceinline__ bool is_mass(float v) { return v > 0.0f && v < INFINITY; }

// A sum as two floats: the second holds what the first rounds away (Knuth's two-sum), so that sums of many elements are exact to some
// 2^-45, at a fraction of the conversions and additions in 64 bits, which took ten times as long here.
struct Sum2 {
  float hi = 0.0f, lo = 0.0f;
  __device__ __forceinline__ void add(float v, float v_lo) {
    const float s = hi + v, b = s - hi;
    lo += (hi - (s - b)) + (v - b) + v_lo;
    hi = s;
  }
  __device__ __forceinline__ double value() const { return (double)hi + (double)lo; }
};

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
  // 16 bytes of p and of q (0 where there are none)
  __device__ __forceinline__ void load(int v, uint4* a, uint4* b) const {
    const int c = column(v);
    *a = *b = make_uint4(0, 0, 0, 0);
    if (v >= n_vec) return;
    if (c >= 0 && c + VEC <= vocab) {
      *a = __ldg((const uint4*)(p + c));
      if (q && same_phase) *b = __ldg((const uint4*)(q + c));
      else if (q) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) ((T*)b)[i] = q[c + i];
      }
    } else {
      for (int i = 0; i < VEC; ++i) {
        if (c + i < 0 || c + i >= vocab) continue;
        ((T*)a)[i] = p[c + i];
        if (q) ((T*)b)[i] = q[c + i];
      }
    }
  }
  // the masses as sums of two floats: a difference of two floats is one rounded and what the rounding lost
  __device__ __forceinline__ void masses(int v, const uint4& a, const uint4& b, float (&x)[VEC], float (&lo)[VEC]) const {
    float pa[VEC], pb[VEC];
    unpack_vector<T>(a, pa);
    unpack_vector<T>(b, pb);
    const int skip = without - column(v);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float d = pa[i] - pb[i], bb = d - pa[i], e = (pa[i] - (d - bb)) - (pb[i] + bb);
      const bool on = is_mass(d) && i != skip;
      x[i] = on ? d : 0.0f;
      lo[i] = on ? e : 0.0f;
    }
  }
};

template <class T>
__global__ void __launch_bounds__(VD_THREADS) verify_draft_kernel(const T* P, size_t ld_p, const T* Q, size_t ld_q, int vocab, const int* tok,
                                                                  const int* offsets, int n_seq, int n_draft, const float* u_accept,
                                                                  const float* u_sample, int* accepted, int* token, int* status) {
  constexpr int VEC = Left<T>::VEC;
  __shared__ int s_first, s_bad;
  __shared__ double mass[2][VR_MAX_CLUSTER * VD_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster_ctarank(), size = (int)cluster_size();
  const int s = (int)cluster_id();
  cluster_arrive_relaxed();
  const int a = offsets[s], e = offsets[s + 1];
  const float u = u_sample[s];
  if (tid == 0) s_first = 0x7fffffff, s_bad = 0;
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
  const int pieces = size * VD_WARPS, piece = rank * VD_WARPS + warp;
  const T* p_row = P + (size_t)(at + s) * ld_p;
  Left<T> left(p_row, Q && at < e ? Q + (size_t)at * ld_q : nullptr, !Q && at < e ? tok[at] : -1, vocab);
  // vectors of an eighth of a piece, in rounds of a warp
  const int rounds = (left.n_vec + 32 * VD_EIGHTHS * pieces - 1) / (32 * VD_EIGHTHS * pieces), eighth = rounds * 32, lo = piece * eighth * VD_EIGHTHS;
  double sums[VD_EIGHTHS], total = 0.0, run = 0.0, want = 0.0;
  int chosen = -1;  // the piece that holds the token
  for (int pass = 0; pass < 2 && chosen < 0; ++pass) {
    if (pass > 0) left = Left<T>(p_row, nullptr, -1, vocab);  // nothing was left: the target's own probabilities
    Sum2 acc[VD_EIGHTHS];
    for (int t = 0; t < rounds; ++t) {
#pragma unroll
      for (int j0 = 0; j0 < VD_EIGHTHS; j0 += 4) {
        uint4 pa[4], qa[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) left.load(lo + (j0 + j) * eighth + t * 32 + lane, pa + j, qa + j);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x[VEC], x_lo[VEC];
          left.masses(lo + (j0 + j) * eighth + t * 32 + lane, pa[j], qa[j], x, x_lo);
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[j0 + j].add(x[i], x_lo[i]);
        }
      }
    }
    double mine = 0.0;
#pragma unroll
    for (int j = 0; j < VD_EIGHTHS; ++j) sums[j] = warp_sum_f64(acc[j].value());
#pragma unroll
    for (int j = 0; j < VD_EIGHTHS; ++j) mine += sums[j];
    if (lane < size) st_cluster(mapa_u32(smem_u32(&mass[pass][piece]), lane), mine);
    cluster_arrive();
    cluster_wait();
    // Running sums over the pieces, two a lane, the same in every warp.  The token's piece is the first with mass whose sum exceeds
    // `want`, or the last with mass where none does.
    const double m0 = 2 * lane < pieces ? mass[pass][2 * lane] : 0.0, m1 = 2 * lane + 1 < pieces ? mass[pass][2 * lane + 1] : 0.0;
    double up = m0 + m1;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const double y = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += y;
    }
    total = __shfl_sync(0xffffffffu, up, 31);
    if (!(total > 0.0)) continue;
    want = u < 0.0f ? 0.0 : u < 1.0f ? (double)u * total : INFINITY;  // (from 1 on, and a NaN: no running sum exceeds it, however it was rounded)
    double in_front = __shfl_up_sync(0xffffffffu, up, 1);  // of the lane's two pieces
    if (lane == 0) in_front = 0.0;
    const unsigned over0 = __ballot_sync(0xffffffffu, m0 > 0.0 && in_front + m0 > want), over1 = __ballot_sync(0xffffffffu, m1 > 0.0 && up > want);
    const unsigned with0 = __ballot_sync(0xffffffffu, m0 > 0.0), with1 = __ballot_sync(0xffffffffu, m1 > 0.0);
    if (over0 | over1) {
      const int l = __ffs(over0 | over1) - 1;
      chosen = 2 * l + !(over0 >> l & 1);
    } else {
      const int l = 31 - __clz(with0 | with1);
      chosen = 2 * l + (with1 >> l & 1);
    }
    run = __shfl_sync(0xffffffffu, in_front, chosen / 2);
    const double m_even = __shfl_sync(0xffffffffu, m0, chosen / 2);
    if (chosen & 1) run += m_even;
  }
  if (chosen < 0 && tid == 0 && rank == 0) token[s] = -1;
  if (chosen != piece) return;
  // the eighth and the vector and the element, by the same rule
  int first = -1, last = -1;
  double run_last = run;
#pragma unroll
  for (int j = 0; j < VD_EIGHTHS; ++j) {
    if (first < 0 && sums[j] > 0.0) {
      last = j;
      run_last = run;
      if (run + sums[j] > want) first = j;
      else run += sums[j];
    }
  }
  run = run_last;
  int found = -1, at_last = -1;
  for (int t = 0; t < rounds && found < 0; ++t) {
    const int v = lo + last * eighth + t * 32 + lane;
    uint4 pa, qa;
    float x[VEC], x_lo[VEC];
    left.load(v, &pa, &qa);
    left.masses(v, pa, qa, x, x_lo);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum += (double)x[i] + (double)x_lo[i];
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
      part += (double)x[i] + (double)x_lo[i];
      if (x[i] > 0.0f) {
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
  // As many CTAs a sequence as run at once for all of them, three on an SM: a second wave costs more than a longer row.  In us, one call after the
  // other, by the cluster's size (drafts with probabilities):
  //   1 of 30000 f32   1: 15.9, 2: 11.0, 4 and 8: 8.3        1 of 151936 f32   1: 51.8, 2: 30.3, 4: 17.8, 8: 13.4       1 of 6000 f32: the same with any
  //   64 of 30000 f32   1: 28.8, 2: 18.5, 4: 12.9, 8: 19.9    96 of 128256 bf16   1: 55.7, 2: 34.1, 4: 25.0, 8: 27.0
  //   200 of 128256 bf16   1: 67.1, 2: 46.7, 4: 45.9, 8: 52.9    1000 of 9000 bf16   1: 35.3, 2: 58.5, 4: 106, 8: 202
  int size = 1;
  while (a.vocab >= 8192 && size < VR_MAX_CLUSTER && (size_t)a.n_seq * size * 2 <= 3 * (size_t)c->num_sms) size *= 2;
  return with_dtype(a.p.dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return launch_clusters(c, verify_draft_kernel<T>, false, a.n_seq, VD_THREADS, size, 0, (const T*)a.p.p, a.p.ld, (const T*)a.q.p, a.q.ld, a.vocab, a.tok, a.offsets,
                           a.n_seq, a.n_draft, a.u_accept, a.u_sample, a.accepted, a.token, c->status_dev);
  });
}

}  // namespace rt
