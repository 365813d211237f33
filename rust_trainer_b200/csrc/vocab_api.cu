// C ABI of the row operations over the vocabulary: checks of the arguments, the device forms, and the host forms over them.
#include "ctx.h"
#include "vocab_rows.h"
#include <math.h>
#include <vector>

namespace {

size_t dtype_bytes(int dtype) { return dtype == RT_DT_F32 ? 4 : 2; }
bool bad_dtype(int dtype) { return dtype != RT_DT_F32 && dtype != RT_DT_BF16 && dtype != RT_DT_F16; }
bool unaligned(const void* p, size_t to) { return (uintptr_t)p % to != 0; }
bool bad_temperature(float t) { return !(t >= 1e-4f && t <= 1e4f); }

// Whether the rows of `in` and `out` share bytes, other than by lying in the same place element by element.  Rows of one pitch may lie between one another;
// where the pitches differ, everything from the first row's start to the last one's end counts.
bool overlap(const void* in, size_t in_ld, int in_dtype, const void* out, size_t out_ld, int out_dtype, size_t rows, size_t vocab) {
  if (in == out && in_dtype == out_dtype && (in_ld == out_ld || rows == 1)) return false;
  const uintptr_t a = (uintptr_t)in, b = (uintptr_t)out;
  const size_t pa = in_ld * dtype_bytes(in_dtype), pb = out_ld * dtype_bytes(out_dtype), wa = vocab * dtype_bytes(in_dtype), wb = vocab * dtype_bytes(out_dtype);
  const size_t na = (rows - 1) * pa + wa, nb = (rows - 1) * pb + wb;
  if (!(a < b + nb && b < a + na)) return false;
  if (pa != pb) return true;
  // the later one's first row begins `at` bytes behind the other's row above it, and reaches into that row or the next one, if there is one
  const bool in_first = a <= b;
  const size_t apart = in_first ? b - a : a - b, at = apart % pa, w_first = in_first ? wa : wb, w_later = in_first ? wb : wa;
  return at < w_first || (at + w_later > pa && apart / pa + 1 < rows);
}

rt_status check_rows(rt_ctx* c, const void* p, int dtype, size_t rows, size_t vocab, size_t ld) {
  if (bad_dtype(dtype)) return c->fail(RT_ERR_BAD_ARG, "rows must be f32, bf16 or f16");
  if (vocab == 0 || vocab > RT_VOCAB_MAX || rows > (1u << 24)) return c->fail(RT_ERR_BAD_SHAPE, "row length or number of rows out of range");
  if (ld < vocab || ld > (1ull << 32)) return c->fail(RT_ERR_BAD_SHAPE, "rows may not lie closer than they are long");
  if (unaligned(p, dtype_bytes(dtype))) return c->fail(RT_ERR_BAD_ARG, "rows are not aligned to their elements");
  return RT_OK;
}

// device temporaries of one call, freed when the call returns
struct Temps {
  std::vector<void*> ptrs;
  ~Temps() {
    for (void* p : ptrs) cudaFree(p);
  }
  template <class T>
  T* get(size_t n) {
    void* p = nullptr;
    if (cudaMalloc(&p, (n ? n : 1) * sizeof(T)) != cudaSuccess) return nullptr;
    ptrs.push_back(p);
    return (T*)p;
  }
  template <class T>
  T* up(const T* host, size_t n, cudaStream_t st) {
    T* d = get<T>(n);
    if (d && n && cudaMemcpyAsync(d, host, n * sizeof(T), cudaMemcpyHostToDevice, st) != cudaSuccess) return nullptr;
    return d;
  }
};

#define RT_DO(expr)                  \
  do {                               \
    const rt_status s__ = (expr);    \
    if (s__ != RT_OK) return s__;    \
  } while (0)

}  // namespace

using namespace rt;

extern "C" {

rt_status rt_top_logits_dev(rt_ctx* c, const void* logits, int dtype, size_t rows, size_t vocab, size_t ld, float temperature, int k,
                            int32_t* index, float* logp, float* lse) {
  if (!c || !logits || !index || !logp) return RT_ERR_BAD_ARG;
  if (rows == 0) return RT_OK;
  RT_DO(check_rows(c, logits, dtype, rows, vocab, ld));
  if (k < 1 || k > RT_TOP_MAX || (size_t)k > vocab) return c->fail(RT_ERR_BAD_SHAPE, "k out of range");
  if (bad_temperature(temperature)) return c->fail(RT_ERR_BAD_ARG, "temperature out of range");
  if (unaligned(index, 4) || unaligned(logp, 4) || unaligned(lse, 4)) return c->fail(RT_ERR_BAD_ARG, "unaligned result");
  RT_CUDA(c, cudaSetDevice(c->device));
  if (launch_top_logits(c, {logits, dtype, ld}, rows, (int)vocab, temperature, k, index, logp, lse))
    return c->fail(RT_ERR_CUDA, "top-logits launch failed");
  return RT_OK;
}

rt_status rt_distill_dev(rt_ctx* c, const void* logits, int dtype, size_t rows, size_t vocab, size_t ld, float temperature,
                         const int32_t* index, const float* teacher_logp, int k, int mode, const float* weight, float* loss, void* dlogits,
                         int d_dtype, size_t d_ld, float* row_scale) {
  if (!c || !logits || !index || !teacher_logp || (!loss && !dlogits)) return RT_ERR_BAD_ARG;
  if (rows == 0) return RT_OK;
  RT_DO(check_rows(c, logits, dtype, rows, vocab, ld));
  if (k < 1 || k > RT_TOP_MAX) return c->fail(RT_ERR_BAD_SHAPE, "k out of range");
  if (bad_temperature(temperature)) return c->fail(RT_ERR_BAD_ARG, "temperature out of range");
  if (mode != RT_DISTILL_RENORM && mode != RT_DISTILL_TAIL) return c->fail(RT_ERR_BAD_ARG, "unknown distillation mode");
  if (unaligned(index, 4) || unaligned(teacher_logp, 4) || unaligned(weight, 4) || unaligned(loss, 4) || unaligned(row_scale, 4))
    return c->fail(RT_ERR_BAD_ARG, "unaligned argument");
  if (row_scale && !dlogits) return c->fail(RT_ERR_BAD_ARG, "row factors without gradients");
  if (dlogits) {
    RT_DO(check_rows(c, dlogits, d_dtype, rows, vocab, d_ld));
    if (overlap(logits, ld, dtype, dlogits, d_ld, d_dtype, rows, vocab)) return c->fail(RT_ERR_BAD_ARG, "gradients overlap the logits");
  }
  RT_CUDA(c, cudaSetDevice(c->device));
  const DistillArgs a{{logits, dtype, ld}, (int)vocab, k, mode, temperature, index, teacher_logp, weight, loss, dlogits,
                      dlogits ? d_dtype : RT_DT_F32, d_ld, row_scale, false};
  if (launch_distill_rows(c, a, rows)) return c->fail(RT_ERR_CUDA, "distillation launch failed");
  return RT_OK;
}

rt_status rt_softmax_dev(rt_ctx* c, const void* logits, int dtype, size_t rows, size_t vocab, size_t ld, float temperature, void* prob,
                         int prob_dtype, size_t prob_ld) {
  if (!c || !logits || !prob) return RT_ERR_BAD_ARG;
  if (rows == 0) return RT_OK;
  RT_DO(check_rows(c, logits, dtype, rows, vocab, ld));
  RT_DO(check_rows(c, prob, prob_dtype, rows, vocab, prob_ld));
  if (bad_temperature(temperature)) return c->fail(RT_ERR_BAD_ARG, "temperature out of range");
  if (overlap(logits, ld, dtype, prob, prob_ld, prob_dtype, rows, vocab)) return c->fail(RT_ERR_BAD_ARG, "probabilities overlap the logits");
  RT_CUDA(c, cudaSetDevice(c->device));
  if (launch_softmax_rows(c, {logits, dtype, ld}, rows, (int)vocab, temperature, prob, prob_dtype, prob_ld))
    return c->fail(RT_ERR_CUDA, "softmax launch failed");
  return RT_OK;
}

rt_status rt_verify_draft_dev(rt_ctx* c, const void* target_prob, size_t target_ld, const void* draft_prob, size_t draft_ld, int dtype,
                              size_t vocab, const int32_t* tok, const int32_t* offsets, size_t n_seq, size_t n_draft, const float* u_accept,
                              const float* u_sample, int32_t* accepted, int32_t* token) {
  if (!c || !target_prob || !offsets || !u_sample || !accepted || !token || (n_draft > 0 && (!tok || !u_accept))) return RT_ERR_BAD_ARG;
  if (n_seq == 0) return n_draft == 0 ? RT_OK : c->fail(RT_ERR_BAD_SHAPE, "drafts without a sequence");
  if (n_seq > (1u << 24) || n_draft > (1u << 24)) return c->fail(RT_ERR_BAD_SHAPE, "too many sequences or drafts");
  RT_DO(check_rows(c, target_prob, dtype, n_seq, vocab, target_ld));
  if (draft_prob) RT_DO(check_rows(c, draft_prob, dtype, n_draft, vocab, draft_ld));
  if (unaligned(tok, 4) || unaligned(offsets, 4) || unaligned(u_accept, 4) || unaligned(u_sample, 4) || unaligned(accepted, 4) || unaligned(token, 4))
    return c->fail(RT_ERR_BAD_ARG, "unaligned argument");
  RT_CUDA(c, cudaSetDevice(c->device));
  const VerifyArgs a{{target_prob, dtype, target_ld}, {n_draft > 0 ? draft_prob : nullptr, dtype, draft_ld}, (int)vocab, tok, offsets,
                     (int)n_seq, (int)n_draft, u_accept, u_sample, accepted, token};
  if (launch_verify_draft(c, a)) return c->fail(RT_ERR_CUDA, "verification launch failed");
  return RT_OK;
}

// ---- host forms

rt_status rt_op_top_logits(rt_ctx* c, const float* logits, size_t rows, size_t vocab, float temperature, int k, int32_t* index, float* logp,
                           float* lse) {
  if (!c || !logits || !index || !logp) return RT_ERR_BAD_ARG;
  if (rows == 0) return RT_OK;
  RT_DO(check_rows(c, logits, RT_DT_F32, rows, vocab, vocab));
  if (k < 1 || k > RT_TOP_MAX) return c->fail(RT_ERR_BAD_SHAPE, "k out of range");
  RT_CUDA(c, cudaSetDevice(c->device));
  Temps t;
  float* z = t.up(logits, rows * vocab, c->stream);
  int32_t* i = t.get<int32_t>(rows * k);
  float *l = t.get<float>(rows * k), *s = t.get<float>(rows);
  if (!z || !i || !l || !s) return c->fail(RT_ERR_CUDA, "out of device memory");
  RT_DO(rt_top_logits_dev(c, z, RT_DT_F32, rows, vocab, vocab, temperature, k, i, l, s));
  RT_CUDA(c, cudaMemcpyAsync(index, i, rows * k * 4, cudaMemcpyDeviceToHost, c->stream));
  RT_CUDA(c, cudaMemcpyAsync(logp, l, rows * k * 4, cudaMemcpyDeviceToHost, c->stream));
  if (lse) RT_CUDA(c, cudaMemcpyAsync(lse, s, rows * 4, cudaMemcpyDeviceToHost, c->stream));
  return c->check_device_status("rt_op_top_logits");
}

rt_status rt_op_distill(rt_ctx* c, const float* logits, size_t rows, size_t vocab, float temperature, const int32_t* index,
                        const float* teacher_logp, int k, int mode, const float* weight, float* loss, float* dlogits) {
  if (!c || !logits || !index || !teacher_logp || !loss) return RT_ERR_BAD_ARG;
  if (rows == 0) return RT_OK;
  RT_DO(check_rows(c, logits, RT_DT_F32, rows, vocab, vocab));
  if (k < 1 || k > RT_TOP_MAX) return c->fail(RT_ERR_BAD_SHAPE, "k out of range");
  RT_CUDA(c, cudaSetDevice(c->device));
  Temps t;
  float* z = t.up(logits, rows * vocab, c->stream);
  int32_t* i = t.up(index, rows * k, c->stream);
  float *l = t.up(teacher_logp, rows * k, c->stream), *w = weight ? t.up(weight, rows, c->stream) : nullptr, *out = t.get<float>(rows);
  if (!z || !i || !l || (weight && !w) || !out) return c->fail(RT_ERR_CUDA, "out of device memory");
  RT_DO(rt_distill_dev(c, z, RT_DT_F32, rows, vocab, vocab, temperature, i, l, k, mode, w, out, dlogits ? z : nullptr, RT_DT_F32, vocab, nullptr));
  RT_CUDA(c, cudaMemcpyAsync(loss, out, rows * 4, cudaMemcpyDeviceToHost, c->stream));
  if (dlogits) RT_CUDA(c, cudaMemcpyAsync(dlogits, z, rows * vocab * 4, cudaMemcpyDeviceToHost, c->stream));
  return c->check_device_status("rt_op_distill");
}

rt_status rt_op_softmax(rt_ctx* c, const float* logits, size_t rows, size_t vocab, float temperature, float* prob) {
  if (!c || !logits || !prob) return RT_ERR_BAD_ARG;
  if (rows == 0) return RT_OK;
  RT_DO(check_rows(c, logits, RT_DT_F32, rows, vocab, vocab));
  RT_CUDA(c, cudaSetDevice(c->device));
  Temps t;
  float* z = t.up(logits, rows * vocab, c->stream);
  if (!z) return c->fail(RT_ERR_CUDA, "out of device memory");
  RT_DO(rt_softmax_dev(c, z, RT_DT_F32, rows, vocab, vocab, temperature, z, RT_DT_F32, vocab));
  RT_CUDA(c, cudaMemcpyAsync(prob, z, rows * vocab * 4, cudaMemcpyDeviceToHost, c->stream));
  return c->check_device_status("rt_op_softmax");
}

rt_status rt_op_verify_draft(rt_ctx* c, const float* target_prob, const float* draft_prob, size_t vocab, const int32_t* tok,
                             const int32_t* offsets, size_t n_seq, const float* u_accept, const float* u_sample, int32_t* accepted,
                             int32_t* token) {
  if (!c || !target_prob || !offsets || !u_sample || !accepted || !token) return RT_ERR_BAD_ARG;
  if (n_seq == 0) return RT_OK;
  if (n_seq > (1u << 24)) return c->fail(RT_ERR_BAD_SHAPE, "too many sequences");
  if (offsets[0] != 0) return c->fail(RT_ERR_BAD_INDEX, "offsets must ascend from 0");
  for (size_t s = 0; s < n_seq; ++s)
    if (offsets[s + 1] < offsets[s]) return c->fail(RT_ERR_BAD_INDEX, "offsets must ascend from 0");
  const size_t n = (size_t)offsets[n_seq];
  if (n > 0 && (!tok || !u_accept)) return c->fail(RT_ERR_BAD_ARG, "drafts missing");
  RT_DO(check_rows(c, target_prob, RT_DT_F32, n + n_seq, vocab, vocab));
  RT_CUDA(c, cudaSetDevice(c->device));
  Temps t;
  float *p = t.up(target_prob, (n + n_seq) * vocab, c->stream), *q = draft_prob ? t.up(draft_prob, n * vocab, c->stream) : nullptr;
  int32_t *d = t.up(tok, n, c->stream), *o = t.up(offsets, n_seq + 1, c->stream), *res = t.get<int32_t>(2 * n_seq);
  float *ua = t.up(u_accept, n, c->stream), *us = t.up(u_sample, n_seq, c->stream);
  if (!p || (draft_prob && !q) || !d || !o || !res || !ua || !us) return c->fail(RT_ERR_CUDA, "out of device memory");
  RT_DO(rt_verify_draft_dev(c, p, vocab, q, vocab, RT_DT_F32, vocab, d, o, n_seq, n, ua, us, res, res + n_seq));
  RT_CUDA(c, cudaMemcpyAsync(accepted, res, n_seq * 4, cudaMemcpyDeviceToHost, c->stream));
  RT_CUDA(c, cudaMemcpyAsync(token, res + n_seq, n_seq * 4, cudaMemcpyDeviceToHost, c->stream));
  return c->check_device_status("rt_op_verify_draft");
}

}  // extern "C"
