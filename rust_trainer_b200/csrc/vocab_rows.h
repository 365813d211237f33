// Launchers of the row operations over the vocabulary (vocab_rows.cu, top_logits.cu, verify_draft.cu).  Every one returns 0, or 3
// when the launch failed; what a kernel finds wrong goes to the ctx's status word.
#pragma once
#include "rt_internal.h"

struct rt_ctx;

namespace rt {

// Rows of one of RT_DT_*, `ld` elements apart.
struct VocabRows {
  const void* p;
  int dtype;
  size_t ld;
};

int launch_softmax_rows(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, void* prob, int prob_dtype, size_t prob_ld);

struct DistillArgs {
  VocabRows z;
  int vocab, k, mode;  // mode: RT_DISTILL_*
  float temperature;
  const int* index;       // [rows x k]
  const float* teacher;   // [rows x k]
  const float* weight;    // [rows] or null
  float* loss;            // [rows] or null
  void* d;                // [rows x vocab] or null, rows d_ld apart
  int d_dtype;
  size_t d_ld;
  float* row_scale;       // [rows] or null: the factor w / T, which d then does not hold
  bool spread;            // f32 rows, f16 gradients with row_scale: these times a power of two, 2^15 as a rule, which row_scale takes back
};
int launch_distill_rows(rt_ctx* c, const DistillArgs& a, size_t rows);

int launch_top_logits(rt_ctx* c, const VocabRows& z, size_t rows, int vocab, float temperature, int k, int* index, float* logp, float* lse);

struct VerifyArgs {
  VocabRows p, q;  // q.p null: drafts without probabilities
  int vocab;
  const int *tok, *offsets;
  int n_seq, n_draft;
  const float *u_accept, *u_sample;
  int *accepted, *token;
};
int launch_verify_draft(rt_ctx* c, const VerifyArgs& a);

}  // namespace rt
