// What the samplers share: a step's bookkeeping for the chosen token.
#pragma once
#include "common.h"

// One workgroup per row of logits [B, V] (bf16 or fp32). temperature <= 0 -> greedy.
// Device-side decode bookkeeping so one decode step is graph-capturable (no host round trip):
//   ctr[b]   : per-row RNG counter (the row's position); null -> `step`
//   out_tok  : sampled token (also the next step's input token)
//   out_lp   : log softmax(logits)[tok] under the untempered distribution
//   conf     : [B, 2] running (sum exp(lp), count) -> mean token probability (llm/openai.go:149-164)
//   active   : rows still generating; cleared on EOS or when the history is full
//   pos/lens : advanced by one for active rows
//   hist     : hist[b * hist_ld + (pos[b] - start[b])] = tok (generation history)
struct SampleArgs {
  const void* logits; int V, ld; float temperature; unsigned seed, step;
  const int* ctr; int* out_tok; float* out_lp; float* conf; int* active; int* pos; int* lens;
  int* hist; const int* start; int hist_ld; int eos0, eos1, eos2, eos3;
};

// The sampler's per-row bookkeeping for the chosen token fi (logprob lp), one thread: token /
// logprob out, confidence running sums, generated-token history, position / length advance, stop
// on EOS or a full history. Every operand is read up front: as `x[b] += ...` statements behind the
// active check they were a chain of dependent memory round trips at the end of every decode step.
__device__ __forceinline__ void sample_bookkeep(const SampleArgs& a, int b, int fi, float lp) {
  const int act = a.active ? a.active[b] : 1;
  const float c0 = a.conf ? a.conf[2 * b] : 0.f, c1 = a.conf ? a.conf[2 * b + 1] : 0.f;
  const int pos = a.pos ? a.pos[b] : 0, st = a.hist ? a.start[b] : 0, len = a.lens ? a.lens[b] : 0;
  if (act == 0) return;
  a.out_tok[b] = fi;
  if (a.out_lp) a.out_lp[b] = lp;
  if (a.conf) { a.conf[2 * b] = c0 + __expf(lp); a.conf[2 * b + 1] = c1 + 1.f; }
  bool stop = (fi == a.eos0 || fi == a.eos1 || fi == a.eos2 || fi == a.eos3);
  if (a.hist) {
    const int gi = pos - st;
    if (gi >= 0 && gi < a.hist_ld) a.hist[(size_t)b * a.hist_ld + gi] = fi;
    if (gi + 1 >= a.hist_ld) stop = true;
  }
  if (a.pos) a.pos[b] = pos + 1;
  if (a.lens) a.lens[b] = len + 1;
  if (stop && a.active) a.active[b] = 0;
}

__device__ __forceinline__ float logit_f(bf16_t x) { return bf2f(x); }
__device__ __forceinline__ float logit_f(float x) { return x; }
