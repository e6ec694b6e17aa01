// Logit controls of the rollout engine (controls.cu): penalties for repeated tokens, biases and token masks,
// and the per-request token state that the penalties read.
#pragma once
#include "../include/common.cuh"

namespace meshy {

// State of ``R`` request slots over a vocabulary of V (W = ceil(V / 32) words a row; entry v is bit v % 32 of word
// v / 32).
struct ControlsView {
  const float* repetition;  // [R], 1: off
  const float* frequency;   // [R], 0: off
  const float* presence;    // [R], 0: off
  uint32_t* seen;           // [R, W] token occurs in the prompt or was generated
  int* counts;              // [R, V] times the token was generated
  const int* bias_ids;      // [R, K], entries outside [0, V) unused; distinct within a row
  const float* bias_vals;   // [R, K]
  const uint32_t* mask;     // [R, W] token allowed
  const int* mask_on;       // [R] nonzero: the mask counts
  int64_t R;
  int V, W, K;
};

// Slot ids come as int32 or int64.
struct SlotIds {
  const void* p;
  bool wide;
};

// State of n requests from their ``total`` tokens so far: row i's are tokens[cu[i] .. cu[i + 1]), of which the first
// n_prompt[i] belong to the prompt. The rows of slots[i] are rewritten; other rows keep their state.
void load_tokens(ControlsView c, SlotIds slots, const int64_t* tokens, int64_t total, const int* cu,
                 const int* n_prompt, int n, cudaStream_t st);
// out[b, v] = penalised, biased and masked logits[b, v]. ``logits`` are fp32 or bf16 with row stride ls; ``out`` is
// fp32 with row stride os and may be ``logits`` itself. With ``fresh`` [B] the token fresh[b] is first counted as
// generated in slot slots[b] (unless it is negative, or done[b] is nonzero). A slot outside [0, R) has no controls.
void apply_logit_controls(const void* logits, bool is_bf16, int64_t ls, ControlsView c, SlotIds slots,
                          const int64_t* fresh, const int* done, int B, float* out, int64_t os, cudaStream_t st);

}  // namespace meshy
