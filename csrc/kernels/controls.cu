// Logit controls: the token state of the requests and its use on the logits (formulas in controls.h).
#include <cuda_runtime.h>

#include "controls.h"

namespace meshy {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ int64_t slot_of(SlotIds s, int i) {
  return s.wide ? reinterpret_cast<const int64_t*>(s.p)[i] : (int64_t) reinterpret_cast<const int*>(s.p)[i];
}

// One CTA per request: clear the row, then one atomic per token (integers: the order does not matter).
__global__ void __launch_bounds__(1024)
    load_tokens_kernel(ControlsView c, SlotIds slots, const int64_t* __restrict__ tokens, int64_t total,
                       const int* __restrict__ cu, const int* __restrict__ n_prompt) {
  const int i = blockIdx.x;
  const int64_t slot = slot_of(slots, i);
  if (slot < 0 || slot >= c.R) return;
  uint32_t* seen = c.seen + slot * c.W;
  int* counts = c.counts + slot * c.V;
  for (int v = threadIdx.x; v < c.W; v += blockDim.x) seen[v] = 0u;
  for (int v = threadIdx.x; v < c.V; v += blockDim.x) counts[v] = 0;
  __syncthreads();
  const int64_t t0 = max(0, cu[i]);
  const int n = (int)(min((int64_t)cu[i + 1], total) - t0), np = n_prompt[i];
  for (int j = threadIdx.x; j < n; j += blockDim.x) {
    const int64_t tok = tokens[t0 + j];
    if (tok < 0 || tok >= c.V) continue;
    atomicOr(&seen[tok / 32], 1u << (tok % 32));
    if (j >= np) atomicAdd(&counts[tok], 1);
  }
}

// One CTA per row.
__global__ void __launch_bounds__(1024)
    controls_kernel(const void* __restrict__ logits, bool is_bf16, int64_t ls, ControlsView c, SlotIds slots,
                    const int64_t* __restrict__ fresh, const int* __restrict__ done, float* __restrict__ out,
                    int64_t os) {
  const int b = blockIdx.x;
  const int64_t slot = slot_of(slots, b);
  const bool on = slot >= 0 && slot < c.R;
  const int64_t r = on ? slot : 0;
  if (on && fresh && threadIdx.x == 0 && !(done && done[b])) {
    const int64_t tok = fresh[b];
    if (tok >= 0 && tok < c.V) {
      c.counts[r * c.V + tok] += 1;
      c.seen[r * c.W + tok / 32] |= 1u << (tok % 32);
    }
  }
  __syncthreads();
  for (int v = threadIdx.x; v < c.V; v += blockDim.x) {
    float z = is_bf16 ? __bfloat162float(reinterpret_cast<const bf16*>(logits)[b * ls + v])
                      : reinterpret_cast<const float*>(logits)[b * ls + v];
    if (on) {
      if ((c.seen[r * c.W + v / 32] >> (v % 32)) & 1u) {
        const float rep = c.repetition[r];
        const float n = (float)c.counts[r * c.V + v];
        z = z > 0.f ? z / rep : z * rep;
        z = z - c.frequency[r] * n - (n > 0.f ? c.presence[r] : 0.f);
      }
      for (int j = 0; j < c.K; ++j)
        if (c.bias_ids[r * c.K + j] == v) z += c.bias_vals[r * c.K + j];
      if (c.mask_on[r] && !((c.mask[r * c.W + v / 32] >> (v % 32)) & 1u)) z = -INFINITY;
    }
    out[b * os + v] = z;
  }
}

}  // namespace

void load_tokens(ControlsView c, SlotIds slots, const int64_t* tokens, int64_t total, const int* cu, const int* n_prompt, int n,
                 cudaStream_t st) {
  if (n == 0) return;
  load_tokens_kernel<<<n, 1024, 0, st>>>(c, slots, tokens, total, cu, n_prompt);
  MESHY_CUDA_CHECK(cudaGetLastError());
}

void apply_logit_controls(const void* logits, bool is_bf16, int64_t ls, ControlsView c, SlotIds slots,
                          const int64_t* fresh, const int* done, int B, float* out, int64_t os, cudaStream_t st) {
  if (B == 0) return;
  controls_kernel<<<B, 1024, 0, st>>>(logits, is_bf16, ls, c, slots, fresh, done, out, os);
  MESHY_CUDA_CHECK(cudaGetLastError());
}

}  // namespace meshy
