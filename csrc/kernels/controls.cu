// Logit controls: the token state of the requests and its use on the logits (formulas in controls.h).
#include <cuda_runtime.h>

#include "../include/sm100.cuh"
#include "controls.h"

namespace meshy {

namespace {

constexpr int kThreads = 64;

__device__ __forceinline__ int64_t slot_of(SlotIds s, int i) {
  return s.wide ? reinterpret_cast<const int64_t*>(s.p)[i] : (int64_t) reinterpret_cast<const int*>(s.p)[i];
}

// ─── token state ───────────────────────────────────────────────────────────
// A row's counts are 4 V bytes that have to be written whatever its tokens are (608 KB at V = 151936), its tokens 8
// bytes each. A cluster of eight CTAs clears the row, an eighth each, and after a cluster barrier adds the tokens, an
// eighth each, with one reduction in L2 per token and bit (integers: the order does not matter). 64 rows of up to
// 16384 tokens take 15 us: the clearing 6, then 1.3 M reductions. Counting spans of the row in shared memory instead
// made every CTA read all tokens (22 us), and so did keeping the bits there, across the cluster (22).
constexpr int kCluster = 8;
constexpr int kLoadThreads = 256;

__global__ void __launch_bounds__(kLoadThreads) __cluster_dims__(kCluster, 1, 1)
    load_tokens_kernel(ControlsView c, SlotIds slots, const int64_t* __restrict__ tokens, int64_t total,
                       const int* __restrict__ cu, const int* __restrict__ n_prompt) {
  const int i = blockIdx.y, at = blockIdx.x * kLoadThreads + threadIdx.x;
  constexpr int kAll = kCluster * kLoadThreads;
  pdl_wait();
  pdl_trigger();
  const int64_t slot = slot_of(slots, i);
  if (slot < 0 || slot >= c.R) return;  // all CTAs of the cluster
  int* counts = c.counts + slot * c.V;
  uint32_t* seen = c.seen + slot * c.W;
  const int64_t t0 = max(0, cu[i]);
  const int n = (int)(min((int64_t)cu[i + 1], total) - t0), np = n_prompt[i];
  const int head = min(c.V, (int)((16 - reinterpret_cast<uintptr_t>(counts) % 16) % 16 / 4)), body = (c.V - head) / 4;
  for (int v = at; v < body; v += kAll) reinterpret_cast<int4*>(counts + head)[v] = make_int4(0, 0, 0, 0);
  if (at < head) counts[at] = 0;
  if (at < c.V - head - 4 * body) counts[head + 4 * body + at] = 0;
  for (int v = at; v < c.W; v += kAll) seen[v] = 0u;
  cluster_sync_all();
#pragma unroll 4
  for (int j = at; j < n; j += kAll) {
    const int64_t v = tokens[t0 + j];
    if (v < 0 || v >= c.V) continue;
    atomicOr(&seen[v / 32], 1u << (v % 32));
    if (j >= np) atomicAdd(&counts[v], 1);
  }
}

// ─── controls ──────────────────────────────────────────────────────────────
// A CTA owns kChunk entries of one row (whole words of both bit rows). Few tokens of a vocabulary have occurred (some
// thousands of 150 thousand), so the work is split: a dense pass copies the logits and writes -inf where the mask
// forbids, with nothing but 16-byte loads and stores; then each thread looks at 16 bits of the seen row and rewrites
// the entries that are set, from their logits and counts. In place the dense pass touches masked entries only, so a
// call costs V / 8 bytes a bit row and what it changes.
// A CTA is a chain of four dependent reads (slot, the row's settings and bits, counts, the entry a bias lands on), so
// the call is bound by how many CTAs are under way: small ones (64 threads: 41.8 us on 256 rows of 128256 bf16 logits,
// 128: 43.3, 256: 48), two seen entries at a time (four: 44.4, for its registers), logits kept as they are stored
// until they are written, biases read at the start. 41.8 us is 4.9 TB/s of the 204 MB that have to move; 64 rows of
// 151936 fp32 logits take 17.8 us (4.5 TB/s).
constexpr int kChunk = 16 * kThreads;

__device__ __forceinline__ float entry(const float* p) { return *p; }
__device__ __forceinline__ float entry(const bf16* p) { return __bfloat162float(*p); }

// E neighbouring logits as they are stored; widened when they are used
template <typename T, int E>
struct Entries;
template <int E>
struct Entries<float, E> {
  float x[E];
  __device__ __forceinline__ void load(const float* p) {
    if constexpr (E == 4)
      *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
    else
      x[0] = *p;
  }
  __device__ __forceinline__ void widen(float* y) const {
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = x[e];
  }
};
template <int E>
struct Entries<bf16, E> {
  uint32_t x[(E + 1) / 2];
  __device__ __forceinline__ void load(const bf16* p) {
    if constexpr (E == 8)
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(p);
    else
      x[0] = *reinterpret_cast<const uint16_t*>(p);
  }
  __device__ __forceinline__ void widen(float* y) const {
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = __uint_as_float(e % 2 ? x[e / 2] & 0xFFFF0000u : x[e / 2] << 16);
  }
};

template <typename T, bool IN_PLACE, bool VEC>
__global__ void __launch_bounds__(kThreads)
    controls_kernel(const T* logits, int64_t ls, ControlsView c, SlotIds slots, const int64_t* __restrict__ fresh,
                    const int* __restrict__ done, float* out, int64_t os) {
  const int b = blockIdx.y, v0 = blockIdx.x * kChunk, v1 = min(c.V, v0 + kChunk), tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();
  const T* z = logits + b * ls;
  float* o = out + b * os;
  constexpr int E = VEC ? (sizeof(T) == 4 ? 4 : 8) : 1, STEPS = kChunk / (E * kThreads), BATCH = STEPS < 4 ? STEPS : 4;
  constexpr uint32_t FIELD = (1u << E) - 1u;
  Entries<T, E> x[BATCH];
  auto load_batch = [&](int k0) {
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int v = v0 + ((k0 + k) * kThreads + tid) * E;
      if (v < v1) x[k].load(z + v);
    }
  };
  auto store = [&](int v, const float* y) {
    if constexpr (VEC) {
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<float4*>(o + v + e) = make_float4(y[e], y[e + 1], y[e + 2], y[e + 3]);
    } else {
      o[v] = y[0];
    }
  };
  if (!IN_PLACE) load_batch(0);  // on their way while the slot is looked up
  const int64_t slot = slot_of(slots, b);
  const bool on = slot >= 0 && slot < c.R;
  if (IN_PLACE && !on) return;
  const int64_t r = on ? slot : 0;
  int* counts = c.counts + r * c.V;
  uint32_t* seen = c.seen + r * c.W;
  const uint32_t* mask = c.mask + r * c.W;
  if (on && fresh) {
    const int64_t tok = done && done[b] ? -1 : fresh[b];
    const bool mine = tok >= v0 && tok < v1;
    if (mine && tid == 0) {
      counts[tok] += 1;
      seen[tok / 32] |= 1u << (tok % 32);
    }
    if (mine) __syncthreads();  // this CTA alone reads the token's count and word
  }
  const float rep = c.repetition[r], freq = c.frequency[r], pres = c.presence[r];
  const bool masked = on && c.mask_on[r] != 0;
  // this thread's bias, looked up early
  int bias_at = -1;
  float bias = 0.f;
  if (on && tid < c.K) {
    bias_at = c.bias_ids[r * c.K + tid];
    bias = c.bias_vals[r * c.K + tid];
  }
  // this thread's 16 entries of the sparse pass: seen, and allowed (the others stay -inf)
  const int w0 = v0 + 16 * tid;
  uint32_t bits = 0u;
  if (on && (rep != 1.f || freq != 0.f || pres != 0.f) && w0 < v1) {
    bits = (seen[w0 / 32] >> (w0 % 32)) & 0xFFFFu;
    if (v1 - w0 < 16) bits &= (1u << (v1 - w0)) - 1u;  // the last word's bits behind the vocabulary are no tokens
    if (masked) bits &= mask[w0 / 32] >> (w0 % 32);
  }
  if (masked) {
    for (int k0 = 0; k0 < STEPS; k0 += BATCH) {
      if (!IN_PLACE && k0 > 0) load_batch(k0);
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int v = v0 + ((k0 + k) * kThreads + tid) * E;
        if (v >= v1) break;
        const uint32_t m = (mask[v / 32] >> (v % 32)) & FIELD;
        if (IN_PLACE && m == FIELD) continue;
        if (IN_PLACE && m != 0u) x[k].load(z + v);
        float y[E];
        x[k].widen(y);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (!((m >> e) & 1u)) y[e] = -INFINITY;
        store(v, y);
      }
    }
  } else if (!IN_PLACE) {
    for (int k0 = 0; k0 < STEPS; k0 += BATCH) {
      if (k0 > 0) load_batch(k0);
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int v = v0 + ((k0 + k) * kThreads + tid) * E;
        if (v >= v1) break;
        float y[E];
        x[k].widen(y);
        store(v, y);
      }
    }
  }
  if (!on) return;
  __syncthreads();  // the dense pass of this chunk is written
  while (bits) {
    constexpr int N = 2;  // entries whose loads are under way together
    int v[N], n[N];
    float y[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = bits ? w0 + __ffs(bits) - 1 : -1;
      bits &= bits - 1u;
      if (v[i] >= 0) {
        n[i] = counts[v[i]];
        y[i] = entry(z + v[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (v[i] >= 0) {
        const float p = y[i] > 0.f ? y[i] / rep : y[i] * rep;
        o[v[i]] = p - freq * (float)n[i] - (n[i] > 0 ? pres : 0.f);
      }
  }
  if (c.K == 0) return;
  // biases, on what this CTA has written (ids of a row are distinct; a masked entry stays -inf)
  __syncthreads();
  if (bias_at >= v0 && bias_at < v1) o[bias_at] += bias;
  for (int j = tid + kThreads; j < c.K; j += kThreads) {
    const int v = c.bias_ids[r * c.K + j];
    if (v >= v0 && v < v1) o[v] += c.bias_vals[r * c.K + j];
  }
}

template <typename T>
void launch_controls(const void* logits, int64_t ls, ControlsView c, SlotIds slots, const int64_t* fresh,
                     const int* done, int B, float* out, int64_t os, cudaStream_t st) {
  const T* z = reinterpret_cast<const T*>(logits);
  const dim3 grid((c.V + kChunk - 1) / kChunk, B);
  // 16 bytes at a time where every row starts on such a boundary and ends on one: 41.8 us on 256 rows of 128256 bf16
  // logits where one at a time takes 56 (64 rows of 151936 fp32: 17.8, 20.2)
  const int e = 16 / sizeof(T);
  const bool vec = c.V % e == 0 && (B == 1 || (ls % e == 0 && os % 4 == 0)) &&
                   reinterpret_cast<uintptr_t>(logits) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
  const bool in_place = logits == out;
  auto go = [&](auto k) { launch_pdl(k, grid, dim3(kThreads), 0, st, z, ls, c, slots, fresh, done, out, os); };
  if (in_place)
    vec ? go(controls_kernel<T, true, true>) : go(controls_kernel<T, true, false>);
  else
    vec ? go(controls_kernel<T, false, true>) : go(controls_kernel<T, false, false>);
}

}  // namespace

void load_tokens(ControlsView c, SlotIds slots, const int64_t* tokens, int64_t total, const int* cu,
                 const int* n_prompt, int n, cudaStream_t st) {
  if (n == 0) return;
  MESHY_CHECK(n <= 65535, "load_tokens: at most 65535 rows");
  launch_pdl(load_tokens_kernel, dim3(kCluster, n), dim3(kLoadThreads), 0, st, c, slots, tokens, total, cu, n_prompt);
}

void apply_logit_controls(const void* logits, bool is_bf16, int64_t ls, ControlsView c, SlotIds slots,
                          const int64_t* fresh, const int* done, int B, float* out, int64_t os, cudaStream_t st) {
  if (B == 0) return;
  MESHY_CHECK(B <= 65535, "apply_logit_controls: at most 65535 rows");
  if (is_bf16)
    launch_controls<bf16>(logits, ls, c, slots, fresh, done, B, out, os, st);
  else
    launch_controls<float>(logits, ls, c, slots, fresh, done, B, out, os, st);
}

}  // namespace meshy
