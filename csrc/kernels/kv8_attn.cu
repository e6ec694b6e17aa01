// Paged decode attention over the 8-bit KV cache (layout in kv8.h).
//
//   s_j = scale a_j (q . n_j),  p = softmax(s),  o = sum_j p_j a'_j n'_j
//
// One CTA per row and query head; each warp takes every so manieth token with the running maximum and sum of its own,
// and the warps' states are joined at the end.
#include <cuda_runtime.h>

#include "kv8.h"

namespace meshy {

namespace {

constexpr int kWarps = 8;

template <int HD>
__global__ void __launch_bounds__(32 * kWarps)
    kv8_attn_kernel(const bf16* __restrict__ q, int64_t qs, int64_t qh, KV8View c, const int* __restrict__ bt,
                    int64_t bt_stride, int max_pages, const int* __restrict__ seq_lens, int Hq, float scale,
                    bf16* __restrict__ out) {
  constexpr int N = HD / 32;
  __shared__ float so[kWarps][HD], sm[kWarps], sl[kWarps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, h = blockIdx.x, b = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  const int hk = h / (Hq / c.Hkv);
  const int64_t n = min((int64_t)max(seq_lens[b], 0), (int64_t)max_pages * c.page);
  float x[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = __bfloat162float(q[b * qs + h * qh + lane * N + i]) * scale;
    o[i] = 0.f;
  }
  for (int64_t t = warp; t < n; t += kWarps) {
    const int64_t pg = bt[b * bt_stride + t / c.page];
    if (pg < 0 || pg >= c.n_pages) continue;
    const int64_t row = (pg * c.Hkv + hk) * c.page + t % c.page;
    const float* a = c.scale + row / kKV8Block * 2;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += x[i] * ((float)c.k[row * HD + lane * N + i] - 128.f);
    s = warp_sum(s) * a[0];
    const float to = fmaxf(m, s), keep = m == -INFINITY ? 0.f : __expf(m - to), p = __expf(s - to);
    m = to;
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * keep + p * a[1] * ((float)c.v[row * HD + lane * N + i] - 128.f);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) so[warp][lane * N + i] = o[i];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  for (int ch = threadIdx.x; ch < HD; ch += 32 * kWarps) {
    float M = -INFINITY, L = 0.f, y = 0.f;
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[w]);
    for (int w = 0; w < kWarps; ++w) {
      const float e = sm[w] == -INFINITY ? 0.f : __expf(sm[w] - M);
      L += sl[w] * e;
      y += so[w][ch] * e;
    }
    out[((int64_t)b * Hq + h) * HD + ch] = __float2bfloat16(L == 0.f ? 0.f : y / L);
  }
}

}  // namespace

void kv8_attention(const bf16* q, int64_t qs, int64_t qh, KV8View c, const int* bt, int64_t bt_stride, int max_pages,
                   const int* seq_lens, int B, int Hq, float scale, bf16* out, cudaStream_t st) {
  if (B == 0) return;
  launch_pdl(c.hd == 128 ? kv8_attn_kernel<128> : kv8_attn_kernel<64>, dim3(Hq, B), dim3(32 * kWarps), 0, st, q, qs, qh,
             c, bt, bt_stride, max_pages, seq_lens, Hq, scale, out);
}

}  // namespace meshy
