// Paged decode attention over the 4-bit KV cache (layout in kv4.h).
//
// s_j = scale * q . (a_j n_j + z_j), p = softmax(s), o = sum_j p_j (a'_j n'_j + z'_j), one pass over the tokens with
// the running maximum and sum of the softmax. One CTA per (row, query head): a thread scores one token of a
// 128-token tile, then sums its channel of V over the tile.
#include <cuda_runtime.h>

#include "kv4.h"

namespace meshy {

namespace {

constexpr int kTile = 128;

__device__ __forceinline__ float block_max(float v, float* sh) {
  v = warp_max(v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sh[threadIdx.x / 32] = v;
  __syncthreads();
  return fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}

__global__ void __launch_bounds__(kTile)
    kv4_attn_kernel(const bf16* __restrict__ q, int64_t qs, int64_t qh, KV4View c, const int* __restrict__ bt,
                    int64_t bt_stride, int max_pages, const int* __restrict__ seq_lens, int Hq, float scale,
                    bf16* __restrict__ out) {
  __shared__ float qv[128], qsum[2], p[kTile], sh[4];
  __shared__ int64_t rows[kTile];
  const int b = blockIdx.x, hq = blockIdx.y, tid = threadIdx.x;
  const int h = hq / (Hq / c.Hkv), hd = c.hd, G = hd / 64;
  const int L = (int)min((int64_t)seq_lens[b], (int64_t)max_pages * c.page);
  if (tid < hd) qv[tid] = __bfloat162float(q[b * qs + hq * qh + tid]);
  __syncthreads();
  if (tid < G) {
    float s = 0.f;
    for (int i = 0; i < 64; ++i) s += qv[tid * 64 + i];
    qsum[tid] = s;
  }
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int t0 = 0; t0 < L; t0 += kTile) {
    const int t = t0 + tid;
    int64_t row = -1;
    if (t < L) {
      const int64_t pg = bt[b * bt_stride + t / c.page];
      if (pg >= 0 && pg < c.n_pages) row = (pg * c.Hkv + h) * c.page + t % c.page;
    }
    __syncthreads();  // qsum; p and rows of the last tile are read
    float s = -INFINITY;
    if (row >= 0) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(c.k + row * (hd / 2));
      s = 0.f;
      for (int grp = 0; grp < G; ++grp) {
        float dot = 0.f;
        for (int u = 0; u < 8; ++u) {
          const uint32_t x = w[u * G + grp];
          for (int e = 0; e < 8; ++e) dot += (float)((x >> (4 * e)) & 15u) * qv[grp * 64 + u * 8 + e];
        }
        const float2 az = __half22float2(c.scale[row * 2 * G + grp]);
        s += az.x * dot + az.y * qsum[grp];
      }
      s *= scale;
    }
    const float m2 = fmaxf(m, block_max(s, sh));
    const float keep = m2 == -INFINITY ? 1.f : expf(m - m2);
    p[tid] = s == -INFINITY ? 0.f : expf(s - m2);
    rows[tid] = row;
    m = m2;
    l *= keep;
    o *= keep;
    __syncthreads();
    const int n = min(kTile, L - t0);
    for (int j = 0; j < n; ++j) {
      l += p[j];
      if (tid < hd && rows[j] >= 0) {
        const int grp = tid / 64, ch = tid % 64;
        const uint32_t x = reinterpret_cast<const uint32_t*>(c.v + rows[j] * (hd / 2))[(ch / 8) * G + grp];
        const float2 az = __half22float2(c.scale[(rows[j] * 2 + 1) * G + grp]);
        o += p[j] * ((float)((x >> (4 * (ch % 8))) & 15u) * az.x + az.y);
      }
    }
  }
  if (tid < hd) out[((int64_t)b * Hq + hq) * hd + tid] = __float2bfloat16(l != 0.f ? o / l : 0.f);
}

}  // namespace

void kv4_attention(const bf16* q, int64_t qs, int64_t qh, KV4View c, const int* bt, int64_t bt_stride, int max_pages,
                   const int* seq_lens, int B, int Hq, float scale, bf16* out, cudaStream_t st) {
  if (B == 0) return;
  kv4_attn_kernel<<<dim3(B, Hq), kTile, 0, st>>>(q, qs, qh, c, bt, bt_stride, max_pages, seq_lens, Hq, scale, out);
  MESHY_CUDA_CHECK(cudaGetLastError());
}

}  // namespace meshy
