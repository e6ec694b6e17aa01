// Paged decode attention over the 4-bit KV cache (layout in kv4.h).
//
//   s_j = scale * sum_g (a_jg (q_g . n_jg) + z_jg sum(q_g)),  p = softmax(s),  o = sum_j p_j (a'_jg n'_j + z'_jg)
//
// The scale and the base of a group leave the channel sums, so the nibbles go to the tensor cores as whole numbers:
// masked in place they are fp16 subnormals (n at bits 0-3 is n 2^-24, at bits 4-7 n 2^-20), exact and with no
// conversion. The power of two is divided out of Q (four of every eight channels carry 1/16) and of the result.
//
// One warp takes 16 tokens at a time (m16n8k16, fp16 in, fp32 sums):
//   S^T [16 tokens, 8 heads] = K [16, hd] Q^T      A rows are tokens: a lane's 16 bytes of a K row are its A registers
//   O^T [16 channels, 8 heads] += V^T [16, 16 tokens] P^T    A rows are channels: two byte permutes pair the tokens
// Query heads that share a KV head fill the 8 columns, so every cached byte is read once for up to 8 heads, straight
// from global memory to registers: nothing passes through shared memory, P changes from accumulator to operand by
// movmatrix. tcgen05 would not help here: operands unpacked in registers would have to be stored to shared or tensor
// memory first, and at 8 query rows the matrix work is a fraction of the unpacking.
//
// P carries the scale of V (x = p a'), so it is kept in fp16's range by a reference (m, A) per warp: x = 64 p a' / A
// with p relative to m. The reference moves only when some x passes 2^15 (then to the true maxima), so most
// tiles take neither the maximum's shuffles nor a rescaling; what falls below fp16's smallest number is less than
// 2^-31 of the largest term.
//
// Work split: the (row, KV head, up to 8 query heads) segments are laid end to end in units of 16 tokens and every
// CTA takes an equal share of the sum, whatever the lengths: the lengths are read on the device, a captured graph
// follows them. A segment that spans CTAs leaves partial sums in a workspace; the last CTA to arrive joins them in
// CTA order, so results do not depend on timing.
#include <cuda_runtime.h>

#include "kv4.h"

namespace meshy {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTok = 16;     // tokens of a tile
constexpr int kHeads = 8;    // query heads of a segment
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBoost = 64.f, kLimit = 32768.f;
constexpr float kMinA = 5.9604645e-8f;  // 2^-24, the smallest fp16

template <int HD>
struct Tile {  // one lane's share of 16 tokens
  uint32_t k[2][HD / 32];     // tokens g, g + 8: words (HD / 32) t ..
  uint32_t v[4][HD / 64];     // tokens 2t, 2t + 1, 2t + 8, 2t + 9: words (HD / 64) g ..
  uint32_t s[2][HD / 32];     // tokens g, g + 8: (a, z) pairs of K's groups, then V's
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t* d, const void* p) {
  if constexpr (N == 4)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "l"(p));
  else if constexpr (N == 2)
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "l"(p));
  else
    asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(d[0]) : "l"(p));
}

__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half2(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }

__device__ __forceinline__ float max_over_rows(float v) {  // over the lanes that share lane % 4
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float sum_over_rows(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Args {
  const bf16* q;
  int64_t qs, qh;
  KV4View c;
  const int* bt;
  int64_t bt_stride;
  int max_pages;
  const int* seq_lens;
  int B, Hq, rep, blocks;  // blocks: groups of kHeads query heads per KV head
  float scale;
  bf16* out;
  float* part;         // [2 CTAs][kHeads][hd + 2]
  unsigned* arrived;   // [segments], zero between launches
};

__device__ __forceinline__ int tokens_of(const Args& a, int b) {
  const int64_t cap = (int64_t)a.max_pages * a.c.page;
  const int n = a.seq_lens[b];
  return n <= 0 ? 0 : (int)min((int64_t)n, cap);
}
__device__ __forceinline__ int tiles_of(int n) { return max(1, (n + kTok - 1) / kTok); }  // an empty row writes its zeros

template <int HD>
__global__ void __launch_bounds__(kThreads, 2) kv4_attn_kernel(const Args a) {
  constexpr int G = HD / 64;
  constexpr int KW = HD / 32;       // K words a lane takes of a row
  constexpr int LD = HD + 4;        // row stride of the merge buffer: spreads the heads over the banks
  __shared__ float so[kWarps][kHeads][LD];
  __shared__ float sm[kWarps][kHeads], sl[kWarps][kHeads];
  __shared__ long long scan[kWarps];
  __shared__ int s_row;
  __shared__ long long s_at;
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int per_row = a.c.Hkv * a.blocks;  // segments of a row

  pdl_wait();
  pdl_trigger();

  // total tiles, and this CTA's share [at, end)
  long long mine = 0;
  for (int b = tid; b < a.B; b += kThreads) mine += tiles_of(tokens_of(a, b));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) scan[warp] = mine;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += scan[w];
  total *= per_row;
  const long long n_cta = min((long long)gridDim.x, (total + kWarps - 1) / kWarps);
  if (blockIdx.x >= n_cta) return;
  long long at = blockIdx.x * total / n_cta;
  const long long end = (blockIdx.x + 1) * total / n_cta;
  // the row that holds tile ``at``
  long long base = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    const int b = b0 + tid;
    const long long n = b < a.B ? (long long)tiles_of(tokens_of(a, b)) * per_row : 0;
    long long incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    long long before = base;
    for (int w = 0; w < warp; ++w) before += scan[w];
    if (at >= before + incl - n && at < before + incl) {
      s_row = b;
      s_at = before + incl - n;
    }
    for (int w = 0; w < kWarps; ++w) base += scan[w];
    if (base > at) break;
  }
  __syncthreads();
  int b = s_row;
  int n_tok = tokens_of(a, b), U = tiles_of(n_tok);
  int hseg = (int)((at - s_at) / U);
  long long seg0 = s_at + (long long)hseg * U;  // first tile of the segment

  const int ppt = a.c.page / kTok;  // tiles of a page
  const float sl2 = a.scale * kLog2e;

  while (at < end) {
    const int hk = hseg / a.blocks, h0 = (hseg % a.blocks) * kHeads;
    const int nh = min(kHeads, a.rep - h0);
    const int first = (int)(at - seg0);
    const int last = (int)min((long long)U, end - seg0);

    // Q fragments: head g, channels of the words this lane reads of a K row; scaled so that the largest is in [2^14, 2^15)
    uint32_t qf[KW][4];
    float cs[2], qs[2][G];
    {
      float x[KW][8], mx = 0.f, sum[G];
#pragma unroll
      for (int i = 0; i < G; ++i) sum[i] = 0.f;
      const bf16* src = a.q + b * a.qs + (int64_t)(hk * a.rep + h0 + g) * a.qh;
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        const int w = KW * t + j;
        uint4 u = make_uint4(0, 0, 0, 0);
        if (g < nh) u = *reinterpret_cast<const uint4*>(src + 64 * (w % G) + 8 * (w / G));
        const uint32_t us[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = unpack_bf16x2(us[e]);
          x[j][2 * e] = f.x;
          x[j][2 * e + 1] = f.y;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          mx = fmaxf(mx, fabsf(x[j][e]));
          sum[j % G] += x[j][e];
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
#pragma unroll
        for (int i = 0; i < G; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
      }
      const int ex = (mx > 0.f && mx < INFINITY) ? min(14 - ilogbf(mx), 126) : 0;
      const float f = ldexpf(1.f, ex), c = ldexpf(sl2, 24 - ex);
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        qf[j][0] = pack_half2(x[j][0] * f, x[j][4] * f);
        qf[j][1] = pack_half2(x[j][1] * f * 0.0625f, x[j][5] * f * 0.0625f);
        qf[j][2] = pack_half2(x[j][2] * f, x[j][6] * f);
        qf[j][3] = pack_half2(x[j][3] * f * 0.0625f, x[j][7] * f * 0.0625f);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        cs[r] = __shfl_sync(0xffffffffu, c, (2 * t + r) * 4);
#pragma unroll
        for (int i = 0; i < G; ++i) qs[r][i] = __shfl_sync(0xffffffffu, sum[i], (2 * t + r) * 4) * sl2;
      }
    }

    float o[G][4][4], z[G][2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, A[G], inv[G];
    bool fresh = true;
#pragma unroll
    for (int i = 0; i < G; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
      z[i][0] = z[i][1] = 0.f;
      A[i] = kMinA;
      inv[i] = kBoost / kMinA;
    }

    const int* row_bt = a.bt + b * a.bt_stride;
    auto page_of = [&](int tile) -> int {
      if (tile >= last || tile * kTok >= n_tok) return -1;
      const int p = row_bt[tile / ppt];
      return p < a.c.n_pages ? p : -1;
    };
    auto load = [&](Tile<HD>& x, int tile, int page) {
      if (page < 0) return;
      const int64_t r = ((int64_t)page * a.c.Hkv + hk) * a.c.page + (tile % ppt) * kTok;
      const uint8_t* kp = a.c.k + r * (HD / 2);
      const uint8_t* vp = a.c.v + r * (HD / 2);
      const __half2* sp = a.c.scale + r * (2 * G);
#pragma unroll
      for (int i = 0; i < 2; ++i) load_words<KW>(x.k[i], kp + (g + 8 * i) * (HD / 2) + t * (4 * KW));
#pragma unroll
      for (int i = 0; i < 2; ++i) load_words<2 * G>(x.s[i], sp + (g + 8 * i) * (2 * G));
#pragma unroll
      for (int i = 0; i < 4; ++i) load_words<G>(x.v[i], vp + (2 * t + (i & 1) + 8 * (i >> 1)) * (HD / 2) + g * (4 * G));
    };
    auto compute = [&](Tile<HD>& x, int tile, int page) {
      if (page < 0) return;
      float acc[G][4];
#pragma unroll
      for (int i = 0; i < G; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        uint32_t w0 = x.k[0][j], w1 = x.k[1][j];
        mma_f16(acc[j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[j][0], qf[j][1]);
        w0 >>= 8;
        w1 >>= 8;
        mma_f16(acc[j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[j][2], qf[j][3]);
      }
      if (tile * kTok + kTok > n_tok) {  // the row ends inside this tile: what lies behind may be anything
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (tile * kTok + g + 8 * i >= n_tok) {
#pragma unroll
            for (int j = 0; j < 2 * G; ++j) x.s[i][j] = 0u;
          }
      }
      // scores: [token g + 8 i][head 2 t + r], base 2, relative to the reference
      float s[2][2], va[2][G], vz[2][G];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float e[2] = {0.f, 0.f}, d[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const float2 k2 = unpack_half2(x.s[i][j]), v2 = unpack_half2(x.s[i][G + j]);
          va[i][j] = v2.x;
          vz[i][j] = v2.y;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            d[r] = fmaf(k2.x, acc[j][2 * i + r], d[r]);
            e[r] = fmaf(k2.y, qs[r][j], e[r]);
          }
        }
        const bool in = tile * kTok + g + 8 * i < n_tok;
#pragma unroll
        for (int r = 0; r < 2; ++r) s[i][r] = in ? fmaf(cs[r], d[r], e[r]) : -INFINITY;
      }
      float p[2][2], y[2][2][G], top = 0.f;
      bool bad = fresh;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          p[i][r] = ex2(s[i][r] - m[r]);
          top = fmaxf(top, p[i][r]);  // of its own: a' may be 0
#pragma unroll
          for (int j = 0; j < G; ++j) {
            y[i][r][j] = p[i][r] * (va[i][j] * inv[j]);
            top = fmaxf(top, y[i][r][j]);
          }
        }
      bad |= !(top <= kLimit);
      if (__any_sync(0xffffffffu, bad)) {
        // move the reference to the true maxima
        fresh = false;
        float keep[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float mn = fmaxf(m[r], max_over_rows(fmaxf(s[0][r], s[1][r])));
          keep[r] = mn == -INFINITY ? 1.f : ex2(m[r] - mn);
          m[r] = mn;
          l[r] *= keep[r];
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const float An = fmaxf(A[j], max_over_rows(fmaxf(va[0][j], va[1][j])));
          const float f = A[j] / An;
          A[j] = An;
          inv[j] = kBoost / An;
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][q][e] *= f * keep[e & 1];
          z[j][0] *= keep[0];
          z[j][1] *= keep[1];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            p[i][r] = m[r] == -INFINITY && s[i][r] == -INFINITY ? 0.f : ex2(s[i][r] - m[r]);
#pragma unroll
            for (int j = 0; j < G; ++j) y[i][r][j] = p[i][r] * (va[i][j] * inv[j]);
          }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += p[0][r] + p[1][r];
#pragma unroll
        for (int j = 0; j < G; ++j) z[j][r] = fmaf(p[0][r], vz[0][j], fmaf(p[1][r], vz[1][j], z[j][r]));
      }
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const uint32_t b0 = transpose8x8(pack_half2(y[0][0][j], y[0][1][j]));
        const uint32_t b1 = transpose8x8(pack_half2(y[1][0][j], y[1][1][j]));
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // channels 8 g + 4 half ..
          const uint32_t sel = half ? 0x7632u : 0x5410u;
          uint32_t x01 = __byte_perm(x.v[0][j], x.v[1][j], sel), x23 = __byte_perm(x.v[2][j], x.v[3][j], sel);
          mma_f16(o[j][2 * half], x01 & 0x000F000Fu, x01 & 0x00F000F0u, x23 & 0x000F000Fu, x23 & 0x00F000F0u, b0, b1);
          x01 >>= 8;
          x23 >>= 8;
          mma_f16(o[j][2 * half + 1], x01 & 0x000F000Fu, x01 & 0x00F000F0u, x23 & 0x000F000Fu, x23 & 0x00F000F0u, b0, b1);
        }
      }
    };

    // a tile in flight while the one before it is computed, its page id one step ahead
    {
      int tile = first + warp;
      int page = page_of(tile), next = page_of(tile + kWarps);
      Tile<HD> x0, x1;
      load(x0, tile, page);
      while (tile < last) {
        int ahead = page_of(tile + 2 * kWarps);
        load(x1, tile + kWarps, next);
        compute(x0, tile, page);
        tile += kWarps;
        page = next;
        next = ahead;
        if (tile >= last) break;
        ahead = page_of(tile + 2 * kWarps);
        load(x0, tile + kWarps, next);
        compute(x1, tile, page);
        tile += kWarps;
        page = next;
        next = ahead;
      }
    }

    // the warp's state: o in units of V, relative to m
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] = sum_over_rows(l[r]);
#pragma unroll
      for (int j = 0; j < G; ++j) {
        z[j][r] = sum_over_rows(z[j][r]);
        const float f0 = A[j] * (16777216.f / kBoost), f1 = A[j] * (1048576.f / kBoost);
        float x[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          x[2 * q] = fmaf(o[j][q][r], f0, z[j][r]);
          x[2 * q + 1] = fmaf(o[j][q][2 + r], f1, z[j][r]);
        }
        float4* d = reinterpret_cast<float4*>(&so[warp][2 * t + r][64 * j + 8 * g]);
        d[0] = make_float4(x[0], x[1], x[2], x[3]);
        d[1] = make_float4(x[4], x[5], x[6], x[7]);
      }
      if (g == 0) {
        sm[warp][2 * t + r] = m[r];
        sl[warp][2 * t + r] = l[r];
      }
    }
    __syncthreads();
    // join the warps; a whole segment is done, a piece of one goes to the workspace
    const bool whole = first == 0 && last == U;
    const int slot = 2 * blockIdx.x + (first == 0 ? 1 : 0);
    bf16* dst = a.out + ((int64_t)b * a.Hq + hk * a.rep + h0) * HD;
    for (int i = tid; i < nh * (HD / 2); i += kThreads) {
      const int h = i / (HD / 2), ch = 2 * (i % (HD / 2));
      float M = -INFINITY, L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[w][h]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = sm[w][h] == -INFINITY ? 0.f : ex2(sm[w][h] - M);
        L = fmaf(sl[w][h], f, L);
        x = fmaf(so[w][h][ch], f, x);
        y = fmaf(so[w][h][ch + 1], f, y);
      }
      if (whole) {
        const float f = L == 0.f ? 0.f : 1.f / L;
        *reinterpret_cast<uint32_t*>(dst + (int64_t)h * HD + ch) = pack_bf16x2(x * f, y * f);
      } else {
        float* pp = a.part + ((int64_t)slot * kHeads + h) * (HD + 2);
        *reinterpret_cast<float2*>(pp + ch) = make_float2(x, y);
        if (ch == 0) *reinterpret_cast<float2*>(pp + HD) = make_float2(M, L);
      }
    }
    if (!whole) {
      const long long c0 = ((seg0 + 1) * n_cta - 1) / total, c1 = ((seg0 + U) * n_cta - 1) / total;
      unsigned* ctr = a.arrived + (int64_t)b * per_row + hseg;
      __threadfence();
      __syncthreads();
      if (tid == 0) s_last = atomicAdd(ctr, 1u) == (unsigned)(c1 - c0);
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int i = tid; i < nh * (HD / 2); i += kThreads) {
          const int h = i / (HD / 2), ch = 2 * (i % (HD / 2));
          float M = -INFINITY, L = 0.f, x = 0.f, y = 0.f;
          for (long long c = c0; c <= c1; ++c) {
            const float* pp = a.part + ((2 * c + (c == c0 ? 1 : 0)) * kHeads + h) * (HD + 2);
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(pp + HD));
            const float2 v = __ldcg(reinterpret_cast<const float2*>(pp + ch));
            if (ml.x == -INFINITY && ml.y == 0.f) continue;
            const float Mn = fmaxf(M, ml.x), f = ex2(M - Mn), e = ex2(ml.x - Mn);
            L = L * f + ml.y * e;
            x = x * f + v.x * e;
            y = y * f + v.y * e;
            M = Mn;
          }
          const float f = L == 0.f ? 0.f : 1.f / L;
          *reinterpret_cast<uint32_t*>(dst + (int64_t)h * HD + ch) = pack_bf16x2(x * f, y * f);
        }
        if (tid == 0) *ctr = 0u;
      }
    }
    __syncthreads();  // the merge buffer is free
    at = seg0 + last;
    if (at < end) {
      seg0 += U;
      if (++hseg == per_row) {
        hseg = 0;
        ++b;
        n_tok = tokens_of(a, b);
        U = tiles_of(n_tok);
      }
    }
  }
}

int sm_count() {
  static int n[64] = {};
  int dev = 0;
  MESHY_CUDA_CHECK(cudaGetDevice(&dev));
  if (!n[dev]) MESHY_CUDA_CHECK(cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev));
  return n[dev];
}

}  // namespace

int kv4_attention_ctas() { return 2 * sm_count(); }
int64_t kv4_attention_segments(int B, int Hq, int Hkv) { return (int64_t)B * Hkv * ((Hq / Hkv + kHeads - 1) / kHeads); }

void kv4_attention(const bf16* q, int64_t qs, int64_t qh, KV4View c, const int* bt, int64_t bt_stride, int max_pages,
                   const int* seq_lens, int B, int Hq, float scale, bf16* out, float* part, unsigned* arrived,
                   cudaStream_t st) {
  if (B == 0) return;
  const int rep = Hq / c.Hkv;
  const Args a{q,  qs,    qh,  c,    bt,     bt_stride, max_pages, seq_lens, B, Hq, rep, (rep + kHeads - 1) / kHeads, scale,
               out, part, arrived};
  const int grid = kv4_attention_ctas();
  if (c.hd == 128)
    launch_pdl(kv4_attn_kernel<128>, dim3(grid), dim3(kThreads), 0, st, a);
  else
    launch_pdl(kv4_attn_kernel<64>, dim3(grid), dim3(kThreads), 0, st, a);
}

}  // namespace meshy
