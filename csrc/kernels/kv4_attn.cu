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
// Query heads that share a KV head fill the 8 columns, so every cached byte is read once for up to 8 heads. P changes
// from accumulator to operand by movmatrix. Each warp keeps a ring of kStages tiles of its own in shared memory, filled
// by 16-byte asynchronous copies, so three tiles are on their way while one is computed and no warp waits for
// another; V's 16-byte chunks are swizzled on the way in (a lane reads 8 bytes of every second token). tcgen05 would not help here: operands unpacked in registers would have to be stored to shared or tensor
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

#include "../include/sm100.cuh"
#include "kv4.h"

namespace meshy {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTok = 16;     // tokens of a tile
constexpr int kHeads = 8;    // query heads of a segment
constexpr int kStages = 4;   // tiles of a warp's ring
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBoost = 64.f;               // x of the largest p and a' right after the reference moved
constexpr float kMaxP = 128.f, kMaxW = 256.f;  // x = p w stays below 2^15
constexpr float kMinA = 5.9604645e-8f;  // 2^-24, the smallest fp16

template <int HD>
struct Ring {  // one stage: 16 tokens of one head
  static constexpr int ROW = HD / 2;             // nibble bytes of a token
  static constexpr int K = 0, V = kTok * ROW, S = 2 * kTok * ROW;
  static constexpr int BYTES = 2 * kTok * ROW + kTok * (HD / 8);  // the pairs take an eighth of the nibbles' bytes
  static constexpr int WARP = kStages * BYTES;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Byte of 16-byte chunk q of a tile's V rows: 128-byte lines, the chunk's place turned by the line, so that the lanes
// of one read (chunks of tokens 0, 2, 4, 6 or 1, 3, 5, 7) fall on different banks.
template <int HD>
__device__ __forceinline__ int v_chunk(int q) {
  return (q / 8) * 128 + ((q % 8) ^ (2 * ((q / 8) % (HD / 32)))) * 16;
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t* d, uint32_t p) {
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(p));
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "r"(p));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(d[0]) : "r"(p));
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
  int ppt;                 // tiles of a page
  int page_bytes;          // nibble bytes of a page, all heads
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

// A CTA's walk over its share of the tiles: segment (b, h), of whose U tiles it has [first, last); ``left`` tiles of the
// share remain from ``first`` on.
struct Walk {
  int b, h, n, U, first, last, left;
  __device__ __forceinline__ void enter(const Args& a) {
    n = tokens_of(a, b);
    U = tiles_of(n);
    last = min(U, first + left);
  }
  __device__ __forceinline__ bool next(const Args& a) {
    left -= last - first;
    if (left <= 0) return false;
    first = 0;
    if (++h == a.c.Hkv * a.blocks) {
      h = 0;
      ++b;
      n = tokens_of(a, b);
      U = tiles_of(n);
    }
    last = min(U, left);
    return true;
  }
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 2) kv4_attn_kernel(const Args a) {
  constexpr int G = HD / 64;
  constexpr int KW = HD / 32;       // K words a lane takes of a row
  constexpr int LD = HD + 4;        // row stride of the merge buffer: spreads the heads over the banks
  using R = Ring<HD>;
  extern __shared__ __align__(128) uint8_t smem[];  // the warps' rings, then the merge buffer
  float* merge = reinterpret_cast<float*>(smem + kWarps * R::WARP);
  float(*so)[kHeads][LD] = reinterpret_cast<float(*)[kHeads][LD]>(merge);
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
  const long long at = blockIdx.x * total / n_cta, end = (blockIdx.x + 1) * total / n_cta;
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
  Walk cur;
  cur.b = s_row;
  {
    const int U = tiles_of(tokens_of(a, cur.b));
    cur.h = (int)((at - s_at) / U);
    cur.first = (int)(at - s_at - (long long)cur.h * U);
  }
  cur.left = (int)(end - at);
  cur.enter(a);
  long long seg0 = at - cur.first;  // the segment's first tile in the sum

  const float sl2 = a.scale * kLog2e;
  const uint32_t ring = smem_u32(smem) + warp * R::WARP;
  // this lane's places in a stage
  const uint32_t k_at = R::K + g * R::ROW + t * (4 * KW), s_at4 = R::S + g * (8 * G);
  uint32_t v_at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at_byte = (2 * t + (i & 1) + 8 * (i >> 1)) * R::ROW + g * (4 * G);
    v_at[i] = R::V + v_chunk<HD>(at_byte / 16) + at_byte % 16;
  }

  // The copies run kStages - 1 tiles ahead of the arithmetic, across the segments; a tile's page id is read one step
  // before its copies start.
  Walk f = cur;
  int f_tile = f.first + warp, f_end = f.n ? f.last : 0, f_pi = f_tile / a.ppt, f_off = f_tile % a.ppt, f_page = -1;
  int f_head = f.h / a.blocks * a.ppt;
  const int step_pi = kWarps / a.ppt, step_off = kWarps % a.ppt;
  const uint8_t* kp = a.c.k + lane * 16;
  const uint8_t* vp = a.c.v + lane * 16;
  const uint8_t* sp = reinterpret_cast<const uint8_t*>(a.c.scale) + lane * 16;
  auto settle = [&]() {  // on this warp's next tile, if its share has one
    while (f_tile >= f_end) {
      if (!f.next(a)) {
        f_page = -1;
        f_end = 0x7fffffff;  // nothing more: the cursor stays on pages that are not there
        f_tile = 0;
        f.left = 0;
        return;
      }
      f_tile = warp;
      f_end = f.n ? f.last : 0;
      f_pi = f_tile / a.ppt;
      f_off = f_tile % a.ppt;
      f_head = f.h / a.blocks * a.ppt;
    }
    if (f.left > 0) f_page = a.bt[f.b * a.bt_stride + f_pi];
  };
  uint32_t valid = 0;  // bit i: the tile i steps ahead has a page
  auto fetch = [&](uint32_t stage, int steps) {
    if ((uint32_t)f_page < (uint32_t)a.c.n_pages) {
      valid |= 1u << steps;
      const int64_t off = (int64_t)f_page * a.page_bytes + (f_head + f_off) * (kTok * R::ROW);
#pragma unroll
      for (int i = 0; i < R::V / 512; ++i) {
        copy16(stage + R::K + (lane + 32 * i) * 16, kp + off + 512 * i);
        copy16(stage + R::V + v_chunk<HD>(lane + 32 * i), vp + off + 512 * i);
      }
      if (lane < (R::BYTES - R::S) / 16) copy16(stage + R::S + lane * 16, sp + (off >> 2));
    }
    copies_commit();
    f_tile += kWarps;
    f_pi += step_pi;
    f_off += step_off;
    if (f_off >= a.ppt) {
      f_off -= a.ppt;
      ++f_pi;
    }
    settle();
  };
  settle();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(ring + i * R::BYTES, i);
  uint32_t stage = ring, ahead = ring + (kStages - 1) * R::BYTES;

  while (true) {
    const int hk = cur.h / a.blocks, h0 = (cur.h % a.blocks) * kHeads;
    const int nh = min(kHeads, a.rep - h0);
    const int b = cur.b;
    const int t_end = cur.n ? cur.last : 0;
    const int cut = cur.n % kTok ? cur.U - 1 : -1;  // the row ends inside this tile

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
#pragma unroll
    for (int i = 0; i < G; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
      z[i][0] = z[i][1] = 0.f;
      A[i] = kMinA;
      inv[i] = kBoost / kMinA;
    }

    for (int tile = cur.first + warp; tile < t_end; tile += kWarps) {
      __syncwarp();  // every lane has read the stage that is filled again
      fetch(ahead, kStages - 1);
      copies_wait<kStages - 1>();
      __syncwarp();
      const uint32_t here = stage;
      ahead = stage;
      stage = stage + R::BYTES == ring + R::WARP ? ring : stage + R::BYTES;
      const bool there = valid & 1u;
      valid >>= 1;
      if (!there) continue;
      uint32_t kw[2][KW], vw[4][G], sw[2][2 * G];
#pragma unroll
      for (int i = 0; i < 2; ++i) load_words<KW>(kw[i], here + k_at + i * 8 * R::ROW);
#pragma unroll
      for (int i = 0; i < 2; ++i) load_words<2 * G>(sw[i], here + s_at4 + i * 8 * (8 * G));
#pragma unroll
      for (int i = 0; i < 4; ++i) load_words<G>(vw[i], here + v_at[i]);
      float acc[G][4];
#pragma unroll
      for (int i = 0; i < G; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        uint32_t w0 = kw[0][j], w1 = kw[1][j];
        mma_f16(acc[j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[j][0], qf[j][1]);
        w0 >>= 8;
        w1 >>= 8;
        mma_f16(acc[j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[j][2], qf[j][3]);
      }
      float e[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
      if (tile == cut) {  // what lies behind the row's end may be anything
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (g + 8 * i >= cur.n % kTok) {
            e[i][0] = e[i][1] = -INFINITY;
#pragma unroll
            for (int j = 0; j < 2 * G; ++j) sw[i][j] = 0u;
          }
      }
      // scores: [token g + 8 i][head 2 t + r], base 2, relative to the reference
      float s[2][2], va[2][G], vz[2][G];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float d[2] = {0.f, 0.f};
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const float2 k2 = unpack_half2(sw[i][j]), v2 = unpack_half2(sw[i][G + j]);
          va[i][j] = v2.x;
          vz[i][j] = v2.y;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            d[r] = fmaf(k2.x, acc[j][2 * i + r], d[r]);
            e[i][r] = fmaf(k2.y, qs[r][j], e[i][r]);
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) s[i][r] = fmaf(cs[r], d[r], e[i][r]);
      }
      float p[2][2], w[2][G], top_p = 0.f, top_w = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          p[i][r] = ex2(s[i][r] - m[r]);
          top_p = fmaxf(top_p, p[i][r]);
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
          w[i][j] = va[i][j] * inv[j];
          top_w = fmaxf(top_w, w[i][j]);
        }
      }
      if (__any_sync(0xffffffffu, top_p > kMaxP || top_w > kMaxW)) {  // the first tile too: there p is infinite
        // move the reference to the true maxima
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
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int r = 0; r < 2; ++r) p[i][r] = m[r] == -INFINITY && s[i][r] == -INFINITY ? 0.f : ex2(s[i][r] - m[r]);
#pragma unroll
          for (int j = 0; j < G; ++j) w[i][j] = va[i][j] * inv[j];
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
        const uint32_t b0 = transpose8x8(pack_half2(p[0][0] * w[0][j], p[0][1] * w[0][j]));
        const uint32_t b1 = transpose8x8(pack_half2(p[1][0] * w[1][j], p[1][1] * w[1][j]));
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // channels 8 g + 4 half ..
          const uint32_t sel = half ? 0x7632u : 0x5410u;
          uint32_t x01 = __byte_perm(vw[0][j], vw[1][j], sel), x23 = __byte_perm(vw[2][j], vw[3][j], sel);
          mma_f16(o[j][2 * half], x01 & 0x000F000Fu, x01 & 0x00F000F0u, x23 & 0x000F000Fu, x23 & 0x00F000F0u, b0, b1);
          x01 >>= 8;
          x23 >>= 8;
          mma_f16(o[j][2 * half + 1], x01 & 0x000F000Fu, x01 & 0x00F000F0u, x23 & 0x000F000Fu, x23 & 0x00F000F0u, b0, b1);
        }
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
    const bool whole = cur.first == 0 && cur.last == cur.U;
    const int slot = 2 * blockIdx.x + (cur.first == 0 ? 1 : 0);
    bf16* dst = a.out + ((int64_t)b * a.Hq + hk * a.rep + h0) * HD;
    for (int i = tid; i < nh * (HD / 2); i += kThreads) {
      const int h = i / (HD / 2), ch = 2 * (i % (HD / 2));
      float M = -INFINITY, L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm[w][h]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float c = sm[w][h] == -INFINITY ? 0.f : ex2(sm[w][h] - M);
        L = fmaf(sl[w][h], c, L);
        x = fmaf(so[w][h][ch], c, x);
        y = fmaf(so[w][h][ch + 1], c, y);
      }
      if (whole) {
        const float c = L == 0.f ? 0.f : 1.f / L;
        *reinterpret_cast<uint32_t*>(dst + (int64_t)h * HD + ch) = pack_bf16x2(x * c, y * c);
      } else {
        float* pp = a.part + ((int64_t)slot * kHeads + h) * (HD + 4);
        *reinterpret_cast<float2*>(pp + ch) = make_float2(x, y);
        if (ch == 0) *reinterpret_cast<float2*>(pp + HD) = make_float2(M, L);
      }
    }
    if (!whole) {
      const long long c0 = ((seg0 + 1) * n_cta - 1) / total;  // the CTAs that share the segment
      const int np = (int)(((seg0 + cur.U) * n_cta - 1) / total - c0) + 1;
      unsigned* ctr = a.arrived + (int64_t)b * per_row + cur.h;
      __threadfence();
      __syncthreads();
      if (tid == 0) s_last = atomicAdd(ctr, 1u) == (unsigned)(np - 1);
      __syncthreads();
      if (s_last) {
        __threadfence();
        static_assert(kWarps == kHeads, "one warp per head");
        // every piece's weight, then the sum of the pieces, a few loads under way at a time
        const float* p0 = a.part + c0 * 2 * kHeads * (HD + 4);
        auto piece = [&](int c, int h) { return p0 + ((2 * c + (c == 0 ? 1 : 0)) * kHeads + h) * (HD + 4); };
        float* wt = merge + warp * np;
        if (warp < nh) {
          float M = -INFINITY, L = 0.f;
          for (int c = lane; c < np; c += 32) {
            const float m1 = __ldcg(piece(c, warp) + HD);
            wt[c] = m1;
            M = fmaxf(M, m1);
          }
          M = warp_max(M);
          for (int c = lane; c < np; c += 32) {
            const float x = wt[c] == -INFINITY ? 0.f : ex2(wt[c] - M);
            wt[c] = x;
            L = fmaf(__ldcg(piece(c, warp) + HD + 1), x, L);
          }
          L = warp_sum(L);
          if (lane == 0) sl[0][warp] = L;
        }
        __syncthreads();
        for (int i = tid; i < nh * (HD / 4); i += kThreads) {
          const int h = i / (HD / 4), ch = 4 * (i % (HD / 4));
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
          for (int c = 0; c < np; ++c) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(piece(c, h) + ch));
            const float e = merge[h * np + c];
            x.x = fmaf(v.x, e, x.x);
            x.y = fmaf(v.y, e, x.y);
            x.z = fmaf(v.z, e, x.z);
            x.w = fmaf(v.w, e, x.w);
          }
          const float L = sl[0][h], e = L == 0.f ? 0.f : 1.f / L;
          *reinterpret_cast<uint2*>(dst + (int64_t)h * HD + ch) =
              make_uint2(pack_bf16x2(x.x * e, x.y * e), pack_bf16x2(x.z * e, x.w * e));
        }
        if (tid == 0) *ctr = 0u;
      }
    }
    seg0 += cur.U;
    if (!cur.next(a)) break;
    __syncthreads();  // the merge buffer is free
  }
  copies_wait<0>();
}

int sm_count() {
  static int n[64] = {};
  int dev = 0;
  MESHY_CUDA_CHECK(cudaGetDevice(&dev));
  if (!n[dev]) MESHY_CUDA_CHECK(cudaDeviceGetAttribute(&n[dev], cudaDevAttrMultiProcessorCount, dev));
  return n[dev];
}

template <int HD>
void launch(const Args& a, cudaStream_t st) {
  constexpr int smem = kWarps * Ring<HD>::WARP + kWarps * kHeads * (HD + 4) * 4;
  static bool set[64] = {};
  int dev = 0;
  MESHY_CUDA_CHECK(cudaGetDevice(&dev));
  if (!set[dev]) {
    MESHY_CUDA_CHECK(cudaFuncSetAttribute(kv4_attn_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    set[dev] = true;
  }
  launch_pdl(kv4_attn_kernel<HD>, dim3(2 * sm_count()), dim3(kThreads), smem, st, a);
}

}  // namespace

int kv4_attention_ctas() { return 2 * sm_count(); }
int64_t kv4_attention_segments(int B, int Hq, int Hkv) { return (int64_t)B * Hkv * ((Hq / Hkv + kHeads - 1) / kHeads); }

void kv4_attention(const bf16* q, int64_t qs, int64_t qh, KV4View c, const int* bt, int64_t bt_stride, int max_pages,
                   const int* seq_lens, int B, int Hq, float scale, bf16* out, float* part, unsigned* arrived,
                   cudaStream_t st) {
  if (B == 0) return;
  const int rep = Hq / c.Hkv;
  const int64_t page_bytes = (int64_t)c.Hkv * c.page * (c.hd / 2);
  MESHY_CHECK(page_bytes < (1LL << 31), "paged_attention_kv4: a page of all heads must be below 2 GB");
  const Args a{q,   qs,   qh,     c, bt, bt_stride, max_pages, seq_lens, B, Hq, rep, (rep + kHeads - 1) / kHeads, c.page / kTok, (int)page_bytes, scale,
               out, part, arrived};
  if (c.hd == 128)
    launch<128>(a, st);
  else
    launch<64>(a, st);
}

}  // namespace meshy
