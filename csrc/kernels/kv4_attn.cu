// Paged decode attention over the 4-bit KV cache (layout in kv4.h).
//
//   s_j = scale * sum_g (a_jg (q_g . n_jg) + z_jg sum(q_g)),  p = softmax(s),  o = sum_j p_j (a'_jg n'_j + z'_jg)
//
// The scale and the base of a group leave the channel sums, so the nibbles go to the tensor cores as whole numbers:
// masked in place they are fp16 subnormals (n at bits 0-3 is n 2^-24, at bits 4-7 n 2^-20), exact and with no
// conversion. The power of two is divided out of Q (four of every eight channels carry 1/16) and of the result.
//
// A warp takes 16 tokens at a time (m16n8k16, fp16 in, fp32 sums):
//   S^T [16 tokens, 8 heads] = K [16, hd] Q^T      A rows are tokens: a lane's 16 bytes of a K row are its A registers
//   O^T [16 channels, 8 heads] += V^T [16, 16 tokens] P^T    A rows are channels: two byte permutes pair the tokens
// Query heads that share a KV head fill the 8 columns, so every cached byte is read once for up to 8 heads. P changes
// from accumulator to operand by movmatrix. The tokens are dealt to the rows so that the lanes that read V together
// read four neighbouring tokens (no bank conflicts). tcgen05 would not help here: operands unpacked in registers would
// have to be stored to shared or tensor memory first, and at 8 query rows the matrix work is a fraction of the
// unpacking.
//
// P carries the scale of V (x = p a'), so it is kept in fp16's range by a reference (m, A) per warp: x = 64 p a' / A
// with p relative to m. The reference moves only when p passes 2^7 or 64 a' / A passes 2^8 (then to the true maxima),
// so most tiles take neither the maximum's shuffles nor a rescaling; what falls below fp16's smallest number is less
// than 2^-30 of the largest term.
//
// Work split: the (row, KV head, up to 8 query heads) segments are laid end to end in units of 16 tokens and every
// CTA takes an equal share of the sum, whatever the lengths: the lengths are read on the device, a captured graph
// follows them. A segment that spans CTAs leaves partial sums in a workspace; the last CTA to arrive joins them in
// CTA order, so results do not depend on timing.
//
// Each warp keeps a ring of kStages units (32 tokens; 16 where a page is not a multiple of 32) of its own in shared
// memory, filled by 16-byte asynchronous copies two units ahead, across the segments, so no warp waits for another
// between joins. The query rows of the next segment come the same way.
#include <cuda_runtime.h>

#include "../include/sm100.cuh"
#include "kv4.h"

namespace meshy {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kTok = 16;                       // tokens of a tile
constexpr int kHeads = 8;                      // query heads of a segment
constexpr int kStages = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBoost = 64.f;                 // x of the largest p and a' right after the reference moved
constexpr float kMaxP = 128.f, kMaxW = 256.f;  // x = p w stays below 2^15
constexpr float kMinA = 5.9604645e-8f;         // 2^-24, the smallest fp16

template <int HD, int NT>  // NT tiles to a unit
struct Cfg {
  static constexpr int ROW = HD / 2;                     // nibble bytes of a token
  static constexpr int PAIRS = HD / 8;                   // bytes of a token's pairs (K and V)
  static constexpr int UTOK = NT * kTok;
  static constexpr int K = 0, V = UTOK * ROW, S = 2 * UTOK * ROW;
  static constexpr int LD = HD + 4;                      // row stride of a warp's state: spreads the heads over the banks
  static constexpr int STAGE = 2 * (2 * kTok * ROW + kTok * PAIRS);  // room for a unit, and for a warp's state
  static_assert(kHeads * LD * 4 <= STAGE && UTOK * (2 * ROW + PAIRS) <= STAGE, "a stage holds either");
  static constexpr int WARP = kStages * STAGE;
  static constexpr int Q = kWarps * WARP;
  static constexpr int QBYTES = kHeads * HD * 2;
  static constexpr int SMEM = Q + 2 * QBYTES;
  static constexpr int PART = HD + 4;                    // floats of a head in the workspace: sums, maximum, normaliser
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {  // zeros where it is not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

// the same with a zero accumulator
__device__ __forceinline__ void mma_f16_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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
  int upp, page_units;     // units of a page, of a page of all heads
  float scale;
  bf16* out;
  float* part;         // [2 CTAs][kHeads][PART]
  unsigned* arrived;   // [segments], zero between launches
};

__device__ __forceinline__ int tokens_of(const Args& a, int b) {
  const int64_t cap = (int64_t)a.max_pages * a.c.page;
  const int n = a.seq_lens[b];
  return n <= 0 ? 0 : (int)min((int64_t)n, cap);
}
template <int UTOK>
__device__ __forceinline__ uint32_t units_of(int n) { return max(1, (n + UTOK - 1) / UTOK); }  // an empty row writes its zeros

// A CTA's walk over its share of the units: segment (b, h), of whose U units it has [first, last); ``left`` units of the
// share remain from ``first`` on.
template <int UTOK>
struct Walk {
  int b, h, n, U, first, last, left;
  __device__ __forceinline__ bool next(const Args& a) {
    left -= last - first;
    if (left <= 0) return false;
    first = 0;
    if (++h == a.c.Hkv * a.blocks) {
      h = 0;
      ++b;
      n = tokens_of(a, b);
      U = units_of<UTOK>(n);
    }
    last = min(U, left);
    return true;
  }
};

// The share of CTA c of n: total / n units, the first total % n CTAs one more.
struct Shares {
  uint32_t per, more;
  __device__ __forceinline__ uint32_t begin(uint32_t c) const { return c * per + min(c, more); }
  __device__ __forceinline__ uint32_t owner(uint32_t unit) const {
    const uint32_t big = more * (per + 1);
    return unit < big ? unit / (per + 1) : more + (unit - big) / per;
  }
};

template <int HD, int NT>
__global__ void __launch_bounds__(kThreads, 2) kv4_attn_kernel(const Args a) {
  using C = Cfg<HD, NT>;
  using W = Walk<C::UTOK>;
  constexpr int G = HD / 64;
  constexpr int KW = HD / 32;  // K words a lane takes of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm[kWarps][kHeads], sl[kWarps][kHeads];
  __shared__ uint32_t scan[kWarps], s_begin;
  __shared__ int s_row, s_last;
  __shared__ const float* so[kWarps];  // the warps' states
  __shared__ W s_cur, s_ahead[kWarps];  // touched once per segment: kept out of the registers
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t per_row = a.c.Hkv * a.blocks;  // segments of a row

  pdl_wait();
  pdl_trigger();

  // all units (row by row), this CTA's share of them and the row it starts in
  uint32_t total = 0, mine = 0, before = 0;
  auto sum_rows = [&](int b0) {  // the units of rows b0 + tid, of the rows before it, and of all up to this block of rows
    mine = b0 + tid < a.B ? units_of<C::UTOK>(tokens_of(a, b0 + tid)) * per_row : 0;
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    before = total + incl - mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
  };
  for (int b0 = 0; b0 < a.B; b0 += kThreads) sum_rows(b0);
  const uint32_t all = total;
  const uint32_t n_cta = min(gridDim.x, (all + kWarps - 1) / kWarps);
  if (blockIdx.x >= n_cta) return;
  const Shares shares{all / n_cta, all % n_cta};
  const uint32_t at = shares.begin(blockIdx.x), end = shares.begin(blockIdx.x + 1);
  if (a.B > kThreads) total = 0;
  for (int b0 = 0; b0 < a.B; b0 += kThreads) {
    if (a.B > kThreads) sum_rows(b0);
    if (at - before < mine) {
      s_row = b0 + tid;
      s_begin = before;
    }
    if (total > at) break;
  }
  __syncthreads();
  uint32_t seg0 = s_begin;  // the segment's first unit in the sum
  int f_unit;
  {
    W w;
    w.b = s_row;
    w.n = tokens_of(a, w.b);
    w.U = units_of<C::UTOK>(w.n);
    w.h = (at - seg0) / w.U;
    seg0 += w.h * w.U;
    w.first = at - seg0;
    w.left = end - at;
    w.last = min(w.U, w.first + w.left);
    f_unit = w.first + warp;
    if (lane == 0) s_ahead[warp] = w;
    if (tid == 0) s_cur = w;
  }
  __syncthreads();

  const int g = lane / 4, t = lane % 4;
  const int tok_g = g / 2 + 4 * (g % 2);  // token of matrix rows g and (8 further on) g + 8; V's are t, t + 4, t + 8, t + 12
  const float sl2 = a.scale * kLog2e;
  const uint32_t ring = smem_u32(smem) + warp * C::WARP;
  // this lane's places in a stage
  const uint32_t k_at = C::K + tok_g * C::ROW + t * (4 * KW), s_at = C::S + tok_g * C::PAIRS;
  const uint32_t v_at = C::V + t * C::ROW + g * (4 * G);

  // Query rows of a segment, a 16-byte chunk per thread (completed with the thread's next group of copies).
  auto copy_q = [&](const W& w, int buf) {
    const int h0 = (w.h % a.blocks) * kHeads, i = tid / (HD / 8);
    if (i < min(kHeads, a.rep - h0))
      copy16(smem_u32(smem) + C::Q + buf * C::QBYTES + tid * 16,
             a.q + w.b * a.qs + (int64_t)(w.h / a.blocks * a.rep + h0 + i) * a.qh + (tid % (HD / 8)) * 8, true);
  };
  copy_q(s_cur, 0);
  copies_commit();

  // The copies run kStages - 1 units ahead of the arithmetic, across the segments; a unit's page id is read one step
  // before its copies start.
  constexpr int kDone = -(1 << 30);  // the share holds no more units for this warp
  int f_end, f_pi, f_off, f_head, f_page;
  const int* f_bt;
  const int step_pi = kWarps / a.upp, step_off = kWarps % a.upp;
  const uint8_t* kp = a.c.k + lane * 16;
  const uint8_t* vp = a.c.v + lane * 16;
  const uint8_t* sp = reinterpret_cast<const uint8_t*>(a.c.scale) + lane * 16;
  auto aim = [&](const W& w) {
    f_end = w.n ? w.last : 0;
    f_pi = f_unit / a.upp;
    f_off = f_unit % a.upp;
    f_head = w.h / a.blocks * a.upp;
    f_bt = a.bt + w.b * a.bt_stride;
  };
  auto settle = [&]() {  // on this warp's next unit, if its share has one
    if (f_unit >= f_end) {
      W w = s_ahead[warp];
      do {
        if (!w.next(a)) {
          f_unit = kDone;
          f_end = 0;
          break;
        }
        f_unit = warp;
        aim(w);
      } while (f_unit >= f_end);
      __syncwarp();
      if (lane == 0) s_ahead[warp] = w;
      __syncwarp();
    }
    f_page = -1;
    if (f_unit >= 0) f_page = f_bt[f_pi];
  };
  uint32_t valid = 0;  // bit i: the unit i steps ahead has a page
  auto fetch = [&](uint32_t stage, int steps) {
    const bool there = (uint32_t)f_page < (uint32_t)a.c.n_pages;
    valid |= (there ? 1u : 0u) << steps;
    const uint32_t n = there ? (uint32_t)f_page * (uint32_t)a.page_units + (uint32_t)(f_head + f_off) : 0u;  // unit of the cache
    const uint8_t* ks = kp + (uint64_t)n * (C::UTOK * C::ROW);
    const uint8_t* vs = vp + (uint64_t)n * (C::UTOK * C::ROW);
    const uint8_t* ss = sp + (uint64_t)n * (C::UTOK * C::PAIRS);
    const uint32_t dst = stage + lane * 16;
#pragma unroll
    for (int i = 0; i < C::UTOK * C::ROW / 512; ++i) {
      copy16(dst + C::K + 512 * i, ks + 512 * i, there);
      copy16(dst + C::V + 512 * i, vs + 512 * i, there);
    }
    if (C::UTOK * C::PAIRS == 512 || lane < C::UTOK * C::PAIRS / 16) copy16(dst + C::S, ss, there);
    copies_commit();
    f_unit += kWarps;
    f_pi += step_pi;
    f_off += step_off;
    if (f_off >= a.upp) {
      f_off -= a.upp;
      ++f_pi;
    }
    settle();
  };
  aim(s_ahead[warp]);
  settle();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(ring + i * C::STAGE, i);
  uint32_t stage = ring, ahead = ring + (kStages - 1) * C::STAGE;
  copies_wait<kStages - 1>();  // Q
  __syncthreads();
  int q_at = 0;

  while (true) {
    const W cur = s_cur;
    const int hk = cur.h / a.blocks, h0 = (cur.h % a.blocks) * kHeads;
    const int nh = min(kHeads, a.rep - h0);
    const int b = cur.b;
    const int u_end = cur.n ? cur.last : 0;

    // Q fragments: head g, channels of the words this lane reads of a K row; scaled so that the largest is in [2^14, 2^15)
    uint32_t qf[KW][4];
    float cs[2], qs[2][G];
    {
      float x[KW][8], mx = 0.f, sum[G];
#pragma unroll
      for (int i = 0; i < G; ++i) sum[i] = 0.f;
      const bf16* src = reinterpret_cast<const bf16*>(smem + C::Q + q_at * C::QBYTES) + g * HD;
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

    float o[G][4][4], z[G][2], m[2] = {0.f, 0.f}, l[2] = {0.f, 0.f}, inv[G];
    float limit = -1.f;  // of p; below 0: no reference yet
#pragma unroll
    for (int i = 0; i < G; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
      z[i][0] = z[i][1] = 0.f;
      inv[i] = kBoost / kMinA;
    }

    if (cur.left > cur.last - cur.first) {  // the next segment's query rows
      W w = cur;
      w.next(a);
      copy_q(w, q_at ^ 1);
    }
    int steps = 0;
    for (int unit = cur.first + warp; unit < u_end; unit += kWarps) {
      __syncwarp();  // every lane has read the stage that is filled again
      fetch(ahead, kStages - 1);
      copies_wait<kStages - 1>();
      __syncwarp();
      const uint32_t here = stage;
      ahead = stage;
      stage = stage + C::STAGE == ring + C::WARP ? ring : stage + C::STAGE;
      // tokens of the unit to be counted; the rest may be anything
      const int count = valid & 1u ? cur.n - unit * C::UTOK : 0;
      valid >>= 1;
      ++steps;
#pragma unroll
      for (int half = 0; half < NT; ++half) {
        uint32_t kw[2][KW], vw[4][G], sw[2][2 * G];
#pragma unroll
        for (int i = 0; i < 2; ++i) load_words<KW>(kw[i], here + k_at + (2 * half + i) * 8 * C::ROW);
#pragma unroll
        for (int i = 0; i < 2; ++i) load_words<2 * G>(sw[i], here + s_at + (2 * half + i) * 8 * C::PAIRS);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<G>(vw[i], here + v_at + (4 * half + i) * 4 * C::ROW);
        float acc[G][4];
#pragma unroll
        for (int j = 0; j < KW; ++j) {
          uint32_t w0 = kw[0][j], w1 = kw[1][j];
          if (j < G)
            mma_f16_first(acc[j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[j][0], qf[j][1]);
          else
            mma_f16(acc[j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[j][0], qf[j][1]);
          w0 >>= 8;
          w1 >>= 8;
          mma_f16(acc[j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[j][2], qf[j][3]);
        }
        // scores: [row g + 8 i][head 2 t + r], base 2, relative to the reference
        float s[2][2], va[2][G], vz[2][G];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float d[2] = {0.f, 0.f}, e[2] = {-m[0], -m[1]};
#pragma unroll
          for (int j = 0; j < G; ++j) {
            const float2 k2 = unpack_half2(sw[i][j]), v2 = unpack_half2(sw[i][G + j]);
            va[i][j] = v2.x;
            vz[i][j] = v2.y;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              d[r] = fmaf(k2.x, acc[j][2 * i + r], d[r]);
              e[r] = fmaf(k2.y, qs[r][j], e[r]);
            }
          }
#pragma unroll
          for (int r = 0; r < 2; ++r) s[i][r] = fmaf(cs[r], d[r], e[r]);
        }
        if (count < (half + 1) * kTok) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (half * kTok + tok_g + 8 * i >= count) {
              s[i][0] = s[i][1] = -INFINITY;
#pragma unroll
              for (int j = 0; j < G; ++j) va[i][j] = vz[i][j] = 0.f;
            }
        }
        float p[2][2], w[2][G], top_p = 0.f, top_w = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            p[i][r] = ex2(s[i][r]);
            top_p = fmaxf(top_p, p[i][r]);
          }
#pragma unroll
          for (int j = 0; j < G; ++j) {
            w[i][j] = va[i][j] * inv[j];
            top_w = fmaxf(top_w, w[i][j]);
          }
        }
        if (__any_sync(0xffffffffu, top_p > limit || top_w > kMaxW)) {
          // move the reference to the true maxima
          float keep[2];
          bool found = false;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float mt = max_over_rows(fmaxf(s[0][r], s[1][r])) + m[r];
            const float mn = limit < 0.f ? mt : fmaxf(m[r], mt);
            keep[r] = limit < 0.f ? 0.f : ex2(m[r] - mn);
            const float shift = mn == -INFINITY ? 0.f : m[r] - mn;
            found |= mn != -INFINITY;
            if (mn != -INFINITY) m[r] = mn;
            l[r] *= keep[r];
            p[0][r] = ex2(s[0][r] + shift);
            p[1][r] = ex2(s[1][r] + shift);
          }
          if (__any_sync(0xffffffffu, found)) limit = kMaxP;
#pragma unroll
          for (int j = 0; j < G; ++j) {
            const float to = fminf(inv[j], kBoost / fmaxf(max_over_rows(fmaxf(va[0][j], va[1][j])), kMinA)), f = to / inv[j];
            inv[j] = to;
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int x = 0; x < 4; ++x) o[j][q][x] *= f * keep[x & 1];
            z[j][0] *= keep[0];
            z[j][1] *= keep[1];
            w[0][j] = va[0][j] * inv[j];
            w[1][j] = va[1][j] * inv[j];
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
    }

    // the warp's state, in the stage that is free: o in units of V, relative to m
    float* state = reinterpret_cast<float*>(smem + (ahead - smem_u32(smem)));
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] = sum_over_rows(l[r]);
#pragma unroll
      for (int j = 0; j < G; ++j) {
        z[j][r] = sum_over_rows(z[j][r]);
        const float f0 = 16777216.f / inv[j], f1 = 1048576.f / inv[j];
        float x[8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          x[2 * q] = fmaf(o[j][q][r], f0, z[j][r]);
          x[2 * q + 1] = fmaf(o[j][q][2 + r], f1, z[j][r]);
        }
        float4* d = reinterpret_cast<float4*>(state + (2 * t + r) * C::LD + 64 * j + 8 * g);
        d[0] = make_float4(x[0], x[1], x[2], x[3]);
        d[1] = make_float4(x[4], x[5], x[6], x[7]);
      }
      if (g == 0) {
        sm[warp][2 * t + r] = limit < 0.f ? -INFINITY : m[r];
        sl[warp][2 * t + r] = l[r];
      }
    }
    if (lane == 0) so[warp] = state;
    if (steps < kStages) {  // after kStages steps the next query rows have arrived anyway
      copies_commit();
      copies_wait<0>();
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
        x = fmaf(so[w][h * C::LD + ch], c, x);
        y = fmaf(so[w][h * C::LD + ch + 1], c, y);
      }
      if (whole) {
        const float c = L == 0.f ? 0.f : 1.f / L;
        *reinterpret_cast<uint32_t*>(dst + (int64_t)h * HD + ch) = pack_bf16x2(x * c, y * c);
      } else {
        float* pp = a.part + ((int64_t)slot * kHeads + h) * C::PART;
        *reinterpret_cast<float2*>(pp + ch) = make_float2(x, y);
        if (ch == 0) *reinterpret_cast<float2*>(pp + HD) = make_float2(M, L);
      }
    }
    if (!whole) {
      const uint32_t c0 = shares.owner(seg0);  // the CTAs that share the segment
      const int np = (int)(shares.owner(seg0 + cur.U - 1) - c0) + 1;
      unsigned* ctr = a.arrived + (int64_t)b * per_row + cur.h;
      __syncthreads();
      if (tid == 0) {
        __threadfence();
        s_last = atomicAdd(ctr, 1u) == (unsigned)(np - 1);
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        // the pieces' maximum and normaliser, a warp per head; then their sum, a few loads under way at a time
        const float* p0 = a.part + (int64_t)c0 * 2 * kHeads * C::PART;
        auto piece = [&](int c, int h) { return p0 + ((2 * c + (c == 0 ? 1 : 0)) * kHeads + h) * C::PART; };
        static_assert(kWarps == kHeads, "a warp per head");
        if (warp < nh) {
          float M = -INFINITY, L = 0.f;
          for (int c = lane; c < np; c += 32) M = fmaxf(M, __ldcg(piece(c, warp) + HD));
          M = warp_max(M);
          for (int c = lane; c < np; c += 32) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(piece(c, warp) + HD));
            L = fmaf(ml.y, ml.x == -INFINITY ? 0.f : ex2(ml.x - M), L);
          }
          L = warp_sum(L);
          if (lane == 0) {
            sm[0][warp] = M;
            sl[0][warp] = L;
          }
        }
        __syncthreads();
        for (int i = tid; i < nh * (HD / 4); i += kThreads) {
          const int h = i / (HD / 4), ch = 4 * (i % (HD / 4));
          const float M = sm[0][h], L = sl[0][h];
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
          for (int c = 0; c < np; ++c) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(piece(c, h) + ch));
            const float m1 = __ldcg(piece(c, h) + HD), e = m1 == -INFINITY ? 0.f : ex2(m1 - M);
            x.x = fmaf(v.x, e, x.x);
            x.y = fmaf(v.y, e, x.y);
            x.z = fmaf(v.z, e, x.z);
            x.w = fmaf(v.w, e, x.w);
          }
          const float e = L == 0.f ? 0.f : 1.f / L;
          *reinterpret_cast<uint2*>(dst + (int64_t)h * HD + ch) =
              make_uint2(pack_bf16x2(x.x * e, x.y * e), pack_bf16x2(x.z * e, x.w * e));
        }
        if (tid == 0) *ctr = 0u;
      }
    }
    seg0 += cur.U;
    if (cur.left <= cur.last - cur.first) break;
    __syncthreads();  // the states have been read
    if (tid == 0) {
      W w = cur;
      w.next(a);
      s_cur = w;
    }
    q_at ^= 1;
    __syncthreads();
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

template <int HD, int NT>
void launch(Args a, cudaStream_t st) {
  using C = Cfg<HD, NT>;
  a.upp = a.c.page / C::UTOK;
  a.page_units = a.c.Hkv * a.upp;
  // units are counted in 32 bits, in the cache and over the rows
  MESHY_CHECK(a.c.n_pages * a.c.Hkv * a.upp < (1LL << 32), "paged_attention_kv4: cache too large");
  MESHY_CHECK((int64_t)a.B * a.c.Hkv * a.blocks * std::max<int64_t>(1, (int64_t)a.max_pages * a.upp) < (1LL << 31),
              "paged_attention_kv4: rows * heads * table width too large");
  static bool set[64] = {};
  int dev = 0;
  MESHY_CUDA_CHECK(cudaGetDevice(&dev));
  if (!set[dev]) {
    MESHY_CUDA_CHECK(cudaFuncSetAttribute(kv4_attn_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    set[dev] = true;
  }
  launch_pdl(kv4_attn_kernel<HD, NT>, dim3(2 * sm_count()), dim3(kThreads), C::SMEM, st, a);
}

}  // namespace

int kv4_attention_ctas() { return 2 * sm_count(); }
int64_t kv4_attention_segments(int B, int Hq, int Hkv) { return (int64_t)B * Hkv * ((Hq / Hkv + kHeads - 1) / kHeads); }

void kv4_attention(const bf16* q, int64_t qs, int64_t qh, KV4View c, const int* bt, int64_t bt_stride, int max_pages,
                   const int* seq_lens, int B, int Hq, float scale, bf16* out, float* part, unsigned* arrived,
                   cudaStream_t st) {
  if (B == 0) return;
  const int rep = Hq / c.Hkv;
  const Args a{q, qs, qh,  c,   bt,    bt_stride, max_pages, seq_lens, B, Hq, rep, (rep + kHeads - 1) / kHeads,
               0, 0,  scale, out, part, arrived};
  const bool pairs = c.page % 32 == 0;
  if (c.hd == 128)
    pairs ? launch<128, 2>(a, st) : launch<128, 1>(a, st);
  else
    pairs ? launch<64, 2>(a, st) : launch<64, 1>(a, st);
}

}  // namespace meshy
