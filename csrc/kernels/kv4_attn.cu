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
constexpr int kStages = 2;
constexpr uint32_t kWholeUnits = 40;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBoost = 2048.f;               // x of the largest p and a' right after the reference moved
constexpr float kGrowP = 8.f, kGrowA = 2.f;    // how far either may pass it: x stays below 2^15
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
  static constexpr int F = Q + 2 * QBYTES;               // two sets of query fragments: matrix B, sums (B too), factors
  static constexpr int F_SUM = 32 * 16 * (HD / 32), F_FACTOR = F_SUM + 2 * 32 * 4, FBYTES = F_FACTOR + kHeads * 4;
  static constexpr int SMEM = F + 2 * FBYTES;
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

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

// CTA c of n has units [begin(c), begin(c + 1)): total / n each, and the rest spread evenly (so that equal segments are
// cut alike).
struct Shares {
  uint32_t total, n, per, more;
  __device__ __forceinline__ uint32_t begin(uint32_t c) const { return c * per + c * more / n; }
  __device__ __forceinline__ uint32_t owner(uint32_t unit) const {
    uint32_t c = min(n - 1, (uint32_t)((float)unit / (float)total * (float)n));
    while (c + 1 < n && begin(c + 1) <= unit) ++c;
    while (begin(c) > unit) --c;
    return c;
  }
};

// A segment (b, h) that the CTA has a piece of: its first unit and its units; then the CTAs that share it.
struct Piece {
  int b, h;
  uint32_t first, n;
  bool last;  // this CTA arrived last
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
  __shared__ int s_row;
  __shared__ Piece s_piece[2];
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
  // a CTA per segment where that makes a few steps of every warp; else as many CTAs as give each warp a unit
  const uint32_t segments = a.B * per_row;
  const uint32_t n_cta = min(gridDim.x, all <= segments * kWholeUnits ? segments : (all + kWarps - 1) / kWarps);
  if (blockIdx.x >= n_cta) return;
  const Shares shares{all, n_cta, all / n_cta, all % n_cta};
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
  // A segment's query rows as matrix fragments, a warp per head: scaled so that the largest is in [2^14, 2^15), a
  // word's channels 0 .. 7 as fp16 pairs (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16; the sums over the groups' channels in
  // units of 2^8 as three fp16 terms, against the bases; the factor that takes all that back, with the softmax scale.
  auto prepare_q = [&](const W& w, int buf) {
    static_assert(kWarps == kHeads, "a warp per head");
    constexpr int CH = HD / 32;  // channels of a lane
    uint8_t* f = smem + C::F + buf * C::FBYTES;
    const bool real = (w.h % a.blocks) * kHeads + warp < a.rep;
    float x[CH], mx = 0.f, sum = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      x[i] = real ? __bfloat162float(reinterpret_cast<const bf16*>(smem + C::Q + buf * C::QBYTES)[warp * HD + lane * CH + i]) : 0.f;
      mx = fmaxf(mx, fabsf(x[i]));
      sum += x[i];
    }
    mx = warp_max(mx);
    const int ex = (mx > 0.f && mx < INFINITY) ? min(14 - ilogbf(mx), 126) : 0;
    const float up = ldexpf(1.f, ex);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int ch = lane * CH + i, word = (ch % 64) / 8 * G + ch / 64, e = ch % 8;
      reinterpret_cast<__half*>(f)[(((word % KW) * 32 + warp * 4 + word / KW) * 4 + e % 4) * 2 + e / 4] =
          __float2half_rn(x[i] * (e % 2 ? up * 0.0625f : up));
    }
#pragma unroll
    for (int o = 1; o < 64 / CH; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const float y0 = __shfl_sync(0xffffffffu, sum, i * 16) * up * 0.00390625f;
      const __half h0 = __float2half_rn(y0);
      const float y1 = y0 - __half2float(h0);
      const __half h1 = __float2half_rn(y1), h2 = __float2half_rn(y1 - __half2float(h1));
      const __half h = lane == 0 ? h0 : lane == 1 ? h1 : lane == 2 ? h2 : __float2half_rn(0.f);
      if (lane < 4) reinterpret_cast<uint32_t*>(f + C::F_SUM)[i * 32 + warp * 4 + lane] = (uint32_t)__half_as_ushort(h) << 16;
    }
    if (lane == 0) reinterpret_cast<float*>(f + C::F_FACTOR)[warp] = ldexpf(sl2, 24 - ex);
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
  copies_wait<kStages - 1>();  // the query rows
  __syncthreads();
  prepare_q(s_cur, 0);
  __syncthreads();
  int q_at = 0, pieces = 0;

  W then = s_cur;
  while (true) {
    const W cur = then;
    const int hk = cur.h / a.blocks, h0 = (cur.h % a.blocks) * kHeads;
    const int nh = min(kHeads, a.rep - h0);
    const int b = cur.b;
    const int u_end = cur.n ? cur.last : 0;

    const uint8_t* frags = smem + C::F + q_at * C::FBYTES;
    uint32_t zf[2] = {0u, 0u};
    float cs[2], ce[2];
#pragma unroll
    for (int i = 0; i < G; ++i) zf[i] = reinterpret_cast<const uint32_t*>(frags + C::F_SUM)[i * 32 + lane];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      cs[r] = reinterpret_cast<const float*>(frags + C::F_FACTOR)[2 * t + r];
      ce[r] = cs[r] * 1.52587890625e-5f;  // the sums are in units of 2^8, the products in 2^24
    }
    const uint32_t f_at = smem_u32(frags) + lane * 16;
    // o, z and l are relative to the reference m: p 2^-m; m < the true maximum, so that x fits fp16 well
    float o[G][4][4], z[G][2], m[2] = {0.f, 0.f}, l[2] = {0.f, 0.f};
    float lim_p = -1.f, lim_a = kMinA * kGrowA;  // lim_p below 0: no reference yet
#pragma unroll
    for (int i = 0; i < G; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
      z[i][0] = z[i][1] = 0.f;
    }
    const bool more = then.next(a);
    if (more) copy_q(then, q_at ^ 1);
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
      // scores: tile n, row g + 8 i, head 2 t + r
      float s[NT][2][2], va[NT][2][G], vz[NT][2][G];
      {
        uint32_t kw[NT][2][KW];
        float acc[NT][G][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) load_words<KW>(kw[n][i], here + k_at + (2 * n + i) * 8 * C::ROW);
#pragma unroll
        for (int j = 0; j < KW; ++j) {
          uint32_t qf[4];
          load_words<4>(qf, f_at + j * 512);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint32_t w0 = kw[n][0][j], w1 = kw[n][1][j];
            if (j < G)
              mma_f16_first(acc[n][j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[0], qf[1]);
            else
              mma_f16(acc[n][j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[0], qf[1]);
            w0 >>= 8;
            w1 >>= 8;
            mma_f16(acc[n][j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[2], qf[3]);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t sw[2][2 * G];
#pragma unroll
          for (int i = 0; i < 2; ++i) load_words<2 * G>(sw[i], here + s_at + (2 * n + i) * 8 * C::PAIRS);
          float e[4];  // sum_g z_g sum(q_g): the pairs (a, z) against (0, sum)
          mma_f16_first(e, sw[0][0], sw[1][0], G == 2 ? sw[0][G - 1] : 0u, G == 2 ? sw[1][G - 1] : 0u, zf[0], zf[1]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float d[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < G; ++j) {
              const float ka = __low2float(*reinterpret_cast<const __half2*>(&sw[i][j]));
              const float2 v2 = unpack_half2(sw[i][G + j]);
              va[n][i][j] = v2.x;
              vz[n][i][j] = v2.y;
              d[0] = fmaf(ka, acc[n][j][2 * i], d[0]);
              d[1] = fmaf(ka, acc[n][j][2 * i + 1], d[1]);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) s[n][i][r] = fmaf(cs[r], d[r], fmaf(ce[r], e[2 * i + r], -m[r]));
          }
        }
      }
      if (count < C::UTOK) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (n * kTok + tok_g + 8 * i >= count) {
              s[n][i][0] = s[n][i][1] = -INFINITY;
#pragma unroll
              for (int j = 0; j < G; ++j) va[n][i][j] = vz[n][i][j] = 0.f;
            }
      }
      float p[NT][2][2], top_p = 0.f, top_a = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            p[n][i][r] = ex2(s[n][i][r]);
            top_p = fmaxf(top_p, p[n][i][r]);
          }
#pragma unroll
          for (int j = 0; j < G; ++j) top_a = fmaxf(top_a, va[n][i][j]);
        }
      if (__any_sync(0xffffffffu, top_p > lim_p || top_a > lim_a)) {
        // move the reference: to the true maxima, less what brings x to kBoost
        const float A0 = lim_a / kGrowA, A = max_over_rows(fmaxf(A0, top_a)), lift = lg2(kBoost / A);
        bool found = false;
        float keep[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float top = s[0][0][r];
#pragma unroll
          for (int n = 0; n < NT; ++n) top = fmaxf(top, fmaxf(s[n][0][r], s[n][1][r]));
          top = max_over_rows(top) + m[r];
          if (lim_p > 0.f) top = fmaxf(top, m[r] + lg2(kBoost / A0));
          const bool real = top != -INFINITY;
          const float to = real ? top - lift : m[r];
          keep[r] = lim_p > 0.f ? ex2(m[r] - to) : 0.f;
          found |= real;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) p[n][i][r] = ex2(s[n][i][r] + (m[r] - to));
          m[r] = to;
          l[r] *= keep[r];
        }
        if (__any_sync(0xffffffffu, found)) lim_p = kBoost / A * kGrowP;
        lim_a = A * kGrowA;
#pragma unroll
        for (int j = 0; j < G; ++j) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[j][q][x] *= keep[x & 1];
          z[j][0] *= keep[0];
          z[j][1] *= keep[1];
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t vw[4][G];
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<G>(vw[i], here + v_at + (4 * n + i) * 4 * C::ROW);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          l[r] += p[n][0][r] + p[n][1][r];
#pragma unroll
          for (int j = 0; j < G; ++j) z[j][r] = fmaf(p[n][0][r], vz[n][0][j], fmaf(p[n][1][r], vz[n][1][j], z[j][r]));
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const uint32_t b0 = transpose8x8(pack_half2(p[n][0][0] * va[n][0][j], p[n][0][1] * va[n][0][j]));
          const uint32_t b1 = transpose8x8(pack_half2(p[n][1][0] * va[n][1][j], p[n][1][1] * va[n][1][j]));
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
        constexpr float f0 = 16777216.f, f1 = 1048576.f;
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
        sm[warp][2 * t + r] = lim_p < 0.f ? -INFINITY : m[r];
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
    if (!whole) {  // at most the first and the last segment of the share
      if (tid == 0) s_piece[pieces] = {b, cur.h, seg0, (uint32_t)cur.U, false};
      ++pieces;
    }
    if (!more) break;
    seg0 += cur.U;
    q_at ^= 1;
    prepare_q(then, q_at);
    __syncthreads();  // the states have been read, the fragments are there
  }
  copies_wait<0>();
  if (pieces == 0) return;
  // The last CTA to arrive at a segment joins its pieces; arrivals wait until the share is done, so that nothing else
  // waits for their round trip.
  __syncthreads();
  if (tid < pieces) {
    Piece& x = s_piece[tid];
    const uint32_t c0 = shares.owner(x.first), np = shares.owner(x.first + x.n - 1) - c0 + 1;
    x.first = c0;
    x.n = np;
    unsigned* ctr = a.arrived + (int64_t)x.b * per_row + x.h;
    unsigned old;
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(ctr) : "memory");
    x.last = old == np - 1;
    if (x.last) *ctr = 0u;
  }
  __syncthreads();
  for (int i = tid; i < pieces * kHeads * (HD / 4); i += kThreads) {
    const Piece& x = s_piece[i / (kHeads * (HD / 4))];
    const int h = i / (HD / 4) % kHeads, ch = 4 * (i % (HD / 4)), hk = x.h / a.blocks, h0 = (x.h % a.blocks) * kHeads;
    if (!x.last || h0 + h >= a.rep) continue;
    const float* p0 = a.part + ((int64_t)x.first * 2 * kHeads + h) * C::PART;
    const int np = x.n;
    float M = -INFINITY, L = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kBatch = 8;
    for (int c0 = 0; c0 < np; c0 += kBatch) {
      float4 v[kBatch];
      float2 ml[kBatch];
      float Mn = M;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int c = c0 + k;
        ml[k] = make_float2(-INFINITY, 0.f);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c < np) {
          const float* pp = p0 + (2 * c + (c == 0 ? 1 : 0)) * kHeads * C::PART;
          ml[k] = __ldcg(reinterpret_cast<const float2*>(pp + HD));
          v[k] = __ldcg(reinterpret_cast<const float4*>(pp + ch));
        }
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) Mn = fmaxf(Mn, ml[k].x);
      const float keep = M == -INFINITY ? 0.f : ex2(M - Mn);
      L *= keep;
      y.x *= keep, y.y *= keep, y.z *= keep, y.w *= keep;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const float e = ml[k].x == -INFINITY ? 0.f : ex2(ml[k].x - Mn);
        L = fmaf(ml[k].y, e, L);
        y.x = fmaf(v[k].x, e, y.x);
        y.y = fmaf(v[k].y, e, y.y);
        y.z = fmaf(v[k].z, e, y.z);
        y.w = fmaf(v[k].w, e, y.w);
      }
      M = Mn;
    }
    const float e = L == 0.f ? 0.f : 1.f / L;
    *reinterpret_cast<uint2*>(a.out + ((int64_t)x.b * a.Hq + hk * a.rep + h0 + h) * HD + ch) =
        make_uint2(pack_bf16x2(y.x * e, y.y * e), pack_bf16x2(y.z * e, y.w * e));
  }
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
