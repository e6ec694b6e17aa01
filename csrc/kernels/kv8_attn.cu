// Paged decode attention over the 8-bit KV cache (layout in kv8.h).
//
//   s_j = scale a_j (q . (u_j - 128)),  p = softmax(s),  o = sum_j p_j a'_j (u'_j - 128)
//
// The 16 tokens of a block share a scale, so scales leave the channel sums and the bytes go to the tensor cores as whole
// numbers: a byte in the low half of a 16-bit word is the fp16 subnormal u 2^-24, exact and with no conversion. The 128
// that u carries too much is a constant of the query in the scores (the accumulators start at -128 sum(q)) and one more
// product in the output (a matrix of -128 against the weights, added before each tile's own product, so that sums stay
// near zero and lose no bits to it).
//
// A warp takes a block at a time (m16n8k16, fp16 in, fp32 sums):
//   S^T [16 tokens, 8 heads] = K [16, hd] Q^T      A rows are tokens: a word of a K row is two operands, masked and moved
//   O^T [16 channels, 8 heads] += V^T [16, 16 tokens] P^T    A rows are channels: a byte permute pairs two tokens' words
// Query heads that share a KV head fill the 8 columns, so every cached byte is read once for up to 8 heads. P changes
// from accumulator to operand by movmatrix. Copies place a row's 16-byte chunks so that lanes that read together, of K
// (rows i and i + 4) and of V (four neighbouring rows), meet in no bank. tcgen05 would not help: the operands would have
// to be unpacked and stored once more before it could read them, and 8 query rows leave it nothing to win.
//
// P carries the scale of V (x = p a'), so a reference m per warp and head keeps it in fp16's range: p is taken relative
// to m, which is set so that the largest p a' seen is 2^11, and moves again only when a later one passes 2^15. So most
// blocks take neither the maximum's shuffles nor a rescaling. x is rounded to fp16's 11 bits, or by 2^-25 where it is
// below 2^-14: less than 2^-35 of the largest. Scales below 2^-64 count as that for the reference, so that p stays below
// 2^79; sums and the normaliser stay in 32 bits.
//
// Eight warps compute and never wait for one another: each keeps a ring of units of its own in shared memory (a unit is
// a block at head width 128, two at 64: the same bytes), filled by 16-byte asynchronous copies units ahead, across the
// segments, and at a segment's end leaves its state in one of kSlots slots and goes on. Four helper warps prepare the
// query fragments of the coming segments and join the eight states of the finished ones. Every wait is bounded; one that
// gives up records an error code. How the work is split over CTAs stands in kv_split.cuh.
#include <climits>

#include <cuda_runtime.h>

#include "../include/kv_split.cuh"
#include "kv8.h"

namespace meshy {

namespace {

using namespace kvsplit;

constexpr int kWarps = 8;  // that compute
constexpr int kHelpers = 4;
constexpr int kThreads = 32 * (kWarps + kHelpers);
constexpr int kTok = kKV8Block;
constexpr int kSlots = 2;  // segments whose fragments or states are held
constexpr Rules kRules{24, 16, 3};
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBoost = 11.f;        // log2 of the largest p a' right after the reference moved
constexpr float kLimit = 32768.f;     // how far later ones may go
constexpr float kMinA = 5.4210109e-20f;  // 2^-64

template <int HD>
struct Cfg {
  static constexpr int NT = 128 / HD;                   // blocks of a unit
  static constexpr int UTOK = NT * kTok;
  static constexpr int BLOCK = kTok * HD;               // bytes of a block of K
  static constexpr int K = 0, V = NT * BLOCK, S = 2 * NT * BLOCK, STAGE = 2 * NT * BLOCK + 16;
  static constexpr int STAGES = 4;
  static constexpr int WARP = STAGES * STAGE;
  static constexpr int LD = HD + 4;                     // row stride of a state: spreads the heads over the banks
  static constexpr int STATES = kWarps * WARP;          // kSlots sets of the warps' states
  static constexpr int STATE = kHeads * LD * 4;
  // kSlots sets of query fragments: matrix B, -128 sum(q), factors
  static constexpr int F = STATES + kSlots * kWarps * STATE;
  static constexpr int KW = HD / 16;                    // K words of a lane and row
  static constexpr int F_BIAS = KW * 32 * 8, F_FACTOR = F_BIAS + kHeads * 4;
  static constexpr int FBYTES = F_FACTOR + kHeads * 4;
  static constexpr int SMEM = F + kSlots * FBYTES;
  static constexpr int PART = HD + 4;                   // floats of a head in the workspace: sums, maximum, normaliser
};

// Where chunk c (16 bytes) of a block's row j stands.
template <int HD>
__device__ __forceinline__ uint32_t chunk_at(int j, int c) {
  if constexpr (HD == 128) return j * 128 + 16 * (c ^ 2 * (j & 3) ^ (j & 4));
  return j / 2 * 128 + ((j ^ j >> 2) & 1) * 64 + 16 * (c ^ (j & 2));
}

__device__ __forceinline__ void helper_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kHelpers) : "memory"); }

struct Args : Rows {
  const bf16* q;
  int64_t qs, qh;
  KV8View c;
  const int* bt;
  int64_t bt_stride;
  int Hq, rep, blocks;   // blocks: groups of kHeads query heads per KV head
  int bpp, page_blocks;  // blocks of a page of one head, of all heads
  float scale;
  bf16* out;
  float* part;        // [2 CTAs][kHeads][PART]
  unsigned* arrived;  // [segments], zero between launches
  int* err;
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) kv8_attn_kernel(const Args a) {
  using C = Cfg<HD>;
  using W = Walk<C::UTOK, kWarps>;
  constexpr int NT = C::NT, KW = C::KW, VW = HD / 32;  // V words of a lane and row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sm[kSlots][kWarps][kHeads], sl[kSlots][kWarps][kHeads];
  __shared__ W s_seg[kSlots], s_ahead[kWarps];
  __shared__ uint64_t ready[kSlots], done[kSlots];  // fragments are there and the states free; the states are there
  __shared__ float weight[kHeads][kWarps], total_max[kHeads], total_sum[kHeads];
  __shared__ Piece s_piece[2];
  __shared__ PlanShared<kThreads> s_plan;
  __shared__ int s_pieces, s_abort, s_ok;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  volatile int* abort_flag = &s_abort;

  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&ready[i], 1);
      mbar_init(&done[i], kWarps);
    }
    s_abort = 0;
    s_pieces = 0;
    fence_mbar_init();
  }
  pdl_wait();
  pdl_trigger();
  const auto plan = make_plan<C::UTOK, kWarps, kThreads>(a, s_plan, kRules);
  if (!plan.work) return;
  const W w0 = plan.w;
  const int pad = plan.pad;
  const float sl2 = a.scale * kLog2e;

  if (warp >= kWarps) {
    // ───────────────────────────── helpers ─────────────────────────────
    const int hw = warp - kWarps, ht = tid - 32 * kWarps;
    // A segment's query rows as matrix fragments, a warp per head: scaled so that the largest is in [2^14, 2^15); -128
    // times their sum, in units of 2^-24 as the products are; the factor that takes the powers back, with the softmax
    // scale (2^12 of it are left to the blocks' scales).
    constexpr int CH = HD / 32;  // channels of a lane
    uint32_t raw[kHeads / kHelpers][CH / 2];
    auto load_q = [&](const W& w) {
      const int h0 = (w.h % a.blocks) * kHeads;
      const bf16* src = a.q + w.b * a.qs + (int64_t)(w.h / a.blocks * a.rep + h0) * a.qh + lane * CH;
#pragma unroll
      for (int k = 0; k < kHeads / kHelpers; ++k) {
        const int h = hw + k * kHelpers;
#pragma unroll
        for (int i = 0; i < CH / 2; ++i)
          raw[k][i] = h0 + h < a.rep ? *reinterpret_cast<const uint32_t*>(src + h * a.qh + 2 * i) : 0u;
      }
    };
    auto prepare = [&](const W& w, int slot) {
      uint8_t* f = smem + C::F + slot * C::FBYTES;
#pragma unroll
      for (int k = 0; k < kHeads / kHelpers; ++k) {
        const int h = hw + k * kHelpers;
        float x[CH];
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
          const float2 y = unpack_bf16x2(raw[k][i]);
          x[2 * i] = y.x;
          x[2 * i + 1] = y.y;
        }
        float mx = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) mx = fmaxf(mx, fabsf(x[i]));
        mx = warp_max(mx);
        const int ex = (mx > 0.f && mx < INFINITY) ? min(14 - ilogbf(mx), 126) : 0;
        const float up = ldexpf(1.f, ex);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int ch = lane * CH + i, t = ch / 16 % 4, w = ch % 16 / 4 + 4 * (ch / 64), e = ch % 4;
          const __half y = __float2half_rn(x[i] * up);
          sum += __half2float(y);
          reinterpret_cast<__half*>(f)[(((w / 2 * 32 + h * 4 + t) * 4) + w % 2 * 2 + e % 2) * 2 + e / 2] = y;
        }
        sum = warp_sum(sum);
        if (lane == 0) {
          reinterpret_cast<float*>(f + C::F_BIAS)[h] = sum * -7.62939453125e-6f;  // -128 2^-24
          reinterpret_cast<float*>(f + C::F_FACTOR)[h] = ldexpf(sl2, 12 - ex);
        }
      }
      if (ht == 0) s_seg[slot] = w;
      helper_sync();
      if (ht == 0) mbar_arrive(&ready[slot]);
    };
    W coming = w0;
    bool more = true;
    load_q(coming);
    for (int i = 0; i < kSlots && more; ++i) {
      prepare(coming, i);
      more = coming.next(a, pad);
      if (more) load_q(coming);  // on its way until a slot is free
    }
    int slot = 0, pieces = 0;
    uint32_t phase = 0;
    while (true) {
      if (ht == 0) s_ok = mbar_wait(&done[slot], phase, abort_flag, a.err, kErrTimeoutEpilogue);
      helper_sync();
      if (!s_ok) break;
      const W w = s_seg[slot];
      const int hk = w.h / a.blocks, h0 = (w.h % a.blocks) * kHeads, nh = min(kHeads, a.rep - h0);
      // the warps' weights: eight neighbouring threads have a head's eight states
      if (ht < kHeads * kWarps) {
        const int h = ht / kWarps, k = ht % kWarps;
        const float m1 = sm[slot][k][h];
        float M = m1;
#pragma unroll
        for (int o = 1; o < kWarps; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float e = m1 == -INFINITY ? 0.f : ex2(m1 - M);
        float L = sl[slot][k][h] * e;
#pragma unroll
        for (int o = 1; o < kWarps; o <<= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        weight[h][k] = e;
        if (k == 0) {
          total_max[h] = M;
          total_sum[h] = L;
        }
      }
      helper_sync();
      // a whole segment is done, a piece of one goes to the workspace
      const bool whole = w.whole();
      const int part = 2 * blockIdx.x + (w.first == 0 ? 1 : 0);
      const float* states = reinterpret_cast<const float*>(smem + C::STATES + slot * kWarps * C::STATE);
      for (int i = ht; i < nh * (HD / 4); i += 32 * kHelpers) {
        const int h = i / (HD / 4), ch = 4 * (i % (HD / 4));
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k = 0; k < kWarps; ++k) {
          const float4 v = *reinterpret_cast<const float4*>(states + k * (C::STATE / 4) + h * C::LD + ch);
          const float e = weight[h][k];
          x.x = fmaf(v.x, e, x.x);
          x.y = fmaf(v.y, e, x.y);
          x.z = fmaf(v.z, e, x.z);
          x.w = fmaf(v.w, e, x.w);
        }
        const float L = total_sum[h];
        if (whole) {
          const float e = L == 0.f ? 0.f : 1.f / L;
          *reinterpret_cast<uint2*>(a.out + ((int64_t)w.b * a.Hq + hk * a.rep + h0 + h) * HD + ch) =
              make_uint2(pack_bf16x2(x.x * e, x.y * e), pack_bf16x2(x.z * e, x.w * e));
        } else {
          float* pp = a.part + ((int64_t)part * kHeads + h) * C::PART;
          *reinterpret_cast<float4*>(pp + ch) = x;
          if (ch == 0) *reinterpret_cast<float2*>(pp + HD) = make_float2(total_max[h], L);
        }
      }
      if (!whole) {  // at most the first and the last segment of the share
        if (ht == 0) s_piece[pieces] = {w.b, w.h, w.begin, (uint32_t)(w.U - pad), false};
        ++pieces;
      }
      if (!w.more()) break;
      helper_sync();  // the states and weights have been read
      if (more) {
        prepare(coming, slot);
        more = coming.next(a, pad);
        if (more) load_q(coming);
      }
      if (++slot == kSlots) {
        slot = 0;
        phase ^= 1;
      }
    }
    if (ht == 0) s_pieces = pieces;
  } else {
    // ───────────────────────────── compute ─────────────────────────────
    const int g = lane / 4, t = lane % 4;
    // token of matrix rows g and (8 further on) g + 8; V's are t, t + 4, t + 8, t + 12
    const int tok_g = g / 2 + 4 * (g % 2);
    const uint32_t ring = smem_u32(smem) + warp * C::WARP;
    // this lane's places in a block: of K, chunk t of row tok_g (and chunk t + 4, 64 bytes across); of V, its channels of
    // rows t and t + 4
    const uint32_t k_at = chunk_at<HD>(tok_g, t);
    const uint32_t v_at = HD == 128 ? chunk_at<HD>(t, g) : chunk_at<HD>(t, g / 2) + g % 2 * 8;
    const uint32_t v_at4 = HD == 128 ? chunk_at<HD>(t + 4, g) : chunk_at<HD>(t + 4, g / 2) + g % 2 * 8;
    constexpr int ROWS = 512 / HD;  // rows of a warp's copy
    const uint32_t copy_at = chunk_at<HD>(lane / (HD / 16), lane % (HD / 16));
    if (lane == 0) s_ahead[warp] = w0;
    __syncwarp();

    // The copies run STAGES - 1 units ahead of the arithmetic, across the segments; a unit's page ids are read one step
    // before its copies start, a block's by every NT-th lane.
    constexpr int kDone = -(1 << 30);  // the share holds no more units for this warp
    const int sub = lane % NT;
    int f_end, f_at, f_wrap, f_page;  // f_at: block within the page of all heads, f_wrap: where this head's part ends
    int f_block, f_blocks;            // of the row: this lane's, all of them
    const int* f_bt;
    const int step_pi = NT * kWarps / a.bpp, step_off = NT * kWarps % a.bpp;
    const uint8_t* kp = a.c.k + lane * 16;
    const uint8_t* vp = a.c.v + lane * 16;
    int f_unit = w0.first_of(warp);
    auto aim = [&](const W& w) {
      f_end = w.end();
      f_block = f_unit * NT + sub;
      f_blocks = (w.n + kTok - 1) / kTok;
      f_at = w.h / a.blocks * a.bpp;
      f_wrap = f_at + a.bpp;
      f_at += f_block % a.bpp;
      f_bt = a.bt + w.b * a.bt_stride + f_block / a.bpp;
    };
    auto settle = [&]() {  // on this warp's next unit, if its share has one
      if (f_unit >= f_end) {
        W w = s_ahead[warp];
        do {
          if (!w.next(a, pad)) {
            f_unit = kDone;
            f_end = 0;
            break;
          }
          f_unit = w.first_of(warp);
          aim(w);
        } while (f_unit >= f_end);
        __syncwarp();
        if (lane == 0) s_ahead[warp] = w;
        __syncwarp();
      }
      f_page = -1;
      if (f_unit >= 0 && (NT == 1 || f_block < f_blocks)) f_page = *f_bt;
    };
    uint32_t valid = 0;  // bits i NT ..: the blocks of the unit i steps ahead have a page
    auto fetch = [&](uint32_t stage, int steps) {
      const bool there = (uint32_t)f_page < (uint32_t)a.c.n_pages;
      const uint32_t n = there ? (uint32_t)f_page * (uint32_t)a.page_blocks + (uint32_t)f_at : 0u;  // block of the cache
      const uint32_t bits = __ballot_sync(0xffffffffu, there) & ((1u << NT) - 1u);
      valid |= bits << (NT * steps);
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        const uint64_t at = (uint64_t)(NT == 1 ? n : __shfl_sync(0xffffffffu, n, x)) * C::BLOCK;
        const bool ok = bits >> x & 1u;
        const uint32_t dst = stage + x * C::BLOCK;
#pragma unroll
        for (int i = 0; i < C::BLOCK / 512; ++i) {
          // the chunk's place depends on the row's bit 2 too: odd copies at head width 128
          const uint32_t to = dst + 512 * i + (HD == 128 && i % 2 ? copy_at ^ 64u : copy_at);
          copy16(to + C::K, kp + at + 512 * i, ok);
          copy16(to + C::V, vp + at + 512 * i, ok);
        }
      }
      if (lane < NT) copy8(stage + C::S + 8 * lane, a.c.scale + 2 * (uint64_t)n, there);
      copies_commit();
      f_unit += kWarps;
      f_block += NT * kWarps;
      f_bt += step_pi;
      f_at += step_off;
      if (f_at >= f_wrap) {
        f_at -= a.bpp;
        ++f_bt;
      }
      settle();
    };
    static_assert(ROWS == (HD == 128 ? 4 : 8), "a copy holds rows of one residue to ROWS");
    aim(w0);
    settle();
    for (int i = 0; i < C::STAGES - 1; ++i) fetch(ring + i * C::STAGE, i);
    uint32_t stage = ring, ahead = ring + (C::STAGES - 1) * C::STAGE;
    int slot = 0;
    uint32_t phase = 0;

    while (true) {
      if (!__all_sync(0xffffffffu, mbar_wait(&ready[slot], phase, abort_flag, a.err, kErrTimeoutMma))) break;
      const W* seg = &s_seg[slot];
      const int n_tok = seg->n, u_end = seg->end();
      int unit = seg->first_of(warp);
      const bool more = seg->more();
      const uint8_t* frags = smem + C::F + slot * C::FBYTES;
      float bias[2], cs[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        bias[r] = reinterpret_cast<const float*>(frags + C::F_BIAS)[2 * t + r];
        cs[r] = reinterpret_cast<const float*>(frags + C::F_FACTOR)[2 * t + r];
      }
      const uint32_t frag_at = smem_u32(frags) + lane * 16;
      // o and l are relative to the reference m: p 2^-m, so that x fits fp16 well
      float o[2 * VW][4], m[2] = {0.f, 0.f}, l[2] = {0.f, 0.f};
      float limit = -1.f;  // below 0: no reference yet
#pragma unroll
      for (int i = 0; i < 2 * VW; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      for (; unit < u_end; unit += kWarps) {
        copies_wait<C::STAGES - 2>();
        __syncwarp();  // and every lane has read the stage that is filled again below
        const uint32_t here = stage;
        // tokens of the unit to be counted; the rest may be anything
        const int count = n_tok - unit * C::UTOK;
        const uint32_t pieces = valid & ((1u << NT) - 1u);
        valid >>= NT;
        fetch(ahead, C::STAGES - 2);
        ahead = stage;
        stage = stage + C::STAGE == ring + C::WARP ? ring : stage + C::STAGE;
        // everything the unit needs from shared memory is asked for at once
        uint32_t kw[NT][2][KW], qf[KW / 2][4], vw[NT][4][VW];
        float2 sc[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            load_words<4>(kw[n][i], here + C::K + n * C::BLOCK + i * (C::BLOCK / 2) + k_at);
            if constexpr (KW == 8) load_words<4>(kw[n][i] + 4, here + C::K + n * C::BLOCK + i * (C::BLOCK / 2) + (k_at ^ 64u));
          }
#pragma unroll
        for (int j = 0; j < KW / 2; ++j) load_words<4>(qf[j], frag_at + j * 512);
#pragma unroll
        for (int n = 0; n < NT; ++n) load_words<2>(reinterpret_cast<uint32_t*>(&sc[n]), here + C::S + 8 * n);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            load_words<VW>(vw[n][i], here + C::V + n * C::BLOCK + i / 2 * (C::BLOCK / 2) + (i % 2 ? v_at4 : v_at));
        // scores: block n, row g + 8 i, head 2 t + r
        float s[NT][2][2];
        {
          float acc[NT][2][4];  // two chains each
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[n][0][0] = acc[n][0][2] = bias[0], acc[n][0][1] = acc[n][0][3] = bias[1];
#pragma unroll
          for (int j = 0; j < KW; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint32_t w0 = kw[n][0][j], w1 = kw[n][1][j];
              const uint32_t a0 = w0 & 0x00FF00FFu, a1 = w1 & 0x00FF00FFu;
              const uint32_t a2 = __byte_perm(w0, 0u, 0x4341), a3 = __byte_perm(w1, 0u, 0x4341);
              if (j == 1)
                mma_f16_first(acc[n][1], a0, a1, a2, a3, qf[j / 2][j % 2 * 2], qf[j / 2][j % 2 * 2 + 1]);
              else
                mma_f16(acc[n][j % 2], a0, a1, a2, a3, qf[j / 2][j % 2 * 2], qf[j / 2][j % 2 * 2 + 1]);
            }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float a1 = sc[n].x * 4096.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                s[n][i][r] = fmaf((acc[n][0][2 * i + r] + acc[n][1][2 * i + r]) * a1, cs[r], -m[r]);
          }
        }
        if (count < C::UTOK || pieces != (1u << NT) - 1u) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (n * kTok >= count || !(pieces >> n & 1u)) sc[n].y = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (n * kTok + tok_g + 8 * i >= count || !(pieces >> n & 1u)) s[n][i][0] = s[n][i][1] = -INFINITY;
          }
        }
        float p[NT][2][2], top_x = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float a1 = fmaxf(sc[n].y, kMinA);
          float top = 0.f;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              p[n][i][r] = ex2(s[n][i][r]);
              top = fmaxf(top, p[n][i][r]);
            }
          top_x = fmaxf(top_x, top * a1);
        }
        if (__any_sync(0xffffffffu, top_x > limit)) {
          // move the reference: to the largest p a', less what brings that to 2^kBoost
          bool found = false;
          float keep[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; ++n) top = fmaxf(top, fmaxf(s[n][0][r], s[n][1][r]) + lg2(fmaxf(sc[n].y, kMinA)));
            top = max_over_rows(top) + m[r];
            if (limit > 0.f) top = fmaxf(top, m[r] + kBoost);
            const bool real = top != -INFINITY;
            const float to = real ? top - kBoost : m[r];
            keep[r] = limit > 0.f ? ex2(m[r] - to) : 0.f;
            found |= real;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 2; ++i) p[n][i][r] = ex2(s[n][i][r] + (m[r] - to));
            m[r] = to;
            l[r] *= keep[r];
          }
          if (__any_sync(0xffffffffu, found)) limit = kLimit;
#pragma unroll
          for (int q = 0; q < 2 * VW; ++q)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[q][x] *= keep[x & 1];
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int r = 0; r < 2; ++r) l[r] += p[n][0][r] + p[n][1][r];
          const uint32_t b0 = transpose8x8(pack_half2(p[n][0][0] * sc[n].y, p[n][0][1] * sc[n].y));
          const uint32_t b1 = transpose8x8(pack_half2(p[n][1][0] * sc[n].y, p[n][1][1] * sc[n].y));
          constexpr uint32_t kBias = 0x80808080u;  // -128 2^-24, twice
#pragma unroll
          for (int j = 0; j < 2 * VW; ++j) mma_f16(o[j], kBias, kBias, kBias, kBias, b0, b1);
#pragma unroll
          for (int j = 0; j < VW; ++j)
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // bytes 2 half, 2 half + 1: rows g and g + 8
              const uint32_t sel = half ? 0x7632u : 0x5410u;
              const uint32_t x = __byte_perm(vw[n][0][j], vw[n][1][j], sel), y = __byte_perm(vw[n][2][j], vw[n][3][j], sel);
              mma_f16(o[2 * j + half], x & 0x00FF00FFu, __byte_perm(x, 0u, 0x4341), y & 0x00FF00FFu,
                      __byte_perm(y, 0u, 0x4341), b0, b1);
            }
        }
      }

      // the warp's state: o in units of V, relative to m
      float* state = reinterpret_cast<float*>(smem + C::STATES + (slot * kWarps + warp) * C::STATE);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] = sum_over_rows(l[r]);
        float4* d = reinterpret_cast<float4*>(state + (2 * t + r) * C::LD + HD / 8 * g);
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          constexpr float f = 16777216.f;
          d[j] = make_float4(o[2 * j][r] * f, o[2 * j][2 + r] * f, o[2 * j + 1][r] * f, o[2 * j + 1][2 + r] * f);
        }
        if (g == 0) {
          sm[slot][warp][2 * t + r] = limit < 0.f ? -INFINITY : m[r];
          sl[slot][warp][2 * t + r] = l[r];
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&done[slot]);
      if (!more) break;
      if (++slot == kSlots) {
        slot = 0;
        phase ^= 1;
      }
    }
    copies_wait<0>();
  }

  __syncthreads();
  const int pieces = s_pieces;
  if (pieces) join_pieces<HD, kThreads>(a, plan.shares, s_piece, pieces, a.part, a.arrived, a.blocks, a.rep, a.Hq, a.out);
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
  using C = Cfg<HD>;
  // blocks are counted in 32 bits, in the cache and over the rows
  MESHY_CHECK(a.c.n_pages * (int64_t)a.page_blocks < (1LL << 32) - 1, "paged_attention_kv8: cache too large");
  MESHY_CHECK((int64_t)a.B * a.per_row * ((int64_t)a.max_pages * a.bpp + 1 + kRules.pad) < (1LL << 31),
              "paged_attention_kv8: rows * heads * table width too large");
  static bool set[64] = {};
  int dev = 0;
  MESHY_CUDA_CHECK(cudaGetDevice(&dev));
  if (!set[dev]) {
    MESHY_CUDA_CHECK(cudaFuncSetAttribute(kv8_attn_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    set[dev] = true;
  }
  launch_pdl(kv8_attn_kernel<HD>, dim3(sm_count()), dim3(kThreads), C::SMEM, st, a);
}

}  // namespace

int64_t kv8_attention_segments(int B, int Hq, int Hkv) { return (int64_t)B * Hkv * ((Hq / Hkv + kHeads - 1) / kHeads); }
int64_t kv8_part_floats() { return (int64_t)2 * sm_count() * kHeads * Cfg<128>::PART; }

void kv8_attention(const bf16* q, int64_t qs, int64_t qh, KV8View c, const int* bt, int64_t bt_stride, int max_pages,
                   const int* seq_lens, int B, int Hq, float scale, bf16* out, float* part, unsigned* arrived, int* err,
                   cudaStream_t st) {
  if (B == 0) return;
  max_pages = std::min(max_pages, (INT_MAX - 63) / c.page);  // lengths are rounded up to units in 32 bits
  Args a;
  const int rep = Hq / c.Hkv, blocks = (rep + kHeads - 1) / kHeads, bpp = c.page / kTok;
  static_cast<Rows&>(a) = {seq_lens, B, max_pages, c.page, c.Hkv * blocks};
  a.q = q, a.qs = qs, a.qh = qh, a.c = c, a.bt = bt, a.bt_stride = bt_stride, a.Hq = Hq, a.rep = rep, a.blocks = blocks;
  a.bpp = bpp, a.page_blocks = c.Hkv * bpp, a.scale = scale, a.out = out, a.part = part, a.arrived = arrived, a.err = err;
  c.hd == 128 ? launch<128>(a, st) : launch<64>(a, st);
}

}  // namespace meshy
