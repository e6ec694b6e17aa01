// Paged decode attention over the 8-bit KV cache (layout in kv8.h).
//
//   s_j = scale a_j (q . (u_j - 128)),  p = softmax(s),  o = sum_j p_j a'_j (u'_j - 128)
//
// The 16 tokens of a block share a scale, so scales leave the channel sums and the bytes go to the tensor cores as whole
// numbers: a byte in the low half of a 16-bit word is the fp16 subnormal u 2^-24, exact and with no conversion. The 128
// that u carries too much is a constant of the query in the scores (the accumulators start at -128 sum(q)) and one more
// product in the output (a matrix of -128 against a block's weights, added before the block's own product, so that sums stay
// near zero and lose no bits to it).
//
// A warp takes a block at a time (m16n8k16, fp16 in, fp32 sums):
//   S^T [16 tokens, 8 heads] = K [16, hd] Q^T      A rows are tokens: a word of a K row is two operands, masked and moved
//   O^T [16 channels, 8 heads] += V^T [16, 16 tokens] P^T    A rows are channels: a byte permute pairs two tokens' words
// Query heads that share a KV head fill the 8 columns, so every cached byte is read once for up to 8 heads. P changes
// from accumulator to operand by movmatrix. The copies swizzle the 16-byte chunks of 128 bytes by the line, and the tokens
// are dealt to the matrix rows so that lanes that read together, of K or of V, meet in no bank. tcgen05 would not help:
// the operands would have to be unpacked and stored once more before it could read them, and 8 query rows leave it nothing
// to win.
//
// P carries the scale of V (x = p a'), so a reference m per warp and head keeps it in fp16's range: p is taken relative
// to m, which is set so that the largest p a' seen is 2^11, and moves again only when a later one passes 2^15. So most
// blocks take neither the maximum's shuffles nor a rescaling. x is rounded to fp16's 11 bits, or by 2^-25 where it is
// below 2^-14: less than 2^-35 of the largest. Scales below 2^-64 count as that for the reference. All of V's scales are
// taken 2^-16 times, which keeps p between 2^-92 (the largest, beside values of 2^126) and 2^95 in fp32's range with the
// weights that count; sums and the normaliser stay in 32 bits. The 11 bits add up to 8e-6 to the bf16 output's error of 1.6e-3
// (root mean square); x in two terms, 22 bits, would take that away for 88.2 us instead of 87.0 on the 8 long rows, 95.5 for
// 92.4 at width 64 and 109.7 for 106.5 on the 256.
//
// Eight warps compute and never wait for one another: each keeps a ring of units of its own in shared memory (a unit is
// a block at head width 128, two at 64: the same bytes), filled by 16-byte asynchronous copies kStages - 1 units ahead,
// across the segments, and at a segment's end leaves its state in one of kSlots slots and goes on. Four helper warps prepare
// the query fragments of the coming segments and join the eight states of the finished ones; the states of a share's last
// segment are joined by all twelve. Every wait is bounded; one that gives up records an error code, and the CTA's pieces are
// counted all the same. How the work is split over CTAs stands in kv_split.cuh.
//
// Measured: 8 rows of 131072 tokens (16 / 2 heads, 128 wide, 538 MB) 87 us, 6.2 TB/s; 128 rows of 16384 at head width 64
// (14 / 2, 540 MB) 92 us, 5.9 TB/s; 256 rows of up to 1500 (32 / 8 heads, 639 MB) 106.5 us, 6.0 TB/s; 64 rows of up to 8192 (12
// / 2, 125 MB) 28 us; one row of 700 tokens 7.2 us. Long rows are bound by memory (a copy runs at 6.5 TB/s; 42 % of the
// issue slots are busy), few tokens by the chain of lengths, page ids, copies, join (3.5 us for a row without tokens).
// Copies of whole 2 KB boxes by TMA took 102 us on the first, units of two blocks at width 128 spilled and took 101. A
// ring of four: 104.5 us on the 256 rows, but 13.9 -> 14.7 on 33 rows of up to 4000 and 13.5 -> 14.6 on one of 32768, as
// three slots did (14.3).
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
constexpr int kStages = 3;
constexpr int kSlots = 2;  // segments whose fragments or states are held
// (us; as in kv_split.cuh) Equal segments up to 32 units are taken whole (a row of 512 tokens with cold caches 8.4, cut 9.1;
// of 700 whole 9.5, cut 9.3); a change of segments counts as 24 units (64 rows of up to 8192 tokens 28.4, 8 units 31.9, 48
// units 28.7, none 33.7; 64 rows of up to 600 and 8 KV heads 17.5, 21.9, 18.1, 39.5); a join is worth 6 steps (64 rows of
// 4096 26.8, 2 steps 30.1, 16 steps 26.8; 8 rows of 131072 88, 2 steps 89.7).
constexpr Rules kRules{32, 24, 6};
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBoost = 11.f;           // log2 of the largest p a' right after the reference moved
constexpr float kLimit = 32768.f;        // how far later ones may go
constexpr float kShrink = 1.52587890625e-5f;       // 2^-16, times V's scales
constexpr float kMinA = 5.42101086e-20f * kShrink;  // 2^-64
constexpr float kUnit = 16777216.f;                // 2^24: the bytes stand for 2^-24 of themselves

template <int HD>
struct Cfg {
  static constexpr int NT = 128 / HD;                   // blocks of a unit
  static constexpr int UTOK = NT * kTok;
  static constexpr int BLOCK = kTok * HD;               // bytes of a block of K
  static constexpr int K = 0, V = NT * BLOCK, STAGE = 2 * NT * BLOCK;
  static constexpr int SCALES = kWarps * kStages * STAGE;  // a pair (K, V) for each block of each stage
  static constexpr int LD = HD + 4;                     // row stride of a state: spreads the heads over the banks
  static constexpr int STATES = SCALES + kWarps * kStages * NT * 8;  // kSlots sets of the warps' states
  static constexpr int STATE = kHeads * LD * 4;
  // kSlots sets of query fragments: matrix B, -128 sum(q), factors
  static constexpr int F = STATES + kSlots * kWarps * STATE;
  static constexpr int KW = HD / 16;                    // K words of a lane and row
  static constexpr int F_BIAS = KW * 32 * 8, F_FACTOR = F_BIAS + kHeads * 4;
  static constexpr int FBYTES = F_FACTOR + kHeads * 4;
  static constexpr int SMEM = F + kSlots * FBYTES;
  static constexpr int PART = HD + 4;                   // floats of a head in the workspace: sums, maximum, normaliser
  static_assert(STAGE == 4096 && SMEM + 4096 <= 232448);
};

// Token of a block that matrix row r (0 .. 7, or those less 8) stands for. Rows 2 i and 2 i + 1 lie in different halves of
// their swizzled lines, and rows 0, 2, 4, 6 (or 1, 3, 5, 7) spread over all eight chunks.
template <int HD>
__device__ __forceinline__ int token_of(int r) {
  if constexpr (HD == 128) return r ^ (r & 1) << 2;
  return (r & 4) + (r & 1 ? 3 - (r & 3) / 2 : (r & 3) / 2);
}
// Where chunk c (16 bytes) of a block's token j stands: lines of 128 bytes, chunks swizzled by the line.
template <int HD>
__device__ __forceinline__ uint32_t chunk_at(int j, int c) {
  if constexpr (HD == 128) return j * 128 + 16 * (c ^ (j & 7));
  return j / 2 * 128 + 16 * ((j % 2 * 4 + c) ^ (j / 2 & 7));
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
  long long wait;  // cycles after which a wait gives up
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    kv8_attn_kernel(const Args a) {
  using C = Cfg<HD>;
  using W = Walk<C::UTOK, kWarps>;
  constexpr int NT = C::NT, KW = C::KW, VW = HD / 32;  // V words of a lane and row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(16) float sm[kSlots][kHeads][kWarps], sl[kSlots][kHeads][kWarps];
  __shared__ W s_seg[kSlots], s_ahead[kWarps];
  __shared__ uint64_t ready[kSlots], done[kSlots];  // fragments are there and the states free; the states are there
  __shared__ Piece s_piece[2];
  __shared__ PlanShared<kThreads> s_plan;
  __shared__ Start<W> s_start;
  __shared__ int s_pieces, s_abort, s_ok;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  volatile int* abort_flag = &s_abort;

  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&ready[i], 1);
      mbar_init(&done[i], kWarps);
    }
    s_abort = 0;
  }
  fence_mbar_init();
  pdl_wait();
  pdl_trigger();
  const auto plan = make_plan<C::UTOK, kWarps, kThreads>(a, s_plan, kRules);
  if (!plan.work) return;
  const W w0 = plan.w;
  const int pad = plan.pad;
  int slot = 0;  // of the segment at hand; at the end, of the share's last

  // The eight warps' states of a segment, joined by n threads of which this is the i-th: a whole segment is done, a piece
  // of one goes to the workspace.
  auto join_states = [&](const W& w, int slot, int i, int n) {
    const int hk = w.h / a.blocks, h0 = (w.h % a.blocks) * kHeads, nh = min(kHeads, a.rep - h0);
    const float* states = reinterpret_cast<const float*>(smem + C::STATES + slot * kWarps * C::STATE);
    for (; i < nh * (HD / 4); i += n) {
      const int h = i / (HD / 4), ch = 4 * (i % (HD / 4));
      float m1[kWarps], l1[kWarps], M = -INFINITY, L = 0.f;
      float4 v[kWarps], x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kWarps; k += 4) {
        *reinterpret_cast<float4*>(m1 + k) = *reinterpret_cast<const float4*>(&sm[slot][h][k]);
        *reinterpret_cast<float4*>(l1 + k) = *reinterpret_cast<const float4*>(&sl[slot][h][k]);
      }
#pragma unroll
      for (int k = 0; k < kWarps; ++k) v[k] = *reinterpret_cast<const float4*>(states + k * (C::STATE / 4) + h * C::LD + ch);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) M = fmaxf(M, m1[k]);
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        const float e = m1[k] == -INFINITY ? 0.f : ex2(m1[k] - M);
        L = fmaf(l1[k], e, L);
        x.x = fmaf(v[k].x, e, x.x);
        x.y = fmaf(v[k].y, e, x.y);
        x.z = fmaf(v[k].z, e, x.z);
        x.w = fmaf(v[k].w, e, x.w);
      }
      constexpr float f = kUnit / kShrink;
      x.x *= f, x.y *= f, x.z *= f, x.w *= f;  // (before the division: L may be as small as p)
      if (w.whole()) {
        const float e = L == 0.f ? 0.f : __fdividef(1.f, L);
        *reinterpret_cast<uint2*>(a.out + ((int64_t)w.b * a.Hq + hk * a.rep + h0 + h) * HD + ch) =
            make_uint2(pack_bf16x2(x.x * e, x.y * e), pack_bf16x2(x.z * e, x.w * e));
      } else {
        float* pp = a.part + ((int64_t)(2 * blockIdx.x + (w.first == 0 ? 1 : 0)) * kHeads + h) * C::PART;
        *reinterpret_cast<float4*>(pp + ch) = x;
        if (ch == 0) *reinterpret_cast<float2*>(pp + HD) = make_float2(M, L);
      }
    }
  };

  if (warp >= kWarps) {
    // ───────────────────────────── helpers ─────────────────────────────
    const int hw = warp - kWarps, ht = tid - 32 * kWarps;
    // A segment's query rows as matrix fragments, a warp per head: scaled so that the largest is in [2^14, 2^15); -128
    // times their sum, in units of 2^-24 as the products are; the factor that takes the query's power back, with the softmax
    // scale.
    constexpr int CH = HD / 32;  // channels of a lane
    const float sl2 = a.scale * kLog2e;
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
      float x[kHeads / kHelpers][CH], mx[kHeads / kHelpers], sum[kHeads / kHelpers], down[kHeads / kHelpers];
#pragma unroll
      for (int k = 0; k < kHeads / kHelpers; ++k) {
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
          const float2 y = unpack_bf16x2(raw[k][i]);
          x[k][2 * i] = y.x;
          x[k][2 * i + 1] = y.y;
        }
        mx[k] = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) mx[k] = fmaxf(mx[k], fabsf(x[k][i]));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < kHeads / kHelpers; ++k) mx[k] = fmaxf(mx[k], __shfl_xor_sync(0xffffffffu, mx[k], o));
#pragma unroll
      for (int k = 0; k < kHeads / kHelpers; ++k) {
        // 2^14 over the largest's power of two; magnitudes below 2^-100 as they are there
        const uint32_t power = min(max(__float_as_uint(mx[k]), 27u << 23), (254u << 23)) & 0x7F800000u;
        const float up = __uint_as_float(((127u + 14u + 127u) << 23) - power);
        down[k] = __uint_as_float(power - (14u << 23));
        sum[k] = 0.f;
        __half y[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          y[i] = __float2half_rn(x[k][i] * up);
          sum[k] += __half2float(y[i]);
        }
        // channel ch: chunk ch / 16 belongs to lane (ch / 16) % 4 of a matrix row, byte e = ch % 4 of its word w; bytes 0, 2
        // are operand 0, bytes 1, 3 operand 1
        const int h = hw + k * kHelpers, ch = lane * CH, t = ch / 16 % 4, w = ch % 16 / 4 + 4 * (ch / 64);
        uint32_t* at = reinterpret_cast<uint32_t*>(f) + (w / 2 * 32 + h * 4 + t) * 4 + w % 2 * 2;
        if constexpr (CH == 4) {
          *reinterpret_cast<__half2*>(at) = __halves2half2(y[0], y[2]);
          *reinterpret_cast<__half2*>(at + 1) = __halves2half2(y[1], y[3]);
        } else {
          reinterpret_cast<__half*>(at)[lane % 2] = y[0];
          reinterpret_cast<__half*>(at + 1)[lane % 2] = y[1];
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < kHeads / kHelpers; ++k) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < kHeads / kHelpers; ++k) {
          reinterpret_cast<float*>(f + C::F_BIAS)[hw + k * kHelpers] = sum[k] * -7.62939453125e-6f;  // -128 2^-24
          reinterpret_cast<float*>(f + C::F_FACTOR)[hw + k * kHelpers] = sl2 * down[k];
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
    if (ht == 64) s_start = {w0, plan.shares, pad};  // (before the first wait; at the kernel's start it costs 0.3 us)
    int pieces = 0;
    uint32_t phase = 0;
    while (true) {
      const W w = s_seg[slot];
      if (!w.whole()) {  // at most the first and the last segment of the share
        if (ht == 32) s_piece[pieces] = piece_of(w, pad, plan.shares);
        ++pieces;
      }
      if (!w.more()) break;
      if (ht == 0) s_ok = mbar_wait(&done[slot], phase, abort_flag, a.err, kErrTimeoutEpilogue, a.wait);
      helper_sync();
      if (!s_ok) break;
      join_states(w, slot, ht, 32 * kHelpers);
      helper_sync();  // the states have been read
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
    const uint32_t ring = smem_u32(smem) + warp * (kStages * C::STAGE);
    float2* const scales = reinterpret_cast<float2*>(smem + C::SCALES) + warp * (kStages * NT);
    // this lane's places in a block: of K, chunk t of row g's token (and chunk t + 4, 64 bytes across); of V, its channels
    // of the tokens of rows 2 t and 2 t + 1; rows 8 further on are tokens 8 further on
    const uint32_t k_at = chunk_at<HD>(token_of<HD>(g), t);
    const uint32_t v_at0 = HD == 128 ? chunk_at<HD>(token_of<HD>(2 * t), g) : chunk_at<HD>(token_of<HD>(2 * t), g / 2) + g % 2 * 8;
    const uint32_t v_at1 =
        HD == 128 ? chunk_at<HD>(token_of<HD>(2 * t + 1), g) : chunk_at<HD>(token_of<HD>(2 * t + 1), g / 2) + g % 2 * 8;
    // at head width 64 the line's bit 2 changes with the half of the block: the chunk's moves too
    constexpr uint32_t kFar = HD == 128 ? 0u : 64u;
    if (lane == 0) s_ahead[warp] = w0;
    __syncwarp();

    // The copies run kStages - 1 units ahead of the arithmetic, across the segments; a unit's page ids are read one step
    // before its copies start.
    constexpr int kDone = -(1 << 30);  // the share holds no more units for this warp
    const int sub = lane % NT;
    int f_end, f_at, f_wrap;  // f_at: block within the page of all heads, f_wrap: where this head's part ends
    int f_block, f_blocks;    // of the row: this lane's, all of them
    const int* f_bt;
    const int step_pi = NT * kWarps / a.bpp, step_off = NT * kWarps % a.bpp;
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
    struct Look {
      int page, at;  // of this lane's block of a unit
    };
    auto look = [&]() {  // at this warp's next unit, if its share has one
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
      Look x{-1, f_at};
      if (f_unit >= 0 && (NT == 1 || f_block < f_blocks)) x.page = *f_bt;
      f_unit += kWarps;
      f_block += NT * kWarps;
      f_bt += step_pi;
      f_at += step_off;
      if (f_at >= f_wrap) {
        f_at -= a.bpp;
        ++f_bt;
      }
      return x;
    };
    uint32_t valid = 0;  // bits i NT ..: the blocks of the unit i steps ahead have a page
    int f_stage = 0;
    // line lane / 8 of every four, chunk lane % 8; the lines' bit 2 is the copy's lowest
    const uint32_t copy_at = lane / 8 * 128 + 16 * (lane % 8 ^ lane / 8);
    const uint8_t* const kp = a.c.k + lane * 16;
    const uint8_t* const vp = a.c.v + lane * 16;
    auto fetch = [&](const Look& x, int steps) {
      const bool there = (uint32_t)x.page < (uint32_t)a.c.n_pages;
      const uint32_t n = there ? (uint32_t)x.page * (uint32_t)a.page_blocks + (uint32_t)x.at : 0u;  // block of the cache
      const uint32_t bits = __ballot_sync(0xffffffffu, there) & ((1u << NT) - 1u);
      valid |= bits << (NT * steps);
      const uint32_t stage = ring + f_stage * C::STAGE;
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        const uint64_t at = (uint64_t)(NT == 1 ? n : __shfl_sync(0xffffffffu, n, b)) * C::BLOCK;
        const bool ok = bits >> b & 1u;
#pragma unroll
        for (int i = 0; i < C::BLOCK / 512; ++i) {
          const uint32_t to = stage + b * C::BLOCK + 512 * i + (i % 2 ? copy_at ^ 64u : copy_at);
          copy16(to + C::K, kp + at + 512 * i, ok);
          copy16(to + C::V, vp + at + 512 * i, ok);
        }
      }
      if (lane < NT) copy8(smem_u32(scales + f_stage * NT + lane), a.c.scale + 2 * (uint64_t)n, there);
      copies_commit();
      f_stage = f_stage + 1 == kStages ? 0 : f_stage + 1;
    };
    aim(w0);
    Look seen;
    {
      Look x[kStages - 1];
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) x[i] = look();
      seen = look();
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) fetch(x[i], i);
    }
    int stage = 0;
    uint32_t phase = 0;

    while (true) {
      if (!__all_sync(0xffffffffu, mbar_wait(&ready[slot], phase, abort_flag, a.err, kErrTimeoutMma, a.wait))) break;
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
        copies_wait<kStages - 2>();
        __syncwarp();  // the copies are there for all, and every lane has read the stage that is filled again below
        const uint32_t here = ring + stage * C::STAGE;
        const float2* sc_at = scales + stage * NT;
        // tokens of the unit to be counted; the rest may be anything
        const int count = n_tok - unit * C::UTOK;
        const uint32_t pieces = valid & ((1u << NT) - 1u);
        valid >>= NT;
        if (++stage == kStages) stage = 0;
        // everything the unit needs from shared memory is asked for at once
        uint32_t kw[NT][2][KW], qf[KW / 2][4], vw[NT][4][VW];
        float2 sc[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t at = here + C::K + n * C::BLOCK + i * (C::BLOCK / 2) + (i ? k_at ^ kFar : k_at);
            load_words<4>(kw[n][i], at);
            if constexpr (KW == 8) load_words<4>(kw[n][i] + 4, at ^ 64u);
          }
#pragma unroll
        for (int j = 0; j < KW / 2; ++j) load_words<4>(qf[j], frag_at + j * 512);
#pragma unroll
        for (int n = 0; n < NT; ++n) sc[n] = sc_at[n], sc[n].y *= kShrink;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            load_words<VW>(vw[n][i], here + C::V + n * C::BLOCK + i / 2 * (C::BLOCK / 2) +
                                         ((i % 2 ? v_at1 : v_at0) ^ (i / 2 ? kFar : 0u)));
        fetch(seen, kStages - 2);
        seen = look();
        // scores: block n, row g + 8 i, head 2 t + r
        float s[NT][2][2];
        {
          constexpr int CHAINS = KW / NT >= 4 ? 4 : 2;  // sums that do not wait for one another
          float acc[NT][CHAINS][4];
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[n][0][0] = acc[n][0][2] = bias[0], acc[n][0][1] = acc[n][0][3] = bias[1];
#pragma unroll
          for (int j = 0; j < KW; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint32_t w0 = kw[n][0][j], w1 = kw[n][1][j];
              const uint32_t a0 = w0 & 0x00FF00FFu, a1 = w1 & 0x00FF00FFu;
              const uint32_t a2 = __byte_perm(w0, 0u, 0x4341), a3 = __byte_perm(w1, 0u, 0x4341);
              if (j > 0 && j < CHAINS)
                mma_f16_first(acc[n][j], a0, a1, a2, a3, qf[j / 2][j % 2 * 2], qf[j / 2][j % 2 * 2 + 1]);
              else
                mma_f16(acc[n][j % CHAINS], a0, a1, a2, a3, qf[j / 2][j % 2 * 2], qf[j / 2][j % 2 * 2 + 1]);
            }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                float x = acc[n][0][2 * i + r] + acc[n][1][2 * i + r];
                if constexpr (CHAINS == 4) x += acc[n][2][2 * i + r] + acc[n][3][2 * i + r];
                // |x| < 2^5: in this order nothing is out of fp32's range unless the score is
                s[n][i][r] = fmaf(x * sc[n].x * cs[r], kUnit, -m[r]);
              }
          }
        }
        if (count < C::UTOK || pieces != (1u << NT) - 1u) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (n * kTok >= count || !(pieces >> n & 1u)) sc[n].y = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (n * kTok + token_of<HD>(g) + 8 * i >= count || !(pieces >> n & 1u)) s[n][i][0] = s[n][i][1] = -INFINITY;
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
          float off[4];
          mma_f16_first(off, kBias, kBias, kBias, kBias, b0, b1);
#pragma unroll
          for (int q = 0; q < 2 * VW; ++q)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[q][x] += off[x & 1];
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

      // the warp's state: o in units of 2^-40 V, relative to m
      float* state = reinterpret_cast<float*>(smem + C::STATES + (slot * kWarps + warp) * C::STATE);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] = sum_over_rows(l[r]);
        float4* d = reinterpret_cast<float4*>(state + (2 * t + r) * C::LD + HD / 8 * g);
#pragma unroll
        for (int j = 0; j < VW; ++j) d[j] = make_float4(o[2 * j][r], o[2 * j][2 + r], o[2 * j + 1][r], o[2 * j + 1][2 + r]);
        if (g == 0) {
          sm[slot][2 * t + r][warp] = limit < 0.f ? -INFINITY : m[r];
          sl[slot][2 * t + r][warp] = l[r];
        }
      }
      if (!more) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&done[slot]);
      if (++slot == kSlots) {
        slot = 0;
        phase ^= 1;
      }
    }
    copies_wait<0>();
  }

  __syncthreads();
  if (s_abort) {
    if (tid == 0) arrive_all(a, s_start, a.arrived);
    return;
  }
  const W w = s_seg[slot];
  join_states(w, slot, tid, kThreads);
  const int pieces = s_pieces;
  if (pieces) {
    __syncthreads();
    join_pieces<HD, kThreads>(a, s_piece, pieces, a.part, a.arrived, a.blocks, a.rep, a.Hq, a.out);
  }
}

template <int HD>
void launch(const Args& a, cudaStream_t st) {
  using C = Cfg<HD>;
  // blocks are counted in 32 bits, in the cache and over the rows
  MESHY_CHECK(a.c.n_pages * (int64_t)a.page_blocks < (1LL << 32) - 1, "paged_attention_kv8: cache too large");
  MESHY_CHECK((int64_t)a.B * a.per_row * ((int64_t)a.max_pages * a.bpp + 1 + kRules.pad) < (1LL << 31),
              "paged_attention_kv8: rows * heads * table width too large");
  launch_split<kv8_attn_kernel<HD>>(kThreads, C::SMEM, a, st);
}

}  // namespace

int64_t kv8_attention_segments(int B, int Hq, int Hkv) { return (int64_t)B * Hkv * ((Hq / Hkv + kHeads - 1) / kHeads); }
int64_t kv8_part_floats() { return (int64_t)2 * sm_count() * kHeads * Cfg<128>::PART; }

void kv8_attention(const bf16* q, int64_t qs, int64_t qh, KV8View c, const int* bt, int64_t bt_stride, int max_pages,
                   const int* seq_lens, int B, int Hq, float scale, bf16* out, float* part, unsigned* arrived, int* err,
                   int64_t wait, cudaStream_t st) {
  if (B == 0) return;
  max_pages = std::min(max_pages, (INT_MAX - 63) / c.page);  // lengths are rounded up to units in 32 bits
  Args a;
  const int rep = Hq / c.Hkv, blocks = (rep + kHeads - 1) / kHeads, bpp = c.page / kTok;
  static_cast<Rows&>(a) = {seq_lens, B, max_pages, c.page, c.Hkv * blocks};
  a.q = q, a.qs = qs, a.qh = qh, a.c = c, a.bt = bt, a.bt_stride = bt_stride, a.Hq = Hq, a.rep = rep, a.blocks = blocks;
  a.bpp = bpp, a.page_blocks = c.Hkv * bpp, a.scale = scale, a.out = out, a.part = part, a.arrived = arrived, a.err = err;
  a.wait = wait < 0 ? kWaitCycles : wait;
  c.hd == 128 ? launch<128>(a, st) : launch<64>(a, st);
}

}  // namespace meshy
