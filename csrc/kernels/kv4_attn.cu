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
// P carries the scale of V (x = p a'), so a reference m per warp and head keeps it in fp16's range: p is taken relative
// to m, which is set so that the largest p a' seen, a' being the larger scale of a token's groups, is 2^11, and moves
// again only when a later one passes 2^15. So most units take neither the maximum's shuffles nor a rescaling. x is
// rounded to fp16's 11 bits, or by 2^-25 where it is below 2^-14: less than 2^-35 of the largest p a'. (A reference for
// the largest p and the largest a' apart lost the values of a long tail where tokens of no weight had values that spread
// 2^16 times as far.) Scales below 2^-24, the smallest there is, count as that, so that p stays below 2^39; sums, the
// normaliser and the bases' part stay in 32 bits.
//
// Work split (kv_split.cuh): units of 32 tokens, 64 at head width 64 (the same bytes, and enough of them under way to hide
// the memory's latency); one CTA per SM.
//
// A unit lies in one page, or, where the page is not a multiple of it, in pieces of 16 or 32 tokens whose page ids
// neighbouring lanes look up (8 rows of 131072 tokens: 68 us with pages of 16, 65 with pages of 64; units of 16 tokens
// took 82 with the former. At head width 64, 128 rows of 16384: 72, 71 and 131).
//
// Eight warps compute and never wait for one another: each keeps a ring of units of its own in shared memory, filled by
// 16-byte asynchronous copies two units ahead, across the segments, and at a segment's end leaves its state in one of
// kSlots slots and goes on. Four helper warps prepare the query fragments of the coming segments and join the eight
// states of the finished ones behind the others' backs. (With the joins in the computing warps' way, 256 rows of about
// 1200 tokens took 105 us instead of 96; two CTAs of eight such warps and 128 registers each ran no faster on long rows
// than one CTA with 168, as one of the two is always favoured and the other finishes alone; copies issued by warps of
// their own left fewer registers and one more wait to a unit: 72 us instead of 66 on 8 rows of 131072 tokens.) Every
// wait is bounded; one that gives up records an error code.
//
// Measured: 8 rows of 131072 tokens (16 / 2 heads, 128 wide, 302 MB) 65-69 us, 4.5 TB/s; 256 rows of up to 1500 (32 / 8
// heads, 360 MB) 88-90 us, 4.1 TB/s; 64 rows of up to 8192 (12 / 2) 28 us; 128 rows of 16384 at head width 64 (14 / 2, 302
// MB) 71 us; one row of 700 tokens 8.4 us. In this schedule the instructions' latency decides, not memory: two computing
// warps on a scheduler keep 51-56 % of its issue slots busy (44 % on the ragged rows), with DRAM at half its rate; about
// 2000 cycles to a unit (products of K 520, P V and the wait for the copies 770, scores 260, the next copies 285). With
// few tokens it is the chain lengths, page id, copies, join (about 8 us).
#include <climits>

#include <cuda_runtime.h>

#include "../include/kv_split.cuh"
#include "kv4.h"

namespace meshy {

namespace {

using namespace kvsplit;

constexpr int kWarps = 8;                      // that compute
constexpr int kHelpers = 4;
constexpr int kThreads = 32 * (kWarps + kHelpers);
constexpr int kTok = 16;                       // tokens of a tile
constexpr int kSlots = 3;                      // segments whose fragments or states are held
// Equal segments up to 24 units are taken whole (one row of 700 tokens 9.0 us; more CTAs, with a join, 9.9; 16 rows of up
// to 1400 tokens 11.2 us where unequal ones get a step of every warp, with up to 24 units 14.9). The number of CTAs goes
// with the root of the work (the root itself took 11.5 and 15.3 us on one row of 8192 and 32768 tokens, twice as many 11.9
// and 15.8, four times 16.4 on the latter). A change of segments counts as 16 units (64 rows of up to 8192 tokens 29.0 us,
// with 8 29.9, with none 35.2; 200 rows of about 800 at head width 64 44.4, 45.5, 48.9; 33 rows of up to 4000 15.5, 16.2,
// 21.5); equal segments are cut alike if that costs fewer than 3 steps (4 rows of 16384 tokens 14.9 us instead of 17.8, 64
// of 4096 22.6 instead of 26.1).
constexpr Rules kRules{24, 16, 3};
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kBoost = 11.f;                 // log2 of the largest p a' right after the reference moved
constexpr float kLimit = 32768.f;              // how far later ones may go
constexpr float kMinA = 5.9604645e-8f;         // 2^-24, the smallest fp16

template <int HD, int NT, int NP>  // NT tiles to a unit, which lie in NP pieces (pages, or parts of one)
struct Cfg {
  static constexpr int ROW = HD / 2;                     // nibble bytes of a token
  static constexpr int PAIRS = HD / 8;                   // bytes of a token's pairs (K and V)
  static constexpr int UTOK = NT * kTok, PTOK = UTOK / NP;  // tokens of a unit, of a piece
  static constexpr int K = 0, V = UTOK * ROW, S = 2 * UTOK * ROW, STAGE = UTOK * (2 * ROW + PAIRS);
  static constexpr int STAGES = 13824 / STAGE;           // 3 units of 32 tokens at head width 128
  static constexpr int WARP = STAGES * STAGE;
  static constexpr int LD = HD + 4;                      // row stride of a state: spreads the heads over the banks
  static constexpr int STATES = kWarps * WARP;           // kSlots sets of the warps' states
  static constexpr int STATE = kHeads * LD * 4;
  // kSlots sets of query fragments: matrix B, sums (B too), factors
  static constexpr int F = STATES + kSlots * kWarps * STATE;
  static constexpr int F_SUM = 32 * 16 * (HD / 32), F_FACTOR = F_SUM + 2 * 32 * 4;
  static constexpr int FBYTES = F_FACTOR + kHeads * 4;
  static constexpr int SMEM = F + kSlots * FBYTES;
  static constexpr int PART = HD + 4;                    // floats of a head in the workspace: sums, maximum, normaliser
};

__device__ __forceinline__ void helper_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kHelpers) : "memory"); }

struct Args : Rows {
  const bf16* q;
  int64_t qs, qh;
  KV4View c;
  const int* bt;
  int64_t bt_stride;
  int Hq, rep, blocks;  // blocks: groups of kHeads query heads per KV head
  int ppp, page_pieces;    // pieces of a page, of a page of all heads
  float scale;
  bf16* out;
  float* part;         // [2 CTAs][kHeads][PART]
  unsigned* arrived;   // [segments], zero between launches
  int* err;
  long long wait;      // cycles after which a wait gives up
};

template <int HD, int NT, int NP>
__global__ void __launch_bounds__(kThreads, 1) kv4_attn_kernel(const Args a) {
  using C = Cfg<HD, NT, NP>;
  using W = Walk<C::UTOK, kWarps>;
  constexpr int G = HD / 64;
  constexpr int KW = HD / 32;  // K words a lane takes of a row
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
    // A segment's query rows as matrix fragments, a warp per head: scaled so that the largest is in [2^14, 2^15), a
    // word's channels 0 .. 7 as fp16 pairs (0, 4), (1, 5) / 16, (2, 6), (3, 7) / 16; the sums over the groups' channels
    // in units of 2^8 as three fp16 terms, against the bases; the factor that takes all that back, with the softmax
    // scale.
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
        float x1[CH];
#pragma unroll
        for (int i = 0; i < CH / 2; ++i) {
          const float2 y = unpack_bf16x2(raw[k][i]);
          x1[2 * i] = y.x;
          x1[2 * i + 1] = y.y;
        }
        float mx = 0.f, sum = 0.f;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          mx = fmaxf(mx, fabsf(x1[i]));
          sum += x1[i];
        }
        mx = warp_max(mx);
        const int ex = (mx > 0.f && mx < INFINITY) ? min(14 - ilogbf(mx), 126) : 0;
        const float up = ldexpf(1.f, ex);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int ch = lane * CH + i, word = (ch % 64) / 8 * G + ch / 64, e = ch % 8;
          reinterpret_cast<__half*>(f)[(((word % KW) * 32 + h * 4 + word / KW) * 4 + e % 4) * 2 + e / 4] =
              __float2half_rn(x1[i] * (e % 2 ? up * 0.0625f : up));
        }
#pragma unroll
        for (int o = 1; o < 64 / CH; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
        for (int i = 0; i < G; ++i) {
          const float y0 = __shfl_sync(0xffffffffu, sum, i * 16) * up * 0.00390625f;
          const __half t0 = __float2half_rn(y0);
          const float y1 = y0 - __half2float(t0);
          const __half t1 = __float2half_rn(y1), t2 = __float2half_rn(y1 - __half2float(t1));
          const __half t = lane == 0 ? t0 : lane == 1 ? t1 : lane == 2 ? t2 : __float2half_rn(0.f);
          if (lane < 4)
            reinterpret_cast<uint32_t*>(f + C::F_SUM)[i * 32 + h * 4 + lane] = (uint32_t)__half_as_ushort(t) << 16;
        }
        if (lane == 0) reinterpret_cast<float*>(f + C::F_FACTOR)[h] = ldexpf(sl2, 24 - ex);
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
      if (ht == 0) s_ok = mbar_wait(&done[slot], phase, abort_flag, a.err, kErrTimeoutEpilogue, a.wait);
      helper_sync();
      if (!s_ok) {  // (so it is if another wait gave up: every segment's states are waited for here)
        pieces = 0;
        if (ht == 0) arrive_all(a, Start<W>{w0, plan.shares, pad}, a.arrived);
        break;
      }
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
        if (ht == 0) s_piece[pieces] = piece_of(w, pad, plan.shares);
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
    // this lane's places in a stage
    const uint32_t k_at = C::K + tok_g * C::ROW + t * (4 * KW), s_at = C::S + tok_g * C::PAIRS;
    const uint32_t v_at = C::V + t * C::ROW + g * (4 * G);
    if (lane == 0) s_ahead[warp] = w0;
    __syncwarp();

    // The copies run STAGES - 1 units ahead of the arithmetic, across the segments; a unit's page ids are read one step
    // before its copies start, a piece's by every NP-th lane.
    constexpr int kDone = -(1 << 30);  // the share holds no more units for this warp
    const int sub = lane % NP;
    int f_end, f_at, f_wrap, f_page;  // f_at: piece within the page of all heads, f_wrap: where this head's part ends
    int f_piece, f_pieces;            // of the row: this lane's, all of them
    const int* f_bt;
    const int step_pi = NP * kWarps / a.ppp, step_off = NP * kWarps % a.ppp;
    const uint8_t* kp = a.c.k + lane * 16;
    const uint8_t* vp = a.c.v + lane * 16;
    const uint8_t* sp = reinterpret_cast<const uint8_t*>(a.c.scale) + lane * 16;
    int f_unit = w0.first_of(warp);
    auto aim = [&](const W& w) {
      f_end = w.end();
      f_piece = f_unit * NP + sub;
      f_pieces = (w.n + C::PTOK - 1) / C::PTOK;
      f_at = w.h / a.blocks * a.ppp;
      f_wrap = f_at + a.ppp;
      f_at += f_piece % a.ppp;
      f_bt = a.bt + w.b * a.bt_stride + f_piece / a.ppp;
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
      if (f_unit >= 0 && (NP == 1 || f_piece < f_pieces)) f_page = *f_bt;
    };
    uint32_t valid = 0;  // bits i NP ..: the pieces of the unit i steps ahead have a page
    auto fetch = [&](uint32_t stage, int steps) {
      const bool there = (uint32_t)f_page < (uint32_t)a.c.n_pages;
      const uint32_t n = there ? (uint32_t)f_page * (uint32_t)a.page_pieces + (uint32_t)f_at : 0u;  // piece of the cache
      const uint32_t dst = stage + lane * 16;
      static_assert(C::UTOK * C::PAIRS == 512, "a lane copies 16 bytes of pairs");
      if constexpr (NP == 1) {
        valid |= (there ? 1u : 0u) << steps;
        const uint8_t* ks = kp + (uint64_t)n * (C::UTOK * C::ROW);
        const uint8_t* vs = vp + (uint64_t)n * (C::UTOK * C::ROW);
        const uint8_t* ss = sp + (uint64_t)n * (C::UTOK * C::PAIRS);
#pragma unroll
        for (int i = 0; i < C::UTOK * C::ROW / 512; ++i) {
          copy16(dst + C::K + 512 * i, ks + 512 * i, there);
          copy16(dst + C::V + 512 * i, vs + 512 * i, there);
        }
        copy16(dst + C::S, ss, there);
      } else {
        const uint32_t bits = __ballot_sync(0xffffffffu, there) & ((1u << NP) - 1u);
        valid |= bits << (NP * steps);
#pragma unroll
        for (int i = 0; i < C::UTOK * C::ROW / 512; ++i) {
          constexpr int N = C::PTOK * C::ROW;
          const int piece = 512 * i / N;
          const uint64_t at = (uint64_t)__shfl_sync(0xffffffffu, n, piece) * N + 512 * i % N;
          copy16(dst + C::K + 512 * i, kp + at, bits >> piece & 1u);
          copy16(dst + C::V + 512 * i, vp + at, bits >> piece & 1u);
        }
        constexpr int N = C::PTOK * C::PAIRS;
        const int piece = lane * 16 / N;
        const uint64_t at = (uint64_t)__shfl_sync(0xffffffffu, n, piece) * N - piece * N;  // sp has lane * 16 already
        copy16(dst + C::S, sp + at, bits >> piece & 1u);
      }
      copies_commit();
      f_unit += kWarps;
      f_piece += NP * kWarps;
      f_bt += step_pi;
      f_at += step_off;
      if (f_at >= f_wrap) {
        f_at -= a.ppp;
        ++f_bt;
      }
      settle();
    };
    aim(w0);
    settle();
    for (int i = 0; i < C::STAGES - 1; ++i) fetch(ring + i * C::STAGE, i);
    uint32_t stage = ring, ahead = ring + (C::STAGES - 1) * C::STAGE;
    int slot = 0;
    uint32_t phase = 0;

    while (true) {
      if (!__all_sync(0xffffffffu, mbar_wait(&ready[slot], phase, abort_flag, a.err, kErrTimeoutMma, a.wait))) break;
      const W* seg = &s_seg[slot];
      const int n_tok = seg->n, u_end = seg->end();
      int unit = seg->first_of(warp);
      const bool more = seg->more();
      const uint8_t* frags = smem + C::F + slot * C::FBYTES;
      uint32_t zf[2] = {0u, 0u};
      float cs[2];
#pragma unroll
      for (int i = 0; i < G; ++i) zf[i] = reinterpret_cast<const uint32_t*>(frags + C::F_SUM)[i * 32 + lane];
#pragma unroll
      for (int r = 0; r < 2; ++r) cs[r] = reinterpret_cast<const float*>(frags + C::F_FACTOR)[2 * t + r];
      const uint32_t frag_at = smem_u32(frags) + lane * 16;
      // o, z and l are relative to the reference m: p 2^-m, so that x fits fp16 well
      float o[G][4][4], z[G][2], m[2] = {0.f, 0.f}, l[2] = {0.f, 0.f};
      float limit = -1.f;  // below 0: no reference yet
#pragma unroll
      for (int i = 0; i < G; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
        z[i][0] = z[i][1] = 0.f;
      }
      for (; unit < u_end; unit += kWarps) {
        copies_wait<C::STAGES - 2>();
        __syncwarp();  // and every lane has read the stage that is filled again below
        const uint32_t here = stage;
        // tokens of the unit to be counted; the rest may be anything
        const int count = n_tok - unit * C::UTOK;
        const uint32_t pieces = valid & ((1u << NP) - 1u);
        valid >>= NP;
        // the next copies first: after the products of K, 8 rows of 131072 tokens took 66.2 us instead of 64.8
        fetch(ahead, C::STAGES - 2);
        ahead = stage;
        stage = stage + C::STAGE == ring + C::WARP ? ring : stage + C::STAGE;
        // everything the unit needs from shared memory is asked for at once
        uint32_t kw[NT][2][KW], qf[KW][4], sw[NT][2][2 * G], vw[NT][4][G];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) load_words<KW>(kw[n][i], here + k_at + (2 * n + i) * 8 * C::ROW);
#pragma unroll
        for (int j = 0; j < KW; ++j) load_words<4>(qf[j], frag_at + j * 512);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) load_words<2 * G>(sw[n][i], here + s_at + (2 * n + i) * 8 * C::PAIRS);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) load_words<G>(vw[n][i], here + v_at + (4 * n + i) * 4 * C::ROW);
        // scores: tile n, row g + 8 i, head 2 t + r
        float s[NT][2][2], va[NT][2][G], vz[NT][2][G];
        {
          float acc[NT][G][4], e[NT][4];
#pragma unroll
          for (int j = 0; j < KW; ++j)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              uint32_t w0 = kw[n][0][j], w1 = kw[n][1][j];
              if (j < G)
                mma_f16_first(acc[n][j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u,
                              qf[j][0], qf[j][1]);
              else
                mma_f16(acc[n][j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[j][0],
                        qf[j][1]);
              w0 >>= 8;
              w1 >>= 8;
              mma_f16(acc[n][j % G], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qf[j][2],
                      qf[j][3]);
            }
#pragma unroll
          for (int n = 0; n < NT; ++n)  // sum_g z_g sum(q_g): the pairs (a, z) against (0, sum)
            mma_f16_first(e[n], sw[n][0][0], sw[n][1][0], G == 2 ? sw[n][0][G - 1] : 0u, G == 2 ? sw[n][1][G - 1] : 0u,
                          zf[0], zf[1]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float d[2] = {0.f, 0.f};
#pragma unroll
              for (int j = 0; j < G; ++j) {
                const float ka = __low2float(*reinterpret_cast<const __half2*>(&sw[n][i][j]));
                const float2 v2 = unpack_half2(sw[n][i][G + j]);
                va[n][i][j] = v2.x;
                vz[n][i][j] = v2.y;
                d[0] = fmaf(ka, acc[n][j][2 * i], d[0]);
                d[1] = fmaf(ka, acc[n][j][2 * i + 1], d[1]);
              }
#pragma unroll
              for (int r = 0; r < 2; ++r)  // the sums are in units of 2^8, the products in 2^24
                s[n][i][r] = fmaf(cs[r], fmaf(e[n][2 * i + r], 1.52587890625e-5f, d[r]), -m[r]);
            }
          }
        }
        if (count < C::UTOK || pieces != (1u << NP) - 1u) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (n * kTok + tok_g + 8 * i >= count || !(pieces >> (n * kTok / C::PTOK) & 1u)) {
                s[n][i][0] = s[n][i][1] = -INFINITY;
#pragma unroll
                for (int j = 0; j < G; ++j) va[n][i][j] = vz[n][i][j] = 0.f;
              }
        }
        float p[NT][2][2], top_x = 0.f;
        auto largest_a = [&](int n, int i) { return fmaxf(kMinA, G == 2 ? fmaxf(va[n][i][0], va[n][i][G - 1]) : va[n][i][0]); };
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float a1 = largest_a(n, i);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              p[n][i][r] = ex2(s[n][i][r]);
              top_x = fmaxf(top_x, p[n][i][r] * a1);
            }
          }
        if (__any_sync(0xffffffffu, top_x > limit)) {
          // move the reference: to the largest p a', less what brings that to 2^kBoost
          bool found = false;
          float keep[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 2; ++i) top = fmaxf(top, s[n][i][r] + lg2(largest_a(n, i)));
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
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            l[r] += p[n][0][r] + p[n][1][r];
#pragma unroll
            for (int j = 0; j < G; ++j)
              z[j][r] = fmaf(p[n][0][r], vz[n][0][j], fmaf(p[n][1][r], vz[n][1][j], z[j][r]));
          }
#pragma unroll
          for (int j = 0; j < G; ++j) {
            const uint32_t b0 = transpose8x8(pack_half2(p[n][0][0] * va[n][0][j], p[n][0][1] * va[n][0][j]));
            const uint32_t b1 = transpose8x8(pack_half2(p[n][1][0] * va[n][1][j], p[n][1][1] * va[n][1][j]));
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // channels 8 g + 4 half ..
              const uint32_t sel = half ? 0x7632u : 0x5410u;
              uint32_t x01 = __byte_perm(vw[n][0][j], vw[n][1][j], sel);
              uint32_t x23 = __byte_perm(vw[n][2][j], vw[n][3][j], sel);
              mma_f16(o[j][2 * half], x01 & 0x000F000Fu, x01 & 0x00F000F0u, x23 & 0x000F000Fu, x23 & 0x00F000F0u, b0,
                      b1);
              x01 >>= 8;
              x23 >>= 8;
              mma_f16(o[j][2 * half + 1], x01 & 0x000F000Fu, x01 & 0x00F000F0u, x23 & 0x000F000Fu, x23 & 0x00F000F0u,
                      b0, b1);
            }
          }
        }
      }

      // the warp's state: o in units of V, relative to m
      float* state = reinterpret_cast<float*>(smem + C::STATES + (slot * kWarps + warp) * C::STATE);
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

  __syncthreads();  // (arrivals wait until the share is done, so that nothing else waits for their round trip)
  const int pieces = s_pieces;
  if (pieces) join_pieces<HD, kThreads>(a, s_piece, pieces, a.part, a.arrived, a.blocks, a.rep, a.Hq, a.out);
}

template <int HD, int NT, int NP>
void launch(Args a, cudaStream_t st) {
  using C = Cfg<HD, NT, NP>;
  a.ppp = a.c.page / C::PTOK;
  a.page_pieces = a.c.Hkv * a.ppp;
  // pieces are counted in 32 bits, in the cache and over the rows
  MESHY_CHECK(a.c.n_pages * a.page_pieces < (1LL << 32) - 1, "paged_attention_kv4: cache too large");
  MESHY_CHECK((int64_t)a.B * a.c.Hkv * a.blocks * (std::max<int64_t>(1, (int64_t)a.max_pages * a.ppp) + kRules.pad) < (1LL << 31),
              "paged_attention_kv4: rows * heads * table width too large");
  launch_split<kv4_attn_kernel<HD, NT, NP>>(kThreads, C::SMEM, a, st);
}

}  // namespace

int kv4_attention_ctas() { return sm_count(); }
int64_t kv4_attention_segments(int B, int Hq, int Hkv) { return (int64_t)B * Hkv * ((Hq / Hkv + kHeads - 1) / kHeads); }

void kv4_attention(const bf16* q, int64_t qs, int64_t qh, KV4View c, const int* bt, int64_t bt_stride, int max_pages,
                   const int* seq_lens, int B, int Hq, float scale, bf16* out, float* part, unsigned* arrived, int* err,
                   int64_t wait, cudaStream_t st) {
  if (B == 0) return;
  const int rep = Hq / c.Hkv;
  max_pages = std::min(max_pages, (INT_MAX - 63) / c.page);  // lengths are rounded up to units in 32 bits
  Args a;
  const int blocks = (rep + kHeads - 1) / kHeads;
  static_cast<Rows&>(a) = {seq_lens, B, max_pages, c.page, c.Hkv * blocks};
  a.q = q, a.qs = qs, a.qh = qh, a.c = c, a.bt = bt, a.bt_stride = bt_stride, a.Hq = Hq, a.rep = rep, a.blocks = blocks;
  a.scale = scale, a.out = out, a.part = part, a.arrived = arrived, a.err = err;
  a.wait = wait < 0 ? kWaitCycles : wait;
  if (c.hd == 128)
    c.page % 32 == 0 ? launch<128, 2, 1>(a, st) : launch<128, 2, 2>(a, st);
  else
    c.page % 64 == 0 ? launch<64, 4, 1>(a, st) : c.page % 32 == 0 ? launch<64, 4, 2>(a, st) : launch<64, 4, 4>(a, st);
}

}  // namespace meshy
