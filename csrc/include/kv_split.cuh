// What the decode attention kernels over quantised paged caches share: instructions, and the split of the work.
//
// The (row, KV head, up to 8 query heads) segments are laid end to end in units of UTOK tokens, and every CTA takes an
// equal share of the sum, whatever the lengths, a change of segments counted as some units: they are read on the device,
// so a captured graph follows them. Within a CTA, unit i belongs to warp i mod WARPS. A segment that spans CTAs leaves
// partial sums in a workspace; the last CTA to arrive joins them in CTA order. So every sum has one order, and results do
// not depend on timing.
#pragma once
#include <atomic>

#include <cuda_fp16.h>

#include "common.cuh"
#include "quotient.cuh"
#include "sm100.cuh"

namespace meshy {
namespace kvsplit {

constexpr int kHeads = 8;  // query heads of a segment

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {  // zeros where it is not
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(there ? 8 : 0) : "memory");
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

struct Rows {
  const int* seq_lens;
  int B, max_pages, page;
  int per_row;  // segments of a row
};

__device__ __forceinline__ int tokens_of(const Rows& a, int b) {
  const int64_t cap = (int64_t)a.max_pages * a.page;
  const int n = a.seq_lens[b];
  return n <= 0 ? 0 : (int)min((int64_t)n, cap);
}
template <int UTOK>
__device__ __forceinline__ uint32_t units_of(int n) {  // an empty row has one too, which writes its zeros
  return max(1, (n + UTOK - 1) / UTOK);
}

// A CTA's walk over its share of the units: segment (b, h), which starts at unit ``begin`` of the sum and of whose U
// units (the last ``pad`` of them empty) the share has [first, last); ``left`` units of the share remain from ``first``
// on.
template <int UTOK, int WARPS>
struct Walk {
  int b, h, n, U, first, last, left;
  uint32_t begin;
  __device__ __forceinline__ bool next(const Rows& a, int pad) {
    left -= last - first;
    if (left <= 0) return false;
    first = 0;
    begin += U;
    if (++h == a.per_row) {
      h = 0;
      ++b;
      n = tokens_of(a, b);
      U = units_of<UTOK>(n) + pad;
    }
    last = min(U, left);
    return true;
  }
  __device__ __forceinline__ bool more() const { return left > last - first; }
  __device__ __forceinline__ int end() const { return min(last, (n + UTOK - 1) / UTOK); }  // of the units with tokens
  __device__ __forceinline__ bool whole() const { return first == 0 && last >= (int)units_of<UTOK>(n); }
  __device__ __forceinline__ int first_of(int warp) const { return first + ((warp - (int)begin - first) & (WARPS - 1)); }
};

__device__ __forceinline__ float sqrt_approx(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// x / d in whole numbers, for quotients below 2^20, r ~ 1 / d
__device__ __forceinline__ uint32_t whole_quotient(uint32_t x, uint32_t d, float r) {
  uint32_t q = (uint32_t)((float)x * r);
  const int rest = (int)(x - q * d);
  if (rest < 0) --q;
  if (rest >= (int)d) ++q;
  return q;
}

// CTA c of n has units [begin(c), begin(c + 1)): total / n each, and the rest spread evenly (so that equal segments are
// cut alike).
struct Shares {
  uint32_t total, n, per, more;
  float r;  // ~ 1 / n
  __device__ __forceinline__ uint32_t begin(uint32_t c) const { return c * per + whole_quotient(c * more, n, r); }
  __device__ __forceinline__ uint32_t owner(uint32_t unit) const {
    uint32_t c = min(n - 1, (uint32_t)((float)unit * rcp_approx((float)total) * (float)n));
    while (c + 1 < n && begin(c + 1) <= unit) ++c;
    while (begin(c) > unit) --c;
    return c;
  }
};

// A segment (b, h) that the CTA has a piece of, and the n CTAs from ``first`` on that share it.
struct Piece {
  int b, h;
  uint32_t first, n;
  bool last;  // this CTA arrived last
};
template <class W>
__device__ __forceinline__ Piece piece_of(const W& w, int pad, const Shares& shares) {
  const uint32_t c0 = shares.owner(w.begin);
  return {w.b, w.h, c0, shares.owner(w.begin + w.U - pad - 1) - c0 + 1, false};
}

// The split's constants, which each kernel measured for itself.
struct Rules {
  uint32_t whole_units;  // units of equal segments that a CTA takes whole
  int pad;               // units that a change of segments costs
  int join_steps;        // steps of a warp that a join is worth
};

// Shared memory of the plan; every thread of the CTA (THREADS) takes part.
template <int THREADS>
struct PlanShared {
  uint32_t scan[THREADS / 32], begin, row0;
  int row, n;
};

template <class W>
struct Plan {
  bool work;  // this CTA has any
  W w;        // where its share starts
  Shares shares;
  int pad;
};

template <int UTOK, int WARPS, int THREADS>
__device__ __forceinline__ Plan<Walk<UTOK, WARPS>> make_plan(const Rows& a, PlanShared<THREADS>& s, const Rules rules) {
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  Plan<Walk<UTOK, WARPS>> p;
  p.work = false;
  // all units (row by row), this CTA's share of them and the row it starts in
  uint32_t total = 0, mine = 0, before = 0;
  int tokens = 0;
  auto sum_rows = [&](int b0) {  // the units of rows b0 + tid, of the rows before it, and of all up to this block of rows
    tokens = b0 + tid < a.B ? tokens_of(a, b0 + tid) : 0;
    mine = b0 + tid < a.B ? units_of<UTOK>(tokens) * (uint32_t)a.per_row : 0;
    uint32_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    __syncthreads();
    if (lane == 31) s.scan[warp] = incl;
    if (b0 == 0 && tid == 0) s.row0 = mine;
    __syncthreads();
    before = total + incl - mine;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += s.scan[w];
      total += s.scan[w];
    }
  };
  for (int b0 = 0; b0 < a.B; b0 += THREADS) sum_rows(b0);
  // A CTA per segment where that makes a few steps of every warp: for equal segments up to ``whole_units``, one step for
  // others, whose shares are cut and joined anyway. Else more of them: the steps shrink with their number, the join grows
  // with it, so the best number goes with the root of the work. Equal segments get a whole number of CTAs each, and are
  // then cut alike, if that costs fewer steps than a join.
  const uint32_t segments = a.B * a.per_row;
  const bool equal = total == s.row0 * a.B;  // or as good as that: the cut is right either way
  uint32_t n_cta = segments;
  if (total > segments * (equal ? rules.whole_units : WARPS))
    n_cta = max(segments, min((total + WARPS - 1) / WARPS, (uint32_t)sqrt_approx((float)total * (float)segments)));
  n_cta = min(gridDim.x, n_cta);
  if (equal && n_cta > segments) {
    const uint32_t even = whole_quotient(n_cta, segments, rcp_approx((float)segments)) * segments;
    if ((float)total * (rcp_approx((float)even) - rcp_approx((float)n_cta)) <= (float)(rules.join_steps * WARPS)) n_cta = even;
  }
  if (blockIdx.x >= n_cta) return p;
  // Where CTAs have several segments, the change from one to the next counts as ``pad`` empty units at a segment's end: a
  // CTA with more segments gets fewer tokens. Where several CTAs share each of equal segments there is no change.
  p.pad = equal && n_cta >= 2 * segments ? 0 : rules.pad;
  const uint32_t all = total + p.pad * segments;
  const uint32_t per = all / n_cta;
  p.shares = Shares{all, n_cta, per, all - per * n_cta, rcp_approx((float)n_cta)};
  const uint32_t at = p.shares.begin(blockIdx.x), end = p.shares.begin(blockIdx.x + 1);
  if (a.B > THREADS) total = 0;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    if (a.B > THREADS) sum_rows(b0);
    const uint32_t row = before + p.pad * a.per_row * (b0 + tid);
    if (b0 + tid < a.B && at - row < mine + p.pad * a.per_row) {
      s.row = b0 + tid;
      s.n = tokens;
      s.begin = row;
    }
    if (total + p.pad * a.per_row * min(b0 + THREADS, a.B) > at) break;
  }
  __syncthreads();
  p.w.b = s.row;
  p.w.n = s.n;
  p.w.U = units_of<UTOK>(p.w.n) + p.pad;
  p.w.h = whole_quotient(at - s.begin, p.w.U, rcp_approx((float)p.w.U));
  p.w.begin = s.begin + p.w.h * p.w.U;
  p.w.first = at - p.w.begin;
  p.w.left = end - at;
  p.w.last = min(p.w.U, p.w.first + p.w.left);
  p.work = !(p.w.first >= p.w.U - p.pad && !p.w.next(a, p.pad));  // something of that segment is left, or another
  return p;
}

// Counts this CTA's piece; true for the last of the segment, which leaves the counter at zero.
__device__ __forceinline__ bool arrive(const Rows& a, const Piece& x, unsigned* arrived) {
  unsigned* ctr = arrived + (int64_t)x.b * a.per_row + x.h;
  unsigned old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(ctr) : "memory");
  const bool last = old == x.n - 1;
  if (last) *ctr = 0u;
  return last;
}

// Where a CTA's share began, kept for one that gives up.
template <class W>
struct Start {
  W w;
  Shares shares;
  int pad;
};
// A CTA in which a wait gave up joins nothing, but one thread counts its pieces all the same: the counters are zero when the
// launch ends, whatever became of it, and the next one's results are right.
template <class W>
__device__ __forceinline__ void arrive_all(const Rows& a, const Start<W>& s, unsigned* arrived) {
  W w = s.w;
  do {
    if (!w.whole()) arrive(a, piece_of(w, s.pad, s.shares), arrived);
  } while (w.next(a, s.pad));
}

// The last CTA to arrive at a segment joins its pieces. ``part``: [2 CTAs][kHeads][HD + 4] floats (sums, maximum,
// normaliser), of which CTA c's segment that began before its share is at 2 c, another at 2 c + 1; ``arrived``: zero
// between launches. Every thread takes part, the CTA's own pieces having been written before a barrier.
template <int HD, int THREADS>
__device__ __forceinline__ void join_pieces(const Rows& a, Piece* piece, int pieces, const float* part, unsigned* arrived,
                                            int blocks, int rep, int Hq, bf16* out) {
  constexpr int PART = HD + 4;
  const int tid = threadIdx.x;
  if (tid < pieces) {
    Piece& x = piece[tid];
    x.last = arrive(a, x, arrived);
  }
  __syncthreads();
  for (int i = tid; i < pieces * kHeads * (HD / 4); i += THREADS) {
    const Piece& x = piece[i / (kHeads * (HD / 4))];
    const int h = i / (HD / 4) % kHeads, ch = 4 * (i % (HD / 4)), hk = x.h / blocks, h0 = (x.h % blocks) * kHeads;
    if (!x.last || h0 + h >= rep) continue;
    const float* p0 = part + ((int64_t)x.first * 2 * kHeads + h) * PART;
    const int np = x.n;
    float M = -INFINITY, L = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kBatch = 16;
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
          const float* pp = p0 + (2 * c + (c == 0 ? 1 : 0)) * kHeads * PART;
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
    *reinterpret_cast<uint2*>(out + ((int64_t)x.b * Hq + hk * rep + h0 + h) * HD + ch) =
        make_uint2(pack_bf16x2(y.x * e, y.y * e), pack_bf16x2(y.z * e, y.w * e));
  }
}

// ─── host ──────────────────────────────────────────────────────────────────

constexpr int kDevices = 64;

inline int sm_count() {
  static std::atomic<int> counts[kDevices];
  int dev = 0, n = 0;
  MESHY_CUDA_CHECK(cudaGetDevice(&dev));
  if ((n = counts[dev].load(std::memory_order_relaxed)) == 0) {
    MESHY_CUDA_CHECK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    counts[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// One CTA to every SM.
template <auto Kernel, class Args>
void launch_split(int threads, int smem, const Args& a, cudaStream_t st) {
  static std::atomic<bool> set[kDevices];
  int dev = 0;
  MESHY_CUDA_CHECK(cudaGetDevice(&dev));
  if (!set[dev].load(std::memory_order_relaxed)) {
    MESHY_CUDA_CHECK(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    set[dev].store(true, std::memory_order_relaxed);
  }
  launch_pdl(Kernel, dim3(sm_count()), dim3(threads), smem, st, a);
}

}  // namespace kvsplit
}  // namespace meshy
