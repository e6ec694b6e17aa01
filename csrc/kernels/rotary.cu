// Rotary positions of a fused QKV projection, and the gradient.
//
//   x^ = x rstd w (with QK-norm),   y_a = m (x^_a cos - x^_b sin),   y_b = m (x^_b cos + x^_a sin)
//   g^ = m R^T g,   dw = sum g^ x rstd,   dx = rstd (g^ w - x rstd mean(g^ w x rstd))
//
// The angle of pair i at position p is p f_i. Far positions would lose it in fp32 (p f has 17 bits before the point at
// 131072), so f_i comes as 2^64 times its turns per position: p times that, in 64 bits, wraps around at whole turns by
// itself, and its upper half is the fraction of a turn to 2^-32, whatever the position.
//
// Everything between reading and writing is in fp32; outputs are rounded once. A group of hd / 8 lanes has a token and
// some of its heads; a lane has four pairs, in the half layout two runs of four channels, or eight channels behind the
// rotated part. Its four angles are worked out once for all its heads; the norm's weights are taken into the sines and
// cosines. Each channel is read and written once, and the memory's rate bounds the calls without norms; it leaves a warp
// only 176 instructions to two heads, so arithmetic is done on pairs of fp32 numbers in one instruction.
//
// Measured: 16384 tokens of 32 + 8 + 8 heads, 128 wide, 66 us forward and 66 back, 6.1 TB/s (loads and stores head by head
// took 148 and 140); with norms and interleaved 88 and 121, where the sums over a head, the chain from them to the stores
// and, back, half the warps (128 registers) count as much as memory: 48 to 57 % of the issue slots are busy. 5003 tokens
// of 16 + 8 + 8 heads with norms 19 and 35 us. 64 tokens of a decode step 2.3 us, a launch.
#include <cuda_runtime.h>

#include "../include/fastdiv.cuh"
#include "rotary.h"

namespace meshy {

namespace {

constexpr int kThreads = 256;
constexpr int C = 8;  // channels of a lane

struct Args {
  RotaryShape s;
  const bf16* qkv;
  int64_t qs;
  const int* pos;
  const uint64_t* turns;
  float factor;
  const bf16* qn;
  const bf16* kn;
  float eps;
  bf16* q;
  bf16* k;
  bf16* v;
  RotaryCache cache;
  const bf16* gq;
  const bf16* gk;
  const bf16* gv;
  bf16* gqkv;
  float* part;
  int nh, splits;             // heads of a group, groups of a token
  FastDiv tokens;             // T
  FastDiv q_items, k_items;   // items of a token in the gradient with norms
  FastDiv v_row;              // 8 bytes each: V's channels of a token
  float inv_hd;
};

// Where a lane's C channels are: two runs of half as many (they follow one another unless the layout is by halves).
struct Place {
  int a, b;
  bool turned;
};
__device__ __forceinline__ Place place_of(const RotaryShape& s, int lane) {
  if (C * lane >= s.rot || s.interleaved) return {C * lane, C * lane + C / 2, C * lane < s.rot};
  return {C / 2 * lane, s.rot / 2 + C / 2 * lane, true};
}

// Two fp32 numbers, and their sums and products in one instruction.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 parts(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// A lane's channels on their way, two to a word: two runs.
struct Raw {
  uint32_t u[C / 2];
};
__device__ __forceinline__ Raw no_raw() {
  Raw r;
#pragma unroll
  for (int i = 0; i < C / 2; ++i) r.u[i] = 0u;
  return r;
}
__device__ __forceinline__ Raw load_raw(const bf16* p, const Place& w) {
  Raw r;
  const uint2 a = __ldg(reinterpret_cast<const uint2*>(p + w.a)), b = __ldg(reinterpret_cast<const uint2*>(p + w.b));
  r.u[0] = a.x, r.u[1] = a.y, r.u[2] = b.x, r.u[3] = b.y;
  return r;
}
__device__ __forceinline__ void store_raw(bf16* p, const Place& w, const Raw& r) {
  *reinterpret_cast<uint2*>(p + w.a) = make_uint2(r.u[0], r.u[1]);
  *reinterpret_cast<uint2*>(p + w.b) = make_uint2(r.u[2], r.u[3]);
}

// The same as C / 2 pairs (a_i, b_i): pair i is channels (i, C / 2 + i) by halves, (2 i, 2 i + 1) interleaved.
struct Pairs {
  static constexpr int N = C / 4;
  F2 a[N], b[N];
};
template <bool INTER>
__device__ __forceinline__ Pairs unpack(const Raw& r) {
  Pairs x;
#pragma unroll
  for (int i = 0; i < C / 4; ++i) {
    const float2 p = unpack_bf16x2(r.u[INTER ? 2 * i : i]), q = unpack_bf16x2(r.u[INTER ? 2 * i + 1 : C / 4 + i]);
    x.a[i] = INTER ? f2(p.x, q.x) : f2(p.x, p.y);
    x.b[i] = INTER ? f2(p.y, q.y) : f2(q.x, q.y);
  }
  return x;
}
template <bool INTER>
__device__ __forceinline__ Raw pack(const Pairs& x) {
  Raw r;
#pragma unroll
  for (int i = 0; i < C / 4; ++i) {
    const float2 a = parts(x.a[i]), b = parts(x.b[i]);
    r.u[INTER ? 2 * i : i] = INTER ? pack_bf16x2(a.x, b.x) : pack_bf16x2(a.x, a.y);
    r.u[INTER ? 2 * i + 1 : C / 4 + i] = INTER ? pack_bf16x2(a.y, b.y) : pack_bf16x2(b.x, b.y);
  }
  return r;
}

// y_a = a ac + b bs, y_b = b bc + a as
struct Turn {
  F2 ac[C / 4], bs[C / 4], bc[C / 4], as[C / 4];
  __device__ __forceinline__ Pairs operator()(const Pairs& x) const {
    Pairs y;
#pragma unroll
    for (int i = 0; i < C / 4; ++i) {
      y.a[i] = fma2(x.b[i], bs[i], x.a[i] * ac[i]);
      y.b[i] = fma2(x.a[i], as[i], x.b[i] * bc[i]);
    }
    return y;
  }
};

// Sine and cosine of a fraction of a turn, given in units of 2^-32: taken to the nearest quarter, the rest by their Taylor
// series, which end 2^-25 (sine 2^-29) from the value at an eighth of a turn.
__device__ __forceinline__ void sine_cosine(uint32_t turn, float& sine, float& cosine) {
  const uint32_t near = turn + 0x20000000u, quarter = near >> 30;
  const float x = (float)((int)(near & 0x3FFFFFFFu) - 0x20000000) * 1.46291807926715968e-9f;  // 2 pi 2^-32
  const float u = x * x;
  float s = fmaf(u, 2.75573192e-6f, -1.98412698e-4f);
  s = fmaf(u, s, 8.33333333e-3f);
  s = fmaf(u, s, -0.166666667f);
  s = fmaf(u * x, s, x);
  float c = fmaf(u, 2.48015873e-5f, -1.38888889e-3f);
  c = fmaf(u, c, 4.16666667e-2f);
  c = fmaf(u, c, -0.5f);
  c = fmaf(u, c, 1.f);
  const bool swap = quarter & 1u;
  sine = __uint_as_float(__float_as_uint(swap ? c : s) ^ (quarter & 2u) << 30);
  cosine = __uint_as_float(__float_as_uint(swap ? s : c) ^ (quarter + 1u & 2u) << 30);
}

// cos and sin of a lane's pairs at position p, times the factor (1 and 0 behind the rotated part).
struct Angles {
  float c[C / 2], s[C / 2];
};
__device__ __forceinline__ Angles angles(const Args& a, const Place& w, int lane, int64_t p) {
  Angles g;
#pragma unroll
  for (int i = 0; i < C / 2; ++i) {
    g.c[i] = 1.f, g.s[i] = 0.f;
    if (!w.turned) continue;
    sine_cosine((uint32_t)(a.turns[C / 2 * lane + i] * (uint64_t)p >> 32), g.s[i], g.c[i]);
    g.c[i] *= a.factor;
    g.s[i] *= a.factor;
  }
  return g;
}
__device__ __forceinline__ Turn turn_of(const Angles& g, bool back) {
  Turn r;
#pragma unroll
  for (int i = 0; i < C / 4; ++i) {
    r.ac[i] = r.bc[i] = f2(g.c[2 * i], g.c[2 * i + 1]);
    const F2 s = f2(g.s[2 * i], g.s[2 * i + 1]), n = f2(-g.s[2 * i], -g.s[2 * i + 1]);
    r.as[i] = back ? n : s;
    r.bs[i] = back ? s : n;
  }
  return r;
}
// after a multiplication by w
__device__ __forceinline__ Turn turn_of(const Angles& g, const Pairs& w) {
  Turn r = turn_of(g, false);
#pragma unroll
  for (int i = 0; i < C / 4; ++i) {
    r.ac[i] = r.ac[i] * w.a[i];
    r.as[i] = r.as[i] * w.a[i];
    r.bc[i] = r.bc[i] * w.b[i];
    r.bs[i] = r.bs[i] * w.b[i];
  }
  return r;
}
__device__ __forceinline__ float sum_products(const Pairs& x, const Pairs& y) {
  F2 s = x.a[0] * y.a[0];
  s = fma2(x.b[0], y.b[0], s);
#pragma unroll
  for (int i = 1; i < C / 4; ++i) {
    s = fma2(x.a[i], y.a[i], s);
    s = fma2(x.b[i], y.b[i], s);
  }
  const float2 p = parts(s);
  return p.x + p.y;
}
__device__ __forceinline__ Pairs times(const Pairs& x, const Pairs& y) {
  Pairs z;
#pragma unroll
  for (int i = 0; i < C / 4; ++i) {
    z.a[i] = x.a[i] * y.a[i];
    z.b[i] = x.b[i] * y.b[i];
  }
  return z;
}
__device__ __forceinline__ Pairs times(const Pairs& x, float f) {
  Pairs z;
#pragma unroll
  for (int i = 0; i < C / 4; ++i) {
    z.a[i] = x.a[i] * f2(f, f);
    z.b[i] = x.b[i] * f2(f, f);
  }
  return z;
}

// The channel of member a (or b) of a lane's pair i.
template <bool INTER>
__device__ __forceinline__ int channel_of(const Place& w, int i, bool b) {
  const int e = INTER ? 2 * i + b : C / 2 * b + i;
  return e < C / 2 ? w.a + e : w.b + e - C / 2;
}

// Lanes of a group, for the sums over a head.
template <int L>
__device__ __forceinline__ uint32_t group_mask() {
  return L == 32 ? 0xffffffffu : ((1u << L) - 1u) << (threadIdx.x % 32 / L * L);
}

// A group's token and heads: neighbouring groups have the same heads of neighbouring tokens, so that a warp does not part.
struct Item {
  bool there;
  int t, h0, h1;
};
template <int L>
__device__ __forceinline__ Item item_of(const Args& a) {
  const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
  if (i >= (int64_t)a.s.T * a.splits) return {false, 0, 0, 0};
  const int k = (int)a.tokens.div((uint32_t)i), h0 = k * a.nh;
  return {true, (int)(i - (int64_t)k * a.s.T), h0, min(a.s.Hq + 2 * a.s.Hkv, h0 + a.nh)};
}

// Heads whose loads are under way together (2 heads: 74 us on the 16384 tokens, 8 heads spill), and heads at hand with
// norms, as many more under way (1 head: 106 us forward and 150 back on the 16384 with norms, for 88 and 121; 4 heads and
// fewer warps: 85 and 133, on the 5003 tokens 21 and 37 for 19 and 35).
constexpr int kBatch = 4;
constexpr int kNormBatch = 2;

// f(x, raw) for each of the n rows of hd channels from ``src`` on.
template <int N, class F>
__device__ __forceinline__ void each_row(const bf16* src, int hd, int n, const Place& w, F f) {
  for (int j = 0; j < n; j += N) {
    Raw raw[N];
#pragma unroll
    for (int x = 0; x < N; ++x)
      if (j + x < n) raw[x] = load_raw(src + (int64_t)(j + x) * hd, w);
#pragma unroll
    for (int x = 0; x < N; ++x)
      if (j + x < n) f(j + x, raw[x]);
  }
}

// (CTAs of an SM, us on the 16384 tokens: without norms 4 66, 3 68; with norms 3 88, 2 96, 4 100.)
template <int L, bool NORM, bool INTER>
__global__ void __launch_bounds__(kThreads, NORM ? 3 : 4) rotary_fwd_kernel(const Args a) {
  const RotaryShape& s = a.s;
  const int lane = threadIdx.x % L;
  pdl_wait();
  pdl_trigger();
  const Item it = item_of<L>(a);
  const bool on = C * lane < s.hd;
  if (!it.there || (!NORM && !on)) return;
  const int t = it.t, HQK = s.Hq + s.Hkv;
  const Place w = on ? place_of(s, lane) : Place{0, 0, false};
  const bf16* src = a.qkv + t * a.qs;
  Angles g;
  if (it.h0 < HQK) g = angles(a, w, lane, a.pos[t]);
  const Turn plain = turn_of(g, false);
  int64_t row = -1;  // of the cache, head 0
  if (a.cache.k && it.h1 > s.Hq) {
    const int64_t slot = a.cache.slots[t], n = a.cache.n_pages * a.cache.page;
    if (slot >= 0 && slot < n) {
      const int64_t p = slot / a.cache.page;
      row = p * s.Hkv * a.cache.page + (slot - p * a.cache.page);
    }
  }
  // heads lo .. hi of one kind, the first of which is head ``at`` of the projection
  auto heads = [&](int at, int n, bf16* dst, bf16* cache, const bf16* weight) {
    const int lo = max(it.h0 - at, 0), hi = min(it.h1 - at, n);
    if (lo >= hi) return;
    bf16* const to = dst ? dst + ((int64_t)t * n + lo) * s.hd : nullptr;
    bf16* const held = cache && row >= 0 ? cache + (row + (int64_t)lo * a.cache.page) * s.hd : nullptr;
    auto put = [&](int x, const Raw& r) {
      if (to) store_raw(to + (int64_t)x * s.hd, w, r);
      if (held) store_raw(held + (int64_t)x * a.cache.page * s.hd, w, r);
    };
    const bf16* from = src + (int64_t)(at + lo) * s.hd;
    if constexpr (NORM) {
      const Raw none = no_raw();
      const Pairs wt = unpack<INTER>(on ? load_raw(weight, w) : none);
      const Turn turned = turn_of(g, wt);
      auto load = [&](int x) { return on && x < hi - lo ? load_raw(from + (int64_t)x * s.hd, w) : none; };
      Raw next[kNormBatch];
#pragma unroll
      for (int x = 0; x < kNormBatch; ++x) next[x] = load(x);
      for (int j = 0; j < hi - lo; j += kNormBatch) {
        Pairs y[kNormBatch];
        float ss[kNormBatch];
#pragma unroll
        for (int x = 0; x < kNormBatch; ++x) {
          y[x] = unpack<INTER>(next[x]);
          next[x] = load(j + kNormBatch + x);
          ss[x] = sum_products(y[x], y[x]);
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
          for (int x = 0; x < kNormBatch; ++x) ss[x] += __shfl_xor_sync(group_mask<L>(), ss[x], o);
#pragma unroll
        for (int x = 0; x < kNormBatch; ++x) {
          if (!on || j + x >= hi - lo) break;
          const float rstd = rsqrtf(ss[x] * a.inv_hd + a.eps);
          put(j + x, pack<INTER>(times(w.turned ? turned(y[x]) : times(y[x], wt), rstd)));
        }
      }
    } else {
      each_row<kBatch>(from, s.hd, hi - lo, w,
                       [&](int x, const Raw& r) { put(x, w.turned ? pack<INTER>(plain(unpack<INTER>(r))) : r); });
    }
  };
  heads(0, s.Hq, a.q, nullptr, a.qn);
  heads(s.Hq, s.Hkv, a.k, a.cache.k, a.kn);
  if (!on) return;
  const int lo = max(it.h0 - HQK, 0), hi = it.h1 - HQK;
  each_row<kBatch>(src + (int64_t)(HQK + lo) * s.hd, s.hd, hi - lo, w, [&](int x, const Raw& r) {
    if (a.v) store_raw(a.v + ((int64_t)t * s.Hkv + lo + x) * s.hd, w, r);
    if (row >= 0) store_raw(a.cache.v + (row + (int64_t)(lo + x) * a.cache.page) * s.hd, w, r);
  });
}

// Without norms the gradient is the turn back; the projection is not read.
template <int L, bool INTER>
__global__ void __launch_bounds__(kThreads, 4) rotary_bwd_kernel(const Args a) {
  const RotaryShape& s = a.s;
  const int lane = threadIdx.x % L;
  pdl_wait();
  pdl_trigger();
  const Item it = item_of<L>(a);
  if (!it.there || C * lane >= s.hd) return;
  const int t = it.t, HQK = s.Hq + s.Hkv;
  const Place w = place_of(s, lane);
  Angles g;
  if (it.h0 < HQK) g = angles(a, w, lane, a.pos[t]);
  const Turn back = turn_of(g, true);
  bf16* dst = a.gqkv + (int64_t)t * (HQK + s.Hkv) * s.hd;
  auto heads = [&](int at, int n, const bf16* grad, bool turned) {
    const int lo = max(it.h0 - at, 0), hi = min(it.h1 - at, n);
    each_row<kBatch>(grad + ((int64_t)t * n + lo) * s.hd, s.hd, hi - lo, w, [&](int x, const Raw& r) {
      store_raw(dst + (int64_t)(at + lo + x) * s.hd, w, turned ? pack<INTER>(back(unpack<INTER>(r))) : r);
    });
  };
  heads(0, s.Hq, a.gq, w.turned);
  heads(s.Hq, s.Hkv, a.gk, w.turned);
  heads(HQK, s.Hkv, a.gv, false);
}

// With norms: the items of all tokens, an item being kNormBatch query (or key) heads of one, are split evenly over a fixed
// number of warps, whose groups take neighbouring ones. A lane keeps its channels' part of the weights' gradients, the
// CTA's groups add theirs up in order and a second kernel adds the CTAs'. So every sum has one order.
constexpr int kNormCtas = 148 * 2;
constexpr int kCopies = 8;

template <int L, bool INTER>
__global__ void __launch_bounds__(kThreads, 2) rotary_norm_bwd_kernel(const Args a) {
  constexpr int GROUPS = kThreads / L, SIDE = 32 / L;
  __shared__ float sums[GROUPS][C * L];
  const RotaryShape& s = a.s;
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  pdl_wait();
  pdl_trigger();
  const int H = s.Hq + 2 * s.Hkv;
  const bool on = C * lane < s.hd;
  const Place w = on ? place_of(s, lane) : Place{0, 0, false};
  constexpr int WARPS = kThreads / 32;
  const int64_t warps = (int64_t)gridDim.x * WARPS, warp = (int64_t)blockIdx.x * WARPS + threadIdx.x / 32;
  const Raw none = no_raw();
#pragma unroll 1
  for (int kind = 0; kind < 2; ++kind) {
    const int N = kind ? s.Hkv : s.Hq, at = kind ? s.Hq : 0;  // heads; where they begin in the projection
    const bf16* grad = kind ? a.gk : a.gq;
    const FastDiv items = kind ? a.k_items : a.q_items;  // of a token
    const Pairs wt = unpack<INTER>(on ? load_raw(kind ? a.kn : a.qn, w) : none);
    Pairs dw = unpack<INTER>(none);
    const int64_t n = (int64_t)s.T * items.d, begin = warp * n / warps, end = (warp + 1) * n / warps;
    // This group's walk: token, first head of the item, rows of the projection and of the gradient there.
    const int64_t i0 = begin + group % SIDE;
    int t = i0 < end ? (int)items.div((uint32_t)i0) : 0, h0 = i0 < end ? (int)(i0 - (int64_t)t * items.d) * kNormBatch : 0;
    int left = (int)(end - begin) - group % SIDE;  // items from this one on
    const int wrap = items.d * kNormBatch;         // where a token's items end, a head behind its last if N is odd
    int64_t from = t * a.qs + (int64_t)(at + h0) * s.hd, to = ((int64_t)t * H + at + h0) * s.hd;
    int64_t gfrom = ((int64_t)t * N + h0) * s.hd;
    struct Load {
      Raw x[kNormBatch], g[kNormBatch];
    };
    auto load = [&]() {
      Load r;
      const int m = on && left > 0 ? N - h0 : 0;
#pragma unroll
      for (int x = 0; x < kNormBatch; ++x) {
        r.x[x] = x < m ? load_raw(a.qkv + from + x * s.hd, w) : none;
        r.g[x] = x < m ? load_raw(grad + gfrom + x * s.hd, w) : none;
      }
      return r;
    };
    Load next = load();
    int p = a.pos[t];
    Turn back;
    int held = -1;  // the token whose angles are at hand
    for (int turns = (int)(end - begin + SIDE - 1) / SIDE; turns > 0; --turns) {
      Pairs y[kNormBatch], z[kNormBatch];
      float ss[kNormBatch], dot[kNormBatch];
#pragma unroll
      for (int x = 0; x < kNormBatch; ++x) {
        y[x] = unpack<INTER>(next.x[x]);
        z[x] = unpack<INTER>(next.g[x]);
      }
      if (__any_sync(0xffffffffu, t != held)) {
        back = turn_of(angles(a, w, lane, p), true);
        held = t;
      }
      const int m = on && left > 0 ? N - h0 : 0;
      bf16* dst = a.gqkv + to;
      left -= SIDE;
      h0 += SIDE * kNormBatch;
      from += SIDE * kNormBatch * s.hd;
      to += SIDE * kNormBatch * s.hd;
      gfrom += SIDE * kNormBatch * s.hd;
      while (h0 >= wrap && left > 0) {
        h0 -= wrap;
        ++t;
        from += a.qs - wrap * s.hd;
        to += (H - wrap) * s.hd;
        gfrom += (N - wrap) * s.hd;
      }
      next = load();
      p = a.pos[t];
#pragma unroll
      for (int x = 0; x < kNormBatch; ++x) {
        if (w.turned) z[x] = back(z[x]);
        ss[x] = sum_products(y[x], y[x]);
        dot[x] = sum_products(times(z[x], wt), y[x]);
      }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
        for (int x = 0; x < kNormBatch; ++x) {
          ss[x] += __shfl_xor_sync(0xffffffffu, ss[x], o);
          dot[x] += __shfl_xor_sync(0xffffffffu, dot[x], o);
        }
#pragma unroll
      for (int x = 0; x < kNormBatch; ++x) {
        if (x >= m) break;
        const float rstd = rsqrtf(ss[x] * a.inv_hd + a.eps);
        const float mean = dot[x] * a.inv_hd * rstd * rstd;  // of the gradient times x rstd, times rstd
        const F2 r2 = f2(rstd, rstd), m2 = f2(-mean, -mean);
        Pairs out;
#pragma unroll
        for (int e = 0; e < C / 4; ++e) {
          dw.a[e] = fma2(z[x].a[e], y[x].a[e] * r2, dw.a[e]);
          dw.b[e] = fma2(z[x].b[e], y[x].b[e] * r2, dw.b[e]);
          out.a[e] = fma2(y[x].a[e], m2, z[x].a[e] * wt.a[e]) * r2;
          out.b[e] = fma2(y[x].b[e], m2, z[x].b[e] * wt.b[e]) * r2;
        }
        store_raw(dst + x * s.hd, w, pack<INTER>(out));
      }
    }
    if (on) {
#pragma unroll
      for (int e = 0; e < C / 2; ++e) {
        const float2 da = parts(dw.a[e / 2]), db = parts(dw.b[e / 2]);
        sums[group][channel_of<INTER>(w, e, false)] = e % 2 ? da.y : da.x;
        sums[group][channel_of<INTER>(w, e, true)] = e % 2 ? db.y : db.x;
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < s.hd; c += kThreads) {
      float x = 0.f;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) x += sums[j][c];
      a.part[((int64_t)blockIdx.x * 2 + kind) * s.hd + c] = x;
    }
    __syncthreads();
  }
  // V's gradient is the output's: CTAs take neighbouring tokens, a thread has kCopies loads under way
  const int64_t t0 = (int64_t)blockIdx.x * s.T / gridDim.x, t1 = (int64_t)(blockIdx.x + 1) * s.T / gridDim.x;
  const uint32_t row = a.v_row.d, n = (uint32_t)(t1 - t0) * row;
  const uint2* vfrom = reinterpret_cast<const uint2*>(a.gv) + t0 * row;
  uint2* vto = reinterpret_cast<uint2*>(a.gqkv + (t0 * H + s.Hq + s.Hkv) * s.hd);
  for (uint32_t c = threadIdx.x; c < n; c += kCopies * kThreads) {
    uint2 u[kCopies];
#pragma unroll
    for (int x = 0; x < kCopies; ++x)
      if (c + x * kThreads < n) u[x] = __ldg(vfrom + c + x * kThreads);
#pragma unroll
    for (int x = 0; x < kCopies; ++x) {
      const uint32_t e = c + x * kThreads, t = a.v_row.div(e);
      if (e < n) vto[(int64_t)t * (H * s.hd / 4) + (e - t * row)] = u[x];
    }
  }
}

// part [n][2][hd] summed over n, columns first .. end: 32 of them to a CTA, every kJoinWarps-th row to a warp.
constexpr int kJoinWarps = 32;

__global__ void __launch_bounds__(32 * kJoinWarps)
    rotary_norm_join_kernel(const float* __restrict__ part, int n, int hd, int first, int end, RotaryWeightGrad wq,
                            RotaryWeightGrad wk) {
  __shared__ float sums[kJoinWarps][32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, c = first + blockIdx.x * 32 + lane;
  pdl_wait();
  pdl_trigger();
  float x = 0.f;
  if (c < end) {
#pragma unroll 10
    for (int i = warp; i < n; i += kJoinWarps) x += part[(int64_t)i * 2 * hd + c];
  }
  sums[warp][lane] = x;
  __syncthreads();
  if (warp || c >= end) return;
  x = 0.f;
#pragma unroll
  for (int j = 0; j < kJoinWarps; ++j) x += sums[j][lane];
  const RotaryWeightGrad& g = c < hd ? wq : wk;
  const int at = c < hd ? c : c - hd;
  if (g.add)
    g.add[at] += x;
  else
    g.out[at] = __float2bfloat16_rn(x);
}

int lanes_of(int hd) { return hd <= 64 ? 8 : hd <= 128 ? 16 : 32; }
void check(const RotaryShape& s) {
  MESHY_CHECK(s.hd % 8 == 0 && s.hd > 0 && s.hd <= 256, "rotary: head_dim must be a multiple of 8, at most 256");
  MESHY_CHECK(s.rot % 8 == 0 && s.rot > 0 && s.rot <= s.hd, "rotary: the rotated part must be a multiple of 8, at most head_dim");
}

// Heads of a group: as many as fill the SMs' threads once, split evenly (twice: 512 tokens of a decode step 6.4 us for 4.7,
// the 5003 tokens with norms 21.8 for 19.2).
int heads_of(const RotaryShape& s, int lanes) {
  const int H = s.Hq + 2 * s.Hkv;
  const int64_t groups = 148LL * 2048 / lanes, splits = std::min<int64_t>(H, groups / std::max(1, s.T) + 1);
  return (int)((H + splits - 1) / splits);
}

template <class F>
void with_lanes(const RotaryShape& s, F f) {
  auto go = [&](auto l) { s.interleaved ? f(l, std::true_type{}) : f(l, std::false_type{}); };
  const int L = lanes_of(s.hd);
  L == 8 ? go(std::integral_constant<int, 8>{})
         : L == 16 ? go(std::integral_constant<int, 16>{}) : go(std::integral_constant<int, 32>{});
}

unsigned blocks_of(const RotaryShape& s, int splits, int lanes) {
  const int64_t groups = (int64_t)s.T * splits, per = kThreads / lanes;
  MESHY_CHECK(groups < (1LL << 31), "rotary: too many rows for one call");
  return (unsigned)((groups + per - 1) / per);
}

}  // namespace

void rotary_fwd(RotaryShape s, const bf16* qkv, int64_t qs, const int* pos, const uint64_t* turns, float factor,
                const bf16* qn, const bf16* kn, float eps, bf16* q, bf16* k, bf16* v, RotaryCache cache,
                cudaStream_t st) {
  check(s);
  if (s.T == 0) return;
  const int lanes = lanes_of(s.hd), nh = heads_of(s, lanes), splits = (s.Hq + 2 * s.Hkv + nh - 1) / nh;
  Args a{s, qkv, qs, pos, turns, factor, qn, kn, eps, q, k, v, cache, nullptr, nullptr, nullptr, nullptr, nullptr, nh,
         splits, FastDiv(s.T), FastDiv(1), FastDiv(1), FastDiv(1), 1.f / s.hd};
  with_lanes(s, [&](auto l, auto inter) {
    auto* kernel = qn ? rotary_fwd_kernel<l.value, true, inter.value> : rotary_fwd_kernel<l.value, false, inter.value>;
    launch_pdl(kernel, dim3(blocks_of(s, splits, lanes)), dim3(kThreads), 0, st, a);
  });
}

bool rotary_shared_grad(RotaryWeightGrad wq, RotaryWeightGrad wk, int hd) {
  return wq.add && wk.add && wq.add < wk.add + hd && wk.add < wq.add + hd;
}

int64_t rotary_part_floats(RotaryShape s) { return (int64_t)kNormCtas * 2 * s.hd; }

void rotary_bwd(RotaryShape s, const bf16* qkv, int64_t qs, const int* pos, const uint64_t* turns, float factor,
                const bf16* qn, const bf16* kn, float eps, const bf16* gq, const bf16* gk, const bf16* gv, bf16* gqkv,
                RotaryWeightGrad wq, RotaryWeightGrad wk, float* part, cudaStream_t st) {
  check(s);
  const int lanes = lanes_of(s.hd), nh = heads_of(s, lanes), splits = (s.Hq + 2 * s.Hkv + nh - 1) / nh;
  Args a{s, qkv, qs, pos, turns, factor, qn, kn, eps, nullptr, nullptr, nullptr, RotaryCache{}, gq, gk, gv, gqkv, part,
         nh, splits, FastDiv(std::max(1, s.T)), FastDiv((s.Hq + kNormBatch - 1) / kNormBatch),
         FastDiv((s.Hkv + kNormBatch - 1) / kNormBatch), FastDiv(s.Hkv * s.hd / 4), 1.f / s.hd};
  if (!qn) {
    if (s.T == 0) return;
    with_lanes(s, [&](auto l, auto inter) {
      launch_pdl(rotary_bwd_kernel<l.value, inter.value>, dim3(blocks_of(s, splits, lanes)), dim3(kThreads), 0, st, a);
    });
    return;
  }
  MESHY_CHECK((int64_t)s.T * a.q_items.d < (1LL << 31) && (int64_t)s.T * a.k_items.d < (1LL << 31),
              "rotary: too many rows for one call");
  const int64_t per = kThreads / lanes, items = (int64_t)s.T * a.q_items.d;  // (an item to a group at least)
  const int ctas = (int)std::min<int64_t>(kNormCtas, (items + per - 1) / per);  // none for no rows: sums of nothing
  if (ctas)
    with_lanes(s, [&](auto l, auto inter) {
      launch_pdl(rotary_norm_bwd_kernel<l.value, inter.value>, dim3(ctas), dim3(kThreads), 0, st, a);
    });
  auto join = [&](int first, int end) {
    launch_pdl(rotary_norm_join_kernel, dim3((end - first + 31) / 32), dim3(32 * kJoinWarps), 0, st, (const float*)part, ctas,
               s.hd, first, end, wq, wk);
  };
  if (rotary_shared_grad(wq, wk, s.hd)) {  // one after the other
    join(0, s.hd);
    join(s.hd, 2 * s.hd);
  } else {
    join(0, 2 * s.hd);
  }
}

}  // namespace meshy
