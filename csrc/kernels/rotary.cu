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
// rotated part. Its four angles are worked out once for all its heads. The memory's rate bounds the large cases (each
// channel is read and written once), latency the small ones.
#include <cuda_runtime.h>

#include "../include/fastdiv.cuh"
#include "rotary.h"

namespace meshy {

namespace {

constexpr int kThreads = 256;

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
  int nh;          // heads of a group
  FastDiv splits;  // groups of a token
};

// Where a lane's eight channels are: two runs of four (they follow one another unless the layout is by halves).
struct Place {
  int a, b;
  bool turned;
};
__device__ __forceinline__ Place place_of(const RotaryShape& s, int lane) {
  const int half = s.rot / 2;
  if (8 * lane >= s.rot) return {8 * lane, 8 * lane + 4, false};
  return s.interleaved ? Place{8 * lane, 8 * lane + 4, true} : Place{4 * lane, half + 4 * lane, true};
}

// Eight channels as a lane has them: x[0..3] the first run, x[4..7] the second.
__device__ __forceinline__ void load8(const bf16* p, const Place& w, uint2 (&u)[2]) {
  u[0] = *reinterpret_cast<const uint2*>(p + w.a);
  u[1] = *reinterpret_cast<const uint2*>(p + w.b);
}
__device__ __forceinline__ void store8(bf16* p, const Place& w, const uint2 (&u)[2]) {
  *reinterpret_cast<uint2*>(p + w.a) = u[0];
  *reinterpret_cast<uint2*>(p + w.b) = u[1];
}
__device__ __forceinline__ void unpack8(const uint2 (&u)[2], float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 lo = unpack_bf16x2(u[i].x), hi = unpack_bf16x2(u[i].y);
    x[4 * i] = lo.x, x[4 * i + 1] = lo.y, x[4 * i + 2] = hi.x, x[4 * i + 3] = hi.y;
  }
}
__device__ __forceinline__ void pack8(const float (&x)[8], uint2 (&u)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    u[i] = make_uint2(pack_bf16x2(x[4 * i], x[4 * i + 1]), pack_bf16x2(x[4 * i + 2], x[4 * i + 3]));
}

struct Angles {
  float c[4], s[4];
};
__device__ __forceinline__ Angles angles(const Args& a, const Place& w, int lane, int t) {
  Angles g;
  const int64_t p = a.pos[t];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    g.c[i] = 1.f, g.s[i] = 0.f;
    if (!w.turned) continue;
    const uint64_t f = a.turns[4 * lane + i] * (uint64_t)p;
    sincospif((float)(int)(f >> 32) * 4.6566129e-10f, &g.s[i], &g.c[i]);  // 2^-31: half turns
    g.c[i] *= a.factor;
    g.s[i] *= a.factor;
  }
  return g;
}

// Pairs are (x[i], x[4 + i]) by halves, (x[2 i], x[2 i + 1]) interleaved.
template <bool BACK>
__device__ __forceinline__ void turn(float (&x)[8], const Angles& g, bool interleaved) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = interleaved ? x[2 * i] : x[i], b = interleaved ? x[2 * i + 1] : x[4 + i];
    const float s = BACK ? -g.s[i] : g.s[i];
    const float ya = a * g.c[i] - b * s, yb = b * g.c[i] + a * s;
    if (interleaved)
      x[2 * i] = ya, x[2 * i + 1] = yb;
    else
      x[i] = ya, x[4 + i] = yb;
  }
}

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int L, bool NORM, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_fwd_kernel(const Args a) {
  const RotaryShape& s = a.s;
  const int lane = threadIdx.x % L;
  const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
  pdl_wait();
  pdl_trigger();
  const int H = s.Hq + 2 * s.Hkv;
  const bool act = i < (int64_t)s.T * a.splits.d && 8 * lane < s.hd;
  const int t = act ? a.splits.div((uint32_t)i) : 0;
  const int h0 = act ? (int)(i - (int64_t)t * a.splits.d) * a.nh : 0, h1 = act ? min(H, h0 + a.nh) : 0;
  const Place w = place_of(s, lane);
  Angles g;
  if (act && h0 < s.Hq + s.Hkv) g = angles(a, w, lane, t);
  int64_t row = -1;  // of the cache, head 0
  if (act && a.cache.k && h1 > s.Hq) {
    const int64_t slot = a.cache.slots[t], n = a.cache.n_pages * a.cache.page;
    if (slot >= 0 && slot < n) {
      const int64_t p = slot / a.cache.page;
      row = p * s.Hkv * a.cache.page + (slot - p * a.cache.page);
    }
  }
  const bf16* src = a.qkv + t * a.qs;
#pragma unroll 4
  for (int j = 0; j < a.nh; ++j) {  // all lanes of a warp take every turn, for the sums
    const int h = h0 + j;
    const bool in = h < h1;
    if (!NORM && !in) break;
    uint2 u[2] = {make_uint2(0, 0), make_uint2(0, 0)};
    if (in) load8(src + (int64_t)h * s.hd, w, u);
    const bool is_q = h < s.Hq, is_v = h >= s.Hq + s.Hkv;
    if (!is_v || NORM) {
      float x[8];
      unpack8(u, x);
      if (NORM) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
        const float rstd = rsqrtf(group_sum<L>(ss) / s.hd + a.eps);
        if (in && !is_v) {
          uint2 nw[2];
          float f[8];
          load8(is_q ? a.qn : a.kn, w, nw);
          unpack8(nw, f);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= rstd * f[e];
        }
      }
      if (in && !is_v) {
        if (w.turned) turn<false>(x, g, INTER);
        pack8(x, u);
      }
    }
    if (!in) continue;
    const int hk = is_v ? h - s.Hq - s.Hkv : h - s.Hq;
    bf16* dst = is_q ? a.q : is_v ? a.v : a.k;
    if (dst) store8(dst + ((int64_t)t * (is_q ? s.Hq : s.Hkv) + (is_q ? h : hk)) * s.hd, w, u);
    if (!is_q && row >= 0) store8((is_v ? a.cache.v : a.cache.k) + (row + (int64_t)hk * a.cache.page) * s.hd, w, u);
  }
}

// Without norms the gradient is the turn back; the projection is not read.
template <int L, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_bwd_kernel(const Args a) {
  const RotaryShape& s = a.s;
  const int lane = threadIdx.x % L;
  const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / L;
  pdl_wait();
  pdl_trigger();
  const int H = s.Hq + 2 * s.Hkv;
  if (i >= (int64_t)s.T * a.splits.d || 8 * lane >= s.hd) return;
  const int t = a.splits.div((uint32_t)i), h0 = (int)(i - (int64_t)t * a.splits.d) * a.nh, h1 = min(H, h0 + a.nh);
  const Place w = place_of(s, lane);
  Angles g;
  if (h0 < s.Hq + s.Hkv) g = angles(a, w, lane, t);
  bf16* dst = a.gqkv + (int64_t)t * H * s.hd;
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const bool is_q = h < s.Hq, is_v = h >= s.Hq + s.Hkv;
    const bf16* src = is_q ? a.gq + ((int64_t)t * s.Hq + h) * s.hd
                           : (is_v ? a.gv : a.gk) + ((int64_t)t * s.Hkv + (is_v ? h - s.Hq - s.Hkv : h - s.Hq)) * s.hd;
    uint2 u[2];
    load8(src, w, u);
    if (!is_v && w.turned) {
      float x[8];
      unpack8(u, x);
      turn<true>(x, g, INTER);
      pack8(x, u);
    }
    store8(dst + (int64_t)h * s.hd, w, u);
  }
}

// With norms: a fixed number of CTAs walk over the tokens, a group a token; a lane keeps its channels' part of the
// weights' gradients, the CTA's groups add theirs up in order and a second kernel adds the CTAs'. So every sum has one
// order.
constexpr int kNormCtas = 148 * 4;

template <int L, bool INTER>
__global__ void __launch_bounds__(kThreads) rotary_norm_bwd_kernel(const Args a) {
  constexpr int GROUPS = kThreads / L;
  __shared__ float sums[GROUPS][8 * L];
  const RotaryShape& s = a.s;
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  pdl_wait();
  pdl_trigger();
  const int H = s.Hq + 2 * s.Hkv;
  const bool on = 8 * lane < s.hd;
  const Place w = place_of(s, lane);
  float wq[8], wk[8], dq[8], dk[8];
  {
    uint2 u[2] = {make_uint2(0, 0), make_uint2(0, 0)};
    if (on) load8(a.qn, w, u);
    unpack8(u, wq);
    if (on) load8(a.kn, w, u);
    unpack8(u, wk);
#pragma unroll
    for (int e = 0; e < 8; ++e) dq[e] = dk[e] = 0.f;
  }
  const float inv = 1.f / s.hd;
  for (int64_t t0 = (int64_t)blockIdx.x * GROUPS; t0 < s.T; t0 += (int64_t)gridDim.x * GROUPS) {
    const int64_t t = t0 + group;
    const bool act = on && t < s.T;
    Angles g;
    if (act) g = angles(a, w, lane, (int)t);
    const bf16* src = a.qkv + t * a.qs;
    bf16* dst = a.gqkv + t * H * s.hd;
    auto head = [&](int h, const bf16* grad, const float (&wt)[8], float (&dw)[8]) {
      uint2 u[2] = {make_uint2(0, 0), make_uint2(0, 0)}, ug[2] = {make_uint2(0, 0), make_uint2(0, 0)};
      if (act) {
        load8(src + (int64_t)h * s.hd, w, u);
        load8(grad, w, ug);
      }
      float x[8], y[8], ss = 0.f, dot = 0.f;
      unpack8(u, x);
      unpack8(ug, y);
      if (act && w.turned) turn<true>(y, g, INTER);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss = fmaf(x[e], x[e], ss);
        dot = fmaf(y[e] * wt[e], x[e], dot);
      }
      const float rstd = rsqrtf(group_sum<L>(ss) * inv + a.eps);
      const float mean = group_sum<L>(dot) * inv * rstd * rstd;  // of the gradient times x rstd, times rstd
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dw[e] = fmaf(y[e], x[e] * rstd, dw[e]);
        y[e] = rstd * (y[e] * wt[e] - x[e] * mean);
      }
      if (act) {
        pack8(y, u);
        store8(dst + (int64_t)h * s.hd, w, u);
      }
    };
#pragma unroll 2
    for (int h = 0; h < s.Hq; ++h) head(h, a.gq + (t * s.Hq + h) * s.hd, wq, dq);
#pragma unroll 2
    for (int h = 0; h < s.Hkv; ++h) head(s.Hq + h, a.gk + (t * s.Hkv + h) * s.hd, wk, dk);
    if (act)
      for (int h = 0; h < s.Hkv; ++h) {
        uint2 u[2];
        load8(a.gv + (t * s.Hkv + h) * s.hd, w, u);
        store8(dst + (int64_t)(s.Hq + s.Hkv + h) * s.hd, w, u);
      }
  }
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    if (on) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sums[group][e < 4 ? w.a + e : w.b + e - 4] = kind ? dk[e] : dq[e];
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
}

// part [n][2][hd] summed over n and added to gqn, gkn: a warp to a column.
__global__ void __launch_bounds__(kThreads)
    rotary_norm_join_kernel(const float* __restrict__ part, int n, int hd, float* __restrict__ gqn,
                            float* __restrict__ gkn) {
  const int c = blockIdx.x * (kThreads / 32) + threadIdx.x / 32, lane = threadIdx.x % 32;
  pdl_wait();
  pdl_trigger();
  if (c >= 2 * hd) return;
  float x = 0.f;
  for (int i = lane; i < n; i += 32) x += part[(int64_t)i * 2 * hd + c];
  x = warp_sum(x);
  if (lane == 0) {
    float* g = c < hd ? gqn + c : gkn + c - hd;
    *g += x;
  }
}

int lanes_of(int hd) { return hd <= 64 ? 8 : hd <= 128 ? 16 : 32; }

void check(const RotaryShape& s) {
  MESHY_CHECK(s.hd % 8 == 0 && s.hd > 0 && s.hd <= 256, "rotary: head_dim must be a multiple of 8, at most 256");
  MESHY_CHECK(s.rot % 8 == 0 && s.rot > 0 && s.rot <= s.hd, "rotary: the rotated part must be a multiple of 8, at most head_dim");
}

// Heads of a group: all of them once the tokens alone fill the SMs' threads.
int heads_of(const RotaryShape& s) {
  const int H = s.Hq + 2 * s.Hkv;
  const int64_t groups = 148LL * 2048 / lanes_of(s.hd);
  return (int)std::max<int64_t>(1, std::min<int64_t>(H, (int64_t)s.T * H / groups));
}

template <class F>
void with_lanes(int hd, bool inter, F f) {
  auto go = [&](auto l) {
    if (inter)
      f(l, std::true_type{});
    else
      f(l, std::false_type{});
  };
  const int L = lanes_of(hd);
  L == 8 ? go(std::integral_constant<int, 8>{}) : L == 16 ? go(std::integral_constant<int, 16>{}) : go(std::integral_constant<int, 32>{});
}

unsigned blocks_of(const RotaryShape& s, int splits) {
  const int64_t groups = (int64_t)s.T * splits, per = kThreads / lanes_of(s.hd);
  MESHY_CHECK(groups < (1LL << 31), "rotary: too many rows for one call");
  return (unsigned)((groups + per - 1) / per);
}

}  // namespace

void rotary_fwd(RotaryShape s, const bf16* qkv, int64_t qs, const int* pos, const uint64_t* turns, float factor,
                const bf16* qn, const bf16* kn, float eps, bf16* q, bf16* k, bf16* v, RotaryCache cache,
                cudaStream_t st) {
  check(s);
  if (s.T == 0) return;
  const int nh = heads_of(s), splits = (s.Hq + 2 * s.Hkv + nh - 1) / nh;
  Args a{s, qkv, qs, pos, turns, factor, qn, kn, eps, q, k, v, cache, nullptr, nullptr, nullptr, nullptr, nullptr, nh,
         FastDiv(splits)};
  with_lanes(s.hd, s.interleaved, [&](auto l, auto inter) {
    auto* kernel = qn ? rotary_fwd_kernel<l.value, true, inter.value> : rotary_fwd_kernel<l.value, false, inter.value>;
    launch_pdl(kernel, dim3(blocks_of(s, splits)), dim3(kThreads), 0, st, a);
  });
}

int64_t rotary_part_floats(RotaryShape s) { return (int64_t)kNormCtas * 2 * s.hd; }

void rotary_bwd(RotaryShape s, const bf16* qkv, int64_t qs, const int* pos, const uint64_t* turns, float factor,
                const bf16* qn, const bf16* kn, float eps, const bf16* gq, const bf16* gk, const bf16* gv, bf16* gqkv,
                float* gqn, float* gkn, float* part, cudaStream_t st) {
  check(s);
  if (s.T == 0) return;
  const int nh = heads_of(s), splits = (s.Hq + 2 * s.Hkv + nh - 1) / nh;
  Args a{s, qkv, qs, pos, turns, factor, qn, kn, eps, nullptr, nullptr, nullptr, RotaryCache{}, gq, gk, gv, gqkv, part,
         nh, FastDiv(splits)};
  if (!qn) {
    with_lanes(s.hd, s.interleaved, [&](auto l, auto inter) {
      launch_pdl(rotary_bwd_kernel<l.value, inter.value>, dim3(blocks_of(s, splits)), dim3(kThreads), 0, st, a);
    });
    return;
  }
  const int per = kThreads / lanes_of(s.hd), ctas = std::min(kNormCtas, (s.T + per - 1) / per);
  with_lanes(s.hd, s.interleaved, [&](auto l, auto inter) {
    launch_pdl(rotary_norm_bwd_kernel<l.value, inter.value>, dim3(ctas), dim3(kThreads), 0, st, a);
  });
  launch_pdl(rotary_norm_join_kernel, dim3((2 * s.hd + kThreads / 32 - 1) / (kThreads / 32)), dim3(kThreads), 0, st,
             (const float*)part, ctas, s.hd, gqn, gkn);
}

}  // namespace meshy
