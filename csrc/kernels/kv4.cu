// 4-bit KV cache: quantising write and read-back (layout in kv4.h).
//
// A group of 64 channels x is kept as a = fp16((hi - lo) / 15), z = fp16(lo) and n = rint((x - z) / a) in [0, 15],
// lo and hi being the group's extremes after clamping x to fp16's range. Scale and base are fp16: at 64 channels to
// a pair they add an eighth to the nibbles, and fp16's 11 bits hold z to a fraction of a step (bf16's 8 would
// lose a step wherever a channel offset is some ten times the spread). Every step is an exactly rounded operation,
// so the bytes are the same wherever the format is computed.
//
// Both kernels move 16 bytes of bf16 against 4 of nibbles per thread and are meant to run at the memory's rate; the
// quotients are what stands in the way (nine channels a clock and SM at that rate), so each is one product and two
// fused multiply-adds with the group's reciprocal instead of a division.
#include <cuda_runtime.h>

#include "kv4.h"

namespace meshy {

namespace {

constexpr int kThreads = 256;
constexpr float kHalfMax = 65504.f;

// n / d for n < 2^31, as (n m) >> s with m = ceil(2^s / d), s = 31 + ceil(log2 d) (Granlund and Montgomery, 1994).
struct FastDiv {
  uint32_t d, m, s;
  explicit FastDiv(uint32_t d_) : d(d_), s(31) {
    while ((1ull << (s - 31)) < d) ++s;
    m = (uint32_t)(((1ull << s) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> s); }
};

// Correctly rounded x / y from y's correctly rounded reciprocal: one Newton step on the quotient with the exact
// remainder (Markstein, 1990).
__device__ __forceinline__ float quotient(float x, float y, float rcp) {
  const float q = x * rcp;
  return fmaf(fmaf(-q, y, x), rcp, q);
}

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 b) { return *reinterpret_cast<uint32_t*>(&b); }

// Row (page, head, place) of the cache that holds head h of a slot; -1: outside.
__device__ __forceinline__ int64_t row_of(const KV4View& c, FastDiv page, int64_t slot, int h) {
  const int64_t n = c.n_pages * c.page;
  if (slot < 0 || slot >= n) return -1;
  const int64_t p = n < (1LL << 31) ? (int64_t)page.div((uint32_t)slot) : slot / c.page;
  return (p * c.Hkv + h) * c.page + (slot - p * c.page);
}

// Eight lanes hold a group, eight channels (one word of nibbles) each.
template <int HD>
__device__ __forceinline__ void quantise(const uint4& u, int lane, uint32_t* row, __half2* pairs) {
  constexpr int G = HD / 64;
  const uint32_t us[4] = {u.x, u.y, u.z, u.w};
  // extremes in bf16, where they are exact; (hi, -lo) side by side through the lanes; a NaN stays one
  __nv_bfloat162 hi2 = as_bf162(us[0]), lo2 = hi2;
#pragma unroll
  for (int q = 1; q < 4; ++q) {
    hi2 = __hmax2_nan(hi2, as_bf162(us[q]));
    lo2 = __hmin2_nan(lo2, as_bf162(us[q]));
  }
  __nv_bfloat162 both = __halves2bfloat162(__hmax_nan(__low2bfloat16(hi2), __high2bfloat16(hi2)),
                                           __hneg(__hmin_nan(__low2bfloat16(lo2), __high2bfloat16(lo2))));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) both = __hmax2_nan(both, as_bf162(__shfl_xor_sync(0xffffffffu, as_u32(both), o)));
  float hi = __low2float(both), lo = -__high2float(both);
  float x[8];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 f = unpack_bf16x2(us[q]);
    x[2 * q] = f.x;
    x[2 * q + 1] = f.y;
  }
  if (hi > kHalfMax || lo < -kHalfMax) {
    hi = fminf(fmaxf(hi, -kHalfMax), kHalfMax);
    lo = fminf(fmaxf(lo, -kHalfMax), kHalfMax);
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = fminf(fmaxf(x[q], -kHalfMax), kHalfMax);
  }
  const __half a = __float2half_rn(quotient(hi - lo, 15.f, 1.f / 15.f)), z = __float2half_rn(lo);
  const float af = __half2float(a), zf = __half2float(z);
  uint32_t word = 0;
  if (af > 0.f) {
    const float rcp = __frcp_rn(af);
    float n[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) n[q] = quotient(x[q] - zf, af, rcp);
    // the base is rounded: only where that moved it by a good part of a step does anything leave [0, 15]
    if (quotient(lo - zf, af, rcp) < -0.5f || quotient(hi - zf, af, rcp) >= 15.5f) {
#pragma unroll
      for (int q = 0; q < 8; ++q) n[q] = fminf(fmaxf(n[q], 0.f), 15.f);
    }
    // adding 1.5 2^23 rounds to whole numbers, halves to even; four of them fit a float's 24 bits side by side
    constexpr float kRound = 12582912.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) n[q] = (n[q] + kRound) - kRound;
    const float h0 = fmaf(fmaf(fmaf(n[3], 16.f, n[2]), 16.f, n[1]), 16.f, n[0]);
    const float h1 = fmaf(fmaf(fmaf(n[7], 16.f, n[6]), 16.f, n[5]), 16.f, n[4]);
    word = __byte_perm(__float_as_uint(h0 + kRound), __float_as_uint(h1 + kRound), 0x5410);
  }
  if (row == nullptr) return;
  row[lane % 8 * G + lane / 8] = word;
  if (lane % 8 == 0) pairs[lane / 8] = __halves2half2(a, z);
}

// HD / 8 lanes per (token, head); each takes its word of K and of V, of kRows (token, head) pairs in one go so that
// their loads are under way together.
constexpr int kRows = 2;

template <int HD>
__global__ void __launch_bounds__(kThreads)
    kv4_write_kernel(const bf16* __restrict__ k, int64_t ks, int64_t kh, const bf16* __restrict__ v, int64_t vs,
                     int64_t vh, const int64_t* __restrict__ slots, uint32_t rows, KV4View c, FastDiv heads, FastDiv page) {
  constexpr int LANES = HD / 8, G = HD / 64, BLOCK = kThreads / LANES;
  const uint32_t lane = threadIdx.x % LANES, th0 = blockIdx.x * (kRows * BLOCK) + threadIdx.x / LANES;
  pdl_wait();
  pdl_trigger();
  uint4 uk[kRows], uv[kRows];
  int64_t r[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const bool act = th0 + u * BLOCK < rows;  // the lanes of a group stay together for the shuffles
    const uint32_t th = act ? th0 + u * BLOCK : 0u, t = heads.div(th), h = th - t * heads.d;
    uk[u] = *reinterpret_cast<const uint4*>(k + t * ks + h * kh + lane * 8);
    uv[u] = *reinterpret_cast<const uint4*>(v + t * vs + h * vh + lane * 8);
    r[u] = act ? row_of(c, page, slots[t], h) : -1;
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    uint32_t* kr = r[u] < 0 ? nullptr : reinterpret_cast<uint32_t*>(c.k + r[u] * (HD / 2));
    uint32_t* vr = r[u] < 0 ? nullptr : reinterpret_cast<uint32_t*>(c.v + r[u] * (HD / 2));
    __half2* pairs = c.scale + r[u] * (2 * G);
    quantise<HD>(uk[u], lane, kr, pairs);
    quantise<HD>(uv[u], lane, vr, pairs + G);
  }
}

// Eight channels of a word: a n + z, rounded once. A nibble masked in place is an fp16 subnormal, n 2^-24 or n 2^-20;
// the scale takes the power back, exactly.
__device__ __forceinline__ uint4 restore(uint32_t w, __half2 pair) {
  const float2 az = __half22float2(pair);
  const float a0 = az.x * 16777216.f, a1 = az.x * 1048576.f;
  float x[8];
#pragma unroll
  for (int q = 0; q < 2; ++q, w >>= 8) {
    const uint32_t y0 = w & 0x000F000Fu, y1 = w & 0x00F000F0u;  // nibbles 2 q, 2 q + 4; 2 q + 1, 2 q + 5
    const float2 n0 = __half22float2(*reinterpret_cast<const __half2*>(&y0));
    const float2 n1 = __half22float2(*reinterpret_cast<const __half2*>(&y1));
    x[2 * q] = fmaf(n0.x, a0, az.y);
    x[2 * q + 4] = fmaf(n0.y, a0, az.y);
    x[2 * q + 1] = fmaf(n1.x, a1, az.y);
    x[2 * q + 5] = fmaf(n1.y, a1, az.y);
  }
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

template <int HD>
__global__ void __launch_bounds__(kThreads)
    kv4_read_kernel(KV4View c, const int64_t* __restrict__ slots, uint32_t rows, bf16* __restrict__ k, bf16* __restrict__ v,
                    FastDiv heads, FastDiv page) {
  constexpr int LANES = HD / 8, G = HD / 64, BLOCK = kThreads / LANES;
  const uint32_t lane = threadIdx.x % LANES, th0 = blockIdx.x * (kRows * BLOCK) + threadIdx.x / LANES;
  pdl_wait();
  pdl_trigger();
  int64_t r[kRows];
  uint32_t wk[kRows], wv[kRows];
  __half2 pk[kRows], pv[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const uint32_t th = th0 + u * BLOCK, t = heads.div(th), h = th - t * heads.d;
    r[u] = th < rows ? row_of(c, page, slots[t], h) : -1;
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    wk[u] = wv[u] = 0u;
    pk[u] = pv[u] = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
    if (r[u] < 0) continue;
    const int at = lane % 8 * G + lane / 8;
    const __half2* pairs = c.scale + r[u] * (2 * G) + lane / 8;
    wk[u] = reinterpret_cast<const uint32_t*>(c.k + r[u] * (HD / 2))[at];
    wv[u] = reinterpret_cast<const uint32_t*>(c.v + r[u] * (HD / 2))[at];
    pk[u] = pairs[0];
    pv[u] = pairs[G];
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const uint32_t th = th0 + u * BLOCK;
    if (th >= rows) continue;
    const int64_t to = (int64_t)th * HD + lane * 8;
    *reinterpret_cast<uint4*>(k + to) = restore(wk[u], pk[u]);
    *reinterpret_cast<uint4*>(v + to) = restore(wv[u], pv[u]);
  }
}

int blocks(int64_t threads) {
  MESHY_CHECK(threads < (1LL << 31), "kv4: too many rows for one call");
  return (int)((threads + kRows * kThreads - 1) / (kRows * kThreads));
}

}  // namespace

void kv4_write(const bf16* k, int64_t ks, int64_t kh, const bf16* v, int64_t vs, int64_t vh, const int64_t* slots,
               int T, KV4View c, cudaStream_t st) {
  if (T == 0) return;
  const int64_t rows = (int64_t)T * c.Hkv;
  launch_pdl(c.hd == 128 ? kv4_write_kernel<128> : kv4_write_kernel<64>, dim3(blocks(rows * (c.hd / 8))), dim3(kThreads), 0, st,
             k, ks, kh, v, vs, vh, slots, (uint32_t)rows, c, FastDiv(c.Hkv), FastDiv(c.page));
}

void kv4_read(KV4View c, const int64_t* slots, int T, bf16* k, bf16* v, cudaStream_t st) {
  if (T == 0) return;
  const int64_t rows = (int64_t)T * c.Hkv;
  launch_pdl(c.hd == 128 ? kv4_read_kernel<128> : kv4_read_kernel<64>, dim3(blocks(rows * (c.hd / 8))), dim3(kThreads), 0, st, c,
             slots, (uint32_t)rows, k, v, FastDiv(c.Hkv), FastDiv(c.page));
}

}  // namespace meshy
