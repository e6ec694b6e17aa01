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
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float n = fminf(fmaxf(quotient(x[q] - zf, af, rcp), 0.f), 15.f);
      // adding 1.5 2^23 rounds to whole numbers, halves to even, and leaves the number in the low bits
      word |= (__float_as_uint(n + 12582912.f) & 15u) << (4 * q);
    }
  }
  if (row == nullptr) return;
  row[lane % 8 * G + lane / 8] = word;
  if (lane % 8 == 0) pairs[lane / 8] = __halves2half2(a, z);
}

// HD / 8 lanes per (token, head); each takes its word of K and of V.
template <int HD>
__global__ void __launch_bounds__(kThreads)
    kv4_write_kernel(const bf16* __restrict__ k, int64_t ks, int64_t kh, const bf16* __restrict__ v, int64_t vs,
                     int64_t vh, const int64_t* __restrict__ slots, uint32_t rows, KV4View c, FastDiv heads, FastDiv page) {
  constexpr int LANES = HD / 8, G = HD / 64;
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x, lane = i % LANES;
  pdl_wait();
  pdl_trigger();
  const bool act = i / LANES < rows;  // the lanes of a group stay together for the shuffles
  const uint32_t th = act ? i / LANES : 0u, t = heads.div(th), h = th - t * heads.d;
  const uint4 uk = *reinterpret_cast<const uint4*>(k + t * ks + h * kh + lane * 8);
  const uint4 uv = *reinterpret_cast<const uint4*>(v + t * vs + h * vh + lane * 8);
  const int64_t r = act ? row_of(c, page, slots[t], h) : -1;
  uint32_t* kr = r < 0 ? nullptr : reinterpret_cast<uint32_t*>(c.k + r * (HD / 2));
  uint32_t* vr = r < 0 ? nullptr : reinterpret_cast<uint32_t*>(c.v + r * (HD / 2));
  __half2* pairs = c.scale + r * (2 * G);
  quantise<HD>(uk, lane, kr, pairs);
  quantise<HD>(uv, lane, vr, pairs + G);
}

// Eight channels of a word: a n + z, rounded once.
__device__ __forceinline__ uint4 restore(uint32_t w, __half2 pair) {
  const float2 az = __half22float2(pair);
  uint32_t o[4];
  float x[8];
#pragma unroll
  for (int q = 0; q < 4; ++q) {  // nibbles q and q + 4 as the low bits of the fp16 numbers 1024 + n
    const uint32_t y = ((w >> (4 * q)) & 0x000F000Fu) | 0x64006400u;
    const float2 n = __half22float2(__hsub2(*reinterpret_cast<const __half2*>(&y), __float2half2_rn(1024.f)));
    x[q] = fmaf(n.x, az.x, az.y);
    x[q + 4] = fmaf(n.y, az.x, az.y);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) o[q] = pack_bf16x2(x[2 * q], x[2 * q + 1]);
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int HD>
__global__ void __launch_bounds__(kThreads)
    kv4_read_kernel(KV4View c, const int64_t* __restrict__ slots, uint32_t rows, bf16* __restrict__ k, bf16* __restrict__ v,
                    FastDiv heads, FastDiv page) {
  constexpr int LANES = HD / 8, G = HD / 64;
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x, lane = i % LANES, th = i / LANES;
  pdl_wait();
  pdl_trigger();
  if (th >= rows) return;
  const uint32_t t = heads.div(th), h = th - t * heads.d;
  const int64_t r = row_of(c, page, slots[t], h);
  uint4 ok = make_uint4(0, 0, 0, 0), ov = ok;
  if (r >= 0) {
    const int at = lane % 8 * G + lane / 8;
    const uint32_t wk = reinterpret_cast<const uint32_t*>(c.k + r * (HD / 2))[at];
    const uint32_t wv = reinterpret_cast<const uint32_t*>(c.v + r * (HD / 2))[at];
    const __half2* pairs = c.scale + r * (2 * G) + lane / 8;
    ok = restore(wk, pairs[0]);
    ov = restore(wv, pairs[G]);
  }
  const int64_t to = (int64_t)th * HD + lane * 8;
  *reinterpret_cast<uint4*>(k + to) = ok;
  *reinterpret_cast<uint4*>(v + to) = ov;
}

int blocks(int64_t threads) {
  MESHY_CHECK(threads < (1LL << 31), "kv4: too many rows for one call");
  return (int)((threads + kThreads - 1) / kThreads);
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
