// 4-bit KV cache: quantising write and read-back (layout in kv4.h).
//
// A group of 64 channels x is kept as a = fp16((hi - lo) / 15), z = fp16(lo) and n = rint((x - z) / a) in [0, 15],
// lo and hi being the group's extremes after clamping x to fp16's range. Scale and base are fp16: at 64 channels to
// a pair they add an eighth to the nibbles, and fp16's 11 bits hold z to a fraction of a step (bf16's 8 would
// lose a step wherever a channel offset is some ten times the spread). Every step is an exactly rounded operation,
// so the bytes are the same wherever the format is computed.
//
// Both kernels should run at the memory's rate; in the write the quotients stand in the way (nine channels a clock and
// SM at that rate), so each is a product and two fused multiply-adds with the group's reciprocal instead of a division,
// on pairs of channels in one instruction. 32768 tokens of 8 heads of 128, at slots of shuffled pages: the write takes
// 36-37 us for 172 MB (4.7 TB/s; instruction issue, 65 % of the slots), the read-back 28-30 us for as much (5.9 TB/s, the
// memory's rate). Decode-size calls take 4 us for both in a stream, launch and latency.
#include <cuda_runtime.h>

#include "kv4.h"

namespace meshy {

namespace {

constexpr int kThreads = 128;
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

// Two fp32 numbers and their sums and products, one instruction to a pair.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// 1 / y, correctly rounded for every positive fp16 number y: the hardware's approximation and one Newton step.
__device__ __forceinline__ float reciprocal(float y) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
  return fmaf(fmaf(-y, r, 1.f), r, r);
}

__device__ __forceinline__ float min_nan(float x, float y) {  // NaN if x is
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}

__device__ __forceinline__ float to_half_range(float x) {  // NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(min_nan(x, kHalfMax)), "f"(-kHalfMax));
  return r;
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

// Four lanes hold a group, sixteen channels (two words of nibbles) each; ``row`` null: nothing is written.
template <int HD>
__device__ __forceinline__ void quantise(const uint4& u0, const uint4& u1, int lane, uint32_t* row, __half2* pairs) {
  constexpr int G = HD / 64;
  const uint32_t us[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
  // extremes in bf16, where they are exact; (hi, -lo) side by side through the lanes; a NaN stays one
  __nv_bfloat162 hi2 = as_bf162(us[0]), lo2 = hi2;
#pragma unroll
  for (int q = 1; q < 8; ++q) {
    hi2 = __hmax2_nan(hi2, as_bf162(us[q]));
    lo2 = __hmin2_nan(lo2, as_bf162(us[q]));
  }
  lo2 = __hneg2(lo2);
  const uint32_t h = as_u32(hi2), l = as_u32(lo2);
  __nv_bfloat162 both = __hmax2_nan(as_bf162(__byte_perm(h, l, 0x5410)), as_bf162(__byte_perm(h, l, 0x7632)));
#pragma unroll
  for (int o = 2; o > 0; o >>= 1) both = __hmax2_nan(both, as_bf162(__shfl_xor_sync(0xffffffffu, as_u32(both), o)));
  const float top = __low2float(both), bot = __high2float(both);  // bot: -lo
  const float hi = to_half_range(top), lo = -to_half_range(bot);  // both ends: a group may lie beyond the range whole
  const __half a = __float2half_rn(quotient(hi - lo, 15.f, 1.f / 15.f)), z = __float2half_rn(lo);
  const float af = __half2float(a), zf = __half2float(z), rcp = af > 0.f ? reciprocal(af) : 0.f;
  // Nothing leaves [0, 15] while rounding moved the base by less than 0.4 steps and the scale by less than 2^-11 of it.
  const bool tight = fabsf(lo) * 0.00048828125f < 0.4f * af && af >= 6.1035156e-5f && fmaxf(top, bot) <= kHalfMax;
  if (row == nullptr) return;
  // Adding 1.5 2^23 rounds to whole numbers, halves to even, and leaves the number in the low bits; the constant's own
  // bits leave the word again.
  const uint64_t nz = pair(-zf, -zf), na = pair(-af, -af), rr = pair(rcp, rcp), round2 = pair(12582912.f, 12582912.f);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    uint64_t n2[4];  // rounded quotients, two to a register pair
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 f = unpack_bf16x2(us[4 * w + q]);
      const uint64_t x = add2(pair(f.x, f.y), nz), y = mul2(x, rr);
      n2[q] = add2(fma2(fma2(y, na, x), rr, y), round2);
    }
    if (!tight) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 f = unpack_bf16x2(us[4 * w + q]);
        const float x0 = fminf(fmaxf(f.x, -kHalfMax), kHalfMax), x1 = fminf(fmaxf(f.y, -kHalfMax), kHalfMax);
        const float n0 = fminf(fmaxf(quotient(x0 - zf, af, rcp), 0.f), 15.f);
        const float n1 = fminf(fmaxf(quotient(x1 - zf, af, rcp), 0.f), 15.f);
        n2[q] = add2(pair(n0, n1), round2);
      }
    }
    constexpr uint32_t kRoundBits = 0x4B400000u;  // 1.5 2^23
    uint32_t word = 0u - kRoundBits * 0x11111111u;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      word += (uint32_t)n2[q] * (1u << (8 * q)) + (uint32_t)(n2[q] >> 32) * (1u << (8 * q + 4));
    row[(lane % 4 * 2 + w) * G + lane / 4] = af > 0.f ? word : 0u;
  }
  if (lane % 4 == 0) pairs[lane / 4] = __halves2half2(a, z);
}

// HD / 16 lanes per token and NH heads of it: a lane takes its words of K and of V of each head; the slot is resolved
// once.
template <int HD, int NH>
__global__ void __launch_bounds__(kThreads)
    kv4_write_kernel(const bf16* __restrict__ k, int64_t ks, int64_t kh, const bf16* __restrict__ v, int64_t vs,
                     int64_t vh, const int64_t* __restrict__ slots, uint32_t items, KV4View c, FastDiv splits,
                     FastDiv page) {
  constexpr int LANES = HD / 16, G = HD / 64;
  const uint32_t lane = threadIdx.x % LANES, i = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  pdl_wait();
  pdl_trigger();
  const bool act = i < items;  // the lanes of a group stay together for the shuffles
  const uint32_t t = act ? splits.div(i) : 0u;
  const int h0 = act ? (i - t * splits.d) * NH : 0;
  const bf16* kp = k + t * ks + h0 * kh + lane * 16;
  const bf16* vp = v + t * vs + h0 * vh + lane * 16;
  const int64_t r = act ? row_of(c, page, slots[t], h0) : -1;
  uint32_t* kr = reinterpret_cast<uint32_t*>(c.k) + r * (HD / 8);
  uint32_t* vr = reinterpret_cast<uint32_t*>(c.v) + r * (HD / 8);
  __half2* pairs = c.scale + r * (2 * G);
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    if (h0 + j >= c.Hkv) kp = k, vp = v, kh = vh = 0;  // any row that is there: nothing of it is written
    const bool in = r >= 0 && h0 + j < c.Hkv;
    const uint4 k0 = reinterpret_cast<const uint4*>(kp)[0], k1 = reinterpret_cast<const uint4*>(kp)[1];
    const uint4 v0 = reinterpret_cast<const uint4*>(vp)[0], v1 = reinterpret_cast<const uint4*>(vp)[1];
    quantise<HD>(k0, k1, lane, in ? kr : nullptr, pairs);
    quantise<HD>(v0, v1, lane, in ? vr : nullptr, pairs + G);
    kp += kh;
    vp += vh;
    kr += (int64_t)c.page * (HD / 8);
    vr += (int64_t)c.page * (HD / 8);
    pairs += (int64_t)c.page * (2 * G);
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

template <int HD, int NH>
__global__ void __launch_bounds__(kThreads)
    kv4_read_kernel(KV4View c, const int64_t* __restrict__ slots, uint32_t items, bf16* __restrict__ k,
                    bf16* __restrict__ v, FastDiv splits, FastDiv page) {
  constexpr int LANES = HD / 8, G = HD / 64;
  const uint32_t lane = threadIdx.x % LANES, i = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  pdl_wait();
  pdl_trigger();
  if (i >= items) return;
  const uint32_t t = splits.div(i);
  const int h0 = (i - t * splits.d) * NH;
  const int64_t r = row_of(c, page, slots[t], h0);
  const int at = lane % 8 * G + lane / 8;
  const uint32_t* kr = reinterpret_cast<const uint32_t*>(c.k) + r * (HD / 8) + at;
  const uint32_t* vr = reinterpret_cast<const uint32_t*>(c.v) + r * (HD / 8) + at;
  const __half2* pairs = c.scale + r * (2 * G) + lane / 8;
  uint32_t wk[NH], wv[NH];
  __half2 pk[NH], pv[NH];
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    wk[j] = wv[j] = 0u;
    pk[j] = pv[j] = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
    if (r < 0 || h0 + j >= c.Hkv) continue;
    const int64_t to = (int64_t)j * c.page;
    wk[j] = kr[to * (HD / 8)];
    wv[j] = vr[to * (HD / 8)];
    pk[j] = pairs[to * (2 * G)];
    pv[j] = pairs[to * (2 * G) + G];
  }
  const int64_t o = ((int64_t)t * c.Hkv + h0) * HD + lane * 8;
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    if (h0 + j >= c.Hkv) break;
    *reinterpret_cast<uint4*>(k + o + j * HD) = restore(wk[j], pk[j]);
    *reinterpret_cast<uint4*>(v + o + j * HD) = restore(wv[j], pv[j]);
  }
}

// Four heads to a thread once that still leaves every SM its threads (32768 tokens of 8 heads: 35.7 us, with two 38.3,
// with eight 38.7); one in a decode step, where a thread's heads come after one another and only latency counts.
constexpr int kManyRows = 1 << 16;

struct Split {
  uint32_t items, heads;  // (token, group of heads) pairs; groups of a token
  int blocks;
};
Split split(int T, const KV4View& c, int nh, int channels) {  // channels of a lane
  const int64_t heads = (c.Hkv + nh - 1) / nh, items = T * heads, per = kThreads / (c.hd / channels);
  MESHY_CHECK(items < (1LL << 31), "kv4: too many rows for one call");
  return {(uint32_t)items, (uint32_t)heads, (int)((items + per - 1) / per)};
}

}  // namespace

void kv4_write(const bf16* k, int64_t ks, int64_t kh, const bf16* v, int64_t vs, int64_t vh, const int64_t* slots,
               int T, KV4View c, cudaStream_t st) {
  if (T == 0) return;
  auto go = [&](auto kernel, int nh) {
    const Split x = split(T, c, nh, 16);
    launch_pdl(kernel, dim3(x.blocks), dim3(kThreads), 0, st, k, ks, kh, v, vs, vh, slots, x.items, c, FastDiv(x.heads),
               FastDiv(c.page));
  };
  const bool many = (int64_t)T * c.Hkv >= kManyRows;
  if (c.hd == 128)
    many ? go(kv4_write_kernel<128, 4>, 4) : go(kv4_write_kernel<128, 1>, 1);
  else
    many ? go(kv4_write_kernel<64, 4>, 4) : go(kv4_write_kernel<64, 1>, 1);
}

void kv4_read(KV4View c, const int64_t* slots, int T, bf16* k, bf16* v, cudaStream_t st) {
  if (T == 0) return;
  auto go = [&](auto kernel, int nh) {
    const Split x = split(T, c, nh, 8);
    launch_pdl(kernel, dim3(x.blocks), dim3(kThreads), 0, st, c, slots, x.items, k, v, FastDiv(x.heads), FastDiv(c.page));
  };
  const bool many = (int64_t)T * c.Hkv >= kManyRows;
  if (c.hd == 128)
    many ? go(kv4_read_kernel<128, 4>, 4) : go(kv4_read_kernel<128, 1>, 1);
  else
    many ? go(kv4_read_kernel<64, 4>, 4) : go(kv4_read_kernel<64, 1>, 1);
}

}  // namespace meshy
