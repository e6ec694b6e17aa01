// 4-bit KV cache: quantising write and read-back (layout in kv4.h).
//
// A group of 64 channels x is kept as a = fp16((hi - lo) / 15), z = fp16(lo) and n = rint((x - z) / a) in [0, 15],
// lo and hi being the group's extremes after clamping x to fp16's range. Scale and base are fp16: at 64 channels to
// a pair they add an eighth to the nibbles, and fp16's 11 bits hold z to a fraction of a step (bf16's 8 would
// lose a step wherever a channel offset is some ten times the spread).
#include <cuda_runtime.h>

#include "kv4.h"

namespace meshy {

namespace {

constexpr int kThreads = 256;
constexpr float kHalfMax = 65504.f;

// Eight lanes hold one group, eight channels (one 32-bit word of nibbles) each; hd / 8 lanes make a row.
__global__ void __launch_bounds__(kThreads)
    kv4_write_kernel(const bf16* __restrict__ k, int64_t ks, int64_t kh, const bf16* __restrict__ v, int64_t vs,
                     int64_t vh, const int64_t* __restrict__ slots, int T, KV4View c) {
  const int lanes = c.hd / 8, G = c.hd / 64;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  int64_t row = i / lanes;  // (token, head, k or v)
  const int lane = (int)(i % lanes);
  const bool act = row < (int64_t)T * c.Hkv * 2;  // whole groups of 8 lanes are in or out
  if (!act) row = 0;
  const int kv = (int)(row & 1);
  const int h = (int)((row >> 1) % c.Hkv);
  const int64_t t = (row >> 1) / c.Hkv;
  const int64_t slot = slots[t];
  const bf16* src = (kv ? v + t * vs + h * vh : k + t * ks + h * kh) + lane * 8;
  const uint4 u = *reinterpret_cast<const uint4*>(src);
  const uint32_t us[4] = {u.x, u.y, u.z, u.w};
  float x[8];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float2 f = unpack_bf16x2(us[q]);
    x[2 * q] = f.x;
    x[2 * q + 1] = f.y;
  }
  float lo = kHalfMax, hi = -kHalfMax;
  bool nan = false;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    nan |= x[q] != x[q];
    x[q] = fminf(fmaxf(x[q], -kHalfMax), kHalfMax);
    lo = fminf(lo, x[q]);
    hi = fmaxf(hi, x[q]);
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    nan |= __shfl_xor_sync(0xffffffffu, (int)nan, o) != 0;
  }
  __half a = __float2half_rn((hi - lo) / 15.f), z = __float2half_rn(lo);
  if (nan) a = z = __float2half_rn(__int_as_float(0x7fc00000));
  const float af = __half2float(a), zf = __half2float(z);
  uint32_t word = 0;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float n = af > 0.f ? fminf(fmaxf(rintf((x[q] - zf) / af), 0.f), 15.f) : 0.f;
    word |= (uint32_t)n << (4 * q);
  }
  if (!act || slot < 0 || slot >= c.n_pages * c.page) return;
  const int64_t r = ((slot / c.page) * c.Hkv + h) * c.page + slot % c.page;
  const int grp = lane / 8, u8 = lane % 8;
  reinterpret_cast<uint32_t*>((kv ? c.v : c.k) + r * (c.hd / 2))[u8 * G + grp] = word;
  if (u8 == 0) c.scale[(r * 2 + kv) * G + grp] = __halves2half2(a, z);
}

__global__ void __launch_bounds__(kThreads)
    kv4_read_kernel(KV4View c, const int64_t* __restrict__ slots, int T, bf16* __restrict__ k, bf16* __restrict__ v) {
  const int lanes = c.hd / 8, G = c.hd / 64;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t row = i / lanes;
  const int lane = (int)(i % lanes);
  if (row >= (int64_t)T * c.Hkv * 2) return;
  const int kv = (int)(row & 1);
  const int64_t th = row >> 1;  // token * Hkv + head
  const int h = (int)(th % c.Hkv);
  const int64_t slot = slots[th / c.Hkv];
  uint4 o = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot < c.n_pages * c.page) {
    const int64_t r = ((slot / c.page) * c.Hkv + h) * c.page + slot % c.page;
    const int grp = lane / 8, u8 = lane % 8;
    const uint32_t w = reinterpret_cast<const uint32_t*>((kv ? c.v : c.k) + r * (c.hd / 2))[u8 * G + grp];
    const float2 az = __half22float2(c.scale[(r * 2 + kv) * G + grp]);
    float x[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = fmaf((float)((w >> (4 * q)) & 15u), az.x, az.y);
    o = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
  *reinterpret_cast<uint4*>((kv ? v : k) + th * c.hd + lane * 8) = o;
}

int blocks(int64_t n) {
  const int64_t b = (n + kThreads - 1) / kThreads;
  MESHY_CHECK(b <= 0x7fffffff, "kv4: too many rows for one launch");
  return (int)b;
}

}  // namespace

void kv4_write(const bf16* k, int64_t ks, int64_t kh, const bf16* v, int64_t vs, int64_t vh, const int64_t* slots,
               int T, KV4View c, cudaStream_t st) {
  if (T == 0) return;
  kv4_write_kernel<<<blocks((int64_t)T * c.Hkv * 2 * (c.hd / 8)), kThreads, 0, st>>>(k, ks, kh, v, vs, vh, slots, T, c);
  MESHY_CUDA_CHECK(cudaGetLastError());
}

void kv4_read(KV4View c, const int64_t* slots, int T, bf16* k, bf16* v, cudaStream_t st) {
  if (T == 0) return;
  kv4_read_kernel<<<blocks((int64_t)T * c.Hkv * 2 * (c.hd / 8)), kThreads, 0, st>>>(c, slots, T, k, v);
  MESHY_CUDA_CHECK(cudaGetLastError());
}

}  // namespace meshy
