// 8-bit KV cache: quantising write and read-back (layout in kv8.h).
//
// A block of 16 tokens of one head is kept as n = rint(x r) in [-127, 127], r the largest number of 8 significant bits
// that is not above 127 / max|x|; the cache holds n + 128 and a = fp32(1 / r). Eight bits for r cost less than 2^-7 of a
// step, and make every decision exact: a bf16 channel times r has 16 significant bits, so one fused multiply-add rounds
// it to a whole number (halves to even) without a rounding before, and the bytes are the same wherever the format is
// computed. 1 / a rounded to 8 bits is r again.
//
// A write that holds a block's first token starts the block anew. Any other takes r' = min(r, r of its own rows); where
// that is below r, the other tokens of the block are requantised, rint(n r' / r): n r' is exact, and no quotient of it
// by r lies so near a half that fp32's rounding could move it there. A token that is written again changes nothing.
//
// A warp owns a block's rows: runs of neighbouring rows of the call whose slots lie in one block. Magnitudes are taken
// in [2^-100, 2^126]; a NaN gives the block the scale NaN (and its new rows the byte 128).
#include <cuda_runtime.h>

#include "../include/fastdiv.cuh"
#include "kv8.h"

namespace meshy {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int B = kKV8Block;
constexpr float kLeast = 7.8886090522101181e-31f;  // 2^-100
constexpr float kMost = 8.5070591730234616e+37f;   // 2^126

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 b) { return *reinterpret_cast<uint32_t*>(&b); }

// Row of head 0 of a slot, counted over (page, head, place); -1: outside.
__device__ __forceinline__ int64_t row_of(const KV8View& c, FastDiv page, int64_t slot) {
  const int64_t n = c.n_pages * c.page;
  if (slot < 0 || slot >= n) return -1;
  const int64_t p = n < (1LL << 31) ? (int64_t)page.div((uint32_t)slot) : slot / c.page;
  return p * c.Hkv * c.page + (slot - p * c.page);
}

// Steps per unit of a block whose largest magnitude is m.
__device__ __forceinline__ float steps(float m) {
  if (m != m) return m;
  const float q = __fdiv_rn(127.f, fminf(fmaxf(m, kLeast), kMost));
  return __uint_as_float(__float_as_uint(q) & 0xFFFF0000u);  // eight significant bits, towards zero
}

// rint(x r) + 128 in the low byte: 1.5 2^23 leaves no bits behind the point.
__device__ __forceinline__ uint32_t level(float x, float r) { return __float_as_uint(fmaf(x, r, 12582912.f + 128.f)); }

__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Eight bytes to bf16 values.
__device__ __forceinline__ uint4 restore(uint2 w, float a) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = __byte_perm(i < 4 ? w.x : w.y, 0x4B000000u, 0x7440 | (i % 4));  // 2^23 + u
    x[i] = (__uint_as_float(u) - (8388608.f + 128.f)) * a;
  }
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

struct WriteArgs {
  const bf16* x[2];  // K and V
  int64_t xs[2], xh[2];
  const int64_t* slots;
  int T, tile;       // rows of the call; rows that a CTA looks at
  KV8View c;
  FastDiv page;
  bf16* out[2];
};

// Rows t0 .. t0 + m of the call, all of one block: head h of K (kv = 0) or V.
template <int HD>
__device__ __forceinline__ void write_run(const WriteArgs& a, int t0, int m, int h, int kv, int lane, int64_t slot) {
  constexpr int L = HD / 8, N = B * L / 32, STEP = 32 / L;  // lanes of a row, rows of a lane, rows side by side
  const int ch = lane % L * 8, r0 = lane / L;
  const bf16* x = (kv ? a.x[1] + t0 * a.xs[1] + h * a.xh[1] : a.x[0] + t0 * a.xs[0] + h * a.xh[0]) + ch;
  const int64_t xs = kv ? a.xs[1] : a.xs[0];
  const int64_t row = __shfl_sync(0xffffffffu, row_of(a.c, a.page, slot), 0);  // lane i has row i's slot
  bf16* out = kv ? a.out[1] : a.out[0];
  if (out) out += ((int64_t)t0 * a.c.Hkv + h) * HD + ch;
  const int64_t os = (int64_t)a.c.Hkv * HD;
  if (row < 0) {  // a slot outside the cache is a run of its own
    if (out && r0 == 0) *reinterpret_cast<uint4*>(out) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int place = (int)(slot % B);  // of row ``lane``
  const int64_t first = row - __shfl_sync(0xffffffffu, place, 0) + (int64_t)h * a.c.page;  // the block's first row
  uint8_t* data = (kv ? a.c.v : a.c.k) + first * HD + ch;
  float* scale = a.c.scale + first / B * 2 + kv;
  const float old = *scale;
  uint4 u[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    u[j] = make_uint4(0, 0, 0, 0);
    if (r0 + j * STEP < m) u[j] = *reinterpret_cast<const uint4*>(x + (r0 + j * STEP) * xs);
  }
  const uint32_t held = __reduce_or_sync(0xffffffffu, lane < m ? 1u << place : 0u);
  // the largest magnitude, in bf16, where it is exact; a NaN stays one
  __nv_bfloat162 top = as_bf162(0u);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    top = __hmax2_nan(top, __hmax2_nan(__habs2(as_bf162(u[j].x)), __habs2(as_bf162(u[j].y))));
    top = __hmax2_nan(top, __hmax2_nan(__habs2(as_bf162(u[j].z)), __habs2(as_bf162(u[j].w))));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = __hmax2_nan(top, as_bf162(__shfl_xor_sync(0xffffffffu, as_u32(top), o)));
  const float t0f = __low2float(top), t1f = __high2float(top);
  const float most = t0f != t0f ? t0f : t1f != t1f ? t1f : fmaxf(t0f, t1f);
  float r = steps(most);
  if (!(held & 1u)) {
    const float r_old = old > 0.f || old != old ? __bfloat162float(__float2bfloat16_rn(__fdiv_rn(1.f, old))) : INFINITY;
    if (r_old != r_old) r = r_old;
    if (r < r_old) {  // requantise the block's other rows
#pragma unroll 1
      for (int p = r0; p < B; p += STEP) {
        if (held >> p & 1u) continue;
        uint2 w = *reinterpret_cast<const uint2*>(data + p * HD);
        uint32_t y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float n = (float)(int)((i < 4 ? w.x : w.y) >> (8 * (i % 4)) & 255u) - 128.f;
          y[i] = level(__fdiv_rn(n * r, r_old), 1.f);
        }
        *reinterpret_cast<uint2*>(data + p * HD) =
            make_uint2(low_bytes(y[0], y[1], y[2], y[3]), low_bytes(y[4], y[5], y[6], y[7]));
      }
    } else if (r >= r_old) {
      r = r_old;
    }
  }
  const float back = __fdiv_rn(1.f, r);
  if (lane == 0) *scale = back;
  const bool far = !(most <= kMost) || r != r;
  if (far && r != r) r = 0.f;  // nothing of a block with a NaN is kept: 128 throughout
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int p = __shfl_sync(0xffffffffu, place, (r0 + j * STEP) % 32);
    if (r0 + j * STEP >= m) continue;
    const uint32_t us[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
    uint32_t y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 f = unpack_bf16x2(us[i]);
      if (far) {
        f.x = fminf(fmaxf(f.x, -kMost), kMost);
        f.y = fminf(fmaxf(f.y, -kMost), kMost);
      }
      y[2 * i] = level(f.x, r);
      y[2 * i + 1] = level(f.y, r);
    }
    const uint2 w = make_uint2(low_bytes(y[0], y[1], y[2], y[3]), low_bytes(y[4], y[5], y[6], y[7]));
    *reinterpret_cast<uint2*>(data + p * HD) = w;
    if (out) *reinterpret_cast<uint4*>(out + (r0 + j * STEP) * os) = restore(w, back);
  }
}

// Block of row t's slot; rows outside the call and slots outside the cache: below zero.
__device__ __forceinline__ int64_t block_of(const WriteArgs& a, int64_t t) {
  if (t < 0 || t >= a.T) return -2;
  const int64_t s = a.slots[t];
  return s < 0 || s >= a.c.n_pages * a.c.page ? -1 : s / B;
}

// A row begins a run unless the row before it has its block; so does one whose block the row 16 before it has too (a
// slot given more than once, as idle rows give the trash page's: no run is longer than a block).
__device__ __forceinline__ bool begins(const WriteArgs& a, int64_t t, int64_t block) {
  return block < 0 || block != block_of(a, t - 1) || block == block_of(a, t - B);
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 4) kv8_write_kernel(const WriteArgs a) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  pdl_wait();
  pdl_trigger();
  const int t0 = blockIdx.x * a.tile;
  // the runs that begin among this CTA's rows
  const int64_t mine = lane < a.tile ? block_of(a, t0 + lane) : -2;
  uint32_t starts = __ballot_sync(0xffffffffu, mine > -2 && begins(a, t0 + lane, mine));
  const int items = 2 * a.c.Hkv;
  // warp w of the grid's row takes every so manieth (head, K or V), run by run
  const int step = gridDim.y * kWarps;
  int item = blockIdx.y * kWarps + warp;
  while (starts) {
    const int t = t0 + __ffs(starts) - 1;
    starts &= starts - 1;
    const int64_t block = block_of(a, t), here = lane < B ? block_of(a, t + lane) : -2;
    const bool in = here == block && (lane == 0 || !begins(a, t + lane, here));
    const int m = __ffs(~__ballot_sync(0xffffffffu, in)) - 1;
    const int64_t slot = lane < m ? a.slots[t + lane] : -1;
    for (; item < items; item += step) write_run<HD>(a, t, m, item / 2, item % 2, lane, slot);
    item -= items;
  }
}

// Lanes of 8 channels; a lane reads its bytes of K and of V of NH heads of a token.
template <int HD, int NH>
__global__ void __launch_bounds__(kThreads)
    kv8_read_kernel(KV8View c, const int64_t* __restrict__ slots, uint32_t items, bf16* __restrict__ k,
                    bf16* __restrict__ v, FastDiv splits, FastDiv page) {
  constexpr int L = HD / 8;
  const uint32_t lane = threadIdx.x % L, i = blockIdx.x * (kThreads / L) + threadIdx.x / L;
  pdl_wait();
  pdl_trigger();
  if (i >= items) return;
  const uint32_t t = splits.div(i);
  const int h0 = (i - t * splits.d) * NH;
  const int64_t r = row_of(c, page, slots[t]);
  uint2 wk[NH], wv[NH];
  float2 a[NH];
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    wk[j] = wv[j] = make_uint2(0u, 0u);
    a[j] = make_float2(0.f, 0.f);
    if (r < 0 || h0 + j >= c.Hkv) continue;
    const int64_t row = r + (int64_t)(h0 + j) * c.page;
    wk[j] = *reinterpret_cast<const uint2*>(c.k + row * HD + lane * 8);
    wv[j] = *reinterpret_cast<const uint2*>(c.v + row * HD + lane * 8);
    a[j] = *reinterpret_cast<const float2*>(c.scale + row / B * 2);
  }
  const int64_t o = ((int64_t)t * c.Hkv + h0) * HD + lane * 8;
#pragma unroll
  for (int j = 0; j < NH; ++j) {
    if (h0 + j >= c.Hkv) break;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(k + o + j * HD) = r < 0 ? zero : restore(wk[j], a[j].x);
    *reinterpret_cast<uint4*>(v + o + j * HD) = r < 0 ? zero : restore(wv[j], a[j].y);
  }
}

}  // namespace

void kv8_write(const bf16* k, int64_t ks, int64_t kh, const bf16* v, int64_t vs, int64_t vh, const int64_t* slots,
               int T, KV8View c, bf16* ko, bf16* vo, cudaStream_t st) {
  if (T == 0) return;
  const int items = 2 * c.Hkv, groups = (items + kWarps - 1) / kWarps;
  // Few rows: a CTA to each, or more, for the latency; many: 16 rows to a CTA, whose warps take the heads of their one or
  // two blocks (32768 tokens of 8 heads: 62.5 us, with 8 rows 65.9, with 32 65.3).
  const bool few = (int64_t)T * items <= 8192;
  const int tile = few ? 1 : 16;
  const WriteArgs a{{k, v}, {ks, vs}, {kh, vh}, slots, T, tile, c, FastDiv(c.page), {ko, vo}};
  const dim3 grid((T + tile - 1) / tile, few ? groups : 1);
  launch_pdl(c.hd == 128 ? kv8_write_kernel<128> : kv8_write_kernel<64>, grid, dim3(kThreads), 0, st, a);
}

void kv8_read(KV8View c, const int64_t* slots, int T, bf16* k, bf16* v, cudaStream_t st) {
  if (T == 0) return;
  auto go = [&](auto kernel, int nh) {
    const int64_t splits = (c.Hkv + nh - 1) / nh, items = T * splits, per = kThreads / (c.hd / 8);
    MESHY_CHECK(items < (1LL << 31), "kv8: too many rows for one call");
    launch_pdl(kernel, dim3((unsigned)((items + per - 1) / per)), dim3(kThreads), 0, st, c, slots, (uint32_t)items, k, v,
               FastDiv((uint32_t)splits), FastDiv(c.page));
  };
  const bool many = (int64_t)T * c.Hkv >= 1 << 16;
  if (c.hd == 128)
    many ? go(kv8_read_kernel<128, 4>, 4) : go(kv8_read_kernel<128, 1>, 1);
  else
    many ? go(kv8_read_kernel<64, 4>, 4) : go(kv8_read_kernel<64, 1>, 1);
}

}  // namespace meshy
