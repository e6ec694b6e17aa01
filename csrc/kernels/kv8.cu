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
// by r lies so near a half that fp32's rounding could move it there. A token that is written again changes nothing. Each such
// growth adds up to half a step of the new scale to the other tokens' errors: (1 + g) / 2 steps at most after g of them.
//
// A warp owns a block's rows: runs of neighbouring rows of the call whose slots lie in one block. Magnitudes are taken
// in [2^-100, 2^126]; a NaN gives the block the scale NaN (and its new rows the byte 128).
//
// Measured: a prompt of 32768 tokens (8 heads, 128 wide) 61 us, 5.6 TB/s of the 340 MB that the call moves: memory, with
// 64 % of the issue slots busy (rounding and packing, about two instructions a channel). 64 rows of a decode step 2.1-2.4
// us (2 heads), with cold caches 4: a launch, the slots, the block's scale and rows, the stores. The read-back of 16384
// tokens 14.4 us; of 64 1.5 us.
#include <cuda_runtime.h>

#include "../include/fastdiv.cuh"
#include "../include/quotient.cuh"
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

// 1 / r, correctly rounded for numbers of eight significant bits: the hardware's approximation and one Newton step.
__device__ __forceinline__ float reciprocal(float r) {
  const float y = rcp_approx(r);
  return fmaf(fmaf(-r, y, 1.f), y, y);
}

// Steps per unit of a block whose largest magnitude is m, a bf16 number: eight significant bits, towards zero. No quotient
// of 127 by such a number lies within 2^-16 below one of eight bits, so an approximation moved up by 2^-20 is cut to the
// same one.
__device__ __forceinline__ float steps(float m) {
  if (m != m) return m;
  const float q = 127.f * rcp_approx(fminf(fmaxf(m, kLeast), kMost)) * 1.00000095367431640625f;
  return __uint_as_float(__float_as_uint(q) & 0xFFFF0000u);
}

// rint(x r) + 128 in the low byte: 1.5 2^23 leaves no bits behind the point.
__device__ __forceinline__ uint32_t level(float x, float r) { return __float_as_uint(fmaf(x, r, 12582912.f + 128.f)); }

__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// n of byte i of a word: u as 2^23 + u, less 2^23 + 128.
__device__ __forceinline__ float number(uint32_t w, int i) {
  return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 | i)) - (8388608.f + 128.f);
}

// Eight bytes to bf16 values.
__device__ __forceinline__ uint4 restore(uint2 w, float a) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = number(i < 4 ? w.x : w.y, i % 4) * a;
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

struct WriteArgs {
  const bf16* x[2];  // K and V
  int64_t xs[2], xh[2];
  const int64_t* slots;
  int T;  // rows of the call
  KV8View c;
  FastDiv page;
  bf16* out[2];
};

// This lane's channels of row t of the call (the first lanes' of a warp), head h of K (kv = 0) or V.
template <int HD>
__device__ __forceinline__ const bf16* row_at(const WriteArgs& a, int64_t t, int h, int kv, int lane) {
  return (kv ? a.x[1] + t * a.xs[1] + h * a.xh[1] : a.x[0] + t * a.xs[0] + h * a.xh[0]) + lane % (HD / 8) * 8;
}

// Rows t0 .. t0 + m of the call, all of one block: head h of K (kv = 0) or V. ``row0``: the first of them, if HAVE.
template <int HD, bool HAVE>
__device__ __forceinline__ void write_run(const WriteArgs& a, int t0, int m, int h, int kv, int lane, int64_t slot,
                                          const uint4& row0) {
  constexpr int L = HD / 8, N = B * L / 32, STEP = 32 / L;  // lanes of a row, rows of a lane, rows side by side
  const int ch = lane % L * 8, r0 = lane / L;
  const bf16* x = row_at<HD>(a, t0, h, kv, lane);
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
  const uint32_t held = __reduce_or_sync(0xffffffffu, lane < m ? 1u << place : 0u);
  const bool anew = held & 1u;
  uint2 was[N];  // the block's rows as they are: a token in three makes its block's scale larger
  if (HAVE && !anew) {
#pragma unroll
    for (int j = 0; j < N; ++j) was[j] = *reinterpret_cast<const uint2*>(data + (r0 + j * STEP) * HD);
  }
  uint4 u[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    u[j] = make_uint4(0, 0, 0, 0);
    if (HAVE && j == 0 && r0 == 0)
      u[j] = row0;
    else if (r0 + j * STEP < m)
      u[j] = *reinterpret_cast<const uint4*>(x + (r0 + j * STEP) * xs);
  }
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
  if (!anew) {
    const float r_old = old > 0.f || old != old ? __bfloat162float(__float2bfloat16_rn(rcp_approx(old))) : INFINITY;
    if (r_old != r_old) r = r_old;
    if (r < r_old) {  // requantise the block's other rows
      if (!HAVE) {
#pragma unroll
        for (int j = 0; j < N; ++j) was[j] = *reinterpret_cast<const uint2*>(data + (r0 + j * STEP) * HD);
      }
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (held >> (r0 + j * STEP) & 1u) continue;
        uint32_t y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float n = number(i < 4 ? was[j].x : was[j].y, i % 4);
          y[i] = level(old > 0.f ? quotient(n * r, r_old, old) : 0.f, 1.f);
        }
        *reinterpret_cast<uint2*>(data + (r0 + j * STEP) * HD) =
            make_uint2(low_bytes(y[0], y[1], y[2], y[3]), low_bytes(y[4], y[5], y[6], y[7]));
      }
    } else if (r >= r_old) {
      r = r_old;
    }
  }
  const float back = reciprocal(r);
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

// A run begins at a row unless the row before it has its block, and at a row whose block the row 16 before it has too (a
// slot given more than once, as idle rows give the trash page's: no run is longer than a block; warps then write one block
// at once, and what it holds is nobody's). A slot outside the cache is a run of its own.
//
// A CTA writes the runs that begin among its TILE rows, 16 at most. With one row, the call's few, latency is what counts:
// its channels are asked for before the slots are known, and the block's other rows before they are known to be needed (64
// rows whose blocks are requantised 2.4 us, 3.3 without; 4 and 13 with cold caches).
template <int HD, int TILE>
__global__ void __launch_bounds__(kThreads, TILE == 1 ? 2 : 4) kv8_write_kernel(const WriteArgs a) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  pdl_wait();
  pdl_trigger();
  const int64_t t0 = (int64_t)blockIdx.x * TILE, n = a.c.n_pages * a.c.page;
  const int items = 2 * a.c.Hkv, step = gridDim.y * kWarps;
  int item = blockIdx.y * kWarps + warp;  // warps take the (head, K or V) of all runs in turn
  uint4 row0 = make_uint4(0, 0, 0, 0);
  if (TILE == 1 && item < items && lane < HD / 8)
    row0 = *reinterpret_cast<const uint4*>(row_at<HD>(a, t0, item / 2, item % 2, lane));
  // slots of rows t0 - 16 + lane and t0 + 16 + lane, and their blocks (outside the cache -1, outside the call -2)
  const int64_t ta = t0 - B + lane, tb = t0 + B + lane;
  const int64_t sa = ta >= 0 && ta < a.T ? a.slots[ta] : -1, sb = tb < a.T ? a.slots[tb] : -1;
  auto block_of = [&](int64_t t, int64_t s) { return t < 0 || t >= a.T ? -2 : s < 0 || s >= n ? -1 : s / B; };
  const int64_t ba = block_of(ta, sa), bb = block_of(tb, sb);
  const int64_t last = __shfl_sync(0xffffffffu, ba, 31), low = __shfl_sync(0xffffffffu, ba, lane % 16 + 16);
  int64_t pa = __shfl_up_sync(0xffffffffu, ba, 1), pb = __shfl_up_sync(0xffffffffu, bb, 1);
  if (lane == 0) pb = last;
  const int64_t first = __shfl_sync(0xffffffffu, ba, lane % 16);  // 16 rows before lane's in the upper half
  const uint32_t begin_a = __ballot_sync(0xffffffffu, ba < 0 || ba != pa || ba == first) >> 16;
  const uint32_t begin_b = __ballot_sync(0xffffffffu, bb < 0 || bb != pb || bb == low) & 0x7FFFu;
  const uint32_t begins = begin_a | begin_b << 16;  // bit r: row t0 + r
  uint32_t starts = begins & (__ballot_sync(0xffffffffu, ba != -2) >> 16) & ((1u << TILE) - 1u);
  while (starts) {
    const int i = __ffs(starts) - 1;
    starts &= starts - 1;
    const uint32_t later = begins >> i >> 1;
    const int m = later ? __ffs(later) : B, at = B + i + lane;  // of the 48 slots at hand
    const int64_t x = __shfl_sync(0xffffffffu, sa, at % 32), y = __shfl_sync(0xffffffffu, sb, at % 32);
    const int64_t slot = lane < m ? (at < 32 ? x : y) : -1;
    for (; item < items; item += step)
      write_run<HD, TILE == 1>(a, (int)t0 + i, m, item / 2, item % 2, lane, slot, row0);
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
  // Few rows: a CTA to each, or more, for the latency. More: 16 rows to a CTA (32768 tokens of 8 heads 62.5 us, with 8 rows
  // 65.9, with 32 65.3), whose warps take the heads of its runs in turn, and as many CTAs to those as make kCtas of
  // them. (us, first a prompt, then a row to a block, as in decoding; 8 heads: 256 rows 4.2, 5.2, by the other rule 3.5,
  // 7.6; 512 rows 4.3, 10.7, by the other 5.6, 10.2, with one CTA to the runs 5.2, 48; 2 heads: 512 rows 3.4, 4.6, by the
  // other 3.1, 6.0; 1024 rows 3.4, 7.6, by the other 4.7, 8.4, with one CTA to the runs 2.9, 15.)
  constexpr int kCtas = 296;
  const bool few = (int64_t)T * groups <= 512;
  const WriteArgs a{{k, v}, {ks, vs}, {kh, vh}, slots, T, c, FastDiv(c.page), {ko, vo}};
  const int tiles = (T + B - 1) / B;
  const dim3 grid = few ? dim3(T, groups) : dim3(tiles, std::max(1, std::min(kCtas / tiles, B * items / kWarps)));
  auto* kernel = c.hd == 128 ? (few ? kv8_write_kernel<128, 1> : kv8_write_kernel<128, B>)
                             : (few ? kv8_write_kernel<64, 1> : kv8_write_kernel<64, B>);
  launch_pdl(kernel, grid, dim3(kThreads), 0, st, a);
}

void kv8_read(KV8View c, const int64_t* slots, int T, bf16* k, bf16* v, cudaStream_t st) {
  if (T == 0) return;
  auto go = [&](auto kernel, int nh) {
    const int64_t splits = (c.Hkv + nh - 1) / nh, items = T * splits, per = kThreads / (c.hd / 8);
    MESHY_CHECK(items < (1LL << 31), "kv8: too many rows for one call");
    launch_pdl(kernel, dim3((unsigned)((items + per - 1) / per)), dim3(kThreads), 0, st, c, slots, (uint32_t)items, k, v,
               FastDiv((uint32_t)splits), FastDiv(c.page));
  };
  // four heads to a lane where there is work for all (8 heads: 512 tokens 2.0 us, one to a lane 1.8; 1024 2.1, 2.6; 16384
  // 14.4, 18.6)
  const bool many = (int64_t)T * c.Hkv >= 8192;
  if (c.hd == 128)
    many ? go(kv8_read_kernel<128, 4>, 4) : go(kv8_read_kernel<128, 1>, 1);
  else
    many ? go(kv8_read_kernel<64, 4>, 4) : go(kv8_read_kernel<64, 1>, 1);
}

}  // namespace meshy
