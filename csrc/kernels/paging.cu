// Block tables and slot maps from request lengths.
//
// Both kernels deal a packed list (pages, tokens) out to rows: entry j belongs to the row i with
// sum(c[:i]) <= j < sum(c[:i + 1]), c the rows' counts. Every CTA scans the counts itself, 256 rows at a time, and
// looks its own entries up in the scanned block by bisection: a few hundred rows are read in the time of one load from
// L2, so one launch does what a scan and a second kernel would. A chain bounds the pages, and the maps of few tokens: lengths,
// the scan, the bisection, the table's entry. Maps of many tokens are bound by instructions (58 % of the issue slots are busy:
// a scan in every CTA, eight steps of bisection on 64-bit ends for every four tokens). Measured: pages and maps of 16 rows
// 1.7 and 2.6 us, 4.3 together; of 256 rows and 1.1 M tokens 1.8 and 6.6, 8.8 together, of which the 14 MB take 2.2.
#include <climits>

#include <cuda_runtime.h>

#include "../include/fastdiv.cuh"
#include "paging.h"

namespace meshy {

namespace {

constexpr int kThreads = 256;
constexpr int kRows = 256;  // scanned at a time (1024: 11.0 us for the tables and maps of 1.1 M tokens of 256 rows, here 8.9)
constexpr int kPer = kRows / kThreads;

struct Scan {
  int64_t ends[kRows + 1];  // ends[i]: entries of the rows before row i of the block, and of all before the block
  int64_t sums[kThreads / 32];
  int rows[kRows], first[kRows];  // the table's row, and the page or token that the row's entries begin with
};

struct Row {
  int count, row, first;
};

// Rows b0 .. b0 + kRows (no entries behind n) into s, the ends from ``carry`` on; returns the new carry.
template <class Load>
__device__ __forceinline__ int64_t scan_rows(Scan& s, int b0, int n, int64_t carry, Load load) {
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  Row r[kPer];
  int64_t mine = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int row = b0 + tid * kPer + i;
    r[i] = row < n ? load(row) : Row{0, 0, 0};
    mine += r[i].count;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  __syncthreads();  // the block before has been used
  if (lane == 31) s.sums[warp] = incl;
  __syncthreads();
  int64_t at = carry + incl - mine;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) at += s.sums[w];
    carry += s.sums[w];
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    s.ends[tid * kPer + i] = at;
    s.rows[tid * kPer + i] = r[i].row;
    s.first[tid * kPer + i] = r[i].first;
    at += r[i].count;
  }
  if (tid == kThreads - 1) s.ends[kRows] = carry;
  __syncthreads();
  return carry;
}

// The row of the scanned block that entry j belongs to: the last i with ends[i] <= j (the rows behind it end later).
__device__ __forceinline__ int find(const Scan& s, int64_t j) {
  int lo = 0;
#pragma unroll
  for (int step = kRows / 2; step > 0; step >>= 1)
    if (s.ends[lo + step] <= j) lo += step;
  return lo;
}

__global__ void __launch_bounds__(kThreads)
    assign_pages_kernel(int* __restrict__ bt, int64_t bt_stride, int R, int M, const int* __restrict__ rows,
                        const int* __restrict__ have, const int* __restrict__ need, int n,
                        const int* __restrict__ pages, int P) {
  __shared__ Scan s;
  pdl_wait();
  pdl_trigger();
  const int64_t j = (int64_t)blockIdx.x * kThreads + threadIdx.x, last = min((int64_t)P, ((int64_t)blockIdx.x + 1) * kThreads);
  int64_t carry = 0;
  for (int b0 = 0; b0 < n && carry < last; b0 += kRows) {
    const int64_t begin = carry;
    carry = scan_rows(s, b0, n, carry, [&](int r) {
      const int h = max(have[r], 0);
      return Row{max(need[r], h) - h, rows[r], h};
    });
    if (j >= begin && j < carry && j < P) {
      const int i = find(s, j);
      const int row = s.rows[i];
      const int64_t col = s.first[i] + (j - s.ends[i]);
      if (row >= 0 && row < R && col < M) bt[row * bt_stride + col] = pages[j];
    }
  }
}

constexpr int kTok = 4;  // neighbouring tokens of a thread

__global__ void __launch_bounds__(kThreads)
    token_maps_kernel(const int* __restrict__ bt, int64_t bt_stride, int R, int M, const int* __restrict__ rows,
                      const int* __restrict__ start, const int* __restrict__ lens, int n, FastDiv page,
                      int* __restrict__ positions, int64_t* __restrict__ slots, int* __restrict__ cu, int total) {
  __shared__ Scan s;
  pdl_wait();
  pdl_trigger();
  const int64_t first = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * kTok;
  const int64_t last = min((int64_t)total, ((int64_t)blockIdx.x + 1) * (kThreads * kTok));
  int pos[kTok] = {0, 0, 0, 0};
  int64_t slot[kTok] = {-1, -1, -1, -1};
  int64_t carry = 0;
  for (int b0 = 0; b0 < n && (carry < last || blockIdx.x == 0); b0 += kRows) {
    const int64_t begin = carry;
    carry = scan_rows(s, b0, n, carry, [&](int r) { return Row{max(lens[r], 0), rows[r], start[r]}; });
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i <= min(kRows, n - b0); i += kThreads) cu[b0 + i] = (int)min(s.ends[i], (int64_t)INT_MAX);
    int i = -1, row = 0, col = -1, pg = -1;
    int64_t end = 0, off = 0;
#pragma unroll
    for (int x = 0; x < kTok; ++x) {
      const int64_t t = first + x;
      if (t < begin || t >= carry || t >= total) continue;
      if (i < 0 || t >= end) {
        i = find(s, t);
        end = s.ends[i + 1];
        row = s.rows[i];
        off = s.first[i] - s.ends[i];
        col = -1;
      }
      const int64_t p = off + t;
      pos[x] = (int)p;
      if (p < 0 || p > INT_MAX || row < 0 || row >= R) continue;
      const int c = (int)page.div((uint32_t)p);
      if (c != col) {
        col = c;
        pg = c < M ? bt[row * bt_stride + c] : -1;
      }
      if (pg >= 0) slot[x] = (int64_t)pg * page.d + (p - (int64_t)c * page.d);
    }
  }
  if (n == 0 && first == 0) cu[0] = 0;
  if (first + kTok <= total) {  // 16 bytes at a time: the outputs start on such boundaries
    *reinterpret_cast<int4*>(positions + first) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    *reinterpret_cast<longlong2*>(slots + first) = make_longlong2(slot[0], slot[1]);
    *reinterpret_cast<longlong2*>(slots + first + 2) = make_longlong2(slot[2], slot[3]);
  } else {
#pragma unroll
    for (int x = 0; x < kTok; ++x)
      if (first + x < total) {
        positions[first + x] = pos[x];
        slots[first + x] = slot[x];
      }
  }
}

}  // namespace

void assign_pages(int* bt, int64_t bt_stride, int R, int M, const int* rows, const int* have, const int* need, int n,
                  const int* pages, int P, cudaStream_t st) {
  if (n == 0 || P == 0) return;
  launch_pdl(assign_pages_kernel, dim3((unsigned)((P + (int64_t)kThreads - 1) / kThreads)), dim3(kThreads), 0, st, bt,
             bt_stride, R, M, rows, have, need, n, pages, P);
}

void token_maps(const int* bt, int64_t bt_stride, int R, int M, const int* rows, const int* start, const int* lens,
                int n, int page, int* positions, int64_t* slots, int* cu, int total, cudaStream_t st) {
  const int64_t per = kThreads * kTok;
  launch_pdl(token_maps_kernel, dim3((unsigned)std::max<int64_t>(1, (total + per - 1) / per)), dim3(kThreads), 0, st,
             bt, bt_stride, R, M, rows, start, lens, n, FastDiv(page), positions, slots, cu, total);
}

}  // namespace meshy
