// Block tables and slot maps of a paged KV cache, made on the device from request lengths (paging.cu).
#pragma once
#include "../include/common.cuh"

namespace meshy {

// Row rows[i] of the table bt [R, M] (row stride bt_stride) gets the next max(0, need[i] - have[i]) of the P pages at
// columns have[i] ..; rows and columns outside the table are not written.
void assign_pages(int* bt, int64_t bt_stride, int R, int M, const int* rows, const int* have, const int* need, int n,
                  const int* pages, int P, cudaStream_t st);
// Tokens start[i] .. start[i] + lens[i] - 1 of each row rows[i], packed: positions and slots [total], cu [n + 1].
// Entries behind the last token: position 0, slot -1.
void token_maps(const int* bt, int64_t bt_stride, int R, int M, const int* rows, const int* start, const int* lens,
                int n, int page, int* positions, int64_t* slots, int* cu, int total, cudaStream_t st);

}  // namespace meshy
