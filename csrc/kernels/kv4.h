// Paged KV cache held in 4 bits (kv4.cu: write and read-back; kv4_attn.cu: decode attention).
//
// One row is one head of one token: ``hd`` channels (64 or 128) in G = hd / 64 groups of 64 neighbours. A group
// keeps a scale ``a`` and a base ``z`` in fp16 and one nibble per channel; nibble n stands for a n + z.
//   k, v   [pages, Hkv, page, hd / 2] bytes. The 32-bit word w of a row holds channels
//          64 (w mod G) + 8 (w div G) + 0..7, the lowest channel in the lowest nibble. Any 8-byte block of a
//          128-channel row (16 bytes for K) therefore holds the same number of channels of both groups, which is
//          what one lane of the attention kernel's matrix fragments needs.
//   scale  [pages, Hkv, page, 2 (k, v), G, 2 (a, z)] fp16
#pragma once
#include <cuda_fp16.h>

#include "../include/common.cuh"

namespace meshy {

struct KV4View {
  uint8_t* k;
  uint8_t* v;
  __half2* scale;
  int64_t n_pages;
  int Hkv, page, hd;
};

// Quantise rows k, v [T, Hkv, hd] bf16 (element strides ks / vs between tokens, kh / vh between heads; inner
// stride 1) into the cache at slots [T] (page * page_size + offset). Slots outside the cache are skipped.
void kv4_write(const bf16* k, int64_t ks, int64_t kh, const bf16* v, int64_t vs, int64_t vh, const int64_t* slots,
               int T, KV4View c, cudaStream_t st);
// The bf16 values the cache stands for at ``slots``: k, v [T, Hkv, hd] contiguous (zero for a slot outside it).
void kv4_read(KV4View c, const int64_t* slots, int T, bf16* k, bf16* v, cudaStream_t st);
// Decode attention of q [B, Hq, hd] (strides qs between rows, qh between heads) over each row's first
// seq_lens[b] tokens, whose pages are bt[b, :]; a row of length 0 gives zeros. A bounded wait inside the kernel that
// gives up (after ``wait`` cycles; below zero: the usual limit) records its code in ``err``; the result is then undefined. ``part`` holds kv4_part_floats(hd) floats, ``arrived``
// kv4_attention_segments() counters that are zero between launches; launches that may run at the same time need
// workspaces of their own.
int kv4_attention_ctas();
int64_t kv4_attention_segments(int B, int Hq, int Hkv);
inline int64_t kv4_part_floats(int hd) { return (int64_t)2 * kv4_attention_ctas() * 8 * (hd + 4); }
void kv4_attention(const bf16* q, int64_t qs, int64_t qh, KV4View c, const int* bt, int64_t bt_stride, int max_pages,
                   const int* seq_lens, int B, int Hq, float scale, bf16* out, float* part, unsigned* arrived, int* err,
                   int64_t wait, cudaStream_t st);

}  // namespace meshy
