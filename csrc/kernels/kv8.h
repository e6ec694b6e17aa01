// Paged KV cache held in 8 bits (kv8.cu: write and read-back; kv8_attn.cu: decode attention).
//
// One row is one head of one token: ``hd`` channels (64 or 128), a byte each. The 16 tokens of a block (slots 16 i ..
// 16 i + 15) share one scale per head, for K and for V:
//   k, v   [pages, Hkv, page, hd] bytes, byte u stands for a (u - 128)
//   scale  [pages, Hkv, page / 16, 2 (k, v)] fp32, a
// a = fp32(1 / r), r the largest number of 8 significant bits that is not above 127 / max|x| over the block.
#pragma once
#include "../include/common.cuh"

namespace meshy {

constexpr int kKV8Block = 16;

struct KV8View {
  uint8_t* k;
  uint8_t* v;
  float* scale;
  int64_t n_pages;
  int Hkv, page, hd;
};

// Quantise rows k, v [T, Hkv, hd] bf16 (element strides ks / vs between tokens, kh / vh between heads; inner stride 1,
// 16-byte aligned rows) into the cache at slots [T] (page * page_size + offset); rows of one block stand together,
// each slot once (a block for which that does not hold is left undefined). Slots outside the cache are skipped.
// ko, vo [T, Hkv, hd]: the values now held (zeros for a slot outside), or null.
void kv8_write(const bf16* k, int64_t ks, int64_t kh, const bf16* v, int64_t vs, int64_t vh, const int64_t* slots,
               int T, KV8View c, bf16* ko, bf16* vo, cudaStream_t st);
// The bf16 values the cache stands for at ``slots``: k, v [T, Hkv, hd] contiguous (zero for a slot outside it).
void kv8_read(KV8View c, const int64_t* slots, int T, bf16* k, bf16* v, cudaStream_t st);
// Decode attention of q [B, Hq, hd] (strides qs between rows, qh between heads) over each row's first seq_lens[b]
// tokens, whose pages are bt[b, :]; a row of length 0 gives zeros. A bounded wait inside the kernel that gives up (after
// ``wait`` cycles; below zero: the usual limit) records its code in ``err``; the result is then undefined. ``part`` holds kv8_part_floats() floats, ``arrived`` kv8_attention_segments() counters that are
// zero between launches; launches that may run at the same time need workspaces of their own.
int64_t kv8_attention_segments(int B, int Hq, int Hkv);
int64_t kv8_part_floats();
void kv8_attention(const bf16* q, int64_t qs, int64_t qh, KV8View c, const int* bt, int64_t bt_stride, int max_pages,
                   const int* seq_lens, int B, int Hq, float scale, bf16* out, float* part, unsigned* arrived, int* err,
                   int64_t wait, cudaStream_t st);

}  // namespace meshy
