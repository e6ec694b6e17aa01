// Rotary positions of a fused QKV projection in any layout and scaling, with QK-norm, and their gradient (rotary.cu).
#pragma once
#include "../include/common.cuh"

namespace meshy {

struct RotaryShape {
  int T, Hq, Hkv, hd;
  int rot;           // rotated channels, the first of a head
  bool interleaved;  // pairs (2 i, 2 i + 1); else (i, i + rot / 2)
};

// A paged cache as a destination of K and V: [pages, Hkv, page, hd], slots [T]; slots outside it are skipped.
struct RotaryCache {
  bf16* k;
  bf16* v;
  const int64_t* slots;
  int64_t n_pages;
  int page;
};

// qkv [T, (Hq + 2 Hkv) hd] (row stride qs) to q, k, v [T, H, hd]; qn, kn [hd] norm weights or null. turns [rot / 2]:
// 2^64 times the turns per position of each pair. The rotated channels are multiplied by ``factor``. k and v may be
// null where ``cache`` takes them.
void rotary_fwd(RotaryShape s, const bf16* qkv, int64_t qs, const int* pos, const uint64_t* turns, float factor,
                const bf16* qn, const bf16* kn, float eps, bf16* q, bf16* k, bf16* v, RotaryCache cache,
                cudaStream_t st);
// Where the gradient of a norm's weights goes: added to fp32, or written in bf16.
struct RotaryWeightGrad {
  float* add;
  bf16* out;
};
// Both are added to the same memory (one weight for queries and keys): that takes a launch for each.
bool rotary_shared_grad(RotaryWeightGrad wq, RotaryWeightGrad wk, int hd);
// gq, gk, gv [T, H, hd] to gqkv [T, (Hq + 2 Hkv) hd]; with norms, the weights' gradients to wq and wk, and ``part`` holds
// rotary_part_floats() floats.
void rotary_bwd(RotaryShape s, const bf16* qkv, int64_t qs, const int* pos, const uint64_t* turns, float factor,
                const bf16* qn, const bf16* kn, float eps, const bf16* gq, const bf16* gk, const bf16* gv, bf16* gqkv,
                RotaryWeightGrad wq, RotaryWeightGrad wk, float* part, cudaStream_t st);
int64_t rotary_part_floats(RotaryShape s);

}  // namespace meshy
