// Reciprocals and quotients in fp32.
#pragma once

namespace meshy {

__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Correctly rounded x / y from y's correctly rounded reciprocal: one Newton step on the quotient with the exact
// remainder (Markstein, 1990).
__device__ __forceinline__ float quotient(float x, float y, float rcp) {
  const float q = x * rcp;
  return fmaf(fmaf(-q, y, x), rcp, q);
}

}  // namespace meshy
