// Hardware exp2 / reciprocal and fp32 arithmetic on two values at once (sm_100a's f32x2 forms, which take
// and give aligned register pairs: neighbouring elements of a vector load or of an accumulator).
#pragma once
#include "common.cuh"

namespace ahb {

AHB_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

AHB_DEVICE float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats in one instruction (the two channels of a lane, or two columns of an accumulator row)
AHB_DEVICE float2 both(float x) { return make_float2(x, x); }
AHB_DEVICE float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
AHB_DEVICE float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
AHB_DEVICE float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
AHB_DEVICE float2 max2(float2 a, float b) { return make_float2(fmaxf(a.x, b), fmaxf(a.y, b)); }

}  // namespace ahb
