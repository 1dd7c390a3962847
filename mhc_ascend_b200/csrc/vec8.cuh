// Eight consecutive values of a row as four pairs, for two-wide fp32 arithmetic.
#pragma once

#include "checkpoint8.cuh"

namespace mhc {

struct V8 {
  float2 a[4];
};
__device__ __forceinline__ V8 v8_zero() {
  V8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v.a[j] = make_float2(0.f, 0.f);
  return v;
}
__device__ __forceinline__ V8 v8_of(const uint4& u) {  // eight bf16 values
  const uint32_t r[4] = {u.x, u.y, u.z, u.w};
  V8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v.a[j] = make_float2(__uint_as_float(r[j] << 16), __uint_as_float(r[j] & 0xffff0000u));
  return v;
}
__device__ __forceinline__ uint4 v8_bf16(const V8& v) {
  uint32_t r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.a[j].x, v.a[j].y);
    r[j] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ void v8_spread(const V8& v, float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = v.a[j].x;
    f[2 * j + 1] = v.a[j].y;
  }
}
__device__ __forceinline__ V8 v8_gather(const float (&f)[8]) {
  V8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v.a[j] = make_float2(f[2 * j], f[2 * j + 1]);
  return v;
}

// A unit as it lies in memory
template <typename T> struct Raw8;
template <> struct Raw8<float> {
  float f[8];
  __device__ __forceinline__ void load(const float* p) { ck_load(p, f); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
  }
  __device__ __forceinline__ V8 values() const { return v8_gather(f); }
};
template <> struct Raw8<__nv_bfloat16> {
  uint4 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void zero() { u = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ V8 values() const { return v8_of(u); }
};
__device__ __forceinline__ void v8_save(float* p, const V8& v) {
  float f[8];
  v8_spread(v, f);
  ck_save(p, f);
}
__device__ __forceinline__ void v8_save(__nv_bfloat16* p, const V8& v) { *reinterpret_cast<uint4*>(p) = v8_bf16(v); }
// Store v and leave what was stored
__device__ __forceinline__ void v8_save_rounded(float* p, V8& v) { v8_save(p, v); }
__device__ __forceinline__ void v8_save_rounded(__nv_bfloat16* p, V8& v) {
  const uint4 u = v8_bf16(v);
  *reinterpret_cast<uint4*>(p) = u;
  v = v8_of(u);
}

// Rows of any width in the tensor's own groups of eight values (units): every access is
// aligned wherever a row starts, and a row's first and last unit may belong to its
// neighbours in part.  Unit of columns c .. c + 7 of a row of cols, c as low as -7:
__device__ __forceinline__ bool v8_edge(int c, int cols) { return c < 0 || c + 8 > cols; }
// its values outside the row as zeros
__device__ __forceinline__ V8 v8_inside(const V8& v, int c, int cols) {
  float f[8];
  v8_spread(v, f);
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = c + j >= 0 && c + j < cols ? f[j] : 0.f;
  return v8_gather(f);
}
// those inside to memory; what was stored stays in v, zeros outside
template <typename T>
__device__ __forceinline__ void v8_save_inside(T* p, V8& v, int c, int cols) {
  float f[8];
  v8_spread(v, f);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool in = c + j >= 0 && c + j < cols;
    if (in) {
      ck_store(p + j, f[j]);
      if (sizeof(T) == 2) f[j] = __bfloat162float(__float2bfloat16_rn(f[j]));
    } else {
      f[j] = 0.f;
    }
  }
  v = v8_gather(f);
}
// a unit of which the tensor has `left` values
template <typename T>
__device__ __forceinline__ V8 v8_load_part(const T* p, int64_t left) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = j < left ? ck_f32(p[j]) : 0.f;
  return v8_gather(f);
}
__device__ __forceinline__ V8 v8_weights_inside(const float* w, int c, int cols) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = c + j >= 0 && c + j < cols ? __ldg(w + c + j) : 0.f;
  return v8_gather(f);
}
// Eight weights, 32-byte aligned
__device__ __forceinline__ V8 v8_weights(const float* w) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(w)), b = __ldg(reinterpret_cast<const float4*>(w + 4));
  V8 v;
  v.a[0] = make_float2(a.x, a.y);
  v.a[1] = make_float2(a.z, a.w);
  v.a[2] = make_float2(b.x, b.y);
  v.a[3] = make_float2(b.z, b.w);
  return v;
}

__device__ __forceinline__ V8 v8_add(const V8& x, const V8& y) {
  V8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v.a[j] = __fadd2_rn(x.a[j], y.a[j]);
  return v;
}
__device__ __forceinline__ V8 v8_mul(const V8& x, const V8& y) {
  V8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v.a[j] = __fmul2_rn(x.a[j], y.a[j]);
  return v;
}
__device__ __forceinline__ V8 v8_scale(const V8& x, float s) {
  V8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v.a[j] = __fmul2_rn(x.a[j], make_float2(s, s));
  return v;
}
__device__ __forceinline__ V8 v8_fma(const V8& x, const V8& y, const V8& z) {
  V8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v.a[j] = __ffma2_rn(x.a[j], y.a[j], z.a[j]);
  return v;
}
__device__ __forceinline__ V8 v8_fma(const V8& x, float y, const V8& z) {
  V8 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) v.a[j] = __ffma2_rn(x.a[j], make_float2(y, y), z.a[j]);
  return v;
}
// r = sqrt(x) and its reciprocal as a sum ir + lo of two fp32 values (a Newton step each on
// the root and on the reciprocal; the residuals are exact in fused products).  v / r * w is
// then v c + v c', c + c' = w (ir + lo): one rounding that counts, in the five operations
// that v / r by a Newton step and its product with w take, which round twice.
struct Root {
  float r, ir, lo;
};
__device__ __forceinline__ Root root_of(double x) {
  const float hi = (float)x, r = sqrtf(hi), ir = 1.0f / r;
  const float rest = (fmaf(-r, r, hi) + (float)(x - (double)hi)) * (0.5f * ir);  // the root is r + rest
  const float lo = fmaf(-rest, ir, fmaf(-r, ir, 1.0f)) * ir;
  return {r, ir, r > 0.f && r <= 3.402823466e38f ? lo : 0.f};
}
__device__ __forceinline__ float normed(float v, float w, const Root& d) {
  const float c = w * d.ir;
  return fmaf(v, c, v * fmaf(w, d.lo, fmaf(w, d.ir, -c)));
}
__device__ __forceinline__ V8 v8_normed(const V8& v, const V8& w, const Root& d) {
  V8 y;
  const float2 ir = make_float2(d.ir, d.ir), lo = make_float2(d.lo, d.lo);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 c = __fmul2_rn(w.a[j], ir);
    const float2 rest = __ffma2_rn(w.a[j], lo, __ffma2_rn(w.a[j], ir, make_float2(-c.x, -c.y)));
    y.a[j] = __ffma2_rn(v.a[j], c, __fmul2_rn(v.a[j], rest));
  }
  return y;
}
// s + x . y, pair by pair
__device__ __forceinline__ float2 v8_dot(const V8& x, const V8& y, float2 s) {
#pragma unroll
  for (int j = 0; j < 4; ++j) s = __ffma2_rn(x.a[j], y.a[j], s);
  return s;
}
// the larger of a and |b|; NaN if either is
__device__ __forceinline__ float max_abs_nan(float a, float b) {
  float y;
  asm("{.reg .f32 t; abs.f32 t, %2; max.NaN.f32 %0, %1, t;}" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float v8_max_abs(const V8& x) {  // NaN if any value is
  float m = 0.f, n = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m = max_abs_nan(m, x.a[j].x);
    n = max_abs_nan(n, x.a[j].y);
  }
  return max_abs_nan(m, n);
}

}  // namespace mhc
