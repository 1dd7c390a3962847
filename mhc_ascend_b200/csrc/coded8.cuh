// 8-bit codes with a fp32 scale for a row or for a group of 128 columns: e4m3 or
// int8 codes [rows, cols] without padding; the scales are dense, one beside the other in a row.
//   a = max |y| of the group, scale = max(a / 448, 2^-100) (int8: a / 127),
//   code = y / scale rounded to nearest, ties to even; it stands for code * scale.
// A group that holds an infinity or a NaN has a NaN scale and stands for NaNs.  The scale is a
// product with the rounded 1 / 448 or 1 / 127, and y / scale is h w times 1 / r and the scale's
// approximate reciprocal: a few units of 2^-24 off the quotients, so that a value next to the
// middle of two codes may take the other one.
#pragma once

#include "checkpoint8.cuh"

namespace mhc {

constexpr int kCodedGroup = 128;
constexpr float kCodedLeast = 0x1p-100f;

inline int64_t coded_groups(int64_t cols, bool grouped) {
  return grouped ? (cols + kCodedGroup - 1) / kCodedGroup : 1;
}

// Scale from the largest |y|, and its reciprocal (the divisions by 448 and by the
// scale as products with a reciprocal: 2 units of 2^-24 each, 2 instructions against
// 20 a group)
__device__ __forceinline__ float coded_scale(float a, bool int8) {
  const float s = fmaxf(a * (int8 ? 1.f / 127.f : 1.f / 448.f), kCodedLeast);
  return a <= 3.402823466e38f ? s : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ float coded_inverse(float scale) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(scale));
  return y;
}
// Whether 1 / r times the reciprocal of a scale (2^100 at most) may pass fp32: h w is then
// multiplied by one after the other.  The same for a whole row.
__device__ __forceinline__ bool coded_apart(float ir) { return ir > 0x1p27f; }

// Two codes from two values that have been divided by the scale, a in the low byte.
__device__ __forceinline__ uint32_t coded_pair(float a, float b, bool int8) {
  if (int8) {
    const uint32_t p = ck_code(fminf(fmaxf(a, -127.f), 127.f), 1.f), q = ck_code(fminf(fmaxf(b, -127.f), 127.f), 1.f);
    return __byte_perm(p, q, 0x7740) & 0xffffu;
  }
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint2 coded_pack(const float (&v)[8], bool int8) {
  if (int8) {
    uint32_t q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = ck_code(fminf(fmaxf(v[j], -127.f), 127.f), 1.f);
    return make_uint2(ck_pack4(q[0], q[1], q[2], q[3]), ck_pack4(q[4], q[5], q[6], q[7]));
  }
  return make_uint2(coded_pair(v[0], v[1], false) | coded_pair(v[2], v[3], false) << 16,
                    coded_pair(v[4], v[5], false) | coded_pair(v[6], v[7], false) << 16);
}
// The values of eight codes; scale as a pair
__device__ __forceinline__ void coded_unpack(uint2 w, float scale, bool int8, float (&v)[8]) {
  const float2 s2 = make_float2(scale, scale);
  if (int8) {
    ck_expand4(w.x, s2, v);
    ck_expand4(w.y, s2, v + 4);
    return;
  }
  const uint32_t u[4] = {w.x & 0xffffu, w.x >> 16, w.y & 0xffffu, w.y >> 16};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)u[j]));
    float2 f;
    asm("{.reg .f16 lo, hi; mov.b32 {lo, hi}, %2; cvt.f32.f16 %0, lo; cvt.f32.f16 %1, hi;}" : "=f"(f.x), "=f"(f.y) : "r"(h));
    f = __fmul2_rn(f, s2);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

// Rows that 8-byte accesses do not fit: through shared memory, as ck_save_any.
__device__ __forceinline__ void coded_save_any(uint8_t* row, int64_t c0, int64_t cols, float* sm, const float (&v)[8],
                                               bool int8) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  *reinterpret_cast<float4*>(sm + ck_word(8 * lane)) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(sm + ck_word(8 * lane + 4)) = make_float4(v[4], v[5], v[6], v[7]);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (c0 + 32 * j + lane < cols)
      row[c0 + 32 * j + lane] = (uint8_t)coded_pair(sm[ck_word(32 * j + lane)], 0.f, int8);
}
__device__ __forceinline__ uint2 coded_load_any(const uint8_t* row, int64_t c, int64_t cols) {
  uint2 w = make_uint2(0u, 0u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (c + j < cols) w.x |= (uint32_t)row[c + j] << (8 * j);
    if (c + 4 + j < cols) w.y |= (uint32_t)row[c + 4 + j] << (8 * j);
  }
  return w;
}

}  // namespace mhc
