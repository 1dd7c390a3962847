// The 8-bit activation checkpoint: format, rounding and expansion.
//
// A row of `cols` values is stored as int8 codes, padded with zeros to
// pitch = 128 * ceil(cols / 128) bytes, and one exponent byte E for each block
// of 32 codes.  With a = max |x| over a block, the block's step is
// 2^(E - 127) for the smallest E >= 1 with a < 127.5 * 2^(E - 127); the code is
// x / step rounded to the nearest integer (ties to even), in [-127, 127], and
// stands for code * step.  E = 255 marks a block that holds an infinity or a
// NaN: all of it stands for NaN, so an overflow still shows after a restore.
// At the largest step, 2^122 (E = 249), a code of 64 would stand for 2^128, past
// fp32 and bf16: codes are held to +-63 there.
//
// Why a power of two: dividing by the step is exact, so the codes depend on
// nothing but the input bits, and code * step (8 significant bits with the
// sign) is exact in bf16, tf32 and fp32, so a matrix product can take the
// restored value in bf16 without a second rounding.  Against a step of a / 127
// it costs 0 to 1 bit; blocks of 32 with a one-byte exponent win that back
// against blocks of 128 with a 4-byte scale at the same size (33/32 bytes a
// value): for normal values the rms error is 0.60% of the values' rms in both.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace mhc {

constexpr int kCkBlock = 32;   // values per exponent
constexpr uint32_t kCkTop = 249;  // the largest exponent byte of finite values
constexpr int kCkPitch = 128;  // rows of codes are padded to a multiple of this

inline __host__ __device__ int64_t ck_pitch(int64_t cols) { return (cols + kCkPitch - 1) / kCkPitch * kCkPitch; }

// Exponent byte of a block from the largest |x| as bits (sign cleared; as
// integers these order as the values do, with infinities and NaNs on top).
// Adding 2^16 carries into the exponent exactly if the significand is at least
// 1.9921875 = 127.5 / 64.
__device__ __forceinline__ uint32_t ck_exponent(uint32_t amax_bits) {
  const uint32_t e = (amax_bits + 0x10000u) >> 23;
  const uint32_t s = e > 7u ? e - 6u : 1u;
  return amax_bits >= 0x7f800000u ? 255u : s;
}
// 1 / step as a float, E in [1, 249]; 0 for E = 255 (the codes are then 0 or
// whatever a NaN rounds to: the exponent alone says NaN)
__device__ __forceinline__ float ck_inverse(uint32_t E) {
  return E == 255u ? 0.f : __uint_as_float((254u - E) << 23);
}
__device__ __forceinline__ float ck_step(uint32_t E) {
  return __uint_as_float(E == 255u ? 0x7fc00000u : E << 23);
}
// Code of one value in the low byte: adding 1.5 * 2^23 rounds x * inv (exact)
// to an integer, ties to even, whose two's complement sits in the low bits.
__device__ __forceinline__ uint32_t ck_code(float x, float inv) {
  return __float_as_uint(fmaf(x, inv, 12582912.0f));
}
__device__ __forceinline__ uint32_t ck_pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Four codes -> four values.  The byte with its sign flipped, set into the low
// byte of 2^23, is 2^23 + 128 + code; the subtraction and the product with the
// step are exact (8 significant bits).
__device__ __forceinline__ void ck_expand4(uint32_t codes, float2 step, float* v) {
  const uint32_t u = codes ^ 0x80808080u;
  const float2 minus = make_float2(-8388736.0f, -8388736.0f);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    float2 f = make_float2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + 2 * j)),
                           __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441 + 2 * j)));
    f = __fmul2_rn(__fadd2_rn(f, minus), step);
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float ck_f32(float v) { return v; }
__device__ __forceinline__ float ck_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void ck_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void ck_store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// A thread works on units of 8 consecutive columns; four lanes hold a block.
// Eight values in one access of 32 (fp32) or 16 (bf16) bytes, aligned to its size:
__device__ __forceinline__ void ck_load(const float* p, float (&v)[8]) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p));
}
__device__ __forceinline__ void ck_load(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(r[j] << 16);
    v[2 * j + 1] = __uint_as_float(r[j] & 0xffff0000u);
  }
}
__device__ __forceinline__ void ck_save(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
               "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
__device__ __forceinline__ void ck_save(__nv_bfloat16* p, const float (&v)[8]) {
  uint4 r;
  __nv_bfloat162 h[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
  r.x = *reinterpret_cast<uint32_t*>(&h[0]); r.y = *reinterpret_cast<uint32_t*>(&h[1]);
  r.z = *reinterpret_cast<uint32_t*>(&h[2]); r.w = *reinterpret_cast<uint32_t*>(&h[3]);
  *reinterpret_cast<uint4*>(p) = r;
}

// Rows whose start or width breaks such accesses go through shared memory: the
// warp's 256 consecutive columns [c0, c0 + 256) move as 8 coalesced accesses of
// one value a lane, and change hands in `sm` (256 words of the warp's own).
// (Columns one a lane throughout took 3 times as long.)  Values past the row's
// end read as zero and are not written.
__device__ __forceinline__ int ck_word(int w) { return w ^ (((w >> 5) & 1) << 2); }  // no bank twice either way
template <typename T>
__device__ __forceinline__ void ck_load_any(const T* row, int64_t c0, int64_t cols, float* sm, float (&v)[8]) {
  const int lane = threadIdx.x & 31;
  float t[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) t[j] = c0 + 32 * j + lane < cols ? ck_f32(row[c0 + 32 * j + lane]) : 0.f;
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j) sm[ck_word(32 * j + lane)] = t[j];
  __syncwarp();
  const float4 a = *reinterpret_cast<const float4*>(sm + ck_word(8 * lane));
  const float4 b = *reinterpret_cast<const float4*>(sm + ck_word(8 * lane + 4));
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void ck_save_any(T* row, int64_t c0, int64_t cols, float* sm, const float (&v)[8]) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
  *reinterpret_cast<float4*>(sm + ck_word(8 * lane)) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(sm + ck_word(8 * lane + 4)) = make_float4(v[4], v[5], v[6], v[7]);
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (c0 + 32 * j + lane < cols) ck_store(row + c0 + 32 * j + lane, sm[ck_word(32 * j + lane)]);
}

// Codes and exponent of the unit that starts at column c of its row.  All
// lanes of the warp take part; values past the row's end are zeros, and `on`
// says whether the unit lies inside the padded row.
__device__ __forceinline__ void ck_encode(float (&v)[8], int8_t* codes, uint8_t* exps, int64_t c, bool on) {
  uint32_t m = abs_bits(v[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) m = max(m, abs_bits(v[j]));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const uint32_t E = ck_exponent(m);
  const float inv = ck_inverse(E);
  if (!on) return;
  if (E == kCkTop) {  // the largest finite values
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fminf(fmaxf(v[j], -63.f * 0x1p122f), 63.f * 0x1p122f);
  }
  uint2 w;
  w.x = ck_pack4(ck_code(v[0], inv), ck_code(v[1], inv), ck_code(v[2], inv), ck_code(v[3], inv));
  w.y = ck_pack4(ck_code(v[4], inv), ck_code(v[5], inv), ck_code(v[6], inv), ck_code(v[7], inv));
  *reinterpret_cast<uint2*>(codes + c) = w;
  if ((threadIdx.x & 3) == 0) exps[c / kCkBlock] = (uint8_t)E;
}

// The values of 8 codes.
__device__ __forceinline__ void ck_decode(uint2 w, uint32_t E, float (&v)[8]) {
  const float2 step = make_float2(ck_step(E), ck_step(E));
  ck_expand4(w.x, step, v);
  ck_expand4(w.y, step, v + 4);
}

}  // namespace mhc
