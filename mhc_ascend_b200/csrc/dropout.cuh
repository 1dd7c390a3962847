// Random numbers of the dropout operators.
//
// The stream is a function of a seed and a position, so a mask is drawn again
// wherever it is needed and never stored: Philox4x32-10 (Salmon, Moraes, Dror,
// Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011) at counter
// (g low, g high, 0, 0) with the seed's two words as key gives the group g of
// eight 16-bit numbers, word by word, low half first.  Value i of a tensor in
// row-major order takes number i % 8 of group position + i / 8 and is dropped
// where that number is below `drop` = round(65536 p).
//
// Why 16 bits a value: the generator's 20 wide products and 40 logical
// operations are shared by eight values, about 8 instructions each, where a
// 32-bit number for each would take 15 of the 22 that HBM leaves a bf16 value
// (two bytes in, two out).  p is then a multiple of 2^-16, and the scale of what
// is kept is exactly 1 / (1 - drop / 65536).
#pragma once

#include "common.cuh"

namespace mhc {

constexpr int kDropGroup = 8;         // numbers of a group
constexpr uint32_t kDropAll = 65536;  // `drop` of p = 1

// Where the numbers come from: device words (seed, position) if given, so that a
// captured graph draws new ones each time, or the values themselves.
struct DropSource {
  const uint64_t* state;
  uint64_t seed, position;
  uint32_t drop;  // 0: no dropout
  float scale;
};

inline DropSource drop_source(const uint64_t* state, uint64_t seed, uint64_t position, int32_t drop) {
  const uint32_t d = (uint32_t)drop;
  return {state, seed, position, d, d >= kDropAll ? 0.f : (float)(65536.0 / (double)(kDropAll - d))};
}

inline int check_drop(const char* what, int32_t drop) {
  MHC_REQUIRE(drop >= 0 && drop <= (int32_t)kDropAll, MHC_ERR_INVALID_ARG, "%s: drop must be in [0, 65536] (got %d)",
              what, (int)drop);
  return MHC_OK;
}

struct DropKey {
  uint32_t k0, k1;
  uint64_t position;
};
__device__ __forceinline__ DropKey drop_key(const DropSource& s) {
  const uint64_t seed = s.state ? s.state[0] : s.seed;
  return {(uint32_t)seed, (uint32_t)(seed >> 32), s.state ? s.state[1] : s.position};
}

// The eight numbers of a group, two a word.
__device__ __forceinline__ uint4 drop_group(const DropKey& key, uint64_t group) {
  const uint64_t g = key.position + group;
  uint32_t x0 = (uint32_t)g, x1 = (uint32_t)(g >> 32), x2 = 0u, x3 = 0u, k0 = key.k0, k1 = key.k1;
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * x0, b = (uint64_t)0xCD9E8D57u * x2;
    x0 = (uint32_t)(b >> 32) ^ x1 ^ k0;
    x1 = (uint32_t)b;
    x2 = (uint32_t)(a >> 32) ^ x3 ^ k1;
    x3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(x0, x1, x2, x3);
}

// Whether each of a word's two numbers keeps its value: the numbers are compared in
// the upper half of a word, where what lies below does not matter.
__device__ __forceinline__ bool keeps_low(uint32_t w, uint32_t drop) { return w << 16 >= drop << 16; }
__device__ __forceinline__ bool keeps_high(uint32_t w, uint32_t drop) { return w >= drop << 16; }

// Apply a group's numbers to eight values: 0 or v * scale (not fused with what
// follows, so that a sum with a dropped value is the same wherever it is formed).
__device__ __forceinline__ void drop_apply(const uint4& n, uint32_t drop, float scale, float (&v)[8]) {
  const uint32_t w[4] = {n.x, n.y, n.z, n.w};
  if (drop >= kDropAll) {  // the shifted comparison has no room for it
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 s = __fmul2_rn(make_float2(v[2 * j], v[2 * j + 1]), make_float2(scale, scale));
    v[2 * j] = keeps_low(w[j], drop) ? s.x : 0.f;
    v[2 * j + 1] = keeps_high(w[j], drop) ? s.y : 0.f;
  }
}

// The same for eight values that start at element i, which need not begin a group.
__device__ __forceinline__ void drop_apply_at(const DropKey& key, uint64_t i, uint32_t drop, float scale, float (&v)[8]) {
  const uint64_t g = i / kDropGroup;
  const uint32_t off = (uint32_t)i % kDropGroup;
  uint4 n = drop_group(key, g);
  if (off) {  // the last 8 - off numbers of this group and the first of the next
    const uint4 m = drop_group(key, g + 1);
    uint32_t w[8] = {n.x, n.y, n.z, n.w, m.x, m.y, m.z, m.w};
    if (off & 4) {
#pragma unroll
      for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
    }
    if (off & 2) {
#pragma unroll
      for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
    }
    if (off & 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 16);
    }
    n = make_uint4(w[0], w[1], w[2], w[3]);
  }
  drop_apply(n, drop, scale, v);
}

}  // namespace mhc
