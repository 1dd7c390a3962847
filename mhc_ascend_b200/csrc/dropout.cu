// Dropout from a counter-based generator (dropout.cuh): one pass, the forward
// and, on the gradient, the backward.
#include "checkpoint8.cuh"
#include "dropout.cuh"

namespace mhc {
namespace {

// Bound by HBM, with 14 instructions a value behind it (ALU 54%): [32768, 4096] bf16 87 us,
// 6.2 TB/s.  Four units a thread share the ten round keys and the addresses (two: 101 us);
// bf16 pairs are scaled as pairs and dropped by masks on the rounded word.
constexpr int kThreads = 256, kUnits = 4;  // units of 8 values a thread

__device__ __forceinline__ void load_raw(const float* p, float (&v)[8]) { ck_load(p, v); }
__device__ __forceinline__ void load_raw(const __nv_bfloat16* p, uint4& v) { v = *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ void put_unit(float* p, float (&v)[8], const uint4& n, uint32_t drop, float scale) {
  drop_apply(n, drop, scale, v);
  ck_save(p, v);
}
// Two bf16 values a word: scaled as pairs, dropped as halves of the result
__device__ __forceinline__ void put_unit(__nv_bfloat16* p, uint4& v, const uint4& n, uint32_t drop, float scale) {
  const uint32_t x[4] = {v.x, v.y, v.z, v.w}, w[4] = {n.x, n.y, n.z, n.w};
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 s = __fmul2_rn(make_float2(__uint_as_float(x[j] << 16), __uint_as_float(x[j] & 0xffff0000u)),
                                make_float2(scale, scale));
    const __nv_bfloat162 b = __floats2bfloat162_rn(s.x, s.y);
    uint32_t r = *reinterpret_cast<const uint32_t*>(&b);
    if (!keeps_low(w[j], drop)) r &= 0xffff0000u;
    if (!keeps_high(w[j], drop)) r &= 0x0000ffffu;
    o[j] = r;
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(o[0], o[1], o[2], o[3]);
}
template <typename T> struct Raw { using type = float[8]; };
template <> struct Raw<__nv_bfloat16> { using type = uint4; };

// EVEN: 16- or 32-byte accesses; the tensor's last, incomplete unit goes value by
// value.  Otherwise through shared memory (a start that is not aligned).
template <typename T, bool EVEN>
__global__ void __launch_bounds__(kThreads)
    dropout_kernel(const T* __restrict__ x, T* __restrict__ out, int64_t count, DropSource src) {
  __shared__ __align__(16) float sm[EVEN ? 1 : kThreads * 8];
  const int64_t first = (int64_t)blockIdx.x * (kThreads * kUnits) + threadIdx.x;
  const DropKey key = drop_key(src);
  if (EVEN && ((int64_t)blockIdx.x + 1) * (kThreads * kUnits * 8) <= count) {
    typename Raw<T>::type v[kUnits];
    x += 8 * first;
    out += 8 * first;
#pragma unroll
    for (int k = 0; k < kUnits; ++k) load_raw(x + k * kThreads * 8, v[k]);
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
      put_unit(out + k * kThreads * 8, v[k], drop_group(key, first + k * kThreads), src.drop, src.scale);
    return;
  }
  float* mine = sm + (EVEN ? 0 : (threadIdx.x >> 5) * 256);
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int k = 0; k < kUnits; ++k) {
    const int64_t u = first + k * kThreads, c = 8 * u;
    float v[8];
    if (EVEN && c + 8 <= count) {
      ck_load(x + c, v);
    } else if (EVEN) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < count ? ck_f32(x[c + j]) : 0.f;
    } else {
      ck_load_any(x, c - 8 * lane, count, mine, v);
    }
    drop_apply(drop_group(key, u), src.drop, src.scale, v);
    if (EVEN && c + 8 <= count) {
      ck_save(out + c, v);
    } else if (EVEN) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < count) ck_store(out + c + j, v[j]);
    } else {
      ck_save_any(out, c - 8 * lane, count, mine, v);
    }
  }
}

template <typename T>
int launch_dropout(const T* x, T* out, int64_t count, const DropSource& src, cudaStream_t st) {
  constexpr uintptr_t align = 8 * sizeof(T) - 1;
  const bool even = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & align) == 0;
  const int64_t blocks = ((count + 7) / 8 + kThreads * kUnits - 1) / (kThreads * kUnits);
  MHC_REQUIRE(blocks < (1ll << 31), MHC_ERR_UNSUPPORTED, "dropout: %lld values are too many", (long long)count);
  ProfScope p("dropout", st);
  if (src.drop >= kDropAll) cudaMemsetAsync(out, 0, (size_t)count * sizeof(T), st);
  else if (even) dropout_kernel<T, true><<<(unsigned)blocks, kThreads, 0, st>>>(x, out, count, src);
  else dropout_kernel<T, false><<<(unsigned)blocks, kThreads, 0, st>>>(x, out, count, src);
  return check_launch("dropout");
}

// One atomic step, so that overlapping calls never get the same numbers.
__global__ void take_kernel(unsigned long long* state, unsigned long long* out, unsigned long long groups) {
  out[0] = state[0];
  out[1] = atomicAdd(state + 1, groups);
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" int mhc_dropout(const void* x, int32_t x_bf16, void* out, int64_t count, int32_t drop, const uint64_t* state,
                           uint64_t seed, uint64_t position, void* stream) {
  MHC_REQUIRE(count >= 0, MHC_ERR_INVALID_ARG, "dropout: count must be >= 0 (got %lld)", (long long)count);
  const int rc = check_drop("dropout", drop);
  if (rc) return rc;
  if (count == 0) return MHC_OK;
  MHC_REQUIRE_PTR(x);
  MHC_REQUIRE_PTR(out);
  MHC_REQUIRE((reinterpret_cast<uintptr_t>(state) & 7) == 0, MHC_ERR_ALIGNMENT, "dropout: state must be 8-byte aligned");
  const DropSource src = drop_source(state, seed, position, drop);
  cudaStream_t st = (cudaStream_t)stream;
  return x_bf16 ? launch_dropout((const __nv_bfloat16*)x, (__nv_bfloat16*)out, count, src, st)
                : launch_dropout((const float*)x, (float*)out, count, src, st);
}

extern "C" int mhc_dropout_take(uint64_t* state, uint64_t* out, int64_t groups, void* stream) {
  MHC_REQUIRE(groups >= 0, MHC_ERR_INVALID_ARG, "dropout_take: groups must be >= 0 (got %lld)", (long long)groups);
  MHC_REQUIRE_PTR(state);
  MHC_REQUIRE_PTR(out);
  MHC_REQUIRE(((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(out)) & 7) == 0, MHC_ERR_ALIGNMENT,
              "dropout_take: state and out must be 8-byte aligned");
  ProfScope p("dropout_take", (cudaStream_t)stream);
  take_kernel<<<1, 1, 0, (cudaStream_t)stream>>>((unsigned long long*)state, (unsigned long long*)out,
                                                 (unsigned long long)groups);
  return check_launch("dropout_take");
}
