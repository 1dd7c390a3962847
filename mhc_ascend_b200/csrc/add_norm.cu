// Residual addition and RMSNorm in one pass over both inputs:
//   h = residual + dropout(branch)      in the residual's type
//   r = sqrt(mean h^2 + eps),  y = h / r * w
// y leaves in the branch's type, with its 8-bit checkpoint (checkpoint8.cuh) if
// wanted, or as 8-bit codes with scales (coded8.cuh).  The norm is of h as it is
// returned, so the backward, which reads h, is the gradient of exactly what the
// forward computed.  Backward: add_norm_bwd.cu.
#include "coded8.cuh"
#include "dropout.cuh"
#include "rows.cuh"

namespace mhc {
namespace {

template <typename TR, typename TB>
struct FwdArgs {
  const TR* res;
  const TB* branch;
  const float* w;
  TR* hidden;
  float* rms;  // nullable
  TB* out;     // plain output
  int8_t* codes;  // its checkpoint, or the codes (nullable in the plain form)
  uint8_t* exps;
  float* scales;
  int64_t rows, cols, pitch, groups;
  float eps;
  bool int8, grouped;
  DropSource drop;
};

// Sum of `a` and largest `m` over the row's threads, the same in each.
template <bool WARP>
__device__ __forceinline__ void row_sum_max(float& a, uint32_t& m, float* red, uint32_t* redm) {
  a = warp_sum(a);
  m = __reduce_max_sync(0xffffffffu, m);
  if (WARP) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (lane == 0) {
    red[warp] = a;
    redm[warp] = m;
  }
  __syncthreads();
  a = warp_sum(lane < nw ? red[lane] : 0.f);
  m = __reduce_max_sync(0xffffffffu, lane < nw ? redm[lane] : 0u);
}

__device__ __forceinline__ float rounded_as(float v, const float*) { return v; }
__device__ __forceinline__ float rounded_as(float v, const __nv_bfloat16*) { return __bfloat162float(__float2bfloat16_rn(v)); }

// h of a unit: residual + branch (dropped), rounded to the residual's type
template <bool EVEN, typename TR, typename TB>
__device__ __forceinline__ void add_unit(const FwdArgs<TR, TB>& p, const DropKey& key, int64_t row, int64_t c, float (&v)[8],
                                         float (&b)[8]) {
  if (p.drop.drop) {
    const uint64_t i = (uint64_t)row * (uint64_t)p.cols + (uint64_t)c;
    if (EVEN) drop_apply(drop_group(key, i / kDropGroup), p.drop.drop, p.drop.scale, b);
    else drop_apply_at(key, i, p.drop.drop, p.drop.scale, b);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = rounded_as(v[j] + b[j], p.hidden);
}

// Output of a unit: h in v, weights in wv
template <bool EVEN, bool CODED, typename TR, typename TB>
__device__ __forceinline__ void put_unit(const FwdArgs<TR, TB>& p, int64_t row, int64_t c, float (&v)[8], const float (&wv)[8],
                                         float ir, float row_scale, float* mine) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = v[j] * ir * wv[j];
  if (CODED) {
    float scale = row_scale;
    if (p.grouped) {  // 16 lanes hold a group
      uint32_t m = abs_bits(v[0]);
#pragma unroll
      for (int j = 1; j < 8; ++j) m = max(m, abs_bits(v[j]));
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      scale = coded_scale(__uint_as_float(m), p.int8);
      if (c < p.cols && (lane & 15) == 0) p.scales[row * p.groups + c / kCodedGroup] = scale;
    }
    const float inv = 1.0f / scale;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= inv;
    uint8_t* to = reinterpret_cast<uint8_t*>(p.codes) + row * p.cols;
    if (EVEN) {
      if (c < p.cols) *reinterpret_cast<uint2*>(to + c) = coded_pack(v, p.int8);
    } else {
      coded_save_any(to, c - 8 * lane, p.cols, mine, v, p.int8);
    }
  } else {
    if (EVEN) {
      if (c < p.cols) ck_save(p.out + row * p.cols + c, v);
    } else {
      ck_save_any(p.out + row * p.cols, c - 8 * lane, p.cols, mine, v);
    }
    if (p.codes) {  // of the output as it is returned
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < p.cols ? rounded_as(v[j], p.out) : 0.f;  // 0 / r is NaN in a row of NaNs
      ck_encode(v, p.codes + row * p.pitch, p.exps + row * (p.pitch / kCkBlock), c, c < p.pitch);
    }
  }
}

constexpr int fwd_threads(int UPT, bool WARP) { return WARP || UPT == 1 ? 256 : UPT == 2 ? 512 : 1024; }

// A row stays in registers between the sum and the output, UPT units a thread.
template <typename TR, typename TB, int UPT, bool WARP, bool EVEN, bool CODED>
__global__ void __launch_bounds__(fwd_threads(UPT, WARP)) add_norm_fwd_kernel(const FwdArgs<TR, TB> p) {
  __shared__ float red[32];
  __shared__ uint32_t redm[32];
  extern __shared__ __align__(16) float sm[];  // uneven rows: 8 a thread
  float* mine = sm + (EVEN ? 0 : (threadIdx.x >> 5) * 256);
  const int lane = threadIdx.x & 31;
  const int64_t row = WARP ? (int64_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (WARP && row >= p.rows) return;
  const TR* rr = p.res + row * p.cols;
  const TB* br = p.branch + row * p.cols;
  const DropKey key = drop_key(p.drop);
  float v[UPT][8], b[UPT][8];
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const int64_t c = unit_col<WARP>(k);
    if (EVEN) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[k][j] = b[k][j] = 0.f;
      if (c < p.cols) {
        ck_load(rr + c, v[k]);
        ck_load(br + c, b[k]);
      }
    } else {
      ck_load_any(rr, c - 8 * lane, p.cols, mine, v[k]);
      ck_load_any(br, c - 8 * lane, p.cols, mine, b[k]);
    }
  }
  float ss = 0.f;
  uint32_t am = 0u;
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const int64_t c = unit_col<WARP>(k);
    add_unit<EVEN>(p, key, row, c, v[k], b[k]);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[k][j], v[k][j], ss);
    if (CODED && !p.grouped) {
      float wv[8];
      load_w(p.w, c, p.cols, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) am = max(am, abs_bits(v[k][j] * wv[j]));
    }
    if (EVEN) {
      if (c < p.cols) ck_save(p.hidden + row * p.cols + c, v[k]);
    } else {
      ck_save_any(p.hidden + row * p.cols, c - 8 * lane, p.cols, mine, v[k]);
    }
  }
  if (CODED) row_sum_max<WARP>(ss, am, red, redm);
  else ss = row_total<WARP>(ss, red);
  const float r = sqrtf(ss / (float)p.cols + p.eps), ir = 1.0f / r;
  const float scale = CODED ? coded_scale(__uint_as_float(am) * ir, p.int8) : 0.f;
  if (WARP ? lane == 0 : threadIdx.x == 0) {
    if (p.rms) p.rms[row] = r;
    if (CODED && !p.grouped) p.scales[row] = scale;
  }
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const int64_t c = unit_col<WARP>(k);
    float wv[8];
    load_w(p.w, c, p.cols, wv);
    put_unit<EVEN, CODED>(p, row, c, v[k], wv, ir, scale, mine);
  }
}

// Rows too long for registers: h is read again, from L2, by the thread that wrote it.
constexpr int kLongThreads = 1024;
template <typename TR, typename TB, bool CODED>
__global__ void __launch_bounds__(kLongThreads) add_norm_fwd_long_kernel(const FwdArgs<TR, TB> p) {
  __shared__ float red[32];
  __shared__ uint32_t redm[32];
  __shared__ __align__(16) float sm[kLongThreads * 8];
  float* mine = sm + (threadIdx.x >> 5) * 256;
  const int lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  const DropKey key = drop_key(p.drop);
  float ss = 0.f;
  uint32_t am = 0u;
  for (int64_t c0 = (threadIdx.x >> 5) * 256; c0 < p.cols; c0 += 8 * kLongThreads) {
    const int64_t c = c0 + 8 * lane;
    float v[8], b[8];
    ck_load_any(p.res + row * p.cols, c0, p.cols, mine, v);
    ck_load_any(p.branch + row * p.cols, c0, p.cols, mine, b);
    add_unit<false>(p, key, row, c, v, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
    if (CODED && !p.grouped) {
      float wv[8];
      load_w(p.w, c, p.cols, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) am = max(am, abs_bits(v[j] * wv[j]));
    }
    ck_save_any(p.hidden + row * p.cols, c0, p.cols, mine, v);
  }
  row_sum_max<false>(ss, am, red, redm);
  const float r = sqrtf(ss / (float)p.cols + p.eps), ir = 1.0f / r;
  const float scale = CODED ? coded_scale(__uint_as_float(am) * ir, p.int8) : 0.f;
  if (threadIdx.x == 0) {
    if (p.rms) p.rms[row] = r;
    if (CODED && !p.grouped) p.scales[row] = scale;
  }
  const int64_t end = CODED ? p.cols : p.pitch;
  for (int64_t c0 = (threadIdx.x >> 5) * 256; c0 < end; c0 += 8 * kLongThreads) {
    const int64_t c = c0 + 8 * lane;
    float v[8], wv[8];
    ck_load_any(static_cast<const TR*>(p.hidden) + row * p.cols, c0, p.cols, mine, v);
    load_w(p.w, c, p.cols, wv);
    put_unit<false, CODED>(p, row, c, v, wv, ir, scale, mine);
  }
}

struct FwdPlan {
  int UPT, threads;  // UPT = 0: the long kernel
  bool warp;
};
FwdPlan fwd_plan(int64_t cols) {
  const int64_t pitch = ck_pitch(cols), U = pitch / 8;
  if (pitch <= kWarpCols) return {pitch <= 256 ? 1 : pitch <= 512 ? 2 : 4, 32 * kWarpRows, true};
  for (int upt : {1, 2, 4})
    if (U <= upt * fwd_threads(upt, false)) return {upt, (int)(((U + upt - 1) / upt + 31) / 32 * 32), false};
  return {0, kLongThreads, false};
}

template <bool CODED, typename TR, typename TB>
int launch_fwd(const FwdArgs<TR, TB>& p, cudaStream_t st) {
  bool even = even_rows<TR>(p.res, p.cols, p.cols) && even_rows<TR>(p.hidden, p.cols, p.cols) &&
              even_rows<TB>(p.branch, p.cols, p.cols);
  even = even && (CODED ? (reinterpret_cast<uintptr_t>(p.codes) & 7) == 0 : even_rows<TB>(p.out, p.cols, p.cols));
  const FwdPlan pl = fwd_plan(p.cols);
  const unsigned blocks = (unsigned)(pl.warp ? (p.rows + kWarpRows - 1) / kWarpRows : p.rows);
  const size_t staging = even ? 0 : (size_t)pl.threads * 32;
  ProfScope prof(CODED ? "add_rmsnorm_coded" : "add_rmsnorm_fwd", st);
#define MHC_GO(UPT, WARP)                                                                                       \
  do {                                                                                                          \
    if (even) add_norm_fwd_kernel<TR, TB, UPT, WARP, true, CODED><<<blocks, pl.threads, staging, st>>>(p);      \
    else add_norm_fwd_kernel<TR, TB, UPT, WARP, false, CODED><<<blocks, pl.threads, staging, st>>>(p);          \
  } while (0)
  if (pl.UPT == 0) add_norm_fwd_long_kernel<TR, TB, CODED><<<blocks, pl.threads, 0, st>>>(p);
  else if (pl.warp && pl.UPT == 1) MHC_GO(1, true);
  else if (pl.warp && pl.UPT == 2) MHC_GO(2, true);
  else if (pl.warp) MHC_GO(4, true);
  else if (pl.UPT == 1) MHC_GO(1, false);
  else if (pl.UPT == 2) MHC_GO(2, false);
  else MHC_GO(4, false);
#undef MHC_GO
  return check_launch("add_rmsnorm");
}

int check_fwd(const char* what, int64_t rows, int64_t cols, float eps, int32_t drop, const uint64_t* state) {
  MHC_REQUIRE(rows >= 0 && cols >= 1, MHC_ERR_INVALID_ARG, "%s: rows must be >= 0 and cols >= 1 (got %lld x %lld)", what,
              (long long)rows, (long long)cols);
  MHC_REQUIRE(cols <= (1ll << 30) && rows < (1ll << 31), MHC_ERR_UNSUPPORTED, "%s: %lld x %lld values are too many", what,
              (long long)rows, (long long)cols);
  MHC_REQUIRE(eps >= 0.f, MHC_ERR_INVALID_ARG, "%s: eps must be >= 0", what);
  MHC_REQUIRE((reinterpret_cast<uintptr_t>(state) & 7) == 0, MHC_ERR_ALIGNMENT, "%s: state must be 8-byte aligned", what);
  return check_drop(what, drop);
}

template <typename F>
int with_types(int32_t a_bf16, int32_t b_bf16, F f) {
  if (a_bf16) return b_bf16 ? f((__nv_bfloat16*)nullptr, (__nv_bfloat16*)nullptr) : f((__nv_bfloat16*)nullptr, (float*)nullptr);
  return b_bf16 ? f((float*)nullptr, (__nv_bfloat16*)nullptr) : f((float*)nullptr, (float*)nullptr);
}

// Codes back to values: one unit of 8 a thread and turn.
template <typename T, bool EVEN>
__global__ void __launch_bounds__(256)
    coded_unpack_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, T* __restrict__ out,
                        int64_t rows, int64_t cols, int64_t U, int64_t groups, bool int8, bool grouped) {
  __shared__ __align__(16) float sm[EVEN ? 1 : 256 * 8];
  float* mine = sm + (EVEN ? 0 : (threadIdx.x >> 5) * 256);
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t row, u;
  if ((uint64_t)i >> 32 || (uint64_t)U >> 32) {
    row = i / U;
    u = i - row * U;
  } else {  // a 64-bit division takes longer than the rest
    row = (uint32_t)i / (uint32_t)U;
    u = (uint32_t)i - (uint32_t)row * (uint32_t)U;
  }
  const int64_t c = 8 * u;
  const bool on = row < rows && c < cols;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (on) {
    const uint8_t* from = codes + row * cols;
    const float scale = scales[row * groups + (grouped ? c / kCodedGroup : 0)];
    coded_unpack(EVEN ? *reinterpret_cast<const uint2*>(from + c) : coded_load_any(from, c, cols), scale, int8, v);
  }
  if (EVEN) {
    if (on) ck_save(out + row * cols + c, v);
  } else {  // U % 32 == 0: the warp is in one row
    ck_save_any(out + row * cols, c - 8 * (threadIdx.x & 31), row < rows ? cols : 0, mine, v);
  }
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" int mhc_add_rmsnorm_fwd(const void* residual, int32_t residual_bf16, const void* branch, int32_t branch_bf16,
                                   const float* weight, void* hidden, void* out, float* rms, int8_t* codes,
                                   uint8_t* exponents, int64_t rows, int64_t cols, float eps, int32_t drop,
                                   const uint64_t* state, uint64_t seed, uint64_t position, void* stream) {
  const char* what = "add_rmsnorm_fwd";
  const int rc = check_fwd(what, rows, cols, eps, drop, state);
  if (rc) return rc;
  if (rows == 0) return MHC_OK;
  MHC_REQUIRE_PTR(residual);
  MHC_REQUIRE_PTR(branch);
  MHC_REQUIRE_PTR(weight);
  MHC_REQUIRE_PTR(hidden);
  MHC_REQUIRE_PTR(out);
  MHC_REQUIRE((codes == nullptr) == (exponents == nullptr), MHC_ERR_INVALID_ARG,
              "%s: codes and exponents must be given together", what);
  MHC_REQUIRE(aligned16(codes) && (reinterpret_cast<uintptr_t>(exponents) & 3) == 0, MHC_ERR_ALIGNMENT,
              "%s: codes must be 16-byte and exponents 4-byte aligned", what);
  return with_types(residual_bf16, branch_bf16, [&](auto* r, auto* b) -> int {
    using TR = std::remove_pointer_t<decltype(r)>;
    using TB = std::remove_pointer_t<decltype(b)>;
    FwdArgs<TR, TB> p = {(const TR*)residual, (const TB*)branch, weight, (TR*)hidden, rms, (TB*)out, codes, exponents, nullptr,
                         rows, cols, ck_pitch(cols), 0, eps, false, false, drop_source(state, seed, position, drop)};
    return launch_fwd<false>(p, (cudaStream_t)stream);
  });
}

extern "C" int mhc_add_rmsnorm_coded(const void* residual, int32_t residual_bf16, const void* branch, int32_t branch_bf16,
                                     const float* weight, void* hidden, void* codes, int32_t codes_int8, float* scales,
                                     int32_t grouped, int64_t rows, int64_t cols, float eps, void* stream) {
  const char* what = "add_rmsnorm_coded";
  const int rc = check_fwd(what, rows, cols, eps, 0, nullptr);
  if (rc) return rc;
  if (rows == 0) return MHC_OK;
  MHC_REQUIRE_PTR(residual);
  MHC_REQUIRE_PTR(branch);
  MHC_REQUIRE_PTR(weight);
  MHC_REQUIRE_PTR(hidden);
  MHC_REQUIRE_PTR(codes);
  MHC_REQUIRE_PTR(scales);
  return with_types(residual_bf16, branch_bf16, [&](auto* r, auto* b) -> int {
    using TR = std::remove_pointer_t<decltype(r)>;
    using TB = std::remove_pointer_t<decltype(b)>;
    FwdArgs<TR, TB> p = {(const TR*)residual, (const TB*)branch, weight, (TR*)hidden, nullptr, nullptr, (int8_t*)codes,
                         nullptr, scales, rows, cols, cols, coded_groups(cols, grouped != 0), eps, codes_int8 != 0,
                         grouped != 0, drop_source(nullptr, 0, 0, 0)};
    return launch_fwd<true>(p, (cudaStream_t)stream);
  });
}

extern "C" int mhc_coded8_unpack(const void* codes, int32_t codes_int8, const float* scales, int32_t grouped, void* out,
                                 int32_t out_bf16, int64_t rows, int64_t cols, void* stream) {
  const char* what = "coded8_unpack";
  const int rc = check_fwd(what, rows, cols, 0.f, 0, nullptr);
  if (rc) return rc;
  if (rows == 0) return MHC_OK;
  MHC_REQUIRE_PTR(codes);
  MHC_REQUIRE_PTR(scales);
  MHC_REQUIRE_PTR(out);
  cudaStream_t st = (cudaStream_t)stream;
  return with_types(out_bf16, 0, [&](auto* o, auto*) -> int {
    using T = std::remove_pointer_t<decltype(o)>;
    const bool even = even_rows<T>(out, cols, cols) && (reinterpret_cast<uintptr_t>(codes) & 7) == 0;
    const int64_t u = (cols + 7) / 8, U = even ? u : (u + 31) / 32 * 32, blocks = (rows * U + 255) / 256;
    MHC_REQUIRE(blocks < (1ll << 31), MHC_ERR_UNSUPPORTED, "coded8_unpack: %lld x %lld values are too many", (long long)rows,
                (long long)cols);
    const int64_t groups = coded_groups(cols, grouped != 0);
    ProfScope prof("coded8_unpack", st);
    if (even) coded_unpack_kernel<T, true><<<(unsigned)blocks, 256, 0, st>>>((const uint8_t*)codes, scales, (T*)out, rows, cols,
                                                                           U, groups, codes_int8 != 0, grouped != 0);
    else coded_unpack_kernel<T, false><<<(unsigned)blocks, 256, 0, st>>>((const uint8_t*)codes, scales, (T*)out, rows, cols, U,
                                                                        groups, codes_int8 != 0, grouped != 0);
    return check_launch("coded8_unpack");
  });
}
