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
#include "vec8.cuh"

namespace mhc {
namespace {

struct FwdArgs {
  const void *res, *branch;
  const float* w;
  void* hidden;
  float* rms;     // nullable
  void* out;      // plain output
  int8_t* codes;  // its checkpoint, or the codes (nullable in the plain form)
  uint8_t* exps;
  float* scales;
  int64_t rows, cols, pitch, groups;
  float eps;
  bool int8, grouped, res16, branch16;
  DropSource drop;
  double share;  // 1 / cols
};

// Sum of `a` and largest `m` (NaN if any is) over the row's threads, the same in each.
template <bool WARP>
__device__ __forceinline__ void row_sum_max(float& a, float& m, float* red, float* redm) {
  auto warp_max_nan = [](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max_abs_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  a = warp_sum(a);
  m = warp_max_nan(m);
  if (WARP) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (lane == 0) {
    red[warp] = a;
    redm[warp] = m;
  }
  __syncthreads();
  a = warp_sum(lane < nw ? red[lane] : 0.f);
  m = warp_max_nan(lane < nw ? redm[lane] : 0.f);
}
// Sum joined in 64 bits
template <bool WARP>
__device__ __forceinline__ double row_sum_d(float a, double* red) {
  const double s = warp_sum_d((double)a);
  if (WARP) return s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (lane == 0) red[warp] = s;
  __syncthreads();
  return warp_sum_d(lane < nw ? red[lane] : 0.0);
}
// Root of a row's mean square from the threads' shares, and the largest `m` (CODED).  The
// plain form keeps what fp32 leaves out, since a step of the kept codes hangs on the last
// bit of the output; codes with scales do without.
template <bool WARP, bool CODED>
__device__ __forceinline__ Root row_root(const FwdArgs& p, float cols, float a, float& m, double* red) {
  if (!CODED) return root_of(row_sum_d<WARP>(a, red) * p.share + (double)p.eps);
  row_sum_max<WARP>(a, m, reinterpret_cast<float*>(red), reinterpret_cast<float*>(red) + 32);
  const float r = sqrtf(a / cols + p.eps);
  return {r, 1.0f / r, 0.f};
}
__device__ __forceinline__ float group_max(float m) {  // over 16 lanes, NaN if any is
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) m = max_abs_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

constexpr int fwd_threads(int UPT, bool WARP) { return WARP || UPT == 1 ? 256 : UPT == 2 ? 512 : 1024; }

// Rows over threads of the kernels below; SMALL: four units a thread of at most 256,
// four blocks an SM.
enum class Lay { kWarp, kBlock, kSmall };

// Bound by HBM: [8192, 4096] fp32 residual, bf16 branch with dropout and kept codes 70 us,
// 6.2 TB/s; [16384, 7168] bf16 140 us, 6.7 TB/s, with dropout and kept codes 191 us (issue
// slots).  A row stays in registers between the sum and the output, UPT units a thread.  EVEN:
// whole units; otherwise units of the tensor's own alignment (vec8.cuh), and the kept
// codes, whose blocks begin with the row, pass through shared memory.  CODED: what is
// kept in registers is h w, and its maxima are taken with the sum (r > 0 is common to
// the row: max |y| = max |h w| / r), so that after the barrier a value costs one product
// and its conversion.
__device__ __forceinline__ int row_word(int c) { return c ^ ((c >> 5) & 7); }  // no bank twice, eight columns a lane

template <typename TR, typename TB, int UPT, Lay LAY, bool CODED, bool EVEN>
__global__ void __launch_bounds__(LAY == Lay::kSmall ? 256 : fwd_threads(UPT, LAY == Lay::kWarp),
                                  LAY == Lay::kSmall ? 4 : LAY == Lay::kBlock && UPT == 2 ? 2 : 1)
    add_norm_fwd_kernel(const FwdArgs p) {
  constexpr bool WARP = LAY == Lay::kWarp;
  __shared__ double red[32];
  extern __shared__ __align__(16) float row_sm[];  // uneven rows with kept codes: pitch words a row
  const int lane = threadIdx.x & 31, cols = (int)p.cols;
  const int64_t row = WARP ? (int64_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (WARP && row >= p.rows) return;
  const int shift = EVEN ? 0 : (int)((row * p.cols) & 7);
  const int c0 = 8 * (WARP ? lane : (int)threadIdx.x) - shift, step = 8 * (WARP ? 32 : (int)blockDim.x);
  const int64_t at = row * p.cols + c0, total = p.rows * p.cols;
  const TR* rr = static_cast<const TR*>(p.res) + at;
  const TB* br = static_cast<const TB*>(p.branch) + at;
  TR* hr = static_cast<TR*>(p.hidden) + at;
  auto edge = [&](int c) { return !EVEN && v8_edge(c, cols); };
  auto weights = [&](int c) { return EVEN ? v8_weights(p.w + c) : v8_weights_inside(p.w, c, cols); };
  Raw8<TR> a[UPT];
  Raw8<TB> b[UPT];
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    a[k].zero();
    b[k].zero();
    if (c0 + k * step < cols && (EVEN || at + k * step + 8 <= total)) {
      a[k].load(rr + k * step);
      b[k].load(br + k * step);
    }
  }
  const DropKey key = drop_key(p.drop);
  V8 v[UPT];
  float2 s2 = make_float2(0.f, 0.f);
  float am = 0.f, gm[UPT];
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const int c = c0 + k * step;
    const bool on = c < cols;
    V8 x = b[k].values(), y = a[k].values();
    if (!EVEN && on && at + k * step + 8 > total) {  // the tensor's last
      y = v8_load_part(rr + k * step, total - at - k * step);
      x = v8_load_part(br + k * step, total - at - k * step);
    }
    if (!CODED && p.drop.drop) {
      float f[8];
      v8_spread(x, f);
      drop_apply(drop_group(key, (uint64_t)(at + k * step) / kDropGroup), p.drop.drop, p.drop.scale, f);
      x = v8_gather(f);
    }
    v[k] = v8_add(y, x);
    if (on) {
      if (edge(c)) v8_save_inside(hr + k * step, v[k], c, cols);
      else v8_save_rounded(hr + k * step, v[k]);
    }
    s2 = v8_dot(v[k], v[k], s2);
    if (CODED) {
      if (on) v[k] = v8_mul(v[k], weights(c));
      gm[k] = v8_max_abs(v[k]);
      if (EVEN && p.grouped) gm[k] = group_max(gm[k]);  // 16 lanes hold a group
      else am = max_abs_nan(am, gm[k]);
    }
  }
  const Root root = row_root<WARP, CODED>(p, (float)cols, s2.x + s2.y, am, red);
  float ir = root.ir;
  const bool first = WARP ? lane == 0 : threadIdx.x == 0;
  if (first && p.rms) p.rms[row] = root.r;
  if (CODED) {
    const float scale = coded_scale(am * ir, p.int8);
    if (first && !p.grouped) p.scales[row] = scale;
    if (coded_apart(ir)) {  // before the loop, where it costs nothing (inside it 1.9 of 129 us)
#pragma unroll
      for (int k = 0; k < UPT; ++k) {
        v[k] = v8_scale(v[k], ir);
        gm[k] *= ir;
      }
      ir = 1.f;
    }
    uint8_t* to = reinterpret_cast<uint8_t*>(p.codes) + at;
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      const int c = c0 + k * step;
      float s = scale;
      if (EVEN && p.grouped) {
        s = coded_scale(gm[k] * ir, p.int8);
        if ((lane & 15) == 0 && c < cols) p.scales[row * p.groups + c / kCodedGroup] = s;
      }
      float f[8];
      v8_spread(v8_scale(v[k], ir * coded_inverse(s)), f);
      if (c < cols) {
        const uint2 w = coded_pack(f, p.int8);
        if (!edge(c)) {
          *reinterpret_cast<uint2*>(to + k * step) = w;
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (c + j >= 0 && c + j < cols) to[k * step + j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
        }
      }
    }
    return;
  }
  TB* out = static_cast<TB*>(p.out) + at;
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    const int c = c0 + k * step;
    V8 y = v8_zero();
    if (c < cols) {
      y = v8_normed(v[k], weights(c), root);
      if (edge(c)) v8_save_inside(out + k * step, y, c, cols);
      else v8_save_rounded(out + k * step, y);
    }
    if (!p.codes) continue;
    float f[8];
    v8_spread(y, f);
    if (EVEN) {  // of the output as it is returned
      ck_encode(f, p.codes + row * p.pitch, p.exps + row * (p.pitch / kCkBlock), c, c < p.pitch);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j >= 0 && c + j < cols) row_sm[row_word(c + j)] = f[j];
    }
  }
  if (!EVEN && p.codes) {
    static_assert(EVEN || CODED || !WARP, "a row's codes pass through the block's shared memory");
    for (int c = cols + (int)threadIdx.x; c < p.pitch; c += blockDim.x) row_sm[row_word(c)] = 0.f;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      const int c = 8 * (int)threadIdx.x + k * step;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = c < p.pitch ? row_sm[row_word(c + j)] : 0.f;
      ck_encode(f, p.codes + row * p.pitch, p.exps + row * (p.pitch / kCkBlock), c, c < p.pitch);
    }
  }
}

// ---------------------------------------------------------------------------
// Any row: through shared memory, and types by a branch.
// ---------------------------------------------------------------------------
__device__ __forceinline__ float rounded_as(float v, bool b16) { return b16 ? __bfloat162float(__float2bfloat16_rn(v)) : v; }

// h of a unit: stored, and its share of the sum and of the maximum
template <bool CODED>
__device__ __forceinline__ void add_unit_any(const FwdArgs& p, const DropKey& key, int64_t row, int64_t c, float* mine,
                                             float (&v)[8], float& ss, float& am) {
  float b[8];
  load_any(p.res, p.res16, row, c, p.cols, mine, v);
  load_any(p.branch, p.branch16, row, c, p.cols, mine, b);
  if (p.drop.drop) drop_apply_at(key, (uint64_t)row * (uint64_t)p.cols + (uint64_t)c, p.drop.drop, p.drop.scale, b);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = rounded_as(v[j] + b[j], p.res16);
    ss = fmaf(v[j], v[j], ss);
  }
  if (CODED && !p.grouped) {
    float wv[8];
    load_w(p.w, c, p.cols, wv);
#pragma unroll
    for (int j = 0; j < 8; ++j) am = max_abs_nan(am, v[j] * wv[j]);
  }
  save_any(p.hidden, p.res16, row, c, p.cols, mine, v);
}
template <bool CODED>
__device__ __forceinline__ void put_unit_any(const FwdArgs& p, int64_t row, int64_t c, float (&v)[8], const Root& root,
                                             float row_scale, float* mine) {
  const int lane = threadIdx.x & 31;
  float wv[8];
  load_w(p.w, c, p.cols, wv);
  if (CODED) {
    float scale = row_scale, m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] *= wv[j];
      m = max_abs_nan(m, v[j]);
    }
    if (p.grouped) {
      scale = coded_scale(group_max(m) * root.ir, p.int8);
      if (c < p.cols && (lane & 15) == 0) p.scales[row * p.groups + c / kCodedGroup] = scale;
    }
    float mult = root.ir * coded_inverse(scale);
    if (coded_apart(root.ir)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= root.ir;
      mult = coded_inverse(scale);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= mult;
    coded_save_any(reinterpret_cast<uint8_t*>(p.codes) + row * p.cols, c - 8 * lane, p.cols, mine, v, p.int8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = normed(v[j], wv[j], root);
    save_any(p.out, p.branch16, row, c, p.cols, mine, v);
    if (p.codes) {  // of the output as it is returned
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = c + j < p.cols ? rounded_as(v[j], p.branch16) : 0.f;  // 0 / r is NaN in a row of NaNs
      ck_encode(v, p.codes + row * p.pitch, p.exps + row * (p.pitch / kCkBlock), c, c < p.pitch);
    }
  }
}

template <int UPT, bool WARP, bool CODED>
__global__ void __launch_bounds__(fwd_threads(UPT, WARP)) add_norm_fwd_any_kernel(const FwdArgs p) {
  __shared__ double red[32];
  __shared__ __align__(16) float sm[fwd_threads(UPT, WARP) * 8];
  float* mine = sm + (threadIdx.x >> 5) * 256;
  const int lane = threadIdx.x & 31;
  const int64_t row = WARP ? (int64_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : (int64_t)blockIdx.x;
  if (WARP && row >= p.rows) return;
  const DropKey key = drop_key(p.drop);
  float v[UPT][8];
  float ss = 0.f, am = 0.f;
#pragma unroll
  for (int k = 0; k < UPT; ++k) add_unit_any<CODED>(p, key, row, unit_col<WARP>(k), mine, v[k], ss, am);
  const Root root = row_root<WARP, CODED>(p, (float)p.cols, ss, am, red);
  const float scale = CODED ? coded_scale(am * root.ir, p.int8) : 0.f;
  if (WARP ? lane == 0 : threadIdx.x == 0) {
    if (p.rms) p.rms[row] = root.r;
    if (CODED && !p.grouped) p.scales[row] = scale;
  }
#pragma unroll
  for (int k = 0; k < UPT; ++k) put_unit_any<CODED>(p, row, unit_col<WARP>(k), v[k], root, scale, mine);
}

// Rows too long for registers (past 32768 columns): h is read again, from L2, by the thread
// that wrote it.
constexpr int kLongThreads = 1024;
template <bool CODED>
__global__ void __launch_bounds__(kLongThreads) add_norm_fwd_long_kernel(const FwdArgs p) {
  __shared__ double red[32];
  __shared__ __align__(16) float sm[kLongThreads * 8];
  float* mine = sm + (threadIdx.x >> 5) * 256;
  const int lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  const DropKey key = drop_key(p.drop);
  float ss = 0.f, am = 0.f;
  for (int64_t c0 = (threadIdx.x >> 5) * 256; c0 < p.cols; c0 += 8 * kLongThreads) {
    float v[8];
    add_unit_any<CODED>(p, key, row, c0 + 8 * lane, mine, v, ss, am);
  }
  const Root root = row_root<false, CODED>(p, (float)p.cols, ss, am, red);
  const float scale = CODED ? coded_scale(am * root.ir, p.int8) : 0.f;
  if (threadIdx.x == 0) {
    if (p.rms) p.rms[row] = root.r;
    if (CODED && !p.grouped) p.scales[row] = scale;
  }
  const int64_t end = CODED ? p.cols : p.pitch;
  for (int64_t c0 = (threadIdx.x >> 5) * 256; c0 < end; c0 += 8 * kLongThreads) {
    float v[8];
    load_any(p.hidden, p.res16, row, c0 + 8 * lane, p.cols, mine, v);
    put_unit_any<CODED>(p, row, c0 + 8 * lane, v, root, scale, mine);
  }
}

enum class Way { kEven, kUneven, kAny };
struct FwdPlan {
  Way way;
  Lay lay;
  int UPT, threads;  // UPT = 0: the long kernel
};
// Rows of 1025 to 8192 columns: where there are many, four units a thread, since more and
// smaller blocks overlap each other's barriers ([16384, 7168] bf16 to e4m3 with a scale for
// each 128: 129 us, 6.4 TB/s, against 162 with two units and 448 threads, 175 with one and
// 896); where there are few, as many threads as there are units ([1, 4096] 2.4 us against 3.3).
// Uneven rows take two units a thread (four spill: [8192, 4097] fp32 residual, bf16 branch,
// kept codes 93 us against 114), and short ones of the plain form the kernel for any row
// ([65536, 250] with kept codes 54 us against 75: its units begin with the row, as the
// codes do; without them too, so that they change no bit of the output).
// aligned: wide accesses fit the tensors' starts; by_column: scales belong to columns.
FwdPlan fwd_plan(int64_t rows, int64_t cols, bool aligned, bool aligned_w, bool by_column, bool coded) {
  const int64_t pitch = ck_pitch(cols), U = pitch / 8, spread = (cols + 7) / 8 + 1;
  const int64_t most = spread > U ? spread : U;  // units of a row wherever it starts
  auto threads = [](int64_t units, int upt) { return (int)(((units + upt - 1) / upt + 31) / 32 * 32); };
  if (aligned && cols % 8 && !by_column) {
    if (most <= 128 && coded) return {Way::kUneven, Lay::kWarp, most <= 32 ? 1 : most <= 64 ? 2 : 4, 32 * kWarpRows};
    if (most > 128 && most <= 1024) return {Way::kUneven, Lay::kBlock, 2, threads(most, 2)};
    if (most > 1024 && most <= 4096) return {Way::kUneven, Lay::kBlock, 4, threads(most, 4)};
  }
  const Way way = aligned && aligned_w && cols % 8 == 0 ? Way::kEven : Way::kAny;
  if (pitch <= kWarpCols) return {way, Lay::kWarp, pitch <= 256 ? 1 : pitch <= 512 ? 2 : 4, 32 * kWarpRows};
  if (way == Way::kEven && U <= 1024 && rows >= 2 * num_sms()) return {way, Lay::kSmall, 4, threads(U, 4)};
  for (int upt : {1, 2, 4})
    if (U <= upt * fwd_threads(upt, false)) return {way, Lay::kBlock, upt, threads(U, upt)};
  return {Way::kAny, Lay::kBlock, 0, kLongThreads};
}

template <bool CODED, typename TR, typename TB>
int launch_fwd(const FwdArgs& p, cudaStream_t st) {
  const bool aligned = even_rows<TR>(p.res, 8, 8) && even_rows<TR>(p.hidden, 8, 8) && even_rows<TB>(p.branch, 8, 8) &&
                       (CODED ? (reinterpret_cast<uintptr_t>(p.codes) & 7) == 0 : even_rows<TB>(p.out, 8, 8));
  const FwdPlan pl = fwd_plan(p.rows, p.cols, aligned, even_rows<float>(p.w, 8, 8), p.grouped, CODED);
  const unsigned blocks = (unsigned)(pl.lay == Lay::kWarp ? (p.rows + kWarpRows - 1) / kWarpRows : p.rows);
  const size_t smem = pl.way == Way::kUneven && p.codes && !CODED ? (size_t)p.pitch * sizeof(float) : 0;
  ProfScope prof(CODED ? "add_rmsnorm_coded" : "add_rmsnorm_fwd", st);
#define MHC_FIT(UPT, LAY, EVEN) add_norm_fwd_kernel<TR, TB, UPT, LAY, CODED, EVEN><<<blocks, pl.threads, smem, st>>>(p)
#define MHC_GO(UPT, LAY)                                                                                    \
  do {                                                                                                      \
    if (pl.way == Way::kEven) MHC_FIT(UPT, LAY, true);                                                      \
    else add_norm_fwd_any_kernel<UPT, LAY == Lay::kWarp, CODED><<<blocks, pl.threads, 0, st>>>(p);          \
  } while (0)
  if (pl.way == Way::kUneven) {
    if (pl.lay == Lay::kWarp) {
      if constexpr (CODED) {  // the plain form's short rows take the kernel for any row
        if (pl.UPT == 1) MHC_FIT(1, Lay::kWarp, false);
        else if (pl.UPT == 2) MHC_FIT(2, Lay::kWarp, false);
        else MHC_FIT(4, Lay::kWarp, false);
      }
    } else if (pl.UPT == 2) {
      MHC_FIT(2, Lay::kBlock, false);
    } else {
      // the limit belongs to the kernel: always what its widest row asks for
      if (smem && cudaFuncSetAttribute(add_norm_fwd_kernel<TR, TB, 4, Lay::kBlock, CODED, false>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, 4096 * 8 * (int)sizeof(float)) != cudaSuccess)
        return fail(MHC_ERR_CUDA, "add_rmsnorm: cannot reserve shared memory for a row");
      MHC_FIT(4, Lay::kBlock, false);
    }
  } else if (pl.UPT == 0) add_norm_fwd_long_kernel<CODED><<<blocks, pl.threads, 0, st>>>(p);
  else if (pl.lay == Lay::kSmall) MHC_FIT(4, Lay::kSmall, true);
  else if (pl.lay == Lay::kWarp && pl.UPT == 1) MHC_GO(1, Lay::kWarp);
  else if (pl.lay == Lay::kWarp && pl.UPT == 2) MHC_GO(2, Lay::kWarp);
  else if (pl.lay == Lay::kWarp) MHC_GO(4, Lay::kWarp);
  else if (pl.UPT == 1) MHC_GO(1, Lay::kBlock);
  else if (pl.UPT == 2) MHC_GO(2, Lay::kBlock);
  else MHC_GO(4, Lay::kBlock);
#undef MHC_GO
#undef MHC_FIT
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

// Codes back to values: units of 8, four a thread and 256 apart, so that one division finds
// the row of all ([16384, 7168] e4m3 to bf16 55 us, 6.4 TB/s; one unit a thread 69 us).  Rows
// of fewer than 256 units are stepped over one by one on the way.
constexpr int kUnpackUnits = 4;
template <typename T, bool EVEN>
__global__ void __launch_bounds__(256)
    coded_unpack_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scales, T* __restrict__ out,
                        int64_t rows, int64_t cols, int64_t U, int64_t groups, bool int8, bool grouped) {
  __shared__ __align__(16) float sm[EVEN ? 1 : 256 * 8];
  float* mine = sm + (EVEN ? 0 : (threadIdx.x >> 5) * 256);
  const int64_t first = (int64_t)blockIdx.x * (256 * kUnpackUnits) + threadIdx.x;
  int64_t row, u;
  if ((uint64_t)first >> 32 || (uint64_t)U >> 32) {
    row = first / U;
    u = first - row * U;
  } else {  // a 64-bit division takes longer than the rest
    row = (uint32_t)first / (uint32_t)U;
    u = (uint32_t)first - (uint32_t)row * (uint32_t)U;
  }
  int64_t at[kUnpackUnits], col[kUnpackUnits];
  uint2 w[kUnpackUnits];
  float scale[kUnpackUnits];
#pragma unroll
  for (int k = 0; k < kUnpackUnits; ++k) {
    at[k] = row;
    col[k] = 8 * u;
    w[k] = make_uint2(0u, 0u);
    scale[k] = 0.f;
    if (row < rows && 8 * u < cols) {
      const uint8_t* from = codes + row * cols;
      scale[k] = scales[row * groups + (grouped ? 8 * u / kCodedGroup : 0)];
      w[k] = EVEN ? *reinterpret_cast<const uint2*>(from + 8 * u) : coded_load_any(from, 8 * u, cols);
    }
    for (u += 256; u >= U; u -= U) ++row;
  }
#pragma unroll
  for (int k = 0; k < kUnpackUnits; ++k) {
    float v[8];
    coded_unpack(w[k], scale[k], int8, v);
    if (EVEN) {
      if (at[k] < rows && col[k] < cols) ck_save(out + at[k] * cols + col[k], v);
    } else {  // U % 32 == 0: the warp is in one row
      ck_save_any(out + at[k] * cols, col[k] - 8 * (threadIdx.x & 31), at[k] < rows ? cols : 0, mine, v);
    }
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
    const FwdArgs p = {residual, branch, weight, hidden, rms, out, codes, exponents, nullptr, rows, cols, ck_pitch(cols), 0,
                       eps, false, false, residual_bf16 != 0, branch_bf16 != 0, drop_source(state, seed, position, drop),
                       1.0 / (double)cols};
    return launch_fwd<false, TR, TB>(p, (cudaStream_t)stream);
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
    const FwdArgs p = {residual, branch, weight, hidden, nullptr, nullptr, (int8_t*)codes, nullptr, scales, rows, cols, cols,
                       coded_groups(cols, grouped != 0), eps, codes_int8 != 0, grouped != 0, residual_bf16 != 0,
                       branch_bf16 != 0, drop_source(nullptr, 0, 0, 0), 1.0 / (double)cols};
    return launch_fwd<true, TR, TB>(p, (cudaStream_t)stream);
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
    const int64_t u = (cols + 7) / 8, U = even ? u : (u + 31) / 32 * 32, blocks = (rows * U + 256 * kUnpackUnits - 1) / (256 * kUnpackUnits);
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
