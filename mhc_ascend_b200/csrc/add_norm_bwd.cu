// Backward of the residual addition with RMSNorm (add_norm.cu), from the hidden
// state h that the forward returned:
//   gi = gh + (g w - h D / (C r^2)) / r,   D = sum_c g w h,   r = sqrt(mean h^2 + eps)
//   g_residual = gi,   g_branch = gi with the forward's dropout,   gw = sum over rows of g h / r
// gh is the gradient that reaches h by other ways (the residual stream's), g the
// output's.  A block (or warp) walks every (its count)-th row and keeps its
// columns' share of gw in registers; the shares leave as one row a block and are
// added in block order: no atomics, the same bits every time.
#include "checkpoint8.cuh"
#include "dropout.cuh"
#include "rows.cuh"
#include "tma.cuh"

namespace mhc {
namespace {

template <typename TR, typename TB>
struct BwdArgs {
  const TR* gh;  // nullable: zero
  const TB* g;
  const TR* h;
  const float* w;
  const float* rms;
  TR* gr;
  TB* gb;  // nullable: not wanted
  float* part;
  int64_t rows, cols;
  DropSource drop;
};

// gi of a unit -> both gradients
template <bool EVEN, typename TR, typename TB>
__device__ __forceinline__ void put_grads(const BwdArgs<TR, TB>& p, const DropKey& key, int64_t row, int64_t c, float (&o)[8],
                                          float* mine) {
  const int lane = threadIdx.x & 31;
  const bool on = c < p.cols;
  if (EVEN) {
    if (on) ck_save(p.gr + row * p.cols + c, o);
  } else {
    ck_save_any(p.gr + row * p.cols, c - 8 * lane, p.cols, mine, o);
  }
  if (p.gb) {
    if (p.drop.drop) {
      const uint64_t i = (uint64_t)row * (uint64_t)p.cols + (uint64_t)c;
      if (EVEN) drop_apply(drop_group(key, i / kDropGroup), p.drop.drop, p.drop.scale, o);
      else drop_apply_at(key, i, p.drop.drop, p.drop.scale, o);
    }
    if (EVEN) {
      if (on) ck_save(p.gb + row * p.cols + c, o);
    } else {
      ck_save_any(p.gb + row * p.cols, c - 8 * lane, p.cols, mine, o);
    }
  }
}

template <bool EVEN, typename T>
__device__ __forceinline__ void get_unit(const T* row, int64_t c, int64_t cols, float* mine, float (&v)[8]) {
  if (EVEN) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (c < cols) ck_load(row + c, v);
  } else {
    ck_load_any(row, c - 8 * (threadIdx.x & 31), cols, mine, v);
  }
}

// ---------------------------------------------------------------------------
// Rows in registers: rows of a warp, and blocks' rows that wide accesses do not fit.
// ---------------------------------------------------------------------------
constexpr int bwd_threads(int UPT, bool WARP) { return WARP || UPT == 1 ? 256 : 512; }

template <typename TR, typename TB, int UPT, bool WARP, bool EVEN>
__global__ void __launch_bounds__(bwd_threads(UPT, WARP), WARP ? 1 : 2) add_norm_bwd_kernel(const BwdArgs<TR, TB> p) {
  let_next_start();
  __shared__ float red[2][32];
  __shared__ __align__(16) float sm[bwd_threads(UPT, WARP) * 8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* mine = sm + warp * 256;
  const DropKey key = drop_key(p.drop);
  float acc[UPT][8];
#pragma unroll
  for (int k = 0; k < UPT; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[k][j] = 0.f;
  const int64_t first = WARP ? (int64_t)blockIdx.x * kWarpRows + warp : (int64_t)blockIdx.x;
  const int64_t hop = WARP ? (int64_t)gridDim.x * kWarpRows : (int64_t)gridDim.x;
  int buf = 0;
  for (int64_t row = first; row < p.rows; row += hop, buf ^= 1) {
    const float r = p.rms[row], ir = 1.0f / r;
    float gw[UPT][8], h[UPT][8], o[UPT][8];
    float d = 0.f;
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      const int64_t c = unit_col<WARP>(k);
      get_unit<EVEN>(p.g + row * p.cols, c, p.cols, mine, gw[k]);
      get_unit<EVEN>(p.h + row * p.cols, c, p.cols, mine, h[k]);
      if (p.gh) {
        get_unit<EVEN>(p.gh + row * p.cols, c, p.cols, mine, o[k]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[k][j] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      float wv[8];
      load_w(p.w, unit_col<WARP>(k), p.cols, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        acc[k][j] = fmaf(gw[k][j] * ir, h[k][j], acc[k][j]);
        gw[k][j] *= wv[j];
        d = fmaf(gw[k][j], h[k][j], d);
      }
    }
    // two buffers: a block writes red[buf] again only after the barrier of the row between
    const float coef = row_total<WARP>(d, red[buf]) / ((float)p.cols * r * r);
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) o[k][j] = fmaf(gw[k][j] - h[k][j] * coef, ir, o[k][j]);
      put_grads<EVEN>(p, key, row, unit_col<WARP>(k), o[k], mine);
    }
  }
  if (WARP) {  // the warps' shares, added in warp order
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < 8; ++j) sm[warp * 256 + j * 32 + lane] = acc[k][j];
      __syncthreads();
      float s = 0.f;
      for (int q = 0; q < kWarpRows; ++q) s += sm[q * 256 + threadIdx.x];
      const int64_t c = (k * 32 + lane) * 8 + warp;  // word j * 32 + lane holds column 8 lane + j
      if (c < p.cols) p.part[(int64_t)blockIdx.x * p.cols + c] = s;
    }
  } else {
#pragma unroll
    for (int k = 0; k < UPT; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t c = unit_col<WARP>(k) + j;
        if (c < p.cols) p.part[(int64_t)blockIdx.x * p.cols + c] = acc[k][j];
      }
  }
}

// ---------------------------------------------------------------------------
// Rows of 1025 to 8192 columns that 16-byte copies fit: each thread copies its own
// units of the rows ahead into shared memory (cp.async), `stages` rows deep, and
// is the only one to read them, so the row's one barrier is that of its sum.
// ---------------------------------------------------------------------------
constexpr int kStagesMost = 4;
constexpr int kStageBytes = 224 * 1024;  // of an SM's blocks together

__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the latest N groups have landed
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A unit in shared memory: 16-byte pieces of all threads side by side.
template <typename T>
__device__ __forceinline__ void unit_copy(unsigned char* at, int unit, int units, const T* from) {
#pragma unroll
  for (int q = 0; q < (int)sizeof(T) / 2; ++q)
    copy16(at + ((size_t)q * units + unit) * 16, reinterpret_cast<const unsigned char*>(from) + 16 * q);
}
__device__ __forceinline__ void unit_read(const unsigned char* at, int unit, int units, float (&v)[8], const float*) {
  const float4 a = *reinterpret_cast<const float4*>(at + (size_t)unit * 16);
  const float4 b = *reinterpret_cast<const float4*>(at + (size_t)(units + unit) * 16);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void unit_read(const unsigned char* at, int unit, int, float (&v)[8], const __nv_bfloat16*) {
  const uint4 a = *reinterpret_cast<const uint4*>(at + (size_t)unit * 16);
  const uint32_t r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(r[j] << 16);
    v[2 * j + 1] = __uint_as_float(r[j] & 0xffff0000u);
  }
}

template <typename TR, typename TB, int UPT, int STAGES>
__global__ void __launch_bounds__(512, 2) add_norm_bwd_ring_kernel(const BwdArgs<TR, TB> p) {
  let_next_start();
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float red[2][16];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  const int units = UPT * (int)blockDim.x;
  constexpr int per = 8 * (2 * (int)sizeof(TR) + (int)sizeof(TB));  // bytes of a unit: gh, h, g
  const size_t at_h = (size_t)units * 8 * sizeof(TR), at_g = 2 * at_h;
  const DropKey key = drop_key(p.drop);
  float acc[UPT][8], wv[UPT][8];
  int c[UPT];
  bool on[UPT];
#pragma unroll
  for (int k = 0; k < UPT; ++k) {
    c[k] = 8 * (k * (int)blockDim.x + tid);
    on[k] = c[k] < p.cols;
    load_w(p.w, c[k], p.cols, wv[k]);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[k][j] = 0.f;
  }
  auto fetch = [&](int64_t row, int s) {
    unsigned char* at = ring + (size_t)s * units * per;
    if (row < p.rows) {
#pragma unroll
      for (int k = 0; k < UPT; ++k)
        if (on[k]) {
          const int u = k * (int)blockDim.x + tid;
          if (p.gh) unit_copy(at, u, units, p.gh + row * p.cols + c[k]);
          unit_copy(at + at_h, u, units, p.h + row * p.cols + c[k]);
          unit_copy(at + at_g, u, units, p.g + row * p.cols + c[k]);
        }
    }
    copies_end();  // a group each time, so that the count of groups is the count of rows
  };
#pragma unroll
  for (int s = 0; s < STAGES; ++s) fetch((int64_t)blockIdx.x + (int64_t)s * gridDim.x, s);
  int s = 0, buf = 0;
  float nr = p.rms[blockIdx.x];
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, buf ^= 1) {
    const unsigned char* at = ring + (size_t)s * units * per;
    const float r = nr, ir = 1.0f / r;
    if (row + gridDim.x < p.rows) nr = p.rms[row + gridDim.x];
    copies_wait<STAGES - 1>();
    float gw[UPT][8], h[UPT][8];
    float d = 0.f;
#pragma unroll
    for (int k = 0; k < UPT; ++k)
      if (on[k]) {
        const int u = k * (int)blockDim.x + tid;
        unit_read(at + at_g, u, units, gw[k], p.g);
        unit_read(at + at_h, u, units, h[k], p.h);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          acc[k][j] = fmaf(gw[k][j] * ir, h[k][j], acc[k][j]);
          gw[k][j] *= wv[k][j];
          d = fmaf(gw[k][j], h[k][j], d);
        }
      }
    d = warp_sum(d);
    if (lane == 0) red[buf][warp] = d;
    __syncthreads();
    float t = lane < nw ? red[buf][lane & 15] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);  // 16 warps at most
    const float coef = __shfl_sync(0xffffffffu, t, 0) / ((float)p.cols * r * r);
#pragma unroll
    for (int k = 0; k < UPT; ++k)
      if (on[k]) {
        float o[8];
        if (p.gh) {
          unit_read(at, k * (int)blockDim.x + tid, units, o, p.gh);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = fmaf(gw[k][j] - h[k][j] * coef, ir, o[j]);
        put_grads<true>(p, key, row, c[k], o, nullptr);
      }
    fetch(row + (int64_t)STAGES * gridDim.x, s);  // into what this thread has just read
    s = s + 1 == STAGES ? 0 : s + 1;
  }
#pragma unroll
  for (int k = 0; k < UPT; ++k)
    if (on[k]) {
      float* q = p.part + (int64_t)blockIdx.x * p.cols + c[k];
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = acc[k][j];
    }
  copies_wait<0>();
}

// ---------------------------------------------------------------------------
// Longer rows: g and h are read twice (the second time from L2), and the block's
// share of gw is kept in shared memory (KEEP) or, past kKeepCols columns, in its row
// of partial sums.  Each unit is always the same thread's.
// ---------------------------------------------------------------------------
constexpr int kLongThreads = 512;
constexpr int64_t kKeepCols = 49152;  // 192 KB

template <typename TR, typename TB, bool EVEN, bool KEEP>
__global__ void __launch_bounds__(kLongThreads) add_norm_bwd_long_kernel(const BwdArgs<TR, TB> p) {
  let_next_start();
  extern __shared__ __align__(16) float keep[];  // [8][units]: value j of unit u at j * units + u
  __shared__ float red[2][32];
  __shared__ __align__(16) float sm[EVEN ? 1 : kLongThreads * 8];
  float* mine = sm + (EVEN ? 0 : (threadIdx.x >> 5) * 256);
  const int lane = threadIdx.x & 31;
  const int64_t units = (p.cols + 7) / 8;
  float* a = KEEP ? keep : p.part + (int64_t)blockIdx.x * p.cols;
  auto slot = [&](int64_t c, int j) -> int64_t { return KEEP ? j * units + c / 8 : c + j; };
  for (int64_t c = 8 * threadIdx.x; c < p.cols; c += 8 * kLongThreads)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < p.cols) a[slot(c, j)] = 0.f;
  const DropKey key = drop_key(p.drop);
  int buf = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, buf ^= 1) {
    const float r = p.rms[row], ir = 1.0f / r;
    const TB* gr = p.g + row * p.cols;
    const TR* hr = p.h + row * p.cols;
    float d = 0.f;
    for (int64_t c0 = 8 * (threadIdx.x & ~31); c0 < p.cols; c0 += 8 * kLongThreads) {
      const int64_t c = c0 + 8 * lane;
      float g[8], h[8], wv[8];
      get_unit<EVEN>(gr, c, p.cols, mine, g);
      get_unit<EVEN>(hr, c, p.cols, mine, h);
      load_w(p.w, c, p.cols, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (c + j < p.cols) a[slot(c, j)] = fmaf(g[j] * ir, h[j], a[slot(c, j)]);
        d = fmaf(g[j] * wv[j], h[j], d);
      }
    }
    const float coef = row_total<false>(d, red[buf]) / ((float)p.cols * r * r);
    for (int64_t c0 = 8 * (threadIdx.x & ~31); c0 < p.cols; c0 += 8 * kLongThreads) {
      const int64_t c = c0 + 8 * lane;
      float g[8], h[8], wv[8], o[8];
      get_unit<EVEN>(gr, c, p.cols, mine, g);
      get_unit<EVEN>(hr, c, p.cols, mine, h);
      load_w(p.w, c, p.cols, wv);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = 0.f;
      if (p.gh) get_unit<EVEN>(p.gh + row * p.cols, c, p.cols, mine, o);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = fmaf(g[j] * wv[j] - h[j] * coef, ir, o[j]);
      put_grads<EVEN>(p, key, row, c, o, mine);
    }
  }
  if (KEEP)
    for (int64_t c = 8 * threadIdx.x; c < p.cols; c += 8 * kLongThreads)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < p.cols) p.part[(int64_t)blockIdx.x * p.cols + c + j] = a[slot(c, j)];
}

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------
enum class Bwd { kWarp, kBlock, kRing, kLong };
struct BwdPlan {
  Bwd kind;
  int UPT, threads, stages, per_sm;
  size_t smem;
};
// `unit`: bytes of 8 columns of gh, h and g
BwdPlan bwd_plan(int64_t cols, bool even, size_t unit) {
  const int64_t U = (cols + 7) / 8;
  if (ck_pitch(cols) <= kWarpCols)
    return {Bwd::kWarp, ck_pitch(cols) <= 256 ? 1 : ck_pitch(cols) <= 512 ? 2 : 4, 32 * kWarpRows, 0, 4, 0};
  if (U > 1024) {
    const size_t keep = cols <= kKeepCols ? (size_t)U * 8 * sizeof(float) : 0;
    return {Bwd::kLong, 0, kLongThreads, 0, keep > 100 * 1024 ? 1 : 2, keep};
  }
  if (!even) {
    const int upt = U <= 256 ? 1 : 2;
    return {Bwd::kBlock, upt, (int)(((U + upt - 1) / upt + 31) / 32 * 32), 0, 2, 0};
  }
  const int upt = U <= 512 ? 1 : 2, threads = (int)(((U + upt - 1) / upt + 31) / 32 * 32);
  const size_t stage = (size_t)upt * threads * unit;
  int per_sm = 1024 / threads;
  per_sm = per_sm < 2 ? 2 : per_sm > 6 ? 6 : per_sm;
  while (per_sm > 1 && 2 * stage > (size_t)kStageBytes / per_sm) --per_sm;
  size_t s = (size_t)kStageBytes / per_sm / stage;
  s = s > kStagesMost ? kStagesMost : s;
  return {Bwd::kRing, upt, threads, (int)s, per_sm, s * stage};
}

// Blocks: as many as run at once (gw leaves as one row a block), no more than
// there are rows for.
int bwd_blocks(const BwdPlan& pl, int64_t rows) {
  const int64_t need = pl.kind == Bwd::kWarp ? (rows + kWarpRows - 1) / kWarpRows : rows;
  const int64_t most = pl.per_sm * (int64_t)num_sms();
  return (int)(need < most ? (need > 0 ? need : 1) : most);
}

template <typename K, typename P>
int go(K kern, int blocks, const BwdPlan& pl, size_t most, const P& p, cudaStream_t st) {
  // The limit on dynamic shared memory belongs to the kernel, not to the launch:
  // it is always set to the most that any width asks for, so that host threads
  // with other widths cannot lower it in between.
  if (most && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess)
    return fail(MHC_ERR_CUDA, "add_rmsnorm_bwd: cannot reserve %zu bytes of shared memory", most);
  kern<<<blocks, pl.threads, pl.smem, st>>>(p);
  return MHC_OK;
}

template <int UPT, typename TR, typename TB>
int go_ring(int blocks, const BwdPlan& pl, const BwdArgs<TR, TB>& p, cudaStream_t st) {
  constexpr size_t most = kStageBytes;
  if (pl.stages == 2) return go(add_norm_bwd_ring_kernel<TR, TB, UPT, 2>, blocks, pl, most, p, st);
  if (pl.stages == 3) return go(add_norm_bwd_ring_kernel<TR, TB, UPT, 3>, blocks, pl, most, p, st);
  return go(add_norm_bwd_ring_kernel<TR, TB, UPT, 4>, blocks, pl, most, p, st);
}

template <typename TR, typename TB>
int launch_bwd(BwdArgs<TR, TB> p, float* grad_weight, size_t workspace_bytes, cudaStream_t st) {
  const bool even = even_rows<TR>(p.gh, p.cols, p.cols) && even_rows<TR>(p.h, p.cols, p.cols) &&
                    even_rows<TB>(p.g, p.cols, p.cols) && even_rows<TR>(p.gr, p.cols, p.cols) &&
                    even_rows<TB>(p.gb, p.cols, p.cols);
  const BwdPlan pl = bwd_plan(p.cols, even, 8 * (2 * sizeof(TR) + sizeof(TB)));
  const int blocks = bwd_blocks(pl, p.rows);
  MHC_REQUIRE(p.part != nullptr && workspace_bytes >= (size_t)blocks * (size_t)p.cols * sizeof(float), MHC_ERR_WORKSPACE,
              "add_rmsnorm_bwd: workspace too small");
  int rc = MHC_OK;
  {
    ProfScope prof("add_rmsnorm_bwd", st);
#define MHC_GO(UPT, WARP)                                                                             \
  (even ? go(add_norm_bwd_kernel<TR, TB, UPT, WARP, true>, blocks, pl, 0, p, st)                      \
        : go(add_norm_bwd_kernel<TR, TB, UPT, WARP, false>, blocks, pl, 0, p, st))
    constexpr size_t keep = kKeepCols * sizeof(float);
    if (pl.kind == Bwd::kRing) rc = pl.UPT == 1 ? go_ring<1>(blocks, pl, p, st) : go_ring<2>(blocks, pl, p, st);
    else if (pl.kind == Bwd::kWarp) rc = pl.UPT == 1 ? MHC_GO(1, true) : pl.UPT == 2 ? MHC_GO(2, true) : MHC_GO(4, true);
    else if (pl.kind == Bwd::kBlock)
      rc = pl.UPT == 1 ? go(add_norm_bwd_kernel<TR, TB, 1, false, false>, blocks, pl, 0, p, st)
                       : go(add_norm_bwd_kernel<TR, TB, 2, false, false>, blocks, pl, 0, p, st);
    else if (pl.smem) rc = even ? go(add_norm_bwd_long_kernel<TR, TB, true, true>, blocks, pl, keep, p, st)
                                : go(add_norm_bwd_long_kernel<TR, TB, false, true>, blocks, pl, keep, p, st);
    else rc = even ? go(add_norm_bwd_long_kernel<TR, TB, true, false>, blocks, pl, 0, p, st)
                   : go(add_norm_bwd_long_kernel<TR, TB, false, false>, blocks, pl, 0, p, st);
#undef MHC_GO
    if (rc == MHC_OK) rc = check_launch("add_rmsnorm_bwd");
    if (rc) return rc;
  }
  ProfScope prof("add_rmsnorm_gw", st);
  launch_early(norm_gw_kernel, dim3((unsigned)((p.cols + 31) / 32)), dim3(256), 0, st, (const float*)p.part, grad_weight,
               blocks, p.cols);
  return check_launch("add_rmsnorm_gw");
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" size_t mhc_add_rmsnorm_bwd_workspace_bytes(int64_t rows, int64_t cols) {
  if (rows < 0 || cols < 1) return 0;
  // the plan depends on types and alignment too: enough for each
  int most = 1;
  for (size_t unit : {48, 64, 80, 96})
    for (bool even : {false, true}) {
      const int b = bwd_blocks(bwd_plan(cols, even, unit), rows);
      most = b > most ? b : most;
    }
  return (size_t)most * (size_t)cols * sizeof(float);
}

extern "C" int mhc_add_rmsnorm_bwd(const void* grad_hidden, const void* grad_out, const void* hidden, int32_t residual_bf16,
                                   int32_t branch_bf16, const float* weight, const float* rms, void* grad_residual,
                                   void* grad_branch, float* grad_weight, int64_t rows, int64_t cols, int32_t drop,
                                   const uint64_t* state, uint64_t seed, uint64_t position, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  const char* what = "add_rmsnorm_bwd";
  MHC_REQUIRE(rows >= 0 && cols >= 1, MHC_ERR_INVALID_ARG, "%s: rows must be >= 0 and cols >= 1 (got %lld x %lld)", what,
              (long long)rows, (long long)cols);
  MHC_REQUIRE(cols <= (1ll << 30) && rows < (1ll << 31), MHC_ERR_UNSUPPORTED, "%s: %lld x %lld values are too many", what,
              (long long)rows, (long long)cols);
  MHC_REQUIRE((reinterpret_cast<uintptr_t>(state) & 7) == 0, MHC_ERR_ALIGNMENT, "%s: state must be 8-byte aligned", what);
  const int rc = check_drop(what, drop);
  if (rc) return rc;
  MHC_REQUIRE_PTR(grad_weight);
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    cudaMemsetAsync(grad_weight, 0, (size_t)cols * sizeof(float), st);
    return check_launch(what);
  }
  MHC_REQUIRE_PTR(grad_out);
  MHC_REQUIRE_PTR(hidden);
  MHC_REQUIRE_PTR(weight);
  MHC_REQUIRE_PTR(rms);
  MHC_REQUIRE_PTR(grad_residual);
  auto run = [&](auto* r, auto* b) -> int {
    using TR = std::remove_pointer_t<decltype(r)>;
    using TB = std::remove_pointer_t<decltype(b)>;
    const BwdArgs<TR, TB> p = {(const TR*)grad_hidden, (const TB*)grad_out, (const TR*)hidden, weight, rms, (TR*)grad_residual,
                               (TB*)grad_branch, (float*)workspace, rows, cols, drop_source(state, seed, position, drop)};
    return launch_bwd(p, grad_weight, workspace_bytes, st);
  };
  if (residual_bf16)
    return branch_bf16 ? run((__nv_bfloat16*)nullptr, (__nv_bfloat16*)nullptr) : run((__nv_bfloat16*)nullptr, (float*)nullptr);
  return branch_bf16 ? run((float*)nullptr, (__nv_bfloat16*)nullptr) : run((float*)nullptr, (float*)nullptr);
}
