// Backward of the residual addition with RMSNorm (add_norm.cu), from the hidden
// state h that the forward returned:
//   gi = gh + (g w - h D / (C r^2)) / r,   D = sum_c g w h,   r = sqrt(mean h^2 + eps)
//   g_residual = gi,   g_branch = gi with the forward's dropout,   gw = sum over rows of g h / r
// gh is the gradient that reaches h by other ways (the residual stream's), g the
// output's.  A block (or warp) walks every (its count)-th row and keeps its
// columns' share of gw in registers; the shares leave as one row a block and are
// added in block order: no atomics, the same bits every time.
#include "dropout.cuh"
#include "rows.cuh"
#include "tma.cuh"
#include "vec8.cuh"

namespace mhc {
namespace {

struct BwdArgs {
  const void* gh;  // nullable: zero
  const void *g, *h;
  const float *w, *rms;
  void *gr, *gb;  // gb nullable: not wanted
  float* part;
  int64_t rows, cols;
  bool res16, branch16;
  DropSource drop;
};

// gi of a unit that starts at element i -> both gradients
template <typename TR, typename TB>
__device__ __forceinline__ void put_grads(const BwdArgs& p, const DropKey& key, int64_t i, const V8& gi) {
  v8_save(static_cast<TR*>(p.gr) + i, gi);
  if (p.gb) {
    V8 o = gi;
    if (p.drop.drop) {
      float f[8];
      v8_spread(gi, f);
      drop_apply(drop_group(key, (uint64_t)i / kDropGroup), p.drop.drop, p.drop.scale, f);
      o = v8_gather(f);
    }
    v8_save(static_cast<TB*>(p.gb) + i, o);
  }
}
__device__ __forceinline__ void put_grads_any(const BwdArgs& p, const DropKey& key, int64_t row, int64_t c, float (&o)[8],
                                              float* mine) {
  save_any(p.gr, p.res16, row, c, p.cols, mine, o);
  if (p.gb) {
    if (p.drop.drop) drop_apply_at(key, (uint64_t)row * (uint64_t)p.cols + (uint64_t)c, p.drop.drop, p.drop.scale, o);
    save_any(p.gb, p.branch16, row, c, p.cols, mine, o);
  }
}

// The warps' shares of the weight's gradient, added in warp order
template <int UPT>
__device__ __forceinline__ void put_warp_parts(const BwdArgs& p, const float (&acc)[UPT][8], float* sm) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
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
}

// gi of a unit at its row's edge
template <typename TR, typename TB>
__device__ __forceinline__ void put_grads_edge(const BwdArgs& p, const DropKey& key, int64_t i, V8 gi, int c, int cols) {
  V8 o = gi;
  v8_save_inside(static_cast<TR*>(p.gr) + i, o, c, cols);
  if (p.gb) {
    if (p.drop.drop) {
      float f[8];
      v8_spread(gi, f);
      drop_apply(drop_group(key, (uint64_t)i / kDropGroup), p.drop.drop, p.drop.scale, f);
      gi = v8_gather(f);
    }
    v8_save_inside(static_cast<TB*>(p.gb) + i, gi, c, cols);
  }
}

// ---------------------------------------------------------------------------
// Rows of at most 1024 columns, one a warp ([65536, 1000] fp32 169 us, 6.2 TB/s; [65536, 256]
// fp32 residual, bf16 branch 56 us, 4.8), whose rows are a multiple of 8 apart.  EVEN:
// whole units; otherwise units of the tensor's own alignment (vec8.cuh): a warp's rows
// all start at the same place of a unit, and its sums go by column through shared memory.
// ---------------------------------------------------------------------------
template <typename TR, typename TB, int UPT, bool EVEN>
__global__ void __launch_bounds__(32 * kWarpRows) add_norm_bwd_warp_kernel(const BwdArgs p) {
  let_next_start();
  __shared__ float sm[EVEN ? kWarpRows * 256 : kWarpRows * 256 * UPT];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, cols = (int)p.cols;
  const int64_t row0 = (int64_t)blockIdx.x * kWarpRows + warp, total = p.rows * cols;
  const int shift = EVEN ? 0 : (int)((row0 * cols) & 7), c0 = 8 * lane - shift;
  const DropKey key = drop_key(p.drop);
  V8 acc[UPT];
#pragma unroll
  for (int k = 0; k < UPT; ++k) acc[k] = v8_zero();
  for (int64_t row = row0; row < p.rows; row += (int64_t)gridDim.x * kWarpRows) {
    const int64_t at = row * cols + c0;
    Raw8<TB> g[UPT];
    Raw8<TR> h[UPT], o[UPT];
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      g[k].zero();
      h[k].zero();
      o[k].zero();
      if (c0 + k * 256 < cols && (EVEN || at + k * 256 + 8 <= total)) {
        g[k].load(static_cast<const TB*>(p.g) + at + k * 256);
        h[k].load(static_cast<const TR*>(p.h) + at + k * 256);
        if (p.gh) o[k].load(static_cast<const TR*>(p.gh) + at + k * 256);
      }
    }
    const float r = p.rms[row], ir = 1.0f / r;
    V8 gw[UPT], hv[UPT], ov[UPT];
    float2 d2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      const int c = c0 + k * 256;
      V8 gv = g[k].values();
      hv[k] = h[k].values();
      ov[k] = o[k].values();
      if (!EVEN && c < cols && v8_edge(c, cols)) {
        if (at + k * 256 + 8 > total) {  // the tensor's last
          const int64_t left = total - at - k * 256;
          gv = v8_load_part(static_cast<const TB*>(p.g) + at + k * 256, left);
          hv[k] = v8_load_part(static_cast<const TR*>(p.h) + at + k * 256, left);
          if (p.gh) ov[k] = v8_load_part(static_cast<const TR*>(p.gh) + at + k * 256, left);
        }
        gv = v8_inside(gv, c, cols);
        hv[k] = v8_inside(hv[k], c, cols);
      }
      acc[k] = v8_fma(v8_scale(gv, ir), hv[k], acc[k]);
      gw[k] = c < cols ? v8_mul(gv, EVEN ? v8_weights(p.w + c) : v8_weights_inside(p.w, c, cols)) : v8_zero();
      d2 = v8_dot(gw[k], hv[k], d2);
    }
    const float coef = -warp_sum(d2.x + d2.y) / ((float)cols * r * r);
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      const int c = c0 + k * 256;
      if (c >= cols) continue;
      const V8 gi = v8_fma(v8_fma(hv[k], coef, gw[k]), ir, ov[k]);
      if (!EVEN && v8_edge(c, cols)) put_grads_edge<TR, TB>(p, key, at + k * 256, gi, c, cols);
      else put_grads<TR, TB>(p, key, at + k * 256, gi);
    }
  }
  if (EVEN) {
    float parts[UPT][8];
#pragma unroll
    for (int k = 0; k < UPT; ++k) v8_spread(acc[k], parts[k]);
    put_warp_parts<UPT>(p, parts, sm);
  } else {
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      float f[8];
      v8_spread(acc[k], f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = c0 + k * 256 + j;
        if (c >= 0 && c < cols) sm[warp * (256 * UPT) + c] = f[j];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += 32 * kWarpRows) {
      float s = 0.f;
      for (int q = 0; q < kWarpRows; ++q) s += sm[q * (256 * UPT) + c];
      p.part[(int64_t)blockIdx.x * cols + c] = s;
    }
  }
}

// ---------------------------------------------------------------------------
// Rows of 1025 to 8192 columns, of any width: units are the tensor's own groups of
// eight values, so that every access is aligned wherever a row starts; a row's first
// and last unit may belong to its neighbours in part.  A block's rows are a multiple
// of 8 apart (or of fewer, as the width allows): they all start at the same place of a
// unit, and a thread keeps its columns, with their weights and sums, over all of them.
// The rows ahead are copied into shared memory (cp.async), `stages` deep, each warp
// what it will read itself, so the row's one barrier is that of its sum.  Copies of
// 512 consecutive bytes a warp and 16-byte pieces stored crosswise: a 32-byte unit a
// lane met every sector twice on its way in ([8192, 4096], fp32 residual, bf16 branch,
// 122 us).  Now 82 us with dropout, 6.5 TB/s; [8192, 7168] 147 us; [8192, 4096] bf16 48 us
// without and 72 us with dropout, where issue slots bound it (70%).
// ---------------------------------------------------------------------------
constexpr int kStagesMost = 4;
constexpr int kStageBytes = 224 * 1024;  // of an SM's blocks together

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_part(uint32_t to, const void* from, uint32_t bytes) {  // zeros behind
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the latest n - 1 groups have landed, 1 <= n <= 4
__device__ __forceinline__ void copies_wait(int n) {
  if (n == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else if (n == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (n == 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// A warp's 256 consecutive values: its lanes copy pieces of 16 bytes side by side.
// need: values that the row wants (a piece that holds none is left out); left: those
// that the tensor has from the warp's first on.
template <bool EVEN, typename T>
__device__ __forceinline__ void span_copy(uint32_t to, const T* from, int need, int left) {
  constexpr int per = 16 / (int)sizeof(T);  // values of a piece
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int q = 0; q < (int)sizeof(T) / 2; ++q) {
    const int piece = 32 * q + lane, e = piece * per;
    const uint32_t at = to + 16u * (sizeof(T) == 4 ? piece ^ ((piece >> 3) & 1) : piece);
    if (e < need && (EVEN || e < left)) {
      if (EVEN || e + per <= left) copy16(at, from + e);
      else copy_part(at, from + e, (uint32_t)(left - e) * sizeof(T));
    }
  }
}
// The lane's unit of them
__device__ __forceinline__ V8 span_read(const unsigned char* at, const float*) {
  const int lane = threadIdx.x & 31, b = (lane >> 2) & 1;
  const float4 x = *reinterpret_cast<const float4*>(at + 16 * ((2 * lane) ^ b));
  const float4 y = *reinterpret_cast<const float4*>(at + 16 * ((2 * lane + 1) ^ b));
  V8 v;
  v.a[0] = make_float2(x.x, x.y);
  v.a[1] = make_float2(x.z, x.w);
  v.a[2] = make_float2(y.x, y.y);
  v.a[3] = make_float2(y.z, y.w);
  return v;
}
__device__ __forceinline__ V8 span_read(const unsigned char* at, const __nv_bfloat16*) {
  return v8_of(*reinterpret_cast<const uint4*>(at + 16 * (threadIdx.x & 31)));
}
// Blocks of up to 576 threads twice an SM (56 registers a thread), larger ones once.
constexpr int ring_blocks(int most) { return most > 576 ? 1 : 2; }

// EVEN: whole units (cols % 8 == 0).  One unit a thread: two (half the threads, twice
// the registers) took as long within 3%.
template <typename TR, typename TB, bool EVEN, int MOST>
__global__ void __launch_bounds__(MOST, ring_blocks(MOST)) add_norm_bwd_ring_kernel(const BwdArgs p, int stages) {
  let_next_start();
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float red[2][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5, cols = (int)p.cols;
  const int shift = EVEN ? 0 : (int)(((int64_t)blockIdx.x * cols) & 7);
  const int c = 8 * tid - shift;  // the unit's first column
  const bool on = c < cols, edge = !EVEN && on && v8_edge(c, cols);
  // a stage: gh, h, g of all warps
  const uint32_t span_r = 256u * sizeof(TR), span_b = 256u * sizeof(TB), at_h = nw * span_r, at_g = 2 * at_h;
  const uint32_t stage = at_g + nw * span_b, ring_end = stages * stage;
  const DropKey key = drop_key(p.drop);
  V8 acc = v8_zero();
  const V8 wv = v8_weights_inside(p.w, c, cols);
  const int64_t hop = (int64_t)gridDim.x * cols, total = p.rows * cols;
  const int need = shift + cols - 256 * warp;
  int64_t ahead = (int64_t)blockIdx.x * cols - shift + 256 * warp;  // element of the warp's next copies
  const uint32_t to_r = smem_u32(ring) + warp * span_r, to_b = smem_u32(ring) + at_g + warp * span_b;
  auto fetch = [&](uint32_t s) {
    if (ahead < total) {
      const int left = EVEN ? 0 : (int)min(total - ahead, (int64_t)1 << 20);
      if (p.gh) span_copy<EVEN>(to_r + s, static_cast<const TR*>(p.gh) + ahead, need, left);
      span_copy<EVEN>(to_r + at_h + s, static_cast<const TR*>(p.h) + ahead, need, left);
      span_copy<EVEN>(to_b + s, static_cast<const TB*>(p.g) + ahead, need, left);
    }
    ahead += hop;
    copies_end();  // a group each time, so that the count of groups is the count of rows
  };
  for (int s = 0; s < stages; ++s) fetch(s * stage);
  uint32_t s = 0;
  int buf = 0;
  int64_t at = (int64_t)blockIdx.x * cols + c;
  // 1 / rms, rounded to nearest since it is common to a row's terms of gw: 32 of the block's
  // rows at once, one a lane (a division a row in every thread: [8192, 2048] bf16 33.9 us, so 33.0)
  float irs = 0.f;
  int turn = 0;
  const float share = 1.0f / (float)cols;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, buf ^= 1, at += hop) {
    if (turn == 0) {
      const int64_t mine = row + (int64_t)lane * gridDim.x;
      if (mine < p.rows) irs = 1.0f / p.rms[mine];
    }
    const float ir = __shfl_sync(0xffffffffu, irs, turn);
    turn = (turn + 1) & 31;
    copies_wait(stages);
    __syncwarp();  // the other lanes' too
    const unsigned char* from = ring + s + warp * span_r;
    V8 g = v8_zero(), h = g;
    float2 d2 = make_float2(0.f, 0.f);
    if (on) {
      g = span_read(ring + s + at_g + warp * span_b, (const TB*)nullptr);
      h = span_read(from + at_h, (const TR*)nullptr);
      if (edge) {
        g = v8_inside(g, c, cols);
        h = v8_inside(h, c, cols);
      }
      acc = v8_fma(v8_scale(g, ir), h, acc);
      g = v8_mul(g, wv);
      d2 = v8_dot(g, h, d2);
    }
    const float d = warp_sum(d2.x + d2.y);
    if (lane == 0) red[buf][warp] = d;
    __syncthreads();
    const float coef = -warp_sum(lane < nw ? red[buf][lane] : 0.f) * share * (ir * ir);
    if (on) {
      const V8 o = p.gh ? span_read(from, (const TR*)nullptr) : v8_zero();
      const V8 gi = v8_fma(v8_fma(h, coef, g), ir, o);
      if (edge) put_grads_edge<TR, TB>(p, key, at, gi, c, cols);
      else put_grads<TR, TB>(p, key, at, gi);
    }
    __syncwarp();  // everyone has read what is now copied over
    fetch(s);
    s = s + stage == ring_end ? 0 : s + stage;
  }
  if (on) v8_save_inside(p.part + (int64_t)blockIdx.x * cols + c, acc, c, cols);
  copies_wait(1);
}

// ---------------------------------------------------------------------------
// Longer rows: g and h are read twice (the second time from L2), and the block's
// share of gw is kept in shared memory (KEEP) or, past kKeepCols columns, in its row
// of partial sums.  Each unit is always the same thread's.  Bound by latency, one or two
// rows an SM: [2000, 16384] bf16 68 us, 3.8 TB/s, [1000, 28672] fp32 residual 102 us, 4.5.
// ---------------------------------------------------------------------------
constexpr int kLongThreads = 512;
constexpr int64_t kKeepCols = 49152;  // 192 KB

__device__ __forceinline__ V8 sums_of(const float4& x, const float4& y) {
  V8 v;
  v.a[0] = make_float2(x.x, x.y);
  v.a[1] = make_float2(x.z, x.w);
  v.a[2] = make_float2(y.x, y.y);
  v.a[3] = make_float2(y.z, y.w);
  return v;
}

template <typename TR, typename TB, bool EVEN>
__global__ void __launch_bounds__(1024) add_norm_bwd_long_kernel(const BwdArgs p) {
  let_next_start();
  extern __shared__ __align__(16) unsigned char keep[];  // halves of a unit's eight sums apart
  __shared__ float red[2][32];
  const int cols = (int)p.cols;
  const int shift = EVEN ? 0 : (int)(((int64_t)blockIdx.x * cols) & 7), U = (shift + cols + 7) / 8;
  const int64_t total = p.rows * cols;
  float4* lo = reinterpret_cast<float4*>(keep);
  float4* hi = lo + U;
  for (int u = threadIdx.x; u < U; u += blockDim.x) lo[u] = hi[u] = make_float4(0.f, 0.f, 0.f, 0.f);
  const DropKey key = drop_key(p.drop);
  auto weights = [&](int c) { return EVEN ? v8_weights(p.w + c) : v8_weights_inside(p.w, c, cols); };
  auto load = [&](const auto* from, int64_t i) -> V8 {  // the unit at element i
    using T = std::remove_const_t<std::remove_pointer_t<decltype(from)>>;
    if (!EVEN && i + 8 > total) return v8_load_part(from + i, total - i);
    Raw8<T> q;
    q.load(from + i);
    return q.values();
  };
  int buf = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, buf ^= 1) {
    const float r = p.rms[row], ir = 1.0f / r;
    const int64_t at = row * cols - shift;
    float2 d2 = make_float2(0.f, 0.f);
#pragma unroll 2
    for (int u = threadIdx.x; u < U; u += blockDim.x) {
      const int c = 8 * u - shift;
      V8 gv = load(static_cast<const TB*>(p.g), at + 8 * u), hv = load(static_cast<const TR*>(p.h), at + 8 * u);
      if (!EVEN && v8_edge(c, cols)) {
        gv = v8_inside(gv, c, cols);
        hv = v8_inside(hv, c, cols);
      }
      const V8 a = v8_fma(v8_scale(gv, ir), hv, sums_of(lo[u], hi[u]));
      lo[u] = make_float4(a.a[0].x, a.a[0].y, a.a[1].x, a.a[1].y);
      hi[u] = make_float4(a.a[2].x, a.a[2].y, a.a[3].x, a.a[3].y);
      d2 = v8_dot(v8_mul(gv, weights(c)), hv, d2);
    }
    const float coef = -row_total<false>(d2.x + d2.y, red[buf]) / ((float)cols * r * r);
#pragma unroll 2
    for (int u = threadIdx.x; u < U; u += blockDim.x) {
      const int c = 8 * u - shift;
      const V8 gw = v8_mul(load(static_cast<const TB*>(p.g), at + 8 * u), weights(c));
      const V8 o = p.gh ? load(static_cast<const TR*>(p.gh), at + 8 * u) : v8_zero();
      const V8 gi = v8_fma(v8_fma(load(static_cast<const TR*>(p.h), at + 8 * u), coef, gw), ir, o);
      if (!EVEN && v8_edge(c, cols)) put_grads_edge<TR, TB>(p, key, at + 8 * u, gi, c, cols);
      else put_grads<TR, TB>(p, key, at + 8 * u, gi);
    }
  }
  for (int u = threadIdx.x; u < U; u += blockDim.x) {
    V8 a = sums_of(lo[u], hi[u]);
    float* to = p.part + (int64_t)blockIdx.x * cols - shift + 8 * u;
    if (EVEN) v8_save(to, a);
    else v8_save_inside(to, a, 8 * u - shift, cols);
  }
}

// ---------------------------------------------------------------------------
// Any row: through shared memory, types by a branch.  In registers up to 8192 columns:
// ---------------------------------------------------------------------------
constexpr int any_threads(int UPT, bool WARP) { return WARP || UPT == 1 ? 256 : 512; }

template <int UPT, bool WARP>
__global__ void __launch_bounds__(any_threads(UPT, WARP)) add_norm_bwd_any_kernel(const BwdArgs p) {
  let_next_start();
  __shared__ float red[2][32];
  __shared__ __align__(16) float sm[any_threads(UPT, WARP) * 8];
  const int warp = threadIdx.x >> 5;
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
    float gw[UPT][8], h[UPT][8];
    float d = 0.f;
#pragma unroll
    for (int k = 0; k < UPT; ++k) {
      const int64_t c = unit_col<WARP>(k);
      load_any(p.g, p.branch16, row, c, p.cols, mine, gw[k]);
      load_any(p.h, p.res16, row, c, p.cols, mine, h[k]);
      float wv[8];
      load_w(p.w, c, p.cols, wv);
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
      const int64_t c = unit_col<WARP>(k);
      float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (p.gh) load_any(p.gh, p.res16, row, c, p.cols, mine, o);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = fmaf(gw[k][j] - h[k][j] * coef, ir, o[j]);
      put_grads_any(p, key, row, c, o, mine);
    }
  }
  if (WARP) {
    put_warp_parts<UPT>(p, acc, sm);
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

template <bool KEEP>
__global__ void __launch_bounds__(kLongThreads) add_norm_bwd_long_any_kernel(const BwdArgs p) {
  let_next_start();
  extern __shared__ __align__(16) unsigned char keep[];  // [8][units] floats: value j of unit u at j * units + u
  __shared__ float red[2][32];
  __shared__ __align__(16) float sm[kLongThreads * 8];
  float* mine = sm + (threadIdx.x >> 5) * 256;
  const int lane = threadIdx.x & 31;
  const int64_t units = (p.cols + 7) / 8;
  float* a = KEEP ? reinterpret_cast<float*>(keep) : p.part + (int64_t)blockIdx.x * p.cols;
  auto slot = [&](int64_t c, int j) -> int64_t { return KEEP ? j * units + c / 8 : c + j; };
  for (int64_t c = 8 * threadIdx.x; c < p.cols; c += 8 * kLongThreads)
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c + j < p.cols) a[slot(c, j)] = 0.f;
  const DropKey key = drop_key(p.drop);
  int buf = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, buf ^= 1) {
    const float r = p.rms[row], ir = 1.0f / r;
    float d = 0.f;
    for (int64_t c0 = 8 * (threadIdx.x & ~31); c0 < p.cols; c0 += 8 * kLongThreads) {
      const int64_t c = c0 + 8 * lane;
      float g[8], h[8], wv[8];
      load_any(p.g, p.branch16, row, c, p.cols, mine, g);
      load_any(p.h, p.res16, row, c, p.cols, mine, h);
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
      float g[8], h[8], wv[8], o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      load_any(p.g, p.branch16, row, c, p.cols, mine, g);
      load_any(p.h, p.res16, row, c, p.cols, mine, h);
      load_w(p.w, c, p.cols, wv);
      if (p.gh) load_any(p.gh, p.res16, row, c, p.cols, mine, o);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = fmaf(g[j] * wv[j] - h[j] * coef, ir, o[j]);
      put_grads_any(p, key, row, c, o, mine);
    }
  }
  if (KEEP)
    for (int64_t c = 8 * threadIdx.x; c < p.cols; c += 8 * kLongThreads)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < p.cols) p.part[(int64_t)blockIdx.x * p.cols + c + j] = a[slot(c, j)];
}

// gw[c] = sum of part[0..blocks)[c]: 32 columns a block, a warp every 32nd partial row, so
// that few loads wait on one another (8 warps a block: 9.3 us for 296 rows of 4096).
__global__ void __launch_bounds__(1024)
    sum_parts_kernel(const float* __restrict__ part, float* __restrict__ gw, int blocks, int64_t cols) {
  __shared__ float s[32][32];
  wait_for_previous();
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float t = 0.f;
  if (c < cols)
#pragma unroll 8
    for (int b = q; b < blocks; b += 32) t += part[(int64_t)b * cols + c];
  s[q][lane] = t;
  __syncthreads();
  if (q == 0 && c < cols) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) a += s[k][lane];
    gw[c] = a;
  }
}

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------
enum class Bwd { kWarp, kRing, kLong, kAny, kAnyWarp, kAnyLong };
struct BwdPlan {
  Bwd kind;
  int UPT, threads, stages, per_sm;
  size_t smem;
};
// aligned: wide accesses fit the tensors' starts, aligned_w: the weights' and the sums'
// too; `unit`: bytes of 8 columns of gh, h and g
BwdPlan bwd_plan(int64_t rows, int64_t cols, bool aligned, bool aligned_w, size_t unit) {
  const int64_t U = (cols + 7) / 8, spread = cols % 8 ? U + 1 : U;  // units of a row wherever it starts
  const bool fit = aligned && (cols % 8 != 0 || aligned_w);
  if (fit && spread <= 128)
    return {Bwd::kWarp, spread <= 32 ? 1 : spread <= 64 ? 2 : 4, 32 * kWarpRows, 0, 4, 0};
  if (aligned && spread <= 1024) {
    const int threads = (int)((spread + 31) / 32 * 32);
    const size_t stage = threads * unit;
    int per_sm = 1152 / threads;
    per_sm = per_sm > 6 ? 6 : per_sm < 1 ? 1 : per_sm;
    while (per_sm > 1 && 2 * stage > (size_t)kStageBytes / per_sm) --per_sm;
    // few rows: half the blocks of wide rows, twice the depth (with the weight's sums, cold:
    // [300, 4096] fp32 16.4 us against 18.4, [1001, 4097] fp32 26.6 against 27.2, [1000, 2560]
    // bf16 18.4 against 20.5, [1100, 4600] bf16 24.6 against 26.6, fp32 residual and bf16 branch
    // [1000, 3001] 24.6 against 25.5; [300, 4096] bf16 and [1100, 4096] fp32 the same)
    if (threads > 288 && rows < 4 * per_sm * (int64_t)num_sms()) per_sm = 1;
    size_t s = (size_t)kStageBytes / per_sm / stage;
    s = s > kStagesMost ? kStagesMost : s;
    return {Bwd::kRing, 1, threads, (int)s, per_sm, s * stage};
  }
  if (U > 1024) {
    const size_t keep = cols <= kKeepCols ? (size_t)spread * 8 * sizeof(float) : 0;
    const int per_sm = keep > 100 * 1024 ? 1 : 2;
    if (fit && keep) return {Bwd::kLong, 0, 1024 / per_sm, 0, per_sm, keep};
    return {Bwd::kAnyLong, 0, kLongThreads, 0, per_sm, keep};
  }
  if (ck_pitch(cols) <= kWarpCols)
    return {Bwd::kAnyWarp, ck_pitch(cols) <= 256 ? 1 : ck_pitch(cols) <= 512 ? 2 : 4, 32 * kWarpRows, 0, 4, 0};
  const int upt = U <= 256 ? 1 : 2;
  return {Bwd::kAny, upt, (int)(((U + upt - 1) / upt + 31) / 32 * 32), 0, 2, 0};
}

// Blocks: as many as run at once (gw leaves as one row a block), no more than
// there are rows for; a block's rows in units start at one place of them.
int bwd_blocks(const BwdPlan& pl, int64_t rows, int64_t cols) {
  const bool warp = pl.kind == Bwd::kWarp || pl.kind == Bwd::kAnyWarp;
  const int64_t need = warp ? (rows + kWarpRows - 1) / kWarpRows : rows;
  int64_t most = pl.per_sm * (int64_t)num_sms();
  if (pl.kind == Bwd::kRing || pl.kind == Bwd::kLong) {
    const int64_t apart = cols % 2 ? 8 : cols % 4 ? 4 : cols % 8 ? 2 : 1;
    most = most < apart ? apart : most / apart * apart;
  }
  return (int)(need < most ? (need > 0 ? need : 1) : most);
}

// The limit on dynamic shared memory belongs to the kernel, not to the launch: it is
// always set to the most that any width asks for, so that host threads with other
// widths cannot lower it in between.
template <typename K>
int allow(K kern, size_t most) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) == cudaSuccess
             ? MHC_OK
             : fail(MHC_ERR_CUDA, "add_rmsnorm_bwd: cannot reserve %zu bytes of shared memory", most);
}

template <typename TR, typename TB>
int launch_bwd(const BwdArgs& p, float* grad_weight, size_t workspace_bytes, cudaStream_t st) {
  const bool aligned = even_rows<TR>(p.gh, 8, 8) && even_rows<TR>(p.h, 8, 8) && even_rows<TB>(p.g, 8, 8) &&
                       even_rows<TR>(p.gr, 8, 8) && even_rows<TB>(p.gb, 8, 8);
  const bool whole = p.cols % 8 == 0;
  const BwdPlan pl = bwd_plan(p.rows, p.cols, aligned, even_rows<float>(p.w, 8, 8) && even_rows<float>(p.part, 8, 8),
                              8 * (2 * sizeof(TR) + sizeof(TB)));
  const int blocks = bwd_blocks(pl, p.rows, p.cols);
  MHC_REQUIRE(p.part != nullptr && workspace_bytes >= (size_t)blocks * (size_t)p.cols * sizeof(float), MHC_ERR_WORKSPACE,
              "add_rmsnorm_bwd: workspace too small");
  constexpr size_t keep = (kKeepCols + 8) * sizeof(float);
  int rc = MHC_OK;
  void (*ring)(const BwdArgs, int) = nullptr;
  void (*plain)(const BwdArgs) = nullptr;
  {
    ProfScope prof("add_rmsnorm_bwd", st);
#define MHC_GO(KERN, ...) KERN<<<blocks, pl.threads, pl.smem, st>>>(__VA_ARGS__)
    switch (pl.kind) {
      case Bwd::kWarp:
        if (whole) {
          if (pl.UPT == 1) MHC_GO((add_norm_bwd_warp_kernel<TR, TB, 1, true>), p);
          else if (pl.UPT == 2) MHC_GO((add_norm_bwd_warp_kernel<TR, TB, 2, true>), p);
          else MHC_GO((add_norm_bwd_warp_kernel<TR, TB, 4, true>), p);
        } else {
          if (pl.UPT == 1) MHC_GO((add_norm_bwd_warp_kernel<TR, TB, 1, false>), p);
          else if (pl.UPT == 2) MHC_GO((add_norm_bwd_warp_kernel<TR, TB, 2, false>), p);
          else MHC_GO((add_norm_bwd_warp_kernel<TR, TB, 4, false>), p);
        }
        break;
      case Bwd::kRing:
        if (pl.threads <= 576) ring = whole ? add_norm_bwd_ring_kernel<TR, TB, true, 576> : add_norm_bwd_ring_kernel<TR, TB, false, 576>;
        else ring = whole ? add_norm_bwd_ring_kernel<TR, TB, true, 1024> : add_norm_bwd_ring_kernel<TR, TB, false, 1024>;
        rc = allow(ring, kStageBytes);
        if (rc) return rc;
        MHC_GO(ring, p, pl.stages);
        break;
      case Bwd::kLong:
        plain = whole ? add_norm_bwd_long_kernel<TR, TB, true> : add_norm_bwd_long_kernel<TR, TB, false>;
        rc = allow(plain, keep);
        if (rc) return rc;
        MHC_GO(plain, p);
        break;
      case Bwd::kAnyWarp:
        if (pl.UPT == 1) MHC_GO((add_norm_bwd_any_kernel<1, true>), p);
        else if (pl.UPT == 2) MHC_GO((add_norm_bwd_any_kernel<2, true>), p);
        else MHC_GO((add_norm_bwd_any_kernel<4, true>), p);
        break;
      case Bwd::kAny:
        if (pl.UPT == 1) MHC_GO((add_norm_bwd_any_kernel<1, false>), p);
        else MHC_GO((add_norm_bwd_any_kernel<2, false>), p);
        break;
      case Bwd::kAnyLong:
        if (pl.smem) {
          rc = allow(add_norm_bwd_long_any_kernel<true>, keep);
          if (rc) return rc;
          MHC_GO(add_norm_bwd_long_any_kernel<true>, p);
        } else {
          MHC_GO(add_norm_bwd_long_any_kernel<false>, p);
        }
    }
#undef MHC_GO
    rc = check_launch("add_rmsnorm_bwd");
    if (rc) return rc;
  }
  ProfScope prof("add_rmsnorm_gw", st);
  launch_early(sum_parts_kernel, dim3((unsigned)((p.cols + 31) / 32)), dim3(1024), 0, st, (const float*)p.part, grad_weight,
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
    for (int way = 0; way < 3; ++way) {
      const int b = bwd_blocks(bwd_plan(rows, cols, way >= 1, way == 2, unit), rows, cols);
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
    const BwdArgs p = {grad_hidden, grad_out, hidden, weight, rms, grad_residual, grad_branch, (float*)workspace, rows, cols,
                       residual_bf16 != 0, branch_bf16 != 0, drop_source(state, seed, position, drop)};
    return launch_bwd<TR, TB>(p, grad_weight, workspace_bytes, st);
  };
  if (residual_bf16)
    return branch_bf16 ? run((__nv_bfloat16*)nullptr, (__nv_bfloat16*)nullptr) : run((__nv_bfloat16*)nullptr, (float*)nullptr);
  return branch_bf16 ? run((float*)nullptr, (__nv_bfloat16*)nullptr) : run((float*)nullptr, (float*)nullptr);
}
