// Log probabilities of given tokens, with entropy and the most likely
// alternatives, and the gradient of the logits.
//
// With m = max x, s = sum exp(x - m) over a row of logits:
//   log p_j = x_j - m - ln s,   H = ln s + sum exp(x - m) (m - x) / s
// (both terms of H are >= 0: nothing cancels).  One pass over the row: a thread
// keeps a running maximum, sum of e = exp(x - m) and sum of e (x - m), and rescales
// them when its maximum moves.  x - m is formed before it is scaled to base 2, so
// the largest value has e = 1 to the bit: s >= 1, no log probability is above 0 and
// no entropy below.  -inf is read as -2^127, so that the forward's products need no
// check: it has e = 0 and a finite x - m.  (The gradient multiplies x - m by a factor of
// any size and does check.)  Rows whose maximum is past 1e38 (of masks alone, or next to
// overflow) are scanned again value by value with those checks.  A row of nothing but
// -inf has s = 0.
//
// The k most likely, ties to the lowest index, in the same pass: every thread also
// notes the maximum of each of its 32-value segments.  The k-th largest of the
// maxima of 2 k or more groups of lanes bounds the k-th largest value from below, so
// only segments whose maximum reaches it are read again (about k of them), and what
// reaches it there is ranked by counting.  Where many values tie, or too few are
// finite, the k are taken one after the other instead.
#include <cooperative_groups.h>

#include "checkpoint8.cuh"

namespace mhc {
namespace {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.44269504088896341f;
constexpr float kLowest = -3.402823466e38f;
constexpr int kPer = 32;          // values of a thread's segment
constexpr int kMostTop = 32;
constexpr int kSegments = 128, kCandidates = 512;  // that the fast selection reads again, and ranks
constexpr int kMostShare = 1 << 18;  // values of a block with alternatives: 32 KB of segments' maxima
constexpr int kMostCluster = 8;

__device__ __forceinline__ float minus_inf() { return __uint_as_float(0xff800000u); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// the larger; NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
constexpr float kTiny = -200.f;     // exp(-200) is 0 in fp32; keeps 0 * inf out of e (x - m)
constexpr float kFloor = -0x1p127f;  // what -inf is read as
constexpr float kPlain = 1e38f;      // rows with a maximum up to this take the short form: x - m stays finite
// x - m of a value with 0 probability can be anything from here on; keeps s (x - m) finite
constexpr float kFar = -1e30f;

// ---------------------------------------------------------------------------
// A row as vectors of 16 bytes from the aligned address at or below its start;
// the vectors at its ends are read value by value, with -inf outside the row.
// ---------------------------------------------------------------------------
template <typename T>
struct Row {
  static constexpr int VE = 16 / (int)sizeof(T);  // values of a vector
  const T* base;  // aligned; value e of the row is base[shift + e]
  int shift, full0, full1, count, V;  // whole vectors, all vectors; a row has at most 2^21 values
  __device__ __forceinline__ Row(const T* row, int vocab) {
    shift = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    base = row - shift;
    V = vocab;
    count = (shift + vocab + VE - 1) / VE;
    full0 = shift ? 1 : 0;
    full1 = (shift + vocab) / VE;
  }
  __device__ __forceinline__ int index(int v) const { return v * VE - shift; }  // of the vector's first value
};

template <typename T>
__device__ __forceinline__ uint4 load_vec(const Row<T>& r, int v, int end) {
  if (v >= r.full0 && v < r.full1 && v < end) return *reinterpret_cast<const uint4*>(r.base + v * Row<T>::VE);
  uint32_t w[4];
  if (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int e = r.index(v) + j;
      w[j] = v < end && e >= 0 && e < r.V ? reinterpret_cast<const uint32_t*>(r.base)[v * 4 + j] : 0xff800000u;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = 0u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int e = r.index(v) + 2 * j + i;
        const uint32_t h =
            v < end && e >= 0 && e < r.V ? reinterpret_cast<const uint16_t*>(r.base)[v * 8 + 2 * j + i] : 0xff80u;
        w[j] |= h << (16 * i);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Values 2 i and 2 i + 1 of a vector
template <typename T>
__device__ __forceinline__ float2 two(const uint4& u, int i) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
// Values below -2^127 become that, NaNs stay
template <typename T>
__device__ __forceinline__ void floor_vec(uint4& u) {
  auto up = [](uint32_t& w) {
    if (sizeof(T) == 4) w = __float_as_uint(max_nan(__uint_as_float(w), kFloor));
    else asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w) : "r"(0xff00ff00u));
  };
  up(u.x);
  up(u.y);
  up(u.z);
  up(u.w);
}
// Largest value of N vectors, NaNs aside
template <typename T, int N>
__device__ __forceinline__ float vec_max(const uint4 (&u)[N]) {
  if (sizeof(T) == 4) {
    float m = kFloor;
#pragma unroll
    for (int q = 0; q < N; ++q)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(u[q].x), __uint_as_float(u[q].y)),
                         fmaxf(__uint_as_float(u[q].z), __uint_as_float(u[q].w))));
    return m;
  }
  uint32_t m = 0xff00ff00u, n = 0xff00ff00u;
  auto up = [](uint32_t& m, uint32_t w) { asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w)); };
#pragma unroll
  for (int q = 0; q < N; ++q) {
    up(m, u[q].x);
    up(n, u[q].y);
    up(m, u[q].z);
    up(n, u[q].w);
  }
  up(m, n);
  return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
}

// ---------------------------------------------------------------------------
// Order of the alternatives: a 64-bit key, larger first; no two are equal.
// NaNs come last.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  const uint32_t b = __float_as_uint(x + 0.f);  // one zero
  const uint32_t o = x != x ? 0u : b ^ ((int32_t)b < 0 ? 0xffffffffu : 0x80000000u);
  return (uint64_t)o << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return o == 0u ? __uint_as_float(0x7fc00000u) : __uint_as_float(o ^ ((int32_t)o < 0 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return ~(uint32_t)key; }

__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(0xffffffffu, v, o);
    v = w > v ? w : v;
  }
  return v;
}

// Sums of a part of a row around its maximum m.
struct Part {
  float m, s, h;
};
__device__ __forceinline__ bool careful(float m) { return !(fabsf(m) <= kPlain); }
// Sums around m as sums around M >= m
__device__ __forceinline__ void rebase(Part& p, float M) {
  const float d = fmaxf(p.m == M ? 0.f : p.m - M, kFar), c = ex2(d * kLog2e);  // equal infinities too
  p.h = c * fmaf(p.s, d, p.h);
  p.s *= c;
  p.m = M;
}
__device__ __forceinline__ float logprob_of(float x, const Part& p) {
  return p.s == 0.f ? minus_inf() : (x - p.m) - logf(p.s);
}
__device__ __forceinline__ float entropy_of(const Part& p) { return p.s == 0.f ? 0.f : logf(p.s) - p.h / p.s; }

// The threads of a row: a block, or a warp of one
template <int THREADS>
__device__ __forceinline__ void row_sync() {
  if (THREADS == 32) __syncwarp();
  else __syncthreads();
}

struct TopShared {
  uint64_t best[kMostTop], joined[kMostTop];  // of the block, of the row's blocks together
  uint64_t cand[kCandidates];
  uint64_t warps[16];
  float maxima[4 * kMostTop];
  int seg[kSegments];
  float bound;
  int segments, candidates;
};

// A block's share [v0, v1) of a row's vectors.  It is walked as [i0, ve): whole
// vectors first, a first one that is not whole (v0 < i0) in the place behind the last.
struct Share {
  int v0, v1, i0, ve, full;  // full: tiles of whole vectors
  // place of vector q of a thread's segment in tile `it`: the threads side by side in full
  // tiles, the warps one behind the other in the last
  template <int THREADS, int VPT>
  __device__ __forceinline__ int walk(int it, int q, int t) const {
    return i0 + it * (THREADS * VPT) + (it < full ? q * THREADS + t : (t & ~31) * VPT + q * 32 + (t & 31));
  }
  __device__ __forceinline__ int at(int v) const { return v == v1 ? v0 : v; }
};

// Threads that the last tile's `left` vectors reach, from thread 0 on
template <int VPT>
__device__ __forceinline__ int lanes_of(int left) {
  const int whole = left / (32 * VPT), rest = left - whole * (32 * VPT);
  return 32 * whole + (rest < 32 ? rest : 32);
}

// The k largest keys of a share into sh.best, in order (0: none left).  segmax:
// maxima of the threads' segments; tm: of all of a thread's.
template <typename T, int THREADS>
__device__ void select_top(const Row<T>& r, const Share& z, int k, int tiles, const float* segmax, float tm, TopShared& sh) {
  constexpr int VE = Row<T>::VE, VPT = kPer / VE, W = THREADS / 32;
  const int tid = threadIdx.x % THREADS, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) sh.segments = sh.candidates = 0;
  // values of a vector that reach the bound, as candidates
  auto push = [&](const uint4& u, int e0, float bound, bool all) {
    uint32_t hits = 0;
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const float2 x = two<T>(u, j / 2);
      const bool in = e0 + j >= 0 && e0 + j < r.V;
      if (in && (all || (j & 1 ? x.y : x.x) >= bound)) hits |= 1u << j;
    }
    if (!hits) return;
    int c = atomicAdd(&sh.candidates, __popc(hits));
#pragma unroll
    for (int j = 0; j < VE; ++j)
      if (hits >> j & 1) {
        const float2 x = two<T>(u, j / 2);
        if (c < kCandidates) sh.cand[c] = key_of(j & 1 ? x.y : x.x, e0 + j);
        ++c;
      }
  };
  bool fast;
  // threads that have values: all of them in a full tile, a warp's place and more in the last
  const int left = z.ve - z.i0, lanes = z.full > 0 ? THREADS : left >= THREADS * VPT ? THREADS : lanes_of<VPT>(left);
  if (lanes < k) {  // 31 vectors at most: all of them
    row_sync<THREADS>();
    for (int vec = z.v0 + tid; vec < z.v1; vec += THREADS) push(load_vec(r, vec, z.v1), r.index(vec), 0.f, true);
    fast = true;
  } else {
    int each = 32;  // lanes of a group
    while (each > 1 && lanes < 2 * k * each) each >>= 1;
    const int groups = (lanes + each - 1) / each;  // that have values: k to 4 k, or a warp each
    float v = tm;
    for (int o = 1; o < each; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane % each == 0 && tid / each < groups) sh.maxima[tid / each] = v;
    row_sync<THREADS>();
    if (tid < groups) {  // the place of each in their order
      const float mine = sh.maxima[tid];
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < groups; ++j) {
        const float m = sh.maxima[j];
        place += m > mine || (m == mine && j < tid);
      }
      if (place == k - 1) sh.bound = mine;
    }
    row_sync<THREADS>();
    const float bound = sh.bound;
    fast = bound > kFloor;  // too few values end below
    if (fast) {
      for (int it = 0; it < tiles; ++it)
        if (segmax[it * THREADS + tid] >= bound) {
          const int i = atomicAdd(&sh.segments, 1);
          if (i < kSegments) sh.seg[i] = it * THREADS + tid;
        }
      row_sync<THREADS>();
      const int n = sh.segments;
      fast = n <= kSegments;
      if (fast)
        for (int i = tid; i < n * VPT; i += THREADS) {
          const int g = sh.seg[i / VPT], walk = z.walk<THREADS, VPT>(g / THREADS, i % VPT, g % THREADS);
          if (walk < z.ve) push(load_vec(r, z.at(walk), z.v1), r.index(z.at(walk)), bound, false);
        }
    }
  }
  row_sync<THREADS>();
  const int c = sh.candidates;
  fast = fast && c <= kCandidates;
  if (fast) {
    for (int i = tid; i < c; i += THREADS) {
      const uint64_t mine = sh.cand[i];
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < c; ++j) rank += sh.cand[j] > mine;
      if (rank < k) sh.best[rank] = mine;
    }
    if (tid >= c && tid < k) sh.best[tid] = 0;  // fewer than k
  }
  if (!fast) {  // one after the other; a thread looks again only when its best is taken
    auto below = [&](uint64_t prev) {
      uint64_t best = 0;
      for (int vec = z.v0 + tid; vec < z.v1; vec += THREADS) {
        const uint4 u = load_vec(r, vec, z.v1);
#pragma unroll
        for (int j = 0; j < VE / 2; ++j) {
          const float2 x = two<T>(u, j);
          const int e = r.index(vec) + 2 * j;
          const uint64_t a = key_of(x.x, e), b = key_of(x.y, e + 1);
          if (e >= 0 && e < r.V && a < prev && a > best) best = a;
          if (e + 1 >= 0 && e + 1 < r.V && b < prev && b > best) best = b;
        }
      }
      return best;
    };
    uint64_t mine = below(~0ull);
    for (int i = 0; i < k; ++i) {
      const uint64_t w = warp_max(mine);
      row_sync<THREADS>();  // everyone has read the last round's
      if (lane == 0) sh.warps[warp] = w;
      row_sync<THREADS>();
      const uint64_t top = warp_max(lane < W ? sh.warps[lane] : 0ull);
      if (tid == 0) sh.best[i] = top;
      if (top != 0 && mine == top) mine = below(top);
    }
  }
  row_sync<THREADS>();
}

struct FwdArgs {
  const void* logits;
  int64_t stride, rows, V;
  const void* targets;
  int64_t ignore;
  float *logprob, *entropy, *top_logprob, *stats;
  int64_t* top_id;
  int top, tiles;
  bool ids64;
};
__device__ __forceinline__ int64_t target_of(const void* t, bool ids64, int64_t row) {
  return ids64 ? static_cast<const int64_t*>(t)[row] : (int64_t)static_cast<const int32_t*>(t)[row];
}
__device__ __forceinline__ float value_of(const float* p) { return *p; }
__device__ __forceinline__ float value_of(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Sums of N vectors around the thread's running maximum.
struct Sums {
  float m;
  float2 s, h;
};
template <typename T, int N>
__device__ __forceinline__ float add_vecs(Sums& a, uint4 (&u)[N]) {
#pragma unroll
  for (int q = 0; q < N; ++q) floor_vec<T>(u[q]);
  const float mx = vec_max<T>(u);
  if (mx > a.m) {
    const float d = fmaxf(a.m - mx, kFar), c = ex2(d * kLog2e);
    a.h.x = c * fmaf(a.s.x, d, a.h.x);
    a.h.y = c * fmaf(a.s.y, d, a.h.y);
    a.s.x *= c;
    a.s.y *= c;
    a.m = mx;
  }
  const float2 minus = make_float2(-a.m, -a.m), scale = make_float2(kLog2e, kLog2e);
#pragma unroll
  for (int q = 0; q < N; ++q)
#pragma unroll
    for (int j = 0; j < Row<T>::VE / 2; ++j) {
      const float2 d = __fadd2_rn(two<T>(u[q], j), minus), t = __fmul2_rn(d, scale);
      const float2 e = make_float2(ex2(t.x), ex2(t.y));
      a.s = __fadd2_rn(a.s, e);
      a.h = __ffma2_rn(e, d, a.h);
    }
  return mx;
}
// The same for one vector in the careful form.
template <typename T>
__device__ __forceinline__ void add_careful(Sums& a, const uint4& u) {
  for (int j = 0; j < Row<T>::VE; ++j) {
    const float2 two_ = two<T>(u, j / 2);
    const float x = j & 1 ? two_.y : two_.x;
    if (x > a.m) {
      const float d = fmaxf(a.m - x, kFar), c = ex2(d * kLog2e);
      a.h.x = c * fmaf(a.s.x, d, a.h.x);
      a.s.x *= c;
      a.m = x;
    }
    const float d = max_nan(x - a.m, kTiny), e = ex2(d * kLog2e);
    a.s.x += e;
    a.h.x = fmaf(e, d, a.h.x);
  }
}

// The row's threads' sums together, the same in each thread.
template <int THREADS>
__device__ __forceinline__ Part block_part(const Sums& a, float (&red)[3][THREADS / 32]) {
  constexpr int W = THREADS / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Part p = {a.m, a.s.x + a.s.y, a.h.x + a.h.y};
  auto join = [](Part& p) {
    float M = p.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    rebase(p, M);
    p.s = warp_sum(p.s);
    p.h = warp_sum(p.h);
  };
  join(p);
  if (W == 1) return p;
  if (lane == 0) {
    red[0][warp] = p.m;
    red[1][warp] = p.s;
    red[2][warp] = p.h;
  }
  __syncthreads();
  p = lane < W ? Part{red[0][lane], red[1][lane], red[2][lane]} : Part{kLowest, 0.f, 0.f};
  join(p);
  return p;
}

// Blocks an SM for the register budget: 16-bit values leave 40 a thread, 32-bit ones
// (a segment is 32 registers) and rows of one warp 64.
template <typename T>
constexpr int fwd_blocks(int threads) { return threads == 32 || sizeof(T) == 4 ? 1024 : 1536; }
constexpr int kRows = 4;  // of a block, where a row takes one warp
constexpr int block_threads(int threads) { return threads == 32 ? 32 * kRows : threads; }

// Shared memory behind a row's segment maxima
inline __host__ __device__ size_t top_bytes(int tiles, int threads) {
  return (size_t)tiles * threads * sizeof(float) + sizeof(TopShared);
}

// One row a cluster of CL blocks, each over its share of the row's vectors; block
// 0 joins the shares through distributed shared memory.  THREADS == 32: a row a warp.
// Bound by HBM, for bf16 with the exponentials behind it (one a value, XU 75%): [8192,
// 65536] bf16 168 us, 6.4 TB/s; [4096, 65536] bf16 89 us, with 5 alternatives 101; [1001,
// 100003] fp32 63 us, 6.4 TB/s.
template <typename T, int THREADS, bool TOP, bool CLUSTER>
__global__ void __launch_bounds__(block_threads(THREADS), fwd_blocks<T>(THREADS) / block_threads(THREADS))
    logprobs_fwd_kernel(const FwdArgs p) {
  constexpr int VE = Row<T>::VE, VPT = kPer / VE, W = THREADS / 32, TILE = THREADS * VPT;
  extern __shared__ __align__(16) unsigned char dyn[];
  const int tid = threadIdx.x % THREADS, lane = tid & 31, place = threadIdx.x / THREADS;
  unsigned char* mine = dyn + (TOP ? place * top_bytes(p.tiles, THREADS) : 0);
  float* segmax = reinterpret_cast<float*>(mine);
  TopShared& sh = *reinterpret_cast<TopShared*>(mine + (size_t)p.tiles * THREADS * sizeof(float));
  __shared__ float red[2][3][W];
  __shared__ Part shared_part;
  const int CL = CLUSTER ? (int)cg::this_cluster().num_blocks() : 1;
  const int rank = CLUSTER ? (int)cg::this_cluster().block_rank() : 0;
  const int64_t row = CLUSTER ? blockIdx.x / CL : THREADS == 32 ? (int64_t)blockIdx.x * kRows + place : blockIdx.x;
  if (THREADS == 32 && row >= p.rows) return;
  const Row<T> r(static_cast<const T*>(p.logits) + row * p.stride, (int)p.V);
  const int each = (r.count + CL - 1) / CL;
  Share z;
  z.v0 = rank * each < r.count ? rank * each : r.count;
  z.v1 = z.v0 + each < r.count ? z.v0 + each : r.count;
  z.i0 = z.v0 > r.full0 ? z.v0 : r.full0;
  z.i0 = z.i0 < z.v1 ? z.i0 : z.v1;
  z.ve = z.v1 + (z.v0 < z.i0);

  Sums a = {kFloor, make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  float tm = kFloor;
  int it = 0;
  // what the given token needs is on its way while the row is read
  int64_t given = -1;
  float at_given = __uint_as_float(0x7fc00000u);
  if (rank == 0 && tid == 0) {
    given = target_of(p.targets, p.ids64, row);
    if (given >= 0 && given < p.V) at_given = value_of(r.base + r.shift + given);
  }
  const int whole = z.v1 < r.full1 ? z.v1 : r.full1;
  int v = z.i0 + tid;
  for (int left = whole - z.i0; left >= TILE; left -= TILE, v += TILE, ++it) {
    uint4 u[VPT];
    const uint4* from = reinterpret_cast<const uint4*>(r.base) + v;
#pragma unroll
    for (int q = 0; q < VPT; ++q) u[q] = from[q * THREADS];
    const float mx = add_vecs<T>(a, u);
    if (TOP) {
      segmax[it * THREADS + tid] = mx;
      tm = fmaxf(tm, mx);
    }
  }
  z.full = it;
  for (; z.i0 + it * TILE < z.ve; ++it) {  // what is left, and the row's ends, to as few warps as it takes
    float mx = kFloor;
    if (z.walk<THREADS, VPT>(it, 0, tid - lane) < z.ve) {
      uint4 u[VPT];
#pragma unroll
      for (int q = 0; q < VPT; ++q) {
        const int w = z.walk<THREADS, VPT>(it, q, tid);
        u[q] = load_vec(r, z.at(w), w < z.ve ? z.v1 : 0);
      }
      mx = add_vecs<T>(a, u);
    }
    if (TOP) {
      segmax[it * THREADS + tid] = mx;
      tm = fmaxf(tm, mx);
    }
  }
  Part part = block_part<THREADS>(a, red[0]);
  if (careful(part.m)) {  // the same for the whole block
    a = {kLowest, make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
    for (int w = z.v0 + tid; w < z.v1; w += THREADS) add_careful<T>(a, load_vec(r, w, z.v1));
    part = block_part<THREADS>(a, red[1]);
  }
  if (TOP) select_top<T, THREADS>(r, z, p.top, it, segmax, tm, sh);
  if (CLUSTER) {
    if (tid == 0) shared_part = part;
    cg::this_cluster().sync();
    if (rank == 0) {
      for (int b = 1; b < CL; ++b) {
        Part o = *cg::this_cluster().map_shared_rank(&shared_part, b);
        if (o.s == 0.f) continue;
        if (part.s == 0.f) {
          part = o;
          continue;
        }
        const float M = fmaxf(part.m, o.m);
        rebase(part, M);
        rebase(o, M);
        part.s += o.s;
        part.h += o.h;
      }
      if (TOP) {
        uint64_t* all = sh.cand;
        for (int i = tid; i < CL * p.top; i += THREADS)
          all[i] = cg::this_cluster().map_shared_rank(sh.best, i / p.top)[i % p.top];
        __syncthreads();
        for (int i = tid; i < CL * p.top; i += THREADS) {
          const uint64_t key = all[i];
          int place = 0;
          for (int j = 0; j < CL * p.top; ++j) place += all[j] > key;
          if (key != 0 && place < p.top) sh.joined[place] = key;
        }
      }
    }
    cg::this_cluster().sync();  // the others' shared memory has been read
    if (rank != 0) return;
  }
  if (TOP && tid < p.top) {
    const uint64_t key = CLUSTER ? sh.joined[tid] : sh.best[tid];
    p.top_logprob[row * p.top + tid] = logprob_of(key_value(key), part);
    p.top_id[row * p.top + tid] = (int64_t)key_index(key);
  }
  if (tid == 0) {
    const bool in = given >= 0 && given < p.V;
    p.logprob[row] = given == p.ignore ? 0.f : in ? logprob_of(at_given, part) : at_given;
    p.entropy[row] = entropy_of(part);
    p.stats[2 * row] = part.m;
    p.stats[2 * row + 1] = part.s;
  }
}

// ---------------------------------------------------------------------------
// Gradient, from the row's m, s and H:
//   gx_j = -p_j (G + gH (ln p_j + H)) + the given tokens' own gradients,
//   G = g_logprob + sum g_top
// and with e = exp(x - m): gx = e (A + B (x - m)).  The few places that have
// a gradient of their own are written again after the block's others.
// ---------------------------------------------------------------------------
struct BwdArgs {
  const void* logits;
  int64_t stride, rows, V;
  const void* targets;
  int64_t ignore;
  const float *stats, *entropy, *g_logprob, *g_entropy, *g_top;
  const int64_t* top_id;
  void* gx;
  int top;
  int64_t chunks;
  int tiles;
  bool ids64;
};
constexpr int kBwdThreads = 256, kBwdTiles = 4;

// Coefficients of a row's gradient in either form
struct Coef {
  float m, A, B;
};
__device__ __forceinline__ float grad_of(float x, const Coef& k) {
  const float d = x - k.m;
  return ex2(d * kLog2e) * fmaf(k.B, max_nan(d, kTiny), k.A);
}
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Gradients of a vector in the short form.  H: with the entropy's (B != 0), whose x - m is held
// above -200 as in the other form, where e is 0 already: B times the distance of a masked value
// passes fp32 for any B past 2, and 0 times that is NaN.  The time stays HBM's ([8192, 65536]
// bf16 326 us, [32768, 4096] 90 us, with and without).
template <typename T, bool H>
__device__ __forceinline__ uint4 grad_vec(const uint4& u, const Coef& k) {
  constexpr int VE = Row<T>::VE;
  const float2 A = make_float2(k.A, k.A), B = make_float2(k.B, k.B), minus = make_float2(-k.m, -k.m),
               scale = make_float2(kLog2e, kLog2e);
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < VE / 2; ++j) {
    const float2 d = __fadd2_rn(two<T>(u, j), minus), t = __fmul2_rn(d, scale);
    const float2 g = __fmul2_rn(make_float2(ex2(t.x), ex2(t.y)),
                                H ? __ffma2_rn(B, make_float2(max_nan(d.x, kTiny), max_nan(d.y, kTiny)), A) : A);
    if (sizeof(T) == 4) {
      w[(2 * j) & 3] = __float_as_uint(g.x);
      w[(2 * j + 1) & 3] = __float_as_uint(g.y);
    } else {
      const __nv_bfloat162 b = __floats2bfloat162_rn(g.x, g.y);
      w[j & 3] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A block takes `tiles` tiles of a row's vectors ([8192, 65536] bf16 321 us, 6.7 TB/s, bound
// by HBM); WARP: rows of 128 vectors at most, one a
// warp and kRows a block.
template <typename T, bool H, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kRows : kBwdThreads) logprobs_bwd_kernel(const BwdArgs p) {
  constexpr int VE = Row<T>::VE, VPT = 4, R = WARP ? kRows : 1;
  __shared__ int64_t at_[R][kMostTop + 1];
  __shared__ float own_[R][kMostTop + 1];
  __shared__ Coef coef_[R];
  __shared__ bool mine_[R];  // whether a place with a gradient of its own is in the range
  const int place = WARP ? threadIdx.x >> 5 : 0, tid = WARP ? threadIdx.x & 31 : threadIdx.x, B_ = WARP ? 32 : blockDim.x;
  int64_t* at = at_[place];
  float* own = own_[place];
  auto sync = [] {
    if (WARP) __syncwarp();
    else __syncthreads();
  };
  const int64_t row = WARP ? (int64_t)blockIdx.x * kRows + place : blockIdx.x / (uint32_t)p.chunks;
  if (WARP && row >= p.rows) return;
  const int chunk = WARP ? 0 : (int)(blockIdx.x - (uint32_t)row * (uint32_t)p.chunks);
  const Row<T> r(static_cast<const T*>(p.logits) + row * p.stride, (int)p.V);
  T* out = static_cast<T*>(p.gx) + row * p.V;
  const int first = chunk * (B_ * VPT * p.tiles);
  int end = first + B_ * VPT * p.tiles;
  end = end < r.count ? end : r.count;
  const bool same = ((reinterpret_cast<uintptr_t>(out) & 15) / sizeof(T)) == (uintptr_t)r.shift;
  auto whole = [&](int a) { return same && a >= r.full0 && a + B_ * VPT <= (end < r.full1 ? end : r.full1); };
  uint4 u[VPT];
  auto load = [&](int a) {  // a tile
    if (whole(a)) {
#pragma unroll
      for (int q = 0; q < VPT; ++q) u[q] = reinterpret_cast<const uint4*>(r.base)[a + q * B_ + tid];
    } else {
#pragma unroll
      for (int q = 0; q < VPT; ++q)
        if (a + q * B_ + tid < end) u[q] = load_vec(r, a + q * B_ + tid, end);
    }
  };
  load(first);
  for (int i = tid; i <= p.top; i += B_) {
    if (i == 0) {
      const int64_t t = target_of(p.targets, p.ids64, row);
      const float g = p.g_logprob ? p.g_logprob[row] : 0.f;
      const bool in = t >= 0 && t < p.V;
      at[0] = in && t != p.ignore ? t : -1;
      // a target outside has a log probability of NaN, and nothing else depends on it
      own[0] = t == p.ignore || !p.g_logprob ? 0.f : in ? g : g * __uint_as_float(0x7fc00000u);
    } else {
      at[i] = p.top_id[row * p.top + i - 1];
      own[i] = p.g_top[row * p.top + i - 1];
    }
  }
  if (p.top) sync();
  if (tid == 0) {
    float G = own[0];
    bool any = false;
    const int lo = r.index(first), hi = r.index(end);
    for (int i = 0; i <= p.top; ++i) {
      if (i) G += own[i];
      any = any || (at[i] >= 0 && at[i] >= lo && at[i] < hi);
    }
    Coef k = {p.stats[2 * row], 0.f, 0.f};
    const float s = p.stats[2 * row + 1];
    if (s != 0.f) {
      const float gh = H ? p.g_entropy[row] : 0.f, inv = 1.0f / s;
      k.A = -inv * (H ? fmaf(gh, p.entropy[row] - logf(s), G) : G);
      k.B = -inv * gh;
    }
    coef_[place] = k;
    mine_[place] = any && s != 0.f;
  }
  sync();
  const Coef k = coef_[place];
  if (careful(k.m)) {  // and rows without anything
    for (int v = first + tid; v < end; v += B_) {
      const uint4 w = load_vec(r, v, end);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float2 x = two<T>(w, j / 2);
        const int e = r.index(v) + j;
        if (e >= 0 && e < p.V) put(out + e, grad_of(j & 1 ? x.y : x.x, k));
      }
    }
  } else {
    for (int a = first; a < end; a += B_ * VPT) {
      if (a != first) load(a);
      uint4* to = reinterpret_cast<uint4*>(out - r.shift) + a + tid;
      if (whole(a)) {
#pragma unroll
        for (int q = 0; q < VPT; ++q) to[q * B_] = grad_vec<T, H>(u[q], k);
      } else {
#pragma unroll
        for (int q = 0; q < VPT; ++q) {
          const int v = a + q * B_ + tid;
          if (v >= end) continue;
          const uint4 g = grad_vec<T, H>(u[q], k);
          if (same && v >= r.full0 && v < r.full1) {
            to[q * B_] = g;
          } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) {
              const int e = r.index(v) + j;
              const float2 x = two<T>(g, j / 2);
              if (e >= 0 && e < p.V) put(out + e, j & 1 ? x.y : x.x);
            }
          }
        }
      }
    }
  }
  if (!mine_[place]) return;
  sync();  // before these places are written again
  const int lo = r.index(first), hi = r.index(end);
  for (int i = tid; i <= p.top; i += B_) {
    const int64_t e = at[i];
    if (e < 0 || e >= p.V || e < lo || e >= hi) continue;
    float g = 0.f;
    bool earliest = true;
    for (int j = 0; j <= p.top; ++j)
      if (at[j] == e) {
        earliest = earliest && j >= i;
        g += own[j];
      }
    if (earliest) put(out + e, g + grad_of(value_of(r.base + r.shift + e), k));
  }
}

template <typename T, int THREADS, bool TOP>
int launch_fwd(FwdArgs p, int CL, cudaStream_t st) {
  constexpr int VE = Row<T>::VE, rows = block_threads(THREADS) / THREADS;
  const int64_t count = (p.V + VE - 1) / VE + 1, each = (count + CL - 1) / CL;
  p.tiles = (int)((each + THREADS * (kPer / VE) - 1) / (THREADS * (kPer / VE)));
  const size_t smem = TOP ? rows * top_bytes(p.tiles, THREADS) : 0;
  ProfScope prof("token_logprobs_fwd", st);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)CL;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.rows + rows - 1) / rows * CL));
  cfg.blockDim = dim3(block_threads(THREADS));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = CL > 1 ? 1 : 0;
  if (CL == 1) cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<T, THREADS, TOP, false>, p);
  else if constexpr (THREADS == 512 || (THREADS == 256 && TOP)) cudaLaunchKernelEx(&cfg, logprobs_fwd_kernel<T, THREADS, TOP, true>, p);
  else return fail(MHC_ERR_UNSUPPORTED, "token_logprobs: no kernel for %d blocks of %d threads a row", CL, THREADS);
  return check_launch("token_logprobs_fwd");
}

template <typename T>
int pick_fwd(const FwdArgs& p, cudaStream_t st) {
  // Few rows: several blocks a row while the GPU has room and a share stays long
  // (joining shares costs 0.5 us, with alternatives 1 to 4: [1, 131072] fp32 8.3 us on
  // one block, 5.9 on four, [1, 32768] 3.7 on one, 4.4 on four).
  int CL = 1;
  while (CL < kMostCluster && p.rows * CL * 2 <= num_sms() && p.V > (int64_t)CL * 49152) CL *= 2;
  while (p.top > 0 && p.V > (int64_t)CL * kMostShare) CL *= 2;  // 8 at most: a row has up to 2^21 values
  MHC_REQUIRE(p.rows * CL < (1ll << 31), MHC_ERR_UNSUPPORTED, "token_logprobs: %lld rows are too many", (long long)p.rows);
  // Small blocks hide each other's ends where there are many rows ([32768, 4096] bf16: 53
  // and 65 us with 32 and 128 threads, [19691, 13632]: 114, 137 and 184 us with 128, 256
  // and 512); few rows want more threads each.
  const int64_t share = (p.V + CL - 1) / CL, blocks = p.rows * CL;
  const int th = share <= 8192 ? (blocks >= 4 * num_sms() ? 32 : 128) : blocks < 2 * num_sms() ? 512 : share <= 32768 ? 128 : 256;
#define MHC_GO(TH) (p.top > 0 ? launch_fwd<T, TH, true>(p, CL, st) : launch_fwd<T, TH, false>(p, CL, st))
  return th == 32 ? MHC_GO(32) : th == 128 ? MHC_GO(128) : th == 256 ? MHC_GO(256) : MHC_GO(512);
#undef MHC_GO
}

int check_args(const char* what, int64_t rows, int64_t vocab, int64_t stride, int32_t top, int32_t bf16, const void* logits) {
  MHC_REQUIRE(rows >= 0 && vocab >= 1, MHC_ERR_INVALID_ARG, "%s: rows must be >= 0 and vocab >= 1 (got %lld x %lld)", what,
              (long long)rows, (long long)vocab);
  MHC_REQUIRE(rows < (1ll << 31) && vocab <= (1ll << 21), MHC_ERR_UNSUPPORTED,
              "%s: at most 2^31 - 1 rows of 2^21 logits (got %lld x %lld)", what, (long long)rows, (long long)vocab);
  MHC_REQUIRE(stride >= vocab || rows <= 1, MHC_ERR_INVALID_ARG, "%s: row_stride %lld < vocab %lld", what, (long long)stride,
              (long long)vocab);
  MHC_REQUIRE(top >= 0 && top <= kMostTop && top <= vocab, MHC_ERR_UNSUPPORTED, "%s: top must be in [0, min(32, vocab)] (got %d)",
              what, (int)top);
  MHC_REQUIRE((reinterpret_cast<uintptr_t>(logits) & (bf16 ? 1 : 3)) == 0, MHC_ERR_ALIGNMENT,
              "%s: logits must be aligned to their type", what);
  return MHC_OK;
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" int mhc_token_logprobs_fwd(const void* logits, int32_t logits_bf16, int64_t row_stride, const void* targets,
                                      int32_t targets_64, int64_t ignore_index, float* logprob, float* entropy,
                                      float* top_logprob, int64_t* top_id, float* stats, int64_t rows, int64_t vocab,
                                      int32_t top, void* stream) {
  const char* what = "token_logprobs_fwd";
  const int rc = check_args(what, rows, vocab, row_stride, top, logits_bf16, logits);
  if (rc) return rc;
  if (rows == 0) return MHC_OK;
  MHC_REQUIRE_PTR(logits);
  MHC_REQUIRE_PTR(targets);
  MHC_REQUIRE_PTR(logprob);
  MHC_REQUIRE_PTR(entropy);
  MHC_REQUIRE_PTR(stats);
  if (top > 0) {
    MHC_REQUIRE_PTR(top_logprob);
    MHC_REQUIRE_PTR(top_id);
  }
  const FwdArgs p = {logits, row_stride, rows, vocab, targets, ignore_index, logprob, entropy, top_logprob, stats, top_id,
                     (int)top, 0, targets_64 != 0};
  return logits_bf16 ? pick_fwd<__nv_bfloat16>(p, (cudaStream_t)stream) : pick_fwd<float>(p, (cudaStream_t)stream);
}

extern "C" int mhc_token_logprobs_bwd(const void* logits, int32_t logits_bf16, int64_t row_stride, const void* targets,
                                      int32_t targets_64, int64_t ignore_index, const float* stats, const float* entropy,
                                      const int64_t* top_id, const float* grad_logprob, const float* grad_entropy,
                                      const float* grad_top, void* grad_logits, int64_t rows, int64_t vocab, int32_t top,
                                      void* stream) {
  const char* what = "token_logprobs_bwd";
  const int rc = check_args(what, rows, vocab, row_stride, top, logits_bf16, logits);
  if (rc) return rc;
  if (rows == 0) return MHC_OK;
  MHC_REQUIRE_PTR(logits);
  MHC_REQUIRE_PTR(targets);
  MHC_REQUIRE_PTR(stats);
  MHC_REQUIRE_PTR(entropy);
  MHC_REQUIRE_PTR(grad_logits);
  if (top > 0) {
    MHC_REQUIRE_PTR(top_id);
    MHC_REQUIRE_PTR(grad_top);
  }
  constexpr int per = 4;  // vectors of a thread and tile
  const int64_t VE = logits_bf16 ? 8 : 4;
  // where rows start in a vector: all at one place, or anywhere
  const int64_t shift = rows == 1 || row_stride % VE == 0 ? (int64_t)(reinterpret_cast<uintptr_t>(logits) & 15) / (logits_bf16 ? 2 : 4) : VE - 1;
  const int64_t count = (shift + vocab + VE - 1) / VE;
  const bool warp = count <= 32 * per;
  // 64 to 256 threads, so that a row has about four tiles of whole vectors ([32768, 8192]
  // bf16 166 us against 212 with 256, [32768, 4096] 86 against 107 with 128)
  int64_t threads = ((count + per * kBwdTiles - 1) / (per * kBwdTiles) + 31) / 32 * 32;
  threads = warp ? 32 * kRows : threads > kBwdThreads ? kBwdThreads : threads < 64 ? 64 : threads;
  // several tiles a block where that leaves enough blocks: its coefficients cost as much as a tile
  int tiles = warp ? 1 : kBwdTiles;
  while (tiles > 1 && rows * ((count + threads * per * tiles - 1) / (threads * per * tiles)) < 16 * (int64_t)num_sms()) --tiles;
  const int64_t chunks = warp ? 1 : (count + threads * per * tiles - 1) / (threads * per * tiles);
  MHC_REQUIRE(rows * chunks < (1ll << 31), MHC_ERR_UNSUPPORTED, "%s: %lld x %lld logits are too many", what, (long long)rows,
              (long long)vocab);
  const BwdArgs p = {logits, row_stride, rows, vocab, targets, ignore_index, stats, entropy, grad_logprob, grad_entropy,
                     grad_top, top_id, grad_logits, (int)top, chunks, tiles, targets_64 != 0};
  cudaStream_t st = (cudaStream_t)stream;
  ProfScope prof(what, st);
  const unsigned blocks = (unsigned)(warp ? (rows + kRows - 1) / kRows : rows * chunks);
#define MHC_GO(T, H)                                                                          \
  do {                                                                                        \
    if (warp) logprobs_bwd_kernel<T, H, true><<<blocks, (unsigned)threads, 0, st>>>(p);       \
    else logprobs_bwd_kernel<T, H, false><<<blocks, (unsigned)threads, 0, st>>>(p);           \
  } while (0)
  if (logits_bf16) {
    if (grad_entropy) MHC_GO(__nv_bfloat16, true);
    else MHC_GO(__nv_bfloat16, false);
  } else {
    if (grad_entropy) MHC_GO(float, true);
    else MHC_GO(float, false);
  }
#undef MHC_GO
  return check_launch(what);
}
