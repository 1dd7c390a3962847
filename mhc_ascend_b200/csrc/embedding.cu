// Embedding lookup into residual streams and the gradient of its table.
//
//   out[t, i, :] = s_i W[id_t, :]                         (i < n streams)
//   gW[v, :]     = sum over t with id_t = v of sum_i s_i g[t, i, :]
//
// The gradient goes by sorted tokens: (id, t) pairs are sorted (stable), so
// that each table row's terms are neighbours and are added in token order by
// one owner.  No float atomics: the same inputs give the same bits.
#include <cooperative_groups.h>

#include "checkpoint8.cuh"

namespace cg = cooperative_groups;

namespace mhc {
namespace {

constexpr int kMaxStreams = 32;
struct Scales {
  float s[kMaxStreams];
};

// units of 4 or 8 values where the layout allows them, of one elsewhere
__device__ __forceinline__ void load_unit(const float* p, float (&v)[4]) {
  const float4 a = __ldcs(reinterpret_cast<const float4*>(p));
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
__device__ __forceinline__ void load_unit(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 a = __ldcs(reinterpret_cast<const uint2*>(p));
  v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u);
  v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
}
__device__ __forceinline__ void load_unit(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p));
  const uint32_t r[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(r[j] << 16);
    v[2 * j + 1] = __uint_as_float(r[j] & 0xffff0000u);
  }
}
template <typename T>
__device__ __forceinline__ void load_unit(const T* p, float (&v)[1]) { v[0] = ck_f32(*p); }

__device__ __forceinline__ void save_unit(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void save_unit(__nv_bfloat16* p, const float (&v)[4]) {
  __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  uint2 r;
  r.x = *reinterpret_cast<uint32_t*>(&a);
  r.y = *reinterpret_cast<uint32_t*>(&b);
  *reinterpret_cast<uint2*>(p) = r;
}
__device__ __forceinline__ void save_unit(float* p, const float (&v)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void save_unit(__nv_bfloat16* p, const float (&v)[8]) { ck_save(p, v); }
template <typename T>
__device__ __forceinline__ void save_unit(T* p, const float (&v)[1]) { ck_store(p, v[0]); }

// ---------------------------------------------------------------------------
// forward: bound by writing the streams.  A block takes tokens_per_block
// tokens, lanes along the row; the row is read once for its n copies.
// ---------------------------------------------------------------------------
template <typename I, typename TW, typename TO, int V>
__global__ void __launch_bounds__(256)
    embed_fwd_kernel(const I* __restrict__ ids, const TW* __restrict__ w, TO* __restrict__ out, int64_t T, int n,
                     int64_t C, int64_t vocab, const __grid_constant__ Scales sc, int lanes) {
  const int64_t t = (int64_t)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes;
  if (t >= T) return;
  const int64_t id = (int64_t)ids[t];
  const bool good = id >= 0 && id < vocab;
  const TW* row = w + id * C;
  TO* o = out + t * n * C;
  for (int64_t c = (int64_t)(threadIdx.x % lanes) * V; c < C; c += (int64_t)lanes * V) {
    float v[V];
    if (good) {
      load_unit(row + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = __uint_as_float(0x7fc00000u);
    }
    for (int i = 0; i < n; ++i) {
      float u[V];
#pragma unroll
      for (int j = 0; j < V; ++j) u[j] = v[j] * sc.s[i];
      save_unit(o + i * C + c, u);
    }
  }
}

// ---------------------------------------------------------------------------
// gradient, launch 1: the sort, and the zeros of the dense gradient.
//
// The first 8 blocks are one cluster that sorts (key, t) by radix digits of up
// to 9 bits, least significant first; block c owns the c-th eighth of the
// positions.  Per digit: a histogram of the block's range in shared memory;
// the exclusive sums over digits and blocks from the others' histograms
// through distributed shared memory; then tiles of 4096 positions are ranked
// (per warp by ballots, across warps by a column sum) and scattered.  The
// lists stay in L2.  Padding and invalid ids get the key V and sort last.
// All other blocks write zeros over gW meanwhile: the sort costs a few
// microseconds a digit on 8 SMs, and hides behind V C stores.
// ---------------------------------------------------------------------------
constexpr int kSortBlocks = 8, kSortThreads = 512, kSortItems = 8, kSortTile = kSortThreads * kSortItems;
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits, kSortWarps = kSortThreads / 32;

template <typename I>
__global__ void __cluster_dims__(kSortBlocks, 1, 1) __launch_bounds__(kSortThreads)
    embed_sort_kernel(const I* __restrict__ ids, uint32_t* ka, uint32_t* va, uint32_t* kb, uint32_t* vb, uint32_t T,
                      uint32_t vocab, int64_t pad, int passes, int bits, char* zero, uint64_t zero_bytes) {
  const int tid = threadIdx.x;
  if (blockIdx.x >= kSortBlocks) {
    const uint64_t nb = gridDim.x - kSortBlocks, b = blockIdx.x - kSortBlocks;
    const uint64_t units = zero_bytes / 16;
#pragma unroll 4
    for (uint64_t u = b * kSortThreads + tid; u < units; u += nb * kSortThreads)
      reinterpret_cast<uint4*>(zero)[u] = make_uint4(0u, 0u, 0u, 0u);
    if (b == 0 && tid < (int)(zero_bytes & 15)) zero[units * 16 + tid] = 0;
    return;
  }
  __shared__ uint32_t hist[kDigits];                 // this block's counts, read by the whole cluster
  __shared__ uint32_t base[kDigits];                 // next free place of each digit for this block
  __shared__ uint32_t wcnt[kSortWarps][kDigits];     // counts, then places, by warp
  __shared__ uint32_t wsum[kSortWarps];
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank();
  const int warp = tid >> 5, lane = tid & 31;
  const uint32_t share = ((T + kSortBlocks - 1) / kSortBlocks + kSortTile - 1) / kSortTile * kSortTile;
  const uint32_t lo = min((uint64_t)rank * share, (uint64_t)T), hi = min((uint64_t)lo + share, (uint64_t)T);
  const uint32_t mask = (1u << bits) - 1u;

  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    uint32_t* kin = (p & 1) ? kb : ka;
    uint32_t* vin = (p & 1) ? vb : va;
    uint32_t* kout = (p & 1) ? ka : kb;
    uint32_t* vout = (p & 1) ? va : vb;
    auto key_at = [&](uint32_t i) -> uint32_t {
      if (p > 0) return __ldcg(kin + i);
      const int64_t id = (int64_t)ids[i];
      return (id >= 0 && id < (int64_t)vocab && id != pad) ? (uint32_t)id : vocab;
    };
    for (int d = tid; d < kDigits; d += kSortThreads) hist[d] = 0;
    __syncthreads();
    for (uint32_t i0 = lo + tid; i0 < hi; i0 += 8 * kSortThreads) {
      uint32_t k[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) k[j] = i0 + j * kSortThreads < hi ? key_at(i0 + j * kSortThreads) : 0u;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j * kSortThreads < hi) atomicAdd(&hist[(k[j] >> shift) & mask], 1u);
    }
    cluster.sync();
    {  // one digit a thread: everyone's count, and the counts of the blocks before this one
      uint32_t all = 0, before = 0;
#pragma unroll
      for (uint32_t c = 0; c < kSortBlocks; ++c) {
        const uint32_t h = *cluster.map_shared_rank(&hist[tid], c);
        all += h;
        if (c < rank) before += h;
      }
      uint32_t inc = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      if (lane == 31) wsum[warp] = inc;
      __syncthreads();
      uint32_t wbase = 0;
      for (int k = 0; k < warp; ++k) wbase += wsum[k];
      base[tid] = wbase + inc - all + before;
    }
    cluster.sync();  // the histograms have been read: the next digit may clear them
    uint32_t key[kSortItems], val[kSortItems];
    auto fetch = [&](uint32_t t0) {
#pragma unroll
      for (int k = 0; k < kSortItems; ++k) {
        const uint32_t i = t0 + warp * (32 * kSortItems) + lane + 32 * k;
        key[k] = i < hi ? key_at(i) : 0xffffffffu;
        val[k] = i < hi ? (p > 0 ? __ldcg(vin + i) : i) : 0u;
      }
    };
    if (lo < hi) fetch(lo);
    for (uint32_t t0 = lo; t0 < hi; t0 += kSortTile) {
      for (int e = tid; e < kSortWarps * kDigits; e += kSortThreads) (&wcnt[0][0])[e] = 0;
      __syncthreads();
      uint32_t place[kSortItems];
      const uint32_t wfirst = t0 + warp * (32 * kSortItems) + lane;
#pragma unroll
      for (int k = 0; k < kSortItems; ++k) {
        const bool on = wfirst + 32 * k < hi;
        const uint32_t d = (key[k] >> shift) & mask;
        uint32_t peers = __ballot_sync(0xffffffffu, on);
        for (int b = 0; b < bits; ++b) {
          const uint32_t m = __ballot_sync(0xffffffffu, (d >> b) & 1u);
          peers &= ((d >> b) & 1u) ? m : ~m;
        }
        uint32_t old = 0;
        if (on) old = wcnt[warp][d];
        __syncwarp();
        place[k] = old + __popc(peers & ((1u << lane) - 1u));
        if (on && (peers & ((1u << lane) - 1u)) == 0) wcnt[warp][d] = old + __popc(peers);
        __syncwarp();
      }
      __syncthreads();
      {
        uint32_t run = base[tid];
        uint32_t c[kSortWarps];
#pragma unroll
        for (int k = 0; k < kSortWarps; ++k) c[k] = wcnt[k][tid];
#pragma unroll
        for (int k = 0; k < kSortWarps; ++k) {
          wcnt[k][tid] = run;
          run += c[k];
        }
        base[tid] = run;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kSortItems; ++k)
        if (wfirst + 32 * k < hi) {
          const uint32_t at = wcnt[warp][(key[k] >> shift) & mask] + place[k];
          __stcg(kout + at, key[k]);
          __stcg(vout + at, val[k]);
        }
      if (t0 + kSortTile < hi) fetch(t0 + kSortTile);
      __syncthreads();
    }
    cluster.sync();  // release / acquire: the lists are whole before the next digit reads them
  }
}

// ---------------------------------------------------------------------------
// gradient, launch 2: sums of the sorted positions, `chunk` of them and a slice of
// the columns a block.  Rows whose tokens all lie in the chunk are written; the
// sums at its two ends, if their rows go on in a neighbour, are kept:
// ends[chunk][0] for a row that began before the chunk, [1] for one that begins in
// it and goes on.  Bound by reading g: 8 or 16 loads of a thread are in flight,
// and blocks that run together read neighbouring slices of the same rows.
// A thread has NC x V columns: V = 4 or 8 in one access, or four single ones, a
// block's width apart, where rows are not aligned.
// launch 3: for each row that begins in a chunk and goes on, its sums are added
// in chunk order and the row is written.
// ---------------------------------------------------------------------------
constexpr int kMaxChunk = 64, kSumThreads = 128, kJoinThreads = 256;

template <typename TG, typename TW, int V, int NC>
__global__ void __launch_bounds__(kSumThreads)
    embed_sum_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ vals,
                     const TG* __restrict__ g, TW* __restrict__ gw, float* __restrict__ ends, uint32_t T,
                     uint32_t vocab, int n, int64_t C, const __grid_constant__ Scales sc, int chunk, uint32_t slices) {
  constexpr int L = NC == 1 ? 8 : 4;  // rows of g in flight
  __shared__ uint32_t sk[kMaxChunk + 2], sv[kMaxChunk];
  __shared__ float ss[kMaxStreams];
  const uint32_t piece = blockIdx.x / slices;
  const uint32_t p0 = piece * chunk;
  const int tid = threadIdx.x;
  if (tid < chunk + 2) {  // sk[1 + j] = key at p0 + j; neighbours on both sides
    const int64_t q = (int64_t)p0 + tid - 1;
    sk[tid] = q >= 0 && q < (int64_t)T ? keys[q] : 0xffffffffu;
  }
  if (tid < chunk) sv[tid] = p0 + tid < T ? vals[p0 + tid] : 0u;
  if (tid < n) ss[tid] = sc.s[tid];
  __syncthreads();
  int len = (int)min((uint32_t)chunk, T - p0);
  while (len > 0 && sk[len] >= vocab) --len;  // padding sorts last
  if (len == 0) return;
  const int64_t c = ((int64_t)(blockIdx.x - piece * slices) * (kSumThreads * NC) + tid) * V;
  if (c >= C) return;
  bool on[NC];
#pragma unroll
  for (int m = 0; m < NC; ++m) on[m] = c + (int64_t)m * kSumThreads * V < C;
  float acc[NC][V];
#pragma unroll
  for (int m = 0; m < NC; ++m)
#pragma unroll
    for (int j = 0; j < V; ++j) acc[m][j] = 0.f;
  int p = 0, i = 0;  // what is added next: stream i of position p
  int first = 0;     // first position of the running row
  const int total = len * n;
  int lp = 0, li = 0;
  const TG* at = g + (int64_t)sv[0] * n * C + c;  // what is loaded next
  for (int q = 0; q < total; q += L) {
    float v[L][NC][V];
#pragma unroll
    for (int k = 0; k < L; ++k)
      if (q + k < total) {
#pragma unroll
        for (int m = 0; m < NC; ++m)
          if (on[m]) load_unit(at + (int64_t)m * kSumThreads * V, v[k][m]);
        at += C;
        if (++li == n) {
          li = 0;
          if (++lp < len) at = g + (int64_t)sv[lp] * n * C + c;
        }
      }
#pragma unroll
    for (int k = 0; k < L; ++k)
      if (q + k < total) {
        const float s = ss[i];
#pragma unroll
        for (int m = 0; m < NC; ++m)
          if (on[m])
#pragma unroll
            for (int j = 0; j < V; ++j) acc[m][j] = fmaf(s, v[k][m][j], acc[m][j]);
        if (++i == n) {
          i = 0;
          const uint32_t key = sk[p + 1];
          const bool more = p + 1 < len && sk[p + 2] == key;
          if (!more) {
            const bool before = first == 0 && sk[0] == key;
            const bool after = p + 1 == len && sk[p + 2] == key;
            float* e = ends + ((int64_t)piece * 2 + (before ? 0 : 1)) * C + c;
#pragma unroll
            for (int m = 0; m < NC; ++m) {
              const int64_t o = (int64_t)m * kSumThreads * V;
              if (on[m]) {
                if (!before && !after) save_unit(gw + (int64_t)key * C + c + o, acc[m]);
                else save_unit(e + o, acc[m]);
              }
#pragma unroll
              for (int j = 0; j < V; ++j) acc[m][j] = 0.f;
            }
            first = p + 1;
          }
          ++p;
        }
      }
  }
}

// A block joins one row's sums over kJoinThreads * V columns; where there are many,
// a warp takes every eighth of them and the eight shares are added in order.
template <typename TW, int V>
__global__ void __launch_bounds__(kJoinThreads)
    embed_join_kernel(const uint32_t* __restrict__ keys, TW* __restrict__ gw, const float* __restrict__ ends,
                      uint32_t T, uint32_t vocab, int64_t C, int chunk, uint32_t slices) {
  __shared__ __align__(16) float part[8][32 * V];
  const uint32_t piece = blockIdx.x / slices;
  const uint32_t p1 = (piece + 1) * chunk;  // first position of the next chunk (exists: the grid is one short)
  const uint32_t p0 = p1 - chunk;
  const uint32_t key = keys[p1], last_key = keys[p1 - 1], first_key = keys[p0], before_key = p0 > 0 ? keys[p0 - 1] : ~0u;
  if (key >= vocab || last_key != key) return;          // no row goes on here
  if (first_key == key && before_key == key) return;    // it began in an earlier chunk
  uint32_t lo = p1, hi = T;                             // first position past the row
  while (lo < hi) {
    const uint32_t m = lo + (hi - lo) / 2;
    if (keys[m] > key) hi = m; else lo = m + 1;
  }
  const uint32_t last = (lo - 1) / chunk, count = last - piece;
  const int64_t c0 = (int64_t)(blockIdx.x - piece * slices) * (kJoinThreads * V);
  if (count <= 16) {
    const int64_t c = c0 + threadIdx.x * V;
    if (c >= C) return;
    float acc[V];
    load_unit(ends + ((int64_t)piece * 2 + 1) * C + c, acc);
#pragma unroll 4
    for (uint32_t m = piece + 1; m <= last; ++m) {
      float v[V];
      load_unit(ends + (int64_t)m * 2 * C + c, v);
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += v[j];
    }
    save_unit(gw + (int64_t)key * C + c, acc);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int sub = 0; sub < 8; ++sub) {
    const int64_t c = c0 + (sub * 32 + lane) * V;
    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
    if (c < C) {
      if (warp == 0) load_unit(ends + ((int64_t)piece * 2 + 1) * C + c, acc);
#pragma unroll 8
      for (uint32_t m = piece + 1 + warp; m <= last; m += 8) {
        float v[V];
        load_unit(ends + (int64_t)m * 2 * C + c, v);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += v[j];
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) part[warp][lane * V + j] = acc[j];
    __syncthreads();
    if (warp == 0 && c < C) {
#pragma unroll
      for (int w = 1; w < 8; ++w)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += part[w][lane * V + j];
      save_unit(gw + (int64_t)key * C + c, acc);
    }
    __syncthreads();
  }
}

int check_embed(const char* what, int64_t T, int32_t n, int64_t C, int64_t vocab, const float* scales) {
  MHC_REQUIRE(T >= 0 && C >= 1 && vocab >= 1, MHC_ERR_INVALID_ARG,
              "%s: tokens must be >= 0, hidden >= 1 and vocab >= 1 (got %lld, %lld, %lld)", what, (long long)T,
              (long long)C, (long long)vocab);
  MHC_REQUIRE(n >= 1 && n <= kMaxStreams, MHC_ERR_UNSUPPORTED, "%s: n must be in [1, %d] (got %d)", what, kMaxStreams,
              n);
  MHC_REQUIRE(T < (1ll << 31) && vocab < (1ll << 31) && C <= (1ll << 22), MHC_ERR_UNSUPPORTED,
              "%s: %lld tokens, %lld rows of %lld are too many", what, (long long)T, (long long)vocab, (long long)C);
  MHC_REQUIRE(scales != nullptr, MHC_ERR_INVALID_ARG, "%s: scales must not be NULL", what);
  return MHC_OK;
}

Scales host_scales(const float* s, int n) {
  Scales r;
  for (int i = 0; i < kMaxStreams; ++i) r.s[i] = i < n ? s[i] : 0.f;
  return r;
}

template <typename I, typename TW, typename TO>
int launch_embed_fwd(const void* ids, const void* w, void* out, int64_t T, int n, int64_t C, int64_t vocab,
                     const Scales& sc, cudaStream_t st) {
  const bool vec = C % 4 == 0 && (reinterpret_cast<uintptr_t>(w) & (4 * sizeof(TW) - 1)) == 0 &&
                   (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(TO) - 1)) == 0;
  const int64_t units = vec ? C / 4 : C;
  int lanes = 1;
  while (lanes < 256 && lanes < units) lanes <<= 1;
  const int64_t per = 256 / lanes, blocks = (T + per - 1) / per;
  ProfScope p("stream_embedding_fwd", st);
  if (vec)
    embed_fwd_kernel<I, TW, TO, 4><<<(unsigned)blocks, 256, 0, st>>>((const I*)ids, (const TW*)w, (TO*)out, T, n, C,
                                                                     vocab, sc, lanes);
  else
    embed_fwd_kernel<I, TW, TO, 1><<<(unsigned)blocks, 256, 0, st>>>((const I*)ids, (const TW*)w, (TO*)out, T, n, C,
                                                                     vocab, sc, lanes);
  return check_launch("stream_embedding_fwd");
}

struct GradPlan {
  size_t list, ends;  // bytes of one list, of the end sums
  int chunk;          // positions of a chunk
  int64_t chunks;
};
// The largest chunk (a power of two to 64) that leaves 2048 blocks: shorter chunks
// join more sums, fewer blocks leave the GPU idle ([128, 32, 1280] in chunks of 32
// took 200 us on its 12 blocks).
GradPlan grad_plan(int64_t T, int64_t C) {
  GradPlan p;
  p.list = ((size_t)T * 4 + 255) / 256 * 256;
  const int64_t slices = (C + 511) / 512;
  p.chunk = kMaxChunk;
  while (p.chunk > 1 && (T + p.chunk - 1) / p.chunk * slices < 2048) p.chunk /= 2;
  p.chunks = (T + p.chunk - 1) / p.chunk;
  p.ends = (size_t)p.chunks * 2 * (size_t)C * sizeof(float);
  return p;
}

template <typename TG, typename TW, int V, int NC>
int launch_embed_sums(const uint32_t* keys, const uint32_t* vals, const void* g, void* gw, float* ends, int64_t T,
                      int n, int64_t C, int64_t vocab, const Scales& sc, const GradPlan& pl, cudaStream_t st) {
  {
    const int64_t slices = (C + kSumThreads * V * NC - 1) / (kSumThreads * V * NC), blocks = pl.chunks * slices;
    MHC_REQUIRE(blocks < (1ll << 31), MHC_ERR_UNSUPPORTED, "stream_embedding_bwd: %lld tokens of %lld are too many",
                (long long)T, (long long)C);
    ProfScope p("stream_embedding_sum", st);
    embed_sum_kernel<TG, TW, V, NC><<<(unsigned)blocks, kSumThreads, 0, st>>>(
        keys, vals, (const TG*)g, (TW*)gw, ends, (uint32_t)T, (uint32_t)vocab, n, C, sc, pl.chunk, (uint32_t)slices);
    const int rc = check_launch("stream_embedding_sum");
    if (rc) return rc;
  }
  if (pl.chunks < 2) return MHC_OK;
  constexpr int W = V == 1 ? 1 : 4;
  const int64_t slices = (C + kJoinThreads * W - 1) / (kJoinThreads * W), blocks = (pl.chunks - 1) * slices;
  MHC_REQUIRE(blocks < (1ll << 31), MHC_ERR_UNSUPPORTED, "stream_embedding_bwd: %lld tokens of %lld are too many",
              (long long)T, (long long)C);
  ProfScope p("stream_embedding_join", st);
  embed_join_kernel<TW, W><<<(unsigned)blocks, kJoinThreads, 0, st>>>(keys, (TW*)gw, ends, (uint32_t)T, (uint32_t)vocab,
                                                                      C, pl.chunk, (uint32_t)slices);
  return check_launch("stream_embedding_join");
}

}  // namespace
}  // namespace mhc

using namespace mhc;

extern "C" int mhc_stream_embedding_fwd(const void* ids, int32_t ids_64, const void* weight, int32_t weight_bf16,
                                        void* out, int32_t out_bf16, const float* scales, int64_t tokens, int32_t n,
                                        int64_t hidden, int64_t vocab, void* stream) {
  const int rc = check_embed("stream_embedding_fwd", tokens, n, hidden, vocab, scales);
  if (rc) return rc;
  if (tokens == 0) return MHC_OK;
  MHC_REQUIRE_PTR(ids);
  MHC_REQUIRE_PTR(weight);
  MHC_REQUIRE_PTR(out);
  const Scales sc = host_scales(scales, n);
  cudaStream_t st = (cudaStream_t)stream;
#define MHC_EMBED(I, TW, TO) launch_embed_fwd<I, TW, TO>(ids, weight, out, tokens, n, hidden, vocab, sc, st)
#define MHC_EMBED_I(I)                                                                                    \
  (weight_bf16 ? (out_bf16 ? MHC_EMBED(I, __nv_bfloat16, __nv_bfloat16) : MHC_EMBED(I, __nv_bfloat16, float)) \
               : (out_bf16 ? MHC_EMBED(I, float, __nv_bfloat16) : MHC_EMBED(I, float, float)))
  return ids_64 ? MHC_EMBED_I(int64_t) : MHC_EMBED_I(int32_t);
#undef MHC_EMBED_I
#undef MHC_EMBED
}

extern "C" size_t mhc_stream_embedding_bwd_workspace_bytes(int64_t tokens, int64_t hidden) {
  if (tokens < 0 || hidden < 1) return 0;
  const GradPlan p = grad_plan(tokens, hidden);
  return 4 * p.list + p.ends;
}

extern "C" int mhc_stream_embedding_bwd(const void* grad_out, int32_t g_bf16, const void* ids, int32_t ids_64,
                                        void* grad_weight, int32_t gw_bf16, const float* scales, int64_t tokens,
                                        int32_t n, int64_t hidden, int64_t vocab, int64_t padding_idx, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  int rc = check_embed("stream_embedding_bwd", tokens, n, hidden, vocab, scales);
  if (rc) return rc;
  MHC_REQUIRE_PTR(grad_weight);
  MHC_REQUIRE(aligned16(grad_weight), MHC_ERR_ALIGNMENT, "stream_embedding_bwd: grad_weight must be 16-byte aligned");
  cudaStream_t st = (cudaStream_t)stream;
  const size_t gw_bytes = (size_t)vocab * (size_t)hidden * (gw_bf16 ? 2 : 4);
  if (tokens == 0) {
    cudaMemsetAsync(grad_weight, 0, gw_bytes, st);
    return check_launch("stream_embedding_bwd");
  }
  MHC_REQUIRE_PTR(grad_out);
  MHC_REQUIRE_PTR(ids);
  MHC_REQUIRE(workspace != nullptr && aligned16(workspace) &&
                  workspace_bytes >= mhc_stream_embedding_bwd_workspace_bytes(tokens, hidden),
              MHC_ERR_WORKSPACE, "stream_embedding_bwd: workspace too small");
  const Scales sc = host_scales(scales, n);
  const GradPlan pl = grad_plan(tokens, hidden);
  char* ws = (char*)workspace;
  uint32_t *ka = (uint32_t*)ws, *va = (uint32_t*)(ws + pl.list), *kb = (uint32_t*)(ws + 2 * pl.list),
           *vb = (uint32_t*)(ws + 3 * pl.list);
  float* ends = (float*)(ws + 4 * pl.list);
  // keys are 0 .. vocab: equal digits of at most 9 bits
  int kbits = 1;
  while ((vocab >> kbits) != 0) ++kbits;
  const int passes = (kbits + kDigitBits - 1) / kDigitBits, bits = (kbits + passes - 1) / passes;
  {
    ProfScope p("stream_embedding_sort", st);
    // clusters of 8 blocks: the first sorts, the others clear, up to two blocks an SM
    const uint64_t want = (gw_bytes + 16 * kSortThreads * 8 - 1) / (16 * kSortThreads * 8);
    const uint64_t most = 2 * (uint64_t)num_sms() - kSortBlocks;
    const unsigned zb = (unsigned)((want < most ? want : most) + kSortBlocks - 1) / kSortBlocks * kSortBlocks;
    const dim3 grid(kSortBlocks + zb);
    if (ids_64)
      embed_sort_kernel<int64_t><<<grid, kSortThreads, 0, st>>>((const int64_t*)ids, ka, va, kb, vb, (uint32_t)tokens,
                                                                (uint32_t)vocab, padding_idx, passes, bits,
                                                                (char*)grad_weight, gw_bytes);
    else
      embed_sort_kernel<int32_t><<<grid, kSortThreads, 0, st>>>((const int32_t*)ids, ka, va, kb, vb, (uint32_t)tokens,
                                                                (uint32_t)vocab, padding_idx, passes, bits,
                                                                (char*)grad_weight, gw_bytes);
    rc = check_launch("stream_embedding_sort");
    if (rc) return rc;
  }
  const uint32_t* keys = (passes & 1) ? kb : ka;
  const uint32_t* vals = (passes & 1) ? vb : va;
  // 16-byte loads of g, and stores of gW of 4 or 8 values
  const bool vec = hidden % (g_bf16 ? 8 : 4) == 0 && aligned16(grad_out);
#define MHC_SUMS(TG, TW, VV)                                                                                        \
  (vec ? launch_embed_sums<TG, TW, VV, 1>(keys, vals, grad_out, grad_weight, ends, tokens, n, hidden, vocab, sc, pl, st) \
       : launch_embed_sums<TG, TW, 1, 4>(keys, vals, grad_out, grad_weight, ends, tokens, n, hidden, vocab, sc, pl, st))
  return g_bf16 ? (gw_bf16 ? MHC_SUMS(__nv_bfloat16, __nv_bfloat16, 8) : MHC_SUMS(__nv_bfloat16, float, 8))
                : (gw_bf16 ? MHC_SUMS(float, __nv_bfloat16, 4) : MHC_SUMS(float, float, 4));
#undef MHC_SUMS
}
