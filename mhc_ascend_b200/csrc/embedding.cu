// Embedding lookup into residual streams and the gradient of its table.
//
//   out[t, i, :] = s_i W[id_t, :]                         (i < n streams)
//   gW[v, :]     = sum over t with id_t = v of sum_i s_i g[t, i, :]
//
// The gradient goes by sorted tokens: (id, t) pairs are sorted (stable), so
// that each table row's terms are neighbours.  They are added in an order that
// the inputs' shape and ids alone decide: in token order within a chunk of at most
// 64 sorted positions, then the chunks' sums (past 256 of them as eight interleaved
// shares).  No float atomics: the same inputs give the same bits.
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
// tokens, lanes along the row; the row is read once for its n copies.  [8192] of
// [65536, 4096], n = 4, about 3600 different ids: fp32 106 us against 91 for the
// rows and the streams at the copy rate, bf16 54 against 46.  Uneven rows go one
// value a lane: [8192, 4, 4095] fp32 155 us, bf16 97, [100003, 2, 1281] bf16 309,
// 1.7 TB/s (2-byte stores).
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
// gradient, launch 1: the sort.  16 blocks, one cluster, sort (key, t) by radix
// digits of up to 9 bits, least significant first; block c owns the c-th sixteenth
// of the positions.  Per digit: a histogram of the block's range in shared memory;
// the exclusive sums over digits and blocks from the others' histograms through
// distributed shared memory; then tiles of 4096 positions are ranked (per warp by
// ballots, across warps by a column sum) and scattered.  The lists stay in L2.
// Padding and invalid ids get the key V and sort last.  (Clusters of 8: 103 us at
// 100003 tokens against 63; ranking by match instructions in place of ballots:
// 15% slower.)
// launch 2, at the same time: zeros over gW, which is most of what is written.  It
// may start as soon as the sort has (programmatic launch) and ends after it, so
// that what follows finds both done.  In one kernel with the sort, whose
// registers and clusters leave a block an SM, 1.07 GB took 197 us, here 143 us
// (a block for each 16 KB: 8 blocks an SM that walk on took 170).
// ---------------------------------------------------------------------------
constexpr int kZeroThreads = 256, kZeroUnroll = 4;

__global__ void __launch_bounds__(kZeroThreads)
    embed_zero_kernel(uint4* __restrict__ zero, uint64_t bytes) {
  let_next_start();
  const uint64_t units = bytes / 16, u = (uint64_t)blockIdx.x * (kZeroThreads * kZeroUnroll) + threadIdx.x;
#pragma unroll
  for (int j = 0; j < kZeroUnroll; ++j)
    if (u + j * kZeroThreads < units) zero[u + j * kZeroThreads] = make_uint4(0u, 0u, 0u, 0u);
  if (blockIdx.x == 0) {
    if (threadIdx.x < (bytes & 15)) reinterpret_cast<char*>(zero)[units * 16 + threadIdx.x] = 0;
    // One block that waits for the sort keeps the whole launch from ending before
    // it; were all to wait, the first of them would keep the others out.
    wait_for_previous();
  }
}

constexpr int kSortBlocks = 16, kSortThreads = 512, kSortItems = 8, kSortTile = kSortThreads * kSortItems;
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits, kSortWarps = kSortThreads / 32;

template <typename I>
__global__ void __cluster_dims__(kSortBlocks, 1, 1) __launch_bounds__(kSortThreads)
    embed_sort_kernel(const I* __restrict__ ids, uint2* la, uint2* lb, uint32_t T,
                      uint32_t vocab, int64_t pad, int passes, int bits) {
  const int tid = threadIdx.x;
  let_next_start();  // the zeros need nothing of this
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
    const uint2* in = (p & 1) ? lb : la;  // (key, token)
    uint2* out = (p & 1) ? la : lb;
    auto key_at = [&](uint32_t i) -> uint32_t {
      if (p > 0) return __ldcg(&in[i].x);
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
    uint2 item[kSortItems];
    auto fetch = [&](uint32_t t0) {
#pragma unroll
      for (int k = 0; k < kSortItems; ++k) {
        const uint32_t i = t0 + warp * (32 * kSortItems) + lane + 32 * k;
        item[k] = make_uint2(0xffffffffu, 0u);
        if (i < hi) item[k] = p > 0 ? __ldcg(in + i) : make_uint2(key_at(i), i);
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
        const uint32_t d = (item[k].x >> shift) & mask;
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
        if (wfirst + 32 * k < hi)
          __stcg(out + wcnt[warp][(item[k].x >> shift) & mask] + place[k], item[k]);
      if (t0 + kSortTile < hi) fetch(t0 + kSortTile);
      __syncthreads();
    }
    cluster.sync();  // release / acquire: the lists are whole before the next digit reads them
  }
}

// ---------------------------------------------------------------------------
// gradient, launch 3: sums of the sorted positions, `chunk` of them and a slice of
// the columns a block.  Rows whose tokens all lie in the chunk are written; the
// sums at its two ends, if their rows go on in a neighbour, are kept:
// ends[chunk][0] for a row that began before the chunk, [1] for one that begins in
// it and goes on.  Bound by reading g: 8 or 16 loads of a thread are in flight,
// and blocks that run together read neighbouring slices of the same rows.
// A thread has 16 bytes of columns.
// launch 4: for each row that begins in a chunk and goes on, its sums are added
// in chunk order and the row is written.
// ---------------------------------------------------------------------------
constexpr int kMaxChunk = 64, kSumThreads = 128, kJoinThreads = 256;

// 16 bytes from an address of any alignment, as 4 words: of two aligned accesses, a
// shift by words, then by bits.  The second access is the next lane's first and
// comes from it by shuffles (read again: 166 us against 158 below).  The
// accesses of several rows are issued before the first shift waits for one.
__device__ __forceinline__ void shift16(uint32_t sh, const uint4& a, const uint4& b, uint32_t (&o)[4]) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t t[6], u[5];
#pragma unroll
  for (int j = 0; j < 6; ++j) t[j] = (sh & 8) ? w[j + 2] : w[j];
#pragma unroll
  for (int j = 0; j < 5; ++j) u[j] = (sh & 4) ? t[j + 1] : t[j];
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = __funnelshift_r(u[j], u[j + 1], (sh & 3) * 8);
}
__device__ __forceinline__ void unit_of_words(const float*, const uint32_t (&o)[4], float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(o[j]);
}
__device__ __forceinline__ void unit_of_words(const __nv_bfloat16*, const uint32_t (&o)[4], float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(o[j] << 16);
    v[2 * j + 1] = __uint_as_float(o[j] & 0xffff0000u);
  }
}

// EVEN: rows of g start on 16 bytes and gW's on four values.  Elsewhere bf16 rows
// are read by shifts and their sums go through shared memory, so that the stores
// are coalesced; fp32 rows are read and written one value a lane ([8192, 4, 4095]:
// 118 us against 162 by shifts, whose registers halve what is in flight; bf16
// [100003, 2, 1281] 152 us by shifts, 268 one value a lane).  What bounds bf16
// there is latency: a warp's four rows in flight, then their sums, then the next
// four; six rows, or registers for more blocks, were slower.
template <typename TG, typename TW, bool EVEN>
__global__ void __launch_bounds__(kSumThreads)
    embed_sum_kernel(const uint2* __restrict__ list, const TG* __restrict__ g, TW* __restrict__ gw,
                     float* __restrict__ ends, uint32_t T, uint32_t vocab, int n, int64_t C,
                     const __grid_constant__ Scales sc, int chunk, uint32_t slices) {
  constexpr int V = 16 / (int)sizeof(TG);
  constexpr int L = EVEN ? 8 : 4;  // rows of g in flight
  constexpr bool SINGLE = !EVEN && sizeof(TG) == 4;
  const int width = blockDim.x;
  let_next_start();
  wait_for_previous();
  __shared__ uint32_t sk[kMaxChunk + 2], sv[kMaxChunk];
  __shared__ float ss[kMaxStreams];
  __shared__ float sums[EVEN || SINGLE ? 1 : kSumThreads * V];
  const uint32_t piece = blockIdx.x / slices;
  const uint32_t p0 = piece * chunk;
  const int tid = threadIdx.x;
  for (int j = tid; j < chunk + 2; j += width) {  // sk[1 + j] = key at p0 + j; neighbours on both sides
    const int64_t q = (int64_t)p0 + j - 1;
    const uint2 e = q >= 0 && q < (int64_t)T ? list[q] : make_uint2(0xffffffffu, 0u);
    sk[j] = e.x;
    if (j >= 1 && j <= chunk) sv[j - 1] = e.y;
  }
  if (tid < n) ss[tid] = sc.s[tid];  // n <= 32 <= width
  __syncthreads();
  int len = (int)min((uint32_t)chunk, T - p0);
  while (len > 0 && sk[len] >= vocab) --len;  // padding sorts last
  if (len == 0) return;
  const int64_t c0 = (int64_t)(blockIdx.x - piece * slices) * (width * V), c = c0 + tid * (SINGLE ? 1 : V);
  const int have = SINGLE ? (int)max((int64_t)0, min((int64_t)V, (C - c + width - 1) / width))
                          : (int)max((int64_t)0, min((int64_t)V, C - c));
  if ((EVEN || SINGLE) && have == 0) return;
  // The aligned accesses around a unit stay inside the tensor unless its token is
  // the first or the last one, or rows are shorter than such an access.
  auto edge = [&](uint32_t token) { return token == 0 || token == T - 1 || C < 16; };
  const bool last = (tid & 31) == 31 || c + V >= C;  // no next lane that loads
  float acc[V];
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
  int p = 0, i = 0;  // what is added next: stream i of position p
  int first = 0;     // first position of the running row
  const int total = len * n;
  int lp = 0, li = 0;
  const TG* at = g + (int64_t)sv[0] * n * C + c;  // what is loaded next
  for (int q = 0; q < total; q += L) {
    uint4 v[L], w[EVEN || SINGLE ? 1 : L];
    uint32_t sh[EVEN || SINGLE ? 1 : L];
#pragma unroll
    for (int k = 0; k < L; ++k)
      if (q + k < total) {
        if constexpr (EVEN) {
          v[k] = __ldcs(reinterpret_cast<const uint4*>(at));
        } else if constexpr (SINGLE) {
          const uint32_t* word = reinterpret_cast<const uint32_t*>(at);
          v[k].x = word[0];
          if (have > 1) v[k].y = word[width];
          if (have > 2) v[k].z = word[2 * width];
          if (have > 3) v[k].w = word[3 * width];
        } else {
          sh[k] = edge(sv[lp]) ? 16u : (uint32_t)reinterpret_cast<uintptr_t>(at) & 15u;  // the same in every lane
          if (have > 0 && sh[k] < 16) {
            const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(at) & ~(uintptr_t)15);
            v[k] = base[0];
            if (last) w[k] = base[1];
          }
        }
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
        float u[V];
        if constexpr (EVEN || SINGLE) {
          const uint32_t o[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
          unit_of_words(g, o, u);
        } else if (sh[k] < 16) {
          uint4 next;
          next.x = __shfl_down_sync(0xffffffffu, v[k].x, 1);
          next.y = __shfl_down_sync(0xffffffffu, v[k].y, 1);
          next.z = __shfl_down_sync(0xffffffffu, v[k].z, 1);
          next.w = __shfl_down_sync(0xffffffffu, v[k].w, 1);
          uint32_t o[4];
          shift16(sh[k], v[k], last ? w[k] : next, o);
          unit_of_words(g, o, u);
        } else {
          const TG* from = g + ((int64_t)sv[p] * n + i) * C + c;
#pragma unroll
          for (int j = 0; j < V; ++j) u[j] = j < have ? ck_f32(from[j]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = fmaf(s, u[j], acc[j]);
        if (++i == n) {
          i = 0;
          const uint32_t key = sk[p + 1];
          const bool more = p + 1 < len && sk[p + 2] == key;
          if (!more) {
            const bool before = first == 0 && sk[0] == key;
            const bool after = p + 1 == len && sk[p + 2] == key;
            float* e = ends + ((int64_t)piece * 2 + (before ? 0 : 1)) * C;
            if (EVEN) {
              if (!before && !after) save_unit(gw + (int64_t)key * C + c, acc);
              else save_unit(e + c, acc);
            } else if (SINGLE) {
#pragma unroll
              for (int j = 0; j < V; ++j)
                if (j < have) {
                  if (!before && !after) ck_store(gw + (int64_t)key * C + c + j * width, acc[j]);
                  else e[c + j * width] = acc[j];
                }
            } else {
              float* mine = sums + (tid & ~31) * V;  // the warp's columns
              __syncwarp();
#pragma unroll
              for (int j = 0; j < V; ++j) mine[(tid & 31) * V + j] = acc[j];
              __syncwarp();
              const int64_t o = c0 + (tid & ~31) * V + (tid & 31);
              const int left = (int)min((int64_t)(32 * V), C - o);  // of the row, from this lane's first on
              if (!before && !after) {
                TW* to = gw + (int64_t)key * C + o;
#pragma unroll
                for (int j = 0; j < V; ++j)
                  if (32 * j < left) ck_store(to + 32 * j, mine[32 * j + (tid & 31)]);
              } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                  if (32 * j < left) e[o + 32 * j] = mine[32 * j + (tid & 31)];
              }
            }
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] = 0.f;
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
    embed_join_kernel(const uint2* __restrict__ list, TW* __restrict__ gw, const float* __restrict__ ends,
                      uint32_t T, uint32_t vocab, int64_t C, int chunk, uint32_t slices) {
  __shared__ __align__(16) float part[8][32 * V];
  wait_for_previous();
  const uint32_t piece = blockIdx.x / slices;
  const uint32_t p1 = (piece + 1) * chunk;  // first position of the next chunk (exists: the grid is one short)
  const uint32_t p0 = p1 - chunk;
  const uint32_t key = list[p1].x, last_key = list[p1 - 1].x, first_key = list[p0].x;
  const uint32_t before_key = p0 > 0 ? list[p0 - 1].x : ~0u;
  if (key >= vocab || last_key != key) return;          // no row goes on here
  if (first_key == key && before_key == key) return;    // it began in an earlier chunk
  uint32_t lo = p1, hi = T;                             // first position past the row
  while (lo < hi) {
    const uint32_t m = lo + (hi - lo) / 2;
    if (list[m].x > key) hi = m; else lo = m + 1;
  }
  const uint32_t last = (lo - 1) / chunk, count = last - piece;
  const int64_t c0 = (int64_t)(blockIdx.x - piece * slices) * (kJoinThreads * V);
  if (count <= 256) {
    const int64_t c = c0 + threadIdx.x * V;
    if (c >= C) return;
    float acc[V];
    load_unit(ends + ((int64_t)piece * 2 + 1) * C + c, acc);
#pragma unroll 16
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
  p.list = ((size_t)T * 8 + 255) / 256 * 256;
  const int64_t slices = (C + 511) / 512;
  p.chunk = kMaxChunk;
  while (p.chunk > 1 && (T + p.chunk - 1) / p.chunk * slices < 2048) p.chunk /= 2;
  p.chunks = (T + p.chunk - 1) / p.chunk;
  p.ends = (size_t)p.chunks * 2 * (size_t)C * sizeof(float);
  return p;
}

template <typename TG, typename TW, bool EVEN>
int launch_embed_sums(const uint2* list, const void* g, void* gw, float* ends, int64_t T,
                      int n, int64_t C, int64_t vocab, const Scales& sc, const GradPlan& pl, cudaStream_t st) {
  {
    // even slices of at most kSumThreads units of 16 bytes
    const int64_t units = (C * (int64_t)sizeof(TG) + 15) / 16, slices = (units + kSumThreads - 1) / kSumThreads;
    const int64_t threads = ((units + slices - 1) / slices + 31) / 32 * 32, blocks = pl.chunks * slices;

    MHC_REQUIRE(blocks < (1ll << 31), MHC_ERR_UNSUPPORTED, "stream_embedding_bwd: %lld tokens of %lld are too many",
                (long long)T, (long long)C);
    ProfScope p("stream_embedding_sum", st);
    launch_early(embed_sum_kernel<TG, TW, EVEN>, dim3((unsigned)blocks), dim3((unsigned)threads), 0, st, list, (const TG*)g,
                 (TW*)gw, ends, (uint32_t)T, (uint32_t)vocab, n, C, sc, pl.chunk, (uint32_t)slices);
    const int rc = check_launch("stream_embedding_sum");
    if (rc) return rc;
  }
  if (pl.chunks < 2) return MHC_OK;
  constexpr int W = EVEN ? 4 : 1;
  const int64_t slices = (C + kJoinThreads * W - 1) / (kJoinThreads * W), blocks = (pl.chunks - 1) * slices;
  MHC_REQUIRE(blocks < (1ll << 31), MHC_ERR_UNSUPPORTED, "stream_embedding_bwd: %lld tokens of %lld are too many",
              (long long)T, (long long)C);
  ProfScope p("stream_embedding_join", st);
  launch_early(embed_join_kernel<TW, W>, dim3((unsigned)blocks), dim3(kJoinThreads), 0, st, list, (TW*)gw, ends, (uint32_t)T,
               (uint32_t)vocab, C, pl.chunk, (uint32_t)slices);
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
  return 2 * p.list + p.ends;
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
  uint2 *la = (uint2*)ws, *lb = (uint2*)(ws + pl.list);
  float* ends = (float*)(ws + 2 * pl.list);
  // keys are 0 .. vocab: equal digits of at most 9 bits
  int kbits = 1;
  while ((vocab >> kbits) != 0) ++kbits;
  const int passes = (kbits + kDigitBits - 1) / kDigitBits, bits = (kbits + passes - 1) / passes;
  {
    ProfScope p("stream_embedding_sort", st);
    auto go = [&](auto kern, auto* id) -> int {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return fail(MHC_ERR_CUDA, "stream_embedding_bwd: no clusters of %d blocks", kSortBlocks);
      kern<<<kSortBlocks, kSortThreads, 0, st>>>(id, la, lb, (uint32_t)tokens, (uint32_t)vocab, padding_idx, passes, bits);
      return MHC_OK;
    };
    rc = ids_64 ? go(embed_sort_kernel<int64_t>, (const int64_t*)ids) : go(embed_sort_kernel<int32_t>, (const int32_t*)ids);
    if (rc) return rc;
    rc = check_launch("stream_embedding_sort");
    if (rc) return rc;
  }
  {
    ProfScope p("stream_embedding_zero", st);
    const uint64_t per = 16ull * kZeroThreads * kZeroUnroll, want = (gw_bytes + per - 1) / per;
    MHC_REQUIRE(want < (1ull << 31), MHC_ERR_UNSUPPORTED, "stream_embedding_bwd: a table of %lld x %lld is too large",
                (long long)vocab, (long long)hidden);
    const cudaError_t e = launch_early(embed_zero_kernel, dim3((unsigned)want), dim3(kZeroThreads), 0, st,
                                       (uint4*)grad_weight, (uint64_t)gw_bytes);
    MHC_REQUIRE(e == cudaSuccess, MHC_ERR_CUDA, "stream_embedding_zero: launch failed: %s", cudaGetErrorString(e));
    rc = check_launch("stream_embedding_zero");
    if (rc) return rc;
  }
  const uint2* list = (passes & 1) ? lb : la;
  const bool even = hidden % (g_bf16 ? 8 : 4) == 0 && aligned16(grad_out);
#define MHC_SUMS(TG, TW)                                                                                            \
  (even ? launch_embed_sums<TG, TW, true>(list, grad_out, grad_weight, ends, tokens, n, hidden, vocab, sc, pl, st)   \
        : launch_embed_sums<TG, TW, false>(list, grad_out, grad_weight, ends, tokens, n, hidden, vocab, sc, pl, st))
  return g_bf16 ? (gw_bf16 ? MHC_SUMS(__nv_bfloat16, __nv_bfloat16) : MHC_SUMS(__nv_bfloat16, float))
                : (gw_bf16 ? MHC_SUMS(float, __nv_bfloat16) : MHC_SUMS(float, float));
#undef MHC_SUMS
}
