// Weight gradient of a linear layer from its input kept in 8 bits, on tcgen05:
//   gW[o, k] = sum_t g[t, o] xh[t, k]
//
// xh is exact in bf16 (checkpoint8.cuh), so a bf16 g makes every product exact
// and the sum is formed in fp32 in tensor memory.  An fp32 g is cut into three
// bf16 terms of 8 significant bits each (exact, by truncation), three MMAs a
// step.
//
// A pair of CTAs (cta_group::2) computes 256 x 256 tiles of gW: M = 256 rows o
// (A = g, 128 of them in each CTA), N = 256 columns k (B = xh, 128 expanded by
// each CTA).  Both operands are MN-major: a token is a row of g and of the
// codes, and the contraction runs over tokens, so neither is transposed.  Why a
// pair: a CTA then expands and stores 128 columns for 128 x 256 products; alone
// it would expand 256, and with the MMAs' own operand reads that is more than
// shared memory's 128 bytes a cycle.
//
// Warps of a CTA: 0 issues the TMA loads of g, 1 the MMAs (of the pair, in the
// even CTA), 2 owns the tensor memory and issues the TMA loads of the codes, 3
// reports g's arrival to the even CTA, 4..11 take finished accumulators, 12..19
// expand: two groups of four warps, each every other stage (a stage is 64
// tokens), turn codes into xh in the 128-byte-swizzled layout that the MMA reads.
// Two accumulators of 256 columns fill tensor memory, so one is read while the
// next is summed.
//
// Accumulating MMAs truncate (a relative shrink of about 2e-8 each, measured on
// the layer's projection), so a chain is kept to 64 MMAs; warps 4..11 add the
// chains in fp32 registers, 128 a thread, which is why registers are moved
// between the roles (setmaxnreg).
//
// 8192 tokens, 4096 x 4096: 280 us a call in a continuous run, 985 TFLOP/s, 60% of
// what cuBLAS reaches in bf16 in a burst and 70% of what it sustains (243 us in
// short runs, 220 under the profiler on a cool GPU).  There the tensor pipe is 67%
// busy, a stage takes about 980 cycles for 512 of MMAs (the operands' traffic alone
// is 640 of shared memory; the rest is hand-overs).
#include "checkpoint8.cuh"
#include "tma.cuh"

namespace mhc {
namespace {

constexpr int kTok = 64;                       // tokens of a stage
constexpr int kTileO = 256, kTileK = 256;      // tile of a pair
constexpr uint32_t kOpBytes = kTok * 128 * 2;  // one operand of one CTA, one stage: 64 tokens x 128 bf16
constexpr int kOutWarp = 4, kOutWarps = 8, kExpandWarp = 12, kExpandWarps = 8;
constexpr int kThreads = 32 * (kExpandWarp + kExpandWarps);
// registers a thread by role; launched with 96 each, and 128 x 32 + 256 x 160 +
// 256 x 64 = 640 x 96
constexpr int kRegsFew = 32, kRegsOut = 160, kRegsExpand = 64;

template <int PLANES>
struct WgCfg {
  static constexpr uint32_t STAGE = (PLANES + 1) * kOpBytes;  // A planes, then B
  static constexpr int STAGES = PLANES == 1 ? 5 : 2;
  static constexpr int CODES = PLANES == 1 ? 4 : 8;           // stages of codes: 64 tokens x 128 bytes each
  // Parities tell a phase from the next only.  A group that has stored stage i knows
  // that the MMAs of stage i - STAGES are done, so before it waits for those of
  // i + 2 - STAGES no earlier phase of that barrier is open; and it meets a stage
  // of codes again itself.
  static_assert(STAGES >= 2 && CODES % 2 == 0, "two groups");
  static constexpr int CHAIN = PLANES == 1 ? 16 : 5;          // stages summed in tensor memory: 64 / 60 MMAs
  static constexpr uint32_t OFF_CODES = STAGES * STAGE;
  static constexpr uint32_t OFF_OUT = OFF_CODES + CODES * kOpBytes / 2;  // 4 KB a warp that writes: 32 x 32 values on their way out
  static constexpr uint32_t OFF_BAR = OFF_OUT + kOutWarps * 4096;
  static constexpr uint32_t SMEM = OFF_BAR + (3 * STAGES + 2 * CODES + 5) * 8 + 16 + 1024;  // + alignment of the ring
  static_assert(SMEM <= 232448, "227 KB a block");
};

struct WgArgs {
  const uint8_t* exps;
  void* gw;
  float* part;           // parts of split tiles: [unit][256][256]
  int64_t T, O, K, pitch;
  int tiles_o, tiles_k;
  int full, splits;      // whole tiles, then each further tile in `splits` parts along the tokens
  int units;
};

// Work of a pair: unit u is a whole tile or a part of one, as a range of stages.
struct Unit {
  int tile_o, tile_k, s0, s1, part;  // part < 0: into gw
};
__device__ __forceinline__ Unit unit_of(const WgArgs& a, int u) {
  Unit r;
  const int nst = (int)((a.T + kTok - 1) / kTok);
  int tile = u;
  r.s0 = 0; r.s1 = nst; r.part = -1;
  if (u >= a.full) {
    const int v = u - a.full, s = v % a.splits;
    tile = a.full + v / a.splits;
    r.part = v;
    r.s0 = (int)((int64_t)nst * s / a.splits);
    r.s1 = (int)((int64_t)nst * (s + 1) / a.splits);
  }
  // bands of 8 tile columns, rows of tiles within a band: pairs that run
  // together read the same few rows of tiles and the same 8 columns from L2
  constexpr int BAND = 8;
  const int band = tile / (BAND * a.tiles_o), w = min(BAND, a.tiles_k - band * BAND), in = tile - band * BAND * a.tiles_o;
  r.tile_o = in / w;
  r.tile_k = band * BAND + in % w;
  return r;
}

__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrive on the barrier at this offset in the even CTA.  What is handed over is
// this CTA's own shared memory (already fenced to the async proxy by its
// writers) and tensor memory, so the release need not reach past the CTA: at
// cluster scope it waits for the warp's code loads in flight, and the 4096^2
// product of 8192 tokens took 648 us instead of 379.
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  asm volatile(
      "{\n .reg .b32 ra;\n mapa.shared::cluster.u32 ra, %0, 0;\n"
      " mbarrier.arrive.shared::cluster.b64 _, [ra];\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ bool poll_cluster(uint32_t addr, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(addr), "r"(parity), "r"(kSuspendNs)
      : "memory");
  return done != 0;
}
// Bounded wait; gives up early once another warp of the CTA has.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* stop) {
  const uint32_t addr = smem_u32(bar);
  if (poll_cluster(addr, parity)) return true;
  const uint64_t t0 = global_ns();
  for (uint32_t it = 0; it < kSpinLimit; ++it) {
    if (poll_cluster(addr, parity)) return true;
    if (*stop) return false;
    if (global_ns() - t0 > kWaitLimitNs) break;
  }
  atomicExch(&g_mhc_device_error, 1);
  *stop = 1;
  return false;
}

// MN-major operand, 128-byte swizzle: atoms of 64 elements x 8 tokens, the next
// 64 elements 8192 bytes on, the next 8 tokens 1024
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// D fp32, A and B bf16, both MN-major, 256 x 256
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) | ((kTileK >> 3) << 17) |
                            ((kTileO >> 4) << 24);
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(kIdesc), "r"(accumulate)
      : "memory");
}
// arrives at this offset in both CTAs once the pair's MMAs issued so far are done
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
}
template <int R>
__device__ __forceinline__ void more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

// Two codes -> two bf16 values.  With the low 7 bits set into the mantissa of
// 128 (0x43nn) a byte reads 128 + low7; less 128, or 256 where its sign is set,
// that is the code, and the product with the power-of-two step is exact.
// sel picks the two bytes.
__device__ __forceinline__ uint32_t expand2(uint32_t low, uint32_t sign, uint32_t sel, __nv_bfloat162 step) {
  uint32_t a = __byte_perm(low, 0x43434343u, sel), k = __byte_perm(sign, 0x43434343u, sel);
  const __nv_bfloat162 d = __hmul2(__hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&k)), step);
  return *reinterpret_cast<const uint32_t*>(&d);
}

// Four values of an output row, `left` of them inside it.
__device__ __forceinline__ void put4(float* p, const float4& v, int64_t left) {
  if (left >= 4 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    *reinterpret_cast<float4*>(p) = v;
  } else {
    const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = w[j];
  }
}
__device__ __forceinline__ void put4(__nv_bfloat16* p, const float4& v, int64_t left) {
  if (left >= 4 && (reinterpret_cast<uintptr_t>(p) & 7) == 0) {
    __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
  } else {
    const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = __float2bfloat16_rn(w[j]);
  }
}

template <int PLANES, typename TW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    wgrad_kernel(const __grid_constant__ CUtensorMap gmap, const __grid_constant__ CUtensorMap cmap, const WgArgs a) {
  using Cfg = WgCfg<PLANES>;
  constexpr int S = Cfg::STAGES, SC = Cfg::CODES;
  extern __shared__ unsigned char raw[];
  unsigned char* ring = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);  // the same offset in both CTAs
  uint64_t* afull = reinterpret_cast<uint64_t*>(ring + Cfg::OFF_BAR);  // [S] this CTA's part of g has landed
  uint64_t* full = afull + S;                                          // [S] (even CTA) both operands of both CTAs
  uint64_t* empty = full + S;                                          // [S] the stage's MMAs are done
  uint64_t* cfull = empty + S;                                         // [SC] codes have landed
  uint64_t* cempty = cfull + SC;                                       // [SC] they have been read
  uint64_t* dfull = cempty + SC;                                       // [2] an accumulator is whole
  uint64_t* dempty = dfull + 2;                                        // [2] (even CTA) it has been read in both CTAs
  uint64_t* idle = dempty + 2;                                         // every MMA issued is done
  uint32_t* tslot = reinterpret_cast<uint32_t*>(idle + 1);
  volatile int* stop = reinterpret_cast<volatile int*>(tslot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tslot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  if (tid == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&afull[s], 1);
      mbar_init(&full[s], kExpandWarps + 2);  // a group of four warps and the report of g, in each CTA
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < SC; ++s) {
      mbar_init(&cfull[s], 1);
      mbar_init(&cempty[s], 4);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&dfull[b], 1);
      mbar_init(&dempty[b], 2 * kOutWarps);
    }
    mbar_init(idle, 1);
    *stop = 0;
    fence_mbar_init();
    prefetch_tmap(&gmap);
    prefetch_tmap(&cmap);
  }
  fence_before();
  __syncthreads();
  cluster_barrier();
  fence_after();
  const uint32_t tmem = *tslot;
  let_next_start();
  wait_for_previous();

  if (warp < kOutWarp) {
    fewer_regs<kRegsFew>();
    if (warp == 0) {
      if (lane == 0) {  // ---- g: two boxes of 64 columns x 64 tokens a plane ----
        int it = 0;
        for (int u = pair; u < a.units && !*stop; u += pairs) {
          const Unit q = unit_of(a, u);
          const int o = q.tile_o * kTileO + (int)rank * 128;
          for (int st = q.s0; st < q.s1; ++st, ++it) {
            const int s = it % S;
            if (it >= S && !wait_bar(&empty[s], (uint32_t)((it / S - 1) & 1), stop)) goto loads_done;
            unsigned char* dst = ring + s * Cfg::STAGE;
            mbar_expect_tx(&afull[s], PLANES * kOpBytes);
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
              tma_load_3d(dst + p * kOpBytes, &gmap, o, st * kTok, p, &afull[s]);
              tma_load_3d(dst + p * kOpBytes + kOpBytes / 2, &gmap, o + 64, st * kTok, p, &afull[s]);
            }
          }
        }
      loads_done:
        // nothing may land after the block is gone
        for (int j = it > S ? it - S : 0; j < it; ++j) mbar_wait(&afull[j % S], (uint32_t)((j / S) & 1));
      }
    } else if (warp == 1) {
      if (lane == 0 && rank == 0) {  // ---- MMAs of the pair ----
        int it = 0, acc = 0;
        for (int u = pair; u < a.units; u += pairs) {
          const Unit q = unit_of(a, u);
          for (int st = q.s0; st < q.s1; ++acc) {
            const int b = acc & 1, end = min(st + Cfg::CHAIN, q.s1);
            if (acc >= 2 && !wait_bar(&dempty[b], (uint32_t)((acc / 2 - 1) & 1), stop)) goto mma_done;
            fence_after();
            const uint32_t d = tmem + 256u * b;
            for (int first = st; st < end; ++st, ++it) {
              const int s = it % S;
              if (!wait_bar(&full[s], (uint32_t)((it / S) & 1), stop)) goto mma_done;
              fence_after();
              const uint32_t base = smem_u32(ring + s * Cfg::STAGE);
#pragma unroll
              for (int p = PLANES - 1; p >= 0; --p)  // smallest terms first
#pragma unroll
                for (int k = 0; k < kTok / 16; ++k)
                  mma_pair(d, mn_desc(base + p * kOpBytes + k * 2048), mn_desc(base + PLANES * kOpBytes + k * 2048),
                           (st > first || p < PLANES - 1 || k > 0) ? 1u : 0u);
              commit_pair(&empty[s]);
            }
            commit_pair(&dfull[b]);
          }
        }
      mma_done:
        commit_pair(idle);
        mbar_wait(idle, 0u);
      }
    } else if (warp == 2) {
      if (lane == 0) {  // ---- codes; columns past the rows' end and tokens past T read as zeros ----
        int it = 0;
        for (int u = pair; u < a.units && !*stop; u += pairs) {
          const Unit q = unit_of(a, u);
          for (int st = q.s0; st < q.s1; ++st, ++it) {
            const int s = it % SC;
            if (it >= SC && !wait_bar(&cempty[s], (uint32_t)((it / SC - 1) & 1), stop)) goto codes_done;
            mbar_expect_tx(&cfull[s], kOpBytes / 2);
            tma_load_2d(ring + Cfg::OFF_CODES + s * (kOpBytes / 2), &cmap, q.tile_k * kTileK + (int)rank * 128, st * kTok,
                        &cfull[s]);
          }
        }
      codes_done:
        for (int j = it > SC ? it - SC : 0; j < it; ++j) mbar_wait(&cfull[j % SC], (uint32_t)((j / SC) & 1));
      }
    } else if (warp == 3) {
      if (lane == 0) {  // ---- g has landed: tell the even CTA ----
        int it = 0;
        for (int u = pair; u < a.units && !*stop; u += pairs) {
          const Unit q = unit_of(a, u);
          for (int st = q.s0; st < q.s1; ++st, ++it) {
            if (!wait_bar(&afull[it % S], (uint32_t)((it / S) & 1), stop)) break;
            arrive_leader(&full[it % S]);
          }
        }
      }
    }
  } else if (warp >= kExpandWarp) {
    // ---- expand: a thread takes one block of 32 codes of two tokens a turn ----
    fewer_regs<kRegsExpand>();
    const int group = (warp - kExpandWarp) >> 2, e = tid & 127;
    const int tok = (e & 7) | ((e >> 5) << 3);  // eight lanes: eight tokens, so that 16-byte stores meet no bank twice
    const int blk = (e >> 3) & 3;               // under the swizzle; the second token is 32 on
    const uint32_t row = (uint32_t)(PLANES * kOpBytes + (blk >> 1) * (kOpBytes / 2) + tok * 128);
    const uint32_t from = (uint32_t)(Cfg::OFF_CODES + tok * 128);
    const int64_t wide = a.pitch / kCkBlock, turn = 2 * kTok * wide;
    // The exponents come from global memory, fetched two turns before their use:
    // the walk is over every other one of the pair's stages.
    int fu = pair, fs = 0, fe = 0;
    int64_t off = 0, t = 0;
    auto enter = [&](int over) {  // the first unit with more than `over` stages left to skip
      while (fu < a.units) {
        const Unit q = unit_of(a, fu);
        fs = q.s0 + over;
        fe = q.s1;
        if (fs < fe) {
          const int64_t k = (int64_t)q.tile_k * kTileK + rank * 128 + blk * 32;
          t = k < a.pitch ? (int64_t)fs * kTok + tok : a.T;  // no columns here: the codes are zeros
          off = t * wide + k / kCkBlock;
          return;
        }
        over = fs - fe;
        fu += pairs;
      }
    };
    auto fetch = [&](uint32_t (&ex)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ex[h] = 1u;
        if (fu < a.units && t + 32 * h < a.T) ex[h] = __ldg(a.exps + off + h * 32 * wide);
      }
      fs += 2;
      off += turn;
      t += 2 * kTok;
      if (fs >= fe && fu < a.units) {
        const int over = fs - fe;
        fu += pairs;
        enter(over);
      }
    };
    int total = 0;
    for (int u = pair; u < a.units; u += pairs) {
      const Unit q = unit_of(a, u);
      total += q.s1 - q.s0;
    }
    uint32_t e0[2], e1[2];
    enter(group);
    fetch(e0);
    fetch(e1);
    auto expand = [&](int it, uint32_t (&ex)[2]) -> bool {
      const int s = it % S, sc = it % SC;
      bool ok = wait_bar(&cfull[sc], (uint32_t)((it / SC) & 1), stop);
      if (!__all_sync(0xffffffffu, ok)) return false;
      uint4 c[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          c[h][j] = *reinterpret_cast<const uint4*>(ring + from + sc * (kOpBytes / 2) + h * 4096 + (((2 * blk + j) ^ (tok & 7)) << 4));
      ok = it < S || wait_bar(&empty[s], (uint32_t)((it / S - 1) & 1), stop);
      if (!__all_sync(0xffffffffu, ok)) return false;
      unsigned char* dst = ring + s * Cfg::STAGE + row;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint16_t sb = ex[h] == 255u ? 0x7fc0 : (uint16_t)(ex[h] << 7);
        const __nv_bfloat162 step = __halves2bfloat162(__ushort_as_bfloat16(sb), __ushort_as_bfloat16(sb));
        const uint32_t w[8] = {c[h][0].x, c[h][0].y, c[h][0].z, c[h][0].w, c[h][1].x, c[h][1].y, c[h][1].z, c[h][1].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 o;
          const uint32_t l0 = w[2 * j] & 0x7f7f7f7fu, s0 = w[2 * j] & 0x80808080u;
          const uint32_t l1 = w[2 * j + 1] & 0x7f7f7f7fu, s1 = w[2 * j + 1] & 0x80808080u;
          o.x = expand2(l0, s0, 0x4140, step);
          o.y = expand2(l0, s0, 0x4342, step);
          o.z = expand2(l1, s1, 0x4140, step);
          o.w = expand2(l1, s1, 0x4342, step);
          *reinterpret_cast<uint4*>(dst + h * 4096 + ((((blk & 1) * 4 + j) ^ (tok & 7)) << 4)) = o;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        arrive_leader(&full[s]);
        // Only now have all lanes used their codes.  Released straight after the
        // loads were issued, the stage was refilled under some of them.
        mbar_arrive(&cempty[sc]);
      }
      fetch(ex);
      return true;
    };
    for (int it = group; it < total; it += 4) {
      if (!expand(it, e0)) break;
      if (it + 2 < total && !expand(it + 2, e1)) break;
    }
  } else {
    // ---- accumulators -> fp32 sums -> gW or a part ----
    more_regs<kRegsOut>();
    const int w8 = warp - kOutWarp, q4 = w8 & 3, half = w8 >> 2;  // 32 rows, 128 columns a warp
    unsigned char* mine = ring + Cfg::OFF_OUT + w8 * 4096;
    const uint32_t src = tmem + ((uint32_t)(32 * q4) << 16) + 128u * half;
    int acc = 0;
    bool ok = true;
    for (int u = pair; u < a.units && ok; u += pairs) {
      const Unit q = unit_of(a, u);
      float sum[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) sum[j] = 0.f;
      for (int st = q.s0; st < q.s1; st += Cfg::CHAIN, ++acc) {
        const int b = acc & 1;
        ok = wait_bar(&dfull[b], (uint32_t)((acc / 2) & 1), stop);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v[16];
          tmem_ld16(src + 256u * b + 16u * i, v);
#pragma unroll
          for (int j = 0; j < 16; ++j) sum[16 * i + j] += v[j];
        }
        fence_before();
        __syncwarp();
        if (lane == 0) arrive_leader(&dempty[b]);
      }
      if (!ok) break;
      // 32 x 32 values at a time through shared memory (16-byte columns exchanged
      // by row, no bank twice), so that eight lanes write 128 bytes of a row
      const int r0 = (int)rank * 128 + 32 * q4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<float4*>(mine + lane * 128 + ((j ^ (lane & 7)) << 4)) =
              make_float4(sum[32 * i + 4 * j], sum[32 * i + 4 * j + 1], sum[32 * i + 4 * j + 2], sum[32 * i + 4 * j + 3]);
        __syncwarp();
        const int col = 128 * half + 32 * i + 4 * (lane & 7);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int r = 4 * j + (lane >> 3);
          const float4 v = *reinterpret_cast<const float4*>(mine + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
          if (q.part >= 0) {
            *reinterpret_cast<float4*>(a.part + ((int64_t)q.part * kTileO + r0 + r) * kTileK + col) = v;
          } else {
            const int64_t o = (int64_t)q.tile_o * kTileO + r0 + r, k = (int64_t)q.tile_k * kTileK + col;
            if (o < a.O) put4(reinterpret_cast<TW*>(a.gw) + o * a.K + k, v, a.K - k);
          }
        }
      }
    }
  }
  // the other CTA may still arrive here, or read this one's operands
  __syncwarp();
  __syncthreads();
  cluster_barrier();
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// Sum of a tile's parts, in order, into gW.
template <typename TW>
__global__ void __launch_bounds__(256)
    wgrad_join_kernel(const WgArgs a) {
  wait_for_previous();
  const Unit q = unit_of(a, a.full + (int)(blockIdx.x / (kTileO / 4)) * a.splits);
  const int rr = (blockIdx.x % (kTileO / 4)) * 4 + (threadIdx.x >> 6), c = (threadIdx.x & 63) * 4;
  const int64_t o = (int64_t)q.tile_o * kTileO + rr, k = (int64_t)q.tile_k * kTileK + c;
  if (o >= a.O || k >= a.K) return;
  const float* p = a.part + ((int64_t)q.part * kTileO + rr) * kTileK + c;
  float4 s = *reinterpret_cast<const float4*>(p);
  for (int i = 1; i < a.splits; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(p + (int64_t)i * kTileO * kTileK);
    s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
  }
  TW* d = reinterpret_cast<TW*>(a.gw) + o * a.K + k;
  const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (k + j < a.K) ck_store(d + j, v[j]);
}

// g as bf16 planes [PLANES][T][width] for the TMA: fp32 cut into three terms of
// 8 bits by truncation (their sum is exact), or rows that the TMA cannot read
// (start or stride not a multiple of 16 bytes) copied.
template <typename TG>
__global__ void __launch_bounds__(256)
    wgrad_planes_kernel(const TG* __restrict__ g, int64_t stride, __nv_bfloat16* __restrict__ out, int64_t T, int64_t O,
                        int64_t width) {
  let_next_start();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < T * width; i += (int64_t)gridDim.x * 256) {
    const int64_t t = i / width, o = i - t * width;
    if constexpr (sizeof(TG) == 2) {
      out[i] = o < O ? g[t * stride + o] : __float2bfloat16_rn(0.f);
    } else {
      float r = o < O ? g[t * stride + o] : 0.f;
      const bool fine = (__float_as_uint(r) & 0x7f800000u) != 0x7f800000u;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        const uint32_t top = __float_as_uint(r) & 0xffff0000u;
        const bool nan = !fine && p == 0 && r != r;
        out[(int64_t)p * T * width + i] = __ushort_as_bfloat16(nan ? (uint16_t)0x7fc0 : (uint16_t)(top >> 16));
        r = fine ? r - __uint_as_float(top) : 0.f;
      }
    }
  }
}

struct WgPlan {
  int tiles_o, tiles_k, full, splits, pairs, units;
  int64_t width;
  size_t part_bytes;
};
WgPlan wg_plan(int64_t T, int64_t O, int64_t K) {
  WgPlan p;
  p.tiles_o = (int)((O + kTileO - 1) / kTileO);
  p.tiles_k = (int)((K + kTileK - 1) / kTileK);
  p.width = (O + 7) / 8 * 8;
  const int tiles = p.tiles_o * p.tiles_k, most = num_sms() / 2;
  const int64_t stages = (T + kTok - 1) / kTok;
  // Whole rounds of tiles, one a pair; the tiles of the last, partial round are
  // split along the tokens over all pairs, at least 4 stages a part.
  const int rest = tiles % most;
  p.full = tiles - rest;
  p.splits = 1;
  if (rest > 0) {
    int64_t s = most / rest;
    if (s > stages / 4) s = stages / 4;
    p.splits = s < 1 ? 1 : (int)s;
  }
  if (p.splits == 1) p.full = tiles;
  p.units = p.full + (tiles - p.full) * p.splits;
  p.pairs = p.units < most ? p.units : most;
  p.part_bytes = (size_t)(tiles - p.full) * p.splits * kTileO * kTileK * sizeof(float);
  return p;
}

template <int PLANES, typename TW>
int launch_wgrad(const CUtensorMap& map, const CUtensorMap& codes, const WgArgs& a, const WgPlan& pl, bool after_planes,
                 cudaStream_t st) {
  auto kern = wgrad_kernel<PLANES, TW>;
  constexpr uint32_t smem = WgCfg<PLANES>::SMEM;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return fail(MHC_ERR_CUDA, "checkpoint8_weight_grad: cannot reserve %u bytes of shared memory", smem);
  {
    ProfScope p("checkpoint8_weight_grad", st);
    const dim3 grid(2 * pl.pairs);
    if (after_planes) launch_early(kern, grid, dim3(kThreads), smem, st, map, codes, a);
    else kern<<<grid, kThreads, smem, st>>>(map, codes, a);
    const int rc = check_launch("checkpoint8_weight_grad");
    if (rc) return rc;
  }
  const int rest = pl.tiles_o * pl.tiles_k - pl.full;
  if (rest == 0) return MHC_OK;
  ProfScope p("checkpoint8_weight_join", st);
  launch_early(wgrad_join_kernel<TW>, dim3((unsigned)rest * (kTileO / 4)), dim3(256), 0, st, a);
  return check_launch("checkpoint8_weight_join");
}

}  // namespace

int wgrad_device_error(int* value, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(value, g_mhc_device_error, sizeof(int));
  const int zero = 0;
  if (e == cudaSuccess && reset) e = cudaMemcpyToSymbol(g_mhc_device_error, &zero, sizeof(int));
  return e == cudaSuccess ? MHC_OK : fail(MHC_ERR_CUDA, "mhc_device_error_word: %s", cudaGetErrorString(e));
}

}  // namespace mhc

using namespace mhc;

extern "C" size_t mhc_checkpoint8_weight_grad_workspace_bytes(int64_t tokens, int64_t out_features,
                                                              int64_t in_features, int32_t g_bf16, int32_t g_aligned) {
  if (tokens < 1 || out_features < 1 || in_features < 1) return 0;
  const WgPlan p = wg_plan(tokens, out_features, in_features);
  const size_t planes = g_bf16 && g_aligned ? 0 : (size_t)tokens * p.width * 2 * (g_bf16 ? 1 : 3);
  return (planes + 255) / 256 * 256 + p.part_bytes;
}

extern "C" int mhc_checkpoint8_weight_grad(const void* grad_out, int32_t g_bf16, int64_t row_stride,
                                           const int8_t* codes, const uint8_t* exponents, void* grad_weight,
                                           int32_t gw_bf16, int64_t tokens, int64_t out_features,
                                           int64_t in_features, void* workspace, size_t workspace_bytes,
                                           void* stream) {
  const char* what = "checkpoint8_weight_grad";
  MHC_REQUIRE(tokens >= 0 && out_features >= 1 && in_features >= 1, MHC_ERR_INVALID_ARG,
              "%s: tokens must be >= 0, out_features and in_features >= 1 (got %lld, %lld, %lld)", what,
              (long long)tokens, (long long)out_features, (long long)in_features);
  MHC_REQUIRE(tokens < (1ll << 30) && out_features <= (1ll << 21) && in_features <= (1ll << 21), MHC_ERR_UNSUPPORTED,
              "%s: %lld tokens, %lld x %lld features are too many", what, (long long)tokens, (long long)out_features,
              (long long)in_features);
  MHC_REQUIRE_PTR(grad_weight);
  cudaStream_t st = (cudaStream_t)stream;
  if (tokens == 0) {
    cudaMemsetAsync(grad_weight, 0, (size_t)out_features * (size_t)in_features * (gw_bf16 ? 2 : 4), st);
    return check_launch(what);
  }
  MHC_REQUIRE_PTR(grad_out);
  MHC_REQUIRE(row_stride >= out_features || tokens == 1, MHC_ERR_INVALID_ARG, "%s: row_stride %lld < out_features %lld",
              what, (long long)row_stride, (long long)out_features);
  MHC_REQUIRE(codes != nullptr && exponents != nullptr, MHC_ERR_INVALID_ARG, "%s: codes and exponents must not be NULL",
              what);
  MHC_REQUIRE(aligned16(codes) && (reinterpret_cast<uintptr_t>(exponents) & 3) == 0, MHC_ERR_ALIGNMENT,
              "%s: codes must be 16-byte and exponents 4-byte aligned", what);
  const WgPlan pl = wg_plan(tokens, out_features, in_features);
  const bool copy = !g_bf16 || !aligned16(grad_out) || (row_stride % 8) != 0;
  const size_t planes = ((size_t)tokens * pl.width * 2 * (g_bf16 ? 1 : 3) + 255) / 256 * 256;
  const size_t need = (copy ? planes : 0) + pl.part_bytes;
  MHC_REQUIRE(need == 0 || (workspace != nullptr && aligned16(workspace) && workspace_bytes >= need),
              MHC_ERR_WORKSPACE, "%s: workspace too small", what);
  const void* src = grad_out;
  int64_t stride = tokens == 1 ? pl.width : row_stride;
  char* ws = (char*)workspace;
  if (copy) {
    ProfScope p("checkpoint8_weight_planes", st);
    const int64_t blocks = (tokens * pl.width + 1023) / 1024, most = 16ll * num_sms();
    const unsigned nb = (unsigned)(blocks < most ? blocks : most);
    if (g_bf16)
      wgrad_planes_kernel<<<nb, 256, 0, st>>>((const __nv_bfloat16*)grad_out, row_stride, (__nv_bfloat16*)ws, tokens,
                                              out_features, pl.width);
    else
      wgrad_planes_kernel<<<nb, 256, 0, st>>>((const float*)grad_out, row_stride, (__nv_bfloat16*)ws, tokens,
                                              out_features, pl.width);
    const int rc = check_launch("checkpoint8_weight_planes");
    if (rc) return rc;
    src = ws;
    stride = pl.width;
    ws += planes;
  }
  CUtensorMap map;
  const int np = g_bf16 ? 1 : 3;
  if (!make_tmap_3d(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, src, copy ? pl.width : out_features, tokens, np, stride * 2,
                    copy ? (uint64_t)tokens * pl.width * 2 : (uint64_t)stride * 2, 64, kTok, 1,
                    CU_TENSOR_MAP_SWIZZLE_128B))
    return fail(MHC_ERR_CUDA, "%s: cannot encode the tensor map", what);
  CUtensorMap cmap;
  if (!make_tmap_2d(&cmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, tokens, ck_pitch(in_features), ck_pitch(in_features),
                    kTok, 128, CU_TENSOR_MAP_SWIZZLE_128B))
    return fail(MHC_ERR_CUDA, "%s: cannot encode the tensor map", what);
  WgArgs a;
  a.exps = exponents; a.gw = grad_weight; a.part = (float*)ws;
  a.T = tokens; a.O = out_features; a.K = in_features; a.pitch = ck_pitch(in_features);
  a.tiles_o = pl.tiles_o; a.tiles_k = pl.tiles_k; a.full = pl.full; a.splits = pl.splits; a.units = pl.units;
  if (g_bf16)
    return gw_bf16 ? launch_wgrad<1, __nv_bfloat16>(map, cmap, a, pl, copy, st) : launch_wgrad<1, float>(map, cmap, a, pl, copy, st);
  return gw_bf16 ? launch_wgrad<3, __nv_bfloat16>(map, cmap, a, pl, copy, st) : launch_wgrad<3, float>(map, cmap, a, pl, copy, st);
}
