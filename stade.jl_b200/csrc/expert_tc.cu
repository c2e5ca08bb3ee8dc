// Products grouped by expert on the tensor cores.
//
// One kernel, tcgen05.mma.cta_group::2 on 256 x 256 tiles, serves the three
// products of expert_mm and expert_mm_b. The MMA's M dimension (256 rows over
// the pair) is always the output's contiguous dimension and its N dimension
// the output's rows:
//
//               M         N              K          A (M x K)        B (N x K)
//   y  = x W    n_o       group's rows   n_i        W[e], M-major    x, K-major
//   xb = yb W^T n_i       group's rows   n_o        W[e], K-major    yb, K-major
//   wb = x^T yb n_o       n_i            its rows   yb, M-major      x, N-major
//
// so a group's ragged end costs what its rows cost: the last tile of a group
// issues MMAs only as wide as its rows (a multiple of 32), columns past the
// group are never stored, and neighbours' values there touch no other column.
// In the third product the ragged dimension is K: the last block's rows past
// the group are set to zero in shared memory, in both operands, before the
// MMAs read them.
//
// A Float32 operand is held as three bf16 planes whose sum is the value (8
// bits of mantissa each, rounded to nearest); the product is the six plane
// products down to 2^-16 of it, each an ordinary K loop over its two planes. The
// planes reach down to bf16's smallest value, 2^-133: operands below 2^-110 lose
// their last bits, below 2^-134 they count as 0. Where the five minor products'
// sum is not finite, an operand is infinite or NaN and the leading product
// gives the result alone: an infinity then stays one, as in a plain product.
//
// The tensor cores' Float32 sums truncate: their error grows with the number
// of MMAs into one accumulator, by about 2^-25 of it each. An accumulator takes
// a few blocks of 64 where the result is Float32 (kChain, kChain16), many where
// it is rounded to 16 bits (kChainRound), before the epilogue warps add it to
// round-to-nearest sums in registers.
//
// What bounds it: 16384 rows in 16 even groups, 2048 -> 4096 in bf16, run at
// 1.3 PFLOP/s for 20 ms (y 211 us, xb 213 us: 0.80 of the measured burst rate of
// a plain product) and at 1.05 for half a second, where the power limit holds
// the clock near 1.5 GHz (a loop of plain library products over the same groups:
// 272 us there, this kernel 260). wb takes 281 us: it also writes 537 MB of
// Float32 (237 us without the stores).
//
// Warp roles per CTA: 0 TMA loads, 1 (of the leader) MMAs, 2 .. 17 epilogue, 18
// zeroes the K tail. Every wait is bounded; one that runs out sets the device
// error word and the kernel leaves.

#include <algorithm>
#include <initializer_list>

#include "expert_tc.cuh"
#include "tcgen05.cuh"
#include "token_ops.cuh"

namespace stade {
namespace {

__device__ int g_expert_tc_error = 0;

using tc5::mbar_arrive;
using tc5::mbar_arrive_tx;
using tc5::mbar_init;
using tc5::smem_u32;
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
  return tc5::mbar_wait_cluster(bar, parity, &g_expert_tc_error);
}

constexpr int kTileN = kExpertTcRows;            // output rows of a tile
constexpr int kHalfM = 128;                      // M rows of one CTA of the pair
constexpr int kBlockK = 64;
constexpr int kTileBytes = 128 * kBlockK * 2;    // one operand tile of one CTA
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kStages = 6;
constexpr int kAcc = 2;                          // TMEM accumulators of kTileN columns
constexpr int kEpiWarps = 16;
constexpr int kThreads = (3 + kEpiWarps) * 32;
constexpr int kBars = 4 * kStages + 2 * kAcc + 1;
constexpr int kOutBytes = 2048;                  // a warp's 16 x 32 block of the output
constexpr int kSmem = kStages * kStageBytes + 1024 + 256 + kEpiWarps * kOutBytes;
static_assert(kSmem <= 232448, "shared memory of a CTA");
static_assert(kBars * 8 + 4 <= 256, "barrier block");
// K blocks of 64 per accumulator where the result is Float32. Measured relative
// error against 64 bits: 1.2e-7, 2.3e-7, 4.7e-7 and 1.0e-6 for 2, 4, 8 and 16
// blocks, whatever K is; weight gradient of 16384 rows in 16 groups, 2048 x
// 4096 in bf16: 365, 298, 285, 278 us (every chain hands an accumulator over).
// Float32 operands keep the tighter sums.
constexpr int kChain = 4, kChain16 = 8;
constexpr int kChainSmall = 64;  // the same for the plane products below 2^-7 of the result
constexpr int kChainRound = 256; // where it is rounded to 16 bits: 3e-5, whatever K is

struct Geom {
  int M;           // output's contiguous extent
  int m_tiles;
  int N;           // wgrad: n_i
  int n_tiles;
  int K;           // rows product: depth
  int planes;
  int chain;       // K blocks per accumulator of the leading product
  bool a_mn, b_mn, bf16, add;
  bool vec;        // output rows in 16-byte pieces
  int64_t ld;      // output row pitch
};

struct Unit {
  int expert, row, rows;   // rows product: tile; wgrad: the group
  int m0, n0, ncols, n_mma, nkb;
};

struct RowSrc {
  const ExpertTile* tiles;
  const int* count;
  __device__ __forceinline__ int total(const Geom& g) const { return *count * g.m_tiles; }
  __device__ __forceinline__ Unit get(int t, const Geom& g) const {
    const int4 v = *reinterpret_cast<const int4*>(tiles + t / g.m_tiles);
    Unit u;
    u.expert = v.x;
    u.row = v.y;
    u.rows = v.z;
    u.m0 = (t % g.m_tiles) * 2 * kHalfM;
    u.n0 = 0;
    u.ncols = v.z;
    u.n_mma = (v.z + 31) / 32 * 32;
    u.nkb = v.x < 0 ? 0 : (g.K + kBlockK - 1) / kBlockK;
    return u;
  }
};
struct GroupSrc {
  const int64_t* bounds;
  int n_e;
  __device__ __forceinline__ int total(const Geom& g) const { return n_e * g.m_tiles * g.n_tiles; }
  __device__ __forceinline__ Unit get(int t, const Geom& g) const {
    // whole tiles of all groups first, the narrow last ones after them: the
    // pairs that a last round leaves with one more unit then have a small one
    const int whole = g.N / kTileN, per = g.m_tiles * whole, first = n_e * per;
    Unit u;
    if (t < first) {
      u.expert = t / per;
      const int r = t - u.expert * per, n = r / g.m_tiles;
      u.m0 = (r - n * g.m_tiles) * 2 * kHalfM;
      u.n0 = n * kTileN;
    } else {
      u.expert = (t - first) / g.m_tiles;
      u.m0 = (t - first - u.expert * g.m_tiles) * 2 * kHalfM;
      u.n0 = whole * kTileN;
    }
    const int64_t a = bounds[u.expert], b = bounds[u.expert + 1];
    u.row = (int)a;
    u.rows = (int)(b - a);
    u.ncols = min(kTileN, g.N - u.n0);
    u.n_mma = (u.ncols + 31) / 32 * 32;
    u.nkb = (u.rows + kBlockK - 1) / kBlockK;
    return u;
  }
};

// The K loop of a unit: `small` blocks of the minor plane products, then nkb
// of the leading one, cut into accumulation chains.
struct Loop {
  int nkb, small, n_small, n_lead;
  __device__ __forceinline__ Loop(int nkb_, const Geom& g) : nkb(nkb_) {
    small = g.planes == 3 ? 5 * nkb : 0;
    n_small = (small + kChainSmall - 1) / kChainSmall;
    n_lead = (nkb + g.chain - 1) / g.chain;
  }
  __device__ __forceinline__ int blocks() const { return small + nkb; }
  __device__ __forceinline__ int chains() const { return max(1, n_small + n_lead); }
  __device__ __forceinline__ void chain(int c, const Geom& g, int* v0, int* v1) const {
    if (c < n_small) {
      *v0 = c * kChainSmall;
      *v1 = min(small, *v0 + kChainSmall);
    } else {
      *v0 = small + (c - n_small) * g.chain;
      *v1 = min(small + nkb, *v0 + g.chain);
    }
  }
  // block v: K block and the planes of A and B
  __device__ __forceinline__ void block(int v, int* kb, int* pa, int* pb) const {
    if (v >= small) {
      *kb = v - small;
      *pa = *pb = 0;
      return;
    }
    *kb = v / 5;
    const int p = v - *kb * 5;           // (0,2) (1,1) (2,0) (0,1) (1,0)
    *pa = p == 1 || p == 4 ? 1 : p == 2 ? 2 : 0;
    *pb = p == 1 || p == 3 ? 1 : p == 0 ? 2 : 0;
  }
};

// ---- output -------------------------------------------------------------------
// A warp's 32 (M) x 16 (output rows) block goes through shared memory so that
// it reaches memory as 16-byte pieces of output rows: straight from the
// accumulator's layout a thread has one value per output row, 16 stores of 2
// or 4 bytes with an address and a bound each (measured, 4096 x 512 x 4096 in
// bf16: 37.8 us with those, 30.0 with these). 16-bit blocks are transposed by
// stmatrix; rows of 64 bytes, 16-byte chunks swizzled so that the eight rows
// of a block fall into different banks. `add` adds the old values before the
// one rounding.
template <class Out>
__device__ __forceinline__ void pack2(float a, float b, uint32_t* r) {
  const Vec<Out, 2> v{{round_to<Out>(a), round_to<Out>(b)}};
  *r = *reinterpret_cast<const uint32_t*>(&v);
}

// Copies 16-byte chunks (or, without vec, single values) between the block in
// shared memory and output rows c0 .. of the tile, rows < ncols, M < lim.
template <class Out, bool LOAD>
__device__ __forceinline__ void copy_block(uint8_t* blk, Out* o, int64_t ld, int rows, int lim,
                                           bool vec, bool add, int lane) {
  constexpr int kPer = 16 / (int)sizeof(Out), kChunks = 32 / kPer;   // chunks of a row: 4 or 8
  auto at = [&](int row, int ch) {
    return blk + row * (kChunks * 16) + 16 * (sizeof(Out) == 2 ? ch ^ ((row >> 1) & 3) : ch);
  };
  if (vec) {
    const int ch = lane % kChunks;
#pragma unroll
    for (int it = 0; it < kChunks / 2; ++it) {
      const int row = it * (32 / kChunks) + lane / kChunks;
      if (row < rows && ch * kPer < lim) {
        int4* p = reinterpret_cast<int4*>(o + row * ld + ch * kPer);
        int4* s = reinterpret_cast<int4*>(at(row, ch));
        if (LOAD) {
          *s = *p;
        } else if (sizeof(Out) == 4 && add) {
          float4 a = *reinterpret_cast<float4*>(s);
          const float4 b = *reinterpret_cast<float4*>(p);
          a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
          *reinterpret_cast<float4*>(p) = a;
        } else {
          *p = *s;
        }
      }
    }
  } else if (lane < lim) {
#pragma unroll 1
    for (int row = 0; row < rows && row < 16; ++row) {
      Out* p = o + row * ld + lane;
      Out* s = reinterpret_cast<Out*>(at(row, lane / kPer)) + lane % kPer;
      if (LOAD) *s = *p;
      else *p = sizeof(Out) == 4 && add ? round_to<Out>(load_acc<Out>(*s) + load_acc<Out>(*p)) : *s;
    }
  }
}

template <class Out>
__device__ __forceinline__ void store_block(float (&sum)[16], uint8_t* blk, Out* o, int64_t ld,
                                            int rows, int lim, bool vec, bool add, int lane) {
  if constexpr (sizeof(Out) == 2) {
    const uint32_t base = smem_u32(blk);
    const int row = (lane & 7) + 8 * (lane >> 4), k = (lane >> 3) & 1;
    if (add) {
      copy_block<Out, true>(blk, o, ld, rows, lim, vec, add, lane);
      __syncwarp();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t a = base + row * 64 + 16 * ((2 * h + k) ^ ((row >> 1) & 3));
      uint32_t r[4];
      if (add) {
        tc5::ldmatrix4_trans(a, r);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const Vec<Out, 2> v = *reinterpret_cast<const Vec<Out, 2>*>(&r[b]);
          sum[8 * h + 2 * b] += load_acc<Out>(v.v[0]);
          sum[8 * h + 2 * b + 1] += load_acc<Out>(v.v[1]);
        }
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) pack2<Out>(sum[8 * h + 2 * b], sum[8 * h + 2 * b + 1], &r[b]);
      tc5::stmatrix4_trans(a, r);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) reinterpret_cast<float*>(blk)[j * 32 + lane] = sum[j];
  }
  __syncwarp();
  copy_block<Out, false>(blk, o, ld, rows, lim, vec, add, lane);
  __syncwarp();
}

// B's maps: boxes of 16, 32, 64 and 128 rows where B is K-major (a tile loads
// its rows with the smallest one that covers them: one copy a block whatever
// the width; pieces of 16 rows measured 85 us more on 16 uneven groups of
// 1,024 rows each, 2048 -> 4096), of 64 where it is N-major.
struct BMaps {
  CUtensorMap m[4];
};

template <bool WGRAD, class Src, class Out>
__global__ void __launch_bounds__(kThreads, 1)
expert_tc_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ BMaps bmaps,
                 Geom g, Src src, Out* __restrict__ out, int n_e) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* tiles = smem_raw + pad;
  uint64_t* bars = reinterpret_cast<uint64_t*>(tiles + kStages * kStageBytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kStages;
  const uint32_t tail0 = empty0 + 8 * kStages;      // K tail landed in this CTA
  const uint32_t ptail0 = tail0 + 8 * kStages;      // the leader's: the peer's tail is zeroed
  const uint32_t tfull0 = ptail0 + 8 * kStages, tempty0 = tfull0 + 8 * kAcc;
  const uint32_t done = tempty0 + 8 * kAcc;
  const uint32_t rank = tc5::cluster_rank();
  const bool leader = rank == 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;

  if (threadIdx.x == 32) {
    tc5::prefetch_map(&amap);
    for (int i = 0; i < 4; ++i) tc5::prefetch_map(&bmaps.m[i]);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
      mbar_init(tail0 + 8 * s, 1);
      mbar_init(ptail0 + 8 * s, 1);
    }
    for (int b = 0; b < kAcc; ++b) {
      mbar_init(tfull0 + 8 * b, 1);
      mbar_init(tempty0 + 8 * b, 2 * kEpiWarps);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tc5::tmem_alloc_pair(smem_u32(tmem_slot), 512);
  tc5::fence_before();
  tc5::cluster_sync();
  tc5::fence_after();
  const uint32_t tmem = *tmem_slot;
  after_previous();        // what is above overlaps the kernels that prepare the operands
  const int total = src.total(g);

  if (warp == 0) {
    if (lane == 0) {
      // ---- TMA loads (both CTAs) ------------------------------------------------
      int i = 0;
      bool ok = true;
      Unit u;
      if (pair < total) u = src.get(pair, g);
      for (int t = pair; t < total && ok; t += npairs) {
        Unit next = u;
        if (t + npairs < total) next = src.get(t + npairs, g);   // in flight during this unit
        const Loop lp(u.nkb, g);
        const int m0 = u.m0 + (int)rank * kHalfM;
        const int half = u.n_mma / 2;
        const int b0 = (WGRAD ? u.n0 : u.row) + (int)rank * half;
        // N-major: boxes of 64 columns; K-major: the map of 16 << bsel rows
        const int bboxes = (half + 63) / 64;
        const int bsel = WGRAD ? 0 : half > 64 ? 3 : half > 32 ? 2 : half > 16 ? 1 : 0;
        const CUtensorMap* bmap = &bmaps.m[bsel];
        const uint32_t bytes = kTileBytes + (WGRAD ? (uint32_t)bboxes * 8192u : 2048u << bsel);
        for (int v = 0; v < lp.blocks(); ++v, ++i) {
          const int s = i % kStages;
          if (!wait(empty0 + 8 * s, ((uint32_t)(i / kStages) & 1u) ^ 1u)) { ok = false; break; }
          int kb, pa, pb;
          lp.block(v, &kb, &pa, &pb);
          const int k0 = kb * kBlockK;
          const uint32_t sa = smem_u32(tiles + s * kStageBytes), sb = sa + kTileBytes;
          if (WGRAD && k0 + kBlockK > u.rows) {
            // the group's K tail: lands here first; warp 18 zeroes its rows past
            // the group, and the leader's arrives on `full` for both CTAs
            const uint32_t tb = tail0 + 8 * s;
            mbar_arrive_tx(tb, bytes);
            tc5::tma_load_3d(sa, &amap, m0, u.row + k0, pa, tb);
            tc5::tma_load_3d(sa + 8192, &amap, m0 + 64, u.row + k0, pa, tb);
            for (int q = 0; q < bboxes; ++q)
              tc5::tma_load_3d(sb + q * 8192, bmap, b0 + 64 * q, u.row + k0, pb, tb);
            continue;
          }
          const uint32_t fb = full0 + 8 * s;
          if (leader) mbar_arrive_tx(fb, 2 * bytes);
          if (WGRAD) {
            tc5::tma_load_3d_pair(sa, &amap, m0, u.row + k0, pa, fb);
            tc5::tma_load_3d_pair(sa + 8192, &amap, m0 + 64, u.row + k0, pa, fb);
            for (int q = 0; q < bboxes; ++q)
              tc5::tma_load_3d_pair(sb + q * 8192, bmap, b0 + 64 * q, u.row + k0, pb, fb);
          } else {
            const int we = pa * n_e + u.expert;
            if (g.a_mn) {
              tc5::tma_load_3d_pair(sa, &amap, m0, k0, we, fb);
              tc5::tma_load_3d_pair(sa + 8192, &amap, m0 + 64, k0, we, fb);
            } else {
              tc5::tma_load_3d_pair(sa, &amap, k0, m0, we, fb);
            }
            tc5::tma_load_3d_pair(sb, bmap, k0, b0, pb, fb);
          }
        }
        u = next;
      }
      // this CTA's copies land before it leaves: the leader sees them on its
      // own barriers, the peer when the leader's MMAs have read them
      for (int j = 0; j < kStages && j < i; ++j) {
        const int last = i - 1 - j;
        wait((leader ? full0 : empty0) + 8 * (last % kStages), (uint32_t)(last / kStages) & 1u);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ---- MMAs --------------------------------------------------------------------
      // descriptors of stage 0; a stage or a K step further is an addition in
      // the address field (building them per MMA kept this thread, not the
      // tensor cores, busy in the third product: 285 us there, 278 us so)
      const uint32_t s0 = smem_u32(tiles);
      const uint64_t a0 = tc5::desc_sw128(s0, g.a_mn ? 8192u : 16u, 1024u, 2u);
      const uint64_t b0 = tc5::desc_sw128(s0 + kTileBytes, g.b_mn ? 8192u : 16u, 1024u, 2u);
      const uint32_t a_step = (g.a_mn ? 2048u : 32u) >> 4, b_step = (g.b_mn ? 2048u : 32u) >> 4;
      int i = 0, c_all = 0;
      bool ok = true;
      Unit u;
      if (pair < total) u = src.get(pair, g);
      for (int t = pair; t < total && ok; t += npairs) {
        Unit next = u;
        if (t + npairs < total) next = src.get(t + npairs, g);
        const Loop lp(u.nkb, g);
        const uint32_t idesc = tc5::idesc_f16(2 * kHalfM, u.n_mma, g.bf16, g.a_mn, g.b_mn);
        for (int c = 0; c < lp.chains() && ok; ++c, ++c_all) {
          const int b = c_all % kAcc;
          const uint32_t acc = tmem + (uint32_t)(b * kTileN);
          if (!wait(tempty0 + 8 * b, ((uint32_t)(c_all / kAcc) & 1u) ^ 1u)) { ok = false; break; }
          tc5::fence_after();
          int v0, v1;
          lp.chain(c, g, &v0, &v1);
          // blocks that can be the group's K tail: the last one, and with
          // three planes any (each plane product has one)
          const int tail_from = lp.small ? 0 : lp.blocks() - 1;
          for (int v = v0; v < v1; ++v, ++i) {
            const int s = i % kStages;
            if (!wait(full0 + 8 * s, (uint32_t)(i / kStages) & 1u)) { ok = false; break; }
            tc5::fence_after();
            const uint64_t ad = a0 + (uint64_t)(s * (kStageBytes >> 4));
            const uint64_t bd = b0 + (uint64_t)(s * (kStageBytes >> 4));
            int rem = kBlockK;             // rows of the K block inside the group
            if (WGRAD && v >= tail_from) {
              int kb, pa, pb;
              lp.block(v, &kb, &pa, &pb);
              rem = u.rows - kb * kBlockK;
            }
#pragma unroll
            for (int j = 0; j < kBlockK / 16; ++j)
              if (16 * j < rem)
                tc5::mma_f16_pair(acc, ad + a_step * j, bd + b_step * j, idesc,
                                  v != v0 || j != 0 ? 1u : 0u);
            tc5::mma_commit_pair(empty0 + 8 * s);
          }
          tc5::mma_commit_pair(tfull0 + 8 * b);
        }
        u = next;
      }
      tc5::mma_commit_pair(done);
    }
    if (lane == 0) wait(done, 0);
    __syncwarp();
  } else if (warp == 2 + kEpiWarps) {
    if (WGRAD) {
      // ---- K tails (both CTAs) ---------------------------------------------------------
      int i = 0;
      uint32_t seen = 0;     // per stage: parity of its next tail
      bool ok = true;
      for (int t = pair; t < total && ok; t += npairs) {
        const Unit u = src.get(t, g);
        const Loop lp(u.nkb, g);
        if (u.rows % kBlockK == 0) {
          i += lp.blocks();
          continue;
        }
        const int half = u.n_mma / 2, bboxes = (half + 63) / 64;
        const int rem = u.rows % kBlockK, upto = (rem + 15) / 16 * 16;
        for (int v = 0; v < lp.blocks(); ++v, ++i) {
          int kb, pa, pb;
          lp.block(v, &kb, &pa, &pb);
          if (kb != u.nkb - 1) continue;
          const int s = i % kStages;
          ok = __all_sync(0xffffffffu, wait(tail0 + 8 * s, (seen >> s) & 1u));
          if (!ok) break;
          seen ^= 1u << s;
          uint8_t* st = tiles + s * kStageBytes;
          const int lines = (upto - rem) * (2 + bboxes);
          for (int l = lane; l < lines * 8; l += 32) {
            const int line = l >> 3, box = line % (2 + bboxes), row = rem + line / (2 + bboxes);
            uint8_t* base = box < 2 ? st + box * 8192 : st + kTileBytes + (box - 2) * 8192;
            *reinterpret_cast<int4*>(base + row * 128 + (l & 7) * 16) = make_int4(0, 0, 0, 0);
          }
          tc5::fence_async_smem();
          __syncwarp();
          if (leader) {
            ok = __all_sync(0xffffffffu, wait(ptail0 + 8 * s, ((seen >> s) & 1u) ^ 1u));
            if (!ok) break;
            if (lane == 0) mbar_arrive(full0 + 8 * s);
          } else if (lane == 0) {
            tc5::mbar_arrive_remote(tc5::mapa(ptail0 + 8 * s, 0));
          }
        }
      }
    }
  } else {
    // ---- epilogue (both CTAs) ---------------------------------------------------------
    const int e = warp - 2;
    const int quad = warp & 3;       // TMEM lanes 32 quad ..
    const int cg = e >> 2;           // 16-column groups cg, cg + 4, cg + 8, cg + 12
    const uint32_t tempty_leader = tc5::mapa(tempty0, 0);
    int c_all = 0;
    bool ok = true;
    Unit u;
    if (pair < total) u = src.get(pair, g);
    for (int t = pair; t < total && ok; t += npairs) {
      Unit next = u;
      if (t + npairs < total) next = src.get(t + npairs, g);
      const Loop lp(u.nkb, g);
      float sum[4][16];
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[q][j] = 0.f;
      for (int c = 0; c < lp.chains(); ++c, ++c_all) {
        const int b = c_all % kAcc;
        ok = __all_sync(0xffffffffu, wait(tfull0 + 8 * b, (uint32_t)(c_all / kAcc) & 1u));
        if (!ok) break;
        tc5::fence_after();
        if (u.nkb > 0) {
          const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * kTileN);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if ((cg + 4 * q) * 16 < u.n_mma) {     // uniform over the warp
              float v[16];
              if constexpr (sizeof(Out) == 2)
                tc5::tmem_ld16_frag(base + (uint32_t)((cg + 4 * q) * 16), v);
              else
                tc5::tmem_ld16(base + (uint32_t)((cg + 4 * q) * 16), v);
#pragma unroll
              for (int j = 0; j < 16; ++j) sum[q][j] += v[j];
            }
          }
          // an infinity's lower planes are 0, and the other operand's mostly, so
          // the minor products make NaN of it: the leading one alone has it right
          if (sizeof(Out) == 4 && c + 1 == lp.n_small) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int j = 0; j < 16; ++j) sum[q][j] = isfinite(sum[q][j]) ? sum[q][j] : 0.f;
          }
        }
        tc5::fence_before();
        __syncwarp();
        if (lane == 0) tc5::mbar_arrive_remote_cta(tempty_leader + 8 * b);
      }
      if (!ok) break;
      const int m = u.m0 + (int)rank * kHalfM + quad * 32;
      if (m < g.M) {
        const int64_t row0 = WGRAD ? (int64_t)u.expert * g.N + u.n0 : (int64_t)u.row;
        uint8_t* blk = reinterpret_cast<uint8_t*>(bars) + 256 + e * kOutBytes;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c0 = (cg + 4 * q) * 16;
          if (c0 < u.ncols)
            store_block<Out>(sum[q], blk, out + (row0 + c0) * g.ld + m, g.ld, u.ncols - c0,
                             g.M - m, g.vec, g.add, lane);
        }
      }
      u = next;
    }
  }

  tc5::fence_before();
  __syncthreads();
  tc5::cluster_sync();
  if (warp == 1) {
    tc5::fence_after();
    tc5::tmem_dealloc_pair(tmem, 512);
  }
}

stade_status operand_map(CUtensorMap* m, const ExpertOperand& o, bool bf16, uint32_t b0,
                         uint32_t b1) {
  const int64_t dims[3] = {o.d0, o.d1, o.d2}, pitch[2] = {o.pitch, o.pitch * o.d1};
  const uint32_t box[3] = {b0, b1, 1};
  return tc5::make_map_16(m, o.p, bf16, dims, pitch, box);
}

template <bool WGRAD, class Src, class Out>
stade_status launch(const ExpertOperand& A, const ExpertOperand& B, const Geom& g, const Src& src,
                    Out* out, int n_e, int64_t units, cudaStream_t s) {
  CUtensorMap am;
  BMaps bm;
  stade_status st = operand_map(&am, A, g.bf16, 64, g.a_mn ? 64 : 128);
  if (st == STADE_OK) st = operand_map(&bm.m[0], B, g.bf16, 64, g.b_mn ? 64 : 16);
  // taller boxes only where a tile can have the rows for them
  for (int i = 1; i < 4 && st == STADE_OK; ++i) {
    if (g.b_mn || B.d1 <= 16 << i) bm.m[i] = bm.m[i - 1];
    else st = operand_map(&bm.m[i], B, g.bf16, 64, 16 << i);
  }
  if (st != STADE_OK) return st;
  auto kern = expert_tc_kernel<WGRAD, Src, Out>;
  STADE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  const int pairs = (int)std::min<int64_t>(units, tc5::sm_count() / 2);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  STADE_CUDA(cudaLaunchKernelEx(&cfg, kern, am, bm, g, src, out, n_e));
  count_launch();
  return STADE_OK;
}

// ---- operand planes ------------------------------------------------------------------
// Eight columns a thread; VEC: source rows are multiples of 16 bytes.
template <class T, int NP, bool VEC>
__global__ void __launch_bounds__(256)
pack_kernel(const T* __restrict__ src, uint16_t* __restrict__ dst, int64_t rows, int64_t cols,
            int64_t pitch) {
  before_next();
  after_previous();
  const int64_t per = pitch / 8, n = rows * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = VEC ? 0 : i / per, c = VEC ? 0 : (i - r * per) * 8;
    alignas(16) T in[8];
    if constexpr (VEC) {       // rows follow each other without a gap
      constexpr int kPieces = 8 * (int)sizeof(T) / 16;
#pragma unroll
      for (int h = 0; h < kPieces; ++h)
        reinterpret_cast<int4*>(in)[h] = reinterpret_cast<const int4*>(src + i * 8)[h];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) in[j] = c + j < cols ? src[r * cols + c + j] : T(0.f);
    }
    const int64_t at = VEC ? i * 8 : r * pitch + c;
    if constexpr (NP == 1) {
      *reinterpret_cast<int4*>(dst + at) = *reinterpret_cast<const int4*>(in);
    } else {
      alignas(16) uint16_t o[NP][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float v = in[j];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          __nv_bfloat16 h = __float2bfloat16_rn(v);
          // a finite value just below 2^128 rounds to infinity: cut it instead
          if (p == 0 && __hisinf(h) && isfinite(v))
            h = __ushort_as_bfloat16((unsigned short)(__float_as_uint(v) >> 16));
          o[p][j] = __bfloat16_as_ushort(h);
          const float f = __bfloat162float(h);
          v = p > 0 || isfinite(f) ? v - f : 0.f;   // exact
        }
      }
#pragma unroll
      for (int p = 0; p < NP; ++p)
        *reinterpret_cast<int4*>(dst + p * rows * pitch + at) =
            *reinterpret_cast<const int4*>(o[p]);
    }
  }
}

}  // namespace

int64_t expert_planes(int dtype) { return dtype == STADE_F32 ? 3 : 1; }

stade_status expert_pack(int dtype, const void* src, void* dst, int64_t rows, int64_t cols,
                         int64_t pitch, cudaStream_t s) {
  const int64_t n = rows * (pitch / 8);
  if (n == 0) return STADE_OK;
  const unsigned blocks = (unsigned)std::min<int64_t>((n + 255) / 256, 148 * 32);
  uint16_t* d = (uint16_t*)dst;
  const bool vec = cols == pitch && row_align(16, {src}) == 16;
  if (dtype == STADE_F32)
    return launch_next(vec ? pack_kernel<float, 3, true> : pack_kernel<float, 3, false>, blocks,
                       256, 0, s, (const float*)src, d, rows, cols, pitch);
  // the two 16-bit types are moved, not computed with
  return launch_next(vec ? pack_kernel<__half, 1, true> : pack_kernel<__half, 1, false>, blocks,
                     256, 0, s, (const __half*)src, d, rows, cols, pitch);
}

stade_status expert_tc_rows(int dtype, const ExpertOperand& in, const ExpertOperand& w, void* out,
                            const ExpertTile* tiles, const int* count, int64_t max_tiles,
                            int64_t n_i, int64_t n_o, bool trans, bool add, cudaStream_t s) {
  Geom g = {};
  g.M = (int)(trans ? n_i : n_o);
  g.K = (int)(trans ? n_o : n_i);
  g.m_tiles = (g.M + 2 * kHalfM - 1) / (2 * kHalfM);
  g.n_tiles = 1;
  g.planes = (int)expert_planes(dtype);
  g.chain = dtype == STADE_F32 ? kChain : kChainRound;
  g.a_mn = !trans;
  g.b_mn = false;
  g.bf16 = dtype != STADE_F16;
  g.add = add;
  g.ld = g.M;
  g.vec = row_align(g.ld * dtype_size(dtype), {out}) == 16;
  const int n_e = (int)(w.d2 / g.planes);
  const RowSrc src{tiles, count};
  const int64_t units = max_tiles * g.m_tiles;
  if (dtype == STADE_F32) return launch<false>(w, in, g, src, (float*)out, n_e, units, s);
  if (dtype == STADE_BF16) return launch<false>(w, in, g, src, (__nv_bfloat16*)out, n_e, units, s);
  return launch<false>(w, in, g, src, (__half*)out, n_e, units, s);
}

stade_status expert_tc_wgrad(int dtype, const ExpertOperand& x, const ExpertOperand& yb, float* wb,
                             const int64_t* bounds, int64_t n_e, int64_t n_i, int64_t n_o, bool add,
                             cudaStream_t s) {
  Geom g = {};
  g.M = (int)n_o;
  g.N = (int)n_i;
  g.m_tiles = (g.M + 2 * kHalfM - 1) / (2 * kHalfM);
  g.n_tiles = (g.N + kTileN - 1) / kTileN;
  g.planes = (int)expert_planes(dtype);
  g.chain = dtype == STADE_F32 ? kChain : kChain16;
  g.a_mn = g.b_mn = true;
  g.bf16 = dtype != STADE_F16;
  g.add = add;
  g.ld = g.M;
  g.vec = row_align(g.ld * 4, {wb}) == 16;
  return launch<true>(yb, x, g, GroupSrc{bounds, (int)n_e}, wb, (int)n_e,
                      n_e * g.m_tiles * g.n_tiles, s);
}

int expert_tc_take_error() {
  int host = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&host, g_expert_tc_error, sizeof(int)) != cudaSuccess) return -1;
  if (host) cudaMemcpyToSymbol(g_expert_tc_error, &zero, sizeof(int));
  return host;
}

}  // namespace stade
