// Products of 8-bit whole numbers on tcgen05 (kind::i8), with a step for every row of A and every row of W:
//
//   C[m,n] = f(sum_k a[m,k] w[n,k]) * a_scales[m] * w_scales[n]
//
// The sums are 32-bit whole numbers and exact (K below 2^17 keeps them in range), f is their one rounding to f32, and C is rounded once from the
// f32 product.  So a result does not depend on tiles, on how K is split, or on the order of anything.
//
// Few output tiles: as gemm_skinny.cuh, with 128 of K where that has 64 (the same bytes).  Bound for a few rows: HBM, W is read once.  W fills the 128-row side of the
// tensor core and the rows of A its N side, NT = 16 .. 128 wide; K is split over a cluster of up to 8 CTAs where tiles are fewer than the SMs can
// take, and the partial sums are added through distributed shared memory.
#pragma once

#include <type_traits>

#include "gemm_skinny.cuh"
#include "ptx.cuh"

namespace tsm100 {
namespace gemm_i8 {

constexpr int kBN = 128;                 // rows of W (columns of C) per tile: the tensor core's M side
constexpr int kBK = 128;                 // 128 bytes: one swizzle row
constexpr int kThreads = 128;
constexpr int kMaxSplit = 8;
constexpr int kWBytes = kBN * kBK;       // 16 KiB of W per stage
constexpr int kMaxStages = 6;
constexpr int kAhead = 8;                // tiles of W that a CTA fetches into the L2 before the kernel before it has ended

template <int NT>
struct Shape {
  static constexpr int kXBytes = NT * kBK;  // rows of A per stage
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kStages = NT <= 16 ? 6 : NT <= 32 ? 5 : NT <= 64 ? 4 : 3;
  static constexpr int kTmemCols = NT < 32 ? 32 : NT;
};

struct alignas(8) Barriers {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t acc_full;
  uint32_t tmem_base;
  uint32_t abort_flag;
};

template <int NT>
constexpr int smem_bytes() {
  return Shape<NT>::kStages * Shape<NT>::kStageBytes + static_cast<int>(sizeof(Barriers)) + 1024;
}
// the partial tile of a split (NT rows x 128 columns, 32 bits) takes the place of the stages
static_assert(Shape<128>::kStages * Shape<128>::kStageBytes >= 128 * kBN * 4 && Shape<16>::kStages * Shape<16>::kStageBytes >= 16 * kBN * 4,
              "the partial tile fits the stages");
static_assert(2 * (smem_bytes<128>() + 1024) <= 227 * 1024 && 2 * (smem_bytes<16>() + 1024) <= 227 * 1024 &&
              2 * (smem_bytes<64>() + 1024) <= 227 * 1024 && 2 * (smem_bytes<32>() + 1024) <= 227 * 1024, "two CTAs per SM");

struct Params {
  const float* a_scales;    // [m]
  const float* w_scales;    // [n]
  int32_t m, n, k;
  int32_t m_blocks, n_blocks;
  int32_t kb_per_cta;       // blocks of 128 of K per CTA of the cluster (every CTA has at least one)
  int32_t vectors;          // rows of C start on 16-byte boundaries, N is a multiple of 4
  int64_t ldc;
  uint32_t* status;
};

__device__ __forceinline__ float scaled(uint32_t sum, float a_scale, float w_scale) { return __int2float_rn(static_cast<int32_t>(sum)) * a_scale * w_scale; }

// grid: (nb * m_blocks + mb) * cluster size + rank; CTAs that share a tile of W are neighbours.
template <typename OutT, int NT>
__global__ void __launch_bounds__(kThreads)
gemm_i8_few_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w, OutT* c, const Params p) {
  using S = Shape<NT>;
  using gemm_skinny::narrow;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Barriers* bars = reinterpret_cast<Barriers*>(smem + S::kStages * S::kStageBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile uint32_t* abort_flag = &bars->abort_flag;

  const uint32_t splits = ptx::cluster_nctarank(), rank = ptx::cluster_ctarank();
  const int t = static_cast<int>(blockIdx.x / splits);
  const int mb = t % p.m_blocks, nb = t / p.m_blocks;
  const int kb_all = (p.k + kBK - 1) / kBK;
  const int kb0 = static_cast<int>(rank) * p.kb_per_cta;
  const int num_kb = min(kb_all - kb0, p.kb_per_cta);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      ptx::mbar_init(&bars->full[s], 1);
      ptx::mbar_init(&bars->empty[s], 1);
    }
    ptx::mbar_init(&bars->acc_full, 1);
    bars->abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(&bars->tmem_base, S::kTmemCols);
    ptx::tmem_relinquish_alloc_permit();
  }
  ptx::tcgen05_fence_before_thread_sync();
  __syncthreads();
  ptx::tcgen05_fence_after_thread_sync();
  const uint32_t tmem_base = bars->tmem_base;
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tmap_a);
    ptx::prefetch_tensormap(&tmap_w);
    // while the kernel before this one runs: its first tiles of W
    for (int i = 0; i < min(num_kb, kAhead); ++i) ptx::prefetch_l2_3d(&tmap_w, (kb0 + i) * kBK, nb * kBN, 0);
  }
  ptx::wait_prior_grid();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < num_kb; ++i) {
        if (!ptx::mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, 181)) break;
        uint8_t* w = smem + stage * S::kStageBytes;
        const int k0 = (kb0 + i) * kBK;
        ptx::mbar_arrive_expect_tx(&bars->full[stage], S::kStageBytes);
        ptx::tma_load_3d(w, &tmap_w, &bars->full[stage], k0, nb * kBN, 0);
        ptx::tma_load_3d(w + kWBytes, &tmap_a, &bars->full[stage], k0, mb * NT, 0);
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = ptx::make_idesc_i8(kBN, NT);
      constexpr uint64_t kmajor = ptx::make_smem_desc_base(16, 1024);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < num_kb; ++i) {
        if (!(ok = ptx::mbar_wait_relaxed(&bars->full[stage], phase, abort_flag, p.status, 182))) break;
        ptx::tcgen05_fence_after_thread_sync();
        const uint32_t w = ptx::smem_u32(smem + stage * S::kStageBytes), x = w + kWBytes;
#pragma unroll
        for (int kk = 0; kk < kBK / 32; ++kk)
          ptx::tcgen05_mma_i8_ss(tmem_base, ptx::smem_desc(kmajor, w + kk * 32), ptx::smem_desc(kmajor, x + kk * 32), idesc, (i | kk) != 0 ? 1u : 0u);
        ptx::tcgen05_commit(&bars->empty[stage]);
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) ptx::tcgen05_commit(&bars->acc_full);
    }
  }
  __syncwarp();

  // ------------------------------ sums -> C ------------------------------
  // The scales, while the products run: lane i has those of rows i, 32 + i ... of A, and those of its own column, or four columns, of C.
  const int rows = min(NT, p.m - mb * NT);
  float as[(NT + 31) / 32], ws[4];
#pragma unroll
  for (int i = 0; i < (NT + 31) / 32; ++i) as[i] = i * 32 + lane < rows ? p.a_scales[mb * NT + i * 32 + lane] : 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = nb * kBN + (splits == 1 ? warp * 32 + lane : lane * 4 + j);
    ws[j] = col < p.n ? p.w_scales[col] : 0.f;
  }
  const bool ready = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->acc_full, 0, abort_flag, p.status, 183));
  ptx::tcgen05_fence_after_thread_sync();
  ptx::launch_dependents();  // not before: gemm_skinny.cuh
  const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
  constexpr int kStep = NT < 32 ? 16 : 32;  // rows of C (TMEM columns) per read
  auto read = [&](int r0, uint32_t (&v)[kStep]) {
    if constexpr (kStep == 16) ptx::tmem_ld_32x32b_x16(lane_addr + r0, v);
    else ptx::tmem_ld_32x32b_x32(lane_addr + r0, v);
    ptx::tmem_ld_wait();
  };
  if (splits == 1) {
    const int col = nb * kBN + warp * 32 + lane;
    if (ready) {
#pragma unroll
      for (int r0 = 0; r0 < NT; r0 += kStep) {
        if (r0 >= rows) break;
        uint32_t v[kStep];
        read(r0, v);
        OutT* dst = c + static_cast<int64_t>(mb * NT + r0) * p.ldc + col;
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
          const OutT x = narrow<OutT>(scaled(v[i], __shfl_sync(0xffffffffu, as[(r0 + i) / 32], (r0 + i) % 32), ws[0]));
          if (col < p.n && r0 + i < rows) dst[i * p.ldc] = x;
        }
      }
    }
  } else {
    // every CTA leaves its partial tile in its stages (all copies into them and products from them have retired) ...
    uint32_t* part = reinterpret_cast<uint32_t*>(smem);
    if (ready) {
#pragma unroll
      for (int r0 = 0; r0 < NT; r0 += kStep) {
        if (r0 >= rows) break;
        uint32_t v[kStep];
        read(r0, v);
#pragma unroll
        for (int i = 0; i < kStep; ++i) part[(r0 + i) * kBN + warp * 32 + lane] = v[i];
      }
    }
    ptx::cluster_sync_all();
    // ... and sums its share of the rows over all of them
    const uint32_t part_addr = ptx::smem_u32(part);
    const int items = rows * (kBN / 4);  // four columns each
    for (int i = static_cast<int>(rank) * kThreads + threadIdx.x; i < items; i += static_cast<int>(splits) * kThreads) {
      uint32_t s[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int q = 0; q < kMaxSplit; ++q)
        if (q < static_cast<int>(splits)) {
          const float4 v = ptx::ld_shared_cluster_f32x4(ptx::mapa_shared(part_addr + i * 16, q));
          s[0] += __float_as_uint(v.x), s[1] += __float_as_uint(v.y), s[2] += __float_as_uint(v.z), s[3] += __float_as_uint(v.w);
        }
      const int row = i / (kBN / 4), col = nb * kBN + lane * 4;  // kBN / 4 is a warp's lanes
      if (col >= p.n) continue;
      const float row_scale = p.a_scales[mb * NT + row];
      OutT* dst = c + static_cast<int64_t>(mb * NT + row) * p.ldc + col;
      OutT x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = narrow<OutT>(scaled(s[j], row_scale, ws[j]));
      if (p.vectors) {
        if constexpr (sizeof(OutT) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(x);
        else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(x);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + j < p.n) dst[j] = x[j];
      }
    }
    ptx::cluster_sync_all();  // nobody's partial tile goes while a peer reads it
  }

  // ------------------------------ teardown ------------------------------------
  if (*abort_flag != 0u) {
    // A wait gave up: give copies and products already in flight time to land before shared and tensor memory are released.
    const unsigned long long t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 1000000ull) {
    }
  }
  ptx::tcgen05_fence_before_thread_sync();
  __syncthreads();
  if (warp == 1) {
    ptx::tcgen05_fence_after_thread_sync();
    ptx::tmem_dealloc(tmem_base, S::kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// Many output tiles: CTA pairs (gemm_tc2.cuh), 256 rows of A by `bn` rows of W a tile
// ---------------------------------------------------------------------------
// Per CTA: warp 0 TMA producer (128 rows of A and half of the tile's rows of W, 128 of K a stage), warp 1 tensor memory and, in the leader, the products
// (M = 256 over the pair, N = bn, K = 32), warps 2..9 this CTA's 128 rows of the sums, of which two sets alternate, scaled and stored as boxes
// (by four warps 497 x 27968 x 192 took 17.6 us, by eight 14.0; K of thousands does not tell them apart).
// Bound: the tensor pipe, 2 M N K: 8192^3 325 us (3.38 POP/s), 8192 x 28672 x 4096 600 (3.2), single CTAs of 128 x 128 1027.  Below that operands from the L2, 64 KB for 128 of K to
// a pair, and what a tile takes to leave, 2.6 us, which the next tile's products do not hide: 4096^3 56 us (41 by the pipe).  Widths from 128 to 256 so that the last wave of tiles is a full one (route.hpp: gemm_i8).
namespace pairs {

constexpr int kPairM = 256, kCtaM = 128, kMaxBN = 256;
constexpr int kStages = 6;
constexpr int kThreads = 320;
constexpr int kABytes = kCtaM * kBK;              // 16 KiB
constexpr int kStageBytes = kABytes + kMaxBN / 2 * kBK;
constexpr int kTmemCols = 512;
constexpr int kGroupM = 16;                       // pair tiles per band (gemm_tc2.cuh)
constexpr int kBoxBytes = 32 * 128;

struct alignas(8) Barriers {
  uint64_t full[kStages];      // used in the leader: both CTAs' bytes of a stage have landed
  uint64_t empty[kStages];     // in each CTA: the products reading the stage have retired
  uint64_t acc_full[2];        // in each CTA: sums complete
  uint64_t acc_empty[2];       // used in the leader: 16 epilogue warps of the pair have drained them
  uint32_t tmem_base;
  uint32_t abort_flag;
};
constexpr int kBarsOff = kStages * kStageBytes + 8 * kBoxBytes;
constexpr int kSmemBytes = kBarsOff + sizeof(Barriers) + 1024;
static_assert(kSmemBytes <= 227 * 1024, "shared memory budget of one CTA");

struct Params {
  const float* a_scales;
  const float* w_scales;
  int32_t m, n, k;
  int32_t bn;                // a multiple of 32, and of a box's columns where C leaves in boxes
  int32_t m_blocks, n_blocks;
  int64_t ldc;
  uint32_t* status;
};

__device__ __forceinline__ void tile_coords(const Params& p, int tile, int& mb, int& nb) {
  const int band_tiles = kGroupM * p.n_blocks, band = tile / band_tiles, first_m = band * kGroupM;
  const int rows_in_band = min(kGroupM, p.m_blocks - first_m), t = tile - band * band_tiles;
  mb = first_m + t % rows_in_band;
  nb = t / rows_in_band;
}

// One warp's 32 rows of a tile's sums (`tmem`: its lanes, first column), scaled, to C from (row0, col0) up to column `end`: as gemm_tc.cuh's store_rows.
// kLoose: rows of C start anywhere.
template <typename OutT, bool kLoose>
__device__ __forceinline__ void store_rows(const CUtensorMap* tmap_c, OutT* c, const Params& p, uint32_t tmem, uint8_t* box, int row0, int col0, int end, int lane) {
  constexpr int kCols = gemm_tc::kBoxCols<OutT>, kHalves = kCols / 32;
  if (row0 >= p.m) return;
  const float as = p.a_scales[min(row0 + lane, p.m - 1)];
  const ptx::f32x2_t as2 = ptx::pack_f32x2(as, as);
  float ws[kHalves], next[kHalves];  // of this lane's columns in a box, asked for a box ahead
  auto ask = [&](int c0) {
#pragma unroll
    for (int h = 0; h < kHalves; ++h) next[h] = p.w_scales[min(c0 + h * 32 + lane, p.n - 1)];
  };
  ask(col0);
#pragma unroll 1
  for (int c0 = col0; c0 < end; c0 += kCols) {
    uint32_t v[kHalves][32];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) ptx::tmem_ld_32x32b_x32(tmem + (c0 - col0) + h * 32, v[h]);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) ws[h] = next[h];
    if (c0 + kCols < end) ask(c0 + kCols);
    ptx::tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int i = 0; i < 32; i += 2) {  // as `scaled`, two at once
        const ptx::f32x2_t x = ptx::pack_f32x2(__int2float_rn(static_cast<int32_t>(v[h][i])), __int2float_rn(static_cast<int32_t>(v[h][i + 1])));
        const ptx::f32x2_t w = ptx::pack_f32x2(__shfl_sync(0xffffffffu, ws[h], i), __shfl_sync(0xffffffffu, ws[h], i + 1));
        float lo, hi;
        ptx::unpack_f32x2(ptx::mul_f32x2(ptx::mul_f32x2(x, as2), w), lo, hi);
        v[h][i] = __float_as_uint(lo), v[h][i + 1] = __float_as_uint(hi);
      }
    if (!kLoose && lane == 0) ptx::tma_store_wait_read<0>();  // the store before has read the buffer
    __syncwarp();
    const uint32_t row = ptx::smem_u32(box) + lane * 128;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t at = row + ((u ^ (lane & 7)) << 4);
      if constexpr (sizeof(OutT) == 4) {
        ptx::st_shared_v4(at, v[0][4 * u], v[0][4 * u + 1], v[0][4 * u + 2], v[0][4 * u + 3]);
      } else {
        using gemm_tc::narrow2;
        const uint32_t(&w)[32] = v[u >> 2];
        const int i = (u & 3) * 8;
        ptx::st_shared_v4(at, narrow2<OutT>(w[i], w[i + 1]), narrow2<OutT>(w[i + 2], w[i + 3]), narrow2<OutT>(w[i + 4], w[i + 5]), narrow2<OutT>(w[i + 6], w[i + 7]));
      }
    }
    if constexpr (kLoose) {
      __syncwarp();
      const int rows = min(32, p.m - row0);
      OutT* dst = c + row0 * p.ldc + c0;
#pragma unroll 4
      for (int r = 0; r < rows; ++r, dst += p.ldc)
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const int x = h * 32 + lane;
          const OutT value = *reinterpret_cast<const OutT*>(box + r * 128 + (((x * static_cast<int>(sizeof(OutT)) >> 4) ^ (r & 7)) << 4) + (x * static_cast<int>(sizeof(OutT)) & 15));
          if (c0 + x < end) dst[x] = value;
        }
      continue;
    }
    ptx::fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      ptx::tma_store_3d(tmap_c, box, c0, row0, 0);
      ptx::tma_store_commit();
    }
  }
}

template <typename OutT, bool kLoose>
__global__ void __launch_bounds__(kThreads, 1)
gemm_i8_pairs_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_c, OutT* c,
                     const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Barriers* bars = reinterpret_cast<Barriers*>(smem + kBarsOff);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();  // 0 = leader
  const int pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
  const int num_tiles = p.m_blocks * p.n_blocks;
  const int num_kb = (p.k + kBK - 1) / kBK;
  volatile uint32_t* abort_flag = &bars->abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(&bars->full[s], 1);
      ptx::mbar_init(&bars->empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(&bars->acc_full[a], 1);
      ptx::mbar_init(&bars->acc_empty[a], 16);
    }
    bars->abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc_pair(&bars->tmem_base, kTmemCols);
    ptx::tmem_relinquish_alloc_permit_pair();
  }
  ptx::tcgen05_fence_before_thread_sync();
  ptx::cluster_sync_all();  // the peer's barriers are initialised before anything signals them
  ptx::tcgen05_fence_after_thread_sync();
  const uint32_t tmem_base = bars->tmem_base;
  ptx::launch_dependents();
  ptx::wait_prior_grid();

  if (warp == 0) {
    // ------------------------------ TMA producer (both CTAs) ------------------
    if (lane == 0) {
      ptx::prefetch_tensormap(&tmap_a);
      ptx::prefetch_tensormap(&tmap_w);
      const uint32_t bytes = 2 * (kABytes + p.bn / 2 * kBK);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = pair; tile < num_tiles && ok; tile += num_pairs) {
        int mb, nb;
        tile_coords(p, tile, mb, nb);
        const int row0 = mb * kPairM + static_cast<int>(rank) * kCtaM, col0 = nb * p.bn + static_cast<int>(rank) * (p.bn / 2);
        const bool backward = ((tile / num_pairs) & 1) != 0;  // every other wave walks K backwards, to find in the L2 what the one before it read last
        for (int kq = 0; kq < num_kb; ++kq) {
          const int k0 = (backward ? num_kb - 1 - kq : kq) * kBK;
          if (!ptx::mbar_wait(&bars->empty[stage], phase ^ 1u, abort_flag, p.status, 184)) {
            ok = false;
            break;
          }
          const uint32_t full_leader = ptx::mapa_shared(ptx::smem_u32(&bars->full[stage]), 0);
          if (rank == 0) ptx::mbar_arrive_expect_tx(&bars->full[stage], bytes);
          uint8_t* to = smem + stage * kStageBytes;
          ptx::tma_load_3d_pair(to, &tmap_a, full_leader, k0, row0, 0);
          ptx::tma_load_3d_pair(to + kABytes, &tmap_w, full_leader, k0, col0, 0);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------ products (leader CTA only) ----------------
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = ptx::make_idesc_i8(kPairM, p.bn);
      constexpr uint64_t kmajor = ptx::make_smem_desc_base(16, 1024);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int local = 0;
      for (int tile = pair; tile < num_tiles && ok; tile += num_pairs, ++local) {
        const int acc = local & 1;
        if (!ptx::mbar_wait(&bars->acc_empty[acc], ((local >> 1) & 1u) ^ 1u, abort_flag, p.status, 185)) break;
        ptx::tcgen05_fence_after_thread_sync();
        const uint32_t d_tmem = tmem_base + acc * kMaxBN;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!ptx::mbar_wait_relaxed(&bars->full[stage], phase, abort_flag, p.status, 186)) {  // relaxed: the data goes straight to the async proxy
            ok = false;
            break;
          }
          ptx::tcgen05_fence_after_thread_sync();
          const uint32_t a = ptx::smem_u32(smem + stage * kStageBytes), w = a + kABytes;
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            ptx::tcgen05_mma_i8_ss_pair(d_tmem, ptx::smem_desc(kmajor, a + kk * 32), ptx::smem_desc(kmajor, w + kk * 32), idesc, (kb | kk) != 0 ? 1u : 0u);
          ptx::tcgen05_commit_pair(&bars->empty[stage], 3);  // frees the stage in both CTAs
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) ptx::tcgen05_commit_pair(&bars->acc_full[acc], 3);
      }
    }
  } else {
    // ------------------------------ sums -> C (both CTAs) ---------------------
    const int quad = warp & 3, side = (warp - 2) >> 2;  // two warps share rows: one the left half of the columns, in whole boxes, one the right
    const int left = (p.bn / 2 + gemm_tc::kBoxCols<OutT> - 1) / gemm_tc::kBoxCols<OutT> * gemm_tc::kBoxCols<OutT>;
    uint8_t* staging = smem + kStages * kStageBytes + (warp - 2) * kBoxBytes;
    int local = 0;
    for (int tile = pair; tile < num_tiles; tile += num_pairs, ++local) {
      const int acc = local & 1;
      int mb, nb;
      tile_coords(p, tile, mb, nb);
      const bool ready = ptx::mbar_wait(&bars->acc_full[acc], (local >> 1) & 1u, abort_flag, p.status, 187);
      if (!__all_sync(0xffffffffu, ready)) break;
      ptx::tcgen05_fence_after_thread_sync();
      const uint32_t from = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * kMaxBN + side * left;
      const int row0 = mb * kPairM + static_cast<int>(rank) * kCtaM + quad * 32, col0 = nb * p.bn + side * left;
      store_rows<OutT, kLoose>(&tmap_c, c, p, from, staging, row0, col0, min(p.n, nb * p.bn + (side ? p.bn : left)), lane);
      ptx::tcgen05_fence_before_thread_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(ptx::smem_u32(&bars->acc_empty[acc]), 0));
    }
    if (!kLoose && lane == 0) ptx::tma_store_wait_all<0>();
  }

  // ------------------------------ teardown ------------------------------------
  if (*abort_flag != 0u) {
    const unsigned long long t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 1000000ull) {
    }
  }
  ptx::tcgen05_fence_before_thread_sync();
  // Neither CTA may leave while the other can still read its shared memory or signal its barriers.
  ptx::cluster_sync_all();
  if (warp == 1) {
    ptx::tcgen05_fence_after_thread_sync();
    ptx::tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

}  // namespace pairs

// Operands whose rows do not start on 16-byte boundaries, as rows that do: src [rows][cols], pitch ld -> dst [rows][pitch], zeros beyond cols.
// A thread has 16 bytes of dst; words of src that hold them, shifted into place, a byte at a time where those reach past the matrix.
struct Operand {
  const uint8_t* src;
  uint4* dst;
  int64_t ld;
  int32_t rows, cols, pitch;
  int32_t blocks;   // of the launch that work on it, 0: it is not copied
};
constexpr int kPadThreads = 256;
__device__ __forceinline__ uint4 load16(const uint8_t* src, int64_t at, int64_t size, int valid) {
  const uintptr_t address = reinterpret_cast<uintptr_t>(src + at), from = address & ~uintptr_t(3);
  const uint32_t bits = static_cast<uint32_t>(address & 3) * 8;
  uint32_t w[5];
  if (valid >= 16 && from >= reinterpret_cast<uintptr_t>(src) && from + 20 <= reinterpret_cast<uintptr_t>(src + size)) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = reinterpret_cast<const uint32_t*>(from)[i];
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = 0u;
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (j < valid) w[j >> 2] |= static_cast<uint32_t>(src[at + j]) << ((j & 3) * 8);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__global__ void __launch_bounds__(kPadThreads) gemm_i8_pad_kernel(const Operand a, const Operand b) {
  ptx::launch_dependents_if_few();
  ptx::wait_prior_grid();
  const bool first = static_cast<int32_t>(blockIdx.x) < a.blocks;
  const Operand& p = first ? a : b;
  const int32_t block = first ? blockIdx.x : blockIdx.x - a.blocks;
  const uint32_t per_row = static_cast<uint32_t>(p.pitch) / 16;
  const int64_t total = static_cast<int64_t>(p.rows) * per_row, step = static_cast<int64_t>(p.blocks) * kPadThreads;
  const int64_t size = static_cast<int64_t>(p.rows - 1) * p.ld + p.cols;
#pragma unroll 2
  for (int64_t i = static_cast<int64_t>(block) * kPadThreads + threadIdx.x; i < total; i += step) {
    const int64_t r = total <= 0xffffffffll ? static_cast<int64_t>(static_cast<uint32_t>(i) / per_row) : i / per_row;
    const int32_t c = static_cast<int32_t>(i - r * per_row) * 16;
    p.dst[i] = load16(p.src, r * p.ld + c, size, p.cols - c);
  }
}

}  // namespace gemm_i8
}  // namespace tsm100
