// Products with 4-bit weights: C[m,n] = a_scale[m] * sum_g scale[n,g] * sum_{k in g} A[m,k] * (q[n,k] - zero[n,g]).
//
// W is [N][K/2] bytes, the even k in the low half.  The inner sums are tcgen05 products of numbers that 16 bits hold exactly, with f32 sums: 128 rows
// of W on the M side, up to 256 rows of A on the N side.  A group's sum comes back from tensor memory, is multiplied by its scale and added in
// f32, so C is rounded once and nothing else.
//
// Bound: with few rows of A reading the weights, 46 of them a clock and SM.  Weights in shared memory would write and read 184 bytes a clock there for the tensor core, more
// than it gives; mma.sync tiles with the weights in registers took 31 us for 16 x 16384 x 4096.  So a thread, which has a row of W, brings 64 k of it from the
// TMA's tile into registers, makes numbers of them with eleven instructions for eight (three shifts, four masks that also set the exponent of 128 + q or 1024 + q, four
// subtractions) and stores them to tensor memory, from where the product takes them.  What bounds it as it is: instructions, 200 a warp for 64 k of its 32
// rows where 88 make the numbers.  With many rows of A the tensor core would be the bound, and the chain of steps of a chunk is.
//
// A CTA has 128 rows of W, up to 256 of A and a range of K, 128 k at a time: eight warps make the weights (four of them the first 64 k, four the others) and bring A's part to
// shared memory in the order in which masks find the weights (of eight k 0 4 1 5 2 6 3 7, K-major, 128-byte swizzle); a warp fetches W by TMA, a warp issues the products.
// Operands have three places and sums two, and a chunk is handed over while the next is made, so that neither stores to tensor memory nor products are waited for.
// K may be split over a cluster; partial sums are added through distributed shared memory in rank order.
//
// More than 64 rows of A (kScaled): a weight is multiplied by its scale and rounded to 16 bits, as a weight of a 16-bit product would have been, and the sums stay
// in tensor memory over all of K: bringing a group's 128 sums a row back cost as much as its products.  A comes in 16 bits (rows in 8 are made such first, w4_dense.cuh),
// by TMA, as it is: the weights' pairs are exchanged instead, four instructions for eight (200 x 5003 x 2048 21.5 us with A through registers, 15.4 this way).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "ptx.cuh"
#include "softmax.cuh"

namespace tsm100 {
namespace w4 {

constexpr int kRows = 128;                 // of W
constexpr int kWorkers = 256, kThreads = kWorkers + 64;  // warp 8: TMA, warp 9: products
constexpr int kChunkK = 128, kStepK = 256;  // a TMA box brings two chunks
constexpr int kSlotBytes = kRows * kStepK / 2;
constexpr int kBuffers = 3;                // of operands
constexpr int kExactTokens = 64;           // rows of A up to which scales are applied to sums

struct Params {
  const void* a;
  const float* a_scales;   // rows in 8 bits, else null
  const void* scales;
  const uint8_t* zeros;    // or null: 8
  void* c;
  int32_t m, n, k, groups;
  int32_t splits;          // CTAs of a cluster along K
  int32_t tokens;          // rows of A a CTA has: a multiple of 16, at most N
  uint32_t* status;
};
struct alignas(8) Barriers {
  uint64_t full[8], empty[8];  // W's slots
  uint64_t ready[2], done[2];  // a chunk's operands are there; its products are
  uint64_t a_full[kBuffers], a_empty[kBuffers];  // kScaled: the places of A's chunks
  uint32_t tmem_base;
  uint32_t abort_flag;
};

// Up to N rows of A; GC groups in a chunk
template <int N, int GC, bool kScaled>
struct Shape {
  static constexpr int kSumsOff = kBuffers * 64;         // columns of tensor memory: weights, then sums
  static constexpr int kTmemUsed = kSumsOff + (kScaled ? N : 2 * GC * N);
  static constexpr int kTmem = kTmemUsed <= 256 ? 256 : 512;
  static constexpr bool kTwo = kTmem == 256 && N <= 32;  // CTAs to an SM
  static constexpr int kSlots = kTwo ? 5 : 6;
  static constexpr int kPlaces = N == 256 ? 2 : kBuffers;  // of A's chunks: what fits
  static constexpr int kActBytes = N * kChunkK * 2;
  static constexpr int kActOff = kSlots * kSlotBytes, kBarsOff = kActOff + kPlaces * kActBytes;
  static constexpr int kSmem = kBarsOff + static_cast<int>(sizeof(Barriers)) + 1024;
  static constexpr int kVecs = kScaled ? 1 : N * kChunkK / 8 / kWorkers;  // eights of A's numbers a worker brings for a chunk
  static_assert(kTmemUsed <= 512 && kSmem <= (kTwo ? 113 : 227) * 1024 && kVecs >= 1, "what an SM has");
  static_assert(N * kRows * 4 <= kBarsOff && kPlaces <= kBuffers, "partial sums lie over the slots");
};

template <bool kBf16>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  if (kBf16) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// 128 + q (bf16) or 1024 + q (f16): exact, and so is taking 128 + zero from it
template <bool kBf16>
constexpr uint32_t kMagic = kBf16 ? 0x43004300u : 0x64006400u;

// Weights k, k + 4 for k = 0 .. 3 of eight, less their zero point.
template <bool kBf16>
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t zero, uint32_t* out) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t h;  // (w >> 4 i & 0x000f000f) | magic in one instruction: left alone, the compiler took two
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(h) : "r"(w >> (4 * i)), "r"(0x000f000fu), "r"(kMagic<kBf16>));
    out[i] = sub2<kBf16>(h, zero);
  }
}

template <bool kBf16>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  if (kBf16) {
    const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Bytes `j` of lo and of hi, whole numbers, as a pair of 16-bit numbers: a byte behind 0x64 is 1024 + byte as f16, behind 0x4b0000 2^23 + byte as f32.
template <typename T>
__device__ __forceinline__ uint32_t i8_to_16(uint32_t lo, uint32_t hi, int j) {
  const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
  if (std::is_same<T, __half>::value) {
    return sub2<false>((__byte_perm(a, b, 0x400 + j * 0x101) & 0x00ff00ffu) | 0x64006400u, 0x64806480u);
  }
  const float x = __uint_as_float(__byte_perm(a, 0x4b000000u, 0x7540 + j)) - 8388736.f, y = __uint_as_float(__byte_perm(b, 0x4b000000u, 0x7540 + j)) - 8388736.f;
  return ptx::pack_bf16x2(x, y);
}

// A whole warp's bounded wait: one vote where the barrier's phase has passed already.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* status, uint32_t site) {
  if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity, abort_flag, status, site));
}

template <int X>
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[X]) {
  if constexpr (X == 32) ptx::tmem_ld_32x32b_x32(at, r);
  else if constexpr (X == 16) ptx::tmem_ld_32x32b_x16(at, r);
  else
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(at) : "memory");
}

template <typename T, int N, int GC, bool kScaled, bool kEight>
__global__ void __launch_bounds__(kThreads, Shape<N, GC, kScaled>::kTwo ? 2 : 1)
gemm_w4_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a, const Params p) {
  static_assert(!kScaled || !kEight, "more than 64 rows come in 16 bits");
  using S = Shape<N, GC, kScaled>;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Barriers* bars = reinterpret_cast<Barriers*>(smem + S::kBarsOff);
  volatile uint32_t* abort_flag = &bars->abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = static_cast<int>(blockIdx.x) % p.splits, row_base = static_cast<int>(blockIdx.x) / p.splits * kRows;
  const int token0 = static_cast<int>(blockIdx.y) * p.tokens;
  const int steps = (p.k + kStepK - 1) / kStepK;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * rank / p.splits), s1 = static_cast<int>(static_cast<int64_t>(steps) * (rank + 1) / p.splits);
  const int first = 2 * s0, chunks = min(2 * s1, (p.k + kChunkK - 1) / kChunkK) - first;
  if (tid == 0) {
    for (int i = 0; i < S::kSlots; ++i) ptx::mbar_init(&bars->full[i], 1), ptx::mbar_init(&bars->empty[i], kWorkers);
    for (int i = 0; i < 2; ++i) ptx::mbar_init(&bars->ready[i], kWorkers), ptx::mbar_init(&bars->done[i], 1);
    if constexpr (kScaled)
      for (int i = 0; i < S::kPlaces; ++i) ptx::mbar_init(&bars->a_full[i], 1), ptx::mbar_init(&bars->a_empty[i], 1);
    bars->abort_flag = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 8 && lane == 0) {
    ptx::prefetch_tensormap(&tmap_w);
    for (int i = 0; i < S::kSlots && s0 + i < s1; ++i) ptx::prefetch_l2_3d(&tmap_w, (s0 + i) * (kStepK / 2), row_base, 0);
  }
  if (warp == 9) {
    ptx::tmem_alloc(&bars->tmem_base, S::kTmem);
    ptx::tmem_relinquish_alloc_permit();
  }
  ptx::tcgen05_fence_before_thread_sync();
  __syncthreads();
  ptx::tcgen05_fence_after_thread_sync();
  const uint32_t tmem = bars->tmem_base, sums_at = tmem + S::kSumsOff;
  ptx::wait_prior_grid();

  constexpr int NH = N / 2;  // a worker's share of a row of sums
  constexpr int X = NH > 32 ? 32 : NH;
  float acc[NH];
#pragma unroll
  for (int i = 0; i < NH; ++i) acc[i] = 0.f;
  const int wg = warp >> 2, row = (warp & 3) * 32 + lane;
  if (warp == 8) {
    if (lane == 0) {
      auto fetch_w = [&](int s) {
        const int i = s - s0, slot = i % S::kSlots;
        if (!ptx::mbar_wait(&bars->empty[slot], ((i / S::kSlots) & 1u) ^ 1u, abort_flag, p.status, 135)) return false;
        ptx::mbar_arrive_expect_tx(&bars->full[slot], kSlotBytes);
        ptx::tma_load_3d(smem + slot * kSlotBytes, &tmap_w, &bars->full[slot], s * (kStepK / 2), row_base, 0);
        return true;
      };
      if constexpr (kScaled) {
        // W keeps kAheadW steps before A: a step's place is free when the products that A's next chunk waits for are about to be
        constexpr int kAheadW = S::kSlots - 2;
        bool more = true;
        for (int s = s0; more && s < min(s0 + kAheadW, s1); ++s) more = fetch_w(s);
        for (int i = 0; more && i < chunks; ++i) {
          if (i % 2 == 0 && s0 + i / 2 + kAheadW < s1) more = fetch_w(s0 + i / 2 + kAheadW);
          const int b = i % S::kPlaces;
          if (!more || !ptx::mbar_wait(&bars->a_empty[b], ((i / S::kPlaces) & 1u) ^ 1u, abort_flag, p.status, 139)) break;
          ptx::mbar_arrive_expect_tx(&bars->a_full[b], static_cast<uint32_t>(p.tokens) * kChunkK * 2);
#pragma unroll
          for (int h = 0; h < kChunkK / 64; ++h)
            ptx::tma_load_3d(smem + S::kActOff + b * S::kActBytes + h * (N * 128), &tmap_a, &bars->a_full[b], (first + i) * kChunkK + h * 64, token0, 0);
        }
      } else {
        for (int s = s0; s < s1; ++s)
          if (!fetch_w(s)) break;
      }
    }
  } else if (warp == 9) {
    const uint32_t idesc = ptx::make_idesc_f16(kRows, static_cast<uint32_t>(p.tokens), false, false, kBf16);
    constexpr uint64_t kmajor = ptx::make_smem_desc_base(16, 1024);
    int b = 0, place = 0;
    uint32_t place_phase = 0;
    for (int i = 0; i < chunks; ++i) {
      const int d = i & 1;
      if (!warp_wait(&bars->ready[d], (i >> 1) & 1u, abort_flag, p.status, 136)) break;
      if (kScaled && !warp_wait(&bars->a_full[place], place_phase, abort_flag, p.status, 140)) break;
      ptx::tcgen05_fence_after_thread_sync();
      if (ptx::elect_one_sync()) {
        const uint32_t act = ptx::smem_u32(smem + S::kActOff + place * S::kActBytes);
#pragma unroll
        for (int kk = 0; kk < kChunkK / 16; ++kk) {
          // nothing behind K: A is zero there, but a weight as far from its zero point as 15, times the last group's scale, may be infinite in 16 bits
          if (kScaled && GC > 1 && (first + i) * kChunkK + kk * 16 >= p.k) break;
          constexpr int kPer = kChunkK / 16 / GC;  // of a group
          ptx::tcgen05_mma_f16_ts(kScaled ? sums_at : sums_at + (d * GC + kk / kPer) * N, tmem + b * 64 + kk * 8,
                                  ptx::smem_desc(kmajor, act + (kk >> 2) * (N * 128) + (kk & 3) * 32), idesc, (kScaled ? i + kk : kk % kPer) != 0 ? 1u : 0u);
        }
        ptx::tcgen05_commit(&bars->done[d]);
        if (kScaled && i + S::kPlaces < chunks) ptx::tcgen05_commit(&bars->a_empty[place]);  // only where it is waited for: none outlives the CTA
      }
      __syncwarp();
      b = b + 1 == kBuffers ? 0 : b + 1;
      if (++place == S::kPlaces) place = 0, place_phase ^= 1u;
    }
  } else {
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    // A chunk's scales and zero points, and its part of A, are fetched two chunks ahead, into the registers that the chunk before has left.
    constexpr int kAhead = 2;
    const int64_t row_groups = static_cast<int64_t>(min(row_base + row, p.n - 1)) * p.groups + first * GC;
    const uint16_t* scale_at = static_cast<const uint16_t*>(p.scales) + row_groups;
    const uint8_t* zero_at = p.zeros ? p.zeros + row_groups : nullptr;
    const int groups_left = min(p.groups - first * GC, chunks * GC);
    // a chunk's groups in one load where they never start inside one
    const bool together = GC > 1 && p.groups % GC == 0 && reinterpret_cast<uintptr_t>(p.scales) % (2 * GC) == 0 && reinterpret_cast<uintptr_t>(p.zeros) % GC == 0;
    uint16_t sc[2][GC];
    uint32_t zp[2];  // a byte a group
    const int last_group = max(groups_left - 1, 0), last_chunk = max((groups_left - 1) / GC, 0);
    // Behind the last group it is fetched again: no product or one with zeros follows, and rows behind N are not stored.
    auto fetch_row = [&](int i, uint16_t (&to)[GC], uint32_t& zero) {
      if (GC > 1 && together) {
        const int at = min(i, last_chunk) * GC;
        if constexpr (GC == 4) {
          const uint2 x = *reinterpret_cast<const uint2*>(scale_at + at);
          to[0] = static_cast<uint16_t>(x.x), to[GC - 3] = static_cast<uint16_t>(x.x >> 16);
          to[GC - 2] = static_cast<uint16_t>(x.y), to[GC - 1] = static_cast<uint16_t>(x.y >> 16);
          if (zero_at) zero = *reinterpret_cast<const uint32_t*>(zero_at + at);
        } else {
          const uint32_t x = *reinterpret_cast<const uint32_t*>(scale_at + at);
          to[0] = static_cast<uint16_t>(x), to[GC - 1] = static_cast<uint16_t>(x >> 16);
          if (zero_at) zero = *reinterpret_cast<const uint16_t*>(zero_at + at);
        }
      } else {
#pragma unroll
        for (int j = 0; j < GC; ++j) to[j] = scale_at[min(i * GC + j, last_group)];
        if (zero_at) {
          zero = 0;
#pragma unroll
          for (int j = 0; j < GC; ++j) zero |= static_cast<uint32_t>(zero_at[min(i * GC + j, last_group)]) << (8 * j);
        }
      }
    };
    using Vec = typename std::conditional<kEight, uint2, uint4>::type;  // eight numbers of A
    const int e8 = tid % 16 * 8, rows_left = min(p.m - token0, p.tokens) - tid / 16;
    const int64_t act_row = static_cast<int64_t>(token0 + tid / 16) * p.k + first * kChunkK + e8;
    const Vec* act_at = reinterpret_cast<const Vec*>(static_cast<const uint8_t*>(p.a) + act_row * (kEight ? 1 : 2));
    const int64_t act_pitch = static_cast<int64_t>(p.k) * 2;  // vectors of sixteen rows
    // chunks in which this thread has something to fetch
    const int act_chunks = rows_left > 0 ? min(chunks, (p.k - first * kChunkK - e8 + kChunkK - 1) / kChunkK) : 0;
    Vec act[kAhead][S::kVecs];
    auto fetch_act = [&](int i, Vec (&to)[S::kVecs]) {
      if constexpr (kScaled) return;
#pragma unroll
      for (int v = 0; v < S::kVecs; ++v) {
        to[v] = Vec{};
        if (i < act_chunks && (v == 0 || v * 16 < rows_left)) to[v] = act_at[i * (kChunkK / 8) + v * act_pitch];
      }
    };
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      zp[b] = 0x08080808u;
      fetch_row(b, sc[b], zp[b]);
      fetch_act(b, act[b]);
    }
    uint16_t sc_of[2][GC];  // of the two chunks whose sums are still out
    bool ok = true;
    auto wait_done = [&](int i) {
      ok = warp_wait(&bars->done[i & 1], (i >> 1) & 1u, abort_flag, p.status, 137);
      ptx::tcgen05_fence_after_thread_sync();
    };
    auto collect = [&](int i, auto which) {  // chunk i's products are done; its sums, times their scales
      [[maybe_unused]] constexpr int d = decltype(which)::value;
      wait_done(i);
      if constexpr (!kScaled) {
        if (!ok) return;
        if constexpr (GC * NH <= 32) {
          uint32_t got[GC][NH];
#pragma unroll
          for (int j = 0; j < GC; ++j) tmem_ld<NH>(sums_at + (d * GC + j) * N + wg * NH + lanes, got[j]);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < GC; ++j) {
            const float f = softmax::Elem<T>::load1(reinterpret_cast<const T*>(&sc_of[d][j]));
#pragma unroll
            for (int e = 0; e < NH; ++e) acc[e] = fmaf(__uint_as_float(got[j][e]), f, acc[e]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < GC; ++j) {
            const float f = softmax::Elem<T>::load1(reinterpret_cast<const T*>(&sc_of[d][j]));
            uint32_t got[X];
            tmem_ld<X>(sums_at + (d * GC + j) * N + wg * NH + lanes, got);
            ptx::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < X; ++e) acc[e] = fmaf(__uint_as_float(got[e]), f, acc[e]);
          }
        }
        ptx::tcgen05_fence_before_thread_sync();
      }
    };
    auto hand_over = [&](int i) {  // chunk i's operands to the tensor core
      ptx::tmem_st_wait();
      ptx::tcgen05_fence_before_thread_sync();
      if constexpr (!kScaled) ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(&bars->ready[i & 1]);
    };
    const uint32_t w_at = ptx::smem_u32(smem) + row * 128;
    uint32_t w_off[2][2];  // the row's 16 bytes of a slot: (chunk, half of its 64 k)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) w_off[c][h] = w_at + (((c * 4 + wg * 2 + h) ^ (row & 7)) << 4);
    uint8_t* act_to = smem + S::kActOff + (tid % 16 >> 3) * (N * 128) + tid / 16 * 128 + (((tid & 7) ^ (tid / 16 & 7)) << 4);
    int slot = 0, b = 0;
    uint32_t full_phase = 0;
    auto chunk = [&](int i, auto which) {
      constexpr int d = decltype(which)::value;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // 32 k of this row, as numbers
        uint32_t x[4], w[16];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(w_off[d][h] + slot * kSlotBytes));
        constexpr int kHalf = GC / 2;  // groups of 64 k
        const int g = GC == 1 ? 0 : (wg ? kHalf : 0) + (GC == 4 ? h : 0);
        const uint32_t zero = (GC == 1 ? zp[d] & 0xffu : zp[d] >> (8 * g) & 0xffu) * 0x10001u + kMagic<kBf16>;
#pragma unroll
        for (int j = 0; j < 4; ++j) unpack8<kBf16>(x[j], zero, w + j * 4);
        if constexpr (kScaled) {
          uint32_t f = sc[d][0];
          if (GC > 1 && g == 1) f = sc[d][GC > 1 ? 1 : 0];
          if (GC > 2 && g == 2) f = sc[d][GC > 2 ? 2 : 0];
          if (GC > 2 && g == 3) f = sc[d][GC > 2 ? 3 : 0];
          f *= 0x10001u;
#pragma unroll
          for (int j = 0; j < 16; ++j) w[j] = mul2<kBf16>(w[j], f);
#pragma unroll
          for (int j = 0; j < 16; j += 4) {  // as A is: 0 1, 2 3, 4 5, 6 7
            const uint32_t y[4] = {w[j], w[j + 1], w[j + 2], w[j + 3]};
            w[j] = __byte_perm(y[0], y[1], 0x5410), w[j + 1] = __byte_perm(y[2], y[3], 0x5410);
            w[j + 2] = __byte_perm(y[0], y[1], 0x7632), w[j + 3] = __byte_perm(y[2], y[3], 0x7632);
          }
        }
        if (h == 0 && i > 0) hand_over(i - 1);  // its stores have had this time to end
        ptx::tmem_st_32x32b_x16(tmem + b * 64 + wg * 32 + h * 16 + lanes, w);
      }
      if (d == 1 || i == chunks - 1) ptx::mbar_arrive(&bars->empty[slot]);
#pragma unroll
      for (int v = 0; v < (kScaled ? 0 : S::kVecs); ++v) {
        const Vec x = act[d][v];
        uint4 y;
        if constexpr (kEight) y = make_uint4(i8_to_16<T>(x.x, x.y, 0), i8_to_16<T>(x.x, x.y, 1), i8_to_16<T>(x.x, x.y, 2), i8_to_16<T>(x.x, x.y, 3));
        else y = make_uint4(__byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
        *reinterpret_cast<uint4*>(act_to + b * S::kActBytes + v * 2048) = y;
      }
      fetch_act(i + kAhead, act[d]);
      if (i >= 2) collect(i - 2, which);  // frees its sums for this chunk, and its operands for the next
#pragma unroll
      for (int j = 0; j < GC; ++j) sc_of[d][j] = sc[d][j];
      fetch_row(i + 2, sc[d], zp[d]);
      b = b + 1 == kBuffers ? 0 : b + 1;
    };
    for (int i = 0; i < chunks && ok; i += 2) {
      ok = warp_wait(&bars->full[slot], full_phase, abort_flag, p.status, 138);
      if (!ok) break;
      chunk(i, std::integral_constant<int, 0>{});
      if (ok && i + 1 < chunks) chunk(i + 1, std::integral_constant<int, 1>{});
      if (++slot == S::kSlots) slot = 0, full_phase ^= 1u;
    }
    if (ok && chunks > 0) hand_over(chunks - 1);
    // the last two, whichever places they have
    if (ok && chunks >= 2) {
      if (chunks & 1) collect(chunks - 2, std::integral_constant<int, 1>{});
      else collect(chunks - 2, std::integral_constant<int, 0>{});
    }
    if (ok && chunks >= 1) {
      if (chunks & 1) collect(chunks - 1, std::integral_constant<int, 0>{});
      else collect(chunks - 1, std::integral_constant<int, 1>{});
    }
    if constexpr (kScaled) {
      if (ok)
#pragma unroll
        for (int c = 0; c < NH; c += X) {
          uint32_t got[X];
          tmem_ld<X>(sums_at + wg * NH + c + lanes, got);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < X; ++e) acc[c + e] = __uint_as_float(got[e]);
        }
    }
  }
  ptx::launch_dependents();
  if (*abort_flag != 0u) {
    // a wait gave up: copies and products in flight end first
    const unsigned long long since = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - since < 1000000ull) {
    }
  }
  ptx::tcgen05_fence_before_thread_sync();
  __syncthreads();
  if (warp == 9) {
    ptx::tcgen05_fence_after_thread_sync();
    ptx::tmem_dealloc(tmem, S::kTmem);
  }

  T* out = static_cast<T*>(p.c);
  const int here = min(p.tokens, p.m - token0);
  if (p.splits == 1) {
    if (warp < 8 && row_base + row < p.n) {
#pragma unroll
      for (int i = 0; i < NH; ++i) {
        const int t = wg * NH + i;
        if (t < here)
          softmax::Elem<T>::store1(out + static_cast<int64_t>(token0 + t) * p.n + row_base + row, kEight || (kScaled && p.a_scales) ? acc[i] * p.a_scales[token0 + t] : acc[i]);
      }
    }
    return;
  }
  // the parts of K, in order
  float* red = reinterpret_cast<float*>(smem);
  if (warp < 8) {
#pragma unroll
    for (int i = 0; i < NH; ++i)
      if (wg * NH + i < here) red[(wg * NH + i) * kRows + row] = acc[i];
  }
  ptx::cluster_sync_all();
  // four rows of W a thread and access (100 x 5003 x 2048 10.7 us; one at a time 14.1)
  for (int i = rank * kThreads + tid; i < here * (kRows / 4); i += p.splits * kThreads) {
    const int j = i / (kRows / 4), t = token0 + j, r = i % (kRows / 4) * 4, left = p.n - row_base - r;
    if (left <= 0) continue;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int q = 0; q < p.splits; ++q) {
      const float4 x = ptx::ld_shared_cluster_f32x4(ptx::mapa_shared(ptx::smem_u32(red + j * kRows + r), q));
      sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
    }
    const float f = kEight || (kScaled && p.a_scales) ? p.a_scales[t] : 1.f;
    alignas(8) T y[4];
    softmax::Elem<T>::store1(y, sum.x * f), softmax::Elem<T>::store1(y + 1, sum.y * f), softmax::Elem<T>::store1(y + 2, sum.z * f);
    softmax::Elem<T>::store1(y + 3, sum.w * f);
    T* to = out + static_cast<int64_t>(t) * p.n + row_base + r;
    if (left >= 4 && reinterpret_cast<uintptr_t>(to) % 8 == 0) {
      *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(y);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) to[e] = y[e];
    }
  }
  ptx::cluster_sync_all();  // the others have read this CTA's sums
}

}  // namespace w4
}  // namespace tsm100
