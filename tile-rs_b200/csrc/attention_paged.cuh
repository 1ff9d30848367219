// Attention of a few new tokens over the pages of their sequences (single tokens above all): a token at position p sees positions 0 .. p.
//
//   o[t,h] = sum_j w_j V[j] / sum_j w_j,   w_j = 2^(s_j - m),   s_j = (q[t,h] . K[j]) log2(e) / sqrt(d),   m = max_j s_j
//
// in one pass over the keys: a running (m, sum, O), rescaled when m grows; parts of a sequence that different warps or CTAs have seen are joined
// by their maxima.
//
// Bound: HBM, the cache is read once.  So the tiles of all (sequence, KV head) pairs are numbered through and every SM takes an equal, contiguous share of
// them, which may begin and end inside a pair: how uneven the sequences are does not matter, and no grid has to be planned from lengths that only the device knows.
// A pair's new tokens times the heads of its group are its rows, up to eight (kWide: sixteen) at a time; more rows are further passes over the pair's keys.
//
// The products are mma.sync tiles with the keys, and V's columns, on the side of sixteen and the rows on the side of eight, S^T = K Q^T and O^T = V^T P^T, so that a
// group of eight heads or fewer leaves none of them idle: half the products, and half the registers, of tiles with the rows on the other side.  P^T is transposed between the two by movmatrix.
// A CTA's warps take the tiles of its share in turn: K and V come by TMA, a box per page or part of one (128-byte swizzle, no multicast), into slots of a warp's own.
// Pages that are no multiple of eight positions are fetched row by row with cp.async instead.
//
// 8 bits: whole numbers become f16 exactly (a byte behind 0x64 is 1024 + byte), K's step multiplies the score and V's the probability, over the
// largest step so far (the accumulator is rescaled when that grows), so that only the probability is rounded.  bf16 queries are brought to f16 by a power of two per row.
#pragma once

#include "attention_decode.cuh"
#include "kv_pages.cuh"
#include "ptx.cuh"

namespace tsm100 {
namespace paged {

namespace mma = attn_decode::mma;

constexpr int kRows = 16;     // of a pass, at most
constexpr int kMaxCtas = 1024;
// What beginning and ending a pair costs, in tiles: shares are as long in tiles and these.  64 sequences of up to 6000 positions in 8 bits, costs of 4, 8, 12, 16, 24, 32 tiles:
// 109, 100, 94, 94, 97, 100 us.  (Heads of 128; taken for 16-bit caches, heads of 64 and wide rows too, unmeasured.)
constexpr int kUnitCost = 16;
template <bool kI8, int D, bool kWide>
struct Tile {
  static constexpr int kWarps = kWide ? 8 : 12, kThreads = kWarps * 32;
  static constexpr int kHeld = kWide ? 16 : 8;            // rows
  static constexpr int kBytes = 4096;                     // of K or of V
  static constexpr int kRowBytes = kI8 ? D : 2 * D;
  static constexpr int kPos = kBytes / kRowBytes;         // 16, 32 or 64 positions
  static constexpr int kSlots = kWide ? 5 : 3;            // per warp
  static constexpr int kRec = D + 4;                      // floats of a row's record: O, maximum, sum; 16-byte rows
  static constexpr int kScales = kI8 ? kPos * 4 : 0;      // bytes beside a slot
  static constexpr int kSmem = kWarps * kSlots * (kBytes + kScales) + kWarps * 8 * kRec * 4 + kWarps * kSlots * 8 + 1024;
  static_assert(kSmem + 224 + 72 * kWarps <= 227 * 1024, "shared memory of one CTA, with what is declared in the kernel");
};

struct Params {
  pages::Cache cache;
  pages::Batch step;
  int32_t heads_q, group;
  int32_t run_log2;   // positions a copy brings: a power of two that divides the page (kTma), else the whole tile
  float scale_log2;   // log2(e) / sqrt(d)
  float* part;        // [CTA][2][kHeld][kRec]: of a pair that began in an earlier share, of one that goes on in the next
  int4* info;         // [CTA]: 1 if a pair of earlier shares ends in this one, 2 if it goes on; sequence and unit of the pair that goes on in the next, or -1
  uint32_t* status;
};

// A sequence's place in the stream.  Its units, the keys of one KV head for up to kHeld rows, are kUnitCost and their tiles long.
struct Seq {
  int b, first, count, len;
  int tiles;      // of a unit
  int passes;     // units of a KV head
  int units;
  int64_t base;   // where it begins
};
// A unit, or a share's part of it.
struct Part {
  Seq seq;
  int unit, begin, end;  // tiles
  int64_t start;         // where the unit begins
  bool there;
};
template <int kPos, int kHeld>
__device__ __forceinline__ int64_t sequence_tiles(const Params& p, int b, Seq& s, uint32_t* status) {
  if (!pages::sequence(p.step, p.cache.page_size, b, s.first, s.count, s.len, status, 143)) return 0;
  s.tiles = (s.len + kPos - 1) / kPos;
  s.passes = static_cast<int>((static_cast<int64_t>(s.count) * p.group + kHeld - 1) / kHeld);
  s.units = s.passes * p.cache.heads;
  return static_cast<int64_t>(s.tiles + kUnitCost) * s.units;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int32_t y, int32_t z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(bar)), "r"(0), "r"(y), "r"(z)
               : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int32_t y, int32_t w) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %3, %5}], [%2];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(bar)), "r"(0), "r"(y), "r"(w)
               : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(ptx::smem_u32(bar))
               : "memory");
}
// Two of the four whole numbers of x, as f16: bytes 0 and 1, 2 and 3, 0 and 2 or 1 and 3 (the selector says which, 4 stands for 0x64).
__device__ __forceinline__ uint32_t i8_pair(uint32_t biased, uint32_t selector) {
  const uint32_t h = __byte_perm(biased, 0x64646464u, selector);  // 1024 + 128 + q
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// f16 has numbers to 2^-14 in full, and probabilities are 1 at most (8 bits: times a step over the largest): weights and their sum are taken 2^15 times as large, so that those
// of keys far behind the first, or beside a large V, keep their bits.  8000 keys of which the first has 2^20 times another's weight and V = 0: f16 off by 1.9e-3, on tcgen05 by 4e-3, with them as they are, by less than 6e-4 so.
template <bool kBf16>
constexpr float kRaised = kBf16 ? 0.f : 15.f;

template <bool kIsBf16>
__device__ __forceinline__ void mma_tile(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (kIsBf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {  // an 8 x 8 tile of 16-bit numbers
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

template <typename T, bool kI8, int D, bool kTma, bool kWide>
__global__ void __launch_bounds__((Tile<kI8, D, kWide>::kThreads), 1)
attention_paged_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const T* __restrict__ q, T* __restrict__ o,
                       const __grid_constant__ Params p) {
  using L = Tile<kI8, D, kWide>;
  constexpr int kWarps = L::kWarps, kThreads = L::kThreads, kHeld = L::kHeld;
  constexpr int NB = kWide ? 2 : 1;  // eights of rows
  constexpr bool kIsBf16 = !std::is_same<T, __half>::value;
  constexpr bool kMmaBf16 = kIsBf16 && !kI8;
  constexpr int TP = L::kPos, N16 = TP / 16, KSTEPS = D / 16, REC = L::kRec, kSlots = L::kSlots, kChunks = L::kRowBytes / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* records = reinterpret_cast<float*>(smem + kWarps * kSlots * (L::kBytes + L::kScales));
  uint64_t* bars = reinterpret_cast<uint64_t*>(records + kWarps * 8 * REC);
  __shared__ int64_t scan[kWarps + 1];
  __shared__ uint32_t abort_word;
  __shared__ int first_seq;
  volatile uint32_t* abort_flag = &abort_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  if (tid == 0) {
    for (int i = 0; i < kWarps * kSlots; ++i) ptx::mbar_init(&bars[i], 1);
    abort_word = 0;
    first_seq = p.step.batch;
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&tmap_k);
    ptx::prefetch_tensormap(&tmap_v);
  }
  ptx::launch_dependents();
  q = ptx::wait_prior_grid(q);

  // The stream: how long it is, and the sequence in which this CTA's share begins.
  const int batch = p.step.batch;
  auto block_scan = [&](int64_t v, int64_t& before) {  // of all threads; answers the total
    int64_t x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    int64_t total = 0;
    before = x - v;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    return total;
  };
  int64_t total = 0, before = 0, own = 0;
  for (int base = 0; base < batch; base += kThreads) {
    Seq s;
    own = base + tid < batch ? sequence_tiles<TP, kHeld>(p, base + tid, s, p.status) : 0;
    total += block_scan(own, before);
  }
  const int64_t per = (total + gridDim.x - 1) / gridDim.x;
  const int64_t t0 = min(total, blockIdx.x * per), t1 = min(total, t0 + per);
  if (t0 < t1) {
    if (batch <= kThreads) {
      if (before <= t0 && t0 < before + own) first_seq = tid, scan[kWarps] = before;
    } else {
      int64_t sum = 0;
      for (int base = 0; base < batch; base += kThreads) {
        Seq s;
        own = base + tid < batch ? sequence_tiles<TP, kHeld>(p, base + tid, s, nullptr) : 0;
        const int64_t here = block_scan(own, before);
        if (sum + before <= t0 && t0 < sum + before + own) first_seq = base + tid, scan[kWarps] = sum + before;
        sum += here;
      }
    }
  }
  __syncthreads();
  if (t0 >= t1) {
    if (tid == 0) p.info[blockIdx.x] = make_int4(0, -1, -1, 0);
    return;
  }
  auto cut = [&](Part& x) {  // what the share has of the unit, from its beginning on
    x.begin = 0;
    x.end = static_cast<int>(min(static_cast<int64_t>(x.seq.tiles), max(t1 - x.start - kUnitCost, static_cast<int64_t>(0))));
    x.there = x.end > 0;
  };
  auto open = [&](Part& x, int b, int64_t base) {  // the first sequence from b on that has units
    for (; b < batch; ++b)
      if (sequence_tiles<TP, kHeld>(p, b, x.seq, nullptr) > 0) break;
    x.seq.b = b, x.seq.base = base;
    x.unit = 0, x.start = base;
  };
  auto next = [&](Part& x) {
    x.start += x.seq.tiles + kUnitCost;
    if (++x.unit == x.seq.units) open(x, x.seq.b + 1, x.start);
    if (x.start >= t1 || x.seq.b >= batch) x.there = false;
    else cut(x);
  };
  // Parts live in shared memory: the CTA's, the one that its thread 0 finds while the warps work on that, and each warp's that its loads have come to.
  __shared__ Part parts[2], parts_ahead[kWarps];
  if (tid == 0) {
    Part x;
    open(x, first_seq, scan[kWarps]);
    x.unit = static_cast<int>((t0 - x.start) / (x.seq.tiles + kUnitCost));
    x.start += static_cast<int64_t>(x.unit) * (x.seq.tiles + kUnitCost);
    cut(x);
    x.begin = static_cast<int>(max(t0 - x.start - kUnitCost, static_cast<int64_t>(0)));
    x.there = x.end > x.begin;
    if (!x.there) next(x);
    parts[0] = x;
    for (int i = 0; i < kWarps; ++i) parts_ahead[i] = x;
  }
  __syncthreads();
  Part& ahead = parts_ahead[warp];

  const uint32_t slots = ptx::smem_u32(smem) + warp * (kSlots * L::kBytes);
  const uint32_t steps = ptx::smem_u32(smem) + kWarps * kSlots * L::kBytes + warp * (kSlots * L::kScales);
  const float* steps_at = reinterpret_cast<const float*>(smem + kWarps * kSlots * L::kBytes + warp * (kSlots * L::kScales));
  uint64_t* full = bars + warp * kSlots;
  const int heads = p.cache.heads, ps = p.cache.page_size;
  const int lb = p.run_log2, run = 1 << lb;  // of the tile's rows, what lies together: see at()
  // where 16 bytes `chunk` of position `pos` of a tile are in its slot
  auto at = [&](int pos, int chunk) -> uint32_t {
    if constexpr (L::kRowBytes == 256) return ((pos >> lb) << (lb + 8)) + ((chunk >> 3) << (lb + 7)) + ((pos & (run - 1)) << 7) + (((chunk & 7) ^ (pos & 7)) << 4);
    else if constexpr (L::kRowBytes == 128) return (pos << 7) + ((chunk ^ (pos & 7)) << 4);
    else return (pos << 6) + ((chunk ^ ((pos >> 1) & 3)) << 4);
  };

  // The warp's tiles, ahead of their use: K and V of a tile in turn.  Tiles are dealt to the warps in turn, across units.
  int load_slot = 0, tile_ahead = ahead.begin + warp, end_ahead = ahead.end, head_ahead = 0, turn_ahead = 0, b_ahead = 0, len_ahead = 0;
  bool load_v = false, more = ahead.there;
  auto look = [&]() {
    b_ahead = ahead.seq.b, len_ahead = ahead.seq.len, end_ahead = ahead.end;
    head_ahead = ahead.seq.passes == 1 ? ahead.unit : ahead.unit / ahead.seq.passes;
  };
  look();
  int row_ahead = 0, at_ahead = 0;  // (lane i) the tile's i-th run: its row of pages times heads, and its first position there
  const int page_bits = (ps & (ps - 1)) == 0 ? 31 - __clz(ps) : -1;
  auto settle = [&]() {  // on to the first unit that has tile_ahead for this warp, and (lane i) the page of the tile's i-th run
    while (more && tile_ahead >= end_ahead) {
      turn_ahead = (turn_ahead + end_ahead - ahead.begin) % kWarps;
      __syncwarp();
      if (lane == 0) next(ahead);
      __syncwarp();
      more = ahead.there;
      look();
      tile_ahead = ahead.begin + (warp >= turn_ahead ? warp - turn_ahead : warp + kWarps - turn_ahead);
    }
    if (!more) return;
    if (kTma) {
      const int pos = tile_ahead * TP + (lane << lb);
      row_ahead = head_ahead, at_ahead = 0;
      if ((lane << lb) < TP && pos < len_ahead) {
        const int nth = page_bits >= 0 ? pos >> page_bits : pos / ps;
        at_ahead = pos - nth * ps;
        int page = p.step.table[static_cast<int64_t>(b_ahead) * p.step.pitch + nth];
        if (page < 0 || page >= p.cache.pages) pages::report(p.status, 144), page = 0;
        row_ahead += page * heads;
      }
    }
  };
  auto issue = [&]() {
    if (!more) {
      if (!kTma) mma::cp_async_commit();
      return;
    }
    const int pos0 = tile_ahead * TP, here = min(TP, len_ahead - pos0);
    const uint32_t dst = slots + load_slot * L::kBytes, dst_steps = steps + load_slot * L::kScales;
    if constexpr (kTma) {
      const int runs = (here + run - 1) >> lb;
      if (lane == 0) ptx::mbar_arrive_expect_tx(&full[load_slot], runs * (run * (L::kRowBytes + (kI8 ? 4 : 0))));
      __syncwarp();
      if (lane < runs) {
        const CUtensorMap* map = load_v ? &tmap_v : &tmap_k;
        const uint32_t to = dst + ((lane << lb) * L::kRowBytes);
        if constexpr (L::kRowBytes == 256) tma_load_4d(to, map, &full[load_slot], at_ahead, row_ahead);
        else tma_load_3d(to, map, &full[load_slot], at_ahead, row_ahead);
        if constexpr (kI8)
          bulk_load(dst_steps + (lane << lb) * 4, (load_v ? p.cache.scales[1] : p.cache.scales[0]) + static_cast<int64_t>(row_ahead) * ps + at_ahead, run * 4, &full[load_slot]);
      }
    } else {
      for (int i = lane; i < TP * kChunks; i += 32) {
        const int r = i / kChunks, c = i % kChunks, pos = pos0 + r;
        const bool ok = r < here;
        const int pg = ok ? max(0, pages::page_of(p.cache, p.step, b_ahead, pos, p.status, 144)) : 0;
        const int64_t row = (static_cast<int64_t>(pg) * heads + head_ahead) * ps + (ok ? pos % ps : 0);
        mma::cp_async_16(dst + at(r, c), static_cast<const uint8_t*>(p.cache.kv[load_v]) + row * L::kRowBytes + c * 16, ok);
        if (kI8 && c == 0) ptx::cp_async_4(dst_steps + r * 4, p.cache.scales[load_v] + row, ok);
      }
      mma::cp_async_commit();
    }
    if (load_v) {
      tile_ahead += kWarps;
      settle();
    }
    load_v = !load_v;
    load_slot = load_slot + 1 == kSlots ? 0 : load_slot + 1;
  };
  settle();
#pragma unroll
  for (int i = 0; i < kSlots; ++i) issue();

  int slot = 0;
  uint32_t phase = 0;
  bool alive = true;
  auto arrived = [&]() {
    if constexpr (kTma) {
      alive = alive && __all_sync(0xffffffffu, ptx::mbar_wait(&full[slot], phase, abort_flag, p.status, 131));
    } else {
      mma::cp_async_wait<kSlots - 1>();
      __syncwarp();
    }
    return alive;
  };
  auto release = [&]() {  // every lane has read the slot: it is filled again
    __syncwarp();
    if (++slot == kSlots) slot = 0, phase ^= 1u;
    issue();
  };
  // What this lane's ldmatrix addresses start from, in a slot: 16 positions, chunk 0 or 1.  A pair of chunks further is the same with bits 5 and 6 turned (no row starts
  // inside them), eight chunks further the run's next 128-byte group.
  uint32_t k_from[N16], v_from[N16];
#pragma unroll
  for (int j = 0; j < N16; ++j) {
    k_from[j] = at(j * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, (lane >> 4) & 1);  // (positions 0-7, chunk 0), (8-15, 0), (0-7, 1), (8-15, 1)
    v_from[j] = at(j * 16 + (lane & 7) + ((lane >> 4) & 1) * 8, (lane >> 3) & 1);  // (positions 0-7, chunk 0), (0-7, 1), (8-15, 0), (8-15, 1)
  }
  const uint32_t group = L::kRowBytes == 256 ? 1u << (lb + 7) : 0u;
  auto pair_of = [&](uint32_t from, int pair) -> uint32_t { return (from ^ ((pair & 3) << 5)) + (pair >= 4 ? group : 0u); };
  uint32_t qb[NB][KSTEPS][2];  // row gr of an eight: its Q as B fragments
  // of rows 2 tq and 2 tq + 1 of an eight, whose scores this lane has at positions gr and gr + 8 of a sixteen
  float q_factor[NB][2];       // what the row of Q was divided by
  int limit[NB][2];            // the last position it sees
  int head_state = 0, tail_b = -1, tail_unit = -1, turn = 0;
  for (int which = 0; parts[which].there; which ^= 1) {
    const Part& now = parts[which];
    const int unit = now.unit, begin = now.begin, end = now.end;
    struct {
      int b, first, count, len, tiles, passes;
    } const seq = {now.seq.b, now.seq.first, now.seq.count, now.seq.len, now.seq.tiles, now.seq.passes};
    if (tid == 0) {  // the others look at it when they have met at the records
      Part x = now;
      next(x);
      parts[which ^ 1] = x;
    }
    const int head = seq.passes == 1 ? unit : unit / seq.passes, row0 = (unit - head * seq.passes) * kHeld;
    const int rows = min(kHeld, seq.count * p.group - row0);
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const bool ok = n * 8 + gr < rows;
      const int r = row0 + (ok ? n * 8 + gr : 0), token = r / p.group;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(q + (static_cast<int64_t>(seq.first + token) * p.heads_q + head * p.group + r % p.group) * D);
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        if (kI8) {  // the four numbers of a fragment lie together in a row of the cache
          const uint2 x = ok ? __ldg(reinterpret_cast<const uint2*>(src + kk * 8 + 2 * tq)) : make_uint2(0u, 0u);
          qb[n][kk][0] = x.x, qb[n][kk][1] = x.y;
        } else {
          qb[n][kk][0] = ok ? __ldg(src + kk * 8 + tq) : 0u;
          qb[n][kk][1] = ok ? __ldg(src + kk * 8 + tq + 4) : 0u;
        }
      }
      float factor = 1.f;
      if constexpr (kI8 && kIsBf16) {
        float top = 0.f;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
          for (int i = 0; i < 2; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(qb[n][kk][i] << 16)), fabsf(__uint_as_float(qb[n][kk][i] & 0xffff0000u))));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the largest magnitude to 2^14 and more: f16 has all eight bits of what lies 2^28 below it, and some down to 2^38.  Over whole numbers that are 0 where the largest
        // is, that is what makes the scores
        const int ex = min(max(static_cast<int>(__float_as_uint(top) >> 23), 20), 254) - 127 - 14;
        factor = __uint_as_float(static_cast<uint32_t>(ex + 127) << 23);
        const float inv = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t& x = qb[n][kk][i];
            x = mma::pack2<false>(__uint_as_float(x << 16) * inv, __uint_as_float(x & 0xffff0000u) * inv);
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        q_factor[n][e] = __shfl_sync(0xffffffffu, factor, (2 * tq + e) * 4) * p.scale_log2;
        const int mine = row0 + min(n * 8 + 2 * tq + e, rows - 1);
        limit[n][e] = seq.len - seq.count + mine / p.group;
      }
    }
    const int least = seq.len - seq.count + row0 / p.group;  // the first row's last position: tiles up to it need no masks
    float oacc[KSTEPS][NB][4];
#pragma unroll
    for (int c = 0; c < KSTEPS; ++c)
#pragma unroll
      for (int n = 0; n < NB; ++n) oacc[c][n][0] = oacc[c][n][1] = oacc[c][n][2] = oacc[c][n][3] = 0.f;
    float m[NB][2], l[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
    float v_top = 0x1p-100f;  // 8 bits: the largest step of V so far, oacc is in units of it; far smaller steps count as zero
    for (int tile = begin + (warp >= turn ? warp - turn : warp + kWarps - turn); tile < end; tile += kWarps) {
      if (!arrived()) break;
      const uint32_t ks = slots + slot * L::kBytes;
      float s[N16][NB][4];
#pragma unroll
      for (int j = 0; j < N16; ++j)
#pragma unroll
        for (int n = 0; n < NB; ++n) s[j][n][0] = s[j][n][1] = s[j][n][2] = s[j][n][3] = 0.f;
      if constexpr (!kI8) {
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
          for (int j = 0; j < N16; ++j) {
            uint32_t ka[4];
            mma::ldmatrix_x4(pair_of(ks + k_from[j], kk), ka);
#pragma unroll
            for (int n = 0; n < NB; ++n) mma_tile<kMmaBf16>(s[j][n], ka[0], ka[1], ka[2], ka[3], qb[n][kk][0], qb[n][kk][1]);
          }
      } else {
#pragma unroll
        for (int kk = 0; kk < KSTEPS; kk += 2)
#pragma unroll
          for (int j = 0; j < N16; ++j) {
            uint32_t kx[4];
            mma::ldmatrix_x4(pair_of(ks + k_from[j], kk / 2), kx);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t x = kx[2 * i] ^ 0x80808080u, y = kx[2 * i + 1] ^ 0x80808080u;
              const uint32_t a0 = i8_pair(x, 0x4140), a1 = i8_pair(y, 0x4140), a2 = i8_pair(x, 0x4342), a3 = i8_pair(y, 0x4342);
#pragma unroll
              for (int n = 0; n < NB; ++n) mma_tile<false>(s[j][n], a0, a1, a2, a3, qb[n][kk + i][0], qb[n][kk + i][1]);
            }
          }
      }
      const int pos = tile * TP + gr;
      const bool masked = (tile + 1) * TP - 1 > least;
#pragma unroll
      for (int j = 0; j < N16; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float step = kI8 ? steps_at[slot * TP + j * 16 + h * 8 + gr] : 1.f;
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) s[j][n][2 * h + e] *= kI8 ? step * q_factor[n][e] : p.scale_log2;
        }
      release();
      if (masked) {
#pragma unroll
        for (int j = 0; j < N16; ++j)
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (pos + j * 16 + (e >> 1) * 8 > limit[n][e & 1]) s[j][n][e] = -INFINITY;
      }
      float a[NB][2];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = -INFINITY;
#pragma unroll
          for (int j = 0; j < N16; ++j) top = fmaxf(top, fmaxf(s[j][n][e], s[j][n][2 + e]));
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          const float most = fmaxf(m[n][e], top), seen = most == -INFINITY ? 0.f : most;  // a row may see nothing of this warp's first tiles
          a[n][e] = ptx::ex2_approx(m[n][e] - seen);
          const float base = seen - kRaised<kMmaBf16>;
          m[n][e] = most;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < N16; ++j) {
            s[j][n][e] = ptx::ex2_approx(s[j][n][e] - base);
            s[j][n][2 + e] = ptx::ex2_approx(s[j][n][2 + e] - base);
            sum += s[j][n][e] + s[j][n][2 + e];
          }
          l[n][e] = fmaf(l[n][e], a[n][e], sum);
        }
      if (!arrived()) break;
      const uint32_t vs = slots + slot * L::kBytes;
      const bool ragged = (tile + 1) * TP > seq.len;
      if constexpr (kI8) {
        float st[N16][2], top = v_top;
#pragma unroll
        for (int j = 0; j < N16; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            st[j][h] = steps_at[slot * TP + j * 16 + h * 8 + gr];
            if (ragged && pos + j * 16 + h * 8 >= seq.len) st[j][h] = 0.f;  // behind the last position may be anything
            top = fmaxf(top, st[j][h]);
          }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float inv = 1.f / top;
#pragma unroll
        for (int n = 0; n < NB; ++n) a[n][0] *= v_top * inv, a[n][1] *= v_top * inv;
        v_top = top;
#pragma unroll
        for (int j = 0; j < N16; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float x = st[j][h] * inv;
#pragma unroll
            for (int n = 0; n < NB; ++n) s[j][n][2 * h] *= x, s[j][n][2 * h + 1] *= x;
          }
      }
      uint32_t pb[N16][NB][2];
#pragma unroll
      for (int j = 0; j < N16; ++j)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) pb[j][n][h] = transposed(mma::pack2<kMmaBf16>(s[j][n][2 * h], s[j][n][2 * h + 1]));
#pragma unroll
      for (int c = 0; c < KSTEPS; ++c)
#pragma unroll
        for (int n = 0; n < NB; ++n) oacc[c][n][0] *= a[n][0], oacc[c][n][1] *= a[n][1], oacc[c][n][2] *= a[n][0], oacc[c][n][3] *= a[n][1];
      if (!kI8 && ragged) {
        // what lies behind the last position weighs nothing, but may be anything
        for (int i = lane; i < TP * kChunks; i += 32)
          if (tile * TP + i / kChunks >= seq.len) ptx::st_shared_v4(vs + at(i / kChunks, i % kChunks), 0u, 0u, 0u, 0u);
        __syncwarp();
      }
#pragma unroll
      for (int c = 0; c < KSTEPS; ++c)
#pragma unroll
        for (int j = 0; j < N16; ++j) {
          uint32_t va[4];
          if constexpr (!kI8) {
            // transposed on load: (d 0-7, positions 0-7), (d 8-15, 0-7), (d 0-7, 8-15), (d 8-15, 8-15)
            mma::ldmatrix_x4_trans(pair_of(vs + v_from[j], c), va);
#pragma unroll
            for (int n = 0; n < NB; ++n) mma_tile<kMmaBf16>(oacc[c][n], va[0], va[1], va[2], va[3], pb[j][n][0], pb[j][n][1]);
          } else if (c % 2 == 0) {
            // the same of pairs of numbers: two positions of column 2 gr and of column 2 gr + 1 in a register, which become rows gr and gr + 8
            mma::ldmatrix_x4_trans(pair_of(vs + v_from[j], c / 2), va);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t x = va[i] ^ 0x80808080u, y = va[2 + i] ^ 0x80808080u;
              const uint32_t a0 = i8_pair(x, 0x4240), a1 = i8_pair(x, 0x4341), a2 = i8_pair(y, 0x4240), a3 = i8_pair(y, 0x4341);
#pragma unroll
              for (int n = 0; n < NB; ++n) mma_tile<false>(oacc[c + i][n], a0, a1, a2, a3, pb[j][n][0], pb[j][n][1]);
            }
          }
        }
      if (!kI8 && ragged && kTma) ptx::fence_proxy_async_smem();  // the zeros before the slot's next copy
      release();
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], off);

    // the warps' records, eight rows at a time
    const bool whole = begin == 0 && end == seq.tiles;
    for (int half = 0; half * 8 < rows; ++half) {
      __syncthreads();  // the records before have been read
      {
        float* rec = records + (warp * 8 + 2 * tq) * REC;
        const float f = kI8 ? v_top : 1.f;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          if (n != half) continue;
#pragma unroll
          for (int c = 0; c < KSTEPS; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (kI8) {
                *reinterpret_cast<float2*>(rec + e * REC + c * 16 + 2 * gr) = make_float2(oacc[c][n][e] * f, oacc[c][n][2 + e] * f);
              } else {
                rec[e * REC + c * 16 + gr] = oacc[c][n][e];
                rec[e * REC + c * 16 + 8 + gr] = oacc[c][n][2 + e];
              }
            }
          if (gr == 0) {
            *reinterpret_cast<float2*>(rec + D) = make_float2(m[n][0], l[n][0]);
            *reinterpret_cast<float2*>(rec + REC + D) = make_float2(m[n][1], l[n][1]);
          }
        }
      }
      __syncthreads();
      for (int i = tid; i < min(8, rows - half * 8) * (D / 4); i += kThreads) {
        const int rr = i / (D / 4), dd = i % (D / 4) * 4;
        const float* rec = records + rr * REC;
        float2 ml[kWarps];
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          ml[w] = *reinterpret_cast<const float2*>(rec + w * 8 * REC + D);
          mm = fmaxf(mm, ml[w].x);
        }
        float ll = 0.f;
        float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          // a warp that has seen nothing weighs nothing; it is added all the same, because one of NaN scores has that maximum too
          const float wgt = ml[w].x == -INFINITY ? 0.f : ptx::ex2_approx(ml[w].x - mm);
          const float4 x = *reinterpret_cast<const float4*>(rec + w * 8 * REC + dd);
          ll = fmaf(ml[w].y, wgt, ll);
          oo.x = fmaf(x.x, wgt, oo.x), oo.y = fmaf(x.y, wgt, oo.y), oo.z = fmaf(x.z, wgt, oo.z), oo.w = fmaf(x.w, wgt, oo.w);
        }
        const int r = half * 8 + rr;
        if (whole) {
          const int token = (row0 + r) / p.group, h = head * p.group + (row0 + r) % p.group;
          const float inv = 1.f / ll;
          *reinterpret_cast<uint2*>(o + (static_cast<int64_t>(seq.first + token) * p.heads_q + h) * D + dd) =
              make_uint2(mma::pack2<kIsBf16>(oo.x * inv, oo.y * inv), mma::pack2<kIsBf16>(oo.z * inv, oo.w * inv));
        } else {
          float* out = p.part + ((static_cast<int64_t>(blockIdx.x) * 2 + (begin == 0 ? 1 : 0)) * kHeld + r) * REC;
          *reinterpret_cast<float4*>(out + dd) = oo;
          if (dd == 0) *reinterpret_cast<float2*>(out + D) = make_float2(mm, ll);
        }
      }
    }
    if (begin > 0) head_state = end == seq.tiles ? 1 : 2;
    else if (end < seq.tiles) tail_b = seq.b, tail_unit = unit;
    turn = (turn + end - begin) % kWarps;
  }
  if (tid == 0) p.info[blockIdx.x] = make_int4(head_state, tail_b, tail_unit, 0);
  if constexpr (!kTma) mma::cp_async_wait<0>();
  if (*abort_flag != 0u) {
    // a wait gave up: copies in flight land before the shared memory is released
    const unsigned long long since = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - since < 1000000ull) {
    }
    __syncthreads();
  }
}

// How many records a unit has that goes on behind the share of this CTA's column: that share's second, and the first of those behind it up to the one it ends in.  A warp
// looks at 32 shares at once.
__device__ __forceinline__ int records_of(const int4* info) {
  const int lane = threadIdx.x & 31;
  int n = 1;
  for (int at = blockIdx.x + 1; at < static_cast<int>(gridDim.x); at += 32) {
    const unsigned on = __ballot_sync(0xffffffffu, at + lane < static_cast<int>(gridDim.x) && __ldcg(&info[at + lane].x) == 2);
    if (on != 0xffffffffu) return n + __ffs(~on);
    n += 32;
  }
  return n;
}

// The records of a pair that several shares have a part of, in order; a warp per row, CTA (x, y) rows 4 y .. of the pair that goes on behind share x.
template <typename T, int D, int kHeld>
__global__ void __launch_bounds__(128)
attention_paged_merge_kernel(T* __restrict__ o, const __grid_constant__ Params p) {
  constexpr int REC = D + 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.y * 4 + warp;
  ptx::launch_dependents();
  ptx::wait_prior_grid();
  const int4 mine = __ldcg(p.info + blockIdx.x);
  if (mine.y < 0) return;
  const int n = records_of(p.info);
  const int first = p.step.starts[mine.y], count = p.step.starts[mine.y + 1] - first;
  const int passes = static_cast<int>((static_cast<int64_t>(count) * p.group + kHeld - 1) / kHeld), head = mine.z / passes, row = mine.z % passes * kHeld + r;
  if (r >= kHeld || row >= count * p.group) return;
  auto record = [&](int i) { return p.part + ((static_cast<int64_t>(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * kHeld + r) * REC; };
  float mm = -INFINITY;
  for (int i = lane; i < n; i += 32) mm = fmaxf(mm, __ldcg(record(i) + D));
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, off));
  float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
  float ll = 0.f;
  for (int base = 0; base < n; base += 32) {
    float w = 0.f;
    if (base + lane < n) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(record(base + lane) + D));
      w = ml.x == -INFINITY ? 0.f : ptx::ex2_approx(ml.x - mm);
      ll = fmaf(ml.y, w, ll);
    }
    const int here = min(32, n - base);
#pragma unroll 8
    for (int i = 0; i < here; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      if (lane < D / 4) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(record(base + i)) + lane);
        oo.x = fmaf(x.x, wi, oo.x), oo.y = fmaf(x.y, wi, oo.y), oo.z = fmaf(x.z, wi, oo.z), oo.w = fmaf(x.w, wi, oo.w);
      }
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, off);
  if (lane < D / 4) {
    const float inv = 1.f / ll;
    constexpr bool kIsBf16 = !std::is_same<T, __half>::value;
    *reinterpret_cast<uint2*>(o + (static_cast<int64_t>(first + row / p.group) * p.heads_q + head * p.group + row % p.group) * D + lane * 4) =
        make_uint2(mma::pack2<kIsBf16>(oo.x * inv, oo.y * inv), mma::pack2<kIsBf16>(oo.z * inv, oo.w * inv));
  }
}

}  // namespace paged
}  // namespace tsm100
