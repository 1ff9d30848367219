// Attention of a few new tokens over pages where many short pieces meet: single tokens of many sequences behind a prefix that they share, or on their encoders' states.
//
// The products, the running softmax and the tiles are those of attention_paged.cuh.  What differs is who works on what: a share of the stream is a WARP's, which goes from unit
// to unit by itself and leaves a record (O, maximum, sum) of every unit that it has a part of; another kernel joins a row's records.  No barrier is
// met after the stream has been measured, and beginning a unit costs the warp a load of its queries instead of costing the CTA two barriers and a merge of all warps' records:
// 64 sequences of 750 positions in the mean, 8 bits, 8 KV heads, 40 us by CTAs, 31 so (3.2 TB/s); 128 of 450 in bf16 62 and 45 (5.2 TB/s).
//
// Bound: HBM.
#pragma once

#include "attention_paged.cuh"

namespace tsm100 {
namespace paged {

// Which keys a token sees.
//   kPast    positions 0 .. its own of its sequence
//   kAll     all positions of its sequence, however many tokens that has (attention to an encoder's states; none: zeros)
//   kShared  the first p.prefix positions, which lie in the same pages for all sequences: all tokens of the call are the rows of one sequence, number -1
//   kRest    positions p.prefix .. its own; a sequence with more than p.large rows is tcgen05's (attention_paged_tc.cuh), any other the other kernel's
//   kBoth    as kShared and as kRest, as two results, in one stream
enum Keys { kPast, kAll, kShared, kRest, kBoth };
// kAll, kRest and kBoth here, kAll, kShared and kRest on tcgen05.  The last three leave records, which attention_paged_join_kernel puts together; here kAll does too.
__host__ __device__ constexpr bool leaves_records(Keys k) { return k == kShared || k == kRest || k == kBoth; }

// Records of rows: D numbers of O, not normalised, the logarithm to base 2 of what the weights were taken against, their sum, six unused, so that rows start on the 32 bytes
// that memory is written by (with two and stores of 16 bytes 64 sequences behind 16384 positions in 8 bits took 104.0 us, so 101.6).  A unit (or block) of rows that one
// share has all of leaves them in `whole`, by token and head; one that is cut, in the shares' places, which `cut` tells by the unit.
template <int D>
constexpr int kRecord = D + 8;
struct Records {
  float* whole;       // [tokens][heads_q]
  float* part;        // [share][2][held], of a unit that began in an earlier share, of one that goes on in the next
  int2* cut;          // the share that the unit's keys begin in, and how many shares there are, 0 if one; [heads_kv][units], kRest: [batch][heads_kv][units]
  int32_t units;      // of a KV head (of a sequence)
  int32_t shares;     // places in part
};

// The tokens of sequence b and the keys that they see; false, and reported, if they contradict each other or the call.  kRest counts positions from the
// prefix on, and so does its table.
template <Keys kKeys, typename P>
__device__ __forceinline__ bool sequence(const P& p, int b, int& first, int& count, int& len, uint32_t* status, uint32_t site) {
  if (kKeys == kPast) return pages::sequence(p.step, p.cache.page_size, b, first, count, len, status, site);
  if (kKeys == kAll) return pages::sequence<false>(p.step, p.cache.page_size, b, first, count, len, status, site) && len > 0;
  if (b < 0) {
    first = 0, count = min(max(p.step.starts[p.step.batch], 0), p.step.tokens), len = p.prefix;
    return count > 0;
  }
  if (!pages::sequence(p.step, p.cache.page_size, b, first, count, len, status, site)) return false;
  len -= p.prefix;
  // the prefix's rows are the tokens before starts[batch]: with starts in no order a sequence may have others
  if (len >= count && first + count <= p.step.starts[p.step.batch]) return true;
  pages::report(status, site);
  return false;
}
template <typename P>
__device__ __forceinline__ bool is_large(const P& p, int count) { return p.large > 0 && static_cast<int64_t>(count) * p.group > p.large; }

// kAll: a sequence without positions has zeros for results.  Of all threads of a grid, which deal each such sequence's out.
template <int D, Keys kKeys, typename T, typename P>
__device__ __forceinline__ void put_zeros(T* o, const P& p) {
  if constexpr (kKeys == kAll) {
    const int64_t threads = static_cast<int64_t>(gridDim.x) * gridDim.y * blockDim.x;
    const int64_t mine = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x;
    for (int b0 = 0; b0 < p.step.batch; b0 += 32) {  // a warp looks at 32 sequences at once
      const int b = b0 + static_cast<int>(threadIdx.x & 31);
      unsigned empty = __ballot_sync(0xffffffffu, b < p.step.batch && p.step.lens[b] == 0);
      for (; empty != 0u; empty &= empty - 1u) {
        int first, count, len;
        if (!pages::sequence<false>(p.step, p.cache.page_size, b0 + __ffs(empty) - 1, first, count, len, nullptr, 0)) continue;
        uint4* to = reinterpret_cast<uint4*>(o + static_cast<int64_t>(first) * p.heads_q * D);
        const int64_t n = static_cast<int64_t>(count) * p.heads_q * (D / 8);
        for (int64_t i = mine; i < n; i += threads) to[i] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }
}

// Rows of a unit, and the places that a warp's loads run ahead by.
template <bool kI8, int D, bool kWide>
struct RowsTile {
  static constexpr int kWarps = kWide ? 8 : 12, kThreads = kWarps * 32;
  static constexpr int kHeld = kWide ? 16 : 8;
  static constexpr int kBytes = 4096;                     // of K or of V
  static constexpr int kRowBytes = kI8 ? D : 2 * D;
  static constexpr int kPos = kBytes / kRowBytes;         // 16, 32 or 64 positions
  static constexpr int kSlots = kWide ? 6 : 4;            // per warp
  static constexpr int kRec = kRecord<D>;                 // floats of a row's record
  static constexpr int kScales = kI8 ? kPos * 4 : 0;      // bytes beside a slot
  static constexpr int kSmem = kWarps * kSlots * (kBytes + kScales) + kWarps * kSlots * 8 + 1024;
  static_assert(kSmem + 2048 + 160 * kWarps <= 227 * 1024, "shared memory of one CTA, with what is declared in the kernel");
};
// What beginning a unit costs a warp, in tiles.
constexpr int kRowsUnitCost = 1;
// A share's tiles at least: a row has as many records as its keys have shares.
constexpr int kRowsMinShare = 3;

struct RowsParams {
  pages::Cache cache;
  pages::Batch step;
  int32_t heads_q, group;
  int32_t run_log2;   // positions a copy brings: a power of two that divides the page (kTma), else the whole tile
  float scale_log2;   // log2(e) / sqrt(d)
  int32_t prefix;     // Keys
  int32_t large;      // 0: no sequence is
  const int32_t* prefix_table;
  Records shared, rest;
  uint32_t* status;
};

template <Keys kKeys, int kPos, int kHeld>
__device__ __forceinline__ int64_t rows_sequence_tiles(const RowsParams& p, int b, Seq& s, uint32_t* status) {
  if (!sequence<kKeys>(p, b, s.first, s.count, s.len, status, 147)) return 0;
  if (b >= 0 && is_large(p, s.count)) return 0;
  s.tiles = (s.len + kPos - 1) / kPos;
  s.passes = static_cast<int>((static_cast<int64_t>(s.count) * p.group + kHeld - 1) / kHeld);
  s.units = s.passes * p.cache.heads;
  return static_cast<int64_t>(s.tiles + kRowsUnitCost) * s.units;
}

template <typename T, bool kI8, int D, bool kTma, bool kWide, Keys kKeys>
__global__ void __launch_bounds__((RowsTile<kI8, D, kWide>::kThreads), 1)
attention_paged_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const T* __restrict__ q, const __grid_constant__ RowsParams p) {
  using L = RowsTile<kI8, D, kWide>;
  constexpr int kWarps = L::kWarps, kThreads = L::kThreads, kHeld = L::kHeld;
  constexpr int NB = kWide ? 2 : 1;  // eights of rows
  constexpr bool kIsBf16 = !std::is_same<T, __half>::value;
  constexpr bool kMmaBf16 = kIsBf16 && !kI8;
  // f16 results from 8 bits: a probability times V's step takes two f16 numbers.  In one, even the weight of a row's first key was rounded, to as many bits as the result has, and
  // results were 1.4 times as far from 64 bits as that alone makes them (2.9e-4, so 2.1e-4).
  constexpr bool kTwoParts = kI8 && !kIsBf16;
  constexpr int TP = L::kPos, N16 = TP / 16, KSTEPS = D / 16, REC = L::kRec, kSlots = L::kSlots, kChunks = L::kRowBytes / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kWarps * kSlots * (L::kBytes + L::kScales));
  __shared__ int64_t scan[kWarps];
  __shared__ uint32_t abort_word;
  // Parts of units: the one that a warp works on (its sequence is found by whichever thread looked at it), and the one that its loads have come to.
  __shared__ Part parts[kWarps], parts_ahead[kWarps];
  volatile uint32_t* abort_flag = &abort_word;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  if (tid == 0) {
    for (int i = 0; i < kWarps * kSlots; ++i) ptx::mbar_init(&bars[i], 1);
    abort_word = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&tmap_k);
    ptx::prefetch_tensormap(&tmap_v);
  }
  ptx::launch_dependents();
  q = ptx::wait_prior_grid(q);

  // The stream: how long it is, and the sequence in which each warp's share begins.
  const int batch = p.step.batch;
  constexpr int kFirst = kKeys == kBoth ? -1 : 0;  // the stream's first sequence
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
  Seq mine;
  for (int base = kFirst; base < batch; base += kThreads) {
    own = base + tid < batch ? rows_sequence_tiles<kKeys, TP, kHeld>(p, base + tid, mine, p.status) : 0;
    total += block_scan(own, before);
  }
  const int64_t shares = static_cast<int64_t>(gridDim.x) * kWarps, per = max((total + shares - 1) / shares, static_cast<int64_t>(kRowsMinShare));
  const int64_t share0 = static_cast<int64_t>(blockIdx.x) * kWarps;
  auto find = [&](int b, int64_t from) {  // the warps whose shares begin in what this thread looked at
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int64_t t = (share0 + w) * per;
      if (from <= t && t < from + own) parts[w].seq = mine, parts[w].seq.b = b, parts[w].seq.base = from;
    }
  };
  if (batch - kFirst <= kThreads) {
    find(kFirst + tid, before);
  } else {
    int64_t sum = 0;
    for (int base = kFirst; base < batch; base += kThreads) {
      own = base + tid < batch ? rows_sequence_tiles<kKeys, TP, kHeld>(p, base + tid, mine, nullptr) : 0;
      const int64_t here = block_scan(own, before);
      find(base + tid, sum + before);
      sum += here;
    }
  }
  __syncthreads();
  const int share = static_cast<int>(share0) + warp;
  const int64_t t0 = min(total, share * per), t1 = min(total, t0 + per);
  if (t0 >= t1) return;
  auto cut = [&](Part& x) {  // what the share has of the unit, from its beginning on
    x.begin = 0;
    x.end = static_cast<int>(min(static_cast<int64_t>(x.seq.tiles), max(t1 - x.start - kRowsUnitCost, static_cast<int64_t>(0))));
    x.there = x.end > 0;
  };
  auto open = [&](Part& x, int b, int64_t base) {  // the first sequence from b on that has units
    for (; b < batch; ++b)
      if (rows_sequence_tiles<kKeys, TP, kHeld>(p, b, x.seq, nullptr) > 0) break;
    x.seq.b = b, x.seq.base = base;
    x.unit = 0, x.start = base;
  };
  auto next = [&](Part& x) {
    x.start += x.seq.tiles + kRowsUnitCost;
    if (++x.unit == x.seq.units) open(x, x.seq.b + 1, x.start);
    if (x.start >= t1 || x.seq.b >= batch) x.there = false;
    else cut(x);
  };
  Part &now = parts[warp], &ahead = parts_ahead[warp];
  if (lane == 0) {
    Part x;
    x.seq = now.seq;
    x.start = x.seq.base;
    x.unit = static_cast<int>((t0 - x.start) / (x.seq.tiles + kRowsUnitCost));
    x.start += static_cast<int64_t>(x.unit) * (x.seq.tiles + kRowsUnitCost);
    cut(x);
    x.begin = static_cast<int>(max(t0 - x.start - kRowsUnitCost, static_cast<int64_t>(0)));
    x.there = x.end > x.begin;
    if (!x.there) next(x);
    now = x, ahead = x;
  }
  __syncwarp();

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

  // The warp's tiles, ahead of their use: K and V of a tile in turn.
  int load_slot = 0, tile_ahead = ahead.begin, end_ahead = ahead.end, head_ahead = 0, b_ahead = 0, len_ahead = 0;
  bool load_v = false, more = ahead.there;
  auto look = [&]() {
    b_ahead = ahead.seq.b, len_ahead = ahead.seq.len, end_ahead = ahead.end;
    head_ahead = ahead.seq.passes == 1 ? ahead.unit : ahead.unit / ahead.seq.passes;
  };
  look();
  int row_ahead = 0, at_ahead = 0;  // (lane i) the tile's i-th run: its row of pages times heads, and its first position there
  const int page_bits = (ps & (ps - 1)) == 0 ? 31 - __clz(ps) : -1;
  auto settle = [&]() {  // on to the first unit that has tile_ahead for this warp, and (lane i) the page of the tile's i-th run
    if (more && tile_ahead >= end_ahead) {
      __syncwarp();
      if (lane == 0) next(ahead);
      __syncwarp();
      more = ahead.there;
      look();
      tile_ahead = ahead.begin;
    }
    if (!more) return;
    if (kTma) {
      const int pos = tile_ahead * TP + (lane << lb);
      row_ahead = head_ahead, at_ahead = 0;
      if ((lane << lb) < TP && pos < len_ahead) {
        const int nth = page_bits >= 0 ? pos >> page_bits : pos / ps;
        at_ahead = pos - nth * ps;
        int page = kKeys == kBoth && b_ahead < 0 ? p.prefix_table[nth] : p.step.table[static_cast<int64_t>(b_ahead) * p.step.pitch + nth];
        if (page < 0 || page >= p.cache.pages) pages::report(p.status, 148), page = 0;
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
        int pg = 0;
        if (kKeys == kBoth && b_ahead < 0) {
          if (ok && ((pg = p.prefix_table[pos / ps]) < 0 || pg >= p.cache.pages)) pages::report(p.status, 148), pg = 0;
        } else if (ok) {
          pg = max(0, pages::page_of(p.cache, p.step, b_ahead, pos, p.status, 148));
        }
        const int64_t row = (static_cast<int64_t>(pg) * heads + head_ahead) * ps + (ok ? pos % ps : 0);
        mma::cp_async_16(dst + at(r, c), static_cast<const uint8_t*>(p.cache.kv[load_v]) + row * L::kRowBytes + c * 16, ok);
        if (kI8 && c == 0) ptx::cp_async_4(dst_steps + r * 4, p.cache.scales[load_v] + row, ok);
      }
      mma::cp_async_commit();
    }
    if (load_v) {
      ++tile_ahead;
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
      alive = alive && __all_sync(0xffffffffu, ptx::mbar_wait(&full[slot], phase, abort_flag, p.status, 188));
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
  for (; now.there;) {
    const int unit = now.unit, begin = now.begin, end = now.end;
    const int64_t start = now.start;
    struct {
      int b, first, count, len, tiles, passes;
    } const seq = {now.seq.b, now.seq.first, now.seq.count, now.seq.len, now.seq.tiles, now.seq.passes};
    __syncwarp();
    if (lane == 0) next(now);  // read when this one is through
    const bool all = kKeys == kAll || (kKeys == kBoth && seq.b < 0);
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
        limit[n][e] = all ? seq.len - 1 : seq.len - seq.count + mine / p.group;
      }
    }
    const int least = all ? seq.len - 1 : seq.len - seq.count + row0 / p.group;  // the first row's last position: tiles up to it need no masks
    float oacc[KSTEPS][NB][4];
#pragma unroll
    for (int c = 0; c < KSTEPS; ++c)
#pragma unroll
      for (int n = 0; n < NB; ++n) oacc[c][n][0] = oacc[c][n][1] = oacc[c][n][2] = oacc[c][n][3] = 0.f;
    float m[NB][2], l[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
    float v_top = 0x1p-100f;  // 8 bits: the largest step of V so far, oacc is in units of it; far smaller steps count as zero
    for (int tile = begin; tile < end; ++tile) {
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
      // Rounded to what the products take, 16 bits: the tensor core's other types are slower, and results are 1.67e-3 to 1.78e-3 from 64 bits in bf16, whose own rounding is 1.65e-3, and
      // 2.1e-4 to 2.3e-4 in f16 (2.07e-4).  The sums above are of what was not rounded.
      uint32_t pb[N16][NB][2], rest[kTwoParts ? N16 : 1][NB][2];
#pragma unroll
      for (int j = 0; j < N16; ++j)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t x = mma::pack2<kMmaBf16>(s[j][n][2 * h], s[j][n][2 * h + 1]);
            pb[j][n][h] = transposed(x);
            if constexpr (kTwoParts) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
              rest[j][n][h] = transposed(mma::pack2<false>(s[j][n][2 * h] - f.x, s[j][n][2 * h + 1] - f.y));
            }
          }
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
              for (int n = 0; n < NB; ++n) {
                mma_tile<false>(oacc[c + i][n], a0, a1, a2, a3, pb[j][n][0], pb[j][n][1]);
                if constexpr (kTwoParts) mma_tile<false>(oacc[c + i][n], a0, a1, a2, a3, rest[j][n][0], rest[j][n][1]);
              }
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

    const bool whole = begin == 0 && end == seq.tiles;
    const Records& to = kKeys == kBoth && seq.b < 0 ? p.shared : p.rest;
    const float f = kI8 ? v_top : 1.f;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = n * 8 + 2 * tq + e;
        if (r >= rows) continue;
        const int token = (row0 + r) / p.group, h = head * p.group + (row0 + r) % p.group;
        float* rec = whole ? to.whole + (static_cast<int64_t>(seq.first + token) * p.heads_q + h) * REC
                           : to.part + ((static_cast<int64_t>(share) * 2 + (begin == 0 ? 1 : 0)) * kHeld + r) * REC;
#pragma unroll
        for (int c = 0; c < KSTEPS; ++c) {
          if (kI8) {
            *reinterpret_cast<float2*>(rec + c * 16 + 2 * gr) = make_float2(oacc[c][n][e] * f, oacc[c][n][2 + e] * f);
          } else {
            rec[c * 16 + gr] = oacc[c][n][e];
            rec[c * 16 + 8 + gr] = oacc[c][n][2 + e];
          }
        }
        if (gr == 0) *reinterpret_cast<float2*>(rec + D) = make_float2(m[n][e] - kRaised<kMmaBf16>, l[n][e]);
      }
    if (lane == 0 && begin == 0) {
      const int last = static_cast<int>((start + kRowsUnitCost + seq.tiles - 1) / per);  // the share that has the unit's last tile
      to.cut[(seq.b < 0 ? 0 : static_cast<int64_t>(seq.b) * heads * to.units) + static_cast<int64_t>(head) * to.units + (unit - head * seq.passes)] =
          make_int2(share, end == seq.tiles ? 0 : last - share + 1);
    }
    __syncwarp();
    if (!alive) break;
  }
  if constexpr (!kTma) mma::cp_async_wait<0>();
  if (*abort_flag != 0u) {
    // a wait gave up: copies in flight land before the shared memory is released
    const unsigned long long since = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - since < 1000000ull) {
    }
  }
}

// What a row's records add up to.  CTA (b, y) has rows of sequence b: D / 4 threads a row, kSplits times, which deal its records out; four are asked for before the first is used.
// Four, or sixteen where rows have more than 40: 4 sequences on 16384 with 2 KV heads, the whole call, 50 us with four and shares of any size (592 records a row), 23 with sixteen and
// kRowsMinShare.
// A part whose scores are all -inf weighs nothing beside another.
struct Join {
  pages::Cache cache;
  pages::Batch step;
  int32_t heads_q, group;
  int32_t all;            // of kAll: there is no prefix, and zeros where there are no positions
  int32_t prefix, large;
  Records shared, rest, rest_large;
  int32_t shared_tokens, large_tokens;  // of a tile, where the records are tcgen05's (256 rows a block); 0: shared_held, rest_held rows a unit
  int32_t shared_held, rest_held;
};
template <int kSplits>
constexpr int kJoinThreads = kSplits == 4 ? 256 : 512;
// A row's records: the first, and what lies between one share's and the next, in numbers.
struct Pieces {
  const float* first;
  const float* next;
  uint32_t step;
  int n;
};
// (Tokens times heads fit 31 bits, so the rows of a KV head and all of them do.)
template <int D>
__device__ __forceinline__ Pieces pieces(const Records& rec, int tile_tokens, uint32_t held, int64_t cut0, uint32_t head, uint32_t group, uint32_t token, uint32_t h, uint32_t row) {
  constexpr uint32_t REC = kRecord<D>;
  uint32_t unit, r;
  if (tile_tokens > 0) {
    unit = token / (2 * tile_tokens);
    const uint32_t t = token - unit * 2 * tile_tokens, g = t >= static_cast<uint32_t>(tile_tokens) ? 1 : 0;
    r = g * 128 + (t - g * tile_tokens) * group + h, held = 256;
  } else {  // 8 or 16
    const uint32_t at = token * group + h;
    unit = held == 8 ? at >> 3 : at >> 4, r = at & (held - 1);
  }
  const int2 cut = __ldcg(rec.cut + cut0 + static_cast<int64_t>(head) * rec.units + unit);
  Pieces x;
  // a kernel that gave up a wait has left some places unwritten: nothing is read by those
  const bool there = cut.x >= 0 && cut.y >= 0 && cut.x < rec.shares && cut.y <= rec.shares - cut.x;
  x.n = there ? max(cut.y, 1) : 0;
  x.step = 2 * held * REC;
  const float* place = rec.part + (static_cast<int64_t>(cut.x) * (2 * held) + r) * REC;
  x.first = cut.y == 0 ? rec.whole + static_cast<int64_t>(row) * REC : place + held * REC;
  x.next = place + x.step;
  return x;
}
template <typename T, int D, int kSplits>
__global__ void __launch_bounds__(kJoinThreads<kSplits>, 1024 / kJoinThreads<kSplits>)
attention_paged_join_kernel(T* o, const __grid_constant__ Join p) {
  constexpr int kLanes = D / 4, kRowsAt = kJoinThreads<kSplits> / kLanes / kSplits, kAtOnce = 4;
  constexpr bool kIsBf16 = !std::is_same<T, __half>::value;
  __shared__ float4 part_x[kSplits][kRowsAt][kLanes];
  __shared__ float2 part_ml[kSplits][kRowsAt];
  ptx::launch_dependents_if_few();
  ptx::wait_prior_grid();
  const int b = static_cast<int>(blockIdx.x);
  int first, count, len;
  if (p.all ? !pages::sequence<false>(p.step, p.cache.page_size, b, first, count, len, nullptr, 0) : !sequence<kRest>(p, b, first, count, len, nullptr, 0)) return;
  const bool large = is_large(p, count);
  const Records& rest = large ? p.rest_large : p.rest;
  const int rest_tokens = large ? p.large_tokens : 0, lane = threadIdx.x % kLanes, split = threadIdx.x / kLanes % kSplits, mine = threadIdx.x / (kLanes * kSplits);
  const uint32_t rows = static_cast<uint32_t>(count) * p.heads_q, group = p.group;
  for (uint32_t i0 = blockIdx.y * kRowsAt; i0 < rows; i0 += gridDim.y * kRowsAt) {
    const uint32_t i = i0 + mine, row = static_cast<uint32_t>(first) * p.heads_q + i;
    float m = -INFINITY, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < rows && len > 0) {
      const uint32_t token = i / static_cast<uint32_t>(p.heads_q), hq = i - token * p.heads_q, head = hq / group, h = hq - head * group;
      Pieces s = {};
      if (!p.all) s = pieces<D>(p.shared, p.shared_tokens, p.shared_held, 0, head, group, first + token, h, row);
      const Pieces r = pieces<D>(rest, rest_tokens, p.rest_held, static_cast<int64_t>(b) * p.cache.heads * rest.units, head, group, token, h, row);
      const int n = s.n + r.n;
      auto record = [&](int at) {
        const bool of_rest = at >= s.n;
        at -= of_rest ? s.n : 0;
        const float* next = of_rest ? r.next : s.next;
        return at == 0 ? (of_rest ? r.first : s.first) : next + static_cast<int64_t>(at - 1) * (of_rest ? r.step : s.step);
      };
      for (int j0 = split; j0 < n; j0 += kSplits * kAtOnce) {
        float2 ml[kAtOnce];
        float4 y[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          const int at = j0 + j * kSplits;
          ml[j] = make_float2(-INFINITY, 0.f), y[j] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (at < n) {
            const float* rec = record(at);
            ml[j] = __ldcg(reinterpret_cast<const float2*>(rec + D)), y[j] = __ldcg(reinterpret_cast<const float4*>(rec) + lane);
          }
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) top = fmaxf(top, ml[j].x);
        const float keep = m == -INFINITY ? 0.f : ptx::ex2_approx(m - top);
        l *= keep, x.x *= keep, x.y *= keep, x.z *= keep, x.w *= keep;
        // a part of no scores but -inf weighs nothing; it is added all the same, because one of NaN scores has that maximum too
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          if (j0 + j * kSplits >= n) break;
          const float w = ml[j].x == -INFINITY ? 0.f : ptx::ex2_approx(ml[j].x - top);
          l = fmaf(w, ml[j].y, l);
          x.x = fmaf(w, y[j].x, x.x), x.y = fmaf(w, y[j].y, x.y), x.z = fmaf(w, y[j].z, x.z), x.w = fmaf(w, y[j].w, x.w);
        }
        m = top;
      }
    }
    __syncthreads();  // what the rows before left has been read
    part_x[split][mine][lane] = x;
    if (lane == 0) part_ml[split][mine] = make_float2(m, l);
    __syncthreads();
    if (split == 0 && i < rows) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < kSplits; ++j) top = fmaxf(top, part_ml[j][mine].x);
      l = 0.f, x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < kSplits; ++j) {
        const float2 ml = part_ml[j][mine];
        const float4 y = part_x[j][mine][lane];
        const float w = ml.x == -INFINITY ? 0.f : ptx::ex2_approx(ml.x - top);
        l = fmaf(w, ml.y, l);
        x.x = fmaf(w, y.x, x.x), x.y = fmaf(w, y.y, x.y), x.z = fmaf(w, y.z, x.z), x.w = fmaf(w, y.w, x.w);
      }
      const float inv = len > 0 ? 1.f / l : 0.f;
      *reinterpret_cast<uint2*>(o + static_cast<int64_t>(row) * D + lane * 4) = make_uint2(mma::pack2<kIsBf16>(x.x * inv, x.y * inv), mma::pack2<kIsBf16>(x.z * inv, x.w * inv));
    }
  }
}

}  // namespace paged
}  // namespace tsm100
