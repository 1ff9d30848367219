// Attention of chunks of new tokens over the pages of their sequences, on tcgen05: a token at position p sees positions 0 .. p.
//
// Semantics and the running softmax as attention_paged.cuh, the pipeline as attention_tc.cuh: two tiles of 128 query rows against steps of 128 keys, S and O in
// tensor memory, a thread per row, probabilities handed over through shared memory, one warp issuing Q K^T a step ahead and one P V.  What differs:
//   * The rows of a tile are tokens times the heads of a group (row = token * group + head), so that a group's heads read K and V once and a chunk of a few tokens
//     still fills a tile.  One TMA box brings them: 64 columns x group x tokens.
//   * The work is one stream, dealt out evenly: blocks of up to two tiles are numbered through (sequence, KV head, block) with the keys they see, and what beginning one
//     costs, as their length, and every SM takes an equal, contiguous share of it, to the step.  Lengths are only known on the device, prompts and single tokens come in
//     one call, and 64 blocks over 148 SMs would leave half of them idle.  A block that is cut leaves (maximum, sum, O) for a merging kernel.  (A block of one tile counts
//     like one of two: two thirds of that cost 2 to 9 % in four mixes of six and gained nothing in the others.  256 keys for beginning a block: 128 cost up to 13 %, 512 up to 7.)
//   * K and V come by pages: boxes of a power of two of positions (8 and more), a lane each.  What a page holds behind the sequence's end is
//     replaced by zeros in V (it has no weight, but may be NaN) and masked in S.
//   * 8 bits (kI8): four warps write the tiles that TMA would have written, whole numbers, which 16 bits hold exactly.  K's steps multiply the scores and V's the
//     probabilities, so that nothing but the probabilities is rounded (with K and V times their steps rounded, errors were 1.6 times as large), and those to f16, whatever q's type
//     is.  They keep their bits by a power of two that follows the largest step and is taken out again with the sum.
//     (Sums of queries times whole numbers are f32 before K's step comes to them: queries end at 2^114.)
//   * Probabilities are rounded to 16 bits, which P V takes them in; their sum is of unrounded ones.  Cross attention in f16 is 2.5e-4 from 64 bits where rounding the result alone
//     makes 2.1e-4, on a shared prefix in bf16 1.8e-3 to 2.0e-3 where it makes 1.65e-3.
// Bound: the tensor core and the exponentials, as there.
#pragma once

#include "attention_paged.cuh"
#include "attention_paged_rows.cuh"
#include "attention_tc.cuh"
#include "kv_pages.cuh"
#include "ptx.cuh"
#include "quantise.cuh"

namespace tsm100 {
namespace paged {
namespace tc {

constexpr int kTileRows = 128, kKeys = 128;
constexpr int kMaxGroup = 128;
constexpr int kBlockCost = 2 * kKeys;  // beginning and ending a block, as a length
constexpr int kMinShare = 4 * kKeys;   // a share's length at least
// How far the maximum that probabilities are taken against may lag, in log2 units.  8 bits: little, for the sake of what follows (the mixed step
// of 12 sequences 203 us, 202 with 8 and three more for the step of V).
template <bool kI8>
constexpr float kLag = kI8 ? 2.f : attn::kRescaleThreshold;
// f16 has numbers to 2^-14 in full: there probabilities and their sum are taken so many powers of two larger that the largest (2^kLag; 8 bits: times a step of less than
// twice 2^v_used) stay within 2^15, and those of keys far behind the first, or beside a large V, keep their bits (attention_paged.cuh).
template <bool kI8, bool kPvBf16>
constexpr float kRaised = kPvBf16 ? 0.f : kI8 ? 14.f - kLag<true> : 15.f - kLag<false>;

template <bool kI8, int D>
struct Shape {
  static constexpr int kThreads = kI8 ? 512 : 384;   // warps 0..3 softmax A, 4..7 softmax B, 8 TMA, 9 Q K^T, 10 P V, 11 planning, 12..15 conversion
  // registers after setmaxnreg; the shares of a block add up to what it was launched with
  static constexpr int kRegsSoftmax = kI8 ? 184 : 216, kRegsOther = kI8 ? 48 : 72, kRegsConvert = 96;
  static constexpr int kHalves = D / 64;
  static constexpr int kHalfBytes = 128 * 128;        // 128 rows x 64 columns
  static constexpr int kTileBytes = kHalves * kHalfBytes;
  static constexpr int kPBytes = 2 * kHalfBytes;
  static constexpr int kRing = D == 128 ? 3 : 6;
  static constexpr int kStepBytes = kI8 ? 2 * kKeys * 4 + 16 : 0;  // of a tile: K's, V's, and the largest of V's that each of the four warps saw; two tiles
  static constexpr int kPOff = 2 * kTileBytes, kRingOff = kPOff + 2 * kPBytes, kStepsOff = kRingOff + kRing * kTileBytes, kBarsOff = kStepsOff + 2 * kStepBytes;
};
static_assert(256 * 184 + 128 * 48 + 128 * 96 <= 512 * 128 && 256 * 216 + 128 * 72 <= 384 * 168, "registers of a block at launch");

// A block, or a share's part of it.  One warp finds them, a few ahead, and the others read them here.
struct Work {
  int b, first, count, len;
  int head, block, token0;   // first token, in the sequence's new ones
  int steps, begin, n;       // of the block, and the part that is this share's
  int n_a;                   // of that, what tile A takes part in (causality)
  int lone, there;           // one tile; false behind the last part
};
constexpr int kPlans = 4;

struct alignas(8) Barriers {
  uint64_t q_full, q_free;
  uint64_t kv_full[6], kv_empty[6];
  uint64_t tail;              // the copies of a V tile that ends behind its sequence
  uint64_t s_full[2], s_free[2], p_ready[2], pv_done[2], o_free[2];
  uint64_t steps_free[2][2];  // [query tile][place]
  uint64_t plan_full[kPlans], plan_empty[kPlans];
  Work plan[kPlans];
  int64_t scan[17];
  int64_t first_base;
  int32_t first_seq;
  uint32_t tmem_base;
  uint32_t abort_flag;
  uint32_t pv_steps;          // steps whose P V has been issued (only grows)
};
// The shared memory of a kernel without variables of its own begins on a 1024-byte boundary (it is checked); there is no room for more.
template <bool kI8, int D>
constexpr int smem_bytes() { return Shape<kI8, D>::kBarsOff + static_cast<int>(sizeof(Barriers)); }
static_assert(smem_bytes<true, 128>() <= 227 * 1024 && smem_bytes<true, 64>() <= 227 * 1024, "shared memory of one CTA");

struct Params {
  pages::Cache cache;
  pages::Batch step;
  int32_t heads_q, group;
  int32_t tokens;      // of a tile: 128 / group
  int32_t run_log2;    // positions of a page's box
  float scale_log2;
  int32_t prefix;      // attention_paged_rows.cuh: Keys
  int32_t large;
  const int32_t* prefix_table;
  Records records;
  float4* part;        // [CTA][2][D / 4][256 rows]: of a block that began in an earlier share, of one that goes on in the next
  float2* part_ml;     // [CTA][2][256]
  int4* info;          // [CTA]: as attention_paged.cuh, with the block's sequence, KV head and number
  uint32_t* status;
};

// The stream of blocks.  A block's length is the keys that its last token sees, and kBlockCost.
struct Seq {
  int b, first, count, len, blocks;
  int64_t per_head, base, end;
};
template <Keys kKeysSeen>
__device__ __forceinline__ int64_t full_blocks(const Params& p, const Seq& s, int64_t i) {  // the length of the first i blocks, which have two tiles
  if (kKeysSeen == kAll || kKeysSeen == kShared) return i * (s.len + kBlockCost);
  const int64_t two = 2 * p.tokens;
  return i * (s.len - s.count + kBlockCost) + two * (i * (i + 1) / 2);
}
template <Keys kKeysSeen>
__device__ __forceinline__ int64_t sequence_length(const Params& p, int b, Seq& s, uint32_t* status) {
  if (!sequence<kKeysSeen>(p, kKeysSeen == kShared ? -1 : b, s.first, s.count, s.len, status, 145)) return 0;
  if (kKeysSeen == kRest && !is_large(p, s.count)) return 0;
  s.blocks = (s.count + 2 * p.tokens - 1) / (2 * p.tokens);
  s.per_head = full_blocks<kKeysSeen>(p, s, s.blocks - 1) + s.len + kBlockCost;
  return s.per_head * p.cache.heads;
}
template <Keys kKeysSeen>
__device__ __forceinline__ int sequences(const Params& p) { return kKeysSeen == kShared ? 1 : p.step.batch; }
template <Keys kKeysSeen>
struct Stream {
  Seq seq;
  int64_t at, end, per;
  __device__ __forceinline__ void open(const Params& p, int b, int64_t base) {  // the first sequence from b on that has blocks
    int64_t n = 0;
    for (; b < sequences<kKeysSeen>(p); ++b)
      if ((n = sequence_length<kKeysSeen>(p, b, seq, nullptr)) > 0) break;
    seq.b = b, seq.base = base, seq.end = base + n;
  }
  __device__ __forceinline__ bool next(const Params& p, Work& w) {
    while (at < end) {
      while (at >= seq.end && seq.b < sequences<kKeysSeen>(p)) open(p, seq.b + 1, seq.end);
      if (seq.b >= sequences<kKeysSeen>(p)) return false;
      const int64_t in_seq = at - seq.base;
      w.head = static_cast<int>(in_seq / seq.per_head);
      const int64_t in_head = in_seq - w.head * seq.per_head;
      int lo = 0, hi = seq.blocks - 1;  // the last block that begins at in_head or before
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (full_blocks<kKeysSeen>(p, seq, mid) <= in_head) lo = mid;
        else hi = mid - 1;
      }
      const bool last = lo == seq.blocks - 1;
      const int64_t from = full_blocks<kKeysSeen>(p, seq, lo), to = last ? seq.per_head : full_blocks<kKeysSeen>(p, seq, lo + 1);
      w.token0 = lo * 2 * p.tokens;
      const int keys = kKeysSeen == kAll || kKeysSeen == kShared ? seq.len : seq.len - seq.count + min(seq.count, w.token0 + 2 * p.tokens);
      w.steps = (keys + kKeys - 1) / kKeys;
      const int64_t stop = min(to, in_head + (end - at));
      auto steps_to = [&](int64_t x) { return static_cast<int>((static_cast<uint32_t>(max(x - from - kBlockCost, static_cast<int64_t>(0))) + kKeys - 1) / kKeys); };
      w.begin = steps_to(in_head);
      w.n = steps_to(stop) - w.begin;
      w.b = seq.b, w.first = seq.first, w.count = seq.count, w.len = seq.len, w.block = lo;
      w.lone = last && seq.count - w.token0 <= p.tokens;
      const int keys_a = kKeysSeen == kAll || kKeysSeen == kShared ? seq.len : seq.len - seq.count + min(seq.count, w.token0 + p.tokens);
      w.n_a = max(0, min(w.n, (keys_a + kKeys - 1) / kKeys - w.begin));
      if constexpr (leaves_records(kKeysSeen)) {
        if (w.n > 0 && w.begin == 0) {
          const int64_t last = seq.base + w.head * seq.per_head + from + kBlockCost + static_cast<int64_t>(w.steps - 1) * kKeys;  // where the last step begins
          p.records.cut[(kKeysSeen == kRest ? static_cast<int64_t>(seq.b) * p.cache.heads * p.records.units : 0) + static_cast<int64_t>(w.head) * p.records.units + lo] =
              make_int2(static_cast<int>(blockIdx.x), w.n == w.steps ? 0 : static_cast<int>(last / per) - static_cast<int>(blockIdx.x) + 1);
        }
      }
      at += stop - in_head;
      if (w.n > 0) return true;
    }
    return false;
  }
};

// pages::page_of, of the prefix's pages for kShared.
template <Keys kKeysSeen>
__device__ __forceinline__ int page_at_position(const Params& p, int b, int pos) {
  if constexpr (kKeysSeen == kShared) {
    const int page = p.prefix_table[pos / p.cache.page_size];
    if (page >= 0 && page < p.cache.pages) return page;
    pages::report(p.status, 146);
    return -1;
  } else {
    return pages::page_of(p.cache, p.step, b, pos, p.status, 146);
  }
}

template <bool kIsBf16, bool kI8, int D, Keys kKeysSeen = kPast>
__global__ void __launch_bounds__(Shape<kI8, D>::kThreads, 1)
attention_paged_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                          uint16_t* __restrict__ o, const __grid_constant__ Params p) {
  using S = Shape<kI8, D>;
  constexpr bool kPvBf16 = kIsBf16 && !kI8;  // of P and V
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((ptx::smem_u32(smem) & 1023u) != 0u) {
    ptx::wait_prior_grid();
    if (threadIdx.x == 0 && !leaves_records(kKeysSeen)) p.info[blockIdx.x] = make_int4(0, -1, 0, 0);
    if (threadIdx.x == 0) atomicCAS(p.status, ptx::kStatusOk, ptx::kStatusWaitTimeout | 174u);
    return;
  }
  uint8_t* smem_q = smem;                  // two tiles
  uint8_t* smem_p = smem + S::kPOff;       // the probabilities of tile A and of tile B
  uint8_t* smem_kv = smem + S::kRingOff;
  Barriers* bars = reinterpret_cast<Barriers*>(smem + S::kBarsOff);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* abort_flag = &bars->abort_flag;
  if (tid == 0) {
    ptx::mbar_init(&bars->q_full, 1);
    ptx::mbar_init(&bars->q_free, 1);
    ptx::mbar_init(&bars->tail, 1);
    for (int s = 0; s < S::kRing; ++s) {
      ptx::mbar_init(&bars->kv_full[s], kI8 ? 128 : 1);
      ptx::mbar_init(&bars->kv_empty[s], 1);
    }
    for (int g = 0; g < 2; ++g) {
      ptx::mbar_init(&bars->s_full[g], 1);
      ptx::mbar_init(&bars->s_free[g], 128);
      ptx::mbar_init(&bars->p_ready[g], 128);
      ptx::mbar_init(&bars->pv_done[g], 1);
      ptx::mbar_init(&bars->o_free[g], 128);
      for (int i = 0; i < 2; ++i) ptx::mbar_init(&bars->steps_free[g][i], 128);
    }
    for (int i = 0; i < kPlans; ++i) {
      ptx::mbar_init(&bars->plan_full[i], 1);
      ptx::mbar_init(&bars->plan_empty[i], kI8 ? 15 : 11);  // the other warps
    }
    bars->abort_flag = 0;
    bars->pv_steps = 0;
    bars->first_seq = sequences<kKeysSeen>(p);
    bars->first_base = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 9) {
    ptx::tmem_alloc(&bars->tmem_base, 512);
    ptx::tmem_relinquish_alloc_permit();
  }
  ptx::tcgen05_fence_before_thread_sync();
  __syncthreads();
  ptx::tcgen05_fence_after_thread_sync();
  const uint32_t tmem_base = bars->tmem_base;
  ptx::launch_dependents();
  ptx::wait_prior_grid();

  // The stream: how long it is, and where this CTA's share begins.
  Stream<kKeysSeen> stream;
  {
    constexpr int kThreads = S::kThreads;
    const int batch = sequences<kKeysSeen>(p);
    auto block_scan = [&](int64_t v, int64_t& before) {  // answers the total
      int64_t x = v;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, off);
        if (lane >= off) x += y;
      }
      __syncthreads();
      if (lane == 31) bars->scan[warp] = x;
      __syncthreads();
      int64_t sum = 0;
      before = x - v;
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) before += bars->scan[w];
        sum += bars->scan[w];
      }
      return sum;
    };
    int64_t total = 0, before = 0;
    Seq s;
    for (int base = 0; base < batch; base += kThreads) total += block_scan(base + tid < batch ? sequence_length<kKeysSeen>(p, base + tid, s, p.status) : 0, before);
    const int64_t per = max((total + gridDim.x - 1) / gridDim.x, static_cast<int64_t>(kMinShare));
    stream.at = min(total, blockIdx.x * per), stream.end = min(total, stream.at + per), stream.per = per;
    int64_t sum = 0;
    for (int base = 0; base < batch; base += kThreads) {
      const int64_t own = base + tid < batch ? sequence_length<kKeysSeen>(p, base + tid, s, nullptr) : 0;
      const int64_t here = block_scan(own, before);
      if (sum + before <= stream.at && stream.at < sum + before + own) bars->first_seq = base + tid, bars->first_base = sum + before;
      sum += here;
    }
    __syncthreads();
  }
  const uint32_t tmem_s = tmem_base;        // S_A at +0, S_B at +128
  const uint32_t tmem_o = tmem_base + 256;  // O_A at +256, O_B at +384
  // The next part, for a whole warp; given back when the warp is through with it.
  int part_no = -1;
  auto take = [&]() -> bool {
    ++part_no;
    const bool ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->plan_full[part_no % kPlans], (part_no / kPlans) & 1u, abort_flag, p.status, 176));
    return ok && bars->plan[part_no % kPlans].there;
  };
  auto give = [&]() {
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&bars->plan_empty[part_no % kPlans]);
  };

  if (warp == 8) {
    // ------------------------------ TMA producer ------------------------------
    ptx::setmaxnreg_dec<S::kRegsOther>();
    if (lane == 0) {
      ptx::prefetch_tensormap(&tmap_q);
      if (!kI8) ptx::prefetch_tensormap(&tmap_k), ptx::prefetch_tensormap(&tmap_v);
    }
    const int run = 1 << p.run_log2, ps = p.cache.page_size;
    int idx0 = 0, tails = 0;
    bool ok = true;
    for (int seg = 0; ok && take(); ++seg) {
      const Work w = bars->plan[part_no % kPlans];
      if (seg > 0 && !(ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->q_free, (seg - 1) & 1u, abort_flag, p.status, 151)))) break;
      if (lane == 0) {
        ptx::mbar_arrive_expect_tx(&bars->q_full, (w.lone ? 1 : 2) * (p.tokens * p.group * 128 * S::kHalves));
        for (int g = 0; g < (w.lone ? 1 : 2); ++g)
          for (int c = 0; c < S::kHalves; ++c)
            ptx::tma_load_3d(smem_q + g * S::kTileBytes + c * S::kHalfBytes, &tmap_q, &bars->q_full, c * 64, w.head * p.group, w.first + w.token0 + g * p.tokens);
      }
      if constexpr (!kI8) {
        // in the order in which the tensor core first needs the tiles: K_0, K_1, V_0, K_2, V_1, ..., K_{n-1}, V_{n-2}, V_{n-1}
        const int my_run = S::kHalves == 2 ? lane >> 1 : lane, half = S::kHalves == 2 ? lane & 1 : 0;
        auto page_at = [&](int step) {  // of this lane's run; asked for a tile ahead
          const int pos = (w.begin + step) * kKeys + my_run * run;
          return my_run * run < kKeys && step < w.n && pos < w.len ? max(0, page_at_position<kKeysSeen>(p, w.b, pos)) : 0;
        };
        const int total = 2 * w.n;
        int page_k = page_at(0), page_v = page_k;
        for (int i = 0; i < total && ok; ++i) {
          const int slot = (idx0 + i) % S::kRing;
          const bool is_v = i == total - 1 || (i >= 2 && (i & 1) == 0);
          const int step = i == 0 ? 0 : i == total - 1 ? w.n - 1 : is_v ? (i >> 1) - 1 : (i + 1) >> 1;
          const int pos0 = (w.begin + step) * kKeys, here = min(kKeys, w.len - pos0), runs = (here + run - 1) >> p.run_log2;
          const int page = is_v ? page_v : page_k;
          // the pages of the next tiles: K runs a step ahead of V
          if (is_v) page_v = page_at(step + 1);
          else page_k = page_at(step + 1);
          if (!(ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->kv_empty[slot], (((idx0 + i) / S::kRing) & 1u) ^ 1u, abort_flag, p.status, 152)))) break;
          const bool ragged = is_v && here < kKeys;
          uint64_t* bar = ragged ? &bars->tail : &bars->kv_full[slot];
          if (lane == 0) ptx::mbar_arrive_expect_tx(bar, runs * run * 128 * S::kHalves);
          __syncwarp();
          if (my_run < runs)
            ptx::tma_load_3d(smem_kv + slot * S::kTileBytes + half * S::kHalfBytes + my_run * run * 128, is_v ? &tmap_v : &tmap_k, bar, half * 64,
                             (pos0 + my_run * run) % ps, page * p.cache.heads + w.head);
          if (ragged) {
            if (!(ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->tail, tails & 1u, abort_flag, p.status, 153)))) break;
            ++tails;
            const uint32_t tile = ptx::smem_u32(smem_kv + slot * S::kTileBytes);
            for (int e = here * 8 + lane; e < kKeys * 8; e += 32)
#pragma unroll
              for (int c = 0; c < S::kHalves; ++c) ptx::st_shared_v4(tile + c * S::kHalfBytes + e * 16, 0u, 0u, 0u, 0u);
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&bars->kv_full[slot]);
          }
        }
        idx0 += total;
      }
      give();
    }
  } else if (warp == 9 || warp == 10) {
    // ------------------------------ MMA issuers --------------------------------
    ptx::setmaxnreg_dec<S::kRegsOther>();
    constexpr uint32_t idesc_qk = ptx::make_idesc_f16(kTileRows, kKeys, false, false, kIsBf16);
    constexpr uint32_t idesc_pv = ptx::make_idesc_f16(kTileRows, D, false, true, kPvBf16);
    constexpr uint64_t kmajor = ptx::make_smem_desc_base(16, 1024);
    constexpr uint64_t v_mnmajor = ptx::make_smem_desc_base(S::kHalfBytes, 1024);
    // everything per MMA is one add on the low word of a descriptor
    constexpr uint32_t k_hi = static_cast<uint32_t>(kmajor >> 32), v_hi = static_cast<uint32_t>(v_mnmajor >> 32);
    constexpr uint32_t k_lo_base = static_cast<uint32_t>(kmajor), v_lo_base = static_cast<uint32_t>(v_mnmajor);
    auto desc64 = [](uint32_t hi, uint32_t lo) -> uint64_t { return (static_cast<uint64_t>(hi) << 32) | lo; };
    // K and V written by TMA are only handed on to the tensor core; written by warps (kI8, the end of a sequence), the wait acquires
    auto wait_kv = [&](int idx, bool written) -> bool {
      uint64_t* bar = &bars->kv_full[idx % S::kRing];
      const uint32_t parity = (idx / S::kRing) & 1u;
      const bool r = kI8 || written ? ptx::mbar_wait(bar, parity, abort_flag, p.status, 154) : ptx::mbar_wait_relaxed(bar, parity, abort_flag, p.status, 155);
      return __all_sync(0xffffffffu, r);
    };
    int idx0 = 0, steps_before = 0;
    int done[2] = {0, 0};       // steps of each tile in earlier segments
    int segs[2] = {0, 0};       // segments that each tile took part in
    bool ok = true;
    for (int seg = 0; ok && take(); ++seg) {
      const Work w = bars->plan[part_no % kPlans];
      auto k_pos = [&](int j) { return idx0 + (j == 0 ? 0 : 2 * j - 1); };
      auto v_pos = [&](int j) { return idx0 + (j == w.n - 1 ? 2 * w.n - 1 : 2 * j + 2); };
      const int n_of[2] = {w.n_a, w.lone ? 0 : w.n};
      if (warp == 9) {
        const uint32_t q_lo = k_lo_base | (ptx::smem_u32(smem_q) >> 4), ring_lo = k_lo_base | (ptx::smem_u32(smem_kv) >> 4);
        ok = __all_sync(0xffffffffu, ptx::mbar_wait_relaxed(&bars->q_full, seg & 1u, abort_flag, p.status, 156));
        ptx::tcgen05_fence_after_thread_sync();
        for (int j = 0; j < w.n && ok; ++j) {
          // not before the P V products of two steps ago are in the tensor core's queue (attention_tc.cuh)
          const int s = steps_before + j;
          if (s >= 2 && !(ok = __all_sync(0xffffffffu, ptx::wait_counter_ge(&bars->pv_steps, static_cast<uint32_t>(s - 1), abort_flag, p.status, 157)))) break;
          if (!(ok = wait_kv(k_pos(j), false))) break;
          ptx::tcgen05_fence_after_thread_sync();
          for (int g = 0; g < 2 && ok; ++g) {
            if (j >= n_of[g]) continue;
            const int c = done[g] + j;
            if (c > 0) {  // every softmax thread of the tile holds the scores before in registers
              ok = __all_sync(0xffffffffu, ptx::mbar_wait_relaxed(&bars->s_free[g], (c - 1) & 1u, abort_flag, p.status, 158 + g));
              ptx::tcgen05_fence_after_thread_sync();
              if (!ok) break;
            }
            const uint32_t a_lo = q_lo + g * (S::kTileBytes >> 4), b_lo = ring_lo + k_pos(j) % S::kRing * (S::kTileBytes >> 4), d = tmem_s + g * 128;
            if (ptx::elect_one_sync()) {
#pragma unroll
              for (int kk = 0; kk < D / 16; ++kk) {
                const uint32_t off = (kk >> 2) * (S::kHalfBytes >> 4) + (kk & 3) * 2;
                ptx::tcgen05_mma_f16_ss(d, desc64(k_hi, a_lo + off), desc64(k_hi, b_lo + off), idesc_qk, kk != 0 ? 1u : 0u);
              }
              ptx::tcgen05_commit(&bars->s_full[g]);
            }
            __syncwarp();
          }
          if (!ok) break;
          if (ptx::elect_one_sync()) {
            ptx::tcgen05_commit(&bars->kv_empty[k_pos(j) % S::kRing]);
            if (j == w.n - 1) ptx::tcgen05_commit(&bars->q_free);
          }
          __syncwarp();
        }
      } else {
        const uint32_t p_lo = k_lo_base | (ptx::smem_u32(smem_p) >> 4), ring_lo = v_lo_base | (ptx::smem_u32(smem_kv) >> 4);
        for (int j = 0; j < w.n && ok; ++j) {
          bool landed = false;
          for (int g = 0; g < 2 && ok; ++g) {
            if (j >= n_of[g]) continue;
            if (j == 0 && segs[g] > 0) {  // the segment before has left tensor memory
              ok = __all_sync(0xffffffffu, ptx::mbar_wait_relaxed(&bars->o_free[g], (segs[g] - 1) & 1u, abort_flag, p.status, 160 + g));
              if (!ok) break;
            }
            ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->p_ready[g], (done[g] + j) & 1u, abort_flag, p.status, 162 + g));
            // V_j after P_j, never before: in a ring of three its slot had K_j, and while that has not landed a wait for V_j's phase, of which the parity is the one before K_j's,
            // would pass at once.  Probabilities say that K_j was read.
            if (ok && !landed) ok = landed = wait_kv(v_pos(j), (w.begin + j + 1) * kKeys > w.len);
            ptx::tcgen05_fence_after_thread_sync();
            if (!ok) break;
            const uint32_t a_lo = p_lo + g * (S::kPBytes >> 4), b_lo = ring_lo + v_pos(j) % S::kRing * (S::kTileBytes >> 4), d = tmem_o + g * 128;
            if (ptx::elect_one_sync()) {
#pragma unroll
              for (int kk = 0; kk < kKeys / 16; ++kk) {
                const uint32_t a_off = (kk >> 2) * (S::kHalfBytes >> 4) + (kk & 3) * 2;
                ptx::tcgen05_mma_f16_ss(d, desc64(k_hi, a_lo + a_off), desc64(v_hi, b_lo + kk * (2048 >> 4)), idesc_pv, (j > 0 || kk != 0) ? 1u : 0u);
              }
              ptx::tcgen05_commit(&bars->pv_done[g]);
            }
            __syncwarp();
          }
          if (!ok) break;
          if (ptx::elect_one_sync()) {
            ptx::tcgen05_commit(&bars->kv_empty[v_pos(j) % S::kRing]);
            *const_cast<volatile uint32_t*>(&bars->pv_steps) = static_cast<uint32_t>(steps_before + j + 1);
          }
          __syncwarp();
        }
      }
      idx0 += 2 * w.n;
      steps_before += w.n;
#pragma unroll
      for (int g = 0; g < 2; ++g) done[g] += n_of[g], segs[g] += n_of[g] > 0 ? 1 : 0;
      give();
    }
  } else if (warp == 11) {
    // ------------------------------ planning -----------------------------------
    ptx::setmaxnreg_dec<S::kRegsOther>();
    if (lane == 0) {
      int head_state = 0, tail_b = -1, tail_head = 0, tail_block = 0;
      stream.open(p, bars->first_seq, bars->first_base);
      for (int i = 0;; ++i) {
        Work w = {};
        w.there = stream.next(p, w) ? 1 : 0;
        if (!ptx::mbar_wait(&bars->plan_empty[i % kPlans], ((i / kPlans) & 1u) ^ 1u, abort_flag, p.status, 177)) break;
        bars->plan[i % kPlans] = w;
        ptx::mbar_arrive(&bars->plan_full[i % kPlans]);
        if (!w.there) break;
        if (w.begin > 0) head_state = w.begin + w.n == w.steps ? 1 : 2;
        else if (w.n < w.steps) tail_b = w.b, tail_head = w.head, tail_block = w.block;
      }
      if (!leaves_records(kKeysSeen)) p.info[blockIdx.x] = make_int4(head_state, tail_b, tail_head, tail_block);
    }
  } else if (kI8 && warp >= 12) {
    // ------------------------------ conversion ---------------------------------
    if constexpr (kI8) {
      ptx::setmaxnreg_dec<S::kRegsConvert>();
      constexpr int kVecs = D / 16;             // 16-byte vectors of a row, and of a thread in a tile
      constexpr int kRowsAt = 128 / kVecs;      // rows that the four warps write at once
      const int cw = warp - 12, ps = p.cache.page_size;
      // A warp has 32 rows of a tile, a lane finds one of them: row (lane / kOwn) * kRowsAt + cw * kOwn + lane % kOwn
      constexpr int kOwn = 32 / kVecs;
      const int my_row = lane / kOwn * kRowsAt + cw * kOwn + lane % kOwn;
      int idx0 = 0, uses[2][2] = {{0, 0}, {0, 0}};  // how often a query tile has read a place's steps
      bool ok = true;
      while (ok && take()) {
        const Work w = bars->plan[part_no % kPlans];
        // A tile's page is asked for three tiles ahead, its steps two and its rows one, so that none of these loads is waited for.
        const int total = 2 * w.n;
        auto second = [&](int i) { return i == total - 1 || (i >= 2 && (i & 1) == 0); };  // V
        auto pos_of = [&](int i) { return (w.begin + (i == 0 ? 0 : i == total - 1 ? w.n - 1 : (i & 1) == 0 ? (i >> 1) - 1 : (i + 1) >> 1)) * kKeys + my_row; };
        int32_t page = -1;        // of this lane's row of a tile
        int64_t row_at = -1;      // -1: behind the sequence's end
        float k_step = 0.f, v_step = 0.f, k_next = 0.f, v_next = 0.f;  // with a tile of K come the steps of both
        uint4 next[kVecs];
        auto ask_page = [&](int i) {
          const int pos = pos_of(i);
          page = i < total && pos < w.len ? (kKeysSeen == kShared ? p.prefix_table : p.step.table + static_cast<int64_t>(w.b) * p.step.pitch)[pos / ps] : 0;
        };
        auto ask_step = [&](int i) {
          const int pos = pos_of(i);
          row_at = -1;
          k_step = v_step = 0.f;
          if (i < total && pos < w.len) {
            if (page < 0 || page >= p.cache.pages) {
              pages::report(p.status, 146);
              page = 0;
            }
            row_at = (static_cast<int64_t>(page) * p.cache.heads + w.head) * ps + pos % ps;
            if (!second(i)) k_step = p.cache.scales[0][row_at], v_step = p.cache.scales[1][row_at];
          }
        };
        auto ask_rows = [&](int i) {
          k_next = k_step, v_next = v_step;
          const uint8_t* from = static_cast<const uint8_t*>(second(i) ? p.cache.kv[1] : p.cache.kv[0]);
#pragma unroll
          for (int v = 0; v < kVecs; ++v) {
            const int64_t at = __shfl_sync(0xffffffffu, row_at, v * kOwn + lane / kVecs);
            next[v] = make_uint4(0u, 0u, 0u, 0u);
            if (at >= 0) next[v] = __ldg(reinterpret_cast<const uint4*>(from + at * D) + lane % kVecs);
          }
        };
        ask_page(0);
        ask_step(0);
        ask_page(1);
        ask_rows(0);
        ask_step(1);
        ask_page(2);
        for (int i = 0; i < total; ++i) {
          uint4 x[kVecs];
#pragma unroll
          for (int v = 0; v < kVecs; ++v) x[v] = next[v];
          const float k_now = k_next, v_now = v_next;
          ask_rows(i + 1);
          ask_step(i + 2);
          ask_page(i + 3);
          const int slot = (idx0 + i) % S::kRing;
          if (!(ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->kv_empty[slot], (((idx0 + i) / S::kRing) & 1u) ^ 1u, abort_flag, p.status, 164)))) break;
          const uint32_t to = ptx::smem_u32(smem_kv + slot * S::kTileBytes);
          const bool is_v = second(i);
#pragma unroll
          for (int v = 0; v < kVecs; ++v) {
            const int row = v * kRowsAt + cw * kOwn + lane / kVecs;
            const uint32_t in[4] = {x[v].x, x[v].y, x[v].z, x[v].w};
            uint32_t out[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              out[e] = kIsBf16 && !is_v ? quant::pair_of<true>(in[e >> 1], (e & 1) != 0) : quant::pair_of<false>(in[e >> 1], (e & 1) != 0);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int chunk = lane % kVecs * 2 + h;
              ptx::st_shared_v4(to + (chunk >> 3) * S::kHalfBytes + row * 128 + (((chunk & 7) ^ (row & 7)) << 4), out[4 * h], out[4 * h + 1], out[4 * h + 2], out[4 * h + 3]);
            }
          }
          if (!is_v) {
            // the steps of this tile go where those of the tile before the last were, once the query tiles that took part in that have read them
            const int j = (i + 1) / 2, place = (idx0 / 2 + j) & 1;
#pragma unroll
            for (int g = 0; g < 2; ++g)
              if (ok && uses[g][place] > 0) ok = __all_sync(0xffffffffu, ptx::mbar_wait(&bars->steps_free[g][place], (uses[g][place] - 1) & 1u, abort_flag, p.status, 175));
            if (!ok) break;
            uses[0][place] += j < w.n_a ? 1 : 0, uses[1][place] += w.lone ? 0 : 1;
            float* steps = reinterpret_cast<float*>(smem + S::kStepsOff + place * S::kStepBytes);
            const float top = softmax::warp_max(v_now);
            steps[my_row] = k_now, steps[kKeys + my_row] = v_now;
            if (lane == 0) steps[2 * kKeys + cw] = top;
          }
          ptx::fence_proxy_async_smem();
          ptx::mbar_arrive(&bars->kv_full[slot]);
        }
        idx0 += total;
        give();
      }
    }
  } else {
    // ------------------------------ softmax / output ---------------------------
    ptx::setmaxnreg_inc<S::kRegsSoftmax>();
    const int g = warp >> 2;                // 0: tile A, 1: tile B
    const int quad = warp & 3;              // TMEM lanes this warp may touch
    const int r = quad * 32 + lane;         // row inside the tile == TMEM lane
    const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t ts = tmem_s + g * 128 + lane_base, to = tmem_o + g * 128 + lane_base;
    const float sl2 = p.scale_log2;
    const uint32_t p_row = ptx::smem_u32(smem_p) + g * S::kPBytes + r * 128;
    const int r_token = r / p.group, r_head = r - r_token * p.group;
    int before = 0, steps_before = 0;       // this tile's steps in earlier segments, and the block's
    bool alive = true;
    while (alive && take()) {
      const Work& w = bars->plan[part_no % kPlans];
      const int n_g = g == 0 ? w.n_a : w.lone ? 0 : w.n;
      const int token = w.token0 + g * p.tokens + r_token;
      const bool row_ok = r_token < p.tokens && token < w.count;
      const bool idle = __all_sync(0xffffffffu, !row_ok);           // no row of this warp exists
      const int limit = kKeysSeen == kAll || kKeysSeen == kShared ? w.len - 1 : w.len - w.count + min(token, w.count - 1);  // last visible position
      float m_used = -INFINITY, l = 0.f;
      int v_used = 0;  // probabilities and their sum are 2^-v_used of what they were
      for (int j = 0; j < n_g; ++j) {
        const int c = before + j;
        bool ready = ptx::mbar_wait(&bars->s_full[g], c & 1u, abort_flag, p.status, 165 + g);
        if (!__all_sync(0xffffffffu, ready)) {
          alive = false;
          break;
        }
        ptx::tcgen05_fence_after_thread_sync();
        if (idle) {  // its probabilities may be anything, but it hands them over in step with the others
          ptx::tcgen05_fence_before_thread_sync();
          ptx::mbar_arrive(&bars->s_free[g]);
          if constexpr (kI8) ptx::mbar_arrive(&bars->steps_free[g][(steps_before + j) & 1]);
          if (j > 0 && !__all_sync(0xffffffffu, ptx::mbar_wait(&bars->pv_done[g], (c - 1) & 1u, abort_flag, p.status, 169 + g))) {
            alive = false;
            break;
          }
          ptx::mbar_arrive(&bars->p_ready[g]);
          continue;
        }
        const int col0 = (w.begin + j) * kKeys;
        const bool masked = col0 + kKeys - 1 > limit;
        uint32_t v[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) ptx::tmem_ld_32x32b_x32(ts + q * 32, v[q]);
        ptx::tmem_ld_wait();
        // the scores are in registers: S_g goes back to the tensor core for the next step's Q K^T
        ptx::tcgen05_fence_before_thread_sync();
        ptx::mbar_arrive(&bars->s_free[g]);
        const int place = (steps_before + j) & 1;
        const uint32_t steps = ptx::smem_u32(smem + S::kStepsOff) + place * S::kStepBytes;
        int v_new = 0;  // the exponent of the largest step of V
        if constexpr (kI8) {
#pragma unroll
          for (int i = 0; i < 128; i += 4) {
            float f[4];
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]) : "r"(steps + i * 4));
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i >> 5][(i & 31) + e] = __float_as_uint(__uint_as_float(v[i >> 5][(i & 31) + e]) * f[e]);
          }
          float f[4];
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3]) : "r"(steps + 2 * kKeys * 4));
          const float top = fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
          // from -80 on: l, which 2^-v_used multiplies, stays finite over 2^31 keys whose V is 0
          v_new = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -80), 100);
        }

        float mx = -INFINITY;
        if (masked) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (col0 + q * 32 + i > limit) v[q][i] = 0xff800000u;  // -inf
              mx = ptx::fmax_nan(mx, __uint_as_float(v[q][i]));
            }
        } else {
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 32; i += 2) mx4[(i >> 1) & 3] = ptx::fmax3_nan(mx4[(i >> 1) & 3], __uint_as_float(v[q][i]), __uint_as_float(v[q][i + 1]));
          mx = ptx::fmax_nan(ptx::fmax_nan(mx4[0], mx4[1]), ptx::fmax_nan(mx4[2], mx4[3]));
        }
        const float m_new = fmaxf(m_used, mx);
        if (j == 0) {
          m_used = m_new;
          v_used = v_new;
        } else {
          const bool grown = kI8 && v_new > v_used;  // alike in all threads of the tile
          const bool need = (m_new - m_used) * sl2 > kLag<kI8> || grown;
          if (__any_sync(0xffffffffu, need)) {
            // O_g is rescaled in place once the P V of the step before has retired
            ready = ptx::mbar_wait(&bars->pv_done[g], (c - 1) & 1u, abort_flag, p.status, 167 + g);
            if (!__all_sync(0xffffffffu, ready)) {
              alive = false;
              break;
            }
            ptx::tcgen05_fence_after_thread_sync();
            // a row of no scores so far has nothing to lose
            const float alpha = need ? ptx::ex2_approx((m_new == -INFINITY ? 0.f : (m_used - m_new) * sl2) + static_cast<float>(grown ? v_used - v_new : 0)) : 1.0f;
            if (need) m_used = m_new;
            if (grown) v_used = v_new;
            l *= alpha;
#pragma unroll 1
            for (int q = 0; q < D / 32; ++q) {
              uint32_t ov[32];
              ptx::tmem_ld_32x32b_x32(to + q * 32, ov);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
              ptx::tmem_st_32x32b_x32(to + q * 32, ov);
            }
            ptx::tmem_st_wait();
            ptx::tcgen05_fence_before_thread_sync();
          }
        }

        // probabilities: exp2, rounded to 16 bits, in the K-major layout of the P V product; of every 8 pairs attn::kPolyPairs avoid MUFU.  A row
        // whose scores so far are all -inf takes them against 0, one with a NaN or +inf among them against NaN (attention_tc.cuh).
        const float ms = (mx != mx || m_used == INFINITY ? NAN : m_used == -INFINITY ? 0.f : m_used * sl2) + (static_cast<float>(v_used) - kRaised<kI8, kPvBf16>);
        const ptx::f32x2_t sl2x2 = ptx::pack_f32x2(sl2, sl2);
        const ptx::f32x2_t nmsx2 = ptx::pack_f32x2(-ms, -ms);
        ptx::f32x2_t lsum[2] = {0ull, 0ull};
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int q = h2 * 2 + (i >> 4), e0 = (i & 15) * 2;
            const ptx::f32x2_t t2 = ptx::fma_f32x2(ptx::pack_f32x2(__uint_as_float(v[q][e0]), __uint_as_float(v[q][e0 + 1])), sl2x2, nmsx2);
            float p0, p1;
            if ((i & 7) < attn::kPolyPairs) {
              ptx::exp2_poly_x2(t2, p0, p1);
            } else {
              float t0, t1;
              ptx::unpack_f32x2(t2, t0, t1);
              p0 = ptx::ex2_approx(t0);
              p1 = ptx::ex2_approx(t1);
            }
            lsum[i & 1] = ptx::add_f32x2(lsum[i & 1], ptx::pack_f32x2(p0, p1));
            if constexpr (kI8) {
              float f0, f1;
              asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(f0), "=f"(f1) : "r"(steps + (kKeys + q * 32 + e0) * 4));
              p0 *= f0, p1 *= f1;
            }
            pk[i] = attn::pack16x2<kPvBf16>(p0, p1);
          }
          if (h2 == 0 && j > 0) {  // P_g is free once the P V of the step before has read it
            ready = ptx::mbar_wait(&bars->pv_done[g], (c - 1) & 1u, abort_flag, p.status, 169 + g);
            if (!__all_sync(0xffffffffu, ready)) {
              alive = false;
              break;
            }
          }
          const uint32_t prow = p_row + h2 * S::kHalfBytes;
#pragma unroll
          for (int q = 0; q < 8; ++q) ptx::st_shared_v4(prow + ((q ^ (r & 7)) << 4), pk[4 * q], pk[4 * q + 1], pk[4 * q + 2], pk[4 * q + 3]);
        }
        if (!alive) break;
        if constexpr (kI8) ptx::mbar_arrive(&bars->steps_free[g][place]);
        float l4[4];
        ptx::unpack_f32x2(lsum[0], l4[0], l4[1]);
        ptx::unpack_f32x2(lsum[1], l4[2], l4[3]);
        l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(&bars->p_ready[g]);
      }
      if (!alive) break;
      const bool whole = w.begin == 0 && w.n == w.steps;
      if (n_g > 0) {
        const bool ready = ptx::mbar_wait(&bars->pv_done[g], (before + n_g - 1) & 1u, abort_flag, p.status, 171 + g);
        if (!__all_sync(0xffffffffu, ready)) {
          alive = false;
          break;
        }
        ptx::tcgen05_fence_after_thread_sync();
      }
      if (!idle) {
        const int64_t rec = static_cast<int64_t>(blockIdx.x) * 2 + (w.begin == 0 ? 1 : 0);
        [[maybe_unused]] const float inv = m_used == -INFINITY ? NAN : 1.0f / l;  // all scores -inf (or NaN): softmax is NaN there
        const int64_t row = static_cast<int64_t>(w.first + token) * p.heads_q + w.head * p.group + r_head;
        [[maybe_unused]] uint16_t* orow = o + row * D;
        [[maybe_unused]] float* record = nullptr;
        if constexpr (leaves_records(kKeysSeen))
          record = whole ? p.records.whole + (row_ok ? row : 0) * kRecord<D> : p.records.part + (rec * 256 + g * kTileRows + r) * kRecord<D>;
#pragma unroll 1
        for (int q = 0; q < D / 32; ++q) {
          uint32_t ov[32];
          if (n_g > 0) {
            ptx::tmem_ld_32x32b_x32(to + q * 32, ov);
            ptx::tmem_ld_wait();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = 0u;
          }
          if constexpr (leaves_records(kKeysSeen)) {
            if (row_ok) {
#pragma unroll
              for (int i = 0; i < 4; ++i) ptx::st_global_v8(record + q * 32 + i * 8, ov + i * 8);
            }
          } else if (whole) {
            if (row_ok) {
#pragma unroll
              for (int t = 0; t < 4; ++t) {
                uint4 x;
                x.x = attn::pack16x2<kIsBf16>(__uint_as_float(ov[8 * t + 0]) * inv, __uint_as_float(ov[8 * t + 1]) * inv);
                x.y = attn::pack16x2<kIsBf16>(__uint_as_float(ov[8 * t + 2]) * inv, __uint_as_float(ov[8 * t + 3]) * inv);
                x.z = attn::pack16x2<kIsBf16>(__uint_as_float(ov[8 * t + 4]) * inv, __uint_as_float(ov[8 * t + 5]) * inv);
                x.w = attn::pack16x2<kIsBf16>(__uint_as_float(ov[8 * t + 6]) * inv, __uint_as_float(ov[8 * t + 7]) * inv);
                reinterpret_cast<uint4*>(orow + q * 32)[t] = x;
              }
            }
          } else {
            float4* part = p.part + (rec * (D / 4) + q * 8) * 256 + g * kTileRows + r;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              part[i * 256] = make_float4(__uint_as_float(ov[4 * i]), __uint_as_float(ov[4 * i + 1]), __uint_as_float(ov[4 * i + 2]), __uint_as_float(ov[4 * i + 3]));
          }
        }
        if constexpr (leaves_records(kKeysSeen)) {
          if (row_ok)
            *reinterpret_cast<float2*>(record + D) =
                make_float2(n_g > 0 ? m_used * sl2 + static_cast<float>(v_used) - kRaised<kI8, kPvBf16> : -INFINITY, n_g > 0 ? l : 0.f);
        } else if (!whole) p.part_ml[rec * 256 + g * kTileRows + r] = make_float2(n_g > 0 ? m_used + static_cast<float>(v_used) / sl2 : -INFINITY, n_g > 0 ? l : 0.f);
      }
      if (n_g > 0) {
        ptx::tcgen05_fence_before_thread_sync();
        ptx::mbar_arrive(&bars->o_free[g]);
      }
      before += n_g;
      steps_before += w.n;
      give();
    }
  }

  // ------------------------------ teardown ------------------------------------
  if (*abort_flag != 0u) {
    const unsigned long long t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 1000000ull) {
    }
  }
  ptx::tcgen05_fence_before_thread_sync();
  __syncthreads();
  if (warp == 9) {
    ptx::tcgen05_fence_after_thread_sync();
    ptx::tmem_dealloc(tmem_base, 512);
  }
}

// The records of a block that several shares have a part of, in order: CTA (x, y) has the block that goes on behind share x and 16 of its columns, a thread a row.
template <bool kIsBf16, int D, Keys kKeysSeen = kPast>
__global__ void __launch_bounds__(256)
attention_paged_tc_merge_kernel(uint16_t* __restrict__ o, const __grid_constant__ Params p) {
  ptx::launch_dependents();
  ptx::wait_prior_grid();
  put_zeros<D, kKeysSeen>(o, p);
  const int4 mine = __ldcg(p.info + blockIdx.x);
  if (mine.y < 0) return;
  const int n = records_of(p.info);
  const int first = p.step.starts[mine.y], count = p.step.starts[mine.y + 1] - first;
  const int g = threadIdx.x >> 7, r = threadIdx.x & 127, r_token = r / p.group;
  const int token = (mine.w * 2 + g) * p.tokens + r_token;
  if (r_token >= p.tokens || token >= count) return;
  auto record = [&](int i) { return static_cast<int64_t>(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0); };
  float gm = -INFINITY;
  for (int i = 0; i < n; ++i) gm = fmaxf(gm, __ldcg(p.part_ml + record(i) * 256 + threadIdx.x).x);
  float acc[16], gl = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = 0.f;
#pragma unroll 2
  for (int i = 0; i < n; ++i) {
    const float2 ml = __ldcg(p.part_ml + record(i) * 256 + threadIdx.x);
    // a part without a visible key weighs 0; it is added all the same, because one of NaN scores has that maximum too
    const float f = ml.x == -INFINITY ? 0.f : ptx::ex2_approx((ml.x - gm) * p.scale_log2);
    gl = fmaf(f, ml.y, gl);
    const float4* part = p.part + (record(i) * (D / 4) + blockIdx.y * 4) * 256 + threadIdx.x;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 x = __ldcg(part + q * 256);
      acc[4 * q] = fmaf(f, x.x, acc[4 * q]), acc[4 * q + 1] = fmaf(f, x.y, acc[4 * q + 1]);
      acc[4 * q + 2] = fmaf(f, x.z, acc[4 * q + 2]), acc[4 * q + 3] = fmaf(f, x.w, acc[4 * q + 3]);
    }
  }
  const float inv = 1.0f / gl;
  uint16_t* orow = o + (static_cast<int64_t>(first + token) * p.heads_q + mine.z * p.group + (r - r_token * p.group)) * D + blockIdx.y * 16;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint4 x;
    x.x = attn::pack16x2<kIsBf16>(acc[8 * h] * inv, acc[8 * h + 1] * inv), x.y = attn::pack16x2<kIsBf16>(acc[8 * h + 2] * inv, acc[8 * h + 3] * inv);
    x.z = attn::pack16x2<kIsBf16>(acc[8 * h + 4] * inv, acc[8 * h + 5] * inv), x.w = attn::pack16x2<kIsBf16>(acc[8 * h + 6] * inv, acc[8 * h + 7] * inv);
    *reinterpret_cast<uint4*>(orow + 8 * h) = x;
  }
}

}  // namespace tc
}  // namespace paged
}  // namespace tsm100
