// pad_evict.cu -- eviction from a paged cache by accumulated attention weight:
// which slots survive (plan) and the copies that make them the first ones
// (move). No counterpart in the reference.
//
// Plan, for one (sequence, KV head) of L > budget slots: rank the slots by
//   (recent first, then weight descending with NaN above all, then slot
//   ascending)
// and keep the first `budget`. Holes are slots below `budget` that are not
// kept, movers are kept slots at or above it; there are equally many, and
// mover i (ascending) goes to hole i (ascending). Attention does not depend on
// the order of the slots, so nothing else has to move, and since sources lie
// at or above `budget` and targets below it, no row is both: the copies are
// free to run in any order.
//
// The ranking is a radix selection on an order-preserving 32-bit key, three
// digits of 11, 11 and 10 bits from the top, which leaves the key T of the
// budget-th slot and how many slots equal to T are kept (those of the lowest
// slots). Weights and positions are read once into shared memory; a pair whose
// slots fill more than one SM's share is spread over a cluster of up to 8 CTAs
// that add up their histograms through distributed shared memory.
//
// Bound: plan -- 8 bytes a slot would take 5 us for 4 x 8 x 118 thousand slots;
// the chain of a gather, three histogram passes, two or three sweeps and the
// exchanges in the cluster takes 41 us, issuing in 38% of the cycles and waiting
// for loads and barriers in the others. 64 x 2 x 2080 slots: 8 us, the latency of
// the same chain. Move -- 2 x row bytes a move: 131 thousand fp16 rows of 256 +
// 256 bytes in 33 us (62% of the copy rate), the rest the latency of its groups of
// loads and stores; a 4-bit row's 4-byte scales, weight and position each cost a
// 32-byte sector both ways, so its 39% of the copy rate over useful bytes is about
// two thirds over sectors.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>
#include <cstdlib>

#include "pad_b200.h"
#include "pad_error.cuh"

namespace {

namespace cg = cooperative_groups;
using pad::cuda_fail;
using pad::fail;

// 512 threads: two CTAs an SM, so that a cluster of 8 finds room.
constexpr int kPlanThreads = 512;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kGather = 8;  // slots of a thread whose loads are in flight together
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr uint32_t kRecentKey = 0xffffffffu, kNanKey = 0xfffffffeu;

struct PlanParams {
  const float* weights;
  const int32_t *slot_positions, *block_table, *seq_lens, *total_lens;
  int32_t *src, *dst, *counts, *new_lens;
  int64_t w1, p1;          // element strides of weights and slot_positions: heads,
  int w0, w2, p0, p2;      // pages and rows
  int64_t bt_stride;
  int hkv, num_pages, page_size, page_shift, max_pages, budget, recent, max_moves;
  int key_cap;  // keys of shared memory per CTA
  int quads;    // four neighbouring slots of a page are 16 aligned bytes
  int32_t* error_flags;
};

// Weight -> key whose unsigned order is the ranking (-0 and +0 are equal).
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return kNanKey;
  const uint32_t b = __float_as_uint(w + 0.f);  // -0 + 0 = +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

struct PlanShared {
  int hist[3][kBins];
  int scan[kPlanWarps];
  int bin, above, in_bin;  // the digit found in a pass, the keys above it and in it
  int eq, movers, holes;  // this CTA's counts, read by the cluster
};

// CACHED: every key lies in shared memory.
template <bool CACHED>
struct SlotKeys {
  const PlanParams& p;
  const uint32_t* cached;
  const float* weights;      // of this KV head
  const int32_t* positions;  // of this KV head, or null
  const int32_t* ids;        // page ids of this sequence
  int first;
  int64_t oldest_recent;     // slots whose position is at least this are recent
  __device__ __forceinline__ int page_slot(int slot) const {
    return p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
  }
  __device__ __forceinline__ const float* weight_at(int page, int row) const {
    return weights + ((int64_t)page * p.w0 + (int64_t)row * p.w2);
  }
  __device__ __forceinline__ const int32_t* position_at(int page, int row) const {
    return positions + ((int64_t)page * p.p0 + (int64_t)row * p.p2);
  }
  __device__ __forceinline__ uint32_t key(float w, int at) const {
    return positions != nullptr && at >= oldest_recent ? kRecentKey : weight_key(w);
  }
  // Slots past the shared-memory share are read again wherever they are needed;
  // those of a page that is none weigh least.
  __device__ __forceinline__ uint32_t at(int slot) const {
    const int i = slot - first;
    if (CACHED || i < p.key_cap) return cached[i];
    const int lp = page_slot(slot), page = __ldg(ids + lp), row = slot - lp * p.page_size;
    if ((unsigned)page >= (unsigned)p.num_pages) return 0u;
    return key(__ldg(weight_at(page, row)), positions != nullptr ? __ldg(position_at(page, row)) : 0);
  }
};

template <int RANKS>
__device__ __forceinline__ void rank_sync() {
  if constexpr (RANKS == 1) __syncthreads();
  else cg::this_cluster().sync();
}

// Largest bin d with (keys in bins above d) < need, searched by every CTA of the
// cluster for itself; a bin's count is summed over the cluster's histograms.
// Sets sh.bin and sh.above.
template <int RANKS>
__device__ __forceinline__ void find_bin(PlanShared& sh, int pass, int need) {
  constexpr int PER = kBins / kPlanThreads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int c[PER] = {}, sum = 0;
  const int top = kBins - PER * (tid + 1);  // thread t holds PER bins from the top
  static_assert(PER == 4, "a thread's bins are one 16-byte load");
  int4 part[RANKS];
#pragma unroll
  for (int r = 0; r < RANKS; ++r) {
    const PlanShared* o = RANKS == 1 ? &sh : cg::this_cluster().map_shared_rank(&sh, r);
    part[r] = *reinterpret_cast<const int4*>(&o->hist[pass][top]);
  }
#pragma unroll
  for (int r = 0; r < RANKS; ++r) {
    c[0] += part[r].w;
    c[1] += part[r].z;
    c[2] += part[r].y;
    c[3] += part[r].x;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) sum += c[i];
  int incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) sh.scan[warp] = incl;
  __syncthreads();
  int above = incl - sum;
#pragma unroll
  for (int x = 0; x < kPlanWarps; ++x) above += x < warp ? sh.scan[x] : 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (above < need && need <= above + c[i]) {
      sh.bin = kBins - 1 - (tid * PER + i);
      sh.above = above;
      sh.in_bin = c[i];
    }
    above += c[i];
  }
  __syncthreads();
}

// Exclusive sum over the block's warps of a per-warp count; *total its sum.
__device__ __forceinline__ int warp_base(PlanShared& sh, int mine, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (lane == 0) sh.scan[warp] = mine;
  __syncthreads();
  const int v = lane < kPlanWarps ? sh.scan[lane] : 0;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  *total = __shfl_sync(0xffffffffu, incl, 31);
  return __shfl_sync(0xffffffffu, incl - v, warp);
}

template <int RANKS, bool CACHED>
__global__ void __launch_bounds__(kPlanThreads, 2) evict_plan_kernel(const __grid_constant__ PlanParams p) {
  extern __shared__ __align__(16) uint32_t keys[];
  __shared__ __align__(16) PlanShared sh;
  const int rank = RANKS == 1 ? 0 : (int)cg::this_cluster().block_rank();
  const int pair = (int)(blockIdx.x / RANKS), b = pair / p.hkv, h = pair % p.hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t cap = (int64_t)p.max_pages * p.page_size;
  const int raw = __ldg(p.seq_lens + b);
  const int n = (int)min((int64_t)max(raw, 0), cap);
  if (raw != n && tid == 0 && rank == 0 && p.error_flags != nullptr) atomicOr(p.error_flags, PAD_FLAG_SEQ_LEN_RANGE);
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = min(n, p.budget);
  int32_t* src = p.src + (int64_t)pair * p.max_moves;
  int32_t* dst = p.dst + (int64_t)pair * p.max_moves;
  int count = 0;
  if (n > p.budget) {
    const int share = ((n + RANKS - 1) / RANKS + 3) / 4 * 4;  // whole quads of slots
    const int first = min(n, rank * share), last = min(n, first + share);
    const SlotKeys<CACHED> key{p,
                               keys,
                               p.weights + h * p.w1,
                               p.slot_positions != nullptr ? p.slot_positions + h * p.p1 : nullptr,
                               p.block_table + (int64_t)b * p.bt_stride,
                               first,
                               p.slot_positions != nullptr ? (int64_t)__ldg(p.total_lens + b) - p.recent : 0};
    for (int x = tid; x < 3 * kBins / 4; x += kPlanThreads)
      reinterpret_cast<int4*>(&sh.hist[0][0])[x] = make_int4(0, 0, 0, 0);
    __syncthreads();
    // keys into shared memory, their top digit counted on the way
    bool bad = false;
    const bool quads = CACHED && p.quads;
    // four neighbouring slots a load (4 x 8 x 118 thousand slots: 52.8 -> 41.3 us)
    constexpr int UQ = kGather / 4;
    for (int s0 = quads ? first : last; s0 < last; s0 += kPlanThreads * 4 * UQ) {
      int page[UQ], row[UQ];
      float4 w[UQ];
      int4 at[UQ];
#pragma unroll
      for (int u = 0; u < UQ; ++u) {
        const int s = s0 + (u * kPlanThreads + tid) * 4, lp = key.page_slot(s);
        row[u] = s - lp * p.page_size;
        page[u] = s < last ? __ldg(key.ids + lp) : -1;
      }
#pragma unroll
      for (int u = 0; u < UQ; ++u) {
        const bool ok = (unsigned)page[u] < (unsigned)p.num_pages;
        bad |= !ok && s0 + (u * kPlanThreads + tid) * 4 < last;
        w[u] = make_float4(0.f, 0.f, 0.f, 0.f);
        at[u] = make_int4(0, 0, 0, 0);
        if (ok) {
          w[u] = __ldg(reinterpret_cast<const float4*>(key.weight_at(page[u], row[u])));
          if (key.positions != nullptr) at[u] = __ldg(reinterpret_cast<const int4*>(key.position_at(page[u], row[u])));
        }
      }
#pragma unroll
      for (int u = 0; u < UQ; ++u) {
        const int s = s0 + (u * kPlanThreads + tid) * 4;
        if (s >= last) continue;
        uint32_t k[4] = {0u, 0u, 0u, 0u};
        if ((unsigned)page[u] < (unsigned)p.num_pages) {
          k[0] = key.key(w[u].x, at[u].x);
          k[1] = key.key(w[u].y, at[u].y);
          k[2] = key.key(w[u].z, at[u].z);
          k[3] = key.key(w[u].w, at[u].w);
        }
        *reinterpret_cast<uint4*>(keys + (s - first)) = make_uint4(k[0], k[1], k[2], k[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (s + j < last) atomicAdd(&sh.hist[0][k[j] >> 21], 1);
      }
    }
    // or one
    for (int s0 = quads ? last : first; s0 < last; s0 += kPlanThreads * kGather) {
      int page[kGather], row[kGather], at[kGather];
      float w[kGather];
#pragma unroll
      for (int u = 0; u < kGather; ++u) {
        const int s = s0 + u * kPlanThreads + tid;
        const int lp = key.page_slot(s);
        row[u] = s - lp * p.page_size;
        page[u] = s < last ? __ldg(key.ids + lp) : -1;
      }
#pragma unroll
      for (int u = 0; u < kGather; ++u) {
        const bool ok = (unsigned)page[u] < (unsigned)p.num_pages;
        bad |= !ok && s0 + u * kPlanThreads + tid < last;
        w[u] = 0.f;
        at[u] = 0;
        if (ok) {
          w[u] = __ldg(key.weight_at(page[u], row[u]));
          if (key.positions != nullptr) at[u] = __ldg(key.position_at(page[u], row[u]));
        }
      }
#pragma unroll
      for (int u = 0; u < kGather; ++u) {
        const int s = s0 + u * kPlanThreads + tid;
        const uint32_t k = (unsigned)page[u] < (unsigned)p.num_pages ? key.key(w[u], at[u]) : 0u;
        if (s < last) {
          if (CACHED || s - first < p.key_cap) keys[s - first] = k;
          atomicAdd(&sh.hist[0][k >> 21], 1);
        }
      }
    }
    if (bad && p.error_flags != nullptr) atomicOr(p.error_flags, PAD_FLAG_BAD_PAGE_ID);
    uint32_t prefix = 0;
    int need = p.budget;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      if (pass > 0) {
        auto count = [&](uint32_t k) {
          if (pass == 1 ? (k >> 21) == prefix : (k >> 10) == prefix)
            atomicAdd(&sh.hist[pass][pass == 1 ? (k >> 10) & 2047u : k & 1023u], 1);
        };
        if constexpr (CACHED) {
#pragma unroll 2
          for (int s = first + tid * 4; s < last; s += kPlanThreads * 4) {
            const uint4 k = *reinterpret_cast<const uint4*>(keys + (s - first));
            count(k.x);
            if (s + 1 < last) count(k.y);
            if (s + 2 < last) count(k.z);
            if (s + 3 < last) count(k.w);
          }
        } else {
#pragma unroll 4
          for (int s = first + tid; s < last; s += kPlanThreads) count(key.at(s));
        }
      }
      rank_sync<RANKS>();
      find_bin<RANKS>(sh, pass, need);
      need -= sh.above;
      prefix = pass == 0 ? (uint32_t)sh.bin : (prefix << (pass == 1 ? 11 : 10)) | (uint32_t)sh.bin;
    }
    // prefix is the key of the budget-th slot; `need` slots equal to it are kept
    const uint32_t T = prefix;
    // each warp walks a contiguous run of the CTA's slots
    const int per = ((last - first + kPlanWarps - 1) / kPlanWarps + 31) / 32 * 32;
    const int lo = min(last, first + warp * per), hi = min(last, lo + per);
    const uint32_t below = (1u << lane) - 1u;
    int eq_base = 0, total;
    const bool all_eq = sh.in_bin == need;  // every slot equal to T is kept: their order does not matter
    if (!all_eq) {
      int eq = 0;
#pragma unroll 4
      for (int s = lo + lane; s - lane < hi; s += 32) eq += __popc(__ballot_sync(0xffffffffu, s < hi && key.at(s) == T));
      eq_base = warp_base(sh, eq, &total);
      if constexpr (RANKS > 1)
        for (int r = 0; r < rank; ++r) eq_base += cg::this_cluster().map_shared_rank(&sh, r)->hist[2][T & 1023u];
    }
    // the slots kept of a run of 32, and the running number of equals before them
    auto kept = [&](int s, int& seen) -> uint32_t {
      const uint32_t k = s < hi ? key.at(s) : 0u;
      if (all_eq) return __ballot_sync(0xffffffffu, s < hi && k >= T);
      const uint32_t e = __ballot_sync(0xffffffffu, s < hi && k == T);
      const uint32_t on = __ballot_sync(0xffffffffu, s < hi && (k > T || (k == T && seen + __popc(e & below) < need)));
      seen += __popc(e);
      return on;
    };
    // Runs below the budget (those not kept are holes), the run across it, and
    // runs above it (those kept are movers).
    const int mid = lo + max(0, min(p.budget, hi) - lo) / 32 * 32;
    const int mid2 = mid < hi && mid < p.budget ? mid + 32 : mid;
    const uint32_t low = p.budget - mid >= 32 ? 0xffffffffu : (1u << max(0, p.budget - mid)) - 1u;  // of the run across
    int holes = 0, movers = 0, seen = eq_base;
#pragma unroll 4
    for (int s = lo + lane; s - lane < mid; s += 32) holes += 32 - __popc(kept(s, seen));
    if (mid2 > mid) {
      const uint32_t on = kept(mid + lane, seen), in = hi - mid >= 32 ? 0xffffffffu : (1u << (hi - mid)) - 1u;
      holes += __popc(~on & low & in);
      movers += __popc(on & ~low);
    }
#pragma unroll 4
    for (int s = mid2 + lane; s - lane < hi; s += 32) movers += __popc(kept(s, seen));
    int hole_at = warp_base(sh, holes, &total);
    if (tid == 0) sh.holes = total;
    int mover_at = warp_base(sh, movers, &total);
    if (tid == 0) sh.movers = total;
    rank_sync<RANKS>();
#pragma unroll
    for (int r = 0; r < RANKS; ++r) {
      const PlanShared* o = RANKS == 1 ? &sh : cg::this_cluster().map_shared_rank(&sh, r);
      const int oh = o->holes, om = o->movers;
      if (r < rank) {
        hole_at += oh;
        mover_at += om;
      }
      count += om;
    }
    seen = eq_base;
    // (never past max_moves unless the inputs change while the kernel runs)
    auto put = [&](int32_t* list, int& at, uint32_t on, int s) {
      const int i = at + __popc(on & below);
      if (((on >> lane) & 1u) && i < p.max_moves) list[i] = s;
      at += __popc(on);
    };
#pragma unroll 4
    for (int s = lo + lane; s - lane < mid; s += 32) put(dst, hole_at, ~kept(s, seen), s);
    if (mid2 > mid) {
      const uint32_t on = kept(mid + lane, seen), in = hi - mid >= 32 ? 0xffffffffu : (1u << (hi - mid)) - 1u;
      put(dst, hole_at, ~on & low & in, mid + lane);
      put(src, mover_at, on & ~low, mid + lane);
    }
#pragma unroll 4
    for (int s = mid2 + lane; s - lane < hi; s += 32) put(src, mover_at, kept(s, seen), s);
    if constexpr (RANKS > 1) cg::this_cluster().sync();  // no CTA leaves while another may read its shared memory
  }
  if (tid == 0 && rank == 0) p.counts[pair] = count;
  for (int x = count + rank * kPlanThreads + tid; x < p.max_moves; x += RANKS * kPlanThreads) {
    src[x] = -1;
    dst[x] = -1;
  }
}
// ----------------------------------------------------------------------------- move
constexpr int kMoveThreads = 256;
constexpr int kMaxCaches = 4;
constexpr int kMoveGrid = 148 * 8;  // every SM full; larger lists loop

struct MoveParams {
  uint8_t* cache[kMaxCaches];
  int64_t s0[kMaxCaches], s1[kMaxCaches], s2[kMaxCaches];  // page, row and head strides in bytes
  int chunks[kMaxCaches], unit_log2[kMaxCaches];           // a row is `chunks` pieces of 2^unit_log2 bytes
  float* weights;
  int32_t* slot_positions;
  const int32_t *block_table, *src, *dst, *counts;
  int64_t w0, w1, w2, p0, p1, p2, bt_stride;
  int64_t items;  // (pair, run of 32 moves) pieces of work
  int hkv, num_pages, page_size, page_shift, max_pages, max_moves, runs;
  int32_t* error_flags;
};

__device__ __forceinline__ uint4 load_piece(const uint8_t* x, int unit_log2) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (unit_log2 == 4) v = *reinterpret_cast<const uint4*>(x);
  else if (unit_log2 == 2) v.x = *reinterpret_cast<const uint32_t*>(x);
  else if (unit_log2 == 1) v.x = *reinterpret_cast<const uint16_t*>(x);
  else v.x = *x;
  return v;
}
__device__ __forceinline__ void store_piece(uint8_t* x, const uint4& v, int unit_log2) {
  if (unit_log2 == 4) *reinterpret_cast<uint4*>(x) = v;
  else if (unit_log2 == 2) *reinterpret_cast<uint32_t*>(x) = v.x;
  else if (unit_log2 == 1) *reinterpret_cast<uint16_t*>(x) = (uint16_t)v.x;
  else *x = (uint8_t)v.x;
}

// A warp takes up to 32 moves of one pair. Lane i looks up move i (slots, pages;
// its weight and position it copies itself), so that the chain of dependent loads
// is walked once for 32 moves; then LPM lanes copy each row, the addresses coming
// from move i's lane by shuffles, UN rounds of loads before their stores.
template <int LPM, int NC>
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const __grid_constant__ MoveParams p) {
  constexpr int MPR = 32 / LPM;           // moves of a round
  constexpr int UN = NC <= 2 ? 4 : 2;     // rounds in flight
  constexpr int ROUNDS = LPM;             // 32 / MPR
  static_assert(ROUNDS % UN == 0, "whole rounds");
  const int lane = threadIdx.x & 31, l = lane % LPM, mine = lane / LPM;
  const int64_t cap = (int64_t)p.max_pages * p.page_size;
  for (int64_t it = (int64_t)blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); it < p.items;
       it += (int64_t)gridDim.x * (kMoveThreads / 32)) {
    const int pair = (int)(it / p.runs), i0 = (int)(it - (int64_t)pair * p.runs) * 32;
    const int left = min(__ldg(p.counts + pair), p.max_moves) - i0;
    if (left <= 0) continue;
    const int b = pair / p.hkv, h = pair % p.hkv;
    // ---- this lane's move
    int sp = 0, dp = 0, sr = 0, dr = 0, bad = 0;
    bool ok = lane < left;
    if (ok) {
      const int64_t at = (int64_t)pair * p.max_moves + i0 + lane;
      const int ss = __ldg(p.src + at), ds = __ldg(p.dst + at);
      if (ss < 0 || ds < 0 || ss >= cap || ds >= cap) {
        bad = PAD_FLAG_SEQ_LEN_RANGE;
      } else {
        const int slp = p.page_shift >= 0 ? ss >> p.page_shift : ss / p.page_size;
        const int dlp = p.page_shift >= 0 ? ds >> p.page_shift : ds / p.page_size;
        sp = __ldg(p.block_table + b * p.bt_stride + slp);
        dp = __ldg(p.block_table + b * p.bt_stride + dlp);
        sr = ss - slp * p.page_size;
        dr = ds - dlp * p.page_size;
        if ((unsigned)sp >= (unsigned)p.num_pages || (unsigned)dp >= (unsigned)p.num_pages) bad = PAD_FLAG_BAD_PAGE_ID;
      }
      ok = bad == 0;
      if (bad != 0 && p.error_flags != nullptr) atomicOr(p.error_flags, bad);
    }
    float w = 0.f;
    int32_t pos = 0;
    if (ok && p.weights != nullptr) w = p.weights[sp * p.w0 + h * p.w1 + sr * p.w2];
    if (ok && p.slot_positions != nullptr) pos = p.slot_positions[sp * p.p0 + h * p.p1 + sr * p.p2];
    const uint32_t good = __ballot_sync(0xffffffffu, ok);
    // ---- the rows
#pragma unroll 1
    for (int r0 = 0; r0 < ROUNDS && r0 * MPR < left; r0 += UN) {
      uint4 v[UN][NC];
      int64_t to[UN][2];  // page and row of the target
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int m = (r0 + u) * MPR + mine;
        const int64_t fp = __shfl_sync(0xffffffffu, sp, m), fr = __shfl_sync(0xffffffffu, sr, m);
        to[u][0] = __shfl_sync(0xffffffffu, dp, m);
        to[u][1] = __shfl_sync(0xffffffffu, dr, m);
        if (!((good >> m) & 1u)) to[u][0] = -1;
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (to[u][0] >= 0 && l < p.chunks[c])
            v[u][c] = load_piece(p.cache[c] + fp * p.s0[c] + fr * p.s1[c] + h * p.s2[c] + ((int64_t)l << p.unit_log2[c]),
                                 p.unit_log2[c]);
      }
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int m = (r0 + u) * MPR + mine;
        const int64_t fp = __shfl_sync(0xffffffffu, sp, m), fr = __shfl_sync(0xffffffffu, sr, m);
        if (to[u][0] < 0) continue;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          uint8_t* row = p.cache[c] + to[u][0] * p.s0[c] + to[u][1] * p.s1[c] + h * p.s2[c];
          if (l < p.chunks[c]) store_piece(row + ((int64_t)l << p.unit_log2[c]), v[u][c], p.unit_log2[c]);
          // rows of more than LPM pieces
          for (int x = l + LPM; x < p.chunks[c]; x += LPM)
            store_piece(row + ((int64_t)x << p.unit_log2[c]),
                        load_piece(p.cache[c] + fp * p.s0[c] + fr * p.s1[c] + h * p.s2[c] + ((int64_t)x << p.unit_log2[c]),
                                   p.unit_log2[c]),
                        p.unit_log2[c]);
        }
      }
    }
    if (ok && p.weights != nullptr) p.weights[dp * p.w0 + h * p.w1 + dr * p.w2] = w;
    if (ok && p.slot_positions != nullptr) p.slot_positions[dp * p.p0 + h * p.p1 + dr * p.p2] = pos;
  }
}

int shift_of(int64_t page_size) {
  return (page_size & (page_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)page_size) : -1;
}

int check_common(const char* what, int64_t batch, int64_t num_kv_heads, int64_t num_pages, int64_t page_size,
                 int64_t max_pages, int64_t bt_stride) {
  if (batch < 0 || num_kv_heads <= 0 || num_pages < 0 || page_size <= 0 || max_pages < 0)
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: negative or zero size", what);
  if (bt_stride < max_pages)
    return fail(PAD_ERR_INVALID_ARGUMENT, "%s: block_table row stride smaller than its width", what);
  if (num_pages > INT32_MAX || page_size > INT32_MAX || max_pages > INT32_MAX ||
      max_pages * page_size > INT32_MAX / 2 || batch > INT32_MAX / num_kv_heads / kMaxCluster)
    return fail(PAD_ERR_UNSUPPORTED, "%s: sizes exceed 32-bit indexing", what);
  return PAD_OK;
}

constexpr int kMaxDevices = 64;

// Keys of shared memory a plan CTA may hold beside its static part.
constexpr int kKeyCapMax = (227 * 1024 - (int)sizeof(PlanShared) - 1024) / 4 / 256 * 256;

}  // namespace

extern "C" int pad_evict_max_moves(int64_t budget, int64_t page_size, int64_t max_pages_per_seq, int64_t* max_moves) {
  if (max_moves == nullptr) return fail(PAD_ERR_INVALID_ARGUMENT, "evict_plan: null output pointer");
  if (budget < 1 || page_size <= 0 || max_pages_per_seq < 0 || (max_pages_per_seq > 0 && page_size > INT64_MAX / max_pages_per_seq))
    return fail(PAD_ERR_INVALID_ARGUMENT, "evict_plan: budget and page_size must be positive");
  *max_moves = std::max<int64_t>(0, std::min(budget, max_pages_per_seq * page_size - budget));
  return PAD_OK;
}

extern "C" int pad_paged_kv_evict_plan(const float* weights, const int32_t* slot_positions, const int32_t* block_table,
                                       const int32_t* seq_lens, const int32_t* total_lens, int32_t* src, int32_t* dst,
                                       int32_t* counts, int32_t* new_lens, int64_t batch, int64_t num_kv_heads,
                                       int64_t num_pages, int64_t page_size, int64_t max_pages_per_seq, int64_t budget,
                                       int64_t recent, const int64_t* weight_strides, const int64_t* position_strides,
                                       int64_t block_table_stride, void* stream, int32_t* error_flags) {
  int st = check_common("evict_plan", batch, num_kv_heads, num_pages, page_size, max_pages_per_seq, block_table_stride);
  if (st != PAD_OK) return st;
  if (budget < 1) return fail(PAD_ERR_INVALID_ARGUMENT, "evict_plan: budget must be at least 1");
  if (recent < 0 || recent > budget)
    return fail(PAD_ERR_INVALID_ARGUMENT, "evict_plan: recent must lie in [0, budget]");
  // (a pool of nothing has no address: no slot of it is read)
  if (recent > 0 && slot_positions == nullptr && num_pages > 0)
    return fail(PAD_ERR_INVALID_ARGUMENT, "evict_plan: recent needs slot_positions");
  if (batch == 0) return PAD_OK;
  int64_t moves = 0;
  if ((st = pad_evict_max_moves(budget, page_size, max_pages_per_seq, &moves)) != PAD_OK) return st;
  if (seq_lens == nullptr || counts == nullptr || new_lens == nullptr ||
      (moves > 0 && ((weights == nullptr && num_pages > 0) || block_table == nullptr || src == nullptr ||
                     dst == nullptr || weight_strides == nullptr)) ||
      (slot_positions != nullptr && (total_lens == nullptr || position_strides == nullptr)))
    return fail(PAD_ERR_INVALID_ARGUMENT, "evict_plan: null pointer argument");
  const int64_t cap = max_pages_per_seq * page_size, pairs = batch * num_kv_heads;
  PlanParams p = {};
  p.weights = weights;
  // without a recent window the positions decide nothing
  p.slot_positions = recent > 0 ? slot_positions : nullptr;
  p.block_table = block_table;
  p.seq_lens = seq_lens;
  p.total_lens = total_lens;
  p.src = src;
  p.dst = dst;
  p.counts = counts;
  p.new_lens = new_lens;
  for (const int64_t* st2 : {weight_strides, p.slot_positions != nullptr ? position_strides : nullptr})
    if (st2 != nullptr && (std::abs(st2[0]) > INT32_MAX || std::abs(st2[2]) > INT32_MAX))
      return fail(PAD_ERR_UNSUPPORTED, "evict_plan: page and row strides must fit 32 bits");
  if (weight_strides != nullptr) {
    p.w0 = (int)weight_strides[0];
    p.w1 = weight_strides[1];
    p.w2 = (int)weight_strides[2];
  }
  if (p.slot_positions != nullptr) {
    p.p0 = (int)position_strides[0];
    p.p1 = position_strides[1];
    p.p2 = (int)position_strides[2];
  }
  p.bt_stride = block_table_stride;
  p.hkv = (int)num_kv_heads;
  p.num_pages = (int)num_pages;
  p.page_size = (int)page_size;
  p.page_shift = shift_of(page_size);
  p.max_pages = (int)max_pages_per_seq;
  auto quads = [&](const void* x, const int64_t* st4) {
    return st4[2] == 1 && st4[0] % 4 == 0 && st4[1] % 4 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  };
  p.quads = page_size % 4 == 0 && weight_strides != nullptr && quads(weights, weight_strides) &&
            (p.slot_positions == nullptr || quads(slot_positions, position_strides));
  p.budget = (int)std::min<int64_t>(budget, INT32_MAX);
  p.recent = (int)std::min<int64_t>(recent, INT32_MAX);
  p.max_moves = (int)moves;
  p.error_flags = error_flags;
  // a CTA per 8192 slots of a sequence, up to a cluster of 8
  int ranks = 1, lg = 0;
  while (ranks < kMaxCluster && cap > (int64_t)ranks * 8192) {
    ranks *= 2;
    ++lg;
  }
  static const void* const kernels[5] = {
      reinterpret_cast<const void*>(&evict_plan_kernel<1, true>), reinterpret_cast<const void*>(&evict_plan_kernel<2, true>),
      reinterpret_cast<const void*>(&evict_plan_kernel<4, true>), reinterpret_cast<const void*>(&evict_plan_kernel<8, true>),
      reinterpret_cast<const void*>(&evict_plan_kernel<8, false>)};
  const int64_t share = (cap + ranks - 1) / ranks;
  p.key_cap = (int)std::min<int64_t>(kKeyCapMax, (share + 255) / 256 * 256);
  if (share > p.key_cap) lg = 4;  // (then ranks is 8)
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  if (device < 0 || device >= kMaxDevices) return fail(PAD_ERR_INVALID_ARGUMENT, "device %d out of range", device);
  static std::atomic<bool> smem_set[kMaxDevices];  // set twice by racing threads at worst
  if (!smem_set[device].load()) {
    for (const void* k : kernels) {
      e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kKeyCapMax * 4);
      if (e != cudaSuccess) return cuda_fail(e, "configuring the evict_plan kernel");
    }
    smem_set[device].store(true);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(pairs * ranks));
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = (size_t)p.key_cap * 4;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {&p};
  e = cudaLaunchKernelExC(&cfg, kernels[lg], args);
  return e == cudaSuccess ? PAD_OK : cuda_fail(e, "launching the evict_plan kernel");
}

extern "C" int pad_paged_kv_move(int64_t num_caches, void* const* caches, const int64_t* row_bytes,
                                 const int64_t* cache_strides, const int32_t* block_table, const int32_t* src,
                                 const int32_t* dst, const int32_t* counts, float* weights, int32_t* slot_positions,
                                 int64_t batch, int64_t num_kv_heads, int64_t num_pages, int64_t page_size,
                                 int64_t max_pages_per_seq, int64_t max_moves, const int64_t* weight_strides,
                                 const int64_t* position_strides, int64_t block_table_stride, void* stream,
                                 int32_t* error_flags) {
  int st = check_common("kv_move", batch, num_kv_heads, num_pages, page_size, max_pages_per_seq, block_table_stride);
  if (st != PAD_OK) return st;
  if (num_caches < 1 || num_caches > kMaxCaches)
    return fail(PAD_ERR_INVALID_ARGUMENT, "kv_move: 1 to %d caches, not %lld", kMaxCaches, (long long)num_caches);
  if (max_moves < 0) return fail(PAD_ERR_INVALID_ARGUMENT, "kv_move: negative or zero size");
  if (max_moves > INT32_MAX) return fail(PAD_ERR_UNSUPPORTED, "kv_move: max_moves exceeds int32");
  if (batch == 0 || max_moves == 0 || num_pages == 0) return PAD_OK;
  if (caches == nullptr || row_bytes == nullptr || cache_strides == nullptr || block_table == nullptr ||
      src == nullptr || dst == nullptr || counts == nullptr || (weights != nullptr && weight_strides == nullptr) ||
      (slot_positions != nullptr && position_strides == nullptr))
    return fail(PAD_ERR_INVALID_ARGUMENT, "kv_move: null pointer argument");
  MoveParams p = {};
  int most = 1;
  for (int c = 0; c < num_caches; ++c) {
    if (caches[c] == nullptr) return fail(PAD_ERR_INVALID_ARGUMENT, "kv_move: null pointer argument");
    if (row_bytes[c] <= 0 || row_bytes[c] > INT32_MAX)
      return fail(PAD_ERR_INVALID_ARGUMENT, "kv_move: row of %lld bytes", (long long)row_bytes[c]);
    const int64_t* s = cache_strides + 3 * c;
    // the widest of 16, 4, 2 and 1 bytes that address and strides allow
    const uint64_t all = (uint64_t)reinterpret_cast<uintptr_t>(caches[c]) | (uint64_t)row_bytes[c] | (uint64_t)s[0] |
                         (uint64_t)s[1] | (uint64_t)s[2];
    p.unit_log2[c] = all % 16 == 0 ? 4 : all % 4 == 0 ? 2 : all % 2 == 0 ? 1 : 0;
    p.cache[c] = static_cast<uint8_t*>(caches[c]);
    p.s0[c] = s[0];
    p.s1[c] = s[1];
    p.s2[c] = s[2];
    p.chunks[c] = (int)(row_bytes[c] >> p.unit_log2[c]);
    most = std::max(most, p.chunks[c]);
  }
  p.weights = weights;
  p.slot_positions = slot_positions;
  p.block_table = block_table;
  p.src = src;
  p.dst = dst;
  p.counts = counts;
  if (weights != nullptr) {
    p.w0 = weight_strides[0];
    p.w1 = weight_strides[1];
    p.w2 = weight_strides[2];
  }
  if (slot_positions != nullptr) {
    p.p0 = position_strides[0];
    p.p1 = position_strides[1];
    p.p2 = position_strides[2];
  }
  p.bt_stride = block_table_stride;
  p.hkv = (int)num_kv_heads;
  p.num_pages = (int)num_pages;
  p.page_size = (int)page_size;
  p.page_shift = shift_of(page_size);
  p.max_pages = (int)max_pages_per_seq;
  p.max_moves = (int)max_moves;
  p.error_flags = error_flags;
  p.runs = (int)((max_moves + 31) / 32);
  p.items = batch * num_kv_heads * (int64_t)p.runs;
  const unsigned grid = (unsigned)std::min<int64_t>((p.items + kMoveThreads / 32 - 1) / (kMoveThreads / 32), kMoveGrid);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  // lanes per move: enough for the widest row's pieces, 16 at most (a 256-byte
  // row's 16 pieces; longer rows loop); two caches keep more rounds in flight
  const int lpm = most <= 4 ? 4 : 16;
  if (num_caches <= 2) {
    if (lpm == 4) kv_move_kernel<4, 2><<<grid, kMoveThreads, 0, s>>>(p);
    else kv_move_kernel<16, 2><<<grid, kMoveThreads, 0, s>>>(p);
  } else {
    if (lpm == 4) kv_move_kernel<4, 4><<<grid, kMoveThreads, 0, s>>>(p);
    else kv_move_kernel<16, 4><<<grid, kMoveThreads, 0, s>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PAD_OK : cuda_fail(e, "launching the kv_move kernel");
}
