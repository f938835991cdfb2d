// Eviction from a paged KV cache by accumulated attention weight, sm_100a.
//
// Per (sequence, KV head) with n > budget tokens: the newest `recent` stay, and of the others the
// budget - recent of the largest weight (NaN above all numbers, ties to the lowest index).  What stays keeps its
// order and moves to slots 0 .. budget - 1 of the sequence's own pages; its weights move along and the freed
// slots' weights become 0.  Sequences of at most `budget` tokens are left as they are.
//
// Two launches.  The selection: one CTA, or one thread-block cluster for long caches, per (sequence, KV head).  The
// weights' order-preserving 32-bit keys are counted into 2048 bins by their first 11 bits; the bin of the last
// key kept is found, its keys set apart, and the other 11 and 10 bits found among those; then the kept tokens are
// numbered in order and listed.  Bound by instructions and latency (128 selections of 4096 from 16K tokens:
// 15 us, 58 % of the issue slots); in a cluster the CTAs add their few used bins to the first one's by
// distributed-shared-memory atomics, integers, so the order does not matter.  Where the bin holds few keys (short
// caches), each is compared with the others instead of two more digits.
//
// The move: bound by HBM, 2 x the kept rows (48 sequences of 16K -> 4096, D = 128, fp16: 1.65 GB in 305 us, selection
// included).  In place, and the list is ascending with list[p] >= p: a row's
// destination is at or before its source.  One CTA moves one column slice of K (or V) of one (sequence, KV
// head), chunk by chunk in list order; a chunk is written only after it and all earlier chunks were read, and a
// chunk's writes end below the next chunk's first source, so reading ahead is free.  Slices make enough CTAs for
// few sequences.  The chunks before the first gap are not touched.  Two chunks of 32 KB in flight in each of three CTAs
// per SM (three in each of two: 92 us instead of 90 us for 16 sequences, 331 us instead of 343 us for 4 of 100000 ->
// 50000; 16 KB chunks: 99 to 135 us).  (One launch,
// with a cluster per (sequence, KV head) that selects and then moves, was 5 us slower for one sequence -- a cluster's
// barriers -- and no faster for many.)
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "device_common.cuh"
#include "kernels.h"

namespace fqkv {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;

// Larger weight, larger key; -0 as +0; every NaN above +inf.  No weight has the key 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (isnan(w)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint32_t ld_dsmem_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void red_dsmem_add(uint32_t addr, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Inclusive sum over the block in thread order; every thread also gets the total.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += u;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  // every warp scans the 32 warps' sums
  static_assert(kSelThreads == 1024, "one lane per warp");
  uint32_t all = warp_sums[lane];
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, all, off);
    if (lane >= off) all += u;
  }
  const uint32_t before = warp ? __shfl_sync(0xffffffffu, all, warp - 1) : 0u;
  all = __shfl_sync(0xffffffffu, all, 31);
  __syncthreads();  // warp_sums may be written again
  *total = all;
  return before + v;
}

constexpr int kMost = 16 * kSelThreads;         // tokens of a step; a slice of one step stays in registers
constexpr int kCand = 4096;                     // keys that share the first digit and fit in shared memory

constexpr int kRanked = 256;                    // and so few that each is compared with every other

struct SelectShared {
  uint32_t hist[2][kBins];  // the next digit's bins are cleared while this one's are in use; then a step's part of the list
  alignas(16) uint32_t cand[kCand];
  uint32_t warp_sums[kSelThreads / 32];
  uint32_t sel[2];          // the digit chosen, and how many keys lie in the bins above it
  uint32_t cands, larger;   // this slice's keys in the first digit's bin, and above it
  uint32_t counts[2];
};

// One slice is read three times: for the first digit's bins, to pick out the keys in the bin chosen (the two other
// digits then look at those alone, unless there are more than kCand of them), and for the list.
// kMine: consecutive tokens of one thread per step (4 where a slice has no more than 4096: the selection and move of one
// sequence of 2112 tokens take 12.2 us, with 16 tokens per thread 15.8 us).
template <int kMine, bool kOneStep>
__device__ void select_tokens(const PagedEvict& a, const float* w, int* list, int rank, int s0, int s1, int k,
                              SelectShared& sm) {
  constexpr int kStep = kMine * kSelThreads;
  const int C = a.cluster, tid = threadIdx.x, lane = tid & 31;
  // f(this thread's first token, its keys) for every step; every thread takes part in every step.  Tokens past the
  // slice have key 0, below every weight's (a key of 0 would be a NaN with the sign bit, and those are mapped away).
  auto fetch = [&](int i0, uint32_t (&key)[kMine]) {
#pragma unroll
    for (int q = 0; q < kMine; q += 4) {  // a row of weights is whole 16-byte pieces
      const float4 x = i0 + q < s1 ? *reinterpret_cast<const float4*>(w + i0 + q) : make_float4(0.f, 0.f, 0.f, 0.f);
      key[q] = weight_key(x.x);
      key[q + 1] = weight_key(x.y);
      key[q + 2] = weight_key(x.z);
      key[q + 3] = weight_key(x.w);
    }
    if (i0 + kMine > s1) {
#pragma unroll
      for (int q = 0; q < kMine; ++q)
        if (i0 + q >= s1) key[q] = 0u;
    }
  };
  uint32_t cached[kOneStep ? kMine : 1];
  if constexpr (kOneStep) fetch(s0 + kMine * tid, cached);
  auto steps = [&](auto&& f) {
    if constexpr (kOneStep) {
      f(s0 + kMine * tid, cached);
    } else {
      for (int c0 = s0; c0 < s1; c0 += kStep) {
        uint32_t key[kMine];
        fetch(c0 + kMine * tid, key);
        f(c0 + kMine * tid, key);
      }
    }
  };

  // ---- the smallest key kept, digit by digit
  uint32_t prefix = 0, mask = 0, need = uint32_t(k);
  for (int i = tid; i < kBins; i += kSelThreads) sm.hist[0][i] = 0;
  if (tid == 0) sm.cands = sm.larger = 0;
  if (C > 1) cluster_sync_all();
  else __syncthreads();
  bool few = false;  // the keys in the first digit's bin are in sm.cand
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const uint32_t digit = pass == 2 ? 1023u : 2047u;
    uint32_t* hist = sm.hist[pass & 1];
    if (few) {
      for (int i = tid; i < int(sm.cands); i += kSelThreads) {
        const uint32_t key = sm.cand[i];
        if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & digit], 1u);
      }
    } else {
      steps([&](int, const uint32_t(&key)[kMine]) {
#pragma unroll
        for (int q = 0; q < kMine; ++q)
          if (key[q] != 0u && (key[q] & mask) == prefix) atomicAdd(&hist[(key[q] >> shift) & digit], 1u);
      });
    }
    for (int i = tid; i < kBins; i += kSelThreads) sm.hist[(pass + 1) & 1][i] = 0;
    __syncthreads();
    if (C > 1) {  // the first CTA gets the others' counts: few of the bins are in use
      if (rank != 0)
        for (int i = tid; i < kBins; i += kSelThreads)
          if (hist[i]) red_dsmem_add(dsmem_addr(smem_u32(&hist[i]), 0), hist[i]);
      cluster_sync_all();
    }
    if (rank == 0) {
      // thread tid: bins 2047 - 2 tid and 2046 - 2 tid
      const uint32_t hi = hist[kBins - 1 - 2 * tid], lo = hist[kBins - 2 - 2 * tid];
      uint32_t total;
      const uint32_t above = block_scan(hi + lo, sm.warp_sums, &total) - hi - lo;
      if (above < need && need <= above + hi + lo) {
        const bool first = need <= above + hi;
        sm.sel[0] = uint32_t(kBins - (first ? 1 : 2) - 2 * tid);
        sm.sel[1] = first ? above : above + hi;
      }
    }
    uint32_t bin, over;
    if (C > 1) {
      cluster_sync_all();
      bin = ld_dsmem_u32(dsmem_addr(smem_u32(&sm.sel[0]), 0));
      over = ld_dsmem_u32(dsmem_addr(smem_u32(&sm.sel[1]), 0));
    } else {
      __syncthreads();
      bin = sm.sel[0];
      over = sm.sel[1];
    }
    // sel is set again behind the next pass's barriers, which every reader has to reach first
    need -= over;
    prefix |= bin << shift;
    mask |= digit << shift;
    if (pass == 0) {
      steps([&](int, const uint32_t(&key)[kMine]) {
        uint32_t mine = 0, above = 0;
#pragma unroll
        for (int q = 0; q < kMine; ++q) {
          mine += (key[q] >> 21) == bin && key[q] != 0u;
          above += (key[q] >> 21) > bin;
        }
        above = __reduce_add_sync(0xffffffffu, above);
        uint32_t incl = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const uint32_t u = __shfl_up_sync(0xffffffffu, incl, off);
          if (lane >= off) incl += u;
        }
        uint32_t at = 0;
        if (lane == 31) {
          atomicAdd(&sm.larger, above);
          at = atomicAdd(&sm.cands, incl);
        }
        at = __shfl_sync(0xffffffffu, at, 31) + incl - mine;
#pragma unroll
        for (int q = 0; q < kMine; ++q)
          if ((key[q] >> 21) == bin && key[q] != 0u) {
            if (at < kCand) sm.cand[at] = key[q];
            ++at;
          }
      });
      __syncthreads();
      few = sm.cands <= kCand;
      if (C == 1 && sm.cands <= kRanked) {
        // Every key of the bin finds its own place (one sequence of 2112 tokens: 26 keys, 0.4 us instead of 2 us for the
        // two other digits).
        const int cands = int(sm.cands);
        if (tid < cands) {
          const uint32_t key = sm.cand[tid];
          uint32_t gt = 0, ge = 0;
          int i = 0;
          for (; i + 4 <= cands; i += 4) {
            const uint4 o = *reinterpret_cast<const uint4*>(&sm.cand[i]);
            gt += (o.x > key) + (o.y > key) + (o.z > key) + (o.w > key);
            ge += (o.x >= key) + (o.y >= key) + (o.z >= key) + (o.w >= key);
          }
          for (; i < cands; ++i) {
            gt += sm.cand[i] > key;
            ge += sm.cand[i] >= key;
          }
          if (gt < need && need <= ge) {  // all threads with this key write the same
            sm.sel[0] = key;
            sm.sel[1] = gt;
          }
        }
        __syncthreads();
        prefix = sm.sel[0];
        need -= sm.sel[1];
        break;
      }
    }
  }

  // ---- numbers of larger and equal keys in the slices before this CTA's
  uint32_t gt_before = 0, eq_before = 0;
  if (C > 1) {
    uint32_t gt = 0, eq = 0;
    if (few) {
      for (int i = tid; i < int(sm.cands); i += kSelThreads) {
        gt += sm.cand[i] > prefix;
        eq += sm.cand[i] == prefix;
      }
    } else {
      steps([&](int, const uint32_t(&key)[kMine]) {
#pragma unroll
        for (int q = 0; q < kMine; ++q) {
          gt += (key[q] >> 21) == (prefix >> 21) && key[q] > prefix;
          eq += key[q] == prefix;
        }
      });
    }
    uint32_t tot_gt, tot_eq;
    block_scan(gt, sm.warp_sums, &tot_gt);
    block_scan(eq, sm.warp_sums, &tot_eq);
    if (tid == 0) {
      sm.counts[0] = sm.larger + tot_gt;
      sm.counts[1] = tot_eq;
    }
    cluster_sync_all();
    for (int r = 0; r < rank; ++r) {
      gt_before += ld_dsmem_u32(dsmem_addr(smem_u32(&sm.counts[0]), r));
      eq_before += ld_dsmem_u32(dsmem_addr(smem_u32(&sm.counts[1]), r));
    }
    cluster_sync_all();  // no CTA leaves while its counts are read
  }

  // ---- the list, in order (a step's counts: larger keys in the low half, equal ones in the high half, at most
  // 16384 each)
  steps([&](int i0, const uint32_t(&key)[kMine]) {
    uint32_t mine = 0;
#pragma unroll
    for (int q = 0; q < kMine; ++q) mine += (key[q] > prefix ? 1u : 0u) + (key[q] == prefix ? 0x10000u : 0u);
    uint32_t total;
    const uint32_t before = block_scan(mine, sm.warp_sums, &total) - mine;
    const uint32_t g = gt_before + (before & 0xffffu);
    uint32_t e = eq_before + (before >> 16);
    const uint32_t base = gt_before + min(eq_before, need);  // of this step in the list
    gt_before += total & 0xffffu;
    eq_before += total >> 16;
    const uint32_t kept = gt_before + min(eq_before, need) - base;
    // By way of shared memory, where it fits: a thread's few entries lie side by side, and stored from here each would be
    // a sector of its own (16 sequences of 0 to 16K: 89.4 against 90.3 us).
    int* stage = reinterpret_cast<int*>(sm.hist[0]);
    const bool staged = kept <= 2 * kBins;
    auto put = [&](int* to) {  // a thread's entries are one after the other
      uint32_t at = g + min(e, need) - base;
#pragma unroll
      for (int q = 0; q < kMine; ++q) {
        const bool is_eq = key[q] == prefix, take = key[q] > prefix || (is_eq && e < need);
        if (take) to[at] = i0 + q;
        at += take;
        e += is_eq;
      }
    };
    if (staged) put(stage);
    else put(list + base);
    if (staged) {
      __syncthreads();
      for (uint32_t i = tid; i < kept; i += kSelThreads) list[base + i] = stage[i];
      __syncthreads();  // the next step's entries come here too
    }
  });
}

// `a.cluster` CTAs per (sequence, KV head), one cluster.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const __grid_constant__ PagedEvict a) {
  __shared__ SelectShared sm;
  // The move is let in only when the selection is over: where both kernels of a call let their successor in at their
  // start, the next call's selection waits beside this one's move, and calls on end take 17.3 instead of 13.9 us (one
  // sequence of 2112 tokens).
  pdl_wait_primary();
  const int C = a.cluster;
  const int rank = int(blockIdx.x) % C, tid = threadIdx.x;
  const int unit = int(blockIdx.x) / C;
  const int n = max(0, min(a.kv.cap, a.kv.seq_lens[unit / a.kv.Hkv]));
  const bool over = n > a.budget;
  if (rank == 0 && tid == 0) a.state[unit] = make_int2(over ? 1 : 0, n);
  if (!over) return;  // the whole cluster
  int* list = a.list + size_t(unit) * a.budget;
  const int m = n - a.recent, k = a.budget - a.recent;  // keep k of the first m, and the rest
  for (int i = rank * kSelThreads + tid; i < a.recent; i += C * kSelThreads) list[k + i] = m + i;
  if (k == 0) return;  // the whole cluster
  const int per = ((m + C - 1) / C + 3) & ~3;
  const int s0 = min(m, rank * per), s1 = min(m, s0 + per);
  const float* w = a.weights + size_t(unit) * a.kv.cap;
  if (per <= 4 * kSelThreads) select_tokens<4, true>(a, w, list, rank, s0, s1, k, sm);
  else if (per <= kMost) select_tokens<16, true>(a, w, list, rank, s0, s1, k, sm);
  else select_tokens<16, false>(a, w, list, rank, s0, s1, k, sm);
}

// ------------------------------------------------------------------ the move
constexpr int kMoveThreads = 512;
constexpr int kMoveVecs = 4;                                // 16-byte pieces per thread and chunk
constexpr int kMoveStages = 2;                              // chunks in flight per CTA
constexpr int kChunkVecs = kMoveThreads * kMoveVecs;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// One column slice of one pool: v 16-byte pieces (2, 4, 8 or 16) of every row.  The lanes of a warp share v lanes per
// row, so each row's addresses are worked out by one lane (one or two rows per lane and chunk) and handed round:
// computing them in every lane took 140 instructions per warp and 512 bytes, 61 % of the issue slots.
// state.x: whether the sequence is over its budget; the first entries of the list (whatever they are, if not) are asked for
// before that is known, which takes a memory round trip off the start.
__device__ void move_rows(const PagedEvict& a, const int2& state, const int* list, const int* row, uint8_t* base,
                          int64_t page_stride, int64_t tok_stride, int v, uint4* ring) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = kChunkVecs / v, shift = 31 - __clz(v);
  const int chunks = (a.budget + rows - 1) / rows;
  const uint32_t my = smem_u32(ring) + tid * 16;
  const int col = 16 * (lane & (v - 1));
  // piece i of a thread belongs to row i * row_step + tid / v of the chunk; a warp has 128 / v rows, numbered
  // i * (32 / v) + lane / v; lane l looks after rows l and l + 32
  const int per = 32 >> shift, warp_rows = kMoveVecs * per, row_step = kMoveThreads >> shift;
  int mine[2];  // place in a chunk of this lane's rows; -1: none
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int s = lane + 32 * r;
    mine[r] = s < warp_rows ? (s / per) * row_step + warp * per + s % per : -1;
  }
  auto hand = [&](unsigned long long x0, unsigned long long x1, int i) -> unsigned long long {
    const int s = i * per + (lane >> shift);
    return __shfl_sync(0xffffffffu, v == 2 && i >= kMoveVecs / 2 ? x1 : x0, s & 31);
  };
  static_assert(kMoveVecs == 4, "v = 2: pieces 0 and 1 lie in rows 0 .. 31, 2 and 3 in rows 32 .. 63");
  // Two steps ahead of the fetch of a chunk its list entries are read, one step ahead its pages.
  int idx[2], page[2], off[2];
  auto read_list = [&](int c) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int p = c * rows + mine[r];
      idx[r] = mine[r] >= 0 && p < a.budget ? list[p] : -1;  // (past the last chunk too)
    }
  };
  auto read_pages = [&]() {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      page[r] = idx[r] < 0 ? 0 : row[a.kv.page_div.div(idx[r])];
      off[r] = idx[r] < 0 ? -1 : a.kv.page_div.mod(idx[r]);  // -1: no row
    }
  };
  // a row's address in the pool, 0 if its page is none of the pool's (recorded)
  auto address = [&](int pg, int o) -> unsigned long long {
    if (unsigned(pg) < unsigned(a.kv.num_pages))
      return reinterpret_cast<unsigned long long>(base + pg * page_stride + o * tok_stride);
    atomicCAS(a.status, kDevOk, kDevBadPage);
    return 0ull;
  };
  unsigned got = 0;  // which of this lane's rows of the chunks in flight were fetched, 2 bits per stage
  auto fetch = [&](int st) {
    got &= ~(3u << (2 * st));
    unsigned long long src[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      src[r] = off[r] >= 0 ? address(page[r], off[r]) : 0ull;
      if (src[r]) got |= 1u << (2 * st + r);
    }
#pragma unroll
    for (int i = 0; i < kMoveVecs; ++i) {
      const unsigned long long x = hand(src[0], src[1], i);
      if (x) cp_async16(my + (st * kChunkVecs + i * kMoveThreads) * 16, reinterpret_cast<const uint8_t*>(x) + col);
    }
    cp_async_commit();
  };
  const int mark = min(a.budget, (tid + 1) * rows) - 1, at_mark = tid < chunks ? list[mark] : -1;
  read_list(0);
  if (!state.x) return;
  // the first chunk with a row that moves: list[p] == p holds up to the first gap and nowhere after it
  int first = 0;
  for (int c0 = 0; c0 < chunks; c0 += kMoveThreads) {
    const int c = c0 + tid;
    const int last = min(a.budget, (c + 1) * rows) - 1;
    const int still = __syncthreads_count(c < chunks && (c0 == 0 ? at_mark : list[last]) == last);
    first += still;
    if (still < kMoveThreads) break;
  }
  if (first) read_list(first);
  read_pages();
  read_list(first + 1);
  for (int c = first; c < first + kMoveStages - 1; ++c) {
    fetch(c % kMoveStages);
    read_pages();
    read_list(c + 2);
  }
  for (int c = first; c < chunks; ++c) {
    const int st = c % kMoveStages;
    int to_page[2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      to_page[r] = (got >> (2 * st + r) & 1u) ? row[a.kv.page_div.div(c * rows + mine[r])] : 0;
    fetch((c + kMoveStages - 1) % kMoveStages);
    read_pages();
    read_list(c + kMoveStages + 1);
    cp_async_wait<kMoveStages - 1>();
    __syncthreads();  // the whole chunk (and all before it) is read: its destinations are free
    unsigned long long dst[2];
#pragma unroll
    for (int r = 0; r < 2; ++r)
      dst[r] = (got >> (2 * st + r) & 1u) ? address(to_page[r], a.kv.page_div.mod(c * rows + mine[r])) : 0ull;
#pragma unroll
    for (int i = 0; i < kMoveVecs; ++i) {
      const unsigned long long x = hand(dst[0], dst[1], i);
      if (x) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(x) + col) = ring[st * kChunkVecs + tid + i * kMoveThreads];
    }
  }
  cp_async_wait<0>();
}

// Page of position p, or -1 (recorded) when the table names none of the pool's.
__device__ __forceinline__ int page_at(const PagedEvict& a, const int* row, int p) {
  const int id = row[a.kv.page_div.div(p)];
  if (unsigned(id) < unsigned(a.kv.num_pages)) return id;
  atomicCAS(a.status, kDevOk, kDevBadPage);
  return -1;
}

// The scales and weights of one (sequence, KV head), by one CTA in list order: a step is read by all threads before
// any of it is written, and lands below the next step's sources.
__device__ void move_scalars(const PagedEvict& a, const int* list, int unit, int2 state) {
  constexpr int kVals = 4;
  const int n = state.y;
  const int tid = threadIdx.x, b = unit / a.kv.Hkv, kh = unit - b * a.kv.Hkv;
  const int* row = a.kv.table + int64_t(b) * a.kv.table_stride;
  const float* w = a.weights + size_t(unit) * a.kv.cap;
  float* wo = a.weights_out + size_t(unit) * a.kv.cap;
  if (!state.x) {
    if (wo != w)
      for (int i = tid; i < n; i += kMoveThreads) wo[i] = w[i];
    return;
  }
  for (int p0 = 0; p0 < a.budget; p0 += kVals * kMoveThreads) {
    int from[kVals];
    float x[kVals];
    __half ks[kVals], vs[kVals];
#pragma unroll
    for (int i = 0; i < kVals; ++i) {
      const int p = p0 + i * kMoveThreads + tid;
      from[i] = p < a.budget ? list[p] : -1;
    }
#pragma unroll
    for (int i = 0; i < kVals; ++i) x[i] = from[i] >= 0 ? w[from[i]] : 0.f;
    if (a.kv.int8) {
#pragma unroll
      for (int i = 0; i < kVals; ++i) {
        const int pg = from[i] >= 0 ? page_at(a, row, from[i]) : -1;
        if (pg >= 0) {
          ks[i] = a.kv.ks[pg * a.kv.ks_page + kh * a.kv.ks_head + a.kv.page_div.mod(from[i])];
          vs[i] = a.kv.vs[pg * a.kv.vs_page + kh * a.kv.vs_head + a.kv.page_div.mod(from[i])];
        } else {
          from[i] = -1;  // no scales
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kVals; ++i) {
      const int p = p0 + i * kMoveThreads + tid;
      if (p >= a.budget) continue;
      wo[p] = x[i];
      const int pg = a.kv.int8 && from[i] >= 0 ? page_at(a, row, p) : -1;
      if (pg >= 0) {
        a.kv.ks[pg * a.kv.ks_page + kh * a.kv.ks_head + a.kv.page_div.mod(p)] = ks[i];
        a.kv.vs[pg * a.kv.vs_page + kh * a.kv.vs_head + a.kv.page_div.mod(p)] = vs[i];
      }
    }
  }
  __syncthreads();  // in place: the last step's sources may lie behind the budget
  for (int p = a.budget + tid; p < n; p += kMoveThreads) wo[p] = 0.f;
}

// Blocks: 2 * slices per (sequence, KV head) for the rows, then one each for the rest, which fills the last wave.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ PagedEvict a) {
  extern __shared__ uint4 ring[];
  pdl_launch_dependents();
  pdl_wait_primary();
  const int jobs = 2 * a.slices, units = a.kv.B * a.kv.Hkv;
  const bool rest = int(blockIdx.x) >= units * jobs;
  const int unit = rest ? int(blockIdx.x) - units * jobs : int(blockIdx.x) / jobs;
  const int2 state = a.state[unit];
  const int* list = a.list + size_t(unit) * a.budget;
  const int b = unit / a.kv.Hkv, kh = unit - b * a.kv.Hkv;
  if (rest) {
    // (here, not in the selection: lens_out may be the lengths that its CTAs read)
    if (kh == 0 && threadIdx.x == 0) a.lens_out[b] = state.x ? a.budget : state.y;
    move_scalars(a, list, unit, state);
    return;
  }
  const int* row = a.kv.table + int64_t(b) * a.kv.table_stride;
  const int job = int(blockIdx.x) - unit * jobs;
  const bool is_v = job >= a.slices;
  const int elt = a.kv.int8 ? 1 : 2;
  const int width = a.kv.D * elt / a.slices;  // bytes
  const int col = (is_v ? job - a.slices : job) * width;
  uint8_t* base = static_cast<uint8_t*>(is_v ? a.kv.v : a.kv.k) + int64_t(kh) * (is_v ? a.kv.v_head : a.kv.k_head) * elt + col;
  move_rows(a, state, list, row, base, (is_v ? a.kv.v_page : a.kv.k_page) * elt, (is_v ? a.kv.v_tok : a.kv.k_tok) * elt,
            width / 16, ring);
}

constexpr size_t kMoveSmem = size_t(kMoveStages) * kChunkVecs * 16;

}  // namespace

cudaError_t evict_prepare() {
  return cudaFuncSetAttribute(evict_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kMoveSmem));
}

cudaError_t launch_evict_paged(const PagedEvict& args, cudaStream_t stream) {
  PagedEvict a = args;
  const int units = a.kv.B * a.kv.Hkv;
  // The move: column slices until about 600 CTAs exist, none narrower than 64 bytes (a DRAM access: 4 sequences of
  // 100000 -> 50000, 8 KV heads, D = 128: 4 slices of 64 bytes 343 us, 8 of 32 bytes 438 us); 32 bytes only where there
  // would not be a CTA per SM (one sequence of 16K -> 4096: 24 us in 64, 22 us in 128 CTAs).  16 sequences of 0 to
  // 16K -> 4096: 2 slices 93 us, 4 slices 90 us; 48 of 12K to 16K: 1 slice 305 us, 2 slices 315 us.
  a.slices = 1;
  const auto width = [&] { return a.kv.D * (a.kv.int8 ? 1 : 2) / a.slices; };
  while ((units * 2 * a.slices < 600 && width() > 64) || (units * 2 * a.slices < a.sms && width() > 32)) a.slices *= 2;
  // The selection: one CTA while a full sequence is about what it holds in registers (one step and a half, so that a
  // table with room to spare for 16K tokens does not pay a cluster's barriers: 22.1 us instead of 25.6 us for one such
  // sequence of 8 KV heads), then clusters of 2, 4 and 8, as long as every CTA has an SM to itself: 1 sequence of 48K ->
  // 12K 42 us in clusters of 2 and 57 us without, 16 of them 347 us and 322 us, 16 of 100K 737 us in 8 and 667 us without.
  a.cluster = 1;
  while (a.cluster < 8 && units * a.cluster * 2 <= a.sms && int64_t(a.cluster) * (kMost + kMost / 2) < a.kv.cap)
    a.cluster *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(units) * unsigned(a.cluster));
  cfg.blockDim = dim3(kSelThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(a.cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, evict_select_kernel, a);
  if (e != cudaSuccess) return e;
  return launch_pdl(evict_move_kernel, dim3((2 * a.slices + 1) * units), dim3(kMoveThreads), kMoveSmem, stream, a);
}

}  // namespace fqkv
