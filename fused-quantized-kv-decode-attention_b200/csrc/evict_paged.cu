// Eviction from a paged KV cache by accumulated attention weight, sm_100a.
//
// Per (sequence, KV head) with n > budget tokens: the newest `recent` stay, and of the others the
// budget - recent of the largest weight (NaN above all numbers, ties to the lowest index).  What stays keeps its
// order and moves to slots 0 .. budget - 1 of the sequence's own pages; its weights move along and the freed
// slots' weights become 0.  Sequences of at most `budget` tokens are left as they are.
//
// Two launches.  The selection: one thread-block cluster per (sequence, KV head); every CTA counts its slice of
// the weights into 2048 bins of the order-preserving 32-bit key, the cluster adds the bins through
// distributed shared memory and narrows the key digit by digit (11, 11 and 10 bits) to the smallest one kept;
// a last pass numbers the kept tokens in order and writes their list.  Bound by latency: five passes over
// 4 bytes per token, from L2 after the first.
//
// The move: bound by HBM, 2 x the kept rows.  In place, and the list is ascending with list[p] >= p: a row's
// destination is at or before its source.  One CTA moves one column slice of K (or V) of one (sequence, KV
// head), chunk by chunk in list order; a chunk is written only after it and all earlier chunks were read, and a
// chunk's writes end below the next chunk's first source, so reading ahead is free.  Slices make enough CTAs for
// few sequences.  The chunks before the first gap are not touched.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "device_common.cuh"
#include "kernels.h"

namespace fqkv {
namespace {

constexpr int kSelThreads = 512;
constexpr int kBins = 2048;

// Larger weight, larger key; -0 as +0; every NaN above +inf.
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
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelThreads / 32; ++w) {
    const uint32_t s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  __syncthreads();  // warp_sums may be written again
  *total = all;
  return before + v;
}

// Cluster of gridDim-independent size `a.cluster` per (sequence, KV head).
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const __grid_constant__ PagedEvict a) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t warp_sums[kSelThreads / 32];
  __shared__ uint32_t sel_bin, sel_above, my_counts[2];
  pdl_launch_dependents();
  pdl_wait_primary();
  const int C = a.cluster;
  const int rank = int(blockIdx.x) % C;
  const int unit = int(blockIdx.x) / C;
  const int tid = threadIdx.x;
  const int n = max(0, min(a.kv.cap, a.kv.seq_lens[unit / a.kv.Hkv]));
  const bool over = n > a.budget;
  if (rank == 0 && tid == 0) a.state[unit] = make_int2(over ? 1 : 0, n);
  if (!over) return;  // the whole cluster

  const float* w = a.weights + size_t(unit) * a.kv.cap;
  int* list = a.list + size_t(unit) * a.budget;
  const int m = n - a.recent, k = a.budget - a.recent;  // keep k of the first m, and the rest
  for (int i = rank * kSelThreads + tid; i < a.recent; i += C * kSelThreads) list[k + i] = m + i;
  if (k == 0) return;  // the whole cluster

  const int per = ((m + C - 1) / C + 3) & ~3;
  const int s0 = min(m, rank * per), s1 = min(m, s0 + per);

  // ---- the smallest key kept, digit by digit
  uint32_t prefix = 0, mask = 0, need = uint32_t(k);
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
    const uint32_t digit = pass == 2 ? 1023u : 2047u;
    for (int i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = s0 + tid; i < s1; i += kSelThreads) {
      const uint32_t key = weight_key(w[i]);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & digit], 1u);
    }
    cluster_sync_all();
    // thread tid: bins 2047 - 4 tid down to 2044 - 4 tid, summed over the cluster
    constexpr int kPer = kBins / kSelThreads;
    uint32_t cnt[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int bin = kBins - 1 - (kPer * tid + i);
      uint32_t v = 0;
      for (int r = 0; r < C; ++r) v += ld_dsmem_u32(dsmem_addr(smem_u32(&hist[bin]), r));
      cnt[i] = v;
      sum += v;
    }
    uint32_t total;
    uint32_t above = block_scan(sum, warp_sums, &total) - sum;  // in the bins above this thread's
    if (above < need && need <= above + sum) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (above < need && need <= above + cnt[i]) {
          sel_bin = uint32_t(kBins - 1 - (kPer * tid + i));
          sel_above = above;
        }
        above += cnt[i];
      }
    }
    cluster_sync_all();  // sel_* are set; every CTA has read the bins
    need -= sel_above;
    prefix |= sel_bin << shift;
    mask |= digit << shift;
    __syncthreads();  // all have read sel_* before the next pass sets them
  }

  // ---- numbers of larger and equal keys in the slices before this CTA's
  uint32_t gt = 0, eq = 0;
  for (int i = s0 + tid; i < s1; i += kSelThreads) {
    const uint32_t key = weight_key(w[i]);
    gt += key > prefix;
    eq += key == prefix;
  }
  uint32_t tot_gt, tot_eq;
  block_scan(gt, warp_sums, &tot_gt);
  block_scan(eq, warp_sums, &tot_eq);
  if (tid == 0) {
    my_counts[0] = tot_gt;
    my_counts[1] = tot_eq;
  }
  cluster_sync_all();
  uint32_t gt_before = 0, eq_before = 0;
  for (int r = 0; r < rank; ++r) {
    gt_before += ld_dsmem_u32(dsmem_addr(smem_u32(&my_counts[0]), r));
    eq_before += ld_dsmem_u32(dsmem_addr(smem_u32(&my_counts[1]), r));
  }
  cluster_sync_all();  // no CTA leaves while its counts are read

  // ---- the list, in order: 4 consecutive tokens per thread and step
  for (int c0 = s0; c0 < s1; c0 += 4 * kSelThreads) {
    uint32_t key[4], mine = 0;  // equal keys in the high half, larger ones in the low half
    const int i0 = c0 + 4 * tid;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      key[i] = i0 + i < s1 ? weight_key(w[i0 + i]) : 0u;
      if (i0 + i < s1) mine += (key[i] > prefix ? 1u : 0u) + (key[i] == prefix ? 0x10000u : 0u);
    }
    uint32_t total;
    const uint32_t before = block_scan(mine, warp_sums, &total) - mine;
    uint32_t g = gt_before + (before & 0xffffu), e = eq_before + (before >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i0 + i >= s1) continue;
      const bool is_gt = key[i] > prefix, is_eq = key[i] == prefix;
      if (is_gt || (is_eq && e < need)) list[g + min(e, need)] = i0 + i;
      g += is_gt;
      e += is_eq;
    }
    gt_before += total & 0xffffu;
    eq_before += total >> 16;
  }
}

// ------------------------------------------------------------------ the move
constexpr int kMoveThreads = 256;
constexpr int kMoveVecs = 4;                                // 16-byte pieces per thread and chunk
constexpr int kMoveStages = 3;                              // chunks in flight per CTA
constexpr int kChunkVecs = kMoveThreads * kMoveVecs;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Page of position p, or -1 (recorded) when the table names none of the pool's.
__device__ __forceinline__ int page_at(const PagedEvict& a, const int* row, int p) {
  const int id = row[a.kv.page_div.div(p)];
  if (unsigned(id) < unsigned(a.kv.num_pages)) return id;
  atomicCAS(a.status, kDevOk, kDevBadPage);
  return -1;
}

// One column slice of one pool: v 16-byte pieces (a power of two) of every row.
__device__ void move_rows(const PagedEvict& a, const int* list, const int* row, uint8_t* base, int64_t page_stride,
                          int64_t tok_stride, int v, uint4* ring) {
  const int tid = threadIdx.x;
  const int rows = kChunkVecs / v, shift = 31 - __clz(v);
  const int chunks = (a.budget + rows - 1) / rows;
  // the first chunk with a row that moves: list[p] == p holds up to the first gap and nowhere after it
  int first = 0;
  for (int c0 = 0; c0 < chunks; c0 += kMoveThreads) {
    const int c = c0 + tid;
    const int last = min(a.budget, (c + 1) * rows) - 1;
    const int still = __syncthreads_count(c < chunks && list[last] == last);
    first += still;
    if (still < kMoveThreads) break;
  }
  const uint32_t my = smem_u32(ring) + tid * 16;
  auto at = [&](int p, int col) -> uint8_t* {
    const int pg = page_at(a, row, p);
    return pg < 0 ? nullptr : base + pg * page_stride + a.kv.page_div.mod(p) * tok_stride + 16 * col;
  };
  unsigned got = 0;  // which pieces of the chunks in flight were fetched, 4 bits per stage
  auto fetch = [&](int c) {
    const int st = c % kMoveStages;
    got &= ~(0xfu << (4 * st));
    if (c < chunks) {
      const uint8_t* src[kMoveVecs];
#pragma unroll
      for (int i = 0; i < kMoveVecs; ++i) {
        const int vec = tid + i * kMoveThreads;
        const int p = c * rows + (vec >> shift);
        src[i] = p < a.budget ? at(list[p], vec & (v - 1)) : nullptr;
      }
#pragma unroll
      for (int i = 0; i < kMoveVecs; ++i)
        if (src[i]) {
          cp_async16(my + (st * kChunkVecs + i * kMoveThreads) * 16, src[i]);
          got |= 1u << (4 * st + i);
        }
    }
    cp_async_commit();
  };
  for (int c = first; c < first + kMoveStages - 1; ++c) fetch(c);
  for (int c = first; c < chunks; ++c) {
    fetch(c + kMoveStages - 1);
    cp_async_wait<kMoveStages - 1>();
    __syncthreads();  // the whole chunk (and all before it) is read: its destinations are free
    const int st = c % kMoveStages;
#pragma unroll
    for (int i = 0; i < kMoveVecs; ++i) {
      if (!(got >> (4 * st + i) & 1u)) continue;
      const int vec = tid + i * kMoveThreads;
      uint8_t* dst = at(c * rows + (vec >> shift), vec & (v - 1));
      if (dst) *reinterpret_cast<uint4*>(dst) = ring[st * kChunkVecs + vec];
    }
  }
  cp_async_wait<0>();
}

// Scales, weights and the new length of one (sequence, KV head), in the same chunk order.
__device__ void move_scalars(const PagedEvict& a, const int* list, const int* row, int unit, int2 state) {
  const int tid = threadIdx.x, kh = unit % a.kv.Hkv;
  const float* w = a.weights + size_t(unit) * a.kv.cap;
  float* wo = a.weights_out + size_t(unit) * a.kv.cap;
  if (kh == 0 && tid == 0) a.lens_out[unit / a.kv.Hkv] = state.x ? a.budget : state.y;
  if (!state.x) {
    if (wo != w)
      for (int i = tid; i < state.y; i += kMoveThreads) wo[i] = w[i];
    return;
  }
  for (int p0 = 0; p0 < a.budget; p0 += kMoveThreads) {
    const int p = p0 + tid;
    const bool on = p < a.budget;
    float x = 0.f;
    __half ks = __half(0.f), vs = __half(0.f);
    bool sc = false;
    if (on) {
      const int s = list[p];
      x = w[s];
      if (a.kv.int8) {
        const int pg = page_at(a, row, s);
        if (pg >= 0) {
          ks = a.kv.ks[pg * a.kv.ks_page + kh * a.kv.ks_head + a.kv.page_div.mod(s)];
          vs = a.kv.vs[pg * a.kv.vs_page + kh * a.kv.vs_head + a.kv.page_div.mod(s)];
          sc = true;
        }
      }
    }
    __syncthreads();
    if (on) {
      wo[p] = x;
      const int pg = sc ? page_at(a, row, p) : -1;
      if (pg >= 0) {
        a.kv.ks[pg * a.kv.ks_page + kh * a.kv.ks_head + a.kv.page_div.mod(p)] = ks;
        a.kv.vs[pg * a.kv.vs_page + kh * a.kv.vs_head + a.kv.page_div.mod(p)] = vs;
      }
    }
  }
  __syncthreads();  // in place: the last chunk's sources may lie behind the budget
  for (int p = a.budget + tid; p < state.y; p += kMoveThreads) wo[p] = 0.f;
}

// Grid: (2 * slices + 1, B * Hkv).
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ PagedEvict a) {
  extern __shared__ uint4 ring[];
  pdl_launch_dependents();
  pdl_wait_primary();
  const int unit = int(blockIdx.y), job = int(blockIdx.x);
  const int2 state = a.state[unit];
  const int* list = a.list + size_t(unit) * a.budget;
  const int b = unit / a.kv.Hkv, kh = unit - b * a.kv.Hkv;
  const int* row = a.kv.table + int64_t(b) * a.kv.table_stride;
  if (job == 2 * a.slices) {
    move_scalars(a, list, row, unit, state);
    return;
  }
  if (!state.x) return;
  const bool is_v = job >= a.slices;
  const int elt = a.kv.int8 ? 1 : 2;
  const int width = a.kv.D * elt / a.slices;  // bytes
  const int col = (is_v ? job - a.slices : job) * width;
  uint8_t* base = static_cast<uint8_t*>(is_v ? a.kv.v : a.kv.k) + int64_t(kh) * (is_v ? a.kv.v_head : a.kv.k_head) * elt + col;
  move_rows(a, list, row, base, (is_v ? a.kv.v_page : a.kv.k_page) * elt, (is_v ? a.kv.v_tok : a.kv.k_tok) * elt,
            width / 16, ring);
}

constexpr size_t kMoveSmem = size_t(kMoveStages) * kChunkVecs * 16;

}  // namespace

cudaError_t evict_prepare() {
  return cudaFuncSetAttribute(evict_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kMoveSmem));
}

cudaError_t launch_evict_paged(const PagedEvict& a, cudaStream_t stream) {
  const int units = a.kv.B * a.kv.Hkv;
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
  return launch_pdl(evict_move_kernel, dim3(2 * a.slices + 1, units), dim3(kMoveThreads), kMoveSmem, stream, a);
}

}  // namespace fqkv
