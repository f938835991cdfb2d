// Rotary embedding with one or several position axes, the fp16 cast of q and the append of k and v to a
// paged KV cache, for any number of tokens (a decode step, packed prompts), sm_100a.
//
// Token t of a fused projection [q heads | k heads | v heads]: pair i of a q or k head is dimensions i and
// i + D/2, turned by the angle whose cosine and sine stand in row pos[axis[i]][t], column i of the tables:
//   y[i] = x[i] c - x[i + D/2] s,   y[i + D/2] = x[i + D/2] c + x[i] s.
// fp32 throughout (the tables too: a table in the model's 16-bit type would cost 2^-9 of every angle);
// q, k and v are rounded once, to fp16.  An int8 cache then takes the fp16 row's codes and scale, bit for bit
// what the per-token quantizer gives for it.
//
// Bound: HBM for prompts (every projected element is read once and written once), launch latency for a decode step;
// a kernel for each.  A thread holds 8 pairs of a head in 16-byte halves and D/16 threads make a head.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "device_common.cuh"
#include "kernels.h"
#include "quant_common.cuh"

namespace fqkv {
namespace {

constexpr int kAppendThreads = 128;
// From how many tokens on the ring pays (32 + 2 x 8 heads, D = 128, bf16 -> fp16 cache, one B200, few-token against
// many-token kernel): 400 to 1000 tokens alike (6.1 to 8.2 us), 2000 tokens 15.1 -> 12.6 us, 8191 tokens 46.5 -> 37.4 us
// (5.4 TB/s); into an int8 cache 51.2 -> 33.9 us.
constexpr int kManyTokens = 1000;
constexpr size_t kMostSmem = 200 * 1024;  // of a block's ring; rows too long for three stages go by the few-token kernel

__device__ __forceinline__ float2 to_f2(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 to_f2(__nv_bfloat162 v) { return __bfloat1622float2(v); }

template <typename T2>
__device__ __forceinline__ void to_f8(const uint4& r, float (&x)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = to_f2(*reinterpret_cast<const T2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Codes of 8 values at scale sc, one byte each (the arithmetic of the quantizer kernels).
__device__ __forceinline__ uint2 codes8(const __half2 (&h)[4], float sc) {
  uint32_t cb[4];
  if (normal_fp16_scale(sc)) {
    const float y = rcp_approx(sc);
    const unsigned long long y2 = f32x2_pack(y, y), ns2 = f32x2_pack(-sc, -sc);
#pragma unroll
    for (int i = 0; i < 4; ++i) cb[i] = code_pair_fast(h[i], ns2, y2);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(h[i]);
      cb[i] = (uint32_t(quant_code<127>(f.x, sc)) & 0xFFu) | ((uint32_t(quant_code<127>(f.y, sc)) & 0xFFu) << 16);
    }
  }
  return make_uint2(__byte_perm(cb[0], cb[1], 0x6420u), __byte_perm(cb[2], cb[3], 0x6420u));
}

constexpr int kThreadsPerHead(int D) { return D / 16; }

// Pairs 8j .. 8j + 7 of head h of one token: turn (q and k heads), round, store or quantize and store.  Every lane of
// a warp takes part (`on`: there is such a head); `kv`: some lane of the warp may hold a k or v head.
template <typename T2, int D, bool kI8>
__device__ __forceinline__ void put_head(const PagedAppend& a, int64_t token, int h, bool on, bool kv, const uint4& rlo,
                                         const uint4& rhi, const float (&c)[8], const float (&s)[8], int page, int off) {
  constexpr int kTPH = kThreadsPerHead(D);
  const int j = threadIdx.x % kTPH;
  float lo[8], hi[8];
  if (on) {
    to_f8<T2>(rlo, lo);
    to_f8<T2>(rhi, hi);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = hi[i] = 0.f;
  }
  const bool is_v = h >= a.Hq + a.kv.Hkv;
  if (!is_v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float l = lo[i], u = hi[i];
      lo[i] = l * c[i] - u * s[i];
      hi[i] = u * c[i] + l * s[i];
    }
  }
  __half2 hl[4], hh[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hl[i] = __floats2half2_rn(lo[2 * i], lo[2 * i + 1]);
    hh[i] = __floats2half2_rn(hi[2 * i], hi[2 * i + 1]);
  }
  if (h < a.Hq) {
    __half* q = a.q_out + (token * a.Hq + h) * D + 8 * j;
    *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(&hl[0]);
    *reinterpret_cast<uint4*>(q + D / 2) = *reinterpret_cast<const uint4*>(&hh[0]);
  }
  if (!kv) return;
  const int kh = is_v ? h - a.Hq - a.kv.Hkv : h - a.Hq;
  if constexpr (!kI8) {
    if (!on || h < a.Hq) return;
    __half* dst = is_v ? static_cast<__half*>(a.kv.v) + page * a.kv.v_page + kh * a.kv.v_head + off * a.kv.v_tok
                       : static_cast<__half*>(a.kv.k) + page * a.kv.k_page + kh * a.kv.k_head + off * a.kv.k_tok;
    *reinterpret_cast<uint4*>(dst + 8 * j) = *reinterpret_cast<const uint4*>(&hl[0]);
    *reinterpret_cast<uint4*>(dst + 8 * j + D / 2) = *reinterpret_cast<const uint4*>(&hh[0]);
  } else {
    __half2 m2 = __habs2(hl[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) m2 = __hmax2_nan(m2, __habs2(hl[i]));
#pragma unroll
    for (int i = 0; i < 4; ++i) m2 = __hmax2_nan(m2, __habs2(hh[i]));
#pragma unroll
    for (int o = 1; o < kTPH; o <<= 1) m2 = __hmax2_nan(m2, __shfl_xor_sync(0xffffffffu, m2, o));
    m2 = __hmax2_nan(m2, __lowhigh2highlow(m2));
    const __half sh = quant_scale_fast<127>(__low2float(m2), __hisnan(__low2half(m2)));
    if (!on || h < a.Hq) return;
    int8_t* dst = is_v ? static_cast<int8_t*>(a.kv.v) + page * a.kv.v_page + kh * a.kv.v_head + off * a.kv.v_tok
                       : static_cast<int8_t*>(a.kv.k) + page * a.kv.k_page + kh * a.kv.k_head + off * a.kv.k_tok;
    const float sc = __half2float(sh);
    *reinterpret_cast<uint2*>(dst + 8 * j) = codes8(hl, sc);
    *reinterpret_cast<uint2*>(dst + 8 * j + D / 2) = codes8(hh, sc);
    if (j == 0) {
      if (is_v) a.kv.vs[page * a.kv.vs_page + kh * a.kv.vs_head + off] = sh;
      else a.kv.ks[page * a.kv.ks_page + kh * a.kv.ks_head + off] = sh;
    }
  }
}

template <int D>
__device__ __forceinline__ void read_angles(const float* table, int j, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    *reinterpret_cast<float4*>(&c[i]) = *reinterpret_cast<const float4*>(&table[8 * j + i]);
    *reinterpret_cast<float4*>(&s[i]) = *reinterpret_cast<const float4*>(&table[D / 2 + 8 * j + i]);
  }
}

// Few tokens: latency.  Grid: (tokens, passes of a token's heads).  T2: the projection's element pairs.
template <typename T2, int D, bool kI8>
__global__ void __launch_bounds__(kAppendThreads) append_few_kernel(const __grid_constant__ PagedAppend a) {
  constexpr int kTPH = kThreadsPerHead(D);
  constexpr int kHeads = kAppendThreads / kTPH;  // heads of a block
  __shared__ __align__(16) float table[D];       // the token's cosines and sines
  pdl_launch_dependents();
  pdl_wait_primary();
  const int64_t token = blockIdx.x;
  const int j = threadIdx.x % kTPH;
  const int h0 = int(blockIdx.y) * kHeads, h = h0 + threadIdx.x / kTPH;
  const bool on = h < a.Hq + 2 * a.kv.Hkv;
  uint4 rlo = make_uint4(0, 0, 0, 0), rhi = rlo;
  if (on) {  // under way while the token's place and angles are looked up
    const uint16_t* x = static_cast<const uint16_t*>(a.qkv) + token * a.qkv_stride + int64_t(h) * D + 8 * j;
    rlo = *reinterpret_cast<const uint4*>(x);
    rhi = *reinterpret_cast<const uint4*>(x + D / 2);
  }
  const int slot = a.slots[token];
  if (slot < 0) return;  // padding
  const int seq = a.seq_ids ? a.seq_ids[token] : int(token);
  const bool placed = seq >= 0 && seq < a.kv.B && slot < a.kv.cap;
  bool good = placed;
  if (threadIdx.x < D) {
    const int i = threadIdx.x % (D / 2), which = threadIdx.x / (D / 2);
    const int axis = a.axes == 1 ? 0 : a.axis_map[i];
    int p = -1;
    if (unsigned(axis) < unsigned(a.axes)) p = a.positions[axis * a.pos_stride + token];
    if (p >= 0 && p < a.table_rows) table[threadIdx.x] = (which ? a.sin_t : a.cos_t)[int64_t(p) * (D / 2) + i];
    else good = false;
  }
  int page = 0;
  if (placed) page = a.kv.table[int64_t(seq) * a.kv.table_stride + a.kv.page_div.div(slot)];
  // a wrong place or angle is recorded and nothing of the token is written
  if (!__syncthreads_and(good)) {
    if (threadIdx.x == 0) atomicCAS(a.status, kDevOk, kDevBadToken);
    return;
  }
  if (unsigned(page) >= unsigned(a.kv.num_pages)) {
    if (threadIdx.x == 0) atomicCAS(a.status, kDevOk, kDevBadPage);
    return;
  }
  float c[8], s[8];
  read_angles<D>(table, j, c, s);
  put_head<T2, D, kI8>(a, token, h, on, h0 + kHeads > a.Hq, rlo, rhi, c, s, page, a.kv.page_div.mod(slot));
}

// Many tokens: bandwidth.  A persistent grid; in every block a producer warp fetches the rows of the block's tokens
// (one bulk copy each) and their angles (4-byte asynchronous copies) into a ring of stages, with the lookups of a
// token's slot, positions and page two and one tokens ahead, and four warps put the heads.
constexpr int kRowStages = 3;

struct RowStage {  // behind the row in a stage
  int slot, page;  // slot < 0: nothing to write
};

__host__ __device__ constexpr size_t row_stage_bytes(int64_t row_bytes, int D) {
  return (size_t(row_bytes) + size_t(D) * 4 + sizeof(RowStage) + 127) & ~size_t(127);
}

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// One arrival on `bar` when this thread's cp.async copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

template <typename T2, int D, bool kI8>
__global__ void __launch_bounds__(kAppendThreads + 32) append_many_kernel(const __grid_constant__ PagedAppend a) {
  constexpr int kTPH = kThreadsPerHead(D);
  constexpr int kHeads = kAppendThreads / kTPH;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kRowStages], empty[kRowStages];
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = a.Hq + 2 * a.kv.Hkv;
  const uint32_t row_bytes = uint32_t(heads) * D * 2;
  const size_t stage_bytes = row_stage_bytes(row_bytes, D);
  const WaitCtl wc{a.status, a.timeout_ns};
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRowStages; ++i) {
      mbar_init(&full[i], 1 + 32);
      mbar_init(&empty[i], kAppendThreads / 32);
    }
    abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait_primary();

  // ------------------------------------------------------------ producer
  if (warp == kAppendThreads / 32) {
    if (a.debug_skip_loads == 1) return;
    constexpr int kPairs = D / 64;  // rotary pairs per lane
    int axis[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) axis[i] = a.axes == 1 ? 0 : a.axis_map[lane + 32 * i];
    // of the token after the next: slot, sequence, the positions of this lane's pairs
    int slot2 = -1, seq2 = 0, pos2[kPairs];
    auto look = [&](int64_t token) {
      slot2 = -1;
      if (token >= a.T) return;
      slot2 = a.slots[token];
      seq2 = a.seq_ids ? a.seq_ids[token] : int(token);
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
        pos2[i] = unsigned(axis[i]) < unsigned(a.axes) ? a.positions[axis[i] * a.pos_stride + token] : -1;
    };
    // of the next one: its page too
    int slot1 = -1, page1 = 0, pos1[kPairs];
    bool placed1 = false;
    auto place = [&]() {
      slot1 = slot2;
      placed1 = slot2 >= 0 && seq2 >= 0 && seq2 < a.kv.B && slot2 < a.kv.cap;
      if (placed1) page1 = a.kv.table[int64_t(seq2) * a.kv.table_stride + a.kv.page_div.div(slot2)];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) pos1[i] = pos2[i];
    };
    look(blockIdx.x);
    place();
    look(int64_t(blockIdx.x) + gridDim.x);
    int it = 0;
    for (int64_t token = blockIdx.x; token < a.T; token += gridDim.x, ++it) {
      const int st = it % kRowStages;
      if (it >= kRowStages) {
        const bool free_stage = !*reinterpret_cast<volatile int*>(&abort_flag) &&
                                mbar_wait(&empty[st], ((it / kRowStages) - 1) & 1, wc, kDevTimeoutEmpty);
        if (!__all_sync(0xffffffffu, free_stage)) break;
      }
      bool good = placed1;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) good = good && pos1[i] >= 0 && pos1[i] < a.table_rows;
      good = __all_sync(0xffffffffu, good);
      const bool known = unsigned(page1) < unsigned(a.kv.num_pages);
      uint8_t* stage = ring + size_t(st) * stage_bytes;
      float* table = reinterpret_cast<float*>(stage + row_bytes);
      const bool put = slot1 >= 0 && good && known, send = put && !a.debug_skip_loads;
      if (lane == 0) {
        // padding is passed over; a wrong place or angle is recorded
        if (slot1 >= 0 && !put) atomicCAS(a.status, kDevOk, good ? kDevBadPage : kDevBadToken);
        *reinterpret_cast<RowStage*>(stage + row_bytes + D * 4) = RowStage{put ? slot1 : -1, page1};
        mbar_arrive_expect_tx(&full[st], put ? row_bytes : 0u);
        if (send) bulk_g2s(stage, static_cast<const uint16_t*>(a.qkv) + token * a.qkv_stride, row_bytes, &full[st]);
      }
      if (send) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const int64_t at = int64_t(pos1[i]) * (D / 2) + lane + 32 * i;
          cp_async4(table + lane + 32 * i, a.cos_t + at);
          cp_async4(table + D / 2 + lane + 32 * i, a.sin_t + at);
        }
      }
      cp_async_arrive(&full[st]);
      place();
      look(token + 2 * int64_t(gridDim.x));
    }
    // The copies in flight land (a bounded wait) before the block's memory goes, whether the consumers are there for them
    // or gave up.
    if (lane == 0)
      for (int i = max(0, it - kRowStages); i < it; ++i)
        mbar_wait(&full[i % kRowStages], (i / kRowStages) & 1, wc, kDevTimeoutDrain);
    return;
  }

  // ------------------------------------------------------------ consumers
  const int j = threadIdx.x % kTPH, hs = threadIdx.x / kTPH;
  int it = 0;
  for (int64_t token = blockIdx.x; token < a.T; token += gridDim.x, ++it) {
    const int st = it % kRowStages;
    const bool ok = a.debug_skip_loads != 2 && mbar_wait(&full[st], (it / kRowStages) & 1, wc, kDevTimeoutFull) &&
                    !*reinterpret_cast<volatile int*>(&abort_flag);
    if (!__all_sync(0xffffffffu, ok)) {
      if (lane == 0) abort_flag = 1;
      break;
    }
    const uint8_t* stage = ring + size_t(st) * stage_bytes;
    const RowStage meta = *reinterpret_cast<const RowStage*>(stage + row_bytes + D * 4);
    if (meta.slot >= 0) {
      float c[8], s[8];
      read_angles<D>(reinterpret_cast<const float*>(stage + row_bytes), j, c, s);
      const int off = a.kv.page_div.mod(meta.slot);
      for (int h0 = 0; h0 < heads; h0 += kHeads) {
        const int h = h0 + hs;
        const bool on = h < heads;
        uint4 rlo = make_uint4(0, 0, 0, 0), rhi = rlo;
        if (on) {
          rlo = *reinterpret_cast<const uint4*>(stage + size_t(h) * D * 2 + 16 * j);
          rhi = *reinterpret_cast<const uint4*>(stage + size_t(h) * D * 2 + D + 16 * j);
        }
        put_head<T2, D, kI8>(a, token, h, on, h0 + kHeads > a.Hq, rlo, rhi, c, s, meta.page, off);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&empty[st]);
  }
}

template <typename T2, int D, bool kI8>
cudaError_t launch_t(const PagedAppend& a, cudaStream_t stream) {
  const int heads = a.Hq + 2 * a.kv.Hkv;
  const size_t smem = kRowStages * row_stage_bytes(int64_t(heads) * D * 2, D);
  if (a.T < kManyTokens || smem > kMostSmem) {
    constexpr int kHeads = kAppendThreads / kThreadsPerHead(D);
    return launch_pdl(append_few_kernel<T2, D, kI8>, dim3(unsigned(a.T), unsigned((heads + kHeads - 1) / kHeads)),
                      dim3(kAppendThreads), 0, stream, a);
  }
  // as many blocks as the rings leave room for, 10 at most (1600 threads)
  const int per_sm = std::max(1, std::min(10, int((kMostSmem + 1024) / (smem + 1024))));
  return launch_pdl(append_many_kernel<T2, D, kI8>, dim3(unsigned(std::min<int64_t>(a.T, int64_t(a.sms) * per_sm))),
                    dim3(kAppendThreads + 32), smem, stream, a);
}

template <typename T2, int D>
cudaError_t launch_d(const PagedAppend& a, cudaStream_t stream) {
  return a.kv.int8 ? launch_t<T2, D, true>(a, stream) : launch_t<T2, D, false>(a, stream);
}

template <typename T2, int D>
cudaError_t prepare_d() {
  cudaError_t e = cudaFuncSetAttribute(append_many_kernel<T2, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       int(kMostSmem));
  if (e != cudaSuccess) return e;
  return cudaFuncSetAttribute(append_many_kernel<T2, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              int(kMostSmem));
}

}  // namespace

cudaError_t append_paged_prepare() {
  cudaError_t e = prepare_d<__half2, 64>();
  if (e == cudaSuccess) e = prepare_d<__half2, 128>();
  if (e == cudaSuccess) e = prepare_d<__nv_bfloat162, 64>();
  if (e == cudaSuccess) e = prepare_d<__nv_bfloat162, 128>();
  return e;
}

cudaError_t launch_append_paged(const PagedAppend& a, bool bf16, cudaStream_t stream) {
  if (bf16) return a.kv.D == 128 ? launch_d<__nv_bfloat162, 128>(a, stream) : launch_d<__nv_bfloat162, 64>(a, stream);
  return a.kv.D == 128 ? launch_d<__half2, 128>(a, stream) : launch_d<__half2, 64>(a, stream);
}

}  // namespace fqkv
