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
// Bound: HBM for prompts (every projected element is read once and written once), launch latency for a
// decode step.  A thread holds 8 pairs of one head in 16-byte halves; D/16 threads make a head, and the
// threads of a block that sit at the same place of their heads go through the token's heads with the same
// 16 table entries in registers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "device_common.cuh"
#include "kernels.h"
#include "quant_common.cuh"

namespace fqkv {
namespace {

constexpr int kAppendThreads = 128;

__device__ __forceinline__ float2 to_f2(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 to_f2(__nv_bfloat162 v) { return __bfloat1622float2(v); }

template <typename T2>
__device__ __forceinline__ void load8(const void* src, float (&x)[8]) {
  const uint4 r = *static_cast<const uint4*>(src);
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

// T2: the projection's element pairs.  Grid: (tokens, parts of a token's heads).
template <typename T2, int D, bool kI8>
__global__ void __launch_bounds__(kAppendThreads) append_paged_kernel(const __grid_constant__ PagedAppend a) {
  constexpr int kTPH = D / 16;                      // threads per head
  constexpr int kHeads = kAppendThreads / kTPH;     // heads per pass
  pdl_launch_dependents();
  pdl_wait_primary();
  const int64_t token = blockIdx.x;
  const int slot = a.slots[token];
  if (slot < 0) return;  // padding
  const int j = threadIdx.x % kTPH, hs = threadIdx.x / kTPH;
  const int seq = a.seq_ids ? a.seq_ids[token] : int(token);

  // the token's place; a wrong one is recorded and nothing of the token is written
  bool good = seq >= 0 && seq < a.kv.B && slot < a.kv.cap;
  for (int x = 0; x < a.axes; ++x) {
    const int p = a.positions[x * a.pos_stride + token];
    good = good && p >= 0 && p < a.table_rows;
  }
  if (!good) {
    if (threadIdx.x == 0) atomicCAS(a.status, kDevOk, kDevBadToken);
    return;
  }
  const int page = a.kv.table[int64_t(seq) * a.kv.table_stride + a.kv.page_div.div(slot)];
  if (unsigned(page) >= unsigned(a.kv.num_pages)) {
    if (threadIdx.x == 0) atomicCAS(a.status, kDevOk, kDevBadPage);
    return;
  }
  const int off = a.kv.page_div.mod(slot);

  // cosines and sines of pairs 8j .. 8j + 7
  float c[8], s[8];
  if (a.axes == 1) {
    const int64_t at = int64_t(a.positions[token]) * (D / 2) + 8 * j;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *reinterpret_cast<float4*>(&c[i]) = *reinterpret_cast<const float4*>(a.cos_t + at + i);
      *reinterpret_cast<float4*>(&s[i]) = *reinterpret_cast<const float4*>(a.sin_t + at + i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned x = unsigned(a.axis_map[8 * j + i]);
      if (x >= unsigned(a.axes)) atomicCAS(a.status, kDevOk, kDevBadToken);
      const int64_t p = a.positions[int64_t(x < unsigned(a.axes) ? x : 0u) * a.pos_stride + token];
      c[i] = a.cos_t[p * (D / 2) + 8 * j + i];
      s[i] = a.sin_t[p * (D / 2) + 8 * j + i];
    }
  }

  const int heads = a.Hq + 2 * a.kv.Hkv;
  const uint16_t* x = static_cast<const uint16_t*>(a.qkv) + token * a.qkv_stride + 8 * j;
  for (int h0 = int(blockIdx.y) * kHeads; h0 < heads; h0 += int(gridDim.y) * kHeads) {
    const int h = h0 + hs;
    const bool on = h < heads;
    float lo[8], hi[8];
    if (on) {
      load8<T2>(x + int64_t(h) * D, lo);
      load8<T2>(x + int64_t(h) * D + D / 2, hi);
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
    const int kh = is_v ? h - a.Hq - a.kv.Hkv : h - a.Hq;
    __half sh = __half(0.f);
    if constexpr (kI8) {
      __half2 m2 = __habs2(hl[0]);
#pragma unroll
      for (int i = 1; i < 4; ++i) m2 = __hmax2_nan(m2, __habs2(hl[i]));
#pragma unroll
      for (int i = 0; i < 4; ++i) m2 = __hmax2_nan(m2, __habs2(hh[i]));
#pragma unroll
      for (int o = 1; o < kTPH; o <<= 1) m2 = __hmax2_nan(m2, __shfl_xor_sync(0xffffffffu, m2, o));
      m2 = __hmax2_nan(m2, __lowhigh2highlow(m2));
      sh = quant_scale_fast<127>(__low2float(m2), __hisnan(__low2half(m2)));
    }
    if (!on) continue;
    if (h < a.Hq) {
      __half* q = a.q_out + (token * a.Hq + h) * D + 8 * j;
      *reinterpret_cast<uint4*>(q) = *reinterpret_cast<const uint4*>(&hl[0]);
      *reinterpret_cast<uint4*>(q + D / 2) = *reinterpret_cast<const uint4*>(&hh[0]);
    } else if constexpr (!kI8) {
      __half* dst = is_v ? static_cast<__half*>(a.kv.v) + page * a.kv.v_page + kh * a.kv.v_head + off * a.kv.v_tok
                         : static_cast<__half*>(a.kv.k) + page * a.kv.k_page + kh * a.kv.k_head + off * a.kv.k_tok;
      *reinterpret_cast<uint4*>(dst + 8 * j) = *reinterpret_cast<const uint4*>(&hl[0]);
      *reinterpret_cast<uint4*>(dst + 8 * j + D / 2) = *reinterpret_cast<const uint4*>(&hh[0]);
    } else {
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
}

template <typename T2, int D>
cudaError_t launch_d(const PagedAppend& a, cudaStream_t stream) {
  constexpr int kHeads = kAppendThreads / (D / 16);
  const int parts = (a.Hq + 2 * a.kv.Hkv + kHeads - 1) / kHeads;
  // Few tokens: a block per pass of heads, for latency.  Many: one block per token reads the table once.
  const dim3 grid(unsigned(a.T), a.T < 512 ? unsigned(parts) : 1u);
  return a.kv.int8 ? launch_pdl(append_paged_kernel<T2, D, true>, grid, dim3(kAppendThreads), 0, stream, a)
                   : launch_pdl(append_paged_kernel<T2, D, false>, grid, dim3(kAppendThreads), 0, stream, a);
}

}  // namespace

cudaError_t launch_append_paged(const PagedAppend& a, bool bf16, cudaStream_t stream) {
  if (bf16) return a.kv.D == 128 ? launch_d<__nv_bfloat162, 128>(a, stream) : launch_d<__nv_bfloat162, 64>(a, stream);
  return a.kv.D == 128 ? launch_d<__half2, 128>(a, stream) : launch_d<__half2, 64>(a, stream);
}

}  // namespace fqkv
