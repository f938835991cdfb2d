// Single-query attention over a paged KV cache with one length per sequence, sm_100a.
//
//   out[b, h] = sum_j softmax_j(q[b, h] . k[b, kh, j] / sqrt(D)) v[b, kh, j],   j < len[b], kh = h / G,
// token j of sequence b in slot j % page of page table[b, j / page] of the pools [P, Hkv, page, D] (fp16,
// or int8 codes with one fp16 scale per token and KV head).  An empty sequence gives zeros.  Optionally
//   weights[b, kh, j] += sum over the group's heads of softmax_j.
//
// Bound: HBM (each K/V byte is read once for all query heads of its KV head; about one multiply-add per
// byte and head).  Work split: the lengths are known only on the device, so the launch cannot cut the work
// by sequence.  All key tiles of all (sequence, KV head) units stand in one line of T tiles and CTA c of a
// persistent grid takes tiles [c * per, (c + 1) * per), per = ceil(T / grid): every CTA streams the same
// number of bytes whatever the lengths are.  A unit that lies inside one CTA's range is finished there; one
// that crosses a border leaves unnormalised fp32 parts (two slots per CTA: the unit its range begins in and
// the one it ends in), merged by the next launch in tile order, so results do not depend on timing.
// Few short units (a choice of the host, by sizes) get a thread-block cluster each instead, which merges its parts
// through distributed shared memory in the same launch.
//
//  * Warp 4 is the producer.  A tile is fetched as boxes of 16, 32, 64 or 128 keys (the largest that divides
//    the page), each inside one page, by 4-D tensor copies over (D, token, head, page) with any 16-byte
//    strides -- tokens outside heads or inside.  The lanes of the warp issue one box each.  Page numbers are
//    read 32 boxes ahead.
//  * Warps 0-3 take 16 (or 32) keys of a tile each.  S = Q K^T by mma m16n8k16 with the heads as rows;
//    O^T += V^T P^T with the head dimension as rows, where the probabilities are the B operand exactly as
//    the score accumulators hold them and 8 heads fill all 8 columns: half the MMAs and half the accumulator
//    registers of the P V order, which leaves half of its 16 rows empty.  More than 8 heads take two column
//    tiles, so up to 16 heads share one pass over K and V.
//  * int8, S: integer MMAs (m16n8k32) on the codes as they lie in memory.  A head's q is a fixed-point number of
//    22 bits, q 2^k = hi 65536 + mid 256 + lo with max |q| 2^k in [2^21, 2^22): an fp16 q is exact in it down to 2^-11 of
//    the largest, so the sums of products are exact integers and the score is rounded only when the three are put
//    together.  Up to 8 heads: rows 0-7 of one MMA are hi, rows 8-15 mid, a second one takes lo.  Against codes
//    converted to fp16 this saves 80 of about 290 instructions per warp and 16 keys at D = 128.
//  * int8, P V: a code becomes the fp16 number 1152 + code by one byte permute (of code + 128), and a second MMA with
//    a constant tile takes 1152 P away again, 16 keys at a time: the subtraction costs tensor-core time, which is
//    there, and no instruction per code; what it rounds is 2^-24 of 1152 P, 7e-5 of a code's step.  The K scale multiplies
//    the score.  The V scale multiplies the probability before it is
//    rounded to fp16, times a power of two that puts the unit's largest V scale so far (by magnitude) in
//    [2^13, 2^14): small scales keep all their bits, and the factor leaves exactly at the end of the unit.
//  * Scores, maxima, sums and outputs are fp32; the probabilities are rounded to fp16 once, as the operand of
//    the second product; the output is rounded once.  fp16 cache: times 2^15 first (1 becomes 32768, below fp16's
//    largest), and O times 2^-15 at the end of a unit, both exact.  So a probability down to 2^-29 of the warp's
//    largest has all its 11 bits (half a step is at most 2^-11 relative), and one below is off by 2^-40 of the
//    largest at most: beside a dominant key the many small ones of a long cache keep their sum (unscaled, half a
//    step is 2^-25: equal weights of 2^-24.5 came out 1.41 times too large, of 2^-25.1 as nothing).
//    O is summed in the MMAs' fp32 accumulators, which cut the last bit: 2^20 tokens in one CTA with equal weights
//    and values of 0.5 to 1 came out 5 to 9e-4 too small.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "device_common.cuh"
#include "kernels.h"

namespace fqkv {
namespace {

constexpr int kWarps = 4;          // consumer warps
constexpr int kThr = 32 * (kWarps + 1);
constexpr int kMergeHeads = 4;     // heads merged per epilogue pass
constexpr int kMaxCluster = 16;

template <int D, bool kI8>
struct Cfg {
  static constexpr int KPW = kI8 ? 32 : 16;    // keys of a tile per consumer warp
  static constexpr int TK = kWarps * KPW;                 // keys per tile
  static constexpr int kBlocks = kI8 ? 1 : D / 64;        // column blocks of a tile (128-byte fp16 rows)
  static constexpr int RB = kI8 ? D : 128;                // bytes of a row of a column block
  static constexpr int kBlockBytes = TK * RB;
  static constexpr int kTileBytes = kBlocks * kBlockBytes;  // K (or V) of one tile
  static constexpr int kScaleBytes = kI8 ? 2 * TK : 0;
  static constexpr int kStageBytes = 2 * kTileBytes + (kI8 ? 1024 : 0);  // scales in a 1 KB tail: tiles stay aligned
  // fp16: as many CTAs as fit beside three stages (3 CTAs of two stages at D = 128 measured within 1 %).
  // int8: 32 keys per warp, so that two independent 16-key chains cover each other's latency, and registers for
  // them: B = 64, 16K, D = 128 301 us; 16 keys per warp and 3 CTAs 316 us (4 CTAs spill: 350 us), 32 keys and 3 CTAs
  // of two stages 354 us (spills).
  static constexpr int kCtas = D == 128 ? 2 : (kI8 ? 3 : 4);
  static constexpr int kStages = 3;
  static constexpr size_t kRingBytes = size_t(kStages) * kStageBytes;
  static constexpr size_t kBarBytes = (2 * kStages * sizeof(uint64_t) + 15) & ~size_t(15);
  static constexpr int kHeadStride = D + 4;               // floats; makes the epilogue's stores conflict-free
  static constexpr size_t kMergeBytes = size_t(kWarps) * (2 * kPagedMaxHeads + kMergeHeads * kHeadStride) * sizeof(float);
  static constexpr size_t kSmemBytes = 1024 + kRingBytes + kBarBytes + kMergeBytes;
};

// Tiled tensor copy of one box of one page into this CTA's shared memory.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w),
        "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// One arrival on `bar` when this thread's cp.async copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Byte offset of 16-byte chunk `chunk` of row `row` of a tile written with the swizzle of its row width: the
// chunk's number XOR the row's place in the swizzle atom.  For a lane's row and chunk parity, the offset of chunk
// 2i + parity is that of `parity` XOR 32 i within a column block (tiles are 1024-byte aligned), so a lane needs
// one logic operation per ldmatrix.
template <int RB>
__device__ __forceinline__ uint32_t blk_off(int row, int c) {
  if constexpr (RB == 128) return uint32_t(row * 128 + ((c ^ (row & 7)) << 4));
  else return uint32_t(row * 64 + ((c ^ ((row >> 1) & 3)) << 4));
}
// Address of chunk 2i + parity from the address `at` of chunk `parity`.
template <int D, bool kI8>
__device__ __forceinline__ uint32_t chunk_at(uint32_t at, int i) {
  constexpr int kPer = Cfg<D, kI8>::RB / 32;  // chunk pairs per column block
  return (at ^ uint32_t((i % kPer) * 32)) + uint32_t((i / kPer) * Cfg<D, kI8>::kBlockBytes);
}

// ------------------------------------------------------------------ the line of tiles
// One stretch of tiles of one unit inside a CTA's range.
struct Part {
  int b, kh, grp;  // the unit: sequence, KV head, head group
  int len, nt;     // the sequence's tokens and tiles
  int t0, t1;      // tiles [t0, t1)
};

// The walk over a CTA's range; every warp runs its own, all lanes alike.
struct Walk {
  const int* lens;
  int B, cap, tk, units_per_seq, groups;
  int per, cur, end;  // tiles per CTA; the range's position and end in the line
  int b, u, t, len, nt;

  __device__ __forceinline__ int length(int i) const { return max(0, min(cap, lens[i])); }
  __device__ __forceinline__ int tiles(int n) const { return (n + tk - 1) / tk; }

  __device__ __forceinline__ void init(const PagedLaunch& a, int tile_keys) {
    const int lane = threadIdx.x & 31;
    lens = a.seq_lens;
    B = a.B;
    cap = a.cap;
    tk = tile_keys;
    groups = a.groups;
    units_per_seq = a.Hkv * a.groups;
    int sum = 0;
    for (int i = lane; i < B; i += 32) sum += tiles(length(i));
    sum = __reduce_add_sync(0xffffffffu, sum);
    const int total = sum * units_per_seq;
    const int grid = int(gridDim.x);
    per = max(1, (total + grid - 1) / grid);
    cur = int(min(int64_t(total), int64_t(blockIdx.x) * per));
    end = min(total, cur + per);
    b = u = t = len = nt = 0;
    if (cur >= end) return;
    int base = 0;
    for (int i0 = 0; i0 < B; i0 += 32) {
      const int n = i0 + lane < B ? length(i0 + lane) : 0;
      int incl = tiles(n) * units_per_seq;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += v;
      }
      const unsigned past = __ballot_sync(0xffffffffu, base + incl > cur);
      if (past) {
        const int l = __ffs(int(past)) - 1;
        b = i0 + l;
        len = __shfl_sync(0xffffffffu, n, l);
        nt = tiles(len);
        const int r = cur - (base + __shfl_sync(0xffffffffu, incl, l) - nt * units_per_seq);
        u = r / nt;
        t = r - u * nt;
        return;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
  }

  // One unit per cluster, its tiles shared out evenly over the cluster's CTAs.
  __device__ __forceinline__ void init_cluster(const PagedLaunch& a, int tile_keys) {
    lens = a.seq_lens;
    B = a.B;
    cap = a.cap;
    tk = tile_keys;
    groups = a.groups;
    units_per_seq = a.Hkv * a.groups;
    per = 0;
    const int unit = int(blockIdx.x) / a.cluster, r = int(blockIdx.x) - unit * a.cluster;
    b = unit / units_per_seq;
    u = unit - b * units_per_seq;
    len = length(b);
    nt = tiles(len);
    t = int(int64_t(nt) * r / a.cluster);
    cur = 0;
    end = int(int64_t(nt) * (r + 1) / a.cluster) - t;
  }

  __device__ __forceinline__ bool next(Part& p) {
    if (cur >= end) return false;
    if (t >= nt) {  // past the unit: the next one, of the next sequence that has tokens
      t = 0;
      if (++u >= units_per_seq) {
        u = 0;
        do {
          if (++b >= B) {  // only if the lengths changed meanwhile
            cur = end;
            return false;
          }
          len = length(b);
          nt = tiles(len);
        } while (nt == 0);
      }
    }
    p.b = b;
    p.kh = u / groups;
    p.grp = u - p.kh * groups;
    p.len = len;
    p.nt = nt;
    p.t0 = t;
    p.t1 = min(nt, t + (end - cur));
    cur += p.t1 - t;
    t = p.t1;
    return true;
  }
};

__device__ __forceinline__ void store_out(const PagedLaunch& a, size_t idx, float v) {
  if (a.out_bf16) static_cast<__nv_bfloat16*>(a.out)[idx] = __float2bfloat16_rn(v);
  else static_cast<__half*>(a.out)[idx] = __float2half_rn(v);
}

__device__ __forceinline__ float2 ld_dsmem_f32x2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}

// Elements idx and idx + 1 (idx even; out is 4-byte aligned).
__device__ __forceinline__ void store_out2(const PagedLaunch& a, size_t idx, float v0, float v1) {
  if (a.out_bf16) *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(a.out) + idx) = __floats2bfloat162_rn(v0, v1);
  else *reinterpret_cast<__half2*>(static_cast<__half*>(a.out) + idx) = __floats2half2_rn(v0, v1);
}

// Two bytes of x (code + 128) as the fp16 numbers 1152 + code.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t x) {
  uint32_t h;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(h) : "r"(x), "r"(0x64646464u), "n"(kSel));
  return h;
}
constexpr uint32_t kMinus1152 = 0xE480E480u;  // two fp16 -1152
constexpr float kProbScale = 32768.f;         // of an fp16 cache's probabilities as MMA operands

// D(16x8, s32) += A(16x32, s8, row) * B(32x8, s8, col).
__device__ __forceinline__ void mma_16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Four q values times the power of two f as three planes of signed bytes: v = hi 65536 + mid 256 + lo, |v| < 2^22.
// x f + 2^23 + 2^22 has the integer v + 2^22 (rounded to nearest) in its mantissa; v + 0x808080 has the digits
// plus 128 in its bytes.
__device__ __forceinline__ void q_planes(const uint2& q, float f, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&q.x));
  const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&q.y));
  auto digits = [&](float z) {
    return uint32_t(__float_as_int(fmaf(z, f, 12582912.f))) + (0x808080u - 0x400000u);
  };
  const uint32_t u0 = digits(x.x), u1 = digits(x.y), u2 = digits(y.x), u3 = digits(y.y);
  const uint32_t p01 = __byte_perm(u0, u1, 0x5140), p23 = __byte_perm(u2, u3, 0x5140);  // lo, lo, mid, mid
  lo = __byte_perm(p01, p23, 0x5410) ^ 0x80808080u;
  mid = __byte_perm(p01, p23, 0x7632) ^ 0x80808080u;
  hi = __byte_perm(__byte_perm(u0, u1, 0x0062), __byte_perm(u2, u3, 0x0062), 0x5410) ^ 0x80808080u;
}

// kNT: column tiles of 8 heads (1: up to 8 heads per unit, 2: up to 16; more heads per KV head take another pass over K and
// V).  64 sequences of 6K to 8K, 8 KV heads, D = 128: fp16 291 us with 8 heads each, 299 with 16, 574 with 17 (floor 288);
// int8 153 us with 8, 230 with 9 and 237 with 16, where two tiles spill 180 bytes, 439 with 17 (floor 146).
// kCl: a thread-block cluster per unit, whose CTAs merge their parts through distributed shared memory.
template <int D, bool kI8, int kNT, bool kCl>
__global__ void __launch_bounds__(kThr, (Cfg<D, kI8>::kCtas)) paged_attn_kernel(const __grid_constant__ PagedLaunch a) {
  using C = Cfg<D, kI8>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((uint32_t(1024) - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kRingBytes);
  uint64_t* empty = full + C::kStages;
  float* sm_m = reinterpret_cast<float*>(smem + C::kRingBytes + C::kBarBytes);  // [kPagedMaxHeads][warps]
  float* sm_l = sm_m + kWarps * kPagedMaxHeads;
  float* sm_o = sm_l + kWarps * kPagedMaxHeads;                // [warps][kMergeHeads][kHeadStride]
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const WaitCtl wc{a.status, a.timeout_ns};

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], kI8 ? 1 + 32 : 1);  // int8: the producer's lanes fetch the scales
      mbar_init(&empty[s], kWarps);
    }
    abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == kWarps && lane == 0) {
    prefetch_tensormap(&a.tmK);
    prefetch_tensormap(&a.tmV);
  }
  __syncthreads();
  pdl_wait_primary();

  Walk walk;
  if constexpr (kCl) walk.init_cluster(a, C::TK);
  else walk.init(a, C::TK);
  Part p;

  // ------------------------------------------------------------ producer
  if (warp == kWarps) {
    int it = 0;
    if (a.debug_skip_loads != 1) {
      const int br = a.box;             // keys per box
      const int nb = C::TK / br;        // boxes per tile: 1, 2, 4 or 8
      constexpr int kKinds = 2 * C::kBlocks;  // copies per box
      const int job_box = lane / kKinds, kind = lane % kKinds;
      const int sc_key = (lane % (C::TK / 8)) * 8;  // int8: 8 scales of K (the lower lanes) or of V
      bool ok = true;
      while (ok && walk.next(p)) {
        const int* row = a.table + int64_t(p.b) * a.table_stride;
        const int first = p.t0 * nb;                                   // boxes counted from the sequence's start
        const int last = min(p.t1 * nb, (p.len + br - 1) / br);        // boxes that hold tokens
        auto page_of = [&](int box) { return box < last ? row[a.page_div.div(box * br)] : 0; };
        int ids = page_of(first + lane), ids_next = page_of(first + 32 + lane), at = 0;
        for (int t = p.t0; t < p.t1 && ok; ++t, ++it, at += nb) {
          if (at == 32) {  // nb divides 32
            ids = ids_next;
            ids_next = page_of(t * nb + 32 + lane);
            at = 0;
          }
          const int st = it % C::kStages;
          if (it >= C::kStages) {
            const bool free_stage = !*reinterpret_cast<volatile int*>(&abort_flag) &&
                                    mbar_wait(&empty[st], ((it / C::kStages) - 1) & 1, wc, kDevTimeoutEmpty);
            if (!__all_sync(0xffffffffu, free_stage)) {
              ok = false;
              break;
            }
          }
          const int boxes = min(nb, last - t * nb);  // a box past the last token is not fetched
          if (lane == 0) mbar_arrive_expect_tx(&full[st], uint32_t(boxes) * br * uint32_t(2 * C::kBlocks * C::RB));
          __syncwarp();
          uint8_t* stage = smem + size_t(st) * C::kStageBytes;
          const int id = __shfl_sync(0xffffffffu, ids, (at + job_box) & 31);
          if (job_box < boxes && !a.debug_skip_loads) {
            const int tok = a.page_div.mod(t * C::TK + job_box * br);
            const bool known = unsigned(id) < unsigned(a.num_pages);
            if (!known && kind == 0) atomicCAS(a.status, kDevOk, kDevBadPage);
            const bool is_v = kind >= C::kBlocks;
            const int blk = kind % C::kBlocks;
            uint8_t* dst = stage + (is_v ? C::kTileBytes : 0) + blk * C::kBlockBytes + job_box * br * C::RB;
            // outside the pool the copy unit writes zeros and reads nothing
            tma_load_4d(dst, is_v ? &a.tmV : &a.tmK, blk * 64, tok, p.kh, known ? id : a.num_pages, &full[st]);
          }
          if constexpr (kI8) {
            // 16-byte pieces of scales, not copies of a box's 32 to 256 bytes: the copy unit's requests are what
            // bounds small pages (D = 64, 16-token pages, B = 64, 4K: 77 us with, 72 us without)
            const int sc_box = sc_key / br;
            const int sid = __shfl_sync(0xffffffffu, ids, (at + sc_box) & 31);
            if (sc_box < boxes && !a.debug_skip_loads) {
              const int pg = unsigned(sid) < unsigned(a.num_pages) ? sid : 0;  // some scales for zero codes
              const int tok = a.page_div.mod(t * C::TK + sc_key);
              const __half* src = lane < C::TK / 8 ? a.Ks + pg * a.ks_page + p.kh * a.ks_head + tok
                                                   : a.Vs + pg * a.vs_page + p.kh * a.vs_head + tok;
              cp_async16(stage + 2 * C::kTileBytes + lane * 16, src);
            }
            cp_async_arrive(&full[st]);
          }
        }
      }
    }
    // The stream's next kernel is let in by a cluster when its last copy is under way, by the line's CTAs only when they
    // leave.  Calls on end (letting it in at the start / here / not at all): cluster, 5 odd int8 sequences 10.1 / 9.5 /
    // 9.5 us, one of 640 tokens 4.9 / 4.8 / 5.2 us (in a graph); line, 6 sequences of 0 to 5000 tokens 16.0 / 15.3 /
    // 14.4 us, 16 of 0 to 8K 51.6 / 50.6 / 49.9 us.
    if constexpr (kCl) pdl_launch_dependents();
    // The copies in flight land (a bounded wait) before the CTA's memory goes: consumers that gave up do not wait for them,
    // and the loop above does not notice that when they did so behind its last free stage.
    if (lane == 0)
      for (int j = max(0, it - C::kStages); j < it; ++j)
        mbar_wait(&full[j % C::kStages], (j / C::kStages) & 1, wc, kDevTimeoutDrain);
    if constexpr (kCl) {  // the whole warp takes part in the consumers' two cluster barriers
      __syncwarp();
      cluster_sync_all();
      cluster_sync_all();
    }
    return;
  }

  // ------------------------------------------------------------ consumers
  const int g = lane >> 2;   // mma row of S: head g (and g + 8)
  const int t4 = lane & 3;
  const int mi = lane >> 3;  // ldmatrix matrix of this lane
  const int rr = lane & 7;   // and row in it
  const int r0 = warp * C::KPW;  // this warp's first key of a tile
  // this lane's row and chunk parity in the ldmatrix of K (keys by 8, then chunks) and of V (chunks, then keys)
  const uint32_t k_off = blk_off<C::RB>(r0 + ((mi >> 1) << 3) + rr, mi & 1);
  const uint32_t v_off = blk_off<C::RB>(r0 + ((mi & 1) << 3) + rr, mi >> 1);
  const uint32_t ring = smem_u32(smem);
  const int ct = threadIdx.x;
  bool alive = a.debug_skip_loads != 2;
  if (!alive && lane == 0) abort_flag = 1;
  int it = 0;

  // a cluster's CTA leaves its part here, in the ring, when all its tiles have been used
  float* cl_ml = reinterpret_cast<float*>(smem);  // [kPagedMaxHeads][2]: maximum, sum
  float* cl_o = cl_ml + 2 * kPagedMaxHeads;       // [kPagedMaxHeads][D]

  // sequences without tokens: zeros, and no parts
  for (int b = int(blockIdx.x); !kCl && b < a.B; b += int(gridDim.x))
    if (a.seq_lens[b] <= 0) {
      for (int i = ct; i < a.Hq * D; i += 32 * kWarps) store_out(a, size_t(b) * a.Hq * D + i, 0.f);
      const int units = a.Hkv * a.groups;
      if (a.unit_info)
        for (int i = ct; i < units; i += 32 * kWarps) a.unit_info[b * units + i] = make_int2(0, 0);
    }

  while (walk.next(p)) {
    const int h0 = p.kh * a.G + p.grp * a.GP;
    const int gvalid = min(a.GP, a.G - p.grp * a.GP);
    const size_t row_base = size_t(p.b) * a.Hq + h0;

    // Q fragments.  fp16: k = 2t, 2t + 1 and 2t + 8, 2t + 9 of every 16 dimensions.  int8: the planes of dimensions
    // 4t .. 4t + 3 and 16 + 4t .. of every 32.
    constexpr int kQ = kI8 ? (kNT == 1 ? 6 : 12) : 2 * kNT, kQS = kI8 ? D / 32 : D / 16;
    uint32_t qa[kQS][kQ];
    float q_scale[kNT];  // int8: softmax scale over the head's fixed-point unit
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      const bool on = g + 8 * nt < gvalid;
      const __half* qrow = static_cast<const __half*>(a.q) + (row_base + g + 8 * nt) * D;
      if constexpr (!kI8) {
#pragma unroll
        for (int kk = 0; kk < kQS; ++kk) {
          qa[kk][2 * nt] = on ? *reinterpret_cast<const uint32_t*>(qrow + 16 * kk + 2 * t4) : 0u;
          qa[kk][2 * nt + 1] = on ? *reinterpret_cast<const uint32_t*>(qrow + 16 * kk + 2 * t4 + 8) : 0u;
        }
      } else {
        uint2 raw[2 * kQS];
        __half2 top2 = __half2half2(__ushort_as_half(0));  // largest magnitude; a NaN stays one
#pragma unroll
        for (int i = 0; i < 2 * kQS; ++i) {
          raw[i] = make_uint2(0u, 0u);
          if (on) {  // q is 4-byte aligned
            raw[i].x = *reinterpret_cast<const uint32_t*>(qrow + 16 * i + 4 * t4);
            raw[i].y = *reinterpret_cast<const uint32_t*>(qrow + 16 * i + 4 * t4 + 2);
          }
        }
#pragma unroll
        for (int i = 0; i < 2 * kQS; ++i) {
          top2 = __hmax2_nan(top2, __habs2(*reinterpret_cast<const __half2*>(&raw[i].x)));
          top2 = __hmax2_nan(top2, __habs2(*reinterpret_cast<const __half2*>(&raw[i].y)));
        }
        top2 = __hmax2_nan(top2, __shfl_xor_sync(0xffffffffu, top2, 1));
        top2 = __hmax2_nan(top2, __shfl_xor_sync(0xffffffffu, top2, 2));
        const __half top1 = __hmax_nan(__low2half(top2), __high2half(top2));
        const uint32_t top = __half_as_ushort(top1) & 0x7fffu;  // inf and NaN: 0x7c00 and above
        // 2^k = 2^(21 - floor(log2 max |q|)), by the exponent field
        const int e = top == 0u ? 127 : (__float_as_int(__half2float(__ushort_as_half(uint16_t(top)))) >> 23);
        const float unit = __int_as_float((127 + 21 + 127 - e) << 23);
        q_scale[nt] = top >= 0x7c00u ? __int_as_float(0x7fc00000) : a.sm_scale_log2 / unit;
#pragma unroll
        for (int kk = 0; kk < kQS; ++kk) {
          uint32_t hi[2], mid[2], lo[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) q_planes(raw[2 * kk + i], unit, hi[i], mid[i], lo[i]);
          if constexpr (kNT == 1) {
            qa[kk][0] = hi[0];
            qa[kk][1] = mid[0];
            qa[kk][2] = hi[1];
            qa[kk][3] = mid[1];
            qa[kk][4] = lo[0];
            qa[kk][5] = lo[1];
          } else {
            qa[kk][nt] = hi[0];
            qa[kk][2 + nt] = hi[1];
            qa[kk][4 + nt] = mid[0];
            qa[kk][6 + nt] = mid[1];
            qa[kk][8 + nt] = lo[0];
            qa[kk][10 + nt] = lo[1];
          }
        }
      }
    }
    float o[kNT][D / 16][4];
    float m_run[kNT], l_run[kNT];
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      m_run[nt] = -INFINITY;
      l_run[nt] = 0.f;
#pragma unroll
      for (int dd = 0; dd < D / 16; ++dd) o[nt][dd][0] = o[nt][dd][1] = o[nt][dd][2] = o[nt][dd][3] = 0.f;
    }
    float frame = 0.f;  // int8: the power of two in the probabilities (0: none yet)

    for (int t = p.t0; t < p.t1; ++t, ++it) {
      const int st = it % C::kStages;
      if (alive) {
        const bool ok = mbar_wait(&full[st], (it / C::kStages) & 1, wc, kDevTimeoutFull) &&
                        !*reinterpret_cast<volatile int*>(&abort_flag);
        alive = __all_sync(0xffffffffu, ok);
        if (!alive && lane == 0) abort_flag = 1;
      }
      if (!alive) continue;
      const uint32_t sk = ring + uint32_t(st) * C::kStageBytes;
      const uint32_t sv = sk + C::kTileBytes;
      const __half* scales = reinterpret_cast<const __half*>(smem + size_t(st) * C::kStageBytes + 2 * C::kTileBytes);
      const int k0 = t * C::TK;

      auto tile = [&](auto mask_tag) {
        constexpr bool kMask = decltype(mask_tag)::value;
        constexpr int NJ = C::KPW / 8;
        // ---- S = Q K^T
        float sc[NJ][4];
#pragma unroll
        for (int kb = 0; kb < C::KPW / 16; ++kb) {
          const uint32_t at = sk + k_off + uint32_t(16 * kb * C::RB);
          if constexpr (!kI8) {
#pragma unroll
            for (int j = 0; j < 2; ++j) sc[2 * kb + j][0] = sc[2 * kb + j][1] = sc[2 * kb + j][2] = sc[2 * kb + j][3] = 0.f;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              uint32_t b[4];
              ldmatrix_x4(chunk_at<D, kI8>(at, kk), b[0], b[1], b[2], b[3]);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                if constexpr (kNT == 1) mma_16816(sc[2 * kb + j], qa[kk][0], 0u, qa[kk][1], 0u, b[2 * j], b[2 * j + 1]);
                else mma_16816(sc[2 * kb + j], qa[kk][0], qa[kk][2], qa[kk][1], qa[kk][3], b[2 * j], b[2 * j + 1]);
              }
            }
          } else {
            constexpr int kAcc = kNT == 1 ? 2 : 3;
            int acc[2][kAcc][4];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int i = 0; i < kAcc; ++i) acc[j][i][0] = acc[j][i][1] = acc[j][i][2] = acc[j][i][3] = 0;
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) {
              uint32_t b[4];  // (keys 0-7, chunk 2 kk), (keys 0-7, 2 kk + 1), (keys 8-15, 2 kk), (keys 8-15, 2 kk + 1)
              ldmatrix_x4(chunk_at<D, kI8>(at, kk), b[0], b[1], b[2], b[3]);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                if constexpr (kNT == 1) {
                  mma_16832(acc[j][0], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], b[2 * j], b[2 * j + 1]);
                  mma_16832(acc[j][1], qa[kk][4], 0u, qa[kk][5], 0u, b[2 * j], b[2 * j + 1]);
                } else {
#pragma unroll
                  for (int i = 0; i < 3; ++i)
                    mma_16832(acc[j][i], qa[kk][4 * i], qa[kk][4 * i + 1], qa[kk][4 * i + 2], qa[kk][4 * i + 3], b[2 * j],
                              b[2 * j + 1]);
                }
              }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 2 * kNT; ++e) {
                const int hi = acc[j][0][e], mid = kNT == 1 ? acc[j][0][2 + e] : acc[j][1][e], lo = acc[j][kAcc - 1][e];
                sc[2 * kb + j][e] = fmaf(float(hi), 65536.f, fmaf(float(mid), 256.f, float(lo)));
              }
          }
        }
        // ---- online softmax in the log2 domain; this lane: heads g (+ 8), keys k0 + r0 + 8j + 2 t4 + e
        float vs[NJ][2];
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int kq = r0 + 8 * j + 2 * t4;
          float2 kf = make_float2(1.f, 1.f);
          if constexpr (kI8) {
            kf = __half22float2(*reinterpret_cast<const __half2*>(scales + kq));
            const float2 vf = __half22float2(*reinterpret_cast<const __half2*>(scales + C::TK + kq));
            vs[j][0] = (!kMask || k0 + kq < p.len) ? vf.x : 0.f;
            vs[j][1] = (!kMask || k0 + kq + 1 < p.len) ? vf.y : 0.f;
          }
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt) {
            const float qs = kI8 ? q_scale[nt] : a.sm_scale_log2;
            sc[j][2 * nt] = (!kMask || k0 + kq < p.len) ? sc[j][2 * nt] * (kI8 ? qs * kf.x : qs) : -INFINITY;
            sc[j][2 * nt + 1] = (!kMask || k0 + kq + 1 < p.len) ? sc[j][2 * nt + 1] * (kI8 ? qs * kf.y : qs) : -INFINITY;
          }
          if (!kCl && a.scores) {  // (with weights the work is never split by clusters)
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
              if (g + 8 * nt < gvalid && (!kMask || k0 + kq < p.len))  // cap is even: the pair stays in the row
                *reinterpret_cast<float2*>(a.scores + (row_base + g + 8 * nt) * size_t(a.cap) + k0 + kq) =
                    make_float2(sc[j][2 * nt], sc[j][2 * nt + 1]);
          }
        }
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt) {
          float mx = -INFINITY;
#pragma unroll
          for (int j = 0; j < NJ; ++j) mx = fmaxf(mx, fmaxf(sc[j][2 * nt], sc[j][2 * nt + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float m_new = fmaxf(m_run[nt], mx);
          if (__any_sync(0xffffffffu, m_new > m_run[nt])) {
            const float alpha = (m_new == -INFINITY) ? 1.f : ex2(m_run[nt] - m_new);
            // O^T's columns are heads 2 t4 and 2 t4 + 1
            const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t4);
            const float a1 = __shfl_sync(0xffffffffu, alpha, 8 * t4 + 4);
#pragma unroll
            for (int dd = 0; dd < D / 16; ++dd) {
              o[nt][dd][0] *= a0;
              o[nt][dd][1] *= a1;
              o[nt][dd][2] *= a0;
              o[nt][dd][3] *= a1;
            }
            l_run[nt] *= alpha;
            m_run[nt] = m_new;
          }
          const float mu = (m_run[nt] == -INFINITY) ? 0.f : m_run[nt];
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            sc[j][2 * nt] = ex2(sc[j][2 * nt] - mu);
            sc[j][2 * nt + 1] = ex2(sc[j][2 * nt + 1] - mu);
            l_run[nt] += sc[j][2 * nt] + sc[j][2 * nt + 1];
          }
        }
        if constexpr (kI8) {
          float vmax = 0.f;
#pragma unroll
          for (int j = 0; j < NJ; ++j) vmax = fmaxf(vmax, fmaxf(fabsf(vs[j][0]), fabsf(vs[j][1])));  // either sign
          vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 1));
          vmax = fmaxf(vmax, __shfl_xor_sync(0xffffffffu, vmax, 2));  // the same in every lane
          if (vmax * frame >= 16384.f || (frame == 0.f && vmax > 0.f)) {
            float k;
            const float f = frame_for(vmax, k);
            const float r = frame == 0.f ? 0.f : f / frame;  // powers of two; O is 0 before the first frame
            frame = f;
#pragma unroll
            for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
              for (int dd = 0; dd < D / 16; ++dd)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[nt][dd][e] *= r;
          }
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            vs[j][0] *= frame;
            vs[j][1] *= frame;
          }
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int kb = 0; kb < C::KPW / 16; ++kb) {
          uint32_t pb[kNT][2];
#pragma unroll
          for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float* s2 = &sc[2 * kb + i][2 * nt];
              pb[nt][i] = kI8 ? pack_half2(s2[0] * vs[2 * kb + i][0], s2[1] * vs[2 * kb + i][1])
                              : pack_half2(s2[0] * kProbScale, s2[1] * kProbScale);
            }
          const uint32_t at = sv + v_off + uint32_t(16 * kb * C::RB);
          if constexpr (!kI8) {
            // The slots past the last token may hold anything, and 0 * inf is NaN: they are masked to zero.
            uint32_t vm0 = 0xffffffffu, vm1 = 0xffffffffu;
            if constexpr (kMask) {
              const int kq = k0 + r0 + 16 * kb + 2 * t4;
              vm0 = (kq < p.len ? 0x0000ffffu : 0u) | (kq + 1 < p.len ? 0xffff0000u : 0u);
              vm1 = (kq + 8 < p.len ? 0x0000ffffu : 0u) | (kq + 9 < p.len ? 0xffff0000u : 0u);
            }
#pragma unroll
            for (int dd = 0; dd < D / 16; ++dd) {
              uint32_t v0, v1, v2, v3;  // (keys 0-7, dims 0-7), (keys 8-15, dims 0-7), (0-7, 8-15), (8-15, 8-15)
              ldmatrix_x4_trans(chunk_at<D, kI8>(at, dd), v0, v1, v2, v3);
              if constexpr (kMask) {
                v0 &= vm0;
                v1 &= vm1;
                v2 &= vm0;
                v3 &= vm1;
              }
#pragma unroll
              for (int nt = 0; nt < kNT; ++nt) mma_16816(o[nt][dd], v0, v2, v1, v3, pb[nt][0], pb[nt][1]);
            }
          } else {
            // a transposed 8 x 16-byte matrix: keys 2 t4, 2 t4 + 1 of dimensions 2g, 2g + 1; row g of the MMA
            // is dimension 2g, row g + 8 is 2g + 1
#pragma unroll
            for (int dd = 0; dd < D / 16; dd += 2) {
              uint32_t v[4];  // (keys 0-7, chunk dd), (keys 8-15, dd), (0-7, dd + 1), (8-15, dd + 1)
              ldmatrix_x4_trans(chunk_at<D, kI8>(at, dd / 2), v[0], v[1], v[2], v[3]);
#pragma unroll
              for (int i = 0; i < 4; ++i) v[i] ^= 0x80808080u;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t lo0 = codes_to_half2<0x4240>(v[2 * i]), hi0 = codes_to_half2<0x4341>(v[2 * i]);
                const uint32_t lo1 = codes_to_half2<0x4240>(v[2 * i + 1]), hi1 = codes_to_half2<0x4341>(v[2 * i + 1]);
#pragma unroll
                for (int nt = 0; nt < kNT; ++nt) {
                  mma_16816(o[nt][dd + i], lo0, hi0, lo1, hi1, pb[nt][0], pb[nt][1]);
                  mma_16816(o[nt][dd + i], kMinus1152, kMinus1152, kMinus1152, kMinus1152, pb[nt][0], pb[nt][1]);
                }
              }
            }
          }
        }
      };
      if (k0 + C::TK <= p.len) tile(std::false_type{});
      else tile(std::true_type{});
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }

    // ---- end of the part: merge the warps; write the output (a whole unit) or one part of it
    const bool whole = p.t0 == 0 && p.t1 == p.nt;
    const size_t slot = size_t(blockIdx.x) * 2 + (p.t0 == 0 ? 1 : 0);
    const float unframe = !kI8 ? 1.f / kProbScale : frame != 0.f ? 1.f / frame : 1.f;
#pragma unroll
    for (int nt = 0; nt < kNT; ++nt) {
      float l = l_run[nt];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if (t4 == 0) {
        sm_m[(g + 8 * nt) * kWarps + warp] = m_run[nt];
        sm_l[(g + 8 * nt) * kWarps + warp] = l;
      }
    }
    for (int hp = 0; hp < gvalid; hp += kMergeHeads) {
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int hl = 8 * nt + 2 * t4 + e - hp;
          if (hl >= 0 && hl < kMergeHeads) {
            float* dst = sm_o + (warp * kMergeHeads + hl) * C::kHeadStride + (kI8 ? 2 * g : g);
#pragma unroll
            for (int dd = 0; dd < D / 16; ++dd) {
              dst[16 * dd] = o[nt][dd][e] * unframe;
              dst[16 * dd + (kI8 ? 1 : 8)] = o[nt][dd][2 + e] * unframe;
            }
          }
        }
      }
      named_bar_sync(1, 32 * kWarps);
      // a warp per head, D / 32 dimensions per lane
      static_assert(kMergeHeads == kWarps, "one head of a pass per warp");
      const int hh = hp + warp;
      if (hh < gvalid) {
        constexpr int kDims = D / 32;
        const float4 m4 = *reinterpret_cast<const float4*>(sm_m + hh * kWarps);
        const float4 l4 = *reinterpret_cast<const float4*>(sm_l + hh * kWarps);
        const float M = fmaxf(fmaxf(m4.x, m4.y), fmaxf(m4.z, m4.w));
        // a warp whose keys all lie past the last token has no say (its sums are 0; a NaN there stays a NaN)
        auto weight = [&](float m) { return m == -INFINITY ? (M == -INFINITY ? 1.f : 0.f) : ex2(m - M); };
        const float wt[kWarps] = {weight(m4.x), weight(m4.y), weight(m4.z), weight(m4.w)};
        const float L = wt[0] * l4.x + wt[1] * l4.y + wt[2] * l4.z + wt[3] * l4.w;
        float O[kDims];
#pragma unroll
        for (int i = 0; i < kDims; ++i) O[i] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float* src = sm_o + (w * kMergeHeads + warp) * C::kHeadStride + lane * kDims;
          float v[kDims];
          if constexpr (kDims == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
          else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
#pragma unroll
          for (int i = 0; i < kDims; ++i) O[i] += wt[w] * v[i];
        }
        if constexpr (kCl) {
          if (alive) {  // this warp has seen every tile arrive, so no copy is on its way into the ring
            if (lane == 0) *reinterpret_cast<float2*>(cl_ml + 2 * hh) = make_float2(M, L);
            float* dst = cl_o + hh * D + lane * kDims;
            if constexpr (kDims == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(O);
            else *reinterpret_cast<float2*>(dst) = *reinterpret_cast<const float2*>(O);
          }
        } else if (whole) {
          const float r = 1.f / L;
#pragma unroll
          for (int i = 0; i < kDims; i += 2) store_out2(a, (row_base + hh) * D + lane * kDims + i, O[i] * r, O[i + 1] * r);
          if (lane == 0 && a.scores) a.row_ml[row_base + hh] = make_float2(M, L);
        } else {
          if (lane == 0) a.part_ml[slot * a.GP + hh] = make_float2(M, L);
          float* dst = a.part_o + (slot * a.GP + hh) * D + lane * kDims;
          if constexpr (kDims == 4) *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(O);
          else *reinterpret_cast<float2*>(dst) = *reinterpret_cast<const float2*>(O);
        }
      }
      named_bar_sync(1, 32 * kWarps);
    }
    // the CTA that a unit begins in says in how many parts it comes, and from which CTA on
    if (!kCl && p.t0 == 0 && ct == 0 && a.unit_info) {
      const int more = p.nt - p.t1;
      a.unit_info[(p.b * a.Hkv + p.kh) * a.groups + p.grp] =
          make_int2(int(blockIdx.x), more ? 1 + (more + walk.per - 1) / walk.per : 0);
    }
  }
  if constexpr (kCl) {
    const int S = a.cluster, r = int(cluster_ctarank());
    const int gvalid = min(a.GP, a.G - (walk.u % a.groups) * a.GP);
    const size_t row_base = size_t(walk.b) * a.Hq + size_t(walk.u / a.groups) * a.G + size_t(walk.u % a.groups) * a.GP;
    // a CTA without tiles has the sum -1, which no other can have; its outputs are never written
    if (walk.end == 0 && ct < gvalid) *reinterpret_cast<float2*>(cl_ml + 2 * ct) = make_float2(-INFINITY, -1.f);
    cluster_sync_all();
    // the outputs, two dimensions at a time, shared out over the cluster; parts always in CTA order
    for (int i = r * (32 * kWarps) + ct; i < gvalid * (D / 2); i += S * 32 * kWarps) {
      const int hh = i / (D / 2), d = 2 * (i - hh * (D / 2));
      const uint32_t ml_at = smem_u32(cl_ml + 2 * hh), o_at = smem_u32(cl_o + hh * D + d);
      float2 ml[kMaxCluster], o[kMaxCluster];
      float M = -INFINITY;
#pragma unroll
      for (int j = 0; j < kMaxCluster; ++j) {
        ml[j] = make_float2(-INFINITY, -1.f);
        o[j] = make_float2(0.f, 0.f);
        if (j < S) {
          ml[j] = ld_dsmem_f32x2(dsmem_addr(ml_at, j));
          o[j] = ld_dsmem_f32x2(dsmem_addr(o_at, j));
        }
        M = fmaxf(M, ml[j].x);
      }
      float L = 0.f;
      float2 O = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < kMaxCluster; ++j) {
        if (ml[j].y == -1.f) continue;
        const float w = M == -INFINITY ? 1.f : ex2(ml[j].x - M);
        L += w * ml[j].y;
        O.x += w * o[j].x;
        O.y += w * o[j].y;
      }
      const bool none = walk.len == 0;  // an empty sequence: zeros
      store_out2(a, (row_base + hh) * D + d, none ? 0.f : O.x / L, none ? 0.f : O.y / L);
    }
    cluster_sync_all();  // nobody leaves while its part is read
  }
}

// ------------------------------------------------------------------ the rest of a call
// One launch after the attention.  Its first blocks merge the units that came in parts: part s of a unit is
// slot 1 of CTA info.x (s = 0) or slot 0 of CTA info.x + s, always taken in this order.  The other blocks, if
// weights are accumulated, add the softmax weights of a stretch of tokens of one (sequence, KV head); they merge
// the parts' maxima and sums for themselves, so that nothing waits for a third launch.
constexpr int kFinishThreads = 256;
constexpr int kFinishWarps = kFinishThreads / 32;

// A unit's parts, none if it was finished in one CTA.  (Lengths that another stream changes during a call could leave
// an entry unwritten; then nothing is followed.)
__device__ __forceinline__ int2 parts_of(const PagedLaunch& a, int unit) {
  const int2 info = a.unit_info[unit];
  const bool legal = info.x >= 0 && info.y >= 0 && info.x < a.grid && info.y <= a.grid - info.x;
  return legal ? info : make_int2(0, 0);
}
__device__ __forceinline__ size_t part_slot(const int2& info, int s) { return (size_t(info.x) + s) * 2 + (s == 0 ? 1 : 0); }

// Maximum and sum of a head over a unit's parts, by one warp; every lane gets both.
__device__ __forceinline__ float2 merge_ml(const PagedLaunch& a, const int2& info, int h) {
  const int lane = threadIdx.x & 31;
  float M = -INFINITY, L = 0.f;
  for (int s = lane; s < info.y; s += 32) {
    const float2 ml = a.part_ml[part_slot(info, s) * a.GP + h];
    const float Mn = fmaxf(M, ml.x);
    L = (Mn == -INFINITY) ? L + ml.y : L * ex2(M - Mn) + ml.y * ex2(ml.x - Mn);
    M = Mn;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float Mo = __shfl_xor_sync(0xffffffffu, M, off), Lo = __shfl_xor_sync(0xffffffffu, L, off);
    const float Mn = fmaxf(M, Mo);
    L = (Mn == -INFINITY) ? L + Lo : L * ex2(M - Mn) + Lo * ex2(Mo - Mn);
    M = Mn;
  }
  return make_float2(M, L);
}

// Merge of `a.merge_heads` heads of one unit, from head h0: the block's warps are shared out over the heads, the warps
// of a head take its parts in turn (4 dimensions per lane; D = 64: half a warp per part), each with its own running
// maximum, so that a part's numbers and its maximum are fetched together.
template <int D>
__device__ void merge_unit(const PagedLaunch& a, const int2& info, int unit, int h0, float* sm_o, float2* sm_ml) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int grp = unit % a.groups, bk = unit / a.groups;
  const int heads = min(min(a.merge_heads, a.GP - h0), a.G - grp * a.GP - h0);  // of this block
  const size_t row0 = size_t(bk / a.Hkv) * a.Hq + size_t(bk % a.Hkv) * a.G + size_t(grp) * a.GP + h0;
  constexpr int kLanes = D / 4, kPer = 32 / kLanes;       // lanes per part, parts per warp and step
  const int share = max(1, kFinishWarps / a.merge_heads);  // warps per head
  const int heads_at_once = kFinishWarps / share;
  const int sub = (warp % share) * kPer + lane / kLanes;  // this lane's place among those of its head and dimension
  const int d = (lane % kLanes) * 4;
  for (int hb = 0; hb < heads; hb += heads_at_once) {
    const int h = hb + warp / share;
    float M = -INFINITY, L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (h < heads) {
#pragma unroll 4
      for (int s = sub; s < info.y; s += share * kPer) {
        const size_t row = part_slot(info, s) * a.GP + h0 + h;
        const float2 ml = a.part_ml[row];
        const float4 o = *reinterpret_cast<const float4*>(a.part_o + row * D + d);
        const float Mn = fmaxf(M, ml.x);
        const float wa = Mn == -INFINITY ? 1.f : ex2(M - Mn), wb = Mn == -INFINITY ? 1.f : ex2(ml.x - Mn);
        M = Mn;
        L = L * wa + ml.y * wb;
        acc.x = acc.x * wa + o.x * wb;
        acc.y = acc.y * wa + o.y * wb;
        acc.z = acc.z * wa + o.z * wb;
        acc.w = acc.w * wa + o.w * wb;
      }
    }
    const int mine = (warp / share) * share * kPer + sub;
    *reinterpret_cast<float4*>(sm_o + mine * D + d) = acc;
    if (d == 0) sm_ml[mine] = make_float2(M, L);
    __syncthreads();
    for (int i = threadIdx.x; i < min(heads_at_once, heads - hb) * D; i += kFinishThreads) {
      const int hh = i / D, e = i - hh * D, first = hh * share * kPer;
      float Mt = -INFINITY, Lt = 0.f, Ot = 0.f;
      for (int k = 0; k < share * kPer; ++k) Mt = fmaxf(Mt, sm_ml[first + k].x);
      for (int k = 0; k < share * kPer; ++k) {
        const float2 ml = sm_ml[first + k];
        const float w = Mt == -INFINITY ? 1.f : ex2(ml.x - Mt);
        Lt += w * ml.y;
        Ot += w * sm_o[(first + k) * D + e];
      }
      store_out(a, (row0 + hb + hh) * D + e, Ot / Lt);
    }
    __syncthreads();
  }
}

// weights[b, kh, j] += sum_h exp2(s[h, j] - M[h]) / L[h], heads in order; 4 tokens per thread.
constexpr int kWeightTokens = 4 * kFinishThreads;

__device__ void add_weights(const PagedLaunch& a, int block, float2* sm_ml) {
  const int chunks = (a.cap + kWeightTokens - 1) / kWeightTokens;
  const int bk = block / chunks, b = bk / a.Hkv, kh = bk - b * a.Hkv;
  const int len = min(a.cap, a.seq_lens[b]);
  const int j0 = (block - bk * chunks) * kWeightTokens;
  if (j0 >= len) return;
  const size_t row = size_t(b) * a.Hq + size_t(kh) * a.G;
  const int j = j0 + 4 * int(threadIdx.x);
  float w[4] = {0.f, 0.f, 0.f, 0.f};
  for (int h0 = 0; h0 < a.G; h0 += kPagedMaxHeads) {  // the heads of a unit at a time
    const int nh = min(kPagedMaxHeads, a.G - h0);
    const int unit = bk * a.groups + h0 / a.GP;
    const int2 info = a.unit_info ? parts_of(a, unit) : make_int2(0, 0);
    for (int h = threadIdx.x >> 5; h < nh; h += kFinishWarps) {
      const float2 ml = info.y ? merge_ml(a, info, h) : a.row_ml[row + h0 + h];
      if ((threadIdx.x & 31) == 0) sm_ml[h] = make_float2(ml.x, 1.f / ml.y);
    }
    __syncthreads();
    if (j < len) {
#pragma unroll 4
      for (int h = 0; h < nh; ++h) {
        // cap and j are multiples of 4; what lies past the length is read but not used
        const float4 s = *reinterpret_cast<const float4*>(a.scores + (row + h0 + h) * size_t(a.cap) + j);
        const float2 ml = sm_ml[h];
        w[0] += ex2(s.x - ml.x) * ml.y;
        w[1] += ex2(s.y - ml.x) * ml.y;
        w[2] += ex2(s.z - ml.x) * ml.y;
        w[3] += ex2(s.w - ml.x) * ml.y;
      }
    }
    __syncthreads();
  }
  if (j >= len) return;
  float* dst = a.weights + (size_t(b) * a.Hkv + kh) * size_t(a.cap) + j;
  if (j + 4 <= len) {
    float4 old = *reinterpret_cast<const float4*>(dst);
    *reinterpret_cast<float4*>(dst) = make_float4(old.x + w[0], old.y + w[1], old.z + w[2], old.w + w[3]);
  } else {
    for (int i = 0; i < len - j; ++i) dst[i] += w[i];
  }
}

template <int D>
__global__ void __launch_bounds__(kFinishThreads) paged_finish_kernel(const __grid_constant__ PagedLaunch a) {
  __shared__ __align__(16) float sm_o[kFinishThreads * 4];
  __shared__ float2 sm_ml[kPagedMaxHeads];  // merge: two per warp
  pdl_launch_dependents();
  pdl_wait_primary();
  if (int(blockIdx.x) >= a.merge_blocks) {
    add_weights(a, int(blockIdx.x) - a.merge_blocks, sm_ml);
    return;
  }
  const int per_unit = (a.GP + a.merge_heads - 1) / a.merge_heads;
  const int unit = int(blockIdx.x) / per_unit;
  const int2 info = parts_of(a, unit);
  if (info.y) merge_unit<D>(a, info, unit, (int(blockIdx.x) - unit * per_unit) * a.merge_heads, sm_o, sm_ml);
}

template <int D, bool kI8>
cudaError_t prepare(PagedOccupancy (&occ)[2]) {
  constexpr size_t smem = Cfg<D, kI8>::kSmemBytes;
  const void* fn[2][2] = {{reinterpret_cast<const void*>(&paged_attn_kernel<D, kI8, 1, false>),
                           reinterpret_cast<const void*>(&paged_attn_kernel<D, kI8, 1, true>)},
                          {reinterpret_cast<const void*>(&paged_attn_kernel<D, kI8, 2, false>),
                           reinterpret_cast<const void*>(&paged_attn_kernel<D, kI8, 2, true>)}};
  for (int i = 0; i < 2; ++i) {
    cudaError_t e = cudaSuccess;
    for (int cl = 0; cl < 2 && e == cudaSuccess; ++cl)
      e = cudaFuncSetAttribute(fn[i][cl], cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(fn[i][1], cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&occ[i].ctas_per_sm, fn[i][0], kThr, smem);
    if (e != cudaSuccess) return e;
    for (int k = 0; k < 4; ++k) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2u << k);
      cfg.blockDim = dim3(kThr);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 2u << k;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, fn[i][1], &cfg) != cudaSuccess) {
        cudaGetLastError();  // an unsupported size is not an error of the library
        n = 0;
      }
      occ[i].clusters[k] = n;
    }
  }
  return cudaSuccess;
}

template <int D, bool kI8, int kNT>
cudaError_t launch_nt(const PagedLaunch& a, cudaStream_t stream) {
  constexpr size_t smem = Cfg<D, kI8>::kSmemBytes;
  if (!a.cluster) return launch_pdl(paged_attn_kernel<D, kI8, kNT, false>, dim3(a.grid), dim3(kThr), smem, stream, a);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.grid);
  cfg.blockDim = dim3(kThr);
  cfg.dynamicSmemBytes = smem;
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
  return cudaLaunchKernelEx(&cfg, paged_attn_kernel<D, kI8, kNT, true>, a);
}

template <int D, bool kI8>
cudaError_t launch(const PagedLaunch& a, cudaStream_t stream) {
  static_assert((2 * kPagedMaxHeads + kPagedMaxHeads * D) * sizeof(float) <= Cfg<D, kI8>::kRingBytes, "a part fits the ring");
  return a.GP > 8 ? launch_nt<D, kI8, 2>(a, stream) : launch_nt<D, kI8, 1>(a, stream);
}

}  // namespace

int paged_tile_keys(bool int8) { return int8 ? Cfg<128, true>::TK : Cfg<128, false>::TK; }

cudaError_t paged_attn_prepare(bool int8, int D, PagedOccupancy (&occ)[2]) {
  if (int8) return D == 128 ? prepare<128, true>(occ) : prepare<64, true>(occ);
  return D == 128 ? prepare<128, false>(occ) : prepare<64, false>(occ);
}

cudaError_t launch_paged_attn(const PagedLaunch& a, cudaStream_t stream) {
  cudaError_t e;
  if (a.int8) e = a.D == 128 ? launch<128, true>(a, stream) : launch<64, true>(a, stream);
  else e = a.D == 128 ? launch<128, false>(a, stream) : launch<64, false>(a, stream);
  if (e == cudaSuccess && (a.unit_info || a.scores)) {
    const int chunks = a.scores ? (a.cap + kWeightTokens - 1) / kWeightTokens : 0;
    const dim3 grid(unsigned(a.merge_blocks) + unsigned(a.B * a.Hkv) * unsigned(chunks));
    e = a.D == 128 ? launch_pdl(paged_finish_kernel<128>, grid, dim3(kFinishThreads), 0, stream, a)
                   : launch_pdl(paged_finish_kernel<64>, grid, dim3(kFinishThreads), 0, stream, a);
  }
  return e;
}

}  // namespace fqkv
