// Block-sparse decode attention over the paged KV pool  cache[page, layer, {k,v}, kv_head, 16, row]:
//   qk_norm_rope_kv_write   q / k RMSNorm, RoPE and the KV page write of new tokens in one
//                           pass, with the key bounds (elementwise min and max of the
//                           stored keys) of every page written
//   select_pages            per (query row, kv head) the pages worth reading, by an upper
//                           bound of the group's scores computed from the key bounds
//   paged_attention_selected  attention of every query row over its selected pages
// Key bounds: bounds[page, layer, kv_head, {min,max}, D], bf16, or e4m3 codes for fp8
// pools (the pool's scale is positive and common to a head, so it does not change an order).
//
// Reference parity: none (the reference reads the whole cache in every decode step).
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "vrm_common.cuh"
#include "vrm_host.h"
#include "vrm_kernels.h"

namespace vrm {

namespace {

constexpr int kPageTok = 16;

// 4, 8 or 16 bytes that are used once: not kept in L1.  Volatile: loads stay where they are
// written, ahead of the arithmetic that hides their latency.
template <int N>
__device__ __forceinline__ void ld_stream(uint32_t* v, const void* p) {
  if constexpr (N == 16)
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "l"(p));
  else if constexpr (N == 8)
    asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "l"(p));
  else
    asm volatile("ld.global.L1::no_allocate.b32 %0, [%1];" : "=r"(v[0]) : "l"(p));
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the e4m3 pair in the low half of v (exact)
__device__ __forceinline__ uint32_t fp8x2_to_half2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)v));
  return r;
}
// the four e4m3 of v (exact)
__device__ __forceinline__ void fp8x4_to_half4(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The sequence of query row t and the tokens the row sees.  Without cu_q rows are
// sequences; with it rows cu_q[b] .. cu_q[b + 1] - 1 are the last tokens of sequence b.
// False: the row lies behind the last sequence.  Called by whole warps.
struct RowOf {
  int seq, n;
};
__device__ __forceinline__ bool find_row(int t, const int* cu_q, const int* context_lens, int B, RowOf& r) {
  if (cu_q == nullptr) {
    r.seq = t;
    r.n = context_lens[t];
    return true;
  }
  const int lane = threadIdx.x & 31;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int b = b0 + lane;
    int lo = 0, hi = 0;
    if (b < B) {
      lo = cu_q[b];
      hi = cu_q[b + 1];
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, b < B && lo <= t && t < hi);
    if (hit) {
      const int src = __ffs(hit) - 1;
      r.seq = b0 + src;
      r.n = context_lens[r.seq] - (__shfl_sync(0xffffffffu, hi, src) - 1 - t);
      return true;
    }
  }
  return false;
}

}  // namespace

// ================================================================ append
// Rows are handled by D / 16 lanes, 16 dims each: dims [8j, 8j + 8) and the same of the
// other half of the head, so that with a rotation over the whole head both dims of every
// rotated pair sit in one lane; a 128-thread block takes kRows rows at a time.
// A block takes a group of q heads or of v heads of a tile of kRows tokens, or one k head of
// a k tile.  With key bounds a k block owns the runs (maximal sequences of adjacent tokens
// in rising slots of one page) that begin in its tile, wherever they end, so every
// page's bounds have one writer and do not depend on the order of the blocks.
//
// Bound by memory for prompts (8192 tokens, 32 + 4 heads: 30.2 us, 5.7 TB/s; with 2 or 8 heads'
// rows in flight a lane instead of 4 35.1 and 35.2 us), by the chain of dependent loads for
// decode steps (1 row 2.9 us, 64 rows of fp8 pages 4.5 us).  Slower forms, 32 + 8 heads: 8192
// tokens with a rotation of half the head 96.7 us (whole head 39.5: each pair passes through
// shared memory), four-bit pages 50.1 (1 row 6.8, 64 rows 10.9: two divisions a value).
template <int D>
struct AppendShape {
  static constexpr int kLanes = D / 16;            // lanes of a row
  static constexpr int kRows = 128 / kLanes;       // rows of a block pass
  static constexpr int kSpan = kRows + kPageTok;   // tokens of a k block (the last run may leave the tile)
};

enum : int { kRotNone = 0, kRotFull = 1, kRotPart = 2 };

// x (16 dims of a row per lane) -> RMSNorm with weight w (null: none), then the rotation
template <int D, int ROT>
__device__ __forceinline__ void norm_rotate(float (&x)[16], const __nv_bfloat16* w, float eps, int j,
                                            const float (&cs)[16], const float* cs_row, int rot_dim, float* scratch) {
  constexpr int kLanes = AppendShape<D>::kLanes;
  if (w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss * (1.f / D) + eps);
    const uint4 wa = *reinterpret_cast<const uint4*>(w + 8 * j);
    const uint4 wb = *reinterpret_cast<const uint4*>(w + D / 2 + 8 * j);
    const uint32_t ws[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[2 * i] *= r * bf16_lo(ws[i]);
      x[2 * i + 1] *= r * bf16_hi(ws[i]);
    }
  }
  if constexpr (ROT == kRotFull) {
#pragma unroll
    for (int i = 0; i < 8; ++i) rope_rotate(x[i], x[8 + i], cs[i], cs[8 + i], x[i], x[8 + i]);
  } else if constexpr (ROT == kRotPart) {
    // the partner of a dim sits in another lane: exchange through the row's scratch
#pragma unroll
    for (int i = 0; i < 16; ++i) scratch[(i < 8 ? 0 : D / 2 - 8) + 8 * j + i] = x[i];
    __syncwarp();
    const int half = rot_dim / 2;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int d = (i < 8 ? 0 : D / 2 - 8) + 8 * j + i;
      float a, b;
      if (d < half) {
        rope_rotate(x[i], scratch[d + half], cs_row[d], cs_row[half + d], a, b);
        x[i] = a;
      } else if (d < rot_dim) {
        rope_rotate(scratch[d - half], x[i], cs_row[d - half], cs_row[d], a, b);
        x[i] = b;
      }
    }
    __syncwarp();
  }
}

__device__ __forceinline__ void unpack8(uint4 v, float* x) {
  x[0] = bf16_lo(v.x);
  x[1] = bf16_hi(v.x);
  x[2] = bf16_lo(v.y);
  x[3] = bf16_hi(v.y);
  x[4] = bf16_lo(v.z);
  x[5] = bf16_hi(v.z);
  x[6] = bf16_lo(v.w);
  x[7] = bf16_hi(v.w);
}
__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ uint2 fp8x4_to_half4(uint32_t v) {
  uint2 r;
  fp8x4_to_half4(v, r.x, r.y);
  return r;
}

// One rounding from fp32 to the page format.  dst: the stored row; `on`: this lane's row is
// stored (all lanes take part in the shuffles).  key: the 16 stored values in the 16-bit
// type the bounds are compared in: f16 for fp8 codes, else bf16 (four-bit values are rounded
// to the bounds' type here; rounding is monotone, so it commutes with min and max).
template <int D, int FMT>
__device__ __forceinline__ void store_kv_row(uint8_t* dst, const float (&x)[16], float scale, int j, bool on,
                                             uint4 (&key)[2]) {
  if constexpr (FMT == kFmtBf16) {
    key[0] = pack8(x);
    key[1] = pack8(x + 8);
    if (on) {
      *reinterpret_cast<uint4*>(dst + 16 * j) = key[0];
      *reinterpret_cast<uint4*>(dst + D + 16 * j) = key[1];
    }
  } else if constexpr (FMT == kFmtFp8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = make_float2(__fdiv_rn(x[4 * i], scale), __fdiv_rn(x[4 * i + 1], scale));
      const float2 b = make_float2(__fdiv_rn(x[4 * i + 2], scale), __fdiv_rn(x[4 * i + 3], scale));
      w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
             ((uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16);
    }
    if (on) {
      *reinterpret_cast<uint2*>(dst + 8 * j) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(dst + D / 2 + 8 * j) = make_uint2(w[2], w[3]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint2 a = fp8x4_to_half4(w[2 * i]), b = fp8x4_to_half4(w[2 * i + 1]);
      key[i] = make_uint4(a.x, a.y, b.x, b.y);
    }
  } else {
    // per 32-dim group (four lanes): scale = (max - min) / 15 and min in fp16, codes
    // against those rounded values
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float mn = x[8 * hf], mx = x[8 * hf];
#pragma unroll
      for (int i = 1; i < 8; ++i) {
        mn = fminf(mn, x[8 * hf + i]);
        mx = fmaxf(mx, x[8 * hf + i]);
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      }
      __half hs = __float2half_rn((mx - mn) / 15.f);
      if (!(__half2float(hs) > 0.f)) hs = __float2half_rn(6.103515625e-05f);   // constant group
      const __half hm = __float2half_rn(mn);
      const float s = __half2float(hs), m = __half2float(hm);
      uint32_t packed = 0;
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float cf = fminf(fmaxf(rintf((x[8 * hf + i] - m) / s), 0.f), 15.f);
        packed |= (uint32_t)cf << (4 * i);
        v[i] = fmaf(cf, s, m);
      }
      key[hf] = pack8(v);
      if (on) {
        *reinterpret_cast<uint32_t*>(dst + hf * (D / 4) + 4 * j) = packed;
        if ((j & 3) == 0)
          *reinterpret_cast<__half2*>(dst + D / 2 + (hf * (D / 64) + j / 4) * 4) = __halves2half2(hs, hm);
      }
    }
  }
}

// Eight stored values (dims 8 d8 ..) of a row of a page, in the bounds' 16-bit type
template <int D, int FMT>
__device__ __forceinline__ uint4 load_key8(const uint8_t* row, int d8) {
  if constexpr (FMT == kFmtBf16) {
    return *reinterpret_cast<const uint4*>(row + 16 * d8);
  } else if constexpr (FMT == kFmtFp8) {
    const uint2 w = *reinterpret_cast<const uint2*>(row + 8 * d8);
    const uint2 a = fp8x4_to_half4(w.x), b = fp8x4_to_half4(w.y);
    return make_uint4(a.x, a.y, b.x, b.y);
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(row + 4 * d8);
    const __half2 sm = *reinterpret_cast<const __half2*>(row + D / 2 + (d8 / 4) * 4);
    const float s = __low2float(sm), m = __high2float(sm);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf((float)((w >> (4 * i)) & 15u), s, m);
    return pack8(v);
  }
}

// min / max of 16-bit pairs; a NaN stays
template <int FMT, bool MAX>
__device__ __forceinline__ uint32_t pick2(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (FMT == kFmtFp8) {
    if constexpr (MAX) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  } else {
    if constexpr (MAX) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  }
  return r;
}
template <int FMT, bool MAX>
__device__ __forceinline__ void pick8(uint4& a, const uint4& b) {
  a.x = pick2<FMT, MAX>(a.x, b.x);
  a.y = pick2<FMT, MAX>(a.y, b.y);
  a.z = pick2<FMT, MAX>(a.z, b.z);
  a.w = pick2<FMT, MAX>(a.w, b.w);
}
__device__ __forceinline__ uint4 shfl_xor4(const uint4& v, int o) {
  return make_uint4(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o),
                    __shfl_xor_sync(0xffffffffu, v.z, o), __shfl_xor_sync(0xffffffffu, v.w, o));
}
// stores eight bounds: finite (infinities become the largest value, a NaN `nan`)
template <int FMT>
__device__ __forceinline__ void store_bound8(void* dst, const uint4& v, float nan) {
  constexpr float kMax = FMT == kFmtFp8 ? 448.f : 3.3895313892515355e38f;
  float x[8];
  if constexpr (FMT == kFmtFp8) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  } else {
    unpack8(v, x);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = x[i] != x[i] ? nan * kMax : fminf(fmaxf(x[i], -kMax), kMax);
  if constexpr (FMT == kFmtFp8) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      w[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i], x[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
             ((uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2], x[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16);
    *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  } else {
    *reinterpret_cast<uint4*>(dst) = pack8(x);
  }
}

template <int D, int FMT, int ROT>
__global__ void __launch_bounds__(128) append_kernel(AppendArgs a) {
  using S = AppendShape<D>;
  constexpr int kLanes = S::kLanes, kRows = S::kRows;
  constexpr int kRowB = PageRow<D, FMT>::kBytes;
  constexpr int kHeads = 4;                // heads whose rows are in flight together
  __shared__ float s_rot[ROT == kRotPart ? kRows * D : 1];
  __shared__ uint4 s_key[S::kSpan * (D / 8)];     // stored keys of the block's tokens
  __shared__ int s_slot[S::kSpan + 1];            // [0]: the token before the tile
  __shared__ int s_run[S::kSpan + 1];             // token of each run's start, then the end of the last
  pdl_launch();
  pdl_wait();
  const int tid = threadIdx.x;
  const int j = tid % kLanes, r0 = tid / kLanes;
  // blocks of the q groups, then of the v groups, then of the k heads, tile by tile
  const int tiles = (a.T + kRows - 1) / kRows, qv = tiles * (a.q_groups + a.v_groups);
  const bool is_k = blockIdx.x >= qv;
  const int tile = is_k ? a.k_tile : kRows;
  const int k_tiles = (a.T + a.k_tile - 1) / a.k_tile;
  const int block = is_k ? blockIdx.x - qv : blockIdx.x;
  const int y = is_k ? block / k_tiles : block / tiles;
  const int tile0 = (is_k ? block % k_tiles : block % tiles) * tile;
  const size_t page_b = (size_t)a.num_layers * 2 * a.KH * kPageTok * kRowB;
  float* scratch = s_rot + (ROT == kRotPart ? r0 * D : 0);

  auto load_row = [&](int t, int head, uint4 (&x)[2]) {
    const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(a.qkv) + (size_t)t * a.ld_qkv + (size_t)head * D;
    x[0] = *reinterpret_cast<const uint4*>(src + 8 * j);
    x[1] = *reinterpret_cast<const uint4*>(src + D / 2 + 8 * j);
  };
  // row of the rotation table of token t; with a whole-head rotation this lane's 8 cos, 8 sin
  auto cos_row = [&](int t, float (&cs)[16]) -> const float* {
    if (ROT == kRotNone) return nullptr;
    int p = a.positions[t];
    if (p < 0 || p >= a.max_pos) {           // outside the table: reported, nearest row taken
      report_error(a.err, kErrBounds);
      p = p < 0 ? 0 : a.max_pos - 1;
    }
    const float* row = a.cos_sin + (size_t)p * a.rot_dim;
    if constexpr (ROT == kRotFull) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(row + (i / 2) * (D / 2) + 8 * j + 4 * (i % 2));
        cs[4 * i] = v.x;
        cs[4 * i + 1] = v.y;
        cs[4 * i + 2] = v.z;
        cs[4 * i + 3] = v.w;
      }
    }
    return row;
  };
  auto page_of = [&](int slot) -> int {      // -1: not stored
    if (slot < 0) return -1;
    const int page = slot / kPageTok;
    if (page >= a.num_pages) {
      report_error(a.err, kErrBounds);
      return -1;
    }
    return page;
  };
  auto kv_row = [&](int page, int slot, int kv, int head) -> uint8_t* {
    return reinterpret_cast<uint8_t*>(a.cache) + (size_t)page * page_b +
           ((((size_t)a.layer * 2 + kv) * a.KH + head) * kPageTok + slot % kPageTok) * (size_t)kRowB;
  };

  if (!is_k && y >= a.q_groups) {
    // ---- v heads
    const int gv = y - a.q_groups;
    const int t = tile0 + r0;
    const bool tok = t < a.T;
    const int slot = tok ? a.slots[t] : -1;
    const int h1 = min(a.KH, (gv + 1) * a.heads_per_group);
    for (int h0 = gv * a.heads_per_group; h0 < h1; h0 += kHeads) {
      uint4 in[kHeads][2];
#pragma unroll
      for (int i = 0; i < kHeads; ++i) load_row(tok ? t : tile0, a.Hq + a.KH + min(h0 + i, h1 - 1), in[i]);
      const int page = page_of(slot);
      const bool on = page >= 0;
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        if (h0 + i >= h1) break;
        float x[16];
        unpack8(in[i][0], x);
        unpack8(in[i][1], x + 8);
        const float sc = FMT == kFmtFp8 ? a.kv_scale[(a.layer * 2 + 1) * a.KH + h0 + i] : 1.f;
        uint4 key[2];
        store_kv_row<D, FMT>(on ? kv_row(page, slot, 1, h0 + i) : nullptr, x, sc, j, on, key);
      }
    }
    return;
  }
  if (!is_k) {
    // ---- q heads
    const int t = tile0 + r0;
    const bool on = t < a.T;
    const int ht = on ? t : tile0;           // rows without a token repeat the tile's first
    float cs[16];
    const float* row = cos_row(ht, cs);
    const int h1 = min(a.Hq, (y + 1) * a.heads_per_group);
    for (int h0 = y * a.heads_per_group; h0 < h1; h0 += kHeads) {
      uint4 in[kHeads][2];
#pragma unroll
      for (int i = 0; i < kHeads; ++i) load_row(ht, min(h0 + i, h1 - 1), in[i]);
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        if (h0 + i >= h1) break;
        float x[16];
        unpack8(in[i][0], x);
        unpack8(in[i][1], x + 8);
        norm_rotate<D, ROT>(x, reinterpret_cast<const __nv_bfloat16*>(a.wq), a.eps, j, cs, row, a.rot_dim, scratch);
        if (on) {
          __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.q_out) + (size_t)t * a.ld_out + (size_t)(h0 + i) * D;
          *reinterpret_cast<uint4*>(dst + 8 * j) = pack8(x);
          *reinterpret_cast<uint4*>(dst + D / 2 + 8 * j) = pack8(x + 8);
        }
      }
    }
    return;
  }
  // ---- one k head
  const int h = y;
  const float sc = FMT == kFmtFp8 ? a.kv_scale[(a.layer * 2 + 0) * a.KH + h] : 1.f;
  const int in_tile = min(tile, a.T - tile0);
  uint4 in[2];
  load_row(r0 < in_tile ? tile0 + r0 : tile0, a.Hq + h, in);
  int first = 0, last = in_tile, runs = 0;
  if (a.bounds != nullptr) {
    if (tid <= in_tile + kPageTok - 1) {     // <= kSpan
      const int i = tile0 + tid - 1;
      s_slot[tid] = i >= 0 && i < a.T ? a.slots[i] : -1;
    }
    __syncthreads();
    // starts of runs, tokens in_tile .. in_tile + 14 included: a run has at most 16 tokens
    const int lane = tid & 31;
    uint64_t starts = 0;
#pragma unroll
    for (int k = 0; k < (S::kSpan + 31) / 32; ++k) {
      const int i = 32 * k + lane;
      bool st = true;
      if (i < in_tile + kPageTok - 1 && tile0 + i < a.T) {
        const int prev = s_slot[i], cur = s_slot[i + 1];
        st = !(prev >= 0 && cur > prev && cur / kPageTok == prev / kPageTok);
      }
      starts |= (uint64_t)__ballot_sync(0xffffffffu, st) << (32 * k);
    }
    const uint64_t own = starts & ((1ull << in_tile) - 1);
    runs = __popcll(own);
    first = runs ? __ffsll((long long)own) - 1 : in_tile;
    last = runs ? __ffsll((long long)(starts >> in_tile << in_tile)) - 1 : in_tile;
    if (tid < in_tile && (own >> tid & 1)) s_run[__popcll(own & ((1ull << tid) - 1))] = tid;
    if (tid == 0) s_run[runs] = last;
  }
  for (int b = 0; b < last; b += kRows) {
    const int k = b + r0, t = tile0 + k;     // this row's token
    if (k >= in_tile && k < last) load_row(t, a.Hq + h, in);
    const bool live = k >= first && k < last;
    const int slot = live ? a.slots[t] : -1;
    float cs[16], x[16];
    const float* row = cos_row(live ? t : tile0, cs);
    unpack8(in[0], x);
    unpack8(in[1], x + 8);
    norm_rotate<D, ROT>(x, reinterpret_cast<const __nv_bfloat16*>(a.wk), a.eps, j, cs, row, a.rot_dim, scratch);
    const int page = page_of(slot);
    const bool on = page >= 0;
    uint4 key[2];
    store_kv_row<D, FMT>(on ? kv_row(page, slot, 0, h) : nullptr, x, sc, j, on, key);
    if (a.bounds != nullptr && live) {
      s_key[k * (D / 8) + j] = key[0];
      s_key[k * (D / 8) + D / 16 + j] = key[1];
    }
  }
  if (a.bounds == nullptr) return;
  __syncthreads();
  // ---- bounds: one warp a run, D / 8 lanes a row, rows up to the run's last.  The run's own
  // come from shared memory, the others from the pool (written by earlier calls).
  constexpr int kPer = D / 8, kGroups = 32 / kPer;
  const int lane = tid & 31, d8 = lane % kPer, grp = lane / kPer;
  for (int run = tid / 32; run < runs; run += 4) {
    const int k0 = s_run[run], k1 = s_run[run + 1];
    const int slot = s_slot[k0 + 1];
    const int page = slot >= 0 && slot / kPageTok < a.num_pages ? slot / kPageTok : -1;
    if (page < 0) continue;
    constexpr uint32_t kInf = FMT == kFmtFp8 ? 0x7C007C00u : 0x7F807F80u;
    uint4 lo = make_uint4(kInf, kInf, kInf, kInf), hi = lo;
    hi.x = hi.y = hi.z = hi.w = kInf | 0x80008000u;
    const uint8_t* base = kv_row(page, 0, 0, h);
    const uint32_t rows = __reduce_or_sync(0xffffffffu, k0 + lane < k1 ? 1u << (s_slot[k0 + 1 + lane] % kPageTok) : 0u);
    const uint32_t others = (0xffffffffu >> __clz(rows)) & ~rows;
    if (others != 0) {
#pragma unroll
      for (int r = 0; r < kPageTok; r += kGroups) {
        if (others >> (r + grp) & 1u) {
          const uint4 v = load_key8<D, FMT>(base + (r + grp) * kRowB, d8);
          pick8<FMT, false>(lo, v);
          pick8<FMT, true>(hi, v);
        }
      }
    }
    for (int k = k0 + grp; k < k1; k += kGroups) {
      const uint4 v = s_key[k * (D / 8) + d8];
      pick8<FMT, false>(lo, v);
      pick8<FMT, true>(hi, v);
    }
#pragma unroll
    for (int o = kPer; o < 32; o <<= 1) {
      pick8<FMT, false>(lo, shfl_xor4(lo, o));
      pick8<FMT, true>(hi, shfl_xor4(hi, o));
    }
    if (grp == 0) {
      constexpr int kEl = FMT == kFmtFp8 ? 1 : 2;
      uint8_t* dst = reinterpret_cast<uint8_t*>(a.bounds) +
                     ((((size_t)page * a.num_layers + a.layer) * a.KH + h) * 2 * D + 8 * d8) * kEl;
      store_bound8<FMT>(dst, lo, -1.f);
      store_bound8<FMT>(dst + D * kEl, hi, 1.f);
    }
  }
}

template <int D, int FMT>
static void launch_append(AppendArgs a, cudaStream_t st) {
  // heads of a q or v block: the rotation table's row is read once a block, so as many as
  // leave a block to every SM.  B200, us with 4 / 8 / 16 / 32 heads a block, this rule's choice
  // in brackets, 32 + 8 heads: 512 tokens (4.5) / 5.5 / 8.4 / 12.8, 2048: 12.1 / 10.9 / (12.9) /
  // 20.2, 2400: 13.8 / 12.4 / 13.0 / (22.9), 3251: 17.3 / 16.4 / 15.3 / (21.5), 4096: 22.1 /
  // 20.7 / 19.8 / (22.7), 6144: 32.1 / 30.9 / 30.7 / (28.8), 8192: 42.1 / 41.3 / 40.7 / (39.5).
  // It suits decode steps and long prompts.  From one block an SM (2353 tokens of 128 dims) to
  // about 5000 tokens 8 or 16 heads are faster, by up to 1.8 times (40 + 8 heads: 2.1): there
  // one block an SM is too few.
  const int tiles = (a.T + AppendShape<D>::kRows - 1) / AppendShape<D>::kRows;
  int per = 4;
  while (per < a.Hq && (long long)tiles * ((a.Hq + 2 * per - 1) / (2 * per)) >= device_sm_count()) per *= 2;
  a.heads_per_group = per;
  a.q_groups = (a.Hq + per - 1) / per;
  a.v_groups = (a.KH + per - 1) / per;
  // In a decode step each token is a run whose page is read back, one warp a run: small k
  // tiles spread them.  In a prompt a run has 16 tokens, and most small tiles have none.
  // B200, us with tiles of 4 / 8 / 16: decode of 64 rows (fp8) 4.5 / 6.0 / 8.2, of 512 rows
  // 10.2 / 8.0 / 11.3; prompts of 512 tokens 5.9 / 4.1 / 5.1, of 2048 22.6 / 17.3 / 16.1.
  a.k_tile = a.bounds == nullptr || a.T > 768 ? 16 : a.T > 256 ? 8 : 4;
  const long long k_blocks = (long long)((a.T + a.k_tile - 1) / a.k_tile) * a.KH;
  const long long blocks = k_blocks + (long long)tiles * (a.q_groups + a.v_groups);
  VRM_REQUIRE(blocks <= INT_MAX, "qk_norm_rope_kv_write: too many tokens");
  const dim3 grid((unsigned)blocks);
  if (a.rot_dim == 0) launch_kernel(append_kernel<D, FMT, kRotNone>, grid, dim3(128), 0, st, a);
  else if (a.rot_dim == D) launch_kernel(append_kernel<D, FMT, kRotFull>, grid, dim3(128), 0, st, a);
  else launch_kernel(append_kernel<D, FMT, kRotPart>, grid, dim3(128), 0, st, a);
}

void qk_norm_rope_kv_write(const AppendArgs& in, cudaStream_t st) {
  if (in.T <= 0) return;
  AppendArgs a = in;
  a.err = error_word();
  VRM_REQUIRE(a.D == 64 || a.D == 128, "qk_norm_rope_kv_write: head_dim must be 64 or 128");
  auto go = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (a.fmt == kFmtQ4) launch_append<D, kFmtQ4>(a, st);
    else if (a.fmt == kFmtFp8) launch_append<D, kFmtFp8>(a, st);
    else launch_append<D, kFmtBf16>(a, st);
  };
  if (a.D == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 64>{});
  VRM_CUDA_CHECK(cudaGetLastError());
}

// ================================================================ page selection
// Score of page p for the group's heads g:  sum_d (up_d * max_pd + dn_d * min_pd) with
// up_d = sum_g max(q_gd, 0), dn_d = sum_g min(q_gd, 0): no key of the page gives the group
// a larger sum of scores (four-bit keys: by more than the bounds' rounding to the nearest
// bf16, 2^-8 sum_d (|up_d max_pd| + |dn_d min_pd|)).
//
// Which page is the last to be taken depends on differences of any size, so the choice is
// the one that 64-bit sums make (products of 8-bit significands are exact there), ties to
// the lowest page.  64-bit arithmetic for every page would cost more than reading it, so
// pages are first scored in fp32 by the tensor cores: bounds go from memory to the A operand
// of an MMA as they are (e4m3 as f16), and the query vector is split into three 16-bit
// parts (24 bits of it) that are columns of B.  With S an upper bound of sum |term|, such a
// score is off by less than E = 2^-17 S (two MMAs in turn add 32 exact products and two sums,
// each off by at most 2^-23 of the sum of their magnitudes: 34 * 2^-23 S = 2^-17.9 S over all
// of them, and the fp32 additions of their sums 2^-20 S), so with the need-th largest score b
// every page above b + 2E is taken, every page below b - 2E is not, and the few between are
// scored again in 64 bits.  How an MMA rounds its sum is not documented: 2^-23 a term is an
// assumption, that it keeps at least the 24 places of fp32 below its largest term.  Measured on
// B200 against exact sums (32 products, exponents up to 20 apart, one term or a cancelling pair
// above 31 terms that lose their last places): at most 8.9 * 2^-23 bf16, 7.9 * 2^-23 f16.
// Whatever fp32 cannot decide (S out of range, non-finite values, more pages between than
// kSelList) is decided by 64-bit scores of all pages.
//
// Bound by the reads while pages stream (64 rows of 32k tokens, fp8 bounds: 56.4 us, 4.8 TB/s;
// 23k tokens, bf16: 58.1 us, 5.1 TB/s), but a row's start and choice (about 15k cycles of
// dependent loads, barriers and shared-memory passes) overlap other rows' reads only in part.
namespace {

// A bound becomes a double by moving its sign, exponent and significand bits into place
// without re-biasing the exponent: the same value times 2^-896 (bf16) or 2^-1016 (e4m3),
// zeros and subnormals included; the query side carries 2^800 against underflow.  The
// common factor does not change an order.
__device__ __forceinline__ double hi_word(uint32_t h) { return __hiloint2double((int)h, 0); }

// the two bf16 of w
__device__ __forceinline__ void bf16x2_to_f64(uint32_t w, double& a, double& b) {
  a = hi_word((uint32_t)((int32_t)(w << 16) >> 3) & 0x8FFFE000u);
  b = hi_word((uint32_t)((int32_t)w >> 3) & 0x8FFFE000u);
}
// the four e4m3 of w
__device__ __forceinline__ void fp8x4_to_f64(uint32_t w, double (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = hi_word((uint32_t)((int32_t)(w << (24 - 8 * i)) >> 7) & 0x80FE0000u);
}

// unsigned keys in the order of the values
__device__ __forceinline__ uint64_t sortable(double s) {
  if (s != s) return ~0ull;                      // a NaN is read first: it is not hidden
  const uint64_t b = (uint64_t)__double_as_longlong(s + 0.0);   // -0 counts as 0
  return (b >> 63) ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ uint32_t sortable(float s) {
  const uint32_t b = __float_as_uint(s + 0.f);
  return (b >> 31) ? ~b : b | (1u << 31);
}
__device__ __forceinline__ float from_sortable(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// Pages decided by the short 64-bit path.  An outlier channel makes E large beside the spread
// of the scores: with 32 and one channel 400 times the others, 64 rows of 2048 pages of fp8
// bounds took 471 us instead of 73, 1 row of 24576 pages 1105 instead of 43.  Beyond 128 pages
// all candidates are scored in 64 bits, by one CTA: with bf16 bounds and one channel 4000 times
// the others 1 row of 2048 pages takes 90 us (8 times: 10), of 24576 pages 1235 (86), 64 rows of
// 2048 pages 489 (92).  A key that was infinite, and so has the largest bound, does the same.
constexpr int kSelList = 128;
constexpr int kSelMaxPages = 24576;              // candidate pages of a row (8 bytes of shared memory each)
constexpr int kBins = 1024;

template <int NT>
struct SelectScratch {
  __align__(16) uint32_t hist[kBins];
  uint32_t scan[NT / 32];
  uint64_t red[2][NT / 32];
  uint32_t border, left, in_bin;
};

// Where the need-th largest of a set of keys lies: it shares the bits `mask` of `prefix`,
// and is the left-th largest of the `in_bin` keys that do.
template <typename K>
struct Border {
  K prefix, mask;
  int shift;                                     // lowest bit of mask
  uint32_t left, in_bin;
  // from the largest and the smallest key: the bits they share are settled
  __device__ __forceinline__ void start(K top, K low, uint32_t need, int n) {
    const K differ = top ^ low;
    shift = differ ? 64 - __clzll((unsigned long long)differ) : 0;
    mask = shift >= (int)sizeof(K) * 8 ? (K)0 : (K)(~(K)0 << shift);
    prefix = top & mask;
    left = need;
    in_bin = (uint32_t)n;
  }
};

// One histogram of the bins bin(0) .. bin(n - 1) (-1: not counted): sc.border becomes the bin
// of the left-th entry from the top, which is its sc.left-th of sc.in_bin.  The bins are
// zero before and after.
template <int NT, typename F>
__device__ __forceinline__ void radix_count(SelectScratch<NT>& sc, int n, uint32_t left, F bin) {
  constexpr int kPer = kBins / NT;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i0 = tid; i0 < n; i0 += 8 * NT) {
    int b[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) b[q] = i0 + q * NT < n ? bin(i0 + q * NT) : -1;
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (b[q] >= 0) atomicAdd(&sc.hist[b[q] % kPer * NT + b[q] / kPer], 1u);
  }
  __syncthreads();
  // suffix sums: thread tid adds up the kPer bins below kBins - tid * kPer
  uint32_t c[kPer], sum = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    uint32_t* p = &sc.hist[q * NT + NT - 1 - tid];
    c[q] = *p;
    *p = 0u;
    sum += c[q];
  }
  uint32_t incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) sc.scan[warp] = incl;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) incl += w < warp ? sc.scan[w] : 0u;
  uint32_t before = incl - sum;
  if (before < left && incl >= left) {           // one thread
#pragma unroll
    for (int q = kPer - 1; q >= 0; --q) {
      if (before < left && before + c[q] >= left) {
        sc.border = kBins - (tid + 1) * kPer + q;
        sc.left = left - before;
        sc.in_bin = c[q];
      }
      before += c[q];
    }
  }
  __syncthreads();
}

// Settles up to 10 more bits of the border of keys key(0) .. key(n - 1)
template <int NT, typename K, typename F>
__device__ __forceinline__ void radix_pass(SelectScratch<NT>& sc, int n, F key, Border<K>& b) {
  const int low = max(0, b.shift - 10);
  radix_count<NT>(sc, n, b.left, [&](int i) -> int {
    const K k = key(i);
    return (k & b.mask) == b.prefix ? (int)((k & (K)~b.mask) >> low) : -1;
  });
  b.prefix |= (K)sc.border << low;
  b.left = sc.left;
  b.in_bin = sc.in_bin;
  b.shift = low;
  b.mask = (K)(~(K)0 << low);
  __syncthreads();
}

}  // namespace

// One cluster of 1, 2, 4 or 8 CTAs per (kv head, query row).  Every CTA scores a slice of
// the row's candidate pages; scores go to the shared memory of the cluster's first CTA,
// which chooses.
//
// The MMAs use the bounds as loads deliver them (with pages as plain rows of A each MMA costs
// four register moves, and 64 rows of 23k tokens took 69 us instead of 58): lane (g, c) reads 16-byte pieces c, c + 4, .. of page g, and
// the four words of a piece are the lane's four A registers.  Words 0 and 2 thereby belong
// to row g, words 1 and 3 to row g + 8: a page fills two rows, the query's parts for even
// words are columns 0..2, for odd words columns 3..5, and a page's score is its first row's
// columns 0..2 plus its second row's 3..5.  (e4m3 words become f16 pairs on the way.)  A warp
// holds kTile pages in registers and requests the next ones' pieces as soon as the MMAs have
// used the present ones'.
template <int D, bool F8, int NT>
__global__ void __launch_bounds__(NT, 512 / NT) select_kernel(SelectArgs a) {
  constexpr int kEl = F8 ? 1 : 2;
  constexpr int kPageB = 2 * D * kEl;            // bounds of one page and kv head
  constexpr int kPieces = kPageB / 64;           // 16-byte pieces of a page per lane: minima, then maxima
  constexpr int kSp = F8 ? 2 : 1;                // MMAs a piece feeds
  constexpr int kSteps = kPieces * kSp;          // MMAs of 8 pages
  constexpr int kSub = kPieces == 8 ? 2 : 4, kTile = 8 * kSub;
  constexpr int kWarps = NT / 32;
  extern __shared__ __align__(16) uint8_t s_dyn[];
  float* s_score = reinterpret_cast<float*>(s_dyn);              // [max_pages] fp32 scores
  int* s_page = reinterpret_cast<int*>(s_dyn) + a.max_pages;     // [max_pages] their pages in the pool
  uint64_t* s_key = reinterpret_cast<uint64_t*>(s_dyn);          // or 64-bit keys, over both
  __shared__ SelectScratch<NT> sc;
  __shared__ double s_q[2 * D];                  // dn, up
  __shared__ __align__(8) uint16_t s_part[3][2 * D];             // their three 16-bit parts
  __shared__ float s_norm[2][kWarps];
  __shared__ uint32_t s_ends[8 * kWarps][3];     // per CTA and warp: largest key, ~smallest key, largest |bound|
  __shared__ uint32_t s_cnt[2][kWarps];
  __shared__ uint64_t s_lkey[kSelList];
  __shared__ int s_lidx[kSelList], s_near[kSelList];
  __shared__ float s_lval[kSelList], s_b;
  __shared__ uint32_t s_count, s_nears;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  pdl_launch();
  pdl_wait();
  const int kvh = blockIdx.y, t = blockIdx.z;
  const int nc = gridDim.x, rank = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;

  // the query vector's loads go out beside the load of the row's length
  __nv_bfloat16 qv[8];
#pragma unroll
  for (int h = 0; h < 8; ++h)
    qv[h] = tid < D && h < a.G ? reinterpret_cast<const __nv_bfloat16*>(a.q)[(size_t)t * a.ld_q + (size_t)(kvh * a.G + h) * D + tid]
                               : __nv_bfloat16(0.f);
  for (int i = tid; i < kBins / 4; i += NT) reinterpret_cast<uint4*>(sc.hist)[i] = make_uint4(0u, 0u, 0u, 0u);
  // and, where the warp's first pages do not depend on it, beside its block-table entries
  const bool early = nc == 1 && a.cu_q == nullptr;
  const int first = a.sinks + warp * kTile + lane;
  const int early_entry = early && lane < kTile && first < a.max_pages ? a.block_tables[(size_t)t * a.bt_stride + first] : 0;
  RowOf row;
  if (!find_row(t, a.cu_q, a.context_lens, a.B, row)) return;      // the same for the whole cluster
  int* out = a.out + ((size_t)t * a.KH + kvh) * a.budget;
  int total = row.n <= 0 ? 0 : (int)(((long long)row.n + kPageTok - 1) / kPageTok);
  total = min(total, a.max_pages);
  if (total <= a.budget) {
    for (int i = rank * NT + tid; i < a.budget; i += nc * NT) out[i] = i < total ? i : -1;
    return;
  }
  const int need = a.budget - a.sinks - a.recent;
  const int n = total - a.sinks - a.recent;      // candidates: pages sinks .. sinks + n - 1, n > need
  if (rank == 0) {
    for (int i = tid; i < a.sinks; i += NT) out[i] = i;
    for (int i = tid; i < a.recent; i += NT) out[a.budget - a.recent + i] = total - a.recent + i;
  }
  if (need <= 0) return;
  if (nc > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this CTA runs

  const int slice = (n + nc - 1) / nc;
  const int c0 = min(n, rank * slice), m = min(n, c0 + slice) - c0;
  const int* bt = a.block_tables + (size_t)row.seq * a.bt_stride + a.sinks;
  const size_t page_stride = (size_t)a.num_layers * a.KH * kPageB;
  const uint8_t* bounds = reinterpret_cast<const uint8_t*>(a.bounds) + ((size_t)a.layer * a.KH + kvh) * kPageB;
  bool odd = false;                              // something that fp32 scores cannot decide

  // lanes below kTile hold the block-table entries of the warp's pages; behind the slice's
  // last page it is repeated: a page that is not the row's would widen its S.  m > 0
  auto entries = [&](int tile) -> int { return bt[c0 + min(tile * kTile + lane, m - 1)]; };
  int* page0 = nullptr;
  auto check = [&](int entry, int tile) -> int {
    const bool bad = entry < 0 || entry >= a.num_pages;
    if (bad) report_error(a.err, kErrBounds);
    odd |= bad;
    entry = bad ? 0 : entry;
    const int i = tile * kTile + lane;
    if (lane < kTile && i < m) page0[c0 + i] = entry;
    return entry;
  };
  const int tiles = (m + kTile - 1) / kTile;
  uint32_t r[kSub][kPieces][4];
  auto load = [&](int sub, int entry) {
    const uint8_t* p = bounds + (size_t)__shfl_sync(0xffffffffu, entry, sub * 8 + g) * page_stride + c * 16;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) ld_stream<16>(r[sub][i], p + i * 64);
  };
  int entry = 0;
  if (warp < tiles) entry = early ? __shfl_sync(0xffffffffu, early_entry, min(lane, m - 1 - warp * kTile)) : entries(warp);
  if (nc > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // the first CTA runs
  float* score0 = nc > 1 ? cluster.map_shared_rank(s_score, 0) : s_score;
  page0 = nc > 1 ? cluster.map_shared_rank(s_page, 0) : s_page;
  int next = 0;
  if (warp < tiles) {
    entry = check(entry, warp);
#pragma unroll
    for (int k = 0; k < kSub; ++k) load(k, entry);
    next = entries(warp + kWarps);
  }
  double qu = 0., qd = 0.;
#pragma unroll
  for (int h = 0; h < 8; ++h) {
    const double x = (double)__bfloat162float(qv[h]);
    if (x >= 0.) qu += x;
    else qd += x;                                // NaN lands here and spoils every score
  }

  // up and dn times the power of two that brings the largest to [1, 2), in three parts
  {
    float mx = (float)fmax(qu, -qd), sum = (float)(qu - qd);
    if (qd != qd) mx = sum = NAN;
    odd |= mx != mx;
    mx = warp_max(mx);
    sum = warp_sum(sum);
    if (lane == 0) {
      s_norm[0][warp] = mx;
      s_norm[1][warp] = sum;
    }
  }
  __syncthreads();
  float qmax = 0.f, l1 = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    qmax = fmaxf(qmax, s_norm[0][w]);
    l1 += s_norm[1][w];
  }
  const int e = (int)(__float_as_uint(qmax) >> 23);
  // f16 parts: another 2^14, so that the last one stays above the subnormals
  const double f = __hiloint2double((1023 + 127 + (F8 ? 14 : 0) - min(max(e, 1), 254)) << 20, 0);
  l1 *= (float)f;
  if (tid < D) {
    s_q[tid] = qd * __hiloint2double((1023 + 800) << 20, 0);
    s_q[D + tid] = qu * __hiloint2double((1023 + 800) << 20, 0);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float x = (float)((k ? qu : qd) * f);
#pragma unroll
      for (int part = 0; part < 3; ++part) {
        if constexpr (F8) {
          const __half h = __float2half_rn(x);
          s_part[part][k * D + tid] = __half_as_ushort(h);
          x -= __half2float(h);
        } else {
          const __nv_bfloat16 h = __float2bfloat16_rn(x);
          s_part[part][k * D + tid] = __bfloat16_as_ushort(h);
          x -= __bfloat162float(h);
        }
      }
    }
  }
  __syncthreads();
  // B operand of step s: columns 0..2 and 3..5
  uint2 qb[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int piece = ((s / kSp) * 4 + c) * (16 / kEl);            // its first element
    const int el = F8 ? piece + (2 * (s % 2) + g / 3) * 4 : piece + (g / 3) * 2;
    const uint16_t* p = &s_part[g % 3][g < 6 ? el : 0];
    qb[s].x = g < 6 ? *reinterpret_cast<const uint32_t*>(p) : 0u;
    qb[s].y = g < 6 ? *reinterpret_cast<const uint32_t*>(p + (F8 ? 2 : 4)) : 0u;
  }

  float s_hi = -INFINITY, s_lo = INFINITY;       // largest and smallest score of the lane, or NaN
  // Largest maximum and most negative minimum of the lane's bounds, 16 bits each: a minimum
  // is not above its maximum, so no bound is larger in magnitude than both.  As integers,
  // positive values rise with their magnitude (signed order), negative ones too (unsigned).
  uint32_t high = 0, deep = 0;
  auto widest = [&](const uint32_t (&w)[4], bool is_max) {
    if (is_max) high = __vimax3_s16x2(__vimax3_s16x2(high, w[0], w[1]), w[2], w[3]);
    else deep = __vimax3_u16x2(__vimax3_u16x2(deep, w[0], w[1]), w[2], w[3]);
  };
  for (int tile = warp; tile < tiles; tile += kWarps) {
    const bool more = tile + kWarps < tiles;
    if (more) {
      entry = check(next, tile + kWarps);
      next = entries(tile + 2 * kWarps);
    }
#pragma unroll
    for (int k = 0; k < kSub; ++k) {
      // two MMAs a sum in the tensor core, the rest in fp32
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s2 = 0; s2 < kSteps; s2 += 2) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = s2; s < s2 + 2; ++s) {
          uint32_t(&w)[4] = r[k][s / kSp];
          const bool is_max = s >= kSteps / 2;
          if constexpr (F8) {
            uint32_t x[4];
            fp8x4_to_half4(w[2 * (s % 2)], x[0], x[2]);
            fp8x4_to_half4(w[2 * (s % 2) + 1], x[1], x[3]);
            mma_f16(acc, x[0], x[1], x[2], x[3], qb[s].x, qb[s].y);
            widest(x, is_max);
          } else {
            mma_bf16_16816(acc, w[0], w[1], w[2], w[3], qb[s].x, qb[s].y);
            widest(w, is_max);
          }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) sum[x] += acc[x];
      }
      if (more) load(k, entry);
      // this lane's columns 2c, 2c + 1: of row g 0..2 are wanted, of row g + 8 3..5
      float v = c == 0 ? sum[0] + sum[1] : c == 1 ? sum[0] + sum[3] : c == 2 ? sum[2] + sum[3] : 0.f;
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      const int i = tile * kTile + k * 8 + g;
      if (c == 0 && i < m) {
        score0[c0 + i] = v;
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(s_hi) : "f"(v));
        asm("min.NaN.f32 %0, %0, %1;" : "+f"(s_lo) : "f"(v));
      }
    }
  }
  // infinite or NaN bounds (as bit patterns they are the largest), or fp32 cannot decide
  const uint32_t wide = __vmaxu2(high & 0x7fff7fffu, deep & 0x7fff7fffu);
  uint32_t big = max(wide << 16, wide & 0xFFFF0000u);
  if constexpr (F8) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&wide));
    big = __float_as_uint(fmaxf(v.x, v.y));
  }
  odd |= !(s_hi < INFINITY && s_lo > -INFINITY);
  if (__any_sync(0xffffffffu, odd)) big = 0x7F800000u;
  big = __reduce_max_sync(0xffffffffu, big);
  uint32_t key_hi = __reduce_max_sync(0xffffffffu, sortable(s_hi));
  uint32_t key_lo_c = __reduce_max_sync(0xffffffffu, ~sortable(s_lo));     // largest complement
  if (lane < 3)
    (nc > 1 ? cluster.map_shared_rank(&s_ends[0][0], 0) : &s_ends[0][0])[(rank * kWarps + warp) * 3 + lane] =
        lane == 0 ? key_hi : lane == 1 ? key_lo_c : big;
  if (tid == 0) s_count = s_nears = 0;
  if (nc > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (rank != 0) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __syncthreads();
  key_hi = key_lo_c = big = 0;
  for (int i = lane; i < nc * kWarps; i += 32) {
    key_hi = max(key_hi, s_ends[i][0]);
    key_lo_c = max(key_lo_c, s_ends[i][1]);
    big = max(big, s_ends[i][2]);
  }
  key_hi = __reduce_max_sync(0xffffffffu, key_hi);
  const uint32_t key_lo = ~__reduce_max_sync(0xffffffffu, key_lo_c);
  big = __reduce_max_sync(0xffffffffu, big);
  const float S = __uint_as_float(big) * l1;
  bool exact = !(S > 8.7e-19f && S < 1.3e36f);   // 2^-60 .. 2^120, and not NaN

  // 64-bit score of candidate i by one warp
  auto score64 = [&](int page) -> uint64_t {
    if (page < 0 || page >= a.num_pages) return 0ull;              // outside the pool: behind every other page
    const uint8_t* b = bounds + (size_t)page * page_stride;
    double s = 0.;
    constexpr int kWords = kPageB / 128;         // 32-bit words per lane
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const uint32_t x = *reinterpret_cast<const uint32_t*>(b + (w * 32 + lane) * 4);
      const int el = (w * 32 + lane) * (4 / kEl);
      if constexpr (F8) {
        double v[4];
        fp8x4_to_f64(x, v);
#pragma unroll
        for (int q = 0; q < 4; ++q) s = fma(s_q[el + q], v[q], s);
      } else {
        double v0, v1;
        bf16x2_to_f64(x, v0, v1);
        s = fma(s_q[el], v0, s);
        s = fma(s_q[el + 1], v1, s);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return sortable(s);
  };

  // warp w owns candidates [w * seg, (w + 1) * seg)
  const int seg = (n + NT - 1) / NT * 32;
  const int g0 = min(n, warp * seg), g1 = min(n, g0 + seg);
  const uint32_t below = (1u << lane) - 1u;      // lanes before this one
  if (!exact) {
    // The need-th largest score lies in [lo, hi]: the bin of a histogram over the range of
    // all scores, then over the edges of that bin, until few share one (scores above hi
    // count in the top bin, which that score is not in).  A bin's edges are off by less than
    // 2^-10 of its width; 2 E = 2^-16 S.
    const float E2 = S * 1.52587890625e-05f;
    float lo = from_sortable(key_lo), hi = from_sortable(key_hi);
    uint32_t in_bin = (uint32_t)n;
    while (in_bin > 8 && hi - lo > E2) {
      const float width = (hi - lo) * (1.f / (kBins - 1)), inv = 1.f / width;
      radix_count<NT>(sc, n, (uint32_t)need, [&](int i) -> int {
        const float v = s_score[i];
        return v > hi ? kBins - 1 : v >= lo ? min(kBins - 2, (int)((v - lo) * inv)) : -1;
      });
      in_bin = sc.in_bin;
      const float l = lo + width * ((float)sc.border - 0x1p-10f), h = lo + width * ((float)(sc.border + 1) + 0x1p-10f);
      lo = fmaxf(lo, l);
      hi = fminf(hi, h);
      __syncthreads();
    }
    lo -= E2;
    hi += E2;
    // list the pages that may go either way, count those above
    uint32_t above = 0, listed_w = 0;
#pragma unroll 4
    for (int i = g0 + lane; i < g1; i += 32) {
      const float v = s_score[i];
      above += v > hi;
      if (v >= lo && v <= hi) {
        ++listed_w;
        const uint32_t at = atomicAdd(&s_count, 1u);
        if (at < kSelList) {
          s_lidx[at] = i;
          s_lval[at] = v;
        }
      }
    }
    above = __reduce_add_sync(0xffffffffu, above);
    listed_w = __reduce_add_sync(0xffffffffu, listed_w);
    if (lane == 0) {
      s_cnt[0][warp] = above;
      s_cnt[1][warp] = listed_w;
    }
    __syncthreads();
    uint32_t take = (uint32_t)need;              // pages of the list to take: 1 .. listed
#pragma unroll
    for (int w = 0; w < kWarps; ++w) take -= s_cnt[0][w];
    const uint32_t listed = s_count;
    exact = listed > kSelList && listed > take;
    if (!exact) {
      if (listed > take) {
        // the need-th largest score b itself, the pages that are surely above it, and those
        // within 2 E of it: all of these are taken, or 64-bit scores tell them apart
        const bool in = (uint32_t)tid < listed;
        const float v = in ? s_lval[tid] : 0.f;
        const int idx = in ? s_lidx[tid] : 0;
        if (in) {
          uint32_t more = 0, same = 0;
          for (uint32_t j = 0; j < listed; ++j) {
            more += s_lval[j] > v;
            same += s_lval[j] == v;
          }
          if (more < take && more + same >= take) s_b = v;
        }
        __syncthreads();
        const bool sure = in && v > s_b + E2, near = in && !sure && v >= s_b - E2;
        const uint32_t sures = __syncthreads_count(sure), nears = __syncthreads_count(near);
        bool taken = sure || near;
        if (sures + nears > take) {
          if (near) s_near[atomicAdd(&s_nears, 1u)] = tid;
          __syncthreads();
          for (uint32_t i = warp; i < nears; i += kWarps) {
            const uint64_t k = score64(s_page[s_lidx[s_near[i]]]);
            if (lane == 0) s_lkey[s_near[i]] = k;
          }
          __syncthreads();
          if (near) {
            const uint64_t k = s_lkey[tid];
            uint32_t better = 0;
            for (uint32_t j = 0; j < nears; ++j) {
              const int o = s_near[j];
              better += s_lkey[o] > k || (s_lkey[o] == k && s_lidx[o] < idx);
            }
            taken = better < take - sures;
          }
        }
        if (in) {
          s_score[idx] = taken ? INFINITY : -INFINITY;
          if (!taken) atomicSub(&s_cnt[1][idx / seg], 1u);
        }
        __syncthreads();
      }
      uint32_t pos = (uint32_t)a.sinks;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) pos += w < warp ? s_cnt[0][w] + s_cnt[1][w] : 0u;
#pragma unroll 4
      for (int i0 = g0; i0 < g1; i0 += 32) {
        const int i = i0 + lane;
        const bool on = i < g1 && s_score[i] >= lo;
        const uint32_t hit = __ballot_sync(0xffffffffu, on);
        if (on) out[pos + __popc(hit & below)] = a.sinks + i;
        pos += __popc(hit);
      }
      return;
    }
  }
  // ---- 64-bit scores of all candidates
  __syncthreads();
  uint64_t top = 0, low_c = 0;
  for (int i = warp; i < n; i += kWarps) {
    const uint64_t k = score64(bt[i]);
    if (lane == 0) s_key[i] = k;
    top = max(top, k);
    low_c = max(low_c, ~k);
  }
  if (lane == 0) {
    sc.red[0][warp] = top;
    sc.red[1][warp] = low_c;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    top = max(top, sc.red[0][w]);
    low_c = max(low_c, sc.red[1][w]);
  }
  Border<uint64_t> b;
  b.start(top, ~low_c, (uint32_t)need, n);
  while (b.shift > 0 && b.in_bin != b.left) radix_pass<NT>(sc, n, [&](int i) { return s_key[i]; }, b);
  // keys above the border's are taken, and of those on it the first `left`
  uint32_t gt = 0, eq = 0;
  for (int i = g0 + lane; i < g1; i += 32) {
    const uint64_t k = s_key[i] & b.mask;
    gt += k > b.prefix;
    eq += k == b.prefix;
  }
  gt = __reduce_add_sync(0xffffffffu, gt);
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) {
    s_cnt[0][warp] = gt;
    s_cnt[1][warp] = eq;
  }
  __syncthreads();
  uint32_t ties = 0, pos = (uint32_t)a.sinks;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    pos += w < warp ? s_cnt[0][w] : 0u;
    ties += w < warp ? s_cnt[1][w] : 0u;
  }
  pos += min(ties, b.left);
  for (int i0 = g0; i0 < g1; i0 += 32) {
    const int i = i0 + lane;
    const uint64_t k = i < g1 ? s_key[i] & b.mask : 0ull;
    const bool tie = i < g1 && k == b.prefix;
    const uint32_t tie_hit = __ballot_sync(0xffffffffu, tie);
    const bool on = i < g1 && (k > b.prefix || (tie && ties + __popc(tie_hit & below) < b.left));
    const uint32_t hit = __ballot_sync(0xffffffffu, on);
    if (on) out[pos + __popc(hit & below)] = a.sinks + i;
    pos += __popc(hit);
    ties += __popc(tie_hit);
  }
}

template <int D, bool F8, int NT>
static void launch_select(const SelectArgs& a, int nc, cudaStream_t st) {
  // by the table's width, not the contexts': where it leaves an SM fewer CTAs, short contexts
  // are slower too.  B200, us, 16000 tokens with tables of 1000 / 4096 / 6144 / 8192 / 12288 /
  // 24576 columns: 64 rows (bf16) 49.7 / 60.9 / 79.8 / 148 / 112 / 131, 32 rows 27.9 / 28.1 /
  // 28.0 / 29.0 / 56.2 / 62.0; 1 row of 32000 tokens 9.9 up to 16384 columns, 10.6 with 24576.
  const size_t smem = (size_t)a.max_pages * sizeof(uint64_t);
  auto kern = select_kernel<D, F8, NT>;
  if (smem > 32 * 1024)
    VRM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelMaxPages * 8));
  const dim3 grid(nc, a.KH, a.T);
  if (nc > 1) launch_kernel_cluster(kern, grid, dim3(NT), dim3(nc, 1, 1), smem, st, a);
  else launch_kernel(kern, grid, dim3(NT), smem, st, a);
}

void select_pages(const SelectArgs& in, cudaStream_t st) {
  if (in.T <= 0) return;
  SelectArgs a = in;
  a.err = error_word();
  VRM_REQUIRE(a.D == 64 || a.D == 128, "select_pages: head_dim must be 64 or 128");
  VRM_REQUIRE(a.max_pages <= kSelMaxPages, "select_pages: more than 24576 pages a sequence");
  VRM_REQUIRE(a.T <= 65535, "select_pages: too many query rows");
  // Few rows: CTAs of 16 warps, one to an SM, and a cluster shares a row's candidates as long
  // as every CTA has its SM.  More: one CTA a row, of 8 warps while two to an SM hold all rows,
  // else of 4, four to an SM.  B200, 8 kv heads of 128 dims (us): 1 row of 32k tokens with 1 / 2 / 4 / 8
  // CTAs 19.1 / 14.2 / 11.3 / 9.9, 4 rows 21.4 / 15.7 / 12.6 / 20.1, 16 rows 25.5 / 31.1 / 41.2 /
  // 54.2; 16, 8 and 4 warps a CTA: 16 rows 25.5, 27.1 (2 CTAs), 36.1; 32 rows of 16k 29.0,
  // 24.8, 33.8; 64 rows of fp8 bounds at 32k -, 62.4, 56.4.
  const long long rows = (long long)a.T * a.KH, sms = device_sm_count();
  int nc = 1;
  while (nc < 8 && rows * nc * 2 <= sms) nc *= 2;
  auto go = [&](auto d, auto f8) {
    constexpr int D = decltype(d)::value;
    constexpr bool F8 = decltype(f8)::value;
    if (rows <= sms) launch_select<D, F8, 512>(a, nc, st);
    else if (rows <= 2 * sms) launch_select<D, F8, 256>(a, 1, st);
    else launch_select<D, F8, 128>(a, 1, st);
  };
  using D128 = std::integral_constant<int, 128>;
  using D64 = std::integral_constant<int, 64>;
  if (a.D == 128) a.f8 ? go(D128{}, std::true_type{}) : go(D128{}, std::false_type{});
  else a.f8 ? go(D64{}, std::true_type{}) : go(D64{}, std::false_type{});
  VRM_CUDA_CHECK(cudaGetLastError());
}

// ================================================================ attention over selected pages
namespace {

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// two four-bit codes held in bits 0..3 and 16..19 -> f16x2 of code * s + m (1024 + code is
// an exact f16 with the code in its significand)
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t v, uint32_t s2, uint32_t m2) {
  const uint32_t x = (v & 0x000F000Fu) | 0x64006400u;
  uint32_t y, r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(0x64006400u));
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(y), "r"(s2), "r"(m2));
  return r;
}

// What a lane (g = lane / 4, c = lane % 4) holds of a page.  K: a quarter of the dims of
// tokens g and g + 8.  V: an eighth of the dims (of g) of tokens 2c, 2c + 1, 2c + 8, 2c + 9.
// Both are read from global memory straight into registers in whole 16-byte (8, 4 for
// narrow rows) pieces; the order of the dims inside a dot product and of the dims over the
// output tiles is free, so the fragments need no shared memory and no exchange.
template <int D, int FMT>
struct Frag {
  static constexpr int kRowB = PageRow<D, FMT>::kBytes;
  static constexpr int kCodeB = FMT == kFmtQ4 ? D / 2 : kRowB;      // bytes of values in a row
  static constexpr int kKB = kCodeB / 4;                            // bytes of a row per lane, K
  static constexpr int kVB = kCodeB / 8;                            // V
  static constexpr int kPK = kKB < 16 ? kKB : 16, kPV = kVB < 16 ? kVB : 16;   // bytes of a piece
  uint32_t k[2][kKB / 4], v[4][kVB / 4];
  uint32_t ks[FMT == kFmtQ4 ? 2 : 1], vs[FMT == kFmtQ4 ? 4 : 1];    // {scale, min}

  template <bool ALL>
  __device__ __forceinline__ void get_k(const uint8_t* kp, int rows, int g, int c) {
    const uint8_t* p0 = kp + g * kRowB + c * kPK;
    const uint8_t* s0 = kp + g * kRowB + D / 2 + (D == 128 ? c : c / 2) * 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (ALL || g + 8 * h < rows) {
#pragma unroll
        for (int i = 0; i < kKB / kPK; ++i) ld_stream<kPK>(&k[h][i * kPK / 4], p0 + h * 8 * kRowB + i * 4 * kPK);
        if constexpr (FMT == kFmtQ4) ld_stream<4>(&ks[h], s0 + h * 8 * kRowB);
      } else {
#pragma unroll
        for (int i = 0; i < kKB / 4; ++i) k[h][i] = 0u;
        if constexpr (FMT == kFmtQ4) ks[h] = 0u;
      }
    }
  }
  template <bool ALL>
  __device__ __forceinline__ void get_v(const uint8_t* vp, int rows, int g, int c) {
    const uint8_t* p0 = vp + 2 * c * kRowB + g * kPV;
    const uint8_t* s0 = vp + 2 * c * kRowB + D / 2 + (D == 128 ? g / 2 : g / 4) * 4;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int r = (h & 1) + 8 * (h >> 1);
      if (ALL || 2 * c + r < rows) {
#pragma unroll
        for (int i = 0; i < kVB / kPV; ++i) ld_stream<kPV>(&v[h][i * kPV / 4], p0 + r * kRowB + i * 8 * kPV);
        if constexpr (FMT == kFmtQ4) ld_stream<4>(&vs[h], s0 + r * kRowB);
      } else {
#pragma unroll
        for (int i = 0; i < kVB / 4; ++i) v[h][i] = 0u;
        if constexpr (FMT == kFmtQ4) vs[h] = 0u;
      }
    }
  }
  // rows >= `rows` (behind the context) are not read and count as zeros
  __device__ __forceinline__ void load_k(const uint8_t* kp, int rows, int g, int c) {
    if (rows == kPageTok) get_k<true>(kp, rows, g, c);
    else get_k<false>(kp, rows, g, c);
  }
  __device__ __forceinline__ void load_v(const uint8_t* vp, int rows, int g, int c) {
    if (rows == kPageTok) get_v<true>(vp, rows, g, c);
    else get_v<false>(vp, rows, g, c);
  }
  // first of the four dims that step s of the score product takes from lane c
  static __device__ __forceinline__ int k_dim(int s, int c) {
    if constexpr (FMT == kFmtBf16) return (c + 4 * (s / 2)) * 8 + 4 * (s % 2);
    else if constexpr (FMT == kFmtFp8) return (c + 4 * (s / 4)) * 16 + 4 * (s % 4);
    else return c * (D / 4) + 4 * s;
  }
  // q's fragment of step s from the eight dims 8 (s / 2) .. of lane c's four-bit piece: the
  // pairs of a code word that one mask takes out are (0, 4), (1, 5) | (2, 6), (3, 7)
  static __device__ __forceinline__ uint2 q4_pairs(const uint2& lo, const uint2& hi, int s) {
    const uint32_t a = s % 2 ? lo.y : lo.x, b = s % 2 ? hi.y : hi.x;
    return make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
  }
  // A fragment of step s: dims k_dim .. + 1 of rows g, g + 8, then k_dim + 2 .. + 3
  __device__ __forceinline__ void k_frag(int s, uint32_t (&a)[4]) const {
    if constexpr (FMT == kFmtBf16) {
      a[0] = k[0][2 * s];
      a[1] = k[1][2 * s];
      a[2] = k[0][2 * s + 1];
      a[3] = k[1][2 * s + 1];
    } else if constexpr (FMT == kFmtFp8) {
      a[0] = fp8x2_to_half2(k[0][s] & 0xffffu);
      a[1] = fp8x2_to_half2(k[1][s] & 0xffffu);
      a[2] = fp8x2_to_half2(k[0][s] >> 16);
      a[3] = fp8x2_to_half2(k[1][s] >> 16);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t s2 = __byte_perm(ks[h], 0, 0x1010), m2 = __byte_perm(ks[h], 0, 0x3232);
        const uint32_t w = k[h][s / 2] >> (8 * (s % 2));        // dims 0 and 4, 1 and 5 of it, or 2 and 6, 3 and 7
        a[h] = codes_to_half2(w, s2, m2);
        a[2 + h] = codes_to_half2(w >> 4, s2, m2);
      }
    }
  }
  // Output tile e: rows 0..7 are dims v_dim(e, g, 0), rows 8..15 v_dim(e, g, 1)
  static __device__ __forceinline__ int v_dim(int e, int g, int hi) {
    if constexpr (FMT == kFmtBf16 && D == 128) return 64 * hi + 8 * g + e;
    else return (D / 8) * g + (D / 16) * hi + e;
  }
  __device__ __forceinline__ void v_frag(int e, uint32_t (&a)[4]) const {
#pragma unroll
    for (int q = 0; q < 4; ++q) {                // a[q]: token pair q / 2, dim half q % 2
      const int t0 = 2 * (q >> 1), hi = q & 1;
      if constexpr (FMT == kFmtBf16) {
        const int w = (D == 128 ? 4 : 2) * hi + e / 2;
        a[q] = __byte_perm(v[t0][w], v[t0 + 1][w], e % 2 ? 0x7632 : 0x5410);
      } else if constexpr (FMT == kFmtFp8) {
        const int dim = (D / 16) * hi + e;
        const uint32_t x = __byte_perm(v[t0][dim / 4], v[t0 + 1][dim / 4], dim % 4 < 2 ? 0x5140 : 0x7362);
        a[q] = fp8x2_to_half2(dim % 2 ? x >> 16 : x);
      } else {
        const int dim = (D / 16) * hi + e;
        const uint32_t x = __byte_perm(v[t0][dim / 8], v[t0 + 1][dim / 8], dim % 8 < 4 ? 0x5410 : 0x7632);
        const uint32_t s2 = __byte_perm(vs[t0], vs[t0 + 1], 0x5410), m2 = __byte_perm(vs[t0], vs[t0 + 1], 0x7632);
        a[q] = codes_to_half2(x >> (4 * (dim % 4)), s2, m2);
      }
    }
  }
};

}  // namespace

// Pages a warp takes at a time and CTAs an SM holds.  Pages of 8 KB (bf16, D = 128): two
// at a time in 255 registers, so that each of the SM's 8 warps has 16 KB under way; narrower
// pages cost more arithmetic a byte, and 16 warps with one page each run better (B200, us:
// 32 rows of bf16 43.9 against 77.9 with one page and 4 CTAs; 128 rows of fp8 92.0 against
// 97.0 with four pages and 2 CTAs, 128 four-bit rows 104.2 against 107.7).
template <int D, int FMT>
struct AttendShape {
  static constexpr bool kWide = FMT == kFmtBf16 && D == 128;
  static constexpr int kTurn = kWide ? 2 : 1, kCtas = kWide ? 2 : 4;
};

// One CTA of 4 warps per (kv head, query row, split); the warps of all splits take the
// row's pages in turn.  Scores are computed transposed, S^T = K Q^T: a page's 16 tokens
// fill the MMA rows and the group's (<= 8) heads its columns; O^T = V^T P^T likewise.  A
// warp requests its next page's K as soon as the scores have used the present one's, and V
// after the outputs, so that loads are in flight all the time.  Splits are the CTAs of one
// cluster: each pushes its partial outputs to the CTAs that finish them, through
// distributed shared memory.  Bound by the reads of the pages (32 rows of 128 bf16 pages:
// 43.9 us, 6.1 TB/s; 128 rows of fp8: 92 us, 5.9 TB/s); one row is bound by the latency of
// its table, pages and merge (7.7 us).
template <int D, int FMT>
__global__ void __launch_bounds__(128, AttendShape<D, FMT>::kCtas) attend_kernel(AttendArgs P) {
  using F = Frag<D, FMT>;
  constexpr int kTurn = AttendShape<D, FMT>::kTurn;
  constexpr int kSteps = D / 16;
  constexpr int kOS = D + 1;                           // odd: the transposed stores meet in two lanes a bank
  __shared__ float s_m[4][8], s_l[4][8];
  __shared__ float s_o[4 * 8 * kOS];
  __shared__ float s_in[8 * D], s_ml[8][2][8];         // what the splits pushed: [split][head][dim], [split][m, l][head]
  __shared__ float s_w[8][8], s_max[8], s_sum[8];      // weights of the parts of a merge, their maximum and sum
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  pdl_launch();
  pdl_wait();
  const int kvh = blockIdx.x, t = blockIdx.y, split = blockIdx.z, nsplit = gridDim.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int G = P.G, KH = P.KH;
  const int stride = 4 * nsplit;
  const int* list = P.pages + ((size_t)t * KH + kvh) * P.S;
  // 32 list entries of this warp, one a lane; the first are requested beside the row's length
  auto entry = [&](int base) -> int { return base + lane * stride < P.S ? list[base + lane * stride] : -1; };
  int lp = entry(split * 4 + warp);

  // Q as the B operand: step s, lane (g, c) holds dims k_dim(s, c) .. + 3 of head g
  uint2 qb[kSteps];
  {
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(P.q) + (size_t)t * P.ld_q + (size_t)(kvh * G + g) * D;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      qb[s] = g < G ? *reinterpret_cast<const uint2*>(q + F::k_dim(s, c)) : make_uint2(0u, 0u);
  }
  // factors of the scores of heads 2c and 2c + 1
  float k_scale = 1.f, v_scale = 1.f;
  if constexpr (FMT == kFmtFp8) {
    k_scale = P.kv_scale[(P.layer * 2 + 0) * KH + kvh];
    v_scale = P.kv_scale[(P.layer * 2 + 1) * KH + kvh];
  }
  // Weights become operands beside V, of its type: bf16 over bf16 pages, in two parts that hold
  // 16 bits of them (with one part outputs were off by 1.9e-3 of their norm instead of 1.7e-3, a
  // bf16 result's own rounding; 32 rows of 128 pages 43.65 -> 43.9 us); f16 over the others, 11
  // bits, which shows in no output's error (1.7e-3 either way).  The latter times 2^14, so that a
  // weight stays whole down to 2^-28 of the largest and counts down to 2^-39.  The sums that
  // divide them are fp32 sums of the weights before that rounding.
  constexpr float kWeight = FMT == kFmtBf16 ? 1.f : 16384.f;
  v_scale *= 1.f / kWeight;
  const float sm_log2 = P.sm_scale * 1.4426950408889634f;
  float scale_log2[2] = {sm_log2 * k_scale, sm_log2 * k_scale};
  RowOf row;
  if (!find_row(t, P.cu_q, P.context_lens, P.B, row)) return;      // the same for the whole cluster
  if (nsplit > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this CTA runs
  const int* bt = P.block_tables + (size_t)row.seq * P.bt_stride;
  const size_t head_b = (size_t)kPageTok * F::kRowB;
  const size_t page_b = (size_t)P.num_layers * 2 * KH * head_b;
  const uint8_t* pool = reinterpret_cast<const uint8_t*>(P.cache) + ((size_t)P.layer * 2 * KH + kvh) * head_b;

  float o[kSteps][4];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  bool seen = false, q_ready = FMT == kFmtBf16;

  for (int base = split * 4 + warp; base < P.S; base += 32 * stride) {
    // physical page and tokens to read of the lane's entry
    int phys = 0, rows = 0;
    if (lp >= 0 && lp < P.max_pages && (long long)lp * kPageTok < row.n) {
      phys = bt[lp];
      if (phys >= 0 && phys < P.num_pages) rows = min(kPageTok, row.n - lp * kPageTok);
      else report_error(P.err, kErrBounds);
    }
    lp = entry(base + 32 * stride);
    uint32_t todo = __ballot_sync(0xffffffffu, rows > 0);
    if (todo == 0) continue;
    seen = true;
    // the pages of a turn: kTurn set bits of todo (rows 0: none left)
    F f[kTurn];
    const uint8_t* kp[kTurn];
    int r[kTurn];
    auto take = [&] {
#pragma unroll
      for (int q = 0; q < kTurn; ++q) {
        const int j = todo ? __ffs(todo) - 1 : 0;
        const int rj = __shfl_sync(0xffffffffu, rows, j);
        kp[q] = pool + (size_t)__shfl_sync(0xffffffffu, phys, j) * page_b;
        r[q] = todo ? rj : 0;
        todo &= todo - 1;
      }
    };
    take();
#pragma unroll
    for (int q = 0; q < kTurn; ++q) f[q].load_k(kp[q], r[q], g, c);
#pragma unroll
    for (int q = 0; q < kTurn; ++q) f[q].load_v(kp[q] + (size_t)KH * head_b, r[q], g, c);
    if (!q_ready) {
      // f16 operands: each head's q times the power of two that brings its largest value to
      // [2^14, 2^15), or 2^126 if that is less: the eight bits of a value stay whole down to
      // 2^-31 of the head's largest.  A head with an infinite value has no finite score: NaN.
      float mx = 0.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        mx = fmaxf(mx, fmaxf(fmaxf(fabsf(bf16_lo(qb[s].x)), fabsf(bf16_hi(qb[s].x))),
                             fmaxf(fabsf(bf16_lo(qb[s].y)), fabsf(bf16_hi(qb[s].y)))));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const uint32_t e = __float_as_uint(mx) >> 23, up = min(253u, 268u - e);
      const float x = __uint_as_float(up << 23);
      const float down = e == 255u ? NAN : __uint_as_float((254u - up) << 23);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        scale_log2[h] = sm_log2 * __shfl_sync(0xffffffffu, down, 4 * (2 * c + h)) * k_scale;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        qb[s].x = pack_half2(bf16_lo(qb[s].x) * x, bf16_hi(qb[s].x) * x);
        qb[s].y = pack_half2(bf16_lo(qb[s].y) * x, bf16_hi(qb[s].y) * x);
      }
      if constexpr (FMT == kFmtQ4) {
#pragma unroll
        for (int s = 0; s < kSteps; s += 2) {
          const uint2 lo = qb[s], hi = qb[s + 1];
          qb[s] = F::q4_pairs(lo, hi, 0);
          qb[s + 1] = F::q4_pairs(lo, hi, 1);
        }
      }
      q_ready = true;
    }
    bool more = true;
    while (more) {
      int r_now[kTurn];
#pragma unroll
      for (int q = 0; q < kTurn; ++q) r_now[q] = r[q];
      more = todo != 0;
      if (more) take();
      float x[kTurn][4], mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int q = 0; q < kTurn; ++q) {
        float sc[4] = {0.f, 0.f, 0.f, 0.f}, sd[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          uint32_t a[4];
          f[q].k_frag(s, a);
          if constexpr (FMT == kFmtBf16) mma_bf16_16816(s % 2 ? sd : sc, a[0], a[1], a[2], a[3], qb[s].x, qb[s].y);
          else mma_f16(s % 2 ? sd : sc, a[0], a[1], a[2], a[3], qb[s].x, qb[s].y);
        }
        if (more) f[q].load_k(kp[q], r[q], g, c);
        // sc[0] = (token g, head 2c), [1] = (g, 2c + 1), [2] = (g + 8, 2c), [3] = (g + 8, 2c + 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[q][i] = (sc[i] + sd[i]) * scale_log2[i % 2];
        if (r_now[q] != kPageTok) {
          if (g >= r_now[q]) x[q][0] = x[q][1] = -INFINITY;
          if (g + 8 >= r_now[q]) x[q][2] = x[q][3] = -INFINITY;
        }
        mx[0] = fmaxf(mx[0], fmaxf(x[q][0], x[q][2]));
        mx[1] = fmaxf(mx[1], fmaxf(x[q][1], x[q][3]));
      }
      float alpha[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 4));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 8));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 16));
        const float m_new = fmaxf(m_run[h], mx[h]);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        alpha[h] = ex2(m_run[h] - m_use);
        m_run[h] = m_new;
        l_run[h] *= alpha[h];
#pragma unroll
        for (int q = 0; q < kTurn; ++q) {
          x[q][h] = ex2(x[q][h] - m_use);
          x[q][2 + h] = ex2(x[q][2 + h] - m_use);
          l_run[h] += x[q][h] + x[q][2 + h];
        }
      }
#pragma unroll
      for (int e = 0; e < kSteps; ++e) {
        o[e][0] *= alpha[0];
        o[e][1] *= alpha[1];
        o[e][2] *= alpha[0];
        o[e][3] *= alpha[1];
      }
#pragma unroll
      for (int q = 0; q < kTurn; ++q) {
        uint32_t pb0, pb1, pl0 = 0, pl1 = 0;                 // weights; bf16: and what they leave
        if constexpr (FMT == kFmtBf16) {
          const uint32_t h0 = pack_bf16x2(x[q][0], x[q][1]), h1 = pack_bf16x2(x[q][2], x[q][3]);
          pb0 = transpose8x8(h0);
          pb1 = transpose8x8(h1);
          pl0 = transpose8x8(pack_bf16x2(x[q][0] - bf16_lo(h0), x[q][1] - bf16_hi(h0)));
          pl1 = transpose8x8(pack_bf16x2(x[q][2] - bf16_lo(h1), x[q][3] - bf16_hi(h1)));
        } else {
          pb0 = transpose8x8(pack_half2(x[q][0] * kWeight, x[q][1] * kWeight));
          pb1 = transpose8x8(pack_half2(x[q][2] * kWeight, x[q][3] * kWeight));
        }
#pragma unroll
        for (int e = 0; e < kSteps; ++e) {
          uint32_t a[4];
          f[q].v_frag(e, a);
          if constexpr (FMT == kFmtBf16) {
            mma_bf16_16816(o[e], a[0], a[1], a[2], a[3], pb0, pb1);
            mma_bf16_16816(o[e], a[0], a[1], a[2], a[3], pl0, pl1);
          } else {
            mma_f16(o[e], a[0], a[1], a[2], a[3], pb0, pb1);
          }
        }
        if (more) f[q].load_v(kp[q] + (size_t)KH * head_b, r[q], g, c);
      }
    }
  }
  // each lane summed its own tokens' weights: the eight lanes that share c hold the rest
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    l_run[q] += __shfl_xor_sync(0xffffffffu, l_run[q], 4);
    l_run[q] += __shfl_xor_sync(0xffffffffu, l_run[q], 8);
    l_run[q] += __shfl_xor_sync(0xffffffffu, l_run[q], 16);
    if (seen && m_run[q] == -INFINITY) l_run[q] = NAN;     // every score -inf: as softmax gives
  }

  // ---- merge the 4 warps
  if (g == 0) {
    s_m[warp][2 * c] = m_run[0];
    s_m[warp][2 * c + 1] = m_run[1];
    s_l[warp][2 * c] = l_run[0];
    s_l[warp][2 * c + 1] = l_run[1];
  }
#pragma unroll
  for (int e = 0; e < kSteps; ++e) {
    float* r0 = s_o + (warp * 8 + 2 * c) * kOS;
    r0[F::v_dim(e, g, 0)] = o[e][0];
    r0[kOS + F::v_dim(e, g, 0)] = o[e][1];
    r0[F::v_dim(e, g, 1)] = o[e][2];
    r0[kOS + F::v_dim(e, g, 1)] = o[e][3];
  }
  __syncthreads();
  // weights of up to 8 partial sums with maxima m(w, h) and sums l(w, h), by one warp: lane
  // (w % 4, h) has parts w and w + 4
  auto weigh = [&](int parts, auto m, auto l) {
    if (warp != 0) return;
    const int h = lane & 7, w = lane >> 3;
    const float m0 = w < parts ? m(w, h) : -INFINITY, m1 = w + 4 < parts ? m(w + 4, h) : -INFINITY;
    const float l0 = w < parts ? l(w, h) : 0.f, l1 = w + 4 < parts ? l(w + 4, h) : 0.f;
    float M = fmaxf(m0, m1);
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 8));
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, 16));
    const float f0 = m0 == -INFINITY ? 0.f : ex2(m0 - M), f1 = m1 == -INFINITY ? 0.f : ex2(m1 - M);
    // no score above -inf anywhere: the sums are 0, or NaN
    float L = M == -INFINITY ? l0 + l1 : (f0 == 0.f ? 0.f : f0 * l0) + (f1 == 0.f ? 0.f : f1 * l1);
    L += __shfl_xor_sync(0xffffffffu, L, 8);
    L += __shfl_xor_sync(0xffffffffu, L, 16);
    s_w[w][h] = f0;
    s_w[w + 4][h] = f1;
    if (w == 0) {
      s_max[h] = M;
      s_sum[h] = L;
    }
    __syncwarp();
  };
  weigh(4, [&](int w, int h) { return s_m[w][h]; }, [&](int w, int h) { return s_l[w][h]; });
  if (nsplit > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // the others run
  if (nsplit > 1 && warp == 0) {
    for (int q = lane >> 3; q < nsplit; q += 4) {
      float* ml = cluster.map_shared_rank(&s_ml[0][0][0], q) + split * 16 + (lane & 7);
      ml[0] = s_max[lane & 7];
      ml[8] = s_sum[lane & 7];
    }
  }
  __syncthreads();
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(P.out) + (size_t)t * P.ld_o + (size_t)kvh * G * D;
  // thread: dims d, d + 1 of heads h0, h0 + 256 / D ..; a split finishes D / nsplit dims of every head
  const int d = 2 * (threadIdx.x % (D / 2)), h0 = threadIdx.x / (D / 2);
  const int own = D / nsplit;
  float* there = nsplit > 1 ? cluster.map_shared_rank(s_in, d / own) + split * 8 * own + d % own : nullptr;
  for (int h = h0; h < G; h += 256 / D) {
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = s_w[w][h];
      if (f != 0.f) {
        x += f * s_o[(w * 8 + h) * kOS + d];
        y += f * s_o[(w * 8 + h) * kOS + d + 1];
      }
    }
    if (nsplit == 1) {
      const float L = s_sum[h];
      *reinterpret_cast<uint32_t*>(out + h * D + d) =
          L == 0.f ? 0u : pack_bf16x2(x / L * v_scale, y / L * v_scale);
    } else {
      there[h * own] = x;
      there[h * own + 1] = y;
    }
  }
  if (nsplit == 1) return;
  cluster.sync();
  weigh(nsplit, [&](int w, int h) { return s_ml[w][0][h]; }, [&](int w, int h) { return s_ml[w][1][h]; });
  __syncthreads();
  for (int i = threadIdx.x; i < G * own; i += 128) {
    const int h = i / own;
    float x = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const float f = q < nsplit ? s_w[q][h] : 0.f;
      if (f != 0.f) x += f * s_in[q * 8 * own + i];
    }
    const float L = s_sum[h];
    out[h * D + split * own + i % own] = __float2bfloat16(L == 0.f ? 0.f : x / L * v_scale);
  }
}

template <int D, int FMT>
static void launch_attend(const AttendArgs& a, cudaStream_t st) {
  // as many splits as keep all CTAs resident at once and leave every warp two pages: more
  // CTAs than that queue, and each costs its start and its merge again (B200, us, splits
  // 1 / 2 / 8: 1 row of bf16 25.1 / 15.6 / 7.6, 16 rows 34.9 / 25.6 / 39.6, 64 rows 84.4 / 96.9 / 139)
  int splits = 1;
  while (splits < 8 && (long long)a.T * a.KH * splits * 2 <= (long long)AttendShape<D, FMT>::kCtas * device_sm_count() &&
         a.S >= 16 * splits)
    splits *= 2;
  const dim3 grid(a.KH, a.T, splits);
  if (splits > 1) launch_kernel_cluster(attend_kernel<D, FMT>, grid, dim3(128), dim3(1, 1, splits), 0, st, a);
  else launch_kernel(attend_kernel<D, FMT>, grid, dim3(128), 0, st, a);
}

void paged_attention_selected(const AttendArgs& in, cudaStream_t st) {
  if (in.T <= 0) return;
  AttendArgs a = in;
  a.err = error_word();
  VRM_REQUIRE(a.D == 64 || a.D == 128, "paged_attention_selected: head_dim must be 64 or 128");
  VRM_REQUIRE(a.G >= 1 && a.G <= 8, "paged_attention_selected: GQA group must be <= 8 heads");
  VRM_REQUIRE(a.T <= 65535, "paged_attention_selected: too many query rows");
  auto go = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (a.fmt == kFmtQ4) launch_attend<D, kFmtQ4>(a, st);
    else if (a.fmt == kFmtFp8) launch_attend<D, kFmtFp8>(a, st);
    else launch_attend<D, kFmtBf16>(a, st);
  };
  if (a.D == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 64>{});
  VRM_CUDA_CHECK(cudaGetLastError());
}

}  // namespace vrm
