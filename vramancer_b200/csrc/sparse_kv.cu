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
#include <cstdlib>
#include <type_traits>

#include "vrm_common.cuh"
#include "vrm_host.h"
#include "vrm_kernels.h"

namespace vrm {

namespace {

constexpr int kPageTok = 16;

// 16-byte / 8-byte / 4-byte loads that do not allocate in L1 (every byte is used once)
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 ld_stream8(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_stream4(const void* p) {
  uint32_t v;
  asm volatile("ld.global.L1::no_allocate.b32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}

__device__ __forceinline__ float fp8_to_f32(uint32_t code) {
  __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3);
  return __half2float(*reinterpret_cast<__half*>(&h));
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
// blockIdx.x is a tile of kRows tokens, blockIdx.y a group of q heads, v heads or one k
// head.  With key bounds a k block owns the runs (maximal sequences of adjacent tokens in
// consecutive slots of one page) that begin in its tile, wherever they end, so every
// page's bounds have one writer and do not depend on the order of the blocks.
template <int D>
struct AppendShape {
  static constexpr int kLanes = D / 16;            // lanes of a row
  static constexpr int kRows = 128 / kLanes;       // rows of a block pass
  static constexpr int kSpan = kRows + kPageTok;   // tokens of a k block (the last run may leave the tile)
};

enum : int { kRotNone = 0, kRotFull = 1, kRotPart = 2 };

// x (16 dims of a row per lane) -> RMSNorm with weight w (null: none), then the rotation
template <int D, int ROT>
__device__ __forceinline__ void norm_rotate(float (&x)[16], const __nv_bfloat16* w, float eps, int j, const float* cs,
                                            int rot_dim, float* scratch) {
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
    for (int q = 0; q < 2; ++q) {
      const float4 c = *reinterpret_cast<const float4*>(cs + 8 * j + 4 * q);
      const float4 s = *reinterpret_cast<const float4*>(cs + D / 2 + 8 * j + 4 * q);
      rope_rotate(x[4 * q], x[8 + 4 * q], c.x, s.x, x[4 * q], x[8 + 4 * q]);
      rope_rotate(x[4 * q + 1], x[9 + 4 * q], c.y, s.y, x[4 * q + 1], x[9 + 4 * q]);
      rope_rotate(x[4 * q + 2], x[10 + 4 * q], c.z, s.z, x[4 * q + 2], x[10 + 4 * q]);
      rope_rotate(x[4 * q + 3], x[11 + 4 * q], c.w, s.w, x[4 * q + 3], x[11 + 4 * q]);
    }
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
        rope_rotate(x[i], scratch[d + half], cs[d], cs[half + d], a, b);
        x[i] = a;
      } else if (d < rot_dim) {
        rope_rotate(scratch[d - half], x[i], cs[d - half], cs[d], a, b);
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

// One rounding from fp32 to the page format; x becomes the value that readers of the row
// see (fp8: the e4m3 code, before the head's scale).  dst: the stored row; `on`: this
// lane's row is stored (all lanes take part in the shuffles).
template <int D, int FMT>
__device__ __forceinline__ void store_kv_row(uint8_t* dst, float (&x)[16], float scale, int j, bool on) {
  if constexpr (FMT == kFmtBf16) {
    const uint4 a = pack8(x), b = pack8(x + 8);
    if (on) {
      *reinterpret_cast<uint4*>(dst + 16 * j) = a;
      *reinterpret_cast<uint4*>(dst + D + 16 * j) = b;
    }
    unpack8(a, x);
    unpack8(b, x + 8);
  } else if constexpr (FMT == kFmtFp8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t q = __nv_cvt_float_to_fp8(__fdiv_rn(x[4 * i + k], scale), __NV_SATFINITE, __NV_E4M3);
        w[i] |= q << (8 * k);
        x[4 * i + k] = fp8_to_f32(q);
      }
    }
    if (on) {
      *reinterpret_cast<uint2*>(dst + 8 * j) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(dst + D / 2 + 8 * j) = make_uint2(w[2], w[3]);
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
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float cf = fminf(fmaxf(rintf((x[8 * hf + i] - m) / s), 0.f), 15.f);
        packed |= (uint32_t)cf << (4 * i);
        x[8 * hf + i] = fmaf(cf, s, m);
      }
      if (on) {
        *reinterpret_cast<uint32_t*>(dst + hf * (D / 4) + 4 * j) = packed;
        if ((j & 3) == 0)
          *reinterpret_cast<__half2*>(dst + D / 2 + (hf * (D / 64) + j / 4) * 4) = __halves2half2(hs, hm);
      }
    }
  }
}

// Eight stored values (dims 8 d8 ..) of a row of a page
template <int D, int FMT>
__device__ __forceinline__ void load_kv8(const uint8_t* row, int d8, float (&v)[8]) {
  if constexpr (FMT == kFmtBf16) {
    unpack8(*reinterpret_cast<const uint4*>(row + 16 * d8), v);
  } else if constexpr (FMT == kFmtFp8) {
    const uint2 w = *reinterpret_cast<const uint2*>(row + 8 * d8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = fp8_to_f32((w.x >> (8 * i)) & 255u);
      v[4 + i] = fp8_to_f32((w.y >> (8 * i)) & 255u);
    }
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(row + 4 * d8);
    const __half2 sm = *reinterpret_cast<const __half2*>(row + D / 2 + (d8 / 4) * 4);
    const float s = __low2float(sm), m = __high2float(sm);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = fmaf((float)((w >> (4 * i)) & 15u), s, m);
  }
}

template <int D, int FMT, int ROT>
__global__ void __launch_bounds__(128) append_kernel(AppendArgs a) {
  using S = AppendShape<D>;
  constexpr int kLanes = S::kLanes, kRows = S::kRows;
  constexpr int kRowB = PageRow<D, FMT>::kBytes;
  __shared__ float s_rot[ROT == kRotPart ? kRows * D : 1];
  __shared__ float s_k[S::kSpan * D];      // stored keys of the block's tokens
  __shared__ int s_slot[S::kSpan];
  __shared__ int s_run[S::kSpan + 1];      // token index of each run's first token
  __shared__ int s_count[2];               // tokens, runs
  pdl_launch();
  pdl_wait();
  const int tid = threadIdx.x;
  const int j = tid % kLanes, r0 = tid / kLanes;
  const int tile0 = blockIdx.x * kRows;
  const size_t page_b = (size_t)a.num_layers * 2 * a.KH * kPageTok * kRowB;
  float* scratch = s_rot + (ROT == kRotPart ? r0 * D : 0);

  auto load_row = [&](int t, int head, float (&x)[16]) {
    const __nv_bfloat16* src = reinterpret_cast<const __nv_bfloat16*>(a.qkv) + (size_t)t * a.ld_qkv + (size_t)head * D;
    unpack8(*reinterpret_cast<const uint4*>(src + 8 * j), x);
    unpack8(*reinterpret_cast<const uint4*>(src + D / 2 + 8 * j), x + 8);
  };
  auto cos_row = [&](int t) -> const float* {
    if (ROT == kRotNone) return nullptr;
    int p = a.positions[t];
    if (p < 0 || p >= a.max_pos) {           // outside the table: reported, nearest row taken
      report_error(a.err, kErrBounds);
      p = p < 0 ? 0 : a.max_pos - 1;
    }
    return a.cos_sin + (size_t)p * a.rot_dim;
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

  int y = blockIdx.y;
  if (y < a.q_groups) {
    // ---- q heads
    const int t = tile0 + r0;
    const bool on = t < a.T;
    const int h1 = min(a.Hq, (y + 1) * a.heads_per_group);
    const float* cs = on ? cos_row(t) : a.cos_sin;
    for (int h = y * a.heads_per_group; h < h1; ++h) {
      float x[16];
      load_row(on ? t : 0, h, x);
      norm_rotate<D, ROT>(x, reinterpret_cast<const __nv_bfloat16*>(a.wq), a.eps, j, cs, a.rot_dim, scratch);
      if (on) {
        __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.q_out) + (size_t)t * a.ld_out + (size_t)h * D;
        *reinterpret_cast<uint4*>(dst + 8 * j) = pack8(x);
        *reinterpret_cast<uint4*>(dst + D / 2 + 8 * j) = pack8(x + 8);
      }
    }
    return;
  }
  y -= a.q_groups;
  if (y < a.v_groups) {
    // ---- v heads
    const int t = tile0 + r0;
    const int slot = t < a.T ? a.slots[t] : -1;
    const int page = page_of(slot);
    const bool on = page >= 0;
    const int h1 = min(a.KH, (y + 1) * a.heads_per_group);
    for (int h = y * a.heads_per_group; h < h1; ++h) {
      float x[16];
      load_row(on ? t : 0, a.Hq + a.KH + h, x);
      const float sc = FMT == kFmtFp8 ? a.kv_scale[(a.layer * 2 + 1) * a.KH + h] : 1.f;
      store_kv_row<D, FMT>(on ? kv_row(page, slot, 1, h) : nullptr, x, sc, j, on);
    }
    return;
  }
  // ---- one k head
  const int h = y - a.v_groups;
  const float sc = FMT == kFmtFp8 ? a.kv_scale[(a.layer * 2 + 0) * a.KH + h] : 1.f;
  int first = tile0, count = min(kRows, a.T - tile0);
  if (a.bounds != nullptr) {
    // the tokens of the runs that begin in this tile
    for (int i = tid; i < S::kSpan; i += 128) s_slot[i] = tile0 + i < a.T ? a.slots[tile0 + i] : -1;
    __syncthreads();
    if (tid == 0) {
      auto joins = [&](int prev, int cur) { return prev >= 0 && cur == prev + 1 && cur % kPageTok != 0; };
      int i = 0, runs = 0;
      if (tile0 > 0) {
        int prev = a.slots[tile0 - 1];
        while (i < count && joins(prev, s_slot[i])) prev = s_slot[i++];
      }
      s_count[0] = i;                        // the first token of this block
      int k = i;
      for (; k < S::kSpan && tile0 + k < a.T; ++k) {
        const bool j0 = k > i && joins(s_slot[k - 1], s_slot[k]);
        if (k >= count && !j0) break;
        if (!j0) s_run[runs++] = k;
      }
      s_run[runs] = k;
      s_count[1] = runs;
    }
    __syncthreads();
    const int skip = s_count[0];
    count = s_run[s_count[1]] - skip;
    if (s_count[1] == 0) count = 0;
    first = tile0 + skip;
  }
  for (int b = 0; b < count; b += kRows) {
    const int t = first + b + r0;
    const bool live = b + r0 < count;
    const int slot = live ? a.slots[t] : -1;
    const int page = page_of(slot);
    const bool on = page >= 0;
    float x[16];
    load_row(on ? t : 0, a.Hq + h, x);
    norm_rotate<D, ROT>(x, reinterpret_cast<const __nv_bfloat16*>(a.wk), a.eps, j, on ? cos_row(t) : a.cos_sin,
                        a.rot_dim, scratch);
    store_kv_row<D, FMT>(on ? kv_row(page, slot, 0, h) : nullptr, x, sc, j, on);
    if (a.bounds != nullptr && live) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s_k[(t - tile0) * D + (i < 8 ? 0 : D / 2 - 8) + 8 * j + i] = x[i];
    }
  }
  if (a.bounds == nullptr) return;
  __syncthreads();
  // ---- bounds: D / 8 threads a run, 8 dims each; rows of the page before the run come
  // from the pool (written by earlier calls), the run's own from shared memory
  constexpr int kTpr = D / 8;
  constexpr float kMax = FMT == kFmtFp8 ? 448.f : 3.3895313892515355e38f;
  const int d8 = tid % kTpr;
  for (int run = tid / kTpr; run < s_count[1]; run += 128 / kTpr) {
    const int k0 = s_run[run], k1 = s_run[run + 1];
    const int slot = s_slot[k0];
    const int page = slot >= 0 && slot / kPageTok < a.num_pages ? slot / kPageTok : -1;
    if (page < 0) continue;
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = INFINITY;
      hi[i] = -INFINITY;
    }
    auto take = [&](const float (&v)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool nan = v[i] != v[i];         // a NaN key may score anything
        lo[i] = fminf(lo[i], nan ? -kMax : v[i]);
        hi[i] = fmaxf(hi[i], nan ? kMax : v[i]);
      }
    };
    const uint8_t* base = kv_row(page, 0, 0, h);
    const int old = slot % kPageTok;
#pragma unroll 5
    for (int r = 0; r < old; ++r) {
      float v[8];
      load_kv8<D, FMT>(base + r * kRowB, d8, v);
      take(v);
    }
    for (int k = k0; k < k1; ++k) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = s_k[k * D + 8 * d8 + i];
      take(v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      lo[i] = fminf(fmaxf(lo[i], -kMax), kMax);
      hi[i] = fminf(fmaxf(hi[i], -kMax), kMax);
    }
    const size_t at = (((size_t)page * a.num_layers + a.layer) * a.KH + h) * 2 * D + 8 * d8;
    if constexpr (FMT == kFmtFp8) {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i / 4] |= (uint32_t)__nv_cvt_float_to_fp8(lo[i], __NV_SATFINITE, __NV_E4M3) << (8 * (i % 4));
        w[2 + i / 4] |= (uint32_t)__nv_cvt_float_to_fp8(hi[i], __NV_SATFINITE, __NV_E4M3) << (8 * (i % 4));
      }
      uint8_t* dst = reinterpret_cast<uint8_t*>(a.bounds) + at;
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      *reinterpret_cast<uint2*>(dst + D) = make_uint2(w[2], w[3]);
    } else {
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.bounds) + at;
      *reinterpret_cast<uint4*>(dst) = pack8(lo);
      *reinterpret_cast<uint4*>(dst + D) = pack8(hi);
    }
  }
}

template <int D, int FMT>
static void launch_append(const AppendArgs& a, cudaStream_t st) {
  const int tiles = (a.T + AppendShape<D>::kRows - 1) / AppendShape<D>::kRows;
  const dim3 grid(tiles, a.q_groups + a.v_groups + a.KH);
  if (a.rot_dim == 0) launch_kernel(append_kernel<D, FMT, kRotNone>, grid, dim3(128), 0, st, a);
  else if (a.rot_dim == D) launch_kernel(append_kernel<D, FMT, kRotFull>, grid, dim3(128), 0, st, a);
  else launch_kernel(append_kernel<D, FMT, kRotPart>, grid, dim3(128), 0, st, a);
}

void qk_norm_rope_kv_write(const AppendArgs& in, cudaStream_t st) {
  if (in.T <= 0) return;
  AppendArgs a = in;
  a.err = error_word();
  VRM_REQUIRE(a.D == 64 || a.D == 128, "qk_norm_rope_kv_write: head_dim must be 64 or 128");
  a.heads_per_group = 4;
  a.q_groups = (a.Hq + a.heads_per_group - 1) / a.heads_per_group;
  a.v_groups = (a.KH + a.heads_per_group - 1) / a.heads_per_group;
  VRM_REQUIRE(a.q_groups + a.v_groups + a.KH <= 65535, "qk_norm_rope_kv_write: too many heads");
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
// a larger sum of scores.  Which page is the last to be taken depends on differences of
// any size, so scores are summed in 64 bits, where products of 8-bit significands are
// exact, and the choice is the one exact arithmetic makes, ties to the lowest page.
//
// A bound becomes a double by moving its sign, exponent and significand bits into place
// without re-biasing the exponent: the same value times 2^-896 (bf16) or 2^-1016 (e4m3),
// zeros and subnormals included.  The common factor (up and dn carry 2^800 against
// underflow) does not change an order.
namespace {

constexpr int kSelThreads = 256;


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

__device__ __forceinline__ uint64_t sortable(double s) {
  if (s != s) return ~0ull;                      // a NaN is read first: it is not hidden
  const uint64_t b = (uint64_t)__double_as_longlong(s + 0.0);   // -0 counts as 0
  return (b >> 63) ? ~b : b | (1ull << 63);
}

}  // namespace

template <int D, bool F8>
__global__ void __launch_bounds__(kSelThreads) select_kernel(SelectArgs a) {
  constexpr int kEl = F8 ? 1 : 2;
  constexpr int kLaneB = D * kEl / 8;            // bytes of a min (or max) row per lane, 8 lanes a page
  constexpr int kDims = D / 8;                   // dims per lane
  extern __shared__ __align__(16) uint64_t s_key[];    // [candidates]
  __shared__ double s_up[D], s_dn[D];
  __shared__ uint32_t s_hist[256];
  __shared__ uint64_t s_sel[2];                  // prefix; entries still to take
  __shared__ uint32_t s_scan[kSelThreads / 32];
  pdl_launch();
  pdl_wait();
  const int kvh = blockIdx.x, t = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  RowOf row;
  if (!find_row(t, a.cu_q, a.context_lens, a.B, row)) return;
  int* out = a.out + ((size_t)t * a.KH + kvh) * a.budget;
  int total = row.n <= 0 ? 0 : (int)(((long long)row.n + kPageTok - 1) / kPageTok);
  total = min(total, a.max_pages);
  if (total <= a.budget) {
    for (int i = tid; i < a.budget; i += kSelThreads) out[i] = i < total ? i : -1;
    return;
  }
  const int need = a.budget - a.sinks - a.recent;
  const int m = total - a.sinks - a.recent;      // candidates: pages sinks .. sinks + m - 1, m > need
  for (int i = tid; i < a.sinks; i += kSelThreads) out[i] = i;
  for (int i = tid; i < a.recent; i += kSelThreads) out[a.budget - a.recent + i] = total - a.recent + i;
  if (need <= 0) return;

  for (int d = tid; d < D; d += kSelThreads) {
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + (size_t)t * a.ld_q + (size_t)kvh * a.G * D + d;
    double up = 0., dn = 0.;
    for (int g = 0; g < a.G; ++g) {
      const double x = (double)__bfloat162float(q[(size_t)g * D]);
      if (x >= 0.) up += x;
      else dn += x;                              // NaN lands here and spoils every score
    }
    const double f = __hiloint2double((1023 + 800) << 20, 0);
    s_up[d] = up * f;
    s_dn[d] = dn * f;
  }
  __syncthreads();

  const int sub = lane & 7, grp = lane >> 3;     // 8 lanes a page, 4 pages a warp
  double up[kDims], dn[kDims];
#pragma unroll
  for (int i = 0; i < kDims; ++i) {
    // 16-byte chunk i / (16 / kEl) of the lane: chunks are dealt round-robin to the lanes
    constexpr int kPer = kLaneB >= 16 ? 16 / kEl : kDims;
    const int d = (i / kPer) * (8 * kPer) + sub * kPer + i % kPer;
    up[i] = s_up[d];
    dn[i] = s_dn[d];
  }
  const int* bt = a.block_tables + (size_t)row.seq * a.bt_stride + a.sinks;
  for (int i0 = warp * 4; i0 < m; i0 += kSelThreads / 32 * 4) {
    const int i = i0 + grp;
    int page = i < m ? bt[i] : -1;
    const bool bad = i < m && (page < 0 || page >= a.num_pages);
    if (bad) report_error(a.err, kErrBounds);
    if (bad) page = -1;
    double s = 0.;
    if (page >= 0) {
      const uint8_t* b = reinterpret_cast<const uint8_t*>(a.bounds) +
                         (((size_t)page * a.num_layers + a.layer) * a.KH + kvh) * (size_t)(2 * D * kEl);
      constexpr int kChunks = kLaneB >= 16 ? kLaneB / 16 : 1;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        if constexpr (!F8) {
          const uint4 lo = ld_stream16(b + c * 128 + sub * 16), hi = ld_stream16(b + D * kEl + c * 128 + sub * 16);
          const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            double x0, x1, y0, y1;
            bf16x2_to_f64(wl[k], x0, x1);
            bf16x2_to_f64(wh[k], y0, y1);
            s = fma(dn[c * 8 + 2 * k], x0, s);
            s = fma(dn[c * 8 + 2 * k + 1], x1, s);
            s = fma(up[c * 8 + 2 * k], y0, s);
            s = fma(up[c * 8 + 2 * k + 1], y1, s);
          }
        } else {
          uint32_t wl[4], wh[4];
          if constexpr (kLaneB == 16) {
            const uint4 lo = ld_stream16(b + sub * 16), hi = ld_stream16(b + D + sub * 16);
            wl[0] = lo.x, wl[1] = lo.y, wl[2] = lo.z, wl[3] = lo.w;
            wh[0] = hi.x, wh[1] = hi.y, wh[2] = hi.z, wh[3] = hi.w;
          } else {
            const uint2 lo = ld_stream8(b + sub * 8), hi = ld_stream8(b + D + sub * 8);
            wl[0] = lo.x, wl[1] = lo.y;
            wh[0] = hi.x, wh[1] = hi.y;
          }
#pragma unroll
          for (int k = 0; k < kDims / 4; ++k) {
            double x[4], z[4];
            fp8x4_to_f64(wl[k], x);
            fp8x4_to_f64(wh[k], z);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s = fma(dn[4 * k + e], x[e], s);
              s = fma(up[4 * k + e], z[e], s);
            }
          }
        }
      }
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (sub == 0 && i < m) s_key[i] = bad ? 0ull : sortable(s);
  }
  __syncthreads();

  // radix selection of the need-th largest key, 8 bits a pass from the top
  uint64_t prefix = 0, left = (uint64_t)need;
  int shift = 56;
  bool all = false;                              // every key with this prefix is taken
  for (;; shift -= 8) {
    s_hist[tid] = 0;
    __syncthreads();
    const uint64_t mask = shift == 56 ? 0ull : ~0ull << (shift + 8);
    for (int i = tid; i < m; i += kSelThreads) {
      const uint64_t k = s_key[i];
      if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    // suffix sums over the 256 bins: thread tid owns bin 255 - tid
    const uint32_t c = s_hist[255 - tid];
    uint32_t incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    for (int w = 0; w < warp; ++w) incl += s_scan[w];
    if (incl >= left && incl - c < left) {
      s_sel[0] = prefix | ((uint64_t)(255 - tid) << shift);
      s_sel[1] = (left - (incl - c)) | (incl == left ? 1ull << 63 : 0ull);
    }
    __syncthreads();
    prefix = s_sel[0];
    left = s_sel[1] & ~(1ull << 63);
    all = s_sel[1] >> 63;
    if (all || shift == 0) break;
  }
  // keys above the prefix are taken, and of those that share it the first `left`
  const uint64_t mask = ~0ull << shift;
  const int per = (m + kSelThreads - 1) / kSelThreads;
  const int i0 = min(m, tid * per), i1 = min(m, i0 + per);
  uint32_t gt = 0, eq = 0;
  for (int i = i0; i < i1; ++i) {
    const uint64_t k = s_key[i] & mask;
    gt += k > prefix;
    eq += k == prefix;
  }
  // exclusive prefix of (gt, eq) over the threads, 16 bits each would overflow: two scans
  __shared__ uint32_t s_scan2[kSelThreads / 32];
  uint32_t ig = gt, ie = eq;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t vg = __shfl_up_sync(0xffffffffu, ig, o), ve = __shfl_up_sync(0xffffffffu, ie, o);
    if (lane >= o) {
      ig += vg;
      ie += ve;
    }
  }
  if (lane == 31) {
    s_scan[warp] = ig;
    s_scan2[warp] = ie;
  }
  __syncthreads();
  ig -= gt;
  ie -= eq;
  for (int w = 0; w < warp; ++w) {
    ig += s_scan[w];
    ie += s_scan2[w];
  }
  uint32_t pos = ig + min(ie, (uint32_t)left);
  for (int i = i0; i < i1; ++i) {
    const uint64_t k = s_key[i] & mask;
    const bool take = k > prefix || (k == prefix && ie < (uint32_t)left);
    ie += k == prefix;
    if (take) out[a.sinks + pos++] = a.sinks + i;
  }
}

template <int D, bool F8>
static void launch_select(const SelectArgs& a, cudaStream_t st) {
  const size_t smem = (size_t)a.max_pages * sizeof(uint64_t);
  auto kern = select_kernel<D, F8>;
  if (smem > 40 * 1024) VRM_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  launch_kernel(kern, dim3(a.KH, a.T), dim3(kSelThreads), smem, st, a);
}

void select_pages(const SelectArgs& in, cudaStream_t st) {
  if (in.T <= 0) return;
  SelectArgs a = in;
  a.err = error_word();
  VRM_REQUIRE(a.D == 64 || a.D == 128, "select_pages: head_dim must be 64 or 128");
  VRM_REQUIRE(a.max_pages <= 24576, "select_pages: more than 24576 pages a sequence");
  VRM_REQUIRE(a.T <= 65535, "select_pages: too many query rows");
  if (a.D == 128) a.f8 ? launch_select<128, true>(a, st) : launch_select<128, false>(a, st);
  else a.f8 ? launch_select<64, true>(a, st) : launch_select<64, false>(a, st);
  VRM_CUDA_CHECK(cudaGetLastError());
}

// ================================================================ attention over selected pages
namespace {

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t fp8x2_to_half2(uint32_t v) {
  __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)v, __NV_E4M3);
  return (uint32_t)h.x | ((uint32_t)h.y << 16);
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
  static constexpr int kKW = kKB / 4, kVW = kVB / 4;                // 32-bit words
  uint32_t k[2][kKW], v[4][kVW];
  uint32_t ks[FMT == kFmtQ4 ? 2 : 1], vs[FMT == kFmtQ4 ? 4 : 1];    // {scale, min}

  template <int W>
  static __device__ __forceinline__ void piece(uint32_t* dst, const uint8_t* p) {
    if constexpr (W == 4) {
      const uint4 x = ld_stream16(p);
      dst[0] = x.x, dst[1] = x.y, dst[2] = x.z, dst[3] = x.w;
    } else if constexpr (W == 2) {
      const uint2 x = ld_stream8(p);
      dst[0] = x.x, dst[1] = x.y;
    } else {
      dst[0] = ld_stream4(p);
    }
  }
  // rows >= `rows` (behind the context) are not read and count as zeros.  Four-bit rows
  // are 8-byte aligned only (16 for D = 128).
  __device__ __forceinline__ void load_k(const uint8_t* kp, int rows, int g, int c) {
    constexpr int W = kKW < 4 ? kKW : 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = g + 8 * h;
      const uint8_t* p = kp + r * kRowB;
      const bool on = r < rows;
#pragma unroll
      for (int i = 0; i < kKW; ++i) k[h][i] = 0u;
      if (FMT == kFmtQ4) ks[FMT == kFmtQ4 ? h : 0] = 0u;
      if (on) {
#pragma unroll
        for (int i = 0; i < kKW / W; ++i) piece<W>(&k[h][i * W], p + (i * 4 + c) * (W * 4));
        if constexpr (FMT == kFmtQ4) ks[h] = ld_stream4(p + D / 2 + (D == 128 ? c : c / 2) * 4);
      }
    }
  }
  __device__ __forceinline__ void load_v(const uint8_t* vp, int rows, int g, int c) {
    constexpr int W = kVW < 4 ? kVW : 4;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int r = 2 * c + (h & 1) + 8 * (h >> 1);
      const uint8_t* p = vp + r * kRowB;
      const bool on = r < rows;
#pragma unroll
      for (int i = 0; i < kVW; ++i) v[h][i] = 0u;
      if (FMT == kFmtQ4) vs[FMT == kFmtQ4 ? h : 0] = 0u;
      if (on) {
#pragma unroll
        for (int i = 0; i < kVW / W; ++i) piece<W>(&v[h][i * W], p + (i * 8 + g) * (W * 4));
        if constexpr (FMT == kFmtQ4) vs[h] = ld_stream4(p + D / 2 + (D == 128 ? g / 2 : g / 4) * 4);
      }
    }
  }
  // first of the four dims that step s of the score product takes from lane c
  static __device__ __forceinline__ int k_dim(int s, int c) {
    if constexpr (FMT == kFmtBf16) return (c + 4 * (s / 2)) * 8 + 4 * (s % 2);
    else if constexpr (FMT == kFmtFp8) return (c + 4 * (s / 4)) * 16 + 4 * (s % 4);
    else return c * (D / 4) + 4 * s;
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
        const uint32_t w = k[h][s / 2] >> (16 * (s % 2));       // two code bytes: four dims
        a[h] = codes_to_half2((w & 0xFu) | ((w & 0xF0u) << 12), s2, m2);
        a[2 + h] = codes_to_half2(((w >> 8) & 0xFu) | ((w & 0xF000u) << 4), s2, m2);
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
        const uint32_t x = __byte_perm(v[t0][dim / 4], v[t0 + 1][dim / 4], 0x40 + 0x11 * (dim % 4));
        a[q] = fp8x2_to_half2(x & 0xffffu);
      } else {
        const int dim = (D / 16) * hi + e, b = dim / 2;
        const uint32_t x = __byte_perm(v[t0][b / 4], v[t0 + 1][b / 4], 0x0400 + 0x0101 * (b % 4));
        const uint32_t s2 = __byte_perm(vs[t0], vs[t0 + 1], 0x5410), m2 = __byte_perm(vs[t0], vs[t0 + 1], 0x7632);
        a[q] = codes_to_half2(dim % 2 ? x >> 4 : x, s2, m2);
      }
    }
  }
};

}  // namespace

// One CTA of 4 warps per (kv head, query row, split); the warps of all splits take the
// row's pages in turn.  Scores are computed transposed, S^T = K Q^T: a page's 16 tokens
// fill the MMA rows and the group's (<= 8) heads its columns; O^T = V^T P^T likewise.
// Splits are the CTAs of one cluster and merge through distributed shared memory.
template <int D, int FMT>
__global__ void __launch_bounds__(128) attend_kernel(AttendArgs P) {
  using F = Frag<D, FMT>;
  constexpr int kSteps = D / 16;
  constexpr int kOS = D + 4;
  __shared__ float s_m[4][8], s_l[4][8];
  __shared__ float s_o[4 * 8 * kOS];
  __shared__ float s_co[8 * D], s_cm[8], s_cl[8];
  pdl_launch();
  pdl_wait();
  const int kvh = blockIdx.x, t = blockIdx.y, split = blockIdx.z, nsplit = gridDim.z;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  const int G = P.G, KH = P.KH;
  RowOf row;
  if (!find_row(t, P.cu_q, P.context_lens, P.B, row)) return;      // the same for the whole cluster
  const int* list = P.pages + ((size_t)t * KH + kvh) * P.S;
  const int* bt = P.block_tables + (size_t)row.seq * P.bt_stride;
  const size_t head_b = (size_t)kPageTok * F::kRowB;
  const size_t page_b = (size_t)P.num_layers * 2 * KH * head_b;
  const uint8_t* pool = reinterpret_cast<const uint8_t*>(P.cache) + ((size_t)P.layer * 2 * KH + kvh) * head_b;

  // Q as the B operand: step s, lane (g, c) holds dims k_dim(s, c) .. + 3 of head g
  uint2 qb[kSteps];
  {
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(P.q) + (size_t)t * P.ld_q + (size_t)(kvh * G + g) * D;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      qb[s] = g < G ? *reinterpret_cast<const uint2*>(q + F::k_dim(s, c)) : make_uint2(0u, 0u);
  }
  float scale_log2 = P.sm_scale * 1.4426950408889634f, v_scale = 1.f;
  if constexpr (FMT == kFmtFp8) {
    scale_log2 *= P.kv_scale[(P.layer * 2 + 0) * KH + kvh];
    v_scale = P.kv_scale[(P.layer * 2 + 1) * KH + kvh];
  }
  if constexpr (FMT != kFmtBf16) {
    // f16 operands: q times the power of two that brings its largest value to [1, 2)
    float mx = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
      mx = fmaxf(mx, fmaxf(fmaxf(fabsf(bf16_lo(qb[s].x)), fabsf(bf16_hi(qb[s].x))),
                           fmaxf(fabsf(bf16_lo(qb[s].y)), fabsf(bf16_hi(qb[s].y)))));
    mx = warp_max(mx);
    const int e = (int)(__float_as_uint(mx) >> 23);
    float f = 1.f;
    if (e > 1 && e < 253) {
      f = __uint_as_float((uint32_t)(254 - e) << 23);
      scale_log2 *= __uint_as_float((uint32_t)e << 23);
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      qb[s].x = pack_half2(bf16_lo(qb[s].x) * f, bf16_hi(qb[s].x) * f);
      qb[s].y = pack_half2(bf16_lo(qb[s].y) * f, bf16_hi(qb[s].y) * f);
    }
  }

  float o[kSteps][4];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  bool seen = false;

  const int stride = 4 * nsplit;
  for (int base = split * 4 + warp; base < P.S; base += 32 * stride) {
    // 32 list entries of this warp: logical page, physical page, tokens to read
    const int i = base + lane * stride;
    const int lp = i < P.S ? list[i] : -1;
    int phys = 0, rows = 0;
    if (lp >= 0 && lp < P.max_pages && (long long)lp * kPageTok < row.n) {
      phys = bt[lp];
      if (phys >= 0 && phys < P.num_pages) rows = min(kPageTok, row.n - lp * kPageTok);
      else report_error(P.err, kErrBounds);
    }
    const int cnt = min(32, (P.S - base + stride - 1) / stride);
    for (int j = 0; j < cnt; ++j) {
      const int r = __shfl_sync(0xffffffffu, rows, j);
      const int ph = __shfl_sync(0xffffffffu, phys, j);
      if (r == 0) continue;
      seen = true;
      const uint8_t* kp = pool + (size_t)ph * page_b;
      F f;
      f.load_k(kp, r, g, c);
      f.load_v(kp + (size_t)KH * head_b, r, g, c);
      float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        uint32_t a[4];
        f.k_frag(s, a);
        if constexpr (FMT == kFmtBf16) mma_bf16_16816(sc, a[0], a[1], a[2], a[3], qb[s].x, qb[s].y);
        else mma_f16(sc, a[0], a[1], a[2], a[3], qb[s].x, qb[s].y);
      }
      // sc[0] = (token g, head 2c), [1] = (g, 2c + 1), [2] = (g + 8, 2c), [3] = (g + 8, 2c + 1)
      float x[4] = {sc[0] * scale_log2, sc[1] * scale_log2, sc[2] * scale_log2, sc[3] * scale_log2};
      if (g >= r) x[0] = x[1] = -INFINITY;
      if (g + 8 >= r) x[2] = x[3] = -INFINITY;
      float mx[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
      float alpha[2], pr[4];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        mx[q] = fmaxf(mx[q], __shfl_xor_sync(0xffffffffu, mx[q], 4));
        mx[q] = fmaxf(mx[q], __shfl_xor_sync(0xffffffffu, mx[q], 8));
        mx[q] = fmaxf(mx[q], __shfl_xor_sync(0xffffffffu, mx[q], 16));
        const float m_new = fmaxf(m_run[q], mx[q]);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        alpha[q] = exp2f(m_run[q] - m_use);
        pr[q] = exp2f(x[q] - m_use);
        pr[2 + q] = exp2f(x[2 + q] - m_use);
        m_run[q] = m_new;
        l_run[q] = l_run[q] * alpha[q] + (pr[q] + pr[2 + q]);
      }
#pragma unroll
      for (int e = 0; e < kSteps; ++e) {
        o[e][0] *= alpha[0];
        o[e][1] *= alpha[1];
        o[e][2] *= alpha[0];
        o[e][3] *= alpha[1];
      }
      uint32_t pb0, pb1;
      if constexpr (FMT == kFmtBf16) {
        pb0 = transpose8x8(pack_bf16x2(pr[0], pr[1]));
        pb1 = transpose8x8(pack_bf16x2(pr[2], pr[3]));
      } else {
        pb0 = transpose8x8(pack_half2(pr[0], pr[1]));
        pb1 = transpose8x8(pack_half2(pr[2], pr[3]));
      }
#pragma unroll
      for (int e = 0; e < kSteps; ++e) {
        uint32_t a[4];
        f.v_frag(e, a);
        if constexpr (FMT == kFmtBf16) mma_bf16_16816(o[e], a[0], a[1], a[2], a[3], pb0, pb1);
        else mma_f16(o[e], a[0], a[1], a[2], a[3], pb0, pb1);
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
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(P.out) + (size_t)t * P.ld_o + (size_t)kvh * G * D;
  for (int idx = threadIdx.x; idx < G * D; idx += 128) {
    const int h = idx / D, d = idx % D;
    float M = fmaxf(fmaxf(s_m[0][h], s_m[1][h]), fmaxf(s_m[2][h], s_m[3][h]));
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (M == -INFINITY) {
        L += s_l[w][h];                                    // 0, or NaN
      } else if (s_m[w][h] != -INFINITY) {
        const float f = exp2f(s_m[w][h] - M);
        L += s_l[w][h] * f;
        acc += s_o[(w * 8 + h) * kOS + d] * f;
      }
    }
    if (nsplit == 1) {
      out[idx] = __float2bfloat16(L == 0.f ? 0.f : acc / L * v_scale);
    } else {
      s_co[idx] = acc;
      if (d == 0) {
        s_cm[h] = M;
        s_cl[h] = L;
      }
    }
  }
  if (nsplit == 1) return;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int n = G * D, per = (n + nsplit - 1) / nsplit;
  const int i0 = split * per, i1 = min(n, i0 + per);
  for (int idx = i0 + threadIdx.x; idx < i1; idx += 128) {
    const int h = idx / D;
    float M = -INFINITY;
    for (int q = 0; q < nsplit; ++q) M = fmaxf(M, cluster.map_shared_rank(s_cm, q)[h]);
    float L = 0.f, acc = 0.f;
    for (int q = 0; q < nsplit; ++q) {
      const float mq = cluster.map_shared_rank(s_cm, q)[h], lq = cluster.map_shared_rank(s_cl, q)[h];
      if (M == -INFINITY) {
        L += lq;
      } else if (mq != -INFINITY) {
        const float w = exp2f(mq - M);
        L += w * lq;
        acc += w * cluster.map_shared_rank(s_co, q)[idx];
      }
    }
    out[idx] = __float2bfloat16(L == 0.f ? 0.f : acc / L * v_scale);
  }
  cluster.sync();     // peers' shared memory stays valid until every CTA has read it
}

template <int D, int FMT>
static void launch_attend(const AttendArgs& a, int splits, cudaStream_t st) {
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
  int splits = 1;
  while (splits < 8 && (long long)a.T * a.KH * splits * 2 <= 2ll * device_sm_count() && a.S >= 8 * splits) splits *= 2;
  auto go = [&](auto d) {
    constexpr int D = decltype(d)::value;
    if (a.fmt == kFmtQ4) launch_attend<D, kFmtQ4>(a, splits, st);
    else if (a.fmt == kFmtFp8) launch_attend<D, kFmtFp8>(a, splits, st);
    else launch_attend<D, kFmtBf16>(a, splits, st);
  };
  if (a.D == 128) go(std::integral_constant<int, 128>{});
  else go(std::integral_constant<int, 64>{});
  VRM_CUDA_CHECK(cudaGetLastError());
}

}  // namespace vrm
