// rope_kv_write into 8-bit pages: rotary embedding of q (in place) and k, a scale per token and head, codes of k and v to the paged cache, one launch.
//
//   k' = R(pos) k      scale = max_i |x_i| / qmax      code_i = round(x_i / scale)      x = k' or v, in 32 bits; qmax 127 (int8) or 448 (e4m3)
//
// A row (one token, one head) lies in d / 8 neighbouring lanes, 16 bytes each, so its largest value takes log2(d / 8) shuffles and nothing is
// stored between: each value is read once and its code written once.  The divisions are the correctly rounded ones: codes are defined by them (a
// product with the reciprocal rounds other values at the half steps), and they hide behind the loads.  The scales stand apart from the codes, so that a
// page's codes stay one block of block_size * d bytes whatever the head size.  Rows with a NaN or an infinity get scale NaN: what reads them sees it.
// Angles are formed from turns in 64 bits, pos * f - rint(pos * f), one per token and frequency: at position 30000 the 32-bit product is off by
// 2e-3 radians, half a bf16 step of the result.
//
// One block handles a token: its sines and cosines are formed once for all heads (a sine per lane and head would take as long as the copy).  A prompt's
// tokens have a block each; a step's few tokens are split over blocks of 8 rows' warps, so that they are in flight at once.
#include "common.cuh"

#include <cuda_fp8.h>
#include <math.h>

namespace {

constexpr int kWarps = 8;

struct QArgs {
  const int* positions;
  const int* slots;
  uint8_t* k;
  uint8_t* v;
  float* k_scale;
  float* v_scale;
  int64_t ld;
  int64_t num_slots;
  int hq, hkv, d, rotary_dim, style, q_off, k_off, v_off, block_size;
  int lanes, per_warp;            // lanes of a row, rows of a warp
  int q_items, kv_items;          // warps' worth of q rows (0: no rotation) and of k (or v) rows
  double turns[128];              // base^(-2 i / rotary_dim) / (2 pi)
};

template <int FMT>
__device__ __forceinline__ uint2 codes8(const float (&f)[8], float scale) {
  uint2 r = make_uint2(0u, 0u);
  if (!(scale > 0.f)) return r;   // a row of zeros, or one that is not finite
  if constexpr (FMT == 1) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = min(127, max(-127, __float2int_rn(__fdiv_rn(f[i], scale))));
      w[i >> 2] |= ((uint32_t)c & 0xffu) << (8 * (i & 3));
    }
    r = make_uint2(w[0], w[1]);
  } else {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f[2 * i], scale), __fdiv_rn(f[2 * i + 1], scale)), __NV_SATFINITE, __NV_E4M3);
    r = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
  }
  return r;
}

template <typename T, int FMT>
__global__ void __launch_bounds__(32 * kWarps) rope_kv_write_q8_kernel(T* __restrict__ qkv, const __grid_constant__ QArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s_cos[128], s_sin[128];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int items = a.q_items + 2 * a.kv_items;
  const int step = gridDim.y * kWarps;
  const int first = blockIdx.y * kWarps + warp;
  const int slot = a.slots[t];
  const bool store = slot >= 0 && (int64_t)slot < a.num_slots;
  T* row = qkv + (int64_t)t * a.ld;
  const int sub = lane / a.lanes, c = (lane % a.lanes) * 8;     // row of the warp, column of the row
  // item -> this lane's vector; rows beyond the last head are the lanes' own business (`live`)
  auto place = [&](int it, int& kind, int& h, T*& p) {
    kind = it < a.q_items ? 0 : it < a.q_items + a.kv_items ? 1 : 2;
    h = (it - (kind == 0 ? 0 : kind == 1 ? a.q_items : a.q_items + a.kv_items)) * a.per_warp + sub;
    p = row + (kind == 0 ? a.q_off : kind == 1 ? a.k_off : a.v_off) + h * a.d + c;
    return sub < a.per_warp && h < (kind == 0 ? a.hq : a.hkv) && (kind != 0 || c < a.rotary_dim) && (kind == 0 || store);
  };
  int kind = 0, h = 0;
  T* p = nullptr;
  uint4 raw = make_uint4(0u, 0u, 0u, 0u);
  bool live = first < items && place(first, kind, h, p);
  if (live) raw = *reinterpret_cast<const uint4*>(p);           // in flight while the angles are formed
  const int half = a.rotary_dim >> 1;
  if (a.style != LLMSS_ROPE_NONE) {
    const double pos = (double)a.positions[t];
    for (int i = threadIdx.x; i < half; i += 32 * kWarps) {
      const double x = pos * a.turns[i];
      sincospif(2.0f * (float)(x - rint(x)), &s_sin[i], &s_cos[i]);
    }
    __syncthreads();
  }
  for (int it = first; it < items; it += step) {
    int kind2 = 0, h2 = 0;
    T* p2 = nullptr;
    uint4 raw2 = make_uint4(0u, 0u, 0u, 0u);
    const bool live2 = it + step < items && place(it + step, kind2, h2, p2);
    if (live2) raw2 = *reinterpret_cast<const uint4*>(p2);
    float f[8];
    unpack8<T>(raw, f);
    if (kind < 2 && a.style == LLMSS_ROPE_GPTJ) {
      if (c < a.rotary_dim) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float sn = s_sin[(c >> 1) + i], cs = s_cos[(c >> 1) + i], x1 = f[2 * i], x2 = f[2 * i + 1];
          f[2 * i] = x1 * cs - x2 * sn;
          f[2 * i + 1] = x2 * cs + x1 * sn;
        }
      }
    } else if (kind < 2 && a.style == LLMSS_ROPE_NEOX) {
      // the partner of column c is half a rotation away, in another lane of the row (half is a multiple of 8)
      const bool lo = c < half;
      const int other = lo ? lane + half / 8 : lane - half / 8;
      float g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = __shfl_sync(0xffffffffu, f[i], other & 31);
      if (c < a.rotary_dim) {
        const int w = lo ? c : c - half;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float sn = s_sin[w + i], cs = s_cos[w + i];
          f[i] = lo ? f[i] * cs - g[i] * sn : f[i] * cs + g[i] * sn;
        }
      }
    }
    if (kind == 0) {
      if (live) *reinterpret_cast<uint4*>(p) = pack8<T>(f);
    } else if (store) {                                          // uniform over the warp
      float m = 0.f;
      bool fin = true;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m = fmaxf(m, fabsf(f[i]));
        fin = fin && isfinite(f[i]);
      }
      if (!fin) m = INFINITY;                                    // a maximum drops NaNs: infinity stands for both
      if (a.per_warp > 1) {
        for (int o = a.lanes >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      } else {
        if (!live) m = 0.f;
        m = warp_max(m);
      }
      const float scale = isfinite(m) ? __fdiv_rn(m, FMT == 1 ? 127.0f : 448.0f) : __int_as_float(0x7fc00000);
      if (live) {
        const int64_t r = ((int64_t)(slot / a.block_size) * a.hkv + h) * a.block_size + slot % a.block_size;
        *reinterpret_cast<uint2*>((kind == 1 ? a.k : a.v) + r * a.d + c) = codes8<FMT>(f, scale);
        if (c == 0) (kind == 1 ? a.k_scale : a.v_scale)[r] = scale;
      }
    }
    kind = kind2;
    h = h2;
    p = p2;
    raw = raw2;
    live = live2;
  }
}

}  // namespace

// qkv [T][>= columns] (row stride ld): q rotated in place, k and v columns read only.  Pages [num_blocks][hkv][block_size][d] of bytes, scales
// [num_blocks][hkv][block_size]; slot < 0 or beyond the pages: the token is not written.  fmt: 1 int8, 2 e4m3.
LLMSS_API int llmss_rope_kv_write_q8(void* qkv, const int* positions, const int* slot_mapping, void* k_pages, void* k_scale, void* v_pages,
                                     void* v_scale, int T, int64_t ld, int hq, int hkv, int d, int rotary_dim, int style, float base, int q_off,
                                     int k_off, int v_off, int block_size, int num_blocks, int fmt, int dtype, cudaStream_t stream) {
  LLMSS_REQUIRE(dtype == LLMSS_F16 || dtype == LLMSS_BF16, "rope_kv_write_q8: dtype must be f16/bf16");
  LLMSS_REQUIRE(fmt == 1 || fmt == 2, "rope_kv_write_q8: page format %d unknown (1 int8, 2 e4m3)", fmt);
  LLMSS_REQUIRE(d > 0 && d % 8 == 0 && d <= 256, "rope_kv_write_q8: head_dim=%d must be a multiple of 8 up to 256", d);
  LLMSS_REQUIRE(hq > 0 && hkv > 0 && block_size > 0 && num_blocks >= 0 && T >= 0, "rope_kv_write_q8: bad sizes (hq=%d hkv=%d block=%d)", hq, hkv, block_size);
  LLMSS_REQUIRE(ld % 8 == 0 && q_off % 8 == 0 && k_off % 8 == 0 && v_off % 8 == 0 && ((uintptr_t)qkv % 16) == 0,
                "rope_kv_write_q8: rows, offsets and stride must be multiples of 16 bytes");
  LLMSS_REQUIRE(q_off >= 0 && k_off >= 0 && v_off >= 0 && (int64_t)q_off + (int64_t)hq * d <= ld && (int64_t)k_off + (int64_t)hkv * d <= ld &&
                    (int64_t)v_off + (int64_t)hkv * d <= ld,
                "rope_kv_write_q8: q/k/v column ranges exceed the row stride");
  LLMSS_REQUIRE((((uintptr_t)k_pages | (uintptr_t)v_pages) % 8) == 0 && (((uintptr_t)k_scale | (uintptr_t)v_scale) % 4) == 0,
                "rope_kv_write_q8: pages must be 8-byte and scales 4-byte aligned");
  LLMSS_REQUIRE(style == LLMSS_ROPE_NONE || style == LLMSS_ROPE_GPTJ || style == LLMSS_ROPE_NEOX, "rope_kv_write_q8: rotation style %d unknown", style);
  LLMSS_REQUIRE(style == LLMSS_ROPE_NONE || (rotary_dim > 0 && rotary_dim <= d && rotary_dim % 16 == 0 && base > 0.f),
                "rope_kv_write_q8: rotary_dim=%d must be a multiple of 16 and <= head_dim, base positive", rotary_dim);
  if (T == 0) return 0;
  QArgs a;
  memset(&a, 0, sizeof(a));
  a.positions = positions;
  a.slots = slot_mapping;
  a.k = (uint8_t*)k_pages;
  a.v = (uint8_t*)v_pages;
  a.k_scale = (float*)k_scale;
  a.v_scale = (float*)v_scale;
  a.ld = ld;
  a.num_slots = (int64_t)num_blocks * block_size;
  a.hq = hq;
  a.hkv = hkv;
  a.d = d;
  a.rotary_dim = style == LLMSS_ROPE_NONE ? 0 : rotary_dim;
  a.style = style;
  a.q_off = q_off;
  a.k_off = k_off;
  a.v_off = v_off;
  a.block_size = block_size;
  a.lanes = d / 8;
  a.per_warp = (a.lanes & (a.lanes - 1)) == 0 ? 32 / a.lanes : 1;
  a.q_items = a.rotary_dim > 0 ? (hq + a.per_warp - 1) / a.per_warp : 0;
  a.kv_items = (hkv + a.per_warp - 1) / a.per_warp;
  for (int i = 0; i < a.rotary_dim / 2; ++i) a.turns[i] = exp2(-2.0 * i / a.rotary_dim * log2((double)base)) / 6.283185307179586476925;
  // one block per token; fewer tokens than fill the 148 SMs some times over: split a token's rows, down to one row per warp
  const int blocks = (a.q_items + 2 * a.kv_items + kWarps - 1) / kWarps;
  const int split = T >= 1184 ? 1 : (1184 + T - 1) / T;
  const dim3 grid(T, split < blocks ? split : blocks);
#define LLMSS_W(T_, F_) LLMSS_CHECK_CUDA(launch_pdl(rope_kv_write_q8_kernel<T_, F_>, grid, dim3(32 * kWarps), 0, stream, (T_*)qkv, a))
  if (dtype == LLMSS_F16) {
    if (fmt == 1) LLMSS_W(__half, 1);
    else LLMSS_W(__half, 2);
  } else {
    if (fmt == 1) LLMSS_W(__nv_bfloat16, 1);
    else LLMSS_W(__nv_bfloat16, 2);
  }
#undef LLMSS_W
  LLMSS_CHECK_CUDA(cudaGetLastError());
  return 0;
}
