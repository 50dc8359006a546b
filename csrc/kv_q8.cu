// rope_kv_write into 8-bit pages: rotary embedding of q (in place) and k, a scale per token and head, codes of k and v to the paged cache, one launch.
//
//   k' = R(pos) k      scale = max_i |x_i| / qmax      code_i = round(x_i / scale)      x = k' or v, in 32 bits; qmax 127 (int8) or 448 (e4m3)
//
// A row (one token, one head) lies in d / 16 neighbouring lanes, two times 16 bytes each, the two halves of a rotated pair in one lane, so its largest value
// takes log2(d / 16) shuffles and nothing is stored between: each value is read once and its code written once.  Codes are defined by the correctly rounded
// quotient x / scale (a product with the reciprocal rounds other values at the half steps).  It is formed from r = 1 / scale, one per row, by Markstein's
// correction: q = x r, q + r (x - q scale); a division per value would make the instructions, not the memory, the bound (8192 tokens of 32 heads of
// 128: 130 us).  The scales stand apart from the codes, so that a
// page's codes stay one block of block_size * d bytes whatever the head size.  Rows with a NaN or an infinity get scale NaN: what reads them sees it.
// Angles are formed from turns in 64 bits, pos * f - rint(pos * f), one per token and frequency: at position 30000 the 32-bit product is off by
// 2e-3 radians, half a bf16 step of the result.
//
// One block handles a token: its sines and cosines are formed once for all heads and stay in registers (a sine per lane and head would take as long as the
// copy).  A prompt's tokens have a block each; a step's few tokens are split over blocks, down to a row's warp each, so that they are in flight at once.
#include "common.cuh"

#include <cuda_fp8.h>
#include <math.h>

namespace {

constexpr int kWarps = 4;

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


// quotients x / scale, correctly rounded for scales of 2^-100 and more, r = 1 / scale
__device__ __forceinline__ void quotients(float (&q)[8], const float (&x)[8], float scale, float r) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    float e0, e1;
    fmul2(q[i], q[i + 1], x[i], x[i + 1], r, r);
    ffma2(e0, e1, q[i], q[i + 1], -scale, -scale, x[i], x[i + 1]);
    ffma2(q[i], q[i + 1], e0, e1, r, r, q[i], q[i + 1]);
  }
}

template <int FMT>
__device__ __forceinline__ uint2 codes8(const float (&q)[8]) {
  if constexpr (FMT == 1) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {               // 1.5 * 2^23 + q: rounded to a whole number, whose low byte is the code
      float a, b;
      fadd2(a, b, q[i], q[i + 1], 12582912.0f, 12582912.0f);
      w[i] = __float_as_uint(a), w[i + 1] = __float_as_uint(b);
    }
    return make_uint2(prmt(prmt(w[0], w[1], 0x0040), prmt(w[2], w[3], 0x0040), 0x5410), prmt(prmt(w[4], w[5], 0x0040), prmt(w[6], w[7], 0x0040), 0x5410));
  } else {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __nv_cvt_float2_to_fp8x2(make_float2(q[2 * i], q[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    return make_uint2(prmt(h[0], h[1], 0x5410), prmt(h[2], h[3], 0x5410));
  }
}

template <typename T, int FMT>
__global__ void __launch_bounds__(32 * kWarps) rope_kv_write_q8_kernel(T* __restrict__ qkv, const __grid_constant__ QArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s_cos[128], s_sin[128];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int step = gridDim.y * kWarps;
  const int first = blockIdx.y * kWarps + warp;
  const int slot = a.slots[t];
  const bool store = slot >= 0 && (int64_t)slot < a.num_slots;
  T* row = qkv + (int64_t)t * a.ld;
  const int64_t at0 = store ? (int64_t)(slot / a.block_size) * a.hkv * a.block_size + slot % a.block_size : 0;   // cache row of head 0
  const int sub = lane / a.lanes, i = lane % a.lanes;           // row of the warp, place in the row
  const int half = a.rotary_dim >> 1;
  // this lane's two vectors of a row (first columns); NEOX: a pair's halves
  const bool apart = a.style == LLMSS_ROPE_NEOX && i < half / 8;
  const int ca = apart ? i * 8 : i * 16, cb = apart ? i * 8 + half : i * 16 + 8;
  const bool turn_a = ca < a.rotary_dim, turn_b = cb < a.rotary_dim, has_b = cb < a.d;
  // items are rows of k, then of v, then of q, per_warp heads each; a warp takes every step-th.  One loop for the three kinds: what a step's few tokens run
  // comes cold from memory, and three loops are three times the instructions
  const int items = 2 * a.kv_items + a.q_items;
  uint4 ra = make_uint4(0u, 0u, 0u, 0u), rb = ra;
  T* p = nullptr;
  bool live = false;
  int kind = 0, h = 0;                                          // 0 k, 1 v, 2 q; head
  auto fetch = [&](int it) {
    kind = it < a.kv_items ? 0 : it < 2 * a.kv_items ? 1 : 2;
    h = (it - min(kind, 2) * a.kv_items) * a.per_warp + sub;
    p = row + (kind == 0 ? a.k_off : kind == 1 ? a.v_off : a.q_off) + h * a.d;
    live = it < items && sub < a.per_warp && (kind == 2 ? turn_a && h < a.hq : store && h < a.hkv);
    ra = rb = make_uint4(0u, 0u, 0u, 0u);
    if (live) {
      ra = *reinterpret_cast<const uint4*>(p + ca);
      if (has_b) rb = *reinterpret_cast<const uint4*>(p + cb);
    }
  };
  fetch(first);                                                 // in flight while the angles are formed
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) cs[e] = 1.f, sn[e] = 0.f;
  if (a.style != LLMSS_ROPE_NONE) {
    const double pos = (double)a.positions[t];
    for (int x = threadIdx.x; x < half; x += 32 * kWarps) {
      const double turns = pos * a.turns[x];
      sincospif(2.0f * (float)(turns - rint(turns)), &s_sin[x], &s_cos[x]);
    }
    __syncthreads();
    // of this lane's pairs: NEOX eight neighbouring ones, GPT-J four of each vector
    const int fa = apart ? ca : ca >> 1, fb = apart ? ca + 4 : cb >> 1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (turn_a) cs[e] = s_cos[fa + e], sn[e] = s_sin[fa + e];
      if (turn_b) cs[4 + e] = s_cos[fb + e], sn[4 + e] = s_sin[fb + e];
    }
  }
  auto turn = [&](float (&x)[8], float (&y)[8]) {
    if (a.style == LLMSS_ROPE_NEOX) {
      if (apart) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float u0, u1, w0, w1;
          fmul2(u0, u1, y[e], y[e + 1], -sn[e], -sn[e + 1]);
          fmul2(w0, w1, x[e], x[e + 1], sn[e], sn[e + 1]);
          ffma2(x[e], x[e + 1], x[e], x[e + 1], cs[e], cs[e + 1], u0, u1);
          ffma2(y[e], y[e + 1], y[e], y[e + 1], cs[e], cs[e + 1], w0, w1);
        }
      }
    } else if (a.style == LLMSS_ROPE_GPTJ) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {                             // columns that are not turned: cos 1, sin 0
        const float x0 = x[2 * e], x1 = x[2 * e + 1], y0 = y[2 * e], y1 = y[2 * e + 1];
        x[2 * e] = x0 * cs[e] - x1 * sn[e];
        x[2 * e + 1] = x1 * cs[e] + x0 * sn[e];
        y[2 * e] = y0 * cs[4 + e] - y1 * sn[4 + e];
        y[2 * e + 1] = y1 * cs[4 + e] + y0 * sn[4 + e];
      }
    }
  };
  constexpr float kTop = FMT == 1 ? 127.0f : 448.0f;
  // the row in x, y (zeros where the lane has none) -> codes and scale of cache row h
  auto put = [&](float (&x)[8], float (&y)[8], bool mine, int h, uint8_t* codes, float* scales) {
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max_nan(m, max_nan(fabsf(x[e]), fabsf(y[e])));
    if (a.per_warp > 1) {
      for (int o = a.lanes >> 1; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    } else {
      if (!mine) m = 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    float scale, q[8], w[8];
    if (__any_sync(0xffffffffu, m > 0.f && m < 0x1p-90f)) {
      // a reciprocal, or what is left of a quotient, might have no 32-bit number; a scale below the normal numbers may be half a step off
      scale = __fdiv_rn(m, kTop);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        q[e] = scale > 0.f ? fminf(kTop, fmaxf(-kTop, __fdiv_rn(x[e], scale))) + 0.f : 0.f;
        w[e] = scale > 0.f ? fminf(kTop, fmaxf(-kTop, __fdiv_rn(y[e], scale))) + 0.f : 0.f;
      }
    } else {
      scale = m * (1.0f / kTop);
      scale = fmaf(fmaf(-scale, kTop, m), 1.0f / kTop, scale);
      const float r = m > 0.f ? __frcp_rn(scale) : 0.f;
      quotients(q, x, scale, r);
      quotients(w, y, scale, r);
    }
    const bool finite = m < INFINITY;                           // not of NaN
    const uint32_t keep = finite ? 0xffffffffu : 0u;
    if (mine) {
      const int64_t at = at0 + h * a.block_size;
      uint8_t* dst = codes + at * a.d;
      const uint2 c = codes8<FMT>(q), d = codes8<FMT>(w);
      *reinterpret_cast<uint2*>(dst + ca) = make_uint2(c.x & keep, c.y & keep);
      if (has_b) *reinterpret_cast<uint2*>(dst + cb) = make_uint2(d.x & keep, d.y & keep);
      if (i == 0) scales[at] = finite ? scale : __int_as_float(0x7fc00000);
    }
  };
  for (int it = first; it < items; it += step) {
    float x[8], y[8];
    unpack8<T>(ra, x);
    unpack8<T>(rb, y);
    const bool mine = live;
    const int kind0 = kind, h0 = h;
    T* to = p;
    fetch(it + step);
    if (kind0 != 1) turn(x, y);
    if (kind0 == 2) {
      if (mine) {
        *reinterpret_cast<uint4*>(to + ca) = pack8<T>(x);
        if (turn_b) *reinterpret_cast<uint4*>(to + cb) = pack8<T>(y);
      }
    } else if (store) {
      put(x, y, mine, h0, kind0 == 0 ? a.k : a.v, kind0 == 0 ? a.k_scale : a.v_scale);
    }
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
  a.lanes = (d + 15) / 16;
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
