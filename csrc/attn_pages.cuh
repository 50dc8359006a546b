// Shared by the kernels of attention over cache pages (attn_pages.cu, attn_pages_few.cu, attn_pages_tile.cu).
//
// Causal attention over a paged cache in 16 or 8 bits, with cached tokens that groups of sequences share.
//
//   s_jk = scale (q_j . K_k)      K_k = ks_k code_k      p = softmax over the keys k <= pos_j      out_j = sum_k p_jk vs_k code_k
//
// A sequence of a group (SharedPrefix) finds its first len keys in the group's pages and the others in its own; a softmax over both is the merge
// of the two parts by their maxima and sums.
#pragma once
#include "common.cuh"

#include <cuda.h>
#include <cuda_fp8.h>

namespace pages {

constexpr int kF16Pages = 0, kInt8 = 1, kE4M3 = 2;    // page formats; 0: the queries' own 16-bit type
constexpr int kScaled16 = 3;                          // inside: 8-bit pages as f16 with an exponent per 64 keys (TileScales)

struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  const float* ks;
  const float* vs;
  const struct TileScales* tile_scales;   // kScaled16: [sequence][hkv][page / 64]
  void* out;
  const int* tables;        // [num_seqs][max_blocks]
  const int* seq_lens;
  const int* cu;            // [num_seqs + 1]
  const int* g_tables;      // [groups][g_max_blocks]
  const int* g_lens;
  const int* g_first;       // [groups + 1]
  int64_t ldq, ldo;
  int num_seqs, total_q, max_blocks, g_max_blocks, groups;
  int hq, hkv, d, page, num_blocks;
  float scale_log2;
};

// sequence that owns query row t (cu ascending), -1: none
__device__ __forceinline__ int seq_of_row(const int* cu, int lo, int hi, int t) {
  if (t < cu[lo] || t >= cu[hi]) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

// group of a sequence, -1: none
__device__ __forceinline__ int group_of_seq(const AttnArgs& a, int s) {
  if (a.groups == 0 || s < a.g_first[0] || s >= a.g_first[a.groups]) return -1;
  int lo = 0, hi = a.groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.g_first[mid] <= s) lo = mid;
    else hi = mid;
  }
  return lo;
}

// a block id that does not exist reads block 0: a wrong table costs a wrong result, not a fault
__device__ __forceinline__ int checked_block(int id, int num_blocks) { return (unsigned)id < (unsigned)num_blocks ? id : 0; }

template <typename T, int FMT>
__device__ __forceinline__ float page_value(const void* p, int64_t i) {
  if constexpr (FMT == kInt8) return (float)reinterpret_cast<const int8_t*>(p)[i];
  else if constexpr (FMT == kE4M3) {
    __nv_fp8_e4m3 c;
    c.__x = reinterpret_cast<const uint8_t*>(p)[i];
    return (float)c;
  } else return to_f32(reinterpret_cast<const T*>(p)[i]);
}

// ---------------------------------------------------------------------------------------------------------------- parts of a softmax
// A part of a row: O [d], then the reference m (log2) and the sum l relative to which O stands, and two numbers of padding; all 32-bit.  Parts of the
// same row join in the merge kernel (attn_pages.cu).
constexpr int kPad = 4;
//
// Lists of few rows (attn_pages_few.cu) are cut where their warps' runs end: `info` says for each (segment, key head) where its parts lie.
struct FewInfo {
  int first_slot;      // of `slots`; < 0: one part, in `whole` (with groups) or already the result (without)
  int first_warp;     // the parts behind the first are the slots 2 j, j = first_warp + 1 .. last_warp (warps' numbers)
  int last_warp;
  int pad;
};

struct PartArgs {
  float* slots;        // [2 warps][rows][d + kPad]
  FewInfo* info;       // [segments][hkv]
  float* whole_own;    // [total_q][hq][d + kPad]
  float* whole_group;
  float* tile_own;     // [splits][total_q][hq][d + kPad]
  float* tile_group;
  int rows;            // of a slot
  int few_own, few_groups;        // lists of sequences / groups are cut into runs
  int own_splits, group_splits;   // or into this many stretches of keys each (0: not)
  int own_chunk, group_chunk;     // keys of a stretch
  int direct;                     // the tiled kernel writes results, not parts
};

struct Seg {
  int lo, hi;          // keys lo .. hi - 1
  int row0, rows;      // query rows (tokens)
  const int* table;
};

// first query row of sequence i, whatever the tables say inside of the call's rows
__device__ __forceinline__ int row_of(const AttnArgs& a, int i) { return min(max(a.cu[min(max(i, 0), a.num_seqs)], 0), a.total_q); }

__device__ __forceinline__ Seg own_segment(const AttnArgs& a, int i) {
  Seg s;
  const int g = group_of_seq(a, i);
  s.row0 = row_of(a, i);
  s.rows = row_of(a, i + 1) - s.row0;
  s.hi = min(a.seq_lens[i], a.max_blocks * a.page);
  s.lo = g < 0 ? 0 : max(0, min(a.g_lens[g], a.g_max_blocks * a.page));
  s.table = a.tables + (int64_t)i * a.max_blocks;
  return s;
}
__device__ __forceinline__ Seg group_segment(const AttnArgs& a, int g) {
  Seg s;
  s.row0 = row_of(a, a.g_first[g]);
  s.rows = row_of(a, a.g_first[g + 1]) - s.row0;
  s.lo = 0;
  s.hi = min(a.g_lens[g], a.g_max_blocks * a.page);
  s.table = a.g_tables + (int64_t)g * a.g_max_blocks;
  return s;
}
// last key that query row t of sequence s sees
__device__ __forceinline__ int row_pos(const AttnArgs& a, int s, int t) {
  return min(a.seq_lens[s] - a.cu[s + 1] + t, a.max_blocks * a.page - 1);
}

__device__ __forceinline__ float exp2_fast(float x) {  // 2^x, one MUFU; 2^-inf = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// ---------------------------------------------------------------------------------------------------------------- a row by itself
// By a warp: the softmax of one row over the keys first, first + step .. below end, in 32 bits; lane i holds the columns i, i + 32 .. .  Looks at no key
// that is not its row's.  M: type of 16-bit pages; row_of(key): its row of the cache.
template <typename T, typename M, int FMT, typename RowOf>
__device__ __forceinline__ void row_softmax(const AttnArgs& a, int tok, int head, int first, int step, int end, RowOf row_of, float (&o)[8], float& m, float& l) {
  const int lane = threadIdx.x & 31;
  float q[8];
  const T* qr = reinterpret_cast<const T*>(a.q) + (int64_t)tok * a.ldq + (int64_t)head * a.d;
  m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = lane + 32 * i < a.d ? to_f32(qr[lane + 32 * i]) : 0.f;
    o[i] = 0.f;
  }
  for (int j = first; j < end; j += step) {
    const int64_t r = row_of(j);
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.d) x = fmaf(q[i], page_value<M, FMT>(a.k, r * a.d + lane + 32 * i), x);
    x = warp_sum(x) * a.scale_log2;
    if constexpr (FMT == kScaled16) x *= a.tile_scales[r / 64].k_up;
    else if constexpr (FMT != kF16Pages) x *= a.ks[r];
    const float mn = fmaxf(m, x), al = m == mn ? 1.f : exp2f(m - mn), p = x == -INFINITY ? 0.f : exp2f(x - mn);
    l = l * al + p;
    float pv = p;
    if constexpr (FMT == kScaled16) pv *= 1.f / a.tile_scales[r / 64].v_down;
    else if constexpr (FMT != kF16Pages) pv *= a.vs[r];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] *= al;
      if (lane + 32 * i < a.d) o[i] = fmaf(pv, page_value<M, FMT>(a.v, r * a.d + lane + 32 * i), o[i]);
    }
    m = mn;
  }
}

// A product over a tile of keys brings a value that is not finite to every row (0 x NaN is NaN), those included that do not see its key.  So a row whose
// result is not finite is looked at once more, by a warp: where a hidden key of its tiles, of `from` .. `to` without first .. last, has such a value, the row
// is formed anew over first .. last alone.  Costs a look at the results of rows that do not see all keys of their tiles: 4 portions of 1000 tokens over 1800
// take as long as before (values looked at as they come into shared memory: 188 -> 205 us); that the code is there at all, 23.7 -> 24.4 us for a step of
// 64 sequences behind 4096 (looked at in front of the rows' stores 24.8, in the merge kernel 25.5).
// Where it happens it is slow, 0.7 us per key of a row and warp: 2 portions of 2000 tokens over 1000, 32 heads, 0.3 ms; with one NaN token near their front 27.
struct RowKeys {
  const int* table;
  int kvh, from, first, last, to;
};
__device__ __forceinline__ int64_t cache_row(const AttnArgs& a, const RowKeys& k, int key) {
  return ((int64_t)checked_block(k.table[key / a.page], a.num_blocks) * a.hkv + k.kvh) * a.page + key % a.page;
}
template <typename M, int FMT>
__device__ __noinline__ bool hidden_unfinite(const AttnArgs& a, const RowKeys& k) {
  bool found = false;
  for (int key = k.from; key <= k.to; ++key) {
    if (key >= k.first && key <= k.last) {
      key = k.last;
      continue;
    }
    const int64_t r = cache_row(a, k, key);
    if constexpr (FMT == kInt8 || FMT == kE4M3) found = found || !(fabsf(a.vs[r]) < INFINITY);
    for (int c = threadIdx.x & 31; c < a.d; c += 32) found = found || !(fabsf(page_value<M, FMT>(a.v, r * a.d + c)) < INFINITY);
  }
  return __any_sync(0xffffffffu, found);
}
// to `part` ([d], maximum, sum), or where that is null to the output
template <typename T, typename M, int FMT>
__device__ __noinline__ void row_anew(const AttnArgs& a, const RowKeys& k, int tok, int head, float* part) {
  float o[8], m, l;
  row_softmax<T, M, FMT>(a, tok, head, k.first, 1, k.last + 1, [&](int key) { return cache_row(a, k, key); }, o, m, l);
  const int lane = threadIdx.x & 31;
  T* out = reinterpret_cast<T*>(a.out) + (int64_t)tok * a.ldo + (int64_t)head * a.d;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (lane + 32 * i >= a.d) continue;
    if (part != nullptr) part[lane + 32 * i] = o[i];
    else out[lane + 32 * i] = from_f32<T>(k.last < k.first ? 0.f : o[i] / l);
  }
  if (part != nullptr && lane == 0) *reinterpret_cast<float2*>(part + a.d) = make_float2(m, l);
}

// Tiles of 64 keys in f16: code * scale / 2^E, E the exponent above the tile's largest scale, so that nothing leaves f16's range and a rounding is 2^-11 of
// the number or, where that is more, 2^-24 of the tile's largest scale.  E is held within -80 .. 120, which is every scale of rows of 16-bit numbers down to
// 2^-80: numbers below 2^-94 lose bits.  What goes with a tile: 2^E of the keys, E and 2^-E of the values.
struct TileScales {
  float k_up, v_exp, v_down, pad;
};
// E from two scales per lane (0 where the list has no key); scales that are not finite do not count, they make their own NaN
__device__ __forceinline__ int tile_exponent(float a, float b) {
  const unsigned x = __float_as_uint(a), y = __float_as_uint(b);
  const unsigned top = __reduce_max_sync(0xffffffffu, max(x < 0x7f800000u ? x : 0u, y < 0x7f800000u ? y : 0u));
  return max(-80, min(120, (int)(top >> 23) - 126));
}
__device__ __forceinline__ float two_to(int e) { return __int_as_float((127 + e) << 23); }
__device__ __forceinline__ TileScales tile_scales(int ek, int ev) {
  TileScales t;
  t.k_up = two_to(ek);
  t.v_exp = (float)ev;
  t.v_down = two_to(-ev);
  t.pad = 0.f;
  return t;
}

// four codes -> code * scale in f16, two words
template <int FMT>
__device__ __forceinline__ void convert4(uint32_t w, float scale, uint32_t& lo, uint32_t& hi) {
  float f[4];
  if constexpr (FMT == kInt8) {
    // 2^23 + (code + 128) as 32-bit numbers, less 2^23 + 128: exact
    w ^= 0x80808080u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t u;
      asm("prmt.b32 %0, %1, %2, %3;" : "=r"(u) : "r"(w), "r"(0x4B000000u), "r"(0x7540 + i));   // bytes: code, 0, 0, 0x4B
      f[i] = __uint_as_float(u);
    }
    fadd2(f[0], f[1], f[0], f[1], -8388736.0f, -8388736.0f);
    fadd2(f[2], f[3], f[2], f[3], -8388736.0f, -8388736.0f);
  } else {
    uint32_t a, b;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(a), "=r"(b) : "r"(w));
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&a)), y = __half22float2(*reinterpret_cast<const __half2*>(&b));
    f[0] = x.x, f[1] = x.y, f[2] = y.x, f[3] = y.y;
  }
  fmul2(f[0], f[1], f[0], f[1], scale, scale);
  fmul2(f[2], f[3], f[2], f[3], scale, scale);
  lo = pack16<__half>(f[0], f[1]);
  hi = pack16<__half>(f[2], f[3]);
}

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, int bytes, uint64_t* bar) {   // addresses and size multiples of 16
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
               "r"(smem_u32(bar))
               : "memory");
}

// pages as rows of bytes, copied in swizzled boxes of box_rows rows by up to 128 bytes
int encode_pages(CUtensorMap* map, const void* base, int64_t rows, int bytes, int box_rows);
// host side: which kernels a call takes, and its scratch
constexpr int kFewWarps = 4;       // attn_pages_few.cu: warps of a block
int few_blocks(int fmt, int d, int rows, int segs);                                       // attn_pages_few.cu: blocks of one launch
// `beside`: starts beside the kernel launched before it, whose results it does not need, and ends behind it
int few_launch(const AttnArgs& a, const PartArgs& p, int fmt, int dtype, int blocks, bool beside, cudaStream_t stream);
int tile_rows(int d, int64_t rows);                                                  // attn_pages_tile.cu: query rows of a block
// row tiles and stretches of keys of sequences (own) and of groups; 0 tiles: not this kernel's
struct TilePlan {
  int own_tiles, group_tiles, rows;
};
int tile_launch(const AttnArgs& a, const PartArgs& p, const TilePlan& t, int fmt, int dtype, cudaStream_t stream);

}  // namespace pages
