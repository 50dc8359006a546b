// Attention over cache pages for up to 16 query rows of a key head (single tokens, some tokens of grouped heads, a few sequences behind a prefix): bound by
// reading the cache.
//
// A warp takes 16 keys at a time, from a ring of its own in shared memory that the copy engine fills (TMA, 128-byte swizzle, two or three units ahead; no
// barrier between warps): keys are the rows (M) of S^T = K Q^T and the head's columns the rows of O^T = V^T P^T, so that 8 query rows cost no more than the
// instruction's narrow side, and what is read becomes fragments without a step between.  The order of a
// product's inner index is free, so a lane's 16 bytes of a key are its columns of D / 16 products one after another, and its 16 bytes of a value row are
// its rows of the output.  8-bit codes become f16 without rounding: e4m3 by the conversion instruction, int8 as (code + 128) 2^-24, which is the f16 whose
// bits are that byte, one logical operation for two.  What 128 adds is taken off the sums: 128 sum q from a score, 128 sum p (of the rounded p, from one
// more product with ones) from an output.  Queries become f16 after division by the power of two below their row's largest value (exact, but for what is 2^-14 of that and smaller).
//
//   x = s log2(e), y = x + log2(vs):  l = sum 2^(x - m),  O = sum 2^(y - m') code,  out = O 2^(m' - m) / l
//
// The scale of a value row joins its probability in the exponent, with a maximum of its own.  Maxima move when a score exceeds them by 8 only, and what is
// rounded to f16 is formed times 2^7, so that it is at most 2^15 whatever the scales are.
//
// Rows of a tree (TREE) see all cached keys and those of the new ones whose bit their mask has: 16 rows are at most 16 new tokens, so that a row's bits are one
// register, looked at in the units behind the cached keys alone.  64 trees of 10 tokens over 1040, 16 heads of 256: 187 us, 0.93 of the copy rate.
//
// The work of a call is the sum of all (sequence, key head) lists in units of 16 keys (32 where a key is 64 bytes); each warp takes an equal run of it,
// wherever sequences begin and end, and waits for no other.  A list within a warp's run is finished there; one that crosses runs leaves its parts in
// scratch, at most two per warp, and the merge kernel joins them.
#include "attn_pages.cuh"

namespace {

using namespace pages;

constexpr int kWarps = kFewWarps;
constexpr int kLeastUnits = 2;     // of a warp's run
constexpr int kKept = 2048;        // lists whose lengths a block keeps in shared memory

template <int FMT, int D, int NT>
struct Few {
  static constexpr int ESZ = FMT == kF16Pages ? 2 : 1;
  static constexpr int SUB = D * ESZ <= 64 ? 2 : 1;   // 16-key parts of a unit
  static constexpr int UNIT = 16 * SUB;
  static constexpr int KW = D * ESZ / 16;             // 32-bit words of a key per lane
  static constexpr int VW = D * ESZ / 32;             // of a value row
  static constexpr int EPC = 16 / ESZ;                // elements of 16 bytes
  static constexpr int KS = D / 16;                   // products of 16 columns
  static constexpr int Q_BYTES = NT * KS * 32 * 8;    // a warp's fragments of a list's queries
  static constexpr int ROW = D * ESZ < 128 ? D * ESZ : 128;   // bytes of a swizzled row: a key is BOXES of them
  static constexpr int BOXES = D * ESZ / ROW;
  static constexpr int HALF = UNIT * D * ESZ;         // keys, or values, of a unit
  static constexpr int STAGES = HALF <= 2048 ? 3 : 2;
  static constexpr int SCALES = FMT == kF16Pages ? 0 : 2 * UNIT * 4;
  static constexpr int FIXED = 1024 + kWarps * (STAGES * (2 * HALF + SCALES + 8) + Q_BYTES);
  static constexpr int MIN_CTAS = 4 * NT * KS <= 64 ? 3 : 2;   // outputs stay in registers; what else a thread holds is about 100
  static int smem(int segs) { return FIXED + 4 * (segs < kKept ? segs : kKept); }
  // blocks of an SM: by registers, and by 228 KB of shared memory less 1 KB per block
  static int ctas(int segs) {
    const int n = 233472 / (smem(segs) + 1024);
    return n < MIN_CTAS ? n : MIN_CTAS;
  }
};

struct FewArgs {
  int segs;            // lists per key head: sequences (own) and groups
  int own;
  int rows;            // query rows of a list at most
  uint32_t page_magic; // (key / 16) 2 this >> 32: the key's page
  int beside;          // wait for the kernel before at the end instead of at the start
};

__device__ __forceinline__ Seg segment(const AttnArgs& a, const FewArgs& f, int i) { return i < f.own ? own_segment(a, i) : group_segment(a, i - f.own); }
template <int UNIT>
__device__ __forceinline__ int units_of(const Seg& s) {
  return s.hi > s.lo && s.rows > 0 ? (s.hi - (s.lo & ~(UNIT - 1)) + UNIT - 1) / UNIT : 0;
}

// bytes 0 and 2 of w, two's complement, as f16 numbers below the normal range: the bits 0x00uu are u 2^-24, u = code + 128, without rounding
__device__ __forceinline__ uint32_t int8_pair(uint32_t w) {
  uint32_t u;
  asm("lop3.b32 %0, %1, 0x00ff00ff, 0x00800080, 0x6a;" : "=r"(u) : "r"(w));   // (w & mask) ^ 0x80 of both
  return u;
}
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {    // low two bytes
  uint32_t r;
  asm("{\n\t.reg .b16 h, x;\n\tmov.b32 {h, x}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_pair_hi(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 h, x;\n\tmov.b32 {x, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {   // 8 x 8 of 16-bit over the warp
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Key of a unit that stands in row i of the first product.  Neighbouring rows lie in chunk places that differ by four, and the even rows in places that
// differ by two, so that under the 128-byte swizzle (chunk ^ key & 7) no eight lanes meet in a bank, neither reading keys nor reading values.
__device__ __forceinline__ int key_of(int i) { return (i & 1) ? ((i - 1) ^ 5) : i; }   // 0 5 2 7 4 1 6 3

// Rows (bits of `rows`) of a list, or of its part (slot >= 0): formed anew over the keys from .. to that they see.
template <typename T, int FMT, int D, bool TREE>
__device__ __noinline__ void rows_anew(const AttnArgs& a, const PartArgs& pa, int own, int seg, int kvh, int from, int to, int slot, unsigned rows) {
  const Seg s = seg < own ? own_segment(a, seg) : group_segment(a, seg - own);
  const int group = a.hq / a.hkv;
  for (; rows != 0; rows &= rows - 1) {
    const int i = __ffs(rows) - 1, tok = s.row0 + i / group, head = kvh * group + i % group;
    const int sq = seg < own ? seg : seq_of_row(a.cu, 0, a.num_seqs, tok), ctx = TREE && sq >= 0 ? tree_context(a, sq) : 0;
    const int last = sq < 0 ? -1 : min(TREE ? ctx - 1 : row_pos(a, sq, tok), min(to, s.hi - 1));
    KeysOf<TREE> k;
    k.table = s.table, k.kvh = kvh, k.from = from, k.first = max(from, s.lo), k.last = last, k.to = to;
    // a prefix's keys are all cached ones: of those behind a row's context, which it does not see, no mask is asked
    if constexpr (TREE) k.to = min(to, seg < own ? s.hi - 1 : last), k.tok = tok, k.ctx = ctx;
    float* whole = (seg < own ? pa.whole_own : pa.whole_group) + ((int64_t)tok * a.hq + head) * (D + kPad);
    row_anew<T, T, FMT, TREE>(a, k, tok, head, slot >= 0 ? pa.slots + ((int64_t)slot * pa.rows + i) * (D + kPad) : a.groups == 0 ? nullptr : whole);
  }
}

template <typename T, int FMT, int D, int NT, bool TREE>
__global__ void __launch_bounds__(32 * kWarps, Few<FMT, D, NT>::MIN_CTAS)
attn_pages_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs a,
                      const __grid_constant__ PartArgs pa, const FewArgs f) {
  using C = Few<FMT, D, NT>;
  using M = typename std::conditional<FMT == kF16Pages, T, __half>::type;   // type of the products
  constexpr int UNIT = C::UNIT, SUB = C::SUB, KW = C::KW, VW = C::VW, KS = C::KS, EPC = C::EPC, STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_ring = smem;                                                   // [warps][STAGES][keys | values]
  float* s_scales = reinterpret_cast<float*>(s_ring + kWarps * STAGES * 2 * C::HALF);   // [warps][STAGES][of keys | of values]
  uint64_t* s_full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(s_scales) + kWarps * STAGES * C::SCALES);   // [warps][STAGES]
  uint2* s_q = reinterpret_cast<uint2*>(s_full + kWarps * STAGES);          // [warps][NT][KS][32] fragments, each lane's its own
  int* s_units = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(s_q) + kWarps * C::Q_BYTES);   // [min(segs, kKept)]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  if (!f.beside) pdl_wait();               // (beside: the kernel before lets this one start when its own wait is over)
  pdl_launch_dependents();                 // the merge reads lengths in front of its wait
  uint8_t* ring = s_ring + warp * STAGES * 2 * C::HALF;
  uint64_t* full = s_full + warp * STAGES;
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }

  s_q += warp * NT * KS * 32 + lane;

  // this warp's run of the lists
  for (int i = threadIdx.x; i < min(f.segs, kKept); i += 32 * kWarps) s_units[i] = units_of<UNIT>(segment(a, f, i));
  __syncthreads();
  auto count = [&](int i) { return i < kKept ? s_units[i] : units_of<UNIT>(segment(a, f, i)); };
  // (the host has checked that all lists together are below 2^31)
  auto scan = [&](int b, int& n) {         // lists b .. b + 31: this lane's units, and those up to it
    n = b + lane < f.segs ? count(b + lane) : 0;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
    return inc;
  };
  int n0;
  const int inc0 = scan(0, n0);
  unsigned units = __shfl_sync(0xffffffffu, inc0, 31);
  for (int b = 32; b < f.segs; b += 32) units += __reduce_add_sync(0xffffffffu, b + lane < f.segs ? count(b + lane) : 0);
  const unsigned total = units * a.hkv;
  const unsigned workers = gridDim.x * kWarps, me = blockIdx.x * kWarps + warp;
  const unsigned per = max((total + workers - 1) / workers, (unsigned)kLeastUnits);
  const unsigned begin = min(per * me, total), end = min(begin + per, total);
  if (begin >= end) {
    pdl_wait();
    return;
  }
  int seg = 0;
  unsigned before = 0;                     // units of the lists of earlier segments, one key head
  for (int b = 0; b < f.segs; b += 32) {
    int n = n0, inc = inc0;
    if (b > 0) inc = scan(b, n);
    const unsigned hit = __ballot_sync(0xffffffffu, (before + inc) * a.hkv > begin);
    if (hit) {
      const int w = __ffs(hit) - 1;
      seg = b + w;
      before += __shfl_sync(0xffffffffu, inc - n, w);
      break;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }

  // f16 ends at 2^16 and has no numbers below 2^-24: what is rounded to it is formed times 2^7 (at most 2^15)
  constexpr float kUp = std::is_same<M, __half>::value ? 7.0f : 0.0f;
  const int group = a.hq / a.hkv;
  auto page_of = [&](int key) { return (int)__umulhi((unsigned)key >> 4 << 1, f.page_magic); };

  // a place in the run: a list, or the part of it that lies in the run, and a unit in it
  struct Place {
    Seg s;
    unsigned before, cur;    // units before the segment (one key head), place of the list's part in the run
    int seg, kvh, n, u0, u1, base, u;
  };
  auto open = [&](Place& w) {              // the list at w.cur
    w.n = count(w.seg);
    while (w.cur >= (w.before + w.n) * a.hkv) {
      w.before += w.n;
      w.n = count(++w.seg);
    }
    w.s = segment(a, f, w.seg);
    const unsigned at = w.cur - w.before * a.hkv;
    w.kvh = at / w.n;
    w.u0 = at - w.kvh * w.n;
    w.u1 = min((unsigned)w.n, w.u0 + (end - w.cur));
    w.base = w.s.lo & ~(UNIT - 1);
    w.u = w.u0;
  };
  const uint64_t policy = l2_policy_evict_first();
  // copies run ahead of the products, from one list into the next
  Place w;
  w.seg = seg, w.before = before, w.cur = begin;
  open(w);
  Place z = w;                             // the products' place
  int blocks[SUB];
  bool more = true;
  auto settle = [&]() {                    // to a unit that exists; its blocks are looked up here and used at the next copy
    while (w.u >= w.u1) {
      w.cur += w.u1 - w.u0;
      if (w.cur >= end) {
        more = false;
        return;
      }
      open(w);
    }
#pragma unroll
    for (int i = 0; i < SUB; ++i) blocks[i] = w.s.table[page_of(min(w.base + w.u * UNIT + i * 16, w.s.hi - 1))];
  };
  auto copy = [&](int stage) {
    uint32_t row[SUB];
#pragma unroll
    for (int i = 0; i < SUB; ++i) {
      const int key = w.base + w.u * UNIT + i * 16;
      row[i] = ((uint32_t)checked_block(blocks[i], a.num_blocks) * a.hkv + w.kvh) * a.page + (key - page_of(key) * a.page);
    }
    if (elect_one()) {
      mbar_arrive_expect_tx(&full[stage], 2 * C::HALF + C::SCALES);
      uint8_t* dst = ring + stage * 2 * C::HALF;
      float* sc = s_scales + (warp * STAGES + stage) * (C::SCALES / 4);
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
#pragma unroll
        for (int b = 0; b < C::BOXES; ++b) {
          tma_load_2d(dst + (i * C::BOXES + b) * 16 * C::ROW, &map_k, &full[stage], b * C::ROW, (int)row[i], policy);
          tma_load_2d(dst + C::HALF + (i * C::BOXES + b) * 16 * C::ROW, &map_v, &full[stage], b * C::ROW, (int)row[i], policy);
        }
        if constexpr (FMT != kF16Pages) {
          bulk_copy(sc + i * 16, a.ks + row[i], 64, &full[stage]);
          bulk_copy(sc + UNIT + i * 16, a.vs + row[i], 64, &full[stage]);
        }
      }
    }
    __syncwarp();
    ++w.u;
    settle();
  };
  settle();
#pragma unroll 1                           // instructions come cold from memory: few of them before the first copies
  for (int i = 0; i < STAGES; ++i)
    if (more) copy(i);
  int stage = 0;
  uint32_t phase = 0;

  // this lane's places in a stage: keys key_of(r), + 8 (chunk t, t + 4 of a row), values of keys 2t, key_of(2t + 1), + 8 (chunk r)
  const int kk = key_of(r), v1 = key_of(2 * t + 1);
  const int k_off = C::ROW == 128 ? kk * 128 + ((t ^ kk) << 4) : kk * 64 + ((t ^ (kk >> 1 & 3)) << 4);
  int v_off[2];
  if constexpr (C::ROW == 128) v_off[0] = 2 * t * 128 + ((r ^ (2 * t)) << 4), v_off[1] = v1 * 128 + ((r ^ v1) << 4);
  else v_off[0] = 2 * t * 64 + (((r >> 1) ^ t) << 4) + (r & 1) * 8, v_off[1] = v1 * 64 + (((r >> 1) ^ (v1 >> 1)) << 4) + (r & 1) * 8;

  for (unsigned cur = begin; cur < end;) {
    const Seg s = z.s;
    const int n = z.n, kvh = z.kvh, u0 = z.u0, u1 = z.u1, base = z.base;
    seg = z.seg;
    const int nrows = min(s.rows * group, f.rows);

    // ---- queries: row r (and r + 8) lies in the four lanes that hold its fragments, a lane's 16 bytes of a key facing its own columns of the row
    float qs[NT][2], qb[NT][2];            // of rows 2t, 2t + 1: score factor, what 128 added to a score
    int pos[NT][2], all_pos = 0x7fffffff, max_pos = -1;   // and their last visible keys; the least and the largest of all rows
    // trees: the last of the cached tokens instead, and a bit for each of the new ones (16 rows are 16 of them at most) that the list has and the row sees
    uint32_t bits[NT][2];
    const int ctx = TREE && seg < f.own ? tree_context(a, seg) : 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int i = nt * 8 + r, tok = s.row0 + i / group;
      const bool live = i < nrows;
      const T* qr = reinterpret_cast<const T*>(a.q) + (int64_t)tok * a.ldq + (int64_t)(kvh * group + i % group) * D + t * EPC;
      uint4 raw[KS / 4][2];                // 16 columns each
#pragma unroll
      for (int c = 0; c < KS / 4; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int d0 = EPC == 16 ? c * 64 + h * 8 : (2 * c + h) * 32;
          raw[c][h] = live ? *reinterpret_cast<const uint4*>(qr + d0) : make_uint4(0u, 0u, 0u, 0u);
        }
      float up = 1.f, f_q = a.scale_log2, sum = 0.f;
      if constexpr (FMT != kF16Pages) {
        float mx = 0.f;
#pragma unroll
        for (int c = 0; c < KS / 4; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x[8];
            unpack8<T>(raw[c][h], x);
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const int e = mx > 0.f && mx < INFINITY ? max(-126, min(126, (int)((__float_as_uint(mx) >> 23) & 255) - 127)) : 0;
        up = __int_as_float((127 - e) << 23);
        f_q *= __int_as_float((127 + e) << 23);
      }
#pragma unroll
      for (int c = 0; c < KS / 4; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint2 w[2] = {make_uint2(raw[c][h].x, raw[c][h].y), make_uint2(raw[c][h].z, raw[c][h].w)};
          if constexpr (FMT != kF16Pages) {
            float x[8];
            unpack8<T>(raw[c][h], x);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float y[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) y[e] = x[4 * k + e] * up;
              // int8: a word's bytes 0, 2 and 1, 3 are converted together
              const __half2 lo = FMT == kInt8 ? __floats2half2_rn(y[0], y[2]) : __floats2half2_rn(y[0], y[1]);
              const __half2 hi = FMT == kInt8 ? __floats2half2_rn(y[1], y[3]) : __floats2half2_rn(y[2], y[3]);
              w[k] = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
              if constexpr (FMT == kInt8) {
                const float2 l2 = __half22float2(lo), h2 = __half22float2(hi);
                sum += (l2.x + l2.y) + (h2.x + h2.y);
              }
            }
          }
          s_q[(nt * KS + (2 * c + h) * 2) * 32] = w[0];
          s_q[(nt * KS + (2 * c + h) * 2 + 1) * 32] = w[1];
        }
      if constexpr (FMT == kInt8) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      }
      int p = -1;
      uint32_t own_bits = 0;
      if (live) {
        const int sq = seg < f.own ? seg : seq_of_row(a.cu, 0, a.num_seqs, tok);
        p = sq < 0 ? -1 : min(TREE ? tree_context(a, sq) - 1 : row_pos(a, sq, tok), s.hi - 1);
        if (TREE && seg < f.own) own_bits = tree_bits(a, tok, 0) & bit_range(max(s.lo, 0) - ctx, s.hi - 1 - ctx);
      }
      all_pos = min(all_pos, __reduce_min_sync(0xffffffffu, live ? p : 0x7fffffff));
      max_pos = max(max_pos, __reduce_max_sync(0xffffffffu, TREE && own_bits != 0 ? ctx + 31 - __clz(own_bits) : p));
      const float f_s = FMT == kInt8 ? f_q * 16777216.f : f_q, f_b = f_q * 128.f * sum;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        qs[nt][c] = __shfl_sync(0xffffffffu, f_s, (2 * t + c) * 4);
        qb[nt][c] = __shfl_sync(0xffffffffu, f_b, (2 * t + c) * 4);
        pos[nt][c] = __shfl_sync(0xffffffffu, p, (2 * t + c) * 4);
        if constexpr (TREE) bits[nt][c] = __shfl_sync(0xffffffffu, own_bits, (2 * t + c) * 4);
      }
    }

    float o[NT][KS][4], m[NT][2], m2[NT][2], l[NT][2];
    float ps[NT][4];                       // sums of the rounded probabilities (int8)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        m[nt][c] = m2[nt][c] = -INFINITY;
        l[nt][c] = 0.f;
        ps[nt][c] = ps[nt][c + 2] = 0.f;
      }
    }

    for (int u = u0; u < u1; ++u) {
      const int tok0 = base + u * UNIT;
      // some key of the unit is hidden from some row: the list's ends, and the causal border
      const bool edge = tok0 < s.lo || tok0 + UNIT - 1 > all_pos;
      float x[SUB][NT][4];
#pragma unroll
      for (int i = 0; i < SUB; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 4; ++c) x[i][nt][c] = 0.f;
      mbar_wait(&full[stage], phase, 90);
      const uint8_t* kb = ring + stage * 2 * C::HALF;
      const uint8_t* vb = kb + C::HALF;
      constexpr int STEPS = 16 / C::ESZ / 4;             // products that a lane's 16 bytes of a key take part in
#pragma unroll
      for (int c = 0; c < KW / 4; ++c) {
#pragma unroll
        for (int i = 0; i < SUB; ++i) {
          uint4 raw[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)                    // chunk t + 4 (c & 1): bit 2 of the place
            raw[h] = *reinterpret_cast<const uint4*>(kb + (i * C::BOXES + (c >> 1)) * 16 * C::ROW + ((k_off ^ ((c & 1) << 6)) + h * 8 * C::ROW));
#pragma unroll
          for (int st = 0; st < STEPS; ++st) {
            uint32_t f0[2], f1[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t* word = reinterpret_cast<const uint32_t*>(&raw[h]);
              if constexpr (FMT == kF16Pages) {
                f0[h] = word[2 * st];
                f1[h] = word[2 * st + 1];
              } else if constexpr (FMT == kInt8) {
                f0[h] = int8_pair(word[st]);
                f1[h] = int8_pair(word[st] >> 8);
              } else {
                f0[h] = e4m3_pair(word[st]);
                f1[h] = e4m3_pair_hi(word[st]);
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint2 qf = s_q[(nt * KS + c * STEPS + st) * 32];
              mma_16816<M>(x[i][nt], f0[0], f0[1], f1[0], f1[1], qf.x, qf.y);
            }
          }
        }
      }
      float kf[SUB][2], lv[SUB][2];
      if constexpr (FMT != kF16Pages) {
        const float* sc = s_scales + (warp * STAGES + stage) * (C::SCALES / 4);
#pragma unroll
        for (int i = 0; i < SUB; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            kf[i][h] = sc[i * 16 + kk + 8 * h];
            lv[i][h] = __log2f(sc[UNIT + i * 16 + kk + 8 * h]);
          }
      }

      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < SUB; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float& z = x[i][nt][c];
            if constexpr (FMT == kInt8) z = kf[i][c >> 1] * fmaf(z, qs[nt][c & 1], -qb[nt][c & 1]);
            else z *= (FMT != kF16Pages ? kf[i][c >> 1] : 1.f) * qs[nt][c & 1];
            if (edge) {
              const int key = tok0 + i * 16 + kk + 8 * (c >> 1);
              if constexpr (TREE) {
                if (key < s.lo || (key > pos[nt][c & 1] && ((unsigned)(key - ctx) > 31u || (bits[nt][c & 1] >> (key - ctx) & 1u) == 0))) z = -INFINITY;
              } else {
                if (key < s.lo || key > pos[nt][c & 1]) z = -INFINITY;
              }
            }
            grow = grow || z > m[nt][c & 1] + 8.f;
            if constexpr (FMT != kF16Pages) grow = grow || z + lv[i][c >> 1] > m2[nt][c & 1] + 8.f;
          }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float a0 = -INFINITY, a1 = -INFINITY;
#pragma unroll
            for (int i = 0; i < SUB; ++i) {
              a0 = fmaxf(a0, fmaxf(x[i][nt][c], x[i][nt][c + 2]));
              if constexpr (FMT != kF16Pages) a1 = fmaxf(a1, fmaxf(x[i][nt][c] + lv[i][0], x[i][nt][c + 2] + lv[i][1]));
            }
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) {
              a0 = fmaxf(a0, __shfl_xor_sync(0xffffffffu, a0, w));
              if constexpr (FMT != kF16Pages) a1 = fmaxf(a1, __shfl_xor_sync(0xffffffffu, a1, w));
            }
            const float mn = fmaxf(m[nt][c], a0), al = m[nt][c] == mn ? 1.f : exp2_fast(m[nt][c] - mn);
            l[nt][c] *= al;
            float al2 = al;
            if constexpr (FMT != kF16Pages) {
              const float mn2 = fmaxf(m2[nt][c], a1);
              al2 = m2[nt][c] == mn2 ? 1.f : exp2_fast(m2[nt][c] - mn2);
              m2[nt][c] = mn2;
            }
            m[nt][c] = mn;
            ps[nt][c] *= al2;
            ps[nt][c + 2] *= al2;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              o[nt][i][c] *= al2;
              o[nt][i][c + 2] *= al2;
            }
          }
      }
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
        uint32_t b0[NT], b1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float p[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float z = x[i][nt][c], mm = m[nt][c & 1] == -INFINITY ? 0.f : m[nt][c & 1] - (FMT == kF16Pages ? kUp : 0.f);
            const float e = exp2_fast(z - mm);
            l[nt][c & 1] += e;
            if constexpr (FMT == kF16Pages) p[c] = e;
            else {
              // a hidden key: 0 whatever its scale is
              const float mm2 = m2[nt][c & 1] == -INFINITY ? 0.f : m2[nt][c & 1] - kUp;
              p[c] = z == -INFINITY ? 0.f : exp2_fast(z + lv[i][c >> 1] - mm2);
            }
          }
          uint32_t w0, w1;
          if constexpr (std::is_same<M, __half>::value) {
            const __half2 h0 = __floats2half2_rn(p[0], p[1]), h1 = __floats2half2_rn(p[2], p[3]);
            w0 = *reinterpret_cast<const uint32_t*>(&h0), w1 = *reinterpret_cast<const uint32_t*>(&h1);
          } else {
            const __nv_bfloat162 h0 = __floats2bfloat162_rn(p[0], p[1]), h1 = __floats2bfloat162_rn(p[2], p[3]);
            w0 = *reinterpret_cast<const uint32_t*>(&h0), w1 = *reinterpret_cast<const uint32_t*>(&h1);
          }
          b0[nt] = transpose8(w0);
          b1[nt] = transpose8(w1);
        }
        if constexpr (FMT == kInt8) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816<M>(ps[nt], 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u, b0[nt], b1[nt]);
        }
        constexpr int CW = VW < 4 ? VW : 4;              // words of a chunk
#pragma unroll
        for (int c = 0; c < VW / CW; ++c) {
          uint32_t vr[4][CW];
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const uint8_t* p = vb + (i * C::BOXES + c) * 16 * C::ROW + v_off[h & 1] + (h >> 1) * 8 * C::ROW;
            if constexpr (CW == 4) {
              const uint4 y = *reinterpret_cast<const uint4*>(p);
              vr[h][0] = y.x, vr[h][1] = y.y, vr[h][2] = y.z, vr[h][3] = y.w;
            } else {
              const uint2 y = *reinterpret_cast<const uint2*>(p);
              vr[h][0] = y.x, vr[h][1] = y.y;
            }
            if (edge) {                                  // what lies in hidden places may be anything: 0 x NaN is NaN
              const int key = tok0 + i * 16 + ((h & 1) ? v1 : 2 * t) + 8 * (h >> 1);
              if (key < s.lo || key > max_pos) {
#pragma unroll
                for (int e = 0; e < CW; ++e) vr[h][e] = 0u;
              }
            }
          }
#pragma unroll
          for (int e = 0; e < CW; ++e) {
            const int w = c * CW + e;
            if constexpr (FMT == kF16Pages) {
              const uint32_t a0 = prmt(vr[0][e], vr[1][e], 0x5410), a1 = prmt(vr[0][e], vr[1][e], 0x7632);
              const uint32_t a2 = prmt(vr[2][e], vr[3][e], 0x5410), a3 = prmt(vr[2][e], vr[3][e], 0x7632);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_16816<M>(o[nt][w], a0, a1, a2, a3, b0[nt], b1[nt]);
            } else {
              uint32_t y[2][4];                          // [keys 2t, 2t + 1 | + 8][byte]
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t x0 = vr[2 * h][e], x1 = vr[2 * h + 1][e];
                if constexpr (FMT == kInt8) {
                  y[h][0] = int8_pair(prmt(x0, x1, 0x0400));
                  y[h][1] = int8_pair(prmt(x0, x1, 0x0501));
                  y[h][2] = int8_pair(prmt(x0, x1, 0x0602));
                  y[h][3] = int8_pair(prmt(x0, x1, 0x0703));
                } else {
                  const uint32_t y0 = prmt(x0, x1, 0x5140), y1 = prmt(x0, x1, 0x7362);
                  y[h][0] = e4m3_pair(y0);
                  y[h][1] = e4m3_pair_hi(y0);
                  y[h][2] = e4m3_pair(y1);
                  y[h][3] = e4m3_pair_hi(y1);
                }
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_16816<M>(o[nt][2 * w], y[0][0], y[0][1], y[1][0], y[1][1], b0[nt], b1[nt]);
                mma_16816<M>(o[nt][2 * w + 1], y[0][2], y[0][3], y[1][2], y[1][3], b0[nt], b1[nt]);
              }
            }
          }
        }
      }
      __syncwarp();                        // every lane has read the stage
      if (more) copy(stage);
      if (++stage == STAGES) stage = 0, phase ^= 1;
    }

    // ---- the list's result, or its part
    unsigned anew = 0;                                 // rows whose result is not finite, perhaps by a value that they do not see (0 x NaN is NaN)
    const bool whole = u0 == 0 && u1 == n;
    const bool last = whole && a.groups == 0;          // the result itself
    const int slot = 2 * (int)me + (cur > begin ? 1 : 0);
    if (u0 == 0 && lane == 0) {
      FewInfo in;
      in.first_slot = whole ? -1 : slot;
      in.first_warp = me;
      in.last_warp = (cur + n - 1) / per;
      in.pad = 0;
      pa.info[(int64_t)seg * a.hkv + kvh] = in;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[nt][c];
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        const int i = nt * 8 + 2 * t + c;
        bool again = false;
        if (FMT != kInt8 && all_pos < max_pos) {       // some row does not see keys that others see (int8: a hidden value is 0 x a number)
          float unfinite = 0.f;                        // NaN where a result is not finite
#pragma unroll
          for (int k = 0; k < KS; ++k) unfinite = fmaf(o[nt][k][c], 0.f, fmaf(o[nt][k][c + 2], 0.f, unfinite));
          const unsigned row = __reduce_or_sync(0xffffffffu, i < nrows && sum == sum && unfinite != 0.f ? 1u << i : 0u);
          again = (row >> i & 1) != 0;
          anew |= row;
        }
        if (i >= nrows || again) continue;
        // what l and O stand relative to
        const float ref = m[nt][c] - (FMT == kF16Pages ? kUp : 0.f);
        float back = 1.f, off = 0.f;
        if constexpr (FMT != kF16Pages) {
          back = m2[nt][c] == -INFINITY ? 0.f : exp2f(m2[nt][c] - kUp - (m[nt][c] == -INFINITY ? 0.f : m[nt][c]));   // no value has a scale: zero
          if constexpr (FMT == kInt8) off = -128.f * ps[nt][c] * back;
        }
        // int8: sums are of code 2^-24.  They are lifted before the factor, which may be as large as the values are
        auto value = [&](float x) { return fmaf(FMT == kInt8 ? x * 16777216.f : x, back, off); };
        const int tok = s.row0 + i / group, head = kvh * group + i % group;
        if (last) {
          // sum is NaN where a score was; a row without a visible key is zero
          const bool sees = pos[nt][c] >= s.lo || (TREE && bits[nt][c] != 0);
          const float inv = 1.0f / sum;
          back *= inv, off *= inv;
          T* dst = reinterpret_cast<T*>(a.out) + (int64_t)tok * a.ldo + (int64_t)head * D;
#pragma unroll
          for (int k = 0; k < KS / 4; ++k) {           // eight neighbouring columns
            const int e = 8 * k, col = VW >= 4 ? ((e / EPC) * 8 + r) * EPC + e % EPC : r * (D / 8) + e;
            float y[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              y[2 * j] = sees ? value(o[nt][4 * k + j][c]) : 0.f;
              y[2 * j + 1] = sees ? value(o[nt][4 * k + j][c + 2]) : 0.f;
            }
            *reinterpret_cast<uint4*>(dst + col) = pack8<T>(y);
          }
        } else {
          float* dst = whole ? (seg < f.own ? pa.whole_own : pa.whole_group) + ((int64_t)tok * a.hq + head) * (D + kPad)
                             : pa.slots + ((int64_t)slot * f.rows + i) * (D + kPad);
#pragma unroll
          for (int k = 0; k < KS / 2; ++k) {
            const int e = 4 * k, col = VW >= 4 ? ((e / EPC) * 8 + r) * EPC + e % EPC : r * (D / 8) + e;
            *reinterpret_cast<float4*>(dst + col) = make_float4(value(o[nt][2 * k][c]), value(o[nt][2 * k][c + 2]), value(o[nt][2 * k + 1][c]), value(o[nt][2 * k + 1][c + 2]));
          }
          if (r == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(ref, sum);
        }
      }
    if (FMT != kInt8 && anew != 0) rows_anew<T, FMT, D, TREE>(a, pa, f.own, seg, kvh, base + u0 * UNIT, base + u1 * UNIT - 1, whole ? -1 : slot, anew);
    cur += u1 - u0;
    if (cur < end) {
      z.cur = cur;
      open(z);
    }
  }
  pdl_wait();
}

template <typename T, int FMT, int D, int NT, bool TREE>
int launch_as(const AttnArgs& a, const PartArgs& p, int blocks, bool beside, cudaStream_t stream) {
  using C = Few<FMT, D, NT>;
  static PerDeviceSmem configured;
  auto kern = attn_pages_few_kernel<T, FMT, D, NT, TREE>;
  FewArgs f;
  f.own = p.few_own ? a.num_seqs : 0;
  f.segs = f.own + (p.few_groups ? a.groups : 0);
  f.rows = p.rows;
  f.page_magic = (uint32_t)(((1ull << 31) + a.page / 16 - 1) / (a.page / 16));
  f.beside = beside;
  const int smem = C::smem(f.segs);
  LLMSS_CHECK_CUDA(configured.ensure(kern, C::smem(kKept)));
  const int64_t rows = (int64_t)a.num_blocks * a.hkv * a.page;
  CUtensorMap map_k, map_v;
  if (int e = encode_pages(&map_k, a.k, rows, D * C::ESZ, 16)) return e;
  if (int e = encode_pages(&map_v, a.v, rows, D * C::ESZ, 16)) return e;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = beside || llmss_pdl_enabled() ? 1 : 0;
  LLMSS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, map_k, map_v, a, p, f));
  return 0;
}
template <typename T, int FMT, int D, int NT>
int launch(const AttnArgs& a, const PartArgs& p, int blocks, bool beside, cudaStream_t stream) {
  return a.masks != nullptr ? launch_as<T, FMT, D, NT, true>(a, p, blocks, beside, stream) : launch_as<T, FMT, D, NT, false>(a, p, blocks, beside, stream);
}

}  // namespace

namespace pages {

#define LLMSS_FEW_D(...)                                      \
  if (d == 64) { constexpr int D = 64; __VA_ARGS__; }         \
  else if (d == 128) { constexpr int D = 128; __VA_ARGS__; }  \
  else { constexpr int D = 256; __VA_ARGS__; }

int few_blocks(int fmt, int d, int rows, int segs) {
  int ctas = 1;
  LLMSS_FEW_D(ctas = fmt == kF16Pages ? (rows <= 8 ? Few<kF16Pages, D, 1>::ctas(segs) : Few<kF16Pages, D, 2>::ctas(segs))
                                      : (rows <= 8 ? Few<kInt8, D, 1>::ctas(segs) : Few<kInt8, D, 2>::ctas(segs)));
  return 148 * ctas;
}

int few_launch(const AttnArgs& a, const PartArgs& p, int fmt, int dtype, int blocks, bool beside, cudaStream_t stream) {
  const int d = a.d;
#define LLMSS_FEW_F(T_)                                                                                                              \
  LLMSS_FEW_D(if (p.rows <= 8) return fmt == kInt8 ? launch<T_, kInt8, D, 1>(a, p, blocks, beside, stream)                           \
                                   : fmt == kE4M3 ? launch<T_, kE4M3, D, 1>(a, p, blocks, beside, stream) : launch<T_, kF16Pages, D, 1>(a, p, blocks, beside, stream); \
              return fmt == kInt8 ? launch<T_, kInt8, D, 2>(a, p, blocks, beside, stream)                                            \
                                  : fmt == kE4M3 ? launch<T_, kE4M3, D, 2>(a, p, blocks, beside, stream) : launch<T_, kF16Pages, D, 2>(a, p, blocks, beside, stream))
  if (dtype == LLMSS_F16) {
    LLMSS_FEW_F(__half);
  }
  LLMSS_FEW_F(__nv_bfloat16);
#undef LLMSS_FEW_F
}

}  // namespace pages
