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
// The scale of a value row joins its probability in the exponent, with a maximum of its own, so that what is rounded to f16 is at most 2^8 whatever the
// scales are.  Maxima move when a score exceeds them by 2^8 only.
//
// The work of a call is the sum of all (sequence, key head) lists in units of 16 keys (32 where a key is 64 bytes); each block takes an equal run of it,
// wherever sequences begin and end, its four warps every fourth unit.  A list within a block's run is finished there; one that crosses runs leaves
// its parts in scratch, at most two per block, and the merge kernel joins them.
#include "attn_pages.cuh"

namespace {

using namespace pages;

constexpr int kWarps = 4;
constexpr int kLeastUnits = 8;     // of a block's run: two per warp
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
  static constexpr int ROWS = 8 * NT;
  static constexpr int LD = D + 4;                    // row of the merge buffer (floats)
  static constexpr int Q_BYTES = NT * KS * 32 * 8;
  static constexpr int ROW = D * ESZ < 128 ? D * ESZ : 128;   // bytes of a swizzled row: a key is BOXES of them
  static constexpr int BOXES = D * ESZ / ROW;
  static constexpr int HALF = UNIT * D * ESZ;         // keys, or values, of a unit
  static constexpr int STAGES = HALF <= 2048 ? 3 : 2;
  static constexpr int SCALES = FMT == kF16Pages ? 0 : 2 * UNIT * 4;
  // without the merge buffer, which has as many rows as the call needs
  static constexpr int FIXED = 1024 + kWarps * STAGES * (2 * HALF + SCALES) + Q_BYTES + ROWS * 12 + kWarps * (3 * ROWS * 4 + STAGES * 8);
  static constexpr int MIN_CTAS = 4 * NT * KS <= 64 ? 3 : 2;   // outputs stay in registers; what else a thread holds is about 100
  static int smem(int rows, int segs) { return FIXED + kWarps * rows * LD * 4 + 4 * (segs < kKept ? segs : kKept); }
  // blocks of an SM: by registers, and by 228 KB of shared memory less 1 KB per block
  static int ctas(int rows, int segs) {
    const int n = 233472 / (smem(rows, segs) + 1024);
    return n < MIN_CTAS ? n : MIN_CTAS;
  }
};

struct FewArgs {
  int segs;            // lists per key head: sequences (own) and groups
  int own;
  int rows;            // of the merge buffer: query rows of a list at most
  uint32_t page_magic; // (key / 16) 2 this >> 32: the key's page
  int beside;          // wait for the kernel before at the end instead of at the start
};

template <int UNIT>
__device__ __forceinline__ Seg segment(const AttnArgs& a, const FewArgs& f, int i) { return i < f.own ? own_segment(a, i) : group_segment(a, i - f.own); }
template <int UNIT>
__device__ __forceinline__ int units_of(const Seg& s) {
  return s.hi > s.lo && s.rows > 0 ? (s.hi - (s.lo & ~(UNIT - 1)) + UNIT - 1) / UNIT : 0;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(s));
  return r;
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

template <typename T, int FMT, int D, int NT>
__global__ void __launch_bounds__(32 * kWarps, Few<FMT, D, NT>::MIN_CTAS)
attn_pages_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs a,
                      const __grid_constant__ PartArgs pa, const FewArgs f) {
  using C = Few<FMT, D, NT>;
  using M = typename std::conditional<FMT == kF16Pages, T, __half>::type;   // type of the products
  constexpr int UNIT = C::UNIT, SUB = C::SUB, KW = C::KW, VW = C::VW, KS = C::KS, EPC = C::EPC, ROWS = C::ROWS, LD = C::LD, STAGES = C::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_ring = smem;                                                   // [warps][STAGES][keys | values]
  float* s_scales = reinterpret_cast<float*>(s_ring + kWarps * STAGES * 2 * C::HALF);   // [warps][STAGES][of keys | of values]
  uint64_t* s_full = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(s_scales) + kWarps * STAGES * C::SCALES);   // [warps][STAGES]
  uint2* s_q = reinterpret_cast<uint2*>(s_full + kWarps * STAGES);          // [NT][KS][32] fragments
  float* s_o = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(s_q) + C::Q_BYTES);   // [warps][rows][LD]
  float* s_m = s_o + kWarps * f.rows * LD;                                  // [warps][ROWS] each: m, m', l
  float* s_m2 = s_m + kWarps * ROWS;
  float* s_l = s_m2 + kWarps * ROWS;
  float* s_qs = s_l + kWarps * ROWS;                                        // [ROWS] score factor
  float* s_qb = s_qs + ROWS;                                                // [ROWS] what 128 added to a score
  int* s_pos = reinterpret_cast<int*>(s_qb + ROWS);                         // [ROWS] last visible key
  int* s_units = s_pos + ROWS;                                              // [min(segs, kKept)]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  if (!f.beside) pdl_wait();
  uint8_t* ring = s_ring + warp * STAGES * 2 * C::HALF;
  uint64_t* full = s_full + warp * STAGES;
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }

  // this block's run of the lists
  for (int i = threadIdx.x; i < min(f.segs, kKept); i += 32 * kWarps) s_units[i] = units_of<UNIT>(segment<UNIT>(a, f, i));
  __syncthreads();
  auto count = [&](int i) { return i < kKept ? s_units[i] : units_of<UNIT>(segment<UNIT>(a, f, i)); };
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
  const unsigned per = max((total + gridDim.x - 1) / gridDim.x, (unsigned)kLeastUnits);
  const unsigned begin = min(per * blockIdx.x, total), end = min(begin + per, total);
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

  // a place in the block's run: a list, or the part of it that lies in the run, and this warp's unit in it
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
    w.s = segment<UNIT>(a, f, w.seg);
    const unsigned at = w.cur - w.before * a.hkv;
    w.kvh = at / w.n;
    w.u0 = at - w.kvh * w.n;
    w.u1 = min((unsigned)w.n, w.u0 + (end - w.cur));
    w.base = w.s.lo & ~(UNIT - 1);
    w.u = w.u0 + warp;
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
    w.u += kWarps;
    settle();
  };
  settle();
#pragma unroll
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

  // a list's queries, read while the list before is finished: rows warp, warp + kWarps ..
  constexpr int QR = ROWS / kWarps, QC = (D + 127) / 128;
  uint2 q_raw[QR][QC];
  int q_pos[QR];
  auto read_queries = [&]() {
#pragma unroll
    for (int k = 0; k < QR; ++k) {
      const int i = warp + k * kWarps, tok = z.s.row0 + i / group;
      const bool live = i < min(z.s.rows * group, f.rows);
      const T* qr = reinterpret_cast<const T*>(a.q) + (int64_t)tok * a.ldq + (int64_t)(z.kvh * group + i % group) * D;
#pragma unroll
      for (int c = 0; c < QC; ++c) {
        q_raw[k][c] = make_uint2(0u, 0u);
        if (live && c * 128 + lane * 4 < D) q_raw[k][c] = *reinterpret_cast<const uint2*>(qr + c * 128 + lane * 4);
      }
      q_pos[k] = -1;
      if (live) {
        const int sq = z.seg < f.own ? z.seg : seq_of_row(a.cu, 0, a.num_seqs, tok);
        q_pos[k] = sq < 0 ? -1 : min(row_pos(a, sq, tok), z.s.hi - 1);
      }
    }
  };
  read_queries();

  for (unsigned cur = begin; cur < end;) {
    const Seg s = z.s;
    const int n = z.n, kvh = z.kvh, u0 = z.u0, u1 = z.u1, base = z.base;
    seg = z.seg;
    const int nrows = min(s.rows * group, f.rows);

    // ---- queries: fragments, score factors, last visible keys
    __syncthreads();                       // the list before is done with the buffers
#pragma unroll
    for (int k = 0; k < QR; ++k) {
      const int i = warp + k * kWarps;
      float up = 1.f, qs = a.scale_log2, sum = 0.f;
      if constexpr (FMT != kF16Pages) {
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < QC; ++c) {
          const T* e = reinterpret_cast<const T*>(&q_raw[k][c]);
#pragma unroll
          for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(to_f32(e[j])));
        }
        m = warp_max(m);
        const int e = m > 0.f && m < INFINITY ? max(-126, min(126, (int)((__float_as_uint(m) >> 23) & 255) - 127)) : 0;
        up = __int_as_float((127 - e) << 23);
        qs *= __int_as_float((127 + e) << 23);
      }
#pragma unroll
      for (int c = 0; c < QC; ++c) {
        const int d0 = c * 128 + lane * 4;
        if (d0 < D) {
          uint2 w = q_raw[k][c];
          if constexpr (FMT != kF16Pages) {
            const T* e = reinterpret_cast<const T*>(&q_raw[k][c]);
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = to_f32(e[j]) * up;
            // int8: a word's bytes 0, 2 and 1, 3 are converted together
            const __half2 lo = FMT == kInt8 ? __floats2half2_rn(x[0], x[2]) : __floats2half2_rn(x[0], x[1]);
            const __half2 hi = FMT == kInt8 ? __floats2half2_rn(x[1], x[3]) : __floats2half2_rn(x[2], x[3]);
            w = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            if constexpr (FMT == kInt8) {
              const float2 l2 = __half22float2(lo), h2 = __half22float2(hi);
              sum += (l2.x + l2.y) + (h2.x + h2.y);
            }
          }
          const int cc = d0 / EPC, step = ((cc >> 2) * EPC + d0 % EPC) / 4;
          s_q[((i >> 3) * KS + step) * 32 + (i & 7) * 4 + (cc & 3)] = w;
        }
      }
      if constexpr (FMT == kInt8) sum = warp_sum(sum);
      if (lane == 0) {
        s_qb[i] = qs * 128.f * sum;
        s_qs[i] = FMT == kInt8 ? qs * 16777216.f : qs;
        s_pos[i] = q_pos[k];
      }
    }
    __syncthreads();
    float qs[NT][2], qb[NT][2];
    int pos[NT][2], all_pos = 0x7fffffff, max_pos = -1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        qs[nt][c] = s_qs[nt * 8 + 2 * t + c];
        qb[nt][c] = s_qb[nt * 8 + 2 * t + c];
        pos[nt][c] = s_pos[nt * 8 + 2 * t + c];
      }
    for (int i = 0; i < nrows; ++i) {
      all_pos = min(all_pos, s_pos[i]);
      max_pos = max(max_pos, s_pos[i]);
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

    for (int u = u0 + warp; u < u1; u += kWarps) {
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
              const uint2 qf = s_q[(nt * KS + c * STEPS + st) * 32 + lane];
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
              if (key < s.lo || key > pos[nt][c & 1]) z = -INFINITY;
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

    // ---- the four warps' parts
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[nt][c];
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        const int i = nt * 8 + 2 * t + c;
        if (i < nrows) {
          if (r == 0) {
            s_m[warp * ROWS + i] = m[nt][c] - (FMT == kF16Pages ? kUp : 0.f);       // what l and O stand relative to
            s_m2[warp * ROWS + i] = (FMT != kF16Pages ? m2[nt][c] : m[nt][c]) - kUp;
            s_l[warp * ROWS + i] = sum;
          }
          float* dst = s_o + (warp * f.rows + i) * LD;
#pragma unroll
          for (int k = 0; k < KS / 2; ++k) {           // rows f[4k] .. f[4k + 3] of the lane: neighbouring columns
            const int e = 4 * k, col = VW >= 4 ? ((e / EPC) * 8 + r) * EPC + e % EPC : r * (D / 8) + e;
            float4 y = make_float4(o[nt][2 * k][c], o[nt][2 * k][c + 2], o[nt][2 * k + 1][c], o[nt][2 * k + 1][c + 2]);
            if constexpr (FMT == kInt8) {
              const float off = -128.f * ps[nt][c];
              y = make_float4(fmaf(y.x, 16777216.f, off), fmaf(y.y, 16777216.f, off), fmaf(y.z, 16777216.f, off), fmaf(y.w, 16777216.f, off));
            }
            *reinterpret_cast<float4*>(dst + col) = y;
          }
        }
      }
    const unsigned next = cur + (u1 - u0);
    if (next < end) {
      z.cur = next;
      open(z);
      read_queries();
    }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == n;
    const bool last = whole && a.groups == 0;          // the result itself
    float* part = nullptr;
    if (!last && !whole) part = pa.slots + (int64_t)(2 * blockIdx.x + (cur > begin ? 1 : 0)) * f.rows * (D + kPad);
    if (u0 == 0 && threadIdx.x == 0) {
      FewInfo in;
      in.first_slot = whole ? -1 : 2 * (int)blockIdx.x + (cur > begin ? 1 : 0);
      in.first_block = blockIdx.x;
      in.last_block = (cur + n - 1) / per;
      in.pad = 0;
      pa.info[(int64_t)seg * a.hkv + kvh] = in;
    }
    for (int e = threadIdx.x; e < nrows * (D / 4); e += 32 * kWarps) {
      const int i = e / (D / 4), c = (e % (D / 4)) * 4;
      float mx = -INFINITY, mx2 = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        mx = fmaxf(mx, s_m[w * ROWS + i]);
        mx2 = fmaxf(mx2, s_m2[w * ROWS + i]);
      }
      const float z = mx == -INFINITY ? 0.f : mx, z2 = mx2 == -INFINITY ? 0.f : mx2;
      float sum = 0.f;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        sum += exp2_fast(s_m[w * ROWS + i] - z) * s_l[w * ROWS + i];
        const float g = exp2_fast(s_m2[w * ROWS + i] - z2);
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * f.rows + i) * LD + c);
        y.x = fmaf(g, v.x, y.x), y.y = fmaf(g, v.y, y.y), y.z = fmaf(g, v.z, y.z), y.w = fmaf(g, v.w, y.w);
      }
      const float back = FMT == kF16Pages ? 1.f : mx2 == -INFINITY ? 0.f : exp2f(z2 - z);   // no value has a scale: zero
      const int tok = s.row0 + i / group, head = kvh * group + i % group;
      if (last) {
        // sum is NaN where a score was; a row without a visible key is zero
        const float inv = s_pos[i] < s.lo ? 0.f : back / sum;
        T w[4] = {from_f32<T>(y.x * inv), from_f32<T>(y.y * inv), from_f32<T>(y.z * inv), from_f32<T>(y.w * inv)};
        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + (int64_t)tok * a.ldo + (int64_t)head * D + c) = *reinterpret_cast<const uint2*>(w);
      } else {
        float* dst = whole ? (seg < f.own ? pa.whole_own : pa.whole_group) + ((int64_t)tok * a.hq + head) * (D + kPad) : part + i * (D + kPad);
        *reinterpret_cast<float4*>(dst + c) = make_float4(y.x * back, y.y * back, y.z * back, y.w * back);
        if (c == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(mx, sum);
      }
    }
    cur = next;
  }
  pdl_wait();
}

template <typename T, int FMT, int D, int NT>
int launch(const AttnArgs& a, const PartArgs& p, int blocks, bool beside, cudaStream_t stream) {
  using C = Few<FMT, D, NT>;
  static PerDeviceSmem configured;
  auto kern = attn_pages_few_kernel<T, FMT, D, NT>;
  FewArgs f;
  f.own = p.few_own ? a.num_seqs : 0;
  f.segs = f.own + (p.few_groups ? a.groups : 0);
  f.rows = p.rows;
  f.page_magic = (uint32_t)(((1ull << 31) + a.page / 16 - 1) / (a.page / 16));
  f.beside = beside;
  const int smem = C::smem(p.rows, f.segs);
  LLMSS_CHECK_CUDA(configured.ensure(kern, C::smem(C::ROWS, kKept)));
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

}  // namespace

namespace pages {

#define LLMSS_FEW_D(...)                                      \
  if (d == 64) { constexpr int D = 64; __VA_ARGS__; }         \
  else if (d == 128) { constexpr int D = 128; __VA_ARGS__; }  \
  else { constexpr int D = 256; __VA_ARGS__; }

int few_blocks(int fmt, int d, int rows, int segs) {
  int ctas = 1;
  LLMSS_FEW_D(ctas = fmt == kF16Pages ? (rows <= 8 ? Few<kF16Pages, D, 1>::ctas(rows, segs) : Few<kF16Pages, D, 2>::ctas(rows, segs))
                                      : (rows <= 8 ? Few<kInt8, D, 1>::ctas(rows, segs) : Few<kInt8, D, 2>::ctas(rows, segs)));
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
