// Attention over cache pages for up to 16 query rows of a key head (single tokens, some tokens of grouped heads, a few sequences behind a prefix): bound by
// reading the cache.
//
// A warp takes 16 keys at a time straight from global memory into the fragments of its products, with no shared memory between: keys are the rows (M) of
// S^T = K Q^T and the head's columns the rows of O^T = V^T P^T, so that 8 query rows cost no more than the instruction's narrow side.  The order of a
// product's inner index is free, so a lane's 16 bytes of a key are its columns of D / 16 products one after another, and its 16 bytes of a value row are
// its rows of the output.  8-bit codes become f16 (which holds both types without rounding) by a byte permutation and a subtraction, or by the conversion
// instruction; queries become f16 after division by the power of two below their row's largest value (exact, but for what is 2^-14 of that and smaller).
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
  static constexpr int SMEM = Q_BYTES + kWarps * ROWS * (LD + 3) * 4 + ROWS * 8;
  // 32-bit numbers that stay in registers: outputs, keys, values; what else a thread holds is about 70
  static constexpr int HELD = 4 * NT * KS + SUB * (2 * KW + 4 * VW);
  static constexpr int MIN_CTAS = HELD <= 96 ? 3 : 2;
};

struct FewArgs {
  int segs;            // lists per key head: sequences (own) and groups
  int own;
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
// bytes 0 and 2 of w, two's complement, as f16: 1024 + (code + 128) is the f16 0x6400 | byte, less 1152
__device__ __forceinline__ uint32_t int8_pair(uint32_t w) {
  uint32_t u, r;
  asm("lop3.b32 %0, %1, 0x00ff00ff, 0x64806480, 0x6a;" : "=r"(u) : "r"(w));   // (w & mask) ^ magic
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0x64806480u));
  return r;
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
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

template <typename T, int FMT, int D, int NT>
__global__ void __launch_bounds__(32 * kWarps, Few<FMT, D, NT>::MIN_CTAS)
attn_pages_few_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ PartArgs pa, const FewArgs f) {
  using C = Few<FMT, D, NT>;
  using M = typename std::conditional<FMT == kF16Pages, T, __half>::type;   // type of the products
  constexpr int UNIT = C::UNIT, SUB = C::SUB, KW = C::KW, VW = C::VW, KS = C::KS, EPC = C::EPC, ROWS = C::ROWS, LD = C::LD;
  extern __shared__ __align__(16) uint8_t smem[];
  uint2* s_q = reinterpret_cast<uint2*>(smem);                              // [NT][KS][32] fragments
  float* s_o = reinterpret_cast<float*>(smem + C::Q_BYTES);                 // [warps][ROWS][LD]
  float* s_m = s_o + kWarps * ROWS * LD;                                    // [warps][ROWS] each: m, m', l
  float* s_m2 = s_m + kWarps * ROWS;
  float* s_l = s_m2 + kWarps * ROWS;
  float* s_qs = s_l + kWarps * ROWS;                                        // [ROWS] score factor
  int* s_pos = reinterpret_cast<int*>(s_qs + ROWS);                         // [ROWS] last visible key
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  if (!f.beside) pdl_wait();

  // this block's run of the lists
  long long units = 0;
  for (int b = 0; b < f.segs; b += 32) {
    int n = 0;
    if (b + lane < f.segs) n = units_of<UNIT>(segment<UNIT>(a, f, b + lane));
    units += __reduce_add_sync(0xffffffffu, n);
  }
  const long long total = units * a.hkv;
  long long per = (total + gridDim.x - 1) / gridDim.x;
  if (per < kLeastUnits) per = kLeastUnits;
  const long long begin = per * blockIdx.x, end = min(begin + per, total);
  if (begin >= end) {
    pdl_wait();
    return;
  }
  int seg = 0;
  long long before = 0;                    // units of the lists of earlier segments, one key head
  for (int b = 0; b < f.segs; b += 32) {
    int n = 0;
    if (b + lane < f.segs) n = units_of<UNIT>(segment<UNIT>(a, f, b + lane));
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += x;
    }
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
  const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.k);
  const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.v);
  for (long long cur = begin; cur < end;) {
    Seg s = segment<UNIT>(a, f, seg);
    int n = units_of<UNIT>(s);
    while (cur >= (before + n) * a.hkv) {  // the next list that has keys
      before += n;
      s = segment<UNIT>(a, f, ++seg);
      n = units_of<UNIT>(s);
    }
    const long long at = cur - before * a.hkv;
    const int kvh = (int)(at / n), u0 = (int)(at - (long long)kvh * n);
    const int u1 = (int)min((long long)n, u0 + (end - cur));
    const int base = s.lo & ~(UNIT - 1);
    const int nrows = min(s.rows * group, ROWS);

    // ---- keys and values of a unit
    uint32_t kr[SUB][2][KW], vr[SUB][4][VW];
    float ks[SUB][2], vs[SUB][2];
    int next_block[SUB];
    auto look_up = [&](int u) {            // blocks of unit u
#pragma unroll
      for (int i = 0; i < SUB; ++i) next_block[i] = u < u1 ? s.table[min(base + u * UNIT + i * 16, s.hi - 1) / a.page] : 0;
    };
    int64_t row[SUB];                      // first key row of the part
    auto place = [&](int u) {
#pragma unroll
      for (int i = 0; i < SUB; ++i)
        row[i] = ((int64_t)checked_block(next_block[i], a.num_blocks) * a.hkv + kvh) * a.page + (base + u * UNIT + i * 16) % a.page;
    };
    auto load_keys = [&]() {
#pragma unroll
      for (int i = 0; i < SUB; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* p = kp + (row[i] + r + 8 * h) * (D * C::ESZ) + t * 16;
#pragma unroll
          for (int c = 0; c < KW / 4; ++c) {
            const uint4 x = load16(p + c * 64);
            kr[i][h][4 * c] = x.x, kr[i][h][4 * c + 1] = x.y, kr[i][h][4 * c + 2] = x.z, kr[i][h][4 * c + 3] = x.w;
          }
          if constexpr (FMT != kF16Pages) ks[i][h] = a.ks[row[i] + r + 8 * h];
        }
    };
    auto load_values = [&]() {
#pragma unroll
      for (int i = 0; i < SUB; ++i) {
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const uint8_t* p = vp + (row[i] + 2 * t + (h & 1) + 8 * (h >> 1)) * (D * C::ESZ);
          if constexpr (VW >= 4) {
#pragma unroll
            for (int c = 0; c < VW / 4; ++c) {
              const uint4 x = load16(p + c * 128 + r * 16);
              vr[i][h][4 * c] = x.x, vr[i][h][4 * c + 1] = x.y, vr[i][h][4 * c + 2] = x.z, vr[i][h][4 * c + 3] = x.w;
            }
          } else {
            const uint2 x = load8(p + r * 8);
            vr[i][h][0] = x.x, vr[i][h][1] = x.y;
          }
        }
        if constexpr (FMT != kF16Pages) {
          vs[i][0] = a.vs[row[i] + r];
          vs[i][1] = a.vs[row[i] + r + 8];
        }
      }
    };
    int u = u0 + warp;
    look_up(u);
    place(u);
    look_up(u + kWarps);
    if (u < u1) {
      load_keys();
      load_values();
    }

    // ---- queries: fragments, score factors, last visible keys
    __syncthreads();                       // the list before is done with the buffers
    for (int i = warp; i < ROWS; i += kWarps) {
      const int tok = s.row0 + i / group;
      const bool live = i < nrows;
      const T* qr = reinterpret_cast<const T*>(a.q) + (int64_t)tok * a.ldq + (int64_t)(kvh * group + i % group) * D;
      uint2 raw[(D + 127) / 128];
      float m = 0.f;
#pragma unroll
      for (int c = 0; c < (D + 127) / 128; ++c) {
        raw[c] = make_uint2(0u, 0u);
        const int d0 = c * 128 + lane * 4;
        if (live && d0 < D) raw[c] = *reinterpret_cast<const uint2*>(qr + d0);
        if constexpr (FMT != kF16Pages) {
          const T* e = reinterpret_cast<const T*>(&raw[c]);
#pragma unroll
          for (int j = 0; j < 4; ++j) m = fmaxf(m, fabsf(to_f32(e[j])));
        }
      }
      float up = 1.f, qs = a.scale_log2;
      if constexpr (FMT != kF16Pages) {
        m = warp_max(m);
        const int e = m > 0.f && m < INFINITY ? max(-126, min(126, (int)((__float_as_uint(m) >> 23) & 255) - 127)) : 0;
        up = __int_as_float((127 - e) << 23);
        qs *= __int_as_float((127 + e) << 23);
      }
#pragma unroll
      for (int c = 0; c < (D + 127) / 128; ++c) {
        const int d0 = c * 128 + lane * 4;
        if (d0 < D) {
          uint2 w = raw[c];
          if constexpr (FMT != kF16Pages) {
            const T* e = reinterpret_cast<const T*>(&raw[c]);
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = to_f32(e[j]) * up;
            // int8: a word's bytes 0, 2 and 1, 3 are converted together
            const __half2 lo = FMT == kInt8 ? __floats2half2_rn(x[0], x[2]) : __floats2half2_rn(x[0], x[1]);
            const __half2 hi = FMT == kInt8 ? __floats2half2_rn(x[1], x[3]) : __floats2half2_rn(x[2], x[3]);
            w = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
          }
          const int cc = d0 / EPC, step = ((cc >> 2) * EPC + d0 % EPC) / 4;
          s_q[((i >> 3) * KS + step) * 32 + (i & 7) * 4 + (cc & 3)] = w;
        }
      }
      if (lane == 0) {
        s_qs[i] = qs;
        int pos = -1;
        if (live) {
          const int sq = seg < f.own ? seg : seq_of_row(a.cu, 0, a.num_seqs, tok);
          pos = sq < 0 ? -1 : min(row_pos(a, sq, tok), s.hi - 1);
        }
        s_pos[i] = pos;
      }
    }
    __syncthreads();
    float qs[NT][2];
    int pos[NT][2], all_pos = 0x7fffffff, max_pos = -1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        qs[nt][c] = s_qs[nt * 8 + 2 * t + c];
        pos[nt][c] = s_pos[nt * 8 + 2 * t + c];
      }
    for (int i = 0; i < nrows; ++i) {
      all_pos = min(all_pos, s_pos[i]);
      max_pos = max(max_pos, s_pos[i]);
    }

    float o[NT][KS][4], m[NT][2], m2[NT][2], l[NT][2];
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
      }
    }

    for (; u < u1; u += kWarps) {
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
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        uint2 qf[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) qf[nt] = s_q[(nt * KS + st) * 32 + lane];
#pragma unroll
        for (int i = 0; i < SUB; ++i) {
          uint32_t f0[2], f1[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if constexpr (FMT == kF16Pages) {
              f0[h] = kr[i][h][2 * st];
              f1[h] = kr[i][h][2 * st + 1];
            } else if constexpr (FMT == kInt8) {
              f0[h] = int8_pair(kr[i][h][st]);
              f1[h] = int8_pair(kr[i][h][st] >> 8);
            } else {
              f0[h] = e4m3_pair(kr[i][h][st]);
              f1[h] = e4m3_pair_hi(kr[i][h][st]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816<M>(x[i][nt], f0[0], f0[1], f1[0], f1[1], qf[nt].x, qf[nt].y);
        }
      }
      float kf[SUB][2], lv[SUB][2];
#pragma unroll
      for (int i = 0; i < SUB; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          kf[i][h] = FMT != kF16Pages ? ks[i][h] : 1.f;
          lv[i][h] = FMT != kF16Pages ? __log2f(vs[i][h]) : 0.f;
        }
      // the next unit's keys go into the same registers
      const int un = u + kWarps;
      place(un);
      look_up(un + kWarps);
      if (un < u1) load_keys();

      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < SUB; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float& z = x[i][nt][c];
            z *= (FMT != kF16Pages ? kf[i][c >> 1] : 1.f) * qs[nt][c & 1];
            if (edge) {
              const int key = tok0 + i * 16 + r + 8 * (c >> 1);
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
              a1 = fmaxf(a1, fmaxf(x[i][nt][c] + lv[i][0], x[i][nt][c + 2] + lv[i][1]));
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
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              o[nt][i][c] *= al2;
              o[nt][i][c + 2] *= al2;
            }
          }
      }
      if (edge) {                          // what lies in hidden places may be anything: 0 x NaN is NaN
#pragma unroll
        for (int i = 0; i < SUB; ++i)
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            const int key = tok0 + i * 16 + 2 * t + (h & 1) + 8 * (h >> 1);
            if (key < s.lo || key > max_pos) {
#pragma unroll
              for (int w = 0; w < VW; ++w) vr[i][h][w] = 0u;
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
        if constexpr (FMT == kF16Pages) {
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            const uint32_t a0 = prmt(vr[i][0][w], vr[i][1][w], 0x5410), a1 = prmt(vr[i][0][w], vr[i][1][w], 0x7632);
            const uint32_t a2 = prmt(vr[i][2][w], vr[i][3][w], 0x5410), a3 = prmt(vr[i][2][w], vr[i][3][w], 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816<M>(o[nt][w], a0, a1, a2, a3, b0[nt], b1[nt]);
          }
        } else {
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            uint32_t e[2][4];              // [keys 2t, 2t+1 | 2t+8, 2t+9][byte]
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t x0 = vr[i][2 * h][w], x1 = vr[i][2 * h + 1][w];
              if constexpr (FMT == kInt8) {
                e[h][0] = int8_pair(prmt(x0, x1, 0x0400));
                e[h][1] = int8_pair(prmt(x0, x1, 0x0501));
                e[h][2] = int8_pair(prmt(x0, x1, 0x0602));
                e[h][3] = int8_pair(prmt(x0, x1, 0x0703));
              } else {
                const uint32_t y0 = prmt(x0, x1, 0x5140), y1 = prmt(x0, x1, 0x7362);
                e[h][0] = e4m3_pair(y0);
                e[h][1] = e4m3_pair_hi(y0);
                e[h][2] = e4m3_pair(y1);
                e[h][3] = e4m3_pair_hi(y1);
              }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_16816<M>(o[nt][2 * w], e[0][0], e[0][1], e[1][0], e[1][1], b0[nt], b1[nt]);
              mma_16816<M>(o[nt][2 * w + 1], e[0][2], e[0][3], e[1][2], e[1][3], b0[nt], b1[nt]);
            }
          }
        }
      }
      if (un < u1) load_values();
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
          float* dst = s_o + (warp * ROWS + i) * LD;
#pragma unroll
          for (int k = 0; k < KS / 2; ++k) {           // rows f[4k] .. f[4k + 3] of the lane: neighbouring columns
            const int e = 4 * k, col = VW >= 4 ? ((e / EPC) * 8 + r) * EPC + e % EPC : r * (D / 8) + e;
            *reinterpret_cast<float4*>(dst + col) = make_float4(o[nt][2 * k][c], o[nt][2 * k][c + 2], o[nt][2 * k + 1][c], o[nt][2 * k + 1][c + 2]);
          }
        }
      }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == n;
    const bool last = whole && a.groups == 0;          // the result itself
    float* part = nullptr;
    if (!last && !whole) part = pa.slots + (int64_t)(2 * blockIdx.x + (cur > begin ? 1 : 0)) * ROWS * (D + kPad);
    if (u0 == 0 && threadIdx.x == 0) {
      FewInfo in;
      in.first_slot = whole ? -1 : 2 * (int)blockIdx.x + (cur > begin ? 1 : 0);
      in.first_block = blockIdx.x;
      in.last_block = (int)((cur + n - 1) / per);
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
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * ROWS + i) * LD + c);
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
    cur += u1 - u0;
  }
  pdl_wait();
}

template <typename T, int FMT, int D, int NT>
int launch(const AttnArgs& a, const PartArgs& p, int blocks, bool beside, cudaStream_t stream) {
  using C = Few<FMT, D, NT>;
  static PerDeviceSmem configured;
  auto kern = attn_pages_few_kernel<T, FMT, D, NT>;
  LLMSS_CHECK_CUDA(configured.ensure(kern, C::SMEM));
  FewArgs f;
  f.own = p.few_own ? a.num_seqs : 0;
  f.segs = f.own + (p.few_groups ? a.groups : 0);
  f.beside = beside;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = beside || llmss_pdl_enabled() ? 1 : 0;
  LLMSS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, a, p, f));
  return 0;
}

}  // namespace

namespace pages {

#define LLMSS_FEW_D(...)                                      \
  if (d == 64) { constexpr int D = 64; __VA_ARGS__; }         \
  else if (d == 128) { constexpr int D = 128; __VA_ARGS__; }  \
  else { constexpr int D = 256; __VA_ARGS__; }

int few_blocks(int fmt, int d, int rows) {
  int ctas = 1;
  LLMSS_FEW_D(ctas = fmt == kF16Pages ? (rows <= 8 ? Few<kF16Pages, D, 1>::MIN_CTAS : Few<kF16Pages, D, 2>::MIN_CTAS)
                                      : (rows <= 8 ? Few<kInt8, D, 1>::MIN_CTAS : Few<kInt8, D, 2>::MIN_CTAS));
  return 148 * ctas;
}

int few_launch(const AttnArgs& a, const PartArgs& p, int fmt, int dtype, int blocks, bool beside, cudaStream_t stream) {
  const int d = a.d;
#define LLMSS_FEW_F(T_)                                                                                                              \
  LLMSS_FEW_D(if (p.rows == 8) return fmt == kInt8 ? launch<T_, kInt8, D, 1>(a, p, blocks, beside, stream)                                   \
                                   : fmt == kE4M3 ? launch<T_, kE4M3, D, 1>(a, p, blocks, beside, stream) : launch<T_, kF16Pages, D, 1>(a, p, blocks, beside, stream); \
              return fmt == kInt8 ? launch<T_, kInt8, D, 2>(a, p, blocks, beside, stream)                                                    \
                                  : fmt == kE4M3 ? launch<T_, kE4M3, D, 2>(a, p, blocks, beside, stream) : launch<T_, kF16Pages, D, 2>(a, p, blocks, beside, stream))
  if (dtype == LLMSS_F16) {
    LLMSS_FEW_F(__half);
  }
  LLMSS_FEW_F(__nv_bfloat16);
#undef LLMSS_FEW_F
}

}  // namespace pages
