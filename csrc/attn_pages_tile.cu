// Attention over cache pages for many query rows of a key head (portions of prompts, the sequences behind a prefix, all heads of a multi-query model) on
// the 5th-generation tensor cores.
//
// A block takes up to 256 rows (128 for 256 columns): a row is a (token, query head) of one key head, so that grouped heads fill a tile's 128 rows and every
// key is read once for all of them.  It walks its keys in tiles of 64:
//
//   loading warps   copy keys and values page by page (cp.async; 8-bit codes through a ring of their own, then converted) into a ring of 128-byte
//                   swizzled tiles, keys a tile ahead of values; what lies outside of the list is filled with zeros and never looked at
//   issuing warp    S_j = Q K_j^T (two S buffers per 128 rows), O += P_j V_j with P_j in tensor memory over S_j
//   softmax warps   a thread per row: its S row from tensor memory, mask, running maximum (moved when exceeded by 2^8) and sum in 32 bits, P back
//
// 8-bit codes are converted once per block for all its rows: code * scale is rounded to the queries' type, which is a rounding of the same size as a
// 16-bit cache has, and well below the code's own step; with the scales multiplied to the scores instead, every row would pay for them.  Copies are not
// TMA's because the conversion and the zeros pass through threads anyway.
//
// A list whose rows are few is cut into stretches of keys (grid x), whose parts the merge kernel joins.
#include "attn_pages.cuh"

namespace {

using namespace pages;
using namespace umma_lo;

constexpr int BM = 128, BN = 64;
constexpr int kLoaders = 4;

template <int FMT, int D, int NQ>
struct Tile {
  static constexpr int ESZ = FMT == kF16Pages ? 2 : 1;
  static constexpr int SOFT = 4 * NQ;                                   // softmax warps
  static constexpr int THREADS = 32 * (SOFT + 1 + kLoaders);
  static constexpr int Q_BYTES = NQ * BM * D * 2;
  static constexpr int SLOT = BN * D * 2;                               // a tile of keys or values
  static constexpr int SLOTS = D == 256 ? (FMT == kF16Pages ? 4 : 3) : 6;
  static constexpr int CH = BN * D * ESZ / 16 / (32 * kLoaders);        // 16-byte chunks of a tile per loading thread
  static constexpr int RAW = FMT == kF16Pages ? 0 : CH * 32 * kLoaders * 20;   // codes, and a scale per chunk
  static constexpr int RAWS = FMT == kF16Pages ? 0 : (D == 256 ? 3 : 4);
  static constexpr int SMEM = 1024 + Q_BYTES + SLOTS * SLOT + RAWS * RAW + 512;
  static constexpr int TMEM = NQ * (2 * BN + D) <= 256 ? 256 : 512;
};

struct TileArgs {
  int own_tiles, group_tiles;     // row tiles of the longest list
  int own_splits, group_splits;
  int own_chunk, group_chunk;     // keys, multiples of BN
  int segs_own;                   // sequences (0: not this launch's)
  int direct;                     // the result itself, not a part
};

// MN-major and K-major halves of descriptors as in umma_lo; instruction descriptor of kind::f16 with 32-bit sums
__host__ __device__ constexpr uint32_t idesc(int fmt, int n, int b_mn) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {   // bytes 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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

// four codes -> code * scale in the 16-bit type, two words
template <typename T, int FMT>
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
  lo = pack16<T>(f[0], f[1]);
  hi = pack16<T>(f[2], f[3]);
}

template <typename T, int FMT, int D, int NQ>
__global__ void __launch_bounds__(Tile<FMT, D, NQ>::THREADS, 1)
attn_pages_tile_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ PartArgs pa, const TileArgs ta) {
  using C = Tile<FMT, D, NQ>;
  constexpr int DSUB = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = smem;                                   // [NQ][DSUB][128 rows][128 bytes]
  uint8_t* s_kv = s_q + C::Q_BYTES;                      // [SLOTS][DSUB][64 keys][128 bytes]
  uint8_t* s_raw = s_kv + C::SLOTS * C::SLOT;            // [RAWS][CH][128 threads] codes, then scales
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_raw + C::RAWS * C::RAW);
  uint64_t* bar_full = bars;                             // [SLOTS]
  uint64_t* bar_empty = bars + C::SLOTS;
  uint64_t* bar_s = bars + 2 * C::SLOTS;                 // [NQ][2] S ready
  uint64_t* bar_p = bar_s + 2 * NQ;                      // [NQ][2] P written
  uint64_t* bar_o = bar_p + 2 * NQ;                      // [NQ][2] P V done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_o + 2 * NQ);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  pdl_wait();

  // the block's list, rows and keys
  const bool is_own = (int)blockIdx.z < ta.segs_own;
  const int tiles = is_own ? ta.own_tiles : ta.group_tiles, splits = is_own ? ta.own_splits : ta.group_splits;
  const int chunk = is_own ? ta.own_chunk : ta.group_chunk;
  if ((int)blockIdx.x >= tiles * splits) return;
  // long causal ranges first
  const int tile = tiles - 1 - (int)blockIdx.x / splits, split = (int)blockIdx.x % splits;
  const Seg s = is_own ? own_segment(a, blockIdx.z) : group_segment(a, blockIdx.z - ta.segs_own);
  const int kvh = blockIdx.y, group = a.hq / a.hkv;
  const int nrows = s.rows * group, n0 = tile * (NQ * BM);
  if (n0 >= nrows) return;
  const int n_last = min(nrows, n0 + NQ * BM) - 1;
  int k_end = s.hi;
  if (is_own) k_end = min(k_end, row_pos(a, blockIdx.z, s.row0 + n_last / group) + 1);
  // stretch `split` of the list; the last one takes what lies behind it (lengths beyond the bounds the call gave)
  const int k_lo = max(s.lo, s.lo + split * chunk);
  const int k_hi = split == splits - 1 ? k_end : min(k_end, s.lo + (split + 1) * chunk);
  const int base = k_lo & ~(BN - 1);
  const int n_tiles = k_hi > k_lo ? (k_hi - base + BN - 1) / BN : 0;

  // queries into their swizzled tiles; rows beyond the last are zeros
  for (int i = threadIdx.x; i < NQ * BM * (D / 8); i += C::THREADS) {
    const int row = i / (D / 8), ch = i % (D / 8), n = n0 + row;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (n < nrows && n_tiles > 0)
      v = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (int64_t)(s.row0 + n / group) * a.ldq + (int64_t)(kvh * group + n % group) * D + ch * 8);
    *reinterpret_cast<uint4*>(s_q + (row / BM) * (BM * D * 2) + (ch >> 3) * (BM * 128) + (row % BM) * 128 + (((ch & 7) ^ (row & 7)) << 4)) = v;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(&bar_full[i], kLoaders);
      mbar_init(&bar_empty[i], 1);
    }
    for (int i = 0; i < 2 * NQ; ++i) {
      mbar_init(&bar_s[i], 1);
      mbar_init(&bar_p[i], 4);
      mbar_init(&bar_o[i], 1);
    }
    fence_mbar_init();
  }
  if (warp == C::SOFT) {
    tmem_alloc(tmem_slot, C::TMEM);
    tmem_relinquish();
  }
  fence_proxy_async_smem();
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto t_s = [&](int q, int b) { return tmem + q * (2 * BN + D) + b * BN; };
  auto t_o = [&](int q) { return tmem + q * (2 * BN + D) + 2 * BN; };
  // places of tiles in the ring: K0, then K_{j+1}, V_j, and V of the last tile
  auto key_at = [&](int j) { return j == 0 ? 0 : 2 * j - 1; };
  auto value_at = [&](int j) { return j + 1 < n_tiles ? 2 * j + 2 : 2 * n_tiles - 1; };

  if (warp > C::SOFT) {
    // ===================== loading warps
    const int tid = threadIdx.x - 32 * (C::SOFT + 1);
    constexpr int PER = D * C::ESZ / 16;                 // chunks of a key
    auto tile_of = [&](int i, bool& value) {             // i-th of the ring -> tile
      if (i == 2 * n_tiles - 1) {
        value = true;
        return n_tiles - 1;
      }
      value = i >= 2 && (i & 1) == 0;
      return i == 0 ? 0 : value ? (i - 2) / 2 : (i + 1) / 2;
    };
    const int total = 2 * n_tiles;
    // cache rows of a tile's four runs of 16 keys (a run lies in one page), one per lane of each four; looked up a tile ahead of the copies
    auto look_up = [&](int j) {
      const int key = base + j * BN + (lane & 3) * 16;
      return key < k_hi ? ((uint32_t)checked_block(__ldg(s.table + key / a.page), a.num_blocks) * a.hkv + kvh) * a.page + key % a.page : 0u;
    };
    uint32_t runs = look_up(0), runs_before = 0, runs_next = 0;       // of the newest tile of keys, of the one before, of the next one
    int newest = -1;
    // turn to the i-th of the ring: its tile, and the cache row of this thread's chunk c with whether that lies in the list
    auto turn = [&](int i, bool& value, uint32_t& mine) {
      const int j = tile_of(i, value);
      if (!value) {
        if (j > 0) runs_before = runs, runs = runs_next;
        newest = j;
        runs_next = look_up(j + 1);
      }
      mine = j == newest ? runs : runs_before;
      return base + j * BN;
    };
    auto place = [&](int first, uint32_t mine, int c, uint32_t& row) {
      const int key = (c * (32 * kLoaders) + tid) / PER;
      row = __shfl_sync(0xffffffffu, mine, key >> 4) + (key & 15);
      return first + key >= s.lo && first + key < k_hi;
    };
    if constexpr (FMT == kF16Pages) {
      constexpr int LAG = C::SLOTS - 2;                  // tiles in flight
      auto finish = [&](int i) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_full[i % C::SLOTS]);
      };
      for (int i = 0; i < total + LAG; ++i) {
        if (i < total) {
          bool value;
          uint32_t mine;
          const int first = turn(i, value, mine);
          mbar_wait(&bar_empty[i % C::SLOTS], ((i / C::SLOTS) & 1) ^ 1, 80);
          const uint32_t dst = smem_u32(s_kv + (i % C::SLOTS) * C::SLOT);
          const uint8_t* src = reinterpret_cast<const uint8_t*>(value ? a.v : a.k);
#pragma unroll
          for (int c = 0; c < C::CH; ++c) {
            uint32_t row;
            const bool in = place(first, mine, c, row);
            const int x = c * (32 * kLoaders) + tid, key = x / PER, ch = x % PER;
            copy16(dst + (ch >> 3) * (BN * 128) + key * 128 + (((ch & 7) ^ (key & 7)) << 4), src + (in ? (uint64_t)row * (D * 2) + ch * 16 : 0), in ? 16 : 0);
          }
        }
        copies_commit();
        if (i >= LAG) {
          copies_wait<LAG>();
          finish(i - LAG);
        }
      }
    } else {
      auto fetch = [&](int i) {
        if (i < total) {
          bool value;
          uint32_t mine;
          const int first = turn(i, value, mine);
          uint8_t* raw = s_raw + (i % C::RAWS) * C::RAW;
          const uint8_t* src = reinterpret_cast<const uint8_t*>(value ? a.v : a.k);
          const float* sc = value ? a.vs : a.ks;
#pragma unroll
          for (int c = 0; c < C::CH; ++c) {
            uint32_t row;
            const bool in = place(first, mine, c, row);
            const int x = c * (32 * kLoaders) + tid;
            copy16(smem_u32(raw + x * 16), src + (in ? (uint64_t)row * D + (x % PER) * 16 : 0), in ? 16 : 0);
            copy4(smem_u32(raw + C::CH * 32 * kLoaders * 16 + x * 4), sc + (in ? row : 0), in ? 4 : 0);
          }
        }
        copies_commit();
      };
      for (int i = 0; i < C::RAWS - 1; ++i) fetch(i);
      for (int i = 0; i < total; ++i) {
        fetch(i + C::RAWS - 1);
        copies_wait<C::RAWS - 1>();                      // a thread converts what it copied itself
        const uint8_t* raw = s_raw + (i % C::RAWS) * C::RAW;
        mbar_wait(&bar_empty[i % C::SLOTS], ((i / C::SLOTS) & 1) ^ 1, 81);
        uint8_t* dst = s_kv + (i % C::SLOTS) * C::SLOT;
#pragma unroll
        for (int c = 0; c < C::CH; ++c) {
          const int x = c * (32 * kLoaders) + tid, key = x / PER, ch = x % PER;
          const uint4 w = *reinterpret_cast<const uint4*>(raw + x * 16);
          const float scale = *reinterpret_cast<const float*>(raw + C::CH * 32 * kLoaders * 16 + x * 4);
          uint4 y[2];
          convert4<T, FMT>(w.x, scale, y[0].x, y[0].y);
          convert4<T, FMT>(w.y, scale, y[0].z, y[0].w);
          convert4<T, FMT>(w.z, scale, y[1].x, y[1].y);
          convert4<T, FMT>(w.w, scale, y[1].z, y[1].w);
          // eight lanes write one key: lanes of odd 64-column halves begin with their second chunk, so that no two meet in a bank
          const int flip = (ch >> 2) & 1;
          uint8_t* to = dst + (ch >> 2) * (BN * 128) + key * 128;
          const int c0 = 2 * (ch & 3) + flip, c1 = c0 ^ 1;
          *reinterpret_cast<uint4*>(to + ((c0 ^ (key & 7)) << 4)) = flip ? y[1] : y[0];
          *reinterpret_cast<uint4*>(to + ((c1 ^ (key & 7)) << 4)) = flip ? y[0] : y[1];
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_full[i % C::SLOTS]);
      }
    }
  } else if (warp == C::SOFT) {
    // ===================== issuing warp: all of it runs the loop, one lane issues
    const int fmt = std::is_same<T, __half>::value ? 0 : 1;
    const uint32_t id_s = idesc(fmt, BN, 0), id_o = idesc(fmt, D, 1);
    const uint32_t q_lo = desc_lo(smem_u32(s_q)), k_lo0 = desc_lo(smem_u32(s_kv)), v_lo0 = desc_lo(smem_u32(s_kv), BN * 128);
    auto scores = [&](int q, int j) {
      const uint32_t ql = q_lo + q * (BM * D * 2 / 16), kl = k_lo0 + (key_at(j) % C::SLOTS) * (C::SLOT / 16);
      if (elect_one()) {
#pragma unroll
        for (int c = 0; c < DSUB; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_ss(t_s(q, j & 1), ql + (c * (BM * 128) + k * 32) / 16, kl + (c * (BN * 128) + k * 32) / 16, id_s, (c | k) ? 1u : 0u);
        umma_commit(&bar_s[q * 2 + (j & 1)]);
        if (q == NQ - 1) umma_commit(&bar_empty[key_at(j) % C::SLOTS]);
      }
      __syncwarp();
    };
    auto wait_full = [&](int i) { mbar_wait(&bar_full[i % C::SLOTS], (i / C::SLOTS) & 1, 82); };
    for (int j = 0; j < min(n_tiles, 2); ++j) {
      wait_full(key_at(j));
      tcgen05_fence_after();
#pragma unroll
      for (int q = 0; q < NQ; ++q) scores(q, j);
    }
    for (int j = 0; j < n_tiles; ++j) {
      const int b = j & 1;
      wait_full(value_at(j));
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        mbar_wait(&bar_p[q * 2 + b], (j >> 1) & 1, 83);
        tcgen05_fence_after();
        const uint32_t vl = v_lo0 + (value_at(j) % C::SLOTS) * (C::SLOT / 16);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < BN / 16; ++k) umma_ts(t_o(q), t_s(q, b) + k * 8, vl + k * 128, id_o, (j > 0 || k > 0) ? 1u : 0u);
          umma_commit(&bar_o[q * 2 + b]);
          if (q == NQ - 1) umma_commit(&bar_empty[value_at(j) % C::SLOTS]);
        }
        __syncwarp();
      }
      if (j + 2 < n_tiles) {
        wait_full(key_at(j + 2));
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          mbar_wait(&bar_o[q * 2 + b], (j >> 1) & 1, 84);    // P_j has been read: S_{j+2} goes over it
          tcgen05_fence_after();
          scores(q, j + 2);
        }
      }
    }
  } else {
    // ===================== softmax: a thread per row
    const int q = warp >> 2, quarter = warp & 3;
    const int n = n0 + q * BM + quarter * 32 + lane;
    const uint32_t off = (uint32_t)(quarter * 32) << 16;
    const bool live = n < nrows;
    const int tok = s.row0 + n / group;
    int pos = 0x7fffffff;                                 // rows beyond the last look at everything and are dropped
    if (live) {
      const int sq = is_own ? (int)blockIdx.z : seq_of_row(a.cu, 0, a.num_seqs, tok);
      pos = sq < 0 ? -1 : row_pos(a, sq, tok);
    }
    pos = min(pos, k_hi - 1);
    const float scale = a.scale_log2;
    // f16 ends at 2^16 and has no numbers below 2^-24: probabilities are formed times 2^7 (at most 2^15), so that those down to 2^-21 keep all bits
    constexpr float kUp = std::is_same<T, __half>::value ? 7.0f : 0.0f;
    float m_run = -INFINITY, l_run = 0.f;
    for (int j = 0; j < n_tiles; ++j) {
      const int b = j & 1, kb = base + j * BN;
      mbar_wait(&bar_s[q * 2 + b], (j >> 1) & 1, 85);
      tcgen05_fence_after();
      float sc[BN];
      {
        uint32_t r[BN / 32][32];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) tmem_ld_32x32b_x32(t_s(q, b) + off + c * 32, r[c]);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < BN / 32; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i) sc[c * 32 + i] = __uint_as_float(r[c][i]);
      }
      const int hi = pos - kb, lo = k_lo - kb;
      if (__any_sync(0xffffffffu, hi < BN - 1 || lo > 0)) {
#pragma unroll
        for (int i = 0; i < BN; ++i)
          if (i > hi || i < lo) sc[i] = -INFINITY;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < BN; i += 8) {
#pragma unroll
        for (int u = 0; u < 4; ++u) mx[u] = fmaxf(mx[u], fmaxf(sc[i + 2 * u], sc[i + 2 * u + 1]));
      }
      const float m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale;
      const bool grow = m_tile > m_run + 8.0f;
      const float m_new = grow ? m_tile : m_run;
      const float alpha = grow && j > 0 ? exp2_fast(m_run - m_new) : 1.0f;
      m_run = m_new;
      const float neg = m_new == -INFINITY ? 0.f : kUp - m_new;
      float la[4] = {0.f, 0.f, 0.f, 0.f}, lb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float e0, e1;
          ffma2(e0, e1, sc[c * 32 + i], sc[c * 32 + i + 1], scale, scale, neg, neg);
          const float p0 = exp2_fast(e0), p1 = exp2_fast(e1);
          fadd2(la[(i >> 1) & 3], lb[(i >> 1) & 3], la[(i >> 1) & 3], lb[(i >> 1) & 3], p0, p1);
          pk[i >> 1] = pack16<T>(p0, p1);
        }
        tmem_st_x16(t_s(q, b) + off + c * 16, pk);
      }
      tmem_st_done();
      const float l_tile = ((la[0] + lb[0]) + (la[1] + lb[1])) + ((la[2] + lb[2]) + (la[3] + lb[3]));
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
        mbar_wait(&bar_o[q * 2 + (b ^ 1)], ((j - 1) >> 1) & 1, 86);
        tcgen05_fence_after();
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(t_o(q) + off + c * 32, r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
          tmem_st_x32(t_o(q) + off + c * 32, r);
        }
        tmem_st_done();
      }
      l_run = l_run * alpha + l_tile;
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_p[q * 2 + b]);
    }
    if (n_tiles > 0) {
      mbar_wait(&bar_o[q * 2 + ((n_tiles - 1) & 1)], ((n_tiles - 1) >> 1) & 1, 87);
      tcgen05_fence_after();
    }
    const int head = kvh * group + n % group;
    // no visible key: zero (the sum is NaN where a score was)
    const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
    T* out = reinterpret_cast<T*>(a.out) + (int64_t)tok * a.ldo + (int64_t)head * D;
    float* part = (is_own ? pa.tile_own : pa.tile_group) + (((int64_t)split * a.total_q + tok) * a.hq + head) * (D + kPad);
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t r[32];
      if (n_tiles > 0) {
        tmem_ld_32x32b_x32(t_o(q) + off + c * 32, r);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) r[i] = 0u;
      }
      if (live) {
        if (ta.direct) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            float f8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f8[e] = __uint_as_float(r[i + e]) * inv;
            *reinterpret_cast<uint4*>(out + c * 32 + i) = pack8<T>(f8);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4) *reinterpret_cast<uint4*>(part + c * 32 + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
        }
      }
    }
    if (live && !ta.direct) *reinterpret_cast<float2*>(part + D) = make_float2(m_run - kUp, l_run);
  }

  tcgen05_fence_before();
  __syncthreads();
  if (warp == C::SOFT) {
    tcgen05_fence_after();
    tmem_dealloc(tmem, C::TMEM);
  }
}

template <typename T, int FMT, int D, int NQ>
int launch(const AttnArgs& a, const PartArgs& p, const TilePlan& t, cudaStream_t stream) {
  using C = Tile<FMT, D, NQ>;
  static_assert(C::SMEM <= 232448, "shared memory of a block");
  static PerDeviceSmem configured;
  auto kern = attn_pages_tile_kernel<T, FMT, D, NQ>;
  LLMSS_CHECK_CUDA(configured.ensure(kern, C::SMEM));
  TileArgs ta;
  ta.own_tiles = t.own_tiles;
  ta.group_tiles = t.group_tiles;
  ta.own_splits = p.own_splits;
  ta.group_splits = p.group_splits;
  ta.own_chunk = p.own_chunk;
  ta.group_chunk = p.group_chunk;
  ta.segs_own = t.own_tiles > 0 ? a.num_seqs : 0;
  ta.direct = a.groups == 0 && p.own_splits == 1;
  const int64_t x = (int64_t)t.own_tiles * p.own_splits, y = (int64_t)t.group_tiles * p.group_splits;
  const dim3 grid((unsigned)(x > y ? x : y), a.hkv, ta.segs_own + (t.group_tiles > 0 ? a.groups : 0));
  LLMSS_REQUIRE(grid.y <= 65535 && grid.z <= 65535 && (x > y ? x : y) < (1ll << 31), "attn_pages: grid too large (%d key heads, %u lists)", a.hkv, grid.z);
  LLMSS_CHECK_CUDA(launch_pdl(kern, grid, dim3(C::THREADS), (size_t)C::SMEM, stream, a, p, ta));
  return 0;
}

template <typename T, int FMT>
int by_size(const AttnArgs& a, const PartArgs& p, const TilePlan& t, cudaStream_t stream) {
  if (a.d == 256) return launch<T, FMT, 256, 1>(a, p, t, stream);
  if (a.d == 128) return t.rows == 256 ? launch<T, FMT, 128, 2>(a, p, t, stream) : launch<T, FMT, 128, 1>(a, p, t, stream);
  return t.rows == 256 ? launch<T, FMT, 64, 2>(a, p, t, stream) : launch<T, FMT, 64, 1>(a, p, t, stream);
}

}  // namespace

namespace pages {

// rows that a block takes: two tiles share its keys where there are more than one tile's rows (and tensor memory holds two)
int tile_rows(int d, int64_t rows) { return d < 256 && rows > BM ? 2 * BM : BM; }

int tile_launch(const AttnArgs& a, const PartArgs& p, const TilePlan& t, int fmt, int dtype, cudaStream_t stream) {
  if (dtype == LLMSS_F16)
    return fmt == kInt8 ? by_size<__half, kInt8>(a, p, t, stream) : fmt == kE4M3 ? by_size<__half, kE4M3>(a, p, t, stream) : by_size<__half, kF16Pages>(a, p, t, stream);
  return fmt == kInt8   ? by_size<__nv_bfloat16, kInt8>(a, p, t, stream)
         : fmt == kE4M3 ? by_size<__nv_bfloat16, kE4M3>(a, p, t, stream)
                        : by_size<__nv_bfloat16, kF16Pages>(a, p, t, stream);
}

}  // namespace pages
