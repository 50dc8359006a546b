// Attention over cache pages for many query rows of a key head (portions of prompts, the sequences behind a prefix, all heads of a multi-query model) on
// the 5th-generation tensor cores.
//
// A block takes up to 256 rows (128 for 256 columns): a row is a (token, query head) of one key head, so that grouped heads fill a tile's 128 rows and every
// key is read once for all of them.  It walks its keys in tiles of 64:
//
//   copying warps   one keys, one values, page by page (TMA), into a ring of 128-byte swizzled tiles, keys a tile ahead of values; 8-bit codes into a
//                   ring of their own (bulk copies), from which
//   converting warps (8-bit) write the tiles.  Values that lie outside of the list become zeros, keys there are never looked at
//   issuing warps   one per 128 rows: S_j = Q K_j^T (two S buffers), O += P_j V_j with P_j in tensor memory over S_j.  (A product takes about 60 clocks to
//                   issue beside the other warps, so that one warp for 256 rows took 2100 clocks a tile where the products take 1100)
//   softmax warps   a thread per row: its S row from tensor memory, mask, running maximum (moved when exceeded by 2^8) and sum in 32 bits, P back
//
// 8-bit codes are converted once per block for all its rows, to f16 whatever the queries' type (code * scale rounded to bf16 is off by as much as the whole
// rest of the arithmetic: 4e-3 of a result instead of 1.8e-3; scales multiplied to scores and probabilities instead cost 100 instructions per row and tile,
// a fifth of the speed).  A power of two per tile keeps them in range (TileScales): that of the keys joins the scores' factor, that of the values the
// exponent of the probabilities, which stand relative to the largest one so far.  bf16 queries become f16 after division by the power of two below their
// row's largest value.  Prompts of many row tiles have their codes converted once for all blocks (attn_pages.cu) and come here as 16-bit pages.
//
// A list whose rows are few is cut into stretches of keys (grid x), whose parts the merge kernel joins.
#include "attn_pages.cuh"

namespace {

using namespace pages;
using namespace umma_lo;

constexpr int BM = 128, BN = 64;

template <int FMT, int D, int NQ>
struct Tile {
  static constexpr int SOFT = 4 * NQ;                                   // softmax warps
  // 8-bit: four warps convert a tile in the time that the products of two times 128 rows take, which is twice that of 128
  static constexpr bool BYTES = FMT == kInt8 || FMT == kE4M3, SCALED = FMT != kF16Pages;
  static constexpr int CONVERT = !BYTES ? 0 : NQ == 2 ? 4 : 8;
  static constexpr int COPY = SOFT + NQ;                                // first copying warp
  static constexpr int THREADS = 32 * (COPY + 2 + CONVERT);
  // 16-bit pages: registers, and shared memory for five tiles where two times 128 rows share them, that leave room for a block of the kernels which run
  // beside this one (with 125 and six, 16 questions behind a prefix took 2 % longer).  Nothing runs beside codes converted before: 128 registers keep
  // them from spilling (4 portions of 1000 tokens over 1800 202 -> 196 us)
  static constexpr int REGS = SCALED ? 128 : 112;
  static constexpr int Q_BYTES = NQ * BM * D * 2;
  static constexpr int SLOT = BN * D * 2;                               // a tile of keys or values
  static constexpr int SLOTS = D == 256 ? (BYTES ? 3 : 4) : NQ == 2 && !BYTES ? 5 : 6;
  static constexpr int RAW = BYTES ? BN * D : 0;                        // a tile of codes
  static constexpr int RAWS = BYTES ? (D == 256 ? 3 : 4) : 0;
  // scales of the last eight tiles, keys' and values', and what goes with a tile: keys of tile j + 8 come after the softmax of tile j, whatever the rings'
  // depths here
  static constexpr int SCALES = (BYTES ? 8 * 2 * BN * 4 : 0) + (SCALED ? 8 * 16 : 0);
  static constexpr int SMEM = 1024 + Q_BYTES + SLOTS * SLOT + RAWS * RAW + SCALES + 512;
  static_assert(SOFT * 32 * (D * 4 + 16) <= Q_BYTES + SLOTS * SLOT, "outputs are staged where queries, keys and values were");
  static constexpr int TMEM = NQ * (2 * BN + D) <= 256 ? 256 : 512;
};

struct TileArgs {
  int own_tiles, group_tiles;     // row tiles of the longest list
  int own_splits, group_splits;
  int own_chunk, group_chunk;     // keys, multiples of BN
  int segs_own;                   // sequences (0: not this launch's)
  int run;                        // keys of a tile that lie in one page: 16, 32 or 64
  uint32_t page_magic;            // (key / 16) 2 this >> 32: the key's page
  int direct;                     // the result itself, not a part
};

// MN-major and K-major halves of descriptors as in umma_lo; instruction descriptor of kind::f16 with 32-bit sums
__host__ __device__ constexpr uint32_t idesc(int fmt, int n, int b_mn) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {   // bytes 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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

// 2^x without the MUFU pipe; 0 for what is below -127 (hidden keys weigh nothing, however large their values), and for NaN
__device__ __forceinline__ float exp2_fma(float x) { return exp2_cubic(fmaxf(x, -127.0f)); }

// what a block computes
struct Block {
  Seg s;
  bool is_own;
  int seg, kvh, split;      // list, key head, stretch of its keys
  int n0, nrows;            // first row, rows of the list
  int k_lo, k_hi;           // keys
};
// groups' lists first, since they are long, and of a list's rows the last first, since they see most
template <int NQ>
__device__ __forceinline__ Block block_of(const AttnArgs& a, const TileArgs& ta) {
  Block b;
  const int in_groups = ta.group_tiles * ta.group_splits * a.hkv * a.groups;      // (group_tiles 0: groups are not this launch's)
  b.is_own = (int)blockIdx.x >= in_groups;
  const int at = b.is_own ? blockIdx.x - in_groups : blockIdx.x;
  const int tiles = b.is_own ? ta.own_tiles : ta.group_tiles, splits = b.is_own ? ta.own_splits : ta.group_splits;
  const int chunk = b.is_own ? ta.own_chunk : ta.group_chunk;
  const int part = at % (tiles * splits), list = at / (tiles * splits);
  b.kvh = list % a.hkv, b.seg = list / a.hkv;
  const int tile = tiles - 1 - part / splits;
  b.split = part % splits;
  b.s = b.is_own ? own_segment(a, b.seg) : group_segment(a, b.seg);
  const int group = a.hq / a.hkv;
  b.nrows = b.s.rows * group, b.n0 = tile * (NQ * BM);
  int k_end = b.s.hi;
  if (b.is_own && b.n0 < b.nrows) k_end = min(k_end, row_pos(a, b.seg, b.s.row0 + (min(b.nrows, b.n0 + NQ * BM) - 1) / group) + 1);
  // stretch `split` of the list; the last one takes what lies behind it (lengths beyond the bounds the call gave)
  b.k_lo = max(b.s.lo, b.s.lo + b.split * chunk);
  b.k_hi = b.split == splits - 1 ? k_end : min(k_end, b.s.lo + (b.split + 1) * chunk);
  return b;
}

// keys of row n of a block's list
template <int NQ>
__device__ __forceinline__ RowKeys keys_of(const AttnArgs& a, const Block& b, int n, int& tok, int& head) {
  const int group = a.hq / a.hkv;
  tok = b.s.row0 + n / group, head = b.kvh * group + n % group;
  const int sq = b.is_own ? b.seg : seq_of_row(a.cu, 0, a.num_seqs, tok);
  return {b.s.table, b.kvh, max(b.k_lo & ~(BN - 1), b.s.lo), b.k_lo, sq < 0 ? -1 : min(row_pos(a, sq, tok), b.k_hi - 1), b.k_hi - 1};
}
// By a softmax warp: of its rows (sums in tensor memory, a lane each) those whose result is not finite because of a hidden key.
template <typename T, int FMT, int D, int NQ>
__device__ __noinline__ unsigned spoiled_rows(const AttnArgs& a, const TileArgs& ta, uint32_t sums, bool mine) {
  using M = typename std::conditional<Tile<FMT, D, NQ>::SCALED, __half, T>::type;
  float x[4] = {0.f, 0.f, 0.f, 0.f};                     // NaN where a sum is not finite
#pragma unroll 1
  for (int c = 0; c < D; c += 32) {
    uint32_t r[32];
    tmem_ld_32x32b_x32(sums + c, r);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      ffma2(x[0], x[1], __uint_as_float(r[i]), __uint_as_float(r[i + 1]), 0.f, 0.f, x[0], x[1]);
      ffma2(x[2], x[3], __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]), 0.f, 0.f, x[2], x[3]);
    }
  }
  unsigned spoiled = 0, rows = __ballot_sync(0xffffffffu, mine && (x[0] + x[1]) + (x[2] + x[3]) != 0.f);
  if (rows == 0) return 0;
  const Block b = block_of<NQ>(a, ta);
  for (; rows != 0; rows &= rows - 1) {
    int tok, head;
    if (hidden_unfinite<M, FMT>(a, keys_of<NQ>(a, b, b.n0 + (threadIdx.x & ~31) + __ffs(rows) - 1, tok, head))) spoiled |= rows & (0u - rows);
  }
  return spoiled;
}
template <typename T, int FMT, int D, int NQ>
__device__ __noinline__ void rows_anew(const AttnArgs& a, const PartArgs& pa, const TileArgs& ta, unsigned rows) {
  using M = typename std::conditional<Tile<FMT, D, NQ>::SCALED, __half, T>::type;
  const Block b = block_of<NQ>(a, ta);
  __syncwarp();                                          // behind the rows as they were
  for (; rows != 0; rows &= rows - 1) {
    int tok, head;
    const RowKeys k = keys_of<NQ>(a, b, b.n0 + (threadIdx.x & ~31) + __ffs(rows) - 1, tok, head);
    float* part = (b.is_own ? pa.tile_own : pa.tile_group) + (((int64_t)b.split * a.total_q + tok) * a.hq + head) * (D + kPad);
    row_anew<T, M, FMT>(a, k, tok, head, ta.direct ? nullptr : part);
  }
}

template <typename T, int FMT, int D, int NQ>
__global__ void __maxnreg__((Tile<FMT, D, NQ>::REGS))
attn_pages_tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnArgs a, const __grid_constant__ PartArgs pa, const __grid_constant__ TileArgs ta) {
  using C = Tile<FMT, D, NQ>;
  using M = typename std::conditional<C::SCALED, __half, T>::type;   // type of the products
  constexpr int DSUB = D / 64;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* s_q = smem;                                   // [NQ][DSUB][128 rows][128 bytes]
  uint8_t* s_kv = s_q + C::Q_BYTES;                      // [SLOTS][DSUB][64 keys][128 bytes]
  uint8_t* s_raw = s_kv + C::SLOTS * C::SLOT;            // [RAWS][64 keys of codes]
  float* s_scale = reinterpret_cast<float*>(s_raw + C::RAWS * C::RAW);   // [8 tiles][keys', values'][64] (8-bit)
  TileScales* s_tile = reinterpret_cast<TileScales*>(s_raw + C::RAWS * C::RAW + C::SCALES) - 8;   // [8 tiles]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_raw + C::RAWS * C::RAW + C::SCALES);
  uint64_t* bar_full = bars;                             // [SLOTS]
  uint64_t* bar_empty = bars + C::SLOTS;
  uint64_t* bar_s = bars + 2 * C::SLOTS;                 // [NQ][2] S ready
  uint64_t* bar_p = bar_s + 2 * NQ;                      // [NQ][2] P written
  uint64_t* bar_o = bar_p + 2 * NQ;                      // [NQ][2] P V done
  uint64_t* bar_q = bar_o + 2 * NQ;                      // [NQ] queries are in place
  uint64_t* bar_part = bar_q + NQ;                       // a tile at the list's end, before its zeros
  uint64_t* bar_raw = bar_part + 1;                      // [RAWS] codes have come
  uint64_t* bar_used = bar_raw + C::RAWS;                // [RAWS] codes have been converted
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_used + C::RAWS);

  // by a shuffle: numbers that the compiler knows to be the same in all lanes need no copies into uniform registers at every product
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (!C::BYTES && threadIdx.x == 32 * C::COPY) {
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  pdl_wait();
  // behind the wait: the kernel for few rows starts beside this one without a wait of its own, and reads what the kernels before this one wrote
  pdl_launch_dependents();

  const Block blk = block_of<NQ>(a, ta);
  const Seg s = blk.s;
  const bool is_own = blk.is_own;
  const int seg = blk.seg, kvh = blk.kvh, split = blk.split, n0 = blk.n0, nrows = blk.nrows, k_lo = blk.k_lo, k_hi = blk.k_hi;
  const int group = a.hq / a.hkv;
  if (n0 >= nrows) return;
  const int base = k_lo & ~(BN - 1);
  const int n_tiles = __shfl_sync(0xffffffffu, k_hi > k_lo ? (k_hi - base + BN - 1) / BN : 0, 0);

  // the copying warps: cache rows of the runs of eight tiles from j on, one per lane (four lanes a tile)
  auto look_up = [&](int j) {
    const int key = base + (j + (lane >> 2)) * BN + min(lane & 3, BN / ta.run - 1) * ta.run;
    if (key >= k_hi) return 0u;
    const int pg = (int)__umulhi((unsigned)key >> 4 << 1, ta.page_magic);
    return ((uint32_t)checked_block(__ldg(s.table + pg), a.num_blocks) * a.hkv + kvh) * a.page + (key - pg * a.page);
  };
  uint32_t run_rows = 0;
  if (warp == C::COPY || warp == C::COPY + 1) run_rows = look_up(0);
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::SLOTS; ++i) {
      mbar_init(&bar_full[i], C::BYTES ? C::CONVERT : 1);
      mbar_init(&bar_empty[i], NQ);
    }
    for (int i = 0; i < 2 * NQ; ++i) {
      mbar_init(&bar_s[i], 1);
      mbar_init(&bar_p[i], 4);
      mbar_init(&bar_o[i], 1);
    }
    for (int i = 0; i < NQ; ++i) mbar_init(&bar_q[i], 4);
    mbar_init(bar_part, 1);
    for (int i = 0; i < C::RAWS; ++i) {
      mbar_init(&bar_raw[i], 1);
      mbar_init(&bar_used[i], C::CONVERT);
    }
    fence_mbar_init();
  }
  if (warp == C::SOFT) {
    tmem_alloc(tmem_slot, C::TMEM);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  auto t_s = [&](int q, int b) { return tmem + q * (2 * BN + D) + b * BN; };
  auto t_o = [&](int q) { return tmem + q * (2 * BN + D) + 2 * BN; };
  // places of tiles in the ring: K0, then K_{j+1}, V_j, and V of the last tile
  auto key_at = [&](int j) { return j == 0 ? 0 : 2 * j - 1; };
  auto value_at = [&](int j) { return j + 1 < n_tiles ? 2 * j + 2 : 2 * n_tiles - 1; };

  if (warp == C::COPY || warp == C::COPY + 1) {
    // ===================== copying warps: all of one runs its loop, one lane issues
    const uint64_t policy = l2_policy_evict_last();
    const int run = ta.run, runs = BN / run;
    uint32_t part_phase = 0;
    // tile j of keys or values from the cache rows of its runs, in lanes from ..
    auto copy = [&](int j, bool value, uint32_t rows, int from, int place) {
      const int first = base + j * BN;
      const int here = min(runs, (k_hi - first + run - 1) / run);       // runs that lie in the list
      // scales of both sides come with the keys: the softmax looks at them before the values are there
      auto scales = [&](uint64_t* bar, uint32_t row, int x) {
        float* to = s_scale + (j & 7) * (2 * BN) + x * run;
        bulk_copy(to, a.ks + row, run * 4, bar);
        bulk_copy(to + BN, a.vs + row, run * 4, bar);
      };
      if constexpr (!C::BYTES) {
        const int slot = place % C::SLOTS;
        mbar_wait(&bar_empty[slot], ((place / C::SLOTS) & 1) ^ 1, 80);     // a slot's first use waits for nobody
        const bool part = value && (first < s.lo || first + BN > k_hi);
        uint64_t* bar = part ? bar_part : &bar_full[slot];
        uint8_t* dst = s_kv + slot * C::SLOT;
        if (elect_one()) {
          mbar_arrive_expect_tx(bar, here * run * D * 2 + (C::SCALED && !value ? 16 : 0));
          if (C::SCALED && !value) bulk_copy(&s_tile[j & 7], a.tile_scales + ((int64_t)seg * a.hkv + kvh) * (a.page / BN) + first / BN, 16, bar);
        }
        for (int x = 0; x < here; ++x) {
          const int row = (int)__shfl_sync(0xffffffffu, rows, from + x);
          if (elect_one()) {
#pragma unroll
            for (int c = 0; c < DSUB; ++c) tma_load_2d(dst + c * (BN * 128) + x * run * 128, value ? &map_v : &map_k, bar, c * 128, row, policy);
          }
        }
        __syncwarp();
        if (part) {
          // zeros where the list does not reach: 0 x NaN would be NaN
          mbar_wait(bar_part, part_phase, 78);
          part_phase ^= 1;
          for (int x = lane; x < BN * DSUB * 8; x += 32) {
            const int key = first + (x >> 3) % BN;
            if (key < s.lo || key >= k_hi) *reinterpret_cast<uint4*>(dst + x * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bar_full[slot]);
        }
      } else {
        const int slot = place % C::RAWS;
        mbar_wait(&bar_used[slot], ((place / C::RAWS) & 1) ^ 1, 80);
        uint8_t* dst = s_raw + slot * C::RAW;
        const uint8_t* src = reinterpret_cast<const uint8_t*>(value ? a.v : a.k);
        if (elect_one()) mbar_arrive_expect_tx(&bar_raw[slot], here * run * (D + (value ? 0 : 8)));
        for (int x = 0; x < here; ++x) {
          const uint32_t row = __shfl_sync(0xffffffffu, rows, from + x);
          if (elect_one()) {
            bulk_copy(dst + x * run * D, src + (uint64_t)row * D, run * D, &bar_raw[slot]);
            if (!value) scales(&bar_raw[slot], row, x);
          }
        }
        __syncwarp();
      }
    };
    const bool value = warp == C::COPY + 1;
    for (int j = 0; j < n_tiles; ++j) {
      if (j > 0 && (j & 7) == 0) run_rows = look_up(j);
      copy(j, value, run_rows, (j & 7) * 4, value ? value_at(j) : key_at(j));
    }
  } else if (warp > C::COPY + 1) {
    // ===================== converting warps
    if constexpr (C::BYTES) {
      const int tid = threadIdx.x - 32 * (C::COPY + 2);
      constexpr int PER = D / 16, KEYS = 32 * C::CONVERT / PER;      // 16-byte chunks of a key, keys between a thread's chunks
      constexpr int CH = BN / KEYS;                                // a thread's chunks of a tile
      const int key0 = tid / PER, ch = tid % PER;                  // this thread's first key, its place in every key
      // eight lanes write one key: lanes of odd 64-column halves begin with their second chunk, so that no two meet in a bank
      const int flip = (ch >> 2) & 1;
      const uint32_t to = (ch >> 2) * (BN * 128) + key0 * 128, c0 = ((2 * (ch & 3) + flip) ^ (key0 & 7)) << 4;
      static_assert(KEYS % 8 == 0, "every eighth key has the same place in the swizzle");
      int slot = 0, raw_slot = 0;
      uint32_t phase = 1, raw_phase = 0;
      auto convert = [&](int j, bool value) {
        const int first = base + j * BN;
        const bool all = first >= s.lo && first + BN <= k_hi;
        const uint8_t* raw = s_raw + raw_slot * C::RAW;
        mbar_wait(&bar_raw[raw_slot], raw_phase, 77);
        uint4 w[CH];
        float scale[CH];
        float* sc = s_scale + (j & 7) * (2 * BN);
        // every warp finds the tile's exponents for itself
        auto inside = [&](int key) { return all || (first + key >= s.lo && first + key < k_hi); };
        auto exponent = [&](const float* x) { return tile_exponent(inside(lane) ? x[lane] : 0.f, inside(lane + 32) ? x[lane + 32] : 0.f); };
        const int ev = exponent(sc + BN);
        int e = ev;
        if (!value) {
          e = exponent(sc);
          if (tid == 0) s_tile[j & 7] = tile_scales(e, ev);
        }
        const float down = two_to(-e);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int key = key0 + c * KEYS;
          w[c] = *reinterpret_cast<const uint4*>(raw + key * D + ch * 16);
          scale[c] = sc[(value ? BN : 0) + key] * down;
          if (!inside(key)) w[c] = make_uint4(0u, 0u, 0u, 0u), scale[c] = 0.f;   // zeros where the list does not reach
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_used[raw_slot]);
        if (++raw_slot == C::RAWS) raw_slot = 0, raw_phase ^= 1;
        mbar_wait(&bar_empty[slot], phase, 81);
        uint8_t* dst = s_kv + slot * C::SLOT + to;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          uint4 y[2];
          convert4<FMT>(w[c].x, scale[c], y[0].x, y[0].y);
          convert4<FMT>(w[c].y, scale[c], y[0].z, y[0].w);
          convert4<FMT>(w[c].z, scale[c], y[1].x, y[1].y);
          convert4<FMT>(w[c].w, scale[c], y[1].z, y[1].w);
          uint8_t* at = dst + c * (KEYS * 128);
          *reinterpret_cast<uint4*>(at + c0) = flip ? y[1] : y[0];
          *reinterpret_cast<uint4*>(at + (c0 ^ 16)) = flip ? y[0] : y[1];
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bar_full[slot]);
        if (++slot == C::SLOTS) slot = 0, phase ^= 1;
      };
      for (int j = 0; j <= n_tiles; ++j) {
        if (j < n_tiles) convert(j, false);
        if (j > 0) convert(j - 1, true);
      }
    }
  } else if (warp >= C::SOFT) {
    // ===================== issuing warps: all of one runs its loop, one lane issues
    const int q = warp - C::SOFT;
    const int fmt = std::is_same<M, __half>::value ? 0 : 1;
    const uint32_t id_s = idesc(fmt, BN, 0), id_o = idesc(fmt, D, 1);
    const uint32_t ql = desc_lo(smem_u32(s_q)) + q * (BM * D * 2 / 16), k_lo = desc_lo(smem_u32(s_kv)), v_lo = desc_lo(smem_u32(s_kv), BN * 128);
    const uint32_t ts = t_s(q, 0), to = t_o(q);
    // places in the ring: keys 0, 1, 3, 5 .., values 2, 4 .. and one behind the last keys
    int k_slot = 0, v_slot = n_tiles > 1 ? 2 : 1;
    uint32_t k_phase = 0, v_phase = 0;
    auto scores = [&](int j) {
      mbar_wait(&bar_full[k_slot], k_phase, 82);
      tcgen05_fence_after();
      const uint32_t kl = k_lo + k_slot * (C::SLOT / 16), d = ts + (j & 1) * BN;
      if (elect_one()) {
#pragma unroll
        for (int c = 0; c < DSUB; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k) umma_ss(d, ql + (c * (BM * 128) + k * 32) / 16, kl + (c * (BN * 128) + k * 32) / 16, id_s, (c | k) ? 1u : 0u);
        umma_commit(&bar_s[q * 2 + (j & 1)]);
        umma_commit(&bar_empty[k_slot]);
      }
      __syncwarp();
      k_slot += j == 0 ? 1 : 2;
      if (k_slot >= C::SLOTS) k_slot -= C::SLOTS, k_phase ^= 1;
    };
    if (n_tiles > 0) mbar_wait(&bar_q[q], 0, 79);
    for (int j = 0; j < min(n_tiles, 2); ++j) scores(j);
    for (int j = 0; j < n_tiles; ++j) {
      const int b = j & 1;
      mbar_wait(&bar_full[v_slot], v_phase, 82);
      mbar_wait(&bar_p[q * 2 + b], (j >> 1) & 1, 83);
      tcgen05_fence_after();
      const uint32_t vl = v_lo + v_slot * (C::SLOT / 16), p = ts + b * BN;
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < BN / 16; ++k) umma_ts(to, p + k * 8, vl + k * 128, id_o, (j > 0 || k > 0) ? 1u : 0u);
        umma_commit(&bar_o[q * 2 + b]);
        umma_commit(&bar_empty[v_slot]);
      }
      __syncwarp();
      v_slot += j + 2 < n_tiles ? 2 : 1;
      if (v_slot >= C::SLOTS) v_slot -= C::SLOTS, v_phase ^= 1;
      if (j + 2 < n_tiles) {
        mbar_wait(&bar_o[q * 2 + b], (j >> 1) & 1, 84);        // P_j has been read: S_{j+2} goes over it
        scores(j + 2);
      }
    }
  } else {
    // ===================== softmax: a thread per row
    const int q = warp >> 2, quarter = warp & 3;
    const int n = n0 + q * BM + quarter * 32 + lane;
    const uint32_t off = (uint32_t)(quarter * 32) << 16;
    const bool live = n < nrows;
    const int tok = s.row0 + n / group;
    const int head = kvh * group + n % group;
    // this warp's 32 rows of queries into their swizzled tile; rows beyond the last are zeros
    float scale = a.scale_log2;
    if (n_tiles > 0) {
      uint8_t* dst = s_q + q * (BM * D * 2);
      const int64_t at = live ? (int64_t)tok * a.ldq + (int64_t)head * D : -1;
      constexpr int LANES = D / 8 < 32 ? D / 8 : 32, STEP = 32 / LANES;    // lanes of a row, rows of one copy of the warp
      const int ch = lane % LANES;
      auto place = [&](int row, int ch) {
        const int rt = quarter * 32 + row;
        return dst + (ch >> 3) * (BM * 128) + rt * 128 + (((ch & 7) ^ (rt & 7)) << 4);
      };
      // loops, not lines: what runs once comes from memory, eight instructions at a time
#pragma unroll 2
      for (int i = 0; i < 32; i += STEP) {
        const int row = i + lane / LANES;
        const int64_t from = __shfl_sync(0xffffffffu, at, row);
        copy16(smem_u32(place(row, ch)), reinterpret_cast<const T*>(a.q) + (from < 0 ? 0 : from + ch * 8), from < 0 ? 0 : 16);
      }
      copies_commit();
      if constexpr (!std::is_same<M, T>::value) {
        // to f16 where they lie, each row by its own thread
        copies_wait<0>();
        __syncwarp();
        uint32_t top = 0;                                 // largest absolute value, as bits: NaN lies above infinity
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          const uint4 w = *reinterpret_cast<const uint4*>(place(lane, c));
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
        }
        top = max(top & 0xffffu, top >> 16) >> 7;         // bf16: eight bits of exponent above seven of fraction
        const int e = top == 255 ? 0 : max(-126, min(126, (int)top - 127));
        const float down = two_to(-e);
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          uint4* to = reinterpret_cast<uint4*>(place(lane, c));
          float x[8];
          unpack8<T>(*to, x);
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] *= down;
          *to = pack8<__half>(x);
        }
        scale *= two_to(e);
      }
    }
    int pos = 0x7fffffff;                                 // rows beyond the last look at everything and are dropped
    if (live) {
      const int sq = is_own ? seg : seq_of_row(a.cu, 0, a.num_seqs, tok);
      pos = sq < 0 ? -1 : row_pos(a, sq, tok);
    }
    pos = min(pos, k_hi - 1);
    if (n_tiles > 0) {
      copies_wait<0>();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_q[q]);
    }
    // f16 ends at 2^16 and has no numbers below 2^-24: probabilities are formed times 2^7 (at most 2^15), so that those down to 2^-21 keep all bits
    constexpr float kUp = std::is_same<M, __half>::value ? 7.0f : 0.0f;
    float m_run = -INFINITY, l_run = 0.f;
    // outputs are sums of probabilities times 2^up: with scales, less the exponent of the values' largest so far.  The sum of probabilities stands relative
    // to the maximum alone then: keys count whose values are far smaller than others
    float up = C::SCALED ? INFINITY : kUp;
    bool partly = false;                                  // some row of the warp does not see some key of its tiles
    bool bad = false;                                     // a score of the row is NaN: so is the result, whatever the exponentials made of it
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
      TileScales ts = {1.f, 0.f, 1.f, 0.f};
      float s_scl = scale;
      if constexpr (C::SCALED) {
        ts = s_tile[j & 7];
        s_scl = scale * ts.k_up;
      }
      const int hi = pos - kb, lo = k_lo - kb;
      if (__any_sync(0xffffffffu, hi < BN - 1 || lo > 0)) {
        partly = true;
#pragma unroll
        for (int i = 0; i < BN; ++i)
          if (i > hi || i < lo) sc[i] = -INFINITY;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < BN; i += 8) {
#pragma unroll
        for (int u = 0; u < 4; ++u) mx[u] = max_nan(mx[u], max_nan(sc[i + 2 * u], sc[i + 2 * u + 1]));
      }
      const float m_tile = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])) * s_scl;
      bad = bad || m_tile != m_tile;
      const bool grow = m_tile > m_run + 8.0f;
      const float m_new = grow ? m_tile : m_run;
      float up_new = up;
      if constexpr (C::SCALED) up_new = fminf(up, kUp - ts.v_exp);
      const float alpha = j > 0 && m_new > -INFINITY && (grow || up_new != up) ? exp2_fast((m_run - m_new) + (up_new - up)) : 1.0f;
      const float fade = C::SCALED ? (j > 0 && grow ? exp2_fast(m_run - m_new) : 1.0f) : alpha;
      m_run = m_new;
      up = up_new;
      // of this tile's probabilities; below 2^-32 they are zeros in f16, and by a factor of 2^-60 their sum still is what it is
      const float lift = C::SCALED ? fmaxf(up + ts.v_exp, -60.0f) : up;
      const float neg = m_new == -INFINITY ? 0.f : lift - m_new;
      float la[4] = {0.f, 0.f, 0.f, 0.f}, lb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float e0, e1;
          ffma2(e0, e1, sc[c * 32 + i], sc[c * 32 + i + 1], s_scl, s_scl, neg, neg);
          // every fourth exponential on the FMA pipe: the MUFU pipe alone would need as many clocks as a tile's products.  Not where warps
          // convert: there instructions are what is short
          const float p0 = exp2_fast(e0), p1 = C::BYTES || (i & 2) ? exp2_fast(e1) : exp2_fma(e1);
          fadd2(la[(i >> 1) & 3], lb[(i >> 1) & 3], la[(i >> 1) & 3], lb[(i >> 1) & 3], p0, p1);
          pk[i >> 1] = pack16<M>(p0, p1);
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
      l_run = l_run * fade + (C::SCALED ? l_tile * exp2_fast(-lift) : l_tile);
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_p[q * 2 + b]);
    }
    if (n_tiles > 0) {
      mbar_wait(&bar_o[q * 2 + ((n_tiles - 1) & 1)], ((n_tiles - 1) >> 1) & 1, 87);
      tcgen05_fence_after();
    }
    // every product has been formed, so queries, keys and values make room: rows go through shared memory, each lane's in a place of its own (a row is
    // 16 bytes longer than a multiple of 128, so that eight lanes never meet in a bank), and from there by the whole warp (a lane's 16 bytes to a row of its
    // own are 32 transactions per instruction: 9600 clocks for 256 rows of 132 numbers; a bulk copy per row: 6400)
    // the other tile's products read keys and values too; its barriers' phases may lie behind by more than one, so that its own warps have to say it
    if constexpr (NQ > 1) asm volatile("bar.sync 1, %0;" ::"n"(32 * C::SOFT) : "memory");
    if (bad) l_run = __int_as_float(0x7fc00000);
    const bool sees = pos >= k_lo;                        // no visible key: zero
    const float down = C::SCALED ? exp2f(-up) : 1.0f;     // of outputs, to the sum's reference
    const float inv = down / l_run;
    const int stride = ta.direct ? D * 2 + 16 : D * 4 + 16;
    uint8_t* stage = smem + (q * BM + quarter * 32) * stride;
    uint8_t* mine = stage + lane * stride;
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
      if (ta.direct) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          float f8[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f8[e] = sees ? __uint_as_float(r[i + e]) * inv : 0.f;
          *reinterpret_cast<uint4*>(mine + c * 64 + i * 2) = pack8<T>(f8);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(mine + c * 128 + i * 4) = make_float4(__uint_as_float(r[i]) * down, __uint_as_float(r[i + 1]) * down, __uint_as_float(r[i + 2]) * down, __uint_as_float(r[i + 3]) * down);
      }
    }
    uint8_t* to = nullptr;
    // (out of line: what a block runs once comes cold from memory.  A direct result may go over the queries: those rows are left out here)
    unsigned anew = 0;
    if constexpr (C::SCALED)
      if (partly) anew = spoiled_rows<T, FMT, D, NQ>(a, ta, t_o(q) + off, live && !bad);
    if (live && (anew >> lane & 1) == 0) {
      if (ta.direct) {
        to = reinterpret_cast<uint8_t*>(reinterpret_cast<T*>(a.out) + (int64_t)tok * a.ldo + (int64_t)head * D);
      } else {
        float* part = (is_own ? pa.tile_own : pa.tile_group) + (((int64_t)split * a.total_q + tok) * a.hq + head) * (D + kPad);
        *reinterpret_cast<float2*>(part + D) = make_float2(C::SCALED ? m_run : m_run - up, l_run);
        to = reinterpret_cast<uint8_t*>(part);
      }
    }
    __syncwarp();
    auto rows_out = [&](auto bytes) {
      constexpr int PER = decltype(bytes)::value / 16, LANES = PER < 32 ? PER : 32;   // 16 bytes of a row per lane
#pragma unroll 4
      for (int i = 0; i < 32; i += 32 / LANES) {
        const int row = i + lane / LANES;
        const uint64_t at = __shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(to), row);
        if (at != 0) {
#pragma unroll
          for (int c = 0; c < PER; c += LANES) {
            const int x = (c + lane % LANES) * 16;
            *reinterpret_cast<uint4*>(at + x) = *reinterpret_cast<const uint4*>(stage + row * stride + x);
          }
        }
      }
    };
    if (ta.direct) rows_out(std::integral_constant<int, D * 2>{});
    else rows_out(std::integral_constant<int, D * 4>{});
    if constexpr (!C::SCALED)
      if (partly) anew = spoiled_rows<T, FMT, D, NQ>(a, ta, t_o(q) + off, live && !bad);
    if (anew != 0) rows_anew<T, FMT, D, NQ>(a, pa, ta, anew);
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
  ta.direct = p.direct;
  ta.page_magic = (uint32_t)(((1ull << 31) + a.page / 16 - 1) / (a.page / 16));
  ta.run = a.page % 64 == 0 ? 64 : a.page % 32 == 0 ? 32 : 16;
  CUtensorMap map_k, map_v;
  memset(&map_k, 0, sizeof(map_k));
  memset(&map_v, 0, sizeof(map_v));
  if (!C::BYTES) {
    const int64_t rows = (int64_t)a.num_blocks * a.hkv * a.page;
    if (int e = encode_pages(&map_k, a.k, rows, D * 2, ta.run)) return e;
    if (int e = encode_pages(&map_v, a.v, rows, D * 2, ta.run)) return e;
  }
  const int64_t blocks = ((int64_t)t.own_tiles * p.own_splits * ta.segs_own + (int64_t)t.group_tiles * p.group_splits * a.groups) * a.hkv;
  LLMSS_REQUIRE(blocks < (1ll << 31), "attn_pages: grid too large (%lld blocks)", (long long)blocks);
  const dim3 grid((unsigned)blocks);
  LLMSS_CHECK_CUDA(launch_pdl(kern, grid, dim3(C::THREADS), (size_t)C::SMEM, stream, map_k, map_v, a, p, ta));
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
  if (fmt == kScaled16) return dtype == LLMSS_F16 ? by_size<__half, kScaled16>(a, p, t, stream) : by_size<__nv_bfloat16, kScaled16>(a, p, t, stream);
  if (dtype == LLMSS_F16)
    return fmt == kInt8 ? by_size<__half, kInt8>(a, p, t, stream) : fmt == kE4M3 ? by_size<__half, kE4M3>(a, p, t, stream) : by_size<__half, kF16Pages>(a, p, t, stream);
  return fmt == kInt8   ? by_size<__nv_bfloat16, kInt8>(a, p, t, stream)
         : fmt == kE4M3 ? by_size<__nv_bfloat16, kE4M3>(a, p, t, stream)
                        : by_size<__nv_bfloat16, kF16Pages>(a, p, t, stream);
}

}  // namespace pages
