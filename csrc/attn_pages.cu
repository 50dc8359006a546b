// Attention over cache pages: the choice of kernels, the merge of their parts, and a simple kernel for every shape.
#include "attn_pages.cuh"

namespace {

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_entry() {
  static EncodeTiled fn = nullptr;
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = (EncodeTiled)p;
  }
  return fn;
}

}  // namespace

namespace pages {

int encode_pages(CUtensorMap* map, const void* base, int64_t rows, int bytes, int box_rows) {
  EncodeTiled enc = encode_entry();
  LLMSS_REQUIRE(enc != nullptr, "attn_pages: cuTensorMapEncodeTiled entry point not available");
  cuuint64_t dims[2] = {(cuuint64_t)bytes, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)bytes};
  cuuint32_t box[2] = {(cuuint32_t)(bytes < 128 ? bytes : 128), (cuuint32_t)box_rows};
  cuuint32_t one[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         bytes < 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  LLMSS_REQUIRE(r == CUDA_SUCCESS, "attn_pages: cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
  return 0;
}

}  // namespace pages

namespace {

using namespace pages;

// ---------------------------------------------------------------------------------------------------------------- any shape
// One block per query row and head, its four warps on keys in turn, everything in 32 bits: head sizes and page sizes that the tiled kernels do not take.
template <typename T, int FMT>
__global__ void __launch_bounds__(128) attn_pages_any_kernel(const __grid_constant__ AttnArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int t = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = seq_of_row(a.cu, 0, a.num_seqs, t);
  if (s < 0) return;
  const int q_len = a.cu[s + 1] - a.cu[s];
  const int len = min(a.seq_lens[s], a.max_blocks * a.page);
  const int seen = min(len, a.seq_lens[s] - q_len + (t - a.cu[s]) + 1);     // keys 0 .. seen - 1
  const int g = group_of_seq(a, s);
  const int shared = g < 0 ? 0 : min(a.g_lens[g], a.g_max_blocks * a.page);
  const int kvh = head / (a.hq / a.hkv);
  float o[8], m, l;
  row_softmax<T, T, FMT>(a, t, head, warp, 4, seen, [&](int j) {
    const int* table = j < shared ? a.g_tables + (int64_t)g * a.g_max_blocks : a.tables + (int64_t)s * a.max_blocks;
    return ((int64_t)checked_block(table[j / a.page], a.num_blocks) * a.hkv + kvh) * a.page + j % a.page;
  }, o, m, l);
  __shared__ float s_m[4], s_l[4], s_o[4][256];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) s_o[warp][lane + 32 * i] = o[i];
  __syncthreads();
  const float mx = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float w[4], sum = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = s_m[i] == -INFINITY && !(s_l[i] != s_l[i]) ? 0.f : exp2f(s_m[i] - mx);
    sum += w[i] * s_l[i];
  }
  T* orow = reinterpret_cast<T*>(a.out) + (int64_t)t * a.ldo + (int64_t)head * a.d;
  for (int c = threadIdx.x; c < a.d; c += 128) {
    const float y = w[0] * s_o[0][c] + w[1] * s_o[1][c] + w[2] * s_o[2][c] + w[3] * s_o[3][c];
    orow[c] = from_f32<T>(seen > 0 ? y / sum : 0.f);     // a row that sees nothing is zero
  }
}

// ---------------------------------------------------------------------------------------------------------------- merge
// A warp per query row and head joins the parts of its softmax: m = max m_i, l = sum l_i 2^(m_i - m), out = sum O_i 2^(m_i - m) / l.  Reads what the
// kernels before it left in L2; launched to start as they end (programmatic dependent launch), so that it costs no launch latency of its own.
// WARPS of them share a row where rows are few: parts are many then, and each costs a read from L2.
template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(256, D < 256 && WARPS == 1 ? 5 : 4) attn_pages_merge_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ PartArgs p) {
  constexpr int N = D / 32, VEC = N < 4 ? N : 4;          // columns of a lane, VEC neighbouring ones
  using Vec = typename std::conditional<VEC == 4, float4, float2>::type;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int w = WARPS == 1 ? blockIdx.x * 8 + warp : blockIdx.x, mine = WARPS == 1 ? 0 : warp;
  const int t = w / a.hq, head = w % a.hq;
  if (t >= a.total_q) return;
  const int s = seq_of_row(a.cu, 0, a.num_seqs, t);      // lengths are not written by the kernels before
  if (s < 0) return;
  const int g = group_of_seq(a, s), group = a.hq / a.hkv, kvh = head / group;
  float o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = 0.f;
  const Seg own = own_segment(a, s);
  const Seg gs = g >= 0 ? group_segment(a, g) : Seg{};
  const bool sees = row_pos(a, s, t) >= 0, has_own = sees && own.hi > own.lo, has_group = sees && g >= 0 && gs.hi > 0;
  // parts lie in up to four runs: the own keys' first and others, the group's first and others (stretches of keys: the others only).  They are added in one
  // loop: with one per run a row waited for memory four times, and for the instructions of each
  // Places are counted in 16 bytes from the scratch's begin (p.slots): 32 bits, since registers decide how many rows are in flight.
  uint32_t run[4] = {0, 0, 0, 0}, step[4] = {0, 0, 0, 0};
  int ends[4] = {0, 0, 0, 0};
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr uint32_t ROW = (D + kPad) / 4;
  const uint32_t slot = p.rows * ROW, at = (uint32_t)(t * a.hq + head) * ROW;
  auto place = [&](const float* x) { return (uint32_t)((x - p.slots) >> 2); };
#pragma unroll
  for (int x = 0; x < 2; ++x) {                           // own keys, the group's
    int first = 0, others = 0;
    if (x == 0 ? has_own : has_group) {
      const Seg& sg = x == 0 ? own : gs;
      if (x == 0 ? p.few_own : p.few_groups) {
        const FewInfo in = p.info[(int64_t)(x == 0 ? s : (p.few_own ? a.num_seqs : 0) + g) * a.hkv + kvh];
        const int n = (t - sg.row0) * group + head % group;
        if (in.first_slot < 0) {
          if (a.groups == 0) return;                      // the result is written already
          run[2 * x] = place(x == 0 ? p.whole_own : p.whole_group) + at;
          first = 1;
        } else if (n < p.rows) {
          run[2 * x] = in.first_slot * slot + n * ROW;
          run[2 * x + 1] = 2 * (in.first_warp + 1) * slot + n * ROW;
          step[2 * x + 1] = 2 * slot;
          first = 1, others = in.last_warp - in.first_warp;
        }
      } else {
        const int chunk = x == 0 ? p.own_chunk : p.group_chunk;
        run[2 * x + 1] = place(x == 0 ? p.tile_own : p.tile_group) + at;
        step[2 * x + 1] = (uint32_t)(a.total_q * a.hq) * ROW;
        others = min(x == 0 ? p.own_splits : p.group_splits, (sg.hi - sg.lo + chunk - 1) / chunk);
      }
    }
    ends[2 * x] = (x > 0 ? ends[1] : 0) + first;
    ends[2 * x + 1] = ends[2 * x] + others;
  }
  // a lane looks at one part's maximum and sum, then all lanes add up the parts with their weights; with WARPS, every WARPS-th part
  const int count = ends[3] > mine ? (ends[3] - mine + WARPS - 1) / WARPS : 0;
  for (int b = 0; b < count; b += 32) {
    const int k = min(32, count - b);
    float2 ml = make_float2(-INFINITY, 0.f);
    uint32_t from = 0;
    if (lane < k) {
      const int x = (b + lane) * WARPS + mine;
      from = x < ends[0] ? run[0] : x < ends[1] ? run[1] + (x - ends[0]) * step[1] : x < ends[2] ? run[2] : run[3] + (x - ends[2]) * step[3];
      ml = *reinterpret_cast<const float2*>(p.slots + (int64_t)from * 4 + D);
    }
    const float mn = fmaxf(m, warp_max(ml.x)), base = mn == -INFINITY ? 0.f : mn;
    const float f = m == mn ? 1.f : exp2f(m - base), e = exp2f(ml.x - base);
    l = l * f + warp_sum(ml.y * e);
    m = mn;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] *= f;
    constexpr int AT_ONCE = 4;                            // parts on their way
    for (int j = 0; j < k; j += AT_ONCE) {
      float w[AT_ONCE];
      Vec v[AT_ONCE][N / VEC];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        w[u] = __shfl_sync(0xffffffffu, e, j + u);        // 0 of lanes without a part
        const float* part = p.slots + (int64_t)__shfl_sync(0xffffffffu, from, j + u) * 4;
#pragma unroll
        for (int i = 0; i < N / VEC; ++i) {
          v[u][i] = Vec{};
          if (w[u] != 0.f) v[u][i] = *reinterpret_cast<const Vec*>(part + i * 32 * VEC + lane * VEC);
        }
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) o[i] = fmaf(w[u], reinterpret_cast<const float*>(&v[u][i / VEC])[i % VEC], o[i]);
    }
  }
  if constexpr (WARPS > 1) {
    __shared__ float s_ml[WARPS][2];
    __shared__ float s_o[WARPS][D];
    if (lane == 0) s_ml[warp][0] = m, s_ml[warp][1] = l;
#pragma unroll
    for (int i = 0; i < N; ++i) s_o[warp][i * 32 + lane] = o[i];      // its own numbers, as they lie in the lane
    __syncthreads();
    if (warp > 0) return;
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < WARPS; ++j) m = fmaxf(m, s_ml[j][0]);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = 0.f;
#pragma unroll
    for (int j = 0; j < WARPS; ++j) {
      const float f = exp2f(s_ml[j][0] - (m == -INFINITY ? 0.f : m));
      l += s_ml[j][1] * f;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = fmaf(s_o[j][i * 32 + lane], f, o[i]);
    }
  }
  // a row that sees nothing, and so has no parts, is zero; NaN where a score was; where all visible scores are minus infinity l is 0, and the row NaN
  const float inv = ends[3] == 0 ? 0.f : 1.f / l;
  T* out = reinterpret_cast<T*>(a.out) + (int64_t)t * a.ldo + (int64_t)head * D;
#pragma unroll
  for (int i = 0; i < N; i += VEC) {
    T v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = from_f32<T>(o[i + e] * inv);
    using Out = typename std::conditional<VEC == 4, uint2, uint32_t>::type;
    Out x;
    memcpy(&x, v, sizeof(x));
    *reinterpret_cast<Out*>(out + i * 32 + lane * VEC) = x;
  }
}

template <typename T, int D>
int launch_merge(const AttnArgs& a, const PartArgs& p, int parts, cudaStream_t stream) {
  const int64_t rows = (int64_t)a.total_q * a.hq;
  // fewer rows than eight warps on each of 148 SMs, many parts of each: 8 sequences of 24000 tokens, 32 heads (28 parts) 83 -> 75 us with the merge; with two
  // parts a row (64 sequences of 1040 tokens, 16 heads) eight warps would cost 6 us of 99
  const bool shared = rows < 1184 && parts >= 8;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3((unsigned)(shared ? rows : (rows + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LLMSS_CHECK_CUDA(cudaLaunchKernelEx(&cfg, shared ? attn_pages_merge_kernel<T, D, 8> : attn_pages_merge_kernel<T, D, 1>, a, p));
  return 0;
}

// ---------------------------------------------------------------------------------------------------------------- codes as 16-bit pages
// 64 keys of one sequence and key head as f16 (TileScales), [sequence][head][pad][d] of keys, then of values; a page per sequence, so that the table names
// itself.  Bound by memory: 1 byte read, 2 written per value.
template <int FMT>
__global__ void __launch_bounds__(256) attn_pages_expand_kernel(const __grid_constant__ AttnArgs a, __half* __restrict__ out, TileScales* __restrict__ scales,
                                                                int* __restrict__ table, int pad) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s_scale[2][64];
  __shared__ int s_exp[2];
  const int s = blockIdx.z, kvh = blockIdx.y, key0 = blockIdx.x * 64;
  if (blockIdx.x == 0 && kvh == 0 && threadIdx.x == 0) table[s] = s;
  const int len = min(min(a.seq_lens[s], a.max_blocks * a.page), pad);
  if (key0 >= len) return;                 // the tiled kernel looks at no tile without a key
  const int per = a.d / 16;
  const int64_t list = ((int64_t)s * a.hkv + kvh) * pad, plane = (int64_t)a.num_seqs * a.hkv * pad;
  auto cache_row = [&](int key) {
    return ((int64_t)checked_block(a.tables[(int64_t)s * a.max_blocks + key / a.page], a.num_blocks) * a.hkv + kvh) * a.page + key % a.page;
  };
  if (threadIdx.x < 128) {
    const int value = threadIdx.x >> 6, key = key0 + (threadIdx.x & 63);
    s_scale[value][threadIdx.x & 63] = key < len ? (value ? a.vs : a.ks)[cache_row(key)] : 0.f;
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int value = threadIdx.x >> 5, lane = threadIdx.x & 31, e = tile_exponent(s_scale[value][lane], s_scale[value][lane + 32]);
    if (lane == 0) s_exp[value] = e;
  }
  __syncthreads();
  if (threadIdx.x == 0) scales[((int64_t)s * a.hkv + kvh) * (pad / 64) + blockIdx.x] = tile_scales(s_exp[0], s_exp[1]);
  const float down[2] = {two_to(-s_exp[0]), two_to(-s_exp[1])};
#pragma unroll 4
  for (int x = threadIdx.x; x < 2 * 64 * per; x += 256) {
    const int value = x >= 64 * per, y = value ? x - 64 * per : x;
    const int at = y / per, key = key0 + at, c = (y % per) * 16;
    if (key >= len) continue;
    const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(value ? a.v : a.k) + cache_row(key) * a.d + c);
    const float scale = s_scale[value][at] * (value ? down[1] : down[0]);
    uint4 lo, hi;
    convert4<FMT>(w.x, scale, lo.x, lo.y);
    convert4<FMT>(w.y, scale, lo.z, lo.w);
    convert4<FMT>(w.z, scale, hi.x, hi.y);
    convert4<FMT>(w.w, scale, hi.z, hi.w);
    __half* to = out + (value * plane + list + key) * a.d + c;
    *reinterpret_cast<uint4*>(to) = lo;
    *reinterpret_cast<uint4*>(to + 8) = hi;
  }
}

// ---------------------------------------------------------------------------------------------------------------- the choice
struct Plan {
  bool any;             // the simple kernel for the whole call
  bool few_own, few_groups;
  int blocks, rows;     // of the kernel for few rows
  TilePlan tile;
  int own_splits, own_chunk, group_splits, group_chunk;
  bool direct;          // the tiled kernel writes the result itself
  int pad;              // codes become 16-bit pages of this many keys first (0: not)
  int64_t slots, info, whole, tile_own, tile_group, expanded, floats;
};

// head sizes and pages of the tiled kernels
bool tiled(int d, int page) { return (d == 64 || d == 128 || d == 256) && page % 16 == 0; }

// Stretches of keys for `blocks` blocks of the tiled kernel, as many as make the call shortest: the blocks' waves over 148 SMs times a block's tiles of 64
// keys, where its start and end take as long as about five (measured: 6000 and 1100 clocks), and a merge that no other part of the call asks for as about
// eight.
void stretches(int64_t blocks, int keys, bool merged, int& splits, int& chunk) {
  const int64_t tiles = (keys + 63) / 64;
  int64_t best = 1, cost = -1;
  for (int64_t n = 1; n <= 148 && n <= (tiles + 1) / 2; ++n) {
    const int64_t c = (blocks * n + 147) / 148 * ((tiles + n - 1) / n + 5) + (n > 1 && !merged ? 8 : 0);
    if (cost < 0 || c < cost) best = n, cost = c;
  }
  chunk = (int)(tiles > 0 ? (tiles + best - 1) / best * 64 : 64);
  splits = keys > 0 ? (keys + chunk - 1) / chunk : 1;
}

// Prefixes by the tiled kernel, a sequence's own keys by the one for few rows: one after the other on all 148 SMs (beside a block of the first there is room for one
// of the second at most), or at the same time, the second on the SMs that fewer stretches of the first leave.  The estimates, in microseconds, were fitted to decode
// steps of 24 to 64 sequences with 60 to 3000 tokens of their own behind 1500 to 12000: a tile of 64 keys 1.15 (8 bits 1.45), an SM reading own keys 88 GB/s
// (8 bits, where it converts, 37) with 0.35 for each list, all of them 6.2 TB/s, starts 7 (8 bits 10) and 7.  64 sequences of 200 tokens behind 4096: 36.9 -> 24.7; of 3000 tokens: 147 -> 134;
// 48 of 300 behind three prefixes of 2500, int8: 41.0 -> 32.5.  All of these with the lengths' own bounds.  A captured step knows more generous ones, the
// estimate follows them, and the gain shrinks: the first with bounds of 4096 on the prefix and 8192 on all tokens 29, of 8192 on both 48; the last as four
// groups of up to 4096 tokens and 48 rows 50, of 2560 tokens and 16 rows 44.  Returns the SMs of the second kernel.
int side_by_side(int64_t lists, int len, double own_lists, double own_bytes, double part_bytes, int d, int fmt, int& splits, int& chunk) {
  const bool wide = fmt == kF16Pages;
  const int64_t tiles = (len + 63) / 64;
  const double start = wide ? 7 : 10, per_tile = (wide ? 1.15 : 1.45) * d / 128, part = part_bytes / 4e6, all = own_bytes / 6.2e6, one = own_bytes / (wide ? 88e3 : 37e3) + 0.35 * own_lists;
  auto prefix = [&](int64_t n) { return start + per_tile * ((lists * n + 147) / 148) * ((tiles + n - 1) / n); };
  auto own = [&](int64_t sms) { return 7 + (one / sms > all ? one / sms : all); };
  // a captured step knows bounds alone, and own keys may be far fewer: prefixes take twice as long as on all SMs at most (64 sequences of 200 tokens behind
  // 4096, all tokens bounded by 8192: 70.6 -> 28.7)
  const double longest = 2 * prefix(splits);
  double best = prefix(splits) + own(148) + part * splits;
  int64_t at = 0;
  for (int64_t n = 1; lists * n < 148 && n <= (tiles + 1) / 2; ++n) {
    const double a = prefix(n), b = own(148 - lists * n), c = (1.1 * a > b ? 1.1 * a : b) + part * n;
    if (a <= longest && c < best) best = c, at = n;
  }
  if (at == 0) return 148;
  chunk = (int)((tiles + at - 1) / at * 64);
  splits = (len + chunk - 1) / chunk;
  return 148 - (int)lists * splits;
}

Plan plan_call(int num_seqs, int max_q, int max_kv, int total_q, int hq, int hkv, int d, int page, int fmt, int groups, int g_max_len, int g_max_rows) {
  Plan p;
  memset(&p, 0, sizeof(p));
  p.any = true;
  if (hkv <= 0 || hq % hkv != 0 || !tiled(d, page)) return p;
  p.any = false;
  const int64_t g = hq / hkv, own = max_q * g, grouped = groups > 0 ? g_max_rows * g : 0;
  // up to 16 rows of a key head fit the narrow side of the warp-level product; a tile of 128 costs the tiled kernel the same whatever is in it
  p.few_own = own <= 16;
  p.few_groups = groups > 0 && grouped <= 16;
  const bool tile_own = !p.few_own, tile_groups = groups > 0 && !p.few_groups;
  p.tile.rows = tile_rows(d, own > 16 && own > grouped ? own : grouped);
  if (tile_own) {
    p.tile.own_tiles = (int)((own + p.tile.rows - 1) / p.tile.rows);
    // behind a prefix a sequence's own keys are few: the longest sequence less the longest prefix stands for them.  A guess costs time alone: the last stretch
    // of a list takes whatever is left of it, and a block without keys is not free (a microsecond on its SM)
    const int keys = groups > 0 ? (max_kv - g_max_len > max_q ? max_kv - g_max_len : max_q) : max_kv;
    stretches((int64_t)p.tile.own_tiles * hkv * num_seqs, keys, groups > 0, p.own_splits, p.own_chunk);
    p.direct = groups == 0 && p.own_splits == 1 && fmt != kF16Pages;      // (16-bit pages come here without groups where a prefix has no tokens, if at all)
    // Every row tile converts all codes for itself, which takes the tiled kernel from 1100 to 2000 clocks per 64 keys; once for all costs a pass over the
    // cache (about 1200 clocks of an SM per 64 keys, and a launch).  4 portions of 1000 tokens over 1800, 16 tiles each: 251 -> 183 us; three tiles 89 -> 87
    // (16 sequences 198 -> 170), two tiles 69 -> 68, one 47 -> 47: from three tiles on.  Up to 1 GB of scratch
    const int64_t pad = ((int64_t)max_kv + 63) / 64 * 64, expanded = (int64_t)num_seqs * hkv * (pad * d + pad / 64 * 4) + (num_seqs + 3) / 4 * 4;
    if (fmt != kF16Pages && groups == 0 && p.tile.own_tiles >= 3 && expanded <= (1ll << 28) && pad <= (1 << 19)) {
      p.pad = (int)pad;
      p.expanded = expanded;
    }
    if (!p.direct) p.tile_own = (int64_t)p.own_splits * total_q * hq * (d + kPad);
  }
  int few_sms = 148;
  if (tile_groups) {
    p.tile.group_tiles = (int)((grouped + p.tile.rows - 1) / p.tile.rows);
    const int64_t lists = (int64_t)p.tile.group_tiles * hkv * groups;
    stretches(lists, g_max_len, true, p.group_splits, p.group_chunk);
    if (p.few_own) {
      // three quarters of the longest: sequences differ, and a tiled kernel that takes longer than the other costs more than one that takes less
      const double keys = 0.75 * (max_kv > g_max_len ? max_kv - g_max_len : 1);
      few_sms = side_by_side(lists, g_max_len, (double)num_seqs * hkv, keys * num_seqs * hkv * d * (fmt == kF16Pages ? 4 : 2), (double)total_q * hq * (d + kPad) * 4, d, fmt,
                             p.group_splits, p.group_chunk);
    }
    p.tile_group = (int64_t)p.group_splits * total_q * hq * (d + kPad);
  }
  if (p.few_own || p.few_groups) {
    p.rows = (int)(p.few_own && (!p.few_groups || own >= grouped) ? own : grouped);
    p.blocks = few_blocks(fmt, d, p.rows, (p.few_own ? num_seqs : 0) + (p.few_groups ? groups : 0)) / 148 * few_sms;
    p.slots = (int64_t)2 * p.blocks * kFewWarps * p.rows * (d + kPad);
    p.info = ((int64_t)(p.few_own ? num_seqs : 0) + (p.few_groups ? groups : 0)) * hkv * 4;
    p.whole = groups > 0 ? (int64_t)total_q * hq * (d + kPad) : 0;
  }
  p.floats = p.slots + p.info + (p.few_own ? p.whole : 0) + (p.few_groups ? p.whole : 0) + p.tile_own + p.tile_group + p.expanded;
  return p;
}

int check_args(const AttnArgs& a, int fmt, int dtype) {
  LLMSS_REQUIRE(dtype == LLMSS_F16 || dtype == LLMSS_BF16, "attn_pages: dtype must be f16/bf16");
  LLMSS_REQUIRE(fmt >= kF16Pages && fmt <= kE4M3, "attn_pages: page format %d unknown", fmt);
  LLMSS_REQUIRE(a.hq > 0 && a.hkv > 0 && a.hq % a.hkv == 0, "attn_pages: bad head grouping hq=%d hkv=%d", a.hq, a.hkv);
  LLMSS_REQUIRE(a.d > 0 && a.d % 8 == 0 && a.d <= 256, "attn_pages: head_dim=%d must be a multiple of 8 up to 256", a.d);
  LLMSS_REQUIRE(a.page > 0 && a.num_blocks > 0 && a.max_blocks >= 0, "attn_pages: bad pages (block_size=%d, %d blocks)", a.page, a.num_blocks);
  LLMSS_REQUIRE((int64_t)a.max_blocks * a.page < (1ll << 31) && (int64_t)a.g_max_blocks * a.page < (1ll << 31), "attn_pages: contexts of 2^31 tokens and more");
  LLMSS_REQUIRE(((int64_t)(a.num_seqs + a.groups) * (a.max_blocks > a.g_max_blocks ? a.max_blocks : a.g_max_blocks)) * (a.page / 16 + 1) * a.hkv < (1ll << 31),
                "attn_pages: lists of 2^35 keys and more (%d sequences of up to %d pages)", a.num_seqs, a.max_blocks);
  LLMSS_REQUIRE((int64_t)a.page * a.page * (a.max_blocks > a.g_max_blocks ? a.max_blocks : a.g_max_blocks) < (1ll << 39), "attn_pages: pages too large (%d)", a.page);
  LLMSS_REQUIRE((int64_t)a.num_blocks * a.hkv * a.page < (1ll << 31), "attn_pages: 2^31 cache rows and more");
  LLMSS_REQUIRE((((uintptr_t)a.ks | (uintptr_t)a.vs) % 16) == 0, "attn_pages: scales must be 16-byte aligned");
  LLMSS_REQUIRE((int64_t)a.hq * a.d <= a.ldq && (int64_t)a.hq * a.d <= a.ldo, "attn_pages: q / out columns exceed the row stride");
  LLMSS_REQUIRE(a.scale_log2 > 0.f && a.scale_log2 < INFINITY, "attn_pages: the score scale must be positive and finite");
  LLMSS_REQUIRE(fmt == kF16Pages || (a.ks != nullptr && a.vs != nullptr), "attn_pages: 8-bit pages need scales");
  LLMSS_REQUIRE(a.groups == 0 || (a.g_tables != nullptr && a.g_lens != nullptr && a.g_first != nullptr), "attn_pages: groups need tables, lengths and firsts");
  LLMSS_REQUIRE(a.ldq % 8 == 0 && a.ldo % 8 == 0 && (((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k | (uintptr_t)a.v) % 16) == 0,
                "attn_pages: q / out rows and pages must be 16-byte aligned");
  return 0;
}

}  // namespace

// Floats of scratch that llmss_attn_pages takes for a call of these sizes (0: none).
LLMSS_API int64_t llmss_attn_pages_scratch_floats(int num_seqs, int max_q, int max_kv, int total_q, int hq, int hkv, int d, int block_size, int fmt,
                                                  int groups, int g_max_len, int g_max_rows) {
  if (num_seqs <= 0 || total_q <= 0 || max_q <= 0) return 0;
  return plan_call(num_seqs, max_q, max_kv, total_q, hq, hkv, d, block_size, fmt, g_max_len > 0 ? groups : 0, g_max_len, g_max_rows).floats;
}

// q [total_q][>= hq * d] (row stride ldq); K / V pages [num_blocks][hkv][block_size][d] of the queries' type (fmt 0) or of bytes with 32-bit scales
// [num_blocks][hkv][block_size] (fmt 1 int8, 2 e4m3); sequence i owns the rows cu_q[i] .. cu_q[i + 1] - 1, the last positions of its seq_lens[i] cached
// tokens.  groups > 0: the sequences g_first[j] .. g_first[j + 1] - 1 find their first g_lens[j] tokens in the pages g_tables[j].  max_q, max_kv,
// g_max_len, g_max_rows bound the lengths.  *launches: kernels launched (null: not wanted).  out is q itself or shares no memory with it.  Rows of sequences without a visible key become zero; rows of no sequence stay as they are.
LLMSS_API int llmss_attn_pages(const void* q, int64_t ldq, const void* k_pages, const float* k_scale, const void* v_pages, const float* v_scale,
                               const int* block_tables, int max_blocks, const int* seq_lens, void* out, int64_t ldo, const int* cu_q, int num_seqs,
                               int max_q, int max_kv, int total_q, int hq, int hkv, int d, int block_size, int num_blocks, float scale, int fmt,
                               int dtype, const int* g_tables, int g_max_blocks, const int* g_lens, const int* g_first, int groups, int g_max_len,
                               int g_max_rows, void* scratch, int64_t scratch_floats, int* launches, cudaStream_t stream) {
  int none = 0;
  if (launches == nullptr) launches = &none;
  *launches = 0;
  AttnArgs a;
  memset(&a, 0, sizeof(a));
  a.q = q;
  a.k = k_pages;
  a.v = v_pages;
  a.ks = k_scale;
  a.vs = v_scale;
  a.out = out;
  a.tables = block_tables;
  a.seq_lens = seq_lens;
  a.cu = cu_q;
  a.g_tables = g_tables;
  a.g_lens = g_lens;
  a.g_first = g_first;
  a.ldq = ldq;
  a.ldo = ldo;
  a.num_seqs = num_seqs;
  a.total_q = total_q;
  a.max_blocks = max_blocks;
  a.g_max_blocks = g_max_blocks;
  a.groups = g_max_len > 0 ? groups : 0;
  a.hq = hq;
  a.hkv = hkv;
  a.d = d;
  a.page = block_size;
  a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  LLMSS_REQUIRE(num_seqs >= 0 && max_q >= 0 && max_kv >= 0 && total_q >= 0 && groups >= 0, "attn_pages: negative size");
  if (num_seqs == 0 || total_q == 0 || max_q == 0) return 0;
  if (int e = check_args(a, fmt, dtype)) return e;
  const Plan plan = plan_call(num_seqs, max_q, max_kv, total_q, hq, hkv, d, block_size, fmt, a.groups, g_max_len, g_max_rows);
  if (!plan.any) {
    LLMSS_REQUIRE(plan.floats == 0 || (scratch != nullptr && scratch_floats >= plan.floats && ((uintptr_t)scratch % 16) == 0), "attn_pages: %lld floats of 16-byte aligned scratch needed",
                  (long long)plan.floats);
    LLMSS_REQUIRE(plan.floats < (1ll << 34), "attn_pages: 64 GB of scratch and more");   // the merge kernel's places
    PartArgs p;
    memset(&p, 0, sizeof(p));
    float* at = (float*)scratch;
    auto take = [&](int64_t n) {
      float* x = at;
      at += n;
      return x;
    };
    p.slots = take(plan.slots);
    p.info = (FewInfo*)take(plan.info);
    p.whole_own = take(plan.few_own ? plan.whole : 0);
    p.whole_group = take(plan.few_groups ? plan.whole : 0);
    p.tile_own = take(plan.tile_own);
    p.tile_group = take(plan.tile_group);
    p.rows = plan.rows;
    p.few_own = plan.few_own;
    p.few_groups = plan.few_groups;
    p.own_splits = plan.own_splits;
    p.own_chunk = plan.own_chunk;
    p.group_splits = plan.group_splits;
    p.group_chunk = plan.group_chunk;
    p.direct = plan.direct;
    const bool tiles = plan.tile.own_tiles > 0 || plan.tile.group_tiles > 0;
    float* expanded = take(plan.expanded);
    if (plan.pad > 0) {
      // from here on the cache is the 16-bit copy, one page per sequence
      const int64_t plane = (int64_t)num_seqs * hkv * plan.pad;
      TileScales* scales = (TileScales*)(expanded + plane * d);
      int* table = (int*)(scales + plane / 64);
      const dim3 grid(plan.pad / 64, hkv, num_seqs);
      LLMSS_REQUIRE(grid.y <= 65535 && grid.z <= 65535, "attn_pages: grid too large (%d key heads, %d sequences)", hkv, num_seqs);
      LLMSS_CHECK_CUDA(fmt == kInt8 ? launch_pdl(attn_pages_expand_kernel<kInt8>, grid, dim3(256), 0, stream, a, (__half*)expanded, scales, table, plan.pad)
                                    : launch_pdl(attn_pages_expand_kernel<kE4M3>, grid, dim3(256), 0, stream, a, (__half*)expanded, scales, table, plan.pad));
      ++*launches;
      a.k = expanded;
      a.v = (const uint16_t*)expanded + plane * d;
      a.tile_scales = scales;
      a.tables = table;
      a.max_blocks = 1;
      a.page = plan.pad;
      a.num_blocks = num_seqs;
      fmt = kScaled16;
    }
    if (tiles) {
      if (int e = tile_launch(a, p, plan.tile, fmt, dtype, stream)) return e;
      ++*launches;
    }
    if (plan.direct) return 0;
    if (plan.few_own || plan.few_groups) {
      if (int e = few_launch(a, p, fmt, dtype, plan.blocks, tiles, stream)) return e;
      ++*launches;
    }
    ++*launches;
    // parts of a row, about: runs of a list, or stretches
    const int64_t lists = ((int64_t)(plan.few_own ? num_seqs : 0) + (plan.few_groups ? a.groups : 0)) * hkv;
    const int64_t runs = lists > 0 ? (int64_t)plan.blocks * kFewWarps / lists : 0;
    const int parts = (int)(runs > plan.own_splits + plan.group_splits ? runs : plan.own_splits + plan.group_splits);
#define LLMSS_MERGE(T_) return d == 64 ? launch_merge<T_, 64>(a, p, parts, stream) : d == 128 ? launch_merge<T_, 128>(a, p, parts, stream) : launch_merge<T_, 256>(a, p, parts, stream)
    if (dtype == LLMSS_F16) LLMSS_MERGE(__half);
    LLMSS_MERGE(__nv_bfloat16);
#undef LLMSS_MERGE
  }
  const dim3 grid(total_q, hq);
  LLMSS_REQUIRE(grid.y <= 65535, "attn_pages: %d heads", hq);
#define LLMSS_ANY(T_, F_) LLMSS_CHECK_CUDA(launch_pdl(attn_pages_any_kernel<T_, F_>, grid, dim3(128), 0, stream, a))
  if (dtype == LLMSS_F16) {
    if (fmt == kInt8) LLMSS_ANY(__half, kInt8);
    else if (fmt == kE4M3) LLMSS_ANY(__half, kE4M3);
    else LLMSS_ANY(__half, kF16Pages);
  } else {
    if (fmt == kInt8) LLMSS_ANY(__nv_bfloat16, kInt8);
    else if (fmt == kE4M3) LLMSS_ANY(__nv_bfloat16, kE4M3);
    else LLMSS_ANY(__nv_bfloat16, kF16Pages);
  }
#undef LLMSS_ANY
  ++*launches;
  LLMSS_CHECK_CUDA(cudaGetLastError());
  return 0;
}
