// Causal attention over a paged cache in 16 or 8 bits, with cached tokens that groups of sequences share.
//
//   s_jk = scale (q_j . K_k)      K_k = ks_k code_k      p = softmax over the keys k <= pos_j      out_j = sum_k p_jk vs_k code_k
//
// A sequence of a group (SharedGroups) finds its first len keys in the group's pages and the others in its own; a softmax over both is the merge
// of the two parts by their maxima and sums.
#include "common.cuh"

#include <cuda_fp8.h>

namespace {

constexpr int kF16Pages = 0, kInt8 = 1, kE4M3 = 2;    // page formats; 0: the queries' own 16-bit type

struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  const float* ks;
  const float* vs;
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
  float q[8], o[8], m = -INFINITY, l = 0.f;
  const T* qr = reinterpret_cast<const T*>(a.q) + (int64_t)t * a.ldq + (int64_t)head * a.d;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    q[i] = lane + 32 * i < a.d ? to_f32(qr[lane + 32 * i]) : 0.f;
    o[i] = 0.f;
  }
  for (int j = warp; j < seen; j += 4) {
    const int* table = j < shared ? a.g_tables + (int64_t)g * a.g_max_blocks : a.tables + (int64_t)s * a.max_blocks;
    const int64_t r = ((int64_t)checked_block(table[j / a.page], a.num_blocks) * a.hkv + kvh) * a.page + j % a.page;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < a.d) x = fmaf(q[i], page_value<T, FMT>(a.k, r * a.d + lane + 32 * i), x);
    x = warp_sum(x) * a.scale_log2;
    if constexpr (FMT != kF16Pages) x *= a.ks[r];
    const float mn = fmaxf(m, x), al = m == mn ? 1.f : exp2f(m - mn), p = x == -INFINITY ? 0.f : exp2f(x - mn);
    l = l * al + p;
    const float pv = FMT != kF16Pages ? p * a.vs[r] : p;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] *= al;
      if (lane + 32 * i < a.d) o[i] = fmaf(pv, page_value<T, FMT>(a.v, r * a.d + lane + 32 * i), o[i]);
    }
    m = mn;
  }
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

int check_args(const AttnArgs& a, int fmt, int dtype) {
  LLMSS_REQUIRE(dtype == LLMSS_F16 || dtype == LLMSS_BF16, "attn_pages: dtype must be f16/bf16");
  LLMSS_REQUIRE(fmt >= kF16Pages && fmt <= kE4M3, "attn_pages: page format %d unknown", fmt);
  LLMSS_REQUIRE(a.hq > 0 && a.hkv > 0 && a.hq % a.hkv == 0, "attn_pages: bad head grouping hq=%d hkv=%d", a.hq, a.hkv);
  LLMSS_REQUIRE(a.d > 0 && a.d % 8 == 0 && a.d <= 256, "attn_pages: head_dim=%d must be a multiple of 8 up to 256", a.d);
  LLMSS_REQUIRE(a.page > 0 && a.num_blocks > 0 && a.max_blocks >= 0, "attn_pages: bad pages (block_size=%d, %d blocks)", a.page, a.num_blocks);
  LLMSS_REQUIRE((int64_t)a.max_blocks * a.page < (1ll << 31) && (int64_t)a.g_max_blocks * a.page < (1ll << 31), "attn_pages: contexts of 2^31 tokens and more");
  LLMSS_REQUIRE((int64_t)a.hq * a.d <= a.ldq && (int64_t)a.hq * a.d <= a.ldo, "attn_pages: q / out columns exceed the row stride");
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
  (void)num_seqs, (void)max_q, (void)max_kv, (void)total_q, (void)hq, (void)hkv, (void)d, (void)block_size, (void)fmt, (void)groups, (void)g_max_len,
      (void)g_max_rows;
  return 0;
}

// q [total_q][>= hq * d] (row stride ldq); K / V pages [num_blocks][hkv][block_size][d] of the queries' type (fmt 0) or of bytes with 32-bit scales
// [num_blocks][hkv][block_size] (fmt 1 int8, 2 e4m3); sequence i owns the rows cu_q[i] .. cu_q[i + 1] - 1, the last positions of its seq_lens[i] cached
// tokens.  groups > 0: the sequences g_first[j] .. g_first[j + 1] - 1 find their first g_lens[j] tokens in the pages g_tables[j].  max_q, max_kv,
// g_max_len, g_max_rows bound the lengths.  out may alias q.  Rows of sequences without a visible key become zero; rows of no sequence stay as they are.
LLMSS_API int llmss_attn_pages(const void* q, int64_t ldq, const void* k_pages, const float* k_scale, const void* v_pages, const float* v_scale,
                               const int* block_tables, int max_blocks, const int* seq_lens, void* out, int64_t ldo, const int* cu_q, int num_seqs,
                               int max_q, int max_kv, int total_q, int hq, int hkv, int d, int block_size, int num_blocks, float scale, int fmt,
                               int dtype, const int* g_tables, int g_max_blocks, const int* g_lens, const int* g_first, int groups, int g_max_len,
                               int g_max_rows, void* scratch, int64_t scratch_floats, cudaStream_t stream) {
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
  a.groups = g_max_len > 0 && g_max_blocks > 0 ? groups : 0;
  a.hq = hq;
  a.hkv = hkv;
  a.d = d;
  a.page = block_size;
  a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  LLMSS_REQUIRE(num_seqs >= 0 && max_q >= 0 && max_kv >= 0 && total_q >= 0 && groups >= 0, "attn_pages: negative size");
  if (num_seqs == 0 || total_q == 0 || max_q == 0) return 0;
  if (int e = check_args(a, fmt, dtype)) return e;
  (void)scratch, (void)scratch_floats;
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
  LLMSS_CHECK_CUDA(cudaGetLastError());
  return 0;
}
