// Attention of one new token of every sequence over its paged key / value cache.
//
// Per sequence and key / value head: S = scale Q K^T for the G query heads that share it, a softmax over the positions
// in one pass (running maximum and sum), O = P V.  Every key and value is read once and used for G heads: the work is
// bound by memory, 1 to 2 operations a byte and head.  So the kernel is built around its loads:
//
//  * The G queries (up to 16) are the columns of 16-wide matrix instructions, whatever G is: the matrix cores have an order of
//    magnitude to spare here, and the vector ALUs, which a dot product per head would fill, stay free.
//  * Keys and values go from memory into registers in the layout that the matrix instructions take, without LDS and without
//    barriers: S^T = K Q^T wants a key's row in pieces of 8 along d, which is how it lies in memory.  O^T = V^T P^T
//    wants 8 keys of one column in a lane.  A lane loads the same piece of a row for 8 keys, 16 lanes a whole row, and turns the 8 x 8
//    block in its registers, one v_perm_b32 per register: row m of fragment i is column m CE + i (CE = DP / 16 columns a lane).
//  * The accumulators of S^T leave a lane with keys 4 g .. 4 g + 3 of both 16-key tiles of a step of one query, which, in that
//    order of the keys, is the second operand of O^T (the lane loads the values of exactly those keys).
//  * The waves of a workgroup take the steps of its share of the positions in turn, each on its own; their results are brought to
//    the common maximum and added through LDS at the end.  A long cache is shared out between `splits` workgroups,
//    each leaving (maximum, sum, sum of p v), which a second launch joins.
//  * The table is read two steps ahead by the scalar unit, so that no step waits for a lookup or drains the loads on the way.
//
// Measured, keys and values out of memory: 16 sequences of 8192 to 32768 in bf16, 8 heads of 128 with 4 queries each, 256 us (5.2 TB/s) and 5 for
// the join; 64 sequences of 256 to 1024, 12 heads of 64, 31 us (4.1 TB/s); 32 sequences of 2048 to 8192 in e4m3, 4 heads of 128 with 8 queries
// each, 38 us (4.4 TB/s) and 5.  Out of the caches all of it takes 136, 19 and 34: the longer ones are bound by memory, and by what one CU draws of
// it (31 B/ns) where the sequences' lengths do not fill all CUs to the end.  One sequence of 1000, 12 heads of 64: 6.1 us and 3.6, the chain of
// table, keys, values and join.
//
// 16-bit types: P is split into values of the type, each nearest to what the ones before leave: three of bf16 have all 24 places of an f32, two of
// f16 have 22, and there is a matrix instruction for each.  (Where values cancel, what P has lost shows in the result: with two of bf16,
// 2^-18 of the largest values.  The third costs long caches less than 1 %, 8 sequences of 256 to 1024, 16 heads of 64, 12.0 us instead of 11.7.)
// f32 runs on v_mfma_f32_16x16x4_f32 with one 16-key tile a step.  e4m3 codes are converted to the queries' type, in which every code has
// an exact value.
#include "paged_rows.h"

namespace lh {

// Shares that n positions take.
__device__ __forceinline__ int paged_parts(const PagedAttnArgs& a, int n) { return (int)(((uint32_t)n + (uint32_t)a.share - 1u) / (uint32_t)a.share); }

// (maximum, sum) of one query over its parts, to every lane of the wave: the lanes take the parts in turn, the lanes' values are
// brought together in a fixed order.
__device__ __forceinline__ float2 paged_join(const float2* ml, int parts, int rows, int lane) {
  float m = -INFINITY, l = 0.0f;
  for (int p = lane; p < parts; p += 64) {
    const float2 x = ml[(int64_t)p * rows];
    const float to = fmaxf(m, x.x), safe = to == -INFINITY ? 0.0f : to;
    l = l * __builtin_amdgcn_exp2f(m - safe) + x.y * __builtin_amdgcn_exp2f(x.x - safe);
    m = to;
  }
  float all = m;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) all = fmaxf(all, __shfl_xor(all, o));
  const float safe = all == -INFINITY ? 0.0f : all;
  l *= __builtin_amdgcn_exp2f(m - safe);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o);
  return make_float2(safe, l);
}

// The first B H workgroups join the parts of a query each: they bring them to the common maximum and add them in the order of the
// positions.  The others, where weights are asked for, take 256 positions of a head of a sequence: weights[b, g, t] += sum over the
// heads of the group of exp2(score - log2 of the head's sum), heads in order; they find that sum for themselves.
template <int QDT, int DP>
__global__ void __launch_bounds__(256) paged_attention_finish(PagedAttnArgs a, int joins, float* weights, int64_t sw_b, int64_t sw_h) {
  constexpr int GROUPS = 256 / DP;
  __shared__ float sums[GROUPS][DP];
  __shared__ float lse[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if ((int)blockIdx.x < joins) {
    const int bh = blockIdx.x, b = bh / a.H, head = bh % a.H;
    const int n = paged_length(a, b), parts = paged_parts(a, n);
    if (parts <= 1) return;  // (written at once)
    const int hk = head / a.G, q_row = head % a.G, col = tid % DP, first = tid / DP;
    const int64_t at = ((int64_t)(b * a.c.heads + hk) * a.groups + q_row / 16) * a.splits * a.rows + q_row % 16;
    // (the first of a thread's parts are requested before the maximum is known)
    constexpr int EARLY = 8;
    float early[EARLY], scale[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; ++i) {
      const int64_t p = at + (int64_t)min(first + i * GROUPS, parts - 1) * a.rows;
      early[i] = a.part_o[p * DP + col], scale[i] = a.part_ml[p].x;
    }
    const float2 ml = paged_join(a.part_ml + at, parts, a.rows, lane);
    float o = 0.0f;
#pragma unroll
    for (int i = 0; i < EARLY; ++i)
      if (first + i * GROUPS < parts) o += early[i] * __builtin_amdgcn_exp2f(scale[i] - ml.x);
#pragma unroll 4
    for (int p = first + EARLY * GROUPS; p < parts; p += GROUPS)
      o += a.part_o[(at + (int64_t)p * a.rows) * DP + col] * __builtin_amdgcn_exp2f(a.part_ml[at + (int64_t)p * a.rows].x - ml.x);
    if (GROUPS > 1) {
      sums[first][col] = o;
      __syncthreads();
      if (first > 0) return;
#pragma unroll
      for (int g = 1; g < GROUPS; ++g) o += sums[g][col];
    }
    if (col < a.c.d) store_from_f32<QDT>(a.out, b * a.so_z + head * a.so_h + col, ml.y == 0.0f ? 0.0f : o * (a.c.v_scale / ml.y));
    return;
  }
  const int per_head = (a.c.capacity() + 255) / 256, bh = (blockIdx.x - joins) / per_head;
  const int b = bh / a.c.heads, hk = bh % a.c.heads;
  const int t0 = (blockIdx.x - joins - bh * per_head) * 256, t = t0 + tid;
  const int n = paged_length(a, b);
  if (t0 >= n) return;
  const int parts = paged_parts(a, n);
  const int64_t first = (int64_t)b * a.H + hk * a.G;
  // (What does not wait for the sums is requested before them: the scores of the first heads and the weight that grows.)
  constexpr int EARLY = 8;
  float early[EARLY], sum = 0.0f, old = 0.0f;
  float* const to = weights + b * sw_b + hk * sw_h + t;
  const float* const scores = a.scores + first * a.cap_pad + t;
#pragma unroll
  for (int g = 0; g < EARLY; ++g) early[g] = t < n && g < a.G ? scores[(int64_t)g * a.cap_pad] : -INFINITY;
  if (t < n) old = *to;
  for (int g0 = 0; g0 < a.G; g0 += 256) {  // (up to 256 heads of a group at a time)
    const int many = min(256, a.G - g0);
    if (g0 > 0) __syncthreads();
    if (parts == 1) {
      if (tid < many) lse[tid] = a.lse[first + g0 + tid];
    } else {
      for (int g = wave; g < many; g += 4) {
        const int64_t at = ((int64_t)bh * a.groups + (g0 + g) / 16) * a.splits * a.rows + (g0 + g) % 16;
        const float2 ml = paged_join(a.part_ml + at, parts, a.rows, lane);
        if (lane == 0) lse[g] = ml.x + __builtin_amdgcn_logf(ml.y);
      }
    }
    __syncthreads();
    auto add = [&](float x, int g) { sum += x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - lse[g]); };
    if (g0 == 0) {
#pragma unroll
      for (int g = 0; g < EARLY; ++g)
        if (g < many) add(early[g], g);
    }
    if (t < n)
#pragma unroll 4
      for (int g = g0 == 0 ? EARLY : 0; g < many; ++g) add(scores[(int64_t)(g0 + g) * a.cap_pad], g);
  }
  if (t < n) *to = old + sum;
}

// ---- host side ------------------------------------------------------------------------------------------------------------

struct PagedPlan {
  int rows, groups, share, splits, dp, cap_pad;
  int mode;
  size_t o_bytes, ml_bytes, score_bytes, lse_bytes;
  size_t total() const { return o_bytes + ml_bytes + score_bytes + lse_bytes; }
};

static bool paged_batch(int64_t B, int64_t H) {
  constexpr int64_t kMost = 1ll << 20;
  return B > 0 && H > 0 && B < kMost && H < kMost && B * H < kMost;
}

static size_t granules(size_t b) { return (b + 255) / 256 * 256; }

static PagedPlan paged_plan(const Paged& c, int cache_dtype, int64_t B, int64_t H, bool with_weights, bool aligned) {
  PagedPlan p = {};
  const int G = (int)(H / c.heads);
  p.rows = G < 16 ? G : 16, p.groups = (G + 15) / 16;
  p.dp = paged_width(c.d);
  const int es = (int)dtype_size(cache_dtype);
  p.mode = paged_mode(c, es, aligned);
  const int64_t items = B * c.heads * p.groups;
  p.share = paged_share(items, c.capacity(), paged_occupancy(cache_dtype, p.dp, p.mode), 2 * (int64_t)c.d * es);
  p.splits = (int)(((int64_t)c.capacity() + p.share - 1) / p.share);
  if (p.splits > 1) {
    p.o_bytes = granules((size_t)items * p.splits * p.rows * p.dp * 4);
    p.ml_bytes = granules((size_t)items * p.splits * p.rows * 8);
  }
  if (with_weights) {
    p.cap_pad = (c.capacity() + 31) / 32 * 32;
    p.score_bytes = granules((size_t)B * H * p.cap_pad * 4);
    p.lse_bytes = granules((size_t)B * H * 4);
  }
  return p;
}

template <int CDT, int QDT, int DP>
static int launch_paged(const PagedAttnArgs& a, int mode, float* weights, int64_t sw_b, int64_t sw_h, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.B * a.c.heads * a.groups * a.splits)), block(kPagedWaves * 64);
  if (mode == kTiles) LH_LAUNCH((paged_attention_kernel<CDT, QDT, DP, kPagedWaves, kTiles, PagedAttnArgs>), grid, block, 0, s, a);
  else if (mode == kWholeRows) LH_LAUNCH((paged_attention_kernel<CDT, QDT, DP, kPagedWaves, kWholeRows, PagedAttnArgs>), grid, block, 0, s, a);
  else LH_LAUNCH((paged_attention_kernel<CDT, QDT, DP, kPagedWaves, kOddRows, PagedAttnArgs>), grid, block, 0, s, a);
  if (const int rc = check_launch("paged_attention")) return rc;
  const int joins = a.splits > 1 ? a.B * a.H : 0;
  const unsigned blocks = joins + (weights ? (unsigned)((a.c.capacity() + 255) / 256 * (int64_t)a.B * a.c.heads) : 0u);
  if (blocks == 0) return LH_OK;
  LH_LAUNCH((paged_attention_finish<QDT, DP>), dim3(blocks), dim3(256), 0, s, a, joins, weights, sw_b, sw_h);
  return check_launch("paged_attention_finish");
}

template <int CDT, int QDT>
static int launch_paged_dp(const PagedAttnArgs& a, int dp, int mode, float* w, int64_t sw_b, int64_t sw_h, hipStream_t s) {
  if (dp == 64) return launch_paged<CDT, QDT, 64>(a, mode, w, sw_b, sw_h, s);
  if (dp == 128) return launch_paged<CDT, QDT, 128>(a, mode, w, sw_b, sw_h, s);
  return launch_paged<CDT, QDT, 256>(a, mode, w, sw_b, sw_h, s);
}

}  // namespace lh

using namespace lh;

extern "C" {

size_t lh_hip_paged_attention_workspace_bytes(const lh_paged_cache* cache, int64_t B, int64_t H, int32_t with_weights) {
  Paged c;
  if (paged_cache(cache, "lh_hip_paged_attention_workspace_bytes", &c) != LH_OK) return 0;
  if (!paged_batch(B, H) || H % c.heads != 0) return 0;
  // (Room for either alignment: a caller may size it with one cache and pass a view of another.)
  const size_t one = paged_plan(c, cache->dtype, B, H, with_weights != 0, true).total(), other = paged_plan(c, cache->dtype, B, H, with_weights != 0, false).total();
  return one > other ? one : other;
}

int lh_hip_paged_attention(const lh_paged_cache* cache, void* out, const void* q, int64_t out_stride_b, int64_t out_stride_h,
                           int64_t q_stride_b, int64_t q_stride_h, const int32_t* lengths, float* weights, int64_t weights_stride_b, int64_t weights_stride_h,
                           int64_t B, int64_t H, float scale, int32_t dtype, void* workspace, size_t workspace_bytes,
                           void* stream) {
  PagedAttnArgs a = {};
  if (const int rc = paged_cache(cache, "lh_hip_paged_attention", &a.c)) return rc;
  if (B == 0) return LH_OK;
  LH_REQUIRE(out && q && lengths, "lh_hip_paged_attention: null pointer");
  LH_REQUIRE(B >= 0 && H > 0 && H % a.c.heads == 0, "lh_hip_paged_attention: %lld heads are no multiple of %d key / value heads", (long long)H, a.c.heads);
  LH_REQUIRE(paged_batch(B, H), "lh_hip_paged_attention: bad batch (fewer than 2^20 heads of sequences)");
  LH_REQUIRE(dtype == cache->dtype || (cache->dtype == LH_F8E4M3 && (dtype == LH_BF16 || dtype == LH_F16)),
             "lh_hip_paged_attention: queries must have the cache's dtype (bf16 or f16 for a cache of e4m3)");
  LH_REQUIRE(weights == nullptr || ((a.c.heads == 1 || weights_stride_h >= a.c.capacity()) && (B <= 1 || weights_stride_b >= a.c.capacity())),
             "lh_hip_paged_attention: rows of the weights overlap");
  LH_REQUIRE(weights == nullptr || (a.c.capacity() + 255) / 256 * B * a.c.heads < (1ll << 23), "lh_hip_paged_attention: too many weights (fewer than 2^31)");
  const PagedPlan p = paged_plan(a.c, cache->dtype, B, H, weights != nullptr, aligned16(a.c.k) && aligned16(a.c.v));
  LH_REQUIRE(p.total() == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && workspace_bytes >= p.total()),
             "lh_hip_paged_attention: workspace too small or not 256-byte aligned: %zu of %zu bytes", workspace_bytes, p.total());
  a.out = out, a.q = q, a.so_z = out_stride_b, a.so_h = out_stride_h, a.sq_z = q_stride_b, a.sq_h = q_stride_h, a.lengths = lengths;
  a.B = (int32_t)B, a.H = (int32_t)H, a.G = (int32_t)(H / a.c.heads);
  a.rows = p.rows, a.groups = p.groups, a.share = p.share, a.splits = p.splits, a.cap_pad = p.cap_pad;
  a.scale_log2e = (float)((double)scale * a.c.k_scale * 1.4426950408889634);
  char* ws = static_cast<char*>(workspace);
  if (p.splits > 1) a.part_o = reinterpret_cast<float*>(ws), a.part_ml = reinterpret_cast<float2*>(ws + p.o_bytes);
  if (weights) a.scores = reinterpret_cast<float*>(ws + p.o_bytes + p.ml_bytes), a.lse = reinterpret_cast<float*>(ws + p.o_bytes + p.ml_bytes + p.score_bytes);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t sb = weights_stride_b, sh = weights_stride_h;
  if (cache->dtype == LH_F8E4M3)
    return dtype == LH_BF16 ? launch_paged_dp<LH_F8E4M3, LH_BF16>(a, p.dp, p.mode, weights, sb, sh, s)
                            : launch_paged_dp<LH_F8E4M3, LH_F16>(a, p.dp, p.mode, weights, sb, sh, s);
  if (dtype == LH_BF16) return launch_paged_dp<LH_BF16, LH_BF16>(a, p.dp, p.mode, weights, sb, sh, s);
  if (dtype == LH_F16) return launch_paged_dp<LH_F16, LH_F16>(a, p.dp, p.mode, weights, sb, sh, s);
  return launch_paged_dp<LH_F32, LH_F32>(a, p.dp, p.mode, weights, sb, sh, s);
}

}  // extern "C"
