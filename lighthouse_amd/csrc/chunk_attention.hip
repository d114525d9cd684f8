// Attention of packed chunks of new tokens over a paged cache: how a call is cut into workgroups, the join of shares of positions, the
// entry points.  The kernel is in chunk_attention_kernel.hip.
#include <algorithm>
#include <utility>

#include "paged_rows.h"

namespace lh {

// A row of the result whose positions were cut into shares: brings them to the common maximum and adds them, in an order that is always the same.
// WAVES of a workgroup have every WAVES-th share each.
template <int QDT, int WAVES>
__device__ __forceinline__ void chunk_join(const ChunkArgs& a, int n, int head, int b, int start, int count) {
  const int lane = threadIdx.x & 63, wave = WAVES > 1 ? threadIdx.x >> 6 : 0, token = n - start;
  const int hk = head / a.G, row = token * a.G + head % a.G, tile = row >> a.tile_shift;
  const int base = min(max(a.lengths[b], 0), a.c.capacity()) - count;
  const int sees = base + (min(count * a.G, (tile + 1) << a.tile_shift) - 1) / a.G + 1;
  if (sees <= a.share) return;  // (written at once)
  const int parts = (sees + a.share - 1) / a.share;
  const int64_t at = chunk_part_row(a, b, hk, row, n, head) * a.splits;
  // Four at a time, asked for together.
  float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int col = 4 * lane < a.width ? 4 * lane : 0;
  for (int p0 = wave; p0 < parts; p0 += 4 * WAVES) {
    float2 ml[4];
    f32x4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t part = at + min(p0 + i * WAVES, parts - 1);
      ml[i] = a.part_ml[part];
      x[i] = *reinterpret_cast<const f32x4*>(a.part_o + part * a.width + col);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i].x);  // (the last one again where there are fewer)
    const float safe = top == -INFINITY ? 0.0f : top, before = __builtin_amdgcn_exp2f(m - safe);
    l *= before;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= before;
    m = top;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p0 + i * WAVES >= parts) break;
      const float w = __builtin_amdgcn_exp2f(ml[i].x - safe);
      l = __builtin_fmaf(ml[i].y, w, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[i][e], w, o[e]);
    }
  }
  if constexpr (WAVES > 1) {
    __shared__ float2 ml[WAVES];
    __shared__ f32x4 x[WAVES][64];
    if (lane == 0) ml[wave] = make_float2(m, l);
    x[wave][lane] = f32x4{o[0], o[1], o[2], o[3]};
    __syncthreads();
    if (wave > 0) return;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) top = fmaxf(top, ml[i].x);
    const float safe = top == -INFINITY ? 0.0f : top;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      const float w = __builtin_amdgcn_exp2f(ml[i].x - safe);
      l = __builtin_fmaf(ml[i].y, w, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[i][lane][e], w, o[e]);
    }
  }
  const float inv = l == 0.0f ? 0.0f : a.c.v_scale / l;
  const int64_t to = n * a.so_n + head * a.so_h + 4 * lane;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (4 * lane + e < a.c.d) store_from_f32<QDT>(a.out, to + e, o[e] * inv);
}

// few: of the sequences with up to few.most rows.  WAVES: a row's, 1 or all 4 of the workgroup.  ALL: rows of the result one after the other;
// otherwise those that a sequence with few rows may have, since no other's positions were cut.
template <int QDT, int WAVES, bool ALL>
__global__ void __launch_bounds__(256) chunk_join_kernel(ChunkArgs a, ChunkArgs few) {
  const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
  int n, head, b, start, count;
  if constexpr (ALL) {
    n = (int)(row / a.H), head = (int)(row - (int64_t)n * a.H);
    if (n >= chunk_start(a, a.B)) return;
    b = chunk_last(a, n, [&](int i) { return chunk_start(a, i); });
    start = chunk_start(a, b), count = max(chunk_start(a, b + 1) - start, 0);
    if (n < start || n - start >= count) return;
  } else {
    const int item = (int)(row / kChunkFew), at = (int)(row % kChunkFew);
    b = item / a.c.heads;
    if (b >= a.B) return;
    start = chunk_start(a, b), count = max(chunk_start(a, b + 1) - start, 0);
    if (at >= count * a.G || count * a.G > kChunkFew) return;
    n = start + at / a.G, head = (item - b * a.c.heads) * a.G + at % a.G;
  }
  if (ALL && count * a.G > few.most) chunk_join<QDT, WAVES>(a, n, head, b, start, count);
  else chunk_join<QDT, WAVES>(few, n, head, b, start, count);
}

template <int QDT>
static void chunk_join_launch(const ChunkArgs& a, const ChunkArgs& few, hipStream_t s) {
  const int64_t rows = (int64_t)a.N * a.H, few_rows = (int64_t)a.B * a.c.heads * kChunkFew;
  // A wave for up to 8 shares, and where the rows are enough to fill the device (4 drafted tokens after 8188 positions, 32 shares: 24.3 us, with
  // four waves 17.7; 1038 tokens of 16 heads, few of them of 12 shares: 88 us, with four 103).  (Where only the
  // sequences with few rows are cut, their rows are that many, or their shares that few.)
  if (a.splits == 1) LH_LAUNCH((chunk_join_kernel<QDT, 1, false>), dim3((unsigned)((few_rows + 3) / 4)), dim3(256), 0, s, a, few);
  else if ((a.splits <= 8 && few.splits <= 8) || rows > 8 * num_cus()) LH_LAUNCH((chunk_join_kernel<QDT, 1, true>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, few);
  else LH_LAUNCH((chunk_join_kernel<QDT, 4, true>), dim3((unsigned)rows), dim3(256), 0, s, a, few);
}

// ---- host side ------------------------------------------------------------------------------------------------------------

static size_t granules(size_t b) { return (b + 255) / 256 * 256; }

// Which kernel a call is for.  The few read every position once for 16 rows; the many have more to do for a tile of 128, however few rows it has.
// Rows of a sequence up to which the few are faster, all alike (few against many, us): 16-bit types 16 (64 sequences of up to 1024, 12 heads of 64: 16
// rows 32.7, 38.0; 17 rows 46.8, 38.3), e4m3, whose codes are half of the bytes, 64 (16 of up to 4096, 4 heads of 128: 64 rows 35.6, 39.1; 80 rows 45.8,
// 41.8), f32 and wide rows 64 and more (8 of up to 2048, 4 heads of 128, f32: 33, 92; 32 of them, 4 heads of 256, bf16: 105, 136).
//
// Of unlike sequences, those with up to 32 rows are for the few, those with more for the many, in two launches: two pieces of 512 among 14 tokens of 16
// heads take 104 us in the kernel of the many, 87 so; of 32 heads 178 and 142.  But all are for the many where there are fewer than 128 rows a
// sequence, so that they may be alike (8 of 20 rows 31 us, 36 in two launches), where a tile of 128 for each would add less than a quarter to the
// rows that there are, and where there are more tiles than workgroups run at once: single tokens, bound by memory, then run beside the others (8
// pieces of 512 among 56 tokens of 32 heads, up to 4096: 392 us, 410 in two launches; 32 of 256 among 224, up to 1024: 257, 270).
enum ChunkPart { kAllFew, kAllMany, kTheFew, kTheMany };
static ChunkPart chunk_part(const Paged& c, int cache_dtype, int64_t N, int64_t B, int64_t H) {
  const int64_t rows = N * (H / c.heads);
  // Where there is little to do at all, tiles of 128 rows are longer chains.  Tiles of 16 rows times positions up to which the few are faster: f16 and bf16 160
  // Ki (26 tokens up to 681, 6 heads of 256 with 3 queries: few 17, many 31; 100 up to 1000, 8 heads of 64: 10, 15; 4 of 64 up to 1000, 4 heads of 128
  // with 2: 18, 20; 69 of 13 heads of 128 up to 1711: 21, 21), f32, whose matrix instructions take 16 times as long, 4 Mi (4 of 48 to 190, 4 heads of 128 with
  // 3: 15, 42; 16 of 1 to 512 up to 2048, 4 heads of 64 with 4: 104, 114; 8 of 1024, 12 heads of 64: 157, 149), but for wide rows (7 of 70 to 278, 8 heads of
  // 256 with 3: 156, 140).
  const int64_t tiles = (rows + 15) / 16 * c.heads;
  if (tiles * c.capacity() <= (cache_dtype == LH_F32 && c.d <= 128 ? 4 << 20 : 160 << 10)) return kAllFew;
  if (rows <= B * (cache_dtype == LH_F32 || cache_dtype == LH_F8E4M3 || c.d > 192 ? 64 : 16)) return kAllFew;
  return rows < 128 * B || rows >= 4 * 128 * B || (rows / 128 + B) * c.heads > 2 * num_cus() ? kAllMany : kTheMany;
}

// A launch has fewer than 2^32 threads.
constexpr int64_t kMostWorkgroups = (1ll << 32) / 256 - 1;

// Positions of each of `splits` shares of a sequence's, which have no fewer than 256; `items` workgroups take a share each.
static int chunk_share(const Paged& c, int64_t splits, int64_t items) {
  const int64_t most = std::min<int64_t>((c.capacity() + 255) / 256, kMostWorkgroups / items);
  splits = splits > most ? most : splits;
  splits = splits < 1 ? 1 : splits;
  return (int)(((c.capacity() + splits - 1) / splits + kPagedShare - 1) / kPagedShare * kPagedShare);
}

// `mode`: how the kernel of the few loads rows.
static ChunkPlan chunk_plan(const Paged& c, int cache_dtype, int64_t N, int64_t B, int64_t H, PagedMode mode, ChunkPart part) {
  ChunkPlan p = {};
  const int64_t G = H / c.heads;
  p.few = part == kAllFew || part == kTheFew;
  p.least = part == kTheMany ? kChunkFew + 1 : 0, p.most = part == kTheFew ? kChunkFew : 0x7fffffff;
  p.tile_rows = p.few ? 16 : 128;
  // No more sequences than tokens have a tile (but where tiles are found by place, each sequence may have an empty one), and the last tile of each
  // may not be full: `tiles` is how many there probably are.
  const int64_t live = B < N ? B : N, full = N * G / p.tile_rows, some = part == kTheMany ? 1 : live;
  p.slots = (int)(part == kTheFew ? 2 * live : full + (B <= kChunkSums ? live : B));
  const int64_t tiles = part == kTheFew || full < some ? some : full, items = (int64_t)p.slots * c.heads;
  if (p.few) {
    p.mode = mode;
    p.width = paged_width(c.d);
    // As many shares of positions as the workgroups that run at once allow for (4 drafted tokens of 8 sequences of up to 4096 positions, 64 tiles:
    // 4 shares 36.3 us, 8 34.0, 12 31.9, 16 36.9; 128 tiles: 4 53.5, 6 48.9, 8 50.8), of no fewer than 256 positions.
    const int per_cu = paged_occupancy(cache_dtype, p.width, p.mode, true);
    p.share = chunk_share(c, (per_cu < 3 ? per_cu : 3) * (int64_t)num_cus() / (tiles * c.heads), items);
  } else {
    p.odd = c.d % (cache_dtype == LH_F32 ? 4 : 8) != 0;
    const int blocks = (c.d + 31) / 32;
    p.blocks = p.odd ? (blocks <= 2 ? 2 : blocks <= 4 ? 4 : 8) : blocks <= 2 ? 2 : blocks <= 4 ? blocks : blocks <= 6 ? 6 : 8;
    p.width = 32 * p.blocks;
    // One share more than that would be a second round of workgroups for a few (a piece of 256 tokens after 16128 positions, 64 tiles: 6 shares
    // 138 us, 8 118, 12 127; of wide rows, of which a CU holds one workgroup, after 7936 positions, 32 tiles: 8 shares 112, 16 127).  But in three
    // shares each, tiles that leave a last round of workgroups mostly empty take a third of it, where a share is long against what its results cost (4
    // pieces of 600 up to 8192, 300 tiles: 323 us, so 238; one of 2300 up to 16384, 568 tiles: 1111, 910; 320 tiles of 64 columns up to 4096: 111, 81, up
    // to 1024: 30, 41).
    const int64_t at_once = (p.blocks > 4 ? 1 : 2) * (int64_t)num_cus(), workgroups = tiles * c.heads;
    const int64_t whole = (workgroups + at_once - 1) / at_once, cut = (3 * workgroups + at_once - 1) / at_once;  // rounds, and thirds of rounds
    const bool thirds = 2 * workgroups > at_once && whole <= 3 && 10 * cut <= 25 * whole && (int64_t)c.capacity() * p.width >= whole << 18;
    p.share = chunk_share(c, thirds ? 3 : at_once / workgroups, items);
  }
  p.splits = (int)(((int64_t)c.capacity() + p.share - 1) / p.share);
  if (p.splits > 1) {
    const size_t rows = (size_t)(part == kTheFew ? B * c.heads * kChunkFew : N * H) * p.splits;
    p.o_bytes = granules(rows * p.width * 4);
    p.ml_bytes = granules(rows * 8);
  }
  return p;
}

static bool chunk_sizes(const Paged& c, int64_t N, int64_t B, int64_t H) {
  return N > 0 && B > 0 && H > 0 && B < (1ll << 20) && N < (1ll << 30) && H < (1ll << 20) && H % c.heads == 0 && N * (H / c.heads) < (1ll << 31) - 256 &&
         N * H < (1ll << 32) && (N * (H / c.heads) / 16 + B) * c.heads < (1ll << 30);
}

}  // namespace lh

using namespace lh;

extern "C" {

size_t lh_hip_paged_attention_chunk_workspace_bytes(const lh_paged_cache* cache, int64_t N, int64_t B, int64_t H) {
  Paged c;
  if (paged_cache(cache, "lh_hip_paged_attention_chunk_workspace_bytes", &c) != LH_OK || !chunk_sizes(c, N, B, H)) return 0;
  // (Room for every way to load rows: a caller may size it with one cache and pass a view of another, of other strides or alignment.)
  const ChunkPart part = chunk_part(c, cache->dtype, N, B, H);
  size_t bytes = 0;
  for (PagedMode mode : {kTiles, kWholeRows, kOddRows}) {
    size_t sum = chunk_plan(c, cache->dtype, N, B, H, mode, part).total();
    if (part == kTheMany) sum += chunk_plan(c, cache->dtype, N, B, H, mode, kTheFew).total();
    bytes = sum > bytes ? sum : bytes;
  }
  return bytes;
}

int lh_hip_paged_attention_chunk(const lh_paged_cache* cache, void* out, const void* q, int64_t out_stride_n, int64_t out_stride_h, int64_t q_stride_n,
                                 int64_t q_stride_h, const int32_t* lengths, const int32_t* starts, int64_t N, int64_t B, int64_t H, float scale,
                                 int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "lh_hip_paged_attention_chunk";
  ChunkArgs a = {};
  if (const int rc = paged_cache(cache, what, &a.c)) return rc;
  if (N == 0 || B == 0) return LH_OK;
  LH_REQUIRE(H > 0 && H % a.c.heads == 0, "%s: %lld heads are no multiple of %d key / value heads", what, (long long)H, a.c.heads);
  LH_REQUIRE(chunk_sizes(a.c, N, B, H), "%s: bad sizes (fewer than 2^20 sequences, 2^30 rows, 2^32 rows of heads)", what);
  LH_REQUIRE(out && q && lengths && starts, "%s: null pointer", what);
  LH_REQUIRE(dtype == cache->dtype || (cache->dtype == LH_F8E4M3 && (dtype == LH_BF16 || dtype == LH_F16)),
             "%s: queries must have the cache's dtype (bf16 or f16 for a cache of e4m3)", what);
  const PagedMode mode = (PagedMode)paged_mode(a.c, (int)dtype_size(cache->dtype), aligned16(a.c.k) && aligned16(a.c.v));
  const ChunkPart part = chunk_part(a.c, cache->dtype, N, B, H);
  const ChunkPlan p = chunk_plan(a.c, cache->dtype, N, B, H, mode, part);
  ChunkPlan f = {};
  if (part == kTheMany) f = chunk_plan(a.c, cache->dtype, N, B, H, mode, kTheFew);
  for (const ChunkPlan* plan : {&std::as_const(p), &std::as_const(f)})
    LH_REQUIRE((int64_t)plan->slots * a.c.heads <= kMostWorkgroups / (plan->splits > 1 ? plan->splits : 1),
               "%s: too many rows and heads for one launch (%lld workgroups, at most 2^24 - 1)", what, (long long)plan->slots * a.c.heads);
  const size_t need = p.total() + f.total();
  LH_REQUIRE(need == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && workspace_bytes >= need),
             "%s: workspace too small or not 256-byte aligned: %zu of %zu bytes", what, workspace_bytes, need);
  a.out = out, a.q = q, a.so_n = out_stride_n, a.so_h = out_stride_h, a.sq_n = q_stride_n, a.sq_h = q_stride_h, a.lengths = lengths, a.starts = starts;
  a.N = (int32_t)N, a.B = (int32_t)B, a.H = (int32_t)H, a.G = (int32_t)(H / a.c.heads), a.by_group = FastDiv((uint32_t)a.G), a.ranked = B > 1 && B <= 32;
  const double factor = (double)scale * a.c.k_scale * 1.4426950408889634;
  a.scale_log2e = scale == 0.0f ? 1.0f : (float)(factor < 0.0 ? -factor : factor);
  a.q_and = scale == 0.0f ? 0u : ~0u, a.q_xor = scale < 0.0f ? (dtype == LH_F32 ? 0x80000000u : 0x80008000u) : 0u;
  LH_REQUIRE(a.scale_log2e > 0.0f && a.scale_log2e < INFINITY, "%s: scale times the keys' scale must be finite", what);
  auto planned = [&](const ChunkPlan& plan, char* space) {
    ChunkArgs x = a;
    x.least = plan.least, x.most = plan.most, x.tile_rows = plan.tile_rows, x.tile_shift = plan.few ? 4 : 7, x.slots = plan.slots;
    x.share = plan.share, x.splits = plan.splits, x.width = plan.width;
    if (plan.splits > 1) x.part_o = reinterpret_cast<float*>(space), x.part_ml = reinterpret_cast<float2*>(space + plan.o_bytes);
    return x;
  };
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  auto launch = [&](const ChunkArgs& x, const ChunkPlan& plan) {
    const auto kernel = cache->dtype == LH_F32    ? (plan.few ? chunk_few_f32 : chunk_many_f32)
                        : cache->dtype == LH_BF16 ? (plan.few ? chunk_few_bf16 : chunk_many_bf16)
                        : cache->dtype == LH_F16  ? (plan.few ? chunk_few_f16 : chunk_many_f16)
                        : dtype == LH_BF16        ? (plan.few ? chunk_few_e4m3_bf16 : chunk_many_e4m3_bf16)
                                                  : (plan.few ? chunk_few_e4m3_f16 : chunk_many_e4m3_f16);
    return kernel(x, plan, s);
  };
  const ChunkArgs main = planned(p, static_cast<char*>(workspace)), few = part == kTheMany ? planned(f, static_cast<char*>(workspace) + p.total()) : main;
  if (const int rc = launch(main, p)) return rc;
  if (part == kTheMany)
    if (const int rc = launch(few, f)) return rc;
  if (need == 0) return LH_OK;
  if (dtype == LH_BF16) chunk_join_launch<LH_BF16>(main, few, s);
  else if (dtype == LH_F16) chunk_join_launch<LH_F16>(main, few, s);
  else chunk_join_launch<LH_F32>(main, few, s);
  return check_launch("chunk_join");
}

}  // extern "C"
