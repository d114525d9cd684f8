// Filling a paged key / value cache and dropping from it the positions that got least attention.  Both move bytes: what
// bounds them is memory, or, for a step of one token per sequence, the launch.
#include "paged.h"

namespace lh {

int paged_cache(const lh_paged_cache* c, const char* what, Paged* out) {
  LH_REQUIRE(c != nullptr, "%s: cache is null", what);
  LH_REQUIRE(c->k && c->v && c->block_table, "%s: null pointer in the cache", what);
  LH_REQUIRE(c->dtype == LH_F32 || c->dtype == LH_BF16 || c->dtype == LH_F16 || c->dtype == LH_F8E4M3,
             "%s: unsupported cache dtype %d", what, c->dtype);
  LH_REQUIRE(c->n_pages > 0 && c->n_pages < (1ll << 31) && c->page_size > 0 && c->page_size < (1ll << 31) &&
                 c->max_pages > 0 && c->max_pages < (1ll << 31) && c->max_pages * c->page_size < (1ll << 31) - 65536,
             "%s: bad page counts (%lld pages of %lld, table of %lld)", what, (long long)c->n_pages,
             (long long)c->page_size, (long long)c->max_pages);
  LH_REQUIRE(c->n_kv_heads > 0 && c->n_kv_heads < 65536 && c->d >= 1 && c->d <= 256, "%s: bad head count %lld or head dimension %lld (1 to 256)",
             what, (long long)c->n_kv_heads, (long long)c->d);
  LH_REQUIRE(c->table_stride >= c->max_pages, "%s: rows of the block table overlap", what);
  for (const lh_strides3* s : {&c->sk, &c->sv})
    LH_REQUIRE((c->page_size == 1 || s->t >= c->d) && (c->n_kv_heads == 1 || s->h >= c->d) && (c->n_pages == 1 || s->z >= c->d),
               "%s: rows of the cache overlap", what);
  LH_REQUIRE(c->k_scale > 0.0f && c->k_scale < INFINITY && c->v_scale > 0.0f && c->v_scale < INFINITY,
             "%s: the scales of the cache must be positive numbers", what);
  *out = Paged{c->k, c->v, c->block_table, c->table_stride, c->sk, c->sv, (int32_t)c->n_pages, (int32_t)c->max_pages,
               (int32_t)c->page_size, (int32_t)c->n_kv_heads, (int32_t)c->d, c->k_scale, c->v_scale,
               FastDiv((uint32_t)c->page_size)};
  return LH_OK;
}

// ---------------------------------------------------------------------------------------------------- append

// (By value: a bit cast of a vector's element itself reads its first one.)
__device__ __forceinline__ float bits_to_f32(uint32_t u) { return __builtin_bit_cast(float, u); }

struct AppendArgs {
  Paged c;
  const void* k;
  const void* v;
  lh_strides3 sk, sv;  // batch, head, token
  const int32_t* positions;
  const int32_t* counts;  // or null: every token counts
  int32_t B, T;
  int32_t per_token;        // chunks of a token's keys and values
  int32_t tokens_per_block;
  FastDiv by_token, by_T, by_chunks, by_heads;
};

// Two floats -> two e4m3 codes in the low half of a word: clamped to the largest finite value, rounded to nearest even;
// a NaN stays one (a comparison keeps it, fmin and fmax would not).
__device__ __forceinline__ float e4m3_clamp(float x) {
  x = x > 448.0f ? 448.0f : x;
  return x < -448.0f ? -448.0f : x;
}
__device__ __forceinline__ uint32_t e4m3_pack2(float a, float b) {
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_clamp(a), e4m3_clamp(b), 0, false) & 0xffffu;
}

// A thread takes one chunk (16 bytes of the source; 8 elements for a cache of 8 bits) of one head's key or value of one
// token; a token's chunks are neighbours, so that both sides are read and written in whole lines whatever the
// layout of heads and tokens.  Any strides and alignment: gfx9 global memory takes 16 bytes at element alignment, the end of
// a row that is no whole chunk goes element by element.
template <int SDT, int CDT>
__global__ void __launch_bounds__(256) kv_append_kernel(AppendArgs a) {
  constexpr int E = SDT == LH_F32 && CDT == LH_F32 ? 4 : 8;
  constexpr int SES = SDT == LH_F32 ? 4 : 2, CES = CDT == LH_F32 ? 4 : CDT == LH_F8E4M3 ? 1 : 2;
  typedef typename Chunk<SES>::type src16;
  const int items = a.per_token * a.tokens_per_block;
  for (int i = threadIdx.x; i < items; i += 256) {
    const int in_block = (int)a.by_token.div(i);
    const int64_t token = (int64_t)blockIdx.x * a.tokens_per_block + in_block;
    if (token >= (int64_t)a.B * a.T) return;
    const int b = (int)a.by_T.div((uint32_t)token), t = (int)token - b * a.T;
    if (a.counts != nullptr && t >= a.counts[b]) continue;
    const int64_t at = (int64_t)a.positions[b] + t;
    if (at < 0 || at >= a.c.capacity()) continue;
    int slot;
    const int page = a.c.page_of(b, (int)at, &slot);
    if (page < 0) continue;
    const int rest = i - in_block * a.per_token;  // [k or v][head][chunk]
    const int row = (int)a.by_chunks.div(rest), col = (rest - row * (int)a.by_chunks.d) * E;
    const bool is_v = row >= a.c.heads;
    const int h = row - (is_v ? a.c.heads : 0);
    const lh_strides3 ss = is_v ? a.sv : a.sk, cs = is_v ? a.c.sv : a.c.sk;
    const uint8_t* src = static_cast<const uint8_t*>(is_v ? a.v : a.k) + (b * ss.z + h * ss.h + t * ss.t + col) * SES;
    uint8_t* dst = static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + (page * cs.z + h * cs.h + slot * cs.t + col) * CES;
    const int n = min(E, a.c.d - col);
    if constexpr (CDT != LH_F8E4M3) {
      if (n == E) {
        *reinterpret_cast<src16*>(dst) = *reinterpret_cast<const src16*>(src);
      } else {
        for (int e = 0; e < n; ++e) {
          if constexpr (SES == 4) reinterpret_cast<uint32_t*>(dst)[e] = reinterpret_cast<const uint32_t*>(src)[e];
          else reinterpret_cast<uint16_t*>(dst)[e] = reinterpret_cast<const uint16_t*>(src)[e];
        }
      }
    } else {
      // x / scale in f32 (a true division: the codes are those of the formula, not of a rounded reciprocal).
      const float scale = is_v ? a.c.v_scale : a.c.k_scale;
      float x[E];
      if (n == E) {
        if constexpr (SES == 2) {
          const src16 w = *reinterpret_cast<const src16*>(src);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[2 * e] = unpack_lo<SDT>(w[e]), x[2 * e + 1] = unpack_hi<SDT>(w[e]);
        } else {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const src16 w = reinterpret_cast<const src16*>(src)[p];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[4 * p + e] = bits_to_f32(w[e]);
          }
        }
        typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
        u32x2_any o;
#pragma unroll
        for (int p = 0; p < 2; ++p)
          o[p] = e4m3_pack2(x[4 * p] / scale, x[4 * p + 1] / scale) | e4m3_pack2(x[4 * p + 2] / scale, x[4 * p + 3] / scale) << 16;
        *reinterpret_cast<u32x2_any*>(dst) = o;
      } else {
        for (int e = 0; e < n; ++e) dst[e] = (uint8_t)e4m3_pack2(load_as_f32<SDT>(src, e) / scale, 0.0f);
      }
    }
  }
}

// ----------------------------------------------------------------------------------------------------- evict

struct EvictArgs {
  Paged c;
  float* weights;  // [B, heads, capacity]
  int64_t sw_b, sw_h;
  const int32_t* lengths;
  int32_t* new_lengths;
  int32_t* kept;  // [B * heads][budget]
  int32_t* held;  // [B * heads]: the length before
  int32_t B, budget, recent;
  int32_t elem_bytes;
  int32_t slices;  // column slices of a row of keys (and of values)
};

__device__ __forceinline__ int evict_length(const EvictArgs& a, int b) { return min(max(a.lengths[b], 0), a.c.capacity()); }

// An order of the weights as unsigned numbers: larger weight, larger number; -0 and 0 alike, a NaN below everything.
__device__ __forceinline__ uint32_t evict_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64;
constexpr int kEvictBins = 2048;  // 11 bits of the key a pass

// Which positions of one head of one sequence stay, in order.  The (budget - recent)-th largest key among the positions that
// are not recent is found by its digits, 11, 11 and 10 bits, from counts in LDS; of the positions that share it the lowest stay.
// Then each wave goes through a contiguous share of the positions: it knows from the shares before it how many
// stay in front, and counts on by ballots.
__global__ void __launch_bounds__(kEvictThreads) kv_evict_select(EvictArgs a) {
  __shared__ uint32_t bins[kEvictBins];
  __shared__ uint32_t wave_sum[kEvictWaves], wave_ties[kEvictWaves];
  __shared__ uint32_t found[2];  // digit, how many of the digit's keys stay
  const int b = blockIdx.x / a.c.heads, h = blockIdx.x % a.c.heads;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = evict_length(a, b);
  if (tid == 0) a.held[blockIdx.x] = n;
  if (n <= a.budget) return;
  const float* w = a.weights + b * a.sw_b + h * a.sw_h;
  const int old = n - a.recent;             // positions that compete
  uint32_t want = a.budget - a.recent;      // of them stay; below `old`
  uint32_t prefix = 0, threshold = 0xffffffffu;
  if (want > 0) {
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < kEvictBins; i += kEvictThreads) bins[i] = 0;
      __syncthreads();
      for (int t = tid; t < old; t += kEvictThreads) {
        const uint32_t key = evict_key(w[t]);
        if (pass == 0 || key >> (shift + bits) == prefix) atomicAdd(&bins[(key >> shift) & ((1u << bits) - 1)], 1u);
      }
      __syncthreads();
      // The digit in which the want-th key from above lies: thread i has the bins 2 i and 2 i + 1 of the order from above.
      const uint32_t c0 = bins[kEvictBins - 1 - 2 * tid], c1 = bins[kEvictBins - 2 - 2 * tid];
      uint32_t s = c0 + c1;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(s, o);
        if (lane >= o) s += up;
      }
      if (lane == 63) wave_sum[wave] = s;
      __syncthreads();
      uint32_t before = s - c0 - c1;
      for (int i = 0; i < wave; ++i) before += wave_sum[i];
      if (before < want && want <= before + c0) found[0] = kEvictBins - 1 - 2 * tid, found[1] = want - before;
      else if (before + c0 < want && want <= before + c0 + c1) found[0] = kEvictBins - 2 - 2 * tid, found[1] = want - before - c0;
      __syncthreads();
      prefix = prefix << bits | found[0];
      want = found[1];
      __syncthreads();
    }
    threshold = prefix;  // the want lowest positions of those with this key stay
  }
  // Shares of the positions, whole multiples of 64.
  const int share = ((n + 63) / 64 + kEvictWaves - 1) / kEvictWaves * 64;
  const int begin = wave * share, end = min(begin + share, n);
  uint32_t above = 0, ties = 0;
  for (int t0 = begin; t0 < end; t0 += 64) {
    const int t = t0 + lane;
    const uint32_t key = t < old ? evict_key(w[t]) : 0;
    above += __popcll(__ballot(t < n && (t >= old || (want > 0 && key > threshold))));
    ties += __popcll(__ballot(t < old && want > 0 && key == threshold));
  }
  if (lane == 0) wave_sum[wave] = above, wave_ties[wave] = ties;
  __syncthreads();
  uint32_t at = 0, tied = 0;
  for (int i = 0; i < wave; ++i) at += wave_sum[i], tied += wave_ties[i];
  at += min(tied, want);
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
  const uint64_t below = (1ull << lane) - 1;
  for (int t0 = begin; t0 < end; t0 += 64) {
    const int t = t0 + lane;
    const uint32_t key = t < old ? evict_key(w[t]) : 0;
    const uint64_t tie = __ballot(t < old && want > 0 && key == threshold);
    const bool stays = t < n && (t >= old || (want > 0 && (key > threshold || (key == threshold && tied + __popcll(tie & below) < want))));
    const uint64_t stay = __ballot(stays);
    if (stays) kept[at + __popcll(stay & below)] = t;
    at += __popcll(stay);
    tied += __popcll(tie);
  }
}

// Rows move up, row kept[j] to row j: kept[j] >= j, so what a block of rows j .. j + R - 1 overwrites no later block reads,
// and within the block every row is in registers before any is written.  A workgroup takes a column slice of 128 bytes
// of the keys or the values of a head, or its weights: slices know nothing of each other.
constexpr int kMoveThreads = 1024;
constexpr int kMoveRows = 4;  // of a thread, in flight at once

__global__ void __launch_bounds__(kMoveThreads) kv_evict_move(EvictArgs a) {
  const int per_head = 1 + 2 * a.slices;
  const int bh = blockIdx.x / per_head, what = blockIdx.x % per_head;
  const int b = bh / a.c.heads, h = bh % a.c.heads;
  // (`lengths` itself is not read here: the new lengths may be written over it.)
  const int n = a.held[bh], tid = threadIdx.x;
  if (what == 0 && h == 0 && tid == 0) a.new_lengths[b] = min(n, a.budget);
  if (n <= a.budget) return;
  const int32_t* kept = a.kept + (int64_t)bh * a.budget;
  if (what == 0) {
    float* w = a.weights + b * a.sw_b + h * a.sw_h;
    for (int j0 = 0; j0 < a.budget; j0 += kMoveThreads) {
      const int j = j0 + tid;
      float x = j < a.budget ? w[kept[j]] : 0.0f;
      asm volatile("" : "+v"(x));  // in a register before anybody writes
      __syncthreads();
      if (j < a.budget) w[j] = x;
    }
    __syncthreads();
    for (int t = a.budget + tid; t < n; t += kMoveThreads) w[t] = 0.0f;
    return;
  }
  const bool is_v = what > a.slices;
  const int slice = (what - 1) % a.slices;
  const lh_strides3 cs = is_v ? a.c.sv : a.c.sk;
  const int es = a.elem_bytes, row_bytes = a.c.d * es;
  uint8_t* base = static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + h * cs.h * es;
  typedef typename Chunk<1>::type any16;
  const int col = slice * 128 + (tid & 7) * 16;  // 8 threads a row
  const int bytes = min(16, row_bytes - col);    // (none, or less than a chunk, where the row ends)
  constexpr int kRows = kMoveThreads / 8;
  auto row = [&](int t) -> uint8_t* {
    int slot;
    const int page = a.c.page_of(b, t, &slot);
    return page < 0 ? nullptr : base + (page * cs.z + slot * cs.t) * es + col;
  };
  for (int j0 = 0; j0 < a.budget; j0 += kRows * kMoveRows) {
    any16 x[kMoveRows];
    uint8_t* to[kMoveRows];
#pragma unroll
    for (int r = 0; r < kMoveRows; ++r) {
      const int j = j0 + r * kRows + (tid >> 3);
      to[r] = nullptr;
      x[r] = any16{0u, 0u, 0u, 0u};
      if (j >= a.budget || bytes <= 0) continue;
      const int from = kept[j];
      if (from == j) continue;
      const uint8_t* src = row(from);
      if (src == nullptr) continue;
      to[r] = row(j);
      if (bytes == 16) {
        x[r] = *reinterpret_cast<const any16*>(src);
      } else {
        uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (e < bytes) words[e >> 2] |= (uint32_t)src[e] << (8 * (e & 3));
        x[r] = any16{words[0], words[1], words[2], words[3]};
      }
    }
#pragma unroll
    for (int r = 0; r < kMoveRows; ++r)
      asm volatile("" : "+v"(x[r][0]), "+v"(x[r][1]), "+v"(x[r][2]), "+v"(x[r][3]));
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kMoveRows; ++r) {
      if (to[r] == nullptr) continue;
      if (bytes == 16) {
        *reinterpret_cast<any16*>(to[r]) = x[r];
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (e < bytes) to[r][e] = (uint8_t)(x[r][e >> 2] >> (8 * (e & 3)));
      }
    }
  }
}

template <int SDT, int CDT>
static int append_launch(const AppendArgs& a, unsigned blocks, hipStream_t s) {
  LH_LAUNCH((kv_append_kernel<SDT, CDT>), dim3(blocks), dim3(256), 0, s, a);
  return check_launch("kv_append");
}

}  // namespace lh

using namespace lh;

extern "C" {

int lh_hip_kv_append(const lh_paged_cache* cache, const void* k, const void* v, int64_t k_stride_b, int64_t k_stride_h,
                     int64_t k_stride_t, int64_t v_stride_b, int64_t v_stride_h, int64_t v_stride_t, const int32_t* positions,
                     const int32_t* counts, int64_t B, int64_t T, int32_t dtype, void* stream) {
  AppendArgs a = {};
  if (const int rc = paged_cache(cache, "lh_hip_kv_append", &a.c)) return rc;
  LH_REQUIRE(k && v && positions, "lh_hip_kv_append: null pointer");
  LH_REQUIRE(B >= 0 && T >= 0 && B < (1ll << 24) && T < (1ll << 24) && B * T < (1ll << 24), "lh_hip_kv_append: bad shape (at most 2^24 tokens)");
  LH_REQUIRE(dtype == LH_F32 || dtype == LH_BF16 || dtype == LH_F16, "lh_hip_kv_append: unsupported dtype %d", dtype);
  LH_REQUIRE(dtype == cache->dtype || cache->dtype == LH_F8E4M3,
             "lh_hip_kv_append: keys and values must have the cache's dtype (any of 16 or 32 bits for a cache of e4m3)");
  if (B == 0 || T == 0) return LH_OK;
  a.k = k, a.v = v, a.sk = {k_stride_b, k_stride_h, k_stride_t}, a.sv = {v_stride_b, v_stride_h, v_stride_t}, a.positions = positions, a.counts = counts;
  a.B = (int32_t)B, a.T = (int32_t)T;
  const int e = dtype == LH_F32 && cache->dtype == LH_F32 ? 4 : 8, chunks = (a.c.d + e - 1) / e;
  a.per_token = 2 * a.c.heads * chunks;
  a.tokens_per_block = a.per_token < 256 ? 256 / a.per_token : 1;
  a.by_token = FastDiv((uint32_t)a.per_token), a.by_T = FastDiv((uint32_t)T), a.by_chunks = FastDiv((uint32_t)chunks);
  const unsigned blocks = (unsigned)((B * T + a.tokens_per_block - 1) / a.tokens_per_block);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache->dtype == LH_F8E4M3) {
    if (dtype == LH_BF16) return append_launch<LH_BF16, LH_F8E4M3>(a, blocks, s);
    if (dtype == LH_F16) return append_launch<LH_F16, LH_F8E4M3>(a, blocks, s);
    return append_launch<LH_F32, LH_F8E4M3>(a, blocks, s);
  }
  if (dtype == LH_F32) return append_launch<LH_F32, LH_F32>(a, blocks, s);
  return append_launch<LH_BF16, LH_BF16>(a, blocks, s);  // (16 bits either way: they are only moved)
}

size_t lh_hip_kv_evict_workspace_bytes(int64_t B, int64_t n_kv_heads, int64_t budget) {
  if (B <= 0 || n_kv_heads <= 0 || budget <= 0) return 0;
  return ((size_t)B * n_kv_heads * (budget + 1) * 4 + 255) / 256 * 256;
}

int lh_hip_kv_evict(const lh_paged_cache* cache, float* weights, int64_t weights_stride_b, int64_t weights_stride_h,
                    const int32_t* lengths, int32_t* new_lengths, int64_t B, int64_t budget, int64_t recent,
                    void* workspace, size_t workspace_bytes, void* stream) {
  EvictArgs a = {};
  if (const int rc = paged_cache(cache, "lh_hip_kv_evict", &a.c)) return rc;
  LH_REQUIRE(weights && lengths && new_lengths, "lh_hip_kv_evict: null pointer");
  LH_REQUIRE(budget >= 1 && recent >= 0 && recent <= budget, "lh_hip_kv_evict: budget must be at least 1, recent between 0 and the budget");
  LH_REQUIRE(B >= 0 && B < (1ll << 20) && B * a.c.heads < (1ll << 16), "lh_hip_kv_evict: bad batch (fewer than 2^16 heads of sequences)");
  LH_REQUIRE((a.c.heads == 1 || weights_stride_h >= a.c.capacity()) && (B <= 1 || weights_stride_b >= a.c.capacity()),
             "lh_hip_kv_evict: rows of the weights overlap");
  if (B == 0) return LH_OK;
  if (budget > a.c.capacity()) budget = a.c.capacity();  // nothing is longer: nothing goes
  if (recent > budget) recent = budget;
  const size_t need = lh_hip_kv_evict_workspace_bytes(B, a.c.heads, budget);
  LH_REQUIRE(workspace != nullptr && workspace_bytes >= need, "lh_hip_kv_evict: workspace too small: %zu of %zu bytes", workspace_bytes, need);
  a.weights = weights, a.sw_b = weights_stride_b, a.sw_h = weights_stride_h;
  a.lengths = lengths, a.new_lengths = new_lengths, a.kept = static_cast<int32_t*>(workspace);
  a.held = a.kept + B * a.c.heads * budget;
  a.B = (int32_t)B, a.budget = (int32_t)budget, a.recent = (int32_t)recent;
  a.elem_bytes = (int32_t)dtype_size(cache->dtype);
  a.slices = (a.c.d * a.elem_bytes + 127) / 128;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  LH_LAUNCH(kv_evict_select, dim3((unsigned)(B * a.c.heads)), dim3(kEvictThreads), 0, s, a);
  if (const int rc = check_launch("kv_evict_select")) return rc;
  LH_LAUNCH(kv_evict_move, dim3((unsigned)(B * a.c.heads * (1 + 2 * a.slices))), dim3(kMoveThreads), 0, s, a);
  return check_launch("kv_evict_move");
}

}  // extern "C"
