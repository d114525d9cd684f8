// Filling a paged key / value cache and dropping from it the positions that got least attention.  Both move bytes: what
// bounds them is memory, or, for a step of one token per sequence, the launch.
#include <cstring>

#include "paged.h"
#include "wave_scan.h"

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
  int32_t T;
  int32_t per_token;      // chunks of a token's keys and values
  int32_t parts;          // workgroups that share them
  int32_t tokens;         // of a sequence that a workgroup takes
  int32_t token_blocks;   // workgroups for T tokens
  FastDiv by_chunks;
  float k_inv, v_inv;     // 1 / scale, rounded, or 0 where the short division does not apply
};

// Two floats, no larger than 448, -> two e4m3 codes in the low half of a word, rounded to nearest even; a NaN stays one.
__device__ __forceinline__ uint32_t e4m3_pack2(float a, float b) { return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu; }
// (Comparisons keep a NaN, fmin and fmax would not.)
__device__ __forceinline__ float e4m3_clamp(float x) {
  x = x > 448.0f ? 448.0f : x;
  return x < -448.0f ? -448.0f : x;
}
// Eight numbers x -> x / scale, clamped to +-448: the quotient that a division rounds, so that the codes are those of the formula and
// not of a rounded reciprocal.  With inv = 1 / scale rounded, q = x inv and r = q scale - x (exact), q - r inv is that quotient
// (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990), but for a
// scale whose mantissa is all ones, and where x or r leaves the normal range: the host passes inv = 0 for scales
// that are not between 2^-60 and 2^60, whose quotients that are not 0 in e4m3 are far from it, and numbers that are not finite
// or far above 448 take the division.  (3 instructions instead of 11: 8 prompts of 1024 tokens, 12 heads of 64, 15.9 -> 11.4 us.)
__device__ __forceinline__ void e4m3_divide(float* x, float scale, float inv) {
  float size = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) size += fabsf(x[e]);
  if (inv != 0.0f && size <= 4096.0f * scale) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float q = x[e] * inv, r = __builtin_fmaf(q, scale, -x[e]);
      x[e] = __builtin_amdgcn_fmed3f(__builtin_fmaf(-r, inv, q), -448.0f, 448.0f);
    }
  } else {
#pragma unroll 1
    for (int e = 0; e < 8; ++e) x[e] = e4m3_clamp(x[e] / scale);
  }
}

// A thread takes one chunk (16 bytes of the source; 8 elements for a cache of 8 bits) of one head's key or value, of several
// tokens of a sequence one after the other, four at a time; a token's chunks are neighbours, so that both sides are read and
// written in whole lines whatever the layout of heads and tokens.  The slot of a token is the same for the workgroup: the scalar
// unit finds it.  Eight prompts of up to 1024 tokens, 12 heads of 64, bf16 into a cache of 8 bits: 12 us from memory, 9 from
// the caches (with a token per workgroup and the slot found by every thread 13.4); one token for each of 64 sequences: 4 us, a launch.  Any
// strides and alignment: gfx9 global memory takes 16 bytes at element alignment, the end of a row that is no whole chunk goes element by element.
template <int SDT, int CDT>
__global__ void __launch_bounds__(256) kv_append_kernel(AppendArgs a) {
  constexpr int E = SDT == LH_F32 && CDT == LH_F32 ? 4 : 8;
  constexpr int SES = SDT == LH_F32 ? 4 : 2, CES = CDT == LH_F32 ? 4 : CDT == LH_F8E4M3 ? 1 : 2;
  constexpr int LOADS = E * SES / 16, BATCH = 4;
  typedef typename Chunk<SES>::type src16;
  const int part = blockIdx.x % a.parts, rest = blockIdx.x / a.parts;
  const int b = rest / a.token_blocks, t0 = (rest - b * a.token_blocks) * a.tokens;
  const int i = part * blockDim.x + threadIdx.x;
  if (i >= a.per_token) return;
  const int row = (int)a.by_chunks.div(i), col = (i - row * (int)a.by_chunks.d) * E;
  const bool is_v = row >= a.c.heads;
  const int h = row - (is_v ? a.c.heads : 0);
  const lh_strides3 ss = is_v ? a.sv : a.sk, cs = is_v ? a.c.sv : a.c.sk;
  const uint8_t* src = static_cast<const uint8_t*>(is_v ? a.v : a.k) + (b * ss.z + h * ss.h + col) * SES;
  uint8_t* dst = static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + (h * cs.h + col) * CES;
  const int n = min(E, a.c.d - col);
  const float scale = is_v ? a.c.v_scale : a.c.k_scale, inv = is_v ? a.v_inv : a.k_inv;
  const int t_end = min(t0 + a.tokens, a.counts == nullptr ? a.T : min(a.T, a.counts[b]));
  const int64_t position = a.positions[b];
#pragma unroll 1
  for (int t1 = t0; t1 < t_end; t1 += BATCH) {
    int page[BATCH], slot[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int64_t at = position + t1 + u;
      page[u] = -1, slot[u] = 0;
      if (t1 + u < t_end && at >= 0 && at < a.c.capacity()) page[u] = a.c.page_of(b, (int)at, &slot[u]);
    }
    if (n == E) {
      src16 w[BATCH][LOADS];
#pragma unroll
      for (int u = 0; u < BATCH; ++u)
        if (page[u] >= 0)
#pragma unroll
          for (int l = 0; l < LOADS; ++l) w[u][l] = reinterpret_cast<const src16*>(src + (int64_t)(t1 + u) * ss.t * SES)[l];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) {
        if (page[u] < 0) continue;
        uint8_t* to = dst + (page[u] * cs.z + slot[u] * cs.t) * CES;
        if constexpr (CDT != LH_F8E4M3) {
          *reinterpret_cast<src16*>(to) = w[u][0];
        } else {
          float x[E];
#pragma unroll
          for (int l = 0; l < LOADS; ++l)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (SES == 2) x[2 * e] = unpack_lo<SDT>(w[u][l][e]), x[2 * e + 1] = unpack_hi<SDT>(w[u][l][e]);
              else x[4 * l + e] = bits_to_f32(w[u][l][e]);
            }
          typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
          e4m3_divide(x, scale, inv);
          u32x2_any o;
#pragma unroll
          for (int p = 0; p < 2; ++p) o[p] = e4m3_pack2(x[4 * p], x[4 * p + 1]) | e4m3_pack2(x[4 * p + 2], x[4 * p + 3]) << 16;
          *reinterpret_cast<u32x2_any*>(to) = o;
        }
      }
    } else {
#pragma unroll 1
      for (int u = 0; u < BATCH; ++u) {
        if (page[u] < 0) continue;
        const uint8_t* from = src + (int64_t)(t1 + u) * ss.t * SES;
        uint8_t* to = dst + (page[u] * cs.z + slot[u] * cs.t) * CES;
        for (int e = 0; e < n; ++e) {
          if constexpr (CDT == LH_F8E4M3) to[e] = (uint8_t)e4m3_pack2(e4m3_clamp(load_as_f32<SDT>(from, e) / scale), 0.0f);
          else if constexpr (SES == 4) reinterpret_cast<uint32_t*>(to)[e] = reinterpret_cast<const uint32_t*>(from)[e];
          else reinterpret_cast<uint16_t*>(to)[e] = reinterpret_cast<const uint16_t*>(from)[e];
        }
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
  int32_t budget, recent;
  int32_t elem_bytes;
  int32_t slices;  // column slices of a row of keys (and of values)
};

__device__ __forceinline__ int evict_length(const EvictArgs& a, int b) { return min(max(a.lengths[b], 0), a.c.capacity()); }

// An order of the weights as unsigned numbers: larger weight, larger number; -0 and 0 alike, a NaN below everything.  Positions that
// stay in any case are above all of them, positions that are not there below.
constexpr uint32_t kKeyAbsent = 0, kKeyNaN = 1, kKeyRecent = 0xffffffffu;
__device__ __forceinline__ uint32_t evict_key(float w) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f), sign = (uint32_t)((int32_t)u >> 31);
  return w != w ? kKeyNaN : u ^ (sign | 0x80000000u);
}

constexpr int kEvictBins = 2048;  // 11 bits of the key a pass

// Which positions of one head of one sequence stay, in order.  The (budget - recent)-th largest key among the positions that
// are not recent is found by its digits, 11, 11 and 10 bits, from counts in LDS, until so few keys share the digits that
// they are ranked against each other; of the positions that share it the lowest stay.  A thread has up to 16 neighbouring
// positions, whose place among those that stay comes from one running sum over the workgroup.  4 waves for tables of up to 4096
// positions, 16 for longer ones; up to 16384 positions the keys stay in registers, a longer sequence reads its weights (which the L2 holds) in
// every pass, 16384 at a time.  What bounds it is the chain of passes: 16384 positions of 32 heads 16 us, 1024 of 192 heads 7.
constexpr int kEvictKeys = 16;   // of a thread
constexpr int kEvictRank = 128;  // keys that are ranked
template <int THREADS>
struct EvictShared {
  // (Weights share a few exponents, so a wave's lanes meet in a few bins: four counts a bin, lanes take turns.)
  // A thread adds up kEvictBins / THREADS neighbours: one element more behind them keeps lanes off each other's banks.
  u32x4 bins[kEvictBins + THREADS];
  unsigned long long wave_sum[THREADS / 64];
  uint32_t found[3];  // digit, how many of the digit's keys stay, how many there are
  uint32_t ranked;
  u32x4 rank[kEvictRank / 4];
};
// The sum over the threads before this one.
template <int THREADS, typename T>
__device__ __forceinline__ T evict_before(EvictShared<THREADS>& s, T mine, T* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const T run = wave_scan(mine);
  if (lane == 63) s.wave_sum[wave] = run;
  __syncthreads();
  T before = run - mine, total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) {
    const T x = (T)s.wave_sum[i];
    before += i < wave ? x : 0;
    total += x;
  }
  *all = total;
  return before;
}

template <int THREADS>
__device__ __forceinline__ void evict_select(const EvictArgs& a, int n, const float* w, EvictShared<THREADS>& s) {
  constexpr int BINS = kEvictBins / THREADS;  // bins a thread adds up
  const int tid = threadIdx.x, lane = tid & 63;
  const int old = n - a.recent;             // positions that compete
  uint32_t want = a.budget - a.recent;      // of them stay; below `old`
  const int mine = n <= THREADS * kEvictKeys ? ((n + THREADS - 1) / THREADS + 3) / 4 * 4 : kEvictKeys;  // positions of a thread
  const int chunks = (n + THREADS * mine - 1) / (THREADS * mine);
  uint32_t keys[kEvictKeys];
  auto load = [&](int chunk) {
    const int t0 = (chunk * THREADS + tid) * mine;
#pragma unroll
    for (int q = 0; q < kEvictKeys; q += 4) {
      if (q >= mine) break;
      if (t0 + q + 4 <= old) {
        const Chunk<4>::type v = *reinterpret_cast<const Chunk<4>::type*>(w + t0 + q);
#pragma unroll
        for (int e = 0; e < 4; ++e) keys[q + e] = evict_key(bits_to_f32(v[e]));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = t0 + q + e;
          keys[q + e] = t < old ? evict_key(w[t]) : t < n ? kKeyRecent : kKeyAbsent;
        }
      }
    }
  };
  // f(position, key) for the thread's positions among `chunk`.
  auto each = [&](int chunk, auto f) {
    const int t0 = (chunk * THREADS + tid) * mine;
#pragma unroll
    for (int q = 0; q < kEvictKeys; q += 4) {
      if (q >= mine) break;
#pragma unroll
      for (int e = 0; e < 4; ++e) f(t0 + q + e, keys[q + e]);
    }
  };
  uint32_t threshold = kKeyRecent - 1;  // (no weight's key)
  load(0);
  if (want > 0) {
    uint32_t prefix = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
#pragma unroll
      for (int i = 0; i < BINS; ++i) s.bins[tid * (BINS + 1) + i] = u32x4{0, 0, 0, 0};
      if (tid == 0) s.ranked = 0;
      if (tid < kEvictRank / 4) s.rank[tid] = u32x4{kKeyAbsent, kKeyAbsent, kKeyAbsent, kKeyAbsent};
      __syncthreads();
      uint32_t* const counts = reinterpret_cast<uint32_t*>(s.bins) + (lane & 3);
      for (int chunk = 0; chunk < chunks; ++chunk) {
        if (chunks > 1) load(chunk);
        each(chunk, [&](int t, uint32_t key) {
          const uint32_t bin = (key >> shift) & ((1u << bits) - 1);
          if ((key - 1u < kKeyRecent - 1u) & ((pass == 0) | (key >> (shift + bits) % 32 == prefix))) {
            // The lanes that share the first one's bin add up first: weights that are all 0 would come one by one.
            const uint64_t same = __ballot(bin == (uint32_t)__builtin_amdgcn_readfirstlane(bin));
            const uint32_t number = same >> lane & 1 ? __popcll(same) : 1u;
            if (number == 1u || __ffsll((unsigned long long)same) - 1 == lane) atomicAdd(&counts[4 * (bin + bin / BINS)], number);
          }
        });
      }
      __syncthreads();
      // The digit in which the want-th key from above lies: thread i has the bins BINS i and on in the order from above.
      uint32_t c[BINS], sum = 0;
#pragma unroll
      for (int i = 0; i < BINS; ++i) {
        const u32x4 x = s.bins[(THREADS - 1 - tid) * (BINS + 1) + BINS - 1 - i];
        sum += c[i] = x[0] + x[1] + x[2] + x[3];
      }
      uint32_t all, before = evict_before<THREADS>(s, sum, &all);
#pragma unroll
      for (int i = 0; i < BINS; ++i) {
        if (before < want && want <= before + c[i]) s.found[0] = kEvictBins - 1 - BINS * tid - i, s.found[1] = want - before, s.found[2] = c[i];
        before += c[i];
      }
      __syncthreads();
      prefix = prefix << bits | s.found[0];
      want = s.found[1];
      const uint32_t left = s.found[2];
      if (pass < 2 && left <= kEvictRank) {
        for (int chunk = 0; chunk < chunks; ++chunk) {
          if (chunks > 1) load(chunk);
          each(chunk, [&](int t, uint32_t key) {
            if ((key - 1u < kKeyRecent - 1u) & (key >> shift == prefix)) reinterpret_cast<uint32_t*>(s.rank)[atomicAdd(&s.ranked, 1u)] = key;
          });
        }
        __syncthreads();
        if (tid < (int)left) {
          const uint32_t key = reinterpret_cast<const uint32_t*>(s.rank)[tid];
          uint32_t above = 0, same = 0;
#pragma unroll 8
          for (uint32_t j = 0; j < (left + 3) / 4; ++j) {
            const u32x4 x = s.rank[j];
#pragma unroll
            for (int e = 0; e < 4; ++e) above += x[e] > key, same += x[e] == key;
          }
          if (above < want && want <= above + same) s.found[0] = key, s.found[1] = want - above;
        }
        __syncthreads();
        prefix = s.found[0], want = s.found[1];
        break;
      }
    }
    threshold = prefix;  // the want lowest positions of those with this key stay
  }
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.budget;
  uint32_t base = 0, base_ties = 0;  // of the chunks before: above the threshold, at it
  for (int chunk = 0; chunk < chunks; ++chunk) {
    if (chunks > 1) load(chunk);
    uint32_t above = 0, ties = 0;
    each(chunk, [&](int, uint32_t key) { above += key > threshold, ties += key == threshold; });
    uint64_t all;
    __syncthreads();
    const uint64_t before = evict_before<THREADS>(s, (uint64_t)ties << 32 | above, &all);
    uint32_t tied = base_ties + (uint32_t)(before >> 32), at = base + (uint32_t)before + min(tied, want);
    each(chunk, [&](int t, uint32_t key) {
      const bool tie = key == threshold;
      if ((key > threshold) | (tie & (tied < want))) kept[at++] = t;
      tied += tie;
    });
    base += (uint32_t)all, base_ties += (uint32_t)(all >> 32);
  }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) kv_evict_select(EvictArgs a) {
  __shared__ EvictShared<THREADS> s;
  const int b = blockIdx.x / a.c.heads, h = blockIdx.x % a.c.heads;
  const int n = evict_length(a, b);
  if (threadIdx.x == 0) a.held[blockIdx.x] = n;
  if (n <= a.budget) return;
  const float* w = a.weights + b * a.sw_b + h * a.sw_h;
  evict_select<THREADS>(a, n, w, s);
}

// Rows move up, row kept[j] to row j: kept[j] >= j, so what a block of rows j .. j + R - 1 overwrites no later block reads,
// and within the block every row is in registers before any is written.  A workgroup takes a column slice of 128 bytes
// of the keys or the values of a head, or its weights: slices know nothing of each other.  What bounds it is that there are only so many slices,
// each a CU's chain of blocks.  Where there are fewer than one for every four CUs they are 64 bytes wide: half a line of memory, but twice
// the CUs.  (Both launches of an eviction, us, slices of 128 and of 64 bytes: 4096 of 16384 positions of 8 heads of 128 in bf16 36.9 and 29.3, of 16 heads 39.4 and
// 37.6, of 32 heads of ragged lengths 48.4 and 50.5, 2048 of 4096 of 64 heads 46.0 and 51.6.)
constexpr int kMoveThreads = 1024;
constexpr int kMoveRows = 2;  // of a thread, in flight at once

// PIECES of 16 bytes: a slice.  WHOLE: rows are whole pieces, and the blocks go through a pipeline: while one is written, the rows of the next, the
// table's entries of the one after it and what `kept` says of the third are on their way.  (Rows of the next block are not among those
// that this one overwrites.  One block after the other, of twice the size, 4096 of 16384 positions of 32 heads took 81 us instead of 48, 512 of 1024 of 192 heads
// of 64 24 instead of 18.)  Lanes that have nothing to move load the first row of all: nothing but the stores branches.
template <int PIECES, bool WHOLE>
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
  const int col = (slice * PIECES + tid % PIECES) * 16;  // a thread each
  const int bytes = min(16, row_bytes - col);    // (none, or less than a chunk, where the row ends)
  constexpr int kRows = kMoveThreads / PIECES;
  if constexpr (WHOLE) {
    struct Block {
      int j[kMoveRows], from[kMoveRows], entry_from[kMoveRows], entry_to[kMoveRows];
    };
    const int64_t table_row = b * a.c.table_stride;
    uint8_t* const cache = base + min(col, row_bytes - 16);
    const bool live = bytes > 0;
    auto look_up = [&](int j0, Block& k) {
#pragma unroll
      for (int r = 0; r < kMoveRows; ++r) k.j[r] = j0 + r * kRows + tid / PIECES, k.from[r] = kept[min(k.j[r], a.budget - 1)];
    };
    auto find_pages = [&](Block& k) {
#pragma unroll
      for (int r = 0; r < kMoveRows; ++r) {
        k.entry_from[r] = a.c.entry(table_row + a.c.by_size.div((uint32_t)k.from[r]));
        k.entry_to[r] = a.c.entry(table_row + a.c.by_size.div((uint32_t)min(k.j[r], a.budget - 1)));
      }
    };
    auto place = [&](int entry, int t) -> uint8_t* {
      const int slot = t - (int)a.c.by_size.div((uint32_t)t) * a.c.size;
      return cache + (entry * cs.z + slot * cs.t) * es;
    };
    auto request = [&](const Block& k, any16* x, uint8_t** to) {
#pragma unroll
      for (int r = 0; r < kMoveRows; ++r) {
        const bool moves = live && k.j[r] < a.budget && k.from[r] != k.j[r] && (uint32_t)k.entry_from[r] < (uint32_t)a.c.pages && (uint32_t)k.entry_to[r] < (uint32_t)a.c.pages;
        x[r] = *reinterpret_cast<const any16*>(moves ? place(k.entry_from[r], k.from[r]) : cache);
        to[r] = moves ? place(k.entry_to[r], k.j[r]) : nullptr;
      }
    };
    constexpr int ROWS = kRows * kMoveRows;
    any16 x[2][kMoveRows];
    uint8_t* to[2][kMoveRows];
    Block k[3];  // of this block, of the next, of the one after it, in turn
    look_up(0, k[0]);
    look_up(ROWS, k[1]);
    find_pages(k[0]);
    find_pages(k[1]);
    look_up(2 * ROWS, k[2]);
    request(k[0], x[0], to[0]);
    // Block at j0: its rows are in x[now], `next` knows the pages of the one behind it, `after` the positions of the one behind that.
    auto step = [&](int j0, int now, Block& own, Block& next, Block& after) {
      find_pages(after);
      look_up(j0 + 3 * ROWS, own);
      request(next, x[now ^ 1], to[now ^ 1]);
#pragma unroll
      for (int r = 0; r < kMoveRows; ++r)
        asm volatile("" : "+v"(x[now][r][0]), "+v"(x[now][r][1]), "+v"(x[now][r][2]), "+v"(x[now][r][3]));
      __syncthreads();
#pragma unroll
      for (int r = 0; r < kMoveRows; ++r)
        if (to[now][r] != nullptr) *reinterpret_cast<any16*>(to[now][r]) = x[now][r];
    };
#pragma unroll 1
    for (int j0 = 0; j0 < a.budget; j0 += 6 * ROWS) {
      step(j0, 0, k[0], k[1], k[2]);
      if (j0 + ROWS < a.budget) step(j0 + ROWS, 1, k[1], k[2], k[0]);
      if (j0 + 2 * ROWS < a.budget) step(j0 + 2 * ROWS, 0, k[2], k[0], k[1]);
      if (j0 + 3 * ROWS < a.budget) step(j0 + 3 * ROWS, 1, k[0], k[1], k[2]);
      if (j0 + 4 * ROWS < a.budget) step(j0 + 4 * ROWS, 0, k[1], k[2], k[0]);
      if (j0 + 5 * ROWS < a.budget) step(j0 + 5 * ROWS, 1, k[2], k[0], k[1]);
    }
    return;
  }
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
      const int j = j0 + r * kRows + tid / PIECES;
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
static int append_launch(const AppendArgs& a, unsigned blocks, unsigned threads, hipStream_t s) {
  LH_LAUNCH((kv_append_kernel<SDT, CDT>), dim3(blocks), dim3(threads), 0, s, a);
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
  a.T = (int32_t)T;
  const int e = dtype == LH_F32 && cache->dtype == LH_F32 ? 4 : 8, chunks = (a.c.d + e - 1) / e;
  a.per_token = 2 * a.c.heads * chunks, a.by_chunks = FastDiv((uint32_t)chunks);
  const unsigned threads = a.per_token >= 256 ? 256 : (unsigned)(a.per_token + 63) / 64 * 64;
  a.parts = (a.per_token + (int)threads - 1) / (int)threads;
  // As many tokens a workgroup as leave about 8 workgroups per CU, 16 at most.
  const int64_t tokens = B * T * a.parts / (8 * num_cus());
  a.tokens = tokens < 1 ? 1 : tokens > 16 ? 16 : (int32_t)tokens;
  a.token_blocks = (int32_t)((T + a.tokens - 1) / a.tokens);
  LH_REQUIRE(B * a.token_blocks * a.parts < (1ll << 24), "lh_hip_kv_append: too many tokens");
  const unsigned blocks = (unsigned)(B * a.token_blocks * a.parts);
  auto short_division = [](float scale) {
    uint32_t bits;
    std::memcpy(&bits, &scale, 4);
    return scale >= 0x1p-60f && scale <= 0x1p60f && (bits & 0x7fffffu) != 0x7fffffu ? 1.0f / scale : 0.0f;
  };
  a.k_inv = short_division(a.c.k_scale), a.v_inv = short_division(a.c.v_scale);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cache->dtype == LH_F8E4M3) {
    if (dtype == LH_BF16) return append_launch<LH_BF16, LH_F8E4M3>(a, blocks, threads, s);
    if (dtype == LH_F16) return append_launch<LH_F16, LH_F8E4M3>(a, blocks, threads, s);
    return append_launch<LH_F32, LH_F8E4M3>(a, blocks, threads, s);
  }
  if (dtype == LH_F32) return append_launch<LH_F32, LH_F32>(a, blocks, threads, s);
  return append_launch<LH_BF16, LH_BF16>(a, blocks, threads, s);  // (16 bits either way: they are only moved)
}

size_t lh_hip_kv_evict_workspace_bytes(int64_t B, int64_t n_kv_heads, int64_t budget) {
  constexpr int64_t kMost = 1ll << 31;
  if (B <= 0 || n_kv_heads <= 0 || budget <= 0 || B >= kMost || n_kv_heads >= kMost || B * n_kv_heads >= (1ll << 16) || budget >= kMost) return 0;
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
  LH_REQUIRE(workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && workspace_bytes >= need,
             "lh_hip_kv_evict: workspace too small or not 256-byte aligned: %zu of %zu bytes", workspace_bytes, need);
  a.weights = weights, a.sw_b = weights_stride_b, a.sw_h = weights_stride_h;
  a.lengths = lengths, a.new_lengths = new_lengths, a.kept = static_cast<int32_t*>(workspace);
  a.held = a.kept + B * a.c.heads * budget;
  a.budget = (int32_t)budget, a.recent = (int32_t)recent;
  a.elem_bytes = (int32_t)dtype_size(cache->dtype);
  const int row_bytes = a.c.d * a.elem_bytes;
  const bool narrow = row_bytes % 16 == 0 && B * a.c.heads * 2 * ((row_bytes + 127) / 128) <= num_cus() / 4;
  a.slices = narrow ? (row_bytes + 63) / 64 : (row_bytes + 127) / 128;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 heads((unsigned)(B * a.c.heads));
  if (a.c.capacity() <= 256 * kEvictKeys) LH_LAUNCH(kv_evict_select<256>, heads, dim3(256), 0, s, a);
  else LH_LAUNCH(kv_evict_select<1024>, heads, dim3(1024), 0, s, a);
  if (const int rc = check_launch("kv_evict_select")) return rc;
  const dim3 moves((unsigned)(B * a.c.heads * (1 + 2 * a.slices)));
  if (row_bytes % 16 != 0) LH_LAUNCH((kv_evict_move<8, false>), moves, dim3(kMoveThreads), 0, s, a);
  else if (narrow) LH_LAUNCH((kv_evict_move<4, true>), moves, dim3(kMoveThreads), 0, s, a);
  else LH_LAUNCH((kv_evict_move<8, true>), moves, dim3(kMoveThreads), 0, s, a);
  return check_launch("kv_evict_move");
}

}  // extern "C"
