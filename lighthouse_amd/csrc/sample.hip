// The next token of a row of logits: temperature, top-k, top-p and min-p, then a draw with a given random number.
//
// With w_i = exp((x_i - max) / T) and the words in falling order of (x, then rising index), each filter keeps a beginning of
// that order: the first k; the words before which less than top_p of the mass lies; the words with w >= min_p.  So what stays
// is described by its last word (cut_x, cut_i), and no row is ever sorted: the last word is found in a histogram of the distance
// max - x, by counts (top-k) or masses (top-p), and then among the few words of the bin it lies in.  The draw is
// a search in the running sum over the indices.
//
// Masses are whole numbers, w in units of 2^-kBits with w from a 64-bit exponential: sums of them are exact in any order, so
// neither the atomics of the histogram nor the split over lanes and waves can change a token, and a sum over
// 131072 words is off by about 1e-12 of the whole: as good as a sum in 64-bit floating point.  (In 32 bits a row of 5000 likely words would
// get another token about once in 10^4 rows.)
//
// One workgroup of 16 waves takes a row; a wave takes a contiguous share of it.
#include "common.h"

namespace lh {

struct SampleArgs {
  int64_t* tokens;
  const void* logits;
  const float* uniform;
  int64_t ld;
  int32_t V;
  int32_t bits;  // of a mass behind the point: V words of weight 1 stay below 2^62
  lh_sample_opts o;
};

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 512;
constexpr int kSampleBatch = 4;  // pieces of a row that a lane has in flight

// (By value: a bit cast of a vector's element itself reads its first one.)
__device__ __forceinline__ float sample_bits(uint32_t u) { return __builtin_bit_cast(float, u); }

template <int DT>
struct SampleRow {
  static constexpr int E = DT == LH_F32 ? 4 : 8;
  const uint8_t* base;
  int V, begin, end, lane;  // of this wave

  __device__ __forceinline__ void load(float* x, int i0) const {
    constexpr int ES = DT == LH_F32 ? 4 : 2;
    if (i0 + E <= V) {
      const typename Chunk<ES>::type w = *reinterpret_cast<const typename Chunk<ES>::type*>(base + (int64_t)i0 * ES);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (DT == LH_F32) x[e] = sample_bits(w[e]);
        else x[2 * e] = unpack_lo<DT>(w[e]), x[2 * e + 1] = unpack_hi<DT>(w[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = i0 + e < V ? load_as_f32<DT>(base, i0 + e) : -INFINITY;
    }
    // No word: NaN, like -inf.
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] != x[e] ? -INFINITY : x[e];
  }
  // f(x, first index) for every piece of the wave's share, in order.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
    for (int i = begin; i < end; i += 64 * E * kSampleBatch) {
      float x[kSampleBatch][E];
#pragma unroll
      for (int p = 0; p < kSampleBatch; ++p) load(x[p], i + p * 64 * E < end ? i + p * 64 * E + lane * E : V);
#pragma unroll
      for (int p = 0; p < kSampleBatch; ++p)
        if (i + p * 64 * E < end) f(x[p], i + p * 64 * E + lane * E);
    }
  }
};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor((unsigned long long)v, o);
  return v;
}

struct SampleShared {
  unsigned long long mass[kSampleBins];
  uint32_t count[kSampleBins];
  float list_x[kSampleList];
  int32_t list_i[kSampleList];
  unsigned long long list_w[kSampleList];
  unsigned long long wave_mass[kSampleWaves];
  uint32_t wave_count[kSampleWaves];
  float wave_lo[kSampleWaves], wave_hi[kSampleWaves];
  int32_t wave_i[kSampleWaves];
  int32_t bin, listed;
  float cut_x;
  int32_t cut_i;
  unsigned long long above_mass;
  uint32_t above_count, in_bin;
};

template <int DT>
struct Sampler {
  static constexpr int E = SampleRow<DT>::E;
  SampleShared& s;
  SampleRow<DT> row;
  int tid, lane, wave;
  float top;       // the largest logit
  double inv_t, unit;
  float cut_x;     // words below (cut_x, cut_i) have been dropped
  int32_t cut_i;

  __device__ __forceinline__ double weight(float x) const { return x == top ? 1.0 : exp(((double)x - (double)top) * inv_t); }
  __device__ __forceinline__ uint64_t mass(float x) const { return (uint64_t)(weight(x) * unit + 0.5); }
  __device__ __forceinline__ bool stays(float x, int i) const { return x > cut_x || (x == cut_x && i <= cut_i); }

  // Finds the last word that stays and makes it the cut: the first `k` words (BY_MASS false), or those before which less than top_p of
  // the mass of what is left lies.
  template <bool BY_MASS>
  __device__ __forceinline__ void cut(uint32_t k, double top_p, float lowest) {
    float hi = top, lo = fmaxf(lowest, BY_MASS ? top - (float)(40.0 / inv_t) : top - 32.0f);
    float below = INFINITY;          // words of this interval are at most this (and at least `from` after the first level)
    float from = -INFINITY;
    uint64_t above = 0, goal = 0;    // mass, or count, in front of the interval; what the last word brings it to, at least
    if (!BY_MASS) goal = k;
#pragma unroll 1
    for (int level = 0;; ++level) {
      const double width = (double)hi - (double)lo;
      const float inv32 = (float)(kSampleBins / (width > 0 ? width : 1.0));
      const double inv64 = kSampleBins / (width > 0 ? width : 1.0);
      // Falls with x: the same expression finds a word's bin when it is counted and when it is listed.
      auto bin_of = [&](float x) -> int {
        if (level == 0) return (int)fminf((hi - x) * inv32, (float)(kSampleBins - 1));
        return (int)fmin(((double)hi - (double)x) * inv64, (double)(kSampleBins - 1));
      };
      auto inside = [&](float x, int i) { return x <= below && x >= from && x > -INFINITY && stays(x, i); };
      for (int i = tid; i < kSampleBins; i += kSampleThreads) s.mass[i] = 0, s.count[i] = 0;
      if (tid == 0) s.listed = 0;
      __syncthreads();
      row.each([&](const float* x, int i0) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (inside(x[e], i0 + e)) {
            const int at = bin_of(x[e]);
            atomicAdd(&s.count[at], 1u);
            if (BY_MASS) atomicAdd(&s.mass[at], (unsigned long long)mass(x[e]));
          }
      });
      __syncthreads();
      // Running sums over the bins, two a thread, from above.
      const uint32_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
      const uint64_t v0 = BY_MASS ? s.mass[2 * tid] : c0, v1 = BY_MASS ? s.mass[2 * tid + 1] : c1;
      uint64_t run = v0 + v1;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint64_t up = __shfl_up((unsigned long long)run, o);
        if (lane >= o) run += up;
      }
      if (lane == 63) s.wave_mass[wave] = run;
      __syncthreads();
      uint64_t before = above + run - v0 - v1, total = above;
      for (int w = 0; w < kSampleWaves; ++w) {
        if (w < wave) before += s.wave_mass[w];
        total += s.wave_mass[w];
      }
      if (BY_MASS && level == 0) {
        // "less than top_p of the mass before it" in whole numbers: before < ceil(top_p * mass).
        goal = (uint64_t)ceil(top_p * (double)total);
        if (goal < 1) goal = 1;
        if (goal > total) goal = total;
      }
      if (goal > total) return;  // (fewer than k words are left: infinite ones)
      if (before < goal && goal <= before + v0) s.bin = 2 * tid, s.above_mass = before, s.in_bin = c0;
      else if (before + v0 < goal && goal <= before + v0 + v1) s.bin = 2 * tid + 1, s.above_mass = before + v0, s.in_bin = c1;
      __syncthreads();
      const int at = s.bin;
      const uint32_t members = s.in_bin;
      above = s.above_mass;
      // The members of the bin: listed if they are few, and their lowest and highest value.
      float low = INFINITY, high = -INFINITY;
      row.each([&](const float* x, int i0) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (inside(x[e], i0 + e) && bin_of(x[e]) == at) {
            low = fminf(low, x[e]), high = fmaxf(high, x[e]);
            if (members <= kSampleList) {
              const int j = atomicAdd(&s.listed, 1);
              s.list_x[j] = x[e], s.list_i[j] = i0 + e;
              if (BY_MASS) s.list_w[j] = mass(x[e]);
            }
          }
      });
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) low = fminf(low, __shfl_xor(low, o)), high = fmaxf(high, __shfl_xor(high, o));
      if (lane == 0) s.wave_lo[wave] = low, s.wave_hi[wave] = high;
      __syncthreads();
      for (int w = 0; w < kSampleWaves; ++w) low = fminf(low, s.wave_lo[w]), high = fmaxf(high, s.wave_hi[w]);
      if (members <= kSampleList) {
        if (tid < (int)members) {  // what lies before this member, in the order
          const float x = s.list_x[tid];
          const int i = s.list_i[tid];
          const uint64_t own = BY_MASS ? s.list_w[tid] : 1;
          uint64_t front = above;
          for (int j = 0; j < (int)members; ++j) {
            const float y = s.list_x[j];
            if (y > x || (y == x && s.list_i[j] < i)) front += BY_MASS ? s.list_w[j] : 1;
          }
          if (front < goal && goal <= front + own) s.cut_x = x, s.cut_i = i;
        }
        __syncthreads();
        cut_x = s.cut_x, cut_i = s.cut_i;
        return;
      }
      if (low == high) {
        // Words of one value: the first of them, by index, as many as reach the goal.
        const uint64_t own = BY_MASS ? mass(low) : 1;
        const uint32_t stay = own == 0 ? members : (uint32_t)((goal - above + own - 1) / own);
        const int last = nth(low, stay);
        cut_x = low, cut_i = last;
        return;
      }
      hi = high, lo = low, below = high, from = low;
      __syncthreads();
    }
  }

  // The index of the n-th word (from 1) of those of this value that stay.
  __device__ __forceinline__ int nth(float value, uint32_t n) {
    uint32_t mine = 0;
    row.each([&](const float* x, int i0) {
#pragma unroll
      for (int e = 0; e < E; ++e) mine += x[e] == value && stays(x[e], i0 + e);
    });
    uint32_t all = mine;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) all += __shfl_xor(all, o);
    if (lane == 0) s.wave_count[wave] = all;
    __syncthreads();
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += s.wave_count[w];
    if (before < n && n <= before + all) {
      row.each([&](const float* x, int i0) {
        uint32_t here = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) here += x[e] == value && stays(x[e], i0 + e);
        uint32_t run = here;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const uint32_t up = __shfl_up(run, o);
          if (lane >= o) run += up;
        }
        uint32_t at = before + run - here;
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (x[e] == value && stays(x[e], i0 + e) && ++at == n) s.cut_i = i0 + e;
        before += __shfl(run, 63);
      });
    }
    __syncthreads();
    return s.cut_i;
  }
};

template <int DT>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  constexpr int E = SampleRow<DT>::E, ES = DT == LH_F32 ? 4 : 2;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float temperature = a.o.temperature ? a.o.temperature[b] : a.o.temperature_all;
  const int top_k = a.o.top_k ? a.o.top_k[b] : a.o.top_k_all;
  const float top_p = a.o.top_p ? a.o.top_p[b] : a.o.top_p_all;
  const float min_p = a.o.min_p ? a.o.min_p[b] : a.o.min_p_all;
  const double u = (double)a.uniform[b];

  const int pieces = (a.V + 64 * E - 1) / (64 * E), share = (pieces + kSampleWaves - 1) / kSampleWaves * (64 * E);
  const int begin = min(wave * (int64_t)share, (int64_t)a.V), end = min(begin + (int64_t)share, (int64_t)a.V);
  const SampleRow<DT> row = {static_cast<const uint8_t*>(a.logits) + b * a.ld * ES, a.V, begin, end, lane};

  // Largest logit, its lowest index, the smallest, how many words.
  float top = -INFINITY, lowest = INFINITY;
  int top_i = 0x7fffffff;
  uint32_t words = 0;
  row.each([&](const float* x, int i0) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (x[e] > top) top = x[e], top_i = i0 + e;
      if (x[e] > -INFINITY) lowest = fminf(lowest, x[e]), ++words;
    }
  });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const float x = __shfl_xor(top, o);
    const int i = __shfl_xor(top_i, o);
    if (x > top || (x == top && i < top_i)) top = x, top_i = i;
    lowest = fminf(lowest, __shfl_xor(lowest, o));
    words += __shfl_xor(words, o);
  }
  if (lane == 0) s.wave_hi[wave] = top, s.wave_i[wave] = top_i, s.wave_lo[wave] = lowest, s.wave_count[wave] = words;
  __syncthreads();
  words = 0;
  for (int w = 0; w < kSampleWaves; ++w) {
    const float x = s.wave_hi[w];
    if (x > top || (x == top && s.wave_i[w] < top_i)) top = x, top_i = s.wave_i[w];
    lowest = fminf(lowest, s.wave_lo[w]);
    words += s.wave_count[w];
  }
  __syncthreads();
  if (words == 0 || !(temperature > 0.0f) || top_k == 1) {
    if (tid == 0) a.tokens[b] = words == 0 ? -1 : top_i;
    return;
  }

  Sampler<DT> f = {s, row, tid, lane, wave, top, 1.0 / (double)temperature, (double)(1ull << a.bits), -INFINITY, -1};
  if (top == INFINITY) f.cut_x = INFINITY, f.cut_i = 0x7fffffff, lowest = top;  // only those
  if (top_k > 0 && (uint32_t)top_k < words) f.template cut<false>((uint32_t)top_k, 0.0, lowest);
  if (top_p < 1.0f) {
    __syncthreads();
    f.template cut<true>(0, (double)top_p, lowest);
  }
  __syncthreads();

  // What stays: its mass by waves, and within a wave by up to 64 groups of pieces, lane g has group g's.
  const double least = min_p > 0.0f ? (double)min_p : 0.0;
  auto left = [&](float x, int i) -> uint64_t {
    if (!(x > -INFINITY) || !f.stays(x, i)) return 0;
    const double w = f.weight(x);
    return w >= least || i == top_i ? (uint64_t)(w * f.unit + 0.5) : 0;
  };
  const int group = ((share / (64 * E) + 63) / 64) * 64 * E;  // words
  uint64_t of_group = 0, total = 0;
  row.each([&](const float* x, int i0) {
    uint64_t m = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) m += left(x[e], i0 + e);
    if (__any(m != 0)) {
      m = wave_sum64(m);
      if (lane == (i0 - lane * E - begin) / group) of_group += m;
      total += m;
    }
  });
  if (lane == 0) s.wave_mass[wave] = total;
  __syncthreads();
  uint64_t before = 0, all = 0;
  for (int w = 0; w < kSampleWaves; ++w) {
    if (w < wave) before += s.wave_mass[w];
    all += s.wave_mass[w];
  }
  // The word whose running sum is the first above u * all: above `goal`, a whole number below `all`.
  uint64_t goal = all - 1;
  if (u < 1.0) goal = u > 0.0 ? (uint64_t)(u * (double)all) : 0;
  if (goal > all - 1) goal = all - 1;
  if (!(before <= goal && goal < before + total)) return;
  uint64_t run = of_group;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t up = __shfl_up((unsigned long long)run, o);
    if (lane >= o) run += up;
  }
  const int g = __popcll(__ballot(before + run <= goal));  // groups that end at or before it
  before += g == 0 ? 0 : __shfl((unsigned long long)run, g - 1);
  for (int i = begin + g * group; i < end; i += 64 * E) {
    const int i0 = i + lane * E;
    float x[E];
    row.load(x, i0);
    uint64_t m[E], own = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) own += m[e] = left(x[e], i0 + e);
    uint64_t sum = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint64_t up = __shfl_up((unsigned long long)sum, o);
      if (lane >= o) sum += up;
    }
    uint64_t at = before + sum - own;
    if (at <= goal && goal < at + own) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (at <= goal && goal < at + m[e]) a.tokens[b] = i0 + e;
        at += m[e];
      }
    }
    before += __shfl((unsigned long long)sum, 63);
    if (before > goal) return;
  }
}

}  // namespace lh

using namespace lh;

extern "C" int lh_hip_sample(int64_t* tokens, const void* logits, const float* uniform, int64_t B, int64_t V, int64_t ld,
                             int32_t dtype, const lh_sample_opts* opts, void* stream) {
  LH_REQUIRE(tokens && logits && uniform && opts, "lh_hip_sample: null pointer");
  LH_REQUIRE(B >= 0 && B < (1ll << 22) && V >= 1 && V < (1ll << 30), "lh_hip_sample: bad shape %lld x %lld", (long long)B, (long long)V);
  LH_REQUIRE(B <= 1 || ld >= V, "lh_hip_sample: rows overlap");
  LH_REQUIRE(dtype == LH_F32 || dtype == LH_BF16 || dtype == LH_F16, "lh_hip_sample: unsupported dtype %d", dtype);
  if (B == 0) return LH_OK;
  SampleArgs a = {tokens, logits, uniform, ld, (int32_t)V, 62, *opts};
  while ((V >> (62 - a.bits)) != 0) --a.bits;
  if (a.bits > 52) a.bits = 52;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)B), block(kSampleThreads);
  if (dtype == LH_F32) LH_LAUNCH(sample_kernel<LH_F32>, grid, block, 0, s, a);
  else if (dtype == LH_BF16) LH_LAUNCH(sample_kernel<LH_BF16>, grid, block, 0, s, a);
  else LH_LAUNCH(sample_kernel<LH_F16>, grid, block, 0, s, a);
  return check_launch("sample");
}
