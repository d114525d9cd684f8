// The next token of a row of logits: temperature, top-k, top-p and min-p, then a draw with a given random number.
//
// With w_i = exp((x_i - max) / T) and the words in falling order of (x, then rising index), each filter keeps a beginning of
// that order: the first k; the words before which less than top_p of the mass lies; the words with w >= min_p.  So what stays
// is described by its last word, and no row is ever sorted.  The draw is a search in the running sum over the indices.
//
// Masses are whole numbers, w in units of 2^-bits with w from a 64-bit exponential (to 6e-12 of itself): sums of them are exact in any
// order, so neither atomics nor the split over lanes and waves can change a token.  (In 32 bits a row of 5000 likely words would get another
// token about once in 10^4 rows.)  What a word has beside whole units is lost, and a row may hold one likely word and unlikely ones
// without end, so the units follow from the sums: 2^-49 of the largest weight for up to 8192 words, which lose half a unit each, 2^-36 of the
// whole at most; the same for each chunk of a longer row, and for the row that its chunks make up, units by their sum.  Where one
// workgroup takes a row of several chunks they are 2^-51, or what the sum leaves room for, and V words lose V 2^-52; in rows without
// chunks down to 2^-60, cut off instead of rounded, and V words lose V 2^-59.  (With units by V alone, such that V likely words fit,
// 131072 unlikely ones lost 2^-28, 2^24 of them 2^-15.)
//
// A row of more than 8192 words is digested first, 8192 words a workgroup: for top-k (up to 512) a chunk lists its own largest words, otherwise
// it adds up its masses, in units of a power of two near its largest word's, and, where a filter will ask for it, by sixteenths of an octave
// of w below it.  Whole powers and a grid that starts at them let another workgroup put the chunks of a row together,
// what falls below its units aside.  That one then has the candidates of top-k to sort, or finds in the sums the bin that the last word lies in, collects the words
// of that bin from the chunks that have any, and evaluates one chunk, the one that the draw falls into.
//
// Rows of one chunk, and what a digest does not settle (top-k above 512, thousands of words in the bin of the cut, infinite logits), take
// one workgroup of 16 waves from the start.  Where few words can stay, they are listed: of the largest word of each of the 1024 threads the K-th
// is at most the K-th of the row, so the words that reach it are K or a few more; the list is sorted in LDS.  Otherwise the last
// word is found in a histogram of the distance max - x, by counts (top-k) or masses (top-p), and then among the words of the bin it
// lies in.
//
// Measured: one row of 50257 f32 with top-k 50 and top-p 6.4 us for the digest and 9.5 for the rest, both a chain of a dozen dependent steps (in one
// workgroup 24); 128 rows of 131072 bf16 with top-p and min-p 21.7 and 25.0 (without a digest 260).  Of that digest about 10 us are the loads and the largest
// word, 4 the masses and 6 their addition to bins in LDS; loading the next chunk during that (103 registers instead of 64, half the waves) took 3 us longer.
#include "common.h"
#include "wave_scan.h"

namespace lh {

constexpr int kChunkWords = 8192, kChunkBins = 512, kChunkList = 1024, kChunks = 64;  // words of a chunk, ..., most chunks of a row
constexpr int kDigestThreads = 512;
constexpr int kChunkBits = 49;  // of a mass behind the point: a chunk's words of weight 1 add up to 2^62

enum SampleMode {  // what a chunk holds: the same for all of a row
  kDigestTop = 1,     // its largest word
  kDigestList = 2,    // its largest words, top_k of them or more, or all
  kDigestTotal = 3,   // its mass (all that is known of a row with a larger top_k)
  kDigestBins = 4     // and by bins
};
struct SampleChunk {
  double power;               // masses are in units of 2^(power - kChunkBits); bins count sixteenths of an octave down from 2^power
  unsigned long long total;
  float top;                  // -inf: no words
  int32_t top_i;
  int32_t listed;             // or -1: the chunk settles nothing
  int32_t mode;
  union {
    unsigned long long bins[kChunkBins];   // the last one holds what lies below, too
    unsigned long long list[kChunkList];
  };
};

struct SampleArgs {
  int64_t* tokens;
  const void* logits;
  const float* uniform;
  int64_t ld;
  int32_t V;
  lh_sample_opts o;
  SampleChunk* chunks;  // [B][n_chunks], or null
  int32_t n_chunks;
  int32_t may_bin;      // whether a row's settings may ask for bins, as far as the host knows them
};

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr int kSampleBins = 2048;
constexpr int kSampleList = 2048;   // words: two a thread
constexpr int kSampleRank = 512;    // words: up to here they are ranked against each other
constexpr int kSampleTopK = 512;    // up to here top-k is tried on a list; also how many words a list for top-p aims at

// (By value: a bit cast of a vector's element itself reads its first one.)
__device__ __forceinline__ float sample_bits(uint32_t u) { return __builtin_bit_cast(float, u); }

template <int DT>
struct SampleRow {
  static constexpr int E = DT == LH_F32 ? 4 : 8;  // words of a piece
  static constexpr int kBatch = DT == LH_F32 ? 6 : 4;  // pieces that a lane has in flight
  const uint8_t* base;
  int V, begin, end, lane;  // of this wave

  __device__ __forceinline__ u32x4 load(int i0) const {
    constexpr int ES = DT == LH_F32 ? 4 : 2;
    if (i0 + E <= V) {
      const typename Chunk<ES>::type w = *reinterpret_cast<const typename Chunk<ES>::type*>(base + (int64_t)i0 * ES);
      return u32x4{w[0], w[1], w[2], w[3]};
    }
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == LH_F32) {
        w[e] = i0 + e < V ? reinterpret_cast<const uint32_t*>(base)[i0 + e] : 0xff800000u;
      } else {
        constexpr uint32_t none = DT == LH_BF16 ? 0xff80u : 0xfc00u;  // -inf
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base);
        const uint32_t lo = i0 + 2 * e < V ? p[i0 + 2 * e] : none, hi = i0 + 2 * e + 1 < V ? p[i0 + 2 * e + 1] : none;
        w[e] = lo | hi << 16;
      }
    }
    return w;
  }
  // Words as numbers; what is no word (NaN) is -inf, -0 is 0.
  __device__ __forceinline__ static void unpack(u32x4 w, float* x) {
    numbers(w, x);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = x[e] >= -INFINITY ? x[e] + 0.0f : -INFINITY;
  }
  __device__ __forceinline__ static void numbers(u32x4 w, float* x) {  // (a NaN as it is)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == LH_F32) x[e] = sample_bits(w[e]);
      else x[2 * e] = unpack_lo<DT>(w[e]), x[2 * e + 1] = unpack_hi<DT>(w[e]);
    }
  }
  // f(x, first index) for every piece of the wave's share, in order.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
    for (int i = begin; i < end; i += 64 * E * kBatch) {
      u32x4 w[kBatch];
#pragma unroll
      for (int p = 0; p < kBatch; ++p)
        if (i + p * 64 * E < end) w[p] = load(i + p * 64 * E + lane * E);
#pragma unroll
      for (int p = 0; p < kBatch; ++p)
        if (i + p * 64 * E < end) {
          float x[E];
          unpack(w[p], x);
          f(x, i + p * 64 * E + lane * E);
        }
    }
  }
};

// all * f, rounded down, or up, for 0 < f < 1 and all < 2^63: f is a whole number of up to 24 bits times a power of two.
__device__ __forceinline__ uint64_t part_of(uint64_t all, float f, bool up) {
  const uint32_t u = __builtin_bit_cast(uint32_t, f), e = u >> 23;
  const uint64_t m = e ? (u & 0x7fffffu) | 0x800000u : u;
  const int shift = 150 - (e ? (int)e : 1);  // at least 24
  const uint64_t hi = __umul64hi(all, m), lo = all * m;
  uint64_t whole, rest;
  if (shift < 64) {
    whole = hi << (64 - shift) | lo >> shift;
    rest = lo & ((1ull << shift) - 1);
  } else {
    const int more = shift - 64;
    whole = more < 64 ? hi >> more : 0;
    rest = lo | (more < 64 ? hi & ((1ull << more) - 1) : hi);
  }
  return whole + (up && rest != 0);
}

// w of a word of a chunk, in the units that the chunk counts in: sixteenths of an octave above 2^(power - bits), t = 16 (x c - power + bits), bits = kChunkBits.
// With n the nearest whole number and f the rest, 2^(t / 16) = 2^(n / 16) 2^(f / 16): a table of sixteenths, and 1 + f p(f) with p of degree 3
// through the values at the Chebyshev nodes (relative error 5.1e-12).  x c - power is rounded once, so words of all chunks keep
// their ratios; what is no word (-inf) comes out as 0 and in the last bin.
struct ChunkScale {
  double c16, offset;
  static constexpr int top = 16 * kChunkBits;  // n of the power itself
  __device__ __forceinline__ ChunkScale(double c, double power) : c16(16.0 * c), offset(16.0 * ((double)kChunkBits - power)) {}
  __device__ __forceinline__ double split(float x, int* n) const {
    const double t = fmax(__builtin_fma((double)x, c16, offset), -32768.0), whole = __builtin_rint(t);
    *n = (int)whole;
    return t - whole;
  }
  __device__ __forceinline__ int bin_of(int n) const { return min(max(top - n, 0), kChunkBins - 1); }
  __device__ __forceinline__ int bin(float x) const {
    int n;
    split(x, &n);
    return bin_of(n);
  }
  __device__ __forceinline__ uint64_t mass(float x, const double* sixteenths, int* bin) const {
    int n;
    const double f = split(x, &n);
    double p = 1.4676329855091502e-07;
    p = __builtin_fma(p, f, 1.3551125679403628e-05);
    p = __builtin_fma(p, f, 0.0009383847927372583);
    p = __builtin_fma(p, f, 0.043321698775062194);
    p = __builtin_fma(p, f, 1.0);
    *bin = bin_of(n);
    return whole_of(__builtin_ldexp(p * sixteenths[n & 15], n >> 4));
  }
  // (A number below 2^52 plus 2^52 has its nearest whole number in the lower bits.)
  __device__ __forceinline__ static uint64_t whole_of(double w) { return __builtin_bit_cast(uint64_t, w + 4503599627370496.0) & ((1ull << 52) - 1); }
};
// 2^(i / 16), i < 16.
__device__ __forceinline__ void fill_sixteenths(double* to) {
  if (threadIdx.x < 16) to[threadIdx.x] = exp2((double)threadIdx.x * 0.0625);
}

// Numbers in the order of floats (no NaN, no -0), and back.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_order(uint32_t k) { return sample_bits(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct SampleShared {
  unsigned long long mass[kSampleBins];  // of a bin; of a word of the list
  alignas(16) unsigned long long list[kSampleList];  // order of x, then falling index, of a word
  uint32_t count[kSampleBins];
  unsigned long long wave_mass[kSampleWaves];
  uint32_t wave_count[kSampleWaves];
  float wave_lo[kSampleWaves], wave_hi[kSampleWaves];
  int32_t wave_i[kSampleWaves];
  int32_t bin, listed, pieces, some;  // (`some`: chunks)
  float cut_x;
  int32_t cut_i;
  unsigned long long above;
  double chunk_power[kChunks], sixteenths[16];
  int32_t chunk_down[kChunks];
  unsigned long long chunk_kept[kChunks];
  uint32_t wave_chunk[kChunks];
};

enum RowKind { kRowOfOne, kRowOfChunks, kRowLong };  // one chunk or less: fixed units; up to kChunks of them; without a digest
template <int DT, RowKind KIND>
struct Sampler {
  static constexpr int E = SampleRow<DT>::E, kMostBits = KIND == kRowLong ? 60 : 51;
  SampleShared& s;
  SampleRow<DT> row;
  int tid, lane, wave;
  float top;       // the largest logit
  double c;        // log2(e) / T
  double inv_t;
  int row_bits;    // of a mass behind the point, unless kRowOfOne
  float cut_x;     // words below (cut_x, cut_i) have been dropped
  int32_t cut_i;

  // 2^t = 2^n 2^f: n + f = t with |f| <= 1/2, 2^f = 1 + f p(f) with p of degree 7 through the values at the
  // Chebyshev nodes of the interval (relative error 2.2e-12, at top exactly 1).
  __device__ __forceinline__ static double fraction(double t, int* n) {
    const double whole = __builtin_rint(t), f = t - whole;
    double p = 1.325080551750225e-06;
    p = __builtin_fma(p, f, 1.5303700711365693e-05);
    p = __builtin_fma(p, f, 0.00015403475186530786);
    p = __builtin_fma(p, f, 0.0013333478473685416);
    p = __builtin_fma(p, f, 0.00961812913523614);
    p = __builtin_fma(p, f, 0.055504109063258665);
    p = __builtin_fma(p, f, 0.24022650695888503);
    p = __builtin_fma(p, f, 0.6931471805568324);
    p = __builtin_fma(p, f, 1.0);
    *n = (int)fmax(whole, -2000.0);
    return p;
  }
  __device__ __forceinline__ double weight(float x) const {
    int n;
    const double p = fraction(((double)x - (double)top) * c, &n);
    return x == top ? 1.0 : __builtin_ldexp(p, n);
  }
  __device__ __forceinline__ uint64_t mass(float x) const {
    int n;
    const double p = fraction(((double)x - (double)top) * c, &n);
    // (Of what is no word, or stands beside infinite ones, t may be -inf or a NaN: it has no mass whatever comes out.)
    uint64_t m;
    const int bits = KIND == kRowOfOne ? kChunkBits : row_bits;
    if constexpr (KIND == kRowLong) m = ChunkScale::whole_of(p * 0x1p51) << 9 >> min(60 - n - bits, 63);  // (up to 2^60, rounded down)
    else m = ChunkScale::whole_of(__builtin_ldexp(p, n + bits));
    return x == top ? 1ull << bits : x > -INFINITY ? m : 0;
  }
  // So many bits that the masses of all words add up to at most 2^61: up to 60, or 51 where a mass comes out of the lower bits of a
  // double (with 64-bit shifts 128 rows of 131072 words, top-k 3000, took 243 us instead of 216).  The sum of all w, in the same order in
  // every run, decides it, in 32 bits: an eighth is added for what 2^20 additions in a lane lose (2^20 steps of 2^-24) and for the exponentials.
  __device__ __forceinline__ int bits_of_row() {
    float sum = 0.0f;
    row.each([&](const float* x, int) {
#pragma unroll
      for (int e = 0; e < E; ++e) sum += x[e] == top ? 1.0f : x[e] > -INFINITY ? __builtin_amdgcn_exp2f((float)(((double)x[e] - (double)top) * c)) : 0.0f;
    });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    __syncthreads();
    if (lane == 0) s.wave_hi[wave] = sum;
    __syncthreads();
    sum = 0.0f;
    for (int w = 0; w < kSampleWaves; ++w) sum += s.wave_hi[w];
    __syncthreads();
    return min(61 - __builtin_amdgcn_frexp_expf(1.125f * sum), kMostBits);
  }
  // The same from the chunks' masses, if they all have one; otherwise 0.  (Relative to the whole octave below the largest word: up to
  // twice the sum.)
  __device__ __forceinline__ int bits_of_chunks(const SampleChunk* chunks, int n_chunks, int mode) const {
    const SampleChunk& mine = chunks[min(lane, n_chunks - 1)];
    const bool own = lane < n_chunks;
    if (mode == kDigestList || __any(own && mine.listed < 0)) return 0;
    double sum = own && mine.total != 0 ? __builtin_ldexp((double)mine.total, (int)fmax(mine.power - floor((double)top * c), -2000.0) - kChunkBits) : 0.0;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    return min(61 - __builtin_amdgcn_frexp_exp(sum), kMostBits);
  }
  __device__ __forceinline__ bool stays(float x, int i) const { return x > cut_x || (x == cut_x && i <= cut_i); }
  __device__ __forceinline__ static unsigned long long entry(float x, int i) { return (unsigned long long)order_of(x) << 32 | (uint32_t)~i; }
  __device__ __forceinline__ static float entry_x(unsigned long long e) { return of_order((uint32_t)(e >> 32)); }
  __device__ __forceinline__ static int entry_i(unsigned long long e) { return (int)~(uint32_t)e; }

  // Sum over the workgroup of all threads before this one; `total` of all.
  __device__ __forceinline__ uint64_t block_before(uint64_t v, uint64_t* total) {
    const uint64_t run = wave_scan(v);
    __syncthreads();
    if (lane == 63) s.wave_mass[wave] = run;
    __syncthreads();
    uint64_t before = run - v, all = 0;
    for (int w = 0; w < kSampleWaves; ++w) {
      if (w < wave) before += s.wave_mass[w];
      all += s.wave_mass[w];
    }
    *total = all;
    return before;
  }

  // The list in falling order; `n` words of it (no two alike), the rest up to a power of two becomes 0.  A few are put where the number of larger
  // ones says; many go through a bitonic network, whose steps over less than a wave's 128 words need no barrier.
  __device__ __forceinline__ void sort(int n) {
    if (n <= kSampleRank) {
      __syncthreads();
      unsigned long long own = 0;
      int place = 0;
      if (tid < n) {
        own = s.list[tid];
        if (tid == 0 && (n & 1)) s.list[n] = 0;
      }
      __syncthreads();
      if (tid < n) {
#pragma unroll 8
        for (int j = 0; j < (n + 1) / 2; ++j) {
          const ulonglong2 o = reinterpret_cast<const ulonglong2*>(s.list)[j];
          place += (o.x > own) + (o.y > own);
        }
      }
      __syncthreads();
      if (tid < n) s.list[place] = own;
      __syncthreads();
      return;
    }
    int size = 2 * kSampleRank;  // (two of a wave's pairs of 128 words at least)
    while (size < n) size <<= 1;
    for (int i = n + tid; i < size; i += kSampleThreads) s.list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        const int i = 2 * tid - (tid & (j - 1));  // the lower of the thread's pair
        if (i < size) {
          const unsigned long long a = s.list[i], b = s.list[i + j];
          if ((a < b) == ((i & k) == 0)) s.list[i] = b, s.list[i + j] = a;
        }
        if (j > 64 || (j == 1 && k >= 128)) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      }
    __syncthreads();
  }

  // Finds the last word that stays and makes it the cut: the first `k` words (BY_MASS false), or those before which less than top_p of
  // the mass of what is left lies.
  template <bool BY_MASS>
  __device__ __forceinline__ void cut(uint32_t k, float top_p, float lowest) {
    float hi = top, lo = fmaxf(lowest, BY_MASS ? top - (float)(20.0 / inv_t) : top - 32.0f);
    float below = INFINITY;          // words of this interval are at most this (and at least `from` after the first level)
    float from = -INFINITY;
    uint64_t above = 0, goal = 0;    // mass, or count, in front of the interval; what the last word brings it to, at least
    if (!BY_MASS) goal = k;
#pragma unroll 1
    for (int level = 0;; ++level) {
      const double width = (double)hi - (double)lo;
      const double inv64 = kSampleBins / (width > 0 ? width : 1.0);
      const float inv32 = (float)inv64;
      // Falls with x: the same expression finds a word's bin when it is counted and when it is listed.
      auto bin_of = [&](float x) -> int {
        if (level == 0) return (int)fminf((hi - x) * inv32, (float)(kSampleBins - 1));
        return (int)fmin(((double)hi - (double)x) * inv64, (double)(kSampleBins - 1));
      };
      auto inside = [&](float x, int i) { return x <= below && x >= from && x > -INFINITY && stays(x, i); };
      for (int i = tid; i < kSampleBins; i += kSampleThreads) {
        if (BY_MASS) s.mass[i] = 0;
        else s.count[i] = 0;
      }
      if (tid == 0) s.listed = 0;
      __syncthreads();
      uint64_t rest = 0;  // of the last bin: what does not come by an atomic
      row.each([&](const float* x, int i0) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if constexpr (BY_MASS) {
            const uint64_t m = mass(x[e]);
            if (inside(x[e], i0 + e)) {
              const int at = bin_of(x[e]);
              if (at == kSampleBins - 1) rest += m;
              else atomicAdd(&s.mass[at], (unsigned long long)m);
            }
          } else if (inside(x[e], i0 + e)) {
            const int at = bin_of(x[e]);
            if (at == kSampleBins - 1) ++rest;
            else atomicAdd(&s.count[at], 1u);
          }
        }
      });
      rest = wave_total(rest);
      if (lane == 0 && rest != 0) {
        if (BY_MASS) atomicAdd(&s.mass[kSampleBins - 1], (unsigned long long)rest);
        else atomicAdd(&s.count[kSampleBins - 1], (uint32_t)rest);
      }
      __syncthreads();
      // Running sums over the bins, two a thread, from above.
      const uint64_t v0 = BY_MASS ? s.mass[2 * tid] : s.count[2 * tid], v1 = BY_MASS ? s.mass[2 * tid + 1] : s.count[2 * tid + 1];
      uint64_t total;
      const uint64_t before = above + block_before(v0 + v1, &total);
      if (BY_MASS && level == 0) {
        // "less than top_p of the mass before it" in whole numbers: before < ceil(top_p * mass).
        goal = top_goal(top_p, total);
      }
      if (goal > above + total) return;  // (fewer than k words are left: infinite ones)
      if (before < goal && goal <= before + v0) s.bin = 2 * tid, s.above = before;
      else if (before + v0 < goal && goal <= before + v0 + v1) s.bin = 2 * tid + 1, s.above = before + v0;
      __syncthreads();
      const int at = s.bin;
      above = s.above;
      // The members of the bin: listed if they are few, and their lowest and highest value.
      float low = INFINITY, high = -INFINITY;
      row.each([&](const float* x, int i0) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (inside(x[e], i0 + e) && bin_of(x[e]) == at) {
            low = fminf(low, x[e]), high = fmaxf(high, x[e]);
            const int j = atomicAdd(&s.listed, 1);
            if (j < kSampleList) s.list[j] = entry(x[e], i0 + e);
          }
      });
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) low = fminf(low, __shfl_xor(low, o)), high = fmaxf(high, __shfl_xor(high, o));
      if (lane == 0) s.wave_lo[wave] = low, s.wave_hi[wave] = high;
      __syncthreads();
      for (int w = 0; w < kSampleWaves; ++w) low = fminf(low, s.wave_lo[w]), high = fmaxf(high, s.wave_hi[w]);
      const int members = s.listed;
      if (members <= kSampleList) {
        sort(members);
        const int j0 = 2 * tid, j1 = j0 + 1;
        const unsigned long long e0 = j0 < members ? s.list[j0] : 0, e1 = j1 < members ? s.list[j1] : 0;
        const uint64_t m0 = j0 >= members ? 0 : BY_MASS ? mass(entry_x(e0)) : 1, m1 = j1 >= members ? 0 : BY_MASS ? mass(entry_x(e1)) : 1;
        uint64_t all;
        const uint64_t front = above + block_before(m0 + m1, &all);
        if (front < goal && goal <= front + m0) s.cut_x = entry_x(e0), s.cut_i = entry_i(e0);
        else if (front + m0 < goal && goal <= front + m0 + m1) s.cut_x = entry_x(e1), s.cut_i = entry_i(e1);
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

  // The draw from the digests of a row's chunks, if they settle it (to every thread alike).
  // `early`: what the wave's chunk's list, or bins, hold in the places 64 i + lane.
  __device__ __forceinline__ bool by_chunks(const SampleChunk* chunks, int n_chunks, unsigned long long (&early)[kChunkBins / 64], int mode, int top_i, uint32_t top_k, float top_p, double least,
                                            float u, int64_t* token) {
    const SampleChunk& mine = chunks[min(lane, n_chunks - 1)];
    const int own = lane < n_chunks ? mine.listed : 0;
    if (__any(own < 0)) return false;
    if (mode == kDigestList) {
      // The candidates, through LDS where all of them fit; those that the largest top_k reach go on the list, by the bins of their distance.
      const uint32_t end = wave_scan((uint32_t)own), all = wave_last(end);
      if (wave == 0) s.wave_chunk[lane] = end - own;
      for (int i = tid; i < kSampleBins; i += kSampleThreads) s.count[i] = 0;
      if (tid == 0) s.listed = 0, s.bin = kSampleBins;
      __syncthreads();
      const float inv = (float)(64.0 * c);  // (sixty-fourths of an octave of w)
      auto bin_of = [&](unsigned long long e) { return (int)fminf((top - entry_x(e)) * inv, (float)(kSampleBins - 1)); };
      const bool staged = all <= kSampleBins;
      for (int k = wave; k < n_chunks; k += kSampleWaves) {
        const int many = __shfl(own, k), at = (int)s.wave_chunk[k];
        for (int j = lane; j < many; j += 64) {
          const unsigned long long e = k == wave && j < 64 ? early[0] : chunks[k].list[j];
          if (staged) s.mass[at + j] = e;
          atomicAdd(&s.count[bin_of(e)], 1u);
        }
      }
      __syncthreads();
      const uint32_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
      uint64_t total;
      const uint64_t before = block_before(c0 + c1, &total);
      if (before < top_k && top_k <= before + c0) s.bin = 2 * tid;
      else if (before + c0 < top_k && top_k <= before + c0 + c1) s.bin = 2 * tid + 1;
      __syncthreads();
      const int last = s.bin;  // (fewer than top_k: all of them)
      auto put = [&](unsigned long long e) {
        if (bin_of(e) <= last) {
          const int at = atomicAdd(&s.listed, 1);
          if (at < kSampleList) s.list[at] = e;
        }
      };
      if (staged) {
        for (int i = tid; i < (int)all; i += kSampleThreads) put(s.mass[i]);
      } else {
        for (int k = wave; k < n_chunks; k += kSampleWaves) {
          const int many = __shfl(own, k);
          for (int j = lane; j < many; j += 64) put(chunks[k].list[j]);
        }
      }
      __syncthreads();
      const int n = s.listed;
      if (n > kSampleList) return false;
      if (n <= 64) {
        if (wave == 0) on_wave(n, top_k, top_p, least, u, token);
        return true;
      }
      return on_list(n, (int)top_k >= n, top_k, top_p, least, u, 0, token);
    }

    if (at_end(u)) return false;  // (which word is the first or last with any weight, masses do not tell)
    // Every wave has the chunks in its lanes.  The row counts octaves from the largest power down, and masses in units in which all
    // of it comes to between 2^60 and 2^61, by `units` octaves above those of the chunk with the largest power.
    const bool words = lane < n_chunks && mine.total != 0;
    const double own_power = words ? mine.power : -INFINITY;
    double power_of_row = own_power;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) power_of_row = fmax(power_of_row, __shfl_xor(power_of_row, o));
    fill_sixteenths(s.sixteenths);
    const int down = words ? (int)fmin(power_of_row - own_power, 80.0) : 80;  // (of what lies 80 octaves below, nothing is left)
    const uint64_t total = words ? mine.total : 0;
    double sum_of_row = __builtin_ldexp((double)total, -down);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum_of_row += __shfl_xor(sum_of_row, o);
    const int units = __builtin_amdgcn_frexp_exp(sum_of_row) - 61;  // -12 to 8
    auto to_row = [&](uint64_t m, int down) { return down + units >= 0 ? m >> min(down + units, 63) : m << -(down + units); };
    if (wave == 0) s.chunk_power[lane] = mine.power, s.chunk_down[lane] = down, s.chunk_kept[lane] = total;
    int last = kChunkBins;                   // words of bins before it stay, and those of it down to the cut
    if (mode == kDigestBins) {
      const uint64_t all = wave_total(to_row(total, down));
      const uint64_t goal = top_p < 1.0f ? top_goal(top_p, all) : ~0ull;
      // The row's bins: a wave adds those of a chunk.
      if (tid < kChunkBins) s.mass[tid] = 0;
      if (tid == 0) s.bin = kChunkBins - 1, s.listed = 0, s.pieces = 0, s.some = 0, s.cut_x = INFINITY, s.cut_i = -1;
      __syncthreads();
      auto fetch = [&](int k) {
#pragma unroll
        for (int i = 0; i < kChunkBins / 64; ++i) early[i] = chunks[k].bins[64 * i + lane];
      };
      for (int k = wave; k < n_chunks; k += kSampleWaves) {
        const int octaves = s.chunk_down[k];
        if (s.chunk_kept[k] == 0) continue;
        if (k != wave) fetch(k);  // (those are there already)
#pragma unroll
        for (int i = 0; i < kChunkBins / 64; ++i) {
          const int at = 64 * i + lane;  // (the last one is not in use)
          if (at < kChunkBins - 1 && at + 16 * octaves < kChunkBins - 1) atomicAdd(&s.mass[at + 16 * octaves], (unsigned long long)to_row(early[i], octaves));
        }
      }
      __syncthreads();
      const uint64_t v = tid < kChunkBins ? s.mass[tid] : 0;
      uint64_t sum;
      const uint64_t before = block_before(v, &sum);
      if (tid < kChunkBins - 1 && before < goal && goal <= before + v) s.bin = tid;
      __syncthreads();
      last = s.bin;
      if (least > 0.0) {  // the bin of the least weight, but none before the largest word's, which stays (least may be above 1)
        const double t = power_of_row - ((double)top * c + log2(least));
        const int of_least = t <= 0.0 ? 0 : (int)fmin(__builtin_rint(16.0 * t), (double)(kChunkBins - 1));
        last = min(last, max(of_least, ChunkScale(c, power_of_row).bin(top)));
      }
      if (last == kChunkBins - 1) return false;
      if (tid == last) s.above = before;
      // What a chunk has in the bins before it, and which chunks have words of it.
      for (int k = wave; k < n_chunks; k += kSampleWaves) {
        const int bins = s.chunk_kept[k] == 0 ? 0 : last - 16 * s.chunk_down[k];
        uint64_t m = 0;
        if (n_chunks > kSampleWaves) fetch(k);
#pragma unroll
        for (int i = 0; i < kChunkBins / 64; ++i) m += 64 * i + lane < bins ? early[i] : 0;
        m = wave_total(m);
        bool some = false;
#pragma unroll
        for (int i = 0; i < kChunkBins / 64; ++i) some |= bins >= 0 && 64 * i + lane == bins && s.chunk_kept[k] != 0 && early[i] != 0;
        if (lane == 0) s.mass[k] = m;
        if (some) s.wave_chunk[atomicAdd(&s.some, 1)] = (uint32_t)k;
      }
      __syncthreads();
      const int some = s.some;
      // The words of the bin.  (First by a range of x, a little too wide, and first the pieces that have any: a few words of a wave's
      // would keep all of it busy with each.  Without, 1000 of 131072 words took 4 us longer.)
      const double wide = 1e-6 * (fabs(power_of_row) + 32.0);
      const float x_hi = (float)((power_of_row - (last - 0.5) / 16.0 + wide) / c), x_lo = (float)((power_of_row - (last + 0.5) / 16.0 - wide) / c);
      constexpr int PIECES = kChunkWords / (kSampleThreads * E), BATCH = 4 / PIECES;
#pragma unroll 1
      for (int c0 = 0; c0 < some; c0 += BATCH) {
        u32x4 w[BATCH * PIECES];
        int at[BATCH * PIECES];
#pragma unroll
        for (int p = 0; p < BATCH * PIECES; ++p) {
          at[p] = (int)s.wave_chunk[min(c0 + p / PIECES, some - 1)] * kChunkWords + (p % PIECES * kSampleThreads + tid) * E;
          w[p] = row.load(at[p]);
        }
#pragma unroll
        for (int p = 0; p < BATCH * PIECES; ++p) {
          float x[E];
          row.numbers(w[p], x);
          bool any = false;
#pragma unroll
          for (int e = 0; e < E; ++e) any |= (x[e] >= x_lo) & (x[e] <= x_hi);
          if (any && c0 + p / PIECES < some) {
            const int j = atomicAdd(&s.pieces, 1);
            if (j < kSampleBins) s.count[j] = (uint32_t)at[p];
          }
        }
      }
      __syncthreads();
      const int pieces = s.pieces;
      if (pieces > kSampleBins) return false;
      for (int j = tid; j < pieces; j += kSampleThreads) {
        const int i0 = (int)s.count[j];
        float x[E];
        row.numbers(row.load(i0), x);
#pragma unroll
        for (int e = 0; e < E; ++e)
          if ((x[e] >= x_lo) & (x[e] <= x_hi) & (x[e] > -INFINITY)) {
            const int at = atomicAdd(&s.listed, 1);
            if (at < kSampleList) s.list[at] = entry(x[e] + 0.0f, i0 + e);
          }
      }
      __syncthreads();
      // Of those the ones that lie in the bin.
      const int range = s.listed;
      if (range > kSampleList) return false;
      unsigned long long member[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (tid + i * kSampleThreads < range) {
          const unsigned long long e = s.list[tid + i * kSampleThreads];
          const int k = entry_i(e) / kChunkWords;
          if (ChunkScale(c, s.chunk_power[k]).bin(entry_x(e)) + 16 * s.chunk_down[k] == last) member[i] = e;
        }
      __syncthreads();
      if (tid == 0) s.listed = 0;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (member[i] != 0) s.list[atomicAdd(&s.listed, 1)] = member[i];
      __syncthreads();
      const int n = s.listed;
      const uint64_t above = s.above;
      if (wave == 0 && lane < n_chunks) s.chunk_kept[lane] = s.mass[lane];
      sort(n);
      const int j0 = 2 * tid, j1 = j0 + 1;
      const unsigned long long e0 = j0 < n ? s.list[j0] : 0, e1 = j1 < n ? s.list[j1] : 0;
      const int k0 = j0 < n ? entry_i(e0) / kChunkWords : 0, k1 = j1 < n ? entry_i(e1) / kChunkWords : 0;
      int bin;
      const uint64_t m0 = j0 < n ? ChunkScale(c, s.chunk_power[k0]).mass(entry_x(e0), s.sixteenths, &bin) : 0;
      const uint64_t m1 = j1 < n ? ChunkScale(c, s.chunk_power[k1]).mass(entry_x(e1), s.sixteenths, &bin) : 0;
      const uint64_t r0 = to_row(m0, s.chunk_down[k0]), r1 = to_row(m1, s.chunk_down[k1]);
      uint64_t of_list, kept;
      const uint64_t front = above + block_before(r0 + r1, &of_list);
      block_before((uint64_t)(j0 < n && front < goal && (weight(entry_x(e0)) >= least || entry_i(e0) == top_i)) +
                       (j1 < n && front + r0 < goal && (weight(entry_x(e1)) >= least || entry_i(e1) == top_i)), &kept);
      if (j0 < (int)kept) atomicAdd(&s.chunk_kept[k0], (unsigned long long)m0);
      if (j1 < (int)kept) atomicAdd(&s.chunk_kept[k1], (unsigned long long)m1);
      if (j0 == (int)kept - 1) s.cut_x = entry_x(e0), s.cut_i = entry_i(e0);
      if (j1 == (int)kept - 1) s.cut_x = entry_x(e1), s.cut_i = entry_i(e1);
    }
    __syncthreads();
    // The chunk that the draw falls into.
    const uint64_t kept = lane < n_chunks ? s.chunk_kept[lane] : 0, own_units = to_row(kept, down);
    const uint64_t run = wave_scan(own_units), all = wave_last(run);
    if (all == 0) return false;  // (the largest word stays: this does not happen, and without it there would be no chunk to find)
    const uint64_t of_row = goal_of(u, all);
    int k = __ffsll((unsigned long long)__ballot(of_row < run)) - 1;
    uint64_t goal = of_row - __shfl((unsigned long long)(run - own_units), k);
    const int by = s.chunk_down[k] + units;  // (below 62: the chunk has a unit of the row's)
    goal = by >= 0 ? goal << by : goal >> -by;
    k = __builtin_amdgcn_readfirstlane(k);
    const ChunkScale scale(c, s.chunk_power[k]);
    const int bin_shift = 16 * s.chunk_down[k];
    cut_x = s.cut_x, cut_i = s.cut_i;
    constexpr int EACH = kChunkWords / kSampleThreads;  // neighbouring words of a thread
    const int i0 = k * kChunkWords + tid * EACH;
    float x[EACH];
#pragma unroll
    for (int p = 0; p < EACH; p += E) row.unpack(row.load(i0 + p), x + p);
    uint64_t m[EACH], sum = 0;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      int bin;
      m[e] = scale.mass(x[e], s.sixteenths, &bin);
      bin += bin_shift;
      if (last < kChunkBins && !(bin < last || (bin == last && stays(x[e], i0 + e)))) m[e] = 0;
      sum += m[e];
    }
    uint64_t of_chunk, at = block_before(sum, &of_chunk);
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      if (at <= goal && goal < at + m[e]) *token = i0 + e;
      at += m[e];
    }
    return true;
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

  // u * all as the whole number that the running sum has to exceed, for u between 0 and 1.
  __device__ __forceinline__ static uint64_t goal_of(float u, uint64_t all) { return part_of(all, u, false); }
  // Another u takes the first word with any weight, or the last one (1 and more, NaN): the largest `rank` among the candidates, 0 or more.
  __device__ __forceinline__ static bool at_end(float u) { return !(u > 0.0f && u < 1.0f); }
  __device__ __forceinline__ static int rank(float u, int i) { return u < 1.0f ? 0x7fffffff - i : i; }
  __device__ __forceinline__ int rank_of(float u, unsigned long long e) const { return weight(entry_x(e)) > 0.0 ? rank(u, entry_i(e)) : -1; }
  __device__ __forceinline__ static int wave_best(int own) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) own = max(own, __shfl_xor(own, o));
    return own;
  }
  __device__ __forceinline__ void take_end(float u, int own, int64_t* token) {
    own = wave_best(own);
    __syncthreads();
    if (lane == 0) s.wave_i[wave] = own;
    __syncthreads();
    for (int w = 0; w < kSampleWaves; ++w) own = max(own, s.wave_i[w]);
    if (tid == 0) *token = rank(u, own);  // (its own inverse)
  }
  __device__ __forceinline__ static uint64_t top_goal(float top_p, uint64_t all) {
    const uint64_t goal = top_p > 0.0f ? part_of(all, top_p, true) : 1;
    return goal < 1 ? 1 : goal;
  }

  // Everything on a list of the largest words, if they are enough: whether they were (to every thread alike).  `mine`: this thread's
  // largest word.  top_k: 0 or at most kSampleTopK.
  __device__ __forceinline__ bool by_list(float mine, uint32_t words, uint32_t top_k, float top_p, double least, float u, int64_t* token) {
    const uint32_t aim = top_k > 0 ? top_k : kSampleTopK;
    // The value that `aim` threads reach: the lower end of its bin among the threads' largest.
    const float lo = top - (float)(32.0 / (top_k > 0 ? 1.0 : inv_t));
    const float inv = (float)kSampleBins / (top - lo);
    for (int i = tid; i < kSampleBins; i += kSampleThreads) s.count[i] = 0;
    if (tid == 0) s.listed = 0, s.bin = -1;
    __syncthreads();
    // (a width that is 0 or infinite sends all of them to one bin: still the lower end of a bin)
    const int bin = mine > -INFINITY ? (int)fminf((top - mine) * inv, (float)(kSampleBins - 1)) : kSampleBins;
    if (bin < kSampleBins) atomicAdd(&s.count[bin], 1u);
    __syncthreads();
    const uint64_t c0 = s.count[2 * tid], c1 = s.count[2 * tid + 1];
    uint64_t threads;
    const uint64_t before = block_before(c0 + c1, &threads);
    if (before < aim && aim <= before + c0) s.bin = 2 * tid;
    else if (before + c0 < aim && aim <= before + c0 + c1) s.bin = 2 * tid + 1;
    __syncthreads();
    float least_x = INFINITY;
    if (s.bin < 0) {
      least_x = -INFINITY;  // fewer threads have words: all of them
    } else {
      if (bin <= s.bin) least_x = mine;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) least_x = fminf(least_x, __shfl_xor(least_x, o));
      if (lane == 0) s.wave_lo[wave] = least_x;
      __syncthreads();
      for (int w = 0; w < kSampleWaves; ++w) least_x = fminf(least_x, s.wave_lo[w]);
    }
    const bool weigh = top_k == 0 && top_p < 1.0f;
    uint64_t all_mass = 0;
    row.each([&](const float* x, int i0) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (weigh) all_mass += mass(x[e]);
        if (x[e] >= least_x && x[e] > -INFINITY) {
          const int j = atomicAdd(&s.listed, 1);
          if (j < kSampleList) s.list[j] = entry(x[e], i0 + e);
        }
      }
    });
    __syncthreads();
    const int n = s.listed;
    if (n > kSampleList) return false;
    uint64_t total = 0;
    if (weigh) block_before(all_mass, &total);
    return on_list(n, (uint32_t)n == words, top_k, top_p, least, u, weigh ? total : 0, token);
  }

  // The lanes' numbers in falling order (no two alike but 0): through LDS, where a lane finds how many are larger.
  __device__ __forceinline__ unsigned long long wave_sort(unsigned long long own) {
    s.list[lane] = own;
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    int place = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const ulonglong2 o = reinterpret_cast<const ulonglong2*>(s.list)[j];
      place += (o.x > own || (o.x == own && 2 * j < lane)) + (o.y > own || (o.y == own && 2 * j + 1 < lane));
    }
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    s.list[place] = own;
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    return s.list[lane];
  }
  // on_list for a list of up to 64 words that is long enough, in one wave.
  __device__ __forceinline__ void on_wave(int n, uint32_t top_k, float top_p, double least, float u, int64_t* token) {
    const unsigned long long e = wave_sort(lane < n ? s.list[lane] : 0);
    const bool first = lane < min((int)top_k, n);
    const uint64_t m = first ? mass(entry_x(e)) : 0, run = wave_scan(m), of_list = wave_last(run);
    const uint64_t goal = top_p < 1.0f ? top_goal(top_p, of_list) : ~0ull;
    const int kept = __popcll(__ballot(lane == 0 || (first && run - m < goal && weight(entry_x(e)) >= least)));
    if (at_end(u)) {
      const int best = wave_best(lane < kept ? rank_of(u, e) : -1);
      if (lane == 0) *token = rank(u, best);
      return;
    }
    const uint64_t own = lane < kept ? m : 0, aim = goal_of(u, wave_total(own));
    const unsigned long long by_index = wave_sort(lane < kept ? (unsigned long long)(uint32_t)~entry_i(e) << 32 | (uint32_t)lane : 0);
    const uint64_t here = lane < kept ? __shfl((unsigned long long)own, (int)(by_index & 63)) : 0, end = wave_scan(here);
    if (end - here <= aim && aim < end) *token = (int)~(uint32_t)(by_index >> 32);
  }

  // The draw from a list of the n largest words.  `complete`: there are no others; `total`: the mass of all words, or 0: that of the first
  // top_k counts.  Returns whether the list was long enough.
  __device__ __forceinline__ bool on_list(int n, bool complete, uint32_t top_k, float top_p, double least, float u, uint64_t total, int64_t* token) {
    sort(n);
    const int j0 = 2 * tid, j1 = j0 + 1;
    const int first = top_k > 0 ? min((int)top_k, n) : n;  // of the list
    const unsigned long long e0 = j0 < first ? s.list[j0] : 0, e1 = j1 < first ? s.list[j1] : 0;
    const uint64_t m0 = j0 < first ? mass(entry_x(e0)) : 0, m1 = j1 < first ? mass(entry_x(e1)) : 0;
    uint64_t of_list;
    uint64_t front = block_before(m0 + m1, &of_list);
    if (total == 0) total = of_list;
    const uint64_t goal = top_p < 1.0f ? top_goal(top_p, total) : ~0ull;
    uint64_t kept;
    block_before((uint64_t)(j0 < first && (j0 == 0 || (front < goal && weight(entry_x(e0)) >= least))) +
                     (j1 < first && front + m0 < goal && weight(entry_x(e1)) >= least), &kept);
    const bool in0 = j0 < (int)kept, in1 = j1 < (int)kept;
    // All of the list stays, and words that are not on it might: it was too short.
    if (kept == (uint64_t)n && !complete && !(top_k > 0 && (int)top_k <= n) && of_list < goal) return false;
    if (at_end(u)) {
      take_end(u, max(in0 ? rank_of(u, e0) : -1, in1 ? rank_of(u, e1) : -1), token);
      return true;
    }
    uint64_t all;
    block_before((in0 ? m0 : 0) + (in1 ? m1 : 0), &all);
    const uint64_t aim_mass = goal_of(u, all);
    // In the order of the indices.
    __syncthreads();
    if (in0) s.list[j0] = (unsigned long long)(uint32_t)~entry_i(e0) << 32 | (uint32_t)j0, s.mass[j0] = m0;
    if (in1) s.list[j1] = (unsigned long long)(uint32_t)~entry_i(e1) << 32 | (uint32_t)j1, s.mass[j1] = m1;
    __syncthreads();
    sort((int)kept);
    const unsigned long long f0 = j0 < (int)kept ? s.list[j0] : 0, f1 = j1 < (int)kept ? s.list[j1] : 0;
    const uint64_t g0 = j0 < (int)kept ? s.mass[(uint32_t)f0] : 0, g1 = j1 < (int)kept ? s.mass[(uint32_t)f1] : 0;
    front = block_before(g0 + g1, &all);
    if (front <= aim_mass && aim_mass < front + g0) *token = (int)~(uint32_t)(f0 >> 32);
    else if (front + g0 <= aim_mass && aim_mass < front + g0 + g1) *token = (int)~(uint32_t)(f1 >> 32);
    return true;
  }
};

// A chunk's words in registers, and what the row's settings will ask of it.
template <int DT>
__global__ void __launch_bounds__(kDigestThreads) sample_digest(SampleArgs a) {
  typedef Sampler<DT, kRowOfChunks> S;
  constexpr int E = SampleRow<DT>::E, ES = DT == LH_F32 ? 4 : 2, PIECES = kChunkWords / (kDigestThreads * E), WAVES = kDigestThreads / 64;
  __shared__ unsigned long long bins[kChunkBins];
  __shared__ unsigned long long wave_mass[WAVES];
  __shared__ float wave_top[WAVES];
  __shared__ int32_t wave_i[WAVES];
  __shared__ int32_t last_bin, listed;
  __shared__ double sixteenths[16];
  const int b = blockIdx.x / a.n_chunks, chunk = blockIdx.x % a.n_chunks, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int first = chunk * kChunkWords;
  const SampleRow<DT> row = {static_cast<const uint8_t*>(a.logits) + b * a.ld * ES, a.V, 0, 0, lane};
  float x[PIECES][E];
  {
    u32x4 raw[PIECES];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) raw[p] = row.load(first + (p * kDigestThreads + tid) * E);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) row.unpack(raw[p], x[p]);
  }
  const float temperature = a.o.temperature ? a.o.temperature[b] : a.o.temperature_all;
  const int top_k = a.o.top_k ? a.o.top_k[b] : a.o.top_k_all;
  const float top_p = a.o.top_p ? a.o.top_p[b] : a.o.top_p_all;
  const float min_p = a.o.min_p ? a.o.min_p[b] : a.o.min_p_all;
  SampleChunk& out = a.chunks[blockIdx.x];

  float top = -INFINITY;
  // f(x, index) for every word of the thread.
  auto each = [&](auto f) {
#pragma unroll
    for (int p = 0; p < PIECES; ++p)
#pragma unroll
      for (int e = 0; e < E; ++e) f(x[p][e], first + (p * kDigestThreads + tid) * E + e);
  };
  fill_sixteenths(sixteenths);
  each([&](float x, int) { top = fmaxf(top, x); });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (lane == 0) wave_top[wave] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) top = fmaxf(top, wave_top[w]);
  int mode = kDigestTotal;
  if (!(temperature > 0.0f) || top_k == 1) mode = kDigestTop;
  else if (top_k > 0 && top_k < a.V) mode = top_k <= kSampleTopK ? kDigestList : kDigestTotal;
  else if (top_p < 1.0f || min_p > 0.0f) mode = kDigestBins;
  int top_i = 0x7fffffff;
  if (mode == kDigestTop || min_p > 1.0f) {  // (otherwise nobody asks which it is)
    each([&](float x, int i) { top_i = x == top && i < top_i ? i : top_i; });
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top_i = min(top_i, __shfl_xor(top_i, o));
    if (lane == 0) wave_i[wave] = top_i;
  } else if (lane == 0) {
    wave_i[wave] = top_i;
  }
  // (The settings and the chunk's largest word are the same for the workgroup: all branches below are uniform.)
  // Left to the row's workgroup: an infinite word, and exponents so large that x c has no places behind the point.
  const double c = 1.0 / (double)temperature * 1.4426950408889634, exponent = (double)top * c;
  const bool some = top > -INFINITY, words = some && fabs(exponent) <= 0x1p40;
  const double power = words ? ceil(exponent) : 0.0;
  const ChunkScale scale(c, power);
  unsigned long long total = 0;
  int in_list = 0;
  if (words && mode == kDigestTotal) {
    each([&](float x, int) {
      int bin;
      total += scale.mass(x, sixteenths, &bin);
    });
  } else if (words && mode == kDigestBins) {
    for (int i = tid; i < kChunkBins; i += kDigestThreads) bins[i] = 0;
    __syncthreads();
    each([&](float x, int) {
      int bin;
      const uint64_t m = scale.mass(x, sixteenths, &bin);
      total += m;
      if (bin < kChunkBins - 1) atomicAdd(&bins[bin], (unsigned long long)m);
    });
    __syncthreads();
    for (int i = tid; i < kChunkBins - 1; i += kDigestThreads) out.bins[i] = bins[i];
  } else if (words && mode == kDigestList) {
    uint32_t* const counts = reinterpret_cast<uint32_t*>(bins);
    for (int i = tid; i < kChunkBins; i += kDigestThreads) counts[i] = 0;
    if (tid == 0) listed = 0, last_bin = kChunkBins - 1;  // fewer than top_k words: all of them
    __syncthreads();
    // (The chunk's own affair: the distance from its largest word in f32 will do, the same expression every time.)
    const float inv = (float)(16.0 * c);
    auto bin_of = [&](float x) { return (int)fminf((top - x) * inv, (float)(kChunkBins - 1)); };
    each([&](float x, int) {
      const int bin = bin_of(x);
      if (bin < kChunkBins - 1 && x > -INFINITY) atomicAdd(&counts[bin], 1u);
    });
    __syncthreads();
    static_assert(kDigestThreads >= kChunkBins, "a bin a thread");
    const uint32_t own = tid < kChunkBins ? counts[tid] : 0, run = wave_scan(own);
    if (lane == 63) wave_mass[wave] = run;
    __syncthreads();
    uint32_t before = run - own;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) before += w < wave ? (uint32_t)wave_mass[w] : 0;
    if (before < (uint32_t)top_k && (uint32_t)top_k <= before + own) last_bin = tid;
    __syncthreads();
    const int last = last_bin;
    each([&](float x, int i) {
      if (x > -INFINITY && bin_of(x) <= last) {
        const int j = atomicAdd(&listed, 1);
        if (j < kChunkList) out.list[j] = S::entry(x, i);
      }
    });
    __syncthreads();
    in_list = listed;
  }
  total = wave_total((uint64_t)total);
  __syncthreads();
  if (lane == 0) wave_mass[wave] = total;
  __syncthreads();
  if (tid == 0) {
    total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) total += wave_mass[w], top_i = min(top_i, wave_i[w]);
    out.power = power, out.total = total, out.top = top, out.top_i = top_i, out.mode = mode;
    out.listed = in_list > kChunkList || (some && !words) ? -1 : in_list;
  }
}

template <int DT, RowKind KIND>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(SampleArgs a) {
  __shared__ SampleShared s;
  constexpr int E = SampleRow<DT>::E, ES = DT == LH_F32 ? 4 : 2;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float temperature = a.o.temperature ? a.o.temperature[b] : a.o.temperature_all;
  const int top_k = a.o.top_k ? a.o.top_k[b] : a.o.top_k_all;
  const float top_p = a.o.top_p ? a.o.top_p[b] : a.o.top_p_all;
  const float min_p = a.o.min_p ? a.o.min_p[b] : a.o.min_p_all;
  const float u = a.uniform[b];

  const int pieces = (a.V + 64 * E - 1) / (64 * E), share = (pieces + kSampleWaves - 1) / kSampleWaves * (64 * E);
  const int begin = min(wave * (int64_t)share, (int64_t)a.V), end = min(begin + (int64_t)share, (int64_t)a.V);
  const SampleRow<DT> row = {static_cast<const uint8_t*>(a.logits) + b * a.ld * ES, a.V, begin, end, lane};

  const double inv_t = 1.0 / (double)temperature;
  const double least = min_p > 0.0f ? (double)min_p : 0.0;
  int bits = 0;
  if constexpr (KIND == kRowOfChunks) {
    const SampleChunk* chunks = a.chunks + (int64_t)b * a.n_chunks;
    const SampleChunk& mine = chunks[min(lane, a.n_chunks - 1)];
    unsigned long long early[kChunkBins / 64];  // (on the way before anything is known)
#pragma unroll
    for (int i = 0; i < kChunkBins / 64; ++i)
      if (i == 0 || a.may_bin) early[i] = chunks[min(wave, a.n_chunks - 1)].list[64 * i + lane];
    float top = mine.top;
    int top_i = mine.top_i;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const float x = __shfl_xor(top, o);
      const int i = __shfl_xor(top_i, o);
      if (x > top || (x == top && i < top_i)) top = x, top_i = i;
    }
    const int mode = __builtin_amdgcn_readfirstlane(mine.mode);
    if (top == -INFINITY || mode == kDigestTop) {
      if (tid == 0) a.tokens[b] = top == -INFINITY ? -1 : top_i;
      return;
    }
    Sampler<DT, KIND> f = {s, row, tid, lane, wave, top, inv_t * 1.4426950408889634, inv_t, kChunkBits, -INFINITY, -1};
    if ((top_k <= kSampleTopK || top_k >= a.V) && top < INFINITY && f.by_chunks(chunks, a.n_chunks, early, mode, top_i, (uint32_t)top_k, top_p, least, u, a.tokens + b)) return;
    if (top < INFINITY) bits = f.bits_of_chunks(chunks, a.n_chunks, mode);
    __syncthreads();
  }

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
  const float mine = top;
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

  Sampler<DT, KIND> f = {s, row, tid, lane, wave, top, inv_t * 1.4426950408889634, inv_t, kChunkBits, -INFINITY, -1};
  if (KIND != kRowOfOne) f.row_bits = bits > 0 ? bits : f.bits_of_row();
  const bool few = top_k > 0 && (uint32_t)top_k < words;
  if (top < INFINITY && (few ? top_k <= kSampleTopK : top_p < 1.0f || least > 0.0))
    if (f.by_list(mine, words, few ? top_k : 0, top_p, least, u, a.tokens + b)) return;
  __syncthreads();
  if (top == INFINITY) f.cut_x = INFINITY, f.cut_i = 0x7fffffff, lowest = top;  // only those
  if (few) f.template cut<false>((uint32_t)top_k, 0.0f, lowest);
  if (top_p < 1.0f) {
    __syncthreads();
    f.template cut<true>(0, top_p, lowest);
  }
  __syncthreads();

  auto keeps = [&](float x, int i) { return x > -INFINITY && f.stays(x, i) && (least == 0.0 || f.weight(x) >= least || i == top_i); };
  if (f.at_end(u)) {
    int best = -1;
    row.each([&](const float* x, int i0) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (keeps(x[e], i0 + e) && f.weight(x[e]) > 0.0) best = max(best, f.rank(u, i0 + e));
    });
    f.take_end(u, best, a.tokens + b);
    return;
  }

  // What stays: its mass by waves, and within a wave by up to 64 groups of pieces, lane g has group g's.
  auto left = [&](float x, int i) -> uint64_t {
    const uint64_t m = f.mass(x);
    return keeps(x, i) ? m : 0;
  };
  const int group = ((share / (64 * E) + 63) / 64) * 64 * E;  // words
  uint64_t of_group = 0, total = 0;
  row.each([&](const float* x, int i0) {
    uint64_t m = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) m += left(x[e], i0 + e);
    if (__any(m != 0)) {
      m = wave_total(m);
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
  const uint64_t goal = f.goal_of(u, all);
  if (!(before <= goal && goal < before + total)) return;
  const uint64_t run = wave_scan(of_group);
  const int g = __popcll(__ballot(before + run <= goal));  // groups that end at or before it
  before += g == 0 ? 0 : __shfl((unsigned long long)run, g - 1);
  for (int i = begin + g * group; i < end; i += 64 * E) {
    const int i0 = i + lane * E;
    float x[E];
    row.unpack(row.load(i0), x);
    uint64_t m[E], own = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) own += m[e] = left(x[e], i0 + e);
    const uint64_t sum = wave_scan(own);
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

static int sample_chunks(int64_t V) {
  const int64_t n = (V + kChunkWords - 1) / kChunkWords;
  return n < 2 || n > kChunks ? 0 : (int)n;
}

template <int DT>
static int launch_sample(const SampleArgs& a, int64_t B, hipStream_t s) {
  if (a.chunks) {
    LH_LAUNCH(sample_digest<DT>, dim3((unsigned)(B * a.n_chunks)), dim3(kDigestThreads), 0, s, a);
    if (const int rc = check_launch("sample_digest")) return rc;
  }
  if (a.chunks) LH_LAUNCH((sample_kernel<DT, kRowOfChunks>), dim3((unsigned)B), dim3(kSampleThreads), 0, s, a);
  else if (a.V <= kChunkWords) LH_LAUNCH((sample_kernel<DT, kRowOfOne>), dim3((unsigned)B), dim3(kSampleThreads), 0, s, a);
  else LH_LAUNCH((sample_kernel<DT, kRowLong>), dim3((unsigned)B), dim3(kSampleThreads), 0, s, a);
  return check_launch("sample");
}

extern "C" {

size_t lh_hip_sample_workspace_bytes(int64_t B, int64_t V) {
  return B <= 0 || B >= (1ll << 18) || V <= 0 ? 0 : ((size_t)B * sample_chunks(V) * sizeof(SampleChunk) + 255) / 256 * 256;
}

int lh_hip_sample(int64_t* tokens, const void* logits, const float* uniform, int64_t B, int64_t V, int64_t ld, int32_t dtype,
                  const lh_sample_opts* opts, void* workspace, size_t workspace_bytes, void* stream) {
  LH_REQUIRE(B >= 0 && B < (1ll << 18) && V >= 1 && V < (1ll << 30) && B * sample_chunks(V) < (1ll << 23),
             "lh_hip_sample: bad shape %lld x %lld (fewer than 2^18 rows, and 2^23 parts of 8192 words)", (long long)B, (long long)V);
  if (B == 0) return LH_OK;
  LH_REQUIRE(tokens && logits && uniform && opts, "lh_hip_sample: null pointer");
  LH_REQUIRE(B == 1 || ld >= V, "lh_hip_sample: rows overlap");
  LH_REQUIRE(dtype == LH_F32 || dtype == LH_BF16 || dtype == LH_F16, "lh_hip_sample: unsupported dtype %d", dtype);
  const size_t need = lh_hip_sample_workspace_bytes(B, V);
  LH_REQUIRE(need == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && workspace_bytes >= need),
             "lh_hip_sample: workspace too small or not 256-byte aligned: %zu of %zu bytes", workspace_bytes, need);
  SampleArgs a = {tokens, logits, uniform, ld, (int32_t)V, *opts, need ? static_cast<SampleChunk*>(workspace) : nullptr, sample_chunks(V), 0};
  a.may_bin = (opts->top_k || opts->top_k_all <= 0 || opts->top_k_all >= V) && (opts->top_p || opts->min_p || opts->top_p_all < 1.0f || opts->min_p_all > 0.0f);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == LH_F32) return launch_sample<LH_F32>(a, B, s);
  if (dtype == LH_BF16) return launch_sample<LH_BF16>(a, B, s);
  return launch_sample<LH_F16>(a, B, s);
}

}  // extern "C"
