// Which pages the sequences of a step hold, and where its packed tokens lie.
//
// The pages that no sequence has are a list whose last `n_free` entries' end is its top.  A step gives back the pages behind what
// the sequences' new lengths need (all of a sequence that ended), in the order of sequences and positions, and then takes what is
// missing from the top, sequence after sequence, while there is enough: both are running sums over the sequences.  So the result does not
// depend on which thread is first.
//
// One workgroup does the pages: a step moves few (4096 for 65536 new tokens in pages of 16), and the sums would need the others to wait for
// each other.  What bounds it is its chain of dependent loads (length, table, list) and barriers: 64 sequences of up to 1024 positions that get a
// token each take 6.7 us with 256 threads (8.6 with 1024), 1024 sequences that get 66432 tokens 19 us, of which 4 loops over about a thousand
// pages each, out of memory, are the larger part.  The tokens' positions and slots are its work too where they are few; otherwise a second
// launch finds each token's sequence by bisection of the running sums (5.2 us for those 66432).
#include "paged.h"
#include "wave_scan.h"

namespace lh {

struct PagesArgs {
  int32_t* table;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* counts;
  int32_t* new_lengths;   // may be `lengths`
  int32_t* free_pages;
  int32_t* n_free;
  int32_t* starts;        // [B + 1]
  int32_t* positions;     // [N]
  int64_t* slots;         // [N]
  int32_t B, P, F, N, size;
  FastDiv by_size;
};

constexpr int kPagesThreads = 1024;

// Running sum over the workgroup's threads, up to and with this one; *all: of all of them.  `sums`: one entry per wave, its own.
template <int WAVES>
__device__ __forceinline__ uint64_t pages_scan(uint64_t v, uint64_t* sums, uint64_t* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan(v);
  __syncthreads();  // (the sums of the call before have been read)
  if (lane == 63) sums[wave] = v;
  __syncthreads();
  uint64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += sums[w];
    total += sums[w];
  }
  *all = total;
  return before + v;
}

// The first of the n ascending sums that is above i.
template <typename T>
__device__ __forceinline__ int first_above(const T* sums, int n, T i) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (sums[mid] > i) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

struct PagesSequence {
  int32_t length, held, need;
  int32_t start;  // its first token
  int64_t count;
  bool fits;  // in the table, and its tokens, if it gets any, among the N
};

__device__ __forceinline__ int pages_for(const PagesArgs& a, int64_t length) {  // (0 <= length <= P size)
  const int whole = (int)a.by_size.div((uint32_t)length);
  return whole + (length > (int64_t)whole * a.size);
}
__device__ __forceinline__ bool pages_valid(const PagesArgs& a, int p) { return (uint32_t)p < (uint32_t)a.F; }

// How many pages sequence b holds: the entries before the first that is none.  In most calls as many as its length needs, which two
// loads at once confirm; otherwise by bisection.
__device__ __forceinline__ int pages_held(const PagesArgs& a, int b, int guess) {
  const int32_t* row = a.table + b * a.table_stride;
  const bool last = guess == 0 || pages_valid(a, row[max(guess - 1, 0)]), next = guess < a.P && pages_valid(a, row[min(guess, a.P - 1)]);
  if (last && !next) return guess;
  int lo = last ? guess + 1 : 0, hi = last ? a.P : guess - 1;
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (pages_valid(a, row[mid])) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void pages_place(const PagesArgs& a, int i, int b, int at) {  // token i at position `at` of b, or -1
  int64_t slot = -1;
  if (at >= 0) {
    const int j = (int)a.by_size.div((uint32_t)at), page = a.table[b * a.table_stride + j];
    if (pages_valid(a, page)) slot = (int64_t)page * a.size + (at - j * a.size);
  }
  a.positions[i] = at;
  a.slots[i] = slot;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) kv_pages_kernel(PagesArgs a) {
  __shared__ uint64_t sums[THREADS];  // running sums of pages, of the sequences of a round
  __shared__ uint64_t scan[THREADS / 64];
  __shared__ uint64_t most;
  __shared__ int32_t from[THREADS];   // a table's entry that the pages begin at
  __shared__ int32_t ends[THREADS];   // running sum of tokens, at most N
  __shared__ int32_t first_at[THREADS];
  const int tid = threadIdx.x;
  const int rounds = (a.B + THREADS - 1) / THREADS;
  const int free_before = min(max(*a.n_free, 0), a.F);
  PagesSequence s = {};
  // Sequence b of this thread; `tokens`: before the round's.
  auto look = [&](int b, uint64_t tokens, uint64_t* round_tokens) {
    s = PagesSequence{};
    if (b < a.B) {
      s.length = min(max(a.lengths[b], 0), a.P * a.size);
      s.count = a.counts[b];
      s.held = pages_held(a, b, pages_for(a, s.length));
    }
    const uint64_t end = tokens + pages_scan<THREADS / 64>((uint64_t)max(s.count, (int64_t)0), scan, round_tokens);
    const int64_t length = s.count < 0 ? 0 : s.length + s.count;
    s.fits = b < a.B && length <= (int64_t)a.P * a.size && (s.count <= 0 || end <= (uint64_t)a.N);
    s.need = s.fits ? pages_for(a, length) : s.held;
    s.start = (int32_t)min(end - (uint64_t)max(s.count, (int64_t)0), (uint64_t)a.N);
    ends[tid] = (int32_t)min(end, (uint64_t)a.N);
    if (b < a.B) a.starts[b + 1] = ends[tid];
  };

  // Pages that go back.
  uint64_t tokens = 0, back = 0, round_tokens = 0;
  if (tid == 0) a.starts[0] = 0;
  for (int round = 0; round < rounds; ++round) {
    const int b = round * THREADS + tid;
    look(b, tokens, &round_tokens);
    uint64_t all;
    const uint64_t up_to = pages_scan<THREADS / 64>((uint64_t)max(s.held - s.need, 0), scan, &all);
    sums[tid] = up_to;
    from[tid] = s.need - (int32_t)(up_to - (uint64_t)max(s.held - s.need, 0));  // (modulo 2^32: what is added to it takes it back)
    __syncthreads();
    for (uint64_t r = tid; r < all; r += THREADS) {
      const int t = first_above(sums, THREADS, r);
      int32_t* entry = a.table + (round * THREADS + t) * a.table_stride + (from[t] + (int32_t)r);
      const uint64_t to = free_before + back + r;
      if (to < (uint64_t)a.F) a.free_pages[to] = *entry;
      *entry = -1;
    }
    back += all;
    tokens += round_tokens;
    __syncthreads();
  }
  // (What the threads wrote to the list and the tables, the barrier above made known to the workgroup.)
  const int there = (int)min((uint64_t)free_before + back, (uint64_t)a.F);

  // Pages that are taken.
  uint64_t wanted = 0, taken = 0;
  tokens = 0;
  for (int round = 0; round < rounds; ++round) {
    const int b = round * THREADS + tid;
    if (rounds > 1) {
      look(b, tokens, &round_tokens);
      tokens += round_tokens;
    } else {
      s.held = min(s.held, s.need);
    }
    const int more = max(s.need - s.held, 0);
    uint64_t all;
    const uint64_t up_to = pages_scan<THREADS / 64>((uint64_t)more, scan, &all);
    const bool gets = s.fits && (more == 0 || wanted + up_to <= (uint64_t)there);
    if (tid == 0) most = 0;
    sums[tid] = up_to;
    from[tid] = s.held - (int32_t)(up_to - (uint64_t)more);
    first_at[tid] = gets && s.count > 0 ? s.length : -1;
    __syncthreads();
    if (gets && more > 0) atomicMax((unsigned long long*)&most, (unsigned long long)up_to);  // (those that get theirs come before those that do not)
    if (b < a.B) {
      a.new_lengths[b] = !gets ? s.length : s.count < 0 ? 0 : s.length + (int32_t)s.count;
      // The first token's position, or that it has none: what the second launch goes by.
      if (s.count > 0 && s.start < a.N) a.positions[s.start] = first_at[tid];
    }
    __syncthreads();
    const uint64_t now = most;
    for (uint64_t r = tid; r < now; r += THREADS) {
      const int t = first_above(sums, THREADS, r);
      a.table[(round * THREADS + t) * a.table_stride + (from[t] + (int32_t)r)] = a.free_pages[there - 1 - (int64_t)(wanted + r)];
    }
    wanted += all;
    taken += now;
    __syncthreads();
  }
  if (tid == 0) *a.n_free = there - (int)taken;
  if (rounds > 1 || a.N > 4 * THREADS) return;
  for (int i = tid; i < a.N; i += THREADS) {
    const int b = first_above(ends, THREADS, i);
    const bool inside = b < a.B && first_at[min(b, THREADS - 1)] >= 0;
    pages_place(a, i, b, inside ? first_at[b] + i - (b == 0 ? 0 : ends[b - 1]) : -1);
  }
}

__global__ void __launch_bounds__(256) kv_pages_tokens(PagesArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.N) return;
  const int b = first_above(a.starts + 1, a.B, i);
  int at = -1;
  if (b < a.B) {
    const int start = a.starts[b];
    // (the sequence's first token's own thread writes what it read)
    const int first = a.positions[start];
    at = first < 0 ? -1 : first + (i - start);
  }
  pages_place(a, i, b, at);
}

}  // namespace lh

using namespace lh;

extern "C" int lh_hip_kv_pages(int32_t* block_table, int64_t table_stride, const int32_t* lengths, const int32_t* counts, int32_t* new_lengths,
                               int32_t* free_pages, int32_t* n_free, int32_t* starts, int32_t* positions, int64_t* slots, int64_t B,
                               int64_t max_pages, int64_t n_pages, int64_t page_size, int64_t N, void* stream) {
  const char* what = "lh_hip_kv_pages";
  LH_REQUIRE(B >= 0 && B < (1ll << 20) && N >= 0 && N < (1ll << 30), "%s: bad counts (%lld sequences, fewer than 2^20; %lld tokens, fewer than 2^30)", what,
             (long long)B, (long long)N);
  LH_REQUIRE(max_pages > 0 && max_pages < (1ll << 31) && page_size > 0 && page_size < (1ll << 31) && max_pages * page_size < (1ll << 31) - 65536 && n_pages > 0 &&
                 n_pages < (1ll << 31),
             "%s: bad page counts (%lld pages of %lld, table of %lld)", what, (long long)n_pages, (long long)page_size, (long long)max_pages);
  LH_REQUIRE(free_pages && n_free && starts && (B == 0 || (block_table && lengths && counts && new_lengths)) && (N == 0 || (positions && slots)),
             "%s: null pointer", what);
  LH_REQUIRE(table_stride >= max_pages || B <= 1, "%s: rows of the block table overlap", what);
  const PagesArgs a = {block_table, table_stride, lengths, counts, new_lengths, free_pages, n_free, starts, positions, slots,
                       (int32_t)B, (int32_t)max_pages, (int32_t)n_pages, (int32_t)N, (int32_t)page_size, FastDiv((uint32_t)page_size)};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool small = B <= 256 && N <= 1024;  // (fewer waves at a barrier, fewer steps of a bisection)
  if (small) LH_LAUNCH((kv_pages_kernel<256>), dim3(1), dim3(256), 0, s, a);
  else LH_LAUNCH((kv_pages_kernel<kPagesThreads>), dim3(1), dim3(kPagesThreads), 0, s, a);
  if (const int rc = check_launch("kv_pages")) return rc;
  if (N == 0 || (B <= kPagesThreads && N <= 4 * kPagesThreads)) return LH_OK;
  LH_LAUNCH(kv_pages_tokens, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, s, a);
  return check_launch("kv_pages_tokens");
}
