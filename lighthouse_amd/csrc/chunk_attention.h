// Attention of packed chunks of new tokens over a paged cache: what its instances and its entry points share.
#pragma once

#include <type_traits>

#include "paged.h"
#include "wave_scan.h"

namespace lh {

struct ChunkArgs {
  Paged c;
  void* out;
  const void* q;
  int64_t so_n, so_h, sq_n, sq_h;
  const int32_t* lengths;  // [B]
  const int32_t* starts;   // [B + 1]
  int32_t N, B, H, G;
  FastDiv by_group;        // rows of a sequence and key / value head: G of a token
  int32_t tile_rows, tile_shift;  // rows a workgroup takes, a power of 2
  int32_t least, most;     // rows of the sequences that the launch is for
  int32_t slots;           // workgroups' places for tiles
  int32_t ranked;          // tiles by weight, or by place
  int32_t share, splits;   // positions a workgroup takes, workgroups for the positions of the table
  float scale_log2e;       // above 0
  uint32_t q_and, q_xor;   // on the queries' words: their signs change, or they become 0
  float* part_o;           // [rows of the result, or as chunk_part_row says][splits][width]
  float2* part_ml;         // [rows][splits]
  int32_t width;           // columns of a row of part_o
};

struct ChunkPlan {
  bool few;                // 16 rows a workgroup, otherwise 128
  int blocks;              // of the many: width of the kernel's rows, in 32 columns
  bool odd;                //   rows that are no whole pieces
  int mode;                // of the few: PagedMode
  int least, most, tile_rows, slots, share, splits, width;
  size_t o_bytes, ml_bytes;
  size_t total() const { return o_bytes + ml_bytes; }
};

constexpr int kChunkFew = 32;     // rows of a sequence: two tiles of the few
constexpr int kChunkSums = 4096;  // sequences whose tiles are found by running sums

// Places for the tiles of sequence b begin at rows / tile_rows (of the rows before it) + b: at least as many as its rows need.
__device__ __forceinline__ int chunk_start(const ChunkArgs& a, int b) { return min(max(a.starts[b], 0), a.N); }
__device__ __forceinline__ int chunk_place(const ChunkArgs& a, int b) { return (int)((uint32_t)(chunk_start(a, b) * a.G) >> a.tile_shift) + b; }
// Where the shares of a row's result lie: token n of the packed ones and `head`, which are `row` (of the sequence) of key / value head hk of sequence b.  By rows of the
// result, or, where the launch is for a few of them, by sequence.
__device__ __forceinline__ int64_t chunk_part_row(const ChunkArgs& a, int b, int hk, int row, int n, int head) {
  return a.most == kChunkFew ? ((int64_t)b * a.c.heads + hk) * kChunkFew + row : (int64_t)n * a.H + head;
}

// The last of the B sequences for which `begins(b) <= at` (ascending), 0 if there is none, by all lanes of a wave: 64 a round.
template <typename F>
__device__ __forceinline__ int chunk_last(const ChunkArgs& a, int at, F begins) {
  const int lane = threadIdx.x & 63;
  int b = 0;
  for (int span = a.B; span > 1;) {
    const int step = (span + 63) / 64;
    const uint64_t before = __builtin_amdgcn_ballot_w64(lane * step < span && begins(min(b + lane * step, a.B - 1)) <= at);
    const int many = (int)__popcll(before), last = many > 0 ? many - 1 : 0;  // (int: an unsigned 0 - 1 is no -1)
    b += last * step;
    span = min(step, span - last * step);
  }
  return __builtin_amdgcn_readfirstlane(b);
}

// The tile that workgroup `rank` of a head takes, heaviest first: for up to 32 sequences (`ranked`) first each one's last tile, then each one's last
// but one, and so on, since a later tile sees more positions; for up to 4096 the tiles in falling order, found by running sums of the lanes' sequences;
// otherwise the places in falling order.  (Those have holes, and the device deals workgroups to its CUs in turn, whether they find work or not: with every
// second place empty half of the CUs did all of it, 64 sequences of 16 rows 105 us instead of 79.)
__device__ __forceinline__ bool chunk_tile(const ChunkArgs& a, int rank, int* seq, int* tile) {
  if (a.ranked) {
    const int lane = threadIdx.x & 63, i = min(lane, a.B - 1);
    const int rows = max(chunk_start(a, i + 1) - chunk_start(a, i), 0) * a.G;
    const int tiles = lane < a.B && rows >= a.least && rows <= a.most ? (int)((uint32_t)(rows + a.tile_rows - 1) >> a.tile_shift) : 0;
    for (int level = 0;;) {  // (of each sequence, counted from its last tile)
      const uint64_t live = __builtin_amdgcn_ballot_w64(tiles > level);
      const int n = (int)__popcll(live);
      if (n == 0) return false;
      int same = tiles > level ? tiles : 0x7fffffff;  // up to here as many sequences have a tile
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) same = min(same, __shfl_xor(same, o));
      same = __builtin_amdgcn_readfirstlane(same);
      const int64_t there = (int64_t)n * (same - level);
      if (rank < there) {
        level += rank / n;
        uint64_t left = live;
        for (int k = rank % n; k > 0; --k) left &= left - 1;
        *seq = (int)__builtin_ctzll(left);
        *tile = __builtin_amdgcn_readlane(tiles, *seq) - 1 - level;
        return true;
      }
      rank -= (int)there;
      level = same;
    }
  }
  if (a.B <= kChunkSums) {
    const int lane = threadIdx.x & 63, per = (a.B + 63) >> 6;
    auto tiles_of = [&](int rows) { return rows >= a.least && rows <= a.most ? (int)((uint32_t)(rows + a.tile_rows - 1) >> a.tile_shift) : 0; };
    uint32_t mine = 0;
    int from = chunk_start(a, min(lane * per, a.B));
    for (int i = 0; i < per; ++i) {
      const int to = chunk_start(a, min(lane * per + i + 1, a.B));
      mine += (uint32_t)tiles_of(max(to - from, 0) * a.G);
      from = to;
    }
    const uint32_t up_to = wave_scan(mine), all = wave_last(up_to);
    if ((uint32_t)rank >= all) return false;
    const uint32_t at = all - 1 - (uint32_t)rank;
    const int owner = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(up_to > at));  // (the last lane's is)
    const uint32_t left = at - (uint32_t)__builtin_amdgcn_readlane((int)(up_to - mine), owner);
    const int b = owner * per + lane;
    const int tiles = lane < per && b < a.B ? tiles_of(max(chunk_start(a, b + 1) - chunk_start(a, b), 0) * a.G) : 0;
    const uint32_t up = wave_scan((uint32_t)tiles);
    const uint64_t above = __builtin_amdgcn_ballot_w64(up > left);
    if (above == 0) return false;
    const int which = (int)__builtin_ctzll(above), has = __builtin_amdgcn_readlane(tiles, which);
    *seq = owner * per + which;
    *tile = (int)(left - (uint32_t)(__builtin_amdgcn_readlane((int)up, which) - has));
    return *tile >= 0 && *tile < has;  // (starts that make no sense may have more tiles than an integer holds)
  }
  const int place = a.slots - 1 - rank;
  *seq = chunk_last(a, place, [&](int i) { return chunk_place(a, i); });
  const int start = __builtin_amdgcn_readfirstlane(chunk_start(a, *seq)), count = __builtin_amdgcn_readfirstlane(chunk_start(a, *seq + 1)) - start;
  *tile = place - __builtin_amdgcn_readfirstlane(chunk_place(a, *seq));
  return *tile >= 0 && count > 0 && count * a.G >= a.least && count * a.G <= a.most && *tile <= (count * a.G - 1) >> a.tile_shift;
}

// Launch the kernel of a pair of types (chunk_attention_kernel.hip and chunk_attention_few.hip, compiled once for each).
int chunk_many_f32(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_many_bf16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_many_f16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_many_e4m3_bf16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_many_e4m3_f16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_few_f32(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_few_bf16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_few_f16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_few_e4m3_bf16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_few_e4m3_f16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);

}  // namespace lh
