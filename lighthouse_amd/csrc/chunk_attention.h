// Attention of packed chunks of new tokens over a paged cache: what its instances and its entry points share.
#pragma once

#include <type_traits>

#include "paged.h"

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
  int32_t slots;           // workgroups' places for tiles
  int32_t share, splits;   // positions a workgroup takes, workgroups for the positions of the table
  float scale_log2e;       // above 0
  uint32_t q_and, q_xor;   // on the queries' words: their signs change, or they become 0
  float* part_o;           // [slots][kv heads][splits][tile_rows][width]
  float2* part_ml;         // [slots][kv heads][splits][tile_rows]
  int32_t width;           // columns of a row of part_o
};

struct ChunkPlan {
  int blocks;              // width of the kernel's rows, in 32 columns
  bool odd;                // rows that are no whole pieces
  bool few;                // 32 rows a workgroup, whose waves share the positions out; otherwise 128, 32 a wave
  int tile_rows, slots, share, splits;
  size_t o_bytes, ml_bytes;
  size_t total() const { return o_bytes + ml_bytes; }
};

// Places for the tiles of sequence b begin at rows / tile_rows (of the rows before it) + b: at least as many as its rows need.
__device__ __forceinline__ int chunk_start(const ChunkArgs& a, int b) { return min(max(a.starts[b], 0), a.N); }
__device__ __forceinline__ int chunk_place(const ChunkArgs& a, int b) { return (int)((uint32_t)(chunk_start(a, b) * a.G) >> a.tile_shift) + b; }

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

// Launches the kernel of a pair of types (in chunk_attention.hip, compiled once for each).
int chunk_launch_f32(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_launch_bf16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_launch_f16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_launch_e4m3_bf16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);
int chunk_launch_e4m3_f16(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s);

}  // namespace lh
