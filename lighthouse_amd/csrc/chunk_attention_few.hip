// Attention of packed chunks with few rows a sequence over a paged cache (a token each, a few drafted ones), for one pair of types: the kernel of
// one token of every sequence, with 16 neighbouring rows of (token, query of the group) where that has the queries of a group.  Like it, it is
// bound by memory, and P is the sum of three values of bf16 or two of f16.  4 tokens each of 8 sequences of 1024 to 4096 positions, bf16, 32 heads
// of 128 over 8: 24.9 us with the join (3.4 TB/s; in tiles of 128 rows 31.2).
#include "paged_rows.h"

#ifndef LH_CHUNK_CDT
#error "compiled with -DLH_CHUNK_CDT=... -DLH_CHUNK_QDT=... -DLH_CHUNK_NAME=..."
#endif

namespace lh {

template <int DP>
static int launch(const ChunkArgs& a, int mode, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.slots * a.c.heads * a.splits)), block(kPagedWaves * 64);
  if (mode == kTiles) LH_LAUNCH((paged_attention_kernel<LH_CHUNK_CDT, LH_CHUNK_QDT, DP, kPagedWaves, kTiles, ChunkArgs>), grid, block, 0, s, a);
  else if (mode == kWholeRows) LH_LAUNCH((paged_attention_kernel<LH_CHUNK_CDT, LH_CHUNK_QDT, DP, kPagedWaves, kWholeRows, ChunkArgs>), grid, block, 0, s, a);
  else LH_LAUNCH((paged_attention_kernel<LH_CHUNK_CDT, LH_CHUNK_QDT, DP, kPagedWaves, kOddRows, ChunkArgs>), grid, block, 0, s, a);
  return check_launch("chunk_attention_few");
}

int LH_CHUNK_NAME(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s) {
  if (a.width == 64) return launch<64>(a, p.mode, s);
  if (a.width == 128) return launch<128>(a, p.mode, s);
  return launch<256>(a, p.mode, s);
}

}  // namespace lh
