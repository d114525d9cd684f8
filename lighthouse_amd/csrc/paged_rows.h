// The kernel of attention over a paged cache for up to 16 rows a workgroup: of one new token of every sequence (paged_attention.hip, which
// says how it works) and of packed chunks with few rows a sequence (chunk_attention_few.hip).
#pragma once

#include <type_traits>

#include "chunk_attention.h"

namespace lh {

struct PagedAttnArgs {
  Paged c;
  void* out;
  const void* q;
  int64_t so_z, so_h, sq_z, sq_h;
  const int32_t* lengths;
  int32_t B, H, G, rows, groups;  // rows = min(G, 16) queries a workgroup, groups = ceil(G / 16) of them
  int32_t share, splits;          // positions a workgroup takes of a sequence, workgroups for the positions of the table
  float scale_log2e;
  float* part_o;   // [B heads groups][splits][rows][DP]
  float2* part_ml; // [B heads groups][splits][rows]
  float* scores;   // [B H][cap_pad], scaled, times log2(e); or null
  float* lse;      // [B H]: log2 of the sum of exp2(scores)
  int32_t cap_pad;
};

__device__ __forceinline__ int paged_length(const PagedAttnArgs& a, int b) { return min(max(a.lengths[b], 0), a.c.capacity()); }

constexpr int kPagedWaves = 4;
typedef float any_f32x4 __attribute__((ext_vector_type(4), aligned(4)));
constexpr int kPagedShare = 32 * kPagedWaves;  // positions a share is a multiple of

template <int DT>
__device__ __forceinline__ f32x4 paged_mma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == LH_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two e4m3 codes (the lower or upper two of a word) as two values of the 16-bit type DT: exact.
template <int DT, bool HI>
__device__ __forceinline__ uint32_t paged_e4m3(uint32_t w) {
  if constexpr (DT == LH_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}

// BYTES from p, of which `left` lie inside the row (elements of ES bytes at their own alignment); the others are 0.  `width`: bytes of a row
// (the same for the wave, which jumps over the loads by element where no piece needs them).  WHOLE: none does.
template <int BYTES, int ES, bool WHOLE>
__device__ __forceinline__ void load_row_piece(uint32_t* out, const uint8_t* p, int left, int width) {
  if (left >= BYTES) {
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) {
        const typename Chunk<ES>::type w = reinterpret_cast<const typename Chunk<ES>::type*>(p)[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) out[4 * i + e] = w[e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < BYTES / 4; ++i) __builtin_memcpy(&out[i], p + 4 * i, 4);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < BYTES / 4; ++i) out[i] = 0;
  if (WHOLE || width % BYTES == 0) return;
#pragma unroll
  for (int i = 0; i < BYTES / 4; ++i) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4 / ES; ++e)
      if (4 * i + ES * e < left) {
        if constexpr (ES == 1) w |= (uint32_t)p[4 * i + e] << (8 * e);
        else if constexpr (ES == 2) w |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[2 * i + e] << (16 * e);
        else w = reinterpret_cast<const uint32_t*>(p)[i];
      }
    out[i] = w;
  }
}

// The first `skip` elements of a piece become 0.
template <int BYTES, int ES>
__device__ __forceinline__ void clear_first(uint32_t* w, int skip) {
#pragma unroll
  for (int i = 0; i < BYTES / 4; ++i) {
    uint32_t keep = 0;
#pragma unroll
    for (int e = 0; e < 4 / ES; ++e) keep |= i * (4 / ES) + e >= skip ? (ES == 4 ? ~0u : ((1u << (8 * ES % 32)) - 1) << (8 * ES * e)) : 0u;
    w[i] &= keep;
  }
}

template <int BYTES>
__device__ __forceinline__ void load_buffer(uint32_t* out, __amdgpu_buffer_rsrc_t r, int offset) {
  if constexpr (BYTES == 4) {
    out[0] = __builtin_amdgcn_raw_buffer_load_b32(r, offset, 0, 0);
  } else if constexpr (BYTES == 8) {
    const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(r, offset, 0, 0);
    out[0] = w[0], out[1] = w[1];
  } else {
    const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = w[e];
  }
}

// All ones where element i of a piece of values is an infinity or a NaN (of e4m3: a NaN), otherwise 0; and not 0 where any of a word is.
template <int ES, int CDT>
__device__ __forceinline__ uint32_t paged_wild(const uint32_t* w, int i) {  // (an exponent of ones carries into the sign's place)
  if constexpr (ES == 4) return (uint32_t)((int32_t)((w[i] & 0x7f800000u) + 0x00800000u) >> 31);
  else if constexpr (ES == 2) return (uint32_t)((int32_t)(((w[i / 2] >> (16 * (i % 2)) & (CDT == LH_BF16 ? 0x7f80u : 0x7c00u)) + (CDT == LH_BF16 ? 0x80u : 0x400u)) << 16) >> 31);
  else return (uint32_t)((int32_t)(((w[i / 4] >> (8 * (i % 4)) & 0x7fu) + 1u) << 24) >> 31);
}
template <int ES, int CDT>
__device__ __forceinline__ uint32_t paged_wild_word(uint32_t w) {
  constexpr uint32_t top = ES == 4 ? 0x7f800000u : ES == 1 ? 0x7f7f7f7fu : CDT == LH_BF16 ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t one = ES == 4 ? 0x00800000u : ES == 1 ? 0x01010101u : CDT == LH_BF16 ? 0x00800080u : 0x04000400u;
  return ((w & top) + one) & ~top & (ES == 4 ? 0x80000000u : ES == 1 ? 0x80808080u : 0x80008000u);
}
// What the lanes of this wave have written to LDS, they read.
__device__ __forceinline__ void paged_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// CDT: the cache's type, QDT: the queries' (the cache's, or a 16-bit type with e4m3).  DP: width that d is padded to.
// kTiles: the pages are multiples of 16 positions and rows 16-byte aligned, so that a tile of 16 keys has one base and its rows
// are loaded through a buffer resource whose size is that of the rows that exist: what lies behind comes back as 0 without a
// test.  Otherwise every lane finds the page of every row it loads; kWholeRows: rows that are whole pieces, however aligned.
enum PagedMode { kTiles, kWholeRows, kOddRows };
// Waves of a SIMD that the registers have to suffice for: as many as they do without scratch memory.
constexpr int paged_occupancy(int cdt, int dp, int mode, bool chunk = false) {
  return dp == 64 ? (mode == kOddRows || (chunk && mode == kWholeRows) ? 3 : 4) : dp == 256 ? 1 : mode == kTiles && cdt != LH_F32 ? 3 : 2;
}
//
// Args: PagedAttnArgs, one token of every sequence: the up to 16 rows are queries of a group, and see all positions.  ChunkArgs, packed tokens:
// 16 neighbouring rows of (token, query of the group), each of which sees the positions up to its token's.
template <int CDT, int QDT, int DP, int NW, int MODE, typename Args>
__global__ void __launch_bounds__(NW * 64, paged_occupancy(CDT, DP, MODE, std::is_same<Args, ChunkArgs>::value)) paged_attention_kernel(Args a) {
  constexpr bool CHUNK = std::is_same<Args, ChunkArgs>::value;
  constexpr bool F32 = CDT == LH_F32, TILES = MODE == kTiles;
  constexpr int ES = CDT == LH_F8E4M3 ? 1 : F32 ? 4 : 2;
  constexpr int KT = F32 ? 1 : 2;            // 16-key tiles a step
  constexpr int KEYS = 16 * KT;
  constexpr int KB = 16;                       // bytes of a piece of a key's row
  constexpr int KE = KB / ES;                  // its elements
  constexpr int KS = DP / 4 / KE;              // pieces a lane takes: columns s 4 KE + g4 KE and on of piece s
  constexpr int CE = DP / 16;                  // columns of a value's row a lane takes
  constexpr int VB = CE * ES;
  constexpr int VP = VB > 16 ? VB / 16 : 1;    // loads for them
  constexpr int VPB = VB / VP;
  constexpr int PARTS = QDT == LH_BF16 ? 3 : 2;  // 16-bit values that a probability is the sum of
  constexpr int kOutside = 0x40000000;         // an offset behind every buffer
  // Rows that are no whole pieces (and longer than one): the last piece moves back to end with the row.  Of a key and a query it gives only the
  // columns that the piece before has not; columns of a value may come from two lanes, which are of one mind.  (By element, 16 sequences of
  // 1024 to 4096, 8 heads of 136 with 4 queries, e4m3: 211 us instead of 73; 32 of 40 to 161, 7 heads of 181 with 16 queries, bf16: 41 instead of 34.)
  const bool k_back = MODE == kOddRows && a.c.d % KE != 0 && a.c.d > KE, v_back = MODE == kOddRows && a.c.d % CE != 0 && a.c.d > CE;
  __shared__ __attribute__((aligned(16))) f32x4 sums[NW / 2][CE][64];
  __shared__ float2 stats[NW][16];
  __shared__ int32_t first_wild[CHUNK ? NW : 1][CHUNK ? DP : 1];

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // An item is a (sequence, key / value head, group of queries).  The first shares of all items come first.  Workgroups whose ids
  // agree modulo 8 run on one XCD: an item's shares go round them, else those of the long sequences could meet on a few.
  int b, hk, item, split, k0, n;
  int q_row, head, token = 0, last_seen = 0, all_see = 0;  // CHUNK: the last position that the lane's row sees, and that every row sees
  int first_row = 0, first_token = 0;                      // CHUNK: of the tile, in its sequence; of the sequence
  bool q_live;
  if constexpr (CHUNK) {
    const int items = a.slots * a.c.heads;
    split = blockIdx.x / items, item = blockIdx.x - split * items, hk = item % a.c.heads, k0 = split * a.share;
    int tile;
    if (!chunk_tile(a, item / a.c.heads, &b, &tile)) return;
    const int start = __builtin_amdgcn_readfirstlane(chunk_start(a, b));
    const int count = max(__builtin_amdgcn_readfirstlane(chunk_start(a, b + 1)) - start, 0);
    const int first = tile << a.tile_shift, rows = min(a.tile_rows, count * a.G - first);
    const int base = __builtin_amdgcn_readfirstlane(min(max(a.lengths[b], 0), a.c.capacity())) - count;
    n = max(base + (int)a.by_group.div((uint32_t)(first + rows - 1)) + 1, 0);  // positions that the last row sees
    q_row = l16, q_live = l16 < rows;
    const int row = first + (q_live ? l16 : 0), of_chunk = (int)a.by_group.div((uint32_t)row);
    token = start + of_chunk, head = hk * a.G + (row - of_chunk * a.G), last_seen = base + of_chunk;
    first_row = first, first_token = start;
    all_see = base + (int)a.by_group.div((uint32_t)first);
  } else {
    const int items = a.B * a.c.heads * a.groups;
    split = blockIdx.x / items;
    item = (int)((blockIdx.x - (unsigned)split * items + split) % (unsigned)items);
    const int group = item % a.groups, rest = item / a.groups;
    hk = rest % a.c.heads, b = rest / a.c.heads, k0 = split * a.share;
    q_row = group * 16 + l16;           // of the G queries
    q_live = q_row < a.G;
    head = hk * a.G + min(q_row, a.G - 1);
  }
  const int table_end = k0 + min(a.c.capacity() - k0, a.share);  // (k0 + share may pass 2^31)
  const int64_t table_row = b * a.c.table_stride;
  int ahead[KT];       // what the table says for a later step
  auto find_pages = [&](int step, int* found) {
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int key = min(k0 + step * KEYS + 16 * t + (TILES ? 0 : l16), table_end - 1);
      found[t] = a.c.entry(table_row + a.c.by_size.div((uint32_t)key));
    }
  };
  // (The share is the host's choice, so that the table is asked without waiting for the length.)
  int head_start[KT];
  find_pages(wave, head_start);
  find_pages(wave + NW, ahead);
  if constexpr (!CHUNK) n = paged_length(a, b);

  // The queries, in the layout of the second operand.
  constexpr int QES = F32 ? 4 : 2, QP = KE * QES / 16;  // 16-byte pieces of a query that go with a piece of a key
  uint32_t qf[KS * QP][4];
  {
    const uint8_t* q = static_cast<const uint8_t*>(a.q);
    if constexpr (CHUNK) q += (token * a.sq_n + head * a.sq_h) * QES;
    else q += (b * a.sq_z + head * a.sq_h) * QES;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < QP; ++i) {
        const int k_d0 = s * (4 * KE) + g4 * KE, back = k_back ? max(k_d0 - (a.c.d - KE), 0) : 0, d0 = k_d0 + i * (16 / QES);
        const int left = !q_live ? 0 : !k_back ? (a.c.d - d0) * QES : k_d0 < a.c.d ? 16 : 0;
        load_row_piece<16, QES, MODE != kOddRows>(qf[s * QP + i], q + (d0 - back) * QES, left, k_back ? 16 : a.c.d * QES);
        if (k_back) clear_first<16, QES>(qf[s * QP + i], back - i * (16 / QES));
        if constexpr (CHUNK)
#pragma unroll
          for (int e = 0; e < 4; ++e) qf[s * QP + i][e] = (qf[s * QP + i][e] & a.q_and) ^ a.q_xor;
      }
  }

  f32x4 acc[CE];
#pragma unroll
  for (int i = 0; i < CE; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m_run = -INFINITY, l_run = 0.0f;

  if (k0 >= n && split > 0) return;
  const int k1 = k0 + min(n - k0, a.share);
  const uint8_t* kb = static_cast<const uint8_t*>(a.c.k);
  const uint8_t* vb = static_cast<const uint8_t*>(a.c.v);
  const int row_bytes = a.c.d * ES;
  uint32_t kr[KT][KS][KB / 4], vr[KT * 4][VB / 4];
  int pages[KT];       // of the step that is requested next: of its tiles, or of the key 16 t + l16 that is the lane's
  int held[KT];        // kTiles: how many rows of its tiles exist
  uint32_t live = 0;   // otherwise: which of the lane's KT * 4 keys do

  int koff[KS], voff[4][VP];
  if constexpr (TILES) {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d0 = s * (4 * KE) + g4 * KE;
      koff[s] = d0 < a.c.d ? l16 * (int)a.c.sk.t * ES + d0 * ES : kOutside;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int p = 0; p < VP; ++p) {
        const int col = l16 * VB + p * VPB;
        voff[r][p] = col < row_bytes ? (g4 * 4 + r) * (int)a.c.sv.t * ES + col : kOutside;
      }
  }
  // kTiles: where the rows of a tile of the next step begin (keys and values are laid out alike), and how many bytes there are.
  int64_t tile_at[KT];
  int tile_bytes[KT];
  auto next_pages = [&](int step, const int* found) {
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int key = k0 + step * KEYS + 16 * t + (TILES ? 0 : l16);
      pages[t] = (uint32_t)found[t] < (uint32_t)a.c.pages && key < k1 ? found[t] : -1;
      if constexpr (TILES) {
        const int slot = key - (int)a.c.by_size.div((uint32_t)key) * a.c.size;
        const int rows = pages[t] < 0 ? 0 : min(16, k1 - key);
        tile_at[t] = rows == 0 ? 0 : (pages[t] * a.c.sk.z + hk * a.c.sk.h + slot * a.c.sk.t) * ES;
        tile_bytes[t] = rows * (int)a.c.sk.t * ES;
      }
    }
  };
  auto request_keys = [&](int step) {
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      if constexpr (TILES) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(kb + tile_at[t]), 0, tile_bytes[t], 0x00020000);
#pragma unroll
        for (int s = 0; s < KS; ++s) load_buffer<KB>(kr[t][s], r, koff[s]);
      } else {
        const int key = k0 + step * KEYS + 16 * t + l16, page = pages[t];
        const int slot = key - (int)a.c.by_size.div((uint32_t)key) * a.c.size;
        const uint8_t* row = kb + (max(page, 0) * a.c.sk.z + hk * a.c.sk.h + slot * a.c.sk.t) * ES;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int d0 = s * (4 * KE) + g4 * KE;
          if (!k_back) {
            load_row_piece<KB, ES, MODE != kOddRows>(kr[t][s], row + d0 * ES, page < 0 ? 0 : (a.c.d - d0) * ES, row_bytes);
          } else {
            const int back = max(d0 - (a.c.d - KE), 0);
            load_row_piece<KB, ES, MODE != kOddRows>(kr[t][s], row + (d0 - back) * ES, page >= 0 && d0 < a.c.d ? KB : 0, KB);
            if ((s + 1) * (4 * KE) > a.c.d) clear_first<KB, ES>(kr[t][s], back);
          }
        }
      }
    }
  };
  auto request_values = [&](int step) {
    live = 0;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      if constexpr (TILES) {
        const int key = k0 + step * KEYS + 16 * t;
        held[t] = pages[t] < 0 ? 0 : min(16, k1 - key);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(vb + tile_at[t]), 0, tile_bytes[t], 0x00020000);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int p = 0; p < VP; ++p) load_buffer<VPB>(vr[t * 4 + r] + p * (VPB / 4), rs, voff[r][p]);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = k0 + step * KEYS + 16 * t + 4 * g4 + r, page = __shfl(pages[t], 4 * g4 + r);
          const int slot = key - (int)a.c.by_size.div((uint32_t)key) * a.c.size;
          const uint8_t* row = vb + (max(page, 0) * a.c.sv.z + hk * a.c.sv.h + slot * a.c.sv.t) * ES;
          const int col = v_back ? min(l16 * CE, a.c.d - CE) : l16 * CE, left = !v_back ? row_bytes - l16 * VB : l16 * CE < a.c.d ? VB : 0;
          load_row_piece<VB, ES, MODE != kOddRows>(vr[t * 4 + r], row + col * ES, page < 0 ? 0 : left, v_back ? VB : row_bytes);
          live |= (page >= 0 ? 1u : 0u) << (t * 4 + r);
        }
      }
    }
  };

  const int steps = (k1 - k0 + KEYS - 1) / KEYS;
  if (wave < steps) {
    next_pages(wave, head_start);
    request_keys(wave);
    request_values(wave);
  }
#pragma unroll 1
  for (int step = wave; step < steps; step += NW) {
    const int next = step + NW;
    next_pages(next, ahead);
    find_pages(next + NW, ahead);
    // S^T: s[t][r] = S[query l16][key 16 t + 4 g4 + r]
    f32x4 s[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      s[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        if constexpr (F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, kr[t][i][e]), __builtin_bit_cast(float, qf[i][e]), s[t], 0, 0, 0);
        } else {
#pragma unroll
          for (int j = 0; j < QP; ++j) {
            u32x4 kf;
            if constexpr (CDT == LH_F8E4M3) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t codes = kr[t][i][2 * j + e];
                kf[2 * e] = paged_e4m3<QDT, false>(codes), kf[2 * e + 1] = paged_e4m3<QDT, true>(codes);
              }
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) kf[e] = kr[t][i][e];
            }
            const uint32_t(&qq)[4] = qf[i * QP + j];
            s[t] = paged_mma<QDT>(kf, u32x4{qq[0], qq[1], qq[2], qq[3]}, s[t]);
          }
        }
      }
    }
    if (next < steps) request_keys(next);  // (the registers of the keys are free again)

    // Softmax: x = s scale log2(e); a position that is not there has -inf.
    f32x4 x[KT];
    bool whole = true;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      x[t] = s[t] * a.scale_log2e;
      if constexpr (TILES) whole = whole && held[t] == 16;
    }
    if constexpr (CHUNK) whole = whole && k0 + (step + 1) * KEYS - 1 <= all_see;
    if (!TILES || !whole) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          bool there;
          if constexpr (TILES) there = 4 * g4 + r < held[t];
          else there = live >> (t * 4 + r) & 1;
          if constexpr (CHUNK) there = there && k0 + step * KEYS + 16 * t + 4 * g4 + r <= last_seen;
          if (!there) x[t][r] = s[t][r] = -INFINITY;
        }
    }
    float mx = x[0][0];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[t][r]);
    if constexpr (!CHUNK)
      if (a.scores != nullptr && q_live) {
        float* to = a.scores + ((int64_t)b * a.H + head) * a.cap_pad + k0 + step * KEYS + 4 * g4;
#pragma unroll
        for (int t = 0; t < KT; ++t) *reinterpret_cast<f32x4*>(to + 16 * t) = x[t];
      }
    // What p is relative to follows the true maximum with a delay: nothing is done until a p would be above 2^10 (which is as
    // accurate as one of 1), or 2^14 in f16, and then by all lanes together.  In f16 it lies 2^12 below the maximum: thousands of positions
    // with 2^-25 of the largest weight, which f16 has no numbers for, have their part in a long row.
    constexpr float slack = QDT == LH_F16 ? 14.0f : 10.0f;
    if (__any(mx > m_run + slack)) {
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      float m_new = fmaxf(m_run, QDT == LH_F16 ? mx - 12.0f : mx);
      if constexpr (CHUNK) m_new = mx > m_run + slack ? m_new : m_run;  // (what other rows see does not reach a row's roundings)
      const float alpha = m_run == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < CE; ++i) acc[i] *= alpha;
    }
    const float off = m_run == -INFINITY ? 0.0f : m_run;  // (nothing there yet: every p is exp2(-inf))
    float p[KT * 4];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // (one rounding of s scale - maximum; where s is -inf the product may be a NaN only for a scale of 0)
        p[t * 4 + r] = x[t][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], a.scale_log2e, -off));
        l_run += p[t * 4 + r];
      }

    // A value that some row does not see must not reach it by a 0 times an infinity: such values become 0, and a column's first one makes a NaN of
    // the rows that see it.
    bool some_wild = false;
    if constexpr (CHUNK)
      if (k0 + (step + 1) * KEYS - 1 > all_see) {
        uint32_t any = 0;
#pragma unroll
        for (int j = 0; j < KT * 4; ++j)
#pragma unroll
          for (int i = 0; i < VB / 4; ++i) any |= paged_wild_word<ES, CDT>(vr[j][i]);
        some_wild = __any(any != 0);
        if (__builtin_expect(some_wild, 0)) {
          for (int c = lane; c < DP; c += 64) first_wild[wave][c] = KEYS + 1;
          paged_wave_sync();
#pragma unroll
          for (int j = 0; j < KT * 4; ++j)
#pragma unroll
            for (int i = 0; i < CE; ++i) {  // (without conditions)
              const uint32_t mask = paged_wild<ES, CDT>(vr[j], i);
              const int col = (v_back ? min(l16 * CE, a.c.d - CE) : l16 * CE) + i, key = 16 * (j / 4) + 4 * g4 + j % 4;  // (of the step)
              atomicMin(&first_wild[wave][col], mask ? key : KEYS + 1);
              vr[j][i * ES / 4] &= ~(ES == 4 ? mask : (mask & ((1u << (8 * ES % 32)) - 1)) << (8 * ES * i % 32));
            }
          paged_wave_sync();
        }
      }

    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < KT * 4; ++j)
#pragma unroll
        for (int i = 0; i < CE; ++i)
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vr[j][i]), p[j], acc[i], 0, 0, 0);
    } else {
      u32x4 part[PARTS];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float p0 = p[2 * e], p1 = p[2 * e + 1];
#pragma unroll
        for (int n = 0; n < PARTS; ++n) {
          part[n][e] = pack2<QDT>(p0, p1);
          p0 -= unpack_lo<QDT>(part[n][e]), p1 -= unpack_hi<QDT>(part[n][e]);
        }
      }
      uint32_t vw[8][CE / 2];  // [key][pair of columns]
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < CE / 2; ++e) {
          if constexpr (CDT == LH_F8E4M3) vw[j][e] = e % 2 ? paged_e4m3<QDT, true>(vr[j][e / 2]) : paged_e4m3<QDT, false>(vr[j][e / 2]);
          else vw[j][e] = vr[j][e];
        }
#pragma unroll
      for (int e = 0; e < CE / 2; ++e) {
        u32x4 even, odd;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          even[j] = __builtin_amdgcn_perm(vw[2 * j + 1][e], vw[2 * j][e], 0x05040100u);
          odd[j] = __builtin_amdgcn_perm(vw[2 * j + 1][e], vw[2 * j][e], 0x07060302u);
        }
#pragma unroll
        for (int n = 0; n < PARTS; ++n) {
          acc[2 * e] = paged_mma<QDT>(even, part[n], acc[2 * e]);
          acc[2 * e + 1] = paged_mma<QDT>(odd, part[n], acc[2 * e + 1]);
        }
      }
    }
    if constexpr (CHUNK)
      if (__builtin_expect(some_wild, 0)) {
        const int sees_up_to = min(max(last_seen - (k0 + step * KEYS), -1), KEYS);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < CE; ++i) {
            const int col = (v_back ? min((4 * g4 + r) * CE, a.c.d - CE) : (4 * g4 + r) * CE) + i;
            acc[i][r] = __uint_as_float(__float_as_uint(acc[i][r]) | (uint32_t)((first_wild[wave][col] - 1 - sees_up_to) >> 31));
          }
      }
    if (next < steps) request_values(next);
  }

  // acc[i][r] = sum p v of query l16, column first_col(r) + i, over this wave's positions and relative to its maximum.
  auto first_col = [&](int r) { return v_back ? min((4 * g4 + r) * CE, a.c.d - CE) : (4 * g4 + r) * CE; };
  l_run += __shfl_xor(l_run, 16);
  l_run += __shfl_xor(l_run, 32);
  if (g4 == 0) stats[wave][l16] = make_float2(m_run, l_run);
  __syncthreads();
  float m_all = -INFINITY, l_all = 0.0f;
#pragma unroll
  for (int w = 0; w < NW; ++w) m_all = fmaxf(m_all, stats[w][l16].x);
  const float m_safe = m_all == -INFINITY ? 0.0f : m_all;
#pragma unroll
  for (int w = 0; w < NW; ++w) l_all += stats[w][l16].y * __builtin_amdgcn_exp2f(stats[w][l16].x - m_safe);
  const float own = __builtin_amdgcn_exp2f(m_run - m_safe);
#pragma unroll
  for (int i = 0; i < CE; ++i) acc[i] *= own;
#pragma unroll
  for (int half = NW / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half)
#pragma unroll
      for (int i = 0; i < CE; ++i) sums[wave - half][i][lane] = acc[i];
    __syncthreads();
    if (wave < half)
#pragma unroll
      for (int i = 0; i < CE; ++i) acc[i] += sums[wave][i][lane];
    if (half > 1) __syncthreads();
  }
  if (wave != 0 || !q_live) return;
  if constexpr (CHUNK) {  // (found again and not held over the steps)
    int of_tile = l16;
    asm volatile("" : "+v"(of_tile));
    q_row = first_row + of_tile;
    const int of_chunk = (int)a.by_group.div((uint32_t)q_row);
    token = first_token + of_chunk, head = hk * a.G + (q_row - of_chunk * a.G);
  }
  if (n > a.share) {
    int64_t part;
    if constexpr (CHUNK) part = chunk_part_row(a, b, hk, q_row, token, head) * a.splits + split;
    else part = ((int64_t)item * a.splits + split) * a.rows + l16;
    if (g4 == 0) a.part_ml[part] = make_float2(m_all, l_all);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < CE; i += 4)
        if ((4 * g4 + r) * CE < a.c.d)
          *reinterpret_cast<any_f32x4*>(a.part_o + part * DP + first_col(r) + i) = any_f32x4{acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]};
    return;
  }
  if constexpr (!CHUNK)
    if (a.lse != nullptr && g4 == 0) a.lse[(int64_t)b * a.H + head] = m_all + __builtin_amdgcn_logf(l_all);
  const float inv = l_all == 0.0f ? 0.0f : a.c.v_scale / l_all;  // (no position there: 0)
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < CE; ++i) {
      const int col = first_col(r) + i;
      if ((4 * g4 + r) * CE < a.c.d && col < a.c.d) {
        if constexpr (CHUNK) store_from_f32<QDT>(a.out, token * a.so_n + head * a.so_h + col, acc[i][r] * inv);
        else store_from_f32<QDT>(a.out, b * a.so_z + head * a.so_h + col, acc[i][r] * inv);
      }
    }
}

// ---- host side ------------------------------------------------------------------------------------------------------------

// `aligned`: keys and values begin at multiples of 16 bytes.
inline bool paged_in_tiles(const Paged& c, int es, bool aligned) {
  const lh_strides3& s = c.sk;
  return aligned && c.size % 16 == 0 && c.d * es % 16 == 0 && s.z == c.sv.z && s.h == c.sv.h && s.t == c.sv.t && s.z * es % 16 == 0 && s.h * es % 16 == 0 &&
         s.t * es % 16 == 0 && 16 * s.t * es < 0x40000000 && s.t >= c.d;
}

// Width that a row is padded to, and how rows are loaded.
inline int paged_width(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
inline int paged_mode(const Paged& c, int es, bool aligned) {
  return paged_in_tiles(c, es, aligned) ? kTiles : c.d * es % 16 == 0 && c.d % (paged_width(c.d) / 16) == 0 ? kWholeRows : kOddRows;
}

// How many positions a workgroup takes of a sequence; `items` (sequence, head, group of queries), `per_cu` workgroups that a CU
// holds at once, `row_bytes` of a position's key and value.  There are to be two workgroups per CU (one, if no more fit; one also where the
// shares would be shorter than 1024 positions, of which their start and end take too much).  (One sequence of 1000, 12 heads of 64: 7.6 us with 128
// positions a share, 9.8 in one; one of 32768, 8 heads of 128: 31.8 with 1024, 33.5 with 512, 362 in one; 4 of 1024 to 4096, 8 heads of 128 with 4 queries: 14.8 with
// 512, 15.8 with 256; heads of 256, 16 sequences of 1024 to 4096: 73 with 2048, 94 with 512.)  With items enough for that, up to 8 per CU
// even out sequences of unlike length, while a share has 512 KB of keys and values, which the join's launch costs nothing against.  (16
// sequences of 8192 to 32768, 8 heads of 128: 255 with 2048, 263 with 512, 384 in one; 64 of 256 to 1024, 12 heads of 64, 30 in one, 33 with 512.)
inline int paged_share(int64_t items, int capacity, int per_cu, int64_t row_bytes) {
  const int64_t cus = num_cus();
  int64_t splits = ((per_cu < 2 ? 1 : 2) * cus + items - 1) / items;
  if (per_cu >= 3) {
    if (capacity < 1024 * splits) splits = (cus + items - 1) / items;
    const int64_t level = (8 * cus + items - 1) / items, most = capacity * row_bytes >> 19;
    splits = splits > level ? splits : level < most ? level : splits > most ? splits : most;
  }
  const int64_t share = (capacity + splits - 1) / splits;
  return (int)((share + kPagedShare - 1) / kPagedShare * kPagedShare);
}

}  // namespace lh
