// Attention of one new token of every sequence over its paged key / value cache.
//
// Per sequence and key / value head: S = scale Q K^T for the G query heads that share it, a softmax over the positions
// in one pass (running maximum and sum), O = P V.  Every key and value is read once and used for G heads: the work is
// bound by memory, 1 to 2 operations a byte and head.  So the kernel is built around its loads:
//
//  * The G queries (up to 16) are the columns of 16-wide matrix instructions, whatever G is: the matrix cores have an order of
//    magnitude to spare here, and the vector ALUs, which a dot product per head would fill, stay free.
//  * Keys and values go from memory into registers in the layout that the matrix instructions take, without LDS and without
//    barriers: S^T = K Q^T wants a key's row in pieces of 8 along d, which is how it lies in memory.  O^T = V^T P^T
//    wants 8 keys of one column in a lane.  A lane loads the same piece of a row for 8 keys, 16 lanes a whole row, and turns the 8 x 8
//    block in its registers, one v_perm_b32 per register: row m of fragment i is column m CE + i (CE = DP / 16 columns a lane).
//  * The accumulators of S^T leave a lane with keys 4 g .. 4 g + 3 of both 16-key tiles of a step of one query, which, in that
//    order of the keys, is the second operand of O^T (the lane loads the values of exactly those keys).
//  * The waves of a workgroup take the steps of its share of the positions in turn, each on its own; their results are brought to
//    the common maximum and added through LDS at the end.  A long cache is shared out between `splits` workgroups,
//    each leaving (maximum, sum, sum of p v), which a second launch joins.
//  * The table is read two steps ahead by the scalar unit, so that no step waits for a lookup or drains the loads on the way.
//
// Measured, keys and values out of memory: 16 sequences of 8192 to 32768 in bf16, 8 heads of 128 with 4 queries each, 256 us (5.2 TB/s) and 5 for
// the join; 64 sequences of 256 to 1024, 12 heads of 64, 31 us (4.1 TB/s); 32 sequences of 2048 to 8192 in e4m3, 4 heads of 128 with 8 queries
// each, 38 us (4.4 TB/s) and 5.  Out of the caches all of it takes 136, 19 and 34: the longer ones are bound by memory, and by what one CU draws of
// it (31 B/ns) where the sequences' lengths do not fill all CUs to the end.  One sequence of 1000, 12 heads of 64: 6.1 us and 3.6, the chain of
// table, keys, values and join.
//
// 16-bit types: P is split into values of the type, each nearest to what the ones before leave: three of bf16 have all 24 places of an f32, two of
// f16 have 22, and there is a matrix instruction for each.  (Where values cancel, what P has lost shows in the result: with two of bf16,
// 2^-18 of the largest values.  The third costs long caches less than 1 %, 8 sequences of 256 to 1024, 16 heads of 64, 12.0 us instead of 11.7.)
// f32 runs on v_mfma_f32_16x16x4_f32 with one 16-key tile a step.  e4m3 codes are converted to the queries' type, in which every code has
// an exact value.
#include "paged.h"

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

constexpr int kPagedWaves = 4;
typedef float any_f32x4 __attribute__((ext_vector_type(4), aligned(4)));
constexpr int kPagedShare = 32 * kPagedWaves;  // positions a share is a multiple of

__device__ __forceinline__ int paged_length(const PagedAttnArgs& a, int b) { return min(max(a.lengths[b], 0), a.c.capacity()); }
// Shares that n positions take.
__device__ __forceinline__ int paged_parts(const PagedAttnArgs& a, int n) { return (int)(((uint32_t)n + (uint32_t)a.share - 1u) / (uint32_t)a.share); }

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

// CDT: the cache's type, QDT: the queries' (the cache's, or a 16-bit type with e4m3).  DP: width that d is padded to.
// kTiles: the pages are multiples of 16 positions and rows 16-byte aligned, so that a tile of 16 keys has one base and its rows
// are loaded through a buffer resource whose size is that of the rows that exist: what lies behind comes back as 0 without a
// test.  Otherwise every lane finds the page of every row it loads; kWholeRows: rows that are whole pieces, however aligned.
enum PagedMode { kTiles, kWholeRows, kOddRows };
// Waves of a SIMD that the registers have to suffice for: as many as they do without scratch memory.
constexpr int paged_occupancy(int cdt, int dp, int mode) {
  return dp == 64 ? (mode == kOddRows ? 3 : 4) : dp == 256 ? 1 : mode == kTiles && cdt != LH_F32 ? 3 : 2;
}
template <int CDT, int QDT, int DP, int NW, int MODE>
__global__ void __launch_bounds__(NW * 64, paged_occupancy(CDT, DP, MODE)) paged_attention_kernel(PagedAttnArgs a) {
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

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // An item is a (sequence, key / value head, group of queries).  The first shares of all items come first.  Workgroups whose ids
  // agree modulo 8 run on one XCD: an item's shares go round them, else those of the long sequences could meet on a few.
  const int items = a.B * a.c.heads * a.groups, split = blockIdx.x / items;
  const int item = (int)((blockIdx.x - (unsigned)split * items + split) % (unsigned)items);
  const int group = item % a.groups, rest = item / a.groups;
  const int hk = rest % a.c.heads, b = rest / a.c.heads;
  const int k0 = split * a.share, table_end = k0 + min(a.c.capacity() - k0, a.share);  // (k0 + share may pass 2^31)
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
  const int n = paged_length(a, b);
  const int q_row = group * 16 + l16;           // of the G queries
  const bool q_live = q_row < a.G;
  const int head = hk * a.G + min(q_row, a.G - 1);

  // The queries, in the layout of the second operand.
  constexpr int QES = F32 ? 4 : 2, QP = KE * QES / 16;  // 16-byte pieces of a query that go with a piece of a key
  uint32_t qf[KS * QP][4];
  {
    const uint8_t* q = static_cast<const uint8_t*>(a.q) + (b * a.sq_z + head * a.sq_h) * QES;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int i = 0; i < QP; ++i) {
        const int k_d0 = s * (4 * KE) + g4 * KE, back = k_back ? max(k_d0 - (a.c.d - KE), 0) : 0, d0 = k_d0 + i * (16 / QES);
        const int left = !q_live ? 0 : !k_back ? (a.c.d - d0) * QES : k_d0 < a.c.d ? 16 : 0;
        load_row_piece<16, QES, MODE != kOddRows>(qf[s * QP + i], q + (d0 - back) * QES, left, k_back ? 16 : a.c.d * QES);
        if (k_back) clear_first<16, QES>(qf[s * QP + i], back - i * (16 / QES));
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
    if (!TILES || !whole) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          bool there;
          if constexpr (TILES) there = 4 * g4 + r < held[t];
          else there = live >> (t * 4 + r) & 1;
          if (!there) x[t][r] = s[t][r] = -INFINITY;
        }
    }
    float mx = x[0][0];
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[t][r]);
    if (a.scores != nullptr && q_live) {
      float* to = a.scores + ((int64_t)b * a.H + head) * a.cap_pad + k0 + step * KEYS + 4 * g4;
#pragma unroll
      for (int t = 0; t < KT; ++t) *reinterpret_cast<f32x4*>(to + 16 * t) = x[t];
    }
    // What p is relative to follows the true maximum with a delay: nothing is done until a p would be above 2^10 (which is as
    // accurate as one of 1), or 2^14 in f16, and then by all lanes together.  In f16 it lies 2^12 below the maximum: thousands of positions
    // with 2^-25 of the largest weight, which f16 has no numbers for, have their part in a long row.
    if (__any(mx > m_run + (QDT == LH_F16 ? 14.0f : 10.0f))) {
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m_run, QDT == LH_F16 ? mx - 12.0f : mx);
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
  if (n > a.share) {
    const int64_t part = ((int64_t)item * a.splits + split) * a.rows + l16;
    if (g4 == 0) a.part_ml[part] = make_float2(m_all, l_all);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < CE; i += 4)
        if ((4 * g4 + r) * CE < a.c.d)
          *reinterpret_cast<any_f32x4*>(a.part_o + part * DP + first_col(r) + i) = any_f32x4{acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]};
    return;
  }
  if (a.lse != nullptr && g4 == 0) a.lse[(int64_t)b * a.H + head] = m_all + __builtin_amdgcn_logf(l_all);
  const float inv = l_all == 0.0f ? 0.0f : a.c.v_scale / l_all;  // (no position there: 0)
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < CE; ++i) {
      const int col = first_col(r) + i;
      if ((4 * g4 + r) * CE < a.c.d && col < a.c.d) store_from_f32<QDT>(a.out, b * a.so_z + head * a.so_h + col, acc[i][r] * inv);
    }
}

// (maximum, sum) of one query over its parts, to every lane of the wave: the lanes take the parts in turn, the lanes' values are
// brought together in a fixed order.
__device__ __forceinline__ float2 paged_join(const float2* ml, int parts, int rows, int lane) {
  float m = -INFINITY, l = 0.0f;
  for (int p = lane; p < parts; p += 64) {
    const float2 x = ml[(int64_t)p * rows];
    const float to = fmaxf(m, x.x), safe = to == -INFINITY ? 0.0f : to;
    l = l * __builtin_amdgcn_exp2f(m - safe) + x.y * __builtin_amdgcn_exp2f(x.x - safe);
    m = to;
  }
  float all = m;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) all = fmaxf(all, __shfl_xor(all, o));
  const float safe = all == -INFINITY ? 0.0f : all;
  l *= __builtin_amdgcn_exp2f(m - safe);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) l += __shfl_xor(l, o);
  return make_float2(safe, l);
}

// The first B H workgroups join the parts of a query each: they bring them to the common maximum and add them in the order of the
// positions.  The others, where weights are asked for, take 256 positions of a head of a sequence: weights[b, g, t] += sum over the
// heads of the group of exp2(score - log2 of the head's sum), heads in order; they find that sum for themselves.
template <int QDT, int DP>
__global__ void __launch_bounds__(256) paged_attention_finish(PagedAttnArgs a, int joins, float* weights, int64_t sw_b, int64_t sw_h) {
  constexpr int GROUPS = 256 / DP;
  __shared__ float sums[GROUPS][DP];
  __shared__ float lse[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if ((int)blockIdx.x < joins) {
    const int bh = blockIdx.x, b = bh / a.H, head = bh % a.H;
    const int n = paged_length(a, b), parts = paged_parts(a, n);
    if (parts <= 1) return;  // (written at once)
    const int hk = head / a.G, q_row = head % a.G, col = tid % DP, first = tid / DP;
    const int64_t at = ((int64_t)(b * a.c.heads + hk) * a.groups + q_row / 16) * a.splits * a.rows + q_row % 16;
    // (the first of a thread's parts are requested before the maximum is known)
    constexpr int EARLY = 8;
    float early[EARLY], scale[EARLY];
#pragma unroll
    for (int i = 0; i < EARLY; ++i) {
      const int64_t p = at + (int64_t)min(first + i * GROUPS, parts - 1) * a.rows;
      early[i] = a.part_o[p * DP + col], scale[i] = a.part_ml[p].x;
    }
    const float2 ml = paged_join(a.part_ml + at, parts, a.rows, lane);
    float o = 0.0f;
#pragma unroll
    for (int i = 0; i < EARLY; ++i)
      if (first + i * GROUPS < parts) o += early[i] * __builtin_amdgcn_exp2f(scale[i] - ml.x);
#pragma unroll 4
    for (int p = first + EARLY * GROUPS; p < parts; p += GROUPS)
      o += a.part_o[(at + (int64_t)p * a.rows) * DP + col] * __builtin_amdgcn_exp2f(a.part_ml[at + (int64_t)p * a.rows].x - ml.x);
    if (GROUPS > 1) {
      sums[first][col] = o;
      __syncthreads();
      if (first > 0) return;
#pragma unroll
      for (int g = 1; g < GROUPS; ++g) o += sums[g][col];
    }
    if (col < a.c.d) store_from_f32<QDT>(a.out, b * a.so_z + head * a.so_h + col, ml.y == 0.0f ? 0.0f : o * (a.c.v_scale / ml.y));
    return;
  }
  const int per_head = (a.c.capacity() + 255) / 256, bh = (blockIdx.x - joins) / per_head;
  const int b = bh / a.c.heads, hk = bh % a.c.heads;
  const int t0 = (blockIdx.x - joins - bh * per_head) * 256, t = t0 + tid;
  const int n = paged_length(a, b);
  if (t0 >= n) return;
  const int parts = paged_parts(a, n);
  const int64_t first = (int64_t)b * a.H + hk * a.G;
  // (What does not wait for the sums is requested before them: the scores of the first heads and the weight that grows.)
  constexpr int EARLY = 8;
  float early[EARLY], sum = 0.0f, old = 0.0f;
  float* const to = weights + b * sw_b + hk * sw_h + t;
  const float* const scores = a.scores + first * a.cap_pad + t;
#pragma unroll
  for (int g = 0; g < EARLY; ++g) early[g] = t < n && g < a.G ? scores[(int64_t)g * a.cap_pad] : -INFINITY;
  if (t < n) old = *to;
  for (int g0 = 0; g0 < a.G; g0 += 256) {  // (up to 256 heads of a group at a time)
    const int many = min(256, a.G - g0);
    if (g0 > 0) __syncthreads();
    if (parts == 1) {
      if (tid < many) lse[tid] = a.lse[first + g0 + tid];
    } else {
      for (int g = wave; g < many; g += 4) {
        const int64_t at = ((int64_t)bh * a.groups + (g0 + g) / 16) * a.splits * a.rows + (g0 + g) % 16;
        const float2 ml = paged_join(a.part_ml + at, parts, a.rows, lane);
        if (lane == 0) lse[g] = ml.x + __builtin_amdgcn_logf(ml.y);
      }
    }
    __syncthreads();
    auto add = [&](float x, int g) { sum += x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - lse[g]); };
    if (g0 == 0) {
#pragma unroll
      for (int g = 0; g < EARLY; ++g)
        if (g < many) add(early[g], g);
    }
    if (t < n)
#pragma unroll 4
      for (int g = g0 == 0 ? EARLY : 0; g < many; ++g) add(scores[(int64_t)(g0 + g) * a.cap_pad], g);
  }
  if (t < n) *to = old + sum;
}

// ---- host side ------------------------------------------------------------------------------------------------------------

struct PagedPlan {
  int rows, groups, share, splits, dp, cap_pad;
  int mode;
  size_t o_bytes, ml_bytes, score_bytes, lse_bytes;
  size_t total() const { return o_bytes + ml_bytes + score_bytes + lse_bytes; }
};

static bool paged_batch(int64_t B, int64_t H) {
  constexpr int64_t kMost = 1ll << 20;
  return B > 0 && H > 0 && B < kMost && H < kMost && B * H < kMost;
}

static size_t granules(size_t b) { return (b + 255) / 256 * 256; }

// `aligned`: keys and values begin at multiples of 16 bytes.
static bool paged_in_tiles(const Paged& c, int es, bool aligned) {
  const lh_strides3& s = c.sk;
  return aligned && c.size % 16 == 0 && c.d * es % 16 == 0 && s.z == c.sv.z && s.h == c.sv.h && s.t == c.sv.t && s.z * es % 16 == 0 && s.h * es % 16 == 0 &&
         s.t * es % 16 == 0 && 16 * s.t * es < 0x40000000 && s.t >= c.d;
}

// How many positions a workgroup takes of a sequence; `items` (sequence, head, group of queries), `per_cu` workgroups that a CU
// holds at once, `row_bytes` of a position's key and value.  There are to be two workgroups per CU (one, if no more fit; one also where the
// shares would be shorter than 1024 positions, of which their start and end take too much).  (One sequence of 1000, 12 heads of 64: 7.6 us with 128
// positions a share, 9.8 in one; one of 32768, 8 heads of 128: 31.8 with 1024, 33.5 with 512, 362 in one; 4 of 1024 to 4096, 8 heads of 128 with 4 queries: 14.8 with
// 512, 15.8 with 256; heads of 256, 16 sequences of 1024 to 4096: 73 with 2048, 94 with 512.)  With items enough for that, up to 8 per CU
// even out sequences of unlike length, while a share has 512 KB of keys and values, which the join's launch costs nothing against.  (16
// sequences of 8192 to 32768, 8 heads of 128: 255 with 2048, 263 with 512, 384 in one; 64 of 256 to 1024, 12 heads of 64, 30 in one, 33 with 512.)
static int paged_share(int64_t items, int capacity, int per_cu, int64_t row_bytes) {
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

static PagedPlan paged_plan(const Paged& c, int cache_dtype, int64_t B, int64_t H, bool with_weights, bool aligned) {
  PagedPlan p = {};
  const int G = (int)(H / c.heads);
  p.rows = G < 16 ? G : 16, p.groups = (G + 15) / 16;
  p.dp = c.d <= 64 ? 64 : c.d <= 128 ? 128 : 256;
  const int es = (int)dtype_size(cache_dtype);
  p.mode = paged_in_tiles(c, es, aligned) ? kTiles : c.d * es % 16 == 0 && c.d % (p.dp / 16) == 0 ? kWholeRows : kOddRows;
  const int64_t items = B * c.heads * p.groups;
  p.share = paged_share(items, c.capacity(), paged_occupancy(cache_dtype, p.dp, p.mode), 2 * (int64_t)c.d * es);
  p.splits = (int)(((int64_t)c.capacity() + p.share - 1) / p.share);
  if (p.splits > 1) {
    p.o_bytes = granules((size_t)items * p.splits * p.rows * p.dp * 4);
    p.ml_bytes = granules((size_t)items * p.splits * p.rows * 8);
  }
  if (with_weights) {
    p.cap_pad = (c.capacity() + 31) / 32 * 32;
    p.score_bytes = granules((size_t)B * H * p.cap_pad * 4);
    p.lse_bytes = granules((size_t)B * H * 4);
  }
  return p;
}

template <int CDT, int QDT, int DP>
static int launch_paged(const PagedAttnArgs& a, int mode, float* weights, int64_t sw_b, int64_t sw_h, hipStream_t s) {
  const dim3 grid((unsigned)((int64_t)a.B * a.c.heads * a.groups * a.splits)), block(kPagedWaves * 64);
  if (mode == kTiles) LH_LAUNCH((paged_attention_kernel<CDT, QDT, DP, kPagedWaves, kTiles>), grid, block, 0, s, a);
  else if (mode == kWholeRows) LH_LAUNCH((paged_attention_kernel<CDT, QDT, DP, kPagedWaves, kWholeRows>), grid, block, 0, s, a);
  else LH_LAUNCH((paged_attention_kernel<CDT, QDT, DP, kPagedWaves, kOddRows>), grid, block, 0, s, a);
  if (const int rc = check_launch("paged_attention")) return rc;
  const int joins = a.splits > 1 ? a.B * a.H : 0;
  const unsigned blocks = joins + (weights ? (unsigned)((a.c.capacity() + 255) / 256 * (int64_t)a.B * a.c.heads) : 0u);
  if (blocks == 0) return LH_OK;
  LH_LAUNCH((paged_attention_finish<QDT, DP>), dim3(blocks), dim3(256), 0, s, a, joins, weights, sw_b, sw_h);
  return check_launch("paged_attention_finish");
}

template <int CDT, int QDT>
static int launch_paged_dp(const PagedAttnArgs& a, int dp, int mode, float* w, int64_t sw_b, int64_t sw_h, hipStream_t s) {
  if (dp == 64) return launch_paged<CDT, QDT, 64>(a, mode, w, sw_b, sw_h, s);
  if (dp == 128) return launch_paged<CDT, QDT, 128>(a, mode, w, sw_b, sw_h, s);
  return launch_paged<CDT, QDT, 256>(a, mode, w, sw_b, sw_h, s);
}

}  // namespace lh

using namespace lh;

extern "C" {

size_t lh_hip_paged_attention_workspace_bytes(const lh_paged_cache* cache, int64_t B, int64_t H, int32_t with_weights) {
  Paged c;
  if (paged_cache(cache, "lh_hip_paged_attention_workspace_bytes", &c) != LH_OK) return 0;
  if (!paged_batch(B, H) || H % c.heads != 0) return 0;
  // (Room for either alignment: a caller may size it with one cache and pass a view of another.)
  const size_t one = paged_plan(c, cache->dtype, B, H, with_weights != 0, true).total(), other = paged_plan(c, cache->dtype, B, H, with_weights != 0, false).total();
  return one > other ? one : other;
}

int lh_hip_paged_attention(const lh_paged_cache* cache, void* out, const void* q, int64_t out_stride_b, int64_t out_stride_h,
                           int64_t q_stride_b, int64_t q_stride_h, const int32_t* lengths, float* weights, int64_t weights_stride_b, int64_t weights_stride_h,
                           int64_t B, int64_t H, float scale, int32_t dtype, void* workspace, size_t workspace_bytes,
                           void* stream) {
  PagedAttnArgs a = {};
  if (const int rc = paged_cache(cache, "lh_hip_paged_attention", &a.c)) return rc;
  if (B == 0) return LH_OK;
  LH_REQUIRE(out && q && lengths, "lh_hip_paged_attention: null pointer");
  LH_REQUIRE(B >= 0 && H > 0 && H % a.c.heads == 0, "lh_hip_paged_attention: %lld heads are no multiple of %d key / value heads", (long long)H, a.c.heads);
  LH_REQUIRE(paged_batch(B, H), "lh_hip_paged_attention: bad batch (fewer than 2^20 heads of sequences)");
  LH_REQUIRE(dtype == cache->dtype || (cache->dtype == LH_F8E4M3 && (dtype == LH_BF16 || dtype == LH_F16)),
             "lh_hip_paged_attention: queries must have the cache's dtype (bf16 or f16 for a cache of e4m3)");
  LH_REQUIRE(weights == nullptr || ((a.c.heads == 1 || weights_stride_h >= a.c.capacity()) && (B <= 1 || weights_stride_b >= a.c.capacity())),
             "lh_hip_paged_attention: rows of the weights overlap");
  LH_REQUIRE(weights == nullptr || (a.c.capacity() + 255) / 256 * B * a.c.heads < (1ll << 23), "lh_hip_paged_attention: too many weights (fewer than 2^31)");
  const PagedPlan p = paged_plan(a.c, cache->dtype, B, H, weights != nullptr, aligned16(a.c.k) && aligned16(a.c.v));
  LH_REQUIRE(p.total() == 0 || (workspace != nullptr && (reinterpret_cast<uintptr_t>(workspace) & 255) == 0 && workspace_bytes >= p.total()),
             "lh_hip_paged_attention: workspace too small or not 256-byte aligned: %zu of %zu bytes", workspace_bytes, p.total());
  a.out = out, a.q = q, a.so_z = out_stride_b, a.so_h = out_stride_h, a.sq_z = q_stride_b, a.sq_h = q_stride_h, a.lengths = lengths;
  a.B = (int32_t)B, a.H = (int32_t)H, a.G = (int32_t)(H / a.c.heads);
  a.rows = p.rows, a.groups = p.groups, a.share = p.share, a.splits = p.splits, a.cap_pad = p.cap_pad;
  a.scale_log2e = (float)((double)scale * a.c.k_scale * 1.4426950408889634);
  char* ws = static_cast<char*>(workspace);
  if (p.splits > 1) a.part_o = reinterpret_cast<float*>(ws), a.part_ml = reinterpret_cast<float2*>(ws + p.o_bytes);
  if (weights) a.scores = reinterpret_cast<float*>(ws + p.o_bytes + p.ml_bytes), a.lse = reinterpret_cast<float*>(ws + p.o_bytes + p.ml_bytes + p.score_bytes);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int64_t sb = weights_stride_b, sh = weights_stride_h;
  if (cache->dtype == LH_F8E4M3)
    return dtype == LH_BF16 ? launch_paged_dp<LH_F8E4M3, LH_BF16>(a, p.dp, p.mode, weights, sb, sh, s)
                            : launch_paged_dp<LH_F8E4M3, LH_F16>(a, p.dp, p.mode, weights, sb, sh, s);
  if (dtype == LH_BF16) return launch_paged_dp<LH_BF16, LH_BF16>(a, p.dp, p.mode, weights, sb, sh, s);
  if (dtype == LH_F16) return launch_paged_dp<LH_F16, LH_F16>(a, p.dp, p.mode, weights, sb, sh, s);
  return launch_paged_dp<LH_F32, LH_F32>(a, p.dp, p.mode, weights, sb, sh, s);
}

}  // extern "C"
