// Attention of packed chunks of new tokens over a paged cache, for one pair of types (the cache's LH_CHUNK_CDT, the queries' LH_CHUNK_QDT).
//
// The rows of a sequence and key / value head are its tokens' queries of the G heads that share it, token by token: row r is token r / G.  A
// workgroup takes a tile of them and walks over the positions up to the last one that any of them sees:
//
//  * Both products are transposed, S^T = K Q^T and O^T = V^T P^T on 32-wide matrix instructions: a lane has one row, its softmax state
//    is a scalar per lane, and the accumulators of S^T are, as sums of 16-bit values, the second operand of O^T.
//  * Keys and values of a step go through registers into LDS, two steps of which are there where that costs a CU no workgroup (the next one's are
//    put there between the two products: 2 % of a short step's time, less of a long one's); they are asked for up to two steps ahead, as far as
//    registers suffice.  Where each position's row lies is looked up before that, one position a thread, so
//    that any page size and any strides cost the same.
//  * 128 rows a workgroup, 32 for each of four waves, 64 positions a step, which all waves read.  (Sequences with few rows have a kernel
//    without LDS, in chunk_attention_few.hip.)
//  * Long caches of few tiles are cut into shares of positions; a second launch joins them.
//
// The arithmetic bounds it: a step of a wave has 48 matrix instructions of 32 cycles at width 128 beside about 290 vector instructions, 32 of them
// exponentials, and the two hardly overlap (2048 tokens after 14336, f16, 32 heads of 128: matrix unit 45 % of the cycles, vector unit 43 %).
// P is held in f32 and enters the second product as the sum of two 16-bit values, each nearest to what is left: off by 2^-16 of it at most in bf16,
// 2^-18 in the mean, and by 2^-22 in f16.  One value would leave 2^-8 and make the result's error against 64 bits up to 1.4 times that of its own
// rounding, 1.0 times with two, and the same row would differ from what the kernel for few rows makes of it (the same 2048 tokens in bf16 609 us with
// one, 757 to 783 with two; 8 prompts of 1024, bf16, 12 heads of 64, 28.6 and 34.0).  A third of bf16 takes 964 and 40.1 us and changes neither of the
// error's first two places.  Everything that was not needed in a step for which nothing has to be masked is behind a uniform branch.
//
// Measured: those 2048 tokens in f16 810 us (636 TFLOP/s of the products that the mask leaves, with half as many again made; 1180 is what a large f16
// product reaches); those prompts 34.0 us (380 TFLOP/s: steps of 24 matrix instructions, half of a tile's last two are masked); 512 tokens each of two
// sequences of 4096 and 2458 positions, e4m3, 16 heads of 128, 70 us and 13 for the join, which moves 34 MB.
#include "chunk_attention.h"

#ifndef LH_CHUNK_CDT
#error "compiled with -DLH_CHUNK_CDT=... -DLH_CHUNK_QDT=... -DLH_CHUNK_NAME=..."
#endif

namespace lh {
namespace {

constexpr int CDT = LH_CHUNK_CDT, QDT = LH_CHUNK_QDT;
constexpr bool F32 = CDT == LH_F32;
constexpr int CES = CDT == LH_F8E4M3 ? 1 : F32 ? 4 : 2;  // bytes of an element in the cache
constexpr int QES = F32 ? 4 : 2;                         // of a query's, and in LDS
constexpr int PE = F32 ? 4 : 8;                          // elements of a piece: 16 bytes in LDS
constexpr int PW = PE * CES / 4;                         // its words in the cache
// The 16-bit type of values and probabilities in the second product, of which a probability is the sum of two.  (Codes of e4m3 are exact in either
// type; in f16 the sum has 22 places instead of 18.)
constexpr int PDT = CDT == LH_F8E4M3 ? LH_F16 : QDT, PARTS = 2;

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ f32x16 mma(u32x4 x, u32x4 y, f32x16 c) {
  if constexpr (DT == LH_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
}

// (By value: a bit cast of a vector's element itself reads its first one.)
__device__ __forceinline__ float f32_of(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ __forceinline__ uint32_t bits_of(float x) { return __builtin_bit_cast(uint32_t, x); }

// The same number, which the compiler takes for another: comparisons with it are made where they are used and not held over the loop (a
// pair of scalar registers each; where those did not suffice, hipcc of ROCm 7.2 put copies of vector registers at the wrong side of the
// lanes' return from a branch).
__device__ __forceinline__ int hide(int x) {
  asm volatile("" : "+s"(x));
  return x;
}

// Waits for this wave's LDS accesses and for the workgroup, but for no load on its way to registers.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A piece of W words whose elements are of ES bytes, moved down by `skip` elements (those behind them become 0).
template <int W, int ES>
__device__ __forceinline__ void move_down(uint32_t* w, int skip) {
  const int bits = skip * ES * 8;
#pragma unroll
  for (int step = 2; step >= 1; step /= 2)
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const uint32_t from = i + step < W ? w[i + step] : 0u;
      w[i] = bits / 32 & step ? from : w[i];
    }
  if constexpr (ES < 4) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = (uint32_t)(((uint64_t)(i + 1 < W ? w[i + 1] : 0u) << 32 | w[i]) >> (bits & 31));
  }
}

// Columns col .. col + PE - 1 of a row of d elements of ES bytes; those behind its end are 0.  The row is there in any case.  ODD: d is no multiple
// of a piece; the last piece is loaded so that it ends with the row and moved down.  SHORT: a row may be shorter than a piece.
template <int ES, bool ODD, bool SHORT>
__device__ __forceinline__ void load_columns(uint32_t* w, const uint8_t* row, int col, int d) {
  constexpr int W = PE * ES / 4;
  if (SHORT && d < PE) {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0;
#pragma unroll
    for (int e = 0; e < PE; ++e)
      if (col + e < d) {
        if constexpr (ES == 4) w[e] = reinterpret_cast<const uint32_t*>(row)[col + e];
        else if constexpr (ES == 2) w[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[col + e] << (16 * (e % 2));
        else w[e / 4] |= (uint32_t)row[col + e] << (8 * (e % 4));
      }
    return;
  }
  const int from = ODD ? min(col, d - PE) : col < d ? col : 0;
  if constexpr (W == 4) {
    const typename Chunk<ES>::type v = *reinterpret_cast<const typename Chunk<ES>::type*>(row + from * ES);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = v[i];
  } else {
    typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
    const u32x2_any v = *reinterpret_cast<const u32x2_any*>(row + from * ES);
    w[0] = v[0], w[1] = v[1];
  }
}
// What of it is not in the row becomes 0, all of it if `there` is (otherwise ones), apart from the load, so that nothing waits for that.  (Masks in
// vector registers: as conditions they would take a pair of scalar ones each.)
template <int ES, bool ODD, bool SHORT>
__device__ __forceinline__ void settle_columns(uint32_t* w, int col, int d, uint32_t there) {
  constexpr int W = PE * ES / 4;
  if (ODD && (!SHORT || d >= PE)) {
    const int skip = max(col - (d - PE), 0);
    if (skip > 0) move_down<W, ES>(w, min(skip, PE - 1));
  }
  const uint32_t keep = there & (uint32_t)((col - d) >> 31);
#pragma unroll
  for (int i = 0; i < W; ++i) w[i] &= keep;
}

// Two e4m3 codes (the lower or upper two of a word) as two values of a 16-bit type: exact.
template <int DT, bool HI>
__device__ __forceinline__ uint32_t of_e4m3(uint32_t w) {
  if constexpr (DT == LH_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}
template <int DT>
__device__ __forceinline__ u32x4 in_lds(const uint32_t* w) {
  if constexpr (CDT == LH_F8E4M3) return u32x4{of_e4m3<DT, false>(w[0]), of_e4m3<DT, true>(w[0]), of_e4m3<DT, false>(w[1]), of_e4m3<DT, true>(w[1])};
  else return u32x4{w[0], w[1], w[2], w[3]};
}
// Not 0 where a piece of values in LDS holds an infinity or a NaN: an exponent of ones carries into the sign's place.
__device__ __forceinline__ uint32_t wild_bits(u32x4 w) {
  constexpr uint32_t top = F32 ? 0x7f800000u : PDT == LH_BF16 ? 0x7f807f80u : 0x7c007c00u, one = F32 ? 0x00800000u : PDT == LH_BF16 ? 0x00800080u : 0x04000400u;
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bits |= (w[i] & top) + one;
  return bits & (F32 ? 0x80000000u : 0x80008000u);
}

// Workgroups that a CU holds, by their registers.
constexpr int occupancy(int blocks, bool odd) { return blocks <= 2 && !F32 && !odd ? 3 : blocks <= 4 ? 2 : 1; }
// Steps ahead whose keys and values are on their way to registers: as many as these suffice for.  0: they are asked for when their place is free.
constexpr int ahead(int blocks, bool odd) { return F32 || (CES == 1 && odd && blocks == 4) ? 0 : blocks == 3 ? 2 : blocks <= 6 ? 1 : 0; }

constexpr int KEYS = 64;  // positions of a step
// Elements from one row to the next: of keys, whose rows are read 16 bytes a lane, so that neighbours lie 4 (f32: 8) banks apart; of values, of
// which 16-bit ones are read four rows at a time, 64 bytes of each: 16 or 48 banks apart.
constexpr int k_row_elems(int blocks) { return 32 * blocks + 8; }
constexpr int v_row_elems(int blocks) { return F32 ? 32 * blocks + 8 : blocks == 3 ? 96 : 32 * blocks + 32; }
constexpr size_t stage_bytes(int blocks) { return (size_t)KEYS * (k_row_elems(blocks) + v_row_elems(blocks)) * QES; }
// Steps that are in LDS: the next one beside the one that is read, where two do not cost a CU a workgroup.
constexpr int stages(int blocks, bool odd) { return 2 * stage_bytes(blocks) <= (occupancy(blocks, odd) == 3 ? 51000 : occupancy(blocks, odd) == 2 ? 77000 : 153000) ? 2 : 1; }
constexpr size_t lds_bytes(int blocks, bool odd) { return stages(blocks, odd) * stage_bytes(blocks); }

// DB: width in 32 columns.
template <int CACHE, int QUERY, int DB, bool ODD>  // (the types: for the name)
__global__ void __launch_bounds__(256, occupancy(DB, ODD)) chunk_attention_kernel(ChunkArgs a) {
  constexpr int D = 32 * DB, KROW = k_row_elems(DB), VROW = v_row_elems(DB);
  constexpr int NI = KEYS / 32;                   // 32-position tiles
  constexpr int CPR = D / PE;                     // pieces of a row
  constexpr int NP = KEYS * CPR / 256;            // pieces a thread brings, of keys and of values
  constexpr int SD = F32 ? D / 8 : D / 16;
  constexpr int RS = ahead(DB, ODD), STAGES = stages(DB, ODD);
  constexpr bool SHORT = ODD && DB == 2;
  constexpr bool TWO = STAGES == 2 || RS == 2;    // steps go by in pairs
  constexpr bool MIDDLE = STAGES == 2 && RS > 0;
  static_assert(NI >= 1 && NP * 256 == KEYS * CPR, "");
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  typedef typename std::conditional<F32, float, uint16_t>::type elem;
  __shared__ int64_t k_at[2][KEYS], v_at[2][KEYS];  // where the rows of a step lie, in elements; 0 where there is none
  __shared__ uint64_t held[8];           // which positions of a step there are (noted up to four steps before they are read)
  __shared__ int32_t wild[2][4], first_wild[D];

  const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int items = a.slots * a.c.heads, split = blockIdx.x / items, item = blockIdx.x - split * items;
  const int hk = item % a.c.heads;
  int b, tile;
  if (!chunk_tile(a, item / a.c.heads, &b, &tile)) return;
  const int start = __builtin_amdgcn_readfirstlane(chunk_start(a, b));
  const int count = max(__builtin_amdgcn_readfirstlane(chunk_start(a, b + 1)) - start, 0);
  const int first = tile << a.tile_shift, rows = min(a.tile_rows, count * a.G - first);
  const int length = __builtin_amdgcn_readfirstlane(min(max(a.lengths[b], 0), a.c.capacity()));
  const int base = length - count;  // position of the sequence's first new token
  const int sees = base + (int)a.by_group.div((uint32_t)(first + rows - 1)) + 1;  // positions that the last row sees
  const int k0 = split * a.share;
  if (k0 >= sees && split > 0) return;
  const int k1 = k0 + max(min(sees - k0, a.share), 0);
  const bool cut = sees > a.share;

  const int row0 = 32 * wave;  // of the wave, in the tile
  const int row = first + row0 + r32;
  const bool row_live = row0 + r32 < rows;
  const int token = (int)a.by_group.div((uint32_t)row), head = hk * a.G + (row - token * a.G);
  const int last_seen = row_live ? min(base + token, k1 - 1) : -1;
  const bool wave_live = row0 < rows;
  const int wave_first = base + (int)a.by_group.div((uint32_t)(first + min(row0, rows - 1)));                  // what its first row sees
  const int wave_last = min(base + (int)a.by_group.div((uint32_t)(first + min(row0 + 31, rows - 1))), k1 - 1);  // and its last one

  // Queries: lane (r32, h) has columns 16 s + 8 h .. + 7 of its row (f32: 8 s + 4 h .. + 3); where the registers do not suffice for them, they are
  // read again in every step.
  constexpr bool Q_HELD = F32 ? DB <= 3 || DB == 6 : !(DB == 8 && ODD);
  const uint8_t* const q = static_cast<const uint8_t*>(a.q) + ((start + (row_live ? token : 0)) * a.sq_n + (row_live ? head : hk * a.G) * a.sq_h) * QES;
  auto query = [&](const uint8_t* from, int s, int d) {
    const int col = (2 * s + h) * PE;
    uint32_t w[4];
    load_columns<QES, ODD, SHORT>(w, from, col, d);
    settle_columns<QES, ODD, SHORT>(w, col, d, row_live ? ~0u : 0u);
    // (A scale below 0 is that of the queries, so that -inf is the score of what a row does not see; with one of 0 they are 0.)
    return (u32x4{w[0], w[1], w[2], w[3]} & a.q_and) ^ a.q_xor;
  };
  u32x4 qf[Q_HELD ? SD : 1];
  if constexpr (Q_HELD)
#pragma unroll
    for (int s = 0; s < SD; ++s) qf[s] = query(q, s, a.c.d);

  f32x16 acc[DB];
#pragma unroll
  for (int j = 0; j < DB; ++j)
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[j][v] = 0.0f;
  // What p is relative to: the maximum, or, in f16, 2^12 below it, so that small probabilities keep their part in a long row (the
  // smallest number of f16 is 2^-24).  It moves only when a p would pass 2^slack.
  constexpr float below = PDT == LH_F16 ? 12.0f : 0.0f, slack = PDT == LH_F16 ? 14.0f : 10.0f;
  float m_run = row_live ? -INFINITY : 0.0f, l_run = 0.0f;  // (a row that is none waits for no maximum)

  const int steps = (k1 - k0 + KEYS - 1) / KEYS;
  const int64_t table_row = b * a.c.table_stride;
  const uint8_t* const kb = static_cast<const uint8_t*>(a.c.k) + hk * a.c.sk.h * CES;
  const uint8_t* const vb = static_cast<const uint8_t*>(a.c.v) + hk * a.c.sv.h * CES;
  // Position k0 + step KEYS + tid, for tid < KEYS: its page, or -1; then where it lies.
  auto look_up = [&](int step) {
    const int key = k0 + step * KEYS + tid;
    return tid < KEYS && key < k1 ? a.c.table[table_row + a.c.by_size.div((uint32_t)key)] : -1;
  };
  auto note = [&](int step, int page) {
    if (tid >= KEYS) return;
    const int key = k0 + step * KEYS + tid;
    const bool there = key < k1 && (uint32_t)page < (uint32_t)a.c.pages;
    const int slot = there ? key - (int)a.c.by_size.div((uint32_t)key) * a.c.size : 0;
    k_at[step & 1][tid] = there ? page * a.c.sk.z + slot * a.c.sk.t : 0;
    v_at[step & 1][tid] = there ? page * a.c.sv.z + slot * a.c.sv.t : 0;
    const uint64_t some = __builtin_amdgcn_ballot_w64(there);
    if (lane == 0) held[step & 7] = some;
  };
  uint32_t kr[RS > 0 ? RS : 1][RS > 0 ? NP : 1][PW], vr[RS > 0 ? RS : 1][RS > 0 ? NP : 1][PW];
  auto request = [&](int step, int i, uint32_t* k, uint32_t* v) {
    const int piece = tid + 256 * i, key = piece / CPR, col = (piece - key * CPR) * PE;
    const int64_t k_row = k_at[step & 1][key], v_row = v_at[step & 1][key];
    const int d = hide(a.c.d);
    load_columns<CES, ODD, SHORT>(k, kb + k_row * CES, col, d);
    load_columns<CES, ODD, SHORT>(v, vb + v_row * CES, col, d);
  };
  auto put = [&](elem* Ks, int i, uint32_t* k, uint32_t* v, uint64_t some, bool full, bool look) {  // into LDS; not 0 where a value is an infinity or a NaN, if asked for
    const int piece = tid + 256 * i, key = piece / CPR, col = (piece - key * CPR) * PE;
    if (!full) {
      const int d = hide(a.c.d);
      const uint32_t there = 0u - ((uint32_t)(some >> key) & 1u);
      settle_columns<CES, ODD, SHORT>(k, col, d, there);
      settle_columns<CES, ODD, SHORT>(v, col, d, there);
    }
    const u32x4 kw = in_lds<QDT>(k), vw = in_lds<PDT>(v);
    *reinterpret_cast<u32x4*>(Ks + key * KROW + col) = kw;
    *reinterpret_cast<u32x4*>(Ks + KEYS * KROW + key * VROW + col) = vw;
    return look ? wild_bits(vw) : 0u;
  };
  // Some row does not see all of a step's positions: those it does not see must not reach it by a 0 times an infinity.
  auto partial = [&](int step) { return k0 + (step + 1) * KEYS > base + (int)a.by_group.div((uint32_t)first) + 1; };
  elem* const stage0 = reinterpret_cast<elem*>(smem);
  constexpr int kStage = STAGES == 2 ? KEYS * (KROW + VROW) : 0;  // elements from one stage to the other
  // A step's keys and values into its stage, those RS steps later on their way.
  auto bring = [&](int step, auto set) {
    constexpr int S = decltype(set)::value;
    elem* const Ks = stage0 + (step & 1) * kStage;
    const bool look = partial(step);
    const uint64_t some = held[step & 7];
    const bool full = __builtin_amdgcn_readfirstlane(a.c.d == D && some == ~0ull);  // nothing of the step has to become 0
    uint32_t odd_one = 0;
    if constexpr (RS > 0) {
#pragma unroll
      for (int i = 0; i < NP; ++i) odd_one |= put(Ks, i, kr[S % RS][i], vr[S % RS][i], some, full, look);
      if (step + RS < steps)
#pragma unroll
        for (int i = 0; i < NP; ++i) request(step + RS, i, kr[S % RS][i], vr[S % RS][i]);
    } else {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        uint32_t k[PW], v[PW];
        request(step, i, k, v);
        odd_one |= put(Ks, i, k, v, some, full, look);
        if (i % (ODD ? 2 : 4) == 1) asm volatile("" ::: "memory");  // (a few of each on their way at once)
      }
    }
    if (look) {
      const bool found = __any(odd_one != 0);
      if (lane == 0) wild[TWO ? step & 1 : 0][wave] = found;
    }
  };
  typedef std::integral_constant<int, 0> even_t;

  // What the table says for later steps: asked for as long ahead as keys and values are, since what is asked for later comes later.
  constexpr int QUEUE = RS > 0 ? RS : 1;
  int queue[QUEUE];
  if (steps > 0) {
    int pages[RS + 2];
#pragma unroll
    for (int i = 0; i < RS + 2; ++i) pages[i] = look_up(i);
#pragma unroll
    for (int i = 0; i < QUEUE; ++i) queue[i] = look_up(RS + 2 + i);
    note(0, pages[0]);
    note(1, pages[1]);
    lds_barrier();
    if constexpr (RS > 0) {
#pragma unroll
      for (int r = 0; r < RS; ++r)
        if (r < steps)
#pragma unroll
          for (int i = 0; i < NP; ++i) request(r, i, kr[r][i], vr[r][i]);
      lds_barrier();  // (where the first ones lie has been read)
#pragma unroll
      for (int i = 2; i < RS + 2; ++i) note(i, pages[i]);
      lds_barrier();
    }
    bring(0, even_t());
  }
  // Step `step`, whose parity is known to the compiler.
  auto take = [&](int step, auto parity) {
    constexpr int P = decltype(parity)::value;
    elem* const Ks = stage0 + P * kStage;
    elem* const Vs = Ks + KEYS * KROW;
    const int j0 = k0 + step * KEYS;
    lds_barrier();  // this step is in its place; the one before has been read
    bool some_wild = false;
    if (partial(step)) some_wild = wild[P][0] | wild[P][1] | wild[P][2] | wild[P][3];
    if (__builtin_expect(some_wild, 0)) {
      // Such values become 0; a column's first one makes a NaN of the rows that see it (below).
      for (int c = tid; c < D; c += 256) first_wild[c] = 0x7fffffff;
      lds_barrier();
#pragma unroll 1
      for (int c = tid; c < KEYS * D; c += 256) {
        elem* const x = Vs + c / D * VROW + c % D;
        const uint32_t bits = F32 ? __builtin_bit_cast(uint32_t, (float)*x) : (uint32_t)*x, top = F32 ? 0x7f800000u : PDT == LH_BF16 ? 0x7f80u : 0x7c00u;
        if ((bits & top) == top) {
          *x = 0;
          atomicMin(&first_wild[c % D], c / D);
        }
      }
      lds_barrier();
    }
    const uint64_t all_held = held[step & 7];
    const bool some_row = wave_live && wave_last >= j0;
    f32x16 s[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[i][v] = 0.0f;
    if (some_row) {
      const uint8_t* q_now = q;
      int d_now = a.c.d;
      if constexpr (!Q_HELD) asm volatile("" : "+v"(q_now), "+s"(d_now));  // (read here, not held over the steps)
#pragma unroll
      for (int e = 0; e < SD; ++e) {
        u32x4 qe;
        if constexpr (Q_HELD) qe = qf[e];
        else qe = query(q_now, e, d_now);
        if (!Q_HELD && (F32 || e % 2 == 1)) asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const u32x4 kf = *reinterpret_cast<const u32x4*>(Ks + (32 * i + r32) * KROW + (2 * e + h) * PE);
          if constexpr (F32) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
              s[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(f32_of(kf[t]), f32_of(qe[t]), s[i], 0, 0, 0);
          } else {
            s[i] = mma<QDT>(kf, qe, s[i]);
          }
        }
      }
      if constexpr (!F32 && Q_HELD) {  // (keys are read from LDS four matrix instructions ahead)
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int e = 0; e < NI * SD - 4; ++e) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);
      }
    }
    // (While the products are made; the other stage has been read.)
    if constexpr (MIDDLE) {
      if (step + 1 < steps) bring(step + 1, std::integral_constant<int, TWO ? 1 - P : 0>());
    }
    if (some_row) {
      // s[i][v] = q . k of row r32 and position j0 + 32 i + 8 (v / 4) + 4 h + v % 4
      const bool whole = j0 + 32 * NI - 1 <= min(wave_first, k1 - 1) && row0 + 31 < rows && all_held == ~0ull;
      if (!whole) {
        // Bit p of `seen`: whether the row sees position j0 + p.
        uint64_t seen = last_seen < j0 ? 0ull : last_seen - j0 >= 63 ? ~0ull : (2ull << (last_seen - j0)) - 1;
        seen = (seen & all_held) >> (4 * h);
        const uint32_t half[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int bit = 8 * (v >> 2) + (v & 3);
            const uint32_t keep = (uint32_t)((int32_t)(half[i] << (31 - bit)) >> 31);  // (bit by bit, no condition)
            s[i][v] = f32_of((bits_of(s[i][v]) & keep) | (0xff800000u & ~keep));
          }
      }
      // The maximum is followed with a delay: nothing moves until a p would pass 2^10, which is as accurate as one of 1.  (Row by row, so that what
      // others see does not reach a row's roundings.)
      float mx = s[0][0];
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) mx = fmaxf(mx, s[i][v]);
      mx *= a.scale_log2e;
      if (__any(mx > m_run + slack)) {
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m_new = mx > m_run + slack ? mx - below : m_run;
        const float safe = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m_run - safe);
        l_run *= alpha;
#pragma unroll
        for (int j = 0; j < DB; ++j) acc[j] *= alpha;
        m_run = m_new;
      }
      const float off = m_run == -INFINITY ? 0.0f : m_run;  // (nothing seen yet: every p is exp2(-inf))
      // p takes the place of s: one rounding of s scale - maximum.
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          s[i][v] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][v], a.scale_log2e, -off));
          l_run += s[i][v];
        }
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const float* vrow = reinterpret_cast<const float*>(Vs) + (32 * i + 8 * (v >> 2) + 4 * h + (v & 3)) * VROW + r32;
#pragma unroll
            for (int j = 0; j < DB; ++j) acc[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(vrow[32 * j], s[i][v], acc[j], 0, 0, 0);
            if (v % (DB > 6 ? 2 : 4) == (DB > 6 ? 1 : 3)) asm volatile("" ::: "memory");  // (values of a few positions fetched ahead)
          }
      } else {
        // Values through the transposing read: lane (g4 = lane / 16, j16 = lane % 16) addresses position 4 h + j16 / 4 of 16 (+ 8 for the second
        // read), columns 32 j + 16 (g4 % 2) + 4 (j16 % 4) .. + 3, and receives 8 positions of one column in the order of p's registers.
        const int tr_row = 4 * h + ((lane & 15) >> 2), tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            u32x4 part[PARTS];  // each nearest to what the ones before leave
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float p0 = s[i][8 * u + 2 * e], p1 = s[i][8 * u + 2 * e + 1];
#pragma unroll
              for (int n = 0; n < PARTS; ++n) {
                part[n][e] = pack2<PDT>(p0, p1);
                p0 -= unpack_lo<PDT>(part[n][e]), p1 -= unpack_hi<PDT>(part[n][e]);
              }
            }
#pragma unroll
            for (int j = 0; j < DB; ++j) {
              const elem* p0 = Vs + (32 * i + 16 * u + tr_row) * VROW + 32 * j + tr_col;
              const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p0);
              const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p0 + 8 * VROW));
              const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
#pragma unroll
              for (int n = 0; n < PARTS; ++n) acc[j] = mma<PDT>(u32x4{l2[0], l2[1], h2[0], h2[1]}, part[n], acc[j]);
            }
          }
      }
      if (__builtin_expect(some_wild, 0)) {
        const int sees_up_to = min(max(last_seen - j0, -1), KEYS);
#pragma unroll
        for (int j = 0; j < DB; ++j)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const uint32_t reached = (uint32_t)((first_wild[32 * j + 8 * (v >> 2) + 4 * h + (v & 3)] - 1 - sees_up_to) >> 31);
            acc[j][v] = f32_of(bits_of(acc[j][v]) | reached);  // (all ones: a NaN)
          }
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // (what waits for memory comes behind the arithmetic)
    if constexpr (!MIDDLE) {
      if (step + 1 < steps) {
        if constexpr (STAGES == 1) lds_barrier();
        bring(step + 1, std::integral_constant<int, TWO ? 1 - P : 0>());
      }
    }
    note(step + RS + 2, queue[P % QUEUE]);
    queue[P % QUEUE] = look_up(step + RS + 2 + QUEUE);
  };
#pragma unroll 1
  for (int step = 0; step < steps; step += TWO ? 2 : 1) {
    take(step, even_t());
    if (TWO && step + 1 < steps) take(step + 1, std::integral_constant<int, TWO ? 1 : 0>());
  }

  // acc[j][v] = sum of p v of row r32, column 32 j + 8 (v / 4) + 4 h + v % 4, relative to m_run
  l_run += __shfl_xor(l_run, 32);
  int again = r32;
  asm volatile("" : "+v"(again));  // (where the row belongs: found again and not held over the steps)
  if (row0 + again >= rows) return;
  const int to_row = first + row0 + again, to_token = (int)a.by_group.div((uint32_t)to_row), to_head = hk * a.G + (to_row - to_token * a.G);
  if (cut) {
    const int64_t part = chunk_part_row(a, b, hk, to_row, start + to_token, to_head) * a.splits + split;
    if (h == 0) a.part_ml[part] = make_float2(m_run, l_run);
    float* to = a.part_o + part * a.width;
#pragma unroll
    for (int j = 0; j < DB; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<f32x4*>(to + 32 * j + 8 * g + 4 * h) = f32x4{acc[j][4 * g], acc[j][4 * g + 1], acc[j][4 * g + 2], acc[j][4 * g + 3]};
    return;
  }
  const float inv = l_run == 0.0f ? 0.0f : a.c.v_scale / l_run;  // (no position seen: 0)
  uint8_t* out = static_cast<uint8_t*>(a.out) + ((start + to_token) * a.so_n + to_head * a.so_h) * QES;
#pragma unroll
  for (int j = 0; j < DB; ++j)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * j + 8 * g + 4 * h, d = hide(a.c.d);
      const float x0 = acc[j][4 * g] * inv, x1 = acc[j][4 * g + 1] * inv, x2 = acc[j][4 * g + 2] * inv, x3 = acc[j][4 * g + 3] * inv;
      if (col + 3 < d) {
        if constexpr (F32) {
          typedef float any_f32x4 __attribute__((ext_vector_type(4), aligned(4)));
          *reinterpret_cast<any_f32x4*>(out + col * 4) = any_f32x4{x0, x1, x2, x3};
        } else {
          typedef uint32_t any_u32x2 __attribute__((ext_vector_type(2), aligned(2)));
          *reinterpret_cast<any_u32x2*>(out + col * 2) = any_u32x2{pack2<QDT>(x0, x1), pack2<QDT>(x2, x3)};
        }
      } else if (ODD) {
        if (col < d) store_from_f32<QDT>(out, col, x0);
        if (col + 1 < d) store_from_f32<QDT>(out, col + 1, x1);
        if (col + 2 < d) store_from_f32<QDT>(out, col + 2, x2);
      }
    }
}

template <int DB, bool ODD>
int launch(const ChunkArgs& a, hipStream_t s) {
  auto kernel = chunk_attention_kernel<CDT, QDT, DB, ODD>;
  constexpr size_t lds = lds_bytes(DB, ODD);
  if (lds > 65536 && !planning())
    LH_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  LH_LAUNCH(kernel, dim3((unsigned)((int64_t)a.slots * a.c.heads * a.splits)), dim3(256), lds, s, a);
  return check_launch("chunk_attention");
}

}  // namespace

int LH_CHUNK_NAME(const ChunkArgs& a, const ChunkPlan& p, hipStream_t s) {
  if (p.odd) {
    if (p.blocks <= 2) return launch<2, true>(a, s);
    if (p.blocks <= 4) return launch<4, true>(a, s);
    return launch<8, true>(a, s);
  }
  switch (p.blocks) {
    case 2: return launch<2, false>(a, s);
    case 3: return launch<3, false>(a, s);
    case 4: return launch<4, false>(a, s);
    case 6: return launch<6, false>(a, s);
    default: return launch<8, false>(a, s);
  }
}

}  // namespace lh
