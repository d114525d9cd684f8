// Rotary positions, and keys and values into the slots of a paged cache.
//
// Column pairs (a, b) of a head, (i, i + R / 2) or (2 i, 2 i + 1) for i < R / 2, turn by the angle position * freqs[i]:
//   a' = a cos - b sin,  b' = b cos + a sin,
// the other columns stay.  A token's angles are the same for all of its heads: a thread makes the eight it needs and uses them for one
// or two heads, whose loads are on their way meanwhile.  The angle is reduced in 64 bits (a position of 10^6 times a frequency of 1 leaves an
// f32 4 places after the point), the reduced one has a sine and cosine by their Taylor series, in f32.
//
// Both operators read and write every value once and are bound by memory, or by the launch for a step of one token a sequence: 8192 tokens of 40
// heads of 128, f16, 36.6 us (4.6 TB/s); keys, values and queries of 8192 tokens, 24 heads of 64, into a cache of e4m3 12.4 us (3.7 TB/s, with
// the vector instructions of angles and quotients beside it); 64 tokens of 24 or 36 heads of 64, 4.3 and 4.9 us.
#include "elements.h"
#include "paged.h"

namespace lh {

struct RotaryArgs {
  const void* q;          // [N, H, d]
  void* out;              // may be q
  int64_t sq_n, sq_h, so_n, so_h;
  const void* k;          // [N, heads, d] each, into the cache
  const void* v;
  int64_t sk_n, sk_h, sv_n, sv_h;
  void* k_cache;
  void* v_cache;
  lh_strides3 ck, cv;
  const int64_t* slots;
  const int32_t* positions;
  const double* freqs;    // [half], radians a position
  float amplitude;
  float k_scale, v_scale, k_inv, v_inv;
  int32_t H, heads, d, half;  // heads of q (0: none), of the cache (0: nothing is stored), columns, pairs that turn (0: none)
  int64_t all_slots;
  FastDiv by_size, by_chunks, by_groups;
  int32_t turning;        // chunks of a head that turn: 8 pairs each
  int32_t threads;
};

// Cosine and sine of 2 pi x, |x| <= 1/8 (what is left out is below 2^-29).
__device__ __forceinline__ void cos_sin_eighth(float x, float* c, float* s) {
  x *= 6.2831853071795865f;
  const float z = x * x;
  float p = __builtin_fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
  p = __builtin_fmaf(z, p, 1.0f / 120.0f);
  p = __builtin_fmaf(z, p, -1.0f / 6.0f);
  *s = __builtin_fmaf(x * z, p, x);
  float t = __builtin_fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  t = __builtin_fmaf(z, t, -1.0f / 720.0f);
  t = __builtin_fmaf(z, t, 1.0f / 24.0f);
  t = __builtin_fmaf(z, t, -0.5f);
  *c = __builtin_fmaf(z, t, 1.0f);
}
// Of position * freq radians.
__device__ __forceinline__ void cos_sin(int position, double freq, float* c, float* s) {
  const double turns = (double)position * (freq * 0.15915494309189533577);  // 1 / (2 pi)
  const double quarters = 4.0 * (turns - __builtin_rint(turns)), whole = __builtin_rint(quarters);  // -2 .. 2
  float c0, s0;
  cos_sin_eighth((float)((quarters - whole) * 0.25), &c0, &s0);
  const int n = (int)whole & 3;
  const float cq = n & 1 ? s0 : c0, sq = n & 1 ? c0 : s0;
  *c = n == 1 || n == 2 ? -cq : cq;
  *s = n >= 2 ? -sq : sq;
}

// A thread takes one chunk, two pieces of 8 columns, of PER heads of a token (of q, keys and values counted through).  The pieces of what turns, of
// what is behind it, and of a value, each are cut in two halves, and a chunk has one of either, so that neighbours read and write neighbouring
// pieces.
template <int SDT, int CDT, bool INTERLEAVED, int PER>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
  constexpr int SES = elem_bytes<SDT>(), CES = elem_bytes<CDT>();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.threads) return;
  const int groups_of_token = (int)a.by_groups.d, chunks = (int)a.by_chunks.d;
  const int rest = (int)a.by_chunks.div((uint32_t)t), chunk = t - rest * chunks;
  const int n = (int)a.by_groups.div((uint32_t)rest), group = rest - n * groups_of_token;
  const int heads_all = a.H + 2 * a.heads;
  const int position = a.half > 0 ? a.positions[n] : 0;
  int64_t page = -1;
  int slot = 0;
  if (a.heads > 0) {
    const int64_t at = a.slots[n];
    if (at >= 0 && at < a.all_slots) {
      page = at < (1ll << 31) ? (int64_t)a.by_size.div((uint32_t)at) : at / a.by_size.d;
      slot = (int)(at - page * a.by_size.d);
    }
  }
  Piece<SDT> lo[PER], hi[PER];
  int c0[PER], c1[PER], n0[PER], n1[PER];  // the pieces' first columns and how many columns they have
  // What each of the PER heads is, and its loads.
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int head = group + i * groups_of_token;
    const bool stored = head >= a.H, value = head >= a.H + a.heads;
    n0[i] = n1[i] = 0, c0[i] = c1[i] = 0;
    if (head < heads_all && (!stored || page >= 0)) {
      if (value || chunk >= a.turning) {
        const int from = value ? 0 : 2 * a.half, at = value ? chunk : chunk - a.turning, chunks_here = (a.d - from + 15) >> 4;
        c0[i] = from + 8 * at, c1[i] = c0[i] + 8 * chunks_here;
        n0[i] = at < chunks_here ? min(a.d - c0[i], 8) : 0, n1[i] = at < chunks_here ? min(max(a.d - c1[i], 0), 8) : 0;
      } else if (INTERLEAVED) {
        c0[i] = 8 * chunk, c1[i] = 8 * (chunk + a.turning);
        n0[i] = min(2 * a.half - c0[i], 8), n1[i] = min(max(2 * a.half - c1[i], 0), 8);
      } else {
        c0[i] = 8 * chunk, c1[i] = a.half + 8 * chunk;
        n0[i] = n1[i] = min(a.half - 8 * chunk, 8);
      }
      const uint8_t* row = value    ? static_cast<const uint8_t*>(a.v) + (n * a.sv_n + (head - a.H - a.heads) * a.sv_h) * SES
                           : stored ? static_cast<const uint8_t*>(a.k) + (n * a.sk_n + (head - a.H) * a.sk_h) * SES
                                    : static_cast<const uint8_t*>(a.q) + (n * a.sq_n + head * a.sq_h) * SES;
      if (n0[i] > 0) lo[i] = load_piece<SDT>(row + (int64_t)c0[i] * SES, n0[i]);
      if (n1[i] > 0) hi[i] = load_piece<SDT>(row + (int64_t)c1[i] * SES, n1[i]);
    }
  }
  float c[8], s[8];
  if (chunk < a.turning) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int pair = INTERLEAVED ? 4 * (e < 4 ? chunk : chunk + a.turning) + e % 4 : 8 * chunk + e;
      cos_sin(position, a.freqs[min(pair, a.half - 1)], &c[e], &s[e]);
      c[e] *= a.amplitude, s[e] *= a.amplitude;
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (n0[i] <= 0) continue;
    const int head = group + i * groups_of_token;
    const bool stored = head >= a.H, value = head >= a.H + a.heads, turns = !value && chunk < a.turning;
    float x[8], y[8];
    piece_to_f32<SDT>(lo[i], x);
    if (n1[i] > 0) {
      piece_to_f32<SDT>(hi[i], y);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = 0.0f;
    }
    if (turns) {
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float xa = x[2 * e], xb = x[2 * e + 1], ya = y[2 * e], yb = y[2 * e + 1];
          x[2 * e] = __builtin_fmaf(xa, c[e], -(xb * s[e])), x[2 * e + 1] = __builtin_fmaf(xb, c[e], xa * s[e]);
          y[2 * e] = __builtin_fmaf(ya, c[4 + e], -(yb * s[4 + e])), y[2 * e + 1] = __builtin_fmaf(yb, c[4 + e], ya * s[4 + e]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float xa = x[e], xb = y[e];
          x[e] = __builtin_fmaf(xa, c[e], -(xb * s[e])), y[e] = __builtin_fmaf(xb, c[e], xa * s[e]);
        }
      }
    }
    if (!stored) {
      uint8_t* to = static_cast<uint8_t*>(a.out) + (n * a.so_n + head * a.so_h) * SES;
      const Piece<SDT> first = turns ? piece_of_f32<SDT>(x) : lo[i], second = turns ? piece_of_f32<SDT>(y) : hi[i];
      store_piece<SDT>(to + (int64_t)c0[i] * SES, first, n0[i]);
      if (n1[i] > 0) store_piece<SDT>(to + (int64_t)c1[i] * SES, second, n1[i]);
    } else {
      const lh_strides3 cs = value ? a.cv : a.ck;
      uint8_t* to = static_cast<uint8_t*>(value ? a.v_cache : a.k_cache) + (page * cs.z + (head - a.H - (value ? a.heads : 0)) * cs.h + slot * cs.t) * CES;
      Piece<CDT> first, second;
      if constexpr (CDT == LH_F8E4M3) {
        const float scale = value ? a.v_scale : a.k_scale, inv = value ? a.v_inv : a.k_inv;
        e4m3_quotients(x, scale, inv);
        e4m3_quotients(y, scale, inv);
        first = piece_of_f32<CDT>(x), second = piece_of_f32<CDT>(y);
      } else {
        first = turns ? piece_of_f32<CDT>(x) : __builtin_bit_cast(Piece<CDT>, lo[i]);
        second = turns ? piece_of_f32<CDT>(y) : __builtin_bit_cast(Piece<CDT>, hi[i]);
      }
      store_piece<CDT>(to + (int64_t)c0[i] * CES, first, n0[i]);
      if (n1[i] > 0) store_piece<CDT>(to + (int64_t)c1[i] * CES, second, n1[i]);
    }
  }
}

template <int SDT, int CDT, bool INTERLEAVED>
static int launch_rotary(RotaryArgs& a, int64_t N, int heads_all, int chunks, hipStream_t s) {
  // Two heads a thread, which share their angles, where one head a thread would fill half of the chip: prompts of 8192 tokens, 24 heads of 64,
  // into e4m3 13.9 us (one head 16.4, four 13.7); 64 tokens of 24 heads 4.4 us (one head 3.8).  (Stores past the
  // caches cost their reader more than they save: 8192 tokens of 40 heads of 128, f16, into one buffer that is read after, 92.5 us; 81.1 kept.)
  const int64_t values = N * heads_all * chunks, at_once = (int64_t)num_cus() * 2048;
  const int per = 2 * values >= at_once ? 2 : 1;
  const int groups = (heads_all + per - 1) / per;
  const int64_t threads = N * groups * chunks;
  LH_REQUIRE(threads < (1ll << 31) - 256, "rotary positions: too many values");
  a.by_groups = FastDiv((uint32_t)groups), a.threads = (int32_t)threads;
  const dim3 grid((unsigned)((threads + 255) / 256)), block(256);
  if (per == 2) LH_LAUNCH((rotary_kernel<SDT, CDT, INTERLEAVED, 2>), grid, block, 0, s, a);
  else LH_LAUNCH((rotary_kernel<SDT, CDT, INTERLEAVED, 1>), grid, block, 0, s, a);
  return check_launch("rotary");
}

template <int SDT>
static int launch_rotary_to(RotaryArgs& a, int64_t N, int cache_dtype, bool interleaved, hipStream_t s) {
  a.turning = (a.half + 7) / 8;
  int chunks = a.turning + (a.d - 2 * a.half + 15) / 16;
  if (a.heads > 0 && chunks < (a.d + 15) / 16) chunks = (a.d + 15) / 16;
  a.by_chunks = FastDiv((uint32_t)chunks);
  const int heads_all = a.H + 2 * a.heads;
  if (cache_dtype == LH_F8E4M3)
    return interleaved ? launch_rotary<SDT, LH_F8E4M3, true>(a, N, heads_all, chunks, s) : launch_rotary<SDT, LH_F8E4M3, false>(a, N, heads_all, chunks, s);
  return interleaved ? launch_rotary<SDT, SDT, true>(a, N, heads_all, chunks, s) : launch_rotary<SDT, SDT, false>(a, N, heads_all, chunks, s);
}

static int launch_rotary_from(RotaryArgs& a, int64_t N, int dtype, int cache_dtype, bool interleaved, hipStream_t s) {
  if (dtype == LH_BF16) return launch_rotary_to<LH_BF16>(a, N, cache_dtype, interleaved, s);
  if (dtype == LH_F16) return launch_rotary_to<LH_F16>(a, N, cache_dtype, interleaved, s);
  return launch_rotary_to<LH_F32>(a, N, cache_dtype, interleaved, s);
}

static int rotary_turn(RotaryArgs* a, const char* what, const lh_rotary* r, int64_t d) {
  LH_REQUIRE(r->positions && r->freqs, "%s: null pointer", what);
  LH_REQUIRE(r->turned >= 2 && r->turned % 2 == 0 && r->turned <= d, "%s: %d of %lld columns cannot turn (an even number)", what, r->turned, (long long)d);
  a->positions = r->positions, a->freqs = r->freqs, a->half = r->turned / 2, a->amplitude = r->amplitude;
  return LH_OK;
}

}  // namespace lh

using namespace lh;

extern "C" {

int lh_hip_rotary(void* out, const void* x, int64_t out_stride_n, int64_t out_stride_h, int64_t x_stride_n, int64_t x_stride_h, const lh_rotary* turn,
                  int64_t N, int64_t H, int64_t d, int32_t dtype, void* stream) {
  const char* what = "lh_hip_rotary";
  RotaryArgs a = {};
  LH_REQUIRE(N >= 0 && N < (1ll << 31) && H >= 0 && H < (1ll << 20) && d >= 1 && d < (1ll << 20), "%s: bad sizes", what);
  LH_REQUIRE(dtype == LH_F32 || dtype == LH_BF16 || dtype == LH_F16, "%s: unsupported dtype %d", what, dtype);
  LH_REQUIRE(turn != nullptr, "%s: null pointer", what);
  if (N == 0 || H == 0) return LH_OK;
  LH_REQUIRE(out && x, "%s: null pointer", what);
  if (const int rc = rotary_turn(&a, what, turn, d)) return rc;
  a.q = x, a.out = out, a.sq_n = x_stride_n, a.sq_h = x_stride_h, a.so_n = out_stride_n, a.so_h = out_stride_h;
  a.H = (int32_t)H, a.d = (int32_t)d;
  return launch_rotary_from(a, N, dtype, dtype, turn->interleaved != 0, reinterpret_cast<hipStream_t>(stream));
}

int lh_hip_kv_store(const lh_paged_cache* cache, const void* k, const void* v, int64_t k_stride_n, int64_t k_stride_h, int64_t v_stride_n,
                    int64_t v_stride_h, const int64_t* slots, void* q_out, const void* q, int64_t out_stride_n, int64_t out_stride_h,
                    int64_t q_stride_n, int64_t q_stride_h, const lh_rotary* turn, int64_t N, int64_t H, int32_t dtype, void* stream) {
  const char* what = "lh_hip_kv_store";
  Paged c;
  if (const int rc = paged_cache(cache, what, &c, false)) return rc;
  RotaryArgs a = {};
  LH_REQUIRE(N >= 0 && N < (1ll << 31) && H >= 0 && H < (1ll << 20), "%s: bad sizes", what);
  LH_REQUIRE(dtype == cache->dtype || (cache->dtype == LH_F8E4M3 && (dtype == LH_F32 || dtype == LH_BF16 || dtype == LH_F16)),
             "%s: keys and values must have the cache's dtype (f32, bf16 or f16 for a cache of e4m3)", what);
  LH_REQUIRE(H == 0 || turn != nullptr, "%s: queries are passed to be turned", what);
  if (N == 0) return LH_OK;
  LH_REQUIRE(k && v && slots && (H == 0 || (q && q_out)), "%s: null pointer", what);
  if (turn)
    if (const int rc = rotary_turn(&a, what, turn, c.d)) return rc;
  a.q = q, a.out = q_out, a.sq_n = q_stride_n, a.sq_h = q_stride_h, a.so_n = out_stride_n, a.so_h = out_stride_h;
  a.k = k, a.v = v, a.sk_n = k_stride_n, a.sk_h = k_stride_h, a.sv_n = v_stride_n, a.sv_h = v_stride_h;
  a.k_cache = c.k, a.v_cache = c.v, a.ck = c.sk, a.cv = c.sv, a.slots = slots;
  a.k_scale = c.k_scale, a.v_scale = c.v_scale, a.k_inv = e4m3_inverse(c.k_scale), a.v_inv = e4m3_inverse(c.v_scale);
  a.H = (int32_t)H, a.heads = c.heads, a.d = c.d, a.all_slots = (int64_t)c.pages * c.size, a.by_size = c.by_size;
  return launch_rotary_from(a, N, dtype, cache->dtype, turn && turn->interleaved != 0, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
