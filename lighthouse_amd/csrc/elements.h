// Rows of elements in pieces of eight, as the kernels that turn, store and normalise rows read and write them: any strides and
// alignment (gfx9 global memory takes 16 bytes at the alignment of an element), the end of a row that is no whole piece by element.
#pragma once

#include "common.h"

namespace lh {

constexpr int kPiece = 8;  // elements

template <int DT>
constexpr int elem_bytes() { return DT == LH_F32 ? 4 : DT == LH_F8E4M3 ? 1 : 2; }

// Eight elements as they lie in memory.
template <int DT>
struct Piece { uint32_t w[kPiece * elem_bytes<DT>() / 4]; };

// The first n (1 to 8) elements from p on; the others are 0.
template <int DT>
__device__ __forceinline__ Piece<DT> load_piece(const void* p, int n) {
  constexpr int ES = elem_bytes<DT>();
  Piece<DT> r;
  if (n >= kPiece) {
#pragma unroll
    for (int l = 0; l < kPiece * ES / 16; ++l) {
      const typename Chunk<ES>::type w = reinterpret_cast<const typename Chunk<ES>::type*>(p)[l];
#pragma unroll
      for (int e = 0; e < 4; ++e) r.w[4 * l + e] = w[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPiece * ES / 4; ++i) r.w[i] = 0;
#pragma unroll
    for (int e = 0; e < kPiece; ++e)
      if (e < n) {
        if constexpr (ES == 4) r.w[e] = reinterpret_cast<const uint32_t*>(p)[e];
        else r.w[e / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(p)[e] << (16 * (e % 2));
      }
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void piece_to_f32(const Piece<DT>& p, float* x) {
#pragma unroll
  for (int e = 0; e < kPiece; ++e) {
    if constexpr (DT == LH_F32) x[e] = __builtin_bit_cast(float, p.w[e]);
    else x[e] = e % 2 ? unpack_hi<DT>(p.w[e / 2]) : unpack_lo<DT>(p.w[e / 2]);
  }
}

// Two floats, no larger than 448, -> two e4m3 codes in the low half of a word, rounded to nearest even; a NaN stays one.
__device__ __forceinline__ uint32_t e4m3_codes(float a, float b) { return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu; }

template <int DT>
__device__ __forceinline__ Piece<DT> piece_of_f32(const float* x) {
  Piece<DT> p;
  if constexpr (DT == LH_F32) {
#pragma unroll
    for (int e = 0; e < kPiece; ++e) p.w[e] = __builtin_bit_cast(uint32_t, x[e]);
  } else if constexpr (DT == LH_F8E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) p.w[i] = e4m3_codes(x[4 * i], x[4 * i + 1]) | e4m3_codes(x[4 * i + 2], x[4 * i + 3]) << 16;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p.w[i] = pack2<DT>(x[2 * i], x[2 * i + 1]);
  }
  return p;
}

// The first n (1 to 8) elements to p.
// STREAM: whole pieces are not kept in the caches.
template <int DT, bool STREAM = false>
__device__ __forceinline__ void store_piece(void* p, const Piece<DT>& v, int n) {
  constexpr int ES = elem_bytes<DT>();
  typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
  if (n >= kPiece) {
    if constexpr (ES == 1) {
      *reinterpret_cast<u32x2_any*>(p) = u32x2_any{v.w[0], v.w[1]};
    } else {
#pragma unroll
      for (int l = 0; l < kPiece * ES / 16; ++l) {
        const typename Chunk<ES>::type w = {v.w[4 * l], v.w[4 * l + 1], v.w[4 * l + 2], v.w[4 * l + 3]};
        if constexpr (STREAM) __builtin_nontemporal_store(w, reinterpret_cast<typename Chunk<ES>::type*>(p) + l);
        else reinterpret_cast<typename Chunk<ES>::type*>(p)[l] = w;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < kPiece; ++e)
      if (e < n) {
        if constexpr (ES == 4) reinterpret_cast<uint32_t*>(p)[e] = v.w[e];
        else if constexpr (ES == 2) reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(v.w[e / 2] >> (16 * (e % 2)));
        else reinterpret_cast<uint8_t*>(p)[e] = (uint8_t)(v.w[e / 4] >> (8 * (e % 4)));
      }
  }
}

// What e4m3_quotients takes for 1 / scale: 0 where the short division below does not apply.
__host__ __device__ inline float e4m3_inverse(float scale) { return scale >= 0x1p-60f && scale <= 0x1p60f ? 1.0f / scale : 0.0f; }

// (Comparisons keep a NaN, fmin and fmax would not.)
__device__ __forceinline__ float e4m3_clamp(float x) {
  x = x > 448.0f ? 448.0f : x;
  return x < -448.0f ? -448.0f : x;
}

// Eight numbers x -> x / scale, clamped to +-448 (a NaN stays one): the quotient that a division rounds, so that the codes are those
// of the formula and not of a rounded reciprocal.  With inv = 1 / scale rounded, q = x inv and r = q scale - x (exact), q - r inv is
// that quotient (Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor", 1990), but where x or r leaves the
// normal range: for scales between 2^-60 and 2^60 such quotients, if not 0 in e4m3, are far from it.  Numbers that are not finite
// or far above 448 take the division.  (3 instructions instead of 11: 8 prompts of 1024 tokens, 12 heads of 64, appended in 11.4 us instead of
// 15.9.)
__device__ __forceinline__ void e4m3_quotients(float* x, float scale, float inv) {
  float size = 0.0f;
#pragma unroll
  for (int e = 0; e < kPiece; ++e) size += fabsf(x[e]);
  if (inv != 0.0f && size <= 4096.0f * scale) {
#pragma unroll
    for (int e = 0; e < kPiece; ++e) {
      const float q = x[e] * inv, r = __builtin_fmaf(q, scale, -x[e]);
      x[e] = __builtin_amdgcn_fmed3f(__builtin_fmaf(-r, inv, q), -448.0f, 448.0f);
    }
  } else {
#pragma unroll 1
    for (int e = 0; e < kPiece; ++e) x[e] = e4m3_clamp(x[e] / scale);
  }
}

}  // namespace lh
