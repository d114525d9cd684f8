// Root-mean-square norm, with a residual's addition before it and a result of 8 bits behind it:
//   s = x + residual,  y = s / sqrt(mean(s^2) + eps) * gamma,  out = y, or e4m3(y / scale).
// Memory bounds it: x, the residual and its sum, and the result once each.  A row stays in the registers of a wave (up to 1024
// columns) or of a workgroup (up to 16384) between its sums, so that nothing is read twice; longer rows are read again, from the caches.
// 8192 rows of 8192, bf16 with a residual, into e4m3 with a scale a row: 90.7 us (5.2 TB/s, what a copy reaches); 64 rows of 768: 4.5 us, a launch and
// one round trip to memory.
#include <algorithm>

#include "elements.h"

namespace lh {

struct RmsArgs {
  void* out;
  const void* x;
  const void* residual;
  void* sum;             // what becomes of the residual
  const float* gamma;
  float* scales;         // one per row that the kernel finds, or null
  int64_t ld_out, ld_x, ld_residual, ld_sum;
  int32_t M, C;
  float eps, scale, scale_inv;  // scale: of all rows, for a result of 8 bits
  int32_t out_dtype;
  int32_t stream;        // the sum is not kept in the caches
};

enum RmsResidual { kNoResidual, kSameResidual, kF32Residual };

__device__ __forceinline__ float rms_wave_sum(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ uint32_t rms_wave_max(uint32_t v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  return v;
}

// Over the row's waves, in a fixed order; `shared` has an entry per wave.
template <int WAVES>
__device__ __forceinline__ float rms_row_sum(float v, float* shared) {
  v = rms_wave_sum(v);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += shared[w];
  }
  return v;
}
template <int WAVES>
__device__ __forceinline__ uint32_t rms_row_max(uint32_t v, uint32_t* shared) {
  v = rms_wave_max(v);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v = max(v, shared[w]);
  }
  return v;
}

// s = x + residual of a piece; the sum is written.
template <int XDT, int RES>
__device__ __forceinline__ void rms_add(const RmsArgs& a, const Piece<XDT>& px, const Piece<RES == kF32Residual ? LH_F32 : XDT>& pr, int64_t row, int col,
                                        int n, bool write, float* s) {
  constexpr int RDT = RES == kF32Residual ? LH_F32 : XDT;
  piece_to_f32<XDT>(px, s);
  if constexpr (RES != kNoResidual) {
    float r[kPiece];
    piece_to_f32<RDT>(pr, r);
#pragma unroll
    for (int e = 0; e < kPiece; ++e) s[e] += r[e];
    if (!write) return;
    uint8_t* const to = static_cast<uint8_t*>(a.sum) + (row * a.ld_sum + col) * elem_bytes<RDT>();
    if (a.stream) store_piece<RDT, true>(to, piece_of_f32<RDT>(s), n);
    else store_piece<RDT>(to, piece_of_f32<RDT>(s), n);
  }
}

__device__ __forceinline__ float rms_square(const float* s) {
  float q = 0.0f;
#pragma unroll
  for (int e = 0; e < kPiece; ++e) q = __builtin_fmaf(s[e], s[e], q);
  return q;
}

__device__ __forceinline__ void rms_scale(float* s, float inv, const Piece<LH_F32>& gamma) {
  float g[kPiece];
  piece_to_f32<LH_F32>(gamma, g);
#pragma unroll
  for (int e = 0; e < kPiece; ++e) s[e] = s[e] * inv * g[e];
}

__device__ __forceinline__ uint32_t rms_largest(const float* y, uint32_t m) {  // (as numbers; a NaN is above all)
#pragma unroll
  for (int e = 0; e < kPiece; ++e) m = max(m, __builtin_bit_cast(uint32_t, y[e]) & 0x7fffffffu);
  return m;
}

__device__ __forceinline__ void rms_store(const RmsArgs& a, int64_t row, int col, int n, float* y, float scale, float inv) {
  uint8_t* out = static_cast<uint8_t*>(a.out);
  const int64_t at = row * a.ld_out + col;
  switch (a.out_dtype) {
    case LH_F8E4M3:
      e4m3_quotients(y, scale, inv);
      store_piece<LH_F8E4M3>(out + at, piece_of_f32<LH_F8E4M3>(y), n);
      break;
    case LH_BF16: store_piece<LH_BF16>(out + 2 * at, piece_of_f32<LH_BF16>(y), n); break;
    case LH_F16: store_piece<LH_F16>(out + 2 * at, piece_of_f32<LH_F16>(y), n); break;
    default: store_piece<LH_F32>(out + 4 * at, piece_of_f32<LH_F32>(y), n); break;
  }
}

// The scale of a row whose largest |y| has the bits m: 448 stands for it; 1 for a row of zeros.  No less than the smallest number, which a
// quotient below half of it would make a 0, and zeros of the row 0 / 0.
__device__ __forceinline__ float rms_row_scale(uint32_t m) {
  const float scale = __builtin_bit_cast(float, m) / 448.0f;
  return m == 0 ? 1.0f : scale == 0.0f ? 0x1p-149f : scale;
}

// WAVES of a row, VPT pieces a thread; a workgroup of one-wave rows has four.
template <int XDT, int RES, int WAVES, int VPT>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) rms_norm_kernel(RmsArgs a) {
  constexpr int RDT = RES == kF32Residual ? LH_F32 : XDT, THREADS = WAVES * 64;
  __shared__ float sums[WAVES];
  __shared__ uint32_t largest[WAVES];
  const int64_t row = WAVES == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= a.M) return;  // (whole rows: no barrier is left out)
  const int tid = threadIdx.x % THREADS;
  const uint8_t* x = static_cast<const uint8_t*>(a.x) + row * a.ld_x * elem_bytes<XDT>();
  const uint8_t* r = static_cast<const uint8_t*>(a.residual) + row * a.ld_residual * elem_bytes<RDT>();
  Piece<XDT> px[VPT];
  Piece<RDT> pr[VPT];
  Piece<LH_F32> pg[VPT];
  float s[VPT][kPiece];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int col = (i * THREADS + tid) * kPiece, n = a.C - col;
    if (n > 0) {
      px[i] = load_piece<XDT>(x + (int64_t)col * elem_bytes<XDT>(), n);
      if constexpr (RES != kNoResidual) pr[i] = load_piece<RDT>(r + (int64_t)col * elem_bytes<RDT>(), n);
    }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int col = (i * THREADS + tid) * kPiece, n = a.C - col;
    if (n > 0) pg[i] = load_piece<LH_F32>(a.gamma + col, n);
  }
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int col = (i * THREADS + tid) * kPiece, n = a.C - col;
    if (n > 0) {
      rms_add<XDT, RES>(a, px[i], pr[i], row, col, n, true, s[i]);
      q += rms_square(s[i]);
    }
  }
  const float inv = 1.0f / sqrtf(rms_row_sum<WAVES>(q, sums) / (float)a.C + a.eps);
  float scale = a.scale, scale_inv = a.scale_inv;
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if ((i * THREADS + tid) * kPiece < a.C) {
      rms_scale(s[i], inv, pg[i]);
      if (a.scales != nullptr) m = rms_largest(s[i], m);
    }
  if (a.scales != nullptr) {
    scale = rms_row_scale(rms_row_max<WAVES>(m, largest));
    scale_inv = e4m3_inverse(scale);
    if (tid == 0) a.scales[row] = scale;
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int col = (i * THREADS + tid) * kPiece, n = a.C - col;
    if (n > 0) rms_store(a, row, col, n, s[i], scale, scale_inv);
  }
}

// Rows that no workgroup's registers hold: passes over x and the residual (whose sum is written in the last, so that it may take the
// residual's place).
template <int XDT, int RES>
__global__ void __launch_bounds__(1024) rms_norm_long(RmsArgs a) {
  constexpr int RDT = RES == kF32Residual ? LH_F32 : XDT, WAVES = 16;
  __shared__ float sums[WAVES];
  __shared__ uint32_t largest[WAVES];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const uint8_t* x = static_cast<const uint8_t*>(a.x) + row * a.ld_x * elem_bytes<XDT>();
  const uint8_t* r = static_cast<const uint8_t*>(a.residual) + row * a.ld_residual * elem_bytes<RDT>();
  auto piece = [&](int col, bool write, float* s) {
    const int n = a.C - col;
    const Piece<XDT> px = load_piece<XDT>(x + (int64_t)col * elem_bytes<XDT>(), n);
    Piece<RDT> pr = {};
    if constexpr (RES != kNoResidual) pr = load_piece<RDT>(r + (int64_t)col * elem_bytes<RDT>(), n);
    rms_add<XDT, RES>(a, px, pr, row, col, n, write, s);
  };
  float q = 0.0f, s[kPiece];
  for (int col = tid * kPiece; col < a.C; col += 1024 * kPiece) {
    piece(col, false, s);
    q += rms_square(s);
  }
  const float inv = 1.0f / sqrtf(rms_row_sum<WAVES>(q, sums) / (float)a.C + a.eps);
  float scale = a.scale, scale_inv = a.scale_inv;
  if (a.scales != nullptr) {
    uint32_t m = 0;
    for (int col = tid * kPiece; col < a.C; col += 1024 * kPiece) {
      piece(col, false, s);
      rms_scale(s, inv, load_piece<LH_F32>(a.gamma + col, a.C - col));
      m = rms_largest(s, m);
    }
    scale = rms_row_scale(rms_row_max<WAVES>(m, largest));
    scale_inv = e4m3_inverse(scale);
    if (tid == 0) a.scales[row] = scale;
  }
  for (int col = tid * kPiece; col < a.C; col += 1024 * kPiece) {
    piece(col, true, s);
    rms_scale(s, inv, load_piece<LH_F32>(a.gamma + col, a.C - col));
    rms_store(a, row, col, a.C - col, s, scale, scale_inv);
  }
}

template <int XDT, int RES>
static int launch_rms_rows(const RmsArgs& a, hipStream_t s) {
  const int pieces = (a.C + kPiece - 1) / kPiece;
  const dim3 four((unsigned)((a.M + 3) / 4)), one((unsigned)a.M);
  if (pieces <= 64) LH_LAUNCH((rms_norm_kernel<XDT, RES, 1, 1>), four, dim3(256), 0, s, a);
  else if (pieces <= 128) LH_LAUNCH((rms_norm_kernel<XDT, RES, 1, 2>), four, dim3(256), 0, s, a);
  else if (pieces <= 256) LH_LAUNCH((rms_norm_kernel<XDT, RES, 4, 1>), one, dim3(256), 0, s, a);
  else if (pieces <= 512) LH_LAUNCH((rms_norm_kernel<XDT, RES, 4, 2>), one, dim3(256), 0, s, a);
  else if (pieces <= 1024) LH_LAUNCH((rms_norm_kernel<XDT, RES, 4, 4>), one, dim3(256), 0, s, a);
  else if (pieces <= 2048) LH_LAUNCH((rms_norm_kernel<XDT, RES, 16, 2>), one, dim3(1024), 0, s, a);
  else LH_LAUNCH((rms_norm_long<XDT, RES>), one, dim3(1024), 0, s, a);
  return check_launch("rms_norm");
}

// A launch has fewer than 2^32 threads, which is 2^26 rows of a wave each, 2^24 of four: more rows are more launches.
template <int XDT, int RES>
static int launch_rms(const RmsArgs& all, hipStream_t s) {
  constexpr int RDT = RES == kF32Residual ? LH_F32 : XDT;
  const int64_t most = (1ll << 32) / (all.C <= 128 * kPiece ? 64 : all.C <= 1024 * kPiece ? 256 : 1024) - 4;
  for (int64_t row = 0; row < all.M; row += most) {
    RmsArgs a = all;
    a.M = (int32_t)std::min<int64_t>(all.M - row, most);
    a.x = static_cast<const uint8_t*>(all.x) + row * all.ld_x * elem_bytes<XDT>();
    a.out = static_cast<uint8_t*>(all.out) + row * all.ld_out * (int64_t)dtype_size(all.out_dtype);
    if (RES != kNoResidual) {
      a.residual = static_cast<const uint8_t*>(all.residual) + row * all.ld_residual * elem_bytes<RDT>();
      a.sum = static_cast<uint8_t*>(all.sum) + row * all.ld_sum * elem_bytes<RDT>();
    }
    if (all.scales != nullptr) a.scales = all.scales + row;
    if (const int rc = launch_rms_rows<XDT, RES>(a, s)) return rc;
  }
  return LH_OK;
}

template <int XDT>
static int launch_rms_residual(const RmsArgs& a, int residual_dtype, hipStream_t s) {
  if (a.residual == nullptr) return launch_rms<XDT, kNoResidual>(a, s);
  if (residual_dtype == XDT) return launch_rms<XDT, kSameResidual>(a, s);
  return launch_rms<XDT, kF32Residual>(a, s);
}

}  // namespace lh

using namespace lh;

extern "C" int lh_hip_rms_norm(void* out, const void* x, const float* gamma, const void* residual, void* residual_out, float* row_scales, float scale,
                               int64_t M, int64_t C, int64_t ld_out, int64_t ld_x, int64_t ld_residual, int64_t ld_residual_out, float eps,
                               int32_t x_dtype, int32_t residual_dtype, int32_t out_dtype, void* stream) {
  const char* what = "lh_hip_rms_norm";
  LH_REQUIRE(M >= 0 && M < (1ll << 31) && C >= 1 && C < (1ll << 30), "%s: bad sizes (%lld rows of %lld)", what, (long long)M, (long long)C);
  LH_REQUIRE(x_dtype == LH_F32 || x_dtype == LH_BF16 || x_dtype == LH_F16, "%s: unsupported x dtype %d", what, x_dtype);
  LH_REQUIRE(out_dtype == LH_F32 || out_dtype == LH_BF16 || out_dtype == LH_F16 || out_dtype == LH_F8E4M3, "%s: unsupported out dtype %d", what, out_dtype);
  LH_REQUIRE(residual == nullptr || residual_dtype == x_dtype || residual_dtype == LH_F32, "%s: the residual must be f32 or have the dtype of x", what);
  LH_REQUIRE((residual == nullptr) == (residual_out == nullptr), "%s: a residual needs a place for its sum", what);
  LH_REQUIRE(out_dtype == LH_F8E4M3 ? row_scales != nullptr || (scale > 0.0f && scale < INFINITY) : row_scales == nullptr,
             "%s: a result of e4m3 needs a positive scale or room for one per row, others take none", what);
  LH_REQUIRE(M <= 1 || (ld_out >= C && (residual == nullptr || ld_residual_out >= C)), "%s: rows of a result overlap", what);
  if (M == 0) return LH_OK;
  LH_REQUIRE(out && x && gamma, "%s: null pointer", what);
  // A sum that the L2 caches (32 MiB) do not hold goes past them: who reads it next comes after the product that reads the result.  (8192 rows of
  // 8192, bf16 with a result of e4m3: 98.5 us kept, 90.6 streamed; from 97.0 to 100.7 us where other buffers are in turn; 4096 columns, f32
  // residuals and smaller sums: within 1% of each other.)
  const bool streaming = residual != nullptr && M * C * (int64_t)dtype_size(residual_dtype) >= 32ll << 20;
  const RmsArgs a = {out, x, residual, residual_out, gamma, row_scales, ld_out, ld_x, ld_residual, ld_residual_out, (int32_t)M, (int32_t)C,
                     eps, scale, e4m3_inverse(scale), out_dtype, streaming};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (x_dtype == LH_BF16) return launch_rms_residual<LH_BF16>(a, residual_dtype, s);
  if (x_dtype == LH_F16) return launch_rms_residual<LH_F16>(a, residual_dtype, s);
  return launch_rms_residual<LH_F32>(a, LH_F32, s);
}
