// Operands of the block-scaled e4m3 Linear (gemm_fp8_block.hip) and the pre-norm in front of it:
//   quant_fp8_group128   activations: one scale per row and 128 columns
//   quant_fp8_block128   weights: one scale per block of 128 rows x 128 columns
//   add_rmsnorm          x += y;  out = x * rsqrt(mean(x^2) + eps) * w  as bf16, as e4m3 / int8 rows with one scale per
//                        row, or as e4m3 rows with one scale per 128 columns
// A scale is max(max|group|, 1e-12) / 448 and an element e4m3(v * (1 / scale)), the rule of the row-wise quantiser in
// step_ew.hip (a row of 128 columns gets the same bytes and scale from both).  The maximum skips NaN (fmaxf) and the NaN
// element becomes the NaN code; an infinite element makes its group's scale infinite and its own code NaN.  int8 rows have a
// NaN scale instead.  This file
// is built with IEEE division and without contraction, so scales and reciprocals are the correctly rounded quotients.
//
// Scales per 128 columns are stored group after group (element (r, g) at scale[g * ld_scale + r]): the GEMM reads the
// scales of consecutive rows of one group.
#include "quant_common.h"

namespace {

constexpr float E4M3_MAX = 448.0f;
constexpr float AMAX_FLOOR = 1e-12f;

// Non-temporal accesses (BIG) for calls whose tensors are together more than twice the 256 MB memory-side cache, so that
// nothing of them would be found there again: group quantiser at [75600, 13824] 535 us against 641 without, norm of
// [75600, 5120] to e4m3 groups 466 against 511 (kernels on a card that ran 501 and 461 at other times).  Below, the producer's result is still there and the consumer finds this
// one's: norm of [32760, 1536] to e4m3 rows 53 us against 66 with them.
constexpr int64_t STREAMED_BYTES = 512 << 20;
constexpr int MAX_DIM = 0x7fffffff - 511;  // columns are counted in 32 bits, in steps of at most 512
constexpr int64_t MAX_BLOCKS = 1 << 24;  // of 256 threads: a dimension of a launch has less than 2^32 threads

template <bool BIG, class V>
LX2V_DEVICE V ld(const V* p) {
  return BIG ? __builtin_nontemporal_load(p) : *p;
}
template <bool BIG, class V>
LX2V_DEVICE void st(V* p, const V& v) {
  if (BIG) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <bool BIG>
LX2V_DEVICE void load8_once(const uint16_t* p, float (&f)[8]) {
  unpack8(ld<BIG>(reinterpret_cast<const u32x4*>(p)), f);
}
template <bool BIG>
LX2V_DEVICE void load8_once(const float* p, float (&f)[8]) {  // (fp32 rows keep ordinary loads: 3 % faster in the norm of [75600, 5120])
  load8(p, f);
}

// All-reduce maximum over the 16 lanes of a DPP row = the 128 columns of one group (8 per lane).
LX2V_DEVICE float max16(float v) {
#define LX2V_ROR_MAX(n) v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + (n), 0xf, 0xf, true)))
  LX2V_ROR_MAX(8);
  LX2V_ROR_MAX(4);
  LX2V_ROR_MAX(2);
  LX2V_ROR_MAX(1);
#undef LX2V_ROR_MAX
  return v;
}
LX2V_DEVICE float max64(float v) {
  v = max16(v);
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
LX2V_DEVICE float absmax8(const float (&f)[8]) {
  float m = fabsf(f[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, fabsf(f[i]));
  return m;
}
// The same where nothing may hide a NaN: infinite if any of the eight is infinite or NaN (magnitudes order as their bit patterns do, NaN last).
LX2V_DEVICE float absmax8_or_inf(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
  return __uint_as_float(min(m, 0x7f800000u));
}
LX2V_DEVICE float scale_e4m3(float amax) { return __fdiv_rn(fmaxf(amax, AMAX_FLOOR), E4M3_MAX); }
LX2V_DEVICE u32x2 cvt8_e4m3(const float (&f)[8], float inv) {
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * inv, f[1] * inv, 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * inv, f[3] * inv, lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * inv, f[5] * inv, 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] * inv, f[7] * inv, hi, true);
  return u32x2{(uint32_t)lo, (uint32_t)hi};
}

// ---- activations: 1 x 128 groups ------------------------------------------------------------------
// A wave owns 8 rows x 512 columns (four groups): 8 independent 16-byte loads per lane in flight, the maximum of a group by four
// DPP rotations, and after the 8 rows 8 of the 16 lanes of a group hold one row's scale each, so the transposed scales leave as
// 32-byte runs.  One read and one write of the data: 3 bytes an element, 6.2 TB/s at [75600, 13824] (16 rows a wave: 4.9, half as
// many waves fit; 4 rows: 5.7).
constexpr int QR = 8;
template <class T, bool BIG>
__global__ __launch_bounds__(256) void quant_fp8_group128_kernel(const T* x, int64_t ldx, const SegSrc src, uint8_t* out, int64_t ldo, float* scale, int64_t lds,
                                                                 int64_t rows, int dim, int col_tiles) {
  const int lane = threadIdx.x & 63;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t r0 = w / col_tiles * QR;
  const int col = (int)(w % col_tiles) * 512 + lane * 8;
  if (r0 >= rows || col - (lane & 15) * 8 >= dim) return;  // whole groups leave: the 16 lanes of a group stay together
  const int n = (int)min((int64_t)QR, rows - r0);
  const bool live = col < dim;
  float keep = 0.f;
  float f[QR][8];
#pragma unroll
  for (int i = 0; i < QR; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
  // Short calls load rows past the last one again, so that no branch parts the loads ([257, 1280] 4.5 us of kernel against
  // 5.3, [4680, 5120] 16.5 against 18.2, inputs from memory).  Long ones wait for each row's before the next row's test: fewer loads
  // at a time, alike at most sizes and better at the largest ([75600, 13824] 535 us against 553, [75600, 5120] 204 against 200).
  if constexpr (BIG) {
#pragma unroll
    for (int i = 0; i < QR; ++i)
      if (live && i < n) load8_once<BIG>(seg_chunk(x, ldx, src, r0 + i, col), f[i]);
  } else if (live) {
#pragma unroll
    for (int i = 0; i < QR; ++i) load8_once<BIG>(seg_chunk(x, ldx, src, r0 + min(i, n - 1), col), f[i]);
  }
#pragma unroll
  for (int i = 0; i < QR; ++i) {
    if (i < n) {
      const float sc = scale_e4m3(max16(absmax8(f[i])));  // (lanes past the row's end hold zeros and take part in the rotations)
      if (i == (lane & 15)) keep = sc;
      if (live) st<BIG>(reinterpret_cast<u32x2*>(out + (r0 + i) * ldo + col), cvt8_e4m3(f[i], __frcp_rn(sc)));
    }
  }
  if ((lane & 15) < n) scale[(int64_t)(col >> 7) * lds + r0 + (lane & 15)] = keep;
}

// ---- weights: 128 x 128 blocks --------------------------------------------------------------------
// One workgroup per block: thread t holds columns 8 (t & 15) .. + 7 of rows (t >> 4) + 16 i.
template <class T>
__global__ __launch_bounds__(256) void quant_fp8_block128_kernel(const T* x, int64_t ldx, uint8_t* out, int64_t ldo, float* scale, int64_t lds, int64_t rows, int dim) {
  const int t = threadIdx.x;
  const int64_t r0 = (int64_t)blockIdx.y * 128 + (t >> 4);
  const int col = blockIdx.x * 128 + (t & 15) * 8;
  const bool live = col < dim;
  float f[8][8], amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
    if (live && r0 + 16 * i < rows) load8(x + (r0 + 16 * i) * ldx + col, f[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, absmax8(f[i]));
  amax = max64(amax);
  __shared__ float part[4];
  if ((t & 63) == 0) part[t >> 6] = amax;
  __syncthreads();
  const float sc = scale_e4m3(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  const float inv = __frcp_rn(sc);
  if (t == 0) scale[(int64_t)blockIdx.y * lds + blockIdx.x] = sc;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (live && r0 + 16 * i < rows) *reinterpret_cast<u32x2*>(out + (r0 + 16 * i) * ldo + col) = cvt8_e4m3(f[i], inv);
}

// ---- residual addition + RMSNorm --------------------------------------------------------------------
// WPR waves share a row, which stays in registers between the two passes, so x and y are read once and x and out written
// once.  The sum, the statistics and the normalised row are fp32: the norm sees the sum before its rounding to the stream's type, and the 8-bit forms round
// the fp32 row once, without a bf16 rounding in between.  Bound by memory: 7 bytes an element with bf16 in and out of e4m3
// (8 of bf16 out), 5.8 TB/s at [75600, 5120].  Four waves a row above 1024 columns: a wave then holds at most 32 columns a lane
// and enough waves fit to cover the loads (e4m3 groups at [75600, 5120] 463 us against 528 with a wave a row, and a single row
// of 5120 has 20 loads' latency less); one wave a row up to 1024, where a fourth of the row would leave lanes idle
// ([65536, 1024] 78 us against 105, [32760, 512] 21 against 30).
enum { FORM_BF16 = -1, FORM_ROW = LX2V_QUANT_FP8_ROW, FORM_GROUP = LX2V_QUANT_FP8_GROUP128, FORM_INT8 = LX2V_QUANT_INT8_ROW };

template <bool BIG>
LX2V_DEVICE void store8(uint16_t* p, const float (&f)[8]) { st<BIG>(reinterpret_cast<u32x4*>(p), pack8(f)); }
template <bool BIG>
LX2V_DEVICE void store8(float* p, const float (&f)[8]) {
  st<BIG>(reinterpret_cast<f32x4*>(p), f32x4{f[0], f[1], f[2], f[3]});
  st<BIG>(reinterpret_cast<f32x4*>(p + 4), f32x4{f[4], f[5], f[6], f[7]});
}

template <class T, int FORM, int WPR, int NC, bool BIG>
__global__ __launch_bounds__(256) void add_rmsnorm_kernel(T* x, int64_t ldx, const uint16_t* y, int64_t ldy, const float* w, void* out, int64_t ldo, float* scale,
                                                          int64_t lds, int64_t rows, int dim, float eps) {
  constexpr int TPR = 64 * WPR;  // threads per row
  __shared__ float part[2][4];
  const int t = threadIdx.x & (TPR - 1);
  const int64_t row = (int64_t)blockIdx.x * (4 / WPR) + threadIdx.x / TPR;
  if (row >= rows) return;  // whole rows leave; with WPR = 4 a workgroup is one row
  const int nchunks = dim >> 3;
  T* xr = x + row * ldx;
  float f[NC][8];
  float ss = 0.f;
  // As in the group quantiser: short calls load without branches in between (lanes past the row's end its last chunk again; one row
  // of 5120 3.4 us of kernel against 3.9, [4680, 5120] 36.4 against 39.3), long ones chunk by chunk ([75600, 5120] 466 against 478).
  if constexpr (BIG) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int ch = t + TPR * c;
#pragma unroll
      for (int j = 0; j < 8; ++j) f[c][j] = 0.f;
      if (ch < nchunks) {
        load8_once<BIG>(xr + ch * 8, f[c]);
        if (y != nullptr) {
          float b[8];
          load8_once<BIG>(y + row * ldy + ch * 8, b);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[c][j] += b[j];
        }
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < NC; ++c) load8_once<BIG>(xr + min(t + TPR * c, nchunks - 1) * 8, f[c]);
    if (y != nullptr) {
      const uint16_t* yr = y + row * ldy;
      float b[NC][8];
#pragma unroll
      for (int c = 0; c < NC; ++c) load8_once<BIG>(yr + min(t + TPR * c, nchunks - 1) * 8, b[c]);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) f[c][j] += b[c][j];
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) f[c][j] = t + TPR * c < nchunks ? f[c][j] : 0.f;
  }
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = __builtin_fmaf(f[c][j], f[c][j], ss);
  ss = wave_sum(ss);
  if constexpr (WPR == 4) {
    if ((t & 63) == 0) part[0][t >> 6] = ss;
    __syncthreads();
    ss = (part[0][0] + part[0][1]) + (part[0][2] + part[0][3]);
  }
  const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)dim) + eps));
  float amax = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int ch = t + TPR * c;
    if (ch < nchunks) {
      if (y != nullptr) store8<BIG>(xr + ch * 8, f[c]);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[c][j] *= rstd;
      if (w != nullptr) {
        float g[8];
        load8(w + ch * 8, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[c][j] *= g[j];
      }
      if constexpr (FORM == FORM_BF16) store8<BIG>(static_cast<uint16_t*>(out) + row * ldo + ch * 8, f[c]);
      if constexpr (FORM == FORM_ROW) amax = fmaxf(amax, absmax8(f[c]));
      if constexpr (FORM == FORM_INT8) amax = fmaxf(amax, absmax8_or_inf(f[c]));
    }
    if constexpr (FORM == FORM_GROUP) {  // (outside the branch: lanes past the row's end hold zeros and take part in the rotations)
      const float sc = scale_e4m3(max16(absmax8(f[c])));
      if (ch < nchunks) {
        st<BIG>(reinterpret_cast<u32x2*>(static_cast<uint8_t*>(out) + row * ldo + ch * 8), cvt8_e4m3(f[c], __frcp_rn(sc)));
        if ((t & 15) == 0) scale[(int64_t)(ch >> 4) * lds + row] = sc;
      }
    }
  }
  if constexpr (FORM == FORM_ROW || FORM == FORM_INT8) {
    amax = max64(amax);
    if constexpr (WPR == 4) {
      if ((t & 63) == 0) part[1][t >> 6] = amax;
      __syncthreads();
      amax = fmaxf(fmaxf(part[1][0], part[1][1]), fmaxf(part[1][2], part[1][3]));
    }
    // int8 codes hold no NaN, so a row with one (in its elements, or because its sum of squares is not finite) says so in its scale
    const bool lost = FORM == FORM_INT8 && !(ss < INFINITY && amax < INFINITY);
    const float sc = FORM == FORM_ROW ? scale_e4m3(amax) : lost ? NAN : __fdiv_rn(amax, 127.0f);
    const float inv = FORM == FORM_ROW ? __frcp_rn(sc) : amax > 0.f ? __fdiv_rn(127.0f, amax) : 0.f;
    if (t == 0) scale[row] = sc;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int ch = t + TPR * c;
      if (ch >= nchunks) continue;
      u32x2 q = {0u, 0u};
      if constexpr (FORM == FORM_ROW) {
        q = cvt8_e4m3(f[c], inv);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float v = fminf(fmaxf(rintf(__fmul_rn(f[c][j], inv)), -128.0f), 127.0f);
          q[j >> 2] |= ((uint32_t)(int)v & 0xffu) << (8 * (j & 3));
        }
      }
      st<BIG>(reinterpret_cast<u32x2*>(static_cast<uint8_t*>(out) + row * ldo + ch * 8), q);
    }
  }
}

template <class T, int FORM>
void add_rmsnorm_launch(T* x, int64_t ldx, const uint16_t* y, int64_t ldy, const float* w, void* out, int64_t ldo, float* scale, int64_t lds, int64_t rows, int dim, float eps,
                        hipStream_t stream) {
  const int nchunks = dim >> 3;
  const bool big = rows * dim * (int64_t)(sizeof(T) + (y ? 2 : 0) + (FORM == FORM_BF16 ? 2 : 1)) > STREAMED_BYTES;
#define LX2V_ARN(WPR, NC)                                                                                                                                                      \
  hipLaunchKernelGGL((big ? add_rmsnorm_kernel<T, FORM, WPR, NC, true> : add_rmsnorm_kernel<T, FORM, WPR, NC, false>), dim3((unsigned)((rows + 4 / WPR - 1) / (4 / WPR))), dim3(256), 0, \
                     stream, x, ldx, y, ldy, w, out, ldo, scale, lds, rows, dim, eps)
  if (nchunks <= 64) LX2V_ARN(1, 1);
  else if (nchunks <= 128) LX2V_ARN(1, 2);
  else if (nchunks <= 256) LX2V_ARN(4, 1);
  else if (nchunks <= 512) LX2V_ARN(4, 2);
  else if (nchunks <= 768) LX2V_ARN(4, 3);
  else LX2V_ARN(4, 4);
#undef LX2V_ARN
}

template <class T>
int add_rmsnorm(const char* what, T* x, int64_t ldx, const uint16_t* y, int64_t ldy, const float* w, void* out, int64_t ldo, float* scale, int64_t lds, int form, int64_t rows,
                int dim, float eps, void* stream) {
  LX2V_REQUIRE(form >= FORM_BF16 && form <= FORM_INT8, LX2V_EINVAL, "%s: unknown output form %d", what, form);
  LX2V_REQUIRE(rows == 0 || (x && out && (form == FORM_BF16 || scale)), LX2V_EINVAL, "%s: null tensor", what);
  LX2V_REQUIRE(rows >= 0 && dim > 0, LX2V_EINVAL, "%s: bad shape rows=%lld dim=%d", what, (long long)rows, dim);
  LX2V_REQUIRE(dim % 8 == 0 && dim <= 8192, LX2V_EUNSUP, "%s: dim=%d must be a multiple of 8 and <= 8192", what, dim);
  LX2V_REQUIRE((dim <= 1024 ? (rows + 3) / 4 : rows) < MAX_BLOCKS, LX2V_EUNSUP, "%s: rows=%lld, a launch has less than 2^24 workgroups", what, (long long)rows);
  LX2V_REQUIRE(ldx % 8 == 0 && ldo % 8 == 0 && ldx >= dim && ldo >= dim, LX2V_EINVAL, "%s: row strides must be multiples of 8 and >= dim", what);
  LX2V_REQUIRE(y == nullptr || (ldy % 8 == 0 && ldy >= dim && lx2v_aligned16(y)), LX2V_EINVAL, "%s: y must be 16-byte aligned with a row stride that is a multiple of 8 and >= dim", what);
  LX2V_REQUIRE(lx2v_aligned16(x) && lx2v_aligned16(w), LX2V_EINVAL, "%s: tensors must be 16-byte aligned", what);
  LX2V_REQUIRE(form == FORM_BF16 ? lx2v_aligned16(out) : (reinterpret_cast<uintptr_t>(out) & 7u) == 0, LX2V_EINVAL, "%s: out must be 16-byte aligned (8-bit rows: 8-byte)", what);
  LX2V_REQUIRE(form != FORM_GROUP || lds >= rows, LX2V_EINVAL, "%s: the stride between groups of scales must be >= rows", what);
  LX2V_REQUIRE(rows == 0 || static_cast<const void*>(x) != out, LX2V_EINVAL, "%s: out may not be x", what);
  if (rows == 0) return LX2V_OK;
  hipStream_t hs = (hipStream_t)stream;
  switch (form) {
    case FORM_BF16: add_rmsnorm_launch<T, FORM_BF16>(x, ldx, y, ldy, w, out, ldo, scale, lds, rows, dim, eps, hs); break;
    case FORM_ROW: add_rmsnorm_launch<T, FORM_ROW>(x, ldx, y, ldy, w, out, ldo, scale, lds, rows, dim, eps, hs); break;
    case FORM_GROUP: add_rmsnorm_launch<T, FORM_GROUP>(x, ldx, y, ldy, w, out, ldo, scale, lds, rows, dim, eps, hs); break;
    default: add_rmsnorm_launch<T, FORM_INT8>(x, ldx, y, ldy, w, out, ldo, scale, lds, rows, dim, eps, hs); break;
  }
  LX2V_CHECK_LAUNCH(what);
  return LX2V_OK;
}

template <class T>
int quant_group128(const T* x, int64_t ldx, const lx2v_kseg* kseg, uint8_t* out, int64_t ldo, float* scale, int64_t lds, int64_t rows, int dim, void* stream) {
  LX2V_REQUIRE(rows == 0 || (x && out && scale), LX2V_EINVAL, "quant_fp8_group128: null tensor");
  LX2V_REQUIRE(rows >= 0 && dim > 0 && dim % 8 == 0, LX2V_EINVAL, "quant_fp8_group128: dim=%d must be a positive multiple of 8", dim);
  LX2V_REQUIRE(dim <= MAX_DIM, LX2V_EUNSUP, "quant_fp8_group128: dim=%d, at most %d columns are supported", dim, MAX_DIM);
  LX2V_REQUIRE(ldx % 8 == 0 && ldo % 8 == 0 && ldo >= dim, LX2V_EINVAL, "quant_fp8_group128: row strides must be multiples of 8, the output's >= dim");
  LX2V_REQUIRE(lx2v_aligned16(x) && (reinterpret_cast<uintptr_t>(out) & 7u) == 0, LX2V_EINVAL, "quant_fp8_group128: x must be 16-byte, out 8-byte aligned");
  LX2V_REQUIRE(lds >= rows, LX2V_EINVAL, "quant_fp8_group128: the stride between groups of scales must be >= rows");
  SegSrc g;
  if (const int rc = seg_src_from(kseg, ldx, dim, "quant_fp8_group128", g); rc != LX2V_OK) return rc;
  if (rows == 0) return LX2V_OK;
  const int col_tiles = (dim + 511) / 512;
  const int64_t blocks = ((rows + QR - 1) / QR * col_tiles + 3) / 4;
  LX2V_REQUIRE(blocks < MAX_BLOCKS, LX2V_EUNSUP, "quant_fp8_group128: rows=%lld, a launch has less than 2^24 workgroups", (long long)rows);
  const bool big = rows * dim * (int64_t)(sizeof(T) + 1) > STREAMED_BYTES;
  auto kernel = big ? quant_fp8_group128_kernel<T, true> : quant_fp8_group128_kernel<T, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, x, ldx, g, out, ldo, scale, lds, rows, dim, col_tiles);
  LX2V_CHECK_LAUNCH("quant_fp8_group128");
  return LX2V_OK;
}

template <class T>
int quant_block128(const T* x, int64_t ldx, uint8_t* out, int64_t ldo, float* scale, int64_t lds, int64_t rows, int dim, void* stream) {
  LX2V_REQUIRE(rows == 0 || (x && out && scale), LX2V_EINVAL, "quant_fp8_block128: null tensor");
  LX2V_REQUIRE(rows >= 0 && dim > 0 && dim % 8 == 0, LX2V_EINVAL, "quant_fp8_block128: dim=%d must be a positive multiple of 8", dim);
  LX2V_REQUIRE(dim <= MAX_DIM, LX2V_EUNSUP, "quant_fp8_block128: dim=%d, at most %d columns are supported", dim, MAX_DIM);
  LX2V_REQUIRE(ldx % 8 == 0 && ldo % 8 == 0 && ldx >= dim && ldo >= dim, LX2V_EINVAL, "quant_fp8_block128: row strides must be multiples of 8 and >= dim");
  LX2V_REQUIRE(lx2v_aligned16(x) && (reinterpret_cast<uintptr_t>(out) & 7u) == 0, LX2V_EINVAL, "quant_fp8_block128: x must be 16-byte, out 8-byte aligned");
  LX2V_REQUIRE(lds >= (dim + 127) / 128, LX2V_EINVAL, "quant_fp8_block128: the row stride of the scales must be >= ceil(dim / 128)");
  LX2V_REQUIRE((rows + 127) / 128 <= 65535, LX2V_EUNSUP, "quant_fp8_block128: rows=%lld, at most 65535 blocks of 128 are supported", (long long)rows);
  if (rows == 0) return LX2V_OK;
  hipLaunchKernelGGL(quant_fp8_block128_kernel<T>, dim3((unsigned)((dim + 127) / 128), (unsigned)((rows + 127) / 128)), dim3(256), 0, (hipStream_t)stream, x, ldx, out, ldo, scale, lds,
                     rows, dim);
  LX2V_CHECK_LAUNCH("quant_fp8_block128");
  return LX2V_OK;
}

}  // namespace

extern "C" int lx2v_quant_fp8_group128(const uint16_t* x, int64_t ldx, const lx2v_kseg* kseg, uint8_t* out, int64_t ldo, float* scale, int64_t ld_scale, int64_t rows, int dim,
                                       void* stream) {
  return quant_group128(x, ldx, kseg, out, ldo, scale, ld_scale, rows, dim, stream);
}

extern "C" int lx2v_quant_fp8_group128_f32(const float* x, int64_t ldx, uint8_t* out, int64_t ldo, float* scale, int64_t ld_scale, int64_t rows, int dim, void* stream) {
  return quant_group128(x, ldx, static_cast<const lx2v_kseg*>(nullptr), out, ldo, scale, ld_scale, rows, dim, stream);
}

extern "C" int lx2v_quant_fp8_block128(const uint16_t* w, int64_t ldw, uint8_t* out, int64_t ldo, float* scale, int64_t ld_scale, int64_t rows, int dim, void* stream) {
  return quant_block128(w, ldw, out, ldo, scale, ld_scale, rows, dim, stream);
}

extern "C" int lx2v_quant_fp8_block128_f32(const float* w, int64_t ldw, uint8_t* out, int64_t ldo, float* scale, int64_t ld_scale, int64_t rows, int dim, void* stream) {
  return quant_block128(w, ldw, out, ldo, scale, ld_scale, rows, dim, stream);
}

extern "C" int lx2v_add_rmsnorm_bf16(uint16_t* x, int64_t ldx, const uint16_t* y, int64_t ldy, const float* w, uint16_t* out, int64_t ldo, int64_t rows, int dim, float eps,
                                     void* stream) {
  return add_rmsnorm("add_rmsnorm", x, ldx, y, ldy, w, out, ldo, static_cast<float*>(nullptr), 0, FORM_BF16, rows, dim, eps, stream);
}

extern "C" int lx2v_add_rmsnorm_f32(float* x, int64_t ldx, const uint16_t* y, int64_t ldy, const float* w, uint16_t* out, int64_t ldo, int64_t rows, int dim, float eps,
                                    void* stream) {
  return add_rmsnorm("add_rmsnorm_f32", x, ldx, y, ldy, w, out, ldo, static_cast<float*>(nullptr), 0, FORM_BF16, rows, dim, eps, stream);
}

extern "C" int lx2v_add_rmsnorm_quant_bf16(uint16_t* x, int64_t ldx, const uint16_t* y, int64_t ldy, const float* w, void* out, int64_t ldo, float* scale, int64_t ld_scale, int form,
                                           int64_t rows, int dim, float eps, void* stream) {
  LX2V_REQUIRE(form != FORM_BF16, LX2V_EINVAL, "add_rmsnorm_quant: unknown output form %d", form);
  return add_rmsnorm("add_rmsnorm_quant", x, ldx, y, ldy, w, out, ldo, scale, ld_scale, form, rows, dim, eps, stream);
}

extern "C" int lx2v_add_rmsnorm_quant_f32(float* x, int64_t ldx, const uint16_t* y, int64_t ldy, const float* w, void* out, int64_t ldo, float* scale, int64_t ld_scale, int form,
                                          int64_t rows, int dim, float eps, void* stream) {
  LX2V_REQUIRE(form != FORM_BF16, LX2V_EINVAL, "add_rmsnorm_quant_f32: unknown output form %d", form);
  return add_rmsnorm("add_rmsnorm_quant_f32", x, ldx, y, ldy, w, out, ldo, scale, ld_scale, form, rows, dim, eps, stream);
}
