// Shared by the quantisers (step_ew.hip: one scale per row; block_quant.hip: one scale per group of 128 columns): the
// source rows they read, plain or stored as column segments.
#pragma once

#include "common.h"

namespace {

// A source row whose columns are stored as segments (lx2v_kseg; seg == 0: a plain row).  All segment
// widths are multiples of 8, so a 16-byte chunk never straddles two segments.
struct SegSrc {
  int64_t seg, stride, split, seg2, stride2, base2, lda2;
};
// Eight consecutive source elements as fp32: bf16 (one 16-byte chunk) or fp32 (two).
LX2V_DEVICE void load8(const uint16_t* p, float (&f)[8]) { unpack8(*reinterpret_cast<const u32x4*>(p), f); }
LX2V_DEVICE void load8(const float* p, float (&f)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = a[i];
    f[4 + i] = b[i];
  }
}
template <class T>
LX2V_DEVICE const T* seg_chunk(const T* x, int64_t ldx, const SegSrc& g, int64_t row, int col) {
  if (g.seg == 0) return x + row * ldx + col;
  if (g.split == 0 || col < g.split) {
    const int64_t s = col / g.seg;
    return x + s * g.stride + row * ldx + (col - s * g.seg);
  }
  const int64_t c2 = col - g.split, t = c2 / g.seg2;
  return x + g.base2 + t * g.stride2 + row * g.lda2 + (c2 - t * g.seg2);
}

// Validates a segmented source description against `dim` and returns its device form (all zero = plain).
int seg_src_from(const lx2v_kseg* kseg, int64_t ldx, int dim, const char* what, SegSrc& g) {
  g = SegSrc{0, 0, 0, 0, 0, 0, 0};
  if (kseg == nullptr) {
    LX2V_REQUIRE(ldx >= dim, LX2V_EINVAL, "%s: row stride smaller than the row", what);
    return LX2V_OK;
  }
  LX2V_REQUIRE(kseg->seg > 0 && kseg->seg % 8 == 0 && kseg->stride % 8 == 0 && ldx >= kseg->seg, LX2V_EINVAL, "%s: segments must be multiples of 8 columns, 8-aligned, inside a row", what);
  const int64_t k1 = kseg->split > 0 ? kseg->split : dim;
  LX2V_REQUIRE(k1 % kseg->seg == 0 && k1 <= dim, LX2V_EINVAL, "%s: region 1 (%lld columns) must hold whole segments of %lld", what, (long long)k1, (long long)kseg->seg);
  if (kseg->split > 0) {
    LX2V_REQUIRE(kseg->seg2 > 0 && kseg->seg2 % 8 == 0 && kseg->stride2 % 8 == 0 && kseg->base2 % 8 == 0 && kseg->lda2 % 8 == 0 && kseg->lda2 >= kseg->seg2 &&
                     (dim - kseg->split) % kseg->seg2 == 0,
                 LX2V_EINVAL, "%s: region 2 must hold whole, 8-aligned segments", what);
  }
  g = SegSrc{kseg->seg, kseg->stride, kseg->split, kseg->seg2, kseg->stride2, kseg->base2, kseg->lda2};
  return LX2V_OK;
}

}  // namespace
