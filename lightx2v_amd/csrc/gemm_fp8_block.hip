// Block-scaled e4m3 Linear, bf16 out:
//   C[m, n] = epilogue( sum_b sa[m, b] sw[n / 128, b] * sum_{k in block b} A8[m, k] W8[n, k]  + bias[n] ),
// blocks b of 128 columns of K; one fp32 scale per row and block of the activation, one per 128 x 128 block of the
// weight.  One v_mfma_f32_16x16x128_f8f6f4 started from zero covers exactly one block b of a 16 x 16 corner; its four
// results a lane are then added to the fp32 accumulators with one fma each, times sa[m, b] * sw[n / 128, b].  The scales
// change with b, so they cannot wait for the epilogue, and they are arbitrary fp32 values, so the power-of-two block
// scales of the MFMA cannot hold them.  The weight rows are the MFMA's first operand: a lane then holds four columns of
// ONE row m, and both scales are one value per lane and corner.
//
// Precision: the instruction adds its 128 products with an fp32-like sum over runs of 8 consecutive k, but within a run
// it keeps only 13 bits below the largest of the eight products (measured).  Against 64 bits that is 1e-5 to 5e-5 of a result, a
// hundredth of its rounding to bf16; widening to bf16 operands would avoid it at half the MFMA rate and twice the LDS
// traffic.  Everything behind the instruction is fp32.
//
// Two kernels.  `tile`: 4 waves (2 x 2), operand tiles of 128 bytes of K per row staged into LDS by LDS-DMA.
// `skinny` (few rows): every wave streams its own weight rows straight into fragment registers, waves split K.
// Rows past M / N and columns past K arrive as zeros (range check of the buffer descriptors).
#include <algorithm>

#include "common.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int BK = 128;
constexpr int EPI_PARTIAL = 3;  // kernel instance that leaves the fp32 sums of a K range in the workspace (internal)

struct Params {
  const uint8_t* A;
  const uint8_t* W;
  const float* a_scale;
  const float* w_scale;
  const float* bias;
  uint16_t* C;
  const uint16_t* resid;
  const float* gate;
  float* partials;  // [split][M][N]
  int64_t lda, ldw, ldc, ldr, lds_a, lds_w;
  int M, N, K;
  int tiles_m, tiles_n;
  int nk;          // K blocks
  int split, per;  // K ranges and K blocks in each
};

template <int N>
struct IntC {
  static constexpr int value = N;
};
template <int B, int E, class F>
LX2V_DEVICE void static_for(F&& f) {
  if constexpr (B < E) {
    f(IntC<B>{});
    static_for<B + 1, E>(f);
  }
}

// Blocks that share an XCD (same blockIdx % 8) get a contiguous run of work items.
LX2V_DEVICE int xcd_remap(int bid, int nwg) {
  const int q = nwg >> 3, r = nwg & 7, xcd = bid & 7;
  const int base = xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q;
  return base + (bid >> 3);
}

LX2V_DEVICE u32x4 raw_descriptor(const void* base, int64_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  u32x4 d;
  d[0] = __builtin_amdgcn_readfirstlane((uint32_t)a);
  d[1] = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));  // stride 0: raw buffer
  d[2] = __builtin_amdgcn_readfirstlane((uint32_t)(bytes < 0 ? 0 : (bytes > 0x7fffffffLL ? 0x7fffffffLL : bytes)));  // loads at or past it return 0
  d[3] = 0x00020000u;
  return d;
}

LX2V_DEVICE f32x4 mfma_block(const i32x8& w, const i32x8& a) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);  // (zero scale operands: the form without block scales)
}

// Four consecutive columns n .. n + 3 of row m: bias, then GELU / gated residual, one rounding.
template <int EPI>
LX2V_DEVICE void finish4(const Params& p, const f32x4& acc, int64_t m, int n) {
  float v[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = acc[j];
  if (p.bias != nullptr) {
    const f32x4 b = *reinterpret_cast<const f32x4*>(p.bias + n);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += b[j];
  }
  if constexpr (EPI == LX2V_EPI_GELU_TANH) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = gelu_tanh(v[j]);
  }
  if constexpr (EPI == LX2V_EPI_RESIDUAL) {
    if (p.gate != nullptr) {
      const f32x4 g = *reinterpret_cast<const f32x4*>(p.gate + n);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= g[j];
    }
    const u32x2 r = *reinterpret_cast<const u32x2*>(p.resid + m * p.ldr + n);
    v[0] += __uint_as_float(r[0] << 16);
    v[1] += __uint_as_float(r[0] & 0xffff0000u);
    v[2] += __uint_as_float(r[1] << 16);
    v[3] += __uint_as_float(r[1] & 0xffff0000u);
  }
  *reinterpret_cast<u32x2*>(p.C + m * p.ldc + n) = u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])};
}

// ---- tile kernel ------------------------------------------------------------------------------------
// Workgroup = 4 waves (2 x 2), wave tile 16 MT x 16 NT, a ring of S operand tiles in LDS.  Slot: A rows | W rows (128
// bytes a row, 16-byte chunk c at position c ^ ((row >> 1) & 7)) | 1 KiB of scales (256 bytes filled by each wave's one
// 4-byte DMA: waves 0 .. the A scales of 64 rows each, wave 3 the weight scales of the tile's one or two row blocks).
template <int MT, int NT, int S>
struct Tile {
  static constexpr int TM = 32 * MT, TN = 32 * NT;
  static constexpr int A_BYTES = TM * BK, W_BYTES = TN * BK;
  static constexpr int SLOT = A_BYTES + W_BYTES + 1024;
  static constexpr int LDS = S * SLOT;
  static constexpr int PA = TM / 32, PW = TN / 32;  // 1 KiB DMA pieces (8 rows) of a wave
  static constexpr int PIECES = PA + PW + 1;
};

template <int MT, int NT, int S, int EPI>
__global__ __launch_bounds__(256) void gemm_fp8_block_tile_kernel(const Params p) {
  using T = Tile<MT, NT, S>;
  __shared__ __attribute__((aligned(16))) char lds[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid >> 1, wn = wid & 1;
  const int fr = lane & 15, fq = lane >> 4;

  const int item = xcd_remap(blockIdx.x, gridDim.x);
  const int part = item % p.split, tile = item / p.split;
  constexpr int GROUP_M = 4;  // row panels that share one sweep over the columns
  const int group_sz = GROUP_M * p.tiles_n, first_m = tile / group_sz * GROUP_M;
  const int gm = min(p.tiles_m - first_m, GROUP_M), in_g = tile % group_sz;
  const int m0 = (first_m + in_g % gm) * T::TM, n0 = in_g / gm * T::TN;
  const int kb0 = part * p.per, nk = min(p.per, p.nk - kb0);

  const uint32_t lds_base = __builtin_amdgcn_readfirstlane((uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds);
  constexpr int NOWHERE = (int)0x80000000u;  // an offset past the end of every descriptor

  // ---- staging: piece q of wave w fills rows 8 (q * 4 + w) .. + 7 of an operand tile (lane L: row L >> 3, position L & 7)
  int a_pv[T::PA], w_pv[T::PW];
  auto chunk_of = [&](int q) __attribute__((always_inline)) { return (lane & 7) ^ (((8 * (q * 4 + wid) + (lane >> 3)) >> 1) & 7); };
  auto set_voff = [&](bool last) __attribute__((always_inline)) {  // `last`: chunks past K go nowhere
    const int left = p.K - (p.nk - 1) * BK;
#pragma unroll
    for (int q = 0; q < T::PA; ++q) a_pv[q] = last && chunk_of(q) * 16 >= left ? NOWHERE : (8 * (q * 4 + wid) + (lane >> 3)) * (int)p.lda + chunk_of(q) * 16;
#pragma unroll
    for (int q = 0; q < T::PW; ++q) w_pv[q] = last && chunk_of(q) * 16 >= left ? NOWHERE : (8 * (q * 4 + wid) + (lane >> 3)) * (int)p.ldw + chunk_of(q) * 16;
  };
  set_voff(false);
  const u32x4 a_rs = raw_descriptor(p.A + (int64_t)m0 * p.lda, min((int64_t)p.M - m0, (int64_t)T::TM) * p.lda);
  const u32x4 w_rs = raw_descriptor(p.W + (int64_t)n0 * p.ldw, min((int64_t)p.N - n0, (int64_t)T::TN) * p.ldw);
  const bool sw_wave = wid == 3, sa_wave = wid < T::TM / 64;
  const int nb = min(((p.N + 127) >> 7) - (n0 >> 7), (T::TN + 127) / 128);  // weight row blocks of the tile
  const int s_pv = sw_wave ? (lane < nb ? lane * (int)p.lds_w * 4 : NOWHERE) : sa_wave ? (64 * wid + lane) * 4 : NOWHERE;

  auto dma16 = [&](uint32_t dst, const u32x4& rs, int voff, uint32_t soff) __attribute__((always_inline)) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(dst)), "v"(voff), "s"(rs), "s"(soff) : "memory");
  };
  auto stage = [&](int j) __attribute__((always_inline)) {  // K block kb0 + j -> slot j % S
    const uint32_t slot = lds_base + (uint32_t)(j % S) * T::SLOT;
    const int kb = kb0 + j;
    if (kb == p.nk - 1 && (p.K & (BK - 1)) != 0) set_voff(true);
    const uint32_t soff = (uint32_t)kb * BK;
#pragma unroll
    for (int q = 0; q < T::PA; ++q) dma16(slot + 1024 * (q * 4 + wid), a_rs, a_pv[q], soff);
#pragma unroll
    for (int q = 0; q < T::PW; ++q) dma16(slot + T::A_BYTES + 1024 * (q * 4 + wid), w_rs, w_pv[q], soff);
    const float* sb = sw_wave ? p.w_scale + (int64_t)(n0 >> 7) * p.lds_w + kb : p.a_scale + (int64_t)kb * p.lds_a + m0;
    const u32x4 s_rs = raw_descriptor(sb, sw_wave ? ((int64_t)(nb - 1) * p.lds_w + 1) * 4 : sa_wave ? ((int64_t)p.M - m0) * 4 : 0);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(slot + T::A_BYTES + T::W_BYTES + 256 * wid)), "v"(s_pv), "s"(s_rs) : "memory");
  };

  int rd_a[2], rd_w[2];  // the lane's 32 bytes of K: chunks 2 fq, 2 fq + 1 of its row; 16 rows on: + 2048 bytes
  {
    const int ar = wm * 16 * MT + fr, wr = wn * 16 * NT + fr;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      rd_a[c] = ar * BK + (((2 * fq + c) ^ ((ar >> 1) & 7)) << 4);
      rd_w[c] = T::A_BYTES + wr * BK + (((2 * fq + c) ^ ((wr >> 1) & 7)) << 4);
    }
  }
  auto frag = [&](const char* base, const int (&rd)[2], int i) __attribute__((always_inline)) -> i32x8 {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(base + rd[0] + i * 2048), hi = *reinterpret_cast<const i32x4*>(base + rd[1] + i * 2048);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int k = 0; k < NT; ++k) acc[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};

#pragma unroll
  for (int j = 0; j < S - 1; ++j)
    if (j < nk) stage(j);
  for (int j = 0; j < nk; ++j) {
    // this wave's pieces of K block j have landed (younger blocks may be in flight); behind the barrier every wave's have, and
    // every wave has left block j - 1, whose slot block j + S - 1 is staged into
    if (j + S - 2 < nk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((S - 2) * T::PIECES) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (j + S - 1 < nk) stage(j + S - 1);
    const char* slot = lds + (j % S) * T::SLOT;
    const float* sc = reinterpret_cast<const float*>(slot + T::A_BYTES + T::W_BYTES);
    const float sw = sc[192 + ((wn * 16 * NT) >> 7)];
    i32x8 wf[NT];
#pragma unroll
    for (int k = 0; k < NT; ++k) wf[k] = frag(slot, rd_w, k);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const i32x8 af = frag(slot, rd_a, i);
      const float s = sc[wm * 16 * MT + i * 16 + fr] * sw;
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        const f32x4 d = mfma_block(wf[k], af);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][k][e] = __builtin_fmaf(d[e], s, acc[i][k][e]);
      }
    }
  }

#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = m0 + wm * 16 * MT + i * 16 + fr;
    if (m >= p.M) continue;
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      const int n = n0 + wn * 16 * NT + k * 16 + fq * 4;
      if (n >= p.N) continue;  // N % 8 == 0: all four columns or none
      if constexpr (EPI == EPI_PARTIAL) *reinterpret_cast<f32x4*>(p.partials + ((int64_t)part * p.M + m) * p.N + n) = acc[i][k];
      else finish4<EPI>(p, acc[i][k], m, n);
    }
  }
}

// Sum of the K ranges in their order, then the epilogue: four columns per thread.
template <int EPI>
__global__ __launch_bounds__(256) void gemm_fp8_block_join_kernel(const Params p) {
  const int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, total = (int64_t)p.M * p.N;
  if (e >= total) return;
  const int64_t m = e / p.N;
  const int n = (int)(e - m * p.N);
  f32x4 v = *reinterpret_cast<const f32x4*>(p.partials + e);
  for (int s = 1; s < p.split; ++s) v += *reinterpret_cast<const f32x4*>(p.partials + s * total + e);
  finish4<EPI>(p, v, m, n);
}

// ---- skinny kernel: M <= 16 MT ------------------------------------------------------------------------
// Workgroup = 8 waves on 16 columns; wave w takes K blocks w, w + 8, ...; a weight row's 128 bytes of a block are one
// cache line, read once, by one wave, into the fragment registers.  The waves' sums meet in LDS in a fixed order.
template <int MT, int EPI>
__global__ __launch_bounds__(512) void gemm_fp8_block_skinny_kernel(const Params p) {
  __shared__ __attribute__((aligned(16))) f32x4 red[8][MT][64];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const uint8_t* wrow = p.W + (int64_t)min(n0 + fr, p.N - 1) * p.ldw + fq * 32;
  const uint8_t* arow[MT];
  int am[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    am[i] = min(i * 16 + fr, p.M - 1);
    arow[i] = p.A + (int64_t)am[i] * p.lda + fq * 32;
  }
  const float* swp = p.w_scale + (int64_t)(n0 >> 7) * p.lds_w;
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto load = [&](const uint8_t* row, int kb) __attribute__((always_inline)) -> i32x8 {
    const int k = kb * BK + fq * 32;  // K % 16 == 0: 16 bytes are inside or outside together
    i32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (k < p.K) lo = *reinterpret_cast<const i32x4*>(row + (int64_t)kb * BK);
    if (k + 16 < p.K) hi = *reinterpret_cast<const i32x4*>(row + (int64_t)kb * BK + 16);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  for (int kb = wid; kb < p.nk; kb += 8) {
    const i32x8 wf = load(wrow, kb);
    const float sw = swp[kb];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const f32x4 d = mfma_block(wf, load(arow[i], kb));
      const float s = p.a_scale[(int64_t)kb * p.lds_a + am[i]] * sw;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = __builtin_fmaf(d[e], s, acc[i][e]);
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) red[wid][i][lane] = acc[i];
  __syncthreads();
  if (wid < MT) {
    f32x4 v = red[0][wid][lane];
#pragma unroll
    for (int w = 1; w < 8; ++w) v += red[w][wid][lane];
    const int m = wid * 16 + fr, n = n0 + fq * 4;
    if (m < p.M && n < p.N) finish4<EPI>(p, v, m, n);
  }
}

int device_cus() {
  static int cus_cached[64];
  int dev = 0, cus = 256;
  if (hipGetDevice(&dev) == hipSuccess && dev >= 0 && dev < 64) {
    if (cus_cached[dev] == 0) {
      int v = 0;
      cus_cached[dev] = (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && v > 0) ? v : 256;
    }
    cus = cus_cached[dev];
  }
  return cus;
}

enum Kind { SKINNY, TILE_64x128, TILE_128x128, TILE_192x256 };
struct Plan {
  Kind kind;
  int tm, tn, split, per;
  int64_t bytes;
};

Plan make_plan(int64_t M, int64_t N, int64_t K, int cus) {
  const int nk = (int)((K + BK - 1) / BK);
  if (M <= 16) return Plan{SKINNY, 16, 16, 1, nk, 0};
  Plan q{TILE_192x256, 192, 256, 1, nk, 0};
  auto tiles = [&](int tm, int tn) { return ((M + tm - 1) / tm) * ((N + tn - 1) / tn); };
  if (tiles(192, 256) < cus) q = Plan{TILE_128x128, 128, 128, 1, nk, 0};
  if (q.kind == TILE_128x128 && (M <= 64 || tiles(128, 128) < cus)) q = Plan{TILE_64x128, 64, 128, 1, nk, 0};
  const int64_t t = tiles(q.tm, q.tn);
  if (q.kind == TILE_64x128 && t < 2 * cus) {
    int split = (int)std::min<int64_t>(2 * cus / t, std::max(1, nk / 4));
    const int per = (nk + split - 1) / split;
    split = (nk + per - 1) / per;
    if (split > 1) {
      q.split = split;
      q.per = per;
      q.bytes = (int64_t)split * M * N * 4;
    }
  }
  return q;
}

template <int MT, int NT, int S, int EPI>
void launch_tile(const Params& p, int64_t items, hipStream_t st) {
  hipLaunchKernelGGL((gemm_fp8_block_tile_kernel<MT, NT, S, EPI>), dim3((unsigned)items), dim3(256), 0, st, p);
}

template <int EPI>
void launch(const Params& p, Kind kind, hipStream_t st) {
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.split;
  switch (kind) {
    case SKINNY:
      if constexpr (EPI != EPI_PARTIAL) hipLaunchKernelGGL((gemm_fp8_block_skinny_kernel<1, EPI>), dim3((unsigned)p.tiles_n), dim3(512), 0, st, p);
      return;
    case TILE_64x128: return launch_tile<2, 4, 3, EPI>(p, items, st);
    case TILE_128x128: return launch_tile<4, 4, 2, EPI>(p, items, st);
    default: return launch_tile<6, 8, 2, EPI>(p, items, st);
  }
}

}  // namespace

extern "C" int64_t lx2v_gemm_fp8_block128_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0 || M >= (1LL << 31) || N >= (1LL << 31) || K >= (1LL << 31)) return 0;
  return make_plan(M, N, K, device_cus()).bytes;
}

extern "C" int lx2v_gemm_fp8_block128(const uint8_t* A, int64_t lda, const float* a_scale, int64_t ld_a_scale, const uint8_t* W, int64_t ldw, const float* w_scale,
                                      int64_t ld_w_scale, const float* bias, uint16_t* C, int64_t ldc, int64_t M, int64_t N, int64_t K, int epilogue, const uint16_t* resid,
                                      int64_t ldr, const float* gate, void* workspace, int64_t workspace_bytes, void* stream) {
  LX2V_REQUIRE(M == 0 || (A && W && C && a_scale && w_scale), LX2V_EINVAL, "gemm_fp8_block128: null tensor");
  LX2V_REQUIRE(M >= 0 && N > 0 && K > 0, LX2V_EINVAL, "gemm_fp8_block128: bad shape M=%lld N=%lld K=%lld", (long long)M, (long long)N, (long long)K);
  LX2V_REQUIRE(M < (1LL << 31) && N < (1LL << 31) && K < (1LL << 31), LX2V_EUNSUP, "gemm_fp8_block128: dimensions must fit in 31 bits");
  LX2V_REQUIRE(K % 16 == 0 && N % 8 == 0, LX2V_EUNSUP, "gemm_fp8_block128: K=%lld must be a multiple of 16, N=%lld of 8", (long long)K, (long long)N);
  LX2V_REQUIRE(lda % 16 == 0 && ldw % 16 == 0 && ldc % 8 == 0, LX2V_EINVAL, "gemm_fp8_block128: fp8 row strides must be multiples of 16, ldc of 8");
  LX2V_REQUIRE(lda >= K && ldw >= K && ldc >= N, LX2V_EINVAL, "gemm_fp8_block128: row stride smaller than the row length");
  LX2V_REQUIRE(lda < (1LL << 22) && ldw < (1LL << 22), LX2V_EUNSUP, "gemm_fp8_block128: fp8 row strides must be below 4 MiB (a tile's rows are addressed with 31 bits)");
  LX2V_REQUIRE(ld_a_scale >= M && ld_w_scale >= (K + BK - 1) / BK, LX2V_EINVAL, "gemm_fp8_block128: ld_a_scale must be >= M, ld_w_scale >= ceil(K / 128)");
  LX2V_REQUIRE(ld_w_scale < (1LL << 28), LX2V_EUNSUP, "gemm_fp8_block128: ld_w_scale=%lld is too large", (long long)ld_w_scale);
  LX2V_REQUIRE(lx2v_aligned16(A) && lx2v_aligned16(W) && lx2v_aligned16(C) && lx2v_aligned16(bias), LX2V_EINVAL, "gemm_fp8_block128: tensors must be 16-byte aligned");
  LX2V_REQUIRE((reinterpret_cast<uintptr_t>(a_scale) & 3u) == 0 && (reinterpret_cast<uintptr_t>(w_scale) & 3u) == 0, LX2V_EINVAL, "gemm_fp8_block128: scales must be 4-byte aligned");
  LX2V_REQUIRE(epilogue == LX2V_EPI_NONE || epilogue == LX2V_EPI_GELU_TANH || epilogue == LX2V_EPI_RESIDUAL, LX2V_EINVAL, "gemm_fp8_block128: unknown epilogue %d", epilogue);
  if (epilogue == LX2V_EPI_RESIDUAL) {
    LX2V_REQUIRE(M == 0 || (resid != nullptr && ldr % 8 == 0 && ldr >= N && lx2v_aligned16(resid)), LX2V_EINVAL, "gemm_fp8_block128: residual epilogue needs an aligned resid with ldr >= N");
    LX2V_REQUIRE(lx2v_aligned16(gate), LX2V_EINVAL, "gemm_fp8_block128: gate must be 16-byte aligned");
  }
  if (M == 0) return LX2V_OK;

  Plan q = make_plan(M, N, K, device_cus());
  if (q.split > 1 && (workspace == nullptr || !lx2v_aligned16(workspace) || workspace_bytes < q.bytes)) {
    q.split = 1;
    q.per = (int)((K + BK - 1) / BK);
  }
  Params p;
  p.A = A; p.W = W; p.a_scale = a_scale; p.w_scale = w_scale; p.bias = bias; p.C = C; p.resid = resid; p.gate = gate; p.partials = reinterpret_cast<float*>(workspace);
  p.lda = lda; p.ldw = ldw; p.ldc = ldc; p.ldr = ldr; p.lds_a = ld_a_scale; p.lds_w = ld_w_scale;
  p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.nk = (int)((K + BK - 1) / BK);
  p.split = q.split;
  p.per = q.per;
  p.tiles_m = (int)((M + q.tm - 1) / q.tm);
  p.tiles_n = (int)((N + q.tn - 1) / q.tn);
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.split, joins = (M * N / 4 + 255) / 256;
  LX2V_REQUIRE(items < (1LL << 31) && (p.split == 1 || joins < (1LL << 31)), LX2V_EUNSUP, "gemm_fp8_block128: too many tiles");
  hipStream_t st = (hipStream_t)stream;
  if (p.split > 1) {
    launch<EPI_PARTIAL>(p, q.kind, st);
    const dim3 grid((unsigned)joins), block(256);
    switch (epilogue) {
      case LX2V_EPI_NONE: hipLaunchKernelGGL(gemm_fp8_block_join_kernel<LX2V_EPI_NONE>, grid, block, 0, st, p); break;
      case LX2V_EPI_GELU_TANH: hipLaunchKernelGGL(gemm_fp8_block_join_kernel<LX2V_EPI_GELU_TANH>, grid, block, 0, st, p); break;
      default: hipLaunchKernelGGL(gemm_fp8_block_join_kernel<LX2V_EPI_RESIDUAL>, grid, block, 0, st, p); break;
    }
  } else {
    switch (epilogue) {
      case LX2V_EPI_NONE: launch<LX2V_EPI_NONE>(p, q.kind, st); break;
      case LX2V_EPI_GELU_TANH: launch<LX2V_EPI_GELU_TANH>(p, q.kind, st); break;
      default: launch<LX2V_EPI_RESIDUAL>(p, q.kind, st); break;
    }
  }
  LX2V_CHECK_LAUNCH("gemm_fp8_block128");
  return LX2V_OK;
}
