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
// Two kernels.  `stream`: 4 waves (2 x 2), operand tiles of 128 bytes of K per row staged into LDS by LDS-DMA, four tile shapes,
// optionally split along K with a second launch (`join`) that adds the parts.  `skinny` (up to 32 rows): every wave streams its own
// weight rows straight into fragment registers, the waves split K.  Rows past M / N and columns past K arrive as zeros (range check of
// the buffer descriptors).
#include <algorithm>
#include <atomic>

#include "common.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int BK = 128;
constexpr int GROUP_M = 4;  // row panels that share one sweep over the columns
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
  uint32_t group_rcp;  // floor(2^32 / (GROUP_M * tiles_n))
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

// Raw buffer of `bytes` from `base`: an access is out of range, and loads 0, when its vector and scalar offsets together reach the extent
// (measured for plain loads and LDS-DMA: neither a scalar offset past the extent nor an extent of 0 makes the comparison wrap).
// An operand tile has at most 256 rows, each below 4 MiB: its extent is below 2^31 and computed in 32 bits.
LX2V_DEVICE u32x4 raw_descriptor(const void* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  u32x4 d;
  d[0] = __builtin_amdgcn_readfirstlane((uint32_t)a);
  d[1] = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));  // stride 0: raw buffer
  d[2] = __builtin_amdgcn_readfirstlane(bytes);  // loads at or past it return 0
  d[3] = 0x00020000u;
  return d;
}

LX2V_DEVICE f32x4 mfma_block(const i32x8& w, const i32x8& a) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);  // (zero scale operands: the form without block scales)
}

// GELU of N values: x * sigmoid(2u), u = sqrt(2/pi) (x + 0.044715 x^3), as x / (1 + 2^(x (c1 + c3 x^2))).  In stages over all N: a
// lone wave would wait behind every exp2 and reciprocal of its own (72 cycles a value one after the other, 56 staged; a tile of
// 192 x 256 holds 192 values a lane).
template <int N>
LX2V_DEVICE void gelu(float (&v)[N]) {
#pragma clang fp reassociate(off)
  constexpr float C1 = -2.f * 0.7978845608028654f * 1.4426950408889634f, C3 = C1 * 0.044715f;
  float e[N];
#pragma unroll
  for (int j = 0; j < N; ++j) e[j] = v[j] * __builtin_fmaf(v[j] * v[j], C3, C1);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < N; ++j) e[j] = __builtin_amdgcn_exp2f(e[j]);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < N; ++j) e[j] = __builtin_amdgcn_rcpf(1.0f + e[j]);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] *= e[j];
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
  if constexpr (EPI == LX2V_EPI_GELU_TANH) gelu(v);
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

// ---- stream kernel ------------------------------------------------------------------------------------
// One wave per SIMD, 4 waves (2 x 2), wave tile 16 MT x 16 NT (within one row block of weight scales), persistent: a workgroup
// walks its output tiles as one stream of K blocks.  Block j is multiplied while block j + 1 is read from LDS into the other
// set of fragment registers (so the LDS reads are spread over the whole block) and the blocks behind it are on their way into
// rings of SA A slots and SW W slots: once every wave has block j in registers, its slots take W(j + SW) with its scales and
// A(j + SA).  (192 x 256, at 75600 x 5120 x 13824 with the gated residual: 4.5 ms = 2.4 PFLOP/s.  The MFMAs are busy 69 % of the
// cycles at a clock that sinks to 1.6 GHz under them; two A slots instead of three: 5.0 ms; eight waves and one set of fragment
// registers: 10.3 ms.)
// LDS: a row's eight 16-byte chunks c lie at c ^ ((row >> 1) & 7).  A lane takes chunks fq and fq + 4 of its row as the two halves of a
// fragment instead of 2 fq and 2 fq + 1 -- any order of K that both operands share gives the same products -- because the LDS serves
// the lanes of a 16-byte read in eights out of two neighbouring quarters, and so all eight hit different banks (counter: no conflicts).
template <int MT_, int NT_, int SA_, int SW_>
struct Stream {
  static constexpr int MT = MT_, NT = NT_, SA = SA_, SW = SW_;
  static constexpr int TM = 32 * MT, TN = 32 * NT;
  static constexpr int A_BYTES = TM * BK, W_BYTES = TN * BK;
  static constexpr int W_AT = SA * A_BYTES, S_AT = W_AT + SW * W_BYTES;
  static constexpr int LDS = S_AT + SW * 1024;
  static_assert(LDS <= 160 * 1024 && SA >= SW && SW >= 2, "LDS of a CU; the order of the waits");
  static constexpr int PA = TM / 32, PW = TN / 32;  // DMA pieces of 1 KiB a wave
  static constexpr int PIECES = PW + 1 + PA;        // W(j + SW), its scales, A(j + SA)
  static constexpr int AHEAD = (SW - 2) * PIECES + (SA > SW ? PA : 0);  // pieces issued behind the last one of block j + 2, at the end of block j
  static constexpr int STEPS = MT * NT;
  static constexpr int RES = STEPS % 3 == 0 ? 3 : 4;  // ring of MFMA results
  static_assert(STEPS % RES == 0, "the ring of results wraps with the block");
  static constexpr int READS = 2 * NT + 3 * MT + 1;
};

// n / d and n % d from floor(2^32 / d): the estimate is the quotient or one less.
LX2V_DEVICE void divmod(uint32_t n, uint32_t d, uint32_t rcp, uint32_t& q, uint32_t& r) {
  q = __umulhi(n, rcp);
  r = n - q * d;
  if (r >= d) {
    ++q;
    r -= d;
  }
}

// Output tile -> its position: contiguous runs of tiles for each XCD, GROUP_M row panels sharing one sweep over the columns.
struct Raster {
  int tiles_m, tiles_n, per_xcd, extra;  // tiles / 8, tiles % 8
  uint32_t rcp;                          // of GROUP_M * tiles_n
};
LX2V_DEVICE void tile_origin(const Raster& g, int vbid, int tm, int tn, int& m0, int& n0) {
  const int xcd = vbid & 7;
  const uint32_t t = (uint32_t)(xcd * g.per_xcd + min(xcd, g.extra) + (vbid >> 3));
  uint32_t sweep, in_g, row, col;
  divmod(t, (uint32_t)(GROUP_M * g.tiles_n), g.rcp, sweep, in_g);
  const uint32_t gm = (uint32_t)min(g.tiles_m - (int)sweep * GROUP_M, GROUP_M);
  divmod(in_g, gm, gm == 4 ? 0x40000000u : gm == 3 ? 0x55555555u : gm == 2 ? 0x80000000u : 0xffffffffu, col, row);
  m0 = (int)(sweep * GROUP_M + row) * tm;
  n0 = (int)col * tn;
}

// The kernel's arguments, read again from memory: what a kernel needs once per output tile only would otherwise occupy scalar
// registers throughout its K loop.
typedef const __attribute__((address_space(4))) Params* ParamsAgain;
LX2V_DEVICE ParamsAgain params_again() {
  uint64_t a = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(a));
  return reinterpret_cast<ParamsAgain>(a);
}

// Accumulator registers a32 .. a255 hold the stream kernel's fragments by name (tools/check_mfma_hazards.py checks that the
// compiler keeps its hands off them).
#define FRAG_CLOBBERS \
  "a32", "a33", "a34", "a35", "a36", "a37", "a38", "a39", "a40", "a41", "a42", "a43", "a44", "a45", "a46", "a47", \
  "a48", "a49", "a50", "a51", "a52", "a53", "a54", "a55", "a56", "a57", "a58", "a59", "a60", "a61", "a62", "a63", \
  "a64", "a65", "a66", "a67", "a68", "a69", "a70", "a71", "a72", "a73", "a74", "a75", "a76", "a77", "a78", "a79", \
  "a80", "a81", "a82", "a83", "a84", "a85", "a86", "a87", "a88", "a89", "a90", "a91", "a92", "a93", "a94", "a95", \
  "a96", "a97", "a98", "a99", "a100", "a101", "a102", "a103", "a104", "a105", "a106", "a107", "a108", "a109", "a110", "a111", \
  "a112", "a113", "a114", "a115", "a116", "a117", "a118", "a119", "a120", "a121", "a122", "a123", "a124", "a125", "a126", "a127", \
  "a128", "a129", "a130", "a131", "a132", "a133", "a134", "a135", "a136", "a137", "a138", "a139", "a140", "a141", "a142", "a143", \
  "a144", "a145", "a146", "a147", "a148", "a149", "a150", "a151", "a152", "a153", "a154", "a155", "a156", "a157", "a158", "a159", \
  "a160", "a161", "a162", "a163", "a164", "a165", "a166", "a167", "a168", "a169", "a170", "a171", "a172", "a173", "a174", "a175", \
  "a176", "a177", "a178", "a179", "a180", "a181", "a182", "a183", "a184", "a185", "a186", "a187", "a188", "a189", "a190", "a191", \
  "a192", "a193", "a194", "a195", "a196", "a197", "a198", "a199", "a200", "a201", "a202", "a203", "a204", "a205", "a206", "a207", \
  "a208", "a209", "a210", "a211", "a212", "a213", "a214", "a215", "a216", "a217", "a218", "a219", "a220", "a221", "a222", "a223", \
  "a224", "a225", "a226", "a227", "a228", "a229", "a230", "a231", "a232", "a233", "a234", "a235", "a236", "a237", "a238", "a239", \
  "a240", "a241", "a242", "a243", "a244", "a245", "a246", "a247", "a248", "a249", "a250", "a251", "a252", "a253", "a254", "a255"

template <class T, int EPI>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void gemm_fp8_block_stream_kernel(const Params p) {
  constexpr int MT = T::MT, NT = T::NT;
  constexpr int STORES = EPI == EPI_PARTIAL ? MT * NT : MT * NT / 2;
  __shared__ __attribute__((aligned(16))) char lds[T::LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid >> 1, wn = wid & 1;
  const int fr = lane & 15, fq = lane >> 4;
  const int ntiles = p.tiles_m * p.tiles_n, grid = gridDim.x;
  // a workgroup's tiles are first, first + grid, ...; EPI_PARTIAL: one K range (blocks kb0 ..) of one tile
  int first = blockIdx.x, kb0 = 0, nk = p.nk, part_id = 0;
  if constexpr (EPI == EPI_PARTIAL) {
    part_id = first / ntiles;
    first -= part_id * ntiles;
    kb0 = part_id * p.per;
    nk = min(p.per, nk - kb0);
  }
  const int my_tiles = first < ntiles ? (ntiles - 1 - first) / grid + 1 : 0;
  const int64_t total = (int64_t)my_tiles * nk;
  if (total == 0) return;

  const Raster raster{p.tiles_m, p.tiles_n, ntiles >> 3, ntiles & 7, p.group_rcp};
  const uint32_t lds_base = __builtin_amdgcn_readfirstlane((uint32_t)(size_t)(__attribute__((address_space(3))) char*)lds);
  constexpr int NOWHERE = (int)0x80000000u;
  const bool sw_wave = wid == 3;  // (waves 0 - 2: 64 rows' scales each; past the tile's rows they read zeros)

  // ---- DMA cursors: W and its scales SW blocks ahead of the multiplied one, A SA blocks ----
  // piece q of wave w: rows 32 q + 8 w + (lane >> 3) of the operand tile; the swizzle is the same for all q
  const int chunk = (lane & 7) ^ ((4 * wid + (lane >> 4)) & 7);
  const int left = p.K - (p.nk - 1) * BK;  // columns of the last block
  const uint32_t last = (uint32_t)(kb0 + nk - 1) * BK;  // offset in a row of the tile's last block ...
  const uint32_t ragged = left < BK && kb0 + nk == p.nk ? last : ~0u;  // ... and of its last block if that is short
  int a_pv, w_pv, s_pv = NOWHERE;
  auto offset = [&](int64_t ld, bool last) __attribute__((always_inline)) -> int {  // of piece 0; `last`: chunks past K go nowhere
    int at = (8 * wid + (lane >> 3)) * (int)ld + chunk * 16;
    asm volatile("" : "+v"(at));  // (a branch around it would make the scalars that meet behind it vector registers)
    return last & (chunk * 16 >= left) ? NOWHERE : at;
  };
  struct Cursor {
    int ord = 0;
    uint32_t soff = 0, step = BK;  // the block's offset in a row (past the last tile it stays 0: an empty descriptor has no scalar offset either)
  } ca, cw;
  u32x4 a_rs, w_rs;
  uint64_t s_base = 0, s_step = 0;  // the scales' descriptor: its base moves on by a block's scales, its extent stays
  uint32_t s_bytes = 0;
  // (the fields are read together: one wait for memory per tile and operand, not one for each field on its first use)
  auto a_tile = [&]() __attribute__((always_inline)) {  // descriptor of the cursor's output tile; past the last one it is empty
    const ParamsAgain p = params_again();
    const uint64_t base = reinterpret_cast<uint64_t>(p->A);
    const int64_t lda = p->lda;
    const int M = p->M;
    asm volatile("" ::"s"(base), "s"(lda), "s"(M));
    const int vbid = ca.ord * grid + first;
    int m0, n0;
    tile_origin(raster, vbid, T::TM, T::TN, m0, n0);
    const int rows = vbid < ntiles ? min(M - m0, T::TM) : 0;
    a_rs = raw_descriptor(reinterpret_cast<const uint8_t*>(base) + (int64_t)(rows ? m0 : 0) * lda, (uint32_t)rows * (uint32_t)lda);
    ca.step = rows ? BK : 0;
    asm volatile("" : "+s"(a_rs), "+s"(ca.step));
  };
  auto w_tile = [&]() __attribute__((always_inline)) {
    const ParamsAgain p = params_again();
    const uint64_t base = reinterpret_cast<uint64_t>(p->W), asb = reinterpret_cast<uint64_t>(p->a_scale), wsb = reinterpret_cast<uint64_t>(p->w_scale);
    const int64_t ldw = p->ldw, lds_w = p->lds_w, lds_a = p->lds_a;
    const int M = p->M, N = p->N;
    asm volatile("" ::"s"(base), "s"(asb), "s"(wsb), "s"(ldw), "s"(lds_w), "s"(lds_a), "s"(M), "s"(N));
    const int vbid = cw.ord * grid + first;
    const bool live = vbid < ntiles;
    int m0, n0;
    tile_origin(raster, vbid, T::TM, T::TN, m0, n0);
    if (!live) m0 = n0 = 0;
    const int rows = live ? min(N - n0, T::TN) : 0;
    w_rs = raw_descriptor(reinterpret_cast<const uint8_t*>(base) + (int64_t)n0 * ldw, (uint32_t)rows * (uint32_t)ldw);
    const int nb = min(((N + 127) >> 7) - (n0 >> 7), (T::TN + 127) / 128);  // weight row blocks of the tile
    const float* sb = sw_wave ? reinterpret_cast<const float*>(wsb) + (int64_t)(n0 >> 7) * lds_w + kb0 : reinterpret_cast<const float*>(asb) + (int64_t)kb0 * lds_a + m0;
    cw.step = live ? BK : 0;
    s_base = reinterpret_cast<uint64_t>(sb);
    s_bytes = !live ? 0u : sw_wave ? ((uint32_t)(nb - 1) * (uint32_t)lds_w + 1) * 4 : (uint32_t)min(M - m0, T::TM) * 4;
    asm volatile("" : "+s"(w_rs), "+s"(s_base), "+s"(s_bytes), "+s"(cw.step));
    s_pv = sw_wave ? (lane < nb ? lane * (int)lds_w * 4 : NOWHERE) : (64 * wid + lane) * 4;
  };
  a_tile();
  w_tile();
  a_pv = offset(p.lda, nk == 1 && ragged == last);
  w_pv = offset(p.ldw, nk == 1 && ragged == last);
  ca.soff = cw.soff = (uint32_t)kb0 * BK;
  {
    const int64_t step = sw_wave ? 4 : p.lds_a * 4;
    s_step = ((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)step >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)step);
  }
  uint32_t dma_base = lds_base + 1024 * (uint32_t)wid, dma_sc;
  asm volatile("" : "+s"(dma_base));
  dma_sc = lds_base + ((dma_base - lds_base) >> 2);
  asm volatile("" : "+s"(dma_sc));
  auto set_m0 = [&](uint32_t base, auto ofsc) __attribute__((always_inline)) { asm volatile("s_add_u32 m0, %0, %1" ::"s"(base), "i"(decltype(ofsc)::value) : "memory", "scc"); };
  auto load16 = [&](const u32x4& rs, int voff, uint32_t soff) __attribute__((always_inline)) {
    asm volatile("buffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(rs), "s"(soff) : "memory");
  };
  auto load4 = [&]() __attribute__((always_inline)) {  // (the descriptor is put together here: as a vector that lives on, the compiler moves it into vector registers)
    asm volatile("s_mov_b64 s[96:97], %1\n\ts_mov_b32 s98, %2\n\ts_mov_b32 s99, 0x20000\n\tbuffer_load_dword %0, s[96:99], 0 offen lds"
                 ::"v"(s_pv), "s"(s_base), "s"(s_bytes) : "memory", "s96", "s97", "s98", "s99");
  };
  // Ring positions: of block j, which the DMA refills, and of block j + 1, which is read.  (Two W slots: W and the scales of block j
  // lie at the parity P of j, known at compile time.)
  uint32_t a_cur = dma_base, a_nxt = dma_base + T::A_BYTES, w_cur = dma_base, w_nxt = dma_base + T::W_BYTES, s_cur = dma_sc, s_nxt = dma_sc + 1024;
  asm volatile("" : "+s"(a_cur), "+s"(a_nxt), "+s"(w_cur), "+s"(w_nxt), "+s"(s_cur), "+s"(s_nxt));
  constexpr bool TWO = T::SW == 2;
  // piece q of a block's DMA, its target and then the load itself: W(j + SW), its scales, A(j + SA)
  auto dma_set = [&](auto Pc, auto qc) __attribute__((always_inline)) {
    constexpr int P = decltype(Pc)::value, q = decltype(qc)::value;
    if constexpr (q < T::PW) set_m0(TWO ? dma_base : w_cur, IntC<T::W_AT + (TWO ? P * T::W_BYTES : 0) + 4096 * q>{});
    else if constexpr (q == T::PW) set_m0(TWO ? dma_sc : s_cur, IntC<T::S_AT + (TWO ? P * 1024 : 0)>{});
    else set_m0(a_cur, IntC<4096 * (q - T::PW - 1)>{});
  };
  const int a_step = 32 * (int)p.lda, w_step = 32 * (int)p.ldw;
  int d_voff = 0;
  auto dma_go = [&](auto qc) __attribute__((always_inline)) {
    constexpr int q = decltype(qc)::value;
    if constexpr (q == 0) d_voff = w_pv;
    if constexpr (q < T::PW) {
      load16(w_rs, d_voff, cw.soff);
      if constexpr (q + 1 < T::PW) d_voff += w_step;
    } else if constexpr (q == T::PW) {
      load4();
    } else {
      if constexpr (q == T::PW + 1) d_voff = a_pv;
      load16(a_rs, d_voff, ca.soff);
      if constexpr (q + 1 < T::PIECES) d_voff += a_step;
    }
    asm volatile("" : "+v"(d_voff));
  };
  // Cursors and rings move on by a block: four pieces of a few scalar instructions, W's (0 - 2) once its DMA of the block is issued,
  // then A's; what the end of a tile needs besides follows in w_turn and a_turn.
  constexpr int MOVES = 4;
  auto move = [&](auto ic) __attribute__((always_inline)) {
    constexpr int i = decltype(ic)::value;
    if constexpr (i == 0) {
      cw.soff += cw.step;
      s_base += s_step;
      asm volatile("" : "+s"(cw.soff), "+s"(s_base));
    } else if constexpr (i == 1 && !TWO) {
      w_cur = w_nxt;
      w_nxt = w_nxt == dma_base + (T::SW - 1) * T::W_BYTES ? dma_base : w_nxt + T::W_BYTES;
      asm volatile("" : "+s"(w_cur), "+s"(w_nxt));
    } else if constexpr (i == 2 && !TWO) {
      s_cur = s_nxt;
      s_nxt = s_nxt == dma_sc + (T::SW - 1) * 1024 ? dma_sc : s_nxt + 1024;
      asm volatile("" : "+s"(s_cur), "+s"(s_nxt));
    } else if constexpr (i == 3) {
      ca.soff += ca.step;
      a_cur = a_nxt;
      a_nxt = a_nxt == dma_base + (T::SA - 1) * T::A_BYTES ? dma_base : a_nxt + T::A_BYTES;
      asm volatile("" : "+s"(ca.soff), "+s"(a_cur), "+s"(a_nxt));
    }
  };
  auto w_turn = [&]() __attribute__((always_inline)) {
    if (cw.soff == ragged) w_pv = offset(params_again()->ldw, true);
    if (cw.soff == last + BK) {
      cw.soff = 0;
      ++cw.ord;
      w_tile();
      if (ragged == last) w_pv = offset(params_again()->ldw, nk == 1);
    }
    asm volatile("" : "+s"(w_rs), "+s"(s_base), "+s"(s_bytes), "+s"(cw.soff), "+s"(cw.step), "+s"(cw.ord), "+s"(dma_base), "+s"(dma_sc));
  };
  auto a_turn = [&]() __attribute__((always_inline)) {
    if (ca.soff == ragged) a_pv = offset(params_again()->lda, true);
    if (ca.soff == last + BK) {
      ca.soff = 0;
      ++ca.ord;
      a_tile();
      if (ragged == last) a_pv = offset(params_again()->lda, nk == 1);
    }
    asm volatile("" : "+s"(a_rs), "+s"(ca.soff), "+s"(ca.step), "+s"(ca.ord), "+s"(a_cur), "+s"(a_nxt));
  };

  // ---- fragments: register set P (0 | 1) = NT W fragments, then MT A fragments, of 8 accumulator registers each ----
  int rd_a[2], rd_w[2];  // LDS addresses of the lane's two 16-byte halves at row block 0 of slot 0 (less this wave's share of a DMA target)
  {
    const int ar = wm * 16 * MT + fr, wr = wn * 16 * NT + fr;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      rd_a[c] = ar * BK + (((fq + 4 * c) ^ ((ar >> 1) & 7)) << 4) - 1024 * wid;
      rd_w[c] = (TWO ? (int)lds_base : -1024 * wid) + T::W_AT + wr * BK + (((fq + 4 * c) ^ ((wr >> 1) & 7)) << 4);
    }
  }
  const int rd_s = T::S_AT + (wm * 16 * MT + fr) * 4, rd_sw = T::S_AT + 768 + ((wn * 16 * NT) >> 7) * 4;
  int at_a[2], at_w[2], at_s = 0;  // where block j + 1 is read (at_s: the offset of its scales' slot)
  auto set_reads = [&](uint32_t a_at, uint32_t w_at, uint32_t s_at) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      at_a[c] = rd_a[c] + (int)a_at;
      at_w[c] = TWO ? rd_w[c] : rd_w[c] + (int)w_at;
    }
    if constexpr (!TWO) at_s = (int)(s_at - dma_sc);
  };
  constexpr int SET = 8 * (NT + MT), FRAG0 = 256 - 2 * SET;
  static_assert(FRAG0 >= 32, "fragments exceed the accumulator registers");
  float sa[MT], sw, s[MT], s_last;
  f32x4 acc[MT][NT];
  f32x4 part[T::RES];
  // `old`, the result of the MFMA two before: handed through the statement, so that its additions stay behind this one --
  // 64 cycles at least after the instruction that made it, which the compiler, not knowing what it is, would not wait for
  auto mm = [&](f32x4& d, f32x4& old, auto wc, auto ac) __attribute__((always_inline)) {
    asm volatile("v_mfma_f32_16x16x128_f8f6f4 %0, a[%2:%3], a[%4:%5], 0"
                 : "=&v"(d), "+v"(old) : "n"(decltype(wc)::value), "n"(decltype(wc)::value + 7), "n"(decltype(ac)::value), "n"(decltype(ac)::value + 7));
  };
  auto add = [&](auto tc, float sc, auto FIRSTc) __attribute__((always_inline)) {  // FIRST: the output tile's first block sets the sums
    constexpr int t = decltype(tc)::value;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[t / NT][t % NT][e] = decltype(FIRSTc)::value ? part[t % T::RES][e] * sc : __builtin_fmaf(part[t % T::RES][e], sc, acc[t / NT][t % NT][e]);
    asm volatile("" : "+v"(acc[t / NT][t % NT]));  // (pinned here: without a use the sums would sink to the end of the block and keep every result alive)
  };
  auto lds_frag = [&](int addr, auto dstc, auto ofsc) __attribute__((always_inline)) {  // 16 bytes a lane into four accumulator registers; waited for at the next barrier
    asm volatile("ds_read_b128 a[%1:%2], %0 offset:%3" ::"v"(addr), "n"(decltype(dstc)::value), "n"(decltype(dstc)::value + 3), "n"(decltype(ofsc)::value) : "memory", FRAG_CLOBBERS);
  };
  // LDS read r of a block into register set P: 2 NT halves of W, 2 MT of A, MT + 1 scales
  auto rd = [&](auto Pc, auto rc) __attribute__((always_inline)) {
    constexpr int P = decltype(Pc)::value, r = decltype(rc)::value;
    if constexpr (r < 2 * NT) lds_frag(at_w[r & 1], IntC<FRAG0 + P * SET + 4 * r>{}, IntC<(TWO ? P * T::W_BYTES : 0) + (r >> 1) * 2048>{});
    else if constexpr (r < 2 * NT + 2 * MT) lds_frag(at_a[r & 1], IntC<FRAG0 + P * SET + 4 * r>{}, IntC<((r - 2 * NT) >> 1) * 2048>{});
    else if constexpr (r < 2 * NT + 3 * MT) sa[r - 2 * NT - 2 * MT] = *reinterpret_cast<const float*>(lds + (TWO ? P * 1024 : at_s) + rd_s + (r - 2 * NT - 2 * MT) * 64);
    else if constexpr (r == 2 * NT + 3 * MT) sw = *reinterpret_cast<const float*>(lds + (TWO ? P * 1024 : at_s) + rd_sw);
  };

  // One block: multiply register set P, read the next one's fragments into set 1 - P, stage into the slots of this one.
  auto block = [&](auto Pc, auto FIRSTc, bool relaxed) __attribute__((always_inline)) {
    constexpr int P = decltype(Pc)::value, Q = 1 - P;
    // the next block is complete in LDS once every wave is past this barrier, and every wave has read its fragments of this one
    // (what was issued behind the next block's last pieces may still be on its way: the pieces of the block after it, an epilogue's stores)
    if (relaxed) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(T::AHEAD + STORES) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(T::AHEAD) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    set_reads(a_nxt, w_nxt, s_nxt);
    s_last = s[MT - 1];
#pragma unroll
    for (int i = 0; i < MT; ++i) s[i] = sa[i] * sw;
    static_for<0, T::STEPS>([&](auto tc) __attribute__((always_inline)) {
      constexpr int t = decltype(tc)::value;
      mm(part[t % T::RES], part[(t + T::RES - 2) % T::RES], IntC<FRAG0 + P * SET + 8 * (t % NT)>{}, IntC<FRAG0 + P * SET + 8 * NT + 8 * (t / NT)>{});
      if constexpr (2 * T::PIECES <= T::STEPS) {
        // Behind the MFMA its shadow of 32 cycles is filled with the four additions (16) and at most three more instructions: a
        // piece's target with two LDS reads in an even step, its load in the next one; the reads left follow, two a step, early
        // enough to be complete at the block's end.
        if constexpr (t < 2 * T::PIECES) {
          if constexpr (t % 2 == 0) dma_set(IntC<P>{}, IntC<t / 2>{});
          else dma_go(IntC<t / 2>{});
        }
        if constexpr (t % 2 == 0 || t >= 2 * T::PIECES) {
          constexpr int r = t < 2 * T::PIECES ? t : 2 * t - 2 * T::PIECES;
          static_for<r, r + 2>([&](auto rc) __attribute__((always_inline)) { rd(IntC<Q>{}, rc); });
        }
      } else {  // few MFMAs: pieces spread over the steps, reads over the first three quarters of them
        constexpr int D = T::STEPS - 1, q0 = t * T::PIECES / D, q1 = (t + 1) * T::PIECES / D;  // (none in the last step: A moves on there)
        static_for<(q0 < T::PIECES ? q0 : T::PIECES), (q1 < T::PIECES ? q1 : T::PIECES)>([&](auto qc) __attribute__((always_inline)) {
          dma_set(IntC<P>{}, qc);
          asm volatile("s_nop 0");
          dma_go(qc);
        });
        constexpr int E = T::STEPS * 3 / 4, r0 = t * T::READS / E, r1 = (t + 1) * T::READS / E;
        static_for<(r0 < T::READS ? r0 : T::READS), (r1 < T::READS ? r1 : T::READS)>([&](auto rc) __attribute__((always_inline)) { rd(IntC<Q>{}, rc); });
      }
      if constexpr (T::STEPS == 8) {
        if constexpr (t >= 5) static_for<t - 5, (t == 7 ? MOVES : t - 4)>(move);
      } else if constexpr (t >= T::STEPS - MOVES) {
        move(IntC<t - (T::STEPS - MOVES)>{});
      }
      __builtin_amdgcn_sched_barrier(0);
      constexpr int last = T::STEPS - 2 + t;
      if constexpr (t >= 2) add(IntC<t - 2>{}, s[(t - 2) / NT], FIRSTc);
      else if constexpr (decltype(FIRSTc)::value) acc[last / NT][last % NT] = f32x4{0.f, 0.f, 0.f, 0.f};
      else add(IntC<last>{}, s_last, FIRSTc);  // the previous block's last two
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  // ---- epilogue: a lane's four columns become eight consecutive ones by swapping lane rows between two column blocks;
  // 16-byte stores through a descriptor of the tile's rows: rows past M and columns past N are dropped ----
  auto epilogue = [&](int m0, int n0) __attribute__((always_inline)) {
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(part[(T::STEPS - 2) % T::RES]), "+v"(part[(T::STEPS - 1) % T::RES]));  // the last MFMAs were issued a few cycles ago
    add(IntC<T::STEPS - 2>{}, s[MT - 1], IntC<0>{});
    add(IntC<T::STEPS - 1>{}, s[MT - 1], IntC<0>{});
    const ParamsAgain p = params_again();
    const uint64_t c_at = reinterpret_cast<uint64_t>(p->C), bias_at = reinterpret_cast<uint64_t>(p->bias), gate_at = reinterpret_cast<uint64_t>(p->gate), resid_at = reinterpret_cast<uint64_t>(p->resid);
    const int64_t ldc = p->ldc, ldr = p->ldr;
    const int M = p->M, N = p->N;
    asm volatile("" ::"s"(c_at), "s"(bias_at), "s"(gate_at), "s"(resid_at), "s"(ldc), "s"(ldr), "s"(M), "s"(N));
    int fr_ = fr, fq_ = fq;
    asm volatile("" : "+v"(fr_), "+v"(fq_));
    if constexpr (EPI == EPI_PARTIAL) {
      const u32x4 d = raw_descriptor(p->partials + ((int64_t)part_id * M + m0) * N, (uint32_t)min(M - m0, T::TM) * (uint32_t)N * 4);
      const auto o_rs = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)d[1] << 32) | d[0]), 0, (int)d[2], 0x00020000);
      static_for<0, MT * NT>([&](auto uc) __attribute__((always_inline)) {
        constexpr int i = decltype(uc)::value / NT, k = decltype(uc)::value % NT;
        const int row = wm * 16 * MT + i * 16 + fr_, n = n0 + wn * 16 * NT + k * 16 + fq_ * 4;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[i][k]), o_rs, m0 + row < M && n < N ? (row * N + n) * 4 : NOWHERE, 0, 0);
      });
      return;
    }
    auto resource = [](uint64_t at, uint32_t bytes) __attribute__((always_inline)) {  // accesses past the end: loads give 0, stores are dropped
      const u32x4 d = raw_descriptor(reinterpret_cast<const void*>(at), bytes);
      return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(((uint64_t)d[1] << 32) | d[0]), 0, (int)d[2], 0x00020000);
    };
    const uint32_t rows = (uint32_t)min(M - m0, T::TM);
    const auto c_rs = resource(c_at + (int64_t)m0 * ldc * 2, ((rows - 1) * (uint32_t)ldc + (uint32_t)N) * 2);
    const auto r_rs = resource(resid_at + (int64_t)m0 * ldr * 2, EPI == LX2V_EPI_RESIDUAL ? ((rows - 1) * (uint32_t)ldr + (uint32_t)N) * 2 : 0);
    const auto b_rs = resource(bias_at, bias_at ? (uint32_t)N * 4 : 0), g_rs = resource(gate_at, EPI == LX2V_EPI_RESIDUAL && gate_at ? (uint32_t)N * 4 : 0);
    // step u = column block pair u / MT, row block u % MT.  Bias and gate are loaded one pair ahead, residual rows RV steps ahead.
    // (the residual form has registers for one pair's bias and gate only)
    constexpr int U = MT * NT / 2, RV = MT, CV = EPI == LX2V_EPI_RESIDUAL ? 1 : 2;
    const int col0 = n0 + wn * 16 * NT + fq_ * 4;
    f32x4 bv[CV][2], gv[CV][2];
    u32x2 rv[RV][2];
    auto fetch_cols = [&](auto kc) __attribute__((always_inline)) {
      constexpr int k2 = decltype(kc)::value;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = (col0 + (2 * k2 + h) * 16) * 4;
        bv[k2 % CV][h] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(b_rs, at, 0, 0));
        if constexpr (EPI == LX2V_EPI_RESIDUAL) {
          gv[k2 % CV][h] = f32x4{1.f, 1.f, 1.f, 1.f};
          if (gate_at != 0) gv[k2 % CV][h] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(g_rs, at, 0, 0));
        }
      }
    };
    auto fetch_rows = [&](auto uc) __attribute__((always_inline)) {
      constexpr int u = decltype(uc)::value;
      if constexpr (EPI == LX2V_EPI_RESIDUAL && u < U) {
        const int at = ((wm * 16 * MT + (u % MT) * 16 + fr_) * (int)ldr + col0 + 2 * (u / MT) * 16) * 2;
#pragma unroll
        for (int h = 0; h < 2; ++h) rv[u % RV][h] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r_rs, at + 32 * h, 0, 0));
      }
    };
    auto store = [&](auto uc, const u32x4& v) __attribute__((always_inline)) {
      constexpr int u = decltype(uc)::value;
      const int row = wm * 16 * MT + (u % MT) * 16 + fr_, n = n0 + wn * 16 * NT + (2 * (u / MT) + (fq_ & 1)) * 16 + (fq_ >> 1) * 8;
      __builtin_amdgcn_raw_buffer_store_b128(v, c_rs, m0 + row < M && n < N ? (row * (int)ldc + n) * 2 : NOWHERE, 0, 0);
    };
    fetch_cols(IntC<0>{});
    static_for<0, RV>([&](auto uc) __attribute__((always_inline)) { fetch_rows(uc); });
    static_for<0, U>([&](auto uc) __attribute__((always_inline)) {
      constexpr int u = decltype(uc)::value, i = u % MT, k2 = u / MT, b = k2 % CV;
      if constexpr (EPI != LX2V_EPI_RESIDUAL && i == 0 && k2 < NT / 2 - 1) fetch_cols(IntC<k2 + 1>{});
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = acc[i][2 * k2 + (e >> 2)][e & 3] + bv[b][e >> 2][e & 3];
      if constexpr (EPI == LX2V_EPI_GELU_TANH) gelu(x);
      uint32_t d[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float* v = x + 4 * h;
        if constexpr (EPI == LX2V_EPI_RESIDUAL) {
          const u32x2 r = rv[u % RV][h];
          v[0] = v[0] * gv[b][h][0] + __uint_as_float(r[0] << 16);
          v[1] = v[1] * gv[b][h][1] + __uint_as_float(r[0] & 0xffff0000u);
          v[2] = v[2] * gv[b][h][2] + __uint_as_float(r[1] << 16);
          v[3] = v[3] * gv[b][h][3] + __uint_as_float(r[1] & 0xffff0000u);
        }
        d[h][0] = pack2(v[0], v[1]);
        d[h][1] = pack2(v[2], v[3]);
      }
      // lane rows fq = 0 .. 3 of block k: columns 4 fq ..; swapping the odd rows of d[0] with the even rows of d[1] leaves row 0
      // with columns 0-7 of block k, row 1 with 0-7 of block k + 1, row 2 with 8-15 of block k, row 3 with 8-15 of block k + 1
      const auto lo = __builtin_amdgcn_permlane16_swap(d[0][0], d[1][0], false, false);
      const auto hi = __builtin_amdgcn_permlane16_swap(d[0][1], d[1][1], false, false);
      const u32x4 out = {lo[0], hi[0], lo[1], hi[1]};
      if constexpr (EPI != LX2V_EPI_RESIDUAL) {
        store(uc, out);
      } else {
        // Memory operations retire in order: a residual load behind a store would wait for its write.  So the results stay, in
        // registers of sums that are done with, until all rows are loaded.
        acc[i][2 * k2] = __builtin_bit_cast(f32x4, out);
        asm volatile("" : "+v"(acc[i][2 * k2]));
        fetch_rows(IntC<u + RV>{});
        if constexpr (i == MT - 1 && k2 < NT / 2 - 1) fetch_cols(IntC<k2 + 1>{});
        if constexpr (u == U - 1) static_for<0, U>([&](auto vc) __attribute__((always_inline)) { store(vc, __builtin_bit_cast(u32x4, acc[decltype(vc)::value % MT][2 * (decltype(vc)::value / MT)])); });
      }
      asm volatile("" ::: FRAG_CLOBBERS);  // (the next block's fragments are in there: nothing of the epilogue may stay in them)
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  // ---- prologue: the first SW W tiles and their scales, the first SA A tiles, then the fragments of block 0 ----
  static_for<0, T::SA>([&](auto bc) __attribute__((always_inline)) {
    constexpr int b = decltype(bc)::value;
    static_for<(b < T::SW ? 0 : T::PW + 1), T::PIECES>([&](auto qc) __attribute__((always_inline)) {
      dma_set(IntC<b & 1>{}, qc);
      asm volatile("s_nop 0");
      dma_go(qc);
    });
    static_for<(b < T::SW ? 0 : 3), MOVES>(move);
    if constexpr (b < T::SW) w_turn();
    a_turn();
  });
  // (the rings are back at slot 0: block 0's)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  set_reads(a_cur, w_cur, s_cur);
  static_for<0, T::READS>([&](auto rc) __attribute__((always_inline)) { rd(IntC<0>{}, rc); });

  int ord = 0, kt = 0;
  bool relaxed = false;
  auto step = [&](auto Pc) __attribute__((always_inline)) {
    if (kt == 0) block(Pc, IntC<1>{}, relaxed);
    else block(Pc, IntC<0>{}, false);
    if (max(cw.soff, ca.soff) >= last) {
      w_turn();
      a_turn();
    }
    relaxed = false;
    if (++kt == nk) {
      int m0, n0;
      tile_origin(raster, ord * grid + first, T::TM, T::TN, m0, n0);
      epilogue(m0, n0);
      relaxed = true;
      kt = 0;
      ++ord;
    }
  };
  for (int64_t j = 0; j < total; j += 2) {
    step(IntC<0>{});
    if (j + 1 < total) step(IntC<1>{});
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA may still be writing this workgroup's LDS when it ends
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

// ---- skinny kernel: M <= 16 MT --------------------------------------------------------------------------
// The weight is read once and the time goes with its bytes, so it goes straight from memory into fragment registers.  Workgroup =
// 8 waves on 16 NT columns; wave w takes the K blocks w, w + 8, ..., U of them at a time: all their loads are issued before the
// first product.  (U = 2 or 4, 8 or 16 waves and non-temporal weight loads measure alike.)  A weight row's 128 bytes of a block are one
// cache line, read by one wave.  The waves' sums meet in LDS and are added in a fixed order.  1 x 30720 x 5120 takes 31 us, 157 MB at
// 5.1 TB/s.
constexpr int SKINNY_WAVES = 8;
template <int MT, int NT, int U, int EPI>
__global__ __launch_bounds__(64 * SKINNY_WAVES) void gemm_fp8_block_skinny_kernel(const Params p) {
  __shared__ __attribute__((aligned(16))) f32x4 red[SKINNY_WAVES][MT * NT][64];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fq = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT;  // (16 NT <= 128 columns inside one row block of weight scales)
  const uint8_t* wrow[NT];
  const uint8_t* arow[MT];
  const float* asp[MT];
#pragma unroll
  for (int k = 0; k < NT; ++k) wrow[k] = p.W + (int64_t)min(n0 + k * 16 + fr, p.N - 1) * p.ldw + fq * 32;
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int m = min(i * 16 + fr, p.M - 1);
    arow[i] = p.A + (int64_t)m * p.lda + fq * 32;
    asp[i] = p.a_scale + m;
  }
  const float* swp = p.w_scale + (int64_t)(n0 >> 7) * p.lds_w;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int k = 0; k < NT; ++k) acc[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Frag {
    i32x4 lo, hi;
  };
  const int k_lane = p.K - fq * 32;  // K % 16 == 0: 16 bytes of a row are inside it or outside it together
  auto load = [&](const uint8_t* row, int kb) __attribute__((always_inline)) -> Frag {
    Frag f = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    const i32x4* at = reinterpret_cast<const i32x4*>(row + (int64_t)kb * BK);
    if (kb * BK < k_lane) f.lo = at[0];
    if (kb * BK + 16 < k_lane) f.hi = at[1];
    return f;
  };
  auto blocks = [&](auto full, int kb) __attribute__((always_inline)) {
    Frag wf[U][NT], af[U][MT];
    float sc[U][MT], sw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = kb + SKINNY_WAVES * u;
      const bool in = decltype(full)::value || b < p.nk;
#pragma unroll
      for (int k = 0; k < NT; ++k) wf[u][k] = in ? load(wrow[k], b) : Frag{{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        af[u][i] = in ? load(arow[i], b) : Frag{{0, 0, 0, 0}, {0, 0, 0, 0}};
        sc[u][i] = in ? asp[i][(int64_t)b * p.lds_a] : 0.f;
      }
      sw[u] = in ? swp[b] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float s = sc[u][i] * sw[u];
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          const f32x4 d = mfma_block(__builtin_shufflevector(wf[u][k].lo, wf[u][k].hi, 0, 1, 2, 3, 4, 5, 6, 7), __builtin_shufflevector(af[u][i].lo, af[u][i].hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][k][e] = __builtin_fmaf(d[e], s, acc[i][k][e]);
        }
      }
  };
  int kb = wid;
  for (; kb + SKINNY_WAVES * (U - 1) < p.nk; kb += SKINNY_WAVES * U) blocks(IntC<1>{}, kb);
  if (kb < p.nk) blocks(IntC<0>{}, kb);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int k = 0; k < NT; ++k) red[wid][i * NT + k][lane] = acc[i][k];
  __syncthreads();
  if (wid < MT * NT) {
    f32x4 v = red[0][wid][lane];
#pragma unroll
    for (int w = 1; w < SKINNY_WAVES; ++w) v += red[w][wid][lane];
    const int m = wid / NT * 16 + fr, n = n0 + wid % NT * 16 + fq * 4;
    if (m < p.M && n < p.N) finish4<EPI>(p, v, m, n);
  }
}

int device_cus() {
  static std::atomic<int> cached[64];  // (calls from several threads at once may all ask: they store the same number)
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int cus = cached[dev].load(std::memory_order_relaxed);
  if (cus == 0) {
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) cus = 256;
    cached[dev].store(cus, std::memory_order_relaxed);
  }
  return cus;
}

enum Kind { SKINNY_16, SKINNY_32, TILE_64x128, TILE_128x128, TILE_128x256, TILE_192x256 };
struct Plan {
  Kind kind;
  int tm, tn, split, per;
  int64_t bytes;
};

// Up to 32 rows the skinny kernel (13 x 5120 x 4096: 9.4 us, the 64 x 128 tile split four ways 12.6; 32 x 5120 x 5120: 12.4 and 14.5;
// at 64 rows its reads of A cost more than they save, 17.4 and 15.2).  Above, the kernel and split whose estimated time is least.
// A tile kernel's time is rounds of tiles, each of K blocks and an overhead (pipeline fill, epilogue, tile switch); measured with
// one tile on nearly every CU, K = 2560 and 10240 (the estimate of a long run of tiles is too large: 551 us at 32760 x 8960 x 1536 + GELU,
// which takes 497; the estimates are only compared with each other):
//   tile        us per K block   us per tile
//   192 x 256        1.08            10          (one wave's 48 MFMAs are 0.64 us at 2.4 GHz; the CU's LDS moves 168 KB meanwhile)
//   128 x 256        0.84             8
//   128 x 128        0.55             5
//   64 x 128         0.41             3
// A split along K adds a launch that reads the partial sums back: 5 us and their bytes, written and read, at 4 TB/s.
// (Calls in a row on the same operands, weights from the memory-side cache; 512 x 10240 x 5120 takes 46 us with all of them from memory.
// 512 x 10240 x 5120: 128 x 256 whole 35.7 us, 192 x 256 44.9, 128 x 128 47.6; 2500 x 1536 x 8960: 128 x 128 whole 43.1,
// 128 x 256 in two parts 46.4; 64 x 5120 x 5120: 64 x 128 in four parts 15.2, whole 20.2; 200 x 5120 x 13824: in three 29.5, 43.9.)
Plan make_plan(int64_t M, int64_t N, int64_t K, int cus) {
  const int nk = (int)((K + BK - 1) / BK);
  if (M <= 16) return Plan{SKINNY_16, 16, 16, 1, nk, 0};
  if (M <= 32) return Plan{SKINNY_32, 32, 32, 1, nk, 0};
  static const struct {
    Kind kind;
    int tm, tn;
    float block, tile;
  } kinds[] = {{TILE_192x256, 192, 256, 1.08f, 10.f}, {TILE_128x256, 128, 256, 0.84f, 8.f}, {TILE_128x128, 128, 128, 0.55f, 5.f}, {TILE_64x128, 64, 128, 0.41f, 3.f}};
  Plan best{TILE_192x256, 192, 256, 1, nk, 0};
  float least = 1e30f;
  for (const auto& k : kinds) {
    const int64_t tiles = ((M + k.tm - 1) / k.tm) * ((N + k.tn - 1) / k.tn);
    for (int want = 1; want <= 16 && (want == 1 || tiles * want <= cus); ++want) {
      const int per = (nk + want - 1) / want, split = (nk + per - 1) / per;
      if (split != want) continue;
      float t = (float)((tiles * split + cus - 1) / cus) * ((float)per * k.block + k.tile);
      const int64_t bytes = split > 1 ? (int64_t)split * M * N * 4 : 0;
      if (split > 1) t += 5.f + (float)bytes * 2e-6f / 4.f;
      if (t < least) {
        least = t;
        best = Plan{k.kind, k.tm, k.tn, split, per, bytes};
      }
    }
  }
  return best;
}

template <int MT, int NT, int U, int EPI>
void launch_skinny(const Params& p, hipStream_t st) {
  if constexpr (EPI != EPI_PARTIAL) hipLaunchKernelGGL((gemm_fp8_block_skinny_kernel<MT, NT, U, EPI>), dim3((unsigned)p.tiles_n), dim3(64 * SKINNY_WAVES), 0, st, p);
}

template <class T, int EPI>
void launch_stream(const Params& p, int64_t items, hipStream_t st) {
  // (a K range is one work item of its own workgroup; whole tiles share the CUs' persistent workgroups)
  const int64_t grid = EPI == EPI_PARTIAL ? items : std::min<int64_t>(items, device_cus());
  hipLaunchKernelGGL((gemm_fp8_block_stream_kernel<T, EPI>), dim3((unsigned)grid), dim3(256), 0, st, p);
}

template <int EPI>
void launch(const Params& p, Kind kind, hipStream_t st) {
  const int64_t items = (int64_t)p.tiles_m * p.tiles_n * p.split;
  switch (kind) {
    case SKINNY_16: return launch_skinny<1, 1, 2, EPI>(p, st);
    case SKINNY_32: return launch_skinny<2, 2, 2, EPI>(p, st);
    case TILE_64x128: return launch_stream<Stream<2, 4, 6, 6>, EPI>(p, items, st);
    case TILE_128x128: return launch_stream<Stream<4, 4, 4, 4>, EPI>(p, items, st);
    case TILE_128x256: return launch_stream<Stream<4, 8, 3, 3>, EPI>(p, items, st);
    default: return launch_stream<Stream<6, 8, 3, 2>, EPI>(p, items, st);
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
  LX2V_REQUIRE(ldc < (1LL << 22) && (epilogue != LX2V_EPI_RESIDUAL || ldr < (1LL << 22)), LX2V_EUNSUP, "gemm_fp8_block128: bf16 row strides must be below 4 Mi elements");
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
  p.group_rcp = (uint32_t)((1ULL << 32) / (uint64_t)(GROUP_M * p.tiles_n));
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
