// anerf_adapter.hip -- a shared projection with a low-rank adapter of its own for every row (gfx950):
//     y[r] = x[r] W^T + b + s_i (x[r] A_i^T) B_i^T          i = the row's adapter, none: the shared projection alone
// and its gradients with W and b frozen:
//     h[r] = s_i x[r] A_i^T,  u[r] = s_i g[r] B_i,  dx = g W + u A_i,  dA_i = sum_r u[r]^T x[r],  dB_i = sum_r g[r]^T h[r]
// Rows are walked in the order of their adapter (positions p; order[p] = row, NULL = rows lie in that order already), adapter i
// owning positions offsets[i] .. offsets[i+1]-1; the rows behind offsets[L] have no adapter.
//   k_thin       h[p] = s_i x[order[p]] A_i^T: one workgroup a piece of 16 or 32 positions of one adapter
//   k_main       x W^T tile by tile; a tile starts with the low-rank term of the adapters whose positions it holds
//   k_thin_grad  dA_i / dB_i as sums over pieces of an adapter's positions, k_thin_grad_sum adds the pieces in order
//   k_few        up to 64 rows with an adapter index each, in any order
//   k_transpose  W, A, B with their last two axes swapped: dx is then the forward product of (g, W^T, B^T, A^T)
#include <math.h>
#include <algorithm>
#include "anerf_rows.h"

namespace anerf {

// ------------------------------------------------------------------------------------------------------------ h = s_i x A_i^T
// HBM-bound on x.  The four waves split the contraction (every fourth 64-byte step), each holding all 16*MB rows x 16*NJ ranks of the
// piece in MFMA accumulators, fed straight from memory: a row of A serves all rows of the piece, and nothing is read twice from HBM.
// 65520 x 688 fp32, rank 8: 32 us, 5.6 TB/s; 8192 x 4096 bf16, 24 adapters of rank 32 (73 MB): 23 us where x was just
// written, from HBM 33, with 16 rows a piece 35; 200 rows
// x 4096 bf16: 13.7 us with 32 rows a piece, 10.2 with 16.  More waves a piece or deeper loads gain nothing: a few pieces are bound by
// what one CU can load.
// Kept as [position][Rp] fp32 (Rp = rank rounded up to 16, zeros behind the rank) for the gradient of B, and, for the 16-bit types, as what k_main
// multiplies with: h as a sum of three (bf16) or two (fp16) values, each the nearest one to what the others leave, [first of 32 ranks | second |
// third] per 32 ranks (16 where there are no more), which meet the same 32 ranks of B one after the other.  They hold the 24 bits of h, 23 in
// fp16, whose range does not hold every h: its rows are scaled first.
// (bf16 by two values, 16 bits of h: rank 32, 8192 x 4096 -> 4096 the same, rank 128, 8192 x 1024 -> 1024 1.5 of 57 us less)
template <int DT> constexpr int pieces_of = DT == ANERF_BF16 ? 3 : DT == ANERF_F16 ? 2 : 1;
// ranks and values of a row's operand form: where 16 ranks are all, two pieces of them lie in what a product contracts, and zeros beside an odd one
__host__ __device__ constexpr int split_ranks(int Rp) { return Rp > 16 ? (Rp + 31) / 32 * 32 : 16; }
template <int DT>
__host__ __device__ constexpr int split_width(int Rp) { return Rp > 16 ? pieces_of<DT> * split_ranks(Rp) : (pieces_of<DT> + 1) / 2 * 32; }

// ranks j .. j+3 of a row
template <int DT>
__device__ __forceinline__ void store_split(f32x4 v, typename Elem<DT>::T* row, int j, int Rp) {
  typedef typename Elem<DT>::T E;
  typedef E four __attribute__((ext_vector_type(4)));
  const int W = Rp > 16 ? 32 : 16;
  E* o = row + pieces_of<DT> * (j & -W) + (j & (W - 1));
  if (pieces_of<DT> == 3 && W == 16) *reinterpret_cast<four*>(o + 48) = four{(E)0.f, (E)0.f, (E)0.f, (E)0.f};
#pragma unroll
  for (int p = 0; p < pieces_of<DT>; ++p) {
    four piece;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      piece[e] = (E)v[e];
      v[e] -= (float)piece[e];                                 // (behind an infinity: NaN; k_main takes h itself where that shows)
    }
    *reinterpret_cast<four*>(o + W * p) = piece;
  }
}

// a row of h is divided by the power of two that brings its largest value into [2^14, 2^15); rows of zeros, infinities and NaN stay
__device__ __forceinline__ int row_exponent(float big) {
  return big > 0.f && __builtin_isfinite(big) ? max(ilogbf(big) - 14, -100) : 0;
}

constexpr int TH_WAVES = 4, TH_DEPTH = 4;
template <int V> struct Const { static constexpr int value = V; };
template <bool C, typename A, typename B> struct Pick { typedef A T; };
template <typename A, typename B> struct Pick<false, A, B> { typedef B T; };

template <int DT, int NJ, int MB>
__global__ void __launch_bounds__(TH_WAVES * 64) k_thin(const typename Elem<DT>::T* __restrict__ x, long long ldx, const int32_t* __restrict__ order,
                                                        const typename Elem<DT>::T* __restrict__ down, const int32_t* __restrict__ offsets,
                                                        int L, long long K, int R, int Rp, const float* __restrict__ scale_of, float scale,
                                                        float* __restrict__ h, typename Elem<DT>::T* __restrict__ split, float* __restrict__ factor,
                                                        int32_t* __restrict__ owner) {
  typedef typename Elem<DT>::T E;
  constexpr int EPC = Elem<DT>::EPC, STEP = 4 * EPC, TH_ROWS = 16 * MB;
  __shared__ f32x4 red[TH_WAVES][MB * NJ][64];
  int a, p0, p1;
  if (!find_piece(offsets, L, TH_ROWS, blockIdx.x, a, p0, p1)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int j0 = blockIdx.y * 16 * NJ;
  const float s_a = scale_of ? scale * scale_of[a] : scale;
  const E* A = down + (long long)a * R * K;
  const E* xr[MB];
  const E* ar[NJ];
#pragma unroll
  for (int m = 0; m < MB; ++m) {
    const int p = min(p0 + 16 * m + i, p1 - 1);      // rows behind the piece repeat its last one; their sums are not stored
    xr[m] = x + (long long)(order ? order[p] : p) * ldx;
  }
#pragma unroll
  for (int n = 0; n < NJ; ++n) ar[n] = A + (long long)min(j0 + 16 * n + i, R - 1) * K;
  f32x4 acc[MB][NJ];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NJ; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  const long long steps = K / STEP;
  auto walk = [&](long long s0, auto depth) {       // `depth` steps of this wave, all their loads in front of the products
    constexpr int D = decltype(depth)::value;
    u32x4 xv[D][MB], av[D][NJ];
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const long long k = (s0 + d * TH_WAVES) * STEP + q * EPC;
#pragma unroll
      for (int m = 0; m < MB; ++m) xv[d][m] = load16(xr[m] + k);
#pragma unroll
      for (int n = 0; n < NJ; ++n) av[d][n] = load16(ar[n] + k);
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int n = 0; n < NJ; ++n)
#pragma unroll
          for (int e = 0; e < Elem<DT>::INSTR; ++e) acc[m][n] = Elem<DT>::mma(av[d][n], xv[d][m], acc[m][n], e);
  };
  long long s = wave;
  for (; s + (TH_DEPTH - 1) * TH_WAVES < steps; s += TH_DEPTH * TH_WAVES) walk(s, Const<TH_DEPTH>());
  for (; s < steps; s += TH_WAVES) walk(s, Const<1>());
  if (steps * STEP < K && wave == (int)(steps % TH_WAVES)) {
    const long long k = steps * STEP + q * EPC;
    u32x4 xv[MB], av[NJ];
#pragma unroll
    for (int m = 0; m < MB; ++m) xv[m] = load_tail<DT>(xr[m], k, K);
#pragma unroll
    for (int n = 0; n < NJ; ++n) av[n] = load_tail<DT>(ar[n], k, K);
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NJ; ++n)
#pragma unroll
        for (int e = 0; e < Elem<DT>::INSTR; ++e) acc[m][n] = Elem<DT>::mma(av[n], xv[m], acc[m][n], e);
  }
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int n = 0; n < NJ; ++n) red[wave][m * NJ + n][lane] = acc[m][n];
  __syncthreads();
  constexpr int LINE = 16 * NJ + 4;
  __shared__ float tile[TH_ROWS * LINE];            // the piece's h, row by row
  for (int f = wave; f < MB * NJ; f += TH_WAVES) {
    f32x4 v = red[0][f][lane];
#pragma unroll
    for (int w = 1; w < TH_WAVES; ++w) v += red[w][f][lane];
    *reinterpret_cast<f32x4*>(tile + (16 * (f / NJ) + i) * LINE + 16 * (f % NJ) + 4 * q) = v;
  }
  __syncthreads();
  // eight lanes a row, four ranks each and turn
  const int r = threadIdx.x >> 3, part = threadIdx.x & 7, p = p0 + r;
  if (r >= TH_ROWS || p >= p1) return;
  if (part == 0 && j0 == 0) owner[p] = a;
  f32x4 v[(4 * NJ + 7) / 8];
  float big = 0.f;
  const int end = DT == ANERF_F32 ? Rp : split_ranks(Rp);
#pragma unroll
  for (int t = 0; t < (4 * NJ + 7) / 8; ++t) {
    const int j = 4 * (part + 8 * t);
    if (j >= 16 * NJ || j0 + j >= end) continue;
    v[t] = *reinterpret_cast<const f32x4*>(tile + r * LINE + j);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[t][e] = j0 + j + e < R ? v[t][e] * s_a : 0.f;          // ranks of the padding: zero
      big = fmaxf(big, fabsf(v[t][e]));
    }
    if (j0 + j < Rp) *reinterpret_cast<f32x4*>(h + (long long)p * Rp + j0 + j) = v[t];
  }
  if constexpr (DT != ANERF_F32) {
    if (DT == ANERF_F16 && gridDim.y > 1) return;              // (k_split_rows needs the whole row)
    float shrink = 1.f;
    if constexpr (DT == ANERF_F16) {
#pragma unroll
      for (int d = 4; d; d >>= 1) big = fmaxf(big, __shfl_xor(big, d));
      const int e = row_exponent(big);
      shrink = ldexpf(1.f, -e);
      if (part == 0) factor[p] = ldexpf(1.f, e);
    }
#pragma unroll
    for (int t = 0; t < (4 * NJ + 7) / 8; ++t) {
      const int j = 4 * (part + 8 * t);
      if (j < 16 * NJ && j0 + j < end) store_split<DT>(v[t] * shrink, split + (long long)p * split_width<DT>(Rp), j0 + j, Rp);
    }
  }
}

// fp16 with more ranks than a workgroup of k_thin holds: the rows' scaling and splitting (8192 rows of rank 128: 5 us)
__global__ void __launch_bounds__(256) k_split_rows(const float* __restrict__ h, const int32_t* __restrict__ kept, int Rp, _Float16* __restrict__ split,
                                                    float* __restrict__ factor) {
  const int p = blockIdx.x * 16 + (threadIdx.x >> 4), i = threadIdx.x & 15;
  if (p >= *kept) return;
  const float* r = h + (long long)p * Rp;
  float big = 0.f;
  for (int j = i; j < Rp; j += 16) big = fmaxf(big, fabsf(r[j]));
#pragma unroll
  for (int d = 8; d; d >>= 1) big = fmaxf(big, __shfl_xor(big, d));
  const int e = row_exponent(big);
  if (i == 0) factor[p] = ldexpf(1.f, e);
  const float down = ldexpf(1.f, -e);
  for (int j = 4 * i; j < split_ranks(Rp); j += 64) {
    const f32x4 v = j < Rp ? *reinterpret_cast<const f32x4*>(r + j) * down : f32x4{0.f, 0.f, 0.f, 0.f};
    store_split<ANERF_F16>(v, split + (long long)p * split_width<ANERF_F16>(Rp), j, Rp);
  }
}

// ------------------------------------------------------------------------------------------------------------------ y = x W^T ...
// BM positions x BN outputs a workgroup of WM x WN waves, 16 x 16 MFMA blocks with W's rows as the first operand, so that a lane ends
// with four consecutive outputs of one row.  The contraction goes through LDS 128 bytes of every row at a time, NS stages deep; 16-byte
// chunk c of row r lies at chunk c ^ (r & 7), which spreads a fragment read over the banks.  DIRECT: global_load_lds_dwordx4, eight rows
// an instruction, the lanes fetching the chunks in the order they have to lie in LDS (16-byte aligned rows); otherwise through registers,
// at any alignment.
// Few tiles: `splits` workgroups share one, each with a contiguous part of the stages, and k_sum_parts adds their fp32 tiles.
// The low-rank term comes first, behind the first stage's loads: for every adapter with positions in the tile h B_i^T is added to the
// blocks of its rows; a block that two adapters share takes it by row (a NaN in one adapter stays with its rows).  Waves with rows of many
// adapters take it row by row.
// fp32 sums of long rows are kept in two levels: every FOLD stages the accumulators are added to a second set.  An instruction adds its four
// products one after the other, so that a chain has Rp (the low-rank term, in the first) + 32 * FOLD + K / (32 * FOLD) additions at most.
// Bound by the matrix units.  In a trace, in turn with a library's plain product of the same rows (us with adapters, without, the library): bf16,
// 8192 x 4096 -> 4096, 24 adapters of rank 32: 269 (1020 TFLOP/s; in a loop of its own 239), 243, 195; 4096 x 2048 -> 2048, 12 of rank 16: 41, 35, 33;
// fp32, 65520 x 688 -> 256, 16 of rank 8: 214 (108 TFLOP/s; rows in order 211), 205, 203; 24000 x 688 -> 256: 87, 75, 94;
// 8192 x 4096 -> 4096, 24 of rank 32: 1901 (145 TFLOP/s), 1873, 1830.
struct MainArgs {
  const void *x, *w, *bias, *up;
  const int32_t *offsets, *order;
  const void* h;               // operand form of h: [M][Rp] fp32, [M][split_width] 16-bit
  const float* factor;         // fp16: power of two of every row of h
  const float* h32;            // [M][Rp]
  const int32_t* owner;        // the positions' adapters
  void* y;
  float* part;                 // splits > 1: fp32 [splits][M][N]
  long long ldx, ldw, K, N;
  long long M;
  int L, R, Rp, splits;
};

constexpr int FOLD = 16;

template <int DT, int BM, int BN, int WM, int WN, int NS, bool DIRECT>
__global__ void __launch_bounds__(WM * WN * 64, BM * BN <= 64 * 64 ? 4 : 2) k_main(MainArgs P) {
  typedef typename Elem<DT>::T E;
  constexpr int EPC = Elem<DT>::EPC, KB = 8 * EPC;        // elements of a 128-byte row piece
  constexpr int NW = WM * WN;
  constexpr int BS = 16, TM = BM / WM, TN = BN / WN, MI = TM / BS, NI = TN / BS;
  constexpr int XL = BM / 8 / NW, WL = BN / 8 / NW;       // 16-byte loads of a lane and stage
  constexpr int STAGE = (BM + BN) * 8;                    // 16-byte units
  extern __shared__ u32x4 lds[];                          // [NS][STAGE]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane % BS, q = lane / BS;
  const int wm = wave % WM, wn = wave / WM;
  // workgroups go round-robin to the 8 XCDs: each XCD gets a contiguous range of the tile order, in which 4 row tiles share a column of W
  long long m0, n0;
  {
    const long long tm = (P.M + BM - 1) / BM, tn = (P.N + BN - 1) / BN, all = tm * tn;
    const unsigned b = P.splits > 1 ? blockIdx.x / P.splits : blockIdx.x;
    const long long xcd = b & 7, t = xcd * (all >> 3) + (xcd < (all & 7) ? xcd : (all & 7)) + (b >> 3);
    const long long g = t / (4 * tn), in = t % (4 * tn);
    const long long rows = tm - 4 * g < 4 ? tm - 4 * g : 4;
    m0 = (4 * g + in % rows) * BM;
    n0 = in / rows * BN;
  }
  // a lane's part of every stage: row r = 8 * (wave + NW * l) + lane / 8, the chunk that has to lie at position lane % 8.  DIRECT: byte
  // offsets of 32 bits against a scalar base that moves with the stage (a vector instruction in the fp32 loop costs matrix time)
  const int sub = lane >> 3, ch = (lane & 7) ^ sub;
  typedef typename Pick<DIRECT, unsigned, long long>::T Off;
  Off xo[XL], wo[WL];
#pragma unroll
  for (int l = 0; l < XL; ++l) {
    long long p = m0 + 8 * (wave + NW * l) + sub;
    if (p >= P.M) p = P.M - 1;
    xo[l] = (Off)(((P.order ? (long long)P.order[p] : p) * P.ldx + ch * EPC) * (long long)sizeof(E));
  }
#pragma unroll
  for (int l = 0; l < WL; ++l) {
    long long n = n0 + 8 * (wave + NW * l) + sub;
    if (n >= P.N) n = P.N - 1;
    wo[l] = (Off)((n * P.ldw + ch * EPC) * (long long)sizeof(E));
  }
  u32x4 rx[XL], rw[WL];
  auto at = [&](int buf, int row8) { return buf * STAGE + row8 * 64; };      // eight rows of 128 bytes
  const unsigned lds0 = (unsigned)reinterpret_cast<size_t>((lds_ptr_t)lds) + wave * 1024;
  auto dma = [&](const void* base, unsigned off, int to) {                   // `to`: 16-byte units behind the wave's eight rows
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds0 + to * 16), "v"(off), "s"(base) : "memory", "m0");
  };
  const int K = (int)P.K;
  auto fetch_regs = [&](int s) {
    const int k = s * KB, left = K - k - ch * EPC;
    const char* xb = static_cast<const char*>(P.x) + (long long)k * sizeof(E);
    const char* wb = static_cast<const char*>(P.w) + (long long)k * sizeof(E);
    if (left >= EPC) {
#pragma unroll
      for (int l = 0; l < XL; ++l) rx[l] = load16(xb + xo[l]);
#pragma unroll
      for (int l = 0; l < WL; ++l) rw[l] = load16(wb + wo[l]);
    } else {
#pragma unroll
      for (int l = 0; l < XL; ++l) rx[l] = load_tail<DT>(reinterpret_cast<const E*>(xb + xo[l]), 0, left);
#pragma unroll
      for (int l = 0; l < WL; ++l) rw[l] = load_tail<DT>(reinterpret_cast<const E*>(wb + wo[l]), 0, left);
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int l = 0; l < XL; ++l) lds[at(buf, wave + NW * l) + lane] = rx[l];
#pragma unroll
    for (int l = 0; l < WL; ++l) lds[at(buf, BM / 8 + wave + NW * l) + lane] = rw[l];
  };
  const int all_stages = (K + KB - 1) / KB, full = K / KB;
  const int part = P.splits > 1 ? blockIdx.x % P.splits : 0;
  const int first = P.splits > 1 ? (int)((long long)all_stages * part / P.splits) : 0;
  const int stages = P.splits > 1 ? (int)((long long)all_stages * (part + 1) / P.splits) : all_stages;      // end of this workgroup's
  // starts stage s; DIRECT: into LDS, otherwise into registers.  In a last, partial stage the chunks behind the row are not there: DIRECT
  // lanes fetch the stage's first chunk in their place, and the products take zeros for them
  auto start = [&](int s, int buf) {
    if constexpr (DIRECT) {
      const char* xb = static_cast<const char*>(P.x) + (long long)s * 128;
      const char* wb = static_cast<const char*>(P.w) + (long long)s * 128;
      if (s < full) {
#pragma unroll
        for (int l = 0; l < XL; ++l) dma(xb, xo[l], at(buf, NW * l));
#pragma unroll
        for (int l = 0; l < WL; ++l) dma(wb, wo[l], at(buf, BM / 8 + NW * l));
      } else {
        const unsigned back = s * KB + ch * EPC < K ? 0u : ch * 16u;
#pragma unroll
        for (int l = 0; l < XL; ++l) dma(xb, xo[l] - back, at(buf, NW * l));
#pragma unroll
        for (int l = 0; l < WL; ++l) dma(wb, wo[l] - back, at(buf, BM / 8 + NW * l));
      }
    } else {
      fetch_regs(s);
    }
  };
#pragma unroll
  for (int s = 0; s < (DIRECT ? NS - 1 : 1); ++s)
    if (first + s < stages) start(first + s, s);
  f32x4 acc[MI][NI];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x4{};

  // ---- low-rank term
  const int kept = P.offsets[P.L];
  if (m0 < kept && part == 0) {
    const int t0 = (int)m0, t1 = min((int)(m0 + BM < P.M ? m0 + BM : P.M), kept);
    const int w0 = t0 + wm * TM;                               // the wave's first position and output
    const long long c0 = n0 + wn * TN;
    const int last_col = (int)(P.N - 1 - c0 < TN ? P.N - 1 - c0 : TN);
    // a product contracts 64 bytes of h's row: 16 fp32 ranks; a piece of 32 ranks of a 16-bit type, or, where 16 are all, two pieces of them
    const bool wide = DT != ANERF_F32 && P.Rp > 16;
    const int times = wide ? pieces_of<DT> : (pieces_of<DT> + 1) / 2;      // products with the same ranks of B
    const int row_bytes = DT == ANERF_F32 ? P.Rp * 4 : 2 * split_width<DT>(P.Rp);
    const char* hw = static_cast<const char*>(P.h) + (long long)w0 * row_bytes + 16 * q;
    int b0 = 0;                                                // of 64 adapters looked at together
    if (P.L > 64) {                                            // first those that hold the tile's first position
      const unsigned long long at = __ballot(64 * lane < P.L && P.offsets[min(64 * lane, P.L)] <= t0);
      b0 = 64 * (63 - __builtin_clzll(at));
    }
    // A wave whose rows are of many adapters (64 rows may be of as many) would take them one after the other, 0.3 us each and 16 ranks.  It
    // takes its rows' dots of `rank` fp32 values instead, whose loads do not wait for one another -- where B's rows are short enough for the
    // first cache to serve them (bf16, rank 16, 1024 x 1024, 48 rows of 64 adapters: 26 -> 17 us; 256 rows x 2048 x 2048 of 500: 50 -> 36; with
    // rank 64 the dots took twice the time).
    bool one_by_one = false;
    if constexpr (MI <= 4) {
      constexpr int many = 3 * MI / 2 * NI;
      if (P.R * (int)sizeof(E) <= 64) {
        int count = 0;
        for (int b = b0; b < P.L && count <= many; b += 64) {
          const int ab = b + lane;
          const int lo = ab < P.L ? P.offsets[ab] : 0, hi = ab < P.L ? P.offsets[ab + 1] : 0;
          count += __popcll(__ballot(hi > lo && hi > w0 && lo < min(w0 + TM, t1)));
          if (__builtin_amdgcn_readlane(hi, 63) >= min(w0 + TM, t1)) break;
        }
        one_by_one = count > many;
      }
      if (one_by_one) {
        typedef E vec __attribute__((ext_vector_type(EPC)));
#pragma unroll
        for (int m0 = 0; m0 < MI; m0 += 2) {                   // two rows of a lane at a time
          const E* br[2];
          const float* hr[2];
          bool has[2];
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            const int p = w0 + BS * (m0 + m) + i;
            has[m] = p < kept;
            br[m] = static_cast<const E*>(P.up) + (has[m] ? (long long)P.owner[p] * P.N : 0) * P.R;
            hr[m] = P.h32 + (long long)(has[m] ? p : t0) * P.Rp;
          }
#pragma unroll
          for (int n = 0; n < NI; ++n) {
            long long at[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const long long col = c0 + BS * n + 4 * q + e;
              at[e] = (col < P.N ? col : P.N - 1) * P.R;
            }
            f32x4 dot[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
            int j = 0;
            for (; j + EPC <= P.R; j += EPC) {
              vec bv[2][4];
              f32x4 hv[2][EPC / 4];
#pragma unroll
              for (int m = 0; m < 2; ++m) {
#pragma unroll
                for (int e = 0; e < 4; ++e) bv[m][e] = __builtin_bit_cast(vec, load16(br[m] + at[e] + j));
#pragma unroll
                for (int k = 0; k < EPC / 4; ++k) hv[m][k] = __builtin_bit_cast(f32x4, load16(hr[m] + j + 4 * k));
              }
#pragma unroll
              for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                  for (int k = 0; k < EPC; ++k) dot[m][e] = fmaf(hv[m][k / 4][k % 4], (float)bv[m][e][k], dot[m][e]);
            }
            for (; j < P.R; ++j)
#pragma unroll
              for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) dot[m][e] = fmaf(hr[m][j], (float)br[m][at[e] + j], dot[m][e]);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[m0 + m][n][e] = has[m] ? dot[m][e] : 0.f;
          }
        }
      }
    }
    // the adapters that own positions of the tile, one after the other
    for (; !one_by_one && b0 < P.L; b0 += 64) {
      const int ab = b0 + lane;
      const int lo = ab < P.L ? P.offsets[ab] : 0, hi = ab < P.L ? P.offsets[ab + 1] : 0;
      unsigned long long owners = __ballot(hi > lo && hi > t0 && lo < t1);
      while (owners) {
        const int l = __builtin_ctzll(owners);
        owners &= owners - 1;
        int r0 = max(__builtin_amdgcn_readlane(lo, l) - w0, 0), r1 = min(__builtin_amdgcn_readlane(hi, l) - w0, TM);
        if (r0 >= r1) continue;                                // none of this wave's
        const E* bw = static_cast<const E*>(P.up) + ((long long)(b0 + l) * P.N + c0) * P.R;
        int j = DT == ANERF_F32 ? 4 * q : wide ? 8 * q : 8 * (q & 1);
        u32x4 bf[NI];
        for (int at = 0, s = 0; at < row_bytes; at += 64) {
          const char* hs = hw + at;
          asm volatile("" : "+s"(r0), "+s"(r1));               // (tests of the blocks are not kept across the loop: registers)
          u32x4 hf[MI];
          if (s == 0) {
#pragma unroll
            for (int n = 0; n < NI; ++n) bf[n] = load_tail<DT>(bw + min(BS * n + i, last_col) * P.R, j, P.R);
          }
#pragma unroll
          for (int m = 0; m < MI; ++m) {
            const int r = min(max(BS * m + i, r0), r1 - 1);
            hf[m] = *reinterpret_cast<const u32x4*>(hs + r * row_bytes);
          }
#pragma unroll
          for (int m = 0; m < MI; ++m) {
            if (BS * m >= r1 || BS * m + BS <= r0) continue;
            if (BS * m >= r0 && BS * m + BS <= r1) {
#pragma unroll
              for (int n = 0; n < NI; ++n)
#pragma unroll
                for (int e = 0; e < Elem<DT>::INSTR; ++e) acc[m][n] = Elem<DT>::mma(bf[n], hf[m], acc[m][n], e);
            } else {
              const bool mine = BS * m + i >= r0 && BS * m + i < r1;
#pragma unroll
              for (int n = 0; n < NI; ++n) {
                f32x4 t = f32x4{};
#pragma unroll
                for (int e = 0; e < Elem<DT>::INSTR; ++e) t = Elem<DT>::mma(bf[n], hf[m], t, e);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[m][n][e] = mine ? acc[m][n][e] + t[e] : acc[m][n][e];
              }
            }
          }
          if (++s == times) s = 0, j += DT == ANERF_F32 ? 16 : 32;
        }
      }
      if (__builtin_amdgcn_readlane(hi, 63) >= t1) break;
    }
    if (DT == ANERF_F16 && !one_by_one) {
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const int p = w0 + BS * m + i;
        const float f = p < kept ? P.factor[p] : 1.f;
#pragma unroll
        for (int n = 0; n < NI; ++n) acc[m][n] *= f;
      }
    }
    // An infinite value of h or B has met pieces of the other's values there, zeros and ones of either sign among them, and infinity times 0
    // is NaN.  Values that are not finite are therefore taken again, from h itself.
    if constexpr (DT != ANERF_F32) {
      float zero = 0.f;
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) zero = fmaf(acc[m][n][e], 0.f, zero);
      if (!one_by_one && __any(!(zero == 0.f))) {
#pragma unroll
        for (int m = 0; m < MI; ++m) {
          const int p = w0 + BS * m + i;
          const bool has = p < kept;
          const E* br = static_cast<const E*>(P.up) + (has ? (long long)P.owner[p] * P.N : 0) * P.R;
          const float* hr = P.h32 + (long long)(has ? p : t0) * P.Rp;
#pragma unroll
          for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if (!has || __builtin_isfinite(acc[m][n][e])) continue;
              const long long col = c0 + BS * n + 4 * q + e;
              const E* b = br + (col < P.N ? col : P.N - 1) * P.R;
              float dot = 0.f;
#pragma unroll 1
              for (int j = 0; j < P.R && dot == dot; ++j) dot = fmaf(hr[j], (float)b[j], dot);      // (NaN stays NaN)
              acc[m][n][e] = dot;
            }
        }
      }
    }
  }

  // ---- x W^T
  constexpr bool F32 = DT == ANERF_F32;
  f32x4 sum[F32 ? MI : 1][F32 ? NI : 1];
  if constexpr (F32) {
#pragma unroll
    for (int m = 0; m < MI; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n) sum[m][n] = f32x4{};
  }
  // A half stage's rows of x are taken in two groups, and every group's fragments are read from LDS while the products of the group
  // before it run (two sets of W's fragments, one of each group of x's), so that the matrix units need not wait for LDS.  The one barrier
  // of a stage lies before its last group's products: there every wave has read the last of stage s, whose buffer stage s + NS may then
  // overwrite, and every wave's loads of stage s + 1 have arrived.
  constexpr int MG = MI / 2;
  static_assert(MI % 2 == 0, "two groups of row blocks a half stage");
  u32x4 wf[2][NI], xf[2][MG];
  // fragment addresses: row i of a block has r & 7 = i & 7, the halves' chunks differ in bit 2
  const int px = (wm * TM + i) * 8, pw = (BM + wn * TN + i) * 8, ch0 = q ^ (i & 7);
  auto read_w = [&](int buf, int h) {
    const u32x4* f = lds + buf * STAGE + pw + (ch0 ^ (4 * h));
#pragma unroll
    for (int n = 0; n < NI; ++n) wf[h][n] = f[n * BS * 8];
  };
  auto read_x = [&](int buf, int h, int g) {
    const u32x4* f = lds + buf * STAGE + px + (ch0 ^ (4 * h));
#pragma unroll
    for (int m = 0; m < MG; ++m) xf[g][m] = f[(g * MG + m) * BS * 8];
  };
  auto products = [&](int h, int g) {
#pragma unroll
    for (int m = 0; m < MG; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n)
#pragma unroll
        for (int e = 0; e < Elem<DT>::INSTR; ++e) acc[g * MG + m][n] = Elem<DT>::mma(wf[h][n], xf[g][m], acc[g * MG + m][n], e);
  };
  // waits for the oldest stage in flight; `all`: of NS - 1
  auto arrive = [&](bool all) {
    if (DIRECT) {
      if (NS > 2 && all) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * (XL + WL)) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __syncthreads();
  };
  if (!DIRECT) put(0);
  arrive(first + NS - 1 <= stages);
  if (DIRECT) {
    if (first + NS - 1 < stages) start(first + NS - 1, NS - 1);
  } else if (first + 1 < stages) {
    start(first + 1, 1);
  }
  read_w(0, 0);
  read_x(0, 0, 0);
  auto zero_behind = [&](u32x4* f, int n, int h) {      // fragments of the partial stage: chunks behind the row
    const bool there = full * KB + (4 * h + q) * EPC < K;
#pragma unroll
    for (int e = 0; e < n; ++e) f[e] = there ? f[e] : u32x4{0, 0, 0, 0};
  };
  auto stage = [&](int s, int buf, auto partial) {
    constexpr bool PART = decltype(partial)::value != 0;
    read_x(buf, 0, 1);
    if (PART) zero_behind(wf[0], NI, 0), zero_behind(xf[0], MG, 0), zero_behind(xf[1], MG, 0);
    products(0, 0);
    read_w(buf, 1);
    read_x(buf, 1, 0);
    if (PART) zero_behind(wf[1], NI, 1), zero_behind(xf[0], MG, 1);
    products(0, 1);
    read_x(buf, 1, 1);
    if (PART) zero_behind(xf[1], MG, 1);
    products(1, 0);
    if (s + 1 < stages) {
      const int next = buf + 1 == NS ? 0 : buf + 1;
      if (!DIRECT) put(next);
      arrive(s + NS <= stages);
      if (s + NS < stages) start(s + NS, buf);
      read_w(next, 0);
      read_x(next, 0, 0);
    }
    products(1, 1);
  };
  // the buffer is a constant of the loop's code: NS stages a turn
  const int whole = DIRECT && full < stages ? full : stages;
  for (int s = first; s < whole; s += NS) {
    stage(s, 0, Const<0>());
    if (s + 1 < whole) stage(s + 1, 1, Const<0>());
    if constexpr (NS > 2) {
      if (s + 2 < whole) stage(s + 2, 2, Const<0>());
    }
    if constexpr (NS > 3) {
      if (s + 3 < whole) stage(s + 3, 3, Const<0>());
    }
    if constexpr (F32) {
      if ((s - first) % FOLD == FOLD - NS) {
#pragma unroll
        for (int m = 0; m < MI; ++m)
#pragma unroll
          for (int n = 0; n < NI; ++n) {
            sum[m][n] += acc[m][n];
            acc[m][n] = f32x4{};
          }
      }
    }
  }
  if (DIRECT && full < stages) stage(full, (full - first) % NS, Const<1>());

  // ---- bias, rounding, store.  A lane holds four outputs of its row in each block.  fp32: 16 bytes, stored as they are
  if constexpr (F32) {
    const float* bias = P.splits > 1 ? nullptr : static_cast<const float*>(P.bias);
    f32x4 add[NI];
    long long row[MI];
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const long long col = n0 + wn * TN + BS * n + 4 * q;
#pragma unroll
      for (int e = 0; e < 4; ++e) add[n][e] = 0.f;
      if (bias && col + 4 <= P.N) {
        __builtin_memcpy(&add[n], bias + col, 16);
      } else if (bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < P.N) add[n][e] = bias[col + e];
      }
    }
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      const long long p = m0 + wm * TM + BS * m + i;
      row[m] = p < P.M ? (P.order ? (long long)P.order[p] : p) : -1;
    }
#pragma unroll
    for (int m = 0; m < MI; ++m) {
      if (row[m] < 0) continue;
      float* yr = P.splits > 1 ? P.part + (part * P.M + row[m]) * P.N : static_cast<float*>(P.y) + row[m] * P.N;
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const long long col = n0 + wn * TN + BS * n + 4 * q;
        f32x4 v = acc[m][n] + sum[m][n];
        if (bias) v += add[n];
        if (col + 4 <= P.N) {
          store16(yr + col, __builtin_bit_cast(u32x4, v));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (col + e < P.N) yr[col + e] = v[e];
        }
      }
    }
    return;
  }
  // 16-bit types: through LDS, a wave's half of its rows at a time, to leave 16 bytes a lane along the rows (8 bytes a lane in 32-byte
  // pieces straight from the registers: 8192 x 4096 outputs 6 us more)
  auto emit = [&](auto one, auto* to, const E* bias) {
    typedef decltype(one) S;
    typedef S four __attribute__((ext_vector_type(4)));
    constexpr int LINE = TN * (int)sizeof(S) + 16, ROWS = MG * BS, PER = 16 / (int)sizeof(S), LPR = TN / PER, RPI = 64 / LPR;
    static_assert(NW * ROWS * LINE <= NS * STAGE * 16 && ROWS % RPI == 0, "the staged rows fit where the stages were");
    char* mine = reinterpret_cast<char*>(lds) + wave * (ROWS * LINE);
    const long long cw = n0 + wn * TN;
    const int r0 = lane / LPR, c = lane % LPR * PER;
    typedef E bias4 __attribute__((ext_vector_type(4)));
    bias4 add[NI];
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const long long col = cw + BS * n + 4 * q;
#pragma unroll
      for (int e = 0; e < 4; ++e) add[n][e] = (E)0.f;
      if (bias && col + 4 <= P.N) {
        __builtin_memcpy(&add[n], bias + col, sizeof(bias4));
      } else if (bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < P.N) add[n][e] = bias[col + e];
      }
    }
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const long long pw = m0 + wm * TM + g * ROWS;
      long long row[ROWS / RPI];
#pragma unroll
      for (int t = 0; t < ROWS / RPI; ++t) {
        const long long p = pw + t * RPI + r0;
        row[t] = p < P.M ? (P.order ? (long long)P.order[p] : p) : -1;
      }
#pragma unroll
      for (int m = 0; m < MG; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n) {
          four o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = acc[g * MG + m][n][e];
            o[e] = (S)(bias ? v + (float)add[n][e] : v);
          }
          *reinterpret_cast<four*>(mine + (BS * m + i) * LINE + (BS * n + 4 * q) * (int)sizeof(S)) = o;
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // the wave's own lines: no barrier
#pragma unroll
      for (int t = 0; t < ROWS / RPI; ++t) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(mine + (t * RPI + r0) * LINE + c * (int)sizeof(S));
        S* o = to + row[t] * P.N + cw + c;
        if (row[t] >= 0) {
          if (cw + c + PER <= P.N) {
            store16(o, v);
          } else {
            typedef S vec __attribute__((ext_vector_type(PER)));
            const vec w = __builtin_bit_cast(vec, v);
#pragma unroll
            for (int e = 0; e < PER; ++e)
              if (cw + c + e < P.N) o[e] = w[e];
          }
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  };
  __syncthreads();                           // every wave is done with the stages
  if constexpr (!F32 && BM == 64 && BN == 64) {
    if (P.splits > 1) {
      emit(0.f, P.part + part * P.M * P.N, static_cast<const E*>(nullptr));
      return;
    }
  }
  if constexpr (!F32) emit(E(), static_cast<E*>(P.y), static_cast<const E*>(P.bias));
}

// y = the parts' sum in order + bias; [M][N] as one row of values (128 x 4096 outputs in 4 parts: 4 us)
template <int DT>
__global__ void __launch_bounds__(256) k_sum_parts(const float* __restrict__ part, int splits, long long all, long long N, const typename Elem<DT>::T* __restrict__ bias,
                                                   typename Elem<DT>::T* __restrict__ y) {
  typedef typename Elem<DT>::T E;
  typedef E out4 __attribute__((ext_vector_type(4)));
  const long long e = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= all) return;
  if (e + 4 <= all) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      f32x4 w;
      __builtin_memcpy(&w, part + s * all + e, 16);
      v += w;
    }
    out4 o;
    long long c = bias ? e % N : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      o[k] = (E)(bias ? v[k] + (float)bias[c] : v[k]);
      c = c + 1 == N ? 0 : c + 1;
    }
    __builtin_memcpy(y + e, &o, sizeof(o));
  } else {
    for (int k = 0; e + k < all; ++k) {
      float v = 0.f;
      for (int s = 0; s < splits; ++s) v += part[s * all + e + k];
      y[e + k] = (E)(bias ? v + (float)bias[(e + k) % N] : v);
    }
  }
}

// -------------------------------------------------------------------------------------------------------- few rows (a decoding step)
// Up to 64 rows, each with an adapter index of its own, no plan: the time is what the shared weight takes to arrive.
//   k_few_thin  h[r][j] = s_i <x[r], A_i[j]>: one wave a value
//   k_few       a workgroup owns 16*NT outputs of all rows; its eight waves take every eighth 128 bytes of W's rows straight into MFMA operands
//               (W is read once, no LDS on its way), x comes from L2, and the waves' sums are added through LDS.  The low-rank term of
//               an output is a dot of `rank` values in fp32, read in front of the loop, so that B's latency hides behind W's.
// bf16, rank 16: one row x 4096 -> 4096 5.7 + 8.0 us (W at 4.2 TB/s); 48 rows x 4096 -> 8192 5.6 + 25 us (67 MB of W, 13 MB of B, and
// 126 MB of x from L2).  The routed kernels take 42 us for the 48 rows, plan included, and catch up where rows are many and outputs few: 64 rows x
// 4096 -> 1024 26.9 us here, 25.7 there (fp32 45.8, 40.7), 4096 -> 4096 27.8 and 36.8, 1024 -> 1024 10.8 and 19.0: the limit is 64 rows.
constexpr int FEW_WAVES = 8;
static_assert(ANERF_FEW_ROWS == 64, "four blocks of 16 rows");

template <typename I>
__device__ __forceinline__ int adapter_of(const void* groups, int r, int L) {
  const I v = static_cast<const I*>(groups)[r];
  return v >= 0 && v < (I)L ? (int)v : -1;
}

template <int DT>
__global__ void __launch_bounds__(256) k_few_thin(const typename Elem<DT>::T* __restrict__ x, long long ldx, const typename Elem<DT>::T* __restrict__ down,
                                                  const void* __restrict__ groups, int wide, int L, long long K, int R, const float* __restrict__ scale_of,
                                                  float scale, float* __restrict__ h) {
  typedef typename Elem<DT>::T E;
  constexpr int EPC = Elem<DT>::EPC;
  typedef E vec __attribute__((ext_vector_type(EPC)));
  const int r = blockIdx.x, j = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int a = wide ? adapter_of<long long>(groups, r, L) : adapter_of<int>(groups, r, L);
  if (a < 0 || j >= R) return;
  const E* xr = x + r * ldx;
  const E* ar = down + ((long long)a * R + j) * K;
  float sum = 0.f;
  const long long whole = K / EPC;
#pragma unroll 4
  for (long long c = lane; c < whole; c += 64) {
    const vec xv = __builtin_bit_cast(vec, load16(xr + c * EPC)), av = __builtin_bit_cast(vec, load16(ar + c * EPC));
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < EPC; ++e) s = fmaf((float)xv[e], (float)av[e], s);
    sum += s;
  }
  const long long c = whole * EPC + lane;
  if (c < K) sum = fmaf((float)xr[c], (float)ar[c], sum);
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) h[r * R + j] = sum * (scale_of ? scale * scale_of[a] : scale);
}

template <int DT, int MT, int NT>
__global__ void __launch_bounds__(FEW_WAVES * 64) k_few(const typename Elem<DT>::T* __restrict__ x, long long ldx, const typename Elem<DT>::T* __restrict__ w,
                                                        const typename Elem<DT>::T* __restrict__ bias, const typename Elem<DT>::T* __restrict__ up,
                                                        const void* __restrict__ groups, int wide, int L, int M, long long K, long long N, int R,
                                                        const float* __restrict__ h, typename Elem<DT>::T* __restrict__ y) {
  typedef typename Elem<DT>::T E;
  constexpr int EPC = Elem<DT>::EPC, STEP = 4 * EPC, DEPTH = MT * NT >= 4 ? 2 : 4;
  typedef E vec __attribute__((ext_vector_type(EPC)));
  constexpr int OUT = 16 * NT, VALUES = OUT * 16 * MT, MINE = (VALUES + FEW_WAVES * 64 - 1) / (FEW_WAVES * 64);
  __shared__ f32x4 red[FEW_WAVES / 2][MT * NT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, q = lane >> 4;
  const long long n0 = (long long)blockIdx.x * OUT;
  // the low-rank term of this thread's outputs: row v / OUT, output n0 + v % OUT
  float thin[MINE];
#pragma unroll
  for (int t = 0; t < MINE; ++t) {
    thin[t] = 0.f;
    const int v = tid + t * FEW_WAVES * 64, r = v / OUT;
    const long long n = n0 + v % OUT;
    if (v >= VALUES || r >= M || n >= N) continue;
    const int a = wide ? adapter_of<long long>(groups, r, L) : adapter_of<int>(groups, r, L);
    if (a < 0) continue;
    const E* br = up + ((long long)a * N + n) * R;
    const float* hr = h + r * R;
    int j = 0;
    for (; j + EPC <= R; j += EPC) {
      const vec b = __builtin_bit_cast(vec, load16(br + j));
#pragma unroll
      for (int e = 0; e < EPC; e += 4) {
        const f32x4 hv = __builtin_bit_cast(f32x4, load16(hr + j + e));
#pragma unroll
        for (int k = 0; k < 4; ++k) thin[t] = fmaf(hv[k], (float)b[e + k], thin[t]);
      }
    }
    for (; j < R; ++j) thin[t] = fmaf(hr[j], (float)br[j], thin[t]);
  }
  const E* wr[NT];
  const E* xr[MT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const long long o = n0 + 16 * n + i;
    wr[n] = w + (o < N ? o : N - 1) * K;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) xr[m] = x + min(16 * m + i, M - 1) * ldx;
  f32x4 acc[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  // two sets of operands: the next turn's loads are in flight while a turn's products run (48 x 4096 -> 8192 bf16: 28.0 -> 24.7 us)
  struct Step {
    u32x4 w[DEPTH][NT], x[DEPTH][MT];
  };
  auto fetch = [&](Step& S, long long s0, auto depth, auto tail) {
#pragma unroll
    for (int d = 0; d < decltype(depth)::value; ++d) {
      const long long k = (s0 + (d >> 1) * 2 * FEW_WAVES + (d & 1)) * STEP + q * EPC;
#pragma unroll
      for (int n = 0; n < NT; ++n) S.w[d][n] = decltype(tail)::value ? load_tail<DT>(wr[n], k, K) : load16(wr[n] + k);
#pragma unroll
      for (int m = 0; m < MT; ++m) S.x[d][m] = decltype(tail)::value ? load_tail<DT>(xr[m], k, K) : load16(xr[m] + k);
    }
  };
  auto products = [&](const Step& S, auto depth) {
#pragma unroll
    for (int d = 0; d < decltype(depth)::value; ++d)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < Elem<DT>::INSTR; ++e) acc[m][n] = Elem<DT>::mma(S.w[d][n], S.x[d][m], acc[m][n], e);
  };
  auto walk = [&](long long s0, auto tail) {
    Step S;
    fetch(S, s0, Const<1>(), tail);
    products(S, Const<1>());
  };
  const long long steps = K / STEP;
  long long s = 2 * wave;
  const long long turn = DEPTH * FEW_WAVES, reach = (DEPTH - 2) * FEW_WAVES + 1;
  if (s + reach < steps) {
    Step S[2];
    fetch(S[0], s, Const<DEPTH>(), Const<0>());
    for (;;) {
      if (s + turn + reach >= steps) { products(S[0], Const<DEPTH>()); s += turn; break; }
      fetch(S[1], s + turn, Const<DEPTH>(), Const<0>());
      products(S[0], Const<DEPTH>());
      s += turn;
      if (s + turn + reach >= steps) { products(S[1], Const<DEPTH>()); s += turn; break; }
      fetch(S[0], s + turn, Const<DEPTH>(), Const<0>());
      products(S[1], Const<DEPTH>());
      s += turn;
    }
  }
  for (; s < steps; s += 2 * FEW_WAVES) {
    walk(s, Const<0>());
    if (s + 1 < steps) walk(s + 1, Const<0>());
  }
  if (steps * STEP < K && wave == (int)(steps % (2 * FEW_WAVES)) / 2) walk(steps, Const<1>());
  // 8 -> 4 -> 2 -> 1 waves
#pragma unroll
  for (int half = FEW_WAVES / 2; half; half >>= 1) {
    if (wave >= half && wave < 2 * half) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) red[wave - half][m * NT + n][lane] = acc[m][n];
    }
    __syncthreads();
    if (wave < half) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] += red[wave][m * NT + n][lane];
    }
    __syncthreads();
  }
  float* out = reinterpret_cast<float*>(red);      // [16 MT rows][OUT + 4]
  constexpr int LD = OUT + 4;
  static_assert(16 * MT * LD * 4 <= sizeof(red), "the sums fit where the waves' parts were");
  if (wave == 0) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int n = 0; n < NT; ++n) *reinterpret_cast<f32x4*>(out + (16 * m + i) * LD + 16 * n + 4 * q) = acc[m][n];
  }
  __syncthreads();
#pragma unroll
  for (int t = 0; t < MINE; ++t) {
    const int v = tid + t * FEW_WAVES * 64, r = v / OUT;
    const long long n = n0 + v % OUT;
    if (v >= VALUES || r >= M || n >= N) continue;
    float f = out[r * LD + v % OUT] + thin[t];
    if (bias) f += (float)bias[n];
    y[r * N + n] = (E)f;
  }
}

// ---------------------------------------------------------------------------------------------------------- gradients of A and B
// part[piece] = sum over the piece's positions p of Z[order[p]][c] * V[p][j]        (Z = x, V = u: dA;  Z = g, V = h: dB)
// The contraction runs over rows, so that v_mfma_f32_16x16x4_f32 takes its operands as they lie in memory: lane (i, q) loads
// columns 4i .. 4i+3 of row q of a group of four, element e being its operand for the block of columns 4i + e, and V[p][16n + i].
// Values of 16-bit types become fp32 on the way (h and u stay whole).  A workgroup owns 64 columns x 16*NJ ranks of a piece; its four waves
// take every fourth group of rows and are added through LDS, a quarter of the sums each.  What bounds it is the latency of Z's loads, so
// the next turn's rows are on their way while a turn's products run, and two waves a SIMD are asked for (with one, whose registers then hold
// more: rank 128, 8192 x (1024 + 1024) fp16, the whole backward 229 instead of 170 us).
// 4096 x (2048 + 2048) bf16, 12 adapters of rank 16: 18 us; 24000 x (688 + 256) fp32, rank 8: 27 us (91 MB).
// BY_RANK: part [piece][Rp][C] (operand order Z, V), else [piece][C][Rp] (V, Z): a lane ends with four values that lie together.
constexpr int TG_WAVES = 4, TG_COLS = 64, TG_DEPTH = 2;

struct GradJob {
  const void* Z;
  const float* V;
  float* part;
  void* out;
  long long ldz, C;
  int rows, blocks, by_rank;          // rows of a piece; workgroups along the columns (the sum's: outputs / 64)
};
struct GradJobs {
  GradJob j[2];
  const int32_t *offsets, *order;
  int L, R, Rp, ways;
};

template <int DT, int NJ, bool BY_RANK>
__device__ __forceinline__ void thin_grad(const GradJobs& G, const GradJob& J, int bx, f32x4 (*red)[4 * NJ][64]) {
  typedef typename Elem<DT>::T E;
  typedef E vec __attribute__((ext_vector_type(4)));
  const E* Z = static_cast<const E*>(J.Z);
  const float* V = J.V;
  const int32_t* order = G.order;
  float* part = J.part;
  const long long ldz = J.ldz, C = J.C;
  const int Rp = G.Rp;
  int a, p0, p1;
  if (!find_piece(G.offsets, G.L, J.rows, blockIdx.y, a, p0, p1)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const long long c = (long long)bx * TG_COLS + 4 * i;
  const int j0 = blockIdx.z * 16 * NJ;
  const bool whole = c + 4 <= C;
  f32x4 acc[4][NJ];
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int n = 0; n < NJ; ++n) acc[e][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  // two sets of operands: the next turn's rows are on their way while a turn's products run
  struct Rows {
    vec z[TG_DEPTH];
    float v[TG_DEPTH][NJ];
  };
  constexpr int TURN = 4 * TG_WAVES * TG_DEPTH;
  auto fetch = [&](Rows& S, int b) {
#pragma unroll
    for (int d = 0; d < TG_DEPTH; ++d) {
      const int p = b + 4 * TG_WAVES * d + q;
      const bool on = p < p1;
#pragma unroll
      for (int e = 0; e < 4; ++e) S.z[d][e] = (E)0.f;
#pragma unroll
      for (int n = 0; n < NJ; ++n) S.v[d][n] = on && j0 + 16 * n < Rp ? V[(long long)p * Rp + j0 + 16 * n + i] : 0.f;
      if (on) {
        const E* zr = Z + (long long)(order ? order[p] : p) * ldz + c;
        if (whole) {
          __builtin_memcpy(&S.z[d], zr, sizeof(vec));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < C) S.z[d][e] = zr[e];
        }
      }
    }
  };
  auto products = [&](const Rows& S) {
#pragma unroll
    for (int d = 0; d < TG_DEPTH; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < NJ; ++n)
          acc[e][n] = BY_RANK ? __builtin_amdgcn_mfma_f32_16x16x4f32((float)S.z[d][e], S.v[d][n], acc[e][n], 0, 0, 0)
                              : __builtin_amdgcn_mfma_f32_16x16x4f32(S.v[d][n], (float)S.z[d][e], acc[e][n], 0, 0, 0);
  };
  {
    Rows S[2];
    int b = p0 + 4 * wave;
    fetch(S[0], b);
    for (; b < p1; b += 2 * TURN) {
      fetch(S[1], b + TURN);
      products(S[0]);
      if (b + TURN >= p1) break;
      fetch(S[0], b + 2 * TURN);
      products(S[1]);
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int n = 0; n < NJ; ++n) red[wave][e * NJ + n][lane] = acc[e][n];
  __syncthreads();
  // every wave adds and stores a quarter
  const long long base = (long long)blockIdx.y * Rp * C, c0 = (long long)bx * TG_COLS;
#pragma unroll
  for (int n = 0; n < NJ; ++n) {
    if (j0 + 16 * n >= Rp) break;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (BY_RANK) {      // register r of block e: column 16q + 4r + e of rank 16n + i; this wave's r is its number
#pragma unroll
      for (int w = 0; w < TG_WAVES; ++w)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += red[w][e * NJ + n][lane][wave];
      const long long col = c0 + 16 * q + 4 * wave;
      float* o = part + base + (long long)(j0 + 16 * n + i) * C + col;
      if (col + 4 <= C) {
        store16(o, __builtin_bit_cast(u32x4, v));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < C) o[e] = v[e];
      }
    } else {            // register r of block e: rank 16n + 4q + r of column 4i + e; this wave's e is its number
#pragma unroll
      for (int w = 0; w < TG_WAVES; ++w) v += red[w][wave * NJ + n][lane];
      if (c + wave < C) *reinterpret_cast<f32x4*>(part + base + (c + wave) * Rp + j0 + 16 * n + 4 * q) = v;
    }
  }
}

template <int DT, int NJ>
__global__ void __launch_bounds__(TG_WAVES * 64, 2) k_thin_grad(GradJobs G) {
  __shared__ f32x4 red[TG_WAVES][4 * NJ][64];
  const int second = (int)blockIdx.x >= G.j[0].blocks;
  const GradJob& J = G.j[second];
  const int bx = (int)blockIdx.x - (second ? G.j[0].blocks : 0);
  if (J.by_rank) thin_grad<DT, NJ, true>(G, J, bx, red);
  else thin_grad<DT, NJ, false>(G, J, bx, red);
}

// adds an adapter's pieces in their order; many pieces an adapter (ways = 4): wave w those of q = w mod 4, then the four sums.
// BY_RANK: out[i][j][c] (dA), else out[i][c][j] (dB).  Adapters without rows get zeros.  4096 x (2048 + 2048), 12 adapters of rank 16: 7 us.
template <int DT>
__global__ void __launch_bounds__(256) k_thin_grad_sum(GradJobs G) {
  typedef typename Elem<DT>::T E;
  __shared__ float red[4][64];
  const int second = (int)blockIdx.x >= G.j[0].blocks;
  const GradJob& J = G.j[second];
  const int bx = (int)blockIdx.x - (second ? G.j[0].blocks : 0), rows = J.rows;
  const int a = blockIdx.y, lane = threadIdx.x & 63;
  int first = 0;
  for (int b = lane; b < a; b += 64) first += (G.offsets[b + 1] - G.offsets[b] + rows - 1) / rows;
#pragma unroll
  for (int d = 32; d; d >>= 1) first += __shfl_xor(first, d);
  const int n = (G.offsets[a + 1] - G.offsets[a] + rows - 1) / rows;
  const long long all = J.C * G.R, stride = J.C * G.Rp;
  E* out = static_cast<E*>(J.out) + a * all;
  const int ways = G.ways, outs = 256 / ways, w = ways == 1 ? 0 : threadIdx.x >> 6, mine = ways == 1 ? threadIdx.x : lane;
  for (long long e0 = (long long)bx * outs; e0 < all; e0 += (long long)J.blocks * outs) {
    const long long e = e0 + mine;
    float v = 0.f;
    if (e < all) {
      const float* src = J.part + first * stride + (J.by_rank ? e : e / G.R * G.Rp + e % G.R);
#pragma unroll 4
      for (int q = w; q < n; q += ways) v += src[q * stride];
    }
    if (ways == 1) {
      if (e < all) out[e] = (E)v;
      continue;
    }
    __syncthreads();
    red[w][lane] = v;
    __syncthreads();
    if (w == 0 && e < all) out[e] = (E)(red[0][lane] + red[1][lane] + (red[2][lane] + red[3][lane]));
  }
}

// ------------------------------------------------------------------------------------------------------------------- transposes
struct TransposeJob {
  const void* in;
  void* out;
  long long rows, cols, batch, tiles, tiles_c;   // in [batch][rows][cols] -> out [batch][cols][ldo], zeros behind the rows
  long long ldo;
};
struct TransposeJobs {
  TransposeJob j[3];
};

// 64 x 64 values a workgroup through LDS, 16 bytes a lane on both sides where the rows allow it.  HBM- and latency-bound: W 2048 x 2048
// and twelve pairs of rank 16, bf16: 6.6 us.
template <typename U>
__global__ void __launch_bounds__(256) k_transpose(TransposeJobs J) {
  constexpr int V = 16 / sizeof(U);
  typedef U vec __attribute__((ext_vector_type(V)));
  __shared__ U t[64][64 + 2];
  long long b = blockIdx.x;
  int k = 0;
  while (k < 2 && b >= J.j[k].tiles * J.j[k].batch) b -= J.j[k].tiles * J.j[k].batch, ++k;
  const TransposeJob& T = J.j[k];
  const U* in = static_cast<const U*>(T.in) + b / T.tiles * T.rows * T.cols;
  U* out = static_cast<U*>(T.out) + b / T.tiles * T.ldo * T.cols;
  const long long r0 = b % T.tiles / T.tiles_c * 64, c0 = b % T.tiles % T.tiles_c * 64;
  constexpr int LANES = 64 / V;      // lanes of a row
  const int x = threadIdx.x % LANES * V;
  for (int r = threadIdx.x / LANES; r < 64; r += 256 / LANES) {
    if (r0 + r >= T.rows) break;
    const U* src = in + (r0 + r) * T.cols + c0 + x;
    if (c0 + x + V <= T.cols) {
      vec v;
      __builtin_memcpy(&v, src, 16);
#pragma unroll
      for (int e = 0; e < V; ++e) t[r][x + e] = v[e];
    } else {
      for (int e = 0; e < V; ++e)
        if (c0 + x + e < T.cols) t[r][x + e] = src[e];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x / LANES; c < 64; c += 256 / LANES) {
    if (c0 + c >= T.cols) break;
    U* dst = out + (c0 + c) * T.ldo + r0 + x;
    if (r0 + x + V <= T.rows) {
      vec v;
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = t[x + e][c];
      __builtin_memcpy(dst, &v, 16);
    } else {
      for (int e = 0; e < V; ++e)
        if (r0 + x + e < T.ldo) dst[e] = r0 + x + e < T.rows ? t[x + e][c] : (U)0;
    }
  }
}

// rows with zeros behind them up to a multiple of 128 bytes, 16-byte aligned: what k_main's direct loads want.  HBM-bound: x 8192 x 4097 and
// W 4096 x 4097 bf16 36 us (202 MB, 5.6 TB/s).
struct PadJob {
  const void* in;
  void* out;
  long long rows, ld;
};
template <int DT>
__global__ void __launch_bounds__(256) k_pad(PadJob a, PadJob b, long long K, long long Kp) {
  typedef typename Elem<DT>::T E;
  constexpr int EPC = Elem<DT>::EPC;
  const unsigned line = (unsigned)(Kp / EPC);
  const long long first = a.rows * line, all = first + b.rows * line;
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < all; t += (long long)gridDim.x * 256) {
    const bool two = t >= first;
    const long long u = two ? t - first : t;
    const long long r = u / line, k = (u - r * line) * EPC;
    const E* src = static_cast<const E*>(two ? b.in : a.in) + r * (two ? b.ld : a.ld);
    *reinterpret_cast<u32x4*>(static_cast<E*>(two ? b.out : a.out) + r * Kp + k) = load_tail<DT>(src, k, K);
  }
}

// ---------------------------------------------------------------------------------------------------------------------- launchers
template <int DT, int BM, int BN, int WM, int WN, bool DIRECT, int NS = 2>
static int run_main(const MainArgs& P, hipStream_t st) {
  static unsigned long long done = 0;
  constexpr int bytes = NS * (BM + BN) * 128;
  const auto kernel = k_main<DT, BM, BN, WM, WN, NS, DIRECT>;
  ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), bytes, &done);
  kernel<<<(unsigned)((P.M + BM - 1) / BM * ((P.N + BN - 1) / BN) * P.splits), WM * WN * 64, bytes, st>>>(P);
  const int rc = check_launch("k_main");
  if (rc || P.splits == 1) return rc;
  typedef typename Elem<DT>::T E;
  const long long all = P.M * P.N;
  k_sum_parts<DT><<<(unsigned)((all + 1023) / 1024), 256, 0, st>>>(P.part, P.splits, all, P.N, static_cast<const E*>(P.bias), static_cast<E*>(P.y));
  return check_launch("k_sum_parts");
}

// Less than one 64 x 64 tile a CU leaves CUs idle and their few waves waiting: the contraction is split until there are 512 workgroups,
// eight stages each at least (128 x 4096 x 4096 bf16: 128 tiles 48 us, 512 workgroups and the sum 35; 256 tiles and more do not gain)
static int split_of(int dtype, long long M, long long K, long long N) {
  const long long tiles = (M + 63) / 64 * ((N + 63) / 64), stages = (K + (dtype == ANERF_F32 ? 31 : 63)) / (dtype == ANERF_F32 ? 32 : 64);
  if (tiles == 0 || tiles >= 256) return 1;
  const long long s = 512 / tiles < stages / 8 ? 512 / tiles : stages / 8;
  return s < 2 ? 1 : s > 16 ? 16 : (int)s;
}

// Tile: the larger, the fewer LDS reads a product (a 256 x 256 tile's waves read 3/8 of what a 64 x 64 tile's do), but the tiles of one CU
// run one after the other, and what the last round leaves idle grows.  Cost: tiles of the busiest CU x size / rate; the rates are
// what the tiles reach where there are many of them, relative to 256 x 128 (bf16, 8192 x 4096 x 4096, rank 8: 256 x 256 271 us, 256 x 128 307,
// 128 x 128 310, 128 x 64 360, 64 x 64 432; 1000 x 1000 x 1000: 45, 29, 25, 19, 16), times what they reach with one or two tiles a CU, whose
// few waves do not hide their waits.  There the contraction is four stages deep in LDS, three of them in flight (bf16, 4096 inputs, 8192
// outputs, two deep -> four deep: 128 rows on 64 x 64 52 -> 28 us, 256 rows 53 -> 41, 512 rows on 128 x 128 63 -> 50); with more tiles a CU two
// stages leave room for more workgroups, and the larger tiles gain nothing from a third.  fp32 is bound by its products: one size is as
// fast as the other (1941 .. 2009 us), and four stages help one tile a CU only (128 x 4096 -> 8192: 99 -> 83 us, 1024 x 2048 -> 2048: 69 -> 71).
template <int DT>
static int launch_main(const MainArgs& P, hipStream_t st) {
  constexpr long long es = sizeof(typename Elem<DT>::T), span = 1ll << 32;      // DIRECT's offsets have 32 bits
  const bool direct = (((uintptr_t)P.x | (uintptr_t)P.w) & 15) == 0 && P.K % Elem<DT>::EPC == 0 && P.ldx % Elem<DT>::EPC == 0 &&
                      P.ldw % Elem<DT>::EPC == 0 && P.M * P.ldx * es < span && P.N * P.ldw * es < span;
  constexpr bool F32 = DT == ANERF_F32;
  auto a_cu = [&](int bm, int bn) { return ((P.M + bm - 1) / bm * ((P.N + bn - 1) / bn) * P.splits + 255) / 256; };      // tiles of the busiest CU
  auto cost = [&](int bm, int bn, double rate, double one, double two) {
    const long long mine = a_cu(bm, bn);
    return (double)mine * bm * bn / (rate * (mine == 1 ? one : mine == 2 ? two : 1.0));
  };
  const double c64 = F32 ? cost(64, 64, 0.97, 0.7, 1.0) : cost(64, 64, 0.6, 0.55, 0.8);
  const double c128 = F32 ? cost(128, 128, 1.0, 0.7, 1.0) : cost(128, 128, 0.87, 0.85, 1.0);
  const bool deep = a_cu(64, 64) <= (F32 ? 1 : 2);
  auto run64 = [&]() { return deep ? run_main<DT, 64, 64, 2, 2, true, 4>(P, st) : run_main<DT, 64, 64, 2, 2, true>(P, st); };
  if (P.splits > 1 || !direct || F32) {
    const bool small = P.splits > 1 || c64 <= c128;
    if (direct) return small ? run64() : run_main<DT, 128, 128, 2, 2, true>(P, st);
    return small ? run_main<DT, 64, 64, 2, 2, false>(P, st) : run_main<DT, 128, 128, 2, 2, false>(P, st);
  }
  if constexpr (!F32) {
    const double c96 = cost(128, 64, 0.75, 0.6, 0.8), c192 = cost(256, 128, 0.97, 1.0, 1.0), c256 = cost(256, 256, 1.05, 1.0, 1.0);
    const double least = fmin(fmin(fmin(c64, c128), c96), fmin(c192, c256));
    if (c256 == least) return run_main<DT, 256, 256, 2, 4, true>(P, st);
    if (c192 == least) return run_main<DT, 256, 128, 4, 2, true>(P, st);
    if (c128 == least) return a_cu(128, 128) == 1 ? run_main<DT, 128, 128, 2, 2, true, 4>(P, st) : run_main<DT, 128, 128, 2, 2, true>(P, st);
    if (c96 < c64) return run_main<DT, 128, 64, 2, 2, true>(P, st);
  }
  return run64();
}

// what k_thin leaves, in one buffer: h fp32 [n_rows][Rp] | operand form [n_rows][split_width] (16-bit types) | factor [n_rows] (fp16) | the positions'
// adapters [n_rows]; byte offsets
struct HLayout {
  int Rp;
  long long split, factor, owner, bytes;
};
static HLayout h_layout(const AnerfAdapterIO& A) {
  HLayout H;
  H.Rp = (A.rank + 15) / 16 * 16;
  const long long part = A.n_rows * H.Rp * 4, line = (A.n_rows + 3) / 4 * 16;
  H.split = part;
  H.factor = A.dtype == ANERF_F32 ? part : part + A.n_rows * 2 * (A.dtype == ANERF_BF16 ? split_width<ANERF_BF16>(H.Rp) : split_width<ANERF_F16>(H.Rp));
  H.owner = H.factor + (A.dtype == ANERF_F16 ? line : 0);
  H.bytes = H.owner + line;
  return H;
}
long long adapter_h_bytes(const AnerfAdapterIO& A) { return h_layout(A).bytes; }
// Rows that cannot be loaded 16 bytes aligned go through registers and smaller tiles (8192 x 4097 x 4096 bf16: 473 us, 4096: 302).  With
// enough outputs a row and rows an output a copy with padded rows costs less (one pass over x and W; from about 1200 of each).
// The width of the copies, 0: none.  ldw > n_in: W's rows lie padded already.
static long long padded_width(const AnerfAdapterIO& A, long long ldw) {
  const long long es = A.dtype == ANERF_F32 ? 4 : 2, epc = 16 / es, Kp = (A.n_in + 8 * epc - 1) / (8 * epc) * (8 * epc);
  const bool odd = A.n_in % epc || A.x_stride % epc || (((uintptr_t)A.x | (uintptr_t)A.weight) & 15);
  if (!odd || A.n_rows < 1280 || A.n_out < 1280 || A.n_in < 256) return 0;
  if (A.n_rows * Kp * es >= (1ll << 32) || A.n_out * Kp * es >= (1ll << 32)) return 0;
  return ldw > A.n_in && ldw != Kp ? 0 : Kp;
}

long long adapter_workspace(const AnerfAdapterIO& A) {
  const int splits = split_of(A.dtype, A.n_rows, A.n_in, A.n_out);
  if (splits > 1) return splits * A.n_rows * A.n_out * 4;
  return padded_width(A, A.n_in) * (A.n_rows + A.n_out) * (A.dtype == ANERF_F32 ? 4 : 2);
}

template <int DT>
static int linear_t(const AnerfAdapterIO& A, long long ldw, void* ws, hipStream_t st) {
  typedef typename Elem<DT>::T E;
  const HLayout H = h_layout(A);
  // pieces of 16 rows while there is at most one for a CU: what bounds few pieces is what one CU can load
  const long long small = pieces_bound(A.n_rows, A.n_adapters, 16), pieces = small <= 256 ? small : pieces_bound(A.n_rows, A.n_adapters, 32);
  const int Rp = H.Rp;
  float* h = reinterpret_cast<float*>(A.h);
  E* split = reinterpret_cast<E*>(static_cast<char*>(A.h) + H.split);
  float* factor = reinterpret_cast<float*>(static_cast<char*>(A.h) + H.factor);
  int32_t* owner = reinterpret_cast<int32_t*>(static_cast<char*>(A.h) + H.owner);
  auto thin = [&](auto kernel, int parts) {
    kernel<<<dim3((unsigned)pieces, parts), TH_WAVES * 64, 0, st>>>(static_cast<const E*>(A.x), A.x_stride, A.order, static_cast<const E*>(A.down), A.offsets,
                                                                  A.n_adapters, A.n_in, A.rank, Rp, A.scale_of, A.scale, h, split, factor, owner);
  };
  if (Rp <= 16) small <= 256 ? thin(k_thin<DT, 1, 1>, 1) : thin(k_thin<DT, 1, 2>, 1);
  else if (Rp <= 32) small <= 256 ? thin(k_thin<DT, 2, 1>, 1) : thin(k_thin<DT, 2, 2>, 1);
  else small <= 256 ? thin(k_thin<DT, 4, 1>, (Rp + 63) / 64) : thin(k_thin<DT, 4, 2>, (Rp + 63) / 64);
  if constexpr (DT == ANERF_F16) {
    if (A.y && Rp > 64) k_split_rows<<<(unsigned)((A.n_rows + 15) / 16), 256, 0, st>>>(h, A.offsets + A.n_adapters, Rp, split, factor);
  }
  const int rc = check_launch("k_thin");
  if (rc || !A.y) return rc;       // (the gradient of A alone needs h only)
  const void* operand = split;
  if constexpr (DT == ANERF_F32) operand = h;
  MainArgs P = {A.x, A.weight, A.bias, A.up, A.offsets, A.order, operand, factor, h, owner, A.y, static_cast<float*>(ws), A.x_stride, ldw, A.n_in, A.n_out,
                A.n_rows, A.n_adapters, A.rank, Rp, split_of(DT, A.n_rows, A.n_in, A.n_out)};
  if (const long long Kp = padded_width(A, ldw)) {
    char* w = static_cast<char*>(ws);
    const bool w_lies = ldw == Kp && ((uintptr_t)A.weight & 15) == 0;
    PadJob jx = {A.x, w, A.n_rows, A.x_stride}, jw = {A.weight, w + A.n_rows * Kp * (long long)sizeof(E), w_lies ? 0 : A.n_out, ldw};
    k_pad<DT><<<2048, 256, 0, st>>>(jx, jw, A.n_in, Kp);
    const int rc = check_launch("k_pad");
    if (rc) return rc;
    P.x = jx.out, P.ldx = Kp;
    if (!w_lies) P.w = jw.out;
    P.ldw = P.K = Kp;
  }
  return launch_main<DT>(P, st);
}

int launch_adapter_linear(const AnerfAdapterIO& A, void* ws, hipStream_t st) {
  switch (A.dtype) {
    case ANERF_F32: return linear_t<ANERF_F32>(A, A.n_in, ws, st);
    case ANERF_BF16: return linear_t<ANERF_BF16>(A, A.n_in, ws, st);
    default: return linear_t<ANERF_F16>(A, A.n_in, ws, st);
  }
}

template <int DT>
static int few_t(const AnerfAdapterIO& A, const void* groups, int wide, hipStream_t st) {
  typedef typename Elem<DT>::T E;
  const E* x = static_cast<const E*>(A.x);
  const int M = (int)A.n_rows;
  float* h = static_cast<float*>(A.h);
  k_few_thin<DT><<<dim3(M, (A.rank + 3) / 4), 256, 0, st>>>(x, A.x_stride, static_cast<const E*>(A.down), groups, wide, A.n_adapters, A.n_in, A.rank,
                                                           A.scale_of, A.scale, h);
  int rc = check_launch("k_few_thin");
  if (rc) return rc;
  auto run = [&](auto kernel, int out) {
    kernel<<<(unsigned)((A.n_out + out - 1) / out), FEW_WAVES * 64, 0, st>>>(x, A.x_stride, static_cast<const E*>(A.weight), static_cast<const E*>(A.bias),
                                                                          static_cast<const E*>(A.up), groups, wide, A.n_adapters, M, A.n_in, A.n_out,
                                                                          A.rank, h, static_cast<E*>(A.y));
  };
  // 32 outputs a workgroup halve what x costs in L2 traffic, where they still fill the chip
  const bool wide_out = A.n_out >= 8192;
  if (M <= 16) wide_out ? run(k_few<DT, 1, 2>, 32) : run(k_few<DT, 1, 1>, 16);
  else if (M <= 32) wide_out ? run(k_few<DT, 2, 2>, 32) : run(k_few<DT, 2, 1>, 16);
  else if (M <= 48) wide_out ? run(k_few<DT, 3, 2>, 32) : run(k_few<DT, 3, 1>, 16);
  else wide_out ? run(k_few<DT, 4, 2>, 32) : run(k_few<DT, 4, 1>, 16);
  return check_launch("k_few");
}

int launch_adapter_few(const AnerfAdapterIO& A, const void* groups, int wide, hipStream_t st) {
  switch (A.dtype) {
    case ANERF_F32: return few_t<ANERF_F32>(A, groups, wide, st);
    case ANERF_BF16: return few_t<ANERF_BF16>(A, groups, wide, st);
    default: return few_t<ANERF_F16>(A, groups, wide, st);
  }
}

// rows of a piece of k_thin_grad: 64 at least, since a piece writes C x Rp floats, and so many that there are about 1024 workgroups -- 512 with
// more than 32 ranks, whose sums weigh more (whole backward of 8192 x (2048 + 2048), rank 64: 225 -> 214 us; rank 16: 324 -> 333)
static int grad_ranks(int Rp) { return Rp <= 16 ? 1 : Rp <= 32 ? 2 : 4; }
static int grad_rows(long long M, long long C, int Rp) {
  const long long blocks = (C + TG_COLS - 1) / TG_COLS * ((Rp + 16 * grad_ranks(Rp) - 1) / (16 * grad_ranks(Rp)));
  const long long want = grad_ranks(Rp) == 4 ? 512 : 1024, pieces = (want + blocks - 1) / blocks;
  const long long rows = ((M + pieces - 1) / pieces + 63) / 64 * 64;
  return (int)(rows < 64 ? 64 : rows);
}

static long long part_floats(long long M, int L, long long C, int Rp) {
  const int rows = grad_rows(M, C, Rp);
  return pieces_bound(M, L, rows) * Rp * C;
}

static AnerfAdapterIO swapped(const AnerfAdapterIO& A) {      // sizes of the product that dx is
  AnerfAdapterIO T = A;
  T.n_in = A.n_out, T.n_out = A.n_in;
  T.x = nullptr, T.weight = nullptr, T.x_stride = 1;      // (not known yet: the worst case where sizes are asked for)
  return T;
}
struct BackwardPlan {
  long long wt_ld, wt, dt, ut, u, part, bytes;     // row length of W^T; byte offsets in the workspace; the parts of dx's product and those of dA, dB share `part`
};
static BackwardPlan backward_plan(const AnerfAdapterIO& A) {
  const long long es = A.dtype == ANERF_F32 ? 4 : 2;
  const int Rp = (A.rank + 15) / 16 * 16;
  auto up16 = [](long long b) { return (b + 255) / 256 * 256; };
  BackwardPlan B;
  long long at = 0;
  B.wt_ld = padded_width(swapped(A), A.n_out);
  if (!B.wt_ld) B.wt_ld = A.n_out;
  B.wt = at, at += up16(A.n_in * B.wt_ld * es);
  B.dt = at, at += up16((long long)A.n_adapters * A.rank * A.n_in * es);
  B.ut = at, at += up16((long long)A.n_adapters * A.rank * A.n_out * es);
  B.u = at, at += up16(h_layout(A).bytes);
  const long long pa = part_floats(A.n_rows, A.n_adapters, A.n_in, Rp), pb = part_floats(A.n_rows, A.n_adapters, A.n_out, Rp);
  const long long pd = adapter_workspace(swapped(A));
  B.part = at, at += up16(std::max((pa + pb) * 4 + 512, pd));
  B.bytes = at;
  return B;
}
long long adapter_backward_workspace(const AnerfAdapterIO& A) { return backward_plan(A).bytes; }

// both sums of an adapter's gradient in one launch each (job 0: dA from (x, u), job 1: dB from (g, h); one of them may be off)
template <int DT>
static int thin_grads(const AnerfAdapterIO& A, const AnerfAdapterGradIO& G, const float* u, float* part, hipStream_t st) {
  const int Rp = (A.rank + 15) / 16 * 16, nj = grad_ranks(Rp);
  GradJobs J = {};
  J.offsets = A.offsets, J.order = A.order, J.L = A.n_adapters, J.R = A.rank, J.Rp = Rp;
  int n = 0;
  long long pieces = 0;
  auto add = [&](const void* Z, long long ldz, const float* V, long long C, void* out, int by_rank) {
    const int rows = grad_rows(A.n_rows, C, Rp);
    const long long mine = pieces_bound(A.n_rows, A.n_adapters, rows);
    J.j[n++] = {Z, V, part, out, ldz, C, rows, (int)((C + TG_COLS - 1) / TG_COLS), by_rank};
    part += (mine * Rp * C + 63) / 64 * 64;
    pieces = std::max(pieces, mine);
  };
  if (G.ddown) add(A.x, A.x_stride, u, A.n_in, G.ddown, 1);
  if (G.dup) add(G.g, G.g_stride, static_cast<const float*>(A.h), A.n_out, G.dup, 0);
  if (n == 0) return ANERF_OK;
  if (pieces > 0) {
    const dim3 grid((unsigned)(J.j[0].blocks + J.j[1].blocks), (unsigned)pieces, (Rp + 16 * nj - 1) / (16 * nj));
    if (nj == 1) k_thin_grad<DT, 1><<<grid, TG_WAVES * 64, 0, st>>>(J);
    else if (nj == 2) k_thin_grad<DT, 2><<<grid, TG_WAVES * 64, 0, st>>>(J);
    else k_thin_grad<DT, 4><<<grid, TG_WAVES * 64, 0, st>>>(J);
    const int rc = check_launch("k_thin_grad");
    if (rc) return rc;
  }
  J.ways = pieces > 8ll * A.n_adapters ? 4 : 1;
  const long long most = std::max(1, 4096 / A.n_adapters), outs = 256 / J.ways;
  for (int k = 0; k < n; ++k) J.j[k].blocks = (int)std::min((J.j[k].C * A.rank + outs - 1) / outs, most);
  k_thin_grad_sum<DT><<<dim3((unsigned)(J.j[0].blocks + J.j[1].blocks), A.n_adapters), 256, 0, st>>>(J);
  return check_launch("k_thin_grad_sum");
}

template <int DT>
static int backward_t(const AnerfAdapterIO& A, const AnerfAdapterGradIO& G, char* ws, hipStream_t st) {
  typedef typename Elem<DT>::T E;
  const BackwardPlan B = backward_plan(A);
  float* u = reinterpret_cast<float*>(ws + B.u);
  float* part = reinterpret_cast<float*>(ws + B.part);
  if (A.n_rows > 0 && (G.dx || G.ddown)) {
    // dx = the forward product of (g, W^T, B^T, A^T); its low-rank middle u is what dA needs
    auto job = [](const void* in, void* out, long long rows, long long cols, long long batch, long long ldo) {
      TransposeJob t = {in, out, rows, cols, batch, (rows + 63) / 64 * ((cols + 63) / 64), (cols + 63) / 64, ldo};
      return t;
    };
    AnerfAdapterIO T = swapped(A);
    T.x = G.g, T.x_stride = G.g_stride, T.weight = ws + B.wt, T.bias = nullptr, T.down = ws + B.ut, T.up = ws + B.dt, T.y = G.dx, T.h = ws + B.u;
    const long long Kp = padded_width(T, A.n_out), ldw = Kp ? Kp : A.n_out;
    TransposeJobs J;
    J.j[0] = job(A.weight, ws + B.wt, A.n_out, A.n_in, G.dx ? 1 : 0, ldw);
    J.j[1] = job(A.down, ws + B.dt, A.rank, A.n_in, G.dx ? A.n_adapters : 0, A.rank);
    J.j[2] = job(A.up, ws + B.ut, A.n_out, A.rank, A.n_adapters, A.n_out);
    long long blocks = 0;
    for (int k = 0; k < 3; ++k) blocks += J.j[k].tiles * J.j[k].batch;
    if constexpr (DT == ANERF_F32) k_transpose<uint32_t><<<(unsigned)blocks, 256, 0, st>>>(J);
    else k_transpose<uint16_t><<<(unsigned)blocks, 256, 0, st>>>(J);
    int rc = check_launch("k_transpose");
    if (rc) return rc;
    rc = linear_t<DT>(T, ldw, ws + B.part, st);
    if (rc) return rc;
  }
  return thin_grads<DT>(A, G, u, part, st);
}

int launch_adapter_backward(const AnerfAdapterIO& A, const AnerfAdapterGradIO& G, void* ws, hipStream_t st) {
  char* w = static_cast<char*>(ws);
  switch (A.dtype) {
    case ANERF_F32: return backward_t<ANERF_F32>(A, G, w, st);
    case ANERF_BF16: return backward_t<ANERF_BF16>(A, G, w, st);
    default: return backward_t<ANERF_F16>(A, G, w, st);
  }
}

}  // namespace anerf
