// anerf_adapter.hip -- a shared projection with a low-rank adapter of its own for every row (gfx950):
//     y[r] = x[r] W^T + b + s_i (x[r] A_i^T) B_i^T          i = the row's adapter, none: the shared projection alone
// and its gradients with W and b frozen:
//     u[r] = g[r] B_i,  dx = g W + s_i u A_i,  dA_i = s_i sum_r u[r]^T x[r],  dB_i = s_i sum_r g[r]^T h[r],  h[r] = x[r] A_i^T
// Rows are walked in the order of their adapter (positions p; order[p] = row, NULL = rows lie in that order already), adapter i
// owning positions offsets[i] .. offsets[i+1]-1; the rows behind offsets[L] have no adapter.
//   k_thin       h[p] = x[order[p]] A_i^T: one workgroup a piece of 32 positions of one adapter
//   k_main       x W^T tile by tile; a tile starts with the low-rank term of the adapters whose positions it holds
//   k_thin_grad  dA_i / dB_i as sums over pieces of an adapter's positions, k_thin_grad_sum adds the pieces in order
//   k_transpose  W, A, B with their last two axes swapped: dx is then the forward product of (g, W^T, B^T, A^T)
#include "anerf_rows.h"

namespace anerf {

// ---------------------------------------------------------------------------------------------------------------- h = x A^T
// HBM-bound on x.  The four waves split the contraction (every fourth 64-byte step), each holding all 32 rows x 16*NJ ranks of the
// piece in MFMA accumulators, fed straight from memory: a row of A serves 32 rows of x, and nothing is read twice from HBM.
constexpr int TH_ROWS = 32, TH_WAVES = 4;

template <int DT, int NJ>
__global__ void __launch_bounds__(TH_WAVES * 64) k_thin(const typename Elem<DT>::T* __restrict__ x, long long ldx, const int32_t* __restrict__ order,
                                                        const typename Elem<DT>::T* __restrict__ down, const int32_t* __restrict__ offsets,
                                                        int L, long long K, int R, int Rp, float* __restrict__ h) {
  typedef typename Elem<DT>::T E;
  constexpr int EPC = Elem<DT>::EPC, STEP = 4 * EPC;
  __shared__ f32x4 red[TH_WAVES][2 * NJ][64];
  int a, p0, p1;
  if (!find_piece(offsets, L, TH_ROWS, blockIdx.x, a, p0, p1)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int j0 = blockIdx.y * 16 * NJ;
  const E* A = down + (long long)a * R * K;
  const E* xr[2];
  const E* ar[NJ];
#pragma unroll
  for (int m = 0; m < 2; ++m) {
    const int p = min(p0 + 16 * m + i, p1 - 1);      // rows behind the piece repeat its last one; their sums are not stored
    xr[m] = x + (long long)(order ? order[p] : p) * ldx;
  }
#pragma unroll
  for (int n = 0; n < NJ; ++n) ar[n] = A + (long long)min(j0 + 16 * n + i, R - 1) * K;
  f32x4 acc[2][NJ];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < NJ; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  const long long steps = K / STEP;
#pragma unroll 4
  for (long long s = wave; s < steps; s += TH_WAVES) {
    const long long k = s * STEP + q * EPC;
    u32x4 xv[2], av[NJ];
#pragma unroll
    for (int m = 0; m < 2; ++m) xv[m] = load16(xr[m] + k);
#pragma unroll
    for (int n = 0; n < NJ; ++n) av[n] = load16(ar[n] + k);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NJ; ++n) acc[m][n] = Elem<DT>::mma(av[n], xv[m], acc[m][n]);
  }
  if (steps * STEP < K && wave == (int)(steps % TH_WAVES)) {
    const long long k = steps * STEP + q * EPC;
    u32x4 xv[2], av[NJ];
#pragma unroll
    for (int m = 0; m < 2; ++m) xv[m] = load_tail<DT>(xr[m], k, K);
#pragma unroll
    for (int n = 0; n < NJ; ++n) av[n] = load_tail<DT>(ar[n], k, K);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int n = 0; n < NJ; ++n) acc[m][n] = Elem<DT>::mma(av[n], xv[m], acc[m][n]);
  }
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int n = 0; n < NJ; ++n) red[wave][m * NJ + n][lane] = acc[m][n];
  __syncthreads();
  for (int f = wave; f < 2 * NJ; f += TH_WAVES) {
    f32x4 v = red[0][f][lane];
#pragma unroll
    for (int w = 1; w < TH_WAVES; ++w) v += red[w][f][lane];
    const int p = p0 + 16 * (f / NJ) + i, j = j0 + 16 * (f % NJ) + 4 * q;
    if (p < p1 && j < Rp) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j + e >= R) v[e] = 0.f;                   // ranks of the padding: zero
      *reinterpret_cast<f32x4*>(h + (long long)p * Rp + j) = v;
    }
  }
}

// ------------------------------------------------------------------------------------------------- one h operand of the low-rank term
// Lane (i, q) wants 16 bytes of its row's h against chunk c of B.  fp32: elements 16c + 4q ...  16-bit types: h is split into the
// nearest value hi and the rest lo, [hi of 16 ranks | lo of the same 16] making one 32-wide step against [B | B], so that h keeps
// 16 (bf16) or 21 (fp16) of its bits; fp16's range does not hold every h, so a row of h is first divided by a power of two.
template <int DT>
__device__ __forceinline__ u32x4 h_operand(const float* __restrict__ hr, int c, int q, float down_scale) {
  if constexpr (DT == ANERF_F32) {
    return __builtin_bit_cast(u32x4, *reinterpret_cast<const f32x4*>(hr + 16 * c + 4 * q));
  } else {
    typedef typename Elem<DT>::T E;
    typedef E vec __attribute__((ext_vector_type(8)));
    vec v;
    const float* s = hr + 16 * c + 8 * (q & 1);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = s[e] * down_scale;
      const E hi = (E)f;
      const float rest = f - (float)hi;
      v[e] = q < 2 ? hi : (E)(__builtin_isfinite(f) && __builtin_isfinite((float)hi) ? rest : 0.f);
    }
    return __builtin_bit_cast(u32x4, v);
  }
}

template <int DT>
__device__ __forceinline__ u32x4 b_operand(const typename Elem<DT>::T* __restrict__ br, int c, int q, int R) {
  const int j = 16 * c + (DT == ANERF_F32 ? 4 * q : 8 * (q & 1));
  return load_tail<DT>(br, j, R);
}

// ------------------------------------------------------------------------------------------------------------------ y = x W^T ...
// BM positions x BN outputs a workgroup, 2 x 2 waves, 16x16 MFMA blocks with W's rows as the first operand, so that a lane ends
// with four consecutive outputs of one row.  The contraction goes through LDS 128 bytes of every row at a time, double-buffered; 16-byte
// chunk c of row r lies at chunk c ^ (r & 7), which spreads a fragment read over the banks.
// The low-rank term comes first: for every adapter with positions in the tile, h B_i^T is formed in accumulators of its own and taken
// over by that adapter's rows alone (a NaN in one adapter stays with its rows), and multiplied by s_i in fp32.
constexpr int MN_THREADS = 256;

struct MainArgs {
  const void *x, *w, *bias, *up;
  const float* scale_of;       // per adapter, or NULL
  const int32_t *offsets, *order;
  const float* h;
  void* y;
  long long ldx, K, N;
  long long M;
  int L, R, Rp;
  float scale;
};

template <int DT, int BM, int BN>
__global__ void __launch_bounds__(MN_THREADS) k_main(MainArgs P) {
  typedef typename Elem<DT>::T E;
  constexpr int EPC = Elem<DT>::EPC, KB = 8 * EPC;        // elements of a 128-byte row piece
  constexpr int MI = BM / 32, NI = BN / 32;               // 16-row / 16-output blocks of a wave
  constexpr int XL = BM / 32, WL = BN / 32;               // 16-byte loads of a thread and stage
  __shared__ u32x4 lds[2][(BM + BN) * 8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, q = lane >> 4;
  const int wm = wave & 1, wn = wave >> 1;
  const long long tiles_n = (P.N + BN - 1) / BN;
  const long long m0 = (long long)blockIdx.x / tiles_n * BM, n0 = (long long)blockIdx.x % tiles_n * BN;
  const E* X = static_cast<const E*>(P.x);
  const E* W = static_cast<const E*>(P.w);
  const int ch = tid & 7;
  const E* xrow[XL];
  const E* wrow[WL];
#pragma unroll
  for (int l = 0; l < XL; ++l) {
    long long p = m0 + (tid >> 3) + 32 * l;
    if (p >= P.M) p = P.M - 1;
    xrow[l] = X + (P.order ? (long long)P.order[p] : p) * P.ldx;
  }
#pragma unroll
  for (int l = 0; l < WL; ++l) {
    long long n = n0 + (tid >> 3) + 32 * l;
    if (n >= P.N) n = P.N - 1;
    wrow[l] = W + n * P.K;
  }
  u32x4 rx[XL], rw[WL];
  auto fetch = [&](long long s) {
    const long long k = s * KB + ch * EPC;
    if (k + EPC <= P.K) {
#pragma unroll
      for (int l = 0; l < XL; ++l) rx[l] = load16(xrow[l] + k);
#pragma unroll
      for (int l = 0; l < WL; ++l) rw[l] = load16(wrow[l] + k);
    } else {
#pragma unroll
      for (int l = 0; l < XL; ++l) rx[l] = load_tail<DT>(xrow[l], k, P.K);
#pragma unroll
      for (int l = 0; l < WL; ++l) rw[l] = load_tail<DT>(wrow[l], k, P.K);
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int l = 0; l < XL; ++l) {
      const int r = (tid >> 3) + 32 * l;
      lds[buf][r * 8 + (ch ^ (r & 7))] = rx[l];
    }
#pragma unroll
    for (int l = 0; l < WL; ++l) {
      const int r = (tid >> 3) + 32 * l;
      lds[buf][(BM + r) * 8 + (ch ^ (r & 7))] = rw[l];
    }
  };
  fetch(0);
  f32x4 acc[MI][NI];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};

  // ---- low-rank term
  long long tile_end = m0 + BM < P.M ? m0 + BM : P.M;
  const int kept = P.offsets[P.L];
  if (m0 < kept) {
    if (tile_end > kept) tile_end = kept;
    int lo = 0, hi = P.L;                    // first adapter that ends behind m0
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (P.offsets[mid + 1] > m0) hi = mid; else lo = mid + 1;
    }
    const int chunks = P.Rp / 16;
    for (int a = lo; a < P.L; ++a) {
      const int a0 = P.offsets[a], a1 = P.offsets[a + 1];
      if (a0 >= tile_end) break;
      if (a1 <= a0) continue;
      const E* B = static_cast<const E*>(P.up) + (long long)a * P.N * P.R;
      const float s = P.scale_of ? P.scale * P.scale_of[a] : P.scale;
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const long long p = m0 + wm * (BM / 2) + 16 * m + i;
        const bool mine = p >= a0 && p < a1;
        if (!__ballot(mine)) continue;
        const float* hr = P.h + (mine ? p : (long long)a0) * P.Rp;
        float ds = 1.f, us = s;
        if constexpr (DT == ANERF_F16) {     // largest |h| of the row -> [1, 2)
          float big = 0.f;
          for (int j = 0; j < P.Rp; j += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(hr + j);
            big = fmaxf(fmaxf(big, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3])));
          }
          if (big > 0.f && __builtin_isfinite(big)) {
            const int e = min(max(ilogbf(big), -100), 100);
            ds = ldexpf(1.f, -e);
            us = s * ldexpf(1.f, e);
          }
        }
#pragma unroll
        for (int n = 0; n < NI; ++n) {
          const long long col = n0 + wn * (BN / 2) + 16 * n + i;
          const E* br = B + (col < P.N ? col : P.N - 1) * P.R;
          f32x4 t = f32x4{0.f, 0.f, 0.f, 0.f};
          for (int c = 0; c < chunks; ++c) t = Elem<DT>::mma(b_operand<DT>(br, c, q, P.R), h_operand<DT>(hr, c, q, ds), t);
          if (mine) acc[m][n] = t * us;
        }
      }
    }
  }

  // ---- x W^T
  const long long stages = (P.K + KB - 1) / KB;
  put(0);
  __syncthreads();
  for (long long s = 0; s < stages; ++s) {
    const int buf = (int)(s & 1);
    if (s + 1 < stages) fetch(s + 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 xf[MI], wf[NI];
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const int r = wm * (BM / 2) + 16 * m + i;
        xf[m] = lds[buf][r * 8 + ((4 * h + q) ^ (r & 7))];
      }
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int r = wn * (BN / 2) + 16 * n + i;
        wf[n] = lds[buf][(BM + r) * 8 + ((4 * h + q) ^ (r & 7))];
      }
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n) acc[m][n] = Elem<DT>::mma(wf[n], xf[m], acc[m][n]);
    }
    if (s + 1 < stages) put(buf ^ 1);
    __syncthreads();
  }

  // ---- bias, rounding, store: lane (i, q) holds outputs 4q .. 4q+3 of its row in every 16x16 block
  const E* bias = static_cast<const E*>(P.bias);
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    const long long p = m0 + wm * (BM / 2) + 16 * m + i;
    if (p >= P.M) continue;
    E* yr = static_cast<E*>(P.y) + (P.order ? (long long)P.order[p] : p) * P.N;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const long long col = n0 + wn * (BN / 2) + 16 * n + 4 * q;
      f32x4 v = acc[m][n];
      typedef E out4 __attribute__((ext_vector_type(4)));
      if (col + 4 <= P.N) {
        if (bias) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += (float)bias[col + e];
        }
        out4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (E)v[e];
        __builtin_memcpy(yr + col, &o, sizeof(o));
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < P.N) yr[col + e] = (E)(bias ? v[e] + (float)bias[col + e] : v[e]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------- gradients of A and B
// part[piece] = sum over the piece's positions p of Z[order[p]][c] * V[p][j]        (Z = x, V = u: dA;  Z = g, V = h: dB)
// The contraction runs over rows, so that v_mfma_f32_16x16x4_f32 takes its operands as they lie in memory: lane (i, q) loads
// columns 4i .. 4i+3 of row q of a group of four, element e being its operand for the block of columns 4i + e, and V[p][16n + i].
// Values of 16-bit types become fp32 on the way (h and u stay whole): up to rank 32 the loads of Z are what bounds it, not the MFMAs.
// A workgroup owns 64 columns x 16*NJ ranks of a piece; its four waves take every fourth group of rows and are added through LDS.
// BY_RANK: part [piece][Rp][C] (operand order Z, V), else [piece][C][Rp] (V, Z): a lane ends with four values that lie together.
constexpr int TG_WAVES = 4, TG_COLS = 64, TG_DEPTH = 4;

template <int DT, int NJ, bool BY_RANK>
__global__ void __launch_bounds__(TG_WAVES * 64) k_thin_grad(const typename Elem<DT>::T* __restrict__ Z, long long ldz, const int32_t* __restrict__ order,
                                                             const float* __restrict__ V, const int32_t* __restrict__ offsets, int L, long long C,
                                                             int Rp, int rows, float* __restrict__ part) {
  typedef typename Elem<DT>::T E;
  typedef E vec __attribute__((ext_vector_type(4)));
  __shared__ f32x4 red[TG_WAVES - 1][4 * NJ][64];
  int a, p0, p1;
  if (!find_piece(offsets, L, rows, blockIdx.y, a, p0, p1)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const long long c = (long long)blockIdx.x * TG_COLS + 4 * i;
  const int j0 = blockIdx.z * 16 * NJ;
  const bool whole = c + 4 <= C;
  f32x4 acc[4][NJ];
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int n = 0; n < NJ; ++n) acc[e][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int b = p0 + 4 * wave; b < p1; b += 4 * TG_WAVES * TG_DEPTH) {
    f32x4 z[TG_DEPTH];
    float v[TG_DEPTH][NJ];
#pragma unroll
    for (int d = 0; d < TG_DEPTH; ++d) {
      const int p = b + 4 * TG_WAVES * d + q;
      const bool on = p < p1;
      z[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NJ; ++n) v[d][n] = on && j0 + 16 * n < Rp ? V[(long long)p * Rp + j0 + 16 * n + i] : 0.f;
      if (on) {
        const E* zr = Z + (long long)(order ? order[p] : p) * ldz + c;
        if (whole) {
          vec w;
          __builtin_memcpy(&w, zr, sizeof(w));
#pragma unroll
          for (int e = 0; e < 4; ++e) z[d][e] = (float)w[e];
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < C) z[d][e] = (float)zr[e];
        }
      }
    }
#pragma unroll
    for (int d = 0; d < TG_DEPTH; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int n = 0; n < NJ; ++n)
          acc[e][n] = BY_RANK ? __builtin_amdgcn_mfma_f32_16x16x4f32(z[d][e], v[d][n], acc[e][n], 0, 0, 0)
                              : __builtin_amdgcn_mfma_f32_16x16x4f32(v[d][n], z[d][e], acc[e][n], 0, 0, 0);
  }
  if (wave) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int n = 0; n < NJ; ++n) red[wave - 1][e * NJ + n][lane] = acc[e][n];
  }
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int w = 0; w < TG_WAVES - 1; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int n = 0; n < NJ; ++n) acc[e][n] += red[w][e * NJ + n][lane];
  const long long base = (long long)blockIdx.y * Rp * C, c0 = (long long)blockIdx.x * TG_COLS;
#pragma unroll
  for (int n = 0; n < NJ; ++n) {
    if (j0 + 16 * n >= Rp) break;
    if (BY_RANK) {      // block e, register r: column 16q + 4r + e of rank 16n + i
      float* o = part + base + (long long)(j0 + 16 * n + i) * C + c0 + 16 * q;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c0 + 16 * q + 4 * r + e < C) o[4 * r + e] = acc[e][n][r];
    } else {            // block e, register r: rank 16n + 4q + r of column 4i + e
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < C) *reinterpret_cast<f32x4*>(part + base + (c + e) * Rp + j0 + 16 * n + 4 * q) = acc[e][n];
    }
  }
}

// adds an adapter's pieces in their order, times s_i.  BY_RANK: out[i][j][c] (dA), else out[i][c][j] (dB).  Adapters without rows get zeros.
template <int DT, bool BY_RANK>
__global__ void __launch_bounds__(256) k_thin_grad_sum(const float* __restrict__ part, const int32_t* __restrict__ offsets, int L, long long C, int R,
                                                       int Rp, int rows, const float* __restrict__ scale_of, float scale,
                                                       typename Elem<DT>::T* __restrict__ out) {
  typedef typename Elem<DT>::T E;
  const int a = blockIdx.y, lane = threadIdx.x & 63;
  int first = 0;
  for (int b = lane; b < a; b += 64) first += (offsets[b + 1] - offsets[b] + rows - 1) / rows;
#pragma unroll
  for (int d = 32; d; d >>= 1) first += __shfl_xor(first, d);
  const int n = (offsets[a + 1] - offsets[a] + rows - 1) / rows;
  const float s = scale_of ? scale * scale_of[a] : scale;
  const long long all = C * R, stride = C * Rp;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < all; e += (long long)gridDim.x * 256) {
    const float* src = part + first * stride + (BY_RANK ? e : e / R * Rp + e % R);
    float v = 0.f;
#pragma unroll 8
    for (int q = 0; q < n; ++q) v += src[q * stride];
    out[(long long)a * all + e] = (E)(v * s);
  }
}

// ------------------------------------------------------------------------------------------------------------------- transposes
struct TransposeJob {
  const void* in;
  void* out;
  long long rows, cols, batch, tiles, tiles_c;   // in [batch][rows][cols] -> out [batch][cols][rows]
};
struct TransposeJobs {
  TransposeJob j[3];
};

template <typename U>
__global__ void __launch_bounds__(256) k_transpose(TransposeJobs J) {
  __shared__ U t[64][65];
  long long b = blockIdx.x;
  int k = 0;
  while (k < 2 && b >= J.j[k].tiles * J.j[k].batch) b -= J.j[k].tiles * J.j[k].batch, ++k;
  const TransposeJob& T = J.j[k];
  const U* in = static_cast<const U*>(T.in) + b / T.tiles * T.rows * T.cols;
  U* out = static_cast<U*>(T.out) + b / T.tiles * T.rows * T.cols;
  const long long r0 = b % T.tiles / T.tiles_c * 64, c0 = b % T.tiles % T.tiles_c * 64;
  const int cx = threadIdx.x & 63, ry = threadIdx.x >> 6;
  for (int r = ry; r < 64; r += 4)
    if (r0 + r < T.rows && c0 + cx < T.cols) t[r][cx] = in[(r0 + r) * T.cols + c0 + cx];
  __syncthreads();
  for (int c = ry; c < 64; c += 4)
    if (c0 + c < T.cols && r0 + cx < T.rows) out[(c0 + c) * T.rows + r0 + cx] = t[cx][c];
}

// ---------------------------------------------------------------------------------------------------------------------- launchers
template <int DT>
static int linear_t(const AnerfAdapterIO& A, hipStream_t st) {
  typedef typename Elem<DT>::T E;
  const int Rp = (A.rank + 15) / 16 * 16;
  const long long pieces = pieces_bound(A.n_rows, A.n_adapters, TH_ROWS);
  const E* x = static_cast<const E*>(A.x);
  const E* down = static_cast<const E*>(A.down);
  if (Rp <= 16)
    k_thin<DT, 1><<<dim3((unsigned)pieces, 1), TH_WAVES * 64, 0, st>>>(x, A.x_stride, A.order, down, A.offsets, A.n_adapters, A.n_in, A.rank, Rp, A.h);
  else if (Rp <= 32)
    k_thin<DT, 2><<<dim3((unsigned)pieces, 1), TH_WAVES * 64, 0, st>>>(x, A.x_stride, A.order, down, A.offsets, A.n_adapters, A.n_in, A.rank, Rp, A.h);
  else
    k_thin<DT, 4><<<dim3((unsigned)pieces, (Rp + 63) / 64), TH_WAVES * 64, 0, st>>>(x, A.x_stride, A.order, down, A.offsets, A.n_adapters, A.n_in,
                                                                                     A.rank, Rp, A.h);
  int rc = check_launch("k_thin");
  if (rc || !A.y) return rc;       // (the gradient of A alone needs h only)
  MainArgs P = {A.x, A.weight, A.bias, A.up, A.scale_of, A.offsets, A.order, A.h, A.y, A.x_stride, A.n_in, A.n_out, A.n_rows, A.n_adapters,
                A.rank, Rp, A.scale};
  // 128 x 128 tiles read each operand half as often as 64 x 64 ones; below one workgroup a CU the smaller ones fill more of the chip
  const long long big = (A.n_rows + 127) / 128 * ((A.n_out + 127) / 128);
  if (big >= 256) {
    k_main<DT, 128, 128><<<(unsigned)big, MN_THREADS, 0, st>>>(P);
  } else {
    const long long tiles = (A.n_rows + 63) / 64 * ((A.n_out + 63) / 64);
    k_main<DT, 64, 64><<<(unsigned)tiles, MN_THREADS, 0, st>>>(P);
  }
  return check_launch("k_main");
}

int launch_adapter_linear(const AnerfAdapterIO& A, hipStream_t st) {
  switch (A.dtype) {
    case ANERF_F32: return linear_t<ANERF_F32>(A, st);
    case ANERF_BF16: return linear_t<ANERF_BF16>(A, st);
    default: return linear_t<ANERF_F16>(A, st);
  }
}

// rows of a piece of k_thin_grad: about 1024 workgroups (a chip full of them twice over), but 64 rows at least (a piece writes C x Rp floats)
static int grad_ranks(int Rp) { return Rp <= 16 ? 1 : Rp <= 32 ? 2 : 4; }
static int grad_rows(long long M, long long C, int Rp) {
  const long long blocks = (C + TG_COLS - 1) / TG_COLS * ((Rp + 16 * grad_ranks(Rp) - 1) / (16 * grad_ranks(Rp)));
  const long long pieces = (1024 + blocks - 1) / blocks;
  const long long rows = ((M + pieces - 1) / pieces + 63) / 64 * 64;
  return (int)(rows < 64 ? 64 : rows);
}

static long long part_floats(long long M, int L, long long C, int Rp) {
  const int rows = grad_rows(M, C, Rp);
  return pieces_bound(M, L, rows) * Rp * C;
}

struct BackwardPlan {
  long long wt, dt, ut, u, part, bytes;     // byte offsets in the workspace
};
static BackwardPlan backward_plan(const AnerfAdapterIO& A) {
  const long long es = A.dtype == ANERF_F32 ? 4 : 2;
  const int Rp = (A.rank + 15) / 16 * 16;
  auto up16 = [](long long b) { return (b + 255) / 256 * 256; };
  BackwardPlan B;
  long long at = 0;
  B.wt = at, at += up16(A.n_in * A.n_out * es);
  B.dt = at, at += up16((long long)A.n_adapters * A.rank * A.n_in * es);
  B.ut = at, at += up16((long long)A.n_adapters * A.rank * A.n_out * es);
  B.u = at, at += up16(A.n_rows * Rp * 4);
  const long long pa = part_floats(A.n_rows, A.n_adapters, A.n_in, Rp), pb = part_floats(A.n_rows, A.n_adapters, A.n_out, Rp);
  B.part = at, at += up16((pa > pb ? pa : pb) * 4);
  B.bytes = at;
  return B;
}
long long adapter_backward_workspace(const AnerfAdapterIO& A) { return backward_plan(A).bytes; }

template <int DT, bool BY_RANK>
static int thin_grad_t(const void* Z, long long ldz, const int32_t* order, const float* V, const AnerfAdapterIO& A, long long C, float* part, void* out,
                       hipStream_t st) {
  typedef typename Elem<DT>::T E;
  const int Rp = (A.rank + 15) / 16 * 16, rows = grad_rows(A.n_rows, C, Rp);
  const long long pieces = pieces_bound(A.n_rows, A.n_adapters, rows);
  if (pieces > 0) {
    const int nj = grad_ranks(Rp);
    const dim3 grid((unsigned)((C + TG_COLS - 1) / TG_COLS), (unsigned)pieces, (Rp + 16 * nj - 1) / (16 * nj));
    auto run = [&](auto kernel) { kernel<<<grid, TG_WAVES * 64, 0, st>>>(static_cast<const E*>(Z), ldz, order, V, A.offsets, A.n_adapters, C, Rp, rows, part); };
    if (nj == 1) run(k_thin_grad<DT, 1, BY_RANK>);
    else if (nj == 2) run(k_thin_grad<DT, 2, BY_RANK>);
    else run(k_thin_grad<DT, 4, BY_RANK>);
    const int rc = check_launch("k_thin_grad");
    if (rc) return rc;
  }
  const long long all = C * A.rank, bx = (all + 255) / 256;
  k_thin_grad_sum<DT, BY_RANK><<<dim3((unsigned)(bx < 4096 ? bx : 4096), A.n_adapters), 256, 0, st>>>(part, A.offsets, A.n_adapters, C, A.rank, Rp, rows,
                                                                                                   A.scale_of, A.scale, static_cast<E*>(out));
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
    auto job = [](const void* in, void* out, long long rows, long long cols, long long batch) {
      TransposeJob t = {in, out, rows, cols, batch, (rows + 63) / 64 * ((cols + 63) / 64), (cols + 63) / 64};
      return t;
    };
    TransposeJobs J;
    J.j[0] = job(A.weight, ws + B.wt, A.n_out, A.n_in, 1);
    J.j[1] = job(A.down, ws + B.dt, A.rank, A.n_in, A.n_adapters);
    J.j[2] = job(A.up, ws + B.ut, A.n_out, A.rank, A.n_adapters);
    long long blocks = 0;
    for (int k = 0; k < 3; ++k) blocks += J.j[k].tiles * J.j[k].batch;
    if constexpr (DT == ANERF_F32) k_transpose<uint32_t><<<(unsigned)blocks, 256, 0, st>>>(J);
    else k_transpose<uint16_t><<<(unsigned)blocks, 256, 0, st>>>(J);
    int rc = check_launch("k_transpose");
    if (rc) return rc;
    AnerfAdapterIO T = A;
    T.x = G.g, T.x_stride = G.g_stride, T.weight = ws + B.wt, T.bias = nullptr, T.down = ws + B.ut, T.up = ws + B.dt;
    T.n_in = A.n_out, T.n_out = A.n_in, T.y = G.dx, T.h = u;
    rc = linear_t<DT>(T, st);
    if (rc) return rc;
  }
  if (G.ddown) {
    const int rc = thin_grad_t<DT, true>(A.x, A.x_stride, A.order, u, A, A.n_in, part, G.ddown, st);
    if (rc) return rc;
  }
  if (G.dup) {
    const int rc = thin_grad_t<DT, false>(G.g, G.g_stride, A.order, A.h, A, A.n_out, part, G.dup, st);
    if (rc) return rc;
  }
  return ANERF_OK;
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
