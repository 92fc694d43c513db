// anerf_rows.hip -- rows put in order of their group and brought back (gfx950).
//   pairs (t, j): row t's j-th group idx[t][j]; a pair whose group is outside 0 .. G-1 is dropped
//   route     stable counting sort of the pairs by group, the dropped ones last: offsets [G+1], source [T*k] (position -> pair),
//             slot [T*k] (pair -> position)
//   out       out[slot[t][j]] = (w[t][j] *) x[t], zero at the dropped pairs' positions
//   back      y[t] = sum_j (w[t][j] *) z[slot[t][j]] over the kept pairs, summed in fp32 in the order of j, rounded once
//   back_grad dz[slot[t][j]] = w[t][j] dy[t],  dw[t][j] = <dy[t], z[slot[t][j]]>
// Every result has one writer and every sum one order: bit-reproducible, no atomics on memory.
#include "anerf_rows.h"

namespace anerf {

constexpr int RT_WAVES = 16, RT_THREADS = RT_WAVES * 64;
constexpr int RT_SINGLE = 4096;     // pairs that one workgroup sorts in one launch: 4 steps of 64 pairs a wave
constexpr int RT_MAX_BLOCKS = 256;

template <typename I>
__device__ __forceinline__ int group_of(const I* __restrict__ idx, long long p, long long n, int G) {
  if (p >= n) return -1;
  const I v = idx[p];
  return v >= 0 && v < (I)G ? (int)v : G;
}

// lanes of the wave that hold the same group (bits = number of bits of G): one ballot a bit
__device__ __forceinline__ unsigned long long same_group(int g, int bits, bool on) {
  unsigned long long m = __ballot(on);
  for (int b = 0; b < bits; ++b) {
    const unsigned long long s = __ballot((g >> b) & 1);
    m &= (g >> b) & 1 ? s : ~s;
  }
  return m;
}

// workgroup b counts the groups of its `chunk` pairs (consecutive ones, so that the sort stays stable) into hist[b][G+1]
template <typename I>
__global__ void __launch_bounds__(RT_THREADS) k_route_count(const I* __restrict__ idx, long long n, int G, int chunk, int32_t* __restrict__ hist) {
  extern __shared__ int cnt[];
  for (int g = threadIdx.x; g <= G; g += RT_THREADS) cnt[g] = 0;
  __syncthreads();
  const long long lo = (long long)blockIdx.x * chunk;
  for (int q = threadIdx.x; q < chunk; q += RT_THREADS) {
    const int g = group_of(idx, lo + q, n, G);
    if (g >= 0) atomicAdd(&cnt[g], 1);      // LDS integer counts: their order does not show
  }
  __syncthreads();
  for (int g = threadIdx.x; g <= G; g += RT_THREADS) hist[(long long)blockIdx.x * (G + 1) + g] = cnt[g];
}

// Positions.  A wave owns a contiguous part of the workgroup's chunk: its counters start at (start of the group) + (pairs of the
// group in earlier workgroups) + (in earlier waves), and it walks its part 64 pairs at a time in order.  hist == NULL: one
// workgroup holds all pairs.  Latency-bound: two passes over the indices, everything else is in LDS.  66 pairs: 3 us; 65520 pairs of 16
// groups: count 4.9 + place 5.2 us, of 128 groups place 8.1 us (the prefix over the workgroups' counts grows with groups x workgroups).
template <typename I>
__global__ void __launch_bounds__(RT_THREADS) k_route_place(const I* __restrict__ idx, long long n, int G, int chunk, int bits,
                                                            const int32_t* __restrict__ hist, int32_t* __restrict__ offsets,
                                                            int32_t* __restrict__ source, int32_t* __restrict__ slot) {
  extern __shared__ int lds[];
  const int W = G + 1;
  int* cnt = lds;                       // [RT_WAVES][W]
  int* total = lds + RT_WAVES * W;      // [W] pairs of the group in the whole call, then its start
  int* before = total + W;              // [W] pairs of the group in earlier workgroups
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const long long lo = (long long)blockIdx.x * chunk;
  const int part = chunk / RT_WAVES;
  for (int e = tid; e < (RT_WAVES + 2) * W; e += RT_THREADS) lds[e] = 0;
  __syncthreads();
  for (int q = lane; q < part; q += 64) {
    const int g = group_of(idx, lo + wave * part + q, n, G);
    if (g >= 0) atomicAdd(&cnt[wave * W + g], 1);
  }
  if (hist) {
    int gp = 1;
    while (gp < W && gp < RT_THREADS) gp <<= 1;
    const int nb = gridDim.x, parts = RT_THREADS / gp, my = tid / gp;
    for (int g = tid % gp; g < W; g += gp) {
      int all = 0, prev = 0;
      for (int b0 = my; b0 < nb; b0 += 8 * parts) {      // eight loads at a time (one after the other: 9.4 us with 128 groups)
        int v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = b0 + u * parts < nb ? hist[(long long)(b0 + u * parts) * W + g] : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          all += v[u];
          prev += b0 + u * parts < (int)blockIdx.x ? v[u] : 0;
        }
      }
      if (all) atomicAdd(&total[g], all);
      if (prev) atomicAdd(&before[g], prev);
    }
  }
  __syncthreads();
  if (!hist)
    for (int g = tid; g < W; g += RT_THREADS) {
      int all = 0;
      for (int w = 0; w < RT_WAVES; ++w) all += cnt[w * W + g];
      total[g] = all;
    }
  __syncthreads();
  if (wave == 0) {                      // exclusive scan of the totals, 64 groups at a time
    int base = 0;
    for (int g0 = 0; g0 < W; g0 += 64) {
      const int g = g0 + lane;
      const int v = g < W ? total[g] : 0;
      int incl = v;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(incl, d);
        if (lane >= d) incl += up;
      }
      if (g < W) {
        total[g] = base + incl - v;
        if (blockIdx.x == 0) offsets[g] = base + incl - v;
      }
      base += __shfl(incl, 63);
    }
  }
  __syncthreads();
  for (int g = tid; g < W; g += RT_THREADS) {
    int at = total[g] + before[g];
    for (int w = 0; w < RT_WAVES; ++w) {
      const int c = cnt[w * W + g];
      cnt[w * W + g] = at;
      at += c;
    }
  }
  __syncthreads();
  volatile int* mine = cnt + wave * W;
  for (int q0 = 0; q0 < part; q0 += 64) {
    const long long p = lo + wave * part + q0 + lane;
    const bool on = q0 + lane < part && p < n;
    const int g = on ? group_of(idx, p, n, G) : 0;
    const unsigned long long m = same_group(g, bits, on);
    int at = 0;
    if (on) at = mine[g];
    __builtin_amdgcn_wave_barrier();
    if (on) {
      const int rank = __popcll(m & ((1ull << lane) - 1));
      if (lane == 63 - __builtin_clzll(m)) mine[g] = at + rank + 1;      // the group's last lane moves the counter on
      source[at + rank] = (int32_t)p;
      slot[p] = at + rank;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

static int route_chunk(long long n) {
  if (n <= RT_SINGLE) return (int)((n + RT_THREADS - 1) / RT_THREADS * RT_THREADS);
  const long long per = (n + RT_MAX_BLOCKS - 1) / RT_MAX_BLOCKS;
  const long long c = (per + RT_THREADS - 1) / RT_THREADS * RT_THREADS;
  return (int)(c < 1024 ? 1024 : c);
}

long long route_workspace(long long n, int G) {
  if (n <= RT_SINGLE) return 0;
  const int chunk = route_chunk(n);
  return (n + chunk - 1) / chunk * (G + 1) * 4;
}

template <typename I>
static int launch_route_t(const I* idx, long long n, int G, int32_t* offsets, int32_t* source, int32_t* slot, int32_t* ws, hipStream_t st) {
  int bits = 0;
  while ((1 << bits) <= G) ++bits;
  const int chunk = n ? route_chunk(n) : RT_THREADS;
  const unsigned lds = (RT_WAVES + 2) * (G + 1) * 4;
  static unsigned long long done = 0;
  ensure_dynamic_lds(reinterpret_cast<const void*>(k_route_place<I>), (RT_WAVES + 2) * (ROWS_MAX_GROUPS + 1) * 4, &done);
  if (n <= RT_SINGLE) {
    k_route_place<I><<<1, RT_THREADS, lds, st>>>(idx, n, G, chunk, bits, nullptr, offsets, source, slot);
  } else {
    const int nb = (int)((n + chunk - 1) / chunk);
    k_route_count<I><<<nb, RT_THREADS, (G + 1) * 4, st>>>(idx, n, G, chunk, ws);
    k_route_place<I><<<nb, RT_THREADS, lds, st>>>(idx, n, G, chunk, bits, ws, offsets, source, slot);
  }
  return check_launch("k_route");
}

int launch_route(const void* idx, int wide, long long n, int G, int32_t* offsets, int32_t* source, int32_t* slot, void* ws, hipStream_t st) {
  return wide ? launch_route_t(static_cast<const long long*>(idx), n, G, offsets, source, slot, static_cast<int32_t*>(ws), st)
              : launch_route_t(static_cast<const int32_t*>(idx), n, G, offsets, source, slot, static_cast<int32_t*>(ws), st);
}

// ---------------------------------------------------------------------------------------------------------------------------
// One wave a row t: its k slots sit in the lanes, and the row is read once and written k times.  16 bytes a lane and access; the
// elements behind the last whole 16 bytes of a row go one by one.  HBM-bound: T*D read + T*k*D written.  65520 x 1080 fp32: 111 us,
// 5.1 TB/s; 8192 x 2048 bf16 to 8 places each: 65 us, 4.7 TB/s.
constexpr int RW_WAVES = 4, RW_BATCH = 4, RW_MAX_X = 1 << 23;

template <int DT, bool WEIGHTED>
__global__ void __launch_bounds__(RW_WAVES * 64) k_rows_out(const typename Elem<DT>::T* __restrict__ x, const float* __restrict__ w,
                                                            const int32_t* __restrict__ slot, const int32_t* __restrict__ end,
                                                            long long T, int k, long long D, typename Elem<DT>::T* __restrict__ out) {
  typedef typename Elem<DT>::T E;
  constexpr int EPC = Elem<DT>::EPC;
  typedef E vec __attribute__((ext_vector_type(EPC)));
  const int lane = threadIdx.x & 63;
  const long long t = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * RW_WAVES + (threadIdx.x >> 6);
  if (t >= T) return;
  const int kept = *end;
  const int myslot = lane < k ? slot[t * k + lane] : 0;
  const float myw = WEIGHTED && lane < k ? w[t * k + lane] : 1.f;
  const E* row = x + t * D;
  const long long whole = D / EPC;
  for (long long c = lane; c < whole; c += 64) {
    const vec v = __builtin_bit_cast(vec, load16(row + c * EPC));
    for (int j = 0; j < k; ++j) {
      const int s = __builtin_amdgcn_readlane(myslot, j);
      vec o = v;
      if (WEIGHTED) {
        const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, myw), j));
#pragma unroll
        for (int e = 0; e < EPC; ++e) o[e] = (E)((float)v[e] * wj);
      }
      store16(out + (long long)s * D + c * EPC, s < kept ? __builtin_bit_cast(u32x4, o) : u32x4{0, 0, 0, 0});
    }
  }
  const long long c = whole * EPC + lane;
  if (c < D) {
    const E v = row[c];
    for (int j = 0; j < k; ++j) {
      const int s = __builtin_amdgcn_readlane(myslot, j);
      const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, myw), j));
      out[(long long)s * D + c] = s < kept ? (WEIGHTED ? (E)((float)v * wj) : v) : (E)0.f;
    }
  }
}

// the way back, the same split: T*k*D read + T*D written.  16384 x 4 x 1024 bf16: 40 us, 4.2 TB/s
template <int DT, bool WEIGHTED>
__global__ void __launch_bounds__(RW_WAVES * 64) k_rows_back(const typename Elem<DT>::T* __restrict__ z, const float* __restrict__ w,
                                                             const int32_t* __restrict__ slot, const int32_t* __restrict__ end,
                                                             long long T, int k, long long D, typename Elem<DT>::T* __restrict__ y) {
  typedef typename Elem<DT>::T E;
  constexpr int EPC = Elem<DT>::EPC;
  typedef E vec __attribute__((ext_vector_type(EPC)));
  const int lane = threadIdx.x & 63;
  const long long t = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * RW_WAVES + (threadIdx.x >> 6);
  if (t >= T) return;
  const int kept = *end;
  const int myslot = lane < k ? slot[t * k + lane] : 0;
  const float myw = WEIGHTED && lane < k ? w[t * k + lane] : 1.f;
  const long long whole = D / EPC;
  for (long long c = lane; c < whole; c += 64) {
    float acc[EPC];
#pragma unroll
    for (int e = 0; e < EPC; ++e) acc[e] = 0.f;
    for (int j = 0; j < k; ++j) {
      const int s = __builtin_amdgcn_readlane(myslot, j);
      if (s >= kept) continue;
      const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, myw), j));
      const vec v = __builtin_bit_cast(vec, load16(z + (long long)s * D + c * EPC));
#pragma unroll
      for (int e = 0; e < EPC; ++e) acc[e] = WEIGHTED ? fmaf((float)v[e], wj, acc[e]) : acc[e] + (float)v[e];
    }
    vec o;
#pragma unroll
    for (int e = 0; e < EPC; ++e) o[e] = (E)acc[e];
    store16(y + t * D + c * EPC, __builtin_bit_cast(u32x4, o));
  }
  const long long c = whole * EPC + lane;
  if (c < D) {
    float acc = 0.f;
    for (int j = 0; j < k; ++j) {
      const int s = __builtin_amdgcn_readlane(myslot, j);
      if (s >= kept) continue;
      const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, myw), j));
      const float v = (float)z[(long long)s * D + c];
      acc = WEIGHTED ? fmaf(v, wj, acc) : acc + v;
    }
    y[t * D + c] = (E)acc;
  }
}

// dz and dw in one pass over z, RW_BATCH choices at a time with one read of dy's row for them.  16384 x 4 x 1024 bf16: 49 us, 302 MB at
// 6.2 TB/s (one choice at a time 66; on the way back, where only z is read, the batch gained nothing)
template <int DT>
__global__ void __launch_bounds__(RW_WAVES * 64) k_rows_back_grad(const typename Elem<DT>::T* __restrict__ dy, const typename Elem<DT>::T* __restrict__ z,
                                                                  const float* __restrict__ w, const int32_t* __restrict__ slot,
                                                                  const int32_t* __restrict__ end, long long T, int k, long long D,
                                                                  typename Elem<DT>::T* __restrict__ dz, float* __restrict__ dw) {
  typedef typename Elem<DT>::T E;
  constexpr int EPC = Elem<DT>::EPC;
  typedef E vec __attribute__((ext_vector_type(EPC)));
  const int lane = threadIdx.x & 63;
  const long long t = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * RW_WAVES + (threadIdx.x >> 6);
  if (t >= T) return;
  const int kept = *end;
  const int myslot = lane < k ? slot[t * k + lane] : 0;
  const float myw = lane < k ? w[t * k + lane] : 0.f;
  const long long whole = D / EPC;
  const E* g = dy + t * D;
  for (int j0 = 0; j0 < k; j0 += RW_BATCH) {
    int sl[RW_BATCH];
    float wj[RW_BATCH], dot[RW_BATCH];
    bool on[RW_BATCH], there[RW_BATCH];
#pragma unroll
    for (int u = 0; u < RW_BATCH; ++u) {
      const int j = min(j0 + u, k - 1);
      sl[u] = __builtin_amdgcn_readlane(myslot, j);
      wj[u] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, myw), j));
      dot[u] = 0.f;
      there[u] = j0 + u < k, on[u] = there[u] && sl[u] < kept;
    }
    for (long long c = lane; c < whole; c += 64) {
      const vec gv = __builtin_bit_cast(vec, load16(g + c * EPC));
      vec zv[RW_BATCH];
#pragma unroll
      for (int u = 0; u < RW_BATCH; ++u)
        if (on[u]) zv[u] = __builtin_bit_cast(vec, load16(z + (long long)sl[u] * D + c * EPC));
#pragma unroll
      for (int u = 0; u < RW_BATCH; ++u) {
        if (!there[u]) continue;
        if (on[u]) {
#pragma unroll
          for (int e = 0; e < EPC; ++e) dot[u] = fmaf((float)gv[e], (float)zv[u][e], dot[u]);
        }
        if (dz) {
          vec r;
#pragma unroll
          for (int e = 0; e < EPC; ++e) r[e] = (E)((float)gv[e] * wj[u]);
          store16(dz + (long long)sl[u] * D + c * EPC, on[u] ? __builtin_bit_cast(u32x4, r) : u32x4{0, 0, 0, 0});
        }
      }
    }
    const long long c = whole * EPC + lane;
    if (c < D) {
      const float gv = (float)g[c];
#pragma unroll
      for (int u = 0; u < RW_BATCH; ++u) {
        if (!there[u]) continue;
        if (on[u]) dot[u] = fmaf(gv, (float)z[(long long)sl[u] * D + c], dot[u]);
        if (dz) dz[(long long)sl[u] * D + c] = on[u] ? (E)(gv * wj[u]) : (E)0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < RW_BATCH; ++u) {
#pragma unroll
      for (int d = 32; d; d >>= 1) dot[u] += __shfl_xor(dot[u], d);
      if (lane == 0 && there[u]) dw[t * k + j0 + u] = on[u] ? dot[u] : 0.f;
    }
  }
}

template <int DT>
static int launch_rows_t(int op, const void* a, const void* b, const float* w, const int32_t* slot, const int32_t* end, long long T, int k,
                         long long D, void* out, float* dw, hipStream_t st) {
  typedef typename Elem<DT>::T E;
  // (a launch has fewer than 2^32 work items along x: 2^25 rows)
  const long long blocks = (T + RW_WAVES - 1) / RW_WAVES, along_x = blocks < RW_MAX_X ? blocks : RW_MAX_X;
  const dim3 grid((unsigned)along_x, (unsigned)((blocks + along_x - 1) / along_x)), block(RW_WAVES * 64);
  const E* in = static_cast<const E*>(a);
  E* o = static_cast<E*>(out);
  if (op == 0) {
    if (w) k_rows_out<DT, true><<<grid, block, 0, st>>>(in, w, slot, end, T, k, D, o);
    else k_rows_out<DT, false><<<grid, block, 0, st>>>(in, w, slot, end, T, k, D, o);
  } else if (op == 1) {
    if (w) k_rows_back<DT, true><<<grid, block, 0, st>>>(in, w, slot, end, T, k, D, o);
    else k_rows_back<DT, false><<<grid, block, 0, st>>>(in, w, slot, end, T, k, D, o);
  } else {
    k_rows_back_grad<DT><<<grid, block, 0, st>>>(in, static_cast<const E*>(b), w, slot, end, T, k, D, o, dw);
  }
  return check_launch("k_rows");
}

// op 0: out, 1: back, 2: back_grad
int launch_rows(int op, int dtype, const void* a, const void* b, const float* w, const int32_t* slot, const int32_t* end, long long T, int k,
                long long D, void* out, float* dw, hipStream_t st) {
  switch (dtype) {
    case ANERF_F32: return launch_rows_t<ANERF_F32>(op, a, b, w, slot, end, T, k, D, out, dw, st);
    case ANERF_BF16: return launch_rows_t<ANERF_BF16>(op, a, b, w, slot, end, T, k, D, out, dw, st);
    default: return launch_rows_t<ANERF_F16>(op, a, b, w, slot, end, T, k, D, out, dw, st);
  }
}

}  // namespace anerf
