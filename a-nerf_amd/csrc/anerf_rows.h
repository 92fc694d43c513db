// anerf_rows.h -- element types and group lookups shared by the row-routing and adapter kernels (gfx950 only).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "anerf.h"
#include "anerf_dev.h"

namespace anerf {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int ROWS_MAX_GROUPS = 1024;   // every wave's group counters live in LDS: 18 x 1025 x 4 bytes
constexpr int ANERF_MAX_RANK = 1024;
constexpr int ROWS_MAX_CHOICES = 64;    // a token's slots sit in the lanes of one wave

// element types of the C ABI: storage type, elements in 16 bytes, and the MFMA products of 16-byte operands.  In a 16 x 16 block lane
// (i = lane % 16, q = lane / 16) holds 16 bytes of row i of each operand, so that a step contracts 64 bytes of a row.  fp32: INSTR = 4
// instructions a step, instruction e contracting element e of the lane groups -- the indices are contracted in another order than
// memory's, the same one for both operands.  The result: lane (i, q) holds column i, rows 4q .. 4q+3.
template <int DT> struct Elem;
template <> struct Elem<ANERF_F32> {
  typedef float T;
  static constexpr int EPC = 4, INSTR = 4;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, int e) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f32x4, a)[e], __builtin_bit_cast(f32x4, b)[e], c, 0, 0, 0);
  }
};
template <> struct Elem<ANERF_BF16> {
  typedef __bf16 T;
  static constexpr int EPC = 8, INSTR = 1;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
template <> struct Elem<ANERF_F16> {
  typedef _Float16 T;
  static constexpr int EPC = 8, INSTR = 1;
  static __device__ __forceinline__ f32x4 mma(u32x4 a, u32x4 b, f32x4 c, int) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

// 16 bytes at any element's alignment: gfx950 takes dwordx4 global accesses at every address
__device__ __forceinline__ u32x4 load16(const void* p) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
__device__ __forceinline__ void store16(void* p, u32x4 v) { __builtin_memcpy(p, &v, 16); }

// 16 bytes of a row of `n` elements from element k on; what lies behind the row reads as zero
template <int DT>
__device__ __forceinline__ u32x4 load_tail(const typename Elem<DT>::T* row, long long k, long long n) {
  constexpr int EPC = Elem<DT>::EPC;
  typedef typename Elem<DT>::T T;
  if (k + EPC <= n) return load16(row + k);
  typedef T vec __attribute__((ext_vector_type(EPC)));
  vec v;
#pragma unroll
  for (int e = 0; e < EPC; ++e) v[e] = k + e < n ? row[k + e] : (T)0.f;
  return __builtin_bit_cast(u32x4, v);
}

// first position of a run of pieces: adapter / group a owns ceil((offsets[a+1] - offsets[a]) / rows) pieces of the work list; the
// whole wave looks up piece `b` (uniform) by scanning the group sizes 64 at a time.  false: fewer pieces than b + 1.
__device__ __forceinline__ bool find_piece(const int32_t* __restrict__ offsets, int n_groups, int rows, int b, int& group, int& p0, int& p1) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int a0 = 0; a0 < n_groups; a0 += 64) {
    const int a = a0 + lane;
    const int lo = a < n_groups ? offsets[a] : 0, hi = a < n_groups ? offsets[a + 1] : 0;
    const int cnt = (hi - lo + rows - 1) / rows;
    int incl = cnt;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int up = __shfl_up(incl, d);
      if (lane >= d) incl += up;
    }
    const unsigned long long past = __ballot(base + incl > b);
    if (past) {
      const int f = __builtin_ctzll(past);
      group = a0 + f;
      const int first = base + __shfl(incl, f) - __shfl(cnt, f);
      p0 = __shfl(lo, f) + (b - first) * rows;
      const int end = __shfl(hi, f);
      p1 = p0 + rows < end ? p0 + rows : end;
      return true;
    }
    base += __shfl(incl, 63);
  }
  return false;
}

// the work list's length is known on the device only; the grid covers its bound
inline long long pieces_bound(long long n_rows, int n_groups, int rows) {
  const long long part = n_rows < n_groups ? n_rows : n_groups;   // groups that can end inside a piece
  return n_rows / rows + part;
}

}  // namespace anerf
