// Device helpers of the attention kernels: rows of any type, rounding, matrix operands, sequences found by a scan.
#pragma once
#include <hip/hip_runtime.h>

#include "attn.h"
#include "exl3_device.h"

namespace ijah {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// ---- rows: 8 elements from element index i of a row matrix (16-byte aligned) as f32, and back (nearest even)
// (the type is a template argument: with a run-time one, the compiler dropped the fp16 branch of a copy whose two conversions
// cancel)
template <int TYPE>
__device__ __forceinline__ f32x8 load8(const RowMat &m, int64_t row, int col) {
  const int64_t i = row * m.ld + col;
  f32x8 o;
  if constexpr (TYPE == kRowF32) {
    const f32x4 a = *(const f32x4 *)((const float *)m.p + i), b = *(const f32x4 *)((const float *)m.p + i + 4);
#pragma unroll
    for (int k = 0; k < 4; k++) o[k] = a[k], o[4 + k] = b[k];
  } else {
    const u32x4 w = *(const u32x4 *)((const uint16_t *)m.p + i);
    if constexpr (TYPE == kRowBf16) {
#pragma unroll
      for (int k = 0; k < 4; k++) {
        o[2 * k] = __uint_as_float(w[k] << 16);
        o[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
      }
    } else {
      const f16x8 h = __builtin_bit_cast(f16x8, w);
#pragma unroll
      for (int k = 0; k < 8; k++) o[k] = (float)h[k];
    }
  }
  return o;
}
__device__ __forceinline__ u32x4 to_bf16x8(const f32x8 &v) {
  bf16x8 o;
#pragma unroll
  for (int k = 0; k < 8; k++) o[k] = (__bf16)v[k];
  return __builtin_bit_cast(u32x4, o);
}
__device__ __forceinline__ u32x4 to_f16x8(const f32x8 &v) {
  f16x8 o;
#pragma unroll
  for (int k = 0; k < 8; k++) o[k] = (_Float16)v[k];
  return __builtin_bit_cast(u32x4, o);
}
template <int TYPE>
__device__ __forceinline__ void store8(const RowMat &m, int64_t row, int col, const f32x8 &v) {
  const int64_t i = row * m.ld + col;
  if constexpr (TYPE == kRowF32) {
    float *p = (float *)m.p + i;
    *(f32x4 *)p = f32x4{v[0], v[1], v[2], v[3]};
    *(f32x4 *)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    *(u32x4 *)((uint16_t *)m.p + i) = TYPE == kRowBf16 ? to_bf16x8(v) : to_f16x8(v);
  }
}
__device__ __forceinline__ void store1(const RowMat &m, int type, int64_t row, int col, float v) {
  const int64_t i = row * m.ld + col;
  if (type == kRowF32) ((float *)m.p)[i] = v;
  else if (type == kRowBf16) ((__bf16 *)m.p)[i] = (__bf16)v;
  else ((_Float16 *)m.p)[i] = (_Float16)v;
}

// ---- 8 signed bytes as fp16 (exact): 1024 + (q + 128) by bytes, minus 1152
__device__ __forceinline__ f16x8 i8_f16(u32x2 w) {
  u32x4 o;
#pragma unroll
  for (int k = 0; k < 2; k++) {
    const uint32_t u = w[k] ^ 0x80808080u;
    o[2 * k] = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u);
    o[2 * k + 1] = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
  }
  f16x8 h = __builtin_bit_cast(f16x8, o);
#pragma unroll
  for (int k = 0; k < 8; k++) h[k] -= (_Float16)1152.f;
  return h;
}

// ---- the sequence in which item `item` of a batch lies, items(b) each: every thread of the workgroup (NT threads)
// calls this; sum: [NT / 64 + 4] words of LDS. Returns the sequence, or -1 behind the last; *before = items of the
// sequences before it, *all = of the whole batch. The sequences are divided among the threads in order, one scan over
// the threads' sums, then the thread whose range holds the item walks it.
template <int NT, typename F>
__device__ int find_item(int n, int64_t item, int64_t *sum, int64_t *before, int64_t *all, F &&items) {
  const int tid = threadIdx.x, per = (n + NT - 1) / NT, lane = tid & 63;
  const int b0 = min(tid * per, n), b1 = min(b0 + per, n);
  int64_t mine = 0;
  for (int b = b0; b < b1; b++) mine += items(b);
  int64_t inc = mine;  // inclusive scan within the wave
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t up = __shfl_up(inc, d);
    if (lane >= d) inc += up;
  }
  __syncthreads();
  if (lane == 63) sum[tid >> 6] = inc;
  if (tid == 0) sum[NT / 64] = -1;
  __syncthreads();
  int64_t base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; w++) {
    if (w < (tid >> 6)) base += sum[w];
    total += sum[w];
  }
  *all = total;
  int64_t at = base + inc - mine;
  if (item >= at && item < at + mine) {
    int b = b0;
    for (;; b++) {
      const int64_t k = items(b);
      if (item < at + k) break;
      at += k;
    }
    sum[NT / 64] = b;
    sum[NT / 64 + 1] = at;
  }
  __syncthreads();
  *before = sum[NT / 64 + 1];
  return (int)sum[NT / 64];
}

}  // namespace ijah
