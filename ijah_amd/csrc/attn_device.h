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

__device__ __forceinline__ int again(int v) {  // v as a value of its own from here on: what follows is computed here, not held
  asm volatile("" : "+v"(v));
  return v;
}
__device__ __forceinline__ const void *again(const void *p) {  // the same of a uniform pointer
  asm volatile("" : "+s"(p));
  return p;
}

// ---- rows: 8 elements from element index i of a row matrix (16-byte aligned) as f32, and back (nearest even)
// (the type is a template argument: with a run-time one, the compiler dropped the fp16 branch of a copy whose two conversions
// cancel)
template <int TYPE>
struct Raw8 {
  u32x4 w[TYPE == kRowF32 ? 2 : 1];
};
template <int TYPE>
__device__ __forceinline__ Raw8<TYPE> load_raw8(const RowMat &m, int64_t row, int col) {
  const int64_t i = row * m.ld + col;
  Raw8<TYPE> r;
  if constexpr (TYPE == kRowF32) {
    r.w[0] = *(const u32x4 *)((const float *)m.p + i);
    r.w[1] = *(const u32x4 *)((const float *)m.p + i + 4);
  } else {
    r.w[0] = *(const u32x4 *)((const uint16_t *)m.p + i);
  }
  return r;
}
template <int TYPE>
__device__ __forceinline__ f32x8 widen8(const Raw8<TYPE> &r) {
  f32x8 o;
  if constexpr (TYPE == kRowF32) {
#pragma unroll
    for (int k = 0; k < 8; k++) o[k] = __uint_as_float(r.w[k >> 2][k & 3]);
  } else if constexpr (TYPE == kRowBf16) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      o[2 * k] = __uint_as_float(r.w[0][k] << 16);
      o[2 * k + 1] = __uint_as_float(r.w[0][k] & 0xFFFF0000u);
    }
  } else {
    const f16x8 h = __builtin_bit_cast(f16x8, r.w[0]);
#pragma unroll
    for (int k = 0; k < 8; k++) o[k] = (float)h[k];
  }
  return o;
}
template <int TYPE>
__device__ __forceinline__ f32x8 load8(const RowMat &m, int64_t row, int col) {
  return widen8<TYPE>(load_raw8<TYPE>(m, row, col));
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

// ---- division of a batch: which sequence the item `item` lies in, with items(b) of each sequence b (32-bit totals: the
// host refuses more). Up to 256 sequences every wave scans the batch on its own, with neither LDS nor a barrier: a lane sums
// its next ceil(n / 64), one scan over the lanes, and the lane whose range holds the item walks it. More sequences are
// divided among all threads of the workgroup.
__device__ __forceinline__ int wave_scan(int x) {  // inclusive sum over the lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // a row's last lane to the next row's: rows 1, 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // lane 31 to rows 2, 3
  return x;
}
constexpr int kWaveScan = 256;
template <int NT>
struct BatchScan {
  int b0, b1, at, mine, total;  // this thread's sequences, the items before them, of them, of the batch
};
// sum: [NT / 64 + 2] words of LDS, the workgroup's from here until the last find
template <int NT, typename F>
__device__ __forceinline__ BatchScan<NT> scan_batch(int n, int *sum, F &&items) {
  BatchScan<NT> s;
  const bool wide = n > kWaveScan;
  const int t = wide ? threadIdx.x : threadIdx.x & 63, per = wide ? (n + NT - 1) / NT : (n + 63) >> 6;
  s.b0 = min(t * per, n);
  s.b1 = min(s.b0 + per, n);
  s.mine = 0;
  for (int b = s.b0; b < s.b1; b++) s.mine += items(b);
  const int inc = wave_scan(s.mine);
  s.at = inc - s.mine;
  s.total = __builtin_amdgcn_readlane(inc, 63);
  if (wide) {
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sum[threadIdx.x >> 6] = inc;
    __syncthreads();
    s.total = 0;
    for (int w = 0; w < NT / 64; w++) {
      if (w < (int)(threadIdx.x >> 6)) s.at += sum[w];
      s.total += sum[w];
    }
  }
  return s;
}
// the sequence of item `item` (uniform, < total), *before = the items of the sequences before it
template <int NT, typename F>
__device__ __forceinline__ int find_item(const BatchScan<NT> &s, int n, int item, int *sum, int *before, F &&items) {
  const bool mine = item >= s.at && item < s.at + s.mine;
  int b = s.b0, at = s.at;
  if (mine) {
    for (;; b++) {
      const int k = items(b);
      if (item < at + k || b + 1 >= s.b1) break;
      at += k;
    }
  }
  if (n > kWaveScan) {
    if (mine) {
      sum[NT / 64] = b;
      sum[NT / 64 + 1] = at;
    }
    __syncthreads();
    b = sum[NT / 64];
    at = sum[NT / 64 + 1];
  } else {
    const int lane = (int)__builtin_ctzll(__ballot(mine) | 1ull << 63);
    b = __builtin_amdgcn_readlane(b, lane);
    at = __builtin_amdgcn_readlane(at, lane);
  }
  *before = __builtin_amdgcn_readfirstlane(at);
  return __builtin_amdgcn_readfirstlane(b);
}

}  // namespace ijah
