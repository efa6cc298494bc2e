// Writing rows into the paged key-value cache and reading them back (layouts in attn.h).
//
// Write: 16 bits c = round(x); 8 bits s = max|x| f32(1 / 127) over the head's dims, c = clamp(round(x / s)). Both are copies with
// a change of layout, bound by HBM when there is enough to move and by the launch and three dependent loads (lengths,
// page id, rows) otherwise.
//
// A workgroup takes one piece (the rows of one sequence that lie in one page) of one key head, so that no two write into
// one 16-byte granule of the values. Thread (token t % 16, part t / 16) holds 8 dims of a token: a wave then reads 16
// rows x 32 dims, and its keys are 64 consecutive granules, 1 KB a store. Values go through LDS once: rows of the tile in,
// 8 keys of one dim out. A granule whose 8 keys all are the piece's is one store; at a piece's ends the values of its
// keys are stored alone, the other bytes belong to other tokens.
#include "attn_device.h"
#include "common.h"

namespace ijah {

namespace {

template <int D>
constexpr int kThreads = 2 * D;  // 16 tokens x D / 8 parts

// the tile in LDS is written and read in words of different widths
typedef uint32_t __attribute__((may_alias)) word;
typedef uint16_t __attribute__((may_alias)) half_word;

struct Piece {
  int b, page, j0, j1, nr_before;  // page id (< 0: none), tokens j0 .. j1 of it; rows before token 0
  int64_t row0;                    // the row of token j0
  int64_t lead0;                   // the first of the nr_before rows
};

// the workgroup's piece; false behind the last
template <int NT>
__device__ __forceinline__ bool find_piece(const KvSeqs &s, int item, int *sum, Piece *p) {
  int before = item, b = item;
  if (s.rows) {
    auto items = [&](int i) { return kv_pieces(kv_seq(s, i)); };
    const BatchScan<NT> sc = scan_batch<NT>(s.n, sum, items);
    if (item >= sc.total) return false;
    b = find_item<NT>(sc, s.n, item, sum, &before, items);
  }
  const KvSeq q = kv_seq(s, b);
  if (!q.nr) return false;
  const int first = q.len - q.nr, p0 = max(first, 0);  // the first row's token; the first token written
  const int k = item - before, pg = p0 / kKvPage + k;
  p->b = b;
  p->nr_before = k == 0 ? p0 - first : 0;
  p->lead0 = q.r0;
  p->j0 = k == 0 ? p0 % kKvPage : 0;
  p->j1 = min(q.len - pg * kKvPage, kKvPage);  // 0 for an empty sequence
  p->row0 = q.r0 + (int64_t)pg * kKvPage + p->j0 - first;
  p->page = -1;
  if (p->j1 > p->j0) {
    const int id = s.table[(int64_t)b * s.ldt + pg];
    if (id >= 0 && id < s.pages) p->page = id;
  }
  return true;
}

template <int KIND, int D, int TYPE>
__global__ __launch_bounds__(kThreads<D>) void kv_write(KvArgs a) {
  constexpr int NT = kThreads<D>, kPitch = D * kv_esize(KIND) + 4;  // bytes of a tile row in LDS
  __shared__ int sum[NT / 64 + 2];
  __shared__ uint32_t amax[2][NT / 64][16];
  __shared__ __align__(16) uint8_t tile[kKvPage * kPitch];
  const int tid = threadIdx.x, tok = tid & 15, part = tid >> 4, h = blockIdx.y;
  Piece p;
  if (!find_piece<NT>(a.s, (int)blockIdx.x, sum, &p) || p.page < 0) return;
  uint8_t *blk = a.base + ((int64_t)p.page * a.H + h) * kv_block_bytes(KIND, D);
  for (int g = p.j0 >> 4; g <= (p.j1 - 1) >> 4; g++) {
    const int j = g * 16 + tok;
    const bool on = j >= p.j0 && j < p.j1;
    f32x8 k, v;
    if (on) {
      k = load8<TYPE>(a.k, p.row0 + j - p.j0, h * D + part * 8);
      v = load8<TYPE>(a.v, p.row0 + j - p.j0, h * D + part * 8);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) k[i] = v[i] = 0.f;
    }
    if constexpr (KIND == kKvI8) {
      // the largest |x| as its bits: an infinity or a NaN is then larger than any number
      uint32_t mk = 0, mv = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        mk = max(mk, __float_as_uint(k[i]) & 0x7FFFFFFFu);
        mv = max(mv, __float_as_uint(v[i]) & 0x7FFFFFFFu);
      }
#pragma unroll
      for (int x = 16; x < 64; x <<= 1) {
        mk = max(mk, (uint32_t)__shfl_xor((int)mk, x));
        mv = max(mv, (uint32_t)__shfl_xor((int)mv, x));
      }
      __syncthreads();  // the round before has read its maxima
      if ((tid & 63) < 16) {
        amax[0][tid >> 6][tok] = mk;
        amax[1][tid >> 6][tok] = mv;
      }
      __syncthreads();
      for (int w = 0; w < NT / 64; w++) {
        mk = max(mk, amax[0][w][tok]);
        mv = max(mv, amax[1][w][tok]);
      }
      auto quant = [](const f32x8 &x, uint32_t m, float *step) {
        const float s = m < 0x7F800000u ? __uint_as_float(m) * (1.f / 127.f) : __builtin_nanf("");
        *step = s;
        u32x2 o = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float c = s > 0.f ? fminf(fmaxf(rintf(x[i] / s), -127.f), 127.f) : 0.f;
          o[i >> 2] |= ((uint32_t)(int)c & 0xFFu) << (8 * (i & 3));
        }
        return o;
      };
      float ks, vs;
      const u32x2 kq = quant(k, mk, &ks), vq = quant(v, mv, &vs);
      if (on) {
        *(u32x2 *)(blk + kv_key_at(KIND, D, j, part * 8)) = kq;
        if (part == 0) {
          *(float *)(blk + kv_step_at(D, 0, j)) = ks;
          *(float *)(blk + kv_step_at(D, 1, j)) = vs;
        }
      }
      word *t = (word *)(tile + j * kPitch + part * 8);
      t[0] = vq[0];
      t[1] = vq[1];
    } else {
      const u32x4 kq = KIND == kKvBf16 ? to_bf16x8(k) : to_f16x8(k), vq = KIND == kKvBf16 ? to_bf16x8(v) : to_f16x8(v);
      if (on) *(u32x4 *)(blk + kv_key_at(KIND, D, j, part * 8)) = kq;
      word *t = (word *)(tile + j * kPitch + part * 16);
#pragma unroll
      for (int i = 0; i < 4; i++) t[i] = vq[i];
    }
  }
  __syncthreads();
  // half granules: the 4 keys 16 (kg, half) + 4 quad + {0..3} of one dim
  constexpr int E = kv_esize(KIND);
  for (int i = tid; i < (D / 16) * 4 * 64; i += NT) {
    const int dl = i & 15, quad = (i >> 4) & 3, g = (i >> 6) & 3, d = (i >> 8) * 16 + dl, j = g * 16 + quad * 4;
    if (j + 4 <= p.j0 || j >= p.j1) continue;
    uint8_t *to = blk + kv_value_at(KIND, D, j, d);
    uint32_t e[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
      e[k] = E == 2 ? *(const half_word *)(tile + (j + k) * kPitch + d * 2) : tile[(j + k) * kPitch + d];
    if (j >= p.j0 && j + 4 <= p.j1) {
      if constexpr (E == 2) *(u32x2 *)to = u32x2{e[0] | e[1] << 16, e[2] | e[3] << 16};
      else *(uint32_t *)to = e[0] | e[1] << 8 | e[2] << 16 | e[3] << 24;
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (j + k >= p.j0 && j + k < p.j1) {
          if constexpr (E == 2) ((uint16_t *)to)[k] = (uint16_t)e[k];
          else to[k] = (uint8_t)e[k];
        }
    }
  }
}

template <int KIND>
__device__ __forceinline__ f32x8 widen(u32x4 w) {  // 8 cached 16-bit values
  f32x8 o;
  if constexpr (KIND == kKvBf16) {
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
  return o;
}
__device__ __forceinline__ f32x8 widen8(u32x2 w, float s) {
  f32x8 o;
#pragma unroll
  for (int k = 0; k < 8; k++) o[k] = (float)(int8_t)(w[k >> 2] >> (8 * (k & 3))) * s;
  return o;
}

template <int KIND, int D, int TYPE>
__global__ __launch_bounds__(kThreads<D>) void kv_read(KvArgs a) {
  constexpr int NT = kThreads<D>, E = kv_esize(KIND), kPitch = D * E + 4;
  __shared__ int sum[NT / 64 + 2];
  __shared__ __align__(16) uint8_t tile[kKvPage * kPitch];
  const int tid = threadIdx.x, tok = tid & 15, part = tid >> 4, h = blockIdx.y;
  Piece p;
  if (!find_piece<NT>(a.s, (int)blockIdx.x, sum, &p)) return;
  const f32x8 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int i = tok; i < p.nr_before; i += 16) {
    store8<TYPE>(a.k, p.lead0 + i, h * D + part * 8, zero);
    store8<TYPE>(a.v, p.lead0 + i, h * D + part * 8, zero);
  }
  if (p.page < 0) {
    for (int j = p.j0 + tok; j < p.j1; j += 16) {
      store8<TYPE>(a.k, p.row0 + j - p.j0, h * D + part * 8, zero);
      store8<TYPE>(a.v, p.row0 + j - p.j0, h * D + part * 8, zero);
    }
    return;
  }
  const uint8_t *blk = a.base + ((int64_t)p.page * a.H + h) * kv_block_bytes(KIND, D);
  // values: half granules (4 keys of a dim) into the tile's rows
  for (int i = tid; i < (D / 16) * 4 * 64; i += NT) {
    const int dl = i & 15, quad = (i >> 4) & 3, g = (i >> 6) & 3, d = (i >> 8) * 16 + dl, j = g * 16 + quad * 4;
    if (j + 4 <= p.j0 || j >= p.j1) continue;
    const uint8_t *from = blk + kv_value_at(KIND, D, j, d);
    if constexpr (E == 2) {
      const u32x2 w = *(const u32x2 *)from;
#pragma unroll
      for (int k = 0; k < 4; k++) *(half_word *)(tile + (j + k) * kPitch + d * 2) = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
    } else {
      const uint32_t w = *(const uint32_t *)from;
#pragma unroll
      for (int k = 0; k < 4; k++) tile[(j + k) * kPitch + d] = (uint8_t)(w >> (8 * k));
    }
  }
  __syncthreads();
  for (int g = p.j0 >> 4; g <= (p.j1 - 1) >> 4; g++) {
    const int j = g * 16 + tok;
    if (j < p.j0 || j >= p.j1) continue;
    f32x8 k, v;
    if constexpr (KIND == kKvI8) {
      k = widen8(*(const u32x2 *)(blk + kv_key_at(KIND, D, j, part * 8)), *(const float *)(blk + kv_step_at(D, 0, j)));
      const word *t = (const word *)(tile + j * kPitch + part * 8);
      v = widen8(u32x2{t[0], t[1]}, *(const float *)(blk + kv_step_at(D, 1, j)));
    } else {
      k = widen<KIND>(*(const u32x4 *)(blk + kv_key_at(KIND, D, j, part * 8)));
      const word *t = (const word *)(tile + j * kPitch + part * 16);
      v = widen<KIND>(u32x4{t[0], t[1], t[2], t[3]});
    }
    store8<TYPE>(a.k, p.row0 + j - p.j0, h * D + part * 8, k);
    store8<TYPE>(a.v, p.row0 + j - p.j0, h * D + part * 8, v);
  }
}

template <typename F>
void each(F &&f) {  // every instance: cache kind, dim, row type
  auto types = [&](auto kind, auto dim) {
    f(kind, dim, std::integral_constant<int, kRowF32>());
    f(kind, dim, std::integral_constant<int, kRowBf16>());
    f(kind, dim, std::integral_constant<int, kRowF16>());
  };
  auto dims = [&](auto kind) {
    types(kind, std::integral_constant<int, 64>());
    types(kind, std::integral_constant<int, 128>());
    types(kind, std::integral_constant<int, 256>());
  };
  dims(std::integral_constant<int, kKvBf16>());
  dims(std::integral_constant<int, kKvF16>());
  dims(std::integral_constant<int, kKvI8>());
}
void launch(const KvArgs &a, bool write, hipStream_t s) {
  const dim3 grid((unsigned)kv_max_pieces(a.s.n, a.s.R, a.s.rows != nullptr), (unsigned)a.H);
  each([&](auto kind, auto dim, auto type) {
    constexpr int K = decltype(kind)::value, D = decltype(dim)::value, T = decltype(type)::value;
    if (a.kind != K || a.D != D || a.type != T) return;
    if (write) hipLaunchKernelGGL((kv_write<K, D, T>), grid, dim3(kThreads<D>), 0, s, a);
    else hipLaunchKernelGGL((kv_read<K, D, T>), grid, dim3(kThreads<D>), 0, s, a);
  });
  IJ_HIP(hipGetLastError());
}

}  // namespace

void launch_kv_write(const KvArgs &a, hipStream_t s) { launch(a, true, s); }
void launch_kv_read(const KvArgs &a, hipStream_t s) { launch(a, false, s); }

}  // namespace ijah
