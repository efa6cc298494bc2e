// Writing rows into the paged key-value cache and reading them back (layouts in attn.h).
//
// Write: 16 bits c = round(x); 8 bits s = max|x| f32(1 / 127) over the head's dims, c = clamp(round(x / s)). Both are copies with
// a change of layout, bound by HBM when there is enough to move and by the launch and three dependent loads (lengths,
// page id, rows) otherwise. 16 sequences of 4096 tokens, 8 heads of 128, bf16 rows: write 110 us (4.9 TB/s) into 16 bits, 89 us
// (4.5 TB/s) into 8; read 107 us (5.0 TB/s) and 92 us (4.4 TB/s). A large copy reaches 5.1 TB/s.
//
// Many rows: a workgroup takes one piece (the rows of one sequence that lie in one page) of one key head, so that no two
// write into one 16-byte granule of the values. Thread (token t % 16, part t / 16) holds 8 dims of a token: a wave then
// reads 16 rows x 32 dims, and its keys are 64 consecutive granules, 1 KB a store. The rows are held as they were loaded until
// their turn: widened they took 172 registers with 8 bits, two waves a SIMD, and 177 us for the write above. Values go
// through LDS once: rows of the tile in, 8 keys of one dim out. A granule whose 8 keys all are the piece's is one store; at a
// piece's ends the values of its keys are stored alone, the other bytes belong to other tokens.
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

// 8 of a row's elements in steps of its largest magnitude (as bits: an infinity or a NaN is larger than any number) / 127.
// x times the step's reciprocal is within 127 (2^-24 + 2^-24) < 2^-15 of the f32 quotient, so both round to the same integer
// unless the product lies within 2^-14 of a half (1 element in 8192) or the reciprocal overflows: then the quotient itself.
__device__ __forceinline__ u32x2 quantise(const f32x8 &x, uint32_t m, float *step) {
  constexpr float kInt = 0x1.8p23f;  // added: a product rounded to an integer, which is the sum's low bits
  const float s = m < 0x7F800000u ? __uint_as_float(m) * (1.f / 127.f) : __builtin_nanf("");
  *step = s;
  const float inv = 1.f / s;
  uint32_t q[8];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const float f = __builtin_fmaf(x[i], inv, kInt);
    far = fmaxf(far, fabsf(__builtin_fmaf(x[i], inv, -(f - kInt))));
    q[i] = __float_as_uint(f);
  }
  if (far > 0.5f - 0x1p-14f || !(inv < 0x1p126f)) {
#pragma unroll
    for (int i = 0; i < 8; i++) q[i] = (uint32_t)(int)(s > 0.f ? fminf(fmaxf(rintf(x[i] / s), -127.f), 127.f) : 0.f);
  }
  u32x2 o;
#pragma unroll
  for (int i = 0; i < 2; i++)
    o[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(q[4 * i + 3], q[4 * i + 2], 0x0C0C0400u),
                                 __builtin_amdgcn_perm(q[4 * i + 1], q[4 * i], 0x0C0C0400u), 0x05040100u);
  return o;
}

template <int KIND, int D, int TYPE>
__global__ __launch_bounds__(kThreads<D>) void kv_write(KvArgs a) {
  constexpr int NT = kThreads<D>, kPitch = D * kv_esize(KIND) + 4;  // bytes of a tile row in LDS
  __shared__ int sum[NT / 64 + 2];
  __shared__ uint32_t amax[2][4][NT / 64][16];
  __shared__ __align__(16) uint8_t tile[kKvPage * kPitch];
  const int tid = threadIdx.x, tok = tid & 15, part = tid >> 4, h = blockIdx.y;
  Piece p;
  if (!find_piece<NT>(a.s, (int)blockIdx.x, sum, &p) || p.page < 0) return;
  uint8_t *blk = a.base + ((int64_t)p.page * a.H + h) * kv_block_bytes(KIND, D);
  // all of the piece's rows are requested at once: four groups of 16 tokens
  Raw8<TYPE> kr[4] = {}, vr[4] = {};
#pragma unroll
  for (int g = 0; g < 4; g++) {
    const int j = g * 16 + tok;
    if (j >= p.j0 && j < p.j1) {
      kr[g] = load_raw8<TYPE>(a.k, p.row0 + j - p.j0, h * D + part * 8);
      vr[g] = load_raw8<TYPE>(a.v, p.row0 + j - p.j0, h * D + part * 8);
    }
  }
  if constexpr (KIND == kKvI8) {
    // the largest |x| as its bits: an infinity or a NaN is then larger than any number
#pragma unroll
    for (int g = 0; g < 4; g++) {
      uint32_t mk = 0, mv = 0;
      const f32x8 k = widen8<TYPE>(kr[g]), v = widen8<TYPE>(vr[g]);
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
      if ((tid & 63) < 16) {
        amax[0][g][tid >> 6][tok] = mk;
        amax[1][g][tid >> 6][tok] = mv;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int g = 0; g < 4; g++) {
    const int j = g * 16 + tok;
    const bool on = j >= p.j0 && j < p.j1;
    const f32x8 k = widen8<TYPE>(kr[g]), v = widen8<TYPE>(vr[g]);
    if constexpr (KIND == kKvI8) {
      uint32_t mk = 0, mv = 0;
#pragma unroll
      for (int w = 0; w < NT / 64; w++) {
        mk = max(mk, amax[0][g][w][tok]);
        mv = max(mv, amax[1][g][w][tok]);
      }
      if (on) {
        float ks, vs;
        const u32x2 kq = quantise(k, mk, &ks), vq = quantise(v, mv, &vs);
        *(u32x2 *)(blk + kv_key_at(KIND, D, j, part * 8)) = kq;
        if (part == 0) {
          *(float *)(blk + kv_step_at(D, 0, j)) = ks;
          *(float *)(blk + kv_step_at(D, 1, j)) = vs;
        }
        word *t = (word *)(tile + j * kPitch + part * 8);
        t[0] = vq[0];
        t[1] = vq[1];
      }
    } else if (on) {
      *(u32x4 *)(blk + kv_key_at(KIND, D, j, part * 8)) = KIND == kKvBf16 ? to_bf16x8(k) : to_f16x8(k);
      const u32x4 vq = KIND == kKvBf16 ? to_bf16x8(v) : to_f16x8(v);
      word *t = (word *)(tile + j * kPitch + part * 16);
#pragma unroll
      for (int i = 0; i < 4; i++) t[i] = vq[i];
    }
  }
  __syncthreads();
  // granules of the values: the keys 4 quad + {0..3} of two groups of 16 (8 bits: of all four) of one dim
  constexpr int E = kv_esize(KIND), G = E == 2 ? 2 : 4;  // groups of a granule
  for (int i = tid; i < (D / 16) * (4 / G) * 64; i += NT) {
    const int dl = i & 15, quad = (i >> 4) & 3, g0 = (i >> 6) % (4 / G) * G, d = (i >> 6) / (4 / G) * 16 + dl;
    const int first = g0 * 16 + quad * 4, last = first + (G - 1) * 16 + 3;
    if (last < p.j0 || first >= p.j1) continue;
    uint8_t *to = blk + kv_value_at(KIND, D, first, d);
    u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int n = 0; n < 4; n++) {
        const int j = first + g * 16 + n, at = (g * 4 + n) * E;  // its byte in the granule
        const uint32_t e = E == 2 ? *(const half_word *)(tile + j * kPitch + d * 2) : tile[j * kPitch + d];
        w[at >> 2] |= e << (at & 3) * 8;
      }
    if (first >= p.j0 && last < p.j1) {
      *(u32x4 *)to = w;
      continue;
    }
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int n = 0; n < 4; n++) {
        const int j = first + g * 16 + n, at = (g * 4 + n) * E;
        if (j >= p.j0 && j < p.j1) {
          const uint32_t e = w[at >> 2] >> (at & 3) * 8;
          if constexpr (E == 2) *(uint16_t *)(to + at) = (uint16_t)e;
          else to[at] = (uint8_t)e;
        }
      }
  }
}

// Few rows of each sequence (a decode step, drafts): a wave takes one row and as many heads as it has lanes for, 8 dims a lane.
// The row's sequence by bisection of the row table (uniform, through the scalar cache); nothing is shared, so there is no LDS
// and no barrier, and a value's dims are stored one by one, 16 bytes apart.
template <int KIND, int D, int TYPE>
__global__ __launch_bounds__(256) void kv_write_rows(KvArgs a) {
  constexpr int kParts = D / 8, kHeads = 64 / kParts;
  const int lane = threadIdx.x & 63, part = lane % kParts;
  const int row = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int h = blockIdx.y * kHeads + lane / kParts;
  if (row >= a.s.R || (!a.s.rows && row >= a.s.n)) return;
  int b = row;
  if (a.s.rows) {  // the last sequence that begins at or before the row
    b = 0;
    for (int lo = 1, hi = a.s.n; lo < hi;) {
      const int mid = (lo + hi) >> 1;
      if (a.s.rows[mid] <= row) b = mid, lo = mid + 1;
      else hi = mid;
    }
  }
  const KvSeq q = kv_seq(a.s, b);
  const int p = q.len - q.nr + row - q.r0;  // the row's token
  if (row < q.r0 || row >= q.r0 + q.nr || p < 0) return;
  const int id = a.s.table[(int64_t)b * a.s.ldt + p / kKvPage], j = p % kKvPage;
  if (id < 0 || id >= a.s.pages || h >= a.H) return;
  uint8_t *blk = a.base + ((int64_t)id * a.H + h) * kv_block_bytes(KIND, D);
  const f32x8 k = load8<TYPE>(a.k, row, h * D + part * 8), v = load8<TYPE>(a.v, row, h * D + part * 8);
  if constexpr (KIND == kKvI8) {
    uint32_t mk = 0, mv = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      mk = max(mk, __float_as_uint(k[i]) & 0x7FFFFFFFu);
      mv = max(mv, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    }
#pragma unroll
    for (int x = 1; x < kParts; x <<= 1) {
      mk = max(mk, (uint32_t)__shfl_xor((int)mk, x));
      mv = max(mv, (uint32_t)__shfl_xor((int)mv, x));
    }
    float ks, vs;
    const u32x2 kq = quantise(k, mk, &ks), vq = quantise(v, mv, &vs);
    *(u32x2 *)(blk + kv_key_at(KIND, D, j, part * 8)) = kq;
    if (part == 0) {
      *(float *)(blk + kv_step_at(D, 0, j)) = ks;
      *(float *)(blk + kv_step_at(D, 1, j)) = vs;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) blk[kv_value_at(KIND, D, j, part * 8 + i)] = (uint8_t)(vq[i >> 2] >> 8 * (i & 3));
  } else {
    *(u32x4 *)(blk + kv_key_at(KIND, D, j, part * 8)) = KIND == kKvBf16 ? to_bf16x8(k) : to_f16x8(k);
    const u32x4 vq = KIND == kKvBf16 ? to_bf16x8(v) : to_f16x8(v);
#pragma unroll
    for (int i = 0; i < 8; i++)
      *(uint16_t *)(blk + kv_value_at(KIND, D, j, part * 8 + i)) = (uint16_t)(vq[i >> 1] >> 16 * (i & 1));
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
  // everything is requested at once: the keys' chunks, the steps, the granules of the values
  constexpr int G = E == 2 ? 2 : 4, VN = (D / 16) * (4 / G) * 64 / NT;  // 16-token groups of a granule; granules of a thread
  u32x4 kq[4], vq[VN];
  float ks[4], vs[4];
#pragma unroll
  for (int g = 0; g < 4; g++) {
    const int j = g * 16 + tok;
    if constexpr (KIND == kKvI8) {
      const u32x2 w = *(const u32x2 *)(blk + kv_key_at(KIND, D, j, part * 8));
      kq[g] = u32x4{w[0], w[1], 0u, 0u};
      ks[g] = *(const float *)(blk + kv_step_at(D, 0, j));
      vs[g] = *(const float *)(blk + kv_step_at(D, 1, j));
    } else {
      kq[g] = *(const u32x4 *)(blk + kv_key_at(KIND, D, j, part * 8));
    }
  }
#pragma unroll
  for (int n = 0; n < VN; n++) {
    const int i = n * NT + tid, d = (i >> 6) / (4 / G) * 16 + (i & 15), first = (i >> 6) % (4 / G) * G * 16 + ((i >> 4) & 3) * 4;
    vq[n] = *(const u32x4 *)(blk + kv_value_at(KIND, D, first, d));
  }
  // (what lies outside of the piece is another's or nobody's: it is read, and goes nowhere)
#pragma unroll
  for (int n = 0; n < VN; n++) {
    const int i = n * NT + tid, d = (i >> 6) / (4 / G) * 16 + (i & 15), first = (i >> 6) % (4 / G) * G * 16 + ((i >> 4) & 3) * 4;
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const int at = (g * 4 + x) * E;
        const uint32_t e = vq[n][at >> 2] >> (at & 3) * 8;
        uint8_t *t = tile + (first + g * 16 + x) * kPitch + d * E;
        if constexpr (E == 2) *(half_word *)t = (uint16_t)e;
        else *t = (uint8_t)e;
      }
  }
  __syncthreads();
#pragma unroll
  for (int g = 0; g < 4; g++) {
    const int j = g * 16 + tok;
    if (j < p.j0 || j >= p.j1) continue;
    f32x8 k, v;
    if constexpr (KIND == kKvI8) {
      const word *t = (const word *)(tile + j * kPitch + part * 8);
      k = widen8(u32x2{kq[g][0], kq[g][1]}, ks[g]);
      v = widen8(u32x2{t[0], t[1]}, vs[g]);
    } else {
      const word *t = (const word *)(tile + j * kPitch + part * 16);
      k = widen<KIND>(kq[g]);
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
  // Few rows of a sequence: by rows, as a piece's workgroup of 64 tokens would idle; many: by pieces, whose stores are whole
  // granules. Row kernel / piece kernel with 256 sequences, 8 heads of 128, us: 16 bits, 1 row each 5.2 / 11.1, 8 rows 14 / 18,
  // 16 rows 34 / 21, 64 rows 88 / 39; 8 bits 5.7 / 15.5, 15 / 22, 26 / 25, 86 / 52.
  const bool few = a.s.R <= 12 * (int64_t)a.s.n;
  each([&](auto kind, auto dim, auto type) {
    constexpr int K = decltype(kind)::value, D = decltype(dim)::value, T = decltype(type)::value;
    if (a.kind != K || a.D != D || a.type != T) return;
    constexpr int kHeads = 512 / D;  // of a wave in kv_write_rows
    if (write && few)
      hipLaunchKernelGGL((kv_write_rows<K, D, T>), dim3((a.s.R + 3) / 4, (a.H + kHeads - 1) / kHeads), dim3(256), 0, s, a);
    else if (write) hipLaunchKernelGGL((kv_write<K, D, T>), grid, dim3(kThreads<D>), 0, s, a);
    else hipLaunchKernelGGL((kv_read<K, D, T>), grid, dim3(kThreads<D>), 0, s, a);
  });
  IJ_HIP(hipGetLastError());
}

}  // namespace

void launch_kv_write(const KvArgs &a, hipStream_t s) { launch(a, true, s); }
void launch_kv_read(const KvArgs &a, hipStream_t s) { launch(a, false, s); }

}  // namespace ijah
