// Causal attention over packed prompts with grouped heads: out_i = sum_{j <= i + nk - nq} softmax_j(scale q_i . k_j) v_j.
//
// One pass over a block's keys with the running maximum and sum of each row (f32, base 2: the scale carries log2 e). Bound
// by the matrix cores and the softmax beside them: 4 D products and about 5 vector operations (one of them an exponential
// at a quarter of the rate) per visible pair.
//
// A workgroup of four waves takes 128 query rows of one head of one sequence, a wave 32 of them; tiles of BN keys and
// values go through LDS. S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16: a lane holds one query row, so its maximum
// needs one lane swap, and the weights that the product of the keys leaves in a lane are those the product of the values
// wants there once the keys of its A operand are taken in the same order (4 half + {0..3}, 8 + 4 half + {0..3}), which
// ds_read_b64_tr_b16 reads transposed from the rows of V.
//
// 32-bit rows are cut into NT = 3 bf16 parts (8 bits each) and each product is the sum of the six part products that
// reach 2^-24: exact to f32's own rounding at six times the matrix work, with f32's range. 16-bit rows are products of
// their own type (NT = 1), the weights rounded to it (2^-9 or 2^-12 of each, as the output itself); sums are f32.
//
// Measured: fp16, 2048 rows over 16048 keys, 16 heads over 2 of 256: 539 us, 935 TFLOP/s (a library product of 8192^3 reaches
// 1213); the matrix cores are busy for 44% of their SIMDs' cycles and the vector ALUs for 42%, mostly one after the other.
// Nine packed sequences of 3231 tokens, bf16, 32 heads over 4 of 128: 38 us, the longest one's last blocks. 32 bits, 4096
// tokens, 64 heads over 8 of 64: 722 us, 1142 TFLOP/s of part products.
#include "attn_device.h"
#include "common.h"

namespace ijah {

namespace {

constexpr float kNegInf = -__builtin_inff();
constexpr int kBM = 128;  // query rows of a workgroup

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <bool F16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// x = part + rest exactly, the part in bf16
__device__ __forceinline__ u32x4 bf16_part(f32x8 &x) {
  const u32x4 w = to_bf16x8(x);
#pragma unroll
  for (int k = 0; k < 4; k++) {
    x[2 * k] -= __uint_as_float(w[k] << 16);
    x[2 * k + 1] -= __uint_as_float(w[k] & 0xFFFF0000u);
  }
  return w;
}

// Where 16-byte chunk c (8 dims) of tile row j lies in LDS, in chunks. Keys are read 32 rows of one chunk at a time, so rows
// are rotated over all chunks of 256 bytes; values are read 4 rows of a pair of chunks at a time per 16 lanes, so pairs
// stay together and four consecutive rows spread over different pairs.
template <int D>
__device__ __forceinline__ int key_chunk(int j, int c) {
  return j * (D / 8) + (c ^ (D == 64 ? (j >> 1) & 7 : j & 15));
}
template <int D>
__device__ __forceinline__ int value_chunk(int j, int c) {
  return j * (D / 8) + (c ^ (D == 64 ? (((j >> 1) & 1) << 1 | ((j >> 2) & 1)) << 1 : ((j & 3) << 1 | ((j >> 2) & 1)) << 1));
}

// the 128 query rows of a workgroup: sequence, head, first row; keys: those that some row of the block sees
struct Block {
  int h, hk, nq, nk, i0, off, keys;
  int64_t q0, k0;
};
// The blocks that see the most keys go first, so that the short ones fill the chip at the end (up to 64 sequences by their
// number of blocks, beyond that each sequence's last first). Workgroups go to the XCDs in turn: where the heads divide
// by their number, an XCD takes an eighth of them, so that the heads of a group read its keys from one L2.
template <int NT>
__device__ __forceinline__ bool find_block(const PromptArgs &a, int *sum, Block *w) {
  constexpr int kXcds = 8;
  const int blocks = gridDim.x / a.Hq, id = blockIdx.x;
  int turn;
  if (a.Hq % kXcds == 0) {
    const int per = a.Hq / kXcds, i = id / kXcds;
    w->h = id % kXcds * per + i % per;
    turn = i / per;
  } else {
    w->h = id % a.Hq;
    turn = id / a.Hq;
  }
  auto bound = [](const int *p, int b, int R) { return kv_clamp(p[b], 0, R); };
  auto q_of = [&](int b) { return max(bound(a.q_rows, b + 1, a.Rq) - bound(a.q_rows, b, a.Rq), 0); };
  auto items = [&](int i) { return (q_of(i) + kBM - 1) / kBM; };
  int b = 0, block;
  if (a.n <= 64) {
    // the longest first over all sequences: level by level of blocks from the highest, a sequence a lane
    const int lane = threadIdx.x & 63, at = min(lane, a.n - 1);
    const int q0 = bound(a.q_rows, at, a.Rq), nq = max(bound(a.q_rows, at + 1, a.Rq) - q0, 0);
    const int k0 = bound(a.k_rows, at, a.Rk), nk = max(bound(a.k_rows, at + 1, a.Rk) - k0, 0);
    const int mine = lane < a.n ? (nq + kBM - 1) / kBM : 0;
    int top = mine;
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = max(top, __shfl_xor(top, x));
    int left = turn;
    for (block = top - 1; block >= 0; block--) {
      const uint64_t has = __ballot(mine > block);
      const int c = __popcll(has);
      if (left < c) {
        // the left-th of them
        const int rank = __popcll(has & ((1ull << lane) - 1));
        b = (int)__builtin_ctzll(__ballot(mine > block && rank == left) | 1ull << 63);
        break;
      }
      left -= c;
      if (has & (has - 1)) continue;
      // one sequence has all the blocks from here on that no other reaches: straight to the next one's level
      int other = mine > block ? 0 : mine;
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) other = max(other, __shfl_xor(other, x));
      const int alone = block - other;  // levels below this one that it has alone
      if (left < alone) {
        block -= 1 + left;
        b = (int)__builtin_ctzll(has);
        break;
      }
      left -= alone;
      block -= alone;
    }
    if (block < 0) return false;
    block = __builtin_amdgcn_readfirstlane(block);
    b = __builtin_amdgcn_readfirstlane(b);
    w->nq = __builtin_amdgcn_readlane(nq, b);
    w->q0 = __builtin_amdgcn_readlane(q0, b);
    w->nk = __builtin_amdgcn_readlane(nk, b);
    w->k0 = __builtin_amdgcn_readlane(k0, b);
  } else {
    const BatchScan<NT> sc = scan_batch<NT>(a.n, sum, items);
    const int item = blocks - 1 - turn;
    if (item >= sc.total) return false;
    int before;
    b = find_item<NT>(sc, a.n, item, sum, &before, items);
    block = item - before;
    const int k0 = bound(a.k_rows, b, a.Rk);
    w->nq = q_of(b);
    w->q0 = bound(a.q_rows, b, a.Rq);
    w->nk = max(bound(a.k_rows, b + 1, a.Rk) - k0, 0);
    w->k0 = k0;
  }
  // uniform, and known to be
  w->nq = __builtin_amdgcn_readfirstlane(w->nq);
  w->q0 = __builtin_amdgcn_readfirstlane((int)w->q0);
  w->nk = __builtin_amdgcn_readfirstlane(w->nk);
  w->k0 = __builtin_amdgcn_readfirstlane((int)w->k0);
  w->i0 = __builtin_amdgcn_readfirstlane(block) * kBM;
  w->off = w->nk - w->nq;
  w->hk = w->h / (a.Hq / a.H);
  w->keys = min(w->nk, min(w->i0 + kBM, w->nq) + w->off);
  return true;
}

// ------------------------------------------------------------------------------------------------ 32-bit rows
template <int D, int BN>
__global__ __launch_bounds__(256) void attn_prompt(PromptArgs a) {
  constexpr int NT = 3, KC = D / 16, DB = D / 32, KB = BN / 32, CH = D / 8, kPlane = BN * D * 2;
  extern __shared__ __align__(16) uint8_t lds[];  // keys [NT][BN][D], values [NT][BN][D]
  __shared__ int sum[6];
  __shared__ uint32_t odd[BN], any;  // keys of the tile whose value is not finite
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5,
            col = lane & 31;
  Block w;
  if (!find_block<256>(a, sum, &w)) return;
  const int nq = w.nq, nk = w.nk, i0 = w.i0, off = w.off, hk = w.hk, h = w.h, keys = w.keys;
  const int64_t q0 = w.q0, k0 = w.k0;
  const int row = i0 + wave * 32 + col;  // this lane's query row in its sequence
  const int last = row + off;            // the last key it sees
  const int all_see = i0 + off;          // every row sees up to here

  // the wave's query rows as B operands; three parts of 256 dims are cut again for each tile (192 registers otherwise)
  constexpr bool kCut = D == 256;
  u32x4 qf[kCut ? 1 : NT][kCut ? 1 : KC];
  f32x8 q32[kCut ? KC : 1];
#pragma unroll
  for (int c = 0; c < KC; c++) {
    const int64_t r = q0 + min(row, nq - 1);
    if constexpr (kCut) {
      q32[c] = load8<kRowF32>(a.q, r, h * D + c * 16 + half * 8);
    } else {
      f32x8 x = load8<kRowF32>(a.q, r, h * D + c * 16 + half * 8);
#pragma unroll
      for (int p = 0; p < NT; p++) qf[p][c] = bf16_part(x);
    }
  }
  f32x16 o[DB];
#pragma unroll
  for (int i = 0; i < DB; i++)
#pragma unroll
    for (int k = 0; k < 16; k++) o[i][k] = 0.f;
  float mx = kNegInf, l = 0.f;
  constexpr int kLoads = BN * CH / 256;  // 8 dims of a key and of a value, of each thread
  // 128 dims: a CU has one workgroup, and registers for the next tile's rows, which are requested before this one is computed
  // (4096 tokens of 32 heads 915 -> 857 us). 64 dims have two workgroups a CU (no gain), 256 dims no registers.
  constexpr bool kAhead = D == 128;
  constexpr int kUnroll = kAhead ? kLoads : 2;
  f32x8 kn[kAhead ? kLoads : 1], vn[kAhead ? kLoads : 1];
  auto load = [&](const RowMat &m, int t0, int n) {
    const int i = n * 256 + tid;
    return load8<kRowF32>(m, k0 + min(t0 + i / CH, nk - 1), hk * D + i % CH * 8);
  };
  auto load_tile = [&](int t0) {
    if constexpr (kAhead) {
#pragma unroll
      for (int n = 0; n < kLoads; n++) {
        kn[n] = load(a.k, t0, n);
        vn[n] = load(a.v, t0, n);
      }
    }
  };
  if (keys > 0) load_tile(0);

  for (int t0 = 0; t0 < keys; t0 += BN) {
    const bool edge = t0 + BN - 1 > all_see || t0 + BN > nk;  // some row does not see some key of the tile
    __syncthreads();
    // ---- the tile into LDS; rows behind the sequence's last key are copies of it. In a tile whose keys not every row
    // sees, a value that is not finite is cleared (0 times it is not 0) and remembered.
    if (edge && tid < BN) odd[tid] = 0;
    if (tid == 0) any = 0;
    __syncthreads();
#pragma unroll kUnroll
    for (int n = 0; n < kLoads; n++) {
      const int i = n * 256 + tid, j = i / CH, c = i % CH;
      f32x8 x, y;
      if constexpr (kAhead) {
        x = kn[n];
        y = vn[n];
      } else {
        x = load(a.k, t0, n);
        y = load(a.v, t0, n);
      }
      if (edge) {
#pragma unroll
        for (int k = 0; k < 8; k++)
          if ((__float_as_uint(y[k]) & 0x7F800000u) == 0x7F800000u) {
            y[k] = 0.f;
            if (t0 + j < nk) odd[j] = any = 1;
          }
      }
#pragma unroll
      for (int p = 0; p < NT; p++) {
        *(u32x4 *)(lds + p * kPlane + key_chunk<D>(j, c) * 16) = bf16_part(x);
        *(u32x4 *)(lds + (NT + p) * kPlane + value_chunk<D>(j, c) * 16) = bf16_part(y);
      }
    }
    if (t0 + BN < keys) load_tile(t0 + BN);
    __syncthreads();
    // ---- scores: lane (row col, keys 32 kb + 8 (i / 4) + 4 half + i % 4)
    f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; kb++)
#pragma unroll
      for (int k = 0; k < 16; k++) s[kb][k] = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; kb++)
#pragma unroll
      for (int c = 0; c < KC; c++) {
        u32x4 kf[NT], qc[NT];
        if constexpr (kCut) {
          f32x8 x = q32[c];
          asm volatile("" : "+v"(x));
#pragma unroll
          for (int p = 0; p < NT; p++) qc[p] = bf16_part(x);
        } else {
#pragma unroll
          for (int p = 0; p < NT; p++) qc[p] = qf[p][c];
        }
#pragma unroll
        for (int p = 0; p < NT; p++)
          kf[p] = *(const u32x4 *)(lds + p * kPlane + key_chunk<D>(kb * 32 + col, c * 2 + half) * 16);
        // smallest products first
        s[kb] = mfma32<false>(kf[2], qc[0], s[kb]);
        s[kb] = mfma32<false>(kf[0], qc[2], s[kb]);
        s[kb] = mfma32<false>(kf[1], qc[1], s[kb]);
        s[kb] = mfma32<false>(kf[1], qc[0], s[kb]);
        s[kb] = mfma32<false>(kf[0], qc[1], s[kb]);
        s[kb] = mfma32<false>(kf[0], qc[0], s[kb]);
      }
    float top = kNegInf;
    const int seen = last - t0 - 4 * half;
#pragma unroll
    for (int kb = 0; kb < KB; kb++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        if (edge && kb * 32 + (i >> 2) * 8 + (i & 3) > min(seen, nk - 1 - t0 - 4 * half)) s[kb][i] = kNegInf;
        top = fmaxf(top, s[kb][i]);
      }
    top = fmaxf(top, xor_lane<32>(top, lane));
    // the maximum that the weights are relative to moves, and the sums with it, only where a weight would pass 2^8
    if (__ballot((top - mx) * a.scale > 8.f)) {
      const float m1 = fmaxf(mx, top), alpha = m1 == kNegInf ? 0.f : __builtin_amdgcn_exp2f((mx - m1) * a.scale);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < DB; i++) o[i] *= alpha;
      mx = m1;
    }
    const float ms = mx == kNegInf ? 0.f : mx * a.scale;
    float add = 0.f;
#pragma unroll
    for (int kb = 0; kb < KB; kb++)
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], a.scale, -ms));
        add += e;
        s[kb][i] = e;
      }
    l += add;
    // ---- sums
#pragma unroll
    for (int kg = 0; kg < BN / 16; kg++) {
      u32x4 pf[NT];
      f32x8 p;
#pragma unroll
      for (int k = 0; k < 8; k++) p[k] = s[kg >> 1][(kg & 1) * 8 + k];
#pragma unroll
      for (int k = 0; k < NT; k++) pf[k] = bf16_part(p);
#pragma unroll
      for (int i = 0; i < DB; i++) {
        u32x4 vf[NT];
#pragma unroll
        for (int k = 0; k < NT; k++) {
          // 16 lanes read 4 keys x 16 dims and get 4 keys of one dim each
          const int j = kg * 16 + half * 4 + ((lane & 15) >> 2), c = i * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
          uint8_t *base = lds + (NT + k) * kPlane + (lane & 1) * 8;
          auto tr = [&](int jj) {
            return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4 *)(base + value_chunk<D>(jj, c) * 16)));
          };
          const u32x2 v0 = tr(j), v1 = tr(j + 8);
          vf[k] = u32x4{v0[0], v0[1], v1[0], v1[1]};
        }
        o[i] = mfma32<false>(vf[2], pf[0], o[i]);
        o[i] = mfma32<false>(vf[0], pf[2], o[i]);
        o[i] = mfma32<false>(vf[1], pf[1], o[i]);
        o[i] = mfma32<false>(vf[1], pf[0], o[i]);
        o[i] = mfma32<false>(vf[0], pf[1], o[i]);
        o[i] = mfma32<false>(vf[0], pf[0], o[i]);
      }
    }
    // ---- rows that see a value that is not finite
    if (edge && any) {
      for (int j = 0; j < min(BN, nk - t0); j++) {
        if (!odd[j] || t0 + j > last) continue;
#pragma unroll
        for (int i = 0; i < DB; i++)
#pragma unroll
          for (int k = 0; k < 16; k++) {
            const int64_t at = (int64_t)(k0 + t0 + j) * a.v.ld + hk * D + i * 32 + (k >> 2) * 8 + half * 4 + (k & 3);
            const float v = ((const float *)a.v.p)[at];
            if ((__float_as_uint(v) & 0x7F800000u) == 0x7F800000u) o[i][k] = __builtin_nanf("");
          }
      }
    }
  }
  l += xor_lane<32>(l, lane);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (row < nq) {
#pragma unroll
    for (int i = 0; i < DB; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int64_t at = (q0 + row) * a.out.ld + h * D + i * 32 + k * 8 + half * 4;
        const f32x4 v = {o[i][4 * k] * inv, o[i][4 * k + 1] * inv, o[i][4 * k + 2] * inv, o[i][4 * k + 3] * inv};
        *(f32x4 *)((float *)a.out.p + at) = v;
      }
  }
}

// ------------------------------------------------------------------------------------------------ 16-bit rows
// Tiles go from HBM to LDS by DMA, the next one while this one is computed (two buffers, one barrier a tile). A DMA of a
// wave fills 1 KB of LDS in lane order, so the rotation of a row's chunks is in the addresses that the lanes read from. The
// buffer resource ends with the sequence's last key: rows behind it arrive as zeros.
template <int D, int BN>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const RowMat &m, const Block &w, int t0) {
  const uint16_t *base = (const uint16_t *)m.p + (w.k0 + t0) * m.ld + w.hk * D;
  return __builtin_amdgcn_make_buffer_rsrc((void *)base, (short)0, (min(w.nk - t0, BN) - 1) * (int)m.ld * 2 + D * 2, 0x00020000);
}

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint32_t at, void *to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)to, 16, at, 0, 0, 0);
}

//
// SPLIT 2: where there are fewer blocks than CUs, eight waves take a block, four of them every other tile each, and the two
// halves' maxima and sums are joined through LDS at the end: a SIMD has two waves then, one's products under the other's
// exponentials. (All of a block's waves meet at every barrier, so what is decided for both tiles is decided alike.)
template <int D, int BN, bool F16, int SPLIT>
__global__ __launch_bounds__(256 * SPLIT, 2) void attn_prompt16(PromptArgs a) {
  constexpr int KC = D / 16, DB = D / 32, KB = BN / 32, CH = D / 8, kTile = BN * D * 2, kRow = D * 2;
  constexpr int kDma = kTile / 1024 / 4;  // of keys, and of values, by each wave
  extern __shared__ __align__(16) uint8_t lds[];  // two buffers of SPLIT times keys [BN][D], values [BN][D]
  __shared__ int sum[4 * SPLIT + 2];
  __shared__ uint32_t odds[SPLIT][BN];  // keys of the tiles whose value is not finite
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, stream = SPLIT == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8),
            wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6 & 3);  // of the stream's four
  __shared__ float jm[SPLIT][SPLIT == 2 ? 4 : 1][64], jl[SPLIT == 2 ? 4 : 1][64];  // the streams' joins
  uint32_t *odd = odds[stream];
  Block w;
  if (!find_block<256 * SPLIT>(a, sum, &w)) return;
  auto row_of = [&](int lane) { return w.i0 + wave * 32 + (lane & 31); };  // a lane's query row in its sequence
  const int all_see = w.i0 + w.off;        // every row of the block sees up to here
  const float scale = a.scale;
  // the last key that any row of the wave sees; a tile behind it is none of its work
  const int wave_last = w.i0 + wave * 32 < w.nq ? min(w.i0 + wave * 32 + 31, w.nq - 1) + w.off : -1;

  // ---- where this lane's DMAs read: row and chunk of LDS chunk (wave * kDma + n) * 64 + lane, in bytes from the tile's first
  // row. The rotation of a row is an exclusive or with a value of the row's number (its own inverse), and the rows of n are a
  // constant apart, so one row offset and one chunk each serve all n.
  constexpr int kStep = 64 / CH;  // rows of a DMA
  auto request = [&](int t0, int buf) {
    const __amdgpu_buffer_rsrc_t rk = tile_rsrc<D, BN>(a.k, w, t0), rv = tile_rsrc<D, BN>(a.v, w, t0);
    uint8_t *to = lds + (buf * SPLIT + stream) * 2 * kTile + wave * kDma * 1024;
    const int at = D == 256 ? again(lane) : lane;  // (256 dims: computed for each tile, there are no registers to hold them)
    const int srow = wave * kDma * kStep + at / CH, schunk = at % CH;
    const uint32_t krow = (uint32_t)(srow * (int)a.k.ld * 2), vrow = (uint32_t)(srow * (int)a.v.ld * 2);
    const uint32_t kchunk = (uint32_t)(key_chunk<D>(srow, schunk) - srow * CH) * 16,
                   vchunk = (uint32_t)(value_chunk<D>(srow, schunk) - srow * CH) * 16;
#pragma unroll
    for (int n = 0; n < kDma; n++)
      dma16(rk, krow + n * kStep * (uint32_t)a.k.ld * 2 + (kchunk ^ key_chunk<D>(n * kStep, 0) % CH * 16), to + n * 1024);
#pragma unroll
    for (int n = 0; n < kDma; n++)
      dma16(rv, vrow + n * kStep * (uint32_t)a.v.ld * 2 + (vchunk ^ value_chunk<D>(n * kStep, 0) % CH * 16),
            to + kTile + n * 1024);
  };
  const int own = stream * BN;  // the stream's tile in a step's SPLIT tiles
  if (own < w.keys) request(own, 0);

  u32x4 qf[KC];
  const int64_t qr = w.q0 + min(row_of(lane), w.nq - 1);
#pragma unroll
  for (int c = 0; c < KC; c++) qf[c] = *(const u32x4 *)((const uint16_t *)a.q.p + qr * a.q.ld + w.h * D + c * 16 + half * 8);
  // ---- where this lane's operands lie in a tile: the first chunk of a key, and of the values of 16 keys 4 of them for each 4
  // lanes. The rotation is an exclusive or, so the other chunks are one too (of the low 256 bytes; the rest is an offset).
  constexpr int KA = D == 64 ? 4 : 8, VA = D == 64 ? 2 : 4;
  const int kat = key_chunk<D>(col, half) * 16;
  const int vat = kTile + value_chunk<D>(half * 4 + ((lane & 15) >> 2), ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) * 16 +
                  (lane & 1) * 8;

  // A value that is not finite must not reach rows that do not see it, as 0 times it. That takes a look at every value of the
  // tiles at the edge, so the block is first computed without; only if something in its sums is not finite is it computed
  // again with such values cleared from those tiles, and made NaN in the rows that do see them.
  f32x16 o[DB];
  float mx, l;
  for (bool careful = false;; careful = true) {
#pragma unroll
  for (int i = 0; i < DB; i++)
#pragma unroll
    for (int k = 0; k < 16; k++) o[i][k] = 0.f;
  mx = kNegInf;
  l = 0.f;
  int buf = 0;
  for (int step = 0; step < w.keys; step += SPLIT * BN, buf ^= 1) {
    const int t0 = step + own;
    // (the last step may have one tile: the other stream then computes what it finds, no key of which anyone sees)
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's part of the tile has arrived
    __syncthreads();                     // everyone's has, and the other buffer is read
    if (t0 + SPLIT * BN < w.keys) request(t0 + SPLIT * BN, buf ^ 1);
    uint8_t *tile = lds + (buf * SPLIT + stream) * 2 * kTile;
    const bool edge = step + SPLIT * BN - 1 > all_see;  // some row does not see some key of the step's tiles
    bool found = false;  // (the same for all of the workgroup)
    if (careful && edge) {
      constexpr uint32_t e = F16 ? 0x7C00u : 0x7F80u;
      bool any = false;
      const int tid = wave * 64 + again(lane);
      u32x4 *vt = (u32x4 *)(tile + kTile);
      for (int i = tid; i < BN * CH; i += 256) {
        if (t0 + i / CH >= w.nk) vt[i] = u32x4{0u, 0u, 0u, 0u};  // behind the last key
        const u32x4 y = vt[i];
#pragma unroll
        for (int k = 0; k < 4; k++) any |= (y[k] & e) == e || (y[k] >> 16 & e) == e;
      }
      if (tid < BN) odd[tid] = 0;
      found = __syncthreads_or(any) != 0;
      if (found) {
        for (int i = tid; i < BN * CH; i += 256) {
          u32x4 y = vt[i];
          uint32_t all = 0;
#pragma unroll
          for (int k = 0; k < 4; k++) {
            const uint32_t bad = ((y[k] & e) == e ? 0xFFFFu : 0u) | ((y[k] >> 16 & e) == e ? 0xFFFF0000u : 0u);
            y[k] &= ~bad;
            all |= bad;
          }
          if (all) {
            vt[i] = y;
            odd[i / CH] = 1;
          }
        }
        __syncthreads();
      }
    }
    if (t0 <= wave_last) {
    // ---- scores: lane (row col, keys 32 kb + 8 (i / 4) + 4 half + i % 4)
    const int ka = again(kat), va = again(vat);  // (the chunks' addresses are computed for each tile: registers)
    f32x16 s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; kb++)
#pragma unroll
      for (int k = 0; k < 16; k++) s[kb][k] = 0.f;
#pragma unroll
    for (int c = 0; c < KC; c++)
#pragma unroll
      for (int kb = 0; kb < KB; kb++) {
        const u32x4 kf = *(const u32x4 *)(tile + (ka ^ c % KA * 32) + kb * 32 * kRow + c / KA * (KA * 32));
        s[kb] = mfma32<F16>(kf, qf[c], s[kb]);
      }
    float top = kNegInf;
    if (edge) {
      const int seen = min(row_of(again(lane)) + w.off, w.nk - 1) - t0 - 4 * half;
#pragma unroll
      for (int kb = 0; kb < KB; kb++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (kb * 32 + (i >> 2) * 8 + (i & 3) > seen) s[kb][i] = kNegInf;
    }
#pragma unroll
    for (int kb = 0; kb < KB; kb++)
#pragma unroll
      for (int i = 0; i < 16; i++) top = fmaxf(top, s[kb][i]);
    top = fmaxf(top, xor_lane<32>(top, lane));
    // the maximum that the weights are relative to moves, and the sums with it, only where a weight would pass 2^8
    if (__ballot((top - mx) * scale > 8.f)) {
      const float m1 = fmaxf(mx, top), alpha = m1 == kNegInf ? 0.f : __builtin_amdgcn_exp2f((mx - m1) * scale);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < DB; i++) o[i] *= alpha;
      mx = m1;
    }
    const float ms = mx == kNegInf ? 0.f : mx * scale;
    float add = 0.f;
    u32x4 pf[BN / 16];
#pragma unroll
    for (int kg = 0; kg < BN / 16; kg++) {
      f32x8 p;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        p[k] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kg >> 1][(kg & 1) * 8 + k], scale, -ms));
        add += p[k];
      }
      pf[kg] = F16 ? to_f16x8(p) : to_bf16x8(p);
    }
    l += add;
    // ---- sums
#pragma unroll
    for (int kg = 0; kg < BN / 16; kg++)
#pragma unroll
      for (int i = 0; i < DB; i++) {
        // 16 lanes read 4 keys x 16 dims and get 4 keys of one dim each
        auto tr = [&](int rows) {
          return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4 *)(tile + (va ^ i % VA * 64) + (kg * 16 + rows) * kRow + i / VA * (VA * 64))));
        };
        const u32x2 v0 = tr(0), v1 = tr(8);
        o[i] = mfma32<F16>(u32x4{v0[0], v0[1], v1[0], v1[1]}, pf[kg], o[i]);
      }
    }
    // ---- rows that see a value that is not finite
    if (__builtin_expect(found, 0)) {
      const int ln = again(lane), last = row_of(ln) + w.off;  // the last key that the lane's row sees
      for (int j = 0; j < min(BN, w.nk - t0); j++) {
        if (!odd[j] || t0 + j > last) continue;
#pragma unroll
        for (int i = 0; i < DB; i++)
#pragma unroll
          for (int k = 0; k < 16; k++) {
            const int64_t at = (w.k0 + t0 + j) * a.v.ld + w.hk * D + i * 32 + (k >> 2) * 8 + (again(ln) >> 5) * 4 + (k & 3);
            const uint32_t v = ((const uint16_t *)again(a.v.p))[at], e = F16 ? 0x7C00u : 0x7F80u;
            if ((v & e) == e) o[i][k] = __builtin_nanf("");
            asm volatile("" ::: "memory");  // (one at a time: this is rare, registers are not)
          }
      }
      __syncthreads();  // `odd` is read
    }
  }
  if (careful) break;
  uint32_t worst = 0;
#pragma unroll
  for (int i = 0; i < DB; i++)
#pragma unroll
    for (int k = 0; k < 16; k++) worst = max(worst, __float_as_uint(o[i][k]) & 0x7FFFFFFFu);
  if (!__syncthreads_or(worst >= 0x7F800000u)) break;
  int first = own;
  asm volatile("" : "+s"(first));  // (computed here, not held through the first time)
  if (own < w.keys) request(first, 0);
  }
  l += xor_lane<32>(l, lane);
  if constexpr (SPLIT == 2) {  // the second stream's sums to the first, a register of all lanes at a time
    jm[stream][wave][lane] = mx;
    __syncthreads();
    const float m1 = fmaxf(mx, jm[stream ^ 1][wave][lane]);
    const float f = mx == kNegInf ? 0.f : __builtin_amdgcn_exp2f((mx - m1) * scale);
    l *= f;
#pragma unroll
    for (int i = 0; i < DB; i++) o[i] *= f;
    f32x4 *js = (f32x4 *)lds + wave * (DB * 4) * 64 + lane;
    if (stream == 1) {
#pragma unroll
      for (int i = 0; i < DB; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) js[(i * 4 + k) * 64] = f32x4{o[i][4 * k], o[i][4 * k + 1], o[i][4 * k + 2], o[i][4 * k + 3]};
      jl[wave][lane] = l;
    }
    __syncthreads();
    if (stream == 1) return;
    l += jl[wave][lane];
#pragma unroll
    for (int i = 0; i < DB; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const f32x4 v = js[(i * 4 + k) * 64];
#pragma unroll
        for (int x = 0; x < 4; x++) o[i][4 * k + x] += v[x];
        if (k == 3) asm volatile("" : "+v"(o[i]));  // (added here, not where they are stored: registers)
      }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int row = row_of(again(lane));
  const void *to = again(a.out.p);
  if (row < w.nq) {
#pragma unroll
    for (int i = 0; i < DB; i++)
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int64_t at = (w.q0 + row) * a.out.ld + w.h * D + i * 32 + k * 8 + half * 4;
        const f32x4 v = {o[i][4 * k] * inv, o[i][4 * k + 1] * inv, o[i][4 * k + 2] * inv, o[i][4 * k + 3] * inv};
        u32x2 r;
        if constexpr (F16) {
          f16x4 x;
#pragma unroll
          for (int y = 0; y < 4; y++) x[y] = (_Float16)v[y];
          r = __builtin_bit_cast(u32x2, x);
        } else {
          bf16x4 x;
#pragma unroll
          for (int y = 0; y < 4; y++) x[y] = (__bf16)v[y];
          r = __builtin_bit_cast(u32x2, x);
        }
        *(u32x2 *)((uint16_t *)to + at) = r;
      }
  }
}

// keys of a tile: what three planes of 256 dims leave room for in LDS; 16 bits: what 256 dims leave registers for
template <int D, int NT>
constexpr int kBN = D == 256 ? 32 : 64;

template <typename F>
void each(F &&f) {  // every instance: dims, parts, fp16
  auto dims = [&](auto nt, auto f16) {
    f(std::integral_constant<int, 64>(), nt, f16);
    f(std::integral_constant<int, 128>(), nt, f16);
    f(std::integral_constant<int, 256>(), nt, f16);
  };
  dims(std::integral_constant<int, 3>(), std::false_type());
  dims(std::integral_constant<int, 1>(), std::false_type());
  dims(std::integral_constant<int, 1>(), std::true_type());
}
template <int D, int NT, int SPLIT = 1>
constexpr int prompt_lds() {  // three parts of keys and values, or two buffers of them for each stream; the join's sums
  constexpr int tiles = (NT == 3 ? 6 : 4 * SPLIT) * kBN<D, NT> * D * 2, join = SPLIT == 2 ? 4 * (D / 32) * 4 * 1024 : 0;
  return tiles > join ? tiles : join;
}

}  // namespace

void launch_attn_prompt(const PromptArgs &a, hipStream_t s) {
  const int64_t blocks = std::min<int64_t>(a.Rq, ((int64_t)a.Rq + (int64_t)(kBM - 1) * a.n) / kBM);  // each sequence's last partial
  // fewer blocks than CUs, and keys enough for two streams of tiles: eight waves a block
  const bool split = blocks * a.Hq <= a.cus && a.Rk >= 512;
  each([&](auto dim, auto nt, auto f16) {
    constexpr int D = decltype(dim)::value, NT = decltype(nt)::value;
    constexpr bool F16 = decltype(f16)::value;
    if (a.D == D && a.type == (NT == 3 ? kRowF32 : F16 ? kRowF16 : kRowBf16))
    {
      const dim3 grid((unsigned)(blocks * a.Hq));
      if constexpr (NT == 3)
        hipLaunchKernelGGL((attn_prompt<D, kBN<D, NT>>), grid, dim3(256), (prompt_lds<D, NT>()), s, a);
      else if (split)
        hipLaunchKernelGGL((attn_prompt16<D, kBN<D, NT>, F16, 2>), grid, dim3(512), (prompt_lds<D, NT, 2>()), s, a);
      else
        hipLaunchKernelGGL((attn_prompt16<D, kBN<D, NT>, F16, 1>), grid, dim3(256), (prompt_lds<D, NT>()), s, a);
    }
  });
  IJ_HIP(hipGetLastError());
}

void init_decode_attrs();
void init_attn_attrs() {
  init_decode_attrs();
  each([&](auto dim, auto nt, auto f16) {
    constexpr int D = decltype(dim)::value, NT = decltype(nt)::value;
    constexpr bool F16 = decltype(f16)::value;
    auto raise = [](const void *f, int bytes) {
      IJ_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    };
    if constexpr (NT == 3) {
      raise((const void *)attn_prompt<D, kBN<D, NT>>, prompt_lds<D, NT>());
    } else {
      raise((const void *)attn_prompt16<D, kBN<D, NT>, F16, 1>, prompt_lds<D, NT>());
      raise((const void *)attn_prompt16<D, kBN<D, NT>, F16, 2>, prompt_lds<D, NT, 2>());
    }
  });
}

}  // namespace ijah
