// Attention of a batch's newest tokens over the paged cache (layouts and the division of work in attn.h).
//
// With s_mj = scale q_m . k_j for the keys j that row m sees, o_m = sum_j e^(s_mj - M_m) v_j / sum_j e^(s_mj - M_m): one pass
// over the pages with the running maximum M and sum L of each row, in f32 and base 2 (the scale carries log2 e). Bound by
// HBM: every key and value is read once, for all query heads of its key head (and all drafts of its sequence) together.
//
// A wave takes a page of 64 keys at a time: S^T = K Q^T on v_mfma_f32_16x16x32 (A: 16 keys, straight from the page's
// granules; B: 16 query rows, from LDS), the softmax in registers (a lane holds one row's keys; quads share rows, so a
// maximum is two lane swaps), O^T += V^T P^T (A: 16 dims; B: the weights, which the page's value order leaves in the right
// lanes). Rows and weights are f32 cut into NS parts of 8 or 11 bits (bf16: three, fp16: two), so that the products carry
// the f32 operand whole; keys and values are what the cache holds, exactly. The matrix cores have the room: 16 x 32
// elements take 16 cycles of one SIMD, HBM brings a CU 6.5 bf16 elements a cycle.
//
// fp16 parts have fp16's range: a query row is scaled by the power of two that brings its largest element under 1 (taken
// back in the scores), weights are 2^14 times themselves (so are the sums L), and the steps of 8-bit values, which are
// weights' factors, are taken relative to the largest power of two that the wave has met (taken back at the end). What a
// part then drops is 2^-24 of the largest element or weight at most.
//
// Work is dealt out in units of a page over as many workgroups as the chip holds (two a CU, one with 256 dims), so a single
// long sequence and a ragged batch fill it alike: one chunk of a group for each workgroup where the groups fit them, else equal
// shares; the device does it, so a captured call follows the lengths. A workgroup's waves take a segment's pages in turn and
// are joined through LDS, the parts of one group through memory by the last of them to arrive (a counter; partials are
// device-coherent stores, so no cache is written back or invalidated). Many rows (drafts, or more than 16 query heads to a
// key head) go in blocks of 32, two blocks of a group side by side so that their reads of a page meet in the caches, and
// their parts are joined by a launch of their own.
//
// Measured: one sequence of 131072 tokens, 2 key heads of 256, bf16: 64 us for 268 MB (4.2 TB/s; a large copy reaches 5.1). 48
// ragged sequences of up to 4000 tokens, 4 key heads of 128, 8 bits: 24 us for 70 MB. One of 37 tokens: 7.5 us, of which the
// call's host side is 5. Sixteen sequences of up to 16000 tokens with up to six drafts of 80 heads over 5 of 128: 76 us for
// 203 MB and 38 GFLOP of part products (40 and 30 us), as products and exponentials of one SIMD overlap little.
#include "attn_device.h"
#include "common.h"

namespace ijah {

namespace {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

constexpr float kNegInf = -__builtin_inff();

// A workgroup has four waves; with up to 128 dims two of them share a CU (256 registers a wave), so that one's joins and
// first requests pass under the other's pages. With 256 dims a wave's keys, values and sums take up to 512 registers.
constexpr int NW = 4, NT = 64 * NW;
IJ_HD constexpr int per_cu(int D) { return D == 256 ? 1 : 2; }

template <int KIND>
struct Num {  // the matrix type of a cache kind, and the parts an f32 operand is cut into
  static constexpr int NS = KIND == kKvBf16 ? 3 : 2;
};

template <int KIND>
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (KIND == kKvBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// the parts of 1, and whether one of a register's two values is not finite (its exponent all ones)
template <int KIND>
constexpr uint32_t kOne = KIND == kKvBf16 ? 0x3F80u : 0x3C00u;
template <int KIND>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {  // all ones in the halves that are not
  constexpr uint32_t e = KIND == kKvBf16 ? 0x7F80u : 0x7C00u;
  return ((w & e) == e ? 0xFFFFu : 0u) | ((w >> 16 & e) == e ? 0xFFFF0000u : 0u);
}
// x = part + rest exactly (the subtraction of a value's own rounding is exact)
template <int KIND>
__device__ __forceinline__ u32x4 part_of(f32x8 &x) {
  const u32x4 w = KIND == kKvBf16 ? to_bf16x8(x) : to_f16x8(x);
  if constexpr (KIND == kKvBf16) {
#pragma unroll
    for (int k = 0; k < 4; k++) {
      x[2 * k] -= __uint_as_float(w[k] << 16);
      x[2 * k + 1] -= __uint_as_float(w[k] & 0xFFFF0000u);
    }
  } else {
    const f16x8 h = __builtin_bit_cast(f16x8, w);
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] -= (float)h[k];
  }
  return w;
}

// 16 bytes of a partial, device-coherent (sc1: past the XCD's own L2), by byte offset in the partials
__device__ __forceinline__ f32x4 part_load(__amdgpu_buffer_rsrc_t r, uint32_t at) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 16));
}
__device__ __forceinline__ void part_store(__amdgpu_buffer_rsrc_t r, uint32_t at, f32x4 v) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, (int)at, 0, 16);
}

// four output elements: dims d .. of the row-th of a sequence's rows of key head h (token, then query head)
template <int D>
__device__ __forceinline__ void store4(const DecArgs &a, int r0, int h, int row, int d, f32x4 v) {
  const int group = a.Hq / a.H, t = row / group;
  const int64_t at = (r0 + t) * a.out.ld + (h * group + row - t * group) * D + d;
  if (a.type == kRowF32) {
    *(f32x4 *)((float *)a.out.p + at) = v;
    return;
  }
  u32x2 w;
  if (a.type == kRowBf16) {
    bf16x4 o4;
#pragma unroll
    for (int k = 0; k < 4; k++) o4[k] = (__bf16)v[k];
    w = __builtin_bit_cast(u32x2, o4);
  } else {
    f16x4 o4;
#pragma unroll
    for (int k = 0; k < 4; k++) o4[k] = (_Float16)v[k];
    w = __builtin_bit_cast(u32x2, o4);
  }
  *(u32x2 *)((uint16_t *)a.out.p + at) = w;
}

// the place of a segment in the batch
struct Group {
  int b, h, rb;  // sequence, key head, which of the sequence's row groups
  KvSeq q;
  DecSeq d;
  int u0;        // the group's first unit (shares), or 0
};

template <int KIND, int D, int RT>
__global__ __launch_bounds__(NT, per_cu(D)) void attn_decode(DecArgs a) {
  constexpr int NS = Num<KIND>::NS, BR = 16 * RT, NB = RT;  // NB: row blocks of a group at most
  constexpr int KC = D / 32;                       // products of 32 dims
  constexpr int KG = KIND == kKvI8 ? KC / 2 : KC;  // granules of 16 keys
  constexpr int DB = D / 16;
  constexpr int VG = KIND == kKvI8 ? 1 : 2;        // granules of 16 dims
  constexpr int BLK = kv_block_bytes(KIND, D), SLOT = dec_slot_floats(D);
  constexpr bool F16 = KIND != kKvBf16;
  constexpr float kLift = F16 ? 14.f : 0.f;
  constexpr bool kAhead = RT == 1;  // the next page's keys are requested a page ahead (two row tiles leave no registers)
  constexpr int kPitch = D + 4;     // of a row of sums in LDS
  // LDS: the query parts [NS][NB][RT][KC][64 lanes] granules; then the waves' sums [NW][BR][kPitch] for their join; then the
  // maxima and sums of the parts that are joined
  extern __shared__ __align__(16) uint8_t lds[];
  u32x4 *qf = (u32x4 *)lds;
  float *js = (float *)lds;
  __shared__ int sum[NW + 2];
  __shared__ float wm[NW][BR], wl[NW][BR];
  float(*pm)[NB * BR] = (float(*)[NB * BR])lds, (*pl)[NB * BR] = pm + kJoins;
  __shared__ int flag;
  __shared__ uint32_t qmax[NB * BR];

  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), quad = lane >> 4,
            col = lane & 15;
  const int group = a.Hq / a.H, W = a.W, me = blockIdx.x;
  auto load_q = [&](int64_t row, int c) {
    return a.type == kRowF32    ? load8<kRowF32>(a.q, row, c)
           : a.type == kRowBf16 ? load8<kRowBf16>(a.q, row, c)
                                : load8<kRowF16>(a.q, row, c);
  };
  // ---- the share
  if (a.apart && tid == 0) a.joins[me].parts = 0;
  auto seq_of = [&](int b) { return dec_seq(kv_seq(a.s, b), group, BR, NB); };
  bool aligned = false;
  int C = 0, chunk = 0, share = 0, u_hi = 0, u = 0;
  Group g;
  {
    int before, k;
    if (a.s.n <= kWaveScan) {
      // every wave for itself; a lane holds up to kPer consecutive sequences
      constexpr int kPer = kWaveScan / 64;
      const int per = (a.s.n + 63) >> 6;
      int un[kPer], gr[kPer], all = 0, groups = 0;  // units of a group, groups; of the lane's sequences
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const int b = lane * per + i;
        un[i] = gr[i] = 0;
        if (i < per && b < a.s.n) {
          const DecSeq d = seq_of(b);
          un[i] = dec_group(d);
          gr[i] = d.blocks * a.H;
        }
        all += un[i] * gr[i];
        groups += gr[i];
      }
      int mine = all, inc = wave_scan(mine);
      all = __builtin_amdgcn_readlane(inc, 63);
      groups = __builtin_amdgcn_readlane(wave_scan(groups), 63);
      if (all == 0) return;
      share = (int)(((uint32_t)all + (uint32_t)W - 1) / (uint32_t)W);
      // chunks of up to four pages a wave more than an equal share, if the groups then fit the workgroups: a second segment
      // (its first loads, its join) costs a workgroup about as much as three more pages for each wave
      if (groups <= W) {
        C = max((share + NW - 1) / NW, RT == 1 ? 1 : 2) * NW;  // (many rows: a part costs about as much as a page)
        for (int t = 0; t < 4 && !aligned; t++, C += aligned ? 0 : NW) {
          int m = 0;
#pragma unroll
          for (int i = 0; i < kPer; i++) m += (int)((uint32_t)(un[i] + C - 1) / (uint32_t)C) * gr[i];
          const int c = wave_scan(m);
          if (__builtin_amdgcn_readlane(c, 63) <= W) {
            aligned = true;
            mine = m;
            inc = c;
            all = __builtin_amdgcn_readlane(c, 63);
          }
        }
      }
      const int item = aligned ? me : share * me;
      if (item >= all) return;
      if (!aligned) {
        u = item;
        u_hi = share < all - u ? u + share : all;
      }
      int at = inc - mine, b = lane * per;
      const uint64_t holds = __ballot(item >= at && item < at + mine);
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const int k = (aligned ? (int)((uint32_t)(un[i] + C - 1) / (uint32_t)C) : un[i]) * gr[i];
        if (i + 1 < per && item >= at + k && b == lane * per + i) {
          at += k;
          b++;
        }
      }
      const int from = (int)__builtin_ctzll(holds | 1ull << 63);
      g.b = __builtin_amdgcn_readlane(b, from);
      before = __builtin_amdgcn_readlane(at, from);
      k = item - before;
    } else {
      auto units = [&](int b) { return dec_units(seq_of(b), a.H); };
      const BatchScan<NT> sc = scan_batch<NT>(a.s.n, sum, units);
      share = (int)(((uint32_t)sc.total + (uint32_t)W - 1) / (uint32_t)W);
      if (share * (int64_t)me >= sc.total) return;
      u = share * me;
      u_hi = share < sc.total - u ? u + share : sc.total;
      g.b = find_item<NT>(sc, a.s.n, u, sum, &before, units);
      k = u - before;
    }
    g.q = kv_seq(a.s, g.b);
    g.d = dec_seq(g.q, group, BR, NB);
    const int size = aligned ? dec_chunks(g.d, C) : dec_group(g.d), i = k / size;
    g.h = i / g.d.blocks;
    g.rb = i - g.h * g.d.blocks;
    g.u0 = aligned ? 0 : before + i * size;
    chunk = k - i * size;
  }
  // of the two workgroups of a CU one goes first, so that one's products run beside the other's exponentials and not beside its
  // products (drafts of 16 sequences 87.5 -> 83.8 us)
  if (per_cu(D) == 2 && (me >> 8 & 1)) __builtin_amdgcn_s_setprio(1);
  for (;;) {  // one segment
    const int size = dec_group(g.d), lo = aligned ? chunk * C : u - g.u0,
              hi = aligned ? min(lo + C, size) : min(u_hi - g.u0, size);  // its units of the group
    const int real = (g.q.len + kKvPage - 1) / kKvPage;  // pages (none: an empty sequence)
    const int pg0 = dec_page(g.d, lo, real), pg1 = dec_page(g.d, hi, real);
    const DecPart part = aligned ? dec_part_chunk(chunk, dec_chunks(g.d, C), me) : dec_part_share(g.u0, g.u0 + size, share);
    const int nb = g.d.nb, row0 = g.rb * nb * BR, nrows = min(g.q.nr * group - row0, nb * BR);  // the group's rows
    // the wave's row block and its turn at the pages: every (NW / nb)-th
    const int wb = nb == 1 ? 0 : wave & 1, ws = nb == 1 ? wave : wave >> 1, step = nb == 1 ? NW : NW / 2;
    const int wrow0 = row0 + wb * BR, wrows = nrows - wb * BR;
    const int *table = a.s.table + (int64_t)g.b * a.s.ldt;
    const int turns = pg0 + ws < pg1 ? (pg1 - pg0 - ws + step - 1) / step : 0;
    // the page ids of the wave's next 64 turns, one a lane
    auto load_ids = [&](int t) { return table[min(pg0 + ws + (t + lane) * step, pg1 - 1)]; };
    int ids = 0, id = 0;
    u32x4 kf[4][KG], vf[DB][VG];
    auto valid = [&](int i) { return i >= 0 && i < a.s.pages; };
    auto block = [&](int i) { return a.base + ((int64_t)(valid(i) ? i : 0) * a.H + g.h) * BLK; };
    auto load_keys = [&](int i) {
      const u32x4 *kp = (const u32x4 *)block(i) + lane;
#pragma unroll
      for (int kb = 0; kb < 4; kb++)
#pragma unroll
        for (int c = 0; c < KG; c++) kf[kb][c] = kp[(kb * KG + c) * 64];
    };
    if (turns) {
      ids = load_ids(0);
      id = __builtin_amdgcn_readlane(ids, 0);
      if constexpr (kAhead) load_keys(id);
    }
    // ---- the group's query rows, scaled, in parts: granule (part, block, tile, chunk, lane) = 8 dims of row `col`
    constexpr int kTile = KC * 64, QN = (NB * RT * kTile + NT - 1) / NT, kPart = NB * RT * kTile;
    const int granules = nb * RT * kTile;
    f32x8 x[QN];
#pragma unroll
    for (int n = 0; n < QN; n++) {
      const int i = n * NT + tid, m = i / kTile * 16 + (i & 15), c = (i >> 6) % KC, qd = (i >> 4) & 3;
      const int d = KIND == kKvI8 ? (c >> 1) * 64 + qd * 16 + (c & 1) * 8 : c * 32 + qd * 8;
      if (i < granules && m < nrows) {
        const int row = row0 + m, t = row / group;
        x[n] = load_q(g.q.r0 + t, (g.h * group + row - t * group) * D + d);
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++) x[n][k] = 0.f;
      }
    }
    __syncthreads();  // the segment before has left LDS
    if constexpr (F16) {
      if (tid < NB * BR) qmax[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int n = 0; n < QN; n++) {
        const int i = n * NT + tid;
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) top = max(top, __float_as_uint(x[n][k]) & 0x7FFFFFFFu);
        if (i < granules) atomicMax(&qmax[i / kTile * 16 + (i & 15)], top);
      }
      __syncthreads();
    }
    auto q_exp = [&](int m) {  // the exponent taken out of row m
      const uint32_t top = qmax[m];
      return top == 0u || top >= 0x7F800000u ? 0 : __builtin_amdgcn_frexp_expf(__uint_as_float(top));
    };
#pragma unroll
    for (int n = 0; n < QN; n++) {
      const int i = n * NT + tid;
      if (i < granules) {
        if constexpr (F16) {
          const int e = -q_exp(i / kTile * 16 + (i & 15));
#pragma unroll
          for (int k = 0; k < 8; k++) x[n][k] = __builtin_amdgcn_ldexpf(x[n][k], e);
        }
#pragma unroll
        for (int p = 0; p < NS; p++) qf[p * kPart + i] = part_of<KIND>(x[n]);
      }
    }
    const u32x4 *wq = qf + wb * RT * kTile + lane;  // the wave's
    // the last token that row col of tile t sees
    int seen[RT];
    float scale[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
      scale[t] = F16 ? __builtin_amdgcn_ldexpf(a.scale, q_exp(wb * BR + t * 16 + col)) : a.scale;
      const int row = wrow0 + t * 16 + col;
      seen[t] = t * 16 + col < wrows ? g.q.len - g.q.nr + row / group : -1;
    }
    const int all_see = g.q.len - g.q.nr + wrow0 / group;  // every row of the block sees up to here
    f32x4 o[RT][DB];
    float mx[RT], l[RT];
    int ve = -200;  // 8 bits: the power of two that the sums are in units of (below any step's)
#pragma unroll
    for (int t = 0; t < RT; t++) {
      mx[t] = kNegInf;
      l[t] = 0.f;
#pragma unroll
      for (int i = 0; i < DB; i++) o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    __syncthreads();
    for (int it = 0; it < turns; it++) {
      const int pg = pg0 + ws + it * step;
      const uint8_t *blk = block(id);
      const u32x4 *vp = (const u32x4 *)(blk + kKvPage * D * kv_esize(KIND)) + lane;
      const bool there = valid(id);  // a page id outside the pool: a page that nobody sees
      const int len = there ? g.q.len : 0;
      if constexpr (!kAhead) load_keys(id);
      auto load_values = [&] {
#pragma unroll
        for (int i = 0; i < DB; i++)
#pragma unroll
          for (int v = 0; v < VG; v++) vf[i][v] = vp[(i * VG + v) * 64];
      };
      f32x4 ks[4], vs[4];
      auto load_steps = [&] {
#pragma unroll
        for (int kb = 0; kb < 4; kb++) {
          ks[kb] = *(const f32x4 *)(blk + kv_step_at(D, 0, kb * 16 + quad * 4));
          vs[kb] = *(const f32x4 *)(blk + kv_step_at(D, 1, kb * 16 + quad * 4));
        }
      };
      if constexpr (kAhead) {
        load_values();
        if constexpr (KIND == kKvI8) load_steps();
      }
      const bool edge = pg * kKvPage + kKvPage - 1 > all_see || !there;  // some row does not see some key of the page
      const int j0 = pg * kKvPage + quad * 4;
      // ---- scores: lane (row col, keys kb * 16 + 4 quad + i)
      f32x4 s[RT][4];
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int kb = 0; kb < 4; kb++) s[t][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; c++) {
        if constexpr (RT > 1 && (KIND == kKvI8 || D == 256)) __builtin_amdgcn_sched_barrier(0);  // (nothing ahead: registers)
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
          for (int p = NS - 1; p >= 0; p--) {
            const u32x4 b = wq[p * kPart + (t * KC + c) * 64];
#pragma unroll
            for (int kb = 0; kb < 4; kb++) {
              u32x4 k;
              if constexpr (KIND == kKvI8) {
                const u32x4 w = kf[kb][c >> 1];
                k = __builtin_bit_cast(u32x4, i8_f16((c & 1) ? u32x2{w[2], w[3]} : u32x2{w[0], w[1]}));
              } else {
                k = kf[kb][c];
              }
              s[t][kb] = mfma<KIND>(k, b, s[t][kb]);
            }
          }
      }
      if constexpr (kAhead) {
        if (it + 1 < turns) {
          if (((it + 1) & 63) == 0) ids = load_ids(it + 1);
          id = __builtin_amdgcn_readlane(ids, (it + 1) & 63);
          load_keys(id);
        }
      } else {
        load_values();
        if constexpr (KIND == kKvI8) load_steps();
        if (it + 1 < turns) {
          if (((it + 1) & 63) == 0) ids = load_ids(it + 1);
          id = __builtin_amdgcn_readlane(ids, (it + 1) & 63);
        }
      }
      float vshift = 1.f;
      if constexpr (KIND == kKvI8) {
        float top = 0.f;
#pragma unroll
        for (int kb = 0; kb < 4; kb++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            if (edge && j0 + kb * 16 + i >= len) vs[kb][i] = 0.f;  // behind the last token a step may be anything
            top = fmaxf(top, vs[kb][i]);
          }
        top = fmaxf(top, xor_lane<16>(top, lane));
        top = fmaxf(top, xor_lane<32>(top, lane));
        const int e = max(ve, top > 0.f ? __builtin_amdgcn_frexp_expf(top) : ve);
        vshift = __builtin_amdgcn_ldexpf(1.f, ve - e);
        ve = e;
#pragma unroll
        for (int kb = 0; kb < 4; kb++) {
#pragma unroll
          for (int i = 0; i < 4; i++) vs[kb][i] = __builtin_amdgcn_ldexpf(vs[kb][i], -e);
        }
      }
      f32x8 p[RT][2];
#pragma unroll
      for (int t = 0; t < RT; t++) {
        const int last = there ? seen[t] : -1;
        float top = kNegInf;
#pragma unroll
        for (int kb = 0; kb < 4; kb++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float v = s[t][kb][i];
            if constexpr (KIND == kKvI8) v *= ks[kb][i];
            if (edge) v = j0 + kb * 16 + i <= last ? v : kNegInf;
            s[t][kb][i] = v;
            top = fmaxf(top, v);
          }
        top = fmaxf(top, xor_lane<16>(top, lane));
        top = fmaxf(top, xor_lane<32>(top, lane));
        // (mx: the running maximum of the products; the scale is positive and comes in with the exponentials)
        const float m1 = fmaxf(mx[t], top), ml = (m1 == kNegInf ? 0.f : m1 * scale[t]) - kLift;
        // (most pages change no maximum; always where the branch costs registers that are not there)
        if (KIND == kKvI8 || (D == 256 && RT == 2) || __ballot(m1 != mx[t])) {
          const float alpha = m1 == kNegInf ? 0.f : __builtin_amdgcn_exp2f((mx[t] - m1) * scale[t]);
          l[t] *= alpha;
#pragma unroll
          for (int i = 0; i < DB; i++) o[t][i] *= alpha * vshift;
        }
        mx[t] = m1;
        float add = 0.f;
#pragma unroll
        for (int kb = 0; kb < 4; kb++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][kb][i], scale[t], -ml));
            add += e;
            if constexpr (KIND == kKvI8) {
              e *= vs[kb][i];
              if (edge) e = j0 + kb * 16 + i <= last ? e : 0.f;  // (a step may be NaN)
            }
            p[t][kb >> 1][(kb & 1) * 4 + i] = e;
          }
        l[t] += add;
      }
      // 16 bits: what lies behind the last token may be anything, and 0 times it too, so it is cleared. Among drafts a value
      // that is not finite must not reach the rows of earlier drafts either: it is taken out of the product, and the sums of
      // the rows that see it are made NaN (which of them, the same product of ones tells).
      bool odd = false;
      auto kept = [&](u32x4 w, int kg) {  // the keys before len (recomputed where it is used: edges are rare, registers are not)
        const int left = again(len - j0) - kg * 32;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int j = (k >> 1) * 16 + (k & 1) * 2;
          w[k] &= (j < left ? 0xFFFFu : 0u) | (j + 1 < left ? 0xFFFF0000u : 0u);
        }
        return w;
      };
      if constexpr (KIND != kKvI8) {
        if (edge && g.q.nr > 1) {
          constexpr uint32_t e = KIND == kKvBf16 ? 0x7F80u : 0x7C00u;
          uint32_t lo = 0, hi = 0;
#pragma unroll
          for (int i = 0; i < DB; i++)
#pragma unroll
            for (int kg = 0; kg < 2; kg++) {
              const u32x4 w = kept(vf[i][kg], kg);
#pragma unroll
              for (int k = 0; k < 4; k++) {
                lo = max(lo, w[k] & e);
                hi = max(hi, w[k] & e << 16);
              }
            }
          odd = __ballot(lo == e || hi == e << 16) != 0;
        }
      }
#pragma unroll
      for (int kg = 0; kg < 2; kg++) {
        __builtin_amdgcn_sched_barrier(0);  // (the groups one after the other: both at once take too many registers)
        u32x4 pf[RT][NS];
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
          for (int k = 0; k < NS; k++) pf[t][k] = part_of<KIND>(p[t][kg]);
#pragma unroll
        for (int i = 0; i < DB; i++) {
          u32x4 v;
          if constexpr (KIND == kKvI8) {
            const u32x4 w = vf[i][0];
            v = __builtin_bit_cast(u32x4, i8_f16(kg ? u32x2{w[2], w[3]} : u32x2{w[0], w[1]}));
          } else {
            v = vf[i][kg];
            if (edge) v = kept(v, kg);
            if (__builtin_expect(odd, 0)) {
              u32x4 one;
#pragma unroll
              for (int k = 0; k < 4; k++) {
                const uint32_t bad = not_finite<KIND>(v[k]);
                one[k] = bad & (kOne<KIND> | kOne<KIND> << 16);
                v[k] &= ~bad;
              }
#pragma unroll
              for (int t = 0; t < RT; t++) {
                const int last = again(seen[t] - j0) - kg * 32;
                u32x4 sees;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                  const int j = (k >> 1) * 16 + (k & 1) * 2;
                  sees[k] = (j <= last ? kOne<KIND> : 0u) | (j + 1 <= last ? kOne<KIND> << 16 : 0u);
                }
                const f32x4 n = mfma<KIND>(one, sees, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                for (int k = 0; k < 4; k++)
                  if (n[k] > 0.f) o[t][i][k] = __builtin_nanf("");
              }
            }
          }
#pragma unroll
          for (int t = 0; t < RT; t++)
#pragma unroll
            for (int k = NS - 1; k >= 0; k--) o[t][i] = mfma<KIND>(v, pf[t][k], o[t][i]);
        }
      }
    }
    if constexpr (KIND == kKvI8) {
#pragma unroll
      for (int t = 0; t < RT; t++)
#pragma unroll
        for (int i = 0; i < DB; i++)
#pragma unroll
          for (int k = 0; k < 4; k++) o[t][i][k] = __builtin_amdgcn_ldexpf(o[t][i][k], ve);
    }
    // ---- the segment's waves joined
    const int tj = again(tid);  // (what follows from it is computed here, not held through the pages)
    const int used = max(min(step, pg1 - pg0), 1);  // waves of a block that had a page; one has the zeros of none
    __syncthreads();  // every wave has read its query parts
#pragma unroll
    for (int t = 0; t < RT; t++) {
      float s = l[t];
      s += xor_lane<16>(s, lane);
      s += xor_lane<32>(s, lane);
      if (quad == 0) {
        wm[wave][t * 16 + col] = mx[t] * scale[t];
        wl[wave][t * 16 + col] = s;
      }
      if (ws < used && t * 16 + col < wrows) {
#pragma unroll
        for (int i = 0; i < DB; i++) *(f32x4 *)(js + (wave * BR + t * 16 + col) * kPitch + i * 16 + quad * 4) = o[t][i];
      }
    }
    __syncthreads();
    const int slot = dec_slot(part, me - part.first) * SLOT;  // in floats
    constexpr int ROWS = NB * BR;
    const __amdgpu_buffer_rsrc_t parts = __builtin_amdgcn_make_buffer_rsrc(a.part, (short)0, (int)(2u * W * SLOT * 4), 0x00020000);
    auto out4 = [&](int m, int d, f32x4 v) { store4<D>(a, g.q.r0, g.h, row0 + m, d, v); };
    for (int i = tj; i < nrows * (D / 4); i += NT) {
      const int m = i / (D / 4), d = i % (D / 4) * 4;
      const int w0 = m / BR, mm = m - w0 * BR;  // the waves w0, w0 + nb, .. hold the row
      float top = kNegInf, s = 0.f;
      for (int w = 0; w < used; w++) top = fmaxf(top, wm[w0 + w * nb][mm]);
      const float ms = top == kNegInf ? 0.f : top;
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      for (int w = 0; w < used; w++) {
        const float f = __builtin_amdgcn_exp2f(wm[w0 + w * nb][mm] - ms);
        s = __builtin_fmaf(wl[w0 + w * nb][mm], f, s);
        v += *(const f32x4 *)(js + ((w0 + w * nb) * BR + mm) * kPitch + d) * f;
      }
      if (part.parts > 1) {
        part_store(parts, (uint32_t)(slot + m * D + d) * 4u, v);
        if (d == 0) {
          st_cg(a.part + slot + ROWS * D + m, top);
          st_cg(a.part + slot + ROWS * D + ROWS + m, s);
        }
      } else {
        out4(m, d, v * (s == 0.f ? 0.f : 1.f / s));
      }
    }
    // ---- the group's shares joined: parts by kJoin, then their joins; or by a launch of its own, that is told which
    if (aligned && a.apart) {
      if (part.parts > 1 && chunk == 0 && tj == 0) a.joins[me] = DecJoin{part.parts, g.q.r0, g.h, row0, nrows};
    } else if (part.parts > 1) {
      // parts k0, k0 + every, .. (cnt of them) into part k0's slot, or into the output
      auto join = [&](int k0, int every, int cnt, bool final) {
        for (int i = tj; i < cnt * ROWS; i += NT) {
          const int k = i / ROWS, m = i % ROWS;
          if (m < nrows) {
            const float *sl = a.part + dec_slot(part, k0 + k * every) * SLOT + ROWS * D;
            pm[k][m] = ld_cg(sl + m);
            pl[k][m] = ld_cg(sl + ROWS + m);
          }
        }
        __syncthreads();
        if (tj < nrows) {  // each part's factor in place of its maximum, the row's maximum and sum
          float top = kNegInf, sum = 0.f;
          for (int k = 0; k < cnt; k++) top = fmaxf(top, pm[k][tj]);
          const float ms = top == kNegInf ? 0.f : top;
          for (int k = 0; k < cnt; k++) {
            const float f = __builtin_amdgcn_exp2f(pm[k][tj] - ms);
            pm[k][tj] = f;
            sum = __builtin_fmaf(pl[k][tj], f, sum);
          }
          if (!final) {
            st_cg(a.part + dec_slot(part, k0) * SLOT + ROWS * D + tj, top);
            st_cg(a.part + dec_slot(part, k0) * SLOT + ROWS * D + ROWS + tj, sum);
          }
          pl[0][tj] = sum == 0.f ? 0.f : 1.f / sum;
        }
        __syncthreads();
        // four dims of a row at a time, kJoin parts' requests in flight and the next ones behind them
        const int items = nrows * (D / 4);
        auto request = [&](f32x4 *in, int i, int r) {
          const int m = i / (D / 4), d = i % (D / 4) * 4;
#pragma unroll
          for (int k = 0; k < kJoin; k++)
            if (r + k < cnt) in[k] = part_load(parts, (uint32_t)(dec_slot(part, k0 + (r + k) * every) * SLOT + m * D + d) * 4u);
        };
        f32x4 in[kJoin] = {}, next[kJoin] = {}, v = {0.f, 0.f, 0.f, 0.f};
        int i = tj, r = 0;
        if (i < items) request(in, i, 0);
        while (i < items) {
          const bool done = r + kJoin >= cnt;  // the item's last round
          const int i1 = done ? i + NT : i, r1 = done ? 0 : r + kJoin;
          if (i1 < items) request(next, i1, r1);
          const int m = i / (D / 4), d = i % (D / 4) * 4;
#pragma unroll
          for (int k = 0; k < kJoin; k++)
            if (r + k < cnt) v += in[k] * pm[r + k][m];
          if (done) {
            if (final) out4(m, d, v * pl[0][m]);
            else part_store(parts, (uint32_t)(dec_slot(part, k0) * SLOT + m * D + d) * 4u, v);
            v = f32x4{0.f, 0.f, 0.f, 0.f};
          }
#pragma unroll
          for (int k = 0; k < kJoin; k++) in[k] = next[k];
          i = i1;
          r = r1;
        }
      };
      auto last_of = [&](uint32_t *c, int n) {  // every wave's stores have arrived; true in the n-th workgroup to come here
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (tj == 0) {
          flag = atomicAdd(c, 1u) == (uint32_t)n - 1u;
          if (flag) st_cg(c, 0u);
        }
        __syncthreads();
        return flag != 0;
      };
      const int k = me - part.first, k0 = k / kJoin * kJoin, cnt = min(part.parts - k0, kJoin);
      const bool one = part.parts <= kJoin;
      if (cnt == 1 || last_of(a.cnt + dec_slot(part, k0), cnt)) {
        if (cnt > 1) join(k0, 1, cnt, one);
        if (!one) {
          const int joins = (part.parts + kJoin - 1) / kJoin;  // at most kJoins
          if (last_of(a.cnt + 2 * W + part.first, joins)) join(0, kJoin, joins, true);
        }
      }
    }
    if (aligned || g.u0 + hi == u_hi) return;
    // ---- the next group
    g.u0 += size;
    u = g.u0;
    if (++g.rb == g.d.blocks) {
      g.rb = 0;
      if (++g.h == a.H) {
        g.h = 0;
        do {
          if (++g.b >= a.s.n) return;  // (not reached: u < total, so a later sequence has rows)
          g.q = kv_seq(a.s, g.b);
          g.d = dec_seq(g.q, group, BR, NB);
        } while (!g.d.blocks);
      }
    }
  }
}

// The parts of the groups that the decode kernel names (rows of several drafts: a part is up to 64 rows, and one workgroup reads
// 40 GB/s of them). Workgroup (the group's first one, 16 rows of it): the rows' factors in LDS, then four dims a thread, kJoin
// parts' loads in flight.
constexpr int kJoinRows = 16;
template <int D>
__global__ __launch_bounds__(256) void attn_join(DecArgs a) {
  constexpr int ROWS = kDecRows, SLOT = dec_slot_floats(D);
  __shared__ float f[kJoin * kJoins][kJoinRows], inv[kJoinRows];
  const DecJoin j = a.joins[blockIdx.x];
  const int m0 = blockIdx.y * kJoinRows, rows = min(j.nrows - m0, kJoinRows), tid = threadIdx.x;
  if (j.parts == 0 || rows <= 0) return;
  const float *base = a.part + (int64_t)blockIdx.x * 2 * SLOT;  // part k's slot: 2 k slots on
  float *sums = inv;
  for (int i = tid; i < j.parts * kJoinRows; i += 256) {
    const int k = i / kJoinRows, m = i % kJoinRows;
    if (m < rows) f[k][m] = base[(int64_t)k * 2 * SLOT + ROWS * D + m0 + m];
  }
  __syncthreads();
  // 16 threads a row
  const int row = tid >> 4, part = tid & 15;
  if (row < rows) {
    float top = kNegInf, sum = 0.f;
    for (int k = part; k < j.parts; k += 16) top = fmaxf(top, f[k][row]);
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float ms = top == kNegInf ? 0.f : top;
    for (int k = part; k < j.parts; k += 16) {
      const float e = __builtin_amdgcn_exp2f(f[k][row] - ms);
      f[k][row] = e;
      sum = __builtin_fmaf(base[(int64_t)k * 2 * SLOT + ROWS * D + ROWS + m0 + row], e, sum);
    }
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) sum += __shfl_xor(sum, x);
    if (part == 0) sums[row] = sum == 0.f ? 0.f : 1.f / sum;
  }
  __syncthreads();
  for (int i = tid; i < rows * (D / 4); i += 256) {
    const int m = i / (D / 4), d = i % (D / 4) * 4;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int r = 0; r < j.parts; r += kJoin) {
      f32x4 in[kJoin];
#pragma unroll
      for (int k = 0; k < kJoin; k++)
        if (r + k < j.parts) in[k] = *(const f32x4 *)(base + (int64_t)(r + k) * 2 * SLOT + (m0 + m) * D + d);
#pragma unroll
      for (int k = 0; k < kJoin; k++)
        if (r + k < j.parts) v += in[k] * f[r + k][m];
    }
    store4<D>(a, j.r0, j.h, j.row0 + m0 + m, d, v * inv[m]);
  }
}

template <int KIND, int D, int RT>
constexpr int lds_bytes() {
  constexpr int q = Num<KIND>::NS * RT * RT * (D / 32) * 1024, j = NW * 16 * RT * (D + 4) * 4, p = 2 * kJoins * 16 * RT * RT * 4;
  return q > j ? (q > p ? q : p) : (j > p ? j : p);
}

template <typename F>
void each(F &&f) {  // every instance
  auto dims = [&](auto kind) {
    auto rows = [&](auto dim) {
      f(kind, dim, std::integral_constant<int, 1>());
      f(kind, dim, std::integral_constant<int, 2>());
    };
    rows(std::integral_constant<int, 64>());
    rows(std::integral_constant<int, 128>());
    rows(std::integral_constant<int, 256>());
  };
  dims(std::integral_constant<int, kKvBf16>());
  dims(std::integral_constant<int, kKvF16>());
  dims(std::integral_constant<int, kKvI8>());
}

}  // namespace

int compute_units() {
  static const int n = [] {
    int dev = 0, cus = 0;
    IJ_HIP(hipGetDevice(&dev));
    IJ_HIP(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev));
    return cus;
  }();
  return n;
}
int decode_grid(int D) { return std::min(compute_units() * per_cu(D), kJoin * kJoins); }  // (256 CUs on an MI355X)

void launch_attn_decode(const DecArgs &args, hipStream_t s) {
  DecArgs a = args;
  // 16 query rows a block while a token's rows fill no more than that, else 32: each block reads the pages once
  const int rt = a.Hq / a.H <= 16 && a.s.R <= a.s.n ? 1 : 2;
  // many rows that may lie in several chunks (of at least two pages a wave): their joins take a launch of their own
  a.apart = rt == 2 && (int64_t)a.s.ldt * 2 > 2 * NW;
  each([&](auto kind, auto dim, auto tiles) {
    constexpr int K = decltype(kind)::value, D = decltype(dim)::value, RT = decltype(tiles)::value;
    if (a.kind == K && a.D == D && rt == RT)
      hipLaunchKernelGGL((attn_decode<K, D, RT>), dim3(a.W), dim3(NT), (lds_bytes<K, D, RT>()), s, a);
  });
  IJ_HIP(hipGetLastError());
  if (!a.apart) return;
  const dim3 grid(a.W, kDecRows / kJoinRows);
  if (a.D == 64) hipLaunchKernelGGL(attn_join<64>, grid, dim3(256), 0, s, a);
  else if (a.D == 128) hipLaunchKernelGGL(attn_join<128>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(attn_join<256>, grid, dim3(256), 0, s, a);
  IJ_HIP(hipGetLastError());
}

void init_decode_attrs() {
  each([&](auto kind, auto dim, auto tiles) {
    IJ_HIP(hipFuncSetAttribute(
        (const void *)attn_decode<decltype(kind)::value, decltype(dim)::value, decltype(tiles)::value>,
        hipFuncAttributeMaxDynamicSharedMemorySize,
        lds_bytes<decltype(kind)::value, decltype(dim)::value, decltype(tiles)::value>()));
  });
}

}  // namespace ijah
