// The paged key-value cache and the attention kernels: layouts, the division of work (plain C++, so that a host program
// can check it), and the launch wrappers.
#pragma once
#include <cstdint>

typedef struct ihipStream_t *hipStream_t;

#ifdef __HIPCC__
#define IJ_HD __host__ __device__ inline __attribute__((always_inline))
#else
#define IJ_HD inline
#endif

namespace ijah {

// ------------------------------------------------------------------------------------------------ a page
// Keys and values of one page and head are one block: keys, values, then (8 bits) the steps of the 64 keys and of the 64
// values, f32. Inside, 16-byte granules in the order in which the lanes of v_mfma_f32_16x16x32 take them, so that every
// load of the decode kernel is 64 lanes x 16 consecutive bytes:
//   keys    A operand, 16 keys x 32 dims: granule (key block kb, dim chunk dc, lane); lane = quad * 16 + key % 16 holds 8
//           dims 32 dc + 8 quad + ... (8 bits: 16 dims 64 dc + 16 quad + ..., two products' worth)
//   values  A operand of the transposed product, 16 dims x 32 keys: granule (dim block db, key group kg, lane); lane =
//           quad * 16 + dim % 16 holds the 8 keys 32 kg + 4 quad + {0..3} and 32 kg + 16 + 4 quad + {0..3}: those whose
//           scores the product of the keys leaves in this quad's lanes, so the softmax weights need no exchange between
//           lanes (8 bits: both key groups of a page in one granule)
// A single new token then touches 16 bytes x dim/8 of the keys and 2 bytes in each of dim granules, 16 neighbours at a
// time, of the values.
constexpr int kKvPage = 64;
enum { kKvBf16 = 0, kKvF16 = 1, kKvI8 = 2 };  // how the cache holds values

IJ_HD constexpr int kv_esize(int kind) { return kind == kKvI8 ? 1 : 2; }
IJ_HD constexpr int kv_block_bytes(int kind, int D) {
  return 2 * kKvPage * D * kv_esize(kind) + (kind == kKvI8 ? 2 * kKvPage * 4 : 0);
}
// byte offsets inside the block of key j's / value j's dim d, and of the steps
IJ_HD constexpr int kv_key_at(int kind, int D, int j, int d) {
  return kind == kKvI8 ? (((j >> 4) * (D >> 6) + (d >> 6)) * 64 + ((d >> 4) & 3) * 16 + (j & 15)) * 16 + (d & 15)
                       : (((j >> 4) * (D >> 5) + (d >> 5)) * 64 + ((d >> 3) & 3) * 16 + (j & 15)) * 16 + (d & 7) * 2;
}
// of the 32 keys of a group, key jj's place in its granule, and the granule's quad
IJ_HD constexpr int kv_pos(int jj) { return ((jj >> 4) & 1) * 4 + (jj & 3); }
IJ_HD constexpr int kv_quad(int jj) { return (jj >> 2) & 3; }
IJ_HD constexpr int kv_value_at(int kind, int D, int j, int d) {
  return kKvPage * D * kv_esize(kind) +
         (kind == kKvI8
              ? ((d >> 4) * 64 + kv_quad(j) * 16 + (d & 15)) * 16 + (j >> 5) * 8 + kv_pos(j & 31)
              : (((d >> 4) * 2 + (j >> 5)) * 64 + kv_quad(j) * 16 + (d & 15)) * 16 + kv_pos(j & 31) * 2);
}
IJ_HD constexpr int kv_step_at(int D, int value, int j) { return 2 * kKvPage * D + (value * kKvPage + j) * 4; }

// ------------------------------------------------------------------------------------------------ sequences
struct KvSeqs {
  int n, ldt, pages, R;  // pages: of the handle; R: rows of the call
  const int *table, *lens, *rows;
};
struct KvSeq {  // sequence b of the batch, clamped
  int len, r0, nr;  // tokens; first row and rows of the call
};
IJ_HD int kv_clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
IJ_HD KvSeq kv_seq(const KvSeqs &s, int b) {
  KvSeq q;
  q.len = kv_clamp(s.lens[b], 0, s.ldt * kKvPage);
  if (s.rows) {
    q.r0 = kv_clamp(s.rows[b], 0, s.R);
    q.nr = kv_clamp(s.rows[b + 1], q.r0, s.R) - q.r0;
  } else {
    q.r0 = b < s.R ? b : s.R;
    q.nr = b < s.R ? 1 : 0;
  }
  return q;
}
// Pieces of a write or read: the pages that the rows of sequence b lie in; a sequence with rows has at least one (its rows
// before token 0 are the first piece's). The grid is sized for kv_max_pieces.
IJ_HD int kv_pieces(const KvSeq &q) {
  if (!q.nr) return 0;
  const int p0 = q.len - q.nr > 0 ? q.len - q.nr : 0;
  return q.len ? (q.len - 1) / kKvPage - p0 / kKvPage + 1 : 1;
}
// rows r of one sequence lie in at most r / 64 + 2 pages, and in at most r
IJ_HD int64_t kv_max_pieces(int n, int R, bool rows) {
  if (!rows) return n < R ? n : R;
  const int64_t a = (int64_t)R / kKvPage + 2 * (int64_t)n;
  return a < R ? a : R;
}

// ------------------------------------------------------------------------------------------------ decode's work
// The batch's work in units of a page for one wave: of one page, one key head and one or two blocks of query rows (two: two
// units, the workgroup's waves split between them, so that their reads of a page meet in the caches), in the order (sequence,
// key head, blocks, page). A (sequence, head, blocks) is a group; a sequence with rows has at least one page (an empty one
// writes its zeros). The W workgroups take consecutive shares, in one of two forms:
//   - aligned: each group is cut into chunks of C units, a workgroup takes one chunk;
//   - else equal shares of ceil(units / W), whatever the lengths: a workgroup may end one group and begin others.
// A group that lies in several shares is joined from one partial each: workgroup w's first segment is in slot 2w, one that
// begins inside its share in 2w + 1. Parts are joined kJoin at a time by the last of them to finish, into the first one's slot
// (whose number names the counter), and these by the last of their joins (at most one group that is continued begins in a
// share, so its first workgroup names that counter): one workgroup reading all of a long sequence's parts would take longer
// than its pages do.
struct DecSeq {
  int pages, nb, blocks;  // pages (at least one); row blocks of a group (1 or 2); groups per key head
};
IJ_HD DecSeq dec_seq(const KvSeq &q, int group, int block_rows, int most_nb) {
  DecSeq d;
  const int rows = q.nr * group;
  d.pages = q.len > 0 ? (q.len + kKvPage - 1) / kKvPage : 1;
  d.nb = rows > block_rows ? most_nb : 1;
  d.blocks = (rows + block_rows * d.nb - 1) / (block_rows * d.nb);
  return d;
}
IJ_HD int dec_group(const DecSeq &d) { return d.pages * d.nb; }                    // units of a group
IJ_HD int dec_chunks(const DecSeq &d, int C) { return (dec_group(d) + C - 1) / C; }  // its chunks
IJ_HD int dec_units(const DecSeq &d, int H) { return dec_group(d) * d.blocks * H; }
// a segment's pages: those whose first unit lies in it (the last share of a group may have none)
IJ_HD int dec_page(const DecSeq &d, int unit, int real_pages) {
  const int p = (unit + d.nb - 1) / d.nb;
  return p < real_pages ? p : real_pages;
}
// the most units that a batch can have: the host refuses batches where this passes 31 bits
IJ_HD int64_t dec_max_units(int n, int ldt, int R, int group, int H, int block_rows) {
  return ((int64_t)R * group / block_rows + n) * H * 2 * ((int64_t)ldt + 1);
}
constexpr int kJoin = 16, kJoins = 32;  // parts of a join, joins of a join of joins: W <= kJoin kJoins
struct DecPart {
  int first, parts, odd;  // the group's first workgroup, how many it has, whether the first one's slot is its second
};
IJ_HD DecPart dec_part_chunk(int chunk, int chunks, int w) { return DecPart{w - chunk, chunks, 0}; }
// the group of units [g0, g1) in shares
IJ_HD DecPart dec_part_share(int g0, int g1, int share) {
  DecPart p;
  p.first = g0 / share;
  p.parts = (g1 - 1) / share - p.first + 1;
  p.odd = g0 != p.first * share ? 1 : 0;
  return p;
}
IJ_HD int dec_slot(const DecPart &p, int k) { return 2 * (p.first + k) + (k == 0 ? p.odd : 0); }  // part k's slot

// ------------------------------------------------------------------------------------------------ launches
enum { kRowF32 = 0, kRowBf16 = 1, kRowF16 = 2 };  // a row matrix's type
struct RowMat {
  const void *p;
  int64_t ld;  // elements between rows
};
struct KvArgs {
  uint8_t *base;   // the layer's pages
  int kind, D, H;  // H: key heads
  KvSeqs s;
  RowMat k, v;     // read: written to
  int type;
};
struct DecJoin {  // a group whose parts a launch of its own joins (parts 0: none), by its first workgroup
  int parts, r0, h, row0, nrows;
};
struct DecArgs {
  const uint8_t *base;
  int kind, D, H, Hq;
  KvSeqs s;
  RowMat q, out;
  int type;
  float scale;     // times log2 e
  float *part;     // [2 W] slots of dec_slot_floats
  uint32_t *cnt;   // [3 W], zero between launches: by slot of a join's first part, then by first workgroup of a group
  DecJoin *joins;  // [W]
  int apart;       // the joins of chunks take a launch of their own
  int W;
};
constexpr int kDecRows = 64;  // query rows of a group at most (the partial slots' size)
IJ_HD constexpr int dec_slot_floats(int D) { return kDecRows * (D + 2); }
struct PromptArgs {
  int n, Hq, H, D, type, Rq, Rk;
  RowMat q, k, v, out;
  const int *q_rows, *k_rows;
  int cus;         // compute units of the device
  float scale;     // times log2 e
};
void launch_kv_write(const KvArgs &a, hipStream_t s);
void launch_kv_read(const KvArgs &a, hipStream_t s);
int compute_units();
int decode_grid(int D);  // workgroups of the decode kernel: what the chip runs at once
void launch_attn_decode(const DecArgs &a, hipStream_t s);
void launch_attn_prompt(const PromptArgs &a, hipStream_t s);
void init_attn_attrs();  // raises the kernels' dynamic LDS limits: before any launch and outside a capture
}  // namespace ijah
