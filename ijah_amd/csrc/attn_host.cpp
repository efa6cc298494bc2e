// Attention entry points (include/ijah_attn.h): argument checks, the cache handle, launches.
#include <cmath>
#include <functional>
#include <limits>

#include "../../include/ijah_attn.h"
#include "attn.h"
#include "common.h"

using namespace ijah;

static const bool g_hooked = (on_device_setup(init_attn_attrs), true);

struct ne_kv {
  ne_kv_desc d;
  int kind = 0, W = 0;
  uint64_t layer_bytes = 0;
  uint8_t *base = nullptr;
  float *part = nullptr;    // decode: the partial slots of W workgroups
  uint32_t *cnt = nullptr;  // decode: 3 W counters, zero between launches
  DecJoin *joins = nullptr; // decode: [W]
  ~ne_kv() {
    for (void *p : {(void *)base, (void *)part, (void *)cnt, (void *)joins})
      if (p) (void)hipFree(p);
  }
};

namespace {

constexpr int kMaxRows = 1 << 22;  // (and 512 threads for each stay below 2^32)

int row_type(int dtype) {
  IJ_CHECK(dtype == NE_F32 || dtype == NE_BF16 || dtype == NE_F16, "rows of type %d (F32, BF16 or F16)", dtype);
  return dtype == NE_F32 ? kRowF32 : dtype == NE_BF16 ? kRowBf16 : kRowF16;
}
void check_dim(int dim) { IJ_CHECK(dim == 64 || dim == 128 || dim == 256, "dim %d (64, 128 or 256)", dim); }
void check_scale(float s) {
  IJ_CHECK(s > 0.f && s < 1e38f, "scale %g (a positive number)", (double)s);
}
constexpr float kLog2e = 1.4426950408889634f;

// R rows of `cols` elements in b from off on, ld elements apart (0: packed); written: not a pack tensor
RowMat rows_of(const ne_buf *b, uint64_t off, int ld, int R, int64_t cols, int type, const char *what, bool written) {
  const uint64_t e = type == kRowF32 ? 4 : 2;
  IJ_CHECK(b, "null %s", what);
  IJ_CHECK(ld == 0 || ld >= cols, "%s: row stride %d below %lld", what, ld, (long long)cols);
  RowMat m;
  m.ld = ld ? ld : cols;
  IJ_CHECK(off % 16 == 0 && (uint64_t)m.ld * e % 16 == 0, "%s: rows must start on 16-byte boundaries", what);
  const uint64_t need = ((uint64_t)(R - 1) * (uint64_t)m.ld + (uint64_t)cols) * e;
  IJ_CHECK(off <= b->size && need <= b->size - off, "%s buffer too small for %d rows of %lld, stride %lld", what, R,
           (long long)cols, (long long)m.ld);
  IJ_CHECK(!written || !b->readonly, "%s is a pack tensor (read-only)", what);
  m.p = (char *)ne_dev(b) + off;
  IJ_CHECK((uintptr_t)m.p % 16 == 0, "%s: rows must start on 16-byte boundaries", what);
  return m;
}
const int *ints_of(const ne_buf *b, uint64_t count, const char *what) {
  IJ_CHECK(b, "null %s", what);
  IJ_CHECK(b->size >= count * 4, "%s buffer too small for %llu i32", what, (unsigned long long)count);
  return (const int *)ne_dev(b);
}
void check_layer(const ne_kv *kv, int layer) {
  IJ_CHECK(kv, "null cache");
  IJ_CHECK(layer >= 0 && layer < kv->d.layers, "layer %d (0..%d)", layer, kv->d.layers - 1);
}
KvSeqs seqs_of(const ne_kv *kv, const ne_kv_seqs *s, int R) {
  IJ_CHECK(s, "null sequences");
  IJ_CHECK(s->n >= 1 && s->n <= kMaxRows, "sequences %d (1..%d)", s->n, kMaxRows);
  IJ_CHECK(s->ldt >= 1 && s->ldt <= std::numeric_limits<int>::max() / kKvPage, "table row length %d (1..%d)", s->ldt,
           std::numeric_limits<int>::max() / kKvPage);
  IJ_CHECK(R >= 1 && R <= kMaxRows, "rows %d (1..%d)", R, kMaxRows);
  IJ_CHECK(s->rows || R == s->n, "%d rows of %d sequences: without `rows` each has one", R, s->n);
  KvSeqs a;
  a.n = s->n;
  a.ldt = s->ldt;
  a.pages = kv->d.pages;
  a.R = R;
  a.table = ints_of(s->table, (uint64_t)s->n * s->ldt, "table");
  a.lens = ints_of(s->lens, s->n, "lens");
  a.rows = s->rows ? ints_of(s->rows, (uint64_t)s->n + 1, "rows") : nullptr;
  return a;
}
KvArgs kv_args(const ne_kv *kv, int layer, const ne_kv_seqs *s, int R, const ne_buf *k, uint64_t k_off, int ldk,
               const ne_buf *v, uint64_t v_off, int ldv, int dtype, bool written) {
  check_layer(kv, layer);
  KvArgs a;
  a.s = seqs_of(kv, s, R);
  a.kind = kv->kind;
  a.D = kv->d.dim;
  a.H = kv->d.heads;
  a.type = row_type(dtype);
  const int64_t cols = (int64_t)a.H * a.D;
  a.k = rows_of(k, k_off, ldk, R, cols, a.type, "k", written);
  a.v = rows_of(v, v_off, ldv, R, cols, a.type, "v", written);
  a.base = kv->base + (uint64_t)layer * kv->layer_bytes;
  return a;
}
// whether two row matrices share bytes (each taken whole, gaps between rows included)
bool overlap(const RowMat &a, int Ra, int64_t ca, const RowMat &b, int Rb, int64_t cb, uint64_t e) {
  const uintptr_t a0 = (uintptr_t)a.p, a1 = a0 + ((uint64_t)(Ra - 1) * a.ld + ca) * e;
  const uintptr_t b0 = (uintptr_t)b.p, b1 = b0 + ((uint64_t)(Rb - 1) * b.ld + cb) * e;
  return a0 < b1 && b0 < a1;
}
template <typename T>
void alloc(T *&p, uint64_t bytes) {
  void *m = nullptr;
  IJ_HIP(hipMalloc(&m, bytes));
  p = (T *)m;
  IJ_HIP(hipMemset(m, 0, bytes));
}
// Runs `work` on the library stream; with gpu_ms, waits and reports its GPU time.
void timed(double *gpu_ms, const std::function<void(hipStream_t)> &work) {
  const hipStream_t s = stream();
  if (!gpu_ms) {
    work(s);
    return;
  }
  struct Event {
    hipEvent_t e = nullptr;
    ~Event() {
      if (e) (void)hipEventDestroy(e);
    }
  } e0, e1;
  IJ_HIP(hipEventCreate(&e0.e));
  IJ_HIP(hipEventCreate(&e1.e));
  IJ_HIP(hipEventRecord(e0.e, s));
  work(s);
  IJ_HIP(hipEventRecord(e1.e, s));
  IJ_HIP(hipEventSynchronize(e1.e));
  float ms = 0.f;
  IJ_HIP(hipEventElapsedTime(&ms, e0.e, e1.e));
  *gpu_ms = ms;
}

}  // namespace

extern "C" {

NE_API ne_kv *ne_kv_create(const ne_kv_desc *d) {
  ne_kv *h = nullptr;
  c_call([&] {
    IJ_CHECK(d, "null desc");
    IJ_CHECK(d->layers >= 1 && d->pages >= 1 && d->heads >= 1, "cache of %d layers, %d pages, %d heads", d->layers,
             d->pages, d->heads);
    check_dim(d->dim);
    IJ_CHECK(d->dtype == NE_BF16 || d->dtype == NE_F16 || d->dtype == NE_I8, "cache of type %d (BF16, F16 or I8)",
             d->dtype);
    IJ_CHECK(d->heads <= 65535 && d->pages <= std::numeric_limits<int>::max() / kKvPage && d->layers <= 65535,
             "cache of %d layers, %d pages, %d heads", d->layers, d->pages, d->heads);
    ensure_device();
    stream();
    auto kv = std::make_unique<ne_kv>();
    kv->d = *d;
    kv->kind = d->dtype == NE_BF16 ? kKvBf16 : d->dtype == NE_F16 ? kKvF16 : kKvI8;
    kv->W = decode_grid(d->dim);
    const uint64_t per_page = (uint64_t)d->heads * kv_block_bytes(kv->kind, d->dim);  // < 2^33
    IJ_CHECK(per_page <= (1ull << 46) / (uint64_t)d->pages / (uint64_t)d->layers, "cache of %d layers, %d pages, %d heads",
             d->layers, d->pages, d->heads);
    kv->layer_bytes = per_page * (uint64_t)d->pages;
    alloc(kv->base, kv->layer_bytes * (uint64_t)d->layers);
    alloc(kv->part, (uint64_t)2 * kv->W * dec_slot_floats(d->dim) * 4);
    alloc(kv->cnt, (uint64_t)3 * kv->W * 4);
    alloc(kv->joins, (uint64_t)kv->W * sizeof(DecJoin));
    IJ_HIP(hipDeviceSynchronize());
    h = kv.release();
  });
  return h;
}
NE_API void ne_kv_free(ne_kv *kv) {
  if (!kv) return;
  c_call([&] { IJ_HIP(hipStreamSynchronize(stream())); });
  delete kv;
}
NE_API int ne_kv_info(const ne_kv *kv, ne_kv_desc *d, uint64_t *bytes) {
  return c_call([&] {
    IJ_CHECK(kv, "null cache");
    if (d) *d = kv->d;
    if (bytes) *bytes = kv->layer_bytes * (uint64_t)kv->d.layers;
  });
}

NE_API int ne_kv_write(ne_kv *kv, int layer, const ne_kv_seqs *s, int R, const ne_buf *k, uint64_t k_off, int ldk,
                       const ne_buf *v, uint64_t v_off, int ldv, int dtype, double *gpu_ms) {
  return c_call([&] {
    const KvArgs a = kv_args(kv, layer, s, R, k, k_off, ldk, v, v_off, ldv, dtype, false);
    timed(gpu_ms, [&](hipStream_t st) { launch_kv_write(a, st); });
  });
}
NE_API int ne_kv_read(const ne_kv *kv, int layer, const ne_kv_seqs *s, int R, ne_buf *k, uint64_t k_off, int ldk, ne_buf *v,
                      uint64_t v_off, int ldv, int dtype, double *gpu_ms) {
  return c_call([&] {
    const KvArgs a = kv_args(kv, layer, s, R, k, k_off, ldk, v, v_off, ldv, dtype, true);
    timed(gpu_ms, [&](hipStream_t st) { launch_kv_read(a, st); });
  });
}

NE_API int ne_attn_decode(ne_kv *kv, int layer, const ne_kv_seqs *s, int R, int heads, const ne_buf *q, uint64_t q_off,
                          int ldq, ne_buf *out, uint64_t out_off, int ldo, int dtype, float scale, double *gpu_ms) {
  return c_call([&] {
    check_layer(kv, layer);
    IJ_CHECK(heads >= 1 && heads % kv->d.heads == 0, "%d query heads over %d key heads", heads, kv->d.heads);
    check_scale(scale);
    DecArgs a;
    a.s = seqs_of(kv, s, R);
    IJ_CHECK(dec_max_units(s->n, s->ldt, R, heads / kv->d.heads, kv->d.heads, 16) < (1ll << 31) &&
                 (int64_t)R * heads < (1ll << 31),
             "%d rows of %d heads over %d tables of %d pages: too much for one call", R, heads, s->n, s->ldt);
    a.kind = kv->kind;
    a.D = kv->d.dim;
    a.H = kv->d.heads;
    a.Hq = heads;
    a.type = row_type(dtype);
    const int64_t cols = (int64_t)heads * a.D;
    a.q = rows_of(q, q_off, ldq, R, cols, a.type, "q", false);
    a.out = rows_of(out, out_off, ldo, R, cols, a.type, "out", true);
    IJ_CHECK((a.q.p == a.out.p && a.q.ld == a.out.ld) ||
                 !overlap(a.q, R, cols, a.out, R, cols, a.type == kRowF32 ? 4 : 2),
             "out overlaps q without being q's own rows");
    a.base = kv->base + (uint64_t)layer * kv->layer_bytes;
    a.scale = scale * kLog2e;
    a.part = kv->part;
    a.cnt = kv->cnt;
    a.joins = kv->joins;
    a.apart = 0;
    a.W = kv->W;
    timed(gpu_ms, [&](hipStream_t st) { launch_attn_decode(a, st); });
  });
}

NE_API int ne_attn_prompt(const ne_attn_prompt_desc *d, double *gpu_ms) {
  return c_call([&] {
    IJ_CHECK(d, "null desc");
    check_dim(d->dim);
    IJ_CHECK(d->kv_heads >= 1 && d->heads >= 1 && d->heads % d->kv_heads == 0, "%d query heads over %d key heads", d->heads,
             d->kv_heads);
    IJ_CHECK(d->n >= 1 && d->n <= kMaxRows, "sequences %d (1..%d)", d->n, kMaxRows);
    IJ_CHECK(d->Rq >= 1 && d->Rq <= kMaxRows && d->Rk >= 1 && d->Rk <= kMaxRows, "rows %d and %d (1..%d)", d->Rq, d->Rk,
             kMaxRows);
    IJ_CHECK(d->k_rows || d->Rk == d->Rq, "%d key rows for %d query rows: without k_rows they are the same", d->Rk, d->Rq);
    IJ_CHECK(((int64_t)d->Rq / 128 + d->n + 1) * d->heads < (1 << 23), "%d rows of %d sequences and %d heads", d->Rq, d->n,
             d->heads);
    check_scale(d->scale);
    ensure_device();
    PromptArgs a;
    a.n = d->n;
    a.Hq = d->heads;
    a.H = d->kv_heads;
    a.D = d->dim;
    a.type = row_type(d->dtype);
    a.Rq = d->Rq;
    a.Rk = d->Rk;
    const int64_t qc = (int64_t)a.Hq * a.D, kc = (int64_t)a.H * a.D;
    a.q = rows_of(d->q, d->q_off, d->ldq, a.Rq, qc, a.type, "q", false);
    a.k = rows_of(d->k, d->k_off, d->ldk, a.Rk, kc, a.type, "k", false);
    a.v = rows_of(d->v, d->v_off, d->ldv, a.Rk, kc, a.type, "v", false);
    a.out = rows_of(d->out, d->out_off, d->ldo, a.Rq, qc, a.type, "out", true);
    const uint64_t e = a.type == kRowF32 ? 4 : 2;
    IJ_CHECK(!overlap(a.q, a.Rq, qc, a.out, a.Rq, qc, e) && !overlap(a.k, a.Rk, kc, a.out, a.Rq, qc, e) &&
                 !overlap(a.v, a.Rk, kc, a.out, a.Rq, qc, e),
             "out overlaps q, k or v");
    IJ_CHECK(a.k.ld < (1 << 22) && a.v.ld < (1 << 22), "row strides %lld and %lld of k and v (below 2^22)",
             (long long)a.k.ld, (long long)a.v.ld);  // (a tile's rows are addressed in 31 bits)
    a.q_rows = ints_of(d->q_rows, (uint64_t)a.n + 1, "q_rows");
    a.k_rows = d->k_rows ? ints_of(d->k_rows, (uint64_t)a.n + 1, "k_rows") : a.q_rows;
    a.cus = compute_units();
    a.scale = d->scale * kLog2e;
    timed(gpu_ms, [&](hipStream_t st) { launch_attn_prompt(a, st); });
  });
}

}  // extern "C"
