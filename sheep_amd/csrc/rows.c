// Several rows a sequence over a paged cache, and that cache's upkeep
// (sml-serve.h): argument checks and launches. The checks come before the
// device is touched, so they refuse alike on a machine without one.
#include "serve.h"

#include <math.h>
#include <stdio.h>
#include <string.h>

int sml_hip_paged_append_axes(const sml_hip_pages * pg, float * qkv, size_t qkv_stride, int n_rows, const int32_t * seq,
                              const int32_t * slot, const int32_t * pos, int n_axis, const uint8_t * axis,
                              const float * cos_t, const float * sin_t, int n_rope, int n_head, float * q_out,
                              void * stream) {
    HX_ENTRY(-1);
    sml_kaxes a;
    memset(&a, 0, sizeof a);
    sv_check_pages(pg, &a.pg);
    if (n_rows < 0 || n_rows > 1 << 22 || n_head < 1 || n_head > 65536) hx_failf("append: %d rows of %d heads", n_rows, n_head);
    if (n_axis < 1 || n_axis > AX_MOST) hx_failf("append: %d axes (1 to %d)", n_axis, AX_MOST);
    const size_t width = ((size_t) n_head + 2 * (size_t) pg->n_kv) * pg->hd;
    if (!qkv || !slot || !pos || !axis || !cos_t || !sin_t || n_rope < 1)
        hx_failf("append: missing rows, slots, positions, axes or rotation tables");
    if (qkv_stride && qkv_stride < width) hx_failf("append: rows of %zu floats %zu apart", width, qkv_stride);
    sv_on_device();
    if (n_rows) {
        a.qkv = qkv; a.stride = qkv_stride ? qkv_stride : width; a.seq = seq; a.slot = slot; a.pos = pos;
        a.cos_t = cos_t; a.sin_t = sin_t; a.q_out = q_out;
        a.n_rows = n_rows; a.n_rope = n_rope; a.n_head = n_head; a.n_axis = n_axis;
        memcpy(a.axis, axis, (size_t) pg->hd / 2);
        char name[40];
        sv_name(name, sizeof name, "sml_rw_append", pg->hd, pg->type);
        const int items = (n_head + pg->n_kv) * (pg->hd / 8) + pg->n_kv * (pg->hd / 4);
        hx_launch(name, (unsigned) n_rows, (unsigned) ceil_div(items, 256), 256, 0, (hipStream_t) stream, &a);
    }
    HX_LEAVE();
    return 0;
}

size_t sml_hip_paged_rows_floats(int n_seq, int n_row, int n_kv, int n_head, int hd, int max_len) {
    if (n_seq < 1 || n_row < 1 || n_kv < 1 || n_head < n_kv || hd < 1 || max_len < 1) return 0;
    const size_t blocks = 2 * (size_t) ceil_div(512, n_kv) + (size_t) (n_seq < n_row ? n_seq : n_row);
    const size_t cols = (size_t) n_row * (size_t) (n_head / n_kv);
    return (size_t) n_kv * blocks * (cols < 128 ? cols : 128) * (size_t) (hd + 2);
}

#define LOG2E 1.44269504088896341f
// A grid of items (y, z) for each KV head (x): the heads of neighbouring items
// run on the same XCDs, whose L2s each hold a head's pages once.
static void items_launch(const char * name, int n_kv, long items, unsigned threads, size_t lds, hipStream_t st, void * a) {
    const long y = items < 32768 ? items : 32768;
    hx_launch3(name, (unsigned) n_kv, (unsigned) y, (unsigned) ((items + y - 1) / y), threads, lds, st, a);
}

// The forms of the kernel: columns of a tile, waves beside each other, groups of
// them over the positions. Eight waves have a CU to themselves; of four, two
// workgroups share one, so that a short tile waits for no long one and one's
// products run beside the other's softmax.
static const struct form { const char * name; int cols, cw, pg; } forms[] = {
    { "rows64", 64, 2, 4 }, { "rows64h", 64, 2, 2 }, { "rows128", 128, 4, 2 }, { "rows128h", 128, 4, 1 }
};

// Tiles of 128 columns read the cache less often; those of 64 waste less of a few
// and make more workgroups. Measured as us a call, 32 heads over 8 of 128, fp16,
// rows x sequences at positions; bfloat16 and heads of 64 go by the same counts,
// which were not measured for them.
static const struct form * form_of(long ncol, long some, int n_kv) {
    const long ncu = hx.ncu, t64 = (ncol + 63) / 64 * n_kv, t128 = (ncol + 127) / 128 * n_kv;
    // long prompts, tiles for both places of every CU and more (128 / 128h / 64h: 4096 at 4096 295 / 291 / 299,
    // 8192 at 8192 1073 / 1023 / 1105, 2000 x 2 at 2000 122 / 103 / 121; but 2600 at 8000 594 / 629 / 626)
    if (t128 > 2 * ncu && ncol >= 2048 * some) return forms + 3;
    // a tile and a half a CU (2048 at 16384 953 / 971 / 1018; 2047 of packed documents, 28 heads over 4, 97 / 152 / 116)
    if (2 * t128 >= 3 * ncu && ncol >= 4096 * some) return forms + 2;
    // four sequences, or more tiles of 64 than CUs (64 / 64h / 128: 8 x 16 to 3000 47 / 36 / 53, 26 x 16 to 8192
    // 49 / 44 / 44, 8 x 48 to 4000 125 / 109 / 144, 33 x 200 to 600 213 / 130 / 164, 560 at 3000 98 / 85 / 89)
    if (some >= 4 || 16 * t64 > 17 * ncu) return forms + 1;
    // fewer (60 at 6000 28.9 / 31.3 / 30.6, 200 at 6000 61 / 62 / 58, 400 at 3000 56 / 61 / 58, 300 x 3 to 3000 70 /
    // 76 / 88)
    return forms;
}

static void rows_launch(sml_krows * a, int hd, int type, hipStream_t st) {
    const int n_kv = a->pg.n_kv, rep = a->n_head / n_kv, n_seq = a->pg.n_seq;
    const int ncol = a->n_row * rep, some = n_seq < a->n_row ? n_seq : a->n_row;
    const struct form * const f = form_of(ncol, some, n_kv);
    a->cols = f->cols;
    a->over = rep > 1 ? (uint32_t) (((1ull << 32) + (unsigned) rep - 1) / (unsigned) rep) : 0;
    // Splits make a workgroup for every place on the card, of 128 positions at least;
    // none where the tiles are more than half as many, of which each could only be one,
    // or as many sequences have rows (32 heads over 8 of 128, fp16, 32 places a KV head, none / split: 256 rows, 16
    // tiles, at 1024 25.5 / 23.9 us, at 8192 117 / 82; 272 rows, 17 tiles, 26.0 / 28.1 and
    // 120 / 123; bfloat16 at 8192 149 / 99 and, 320 rows, 153 / 155). That holds for
    // tiles as long as each other: 8 sequences of up to 128 rows at 500 to 4000 take 94 us
    // for 51 with splits, and a long sequence of one row beside a prompt's 256 rows is walked by
    // one workgroup a KV head (at 65536 774 us, apart 19 and 46).
    const int want = ceil_div((f->cw * f->pg == 8 ? 1 : 2) * (hx.ncu < 256 ? hx.ncu : 256), n_kv);
    a->least = 2;
    const int split = n_seq <= AT_SHARED && some < want && 2 * ceil_div(ncol, a->cols) <= want && a->max_len > RW_BLOCK * a->least;
    a->want = split ? want : 0;
    const long tiles = n_seq == 1 ? ceil_div(ncol, a->cols) : (long) ncol / a->cols + (split ? some : n_seq);
    const long items = split && tiles < want ? want : tiles;
    a->items = (int) items;
    a->part_cols = ncol < a->cols ? ncol : a->cols;
    // LDS: two stages a group, their positions and what they hold that is not finite, and the
    // columns' ranges; at the end the groups' sums; behind both a bit for each column's dims
    const size_t stages = (size_t) f->pg * 2 * (4 * 32 * hd + 4 * 32 + 4 * f->cw + 4 * hd) + (16 + 20 * 32 + 4 * 32 * f->pg) * f->cw;
    const size_t joined = (size_t) f->pg * f->cols * ((hd + 4) * 4 + 8);
    char base[24], name[40];
    snprintf(base, sizeof base, "sml_rw_%s%s", f->name, a->cap > 0.0f || a->slope ? "r" : "");
    sv_name(name, sizeof name, base, hd, type);
    items_launch(name, n_kv, items, 64 * (unsigned) (f->cw * f->pg), (stages > joined ? stages : joined) + (size_t) f->cols * hd / 8, st, a);
    if (split) {
        // a wave a column while that makes at most two workgroups a CU (us of the
        // merge at 4 / 16 columns a workgroup: one tile of 32 columns, 32 splits 4.0 /
        // 5.5, 16 sequences of 36 to 104 columns 10.6 / 5.9)
        const int per = tiles * (a->cols / 4) * n_kv <= 2L * hx.ncu ? 4 : 16;
        snprintf(name, sizeof name, "sml_rw_merge%d%s", per, hd == 64 ? "_d64" : "");
        items_launch(name, n_kv, tiles * (a->cols / per), 256, 0, st, a);
    }
}

int sml_hip_paged_attention_rows(const sml_hip_pages * pg, const sml_hip_rows * rows, const float * q, size_t q_stride,
                                 int n_head, float scale, float * part, float * out, void * stream) {
    HX_ENTRY(-1);
    sml_krows a;
    memset(&a, 0, sizeof a);
    sv_check_pages(pg, &a.pg);
    if (!rows || !rows->start || !rows->len) hx_failf("rows' attention: missing starts or lengths");
    if (rows->n_row < 0 || rows->n_row > 65535 || rows->max_len < 0)
        hx_failf("rows' attention: %d rows, lengths up to %d", rows->n_row, rows->max_len);
    if (rows->tree && (rows->tree_words < 1 || rows->tree_words > 2048))
        hx_failf("rows' attention: %d words of a tree's bits a row (1 to 2048)", rows->tree_words);
    if (n_head < 1 || n_head % pg->n_kv || n_head / pg->n_kv > 16)
        hx_failf("rows' attention: %d heads over %d kv heads (1 to 16 each)", n_head, pg->n_kv);
    const float sc = scale != 0.0f ? scale : 1.0f / sqrtf((float) pg->hd);
    if (!(rows->cap >= 0.0f) || isinf(rows->cap * LOG2E) ||
        (rows->cap > 0.0f && !(fabsf(sc) <= 0x1p100f * rows->cap && rows->cap <= 0x1p100f * fabsf(sc))))
        hx_failf("rows' attention: scores capped at %g", (double) rows->cap);
    if (!q || !part || !out) hx_failf("rows' attention: missing rows, workspace or output");
    if (!al16(part)) hx_failf("rows' attention: workspace off a 16-byte boundary");
    const size_t width = (size_t) n_head * pg->hd;
    if (q_stride && q_stride < width) hx_failf("rows' attention: rows of %zu floats %zu apart", width, q_stride);
    sv_on_device();
    if (rows->n_row) {
        a.q = q; a.q_stride = q_stride ? q_stride : width; a.part = part; a.out = out;
        a.start = rows->start; a.len = rows->len; a.first = rows->first; a.last = rows->last; a.pos = rows->pos;
        a.tree = rows->tree; a.words = rows->tree_words; a.slope = rows->slope; a.cap = rows->cap;
        a.sign = sc < 0.0f ? -1.0f : 1.0f;
        a.scale = rows->cap > 0.0f ? fabsf(sc) / rows->cap : fabsf(sc) * LOG2E;
        a.cap = rows->cap * LOG2E;
        a.n_head = n_head; a.n_row = rows->n_row;
        const long cap = (long) pg->seq_pages * pg->page_size;
        a.max_len = rows->max_len < cap ? rows->max_len : (int) cap;
        rows_launch(&a, pg->hd, pg->type, (hipStream_t) stream);
    }
    HX_LEAVE();
    return 0;
}

// The layers of a cache whose pages pg describes.
static void check_layers(const sml_hip_pages * pg, int n_layer, int least, size_t layer_stride) {
    const size_t page = (size_t) pg->page_size * pg->n_kv * pg->hd;
    if (n_layer < least || n_layer > 16384) hx_failf("paged cache: %d layers (%d to 16384)", n_layer, least);
    if (n_layer > 1 && (layer_stride < page || layer_stride % 8))
        hx_failf("paged cache: layers of %zu values a page %zu apart (a multiple of 8)", page, layer_stride);
}

int sml_hip_draft_accept(const sml_hip_pages * pg, int n_layer, size_t layer_stride, int n_row, const int32_t * start,
                         const int32_t * len, const int32_t * tok, const int32_t * parent, const int32_t * pick,
                         int max_kept, int32_t * n_kept, int32_t * kept, int32_t * next, int32_t * len_out,
                         void * stream) {
    HX_ENTRY(-1);
    sml_kaccept a;
    memset(&a, 0, sizeof a);
    sv_check_pages(pg, &a.pg);
    check_layers(pg, n_layer, 0, layer_stride);
    if (n_row < 0 || n_row > 1 << 22 || max_kept < 1 || max_kept > AC_MOST)
        hx_failf("accept: %d rows, %d kept a sequence (1 to %d)", n_row, max_kept, AC_MOST);
    if (!start || !len || (n_row && (!tok || !parent || !pick))) hx_failf("accept: missing starts, lengths, tokens, parents or picks");
    if (len_out == len) hx_failf("accept: lengths in place");
    sv_on_device();
    a.layer_stride = n_layer > 1 ? layer_stride : 0; a.n_layer = n_layer;
    a.start = start; a.len = len; a.tok = tok; a.parent = parent; a.pick = pick;
    a.n_kept = n_kept; a.kept = kept; a.next = next; a.len_out = len_out; a.n_row = n_row; a.most = max_kept;
    const long units = 2L * n_layer * pg->n_kv * pg->hd / 8;
    hx_launch("sml_rw_accept", (unsigned) (units ? (units + 255) / 256 : 1), (unsigned) pg->n_seq, 256, 0, (hipStream_t) stream, &a);
    HX_LEAVE();
    return 0;
}

#define FK_BLOCK (256 * 4 * 8)                        // values a workgroup copies
// Workgroups that a page of one pool takes.
static unsigned page_groups(const sml_hip_pages * pg) {
    return (unsigned) (((long) pg->page_size * pg->n_kv * pg->hd + FK_BLOCK - 1) / FK_BLOCK);
}

int sml_hip_paged_fork(const sml_hip_pages * pg, int n_layer, size_t layer_stride, const int32_t * len, int n_fork,
                       const int32_t * parent, const int32_t * fresh, int32_t * table_out, int32_t * len_out,
                       void * stream) {
    HX_ENTRY(-1);
    sml_kfork a;
    memset(&a, 0, sizeof a);
    sv_check_pages(pg, &a.pg);
    check_layers(pg, n_layer, 1, layer_stride);
    if (n_fork < 0 || n_fork > 65535) hx_failf("fork: %d sequences", n_fork);
    if (!len || !parent || !fresh || !table_out || !len_out) hx_failf("fork: missing lengths, parents, pages or outputs");
    if (table_out == pg->table || len_out == len) hx_failf("fork: table or lengths in place");
    sv_on_device();
    if (n_fork) {
        a.layer_stride = n_layer > 1 ? layer_stride : 0; a.n_layer = n_layer;
        a.len = len; a.n_fork = n_fork; a.parent = parent; a.fresh = fresh; a.table_out = table_out; a.len_out = len_out;
        hx_launch3("sml_rw_fork", page_groups(pg), (unsigned) n_fork, 2 * (unsigned) n_layer, 256, 0, (hipStream_t) stream, &a);
    }
    HX_LEAVE();
    return 0;
}

int sml_hip_paged_compact(const sml_hip_pages * pg, int n_layer, size_t layer_stride, int n_move, const int32_t * src,
                          const int32_t * dst, int32_t * table, void * stream) {
    HX_ENTRY(-1);
    sml_kcompact a;
    memset(&a, 0, sizeof a);
    sv_check_pages(pg, &a.pg);
    check_layers(pg, n_layer, 1, layer_stride);
    if (n_move < 0 || n_move > 65534) hx_failf("compact: %d pages", n_move);
    if (n_move && (!src || !dst)) hx_failf("compact: missing pages");
    sv_on_device();
    if (n_move) {
        a.layer_stride = n_layer > 1 ? layer_stride : 0; a.n_layer = n_layer;
        a.src = src; a.dst = dst; a.table = table; a.n_move = n_move;
        hx_launch3("sml_rw_compact", page_groups(pg), (unsigned) n_move + (table != NULL), 2 * (unsigned) n_layer, 256, 0,
                   (hipStream_t) stream, &a);
    }
    HX_LEAVE();
    return 0;
}
