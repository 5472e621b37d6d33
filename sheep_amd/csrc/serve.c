// The operators of a step that serves many requests at once (sml-serve.h):
// argument checks and launches. The checks come before the device is touched,
// so they refuse alike on a machine without one.
#include "serve.h"

#include <math.h>
#include <stdio.h>
#include <string.h>

// The device of sml_hip_init has to be the calling thread's: the stream and
// the buffers of another one would meet kernels loaded for this one.
void sv_on_device(void) {
    if (!hx.inited) hx_init(0);
    int d = -1;
    HX(hipGetDevice(&d));
    if (d != hx.device) hx_failf("device %d is current, the library runs on device %d", d, hx.device);
}

void sv_check_pages(const sml_hip_pages * p, sml_kpages * k) {
    if (!p || !p->k || !p->v || !p->table) hx_failf("paged cache: missing pools or table");
    if (p->type != SML_F16 && p->type != SML_BF16) hx_failf("paged cache: type %d", p->type);
    if (p->hd != 64 && p->hd != 128) hx_failf("paged cache: head_dim %d (64 or 128)", p->hd);
    if (p->n_kv < 1 || p->n_kv > 4096) hx_failf("paged cache: %d kv heads", p->n_kv);
    if (p->page_size < 16 || p->page_size > 65536 || (p->page_size & (p->page_size - 1)))
        hx_failf("paged cache: pages of %d positions (a power of two, 16..65536)", p->page_size);
    const size_t page = (size_t) p->page_size * p->n_kv * p->hd;
    if (page > (size_t) 1 << 30) hx_failf("paged cache: pages of %zu values", page);
    if (p->page_stride && (p->page_stride < page || p->page_stride % 8))
        hx_failf("paged cache: page stride %zu for pages of %zu values (a multiple of 8)", p->page_stride, page);
    if (p->n_pages < 1 || p->n_seq < 1 || p->n_seq > 65535 || p->seq_pages < 1)
        hx_failf("paged cache: %d pages, %d sequences of %d pages", p->n_pages, p->n_seq, p->seq_pages);
    if ((uint64_t) p->seq_pages * (uint64_t) p->page_size > (uint64_t) 1 << 30)
        hx_failf("paged cache: %d pages of %d positions a sequence", p->seq_pages, p->page_size);
    if (!al16(p->k) || !al16(p->v)) hx_failf("paged cache: pools off 16-byte boundaries");
    memset(k, 0, sizeof *k);
    k->k = p->k; k->v = p->v; k->table = p->table;
    k->page_stride = p->page_stride ? p->page_stride : page;
    k->n_pages = p->n_pages; k->page_shift = __builtin_ctz((unsigned) p->page_size);
    k->n_seq = p->n_seq; k->seq_pages = p->seq_pages; k->n_kv = p->n_kv; k->hd = p->hd;
}

void sv_name(char * s, size_t n, const char * base, int hd, int type) {
    snprintf(s, n, "%s%s%s", base, hd == 64 ? "_d64" : "", type == SML_BF16 ? "_bf" : "");
}

int sml_hip_paged_append(const sml_hip_pages * pg, float * qkv, size_t qkv_stride, int n_rows, const int32_t * seq,
                         const int32_t * pos, const float * cos_t, const float * sin_t, int n_rope, int n_head,
                         float * q_out, void * stream) {
    HX_ENTRY(-1);
    sml_kappend a;
    memset(&a, 0, sizeof a);
    sv_check_pages(pg, &a.pg);
    if (n_rows < 0 || n_rows > 1 << 22 || n_head < 1 || n_head > 65536) hx_failf("append: %d rows of %d heads", n_rows, n_head);
    const size_t width = ((size_t) n_head + 2 * (size_t) pg->n_kv) * pg->hd;
    if (!qkv || !pos || !cos_t || !sin_t || n_rope < 1) hx_failf("append: missing rows, positions or rotation tables");
    if (qkv_stride && qkv_stride < width) hx_failf("append: rows of %zu floats %zu apart", width, qkv_stride);
    sv_on_device();
    if (n_rows) {
        a.qkv = qkv; a.stride = qkv_stride ? qkv_stride : width; a.seq = seq; a.pos = pos;
        a.cos_t = cos_t; a.sin_t = sin_t; a.q_out = q_out; a.n_rope = n_rope; a.n_head = n_head;
        char name[40];
        sv_name(name, sizeof name, "sml_sv_append", pg->hd, pg->type);
        const int items = (n_head + pg->n_kv) * (pg->hd / 8) + pg->n_kv * (pg->hd / 4);
        hx_launch(name, (unsigned) n_rows, (unsigned) ceil_div(items, 256), 256, 0, (hipStream_t) stream, &a);
    }
    HX_LEAVE();
    return 0;
}

size_t sml_hip_paged_part_floats(int n_seq, int n_head, int hd, int max_len) {
    if (n_seq < 1 || n_head < 1 || hd < 1 || max_len < 1) return 0;
    const int ns = ceil_div(max_len, 64);
    return (size_t) n_seq * (size_t) n_head * (size_t) (ns < 256 ? ns : 256) * (size_t) (hd + 2);
}

int sml_hip_paged_attention(const sml_hip_pages * pg, const float * q, size_t q_stride, const int32_t * len,
                            int max_len, int n_head, float scale, float * part, float * out, void * stream) {
    HX_ENTRY(-1);
    sml_kattend a;
    memset(&a, 0, sizeof a);
    sv_check_pages(pg, &a.pg);
    if (n_head < 1 || n_head % pg->n_kv || n_head / pg->n_kv > 16)
        hx_failf("paged attention: %d heads over %d kv heads (1 to 16 each)", n_head, pg->n_kv);
    if (!q || !len || !part || !out || max_len < 0) hx_failf("paged attention: missing buffers, or lengths up to %d", max_len);
    if (!al16(part)) hx_failf("paged attention: workspace off a 16-byte boundary");
    const size_t width = (size_t) n_head * pg->hd;
    if (q_stride && q_stride < width) hx_failf("paged attention: rows of %zu floats %zu apart", width, q_stride);
    sv_on_device();
    a.q = q; a.q_stride = q_stride ? q_stride : width; a.len = len; a.part = part; a.out = out;
    a.scale = (scale != 0.0f ? scale : 1.0f / sqrtf((float) pg->hd)) * 1.44269504088896341f;
    a.n_head = n_head;
    const long cap = (long) pg->seq_pages * pg->page_size;
    a.max_len = max_len < cap ? max_len : (int) cap;
    // splits of 128 positions (a tile a wave) at least, and no more than the
    // workspace's of the longest sequence
    a.nsplit = ceil_div(max_len > 1 ? max_len : 1, 64);
    if (a.nsplit > 256) a.nsplit = 256;
    // Two workgroups a CU, 512, where the lengths are shared out (48
    // sequences up to 8192 / one at 65537 / 16 of 2000 / 32 of 1000 to 9000 with
    // 12 heads over 2, us: 512 55, 36, 32, 24; 768 54, 37, 37, 27; 1024 52, 37, 35,
    // 27).
    // Up to 512 positions a sequence is one split, with no merge (whole / split:
    // one sequence of 256 5.9 / 8.0 us, of 512 8.0 / 8.5, of 768 9.9 / 8.8; 64 of
    // 512 23 / 26).
    const int n = a.max_len > 1 ? a.max_len : 1, shared = pg->n_seq <= AT_SHARED;
    const int least = shared && n > 512 ? 128 : 512;
    a.chunk = least * ceil_div(n, least * 256);
    a.want = shared ? ceil_div(2 * hx.ncu, pg->n_kv) : 0;
    // every sequence's first split, and those that the lengths can make beyond
    long grid = ceil_div(n, a.chunk);
    if (shared) {
        grid *= pg->n_seq;
        if (grid > (long) a.want + pg->n_seq) grid = (long) a.want + pg->n_seq;
    }
    char name[40];
    sv_name(name, sizeof name, "sml_sv_attend", pg->hd, pg->type);
    hx_launch3(name, (unsigned) pg->n_kv, (unsigned) grid, shared ? 1 : (unsigned) pg->n_seq, 256, 0, (hipStream_t) stream, &a);
    if (n > a.chunk) {
        // more threads a row while the workgroups are at most 2 a CU (measured
        // beside the kernel)
        const int nt = (long) n_head * pg->n_seq <= 2L * hx.ncu ? 512 : 256;
        snprintf(name, sizeof name, "sml_sv_merge%s_%d", pg->hd == 64 ? "_d64" : "", nt);
        hx_launch(name, (unsigned) n_head, (unsigned) pg->n_seq, (unsigned) nt, 0, (hipStream_t) stream, &a);
    }
    HX_LEAVE();
    return 0;
}

size_t sml_hip_logits_part_bytes(int n_row, int n_vocab) {
    if (n_row < 1 || n_vocab < 1) return 0;
    return (size_t) n_row * (size_t) ceil_div(n_vocab, LG_RANGE) * sizeof(int4);
}

int sml_hip_logits_adjust(const float * logits, size_t stride, int n_row, int n_vocab, const sml_hip_rules * rules,
                          float * out, size_t out_stride, int32_t * tok, void * part, void * stream) {
    HX_ENTRY(-1);
    if (n_row < 0 || n_row > 65535 || n_vocab < 1 || n_vocab > 1 << 30)
        hx_failf("logits: %d rows of %d", n_row, n_vocab);
    if (!logits || (!out && !tok) || (tok && !part)) hx_failf("logits: missing rows, output or workspace");
    if ((stride && stride < (size_t) n_vocab) || (out_stride && out_stride < (size_t) n_vocab))
        hx_failf("logits: rows of %d floats %zu and %zu apart", n_vocab, stride, out_stride);
    sml_klogits a;
    memset(&a, 0, sizeof a);
    a.logits = logits; a.out = out; a.tok = tok; a.part = part; a.n_vocab = n_vocab;
    a.stride = stride ? stride : (size_t) n_vocab;
    a.out_stride = out_stride ? out_stride : (size_t) n_vocab;
    if (out == logits && a.out_stride != a.stride) hx_failf("logits: in place with strides %zu and %zu", a.stride, a.out_stride);
    if (tok && ((uintptr_t) part & 15u)) hx_failf("logits: workspace off a 16-byte boundary");
    if (rules) {
        const sml_hip_rules * r = rules;
        if (r->n_hist < 0 || r->n_hist > 1 << 30 || r->n_bias < 0 || r->n_bias > 1 << 30 || r->n_mask < 0)
            hx_failf("logits: %d ids, %d biases, %d masks", r->n_hist, r->n_bias, r->n_mask);
        if (r->hist && r->n_hist && (r->rep || r->presence || r->frequency)) {
            if (!r->hist_start) hx_failf("logits: a history without hist_start");
            a.hist = r->hist; a.hist_start = r->hist_start; a.n_prompt = r->n_prompt; a.n_hist = r->n_hist;
            a.rep = r->rep; a.presence = r->presence; a.frequency = r->frequency;
        }
        if (r->bias && r->n_bias) {
            if (!r->bias_id || !r->bias_start) hx_failf("logits: biases without bias_id or bias_start");
            a.bias = r->bias; a.bias_id = r->bias_id; a.bias_start = r->bias_start; a.n_bias = r->n_bias;
        }
        if (r->mask) {
            if (!r->mask_row && r->n_mask < n_row) hx_failf("logits: %d masks for %d rows without mask_row", r->n_mask, n_row);
            a.mask = r->mask; a.mask_row = r->mask_row; a.n_mask = r->n_mask;
        }
    }
    sv_on_device();
    if (n_row) {
        a.n_part = ceil_div(n_vocab, LG_RANGE);
        // one word a thread while the workgroups are at most 2 a CU (a call of
        // latencies), else half the threads with two (measured beside the kernel)
        const int wide = (long) a.n_part * n_row <= 2L * hx.ncu;
        hx_launch(wide ? "sml_sv_logits_512_1" : "sml_sv_logits_256_2", (unsigned) a.n_part, (unsigned) n_row,
                  wide ? 512 : 256, 0, (hipStream_t) stream, &a);
        if (tok) hx_launch("sml_sv_pick", (unsigned) n_row, 1, 64, 0, (hipStream_t) stream, &a);
    }
    HX_LEAVE();
    return 0;
}

size_t sml_hip_lora_work_floats(int rank, int n_row) {
    if (rank < 1 || n_row < 1) return 0;
    const size_t split = 32 * (size_t) n_row < 8192 ? 32 * (size_t) n_row : 8192;
    return (size_t) rank * (split > (size_t) n_row ? split : (size_t) n_row);
}

#define LD_ROWS 16                                    // rows of a tile

// The workgroups of a product that run at once: two a CU by their registers, if
// the CU's LDS (a little of it is theirs beside lds) holds them. It does not
// where bf16's three parts meet 32 ranks of A or, at 32 rows, 256 ranks of B
// (us a call of bf16 with these taken for two a CU / so: 80 rows of 16 adapters,
// 14336 to 4096, rank 64 32.1 / 29.0, 256 rows 32.9 / 27.1, 509 rows of 4096 to
// 4096, rank 256 64 / 45, of 4 adapters in runs 53 / 38; the most that lose, 128
// rows of 64 adapters 75 / 79).
static int at_once(size_t lds) { return hx.ncu * (2 * (lds + 256) <= 160 << 10 ? 2 : 1); }

// One launch or two, as measured beside the kernels. One: up to 16 rows of rank
// up to 64, sums that fit LDS, at most 2.5 workgroups a CU, and few row products a
// wave (rounds of its 8 ranks of 512 inputs, each taking the adapter's rows one
// by one): 8 if the rows share the pool's adapters alike, 16 if all had one.
// Which adapters they have only the device knows: where all rows have the same
// one of a pool as large as the batch, one launch loses what two would save (us
// with one launch, a row each of its own adapter / all of one, and two launches,
// all of one; rank 16, 4096 to 4096: 4 rows 5.8 / 7.4, 11.1, 8 rows 6.5 / 10.1,
// 11.1, 16 rows 8.0 / 15.6, 11.0; 14336 to 4096: 4 rows 9.7 / 15.1, 13.0; rank 64,
// 4096 to 4096: 4 rows 11.0 / 17.5, 12.6).
static void lora_launch(sml_klora * a, int bf, hipStream_t st) {
    const int parts = bf ? 3 : 2, nslice = ceil_div(a->n_in, LF_SLICE), few = a->n_row < 16 ? a->n_row : 16;
    const size_t sums = (size_t) nslice * 16 * (size_t) a->rank * 4;
    const long rounds = ceil_div(nslice * (a->rank / 8), LF_WAVES);
    if (a->n_row <= 16 && a->rank <= LF_RANK && sums <= 96 << 10 && a->n_row * rounds <= 16 &&
        ceil_div(a->n_row, a->n_adapter) * rounds <= 8 && (long) ceil_div(a->n_out, LF_OUT) * few <= 5L * hx.ncu / 2) {
        hx_launch(bf ? "sml_sv_lora_few_bf" : "sml_sv_lora_few", (unsigned) ceil_div(a->n_out, LF_OUT), (unsigned) few,
                  64 * LF_WAVES, (size_t) parts * 16 * LF_LD * 2 + 64 + sums, st, a);
        return;
    }
    a->sorted = a->n_row > 32 && a->n_row <= LS_ROWS && a->n_adapter > 1 && a->n_adapter <= LS_ADAPTERS;
    // t: the inputs split for half a workgroup a CU of 64 ranks, twice as many of
    // up to 16, as far as the workspace holds them (509 rows, us a call at half /
    // so / twice: rank 64, 4096 to 14336 30.6 / 29.5 / 33.3, rank 16, 14336 to
    // 4096 21.1 / 20.0 / -): every workgroup of y joins them, so that splits times
    // ranks stay within 768 too (14336 to 4096, with that and without: 16 rows,
    // rank 64 16.2 / 20.8, 32 rows, rank 128 19.6 / 31.8, 1 row, rank 256 22.6 /
    // 21.9).
    const int ntile = ceil_div(a->n_row, LD_ROWS), ngroup = ceil_div(a->rank, 64);
    int most = 8192 / a->n_row < 32 ? 8192 / a->n_row : 32;
    if (most > 768 / a->rank) most = 768 / a->rank;
    const int want = ceil_div(a->rank <= 16 ? hx.ncu : hx.ncu / 2, ntile * ngroup);
    if (most > want) most = want;
    if (most < 1) most = 1;
    a->chunk = LD_TILE;
    while (ceil_div(a->n_in, a->chunk) > most) a->chunk += LD_TILE;
    a->nsplit = ceil_div(a->n_in, a->chunk);
    // 32 ranks a workgroup, of low ranks or few rows 16 (us a call at 16 / 32: 16
    // rows, rank 64, 14336 to 4096 16.2 / 17.3, 32 rows, rank 16, 4096 to 4096 11.3
    // / 11.6; 144 rows, rank 64, 14336 to 4096 21.0 / 18.2)
    const int rt = a->rank <= 16 || a->n_row <= 64 ? 1 : 2;
    // y: 32 rows a workgroup of a prompt (us a call at 16 / 32, one adapter: 192
    // rows, 4096 to 14336, rank 64 17.8 / 19.3, 14336 to 4096 19.5 / 23.4; 384
    // rows 24.5 / 24.3 and 23.8 / 25.9, 1536 to 8960, rank 8 18.7 / 14.9; 509
    // rows of 4 adapters in runs 33.6 / 31.5, 30.8 / 27.0 at rank 16), and the
    // workgroups that run at once, never more (the same case with 256 / 512 /
    // 1024: 35 / 30 / 34; 192 rows, rank 64, with 576: 24.8 for 17.8). A
    // row tile's workgroups are a multiple of 8, so that the same outputs' B goes
    // to the same XCD's L2, where that drops few of them (320 rows, rank 64, 48
    // for 51: 22.7 / 24.8; 700 rows, rank 16, 16 for 23: 29.0 / 27.5).
    const int rb = a->n_row <= 256 ? 1 : 2, nrt = ceil_div(a->n_row, 16 * rb);
    // (the sort's counts, 8 KB, fit before the rest)
    const size_t lds_d = (size_t) LD_WAVES * LD_WAVE_LDS(parts, rt),
                 lds_u = (size_t) 4 * LU_OUT * LD_ROW + (size_t) 16 * rb * (4 + (size_t) parts * ((size_t) ngroup * 64 + 8) * 2);
    const int once_d = at_once(lds_d), once_u = at_once(lds_u);
    int gx = once_u / nrt;
    if (gx >= 24) gx -= gx % 8;
    if (gx > ceil_div(a->n_out, 4 * LU_OUT)) gx = ceil_div(a->n_out, 4 * LU_OUT);
    if (gx < 1) gx = 1;
    // a tile's distinct adapters are shared out while both launches then stay
    // within the workgroups that run at once (us a call with 1 / 2 / 4 / 8 / 16
    // shares, rank 16: 32 rows of 32 adapters, 4096 to 4096 35 / 25 / 18.5 / 15.3 /
    // 14.2, 4096 to 14336 35 / 25.5 / 20.3 / 25 / 33; 64 of 64, 4096 to 4096 46 / 35
    // / 29 / 26 / 38, 14336 to 4096 53 / 39 / 33 / 41 / 68; 128 of 64, 4096 to 14336
    // 41 / 49 / 67)
    const int down = a->nsplit * ntile * ceil_div(a->rank, 16 * rt), up = gx * nrt;
    int nz = 1;
    while (2 * nz <= few && 2 * nz <= a->n_adapter && 2 * nz * down <= once_d && 2 * nz * up <= once_u) nz *= 2;
    char name[40];
    snprintf(name, sizeof name, "sml_sv_lora_down%d%s", rt, bf ? "_bf" : "");
    hx_launch3(name, (unsigned) a->nsplit, (unsigned) ntile, (unsigned) (nz * ceil_div(a->rank, 16 * rt)), 64 * LD_WAVES,
               lds_d, st, a);
    snprintf(name, sizeof name, "sml_sv_lora_up%d%s", rb, bf ? "_bf" : "");
    hx_launch3(name, (unsigned) gx, (unsigned) nrt, (unsigned) nz, 256, lds_u, st, a);
}

int sml_hip_lora_add(const sml_hip_adapters * ad, const float * x, size_t x_stride, int n_row, const int32_t * adapter,
                     const float * base, float * y, size_t y_stride, float * work, void * stream) {
    HX_ENTRY(-1);
    if (!ad || !ad->a || !ad->b) hx_failf("adapters: missing pools");
    if (ad->type != SML_F16 && ad->type != SML_BF16) hx_failf("adapters: type %d", ad->type);
    if (ad->n_adapter < 1 || ad->rank < 8 || ad->rank > 256 || ad->rank % 8)
        hx_failf("adapters: %d of rank %d (a multiple of 8 up to 256)", ad->n_adapter, ad->rank);
    if (ad->n_in < 8 || ad->n_in % 8 || ad->n_in > 1 << 24 || ad->n_out < 1 || ad->n_out > 1 << 24)
        hx_failf("adapters: %d inputs (a multiple of 8), %d outputs", ad->n_in, ad->n_out);
    if (!al16(ad->a) || !al16(ad->b)) hx_failf("adapters: pools off 16-byte boundaries");
    if (n_row < 0 || n_row > 65535) hx_failf("adapters: %d rows", n_row);
    if (!x || !adapter || !y || !work) hx_failf("adapters: missing rows, ids, output or workspace");
    if ((x_stride && x_stride < (size_t) ad->n_in) || (y_stride && y_stride < (size_t) ad->n_out))
        hx_failf("adapters: rows of %d and %d floats %zu and %zu apart", ad->n_in, ad->n_out, x_stride, y_stride);
    sv_on_device();
    if (n_row) {
        sml_klora a;
        memset(&a, 0, sizeof a);
        a.a = ad->a; a.b = ad->b; a.scale = ad->scale; a.ranks = ad->ranks; a.adapter = adapter;
        a.x = x; a.base = base; a.y = y; a.work = work;
        a.x_stride = x_stride ? x_stride : (size_t) ad->n_in;
        a.y_stride = y_stride ? y_stride : (size_t) ad->n_out;
        a.n_adapter = ad->n_adapter; a.rank = ad->rank; a.n_in = ad->n_in; a.n_out = ad->n_out; a.n_row = n_row;
        lora_launch(&a, ad->type == SML_BF16, (hipStream_t) stream);
    }
    HX_LEAVE();
    return 0;
}
