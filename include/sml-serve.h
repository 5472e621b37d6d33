// Operators of a step that serves many requests at once, on device buffers:
// a paged key/value cache and the attention of one new token a sequence, or of
// several (a draft's tree, a prompt's chunk), over it, what such a cache's
// upkeep takes (accepted drafts, forks, compaction), low-rank adapters beside a
// shared projection, and penalties, biases and grammar masks on logits with the
// greedy pick. They stand beside the
// contiguous cache, the products and the pick of sml-hip.h, whose conventions
// hold here: device pointers unless a comment says host, 0 on success and -1
// on failure with the reason in sml_hip_last_error(). The reference has no
// counterpart of any of them: it keeps one contiguous cache per sequence
// (sml/sml-run.c:3414-3434) and picks greedily (sml/sml-run.c:3539-3544).
//
// Every call enqueues its launches on `stream` (a hipStream_t; NULL: the null
// stream, where the rest of the kernel-level ABI runs), allocates nothing,
// never waits and may be captured into a HIP graph once sml_hip_init has run.
// Buffers used on another stream than the one they were filled on are the
// caller's to order, by events: so are the results of sml-hip.h's products,
// which run on the null stream (and are not captured with these calls), for a
// stream that does not wait for it. Workspaces are the caller's too: calls that
// may overlap (on two streams, or in two graphs replayed side by side) need one
// each; nothing in a workspace outlives its call. The calls are made by one host
// thread at a time, with the device of sml_hip_init current; with another
// device current they are refused.
#pragma once
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

// The 16-bit type of a cache or an adapter pool.
enum { SML_F16 = 0, SML_BF16 = 1 };

// ------------------------------------------------------------ paged cache
// One layer's keys and values in pages of page_size positions (a power of
// two, 16..65536), each [page_size][n_kv][hd] (hd 64 or 128) in each pool.
// Position p of sequence s lies in page table[s * seq_pages + p / page_size].
// A table entry outside 0..n_pages-1 (-1 by custom) is no page: nothing is
// written there, and attention leaves its positions out.
// Sequences may name the same pages (a common prefix, or several rows of one
// request).
typedef struct {
    uint16_t * k, * v;            // the pools, 16-byte aligned
    const int32_t * table;        // [n_seq][seq_pages]
    size_t page_stride;           // values from one page to the next in a pool, a multiple of 8
                                  //   (0: page_size * n_kv * hd), so layers may share pages
    int n_pages, page_size;
    int n_seq, seq_pages;         // seq_pages * page_size at most 2^30
    int n_kv, hd, type;           // type: SML_F16 or SML_BF16
} sml_hip_pages;

// Append n_rows new tokens (0..2^22). Row r of qkv (qkv_stride floats apart,
// 0: (n_head + 2 * n_kv) * hd) holds a token's q, k and v after bias, as the
// stacked product leaves them; it is position pos[r] of sequence seq[r] (seq
// NULL: sequence r). q and k are rotated by their position (halved pairs,
// table rows of hd / 2), k and v rounded to the cache's type (nearest even)
// and written to their page; the rotated q goes to q_out [n_rows][n_head*hd]
// (apart from qkv), or back to its place in qkv when q_out is NULL. In fp16 the cache then holds
// what sml_hip_attention would have written, bit for bit.
// A row is left out, its q_out included, when its position is negative or at
// or past n_rope or seq_pages * page_size, its sequence is outside 0..n_seq-1
// or its page is none: rows of padding carry position -1. The rows of one
// call are for distinct places; where some share one (a position twice, or a page
// that two sequences name), each value there is one of theirs, not all of them
// the same row's.
int sml_hip_paged_append(const sml_hip_pages * pg, float * qkv, size_t qkv_stride, int n_rows, const int32_t * seq,
                         const int32_t * pos, const float * cos_t, const float * sin_t, int n_rope, int n_head,
                         float * q_out, void * stream);

// Floats of the workspace of sml_hip_paged_attention:
// n_seq * n_head * min(256, ceil(max_len / 64)) * (hd + 2).
size_t sml_hip_paged_part_floats(int n_seq, int n_head, int hd, int max_len);
// Attention of one token a sequence: q row b (q_stride floats apart, 0:
// n_head * hd; rotated already) over the first len[b] positions of sequence b,
// scaled by `scale` (0: 1 / sqrt(hd)), into out [n_seq][n_head * hd]. n_head is
// a multiple of n_kv, at most 16 query heads per KV head. max_len (host) bounds
// every length and sizes the launch (a tight bound is faster); a longer len[b]
// is cut to it and to seq_pages * page_size, a negative one is 0. Positions
// past the length and on absent pages count for nothing, whatever their memory
// holds. A sequence with no position left, or with no score above -infinity,
// gets zeros. Softmax statistics and sums are fp32; q and the weights meet the
// cache in the matrix cores as sums of 16-bit parts that together hold them to
// fp32's accuracy. Finite queries, keys and values give finite outputs wherever
// fp32 holds q * scale, the sums of |q_d k_d|, twice those times |scale|, and
// the sums of weight * |value|, the largest weight 1; an infinite or NaN value that
// a sequence does attend over makes its dim of its KV head's outputs infinite or
// NaN, however small its weight, and no other; an infinite or NaN query makes its
// own head's outputs NaN. So does a key of its KV head's, unless the score is
// -infinity: that has no weight (such a position's values that are not finite may
// count or not). How the positions are split follows all of the lengths: a
// sequence's sums depend on the others by their rounding alone, and equal calls
// give equal bits.
int sml_hip_paged_attention(const sml_hip_pages * pg, const float * q, size_t q_stride, const int32_t * len,
                            int max_len, int n_head, float scale, float * part, float * out, void * stream);

// ------------------------------------------------------------ several rows a sequence
// Append with the place and the rotation of a row apart: row r goes to position
// slot[r] of its sequence's pages, and pair d of its q and k (halved pairs, d <
// hd / 2) is turned by row pos[axis[d] * n_rows + r] of the tables. One axis: the
// drafts of a tree, whose siblings share a position and not a slot. Several (at
// most 4): time, height and width of an image's or a video's rows, axis giving
// each pair its own in sections, in turn or as the model has it. axis lies in
// host memory ([hd / 2], read before the call returns); a pair whose axis is
// n_axis or more is not turned.
// Everything else is sml_hip_paged_append's: a row is left out when its slot is
// outside the sequence's pages, any of its n_axis positions outside
// 0..n_rope - 1, its sequence outside 0..n_seq - 1 or its page none.
int sml_hip_paged_append_axes(const sml_hip_pages * pg, float * qkv, size_t qkv_stride, int n_rows, const int32_t * seq,
                              const int32_t * slot, const int32_t * pos, int n_axis, const uint8_t * axis,
                              const float * cos_t, const float * sin_t, int n_rope, int n_head, float * q_out,
                              void * stream);

// New rows of ragged sequences and what each of them attends to. Rows
// start[b] .. start[b+1] - 1 are sequence b's m newest positions: they lie in its
// slots h .. len[b] - 1, h = len[b] - m, in order (appended already).
typedef struct {
    const int32_t * start;        // [n_seq + 1], not falling; clamped to 0..n_row
    const int32_t * len;          // [n_seq] the sequence's positions, its new rows among them
    // Row r attends to slots first[r] .. last[r] - 1. first NULL: 0; last NULL:
    // up to its own slot, that included, or with a tree up to h. A window, packed
    // documents, a prefix that all of its rows see, or an empty row of padding
    // are these two.
    const int32_t * first, * last;   // [n_row]
    // and to slot h + j for each bit j set (bit j % 32 of word j / 32), j < m: a
    // drafted row's ancestors and itself
    const uint32_t * tree;        // [n_row][tree_words], NULL: none
    // The bias of distance: slope[head] * |the row's position - the slot's| is
    // subtracted from a score. A new row's position, and its slot's, is pos[r]
    // (NULL: its slot); an earlier slot's is its number.
    const int32_t * pos;          // [n_row], at most 2^30 in size
    const float * slope;          // [n_head], NULL: no bias
    float cap;                    // a score s becomes cap * tanh(s / cap) before the bias; 0: it stays.
                                  //   Within a factor of 2^100 of |scale|
    int tree_words;
    int n_row;                    // 0..65535
    int max_len;                  // (host) bounds every length, as above
} sml_hip_rows;

// Floats of the workspace of sml_hip_paged_attention_rows: n_kv * (2 *
// ceil(512 / n_kv) + min(n_seq, n_row)) * min(128, n_row * n_head / n_kv) * (hd + 2).
size_t sml_hip_paged_rows_floats(int n_seq, int n_row, int n_kv, int n_head, int hd, int max_len);
// Attention of every new row over its sequence's pages, each page read once for
// the rows and heads that share it: q row r (q_stride floats apart, 0: n_head *
// hd; rotated already), scaled by `scale` (0: 1 / sqrt(hd)), into row r of out
// [n_row][n_head * hd]. n_head is a multiple of n_kv, at most 16 query heads per
// KV head. A longer len[b] is cut to max_len and to seq_pages * page_size, a
// negative one is 0. Slots past the length and on absent pages are nobody's.
// What a row does not attend to does not count, whatever its memory holds, and
// also where other rows of the call do attend to it; a row with no slot left, or
// with no score above -infinity, gets zeros. Rows outside every sequence's are
// left as they were. Precision, ranges and infinities are
// sml_hip_paged_attention's; the cap and the bias are fp32, and a key's infinite
// score may be the cap's, with its sign. How the positions are
// split follows all of the lengths: a row's sums depend on the other rows by
// their rounding alone, and equal calls give equal bits.
int sml_hip_paged_attention_rows(const sml_hip_pages * pg, const sml_hip_rows * rows, const float * q, size_t q_stride,
                                 int n_head, float scale, float * part, float * out, void * stream);

// ------------------------------------------------------------ the cache's upkeep
// These act on n_layer layers of one cache at once, which share pg's table: layer
// l's pools lie l * layer_stride values behind pg's (a multiple of 8, at least a
// page; unused with one layer). Both ways of laying layers out are meant: whole
// pools one after another, or each page's layers side by side (page_stride).

// What the picks of a drafted step accept. Row start[b] of sequence b is the last
// token that was sure, the others are its drafted tree: tok[r] is the token
// drafted at row r, parent[r] the number in the sequence (0: the root) of the row
// it follows, which comes before it, pick[r] the model's pick behind row r
// (sml_hip_logits_adjust's tok). From the root on, the path goes on to the first
// child whose token is its row's pick, until there is none or max_kept (1..1024)
// rows are kept. Out: n_kept[b]; kept[b][j], the path's rows by number; next[b][j],
// the tokens that follow them (row j's pick; the last is the next step's root);
// both [n_seq][max_kept], -1 behind; len_out[b] = len[b] - m + n_kept[b] (apart
// from len; a negative len[b] is 0). Keys and values of the path's rows move to
// slots h, h + 1 and on, in all layers, where both slots have pages; n_layer 0 moves
// nothing. Any of the outputs may be NULL. A sequence of no rows keeps none. The
// slots of new rows belong to one sequence alone.
int sml_hip_draft_accept(const sml_hip_pages * pg, int n_layer, size_t layer_stride, int n_row, const int32_t * start,
                         const int32_t * len, const int32_t * tok, const int32_t * parent, const int32_t * pick,
                         int max_kept, int32_t * n_kept, int32_t * kept, int32_t * next, int32_t * len_out,
                         void * stream);

// n_fork (0..65535) sequences that go on from others: row i of table_out
// [n_fork][seq_pages] (apart from pg's table) gets the full pages of sequence
// parent[i]'s first len[parent[i]] positions; the page after them, if it is
// begun, is fresh[i], into which the positions it has are copied in all layers;
// -1 behind. len_out[i] = len[parent[i]] (apart from len), cut to 0..seq_pages *
// page_size. fresh[i] outside 0..n_pages - 1 copies nothing and names the
// parent's page itself: for the one child that goes on in it. A parent outside
// 0..n_seq - 1 gives an empty sequence. Fresh pages are distinct and nobody's
// before the call; of an absent page nothing is copied.
int sml_hip_paged_fork(const sml_hip_pages * pg, int n_layer, size_t layer_stride, const int32_t * len, int n_fork,
                       const int32_t * parent, const int32_t * fresh, int32_t * table_out, int32_t * len_out,
                       void * stream);

// n_move (0..65534) pages moved: page src[i] is copied to page dst[i] in all
// layers, and every entry of table ([n_seq][seq_pages], as a rule pg's; NULL:
// none) that names src[i] names dst[i] then, whichever sequences share it. src is
// ascending; dst are distinct pages that nobody names and that are none of src.
// Pages outside 0..n_pages - 1 move nothing.
int sml_hip_paged_compact(const sml_hip_pages * pg, int n_layer, size_t layer_stride, int n_move, const int32_t * src,
                          const int32_t * dst, int32_t * table, void * stream);

// ------------------------------------------------------------ logits
// What changes a row of logits before the pick; any of the parts may be NULL.
typedef struct {
    // the row's tokens so far: ids hist[hist_start[b] .. hist_start[b+1]), the
    // first n_prompt[b] of them (NULL: none) its prompt, the rest generated
    const int32_t * hist;         // [n_hist], at most 2^30
    const int32_t * hist_start;   // [n_row + 1], clamped to 0..n_hist
    const int32_t * n_prompt;     // [n_row]
    int n_hist;
    // per row, each NULL for none: rep divides a positive logit of a token in
    // the list and multiplies another; then frequency times its generated
    // count is subtracted, then presence if that count is not 0
    const float * rep, * presence, * frequency;
    // then bias[i] is added to token bias_id[i], i in bias_start[b] ..
    // bias_start[b+1]; of a token listed twice the last entry counts
    const int32_t * bias_id;      // [n_bias], at most 2^30
    const float * bias;
    const int32_t * bias_start;   // [n_row + 1], clamped to 0..n_bias
    int n_bias;
    // then tokens whose bit is 0 become -infinity: bit t % 32 of word t / 32
    // of mask row mask_row[b] ([n_mask][ceil(n_vocab / 32)]; -1: no mask; any
    // other id outside 0..n_mask-1 permits nothing); mask_row NULL: row b's
    // mask is b, and n_mask at least n_row
    const uint32_t * mask;
    const int32_t * mask_row;     // [n_row]
    int n_mask;
} sml_hip_rules;

// Bytes of the pick's workspace: n_row * ceil(n_vocab / 2048) * 16.
size_t sml_hip_logits_part_bytes(int n_row, int n_vocab);
// Rows of n_vocab logits (stride floats apart, 0: n_vocab) under the rules
// (NULL: none), into out (out_stride floats apart, 0: n_vocab; out may be
// logits with the same stride, or NULL for the pick alone). tok (NULL: no
// pick) receives each row's greedy pick: what sml_hip_argmax's serial loop
// finds among the tokens the mask permits, -1 where it permits none. part is
// the pick's workspace (unused without tok). Ids outside 0..n_vocab-1 are
// passed over. n_row 0..65535, n_vocab 1..2^30.
int sml_hip_logits_adjust(const float * logits, size_t stride, int n_row, int n_vocab, const sml_hip_rules * rules,
                          float * out, size_t out_stride, int32_t * tok, void * part, void * stream);

// ------------------------------------------------------------ adapters
// Low-rank adapters of one projection: adapter i adds
// scale[i] * B_i (A_i x), A_i [rank][n_in] and B_i [n_out][rank] row-major in
// pools of one 16-bit type.
typedef struct {
    const uint16_t * a;           // [n_adapter][rank][n_in], 16-byte aligned
    const uint16_t * b;           // [n_adapter][n_out][rank], 16-byte aligned
    const float * scale;          // [n_adapter], NULL: 1
    const int32_t * ranks;        // [n_adapter] each adapter's own rank (0..rank; what lies past it is
                                  //   not used), NULL: rank
    int n_adapter, rank;          // rank a multiple of 8 up to 256
    int n_in, n_out, type;        // n_in a multiple of 8; type: SML_F16 or SML_BF16
} sml_hip_adapters;

// Floats of the workspace of sml_hip_lora_add: rank * max(n_row, min(32 * n_row, 8192)).
size_t sml_hip_lora_work_floats(int rank, int n_row);
// y[r] = base[r] + scale * B (A x[r]) for n_row rows (0..65535) with adapter
// adapter[r] each; an id outside 0..n_adapter-1 (-1 by custom) adds nothing:
// the row is its base, signs of zeros and NaN included.
// x rows lie x_stride floats apart (0: n_in), y's and base's y_stride (0:
// n_out); base may be y, or NULL for zeros; x and work lie apart from y.
// Products and sums are fp32, their order set by the call's shape: a row's bits
// do not depend on the other rows or on which adapters they have, and an
// infinity or NaN in a row or an adapter reaches only the rows it belongs to.
// It follows sml_hip_gemm, whose output is its base, and takes the unquantized
// input of that product.
int sml_hip_lora_add(const sml_hip_adapters * ad, const float * x, size_t x_stride, int n_row, const int32_t * adapter,
                     const float * base, float * y, size_t y_stride, float * work, void * stream);

#ifdef __cplusplus
}
#endif
