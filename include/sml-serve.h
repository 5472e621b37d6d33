// Operators of a step that serves many requests at once, on device buffers:
// a paged key/value cache and the attention of one new token a sequence over
// it, low-rank adapters beside a shared projection, and penalties, biases and
// grammar masks on logits with the greedy pick. They stand beside the
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
// the sums of weight * |value|, the largest weight 1; an infinite key or value
// that a sequence does attend over makes its KV head's outputs NaN, an infinite
// query its own head's. How the positions are split follows all of the lengths:
// a sequence's sums depend on the others by their rounding alone, and equal
// calls give equal bits.
int sml_hip_paged_attention(const sml_hip_pages * pg, const float * q, size_t q_stride, const int32_t * len,
                            int max_len, int n_head, float scale, float * part, float * out, void * stream);

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
