// Kernels of several rows a sequence over a paged cache, and of that cache's
// upkeep (sml-serve.h): the append with axes, the rows' attention, accepted
// drafts, forks and moved pages.
#include "serve_dev.h"

// ---------------------------------------------------------------- append
//
// The rotation of sml_sv_append with a position for each pair: a thread's four
// pairs look up their axis (in the arguments) and its position, and their angles
// come in one load where the axis is one. Latency bounds 59 rows (3.8 us, 2.7 MB, 32
// heads over 8 of 128), the stream 1369 (6.4 us, 22 MB, 12 heads over 2 of 128 with
// three axes, whose 288 items a row are 512 threads; 6.6 with an angle a load). A row
// as one workgroup of 512 threads was no faster.
template <int D, int BF>
__device__ __forceinline__ void axes_body(const sml_kaxes & a) {
    constexpr int HQ = D / 8;                         // threads of a rotated head
    const int r = blockIdx.x, i = blockIdx.y * blockDim.x + threadIdx.x;
    const int s = a.seq ? a.seq[r] : r, p = a.slot[r];
    if (p < 0 || p >> a.pg.page_shift >= a.pg.seq_pages || s < 0 || s >= a.pg.n_seq) return;
    int pos[AX_MOST];
    #pragma unroll
    for (int x = 0; x < AX_MOST; x++) {
        pos[x] = x < a.n_axis ? a.pos[(size_t) x * a.n_rows + r] : 0;
        if (pos[x] < 0 || pos[x] >= a.n_rope) return;
    }
    const int page = page_of(a.pg, s, p >> a.pg.page_shift);
    if (page < 0) return;
    const int nrot = (a.n_head + a.pg.n_kv) * HQ;
    if (i >= nrot + a.pg.n_kv * (D / 4)) return;
    float * row = a.qkv + (size_t) r * a.stride;
    const size_t at = (size_t) page * a.pg.page_stride +
                      (size_t) (p & ((1 << a.pg.page_shift) - 1)) * (a.pg.n_kv * D);
    if (i >= nrot) {
        const int d = 4 * (i - nrot);
        const v4f x = *(const v4fu *) (row + (size_t) (a.n_head + a.pg.n_kv) * D + d);
        ushort4 w = { to16<BF>(x[0]), to16<BF>(x[1]), to16<BF>(x[2]), to16<BF>(x[3]) };
        *(ushort4 *) (a.pg.v + at + d) = w;
        return;
    }
    const int h = i / HQ, d = 4 * (i % HQ);
    float * x = row + (size_t) h * D + d;
    const v4f lo = *(const v4fu *) x, hi = *(const v4fu *) (x + D / 2);
    v4f y0 = lo, y1 = hi;
    auto of_axis = [&](uint32_t ax) { return (size_t) (ax == 0 ? pos[0] : ax == 1 ? pos[1] : ax == 2 ? pos[2] : pos[3]) * (D / 2) + d; };
    const uint32_t four = a.axis[d / 4];
    if (four == (four & 255u) * 0x01010101u) {
        if ((four & 255u) < (uint32_t) a.n_axis) {
            const size_t o = of_axis(four & 255u);
            const v4f c = *(const v4fu *) (a.cos_t + o), sn = *(const v4fu *) (a.sin_t + o);
            #pragma unroll
            for (int e = 0; e < 4; e++) {
                y0[e] = __builtin_fmaf(lo[e], c[e], -(hi[e] * sn[e]));
                y1[e] = __builtin_fmaf(lo[e], sn[e], hi[e] * c[e]);
            }
        }
    } else {
        #pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t ax = four >> (8 * e) & 255u;
            if (ax < (uint32_t) a.n_axis) {
                const size_t o = of_axis(ax) + e;
                const float c = a.cos_t[o], sn = a.sin_t[o];
                y0[e] = __builtin_fmaf(lo[e], c, -(hi[e] * sn));
                y1[e] = __builtin_fmaf(lo[e], sn, hi[e] * c);
            }
        }
    }
    if (h < a.n_head) {
        float * q = a.q_out ? a.q_out + ((size_t) r * a.n_head + h) * D + d : x;
        *(v4fu *) q = y0;
        *(v4fu *) (q + D / 2) = y1;
        return;
    }
    uint16_t * k = a.pg.k + at + (size_t) (h - a.n_head) * D + d;
    ushort4 w0 = { to16<BF>(y0[0]), to16<BF>(y0[1]), to16<BF>(y0[2]), to16<BF>(y0[3]) };
    ushort4 w1 = { to16<BF>(y1[0]), to16<BF>(y1[1]), to16<BF>(y1[2]), to16<BF>(y1[3]) };
    *(ushort4 *) k = w0;
    *(ushort4 *) (k + D / 2) = w1;
}
#define AXES(D, BF, name) \
    extern "C" __global__ __launch_bounds__(256) void name(const sml_kaxes a) { axes_body<D, BF>(a); }
AXES(128, 0, sml_rw_append)
AXES(128, 1, sml_rw_append_bf)
AXES(64, 0, sml_rw_append_d64)
AXES(64, 1, sml_rw_append_d64_bf)

// ---------------------------------------------------------------- attention
//
// out = sum_t 2^(s_t - m) v_t / sum_t 2^(s_t - m) over the slots a row attends
// to, s_t = log2(e) (cap tanh(scale q.k_t / cap) - slope |distance|), in one pass
// over the cache with a running base m.
//
// The (row, query head) pairs of a sequence and KV head are columns, a row's
// heads side by side. A workgroup of eight or four waves takes a tile of
// 64 or 128 of them and a split of the positions: CW waves of 32 columns side by
// side, and PG such groups that take blocks of 32 positions in turn and are joined
// in LDS at the end.
// The matrix cores take S^T = K Q^T and O^T = V^T P^T in tiles of 32 x 32, columns
// in the columns. With the lane's c = lane % 32, g = lane / 32:
// - K is read from LDS as the first operand: lane (c, g) takes position c's dims
//   16j + 8g..; score e comes back as position 8 (e / 4) + 4g + e % 4 of column c.
// - That is just what the second product takes as P^T if its inner index 8g + i
//   stands for position 4g + i of 16 (i < 4) or 8 + 4g + i - 4: P never crosses
//   lanes.
// - V^T comes by transposing LDS reads (ds_read_b64_tr_b16: 16 lanes read 4 rows
//   of 16 dims and take a dim's 4 rows each) in the same order, and lane (c, g)
//   ends with dims 32u + 8 (e / 4) + 4g + e % 4 of column c: the base's rescaling is
//   a lane's own.
// q and the weights are split into 16-bit parts, as in sml_sv_attend, whose base
// and room these are. K and V go from memory to LDS without registers, a block
// ahead, 16-byte words swizzled by row so that both kinds of read spread over the
// banks; a chunk of the table is a lane's entry each, looked up 1024 positions ahead.
// (An entry is compared with n_pages where it is loaded, so every 1024 positions the
// wave waits for it and for the copies in flight.)
//
// What bounds it: of many rows the matrix cores' rate on real data (2048 rows at
// 16384, 32 heads over 8 of 128: 552 TFLOP/s of the formula, which in fp16's two
// parts is 1104 of the 1217 that a large library product reaches; bf16 436, which
// in three parts is 1308 of 1277). The same columns as 16 x 16 tiles took 10 to 20%
// longer (a matrix instruction keeps the vector unit from issuing for more than
// half of its time, so fewer and larger ones leave it more), 16 columns a wave
// twice the LDS reads. A next block's scores made during this one's softmax,
// with three stages, gained nothing: the two waves of a SIMD do that for each
// other. Neither did a third stage alone (of 128 columns and eight waves, 16 x 26
// rows 45 us for 46, 2047 rows of packed documents in bfloat16 155 for 151) nor a
// wave's priority raised in its products or its softmax. Of few rows the chain of
// latencies bounds it (place, table, rows, products, joining: 8.7 us at 4095
// positions), then the cache's stream.
//
// Masks cost a block only where it is not whole for all of a wave's columns: each
// lane then makes its column's 32 bits of the block, of the range, the tree and
// the pages that are there. What a column does not attend to has no weight, but
// 0 times a NaN or an infinity is none either: rows that no column of the tile
// may see are loaded as zeros, and where columns differ, each wave looks its share
// of the values through on its arrival, puts zeros for those that are not finite
// and notes their positions: a column that attends to one gets NaN in its dim
// (spoiled), as the products leave an infinity or NaN there where columns agree.
//
// Lengths and counts are ragged and on the device: every wave sums them up and
// finds its workgroup's tile and split (rows_place), splits of one size for all
// but cut to what a tile's rows see. Calls with tiles enough are not split, nor
// sequences past AT_SHARED, whose tiles are found by halving.
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

// What no column may see is read from here.
__device__ const __align__(16) uint8_t rw_zeros[16] = { 0 };

// 16 bytes a lane straight into LDS, from an address of its own or from base + off,
// the wave's 64 lanes side by side from dst (a wave-uniform address) on; the caller
// waits (vmcnt) and then meets the other waves before any of the bytes is read.
// Written out because the compiler, which cannot tell the buffers apart, otherwise
// waits for every copy in flight before the next LDS read.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"             // m0 among the clobbers: it is what the statement sets
__device__ __forceinline__ void copy_lds16(const void * src, const void * dst) {
    const uint32_t at = (uint32_t) (uintptr_t) (const __attribute__((address_space(3))) void *) dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(__builtin_amdgcn_readfirstlane(at)), "v"(src) : "m0", "memory");
}
__device__ __forceinline__ void copy_lds16(const void * base, uint32_t off, const void * dst) {
    const uint32_t at = (uint32_t) (uintptr_t) (const __attribute__((address_space(3))) void *) dst;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(__builtin_amdgcn_readfirstlane(at)), "v"(off), "s"(base) : "m0", "memory");
}
#pragma clang diagnostic pop

// col / rep: rep is at most 16 and col below 2^21, so that the high word of a
// product with 2^32 / rep, rounded up, is it.
__device__ __forceinline__ int rows_over(const sml_krows & a, int col) { return a.over ? (int) __umulhi((unsigned) col, a.over) : col; }

struct rows_of { int s0, m, n; };                     // a sequence's first row, its rows and its positions
__device__ __forceinline__ rows_of rows_seq(const sml_krows & a, int b) {
    rows_of x;
    x.s0 = min(max(a.start[b], 0), a.n_row);
    x.m = min(max(a.start[b + 1], x.s0), a.n_row) - x.s0;
    x.n = min(max(a.len[b], 0), a.max_len);
    return x;
}
// The sum of v over the wave's lanes.
__device__ __forceinline__ float wave_total(float v) {
    v += dpp_f<0x111>(v);                             // row_shr 1, 2, 4, 8: lane 15 of a row has its sum
    v += dpp_f<0x112>(v);
    v += dpp_f<0x114>(v);
    v += dpp_f<0x118>(v);
    const int x = __builtin_bit_cast(int, v);
    return (__builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 15)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 31))) +
           (__builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 47)) + __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, 63)));
}
// The least and the largest of the first 32 lanes.
__device__ __forceinline__ int least32(int v) {
    v = min(v, dpp_i<0xB1>(v)); v = min(v, dpp_i<0x4E>(v)); v = min(v, dpp_i<0x141>(v)); v = min(v, dpp_i<0x140>(v));
    return min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
}
__device__ __forceinline__ int most32(int v) {
    v = max(v, dpp_i<0xB1>(v)); v = max(v, dpp_i<0x4E>(v)); v = max(v, dpp_i<0x141>(v)); v = max(v, dpp_i<0x140>(v));
    return max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
}

struct rows_block { int t, pa, pb; uint64_t aa, ab; };  // a step's start, a group's block's two pages and their places in a pool
struct rows_at { int b, tile, count, split, item; rows_of sq; };  // a tile, its splits, this one's number, the first's among all items
// Item i's (or, of TILES, tile i's) place; false past the last. Numbers run through
// the items without a gap, so that workgroups that run at once lie evenly (64
// sequences of up to 8 rows to 2000 in 75 us, 91 with gaps). Of more sequences than
// AT_SHARED, which are not split, b's tiles are numbered from start[b] * rep / cols +
// b on, which leaves each as many numbers as it has tiles, and the number says whose
// it is.
template <bool TILES>
__device__ __forceinline__ bool rows_place(const sml_krows & a, int i, int lane, rows_at & p) {
    const int rep = a.n_head / a.pg.n_kv, cols = a.cols, cl = __builtin_ctz(a.cols);
    const bool turned = !a.first && !a.last;          // causal rows: the last tiles see most, and begin
    if (a.pg.n_seq > AT_SHARED) {
        int lo = 0, hi = a.pg.n_seq;
        while (hi - lo > 1) {
            const int step = (hi - lo + 63) / 64, at = lo + lane * step;
            const bool in = at < hi && (min(max(a.start[at], 0), a.n_row) * rep >> cl) + at <= i;
            const unsigned long long hit = __ballot(in);
            const int k = hit ? 63 - __builtin_clzll(hit) : 0;
            lo += k * step;
            hi = min(hi, lo + step);
        }
        p.sq = rows_seq(a, lo);
        p.b = lo;
        const int e = i - ((p.sq.s0 * rep >> cl) + lo), nt = (p.sq.m * rep + cols - 1) >> cl;
        p.tile = turned ? nt - 1 - e : e;
        p.count = 1;
        p.split = 0;
        p.item = i;
        return e >= 0 && e < nt;
    }
    if (a.pg.n_seq == 1) {
        p.sq = rows_seq(a, 0);
        const int nb = (p.sq.n + RW_BLOCK - 1) / RW_BLOCK, nt = (p.sq.m * rep + cols - 1) >> cl, most = max(a.want / max(nt, 1), 1);
        const int chunk = max(a.least, (nb + most - 1) / most);
        p.b = 0;
        p.count = max((nb + chunk - 1) / chunk, 1);
        p.tile = TILES || p.count == 1 ? i : i / p.count;
        p.split = TILES ? 0 : i - p.tile * p.count;
        p.item = p.tile * p.count;
        if (turned) p.tile = nt - 1 - p.tile;
        return p.item < nt * p.count;
    }
    // The blocks of a split (want 0: all): what makes want of them in all if each
    // tile's came out even, and more until they are no more than that; else a tile's
    // each. How many that makes of a tile's blocks need not be exact, but the same
    // everywhere: a product with the reciprocal, rounded up.
    rows_of x[AT_SHARED / 64];
    int nb[AT_SHARED / 64], nt[AT_SHARED / 64];
    float sum = 0.0f;
    #pragma unroll
    for (int k = 0; k < AT_SHARED / 64; k++)
        if (k == 0 || 64 * k < a.pg.n_seq) {
            x[k] = rows_of{0, 0, 0};
            if (64 * k + lane < a.pg.n_seq) x[k] = rows_seq(a, 64 * k + lane);
            nt[k] = (x[k].m * rep + cols - 1) >> cl;
            nb[k] = (x[k].n + RW_BLOCK - 1) / RW_BLOCK;
            sum += (float) nt[k] * (float) nb[k];
        }
    sum = wave_total(sum);
    int chunk = a.want ? max(a.least, (int) (sum * 1.0001f / (float) a.want) + 1) : 1 << 30;
    float per = __builtin_amdgcn_rcpf((float) chunk);
    auto splits = [&](int blocks) { return max((int) __builtin_ceilf((float) blocks * per), 1); };
    for (int tries = 0; a.want && tries < 8; tries++) {
        float made = 0.0f;
        #pragma unroll
        for (int k = 0; k < AT_SHARED / 64; k++)
            if (k == 0 || 64 * k < a.pg.n_seq) made += (float) (nt[k] * splits(nb[k]));
        made = wave_total(made);
        if (made <= (float) a.want) break;
        chunk = tries < 6 ? chunk + (int) ((float) chunk * (made / (float) a.want - 1.0f)) + 1 : 1 << 30;
        per = __builtin_amdgcn_rcpf((float) chunk);
    }
    p.item = 0;
    #pragma unroll
    for (int k = 0; k < AT_SHARED / 64; k++)
        if (k == 0 || 64 * k < a.pg.n_seq) {
            const int count = splits(nb[k]);
            const int items = wave_scan(nt[k] * count), mine = TILES ? wave_scan(nt[k]) : items;
            const unsigned long long hit = __ballot(mine > i);
            if (hit) {
                const int l = __builtin_ctzll(hit), n = __builtin_amdgcn_readlane(nt[k], l);
                p.b = 64 * k + l;
                p.count = __builtin_amdgcn_readlane(count, l);
                p.sq.s0 = __builtin_amdgcn_readlane(x[k].s0, l);
                p.sq.m = __builtin_amdgcn_readlane(x[k].m, l);
                p.sq.n = __builtin_amdgcn_readlane(x[k].n, l);
                const int e = i - (__builtin_amdgcn_readlane(mine, l) - (TILES ? n : n * p.count));
                p.tile = TILES || p.count == 1 ? e : e / p.count;
                p.split = TILES ? 0 : e - p.tile * p.count;
                p.item += __builtin_amdgcn_readlane(items, l) - n * p.count + p.tile * p.count;
                if (turned) p.tile = n - 1 - p.tile;
                return true;
            }
            i -= __builtin_amdgcn_readlane(mine, 63);
            p.item += __builtin_amdgcn_readlane(items, 63);
        }
    return false;
}
__device__ __forceinline__ int rows_item() { return (int) (blockIdx.z * gridDim.y + blockIdx.y); }
// The sums of an item's columns, and their bases and weights' sums.
__device__ __forceinline__ float * part_o(const sml_krows & a, int kh, int item, int d) {
    return a.part + ((size_t) kh * a.items + item) * a.part_cols * d;
}
__device__ __forceinline__ float2 * part_ml(const sml_krows & a, int kh, int item, int d) {
    return (float2 *) (a.part + (size_t) a.pg.n_kv * a.items * a.part_cols * d) + ((size_t) kh * a.items + item) * a.part_cols;
}

// tanh(y) for |y| up to 0.625: y times a polynomial of y^2, fitted to the relative
// error on that range (1.1e-8 as its coefficients are rounded, 1.1e-7 as evaluated;
// five unrounded ones reach 4.4e-9). Past it 1 - 2 / (e^2y + 1), whose cancellation
// costs less than a bit there. (The Cephes library's tanhf has the same two ranges.)
__device__ __forceinline__ float tanh_small(float y) {
    const float z = y * y;
    float p = __builtin_fmaf(-0.0056599886f, z, 0.020590989f);
    p = __builtin_fmaf(p, z, -0.053721067f);
    p = __builtin_fmaf(p, z, 0.13331127f);
    p = __builtin_fmaf(p, z, -0.33333260f);
    return y * __builtin_fmaf(p, z, 1.0f);
}
__device__ __forceinline__ float tanh_any(float y) {
    const float e = __builtin_amdgcn_exp2f(y * 2.88539008177792681f);
    const float t = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(e + 1.0f), 1.0f);
    return fabsf(y) > 0.625f ? t : tanh_small(y);
}

// The parts of two weights, as parts_of makes them; fp16's remainders are a mixed
// instruction each if the compiler does not know that m1 is -1.
template <int BF>
__device__ __forceinline__ void weights_of(float x, float y, float m1, typename Mx<BF>::v8 (&p)[Mx<BF>::parts], int e) {
    if constexpr (BF) parts_of<BF>(x, y, p, e);
    else {
        typedef _Float16 v2h __attribute__((ext_vector_type(2)));
        typedef float v2f __attribute__((ext_vector_type(2)));
        const v2h h = __builtin_convertvector(v2f{x, y}, v2h);
        const v2h l = __builtin_convertvector(v2f{__builtin_fmaf((float) h[0], m1, x), __builtin_fmaf((float) h[1], m1, y)}, v2h);
        p[0][e] = h[0];
        p[0][e + 1] = h[1];
        p[1][e] = l[0];
        p[1][e + 1] = l[1];
    }
}

// Bits lo..hi-1 of 32.
__device__ __forceinline__ uint32_t bits_range(int lo, int hi) {
    lo = min(max(lo, 0), 32);
    hi = min(max(hi, 0), 32);
    return lo < hi ? (~0u >> (32 - (hi - lo))) << lo : 0;
}

// A form of the rows' attention: CW waves of 32 columns beside each other, PG
// groups of them; two stages of 32 positions a group, where the groups' joined
// sums end, and the dims that are no longer finite, behind both.
template <int D, int CW, int PG> struct RowsForm {
    static constexpr int stages = PG * 2 * 4 * 32 * D;
    static constexpr int joined = PG * 32 * CW * (D + 4) * 4;
    static constexpr int filled = stages + PG * 2 * 4 * (32 + CW + D) + (16 + 20 * 32 + 4 * 32 * PG) * CW, joining = joined + PG * 32 * CW * 8;
    static constexpr int spoiled = filled > joining ? filled : joining;
};

template <int BF> struct Mx32;
template <> struct Mx32<0> {
    static __device__ __forceinline__ v16f mul(Mx<0>::v8 a, Mx<0>::v8 b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mx32<1> {
    static __device__ __forceinline__ v16f mul(Mx<1>::v8 a, Mx<1>::v8 b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};

// CW waves side by side take 32 CW columns; PG such groups take the blocks of a
// split in turn and are joined in LDS at the end.
template <int D, int BF, int CW, int PG, bool RULES>
__device__ __forceinline__ void rows_body(const sml_krows & a) {
    using M = Mx<BF>;
    using MM = Mx32<BF>;
    typedef typename M::v8 v8;
    using F = RowsForm<D, CW, PG>;
    constexpr int NJ = D / 16, E = D / 32, NP = M::parts, RB = 2 * D, W = CW * PG, KB = 32, POOL = KB * RB, STAGE = 2 * POOL;
    constexpr int RC = 1024 / RB, NC = KB / RC / CW;  // rows of a copy, a wave's copies of a block's keys
    static_assert(NC >= 1 && RC <= 16, "");
    extern __shared__ __align__(16) uint8_t lds[];    // the groups' stages; their new rows' positions, positions whose V is not finite, ranges
    const int kh = blockIdx.x, tid = threadIdx.x, lane = tid & 63, c = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), pgi = wave % PG, cw = wave / PG;
    uint8_t * const stages = lds + pgi * 2 * STAGE;
    int * const kpos = (int *) (lds + F::stages) + pgi * 2 * KB;
    uint32_t * const found = (uint32_t *) (lds + F::stages + 4 * PG * 2 * KB) + pgi * 2 * CW;
    int * const red = (int *) (lds + F::stages + 4 * PG * 2 * (KB + CW));
    int4 * const about = (int4 *) (red + 4 * CW);     // of the columns, for the masks: range, tree's bits
    int * const owner = (int *) (about + 32 * CW);    // and their rows, -1 for those that attend to nothing
    uint8_t * const dims = (uint8_t *) (owner + 32 * CW) + pgi * 2 * KB * (D / 8);   // those of the positions found, a bit each
    uint32_t * const hits = (uint32_t *) ((uint8_t *) (owner + 32 * CW) + PG * 2 * KB * (D / 8)) + 32 * wave;   // which of them a column attends to
    uint32_t * const spoiled = (uint32_t *) (lds + F::spoiled);   // [column][E] and of the columns that attend to them
    rows_at p;
    if (!rows_place<false>(a, rows_item(), lane, p)) return;
    const rows_of sq = p.sq;
    const int rep = a.n_head / a.pg.n_kv, ncol = sq.m * rep, past = sq.n - sq.m, kvd = a.pg.n_kv * D;
    const int sh = a.pg.page_shift, pmask = (1 << sh) - 1;
    const int32_t * const tab = a.pg.table + (size_t) p.b * a.pg.seq_pages;

    // the lane's column: its row's range, its tree's bits (if they are no more than 64) and its position
    const int col0 = p.tile * a.cols, col = col0 + 32 * cw + c, in_seq = rows_over(a, min(col, ncol - 1));
    const bool mine = col < ncol;
    const int r = sq.s0 + in_seq, h = kh * rep + (min(col, ncol - 1) - in_seq * rep);
    const int lo = a.first ? max(a.first[r], 0) : 0;
    const int hi = max(min(a.last ? a.last[r] : a.tree ? past : past + in_seq + 1, sq.n), 0);
    const int nbit = a.tree ? min(sq.m, 32 * a.words) : 0;
    uint64_t tw = 0;
    if (nbit) {
        const uint32_t * const bits = a.tree + (size_t) r * a.words;
        tw = bits[0];
        if (a.words > 1) tw |= (uint64_t) bits[1] << 32;
    }
    const bool range = lo < hi;
    // what any column of the wave, of the tile attends to lies in w_lo..w_hi, t_lo..t_hi;
    // every one that attends to anything has all of f_lo..f_hi (t_flo.. of the tile)
    int w_lo = 0x7fffffff, w_hi = 0, f_lo = 0, f_hi = 0x7fffffff, t_lo, t_hi, t_flo, t_fhi;
    const bool any = col0 + 32 * cw < ncol;
    if (!a.first && !a.last && past >= 0) {
        // no loads to wait for: a tree's rows all see the past, causal ones more from row to row
        if (a.tree) {
            t_lo = 0;
            t_hi = past + nbit;
            t_flo = past > 0 ? 0 : 0x7fffffff;
            t_fhi = past;
        } else {
            t_lo = t_flo = 0;
            t_hi = past + rows_over(a, min(col0 + a.cols, ncol) - 1) + 1;
            t_fhi = past + rows_over(a, col0) + 1;
        }
        if (any) {
            w_lo = 0;
            w_hi = a.tree ? t_hi : __builtin_amdgcn_readlane(hi, 31);
            f_lo = t_flo;
            f_hi = a.tree ? t_fhi : __builtin_amdgcn_readlane(hi, 0);
        }
    } else {
        const bool tree = nbit && (tw || a.words > 2);
        if (mine && range) { w_lo = lo; w_hi = hi; }
        if (mine && tree && past + nbit > 0) { w_lo = min(w_lo, max(past, 0)); w_hi = max(w_hi, min(past + nbit, sq.n)); }
        if (mine && (range || tree)) { f_lo = range ? lo : 0x7fffffff; f_hi = range ? hi : 0; }
        t_lo = w_lo = least32(w_lo);
        t_hi = w_hi = most32(w_hi);
        t_flo = f_lo = most32(f_lo);
        t_fhi = f_hi = least32(f_hi);
        if (!lane && !pgi) { red[4 * cw] = w_lo; red[4 * cw + 1] = w_hi; red[4 * cw + 2] = f_lo; red[4 * cw + 3] = f_hi; }
        __syncthreads();
        #pragma unroll
        for (int w = 0; w < CW; w++) {
            t_lo = min(t_lo, red[4 * w]);
            t_hi = max(t_hi, red[4 * w + 1]);
            t_flo = max(t_flo, red[4 * w + 2]);
            t_fhi = min(t_fhi, red[4 * w + 3]);
        }
        t_lo = __builtin_amdgcn_readfirstlane(t_lo);
        t_hi = __builtin_amdgcn_readfirstlane(t_hi);
        t_flo = __builtin_amdgcn_readfirstlane(t_flo);
        t_fhi = __builtin_amdgcn_readfirstlane(t_fhi);
    }
    // this split's blocks
    int t_at = 0, t_end = 0;
    if (t_lo < t_hi) {
        const int b0 = t_lo / RW_BLOCK, nb = (t_hi + RW_BLOCK - 1) / RW_BLOCK - b0, per = p.count == 1 ? nb : (nb + p.count - 1) / p.count;
        t_at = (b0 + p.split * per) * RW_BLOCK;
        t_end = min((b0 + min(nb, (p.split + 1) * per)) * RW_BLOCK, t_hi);
    }

    // Pages of 64 times 16 positions from t_tab on, one a lane (negative: none), and
    // of as many behind; where in a pool the first of the 16 lies, in bytes.
    auto look = [&](int t) {
        t += 16 * lane;
        const int e = t < t_end ? tab[t >> sh] : -1;
        return e < a.pg.n_pages ? e : -1;
    };
    int t_tab = t_at, ent = look(t_at), next = look(t_at + 1024);
    // the query: lane (c, g) holds dims 16j + 8g.. of column c
    v4f x[2 * NJ];
    {
        const float * qp = a.q + (size_t) r * a.q_stride + (size_t) h * D + 8 * g;
        #pragma unroll
        for (int j = 0; j < 2 * NJ; j++) x[j] = *(const v4fu *) (qp + 16 * (j / 2) + 4 * (j % 2));
    }
    const int qpos = RULES && a.pos ? a.pos[r] : past + in_seq;
    uint64_t at_ent;
    auto place = [&]() { at_ent = 2 * ((uint64_t) max(ent, 0) * a.pg.page_stride + (uint64_t) (uint32_t) (((t_tab + 16 * lane) & pmask) * kvd + kh * D)); };
    place();
    // the next step (a block of each group) at or after t with a page
    constexpr int STEP = PG * KB;
    auto seek = [&](int t) {
        while (t < t_end) {
            if (t - t_tab >= 1024) {
                t_tab += 1024;
                ent = next;
                next = look(t_tab + 1024);
                place();
                continue;
            }
            if (__ballot(ent >= 0) >> ((t - t_tab) >> 4) & ((1ull << (STEP / 16)) - 1)) break;
            t += STEP;
        }
        return t;
    };
    // a group's block of the step at t: the pages of its two halves, and where these lie
    auto locate = [&](int t) {
        rows_block x = { t, -1, -1, 0, 0 };
        if (t < t_end) {
            const int i = ((t - t_tab) >> 4) + 2 * pgi;
            x.pa = __builtin_amdgcn_readlane(ent, i);
            x.pb = __builtin_amdgcn_readlane(ent, i + 1);
            x.aa = (uint64_t) (uint32_t) __builtin_amdgcn_readlane((int) (at_ent >> 32), i) << 32 | (uint32_t) __builtin_amdgcn_readlane((int) at_ent, i);
            x.ab = (uint64_t) (uint32_t) __builtin_amdgcn_readlane((int) (at_ent >> 32), i + 1) << 32 | (uint32_t) __builtin_amdgcn_readlane((int) at_ent, i + 1);
        }
        return x;
    };
    // A lane of a copy: its row and its word there; word w of row x lies at w ^ swz(x).
    // (A row's words fill its bytes to the power of two, so that another copy's
    // swizzle is an exclusive or of the offset.)
    auto swz_k = [](int x) { return D == 128 ? x & 15 : (x >> 1) & 7; };
    auto swz_v = [](int x) { return D == 128 ? 2 * (x & 7) : (x >> 1) & 7; };
    const int crow = RC * cw + lane / (RB / 16), cword = lane % (RB / 16);
    const uint32_t koff = 2u * (uint32_t) ((crow & 15) * kvd + 8 * (cword ^ swz_k(crow)));
    const uint32_t voff = 2u * (uint32_t) ((crow & 15) * kvd + 8 * (cword ^ swz_v(crow)));
    auto fetch = [&](uint8_t * st, bool values, const rows_block & x) {
        const int from = x.t + pgi * KB;
        const uint8_t * const pool = (const uint8_t *) (values ? a.pg.v : a.pg.k);
        if (x.pa >= 0 && x.pb >= 0 && from >= t_lo && from + KB <= t_hi) {
            #pragma unroll
            for (int e = 0; e < NC; e++) {
                const int row0 = RC * (CW * e + cw), turn = 16 * (values ? swz_v(RC * CW * e) : swz_k(RC * CW * e));
                copy_lds16(pool + (row0 < 16 ? x.aa : x.ab) + (uint32_t) (2 * ((RC * CW * e) & 15) * kvd), (values ? voff : koff) ^ turn, st + row0 * RB);
            }
        } else {
            #pragma unroll 1
            for (int e = 0; e < NC; e++) {
                const int row0 = RC * (CW * e + cw), row = RC * CW * e + crow, pos = from + row;
                const bool in = (row0 < 16 ? x.pa : x.pb) >= 0 && pos >= t_lo && pos < t_hi;
                const uint8_t * at = pool + (row0 < 16 ? x.aa : x.ab) + 2u * (uint32_t) ((row & 15) * kvd + 8 * (cword ^ (values ? swz_v(row) : swz_k(row))));
                copy_lds16(in ? (const void *) at : (const void *) rw_zeros, st + row0 * RB);
            }
        }
    };
    // The positions of a block's new rows; they are in LDS with the block. (Chosen from
    // as they are loaded: the wave waits for them, behind the copies that it has begun.)
    int at_pos = 0;
    auto fetch_pos = [&](int t) {
        if (RULES && a.slope && a.pos && t + pgi * KB + KB > past && cw == 0)
        {
            const int slot = t + pgi * KB + lane, i = min(max(slot - past, 0), max(sq.m - 1, 0));
            at_pos = a.pos[sq.s0 + i];
            if (slot < past) at_pos = slot;
        }
    };
    auto keep_pos = [&](int * kp) {
        if (RULES && a.slope && a.pos && cw == 0 && lane < KB) kp[lane] = at_pos;
    };
    rows_block b0 = locate(seek(t_at));
    if (b0.t < t_end) {
        fetch(stages, false, b0);
        fetch(stages + POOL, true, b0);
        fetch_pos(b0.t);
    }

    const bool some = mine && (range || (nbit && (tw || a.words > 2)));      // does it attend to anything
    if (!pgi && !g) {
        about[32 * cw + c] = some ? make_int4(lo, hi, (int) (uint32_t) tw, (int) (uint32_t) (tw >> 32)) : make_int4(0, 0, 0, 0);
        owner[32 * cw + c] = some ? r : -1;
    }
    for (int x = tid; x < 32 * CW * E; x += 64 * W) spoiled[x] = 0;
    // the query in parts
    v8 q[NJ][NP];
    float back;                                       // what a product of the scaled q is multiplied by
    int ex;
    {
        float mx = 0.0f;
        #pragma unroll
        for (int j = 0; j < 2 * NJ; j++)
            #pragma unroll
            for (int k = 0; k < 4; k++) mx = fmaxf(mx, fabsf(x[j][k]));
        if (a.sign < 0.0f) {
            #pragma unroll
            for (int j = 0; j < 2 * NJ; j++) x[j] = -x[j];
        }
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        ex = BF ? 0 : scale_of(mx);
        #pragma unroll
        for (int j = 0; j < NJ; j++)
            #pragma unroll
            for (int e = 0; e < 8; e += 2)
                parts_of<BF>(__builtin_amdgcn_ldexpf(x[2 * j + e / 4][e % 4], -ex), __builtin_amdgcn_ldexpf(x[2 * j + e / 4][e % 4 + 1], -ex), q[j], e);
        back = __builtin_amdgcn_ldexpf(a.scale, ex);
    }
    // Over the cap, the factor may leave fp32's room where scores or the cap do not.
    // Below 2^-110 (products are below 2^34) a tanh is its argument, also one 2^60 as
    // large: the cap gives these up. Past the largest, scores are 0 or the cap.
    float cap = a.cap;
    if (RULES && !BF && a.cap > 0.0f) {
        const bool far = back < 0x1p-110f;
        back = fminf(far ? __builtin_amdgcn_ldexpf(a.scale, ex + 60) : back, 0x1.fffffep127f);
        cap = far ? __builtin_amdgcn_ldexpf(cap, -60) : cap;
    }
    const int q0 = qpos - 4 * g;                      // the row's position, less where the lane's first score is
    const float slope = RULES && a.slope ? -1.44269504088896341f * a.slope[h] : 0.0f;
    // log2 weights are f times the settled scores. Masked ones are -infinity, of which
    // 0 would make NaN: a factor that fp32 does not hold (a row of q below 2^-137, or
    // a scale as small) becomes its least, and scores stay below 2^-115.
    const float f = RULES ? 1.0f : fmaxf(back, 0x1p-149f);

    v16f o[E];
    #pragma unroll
    for (int u = 0; u < E; u++)
        #pragma unroll
        for (int e = 0; e < 16; e++) o[u][e] = 0.0f;
    float base = -INFINITY, l = 0.0f;

    const int krow = c * RB, kx = swz_k(c);
    // the V row that this lane reads for its 16, and its eight bytes there
    const int vrow = 4 * g + ((lane & 15) >> 2), q16 = (lane >> 4) & 1;
    const int vx = D == 128 ? vrow : g, vat = POOL + vrow * RB + (D == 128 ? 8 * (lane & 3) : 16 * (((lane >> 1) & 1) ^ ((lane >> 3) & 1)) + 8 * (lane & 1));
    // Values that are not finite among those that this wave has fetched, where columns
    // differ: zeros in their place; their positions in the block and, a byte a lane, dims.
    auto screen = [&](uint8_t * st, uint8_t * of) {
        uint32_t bad = 0;
        #pragma unroll 1
        for (int e = 0; e < NC; e++) {
            const int row0 = RC * (CW * e + cw);
            v4u * const at = (v4u *) (st + POOL + row0 * RB + 16 * lane);
            v4u x = *at;
            auto ones = [&](int k) {                  // an exponent of all ones carries into the top bit
                return BF ? ((x[k] & 0x7F807F80u) + 0x00800080u) & 0x80008000u : ((x[k] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
            };
            const uint64_t hit = __ballot((ones(0) | ones(1) | ones(2) | ones(3)) != 0);
            if (hit) {
                int ln = lane;                        // so that no register is kept for what follows from it
                asm volatile("" : "+v"(ln));
                const int row = row0 + ln / (RB / 16);
                uint32_t mark = 0;
                #pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t up = ones(k);
                    x[k] &= ~((up >> 15) * 0xFFFFu);
                    mark |= (up >> 15 & 1u | up >> 30) << (2 * k);
                }
                *at = x;
                of[row * (D / 8) + (ln % (RB / 16) ^ swz_v(row))] = (uint8_t) mark;
                #pragma unroll 1
                for (int k = 0; k < RC; k++)
                    if (hit >> (64 / RC * k) & ((1ull << (64 / RC)) - 1)) bad |= 1u << (row0 + k);
            }
        }
        return bad;
    };

    float m1;
    asm("v_mov_b32 %0, -1.0" : "=v"(m1));
    // The scores, their keys NK ahead; a tile's dims of 16 positions' values; the sums.
    // (bfloat16's three parts leave few registers.)
    constexpr int NK = BF ? 4 : NJ, NV = BF ? 2 : E;
    auto products = [&](const uint8_t * st) {
        auto key = [&](int e) { return *(const v8 *) (st + krow + 16 * ((2 * e + g) ^ kx)); };
        v8 ka[NK];
        #pragma unroll
        for (int e = 0; e < NK; e++) ka[e] = key(e);
        __builtin_amdgcn_sched_barrier(0);
        v16f s;
        #pragma unroll
        for (int e = 0; e < 16; e++) s[e] = 0.0f;
        #pragma unroll
        for (int e = 0; e < NJ; e++) {
            #pragma unroll
            for (int k = 0; k < NP; k++) s = MM::mul(ka[e % NK], q[e][k], s);
            if (e + NK < NJ) ka[e % NK] = key(e + NK);
            if (NK < NJ) __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        return s;
    };
    auto value = [&](const uint8_t * st, int u, int k) {
        typedef __attribute__((address_space(3))) v4s lv4s;
        const uint8_t * const vr = st + vat + 16 * k * RB;
        const v4s x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s *) (vr + (((2 * u + q16) ^ vx) << 5)));
        const v4s x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s *) (vr + 8 * RB + (((2 * u + q16) ^ (D == 128 ? vx : vx | 2)) << 5)));
        return __builtin_bit_cast(v8, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto sums = [&](const v8 & vv, int u, const v8 (&w)[NP]) {
        #pragma unroll
        for (int y = 0; y < NP; y++) o[u] = MM::mul(vv, w[y], o[u]);
    };
    // The dims of the positions found in a block marked for the columns that attend to them.
    auto spoil = [&](const uint8_t * of, uint32_t bad) {
        int ln = lane;                                // so that no register is kept for what follows from it
        asm volatile("" : "+v"(ln));
        const uint32_t hit = hits[ln & 31];
        #pragma unroll 1
        for (; bad; bad &= bad - 1) {
            const int y = __builtin_ctz(bad);
            if (hit >> y & 1)
                #pragma unroll 1
                for (int u = ln >> 5; u < E; u += 2) atomicOr(&spoiled[(32 * cw + (ln & 31)) * E + u], ((const uint32_t *) of)[y * E + u]);
        }
    };
    // Scores of positions t.., whose pages are pa and pb, under the rules and the
    // masks; the base that their weights have. Score e is position at(e) + 4g.
    auto at = [](int e) { return 8 * (e >> 2) + (e & 3); };
    auto settle = [&](v16f & s, const int * kp, int t, int pa, int pb, uint32_t bad) {
        if constexpr (RULES) {
            float top = 0.0f;
            #pragma unroll
            for (int e = 0; e < 16; e++) { s[e] *= back; top = fmaxf(top, fabsf(s[e])); }
            if (a.cap > 0.0f) {
                if (__any(!(top <= 0.625f))) {
                    #pragma unroll
                    for (int e = 0; e < 16; e++) s[e] = cap * tanh_any(s[e]);
                } else {
                    #pragma unroll
                    for (int e = 0; e < 16; e++) s[e] = cap * tanh_small(s[e]);
                }
            }
            if (a.slope) {
                const float d0 = (float) (t - q0);
                if (a.pos && t + 32 > past) {
                    const int4 * const at4 = (const int4 *) kp + g;
                    #pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int4 y = at4[2 * k];
                        const int x4[4] = { y.x, y.y, y.z, y.w };
                        #pragma unroll
                        for (int e = 0; e < 4; e++) s[4 * k + e] = __builtin_fmaf(slope, fabsf((float) (x4[e] - 4 * g - q0)), s[4 * k + e]);
                    }
                } else {
                    #pragma unroll
                    for (int e = 0; e < 16; e++) s[e] = __builtin_fmaf(slope, fabsf(d0 + (float) at(e)), s[e]);
                }
            }
        }
        if (pa < 0 || pb < 0 || t < f_lo || t + 32 > f_hi) {
            const int4 mask = about[32 * cw + c];
            uint32_t vm = bits_range(mask.x - t, mask.y - t);
            const int j0 = t - past;
            if (nbit && j0 + 32 > 0 && j0 < nbit) {
                uint64_t y = (uint64_t) (uint32_t) mask.w << 32 | (uint32_t) mask.z;
                const int w0 = j0 >> 5;               // bits 32 w0.. of the row, 64 of them
                if (a.words > 2) {
                    const int row = owner[32 * cw + c];   // the bits' load waits for the copies in flight, too
                    const uint32_t * const bits = a.tree + (size_t) max(row, 0) * a.words;
                    y = (uint64_t) (w0 + 1 >= 0 && w0 + 1 < a.words ? bits[w0 + 1] : 0u) << 32 | (w0 >= 0 && w0 < a.words ? bits[w0] : 0u);
                    if (row < 0) y = 0;
                } else if (w0) {
                    y = w0 == -1 ? y << 32 : w0 == 1 ? y >> 32 : 0;
                }
                vm |= (uint32_t) (y >> (j0 & 31)) & bits_range(-j0, nbit - j0);
            }
            vm &= bits_range(0, sq.n - t);
            if (pa < 0) vm &= 0xFFFF0000u;
            if (pb < 0) vm &= 0x0000FFFFu;
            if (bad) hits[c] = vm;
            vm >>= 4 * g;
            #pragma unroll
            for (int e = 0; e < 16; e++) s[e] = (vm >> at(e)) & 1 ? s[e] : -INFINITY;
        } else if (bad) {
            hits[c] = some ? ~0u : 0u;
        }
        float mx = -INFINITY;
        #pragma unroll
        for (int e = 0; e < 16; e++) mx = fmaxf(mx, s[e]);
        mx *= f;
        if (__any(mx > base + M::room)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float to = mx > base + M::room ? mx + M::lift : base;
            const float al = __builtin_amdgcn_exp2f(base - (to == -INFINITY ? 0.0f : to));
            l *= al;
            #pragma unroll
            for (int u = 0; u < E; u++)
                #pragma unroll
                for (int e = 0; e < 16; e++) o[u][e] *= al;
            base = to;
        }
    };
    auto weights = [&](const v16f & s, v8 (&w)[2][NP]) {
        const float bu = base == -INFINITY ? 0.0f : base;
        #pragma unroll
        for (int e = 0; e < 16; e += 2) {
            const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], f, -bu)), w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e + 1], f, -bu));
            l += w0;
            l += w1;
            weights_of<BF>(w0, w1, m1, w[e >> 3], e & 7);
        }
    };
    rows_block b1 = locate(seek(b0.t + STEP));        // the next block; b2: the one behind it
    // Two stages, one in use and one that is filled.
    int i0 = 0;
    while (b0.t < t_end) {
        const int cur = b0.t + pgi * KB;
        uint8_t * const st = stages + i0 * STAGE;
        const bool differ = cur < t_flo || cur + KB > t_fhi;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        keep_pos(kpos + i0 * KB);
        if (differ) {
            const uint32_t bad = screen(st, dims + i0 * KB * (D / 8));
            if (!lane) found[i0 * CW + cw] = bad;
        }
        __syncthreads();                          // the block is whole, and nobody reads the last one
        if (b1.t < t_end) {
            fetch(stages + (i0 ^ 1) * STAGE, false, b1);
            fetch(stages + (i0 ^ 1) * STAGE + POOL, true, b1);
            fetch_pos(b1.t);
        }
        const rows_block b2 = b1.t < t_end ? locate(seek(b1.t + STEP)) : b1;
        if (cur < t_end && cur < w_hi && cur + KB > w_lo) {
            v16f s = products(st);
            v8 w[2][NP], vv[NV];
            #pragma unroll
            for (int u = 0; u < NV; u++) vv[u] = value(st, u % E, u / E);
            __builtin_amdgcn_sched_barrier(0);
            uint32_t bad = 0;
            if (differ) {
                #pragma unroll
                for (int y = 0; y < CW; y++) bad |= found[i0 * CW + y];
                bad = (uint32_t) __builtin_amdgcn_readfirstlane((int) bad);
            }
            settle(s, kpos + i0 * KB, cur, b0.pa, b0.pb, bad);
            weights(s, w);
            #pragma unroll
            for (int u = 0; u < 2 * E; u++) {
                sums(vv[u % NV], u % E, w[u / E]);
                if (u + NV < 2 * E) vv[u % NV] = value(st, (u + NV) % E, (u + NV) / E);
                if (NV < E) __builtin_amdgcn_sched_barrier(0);
            }
            if (bad) spoil(dims + i0 * KB * (D / 8), bad);
        }
        b0 = b1;
        b1 = b2;
        i0 ^= 1;
    }

    l += __shfl_xor(l, 32);
    if (!some) { base = -INFINITY; l = 0.0f; }
    // The groups joined: their sums over the stages, rows of D + 4 floats on
    // different banks, their bases and weights' sums behind.
    constexpr int QT = 32 * CW, LD = D + 4;
    float * const so = (float *) lds;
    float2 * const sml = (float2 *) (lds + F::joined);
    __syncthreads();                                  // all are done with the stages
    {
        const int pc = 32 * cw + c;
        float * const to = so + (size_t) (pgi * QT + pc) * LD + 4 * g;
        #pragma unroll
        for (int u = 0; u < E; u++)
            #pragma unroll
            for (int k = 0; k < 4; k++) *(v4f *) (to + 32 * u + 8 * k) = v4f{o[u][4 * k], o[u][4 * k + 1], o[u][4 * k + 2], o[u][4 * k + 3]};
        if (!g) sml[pgi * QT + pc] = make_float2(base, l);
    }
    __syncthreads();
    #pragma unroll 1
    for (int x = tid; x < QT * (D / 4); x += 64 * W) {
        const int pc = x / (D / 4), d = 4 * (x % (D / 4)), col = col0 + pc;
        if (col >= ncol) break;
        float2 ml[PG];
        v4f v[PG];
        #pragma unroll
        for (int k = 0; k < PG; k++) { ml[k] = sml[k * QT + pc]; v[k] = *(const v4f *) (so + (size_t) (k * QT + pc) * LD + d); }
        float m = ml[0].x;
        #pragma unroll
        for (int k = 1; k < PG; k++) m = fmaxf(m, ml[k].x);
        const float mu = m == -INFINITY ? 0.0f : m;
        float ls = 0.0f;
        v4f os = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        #pragma unroll
        for (int k = 0; k < PG; k++) {
            const bool none = ml[k].x == -INFINITY && ml[k].y == 0.0f;    // what its sums hold counts for nothing
            const float f = __builtin_amdgcn_exp2f(ml[k].x - mu);
            ls += none ? 0.0f : f * ml[k].y;
            #pragma unroll
            for (int e = 0; e < 4; e++) os[e] = none ? os[e] : __builtin_fmaf(f, v[k][e], os[e]);
        }
        const uint32_t dims = spoiled[pc * E + d / 32] >> (d & 31);
        #pragma unroll
        for (int e = 0; e < 4; e++) os[e] = dims >> e & 1 ? NAN : os[e];
        if (p.count == 1) {
            const int i = rows_over(a, col);
            #pragma unroll
            for (int e = 0; e < 4; e++) os[e] = ls != 0.0f ? os[e] / ls : 0.0f;
            *(v4fu *) (a.out + ((size_t) (sq.s0 + i) * a.n_head + kh * rep + (col - i * rep)) * D + d) = os;
        } else {
            if (!d) part_ml(a, kh, p.item + p.split, D)[pc] = make_float2(m, ls);
            *(v4f *) (part_o(a, kh, p.item + p.split, D) + (size_t) pc * D + d) = os;
        }
    }
}
// Two waves a SIMD: at three or four, heads of 64 spill (509 rows at 2040 30.7 us
// so, 37.5 with two workgroups a CU).
#define ROWS(D, BF, CW, PG, name, sfx) \
    extern "C" __global__ __launch_bounds__(64 * CW * PG, 2) void name##sfx(const sml_krows a) { rows_body<D, BF, CW, PG, false>(a); } \
    extern "C" __global__ __launch_bounds__(64 * CW * PG, 2) void name##r##sfx(const sml_krows a) { rows_body<D, BF, CW, PG, true>(a); }
#define ROWS4(CW, PG, name) \
    ROWS(128, 0, CW, PG, name, ) \
    ROWS(128, 1, CW, PG, name, _bf) \
    ROWS(64, 0, CW, PG, name, _d64) \
    ROWS(64, 1, CW, PG, name, _d64_bf)
ROWS4(2, 4, sml_rw_rows64)
ROWS4(4, 2, sml_rw_rows128)
ROWS4(2, 2, sml_rw_rows64h)
ROWS4(4, 1, sml_rw_rows128h)

// The splits of a tile joined, C columns a workgroup: the bases of a column's splits
// shared out over its 256 / C lanes, then the splits over each 16 of them, which
// take a few dims each. Latency bounds it.
template <int D, int C>
__device__ __forceinline__ void rows_merge_body(const sml_krows & a) {
    constexpr int LC = 256 / C, SG = LC / 16;         // a column's lanes, and how many splits they take at once
    __shared__ float f[C][RW_SPLITS + 1];
    const int kh = blockIdx.x, tid = threadIdx.x, lane = tid & 63, c = tid / LC, lc = tid % LC, l = tid & 15, share = lc / 16;
    const int groups = a.cols / C, unit = rows_item();
    rows_at p;
    if (!rows_place<true>(a, unit / groups, lane, p) || p.count == 1) return;
    const int rep = a.n_head / a.pg.n_kv, pc = C * (unit % groups) + c, col = p.tile * a.cols + pc;
    if (p.item + p.count > a.items || p.count > RW_SPLITS) return;
    if (p.tile * a.cols + pc - c >= p.sq.m * rep) return;
    const bool mine = col < p.sq.m * rep;
    const float2 * ml = part_ml(a, kh, p.item, D) + (mine ? pc : 0);
    const float * po = part_o(a, kh, p.item, D) + (size_t) (mine ? pc : 0) * D + 4 * l;
    const size_t step = (size_t) a.part_cols;
    float m = -INFINITY;
    for (int s = lc; s < p.count; s += LC) m = fmaxf(m, ml[s * step].x);
    m = LC == 64 ? wave_max(m) : max16(m);
    const float mu = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
    for (int s = lc; s < p.count; s += LC) {
        const float2 y = ml[s * step];
        const float e = __builtin_amdgcn_exp2f(y.x - mu);
        const bool none = y.x == -INFINITY && y.y == 0.0f;    // what lies there counts for nothing
        f[c][s] = none ? -1.0f : e;
        if (!none) sum += e * y.y;
    }
    sum = LC == 64 ? wave_sum(sum) : sum16(sum);
    wave_lds();
    v4f o[D / 64];
    #pragma unroll
    for (int u = 0; u < D / 64; u++) o[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    #pragma unroll 8
    for (int s = share; s < p.count; s += SG) {
        const float e = f[c][s];
        #pragma unroll
        for (int u = 0; u < D / 64; u++) {
            const v4f y = *(const v4f *) (po + s * step * D + 64 * u);
            #pragma unroll
            for (int k = 0; k < 4; k++) o[u][k] = e >= 0.0f || e != e ? __builtin_fmaf(e, y[k], o[u][k]) : o[u][k];
        }
    }
    if constexpr (SG > 1) {
        #pragma unroll
        for (int u = 0; u < D / 64; u++)
            #pragma unroll
            for (int k = 0; k < 4; k++) {
                o[u][k] += __shfl_xor(o[u][k], 16);
                o[u][k] += __shfl_xor(o[u][k], 32);
            }
    }
    if (share || !mine) return;
    const int i = rows_over(a, col);
    float * const to = a.out + ((size_t) (p.sq.s0 + i) * a.n_head + kh * rep + (col - i * rep)) * D + 4 * l;
    #pragma unroll
    for (int u = 0; u < D / 64; u++) {
        v4f y;
        #pragma unroll
        for (int k = 0; k < 4; k++) y[k] = sum == 0.0f ? 0.0f : o[u][k] / sum;
        *(v4fu *) (to + 64 * u) = y;
    }
}
#define MERGE(D, C, name) \
    extern "C" __global__ __launch_bounds__(256) void name(const sml_krows a) { rows_merge_body<D, C>(a); }
MERGE(128, 4, sml_rw_merge4)
MERGE(128, 16, sml_rw_merge16)
MERGE(64, 4, sml_rw_merge4_d64)
MERGE(64, 16, sml_rw_merge16_d64)

// ---------------------------------------------------------------- layers of a cache

// Unit z's pool of the layers: even numbers keys, odd ones values.
__device__ __forceinline__ uint16_t * pool_of(const sml_kpages & pg, size_t layer_stride, int z) {
    return (z & 1 ? pg.v : pg.k) + (size_t) (z >> 1) * layer_stride;
}

// ---------------------------------------------------------------- accepted drafts
//
// Every workgroup walks its sequence's tree for itself: a step is the first row
// behind the present one that follows it with its pick, 64 rows looked at a time
// by one wave (up to 64 in all are loaded once, a lane each). A thread then moves 16
// bytes of a position in one pool, a few of the path's rows at a time, in order: a
// row's new place lies before every later row's old one, so nothing is overwritten
// that is still to be read. Latency bounds it, the walk's chain of loads and then the
// path's copies: 3.6 us for 8 rows in 32 layers, 4.3 for 16 sequences of up to 26 in
// 28 (3.9 and 4.8 with a load a step of the walk and a row's copy at a time).
#define AC_AHEAD 4
extern "C" __global__ __launch_bounds__(256) void sml_rw_accept(const sml_kaccept a) {
    __shared__ int path[AC_MOST], count;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int s0 = min(max(a.start[b], 0), a.n_row), s1 = min(max(a.start[b + 1], s0), a.n_row), m = s1 - s0;
    const int cap = a.pg.seq_pages << a.pg.page_shift, past = max(a.len[b], 0) - m;
    if (tid < 64) {
        int k = 0, at = 0;
        if (m > 0) {
            if (!lane) path[0] = 0;
            k = 1;
        }
        if (m > 0 && m <= 64) {                       // a row a lane
            const bool in = lane < m;
            const int up = in ? a.parent[s0 + lane] : -1, tok = in ? a.tok[s0 + lane] : 0, pick = in ? a.pick[s0 + lane] : -1;
            while (k < a.most) {
                const int want = __builtin_amdgcn_readlane(pick, at);
                const unsigned long long hit = __ballot(want >= 0 && lane > at && up == at && tok == want);
                if (!hit) break;
                at = __builtin_ctzll(hit);
                if (!lane) path[k] = at;
                k++;
            }
        } else if (m > 0) {
            while (k < a.most) {
                const int want = a.pick[s0 + at];
                if (want < 0) break;
                int next = -1;
                for (int j0 = at + 1; j0 < m; j0 += 64) {
                    const int j = j0 + lane;
                    const unsigned long long hit = __ballot(j < m && a.parent[s0 + j] == at && a.tok[s0 + j] == want);
                    if (hit) { next = j0 + __builtin_ctzll(hit); break; }
                }
                if (next < 0) break;
                if (!lane) path[k] = next;
                at = next;
                k++;
            }
        }
        if (!lane) count = k;
    }
    __syncthreads();
    const int k = count;
    if (!blockIdx.x) {
        if (!tid) {
            if (a.n_kept) a.n_kept[b] = k;
            if (a.len_out) a.len_out[b] = past + k;
        }
        for (int j = tid; j < a.most; j += 256) {
            if (a.kept) a.kept[(size_t) b * a.most + j] = j < k ? path[j] : -1;
            if (a.next) a.next[(size_t) b * a.most + j] = j < k ? a.pick[s0 + path[j]] : -1;
        }
    }
    const int row = a.pg.n_kv * a.pg.hd / 8;          // 16-byte units of a position
    const uint32_t u = blockIdx.x * 256 + tid, z = u / (uint32_t) row;    // 2^31 units at most
    if (u >= 2u * (uint32_t) a.n_layer * (uint32_t) row) return;
    uint16_t * const pool = pool_of(a.pg, a.layer_stride, (int) z) + 8 * (u - z * (uint32_t) row);
    const int sh = a.pg.page_shift, pmask = (1 << sh) - 1;
    for (int j0 = 1; j0 < k; j0 += AC_AHEAD) {
        v4u w[AC_AHEAD];
        v4u * to[AC_AHEAD];
        #pragma unroll
        for (int e = 0; e < AC_AHEAD; e++) {
            const int j = j0 + e;
            to[e] = NULL;
            if (j >= k) continue;
            const int from = past + path[j], at = past + j;
            if (from == at || at < 0 || from >= cap) continue;
            const int pf = page_of(a.pg, b, from >> sh), pt = page_of(a.pg, b, at >> sh);
            if (pf < 0 || pt < 0) continue;
            w[e] = *(const v4u *) (pool + (size_t) pf * a.pg.page_stride + (size_t) (from & pmask) * 8 * row);
            to[e] = (v4u *) (pool + (size_t) pt * a.pg.page_stride + (size_t) (at & pmask) * 8 * row);
        }
        #pragma unroll
        for (int e = 0; e < AC_AHEAD; e++)
            if (to[e]) *to[e] = w[e];
    }
}

// ---------------------------------------------------------------- forks
//
// A workgroup copies 16 KB of the begun page in one pool; the first of a fork's
// also writes its row of the table. Its parts of the page are in flight at once, and
// enough workgroups wait at once to fill the stream: 64 forks of 16 sequences in
// 28 layers 16.5 us (94 MB, of which reads meet in the caches; 29 behind emptied
// ones), 4 of one in 32 layers 4.2, a launch's latency.
#define FK_UNITS 4                // 16-byte units a thread
extern "C" __global__ __launch_bounds__(256) void sml_rw_fork(const sml_kfork a) {
    const int i = blockIdx.y, tid = threadIdx.x, sh = a.pg.page_shift;
    const int b = a.parent[i], cap = a.pg.seq_pages << sh;
    const bool there = b >= 0 && b < a.pg.n_seq;
    const int n = there ? min(max(a.len[b], 0), cap) : 0, full = n >> sh, part = n & ((1 << sh) - 1);
    const int32_t * const from = a.pg.table + (size_t) (there ? b : 0) * a.pg.seq_pages;
    const int fresh = a.fresh[i];
    const bool copies = fresh >= 0 && fresh < a.pg.n_pages;
    if (!blockIdx.x && !blockIdx.z) {
        for (int p = tid; p < a.pg.seq_pages; p += 256)
            a.table_out[(size_t) i * a.pg.seq_pages + p] =
                p < full || (p == full && part && !copies) ? from[p] : p == full && part ? fresh : -1;
        if (!tid) a.len_out[i] = n;
    }
    if (!part || !copies || (int) blockIdx.z >= 2 * a.n_layer) return;
    const int src = page_of(a.pg, b, full);
    if (src < 0 || src == fresh) return;
    const long units = (long) part * a.pg.n_kv * a.pg.hd / 8;
    uint16_t * const pool = pool_of(a.pg, a.layer_stride, blockIdx.z);
    const v4u * const s = (const v4u *) (pool + (size_t) src * a.pg.page_stride);
    v4u * const d = (v4u *) (pool + (size_t) fresh * a.pg.page_stride);
    const long u0 = (long) blockIdx.x * (256 * FK_UNITS) + tid;
    #pragma unroll
    for (int e = 0; e < FK_UNITS; e++) {
        const long u = u0 + 256 * e;
        if (u < units) d[u] = s[u];
    }
}

// ---------------------------------------------------------------- moved pages
//
// A workgroup copies 16 KB of a page in one pool; behind the moves' workgroups
// (y) come those that rename the table's entries, each found among the
// ascending sources by halving. The stream bounds it: 121 pages' 444 MB, read and
// written, 90 us, as a large copy would take 86; 9 pages 6.4.
extern "C" __global__ __launch_bounds__(256) void sml_rw_compact(const sml_kcompact a) {
    const int tid = threadIdx.x;
    if ((int) blockIdx.y == a.n_move) {
        const long entries = (long) a.pg.n_seq * a.pg.seq_pages;
        const long step = (long) gridDim.x * gridDim.z * 256;
        for (long e = ((long) blockIdx.z * gridDim.x + blockIdx.x) * 256 + tid; e < entries; e += step) {
            const int p = a.table[e];
            if (p < 0 || p >= a.pg.n_pages) continue;
            int lo = 0, hi = a.n_move;                // src[lo] <= p, if any is
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (a.src[mid] <= p) lo = mid;
                else hi = mid;
            }
            const int to = a.dst[lo];
            if (a.src[lo] == p && to >= 0 && to < a.pg.n_pages) a.table[e] = to;
        }
        return;
    }
    const int src = a.src[blockIdx.y], dst = a.dst[blockIdx.y];
    if (src < 0 || src >= a.pg.n_pages || dst < 0 || dst >= a.pg.n_pages || src == dst) return;
    const long units = ((long) a.pg.n_kv * a.pg.hd / 8) << a.pg.page_shift;
    uint16_t * const pool = pool_of(a.pg, a.layer_stride, blockIdx.z);
    const v4u * const s = (const v4u *) (pool + (size_t) src * a.pg.page_stride);
    v4u * const d = (v4u *) (pool + (size_t) dst * a.pg.page_stride);
    const long u0 = (long) blockIdx.x * (256 * FK_UNITS) + tid;
    #pragma unroll
    for (int e = 0; e < FK_UNITS; e++) {
        const long u = u0 + 256 * e;
        if (u < units) d[u] = s[u];
    }
}
