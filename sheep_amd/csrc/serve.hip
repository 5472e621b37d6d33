// Kernels of a step that serves many requests at once (sml-serve.h): the paged
// cache's append and attention, low-rank adapters, and the rules on logits.
#include "dev.h"

typedef float v4f __attribute__((ext_vector_type(4)));
// four floats at a float's alignment: rows start at any stride
typedef float v4fu __attribute__((ext_vector_type(4), aligned(4)));

// float to the 16-bit type, to nearest even, and back
template <int BF> __device__ __forceinline__ uint16_t to16(float f) {
    if constexpr (BF) return __builtin_bit_cast(uint16_t, (__bf16) f);
    else return f2h(f);
}
template <int BF> __device__ __forceinline__ float of16(uint16_t h) {
    if constexpr (BF) return __builtin_bit_cast(float, (uint32_t) h << 16);
    else return h2f(h);
}

// What a wave's lanes wrote to its own part of LDS is there for all of them.
__device__ __forceinline__ void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The page of entry i of sequence s, or -1.
__device__ __forceinline__ int page_of(const sml_kpages & pg, int s, int i) {
    const int p = pg.table[(size_t) s * pg.seq_pages + i];
    return p >= 0 && p < pg.n_pages ? p : -1;
}

// ---------------------------------------------------------------- append
//
// A thread takes four rotation pairs (d, d + hd/2) of one head of q or k, or
// four values of v. The pair's products are the decode kernels' (one rounded,
// the other fused), so a float16 cache equals the contiguous one. It reads and
// writes each value once; what bounds it is the launch (16 tokens, 32 heads over
// 8 of 128: 2.9 us of kernel in a call of 5.4) until the rows are thousands (1021
// tokens, 12 over 2: 16 MB in 4.2 us, 3.9 TB/s). Four pairs a thread make every
// access 8 or 16 bytes.
template <int D, int BF>
__device__ __forceinline__ void append_body(const sml_kappend & a) {
    constexpr int HQ = D / 8;                         // threads of a rotated head
    const int r = blockIdx.x, i = blockIdx.y * blockDim.x + threadIdx.x;
    const int s = a.seq ? a.seq[r] : r, p = a.pos[r];
    if (p < 0 || p >= a.n_rope || p >> a.pg.page_shift >= a.pg.seq_pages || s < 0 || s >= a.pg.n_seq) return;
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
    const v4f c = *(const v4fu *) (a.cos_t + (size_t) p * (D / 2) + d), sn = *(const v4fu *) (a.sin_t + (size_t) p * (D / 2) + d);
    v4f y0, y1;
    #pragma unroll
    for (int e = 0; e < 4; e++) {
        y0[e] = __builtin_fmaf(lo[e], c[e], -(hi[e] * sn[e]));
        y1[e] = __builtin_fmaf(lo[e], sn[e], hi[e] * c[e]);
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
#define APPEND(D, BF, name) \
    extern "C" __global__ __launch_bounds__(256) void name(const sml_kappend a) { append_body<D, BF>(a); }
APPEND(128, 0, sml_sv_append)
APPEND(128, 1, sml_sv_append_bf)
APPEND(64, 0, sml_sv_append_d64)
APPEND(64, 1, sml_sv_append_d64_bf)

// ---------------------------------------------------------------- attention
//
// out = sum_i 2^(s_i - m) v_i / sum_i 2^(s_i - m), s_i = scale log2(e) q.k_i,
// in one pass over the cache with a running base m. Nothing is read twice and
// the arithmetic is 4 operations a value of up to 16 heads, so the cache's
// bytes bound it: everything else is arranged to keep loads in flight.
//
// A workgroup takes a split of a sequence's positions for one KV head, its
// waves alternate tiles of 32 positions, and a wave keeps all of a tile in
// registers while the next is on its way. The matrix cores take
// S^T = K Q^T and O^T = V^T P^T, heads in the columns (the unused of the 16
// are zero). With the lane's c = lane % 16, g = lane / 16:
// - K is the first operand as the cache stores it: lane (c, g) takes 16 bytes of
//   position c's row, dims 32j + 8g.. for product j. Loads in that order would
//   touch 16 rows in 16 consecutive lanes, a cache line a lane: the rows are
//   loaded whole and handed over through the wave's part of LDS.
// - S comes back as positions 4g + r of head c, which is just what the second
//   product takes as its P^T operand if its inner index 8g + i stands for
//   position 4g + i of the first 16 positions (i < 4) or of the second: P
//   never crosses lanes.
// - V's rows of those 8 positions are loaded whole, 16 lanes a row, dims
//   (D/16)c.. each; the product u takes dim (D/16)c + u of every lane, so V^T
//   is 4 D/16 byte permutes in the lane, and lane (c, g) ends with dims
//   (D/4)g.. of head c: the base's rescaling is a lane's own too.
// q and the weights are split into parts of the cache's type (two of fp16,
// three of bf16: 22 and 24 bits), a matrix instruction each. fp16 has little
// range: q's row is scaled by a power of two to below 2^11 first, and the base
// starts 10 below the first maximum and moves when a score passes it by 15, so
// that weights lie up to 2^15 and those that fp16's smallest steps round are
// 2^-34 of the largest. bf16 has fp32's, and so may its keys and values: there
// q stays as it is, and the base starts 4 above the maximum and moves when a
// score passes it: weights of 1 at most leave the largest values their room, and
// of 1/16 the smallest. (The base thus moves when the maximum has risen by 5 or
// 4, which few tiles see. A base that is the maximum itself moves in most: one
// at 65537 29.2 us for 28.8 on warm caches, 48 up to 8192 43.4 for 42.7.)
//
// Pages are looked up a tile ahead, once per 16 positions (a page is a
// multiple of 16). Positions past the length or on absent pages are loaded
// from where memory is (the rest of the page, or page 0), their scores
// replaced by -infinity and their V rows by zeros; tiles of absent pages alone
// are passed over.
//
// Lengths are ragged and the host knows only a bound of them, so the device
// shares the work out: every wave sums the lengths and finds its workgroup's
// sequence and split (at_place), splits of one size for all. Past AT_SHARED
// sequences, whose sum would cost too much, splits have a fixed size and the
// grid every sequence's most (want 0).
//
// Measured with the merge, 32 heads over 8 of 128, fp16: 48 sequences up to
// 8192 (202 MB) 55 us = 3.7 TB/s (60 with fixed splits of 512 and K in the
// matrix cores' order from memory), one at 4095 10.2 us, of which 5.9 are this
// kernel's chain of latencies (length, table, rows, joining) and 3.6 the
// merge's; bf16, 28 over 4, one at 65537 (134 MB) 34.7 us = 3.9 TB/s. A large
// copy reaches 4.8 TB/s. Two workgroups (212 registers, bf16 228) a CU: held to
// three, 58 and 52 us.
#define AT_WAVES 4

// The positions a sequence attends over.
__device__ __forceinline__ int at_len(const sml_kattend & a, int b) { return min(max(a.len[b], 0), a.max_len); }
// The inclusive sums of v over the wave's lanes.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);           // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);           // row_bcast 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);           // row_bcast 31 into rows 2 and 3
    return v;
}
// The positions of a split, by one wave: a multiple of 128, a.chunk at least,
// else what makes a.want splits in all (counted in units of 128 positions:
// AT_SHARED lengths of 2^30 stay below 2^31).
__device__ __forceinline__ int at_size(const sml_kattend & a, int lane) {
    if (!a.want) return a.chunk;
    unsigned t = 0;
    if (a.pg.n_seq == 1) {
        t = (unsigned) (at_len(a, 0) + 127) >> 7;
    } else {
        #pragma unroll 4
        for (int b = lane; b < a.pg.n_seq; b += 64) t += (unsigned) (at_len(a, b) + 127) >> 7;
        t = (unsigned) __builtin_amdgcn_readlane(wave_scan((int) t), 63);
    }
    return max(a.chunk, (int) min((t + a.want - 1) / a.want, 1u << 23) * 128);
}
// A sequence of n positions in splits of about chunk: equal ones, to a tile of
// 32; per is their size. At least one (an empty sequence's writes its zeros).
__device__ __forceinline__ int at_splits(int n, int chunk, int & per) {
    const int p = max((n + chunk - 1) / chunk, 1);
    per = max(((n + p - 1) / p + 31) & ~31, 32);
    return max((n + per - 1) / per, 1);
}
// Split i of all, in the sequences' order: its sequence, its number there,
// their size and count; false past the last.
__device__ __forceinline__ bool at_place(const sml_kattend & a, int i, int lane, int & b, int & split, int & per, int & count) {
    const int chunk = at_size(a, lane);
    if (!a.want || a.pg.n_seq == 1) {
        b = blockIdx.z;
        split = i;
        count = at_splits(at_len(a, b), chunk, per);
        return i < count;
    }
    for (int b0 = 0; b0 < a.pg.n_seq; b0 += 64) {
        int pl = 32, cl = 0;
        if (b0 + lane < a.pg.n_seq) cl = at_splits(at_len(a, b0 + lane), chunk, pl);
        const int sum = wave_scan(cl);
        const unsigned long long at = __ballot(sum > i);
        if (at) {
            const int l = __builtin_ctzll(at);
            b = b0 + l;
            count = __builtin_amdgcn_readlane(cl, l);
            per = __builtin_amdgcn_readlane(pl, l);
            split = i - (__builtin_amdgcn_readlane(sum, l) - count);
            return true;
        }
        i -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

template <int BF> struct Mx;
template <> struct Mx<0> {
    typedef _Float16 t;
    typedef t v8 __attribute__((ext_vector_type(8)));
    static constexpr int parts = 2;
    static constexpr float lift = -10.0f, room = 15.0f;   // of the base over a maximum, of a score over the base
    static __device__ __forceinline__ v4f mul(v8 a, v8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mx<1> {
    typedef __bf16 t;
    typedef t v8 __attribute__((ext_vector_type(8)));
    static constexpr int parts = 3;
    static constexpr float lift = 4.0f, room = 0.0f;
    static __device__ __forceinline__ v4f mul(v8 a, v8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// Powers of two: the one that brings values up to mx below 2^11, and back.
__device__ __forceinline__ int scale_of(float mx) {
    return mx > 0.0f && mx < INFINITY ? __builtin_amdgcn_frexp_expf(mx) - 11 : 0;
}

// Elements e and e + 1 of the parts of x and y: each part what its type holds of
// what is left, which the subtraction leaves exactly. fp16 rounds (the scaled
// values stay below its largest); bfloat16 cuts off, so that the largest fp32
// values do not round up to an infinity, and three cut parts of 8 bits are all
// of the 24.
template <int BF>
__device__ __forceinline__ void parts_of(float x, float y, typename Mx<BF>::v8 (&p)[Mx<BF>::parts], int e) {
    typedef typename Mx<BF>::t v2t __attribute__((ext_vector_type(2)));
    typedef float v2f __attribute__((ext_vector_type(2)));
    #pragma unroll
    for (int k = 0; k < Mx<BF>::parts; k++) {
        v2t h;
        if constexpr (BF) h = __builtin_bit_cast(v2t, __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u));
        else h = __builtin_convertvector(v2f{x, y}, v2t);
        p[k][e] = h[0];
        p[k][e + 1] = h[1];
        x = __builtin_fmaf((float) h[0], -1.0f, x);
        y = __builtin_fmaf((float) h[1], -1.0f, y);
    }
}

template <int D, int BF>
__device__ __forceinline__ void attend_body(const sml_kattend & a) {
    using M = Mx<BF>;
    typedef typename M::v8 v8;
    constexpr int NJ = D / 32, E = D / 16, NP = M::parts, W = AT_WAVES;
    typedef unsigned vrow __attribute__((ext_vector_type(E / 2)));
    constexpr int KR = 2 * D + 16;                    // bytes of a K row in LDS: 16 rows fall on different banks
    __shared__ __align__(16) uint8_t lds[W * 32 * KR];  // a wave's 32 K rows; at the end its sums
    static_assert(32 * KR >= 16 * (D + 4) * 4, "");
    __shared__ float sm[W][16], sl[W][16];
    const int kh = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    int b, split, per, count;
    if (!at_place(a, blockIdx.y, lane, b, split, per, count)) return;
    const int n = at_len(a, b), t0 = split * per, t1 = min(n, t0 + per);
    const int rep = a.n_head / a.pg.n_kv, kvd = a.pg.n_kv * D;
    const int sh = a.pg.page_shift, pmask = (1 << sh) - 1;
    const int32_t * const tab = a.pg.table + (size_t) b * a.pg.seq_pages;

    // the query: lane (c, g) holds dims 32j + 8g.. of head c, in parts
    v8 q[NJ][NP];
    float back;                                       // what a product of the scaled q is multiplied by
    {
        float x[NJ][8], mx = 0.0f;
        const float * qp = a.q + (size_t) b * a.q_stride + (size_t) (kh * rep + min(c, rep - 1)) * D + 8 * g;
        #pragma unroll
        for (int j = 0; j < NJ; j++)
            #pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const v4f v = *(const v4fu *) (qp + 32 * j + e);
                #pragma unroll
                for (int i = 0; i < 4; i++) { x[j][e + i] = c < rep ? v[i] : 0.0f; mx = fmaxf(mx, fabsf(x[j][e + i])); }
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const int ex = BF ? 0 : scale_of(mx);
        #pragma unroll
        for (int j = 0; j < NJ; j++)
            #pragma unroll
            for (int e = 0; e < 8; e += 2)
                parts_of<BF>(__builtin_amdgcn_ldexpf(x[j][e], -ex), __builtin_amdgcn_ldexpf(x[j][e + 1], -ex), q[j], e);
        back = __builtin_amdgcn_ldexpf(a.scale, ex);
    }

    v4f o[E];
    #pragma unroll
    for (int u = 0; u < E; u++) o[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float base = -INFINITY, l = 0.0f;

    // the next tile at or after t (this wave's) that has a page, and its two
    // pages (-1: absent)
    int pa = -1, pb = -1;
    auto seek = [&](int t) {
        for (; t < t1; t += 32 * W) {
            pa = tab[t >> sh];
            pb = t + 16 < t1 ? tab[(t + 16) >> sh] : -1;
            pa = pa >= 0 && pa < a.pg.n_pages ? pa : -1;
            pb = pb >= 0 && pb < a.pg.n_pages ? pb : -1;
            if (pa >= 0 || pb >= 0) break;
        }
        return t;
    };
    constexpr int LK = D / 8, RK = 64 / LK;           // lanes of a K row, rows of a load
    v4u kr[2][16 / RK];
    vrow vr[8];
    uint8_t * const lk = lds + wave * 32 * KR;
    uint32_t koff[16 / RK];
    #pragma unroll
    for (int i = 0; i < 16 / RK; i++) koff[i] = 2u * (uint32_t) ((RK * i + lane / LK) * kvd + 8 * (lane % LK));
    uint32_t voff[4];
    #pragma unroll
    for (int i = 0; i < 4; i++) voff[i] = 2u * (uint32_t) ((4 * g + i) * kvd + E * c);
    // the places of a tile's two halves in a pool
    auto place = [&](int page, int t) {
        return (size_t) max(page, 0) * a.pg.page_stride + (size_t) (t & pmask) * kvd + (size_t) kh * D;
    };
    auto load_k = [&](size_t xa, size_t xb) {
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            const GLOBAL char * p = (const GLOBAL char *) (a.pg.k + (h ? xb : xa));
            #pragma unroll
            for (int i = 0; i < 16 / RK; i++) kr[h][i] = *(const GLOBAL v4u *) (p + koff[i]);
        }
    };
    auto load_v = [&](size_t xa, size_t xb) {
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            const GLOBAL char * p = (const GLOBAL char *) (a.pg.v + (h ? xb : xa));
            #pragma unroll
            for (int i = 0; i < 4; i++) vr[4 * h + i] = *(const GLOBAL vrow *) (p + voff[i]);
        }
    };

    int t = seek(t0 + 32 * wave);
    if (t < t1) {
        const size_t xa = place(pa, t), xb = place(pb, t + 16);
        load_k(xa, xb);
        load_v(xa, xb);
    }
    while (t < t1) {
        const bool ha = pa >= 0, hb = pb >= 0, whole = ha && hb && t + 32 <= t1;
        const int tn = seek(t + 32 * W);
        const size_t xa = place(pa, tn), xb = place(pb, tn + 16);
        #pragma unroll
        for (int h = 0; h < 2; h++)
            #pragma unroll
            for (int i = 0; i < 16 / RK; i++) *(v4u *) (lk + (16 * h + RK * i + lane / LK) * KR + 16 * (lane % LK)) = kr[h][i];
        wave_lds();
        if (tn < t1) load_k(xa, xb);
        v4f s[2];
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            s[h] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            #pragma unroll
            for (int j = 0; j < NJ; j++) {
                const v8 kj = *(const v8 *) (lk + (16 * h + c) * KR + 64 * j + 16 * g);
                #pragma unroll
                for (int k = 0; k < NP; k++) s[h] = M::mul(kj, q[j][k], s[h]);
            }
        }
        wave_lds();                                   // all read before the next tile is written
        // the lane's scores: positions 4g + r of either half
        float mx = -INFINITY;
        #pragma unroll
        for (int h = 0; h < 2; h++)
            #pragma unroll
            for (int r = 0; r < 4; r++) s[h][r] *= back;
        if (!whole) {
            #pragma unroll
            for (int h = 0; h < 2; h++)
                #pragma unroll
                for (int r = 0; r < 4; r++) {
                    const bool in = (h ? hb : ha) && t + 16 * h + 4 * g + r < t1;
                    s[h][r] = in ? s[h][r] : -INFINITY;
                    if (!in) vr[4 * h + r] = vrow(0u);
                }
        }
        #pragma unroll
        for (int h = 0; h < 2; h++)
            #pragma unroll
            for (int r = 0; r < 4; r++) mx = fmaxf(mx, s[h][r]);
        if (__any(mx > base + M::room)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float to = mx > base + M::room ? mx + M::lift : base;
            const float al = __builtin_amdgcn_exp2f(base - (to == -INFINITY ? 0.0f : to));
            l *= al;
            #pragma unroll
            for (int u = 0; u < E; u++)
                #pragma unroll
                for (int r = 0; r < 4; r++) o[u][r] *= al;
            base = to;
        }
        const float bu = base == -INFINITY ? 0.0f : base;
        v8 p[NP];
        #pragma unroll
        for (int h = 0; h < 2; h++)
            #pragma unroll
            for (int r = 0; r < 4; r += 2) {
                const float w0 = __builtin_amdgcn_exp2f(s[h][r] - bu), w1 = __builtin_amdgcn_exp2f(s[h][r + 1] - bu);
                l += w0;
                l += w1;
                parts_of<BF>(w0, w1, p, 4 * h + r);
            }
        #pragma unroll
        for (int u = 0; u < E; u++) {
            v4u w;
            #pragma unroll
            for (int i = 0; i < 4; i++)
                w[i] = __builtin_amdgcn_perm(vr[2 * i + 1][u / 2], vr[2 * i][u / 2], u & 1 ? 0x07060302u : 0x05040100u);
            #pragma unroll
            for (int k = 0; k < NP; k++) o[u] = M::mul(__builtin_bit_cast(v8, w), p[k], o[u]);
        }
        if (tn < t1) load_v(xa, xb);
        t = tn;
    }

    // the waves' sums joined: wave w's head c, dims (D/4)g + Er + u
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();                                  // the K rows are done with
    float (* const so)[16][D + 4] = (float (*)[16][D + 4]) lds;
    if (c < rep) {
        #pragma unroll
        for (int r = 0; r < 4; r++)
            #pragma unroll
            for (int u = 0; u < E; u++) so[wave][c][(D / 4) * g + E * r + u] = o[u][r];
        if (!g) { sm[wave][c] = base; sl[wave][c] = l; }
    }
    __syncthreads();
    const size_t row0 = (size_t) b * a.n_head + (size_t) kh * rep;
    for (int i = tid; i < rep * D; i += 64 * W) {
        const int h = i / D, d = i % D;
        float m = sm[0][h];
        #pragma unroll
        for (int w = 1; w < W; w++) m = fmaxf(m, sm[w][h]);
        const float mu = m == -INFINITY ? 0.0f : m;
        float os = 0.0f, ls = 0.0f;
        #pragma unroll
        for (int w = 0; w < W; w++) {
            const float f = __builtin_amdgcn_exp2f(sm[w][h] - mu);
            os += f * so[w][h][d];
            ls += f * sl[w][h];
        }
        if (count == 1) {
            a.out[(row0 + h) * D + d] = ls == 0.0f ? 0.0f : os / ls;
        } else {
            const size_t at = (row0 + h) * a.nsplit + split;
            a.part[at * D + d] = os;
            if (!d) *(float2 *) (a.part + (size_t) a.pg.n_seq * a.n_head * a.nsplit * D + 2 * at) = make_float2(m, ls);
        }
    }
}

// The splits of a row joined: a workgroup a (sequence, head), D threads a
// share of its splits. Latency bounds it: the lengths, the splits' bases, then
// each share's rows, eight in flight. us a call with its attention, 256 / 512 /
// 1024 threads: 28 heads, one sequence at 65537 (129 splits) 30.6 / 29.2 / 29.7,
// 32 heads, 4 of 3000 17.0 / 16.3 / 16.4, but 200 of up to 2000 (6400 workgroups)
// 74 / 80 / 93.
template <int D, int NT>
__device__ __forceinline__ void attend_merge_body(const sml_kattend & a) {
    constexpr int S = NT / D;                         // shares
    __shared__ float f[256], red[S][D], sred[NT / 64];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    int per;
    const int ns = at_splits(at_len(a, b), at_size(a, tid & 63), per);
    if (ns == 1) return;                              // written already
    const size_t row = (size_t) b * a.n_head + h;
    const float * po = a.part + row * a.nsplit * D;
    const float2 * pm = (const float2 *) (a.part + (size_t) a.pg.n_seq * a.n_head * a.nsplit * D) + row * a.nsplit;
    const float2 ml = tid < ns ? pm[tid] : make_float2(-INFINITY, 0.0f);
    float m = wave_max(ml.x);
    if (!(tid & 63)) sred[tid >> 6] = m;
    __syncthreads();
    m = sred[0];
    #pragma unroll
    for (int w = 1; w < NT / 64; w++) m = fmaxf(m, sred[w]);
    const float e = __builtin_amdgcn_exp2f(ml.x - (m == -INFINITY ? 0.0f : m));
    if (NT == 256 || tid < 256) f[tid] = e;
    __syncthreads();                                  // f is whole, and sred read by all
    const float lw = wave_sum(e * ml.y);
    if (!(tid & 63)) sred[tid >> 6] = lw;
    const int d = tid % D, s0 = tid / D;
    float o = 0.0f;
    #pragma unroll 8
    for (int i = s0; i < ns; i += S) o += f[i] * po[(size_t) i * D + d];
    red[s0][d] = o;
    __syncthreads();
    if (tid >= D) return;
    float l = 0.0f;
    #pragma unroll
    for (int w = 0; w < NT / 64; w++) l += sred[w];
    #pragma unroll
    for (int s = 1; s < S; s++) o += red[s][d];
    a.out[row * D + d] = l == 0.0f ? 0.0f : o / l;
}
#define MERGE(D, NT, name) \
    extern "C" __global__ __launch_bounds__(NT) void name##_##NT(const sml_kattend a) { attend_merge_body<D, NT>(a); }
MERGE(128, 256, sml_sv_merge)
MERGE(128, 512, sml_sv_merge)
MERGE(64, 256, sml_sv_merge_d64)
MERGE(64, 512, sml_sv_merge_d64)

#define ATTEND(D, BF, name) \
    extern "C" __global__ __launch_bounds__(64 * AT_WAVES) void name(const sml_kattend a) { attend_body<D, BF>(a); }
ATTEND(128, 0, sml_sv_attend)
ATTEND(128, 1, sml_sv_attend_bf)
ATTEND(64, 0, sml_sv_attend_d64)
ATTEND(64, 1, sml_sv_attend_d64_bf)

// ---------------------------------------------------------------- logits
//
// A workgroup takes LG_RANGE tokens of a row, K words of four a thread. Its
// logits and mask bits are on their way while it counts the row's history and
// finds the biases of its own tokens in LDS (whole numbers, so the order of
// the atomics does not show); then the rules are applied in the order the
// header gives, with no contraction, and the greedy pick's candidate is kept.
// The logits, read and written once, bound the large calls; every workgroup
// reads its row's whole history, which stays in L2. A small call is a chain of
// latencies (the list's bounds, the list, LDS, the biases), and its code's own
// loading counts: the listed tokens go through one copy of the rules (one
// division), not sixteen unrolled (1 row of 128256: 10.3 us so, 6.0 with).
//
// us a call with the pick, 512 threads of one word / 256 of two / 4096 tokens a
// workgroup, 512 threads of two / 256 of four (128256 tokens, masks, histories
// of 2047, from 16 rows four batches in turn): 1 row 7.3 / 8.3 / 8.1 / 10.9 (5.4
// and 1.4 of the first its kernels'), 12 rows 9.0 / 9.4 / 10.1 / 12.0, 16 rows
// 10.5 / 10.5 / 11.0 / 13.0, 32 rows 15.5 / 14.6 / 14.7 / 15.6, 96 rows 38.5 /
// 30.8 / 33.9 / 42; histories of 65536: 1 row 15 / 23 / 17 / 28, 16 rows 18 / 25
// / 24 / 29, 96 rows 59 / 54 / 55 / 66. So 256 threads of two lose up to 30%
// where histories are that long. The 96 rows' first kernel streams their 99 MB
// at 4.1 TB/s. The pick looks for the largest value first and for its place in
// the lanes that have it; with an index carried beside every value a word of
// four took 213 instructions, and the 96 rows 2 us more.
#define LG_SEEN 0x80000000u

// The largest value and the smallest index over the wave's lanes.
__device__ __forceinline__ float wave_top(float v) {
    const int r = __builtin_bit_cast(int, max16(v));
    const float a = __builtin_bit_cast(float, __builtin_amdgcn_readlane(r, 0)), b = __builtin_bit_cast(float, __builtin_amdgcn_readlane(r, 16));
    const float c = __builtin_bit_cast(float, __builtin_amdgcn_readlane(r, 32)), d = __builtin_bit_cast(float, __builtin_amdgcn_readlane(r, 48));
    return fmaxf(fmaxf(a, b), fmaxf(c, d));
}
__device__ __forceinline__ unsigned wave_least(unsigned v) {
    v = min(v, (unsigned) dpp_i<0xB1>((int) v));
    v = min(v, (unsigned) dpp_i<0x4E>((int) v));
    v = min(v, (unsigned) dpp_i<0x141>((int) v));
    v = min(v, (unsigned) dpp_i<0x140>((int) v));
    const unsigned a = (unsigned) __builtin_amdgcn_readlane((int) v, 0), b = (unsigned) __builtin_amdgcn_readlane((int) v, 16);
    const unsigned c = (unsigned) __builtin_amdgcn_readlane((int) v, 32), d = (unsigned) __builtin_amdgcn_readlane((int) v, 48);
    return min(min(a, b), min(c, d));
}
// Of the lanes' candidates (value, index; NaN loses, LG_NONE is none) the
// lowest index of the largest value; of their first permitted tokens (twice the
// index, plus 1 if the value is NaN) the first.
__device__ __forceinline__ void pick_wave(float & bv, unsigned & bi, unsigned & first) {
    const float top = wave_top(bv);
    bi = wave_least(bv == top ? bi : 0x7fffffffu);
    bv = top;
    first = wave_least(first);
}
#define LG_NONE 0x7fffffffu                           // no index
#define LG_FIRST 0xffffffffu                          // nothing permitted

__device__ __forceinline__ float pick4(v4f v, int e) { return e & 2 ? (e & 1 ? v[3] : v[2]) : (e & 1 ? v[1] : v[0]); }
__device__ __forceinline__ unsigned pick4(v4u v, int e) { return e & 2 ? (e & 1 ? v[3] : v[2]) : (e & 1 ? v[1] : v[0]); }

template <int NT, int K>
__device__ __forceinline__ void logits_body(const sml_klogits & a) {
    #pragma clang fp contract(off)
    static_assert(NT * K * 4 == LG_RANGE, "");
    __shared__ __align__(16) unsigned cnt[LG_RANGE];     // generated count, LG_SEEN if listed at all
    __shared__ __align__(16) unsigned bia[LG_RANGE];     // the last bias entry's index + 1
    __shared__ float rv[NT / 64];
    __shared__ unsigned ri[NT / 64], rf[NT / 64];
    const int row = blockIdx.y, t0 = blockIdx.x * LG_RANGE, tid = threadIdx.x;
    const int nt = min(LG_RANGE, a.n_vocab - t0);
    const float * x = a.logits + (size_t) row * a.stride + t0;
    const int mr = !a.mask ? -1 : a.mask_row ? a.mask_row[row] : row;
    const bool none = mr < -1 || mr >= a.n_mask;      // a mask that is not there permits nothing
    v4f l[K];
    uint32_t ok[K];                                   // bits 0..3: permitted and inside the row
    #pragma unroll
    for (int i = 0; i < K; i++) {
        const int j = 4 * (NT * i + tid);
        l[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (j + 4 <= nt) l[i] = *(const v4fu *) (x + j);
        else
            for (int e = 0; e < 3; e++) if (j + e < nt) l[i][e] = x[j + e];
        ok[i] = j >= nt ? 0u : j + 4 <= nt ? 15u : (1u << (nt - j)) - 1u;
        if (a.mask && mr != -1) {
            uint32_t w = 0;
            if (!none && j < nt) w = a.mask[(size_t) mr * ((a.n_vocab + 31) / 32) + ((t0 + j) >> 5)] >> (j & 31);
            ok[i] &= w;
        }
    }
    if (a.hist || a.bias) {
        #pragma unroll
        for (int i = 0; i < K; i++) {
            if (a.hist) *(v4u *) (cnt + 4 * (NT * i + tid)) = v4u(0u);
            if (a.bias) *(v4u *) (bia + 4 * (NT * i + tid)) = v4u(0u);
        }
        __syncthreads();
    }
    if (a.hist) {
        const int h0 = min(max(a.hist_start[row], 0), a.n_hist), h1 = min(max(a.hist_start[row + 1], 0), a.n_hist);
        const int gen = h0 + (a.n_prompt ? min(max(a.n_prompt[row], 0), max(h1 - h0, 0)) : 0);
        auto take = [&](int i, unsigned t) {
            if (t < (unsigned) nt) {
                if (i >= gen) atomicAdd(&cnt[t], 1u);
                atomicOr(&cnt[t], LG_SEEN);
            }
        };
        // sixteen ids a thread in flight, most of them another workgroup's
        typedef int v4iu __attribute__((ext_vector_type(4), aligned(4)));
        int i = h0 + 4 * tid;
        for (; i + 12 * NT + 4 <= h1; i += 16 * NT) {
            v4i t[4];
            #pragma unroll
            for (int k = 0; k < 4; k++) t[k] = *(const v4iu *) (a.hist + i + 4 * NT * k) - t0;
            #pragma unroll
            for (int k = 0; k < 4; k++)
                if (min(min((unsigned) t[k][0], (unsigned) t[k][1]), min((unsigned) t[k][2], (unsigned) t[k][3])) < (unsigned) nt) {
                    #pragma unroll
                    for (int e = 0; e < 4; e++) take(i + 4 * NT * k + e, (unsigned) t[k][e]);
                }
        }
        for (; i < h1; i += 4 * NT) {
            int t[4];
            #pragma unroll
            for (int e = 0; e < 4; e++) t[e] = a.hist[min(i + e, h1 - 1)] - t0;
            #pragma unroll
            for (int e = 0; e < 4; e++) if (i + e < h1) take(i + e, (unsigned) t[e]);
        }
    }
    if (a.bias) {
        const int b0 = min(max(a.bias_start[row], 0), a.n_bias), b1 = min(max(a.bias_start[row + 1], 0), a.n_bias);
        for (int i = b0 + tid; i < b1; i += NT) {
            const int t = a.bias_id[i] - t0;
            if ((unsigned) t < (unsigned) nt) atomicMax(&bia[t], (unsigned) i + 1);
        }
    }
    const float rep = a.rep ? a.rep[row] : 1.0f, fr = a.frequency ? a.frequency[row] : 0.0f,
                pr = a.presence ? a.presence[row] : 0.0f;
    if (a.hist || a.bias) __syncthreads();
    float bv = -INFINITY;
    #pragma unroll
    for (int i = 0; i < K; i++) {
        const int j = 4 * (NT * i + tid);
        v4u c = v4u(0u), k = v4u(0u);
        if (a.hist) c = *(const v4u *) (cnt + j);
        if (a.bias) k = *(const v4u *) (bia + j);
        // the few listed tokens one by one: one copy of the division
        unsigned todo = (c[0] | k[0] ? 1u : 0u) | (c[1] | k[1] ? 2u : 0u) | (c[2] | k[2] ? 4u : 0u) | (c[3] | k[3] ? 8u : 0u);
        while (todo) {
            const int e = __builtin_ctz(todo);
            todo &= todo - 1;
            float v = pick4(l[i], e);
            const unsigned ce = pick4(c, e), m = ce & ~LG_SEEN, ke = pick4(k, e);
            if (ce && a.rep) v = v > 0.0f ? v / rep : v * rep;
            if (m && a.frequency) v = v - fr * (float) m;
            if (m && a.presence) v = v - pr;
            if (ke) v = v + a.bias[ke - 1];
            #pragma unroll
            for (int f = 0; f < 4; f++) l[i][f] = e == f ? v : l[i][f];
        }
        ok[i] &= 15u;
        if (ok[i] != 15u) {
            #pragma unroll
            for (int e = 0; e < 4; e++) l[i][e] = ok[i] >> e & 1 ? l[i][e] : -INFINITY;
        }
        bv = fmaxf(bv, fmaxf(fmaxf(l[i][0], l[i][1]), fmaxf(l[i][2], l[i][3])));
        if (a.out) {
            float * y = a.out + (size_t) row * a.out_stride + t0 + j;
            if (j + 4 <= nt) *(v4fu *) y = l[i];
            else
                for (int e = 0; e < 3; e++) if (j + e < nt) y[e] = l[i][e];
        }
    }
    if (!a.tok) return;
    // the wave's largest value, then the lanes that have it look for its place
    // (indices rise over the words, the waves, the lanes)
    const float top = wave_top(bv);
    unsigned bi = LG_NONE, first = LG_FIRST;
    if (bv == top) {
        #pragma unroll
        for (int i = K - 1; i >= 0; i--)
            #pragma unroll
            for (int e = 3; e >= 0; e--) bi = (ok[i] >> e & 1) && l[i][e] == top ? (unsigned) (t0 + 4 * (NT * i + tid) + e) : bi;
    }
    #pragma unroll
    for (int i = K - 1; i >= 0; i--) {
        const int e = __builtin_ctz(ok[i] | 16u);
        const float v = pick4(l[i], e);
        first = ok[i] ? 2u * (unsigned) (t0 + 4 * (NT * i + tid) + e) + (v != v) : first;
    }
    bi = wave_least(bi);
    first = wave_least(first);
    if ((tid & 63) == 0) { rv[tid >> 6] = top; ri[tid >> 6] = bi; rf[tid >> 6] = first; }
    __syncthreads();
    if (tid >= 64) return;
    bv = tid < NT / 64 ? rv[tid] : -INFINITY;
    bi = tid < NT / 64 ? ri[tid] : LG_NONE;
    first = tid < NT / 64 ? rf[tid] : LG_FIRST;
    pick_wave(bv, bi, first);
    if (!tid) a.part[(size_t) row * a.n_part + blockIdx.x] = make_int4(__float_as_int(bv), (int) bi, (int) first, 0);
}
#define LOGITS(NT, K) \
    extern "C" __global__ __launch_bounds__(NT) void sml_sv_logits_##NT##_##K(const sml_klogits a) { logits_body<NT, K>(a); }
LOGITS(512, 1)
LOGITS(256, 2)

// The pick over a row's blocks: the first permitted token if it is NaN (the
// serial loop never leaves it), else the lowest index of the largest value.
extern "C" __global__ __launch_bounds__(64) void sml_sv_pick(const sml_klogits a) {
    const int row = blockIdx.x;
    float bv = -INFINITY;
    unsigned bi = LG_NONE, first = LG_FIRST;
    for (int i = threadIdx.x; i < a.n_part; i += 64) {
        const int4 p = a.part[(size_t) row * a.n_part + i];
        const float v = __int_as_float(p.x);
        // a lane's blocks come in order: only a larger value displaces, or any
        // index where there was none
        if (v > bv || bi == LG_NONE) { bv = v; bi = (unsigned) p.y; }
        first = min(first, (unsigned) p.z);
    }
    pick_wave(bv, bi, first);
    if (!threadIdx.x) a.tok[row] = first == LG_FIRST ? -1 : first & 1 ? (int) (first >> 1) : (int) bi;
}

// ---------------------------------------------------------------- adapters
//
// y = base + scale B (A x). Rows come in tiles of 16; a tile's distinct adapters
// are taken one by one, all of its rows computed with each and those of the
// adapter's own rows kept. Rows never mix in a product, so a row sees nothing
// of the others, and no sorting of requests is needed: requests of a tile that
// share an adapter read it once, those that do not read each their own, which
// is the least there is to read.
//
// fp32 x and t meet the 16-bit matrices as parts of their type (fp16: two, and
// each row scaled by a power of two to below 2^11 first; bf16: three), 22 or 24
// bits, summed in fp32.
//
// A few rows take one launch (lora_few_body), others two: t = A x, split over
// the inputs, then y, whose workgroups join the splits. us a call, one launch /
// two (fp16; "8 of 4" is 8 rows of 4 adapters):
//   rank 16, 4096 to 4096: 1 of 1 5.3 / 10.6, 4 of 4 5.8 / 11.3, 8 of 1 10.1 /
//   11.3, 16 of 16 7.9 / 18; 4096 to 14336: 4 of 4 6.0 / 11.6, 8 of 8 (448
//   workgroups) 11.6 / 13.9, 12 of 12 (672) 18.3 / 15.8; 14336 to 4096: 1 of 1
//   8.9 / 12.4, 4 of 4 9.6 / 13.3, 4 of 1 14.9 / 12.8; rank 64, 4096 to 4096: 4 of
//   4 10.9 / 13.4, 4 of 1 17.4 / 12.5; rank 8, 1536 to 8960: 16 of 16 (560) 16.5
//   / 18.
// So one launch pays while its waves have few rows' products to make in their
// lanes and the workgroups, each reading its adapter's A again, are not many.

// The valid adapter id of a row, or -1.
__device__ __forceinline__ int adapter_of(const sml_klora & a, int row) {
    const int id = a.adapter[min(max(row, 0), a.n_row - 1)];
    return row >= 0 && row < a.n_row && id >= 0 && id < a.n_adapter ? id : -1;
}
__device__ __forceinline__ int rank_of(const sml_klora & a, int id) {
    return a.ranks ? min(max(a.ranks[id], 0), a.rank) : a.rank;
}

// The rows of tile positions row0 .. row0 + nr - 1 into rows (-1 past the last):
// the caller's order, or (a.sorted) that of their adapters, rows without one
// last, so that a mixed batch's tiles hold few adapters each. A counting sort
// every workgroup makes for itself: 64 rows a wave, each distinct adapter's
// lanes by ballot; cnt holds (n_adapter + 1) counts of every 64 rows. It takes
// 1.7 us of a call's two launches, 0.6 where the rows lie in runs and stay. Rows
// of 16 adapters in turn, us a call in the caller's order / by adapter (4096 to
// 14336, rank 64): 32 rows 22.9 / 22.8, 64 29 / 23, 128 46 / 26, 509 92 / 36.
template <int NW>
__device__ __forceinline__ void tile_rows(const sml_klora & a, int row0, int nr, int * rows, int * cnt, int * wsum) {
    constexpr int PER = LS_ROWS / 64 / NW;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (!a.sorted) {
        if (tid < nr) rows[tid] = row0 + tid < a.n_row ? row0 + tid : -1;
        __syncthreads();
        return;
    }
    const int nch = (a.n_row + 63) / 64, m = (a.n_adapter + 1) * nch;
    int key[PER], rank[PER], turns = 0;
    #pragma unroll
    for (int i = 0; i < PER; i++) {
        const int row = 64 * (wave + NW * i) + lane;
        key[i] = -1;
        if (row < a.n_row) {
            key[i] = adapter_of(a, row);
            if (key[i] < 0) key[i] = a.n_adapter;
        }
        turns += __builtin_popcountll(__ballot(key[i] != __shfl_down(key[i], 1)));
    }
    if (!lane) wsum[wave] = turns;
    for (int i = tid; i < m; i += 64 * NW) cnt[i] = 0;
    __syncthreads();
    turns = 0;
    #pragma unroll
    for (int w = 0; w < NW; w++) turns += wsum[w];
    // runs already, as prompts come: at most about a change a tile
    const bool runs = 16 * turns <= a.n_row;
    if (tid < nr) rows[tid] = runs && row0 + tid < a.n_row ? row0 + tid : -1;
    __syncthreads();                                  // wsum is read by all
    if (runs) return;
    #pragma unroll
    for (int i = 0; i < PER; i++) {
        rank[i] = 0;
        for (unsigned long long left = __ballot(key[i] >= 0); left;) {
            const int cur = __builtin_amdgcn_readlane(key[i], __builtin_ctzll(left));
            const unsigned long long at = __ballot(key[i] == cur);
            left &= ~at;
            if (key[i] == cur) rank[i] = __builtin_amdgcn_mbcnt_hi((unsigned) (at >> 32), __builtin_amdgcn_mbcnt_lo((unsigned) at, 0));
            if (!lane) cnt[cur * nch + wave + NW * i] = __builtin_popcountll(at);
        }
    }
    __syncthreads();
    // exclusive sums, adapter by adapter
    const int each = (m + 64 * NW - 1) / (64 * NW), e0 = min(tid * each, m), e1 = min(e0 + each, m);
    int sum = 0;
    for (int i = e0; i < e1; i++) sum += cnt[i];
    int before = wave_scan(sum);
    if (lane == 63) wsum[wave] = before;
    before -= sum;
    __syncthreads();
    for (int w = 0; w < wave; w++) before += wsum[w];
    for (int i = e0; i < e1; i++) { const int v = cnt[i]; cnt[i] = before; before += v; }
    __syncthreads();
    #pragma unroll
    for (int i = 0; i < PER; i++)
        if (key[i] >= 0) {
            const int p = cnt[key[i] * nch + wave + NW * i] + rank[i] - row0;
            if (p >= 0 && p < nr) rows[p] = 64 * (wave + NW * i) + lane;
        }
    __syncthreads();
}

// The rows of a tile (bits of valid, id: the lane's) whose adapter is the z-th,
// z + nz-th, ... distinct one.
__device__ __forceinline__ unsigned long long my_rows(int id, unsigned long long valid, int z, int nz) {
    if (nz == 1) return valid;
    unsigned long long mine = 0;
    for (int k = 0; valid; k++) {
        const unsigned long long m = __ballot(id == __builtin_amdgcn_readlane(id, __builtin_ctzll(valid))) & valid;
        if (k % nz == z) mine |= m;
        valid &= ~m;
    }
    return mine;
}

// A x: a workgroup takes a tile of 16 rows, RT of 16 ranks and a split of the
// inputs, a wave every eighth 64 of those. The matrix cores want 16 rows in 16
// consecutive lanes, and loads in that order cost a cache line a lane (16
// bytes a cycle and CU measured): rows are loaded whole, 128 or 256 bytes in
// consecutive lanes, and handed over through the wave's part of LDS, at a
// stride of LD_ROW bytes that spreads 16 rows over all banks. 509 rows of 4096,
// rank 64: 8.4 us, of which a second adapter in a tile's rows takes 2; the
// reads of x alone (8 MB, each once) would be 2.
template <int BF, int RT>
__device__ __forceinline__ void lora_down_body(const sml_klora & a) {
    using M = Mx<BF>;
    typedef typename M::v8 v8;
    typedef typename M::t T;
    typedef T v4t __attribute__((ext_vector_type(4)));
    constexpr int NP = M::parts, NR = 16 * RT, RS = NR + 1;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint8_t * const la = lds + wave * LD_WAVE_LDS(NP, RT);          // [rank][LD_ROW]
    uint8_t * const lx = la + NR * LD_ROW;                          // [part][row][LD_ROW]
    int * const le = (int *) (lx + NP * 16 * LD_ROW);               // [row]
    const int split = blockIdx.x, row0 = blockIdx.y * 16, ngroup = (a.rank + NR - 1) / NR, nz = gridDim.z / ngroup;
    const int j0 = (blockIdx.z % ngroup) * NR, z = blockIdx.z / ngroup;
    const int k0 = split * a.chunk, k1 = min(a.n_in, k0 + a.chunk);
    __shared__ int rows[16], wsum[LD_WAVES];
    tile_rows<LD_WAVES>(a, row0, 16, rows, (int *) lds, wsum);
    const int id = adapter_of(a, rows[c]), nt = min(RT, (a.rank - j0 + 15) / 16);
    const unsigned all = (unsigned) my_rows(id, (unsigned) (__ballot(id >= 0) & 0xFFFFu), z, nz);
    if (!all) return;
    const int first = __builtin_amdgcn_readlane(id, __builtin_ctz(all));

    const float * xrow[4];
    #pragma unroll
    for (int i = 0; i < 4; i++) xrow[i] = a.x + (size_t) max(rows[4 * i + g], 0) * a.x_stride;
    v4f xr[4];
    v4u ar[2 * RT], an[2 * RT];
    auto load_x = [&](int kb) {
        const int kk = min(kb + 4 * c, k1 - 4);
        #pragma unroll
        for (int i = 0; i < 4; i++) xr[i] = *(const GLOBAL v4fu *) (xrow[i] + kk);
    };
    auto load_a = [&](v4u (&r)[2 * RT], int ad, int kb) {
        const int kk = min(kb + 8 * (lane & 7), k1 - 8);
        const uint16_t * w = a.a + (size_t) ad * a.rank * a.n_in + kk;
        #pragma unroll
        for (int i = 0; i < 2 * RT; i++)
            if (i < 2 * nt) r[i] = *(const GLOBAL v4u *) (w + (size_t) min(j0 + 8 * i + (lane >> 3), a.rank - 1) * a.n_in);
    };
    v4f tot[RT];
    #pragma unroll
    for (int t = 0; t < RT; t++) tot[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    int kb = k0 + wave * 64;
    if (kb < k1) { load_x(kb); load_a(ar, first, kb); }
    for (; kb < k1; kb += 64 * LD_WAVES) {
        // x's parts, each row scaled for fp16: 16 lanes a row
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            if (kb + 4 * c >= k1) xr[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            int ex = 0;
            if constexpr (!BF) {
                ex = scale_of(max16(fmaxf(fmaxf(fabsf(xr[i][0]), fabsf(xr[i][1])), fmaxf(fabsf(xr[i][2]), fabsf(xr[i][3])))));
                #pragma unroll
                for (int e = 0; e < 4; e++) xr[i][e] = __builtin_amdgcn_ldexpf(xr[i][e], -ex);
                if (!c) le[4 * i + g] = ex;
            }
            v8 p[NP];
            parts_of<BF>(xr[i][0], xr[i][1], p, 0);
            parts_of<BF>(xr[i][2], xr[i][3], p, 2);
            #pragma unroll
            for (int k = 0; k < NP; k++)
                *(v4t *) (lx + (k * 16 + 4 * i + g) * LD_ROW + 8 * c) = __builtin_shufflevector(p[k], p[k], 0, 1, 2, 3);
        }
        const int kn = kb + 64 * LD_WAVES;
        if (kn < k1) load_x(kn);
        // the tile's adapters one by one: each one's rows keep its products
        unsigned left = all;
        for (int cur = first; left;) {
            #pragma unroll
            for (int i = 0; i < 2 * RT; i++)
                if (i < 2 * nt) {
                    if (kb + 8 * (lane & 7) >= k1) ar[i] = v4u(0u);
                    *(v4u *) (la + (8 * i + (lane >> 3)) * LD_ROW + 16 * (lane & 7)) = ar[i];
                }
            wave_lds();
            const bool mine = id == cur;
            left &= ~(unsigned) __ballot(mine);
            const int then = left ? __builtin_amdgcn_readlane(id, __builtin_ctz(left)) : first;
            if (left || kn < k1) load_a(an, then, left ? kb : kn);
            const int ex = BF ? 0 : le[c];
            v8 xp[2][NP];
            #pragma unroll
            for (int s = 0; s < 2; s++)
                #pragma unroll
                for (int i = 0; i < NP; i++) xp[s][i] = *(const v8 *) (lx + (i * 16 + c) * LD_ROW + 64 * s + 16 * g);
            #pragma unroll
            for (int t = 0; t < RT; t++)
                if (t < nt) {
                    v4f acc = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                    #pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const v8 w = *(const v8 *) (la + (16 * t + c) * LD_ROW + 64 * s + 16 * g);
                        #pragma unroll
                        for (int i = 0; i < NP; i++) acc = M::mul(w, xp[s][i], acc);
                    }
                    #pragma unroll
                    for (int r = 0; r < 4; r++) tot[t][r] += mine ? __builtin_amdgcn_ldexpf(acc[r], ex) : 0.0f;
                }
            wave_lds();                               // all read before the next is written
            cur = then;
            #pragma unroll
            for (int i = 0; i < 2 * RT; i++) ar[i] = an[i];
        }
    }
    __syncthreads();                                  // the waves' parts become one
    float * const red = (float *) lds;                // [wave][row][RS]
    #pragma unroll
    for (int t = 0; t < RT; t++)
        #pragma unroll
        for (int r = 0; r < 4; r++) red[(wave * 16 + c) * RS + 16 * t + 4 * g + r] = tot[t][r];
    __syncthreads();
    for (int i = tid; i < 16 * NR; i += 64 * LD_WAVES) {
        const int rw = i / NR, j = i % NR;
        float s = 0.0f;
        #pragma unroll
        for (int v = 0; v < LD_WAVES; v++) s += red[(v * 16 + rw) * RS + j];
        if ((all >> rw & 1) && j0 + j < a.rank)
            a.work[((size_t) (row0 + rw) * a.nsplit + split) * a.rank + j0 + j] = s;
    }
}

// Both products of up to 16 rows in one launch: a workgroup of 16 waves computes
// t of one adapter's rows (all of n_in, the waves sharing it), then 256 outputs
// of theirs. Each workgroup reads its adapter's whole A again, from L2: less
// than a second launch costs while A is small. A step holds a row or two of an
// adapter, too few for the matrix cores' 16 columns (converting all 16 made
// this 12.6 us for 8.5): the first product is a lane's own fused multiply-adds
// on 8 inputs of 8 ranks at a time, summed over the wave by halves. 16 rows of
// 11 adapters, 4096 to 4096, rank 16: 8.4 us, a chain of latencies (ids, A and x,
// two exchanges in LDS, B) around 4 MB that would take 1; behind the L2s they are
// 15, since an adapter's output blocks lie on all XCDs, and each fetches its A
// and x.
template <int BF>
__device__ __forceinline__ void lora_few_body(const sml_klora & a) {
    using M = Mx<BF>;
    typedef typename M::v8 v8;
    typedef typename M::t T;
    constexpr int NP = M::parts, LD = LF_LD;
    extern __shared__ __align__(16) uint8_t lds[];
    T * const tp = (T *) lds;                         // [part][row][LD]
    int * const ex_s = (int *) (tp + NP * 16 * LD);   // [row]
    float * const red = (float *) (ex_s + 16);        // [slice][row][rank]
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nz = gridDim.y, z = blockIdx.y;
    const int o0 = blockIdx.x * LF_OUT + wave * 16, o = o0 + 4 * g, row = c;
    const int id = adapter_of(a, row), nrg = a.rank / 8, nslice = (a.n_in + LF_SLICE - 1) / LF_SLICE;
    const bool live = row < a.n_row;
    const float zero = a.base ? -0.0f : 0.0f;         // of outputs whose base follows behind: -0 leaves it as it is
    v4f base = v4f{zero, zero, zero, zero};
    if (a.base && live && o + 4 <= a.n_out) base = *(const v4fu *) (a.base + (size_t) row * a.y_stride + o);
    unsigned left = (unsigned) (__ballot(id >= 0) & 0xFFFFu);
    unsigned none = a.base == a.y ? 0u : (unsigned) (__ballot(id < 0 && live) & 0xFFFFu);
    for (int k = 0; left | none; k++) {
        int cur = -1;
        unsigned mine = none;
        if (left) {
            cur = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
            mine = (unsigned) (__ballot(id == cur) & 0xFFFFu);
            left &= ~mine;
        } else {
            none = 0;
        }
        if (k % nz != z) continue;
        v4f acc = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        int ex = 0;
        if (cur >= 0) {
            const int rk = rank_of(a, cur);
            const uint16_t * wa = a.a + (size_t) cur * a.rank * a.n_in, * wb = a.b + (size_t) cur * a.n_out * a.rank;
            v4u bw[2];
            #pragma unroll
            for (int s = 0; s < 2; s++) {
                const int kk = 32 * s + 8 * g;
                bw[s] = *(const GLOBAL v4u *) (wb + (size_t) min(o0 + c, a.n_out - 1) * a.rank + (kk < a.rank ? kk : 0));
            }
            for (int u = wave; u < nrg * nslice; u += LF_WAVES) {
                const int slice = u / nrg, rg = u - slice * nrg, kk = LF_SLICE * slice + 8 * lane;
                const bool in = kk < a.n_in;
                v4u w[8];
                #pragma unroll
                for (int i = 0; i < 8; i++) w[i] = *(const GLOBAL v4u *) (wa + (size_t) (8 * rg + i) * a.n_in + (in ? kk : 0));
                for (unsigned m = mine; m; m &= m - 1) {
                    const int r = __builtin_ctz(m);
                    const float * x = a.x + (size_t) r * a.x_stride + (in ? kk : 0);
                    const v4f x0 = *(const GLOBAL v4fu *) x, x1 = *(const GLOBAL v4fu *) (x + 4);
                    float t[8];
                    #pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const v8 h = __builtin_bit_cast(v8, w[i]);
                        t[i] = 0.0f;
                        #pragma unroll
                        for (int e = 0; e < 4; e++) {
                            t[i] = __builtin_fmaf((float) h[e], x0[e], t[i]);
                            t[i] = __builtin_fmaf((float) h[e + 4], x1[e], t[i]);
                        }
                        if (!in) t[i] = 0.0f;
                    }
                    // 8 sums over 64 lanes: lane l ends with that of 4 l5 + 2 l4 + l3
                    #pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float s = lane & 32 ? t[i] : t[i + 4];
                        t[i] = (lane & 32 ? t[i + 4] : t[i]) + __shfl_xor(s, 32);
                    }
                    #pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float s = lane & 16 ? t[i] : t[i + 2];
                        t[i] = (lane & 16 ? t[i + 2] : t[i]) + __shfl_xor(s, 16);
                    }
                    const float s = lane & 8 ? t[0] : t[1];
                    t[0] = (lane & 8 ? t[1] : t[0]) + __shfl_xor(s, 8);
                    t[0] += dpp_f<0xB1>(t[0]); t[0] += dpp_f<0x4E>(t[0]); t[0] += dpp_f<0x141>(t[0]);
                    if (!(lane & 7)) red[(slice * 16 + r) * a.rank + 8 * rg + (lane >> 3 & 1) + 2 * (lane >> 4 & 1) + 4 * (lane >> 5)] = t[0];
                }
            }
            __syncthreads();
            // wave w joins row w: lane j its rank j
            if (mine >> wave & 1) {
                float v = 0.0f;
                if (lane < rk)
                    for (int s = 0; s < nslice; s++) v += red[(s * 16 + wave) * a.rank + lane];
                v *= a.scale ? a.scale[cur] : 1.0f;
                const int et = BF ? 0 : scale_of(wave_max(fabsf(v)));
                v8 p[NP];
                parts_of<BF>(__builtin_amdgcn_ldexpf(v, -et), 0.0f, p, 0);
                #pragma unroll
                for (int i = 0; i < NP; i++) tp[(i * 16 + wave) * LD + lane] = p[i][0];
                if (!lane) ex_s[wave] = et;
            }
            __syncthreads();
            #pragma unroll
            for (int s = 0; s < 2; s++)
                if (32 * s < rk) {
                    const int kk = 32 * s + 8 * g;
                    #pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int j = kk + 2 * i;
                        bw[s][i] = j + 1 < rk ? bw[s][i] : j < rk ? bw[s][i] & 0xFFFFu : 0u;
                    }
                    #pragma unroll
                    for (int i = 0; i < NP; i++)
                        acc = M::mul(__builtin_bit_cast(v8, bw[s]), *(const v8 *) (tp + (i * 16 + c) * LD + kk), acc);
                }
            ex = ex_s[c];
            __syncthreads();                          // red and tp are the next adapter's
        }
        if (!(mine >> c & 1) || o >= a.n_out) continue;
        float * y = a.y + (size_t) row * a.y_stride + o;
        v4f d;
        #pragma unroll
        for (int r = 0; r < 4; r++) d[r] = base[r] + (cur < 0 ? -0.0f : __builtin_amdgcn_ldexpf(acc[r], ex));
        if (o + 4 <= a.n_out) *(v4fu *) y = d;
        else
            for (int r = 0; r < 3; r++)
                if (o + r < a.n_out) y[r] = d[r] + (a.base ? a.base[(size_t) row * a.y_stride + o + r] : -0.0f);
    }
}

// A workgroup takes RB tiles of 16 rows and, wave by wave, every so many blocks
// of 64 outputs: t is joined, scaled and split into parts in LDS once, and the
// waves then stream B and the base past it with no barrier, the next block's
// on their way before the present one's products. Rows are the products'
// rows, and column c of product u is output 4c + u of the block: a lane then
// holds four outputs side by side and 16 lanes 256 bytes of a row. B's rows
// come through the wave's part of LDS as A's do above. 509 rows to 14336, rank
// 64: 22 us, 58 MB of base and y at 2.7 TB/s: about 3 us join t's splits ahead of
// the first product, and tiles that hold two adapters take 4 more.
template <int BF, int RB>
__device__ __forceinline__ void lora_up_body(const sml_klora & a) {
    using M = Mx<BF>;
    typedef typename M::v8 v8;
    typedef typename M::t T;
    typedef T v4t __attribute__((ext_vector_type(4)));
    extern __shared__ __align__(16) uint8_t lds[];
    constexpr int NR = 16 * RB, NP = M::parts;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nz = gridDim.z, z = blockIdx.z;
    uint8_t * const lb = lds + wave * LU_OUT * LD_ROW;              // [16 u + c][LD_ROW], output 4c + u
    int * const ex_s = (int *) (lds + 4 * LU_OUT * LD_ROW);         // [row]
    T * const tp = (T *) (ex_s + NR);                               // [part][row][ld]
    const int ld = (a.rank + 63) / 64 * 64 + 8, row0 = blockIdx.y * NR;

    __shared__ int rows[NR], wsum[4];
    tile_rows<4>(a, row0, NR, rows, (int *) lds, wsum);
    const int myrow = lane < NR ? rows[lane] : -1;

    // the rows of this workgroup: of its adapters and, once, those without
    const int id = adapter_of(a, myrow);
    const unsigned long long valid = my_rows(id, __ballot(id >= 0), z, nz);
    const unsigned long long all = valid | (z || a.base == a.y ? 0 : __ballot(id < 0 && myrow >= 0));
    if (!all) return;
    const int rk_l = id < 0 ? 0 : rank_of(a, id);     // of the lane's row
    const float sc_l = id < 0 || !a.scale ? 1.0f : a.scale[id];
    const int first = valid ? __builtin_amdgcn_readlane(id, __builtin_ctzll(valid)) : -1;
    const unsigned long long mine4 = all >> (4 * g);  // bit 16h + r: row 16h + 4g + r

    int yrow[RB][4];                                  // row of position 16h + 4g + r
    #pragma unroll
    for (int h = 0; h < RB; h++)
        #pragma unroll
        for (int r = 0; r < 4; r++) yrow[h][r] = rows[16 * h + 4 * g + r];

    const int jump = gridDim.x * 4 * LU_OUT;
    v4u br[8];
    v4f base[RB][4], bn[RB][4];
    // 64 outputs' ranks k0.. (up to 64), 8 lanes a row
    auto load_b = [&](int ad, int o0, int k0) {
        const int kk = k0 + 8 * (lane & 7);
        const uint16_t * b = a.b + (size_t) max(ad, 0) * a.n_out * a.rank + (kk < a.rank ? kk : 0);
        #pragma unroll
        for (int i = 0; i < 8; i++) br[i] = *(const GLOBAL v4u *) (b + (size_t) min(o0 + 8 * i + (lane >> 3), a.n_out - 1) * a.rank);
    };
    // adding -0 leaves any sum as it is: what other rows' adapters add, and
    // where the last outputs' base follows behind
    const float zero = a.base ? -0.0f : 0.0f;
    auto load_base = [&](v4f (&v)[RB][4], int o0) {
        const int o = o0 + 4 * c;
        #pragma unroll
        for (int h = 0; h < RB; h++)
            #pragma unroll
            for (int r = 0; r < 4; r++) {
                v[h][r] = v4f{zero, zero, zero, zero};
                if (a.base && (mine4 >> (16 * h + r) & 1) && o + 4 <= a.n_out)
                    v[h][r] = *(const GLOBAL v4fu *) (a.base + (size_t) yrow[h][r] * a.y_stride + o);
            }
    };
    int o0 = (blockIdx.x * 4 + wave) * LU_OUT;
    if (o0 < a.n_out) { load_base(base, o0); load_b(first, o0, 0); }     // neither needs t

    // t's rows: lr lanes of 4 values each, times sg lanes that share the splits
    // where the tile leaves threads over; up to four rows a thread at once
    int lr = 2;
    while (4 * lr < a.rank) lr *= 2;
    const int sg = max(256 / NR / lr, 1), lanes = lr * sg;
    const int q = tid & (lr - 1), s0 = tid / lr & (sg - 1), step = 256 / lanes;
    const bool inq = 4 * q < a.rank;
    // zeros from the rank to the next multiple of 64
    for (int i = tid, n8 = (ld - 8 - a.rank) / 8; i < NP * NR * n8; i += 256)
        *(v4u *) (tp + (size_t) (i / n8) * ld + a.rank + 8 * (i % n8)) = v4u(0u);
    for (int r0 = tid / lanes; r0 < NR; r0 += 4 * step) {
        v4f v[4];
        #pragma unroll
        for (int i = 0; i < 4; i++) v[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        #pragma unroll 4
        for (int s = s0; s < a.nsplit; s += sg)
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = row0 + r0 + i * step;
                if (r0 + i * step < NR && row < a.n_row && inq)
                    v[i] += *(const v4fu *) (a.work + ((size_t) row * a.nsplit + s) * a.rank + 4 * q);
            }
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = r0 + i * step;
            const int rr = __shfl(rk_l, r & 63);
            const float sc = __shfl(sc_l, r & 63);
            for (int o = lr; o < lanes; o *= 2)
                #pragma unroll
                for (int e = 0; e < 4; e++) v[i][e] += __shfl_xor(v[i][e], o);
            float mx = 0.0f;
            #pragma unroll
            for (int e = 0; e < 4; e++) { v[i][e] = 4 * q + e < rr ? v[i][e] * sc : 0.0f; mx = fmaxf(mx, fabsf(v[i][e])); }
            int ex = 0;
            if constexpr (!BF) {
                for (int o = 1; o < lr; o *= 2) mx = fmaxf(mx, __shfl_xor(mx, o));
                ex = scale_of(mx);
            }
            v8 p[NP];
            #pragma unroll
            for (int e = 0; e < 4; e += 2)
                parts_of<BF>(__builtin_amdgcn_ldexpf(v[i][e], -ex), __builtin_amdgcn_ldexpf(v[i][e + 1], -ex), p, e);
            if (r < NR && inq && !s0) {
                #pragma unroll
                for (int k = 0; k < NP; k++)
                    *(v4t *) (tp + ((size_t) k * NR + r) * ld + 4 * q) = __builtin_shufflevector(p[k], p[k], 0, 1, 2, 3);
            }
            if (r < NR && !(tid & (lanes - 1))) ex_s[r] = ex;
        }
    }
    __syncthreads();
    int idr[RB][4], ex[RB][4];                        // of row 16h + 4g + r
    #pragma unroll
    for (int h = 0; h < RB; h++)
        #pragma unroll
        for (int r = 0; r < 4; r++) { idr[h][r] = __shfl(id, 16 * h + 4 * g + r); ex[h][r] = ex_s[16 * h + 4 * g + r]; }
    for (; o0 < a.n_out; o0 += jump) {
        const bool more = o0 + jump < a.n_out;
        if (more) load_base(bn, o0 + jump);
        // the tile's adapters one by one: each one's rows take its products
        unsigned long long left = valid;
        int cur = first;
        while (left) {
            const int rk = rank_of(a, cur);
            const unsigned long long rest = left & ~__ballot(id == cur);
            const int then = rest ? __builtin_amdgcn_readlane(id, __builtin_ctzll(rest)) : first;
            v4f acc[RB][4];
            #pragma unroll
            for (int h = 0; h < RB; h++)
                #pragma unroll
                for (int u = 0; u < 4; u++) acc[h][u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            int k0 = 0;
            do {
                // zeros past the adapter's rank (t is zero there too), output
                // 8i + l/8 of the block to its product's row
                const int keep = rk - k0 - 8 * (lane & 7);
                #pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (keep < 8) {
                        #pragma unroll
                        for (int e = 0; e < 4; e++) br[i][e] = 2 * e + 1 < keep ? br[i][e] : 2 * e < keep ? br[i][e] & 0xFFFFu : 0u;
                    }
                    const int o = 8 * i + (lane >> 3);
                    *(v4u *) (lb + (16 * (o & 3) + (o >> 2)) * LD_ROW + 16 * (lane & 7)) = br[i];
                }
                wave_lds();
                const int kc = k0;
                k0 += 64;
                if (k0 < rk) load_b(cur, o0, k0);
                else if (rest || more) load_b(then, rest ? o0 : o0 + jump, 0);
                #pragma unroll
                for (int s = 0; s < 2; s++)
                    if (kc + 32 * s < rk) {
                        v8 w[4];
                        #pragma unroll
                        for (int u = 0; u < 4; u++) w[u] = *(const v8 *) (lb + (16 * u + c) * LD_ROW + 64 * s + 16 * g);
                        #pragma unroll
                        for (int h = 0; h < RB; h++)
                            #pragma unroll
                            for (int i = 0; i < NP; i++) {
                                const v8 tv = *(const v8 *) (tp + ((size_t) i * NR + 16 * h + c) * ld + kc + 32 * s + 8 * g);
                                #pragma unroll
                                for (int u = 0; u < 4; u++) acc[h][u] = M::mul(tv, w[u], acc[h][u]);
                            }
                    }
                wave_lds();                           // all read before the next is written
            } while (k0 < rk);
            #pragma unroll
            for (int h = 0; h < RB; h++)
                #pragma unroll
                for (int r = 0; r < 4; r++)
                    #pragma unroll
                    for (int u = 0; u < 4; u++) base[h][r][u] += idr[h][r] == cur ? __builtin_amdgcn_ldexpf(acc[h][u][r], ex[h][r]) : -0.0f;
            left = rest;
            cur = then;
        }
        const int o = o0 + 4 * c;
        #pragma unroll
        for (int h = 0; h < RB; h++)
            #pragma unroll
            for (int r = 0; r < 4; r++) {
                const size_t at = (size_t) yrow[h][r] * a.y_stride + o;
                if (!(mine4 >> (16 * h + r) & 1)) continue;
                if (o + 4 <= a.n_out) *(GLOBAL v4fu *) (a.y + at) = base[h][r];
                else
                    for (int e = 0; e < 3; e++)
                        if (o + e < a.n_out) a.y[at + e] = base[h][r][e] + (a.base ? a.base[at + e] : -0.0f);
            }
        #pragma unroll
        for (int h = 0; h < RB; h++)
            #pragma unroll
            for (int r = 0; r < 4; r++) base[h][r] = bn[h][r];
    }
}
#define LORA(BF, sfx) \
    extern "C" __global__ __launch_bounds__(64 * LD_WAVES) void sml_sv_lora_down2##sfx(const sml_klora a) { lora_down_body<BF, 2>(a); } \
    extern "C" __global__ __launch_bounds__(64 * LD_WAVES) void sml_sv_lora_down1##sfx(const sml_klora a) { lora_down_body<BF, 1>(a); } \
    extern "C" __global__ __launch_bounds__(256) void sml_sv_lora_up2##sfx(const sml_klora a) { lora_up_body<BF, 2>(a); } \
    extern "C" __global__ __launch_bounds__(256) void sml_sv_lora_up1##sfx(const sml_klora a) { lora_up_body<BF, 1>(a); } \
    extern "C" __global__ __launch_bounds__(64 * LF_WAVES) void sml_sv_lora_few##sfx(const sml_klora a) { lora_few_body<BF>(a); }
LORA(0, )
LORA(1, _bf)
