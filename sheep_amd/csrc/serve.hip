// Kernels of a step that serves many requests at once (sml-serve.h): the paged
// cache's append and attention, low-rank adapters, and the rules on logits.
#include "dev.h"

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
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

// The page of entry i of sequence s, or -1.
__device__ __forceinline__ int page_of(const sml_kpages & pg, int s, int i) {
    const int p = pg.table[(size_t) s * pg.seq_pages + i];
    return p >= 0 && p < pg.n_pages ? p : -1;
}

// ---------------------------------------------------------------- append
//
// A thread takes four rotation pairs (d, d + hd/2) of one head of q or k, or
// four values of v. The pair's products are the decode kernels' (one rounded,
// the other fused), so a float16 cache equals the contiguous one.
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
// registers (no LDS until the waves' sums are joined). The matrix cores take
// S^T = K Q^T and O^T = V^T P^T, heads in the columns (the unused of the 16
// are zero). With the lane's c = lane % 16, g = lane / 16:
// - K is the first operand as the cache stores it: lane (c, g) loads 16 bytes
//   of position c's row, dims 32j + 8g.. for product j.
// - S comes back as positions 4g + r of head c, which is just what the second
//   product takes as its P^T operand if its inner index 8g + i stands for
//   position 4g + i of the first 16 positions (i < 4) or of the second: P
//   never crosses lanes.
// - V's rows of those 8 positions are loaded whole, 16 lanes a row, dims
//   (D/16)c.. each; the product u takes dim (D/16)c + u of every lane, so V^T
//   is 4 D/16 byte permutes in the lane, and lane (c, g) ends with dims
//   (D/4)g.. of head c: the base's rescaling is a lane's own too.
// q and the weights are split into parts of the cache's type (two of fp16,
// three of bf16: 22 and 24 bits), a matrix instruction each; q's row is scaled
// by a power of two to below 2^11 first so that fp16 holds it. The base
// starts 10 below the first maximum and moves when a score passes it by 15:
// weights then lie up to 2^15, fp16's range, and those that its smallest
// steps round are 2^-34 of the largest.
//
// Pages are looked up a tile ahead, once per 16 positions (a page is a
// multiple of 16). Positions past the length or on absent pages are loaded
// from where memory is (the rest of the page, or page 0), their scores
// replaced by -infinity and their V rows by zeros; tiles of absent pages alone
// are passed over.
#define AT_WAVES 4

template <int BF> struct Mx;
template <> struct Mx<0> {
    typedef _Float16 t;
    typedef t v8 __attribute__((ext_vector_type(8)));
    static constexpr int parts = 2;
    static __device__ __forceinline__ v4f mul(v8 a, v8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mx<1> {
    typedef __bf16 t;
    typedef t v8 __attribute__((ext_vector_type(8)));
    static constexpr int parts = 3;
    static __device__ __forceinline__ v4f mul(v8 a, v8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// Powers of two: the one that brings values up to mx below 2^11, and back.
__device__ __forceinline__ int scale_of(float mx) {
    return mx > 0.0f && mx < INFINITY ? __builtin_amdgcn_frexp_expf(mx) - 11 : 0;
}

// element e of the parts of x: each part the rounding of what is left
template <int BF>
__device__ __forceinline__ void parts_of(float x, typename Mx<BF>::v8 (&p)[Mx<BF>::parts], int e) {
    #pragma unroll
    for (int k = 0; k < Mx<BF>::parts; k++) {
        const typename Mx<BF>::t h = (typename Mx<BF>::t) x;
        p[k][e] = h;
        x -= (float) h;
    }
}

template <int D, int BF>
__device__ __forceinline__ void attend_body(const sml_kattend & a) {
    using M = Mx<BF>;
    typedef typename M::v8 v8;
    constexpr int NJ = D / 32, E = D / 16, NP = M::parts, W = AT_WAVES;
    typedef unsigned vrow __attribute__((ext_vector_type(E / 2)));
    __shared__ float so[W][16][D + 4], sm[W][16], sl[W][16];
    const int kh = blockIdx.x, split = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 15, g = lane >> 4;
    const int n = min(a.len[b], a.max_len), t0 = split * a.chunk, t1 = min(n, t0 + a.chunk);
    if (t0 >= t1 && a.nsplit > 1) return;             // the merge takes the splits below the length only
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
        const int ex = scale_of(mx);
        #pragma unroll
        for (int j = 0; j < NJ; j++)
            #pragma unroll
            for (int e = 0; e < 8; e++) parts_of<BF>(__builtin_amdgcn_ldexpf(x[j][e], -ex), q[j], e);
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
    v4u kr[2][NJ];
    vrow vr[8];
    const uint32_t koff = 2u * (uint32_t) (c * kvd + 8 * g);
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
            for (int j = 0; j < NJ; j++) kr[h][j] = *(const GLOBAL v4u *) (p + koff + 64 * j);
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
        v4f s[2];
        #pragma unroll
        for (int h = 0; h < 2; h++) {
            s[h] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            #pragma unroll
            for (int j = 0; j < NJ; j++)
                #pragma unroll
                for (int k = 0; k < NP; k++) s[h] = M::mul(__builtin_bit_cast(v8, kr[h][j]), q[j][k], s[h]);
        }
        if (tn < t1) load_k(xa, xb);
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
        if (__any(mx > base + 15.0f)) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float to = mx > base + 15.0f ? mx - 10.0f : base;
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
            for (int r = 0; r < 4; r++) {
                const float w = __builtin_amdgcn_exp2f(s[h][r] - bu);
                l += w;
                parts_of<BF>(w, p, 4 * h + r);
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
        if (a.nsplit == 1) {
            a.out[(row0 + h) * D + d] = ls == 0.0f ? 0.0f : os / ls;
        } else {
            const size_t at = (row0 + h) * a.nsplit + split;
            a.part[at * D + d] = os;
            if (!d) *(float2 *) (a.part + (size_t) a.pg.n_seq * a.n_head * a.nsplit * D + 2 * at) = make_float2(m, ls);
        }
    }
}

// The splits of a row joined: a workgroup a (sequence, head), D threads a
// share of its splits.
#define AM_THREADS 256
template <int D>
__device__ __forceinline__ void attend_merge_body(const sml_kattend & a) {
    constexpr int S = AM_THREADS / D;                 // shares
    __shared__ float f[256], red[S][D], sred[AM_THREADS / 64];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int n = min(a.len[b], a.max_len), ns = n > 0 ? (n + a.chunk - 1) / a.chunk : 0;
    const size_t row = (size_t) b * a.n_head + h;
    const float * po = a.part + row * a.nsplit * D;
    const float2 * pm = (const float2 *) (a.part + (size_t) a.pg.n_seq * a.n_head * a.nsplit * D) + row * a.nsplit;
    const float2 ml = tid < ns ? pm[tid] : make_float2(-INFINITY, 0.0f);
    float m = wave_max(ml.x);
    if (!(tid & 63)) sred[tid >> 6] = m;
    __syncthreads();
    m = sred[0];
    #pragma unroll
    for (int w = 1; w < AM_THREADS / 64; w++) m = fmaxf(m, sred[w]);
    const float e = __builtin_amdgcn_exp2f(ml.x - (m == -INFINITY ? 0.0f : m));
    f[tid] = e;
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
    for (int w = 0; w < AM_THREADS / 64; w++) l += sred[w];
    #pragma unroll
    for (int s = 1; s < S; s++) o += red[s][d];
    a.out[row * D + d] = l == 0.0f ? 0.0f : o / l;
}
extern "C" __global__ __launch_bounds__(AM_THREADS) void sml_sv_merge(const sml_kattend a) { attend_merge_body<128>(a); }
extern "C" __global__ __launch_bounds__(AM_THREADS) void sml_sv_merge_d64(const sml_kattend a) { attend_merge_body<64>(a); }

#define ATTEND(D, BF, name) \
    extern "C" __global__ __launch_bounds__(64 * AT_WAVES) void name(const sml_kattend a) { attend_body<D, BF>(a); }
ATTEND(128, 0, sml_sv_attend)
ATTEND(128, 1, sml_sv_attend_bf)
ATTEND(64, 0, sml_sv_attend_d64)
ATTEND(64, 1, sml_sv_attend_d64_bf)

// ---------------------------------------------------------------- logits
//
// A workgroup takes LG_RANGE tokens of a row. It counts the row's history and
// finds the biases of its own tokens in LDS (whole numbers, so the order of
// the atomics does not show), then applies the rules to its logits in the
// order the header gives, with no contraction, and keeps the greedy pick's
// candidate.
#define LG_RANGE 4096
#define LG_SEEN 0x80000000u

__device__ __forceinline__ void amax_take(float v, int i, float & bv, int & bi) {
    if (v > bv || (v == bv && i < bi)) { bv = v; bi = i; }
}

extern "C" __global__ __launch_bounds__(256) void sml_sv_logits(const sml_klogits a) {
    #pragma clang fp contract(off)
    __shared__ unsigned cnt[LG_RANGE];                // generated count, LG_SEEN if listed at all
    __shared__ int bia[LG_RANGE];                     // the last bias entry's index + 1
    __shared__ float bv_s[4];
    __shared__ int bi_s[4], fi_s[4], fn_s[4];
    const int row = blockIdx.y, t0 = blockIdx.x * LG_RANGE, tid = threadIdx.x;
    const int nt = min(LG_RANGE, a.n_vocab - t0);
    for (int i = tid; i < LG_RANGE; i += 256) { cnt[i] = 0; bia[i] = 0; }
    __syncthreads();
    if (a.hist) {
        const int h0 = min(max(a.hist_start[row], 0), a.n_hist), h1 = min(max(a.hist_start[row + 1], 0), a.n_hist);
        const int np = a.n_prompt ? a.n_prompt[row] : 0;
        for (int i = h0 + tid; i < h1; i += 256) {
            const int t = a.hist[i];
            if (t < t0 || t - t0 >= nt) continue;
            if (i - h0 >= np) atomicAdd(&cnt[t - t0], 1u);
            atomicOr(&cnt[t - t0], LG_SEEN);
        }
    }
    if (a.bias) {
        const int b0 = min(max(a.bias_start[row], 0), a.n_bias), b1 = min(max(a.bias_start[row + 1], 0), a.n_bias);
        for (int i = b0 + tid; i < b1; i += 256) {
            const int t = a.bias_id[i];
            if (t >= t0 && t - t0 < nt) atomicMax(&bia[t - t0], i + 1);
        }
    }
    __syncthreads();
    const float rep = a.rep ? a.rep[row] : 1.0f, fr = a.frequency ? a.frequency[row] : 0.0f,
                pr = a.presence ? a.presence[row] : 0.0f;
    const int mr = !a.mask ? -1 : a.mask_row ? a.mask_row[row] : row;
    const bool none = mr < -1 || mr >= a.n_mask;
    const uint32_t * mask = mr < 0 || none ? nullptr : a.mask + (size_t) mr * ((a.n_vocab + 31) / 32);
    float bv = -INFINITY;
    int bi = 0x7fffffff, fi = 0x7fffffff, fn = 0;
    for (int j = tid; j < nt; j += 256) {
        const int t = t0 + j;
        float l = a.logits[(size_t) row * a.stride + t];
        const unsigned c = cnt[j];
        if (c) {
            if (a.rep) l = l > 0.0f ? l / rep : l * rep;
            if (c & ~LG_SEEN) {
                if (a.frequency) l = l - fr * (float) (c & ~LG_SEEN);
                if (a.presence) l = l - pr;
            }
        }
        if (bia[j]) l = l + a.bias[bia[j] - 1];
        const bool ok = a.mask == nullptr || mr == -1 || (mask && (mask[t >> 5] >> (t & 31) & 1));
        if (a.out) a.out[(size_t) row * a.out_stride + t] = ok ? l : -INFINITY;
        if (ok) {
            if (fi == 0x7fffffff) { fi = t; fn = l != l; }
            amax_take(l, t, bv, bi);
        }
    }
    if (!a.tok) return;
    #pragma unroll
    for (int o = 32; o; o >>= 1) {
        const float ov = __shfl_xor(bv, o);
        const int oi = __shfl_xor(bi, o), of = __shfl_xor(fi, o), on = __shfl_xor(fn, o);
        amax_take(ov, oi, bv, bi);
        if (of < fi) { fi = of; fn = on; }
    }
    if ((tid & 63) == 0) { bv_s[tid >> 6] = bv; bi_s[tid >> 6] = bi; fi_s[tid >> 6] = fi; fn_s[tid >> 6] = fn; }
    __syncthreads();
    if (tid) return;
    for (int w = 1; w < 4; w++) {
        amax_take(bv_s[w], bi_s[w], bv, bi);
        if (fi_s[w] < fi) { fi = fi_s[w]; fn = fn_s[w]; }
    }
    a.part[(size_t) row * a.n_part + blockIdx.x] = make_int4(__float_as_int(bv), bi, fi, fn);
}

// The pick over a row's blocks: the first permitted token if it is NaN (the
// serial loop never leaves it), else the lowest index of the largest value.
extern "C" __global__ __launch_bounds__(64) void sml_sv_pick(const sml_klogits a) {
    const int row = blockIdx.x;
    float bv = -INFINITY;
    int bi = 0x7fffffff, fi = 0x7fffffff, fn = 0;
    for (int i = threadIdx.x; i < a.n_part; i += 64) {
        const int4 p = a.part[(size_t) row * a.n_part + i];
        amax_take(__int_as_float(p.x), p.y, bv, bi);
        if (p.z < fi) { fi = p.z; fn = p.w; }
    }
    #pragma unroll
    for (int o = 32; o; o >>= 1) {
        const float ov = __shfl_xor(bv, o);
        const int oi = __shfl_xor(bi, o), of = __shfl_xor(fi, o), on = __shfl_xor(fn, o);
        amax_take(ov, oi, bv, bi);
        if (of < fi) { fi = of; fn = on; }
    }
    if (!threadIdx.x) a.tok[row] = fi == 0x7fffffff ? -1 : fn ? fi : bi;
}

// ---------------------------------------------------------------- adapters
//
// y = base + scale B (A x), two launches: t = A x of every row under its own
// adapter (split over the inputs, joined by the second launch's prologue), then
// y. Rows come in tiles of 16, the matrix cores' columns: a workgroup takes the
// distinct adapters among its tile's rows one by one, computes all columns
// with each and stores those of its rows. Columns never mix, so a row sees
// nothing of the others, and no sorting of requests is needed: requests that
// share an adapter in a tile read it once, those that do not read each their
// own, which is the least there is to read.
//
// fp32 x and t meet the 16-bit matrices as parts of their type (fp16: two, and
// each row scaled by a power of two to below 2^11 first; bf16: three), 22 or 24
// bits, summed in fp32.
#define LD_WAVES 8
#define LD_STEPS 4                                    // inner products of 32 a wave holds at once
#define LD_TILE (LD_WAVES * LD_STEPS * 32)            // inputs a workgroup takes at once

// The valid adapter id of a row, or -1.
__device__ __forceinline__ int adapter_of(const sml_klora & a, int row) {
    const int id = row < a.n_row ? a.adapter[row] : -1;
    return id >= 0 && id < a.n_adapter ? id : -1;
}
__device__ __forceinline__ int rank_of(const sml_klora & a, int id) {
    return a.ranks ? min(max(a.ranks[id], 0), a.rank) : a.rank;
}

template <int BF, int RT>
__device__ __forceinline__ void lora_down_body(const sml_klora & a) {
    using M = Mx<BF>;
    typedef typename M::v8 v8;
    __shared__ float red[LD_WAVES][16][16 * RT + 1];
    const int row0 = blockIdx.x * 16, split = blockIdx.y, tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int ngroup = (a.rank + 16 * RT - 1) / (16 * RT), nz = gridDim.z / ngroup;
    const int j0 = (blockIdx.z % ngroup) * 16 * RT, z = blockIdx.z / ngroup;
    const int k0 = split * a.chunk, k1 = min(a.n_in, k0 + a.chunk);
    const int id = adapter_of(a, row0 + c);
    const float * x = a.x + (size_t) min(row0 + c, a.n_row - 1) * a.x_stride;

    unsigned left = (unsigned) (__ballot(id >= 0) & 0xFFFFu);
    for (int k = 0; left; k++) {
        const int cur = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
        const unsigned mine = (unsigned) (__ballot(id == cur) & 0xFFFFu);
        left &= ~mine;
        if (k % nz != z) continue;
        const int rk = rank_of(a, cur);
        if (j0 >= rk) continue;
        const int nt = min(RT, (rk - j0 + 15) / 16);
        const uint16_t * w = a.a + (size_t) cur * a.rank * a.n_in;
        v4f tot[RT];
        #pragma unroll
        for (int t = 0; t < RT; t++) tot[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        for (int kb = k0 + wave * 32 * LD_STEPS; kb < k1; kb += LD_TILE) {
            float xv[LD_STEPS][8], mx = 0.0f;
            v4u wv[RT][LD_STEPS];
            #pragma unroll
            for (int s = 0; s < LD_STEPS; s++) {
                const int kk = kb + 32 * s + 8 * g;
                #pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const v4f v = *(const GLOBAL v4fu *) (x + (kk < k1 ? kk + e : 0));
                    #pragma unroll
                    for (int i = 0; i < 4; i++) xv[s][e + i] = kk < k1 ? v[i] : 0.0f;
                }
            }
            #pragma unroll
            for (int t = 0; t < RT; t++)
                if (t < nt) {
                    const uint16_t * wr = w + (size_t) min(j0 + 16 * t + c, rk - 1) * a.n_in;
                    #pragma unroll
                    for (int s = 0; s < LD_STEPS; s++) {
                        const int kk = kb + 32 * s + 8 * g;
                        wv[t][s] = *(const GLOBAL v4u *) (wr + (kk < k1 ? kk : 0));
                        if (kk >= k1) wv[t][s] = v4u(0u);
                    }
                }
            #pragma unroll
            for (int s = 0; s < LD_STEPS; s++)
                #pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(xv[s][e]));
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const int ex = BF ? 0 : scale_of(mx);
            v8 p[LD_STEPS][M::parts];
            #pragma unroll
            for (int s = 0; s < LD_STEPS; s++)
                #pragma unroll
                for (int e = 0; e < 8; e++) parts_of<BF>(__builtin_amdgcn_ldexpf(xv[s][e], -ex), p[s], e);
            #pragma unroll
            for (int t = 0; t < RT; t++)
                if (t < nt) {
                    v4f acc = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                    #pragma unroll
                    for (int s = 0; s < LD_STEPS; s++)
                        #pragma unroll
                        for (int i = 0; i < M::parts; i++) acc = M::mul(__builtin_bit_cast(v8, wv[t][s]), p[s][i], acc);
                    #pragma unroll
                    for (int r = 0; r < 4; r++) tot[t][r] += __builtin_amdgcn_ldexpf(acc[r], ex);
                }
        }
        #pragma unroll
        for (int t = 0; t < RT; t++)
            #pragma unroll
            for (int r = 0; r < 4; r++) red[wave][c][16 * t + 4 * g + r] = tot[t][r];
        __syncthreads();
        for (int i = tid; i < 256 * RT; i += 64 * LD_WAVES) {
            const int rw = i / (16 * RT), j = i % (16 * RT);
            float s = 0.0f;
            #pragma unroll
            for (int v = 0; v < LD_WAVES; v++) s += red[v][rw][j];
            if ((mine >> rw & 1) && j0 + j < rk)
                a.work[((size_t) (row0 + rw) * a.nsplit + split) * a.rank + j0 + j] = s;
        }
        __syncthreads();
    }
}

// RB tiles of 16 rows and 4 waves of OT tiles of 16 outputs a workgroup.
template <int BF, int RB, int OT>
__device__ __forceinline__ void lora_up_body(const sml_klora & a) {
    using M = Mx<BF>;
    typedef typename M::v8 v8;
    typedef typename M::t T;
    extern __shared__ __align__(16) uint8_t lds[];
    constexpr int NR = 16 * RB, NP = M::parts;
    const int ld = a.rank + 8;                        // values of a row of t's parts in LDS
    T * const tp = (T *) lds;                         // [part][row][ld]
    int * const ex_s = (int *) (lds + (size_t) NP * NR * ld * 2);
    const int row0 = blockIdx.y * NR, tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nz = gridDim.z, z = blockIdx.z;
    const int o0 = (blockIdx.x * 4 + wave) * 16 * OT;

    // t: the splits' sums, scaled, in parts; lr lanes of 4 values a row
    {
        int lr = 2;
        while (4 * lr < a.rank) lr *= 2;
        const int q = tid & (lr - 1), step = 256 / lr;
        for (int r = tid / lr; r < NR; r += step) {
            const int row = min(row0 + r, a.n_row - 1), id = adapter_of(a, row), rk = id < 0 ? 0 : rank_of(a, id);
            const float sc = id < 0 ? 0.0f : a.scale ? a.scale[id] : 1.0f;
            const float * t = a.work + (size_t) row * a.nsplit * a.rank + 4 * q;
            v4f v = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            if (4 * q < rk)
                for (int s = 0; s < a.nsplit; s++) v += *(const v4fu *) (t + (size_t) s * a.rank);
            float mx = 0.0f;
            #pragma unroll
            for (int e = 0; e < 4; e++) { v[e] = 4 * q + e < rk ? v[e] * sc : 0.0f; mx = fmaxf(mx, fabsf(v[e])); }
            for (int o = 1; o < lr; o *= 2) mx = fmaxf(mx, __shfl_xor(mx, o));
            const int ex = BF ? 0 : scale_of(mx);
            if (4 * q < a.rank) {
                v8 p[NP];
                #pragma unroll
                for (int e = 0; e < 4; e++) parts_of<BF>(__builtin_amdgcn_ldexpf(v[e], -ex), p, e);
                #pragma unroll
                for (int k = 0; k < NP; k++)
                    #pragma unroll
                    for (int e = 0; e < 4; e++) tp[((size_t) k * NR + r) * ld + 4 * q + e] = p[k][e];
            }
            if (!q) ex_s[r] = ex;
        }
    }
    __syncthreads();
    const int id = lane < NR ? adapter_of(a, row0 + lane) : -1;
    unsigned long long left = __ballot(id >= 0), none = ~left;
    for (int k = 0; left || none; k++) {
        // the rows without an adapter are taken like those of one more
        int cur = -1;
        unsigned long long mine = none;
        if (left) {
            cur = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
            mine = __ballot(id == cur);
            left &= ~mine;
        } else {
            none = 0;
        }
        if (k % nz != z || (cur < 0 && a.base == a.y)) continue;
        const int rk = cur < 0 ? 0 : rank_of(a, cur);
        const uint16_t * w = a.b + (size_t) max(cur, 0) * a.n_out * a.rank;
        v4f acc[RB][OT];
        #pragma unroll
        for (int b = 0; b < RB; b++)
            #pragma unroll
            for (int u = 0; u < OT; u++) acc[b][u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k0 = 0; k0 < rk; k0 += 32) {
            const int kk = k0 + 8 * g, at = kk < a.rank ? kk : 0;
            v4u wv[OT];
            #pragma unroll
            for (int u = 0; u < OT; u++) {
                wv[u] = *(const GLOBAL v4u *) (w + (size_t) min(o0 + 16 * u + c, a.n_out - 1) * a.rank + at);
                if (k0 + 32 > rk) {
                    #pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int j = kk + 2 * i;
                        wv[u][i] = j + 1 < rk ? wv[u][i] : j < rk ? wv[u][i] & 0xFFFFu : 0u;
                    }
                }
            }
            #pragma unroll
            for (int b = 0; b < RB; b++)
                #pragma unroll
                for (int i = 0; i < NP; i++) {
                    v8 tv = *(const v8 *) (tp + ((size_t) i * NR + 16 * b + c) * ld + at);
                    if (kk >= a.rank) tv = __builtin_bit_cast(v8, v4u(0u));
                    #pragma unroll
                    for (int u = 0; u < OT; u++) acc[b][u] = M::mul(__builtin_bit_cast(v8, wv[u]), tv, acc[b][u]);
                }
        }
        #pragma unroll
        for (int b = 0; b < RB; b++) {
            const int row = row0 + 16 * b + c;
            if (!(mine >> (16 * b + c) & 1) || row >= a.n_row) continue;
            const int ex = ex_s[16 * b + c];
            #pragma unroll
            for (int u = 0; u < OT; u++) {
                const int o = o0 + 16 * u + 4 * g;
                const size_t at = (size_t) row * a.y_stride + o;
                v4f d;
                #pragma unroll
                for (int r = 0; r < 4; r++) d[r] = __builtin_amdgcn_ldexpf(acc[b][u][r], ex);
                if (o + 4 <= a.n_out) {
                    if (a.base) d += *(const v4fu *) (a.base + at);
                    *(v4fu *) (a.y + at) = d;
                } else {
                    #pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (o + r < a.n_out) a.y[at + r] = (a.base ? a.base[at + r] : 0.0f) + d[r];
                }
            }
        }
    }
}
#define LORA_DOWN(BF, RT, name) \
    extern "C" __global__ __launch_bounds__(64 * LD_WAVES) void name(const sml_klora a) { lora_down_body<BF, RT>(a); }
LORA_DOWN(0, 1, sml_sv_lora_down_t1)
LORA_DOWN(1, 1, sml_sv_lora_down_t1_bf)
LORA_DOWN(0, 4, sml_sv_lora_down_t4)
LORA_DOWN(1, 4, sml_sv_lora_down_t4_bf)
#define LORA_UP(BF, RB, OT, name) \
    extern "C" __global__ __launch_bounds__(256) void name(const sml_klora a) { lora_up_body<BF, RB, OT>(a); }
LORA_UP(0, 1, 1, sml_sv_lora_up_b1)
LORA_UP(1, 1, 1, sml_sv_lora_up_b1_bf)
LORA_UP(0, 4, 2, sml_sv_lora_up_b4)
LORA_UP(1, 4, 2, sml_sv_lora_up_b4_bf)
