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
// One workgroup a query head, a wave every fourth position.
template <int D, int BF>
__device__ __forceinline__ void attend_body(const sml_kattend & a) {
    constexpr int E = D / 64;
    __shared__ float so[4][D], sm[4], sl[4];
    const int h = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = min(a.len[b], a.max_len), kh = h / (a.n_head / a.pg.n_kv);
    float q[E], o[E], m = -INFINITY, l = 0.0f;
    #pragma unroll
    for (int e = 0; e < E; e++) {
        q[e] = a.q[(size_t) b * a.q_stride + (size_t) h * D + lane * E + e] * a.scale;
        o[e] = 0.0f;
    }
    for (int p = w; p < n; p += 4) {
        const int page = page_of(a.pg, b, p >> a.pg.page_shift);
        if (page < 0) continue;
        const size_t at = (size_t) page * a.pg.page_stride +
                          (size_t) (p & ((1 << a.pg.page_shift) - 1)) * (a.pg.n_kv * D) + (size_t) kh * D + lane * E;
        float s = 0.0f;
        #pragma unroll
        for (int e = 0; e < E; e++) s += q[e] * of16<BF>(a.pg.k[at + e]);
        s = wave_sum(s);
        const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m - mu), pr = __builtin_amdgcn_exp2f(s - mu);
        l = l * al + pr;
        #pragma unroll
        for (int e = 0; e < E; e++) o[e] = o[e] * al + pr * of16<BF>(a.pg.v[at + e]);
        m = mn;
    }
    #pragma unroll
    for (int e = 0; e < E; e++) so[w][lane * E + e] = o[e];
    if (!lane) { sm[w] = m; sl[w] = l; }
    __syncthreads();
    if ((int) threadIdx.x >= D) return;
    float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), ll = 0.0f, oo = 0.0f;
    if (mm == -INFINITY) mm = 0.0f;
    for (int i = 0; i < 4; i++) {
        const float e = __builtin_amdgcn_exp2f(sm[i] - mm);
        ll += e * sl[i];
        oo += e * so[i][threadIdx.x];
    }
    a.out[((size_t) b * a.n_head + h) * D + threadIdx.x] = ll == 0.0f ? 0.0f : oo / ll;
}
#define ATTEND(D, BF, name) \
    extern "C" __global__ __launch_bounds__(256) void name(const sml_kattend a) { attend_body<D, BF>(a); }
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
// Two launches: t = A x of a row's adapter, then y = base + scale * B t.
template <int BF>
__device__ __forceinline__ void lora_down_body(const sml_klora & a) {
    const int j = blockIdx.x, r = blockIdx.y, ad = a.adapter[r];
    if (ad < 0 || ad >= a.n_adapter || (a.ranks && j >= a.ranks[ad])) return;
    const uint16_t * w = a.a + ((size_t) ad * a.rank + j) * a.n_in;
    const float * x = a.x + (size_t) r * a.x_stride;
    float s = 0.0f;
    for (int i = threadIdx.x; i < a.n_in; i += 64) s += x[i] * of16<BF>(w[i]);
    s = wave_sum(s);
    if (!threadIdx.x) a.work[(size_t) r * a.rank + j] = s;
}
template <int BF>
__device__ __forceinline__ void lora_up_body(const sml_klora & a) {
    const int o = blockIdx.x * 256 + threadIdx.x, r = blockIdx.y, ad = a.adapter[r];
    if (o >= a.n_out) return;
    const size_t at = (size_t) r * a.y_stride + o;
    float y = a.base ? a.base[at] : 0.0f;
    if (ad >= 0 && ad < a.n_adapter) {
        const int rk = a.ranks ? min(a.ranks[ad], a.rank) : a.rank;
        const uint16_t * w = a.b + ((size_t) ad * a.n_out + o) * a.rank;
        const float * t = a.work + (size_t) r * a.rank;
        float s = 0.0f;
        for (int j = 0; j < rk; j++) s += t[j] * of16<BF>(w[j]);
        y += (a.scale ? a.scale[ad] : 1.0f) * s;
    }
    a.y[at] = y;
}
extern "C" __global__ __launch_bounds__(64) void sml_sv_lora_down(const sml_klora a) { lora_down_body<0>(a); }
extern "C" __global__ __launch_bounds__(64) void sml_sv_lora_down_bf(const sml_klora a) { lora_down_body<1>(a); }
extern "C" __global__ __launch_bounds__(256) void sml_sv_lora_up(const sml_klora a) { lora_up_body<0>(a); }
extern "C" __global__ __launch_bounds__(256) void sml_sv_lora_up_bf(const sml_klora a) { lora_up_body<1>(a); }
