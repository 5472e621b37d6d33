// Kernels of several rows a sequence over a paged cache, and of that cache's
// upkeep (sml-serve.h): the append with axes, the rows' attention, accepted
// drafts, forks and moved pages.
#include "serve_dev.h"

// ---------------------------------------------------------------- append
//
// The rotation of sml_sv_append with a position for each pair: a thread's four
// pairs look up their axis (in the arguments) and its position.
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
    v4f y0, y1;
    #pragma unroll
    for (int e = 0; e < 4; e++) {
        const int ax = a.axis[d + e];
        float c = 1.0f, sn = 0.0f;
        if (ax < a.n_axis) {
            const size_t o = (size_t) (ax == 0 ? pos[0] : ax == 1 ? pos[1] : ax == 2 ? pos[2] : pos[3]) * (D / 2) + d + e;
            c = a.cos_t[o];
            sn = a.sin_t[o];
            y0[e] = __builtin_fmaf(lo[e], c, -(hi[e] * sn));
            y1[e] = __builtin_fmaf(lo[e], sn, hi[e] * c);
        } else {
            y0[e] = lo[e];
            y1[e] = hi[e];
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

// The sequence of row r: the last whose rows begin at or before it. -1 where
// the row is nobody's.
__device__ __forceinline__ int row_seq(const sml_krows & a, int r) {
    int lo = 0, hi = a.pg.n_seq;                      // start[lo] <= r < start[hi], if they do not fall
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.start[mid] <= r) lo = mid;
        else hi = mid;
    }
    return a.start[lo] <= r && r < a.start[lo + 1] ? lo : -1;
}

// A workgroup a row and head, its waves alternating chunks of 64 positions, a
// position a lane for the scores and dims a lane for the sum of values: fp32
// throughout.
template <int D, int BF>
__device__ __forceinline__ void rows_body(const sml_krows & a) {
    __shared__ float q[D], pw[4][64], so[4][D], sm[4], sl[4];
    const int h = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = row_seq(a, r);
    if (b < 0) return;
    const int s0 = min(max(a.start[b], 0), a.n_row), s1 = min(max(a.start[b + 1], s0), a.n_row);
    const int n = min(max(a.len[b], 0), a.max_len), m = s1 - s0, past = n - m, own = past + r - s0;
    const int lo = a.first ? max(a.first[r], 0) : 0;
    const int hi = min(a.last ? a.last[r] : a.tree ? past : own + 1, n);
    const int kh = h / (a.n_head / a.pg.n_kv), kvd = a.pg.n_kv * D, sh = a.pg.page_shift, pmask = (1 << sh) - 1;
    const uint32_t * bits = a.tree ? a.tree + (size_t) r * a.words : nullptr;
    const int qpos = a.pos ? a.pos[r] : own;
    if (tid < D) q[tid] = a.q[(size_t) r * a.q_stride + (size_t) h * D + tid];
    __syncthreads();
    const float slope = a.slope ? a.slope[h] : 0.0f;
    float m_run = -INFINITY, l = 0.0f, o[D / 64];
    #pragma unroll
    for (int u = 0; u < D / 64; u++) o[u] = 0.0f;
    for (int t0 = 64 * wave; t0 < n; t0 += 256) {
        const int t = t0 + lane, j = t - past;
        bool see = t < n && t >= lo && t < hi;
        if (bits && t < n && j >= 0 && j < m && j < 32 * a.words) see |= (bits[j >> 5] >> (j & 31)) & 1;
        int page = see ? page_of(a.pg, b, t >> sh) : -1;
        see &= page >= 0;
        size_t at = see ? (size_t) page * a.pg.page_stride + (size_t) (t & pmask) * kvd + (size_t) kh * D : 0;
        float s = -INFINITY;
        if (see) {
            s = 0.0f;
            for (int d = 0; d < D; d += 8) {
                const v4u w = *(const v4u *) (a.pg.k + at + d);
                #pragma unroll
                for (int e = 0; e < 4; e++) {
                    s = __builtin_fmaf(of16<BF>((uint16_t) (w[e] & 0xFFFF)), q[d + 2 * e], s);
                    s = __builtin_fmaf(of16<BF>((uint16_t) (w[e] >> 16)), q[d + 2 * e + 1], s);
                }
            }
            s *= a.scale;
            if (a.cap > 0.0f) s = a.cap * tanhf(s / a.cap);
            if (a.slope) {
                const int kpos = j >= 0 && a.pos ? a.pos[s0 + j] : t;
                s -= slope * fabsf((float) (qpos - kpos));
            }
        }
        const float top = fmaxf(m_run, wave_max(s)), tu = top == -INFINITY ? 0.0f : top;
        const float al = expf(m_run - tu), p = see ? expf(s - tu) : 0.0f;
        m_run = top;
        l = l * al + p;
        pw[wave][lane] = p;
        wave_lds();
        #pragma unroll
        for (int u = 0; u < D / 64; u++) o[u] *= al;
        const unsigned long long any = __ballot(see);
        for (int i = 0; i < 64; i++) {
            if (!((any >> i) & 1)) continue;
            const float w = pw[wave][i];
            const size_t v = ((size_t) (unsigned) __shfl((int) (at >> 32), i) << 32) | (unsigned) __shfl((int) at, i);
            #pragma unroll
            for (int u = 0; u < D / 64; u++) o[u] = __builtin_fmaf(w, of16<BF>(a.pg.v[v + 64 * u + lane]), o[u]);
        }
        wave_lds();
    }
    l = wave_sum(l);
    if (!lane) { sm[wave] = m_run; sl[wave] = l; }
    #pragma unroll
    for (int u = 0; u < D / 64; u++) so[wave][64 * u + lane] = o[u];
    __syncthreads();
    if (tid >= D) return;
    float top = sm[0];
    for (int w = 1; w < 4; w++) top = fmaxf(top, sm[w]);
    const float tu = top == -INFINITY ? 0.0f : top;
    float os = 0.0f, ls = 0.0f;
    for (int w = 0; w < 4; w++) {
        const float f = expf(sm[w] - tu);
        os += f * so[w][tid];
        ls += f * sl[w];
    }
    a.out[((size_t) r * a.n_head + h) * D + tid] = ls == 0.0f ? 0.0f : os / ls;
}
#define ROWS(D, BF, name) \
    extern "C" __global__ __launch_bounds__(256) void name(const sml_krows a) { rows_body<D, BF>(a); }
ROWS(128, 0, sml_rw_rows)
ROWS(128, 1, sml_rw_rows_bf)
ROWS(64, 0, sml_rw_rows_d64)
ROWS(64, 1, sml_rw_rows_d64_bf)

// ---------------------------------------------------------------- layers of a cache

// Unit z's pool of the layers: even numbers keys, odd ones values.
__device__ __forceinline__ uint16_t * pool_of(const sml_kpages & pg, size_t layer_stride, int z) {
    return (z & 1 ? pg.v : pg.k) + (size_t) (z >> 1) * layer_stride;
}

// ---------------------------------------------------------------- accepted drafts
//
// Every workgroup walks its sequence's tree for itself: a step is the first row
// behind the present one that follows it with its pick, 64 rows looked at a time
// by one wave. A thread then moves 16 bytes of a position in one pool, the
// path's rows in order: a row's new place lies before every later row's old one,
// so nothing is overwritten that is still to be read.
extern "C" __global__ __launch_bounds__(256) void sml_rw_accept(const sml_kaccept a) {
    __shared__ int path[AC_MOST], count;
    const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int s0 = min(max(a.start[b], 0), a.n_row), s1 = min(max(a.start[b + 1], s0), a.n_row), m = s1 - s0;
    const int cap = a.pg.seq_pages << a.pg.page_shift, n = min(max(a.len[b], 0), cap), past = n - m;
    if (tid < 64) {
        int k = 0, at = 0;
        if (m > 0) {
            if (!lane) path[0] = 0;
            k = 1;
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
    const long u = (long) blockIdx.x * 256 + tid;
    if (u >= (long) 2 * a.n_layer * row) return;
    uint16_t * const pool = pool_of(a.pg, a.layer_stride, (int) (u / row)) + 8 * (u % row);
    const int sh = a.pg.page_shift, pmask = (1 << sh) - 1;
    for (int j = 1; j < k; j++) {
        const int from = past + path[j], to = past + j;
        if (from == to || to < 0) continue;
        const int pf = page_of(a.pg, b, from >> sh), pt = page_of(a.pg, b, to >> sh);
        if (pf < 0 || pt < 0) continue;
        const v4u w = *(const v4u *) (pool + (size_t) pf * a.pg.page_stride + (size_t) (from & pmask) * 8 * row);
        *(v4u *) (pool + (size_t) pt * a.pg.page_stride + (size_t) (to & pmask) * 8 * row) = w;
    }
}

// ---------------------------------------------------------------- forks
//
// A workgroup copies 16 KB of the begun page in one pool; the first of a fork's
// also writes its row of the table.
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
// ascending sources by halving.
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
