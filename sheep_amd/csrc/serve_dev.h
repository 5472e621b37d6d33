// Device code shared by the kernels over a paged cache (serve.hip, rows.hip).
#pragma once
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

// ---------------------------------------------------------------- values in 16-bit parts
//
// The matrix cores take fp32 values as sums of 16-bit parts: two of fp16, three
// of bfloat16. lift and room: of a softmax's base (beside the attention).
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
