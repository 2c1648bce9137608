// psfm_linear_kernels.h — the pointwise product's kernels, one instance set per type (gfx950).
//
//   product   one output tile [BI, BJ] per workgroup on the matrix cores (k_forward: with the epilogue; k_pair:
//             dx's and dw's tiles in one launch).  LDS holds two or three stages of 128 bytes of reduction per output
//             row and column (64 values of 16 bits, 32 of 32): while one is multiplied the next ones' global
//             loads are in flight.  The product is taken as D = Q P^T, so that a lane's four results are
//             four consecutive columns of one output row.
//   k_skinny  at most 32 rows: no tiles, W straight from memory into the matrix instructions.
//   k_finish  sums split products in the order of their splits, and the bias gradient's parts.
//   k_dz      dz = drop(dy) act'(z) and its column sums as a pass of its own, where the products would make
//             it too often.
#pragma once
#include <type_traits>

#include "psfm_linear.h"

namespace psfm {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));

// LDS by its own address space: the compiler follows such pointers to their object (the waits for loads into it)
#define PSFM_LDS __attribute__((address_space(3)))
typedef PSFM_LDS uint8_t lds8;

template <typename T>
constexpr int CHUNK = 16 / (int)sizeof(T);   // values of one 16-byte chunk

// ---- activations, in fp32, of N values under one (uniform) choice ------------------------------
// v_rcp_f32 is good to one step of fp32, the IEEE division around it costs ten instructions
__device__ __forceinline__ float sigmoidf(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

// The normal distribution function and exp(-z^2 / 2).  Both branches keep the lower tail's own scale.  fp32: erfcf.  16 bits,
// sharing the density's exponential: erfc(x) = (a1 t + .. + a8 t^8) exp(-x^2), t = 1 / (1 + 0.44 x), x = |z| / sqrt(2).
// The a are a fit of least relative error over x = 0 .. 10 (linear programming; 1 at x = 0): 1.8e-7, 5.7e-7 in fp32.
template <typename T>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    e = __expf(-0.5f * z * z);
    if constexpr (sizeof(T) == 4) {
        return 0.5f * erfcf(-0.70710678118654752f * z);
    } else {
        const float t = __builtin_amdgcn_rcpf(1.0f + 0.44f * 0.70710678118654752f * fabsf(z));
        const float a = t * (0.294311702f + t * (-0.276345044f + t * 0.0707828626f));
        const float q = t * (0.248222306f + t * (0.24884516f + t * (0.217515379f + t * (0.214997917f + t * (-0.0183302537f + a)))));
        const float low = 0.5f * q * e;
        return z < 0.0f ? low : 1.0f - low;
    }
}

template <typename T, int N>
__device__ __forceinline__ void act_of(int act, float (&z)[N]) {
#define PSFM_EACH(F)                         \
    _Pragma("unroll") for (int k = 0; k < N; ++k) { \
        const float v = z[k];                \
        z[k] = F;                            \
    }                                        \
    break;
    float e;
    switch (act) {
        case PSFM_ACT_RELU: PSFM_EACH(v < 0.0f ? 0.0f : v)     // NaN stays
        case PSFM_ACT_SIGMOID: PSFM_EACH(sigmoidf(v))
        case PSFM_ACT_ELU: PSFM_EACH(v > 0.0f ? v : expm1f(v))
        case PSFM_ACT_SILU: PSFM_EACH(v * sigmoidf(v))
        case PSFM_ACT_GELU: PSFM_EACH(v * normal_cdf<T>(v, e))
        default: break;
    }
#undef PSFM_EACH
}

__device__ __forceinline__ float slope_silu(float z) {
    const float s = sigmoidf(z);
    return s * (1.0f + z * (1.0f - s));
}
// of exp(-|z|): 1 - s has lost both tails' scale
__device__ __forceinline__ float slope_sigmoid(float z) {
    const float e = __expf(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e);
    return e * r * r;
}
template <typename T>
__device__ __forceinline__ float slope_gelu(float z) {
    float e;
    const float c = normal_cdf<T>(z, e);
    return c + z * e * 0.39894228040143268f;
}
template <typename T, int N>
__device__ __forceinline__ void times_slope(int act, const float (&z)[N], float (&d)[N]) {
#define PSFM_EACH(F) \
    _Pragma("unroll") for (int k = 0; k < N; ++k) d[k] *= F; \
    break;
    switch (act) {
        case PSFM_ACT_RELU:   // a selection: an infinite gradient of a value below 0 is none, and NaN passes its own
            _Pragma("unroll") for (int k = 0; k < N; ++k) d[k] = z[k] <= 0.0f ? 0.0f : d[k];
            break;
        case PSFM_ACT_SIGMOID: PSFM_EACH(slope_sigmoid(z[k]))
        case PSFM_ACT_ELU: PSFM_EACH((z[k] > 0.0f ? 1.0f : __expf(z[k])))
        case PSFM_ACT_SILU: PSFM_EACH(slope_silu(z[k]))
        case PSFM_ACT_GELU: PSFM_EACH(slope_gelu<T>(z[k]))
        default: break;
    }
#undef PSFM_EACH
}

// What z is kept in for the backward pass.  The slope is taken at it, so its rounding adds to dz's own: |z act''| reaches
// |act'| (sigmoid, elu), and bf16's would weigh as much as dz's.  fp16 has 8 times bf16's steps in the same
// bytes; beyond its range (+-65504) every slope has reached its limit.  fp16 products keep z in fp32.  ReLU
// needs the sign alone, in the type itself.
template <typename T>
struct KeptZ {
    using type = float;
};
template <>
struct KeptZ<__bf16> {
    using type = _Float16;
};

// ---- chunks of up to 16 bytes at any alignment that the type has -------------------------------
template <typename T>
__device__ __forceinline__ u4v load_chunk(const T* p) {
    return *reinterpret_cast<const u4v*>(p);
}
template <typename T>
__device__ __forceinline__ u4v load_part(const T* p, int n) {   // the first n values, zeros behind
    union {
        u4v v;
        T t[CHUNK<T>];
    } u;
    u.v = u4v{0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < CHUNK<T>; ++k)
        if (k < n) u.t[k] = p[k];
    return u.v;
}
// n in 0 .. CHUNK values at p; VEC: n is 0 or CHUNK and p is 16-byte aligned
template <typename T, bool VEC>
__device__ __forceinline__ u4v load_n(const T* p, int n) {
    if (n >= CHUNK<T>) {
        if (VEC) return load_chunk(p);
        u4v v;
        __builtin_memcpy(&v, p, 16);
        return v;
    }
    return VEC ? u4v{0, 0, 0, 0} : load_part(p, n);
}

// ---- runs of N consecutive values, the first n of them there, at any alignment that the type has ---
template <typename T, int N>
__device__ __forceinline__ void store_run(T* p, const float (&v)[N], int n) {
    typedef T TN __attribute__((ext_vector_type(N)));
    if (n >= N) {
        TN t;
#pragma unroll
        for (int k = 0; k < N; ++k) t[k] = (T)v[k];
        __builtin_memcpy(p, &t, sizeof(T) * N);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < n) p[k] = (T)v[k];
    }
}
template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, float (&v)[N], int n) {
    typedef T TN __attribute__((ext_vector_type(N)));
    if (n >= N) {
        TN t;
        __builtin_memcpy(&t, p, sizeof(T) * N);
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = (float)t[k];
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = k < n ? (float)p[k] : 0.0f;
    }
}

// ---- the epilogue of columns j .. j + N - 1 (j % 4 = 0; those below J exist) of row i -----------------
// Its inputs: bias[j ..], or zeros, and res[i, j ..].
template <typename T, bool FULL, int N>
__device__ __forceinline__ void bias_run(const LinearEpi& e, int64_t J, int64_t j, float (&b)[N]) {
    if (FULL && e.bias && j < J) {
        load_run((const T*)e.bias + j, b, J - j < N ? (int)(J - j) : N);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) b[k] = 0.0f;
    }
}
template <typename T, bool FULL, int N>
__device__ __forceinline__ void res_run(const LinearEpi& e, int64_t I, int64_t J, int64_t i, int64_t j, T (&r)[N]) {
    if (!FULL || !e.res || i >= I || j >= J) return;
    const T* p = (const T*)e.res + i * e.ldr + j;
    if (J - j >= N) {
        __builtin_memcpy(r, p, sizeof(T) * N);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < J - j) r[k] = p[k];
    }
}
template <typename T, bool FULL, int N>
__device__ __forceinline__ void epilogue(const LinearEpi& e, const PhiloxKey& key, KeepBits<N>& keep, int64_t J, int64_t i,
                                         int64_t j, float (&v)[N], const float (&b)[N], const T (&r)[N]) {
    const int n = J - j < N ? (int)(J - j) : N;
    const int64_t at = i * J + j;
    if (!FULL) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] *= e.alpha;
        store_run((T*)e.out + at, v, n);
        return;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += b[k];
    if (e.z) {
        using Z = typename KeptZ<T>::type;
        if (e.act == PSFM_ACT_RELU) {
            store_run((T*)e.z + at, v, n);
        } else if (sizeof(Z) == 2) {
            float c[N];
#pragma unroll
            for (int k = 0; k < N; ++k) c[k] = v[k] != v[k] ? v[k] : fminf(fmaxf(v[k], -65504.0f), 65504.0f);
            store_run((Z*)e.z + at, c, n);
        } else {
            store_run((Z*)e.z + at, v, n);
        }
    }
    act_of<T>(e.act, v);
    if (e.drop.rng) drop_run(e.drop, key, keep, J, mask_row(e.drop, i), j, e.drop.scale, v);
    if (e.res) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += (float)r[k];
    }
    store_run((T*)e.out + at, v, n);
}
template <typename T, bool FULL, int N>
__device__ __forceinline__ void epilogue(const LinearEpi& e, const PhiloxKey& key, KeepBits<N>& keep, int64_t I, int64_t J,
                                         int64_t i, int64_t j, float (&v)[N]) {
    float b[N];
    T r[N];
    bias_run<T, FULL>(e, J, j, b);
    res_run<T, FULL>(e, I, J, i, j, r);
    epilogue<T, FULL>(e, key, keep, J, i, j, v, b, r);
}

// ---- LDS images ----------------------------------------------------------------------------
// Straight operand: one 128-byte row of reduction per output row; its eight 16-byte chunks are XORed by the
// row so that 16 lanes reading the same chunk of 16 rows hit 16 bank quads.  Turned operand: one row per
// reduction index, chunks XORed so that the reads (16 bits: transposing, 4 rows x 32 bytes a 16-lane group;
// 32 bits: 128 or 256 bytes of a row a group, the groups 4 rows apart) spread over the banks.
__device__ __forceinline__ int swz_straight(int row) { return (row >> 1) & 7; }
template <typename T, int B>
__device__ __forceinline__ int swz_turned(int row) {
    if (sizeof(T) == 4) return (((row >> 2) & 1) << 3) | (((row >> 3) & 1) << 2);
    if (B == 64) return (((row >> 1) & 1) | (((row >> 3) & 1) << 1)) << 1;
    return ((row & 3) | (((row >> 3) & 1) << 2)) << 1;
}

// Thread t's share of a stage, NC chunks: global -> registers, registers -> LDS.
template <typename T, int B, int NTH, bool TURNED, bool VEC>
struct Stager {
    static constexpr int NC = B * 8 / NTH, V = CHUNK<T>, CPR = B * (int)sizeof(T) / 16;
    u4v r[NC];

    // (row, column) in the operand's own matrix of chunk q of the stage at rows b0 .., reduction r0 ..
    static __device__ __forceinline__ void place(int q, int64_t b0, int64_t r0, int64_t& row, int64_t& col) {
        const int c = q * NTH + threadIdx.x;
        row = TURNED ? r0 + c / CPR : b0 + c / 8;
        col = TURNED ? b0 + (int64_t)(c % CPR) * V : r0 + (c % 8) * V;
    }
    // values of the chunk that exist: rows below ext (turned: rend), columns below rend (turned: ext)
    static __device__ __forceinline__ int there(int64_t row, int64_t col, int64_t ext, int64_t rend) {
        const int64_t left = row < (TURNED ? rend : ext) ? (TURNED ? ext : rend) - col : 0;
        return left >= V ? V : left > 0 ? (int)left : 0;
    }
    // Whether every chunk of a stage may be read whole: the reduction does not end inside it, and where a chunk reaches
    // over its row's end (turned: the tile's last columns, by V - 1 values at most; what it takes from there is
    // never stored) there is as much of the operand behind the stage's last row.
    static __device__ __forceinline__ bool whole(int64_t ld, int64_t b0, int64_t ext, int64_t r0, int64_t rend, int64_t all) {
        constexpr int BR = 128 / (int)sizeof(T);
        return r0 + BR <= rend && (!TURNED || b0 + B <= ext || (all - r0 - BR) * ld >= V - 1);
    }
    // all: the reduction's end in the operand, behind this split's too
    __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t b0, int64_t ext, int64_t r0, int64_t rend,
                                         int64_t all) {
        // uniform: no bounds a chunk (aligned chunks are whole or none, and reading the none ones costs more)
        if (!VEC && whole(ld, b0, ext, r0, rend, all)) {
#pragma unroll
            for (int q = 0; q < NC; ++q) {
                int64_t row, col;
                place(q, b0, r0, row, col);
                if (!TURNED && row >= ext) row = ext - 1;
                if (TURNED && col >= ext) col = b0;
                __builtin_memcpy(&r[q], base + row * ld + col, 16);
            }
            return;
        }
#pragma unroll
        for (int q = 0; q < NC; ++q) {
            int64_t row, col;
            place(q, b0, r0, row, col);
            const int n = there(row, col, ext, rend);
            r[q] = load_n<T, VEC>(base + (n > 0 ? row * ld + col : 0), n);
        }
    }
    static __device__ __forceinline__ void put(lds8* lds, int q, u4v v) {
        const int c = q * NTH + threadIdx.x;
        const int row = TURNED ? c / CPR : c / 8, ch = TURNED ? c % CPR : c % 8;
        const int x = TURNED ? swz_turned<T, B>(row) : swz_straight(row);
        *(PSFM_LDS u4v*)(lds + row * (TURNED ? CPR * 16 : 128) + ((ch ^ x) << 4)) = v;
    }
    __device__ __forceinline__ void store(lds8* lds) const {
#pragma unroll
        for (int q = 0; q < NC; ++q) put(lds, q, r[q]);
    }
};

// The same without registers: the loads write LDS themselves, 16 bytes a lane in lane order, so the chunks' order in
// a row is turned in the addresses that they read.  Whole chunks only.  A row or column that does not exist reads
// the last one that does (what it gives is never stored); behind the reduction's end there are zeros.
__device__ const uint4 zeros16 = {0, 0, 0, 0};

template <typename T, int B, int NTH, bool TURNED>
struct DmaStager {
    static constexpr int NC = B * 8 / NTH, V = CHUNK<T>, CPR = B * (int)sizeof(T) / 16, BR = 128 / (int)sizeof(T);
    const T* p[NC];       // this lane's chunks of the next stage
    int r[NC];            // their reduction index in the stage
    int64_t stride;       // from stage to stage

    __device__ __forceinline__ void at(const T* base, int64_t ld, int64_t b0, int64_t ext, int64_t r0) {
        stride = TURNED ? BR * ld : BR;
#pragma unroll
        for (int q = 0; q < NC; ++q) {
            const int c = q * NTH + threadIdx.x, row = TURNED ? c / CPR : c / 8;
            const int ch = TURNED ? (c % CPR) ^ swz_turned<T, B>(row) : (c % 8) ^ swz_straight(row);
            const int64_t want = b0 + (TURNED ? ch * V : row), last = TURNED ? ext - V : ext - 1;
            const int64_t out = want < last ? want : last;
            r[q] = TURNED ? row : ch * V;
            p[q] = base + (TURNED ? (r0 + row) * ld + out : out * ld + r0 + ch * V);
        }
    }
    // left: reduction elements from this stage on
    __device__ __forceinline__ void load(lds8* lds, int64_t left) {
        typedef __attribute__((address_space(1))) const void gvoid;
        typedef PSFM_LDS void lvoid;
#pragma unroll
        for (int q = 0; q < NC; ++q) {
            const T* src = p[q];
            if (left < BR && r[q] >= left) src = (const T*)&zeros16;
            __builtin_amdgcn_global_load_lds((gvoid*)src, (lvoid*)(lds + (q * NTH + (threadIdx.x & ~63)) * 16), 16, 0, 0);
            p[q] += stride;
        }
    }
};

// The same of dz, made from dy and z on the way to LDS, with the sums of this thread's columns (turned: they stay
// the same in all its chunks) before dz is rounded to the type for the matrix cores.  16 bits: what that rounding leaves
// goes to a second image and a second product, so that a gradient has one rounding and not two (few values are summed
// here at times, and then the two showed: up to 1.6 times the error of one).  These products wait for memory,
// not for the matrix cores.  No activation, or ReLU: dz is dy's own value or 0, and nothing is left.
template <typename T, int B, int NTH, bool TURNED, bool VEC>
struct DzStager : Stager<T, B, NTH, TURNED, VEC> {
    using S = Stager<T, B, NTH, TURNED, VEC>;
    using Z = typename KeptZ<T>::type;
    static constexpr int V = S::V, ZN = (int)sizeof(Z) * V / 16;
    u4v z[S::NC][ZN];
    float sum[V];
    KeepBits<V> keep;

    __device__ __forceinline__ void load(const GemmArgs& A, int64_t b0, int64_t ext, int64_t r0, int64_t rend) {
        S::load((const T*)A.P, A.ldp, b0, ext, r0, rend, A.R);
        if (!A.dz.z) return;
        const bool relu = A.dz.act == PSFM_ACT_RELU;
#pragma unroll
        for (int q = 0; q < S::NC; ++q) {
            int64_t row, col;
            S::place(q, b0, r0, row, col);
            const int n = S::there(row, col, ext, rend);
            const int64_t at = n > 0 ? row * A.ldp + col : 0;
            if (relu || sizeof(Z) == sizeof(T)) {
                z[q][0] = load_n<T, VEC>((const T*)A.dz.z + at, n);   // the same bytes, T or Z
            } else {
#pragma unroll
                for (int h = 0; h < ZN; ++h) {
                    constexpr int ZV = 16 / (int)sizeof(Z);
                    z[q][h] = load_n<Z, VEC>((const Z*)A.dz.z + at + (n > h * ZV ? h * ZV : 0),
                                             n > h * ZV ? (n - h * ZV < ZV ? n - h * ZV : ZV) : 0);
                }
            }
        }
    }
    static __device__ __forceinline__ bool has_rest(const GemmArgs& A) {
        return sizeof(T) == 2 && A.dz.z && A.dz.act != PSFM_ACT_RELU;
    }
    // rest: the second image
    __device__ __forceinline__ void store(lds8* lds, lds8* rest, const GemmArgs& A, const PhiloxKey& key, int64_t b0,
                                          int64_t r0) {
        typedef T TV __attribute__((ext_vector_type(V)));
#pragma unroll
        for (int q = 0; q < S::NC; ++q) {
            float d[V];
            const TV t = __builtin_bit_cast(TV, S::r[q]);
#pragma unroll
            for (int k = 0; k < V; ++k) d[k] = (float)t[k];
            if (A.dz.z) {
                float zv[V];
                const TV zt = __builtin_bit_cast(TV, z[q][0]);
                if (A.dz.act == PSFM_ACT_RELU) {
#pragma unroll
                    for (int k = 0; k < V; ++k) zv[k] = (float)zt[k];
                } else {
#pragma unroll
                    for (int h = 0; h < ZN; ++h) {
                        typedef Z ZV __attribute__((ext_vector_type(16 / sizeof(Z))));
                        const ZV zz = __builtin_bit_cast(ZV, z[q][h]);
#pragma unroll
                        for (int k = 0; k < 16 / (int)sizeof(Z); ++k) zv[h * (16 / (int)sizeof(Z)) + k] = (float)zz[k];
                    }
                }
                times_slope<T>(A.dz.act, zv, d);
            }
            if (A.dz.drop.rng) {   // last: a dropped value is 0 whatever dy and z hold
                int64_t row, col;
                S::place(q, b0, r0, row, col);
                drop_run(A.dz.drop, key, keep, A.ldp, mask_row(A.dz.drop, row), col, 1.0f, d);
            }
            TV o;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                o[k] = (T)d[k];
                if (TURNED) sum[k] += d[k];
            }
            S::put(lds, q, __builtin_bit_cast(u4v, o));
            if constexpr (sizeof(T) == 2) {
                if (has_rest(A)) {
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float high = (float)o[k];
                        o[k] = (T)(fabsf(high) < INFINITY ? d[k] - high : 0.0f);   // nothing is left of an infinity
                    }
                    S::put(rest, q, __builtin_bit_cast(u4v, o));
                }
            }
        }
    }
};

// One lane's operand of a matrix instruction step (64 bytes of reduction: 32 values of 16 bits, 16 of 32): the 16
// output rows or columns b .. b + 15, lane l holds row l % 16, reduction chunk l / 16.
template <typename T, int B, bool TURNED>
__device__ __forceinline__ u4v fragment(const lds8* lds, int b, int ks) {
    const int l = threadIdx.x & 63, g = l >> 4, n = l & 15;
    if (!TURNED) {
        const int row = b + n;
        return *(const PSFM_LDS u4v*)(lds + row * 128 + (((ks * 4 + g) ^ swz_straight(row)) << 4));
    }
    if constexpr (sizeof(T) == 2) {
        constexpr int RB = B * 2;
        // a 16-lane group reads 4 rows x 16 values, lane n gets column n of the 4 rows
        typedef PSFM_LDS s4 lds_s4;
        const int ch = (b >> 3) + ((n & 3) >> 1), r0 = ks * 32 + 8 * g + (n >> 2), r1 = r0 + 4;
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s4*)(lds + r0 * RB + ((ch ^ swz_turned<T, B>(r0)) << 4) + 8 * (n & 1)));
        const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s4*)(lds + r1 * RB + ((ch ^ swz_turned<T, B>(r1)) << 4) + 8 * (n & 1)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(u4v, (s8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
    }
    __builtin_unreachable();   // turned 32-bit operands: fragments_turned32
}

// S of them of a turned 32-bit operand.  Lane n takes the S neighbouring output rows b + S n + s of each reduction
// index, one read of 4 S bytes, so operand s holds every S-th output row: `product` puts the results in order.
template <int S, int B, int ks>
__device__ __forceinline__ void fragments_turned32(const lds8* lds, int b, u4v (&f)[S]) {
    static_assert(S == 2 || S == 4, "a read of 8 or 16 bytes");
    typedef unsigned int uSv __attribute__((ext_vector_type(S)));
    const int l = threadIdx.x & 63, g = l >> 4, col = b + S * (l & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = ks * 16 + 4 * g + i;
        const uSv v = *(const PSFM_LDS uSv*)(lds + row * B * 4 + (((col >> 2) ^ swz_turned<float, B>(row)) << 4) + 4 * (col & 3));
#pragma unroll
        for (int s = 0; s < S; ++s) f[s][i] = v[s];
    }
}

// S of them of a turned 16-bit operand, 16 output rows apart, where the stages are filled by loads into LDS: behind such
// a load the compiler puts a wait for all of them before the first transposing read (it does not follow the object
// that this read reads, as it does for plain reads), so the reads are written out with their own wait.
// One address serves all: the operands' chunks differ in bits that the swizzle XORs (s << 5), the rows of the second half
// and of the second step lie a constant away and are swizzled alike.  It is hidden from the optimiser each
// time, which would keep every operand's own and spill.
template <int S, int B, int ks>
__device__ __forceinline__ void fragments_turned(const lds8* lds, int b, u4v (&f)[S]) {
    constexpr int RB = B * 2, U = S % 4 == 0 ? 4 : 2;
    static_assert(S % 2 == 0 && S * 2 <= B / 8, "operands within a row");
    const int l = threadIdx.x & 63, g = l >> 4, n = l & 15, row = 8 * g + (n >> 2), ch = (b >> 3) + ((n & 3) >> 1);
    typedef unsigned int u2v __attribute__((ext_vector_type(2)));
    uint32_t at = (uint32_t)(uintptr_t)(lds + row * RB + ((ch ^ swz_turned<__bf16, B>(row)) << 4) + 8 * (n & 1));
    asm volatile("" : "+v"(at));
    constexpr int o0 = ks * 32 * RB, o1 = o0 + 4 * RB;
#pragma unroll
    for (int s = 0; s < S; s += U) {
        u2v v[2 * U];
        if constexpr (U == 4)
            asm volatile(
                "ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
                : "v"(at ^ s << 5), "v"(at ^ (s + 1) << 5), "v"(at ^ (s + 2) << 5), "v"(at ^ (s + 3) << 5), "n"(o0),
                  "n"(o1)
                : "memory");
        else
            asm volatile(
                "ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
                "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
                : "v"(at ^ s << 5), "v"(at ^ (s + 1) << 5), "n"(o0), "n"(o1)
                : "memory");
#pragma unroll
        for (int q = 0; q < U; ++q) f[s + q] = u4v{v[2 * q][0], v[2 * q][1], v[2 * q + 1][0], v[2 * q + 1][1]};
    }
}

// The S operands of a wave's step.
template <typename T, int S, int B, bool TURNED, bool DMA, int ks>
__device__ __forceinline__ void fragments(const lds8* lds, int b, u4v (&f)[S]) {
    if constexpr (TURNED && sizeof(T) == 4) {
        fragments_turned32<S, B, ks>(lds, b, f);
    } else if constexpr (TURNED && DMA) {
        fragments_turned<S, B, ks>(lds, b, f);
    } else {
#pragma unroll
        for (int s = 0; s < S; ++s) f[s] = fragment<T, B, TURNED>(lds, b + 16 * s, ks);
    }
}

template <typename T>
__device__ __forceinline__ f4 mma(u4v a, u4v b, f4 c) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)   // the four steps of four values take the same reduction order of both operands
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
        return c;
    } else if constexpr (__is_same(T, __bf16)) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
}

// Workgroup id -> tile: the eight XCDs take turns in the id, so each gets a run of consecutive tiles (its L2
// keeps their operands), and a run walks 8 tile rows before the next tile column.
__device__ __forceinline__ uint32_t xcd_run(uint32_t id, uint32_t n) {
    const uint32_t x = id & 7, k = id >> 3, per = n >> 3, more = n & 7;
    return x * per + (x < more ? x : more) + k;
}

// Stages in LDS.  Two; three of the smallest tile where loads go into LDS and the reduction is long (DEEP), so that two
// are on their way while one is multiplied: a CU with few workgroups waits for memory (4096 x 512 x 2048 bf16: 21.2 us
// with two, 15.9 with three; 512 x 4096 x 4096: 38.8, 32.5).  Short ones live from workgroups a CU instead (184320 x
// 64 x 32: 21 us with two and five a CU, 23.4 with three and three a CU).
constexpr int DEEP_STAGES = 5;   // of reduction, at least
template <bool DMA, bool DEEP>
constexpr int STAGES = DMA && DEEP ? 3 : 2;

// A stage's images: P, Q, and what dz's rounding left of P.
template <typename T, int BI, int BJ, bool DZ>
constexpr int STAGE_BYTES = (BI + BJ + (DZ && sizeof(T) == 2 ? BI : 0)) * 128;

// Tile `id` of `count` of a product.  WI x WJ waves.  The stages are objects of their own, and the loop is written out for
// them, so that the compiler sees that the reads of one do not wait for the loads into another.
template <typename T, int BI, int BJ, int WI, int WJ, bool PT, bool QT, bool VEC, bool FULL, bool DZ, bool DEEP>
__device__ __forceinline__ void product(const GemmArgs& A, uint32_t id, uint32_t count,
                                        uint8_t (&stage0)[STAGE_BYTES<T, BI, BJ, DZ>], lds8* s1, lds8* s2) {
    constexpr int NTH = 64 * WI * WJ, BR = 128 / (int)sizeof(T), SI = BI / WI / 16, SJ = BJ / WJ / 16, V = CHUNK<T>;
    constexpr bool DMA = VEC && !DZ;
    const uint32_t tiles = A.ti * A.tj, w = xcd_run(id, count), split = w / tiles, t = w - split * tiles;
    const uint32_t band = t / (8 * A.tj), in = t - band * 8 * A.tj, high = A.ti - band * 8 < 8 ? A.ti - band * 8 : 8;
    const int64_t i0 = (int64_t)(band * 8 + in % high) * BI, j0 = (int64_t)(in / high) * BJ;
    const int64_t r0 = split * A.rsplit, rend = r0 + A.rsplit < A.R ? r0 + A.rsplit : A.R;
    const int nk = (int)((rend - r0 + BR - 1) / BR);
    const int wave = threadIdx.x >> 6, wi = wave % WI, wj = wave / WI;

    f4 acc[SI][SJ];
#pragma unroll
    for (int a = 0; a < SI; ++a)
#pragma unroll
        for (int b = 0; b < SJ; ++b) acc[a][b] = f4{0, 0, 0, 0};
    using SP = std::conditional_t<DZ, DzStager<T, BI, NTH, PT, VEC>,
                                  std::conditional_t<DMA, DmaStager<T, BI, NTH, PT>, Stager<T, BI, NTH, PT, VEC>>>;
    using SQ = std::conditional_t<DMA, DmaStager<T, BJ, NTH, QT>, Stager<T, BJ, NTH, QT, VEC>>;
    SP sp;
    SQ sq;
    const T* P = (const T*)A.P;
    const T* Q = (const T*)A.Q;
    PhiloxKey dkey{};
    if constexpr (DZ) {
        if (A.dz.drop.rng) dkey = philox_key(A.dz.drop.rng);
#pragma unroll
        for (int k = 0; k < V; ++k) sp.sum[k] = 0;
    }
    if constexpr (DMA) {
        sp.at(P, A.ldp, i0, A.I, r0);
        sq.at(Q, A.ldq, j0, A.J, r0);
    }
    // the stage at reduction r: its loads go out, into LDS or registers; what came to registers is put to LDS
    auto fetch = [&](lds8* lds, int64_t r) {
        if constexpr (DMA) {
            sp.load(lds, rend - r);
            sq.load(lds + BI * 128, rend - r);
        } else {
            if constexpr (DZ)
                sp.load(A, i0, A.I, r, rend);
            else
                sp.load(P, A.ldp, i0, A.I, r, rend, A.R);
            sq.load(Q, A.ldq, j0, A.J, r, rend, A.R);
        }
    };
    auto put = [&](lds8* lds, int64_t r) {
        if constexpr (!DMA) {
            if constexpr (DZ)
                sp.store(lds, lds + (BI + BJ) * 128, A, dkey, i0, r);
            else
                sp.store(lds);
            sq.store(lds + BI * 128);
        }
    };
    bool has_rest = false;
    if constexpr (DZ) has_rest = SP::has_rest(A);
    auto multiply_step = [&](const lds8* lp, auto ks) {
        u4v fp[SI], fq[SJ];
        fragments<T, SJ, BJ, QT, DMA, ks.value>(lp + BI * 128, wj * (BJ / WJ), fq);
        fragments<T, SI, BI, PT, DMA, ks.value>(lp, wi * (BI / WI), fp);
#pragma unroll
        for (int a = 0; a < SI; ++a)
#pragma unroll
            for (int b = 0; b < SJ; ++b) acc[a][b] = mma<T>(fq[b], fp[a], acc[a][b]);
        if constexpr (DZ && sizeof(T) == 2) {
            if (has_rest) {
                fragments<T, SI, BI, PT, DMA, ks.value>(lp + (BI + BJ) * 128, wi * (BI / WI), fp);
#pragma unroll
                for (int a = 0; a < SI; ++a)
#pragma unroll
                    for (int b = 0; b < SJ; ++b) acc[a][b] = mma<T>(fq[b], fp[a], acc[a][b]);
            }
        }
    };
    auto multiply = [&](const lds8* lp) {
        multiply_step(lp, std::integral_constant<int, 0>());
        multiply_step(lp, std::integral_constant<int, 1>());
    };
    lds8* const s0 = (lds8*)&stage0[0];
    if constexpr (DMA) {
        constexpr int NST = STAGES<true, DEEP>, LOADS = SP::NC + SQ::NC;
        constexpr int WAIT_ALL = 0x70;   // s_waitcnt's vmcnt and lgkmcnt at 0 (vmcnt: the low four bits), expcnt at its top
        static_assert(NST == 2 || LOADS < 16, "vmcnt's low bits");
        lds8* const st[3] = {s0, s1, s2};
        // Behind the barrier stage k has landed, for every wave, and the one before it has been read, so that the next but
        // one can be loaded over it.  The barrier is bare: a fence would wait for all loads.
        auto step = [&](auto i, int k) {
            asm volatile("" ::: "memory");
            if (NST == 3 && k + 1 < nk)
                __builtin_amdgcn_s_waitcnt(WAIT_ALL | LOADS);   // stage k + 1 may be on its way
            else
                __builtin_amdgcn_s_waitcnt(WAIT_ALL);
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (k + NST - 1 < nk) fetch(st[(i.value + NST - 1) % NST], r0 + (int64_t)(k + NST - 1) * BR);
            multiply(st[i.value]);
        };
        // the same with a stage to load for certain: then the compiler can tell that the older loads have landed
        auto step_on = [&](auto i, int k) {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(WAIT_ALL | LOADS);
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            fetch(st[(i.value + 2) % 3], r0 + (int64_t)(k + 2) * BR);
            multiply(st[i.value]);
        };
        int k = 0;
        if (NST == 3 && nk > 4) {
            fetch(st[0], r0);
            fetch(st[1], r0 + BR);
            do {
                step_on(std::integral_constant<int, 0>(), k);
                step_on(std::integral_constant<int, 1>(), k + 1);
                step_on(std::integral_constant<int, 2>(), k + 2);
                k += 3;
            } while (k + 4 < nk);
        } else {
#pragma unroll
            for (int q = 0; q < NST - 1; ++q)
                if (q < nk) fetch(st[q], r0 + (int64_t)q * BR);
        }
        for (; k < nk; k += NST) {
            step(std::integral_constant<int, 0>(), k);
            if (k + 1 < nk) step(std::integral_constant<int, 1>(), k + 1);
            if constexpr (NST == 3)
                if (k + 2 < nk) step(std::integral_constant<int, 2>(), k + 2);
        }
        __syncthreads();
    } else {
        // the stage that is filled: its last readers passed the barrier before this step
        auto step = [&](const lds8* now, lds8* next, int k) {
            const bool more = k + 1 < nk;
            const int64_t r = r0 + (int64_t)(k + 1) * BR;
            if (more) fetch(next, r);
            multiply(now);
            if (more) put(next, r);
            __syncthreads();
        };
        if (nk > 0) {
            fetch(s0, r0);
            put(s0, r0);
        }
        __syncthreads();
        for (int k = 0; k < nk; k += 2) {
            step(s0, s1, k);
            if (k + 1 < nk) step(s1, s0, k + 1);
        }
    }

    if constexpr (DZ && PT) {
        if (j0 == 0 && (A.dz.cols || A.dz.db)) {   // the bias gradient: this tile's columns, over this split's rows
            constexpr int CPR = BI / V, RP = NTH / CPR;
            static_assert(RP * BI * 4 <= (int)sizeof(stage0), "column sums");
            float* sums = reinterpret_cast<float*>(&stage0[0]);
#pragma unroll
            for (int k = 0; k < V; ++k) sums[threadIdx.x / CPR * BI + threadIdx.x % CPR * V + k] = sp.sum[k];
            __syncthreads();
            for (int c = threadIdx.x; c < BI && i0 + c < A.I; c += NTH) {
                float s = 0;
#pragma unroll 8
                for (int r = 0; r < RP; ++r) s += sums[r * BI + c];
                if (A.splits > 1)
                    A.dz.cols[split * A.I + i0 + c] = s;
                else
                    ((T*)A.dz.db)[i0 + c] = (T)(A.e.alpha * s);
            }
            __syncthreads();
        }
    }

    // A lane holds row row_of(a) and, for q = 0 .. SJ - 1, the columns col_of(q) .. + 3 of it (fragments_turned32: every SJ-th
    // or SI-th is its operand's).
    const int l = threadIdx.x & 63, g = l >> 4, n = l & 15;
    constexpr bool ROWS32 = PT && sizeof(T) == 4, COLS32 = QT && sizeof(T) == 4;
    auto row_of = [&](int a) { return wi * (BI / WI) + (ROWS32 ? SI * n + a : 16 * a + n); };
    auto col_of = [&](int q) { return wj * (BJ / WJ) + (COLS32 ? 4 * SJ * g + 4 * q : 16 * q + 4 * g); };
    auto four = [&](int a, int q) {
        if constexpr (!COLS32) return acc[a][q];
        f4 v;
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = acc[a][(4 * q + t) % SJ][(4 * q + t) / SJ];
        return v;
    };
    if (A.splits > 1) {
#pragma unroll
        for (int a = 0; a < SI; ++a) {
            const int64_t i = i0 + row_of(a);
#pragma unroll
            for (int q = 0; q < SJ; ++q) {
                const int64_t j = j0 + col_of(q);
                if (i >= A.I || j >= A.J) continue;
                const f4 x = four(a, q);
                const float v[4] = {x[0], x[1], x[2], x[3]};
                store_run(A.part + (split * A.I + i) * A.J + j, v, A.J - j < 4 ? (int)(A.J - j) : 4);
            }
        }
        return;
    }
    // The epilogue reads the tile back from LDS, 16 bytes of output a thread and whole row segments a wave, in a
    // short loop: unrolled over the accumulators it was 64 copies of the activations and generators, and the
    // instruction fetch took four times the product (silu at 4096 x 8192 x 2048: 884 us, 185 without it).
    // 16-byte chunks are XORed by the row: the 16 rows of a store hit 16 bank quads.  The tile goes through the
    // first stage in bands of rows.
    constexpr int BANDS = (BI * BJ * 4 + (int)sizeof(stage0) - 1) / (int)sizeof(stage0), BAND = BI / BANDS;
    constexpr int CPR = BJ / V, RPP = NTH / CPR;
    static_assert(BI % BANDS == 0 && BAND % 16 == 0 && BAND * BJ * 4 <= (int)sizeof(stage0) && NTH % CPR == 0 &&
                      BAND % RPP == 0, "epilogue tile");
    float* tile = reinterpret_cast<float*>(&stage0[0]);
    PhiloxKey key{};
    if (FULL && A.e.drop.rng) key = philox_key(A.e.drop.rng);
    KeepBits<V> keep;
    const int col = threadIdx.x % CPR * V;
#pragma unroll
    for (int band = 0; band < BANDS; ++band) {
        if (band) __syncthreads();
#pragma unroll
        for (int a = 0; a < SI; ++a) {
            const int i = row_of(a) - band * BAND;
            if (i < 0 || i >= BAND) continue;
#pragma unroll
            for (int q = 0; q < SJ; ++q)
                *reinterpret_cast<f4*>(tile + i * BJ + (((col_of(q) >> 2) ^ (i & 15)) << 2)) = four(a, q);
        }
        __syncthreads();
        const int64_t ib = i0 + band * BAND;
        if (j0 + col < A.J) {
#pragma unroll 1
            for (int i = threadIdx.x / CPR; i < BAND && ib + i < A.I; i += RPP) {
                float v[V];
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    const f4 x = *reinterpret_cast<const f4*>(tile + i * BJ + (((col / 4 + q) ^ (i & 15)) << 2));
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[4 * q + k] = x[k];
                }
                epilogue<T, FULL>(A.e, key, keep, A.I, A.J, ib + i, j0 + col, v);
            }
        }
    }
}

#define PSFM_STAGES(DMA, DZ)                                                                               \
    constexpr int BYTES = STAGE_BYTES<T, BI, BJ, DZ>;                                                      \
    __shared__ __attribute__((aligned(16))) uint8_t stage0[BYTES], stage1[BYTES], stage2[STAGES<DMA, DEEP> == 3 ? BYTES : 16]; \
    lds8* const s1 = (lds8*)&stage1[0];                                                                    \
    lds8* const s2 = (lds8*)&stage2[0];

template <typename T, int BI, int BJ, int WI, int WJ, bool VEC, bool DEEP>
__global__ __launch_bounds__(64 * WI * WJ, 2) void k_forward(const GemmArgs A) {
    PSFM_STAGES(VEC, false)
    product<T, BI, BJ, WI, WJ, false, false, VEC, true, false, DEEP>(A, blockIdx.x, gridDim.x, stage0, s1, s2);
}

template <typename T, int BI, int BJ, int WI, int WJ, bool VEC, bool DZ, bool DEEP>
__global__ __launch_bounds__(64 * WI * WJ, 2) void k_pair(const PairArgs A) {
    PSFM_STAGES(VEC && !DZ, DZ)
    if (blockIdx.x < A.ndw)
        product<T, BI, BJ, WI, WJ, true, true, VEC, false, DZ, DEEP>(A.dw, blockIdx.x, A.ndw, stage0, s1, s2);
    else
        product<T, BI, BJ, WI, WJ, false, true, VEC, false, DZ, DEEP>(A.dx, blockIdx.x - A.ndw, A.ndx, stage0, s1, s2);
}
#undef PSFM_STAGES

// y of 16 columns and up to 16 MT rows.  The 8 waves take turns in the reduction, 128 bytes of each row (two steps) a
// turn; each reads 16 rows of W straight into the matrix instructions' operands, U steps in flight, and x's few rows
// from the caches.
constexpr int SKINNY_WAVES = SKINNY_THREADS / 64;

template <typename T, int MT, bool VEC>
__global__ __launch_bounds__(64 * SKINNY_WAVES) void k_skinny(const SkinnyArgs A) {
    constexpr int V = CHUNK<T>, STEP = 4 * V, U = 16 / MT;
    __shared__ f4 part[SKINNY_WAVES][MT][64];
    const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, g = l >> 4, n = l & 15;
    const int64_t j0 = (int64_t)blockIdx.x * 16, j = j0 + n;
    const T* w = (const T*)A.w + (j < A.N ? j * A.K : 0);
    f4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = f4{0, 0, 0, 0};
    // the epilogue's thread, in the first MT waves: 4 columns (lane group g of the results) of one row.  Its inputs
    // are on their way while W is read (1 x 512 x 512 bf16: 4.25 -> 4.08 us; in the tiles the registers cost more than that gave).
    const int64_t i = wave * 16 + n, jj = j0 + 4 * g;
    float bias[4];
    T res[4];
    bias_run<T, true>(A.e, A.N, jj, bias);
    res_run<T, true>(A.e, A.M, A.N, i, jj, res);
    for (int64_t k0 = (int64_t)wave * 2 * STEP; k0 < A.K; k0 += SKINNY_WAVES * U * STEP) {
        u4v fw[U], fx[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t k = k0 + (u / 2 * 2 * SKINNY_WAVES + u % 2) * STEP + g * V, left = A.K - k;
            const int have = left >= V ? V : left > 0 ? (int)left : 0;
            fw[u] = load_n<T, VEC>(w + (have ? k : 0), j < A.N ? have : 0);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const int64_t row = m * 16 + n;
                fx[u][m] = load_n<T, VEC>((const T*)A.x + (row < A.M && have ? row * A.ldx + k : 0), row < A.M ? have : 0);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[m] = mma<T>(fw[u], fx[u][m], acc[m]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) part[wave][m][l] = acc[m];
    __syncthreads();
    if (wave >= MT) return;
    PhiloxKey key{};
    if (A.e.drop.rng) key = philox_key(A.e.drop.rng);
    if (i >= A.M || jj >= A.N) return;
    float v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < SKINNY_WAVES; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += part[s][wave][l][k];
    KeepBits<4> keep;
    epilogue<T, true>(A.e, key, keep, A.N, i, jj, v, bias, res);
}

// Split products: 256 / SL groups of four columns a workgroup, SL threads a group, each summing every SL-th split;
// the SL sums are added in order, then the epilogue.
template <typename T, bool FULL, int SL>
__device__ __forceinline__ void join(const GemmArgs& A, uint32_t block, f4* sums) {
    constexpr int G = 256 / SL;
    // a split product is small: its groups are counted in 32 bits
    const uint32_t cb = (uint32_t)((A.J + 3) >> 2), q = threadIdx.x % G, lane = threadIdx.x / G, id = block * G + q,
                   row = id / cb;
    const int64_t i = row, j = (int64_t)(id - row * cb) * 4;
    const int n = A.J - j < 4 ? (int)(A.J - j) : 4;
    const bool in = row < A.I;
    float v[4] = {0, 0, 0, 0};
    if (in) {
        const float* p = A.part + i * A.J + j;
#pragma unroll 4
        for (int s = lane; s < A.splits; s += SL) {
            float t[4];
            load_run(p + (int64_t)s * A.I * A.J, t, n);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += t[k];
        }
    }
    if (SL > 1) {
        sums[lane * G + q] = f4{v[0], v[1], v[2], v[3]};
        __syncthreads();
        if (lane) return;
        for (int s = 1; s < SL; ++s)
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += sums[s * G + q][k];
    }
    if (!in) return;
    PhiloxKey key{};
    if (FULL && A.e.drop.rng) key = philox_key(A.e.drop.rng);
    KeepBits<4> keep;
    epilogue<T, FULL>(A.e, key, keep, A.I, A.J, i, j, v);
}

// Up to JOIN_FEW splits one thread a group sums them all: 512 x 1024 over 4096 forward in bf16 16.1 us, 21.0 with JOIN_LANES;
// gradients of 30720 x 32 x 64, hundreds of splits: 16.2 with JOIN_LANES, 35.3 with one.
constexpr int JOIN_FEW = 8, JOIN_LANES = 16;

inline int64_t join_blocks(const GemmArgs& a) {
    const int64_t groups = a.I * ((a.J + 3) >> 2), per = a.splits <= JOIN_FEW ? 256 : 256 / JOIN_LANES;
    return (groups + per - 1) / per;
}
template <typename T, bool FULL>
__device__ __forceinline__ void join_any(const GemmArgs& A, uint32_t block, f4* sums) {
    if (A.splits <= JOIN_FEW)
        join<T, FULL, 1>(A, block, sums);
    else
        join<T, FULL, JOIN_LANES>(A, block, sums);
}

template <typename T>
__global__ __launch_bounds__(256) void k_join(const GemmArgs A) {
    __shared__ f4 sums[256];
    join_any<T, true>(A, blockIdx.x, sums);
}

// The bias gradient's parts: 16 columns a workgroup, 16 threads a column.
template <typename T>
__global__ __launch_bounds__(FINISH_THREADS) void k_finish(const FinishArgs A) {
    __shared__ f4 sums[256];
    if (blockIdx.x < A.ndx) {
        join_any<T, false>(A.dx, blockIdx.x, sums);
    } else if (blockIdx.x < A.ndx + A.ndw) {
        join_any<T, false>(A.dw, blockIdx.x - A.ndx, sums);
    } else {
        float* cs = reinterpret_cast<float*>(sums);
        const int c = threadIdx.x & 15, q = threadIdx.x >> 4;
        const int64_t col = (int64_t)(blockIdx.x - A.ndx - A.ndw) * 16 + c;
        float s = 0;
        if (col < A.N) {
#pragma unroll 8
            for (int64_t p = q; p < A.parts; p += 16) s += A.cols[p * A.N + col];
        }
        cs[q * 16 + c] = s;
        __syncthreads();
        if (q || col >= A.N) return;
        for (int r = 1; r < 16; ++r) s += cs[r * 16 + c];
        ((T*)A.db)[col] = (T)(A.alpha * s);
    }
}

// Workgroup (x, y): CB chunks of columns from x * CB, rows y * rows ..; 256 / CB rows at a time.
template <typename T, int CB>
__global__ __launch_bounds__(DZ_THREADS) void k_dz(const DzPassArgs A) {
    constexpr int RP = DZ_THREADS / CB, V = CHUNK<T>;
    __shared__ float sums[RP][CB * V];
    const int cx = threadIdx.x % CB, ry = threadIdx.x / CB;
    const int64_t j = ((int64_t)blockIdx.x * CB + cx) * V;
    const int n = A.N - j < V ? (int)(A.N - j) : V;
    const int64_t m0 = (int64_t)blockIdx.y * A.rows, m1 = m0 + A.rows < A.M ? m0 + A.rows : A.M;
    const DropArgs& drop = A.dz.drop;
    PhiloxKey key{};
    if (drop.rng) key = philox_key(drop.rng);
    KeepBits<V> keep;
    float sum[V];
#pragma unroll
    for (int k = 0; k < V; ++k) sum[k] = 0;
    if (n > 0) {
        for (int64_t m = m0 + ry; m < m1; m += RP) {
            float d[V];
            load_run((const T*)A.dy + m * A.N + j, d, n);
            if (A.dz.z) {
                float z[V];
                if (A.dz.act == PSFM_ACT_RELU)
                    load_run((const T*)A.dz.z + m * A.N + j, z, n);
                else
                    load_run((const typename KeptZ<T>::type*)A.dz.z + m * A.N + j, z, n);
                times_slope<T>(A.dz.act, z, d);
            }
            // last: a dropped value is 0 whatever dy and z hold
            if (drop.rng) drop_run(drop, key, keep, A.N, mask_row(drop, m), j, 1.0f, d);
            if (A.out) store_run((T*)A.out + m * A.N + j, d, n);
#pragma unroll
            for (int k = 0; k < V; ++k) sum[k] += d[k];
        }
    }
    if (!A.dz.cols) return;
#pragma unroll
    for (int k = 0; k < V; ++k) sums[ry][cx * V + k] = sum[k];
    __syncthreads();
    for (int c = threadIdx.x; c < CB * V; c += DZ_THREADS) {
        const int64_t col = (int64_t)blockIdx.x * CB * V + c;
        if (col >= A.N) continue;
        float s = 0;
#pragma unroll
        for (int r = 0; r < RP; ++r) s += sums[r][c];
        A.dz.cols[blockIdx.y * A.N + col] = s;
    }
}

// ---- launches --------------------------------------------------------------------------------
template <typename T>
bool deep(const GemmArgs& a) {
    return a.rsplit >= DEEP_STAGES * (128 / (int64_t)sizeof(T)) && a.R >= DEEP_STAGES * (128 / (int64_t)sizeof(T));
}

template <typename T, int BI, int BJ, int WI, int WJ, bool DEEP>
void launch_forward(bool vec, const GemmArgs& a, hipStream_t s) {
    static_assert(64 * WI * WJ == LINEAR_TILES[BI == 64 ? 0 : BI == 128 ? 1 : 2].threads, "a launch's threads");
    if (vec)
        k_forward<T, BI, BJ, WI, WJ, true, DEEP><<<dim3(a.blocks()), 64 * WI * WJ, 0, s>>>(a);
    else
        k_forward<T, BI, BJ, WI, WJ, false, false><<<dim3(a.blocks()), 64 * WI * WJ, 0, s>>>(a);
}
template <typename T>
int forward_of(int variant, bool vec, const GemmArgs& a, hipStream_t s) {
    if (variant == 0 && deep<T>(a))
        launch_forward<T, 64, 64, 2, 2, true>(vec, a, s);
    else if (variant == 0)
        launch_forward<T, 64, 64, 2, 2, false>(vec, a, s);
    else if (variant == 1 || sizeof(T) == 4)
        launch_forward<T, 128, 128, 2, 2, false>(vec, a, s);
    else if constexpr (sizeof(T) == 2)
        launch_forward<T, 256, 256, 2, 4, false>(vec, a, s);
    return (int)hipGetLastError();
}

template <typename T, int BI, int BJ, int WI, int WJ, bool DZ, bool DEEP>
void launch_pair(bool vec, const PairArgs& a, hipStream_t s) {
    const dim3 grid(a.ndx + a.ndw), block(64 * WI * WJ);
    if (vec)
        k_pair<T, BI, BJ, WI, WJ, true, DZ, DEEP><<<grid, block, 0, s>>>(a);
    else
        k_pair<T, BI, BJ, WI, WJ, false, DZ, false><<<grid, block, 0, s>>>(a);
}
// dz is made on the way only in the smallest tiles: the others have no registers left for it
template <typename T>
int pair_of(int variant, bool vec, bool dz, const PairArgs& a, hipStream_t s) {
    if (variant == 0 && dz)
        launch_pair<T, 64, 64, 2, 2, true, false>(vec, a, s);
    else if (variant == 0 && (a.ndx == 0 || deep<T>(a.dx)) && (a.ndw == 0 || deep<T>(a.dw)))
        launch_pair<T, 64, 64, 2, 2, false, true>(vec, a, s);
    else if (variant == 0)
        launch_pair<T, 64, 64, 2, 2, false, false>(vec, a, s);
    else if (variant == 1 || sizeof(T) == 4)
        launch_pair<T, 128, 128, 2, 2, false, false>(vec, a, s);
    else if constexpr (sizeof(T) == 2)   // whole chunks only
        k_pair<T, 256, 256, 2, 4, true, false, false><<<dim3(a.ndx + a.ndw), 512, 0, s>>>(a);
    return (int)hipGetLastError();
}

template <typename T>
int skinny_of(bool vec, const SkinnyArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)((a.N + 15) / 16)), block(64 * SKINNY_WAVES);
    if (a.M <= 16)
        vec ? k_skinny<T, 1, true><<<grid, block, 0, s>>>(a) : k_skinny<T, 1, false><<<grid, block, 0, s>>>(a);
    else
        vec ? k_skinny<T, 2, true><<<grid, block, 0, s>>>(a) : k_skinny<T, 2, false><<<grid, block, 0, s>>>(a);
    return (int)hipGetLastError();
}

template <typename T>
int join_of(const GemmArgs& a, hipStream_t s) {
    k_join<T><<<dim3((unsigned)join_blocks(a)), 256, 0, s>>>(a);
    return (int)hipGetLastError();
}

template <typename T>
int finish_of(FinishArgs& a, hipStream_t s) {
    a.ndx = a.dx.splits > 1 ? (uint32_t)join_blocks(a.dx) : 0;
    a.ndw = a.dw.splits > 1 ? (uint32_t)join_blocks(a.dw) : 0;
    a.ncol = a.db ? (uint32_t)((a.N + 15) / 16) : 0;
    if (a.ndx + a.ndw + a.ncol == 0) return 0;
    k_finish<T><<<dim3(a.ndx + a.ndw + a.ncol), FINISH_THREADS, 0, s>>>(a);
    return (int)hipGetLastError();
}

template <typename T>
int dz_of(const DzPassArgs& a, int64_t gx, int64_t gy, hipStream_t s) {
    const dim3 grid((unsigned)gx, (unsigned)gy);
    if (a.N <= DZ_NARROW * CHUNK<T>)
        k_dz<T, DZ_NARROW><<<grid, DZ_THREADS, 0, s>>>(a);
    else
        k_dz<T, DZ_WIDE><<<grid, DZ_THREADS, 0, s>>>(a);
    return (int)hipGetLastError();
}

template <typename T>
LinearOps ops() {
    return LinearOps{forward_of<T>, join_of<T>, skinny_of<T>, pair_of<T>, finish_of<T>, dz_of<T>};
}

}  // namespace
}  // namespace psfm
