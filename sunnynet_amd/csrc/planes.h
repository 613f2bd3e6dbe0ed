// Products of fp32 precision on the bf16 matrix cores: operands held as sums of
// bf16 planes (x = p0 + p1 + p2, each the rounding of what the planes before it
// leave). Three planes hold all 24 bits of an fp32 value, two an fp16 value, one a
// bf16 value, so the products of planes whose indices sum to less than LIM carry
// 8 LIM bits: LIM = 3 is fp32 to its last bit or two. Range is bf16's, which is
// fp32's, so nothing is scaled. A non-finite value leaves NaN planes.
//
// A 16x16x32 product reads eight contraction elements per lane. A lane's group
// g = lane / 16 holds, in this file's order, elements 4g..4g+3 and 16+4g..16+4g+3 of
// the 32: the rows that the lane holds of two 16x16 results stacked along that axis.
// So a result is the next product's right operand without leaving its registers, and
// tiles in LDS store their columns in the same order (perm_col).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace snhip {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct ElemPlanes;             // planes that hold a value of T exactly
template <> struct ElemPlanes<float> { static constexpr int n = 3; };
template <> struct ElemPlanes<_Float16> { static constexpr int n = 2; };
template <> struct ElemPlanes<__bf16> { static constexpr int n = 1; };

// One lane's operand of a product: P planes of eight elements.
template <int P> struct Frag { bf16x8 p[P]; };

template <int P> __device__ __forceinline__ Frag<P> split8(const float* x) {
    Frag<P> f;
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
    for (int p = 0; p < P; p++) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            f.p[p][i] = (__bf16)r[i];
            r[i] = r[i] - (float)f.p[p][i];
        }
    }
    return f;
}

// acc += a b over the plane pairs with i + j < LIM, the smallest first.
template <int LIM, int NA, int NB>
__device__ __forceinline__ f32x4 mma(const Frag<NA>& a, const Frag<NB>& b, f32x4 acc) {
#pragma unroll
    for (int s = LIM - 1; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < NA; i++) {
            const int j = s - i;
            if (j >= 0 && j < NB)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.p[i], b.p[j], acc, 0, 0, 0);
        }
    return acc;
}

// Where column c of a row is stored (a multiple of 4 columns moves as one).
__host__ __device__ constexpr int perm_col(int c) {
    return (c & ~31) + ((c & 12) << 1) + ((c & 16) >> 2) + (c & 3);
}

// A tile of P planes of R rows and C columns in LDS. Rows are padded by 8 elements
// (16 bytes), which spreads a product's 16 rows over the banks.
template <int P, int R, int C> struct Tile {
    static constexpr int ld = C + 8;
    static constexpr int elems = P * R * ld;
    __bf16* s;
    __device__ __forceinline__ __bf16* at(int p, int r, int c) const { return s + (p * R + r) * ld + c; }
    // The operand of rows r0..r0+15, contraction columns 32 ks..32 ks + 31.
    template <int Q = P> __device__ __forceinline__ Frag<Q> frag(int r0, int ks, int lane) const {
        Frag<Q> f;
#pragma unroll
        for (int p = 0; p < Q; p++)
            f.p[p] = *reinterpret_cast<const bf16x8*>(at(p, r0 + (lane & 15), 32 * ks + 8 * (lane >> 4)));
        return f;
    }
    // Four neighbouring columns (c a multiple of 4) of one row.
    __device__ __forceinline__ void put4(int r, int c, const float* x) const {
        float t[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int p = 0; p < P; p++) {
            bf16x4 h;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                h[i] = (__bf16)t[i];
                t[i] = t[i] - (float)h[i];
            }
            *reinterpret_cast<bf16x4*>(at(p, r, perm_col(c))) = h;
        }
    }
    __device__ __forceinline__ void put(int r, int c, float x) const {
#pragma unroll
        for (int p = 0; p < P; p++) {
            const __bf16 h = (__bf16)x;
            *at(p, r, perm_col(c)) = h;
            x = x - (float)h;
        }
    }
    __device__ __forceinline__ float get(int r, int c) const {
        float x = 0.f;
#pragma unroll
        for (int p = P - 1; p >= 0; p--) x += (float)*at(p, r, perm_col(c));
        return x;
    }
};

// Eight consecutive elements from `src`, of which the first `n` exist (the rest
// are 0). vec: the address is 16-byte aligned.
template <typename T> __device__ __forceinline__ void load8(const T* src, int n, bool vec, float* x) {
    if (vec && n >= 8) {
        if constexpr (sizeof(T) == 4) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(src), b = *reinterpret_cast<const f32x4*>(src + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = a[i], x[4 + i] = b[i];
        } else {
            typedef T T8 __attribute__((ext_vector_type(8)));
            const T8 a = *reinterpret_cast<const T8*>(src);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = (float)a[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = i < n ? (float)src[i] : 0.f;
    }
}

}  // namespace snhip
