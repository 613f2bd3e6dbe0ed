// Products of fp32 precision on the bf16 matrix cores: operands held as sums of
// bf16 planes (x = p0 + p1 + p2, each the rounding of what the planes before it
// leave). Three planes hold all 24 bits of an fp32 value, two an fp16 value, one a
// bf16 value, so the products of planes whose indices sum to less than LIM carry
// 8 LIM bits: LIM = 3 is fp32 to its last bit or two. Range is bf16's, which is
// fp32's, so nothing is scaled. A non-finite value leaves NaN planes.
//
// A 16x16x32 product reads eight contraction elements per lane: lane group g = lane / 16
// holds elements 8g..8g+7 of the 32, of row (left) or column (right) lane % 16. Of the
// 16x16 result the lane holds rows 4g..4g+3 of column lane % 16. Two results make 32
// rows, and which row of the matrix a row of a left operand stands for is free: with row
// i of result m standing for row pair_row(m, i) = 8 (i / 4) + 4 m + i % 4, the lane holds
// rows 8g..8g+7 of its column, in order. So a pair of results is the next product's
// right operand without leaving its registers.
//
// Tiles in LDS are row by row, eight neighbouring values (16 bytes a plane) to a write.
// An operand whose contraction runs along a row is read as it stands (frag); one whose
// contraction runs down the columns through the transposing LDS read (tfrag), which
// hands four rows of a 4x16 block to the lane of each column.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "bufio.h"

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
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    Frag<P> f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {       // by pairs: one instruction rounds and packs two
        f32x2 r = {x[i], x[i + 1]};
#pragma unroll
        for (int p = 0; p < P; p++) {
            const bf16x2 h = __builtin_convertvector(r, bf16x2);
            f.p[p][i] = h[0];
            f.p[p][i + 1] = h[1];
            if (p + 1 < P) r = r - __builtin_convertvector(h, f32x2);
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

// The same for N left operands at once: neighbouring products are independent, so none
// waits for the one before it.
template <int LIM, int N, int NA, int NB>
__device__ __forceinline__ void mma_n(const Frag<NA> (&a)[N], const Frag<NB>& b, f32x4 (&acc)[N]) {
#pragma unroll
    for (int s = LIM - 1; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < NA; i++) {
            const int j = s - i;
            if (j >= 0 && j < NB)
#pragma unroll
                for (int n = 0; n < N; n++)
                    acc[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[n].p[i], b.p[j], acc[n], 0, 0, 0);
        }
}

__device__ __forceinline__ int pair_row(int m, int i) { return 8 * (i >> 2) + 4 * m + (i & 3); }

// A tile of P planes of R rows and C columns in LDS. Rows are padded by 16 bytes, which
// spreads the 16 rows of a frag over the banks; a tile that is only read transposed does
// better with rows 64 bytes apart modulo 256, which spreads the four rows of a tfrag.
template <int P, int R, int C, int PAD = 8> struct Tile {
    static constexpr int ld = C + PAD;
    static constexpr int elems = P * R * ld;
    __bf16* s;
    __device__ __forceinline__ __bf16* at(int p, int r, int c) const { return s + (p * R + r) * ld + c; }
    // Row `row` (one per lane % 16), contraction columns c0..c0 + 31.
    template <int Q = P> __device__ __forceinline__ Frag<Q> frag(int row, int c0, int lane) const {
        Frag<Q> f;
#pragma unroll
        for (int p = 0; p < Q; p++) f.p[p] = *reinterpret_cast<const bf16x8*>(at(p, row, c0 + 8 * (lane >> 4)));
        return f;
    }
    // Contraction rows r0..r0 + 31; the lane's column is that of lane % 16 in the four
    // blocks of four columns, of which the one at `block` is this lane's to fetch
    // (block index lane % 4): columns 16 t + i: block = 16 t + 4 (lane % 4); columns
    // pair_row(m, i): block = 8 (lane % 4) + 4 m. The whole wave takes part.
    template <int Q = P> __device__ __forceinline__ Frag<Q> tfrag(int r0, int block, int lane) const {
        Frag<Q> f;
        const int r = r0 + 8 * (lane >> 4) + ((lane >> 2) & 3);
#pragma unroll
        for (int p = 0; p < Q; p++) {
            const bf16x4 lo = tread(at(p, r, block)), hi = tread(at(p, r + 4, block));
            f.p[p] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return f;
    }
    static __device__ __forceinline__ bf16x4 tread(__bf16* a) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds4;
        return __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)a));
    }
    // Eight neighbouring columns (c a multiple of 8) of one row.
    __device__ __forceinline__ void put8(int r, int c, const float* x) const { put8(r, c, split8<P>(x)); }
    __device__ __forceinline__ void put8(int r, int c, const Frag<P>& f) const {
#pragma unroll
        for (int p = 0; p < P; p++) *reinterpret_cast<bf16x8*>(at(p, r, c)) = f.p[p];
    }
    __device__ __forceinline__ void put(int r, int c, float x) const {
#pragma unroll
        for (int p = 0; p < P; p++) {
            const __bf16 h = (__bf16)x;
            *at(p, r, c) = h;
            x = x - (float)h;
        }
    }
    __device__ __forceinline__ float get(int r, int c) const {
        float x = 0.f;
#pragma unroll
        for (int p = P - 1; p >= 0; p--) x += (float)*at(p, r, c);
        return x;
    }
};

template <typename T> using Vec8 = T __attribute__((ext_vector_type(8)));

// Eight consecutive floats from a 16-byte aligned address.
__device__ __forceinline__ Vec8<float> load_floats8(const float* src) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(src), b = *reinterpret_cast<const f32x4*>(src + 4);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A window of n rows of `len` elements, `stride` elements apart, as a buffer: an offset
// past it reads 0 and writes nothing, so no row or column needs a branch. kNowhere is
// such an offset. Strides are below 2^24 elements, so offsets fit 32 bits.
constexpr int kNowhere = (int)0x80000000u;
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_window(const T* p, int64_t stride, int n, int len) {
    return make_rsrc(p, (uint32_t)((uint32_t)(n - 1) * (uint32_t)stride + (uint32_t)len) * (uint32_t)sizeof(T));
}
template <typename T> __device__ __forceinline__ T buf_load(__amdgpu_buffer_rsrc_t r, int off) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
    else return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0));
}
// The same as a register of its own, to be held while later work runs: 16-bit values
// would be packed in pairs on arrival, which waits for them.
template <typename T> __device__ __forceinline__ unsigned buf_load_bits(__amdgpu_buffer_rsrc_t r, int off) {
    if constexpr (sizeof(T) == 4) return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
    else return (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
}
template <typename T> __device__ __forceinline__ float float_of_bits(unsigned b) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(b);
    else return (float)__builtin_bit_cast(T, (unsigned short)b);
}
template <typename T> __device__ __forceinline__ void buf_store(__amdgpu_buffer_rsrc_t r, int off, T x) {
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), r, off, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(short, x), r, off, 0, 0);
}
__device__ __forceinline__ f32x4 buf_load4(__amdgpu_buffer_rsrc_t r, int off) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
__device__ __forceinline__ void buf_store4(__amdgpu_buffer_rsrc_t r, int off, f32x4 x) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), r, off, 0, 0);
}
// Eight elements from `off`, of which the first n are wanted (n < 8 only without vec);
// vec: 16-byte aligned.
template <typename T> __device__ __forceinline__ Vec8<T> buf_load8(__amdgpu_buffer_rsrc_t r, int off, int n, bool vec) {
    Vec8<T> x;
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const f32x4 a = buf_load4(r, off), b = buf_load4(r, off + 16);
            x = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            x = __builtin_bit_cast(Vec8<T>, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = buf_load<T>(r, i < n ? off + i * (int)sizeof(T) : kNowhere);
    }
    return x;
}

// The planes of eight elements, without arithmetic where one plane is the value.
template <typename T> __device__ __forceinline__ Frag<ElemPlanes<T>::n> split_raw8(const Vec8<T>& v) {
    if constexpr (ElemPlanes<T>::n == 1) {
        return Frag<1>{{v}};
    } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)v[i];
        return split8<ElemPlanes<T>::n>(x);
    }
}

// Sum over the 16 lanes of a row, by row-local lane exchanges in the adder's operand.
template <int CTRL> __device__ __forceinline__ float add_dpp(float x) {
    return x + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float sum16(float x) {
    x = add_dpp<0xb1>(x);         // lanes 1, 0, 3, 2
    x = add_dpp<0x4e>(x);         // 2, 3, 0, 1
    x = add_dpp<0x141>(x);        // mirrored within 8
    return add_dpp<0x140>(x);     // and within 16
}

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
