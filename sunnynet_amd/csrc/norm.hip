// Layer norm over rows, forward and backward.
//
//   xh = (x - mean) rstd     y = xh w + b
//   dx = rstd (e - mean(e) - xh mean(e xh)), e = dy w
//   dw = sum over rows of dy xh             db = sum over rows of dy
//
// Bound by HBM: forward one read and one write of the rows, backward two reads and one
// write. WPR waves hold one row in registers, NV vectors of eight values a lane, so
// the mean, the centred variance and the result come from one read. The backward's
// lanes keep their columns from row to row and add up dw and db in registers; a block
// leaves one partial row of each, and a second kernel sums those in a fixed order.
#include "common.h"
#include "planes.h"
#include "snhip_ops.h"

namespace snhip {
namespace {

constexpr int kNormMaxD = 16384;
constexpr int kNormBlocks = 256;       // partial rows of the backward, at most: a block a CU

template <typename T> __device__ __forceinline__ void store8(T* dst, int n, bool vec, const float* x) {
    if (vec && n >= 8) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<f32x4*>(dst) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4*>(dst + 4) = f32x4{x[4], x[5], x[6], x[7]};
        } else {
            typedef T T8 __attribute__((ext_vector_type(8)));
            T8 t;
#pragma unroll
            for (int i = 0; i < 8; i++) t[i] = (T)x[i];
            *reinterpret_cast<T8*>(dst) = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) dst[i] = (T)x[i];
    }
}

// Sum of one value per lane over the WPR waves of a row; `slot` holds one float per
// wave of the block, and consecutive calls need different ones.
template <int WPR> __device__ __forceinline__ float row_sum(float x, float* slot, int wave) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    if constexpr (WPR > 1) {
        slot[wave] = x;
        __syncthreads();
        x = 0.f;
        for (int i = 0; i < WPR; i++) x += slot[wave / WPR * WPR + i];
    }
    return x;
}

constexpr int norm_waves(int wpr) { return wpr < 4 ? 4 : wpr; }     // waves of a block

// 32768 rows of 1024 in bf16: 25 to 26 us, 5.1 to 5.4 TB/s.
template <typename T, int NV, int WPR>
__global__ __launch_bounds__(64 * norm_waves(WPR)) void k_norm_fwd(const T* x, const float* w, const float* b, T* y,
                                                                   float* mean, float* rstd, int64_t R, int D,
                                                                   float eps, bool vec) {
    __shared__ float slot[2][norm_waves(WPR)];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * (norm_waves(WPR) / WPR) + wave / WPR;
    const bool live = row < R;       // a dead row still takes part in the block's barriers
    float v[NV][8], s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = ((i * WPR + wave % WPR) * 64 + lane) * 8;
        load8(x + row * D + c, live ? D - c : 0, vec, v[i]);
#pragma unroll
        for (int j = 0; j < 8; j++) s += v[i][j];
    }
    const float mu = row_sum<WPR>(s, slot[0], wave) / (float)D;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = ((i * WPR + wave % WPR) * 64 + lane) * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            v[i][j] = c + j < D ? v[i][j] - mu : 0.f;
            s = fmaf(v[i][j], v[i][j], s);
        }
    }
    const float rs = 1.f / sqrtf(row_sum<WPR>(s, slot[1], wave) / (float)D + eps);
    if (!live) return;
    if (mean && lane == 0 && wave % WPR == 0) {
        mean[row] = mu;
        rstd[row] = rs;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = ((i * WPR + wave % WPR) * 64 + lane) * 8;
#pragma unroll
        for (int j = 0; j < 8; j++) v[i][j] *= rs;
        if (w) {
            float t[8];
            load8(w + c, D - c, vec, t);
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] *= t[j];
        }
        if (b) {
            float t[8];
            load8(b + c, D - c, vec, t);
#pragma unroll
            for (int j = 0; j < 8; j++) v[i][j] += t[j];
        }
        store8(y + row * D + c, D - c, vec, v[i]);
    }
}

constexpr int kBwdWaves = 16;          // waves of a block of the backward

// 32768 rows of 1024 in bf16: 39 us, 5.1 TB/s. Rows wider than 4096 spill 7 to 23 of 128
// registers.
template <typename T, int NV, int WPR>
__global__ __launch_bounds__(64 * kBwdWaves) void k_norm_bwd(const T* dy, const T* x, const float* w, const float* mean,
                                                             const float* rstd, T* dx, float* part, int64_t R, int D,
                                                             bool vec) {
    constexpr int RPB = kBwdWaves / WPR;
    __shared__ float slot[4][kBwdWaves];
    __shared__ float acc[RPB][RPB > 1 ? NV * WPR * 512 : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr bool hold = WPR <= 4;       // the weights too; wider rows have no registers left
    float ws[NV][8], aw[NV][8], ab[NV][8];
    auto weights = [&](int i) {
        const int c = ((i * WPR + wave % WPR) * 64 + lane) * 8;
        if (w) load8(w + c, D - c, vec, ws[i]);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (!w) ws[i][j] = 1.f;
    };
#pragma unroll
    for (int i = 0; i < NV; i++) {
        if (hold) weights(i);
#pragma unroll
        for (int j = 0; j < 8; j++) aw[i][j] = ab[i][j] = 0.f;
    }
    int odd = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < R; r0 += (int64_t)gridDim.x * RPB, odd ^= 2) {
        const int64_t row = r0 + wave / WPR;
        const bool live = row < R;
        const float mu = live ? mean[row] : 0.f, rs = live ? rstd[row] : 0.f;
        float g[NV][8], h[NV][8], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = ((i * WPR + wave % WPR) * 64 + lane) * 8;
            load8(dy + row * D + c, live ? D - c : 0, vec, g[i]);
            load8(x + row * D + c, live ? D - c : 0, vec, h[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = ((i * WPR + wave % WPR) * 64 + lane) * 8;
            if (!hold) weights(i);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                h[i][j] = live && c + j < D ? (h[i][j] - mu) * rs : 0.f;
                aw[i][j] = fmaf(g[i][j], h[i][j], aw[i][j]);
                ab[i][j] += g[i][j];
                g[i][j] *= ws[i][j];
                s1 += g[i][j];
                s2 = fmaf(g[i][j], h[i][j], s2);
            }
        }
        if (!dx) continue;
        const float m1 = row_sum<WPR>(s1, slot[odd], wave) / (float)D;
        const float m2 = row_sum<WPR>(s2, slot[odd + 1], wave) / (float)D;
        if (live)
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = ((i * WPR + wave % WPR) * 64 + lane) * 8;
#pragma unroll
                for (int j = 0; j < 8; j++) g[i][j] = rs * (g[i][j] - m1 - h[i][j] * m2);
                store8(dx + row * D + c, D - c, vec, g[i]);
            }
    }
    if (!part) return;
    // one partial row of dw, then of db, per block
#pragma unroll
    for (int k = 0; k < 2; k++) {
        float* out = part + (blockIdx.x * (int64_t)2 + k) * D;
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    acc[wave / WPR][((i * WPR + wave % WPR) * 64 + lane) * 8 + j] = k ? ab[i][j] : aw[i][j];
            __syncthreads();
            for (int c = threadIdx.x; c < D; c += 64 * kBwdWaves) {
                float t = 0.f;
                for (int i = 0; i < RPB; i++) t += acc[i][c];
                out[c] = t;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = ((i * WPR + wave % WPR) * 64 + lane) * 8;
                store8(out + c, D - c, false, k ? ab[i] : aw[i]);
            }
        }
    }
}

// dw (blockIdx.y = 0) or db (1): 64 columns of n partial rows, 16 waves. 256 rows of 1024:
// 4 us; 1024 rows, from four times the blocks, took 20.
__global__ __launch_bounds__(1024) void k_norm_sum(const float* part, float* dw, float* db, int n, int D) {
    __shared__ float s[16][64];
    float* out = blockIdx.y ? db : dw;
    if (!out) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
    float t = 0.f;
    if (c < D)
#pragma unroll 16
        for (int i = wave; i < n; i += 16) t += part[((int64_t)2 * i + blockIdx.y) * D + c];
    s[wave][lane] = t;
    __syncthreads();
    if (wave == 0 && c < D) {
        t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) t += s[i][lane];
        out[c] = t;
    }
}

// Waves per row: the fewest whose lanes hold the row in two vectors each.
template <typename F> snhip_status norm_shape(int64_t D, F f) {
    if (D <= 512) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 1>());
    if (D <= 1024) return f(std::integral_constant<int, 2>(), std::integral_constant<int, 1>());
    if (D <= 2048) return f(std::integral_constant<int, 2>(), std::integral_constant<int, 2>());
    if (D <= 4096) return f(std::integral_constant<int, 2>(), std::integral_constant<int, 4>());
    if (D <= 8192) return f(std::integral_constant<int, 2>(), std::integral_constant<int, 8>());
    return f(std::integral_constant<int, 2>(), std::integral_constant<int, 16>());
}

int norm_wpr(int64_t D) { return D <= 1024 ? 1 : D <= 2048 ? 2 : D <= 4096 ? 4 : D <= 8192 ? 8 : 16; }

// Blocks of the backward, one partial row each.
int64_t norm_blocks(int64_t R, int64_t D) {
    const int64_t rpb = kBwdWaves / norm_wpr(D), n = (R + rpb - 1) / rpb;
    return n < kNormBlocks ? n : kNormBlocks;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T>
snhip_status norm_fwd_t(const void* x, const float* w, const float* b, void* y, float* mean, float* rstd, int64_t R,
                        int64_t D, float eps, hipStream_t st) {
    const bool vec = D % 8 == 0 && aligned(x) && aligned(y) && aligned(w) && aligned(b);
    return norm_shape(D, [&](auto nv, auto wpr) -> snhip_status {
        constexpr int NV = decltype(nv)::value, WPR = decltype(wpr)::value, RPB = norm_waves(WPR) / WPR;
        // a grid holds fewer than 2^32 threads: more rows go in several launches
        constexpr int64_t most = (int64_t)RPB << 21;
        for (int64_t r = 0; r < R; r += most) {
            const int64_t n = R - r < most ? R - r : most;
            k_norm_fwd<T, NV, WPR><<<(unsigned)((n + RPB - 1) / RPB), 64 * norm_waves(WPR), 0, st>>>(
                (const T*)x + r * D, w, b, (T*)y + r * D, mean ? mean + r : nullptr, rstd ? rstd + r : nullptr, n,
                (int)D, eps, vec);
            SNHIP_CHECK(hipGetLastError());
        }
        return SNHIP_OK;
    });
}

template <typename T>
snhip_status norm_bwd_t(const void* dy, const void* x, const float* w, const float* mean, const float* rstd, void* dx,
                        float* dw, float* db, float* ws, int64_t R, int64_t D, hipStream_t st) {
    const bool vec = D % 8 == 0 && aligned(dy) && aligned(x) && aligned(w) && aligned(dx);
    const int n = (int)norm_blocks(R, D);
    const bool sums = dw || db;
    return norm_shape(D, [&](auto nv, auto wpr) -> snhip_status {
        constexpr int NV = decltype(nv)::value, WPR = decltype(wpr)::value;
        k_norm_bwd<T, NV, WPR><<<n, 64 * kBwdWaves, 0, st>>>(
            (const T*)dy, (const T*)x, w, mean, rstd, (T*)dx, sums ? ws : nullptr, R, (int)D, vec);
        SNHIP_CHECK(hipGetLastError());
        if (sums) {
            k_norm_sum<<<dim3((unsigned)((D + 63) / 64), 2), 1024, 0, st>>>(ws, dw, db, n, (int)D);
            SNHIP_CHECK(hipGetLastError());
        }
        return SNHIP_OK;
    });
}

bool norm_bad(int64_t R, int64_t D, int32_t dtype) {
    return R < 1 || R > INT32_MAX || D < 1 || D > kNormMaxD || dtype < SNHIP_F32 || dtype > SNHIP_F16;
}

}  // namespace
}  // namespace snhip

using namespace snhip;

extern "C" {

snhip_status snhip_op_norm_fwd_dev(const void* x, const float* w, const float* b, void* y, float* mean, float* rstd,
                                   int64_t R, int64_t D, float eps, int32_t dtype, void* stream) {
    if (norm_bad(R, D, dtype) || !x || !y || !mean != !rstd) return SNHIP_E_INVAL;
    const hipStream_t st = as_stream(stream);
    if (dtype == SNHIP_F32) return norm_fwd_t<float>(x, w, b, y, mean, rstd, R, D, eps, st);
    if (dtype == SNHIP_BF16) return norm_fwd_t<__bf16>(x, w, b, y, mean, rstd, R, D, eps, st);
    return norm_fwd_t<_Float16>(x, w, b, y, mean, rstd, R, D, eps, st);
}

int64_t snhip_op_norm_bwd_floats(int64_t R, int64_t D) { return norm_bad(R, D, 0) ? 0 : 2 * D * norm_blocks(R, D); }

snhip_status snhip_op_norm_bwd_dev(const void* dy, const void* x, const float* w, const float* mean,
                                   const float* rstd, void* dx, float* dw, float* db, float* ws, int64_t R, int64_t D,
                                   int32_t dtype, void* stream) {
    if (norm_bad(R, D, dtype) || !dy || !x || !mean || !rstd || ((dw || db) && !ws)) return SNHIP_E_INVAL;
    const hipStream_t st = as_stream(stream);
    if (dtype == SNHIP_F32) return norm_bwd_t<float>(dy, x, w, mean, rstd, dx, dw, db, ws, R, D, st);
    if (dtype == SNHIP_BF16) return norm_bwd_t<__bf16>(dy, x, w, mean, rstd, dx, dw, db, ws, R, D, st);
    return norm_bwd_t<_Float16>(dy, x, w, mean, rstd, dx, dw, db, ws, R, D, st);
}

}  // extern "C"
