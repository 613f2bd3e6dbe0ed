// The common norm of many tensors and the scaling to a bound: gradient clipping.
//
//   norm = sqrt(sum of all x^2)        y = x min(1, max_norm / (norm + 1e-6))
//
// Bound by memory: every x is read for the sum, and once more, with y written, where the
// factor is not 1. The tensors' addresses and sizes travel in the kernels' arguments, 128
// tensors a launch: nothing is copied to the device and nothing kept, so a capture holds
// all of it. Work goes by pieces of kClipPiece elements, which a block finds by the pieces'
// running count; a block sums the squares of its pieces in 64 bits (a square of fp32 does
// not overflow there) into one partial sum, and the blocks of the second kernel each add
// all partial sums again in the same order, which is cheaper than a launch between the two.
// 102 M fp32 values: 74 us for the sums, 164 for the scaling (5.1 and 5.0 TB/s; the sums find
// part of what an earlier pass read in the cache).
// The second kernels go through the pieces backwards: what the first ones read last is still
// in the last-level cache (256 MB), and what they write is kept out of it (102 M fp32: 249 us
// with ordinary stores, 238 so; bf16 135 and 114).
#include <algorithm>
#include <vector>

#include "common.h"
#include "planes.h"
#include "snhip_ops.h"

namespace snhip {
namespace {

constexpr int kClipTensors = 128, kClipBlocks = 1024;
constexpr int64_t kClipPiece = 8192;
constexpr int64_t kClipMost = (int64_t)1 << 36;       // elements of a tensor: 128 of them make at most 2^30 pieces

struct ClipTable {
    const void* x[kClipTensors];
    void* y[kClipTensors];
    int64_t n[kClipTensors];
    int first[kClipTensors + 1];       // pieces before tensor i
    unsigned char dtype[kClipTensors];
    int count;
};
static_assert(sizeof(ClipTable) <= 3900, "kernel arguments");

// f(first of eight elements, how many of them exist) of a piece, for this thread's part.
template <typename F> __device__ __forceinline__ void clip_each(int64_t n, int64_t piece, F f) {
    const int64_t i0 = piece * kClipPiece, i1 = i0 + kClipPiece < n ? i0 + kClipPiece : n;
#pragma unroll 2
    for (int64_t i = i0 + 8 * (int)threadIdx.x; i < i1; i += 8 * 256) f(i, (int)(i1 - i < 8 ? i1 - i : 8));
}

template <typename T> __device__ __forceinline__ double clip_squares(const T* x, int64_t n, int64_t piece) {
    const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0;
    double s = 0.;
    clip_each(n, piece, [&](int64_t i, int m) {
        float v[8];
        load8<T>(x + i, m, vec, v);
#pragma unroll
        for (int e = 0; e < 8; e++) s = fma((double)v[e], (double)v[e], s);
    });
    return s;
}

template <typename T> __device__ __forceinline__ void clip_scale(const T* x, T* y, int64_t n, int64_t piece, float factor) {
    const bool vec = (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % 16 == 0;
    clip_each(n, piece, [&](int64_t i, int m) {
        float v[8];
        load8<T>(x + i, m, vec, v);
        if (vec && m == 8) {
            typedef T T8 __attribute__((ext_vector_type(8), aligned(16)));
            T8 o;
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = (T)(v[e] * factor);
            __builtin_nontemporal_store(o, reinterpret_cast<T8*>(y + i));
        } else {
            for (int e = 0; e < m; e++) y[i + e] = (T)(v[e] * factor);
        }
    });
}

// f(tensor, its piece) for the pieces of this block, from the first or from the last.
template <bool BACK, typename F> __device__ __forceinline__ void clip_pieces(const ClipTable& t, F f) {
    const int all = t.first[t.count];
    for (int i = blockIdx.x; i < all; i += gridDim.x) {
        const int p = BACK ? all - 1 - i : i;
        int lo = 0, hi = t.count - 1;          // the last tensor that begins at or before p
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (t.first[mid] <= p) lo = mid;
            else hi = mid - 1;
        }
        f(lo, p - t.first[lo]);
    }
}

__device__ __forceinline__ double clip_block_sum(double v) {
    __shared__ double w[4];
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) w[threadIdx.x >> 6] = v;
    __syncthreads();
    return (w[0] + w[1]) + (w[2] + w[3]);
}

__global__ __launch_bounds__(256) void k_clip_sum(ClipTable t, double* partial) {
    double s = 0.;
    clip_pieces<false>(t, [&](int i, int64_t piece) {
        if (t.dtype[i] == SNHIP_F32) s += clip_squares(static_cast<const float*>(t.x[i]), t.n[i], piece);
        else if (t.dtype[i] == SNHIP_BF16) s += clip_squares(static_cast<const __bf16*>(t.x[i]), t.n[i], piece);
        else s += clip_squares(static_cast<const _Float16*>(t.x[i]), t.n[i], piece);
    });
    s = clip_block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double clip_norm(const double* partial, int64_t partials) {
    double s = 0.;
    for (int64_t i = threadIdx.x; i < partials; i += 256) s += partial[i];
    return sqrt(clip_block_sum(s));
}

__global__ __launch_bounds__(256) void k_clip_norm(const double* partial, int64_t partials, float* norm) {
    const double n = clip_norm(partial, partials);
    if (threadIdx.x == 0) *norm = (float)n;
}

__global__ __launch_bounds__(256) void k_clip_scale(ClipTable t, const double* partial, int64_t partials, double max_norm, float* norm) {
    // a bound without end scales nothing, beside an infinite value neither
    const double n = clip_norm(partial, partials), f = isinf(max_norm) && isinf(n) ? 1. : max_norm / (n + 1e-6);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const float factor = f >= 1. ? 1.f : (float)f;         // NaN stays
    clip_pieces<true>(t, [&](int i, int64_t piece) {
        if (factor == 1.f && t.x[i] == t.y[i]) return;
        if (t.dtype[i] == SNHIP_F32) clip_scale(static_cast<const float*>(t.x[i]), static_cast<float*>(t.y[i]), t.n[i], piece, factor);
        else if (t.dtype[i] == SNHIP_BF16)
            clip_scale(static_cast<const __bf16*>(t.x[i]), static_cast<__bf16*>(t.y[i]), t.n[i], piece, factor);
        else clip_scale(static_cast<const _Float16*>(t.x[i]), static_cast<_Float16*>(t.y[i]), t.n[i], piece, factor);
    });
}

// Whether any y overlaps another y or an x other than the one it replaces.
bool clip_overlaps(const SnHipClip& c) {
    struct Span {
        uintptr_t a, e;
        bool out;
    };
    std::vector<Span> s;
    s.reserve((size_t)c.count * 2);
    for (int64_t i = 0; i < c.count; i++) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(c.x[i]), y = reinterpret_cast<uintptr_t>(c.y[i]),
                        b = (uintptr_t)c.n[i] * (c.dtype[i] == SNHIP_F32 ? 4 : 2);
        if (!b) continue;
        s.push_back({y, y + b, true});
        if (x != y) s.push_back({x, x + b, false});
    }
    std::sort(s.begin(), s.end(), [](const Span& a, const Span& b) { return a.a < b.a; });
    uintptr_t any = 0, out = 0;        // ends of what came before
    for (const Span& p : s) {
        if (p.a < (p.out ? any : out)) return true;
        any = std::max(any, p.e);
        if (p.out) out = std::max(out, p.e);
    }
    return false;
}

int64_t clip_launches(int64_t count) { return (count + kClipTensors - 1) / kClipTensors; }

snhip_status clip_run(const SnHipClip& c, float* norm, hipStream_t st) {
    for (int64_t i = 0; i < c.count; i++)
        if (c.n[i] < 0 || c.n[i] >= kClipMost || c.dtype[i] < SNHIP_F32 || c.dtype[i] > SNHIP_F16 ||
            (c.n[i] && (!c.x[i] || (c.y && !c.y[i]))))
            return SNHIP_E_INVAL;
    if (c.y && clip_overlaps(c)) return SNHIP_E_INVAL;
    std::vector<ClipTable> tables;
    for (int64_t at = 0; at < c.count; at++) {
        const int64_t pieces = (c.n[at] + kClipPiece - 1) / kClipPiece;
        if (!pieces) continue;
        if (tables.empty() || tables.back().count == kClipTensors) {
            tables.emplace_back();
            tables.back().count = tables.back().first[0] = 0;
        }
        ClipTable& t = tables.back();
        t.x[t.count] = c.x[at];
        t.y[t.count] = c.y ? c.y[at] : nullptr;
        t.n[t.count] = c.n[at];
        t.dtype[t.count] = (unsigned char)c.dtype[at];
        t.first[t.count + 1] = t.first[t.count] + (int)pieces;
        t.count++;
    }
    auto grid = [&](const ClipTable& t) { return (unsigned)std::min<int64_t>(t.first[t.count], kClipBlocks); };
    int64_t partials = 0;
    for (const ClipTable& t : tables) {
        k_clip_sum<<<grid(t), 256, 0, st>>>(t, c.ws + partials);
        SNHIP_CHECK(hipGetLastError());
        partials += grid(t);
    }
    if (!c.y || !partials) {
        k_clip_norm<<<1, 256, 0, st>>>(c.ws, partials, norm);
        SNHIP_CHECK(hipGetLastError());
    } else {
        for (size_t i = tables.size(); i-- > 0;) {
            k_clip_scale<<<grid(tables[i]), 256, 0, st>>>(tables[i], c.ws, partials, c.max_norm, i ? nullptr : norm);
            SNHIP_CHECK(hipGetLastError());
        }
    }
    return SNHIP_OK;
}

}  // namespace
}  // namespace snhip

using namespace snhip;

extern "C" {

int64_t snhip_op_clip_doubles(int64_t count) {
    return count < 0 || count >= 1 << 20 ? 0 : std::max<int64_t>(1, clip_launches(count)) * kClipBlocks;
}

snhip_status snhip_op_clip_dev(const SnHipClip* c, float* norm, void* stream) {
    if (!c || !norm || !c->ws || c->count < 0 || c->count >= 1 << 20 || (c->count && (!c->x || !c->n || !c->dtype)))
        return SNHIP_E_INVAL;
    try {
        return clip_run(*c, norm, as_stream(stream));
    } catch (...) {
        return SNHIP_E_NOMEM;          // of the host
    }
}

}  // extern "C"
