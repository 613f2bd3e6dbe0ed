// Shared pieces of the gated delta rule's kernels (delta.hip, deltabwd.hip).
//
// Mathematics, per sequence and value head, in chunks of C = 32 tokens. With c the
// running sum of g inside the chunk, G_i = exp(c_i), D_ij = exp(c_i - c_j) for j <= i
// (0 above), S the state before the chunk and everything row by token:
//   N_ij = D_ij k_i.k_j (j < i)              M = (I + N diag(beta))^-1
//   X = V - G (K S)    E = M X (the errors)  U = beta E (the writes)
//   P_ij = scale D_ij q_i.k_j (j <= i)       O = scale G (Q S) + P U
//   S' = G_C S + K^T (L U)                   L_j = exp(c_C - c_j)
// All exponents are differences of running sums, held in 64 bits: their difference
// keeps its digits after a strong decay. They are never positive for g <= 0.
//
// M, P, G, L and beta depend on no state: k_delta_prep makes them for all chunks at
// once. What is left is sequential over chunks but independent over the columns of V:
// a wave owns 16 of them and keeps its (K, 16) of the state in registers, where the
// results of one product are the operand of the next (planes.h); LDS only holds the
// tiles that all columns share. Rows of K and tokens are both taken in pair_row's order.
#pragma once

#include <type_traits>

#include "common.h"
#include "planes.h"
#include "snhip_ops.h"

namespace snhip {

constexpr int kDC = 32;                            // tokens per chunk
// Per chunk and head, in floats: M and P as three bf16 planes of 32 x 32 each, then G, L
// and beta (32 each).
constexpr int kDeltaP = 3 * kDC * kDC / 2, kDeltaG = 2 * kDeltaP, kDeltaChunk = kDeltaG + 3 * kDC;

// Tokens of a call: positions inside a sequence, and a part's end past it, fit 32 bits.
constexpr int64_t kDeltaTokens = (1 << 30) - 1;
// Chunks of a call: the kernels launch up to 512 threads for each, in one dimension of a
// grid that holds fewer than 2^32.
constexpr int64_t kDeltaSlots = (1 << 23) - 1;
// The longest call that runs token by token without workspaces. 12 tokens, calls with their
// host work: one sequence, 12 heads of 64 in fp32, 13.2 us token by token and 18.7 in chunks;
// 64 sequences, 16 heads of 128 in bf16, 45 and 78 (57 and 78 at 16 tokens).
constexpr int kDeltaStepTokens = 12;
// Waves of a block of the scans, 16 columns of V each.
constexpr int kDeltaW = 4;
// Token strides stay below this, so that offsets inside a chunk fit 32 bits.
constexpr int64_t kDeltaStride = 1 << 24;

struct DeltaP {
    SnHipDelta d;
    int64_t slots, groups;  // chunk slots of all sequences; groups of NS chunks
    int KP, VP;             // K and V padded: saved states are (KP, VP), errors (VP, 32 NS)
    int rep;                // value heads per query and key head
    int segs, seg_chunks;   // parts of a sequence that are scanned at once, and their chunks
    float* seg_state;       // per sequence, part and head: delta_seg_floats
    bool vec;               // every eight elements of a row of q or k are 16-byte aligned
};

// Whether a call's sizes and type are in the documented ranges.
inline bool delta_in_range(const SnHipDelta& d) {
    return d.B >= 1 && d.T >= 1 && d.N >= 1 && d.N <= 65535 && d.H >= 1 && d.H <= 65535 && d.Hk >= 1 &&
           d.H % d.Hk == 0 && d.K >= 1 && d.K <= 128 && d.V >= 1 && d.V <= 4096 && d.T <= kDeltaTokens / d.B &&
           (d.cu ? d.B == 1 : d.N == d.B) && d.H * d.V < kDeltaStride && d.H * d.K < kDeltaStride &&
           d.dtype >= SNHIP_F32 && d.dtype <= SNHIP_F16;
}

__host__ __device__ inline int64_t delta_slots(const SnHipDelta& d) {
    return d.cu ? d.T / kDC + d.N : d.B * ((d.T + kDC - 1) / kDC);
}
__host__ __device__ inline int delta_kp(int64_t K) { return K <= 64 ? 64 : 128; }
__host__ __device__ inline int delta_vp(int64_t V) { return (int)((V + 15) / 16 * 16); }

// The backward takes NS chunks at a time, and states are kept per such group. Two halve the
// bytes of the states: forward and backward of 8 x 2048 tokens, 16 heads of 128 in bf16,
// take 1.05 ms with two and 1.35 with one. Heads of up to 64 have a quarter of those bytes,
// and their tiles of one chunk leave room for more blocks on a CU (0.65 ms with one, 0.73
// with two); three planes of fp32 leave no room for two.
__host__ __device__ constexpr int delta_ns(int64_t dtype, int64_t K) { return dtype == SNHIP_F32 || K <= 64 ? 1 : 2; }
__host__ __device__ inline int64_t delta_groups(const SnHipDelta& d) {
    const int64_t n = kDC * delta_ns(d.dtype, d.K);
    return d.cu ? d.T / n + d.N : d.B * ((d.T + n - 1) / n);
}
// What the forward keeps for the backward, per group and head: S (KP, VP) before it, and
// behind all of those E^T (VP, 32 NS).
__host__ __device__ inline float* delta_state(const DeltaP& a, int64_t group, int h) {
    return a.d.states + (group * a.d.H + h) * (int64_t)(a.VP * a.KP);
}
__host__ __device__ inline float* delta_errors(const DeltaP& a, int64_t group, int h) {
    return a.d.states + a.groups * a.d.H * (int64_t)(a.VP * a.KP) +
           (group * a.d.H + h) * (int64_t)(a.VP * kDC * delta_ns(a.d.dtype, a.d.K));
}

// Few heads and a long sequence leave the scan a handful of waves. Then the sequence is
// scanned in parts: over a part the state is an affine map of the state before it,
// S' = A S + B, where B is what the scan makes of S = 0 and A what it makes of S = I with
// no values: K more columns. One pass makes A and B of all parts, a small kernel joins
// them, and the ordinary scan runs over all parts at once from their true states. This is
// 2 to 3 times the work. Per part and head: (KP, VP + KP) for [B A], then (KP, VP) for S.
__host__ __device__ inline int64_t delta_seg_floats(int KP, int VP) { return (int64_t)KP * (2 * VP + KP); }
// Waves that fill the card (256 CUs of four SIMDs), and the fewest chunks worth a part.
constexpr int kDeltaWaves = 1024, kDeltaSegChunks = 32;
inline int delta_segs(const SnHipDelta& d) {
    const int64_t waves = (int64_t)d.H * d.N * (delta_vp(d.V) / 16), chunks = (d.T + kDC - 1) / kDC;
    int64_t n = kDeltaWaves / waves;
    if (n > chunks / kDeltaSegChunks) n = chunks / kDeltaSegChunks;
    // Below four parts the second pass and the join take what the first one gives. 16384
    // tokens, 16 heads of 128 in fp16: 1,776 us in one part, 537 in eight.
    return n < 4 ? 1 : n > 16 ? 16 : (int)n;
}

// A sequence: its first token as a row of the contiguous arrays, its batch entry and
// first token there, its length, and the slot of its first chunk. With cu the slots of
// a sequence begin at cu[n] / 32 + n, which leaves every sequence enough of them.
struct DeltaSeq {
    int64_t row, b, t0, slot, group;
    int len;
};
__device__ __forceinline__ int64_t delta_edge(const SnHipDelta& d, int64_t n) {
    const int64_t e = d.cu[n];
    return e < 0 ? 0 : e > d.T ? d.T : e;
}
__device__ __forceinline__ DeltaSeq delta_seq(const SnHipDelta& d, int64_t n) {
    DeltaSeq s;
    if (d.cu) {
        const int64_t a = delta_edge(d, n), e = delta_edge(d, n + 1);
        s.row = s.t0 = a;
        s.b = 0;
        s.len = (int)(e > a ? e - a : 0);
        s.slot = a / kDC + n;
        s.group = a / (kDC * delta_ns(d.dtype, d.K)) + n;
    } else {
        s.row = n * d.T;
        s.t0 = 0;
        s.b = n;
        s.len = (int)d.T;
        s.slot = n * ((d.T + kDC - 1) / kDC);
        const int64_t c = kDC * delta_ns(d.dtype, d.K);
        s.group = n * ((d.T + c - 1) / c);
    }
    return s;
}
// The sequence and chunk of a slot (C = kDC), or the sequence and group of a group's
// number (C = kDC NS); false for one that is not used.
template <int C> __device__ __forceinline__ bool delta_chunk_of(const SnHipDelta& d, int64_t slot, DeltaSeq* s, int* chunk) {
    int64_t n;
    if (d.cu) {
        int64_t lo = 0, hi = d.N - 1;          // the last sequence that begins at or before the slot
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) / 2;
            if (delta_edge(d, mid) / C + mid <= slot) lo = mid;
            else hi = mid - 1;
        }
        n = lo;
    } else {
        n = slot / ((d.T + C - 1) / C);
    }
    *s = delta_seq(d, n);
    const int64_t c = slot - (C == kDC ? s->slot : s->group);
    *chunk = (int)c;
    return c >= 0 && c * C < s->len;
}

template <typename T>
__device__ __forceinline__ const T* delta_at(const void* p, const int64_t* st, int64_t b, int64_t t, int64_t h) {
    return static_cast<const T*>(p) + b * st[0] + t * st[1] + h * st[2];
}

// An (R, KP) tile of a (tokens, K) array on its way from memory to LDS, held by NTH
// threads: rows from n on and columns from K on are 0.
template <typename T, int KP, int NTH, bool VEC, int R = kDC> struct RowsFetch {
    static constexpr int P = ElemPlanes<T>::n, N = (R * KP / 8 + NTH - 1) / NTH;
    static constexpr bool whole = R * KP / 8 % NTH == 0;
    Vec8<T> x[N];
    int off[N];            // of this thread's vectors in any chunk
    __device__ __forceinline__ void init(int64_t stride, int K, int tid) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = tid + j * NTH, t = i / (KP / 8), c = i % (KP / 8) * 8;
            off[j] = c < K ? (t * (int)stride + c) * (int)sizeof(T) : kNowhere;
        }
    }
    __device__ __forceinline__ void load(const T* src, int64_t stride, int n, int K, int tid) {
        const __amdgpu_buffer_rsrc_t r = rows_window(src, stride, n, K);
#pragma unroll
        for (int j = 0; j < N; j++) x[j] = buf_load8<T>(r, off[j], K - (tid + j * NTH) % (KP / 8) * 8, VEC);
    }
    __device__ __forceinline__ void store(Tile<P, R, KP> to, int tid) const {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = tid + j * NTH, t = i / (KP / 8), c = i % (KP / 8) * 8;
            if (whole || t < R) to.put8(t, c, split_raw8<T>(x[j]));
        }
    }
};

// The three planes of a (32, 32) matrix of a chunk's record (at float `at`), likewise.
// The matrix's place is part of the vector offset, which the hardware checks against the
// record; threads past the planes fetch nothing.
template <int NTH> struct MatFetch {
    static constexpr int Q = 3;
    static constexpr int N = (Q * 128 + NTH - 1) / NTH;
    static constexpr bool whole = Q * 128 % NTH == 0;
    bf16x8 x[N];
    // Of vector i, in bytes from the record's start.
    static constexpr int offset(int i, int at) { return whole || i < Q * 128 ? at * 4 + i * 16 : kNowhere; }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rec, int at, int tid) {
#pragma unroll
        for (int j = 0; j < N; j++)
            x[j] = __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(rec, offset(tid + j * NTH, at), 0, 0));
    }
    __device__ __forceinline__ void store(Tile<Q, kDC, kDC> to, int tid) const {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = tid + j * NTH;
            if (whole || i < Q * 128) *reinterpret_cast<bf16x8*>(to.at(i >> 7, (i >> 2) & 31, (i & 3) * 8)) = x[j];
        }
    }
};

// f(element type, padded K, vector loads) of a call, as values of types that name them.
template <typename F> snhip_status delta_pick(const DeltaP& a, F f) {
    auto by_vec = [&](auto t, auto kp) {
        return a.vec ? f(t, kp, std::true_type()) : f(t, kp, std::false_type());
    };
    auto by_k = [&](auto t) {
        return a.KP == 64 ? by_vec(t, std::integral_constant<int, 64>()) : by_vec(t, std::integral_constant<int, 128>());
    };
    return a.d.dtype == SNHIP_F32 ? by_k(float()) : a.d.dtype == SNHIP_BF16 ? by_k(__bf16()) : by_k(_Float16());
}

// g as the kernels use it: exp(-200) is 0 in fp32, and a sum of 32 such stays finite.
__device__ __forceinline__ float delta_decay(float g) { return g < -200.f ? -200.f : g; }

}  // namespace snhip
