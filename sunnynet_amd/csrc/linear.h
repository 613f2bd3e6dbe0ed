// Linear attention with a decay for each head (linear*.hip).
//
// Mathematics, per sequence and value head, with a = exp(g):
//   S_t = a_t S_{t-1} + k_t v_t^T        out_t = scale S_t^T q_t
// and, with R_t the gradient of S_t, R_t = a_{t+1} R_{t+1} + scale q_t dO_t^T:
//   dq_t = scale S_t dO_t        dv_t = R_t^T k_t        dk_t = R_t v_t
//   dg_t = sum over i >= t of (q_i.dq_i - k_i.dk_i) + <S_T, dS_T>
// (a token's own share is the same in q_i.dq_i and in k_i.dk_i and left out of both, not
// cancelled). All four are one recurrence of rows A, B (contracted) and C (columns):
//   y_i = sum over j of w_ij (A_i.B_j) C_j + (row factor) S^T A_i,   S += B_j C_j^T
// out: (q, k, v) forward in time; dq: (dO, v, k) forward, on S transposed; dv: (k, q, dO)
// backward in time, on R; dk: (v, dO, q) backward, on R transposed. So one kernel does all.
//
// In chunks of C tokens, c the running sum of g inside the chunk, held in 64 bits (their
// differences keep their digits after a strong decay):
//   forward:   P_ij = scale e^(c_i - c_j) A_i.B_j (j <= i)   y = scale e^(c_i) A S + P C
//              S' = e^(c_C) S + sum of B_j e^(c_C - c_j) C_j^T
//   backward:  P_ij = scale e^(c_j - c_i) A_i.B_j (j >= i)   y = e^(c_C - c_i) A S + P C
//              S' = e^(c_C) S + sum of B_j scale e^(c_j) C_j^T
//
// Without a correction the state of a part of a sequence is an affine map of the state
// before it whose matrix is one number, e^(sum of g): parts of a sequence are summed from
// zero at once (k_lin, STATE), joined (k_lin_join), and then run from their true states.
//
// Products are of fp32 precision (planes.h): a wave owns 16 NC columns of C and keeps its
// rows of S in registers, as results that are the next product's operand.
#pragma once

#include "common.h"
#include "planes.h"
#include "snhip_ops.h"

namespace snhip {

constexpr int64_t kLinTokens = (1 << 30) - 1;      // positions fit 32 bits
constexpr int64_t kLinStride = 1 << 24;            // token strides: offsets inside a chunk fit 32 bits
constexpr int kLinWaves = 4;                       // of a block, and so the parts of a dot
constexpr int kLinRows = 128;                      // contracted rows of a block: all of K, or of a block of V

// A call's sizes, and the parts into which its sequences are cut: `part` tokens each. The
// parts of sequence n are the slots from first(n) on.
struct LinShape {
    const float* g;
    const int32_t* cu;
    int64_t B, T, N, H, K, V, slots;
    int part;               // tokens
    int per_seq;            // parts of a sequence, without cu
    bool head_g;            // g is (H), not (B,T,H)
    bool split;             // more parts than one per sequence can be
    bool narrow;            // blocks of 64 columns, not 128
    float scale;
};

struct LinSeq {
    int64_t row, b, t0;     // first token: as a row of contiguous arrays, batch entry, place there
    int64_t slot;           // of its first part
    int len;
};
__device__ __forceinline__ int64_t lin_edge(const LinShape& d, int64_t n) {
    const int64_t e = d.cu[n];
    return e < 0 ? 0 : e > d.T ? d.T : e;
}
__device__ __forceinline__ LinSeq lin_seq(const LinShape& d, int64_t n) {
    LinSeq s;
    if (d.cu) {
        const int64_t a = lin_edge(d, n), e = lin_edge(d, n + 1);
        s.row = s.t0 = a;
        s.b = 0;
        s.len = (int)(e > a ? e - a : 0);
        s.slot = (unsigned)a / (unsigned)d.part + n;
    } else {
        s.row = n * d.T;
        s.t0 = 0;
        s.b = n;
        s.len = (int)d.T;
        s.slot = n * d.per_seq;
    }
    return s;
}
// The sequence and part of a slot, for a whole wave. False for a slot that is not used; an
// empty sequence has one part of no tokens. The lanes look at 64 sequences a step (by halves
// a step is a load's latency for each bit of N).
__device__ __forceinline__ bool lin_part_of(const LinShape& d, unsigned slot, LinSeq* s, int64_t* seq, int* part) {
    unsigned n = 0;                            // the last sequence that begins at or before the slot
    if (d.cu) {
        for (unsigned left = (unsigned)d.N; left > 1;) {
            const unsigned step = (left + 63) / 64, i = (threadIdx.x & 63) * step;
            const bool before = i < left && (unsigned)lin_edge(d, n + i) / (unsigned)d.part + n + i <= slot;
            const unsigned some = __popcll(__ballot(before)), to = some ? (some - 1) * step : 0;
            n += to;
            left = step < left - to ? step : left - to;
        }
    } else {
        n = slot / (unsigned)d.per_seq;
    }
    *s = lin_seq(d, n);
    *seq = n;
    const int64_t p = (int64_t)slot - s->slot;
    *part = (int)p;
    return p == 0 || (p > 0 && p * d.part < s->len);
}

// An operand of (tokens, heads, columns): strides in elements, last axis contiguous; `rep`
// value heads share one of its heads.
struct LinRows {
    const void* p;
    int64_t st[3];          // batch, token, head
    int rep;
};
template <typename T> __device__ __forceinline__ const T* lin_at(const LinRows& r, int64_t b, int64_t t, int64_t h) {
    return static_cast<const T*>(r.p) + b * r.st[0] + t * r.st[1] + h / r.rep * r.st[2];
}

// One recurrence. States are (K, V) in memory; in the runs with dots (dq and dk) the rows of S
// are V's.
struct LinPass {
    LinRows A, B, C, X;     // X: with which y is multiplied for the decay's gradient
    int rows, cols;         // A's and C's columns
    bool vec;               // every eight elements of a row of A, B, C and X are 16-byte aligned (X's too)
    const float* begin;     // (N,H,K,V) the state at the sequence's (backward: last) first token, or null
    float* end;             // (N,H,K,V) the state after all tokens, or null
    float* parts;           // (slots,H,K,V): of every part the state it begins with (STATE: writes its own sum)
    float* decay;           // (slots,H): STATE writes e^(sum of g)
    void* y;                // T (B,T,H / y_rep,cols), or fp32 per slice (y_f32)
    int y_rep;
    bool y_f32;
    bool y_vec;             // every four elements of a row of y are aligned
    float* dot;             // (blocks of rows, blocks of columns, waves, H, B T): a wave's part of X_i.y_i without the token's own share
};


// Runs a pass: kind 0 plain, 1 with dots, 2 states of the parts.
snhip_status lin_run_f32(const LinShape& d, const LinPass& a, bool rev, int kind, hipStream_t st);
snhip_status lin_run_bf16(const LinShape& d, const LinPass& a, bool rev, int kind, hipStream_t st);
snhip_status lin_run_f16(const LinShape& d, const LinPass& a, bool rev, int kind, hipStream_t st);

// g as the kernels use it: exp(-200) is 0 in fp32, and a sum of such stays finite.
__device__ __forceinline__ float lin_decay(float g) { return g < -200.f ? -200.f : g; }

}  // namespace snhip
