// Gated delta rule, forward: the per-chunk matrices, the chunked scan and the
// token-by-token form. Mathematics and layout: delta.h.
#include "delta.h"

namespace snhip {
namespace {

// M, P, G, L, beta of one chunk and value head: a block of four waves, one 16x16 tile
// of the 32x32 matrices each. The inverse of the unit lower triangular I + A,
// A = N diag(beta), goes by halves: its two diagonal 16x16 blocks by forward substitution,
// a column per lane, then M10 = -M11 A10 M00. M and P are left as the planes in which the
// scans multiply them. Bound by the latency of its steps, hidden by the blocks of a CU:
// 50 us for 8 x 2048 tokens, 16 heads of 128 in bf16 (4.7 TB/s of what its blocks read
// and write).
template <typename T, int KP, bool VEC>
__global__ __launch_bounds__(256) void k_delta_prep(DeltaP a) {
    constexpr int P = ElemPlanes<T>::n;
    __shared__ alignas(16) __bf16 sk[Tile<P, kDC, KP>::elems], sq[Tile<P, kDC, KP>::elems];
    __shared__ double sc[kDC];
    __shared__ float sb[kDC], sA[kDC][kDC + 1], sM[kDC][kDC + 1], sP[kDC][kDC + 1], sT[16][17];
    const SnHipDelta& d = a.d;
    const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15;
    DeltaSeq s;
    int chunk;
    if (!delta_chunk_of<kDC>(d, blockIdx.x, &s, &chunk)) return;
    const int64_t t0 = (int64_t)chunk * kDC;
    const int n = (int)(s.len - t0 < kDC ? s.len - t0 : kDC);
    const Tile<P, kDC, KP> K{sk}, Q{sq};
    RowsFetch<T, KP, 256, VEC> fk, fq;
    fk.init(d.k_stride[1], (int)d.K, tid);
    fq.init(d.q_stride[1], (int)d.K, tid);
    fk.load(delta_at<T>(d.k, d.k_stride, s.b, s.t0 + t0, h / a.rep), d.k_stride[1], n, (int)d.K, tid);
    fq.load(delta_at<T>(d.q, d.q_stride, s.b, s.t0 + t0, h / a.rep), d.q_stride[1], n, (int)d.K, tid);
    if (wave == 0) {
        const int64_t at = (s.row + t0 + lane) * d.H + h;
        double c = lane < n ? (double)delta_decay(d.g[at]) : 0.0;
#pragma unroll
        for (int o = 1; o < kDC; o <<= 1) {
            const double y = __shfl_up(c, o, kDC);
            if ((lane & 31) >= o) c += y;
        }
        if (lane < kDC) {
            sc[lane] = c;
            sb[lane] = lane < n ? d.beta[at] : 0.f;
        }
    }
    fk.store(K, tid);
    fq.store(Q, tid);
    __syncthreads();
    float* out = d.chunks + ((int64_t)blockIdx.x * d.H + h) * kDeltaChunk;
    const int ti = wave >> 1, tj = wave & 1, col = tj * 16 + l16;
    f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
    if (tj <= ti) {
#pragma unroll
        for (int c = 0; c < KP; c += 32) {
            const Frag<P> b = K.frag(16 * tj + l16, c, lane);
            kk = mma<3>(K.frag(16 * ti + l16, c, lane), b, kk);
            qk = mma<3>(Q.frag(16 * ti + l16, c, lane), b, qk);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int row = ti * 16 + (lane >> 4) * 4 + r;
        const float D = col <= row ? expf((float)(sc[row] - sc[col])) : 0.f;
        sA[row][col] = col < row ? sb[col] * D * kk[r] : 0.f;
        sP[row][col] = col <= row ? (float)d.scale * D * qk[r] : 0.f;
    }
    if (tid < kDC) {
        out[kDeltaG + tid] = expf((float)sc[tid]);
        out[kDeltaG + kDC + tid] = expf((float)(sc[kDC - 1] - sc[tid]));
        out[kDeltaG + 2 * kDC + tid] = sb[tid];
    }
    __syncthreads();
    if (tid < 32) {
        const int o = tid & 16, c = tid & 15;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float v = i == c ? 1.f : 0.f;
#pragma unroll
            for (int j = 0; j < i; j++) v = fmaf(-sA[o + i][o + j], x[j], v);
            x[i] = v;
            sM[o + i][o + c] = v;
        }
    }
    __syncthreads();
    {
        const int i = tid >> 4, j = tid & 15;
        float v = 0.f;
#pragma unroll
        for (int l = 0; l < 16; l++) v = fmaf(sA[16 + i][l], sM[l][j], v);
        sT[i][j] = v;
        sM[i][16 + j] = 0.f;
    }
    __syncthreads();
    {
        const int i = tid >> 4, j = tid & 15;
        float v = 0.f;
#pragma unroll
        for (int l = 0; l < 16; l++) v = fmaf(-sM[16 + i][16 + l], sT[l][j], v);
        sM[16 + i][j] = v;
    }
    __syncthreads();
    {
        // eight values a thread: M by the first two waves, P by the others
        const int i = tid & 127, row = i >> 2, c = (i & 3) * 8;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = tid < 128 ? sM[row][c + j] : sP[row][c + j];
        const Frag<3> f = split8<3>(x);
        float* to = out + (tid < 128 ? 0 : kDeltaP) + i * 4;
#pragma unroll
        for (int p = 0; p < 3; p++) *reinterpret_cast<bf16x8*>(to + p * 512) = f.p[p];
    }
}

// The scan over chunks: kDeltaW waves, 16 columns of V each. The next chunk's tiles are
// fetched into registers while this one is worked on, and put into the other half of LDS:
// one barrier per chunk, no wait for memory in between. Bound by the chain of a chunk's
// products (each waits for the one before), of which a SIMD has one to three waves to
// overlap: 8 x 2048 tokens, 16 heads of 128 in bf16 take 217 us, 286 with the states and
// errors kept for the backward. PASS 0 scans whole sequences or, from
// the states that the join left, the parts of sequences; PASS 1 makes the parts' maps:
// columns from VP on are those of A, and there is no output.
template <typename T, int KP, bool VEC, int PASS>
__global__ __launch_bounds__(64 * kDeltaW) void k_delta_scan(DeltaP a, T* out, float* send) {
    constexpr int P = ElemPlanes<T>::n, NK = KP / 16, W = kDeltaW, NTH = 64 * W;
    constexpr int NS = sizeof(T) == 4 || KP == 64 ? 1 : 2;
    typedef Tile<P, kDC, KP> Rows;
    typedef Tile<3, kDC, kDC> Mat;
    __shared__ alignas(16) __bf16 sk[2][Rows::elems], sq[2][Rows::elems], sm[2][Mat::elems], sp[2][Mat::elems];
    __shared__ alignas(16) float sv[2][3 * kDC];
    const SnHipDelta& d = a.d;
    const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g8 = (lane >> 4) * 8;
    const int64_t seq = blockIdx.z / a.segs;
    const int seg = blockIdx.z % a.segs;
    const DeltaSeq s = delta_seq(d, seq);
    const int begin = seg * a.seg_chunks * kDC;
    // a part that the sequence does not reach, or (for the maps) whose end is the sequence's
    if (seg && begin >= s.len) return;
    const bool last = a.segs == 1 || begin + a.seg_chunks * kDC >= s.len;
    if (PASS == 1 && (last || (seg == 0 && (int)blockIdx.x * 16 * W >= a.VP))) return;      // part 0's A is not used
    const int stop = last ? s.len : begin + a.seg_chunks * kDC;
    const int v = (blockIdx.x * W + wave) * 16 + l16, V = (int)d.V, Kd = (int)d.K;
    const int64_t sbase = (seq * d.H + h) * d.K * d.V;
    float* part = a.segs > 1 ? a.seg_state + ((seq * a.segs + seg) * d.H + h) * delta_seg_floats(KP, a.VP) : nullptr;
    const T* kp = delta_at<T>(d.k, d.k_stride, s.b, s.t0, h / a.rep);
    const T* qp = delta_at<T>(d.q, d.q_stride, s.b, s.t0, h / a.rep);
    const T* vp = delta_at<T>(d.v, d.v_stride, s.b, s.t0, h);
    const float* rec = d.chunks + (s.slot * d.H + h) * kDeltaChunk;

    f32x4 S[NK];           // S[2 p + e][r] is row 32 p + g8 + 4 e + r of column v
#pragma unroll
    for (int kt = 0; kt < NK; kt++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int k = (kt >> 1) * 32 + g8 + 4 * (kt & 1) + r;
            if (PASS == 1 && v >= a.VP) S[kt][r] = k == v - a.VP ? 1.f : 0.f;
            else if (seg == 0) S[kt][r] = d.s0 && k < Kd && v < V ? d.s0[sbase + (int64_t)k * V + v] : 0.f;
            else S[kt][r] = PASS == 0 && v < a.VP ? part[(int64_t)KP * (a.VP + KP) + k * a.VP + v] : 0.f;
        }
    RowsFetch<T, KP, NTH, VEC> fk, fq;
    MatFetch<NTH> fm, fp;
    float fv[(3 * kDC + NTH - 1) / NTH];
    unsigned vv[8];
    fk.init(d.k_stride[1], Kd, tid);
    fq.init(d.q_stride[1], Kd, tid);
    const int E = (int)sizeof(T), v_step = (int)d.v_stride[1] * E, v_off = v < V ? g8 * v_step + v * E : kNowhere;
    const int o_step = (int)d.H * V * E, o_off = v < V ? g8 * o_step + v * E : kNowhere;
    auto fetch = [&](int t0) {
        const int n = s.len - t0 < kDC ? s.len - t0 : kDC;
        const __amdgpu_buffer_rsrc_t r = make_rsrc(rec + (int64_t)(t0 / kDC) * d.H * kDeltaChunk, kDeltaChunk * 4);
        fk.load(kp + t0 * d.k_stride[1], d.k_stride[1], n, Kd, tid);
        if (PASS == 0) fq.load(qp + t0 * d.q_stride[1], d.q_stride[1], n, Kd, tid);
        fm.load(r, 0, tid);
        if (PASS == 0) fp.load(r, kDeltaP, tid);
#pragma unroll
        for (int j = 0; j * NTH < 3 * kDC; j++) fv[j] = buf_load<float>(r, (kDeltaG + tid + j * NTH) * 4);
        const __amdgpu_buffer_rsrc_t rv = rows_window(vp + t0 * d.v_stride[1], d.v_stride[1], n, V);
#pragma unroll
        for (int i = 0; i < 8; i++) vv[i] = buf_load_bits<T>(rv, v_off + i * v_step);
    };
    auto store = [&](int b) {
        fk.store(Rows{sk[b]}, tid);
        fm.store(Mat{sm[b]}, tid);
        if (PASS == 0) {
            fq.store(Rows{sq[b]}, tid);
            fp.store(Mat{sp[b]}, tid);
        }
#pragma unroll
        for (int j = 0; j * NTH < 3 * kDC; j++)
            if (tid + j * NTH < 3 * kDC) sv[b][tid + j * NTH] = fv[j];
    };
    if (begin < stop) {
        fetch(begin);
        store(0);
    }
    barrier_lds();
    for (int t0 = begin, b = 0; t0 < stop; t0 += kDC, b ^= 1) {
        const int n = s.len - t0 < kDC ? s.len - t0 : kDC;
        const Rows K{sk[b]}, Q{sq[b]};
        float vc[8];
#pragma unroll
        for (int i = 0; i < 8; i++) vc[i] = float_of_bits<T>(vv[i]);
        const bool more = t0 + kDC < stop;
        if (more) fetch(t0 + kDC);
        if (PASS == 0 && d.states && t0 % (kDC * NS) == 0) {       // S (KP, VP) before the group, for the backward
            const __amdgpu_buffer_rsrc_t st =
                make_rsrc(delta_state(a, s.group + t0 / (kDC * NS), h), (uint32_t)(a.VP * KP * 4));
            const int at = v < a.VP ? (g8 * a.VP + v) * 4 : kNowhere;
#pragma unroll
            for (int kt = 0; kt < NK; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(S[kt][r]), st, at,
                                                          ((kt >> 1) * 32 + 4 * (kt & 1) + r) * a.VP * 4, 0);
        }
        f32x4 ks[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}}, o[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int p = 0; p < KP / 32; p++) {
            float x[8];
#pragma unroll
            for (int r = 0; r < 4; r++) x[r] = S[2 * p][r], x[4 + r] = S[2 * p + 1][r];
            const Frag<3> f = split8<3>(x);
            const Frag<P> kf[2] = {K.frag(pair_row(0, l16), 32 * p, lane), K.frag(pair_row(1, l16), 32 * p, lane)},
                          qf[2] = {Q.frag(pair_row(0, l16), 32 * p, lane), Q.frag(pair_row(1, l16), 32 * p, lane)};
            mma_n<3>(kf, f, ks);
            if (PASS == 0) mma_n<3>(qf, f, o);
        }
        float G[8], L[8], be[8], x[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const f32x4 t0v = *reinterpret_cast<const f32x4*>(&sv[b][g8 + i]),
                        t1v = *reinterpret_cast<const f32x4*>(&sv[b][kDC + g8 + i]),
                        t2v = *reinterpret_cast<const f32x4*>(&sv[b][2 * kDC + g8 + i]);
#pragma unroll
            for (int r = 0; r < 4; r++) G[i + r] = t0v[r], L[i + r] = t1v[r], be[i + r] = t2v[r];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = vc[i] - G[i] * ks[i >> 2][i & 3];
            o[i >> 2][i & 3] *= (float)d.scale * G[i];
        }
        const Frag<3> X = split8<3>(x);
        const Mat M{sm[b]};
        const Frag<3> mf[2] = {M.frag(pair_row(0, l16), 0, lane), M.frag(pair_row(1, l16), 0, lane)};
        f32x4 e[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        mma_n<3>(mf, X, e);
#pragma unroll
        for (int m = 0; m < 2; m++) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[4 * m + r] = e[m][r] * be[4 * m + r];
                y[4 * m + r] = x[4 * m + r] * L[4 * m + r];
            }
        }
        if (PASS == 0 && d.states) {
            const __amdgpu_buffer_rsrc_t re =
                make_rsrc(delta_errors(a, s.group + t0 / (kDC * NS), h), (uint32_t)(a.VP * kDC * NS * 4));
#pragma unroll
            for (int m = 0; m < 2; m++)
                buf_store4(re, (v * kDC * NS + t0 % (kDC * NS) + g8 + 4 * m) * 4, e[m]);
        }
        const Frag<3> U = split8<3>(x);
        const Frag<3> LU = split8<3>(y);
        const float decay = sv[b][kDC - 1];
#pragma unroll
        for (int k4 = 0; k4 < NK; k4 += 4) {
            Frag<P> kf[4];
            f32x4 t[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                kf[i] = K.tfrag(0, ((k4 + i) >> 1) * 32 + 8 * (lane & 3) + 4 * (i & 1), lane);
                t[i] = S[k4 + i] * decay;
            }
            mma_n<3>(kf, LU, t);
#pragma unroll
            for (int i = 0; i < 4; i++) S[k4 + i] = t[i];
        }
        if constexpr (PASS == 0) {
        const __amdgpu_buffer_rsrc_t ro =
            rows_window(out + ((s.row + t0) * d.H + h) * (int64_t)V, d.H * (int64_t)V, n, V);
#pragma unroll
        for (int m = 0; m < 2; m++) {
            o[m] = mma<3>(Mat{sp[b]}.frag(pair_row(m, l16), 0, lane), U, o[m]);
#pragma unroll
            for (int r = 0; r < 4; r++) buf_store<T>(ro, o_off + (4 * m + r) * o_step, (T)o[m][r]);
        }
        }
        if (more) store(b ^ 1);
        barrier_lds();
    }
    if (PASS == 1 && v < a.VP + KP)
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int k = (kt >> 1) * 32 + g8 + 4 * (kt & 1) + r;
                part[k * (a.VP + KP) + v] = S[kt][r];
            }
    if (PASS == 0 && last && send && v < V)
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int k = (kt >> 1) * 32 + g8 + 4 * (kt & 1) + r;
                if (k < Kd) send[sbase + (int64_t)k * V + v] = S[kt][r];
            }
}

// Joins the parts of a sequence: S after a part is A S + B. A block owns 16 columns of S, a
// wave of it 32 rows: its rows of A come from memory, a part ahead, and the waves hand each
// other their rows of S through LDS. Part 0 began with the sequence's own state, so its B
// is the state after it. Sequential over parts: 20 us for 16 heads of 128 in 8 parts, 82
// with one wave per 16 columns.
template <int KP> __global__ __launch_bounds__(2 * KP) void k_delta_join(DeltaP a) {
    constexpr int NP = KP / 32;
    __shared__ alignas(16) bf16x8 sf[2][NP][3][64];
    const SnHipDelta& d = a.d;
    const int h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, g8 = (lane >> 4) * 8,
              v = blockIdx.x * 16 + l16, ld = a.VP + KP, row0 = 32 * wave;
    const DeltaSeq s = delta_seq(d, blockIdx.z);
    const int64_t step = d.H * delta_seg_floats(KP, a.VP);
    float* part = a.seg_state + (blockIdx.z * (int64_t)a.segs * d.H + h) * delta_seg_floats(KP, a.VP);
    Vec8<float> na[2][NP] = {};
    float nb[8];
    auto fetch = [&](const float* from, bool with_a) {
#pragma unroll
        for (int i = 0; i < 8; i++) nb[i] = from[(row0 + g8 + i) * ld + v];
        if (with_a)
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
                for (int p = 0; p < NP; p++)
                    na[m][p] = load_floats8(from + (row0 + pair_row(m, l16)) * ld + a.VP + 32 * p + g8);
    };
    fetch(part, false);
    for (int seg = 0; seg + 1 < a.segs && (seg + 1) * a.seg_chunks * kDC < s.len; seg++, part += step) {
        f32x4 t[2] = {{nb[0], nb[1], nb[2], nb[3]}, {nb[4], nb[5], nb[6], nb[7]}};
        Frag<3> fa[2][NP];
#pragma unroll
        for (int m = 0; m < 2; m++)
#pragma unroll
            for (int p = 0; p < NP; p++) fa[m][p] = split_raw8<float>(na[m][p]);
        const bool more = seg + 2 < a.segs && (seg + 2) * a.seg_chunks * kDC < s.len;
        if (more) fetch(part + step, true);
        if (seg)
#pragma unroll
            for (int p = 0; p < NP; p++) {
                Frag<3> f;
#pragma unroll
                for (int i = 0; i < 3; i++) f.p[i] = sf[seg & 1][p][i][lane];
#pragma unroll
                for (int m = 0; m < 2; m++) t[m] = mma<3>(fa[m][p], f, t[m]);
            }
        float* next = part + step + (int64_t)KP * ld;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = t[i >> 2][i & 3];
            next[(row0 + g8 + i) * a.VP + v] = x[i];
        }
        const Frag<3> f = split8<3>(x);
#pragma unroll
        for (int i = 0; i < 3; i++) sf[(seg + 1) & 1][wave][i][lane] = f.p[i];
        barrier_lds();
    }
}

// Token by token. A wave owns 32 columns of V of one sequence and head: lane (kg, vg)
// holds rows kg RPT .. + RPT - 1 and four columns, all in registers from one read of the
// state to one write. q.S' = a q.S + (q.k) u, so one pass over the state gives both
// read-outs. Bound by the state's bytes; for one sequence by the latency of its reads, so
// all of them are on their way before the first is used: 22 us (6.1 TB/s) for 64 sequences
// of 16 heads of 128, 4 us for one of 12 heads of 64. FOUR: V is a multiple of four.
template <typename T, int RPT, bool VEC, bool FOUR>
__global__ __launch_bounds__(64) void k_delta_step(DeltaP a, T* out, const float* s0, float* send) {
    const SnHipDelta& d = a.d;
    const int h = blockIdx.y, lane = threadIdx.x, kg = lane >> 3, k0 = kg * RPT, E = (int)sizeof(T);
    const int V = (int)d.V, Kd = (int)d.K, v0 = blockIdx.x * 32 + (lane & 7) * 4;
    const DeltaSeq s = delta_seq(d, blockIdx.z);
    const int64_t sbase = ((int64_t)blockIdx.z * d.H + h) * d.K * d.V;
    Vec8<T> nq[RPT / 8], nk[RPT / 8];
    unsigned nv[4];
    float ng, nb;
    auto fetch = [&](int t) {
        const __amdgpu_buffer_rsrc_t rq = rows_window(delta_at<T>(d.q, d.q_stride, s.b, s.t0 + t, h / a.rep), 0, 1, Kd),
                                     rk = rows_window(delta_at<T>(d.k, d.k_stride, s.b, s.t0 + t, h / a.rep), 0, 1, Kd),
                                     rv = rows_window(delta_at<T>(d.v, d.v_stride, s.b, s.t0 + t, h), 0, 1, V);
        const int64_t row = (s.row + t) * d.H + h;
        ng = d.g[row];
        nb = d.beta[row];
#pragma unroll
        for (int i = 0; i < RPT / 8; i++) {
            nq[i] = buf_load8<T>(rq, (k0 + 8 * i) * E, Kd - k0 - 8 * i, VEC);
            nk[i] = buf_load8<T>(rk, (k0 + 8 * i) * E, Kd - k0 - 8 * i, VEC);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) nv[j] = buf_load_bits<T>(rv, (v0 + j) * E);
    };
    if (s.len > 0) fetch(0);
    // rows from K on lie past the state's bytes, and read as 0; so does a state that is not there
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(s0 ? s0 + sbase : nullptr, s0 ? (uint32_t)(Kd * V * 4) : 0u);
    auto place = [&](int i, int j) { return v0 + j < V ? ((k0 + i) * V + v0 + j) * 4 : kNowhere; };
    f32x4 S[RPT];
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        if constexpr (FOUR) {
            S[i] = buf_load4(rs, place(i, 0));
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) S[i][j] = buf_load<float>(rs, place(i, j));
        }
    }
    for (int t = 0; t < s.len; t++) {
        float q[RPT], k[RPT], vv[4];
#pragma unroll
        for (int i = 0; i < RPT; i++) q[i] = (float)nq[i / 8][i % 8], k[i] = (float)nk[i / 8][i % 8];
#pragma unroll
        for (int j = 0; j < 4; j++) vv[j] = float_of_bits<T>(nv[j]);
        const float al = expf(ng), be = nb;
        if (t + 1 < s.len) fetch(t + 1);
        f32x4 sk = {0, 0, 0, 0}, sq = {0, 0, 0, 0};
        float qk = 0.f;
#pragma unroll
        for (int i = 0; i < RPT; i++) {
            qk = fmaf(q[i], k[i], qk);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                sk[j] = fmaf(S[i][j], k[i], sk[j]);
                sq[j] = fmaf(S[i][j], q[i], sq[j]);
            }
        }
#pragma unroll
        for (int o = 8; o < 64; o <<= 1) {
            qk += __shfl_xor(qk, o);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                sk[j] += __shfl_xor(sk[j], o);
                sq[j] += __shfl_xor(sq[j], o);
            }
        }
        f32x4 u;
        const __amdgpu_buffer_rsrc_t ro = rows_window(out + ((s.row + t) * d.H + h) * (int64_t)V, 0, 1, V);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            u[j] = be * (vv[j] - al * sk[j]);
            buf_store<T>(ro, kg == 0 ? (v0 + j) * E : kNowhere, (T)((float)d.scale * (al * sq[j] + qk * u[j])));
        }
#pragma unroll
        for (int i = 0; i < RPT; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) S[i][j] = fmaf(k[i], u[j], al * S[i][j]);
    }
    if (!send) return;
    const __amdgpu_buffer_rsrc_t rt = make_rsrc(send + sbase, (uint32_t)(Kd * V * 4));
#pragma unroll
    for (int i = 0; i < RPT; i++) {
        if constexpr (FOUR) {
            buf_store4(rt, place(i, 0), S[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) buf_store<float>(rt, place(i, j), S[i][j]);
        }
    }
}

template <typename T, int KP, bool VEC>
snhip_status step_t(const DeltaP& a, void* out, float* send, hipStream_t st) {
    const dim3 grid((unsigned)((a.d.V + 31) / 32), (unsigned)a.d.H, (unsigned)a.d.N);
    if (a.d.V % 4 == 0) k_delta_step<T, KP / 8, VEC, true><<<grid, 64, 0, st>>>(a, (T*)out, a.d.s0, send);
    else k_delta_step<T, KP / 8, VEC, false><<<grid, 64, 0, st>>>(a, (T*)out, a.d.s0, send);
    SNHIP_CHECK(hipGetLastError());
    return SNHIP_OK;
}

template <typename T, int KP, bool VEC>
snhip_status fwd_t(const DeltaP& a, void* out, float* send, hipStream_t st) {
    k_delta_prep<T, KP, VEC><<<dim3((unsigned)a.slots, (unsigned)a.d.H), 256, 0, st>>>(a);
    SNHIP_CHECK(hipGetLastError());
    const unsigned H = (unsigned)a.d.H, N = (unsigned)a.d.N, per = 16 * kDeltaW;
    if (a.segs > 1) {
        k_delta_scan<T, KP, VEC, 1><<<dim3((a.VP + KP + per - 1) / per, H, N * a.segs), 64 * kDeltaW, 0, st>>>(a, nullptr, nullptr);
        SNHIP_CHECK(hipGetLastError());
        k_delta_join<KP><<<dim3(a.VP / 16, H, N), 2 * KP, 0, st>>>(a);
        SNHIP_CHECK(hipGetLastError());
    }
    k_delta_scan<T, KP, VEC, 0><<<dim3((a.VP + per - 1) / per, H, N * a.segs), 64 * kDeltaW, 0, st>>>(a, (T*)out, send);
    SNHIP_CHECK(hipGetLastError());
    return SNHIP_OK;
}

}  // namespace

// Checks d and fills in what the kernels derive from it.
snhip_status delta_args(const SnHipDelta* d, DeltaP* a) {
    if (!d || !d->q || !d->k || !d->v || !d->g || !d->beta) return SNHIP_E_INVAL;
    if (!delta_in_range(*d)) return SNHIP_E_INVAL;
    for (const void* w : {(const void*)d->chunks, (const void*)d->states})
        if (reinterpret_cast<uintptr_t>(w) % 16) return SNHIP_E_INVAL;
    for (const int64_t* st : {d->q_stride, d->k_stride, d->v_stride})
        if (st[1] < 0 || st[1] >= kDeltaStride) return SNHIP_E_INVAL;
    a->d = *d;
    a->slots = delta_slots(*d);
    a->groups = delta_groups(*d);
    a->segs = delta_segs(*d);
    a->seg_chunks = (int)(((d->T + kDC - 1) / kDC + a->segs - 1) / a->segs);
    if (d->dtype != SNHIP_F32) a->seg_chunks += a->seg_chunks & 1;      // whole groups of the backward
    a->seg_state = d->chunks + delta_slots(*d) * d->H * kDeltaChunk;
    a->KP = delta_kp(d->K);
    a->VP = delta_vp(d->V);
    a->rep = (int)(d->H / d->Hk);
    const int64_t step = d->dtype == SNHIP_F32 ? 4 : 8;       // elements of 16 bytes
    auto vec = [&](const void* p, const int64_t* s) {
        return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s[0] % step == 0 && s[1] % step == 0 && s[2] % step == 0;
    };
    a->vec = d->K % 8 == 0 && vec(d->q, d->q_stride) && vec(d->k, d->k_stride);
    return SNHIP_OK;
}

}  // namespace snhip

using namespace snhip;

extern "C" {

int64_t snhip_op_delta_chunk_floats(const SnHipDelta* d) {
    if (!d || !delta_in_range(*d) || delta_slots(*d) > kDeltaSlots) return 0;
    const int64_t segs = delta_segs(*d);
    return delta_slots(*d) * d->H * kDeltaChunk +
           (segs > 1 ? d->N * segs * d->H * delta_seg_floats(delta_kp(d->K), delta_vp(d->V)) : 0);
}
int64_t snhip_op_delta_state_floats(const SnHipDelta* d) {
    if (!d || !delta_in_range(*d) || delta_slots(*d) > kDeltaSlots) return 0;
    return delta_groups(*d) * d->H * delta_vp(d->V) * (kDC * delta_ns(d->dtype, d->K) + (int64_t)delta_kp(d->K));
}

snhip_status snhip_op_delta_step_dev(const SnHipDelta* d, void* out, float* send, void* stream) {
    DeltaP a;
    const snhip_status rc = delta_args(d, &a);
    if (rc != SNHIP_OK || !out || !send) return SNHIP_E_INVAL;
    return delta_pick(a, [&](auto t, auto kp, auto vec) {
        return step_t<decltype(t), decltype(kp)::value, decltype(vec)::value>(a, out, send, as_stream(stream));
    });
}

snhip_status snhip_op_delta_fwd_dev(const SnHipDelta* d, void* out, float* send, void* stream) {
    DeltaP a;
    const snhip_status rc = delta_args(d, &a);
    if (rc != SNHIP_OK || !out) return SNHIP_E_INVAL;
    const hipStream_t st = as_stream(stream);
    if (!d->chunks) {
        if (d->cu || d->states || d->T > kDeltaStepTokens) return SNHIP_E_INVAL;
        return delta_pick(a, [&](auto t, auto kp, auto vec) {
            return step_t<decltype(t), decltype(kp)::value, decltype(vec)::value>(a, out, send, st);
        });
    }
    if (a.slots > kDeltaSlots) return SNHIP_E_INVAL;
    return delta_pick(a, [&](auto t, auto kp, auto vec) {
        return fwd_t<decltype(t), decltype(kp)::value, decltype(vec)::value>(a, out, send, st);
    });
}

}  // extern "C"
