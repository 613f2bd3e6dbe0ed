// Gated delta rule, backward. With dS the gradient of the state after a chunk
// (names of delta.h):
//   dU = P^T dO + L (K dS)       W = M^T (beta dU) = dV
//   dS before = G_C dS + scale Q^T (G dO) - K^T (G W)
// is sequential over chunks, from the last to the first, and independent over the
// columns of V (k_delta_rscan); it leaves W, each chunk's dS, and its columns' part of
// E_i.dU_i. The rest is a sum over V per chunk (k_delta_local):
//   Y_ij = scale D_ij beta_j dO_i.E_j (j <= i)   Z_ij = W_i.E_j, F_ij = -D_ij beta_j Z_ij (j < i)
//   dQ = scale G (dO S^T) + Y K
//   dK = L beta (E dS^T) - G (W S^T) + Y^T Q + (F + F^T) K
//   dbeta_j = E_j.dU_j - sum over i > j in j's chunk of Z_ij D_ij k_i.k_j
// and, with H = Y (q.k) + F (k.k) elementwise below the diagonal (on it a decay of 1
// has no gradient: its two shares are left out, not cancelled),
//   dg_t = sum over i >= t of [ sum_j H_ij - sum_j H_ji
//                               + scale G q_i.(dO S^T)_i - G k_i.(W S^T)_i ]
//          + sum over i < t of L beta k_i.(E dS^T)_i + G_C <S, dS>.
#include "delta.h"

namespace snhip {

snhip_status delta_args(const SnHipDelta* d, DeltaP* a);

namespace {

// Per group of NS chunks and head: W^T (VP, 32 NS), dS (KP, VP) after the group, and
// (VP / 16, 32 NS) sums of E dU over 16 columns.
struct DeltaWs {
    float* w;
    float* ds;
    float* eu;
};
__host__ __device__ inline DeltaWs delta_ws(const DeltaP& a, float* ws, int64_t group, int h) {
    const int64_t i = group * a.d.H + h, n = a.groups * a.d.H, c = kDC * delta_ns(a.d.dtype, a.d.K), w = c * a.VP,
                  ds = (int64_t)a.VP * a.KP;
    return {ws + i * w, ws + n * w + i * ds, ws + n * (w + ds) + i * (a.VP / 16 * c)};
}

// The scan from the last chunk to the first, laid out as the forward's: a wave owns 16
// columns of V and holds its (K, 16) of dS in registers, the chunk before is fetched while
// one is worked on. Bound by the chain of a chunk's products and by what it leaves in
// memory: 298 us for 8 x 2048 tokens, 16 heads of 128 in bf16.
template <typename T, int KP, bool VEC>
__global__ __launch_bounds__(64 * kDeltaW) void k_delta_rscan(DeltaP a, SnHipDeltaGrad gr) {
    constexpr int P = ElemPlanes<T>::n, NK = KP / 16, W = kDeltaW, NTH = 64 * W, NS = sizeof(T) == 4 || KP == 64 ? 1 : 2, C = kDC * NS;
    typedef Tile<P, kDC, KP> Rows;
    typedef Tile<3, kDC, kDC> Mat;
    __shared__ alignas(16) __bf16 sk[2][Rows::elems], sq[2][Rows::elems], sm[2][Mat::elems], sp[2][Mat::elems];
    __shared__ alignas(16) float sv[2][3 * kDC];
    const SnHipDelta& d = a.d;
    const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g8 = (lane >> 4) * 8;
    const DeltaSeq s = delta_seq(d, blockIdx.z);
    const int v = (blockIdx.x * W + wave) * 16 + l16, V = (int)d.V, Kd = (int)d.K;
    const int64_t sbase = ((int64_t)blockIdx.z * d.H + h) * d.K * d.V;
    const T* kp = delta_at<T>(d.k, d.k_stride, s.b, s.t0, h / a.rep);
    const T* qp = delta_at<T>(d.q, d.q_stride, s.b, s.t0, h / a.rep);
    const T* dop = static_cast<const T*>(gr.dout) + (s.row * d.H + h) * (int64_t)V;
    const float* rec = d.chunks + (s.slot * d.H + h) * kDeltaChunk;

    f32x4 S[NK];           // dS, rows as k_delta_scan holds S
#pragma unroll
    for (int kt = 0; kt < NK; kt++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int k = (kt >> 1) * 32 + g8 + 4 * (kt & 1) + r;
            S[kt][r] = gr.dsend && k < Kd && v < V ? gr.dsend[sbase + (int64_t)k * V + v] : 0.f;
        }
    RowsFetch<T, KP, NTH, VEC> fk, fq;
    MatFetch<NTH> fm, fp;
    float fv[(3 * kDC + NTH - 1) / NTH];
    unsigned vv[8];
    f32x4 ev[2];
    fk.init(d.k_stride[1], Kd, tid);
    fq.init(d.q_stride[1], Kd, tid);
    const int E = (int)sizeof(T), o_step = (int)d.H * V * E, o_off = v < V ? g8 * o_step + v * E : kNowhere;
    auto fetch = [&](int t0) {
        const int n = s.len - t0 < kDC ? s.len - t0 : kDC;
        const __amdgpu_buffer_rsrc_t r = make_rsrc(rec + (int64_t)(t0 / kDC) * d.H * kDeltaChunk, kDeltaChunk * 4);
        fk.load(kp + t0 * d.k_stride[1], d.k_stride[1], n, Kd, tid);
        fq.load(qp + t0 * d.q_stride[1], d.q_stride[1], n, Kd, tid);
        fm.load(r, 0, tid);
        fp.load(r, kDeltaP, tid);
#pragma unroll
        for (int j = 0; j * NTH < 3 * kDC; j++) fv[j] = buf_load<float>(r, (kDeltaG + tid + j * NTH) * 4);
        const __amdgpu_buffer_rsrc_t ro = rows_window(dop + t0 * d.H * V, d.H * V, n, V);
#pragma unroll
        for (int i = 0; i < 8; i++) vv[i] = buf_load_bits<T>(ro, o_off + i * o_step);
        const __amdgpu_buffer_rsrc_t re = make_rsrc(delta_errors(a, s.group + t0 / C, h), (uint32_t)(a.VP * C * 4));
#pragma unroll
        for (int m = 0; m < 2; m++) ev[m] = buf_load4(re, (v * C + t0 % C + g8 + 4 * m) * 4);
    };
    auto store = [&](int b) {
        fk.store(Rows{sk[b]}, tid);
        fq.store(Rows{sq[b]}, tid);
        fm.store(Mat{sm[b]}, tid);
        fp.store(Mat{sp[b]}, tid);
#pragma unroll
        for (int j = 0; j * NTH < 3 * kDC; j++)
            if (tid + j * NTH < 3 * kDC) sv[b][tid + j * NTH] = fv[j];
    };
    const int last = s.len > 0 ? (s.len - 1) / kDC * kDC : -1;
    if (last >= 0) {
        fetch(last);
        store(0);
    }
    barrier_lds();
    for (int t0 = last, b = 0; t0 >= 0; t0 -= kDC, b ^= 1) {
        const Rows K{sk[b]}, Q{sq[b]};
        const Mat M{sm[b]}, PM{sp[b]};
        const DeltaWs w = delta_ws(a, gr.ws, s.group + t0 / C, h);
        const int n = s.len - t0 < kDC ? s.len - t0 : kDC;
        float G[8], L[8], be[8], x[8], y[8], od[8];
        const f32x4 e[2] = {ev[0], ev[1]};
#pragma unroll
        for (int i = 0; i < 8; i++) od[i] = float_of_bits<T>(vv[i]);
        if (t0 > 0) fetch(t0 - kDC);
        const __amdgpu_buffer_rsrc_t rds = make_rsrc(w.ds, (uint32_t)(a.VP * KP * 4)),
                                     rw = make_rsrc(w.w, (uint32_t)(a.VP * C * 4)),
                                     reu = make_rsrc(w.eu, (uint32_t)(a.VP / 16 * C * 4));
        const int at = v < a.VP ? (g8 * a.VP + v) * 4 : kNowhere;
        if (NS == 1 || t0 % C || t0 == last)       // the group's last chunk
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(S[kt][r]), rds, at,
                                                      ((kt >> 1) * 32 + 4 * (kt & 1) + r) * a.VP * 4, 0);
        f32x4 du[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int p = 0; p < KP / 32; p++) {
#pragma unroll
            for (int r = 0; r < 4; r++) x[r] = S[2 * p][r], x[4 + r] = S[2 * p + 1][r];
            const Frag<3> f = split8<3>(x);
            const Frag<P> kf[2] = {K.frag(pair_row(0, l16), 32 * p, lane), K.frag(pair_row(1, l16), 32 * p, lane)};
            mma_n<3>(kf, f, du);
        }
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            const f32x4 t0v = *reinterpret_cast<const f32x4*>(&sv[b][g8 + i]),
                        t1v = *reinterpret_cast<const f32x4*>(&sv[b][kDC + g8 + i]),
                        t2v = *reinterpret_cast<const f32x4*>(&sv[b][2 * kDC + g8 + i]);
#pragma unroll
            for (int r = 0; r < 4; r++) G[i + r] = t0v[r], L[i + r] = t1v[r], be[i + r] = t2v[r];
        }
        const Frag<P> dO = split8<P>(od);
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = od[i] * ((float)d.scale * G[i]);
        const Frag<3> GdO = split8<3>(y);
#pragma unroll
        for (int i = 0; i < 8; i++) du[i >> 2][i & 3] *= L[i];
        const Frag<3> pf[2] = {PM.tfrag(0, 8 * (lane & 3), lane), PM.tfrag(0, 8 * (lane & 3) + 4, lane)};
        mma_n<3>(pf, dO, du);
#pragma unroll
        for (int m = 0; m < 2; m++) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                x[4 * m + r] = du[m][r] * be[4 * m + r];
                const float eu = sum16(e[m][r] * du[m][r]);
                buf_store<float>(reu, l16 == 0 ? ((v >> 4) * C + t0 % C + g8 + 4 * m + r) * 4 : kNowhere, eu);
            }
        }
        const Frag<3> dE = split8<3>(x);
        const __amdgpu_buffer_rsrc_t rdv =
            rows_window(static_cast<T*>(gr.dv) + ((s.row + t0) * d.H + h) * (int64_t)V, d.H * (int64_t)V, n, V);
        const Frag<3> mf[2] = {M.tfrag(0, 8 * (lane & 3), lane), M.tfrag(0, 8 * (lane & 3) + 4, lane)};
        f32x4 wm[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        mma_n<3>(mf, dE, wm);
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const f32x4 wv = wm[m];
            buf_store4(rw, (v * C + t0 % C + g8 + 4 * m) * 4, wv);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                buf_store<T>(rdv, o_off + (4 * m + r) * o_step, (T)wv[r]);
                y[4 * m + r] = -wv[r] * G[4 * m + r];
            }
        }
        const Frag<3> GW = split8<3>(y);
        const float decay = sv[b][kDC - 1];
#pragma unroll
        for (int k4 = 0; k4 < NK; k4 += 4) {
            Frag<P> kf[4], qf[4];
            f32x4 t[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int block = ((k4 + i) >> 1) * 32 + 8 * (lane & 3) + 4 * (i & 1);
                qf[i] = Q.tfrag(0, block, lane);
                kf[i] = K.tfrag(0, block, lane);
                t[i] = S[k4 + i] * decay;
            }
            mma_n<3>(qf, GdO, t);
            mma_n<3>(kf, GW, t);
#pragma unroll
            for (int i = 0; i < 4; i++) S[k4 + i] = t[i];
        }
        if (t0 > 0) store(b ^ 1);
        barrier_lds();
    }
    if (gr.ds0 && v < V)
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int k = (kt >> 1) * 32 + g8 + 4 * (kt & 1) + r;
                if (k < Kd) gr.ds0[sbase + (int64_t)k * V + v] = S[kt][r];
            }
}

// The row of tile i of a lower triangle, counted by rows: 0; 1, 1; 2, 2, 2; ...
__device__ __forceinline__ int delta_tile_row(int i) { return i < 1 ? 0 : i < 3 ? 1 : i < 6 ? 2 : 3; }

// The lane's place in a phase of a loop, as a value of that phase: the addresses that it
// makes are not carried around the loop in registers.
struct LanePlace {
    int lane, l16, g4, g8, blk16, blkp;
    __device__ __forceinline__ explicit LanePlace(int l) {
        asm volatile("" : "+v"(l));
        lane = l & 63;
        l16 = lane & 15;
        g4 = lane >> 4 << 2;
        g8 = 2 * g4;
        blk16 = 4 * (lane & 3);
        blkp = 8 * (lane & 3);
    }
};

__device__ __forceinline__ float sum_groups(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// One group of NS chunks (C = 32 NS tokens, taken as one chunk) of one query and key head:
// a block of KP / 16 waves runs over the value heads that share it, so dq and dk are summed
// in registers. Per head and 64 columns of V, E, W and dO go through LDS (E and W by
// column, as the scans leave them, read transposed), and a wave owns 16 columns of K in the
// products with S and dS; Y and F are made by tiles of 16x16, a wave taking every
// (KP / 16)-th. What the next step reads is fetched into registers a step ahead. Bound by
// the bytes of S and dS, and by the latency of its steps (one block of eight waves on a CU
// waits in 60 % of its cycles; in 16 bits with K > 64 it has all 256 registers and spills 7):
// 510 us for 8 x 2048 tokens, 16 heads of 128 in bf16.
template <typename T, int KP, bool VEC>
__global__ __launch_bounds__(4 * KP, 2) void k_delta_local(DeltaP a, SnHipDeltaGrad gr, bool vec_o) {
    constexpr int NS = sizeof(T) == 4 || KP == 64 ? 1 : 2, C = kDC * NS, NM = 2 * NS;      // NM tiles of 16 tokens
    constexpr int P = ElemPlanes<T>::n, VT = 64, NW = KP / 16, NTH = 64 * NW;
    constexpr int TILES = NM * (NM + 1) / 2, NT = (2 * TILES + NW - 1) / NW;   // of Y, then of F; per wave
    typedef Tile<P, C, KP> Rows;
    // C = 32: rows of 64 bytes; C = 64: of 192, where LDS holds that beside the 16-bit tiles
    typedef Tile<3, VT, C, NS == 1 ? 0 : P == 1 ? 32 : 8> Cols;
    typedef Tile<3, C, C> Mat;
    static_assert(Cols::elems >= Mat::elems, "Y and F take the places of E and W");
    __shared__ alignas(16) __bf16 sk[Rows::elems], sq[Rows::elems], se[Cols::elems], sw[Cols::elems],
        so[Tile<P, C, VT>::elems];
    __shared__ float sG[C], sL[C], sB[C], seu[C], kread[NW][C], kwrite[NW][C], trow[2 * TILES][16], tcol[2 * TILES][16],
        tzk[TILES][16], dots[NW];
    __shared__ double sc[C];
    const SnHipDelta& d = a.d;
    const int hk = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15,
              g8 = (lane >> 4) * 8;
    DeltaSeq s;
    int group;
    if (!delta_chunk_of<C>(d, blockIdx.x, &s, &group)) return;
    const int64_t t0 = (int64_t)group * C;
    const int n = (int)(s.len - t0 < C ? s.len - t0 : C), V = (int)d.V, Kd = (int)d.K;
    const Rows K{sk}, Q{sq};
    const Cols ET{se}, WT{sw};
    const Tile<P, C, VT> DO{so};
    const Mat Y{se}, FF{sw};
    RowsFetch<T, KP, NTH, VEC, C> fk, fq;
    fk.init(d.k_stride[1], Kd, tid);
    fq.init(d.q_stride[1], Kd, tid);
    fk.load(delta_at<T>(d.k, d.k_stride, s.b, s.t0 + t0, hk), d.k_stride[1], n, Kd, tid);
    fq.load(delta_at<T>(d.q, d.q_stride, s.b, s.t0 + t0, hk), d.q_stride[1], n, Kd, tid);

    // Fetches ahead. Tiles: 64 columns of V of E^T, then of W^T (C / 8 vectors of eight tokens
    // a column; those of a chunk that the sequence does not reach were never written and
    // count as 0), and dO (eight vectors a token).
    constexpr int EV = VT * C / 8, NEW = 2 * EV / NTH, NO = (C * 8 + NTH - 1) / NTH;
    Vec8<float> pe[NEW];
    Vec8<T> po[NO];
    const int o_step = (int)d.H * V;
    auto fetch_tiles = [&](int h, int vt) {
        const uint32_t bytes = (uint32_t)(a.VP * C * 4);
        const __amdgpu_buffer_rsrc_t re = make_rsrc(delta_errors(a, blockIdx.x, h), bytes),
                                     rw = make_rsrc(delta_ws(a, gr.ws, blockIdx.x, h).w, bytes);
#pragma unroll
        for (int j = 0; j < NEW; j++) {
            const int u = tid + j * NTH, c = u % (C / 8) * 8;
            const int at = (c & ~(kDC - 1)) < n ? (vt * C + u % EV * 8) * 4 : kNowhere;
            pe[j] = buf_load8<float>(u < EV ? re : rw, at, 8, true);
        }
        const T* op = static_cast<const T*>(gr.dout) + ((s.row + t0) * d.H + h) * (int64_t)V;
        const __amdgpu_buffer_rsrc_t ro = rows_window(op, o_step, n, V);
#pragma unroll
        for (int j = 0; j < NO; j++) {
            const int u = tid + j * NTH, c = vt + (u & 7) * 8;
            po[j] = buf_load8<T>(ro, c < V && u < C * 8 ? ((u >> 3) * o_step + c) * (int)sizeof(T) : kNowhere, V - c, vec_o);
        }
    };
    // States: 32 columns of V from `v0` on of S and dS, the rows of K of this wave.
    const int kc = wave * 16;
    Vec8<float> ps, pd;
    auto fetch_states = [&](int h, int v0) {
        const int at = v0 + g8 < a.VP ? ((kc + l16) * a.VP + v0 + g8) * 4 : kNowhere;
        ps = buf_load8<float>(make_rsrc(delta_state(a, blockIdx.x, h), (uint32_t)(a.VP * KP * 4)), at, 8, true);
        pd = buf_load8<float>(make_rsrc(delta_ws(a, gr.ws, blockIdx.x, h).ds, (uint32_t)(a.VP * KP * 4)), at, 8, true);
    };
    fetch_tiles(hk * a.rep, 0);
    fetch_states(hk * a.rep, 0);
    fk.store(K, tid);
    fq.store(Q, tid);
    f32x4 dq[NM], dk[NM];
#pragma unroll
    for (int m = 0; m < NM; m++) dq[m] = dk[m] = f32x4{0, 0, 0, 0};

    for (int h = hk * a.rep, end = h + a.rep; h < end; h++) {
        if (wave == NW - 1) {        // decays, and the parts of E dU
            const int64_t at = (s.row + t0 + lane) * d.H + h;
            double c = lane < n ? (double)delta_decay(d.g[at]) : 0.0;
#pragma unroll
            for (int o = 1; o < C; o <<= 1) {
                const double y = __shfl_up(c, o, C);
                if ((lane & (C - 1)) >= o) c += y;
            }
            const double last = __shfl(c, C - 1, C);
            if (lane < C) {
                sc[lane] = c;
                sG[lane] = expf((float)c);
                sL[lane] = expf((float)(last - c));
                sB[lane] = lane < n ? d.beta[at] : 0.f;
                const float* eu = delta_ws(a, gr.ws, blockIdx.x, h).eu;
                float t = 0.f;
                if (lane < n)
                    for (int i = 0; i < a.VP / 16; i++) t += eu[i * C + lane];
                seu[lane] = t;
            }
        }
        f32x4 small[NT], q1[NM], k1[NM], k2[NM];
#pragma unroll
        for (int j = 0; j < NT; j++) small[j] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int m = 0; m < NM; m++) q1[m] = k1[m] = k2[m] = f32x4{0, 0, 0, 0};
        float ss = 0.f;
        for (int vt = 0; vt < a.VP; vt += VT) {
#pragma unroll
            for (int j = 0; j < NEW; j++) {
                const int u = tid + j * NTH, r = u % EV / (C / 8), c = u % (C / 8) * 8;
                (u < EV ? ET : WT).put8(r, c, split_raw8<float>(pe[j]));
            }
#pragma unroll
            for (int j = 0; j < NO; j++) {
                const int u = tid + j * NTH;
                if (u < C * 8) DO.put8(u >> 3, (u & 7) * 8, split_raw8<T>(po[j]));
            }
            barrier_lds();
            if (vt + VT < a.VP) fetch_tiles(h, vt + VT);
            else if (h + 1 < end) fetch_tiles(h + 1, 0);
            const int nv = a.VP - vt < VT ? (a.VP - vt + 31) & ~31 : VT;       // whole 32s
            const LanePlace L(lane);
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const int task = wave + j * NW, ti = delta_tile_row(task % TILES), tj = task % TILES - ti * (ti + 1) / 2;
                if (task < 2 * TILES)
                    for (int i = 0; i < nv; i += 32) {
                        const Frag<3> b = ET.tfrag(i, 16 * tj + L.blk16, L.lane);
                        small[j] = task < TILES ? mma<3>(DO.frag(16 * ti + L.l16, i, L.lane), b, small[j])
                                                : mma<3>(WT.tfrag(i, 16 * ti + L.blk16, L.lane), b, small[j]);
                    }
                __builtin_amdgcn_sched_barrier(0);       // reads of later tiles would need registers
            }
            for (int i = 0; i < nv; i += 32) {
#pragma unroll
                for (int l = 0; l < 8; l++) ss = fmaf(ps[l], pd[l], ss);
                const Frag<3> b = split_raw8<float>(ps), e = split_raw8<float>(pd);
                if (vt + i + 32 < a.VP) fetch_states(h, vt + i + 32);
                else if (h + 1 < end) fetch_states(h + 1, 0);
#pragma unroll
                for (int m = 0; m < NM; m++) {
                    const int r = 32 * (m >> 1), q = m & 1;
                    q1[m] = mma<3>(DO.frag(r + pair_row(q, L.l16), i, L.lane), b, q1[m]);
                    k1[m] = mma<3>(WT.tfrag(i, r + L.blkp + 4 * q, L.lane), b, k1[m]);
                    k2[m] = mma<3>(ET.tfrag(i, r + L.blkp + 4 * q, L.lane), e, k2[m]);
                    if (m & 1) __builtin_amdgcn_sched_barrier(0);
                }
            }
            barrier_lds();
        }
        ss = sum_groups(sum16(ss));
        if (lane == 0) dots[wave] = ss;
        // Y's upper tiles are 0
        for (int i = tid; i < C * C / 8; i += NTH) {
            const int row = i / (C / 8), c = i % (C / 8) * 8;
            if (c / 16 > row / 16) Y.put8(row, c, Frag<3>{});
        }
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const LanePlace L(lane);
            // a tile of Y with its part of H, or of F with its part
            const int task = wave + j * NW, tile = task % TILES, ti = delta_tile_row(tile), tj = tile - ti * (ti + 1) / 2;
            if (task >= 2 * TILES) break;
            const Rows A{task < TILES ? sq : sk};
            f32x4 qk = {0, 0, 0, 0};       // q.k, or k.k
#pragma unroll
            for (int c = 0; c < KP; c += 32)
                qk = mma<3>(A.frag(16 * ti + L.l16, c, L.lane), K.frag(16 * tj + L.l16, c, L.lane), qk);
            const int col = tj * 16 + L.l16;
            const float bj = sB[col];
            float hsum = 0.f, zsum = 0.f, f[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * ti + L.g4 + r;
                const float D = col <= row ? expf((float)(sc[row] - sc[col])) : 0.f;
                float e;
                if (task < TILES) {
                    const float y = (float)d.scale * D * bj * small[j][r];
                    e = col < row ? y * qk[r] : 0.f;
                    Y.put(row, col, y);
                } else {
                    const float zd = col < row ? D * small[j][r] : 0.f;
                    f[r] = -bj * zd;
                    e = f[r] * qk[r];
                    if (ti / 2 == tj / 2) zsum = fmaf(zd, qk[r], zsum);     // dU has the other chunks' part
                    if (ti != tj) {
                        FF.put(row, col, f[r]);
                        FF.put(col, row, f[r]);
                    }
                }
                const float er = sum16(e);
                if (L.l16 == 0) trow[task][L.g4 + r] = er;
                hsum += e;
            }
            hsum = sum_groups(hsum);
            if (L.lane < 16) tcol[task][lane] = hsum;
            if (task >= TILES) {
                zsum = sum_groups(zsum);
                if (L.lane < 16) tzk[tile][lane] = zsum;
                if (ti == tj) {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        // F_ji of this lane's (i, j): row j of column i, in lane 16 (j / 4) + i
                        float t = 0.f;
#pragma unroll
                        for (int rr = 0; rr < 4; rr++) {
                            const float x = __shfl(f[rr], (L.l16 >> 2) * 16 + L.g4 + r);
                            if ((L.l16 & 3) == rr) t = x;
                        }
                        FF.put(16 * ti + L.g4 + r, col, f[r] + t);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        barrier_lds();
        const LanePlace L(lane);
        Frag<P> bk[NS], bq[NS];
#pragma unroll
        for (int i = 0; i < NS; i++) {
            bk[i] = K.tfrag(32 * i, kc + L.blk16, L.lane);
            bq[i] = Q.tfrag(32 * i, kc + L.blk16, L.lane);
        }
#pragma unroll
        for (int m = 0; m < NM; m++) {
            const int b32 = 32 * (m >> 1), q = m & 1;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int t = b32 + L.g8 + 4 * q + r;
                const float qv = Q.get(t, kc + L.l16), kv = K.get(t, kc + L.l16), G = sG[t];
                q1[m][r] *= (float)d.scale * G;
                k1[m][r] *= -G;
                k2[m][r] *= sL[t] * sB[t];
                const float cr = sum16(fmaf(qv, q1[m][r], kv * k1[m][r])), cw = sum16(kv * k2[m][r]);
                if (L.l16 == 0) {
                    kread[wave][t] = cr;
                    kwrite[wave][t] = cw;
                }
            }
            f32x4 t = k1[m] + k2[m];
#pragma unroll
            for (int i = 0; i < NS; i++) {
                if (32 * i <= b32) q1[m] = mma<3>(Y.frag(b32 + pair_row(q, L.l16), 32 * i, L.lane), bk[i], q1[m]);
                if (32 * i >= b32) t = mma<3>(Y.tfrag(32 * i, b32 + L.blkp + 4 * q, L.lane), bq[i], t);
                t = mma<3>(FF.frag(b32 + pair_row(q, L.l16), 32 * i, L.lane), bk[i], t);
            }
            dq[m] += q1[m];
            dk[m] += t;
            __builtin_amdgcn_sched_barrier(0);
        }
        barrier_lds();
        if (tid < C) {
            // dg_t: reads and H by later tokens, less H's columns there, and the writes of
            // earlier ones (a write's share in dc_C less its own dc is left of its token)
            const int t = tid, hi = t >> 4, lo = t & 15;
            float dc = 0.f, db = seu[t], wr = 0.f, all = 0.f;
            for (int i = 0; i < NM; i++) {         // tile (hi, i) of its row, (i, hi) of its column
                if (i <= hi)
                    dc += trow[hi * (hi + 1) / 2 + i][lo] + trow[TILES + hi * (hi + 1) / 2 + i][lo];
                if (i >= hi) {
                    const int c = i * (i + 1) / 2 + hi;
                    dc -= tcol[c][lo] + tcol[TILES + c][lo];
                    db -= tzk[c][lo];
                }
            }
            for (int i = 0; i < NW; i++) {
                dc += kread[i][t];
                wr += kwrite[i][t];
                all += dots[i];
            }
#pragma unroll
            for (int o = 1; o < C; o <<= 1) {
                const float x = __shfl_down(dc, o, C), y = __shfl_up(wr, o, C);
                if (t + o < C) dc += x;
                if (t >= o) wr += y;
            }
            const float before = __shfl_up(wr, 1, C);
            dc += (t ? before : 0.f) + sG[C - 1] * all;
            if (t < n) {
                gr.dg[(s.row + t0 + t) * d.H + h] = dc;
                gr.dbeta[(s.row + t0 + t) * d.H + h] = db;
            }
        }
        barrier_lds();        // sc and the sums are the next head's
    }
    if (kc + l16 >= Kd) return;
#pragma unroll
    for (int i = 0; i < 4 * NM; i++) {
        const int t = 32 * (i >> 3) + g8 + (i & 7);
        const int64_t at = ((s.row + t0 + t) * d.Hk + hk) * (int64_t)Kd + kc + l16;
        if (t < n) {
            static_cast<T*>(gr.dq)[at] = (T)dq[i >> 2][i & 3];
            static_cast<T*>(gr.dk)[at] = (T)dk[i >> 2][i & 3];
        }
    }
}

template <typename T, int KP, bool VEC>
snhip_status bwd_t(const DeltaP& a, const SnHipDeltaGrad& gr, hipStream_t st) {
    const dim3 grid((unsigned)((a.VP / 16 + kDeltaW - 1) / kDeltaW), (unsigned)a.d.H, (unsigned)a.d.N);
    k_delta_rscan<T, KP, VEC><<<grid, 64 * kDeltaW, 0, st>>>(a, gr);
    SNHIP_CHECK(hipGetLastError());
    const bool vec_o = a.d.V % 8 == 0 && reinterpret_cast<uintptr_t>(gr.dout) % 16 == 0;
    k_delta_local<T, KP, VEC><<<dim3((unsigned)a.groups, (unsigned)a.d.Hk), 4 * KP, 0, st>>>(a, gr, vec_o);
    SNHIP_CHECK(hipGetLastError());
    return SNHIP_OK;
}

}  // namespace
}  // namespace snhip

using namespace snhip;

extern "C" {

int64_t snhip_op_delta_bwd_floats(const SnHipDelta* d) {
    if (!d || !delta_in_range(*d) || delta_slots(*d) > kDeltaSlots) return 0;
    const int64_t c = kDC * delta_ns(d->dtype, d->K);
    return delta_groups(*d) * d->H * delta_vp(d->V) * (c + delta_kp(d->K) + c / 16);
}

snhip_status snhip_op_delta_bwd_dev(const SnHipDelta* d, const SnHipDeltaGrad* gr, void* stream) {
    DeltaP a;
    const snhip_status rc = delta_args(d, &a);
    if (rc != SNHIP_OK || a.slots > kDeltaSlots || !gr || !d->chunks || !d->states || !gr->dout || !gr->dq || !gr->dk || !gr->dv ||
        !gr->dg || !gr->dbeta || !gr->ws || reinterpret_cast<uintptr_t>(gr->ws) % 16)
        return SNHIP_E_INVAL;
    const hipStream_t st = as_stream(stream);
    return delta_pick(a, [&](auto t, auto kp, auto vec) {
        return bwd_t<decltype(t), decltype(kp)::value, decltype(vec)::value>(a, *gr, st);
    });
}

}  // extern "C"
