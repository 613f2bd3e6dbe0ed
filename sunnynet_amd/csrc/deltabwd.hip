// Gated delta rule, backward. With dS the gradient of the state after a chunk
// (names of delta.h):
//   dU = P^T dO + L (K dS)       dR = M^T dU        dV = beta dR
//   dS before = G_C dS + scale Q^T (G dO) - K^T (beta G dR)
// is sequential over chunks, from the last to the first, and independent over the
// columns of V (k_delta_rscan); it leaves dR and each chunk's dS. The rest is a sum
// over V per chunk (k_delta_local), with X = V - G (K S), U = M (beta X):
//   dP = dO U^T (j <= i)         Z = dR U^T (j < i; dA = -Z)
//   dQ = scale G (dO S^T) + Y K,            Y_ij = scale D_ij dP_ij
//   dK = L (U dS^T) - beta G (dR S^T) + Y^T Q + (F + F^T) K,  F_ij = -beta_i D_ij Z_ij
//   dbeta_i = dR_i.X_i - sum_j Z_ij D_ij k_i.k_j
// and, with E = Y (q.k) + F (k.k) elementwise below the diagonal (on it a decay of 1
// has no gradient: its two shares are left out, not cancelled),
//   dg_t = sum over i >= t of [ sum_j E_ij - sum_j E_ji
//                               + scale G q_i.(dO S^T)_i - beta G k_i.(dR S^T)_i ]
//          + sum over i < t of L k_i.(U dS^T)_i + G_C <S, dS>.
#include "delta.h"

namespace snhip {

snhip_status delta_args(const SnHipDelta* d, DeltaP* a);

namespace {

// Per slot and head: dR (32, VP), then dS^T (VP, KP) after the chunk.
struct DeltaWs {
    float* dr;
    float* ds;
};
__host__ __device__ inline DeltaWs delta_ws(const DeltaP& a, float* ws, int64_t slot, int h) {
    const int64_t i = slot * a.d.H + h, nr = a.slots * a.d.H * kDC * a.VP;
    return {ws + i * kDC * a.VP, ws + nr + i * (int64_t)(a.VP * a.KP)};
}

// Rows of 16x16 results that belong to this lane's column: 16 m + 4 (lane / 16) + r.
__device__ __forceinline__ int res_row(int m, int lane, int r) { return 16 * m + (lane >> 4) * 4 + r; }

template <typename T, int KP, int W>
__global__ __launch_bounds__(64 * W) void k_delta_rscan(DeltaP a, SnHipDeltaGrad gr) {
    constexpr int P = ElemPlanes<T>::n, NK = KP / 16;
    __shared__ alignas(16) __bf16 sk[Tile<P, kDC, KP>::elems], skt[Tile<P, KP, kDC>::elems],
        sqt[Tile<P, KP, kDC>::elems], sm[Tile<3, kDC, kDC>::elems], sp[Tile<3, kDC, kDC>::elems];
    __shared__ alignas(16) float sv[3 * kDC];
    const SnHipDelta& d = a.d;
    const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g4 = (lane >> 4) * 4;
    const DeltaSeq s = delta_seq(d, blockIdx.z);
    const int v = (blockIdx.x * W + wave) * 16 + (lane & 15), V = (int)d.V, Kd = (int)d.K;
    const Tile<P, kDC, KP> K{sk}, none{nullptr};
    const Tile<P, KP, kDC> KT{skt}, QT{sqt};
    const Tile<3, kDC, kDC> MT{sm}, PT{sp};
    const int64_t sbase = ((int64_t)blockIdx.z * d.H + h) * d.K * d.V;

    f32x4 S[NK];
#pragma unroll
    for (int kt = 0; kt < NK; kt++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int k = kt * 16 + g4 + r;
            S[kt][r] = gr.dsend && k < Kd && v < V ? gr.dsend[sbase + (int64_t)k * V + v] : 0.f;
        }
    for (int c = (s.len + kDC - 1) / kDC - 1; c >= 0; c--) {
        const int t0 = c * kDC, n = s.len - t0 < kDC ? s.len - t0 : kDC;
        const float* pre = d.chunks + ((s.slot + c) * d.H + h) * kDeltaChunk;
        const DeltaWs w = delta_ws(a, gr.ws, s.slot + c, h);
        __syncthreads();
        stage_tile<T, P, KP, true, true>(delta_at<T>(d.k, d.k_stride, s.b, s.t0 + t0, h / a.rep), d.k_stride[1], n,
                                         Kd, a.vec_k, K, KT, tid, 64 * W);
        stage_tile<T, P, KP, false, true>(delta_at<T>(d.q, d.q_stride, s.b, s.t0 + t0, h / a.rep), d.q_stride[1],
                                          n, Kd, a.vec_q, none, QT, tid, 64 * W);
        stage_mat<3, true>(pre, MT, tid, 64 * W);
        stage_mat<3, true>(pre + kDeltaP, PT, tid, 64 * W);
        for (int i = tid; i < 3 * kDC; i += 64 * W) sv[i] = pre[kDeltaG + i];
        __syncthreads();
        if (v < a.VP)
#pragma unroll
            for (int kt = 0; kt < NK; kt++)
                *reinterpret_cast<f32x4*>(w.ds + (int64_t)v * KP + kt * 16 + g4) = S[kt];
        const T* dop = static_cast<const T*>(gr.dout) + ((s.row + t0) * d.H + h) * (int64_t)V + v;
        float x[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int t = res_row(i >> 2, lane, i & 3);
            x[i] = t < n && v < V ? (float)dop[(int64_t)t * d.H * V] : 0.f;
            y[i] = x[i] * ((float)d.scale * sv[t]);
        }
        const Frag<P> dO = split8<P>(x);
        const Frag<3> GdO = split8<3>(y);
        f32x4 du[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int i = 0; i < KP / 32; i++) {
#pragma unroll
            for (int r = 0; r < 4; r++) x[r] = S[2 * i][r], x[4 + r] = S[2 * i + 1][r];
            const Frag<3> b = split8<3>(x);
#pragma unroll
            for (int m = 0; m < 2; m++) du[m] = mma<3>(K.frag(16 * m, i, lane), b, du[m]);
        }
#pragma unroll
        for (int m = 0; m < 2; m++) {
#pragma unroll
            for (int r = 0; r < 4; r++) du[m][r] *= sv[kDC + res_row(m, lane, r)];
            du[m] = mma<3>(PT.frag(16 * m, 0, lane), dO, du[m]);
#pragma unroll
            for (int r = 0; r < 4; r++) x[4 * m + r] = du[m][r];
        }
        const Frag<3> dU = split8<3>(x);
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const f32x4 dr = mma<3>(MT.frag(16 * m, 0, lane), dU, f32x4{0, 0, 0, 0});
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int t = res_row(m, lane, r);
                if (v < a.VP) w.dr[(int64_t)t * a.VP + v] = dr[r];
                y[4 * m + r] = -dr[r] * sv[2 * kDC + t] * sv[t];
            }
        }
        const Frag<3> BdR = split8<3>(y);
        const float decay = sv[kDC - 1];
#pragma unroll
        for (int kt = 0; kt < NK; kt++) {
            S[kt] = mma<3>(QT.frag(16 * kt, 0, lane), GdO, S[kt] * decay);
            S[kt] = mma<3>(KT.frag(16 * kt, 0, lane), BdR, S[kt]);
        }
    }
    if (gr.ds0 && v < V)
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int k = kt * 16 + g4 + r;
                if (k < Kd) gr.ds0[sbase + (int64_t)k * V + v] = S[kt][r];
            }
}

// Sum over the 16 lanes that hold one result row, or over the four lane groups.
__device__ __forceinline__ float sum16(float x) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) x += __shfl_xor(x, o);
    return x;
}
__device__ __forceinline__ float sum_groups(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// One chunk of one query and key head: a block of eight waves runs over the value
// heads that share it, so dq and dk are summed in registers. Per head and 128 columns
// of V a wave first owns 16 columns (X, U, dV), then 16 columns of K (the products
// with S and dS); the 32x32 matrices are made by three waves, a tile of 16x16 each.
template <typename T, int KP>
__global__ __launch_bounds__(512) void k_delta_local(DeltaP a, SnHipDeltaGrad gr) {
    constexpr int P = ElemPlanes<T>::n, VT = 128;
    constexpr int KT1 = Tile<P, KP, kDC>::elems, V3 = Tile<3, kDC, VT>::elems, X1 = Tile<3, kDC, kDC>::elems;
    constexpr int VPH = 2 * V3 + Tile<P, kDC, VT>::elems;       // U, dR, dO, then K^T and Q^T
    constexpr int OV = VPH > 2 * KT1 ? VPH : 2 * KT1;
    __shared__ alignas(16) __bf16 sk[Tile<P, kDC, KP>::elems], sq[Tile<P, kDC, KP>::elems], sov[OV], sx[3 * X1];
    __shared__ alignas(16) float sv[3 * kDC];
    __shared__ float red[8][kDC], kread[8][kDC], kwrite[8][kDC], trow[3][16], tzk[3][16], tcol[3][16], dots[8];
    __shared__ double sc[kDC];
    const SnHipDelta& d = a.d;
    const int hk = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g4 = (lane >> 4) * 4, l16 = lane & 15;
    DeltaSeq s;
    int chunk;
    if (!delta_chunk_of(d, blockIdx.x, &s, &chunk)) return;
    const int64_t t0 = (int64_t)chunk * kDC;
    const int n = (int)(s.len - t0 < kDC ? s.len - t0 : kDC), V = (int)d.V, Kd = (int)d.K;
    const Tile<P, kDC, KP> K{sk}, Q{sq}, none{nullptr};
    const Tile<P, KP, kDC> KT{sov}, QT{sov + KT1}, nonet{nullptr};
    const Tile<3, kDC, VT> U{sov}, DR{sov + V3};
    const Tile<P, kDC, VT> DO{sov + 2 * V3};
    const Tile<3, kDC, kDC> M{sx}, Y{sx}, YT{sx + X1}, FF{sx + 2 * X1};
    const T* kp = delta_at<T>(d.k, d.k_stride, s.b, s.t0 + t0, hk);
    const T* qp = delta_at<T>(d.q, d.q_stride, s.b, s.t0 + t0, hk);
    stage_tile<T, P, KP, true, false>(kp, d.k_stride[1], n, Kd, a.vec_k, K, nonet, tid, 512);
    stage_tile<T, P, KP, true, false>(qp, d.q_stride[1], n, Kd, a.vec_q, Q, nonet, tid, 512);
    const int k0 = wave * 16;
    const bool kwave = k0 < KP;
    f32x4 dq[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}}, dk[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    const int ti = wave == 0 ? 0 : 1, tj = wave == 2 ? 1 : 0;     // waves 0..2: tiles (0,0), (1,0), (1,1)

    for (int h = hk * a.rep; h < (hk + 1) * a.rep; h++) {
        const float* pre = d.chunks + ((int64_t)blockIdx.x * d.H + h) * kDeltaChunk;
        const float* st = d.states + ((int64_t)blockIdx.x * d.H + h) * (int64_t)(a.VP * KP);
        const DeltaWs w = delta_ws(a, gr.ws, blockIdx.x, h);
        __syncthreads();
        stage_mat<3, false>(pre, M, tid, 512);
        for (int i = tid; i < 3 * kDC; i += 512) sv[i] = pre[kDeltaG + i];
        if (wave == 7) {
            const int64_t at = (s.row + t0 + lane) * d.H + h;
            double c = lane < n ? (double)delta_decay(d.g[at]) : 0.0;
#pragma unroll
            for (int o = 1; o < kDC; o <<= 1) {
                const double y = __shfl_up(c, o, kDC);
                if ((lane & 31) >= o) c += y;
            }
            if (lane < kDC) sc[lane] = c;
        }
        __syncthreads();
        f32x4 dp = {0, 0, 0, 0}, z = {0, 0, 0, 0};
        f32x4 q1[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}}, k1[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}},
              k2[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
        float bsum[8] = {0, 0, 0, 0, 0, 0, 0, 0}, ss = 0.f;
        for (int vt = 0; vt < a.VP; vt += VT) {
            const int vl = wave * 16 + l16, v = vt + vl;
            float u[8], dr[8], o[8];
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = dr[i] = o[i] = 0.f;
            if (vt + wave * 16 < a.VP) {
                f32x4 ks[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
                for (int i = 0; i < KP / 32; i++) {
                    const float* p = st + (int64_t)v * KP + 32 * i + g4;
                    const f32x4 lo = *reinterpret_cast<const f32x4*>(p), hi = *reinterpret_cast<const f32x4*>(p + 16);
                    const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    const Frag<3> b = split8<3>(x);
#pragma unroll
                    for (int m = 0; m < 2; m++) ks[m] = mma<3>(K.frag(16 * m, i, lane), b, ks[m]);
                }
                const T* vp = delta_at<T>(d.v, d.v_stride, s.b, s.t0 + t0, h) + v;
                const int64_t at = ((s.row + t0) * d.H + h) * (int64_t)V + v;
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int t = res_row(i >> 2, lane, i & 3);
                    const bool live = t < n && v < V;
                    const float xx = (live ? (float)vp[t * d.v_stride[1]] : 0.f) - sv[t] * ks[i >> 2][i & 3];
                    dr[i] = w.dr[(int64_t)t * a.VP + v];
                    o[i] = live ? (float)static_cast<const T*>(gr.dout)[at + (int64_t)t * d.H * V] : 0.f;
                    if (live) static_cast<T*>(gr.dv)[at + (int64_t)t * d.H * V] = (T)(sv[2 * kDC + t] * dr[i]);
                    bsum[i] = fmaf(dr[i], xx, bsum[i]);
                    x[i] = sv[2 * kDC + t] * xx;
                }
                const Frag<3> R = split8<3>(x);
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    const f32x4 um = mma<3>(M.frag(16 * m, 0, lane), R, f32x4{0, 0, 0, 0});
#pragma unroll
                    for (int r = 0; r < 4; r++) u[4 * m + r] = um[r];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int t = res_row(i >> 2, lane, i & 3);
                U.put(t, vl, u[i]);
                DR.put(t, vl, dr[i]);
                DO.put(t, vl, o[i]);
            }
            __syncthreads();
            const int nv = (a.VP - vt < VT ? a.VP - vt + 31 : VT) / 32;
            if (wave < 3)
                for (int i = 0; i < nv; i++) {
                    const Frag<3> b = U.frag(16 * tj, i, lane);
                    dp = mma<3>(DO.frag(16 * ti, i, lane), b, dp);
                    z = mma<3>(DR.frag(16 * ti, i, lane), b, z);
                }
            if (kwave)
                for (int i = 0; i < nv; i++) {
                    float x[8], y[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int vv = vt + 32 * i + g4 + (j & 3) + (j >> 2) * 16;
                        x[j] = vv < a.VP ? st[(int64_t)vv * KP + k0 + l16] : 0.f;
                        y[j] = vv < a.VP ? w.ds[(int64_t)vv * KP + k0 + l16] : 0.f;
                        ss = fmaf(x[j], y[j], ss);
                    }
                    const Frag<3> b = split8<3>(x), e = split8<3>(y);
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        q1[m] = mma<3>(DO.frag(16 * m, i, lane), b, q1[m]);
                        k1[m] = mma<3>(DR.frag(16 * m, i, lane), b, k1[m]);
                        k2[m] = mma<3>(U.frag(16 * m, i, lane), e, k2[m]);
                    }
                }
            __syncthreads();
        }
        // the V tiles are done with: K and Q by column take their place
        stage_tile<T, P, KP, false, true>(kp, d.k_stride[1], n, Kd, a.vec_k, none, KT, tid, 512);
        stage_tile<T, P, KP, false, true>(qp, d.q_stride[1], n, Kd, a.vec_q, none, QT, tid, 512);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float b = sum16(bsum[i]);
            if (l16 == 0) red[wave][res_row(i >> 2, lane, i & 3)] = b;
        }
        ss = sum16(sum_groups(ss));
        if (lane == 0) dots[wave] = ss;
        if (wave < 3) {
            f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < KP / 32; i++) {
                const Frag<P> b = K.frag(16 * tj, i, lane);
                kk = mma<3>(K.frag(16 * ti, i, lane), b, kk);
                qk = mma<3>(Q.frag(16 * ti, i, lane), b, qk);
            }
            const int col = tj * 16 + l16;
            float esum = 0.f;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = res_row(ti, lane, r);
                const float D = col <= row ? expf((float)(sc[row] - sc[col])) : 0.f;
                const float zd = col < row ? D * z[r] : 0.f, f = -sv[2 * kDC + row] * zd;
                const float y = (float)d.scale * D * dp[r], e = col < row ? y * qk[r] + f * kk[r] : 0.f;
                const float er = sum16(e), zr = sum16(zd * kk[r]);
                if (l16 == 0) {
                    trow[wave][g4 + r] = er;
                    tzk[wave][g4 + r] = zr;
                }
                esum += e;
                z[r] = f;
                Y.put(row, col, y);
                YT.put(col, row, y);
                if (ti != tj) {
                    Y.put(col, row, 0.f);
                    YT.put(row, col, 0.f);
                    FF.put(row, col, f);
                    FF.put(col, row, f);
                }
            }
            esum = sum_groups(esum);
            if (lane < 16) tcol[wave][lane] = esum;
            if (ti == tj) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    // F_ji of this lane's (i, j): row j of column i, in lane 16 (j / 4) + i
                    float t = 0.f;
#pragma unroll
                    for (int rr = 0; rr < 4; rr++) {
                        const float x = __shfl(z[rr], (l16 >> 2) * 16 + g4 + r);
                        if ((l16 & 3) == rr) t = x;
                    }
                    FF.put(res_row(ti, lane, r), col, z[r] + t);
                }
            }
        }
        __syncthreads();
        if (kwave) {
            const int kc = k0 + l16;
            const Frag<P> bk = KT.frag(k0, 0, lane), bq = QT.frag(k0, 0, lane);
#pragma unroll
            for (int m = 0; m < 2; m++) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int t = res_row(m, lane, r);
                    const float G = sv[t], qv = Q.get(t, kc), kv = K.get(t, kc);
                    q1[m][r] *= (float)d.scale * G;
                    k1[m][r] *= -sv[2 * kDC + t] * G;
                    k2[m][r] *= sv[kDC + t];
                    const float cr = sum16(qv * q1[m][r] + kv * k1[m][r]), cw = sum16(kv * k2[m][r]);
                    if (l16 == 0) {
                        kread[wave][t] = cr;
                        kwrite[wave][t] = cw;
                    }
                }
                q1[m] = mma<3>(Y.frag(16 * m, 0, lane), bk, q1[m]);
                k1[m] = mma<3>(YT.frag(16 * m, 0, lane), bq, k1[m] + k2[m]);
                k1[m] = mma<3>(FF.frag(16 * m, 0, lane), bk, k1[m]);
                dq[m] += q1[m];
                dk[m] += k1[m];
            }
        }
        __syncthreads();
        if (tid < kDC) {
            // dg_t: reads and E by later tokens, less E's columns there, and the writes of
            // earlier ones (a write's share in dc_C less its own dc is left of its token)
            const int t = tid, hi = t >> 4, lo = t & 15;
            float dc = hi ? trow[1][lo] + trow[2][lo] - tcol[2][lo] : trow[0][lo] - tcol[0][lo] - tcol[1][lo];
            float db = hi ? -tzk[1][lo] - tzk[2][lo] : -tzk[0][lo];
            float wr = 0.f, all = 0.f;
            for (int i = 0; i < KP / 16; i++) {
                dc += kread[i][t];
                wr += kwrite[i][t];
                all += dots[i];
            }
            for (int i = 0; i < 8; i++) db += red[i][t];
#pragma unroll
            for (int o = 1; o < kDC; o <<= 1) {
                const float x = __shfl_down(dc, o, kDC), y = __shfl_up(wr, o, kDC);
                if (t + o < kDC) dc += x;
                if (t >= o) wr += y;
            }
            const float before = __shfl_up(wr, 1, kDC);
            dc += (t ? before : 0.f) + sv[kDC - 1] * all;
            if (t < n) {
                gr.dg[(s.row + t0 + t) * d.H + h] = dc;
                gr.dbeta[(s.row + t0 + t) * d.H + h] = db;
            }
        }
    }
    if (kwave && k0 + l16 < Kd)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int t = res_row(i >> 2, lane, i & 3);
            const int64_t at = ((s.row + t0 + t) * d.Hk + hk) * (int64_t)Kd + k0 + l16;
            if (t < n) {
                static_cast<T*>(gr.dq)[at] = (T)dq[i >> 2][i & 3];
                static_cast<T*>(gr.dk)[at] = (T)dk[i >> 2][i & 3];
            }
        }
}

template <typename T, int KP>
snhip_status bwd_t(const DeltaP& a, const SnHipDeltaGrad& gr, hipStream_t st) {
    const int strips = a.VP / 16, W = strips >= 4 ? 4 : strips >= 2 ? 2 : 1;
    const dim3 grid((unsigned)((strips + W - 1) / W), (unsigned)a.d.H, (unsigned)a.d.N);
    if (W == 4) k_delta_rscan<T, KP, 4><<<grid, 256, 0, st>>>(a, gr);
    else if (W == 2) k_delta_rscan<T, KP, 2><<<grid, 128, 0, st>>>(a, gr);
    else k_delta_rscan<T, KP, 1><<<grid, 64, 0, st>>>(a, gr);
    SNHIP_CHECK(hipGetLastError());
    k_delta_local<T, KP><<<dim3((unsigned)a.slots, (unsigned)a.d.Hk), 512, 0, st>>>(a, gr);
    SNHIP_CHECK(hipGetLastError());
    return SNHIP_OK;
}

}  // namespace
}  // namespace snhip

using namespace snhip;

extern "C" {

int64_t snhip_op_delta_bwd_floats(const SnHipDelta* d) {
    return d ? delta_slots(*d) * d->H * delta_vp(d->V) * (kDC + (int64_t)delta_kp(d->K)) : 0;
}

snhip_status snhip_op_delta_bwd_dev(const SnHipDelta* d, const SnHipDeltaGrad* gr, void* stream) {
    DeltaP a;
    const snhip_status rc = delta_args(d, &a);
    if (rc != SNHIP_OK || !gr || !d->chunks || !d->states || !gr->dout || !gr->dq || !gr->dk || !gr->dv ||
        !gr->dg || !gr->dbeta || !gr->ws)
        return SNHIP_E_INVAL;
    const hipStream_t st = as_stream(stream);
    if (a.KP == 64) {
        if (d->dtype == SNHIP_F32) return bwd_t<float, 64>(a, *gr, st);
        if (d->dtype == SNHIP_BF16) return bwd_t<__bf16, 64>(a, *gr, st);
        return bwd_t<_Float16, 64>(a, *gr, st);
    }
    if (d->dtype == SNHIP_F32) return bwd_t<float, 128>(a, *gr, st);
    if (d->dtype == SNHIP_BF16) return bwd_t<__bf16, 128>(a, *gr, st);
    return bwd_t<_Float16, 128>(a, *gr, st);
}

}  // extern "C"
