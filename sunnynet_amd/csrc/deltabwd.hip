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

// Per slot and head: dR^T (VP, 32), then dS^T (VP, KP) after the chunk.
struct DeltaWs {
    float* dr;
    float* ds;
};
__host__ __device__ inline DeltaWs delta_ws(const DeltaP& a, float* ws, int64_t slot, int h) {
    const int64_t i = slot * a.d.H + h, nr = a.slots * a.d.H * kDC * a.VP;
    return {ws + i * kDC * a.VP, ws + nr + i * (int64_t)(a.VP * a.KP)};
}

template <typename T, int KP, bool VEC>
__global__ __launch_bounds__(64 * kDeltaW) void k_delta_rscan(DeltaP a, SnHipDeltaGrad gr) {
    constexpr int P = ElemPlanes<T>::n, NK = KP / 16, W = kDeltaW, NTH = 64 * W;
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
    MatFetch<3, NTH> fm, fp;
    float fv[(3 * kDC + NTH - 1) / NTH];
    unsigned vv[8];
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
        const DeltaWs w = delta_ws(a, gr.ws, s.slot + t0 / kDC, h);
        float G[8], L[8], be[8], x[8], y[8];
        float od[8];
#pragma unroll
        for (int i = 0; i < 8; i++) od[i] = float_of_bits<T>(vv[i]);
        if (t0 > 0) fetch(t0 - kDC);
        const __amdgpu_buffer_rsrc_t rds = make_rsrc(w.ds, (uint32_t)(a.VP * KP * 4)),
                                     rdr = make_rsrc(w.dr, (uint32_t)(a.VP * kDC * 4));
#pragma unroll
        for (int kt = 0; kt < NK; kt++)
            buf_store4(rds, (v * KP + g8) * 4 + ((kt >> 1) * 32 + 4 * (kt & 1)) * 4, S[kt]);
        f32x4 du[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int p = 0; p < KP / 32; p++) {
#pragma unroll
            for (int r = 0; r < 4; r++) x[r] = S[2 * p][r], x[4 + r] = S[2 * p + 1][r];
            const Frag<3> f = split8<3>(x);
#pragma unroll
            for (int m = 0; m < 2; m++) du[m] = mma<3>(K.frag(pair_row(m, l16), 32 * p, lane), f, du[m]);
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
        for (int m = 0; m < 2; m++) {
#pragma unroll
            for (int r = 0; r < 4; r++) du[m][r] *= L[4 * m + r];
            du[m] = mma<3>(PM.tfrag(0, 8 * (lane & 3) + 4 * m, lane), dO, du[m]);
#pragma unroll
            for (int r = 0; r < 4; r++) x[4 * m + r] = du[m][r];
        }
        const Frag<3> dU = split8<3>(x);
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const f32x4 dr = mma<3>(M.tfrag(0, 8 * (lane & 3) + 4 * m, lane), dU, f32x4{0, 0, 0, 0});
            buf_store4(rdr, (v * kDC + g8 + 4 * m) * 4, dr);
#pragma unroll
            for (int r = 0; r < 4; r++) y[4 * m + r] = -dr[r] * be[4 * m + r] * G[4 * m + r];
        }
        const Frag<3> BdR = split8<3>(y);
        const float decay = sv[b][kDC - 1];
#pragma unroll
        for (int kt = 0; kt < NK; kt++) {
            const int block = (kt >> 1) * 32 + 8 * (lane & 3) + 4 * (kt & 1);
            S[kt] = mma<3>(Q.tfrag(0, block, lane), GdO, S[kt] * decay);
            S[kt] = mma<3>(K.tfrag(0, block, lane), BdR, S[kt]);
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

__device__ __forceinline__ float sum_groups(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

// One chunk of one query and key head: a block of four waves runs over the value heads
// that share it, so dq and dk are summed in registers. Per head and 64 columns of V a
// wave first owns 16 columns (X, U, dV), then KP / 4 columns of K (the products with S
// and dS); the 32x32 matrices are made by three waves, a 16x16 tile each. U and dR lie
// in LDS by column of V, as the waves hold them, and are read transposed.
template <typename T, int KP, bool VEC>
__global__ __launch_bounds__(256, 2) void k_delta_local(DeltaP a, SnHipDeltaGrad gr, bool vec_o) {
    constexpr int P = ElemPlanes<T>::n, VT = 64, NC = KP / 64;     // NC tiles of 16 columns of K a wave
    typedef Tile<P, kDC, KP> Rows;
    typedef Tile<3, VT, kDC> Cols;
    typedef Tile<3, kDC, kDC> Mat;
    __shared__ alignas(16) __bf16 sk[Rows::elems], sq[Rows::elems], su[Cols::elems], sr[Cols::elems],
        so[Tile<P, kDC, VT>::elems], sx[2 * Mat::elems];
    __shared__ alignas(16) float sv[3 * kDC];
    __shared__ float red[4][kDC], kread[4][kDC], kwrite[4][kDC], trow[3][16], tzk[3][16], tcol[3][16], dots[4];
    __shared__ double sc[kDC];
    const SnHipDelta& d = a.d;
    const int hk = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g4 = (lane >> 4) * 4, g8 = 2 * g4,
              l16 = lane & 15, blk16 = 4 * (lane & 3), blkp = 8 * (lane & 3);
    DeltaSeq s;
    int chunk;
    if (!delta_chunk_of(d, blockIdx.x, &s, &chunk)) return;
    const int64_t t0 = (int64_t)chunk * kDC;
    const int n = (int)(s.len - t0 < kDC ? s.len - t0 : kDC), V = (int)d.V, Kd = (int)d.K;
    const Rows K{sk}, Q{sq};
    const Cols UT{su}, RT{sr};
    const Tile<P, kDC, VT> DO{so};
    const Mat M{sx}, Y{sx}, FF{sx + Mat::elems};        // Y takes M's place
    RowsFetch<T, KP, 256, VEC> f;
    f.init(d.k_stride[1], Kd, tid);
    f.load(delta_at<T>(d.k, d.k_stride, s.b, s.t0 + t0, hk), d.k_stride[1], n, Kd, tid);
    f.store(K, tid);
    f.init(d.q_stride[1], Kd, tid);
    f.load(delta_at<T>(d.q, d.q_stride, s.b, s.t0 + t0, hk), d.q_stride[1], n, Kd, tid);
    f.store(Q, tid);
    f32x4 dq[NC][2], dk[NC][2];
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
        for (int m = 0; m < 2; m++) dq[j][m] = dk[j][m] = f32x4{0, 0, 0, 0};
    const int ti = wave == 0 ? 0 : 1, tj = wave == 2 ? 1 : 0;     // waves 0..2: tiles (0,0), (1,0), (1,1)

    for (int h = hk * a.rep; h < (hk + 1) * a.rep; h++) {
        const float* rec = d.chunks + ((int64_t)blockIdx.x * d.H + h) * kDeltaChunk;
        const float* st = d.states + ((int64_t)blockIdx.x * d.H + h) * (int64_t)(a.VP * KP);
        const DeltaWs w = delta_ws(a, gr.ws, blockIdx.x, h);
        const T* vp = delta_at<T>(d.v, d.v_stride, s.b, s.t0 + t0, h);
        const int64_t at0 = ((s.row + t0) * d.H + h) * (int64_t)V;
        __syncthreads();
        {
            MatFetch<3, 256> fm;
            fm.load(make_rsrc(rec, kDeltaChunk * 4), 0, tid);
            fm.store(M, tid);
        }
        if (tid < 3 * kDC) sv[tid] = rec[kDeltaG + tid];
        if (wave == 3) {
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
        float G[8], be[8];
#pragma unroll
        for (int i = 0; i < 8; i++) G[i] = sv[g8 + i], be[i] = sv[2 * kDC + g8 + i];
        f32x4 dp = {0, 0, 0, 0}, z = {0, 0, 0, 0}, q1[NC][2], k1[NC][2], k2[NC][2];
#pragma unroll
        for (int j = 0; j < NC; j++)
#pragma unroll
            for (int m = 0; m < 2; m++) q1[j][m] = k1[j][m] = k2[j][m] = f32x4{0, 0, 0, 0};
        float bsum[8] = {0, 0, 0, 0, 0, 0, 0, 0}, ss = 0.f;
        for (int vt = 0; vt < a.VP; vt += VT) {
            const int vl = wave * 16 + l16, v = vt + vl;
            {
                const int t = tid >> 3, c = (tid & 7) * 8;
                const T* op = static_cast<const T*>(gr.dout) + at0 + (int64_t)t * d.H * V + vt + c;
                DO.put8(t, c, split_raw8<T>(load_raw8(op, t < n ? V - vt - c : 0, vec_o)));
            }
            float x[8], dr[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = dr[i] = 0.f;
            if (vt + wave * 16 < a.VP) {
                f32x4 ks[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
                float vv[8];
#pragma unroll
                for (int i = 0; i < 8; i++) vv[i] = g8 + i < n && v < V ? (float)vp[(g8 + i) * d.v_stride[1] + v] : 0.f;
                const Vec8<float> rv = load_raw8(w.dr + (int64_t)v * kDC + g8, 8, true);
#pragma unroll
                for (int p = 0; p < KP / 32; p++) {
                    const Frag<3> b = split_raw8<float>(load_raw8(st + (int64_t)v * KP + 32 * p + g8, 8, true));
#pragma unroll
                    for (int m = 0; m < 2; m++) ks[m] = mma<3>(K.frag(pair_row(m, l16), 32 * p, lane), b, ks[m]);
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float xx = vv[i] - G[i] * ks[i >> 2][i & 3];
                    dr[i] = rv[i];
                    if (g8 + i < n && v < V)
                        static_cast<T*>(gr.dv)[at0 + (int64_t)(g8 + i) * d.H * V + v] = (T)(be[i] * dr[i]);
                    bsum[i] = fmaf(dr[i], xx, bsum[i]);
                    x[i] = be[i] * xx;
                }
                const Frag<3> R = split8<3>(x);
#pragma unroll
                for (int m = 0; m < 2; m++) {
                    const f32x4 u = mma<3>(M.frag(pair_row(m, l16), 0, lane), R, f32x4{0, 0, 0, 0});
#pragma unroll
                    for (int r = 0; r < 4; r++) x[4 * m + r] = u[r];
                }
            }
            UT.put8(vl, g8, x);
            RT.put8(vl, g8, dr);
            __syncthreads();
            const int nv = a.VP - vt < VT ? (a.VP - vt + 31) & ~31 : VT;       // whole 32s
            if (wave < 3)
                for (int i = 0; i < nv; i += 32) {
                    const Frag<3> b = UT.tfrag(i, 16 * tj + blk16, lane);
                    dp = mma<3>(DO.frag(16 * ti + l16, i, lane), b, dp);
                    z = mma<3>(RT.tfrag(i, 16 * ti + blk16, lane), b, z);
                }
            for (int i = 0; i < nv; i += 32) {
#pragma unroll
                for (int j = 0; j < NC; j++) {
                    const int kc = (wave * NC + j) * 16 + l16;
                    float sx8[8], dx8[8];
#pragma unroll
                    for (int l = 0; l < 8; l++) {
                        const int vv = vt + i + g8 + l;
                        sx8[l] = vv < a.VP ? st[(int64_t)vv * KP + kc] : 0.f;
                        dx8[l] = vv < a.VP ? w.ds[(int64_t)vv * KP + kc] : 0.f;
                        ss = fmaf(sx8[l], dx8[l], ss);
                    }
                    const Frag<3> b = split8<3>(sx8), e = split8<3>(dx8);
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        q1[j][m] = mma<3>(DO.frag(pair_row(m, l16), i, lane), b, q1[j][m]);
                        k1[j][m] = mma<3>(RT.tfrag(i, blkp + 4 * m, lane), b, k1[j][m]);
                        k2[j][m] = mma<3>(UT.tfrag(i, blkp + 4 * m, lane), e, k2[j][m]);
                    }
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float b = sum16(bsum[i]);
            if (l16 == 0) red[wave][g8 + i] = b;
        }
        ss = sum_groups(sum16(ss));
        if (lane == 0) dots[wave] = ss;
        if (wave < 3) {
            f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < KP; c += 32) {
                const Frag<P> b = K.frag(16 * tj + l16, c, lane);
                kk = mma<3>(K.frag(16 * ti + l16, c, lane), b, kk);
                qk = mma<3>(Q.frag(16 * ti + l16, c, lane), b, qk);
            }
            const int col = tj * 16 + l16;
            float esum = 0.f;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int row = 16 * ti + g4 + r;
                const float D = col <= row ? expf((float)(sc[row] - sc[col])) : 0.f;
                const float zd = col < row ? D * z[r] : 0.f, ff = -sv[2 * kDC + row] * zd;
                const float y = (float)d.scale * D * dp[r], e = col < row ? y * qk[r] + ff * kk[r] : 0.f;
                const float er = sum16(e), zr = sum16(zd * kk[r]);
                if (l16 == 0) {
                    trow[wave][g4 + r] = er;
                    tzk[wave][g4 + r] = zr;
                }
                esum += e;
                z[r] = ff;
                Y.put(row, col, y);
                if (ti != tj) {
                    FF.put(row, col, ff);
                    FF.put(col, row, ff);
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
                    FF.put(16 * ti + g4 + r, col, z[r] + t);
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++) Y.put(g4 + r, 16 + l16, 0.f);
        }
        __syncthreads();
        float cr[8], cw[8];
#pragma unroll
        for (int i = 0; i < 8; i++) cr[i] = cw[i] = 0.f;
#pragma unroll
        for (int j = 0; j < NC; j++) {
            const int kc = (wave * NC + j) * 16;
            const Frag<P> bk = K.tfrag(0, kc + blk16, lane), bq = Q.tfrag(0, kc + blk16, lane);
#pragma unroll
            for (int m = 0; m < 2; m++) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = 4 * m + r, t = g8 + i;
                    const float qv = Q.get(t, kc + l16), kv = K.get(t, kc + l16);
                    q1[j][m][r] *= (float)d.scale * G[i];
                    k1[j][m][r] *= -be[i] * G[i];
                    k2[j][m][r] *= sv[kDC + t];
                    cr[i] = fmaf(qv, q1[j][m][r], fmaf(kv, k1[j][m][r], cr[i]));
                    cw[i] = fmaf(kv, k2[j][m][r], cw[i]);
                }
                dq[j][m] += mma<3>(Y.frag(pair_row(m, l16), 0, lane), bk, q1[j][m]);
                f32x4 t = mma<3>(Y.tfrag(0, blkp + 4 * m, lane), bq, k1[j][m] + k2[j][m]);
                dk[j][m] += mma<3>(FF.frag(pair_row(m, l16), 0, lane), bk, t);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float r = sum16(cr[i]), wr = sum16(cw[i]);
            if (l16 == 0) {
                kread[wave][g8 + i] = r;
                kwrite[wave][g8 + i] = wr;
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
            for (int i = 0; i < 4; i++) {
                dc += kread[i][t];
                wr += kwrite[i][t];
                all += dots[i];
                db += red[i][t];
            }
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
#pragma unroll
    for (int j = 0; j < NC; j++) {
        const int kc = (wave * NC + j) * 16 + l16;
        if (kc >= Kd) continue;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int64_t at = ((s.row + t0 + g8 + i) * d.Hk + hk) * (int64_t)Kd + kc;
            if (g8 + i < n) {
                static_cast<T*>(gr.dq)[at] = (T)dq[j][i >> 2][i & 3];
                static_cast<T*>(gr.dk)[at] = (T)dk[j][i >> 2][i & 3];
            }
        }
    }
}

template <typename T, int KP, bool VEC>
snhip_status bwd_t(const DeltaP& a, const SnHipDeltaGrad& gr, hipStream_t st) {
    const dim3 grid((unsigned)((a.VP / 16 + kDeltaW - 1) / kDeltaW), (unsigned)a.d.H, (unsigned)a.d.N);
    k_delta_rscan<T, KP, VEC><<<grid, 64 * kDeltaW, 0, st>>>(a, gr);
    SNHIP_CHECK(hipGetLastError());
    const bool vec_o = a.d.V % 8 == 0 && reinterpret_cast<uintptr_t>(gr.dout) % 16 == 0;
    k_delta_local<T, KP, VEC><<<dim3((unsigned)a.slots, (unsigned)a.d.Hk), 256, 0, st>>>(a, gr, vec_o);
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
    return delta_pick(a, [&](auto t, auto kp, auto vec) {
        return bwd_t<decltype(t), decltype(kp)::value, decltype(vec)::value>(a, *gr, st);
    });
}

}  // extern "C"
