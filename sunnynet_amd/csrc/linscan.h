// The recurrence of linear.h over chunks, for one element type (linscan_*.hip).
#pragma once

#include <type_traits>

#include "linear.h"

namespace snhip {
namespace {

// A value of the place where it is used: what it makes, addresses mostly, is made there and
// not carried around a loop in registers.
__device__ __forceinline__ int here(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// An (R, W) tile of a (tokens, columns) array on its way from memory to LDS, held by 256
// threads: tokens from n on and columns from `cols` on are 0 (a stride below `cols` would let
// the window alone hand out other rows).
template <typename T, int R, int W> struct LinFetch {
    static constexpr int P = ElemPlanes<T>::n, N = R * W / 8 / 256;
    static_assert(R * W / 8 % 256 == 0);
    Vec8<T> x[N];
    __device__ __forceinline__ void load(const T* src, int64_t stride, int n, int cols, bool vec, int tid) {
        const __amdgpu_buffer_rsrc_t r = rows_window(src, stride, n, cols);
        const int step = (int)stride;
        if (vec) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int i = tid + j * 256, t = i / (W / 8), c = i % (W / 8) * 8;
                x[j] = buf_load8<T>(r, t < n && c < cols ? (t * step + c) * (int)sizeof(T) : kNowhere, 8, true);
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int i = here(tid) + j * 256, t = i / (W / 8), c = i % (W / 8) * 8;
                x[j] = buf_load8<T>(r, (t * step + c) * (int)sizeof(T), t < n ? cols - c : 0, false);
            }
        }
    }
    template <typename Tl> __device__ __forceinline__ void store(Tl to, int tid) const {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = tid + j * 256;
            to.put8(i / (W / 8), i % (W / 8) * 8, split_raw8<T>(x[j]));
        }
    }
};

// Values of a fragment, its planes added from the smallest.
template <int P> __device__ __forceinline__ void join8(const Frag<P>& f, float* x) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        x[i] = (float)f.p[P - 1][i];
#pragma unroll
        for (int p = P - 2; p >= 0; p--) x[i] += (float)f.p[p][i];
    }
}

// The row of tile i of a lower triangle, counted by rows: 0; 1, 1; 2, 2, 2; 3, ...
__device__ __forceinline__ int lin_tile_row(int i) { return i < 1 ? 0 : i < 3 ? 1 : i < 6 ? 2 : 3; }

// One part of one sequence and head, 64 NC columns: four waves of 16 NC columns each. REV:
// backward in time. DOT: with X.y. STATE: only the part's sum of B C^T. The next chunk's
// tiles are fetched into registers while this one is worked on.
template <typename T, int DP, int NC, bool REV, bool DOT, bool STATE>
__global__ __launch_bounds__(256, ElemPlanes<T>::n == 1 ? 2 : 1) void k_lin(LinShape d, LinPass a) {
    constexpr int P = ElemPlanes<T>::n, C = LinChunk<T>::n, NB = C / 32, NK = DP / 16, W = 64 * NC, E = (int)sizeof(T);
    typedef Tile<P, C, DP> Rows;
    typedef Tile<P, C, W> Cols;
    typedef Tile<3, C, C> Mat;
    __shared__ alignas(16) __bf16 sa[STATE ? 8 : Rows::elems], sb[Rows::elems], sc[Cols::elems], sp[STATE ? 8 : Mat::elems];
    __shared__ struct { double c[C]; float row[C], upd[C]; } s;      // a chunk's running sums, row factors and weights
    __shared__ float sdiag[DOT ? C : 1];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int lane = tid & 63, l16 = lane & 15, g8 = (lane >> 4) * 8;
    const int h = blockIdx.y, ncol = (a.cols + W - 1) / W;
    const int col_block = blockIdx.z % ncol, row_block = blockIdx.z / ncol;
    const int rows = a.rows - row_block * kLinRows < DP ? a.rows - row_block * kLinRows : DP;
    const int cols = a.cols - col_block * W < W ? a.cols - col_block * W : W;
    LinSeq q;
    int64_t seq;
    int part;
    if (!lin_part_of(d, blockIdx.x, &q, &seq, &part)) return;
    const int begin = part * d.part;
    const bool last = begin + d.part >= q.len, first_run = REV ? last : part == 0, last_run = REV ? part == 0 : last;
    if (STATE && last_run) return;             // nothing begins with it
    const int stop = last ? q.len : begin + d.part;
    const Rows A{sa}, Bt{sb};
    const Cols Ct{sc};
    const Mat Pm{sp};

    // place of row i, column j of this block's S in a (K, V) state
    const int r0 = row_block * kLinRows, c0 = col_block * W + wave * 16 * NC;
    const int64_t rs = a.turned ? 1 : d.V, cs = a.turned ? d.V : 1, kv = d.K * d.V;
    auto each_state = [&](auto f) {
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
            for (int kt = 0; kt < NK; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = (kt >> 1) * 32 + g8 + 4 * (kt & 1) + r, j = c0 + 16 * n + l16;
                    f(n, kt, r, (r0 + i) * rs + j * cs, i < rows && j < a.cols);
                }
    };
    f32x4 S[NC][NK];       // S[n][2 p + e][r] is row 32 p + g8 + 4 e + r of column 16 n + l16
    {
        const float* from = first_run ? (a.begin ? a.begin + (seq * d.H + h) * kv : nullptr)
                                      : a.parts + ((int64_t)blockIdx.x * d.H + h) * kv;
        if (STATE) from = nullptr;
        each_state([&](int n, int kt, int r, int64_t at, bool in) { S[n][kt][r] = from && in ? from[at] : 0.f; });
    }
    LinFetch<T, C, DP> fa, fb;
    LinFetch<T, C, W> fc;
    float fg = 0.f;
    const T* ap = STATE ? nullptr : lin_at<T>(a.A, q.b, q.t0, h) + r0;
    const T* bp = lin_at<T>(a.B, q.b, q.t0, h) + r0;
    const T* cp = lin_at<T>(a.C, q.b, q.t0, h) + col_block * W;
    const T* xp = DOT ? lin_at<T>(a.X, q.b, q.t0, h) : nullptr;
    auto fetch = [&](int t0) {
        const int n = q.len - t0 < C ? q.len - t0 : C;
        if (!STATE) fa.load(ap + t0 * a.A.st[1], a.A.st[1], n, rows, a.vec, tid);
        fb.load(bp + t0 * a.B.st[1], a.B.st[1], n, rows, a.vec, tid);
        fc.load(cp + t0 * a.C.st[1], a.C.st[1], n, cols, a.vec, tid);
        if (wave == 0) fg = lane < n ? d.g[d.head_g ? h : (q.row + t0 + lane) * d.H + h] : 0.f;
    };
    auto store = [&]() {
        if (!STATE) fa.store(A, tid);
        fb.store(Bt, tid);
        fc.store(Ct, tid);
        if (wave == 0) {
            double c = (double)lin_decay(fg);
#pragma unroll
            for (int o = 1; o < C; o <<= 1) {
                const double y = __shfl_up(c, o);
                if (lane >= o) c += y;
            }
            const double end = __shfl(c, C - 1);
            if (lane < C) {
                s.c[lane] = c;
                const float in = expf((float)c), out = expf((float)(end - c));
                s.row[lane] = REV ? out : d.scale * in;
                s.upd[lane] = REV ? d.scale * in : out;
            }
        }
    };
    if constexpr (!STATE) {                    // the tiles beside the diagonal that products of 32 read
        for (int i = tid; i < 3 * C * C / 8; i += 256) {
            const int p = i / (C * C / 8), k = i % (C * C / 8);
            *reinterpret_cast<bf16x8*>(Pm.at(p, k / (C / 8), k % (C / 8) * 8)) = bf16x8{};
        }
    }
    const int n_chunks = (stop - begin + C - 1) / C;
    auto chunk_at = [&](int i) { return begin + (REV ? n_chunks - 1 - i : i) * C; };
    double total = 0.;
    if (n_chunks > 0) {
        fetch(chunk_at(0));
        store();
    }
    barrier_lds();
    for (int ci = 0; ci < n_chunks; ci++) {
        const int t0 = chunk_at(ci), n = q.len - t0 < C ? q.len - t0 : C;
        const bool more = ci + 1 < n_chunks;
        if (more) fetch(chunk_at(ci + 1));
        lane = here(lane);
        l16 = lane & 15;
        g8 = (lane >> 4) * 8;
        const double c_end = s.c[C - 1];
        const float decay = expf((float)c_end);
        total += c_end;
        f32x4 y[NC][NB][2];
        if constexpr (!STATE) {
            // P, made transposed: a lane has four neighbouring columns of one row
            constexpr int NT = C / 16;
#pragma unroll
            for (int t = wave; t < NT * (NT + 1) / 2; t += 4) {
                const int hi = lin_tile_row(t), lo = t - hi * (hi + 1) / 2, ti = REV ? lo : hi, tj = REV ? hi : lo;
                f32x4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < DP; p += 32)
                    acc = mma<3>(Bt.frag(16 * tj + l16, p, lane), A.frag(16 * ti + l16, p, lane), acc);
                const int i = 16 * ti + l16, j0 = 16 * tj + (lane >> 4) * 4;
                const double ci_ = s.c[i];
                float x[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int j = j0 + r;
                    const double gap = REV ? s.c[j] - ci_ : ci_ - s.c[j];
                    x[r] = (REV ? j >= i : j <= i) ? d.scale * expf((float)gap) * acc[r] : 0.f;
                    if (DOT && j == i) {
                        sdiag[i] = x[r];
                        x[r] = 0.f;
                    }
                }
#pragma unroll
                for (int p = 0; p < 3; p++) {
                    bf16x4 o;
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        o[r] = (__bf16)x[r];
                        x[r] -= (float)o[r];
                    }
                    *reinterpret_cast<bf16x4*>(Pm.at(p, i, j0)) = o;
                }
            }
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int m = 0; m < 2; m++) y[c][b][m] = {0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < DP / 32; p++) {
                Frag<3> f[NC];
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    float x[8];
#pragma unroll
                    for (int r = 0; r < 4; r++) x[r] = S[c][2 * p][r], x[4 + r] = S[c][2 * p + 1][r];
                    f[c] = split8<3>(x);
                }
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const Frag<P> af[2] = {A.frag(32 * b + pair_row(0, l16), 32 * p, lane),
                                           A.frag(32 * b + pair_row(1, l16), 32 * p, lane)};
#pragma unroll
                    for (int c = 0; c < NC; c++) mma_n<3>(af, f[c], y[c][b]);
                }
            }
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float f = s.row[32 * b + g8 + i];
#pragma unroll
                    for (int c = 0; c < NC; c++) y[c][b][i >> 2][i & 3] *= f;
                }
        }
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int kt = 0; kt < NK; kt++) S[c][kt] *= decay;
        Frag<P> cf[NB][NC];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            Frag<3> u[NC];
#pragma unroll
            for (int c = 0; c < NC; c++) {
                cf[b][c] = Ct.tfrag(32 * b, wave * 16 * NC + 16 * c + 4 * (lane & 3), lane);
                float x[8];
                join8(cf[b][c], x);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] *= s.upd[32 * b + g8 + i];
                u[c] = split8<3>(x);
            }
#pragma unroll
            for (int k2 = 0; k2 < NK; k2 += 2) {
                const Frag<P> bf[2] = {Bt.tfrag(32 * b, 16 * k2 + 8 * (lane & 3), lane),
                                       Bt.tfrag(32 * b, 16 * k2 + 8 * (lane & 3) + 4, lane)};
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    f32x4 t[2] = {S[c][k2], S[c][k2 + 1]};
                    mma_n<3>(bf, u[c], t);
                    S[c][k2] = t[0];
                    S[c][k2 + 1] = t[1];
                }
            }
        }
        unsigned xv[DOT ? NC * NB * 8 : 1];
        if constexpr (DOT) {
            const __amdgpu_buffer_rsrc_t r = rows_window(xp + t0 * a.X.st[1], a.X.st[1], n, a.cols);
            const int step = (int)a.X.st[1] * E;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const int j = c0 + 16 * c + l16, off = j < a.cols ? (32 * b + g8) * step + j * E : kNowhere;
#pragma unroll
                    for (int i = 0; i < 8; i++) xv[(b * NC + c) * 8 + i] = buf_load_bits<T>(r, off + i * step);
                }
        }
        barrier_lds();
        if (more) store();                     // only P is read from here on
        if constexpr (!STATE) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int jb = REV ? b : 0; jb < (REV ? NB : b + 1); jb++) {
                    const Frag<3> pf[2] = {Pm.frag(32 * b + pair_row(0, l16), 32 * jb, lane),
                                           Pm.frag(32 * b + pair_row(1, l16), 32 * jb, lane)};
#pragma unroll
                    for (int c = 0; c < NC; c++) mma_n<3>(pf, cf[jb][c], y[c][b]);
                }
            if constexpr (DOT) {
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    float own[NC][8];
#pragma unroll
                    for (int c = 0; c < NC; c++) join8(cf[b][c], own[c]);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int t = 32 * b + g8 + i;
                        float e = 0.f;
#pragma unroll
                        for (int c = 0; c < NC; c++) {
                            f32x4& o = y[c][b][i >> 2];
                            e = fmaf(float_of_bits<T>(xv[(b * NC + c) * 8 + i]), o[i & 3], e);
                            o[i & 3] = fmaf(sdiag[t], own[c][i], o[i & 3]);
                        }
                        e = sum16(e);
                        if (l16 == 0 && t < n)
                            a.dot[((row_block * 4 + wave) * (d.B * d.T) + q.row + t0 + t) * d.H + h] = e;
                    }
                }
            }
            const int64_t HY = d.H / a.y_rep, row = q.row + t0;
            const int64_t slice = a.y_f32 ? ((int64_t)row_block * a.y_rep + h % a.y_rep) * (d.B * d.T) : 0;
            const int64_t at = ((slice + row) * HY + h / a.y_rep) * a.cols;
            const int64_t step = HY * a.cols;
            auto put = [&](auto zero) {
                typedef decltype(zero) U;
                const __amdgpu_buffer_rsrc_t ry = rows_window(static_cast<const U*>(a.y) + at, step, n, a.cols);
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        const int j = c0 + 16 * c + l16;
                        const int off = j < a.cols ? ((32 * b + g8) * (int)step + j) * (int)sizeof(U) : kNowhere;
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            buf_store<U>(ry, off + i * (int)step * (int)sizeof(U), (U)y[c][b][i >> 2][i & 3]);
                    }
            };
            if (a.y_f32) put(0.f);
            else put(T(0.f));
        }
        barrier_lds();
    }
    if (STATE) {
        float* to = a.parts + ((int64_t)blockIdx.x * d.H + h) * kv;
        each_state([&](int n, int kt, int r, int64_t at, bool in) {
            if (in) to[at] = S[n][kt][r];
        });
        if (tid == 0 && blockIdx.z == 0) a.decay[(int64_t)blockIdx.x * d.H + h] = expf((float)total);
    } else if (last_run && a.end) {
        float* to = a.end + (seq * d.H + h) * kv;
        each_state([&](int n, int kt, int r, int64_t at, bool in) {
            if (in) to[at] = S[n][kt][r];
        });
    }
}

template <typename T> snhip_status lin_run(const LinShape& d, const LinPass& a, bool rev, int kind, hipStream_t st) {
    auto go = [&](auto dp, auto nc, auto back, auto dot, auto state) -> snhip_status {
        constexpr int W = 64 * decltype(nc)::value;
        const int64_t z = (int64_t)((a.cols + W - 1) / W) * ((a.rows + kLinRows - 1) / kLinRows);
        const dim3 grid((unsigned)d.slots, (unsigned)d.H, (unsigned)z);
        k_lin<T, decltype(dp)::value, decltype(nc)::value, decltype(back)::value, decltype(dot)::value,
              decltype(state)::value><<<grid, 256, 0, st>>>(d, a);
        SNHIP_CHECK(hipGetLastError());
        return SNHIP_OK;
    };
    typedef std::integral_constant<int, 1> one;
    typedef std::integral_constant<int, 2> two;
    auto by_kind = [&](auto dp, auto nc, auto back) {
        if (kind == 0) return go(dp, nc, back, std::false_type(), std::false_type());
        if (kind == 1) return go(dp, nc, back, std::true_type(), std::false_type());
        return go(dp, nc, back, std::false_type(), std::true_type());
    };
    auto by_dir = [&](auto dp, auto nc) {
        return rev ? by_kind(dp, nc, std::true_type()) : by_kind(dp, nc, std::false_type());
    };
    auto by_cols = [&](auto dp) { return a.cols <= 64 ? by_dir(dp, one()) : by_dir(dp, two()); };
    return a.rows <= 64 ? by_cols(std::integral_constant<int, 64>()) : by_cols(std::integral_constant<int, 128>());
}

}  // namespace
}  // namespace snhip
