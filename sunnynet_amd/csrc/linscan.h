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

__device__ __forceinline__ float exp2_of(double x) { return __builtin_amdgcn_exp2f((float)x); }

// Values of a fragment, its planes added from the smallest.
template <int P> __device__ __forceinline__ void join8(const Frag<P>& f, float* x) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        x[i] = (float)f.p[P - 1][i];
#pragma unroll
        for (int p = P - 2; p >= 0; p--) x[i] += (float)f.p[p][i];
    }
}

template <int P> __device__ __forceinline__ void join4(const Frag<P>& f, float* x) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[i] = (float)f.p[P - 1][i];
#pragma unroll
        for (int p = P - 2; p >= 0; p--) x[i] += (float)f.p[p][i];
    }
}

// acc[m][n] += a[n] b[m] (mma): N M products next to each other, none of which waits for another.
template <int LIM, int N, int M, int NA, int NB>
__device__ __forceinline__ void mma_nm(const Frag<NA> (&a)[N], const Frag<NB> (&b)[M], f32x4 (&acc)[M][N]) {
#pragma unroll
    for (int s = LIM - 1; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < NA; i++) {
            const int j = s - i;
            if (j >= 0 && j < NB)
#pragma unroll
                for (int m = 0; m < M; m++)
#pragma unroll
                    for (int n = 0; n < N; n++)
                        acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[n].p[i], b[m].p[j], acc[m][n], 0, 0, 0);
        }
}

// Four neighbouring elements from `off`, of which the first n exist. vec: aligned, all exist.
template <typename T> __device__ __forceinline__ void buf_load4e(__amdgpu_buffer_rsrc_t r, int off, int n, bool vec, float* x) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const f32x4 v = buf_load4(r, off);
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = v[i];
        } else {
            typedef T T4 __attribute__((ext_vector_type(4)));
            const T4 v = __builtin_bit_cast(T4, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = (float)v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (float)buf_load<T>(r, i < n ? off + i * (int)sizeof(T) : kNowhere);
    }
}
template <typename T> __device__ __forceinline__ void buf_store4e(__amdgpu_buffer_rsrc_t r, int off, int n, bool vec, f32x4 x) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (vec) {
        if constexpr (sizeof(T) == 4) buf_store4(r, off, x);
        else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, __builtin_convertvector(x, T4)), r, off, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) buf_store<T>(r, i < n ? off + i * (int)sizeof(T) : kNowhere, (T)x[i]);
    }
}

// The row of tile i of a lower triangle, counted by rows: 0; 1, 1; 2, 2, 2; 3, ...
__device__ __forceinline__ int lin_tile_row(int i) { return i < 1 ? 0 : i < 3 ? 1 : i < 6 ? 2 : 3; }

// One part of one sequence and head, 64 NC columns: four waves of 16 NC columns each. REV:
// backward in time. DOT: with X.y. STATE: only the part's sum of B C^T. The next chunk's
// tiles are fetched into registers while this one is worked on.
template <typename T, int DP, int NC, bool REV, bool DOT, bool STATE>
__global__ __launch_bounds__(256, ElemPlanes<T>::n == 1 ? 2 : 1) void k_lin(LinShape d, LinPass a) {
    constexpr int P = ElemPlanes<T>::n, C = LinChunk<T>::n, NB = C / 32, NT = C / 16, NK = DP / 16, W = 64 * NC, E = (int)sizeof(T);
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
    const T* xp = DOT ? lin_at<T>(a.X, q.b, q.t0, h) + col_block * W : nullptr;
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
            double c = (double)lin_decay(fg) * 1.4426950408889634074;         // powers of two from here on
#pragma unroll
            for (int o = 1; o < C; o <<= 1) {
                const double y = __shfl_up(c, o);
                if (lane >= o) c += y;
            }
            const double end = __shfl(c, C - 1);
            if (lane < C) {
                s.c[lane] = c;
                const float in = exp2_of(c), out = exp2_of(end - c);
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
        const float decay = exp2_of(c_end);
        total += c_end;
        f32x4 y[NT][NC];       // y[t][c][r] is token 16 t + l16 of column 16 c + 4 (lane / 16) + r
        if constexpr (!STATE) {
            // P, made transposed: a lane has four neighbouring columns of one row
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
                    x[r] = (REV ? j >= i : j <= i) ? d.scale * exp2_of(gap) * acc[r] : 0.f;
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
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int c = 0; c < NC; c++) y[t][c] = {0, 0, 0, 0};
#pragma unroll
            for (int p = 0; p < DP / 32; p++) {
                Frag<3> f[NC];
                Frag<P> af[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) af[t] = A.frag(16 * t + l16, 32 * p, lane);
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    float x[8];
#pragma unroll
                    for (int r = 0; r < 4; r++) x[r] = S[c][2 * p][r], x[4 + r] = S[c][2 * p + 1][r];
                    f[c] = split8<3>(x);
                }
                mma_nm<3>(f, af, y);
            }
#pragma unroll
            for (int t = 0; t < NT; t++) {
                const float f = s.row[16 * t + l16];
#pragma unroll
                for (int c = 0; c < NC; c++) y[t][c] *= f;
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
        // what the dots take: X, and C of the token itself, whose share is added after them
        const int j4 = wave * 16 * NC + (lane >> 4) * 4;       // this lane's first column in C
        float xv[DOT ? NT : 1][NC][4];
        Frag<P> own[DOT ? NT : 1][NC];
        if constexpr (DOT) {
            const __amdgpu_buffer_rsrc_t r = rows_window(xp + t0 * a.X.st[1], a.X.st[1], n, cols);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const int j = j4 + 16 * c;
                    buf_load4e<T>(r, j < cols ? ((16 * t + l16) * (int)a.X.st[1] + j) * E : kNowhere, cols - j, a.vec, xv[t][c]);
                }
        }
        if constexpr (DOT) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int p = 0; p < P; p++)
                        *reinterpret_cast<bf16x4*>(&own[t][c].p[p]) = *reinterpret_cast<const bf16x4*>(Ct.at(p, 16 * t + l16, j4 + 16 * c));
        }
        barrier_lds();
        if (more) store();                     // only P is read from here on
        if constexpr (!STATE) {
#pragma unroll
            for (int jb = 0; jb < NB; jb++) {
#pragma unroll
                for (int t2 = 0; t2 < NT; t2 += 2) {
                    if (REV ? t2 > 2 * jb : t2 < 2 * jb) continue;
                    const Frag<3> pf[2] = {Pm.frag(16 * t2 + l16, 32 * jb, lane), Pm.frag(16 * t2 + 16 + l16, 32 * jb, lane)};
                    f32x4 o[2][NC];
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int c = 0; c < NC; c++) o[m][c] = y[t2 + m][c];
                    mma_nm<3>(cf[jb], pf, o);
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int c = 0; c < NC; c++) y[t2 + m][c] = o[m][c];
                }
            }
            if constexpr (DOT) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float w = sdiag[16 * t + l16];
                    float e = 0.f;
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        float o[4];
                        join4(own[t][c], o);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            e = fmaf(xv[t][c][r], y[t][c][r], e);
                            y[t][c][r] = fmaf(w, o[r], y[t][c][r]);
                        }
                    }
                    e += __shfl_xor(e, 16);
                    e += __shfl_xor(e, 32);
                    if (lane < 16 && 16 * t + lane < n)
                        a.dot[((int64_t)(row_block * 4 + wave) * d.H + h) * (d.B * d.T) + q.row + t0 + 16 * t + lane] = e;
                }
            }
            const int64_t HY = d.H / a.y_rep, row = q.row + t0;
            const int64_t slice = a.y_f32 ? ((int64_t)row_block * a.y_rep + h % a.y_rep) * (d.B * d.T) : 0;
            const int64_t step = HY * a.cols, at = ((slice + row) * HY + h / a.y_rep) * a.cols + col_block * W;
            auto put = [&](auto zero) {
                typedef decltype(zero) U;
                const __amdgpu_buffer_rsrc_t ry = rows_window(static_cast<const U*>(a.y) + at, step, n, cols);
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        const int j = j4 + 16 * c;
                        const int off = j < cols ? ((16 * t + l16) * (int)step + j) * (int)sizeof(U) : kNowhere;
                        buf_store4e<U>(ry, off, cols - j, a.y_vec, y[t][c]);
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
        if (tid == 0 && blockIdx.z == 0) a.decay[(int64_t)blockIdx.x * d.H + h] = exp2_of(total);
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
