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

// Running sums over lanes: within rows of 16 by shifts, then the rows before.
template <int CTRL> __device__ __forceinline__ double add_shifted(double x) {
    const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, 0xf, 0xf, true),
              hi = __builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, 0xf, 0xf, true);
    return x + __hiloint2double(hi, lo);
}
__device__ __forceinline__ double lane_value(double x, int l) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), l), __builtin_amdgcn_readlane(__double2loint(x), l));
}
__device__ __forceinline__ double running_sum(double x, int lane) {
    x = add_shifted<0x111>(x);
    x = add_shifted<0x112>(x);
    x = add_shifted<0x114>(x);
    x = add_shifted<0x118>(x);
    const double a = lane_value(x, 15), b = a + lane_value(x, 31), c = b + lane_value(x, 47);
    return x + (lane < 16 ? 0. : lane < 32 ? a : lane < 48 ? b : c);
}

// A tile of P planes of R rows and C columns in LDS without padding (planes.h has one with):
// the 16-byte units of a row are permuted by an exclusive or with bits of the row, chosen so
// that both ways of reading spread over the banks. The 16 rows of a frag meet 16 different
// units, and the four rows that a transposing read takes at once lie four units apart.
template <int P, int R, int C> struct SwTile {
    static constexpr int elems = P * R * C, U = C / 8, G = 16 / U;         // units of a row, rows of 256 bytes
    static_assert(U == 16 || U == 8 || U == 4);
    __bf16* s;
    static __device__ __forceinline__ int mix(int r) {
        const int x = r / G;
        return U == 16 ? (x & 3) << 2 | (x >> 2 & 3) : U == 8 ? (x & 1) << 2 | (x >> 1 & 3) : x & 3;
    }
    __device__ __forceinline__ __bf16* at(int p, int r, int c) const {
        return s + (p * R + r) * C + (((c >> 3) ^ mix(r)) << 3) + (c & 7);
    }
    // Row r0 + lane % 16 (r0 a multiple of 16), columns c0..c0 + 31 as the contraction.
    __device__ __forceinline__ Frag<P> frag(int r0, int c0, int lane) const {
        Frag<P> f;
#pragma unroll
        for (int p = 0; p < P; p++)
            f.p[p] = *reinterpret_cast<const bf16x8*>(s + (p * R + r0) * C + (lane & 15) * C +
                                                      (((c0 >> 3) + (lane >> 4)) ^ mix(lane & 15)) * 8);
        return f;
    }
    // Rows r0..r0 + 31 as the contraction (r0 a multiple of 32); the lane fetches its row's
    // four columns from `block` on, see planes.h.
    __device__ __forceinline__ Frag<P> tfrag(int r0, int block, int lane) const {
        Frag<P> f;
        const int r = 8 * (lane >> 4) + ((lane >> 2) & 3), u = block >> 3, e = block & 7;
#pragma unroll
        for (int p = 0; p < P; p++) {
            const bf16x4 lo = Tile<P, R, C>::tread(s + (p * R + r0) * C + r * C + (u ^ mix(r)) * 8 + e),
                         hi = Tile<P, R, C>::tread(s + (p * R + r0 + 4) * C + r * C + (u ^ mix(r + 4)) * 8 + e);
            f.p[p] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return f;
    }
    __device__ __forceinline__ void put8(int r, int c, const Frag<P>& f) const {
#pragma unroll
        for (int p = 0; p < P; p++) *reinterpret_cast<bf16x8*>(at(p, r, c)) = f.p[p];
    }
};

// An (R, W) tile of a (tokens, columns) array on its way from memory to LDS, held by NTH
// threads: tokens from n on and columns from `cols` on are 0 (a stride below `cols` would let
// the window alone hand out other rows).
template <typename T, int R, int W, int NTH> struct LinFetch {
    static constexpr int N = R * W / 8 / NTH;
    static_assert(R * W / 8 % NTH == 0);
    Vec8<T> x[N];
    __device__ __forceinline__ void load(const T* src, int64_t stride, int n, int cols, bool vec, int tid) {
        const __amdgpu_buffer_rsrc_t r = rows_window(src, stride, n, cols);
        const int step = (int)stride;
        if (vec) {
            const int t0 = tid / (W / 8), c = tid % (W / 8) * 8, off = (t0 * step + c) * (int)sizeof(T);
            constexpr int more = NTH / (W / 8);            // rows from one vector of a thread to the next
#pragma unroll
            for (int j = 0; j < N; j++)
                x[j] = buf_load8<T>(r, t0 + j * more < n && c < cols ? off + j * more * step * (int)sizeof(T) : kNowhere, 8, true);
        } else {
#pragma unroll
            for (int j = 0; j < N; j++) {
                const int i = here(tid) + j * NTH, t = i / (W / 8), c = i % (W / 8) * 8;
                x[j] = buf_load8<T>(r, (t * step + c) * (int)sizeof(T), t < n ? cols - c : 0, false);
            }
        }
    }
    template <typename Tl> __device__ __forceinline__ void store(Tl to, int tid) const {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = tid + j * NTH;
            to.put8(i / (W / 8), i % (W / 8) * 8, split_raw8<T>(x[j]));
        }
    }
};

__device__ __forceinline__ float exp2_of(double x) { return __builtin_amdgcn_exp2f((float)x); }

// Value e of a fragment, its planes added from the smallest.
template <int P> __device__ __forceinline__ float value_of(const Frag<P>& f, int e) {
    float x = (float)f.p[P - 1][e];
#pragma unroll
    for (int p = P - 2; p >= 0; p--) x += (float)f.p[p][e];
    return x;
}
// Values e and e + 1 of a fragment: eight bits a plane by truncation, which makes three planes
// exact, and the bits of a plane one instruction's to pack (a rounding one takes longer).
__device__ __forceinline__ void split2(float x, float y, Frag<3>& f, int e) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    unsigned u = __float_as_uint(x), v = __float_as_uint(y);
#pragma unroll
    for (int p = 0; p < 3; p++) {
        const bf16x2 h = __builtin_bit_cast(bf16x2, __builtin_amdgcn_perm(v, u, 0x07060302));
        f.p[p][e] = h[0];
        f.p[p][e + 1] = h[1];
        u = __float_as_uint(__uint_as_float(u) - __uint_as_float(u & 0xffff0000u));
        v = __float_as_uint(__uint_as_float(v) - __uint_as_float(v & 0xffff0000u));
    }
}
// f(plane of three, plane of the other) for the plane pairs of a product of fp32 precision
// (planes.h), the smallest first.
template <int PAIRS, typename F> __device__ __forceinline__ void each_product(F f) {
    constexpr int P = PAIRS == 3 ? 1 : PAIRS == 5 ? 2 : 3;
#pragma unroll
    for (int s = 2; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (s - i >= 0 && s - i < P) f(i, s - i);
}

// Spreads `steps` steps evenly over `all` products, also where the numbers do not divide: whether
// one is due after product m, and which. Each is, once, in order.
constexpr bool lin_due(int m, int all, int steps) { return (m + 1) * steps / all > m * steps / all; }
constexpr int lin_step_at(int m, int all, int steps) { return m * steps / all; }

// Four neighbouring elements from `off`, of which the first n exist. vec: aligned, all exist.
template <typename T> struct Vec4 { typedef T type __attribute__((ext_vector_type(4))); };
template <typename T> __device__ __forceinline__ typename Vec4<T>::type buf_load4e(__amdgpu_buffer_rsrc_t r, int off, int n, bool vec) {
    typedef typename Vec4<T>::type T4;
    if (vec) {
        if constexpr (sizeof(T) == 4) return buf_load4(r, off);
        else return __builtin_bit_cast(T4, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
    }
    T4 x;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = buf_load<T>(r, i < n ? off + i * (int)sizeof(T) : kNowhere);
    return x;
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
// backward in time. DOT: with X.y, and S transposed, its rows V's (dq, dk). STATE: only the
// part's sum of B C^T. The next chunk's tiles are fetched into registers while this one is
// worked on, two barriers a chunk.
//
// Bound first by the issue of matrix and vector instructions, which do not run side by side on
// this card (two waves on a SIMD take 65 ns each for 8 v_mfma_f32_16x16x32, 49 for 40
// v_sub_f32, and 124 for both in turn): a wave and chunk of 64 bf16 tokens and 128 x 32 of S is
// 240 matrix and about 1,280 vector instructions, half of them splitting S and C times its
// weight into planes. 8 x 2048 tokens, 16 heads of 128 in bf16, in 512 parts: 102 us for the
// output and for dv, 120 for dq and for dk with their dots, 47 for the parts' sums. Of the
// output's 102, 61 are that issue, about 22 waits for LDS, barriers and the fetch (a quarter of
// the waves' time by the counters), the rest starts and ends. Its 314 MB would take 62 by
// themselves. A chunk of 64 takes S apart half as often as one of 32,
// but has to leave LDS for a second block on the CU, without which every wait stands (fp16,
// 8 x 2048 tokens: 237 us with 64, 189 with 32; fp32, chunks of 32, held to the registers of
// two blocks: 318 -> 270). Two column tiles a wave halve the LDS reads and P's share (8 waves
// of 16 columns: 155 us).
template <typename T, int DP, int NC, bool REV, bool DOT, bool STATE>
__global__ __launch_bounds__(256, 2) void k_lin(LinShape d, LinPass a) {
    constexpr int P = ElemPlanes<T>::n, C = P == 1 || (P == 2 && STATE) ? 64 : 32, NB = C / 32, NT = C / 16,
                  NK = DP / 16, NW = kLinWaves, W = 64 * NC, PAIRS = P == 1 ? 3 : P == 2 ? 5 : 6, NTH = 256, E = (int)sizeof(T);
    // With five or six partial products they are summed before S takes them up, by one rounding
    // with the decay. Each added to S by itself left 17 2^-24 (rms, fp32) after 128 chunks
    // without a decay, this 3.7, for 1 to 2 % of the time. bf16's three, in chunks twice as long,
    // leave 6.6 there; their sums would spill.
    constexpr bool APART = P > 1;
    typedef SwTile<P, C, DP> Rows;
    typedef SwTile<P, C, W> Cols;
    typedef SwTile<3, C, C> Mat;
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
    f32x4 S[NC][NK];       // S[c][2 p + e][r] is row 32 p + g8 + 4 e + r of column 16 c + l16
    const int64_t kv = d.K * d.V;
    const int rs = (DOT ? 1 : (int)d.V) * 4, cs = (DOT ? (int)d.V : 1) * 4;
    auto each_state = [&](auto f) {
        const int g = here(g8), j0 = c0 + here(l16);
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int j = j0 + 16 * c, at = (r0 + g) * rs + j * cs;
#pragma unroll
            for (int kt = 0; kt < NK; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int i = (kt >> 1) * 32 + 4 * (kt & 1) + r;
                    f(S[c][kt], r, g + i < rows && j < a.cols ? at + i * rs : kNowhere);
                }
        }
    };
    auto state_at = [&](const float* p, int64_t n) {
        return make_rsrc(p ? p + (n * d.H + h) * kv : nullptr, p ? (uint32_t)kv * 4u : 0u);
    };
    {
        const float* const from = STATE ? nullptr : first_run ? a.begin : a.parts;
        const __amdgpu_buffer_rsrc_t st = state_at(from, first_run ? seq : (int64_t)blockIdx.x);
        if (DOT && d.V % 4 == 0) {             // four rows lie next to each other: 128 -> 120 us
            each_state([&](f32x4& x, int r, int at) { if (r == 0) x = buf_load4(st, at); });
        } else {
            each_state([&](f32x4& x, int r, int at) { x[r] = buf_load<float>(st, at); });
        }
    }
    LinFetch<T, C, DP, NTH> fa, fb;
    LinFetch<T, C, W, NTH> fc;
    float fg = 0.f;
    const T* ap = STATE ? nullptr : lin_at<T>(a.A, q.b, q.t0, h) + r0;
    const T* bp = lin_at<T>(a.B, q.b, q.t0, h) + r0;
    const T* cp = lin_at<T>(a.C, q.b, q.t0, h) + col_block * W;
    const T* xp = DOT ? lin_at<T>(a.X, q.b, q.t0, h) + col_block * W : nullptr;
    // rows of y lie `step` elements apart, the sequence's first at y_at
    const int step = (int)(d.H / a.y_rep) * a.cols;
    const int64_t slice = a.y_f32 ? ((int64_t)row_block * a.y_rep + h % a.y_rep) * (d.B * d.T) : 0;
    const int64_t y_at = (slice + q.row) * step + h / a.y_rep * a.cols + col_block * W;
    auto fetch = [&](int t0) {
        const int n = q.len - t0 < C ? q.len - t0 : C, tid = here((int)threadIdx.x), lane = tid & 63;
        if (!STATE) fa.load(ap + t0 * a.A.st[1], a.A.st[1], n, rows, a.vec, tid);
        fb.load(bp + t0 * a.B.st[1], a.B.st[1], n, rows, a.vec, tid);
        fc.load(cp + t0 * a.C.st[1], a.C.st[1], n, cols, a.vec, tid);
        if (wave == 0) fg = lane < n ? d.g[d.head_g ? h : (q.row + t0 + lane) * d.H + h] : 0.f;
    };
    auto store = [&]() {
        const int tid = here((int)threadIdx.x), lane = tid & 63;
        if (!STATE) fa.store(A, tid);
        fb.store(Bt, tid);
        fc.store(Ct, tid);
        if (wave == 0) {
            // powers of two from here on
            const double c = running_sum(lane < C ? (double)lin_decay(fg) * 1.4426950408889634074 : 0., lane),
                         end = lane_value(c, C - 1);
            if (lane < C) {
                s.c[lane] = c;
                const float in = exp2_of(c), out = exp2_of(end - c);
                s.row[lane] = REV ? out : d.scale * in;
                s.upd[lane] = REV ? d.scale * in : out;
            }
        }
    };
    if constexpr (!STATE) {                    // the tiles beside the diagonal that products of 32 read
        for (int i = tid; i < 3 * C * C / 8; i += NTH) {
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
        lane = here(lane);
        l16 = lane & 15;
        g8 = (lane >> 4) * 8;
        const double c_end = s.c[C - 1];
        const float decay = exp2_of(c_end);
        total += c_end;
        f32x4 y[NT][NC];       // y[t][c][r] is token 16 t + l16 of column 16 c + 4 (lane / 16) + r
        Frag<P> cf[NB][NC];    // C by columns, and its rows times the weights, which S takes up
        Frag<3> u[2][NC];
        constexpr int STEPS = 4 * NC;          // pairs of values of a step's operands
        auto columns_of = [&](int b) {
#pragma unroll
            for (int c = 0; c < NC; c++) cf[b][c] = Ct.tfrag(32 * b, wave * 16 * NC + 16 * c + 4 * (lane & 3), lane);
        };
        auto weigh = [&](int b, int i) {       // pair i of the operand
            const int c = i >> 2, e = 2 * (i & 3);
            const float2 w = *reinterpret_cast<const float2*>(&s.upd[32 * b + g8 + e]);
            split2(value_of(cf[b][c], e) * w.x, value_of(cf[b][c], e + 1) * w.y, u[b & 1][c], e);
        };
        if constexpr (!STATE) {
            // P, made transposed: a lane has four neighbouring columns of one row. A wave makes
            // every fourth tile; where there is none left, the last once more (the same values).
            constexpr int TILES = NT * (NT + 1) / 2;
#pragma unroll
            for (int k = 0; k < TILES; k += NW) {
                const int t = wave + k < TILES ? wave + k : TILES - 1;
                const int hi = lin_tile_row(t), lo = t - hi * (hi + 1) / 2, ti = REV ? lo : hi, tj = REV ? hi : lo;
                const int i = 16 * ti + l16, j0 = 16 * tj + (lane >> 4) * 4;
                f32x4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < DP; p += 32) acc = mma<3>(Bt.frag(16 * tj, p, lane), A.frag(16 * ti, p, lane), acc);
                const double ci_ = s.c[i];
                double cj[4];
#pragma unroll
                for (int r = 0; r < 4; r++) cj[r] = s.c[j0 + r];
                float x[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float w = d.scale * exp2_of(REV ? cj[r] - ci_ : ci_ - cj[r]) * acc[r];
                    x[r] = (REV ? j0 + r >= i : j0 + r <= i) ? w : 0.f;
                    if (DOT && j0 + r == i) {
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
            // Written in the order in which it is to run: the next step's operands are made
            // between this step's products.
            Frag<3> f[2][NC];
            Frag<P> af[2][NT];
            auto rows_of_a = [&](int p) {
#pragma unroll
                for (int t = 0; t < NT; t++) af[p & 1][t] = A.frag(16 * t, 32 * p, lane);
            };
            auto planes_of = [&](int p, int i) {
                const int c = i >> 2, e = 2 * (i & 3);
                const f32x4& x = S[c][2 * p + (e >> 2)];
                split2(x[e & 3], x[(e & 3) + 1], f[p & 1][c], e);
            };
            rows_of_a(0);
#pragma unroll
            for (int i = 0; i < STEPS; i++) planes_of(0, i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < DP / 32; p++) {
                if (p + 1 < DP / 32) rows_of_a(p + 1);
                else columns_of(0);
                int m = 0;
                each_product<PAIRS>([&](int i, int j) {
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int c = 0; c < NC; c++) {
                            y[t][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[p & 1][c].p[i], af[p & 1][t].p[j], y[t][c], 0, 0, 0);
                            constexpr int all = PAIRS * NT * NC;
                            static_assert(all >= STEPS);
                            if (lin_due(m, all, STEPS)) {
                                const int made = lin_step_at(m, all, STEPS);
                                if (p + 1 < DP / 32) planes_of(p + 1, made);
                                else weigh(0, made);
                                __builtin_amdgcn_sched_barrier(0);
                            }
                            m++;
                        }
                });
            }
        } else {
            columns_of(0);
#pragma unroll
            for (int i = 0; i < STEPS; i++) weigh(0, i);
        }
        if (more && !DOT) fetch(chunk_at(ci + 1));
        Frag<P> bf[2][2];
        auto columns_of_b = [&](int i) {       // step i: 32 rows of S, of 32 tokens
            const int b = i / (NK / 2), k2 = i % (NK / 2) * 2;
#pragma unroll
            for (int e = 0; e < 2; e++) bf[i & 1][e] = Bt.tfrag(32 * b, 16 * k2 + 8 * (lane & 3) + 4 * e, lane);
        };
        columns_of_b(0);             // with the dots' registers a step ahead is too much
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if (b + 1 < NB) columns_of(b + 1);
            else if (DOT && more) fetch(chunk_at(ci + 1));         // later: one of them would spill (134 -> 128 us)
            int m = 0;
#pragma unroll
            for (int k = 0; k < NK / 2; k++) {
                const int i = b * (NK / 2) + k;
                if (i + 1 < NB * NK / 2) columns_of_b(i + 1);
                f32x4 sum[2][NC];
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        if (APART && b == 0) sum[e][c] = {0, 0, 0, 0};
                        else if (b == 0) S[c][2 * k + e] *= decay;
                    }
                each_product<PAIRS>([&](int pj, int pi) {          // u's plane pj, B's pi
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int c = 0; c < NC; c++) {
                            f32x4& x = APART && b == 0 ? sum[e][c] : S[c][2 * k + e];
                            x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf[i & 1][e].p[pi], u[b & 1][c].p[pj], x, 0, 0, 0);
                            constexpr int all = PAIRS * NK * NC;
                            static_assert(all >= STEPS && NT <= STEPS);
                            if (lin_due(m, all, STEPS)) {
                                const int made = lin_step_at(m, all, STEPS);
                                if (b + 1 < NB) weigh(b + 1, made);
                                else if constexpr (!STATE)
                                    if (made < NT) {
                                        const float r = s.row[16 * made + l16];
#pragma unroll
                                        for (int q = 0; q < NC; q++) y[made][q] *= r;
                                    }
                                __builtin_amdgcn_sched_barrier(0);
                            }
                            m++;
                        }
                });
                if (APART && b == 0)
#pragma unroll
                    for (int e = 0; e < 2; e++)
#pragma unroll
                        for (int c = 0; c < NC; c++) {
                            f32x4& x = S[c][2 * k + e];
#pragma unroll
                            for (int r = 0; r < 4; r++) x[r] = fmaf(x[r], decay, sum[e][c][r]);
                            asm volatile("" : "+v"(x));        // here, not at the chunk's end with all sums held (spills)
                        }
            }
        }
        const int j4 = wave * 16 * NC + (lane >> 4) * 4;       // this lane's first column in C
        typename Vec4<T>::type xv[DOT ? NT : 1][NC];
        if constexpr (DOT) {
            const __amdgpu_buffer_rsrc_t r = rows_window(xp + t0 * a.X.st[1], a.X.st[1], n, cols);
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const int j = j4 + 16 * c;
                    xv[t][c] = buf_load4e<T>(r, j < cols ? ((16 * t + l16) * (int)a.X.st[1] + j) * E : kNowhere, cols - j, a.vec);
                }
        }
        Frag<P> own[DOT ? NT : 1][NC];         // C of the token itself, whose share is added after the dots
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
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!STATE) {
#pragma unroll
            for (int jb = 0; jb < NB; jb++)
#pragma unroll
                for (int t2 = 0; t2 < NT; t2 += 2) {
                    if (REV ? t2 > 2 * jb : t2 < 2 * jb) continue;
                    const Frag<3> pf[2] = {Pm.frag(16 * t2, 32 * jb, lane), Pm.frag(16 * t2 + 16, 32 * jb, lane)};
                    each_product<PAIRS>([&](int pj, int pi) {      // P's plane pj, C's pi
#pragma unroll
                        for (int m = 0; m < 2; m++)
#pragma unroll
                            for (int c = 0; c < NC; c++)
                                y[t2 + m][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(cf[jb][c].p[pi], pf[m].p[pj], y[t2 + m][c], 0, 0, 0);
                    });
                }
            if constexpr (DOT) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const float w = sdiag[16 * t + l16];
                    float e = 0.f;
#pragma unroll
                    for (int c = 0; c < NC; c++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            e = fmaf((float)xv[t][c][r], y[t][c][r], e);
                            y[t][c][r] = fmaf(w, value_of(own[t][c], r), y[t][c][r]);
                        }
                    e += __shfl_xor(e, 16);
                    e += __shfl_xor(e, 32);
                    if (lane < 16 && 16 * t + lane < n)
                        a.dot[((int64_t)((row_block * ncol + col_block) * NW + wave) * d.H + h) * (d.B * d.T) + q.row + t0 + 16 * t + lane] = e;
                }
            }
            const int64_t at = y_at + t0 * (int64_t)step;
            auto put = [&](auto zero) {
                typedef decltype(zero) U;
                const __amdgpu_buffer_rsrc_t ry = rows_window(static_cast<const U*>(a.y) + at, step, n, cols);
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const int j = j4 + 16 * c, off = j < cols ? (l16 * step + j) * (int)sizeof(U) : kNowhere;
#pragma unroll
                    for (int t = 0; t < NT; t++)           // what is added to kNowhere stays outside
                        buf_store4e<U>(ry, off + 16 * t * step * (int)sizeof(U), cols - j, a.y_vec, y[t][c]);
                }
            };
            if (a.y_f32) put(0.f);
            else put(T(0.f));
        }
        barrier_lds();
    }
    if (STATE || (last_run && a.end)) {
        const __amdgpu_buffer_rsrc_t st = state_at(STATE ? a.parts : a.end, STATE ? (int64_t)blockIdx.x : seq);
        each_state([&](f32x4& x, int r, int at) { buf_store<float>(st, at, x[r]); });
    }
    if (STATE && tid == 0 && blockIdx.z == 0) a.decay[(int64_t)blockIdx.x * d.H + h] = exp2_of(total);
}

template <typename T> snhip_status lin_run(const LinShape& d, const LinPass& a, bool rev, int kind, hipStream_t st) {
    auto go = [&](auto dp, auto nc, auto back, auto dot, auto state) -> snhip_status {
        constexpr int NC = decltype(nc)::value;
        const int64_t z = (int64_t)((a.cols + 64 * NC - 1) / (64 * NC)) * ((a.rows + kLinRows - 1) / kLinRows);
        const dim3 grid((unsigned)d.slots, (unsigned)d.H, (unsigned)z);
        k_lin<T, decltype(dp)::value, NC, decltype(back)::value, decltype(dot)::value, decltype(state)::value>
            <<<grid, 256, 0, st>>>(d, a);
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
    auto by_cols = [&](auto dp) { return a.cols <= 64 || d.narrow ? by_dir(dp, one()) : by_dir(dp, two()); };
    return a.rows <= 64 ? by_cols(std::integral_constant<int, 64>()) : by_cols(std::integral_constant<int, 128>());
}

}  // namespace
}  // namespace snhip
