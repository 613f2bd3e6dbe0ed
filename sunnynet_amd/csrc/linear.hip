// Linear attention with a decay for each head: the token-by-token form, the small kernels
// around the recurrence (linscan.h), and the C entry points. Mathematics: linear.h.
#include <type_traits>

#include "linear.h"

namespace snhip {
namespace {

// Token by token. A wave owns 32 columns of V of one sequence and head: lane (kg, vg)
// holds rows kg RPT .. + RPT - 1 and four columns, all in registers from one read of the
// state to one write, every read on its way before the first is used. Bound by the state's
// bytes: 22.7 us (5.9 TB/s) for 64 sequences of 16 heads of 128; for one sequence by latency.
// FOUR: V is a multiple of four.
template <typename T, int RPT, bool FOUR>
__global__ __launch_bounds__(64) void k_lin_step(LinShape d, LinRows q, LinRows k, LinRows v, bool vec, T* out,
                                                 const float* s0, float* send) {
    const int h = blockIdx.y, lane = threadIdx.x, kg = lane >> 3, k0 = kg * RPT, E = (int)sizeof(T);
    const int V = (int)d.V, Kd = (int)d.K, v0 = blockIdx.x * 32 + (lane & 7) * 4;
    const int64_t n = blockIdx.z, row = n * d.T, base = (n * d.H + h) * d.K * d.V;
    Vec8<T> nq[RPT / 8], nk[RPT / 8];
    unsigned nv[4];
    float ng;
    auto fetch = [&](int t) {
        const __amdgpu_buffer_rsrc_t rq = rows_window(lin_at<T>(q, n, t, h), 0, 1, Kd),
                                     rk = rows_window(lin_at<T>(k, n, t, h), 0, 1, Kd),
                                     rv = rows_window(lin_at<T>(v, n, t, h), 0, 1, V);
        ng = d.g[d.head_g ? h : (row + t) * d.H + h];
#pragma unroll
        for (int i = 0; i < RPT / 8; i++) {
            nq[i] = buf_load8<T>(rq, (k0 + 8 * i) * E, Kd - k0 - 8 * i, vec);
            nk[i] = buf_load8<T>(rk, (k0 + 8 * i) * E, Kd - k0 - 8 * i, vec);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) nv[j] = buf_load_bits<T>(rv, (v0 + j) * E);
    };
    if (d.T > 0) fetch(0);
    // rows from K on lie past the state's bytes, and read as 0; so does a state that is not there
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(s0 ? s0 + base : nullptr, s0 ? (uint32_t)(Kd * V * 4) : 0u);
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
    for (int t = 0; t < (int)d.T; t++) {
        float qf[RPT], kf[RPT], vv[4];
#pragma unroll
        for (int i = 0; i < RPT; i++) qf[i] = (float)nq[i / 8][i % 8], kf[i] = (float)nk[i / 8][i % 8];
#pragma unroll
        for (int j = 0; j < 4; j++) vv[j] = float_of_bits<T>(nv[j]);
        const float al = expf(lin_decay(ng));
        if (t + 1 < (int)d.T) fetch(t + 1);
        f32x4 o = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < RPT; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                S[i][j] = fmaf(kf[i], vv[j], al * S[i][j]);
                o[j] = fmaf(S[i][j], qf[i], o[j]);
            }
#pragma unroll
        for (int l = 8; l < 64; l <<= 1)
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] += __shfl_xor(o[j], l);
        const __amdgpu_buffer_rsrc_t ro = rows_window(out + ((row + t) * d.H + h) * (int64_t)V, 0, 1, V);
#pragma unroll
        for (int j = 0; j < 4; j++) buf_store<T>(ro, kg == 0 ? (v0 + j) * E : kNowhere, (T)(d.scale * o[j]));
    }
    if (!send) return;
    const __amdgpu_buffer_rsrc_t rt = make_rsrc(send + base, (uint32_t)(Kd * V * 4));
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

// Joins the parts of a sequence, a thread per element of the state, or four of them: the parts' own sums
// become the states that they begin with (REV: end with, from the last part back). Bound by
// memory: 12.5 us for 3 of 4 parts of 8 x 16 states of 128 x 128 (4.7 TB/s).
template <typename F, bool REV>
__global__ __launch_bounds__(256) void k_lin_join(LinShape d, float* all, const float* decay, const float* begin) {
    const int64_t kv = d.K * d.V / (sizeof(F) / 4), i = blockIdx.x * (int64_t)256 + threadIdx.x, h = blockIdx.y, seq = blockIdx.z;
    if (i >= kv) return;
    F* const parts = reinterpret_cast<F*>(all);
    const LinSeq s = lin_seq(d, seq);
    const int np = (s.len + d.part - 1) / d.part;
    F run = {};
    if (begin) run = reinterpret_cast<const F*>(begin)[(seq * d.H + h) * kv + i];
    auto slot = [&](int p) { return (s.slot + (REV ? np - 1 - p : p)) * d.H + h; };
    constexpr int U = 8;                       // steps whose reads are on their way at once
    F own[U + 1] = {};
    if (np > 1) own[0] = parts[slot(0) * kv + i];
    for (int p0 = 0; p0 + 1 < np; p0 += U) {
        float a[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (p0 + u + 1 < np) a[u] = decay[slot(p0 + u)];
            if (p0 + u + 2 < np) own[u + 1] = parts[slot(p0 + u + 1) * kv + i];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (p0 + u + 1 >= np) continue;
            run = run * a[u] + own[u];
            parts[slot(p0 + u + 1) * kv + i] = run;
        }
        own[0] = own[U];
    }
}

// The decay's gradient over one part and head: e_t = q_t.dq_t - k_t.dk_t summed from the
// part's last token back, from <S, R> at its end. Sums in 64 bits. dg: (B,T,H), or the
// part's total in `sums` (slots, H). Waits for its reads, the two states before any token: 22 us
// for 8 x 4 parts, 16 heads of 128 x 128 (3.4 TB/s; its waves wait 77 % of their time).
__global__ __launch_bounds__(256) void k_lin_dg(LinShape d, const float* dots, int waves, const float* s_parts, const float* r_parts,
                                                const float* send, const float* dsend, float* dg, double* sums) {
    __shared__ double sw[4];
    const int h = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t kv = d.K * d.V, all = d.B * d.T;
    LinSeq s;
    int64_t seq;
    int part;
    if (!lin_part_of(d, blockIdx.x, &s, &seq, &part)) {
        if (d.head_g && tid == 0) sums[blockIdx.x * d.H + h] = 0.;
        return;
    }
    const int begin = part * d.part;
    const bool last = begin + d.part >= s.len;
    const int stop = last ? s.len : begin + d.part;
    const float* x = last ? (dsend ? send + (seq * d.H + h) * kv : nullptr) : s_parts + ((blockIdx.x + 1) * d.H + h) * kv;
    const float* y = last ? (dsend ? dsend + (seq * d.H + h) * kv : nullptr) : r_parts + (blockIdx.x * d.H + h) * kv;
    auto block_sum = [&](double v) {
        for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
        __syncthreads();
        if (lane == 0) sw[wave] = v;
        __syncthreads();
        return (sw[0] + sw[1]) + (sw[2] + sw[3]);
    };
    double carry = 0., total = 0.;
    if (x && kv % 4 == 0 && (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % 16 == 0) {
#pragma unroll 4
        for (int i = 4 * tid; i < (int)kv; i += 1024) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(x + i), b = *reinterpret_cast<const f32x4*>(y + i);
            carry += ((double)a[0] * b[0] + (double)a[1] * b[1]) + ((double)a[2] * b[2] + (double)a[3] * b[3]);
        }
    } else if (x) {
        for (int i = tid; i < (int)kv; i += 256) carry += (double)x[i] * (double)y[i];
    }
    carry = block_sum(carry);
    for (int t0 = stop; t0 > begin; t0 -= 256) {           // thread 0 the last token
        const int t = t0 - 1 - tid;
        double e = 0.;
        const int64_t row = (s.row + t) * d.H + h;
        if (t >= begin)
            for (int w = 0; w < waves; w++) {
                const float* x = dots + (w * d.H + h) * all + s.row + t;
                e += (double)x[0] - (double)x[waves * d.H * all];
            }
        for (int o = 1; o < 64; o <<= 1) {
            const double z = __shfl_up(e, o);
            if (lane >= o) e += z;
        }
        __syncthreads();
        if (lane == 63) sw[wave] = e;
        __syncthreads();
        double before = carry;
        for (int w = 0; w < wave; w++) before += sw[w];
        carry += (sw[0] + sw[1]) + (sw[2] + sw[3]);
        e += before;
        if (t >= begin) {
            total += e;
            if (!d.head_g) dg[row] = (float)e;
        }
    }
    if (d.head_g) {
        total = block_sum(total);
        if (tid == 0) sums[blockIdx.x * d.H + h] = total;
    }
}

__global__ __launch_bounds__(64) void k_lin_dg_heads(LinShape d, const double* sums, float* dg) {
    const int h = blockIdx.x;
    double v = 0.;
    for (int64_t i = threadIdx.x; i < d.slots; i += 64) v += sums[i * d.H + h];
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if (threadIdx.x == 0) dg[h] = (float)v;
}

// Adds `count` fp32 slices of n values, in order, and rounds.
template <typename T> __global__ __launch_bounds__(256) void k_lin_add(const float* x, T* y, int64_t n, int count, LinShape d, int64_t per) {
    for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < n; i += gridDim.x * (int64_t)256) {
        if (d.cu) {                            // rows of no sequence were not written
            const int64_t t = i / per;
            if (t < lin_edge(d, 0) || t >= lin_edge(d, d.N)) continue;
        }
        float v = 0.f;
        for (int c = 0; c < count; c++) v += x[c * n + i];
        y[i] = (T)v;
    }
}

// Clears the rows of no sequence, before the first edge and from the last on, of up to four
// arrays. A launch of 2 us, where clearing whole arrays first took 4 to 5 each.
struct LinClear {
    struct { char* p; int64_t row; } at[4];    // bytes of a row, an even number
};
__global__ __launch_bounds__(256) void k_lin_clear(LinShape d, LinClear c) {
    const int64_t first = lin_edge(d, 0), last = lin_edge(d, d.N), i0 = blockIdx.x * (int64_t)256 + threadIdx.x, n = gridDim.x * (int64_t)256;
    char* const p = c.at[blockIdx.y].p;
    const int64_t row = c.at[blockIdx.y].row;
    auto clear = [&](char* a, char* e) {
        char* const a16 = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(a) + 15) & ~(uintptr_t)15);
        char* const e16 = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(e) & ~(uintptr_t)15);
        if (a16 >= e16) {
            for (char* x = a + 2 * i0; x < e; x += 2 * n) *reinterpret_cast<short*>(x) = 0;
            return;
        }
        for (char* x = a + 2 * i0; x < a16; x += 2 * n) *reinterpret_cast<short*>(x) = 0;
        for (char* x = a16 + 16 * i0; x < e16; x += 16 * n) *reinterpret_cast<u32x4*>(x) = u32x4{};
        for (char* x = e16 + 2 * i0; x < e; x += 2 * n) *reinterpret_cast<short*>(x) = 0;
    };
    if (first > 0) clear(p, p + first * row);
    if (last < d.T) clear(p + last * row, p + d.T * row);
}
snhip_status lin_clear(const LinShape& s, const LinClear& c, int arrays, hipStream_t st) {
    k_lin_clear<<<dim3((unsigned)(s.T < 64 ? 1 : s.T / 64 < 256 ? s.T / 64 : 256), (unsigned)arrays), 256, 0, st>>>(s, c);
    SNHIP_CHECK(hipGetLastError());
    return SNHIP_OK;
}

bool lin_in_range(const SnHipLinear& d) {
    return d.B >= 1 && d.T >= 1 && d.N >= 1 && d.N <= 65535 && d.H >= 1 && d.H <= 65535 && d.Hk >= 1 &&
           d.H % d.Hk == 0 && d.K >= 1 && d.K <= 128 && d.V >= 1 && d.V <= 4096 && d.T <= kLinTokens / d.B &&
           (d.cu ? d.B == 1 : d.N == d.B) && d.H * d.V < kLinStride / 2 && d.H * d.K < kLinStride / 2 &&
           d.dtype >= SNHIP_F32 && d.dtype <= SNHIP_F16;
}

// Blocks that fill the card: two a CU, or three where K and V are at most 64 (16 x 1024 tokens
// of 16 heads of 64 in bf16: 66 us and 61), and not one more: a few blocks in a second round
// take as long as all (the output of 16384 tokens of 12 heads of 128, bf16: 96 us in 516
// blocks, 77 in 444). And the fewest tokens worth a part: 3 x 333 tokens of 5 heads, all kernels of a
// training pass, 100 us with 64, 133 with 128, 210 with 256.
constexpr int64_t kLinBlocks = 512, kLinSmall = 768, kLinPart = 64;

void lin_shape(const SnHipLinear& d, LinShape* s) {
    const int64_t tokens = d.B * d.T;
    // Blocks of 64 columns where even the shortest parts leave CUs idle: 16 us less of those 100.
    s->narrow = tokens * d.H * ((d.V + 127) / 128) / kLinPart < 256;
    const int64_t blocks = d.H * (s->narrow ? (d.V + 63) / 64 : (d.V + 127) / 128);
    const int64_t fit = (d.K <= 64 && d.V <= 64 ? kLinSmall : kLinBlocks) / (blocks * d.B), parts = fit < 1 ? 1 : fit;
    int64_t part = (d.T + parts - 1) / parts;
    part = ((part < kLinPart ? kLinPart : part) + 63) / 64 * 64;
    if (part > d.T) part = (d.T + 63) / 64 * 64;
    s->g = d.g;
    s->cu = d.cu;
    s->B = d.B, s->T = d.T, s->N = d.N, s->H = d.H, s->K = d.K, s->V = d.V;
    s->part = (int)part;
    s->per_seq = (int)((d.T + part - 1) / part);
    s->slots = d.cu ? d.T / part + d.N : d.B * s->per_seq;
    s->split = part < d.T;
    s->head_g = d.head_g != 0;
    s->scale = (float)d.scale;
}

int64_t parts_floats(const LinShape& s) { return s.split ? (s.slots * s.H * (s.K * s.V + 1) + 3) / 4 * 4 : 0; }

// The parts' sums of the decay's gradient, in 64 bits.
int64_t lin_sums_floats(const LinShape& s) { return (2 * s.slots * s.H + 3) / 4 * 4; }

// Slices of dq and dk: value heads that share a head, blocks of 128 columns of V.
int64_t lin_row_blocks(const SnHipLinear& d) { return (d.V + kLinRows - 1) / kLinRows; }
// Parts of a dot of X and y: waves of all blocks of K's columns, for each block of V's rows.
int64_t lin_dots(const SnHipLinear& d, const LinShape& s) {
    return kLinWaves * lin_row_blocks(d) * (s.narrow ? (d.K + 63) / 64 : 1);
}
int64_t lin_slices(const SnHipLinear& d) { return d.H / d.Hk * lin_row_blocks(d); }

bool aligned8(const void* p, const int64_t* st, int64_t cols, int64_t dtype) {
    const int64_t step = dtype == SNHIP_F32 ? 4 : 8;      // elements of 16 bytes
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && st[0] % step == 0 && st[1] % step == 0 && st[2] % step == 0 && cols % 8 == 0;
}

// Whether every four elements of rows of `cols` are aligned.
bool lin_four(const void* p, int64_t cols, int64_t dtype) {
    return cols % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (dtype == SNHIP_F32 ? 16 : 8) == 0;
}

LinRows rows_of(const void* p, const int64_t* st, int64_t rep) { return {p, {st[0], st[1], st[2]}, (int)rep}; }

snhip_status lin_run_any(const SnHipLinear& d, const LinShape& s, const LinPass& a, bool rev, int kind, hipStream_t st) {
    return d.dtype == SNHIP_F32    ? lin_run_f32(s, a, rev, kind, st)
           : d.dtype == SNHIP_BF16 ? lin_run_bf16(s, a, rev, kind, st)
                                   : lin_run_f16(s, a, rev, kind, st);
}

snhip_status lin_join(const LinShape& s, bool rev, float* parts, const float* begin, hipStream_t st) {
    const float* decay = parts + s.slots * s.H * s.K * s.V;
    const bool four = s.K * s.V % 4 == 0 && reinterpret_cast<uintptr_t>(begin) % 16 == 0;
    const dim3 grid((unsigned)((s.K * s.V / (four ? 4 : 1) + 255) / 256), (unsigned)s.H, (unsigned)s.N);
    if (four && rev) k_lin_join<f32x4, true><<<grid, 256, 0, st>>>(s, parts, decay, begin);
    else if (four) k_lin_join<f32x4, false><<<grid, 256, 0, st>>>(s, parts, decay, begin);
    else if (rev) k_lin_join<float, true><<<grid, 256, 0, st>>>(s, parts, decay, begin);
    else k_lin_join<float, false><<<grid, 256, 0, st>>>(s, parts, decay, begin);
    SNHIP_CHECK(hipGetLastError());
    return SNHIP_OK;
}

template <typename T>
snhip_status step_t(const SnHipLinear& d, const LinShape& s, void* out, float* send, hipStream_t st) {
    const int64_t rep = d.H / d.Hk;
    const LinRows q = rows_of(d.q, d.q_stride, rep), k = rows_of(d.k, d.k_stride, rep), v = rows_of(d.v, d.v_stride, 1);
    const bool vec = aligned8(d.q, d.q_stride, d.K, d.dtype) && aligned8(d.k, d.k_stride, d.K, d.dtype);
    const dim3 grid((unsigned)((d.V + 31) / 32), (unsigned)d.H, (unsigned)d.N);
    auto go = [&](auto rpt, auto four) {
        k_lin_step<T, decltype(rpt)::value, decltype(four)::value><<<grid, 64, 0, st>>>(s, q, k, v, vec, (T*)out, d.s0, send);
    };
    auto by_v = [&](auto rpt) { d.V % 4 == 0 ? go(rpt, std::true_type()) : go(rpt, std::false_type()); };
    if (d.K <= 64) by_v(std::integral_constant<int, 8>());
    else by_v(std::integral_constant<int, 16>());
    SNHIP_CHECK(hipGetLastError());
    return SNHIP_OK;
}

snhip_status lin_step(const SnHipLinear& d, const LinShape& s, void* out, float* send, hipStream_t st) {
    return d.dtype == SNHIP_F32    ? step_t<float>(d, s, out, send, st)
           : d.dtype == SNHIP_BF16 ? step_t<__bf16>(d, s, out, send, st)
                                   : step_t<_Float16>(d, s, out, send, st);
}

template <typename T> snhip_status add_t(const LinShape& s, const float* x, void* y, int64_t n, int64_t count, int64_t per, hipStream_t st) {
    const int64_t blocks = (n + 255) / 256;
    k_lin_add<T><<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, st>>>(x, (T*)y, n, (int)count, s, per);
    SNHIP_CHECK(hipGetLastError());
    return SNHIP_OK;
}

}  // namespace

// Checks d and derives the shape from it.
snhip_status lin_args(const SnHipLinear* d, LinShape* s) {
    if (!d || !d->q || !d->k || !d->v || !d->g || !lin_in_range(*d)) return SNHIP_E_INVAL;
    if (reinterpret_cast<uintptr_t>(d->parts) % 16) return SNHIP_E_INVAL;
    for (const int64_t* st : {d->q_stride, d->k_stride, d->v_stride})
        if (st[1] < 0 || st[1] >= kLinStride) return SNHIP_E_INVAL;
    lin_shape(*d, s);
    return SNHIP_OK;
}

}  // namespace snhip

using namespace snhip;

extern "C" {

int64_t snhip_op_linear_parts_floats(const SnHipLinear* d) {
    if (!d || !lin_in_range(*d)) return 0;
    LinShape s;
    lin_shape(*d, &s);
    return parts_floats(s);
}

int64_t snhip_op_linear_bwd_floats(const SnHipLinear* d) {
    if (!d || !lin_in_range(*d)) return 0;
    LinShape s;
    lin_shape(*d, &s);
    const int64_t tokens = d->B * d->T, slices = lin_slices(*d);
    return lin_sums_floats(s) + parts_floats(s) + 2 * lin_dots(*d, s) * tokens * d->H +
           (slices > 1 ? slices * tokens * d->Hk * d->K : 0);
}

snhip_status snhip_op_linear_step_dev(const SnHipLinear* d, void* out, float* send, void* stream) {
    LinShape s;
    if (lin_args(d, &s) != SNHIP_OK || d->cu || !out || !send) return SNHIP_E_INVAL;
    return lin_step(*d, s, out, send, as_stream(stream));
}

snhip_status snhip_op_linear_fwd_dev(const SnHipLinear* d, void* out, float* send, void* stream) {
    LinShape s;
    if (lin_args(d, &s) != SNHIP_OK || !out || (s.split && !d->parts)) return SNHIP_E_INVAL;
    const hipStream_t st = as_stream(stream);
    const int64_t rep = d->H / d->Hk;
    LinPass a = {};
    a.A = rows_of(d->q, d->q_stride, rep);
    a.B = rows_of(d->k, d->k_stride, rep);
    a.C = rows_of(d->v, d->v_stride, 1);
    a.rows = (int)d->K, a.cols = (int)d->V;
    a.vec = aligned8(d->q, d->q_stride, d->K, d->dtype) && aligned8(d->k, d->k_stride, d->K, d->dtype) &&
            aligned8(d->v, d->v_stride, d->V, d->dtype);
    a.begin = d->s0;
    a.end = send;
    a.parts = d->parts;
    a.decay = d->parts + s.slots * s.H * s.K * s.V;
    a.y = out;
    a.y_rep = 1;
    a.y_vec = lin_four(out, d->V, d->dtype);
    if (d->cu) {
        const snhip_status rc = lin_clear(s, {{{static_cast<char*>(out), d->H * d->V * (d->dtype == SNHIP_F32 ? 4 : 2)}}}, 1, st);
        if (rc != SNHIP_OK) return rc;
    }
    if (s.split) {
        snhip_status rc = lin_run_any(*d, s, a, false, 2, st);
        if (rc == SNHIP_OK) rc = lin_join(s, false, d->parts, d->s0, st);
        if (rc != SNHIP_OK) return rc;
    }
    return lin_run_any(*d, s, a, false, 0, st);
}

snhip_status snhip_op_linear_bwd_dev(const SnHipLinear* d, const SnHipLinearGrad* gr, void* stream) {
    LinShape s;
    if (lin_args(d, &s) != SNHIP_OK || !gr || !gr->dout || !gr->dq || !gr->dk || !gr->dv || !gr->dg || !gr->ws ||
        (gr->dsend && !gr->send) || (s.split && !d->parts) || reinterpret_cast<uintptr_t>(gr->ws) % 16)
        return SNHIP_E_INVAL;
    const hipStream_t st = as_stream(stream);
    const int64_t rep = d->H / d->Hk, tokens = d->B * d->T, slices = lin_slices(*d);
    double* const sums = reinterpret_cast<double*>(gr->ws);
    float* const parts = gr->ws + lin_sums_floats(s);
    float* const dots = parts + parts_floats(s);
    const int64_t waves = lin_dots(*d, s);
    float* const slice = dots + 2 * waves * tokens * d->H;
    const int64_t dout_st[3] = {d->T * d->H * d->V, d->H * d->V, d->V};
    const LinRows q = rows_of(d->q, d->q_stride, rep), k = rows_of(d->k, d->k_stride, rep), v = rows_of(d->v, d->v_stride, 1),
                  o = rows_of(gr->dout, dout_st, 1);
    const bool vec = aligned8(d->q, d->q_stride, d->K, d->dtype) && aligned8(d->k, d->k_stride, d->K, d->dtype) &&
                     aligned8(d->v, d->v_stride, d->V, d->dtype) && aligned8(gr->dout, dout_st, d->V, d->dtype);
    LinPass a = {};
    a.vec = vec;
    a.y_rep = 1;
    // dv and ds0, and the gradients of the parts' states
    a.A = k, a.B = q, a.C = o;
    a.rows = (int)d->K, a.cols = (int)d->V;
    a.begin = gr->dsend;
    a.end = gr->ds0;
    a.parts = parts;
    a.decay = parts + s.slots * s.H * s.K * s.V;
    a.y = gr->dv;
    a.y_vec = lin_four(gr->dv, d->V, d->dtype);
    snhip_status rc = SNHIP_OK;
    if (d->cu) {
        const int64_t e = d->dtype == SNHIP_F32 ? 4 : 2;
        rc = lin_clear(s, {{{static_cast<char*>(gr->dv), d->H * d->V * e}, {static_cast<char*>(gr->dq), d->Hk * d->K * e},
                            {static_cast<char*>(gr->dk), d->Hk * d->K * e}, {reinterpret_cast<char*>(gr->dg), d->H * 4}}},
                       s.head_g ? 3 : 4, st);
    }
    if (rc == SNHIP_OK && s.split) {
        rc = lin_run_any(*d, s, a, true, 2, st);
        if (rc == SNHIP_OK) rc = lin_join(s, true, parts, gr->dsend, st);
    }
    if (rc == SNHIP_OK) rc = lin_run_any(*d, s, a, true, 0, st);
    auto turned = [&](const LinRows& A, const LinRows& B, const LinRows& C, const LinRows& X, const float* begin, float* at,
                      float* dot, void* y, bool rev) {
        LinPass b = {};
        b.vec = vec;
        b.A = A, b.B = B, b.C = C, b.X = X;
        b.rows = (int)d->V, b.cols = (int)d->K;
        b.begin = begin;
        b.parts = at;
        b.y_rep = (int)rep;
        b.y_f32 = slices > 1;
        b.y = slices > 1 ? slice : y;
        b.y_vec = lin_four(b.y, d->K, slices > 1 ? SNHIP_F32 : d->dtype);
        b.dot = dot;
        snhip_status r = lin_run_any(*d, s, b, rev, 1, st);
        if (r != SNHIP_OK || slices == 1) return r;
        const int64_t n = tokens * d->Hk * d->K, per = d->Hk * d->K;
        return d->dtype == SNHIP_F32    ? add_t<float>(s, slice, y, n, slices, per, st)
               : d->dtype == SNHIP_BF16 ? add_t<__bf16>(s, slice, y, n, slices, per, st)
                                        : add_t<_Float16>(s, slice, y, n, slices, per, st);
    };
    if (rc == SNHIP_OK) rc = turned(o, v, k, q, d->s0, d->parts, dots, gr->dq, false);
    if (rc == SNHIP_OK) rc = turned(v, o, q, k, gr->dsend, parts, dots + waves * tokens * d->H, gr->dk, true);
    if (rc != SNHIP_OK) return rc;
    k_lin_dg<<<dim3((unsigned)s.slots, (unsigned)s.H), 256, 0, st>>>(s, dots, (int)waves, d->parts, parts, gr->send,
                                                                    gr->dsend, gr->dg, sums);
    SNHIP_CHECK(hipGetLastError());
    if (s.head_g) {
        k_lin_dg_heads<<<(unsigned)s.H, 64, 0, st>>>(s, sums, gr->dg);
        SNHIP_CHECK(hipGetLastError());
    }
    return SNHIP_OK;
}

}  // extern "C"
