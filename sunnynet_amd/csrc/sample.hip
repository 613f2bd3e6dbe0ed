// The next token of every row of logits from one given random number per row.
//
// With m the largest logit, token i weighs exp((x_i - m) / T). The filters keep, in the
// descending order of the logits, a prefix each: top-k by count, top-p by share, min-p by
// weight. So a row needs no sort: it needs the place at which a prefix ends. A block has a
// row, which it reads again in each pass (from L2: the first pass has brought it there), and
//   - counts, or sums, the row into 2048 bins of equal width of (m - x) / T in LDS, down to
//     where weights are 0, and finds the bin in which the prefix ends;
//   - takes that bin's few tokens (for top-k all tokens from it up, if few) into a list and
//     orders them by comparing all pairs; a bin of many (equal logits, mostly) is divided
//     again by the bits of the logits until it is one value, whose tokens go by index;
//   - sums the kept weights by groups of 256 neighbouring indices and walks those sums to
//     the first index up to which they exceed u of their total.
//
// Weights are computed in 64 bits and summed as whole numbers (scaled by a power of two
// that lets a row's sum stay below 2^62): sums do not depend on their order, so neither
// the LDS atomics nor the division of the row change a result, and the rounding of a
// weight (2^-42 of the largest for 2^20 tokens, 2^-47 for 32000) is far below what a sum
// of 32-bit floats would leave.
//
// With few rows the time is that of one block's passes, not of HBM: per 4,096 fp32 tokens
// a pass takes 0.24 us to read them (70 GB/s, one CU's share of L2; more slabs on their way
// at once change nothing), 0.4 to count them, 1.1 to weigh them (instruction issue). 64 rows of 32000: 7 us for the
// largest logit alone, 16 us without filters, 15 us with top-k 40, 33 us with top-p 0.9.
#include "common.h"
#include "planes.h"
#include "snhip_ops.h"

namespace snhip {
namespace {

constexpr int kBins = 2048;
constexpr int kGroup = 256;                  // neighbouring tokens of a wave: four a lane
constexpr int kList = 256;
constexpr int kFracs = 128;                  // of 16 with a polynomial of degree 6: 25.1 us, not 24.4, for 65536
constexpr float kRange = 44.f;               // exp(-44) is 0 in the scaled weights
typedef unsigned long long u64;

// Larger logits have larger keys; -0 and 0 are one.
__device__ __forceinline__ unsigned sort_key(float x) {
    const unsigned b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(unsigned k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct Shared {
    u64 sum[kBins];                // of bins
    unsigned count[kBins];
    double exp2[kFracs];           // 2^(j / kFracs + bits)
    u64 wsum[16];
    unsigned wcount[16];
    float lx[kList];               // the list: logits, indices, weights
    int li[kList];
    u64 lw[kList];
    float wmax[16];
    int windex[16];
    unsigned listed, low_key, high_key;
    int bin, pick;
    u64 above_sum, total;
    unsigned above_count;
    u64 group[(1 << 20) / kGroup];        // kept weight of kGroup neighbouring tokens
};

// exp((x - m) / T) 2^bits, in 64 bits: 2^(n / kFracs + bits) from the table, the rest (below
// log 2 / (2 kFracs)) by its Taylor polynomial of degree 4, 1e-15 of the value. n comes from
// adding 1.5 2^52, whose last bits it is; its power of two is added to the exponent's bits.
// Below 2^-70 the value stays 2^-70, which rounds to the whole number 0.
struct Weights {
    double m, step, low;           // step: kFracs / (T log 2)
    __device__ __forceinline__ double real(float x, const Shared& s) const {
        constexpr double c = 0x1.8p52, l = 0.69314718055994530942 / kFracs;
        const double t = fmax(((double)x - m) * step, -kFracs * 70.), q = t + c, r = t - (q - c);
        const int i = (int)(unsigned)__double_as_longlong(q);
        const double p = fma(r, fma(r, fma(r, fma(r, l * l * l * l / 24., l * l * l / 6.), l * l / 2.), l), 1.);
        const double w = s.exp2[i & (kFracs - 1)] * p;
        return __hiloint2double(__double2hiint(w) + ((i & -kFracs) * ((1 << 20) / kFracs)), __double2loint(w));
    }
    // Rounded to a whole number (below 2^52), by adding 2^52.
    __device__ __forceinline__ u64 whole(double w) const {
        return (u64)__double_as_longlong(w + 0x1p52) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ u64 operator()(float x, const Shared& s) const { return whole(real(x, s)); }
};

// Sum over the wave: rows of 16 lanes by row-local exchanges, then four scalars.
template <int CTRL> __device__ __forceinline__ u64 add_dpp64(u64 x) {
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)x, CTRL, 0xf, 0xf, true),
                   hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(x >> 32), CTRL, 0xf, 0xf, true);
    return x + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 wave_sum(u64 x) {
    x = add_dpp64<0xb1>(x);
    x = add_dpp64<0x4e>(x);
    x = add_dpp64<0x141>(x);
    x = add_dpp64<0x140>(x);
    u64 t = 0;
#pragma unroll
    for (int l = 0; l < 64; l += 16)
        t += (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(x >> 32), l) << 32 |
             (unsigned)__builtin_amdgcn_readlane((int)(unsigned)x, l);
    return t;
}

// A row, read where it is used: a slab of 4 TH tokens at a time, the next one on its way
// (a row of 65536 fp32 is 256 KB, in L2 after the first pass; held in registers it made
// every pass spill). A thread has four neighbouring tokens of a slab, from first(j) on. In
// the last, partial slab that is at most V - 4, so that every read is of four tokens inside
// the row; those that a neighbour has already, and whole reads past the end, count as -inf.
// Rows of fewer than four tokens (ONE) are read one by one.
template <typename T, bool ONE, int TH> struct RowData {
    static constexpr int threads = TH, waves = TH / 64, slab = 4 * TH;
    typedef T T4 __attribute__((ext_vector_type(4)));
    const T* p;
    int V, full, slabs;            // whole slabs, and all
    __device__ __forceinline__ void init(const T* at, int n) {
        p = at;
        V = n;
        full = V / slab;
        slabs = (V + slab - 1) / slab;
    }
    __device__ __forceinline__ int first(int j) const {
        const int i = j * slab + 4 * (int)threadIdx.x;
        return ONE || i < V - 4 ? i : V - 4;
    }
    __device__ __forceinline__ T4 fetch(int i) const {
        typedef T4 T4any __attribute__((aligned(sizeof(T))));
        if constexpr (ONE) {
            T4 t;
#pragma unroll
            for (int e = 0; e < 4; e++) t[e] = p[i + e < V ? i + e : V - 1];
            return t;
        } else {
            return *reinterpret_cast<const T4any*>(p + i);
        }
    }
    __device__ __forceinline__ f32x4 load(int j) const {
        const int want = j * slab + 4 * (int)threadIdx.x, i = first(j);
        const T4 t = fetch(i);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = i + e >= want && i + e < V ? (float)t[e] : -INFINITY;
        return v;
    }
    // f(slab, first index, four logits) for this thread's part of every slab.
    template <typename F> __device__ __forceinline__ void each_slab(F f) const {
        if (full) {
            int i = 4 * (int)threadIdx.x;
            T4 t = fetch(i);
#pragma unroll 1
            for (int j = 0; j < full; j++, i += slab) {
                const T4 next = fetch(j + 1 < full ? i + slab : i);
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = (float)t[e];
                f(j, i, v);
                t = next;
            }
        }
        if (full < slabs) f(full, first(full), load(full));
    }
    // f(index, logit) for every token of this thread.
    template <typename F> __device__ __forceinline__ void each(F f) const {
        each_slab([&](int, int i, f32x4 v) {
#pragma unroll
            for (int e = 0; e < 4; e++) f(i + e, v[e]);
        });
    }
};

template <int TH> __device__ __forceinline__ void clear_bins(Shared& s) {
    for (int i = threadIdx.x; i < kBins; i += TH) {
        s.sum[i] = 0;
        s.count[i] = 0;
    }
    if (threadIdx.x == 0) {
        s.bin = -1;
        s.listed = 0;
        s.low_key = ~0u;
        s.high_key = 0;
    }
}

// The last used bin before which fewer than `limit` tokens lie (or, by sum, a weight of
// at most `limit`), counting from (count, sum) above the first bin. -1: no bin is used.
// Leaves the bin and what lies above it in s.
template <int TH> __device__ __forceinline__ void end_bin(bool by_sum, u64 limit, unsigned count, u64 sum, Shared& s) {
    constexpr int NB = kBins / TH, NW = TH / 64;          // bins of a thread
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __syncthreads();
    unsigned ci[NB], c = 0;
    u64 ti[NB], t = 0;
#pragma unroll
    for (int i = 0; i < NB; i++) {
        ci[i] = s.count[NB * tid + i];
        ti[i] = s.sum[NB * tid + i];
        c += ci[i];
        t += ti[i];
    }
    const unsigned mine_c = c;
    const u64 mine_t = t;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned y = __shfl_up(c, o);
        const u64 z = __shfl_up(t, o);
        if (lane >= o) c += y, t += z;
    }
    if (lane == 63) s.wcount[wave] = c, s.wsum[wave] = t;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) {
        c += w < wave ? s.wcount[w] : 0;
        t += w < wave ? s.wsum[w] : 0;
    }
    c += count - mine_c;               // above the first of this thread's bins
    t += sum - mine_t;
    int mine = -1;
    unsigned above_c = 0;
    u64 above_t = 0;
#pragma unroll
    for (int i = 0; i < NB; i++) {
        if (ci[i] && (by_sum ? t <= limit : c < limit)) mine = NB * tid + i, above_c = c, above_t = t;
        c += ci[i];
        t += ti[i];
    }
    if (mine >= 0) atomicMax(&s.bin, mine);
    __syncthreads();
    if (mine >= 0 && mine == s.bin) {
        s.above_count = above_c;
        s.above_sum = above_t;
    }
    __syncthreads();
}

// Where a prefix ends: tokens above `x`, and of those equal to it the indices below
// `end`, are in it.
struct Cut {
    float x;
    int end;
    __device__ __forceinline__ bool keeps(int i, float y) const { return (y > x) | ((y == x) & (i < end)); }
};

// The first index at which the running total of val(i, x) over indices exceeds
// point(total); -1 if there is none.
template <typename D, typename F, typename G> __device__ __forceinline__ int find_index(D& row, Shared& s, F val, G point_of) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __syncthreads();
    if (tid == 0) s.pick = s.bin = -1;
    row.each_slab([&](int j, int i, f32x4 x) {
        u64 v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = val(i + e, x[e]);
        const u64 t = wave_sum(v[0] + v[1] + (v[2] + v[3]));
        if (lane == 0) s.group[j * D::waves + wave] = t;
    });
    __syncthreads();
    // wave 0 walks the groups, 64 at a time
    const u64* g = s.group;
    const int n = row.slabs * D::waves;
    if (wave == 0) {
        u64 before = 0, total = 0;
        for (int i = lane; i < n; i += 64) total += g[i];
        total = wave_sum(total);
        if (lane == 0) s.total = total;
        const u64 point = point_of(total);
        for (int i = 0; i < n; i += 64) {
            u64 t = i + lane < n ? g[i + lane] : 0;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const u64 y = __shfl_up(t, o);
                if (lane >= o) t += y;
            }
            const u64 m = __ballot(before + t > point);
            if (m) {
                const int l = __ffsll(m) - 1;
                const u64 upto = before + __shfl(t, l);
                if (lane == 0) {
                    s.bin = i + l;
                    s.above_sum = upto - g[i + l];
                }
                break;
            }
            before += __shfl(t, 63);
        }
    }
    __syncthreads();
    const int at = s.bin;
    const u64 point = point_of(s.total);
    if (at >= 0 && wave == at % D::waves) {
        const f32x4 x = row.load(at / D::waves);
        const int i = row.first(at / D::waves);
        u64 w[4], t = 0;
#pragma unroll
        for (int e = 0; e < 4; e++) t += w[e] = val(i + e, x[e]);
        u64 run = t;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const u64 y = __shfl_up(run, o);
            if (lane >= o) run += y;
        }
        run += s.above_sum;
        const u64 m = __ballot(run > point);
        if (m && lane == __ffsll(m) - 1) {
            run -= t;
            int e = 0;
            while (e < 3 && run + w[e] <= point) run += w[e++];
            s.pick = i + e;
        }
    }
    __syncthreads();
    return s.pick;
}

// The cut of a prefix that ends among the tokens with keys [low, high], of which there
// are many: by the bits of the keys, then by index.
template <typename D>
__device__ __forceinline__ Cut cut_by_keys(D& row, const Weights& w, unsigned low, unsigned high, bool by_sum, u64 limit,
                           unsigned count, u64 sum, Shared& s) {
    for (;;) {
        const unsigned span = high - low;         // bins of 2^shift keys, the first at `high`
        int shift = 0;
        while ((span >> shift) >= kBins) shift++;
        __syncthreads();
        clear_bins<D::threads>(s);
        __syncthreads();
        row.each([&](int i, float x) {
            const unsigned k = sort_key(x);
            if (k >= low && k <= high) {
                const unsigned b = (high - k) >> shift;
                atomicAdd(&s.count[b], 1u);
                if (by_sum) atomicAdd(&s.sum[b], w(x, s));
            }
        });
        end_bin<D::threads>(by_sum, limit, count, sum, s);
        count = s.above_count;
        sum = s.above_sum;
        high -= (unsigned)s.bin << shift;
        const unsigned width = (1u << shift) - 1;
        low = high - low > width ? high - width : low;
        if (!shift) break;
    }
    const float x = key_logit(high);
    if (!by_sum) return {x, INT32_MAX};           // all that equal the k-th stay
    const u64 one = w(x, s), room = limit - sum;
    u64 n = row.V;                                // room / one + 1 of them stay
    if (one && (double)room < (double)one * (double)row.V) {
        n = (u64)((double)room / (double)one);
        while (n * one > room) n--;
        while (n * one <= room) n++;
    }
    if (n >= (u64)row.V) return {x, INT32_MAX};
    const int end = find_index(row, s, [&](int, float y) -> u64 { return y == x; }, [&](u64) { return n; });
    return {x, end < 0 ? INT32_MAX : end};
}

// The block's threads in groups of equal size, one group per listed token.
struct ListView {
    int n, per, me;                // listed tokens, threads a group, this group's token
    __device__ __forceinline__ ListView(int n_, int threads) : n(n_) {
        per = threads / (n <= 64 ? 64 : n <= 128 ? 128 : kList);
        me = (int)threadIdx.x / per;
    }
    __device__ __forceinline__ bool first() const { return me < n && (int)threadIdx.x % per == 0; }
    // Sum over the listed tokens j of f(j), in every thread of the group.
    template <typename V, typename F> __device__ __forceinline__ V sum(F f) const {
        V t = 0;
#pragma unroll 4
        for (int j = (int)threadIdx.x % per; j < n; j += per) t += f(j);
        for (int o = 1; o < per; o <<= 1) t += __shfl_xor(t, o);
        return t;
    }
};
template <typename T, bool ONE, int TH>
__global__ __launch_bounds__(TH) void k_sample(SnHipSample a, int* tokens, int* drew) {
    constexpr int NW = TH / 64;
    static_assert(TH >= kList && NW <= 16);
    __shared__ Shared s;
    const int64_t b = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    RowData<T, ONE, TH> row;
    row.init(static_cast<const T*>(a.logits) + b * a.stride, (int)a.V);
    const double temperature = a.temperature ? a.temperature[b] : a.temperature0;
    const double top_p = a.top_p ? a.top_p[b] : a.top_p0, min_p = a.min_p ? a.min_p[b] : a.min_p0;
    const int64_t top_k = a.top_k ? a.top_k[b] : a.top_k0;
    const double u = a.u[b];
    int bits = 0;                  // a row's sum of weights of up to 2^bits stays below 2^62
    while ((1 << bits) < row.V) bits++;
    bits = 62 - bits < 51 ? 62 - bits : 51;
    if (tid < kFracs) s.exp2[tid] = ldexp(exp2((double)tid / kFracs), bits);
    clear_bins<TH>(s);

    // the largest logit; a NaN makes it NaN
    float m = -INFINITY;
    bool nan = false;
    row.each([&](int, float x) {
        m = fmaxf(m, x);
        nan |= x != x;
    });
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (__any(nan)) m = NAN;
    if (lane == 0) s.wmax[wave] = m;
    __syncthreads();
    m = s.wmax[0];
    for (int w = 1; w < NW; w++) m = s.wmax[w] > m || s.wmax[w] != s.wmax[w] ? s.wmax[w] : m;
    // written so that one NaN wins: a NaN m compares false, and a later number does not replace it
    const double zmax = (double)m / temperature;
    auto first_max = [&] {
        int at = row.V;
        row.each([&](int i, float x) {
            if ((m != m ? x != x : x == m) && i < at) at = i;
        });
        for (int o = 32; o; o >>= 1) {
            const int y = __shfl_xor(at, o);
            at = at < y ? at : y;
        }
        __syncthreads();
        if (lane == 0) s.windex[wave] = at;
        __syncthreads();
        for (int w = 0; w < NW; w++) at = at < s.windex[w] ? at : s.windex[w];
        if (tid == 0) {
            tokens[b] = at;
            if (drew) drew[b] = 0;
        }
    };
    auto chosen = [&](int at) {
        if (tid == 0) {
            tokens[b] = at;
            if (drew) drew[b] = 1;
        }
    };
    if (!(temperature > 0.) || !(fabs(zmax) < INFINITY)) return first_max();
    auto point_of = [&](u64 total) -> u64 {
        const u64 point = u > 0. ? (u64)(fmin(u, 1.) * (double)total) : 0;
        return total && point >= total ? total - 1 : point;
    };
    Weights w;
    w.m = (double)m;
    w.step = fmin(kFracs / (0.69314718055994530942 * temperature), 1e300);
    w.low = min_p * ldexp(1., bits);
    // in halves, whose difference is finite for any two finite logits
    const float per = (float)fmin(2. * kBins / ((double)kRange * temperature), 1e30), half = 0.5f * m;
    auto bin_of = [&](float x) { return (int)fminf(fmaf(x, -0.5f, half) * per, 2.f * kBins); };     // kBins and up: weight 0

    Cut cut{-INFINITY, INT32_MAX};
    const bool some_k = top_k > 0 && top_k < row.V, some_p = top_p > 0. && top_p < 1.;
    if (some_k) {
        row.each([&](int, float x) {
            const int i = bin_of(x);
            if (i < kBins) atomicAdd(&s.count[i], 1u);
        });
        end_bin<TH>(false, (u64)top_k, 0, 0, s);
        const int last = s.bin;
        const unsigned above = s.above_count, in = s.count[last];
        const bool all = above + in <= (unsigned)kList;          // every candidate fits the list
        row.each([&](int i, float x) {
            const int q = bin_of(x);
            if (q == last || (all && q < last)) {
                const unsigned at = atomicAdd(&s.listed, 1u);
                if (at < (unsigned)kList) s.lx[at] = x, s.li[at] = i;
                if (!all) {
                    atomicMin(&s.low_key, sort_key(x));
                    atomicMax(&s.high_key, sort_key(x));
                }
            }
        });
        __syncthreads();
        if (all) {
            // the rest on the list alone: a group of threads per token
            const ListView list((int)s.listed, TH);
            const int n = list.n, me = list.me;
            const float x = me < n ? s.lx[me] : 0.f;
            const int at = me < n ? s.li[me] : 0;
            const unsigned rank = list.sum<unsigned>([&](int j) -> unsigned { return s.lx[j] > x; });
            u64 mine = me < n && rank < (u64)top_k ? w(x, s) : 0;
            if (list.first()) s.lw[me] = mine;
            __syncthreads();
            const u64 total = list.sum<u64>([&](int j) { return s.lw[j]; });
            if (some_p) {
                const u64 before = list.sum<u64>([&](int j) -> u64 {
                    return s.lx[j] > x || (s.lx[j] == x && s.li[j] < at) ? s.lw[j] : 0;
                });
                if (before > (u64)(top_p * (double)total)) mine = 0;
            }
            if (mine && w.real(x, s) < w.low) mine = 0;
            __syncthreads();
            if (list.first()) s.lw[me] = mine;
            if (tid == 0) s.pick = -1;
            __syncthreads();
            const u64 kept = list.sum<u64>([&](int j) { return s.lw[j]; });
            const u64 before = list.sum<u64>([&](int j) -> u64 { return s.li[j] < at ? s.lw[j] : 0; });
            const u64 point = point_of(kept);
            if (list.first() && mine && before <= point && point < before + mine) s.pick = at;
            __syncthreads();
            if (s.pick < 0) return first_max();        // min-p leaves nothing
            return chosen(s.pick);
        } else if (in <= (unsigned)kList) {
            const ListView list((int)s.listed, TH);
            const int n = list.n, me = list.me;
            const float x = me < n ? s.lx[me] : 0.f;
            const unsigned rank = above + list.sum<unsigned>([&](int j) -> unsigned { return s.lx[j] > x; });
            // the smallest kept one: fewer than k above it, and k with its equals
            const unsigned upto = rank + list.sum<unsigned>([&](int j) -> unsigned { return s.lx[j] == x; });
            if (list.first() && rank < (u64)top_k && (upto >= (u64)top_k || upto == above + in)) s.wmax[0] = x;
            __syncthreads();
            cut.x = s.wmax[0];
        } else {
            cut = cut_by_keys(row, w, s.low_key, s.high_key, false, (u64)top_k, above, 0, s);
        }
        __syncthreads();
        clear_bins<TH>(s);
        __syncthreads();
    }
    if (some_p) {
        u64 t = 0;
        row.each_slab([&](int, int, f32x4 x) {
            u64 y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = w(x[e], s);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = bin_of(x[e]);
                if (i < kBins && x[e] >= cut.x) {
                    t += y[e];
                    atomicAdd(&s.count[i], 1u);
                    atomicAdd(&s.sum[i], y[e]);
                }
            }
        });
        t = wave_sum(t);
        if (lane == 0) s.wsum[wave] = t;
        __syncthreads();
        t = 0;
        for (int i = 0; i < NW; i++) t += s.wsum[i];
        const u64 limit = (u64)(top_p * (double)t);
        end_bin<TH>(true, limit, 0, 0, s);
        const int last = s.bin;
        const u64 above = s.above_sum;
        const unsigned in = s.count[last];
        const float floor_x = cut.x;
        row.each([&](int i, float x) {
            if (bin_of(x) == last && x >= floor_x) {
                const unsigned at = atomicAdd(&s.listed, 1u);
                if (at < (unsigned)kList) s.lx[at] = x, s.li[at] = i, s.lw[at] = w(x, s);
                if (in > (unsigned)kList) {
                    atomicMin(&s.low_key, sort_key(x));
                    atomicMax(&s.high_key, sort_key(x));
                }
            }
        });
        __syncthreads();
        if (in <= (unsigned)kList) {
            // in order, the last token before which the sum is within the limit
            const ListView list((int)s.listed, TH);
            const int n = list.n, me = list.me;
            const float x = me < n ? s.lx[me] : 0.f;
            const int at = me < n ? s.li[me] : 0;
            const u64 before = above + list.sum<u64>([&](int j) -> u64 {
                return s.lx[j] > x || (s.lx[j] == x && s.li[j] < at) ? s.lw[j] : 0;
            });
            const bool in_it = me < n && before <= limit;
            const unsigned rank = list.sum<unsigned>([&](int j) -> unsigned {
                return s.lx[j] > x || (s.lx[j] == x && s.li[j] < at);
            });
            __syncthreads();
            if (tid == 0) s.pick = -1;
            __syncthreads();
            if (in_it && list.first()) atomicMax(&s.pick, (int)rank);
            __syncthreads();
            if (in_it && list.first() && (int)rank == s.pick) {
                s.wmax[0] = x;
                s.windex[0] = at + 1;
            }
            __syncthreads();
            cut = {s.wmax[0], s.windex[0]};
        } else {
            cut = cut_by_keys(row, w, s.low_key, s.high_key, true, limit, s.above_count, above, s);
        }
    }
    // weights first, choices after: a branch per token would wait for the table token by token
    auto kept = [&](int i, float x) -> u64 {
        const double y = w.real(x, s);
        const u64 n = w.whole(y);
        return (cut.keeps(i, x) & !(y < w.low)) ? n : 0;
    };
    const int pick = find_index(row, s, kept, point_of);
    if (pick < 0) return first_max();
    chosen(pick);
}

template <typename T> snhip_status sample_t(const SnHipSample& all, int* tokens, int* drew, hipStream_t st) {
    // A row of 16 waves is done sooner, two rows of 8 waves share a CU's LDS and registers:
    // 8 for more rows than CUs (top-p 0.9, 512 rows of 12000: 27 us against 39; of 65536: 108
    // against 126) and for short rows, whose barriers weigh more (one row of 1000: 10.2
    // against 11.9); 16 otherwise (64 rows of 32000: 33 against 37; of 8000: 17 both).
    // A grid holds fewer than 2^32 threads: more rows go in several launches.
    constexpr int64_t most = 1 << 22;
    for (int64_t r = 0; r < all.B; r += most) {
        SnHipSample a = all;
        const unsigned B = (unsigned)(all.B - r < most ? all.B - r : most);
        a.logits = static_cast<const T*>(all.logits) + r * all.stride;
        a.u += r;
        if (a.temperature) a.temperature += r;
        if (a.top_k) a.top_k += r;
        if (a.top_p) a.top_p += r;
        if (a.min_p) a.min_p += r;
        int* told = drew ? drew + r : nullptr;
        if (a.V < 4) k_sample<T, true, 512><<<B, 512, 0, st>>>(a, tokens + r, told);
        else if (B > 256 || a.V <= 8192) k_sample<T, false, 512><<<B, 512, 0, st>>>(a, tokens + r, told);
        else k_sample<T, false, 1024><<<B, 1024, 0, st>>>(a, tokens + r, told);
        SNHIP_CHECK(hipGetLastError());
    }
    return SNHIP_OK;
}

}  // namespace
}  // namespace snhip

using namespace snhip;

extern "C" {

snhip_status snhip_op_sample_drew_dev(const SnHipSample* s, int32_t* tokens, int32_t* drew, void* stream) {
    if (!s || !s->logits || !s->u || !tokens || s->B < 1 || s->B > INT32_MAX || s->V < 1 || s->V > (1 << 20) ||
        s->stride < 0 || s->dtype < SNHIP_F32 || s->dtype > SNHIP_F16)
        return SNHIP_E_INVAL;
    const hipStream_t st = as_stream(stream);
    if (s->dtype == SNHIP_F32) return sample_t<float>(*s, tokens, drew, st);
    if (s->dtype == SNHIP_BF16) return sample_t<__bf16>(*s, tokens, drew, st);
    return sample_t<_Float16>(*s, tokens, drew, st);
}

snhip_status snhip_op_sample_dev(const SnHipSample* s, int32_t* tokens, void* stream) {
    return snhip_op_sample_drew_dev(s, tokens, nullptr, stream);
}

}  // extern "C"
