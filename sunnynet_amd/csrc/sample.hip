// The next token of every row of logits from one given random number per row.
//
// With z = logit / T and m = max z, token i weighs exp(z_i - m). The filters keep, in
// the descending order of z, a prefix each: top-k by count, top-p by share, min-p by
// weight. So a row needs no sort: it needs the value at which a prefix ends. That value
// is found on a monotone 32-bit image of the logit (sort_key), 2048 bins at a time:
// counts or sums per bin in LDS, the bin in which the prefix ends, then the same over
// that bin's keys until it is one key. The token is the first index up to which the kept
// weights sum to more than u of their total; a wave sums a span of indices, and the span
// that holds the point is divided again.
//
// Weights are computed in 64 bits and summed as whole numbers (scaled by a power of two
// that lets a row's sum stay below 2^62): sums do not depend on their order, so neither
// the LDS atomics nor the division of the row change a result, and the rounding of a
// weight (2^-42 of the largest for 2^20 tokens, 2^-47 for 32000) is far below what a
// sum of 32-bit floats would leave.
#include "common.h"
#include "snhip_ops.h"

namespace snhip {
namespace {

constexpr int kBins = 2048;
constexpr int kThreads = 1024, kWaves = kThreads / 64;
typedef unsigned long long u64;

__device__ __forceinline__ float logit_f(float x) { return x; }
__device__ __forceinline__ float logit_f(__bf16 x) { return (float)x; }
__device__ __forceinline__ float logit_f(_Float16 x) { return (float)x; }

// Larger logits have larger keys; -0 and 0 are one.
__device__ __forceinline__ unsigned sort_key(float x) {
    const unsigned b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Row {
    double temperature, zmax, scale;
};

// The weight of a logit as a whole number; a NaN or a logit of -inf weighs nothing.
__device__ __forceinline__ u64 weight(const Row& r, float x) {
    const double w = exp((double)x / r.temperature - r.zmax);
    return w > 0. ? (u64)rint(w * r.scale) : 0;
}

struct Shared {
    u64 sum[kBins];
    unsigned count[kBins];
    u64 wsum[kWaves];
    unsigned wcount[kWaves];
    u64 pick_sum;              // what the search found
    unsigned pick_bin, pick_count;
    float wmax[kWaves];
    int warg[kWaves], wnan[kWaves];
};

__device__ __forceinline__ u64 wave_sum(u64 x) {
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// In the descending order of keys from `top` down, where a prefix ends: the key of the
// last token before which `limit` is not yet passed (by count: fewer than `limit` tokens
// before it; by sum: the weights before it sum to at most `limit`). Also the number and
// sum of the tokens above that key. Tokens below `low` do not take part.
struct Cut {
    unsigned key, above;
    u64 sum;
};
template <typename T>
__device__ Cut find_cut(const T* x, int V, const Row& row, unsigned top, unsigned low, bool by_sum, u64 limit,
                        Shared& s) {
    const int tid = threadIdx.x;
    Cut c{0, 0, 0};
    unsigned hi = top, lo = low;               // the keys in question
    for (;;) {
        const unsigned span = hi - lo;         // bins of 2^shift keys, the first at hi
        int shift = 0;
        while ((span >> shift) >= kBins) shift++;
        for (int i = tid; i < kBins; i += kThreads) {
            s.sum[i] = 0;
            s.count[i] = 0;
        }
        __syncthreads();
        for (int i = tid; i < V; i += kThreads) {
            const float f = logit_f(x[i]);
            const unsigned k = sort_key(f);
            if (f == f && k >= lo && k <= hi) {
                const unsigned b = (hi - k) >> shift;
                atomicAdd(&s.count[b], 1u);
                atomicAdd(&s.sum[b], weight(row, f));
            }
        }
        __syncthreads();
        if (tid == 0) {                        // the bin in which the prefix ends
            u64 sum = c.sum;
            unsigned n = c.above, b = 0, last = 0;
            u64 lsum = sum;
            unsigned ln = n;
            bool any = false;
            for (b = 0; b < kBins; b++) {
                if (!s.count[b]) continue;
                if (any && (by_sum ? sum > limit : n >= limit)) break;
                any = true;
                last = b;
                lsum = sum;
                ln = n;
                sum += s.sum[b];
                n += s.count[b];
            }
            s.pick_bin = last;
            s.pick_sum = lsum;
            s.pick_count = ln;
        }
        __syncthreads();
        c.sum = s.pick_sum;
        c.above = s.pick_count;
        hi = hi - (s.pick_bin << shift);
        const unsigned width = (1u << shift) - 1;
        lo = hi - lo > width ? hi - width : lo;
        __syncthreads();
        if (!shift) {
            c.key = hi;
            return c;
        }
    }
}

// The first index at which a running total over indices [0, V) of val(i) exceeds
// `point`, and the total before its span; V if there is none. The row is divided into
// kWaves spans, the span with the point again, down to 64 indices.
template <typename F> __device__ int find_index(int V, u64 point, Shared& s, F val) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int lo = 0, hi = V;
    u64 before = 0;
    while (hi - lo > 64) {
        const int span = ((hi - lo + kWaves - 1) / kWaves + 63) & ~63;
        const int a = lo + wave * span, e = a + span < hi ? a + span : hi;
        u64 t = 0;
        for (int i = a + lane; i < e; i += 64) t += val(i);
        t = wave_sum(t);
        __syncthreads();
        if (lane == 0) s.wsum[wave] = t;
        __syncthreads();
        int w = 0;
        u64 sum = before;
        while (w < kWaves && sum + s.wsum[w] <= point) sum += s.wsum[w++];
        if (w == kWaves) return V;
        before = sum;
        lo = lo + w * span;
        hi = lo + span < hi ? lo + span : hi;
    }
    // every wave does the same last step
    u64 t = lo + lane < hi ? val(lo + lane) : 0;
    for (int o = 1; o < 64; o <<= 1) {
        const u64 y = __shfl_up(t, o);
        if (lane >= o) t += y;
    }
    const u64 m = __ballot(lo + lane < hi && before + t > point);
    return m ? lo + __ffsll(m) - 1 : V;
}

template <typename T> __global__ __launch_bounds__(kThreads) void k_sample(SnHipSample a, int* tokens) {
    __shared__ Shared s;
    const int64_t b = blockIdx.x;
    const int V = (int)a.V, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* x = static_cast<const T*>(a.logits) + b * a.stride;
    Row row;
    row.temperature = a.temperature ? a.temperature[b] : a.temperature0;
    const double top_p = a.top_p ? a.top_p[b] : a.top_p0, min_p = a.min_p ? a.min_p[b] : a.min_p0;
    const int64_t top_k = a.top_k ? a.top_k[b] : a.top_k0;

    // the first maximal logit; NaN counts as maximal
    float m = -INFINITY;
    int at = V, nan = V;
    for (int i = tid; i < V; i += kThreads) {
        const float f = logit_f(x[i]);
        if (f != f) nan = nan < i ? nan : i;
        else if (at == V || f > m) m = f, at = i;
    }
    for (int o = 32; o; o >>= 1) {
        const float om = __shfl_xor(m, o);
        const int oa = __shfl_xor(at, o), on = __shfl_xor(nan, o);
        if (oa < V && (at == V || om > m || (om == m && oa < at))) m = om, at = oa;
        nan = nan < on ? nan : on;
    }
    if (lane == 0) s.wmax[wave] = m, s.warg[wave] = at, s.wnan[wave] = nan;
    __syncthreads();
    m = s.wmax[0], at = s.warg[0], nan = s.wnan[0];
    for (int w = 1; w < kWaves; w++) {
        const int oa = s.warg[w];
        if (oa < V && (at == V || s.wmax[w] > m || (s.wmax[w] == m && oa < at))) m = s.wmax[w], at = oa;
        nan = nan < s.wnan[w] ? nan : s.wnan[w];
    }
    const int greedy = nan < V ? nan : at;
    row.zmax = (double)m / row.temperature;
    int bits = 0;
    while ((1 << bits) < V) bits++;
    row.scale = ldexp(1.0, 62 - bits);
    if (!(row.temperature > 0.) || nan < V || !(fabs(row.zmax) < INFINITY)) {
        if (tid == 0) tokens[b] = greedy;
        return;
    }
    const unsigned top = sort_key(m), all = sort_key(-INFINITY);
    unsigned low = all;                        // the smallest key that is kept
    int ties = V;                              // and the first index from which it is not
    if (top_k > 0 && top_k < V) low = find_cut(x, V, row, top, all, false, (u64)top_k, s).key;
    if (top_p > 0. && top_p < 1.) {
        __syncthreads();
        u64 t = 0;
        for (int i = tid; i < V; i += kThreads) {
            const float f = logit_f(x[i]);
            if (sort_key(f) >= low) t += weight(row, f);
        }
        t = wave_sum(t);
        if (lane == 0) s.wsum[wave] = t;
        __syncthreads();
        t = 0;
        for (int w = 0; w < kWaves; w++) t += s.wsum[w];
        const u64 limit = (u64)(top_p * (double)t);
        const Cut c = find_cut(x, V, row, top, low, true, limit, s);
        low = c.key;
        // of the equal ones at the end, those before which the sum is at most the limit
        const unsigned kb = low & 0x80000000u ? low & 0x7fffffffu : ~low;
        const u64 w = weight(row, __uint_as_float(kb));
        const u64 n = w ? (limit - c.sum) / w + 1 : V;
        if (n < (u64)V) ties = find_index(V, n, s, [&](int i) -> u64 { return sort_key(logit_f(x[i])) == low; });
    }
    auto kept = [&](int i) -> u64 {
        const float f = logit_f(x[i]);
        const unsigned k = sort_key(f);
        if (k < low || (k == low && i >= ties)) return 0;
        const double w = exp((double)f / row.temperature - row.zmax);
        return w < min_p ? 0 : (u64)rint(w * row.scale);
    };
    __syncthreads();
    u64 t = 0;
    for (int i = tid; i < V; i += kThreads) t += kept(i);
    t = wave_sum(t);
    if (lane == 0) s.wsum[wave] = t;
    __syncthreads();
    t = 0;
    for (int w = 0; w < kWaves; w++) t += s.wsum[w];
    const double u = a.u[b];
    u64 point = u > 0. ? (u64)(u * (double)t) : 0;
    if (t && point >= t) point = t - 1;
    const int pick = t ? find_index(V, point, s, kept) : greedy;
    if (tid == 0) tokens[b] = pick;
}

}  // namespace
}  // namespace snhip

using namespace snhip;

extern "C" snhip_status snhip_op_sample_dev(const SnHipSample* s, int32_t* tokens, void* stream) {
    if (!s || !s->logits || !s->u || !tokens || s->B < 1 || s->B > INT32_MAX || s->V < 1 || s->V > (1 << 20) ||
        s->stride < 0 || s->dtype < SNHIP_F32 || s->dtype > SNHIP_F16)
        return SNHIP_E_INVAL;
    const hipStream_t st = as_stream(stream);
    if (s->dtype == SNHIP_F32) k_sample<float><<<(unsigned)s->B, kThreads, 0, st>>>(*s, tokens);
    else if (s->dtype == SNHIP_BF16) k_sample<__bf16><<<(unsigned)s->B, kThreads, 0, st>>>(*s, tokens);
    else k_sample<_Float16><<<(unsigned)s->B, kThreads, 0, st>>>(*s, tokens);
    SNHIP_CHECK(hipGetLastError());
    return SNHIP_OK;
}
