// The embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   y_i = scale table[id_i]        dtable[r] = scale (sum of dy_i over the i with id_i = r)
//
// An id outside [0, R) names no row: y_i is 0 and dy_i goes nowhere.
//
// Lookup: bound by memory. A thread copies 16 bytes of a row: 20 us for 32768 rows of 1024 in
// bf16 (4.4 TB/s of what is read and written).
//
// Gradient: the tokens are sorted by id, stably, so a row's tokens lie next to each other
// in the order of the batch, and no sum needs an atomic: the same call gives the same bits.
// The sort goes by digits of up to 10 bits, the lowest first, two passes up to 2^20 rows. In
// a pass a block ranks one tile of the tokens: it counts its waves' digits in LDS, adds what
// the tiles and digits before it count, and a wave then walks its tokens 64 at a time,
// ranking equal digits by ballots. Each pass' digits are counted by a launch of their own: by
// atomics beside the pass before it took 10 us more where an id is frequent.
// A wave then takes some neighbouring sorted tokens and 16 bytes a lane of the columns, sums
// runs of one id in fp32 and writes the rows that lie inside it; runs that go on in a
// neighbour's tokens are left as partial sums, which k_embed_join adds in order. Rows that
// no token names are cleared by blocks of their own beside these.
// Rows of up to half a wave's columns share a wave, and a wave joins a group's run by itself
// unless it is long (524288 tokens of text, 64 columns in bf16: 208 us without either, 90 so).
// 32768 tokens of text, a table of 32000 x 1024 in bf16: two passes of 3.5 us to count and 7.7 (the
// latency of their steps), sums 30, joins 10; up to 4096 tokens one block sorts alone.
#include <type_traits>

#include "common.h"
#include "planes.h"
#include "snhip_ops.h"

namespace snhip {
namespace {

// At most so many tiles, of at least so many tokens; up to how many one block sorts alone.
constexpr int kEmbedTiles = 128, kEmbedTile = 1024, kEmbedAlone = 4096;
constexpr int kEmbedBits = 10, kEmbedBins = 1 << kEmbedBits, kEmbedWaves = 8;

template <typename T> constexpr int kLane = 16 / (int)sizeof(T);      // columns of a lane

struct EmbedP {
    const void* ids;
    bool wide;                  // 64-bit ids
    int64_t n, R, D;
    int tile, tiles;            // tokens of a tile
    int passes, bits;           // of a digit
    unsigned* key[2];           // sorted ids (R: none), and their tokens
    int* at[2];
    int* count;                 // (tiles, 2^bits), of the pass that runs
    float* part;                // (groups, 2, ld): sums of the runs that a group shares with its neighbours
    int64_t ld;                 // D up to a multiple of 8
    int group;                  // sorted tokens of a wave
    int64_t groups;
    int lanes;                  // log2 of the lanes that a group's columns take (64: or more)
    float scale;
};

__device__ __forceinline__ unsigned embed_key(const EmbedP& a, int64_t i) {
    const int64_t id = a.wide ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
    return id < 0 || id >= a.R ? (unsigned)a.R : (unsigned)id;
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void k_embed(EmbedP a, const T* table, T* y, int per) {
    constexpr int L = kLane<T>;
    const int cols = (int)((a.D + L - 1) / L);
    for (int64_t i0 = blockIdx.x * (int64_t)per; i0 < a.n; i0 += gridDim.x * (int64_t)per) {
    const int rows = (int)(a.n - i0 < per ? a.n - i0 : per);
    for (int j = threadIdx.x; j < rows * cols; j += 256) {
        const int r = j / cols, c = (j - r * cols) * L;
        const unsigned id = embed_key(a, i0 + r);
        const bool none = id >= (unsigned)a.R;
        const T* from = table + (none ? 0 : (int64_t)id * a.D) + c;
        T* to = y + (i0 + r) * a.D + c;
        typedef T V __attribute__((ext_vector_type(L)));
        if constexpr (VEC) {
            const V x = *reinterpret_cast<const V*>(from);
            V o;
#pragma unroll
            for (int e = 0; e < L; e++) o[e] = none ? (T)0.f : (T)(a.scale * (float)x[e]);
            *reinterpret_cast<V*>(to) = o;
        } else {
            for (int e = 0; e < L && c + e < a.D; e++) to[e] = none ? (T)0.f : (T)(a.scale * (float)from[e]);
        }
    }
    }
}

// Counts a pass' digits of a tile.
__global__ __launch_bounds__(1024) void k_embed_count(EmbedP a, int p) {
    __shared__ int bin[kEmbedBins];
    const int tid = threadIdx.x, bins = 1 << a.bits, shift = p * a.bits;
    const unsigned* const from = a.key[(p + 1) & 1];
    if (tid < bins) bin[tid] = 0;
    __syncthreads();
    const int64_t t0 = blockIdx.x * (int64_t)a.tile, t1 = t0 + a.tile < a.n ? t0 + a.tile : a.n;
    for (int64_t i = t0 + tid; i < t1; i += 1024) atomicAdd(&bin[((p ? from[i] : embed_key(a, i)) >> shift) & (bins - 1)], 1);
    __syncthreads();
    if (tid < bins) a.count[(int64_t)blockIdx.x * bins + tid] = bin[tid];
}

// Puts a tile's tokens in the places that passes p0 to p1 - 1 give them (more than one only
// where the tile is all there is: then its own counts are all counts). A thread has PER
// neighbouring digits.
template <int PER> __global__ __launch_bounds__(64 * kEmbedWaves) void k_embed_sort(EmbedP a, int p0, int p1) {
    constexpr int NW = kEmbedWaves, NTH = 64 * NW, BINS = PER * NTH;
    __shared__ int next[NW][BINS];             // of a wave: its tokens of a digit, then the place of the next
    __shared__ int wsum[NW];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = 1 << a.bits;
    const int64_t t0 = blockIdx.x * (int64_t)a.tile, t1 = t0 + a.tile < a.n ? t0 + a.tile : a.n;
    const int64_t per = (a.tile + NTH - 1) / NTH * 64, w0 = t0 + wave * per, w1 = w0 + per < t1 ? w0 + per : t1;
    for (int p = p0; p < p1; p++) {
        const int shift = p * a.bits;
        const unsigned* const from = a.key[(p + 1) & 1];
        const int* const from_at = a.at[(p + 1) & 1];
        auto key_of = [&](int64_t i) { return p ? from[i] : embed_key(a, i); };
        for (int i = tid; i < NW * BINS; i += NTH) next[0][i] = 0;
        __syncthreads();
        for (int64_t i = w0 + lane; i < w1; i += 64) atomicAdd(&next[wave][(key_of(i) >> shift) & (bins - 1)], 1);
        __syncthreads();
        // where this tile's tokens of a digit begin: after all smaller digits and earlier tiles
        int before[PER] = {}, all[PER] = {}, sum = 0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int b = tid * PER + j;
            if (a.tiles == 1) {
#pragma unroll
                for (int w = 0; w < NW; w++) all[j] += next[w][b];
            } else if (b < bins) {
#pragma unroll 8
                for (int t = 0; t < a.tiles; t++) {
                    const int c = a.count[(int64_t)t * bins + b];
                    before[j] += t < (int)blockIdx.x ? c : 0;
                    all[j] += c;
                }
            }
            sum += all[j];
        }
        int run = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(run, o);
            if (lane >= o) run += y;
        }
        if (lane == 63) wsum[wave] = run;
        __syncthreads();
        int first = run - sum;
        for (int w = 0; w < wave; w++) first += wsum[w];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            int place = first + before[j];
            first += all[j];
#pragma unroll
            for (int w = 0; w < NW; w++) {
                const int c = next[w][tid * PER + j];
                next[w][tid * PER + j] = place;
                place += c;
            }
        }
        __syncthreads();
        unsigned* const key = a.key[p & 1];
        int* const at = a.at[p & 1];
        for (int64_t i0 = w0; i0 < w1; i0 += 64) {
            const int64_t i = i0 + lane;
            const bool live = i < w1;
            const unsigned k = live ? key_of(i) : 0;
            const int token = live ? (p ? from_at[i] : (int)i) : 0, digit = (int)(k >> shift) & (bins - 1);
            unsigned long long same = __ballot(live);
            for (int b = 0; b < a.bits; b++) {
                const unsigned long long one = __ballot(digit >> b & 1);
                same &= digit >> b & 1 ? one : ~one;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1)), to = next[wave][digit] + rank;
            // a wave's LDS accesses keep their order: all lanes have read before one writes
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (live && rank == 0) next[wave][digit] = to + __popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (live) {
                key[to] = k;
                at[to] = token;
            }
        }
        __syncthreads();
    }
}

// L neighbouring columns of a row, of which the first n exist, as floats. VEC: all exist,
// 16-byte aligned.
template <typename T, int L, bool VEC> __device__ __forceinline__ void embed_load(const T* p, int n, float* x) {
    typedef T V __attribute__((ext_vector_type(L), aligned(16)));
    if constexpr (VEC) {
        const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
        for (int e = 0; e < L; e++) x[e] = (float)v[e];
    } else {
#pragma unroll
        for (int e = 0; e < L; e++) x[e] = e < n ? (float)p[e] : 0.f;
    }
}
template <typename T, int L, bool VEC> __device__ __forceinline__ void embed_store(T* p, int n, const float* x, float scale) {
    typedef T V __attribute__((ext_vector_type(L), aligned(16)));
    if constexpr (VEC) {
        V v;
#pragma unroll
        for (int e = 0; e < L; e++) v[e] = (T)(scale * x[e]);
        *reinterpret_cast<V*>(p) = v;
    } else {
#pragma unroll
        for (int e = 0; e < L; e++)
            if (e < n) p[e] = (T)(scale * x[e]);
    }
}

// Blocks before `fill`: four waves, a group of sorted tokens and 64 lanes of columns each,
// or with NARROW rows several groups. The others clear the unused ones of 64 rows each.
template <typename T, bool VEC, bool NARROW>
__global__ __launch_bounds__(256) void k_embed_grad(EmbedP a, const T* dy, T* out, int slices, int64_t fill) {
    constexpr int L = kLane<T>, U = 8;
    const int lg = NARROW ? a.lanes : 6, subs = 64 >> lg;      // groups of a wave
    const int lane = threadIdx.x & 63, sub = NARROW ? lane >> lg : 0, own = NARROW ? lane & ((1 << lg) - 1) : lane;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned* const key = a.key[(a.passes - 1) & 1];
    const int* const at = a.at[(a.passes - 1) & 1];
    if (blockIdx.x >= fill) {
        const int64_t r0 = (blockIdx.x - fill) * 64;
        // a lane looks for its row's first token among the sorted ones: no run is walked, however long
        int64_t lo = 0, hi = a.n;
        while (lo < hi) {
            const int64_t mid = (lo + hi) / 2;
            if (key[mid] < (unsigned)r0 + lane) lo = mid + 1;
            else hi = mid;
        }
        const unsigned long long used = __ballot(lo < a.n && key[lo] == (unsigned)r0 + lane);
        const float zero[L] = {};
        for (int r = wave * subs + sub; r < 64 && r0 + r < a.R; r += 4 * subs)
            if (!(used >> r & 1))
                for (int64_t c = own * L; c < a.D; c += 64 * L)
                    embed_store<T, L, VEC>(out + (r0 + r) * a.D + c, (int)(a.D - c < L ? a.D - c : L), zero, 0.f);
        return;
    }
    const int64_t task = blockIdx.x * (int64_t)4 + wave, g = NARROW ? task * subs + sub : task / slices;
    if (g >= a.groups) return;
    const int64_t c = (NARROW ? 0 : task % slices * 64 * L) + own * L, i0 = g * a.group, i1 = i0 + a.group < a.n ? i0 + a.group : a.n;
    const int n = (int)(a.D - c < L ? a.D - c : L);
    float sum[L] = {};
    unsigned now = key[i0];
    if (now >= (unsigned)a.R) return;                   // as all after it: tokens of no row
    bool open = i0 > 0 && key[i0 - 1] == now;           // the run began before this group
    auto flush = [&](bool goes_on) {
        if (now < (unsigned)a.R && c < a.D) {
            if (open || goes_on) embed_store<float, L, true>(a.part + (g * 2 + (open ? 0 : 1)) * a.ld + c, L, sum, 1.f);
            else embed_store<T, L, VEC>(out + (int64_t)now * a.D + c, n, sum, a.scale);
        }
    };
    for (int64_t i = i0; i < i1; i += U) {
        float x[U][L];
        unsigned k[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t j = i + u < i1 ? i + u : i1 - 1;
            k[u] = key[j];
            if (c < a.D) embed_load<T, L, VEC>(dy + (int64_t)at[j] * a.D + c, n, x[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (i + u >= i1) continue;
            if (k[u] != now) {
                flush(false);
                now = k[u];
                open = false;
#pragma unroll
                for (int e = 0; e < L; e++) sum[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < L; e++) sum[e] += x[u][e];
        }
    }
    flush(i1 < a.n && key[i1] == now);
}

// Adds the partial sums of the runs that begin in a group and end in a later one, for 64
// lanes of columns (NARROW: lanes that are left share the groups): a wave for a group whose run
// ends within a step of loads, then all four of the block's for a longer one, in turn.
template <typename T, bool VEC, bool NARROW> __global__ __launch_bounds__(256) void k_embed_join(EmbedP a, T* out, int slices) {
    constexpr int L = kLane<T>, U = 8;
    __shared__ float part[3][64][L + 1];
    __shared__ int runs[4];                    // of a wave's group: groups that its run goes on in, where they are many
    const unsigned* const key = a.key[(a.passes - 1) & 1];
    const int lg = NARROW ? a.lanes : 6, subs = 64 >> lg, lane = threadIdx.x & 63;
    const int sub = NARROW ? lane >> lg : 0, own = NARROW ? lane & ((1 << lg) - 1) : lane;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t g0 = blockIdx.x / slices * 4, c = (blockIdx.x % slices) * 64 * L + own * L;
    const int n = (int)(a.D - c < L ? a.D - c : L);
    auto id_of = [&](int64_t g) { return key[(g + 1) * a.group - 1]; };          // of a group's last token
    // how many groups after g the run of g's last token goes on in
    auto length = [&](int64_t g) {
        const int64_t i0 = g * a.group;
        if (i0 + a.group >= a.n) return 0;
        const unsigned k = id_of(g);
        if (key[i0 + a.group] != k || k >= (unsigned)a.R || (i0 > 0 && key[i0 - 1] == k)) return 0;
        auto in = [&](int64_t j) { return (g + j) * a.group < a.n && key[(g + j) * a.group] == k; };
        int64_t lo = 1, hi = 2;                // in(lo), by doubling not in(hi)
        while (in(hi)) lo = hi, hi *= 2;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) / 2;
            if (in(mid)) lo = mid;
            else hi = mid;
        }
        return (int)lo;
    };
    float sum[L];
    auto add = [&](int64_t g, int m, int w, int waves) {       // this wave's share of m groups after g, and g's own
        const int step = waves * subs;
#pragma unroll
        for (int e = 0; e < L; e++) sum[e] = 0.f;
        if (c < a.D) {
            if (w == 0 && sub == 0) embed_load<float, L, true>(a.part + (g * 2 + 1) * a.ld + c, L, sum);
            for (int q = 1 + w * subs + sub; q <= m; q += step * U) {
                float x[U][L];
#pragma unroll
                for (int u = 0; u < U; u++)
                    embed_load<float, L, true>(a.part + (g + (q + step * u <= m ? q + step * u : m)) * 2 * a.ld + c, L, x[u]);
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (q + step * u > m) continue;
#pragma unroll
                    for (int e = 0; e < L; e++) sum[e] += x[u][e];
                }
            }
        }
        if (NARROW)
            for (int o = 1 << lg; o < 64; o <<= 1)
#pragma unroll
                for (int e = 0; e < L; e++) sum[e] += __shfl_xor(sum[e], o);
    };
    auto put = [&](int64_t g) {
        if (sub == 0 && c < a.D) embed_store<T, L, VEC>(out + (int64_t)id_of(g) * a.D + c, n, sum, a.scale);
    };
    const int m = length(g0 + wave);
    const bool alone = m <= subs * U;
    if (m > 0 && alone) {
        add(g0 + wave, m, 0, 1);
        put(g0 + wave);
    }
    if (lane == 0) runs[wave] = alone ? 0 : m;
    __syncthreads();
    for (int r = 0; r < 4; r++) {
        if (!runs[r]) continue;
        add(g0 + r, runs[r], wave, 4);
        if (wave)
#pragma unroll
            for (int e = 0; e < L; e++) part[wave - 1][lane][e] = sum[e];
        __syncthreads();
        if (!wave) {
#pragma unroll
            for (int e = 0; e < L; e++) sum[e] = (sum[e] + part[0][lane][e]) + (part[1][lane][e] + part[2][lane][e]);
            put(g0 + r);
        }
        __syncthreads();
    }
}

constexpr int64_t kEmbedRows = 1 << 28, kEmbedCols = 1 << 20, kEmbedTokens = INT32_MAX;

bool embed_in_range(int64_t n, int64_t R, int64_t D, int dtype) {
    return n >= 1 && n <= kEmbedTokens && R >= 1 && R <= kEmbedRows && D >= 1 && D <= kEmbedCols && dtype >= SNHIP_F32 &&
           dtype <= SNHIP_F16;
}

// Sizes of a call, and its workspace's parts where there is one. Returns its bytes.
int64_t embed_plan(EmbedP* a, const void* ids, bool wide, int64_t n, int64_t R, int64_t D, float scale, int dtype, char* ws) {
    a->ids = ids;
    a->wide = wide;
    a->n = n, a->R = R, a->D = D;
    a->scale = scale;
    int64_t tiles = n <= kEmbedAlone ? 1 : (n + kEmbedTile - 1) / kEmbedTile;
    if (tiles > kEmbedTiles) tiles = kEmbedTiles;
    a->tile = (int)((n + tiles - 1) / tiles);
    a->tiles = (int)((n + a->tile - 1) / a->tile);
    int bits = 1;
    while (R >> bits) bits++;                    // of R itself, which stands for no row
    a->passes = (bits + kEmbedBits - 1) / kEmbedBits;
    a->bits = (bits + a->passes - 1) / a->passes;
    const int64_t lane = dtype == SNHIP_F32 ? 4 : 8, lanes = 64 * lane, slices = (D + lanes - 1) / lanes;
    a->lanes = 6;
    while (a->lanes > 0 && D <= lane << (a->lanes - 1)) a->lanes--;
    // Enough waves to fill the card, and runs as long as they may be; past 2^23 groups and
    // slices longer ones, so that a grid (of fewer than 2^32 threads) holds them.
    int64_t group = (n * slices >> (6 - a->lanes)) / 4096;
    group = group < 8 ? 8 : group > 64 ? 64 : group;
    if (n * slices / group >= 1 << 23) group = (n * slices >> 22) + 1;
    a->group = (int)group;
    a->groups = (n + a->group - 1) / a->group;
    a->ld = (D + 7) / 8 * 8;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        char* p = ws + at;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    a->part = reinterpret_cast<float*>(take(a->groups * 2 * a->ld * 4));
    for (int i = 0; i < 2; i++) {
        a->key[i] = reinterpret_cast<unsigned*>(take(4 * n));
        a->at[i] = reinterpret_cast<int*>(take(4 * n));
    }
    a->count = reinterpret_cast<int*>(take(a->tiles > 1 ? (int64_t)a->tiles * (4 << a->bits) : 0));
    return at;
}

bool embed_vec(const void* x, const void* y, int64_t D, int dtype) {
    return (reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % 16 == 0 && D % (dtype == SNHIP_F32 ? 4 : 8) == 0;
}

template <typename T> snhip_status embed_fwd_t(const EmbedP& a, const void* table, void* y, bool vec, hipStream_t st) {
    const int64_t cols = (a.D + kLane<T> - 1) / kLane<T>, per = cols >= 1024 ? 1 : 1024 / cols;
    const int64_t blocks = (a.n + per - 1) / per, grid = blocks < (1 << 20) ? blocks : 1 << 20;
    if (vec) k_embed<T, true><<<(unsigned)grid, 256, 0, st>>>(a, (const T*)table, (T*)y, (int)per);
    else k_embed<T, false><<<(unsigned)grid, 256, 0, st>>>(a, (const T*)table, (T*)y, (int)per);
    SNHIP_CHECK(hipGetLastError());
    return SNHIP_OK;
}

template <typename T> snhip_status embed_bwd_t(const EmbedP& a, const void* dy, void* out, bool vec, hipStream_t st) {
    const int64_t lanes = 64 * kLane<T>, slices = (a.D + lanes - 1) / lanes, subs = 64 >> a.lanes,
                  tasks = ((a.groups + subs - 1) / subs * slices + 3) / 4, blocks = tasks + (a.R + 63) / 64;
    auto go = [&](auto v, auto narrow) -> snhip_status {
        constexpr bool VEC = decltype(v)::value, NARROW = decltype(narrow)::value;
        k_embed_grad<T, VEC, NARROW><<<(unsigned)blocks, 256, 0, st>>>(a, (const T*)dy, (T*)out, (int)slices, tasks);
        SNHIP_CHECK(hipGetLastError());
        if (a.groups > 1) {
            k_embed_join<T, VEC, NARROW><<<(unsigned)((a.groups + 3) / 4 * slices), 256, 0, st>>>(a, (T*)out, (int)slices);
            SNHIP_CHECK(hipGetLastError());
        }
        return SNHIP_OK;
    };
    typedef std::true_type yes;
    typedef std::false_type no;
    if (a.lanes < 6) return vec ? go(yes(), yes()) : go(no(), yes());
    return vec ? go(yes(), no()) : go(no(), no());
}

}  // namespace
}  // namespace snhip

using namespace snhip;

extern "C" {

snhip_status snhip_op_embed_fwd_dev(const void* table, const void* ids, int32_t wide, void* y, int64_t n, int64_t R,
                                    int64_t D, float scale, int32_t dtype, void* stream) {
    if (!table || !ids || !y || !embed_in_range(n, R, D, dtype)) return SNHIP_E_INVAL;
    EmbedP a = {};
    a.ids = ids, a.wide = wide != 0, a.n = n, a.R = R, a.D = D, a.scale = scale;
    const bool vec = embed_vec(table, y, D, dtype);
    const hipStream_t st = as_stream(stream);
    return dtype == SNHIP_F32    ? embed_fwd_t<float>(a, table, y, vec, st)
           : dtype == SNHIP_BF16 ? embed_fwd_t<__bf16>(a, table, y, vec, st)
                                 : embed_fwd_t<_Float16>(a, table, y, vec, st);
}

int64_t snhip_op_embed_bwd_bytes(int64_t n, int64_t R, int64_t D, int32_t dtype) {
    if (!embed_in_range(n, R, D, dtype)) return 0;
    EmbedP a;
    return embed_plan(&a, nullptr, false, n, R, D, 1.f, dtype, nullptr);
}

snhip_status snhip_op_embed_bwd_dev(const void* dy, const void* ids, int32_t wide, void* dtable, void* ws, int64_t n, int64_t R,
                                    int64_t D, float scale, int32_t dtype, void* stream) {
    if (!dy || !ids || !dtable || !ws || reinterpret_cast<uintptr_t>(ws) % 16 || !embed_in_range(n, R, D, dtype))
        return SNHIP_E_INVAL;
    EmbedP a;
    embed_plan(&a, ids, wide != 0, n, R, D, scale, dtype, static_cast<char*>(ws));
    const hipStream_t st = as_stream(stream);
    auto sort = [&](int p0, int p1) {
        if (a.bits < kEmbedBits) k_embed_sort<1><<<(unsigned)a.tiles, 64 * kEmbedWaves, 0, st>>>(a, p0, p1);
        else k_embed_sort<2><<<(unsigned)a.tiles, 64 * kEmbedWaves, 0, st>>>(a, p0, p1);
        return hipGetLastError();
    };
    if (a.tiles == 1) {
        SNHIP_CHECK(sort(0, a.passes));
    } else {
        for (int p = 0; p < a.passes; p++) {
            k_embed_count<<<(unsigned)a.tiles, 1024, 0, st>>>(a, p);
            SNHIP_CHECK(hipGetLastError());
            SNHIP_CHECK(sort(p, p + 1));
        }
    }
    const bool vec = embed_vec(dy, dtable, D, dtype);
    return dtype == SNHIP_F32    ? embed_bwd_t<float>(a, dy, dtable, vec, st)
           : dtype == SNHIP_BF16 ? embed_bwd_t<__bf16>(a, dy, dtable, vec, st)
                                 : embed_bwd_t<_Float16>(a, dy, dtable, vec, st);
}

}  // extern "C"
