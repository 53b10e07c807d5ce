// Sampling of logits rows with temperature, top-k, top-p and min-p from given random numbers.
//
// Definition (exact: every mass is an integer, so that the token is the same however the work is
// split):
//   m    = max_i l_i (a NaN counts as -inf);  w_i = rint(2^44 exp((l_i - m) / T)), in 64 bits
//   order: by l, the largest first, of equal ones the lowest index first
//   K    = the first top_k ids in order (all: top_k <= 0), of those the ones with w_i >= min_p 2^44
//   N    = the ids of K in order up to the first at which their mass reaches
//          max(1, ceil(top_p W)), W the mass of K (all of K: top_p >= 1)
//   r    = floor(u M), M the mass of N (in double, at most M - 1)
//   token = the smallest id of N whose inclusive mass, in the order of ids, exceeds r; -1 where no
//          id has mass.
// The exponential is evaluated in 64 bits (a relative error of some 2^-50), so that w_i is the
// definition's up to one unit of 2^44 in rare cases, and a token's chance of being another one
// some 2^-44 an id. V < 2^20 keeps every sum below 2^64.
//
// What bounds it: few rows by the launches and the chain of a row's last workgroup, many rows by the
// logits' bytes and the 64-bit exponentials. The steps:
//   no top-k, no top-p   1. the maximum  2. masses by tile (a pass of a workgroup's loads); the tile
//                        that holds r and the id within it
//   top-p                1. the maximum  2. a histogram of masses by logit  3. masses by tile of the
//                        ids that are surely in N, and a list of the ids of the bin in which N ends;
//                        N's end in that list, then the tile as above
//   top-k                1. the maxima of runs of 32 logits: the top_k-th largest of those, and the logit
//                        at which masses end, bound the top_k-th logit from below  2. a list of the ids
//                        above the bound, from the runs that reach it; the ends of K and N in it, and the
//                        draw
// Top-p's third step is done so too where few runs reach N's end.
// Rows of a large vocabulary are cut into blocks of a workgroup each, a launch a step, and what follows
// the last step's pass is done by the row's last workgroup to arrive. Small vocabularies take one
// launch, a workgroup a row. A list that does not fit in LDS is read from the workspace (top-p of flat
// rows, where thousands of ids have the mass at which N ends: 33 rows of 151936 logits of N(0, 1) 54 us, of
// N(0, 4^2) 33), and where it does not fit there either, or top_k is in the thousands, the choice is made
// from the row itself, some ten passes of a workgroup (top_k = 5000 of 151936: 341 to 368 us). Equal logits
// under top-p are the slowest, their masses added to one word: 2.2 ms, 33 rows 3.5.
#include "common.hpp"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace efm {

int prefill_cus();

constexpr int kFiltThreads = 256;                // of a block of a row
constexpr int kFiltListThreads = 512;
constexpr int kFiltMaxVocab = 1 << 20;
constexpr double kFiltOne = 17592186044416.0;   // 2^44
constexpr int kFiltBlocks = 128;                 // of a row, at most
constexpr int kFiltTiles = 1024;                 // of a row: 1024 logits or more each
constexpr int kFiltMassBins = 1024, kFiltBinsPerOctave = 22;   // masses from 2^0 to below 2^-46
constexpr int kFiltRuns = 5120;                  // runs of neighbouring logits whose maxima are kept, at most
constexpr int kFiltRunBins = 1024;
constexpr int kFiltHeld = 1024, kFiltHeldK = 2048;   // entries of a list that a workgroup holds with their masses; top-k
constexpr int kFiltLong = 8192;                  // entries of a row's list in the workspace
constexpr int kFiltOneVocab = 16384;             // vocabularies of one launch

// One row's part of the workspace.
struct FiltRow {
    unsigned long long mass_bins[kFiltMassBins];
    uint32_t counter, count;
    uint32_t pad[2];
    float bmax[kFiltBlocks];
    unsigned long long tile[kFiltTiles];
    unsigned long long list[kFiltLong];   // key << 32 | id
    float run[kFiltRuns];
};
static_assert(sizeof(FiltRow) % 16 == 0, "rows of the workspace stay aligned");

struct FiltArgs {
    const void* logits;
    int64_t stride;
    int V, top_k;
    float top_p;
    double to_log2;       // log2(e) / T
    float to_log2f, low;  // a logit with (l - m) to_log2f <= low has no mass that counts
    float reach;          // low / to_log2f
    float to_bin;         // bins a unit of m - l
    uint64_t min_mass;    // max(1, ceil(min_p 2^44))
    const float* u;
    int32_t* out;
    FiltRow* ws;
    int blocks, chunk;    // of a row; logits of a block
    int run_lanes, runs;  // 16-byte loads of a run; runs of a row
};

enum { kFiltAll, kFiltTopP, kFiltTopK };

// w of a logit, m the row's largest. 2^t, t = (l - m) log2(e) / T, is 2^n 2^f with the series of
// exp(f ln 2), |f| <= 1/2: the term after the last is below 2^-52. Adding 1.5 2^52 rounds t to an integer,
// and a last step to p 2^(n + 44) + 2^52 leaves w in the low bits. Without branches, so that a thread's
// logits go through side by side (33 rows of 151936: 15.1 -> 11.9 us for the masses by bin).
__device__ __forceinline__ uint64_t filt_mass(const FiltArgs& a, float l, float m) {
    const double t = l == m ? 0.0 : ((double)l - (double)m) * a.to_log2;
    const double near = t + 6755399441055744.0, f = t - (near - 6755399441055744.0);
    constexpr double c = 0.69314718055994530942, c2 = c * c / 2, c3 = c2 * c / 3, c4 = c3 * c / 4, c5 = c4 * c / 5, c6 = c5 * c / 6,
                     c7 = c6 * c / 7, c8 = c7 * c / 8, c9 = c8 * c / 9, c10 = c9 * c / 10, c11 = c10 * c / 11, c12 = c11 * c / 12;
    double p = c12;
    p = __builtin_fma(p, f, c11);
    p = __builtin_fma(p, f, c10);
    p = __builtin_fma(p, f, c9);
    p = __builtin_fma(p, f, c8);
    p = __builtin_fma(p, f, c7);
    p = __builtin_fma(p, f, c6);
    p = __builtin_fma(p, f, c5);
    p = __builtin_fma(p, f, c4);
    p = __builtin_fma(p, f, c3);
    p = __builtin_fma(p, f, c2);
    p = __builtin_fma(p, f, c);
    p = __builtin_fma(p, f, 1.0);
    const double scale = __builtin_bit_cast(double, (uint64_t)((uint32_t)__builtin_bit_cast(uint64_t, near) + 44u + 1023u) << 52);
    const uint64_t w = __builtin_bit_cast(uint64_t, __builtin_fma(p, scale, 4503599627370496.0)) & 0xfffffffffffffull;
    // fp32 decides what is far below (no 2^n is made of those); the largest is there even where it is infinite
    const bool counts = (l == m) | ((l - m) * a.to_log2f > a.low);
    return (counts & (w >= a.min_mass)) ? w : 0;
}

// Bin of a mass histogram, 0 for the largest logit; it rises as the logit falls.
__device__ __forceinline__ int filt_bin(const FiltArgs& a, float l, float m) {
    const float x = l == m ? 0.f : (m - l) * a.to_bin;
    return x < (float)(kFiltMassBins - 1) ? (int)x : kFiltMassBins - 1;
}

// Unsigned keys that order as the logits do (zeros of both signs alike), and back.
__device__ __forceinline__ uint32_t filt_key(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float filt_logit(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key); }

__device__ __forceinline__ float filt_clean(float l) { return l == l ? l : -INFINITY; }

constexpr int kFiltBatch = 4;   // 16-byte loads of a thread under way

// 16 bytes of a row's logits from i on, -inf past the end. A row that does not start on 16 bytes, as three of four (bf16: seven
// of eight) do where the vocabulary is odd, is loaded an element at a time (33 rows of 151935 against 151936, fp32 and bf16: top-k 17 | 13 and
// 18 | 13 us, top-p 43 | 37 and 54 | 39, min-p 19 | 12 and 23 | 13).
template <bool BF16>
__device__ __forceinline__ uint4 filt_raw(const void* row, bool aligned, int i, int end) {
    constexpr int E = BF16 ? 8 : 4;
    if (aligned && i + E <= end) return *reinterpret_cast<const uint4*>(static_cast<const char*>(row) + (int64_t)i * (BF16 ? 2 : 4));
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (BF16) {
            const uint16_t* const p = static_cast<const uint16_t*>(row);
            const uint32_t lo = i + 2 * e < end ? p[i + 2 * e] : 0xff80u, hi = i + 2 * e + 1 < end ? p[i + 2 * e + 1] : 0xff80u;
            w[e] = lo | hi << 16;
        } else {
            w[e] = i + e < end ? static_cast<const uint32_t*>(row)[i + e] : 0xff800000u;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool BF16>
__device__ __forceinline__ void filt_unpack(const uint4& x, float* l) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if constexpr (BF16) l[2 * e] = lo_f32(w[e]), l[2 * e + 1] = hi_f32(w[e]);
        else l[e] = __uint_as_float(w[e]);
    }
}

// A row's logits [first, end), first a multiple of a tile: f(tile of the range, first id, the thread's
// E logits as they are (-inf past the end), how many of them there are), by all threads together.
template <int NT, bool BF16, typename F>
__device__ __forceinline__ void filt_tiles(const void* row, int first, int end, F f) {
    constexpr int E = BF16 ? 8 : 4, U = kFiltBatch, TILE = E * NT;
    const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
    for (int t0 = 0; first + t0 * TILE < end; t0 += U) {
        uint4 x[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int i = first + (t0 + j) * TILE + (int)threadIdx.x * E;
            x[j] = filt_raw<BF16>(row, aligned, i, end);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int i = first + (t0 + j) * TILE + (int)threadIdx.x * E;
            if (first + (t0 + j) * TILE >= end) break;
            float l[E];
            filt_unpack<BF16>(x[j], l);
            f(t0 + j, i, l, min(max(end - i, 0), E));
        }
    }
}

// A 64-bit value moved across lanes, 0 where the source is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t filt_dpp(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return (uint64_t)hi << 32 | lo;
}

// Inclusive sums over the lanes of a wave: shifts by 1, 2, 4 and 8 within 16 lanes, then the ends of
// the rows of 16.
__device__ __forceinline__ uint64_t filt_wave_scan(uint64_t v) {
    v += filt_dpp<0x111, 0xf>(v);
    v += filt_dpp<0x112, 0xf>(v);
    v += filt_dpp<0x114, 0xf>(v);
    v += filt_dpp<0x118, 0xf>(v);
    v += filt_dpp<0x142, 0xa>(v);
    v += filt_dpp<0x143, 0xc>(v);
    return v;
}

// Their last, in every lane.
__device__ __forceinline__ uint64_t filt_last_lane(uint64_t v) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}

template <int NT>
struct FiltShared {
    unsigned long long red[NT / kWave];
    unsigned long long sel[2];
    unsigned long long bins[2][256];
    uint32_t counts[2][256];
    float redf[2][NT / kWave];
    uint32_t flag, found[3];
};

// Sum of the values of the threads before this one, and of all.
template <int NT>
__device__ __forceinline__ uint64_t filt_scan(uint64_t v, FiltShared<NT>& s, uint64_t* total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint64_t incl = filt_wave_scan(v);
    __syncthreads();
    if (lane == kWave - 1) s.red[wave] = incl;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / kWave; ++w) {
        if (w < wave) before += s.red[w];
        all += s.red[w];
    }
    *total = all;
    return before + incl - v;
}

template <int NT>
__device__ __forceinline__ uint64_t filt_sum(uint64_t v, FiltShared<NT>& s) {
    uint64_t all;
    filt_scan<NT>(v, s, &all);
    return all;
}

// The largest m and the smallest *least of the workgroup.
template <int NT>
__device__ __forceinline__ float filt_max(float m, float* least, FiltShared<NT>& s) {
    m = wave_max_uniform(m);
    const float n = wave_max_uniform(-*least);
    if (threadIdx.x % kWave == 0) s.redf[0][threadIdx.x / kWave] = m, s.redf[1][threadIdx.x / kWave] = n;
    __syncthreads();
    m = s.redf[0][0];
    float z = s.redf[1][0];
#pragma unroll
    for (int w = 1; w < NT / kWave; ++w) m = fmaxf(m, s.redf[0][w]), z = fmaxf(z, s.redf[1][w]);
    *least = -z;
    return m;
}

// What the choices so far keep: keys above `key`, and of those equal to it the ids up to `id`.
struct FiltCut {
    uint32_t key;
    int id;
    __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= id); }
};

// floor(u M), at most M - 1. M may be anything below 2^64; 2^64 - 2^11 is the largest double there.
__device__ __forceinline__ uint64_t filt_draw(float u, uint64_t M) {
    const double x = (double)u * (double)M;
    const uint64_t r = x > 0.0 ? (uint64_t)__builtin_fmin(x, 18446744073709549568.0) : 0ull;
    return r < M ? r : M - 1;
}

__device__ __forceinline__ uint64_t filt_need(float top_p, uint64_t W) {
    const uint64_t need = (uint64_t)__builtin_ceil((double)top_p * (double)W);
    return need < 1 ? 1 : need > W ? W : need;
}

// Last of the 2^shift values from lo on, no further than hi. The difference is compared: lo + 2^shift may pass 2^32, where
// the lowest logits' keys lie.
constexpr uint32_t filt_bin_end(uint32_t lo, uint32_t hi, int shift) {
    const uint32_t past = (1u << shift) - 1;
    return hi - lo > past ? lo + past : hi;
}
static_assert(filt_bin_end(0xff5fffffu, 0xff7fffffu, 24) == 0xff7fffffu && filt_bin_end(0xff5fffffu, 0xffffffffu, 16) == 0xff60fffeu &&
              filt_bin_end(5, 5, 0) == 5 && filt_bin_end(0, ~0u, 24) == 0xffffffu);

// The entry that holds unit `rank` of the weights of a source, each(f): f(id, key, whether it is one, weight()) by whole
// waves where ROW; in the sampler's order (keys of [low, high]), or by id alone (ids of [low, high]). The range that may
// hold it is cut into 256 bins until one entry is left, four times for keys and three for the ids of equal keys at most;
// weights outside it are not asked for. A rank that the sum of the weights does not reach keeps every entry.
template <int NT, bool ROW, typename Each>
__device__ __forceinline__ FiltCut filt_pick(bool by_id, uint32_t low, uint32_t high, uint64_t rank, const FiltArgs& a, FiltShared<NT>& s,
                                             Each each) {
    const int tid = threadIdx.x;
    bool ids = by_id;
    uint32_t lo = by_id ? low : ~high, hi = by_id ? high : ~low, tie = 0;   // of ~key, or of the ids with ~key = tie
    __syncthreads();
    if (tid < 256) s.bins[0][tid] = 0, s.counts[0][tid] = 0;
    __syncthreads();
#pragma unroll 1
    for (int step = 0; step < 8; ++step) {
        const int b = step & 1, bits = 32 - __builtin_clz(hi - lo | 1u), shift = max(bits - 8, 0);
        auto value = [&](int i, uint32_t k) { return ids ? (uint32_t)i : ~k; };
        auto active = [&](int i, uint32_t k) { return value(i, k) >= lo && value(i, k) <= hi && (!ids || by_id || ~k == tie); };
        each([&](int i, uint32_t k, bool in, auto weight) {
            uint64_t w = 0;
            if (in && active(i, k)) w = weight();
            const uint32_t bin = (value(i, k) - lo) >> shift;
            if constexpr (ROW) {   // a wave whose entries share a bin, as equal logits do, adds once
                const uint64_t lanes = __ballot(w != 0);
                if (lanes == 0) return;
                const uint32_t bin0 = (uint32_t)__builtin_amdgcn_readlane((int)bin, __builtin_ctzll(lanes));
                if (__ballot(w != 0 && bin != bin0) == 0) {
                    w = filt_last_lane(filt_wave_scan(w));
                    if (tid % kWave == 0) {
                        atomicAdd(&s.bins[b][bin0 & 255u], (unsigned long long)w);
                        atomicAdd(&s.counts[b][bin0 & 255u], (uint32_t)__builtin_popcountll(lanes));
                    }
                    return;
                }
            }
            if (w == 0) return;
            atomicAdd(&s.bins[b][bin & 255u], (unsigned long long)w);
            atomicAdd(&s.counts[b][bin & 255u], 1u);
        });
        if (tid < 256) s.bins[1 - b][tid] = 0, s.counts[1 - b][tid] = 0;
        __syncthreads();
        uint64_t all;
        const uint64_t own = tid < 256 ? s.bins[b][tid] : 0ull, excl = filt_scan<NT>(own, s, &all);
        if (all <= rank) return FiltCut{0u, a.V};   // at the first step, if at all
        if (excl <= rank && rank - excl < own) s.sel[0] = tid, s.sel[1] = excl, s.found[2] = s.counts[b][tid];
        __syncthreads();
        rank -= s.sel[1];
        lo += ((uint32_t)s.sel[0] & 255u) << shift, hi = filt_bin_end(lo, hi, shift);
        if (s.found[2] == 1) {
            each([&](int i, uint32_t k, bool in, auto weight) {
                if (in && active(i, k) && weight() != 0) s.found[0] = k, s.found[1] = (uint32_t)i;
            });
            __syncthreads();
            return FiltCut{s.found[0], (int)s.found[1]};
        }
        if (shift == 0) {   // equal keys: by id
            if (ids) break;
            ids = true, tie = lo, lo = 0, hi = (uint32_t)a.V - 1;
        }
    }
    return FiltCut{~0u, 0};
}

// K, N and the draw over a list, each(f): f(id, key, mass), `count` entries with keys of [low, high]. W: the
// mass that top_p is of (0: K's).
template <int NT, typename Each>
__device__ __forceinline__ int filt_choose(const FiltArgs& a, uint32_t low, uint32_t high, uint32_t count, uint64_t W, float u, FiltShared<NT>& s,
                                           Each each) {
    FiltCut kept{0u, a.V};
    if ((uint32_t)a.top_k < count)
        kept = filt_pick<NT, false>(false, low, high, (uint64_t)a.top_k - 1, a, s,
                                    [&](auto f) { each([&](int i, uint32_t k, uint64_t) { f(i, k, true, [] { return (uint64_t)1; }); }); });
    auto left = [&](auto f) { each([&](int i, uint32_t k, uint64_t w) { f(i, k, kept.keeps(k, i), [=] { return w; }); }); };
    auto total = [&]() {
        uint64_t sum = 0;
        each([&](int i, uint32_t k, uint64_t w) { sum += kept.keeps(k, i) ? w : 0ull; });
        return filt_sum<NT>(sum, s);
    };
    uint64_t M = total();
    if (a.top_p < 1.0f) {
        kept = filt_pick<NT, false>(false, low, high, filt_need(a.top_p, W != 0 ? W : M) - 1, a, s, left);
        M = total();
    }
    return filt_pick<NT, false>(true, 0, (uint32_t)a.V - 1, filt_draw(u, M), a, s, left).id;
}

// The same where every thread has an entry at most (x: ~key << 32 | id, and its mass w), by ranks: the
// entries before one are counted, it moves to that place, and K, N and the draw are prefix sums. W: the
// mass that top_p is of (0: K's). order and mass are LDS of NT entries each.
template <int NT>
__device__ __forceinline__ int filt_choose_held(const FiltArgs& a, uint32_t count, unsigned long long x, uint64_t w, uint64_t W, float u,
                                                unsigned long long* order, unsigned long long* mass, FiltShared<NT>& s) {
    const int tid = threadIdx.x, wave0 = tid / kWave * kWave;
    uint32_t* const ids = reinterpret_cast<uint32_t*>(order);
    __syncthreads();
    order[tid] = x;   // ~0 for threads without one
    __syncthreads();
    if (a.top_k < (int)count || a.top_p < 1.0f) {
        int at = 0;
        if (wave0 < (int)count)
            for (int j = 0; j < (int)count; j += 16) {
                ulonglong2 y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = reinterpret_cast<const ulonglong2*>(order + j)[i];
#pragma unroll
                for (int i = 0; i < 8; ++i) at += (y[i].x < x) + (y[i].y < x);
            }
        __syncthreads();
        if (tid < (int)count) order[at] = x, mass[at] = w;
        __syncthreads();
        x = order[tid];
        w = tid < (int)count && tid < a.top_k ? mass[tid] : 0ull;
        if (a.top_p < 1.0f) {
            uint64_t all;
            const uint64_t before = filt_scan<NT>(w, s, &all);
            if (before >= filt_need(a.top_p, W != 0 ? W : all)) w = 0;
        }
    }
    // what has mass, in the order of ids
    const uint32_t id = w != 0 ? (uint32_t)x : ~0u;
    __syncthreads();
    ids[tid] = id;
    mass[tid] = 0;
    __syncthreads();
    int at = 0;
    if (wave0 < (int)count)
        for (int j = 0; j < (int)count; j += 16) {
            uint4 y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = reinterpret_cast<const uint4*>(ids + j)[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) at += (y[i].x < id) + (y[i].y < id) + (y[i].z < id) + (y[i].w < id);
        }
    if (w != 0) ids[NT + at] = id, mass[at] = w;
    __syncthreads();
    uint64_t M;
    const uint64_t own = mass[tid], excl = filt_scan<NT>(own, s, &M), r = filt_draw(u, M);
    if (excl <= r && r - excl < own) s.found[0] = ids[NT + tid];
    __syncthreads();
    return (int)s.found[0];
}

// Keys that a bin's logits can have, with 2^-20 of each of the terms to spare.
__device__ __forceinline__ void filt_bin_keys(const FiltArgs& a, float m, int bin, uint32_t* from, uint32_t* to) {
    *from = 0u, *to = filt_key(m);
    if (!(m < INFINITY)) return;
    const double spare = 0x1p-20 * __builtin_fabs((double)m), one = 1.0 / (double)a.to_bin;
    if (bin < kFiltMassBins - 1) *from = filt_key((float)((double)m - (bin + 1) * one * (1.0 + 0x1p-20) - spare));
    *to = min(*to, filt_key((float)((double)m - bin * one * (1.0 - 0x1p-20) + spare)));
}

// The draw from the masses by tile, in `tile`, of what the cut keeps.
template <int NT, bool BF16>
__device__ __forceinline__ int filt_tile_draw(const FiltArgs& a, const void* row, float m, float u, const FiltCut& kept, const unsigned long long* tile,
                                              FiltShared<NT>& s) {
    constexpr int E = BF16 ? 8 : 4, TILE = E * NT, PER = kFiltTiles / NT;
    const int tid = threadIdx.x;
    uint64_t own = 0, M, h[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) own += h[i] = tile[tid * PER + i];
    uint64_t excl = filt_scan<NT>(own, s, &M);
    const uint64_t r = filt_draw(u, M);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (excl <= r && r - excl < h[i]) s.sel[0] = tid * PER + i, s.sel[1] = excl;
        excl += h[i];
    }
    __syncthreads();
    const int t = (int)min((uint32_t)s.sel[0], (uint32_t)(a.V - 1) / TILE);
    const uint64_t rest = r - s.sel[1];
    filt_tiles<NT, BF16>(row, t * TILE, min(t * TILE + TILE, a.V), [&](int, int i, const float (&l)[E], int) {
        uint64_t y[E], sum = 0, all;
#pragma unroll
        for (int e = 0; e < E; ++e) sum += y[e] = kept.keeps(filt_key(filt_clean(l[e])), i + e) ? filt_mass(a, filt_clean(l[e]), m) : 0ull;
        uint64_t at = filt_scan<NT>(sum, s, &all);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (at <= rest && rest - at < y[e]) s.found[0] = i + e;
            at += y[e];
        }
    });
    __syncthreads();
    return (int)s.found[0];
}

// The choice where the list does not fit, from the row itself, a pass a step of filt_pick. bin < 0: from the start, of
// what may have mass; otherwise N ends in that bin of masses, `above` is the mass of the bins before it and `tile` theirs by tile.
template <int NT, bool BF16>
__device__ __forceinline__ int filt_choose_row(const FiltArgs& a, const void* row, float m, float u, int bin, uint64_t above, uint64_t W,
                                               unsigned long long* tile, FiltShared<NT>& s) {
    constexpr int E = BF16 ? 8 : 4;
    // what may have mass, with 2^-20 of each of the terms to spare
    const uint32_t least = filt_key(m + a.reach * (1.f + 0x1p-20f) - (m < INFINITY ? 0x1p-20f * fabsf(m) : 0.f));
    FiltCut kept{bin < 0 ? least : 0u, a.V};
    uint64_t sum = 0;
    bool tiles = false;   // the pass adds masses by tile
    auto pass = [&](auto f) {
        filt_tiles<NT, BF16>(row, 0, a.V, [&](int t, int i, const float (&l)[E], int n) {
            uint64_t y = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = filt_clean(l[e]);
                const uint32_t k = filt_key(x);
                y += f(i + e, k, x, e < n && kept.keeps(k, i + e) && (bin < 0 || filt_bin(a, x, m) == bin));
            }
            if (!tiles) return;
            y = filt_last_lane(filt_wave_scan(y));
            if (threadIdx.x % kWave == 0 && y != 0) atomicAdd(&tile[t], (unsigned long long)y);
        });
    };
    auto masses = [&](auto f) {
        pass([&](int i, uint32_t k, float x, bool in) {
            f(i, k, in, [&] { return filt_mass(a, x, m); });
            return 0ull;
        });
    };
    const uint32_t high = filt_key(m);
    if (bin >= 0) {
        uint32_t from, to;
        filt_bin_keys(a, m, bin, &from, &to);
        kept = filt_pick<NT, true>(false, from, to, filt_need(a.top_p, W) - 1 - above, a, s, masses);
    } else {
        for (int i = threadIdx.x; i < kFiltTiles; i += NT) tile[i] = 0;
        if (a.top_k < a.V)
            kept = filt_pick<NT, true>(false, least, high, (uint64_t)a.top_k - 1, a, s, [&](auto f) {
                pass([&](int i, uint32_t k, float, bool in) {
                    f(i, k, in, [] { return (uint64_t)1; });
                    return 0ull;
                });
            });
        if (a.top_p < 1.0f) {
            pass([&](int, uint32_t, float x, bool in) {
                if (in) sum += filt_mass(a, x, m);
                return 0ull;
            });
            W = filt_sum<NT>(sum, s);
            kept = filt_pick<NT, true>(false, kept.key, high, filt_need(a.top_p, W) - 1, a, s, masses);
        }
    }
    tiles = true;
    pass([&](int, uint32_t, float x, bool in) { return in ? filt_mass(a, x, m) : (uint64_t)0; });
    __syncthreads();
    return filt_tile_draw<NT, BF16>(a, row, m, u, kept, tile, s);
}

// Top-k: what a logit has to reach to be listed. Logits fall into bins of equal width from the row's
// maximum down to the smallest maximum of a run, or to where a logit has no mass if that is higher, and
// those of the bins down to the one at which the runs are top_k are listed; where that is the last one,
// all that has mass. (Bins down to the smallest maximum whatever it is: with a few ids masked by -1e4 or
// less all that matters is in one bin, a row of 151936 and top_k 50 329 us instead of 12.)
struct FiltBound {
    float m, least;   // the row's maximum; listed from least on: one comparison a logit, which a NaN fails
    // Logits up to `far` below m, with 2^-22 of both to spare for the roundings by which far and the distances were found
    // (listing more is no mistake); never -inf.
    __device__ __forceinline__ FiltBound(float m, float far) : m(m) {
        const float spare = m < INFINITY ? 0x1p-22f * (fabsf(m) + far) : 0.f;
        least = fmaxf(m - (far + spare), -FLT_MAX);
    }
    __device__ __forceinline__ bool takes(float l) const { return l >= least; }
};

// From the maxima of the row's runs; pick(run) for the runs that hold such logits. What would be in the last bin is not
// counted but added to words behind the bins that nothing reads: thousands of runs may be in it, and additions to one word
// go one at a time (151936 logits, top-k 50, min-p 0.02: 9.3 -> 13.3 us; a branch around them: 2000 logits 8.0 -> 8.5).
template <int NT, typename Pick>
__device__ __forceinline__ FiltBound filt_bound(const FiltArgs& a, const float* run, uint32_t* bins, FiltShared<NT>& s, Pick pick) {
    constexpr int PER = kFiltRunBins / NT, HELD = kFiltRuns / NT;
    const int tid = threadIdx.x;
    float x[HELD], m = -INFINITY, least = INFINITY;
#pragma unroll
    for (int i = 0; i < HELD; ++i) x[i] = run[min(i * NT + tid, a.runs - 1)];
#pragma unroll
    for (int i = 0; i < PER; ++i) bins[i * NT + tid] = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        x[i] = i * NT + tid < a.runs ? x[i] : -INFINITY;
        m = fmaxf(m, x[i]);
        least = x[i] > -INFINITY ? fminf(least, x[i]) : least;
    }
    m = filt_max<NT>(m, &least, s);
    least = fmaxf(least, m + a.reach);
    // few runs for so large a top_k, equal runs or infinite ones: all that has mass is listed
    float far = -a.reach;
    const float width = (float)(kFiltRunBins - 1) / (m - least);
    if (a.top_k <= a.runs && width < INFINITY && width > 0.f) {
#pragma unroll
        for (int i = 0; i < HELD; ++i)
            if (i * NT < a.runs) {
                const float bin = (m - x[i]) * width;
                atomicAdd(&bins[bin < kFiltRunBins - 1 ? (int)bin : kFiltRunBins + tid % kWave], 1u);
            }
        __syncthreads();
        uint32_t own = 0, c[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) own += c[i] = bins[tid * PER + i];
        uint64_t all, excl = filt_scan<NT>(own, s, &all);
        const uint64_t rank = (uint64_t)a.top_k - 1;
        if (all > rank) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (excl <= rank && rank - excl < c[i]) s.sel[0] = tid * PER + i;
                excl += c[i];
            }
            __syncthreads();
            far = (float)((int)s.sel[0] + 1) / width;
        }
    }
    const FiltBound b(m, far);
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (i * NT < a.runs && b.takes(x[i])) pick(i * NT + tid);
    return b;
}

// Top-p: the bin in which N ends. *above: the mass of the bins before it, *W: of all.
template <int NT>
__device__ __forceinline__ int filt_mass_cut(const FiltArgs& a, const unsigned long long* bins, FiltShared<NT>& s, uint64_t* above, uint64_t* W) {
    constexpr int PER = kFiltMassBins / NT;
    uint64_t h[PER], own = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) own += h[i] = bins[threadIdx.x * PER + i];
    uint64_t excl = filt_scan<NT>(own, s, W);
    const uint64_t rank = filt_need(a.top_p, *W) - 1;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (excl <= rank && rank - excl < h[i]) s.sel[0] = threadIdx.x * PER + i, s.sel[1] = excl;
        excl += h[i];
    }
    __syncthreads();
    *above = s.sel[1];
    return (int)s.sel[0];
}

// Shared memory of the last step: the list with its masses, and the tiles' masses.
template <int H>
struct FiltLast {
    static constexpr int kHeld = H;
    unsigned long long list[H];
    unsigned long long mass[H];
    unsigned long long tile[kFiltTiles];
    uint32_t count, base;
};

// The maximum of [first, end) and, where runs is not null, those of the row's runs in it.
template <int NT, bool BF16>
__device__ __forceinline__ float filt_maxima(const FiltArgs& a, const void* row, int first, int end, float* runs) {
    constexpr int E = BF16 ? 8 : 4;
    float m = -INFINITY;
    const int lanes = a.run_lanes, lg = __builtin_ctz(lanes);
    filt_tiles<NT, BF16>(row, first, end, [&](int, int i, const float (&l)[E], int) {
        float x = l[0];
#pragma unroll
        for (int e = 1; e < E; ++e) x = fmaxf(x, l[e]);
        x = fmaxf(x, -INFINITY);   // not a NaN
        m = fmaxf(m, x);
        if (runs == nullptr) return;
        if (lanes >= 2) x = fmaxf(x, dpp_f32<0xB1>(x));
        if (lanes >= 4) x = fmaxf(x, dpp_f32<0x4E>(x));
        if (lanes >= 8) x = fmaxf(x, dpp_f32<0x141>(x));
        if (lanes >= 16) x = fmaxf(x, dpp_f32<0x140>(x));
        if (lanes >= 32) x = fmaxf(x, __shfl_xor(x, 16, kWave));
        if (lanes >= 64) x = fmaxf(x, __shfl_xor(x, 32, kWave));
        const int r = (i / E) >> lg;
        if ((threadIdx.x & (lanes - 1)) == 0 && r < a.runs) runs[r] = x;
    });
    return m;
}

template <int NT, bool BF16>
__device__ __forceinline__ void filt_mass_bins(const FiltArgs& a, const void* row, int first, int end, float m, unsigned long long* bins) {
    constexpr int E = BF16 ? 8 : 4;
    filt_tiles<NT, BF16>(row, first, end, [&](int, int, const float (&l)[E], int) {
        uint64_t x[E];
        uint64_t any = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) any |= x[e] = filt_mass(a, filt_clean(l[e]), m);
        if (any == 0) return;
#pragma unroll
        for (int e = 0; e < E; ++e) atomicAdd(&bins[filt_bin(a, filt_clean(l[e]), m)], (unsigned long long)x[e]);
    });
}

// The last step's pass: top-k: ids within the bound are listed; top-p: masses of bins < bin by tile, ids
// of `bin` are listed; neither: masses by tile. Tiles count from the range's first. Most logits are below
// what any of that takes: one comparison each, and a NaN goes the careful way.
template <int NT, bool BF16, int MODE, typename Last>
__device__ __forceinline__ void filt_gather(const FiltArgs& a, const void* row, int first, int end, float m, int bin, const FiltBound& bound,
                                            Last& z) {
    constexpr int E = BF16 ? 8 : 4;
    auto enlist = [&](int i, float l) {
        const uint32_t at = atomicAdd(&z.count, 1u);
        if (at < Last::kHeld) z.list[at] = (unsigned long long)filt_key(l) << 32 | (uint32_t)i;
    };
    const float past = bin < kFiltMassBins - 1 ? (float)(bin + 1) : INFINITY;
    if constexpr (MODE == kFiltTopP) {
        // What is above the bin is listed too at first, if it fits: its masses then take full waves.
        filt_tiles<NT, BF16>(row, first, end, [&](int, int i, const float (&l)[E], int n) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < n && !((m - l[e]) * a.to_bin >= past)) enlist(i + e, filt_clean(l[e]));
        });
        __syncthreads();
        const uint32_t listed = z.count;
        __syncthreads();
        if (threadIdx.x == 0) z.count = 0;
        unsigned long long x[Last::kHeld / NT];
#pragma unroll
        for (int j = 0; j < Last::kHeld / NT; ++j) x[j] = z.list[j * NT + threadIdx.x];
        __syncthreads();
        if (listed <= Last::kHeld) {
#pragma unroll
            for (int j = 0; j < Last::kHeld / NT; ++j) {
                if (j * NT + threadIdx.x >= listed) break;
                const float l = filt_logit((uint32_t)(x[j] >> 32));
                if (filt_bin(a, l, m) == bin) z.list[atomicAdd(&z.count, 1u)] = x[j];
                else atomicAdd(&z.tile[((int)(uint32_t)x[j] - first) / (E * NT)], (unsigned long long)filt_mass(a, l, m));
            }
            return;
        }
    }
    filt_tiles<NT, BF16>(row, first, end, [&](int t, int i, const float (&l)[E], int n) {
        bool some = false;
#pragma unroll
        for (int e = 0; e < E; ++e)
            some |= MODE == kFiltTopK ? bound.takes(l[e]) : MODE == kFiltTopP ? !((m - l[e]) * a.to_bin >= past) : !((l[e] - m) * a.to_log2f <= a.low);
        if (MODE == kFiltTopK && some) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < n && bound.takes(l[e])) enlist(i + e, l[e]);
        }
        if constexpr (MODE != kFiltTopK) {
            if (!__any(some)) return;
            uint64_t y = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) {   // there is none past the end: -inf
                const float x = filt_clean(l[e]);
                const uint64_t w = filt_mass(a, x, m);
                if constexpr (MODE == kFiltTopP) {
                    const int b = filt_bin(a, x, m);
                    y += b < bin ? w : 0ull;
                    if (b == bin && e < n) enlist(i + e, x);
                } else {
                    y += w;
                }
            }
            y = filt_last_lane(filt_wave_scan(y));
            if (threadIdx.x % kWave == 0) atomicAdd(&z.tile[t], (unsigned long long)y);
        }
    });
}

// Lists the logits within the bound of n picked runs.
template <int NT, bool BF16, typename Last>
__device__ __forceinline__ void filt_list_runs(const FiltArgs& a, const void* row, const uint32_t* picked, int n, const FiltBound& bound, Last& z) {
    constexpr int E = BF16 ? 8 : 4;
    const int lg = __builtin_ctz(a.run_lanes), all = n << lg;
    const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
    for (int i0 = threadIdx.x; i0 < all; i0 += 4 * NT) {
        uint4 x[4];
        int at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = min(i0 + j * NT, all - 1);
            at[j] = (((int)picked[i >> lg] << lg) + (i & (a.run_lanes - 1))) * E;
            if (i0 + j * NT < all) x[j] = filt_raw<BF16>(row, aligned, at[j], a.V);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i0 + j * NT >= all) break;
            float l[E];
            filt_unpack<BF16>(x[j], l);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (at[j] + e < a.V && bound.takes(l[e])) {
                    const uint32_t to = atomicAdd(&z.count, 1u);
                    if (to < Last::kHeld) z.list[to] = (unsigned long long)filt_key(l[e]) << 32 | (uint32_t)(at[j] + e);
                }
            }
        }
    }
}

// The choice from a row's list (`count` entries, in z or in `list`) and its tiles' masses (in z.tile).
template <int NT, bool BF16, int MODE, typename Last>
__device__ __forceinline__ int filt_last(const FiltArgs& a, const void* row, float m, float u, int bin, uint64_t above, uint64_t W, uint32_t count,
                                         const unsigned long long* list, FiltShared<NT>& s, Last& z) {
    const int tid = threadIdx.x;
    const uint32_t high = filt_key(m);
    if (m == -INFINITY) return -1;
    if (MODE == kFiltTopP && list != nullptr && count > Last::kHeld && count <= kFiltLong) {
        // from the list in the workspace; masses of what is in question only
        auto each = [&](auto f) {
            constexpr int U = 8;
            for (uint32_t i0 = tid; i0 < count; i0 += U * NT) {
                unsigned long long x[U];
#pragma unroll
                for (int j = 0; j < U; ++j) x[j] = __hip_atomic_load(&list[min(i0 + j * NT, count - 1)], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                for (int j = 0; j < U; ++j)
                    if (i0 + j * NT < count)
                        f((int)(uint32_t)x[j], (uint32_t)(x[j] >> 32), true, [&] { return filt_mass(a, filt_logit((uint32_t)(x[j] >> 32)), m); });
            }
        };
        uint32_t from, to;
        filt_bin_keys(a, m, bin, &from, &to);
        const FiltCut kept = filt_pick<NT, false>(false, from, to, filt_need(a.top_p, W) - 1 - above, a, s, each);
        each([&](int i, uint32_t k, bool, auto weight) {
            if (kept.keeps(k, i) && i < a.V) atomicAdd(&z.tile[i / ((BF16 ? 8 : 4) * NT)], (unsigned long long)weight());
        });
        __syncthreads();
        return filt_tile_draw<NT, BF16>(a, row, m, u, kept, z.tile, s);
    }
    if (MODE != kFiltAll && count > Last::kHeld) return filt_choose_row<NT, BF16>(a, row, m, u, MODE == kFiltTopP ? bin : -1, above, W, z.tile, s);
    if (MODE == kFiltTopK && count <= NT) {
        unsigned long long x = tid < (int)count ? z.list[tid] : 0ull;
        const uint64_t mass = tid < (int)count ? filt_mass(a, filt_logit((uint32_t)(x >> 32)), m) : 0ull;
        x = tid < (int)count ? (unsigned long long)~(uint32_t)(x >> 32) << 32 | (uint32_t)x : ~0ull;
        return filt_choose_held<NT>(a, count, x, mass, W, u, z.list, z.mass, s);
    }
    uint32_t low = ~0u;
    for (uint32_t i = tid; i < count; i += NT) {
        const unsigned long long x = list != nullptr ? __hip_atomic_load(&list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : z.list[i];
        z.list[i] = x;
        z.mass[i] = filt_mass(a, filt_logit((uint32_t)(x >> 32)), m);
        low = min(low, (uint32_t)(x >> 32));
    }
    auto each = [&](auto f) {
        for (uint32_t i = tid; i < count; i += NT) f((int)(uint32_t)z.list[i], (uint32_t)(z.list[i] >> 32), (uint64_t)z.mass[i]);
    };
    if constexpr (MODE != kFiltAll) {   // the least key listed
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) low = min(low, (uint32_t)__shfl_xor((int)low, off, kWave));
        if (tid % kWave == 0) s.counts[0][tid / kWave] = low;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / kWave; ++w) low = min(low, s.counts[0][w]);
    }
    if constexpr (MODE == kFiltTopK) return filt_choose<NT>(a, low, high, count, W, u, s, each);
    constexpr int TILE = (BF16 ? 8 : 4) * NT;
    FiltCut kept{0u, a.V};
    if constexpr (MODE == kFiltTopP) {
        kept = filt_pick<NT, false>(false, low, high, filt_need(a.top_p, W) - 1 - above, a, s, [&](auto f) {
            each([&](int i, uint32_t k, uint64_t w) { f(i, k, true, [=] { return w; }); });
        });
        each([&](int i, uint32_t k, uint64_t w) {
            if (w != 0 && kept.keeps(k, i) && i < a.V) atomicAdd(&z.tile[i / TILE], (unsigned long long)w);
        });
        __syncthreads();
    }
    return filt_tile_draw<NT, BF16>(a, row, m, u, kept, z.tile, s);
}

template <bool BF16>
__device__ __forceinline__ const char* filt_row(const FiltArgs& a, unsigned r) {
    return static_cast<const char*>(a.logits) + (int64_t)r * a.stride * (BF16 ? 2 : 4);
}

// 1. Block maxima, and those of runs.
template <bool BF16>
__global__ __launch_bounds__(kFiltThreads) void filt_max_kernel(FiltArgs a) {
    __shared__ FiltShared<kFiltThreads> s;
    FiltRow& w = a.ws[blockIdx.y];
    const int first = blockIdx.x * a.chunk, end = min(first + a.chunk, a.V);
    float m = filt_maxima<kFiltThreads, BF16>(a, filt_row<BF16>(a, blockIdx.y), first, end, a.runs > 0 ? w.run : nullptr), least = 0.f;
    m = filt_max<kFiltThreads>(m, &least, s);
    if (threadIdx.x == 0) w.bmax[blockIdx.x] = m;
    if (blockIdx.x == 0) {   // what the next steps add to
        for (int i = threadIdx.x; i < kFiltMassBins; i += kFiltThreads) w.mass_bins[i] = 0;
        if (threadIdx.x == 0) w.counter = 0, w.count = 0;
    }
}

// The row's maximum, from its blocks'.
__device__ __forceinline__ float filt_row_max(const FiltArgs& a, const FiltRow& w, FiltShared<kFiltThreads>& s) {
    float least = 0.f;
    return filt_max<kFiltThreads>(threadIdx.x < a.blocks ? w.bmax[threadIdx.x] : -INFINITY, &least, s);
}

// 2. top-p: masses by bin.
template <bool BF16>
__global__ __launch_bounds__(kFiltThreads) void filt_mass_kernel(FiltArgs a) {
    __shared__ FiltShared<kFiltThreads> s;
    __shared__ unsigned long long bins[kFiltMassBins];
    const int tid = threadIdx.x, first = blockIdx.x * a.chunk, end = min(first + a.chunk, a.V);
    FiltRow& w = a.ws[blockIdx.y];
    for (int i = tid; i < kFiltMassBins; i += kFiltThreads) bins[i] = 0;
    const float m = filt_row_max(a, w, s);
    filt_mass_bins<kFiltThreads, BF16>(a, filt_row<BF16>(a, blockIdx.y), first, end, m, bins);
    __syncthreads();
    for (int i = tid; i < kFiltMassBins; i += kFiltThreads)
        if (bins[i] != 0) __hip_atomic_fetch_add(&w.mass_bins[i], bins[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The last step: see the top. What a row's blocks hand to its last workgroup goes through agent-scope
// stores that have returned before the block counts in, and agent-scope loads.
template <bool BF16, int MODE>
__global__ __launch_bounds__(kFiltThreads) void filt_draw_kernel(FiltArgs a) {
    constexpr int NT = kFiltThreads, TILE = (BF16 ? 8 : 4) * NT;
    __shared__ FiltShared<NT> s;
    __shared__ FiltLast<kFiltHeld> z;
    __shared__ uint32_t picked[MODE == kFiltTopP ? kFiltHeld / 4 : 1];
    __shared__ uint32_t n_picked;
    const int tid = threadIdx.x;
    FiltRow& w = a.ws[blockIdx.y];
    const char* const row = filt_row<BF16>(a, blockIdx.y);
    const int first = blockIdx.x * a.chunk, end = min(first + a.chunk, a.V), tiles = (end - first + TILE - 1) / TILE;
    if (tid == 0) z.count = 0, n_picked = 0;
    for (int i = tid; i < tiles; i += NT) z.tile[i] = 0;
    int bin = 0;
    uint64_t above = 0, W = 0;
    const FiltBound bound(0.f, 0.f);
    const float m = filt_row_max(a, w, s);
    if constexpr (MODE == kFiltTopP) {
        float x[kFiltRuns / NT];
#pragma unroll
        for (int i = 0; i < kFiltRuns / NT; ++i) x[i] = w.run[min(i * NT + tid, a.runs - 1)];
        bin = filt_mass_cut<NT>(a, w.mass_bins, s, &above, &W);
        // the runs that reach N's end
        const FiltBound reach(m, bin < kFiltMassBins - 1 ? (float)(bin + 1) / a.to_bin : INFINITY);
        uint32_t mine = 0;
#pragma unroll
        for (int i = 0; i < kFiltRuns / NT; ++i) mine += i * NT + tid < a.runs && reach.takes(x[i]);
        const uint64_t few = filt_sum<NT>(mine, s);
        constexpr int E = BF16 ? 8 : 4;
        if (few * (E * a.run_lanes) <= kFiltHeld) {   // the first block has them all, and whatever they hold fits in its list
            if (blockIdx.x != 0) return;
#pragma unroll
            for (int i = 0; i < kFiltRuns / NT; ++i)
                if (i * NT + tid < a.runs && reach.takes(x[i])) picked[atomicAdd(&n_picked, 1u)] = i * NT + tid;
            __syncthreads();
            filt_list_runs<NT, BF16>(a, row, picked, (int)n_picked, reach, z);
            __syncthreads();
            const int token = filt_last<NT, BF16, kFiltTopK>(a, row, m, a.u[blockIdx.y], bin, 0, W, z.count, nullptr, s, z);
            if (tid == 0) a.out[blockIdx.y] = token;
            return;
        }
    }
    __syncthreads();
    if (m > -INFINITY) filt_gather<NT, BF16, MODE>(a, row, first, end, m, bin, bound, z);
    __syncthreads();
    if constexpr (MODE != kFiltAll) {
        const uint32_t n = z.count;
        // a block whose part does not fit makes the row's list overflow
        if (tid == 0 && n != 0)
            z.base = __hip_atomic_fetch_add(&w.count, n <= kFiltHeld ? n : (uint32_t)kFiltLong + 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (n <= kFiltHeld)
            for (uint32_t i = tid; i < n; i += NT)
                if (z.base + i < kFiltLong) __hip_atomic_store(&w.list[z.base + i], z.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    for (int i = tid; i < tiles; i += NT)
        __hip_atomic_store(&w.tile[first / TILE + i], z.tile[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0)
        s.flag = __hip_atomic_fetch_add(&w.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)a.blocks - 1;
    __syncthreads();
    if (!s.flag) return;

    // ---- the row's last workgroup
    const float u = a.u[blockIdx.y];
    const uint32_t count = MODE == kFiltAll ? 0u : __hip_atomic_load(&w.count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int all = (a.V + TILE - 1) / TILE;
#pragma unroll
    for (int i = 0; i < kFiltTiles / NT; ++i) {
        const int t = i * NT + tid;
        z.tile[t] = t < all ? __hip_atomic_load(&w.tile[t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0ull;
    }
    __syncthreads();
    const int token = filt_last<NT, BF16, MODE>(a, row, m, u, bin, above, W, count, w.list, s, z);
    if (tid == 0) a.out[blockIdx.y] = token;
}

// Top-k, after the maxima: a workgroup a row. Only runs whose maximum is within the bound
// hold logits to be listed, some top_k of them, so that the row is read once in all.
template <int NT, bool BF16>
__global__ __launch_bounds__(NT) void filt_list_kernel(FiltArgs a) {
    constexpr int E = BF16 ? 8 : 4;
    __shared__ FiltShared<NT> s;
    __shared__ FiltLast<kFiltHeldK> z;
    __shared__ uint32_t run_bins[kFiltRunBins + kWave];
    __shared__ uint32_t picked[kFiltHeldK];
    __shared__ uint32_t n_picked;
    const int tid = threadIdx.x;
    const FiltRow& w = a.ws[blockIdx.x];
    const char* const row = filt_row<BF16>(a, blockIdx.x);
    const float u = a.u[blockIdx.x];
    if (tid == 0) z.count = 0, n_picked = 0;
    const FiltBound bound = filt_bound<NT>(a, w.run, run_bins, s, [&](int r) {
        const uint32_t at = atomicAdd(&n_picked, 1u);
        if (at < kFiltHeldK) picked[at] = r;
    });
    __syncthreads();
    const uint32_t n = n_picked;
    if (n <= kFiltHeldK) filt_list_runs<NT, BF16>(a, row, picked, (int)n, bound, z);
    __syncthreads();
    const uint32_t count = n <= kFiltHeldK ? z.count : kFiltHeldK + 1;
    const int token = filt_last<NT, BF16, kFiltTopK>(a, row, bound.m, u, 0, 0, 0, count, nullptr, s, z);
    if (tid == 0) a.out[blockIdx.x] = token;
}

// All steps in one launch, a workgroup a row.
template <int NT, bool BF16, int MODE>
__global__ __launch_bounds__(NT) void filt_one_kernel(FiltArgs a) {
    __shared__ FiltShared<NT> s;
    __shared__ FiltLast<MODE == kFiltTopK ? kFiltHeldK : kFiltHeld> z;
    __shared__ uint32_t run_bins[MODE == kFiltTopK ? kFiltRunBins + kWave : 1];
    __shared__ float runs[MODE == kFiltTopK ? kFiltRuns : 1];
    __shared__ unsigned long long masses[MODE == kFiltTopP ? kFiltMassBins : 1];
    const int tid = threadIdx.x;
    const char* const row = filt_row<BF16>(a, blockIdx.x);
    if (tid == 0) z.count = 0;
    for (int i = tid; i < kFiltTiles; i += NT) z.tile[i] = 0;
    if constexpr (MODE == kFiltTopP)
        for (int i = tid; i < kFiltMassBins; i += NT) masses[i] = 0;
    float m = filt_maxima<NT, BF16>(a, row, 0, a.V, MODE == kFiltTopK ? runs : nullptr), least = 0.f;
    int bin = 0;
    uint64_t above = 0, W = 0;
    FiltBound bound(0.f, 0.f);
    if constexpr (MODE == kFiltTopK) {
        __syncthreads();
        bound = filt_bound<NT>(a, runs, run_bins, s, [](int) {});
        m = bound.m;
    } else {
        m = filt_max<NT>(m, &least, s);
    }
    if constexpr (MODE == kFiltTopP) {
        filt_mass_bins<NT, BF16>(a, row, 0, a.V, m, masses);
        __syncthreads();
        bin = filt_mass_cut<NT>(a, masses, s, &above, &W);
    }
    __syncthreads();
    if (m > -INFINITY) filt_gather<NT, BF16, MODE>(a, row, 0, a.V, m, bin, bound, z);
    __syncthreads();
    const int token = filt_last<NT, BF16, MODE>(a, row, m, a.u[blockIdx.x], bin, above, W, z.count, nullptr, s, z);
    if (tid == 0) a.out[blockIdx.x] = token;
}

// Blocks of a row: some four workgroups a CU in all, blocks of whole tiles.
static void filt_split(int64_t rows, int64_t vocab, int* blocks, int* chunk) {
    const int64_t want = std::min<int64_t>(kFiltBlocks, std::max<int64_t>(1, 4 * prefill_cus() / rows));
    const int64_t c = ((vocab + want - 1) / want + 2047) / 2048 * 2048;
    *chunk = (int)c;
    *blocks = (int)((vocab + c - 1) / c);
}

// NT: a row of 16384 and top-p take 44 us with 256 threads and 32 with 512, a row of 2048 12.7 and 14.0; rows beyond the
// CUs share them (1000 rows of 8192: 67 and 91).
template <int NT, bool BF16>
static void filt_launch_one(const FiltArgs& a, int64_t rows, hipStream_t stream) {
    const dim3 grid((unsigned)rows), t(NT);
    if (a.top_k < a.V) hipLaunchKernelGGL((filt_one_kernel<NT, BF16, kFiltTopK>), grid, t, 0, stream, a);
    else if (a.top_p < 1.0f) hipLaunchKernelGGL((filt_one_kernel<NT, BF16, kFiltTopP>), grid, t, 0, stream, a);
    else hipLaunchKernelGGL((filt_one_kernel<NT, BF16, kFiltAll>), grid, t, 0, stream, a);
}

template <bool BF16>
static void filt_launch(FiltArgs a, int64_t rows, hipStream_t stream) {
    const int vectors = (a.V + (BF16 ? 7 : 3)) / (BF16 ? 8 : 4);
    while ((vectors + a.run_lanes - 1) / a.run_lanes > kFiltRuns) a.run_lanes *= 2;
    a.runs = (vectors + a.run_lanes - 1) / a.run_lanes;
    if (a.V <= kFiltOneVocab) {
        if (a.V > kFiltOneVocab / 4 && rows <= prefill_cus()) filt_launch_one<512, BF16>(a, rows, stream);
        else filt_launch_one<256, BF16>(a, rows, stream);
        return;
    }
    const bool list = a.top_k < a.V;
    filt_split(rows, a.V, &a.blocks, &a.chunk);
    const dim3 t(kFiltThreads), grid(a.blocks, (unsigned)rows);
    if (!list && a.top_p >= 1.0f) a.runs = 0;
    hipLaunchKernelGGL(filt_max_kernel<BF16>, grid, t, 0, stream, a);
    if (list) {
        hipLaunchKernelGGL((filt_list_kernel<kFiltListThreads, BF16>), dim3((unsigned)rows), dim3(kFiltListThreads), 0, stream, a);
    } else if (a.top_p < 1.0f) {
        hipLaunchKernelGGL(filt_mass_kernel<BF16>, grid, t, 0, stream, a);
        hipLaunchKernelGGL((filt_draw_kernel<BF16, kFiltTopP>), grid, t, 0, stream, a);
    } else {
        hipLaunchKernelGGL((filt_draw_kernel<BF16, kFiltAll>), grid, t, 0, stream, a);
    }
}

}  // namespace efm

using namespace efm;

extern "C" size_t efm_sampler_filtered_workspace_bytes(int64_t rows, int64_t vocab) {
    return rows <= 0 || vocab <= kFiltOneVocab ? 0 : (size_t)rows * sizeof(FiltRow);
}

extern "C" int efm_sampler_filtered(int64_t rows, int64_t vocab, const void* logits, int32_t logits_dtype, int64_t logits_stride,
                                    float temperature, int32_t top_k, float top_p, float min_p, const float* uniforms,
                                    int32_t* token_out, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (rows < 0 || vocab <= 0 || vocab >= kFiltMaxVocab)   // V < 2^20 keeps sums of masses below 2^64
        return set_error(EFM_ERR_INVALID_ARGUMENT, "sampler_filtered: %lld rows of %lld logits (below %d)", (long long)rows,
                         (long long)vocab, kFiltMaxVocab);
    if (logits_dtype != EFM_DTYPE_F32 && logits_dtype != EFM_DTYPE_BF16)
        return set_error(EFM_ERR_UNSUPPORTED, "sampler_filtered: logits dtype %d (fp32 or bf16)", logits_dtype);
    if (logits_stride != 0 && logits_stride < vocab)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "sampler_filtered: logits_stride %lld below the vocabulary", (long long)logits_stride);
    // past 1e36 logits whose distance overflows in fp32 would have mass (FLT_MAX / 1e36 is far above the 31.2 at which none is left)
    if (!(temperature >= 1e-6f) || !(temperature <= 1e36f))
        return set_error(EFM_ERR_INVALID_ARGUMENT,
                         "sampler_filtered: temperature must be of [1e-6, 1e36] (below that sampling is greedy)");
    if (!(top_p > 0.0f)) return set_error(EFM_ERR_INVALID_ARGUMENT, "sampler_filtered: top_p must be > 0");
    if (!(min_p <= 1.0f)) return set_error(EFM_ERR_INVALID_ARGUMENT, "sampler_filtered: min_p must be at most 1");
    if (!logits || !uniforms || !token_out) return set_error(EFM_ERR_INVALID_ARGUMENT, "sampler_filtered: null pointer");
    const uintptr_t el = logits_dtype == EFM_DTYPE_BF16 ? 2 : 4;
    if (reinterpret_cast<uintptr_t>(logits) % el != 0 || ((reinterpret_cast<uintptr_t>(uniforms) | reinterpret_cast<uintptr_t>(token_out)) & 3u) != 0)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "sampler_filtered: misaligned pointer");
    if (rows == 0) return EFM_OK;
    if (rows > 65535) return set_error(EFM_ERR_UNSUPPORTED, "sampler_filtered: %lld rows", (long long)rows);
    const size_t need = efm_sampler_filtered_workspace_bytes(rows, vocab);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
        return set_error(EFM_ERR_WORKSPACE, "sampler_filtered: workspace of %zu bytes required", need);
    if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "sampler_filtered: workspace must be 16-byte aligned");
    FiltArgs a;
    a.logits = logits;
    a.stride = logits_stride != 0 ? logits_stride : vocab;
    a.V = (int)vocab;
    a.top_k = top_k > 0 && top_k < vocab ? top_k : (int)vocab;
    a.top_p = top_p;
    a.to_log2 = 1.4426950408889634074 / (double)temperature;
    a.min_mass = std::max<uint64_t>(1, min_p > 0.f ? (uint64_t)std::ceil((double)min_p * kFiltOne) : 0);
    a.to_log2f = (float)a.to_log2;
    a.low = (float)(std::log2((double)a.min_mass - 0.5) - 44.0 - 0.01);   // fp32 moves (l - m) log2(e) / T by 46 2^-22 at most
    a.reach = (float)((double)a.low / a.to_log2);
    a.to_bin = (float)(a.to_log2 * kFiltBinsPerOctave);
    a.u = uniforms;
    a.out = token_out;
    a.ws = need > 0 ? static_cast<FiltRow*>(workspace) : nullptr;
    a.blocks = a.chunk = a.runs = 0;
    a.run_lanes = 1;
    if (logits_dtype == EFM_DTYPE_BF16) filt_launch<true>(a, rows, stream);
    else filt_launch<false>(a, rows, stream);
    return check_launch("sampler_filtered");
}
