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
// logits' bytes and the 64-bit exponentials. A large vocabulary is cut into blocks of a workgroup each:
//   no top-k, no top-p   1. block maxima  2. masses of tiles; the row's last workgroup finds the tile
//                        that holds r and the id within it
//   top-p                1. block maxima  2. histogram of masses by logit  3. masses by tile of the ids
//                        that are surely in N, and a list of the ids of the bin in which N ends; the
//                        last workgroup finds N's end in that list and goes on as above
//   top-k                1. block maxima and a histogram of counts by logit  2. a list of the ids that
//                        may be in K; the last workgroup finds the ends of K and N in it and draws
// A small vocabulary goes through the same steps in one launch, a workgroup a row. Where the list's
// masses do not fit in LDS, or the list not in its place (thousands of equal logits), the last
// workgroup works from the list in memory or from the row itself.
#include "common.hpp"

#include <algorithm>
#include <cmath>

namespace efm {

int prefill_cus();

constexpr int kFiltThreads = 256;
constexpr int kFiltWaves = kFiltThreads / kWave;
constexpr int kFiltMaxVocab = 1 << 20;
constexpr double kFiltOne = 17592186044416.0;   // 2^44
constexpr int kFiltBlocks = 128;                 // of a row, at most
constexpr int kFiltTiles = 1024;                 // of a row: passes of a workgroup's loads, 1024 logits or more each
constexpr int kFiltMassBins = 1024, kFiltBinsPerOctave = 22;   // masses from 2^0 to below 2^-46
constexpr int kFiltCountBins = 4096, kFiltCountShift = 20;     // sign, exponent and three bits of the logit
constexpr int kFiltList = 4096;
constexpr int kFiltHeld = 1024;                  // entries of a list that a workgroup holds with their masses
constexpr int kFiltOneVocab = 16384;             // rows of one launch

// One row's part of the workspace. hist, counter and count are zero between calls.
struct FiltRow {
    union {
        unsigned long long mass[kFiltMassBins];
        uint32_t count[kFiltCountBins];
    } hist;
    uint32_t counter, count;
    uint32_t pad[2];
    float bmax[kFiltBlocks];
    unsigned long long tile[kFiltTiles];
    unsigned long long list[kFiltList];   // key << 32 | id
};
static_assert(sizeof(FiltRow) % 16 == 0, "rows of the workspace stay aligned");

struct FiltArgs {
    const void* logits;
    int64_t stride;
    int V, top_k;
    float top_p;
    double to_log2;       // log2(e) / T
    float to_log2f, low;  // a logit with (l - m) to_log2f <= low has no mass that counts
    float to_bin;         // bins a unit of m - l
    uint64_t min_mass;    // max(1, ceil(min_p 2^44))
    const float* u;
    int32_t* out;
    FiltRow* ws;
    int blocks, chunk;    // of a row; logits of a block
};

enum { kFiltAll, kFiltTopP, kFiltTopK };

// w of a logit, m the row's largest. 2^t, t = (l - m) log2(e) / T, as 2^n 2^f with the series of
// exp(f ln 2), |f| <= 1/2: the term after the last is below 2^-52. Adding 2^52 rounds to an integer.
__device__ __forceinline__ uint64_t filt_mass(const FiltArgs& a, float l, float m) {
    if (l != m && !((l - m) * a.to_log2f > a.low)) return 0;
    const double t = l == m ? 0.0 : ((double)l - (double)m) * a.to_log2;
    const double n = __builtin_rint(t), f = (t - n) * 0.69314718055994530942;
    double p = 1.0 / 479001600.0;
    p = __builtin_fma(p, f, 1.0 / 39916800.0);
    p = __builtin_fma(p, f, 1.0 / 3628800.0);
    p = __builtin_fma(p, f, 1.0 / 362880.0);
    p = __builtin_fma(p, f, 1.0 / 40320.0);
    p = __builtin_fma(p, f, 1.0 / 5040.0);
    p = __builtin_fma(p, f, 1.0 / 720.0);
    p = __builtin_fma(p, f, 1.0 / 120.0);
    p = __builtin_fma(p, f, 1.0 / 24.0);
    p = __builtin_fma(p, f, 1.0 / 6.0);
    p = __builtin_fma(p, f, 0.5);
    p = __builtin_fma(p, f, 1.0);
    p = __builtin_fma(p, f, 1.0);
    const uint64_t w = __builtin_bit_cast(uint64_t, __builtin_ldexp(p, (int)n + 44) + 4503599627370496.0) & 0xfffffffffffffull;
    return w >= a.min_mass ? w : 0;
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

// A row's logits [first, end), first a multiple of a tile: f(tile of the range, first id, the thread's
// E logits as they are (-inf past the end), how many of them there are), by all threads together; 16
// bytes a thread, four under way.
template <bool BF16, typename F>
__device__ __forceinline__ void filt_tiles(const void* row, int first, int end, F f) {
    constexpr int E = BF16 ? 8 : 4, U = 4, TILE = E * kFiltThreads;
    const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
    for (int t0 = 0; first + t0 * TILE < end; t0 += U) {
        uint4 x[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int i = first + (t0 + j) * TILE + (int)threadIdx.x * E;
            if (aligned && i + E <= end) {
                x[j] = *reinterpret_cast<const uint4*>(static_cast<const char*>(row) + (int64_t)i * (BF16 ? 2 : 4));
            } else {
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
                x[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int i = first + (t0 + j) * TILE + (int)threadIdx.x * E;
            if (first + (t0 + j) * TILE >= end) break;
            float l[E];
            const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (BF16) l[2 * e] = lo_f32(w[e]), l[2 * e + 1] = hi_f32(w[e]);
                else l[e] = __uint_as_float(w[e]);
            }
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

struct FiltShared {
    unsigned long long red[kFiltWaves];
    unsigned long long sel[2];
    unsigned long long bins[2][kFiltThreads];
    uint32_t counts[2][kFiltThreads];
    float redf[kFiltWaves];
    uint32_t flag, found[3];
};

// Sum of the values of the threads before this one, and of all.
__device__ __forceinline__ uint64_t filt_scan(uint64_t v, FiltShared& s, uint64_t* total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint64_t incl = filt_wave_scan(v);
    __syncthreads();
    if (lane == kWave - 1) s.red[wave] = incl;
    __syncthreads();
    uint64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kFiltWaves; ++w) {
        if (w < wave) before += s.red[w];
        all += s.red[w];
    }
    *total = all;
    return before + incl - v;
}

__device__ __forceinline__ uint64_t filt_sum(uint64_t v, FiltShared& s) {
    uint64_t all;
    filt_scan(v, s, &all);
    return all;
}

__device__ __forceinline__ float filt_max(float m, FiltShared& s) {
    m = wave_max_uniform(m);
    if (threadIdx.x % kWave == 0) s.redf[threadIdx.x / kWave] = m;
    __syncthreads();
    m = s.redf[0];
#pragma unroll
    for (int w = 1; w < kFiltWaves; ++w) m = fmaxf(m, s.redf[w]);
    return m;
}

// What the choices so far keep: keys above `key`, and of those equal to it the ids up to `id`.
struct FiltCut {
    uint32_t key;
    int id;
    __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= id); }
};

// floor(u M), at most M - 1.
__device__ __forceinline__ uint64_t filt_draw(float u, uint64_t M) {
    const double x = (double)u * (double)M;
    const uint64_t r = x > 0.0 ? (uint64_t)__builtin_fmin(x, 9.2e18) : 0ull;
    return r < M ? r : M - 1;
}

__device__ __forceinline__ uint64_t filt_need(float top_p, uint64_t W) {
    const uint64_t need = (uint64_t)__builtin_ceil((double)top_p * (double)W);
    return need < 1 ? 1 : need > W ? W : need;
}

// The entry that holds unit `rank` of the weights of a source of (id, key, weight), each(f): in the
// sampler's order (keys of [low, high]), or by id alone (ids of [low, high]). The range that may hold
// it is cut into 256 bins until one entry is left, four times for keys and three for the ids of equal
// keys at most. rank is below the sum of the weights; were it not (a workspace that was not zeroed),
// the entry is any.
template <typename Each>
__device__ __forceinline__ FiltCut filt_pick(bool by_id, uint32_t low, uint32_t high, uint64_t rank, const FiltArgs& a, FiltShared& s, Each each) {
    const int tid = threadIdx.x;
    bool ids = by_id;
    uint32_t lo = by_id ? low : ~high, hi = by_id ? high : ~low, tie = 0;   // of ~key, or of the ids with ~key = tie
    __syncthreads();
    s.bins[0][tid] = 0, s.counts[0][tid] = 0;
    __syncthreads();
    for (int step = 0; step < 8; ++step) {
        const int b = step & 1, bits = 32 - __builtin_clz(hi - lo | 1u), shift = max(bits - 8, 0);
        auto value = [&](int i, uint32_t k) { return ids ? (uint32_t)i : ~k; };
        auto active = [&](int i, uint32_t k, uint64_t w) {
            return w != 0 && value(i, k) >= lo && value(i, k) <= hi && (!ids || by_id || ~k == tie);
        };
        each([&](int i, uint32_t k, uint64_t w) {
            if (!active(i, k, w)) return;
            const uint32_t bin = (value(i, k) - lo) >> shift;
            atomicAdd(&s.bins[b][bin], (unsigned long long)w);
            atomicAdd(&s.counts[b][bin], 1u);
        });
        s.bins[1 - b][tid] = 0, s.counts[1 - b][tid] = 0;
        __syncthreads();
        uint64_t all;
        const uint64_t own = s.bins[b][tid], excl = filt_scan(own, s, &all);
        if (excl <= rank && rank - excl < own) s.sel[0] = tid, s.sel[1] = excl, s.found[2] = s.counts[b][tid];
        __syncthreads();
        rank -= s.sel[1];
        lo += ((uint32_t)s.sel[0] & (kFiltThreads - 1)) << shift, hi = min(hi, lo + ((1u << shift) - 1));
        if (s.found[2] == 1) {
            each([&](int i, uint32_t k, uint64_t w) {
                if (active(i, k, w)) s.found[0] = k, s.found[1] = (uint32_t)i;
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

// K, N and the draw over a source of `count` entries (id, key, mass), each(f), keys of [low, high].
template <typename Each>
__device__ __forceinline__ int filt_choose(const FiltArgs& a, uint32_t low, uint32_t high, uint32_t count, float u, FiltShared& s, Each each) {
    FiltCut kept{0u, a.V};
    if ((uint32_t)a.top_k < count)
        kept = filt_pick(false, low, high, (uint64_t)a.top_k - 1, a, s, [&](auto f) { each([&](int i, uint32_t k, uint64_t) { f(i, k, 1ull); }); });
    auto left = [&](auto f) { each([&](int i, uint32_t k, uint64_t w) { f(i, k, kept.keeps(k, i) ? w : 0ull); }); };
    auto total = [&]() {
        uint64_t sum = 0;
        left([&](int, uint32_t, uint64_t w) { sum += w; });
        return filt_sum(sum, s);
    };
    uint64_t M = total();
    if (a.top_p < 1.0f) {
        kept = filt_pick(false, low, high, filt_need(a.top_p, M) - 1, a, s, left);
        M = total();
    }
    return filt_pick(true, 0, (uint32_t)a.V - 1, filt_draw(u, M), a, s, left).id;
}

// The same over the row itself: for what fits nowhere.
template <bool BF16>
__device__ __noinline__ int filt_choose_row(const FiltArgs& a, const void* row, float m, float u, FiltShared& s) {
    return filt_choose(a, 0u, ~0u, (uint32_t)a.V, u, s, [&](auto f) {
        filt_tiles<BF16>(row, 0, a.V, [&](int, int i, const auto& l, int n) {
            constexpr int E = BF16 ? 8 : 4;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e < n) f(i + e, filt_key(filt_clean(l[e])), filt_mass(a, filt_clean(l[e]), m));
        });
    });
}

// The least logit of a bin of counts.
__device__ __forceinline__ float filt_bin_logit(int bin) {
    return bin <= (int)(0x007fffffu >> kFiltCountShift) ? -INFINITY : filt_logit((uint32_t)bin << kFiltCountShift);
}

constexpr int kFiltPer = kFiltCountBins / kFiltThreads;
// A thread's 16 bins of a count histogram in LDS lie side by side, with a word between the threads'.
__device__ __forceinline__ int filt_slot(int bin) { return bin + bin / kFiltPer; }
constexpr int kFiltSlots = kFiltCountBins + kFiltThreads;

// The bin that holds the top_k-th logit; the thread has the counts of bins high, high - 1, ... .
__device__ __forceinline__ int filt_count_cut(const FiltArgs& a, const uint32_t (&c)[kFiltPer], int high, FiltShared& s) {
    uint32_t own = 0;
#pragma unroll
    for (int i = 0; i < kFiltPer; ++i) own += c[i];
    uint64_t all, excl = filt_scan(own, s, &all);
    const uint64_t rank = (uint64_t)a.top_k - 1;
    if (excl <= rank && rank - excl < own) {
        int at = 0;
#pragma unroll
        for (int i = 0; i < kFiltPer; ++i) {
            if (excl <= rank) at = high - i;
            excl += c[i];
        }
        s.sel[0] = at;
    }
    __syncthreads();
    return (int)s.sel[0];
}

// The bin in which N ends; the thread has the masses of four bins. *above: the mass of the bins before
// it, *W: of all.
__device__ __forceinline__ int filt_mass_cut(const FiltArgs& a, const uint64_t (&h)[4], FiltShared& s, uint64_t* above, uint64_t* W) {
    uint64_t excl = filt_scan(h[0] + h[1] + h[2] + h[3], s, W);
    const uint64_t rank = filt_need(a.top_p, *W) - 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (excl <= rank && rank - excl < h[i]) s.sel[0] = threadIdx.x * 4 + i, s.sel[1] = excl;
        excl += h[i];
    }
    __syncthreads();
    *above = s.sel[1];
    return (int)s.sel[0];
}

// Shared memory of the last step: the list with its masses, and the tiles' masses.
struct FiltLast {
    unsigned long long list[kFiltHeld];
    unsigned long long mass[kFiltHeld];
    unsigned long long tile[kFiltTiles];
    uint32_t count, base;
};

// A block's part of the last step: top-k: ids of bins >= bin are listed; top-p: masses of bins < bin by
// tile, ids of `bin` are listed; neither: masses by tile. Tiles count from the block's first. Most logits
// are below what any of that takes: one comparison each, and a NaN goes the careful way.
template <bool BF16, int MODE>
__device__ __forceinline__ void filt_gather(const FiltArgs& a, const void* row, int first, int end, float m, int bin, FiltLast& z) {
    constexpr int E = BF16 ? 8 : 4;
    auto enlist = [&](int i, float l) {
        const uint32_t at = atomicAdd(&z.count, 1u);
        if (at < kFiltHeld) z.list[at] = (unsigned long long)filt_key(l) << 32 | (uint32_t)i;
    };
    const float least = filt_bin_logit(bin), past = bin < kFiltMassBins - 1 ? (float)(bin + 1) : INFINITY;
    filt_tiles<BF16>(row, first, end, [&](int t, int i, const float (&l)[E], int n) {
        bool some = false;
#pragma unroll
        for (int e = 0; e < E; ++e)
            some |= MODE == kFiltTopK ? l[e] >= least : MODE == kFiltTopP ? !((m - l[e]) * a.to_bin >= past) : !((l[e] - m) * a.to_log2f <= a.low);
        uint64_t y = 0;
        if (some) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = filt_clean(l[e]);
                if constexpr (MODE == kFiltTopK) {
                    if (e < n && x >= least) enlist(i + e, x);
                } else if constexpr (MODE == kFiltTopP) {
                    const int b = filt_bin(a, x, m);
                    if (b < bin) y += filt_mass(a, x, m);
                    else if (b == bin && e < n) enlist(i + e, x);
                } else {
                    y += filt_mass(a, x, m);   // there is none past the end: -inf
                }
            }
        }
        if (MODE != kFiltTopK && __any(y != 0)) {
            y = filt_last_lane(filt_wave_scan(y));
            if (threadIdx.x % kWave == 0) atomicAdd(&z.tile[t], (unsigned long long)y);
        }
    });
}

// The choice from a row's list (`count` entries, in z or in `list`) and its tiles' masses (in z.tile).
template <bool BF16, int MODE>
__device__ __forceinline__ int filt_last(const FiltArgs& a, const void* row, float m, float u, int bin, uint64_t above, uint64_t W,
                                         uint32_t count, const unsigned long long* list, FiltShared& s, FiltLast& z) {
    const int tid = threadIdx.x;
    const uint32_t high = filt_key(m), low = filt_key(filt_bin_logit(bin));   // the keys of top-k's list
    if (m == -INFINITY) return -1;
    if (count > (list != nullptr && MODE == kFiltTopK ? kFiltList : kFiltHeld)) return filt_choose_row<BF16>(a, row, m, u, s);
    if (MODE == kFiltTopK && count > kFiltHeld)
        return filt_choose(a, low, high, count, u, s, [&](auto f) {
            for (uint32_t i = tid; i < count; i += kFiltThreads) {
                const unsigned long long x = __hip_atomic_load(&list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                f((int)(uint32_t)x, (uint32_t)(x >> 32), filt_mass(a, filt_logit((uint32_t)(x >> 32)), m));
            }
        });
    for (uint32_t i = tid; i < count; i += kFiltThreads) {
        const unsigned long long x = list != nullptr ? __hip_atomic_load(&list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : z.list[i];
        z.list[i] = x;
        z.mass[i] = filt_mass(a, filt_logit((uint32_t)(x >> 32)), m);
    }
    __syncthreads();
    auto each = [&](auto f) {
        for (uint32_t i = tid; i < count; i += kFiltThreads) f((int)(uint32_t)z.list[i], (uint32_t)(z.list[i] >> 32), (uint64_t)z.mass[i]);
    };
    if constexpr (MODE == kFiltTopK) return filt_choose(a, low, high, count, u, s, each);
    constexpr int E = BF16 ? 8 : 4, TILE = E * kFiltThreads;
    FiltCut kept{0u, a.V};
    if constexpr (MODE == kFiltTopP) {
        kept = filt_pick(false, 0u, high, filt_need(a.top_p, W) - 1 - above, a, s, each);
        each([&](int i, uint32_t k, uint64_t w) {
            if (w != 0 && kept.keeps(k, i) && i < a.V) atomicAdd(&z.tile[i / TILE], (unsigned long long)w);
        });
        __syncthreads();
    }
    uint64_t own = 0, M, h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) own += h[i] = z.tile[tid * 4 + i];
    uint64_t excl = filt_scan(own, s, &M);
    const uint64_t r = filt_draw(u, M);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (excl <= r && r - excl < h[i]) s.sel[0] = tid * 4 + i, s.sel[1] = excl;
        excl += h[i];
    }
    __syncthreads();
    const int t = (int)min((uint32_t)s.sel[0], (uint32_t)(a.V - 1) / TILE);
    const uint64_t rest = r - s.sel[1];
    filt_tiles<BF16>(row, t * TILE, min(t * TILE + TILE, a.V), [&](int, int i, const float (&l)[E], int) {
        uint64_t y[E], sum = 0, all;
#pragma unroll
        for (int e = 0; e < E; ++e) sum += y[e] = kept.keeps(filt_key(filt_clean(l[e])), i + e) ? filt_mass(a, filt_clean(l[e]), m) : 0ull;
        uint64_t at = filt_scan(sum, s, &all);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (at <= rest && rest - at < y[e]) s.found[0] = i + e;
            at += y[e];
        }
    });
    __syncthreads();
    return (int)s.found[0];
}

template <bool BF16>
__device__ __forceinline__ const char* filt_row(const FiltArgs& a, unsigned r) {
    return static_cast<const char*>(a.logits) + (int64_t)r * a.stride * (BF16 ? 2 : 4);
}

// 1. Block maxima; top-k: a histogram of counts, of which a block adds the bins that its own first
// top_k logits reach (lower ones cannot be among the row's).
template <bool BF16, int MODE>
__global__ __launch_bounds__(kFiltThreads) void filt_max_kernel(FiltArgs a) {
    constexpr int E = BF16 ? 8 : 4;
    __shared__ FiltShared s;
    __shared__ uint32_t bins[MODE == kFiltTopK ? kFiltSlots : 1];
    const int tid = threadIdx.x, block = blockIdx.x;
    FiltRow& w = a.ws[blockIdx.y];
    const int first = block * a.chunk, end = min(first + a.chunk, a.V);
    if constexpr (MODE == kFiltTopK) {
        for (int i = tid; i < kFiltSlots; i += kFiltThreads) bins[i] = 0;
        __syncthreads();
    }
    float m = -INFINITY;
    filt_tiles<BF16>(filt_row<BF16>(a, blockIdx.y), first, end, [&](int, int, const float (&l)[E], int n) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            m = fmaxf(m, l[e]);   // not a NaN
            if (MODE == kFiltTopK && e < n) atomicAdd(&bins[filt_slot(filt_key(filt_clean(l[e])) >> kFiltCountShift)], 1u);
        }
    });
    m = filt_max(m, s);   // the counts are whole behind its barrier
    if (tid == 0) w.bmax[block] = m;
    if constexpr (MODE == kFiltTopK) {
        const int high = kFiltCountBins - 1 - tid * kFiltPer;   // the thread's bins, from the highest
        uint32_t c[kFiltPer], own = 0;
#pragma unroll
        for (int i = 0; i < kFiltPer; ++i) own += c[i] = bins[filt_slot(high - i)];
        uint64_t all;
        uint64_t above = filt_scan(own, s, &all);
#pragma unroll
        for (int i = 0; i < kFiltPer; ++i) {
            if (c[i] != 0 && above < (uint64_t)a.top_k)
                __hip_atomic_fetch_add(&w.hist.count[high - i], c[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            above += c[i];
        }
    }
}

// The row's maximum, from its blocks'.
__device__ __forceinline__ float filt_row_max(const FiltArgs& a, const FiltRow& w, FiltShared& s) {
    return filt_max(threadIdx.x < a.blocks ? w.bmax[threadIdx.x] : -INFINITY, s);
}

template <bool BF16>
__device__ __forceinline__ void filt_mass_bins(const FiltArgs& a, const void* row, int first, int end, float m, unsigned long long* bins) {
    constexpr int E = BF16 ? 8 : 4;
    filt_tiles<BF16>(row, first, end, [&](int, int, const float (&l)[E], int) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint64_t x = filt_mass(a, filt_clean(l[e]), m);
            if (x != 0) atomicAdd(&bins[filt_bin(a, l[e], m)], (unsigned long long)x);
        }
    });
}

// 2. top-p: masses by bin.
template <bool BF16>
__global__ __launch_bounds__(kFiltThreads) void filt_mass_kernel(FiltArgs a) {
    __shared__ FiltShared s;
    __shared__ unsigned long long bins[kFiltMassBins];
    const int tid = threadIdx.x, first = blockIdx.x * a.chunk, end = min(first + a.chunk, a.V);
    FiltRow& w = a.ws[blockIdx.y];
    for (int i = tid; i < kFiltMassBins; i += kFiltThreads) bins[i] = 0;
    const float m = filt_row_max(a, w, s);
    filt_mass_bins<BF16>(a, filt_row<BF16>(a, blockIdx.y), first, end, m, bins);
    __syncthreads();
    for (int i = tid; i < kFiltMassBins; i += kFiltThreads)
        if (bins[i] != 0) __hip_atomic_fetch_add(&w.hist.mass[i], bins[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The last step: see the top. What a row's blocks hand to its last workgroup goes through agent-scope
// stores that have returned before the block counts in, and agent-scope loads.
template <bool BF16, int MODE>
__global__ __launch_bounds__(kFiltThreads) void filt_draw_kernel(FiltArgs a) {
    constexpr int TILE = (BF16 ? 8 : 4) * kFiltThreads;
    __shared__ FiltShared s;
    __shared__ FiltLast z;
    const int tid = threadIdx.x;
    FiltRow& w = a.ws[blockIdx.y];
    const char* const row = filt_row<BF16>(a, blockIdx.y);
    const int first = blockIdx.x * a.chunk, end = min(first + a.chunk, a.V), tiles = (end - first + TILE - 1) / TILE;
    if (tid == 0) z.count = 0;
    if constexpr (MODE != kFiltTopK)
        for (int i = tid; i < tiles; i += kFiltThreads) z.tile[i] = 0;
    // where K or N ends: the bin, and what lies above it
    int bin = 0;
    uint64_t above = 0, W = 0;
    uint32_t c[kFiltPer];
    uint64_t h[4];
    const int high = kFiltCountBins - 1 - tid * kFiltPer;
    if constexpr (MODE == kFiltTopK) {
#pragma unroll
        for (int i = 0; i < kFiltPer; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(&w.hist.count[high - i - 3]);
            c[i] = x.w, c[i + 1] = x.z, c[i + 2] = x.y, c[i + 3] = x.x;
        }
    }
    if constexpr (MODE == kFiltTopP) {
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = w.hist.mass[tid * 4 + i];
    }
    const float m = filt_row_max(a, w, s);
    if constexpr (MODE == kFiltTopK) bin = filt_count_cut(a, c, high, s);
    if constexpr (MODE == kFiltTopP) bin = filt_mass_cut(a, h, s, &above, &W);
    if (m > -INFINITY) filt_gather<BF16, MODE>(a, row, first, end, m, bin, z);
    __syncthreads();
    if constexpr (MODE != kFiltAll) {
        const uint32_t n = z.count;
        // a block whose part does not fit makes the row's list overflow
        if (tid == 0 && n != 0)
            z.base = __hip_atomic_fetch_add(&w.count, n <= kFiltHeld ? n : (uint32_t)kFiltList + 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (n <= kFiltHeld)
            for (uint32_t i = tid; i < n; i += kFiltThreads)
                if (z.base + i < kFiltList) __hip_atomic_store(&w.list[z.base + i], z.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if constexpr (MODE != kFiltTopK)
        for (int i = tid; i < tiles; i += kFiltThreads)
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
    if constexpr (MODE != kFiltTopK) {
        const int all = (a.V + TILE - 1) / TILE;
#pragma unroll
        for (int i = 0; i < kFiltTiles / kFiltThreads; ++i) {
            const int t = i * kFiltThreads + tid;
            z.tile[t] = t < all ? __hip_atomic_load(&w.tile[t], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0ull;
        }
    }
    __syncthreads();
    if (tid == 0) w.counter = 0, w.count = 0;
    if constexpr (MODE == kFiltTopK)
        for (int i = tid; i < kFiltCountBins; i += kFiltThreads) w.hist.count[i] = 0;
    if constexpr (MODE == kFiltTopP)
        for (int i = tid; i < kFiltMassBins; i += kFiltThreads) w.hist.mass[i] = 0;
    const int token = filt_last<BF16, MODE>(a, row, m, u, bin, above, W, count, w.list, s, z);
    if (tid == 0) a.out[blockIdx.y] = token;
}

// Small vocabularies: all steps in one launch, a workgroup a row.
template <bool BF16, int MODE>
__global__ __launch_bounds__(kFiltThreads) void filt_one_kernel(FiltArgs a) {
    constexpr int E = BF16 ? 8 : 4;
    __shared__ FiltShared s;
    __shared__ FiltLast z;
    __shared__ uint32_t counts[MODE == kFiltTopK ? kFiltSlots : 1];
    __shared__ unsigned long long masses[MODE == kFiltTopP ? kFiltMassBins : 1];
    const int tid = threadIdx.x;
    const char* const row = filt_row<BF16>(a, blockIdx.x);
    if (tid == 0) z.count = 0;
    for (int i = tid; i < kFiltTiles; i += kFiltThreads) z.tile[i] = 0;
    if constexpr (MODE == kFiltTopK) {
        for (int i = tid; i < kFiltSlots; i += kFiltThreads) counts[i] = 0;
        __syncthreads();
    }
    if constexpr (MODE == kFiltTopP)
        for (int i = tid; i < kFiltMassBins; i += kFiltThreads) masses[i] = 0;
    float m = -INFINITY;
    filt_tiles<BF16>(row, 0, a.V, [&](int, int, const float (&l)[E], int n) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            m = fmaxf(m, l[e]);
            if (MODE == kFiltTopK && e < n) atomicAdd(&counts[filt_slot(filt_key(filt_clean(l[e])) >> kFiltCountShift)], 1u);
        }
    });
    m = filt_max(m, s);
    int bin = 0;
    uint64_t above = 0, W = 0;
    if constexpr (MODE == kFiltTopK) {
        const int high = kFiltCountBins - 1 - tid * kFiltPer;
        uint32_t c[kFiltPer];
#pragma unroll
        for (int i = 0; i < kFiltPer; ++i) c[i] = counts[filt_slot(high - i)];
        bin = filt_count_cut(a, c, high, s);
    }
    if constexpr (MODE == kFiltTopP) {
        filt_mass_bins<BF16>(a, row, 0, a.V, m, masses);
        __syncthreads();
        uint64_t h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = masses[tid * 4 + i];
        bin = filt_mass_cut(a, h, s, &above, &W);
    }
    if (m > -INFINITY) filt_gather<BF16, MODE>(a, row, 0, a.V, m, bin, z);
    __syncthreads();
    const int token = filt_last<BF16, MODE>(a, row, m, a.u[blockIdx.x], bin, above, W, z.count, nullptr, s, z);
    if (tid == 0) a.out[blockIdx.x] = token;
}

// Blocks of a row: some four workgroups a CU in all, blocks of whole tiles.
static void filt_split(int64_t rows, int64_t vocab, int* blocks, int* chunk) {
    const int64_t want = std::min<int64_t>(kFiltBlocks, std::max<int64_t>(1, 4 * prefill_cus() / rows));
    const int64_t c = ((vocab + want - 1) / want + 2047) / 2048 * 2048;
    *chunk = (int)c;
    *blocks = (int)((vocab + c - 1) / c);
}

template <bool BF16>
static void filt_launch(const FiltArgs& a, int64_t rows, hipStream_t stream) {
    const dim3 t(kFiltThreads), grid(a.blocks, (unsigned)rows), one((unsigned)rows);
    const bool k = a.top_k < a.V, p = a.top_p < 1.0f;
    if (a.ws == nullptr) {
        if (k) hipLaunchKernelGGL((filt_one_kernel<BF16, kFiltTopK>), one, t, 0, stream, a);
        else if (p) hipLaunchKernelGGL((filt_one_kernel<BF16, kFiltTopP>), one, t, 0, stream, a);
        else hipLaunchKernelGGL((filt_one_kernel<BF16, kFiltAll>), one, t, 0, stream, a);
        return;
    }
    if (k) {
        hipLaunchKernelGGL((filt_max_kernel<BF16, kFiltTopK>), grid, t, 0, stream, a);
        hipLaunchKernelGGL((filt_draw_kernel<BF16, kFiltTopK>), grid, t, 0, stream, a);
        return;
    }
    hipLaunchKernelGGL((filt_max_kernel<BF16, kFiltAll>), grid, t, 0, stream, a);
    if (p) {
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
    if (!(temperature >= 1e-6f) || !(temperature < INFINITY))
        return set_error(EFM_ERR_INVALID_ARGUMENT,
                         "sampler_filtered: temperature must be finite and >= 1e-6 (below that sampling is greedy)");
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
    a.to_bin = (float)(a.to_log2 * kFiltBinsPerOctave);
    a.u = uniforms;
    a.out = token_out;
    a.ws = need > 0 ? static_cast<FiltRow*>(workspace) : nullptr;
    filt_split(rows, vocab, &a.blocks, &a.chunk);
    if (logits_dtype == EFM_DTYPE_BF16) filt_launch<true>(a, rows, stream);
    else filt_launch<false>(a, rows, stream);
    return check_launch("sampler_filtered");
}
