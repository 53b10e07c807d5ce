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
//   no top-k, no top-p   1. block maxima  2. block masses; the row's last workgroup finds the block
//                        that holds r and the id within it
//   top-p                1. block maxima  2. histogram of masses by logit  3. masses of the ids that
//                        are surely in N by block, and a list of the ids of the bin in which N ends;
//                        the last workgroup orders that list and goes on as above
//   top-k                1. block maxima and a histogram of counts by logit  2. a list of the ids that
//                        may be in K; the last workgroup orders it and draws
// A list that does not fit (thousands of equal logits) sends the row's last workgroup through the
// row itself, digit by digit: filt_select below, which is also what the small vocabularies run on, a
// workgroup a row with the row in LDS.
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
constexpr int kFiltMassBins = 1024, kFiltBinsPerOctave = 22;   // masses from 2^0 to below 2^-46
constexpr int kFiltCountBins = 4096, kFiltCountShift = 20;     // sign, exponent and three bits of the logit
constexpr int kFiltMaxTiles = kFiltThreads;      // a block's passes of a workgroup's loads, 1024 logits or more each
constexpr int kFiltList = 4096;
constexpr int kFiltSort = 1024;
constexpr int kFiltLdsVocab = 14336;             // rows that a workgroup holds in LDS

// One row's part of the workspace. hist, counter and count are zero between calls.
struct FiltRow {
    union {
        unsigned long long mass[kFiltMassBins];
        uint32_t count[kFiltCountBins];
    } hist;
    uint32_t counter, count;
    uint32_t pad[2];
    float bmax[kFiltBlocks];
    unsigned long long bmass[kFiltBlocks];
    unsigned long long list[kFiltList];   // ~key << 32 | id: ascending in the sampler's order
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

// f(id, logit) for the logits of [first, end) of a row: 16 bytes a thread, four under way.
template <bool BF16, typename F>
__device__ __forceinline__ void filt_each(const void* row, int first, int end, F f) {
    constexpr int E = BF16 ? 8 : 4, U = 4;
    const int tid = threadIdx.x;
    int done = first;
    if ((reinterpret_cast<uintptr_t>(row) & 15) == 0) {   // first is a multiple of 8
        const int whole = (end - first) / E;
        const uint4* const p = reinterpret_cast<const uint4*>(static_cast<const char*>(row) + (int64_t)first * (BF16 ? 2 : 4));
        for (int v0 = tid; v0 < whole; v0 += U * kFiltThreads) {
            uint4 x[U];
#pragma unroll
            for (int j = 0; j < U; ++j)
                if (v0 + j * kFiltThreads < whole) x[j] = p[v0 + j * kFiltThreads];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int v = v0 + j * kFiltThreads;
                if (v >= whole) break;
                const int i = first + v * E;
                const uint32_t w[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (BF16) {
                        f(i + 2 * e, filt_clean(lo_f32(w[e])));
                        f(i + 2 * e + 1, filt_clean(hi_f32(w[e])));
                    } else {
                        f(i + e, filt_clean(__uint_as_float(w[e])));
                    }
                }
            }
        }
        done = first + whole * E;
    }
    for (int i = done + tid; i < end; i += kFiltThreads) {
        if constexpr (BF16) f(i, filt_clean(bf16_to_f32(static_cast<const uint16_t*>(row)[i])));
        else f(i, filt_clean(static_cast<const float*>(row)[i]));
    }
}

__device__ __forceinline__ uint64_t filt_wave_scan(uint64_t v, int lane) {
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const uint64_t o = __shfl_up(v, off, kWave);
        if (lane >= off) v += o;
    }
    return v;
}

struct FiltShared {
    unsigned long long red[kFiltWaves];
    unsigned long long sel[2];
    unsigned long long bins[kFiltThreads];
    float redf[kFiltWaves];
    uint32_t flag;
};

// Sum of the values of the threads before this one, and of all.
__device__ __forceinline__ uint64_t filt_scan(uint64_t v, FiltShared& s, uint64_t* total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint64_t incl = filt_wave_scan(v, lane);
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

// The thread whose `own` units hold unit `rank` (from 0), in the order of threads, and the units
// before it; rank is below the total.
__device__ __forceinline__ int filt_find(uint64_t own, uint64_t rank, FiltShared& s, uint64_t* before) {
    uint64_t all;
    const uint64_t excl = filt_scan(own, s, &all);
    if (excl <= rank && rank - excl < own) s.sel[0] = threadIdx.x, s.sel[1] = excl;
    __syncthreads();
    *before = s.sel[1];
    return (int)s.sel[0];
}

__device__ __forceinline__ float filt_max(float m, FiltShared& s) {
    m = wave_max(m);
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

// The whole choice over any source of (id, logit), each(f), by histograms of eight bits at a time.
template <typename Each>
__device__ int filt_select(const FiltArgs& a, float m, float u, FiltShared& s, Each each) {
    const int tid = threadIdx.x;
    uint64_t before;
    // The bins of `digit` of what take(i, k) takes, and the one that holds unit `rank` of `weight`.
    auto pass = [&](auto take, auto digit, auto weight, uint64_t& rank) {
        __syncthreads();
        s.bins[tid] = 0;
        __syncthreads();
        each([&](int i, float l) {
            const uint32_t k = filt_key(l);
            if (!take(i, k)) return;
            const uint64_t w = weight(l);
            if (w != 0) atomicAdd(&s.bins[digit(i, k)], (unsigned long long)w);
        });
        __syncthreads();
        const int bin = filt_find(s.bins[tid], rank, s, &before);
        rank -= before;
        return (uint32_t)bin;
    };
    auto by_id = [&](auto take, auto weight, uint64_t rank) {
        uint32_t top = 0;
        for (int shift = 16; shift >= 0; shift -= 8) {
            const uint32_t bin = pass([&](int i, uint32_t k) { return take(i, k) && (uint32_t)i >> shift >> 8 == top; },
                                      [&](int i, uint32_t) { return (uint32_t)i >> shift & 255; }, weight, rank);
            top = top << 8 | bin;
        }
        return (int)top;
    };
    auto cut_at = [&](const FiltCut& kept, auto weight, uint64_t rank) {
        uint32_t prefix = 0, mask = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            const uint32_t bin = pass([&](int i, uint32_t k) { return (k & mask) == prefix && kept.keeps(k, i); },
                                      [&](int, uint32_t k) { return 255 - (k >> shift & 255); }, weight, rank);
            prefix |= (255 - bin) << shift;
            mask |= 255u << shift;
        }
        return FiltCut{prefix, by_id([&](int i, uint32_t k) { return k == prefix && kept.keeps(k, i); }, weight, rank)};
    };
    auto mass = [&](float l) { return filt_mass(a, l, m); };
    auto total = [&](const FiltCut& kept) {
        uint64_t sum = 0, all;
        each([&](int i, float l) { sum += kept.keeps(filt_key(l), i) ? mass(l) : 0ull; });
        filt_scan(sum, s, &all);
        return all;
    };
    FiltCut kept{0u, a.V};
    if (a.top_k < a.V) kept = cut_at(kept, [](float) { return 1ull; }, (uint64_t)a.top_k - 1);
    uint64_t M = total(kept);
    if (a.top_p < 1.0f) {
        kept = cut_at(kept, mass, filt_need(a.top_p, M) - 1);
        M = total(kept);
    }
    return by_id([&](int i, uint32_t k) { return kept.keeps(k, i); }, mass, filt_draw(u, M));
}

// Sorts v[0, N), N a power of two, ascending.
__device__ __forceinline__ void filt_sort(unsigned long long* v, int N) {
    for (int k = 2; k <= N; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            for (int t = threadIdx.x; t < N / 2; t += kFiltThreads) {
                const int lo = (t & ~(j - 1)) * 2 | (t & (j - 1)), hi = lo | j;
                const unsigned long long x = v[lo], y = v[hi];
                if ((x > y) == ((lo & k) == 0)) v[lo] = y, v[hi] = x;
            }
        }
    __syncthreads();
}

// 1. Block maxima; top-k: a histogram of counts, of which a block adds the bins that its own first
// top_k logits reach (lower ones cannot be among the row's).
template <bool BF16, int MODE>
__global__ __launch_bounds__(kFiltThreads) void filt_max_kernel(FiltArgs a) {
    __shared__ FiltShared s;
    __shared__ uint32_t bins[MODE == kFiltTopK ? kFiltCountBins : 1];
    constexpr int PER = kFiltCountBins / kFiltThreads;
    const int tid = threadIdx.x, block = blockIdx.x;
    FiltRow& w = a.ws[blockIdx.y];
    const char* const row = static_cast<const char*>(a.logits) + (int64_t)blockIdx.y * a.stride * (BF16 ? 2 : 4);
    const int first = block * a.chunk, end = min(first + a.chunk, a.V);
    if constexpr (MODE == kFiltTopK) {
        for (int i = tid; i < kFiltCountBins; i += kFiltThreads) bins[i] = 0;
        __syncthreads();
    }
    float m = -INFINITY;
    filt_each<BF16>(row, first, end, [&](int, float l) {
        m = fmaxf(m, l);
        if constexpr (MODE == kFiltTopK) atomicAdd(&bins[filt_key(l) >> kFiltCountShift], 1u);
    });
    m = filt_max(m, s);   // the counts are whole behind its barrier
    if (tid == 0) w.bmax[block] = m;
    if constexpr (MODE == kFiltTopK) {
        const int high = kFiltCountBins - 1 - tid * PER;   // the thread's bins, from the highest
        uint32_t own = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) own += bins[high - i];
        uint64_t all;
        uint64_t above = filt_scan(own, s, &all);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t c = bins[high - i];
            if (c != 0 && above < (uint64_t)a.top_k)
                __hip_atomic_fetch_add(&w.hist.count[high - i], c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            above += c;
        }
    }
}

// The row's maximum, from its blocks'.
__device__ __forceinline__ float filt_row_max(const FiltArgs& a, const FiltRow& w, FiltShared& s) {
    return filt_max(threadIdx.x < a.blocks ? w.bmax[threadIdx.x] : -INFINITY, s);
}

// 2. top-p: masses by bin.
template <bool BF16>
__global__ __launch_bounds__(kFiltThreads) void filt_mass_kernel(FiltArgs a) {
    __shared__ FiltShared s;
    __shared__ unsigned long long bins[kFiltMassBins];
    const int tid = threadIdx.x, first = blockIdx.x * a.chunk, end = min(first + a.chunk, a.V);
    FiltRow& w = a.ws[blockIdx.y];
    const char* const row = static_cast<const char*>(a.logits) + (int64_t)blockIdx.y * a.stride * (BF16 ? 2 : 4);
    for (int i = tid; i < kFiltMassBins; i += kFiltThreads) bins[i] = 0;
    const float m = filt_row_max(a, w, s);
    __syncthreads();
    filt_each<BF16>(row, first, end, [&](int, float l) {
        const uint64_t x = filt_mass(a, l, m);
        if (x != 0) atomicAdd(&bins[filt_bin(a, l, m)], (unsigned long long)x);
    });
    __syncthreads();
    for (int i = tid; i < kFiltMassBins; i += kFiltThreads)
        if (bins[i] != 0) __hip_atomic_fetch_add(&w.hist.mass[i], bins[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The last step: see the top. What a row's blocks hand to its last workgroup goes through agent-scope
// stores that have returned before the block counts in, and agent-scope loads.
template <bool BF16, int MODE>
__global__ __launch_bounds__(kFiltThreads) void filt_draw_kernel(FiltArgs a) {
    __shared__ FiltShared s;
    __shared__ unsigned long long buf[kFiltSort];   // the block's part of the list, then the row's list
    __shared__ unsigned long long sums[kFiltBlocks];
    __shared__ uint32_t s_count, s_base;
    const int tid = threadIdx.x, block = blockIdx.x;
    FiltRow& w = a.ws[blockIdx.y];
    const char* const row = static_cast<const char*>(a.logits) + (int64_t)blockIdx.y * a.stride * (BF16 ? 2 : 4);
    const int first = block * a.chunk, end = min(first + a.chunk, a.V);
    if (tid == 0) s_count = 0;
    const float m = filt_row_max(a, w, s);
    // where K or N ends: the bin, and what lies above it
    int bin = 0;
    uint64_t above = 0, W = 0;
    if constexpr (MODE == kFiltTopK) {
        constexpr int PER = kFiltCountBins / kFiltThreads;
        const int high = kFiltCountBins - 1 - tid * PER;
        uint32_t c[PER], own = 0;
#pragma unroll
        for (int i = 0; i < PER; i += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(&w.hist.count[high - i - 3]);
            c[i] = x.w, c[i + 1] = x.z, c[i + 2] = x.y, c[i + 3] = x.x;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) own += c[i];
        uint64_t all, excl = filt_scan(own, s, &all);
        const uint64_t rank = (uint64_t)a.top_k - 1;
        if (excl <= rank && rank - excl < own) {
            int at = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (excl <= rank) at = high - i;
                excl += c[i];
            }
            s.sel[0] = at;
        }
        __syncthreads();
        bin = (int)s.sel[0];
    }
    if constexpr (MODE == kFiltTopP) {
        constexpr int PER = kFiltMassBins / kFiltThreads;
        uint64_t h[PER], own = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) own += h[i] = w.hist.mass[tid * PER + i];
        uint64_t excl = filt_scan(own, s, &W);
        const uint64_t rank = filt_need(a.top_p, W) - 1;
        if (excl <= rank && rank - excl < own) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (excl <= rank) s.sel[0] = tid * PER + i, s.sel[1] = excl;
                excl += h[i];
            }
        }
        __syncthreads();
        bin = (int)s.sel[0], above = s.sel[1];
    }
    __syncthreads();
    uint64_t mine = 0;
    auto enlist = [&](int i, uint32_t key) {
        const unsigned long long x = (unsigned long long)~key << 32 | (uint32_t)i;
        const uint32_t at = atomicAdd(&s_count, 1u);
        if (at < kFiltSort) buf[at] = x;
    };
    if (m > -INFINITY)
        filt_each<BF16>(row, first, end, [&](int i, float l) {
            if constexpr (MODE == kFiltTopK) {
                const uint32_t k = filt_key(l);
                if ((int)(k >> kFiltCountShift) >= bin) enlist(i, k);
            } else if constexpr (MODE == kFiltTopP) {
                const int b = filt_bin(a, l, m);
                if (b < bin) mine += filt_mass(a, l, m);
                else if (b == bin) enlist(i, filt_key(l));
            } else {
                mine += filt_mass(a, l, m);
            }
        });
    if constexpr (MODE != kFiltTopK) {
        uint64_t all;
        filt_scan(mine, s, &all);
        mine = all;
    }
    __syncthreads();
    if constexpr (MODE != kFiltAll) {
        const uint32_t n = s_count;
        if (tid == 0 && n != 0) {
            // a block whose part does not fit makes the row's list overflow
            s_base = __hip_atomic_fetch_add(&w.count, n <= kFiltSort ? n : (uint32_t)kFiltList + 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (n <= kFiltSort)
            for (uint32_t i = tid; i < n; i += kFiltThreads)
                if (s_base + i < kFiltList) __hip_atomic_store(&w.list[s_base + i], buf[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (MODE != kFiltTopK && tid == 0) __hip_atomic_store(&w.bmass[block], mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0)
        s.flag = __hip_atomic_fetch_add(&w.counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)a.blocks - 1;
    __syncthreads();
    if (!s.flag) return;

    // ---- the row's last workgroup
    const float u = a.u[blockIdx.y];
    const uint32_t count = MODE == kFiltAll ? 0u : __hip_atomic_load(&w.count, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (tid == 0) w.counter = 0, w.count = 0;
    if constexpr (MODE == kFiltTopK)
        for (int i = tid; i < kFiltCountBins; i += kFiltThreads) w.hist.count[i] = 0;
    if constexpr (MODE == kFiltTopP)
        for (int i = tid; i < kFiltMassBins; i += kFiltThreads) w.hist.mass[i] = 0;
    if (m == -INFINITY) {
        if (tid == 0) a.out[blockIdx.y] = -1;
        return;
    }
    if (count > kFiltSort) {
        int token;
        if (MODE == kFiltTopK && count <= kFiltList)
            token = filt_select(a, m, u, s, [&](auto f) {
                for (uint32_t i = tid; i < count; i += kFiltThreads) {
                    const unsigned long long x = __hip_atomic_load(&w.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    f((int)(uint32_t)x, filt_logit(~(uint32_t)(x >> 32)));
                }
            });
        else
            token = filt_select(a, m, u, s, [&](auto f) { filt_each<BF16>(row, 0, a.V, f); });
        if (tid == 0) a.out[blockIdx.y] = token;
        return;
    }
    // the list in the sampler's order; a thread has PER neighbours of it
    constexpr int PER = kFiltSort / kFiltThreads;
    uint64_t x[PER];
    uint64_t mass[PER];
    int N = 0;
    if constexpr (MODE != kFiltAll) {
        N = 2;
        while (N < (int)count) N *= 2;
        for (int i = tid; i < N; i += kFiltThreads)
            buf[i] = i < (int)count ? __hip_atomic_load(&w.list[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : ~0ull;
        filt_sort(buf, N);
        uint64_t own = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = tid * PER + i;
            x[i] = at < N ? buf[at] : ~0ull;
            mass[i] = 0;
            if (at < (int)count && (MODE == kFiltTopP || at < a.top_k)) mass[i] = filt_mass(a, filt_logit(~(uint32_t)(x[i] >> 32)), m);
            own += mass[i];
        }
        if (MODE == kFiltTopP || a.top_p < 1.0f) {
            uint64_t all, before = filt_scan(own, s, &all);
            const uint64_t need = MODE == kFiltTopP ? filt_need(a.top_p, W) - above : filt_need(a.top_p, all);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint64_t y = mass[i];
                if (before >= need) mass[i] = 0;
                before += y;
            }
        }
    }
    if constexpr (MODE == kFiltTopK) {
        // the draw, in the order of ids: masses join their ids
        __syncthreads();
        uint64_t own = 0, M;
#pragma unroll
        for (int i = 0; i < PER; ++i) own += mass[i];
        filt_scan(own, s, &M);
        const uint64_t r = filt_draw(u, M);
        // ids of kept ones with their places, sorted by id
        __shared__ unsigned long long masses[kFiltSort];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = tid * PER + i;
            if (at < N) buf[at] = mass[i] != 0 ? (x[i] & 0xffffffffull) << 32 | (uint32_t)at : ~0ull, masses[at] = mass[i];
        }
        filt_sort(buf, N);
        own = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = tid * PER + i;
            x[i] = at < N ? buf[at] : ~0ull;
            mass[i] = x[i] != ~0ull ? masses[(uint32_t)x[i]] : 0ull;
            own += mass[i];
        }
        uint64_t excl = filt_scan(own, s, &M);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (excl <= r && r - excl < mass[i]) a.out[blockIdx.y] = (int32_t)(x[i] >> 32);
            excl += mass[i];
        }
    } else {
        // masses of the blocks, and of the list's kept ids in theirs
        FiltCut kept{0u, a.V};
        __syncthreads();
        if (tid < kFiltBlocks)
            sums[tid] = tid < a.blocks ? __hip_atomic_load(&w.bmass[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0ull;
        __syncthreads();
        if constexpr (MODE == kFiltTopP) {
            // the last that is kept: its successor is not
            unsigned long long last = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (mass[i] != 0) {
                    atomicAdd(&sums[(uint32_t)x[i] / (uint32_t)a.chunk], (unsigned long long)mass[i]);
                    last = x[i];   // neighbours ascend
                }
            if (tid == 0) s.sel[0] = 0;
            __syncthreads();
            if (last != 0) atomicMax(&s.sel[0], last);
            __syncthreads();
            last = s.sel[0];
            kept = FiltCut{~(uint32_t)(last >> 32), (int)(uint32_t)last};
            __syncthreads();
        }
        uint64_t before, M;
        const uint64_t own = tid < kFiltBlocks ? sums[tid] : 0ull;
        filt_scan(own, s, &M);
        uint64_t r = filt_draw(u, M);
        const int b = filt_find(own, r, s, &before);
        r -= before;
        // the block's tiles of 256 vectors, then the id
        constexpr int TILE = kFiltThreads * (BF16 ? 8 : 4);
        const int b0 = b * a.chunk, b1 = min(b0 + a.chunk, a.V);
        auto weigh = [&](int i, float l) { return kept.keeps(filt_key(l), i) ? filt_mass(a, l, m) : 0ull; };
        __syncthreads();
        s.bins[tid] = 0;
        __syncthreads();
        filt_each<BF16>(row, b0, b1, [&](int i, float l) {
            const uint64_t y = weigh(i, l);
            if (y != 0) atomicAdd(&s.bins[(i - b0) / TILE], (unsigned long long)y);
        });
        __syncthreads();
        const int t = filt_find(s.bins[tid], r, s, &before);
        r -= before;
        const int t0 = b0 + t * TILE;
        constexpr int E = TILE / kFiltThreads;
        uint64_t y[E], sum = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = t0 + tid * E + e;
            y[e] = 0;
            if (i < b1) {
                float l;
                if constexpr (BF16) l = bf16_to_f32(reinterpret_cast<const uint16_t*>(row)[i]);
                else l = reinterpret_cast<const float*>(row)[i];
                y[e] = weigh(i, filt_clean(l));
            }
            sum += y[e];
        }
        uint64_t excl = filt_scan(sum, s, &M);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (excl <= r && r - excl < y[e]) a.out[blockIdx.y] = t0 + tid * E + e;
            excl += y[e];
        }
    }
}

// Small vocabularies: a workgroup a row, the row in LDS.
template <bool BF16>
__global__ __launch_bounds__(kFiltThreads) void filt_row_kernel(FiltArgs a) {
    __shared__ FiltShared s;
    extern __shared__ float held[];
    const int tid = threadIdx.x;
    const char* const row = static_cast<const char*>(a.logits) + (int64_t)blockIdx.x * a.stride * (BF16 ? 2 : 4);
    float m = -INFINITY;
    filt_each<BF16>(row, 0, a.V, [&](int i, float l) { m = fmaxf(m, l), held[i] = l; });
    m = filt_max(m, s);
    int token = -1;
    if (m > -INFINITY)
        token = filt_select(a, m, a.u[blockIdx.x], s, [&](auto f) {
            for (int i = tid; i < a.V; i += kFiltThreads) f(i, held[i]);
        });
    if (tid == 0) a.out[blockIdx.x] = token;
}

// Blocks of a row: some four workgroups a CU in all, blocks of whole passes of a workgroup's loads.
static void filt_split(int64_t rows, int64_t vocab, int* blocks, int* chunk) {
    const int64_t want = std::min<int64_t>(kFiltBlocks, std::max<int64_t>(1, (4 * prefill_cus() + rows - 1) / rows));
    int64_t c = std::min<int64_t>((vocab + want - 1) / want, kFiltMaxTiles * kFiltThreads * 4 - 2047);
    c = (c + 2047) / 2048 * 2048;
    *chunk = (int)c;
    *blocks = (int)((vocab + c - 1) / c);
}

template <bool BF16>
static void filt_launch(const FiltArgs& a, int64_t rows, hipStream_t stream) {
    const dim3 t(kFiltThreads);
    if (a.ws == nullptr) {
        hipLaunchKernelGGL(filt_row_kernel<BF16>, dim3((unsigned)rows), t, (unsigned)a.V * sizeof(float), stream, a);
        return;
    }
    const dim3 grid(a.blocks, (unsigned)rows);
    if (a.top_k < a.V) {
        hipLaunchKernelGGL((filt_max_kernel<BF16, kFiltTopK>), grid, t, 0, stream, a);
        hipLaunchKernelGGL((filt_draw_kernel<BF16, kFiltTopK>), grid, t, 0, stream, a);
        return;
    }
    hipLaunchKernelGGL((filt_max_kernel<BF16, kFiltAll>), grid, t, 0, stream, a);
    if (a.top_p < 1.0f) {
        hipLaunchKernelGGL(filt_mass_kernel<BF16>, grid, t, 0, stream, a);
        hipLaunchKernelGGL((filt_draw_kernel<BF16, kFiltTopP>), grid, t, 0, stream, a);
    } else {
        hipLaunchKernelGGL((filt_draw_kernel<BF16, kFiltAll>), grid, t, 0, stream, a);
    }
}

}  // namespace efm

using namespace efm;

extern "C" size_t efm_sampler_filtered_workspace_bytes(int64_t rows, int64_t vocab) {
    return rows <= 0 || vocab <= kFiltLdsVocab ? 0 : (size_t)rows * sizeof(FiltRow);
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
