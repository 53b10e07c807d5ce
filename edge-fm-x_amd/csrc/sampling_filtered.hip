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
#include "common.hpp"

#include <cmath>

namespace efm {

constexpr int kFiltThreads = 1024;
constexpr int kFiltWaves = kFiltThreads / kWave;
constexpr int kFiltMaxVocab = 1 << 20;
constexpr double kFiltOne = 17592186044416.0;   // 2^44

struct FiltArgs {
    const void* logits;
    int64_t stride;
    int V, top_k;
    float top_p;
    double to_log2;      // log2(e) / T
    uint64_t min_mass;   // max(1, ceil(min_p 2^44))
    const float* u;
    int32_t* out;
};

// w of a logit, m the row's largest. 2^t, t = (l - m) log2(e) / T, as 2^n 2^f with the series of
// exp(f ln 2), |f| <= 1/2: the term after the last is below 2^-52. Adding 2^52 rounds to an integer.
__device__ __forceinline__ uint64_t filt_mass(float l, float m, double to_log2) {
    const double t = l == m ? 0.0 : ((double)l - (double)m) * to_log2;
    if (!(t > -46.0)) return 0;
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
    const double w = __builtin_ldexp(p, (int)n + 44) + 4503599627370496.0;
    return __builtin_bit_cast(uint64_t, w) & 0xfffffffffffffull;
}

// Unsigned keys that order as the logits do (zeros of both signs alike).
__device__ __forceinline__ uint32_t filt_key(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float filt_clean(float l) { return l == l ? l : -INFINITY; }

template <bool BF16>
__device__ __forceinline__ float filt_load(const void* row, int i) {
    if constexpr (BF16) return filt_clean(bf16_to_f32(static_cast<const uint16_t*>(row)[i]));
    else return filt_clean(static_cast<const float*>(row)[i]);
}

// f(id, logit) for every logit of the row.
template <bool BF16, typename F>
__device__ __forceinline__ void filt_each(const void* row, int V, F f) {
    for (int i = threadIdx.x; i < V; i += kFiltThreads) f(i, filt_load<BF16>(row, i));
}

__device__ __forceinline__ uint64_t filt_wave_scan(uint64_t v, int lane) {
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const uint64_t o = __shfl_up(v, off, kWave);
        if (lane >= off) v += o;
    }
    return v;
}

// Sum of the values of the threads before this one, and of all.
__device__ __forceinline__ uint64_t filt_scan(uint64_t v, unsigned long long* red, uint64_t* total) {
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint64_t incl = filt_wave_scan(v, lane);
    __syncthreads();
    if (lane == kWave - 1) red[wave] = incl;
    __syncthreads();
    uint64_t before = 0, all = 0;
    for (int w = 0; w < kFiltWaves; ++w) {
        if (w < wave) before += red[w];
        all += red[w];
    }
    *total = all;
    return before + incl - v;
}

// The bin that holds unit `rank` (from 0) of the 1024 bins' contents in the order of the threads'
// bins, and what lies before that bin; every thread gets both. rank is below the total.
__device__ __forceinline__ int filt_find(uint64_t own, uint64_t rank, unsigned long long* red, unsigned long long* sel, uint64_t* before) {
    uint64_t all;
    const uint64_t excl = filt_scan(own, red, &all);
    if (excl <= rank && rank < excl + own) sel[0] = threadIdx.x, sel[1] = excl;
    __syncthreads();
    *before = sel[1];
    return (int)sel[0];
}

// What the choices so far keep: keys above `key`, and of those equal to it the ids up to `id`.
struct FiltCut {
    uint32_t key;
    int id;
    __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= id); }
};

// One workgroup a row, every pass over the row itself.
template <bool BF16>
__global__ __launch_bounds__(kFiltThreads) void filt_row_kernel(FiltArgs a) {
    __shared__ unsigned long long hist[1024];
    __shared__ unsigned long long red[kFiltWaves];
    __shared__ unsigned long long sel[2];
    __shared__ float redf[kFiltWaves];
    const int tid = threadIdx.x;
    const char* const row = static_cast<const char*>(a.logits) + (int64_t)blockIdx.x * a.stride * (BF16 ? 2 : 4);
    float m = -INFINITY;
    filt_each<BF16>(row, a.V, [&](int, float l) { m = fmaxf(m, l); });
    m = wave_max(m);
    if (tid % kWave == 0) redf[tid / kWave] = m;
    __syncthreads();
    for (int w = 0; w < kFiltWaves; ++w) m = fmaxf(m, redf[w]);
    if (m == -INFINITY) {
        if (tid == 0) a.out[blockIdx.x] = -1;
        return;
    }
    auto mass = [&](float l) {
        const uint64_t w = filt_mass(l, m, a.to_log2);
        return w >= a.min_mass ? w : 0ull;
    };
    // A weight of each id, 1 or its mass, is histogrammed digit by digit from the top; of ids with the
    // same key the lowest count first. The cut keeps weights up to and with unit `rank`.
    auto cut_at = [&](const FiltCut& kept, uint64_t rank, auto weight) {
        uint32_t prefix = 0, mask = 0;
        uint64_t before;
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            hist[tid] = 0;
            __syncthreads();
            filt_each<BF16>(row, a.V, [&](int i, float l) {
                const uint32_t k = filt_key(l);
                if ((k & mask) == prefix && kept.keeps(k, i)) {
                    const uint64_t w = weight(l);
                    if (w != 0) atomicAdd(&hist[255 - (k >> shift & 255)], (unsigned long long)w);
                }
            });
            __syncthreads();
            const int bin = filt_find(hist[tid], rank, red, sel, &before);
            rank -= before;
            prefix |= (uint32_t)(255 - bin) << shift;
            mask |= 255u << shift;
        }
        // among the ids of this key, by id
        uint32_t top = 0;
        for (int shift = 10; shift >= 0; shift -= 10) {
            __syncthreads();
            hist[tid] = 0;
            __syncthreads();
            filt_each<BF16>(row, a.V, [&](int i, float l) {
                const uint32_t k = filt_key(l);
                if (k == prefix && kept.keeps(k, i) && (shift == 10 || (uint32_t)i >> 10 == top)) {
                    const uint64_t w = weight(l);
                    if (w != 0) atomicAdd(&hist[i >> shift & 1023], (unsigned long long)w);
                }
            });
            __syncthreads();
            const int bin = filt_find(hist[tid], rank, red, sel, &before);
            rank -= before;
            top = shift == 10 ? (uint32_t)bin : top << 10 | (uint32_t)bin;
        }
        return FiltCut{prefix, (int)top};
    };
    auto total = [&](const FiltCut& kept) {
        uint64_t s = 0, all;
        filt_each<BF16>(row, a.V, [&](int i, float l) { s += kept.keeps(filt_key(l), i) ? mass(l) : 0ull; });
        filt_scan(s, red, &all);
        return all;
    };
    FiltCut kept{0u, a.V};
    if (a.top_k > 0 && a.top_k < a.V) kept = cut_at(kept, (uint64_t)a.top_k - 1, [](float) { return 1ull; });
    if (a.top_p < 1.0f) {
        const uint64_t W = total(kept);
        uint64_t need = (uint64_t)__builtin_ceil((double)a.top_p * (double)W);
        need = need < 1 ? 1 : need > W ? W : need;
        kept = cut_at(kept, need - 1, mass);
    }
    const uint64_t M = total(kept);
    const double x = (double)a.u[blockIdx.x] * (double)M;
    uint64_t r = x > 0.0 ? (uint64_t)__builtin_fmin(x, 9.2e18) : 0ull;
    r = r < M ? r : M - 1;
    uint64_t before;
    uint32_t top = 0;
    for (int shift = 10; shift >= 0; shift -= 10) {
        __syncthreads();
        hist[tid] = 0;
        __syncthreads();
        filt_each<BF16>(row, a.V, [&](int i, float l) {
            if (!kept.keeps(filt_key(l), i) || (shift == 0 && (uint32_t)i >> 10 != top)) return;
            const uint64_t w = mass(l);
            if (w != 0) atomicAdd(&hist[i >> shift & 1023], (unsigned long long)w);
        });
        __syncthreads();
        const int bin = filt_find(hist[tid], r, red, sel, &before);
        r -= before;
        top = shift == 10 ? (uint32_t)bin : top << 10 | (uint32_t)bin;
    }
    if (tid == 0) a.out[blockIdx.x] = (int32_t)top;
}

}  // namespace efm

using namespace efm;

extern "C" size_t efm_sampler_filtered_workspace_bytes(int64_t rows, int64_t vocab) {
    (void)rows, (void)vocab;
    return 0;
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
    if (rows > (1 << 20)) return set_error(EFM_ERR_UNSUPPORTED, "sampler_filtered: %lld rows", (long long)rows);
    FiltArgs a;
    a.logits = logits;
    a.stride = logits_stride != 0 ? logits_stride : vocab;
    a.V = (int)vocab;
    a.top_k = top_k;
    a.top_p = top_p;
    a.to_log2 = 1.4426950408889634074 / (double)temperature;
    a.min_mass = min_p > 0.f ? (uint64_t)std::ceil((double)min_p * kFiltOne) : 1;
    if (a.min_mass < 1) a.min_mass = 1;
    a.u = uniforms;
    a.out = token_out;
    if (logits_dtype == EFM_DTYPE_BF16) hipLaunchKernelGGL(filt_row_kernel<true>, dim3((unsigned)rows), dim3(kFiltThreads), 0, stream, a);
    else hipLaunchKernelGGL(filt_row_kernel<false>, dim3((unsigned)rows), dim3(kFiltThreads), 0, stream, a);
    return check_launch("sampler_filtered");
}
