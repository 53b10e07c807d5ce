// Norm of queries and keys per head, position rotation and cache write in one pass, into a bf16
// cache or an FP4 one (fp4.hpp), and the FP4 cache read back.
//
// For a head's row x: y = x * rsqrt(mean(x^2) + eps) * w (without weights y = x), then the pair
// (d, d + hd / 2) of y is turned by the angle pos * theta^(-2 d / hd) / rope_scale. A row is
// rounded once, at the end. The angle is reduced in 64 bits (in turns: pos times a 64-bit
// frequency, less its whole part), so far positions lose nothing; sine and cosine are computed
// once a token and shared by its heads through LDS. Keys of an FP4 cache are computed in 64 bits
// throughout, a small part of the row's work: a value next to a border of the grid lands on its
// own side, whatever the order of a sum.
#include "fp4.hpp"

#include <cmath>

namespace efm {

int validate_attention_ctx(const efm_attention_ctx* c, const char* who);

struct QkWriteArgs {
    const bf16_t* qkv;       // [S, qkv_sn]: q at 0, k at Hq*hd, v at (Hq+Hkv)*hd
    const bf16_t* q_w;       // [hd] or NULL
    const bf16_t* k_w;
    bf16_t* q_out;           // NULL: queries are not wanted
    bf16_t* k_cache;         // bf16 cache
    bf16_t* v_cache;
    uint8_t* cache;          // FP4 cache
    const uint32_t* d_kv_len;
    const int32_t* pos;      // [3, pos_stride] or NULL
    int64_t qkv_sn;
    int64_t q_sn, q_sh, k_sn, k_sh, v_sn, v_sh;
    int64_t pos_stride;
    uint32_t max_rows, S, base;
    int Hq, Hkv, rotate, cum0, cum1;
    uint32_t q_off, k_off;
    float eps;
    double turns[kMaxHalfDim];   // theta^(-2 d / hd) / rope_scale / (2 pi)
};

// Row y of 8 values from the lane's 8 and, in `other`, those of the lane that holds the other half
// of its pairs; lo: this lane holds the first half.
template <typename T>
__device__ __forceinline__ void turn8(T* x, const double2* cs, int lane_mask, bool lo) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const T o = __shfl_xor(x[e], lane_mask, kWave);
        const T c = (T)cs[e].x, s = (T)cs[e].y;
        x[e] = lo ? x[e] * c - o * s : x[e] * c + o * s;
    }
}

template <typename T, int LANES>
__device__ __forceinline__ void norm8(T* x, uint4 weight, T eps) {
    T sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += x[e] * x[e];
#pragma unroll
    for (int m = 1; m < LANES; m *= 2) sum += __shfl_xor(sum, m, kWave);
    const T r = (T)1 / sqrt(sum / (T)(8 * LANES) + eps);
    float w[8];
    unpack8(weight, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * r * (T)w[e];
}

// One workgroup a token; HD / 8 lanes a head.
template <int HD, bool FP4>
__global__ __launch_bounds__(256) void qk_norm_rope_write_kernel(QkWriteArgs a) {
    constexpr int LANES = HD / 8, HALF = HD / 2;
    __shared__ double2 cs[2][HALF];   // [query, key] (cos, sin)
    const uint32_t t = blockIdx.x;
    uint32_t base = a.base;
    if (a.d_kv_len != nullptr) {
        const uint32_t L = a.d_kv_len[0];
        if (L < a.S || L > a.max_rows) return;
        base = L - a.S;
    }
    const uint32_t row = base + t;
    const bf16_t* const src = a.qkv + (int64_t)t * a.qkv_sn;
    if (a.rotate) {
        for (int i = threadIdx.x; i < HD; i += 256) {
            const int d = i % HALF, is_k = i / HALF;
            double p;
            if (a.pos != nullptr) p = (double)a.pos[(d < a.cum0 ? 0 : d < a.cum1 ? 1 : 2) * a.pos_stride + t];
            else p = (double)row + (double)(is_k ? a.k_off : a.q_off);
            const double turn = p * a.turns[d];
            double s, c;
            sincospi(2.0 * (turn - rint(turn)), &s, &c);
            cs[is_k][d] = make_double2(c, s);
        }
        __syncthreads();
    }
    const KvFp4Layout lay(KvFp4Layout::rows(a.max_rows), a.Hkv, HD);
    const int j = threadIdx.x % LANES;
    const bool lo = j < LANES / 2;
    const int heads = a.Hq + 2 * a.Hkv;
    const int first = a.q_out != nullptr ? 0 : a.Hq;
    // whole waves walk the heads together: lanes exchange halves inside a head
    for (int h0 = first + threadIdx.x / kWave * (kWave / LANES); h0 < heads; h0 += 256 / LANES) {
        const int h = h0 + threadIdx.x % kWave / LANES;
        const bool on = h < heads;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (on) raw = *reinterpret_cast<const uint4*>(src + (int64_t)h * HD + 8 * j);
        const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + a.Hkv;
        const bf16_t* const w = is_q ? a.q_w : a.k_w;
        if constexpr (FP4) {
            if (__any(is_k)) {
                float f[8];
                unpack8(raw, f);
                double x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (double)f[e];
                if (a.k_w != nullptr) norm8<double, LANES>(x, reinterpret_cast<const uint4*>(a.k_w)[j], (double)a.eps);
                if (a.rotate) turn8<double>(x, &cs[1][8 * (j % (LANES / 2))], LANES / 2, lo);
                uint64_t top = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    top = max(top, (uint64_t)(__double_as_longlong(x[e]) & 0x7fffffffffffffffll));
                top = max(top, (uint64_t)__shfl_xor((unsigned long long)top, 1, kWave));
                top = max(top, (uint64_t)__shfl_xor((unsigned long long)top, 2, kWave));
                const uint32_t byte = fp4_scale_byte(top);
                const uint32_t word = fp4_encode8(x, byte);
                if (is_k) {
                    const int kh = h - a.Hq;
                    *reinterpret_cast<uint32_t*>(a.cache + lay.k(kh) + lay.k_word(row, j)) = word;
                    if (j % 4 == 0) a.cache[lay.ks(kh) + lay.k_scale(row, j)] = (uint8_t)byte;
                }
            }
        }
        float x[8];
        unpack8(raw, x);
        if (FP4 ? __any(on && !is_q && !is_k) : false) {
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            top = max(top, (uint32_t)__shfl_xor((int)top, 1, kWave));
            top = max(top, (uint32_t)__shfl_xor((int)top, 2, kWave));
            const uint32_t byte = fp4_scale_byte(top);
            if (on && !is_q && !is_k) {
                const int vh = h - a.Hq - a.Hkv;
                *reinterpret_cast<uint32_t*>(a.cache + lay.v(vh) + lay.v_word(row, j)) = fp4_encode8(x, byte);
                if (j % 4 == 0) a.cache[lay.vs(vh) + lay.v_scale(row, j)] = (uint8_t)byte;
            }
        }
        // queries, and keys of a bf16 cache
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[e];
        if (w != nullptr) norm8<float, LANES>(y, reinterpret_cast<const uint4*>(w)[j], a.eps);
        if (a.rotate) turn8<float>(y, &cs[is_q ? 0 : 1][8 * (j % (LANES / 2))], LANES / 2, lo);
        if (!on) continue;
        if (is_q) {
            *reinterpret_cast<uint4*>(a.q_out + (int64_t)t * a.q_sn + (int64_t)h * a.q_sh + 8 * j) = pack8(y);
        } else if (!FP4) {
            if (is_k)
                *reinterpret_cast<uint4*>(a.k_cache + (int64_t)row * a.k_sn + (int64_t)(h - a.Hq) * a.k_sh + 8 * j) = pack8(y);
            else
                *reinterpret_cast<uint4*>(a.v_cache + (int64_t)row * a.v_sn + (int64_t)(h - a.Hq - a.Hkv) * a.v_sh + 8 * j) = raw;
        }
    }
}

// One lane for 8 channels of a row.
template <int HD>
__global__ __launch_bounds__(256) void kv_fp4_read_kernel(const uint8_t* cache, KvFp4Layout lay, uint32_t first, int64_t octets,
                                                          uint4* k_out, uint4* v_out) {
    const int64_t i = blockIdx.x * 256ll + threadIdx.x;
    if (i >= octets) return;
    const int j = (int)(i % (HD / 8)), h = (int)(i / (HD / 8) % lay.Hkv);
    const size_t row = first + (size_t)(i / (HD / 8) / lay.Hkv);
    if (k_out != nullptr) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(cache + lay.k(h) + lay.k_word(row, j));
        k_out[i] = __builtin_bit_cast(uint4, fp4_unpack8(w, fp4_scale(cache[lay.ks(h) + lay.k_scale(row, j)])));
    }
    if (v_out != nullptr) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(cache + lay.v(h) + lay.v_word(row, j));
        v_out[i] = __builtin_bit_cast(uint4, fp4_unpack8(w, fp4_scale(cache[lay.vs(h) + lay.v_scale(row, j)])));
    }
}

static bool qk_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static int qk_write(const char* who, bool fp4, const efm_attention_ctx* ctx, const void* qkv, int64_t qkv_stride_n,
                    const void* q_norm_w, const void* k_norm_w, float eps, void* q_out, void* k_cache, void* v_cache,
                    uint32_t max_rows, uint32_t seq_len, uint32_t base, const uint32_t* d_kv_len,
                    const int32_t* position_ids, int32_t position_stride, int32_t s0, int32_t s1, int32_t s2,
                    hipStream_t stream) {
    const int rc = validate_attention_ctx(ctx, who);
    if (rc) return rc;
    if (!qkv || !k_cache || (!fp4 && !v_cache)) return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    const int64_t hd = ctx->head_dim, Hq = ctx->num_qo_heads, Hkv = ctx->num_kv_heads;
    const int64_t width = (Hq + 2 * Hkv) * hd;
    if (Hq > (1 << 16)) return set_error(EFM_ERR_UNSUPPORTED, "%s: %lld query heads", who, (long long)Hq);
    QkWriteArgs a;
    a.qkv_sn = qkv_stride_n ? qkv_stride_n : width;
    if (a.qkv_sn < width || a.qkv_sn % 8 != 0)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: qkv_stride_n %lld (at least %lld, a multiple of 8)", who,
                         (long long)a.qkv_sn, (long long)width);
    if (!qk_aligned(qkv) || !qk_aligned(q_norm_w) || !qk_aligned(k_norm_w) || !qk_aligned(q_out) || !qk_aligned(k_cache) ||
        !qk_aligned(v_cache))
        return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: pointers must be 16-byte aligned", who);
    if ((q_norm_w || k_norm_w) && !(eps >= 0.f)) return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: eps %g", who, (double)eps);
    if (max_rows > (1u << 24)) return set_error(EFM_ERR_UNSUPPORTED, "%s: max_rows %u too large", who, max_rows);
    if (seq_len > max_rows || (d_kv_len == nullptr && base > max_rows - seq_len))
        return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: rows %u + %u do not fit max_rows %u", who, base, seq_len, max_rows);
    const bool rotate = ctx->pos_encoding == EFM_POS_ROPE_LLAMA;
    if (position_ids != nullptr) {
        if (!rotate) return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: position_ids without a position encoding", who);
        if (s0 < 0 || s1 < 0 || s2 < 0 || (int64_t)s0 + s1 + s2 != hd / 2)
            return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: sections %d+%d+%d must sum to head_dim/2 = %lld", who, s0, s1, s2,
                             (long long)(hd / 2));
        if (position_stride < 0 || (uint32_t)position_stride < seq_len)
            return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: position_stride < seq_len", who);
    }
    if (seq_len == 0) return EFM_OK;
    a.qkv = static_cast<const bf16_t*>(qkv);
    a.q_w = static_cast<const bf16_t*>(q_norm_w);
    a.k_w = static_cast<const bf16_t*>(k_norm_w);
    a.q_out = static_cast<bf16_t*>(q_out);
    a.k_cache = fp4 ? nullptr : static_cast<bf16_t*>(k_cache);
    a.v_cache = static_cast<bf16_t*>(v_cache);
    a.cache = fp4 ? static_cast<uint8_t*>(k_cache) : nullptr;
    a.d_kv_len = d_kv_len;
    a.pos = position_ids;
    a.pos_stride = position_stride;
    a.q_sn = ctx->q_stride_n ? ctx->q_stride_n : Hq * hd;
    a.q_sh = ctx->q_stride_h ? ctx->q_stride_h : hd;
    a.k_sn = ctx->k_stride_n ? ctx->k_stride_n : Hkv * hd;
    a.k_sh = ctx->k_stride_h ? ctx->k_stride_h : hd;
    a.v_sn = ctx->kv_stride_n ? ctx->kv_stride_n : Hkv * hd;
    a.v_sh = ctx->kv_stride_h ? ctx->kv_stride_h : hd;
    a.max_rows = max_rows;
    a.S = seq_len;
    a.base = base;
    a.Hq = (int)Hq;
    a.Hkv = (int)Hkv;
    a.rotate = rotate;
    a.cum0 = s0;
    a.cum1 = s0 + s1;
    a.q_off = ctx->q_rope_pos_offset;
    a.k_off = ctx->k_rope_pos_offset;
    a.eps = eps;
    for (int d = 0; d < kMaxHalfDim; ++d)
        a.turns[d] = rotate && d < hd / 2 ? exp(-2.0 * d / (double)hd * log((double)ctx->rope_theta)) /
                                                (double)ctx->rope_scale / 6.283185307179586476925
                                          : 0.0;
    const dim3 grid(seq_len), block(256);
    if (hd == 128 && fp4) hipLaunchKernelGGL((qk_norm_rope_write_kernel<128, true>), grid, block, 0, stream, a);
    else if (hd == 128) hipLaunchKernelGGL((qk_norm_rope_write_kernel<128, false>), grid, block, 0, stream, a);
    else if (fp4) hipLaunchKernelGGL((qk_norm_rope_write_kernel<64, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((qk_norm_rope_write_kernel<64, false>), grid, block, 0, stream, a);
    return check_launch(who);
}

}  // namespace efm

using namespace efm;

extern "C" int efm_qk_norm_rope_write_kv(const efm_attention_ctx* ctx, const void* qkv, int64_t qkv_stride_n,
                                         const void* q_norm_w, const void* k_norm_w, float eps, void* q_out, void* k_cache,
                                         void* v_cache, uint32_t max_rows, uint32_t seq_len, uint32_t base,
                                         const uint32_t* d_kv_len, const int32_t* position_ids, int32_t position_stride,
                                         int32_t section0, int32_t section1, int32_t section2, hipStream_t stream) {
    return qk_write("qk_norm_rope_write_kv", false, ctx, qkv, qkv_stride_n, q_norm_w, k_norm_w, eps, q_out, k_cache, v_cache,
                    max_rows, seq_len, base, d_kv_len, position_ids, position_stride, section0, section1, section2, stream);
}

extern "C" int efm_qk_norm_rope_write_kv_fp4(const efm_attention_ctx* ctx, const void* qkv, int64_t qkv_stride_n,
                                             const void* q_norm_w, const void* k_norm_w, float eps, void* q_out, void* cache,
                                             uint32_t max_rows, uint32_t seq_len, uint32_t base, const uint32_t* d_kv_len,
                                             const int32_t* position_ids, int32_t position_stride, int32_t section0,
                                             int32_t section1, int32_t section2, hipStream_t stream) {
    return qk_write("qk_norm_rope_write_kv_fp4", true, ctx, qkv, qkv_stride_n, q_norm_w, k_norm_w, eps, q_out, cache, nullptr,
                    max_rows, seq_len, base, d_kv_len, position_ids, position_stride, section0, section1, section2, stream);
}

extern "C" size_t efm_kv_fp4_bytes(const efm_attention_ctx* ctx, uint32_t max_rows) {
    if (validate_attention_ctx(ctx, "kv_fp4_bytes") != EFM_OK) return 0;
    return KvFp4Layout(KvFp4Layout::rows(max_rows), (int)ctx->num_kv_heads, (int)ctx->head_dim).bytes();
}

extern "C" int efm_kv_fp4_read(const efm_attention_ctx* ctx, const void* cache, uint32_t max_rows, uint32_t first, uint32_t rows,
                               void* k_out, void* v_out, hipStream_t stream) {
    const int rc = validate_attention_ctx(ctx, "kv_fp4_read");
    if (rc) return rc;
    if (!cache || (!k_out && !v_out)) return set_error(EFM_ERR_INVALID_ARGUMENT, "kv_fp4_read: null pointer");
    if (!qk_aligned(cache) || !qk_aligned(k_out) || !qk_aligned(v_out))
        return set_error(EFM_ERR_INVALID_ARGUMENT, "kv_fp4_read: pointers must be 16-byte aligned");
    if (max_rows > (1u << 24)) return set_error(EFM_ERR_UNSUPPORTED, "kv_fp4_read: max_rows %u too large", max_rows);
    if (first > max_rows || rows > max_rows - first)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "kv_fp4_read: rows %u + %u do not fit max_rows %u", first, rows, max_rows);
    if (rows == 0) return EFM_OK;
    const KvFp4Layout lay(KvFp4Layout::rows(max_rows), (int)ctx->num_kv_heads, (int)ctx->head_dim);
    const int64_t octets = (int64_t)rows * ctx->num_kv_heads * (ctx->head_dim / 8);
    if (octets > (1ll << 38)) return set_error(EFM_ERR_UNSUPPORTED, "kv_fp4_read: too many rows");
    const dim3 grid((unsigned)((octets + 255) / 256));
    if (ctx->head_dim == 128)
        hipLaunchKernelGGL(kv_fp4_read_kernel<128>, grid, dim3(256), 0, stream, static_cast<const uint8_t*>(cache), lay, first,
                           octets, static_cast<uint4*>(k_out), static_cast<uint4*>(v_out));
    else
        hipLaunchKernelGGL(kv_fp4_read_kernel<64>, grid, dim3(256), 0, stream, static_cast<const uint8_t*>(cache), lay, first,
                           octets, static_cast<uint4*>(k_out), static_cast<uint4*>(v_out));
    return check_launch("kv_fp4_read");
}
