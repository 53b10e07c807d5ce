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
//
// Bound by memory once there are many tokens: 4096 tokens of 28/4 heads of 128 into a bf16 cache read
// and write 76 MB in 14.4 us (5.2 TB/s, a copy's rate), into an FP4 cache 70 MB in 16 us. A token by itself
// takes 3.1 us (bf16) and 3.9 us (FP4), of which an empty launch is 2: the rest is one chain of a load,
// the angle's sine and cosine in 64 bits, the norm's sum, and the store. Reading 4096 such rows of an FP4
// cache back (8.4 MB written) takes 5 us.
#include "fp4.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace efm {

int validate_attention_ctx(const efm_attention_ctx* c, const char* who);
int prefill_cus();

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
    int q_off, k_off;   // as in the other operators: 2^31 and more are below zero
    float eps;
    double turns[kMaxHalfDim];   // theta^(-2 d / hd) / rope_scale / (2 pi)
};

// A value of 4 or 8 bytes from another lane of the row.
template <int CTRL, typename T>
__device__ __forceinline__ T dpp(T v) {
    auto move = [](uint32_t w) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w, CTRL, 0xf, 0xf, false); };
    if constexpr (sizeof(T) == 4) {
        return __builtin_bit_cast(T, move(__builtin_bit_cast(uint32_t, v)));
    } else {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(T, (uint64_t)move((uint32_t)(u >> 32)) << 32 | move((uint32_t)u));
    }
}

// Sum over the LANES lanes of a row, alike in all of them.
template <int LANES, typename T>
__device__ __forceinline__ T row_sum(T v) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    return LANES == 16 ? v + dpp<0x140>(v) : v;
}

// The largest of four lanes, which hold a group of 32 channels.
template <typename T>
__device__ __forceinline__ T group_max(T v) {
    v = max(v, dpp<0xB1>(v));
    return max(v, dpp<0x4E>(v));
}

// The value of the lane that holds the other half of this lane's pairs, LANES / 2 away.
template <int LANES, typename T>
__device__ __forceinline__ T row_other(T v) {
    return LANES == 16 ? dpp<0x128>(v) : dpp<0x141>(dpp<0x1B>(v));
}

__device__ __forceinline__ float inv_sqrt(float v) { return rsqrtf(v); }
__device__ __forceinline__ double inv_sqrt(double v) { return 1.0 / sqrt(v); }

template <typename T, int LANES>
__device__ __forceinline__ void norm8(T* x, uint4 weight, T eps) {
    T sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += x[e] * x[e];
    const T r = inv_sqrt(row_sum<LANES>(sum) / (T)(8 * LANES) + eps);
    float w[8];
    unpack8(weight, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * r * (T)w[e];
}

// cs: (cos, sin), the sine negated for lanes of the first half.
template <typename T, int LANES, typename CS>
__device__ __forceinline__ void turn8(T* x, CS cs) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        // 64-bit pairs one after another: all eight at once would cost 20 registers, and with them waves
        if constexpr (sizeof(T) == 8) __builtin_amdgcn_sched_barrier(0);
        const T o = row_other<LANES>(x[e]);
        const auto v = cs(e);
        x[e] = x[e] * (T)v.x + o * (T)v.y;
    }
}

// HD / 8 lanes a row of a head, 64 / (HD / 8) rows a wave. TOKENS: a workgroup takes that many
// consecutive tokens, and a wave their rows of a head, so that all its lanes do the same (a row of
// Q, K or V) and the words of a V block's rows leave together. Otherwise a workgroup takes one token,
// and a wave several heads of it. Either way a lane keeps its token and channels: sines and cosines
// stay in its registers for the queries, and the next two rows are on their way while it works on one.
template <int HD, bool FP4, bool TOKENS>
__global__ __launch_bounds__(TOKENS ? 512 : 1024) void qk_norm_rope_write_kernel(QkWriteArgs a) {
    constexpr int LANES = HD / 8, HALF = HD / 2, ROWS = kWave / LANES, T = TOKENS ? ROWS : 1, HL = LANES / 2;
    // (cos, sin) of [query, key], of both where their offsets agree; channel d at (d % 8) * HL + d / 8, so
    // that the lanes of a row read beside each other
    __shared__ double2 cs[2][T][HALF + 8];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
    const int sub = lane / LANES, j = lane % LANES;
    const uint32_t t0 = blockIdx.x * T, t = TOKENS ? t0 + sub : t0;
    const bool on = t < a.S, lo = j < HL;
    const int first = a.q_out != nullptr ? 0 : a.Hq, heads = a.Hq + 2 * a.Hkv;
    const bf16_t* const src = a.qkv + (int64_t)(on ? t : t0) * a.qkv_sn + 8 * j;
    const int step = TOKENS ? waves : waves * ROWS;
    int h = first + (TOKENS ? wave : wave * ROWS + sub);
    auto request = [&](int head) { return *reinterpret_cast<const uint4*>(src + (int64_t)min(head, heads - 1) * HD); };
    uint4 next[2] = {request(h), request(h + step)};
    uint4 qw = make_uint4(0, 0, 0, 0), kw = qw;
    if (a.q_w != nullptr) qw = reinterpret_cast<const uint4*>(a.q_w)[j];
    if (!FP4 && a.k_w != nullptr) kw = reinterpret_cast<const uint4*>(a.k_w)[j];
    uint32_t base = a.base;
    if (a.d_kv_len != nullptr) {
        const uint32_t L = a.d_kv_len[0];
        if (L < a.S || L > a.max_rows) return;
        base = L - a.S;
    }
    const uint32_t row = base + t;
    const int same = a.pos != nullptr || a.q_off == a.k_off;
    if (a.rotate) {
        for (int i = threadIdx.x; i < (same ? 1 : 2) * T * HALF; i += blockDim.x) {
            const int at = i % HALF, d = at % HL * 8 + at / HL, tt = i / HALF % T, is_k = i / HALF / T;
            double p;
            if (a.pos != nullptr)
                p = (double)a.pos[(d < a.cum0 ? 0 : d < a.cum1 ? 1 : 2) * a.pos_stride + min(t0 + tt, a.S - 1)];
            else p = (double)(base + t0 + tt) + (double)(is_k ? a.k_off : a.q_off);
            const double turn = p * a.turns[d];
            double s, c;
            sincospi(2.0 * (turn - rint(turn)), &s, &c);
            cs[is_k][tt][at] = make_double2(c, s);
        }
        __syncthreads();
    }
    float2 csq[8];
    if (a.rotate) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const double2 v = cs[0][TOKENS ? sub : 0][e * HL + j % HL];
            csq[e] = make_float2((float)v.x, lo ? -(float)v.y : (float)v.y);
        }
    }
    const KvFp4Layout lay(KvFp4Layout::rows(a.max_rows), a.Hkv, HD);
    for (; __any(h < heads); h += step) {
        const uint4 raw = next[0];
        next[0] = next[1];
        next[1] = request(h + 2 * step);
        const bool is_q = h < a.Hq, is_k = !is_q && h < a.Hq + a.Hkv, is_v = !is_q && !is_k && h < heads;
        if (__any(is_q)) {
            float x[8];
            unpack8(raw, x);
            if (a.q_w != nullptr) norm8<float, LANES>(x, qw, a.eps);
            if (a.rotate) turn8<float, LANES>(x, [&](int e) { return csq[e]; });
            if (is_q && on)
                *reinterpret_cast<uint4*>(a.q_out + (int64_t)t * a.q_sn + (int64_t)h * a.q_sh + 8 * j) = pack8(x);
        }
        if (__any(is_k)) {
            using Y = std::conditional_t<FP4, double, float>;
            float x[8];
            unpack8(raw, x);
            Y y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = (Y)x[e];
            if (a.k_w != nullptr) norm8<Y, LANES>(y, FP4 ? reinterpret_cast<const uint4*>(a.k_w)[j] : kw, (Y)a.eps);
            if (a.rotate) {
                int at = j % HL;
                asm volatile("" : "+v"(at));   // read here: held over the loop, they would cost 32 registers
                turn8<Y, LANES>(y, [&](int e) {
                    const double2 v = cs[same ? 0 : 1][TOKENS ? sub : 0][e * HL + at];
                    return make_double2(v.x, lo ? -v.y : v.y);
                });
            }
            const int kh = h - a.Hq;
            if constexpr (FP4) {
                uint64_t top = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, (uint64_t)(__double_as_longlong(y[e]) & 0x7fffffffffffffffll));
                const uint32_t byte = fp4_scale_byte(group_max(top)), word = fp4_encode8(y, byte);
                if (is_k && on) {
                    *reinterpret_cast<uint32_t*>(a.cache + lay.k(kh) + lay.k_word(row, j)) = word;
                    if (j % 4 == 0) a.cache[lay.ks(kh) + lay.k_scale(row, j)] = (uint8_t)byte;
                }
            } else if (is_k && on) {
                *reinterpret_cast<uint4*>(a.k_cache + (int64_t)row * a.k_sn + (int64_t)kh * a.k_sh + 8 * j) = pack8(y);
            }
        }
        if (__any(is_v)) {
            const int vh = h - a.Hq - a.Hkv;
            if constexpr (FP4) {
                float x[8];
                unpack8(raw, x);
                uint32_t top = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
                const uint32_t byte = fp4_scale_byte(group_max(top)), word = fp4_encode8(x, byte);
                if (is_v && on) {
                    *reinterpret_cast<uint32_t*>(a.cache + lay.v(vh) + lay.v_word(row, j)) = word;
                    if (j % 4 == 0) a.cache[lay.vs(vh) + lay.v_scale(row, j)] = (uint8_t)byte;
                }
            } else if (is_v && on) {
                *reinterpret_cast<uint4*>(a.v_cache + (int64_t)row * a.v_sn + (int64_t)vh * a.v_sh + 8 * j) = raw;
            }
        }
    }
}

// One lane for 8 channels of a row of head head0 + blockIdx.y: keys (blockIdx.z == 0) row after row, values 8 rows
// of an octet beside each other as they lie.
template <int HD>
__global__ __launch_bounds__(256) void kv_fp4_read_kernel(const uint8_t* cache, KvFp4Layout lay, int head0, uint32_t first,
                                                          uint32_t rows, uint4* k_out, uint4* v_out) {
    constexpr uint32_t J = HD / 8;
    const bool values = blockIdx.z == 1;
    uint4* const out = values ? v_out : k_out;
    if (out == nullptr) return;
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;   // rows <= 2^24
    const int h = head0 + blockIdx.y, j = (int)(values ? i / 8 % J : i % J);
    const uint32_t row = values ? (first / 8 + i / 8 / J) * 8 + i % 8 : first + i / J;
    if (row < first || row >= first + rows) return;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(cache + (values ? lay.v(h) + lay.v_word(row, j) : lay.k(h) + lay.k_word(row, j)));
    const uint32_t byte = cache[values ? lay.vs(h) + lay.v_scale(row, j) : lay.ks(h) + lay.k_scale(row, j)];
    out[((int64_t)(row - first) * lay.Hkv + h) * J + j] = __builtin_bit_cast(uint4, fp4_unpack8(w, fp4_scale(byte)));
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
    a.q_off = (int)ctx->q_rope_pos_offset;
    a.k_off = (int)ctx->k_rope_pos_offset;
    a.eps = eps;
    if (rotate) {
        const double l = log((double)ctx->rope_theta), scale = ctx->rope_scale;
        for (int d = 0; d < hd / 2; ++d) a.turns[d] = exp(-2.0 * d / (double)hd * l) / scale / 6.283185307179586476925;
    }
    // A token a workgroup spreads few tokens over the chip; from ten of its waves a CU on (bf16: 24), tokens
    // together do less apiece. Measured (us, one / together; FP4 with the rows read back, 2 to 2.5 of it):
    // 28/4 heads of 128, FP4: 64 tokens 6.3 / 7.4, 256 6.8 / 7.7, 284 8.2 / 7.7, 512 9.0 / 8.1, 1024 14.4 /
    // 9.9; bf16: 64 3.4 / 4.6, 512 4.6 / 5.2, 682 6.2 / 5.7, 1024 9.2 / 6.6, 4096 25.8 / 14.5. 12/2 heads, FP4:
    // 500 tokens 6.8 / 6.8, 1024 7.7 / 7.3; bf16: 1300 5.1 / 5.4, 1536 5.5 / 5.7, 2000 7.2 / 6.3. 14/2 heads of
    // 64, FP4: 700 tokens 6.8 / 6.8, 2000 10.2 / 7.4; bf16: 1500 4.9 / 4.5, 2000 5.4 / 4.7, 2500 7.0 / 5.8.
    // Eight waves for tokens together: 4096 of 28/4 heads into a bf16 cache 14.5, with six 15.5, twelve 16.1;
    // 1344 of 16/2 heads 6.0, with five 6.4, ten 6.2.
    auto launch = [&](auto hdc, auto fc) {
        constexpr int HD = decltype(hdc)::value, ROWS = kWave * 8 / HD;
        constexpr bool F = decltype(fc)::value;
        const int64_t heads = (q_out ? Hq : 0) + 2 * Hkv, waves = std::min<int64_t>(16, (heads + ROWS - 1) / ROWS);
        if (seq_len * waves >= (F ? 10 : 24) * (int64_t)prefill_cus())
            hipLaunchKernelGGL((qk_norm_rope_write_kernel<HD, F, true>), dim3((seq_len + ROWS - 1) / ROWS),
                               dim3(kWave * (unsigned)std::min<int64_t>(8, heads)), 0, stream, a);
        else
            hipLaunchKernelGGL((qk_norm_rope_write_kernel<HD, F, false>), dim3(seq_len), dim3(kWave * (unsigned)waves), 0,
                               stream, a);
    };
    using std::integral_constant;
    if (hd == 128 && fp4) launch(integral_constant<int, 128>{}, std::true_type{});
    else if (hd == 128) launch(integral_constant<int, 128>{}, std::false_type{});
    else if (fp4) launch(integral_constant<int, 64>{}, std::true_type{});
    else launch(integral_constant<int, 64>{}, std::false_type{});
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
    if (validate_attention_ctx(ctx, "kv_fp4_bytes") != EFM_OK || ctx->num_qo_heads > (1u << 16) || max_rows > (1u << 24)) return 0;
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
    if (ctx->num_qo_heads > (1u << 16))
        return set_error(EFM_ERR_UNSUPPORTED, "kv_fp4_read: %u query heads", ctx->num_qo_heads);
    if (first > max_rows || rows > max_rows - first)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "kv_fp4_read: rows %u + %u do not fit max_rows %u", first, rows, max_rows);
    if (rows == 0) return EFM_OK;
    const KvFp4Layout lay(KvFp4Layout::rows(max_rows), (int)ctx->num_kv_heads, (int)ctx->head_dim);
    // a head's lanes for values' whole blocks of 8 rows; keys take no more
    const uint32_t lanes = (rows + 14) / 8 * 8 * (ctx->head_dim / 8);
    const uint32_t grid_heads = 65535;   // a grid holds one head less than a cache may have
    auto launch = [&](auto hdc) {
        for (uint32_t h = 0; h < ctx->num_kv_heads; h += grid_heads)
            hipLaunchKernelGGL(kv_fp4_read_kernel<decltype(hdc)::value>,
                               dim3((lanes + 255) / 256, std::min(ctx->num_kv_heads - h, grid_heads), 2), dim3(256), 0, stream,
                               static_cast<const uint8_t*>(cache), lay, (int)h, first, rows, static_cast<uint4*>(k_out),
                               static_cast<uint4*>(v_out));
    };
    if (ctx->head_dim == 128) launch(std::integral_constant<int, 128>{});
    else launch(std::integral_constant<int, 64>{});
    return check_launch("kv_fp4_read");
}
