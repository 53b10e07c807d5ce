// Attention over an FP4 cache (fp4.hpp) on gfx950: one query row (decode) or several (a turn's or
// a prompt's rows), GQA, causal or not.
//
// Query rows of the heads that share a KV head are flattened (row r: token r / G, head r % G) and
// taken 16 at a time: the matrix cores multiply 16 keys by 16 rows by 32 channels, S^T = K Q^T
// with the keys as the first operand. A lane then holds, for one row, 8 consecutive keys of a
// 32-key tile (the keys of the two 16-key operands are interleaved so), which is what the second
// product O^T = V^T P^T takes from it as its second operand: P never moves between lanes. The
// codes become bf16 in registers, exactly.
// A workgroup's waves take every NW-th tile of its split of the keys, each with the running
// maximum and sum of its own softmax; their outputs meet in LDS. Where the keys are split over
// workgroups too, those write unnormalised outputs with (maximum, sum), and a second kernel joins
// them.
#include "fp4.hpp"

#include <algorithm>
#include <cmath>

namespace efm {

int validate_attention_ctx(const efm_attention_ctx* c, const char* who);
int prefill_cus();

struct KvFp4Args {
    const bf16_t* q;
    const uint8_t* cache;
    bf16_t* o;
    float* o_part;             // [splits][Hkv][rows][HD]
    float* ml_part;            // [splits][Hkv][rows][2]
    const uint32_t* d_kv_len;
    size_t T;
    int64_t q_sn, q_sh;
    uint32_t kv_len, max_kv_len, S;
    int Hq, Hkv, G, causal;
    int rows;                  // S * G
    int split_tiles, splits;   // 32-key tiles of a split
    float scale;               // log2(e) / sqrt(HD)
};

__device__ __forceinline__ float max_over_groups(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}

template <int HD>
struct KvFp4Tile {
    static constexpr int W = HD / 32;      // words a lane takes of a key
    uint32_t k[2][W], ks[2];
    uint32_t v[8];
    uint2 vs;
};

template <int HD, int NW>
__global__ __launch_bounds__(NW * kWave) void kv_fp4_attn_kernel(KvFp4Args a) {
    constexpr int W = HD / 32, MT = HD / 16;   // channel tiles of O^T
    constexpr int LDO = HD + 4;
    __shared__ float so[NW][16][LDO];
    __shared__ float sml[NW][16][2];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, l = lane % 16, g = lane / 16;
    const int r0 = blockIdx.x * 16, kvh = blockIdx.y, split = blockIdx.z;
    uint32_t L = a.kv_len;
    if (a.d_kv_len != nullptr) L = min(a.d_kv_len[0], a.max_kv_len);
    const int row = r0 + l, tok = row / a.G, head = kvh * a.G + row % a.G;
    const bool row_on = row < a.rows;
    // keys that the lane's row sees, and that any row of the block does
    const int sees = !row_on ? 0 : a.causal ? (int)L - (int)a.S + tok + 1 : (int)L;
    const int last = min(r0 + 15, a.rows - 1) / a.G;
    const int block_sees = a.causal ? (int)L - (int)a.S + last + 1 : (int)L;
    const int first_sees = a.causal ? (int)L - (int)a.S + r0 / a.G + 1 : (int)L;   // the fewest
    const int tile_end = min((block_sees + 31) / 32, (split + 1) * a.split_tiles);

    const KvFp4Layout lay(a.T, a.Hkv, HD);
    const uint8_t* const kc = a.cache + lay.k(kvh);
    const uint8_t* const vc = a.cache + lay.v(kvh);
    const uint8_t* const ksc = a.cache + lay.ks(kvh);
    const uint8_t* const vsc = a.cache + lay.vs(kvh);
    const int oct = HD == 128 ? l : l % 8;                     // the lane's octet of channels
    const int oshift = HD == 128 ? 0 : 16 * (l / 8);           // head_dim 64: two lanes share an octet

    bf16x8_t qf[W];
#pragma unroll
    for (int w = 0; w < W; ++w) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (row_on) u = *reinterpret_cast<const uint4*>(a.q + (int64_t)tok * a.q_sn + (int64_t)head * a.q_sh + 32 * w + 8 * g);
        qf[w] = __builtin_bit_cast(bf16x8_t, u);
    }
    f32x4_t o[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, sum = 0.f;

    for (int t = split * a.split_tiles + wave; t < tile_end; t += NW) {
        KvFp4Tile<HD> c;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const size_t key = (size_t)t * 32 + 8 * (l / 4) + 4 * i + l % 4;
            const uint8_t* p = kc + key * (HD / 2) + g * (HD / 8);
            if constexpr (HD == 128) {
                const uint4 u = load_stream16(p);
                c.k[i][0] = u.x, c.k[i][1] = u.y, c.k[i][2] = u.z, c.k[i][3] = u.w;
                c.ks[i] = *reinterpret_cast<const uint32_t*>(ksc + key * 4);
            } else {
                const uint2 u = *reinterpret_cast<const uint2*>(p);
                c.k[i][0] = u.x, c.k[i][1] = u.y;
                c.ks[i] = *reinterpret_cast<const uint16_t*>(ksc + key * 2);
            }
        }
        const size_t blk = (size_t)t * 4 + g;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 u = load_stream16(vc + (blk * (HD / 8) + oct) * 32 + 16 * i);
            c.v[4 * i] = u.x, c.v[4 * i + 1] = u.y, c.v[4 * i + 2] = u.z, c.v[4 * i + 3] = u.w;
        }
        c.vs = *reinterpret_cast<const uint2*>(vsc + (blk * W + oct / 4) * 8);

        f32x4_t s[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w)
                s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    fp4_unpack8(c.k[i][w], fp4_scale((c.ks[i] >> (8 * w)) & 255)), qf[w], s[i], 0, 0, 0);
        }
        // the lane's keys: key0 + 4 i + r
        const int key0 = t * 32 + 8 * g;
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = s[i / 4][i % 4] * a.scale;
        if (t * 32 + 32 > first_sees || r0 + 16 > a.rows) {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = key0 + i < sees ? p[i] : -INFINITY;
        }
        float top = p[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, p[i]);
        top = fmaxf(m, max_over_groups(top));
        if (__any(top > m)) {
            const float alpha = top == -INFINITY ? 1.f : exp2f(m - top);
            sum *= alpha;
#pragma unroll
            for (int i = 0; i < MT; ++i) o[i] *= alpha;
            m = top;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float part = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = exp2f(p[i] - ref);
            part += p[i];
        }
        sum += part;
        const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, pack8(p));

        // values of keys past the end are zero, and so are NaN groups, whose rows get their NaN below
        uint32_t vb[8];
        bool nan = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            vb[i] = ((i < 4 ? c.vs.x : c.vs.y) >> (8 * (i % 4))) & 255;
            const bool off = key0 + i >= (int)L;
            if (off || vb[i] == kFp4ScaleNan) {
                nan |= !off;
                c.v[i] = 0;
                if (off) vb[i] = 0;
            }
        }
        const bool any_nan = __any(nan);
#pragma unroll
        for (int b = 0; b < MT / 2; ++b) {
            uint32_t e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float sc = fp4_scale(vb[i] == kFp4ScaleNan ? 0 : vb[i]);
                const uint32_t word = c.v[i] >> oshift;
                e[i] = b == 0 ? fp4_pair<0>(word, sc) : b == 1 ? fp4_pair<1>(word, sc)
                     : b == 2 ? fp4_pair<2>(word, sc) : fp4_pair<3>(word, sc);
            }
            uint4 lo, hi;
            lo.x = __builtin_amdgcn_perm(e[1], e[0], 0x05040100), hi.x = __builtin_amdgcn_perm(e[1], e[0], 0x07060302);
            lo.y = __builtin_amdgcn_perm(e[3], e[2], 0x05040100), hi.y = __builtin_amdgcn_perm(e[3], e[2], 0x07060302);
            lo.z = __builtin_amdgcn_perm(e[5], e[4], 0x05040100), hi.z = __builtin_amdgcn_perm(e[5], e[4], 0x07060302);
            lo.w = __builtin_amdgcn_perm(e[7], e[6], 0x05040100), hi.w = __builtin_amdgcn_perm(e[7], e[6], 0x07060302);
            o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, lo), pf, o[2 * b], 0, 0, 0);
            o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, hi), pf, o[2 * b + 1], 0, 0, 0);
        }
        if (any_nan) {
            // the output of a row that sees a key with a NaN group is NaN in the group's channels
            for (int k = 0; k < 32; ++k) {
                if (t * 32 + k >= (int)L) break;
                const bool seen = t * 32 + k < sees;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int ch = HD == 128 ? 8 * (4 * g + r) : 8 * ((4 * g + r) % 8);
                    const bool bad = vsc[((size_t)(t * 4 + k / 8) * W + ch / 32) * 8 + k % 8] == kFp4ScaleNan;
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        if (bad && seen) o[i][r] = __builtin_nanf("");
                }
            }
        }
    }
    sum += __shfl_xor(sum, 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);
    if (g == 0) sml[wave][l][0] = m, sml[wave][l][1] = sum;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int op = 4 * g + r, d = HD == 128 ? 8 * op : 8 * (op % 8) + 4 * (op / 8);
#pragma unroll
        for (int i = 0; i < MT; i += 4)
            *reinterpret_cast<float4*>(&so[wave][l][d + i]) = make_float4(o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * (HD / 4); e += NW * kWave) {
        const int r = e / (HD / 4), d = e % (HD / 4) * 4, gr = r0 + r;
        if (gr >= a.rows) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sml[w][r][0]);
        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = M == -INFINITY ? 1.f : exp2f(sml[w][r][0] - M);
            const float4 x = *reinterpret_cast<const float4*>(&so[w][r][d]);
            t.x += f * x.x, t.y += f * x.y, t.z += f * x.z, t.w += f * x.w;
            den += f * sml[w][r][1];
        }
        if (a.splits == 1) {
            const float inv = den == 0.f ? 0.f : 1.f / den;
            const int tk = gr / a.G, h = kvh * a.G + gr % a.G;
            *reinterpret_cast<uint2*>(a.o + ((int64_t)tk * a.Hq + h) * HD + d) =
                make_uint2(pack_bf16x2(t.x * inv, t.y * inv), pack_bf16x2(t.z * inv, t.w * inv));
        } else {
            const int64_t at = ((int64_t)split * a.Hkv + kvh) * a.rows + gr;
            *reinterpret_cast<float4*>(a.o_part + at * HD + d) = t;
            if (d == 0) *reinterpret_cast<float2*>(a.ml_part + at * 2) = make_float2(M, den);
        }
    }
}

// HD / 4 lanes a row: the outputs of its splits, weighted by exp2(m_s - max m).
template <int HD>
__global__ __launch_bounds__(256) void kv_fp4_merge_kernel(KvFp4Args a) {
    const int per = 256 / (HD / 4);
    const int64_t r = (int64_t)blockIdx.x * per + threadIdx.x / (HD / 4);
    const int d = threadIdx.x % (HD / 4) * 4;
    const int64_t all = (int64_t)a.Hkv * a.rows;
    if (r >= all) return;
    uint32_t L = a.kv_len;
    if (a.d_kv_len != nullptr) L = min(a.d_kv_len[0], a.max_kv_len);
    const int used = min(a.splits, ((int)L + a.split_tiles * 32 - 1) / (a.split_tiles * 32));
    float M = -INFINITY;
    for (int s = 0; s < used; ++s) M = fmaxf(M, a.ml_part[(s * all + r) * 2]);
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    float den = 0.f;
    for (int s = 0; s < used; ++s) {
        const float2 ml = *reinterpret_cast<const float2*>(a.ml_part + (s * all + r) * 2);
        const float f = M == -INFINITY ? 1.f : exp2f(ml.x - M);
        const float4 x = *reinterpret_cast<const float4*>(a.o_part + (s * all + r) * HD + d);
        t.x += f * x.x, t.y += f * x.y, t.z += f * x.z, t.w += f * x.w;
        den += f * ml.y;
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    const int kvh = (int)(r / a.rows), gr = (int)(r % a.rows), tk = gr / a.G, h = kvh * a.G + gr % a.G;
    *reinterpret_cast<uint2*>(a.o + ((int64_t)tk * a.Hq + h) * HD + d) =
        make_uint2(pack_bf16x2(t.x * inv, t.y * inv), pack_bf16x2(t.z * inv, t.w * inv));
}

struct KvFp4Plan {
    int split_tiles, splits;
    size_t o_bytes, ml_bytes;
};

static KvFp4Plan kv_fp4_plan(const efm_attention_ctx* c, uint32_t S, uint32_t kv_len) {
    const int G = (int)(c->num_qo_heads / c->num_kv_heads);
    const int64_t rows = (int64_t)S * G, blocks = (rows + 15) / 16 * c->num_kv_heads;
    const int tiles = (int)((kv_len + 31) / 32);
    // two workgroups of 4 waves a CU, and at least a tile for each wave of a split
    const int64_t want = std::max<int64_t>(1, 512 / std::max<int64_t>(1, blocks));
    KvFp4Plan p;
    p.split_tiles = std::max(4, (int)((tiles + want - 1) / want));
    p.splits = std::max(1, (tiles + p.split_tiles - 1) / p.split_tiles);
    p.o_bytes = p.splits == 1 ? 0 : (size_t)p.splits * c->num_kv_heads * rows * c->head_dim * sizeof(float);
    p.ml_bytes = p.splits == 1 ? 0 : (size_t)p.splits * c->num_kv_heads * rows * 2 * sizeof(float);
    return p;
}

static int kv_fp4_attention(const char* who, const efm_attention_ctx* ctx, const void* q, const void* cache, uint32_t max_rows,
                            void* o, uint32_t S, uint32_t kv_len, const uint32_t* d_kv_len, uint32_t max_kv_len, int causal,
                            void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const int rc = validate_attention_ctx(ctx, who);
    if (rc) return rc;
    if (ctx->pos_encoding != EFM_POS_NONE)
        return set_error(EFM_ERR_UNSUPPORTED, "%s: pos_encoding must be EFM_POS_NONE (the cache holds rotated keys)", who);
    if (!q || !cache || !o) return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: null tensor pointer", who);
    const uint32_t bound = d_kv_len != nullptr ? max_kv_len : kv_len;
    if (d_kv_len != nullptr && max_kv_len == 0)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: max_kv_len must be > 0 with d_kv_len", who);
    if (max_rows > (1u << 24)) return set_error(EFM_ERR_UNSUPPORTED, "%s: max_rows %u too large", who, max_rows);
    if (bound > max_rows) return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: %u rows of a cache of %u", who, bound, max_rows);
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(o)) & 15u) != 0)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: pointers must be 16-byte aligned", who);
    if (S == 0) return EFM_OK;
    const int hd = (int)ctx->head_dim;
    const KvFp4Plan p = kv_fp4_plan(ctx, S, bound);
    if (p.splits > 1 && (workspace == nullptr || workspace_bytes < p.o_bytes + p.ml_bytes))
        return set_error(EFM_ERR_WORKSPACE, "%s: workspace of %zu bytes required", who, p.o_bytes + p.ml_bytes);
    if (p.splits > 1 && (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", who);
    KvFp4Args a;
    a.q = static_cast<const bf16_t*>(q);
    a.cache = static_cast<const uint8_t*>(cache);
    a.o = static_cast<bf16_t*>(o);
    a.o_part = static_cast<float*>(workspace);
    a.ml_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.o_bytes);
    a.d_kv_len = d_kv_len;
    a.T = KvFp4Layout::rows(max_rows);
    a.q_sn = ctx->q_stride_n ? ctx->q_stride_n : (int64_t)ctx->num_qo_heads * hd;
    a.q_sh = ctx->q_stride_h ? ctx->q_stride_h : hd;
    a.kv_len = kv_len;
    a.max_kv_len = max_kv_len;
    a.S = S;
    a.Hq = (int)ctx->num_qo_heads;
    a.Hkv = (int)ctx->num_kv_heads;
    a.G = a.Hq / a.Hkv;
    a.causal = causal != 0;
    a.rows = (int)S * a.G;
    a.split_tiles = p.split_tiles;
    a.splits = p.splits;
    a.scale = 1.4426950408889634f / sqrtf((float)hd);
    const dim3 grid((a.rows + 15) / 16, a.Hkv, p.splits);
    const unsigned merge = (unsigned)(((int64_t)a.Hkv * a.rows + 256 / (hd / 4) - 1) / (256 / (hd / 4)));
    if (hd == 128) {
        hipLaunchKernelGGL((kv_fp4_attn_kernel<128, 4>), grid, dim3(256), 0, stream, a);
        if (p.splits > 1) hipLaunchKernelGGL(kv_fp4_merge_kernel<128>, dim3(merge), dim3(256), 0, stream, a);
    } else {
        hipLaunchKernelGGL((kv_fp4_attn_kernel<64, 4>), grid, dim3(256), 0, stream, a);
        if (p.splits > 1) hipLaunchKernelGGL(kv_fp4_merge_kernel<64>, dim3(merge), dim3(256), 0, stream, a);
    }
    return check_launch(who);
}

}  // namespace efm

using namespace efm;

extern "C" size_t efm_attention_decode_kv_fp4_workspace_bytes(const efm_attention_ctx* ctx, uint32_t max_kv_len) {
    if (validate_attention_ctx(ctx, "attention_decode_kv_fp4_workspace_bytes") != EFM_OK) return 0;
    const KvFp4Plan p = kv_fp4_plan(ctx, 1, max_kv_len);
    return p.o_bytes + p.ml_bytes;
}

extern "C" int efm_attention_decode_kv_fp4(const efm_attention_ctx* ctx, const void* q, const void* cache, uint32_t max_rows,
                                           void* o, uint32_t kv_len, const uint32_t* d_kv_len, uint32_t max_kv_len,
                                           void* workspace, size_t workspace_bytes, hipStream_t stream) {
    return kv_fp4_attention("attention_decode_kv_fp4", ctx, q, cache, max_rows, o, 1, kv_len, d_kv_len, max_kv_len, 0,
                            workspace, workspace_bytes, stream);
}

extern "C" size_t efm_attention_prefill_kv_fp4_workspace_bytes(const efm_attention_ctx* ctx, uint32_t qo_len,
                                                               uint32_t kv_len) {
    if (validate_attention_ctx(ctx, "attention_prefill_kv_fp4_workspace_bytes") != EFM_OK) return 0;
    const KvFp4Plan p = kv_fp4_plan(ctx, qo_len, kv_len);
    return p.o_bytes + p.ml_bytes;
}

extern "C" int efm_attention_prefill_kv_fp4(const efm_attention_ctx* ctx, const void* q, const void* cache, uint32_t max_rows,
                                            void* o, uint32_t qo_len, uint32_t kv_len, int32_t causal, void* workspace,
                                            size_t workspace_bytes, hipStream_t stream) {
    if (kv_len < qo_len)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "attention_prefill_kv_fp4: kv_len %u < qo_len %u", kv_len, qo_len);
    if (qo_len > (1u << 20)) return set_error(EFM_ERR_UNSUPPORTED, "attention_prefill_kv_fp4: sequence too long");
    return kv_fp4_attention("attention_prefill_kv_fp4", ctx, q, cache, max_rows, o, qo_len, kv_len, nullptr, 0, causal,
                            workspace, workspace_bytes, stream);
}
