// Attention over an FP4 cache (fp4.hpp) on gfx950: one query row (decode) or several (a turn's or
// a prompt's rows), GQA, causal or not.
//
// Query rows of the heads that share a KV head are flattened (row r: token r / G, head r % G) and
// taken 16 at a time: the matrix cores multiply 16 keys by 16 rows by 32 channels, S^T = K Q^T
// with the keys as the first operand. A lane then holds, for one row, 8 consecutive keys of a
// 32-key tile (the keys of the two 16-key operands are interleaved so), which is what the second
// product O^T = V^T P^T takes from it as its second operand: P never moves between lanes. The
// codes become bf16 in registers, exactly. P is rounded to bf16 there, the type of the matrix cores'
// products (a relative 2^-9 a weight: outputs move by 0.0013 to 0.0016 of their size before their own
// rounding to bf16, which moves them by 0.0017); maxima, sums and outputs stay in fp32, the sums over P unrounded.
// A workgroup's waves take every NW-th tile of its split of the keys, each with the running
// maximum and sum of its own softmax; their outputs meet in LDS (many rows: a kernel of its own,
// below). Where the keys are split over workgroups too, those write unnormalised outputs with
// (maximum, sum), and a second kernel joins them.
#include "fp4.hpp"

#include <algorithm>
#include <cmath>
#include <utility>

namespace efm {

int validate_attention_ctx(const efm_attention_ctx* c, const char* who);
int prefill_cus();

constexpr int kKvFp4MaxSplits = 256;   // threads of a workgroup that joins them
constexpr float kKvFp4Lazy = 8.f;

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
    int tiles;                 // of all keys there may be
    int cus;
    float scale;               // log2(e) / sqrt(HD)
};

// Values of lanes l, l + 16, l + 32 and l + 48 combined, in all four.
template <typename F>
__device__ __forceinline__ float over_groups(float v, F f) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// What a lane holds of a 32-key tile: of each of its two 16-key operands a key's words and scale
// bytes, and 8 consecutive keys' words of one octet of channels with their scale bytes.
template <int HD>
struct KvFp4Tile {
    static constexpr int W = HD / 32;
    uint32_t k[2][W], ks[2], v[8], vs[2];
};

// The first half of the softmax step of NT tiles of 32 keys for the lane's row: masks s, its products with
// keys key0 .. key0 + 7 of each tile, and returns what their exponents are relative to. m, sum and the
// outputs so far follow a maximum larger by 2^kKvFp4Lazy in weights, which is rare past a row's first
// keys: weights of up to that and their sums are as exact in bf16 and fp32 as those of up to 1.
template <int MT, int NT>
__device__ __forceinline__ float kv_fp4_maximum(f32x4_t (*s)[2], int key0, bool masked, int sees, float scale, float& m, float& sum,
                                                f32x4_t* o) {
    // v_maximum3_f32 takes three operands as they are; a NaN among them leaves m, and makes the row's sum NaN
    auto larger = [](float x, float y) { return __builtin_elementwise_maximum(x, y); };
    float tops[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (masked) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[t][i / 4][i % 4] = key0 + 32 * t + i < sees ? s[t][i / 4][i % 4] : -INFINITY;
        }
        const f32x4_t x = s[t][0], y = s[t][1];
        tops[t] = larger(larger(larger(larger(x[0], x[1]), x[2]), larger(larger(x[3], y[0]), y[1])), larger(y[2], y[3]));
    }
    float top = NT == 1 ? tops[0] : larger(tops[0], tops[NT - 1]);
    top = larger(m, over_groups(top, larger));
    if (__any(top > m + kKvFp4Lazy / scale)) {
        const float alpha = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - top) * scale);
        sum *= alpha;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[i] *= alpha;
        m = top;
    }
    return m == -INFINITY ? 0.f : m * scale;
}

// The whole step; pf: the weights as second operands of the second product.
template <int MT, int NT>
__device__ __forceinline__ void kv_fp4_softmax(f32x4_t (*s)[2], int key0, bool masked, int sees, float scale, float& m, float& sum,
                                               f32x4_t* o, bf16x8_t* pf) {
    const float ref = kv_fp4_maximum<MT, NT>(s, key0, masked, sees, scale, m, sum, o);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        float p[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[t][i / 4][i % 4], scale, -ref));
        sum += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        pf[t] = __builtin_bit_cast(bf16x8_t, pack8(p));
    }
}

// NaN in the channels of key k's NaN groups, for the rows that see it.
template <int HD, int NQ>
__device__ __forceinline__ void kv_fp4_put_nan(const uint8_t* vs, const KvFp4Layout& lay, int k, int g, const int* sees,
                                               f32x4_t (*o)[HD / 16]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int oct = HD == 128 ? 4 * g + r : (4 * g + r) % 8;
        const bool bad = vs[lay.v_scale(k, oct)] == kFp4ScaleNan;
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int i = 0; i < HD / 16; ++i)
                if (bad && k < sees[n]) o[n][i][r] = __builtin_nanf("");
    }
}

// NQ x 16 rows a workgroup; the waves walk the tiles of its split. Bound by memory while rows are
// few: 4.25 bits a value, two tiles of loads (4.3 KB each a wave) under way.
template <int HD, int NW, int NQ>
__global__ __launch_bounds__(NW * kWave, NQ == 1 ? (HD == 128 ? 3 : 4) : NQ == 2 ? 2 : 1) void kv_fp4_attn_kernel(KvFp4Args a) {
    constexpr int W = HD / 32, MT = HD / 16;   // channel tiles of O^T
    constexpr int LDO = HD + 4;
    __shared__ float so[NW][16][LDO];
    __shared__ float sml[NQ][NW][16][2];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, l = lane % 16, g = lane / 16;
    // row blocks from the last, which see the most keys, the KV heads side by side
    const int r0 = ((int)(gridDim.x / a.Hkv) - 1 - (int)(blockIdx.x / a.Hkv)) * (16 * NQ), kvh = blockIdx.x % a.Hkv, split = blockIdx.z;
    const KvFp4Layout lay(a.T, a.Hkv, HD);
    const int oct = HD == 128 ? l : l % 8;            // the lane's octet of channels
    const int oshift = HD == 128 ? 0 : 16 * (l / 8);  // head_dim 64: two lanes share an octet
    const int kr = 8 * (l / 4) + l % 4;               // the lane's key in the first operand; the second's is 4 on
    // 64-bit bases of the head, 32-bit offsets within it (max_rows <= 2^24)
    const uint8_t* const kc = a.cache + lay.k(kvh) + kr * (HD / 2) + g * (HD / 8);
    const uint8_t* const vc = a.cache + lay.v(kvh) + (g * (HD / 8) + oct) * 32;
    const uint8_t* const ksc = a.cache + lay.ks(kvh) + kr * W;
    const uint8_t* const vsc = a.cache + lay.vs(kvh) + (g * W + oct / 4) * 8;
    auto load = [&](KvFp4Tile<HD>& c, int t) {
        const uint32_t ko = (uint32_t)t * (32 * HD / 2), so_ = (uint32_t)t * (32 * W);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint8_t* p = kc + ko + i * (4 * HD / 2);
            if constexpr (HD == 128) {
                const uint4 u = load_stream16(p);
                c.k[i][0] = u.x, c.k[i][1] = u.y, c.k[i][2] = u.z, c.k[i][3] = u.w;
                c.ks[i] = *reinterpret_cast<const uint32_t*>(ksc + so_ + i * 4 * W);
            } else {
                const uint2 u = *reinterpret_cast<const uint2*>(p);
                c.k[i][0] = u.x, c.k[i][1] = u.y;
                c.ks[i] = *reinterpret_cast<const uint16_t*>(ksc + so_ + i * 4 * W);
            }
            const uint4 u = load_stream16(vc + ko + 16 * i);
            c.v[4 * i] = u.x, c.v[4 * i + 1] = u.y, c.v[4 * i + 2] = u.z, c.v[4 * i + 3] = u.w;
        }
        const uint2 u = *reinterpret_cast<const uint2*>(vsc + so_);
        c.vs[0] = u.x, c.vs[1] = u.y;
    };
    // the first tile is requested before the length is known: the cache holds it
    int t = split * a.split_tiles + wave;
    KvFp4Tile<HD> ta, tb;
    if (t < min(a.tiles, (split + 1) * a.split_tiles)) load(ta, t);
    uint32_t L = a.kv_len;
    if (a.d_kv_len != nullptr) L = min(a.d_kv_len[0], a.max_kv_len);
    // keys that the lane's row of query tile n sees
    int sees[NQ];
    bf16x8_t qf[NQ][W];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int row = r0 + 16 * n + l, tok = row / a.G, head = kvh * a.G + row % a.G;
        const bool on = row < a.rows;
        sees[n] = !on ? 0 : a.causal ? (int)L - (int)a.S + tok + 1 : (int)L;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (on) u = *reinterpret_cast<const uint4*>(a.q + (int64_t)tok * a.q_sn + (int64_t)head * a.q_sh + 32 * w + 8 * g);
            qf[n][w] = __builtin_bit_cast(bf16x8_t, u);
        }
    }
    // keys that any row sees, and that every row sees
    const int last = min(r0 + 16 * NQ - 1, a.rows - 1) / a.G;
    const int any_sees = a.causal ? (int)L - (int)a.S + last + 1 : (int)L;
    const int all_see = r0 + 16 * NQ > a.rows ? 0 : a.causal ? (int)L - (int)a.S + r0 / a.G + 1 : (int)L;
    const int tile_end = min((any_sees + 31) / 32, (split + 1) * a.split_tiles);

    f32x4_t o[NQ][MT];
    float m[NQ], sum[NQ];   // largest product and sum of a row's weights, of the lane's keys
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        m[n] = -INFINITY, sum[n] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[n][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    auto process = [&](KvFp4Tile<HD>& c, int t) {
        // S^T: the lane gets keys key0 + 4 i + r of its row. The conversion takes the scale's exponent
        // bits alone, so the word's other scales need not be cleared.
        f32x4_t s[NQ][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) s[n][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const bf16x8_t kf = fp4_unpack8(c.k[i][w], fp4_scale_at(c.ks[i], w));
#pragma unroll
                for (int n = 0; n < NQ; ++n)
                    s[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[n][w], s[n][i], 0, 0, 0);
            }
        }
        const int key0 = t * 32 + 8 * g;
        // Values of keys past the end are made zero, and so are NaN groups; the rows that see those get
        // their NaN below.
        bool nan = false;
        const bool cut = t * 32 + 32 > (int)L;
        const uint32_t ff = ((c.vs[0] & 0x7f7f7f7fu) + 0x01010101u) & c.vs[0], fg = ((c.vs[1] & 0x7f7f7f7fu) + 0x01010101u) & c.vs[1];
        if (cut || __any(((ff | fg) & 0x80808080u) != 0)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t byte = (c.vs[i / 4] >> (8 * (i % 4))) & 255;
                const bool off = key0 + i >= (int)L;
                if (off || byte == kFp4ScaleNan) {
                    nan |= !off;
                    c.v[i] = 0;
                    c.vs[i / 4] &= ~(255u << (8 * (i % 4)));
                }
            }
            nan = __any(nan);
        }
        bf16x8_t pf[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
            kv_fp4_softmax<MT, 1>(&s[n], key0, t * 32 + 32 > all_see, sees[n], a.scale, m[n], sum[n], o[n], &pf[n]);
        // O^T: byte b of the words is two channels of each key; pairs of keys of one channel are put
        // together for the first operand
        [&]<int... B>(std::integer_sequence<int, B...>) {
            ([&] {
                uint32_t e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = fp4_pair<B>(c.v[i] >> oshift, fp4_scale_at(c.vs[i / 4], i % 4));
                uint4 lo, hi;
                lo.x = __builtin_amdgcn_perm(e[1], e[0], 0x05040100), hi.x = __builtin_amdgcn_perm(e[1], e[0], 0x07060302);
                lo.y = __builtin_amdgcn_perm(e[3], e[2], 0x05040100), hi.y = __builtin_amdgcn_perm(e[3], e[2], 0x07060302);
                lo.z = __builtin_amdgcn_perm(e[5], e[4], 0x05040100), hi.z = __builtin_amdgcn_perm(e[5], e[4], 0x07060302);
                lo.w = __builtin_amdgcn_perm(e[7], e[6], 0x05040100), hi.w = __builtin_amdgcn_perm(e[7], e[6], 0x07060302);
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    o[n][2 * B] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, lo), pf[n], o[n][2 * B], 0, 0, 0);
                    o[n][2 * B + 1] =
                        __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, hi), pf[n], o[n][2 * B + 1], 0, 0, 0);
                }
            }(), ...);
        }(std::make_integer_sequence<int, MT / 2>{});
        if (nan)
            for (int k = t * 32; k < min(t * 32 + 32, (int)L); ++k)
                kv_fp4_put_nan<HD, NQ>(a.cache + lay.vs(kvh), lay, k, g, sees, o);
    };
    // two tiles' registers in turn: the next tile is requested before a tile is multiplied
    while (t < tile_end) {
        load(tb, min(t + NW, tile_end - 1));
        process(ta, t);
        t += NW;
        if (t >= tile_end) break;
        load(ta, min(t + NW, tile_end - 1));
        process(tb, t);
        t += NW;
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const float den = over_groups(sum[n], [](float x, float y) { return x + y; });
        if (g == 0) sml[n][wave][l][0] = m[n] * a.scale, sml[n][wave][l][1] = den;
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        if (n > 0) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int op = 4 * g + r, d = HD == 128 ? 8 * op : 8 * (op % 8) + 4 * (op / 8);
#pragma unroll
            for (int i = 0; i < MT; i += 4)
                *reinterpret_cast<float4*>(&so[wave][l][d + i]) = make_float4(o[n][i][r], o[n][i + 1][r], o[n][i + 2][r], o[n][i + 3][r]);
        }
        __syncthreads();
        for (int e = threadIdx.x; e < 16 * (HD / 4); e += NW * kWave) {
            const int r = e / (HD / 4), d = e % (HD / 4) * 4, gr = r0 + 16 * n + r;
            if (gr >= a.rows) continue;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < NW; ++w) M = fmaxf(M, sml[n][w][r][0]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float den = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(sml[n][w][r][0] - M);
                const float4 x = *reinterpret_cast<const float4*>(&so[w][r][d]);
                acc.x += f * x.x, acc.y += f * x.y, acc.z += f * x.z, acc.w += f * x.w;
                den += f * sml[n][w][r][1];
            }
            if (a.splits == 1) {
                const float inv = den == 0.f ? 0.f : 1.f / den;
                const int tk = gr / a.G, h = kvh * a.G + gr % a.G;
                *reinterpret_cast<uint2*>(a.o + ((int64_t)tk * a.Hq + h) * HD + d) =
                    make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
            } else {
                const int64_t at = ((int64_t)split * a.Hkv + kvh) * a.rows + gr;
                if (tile_end > split * a.split_tiles) *reinterpret_cast<float4*>(a.o_part + at * HD + d) = acc;
                if (d == 0) *reinterpret_cast<float2*>(a.ml_part + at * 2) = make_float2(M, den);
            }
        }
    }
}

// Joins the splits of a row, weighted by exp2(m_s - max m): NT threads a row, HD / 4 across its
// channels by P lanes that take every P-th split each and are added in order. Many rows have few
// splits: a wave each; a decode step's few rows have many: a workgroup each.
template <int HD, int NT>
__global__ __launch_bounds__(256) void kv_fp4_merge_kernel(KvFp4Args a) {
    constexpr int C = HD / 4, P = NT / C, CH = 8, RW = 256 / NT;   // at most NT splits
    __shared__ float wt[RW][NT], red_max[4], red_sum[4];
    __shared__ float4 part[RW][P][C];
    const int64_t all = (int64_t)a.Hkv * a.rows;
    const int rw = threadIdx.x / NT, tid = threadIdx.x % NT, c = tid % C, lane_p = tid / C;
    const int64_t r = (int64_t)blockIdx.x * RW + rw, rr = min(r, all - 1);
    // Every split has written its (maximum, sum); one that has no keys for the row has (-inf, 0), and
    // perhaps no output. The first outputs are requested before that is known.
    float4 x[CH];
    const float* const op = a.o_part + rr * HD + c * 4;
    auto request = [&](int s0) {
#pragma unroll
        for (int k = 0; k < CH; ++k)
            x[k] = s0 + k * P < a.splits ? *reinterpret_cast<const float4*>(op + (int64_t)(s0 + k * P) * all * HD) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    request(lane_p);
    const float2 ml = tid < a.splits ? *reinterpret_cast<const float2*>(a.ml_part + ((int64_t)tid * all + rr) * 2) : make_float2(-INFINITY, 0.f);
    float M = wave_max_uniform(ml.x);
    if constexpr (NT == 256) {
        if (tid % kWave == 0) red_max[tid / kWave] = M;
        __syncthreads();
        M = fmaxf(fmaxf(red_max[0], red_max[1]), fmaxf(red_max[2], red_max[3]));
    }
    const bool used = ml.y != 0.f || ml.x != -INFINITY;
    const float f = M == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(ml.x - M);
    if (tid < a.splits) wt[rw][tid] = used ? f : -1.f;
    float den = wave_total(used ? f * ml.y : 0.f);
    if constexpr (NT == 256) {
        if (tid % kWave == 0) red_sum[tid / kWave] = den;
    }
    __syncthreads();
    if constexpr (NT == 256) den = (red_sum[0] + red_sum[1]) + (red_sum[2] + red_sum[3]);
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = lane_p; s0 < a.splits; s0 += CH * P) {
        if (s0 != lane_p) request(s0);
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const float w = s0 + k * P < a.splits ? wt[rw][s0 + k * P] : -1.f;
            if (w < 0.f) continue;
            t.x += w * x[k].x, t.y += w * x[k].y, t.z += w * x[k].z, t.w += w * x[k].w;
        }
    }
    part[rw][lane_p][c] = t;
    __syncthreads();
    if (lane_p > 0 || r >= all) return;
#pragma unroll
    for (int p = 1; p < P; ++p) {
        const float4 y = part[rw][p][c];
        t.x += y.x, t.y += y.y, t.z += y.z, t.w += y.w;
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
    const int kvh = (int)(r / a.rows), gr = (int)(r % a.rows), tk = gr / a.G, h = kvh * a.G + gr % a.G;
    *reinterpret_cast<uint2*>(a.o + ((int64_t)tk * a.Hq + h) * HD + c * 4) =
        make_uint2(pack_bf16x2(t.x * inv, t.y * inv), pack_bf16x2(t.z * inv, t.w * inv));
}

// Many rows: four waves with 32 rows each share the keys. 64 keys (a stage) at a time the waves make
// a quarter of the stage's operands each, the codes of the next stage unpacked into LDS in the order
// in which the lanes take them: unpacking costs a row an eighth of what it does above. A wave's own
// instructions alternate: unpacking goes out between the first products, the second tile's exponentials
// between the first tile's second products, and a wave at its products goes before the other on its SIMD,
// which so falls to its softmax (4096 rows of 28/4 heads: 150 us one after the other, 143 alternating, 122 with
// the priority). 4096 rows 970 TFLOP/s, 8192 rows 1090; fewer rows are bound by workgroups that see more
// keys than others.
// Heads of 128; the keys are not split, since there are rows enough.
__global__ __launch_bounds__(256, 2) void kv_fp4_rows_kernel(KvFp4Args a) {
    constexpr int HD = 128, W = HD / 32, MT = HD / 16, NQ = 2;
    constexpr int FRAGS = 2 * W + MT;                // 1 KB operands of a 32-key tile: keys [2][W], values [MT]
    constexpr int AHEAD = 4;
    __shared__ uint4 frag[2][2][FRAGS][kWave];       // [buffer][tile of the stage]
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), l = lane % 16, g = lane / 16;
    // Row blocks from the last, which see the most keys, the KV heads side by side. The second workgroup to
    // arrive at a CU is the lighter the heavier its first (2500 rows of 28/4 heads 70 us, 75 in plain order).
    int rank = blockIdx.x;
    const int resident = min((int)gridDim.x, 2 * a.cus);
    if (rank >= a.cus && rank < resident) rank = a.cus + resident - 1 - rank;
    const int r0 = ((int)(gridDim.x / a.Hkv) - 1 - rank / a.Hkv) * (64 * NQ), kvh = rank % a.Hkv;
    const KvFp4Layout lay(a.T, a.Hkv, HD);
    const int L = (int)a.kv_len;
    int sees[NQ];
    bf16x8_t qf[NQ][W];
    const int w0 = r0 + wave * 16 * NQ;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int row = w0 + 16 * n + l, tok = row / a.G, head = kvh * a.G + row % a.G;
        const bool on = row < a.rows;
        sees[n] = !on ? 0 : a.causal ? L - (int)a.S + tok + 1 : L;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            uint4 u = make_uint4(0, 0, 0, 0);
            if (on) u = *reinterpret_cast<const uint4*>(a.q + (int64_t)tok * a.q_sn + (int64_t)head * a.q_sh + 32 * w + 8 * g);
            qf[n][w] = __builtin_bit_cast(bf16x8_t, u);
        }
    }
    // keys that any row of the workgroup sees; that any and every row of the wave sees
    const int last = min(r0 + 64 * NQ - 1, a.rows - 1) / a.G;
    const int any_sees = a.causal ? L - (int)a.S + last + 1 : L;
    const int wave_sees = w0 >= a.rows ? 0 : a.causal ? L - (int)a.S + min(w0 + 16 * NQ - 1, a.rows - 1) / a.G + 1 : L;
    const int all_see = w0 + 16 * NQ > a.rows ? 0 : a.causal ? L - (int)a.S + w0 / a.G + 1 : L;
    const int stages = (any_sees + 63) / 64;

    // this wave's part of a stage: tile wave / 2, operand wave % 2 of the keys, bytes (HD / 64) (wave % 2) on of
    // the values' words
    const int part = wave % 2;
    const int oshift = part * (HD / 8);
    const int kr = (wave / 2) * 32 + 8 * (l / 4) + 4 * part + l % 4;
    const uint8_t* const kc = a.cache + lay.k(kvh) + kr * (HD / 2) + g * (HD / 8);
    const uint8_t* const vc = a.cache + lay.v(kvh) + (((wave / 2) * 4 + g) * (HD / 8) + l) * 32;
    const uint8_t* const ksc = a.cache + lay.ks(kvh) + kr * W;
    const uint8_t* const vsc = a.cache + lay.vs(kvh) + (((wave / 2) * 4 + g) * W + l / 4) * 8;
    const int tile_max = (int)(a.T / 32) - 1;   // the cache's last tile; a stage may end past it
    uint32_t ck[W], cks, cv[8], cvs[2];
    bool saw_nan = false;
    auto load = [&](int st) {
        const int t = min(2 * st + wave / 2, tile_max) - wave / 2;   // the bases are at the wave's tile of stage 0
        const int ko = t * (32 * HD / 2), sof = t * (32 * W);
        const uint4 c = *reinterpret_cast<const uint4*>(kc + ko);
        ck[0] = c.x, ck[1] = c.y, ck[2] = c.z, ck[3] = c.w;
        cks = *reinterpret_cast<const uint32_t*>(ksc + sof);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 u = *reinterpret_cast<const uint4*>(vc + ko + 16 * i);
            cv[4 * i] = u.x, cv[4 * i + 1] = u.y, cv[4 * i + 2] = u.z, cv[4 * i + 3] = u.w;
        }
        const uint2 u = *reinterpret_cast<const uint2*>(vsc + sof);
        cvs[0] = u.x, cvs[1] = u.y;
    };
    // The codes at hand, of stage st, are unpacked into a buffer in 24 pieces, which go out between the
    // matrix instructions. Before that, values past the end and NaN groups are made zeros.
    auto clean = [&](int st) {
        const int key0 = (2 * st + wave / 2) * 32 + 8 * g;
        const uint32_t ff = ((cvs[0] & 0x7f7f7f7fu) + 0x01010101u) & cvs[0], fg = ((cvs[1] & 0x7f7f7f7fu) + 0x01010101u) & cvs[1];
        if (st * 64 + 64 > L || __any(((ff | fg) & 0x80808080u) != 0)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t byte = (cvs[i / 4] >> (8 * (i % 4))) & 255;
                const bool off = key0 + i >= L;
                if (off || byte == kFp4ScaleNan) {
                    saw_nan |= !off;
                    cv[i] = 0;
                    cvs[i / 4] &= ~(255u << (8 * (i % 4)));
                }
            }
        }
    };
    constexpr int PIECES = W + 2 * 10;
    uint32_t e[8];
    auto unpack = [&](auto pc, int b) {
        constexpr int P = decltype(pc)::value, V = P - W, B = V / 10, I = V % 10;
        uint4 (*const f)[kWave] = frag[b][wave / 2];
        if constexpr (P < W) {
            f[part * W + P][lane] = __builtin_bit_cast(uint4, fp4_unpack8(ck[P], fp4_scale_at(cks, P)));
        } else if constexpr (I < 8) {
            e[I] = fp4_pair<B>(cv[I] >> oshift, fp4_scale_at(cvs[I / 4], I % 4));
        } else {
            constexpr uint32_t half = I == 8 ? 0x05040100 : 0x07060302;
            f[2 * W + part * (MT / 2) + 2 * B + I - 8][lane] =
                make_uint4(__builtin_amdgcn_perm(e[1], e[0], half), __builtin_amdgcn_perm(e[3], e[2], half),
                           __builtin_amdgcn_perm(e[5], e[4], half), __builtin_amdgcn_perm(e[7], e[6], half));
        }
    };
    // f(0) to f(n - 1)
    auto each = [](auto nc, auto&& f) {
        [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
        (std::make_integer_sequence<int, decltype(nc)::value>{});
    };

    f32x4_t o[NQ][MT];
    float m[NQ], sum[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        m[n] = -INFINITY, sum[n] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[n][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    auto meet = [&]() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    using std::integral_constant;
    load(0);   // every row sees a key
    clean(0);
    each(integral_constant<int, PIECES>{}, [&](auto pc) { unpack(pc, 0); });
    load(min(1, stages - 1));
    for (int st = 0; st < stages; ++st) {
        const int b = st & 1;
        meet();   // this stage is in LDS, and the other buffer is read out
        // the stage's operands in the order of their use: keys of both tiles, values of both; AHEAD reads under way
        bf16x8_t ring[AHEAD];
        auto read = [&](auto fc) {
            constexpr int F = decltype(fc)::value, T = F < 4 * W ? F / (2 * W) : (F - 4 * W) / MT, X = F < 4 * W ? F % (2 * W) : 2 * W + (F - 4 * W) % MT;
            if constexpr (F < 2 * FRAGS) ring[F % AHEAD] = __builtin_bit_cast(bf16x8_t, frag[b][T][X][lane]);
        };
        each(integral_constant<int, AHEAD>{}, read);
        clean(st + 1);   // past the last stage: the last one once more, into a buffer that nothing reads
        f32x4_t s[NQ][2][2];
        __builtin_amdgcn_s_setprio(1);
        each(integral_constant<int, 4 * W>{}, [&](auto fc) {
            constexpr int F = decltype(fc)::value, T = F / (2 * W), I = F / W % 2;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                s[n][T][I] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ring[F % AHEAD], qf[n][F % W], F % W == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : s[n][T][I], 0, 0, 0);
                if (n == 1) read(integral_constant<int, F + AHEAD>{});
                constexpr int P0 = F * PIECES / (4 * W), P1 = (F + 1) * PIECES / (4 * W), PM = (P0 + P1) / 2;
                if (n == 0) each(integral_constant<int, PM - P0>{}, [&](auto pc) { unpack(integral_constant<int, P0 + decltype(pc)::value>{}, 1 - b); });
                else each(integral_constant<int, P1 - PM>{}, [&](auto pc) { unpack(integral_constant<int, PM + decltype(pc)::value>{}, 1 - b); });
                __builtin_amdgcn_sched_barrier(0);
            }
        });
        __builtin_amdgcn_s_setprio(0);
        load(min(st + 2, stages - 1));
        bf16x8_t pf[NQ][2];
        float ref[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
            ref[n] = kv_fp4_maximum<MT, 2>(s[n], st * 64 + 8 * g, st * 64 + 64 > all_see, sees[n], a.scale, m[n], sum[n], o[n]);
        uint4 pw[NQ];
        // weights E and E + 1 of a row's tile
        auto weigh = [&](int n, int t, auto ec) {
            constexpr int E = decltype(ec)::value;
            const float x = __builtin_amdgcn_exp2f(fmaf(s[n][t][E / 4][E % 4], a.scale, -ref[n]));
            const float y = __builtin_amdgcn_exp2f(fmaf(s[n][t][E / 4][E % 4 + 1], a.scale, -ref[n]));
            sum[n] += x + y;
            reinterpret_cast<uint32_t*>(&pw[n])[E / 2] = pack_bf16x2(x, y);
        };
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            each(integral_constant<int, 4>{}, [&](auto ec) { weigh(n, 0, integral_constant<int, 2 * decltype(ec)::value>{}); });
            pf[n][0] = __builtin_bit_cast(bf16x8_t, pw[n]);
        }
        __builtin_amdgcn_s_setprio(1);
        each(integral_constant<int, 2 * MT>{}, [&](auto fc) {
            constexpr int F = decltype(fc)::value, T = F / MT, I = F % MT;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                o[n][I] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ring[(4 * W + F) % AHEAD], pf[n][T], o[n][I], 0, 0, 0);
                if (n == 1) read(integral_constant<int, 4 * W + F + AHEAD>{});
                // the second tile's weights, beside the first tile's products
                if (T == 0 && n == 1) weigh(F / 4, 1, integral_constant<int, 2 * (F % 4)>{});
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (T == 0 && I == MT - 1) {
#pragma unroll
                for (int n = 0; n < NQ; ++n) pf[n][1] = __builtin_bit_cast(bf16x8_t, pw[n]);
            }
        });
        __builtin_amdgcn_s_setprio(0);
    }
    // NaN groups of values reach the outputs of the rows that see them
    meet();
    int* const flag = reinterpret_cast<int*>(&frag[0][0][0][0]);
    const bool wave_saw = __any(saw_nan);
    if (lane == 0) flag[wave] = wave_saw;
    meet();
    if (flag[0] | flag[1] | flag[2] | flag[3])
        for (int k = 0; k < wave_sees; ++k)
            kv_fp4_put_nan<HD, NQ>(a.cache + lay.vs(kvh), lay, k, g, sees, o);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const float den = over_groups(sum[n], [](float x, float y) { return x + y; });
        const int gr = w0 + 16 * n + l;
        if (gr >= a.rows) continue;
        const float inv = den == 0.f ? 0.f : 1.f / den;
        const int tk = gr / a.G, h = kvh * a.G + gr % a.G;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            bf16_t* const dst = a.o + ((int64_t)tk * a.Hq + h) * HD + 8 * (4 * g + r);
#pragma unroll
            for (int i = 0; i < MT; i += 4)
                *reinterpret_cast<uint2*>(dst + i) = make_uint2(pack_bf16x2(o[n][i][r] * inv, o[n][i + 1][r] * inv),
                                                               pack_bf16x2(o[n][i + 2][r] * inv, o[n][i + 3][r] * inv));
        }
    }
}

struct KvFp4Plan {
    bool shared;                           // kv_fp4_rows_kernel
    int nw, nq, split_tiles, splits;
    size_t o_bytes, ml_bytes;              // partial outputs and (maximum, sum)
    size_t total() const { return o_bytes + ml_bytes; }
};

// Measured on 256 CUs (us). One row: 200 keys of 14/2 heads 3.8 in one workgroup a head, 6.3 split; 500
// keys of 12/2 heads 5.4 and 6.6; 700 keys of 12/2 heads 6.8 and 6.6, of 14/2 heads of 64 5.5 and 6.3; 2000
// keys of 28/4 heads 7.2 in workgroups of four waves, 7.4 of eight; 32771 keys 11.9 with up to 512
// workgroups, 10.9 with 256. Rows, kv_fp4_attn_kernel with 16 and with 32 rows a workgroup: 37 rows behind 8000 of
// 12/2 heads 13 / 16, 512 behind 512 of 28/4 heads 22 / 17. kv_fp4_attn_kernel with 32 and kv_fp4_rows_kernel, by the
// latter's workgroups: behind as many rows, 28/4 heads, 372 of them 87 / 95, 396 101 / 100, 416 107 / 105, 448
// 117 / 104, 484 138 / 120, and behind 8000 416 303 / 272; 16/2 heads 376 140 / 159, 414 172 / 176, 448 190 / 176; 12/2
// heads 404 217 / 226, 442 244 / 246, 516 346 / 323. Alone, 28/4 heads, 448 51 / 52, 484 58 / 60, 548 70.7 / 69.2,
// 640 92 / 83; 12/2 heads 564 142 / 152, 640 178 / 181; 10000 rows of them 364 / 283. 13/8 of the CUs
// lies between the head layouts' borders: 396 workgroups of 28/4 heads behind 4000 keys take 172 instead of 160.
static KvFp4Plan kv_fp4_plan(const efm_attention_ctx* c, uint32_t S, uint32_t kv_len, bool causal) {
    const int64_t Hkv = c->num_kv_heads, rows = (int64_t)S * (c->num_qo_heads / Hkv), cus = prefill_cus();
    const int tiles = (int)(((int64_t)kv_len + 31) / 32);
    auto blocks_of = [&](int n) { return (rows + n - 1) / n * Hkv; };
    KvFp4Plan p = {};
    // The shared kernel's 128-row workgroups pay where they fill the CUs' places (two each) and more, or nearly
    // fill them and differ little in their keys.
    const int64_t shared = blocks_of(128);
    p.shared = c->head_dim == 128 && S > 1 &&
               (2 * shared >= 5 * cus || (8 * shared >= 13 * cus && (!causal || kv_len >= S + S / 2)));
    p.nq = blocks_of(16) >= 2 * cus ? 2 : 1;
    p.nw = p.nq == 2 ? 4 : 8;
    const int64_t blocks = p.shared ? shared : blocks_of(16 * p.nq);
    int least = p.nw;   // tiles of a split: one for each wave
    if (S == 1) {
        // few tiles: one workgroup a head and no second launch; else four waves until there is one a CU
        const int alone = (c->head_dim == 64 ? 3 : 2) * 8;
        if (tiles <= alone) least = alone;
        else if ((tiles + 3) / 4 * blocks <= cus) p.nw = least = 4;
    }
    const int64_t want = std::max<int64_t>(1, cus / blocks);   // one workgroup a CU where keys are split
    p.split_tiles = std::max({least, (int)((tiles + want - 1) / want), (tiles + kKvFp4MaxSplits - 1) / kKvFp4MaxSplits});
    p.splits = std::max(1, (tiles + p.split_tiles - 1) / p.split_tiles);
    if (p.splits > 1) {
        p.o_bytes = (size_t)p.splits * Hkv * rows * c->head_dim * sizeof(float);
        p.ml_bytes = (size_t)p.splits * Hkv * rows * 2 * sizeof(float);
    }
    return p;
}

// Bytes that hold the partial results of every call of up to S rows behind up to kv_len keys. A call's
// own need goes up and down with its sizes; splits <= min(tiles, CUs / blocks of 16 rows) bounds it.
static size_t kv_fp4_workspace(const efm_attention_ctx* c, uint32_t S, uint32_t kv_len) {
    const int64_t tiles = ((int64_t)kv_len + 31) / 32, cus = prefill_cus();
    if (tiles <= 8) return 0;
    const int64_t rows = std::min(std::min(tiles, cus) * S * (int64_t)c->num_qo_heads, 16 * cus);
    return rows * (c->head_dim + 2) * sizeof(float);
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
    if (ctx->num_qo_heads > (1u << 16) || (uint64_t)S * ctx->num_qo_heads > (1ull << 30))
        return set_error(EFM_ERR_UNSUPPORTED, "%s: %u rows of %u query heads", who, S, ctx->num_qo_heads);
    const int hd = (int)ctx->head_dim;
    const KvFp4Plan p = kv_fp4_plan(ctx, S, bound, causal != 0);
    const int64_t rows = (int64_t)S * (ctx->num_qo_heads / ctx->num_kv_heads), block = p.shared ? 128 : 16 * p.nq;
    const int64_t groups = (rows + block - 1) / block * ctx->num_kv_heads;
    const int threads = kWave * (p.shared ? 4 : p.nw);
    if (groups * threads > kGridThreads)
        return set_error(EFM_ERR_UNSUPPORTED, "%s: %u rows of %u query heads", who, S, ctx->num_qo_heads);
    if (p.total() > 0 && (workspace == nullptr || workspace_bytes < p.total()))
        return set_error(EFM_ERR_WORKSPACE, "%s: workspace of %zu bytes required", who, p.total());
    if (p.total() > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", who);
    const KvFp4Layout lay(KvFp4Layout::rows(max_rows), (int)ctx->num_kv_heads, hd);
    KvFp4Args a;
    a.q = static_cast<const bf16_t*>(q);
    a.cache = static_cast<const uint8_t*>(cache);
    a.o = static_cast<bf16_t*>(o);
    a.o_part = static_cast<float*>(workspace);
    a.ml_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.o_bytes);
    a.d_kv_len = d_kv_len;
    a.T = lay.T;
    a.q_sn = ctx->q_stride_n ? ctx->q_stride_n : (int64_t)ctx->num_qo_heads * hd;
    a.q_sh = ctx->q_stride_h ? ctx->q_stride_h : hd;
    a.kv_len = kv_len;
    a.max_kv_len = max_kv_len;
    a.S = S;
    a.Hq = (int)ctx->num_qo_heads;
    a.Hkv = (int)ctx->num_kv_heads;
    a.G = a.Hq / a.Hkv;
    a.causal = causal != 0;
    a.rows = (int)rows;
    a.split_tiles = p.split_tiles;
    a.splits = p.splits;
    a.tiles = (int)((bound + 31) / 32);
    a.cus = prefill_cus();
    a.scale = 1.4426950408889634f / sqrtf((float)hd);
    const dim3 grid((unsigned)groups, 1, p.splits);
    const int64_t all = (int64_t)a.Hkv * a.rows;
    auto launch = [&](auto hdc) {
        constexpr int HD = decltype(hdc)::value;
        if (p.shared) hipLaunchKernelGGL(kv_fp4_rows_kernel, grid, dim3(threads), 0, stream, a);
        else if (p.nq == 2) hipLaunchKernelGGL((kv_fp4_attn_kernel<HD, 4, 2>), grid, dim3(threads), 0, stream, a);
        else if (p.nw == 4) hipLaunchKernelGGL((kv_fp4_attn_kernel<HD, 4, 1>), grid, dim3(threads), 0, stream, a);
        else hipLaunchKernelGGL((kv_fp4_attn_kernel<HD, 8, 1>), grid, dim3(threads), 0, stream, a);
        if (p.splits > 1 && p.splits <= kWave && all >= 256)
            hipLaunchKernelGGL((kv_fp4_merge_kernel<HD, kWave>), dim3((unsigned)((all + 3) / 4)), dim3(256), 0, stream, a);
        else if (p.splits > 1)
            hipLaunchKernelGGL((kv_fp4_merge_kernel<HD, 256>), dim3((unsigned)all), dim3(256), 0, stream, a);
    };
    if (hd == 128) launch(std::integral_constant<int, 128>{});
    else launch(std::integral_constant<int, 64>{});
    return check_launch(who);
}

}  // namespace efm

using namespace efm;

extern "C" size_t efm_attention_decode_kv_fp4_workspace_bytes(const efm_attention_ctx* ctx, uint32_t max_kv_len) {
    if (validate_attention_ctx(ctx, "attention_decode_kv_fp4_workspace_bytes") != EFM_OK) return 0;
    return kv_fp4_workspace(ctx, 1, max_kv_len);
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
    return kv_fp4_workspace(ctx, qo_len, kv_len);
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
