// Attention of a tree of drafted tokens over a bf16 cache that holds their own keys in its last rows
// (gfx950, bf16 in, fp32 softmax). Node i sees the L - n rows before the tree and, of the tree's n
// rows, those with a bit in its mask.
//
// The query rows of the heads that share a KV head are flattened (row r: node r / G, head r % G) and
// taken 32 at a time; S^T = K Q^T and O^T = V^T P^T go to the 32 x 32 x 16 matrix instructions with
// the keys as the first operand, so that a lane holds one row's scores and P enters the second
// product from the registers that it was made in (layouts in attn_split.hpp and attn_pipe.hpp). A
// workgroup's waves take every KW-th tile of its split of the keys, each through LDS of its own.
// Where the keys are split over workgroups too, those write unnormalised outputs with (maximum,
// sum), and a second kernel joins them.
//
// P is rounded to bf16 for the second product, and the sums are over the rounded P, so that the
// weights of a row add up to one; maxima, sums and outputs stay in fp32.
#include "attn_split.hpp"
#include "common.hpp"

#include <algorithm>
#include <type_traits>

namespace efm {

int validate_attention_ctx(const efm_attention_ctx* c, const char* who);
int prefill_cus();

constexpr int kTreeMaxSplits = 256;
constexpr float kTreeLazy = 8.f;   // a maximum is followed once it is exceeded by 2^8 in weights

struct TreeArgs {
    const bf16_t* q;
    const bf16_t* k;
    const bf16_t* v;
    bf16_t* o;
    const uint64_t* mask;
    float* o_part;    // [splits][Hkv][rows][HD]
    float* ml_part;   // [splits][Hkv][rows][2]
    const uint32_t* d_kv_len;
    uint32_t kv_len, max_kv_len;
    int n, words, Hq, Hkv, G, rows;   // rows: n * G
    int64_t q_sn, q_sh, k_sh, v_sh;
    int k_sn, v_sn;
    int blocks, splits, split_tiles;
    float scale;      // log2(e) / sqrt(HD)
};

// Rows attended; 0 where the device's length cannot be (the outputs are then zero).
__device__ __forceinline__ int tree_len(const TreeArgs& a) {
    if (a.d_kv_len == nullptr) return (int)a.kv_len;
    const uint32_t L = a.d_kv_len[0];
    return L >= (uint32_t)a.n && L <= a.max_kv_len ? (int)L : 0;
}

// Bit i: the node sees key k0 + i, for the KT keys from k0; c0: k0's place in the tree (negative in
// the rows before it).
template <int KT>
__device__ __forceinline__ uint64_t tree_window(const uint64_t* row, int words, int c0) {
    if (c0 <= -KT) return ~0ull;
    if (c0 < 0) return row[0] << -c0 | ((1ull << -c0) - 1);
    const int w = c0 / 64, sh = c0 % 64;
    uint64_t bits = w < words ? row[w] >> sh : 0ull;
    if (sh != 0 && w + 1 < words) bits |= row[w + 1] << (64 - sh);
    return bits;
}

// A bf16 pair with zeros in the place of infinities and NaN.
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
    return w;
}

// Channels 4 c to 4 c + 3 of a row: the output, or what a split hands on. some: the split has keys.
template <int HD>
__device__ __forceinline__ void tree_store(const TreeArgs& a, int kvh, int split, int row, int c, float m, float l, const float4& acc, bool some) {
    if (a.splits == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<uint2*>(a.o + ((int64_t)(row / a.G) * a.Hq + kvh * a.G + row % a.G) * HD + c * 4) =
            make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
        return;
    }
    const int64_t at = ((int64_t)split * a.Hkv + kvh) * a.rows + row;
    if (some) *reinterpret_cast<float4*>(a.o_part + at * HD + c * 4) = acc;
    if (c == 0) *reinterpret_cast<float2*>(a.ml_part + at * 2) = make_float2(m, l);
}

template <int HD, int KW>
__global__ __launch_bounds__(KW * kWave, 2) void tree_attn_kernel(TreeArgs a) {
    typedef SplitTile<HD> T;
    constexpr int KT = T::kKeys, NH = KT / 32, KS = HD / 16, DT = HD / 32, NL = T::kLoads, KB = KT / 16;
    constexpr int SLOT = 2 * T::kBytes, CPR = HD / 4;
    typedef short s4_t __attribute__((ext_vector_type(4)));
    __shared__ __align__(1024) unsigned char smem[KW * SLOT];
    __shared__ float ml[2][KW][32];

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
    const int ql = lane % 32, hh = lane / 32;
    // the row blocks of a (head, split) are 8 workgroups apart: on one XCD, whose L2 they share
    const int xcd = blockIdx.x % 8, rest = blockIdx.x / 8;
    const int unit = rest / a.blocks * 8 + xcd, block = rest % a.blocks;
    if (unit >= a.Hkv * a.splits) return;
    const int kvh = unit % a.Hkv, split = unit / a.Hkv;
    const int r0 = block * 32, row = r0 + ql, node = min(row, a.rows - 1) / a.G, head = kvh * a.G + min(row, a.rows - 1) % a.G;

    const int L = tree_len(a), before = L - a.n;   // rows before the tree
    const int tiles = (L + KT - 1) / KT;
    const int tile_end = min(tiles, (split + 1) * a.split_tiles);
    int t = split * a.split_tiles + wave;

    const char* const kbase = reinterpret_cast<const char*>(a.k + kvh * a.k_sh);
    const char* const vbase = reinterpret_cast<const char*>(a.v + kvh * a.v_sh);
    unsigned char* const kslot = smem + wave * SLOT;
    unsigned char* const vslot = kslot + T::kBytes;
    const int pr = lane / T::kChunks, pc = lane % T::kChunks;
    auto issue = [&](const char* base, int sn, int k0, unsigned char* slot, auto is_v) {
        const char* const t0 = base + (int64_t)k0 * sn * 2;
        const bool whole = k0 + KT <= L;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int rr = i * T::kRows + pr;
            const int c = pc ^ (decltype(is_v)::value ? T::v_swz(rr) : T::k_swz(rr));
            const int r = whole ? rr : min(rr, L - 1 - k0);   // rows past the end read the last row
            __builtin_amdgcn_global_load_lds(static_cast<const void*>(t0 + (uint32_t)((r * sn + c * 8) * 2)),
                                             (__attribute__((address_space(3))) void*)(slot + i * 1024), 16, 0, 0);
        }
    };
    auto issue_k = [&](int tt) { issue(kbase, a.k_sn, tt * KT, kslot, std::false_type{}); };
    auto issue_v = [&](int tt) { issue(vbase, a.v_sn, tt * KT, vslot, std::true_type{}); };

    // Q, the second operand: d = 16 ks + 8 hh + e
    bf16x8_t qf[KS];
    {
        const bf16_t* qp = a.q + node * a.q_sn + head * a.q_sh;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            Pack8 x;
            x.u = *reinterpret_cast<const uint4*>(qp + ks * 16 + hh * 8);
            qf[ks] = x.v;
        }
    }
    if (t < tile_end) {
        issue_k(t);
        issue_v(t);
    }
    f32x16_t oacc[DT];
#pragma unroll
    for (int tt = 0; tt < DT; ++tt)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[tt][e] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    const uint64_t* const bits_row = a.mask + (int64_t)node * a.words;

    const uint32_t lk = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)kslot);
    uint32_t ka[KS], va[DT];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ka[ks] = lk + (uint32_t)(ql * T::kRow + (((ks * 2 + hh) ^ T::k_swz(ql)) << 4));
    {
        const int g = lane >> 4, j = lane & 15, rr = (g >> 1) * 4 + (j >> 2);
#pragma unroll
        for (int tt = 0; tt < DT; ++tt) {
            const int d = tt * 32 + 16 * (g & 1) + 4 * (j & 3);
            va[tt] = lk + (uint32_t)(T::kBytes + rr * T::kRow + (((d >> 3) ^ T::v_swz(rr)) << 4) + ((d & 7) << 1));
        }
    }
    const float lazy = kTreeLazy / a.scale;
    for (; t < tile_end; t += KW) {
        const bool more = t + KW < tile_end;
        const int kb0 = t * KT;
        const bool masked = kb0 + KT > before;
        uint64_t bits = ~0ull;
        if (masked) {   // requested before the waits below
            bits = tree_window<KT>(bits_row, a.words, kb0 - before);
            if (L - kb0 < 64) bits &= (1ull << (L - kb0)) - 1;
            asm volatile("" : "+v"(bits));
            attn_pipe::vm_wait<0>();
        } else {
            attn_pipe::vm_wait<NL>();   // K has landed; V may be under way
        }
        asm volatile("" ::: "memory");
        bf16x8_t kf[NH][KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            attn_pipe::read_b128<0>(kf[0][ks], ka[ks]);
            if constexpr (NH == 2) attn_pipe::read_b128<32 * T::kRow>(kf[1][ks], ka[ks]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(kf[h][ks]));
        // Values that a row does not see take no part in its output whatever they are: a zero weight
        // times an infinity would be a NaN. V of the tree's rows and of rows past the end is made
        // finite here, and what was not is added below where it is seen.
        bool odd = false;
        if (masked) {
            uint4* const vp = reinterpret_cast<uint4*>(vslot);
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const uint4 x = vp[i * 64 + lane];
                const uint4 y = make_uint4(finite_pair(x.x), finite_pair(x.y), finite_pair(x.z), finite_pair(x.w));
                if (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w) {
                    odd = true;
                    vp[i * 64 + lane] = y;
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
        if (more) issue_k(t + KW);
        // S^T - m; element e of s[h]: key kb0 + 32 h + 8 (e / 4) + 4 hh + e % 4 of the lane's row
        const float start = m_run == -INFINITY ? 0.f : -m_run;
        f32x16_t s[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[h][e] = start;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s[h] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[h][ks], qf[ks], s[h], 0, 0, 0);
        }
        if (!masked) {
            if (more) attn_pipe::vm_wait<NL>();
            else attn_pipe::vm_wait<0>();
        }
        asm volatile("" ::: "memory");
        s4_t vf[KB][DT][2];
#pragma unroll
        for (int tt = 0; tt < DT; ++tt) {
            attn_pipe::read_tr16<0>(vf[0][tt][0], va[tt]);
            attn_pipe::read_tr16<8 * T::kRow>(vf[0][tt][1], va[tt]);
            attn_pipe::read_tr16<16 * T::kRow>(vf[1][tt][0], va[tt]);
            attn_pipe::read_tr16<24 * T::kRow>(vf[1][tt][1], va[tt]);
            if constexpr (KB == 4) {
                attn_pipe::read_tr16<32 * T::kRow>(vf[KB - 2][tt][0], va[tt]);
                attn_pipe::read_tr16<40 * T::kRow>(vf[KB - 2][tt][1], va[tt]);
                attn_pipe::read_tr16<48 * T::kRow>(vf[KB - 1][tt][0], va[tt]);
                attn_pipe::read_tr16<56 * T::kRow>(vf[KB - 1][tt][1], va[tt]);
            }
        }
        if (masked) {
            const uint64_t mine = bits >> (4 * hh);
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s[h][e] = (mine >> (32 * h + 8 * (e / 4) + e % 4) & 1) ? s[h][e] : -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, s[h][e]);
        {
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        }
        if (__any((m_run == -INFINITY && top > -INFINITY) || top > lazy)) {
            // a row may see none of its wave's first tiles: its maximum stays -inf, its weights are 0
            const float m_new = fmaxf(m_run, top - start);
            const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run - m_new) * a.scale);
            const float shift = m_new == -INFINITY ? 0.f : m_new + start;
            l_run *= alpha;
#pragma unroll
            for (int tt = 0; tt < DT; ++tt)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[tt][e] *= alpha;
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[h][e] -= shift;
            m_run = m_new;
        }
        Pack8 pb[KB];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            float p[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(s[h][e] * a.scale);
            pb[2 * h].u = pack8(&p[0]);
            pb[2 * h + 1].u = pack8(&p[8]);
        }
        float psum = 0.f;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            psum = add_bf16_pair(pb[b].u.x, psum);
            psum = add_bf16_pair(pb[b].u.y, psum);
            psum = add_bf16_pair(pb[b].u.z, psum);
            psum = add_bf16_pair(pb[b].u.w, psum);
        }
        {
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(psum), __float_as_uint(psum), false, false);
            l_run += __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int tt = 0; tt < DT; ++tt) asm volatile("" : "+v"(vf[kb][tt][0]), "+v"(vf[kb][tt][1]));
        if (more) issue_v(t + KW);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int tt = 0; tt < DT; ++tt) {
                union {
                    s4_t h[2];
                    bf16x8_t v;
                } vv;
                vv.h[0] = vf[kb][tt][0];
                vv.h[1] = vf[kb][tt][1];
                oacc[tt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vv.v, pb[kb].v, oacc[tt], 0, 0, 0);
            }
        if (__any(odd)) {
            // the values that were not finite, from memory: rows that see the key add them
            const int keys = min(KT, L - kb0);
            for (int j = 0; j < keys; ++j) {
                const bf16_t* const vr = reinterpret_cast<const bf16_t*>(vbase) + (int64_t)(kb0 + j) * a.v_sn;
                const bool seen = bits >> j & 1;
#pragma unroll
                for (int tt = 0; tt < DT; ++tt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int d = tt * 32 + (e / 4) * 8 + hh * 4 + e % 4;
                        const uint32_t x = vr[d];
                        if (seen && (x & 0x7f80u) == 0x7f80u) oacc[tt][e] += bf16_to_f32(x);
                    }
            }
        }
    }

    // the waves' outputs meet in LDS (float4 chunk c of row r at c ^ (r & 15))
    {
        float4* const part = reinterpret_cast<float4*>(kslot);
#pragma unroll
        for (int tt = 0; tt < DT; ++tt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                part[ql * CPR + ((tt * 8 + g * 2 + hh) ^ (ql & 15))] =
                    make_float4(oacc[tt][g * 4], oacc[tt][g * 4 + 1], oacc[tt][g * 4 + 2], oacc[tt][g * 4 + 3]);
        if (hh == 0) {
            ml[0][wave][ql] = m_run * a.scale;
            ml[1][wave][ql] = l_run;
        }
    }
    __syncthreads();
    for (int idx = tid; idx < 32 * CPR; idx += KW * kWave) {
        const int r = idx / CPR, c = idx % CPR, gr = r0 + r;
        if (gr >= a.rows) continue;
        float m = ml[0][0][r];
#pragma unroll
        for (int w = 1; w < KW; ++w) m = fmaxf(m, ml[0][w][r]);
        float l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            // a wave that saw nothing of the row has no part in it
            if (ml[0][w][r] == -INFINITY && ml[1][w][r] == 0.f) continue;
            const float x = __builtin_amdgcn_exp2f(ml[0][w][r] - m);
            const float4 y = reinterpret_cast<const float4*>(smem + w * SLOT)[r * CPR + (c ^ (r & 15))];
            l += x * ml[1][w][r];
            acc.x += x * y.x;
            acc.y += x * y.y;
            acc.z += x * y.z;
            acc.w += x * y.w;
        }
        tree_store<HD>(a, kvh, split, gr, c, m, l, acc, tile_end > split * a.split_tiles);
    }
}

// Many rows: a workgroup takes 128 rows. Tiles of 64 keys go through a ring in LDS that its eight waves
// read in common; a wave takes 32 rows and one half of a tile's keys. Two waves a SIMD, so that one's
// softmax runs beside the other's products, and a ring of S tiles, S - 1 of them under way.
template <int HD>
__global__ __launch_bounds__(512, 2) void tree_rows_kernel(TreeArgs a) {
    typedef SplitTile<HD> T;
    constexpr int KT = 64, KS = HD / 16, DT = HD / 32, CPR = HD / 4, S = HD == 128 ? 4 : 6;
    constexpr int TILE = KT * T::kRow, STAGE = 2 * TILE;   // bytes: keys or values; both
    constexpr int NL = TILE / 1024 / 8;                    // loads of a wave: keys, and as many of values
    typedef short s4_t __attribute__((ext_vector_type(4)));
    constexpr int SMEM = S * STAGE > 8 * 32 * HD * 4 ? S * STAGE : 8 * 32 * HD * 4;   // the ring, later the outputs
    __shared__ __align__(1024) unsigned char smem[SMEM];
    __shared__ float ml[2][2][128];
    __shared__ int s_odd;

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, grp = wave / 4, wg = wave % 4;
    const int ql = lane % 32, hh = lane / 32;
    const int xcd = blockIdx.x % 8, rest = blockIdx.x / 8;
    const int unit = rest / a.blocks * 8 + xcd, block = rest % a.blocks;
    if (unit >= a.Hkv * a.splits) return;
    const int kvh = unit % a.Hkv, split = unit / a.Hkv;
    const int r0 = block * 128, row = min(r0 + wg * 32 + ql, a.rows - 1), node = row / a.G, head = kvh * a.G + row % a.G;
    const bool idle = r0 + wg * 32 >= a.rows;   // a wave without rows helps to load

    const int L = tree_len(a), before = L - a.n;
    const int t0 = split * a.split_tiles, tile_end = min((L + KT - 1) / KT, t0 + a.split_tiles), tiles = max(tile_end - t0, 0);
    if (tid == 0) s_odd = -1;

    const char* const kbase = reinterpret_cast<const char*>(a.k + kvh * a.k_sh);
    const char* const vbase = reinterpret_cast<const char*>(a.v + kvh * a.v_sh);
    const int pr = lane / T::kChunks, pc = lane % T::kChunks;
    auto issue = [&](int t, int slot) {
        const int k0 = t * KT;
        const bool whole = k0 + KT <= L;
        unsigned char* const dst = smem + slot * STAGE + wave * 1024;
#pragma unroll
        for (int i = 0; i < 2 * NL; ++i) {
            const bool is_v = i >= NL;
            const int rr = ((i % NL) * 8 + wave) * T::kRows + pr;
            const int c = pc ^ (is_v ? T::v_swz(rr) : T::k_swz(rr));
            const int r = whole ? rr : min(rr, L - 1 - k0);   // rows past the end read the last row
            const int sn = is_v ? a.v_sn : a.k_sn;
            const char* const src = (is_v ? vbase : kbase) + (int64_t)k0 * sn * 2 + (uint32_t)((r * sn + c * 8) * 2);
            __builtin_amdgcn_global_load_lds(static_cast<const void*>(src),
                                             (__attribute__((address_space(3))) void*)(dst + (is_v ? TILE : 0) + (i % NL) * 8192), 16, 0, 0);
        }
    };
    bf16x8_t qf[KS];
    {
        const bf16_t* qp = a.q + node * a.q_sn + head * a.q_sh;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            Pack8 x;
            x.u = *reinterpret_cast<const uint4*>(qp + ks * 16 + hh * 8);
            qf[ks] = x.v;
        }
    }
    for (int i = 0; i < S - 1; ++i)
        if (i < tiles) issue(t0 + i, i);
    f32x16_t oacc[DT];
#pragma unroll
    for (int tt = 0; tt < DT; ++tt)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[tt][e] = 0.f;
    float m_run = -INFINITY, l_part = 0.f;
    const uint64_t* const bits_row = a.mask + (int64_t)node * a.words;
    const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)smem);
    uint32_t koff[KS], voff[DT];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) koff[ks] = lds + (uint32_t)((grp * 32 + ql) * T::kRow + (((ks * 2 + hh) ^ T::k_swz(ql)) << 4));
    {
        const int g = lane >> 4, j = lane & 15, rr = (g >> 1) * 4 + (j >> 2);
#pragma unroll
        for (int tt = 0; tt < DT; ++tt) {
            const int d = tt * 32 + 16 * (g & 1) + 4 * (j & 3);
            voff[tt] = lds + (uint32_t)(TILE + (grp * 32 + rr) * T::kRow + (((d >> 3) ^ T::v_swz(rr)) << 4) + ((d & 7) << 1));
        }
    }
    const float lazy = kTreeLazy / a.scale;
    auto meet = [] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    for (int st = 0; st < tiles; ++st) {
        const int k0 = (t0 + st) * KT, kb0 = k0 + grp * 32;
        const bool masked = k0 + KT > before;   // the tile has rows of the tree: the same in every wave
        const uint32_t slot = (uint32_t)(st % S);
        uint64_t bits = ~0ull;
        if (masked) {
            bits = tree_window<32>(bits_row, a.words, kb0 - before);
            bits &= L - kb0 >= 32 ? 0xffffffffull : L - kb0 > 0 ? (1ull << (L - kb0)) - 1 : 0ull;
            asm volatile("" : "+v"(bits));
        }
        switch (min(S - 2, tiles - 1 - st)) {   // tiles that may be under way
            case 0: attn_pipe::vm_wait<0>(); break;
            case 1: attn_pipe::vm_wait<2 * NL>(); break;
            case 2: attn_pipe::vm_wait<4 * NL>(); break;
            case 3: attn_pipe::vm_wait<6 * NL>(); break;
            default: attn_pipe::vm_wait<8 * NL>(); break;
        }
        meet();   // the tile is there, and the slot of the one before is read out
        unsigned char* const stage = smem + slot * STAGE;
        if (masked) {
            // values that are not finite are made zeros, and added below where they are seen
            bool odd = false;
            uint4* const vp = reinterpret_cast<uint4*>(stage + TILE);
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const uint4 x = vp[(i * 8 + wave) * 64 + lane];
                const uint4 y = make_uint4(finite_pair(x.x), finite_pair(x.y), finite_pair(x.z), finite_pair(x.w));
                if (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w) {
                    odd = true;
                    vp[(i * 8 + wave) * 64 + lane] = y;
                }
            }
            if (__any(odd) && lane == 0) s_odd = st;
            meet();
        }
        if (st + S - 1 < tiles) issue(t0 + st + S - 1, (st + S - 1) % S);
        if (idle || kb0 >= L) continue;
        const uint32_t at = slot * STAGE;
        // S^T; element e: key kb0 + 8 (e / 4) + 4 hh + e % 4 of the lane's row
        f32x16_t s;
        bf16x8_t kf[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) attn_pipe::read_b128<0>(kf[ks], koff[ks] + at);
        s4_t vf[2][DT][2];
        auto read_v = [&](auto kbc) {
            constexpr int kb = decltype(kbc)::value;
#pragma unroll
            for (int tt = 0; tt < DT; ++tt) {
                attn_pipe::read_tr16<(kb * 16) * T::kRow>(vf[kb][tt][0], voff[tt] + at);
                attn_pipe::read_tr16<(kb * 16 + 8) * T::kRow>(vf[kb][tt][1], voff[tt] + at);
            }
        };
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(KS / 2) : "memory");
#pragma unroll
        for (int ks = 0; ks < KS / 2; ++ks) asm volatile("" : "+v"(kf[ks]));
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS / 2; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks], qf[ks], s, 0, 0, 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int ks = KS / 2; ks < KS; ++ks) asm volatile("" : "+v"(kf[ks]));
#pragma unroll
        for (int ks = KS / 2; ks < KS; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks], qf[ks], s, 0, 0, 0);
        read_v(std::integral_constant<int, 0>{});
        read_v(std::integral_constant<int, 1>{});
        if (masked) {
            const uint32_t mine = (uint32_t)bits >> (4 * hh);
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = (mine >> (8 * (e / 4) + e % 4) & 1) ? s[e] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(top, s[e]);
        {
            const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
        }
        if (__any(top > m_run + lazy)) {   // -inf: whatever is seen first
            const float m_new = fmaxf(m_run, top);
            const float alpha = m_run == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m_run - m_new) * a.scale);
            l_part *= alpha;
#pragma unroll
            for (int tt = 0; tt < DT; ++tt)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[tt][e] *= alpha;
            m_run = m_new;
        }
        const float ref = m_run == -INFINITY ? 0.f : m_run * a.scale;
        Pack8 pb[2];
        {
            float p[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale, -ref));
            pb[0].u = pack8(&p[0]);
            pb[1].u = pack8(&p[8]);
        }
        float psum = 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            psum = add_bf16_pair(pb[b].u.x, psum);
            psum = add_bf16_pair(pb[b].u.y, psum);
            psum = add_bf16_pair(pb[b].u.z, psum);
            psum = add_bf16_pair(pb[b].u.w, psum);
        }
        l_part += psum;   // of the lane's half of the keys
        auto pv = [&](int kb) {
#pragma unroll
            for (int tt = 0; tt < DT; ++tt) {
                asm volatile("" : "+v"(vf[kb][tt][0]), "+v"(vf[kb][tt][1]));
                union {
                    s4_t h[2];
                    bf16x8_t v;
                } vv;
                vv.h[0] = vf[kb][tt][0];
                vv.h[1] = vf[kb][tt][1];
                oacc[tt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vv.v, pb[kb].v, oacc[tt], 0, 0, 0);
            }
        };
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(2 * DT) : "memory");
        pv(0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        pv(1);
        if (masked && s_odd == st) {
            const int keys = min(32, L - kb0);
            for (int j = 0; j < keys; ++j) {
                const bf16_t* const vr = reinterpret_cast<const bf16_t*>(vbase) + (int64_t)(kb0 + j) * a.v_sn;
                const bool seen = bits >> j & 1;
#pragma unroll
                for (int tt = 0; tt < DT; ++tt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const uint32_t x = vr[tt * 32 + (e / 4) * 8 + hh * 4 + e % 4];
                        if (seen && (x & 0x7f80u) == 0x7f80u) oacc[tt][e] += bf16_to_f32(x);
                    }
            }
        }
    }
    float l_run;
    {
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_part), __float_as_uint(l_part), false, false);
        l_run = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    }
    // the groups' outputs meet in LDS (float4 chunk c of row r at c ^ (r & 15))
    meet();
    {
        float4* const part = reinterpret_cast<float4*>(smem + (grp * 4 + wg) * 32 * HD * 4);
#pragma unroll
        for (int tt = 0; tt < DT; ++tt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                part[ql * CPR + ((tt * 8 + g * 2 + hh) ^ (ql & 15))] =
                    make_float4(oacc[tt][g * 4], oacc[tt][g * 4 + 1], oacc[tt][g * 4 + 2], oacc[tt][g * 4 + 3]);
        if (hh == 0) {
            ml[0][grp][wg * 32 + ql] = m_run * a.scale;
            ml[1][grp][wg * 32 + ql] = l_run;
        }
    }
    __syncthreads();
    for (int idx = tid; idx < 128 * CPR; idx += 512) {
        const int r = idx / CPR, c = idx % CPR, gr = r0 + r;
        if (gr >= a.rows) break;
        const float m = fmaxf(ml[0][0][r], ml[0][1][r]);
        float l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            if (ml[0][g][r] == -INFINITY && ml[1][g][r] == 0.f) continue;   // it saw nothing of the row
            const float x = __builtin_amdgcn_exp2f(ml[0][g][r] - m);
            const float4 y = reinterpret_cast<const float4*>(smem + (g * 4 + r / 32) * 32 * HD * 4)[r % 32 * CPR + (c ^ (r & 15))];
            l += x * ml[1][g][r];
            acc.x += x * y.x;
            acc.y += x * y.y;
            acc.z += x * y.z;
            acc.w += x * y.w;
        }
        tree_store<HD>(a, kvh, split, gr, c, m, l, acc, tiles > 0);
    }
}

// Joins the splits of a row: a wave a row, HD / 4 lanes across its channels, the rest over the splits.
template <int HD>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
    constexpr int C = HD / 4, P = kWave / C, CH = 8;
    __shared__ float wt[4][kTreeMaxSplits];
    const int64_t all = (int64_t)a.Hkv * a.rows;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, c = lane % C, part = lane / C;
    const int64_t r = (int64_t)blockIdx.x * 4 + wave, rr = min(r, all - 1);
    float M = -INFINITY;
    float2 mine[kTreeMaxSplits / kWave];
#pragma unroll
    for (int i = 0; i < kTreeMaxSplits / kWave; ++i) {
        const int s = i * kWave + lane;
        mine[i] = s < a.splits ? *reinterpret_cast<const float2*>(a.ml_part + ((int64_t)s * all + rr) * 2) : make_float2(-INFINITY, 0.f);
        M = fmaxf(M, mine[i].x);
    }
    M = wave_max_uniform(M);
    float den = 0.f;
#pragma unroll
    for (int i = 0; i < kTreeMaxSplits / kWave; ++i) {
        const bool used = mine[i].x != -INFINITY || mine[i].y != 0.f;   // the others may have no output
        const float f = used ? __builtin_amdgcn_exp2f(mine[i].x - M) : 0.f;
        den += used ? f * mine[i].y : 0.f;
        wt[wave][i * kWave + lane] = used ? f : -1.f;
    }
    den = wave_total(den);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    const float* const op = a.o_part + rr * HD + c * 4;
    for (int s0 = part; s0 < a.splits; s0 += CH * P) {
        float4 x[CH];
        float w[CH];
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const int s = s0 + k * P;
            w[k] = s < a.splits ? wt[wave][s] : -1.f;
            if (!(w[k] < 0.f)) x[k] = *reinterpret_cast<const float4*>(op + (int64_t)s * all * HD);
        }
#pragma unroll
        for (int k = 0; k < CH; ++k)
            if (!(w[k] < 0.f)) t.x += w[k] * x[k].x, t.y += w[k] * x[k].y, t.z += w[k] * x[k].z, t.w += w[k] * x[k].w;
    }
    // the parts of a channel are C lanes apart
#pragma unroll
    for (int off = C; off < kWave; off *= 2) {
        t.x += __shfl_xor(t.x, off, kWave), t.y += __shfl_xor(t.y, off, kWave);
        t.z += __shfl_xor(t.z, off, kWave), t.w += __shfl_xor(t.w, off, kWave);
    }
    if (part > 0 || r >= all) return;
    const float inv = den == 0.f ? 0.f : 1.f / den;
    const int kvh = (int)(r / a.rows), gr = (int)(r % a.rows);
    *reinterpret_cast<uint2*>(a.o + ((int64_t)(gr / a.G) * a.Hq + kvh * a.G + gr % a.G) * HD + c * 4) =
        make_uint2(pack_bf16x2(t.x * inv, t.y * inv), pack_bf16x2(t.z * inv, t.w * inv));
}

struct TreePlan {
    bool many;   // tree_rows_kernel
    int blocks, splits, split_tiles;
    size_t o_bytes, ml_bytes;
    size_t total() const { return o_bytes + ml_bytes; }
};

static TreePlan tree_plan(const efm_attention_ctx* c, uint32_t n, uint32_t kv_len) {
    const int hd = (int)c->head_dim, Hkv = (int)c->num_kv_heads;
    const int64_t rows = (int64_t)n * (c->num_qo_heads / c->num_kv_heads), cus = prefill_cus();
    TreePlan p = {};
    p.many = rows > 64;
    const int keys = p.many || hd == 64 ? 64 : 32, waves = 4;
    const int64_t tiles = ((int64_t)kv_len + keys - 1) / keys;
    p.blocks = (int)(p.many ? (rows + 127) / 128 : (rows + 31) / 32);
    // workgroups: one a CU of the large ones, two of the small
    const int64_t want = std::max<int64_t>(1, (p.many ? 1 : 2) * cus / ((int64_t)p.blocks * Hkv));
    p.split_tiles = (int)std::max<int64_t>({p.many ? 4 : 2 * waves, (tiles + want - 1) / want, (tiles + kTreeMaxSplits - 1) / kTreeMaxSplits});
    p.splits = (int)std::max<int64_t>(1, (tiles + p.split_tiles - 1) / p.split_tiles);
    if (p.splits > 1) {
        p.o_bytes = (size_t)p.splits * Hkv * rows * hd * sizeof(float);
        p.ml_bytes = (size_t)p.splits * Hkv * rows * 2 * sizeof(float);
    }
    return p;
}

// Bytes that hold the partial results of every call of up to n nodes over up to kv_len rows: a call's
// own need goes up and down with its sizes, and splits <= min(tiles, workgroups wanted / row blocks).
static size_t tree_workspace(const efm_attention_ctx* c, uint32_t n, uint32_t kv_len) {
    const int64_t tiles = ((int64_t)kv_len + 31) / 32, cus = prefill_cus();
    if (kv_len <= 256) return 0;
    const int64_t splits = std::min<int64_t>(tiles, kTreeMaxSplits);
    const int64_t rows = std::min(splits * n * (int64_t)c->num_qo_heads, 128 * cus);   // workgroups' rows: 128 a CU, or twice 32
    return (size_t)rows * (c->head_dim + 2) * sizeof(float);
}

}  // namespace efm

using namespace efm;

extern "C" size_t efm_attention_tree_workspace_bytes(const efm_attention_ctx* ctx, uint32_t nodes, uint32_t max_kv_len) {
    if (validate_attention_ctx(ctx, "attention_tree_workspace_bytes") != EFM_OK) return 0;
    if (nodes > EFM_DRAFT_TREE_MAX_NODES || max_kv_len > (1u << 24)) return 0;
    return tree_workspace(ctx, nodes, max_kv_len);
}

extern "C" int efm_attention_tree(const efm_attention_ctx* ctx, const void* q, const void* k, const void* v, const uint64_t* mask,
                                  void* o, uint32_t nodes, uint32_t kv_len, const uint32_t* d_kv_len, uint32_t max_kv_len,
                                  void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const int rc = validate_attention_ctx(ctx, "attention_tree");
    if (rc) return rc;
    if (ctx->pos_encoding != EFM_POS_NONE)
        return set_error(EFM_ERR_UNSUPPORTED, "attention_tree: pos_encoding must be EFM_POS_NONE (a node's position is not its row)");
    if (!q || !k || !v || !mask || !o) return set_error(EFM_ERR_INVALID_ARGUMENT, "attention_tree: null tensor pointer");
    if (nodes == 0) return set_error(EFM_ERR_INVALID_ARGUMENT, "attention_tree: a tree has a node at least");
    if (nodes > EFM_DRAFT_TREE_MAX_NODES)
        return set_error(EFM_ERR_UNSUPPORTED, "attention_tree: %u nodes, %d at most", nodes, EFM_DRAFT_TREE_MAX_NODES);
    const uint32_t bound = d_kv_len != nullptr ? max_kv_len : kv_len;
    if (bound < nodes) return set_error(EFM_ERR_INVALID_ARGUMENT, "attention_tree: %u rows with %u nodes among them", bound, nodes);
    if (bound > (1u << 24)) return set_error(EFM_ERR_UNSUPPORTED, "attention_tree: %u rows", bound);
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
          reinterpret_cast<uintptr_t>(o)) & 15u) != 0 || (reinterpret_cast<uintptr_t>(mask) & 7u) != 0 ||
        (reinterpret_cast<uintptr_t>(d_kv_len) & 3u) != 0)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "attention_tree: misaligned pointer");
    // offsets inside a tile are of 32 bits
    if (ctx->k_stride_n >= (1u << 24) || ctx->kv_stride_n >= (1u << 24) || ctx->num_qo_heads > (1u << 14))
        return set_error(EFM_ERR_UNSUPPORTED, "attention_tree: row strides %u and %u, %u query heads", ctx->k_stride_n, ctx->kv_stride_n,
                         ctx->num_qo_heads);
    const int hd = (int)ctx->head_dim;
    const TreePlan p = tree_plan(ctx, nodes, bound);
    if (p.total() > 0 && (workspace == nullptr || workspace_bytes < p.total()))
        return set_error(EFM_ERR_WORKSPACE, "attention_tree: workspace of %zu bytes required", p.total());
    if (p.total() > 0 && (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "attention_tree: workspace must be 16-byte aligned");
    const int Hq = (int)ctx->num_qo_heads, Hkv = (int)ctx->num_kv_heads;
    TreeArgs a;
    a.q = static_cast<const bf16_t*>(q);
    a.k = static_cast<const bf16_t*>(k);
    a.v = static_cast<const bf16_t*>(v);
    a.o = static_cast<bf16_t*>(o);
    a.mask = mask;
    a.o_part = static_cast<float*>(workspace);
    a.ml_part = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.o_bytes);
    a.d_kv_len = d_kv_len;
    a.kv_len = kv_len;
    a.max_kv_len = max_kv_len;
    a.n = (int)nodes;
    a.words = ((int)nodes + 63) / 64;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.G = Hq / Hkv;
    a.rows = a.n * a.G;
    a.q_sn = ctx->q_stride_n ? (int64_t)ctx->q_stride_n : (int64_t)Hq * hd;
    a.q_sh = ctx->q_stride_h ? (int64_t)ctx->q_stride_h : hd;
    a.k_sn = ctx->k_stride_n ? (int)ctx->k_stride_n : Hkv * hd;
    a.k_sh = ctx->k_stride_h ? (int64_t)ctx->k_stride_h : hd;
    a.v_sn = ctx->kv_stride_n ? (int)ctx->kv_stride_n : Hkv * hd;
    a.v_sh = ctx->kv_stride_h ? (int64_t)ctx->kv_stride_h : hd;
    a.blocks = p.blocks;
    a.splits = p.splits;
    a.split_tiles = p.split_tiles;
    a.scale = 1.4426950408889634f / sqrtf((float)hd);
    const int64_t units = ((int64_t)Hkv * p.splits + 7) / 8 * 8, all = (int64_t)Hkv * a.rows;
    const dim3 grid((unsigned)(units * p.blocks)), joins((unsigned)((all + 3) / 4));
    if (hd == 128) {
        if (p.many) hipLaunchKernelGGL(tree_rows_kernel<128>, grid, dim3(512), 0, stream, a);
        else hipLaunchKernelGGL((tree_attn_kernel<128, 4>), grid, dim3(256), 0, stream, a);
        if (p.splits > 1) hipLaunchKernelGGL(tree_merge_kernel<128>, joins, dim3(256), 0, stream, a);
    } else {
        if (p.many) hipLaunchKernelGGL(tree_rows_kernel<64>, grid, dim3(512), 0, stream, a);
        else hipLaunchKernelGGL((tree_attn_kernel<64, 4>), grid, dim3(256), 0, stream, a);
        if (p.splits > 1) hipLaunchKernelGGL(tree_merge_kernel<64>, joins, dim3(256), 0, stream, a);
    }
    return check_launch("attention_tree");
}
