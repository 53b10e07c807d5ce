// Attention of a tree of drafted tokens over a bf16 cache that holds their own keys in its last rows (gfx950, bf16 in,
// fp32 softmax). Node i sees the L - n rows before the tree and, of the tree's n rows, those with a bit in its mask.
//
// The query rows of the heads that share a KV head are flattened (row r: node r / G, head r % G) and taken 32 a wave;
// S^T = K Q^T and O^T = V^T P^T go to the 32 x 32 x 16 matrix instructions with the keys as the first operand, so that
// a lane holds one row's scores and P enters the second product from the registers that it was made in (layouts in
// attn_split.hpp and attn_pipe.hpp). The keys are split over waves and workgroups; parts carry unnormalised outputs
// with (maximum, sum) and are joined in LDS, and a second kernel joins those of different workgroups.
//
// P is rounded to bf16 for the second product, and the sums are over the rounded P, so that the weights of a row add up
// to one; maxima, sums and outputs stay in fp32.
//
// A short context is bound by latencies: a launch, a length and a tile that come from memory, the join. A long one reads
// the cache at half of the memory's rate: a step's chain takes twice its matrix instructions' time, and the parts that the
// splits write and the second launch weigh as much as a third (33 nodes at 32000 rows of 4 heads of 128: 66 MB and 16 MB
// of parts in 25 us, the join 5 us).
#include "attn_split.hpp"
#include "common.hpp"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace efm {

int validate_attention_ctx(const efm_attention_ctx* c, const char* who);
int prefill_cus();

constexpr int kTreeMaxSplits = 256;
constexpr int kTreeMany = 16000, kTreeWhole = 12, kTreeLeast = 4;   // tree_plan
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
    int bound;                        // rows that the cache holds
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

// The 64 bits of a node's mask from key c0 of the tree on, which may be before it: bit i says that the node sees key
// c0 + i. request() may come long before get(), which waits for it.
struct TreeBits {
    uint64_t lo, hi;
    __device__ __forceinline__ void request(const uint64_t* row, int words, int c0) {
        const int w = max(c0, 0) / 64;
        lo = row[min(w, words - 1)], hi = row[min(w + 1, words - 1)];
    }
    __device__ __forceinline__ uint64_t get(int words, int c0) const {
        if (c0 <= -64) return ~0ull;
        if (c0 < 0) return lo << -c0 | ((1ull << -c0) - 1);
        const int w = c0 / 64, sh = c0 % 64;
        const uint64_t a = w < words ? lo >> sh : 0ull, b = w + 1 < words ? hi << 1 << (63 - sh) : 0ull;
        return a | b;
    }
};

typedef short tree_s4_t __attribute__((ext_vector_type(4)));   // four values of a lane

// Whether words of bf16 pairs hold infinities or NaN: an exponent of ones carries into the bit above it.
struct TreeOdd {
    uint32_t sum = 0;
    __device__ __forceinline__ void look(uint32_t w) { sum |= (w & 0x7f807f80u) + 0x00800080u; }
    __device__ __forceinline__ void look(tree_s4_t x) {
        const uint2 w = __builtin_bit_cast(uint2, x);
        look(w.x), look(w.y);
    }
    __device__ __forceinline__ bool any() const { return __any((sum & 0x80008000u) != 0); }
};

// A score, or -inf where bit i is not set.
__device__ __forceinline__ float tree_masked(float s, uint32_t bits, int i) {
    const uint32_t seen = (uint32_t)((int)(bits << (31 - i)) >> 31);
    return __uint_as_float((__float_as_uint(s) & seen) | (0xff800000u & ~seen));
}

// A bf16 pair with zeros in the place of infinities and NaN.
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
    return w;
}

__device__ __forceinline__ tree_s4_t tree_finite(tree_s4_t x) {
    uint2 w = __builtin_bit_cast(uint2, x);
    w = make_uint2(finite_pair(w.x), finite_pair(w.y));
    return __builtin_bit_cast(tree_s4_t, w);
}

// The first n of four values, zeros in the place of the others.
__device__ __forceinline__ tree_s4_t tree_first(tree_s4_t x, int n) {
    const uint64_t keep = n <= 0 ? 0ull : n >= 4 ? ~0ull : (1ull << (16 * n)) - 1;
    return __builtin_bit_cast(tree_s4_t, __builtin_bit_cast(uint64_t, x) & keep);
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

// What a workgroup works at. Workgroups go to the 8 XCDs in turn: an XCD takes an eighth of all workgroups, the row
// blocks of a (split, head) side by side, which share the tiles in its L2. (Whole pairs to the XCDs in turn leave some of
// them idle where the pairs are few or no multiple of 8: 1000 nodes at 2000 rows 53 -> 191 us.)
__device__ __forceinline__ bool tree_place(const TreeArgs& a, int& kvh, int& split, int& block) {
    const int all = a.Hkv * a.splits * a.blocks, xcd = blockIdx.x % 8, at = xcd * all / 8 + (int)(blockIdx.x / 8);
    if (at >= (xcd + 1) * all / 8) return false;
    block = at % a.blocks, kvh = at / a.blocks % a.Hkv, split = at / a.blocks / a.Hkv;
    return true;
}

// Adds what is not finite of channels 4 c to 4 c + 3 of the values of keys [j0, j1) that a row sees.
__device__ __forceinline__ void tree_not_finite(const TreeArgs& a, const char* vbase, int row, int c, int before, int j0, int j1, float4& acc) {
    const uint64_t* const bits = a.mask + (int64_t)(row / a.G) * a.words;
#pragma unroll 1
    for (int j = j0; j < j1; ++j) {
        const int at = j - before;
        if (at >= 0 && !(bits[at / 64] >> at % 64 & 1)) continue;
        const uint2 x = *reinterpret_cast<const uint2*>(vbase + ((int64_t)j * a.v_sn + c * 4) * 2);
        acc.x += (x.x & 0x7f80u) == 0x7f80u ? lo_f32(x.x) : 0.f;
        acc.y += (x.x & 0x7f800000u) == 0x7f800000u ? hi_f32(x.x) : 0.f;
        acc.z += (x.y & 0x7f80u) == 0x7f80u ? lo_f32(x.y) : 0.f;
        acc.w += (x.y & 0x7f800000u) == 0x7f800000u ? hi_f32(x.y) : 0.f;
    }
}

// Joins the outputs of P parts of a workgroup, part(p, row, chunk), with the rows' maxima at ml[p * R + row] and sums at
// ml[(P + p) * R + row]; N chunks of four channels a thread. A part that saw nothing of a row has none in it.
template <int HD, int P, int N, typename Part, typename Last>
__device__ __forceinline__ void tree_join(const TreeArgs& a, int tid, int threads, int kvh, int split, int r0, bool some, Part part,
                                          const float* ml, int R, Last last) {
    constexpr int CPR = HD / 4;
    const int c = tid % CPR, step = threads / CPR;
    // a row's weights once, the outputs of two rows under way
#pragma unroll 2
    for (int i = 0; i < N; ++i) {
        const int r = tid / CPR + i * step, gr = r0 + r;
        float mp[P], lp[P], m = -INFINITY, l = 0.f;
        float4 y[P], acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int p = 0; p < P; ++p) mp[p] = ml[p * R + r], lp[p] = ml[(P + p) * R + r], y[p] = part(p, r, c);
#pragma unroll
        for (int p = 0; p < P; ++p) m = fmaxf(m, mp[p]);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const bool used = mp[p] != -INFINITY || lp[p] != 0.f;
            const float x = used ? __builtin_amdgcn_exp2f(mp[p] - m) : 0.f;
            l += used ? x * lp[p] : 0.f;
            acc.x += used ? x * y[p].x : 0.f;
            acc.y += used ? x * y[p].y : 0.f;
            acc.z += used ? x * y[p].z : 0.f;
            acc.w += used ? x * y[p].w : 0.f;
        }
        if (gr < a.rows) {
            last(gr, c, acc);
            tree_store<HD>(a, kvh, split, gr, c, m, l, acc, some);
        }
    }
}

// f(0) to f(N - 1), the index a constant.
template <int N, typename F>
__device__ __forceinline__ void tree_each(F f) {
    [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
    (std::make_integer_sequence<int, N>{});
}

// Little work: 32 rows a workgroup, whose waves take every KW-th tile of 8 KB of keys and 8 KB of values, each through a
// slot of its own in LDS that is requested again as soon as it is read out, so that no wave waits for another
// before the end. Two workgroups share a CU: one's products run while the other's tiles arrive. (Two slots a wave and
// loads two tiles ahead, one workgroup a CU: 11.4 -> 12.3 us for 24 nodes at 2003 rows, 28 -> 61 us for 250 at 3900.)
template <int HD>
__global__ __launch_bounds__(256, 2) void tree_few_kernel(TreeArgs a) {
    typedef SplitTile<HD> T;
    constexpr int KW = 4, KT = T::kKeys, NH = KT / 32, KS = HD / 16, DT = HD / 32, NL = T::kLoads, KB = KT / 16;
    constexpr int SLOT = 2 * T::kBytes, CPR = HD / 4;
    __shared__ __align__(1024) unsigned char smem[KW * SLOT];
    __shared__ float ml[2][KW][32];
    __shared__ int s_odd[KW];
    static_assert(32 * HD * 4 <= SLOT && 32 * CPR % (KW * kWave) == 0, "a wave's outputs fit in its slot");

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
    const int ql = lane % 32, hh = lane / 32;
    int kvh, split, block;
    if (!tree_place(a, kvh, split, block)) return;
    const int r0 = block * 32, row = min(r0 + ql, a.rows - 1), node = row / a.G, head = kvh * a.G + row % a.G;
    const int bound = a.bound, t0 = split * a.split_tiles;
    int t = t0 + wave;

    const char* const kbase = reinterpret_cast<const char*>(a.k + kvh * a.k_sh);
    const char* const vbase = reinterpret_cast<const char*>(a.v + kvh * a.v_sh);
    unsigned char* const kslot = smem + wave * SLOT;
    unsigned char* const vslot = kslot + T::kBytes;
    const int pr = lane / T::kChunks, pc = lane % T::kChunks;
    auto issue = [&](const char* base, int sn, int k0, unsigned char* slot, auto is_v) {
        const char* const tile = base + (int64_t)k0 * sn * 2;
        const bool whole = k0 + KT <= bound;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int rr = i * T::kRows + pr;
            const int c = pc ^ (decltype(is_v)::value ? T::v_swz(rr) : T::k_swz(rr));
            const int r = whole ? rr : min(rr, bound - 1 - k0);   // rows past the end read the last row
            __builtin_amdgcn_global_load_lds(static_cast<const void*>(tile + (uint32_t)((r * sn + c * 8) * 2)),
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
    // the first tile is requested before the length is known: the cache holds `bound` rows
    if (t < min((bound + KT - 1) / KT, t0 + a.split_tiles)) {
        issue_k(t);
        issue_v(t);
    }
    const int L = tree_len(a), before = L - a.n;   // rows before the tree
    const int tile_end = min((L + KT - 1) / KT, t0 + a.split_tiles);
    // Q has landed here: a first use in the loop would wait for every load under way, each time
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
    f32x16_t oacc[DT];
#pragma unroll
    for (int tt = 0; tt < DT; ++tt)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[tt][e] = 0.f;
    float m_run = -INFINITY, l_part = 0.f;   // the largest score so far; the sum over the lane's half of the keys
    bool odd = false;
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
            TreeBits window;
            window.request(bits_row, a.words, kb0 - before);
            bits = window.get(a.words, kb0 - before);
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
        if (more) issue_k(t + KW);
        // S^T; element e of s[h]: key kb0 + 32 h + 8 (e / 4) + 4 hh + e % 4 of the lane's row
        f32x16_t s[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[h][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s[h] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[h][ks], qf[ks], s[h], 0, 0, 0);
        }
        if (!masked) {
            if (more) attn_pipe::vm_wait<NL>();
            else attn_pipe::vm_wait<0>();
        }
        asm volatile("" ::: "memory");
        tree_s4_t vf[KB][DT][2];
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
                for (int e = 0; e < 16; ++e) s[h][e] = tree_masked(s[h][e], (uint32_t)(mine >> (32 * h)), 8 * (e / 4) + e % 4);
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
        if (__any(top > m_run + lazy)) {   // from -inf: whatever is seen first
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
        Pack8 pb[KB];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            float p[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[h][e], a.scale, -ref));
            pb[2 * h].u = pack8(&p[0]);
            pb[2 * h + 1].u = pack8(&p[8]);
        }
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            l_part = add_bf16_pair(pb[b].u.x, l_part);
            l_part = add_bf16_pair(pb[b].u.y, l_part);
            l_part = add_bf16_pair(pb[b].u.z, l_part);
            l_part = add_bf16_pair(pb[b].u.w, l_part);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int tt = 0; tt < DT; ++tt) asm volatile("" : "+v"(vf[kb][tt][0]), "+v"(vf[kb][tt][1]));
        if (more) issue_v(t + KW);
        // Values that a row does not see take no part in its output whatever they are: a zero weight times an infinity
        // would be a NaN. V of the tree's rows and of rows past the end is made finite here, and what was not of the
        // tree's rows is added at the end where it is seen. (Rows past the end among those looked for: 200 nodes
        // behind 2000 rows 19 -> 72 us whenever the cache holds a NaN there, 1000 nodes 46 -> 1100.)
        if (masked) {
            TreeOdd look;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int tt = 0; tt < DT * 2; ++tt) {
                    look.look(vf[kb][tt / 2][tt % 2]);
                }
            if (look.any()) {
                const int left = L - kb0 - 4 * hh;   // the lane's keys: 16 kb + 8 (tt % 2) + 0 to 3 of these
                TreeOdd seen;
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int tt = 0; tt < DT * 2; ++tt) {
                        const tree_s4_t x = tree_first(vf[kb][tt / 2][tt % 2], left - 16 * kb - 8 * (tt % 2));
                        seen.look(x);
                        vf[kb][tt / 2][tt % 2] = tree_finite(x);
                    }
                odd |= seen.any();
            }
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int tt = 0; tt < DT; ++tt) {
                union {
                    tree_s4_t h[2];
                    bf16x8_t v;
                } vv;
                vv.h[0] = vf[kb][tt][0];
                vv.h[1] = vf[kb][tt][1];
                oacc[tt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vv.v, pb[kb].v, oacc[tt], 0, 0, 0);
            }
    }
    attn_pipe::vm_wait<0>();   // a tile past the length
    asm volatile("" ::: "memory");

    // the waves' outputs meet in LDS (float4 chunk c of row r at c ^ (r & 15))
    {
        float4* const part = reinterpret_cast<float4*>(kslot);
#pragma unroll
        for (int tt = 0; tt < DT; ++tt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                part[ql * CPR + ((tt * 8 + g * 2 + hh) ^ (ql & 15))] =
                    make_float4(oacc[tt][g * 4], oacc[tt][g * 4 + 1], oacc[tt][g * 4 + 2], oacc[tt][g * 4 + 3]);
        const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_part), __float_as_uint(l_part), false, false);
        if (hh == 0) {
            ml[0][wave][ql] = m_run * a.scale;
            ml[1][wave][ql] = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
        }
        odd = __any(odd);
        if (lane == 0) s_odd[wave] = odd;
    }
    __syncthreads();
    odd = false;
#pragma unroll
    for (int w = 0; w < KW; ++w) odd |= s_odd[w] != 0;
    tree_join<HD, KW, 32 * CPR / (KW * kWave)>(a, tid, KW * kWave, kvh, split, r0, tile_end > t0, [&](int w, int r, int c) {
        return reinterpret_cast<const float4*>(smem + w * SLOT)[r * CPR + (c ^ (r & 15))];
    }, &ml[0][0][0], 32, [&](int gr, int c, float4& acc) {
        if (odd) tree_not_finite(a, vbase, gr, c, before, max(before / KT, t0) * KT, min(L, tile_end * KT), acc);
    });
}

// Much work: a workgroup takes 128 rows, 32 a wave, and two groups of four waves take every other tile of
// 64 keys. A group's tiles go through a ring of two in LDS that its waves read in common; the next tile is
// requested before a tile is multiplied. A step takes 2.1 us, of which the matrix instructions need 0.93 (32 cycles
// each, two waves a SIMD) and the exponentials and sums about as much; keeping the groups half a step apart, or letting
// each run on without the other, made it no faster (30 -> 31 to 33 us for 33 nodes at 32000 rows).
template <int HD>
__global__ __launch_bounds__(512, 2) void tree_rows_kernel(TreeArgs a) {
    typedef SplitTile<HD> T;
    constexpr int KT = 64, KS = HD / 16, DT = HD / 32, CPR = HD / 4;
    constexpr int TILE = KT * T::kRow, STAGE = 2 * TILE, RING = 2 * STAGE;   // bytes: keys or values; both; a group's ring
    constexpr int NL = TILE / 1024 / 4;                                      // loads of a wave: keys, and as many of values
    static_assert(DT % 2 == 0 && 8 * DT / 2 * 4 * 1024 <= 2 * RING, "half of the outputs fits in the rings");
    __shared__ __align__(1024) unsigned char smem[2 * RING];
    __shared__ float ml[2][2][128];
    __shared__ int s_odd;

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave, grp = wave / 4, wg = wave % 4;
    const int ql = lane % 32, hh = lane / 32;
    int kvh, split, block;
    if (!tree_place(a, kvh, split, block)) return;
    const int r0 = block * 128, row = min(r0 + wg * 32 + ql, a.rows - 1), node = row / a.G, head = kvh * a.G + row % a.G;
    const bool idle = r0 + wg * 32 >= a.rows;   // a wave without rows helps to load

    const char* const kbase = reinterpret_cast<const char*>(a.k + kvh * a.k_sh);
    const char* const vbase = reinterpret_cast<const char*>(a.v + kvh * a.v_sh);
    unsigned char* const ring = smem + grp * RING;
    // Loads of a wave: rows (4 i + wg) kRows + pr of a tile, the chunk that belongs at its place, which is the same
    // in all of them: one offset a lane serves.
    const int pr = lane / T::kChunks, pc = lane % T::kChunks, row0 = wg * T::kRows + pr;
    static_assert(4 * T::kRows % 16 == 0, "the swizzles repeat after 16 rows");
    const uint32_t koff0 = (uint32_t)(row0 * a.k_sn * 2 + ((pc ^ T::k_swz(row0)) << 4));
    const uint32_t voff0 = (uint32_t)(row0 * a.v_sn * 2 + ((pc ^ T::v_swz(row0)) << 4));
    const int bound = a.bound, t0 = split * a.split_tiles;
    auto issue = [&](int t, int slot) {
        const int k0 = t * KT;
        unsigned char* const dst = ring + slot * STAGE + wg * 1024;
        if (k0 + KT <= bound) {
            const char* const kt = kbase + (int64_t)k0 * a.k_sn * 2;
            const char* const vt = vbase + (int64_t)k0 * a.v_sn * 2;
#pragma unroll
            for (int i = 0; i < NL; ++i)
                __builtin_amdgcn_global_load_lds(static_cast<const void*>(kt + (int64_t)i * 4 * T::kRows * a.k_sn * 2 + koff0),
                                                 (__attribute__((address_space(3))) void*)(dst + i * 4096), 16, 0, 0);
#pragma unroll
            for (int i = 0; i < NL; ++i)
                __builtin_amdgcn_global_load_lds(static_cast<const void*>(vt + (int64_t)i * 4 * T::kRows * a.v_sn * 2 + voff0),
                                                 (__attribute__((address_space(3))) void*)(dst + TILE + i * 4096), 16, 0, 0);
            return;
        }
#pragma unroll
        for (int i = 0; i < 2 * NL; ++i) {   // rows past the end read the last row
            const bool is_v = i >= NL;
            const int rr = (i % NL) * 4 * T::kRows + row0, r = min(rr, bound - 1 - k0);
            const int c = pc ^ (is_v ? T::v_swz(rr) : T::k_swz(rr));
            const int sn = is_v ? a.v_sn : a.k_sn;
            const char* const src = (is_v ? vbase : kbase) + (int64_t)k0 * sn * 2 + (uint32_t)((r * sn + c * 8) * 2);
            __builtin_amdgcn_global_load_lds(static_cast<const void*>(src),
                                             (__attribute__((address_space(3))) void*)(dst + (is_v ? TILE : 0) + (i % NL) * 4096), 16, 0, 0);
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
    // The first tile is requested before the length is known: the cache holds `bound` rows.
    if (t0 + grp < min((bound + KT - 1) / KT, t0 + a.split_tiles)) issue(t0 + grp, 0);
    const int L = tree_len(a), before = L - a.n;   // rows before the tree
    const int tile_end = min((L + KT - 1) / KT, t0 + a.split_tiles);
    const int steps = tile_end > t0 ? (tile_end - t0 + 1) / 2 : 0;
    if (tid == 0) s_odd = 0;
    // Q has landed here: a first use in the loop would wait for every load under way, each time
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
    f32x16_t oacc[DT];
#pragma unroll
    for (int tt = 0; tt < DT; ++tt)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[tt][e] = 0.f;
    float m_run = -INFINITY, l_part = 0.f;   // the largest score so far; the sum over the lane's half of the keys
    const uint64_t* const bits_row = a.mask + (int64_t)node * a.words;
    const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)ring);
    uint32_t koff[KS], voff[DT];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) koff[ks] = lds + (uint32_t)(ql * T::kRow + (((ks * 2 + hh) ^ T::k_swz(ql)) << 4));
    {
        const int g = lane >> 4, j = lane & 15, rr = (g >> 1) * 4 + (j >> 2);
#pragma unroll
        for (int tt = 0; tt < DT; ++tt) {
            const int d = tt * 32 + 16 * (g & 1) + 4 * (j & 3);
            voff[tt] = lds + (uint32_t)(TILE + rr * T::kRow + (((d >> 3) ^ T::v_swz(rr)) << 4) + ((d & 7) << 1));
        }
    }
    const float lazy = kTreeLazy / a.scale;
    auto meet = [] {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    TreeBits window = {};
    if (steps > 0 && (t0 + grp) * KT + KT > before) window.request(bits_row, a.words, (t0 + grp) * KT - before);
    for (int st = 0; st < steps; ++st) {
        const int t = t0 + 2 * st + grp, kb0 = t * KT;
        const bool on = t < tile_end, masked = kb0 + KT > before;
        // whether either group's tile is of the tree's rows: the same in every wave
        const bool clean = (t0 + 2 * st + 1) * KT + KT > before;
        attn_pipe::vm_wait<0>();
        uint64_t bits = ~0ull;
        if (on && masked) {
            bits = window.get(a.words, kb0 - before);
            if (L - kb0 < 64) bits &= (1ull << (L - kb0)) - 1;
        }
        meet();   // the tile is there, and the other slot is read out
        if (clean) {
            // values that are not finite are made zeros, and added at the end where they are seen; a quarter a wave
            if (on && masked) {
                uint4* const vp = reinterpret_cast<uint4*>(ring + (st & 1) * STAGE + TILE);
                uint4 x[NL];
                TreeOdd look;
#pragma unroll
                for (int i = 0; i < NL; ++i) {
                    x[i] = vp[(i * 4 + wg) * 64 + lane];
                    look.look(x[i].x), look.look(x[i].y), look.look(x[i].z), look.look(x[i].w);
                }
                if (look.any()) {   // of rows past the end: zeros, and nothing to add
                    TreeOdd seen;
#pragma unroll
                    for (int i = 0; i < NL; ++i) {
                        if (i * 4 * T::kRows + row0 >= L - kb0) x[i] = make_uint4(0, 0, 0, 0);
                        seen.look(x[i].x), seen.look(x[i].y), seen.look(x[i].z), seen.look(x[i].w);
                    }
                    if (seen.any() && lane == 0) s_odd = 1;
#pragma unroll
                    for (int i = 0; i < NL; ++i)
                        vp[(i * 4 + wg) * 64 + lane] = make_uint4(finite_pair(x[i].x), finite_pair(x[i].y), finite_pair(x[i].z), finite_pair(x[i].w));
                }
            }
            meet();
        }
        if (t + 2 < tile_end) {
            issue(t + 2, (st + 1) & 1);
            if (kb0 + 3 * KT > before) window.request(bits_row, a.words, kb0 + 2 * KT - before);
        }
        if (!on || idle) continue;
        const uint32_t at = (uint32_t)((st & 1) * STAGE);
        // S^T; element e of s[h]: key kb0 + 32 h + 8 (e / 4) + 4 hh + e % 4 of the lane's row
        f32x16_t s[2];
        bf16x8_t kf[2][KS];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (h == 0) attn_pipe::read_b128<0>(kf[h][ks], koff[ks] + at);
                else attn_pipe::read_b128<32 * T::kRow>(kf[h][ks], koff[ks] + at);
            }
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(KS) : "memory");
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(kf[0][ks]));
#pragma unroll
        for (int e = 0; e < 16; ++e) s[0][e] = 0.f, s[1][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[0][ks], qf[ks], s[0], 0, 0, 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(kf[1][ks]));
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[1][ks], qf[ks], s[1], 0, 0, 0);
        tree_s4_t vf[4][DT][2];
        auto read_v = [&](auto kbc) {
            constexpr int kb = decltype(kbc)::value;
#pragma unroll
            for (int tt = 0; tt < DT; ++tt) {
                attn_pipe::read_tr16<(kb * 16) * T::kRow>(vf[kb][tt][0], voff[tt] + at);
                attn_pipe::read_tr16<(kb * 16 + 8) * T::kRow>(vf[kb][tt][1], voff[tt] + at);
            }
        };
        read_v(std::integral_constant<int, 0>{});
        read_v(std::integral_constant<int, 1>{});
        if (masked) {
            const uint64_t mine = bits >> (4 * hh);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[h][e] = tree_masked(s[h][e], (uint32_t)(mine >> (32 * h)), 8 * (e / 4) + e % 4);
        }
        float top = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int e = 1; e < 16; ++e) top = fmaxf(fmaxf(top, s[0][e]), s[1][e]);
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
        Pack8 pb[4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float p[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[h][e], a.scale, -ref));
            pb[2 * h].u = pack8(&p[0]);
            pb[2 * h + 1].u = pack8(&p[8]);
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            l_part = add_bf16_pair(pb[b].u.x, l_part);
            l_part = add_bf16_pair(pb[b].u.y, l_part);
            l_part = add_bf16_pair(pb[b].u.z, l_part);
            l_part = add_bf16_pair(pb[b].u.w, l_part);
        }
        auto pv = [&](int kb) {
#pragma unroll
            for (int tt = 0; tt < DT; ++tt) {
                asm volatile("" : "+v"(vf[kb][tt][0]), "+v"(vf[kb][tt][1]));
                union {
                    tree_s4_t h[2];
                    bf16x8_t v;
                } vv;
                vv.h[0] = vf[kb][tt][0];
                vv.h[1] = vf[kb][tt][1];
                oacc[tt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vv.v, pb[kb].v, oacc[tt], 0, 0, 0);
            }
        };
        // a block's reads go out once the block two before has landed
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(2 * DT) : "memory");
        pv(0);
        read_v(std::integral_constant<int, 2>{});
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(2 * DT) : "memory");
        pv(1);
        read_v(std::integral_constant<int, 3>{});
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(2 * DT) : "memory");
        pv(2);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        pv(3);
    }
    attn_pipe::vm_wait<0>();   // a tile past the length
    // The groups' outputs meet: each joins one half of the channels, and hands the other group's half over in LDS.
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_part), __float_as_uint(l_part), false, false);
    const float l_run = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    meet();
    constexpr int HALF = DT / 2, PARTS = HALF * 4;
    float4* const mine = reinterpret_cast<float4*>(smem + wave * PARTS * 1024) + lane;
    const float4* const other = reinterpret_cast<const float4*>(smem + (wave ^ 4) * PARTS * 1024) + lane;
    tree_each<PARTS>([&](auto ic) {
        constexpr int I = decltype(ic)::value / 4, G = decltype(ic)::value % 4 * 4;
        const f32x16_t& x = grp == 0 ? oacc[HALF + I] : oacc[I];
        mine[decltype(ic)::value * 64] = make_float4(x[G], x[G + 1], x[G + 2], x[G + 3]);
    });
    if (hh == 0) {
        ml[0][grp][wg * 32 + ql] = m_run * a.scale;
        ml[1][grp][wg * 32 + ql] = l_run;
    }
    __syncthreads();
    const float m0 = m_run * a.scale, m1 = ml[0][grp ^ 1][wg * 32 + ql], l1 = ml[1][grp ^ 1][wg * 32 + ql], m = fmaxf(m0, m1);
    const bool any0 = m0 != -INFINITY || l_run != 0.f, any1 = m1 != -INFINITY || l1 != 0.f;   // a group that saw nothing has no part
    const float x0 = any0 ? __builtin_amdgcn_exp2f(m0 - m) : 0.f, x1 = any1 ? __builtin_amdgcn_exp2f(m1 - m) : 0.f;
    const float l = (any0 ? x0 * l_run : 0.f) + (any1 ? x1 * l1 : 0.f);
    const bool odd = s_odd != 0;
    const int gr = r0 + wg * 32 + ql;
    if (gr >= a.rows) return;
    tree_each<PARTS>([&](auto ic) {
        constexpr int I = decltype(ic)::value / 4, G = decltype(ic)::value % 4 * 4;
        const f32x16_t& x = grp == 0 ? oacc[I] : oacc[HALF + I];
        const float4 y = other[decltype(ic)::value * 64];
        const int c = (grp * HALF + I) * 8 + G / 2 + hh;
        float4 acc = make_float4((any0 ? x0 * x[G] : 0.f) + (any1 ? x1 * y.x : 0.f), (any0 ? x0 * x[G + 1] : 0.f) + (any1 ? x1 * y.y : 0.f),
                                 (any0 ? x0 * x[G + 2] : 0.f) + (any1 ? x1 * y.z : 0.f), (any0 ? x0 * x[G + 3] : 0.f) + (any1 ? x1 * y.w : 0.f));
        if (odd) tree_not_finite(a, vbase, gr, c, before, max(before / KT, t0) * KT, min(L, tile_end * KT), acc);
        tree_store<HD>(a, kvh, split, gr, c, m, l, acc, tile_end > t0);
    });
}

// Joins the splits of a row: TPR threads a row, HD / 4 across its channels and P over the splits. The first
// outputs are requested before it is known which splits have any. 4000 rows of 8 splits, 16 MB: 5.0 us.
template <int HD, int TPR>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
    constexpr int C = HD / 4, P = TPR / C, CH = 4, RW = 256 / TPR;
    __shared__ float wt[RW][kTreeMaxSplits];
    __shared__ float4 parts[RW][P][C];
    __shared__ float red[2][4];
    const int64_t all = (int64_t)a.Hkv * a.rows;
    const int rw = threadIdx.x / TPR, tid = threadIdx.x % TPR, c = tid % C, part = tid / C;
    const int64_t r = (int64_t)blockIdx.x * RW + rw, rr = min(r, all - 1);
    const float* const op = a.o_part + rr * HD + c * 4;
    float4 x[CH];
    auto request = [&](int s0) {
#pragma unroll
        for (int k = 0; k < CH; ++k) x[k] = *reinterpret_cast<const float4*>(op + (int64_t)min(s0 + k * P, a.splits - 1) * all * HD);
    };
    request(part);
    constexpr int N = kTreeMaxSplits / TPR;
    float2 mine[N];
#pragma unroll
    for (int i = 0; i < N; ++i) mine[i] = *reinterpret_cast<const float2*>(a.ml_part + ((int64_t)min(i * TPR + tid, a.splits - 1) * all + rr) * 2);
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (i * TPR + tid >= a.splits) mine[i] = make_float2(-INFINITY, 0.f);
        M = fmaxf(M, mine[i].x);
    }
    M = wave_max_uniform(M);
    if constexpr (TPR == 256) {
        if (tid % kWave == 0) red[0][tid / kWave] = M;
        __syncthreads();
        M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    }
    float den = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool used = mine[i].x != -INFINITY || mine[i].y != 0.f;   // the others may have no output
        const float f = used ? __builtin_amdgcn_exp2f(mine[i].x - M) : 0.f;
        den += used ? f * mine[i].y : 0.f;
        wt[rw][i * TPR + tid] = used ? f : -1.f;
    }
    den = wave_total(den);
    if constexpr (TPR == 256) {
        if (tid % kWave == 0) red[1][tid / kWave] = den;
    }
    __syncthreads();
    if constexpr (TPR == 256) den = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = part; s0 < a.splits; s0 += CH * P) {
        if (s0 != part) request(s0);
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const float w = s0 + k * P < a.splits ? wt[rw][s0 + k * P] : -1.f;
            const bool on = !(w < 0.f);
            t.x += on ? w * x[k].x : 0.f, t.y += on ? w * x[k].y : 0.f, t.z += on ? w * x[k].z : 0.f, t.w += on ? w * x[k].w : 0.f;
        }
    }
    parts[rw][part][c] = t;
    __syncthreads();
    if (part > 0 || r >= all) return;
#pragma unroll
    for (int p = 1; p < P; ++p) {
        const float4 y = parts[rw][p][c];
        t.x += y.x, t.y += y.y, t.z += y.z, t.w += y.w;
    }
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

// tree_few_kernel or tree_rows_kernel: the first starts and joins faster and takes masks better, the second reads a tile
// for four times as many rows. With the tiles of 8 KB before the tree that blocks of 32 rows visit, both measured in us:
//   630 (24 nodes, 2000 rows) 10.3 | 13.8    8000 (33, 8000) 20.0 | 22.8       11000 (100, 4000) 23.7 | 25.5
//   15400 (250, 3900) 27.6 | 28.3            15800 (500, 2000) 31.2 | 30.7     16000 (33, 16000) 26.5 | 23.5
//   16000 (1000, 1000) 36.2 | 42.4           16500 (700, 1500) 34.5 | 35.8     31500 (1000, 2000) 47.2 | 48.2
//   32000 (33, 32000) 41.2 | 31.7            head_dim 64: 14000 (1000, 2000) 27.9 | 34.0
// The visits alone do not tell few row blocks over a long context from many over a short one: from 16000 on the second
// is taken for 700 and 1000 nodes too, where it is slower by 2 to 17 %.
// A workgroup a CU, or two where a row block has fewer than four splits, whose join is cheap (250 nodes at 3900 rows
// 39 -> 28 us; 24 nodes at 32000, 25 splits instead of 51, 25 -> 20 us). Up to twelve tiles are not split (five: 6.3 us, in
// two splits 7.8), more into splits of a tile a wave at least (24 nodes at 2003 10.2 us, two tiles a wave 10.8, three 11.4).
static TreePlan tree_plan(const efm_attention_ctx* c, uint32_t n, uint32_t kv_len) {
    const int hd = (int)c->head_dim, Hkv = (int)c->num_kv_heads;
    const int64_t rows = (int64_t)n * (c->num_qo_heads / c->num_kv_heads), cus = prefill_cus();
    TreePlan p = {};
    const int few = hd == 128 ? 32 : 64;   // keys of 8 KB
    p.many = (rows + 31) / 32 * Hkv * (((int64_t)(kv_len - n) + few - 1) / few) >= kTreeMany;
    const int keys = p.many ? 64 : few;
    const int64_t tiles = ((int64_t)kv_len + keys - 1) / keys;
    p.blocks = (int)((rows + (p.many ? 127 : 31)) / (p.many ? 128 : 32));
    const int64_t pairs = (int64_t)p.blocks * Hkv, each = !p.many && cus / pairs < 4 ? 2 : 1;
    const int64_t want = std::max<int64_t>(1, each * cus / pairs);
    p.split_tiles = (int)std::max<int64_t>({tiles <= kTreeWhole ? tiles : kTreeLeast, (tiles + want - 1) / want, (tiles + kTreeMaxSplits - 1) / kTreeMaxSplits});
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
    if (kv_len <= 256) return 0;   // one split in either kernel
    const int64_t splits = std::min<int64_t>(tiles, kTreeMaxSplits);
    const int64_t rows = std::min(splits * n * (int64_t)c->num_qo_heads, 128 * cus);   // 128 rows a workgroup at most
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
    a.bound = (int)bound;
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
    const int64_t all = (int64_t)Hkv * a.rows;
    const dim3 grid((unsigned)(((int64_t)Hkv * p.splits * p.blocks + 7) / 8 * 8));
    auto launch = [&](auto hdc) {
        constexpr int HD = decltype(hdc)::value;
        if (p.many) hipLaunchKernelGGL(tree_rows_kernel<HD>, grid, dim3(512), 0, stream, a);
        else hipLaunchKernelGGL(tree_few_kernel<HD>, grid, dim3(256), 0, stream, a);
        if (p.splits > 8) hipLaunchKernelGGL((tree_merge_kernel<HD, 256>), dim3((unsigned)all), dim3(256), 0, stream, a);
        else if (p.splits > 1) hipLaunchKernelGGL((tree_merge_kernel<HD, 64>), dim3((unsigned)((all + 3) / 4)), dim3(256), 0, stream, a);
    };
    if (hd == 128) launch(std::integral_constant<int, 128>{});
    else launch(std::integral_constant<int, 64>{});
    return check_launch("attention_tree");
}
