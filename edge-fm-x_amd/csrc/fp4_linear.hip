// Linear layers with FP4 weights (fp4.hpp) on gfx950: quantisation and packing of the weights,
// y = x W^T (+ bias) and the fused gate / up projection with SwiGLU.
//
// Packed weights: tiles of 16 rows by blocks of 128 columns, 1 KB each, in the order in which a
// wave's lanes take them as the second operand of v_mfma_f32_16x16x32_bf16: lane l holds, for
// row l % 16, the words of columns 32 w + 8 (l / 16) .. + 7, w = 0..3. One 16-byte load a lane
// feeds the four MFMAs of a block, and a wave's loads are whole contiguous kilobytes. The scale
// bytes follow all tiles, four to a row and block. Rows and columns past the matrix are zero.
#include "attn_pipe.hpp"
#include "fp4.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

namespace efm {

int prefill_cus();

constexpr int kW4Rows = 16, kW4Cols = 128;

struct Fp4Weights {
    const uint8_t* codes;    // [tiles][blocks][64 lanes][16 bytes]
    const uint8_t* scales;   // [tiles][blocks][16 rows][4 bytes]
    int tiles, blocks;
};

static int w4_tiles(int64_t out) { return (int)((out + kW4Rows - 1) / kW4Rows); }
static int w4_blocks(int64_t in) { return (int)((in + kW4Cols - 1) / kW4Cols); }

static size_t w4_code_bytes(int64_t in, int64_t out) { return (size_t)w4_tiles(out) * w4_blocks(in) * 1024; }
static size_t w4_packed_bytes(int64_t in, int64_t out) { return w4_code_bytes(in, out) / 16 * 17; }

static Fp4Weights w4_weights(int64_t in, int64_t out, const void* packed) {
    const uint8_t* p = static_cast<const uint8_t*>(packed);
    return Fp4Weights{p, p + w4_code_bytes(in, out), w4_tiles(out), w4_blocks(in)};
}

// One lane for 8 values, four lanes for a group. Bound by memory: 3584 x 37888 in 61 us (5.6 TB/s).
__global__ __launch_bounds__(256) void fp4_quantize_kernel(const uint4* w, uint32_t* codes, uint8_t* scales, int64_t octets) {
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < octets; i += gridDim.x * 256ll) {   // octets % 4 == 0
        float x[8];
        unpack8(w[i], x);
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
        top = max(top, (uint32_t)__shfl_xor((int)top, 1, kWave));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2, kWave));
        const uint32_t byte = fp4_scale_byte(top);
        codes[i] = fp4_encode8(x, byte);
        if (i % 4 == 0) scales[i / 4] = (uint8_t)byte;
    }
}

// One wave for a tile's block. Its lanes gather words of 16 rows, a row's length apart: 3584 x 37888 in 54 to 61
// us (2.5 TB/s read and written), once, as the weights are loaded.
__global__ __launch_bounds__(256) void fp4_pack_kernel(const uint8_t* codes, const uint8_t* scales, uint4* out_codes,
                                                       uint32_t* out_scales, int64_t in, int64_t out, int blocks,
                                                       int64_t total) {
    const int lane = threadIdx.x % kWave, g = lane / 16;
    for (int64_t t = blockIdx.x * 4ll + threadIdx.x / kWave; t < total; t += gridDim.x * 4ll) {
        const int64_t row = t / blocks * kW4Rows + lane % 16, col = t % blocks * kW4Cols;
        uint32_t w[4] = {0, 0, 0, 0}, s = 0;
        if (row < out) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (col + 32 * i >= in) break;
                w[i] = *reinterpret_cast<const uint32_t*>(codes + (row * in + col + 32 * i + 8 * g) / 2);
                s |= (uint32_t)scales[(row * in + col) / 32 + i] << (8 * i);
            }
        }
        out_codes[t * 64 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
        if (lane < 16) out_scales[t * 16 + lane] = s;
    }
}

enum { W4_BF16 = 0, W4_F32 = 1, W4_SWIGLU = 2 };

struct W4Args {
    const bf16_t* x;
    Fp4Weights w;
    const bf16_t* bias;
    void* y;
    int64_t M, N, K;   // N: columns of y
};

// Four consecutive columns of a row of y, `left` of them inside the matrix. Whole fours go as one
// store whatever their alignment, which the hardware takes.
template <bool F32>
__device__ __forceinline__ void w4_store4(void* y, int64_t at, const float* v, int64_t left) {
    if constexpr (F32) {
        float* o = static_cast<float*>(y) + at;
        if (left >= 4) {
            __builtin_memcpy(o, v, 16);
        } else {
            for (int e = 0; e < left; ++e) o[e] = v[e];
        }
    } else {
        bf16_t* o = static_cast<bf16_t*>(y) + at;
        if (left >= 4) {
            const uint2 p = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
            __builtin_memcpy(o, &p, 8);
        } else {
            for (int e = 0; e < left; ++e) o[e] = (bf16_t)f32_to_bf16(v[e]);
        }
    }
}

// One to four rows of x, bound by the stream of the weights: a workgroup takes NT tiles of weight rows
// (SwiGLU: NT / 2 tiles of up and the NT / 2 of gate beside them); its waves take every KW-th block of
// K each and add their sums through LDS in the order of the waves. A wave has P blocks of codes and
// scales under way in registers. x sits in LDS where it fits (XLDS), since 64 lanes that ask for the
// same few bytes of it cost the address unit as much as 64 that ask for codes (1 x 18944 -> 3584 9.2 us
// against 13.3, 1 x 3584 -> 2 x 18944 SwiGLU 13.5 against 15.0).
template <int NT, int P, int EPI, bool XLDS>
__global__ __launch_bounds__(1024) void fp4_linear_kernel(W4Args a) {
    extern __shared__ __align__(16) float red[];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), KW = blockDim.x / kWave;
    const int g = lane / 16, l = lane % 16;
    const int half = a.w.tiles / 2;
    const uint8_t* wp[NT];
    const uint8_t* sp[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int tile = EPI == W4_SWIGLU ? min((int)blockIdx.x * (NT / 2) + j % (NT / 2), half - 1) + (j < NT / 2 ? 0 : half)
                                          : min((int)blockIdx.x * NT + j, a.w.tiles - 1);
        wp[j] = a.w.codes + (size_t)tile * a.w.blocks * 1024 + lane * 16;
        sp[j] = a.w.scales + (size_t)tile * a.w.blocks * 64 + l * 4;
    }
    // not in LDS: rows past the last, and columns past the last row's, are asked for past the buffer's end and
    // come as zeros. All of the offset is in the lane's register, since a scalar offset is outside the check
    // of that end.
    const __amdgpu_buffer_rsrc_t xb =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(a.x), (short)0, (int)(a.M * a.K * 2), 0x00020000);
    const uint32_t xo = l < a.M ? (uint32_t)(l * a.K + 8 * g) * 2 : 0x80000000u;
    // in LDS, behind the sums: row r at r * (K + 8) values, so that the rows' reads meet different banks
    unsigned char* const xl = reinterpret_cast<unsigned char*>(red) + (size_t)KW * NT * 1024;
    const unsigned char* const xr = xl + (l < a.M ? l : 0) * (a.K * 2 + 16) + 16 * g;
    auto stage_x = [&]() {
        const int per = (int)(a.K / 8);
        for (int i = threadIdx.x; i < (int)a.M * per; i += blockDim.x) {
            const int r = i / per, c = i % per;
            *reinterpret_cast<uint4*>(xl + r * (a.K * 2 + 16) + c * 16) = reinterpret_cast<const uint4*>(a.x + r * a.K)[c];
        }
        __syncthreads();
    };
    f32x4_t acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
    uint4 w[P][NT];
    u32x4_t x[P][4];
    uint32_t s[P][NT];
    auto load = [&](int st, int b) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            w[st][j] = load_stream16(wp[j] + (size_t)b * 1024);
            s[st][j] = *reinterpret_cast<const uint32_t*>(sp[j] + (size_t)b * 64);
        }
        if constexpr (!XLDS) {
#pragma unroll
            for (int q = 0; q < 4; ++q) x[st][q] = __builtin_amdgcn_raw_buffer_load_b128(xb, (int)(xo + (b * kW4Cols + 32 * q) * 2), 0, 0);
        }
    };
    auto multiply = [&](int st, int b) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if ((int64_t)b * kW4Cols + 32 * q >= a.K) break;
            bf16x8_t xf;
            if constexpr (XLDS) xf = *reinterpret_cast<const bf16x8_t*>(xr + (b * kW4Cols + 32 * q) * 2);
            else xf = __builtin_bit_cast(bf16x8_t, x[st][q]);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const bf16x8_t wf = fp4_unpack8(q == 0 ? w[st][j].x : q == 1 ? w[st][j].y : q == 2 ? w[st][j].z : w[st][j].w,
                                                fp4_scale_at(s[st][j], q));
                acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, wf, acc[j], 0, 0, 0);
            }
        }
    };
    // the wave's blocks: wave, wave + KW, ...; n of them
    const int n = wave < a.w.blocks ? (a.w.blocks - 1 - wave) / KW + 1 : 0;
    auto block = [&](int i) { return wave + i * KW; };
    if (n >= P) {
#pragma unroll
        for (int st = 0; st < P; ++st) load(st, block(st));
    }
    if constexpr (XLDS) stage_x();
    if (n >= P) {
        int i = 0;
        for (; i + 2 * P <= n; i += P)
#pragma unroll
            for (int st = 0; st < P; ++st) {
                multiply(st, block(i + st));
                load(st, block(i + st + P));
            }
#pragma unroll
        for (int st = 0; st < P; ++st) {
            multiply(st, block(i + st));
            if (i + P + st < n) load(st, block(i + P + st));
        }
#pragma unroll
        for (int st = 0; st + 1 < P; ++st)
            if (i + P + st < n) multiply(st, block(i + P + st));
    } else {
        for (int i = 0; i < n; ++i) {
            load(0, block(i));
            multiply(0, block(i));
        }
    }
    f32x4_t* const part = reinterpret_cast<f32x4_t*>(red);
#pragma unroll
    for (int j = 0; j < NT; ++j) part[(wave * NT + j) * kWave + lane] = acc[j];
    __syncthreads();
    constexpr int NO = EPI == W4_SWIGLU ? NT / 2 : NT;   // column tiles of y
    for (int e = threadIdx.x; e < NO * 16 * (int)a.M; e += blockDim.x) {
        const int n16 = e % 16, j = e / 16 % NO, m = e / 16 / NO;   // m < 4: row m of the first four
        const int64_t col = ((int64_t)blockIdx.x * NO + j) * 16 + n16;
        if (col >= a.N) continue;
        auto total = [&](int jj) {
            float t = 0.f;
            for (int k = 0; k < KW; ++k) t += red[((k * NT + jj) * kWave + n16) * 4 + m];
            return t;
        };
        const int64_t at = m * a.N + col;
        if constexpr (EPI == W4_SWIGLU) {
            const float u = round_bf16(total(j)), gate = round_bf16(total(j + NO));
            static_cast<bf16_t*>(a.y)[at] = (bf16_t)f32_to_bf16(silu_f32(gate) * u);
        } else {
            const float t = total(j) + (a.bias != nullptr ? bf16_to_f32(a.bias[col]) : 0.f);
            if constexpr (EPI == W4_F32) static_cast<float*>(a.y)[at] = t;
            else static_cast<bf16_t*>(a.y)[at] = (bf16_t)f32_to_bf16(t);
        }
    }
}

// Five rows of x and more: KG groups, each with a part of K, of WN waves that share 16 TM rows of x and take
// 16 TN weight rows each; a group of one wave meets no barrier. x, 64 columns (a slab) at a time, and the
// codes and scales, 128 columns (a block) at a time, go straight into rings of D and R places in LDS,
// D - 1 slabs ahead. In LDS the 16-byte chunk c of a row r of x
// sits at c ^ (r / 2 % 8), so that sixteen rows' reads meet all banks. The weights are the first
// operand: a lane ends with four consecutive columns of a row of y.
constexpr int w4_swz(int r) { return (r >> 1) & 7; }

// 16 bytes a lane from base + off, off a lane's own, into consecutive places at dst; zeros past `bytes`. The
// scalar offset of the load stays 0: it is outside the check of that end.
__device__ __forceinline__ void w4_dma16(const void* base, uint32_t bytes, uint32_t off, void* dst) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)dst, 16, (int)off, 0, 0, 0);
}
// 4 bytes a lane.
__device__ __forceinline__ void w4_dma4(const void* src, void* dst) {
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)dst, 4, 0, 0);
}
template <int IMM>
__device__ __forceinline__ void w4_read32(uint32_t& dst, uint32_t addr) {
    asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(dst) : "v"(addr), "n"(IMM) : "memory");
}

// LDS of a group: D slabs of x, (D + 1) / 2 blocks of codes and scales.
constexpr int kW4Ring = 3;
constexpr int w4_tile_lds(int tm, int tn, int wn) {
    return kW4Ring * 2048 * tm + (kW4Ring + 1) / 2 * (1024 * wn * tn + 256 * wn);
}
// Waves a SIMD to compile for: two while two workgroups of four waves fit LDS.
constexpr int w4_tile_waves(int tm, int tn, int wn, int kg) {
    return wn * kg > 4 ? wn * kg / 4 : w4_tile_lds(tm, tn, wn) * kg <= 80 * 1024 && tm * tn <= 16 ? 2 : 1;
}

template <int TM, int TN, int WN, int KG, int EPI>
__global__ __launch_bounds__(64 * WN * KG, w4_tile_waves(TM, TN, WN, KG)) void fp4_linear_tile_kernel(W4Args a, int mt, int nt) {
    constexpr int D = kW4Ring, NW = WN, BM = 16 * TM;   // NW: waves of a group
    constexpr int XS = BM * 128, WS = WN * TN * 1024;   // bytes of a slab of x, of a block of codes
    constexpr int LX = XS / 1024 / NW, LW = TN;         // 1 KB loads of x a wave and slab; tiles whose codes a wave fetches
    constexpr int NO = EPI == W4_SWIGLU ? TN / 2 : TN;  // column tiles of y a wave
    constexpr int R = (D + 1) / 2;                      // blocks of codes in their ring
    constexpr int W0 = D * XS, S0 = W0 + R * WS;
    // loads that may be under way behind the barrier of an even and of an odd slab
    constexpr int AHEAD0 = (D - 2) * LX + (D - 1) / 2 * (LW + 1), AHEAD1 = (D - 2) * LX + (D - 2) / 2 * (LW + 1);
    static_assert(D >= 3 && XS % (1024 * NW) == 0 && LW <= 4 && AHEAD0 < 64, "the waits below count these loads");
    constexpr int SS = 256 * NW, GS = S0 + R * SS;       // scales of a block; LDS of a group
    static_assert(KG == 1 || (KG - 1) * NW * TM * TN * 1024 <= KG * GS, "the groups' sums fit where their rings were");
    __shared__ __align__(1024) unsigned char smem_all[KG * GS];
    // consecutive workgroups of an XCD (one L2) share rows of weights and sweep x
    const int total = mt * nt, per = (total + 7) / 8;
    const int t = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if (t >= total) return;
    const int64_t m0 = (int64_t)(t % mt) * BM;
    const int nb = t / mt;
    const int wave4 = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), wave = wave4 % NW, grp = wave4 / NW, lane = threadIdx.x % kWave;
    const int l = lane % 16, g = lane / 16;
    const int half = a.w.tiles / 2;
    // the group's blocks and slabs: a KG-th of K
    const int gb = (a.w.blocks + KG - 1) / KG, blk0 = grp * gb, sl0 = 2 * blk0;
    const int all_slabs = (int)((a.K + 63) / 64), slabs = min(2 * gb, all_slabs - sl0);
    unsigned char* const smem = smem_all + grp * GS;
    // weight tile u of the workgroup: u / TN is the wave's column, u % TN its tile there
    auto tile = [&](int u) {
        const int c = (nb * WN + u / TN) * NO, j = u % TN;
        return EPI == W4_SWIGLU ? min(c + j % NO, half - 1) + (j < NO ? 0 : half) : min(c + j, a.w.tiles - 1);
    };
    const uint8_t* wp[LW];
#pragma unroll
    for (int i = 0; i < LW; ++i) wp[i] = a.w.codes + (size_t)tile(wave * LW + i) * a.w.blocks * 1024;
    const uint8_t* const sp = a.w.scales + (size_t)tile(wave * LW + lane / 16 % LW) * a.w.blocks * 64 + l * 4;
    // x: rows past the last repeat it. A last slab of 32 columns reads past its rows' ends, inside x or
    // as zeros past its end; nothing multiplies what it reads there.
    const unsigned char* const xbase = reinterpret_cast<const unsigned char*>(a.x + m0 * a.K);
    const uint32_t xbytes = (uint32_t)min((a.M - m0) * a.K * 2, (int64_t)0x7fffffff);
    uint32_t xv[LX];
#pragma unroll
    for (int i = 0; i < LX; ++i) {
        const int r = (i * NW + wave) * 8 + lane / 8;
        xv[i] = (uint32_t)(min((int64_t)r, a.M - 1 - m0) * a.K * 2 + (((lane % 8) ^ w4_swz(r)) << 4));
    }
    // loads past the end repeat the last slab and block into places that nothing reads
    auto load_x = [&](int slab, int i) {
        w4_dma16(xbase, xbytes, xv[i] + (uint32_t)min(sl0 + slab, all_slabs - 1) * 128, smem + slab % D * XS + (i * NW + wave) * 1024);
    };
    auto load_w = [&](int b, int i) {
        const size_t at = (size_t)min(blk0 + b, a.w.blocks - 1);
        if (i < LW)
            w4_dma16(wp[i < LW ? i : 0] + at * 1024, 1024, lane * 16, smem + W0 + b % R * WS + (wave * LW + i) * 1024);
        else
            w4_dma4(sp + at * 64, smem + S0 + b % R * SS + wave * 256);
    };
    const uint32_t lds = (uint32_t)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) unsigned char*)smem);
    uint32_t xa[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) xa[q] = lds + (uint32_t)(l * 128 + (((q * 4 + g) ^ w4_swz(l)) << 4));
    const uint32_t wa = lds + (uint32_t)(W0 + wave * TN * 1024 + lane * 16);
    const uint32_t sa = lds + (uint32_t)(S0 + wave * 256 + l * 4);   // tile j: its loader's place, 64 (j % LW) on

    f32x4_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
    u32x4_t w[2][TN];    // codes and scales of a block, in registers one slab before they are needed
    uint32_t s[2][TN], sc[TN];
    bf16x8_t xf[2][TM];
    u32x4_t wf[2][TN];
    auto read_x = [&](auto ic, auto qc, uint32_t at) {
        constexpr int I = decltype(ic)::value, Q = decltype(qc)::value;
        if constexpr (I < TM) attn_pipe::read_b128<I * 2048>(xf[Q][I], xa[Q] + at);
    };
    auto read_w = [&](auto jc, auto bc, uint32_t b) {
        constexpr int J = decltype(jc)::value, B = decltype(bc)::value;
        if constexpr (J >= 0 && J < TN) {
            attn_pipe::read_b128<J * 1024>(w[B][J], wa + b * WS);
            w4_read32<J / LW * 256 + J % LW * 64>(s[B][J], sa + b * SS);
        }
    };
    auto landed = [&]() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
    auto tie_x = [&](int q) {
#pragma unroll
        for (int i = 0; i < TM; ++i) asm volatile("" : "+v"(xf[q][i]));
    };
    auto tie_w = [&](int b) {
#pragma unroll
        for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(w[b][j]), "+v"(s[b][j]));
    };
    // Unpacking of word I of the codes in w[B] into wf[Q], in 5 TN instructions: piece P is the scale
    // (P % 5 == 0) of tile P / 5 or two of its values. The conversion takes the scale's exponent
    // bits alone, so the other scales of the word need not be cleared.
    auto unpack = [&](auto pc, auto bc, auto ic, auto qc) {
        constexpr int P = decltype(pc)::value, B = decltype(bc)::value, I = decltype(ic)::value, Q = decltype(qc)::value;
        if constexpr (P < 5 * TN) {
            constexpr int J = P / 5, E = P % 5 - 1;
            if constexpr (E < 0) {
                sc[J] = I < 3 ? s[B][J] << (23 - 8 * I) : s[B][J] >> 1;
                asm volatile("" : "+v"(sc[J]));
            } else {
                uint32_t v = fp4_pair<E>(w[B][J][I], __uint_as_float(sc[J]));
                asm volatile("" : "+v"(v));   // here, not beside its use
                wf[Q][J][E] = v;
            }
        }
    };
    // the MFMAs of a 32-column step; `beside(I)` is what goes out behind MFMA I
    constexpr int NM = TM * TN;
    auto step = [&](auto qc, auto&& beside) {
        constexpr int Q = decltype(qc)::value;
        [&]<int... I>(std::integer_sequence<int, I...>) {
            ((acc[I / TN][I % TN] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, wf[Q][I % TN]), xf[Q][I / TN],
                                                                            acc[I / TN][I % TN], 0, 0, 0),
              beside(std::integral_constant<int, I>{}), __builtin_amdgcn_sched_barrier(0)),
             ...);
        }(std::make_integer_sequence<int, TM * TN>{});
    };
    // pieces P of `n` that go out behind MFMA I when they are spread over the step
    auto spread = [&](auto ic, auto nc, auto&& f) {
        constexpr int I = decltype(ic)::value, N = decltype(nc)::value, P0 = (I * N + NM - 1) / NM, P1 = ((I + 1) * N + NM - 1) / NM;
        [&]<int... P>(std::integer_sequence<int, P...>) { (f(std::integral_constant<int, P0 + P>{}), ...); }
        (std::make_integer_sequence<int, P1 - P0>{});
    };
    constexpr std::integral_constant<int, 0> c0{};
    constexpr std::integral_constant<int, 1> c1{};
    constexpr std::integral_constant<int, 5 * TN> pieces{};
    auto load_block = [&](int b) {
#pragma unroll
        for (int i = 0; i <= LW; ++i) load_w(b, i);
    };
    // as if slabs -(D - 1) to -1 had sent them
    load_block(0);
#pragma unroll
    for (int v = 1 - D; v < 0; ++v) {
        if (v % 2 == 0) load_block(v / 2 + R);
#pragma unroll
        for (int i = 0; i < LX; ++i) load_x(v + D - 1, i);
    }
    auto meet = [&]() {   // the waves of a group; one alone has nobody to wait for
        asm volatile("" ::: "memory");
        if constexpr (NW > 1) __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    attn_pipe::vm_wait<AHEAD1>();
    meet();
    [&]<int... I>(std::integer_sequence<int, I...>) {
        (read_x(std::integral_constant<int, I>{}, c0, 0u), ...);
        (read_w(std::integral_constant<int, I>{}, c0, 0u), ...);
    }(std::make_integer_sequence<int, (TM > TN ? TM : TN)>{});
    landed();
    tie_w(0);
    meet();   // block 0's place is refilled from here on
    load_block(R);
    [&]<int... P>(std::integer_sequence<int, P...>) {
        (unpack(std::integral_constant<int, P>{}, c0, c0, c0), ...);
    }(std::make_integer_sequence<int, 5 * TN>{});

    // Slab sl, the half H of block sl / 2, whose codes are in w[B]. Step 0 runs with the reads of
    // step 1, the unpacking for it, the loads of x D - 1 slabs ahead into the place of slab sl - 1
    // and, in a block's second half, the reads of the next block's codes; then the barrier: this
    // slab is in registers everywhere and the next one has landed; step 1 runs with the reads and
    // the unpacking for the next slab's step 0 and, in the second half, the loads of the codes R
    // blocks ahead of the next block into its place.
    auto slab_step = [&](int sl, auto hc, auto bc) {
        constexpr int H = decltype(hc)::value, B = decltype(bc)::value;
        constexpr std::integral_constant<int, 1 - B> other{};
        constexpr std::integral_constant<int, (H == 0 ? B : 1 - B)> next{};
        const uint32_t xo = (uint32_t)(sl % D * XS), xn = (uint32_t)((sl + 1) % D * XS), bn = (uint32_t)((sl / 2 + 1) % R);
        landed();
        tie_x(0);
        step(c0, [&](auto ic) {
            constexpr int I = decltype(ic)::value;
            read_x(ic, c1, xo);
            if constexpr (H == 1) read_w(ic, other, bn);
            spread(ic, pieces, [&](auto pc) { unpack(pc, bc, std::integral_constant<int, 2 * H + 1>{}, c1); });
            spread(ic, std::integral_constant<int, LX>{}, [&](auto pc) { load_x(sl + D - 1, decltype(pc)::value); });
        });
        landed();
        tie_x(1);
        if constexpr (H == 1) tie_w(1 - B);
        attn_pipe::vm_wait<(H == 0 ? AHEAD0 : AHEAD1)>();
        meet();
        if ((int64_t)(sl0 + sl) * 64 + 32 >= a.K) return;
        step(c1, [&](auto ic) {
            constexpr int I = decltype(ic)::value;
            read_x(ic, c0, xn);
            spread(ic, pieces, [&](auto pc) { unpack(pc, next, std::integral_constant<int, (H == 0 ? 2 : 0)>{}, c0); });
            if constexpr (H == 1)
                spread(ic, std::integral_constant<int, LW + 1>{}, [&](auto pc) { load_w(sl / 2 + 1 + R, decltype(pc)::value); });
        });
    };
    auto part = [&](int sl, auto hc, auto bc) {
        if (sl < slabs) slab_step(sl, hc, bc);
        else if (KG > 1 && sl < 2 * gb) meet();   // the other groups' slabs
    };
    for (int sl = 0; sl < (KG > 1 ? 2 * gb : slabs); sl += 4) {
        part(sl, c0, c0);
        part(sl + 1, c1, c0);
        part(sl + 2, c0, c1);
        part(sl + 3, c1, c1);
    }
    const int ct0 = (nb * WN + wave) * NO;   // first column tile of y
    float bias[NO][4] = {};                // all requested at once
    if (EPI != W4_SWIGLU && a.bias != nullptr) {
#pragma unroll
        for (int j = 0; j < NO; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) bias[j][e] = bf16_to_f32(a.bias[min((int64_t)(ct0 + j) * 16 + 4 * g + e, a.N - 1)]);
    }
    landed();
    tie_x(0);
    attn_pipe::vm_wait<0>();
    if constexpr (KG > 1) {
        // the groups' sums in their order
        f32x4_t* const sums = reinterpret_cast<f32x4_t*>(smem_all);
        auto at = [&](int gr, int i, int j) { return (((gr - 1) * NW + wave) * TM * TN + i * TN + j) * kWave + lane; };
        __syncthreads();
        if (grp > 0) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) sums[at(grp, i, j)] = acc[i][j];
        }
        __syncthreads();
        if (grp > 0) return;
#pragma unroll
        for (int gr = 1; gr < KG; ++gr)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] += sums[at(gr, i, j)];
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int64_t row = m0 + i * 16 + l;
        if (row >= a.M) continue;
#pragma unroll
        for (int j = 0; j < NO; ++j) {
            const int64_t col = (int64_t)(ct0 + j) * 16 + 4 * g;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (EPI == W4_SWIGLU) v[e] = silu_f32(round_bf16(acc[i][j + NO][e])) * round_bf16(acc[i][j][e]);
                else v[e] = acc[i][j][e] + bias[j][e];
            }
            w4_store4<EPI == W4_F32>(a.y, row * a.N + col, v, a.N - col);
        }
    }
}

static int w4_check(const char* who, int64_t in, int64_t out) {
    if (in <= 0 || out <= 0)
        return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: bad shape in=%lld out=%lld", who, (long long)in, (long long)out);
    if (in % kFp4Group != 0)
        return set_error(EFM_ERR_UNSUPPORTED, "%s: in_features must be a multiple of 32 (got %lld)", who, (long long)in);
    if (in > (1 << 20) || out > (1 << 24))
        return set_error(EFM_ERR_UNSUPPORTED, "%s: shape too large (in=%lld out=%lld)", who, (long long)in, (long long)out);
    return EFM_OK;
}

static bool w4_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr int kW4FewRows = 4;

// Waves of a workgroup: 16 while it is alone on its CU, else 8, and no more than blocks of K. One tile
// of weight rows each (SwiGLU: one of up and one of gate), two where there are thousands (152064 x
// 3584: 46 us, 60 with one). Two blocks under way where a wave has three or more to go, and always where
// x is outside LDS, from 48 blocks on; SwiGLU's sums of two tiles a wave put x outside from 32 on, where
// 16 waves have one under way.
template <int EPI>
static void w4_launch_few(const W4Args& a, int cus, hipStream_t stream) {
    const int half = EPI == W4_SWIGLU ? 2 : 1;
    const bool wide = EPI != W4_SWIGLU && a.w.tiles >= 16 * cus;
    const int nt = wide ? 2 : half, groups = (a.w.tiles / half + (wide ? 1 : 0)) / (wide ? 2 : 1);
    int kw = groups <= 2 * cus ? 16 : 8;
    while (kw > 1 && kw / 2 >= a.w.blocks) kw /= 2;
    const size_t sums = (size_t)kw * nt * 1024, x = (size_t)a.M * (a.K * 2 + 16);
    const bool xlds = sums + x <= 64 * 1024;
    const bool two = a.w.blocks >= 3 * kw || (EPI != W4_SWIGLU && !xlds);
    auto go = [&](auto ntc, auto pc, auto xc) {
        constexpr int NT = decltype(ntc)::value, P = decltype(pc)::value;
        if (nt != NT || two != (P == 2) || xlds != decltype(xc)::value) return;
        hipLaunchKernelGGL((fp4_linear_kernel<NT, P, EPI, decltype(xc)::value>), dim3(groups), dim3(kw * kWave),
                           sums + (xlds ? x : 0), stream, a);
    };
    using std::integral_constant;
    auto each = [&](auto ntc) {
        go(ntc, integral_constant<int, 1>{}, std::true_type{});
        go(ntc, integral_constant<int, 2>{}, std::true_type{});
        if constexpr (EPI == W4_SWIGLU) go(ntc, integral_constant<int, 1>{}, std::false_type{});
        go(ntc, integral_constant<int, 2>{}, std::false_type{});
    };
    if constexpr (EPI != W4_SWIGLU) each(integral_constant<int, 1>{});
    each(integral_constant<int, 2>{});
}

// The forms of the tile kernel, and what a launch of each takes in us, fitted to sweeps of 1 to 4096
// rows over the projections of the models' dimensions on 256 CUs: fixed + per_group * x + slabs *
// max(alone * rounds, full * x), x the workgroups that the busiest CU has (their mean and its ceiling,
// weighted), rounds = x / resident, slabs those that one group of waves walks. The form that it picks
// is 0.7 % off the best of them over the sweeps.
struct W4Form {
    int tm, tn, wn, kg, resident;
    float alone, full, fixed, per_group, mean;
};
constexpr W4Form kW4Forms[] = {
    // few rows: each wave a part of K and rings of its own
    {1, 1, 1, 8, 2, 0.197f, 0.247f, 2.71f, 0.37f, 0.38f},
    {1, 2, 1, 2, 4, 0.259f, 0.069f, 1.66f, 0.41f, 0.00f},
    {1, 2, 1, 4, 3, 0.238f, 0.153f, 2.29f, 0.54f, 0.25f},
    {1, 2, 1, 8, 1, 0.100f, 0.318f, 1.89f, 1.67f, 0.20f},
    {2, 2, 1, 2, 4, 0.288f, 0.119f, 1.87f, 0.65f, 0.49f},
    {2, 2, 1, 4, 2, 0.304f, 0.235f, 2.14f, 1.07f, 0.45f},
    {2, 2, 1, 8, 1, 0.333f, 0.453f, 2.13f, 2.07f, 0.26f},
    {2, 4, 1, 2, 3, 0.394f, 0.159f, 1.50f, 1.45f, 0.19f},
    // two or four waves beside each other share x, in groups that split K or alone
    {2, 2, 2, 4, 1, 0.331f, 0.390f, 1.50f, 2.30f, 0.15f},
    {2, 2, 4, 2, 2, 0.327f, 0.289f, 2.51f, 1.07f, 0.24f},
    {2, 2, 4, 1, 4, 0.284f, 0.125f, 1.50f, 0.95f, 0.00f},
    {4, 2, 4, 1, 3, 0.290f, 0.252f, 3.21f, 0.62f, 0.51f},
    {6, 2, 4, 1, 2, 0.332f, 0.350f, 3.84f, 0.93f, 0.63f},
    {8, 2, 4, 1, 2, 0.382f, 0.447f, 4.53f, 1.23f, 0.64f},
    {4, 4, 4, 1, 2, 0.420f, 0.393f, 4.26f, 2.01f, 0.45f},
    {6, 4, 4, 1, 2, 0.519f, 0.518f, 4.77f, 2.72f, 0.37f},
};
constexpr int kW4FormCount = sizeof(kW4Forms) / sizeof(kW4Forms[0]);

struct W4Tiles {
    int64_t mt, nt;
};

static W4Tiles w4_tiles_of(const W4Form& f, const W4Args& a, bool swiglu) {
    const int cols = 16 * f.wn * (swiglu ? f.tn / 2 : f.tn), rows = 16 * f.tm;
    return W4Tiles{(a.M + rows - 1) / rows, (a.N + cols - 1) / cols};
}

static int w4_pick(const W4Args& a, bool swiglu, int cus) {
    int best = -1;
    double least = 0;
    for (int i = 0; i < kW4FormCount; ++i) {
        const W4Form& f = kW4Forms[i];
        if (swiglu && f.tn % 2 != 0) continue;
        const W4Tiles t = w4_tiles_of(f, a, swiglu);
        const double load = (double)t.mt * t.nt / cus, x = f.mean * load + (1 - f.mean) * std::ceil(load);
        const double slabs = 2 * ((a.w.blocks + f.kg - 1) / f.kg);
        const double us = f.fixed + f.per_group * x + slabs * std::max(f.alone * std::max(1.0, x / f.resident), f.full * x);
        if (best < 0 || us < least) best = i, least = us;
    }
    return best;
}

// Steps of 64 columns that a wave of the form walks: groups of waves take whole blocks of two.
static int w4_steps(const W4Form& f, int64_t K, int blocks) {
    return f.kg > 1 ? 2 * ((blocks + f.kg - 1) / f.kg) : (int)((K + 63) / 64);
}

template <int EPI>
static int w4_launch(const char* who, const W4Args& a, hipStream_t stream) {
    const int cus = prefill_cus();
    if (a.M <= kW4FewRows) {
        w4_launch_few<EPI>(a, cus, stream);
        return check_launch(who);
    }
    const int pick = w4_pick(a, EPI == W4_SWIGLU, cus);
    const W4Tiles t = w4_tiles_of(kW4Forms[pick], a, EPI == W4_SWIGLU);
    if ((t.mt * t.nt + 7) / 8 * 8 * (kWave * kW4Forms[pick].wn * kW4Forms[pick].kg) > kGridThreads)
        return set_error(EFM_ERR_UNSUPPORTED, "%s: too many tiles", who);
    const dim3 grid((unsigned)((t.mt * t.nt + 7) / 8 * 8));
    auto go = [&](auto ic) {
        constexpr W4Form f = kW4Forms[decltype(ic)::value];
        if constexpr (EPI != W4_SWIGLU || f.tn % 2 == 0) {
            if (pick == decltype(ic)::value)
                hipLaunchKernelGGL((fp4_linear_tile_kernel<f.tm, f.tn, f.wn, f.kg, EPI>), grid,
                                   dim3(kWave * f.wn * f.kg), 0, stream, a, (int)t.mt, (int)t.nt);
        }
    };
    [&]<int... I>(std::integer_sequence<int, I...>) { (go(std::integral_constant<int, I>{}), ...); }
    (std::make_integer_sequence<int, kW4FormCount>{});
    return check_launch(who);
}

}  // namespace efm

using namespace efm;

extern "C" size_t efm_fp4_packed_bytes(int64_t in_features, int64_t out_features) {
    return w4_check("fp4_packed_bytes", in_features, out_features) == EFM_OK ? w4_packed_bytes(in_features, out_features) : 0;
}

extern "C" int efm_fp4_quantize(int64_t in_features, int64_t out_features, const void* w, uint8_t* codes, uint8_t* scales,
                                hipStream_t stream) {
    const int rc = w4_check("fp4_quantize", in_features, out_features);
    if (rc) return rc;
    if (!w || !codes || !scales) return set_error(EFM_ERR_INVALID_ARGUMENT, "fp4_quantize: null pointer");
    if (!w4_aligned(w) || !w4_aligned(codes))
        return set_error(EFM_ERR_INVALID_ARGUMENT, "fp4_quantize: w and codes must be 16-byte aligned");
    const int64_t octets = in_features * out_features / 8;
    hipLaunchKernelGGL(fp4_quantize_kernel, dim3((unsigned)std::min<int64_t>(8192, (octets + 255) / 256)), dim3(256), 0, stream,
                       static_cast<const uint4*>(w), reinterpret_cast<uint32_t*>(codes), scales, octets);
    return check_launch("fp4_quantize");
}

extern "C" int efm_fp4_pack(int64_t in_features, int64_t out_features, const uint8_t* codes, const uint8_t* scales,
                            void* packed, hipStream_t stream) {
    const int rc = w4_check("fp4_pack", in_features, out_features);
    if (rc) return rc;
    if (!codes || !scales || !packed) return set_error(EFM_ERR_INVALID_ARGUMENT, "fp4_pack: null pointer");
    if (!w4_aligned(codes) || !w4_aligned(packed))
        return set_error(EFM_ERR_INVALID_ARGUMENT, "fp4_pack: codes and packed must be 16-byte aligned");
    const int64_t total = (int64_t)w4_tiles(out_features) * w4_blocks(in_features);
    uint8_t* p = static_cast<uint8_t*>(packed);
    hipLaunchKernelGGL(fp4_pack_kernel, dim3((unsigned)std::min(kGridThreads / 256, (total + 3) / 4)), dim3(256), 0, stream, codes, scales,
                       reinterpret_cast<uint4*>(p), reinterpret_cast<uint32_t*>(p + w4_code_bytes(in_features, out_features)),
                       in_features, out_features, w4_blocks(in_features), total);
    return check_launch("fp4_pack");
}

static int w4_check_call(const char* who, int64_t m, int64_t in, int64_t out, const void* x, const void* packed, const void* y) {
    if (m < 0) return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: bad shape m=%lld", who, (long long)m);
    const int rc = w4_check(who, in, out);
    if (rc) return rc;
    if (m > (1 << 20)) return set_error(EFM_ERR_UNSUPPORTED, "%s: m=%lld too large", who, (long long)m);
    if (!x || !packed || !y) return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    if (!w4_aligned(x) || !w4_aligned(packed))
        return set_error(EFM_ERR_INVALID_ARGUMENT, "%s: x and the packed weights must be 16-byte aligned", who);
    return EFM_OK;
}

extern "C" size_t efm_linear_fp4_workspace_bytes(int64_t m, int64_t in_features, int64_t out_features) {
    return 0;
}

extern "C" int efm_linear_fp4(int64_t m, int64_t in_features, int64_t out_features, const void* x, const void* w_packed,
                              const void* bias, void* y, int32_t out_dtype, void* workspace, size_t workspace_bytes,
                              hipStream_t stream) {
    const int rc = w4_check_call("linear_fp4", m, in_features, out_features, x, w_packed, y);
    if (rc) return rc;
    if (out_dtype != EFM_DTYPE_BF16 && out_dtype != EFM_DTYPE_F32)
        return set_error(EFM_ERR_UNSUPPORTED, "linear_fp4: output dtype %d not supported", out_dtype);
    if (m == 0) return EFM_OK;
    const W4Args a{static_cast<const bf16_t*>(x), w4_weights(in_features, out_features, w_packed),
                   static_cast<const bf16_t*>(bias), y, m, out_features, in_features};
    return out_dtype == EFM_DTYPE_F32 ? w4_launch<W4_F32>("linear_fp4", a, stream) : w4_launch<W4_BF16>("linear_fp4", a, stream);
}

extern "C" int32_t efm_testing_fp4_linear_form(int64_t m, int64_t in_features, int64_t out_features, int32_t swiglu,
                                               int32_t* forms, int32_t* steps) {
    const bool s = swiglu != 0;
    if (w4_check("testing_fp4_linear_form", in_features, s ? 2 * out_features : out_features) != EFM_OK || m <= kW4FewRows ||
        forms == nullptr || steps == nullptr)
        return -1;
    const W4Args a{nullptr, w4_weights(in_features, s ? 2 * out_features : out_features, nullptr), nullptr, nullptr, m, out_features,
                   in_features};
    const int pick = w4_pick(a, s, prefill_cus());
    *forms = (int32_t)std::count_if(kW4Forms, kW4Forms + kW4FormCount, [&](const W4Form& f) { return !s || f.tn % 2 == 0; });
    *steps = w4_steps(kW4Forms[pick], in_features, a.w.blocks);
    return pick;
}

extern "C" size_t efm_fused_gate_up_swiglu_fp4_workspace_bytes(int64_t m, int64_t hidden, int64_t inter) {
    return 0;
}

extern "C" int efm_fused_gate_up_swiglu_fp4(int64_t m, int64_t hidden, int64_t inter, const void* x, const void* w_packed,
                                            void* out, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (inter > 0 && inter % kW4Rows != 0)
        return set_error(EFM_ERR_UNSUPPORTED, "fused_gate_up_swiglu_fp4: inter must be a multiple of 16 (got %lld)",
                         (long long)inter);
    const int rc = w4_check_call("fused_gate_up_swiglu_fp4", m, hidden, 2 * inter, x, w_packed, out);
    if (rc) return rc;
    if (m == 0) return EFM_OK;
    const W4Args a{static_cast<const bf16_t*>(x), w4_weights(hidden, 2 * inter, w_packed), nullptr, out, m, inter, hidden};
    return w4_launch<W4_SWIGLU>("fused_gate_up_swiglu_fp4", a, stream);
}
