// Linear layers with FP4 weights (fp4.hpp) on gfx950: quantisation and packing of the weights,
// y = x W^T (+ bias) and the fused gate / up projection with SwiGLU.
//
// Packed weights: tiles of 16 rows by blocks of 128 columns, 1 KB each, in the order in which a
// wave's lanes take them as the second operand of v_mfma_f32_16x16x32_bf16: lane l holds, for
// row l % 16, the words of columns 32 w + 8 (l / 16) .. + 7, w = 0..3. One 16-byte load a lane
// feeds the four MFMAs of a block, and a wave's loads are whole contiguous kilobytes. The scale
// bytes follow all tiles, four to a row and block. Rows and columns past the matrix are zero.
#include "fp4.hpp"

#include <algorithm>

namespace efm {

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

// One lane for 8 values, four lanes for a group.
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

// One wave for a tile's block.
__global__ __launch_bounds__(256) void fp4_pack_kernel(const uint8_t* codes, const uint8_t* scales, uint4* out_codes,
                                                       uint32_t* out_scales, int64_t in, int64_t out, int blocks,
                                                       int64_t total) {
    const int64_t t = blockIdx.x * 4ll + threadIdx.x / kWave;
    if (t >= total) return;
    const int lane = threadIdx.x % kWave, g = lane / 16;
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

enum { W4_BF16 = 0, W4_F32 = 1, W4_SWIGLU = 2 };

struct W4Args {
    const bf16_t* x;
    Fp4Weights w;
    const bf16_t* bias;
    void* y;
    int64_t M, N, K;   // N: columns of y
};

// A workgroup takes 16 MT rows of x and NT tiles of weight rows (SwiGLU: NT / 2 tiles of up and
// the NT / 2 of gate beside them); its waves take every KW-th block of K each and add their sums
// through LDS in the order of the waves.
template <int MT, int NT, int EPI>
__global__ void fp4_linear_kernel(W4Args a) {
    extern __shared__ __align__(16) float red[];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, KW = blockDim.x / kWave;
    const int g = lane / 16, l = lane % 16;
    const int half = a.w.tiles / 2;
    auto tile = [&](int j) {
        if (EPI == W4_SWIGLU) return min((int)blockIdx.x * (NT / 2) + j % (NT / 2), half - 1) + (j < NT / 2 ? 0 : half);
        return min((int)blockIdx.x * NT + j, a.w.tiles - 1);
    };
    const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
    f32x4_t acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    for (int b = wave; b < a.w.blocks; b += KW) {
        uint4 w[NT];
        uint32_t s[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const size_t at = (size_t)tile(j) * a.w.blocks + b;
            w[j] = load_stream16(a.w.codes + at * 1024 + lane * 16);
            s[j] = *reinterpret_cast<const uint32_t*>(a.w.scales + at * 64 + l * 4);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t k = (int64_t)b * kW4Cols + 32 * i;
            if (k >= a.K) break;
            bf16x8_t wf[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j)
                wf[j] = fp4_unpack8(i == 0 ? w[j].x : i == 1 ? w[j].y : i == 2 ? w[j].z : w[j].w,
                                    fp4_scale((s[j] >> (8 * i)) & 255));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const int64_t m = min(m0 + mt * 16 + l, a.M - 1);
                const bf16x8_t xf = *reinterpret_cast<const bf16x8_t*>(a.x + m * a.K + k + 8 * g);
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[mt][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf, wf[j], acc[mt][j], 0, 0, 0);
            }
        }
    }
    f32x4_t* const part = reinterpret_cast<f32x4_t*>(red);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[((wave * MT + mt) * NT + j) * kWave + lane] = acc[mt][j];
    __syncthreads();
    constexpr int NO = EPI == W4_SWIGLU ? NT / 2 : NT;   // column tiles of y
    for (int e = threadIdx.x; e < MT * NO * 256; e += blockDim.x) {
        const int n = e % 16, m = e / 16 % 16, j = e / 256 % NO, mt = e / 256 / NO;
        const int64_t row = m0 + mt * 16 + m, col = ((int64_t)blockIdx.x * NO + j) * 16 + n;
        if (row >= a.M || col >= a.N) continue;
        auto total = [&](int jj) {
            float t = 0.f;
            for (int k = 0; k < KW; ++k) t += red[(((k * MT + mt) * NT + jj) * kWave + m / 4 * 16 + n) * 4 + m % 4];
            return t;
        };
        const int64_t at = row * a.N + col;
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

template <int EPI>
static int w4_launch(const W4Args& a, hipStream_t stream) {
    const int KW = std::max(1, std::min(4, a.w.blocks));
    constexpr int NT = EPI == W4_SWIGLU ? 2 : 1;
    const int cols = EPI == W4_SWIGLU ? a.w.tiles / 2 : a.w.tiles;
    hipLaunchKernelGGL((fp4_linear_kernel<1, NT, EPI>), dim3(cols, (unsigned)((a.M + 15) / 16)), dim3(KW * kWave),
                       (size_t)KW * NT * 1024, stream, a);
    return check_launch("linear_fp4");
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
    hipLaunchKernelGGL(fp4_pack_kernel, dim3((unsigned)((total + 3) / 4)), dim3(256), 0, stream, codes, scales,
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
    return out_dtype == EFM_DTYPE_F32 ? w4_launch<W4_F32>(a, stream) : w4_launch<W4_BF16>(a, stream);
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
    return w4_launch<W4_SWIGLU>(a, stream);
}
