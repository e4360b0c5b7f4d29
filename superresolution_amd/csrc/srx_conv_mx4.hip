// gfx950 kernel of the convolution whose input and filter are held in the 4-bit block form (srx_mx4.h).
//
//   out[pixel][o] = act(bias[o] + sum over taps (i, j) and channels c of in[pixel + (i - padTop, j - padLeft)][c] * w[o][i][j][c])
//
// as an implicit matrix product on v_mfma_scale_f32_32x32x64_f8f6f4: rows = output channels, columns = pixels, and a
// reduction over the blocks of 32 channels of every tap, numbered kb = tap * (blocks of a pixel) + block.  One
// instruction multiplies two blocks: lanes 0-31 hold one of them for 32 rows (or columns), lanes 32-63 the other, 16
// bytes and one scale byte each, so that the two blocks may come from different taps.  fp32 accumulation.
#include "srx_mx4.h"

namespace srx {

using namespace dev;

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct ConvMxArgs
{
    const uint8_t *codes, *scales;    // [pixels][blocks][16], [pixels][blocks]
    const uint8_t *wCodes, *wScales;  // [O][taps * blocks][16], [O][taps * blocks]
    const void* bias;
    void* out;
    int pixels, H, W, O, kw, padTop, padLeft;
    int blocks, total;                // blocks of a pixel, blocks of the whole reduction
    int tilesO;
    int activation;
};

constexpr int kChunk = 8;             // blocks staged at a time: four instructions' worth

// Position of block `b` of row `row` in LDS: rows are 128 bytes apart, and the exclusive-or spreads the 16 rows that
// one pass of a ds_read_b128 covers over all 64 banks.
__device__ __forceinline__ int slot(int row, int b) { return row * (kChunk * kMxBytes) + ((b ^ ((row >> 1) & 7)) << 4); }

__device__ __forceinline__ i32x8 widen(const uint4& v)
{
    return i32x8{int(v.x), int(v.y), int(v.z), int(v.w), 0, 0, 0, 0};
}

// A workgroup makes BO output channels of BP pixels; wave w makes 32 * FO channels of 32 * FP pixels.
template <typename T, int BO, int BP, int FO, int FP>
__global__ __launch_bounds__(kThreads) void ConvMxKernel(const ConvMxArgs a)
{
    static_assert(BO * BP == 4 * 32 * FO * 32 * FP, "four waves");
    __shared__ __attribute__((aligned(16))) uint8_t sW[BO * kChunk * kMxBytes], sX[BP * kChunk * kMxBytes];
    __shared__ unsigned sWs[BO * 2], sXs[BP * 2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, l = lane & 31;
    const int o0 = int(blockIdx.x % a.tilesO) * BO;
    const int64_t m0 = int64_t(blockIdx.x / a.tilesO) * BP;
    constexpr int kWavesO = BO / (32 * FO);
    const int wo = (wave % kWavesO) * 32 * FO, wp = (wave / kWavesO) * 32 * FP;

    f32x16 acc[FO][FP];
#pragma unroll
    for (int i = 0; i < FO; ++i)
#pragma unroll
        for (int j = 0; j < FP; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    // block kb of pixel m: the offset of its bytes, or -1 outside the image or the reduction
    const auto xBlock = [&](int64_t m, int kb) -> int64_t {
        if (m >= a.pixels || kb >= a.total) return -1;
        const int tap = kb / a.blocks, cb = kb - tap * a.blocks;
        const int ky = tap / a.kw, kx = tap - ky * a.kw;
        const int row = int(m) / a.W, x = int(m) - row * a.W + kx - a.padLeft, y = row % a.H + ky - a.padTop;
        if (x < 0 || x >= a.W || y < 0 || y >= a.H) return -1;
        return (m + int64_t(ky - a.padTop) * a.W + kx - a.padLeft) * a.blocks + cb;
    };
    const auto wBlock = [&](int o, int kb) -> int64_t { return o < a.O && kb < a.total ? int64_t(o) * a.total + kb : -1; };

    for (int k0 = 0; k0 < a.total; k0 += kChunk)
    {
        __syncthreads();
        for (int u = tid; u < BO * kChunk; u += kThreads)
        {
            const int64_t at = wBlock(o0 + (u >> 3), k0 + (u & 7));
            uint4 v = uint4{0, 0, 0, 0};
            if (at >= 0) __builtin_memcpy(&v, a.wCodes + at * kMxBytes, 16);
            *reinterpret_cast<uint4*>(sW + slot(u >> 3, u & 7)) = v;
            reinterpret_cast<uint8_t*>(sWs)[u] = at >= 0 ? a.wScales[at] : 0;
        }
        for (int u = tid; u < BP * kChunk; u += kThreads)
        {
            const int64_t at = xBlock(m0 + (u >> 3), k0 + (u & 7));
            uint4 v = uint4{0, 0, 0, 0};
            if (at >= 0) __builtin_memcpy(&v, a.codes + at * kMxBytes, 16);
            *reinterpret_cast<uint4*>(sX + slot(u >> 3, u & 7)) = v;
            reinterpret_cast<uint8_t*>(sXs)[u] = at >= 0 ? a.scales[at] : 0;
        }
        __syncthreads();
        // step s multiplies the blocks s (lanes 0-31) and 4 + s (lanes 32-63): a lane's four scales are one word
        unsigned ws[FO], xs[FP];
#pragma unroll
        for (int i = 0; i < FO; ++i) ws[i] = sWs[(wo + 32 * i + l) * 2 + h];
#pragma unroll
        for (int j = 0; j < FP; ++j) xs[j] = sXs[(wp + 32 * j + l) * 2 + h];
#define SRX_STEP(S)                                                                                                    \
        {                                                                                                              \
            i32x8 w[FO], x[FP];                                                                                        \
            _Pragma("unroll") for (int i = 0; i < FO; ++i)                                                             \
                w[i] = widen(*reinterpret_cast<const uint4*>(sW + slot(wo + 32 * i + l, 4 * h + S)));                  \
            _Pragma("unroll") for (int j = 0; j < FP; ++j)                                                             \
                x[j] = widen(*reinterpret_cast<const uint4*>(sX + slot(wp + 32 * j + l, 4 * h + S)));                  \
            _Pragma("unroll") for (int i = 0; i < FO; ++i)                                                             \
                _Pragma("unroll") for (int j = 0; j < FP; ++j)                                                         \
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[i], x[j], acc[i][j], 4, 4, S, ws[i], S, xs[j]); \
        }
        SRX_STEP(0)
        SRX_STEP(1)
        SRX_STEP(2)
        SRX_STEP(3)
#undef SRX_STEP
    }

    // a lane holds, for its pixel, output channels 8 * (r >> 2) + 4 * h + (r & 3) of every 32
    T* out = static_cast<T*>(a.out);
    const T* bias = static_cast<const T*>(a.bias);
#pragma unroll
    for (int j = 0; j < FP; ++j)
    {
        const int64_t m = m0 + wp + 32 * j + l;
        if (m >= a.pixels) continue;
#pragma unroll
        for (int i = 0; i < FO; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
            {
                const int o = o0 + wo + 32 * i + 8 * (r >> 2) + 4 * h + (r & 3);
                if (o >= a.O) continue;
                float v = acc[i][j][r];
                if (bias) v += (float)bias[o];
                out[m * a.O + o] = (T)activate(v, a.activation);
            }
    }
}

template <int BO, int BP, int FO, int FP>
hipError_t launch(bool half, const ConvMxArgs& args, hipStream_t s)
{
    ConvMxArgs a = args;
    a.tilesO = (a.O + BO - 1) / BO;
    const int64_t grid = int64_t(a.tilesO) * ((int64_t(a.pixels) + BP - 1) / BP);
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    if (half) hipLaunchKernelGGL((ConvMxKernel<f16, BO, BP, FO, FP>), dim3(unsigned(grid)), dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL((ConvMxKernel<float, BO, BP, FO, FP>), dim3(unsigned(grid)), dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t LaunchConvMx4(const ML::Operator& op, const uint8_t* codes, const uint8_t* scales, const uint8_t* filterCodes,
                         const uint8_t* filterScales, const void* bias, void* out, hipStream_t s)
{
    ConvMxArgs a{};
    a.codes = codes;
    a.scales = scales;
    a.wCodes = filterCodes;
    a.wScales = filterScales;
    a.bias = bias;
    a.out = out;
    a.H = int(op.inputSizes[2]);
    a.W = int(op.inputSizes[3]);
    a.pixels = int(op.inputSizes[0]) * a.H * a.W;
    a.O = int(op.filterSizes[0]);
    a.kw = int(op.filterSizes[3]);
    a.padTop = int(op.padTop);
    a.padLeft = int(op.padLeft);
    a.blocks = int(mxBlocks(op.inputSizes[1]));
    a.total = int(op.filterSizes[2] * op.filterSizes[3]) * a.blocks;
    a.activation = int(op.activation);
    return launch<64, 128, 1, 2>(op.dataType == ML::TensorDataType::FLOAT16, a, s);
}

}  // namespace srx
