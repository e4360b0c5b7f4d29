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

// Division of numbers below 2^31 by a constant d: (mulhi(n, mul) + n) >> shift.
struct Divider
{
    unsigned mul = 0, shift = 0, d = 1;
    Divider() = default;
    explicit Divider(unsigned by) : d(by)
    {
        while ((uint64_t(1) << shift) < by) ++shift;
        mul = unsigned((uint64_t(1) << 32) * ((uint64_t(1) << shift) - by) / by + 1);
    }
    __device__ __forceinline__ unsigned operator()(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

struct ConvMxArgs
{
    const uint8_t *codes, *scales;    // [pixels][blocks][16], [pixels][blocks]
    const uint8_t *wCodes, *wScales;  // [O][total][16], [O][total]
    const void* bias;
    void* out;
    int pixels, H, W, O, kw, taps, padTop, padLeft;
    int blocks, total;                // blocks of a pixel, blocks of the whole reduction
    Divider byW, byH, byBlocks, byKw, byTilesO;
    int tilesO;
    int activation;
};

constexpr int kChunk = 8;             // blocks staged at a time: four instructions' worth
constexpr int kRow = kChunk * kMxBytes;

// Position of block `b` of row `row` in LDS: rows are 128 bytes apart, and the exclusive-or spreads the 16 rows that
// one pass of a ds_read_b128 covers over all 64 banks.
__device__ __forceinline__ int slot(int row, int b) { return row * kRow + ((b ^ ((row >> 1) & 7)) << 4); }

__device__ __forceinline__ i32x8 widen(const uint4& v)
{
    return i32x8{int(v.x), int(v.y), int(v.z), int(v.w), 0, 0, 0, 0};
}

// Buffer descriptors of everything from `p` on: offsets below kRange are read, others give zeros.  A lane that has
// nothing to read takes the offset kRange.  Scales lie at a sixteenth of their codes' offsets.
constexpr unsigned kRange = 0x80000000u;
__device__ __forceinline__ i32x4 descriptor(const uint8_t* p, unsigned range)
{
    const uint64_t at = reinterpret_cast<uint64_t>(p);
    return i32x4{int(unsigned(at)), int(unsigned(at >> 32) & 0xffffu), int(range), 0x00027000};
}
// 16 bytes a lane from memory to LDS, lane after lane from the address `lds` on, without registers.  The compiler does
// not count this load: whoever reads the data waits for it (vmcnt) and for the other waves (s_barrier) first.
__device__ __forceinline__ void loadToLds(i32x4 from, unsigned offset, unsigned lds)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(from) : "memory");
}
__device__ __forceinline__ unsigned loadWord(i32x4 from, unsigned offset)
{
    return __builtin_amdgcn_raw_buffer_load_b32(__builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uint64_t(unsigned(from[0])) | uint64_t(unsigned(from[1])) << 32), 0, from[2], from[3]), offset, 0, 0);
}
__device__ __forceinline__ unsigned loadByte(i32x4 from, unsigned offset)
{
    return __builtin_amdgcn_raw_buffer_load_b8(__builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uint64_t(unsigned(from[0])) | uint64_t(unsigned(from[1])) << 32), 0, from[2], from[3]), offset, 0, 0);
}

// Bias, activation and stores of a wave's 32 * FO channels of 32 * FP pixels.  A lane holds, for its pixel, output channels
// 8 * (r >> 2) + 4 * h + (r & 3) of every 32; the wave turns 32 pixels at a time in its own part of LDS, so that whole
// rows of channels are stored.
template <typename T, int FO, int FP, int ACT>
__device__ __forceinline__ void finish(const ConvMxArgs& a, const f32x16 (&acc)[FO][FP], const float* bias, uint8_t* mine, int64_t m0, int o0, int lane)
{
    constexpr int kOutRow = 32 * FO * int(sizeof(T)) + 16;
    constexpr int kN = 16 / int(sizeof(T)), kPerRow = 32 * FO / kN;   // elements of a store, stores of a pixel
    typedef T T4 __attribute__((ext_vector_type(4)));
    const int h = lane >> 5, l = lane & 31;
    T* out = static_cast<T*>(a.out);
#pragma unroll
    for (int j = 0; j < FP; ++j)
    {
#pragma unroll
        for (int i = 0; i < FO; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
            {
                const int o = 32 * i + 8 * g + 4 * h;
                const f32x4 b = *reinterpret_cast<const f32x4*>(bias + o);
                T4 v4;
#pragma unroll
                for (int k = 0; k < 4; ++k) v4[k] = (T)activate(acc[i][j][4 * g + k] + b[k], ACT);
                *reinterpret_cast<T4*>(mine + l * kOutRow + o * int(sizeof(T))) = v4;
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < 32 * kPerRow / 64; ++u)
        {
            const int px = (u * 64 + lane) / kPerRow, part = (u * 64 + lane) % kPerRow;
            const int64_t m = m0 + 32 * j + px;
            const int o = o0 + part * kN;
            const uint4 v = *reinterpret_cast<const uint4*>(mine + px * kOutRow + part * 16);
            if (m >= a.pixels) continue;
            T* dst = out + m * a.O + o;
            if (o + kN <= a.O) __builtin_memcpy(dst, &v, 16);
            else
            {
                T e[kN];
                __builtin_memcpy(e, &v, 16);
#pragma unroll
                for (int k = 0; k < kN; ++k)
                    if (o + k < a.O) dst[k] = e[k];
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// A workgroup (four waves) makes BO output channels of BP pixels; wave w makes 32 * FO channels of 32 * FP pixels.
// The reduction goes in chunks of eight blocks through two buffers in LDS: while one is multiplied, the next is on its
// way from memory to the other (one barrier a chunk).
//   WITHIN: no chunk crosses from one tap to the next (each tap's blocks are padded to whole chunks), so that a tap's
//           offsets are found once; otherwise blocks are numbered through and every thread finds its own tap.
//   WORDS:  the blocks of a pixel come in fours, so that a lane's four scales of a chunk are one word, read right into
//           the lane that needs it; otherwise scales are staged in LDS byte by byte.
template <typename T, int BO, int BP, int FO, int FP, bool WITHIN, bool WORDS>
__global__ __launch_bounds__(kThreads) void ConvMxKernel(const ConvMxArgs a)
{
    static_assert(BO * BP == 4 * 32 * FO * 32 * FP, "four waves");
    constexpr int kCodes = (BO + BP) * kRow, kStage = kCodes + (WORDS ? 0 : (BO + BP) * kChunk);
    constexpr int kOutRow = 32 * FO * int(sizeof(T)) + 16;            // bytes of a pixel in the epilogue, padded
    constexpr int kLds = 2 * kStage > 4 * 32 * kOutRow ? 2 * kStage : 4 * 32 * kOutRow;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
    __shared__ __attribute__((aligned(16))) float sBias[BO];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l = lane & 31;
    const unsigned tileP = a.byTilesO(blockIdx.x);
    const int o0 = int(blockIdx.x - tileP * a.tilesO) * BO;
    const int64_t m0 = int64_t(tileP) * BP;
    constexpr int kWavesO = BO / (32 * FO);
    const int wo = (wave % kWavesO) * 32 * FO, wp = (wave / kWavesO) * 32 * FP;
    const unsigned ldsAt = unsigned(uintptr_t((__attribute__((address_space(3))) uint8_t*)lds));

    // Staging: eight threads a row of codes, rows 32 apart; a thread's place in LDS is fixed, so the swizzle picks its block.
    constexpr int kXRows = BP / 32, kWRows = BO / 32;
    const int sr = tid >> 3, sb = (tid & 7) ^ ((sr >> 1) & 7);
    const int pixelBytes = a.blocks * kMxBytes;
    const unsigned rowBytes = unsigned(a.W) * unsigned(pixelBytes);     // below 2^31 where it is used (!WITHIN)
    const auto place = [&](int64_t m, int& y, int& x) {
        const unsigned row = a.byW(unsigned(m));
        x = int(unsigned(m) - row * unsigned(a.W));
        y = m < a.pixels ? int(row - a.byH(row) * unsigned(a.H)) : INT32_MIN / 2;   // never inside
    };
    int y[kXRows], x[kXRows], fy[FP], fx[FP];
#pragma unroll
    for (int i = 0; i < kXRows; ++i) place(m0 + sr + 32 * i, y[i], x[i]);
    if (WORDS)
    {
#pragma unroll
        for (int j = 0; j < FP; ++j) place(m0 + wp + 32 * j + l, fy[j], fx[j]);
    }
    const auto inside = [&](int yy, int xx) { return unsigned(yy) < unsigned(a.H) && unsigned(xx) < unsigned(a.W); };

    // where the next chunk is
    int tap = 0, c0 = 0, k0 = 0;                                        // WITHIN: tap and block of the pixel; else block of all
    const uint8_t *xBase = nullptr, *zBase = nullptr;
    unsigned xOff[kXRows], wOff[kWRows], zOff[FP], vOff[FO];
#pragma unroll
    for (int i = 0; i < kWRows; ++i) wOff[i] = o0 + sr + 32 * i < a.O ? unsigned((sr + 32 * i) * a.total + sb) * kMxBytes : kRange;
    if (WORDS)
    {
#pragma unroll
        for (int i = 0; i < FO; ++i) vOff[i] = o0 + wo + 32 * i + l < a.O ? unsigned((wo + 32 * i + l) * a.total + 4 * h) : kRange;
    }
    const auto enterTap = [&]() {
        const int ky = int(a.byKw(unsigned(tap))), dy = ky - a.padTop, dx = tap - ky * a.kw - a.padLeft;
        xBase = a.codes + (m0 + int64_t(dy) * a.W + dx) * pixelBytes;
        zBase = a.scales + (m0 + int64_t(dy) * a.W + dx) * a.blocks;
#pragma unroll
        for (int i = 0; i < kXRows; ++i) xOff[i] = inside(y[i] + dy, x[i] + dx) ? unsigned((sr + 32 * i) * a.blocks + sb) * kMxBytes : kRange;
        if (WORDS)
        {
#pragma unroll
            for (int j = 0; j < FP; ++j) zOff[j] = inside(fy[j] + dy, fx[j] + dx) ? unsigned((wp + 32 * j + l) * a.blocks + 4 * h) : kRange;
        }
    };
    if (WITHIN) enterTap();
    else
    {
        xBase = a.codes + (m0 - int64_t(a.padTop) * a.W - a.padLeft) * pixelBytes;
        zBase = a.scales + (m0 - int64_t(a.padTop) * a.W - a.padLeft) * a.blocks;
    }

    unsigned xs[FP], ws[FO], nextX[FP], nextW[FO], xz[kXRows], wz[kWRows];
    const auto fetch = [&](int stage) {
        const int block = WITHIN ? c0 : 0;
        const int kb = WITHIN ? tap * a.blocks + c0 : k0;
        const bool in = WITHIN ? c0 + sb < a.blocks : k0 + sb < a.total;
        const i32x4 xd = descriptor(xBase + int64_t(block) * kMxBytes, kRange), wd = descriptor(a.wCodes + (int64_t(o0) * a.total + kb) * kMxBytes, kRange);
        const i32x4 zd = descriptor(zBase + block, WORDS ? kRange : kRange >> 4), vd = descriptor(a.wScales + int64_t(o0) * a.total + kb, WORDS ? kRange : kRange >> 4);
        const unsigned at = ldsAt + stage + wave * 1024;
        unsigned off[kXRows];
        if (WITHIN)
        {
#pragma unroll
            for (int i = 0; i < kXRows; ++i) off[i] = in ? xOff[i] : kRange;
        }
        else
        {
            const int t = int(a.byBlocks(unsigned(k0 + sb))), ky = int(a.byKw(unsigned(t))), kx = t - ky * a.kw;
            const unsigned from = unsigned(ky) * rowBytes + unsigned(kx * pixelBytes + (k0 + sb - t * a.blocks) * kMxBytes);
#pragma unroll
            for (int i = 0; i < kXRows; ++i)
                off[i] = in && inside(y[i] + ky - a.padTop, x[i] + kx - a.padLeft) ? from + unsigned((sr + 32 * i) * pixelBytes) : kRange;
        }
#pragma unroll
        for (int i = 0; i < kWRows; ++i) loadToLds(wd, in ? wOff[i] : kRange, at + i * 4096);
#pragma unroll
        for (int i = 0; i < kXRows; ++i) loadToLds(xd, off[i], at + BO * kRow + i * 4096);
        if (WORDS && WITHIN)
        {
            const bool zin = c0 + 4 * h < a.blocks;
#pragma unroll
            for (int i = 0; i < FO; ++i) nextW[i] = loadWord(vd, zin ? vOff[i] : kRange);
#pragma unroll
            for (int j = 0; j < FP; ++j) nextX[j] = loadWord(zd, zin ? zOff[j] : kRange);
        }
        else if (WORDS)
        {
            const int kz = k0 + 4 * h;
            const int t = int(a.byBlocks(unsigned(kz))), ky = int(a.byKw(unsigned(t))), kx = t - ky * a.kw;
            const bool zin = kz < a.total;
            const unsigned from = (unsigned(ky) * rowBytes + unsigned(kx * pixelBytes)) / kMxBytes + unsigned(kz - t * a.blocks);
#pragma unroll
            for (int i = 0; i < FO; ++i) nextW[i] = loadWord(vd, zin ? vOff[i] : kRange);
#pragma unroll
            for (int j = 0; j < FP; ++j)
                nextX[j] = loadWord(zd, zin && inside(fy[j] + ky - a.padTop, fx[j] + kx - a.padLeft) ? from + unsigned((wp + 32 * j + l) * a.blocks) : kRange);
        }
        else
        {
#pragma unroll
            for (int i = 0; i < kWRows; ++i) wz[i] = loadByte(vd, (in ? wOff[i] : kRange) / kMxBytes);
#pragma unroll
            for (int i = 0; i < kXRows; ++i) xz[i] = loadByte(zd, off[i] / kMxBytes);
        }
        if (WITHIN)
        {
            c0 += kChunk;
            if (c0 >= a.blocks) { c0 = 0; ++tap; if (tap < a.taps) enterTap(); }
        }
        else k0 += kChunk;
    };
    // after fetch(stage): what does not go to LDS by itself
    const auto settle = [&](int stage) {
        if (WORDS)
        {
#pragma unroll
            for (int i = 0; i < FO; ++i) ws[i] = nextW[i];
#pragma unroll
            for (int j = 0; j < FP; ++j) xs[j] = nextX[j];
        }
        else
        {
            uint8_t* z = lds + stage + kCodes;
#pragma unroll
            for (int i = 0; i < kWRows; ++i) z[(sr + 32 * i) * kChunk + sb] = uint8_t(wz[i]);
#pragma unroll
            for (int i = 0; i < kXRows; ++i) z[(BO + sr + 32 * i) * kChunk + sb] = uint8_t(xz[i]);
        }
    };

    f32x16 acc[FO][FP];
#pragma unroll
    for (int i = 0; i < FO; ++i)
#pragma unroll
        for (int j = 0; j < FP; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    fetch(0);
    for (int o = tid; o < BO; o += kThreads)
        sBias[o] = a.bias && o0 + o < a.O ? (float)static_cast<const T*>(a.bias)[o0 + o] : 0.0f;
    settle(0);
    const int chunks = WITHIN ? a.taps * ((a.blocks + kChunk - 1) / kChunk) : (a.total + kChunk - 1) / kChunk;
    int stage = 0, left = WITHIN ? a.blocks : a.total;                  // blocks left in the tap / in all
    for (int c = 0; c < chunks; ++c)
    {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const uint8_t* from = lds + stage;
        stage = kStage - stage;
        if (c + 1 < chunks) fetch(stage);
        if (!WORDS)
        {
            const unsigned* z = reinterpret_cast<const unsigned*>(from + kCodes);
#pragma unroll
            for (int i = 0; i < FO; ++i) ws[i] = z[(wo + 32 * i + l) * 2 + h];
#pragma unroll
            for (int j = 0; j < FP; ++j) xs[j] = z[(BO + wp + 32 * j + l) * 2 + h];
        }
        // step s multiplies the blocks s (lanes 0-31) and 4 + s (lanes 32-63): a lane's four scales are one word
#define SRX_STEP(S)                                                                                                    \
        if (S < left)                                                                                                  \
        {                                                                                                              \
            i32x8 wf[FO], xf[FP];                                                                                      \
            _Pragma("unroll") for (int i = 0; i < FO; ++i)                                                             \
                wf[i] = widen(*reinterpret_cast<const uint4*>(from + slot(wo + 32 * i + l, 4 * h + S)));               \
            _Pragma("unroll") for (int j = 0; j < FP; ++j)                                                             \
                xf[j] = widen(*reinterpret_cast<const uint4*>(from + BO * kRow + slot(wp + 32 * j + l, 4 * h + S)));   \
            _Pragma("unroll") for (int i = 0; i < FO; ++i)                                                             \
                _Pragma("unroll") for (int j = 0; j < FP; ++j)                                                         \
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[i], xf[j], acc[i][j], 4, 4, S, ws[i], S, xs[j]); \
        }
        SRX_STEP(0)
        SRX_STEP(1)
        SRX_STEP(2)
        SRX_STEP(3)
#undef SRX_STEP
        left -= kChunk;
        if (WITHIN && left <= 0) left = a.blocks;
        if (c + 1 < chunks) settle(stage);
    }
    __syncthreads();
    uint8_t* mine = lds + wave * 32 * kOutRow;
    if (a.activation == 0) finish<T, FO, FP, 0>(a, acc, sBias + wo, mine, m0 + wp, o0 + wo, lane);
    else if (a.activation == 1) finish<T, FO, FP, 1>(a, acc, sBias + wo, mine, m0 + wp, o0 + wo, lane);
    else finish<T, FO, FP, 2>(a, acc, sBias + wo, mine, m0 + wp, o0 + wo, lane);
}

template <typename T, int BO, int BP, int FO, int FP>
hipError_t launch(const ConvMxArgs& args, hipStream_t s)
{
    ConvMxArgs a = args;
    a.tilesO = (a.O + BO - 1) / BO;
    a.byTilesO = Divider(unsigned(a.tilesO));
    const int64_t grid = int64_t(a.tilesO) * ((int64_t(a.pixels) + BP - 1) / BP);
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    const dim3 g(static_cast<unsigned>(grid)), block(kThreads);
    // Numbered-through blocks need all taps of a tile within the range of one descriptor.
    const int64_t span = ((int64_t(a.taps / a.kw) * a.W + a.kw + BP) * a.blocks + a.total) * kMxBytes;
    const bool within = a.taps == 1 || a.blocks % kChunk == 0 || span >= int64_t(kRange);
    const bool words = a.blocks % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.scales) | reinterpret_cast<uintptr_t>(a.wScales)) & 3) == 0;
    if (within && words) hipLaunchKernelGGL((ConvMxKernel<T, BO, BP, FO, FP, true, true>), g, block, 0, s, a);
    else if (within) hipLaunchKernelGGL((ConvMxKernel<T, BO, BP, FO, FP, true, false>), g, block, 0, s, a);
    else if (words) hipLaunchKernelGGL((ConvMxKernel<T, BO, BP, FO, FP, false, true>), g, block, 0, s, a);
    else hipLaunchKernelGGL((ConvMxKernel<T, BO, BP, FO, FP, false, false>), g, block, 0, s, a);
    return hipGetLastError();
}

template <int BO, int BP, int FO, int FP>
hipError_t launch(bool half, const ConvMxArgs& a, hipStream_t s)
{
    return half ? launch<f16, BO, BP, FO, FP>(a, s) : launch<float, BO, BP, FO, FP>(a, s);
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
    a.taps = int(op.filterSizes[2] * op.filterSizes[3]);
    a.total = a.taps * a.blocks;
    a.byW = Divider(unsigned(a.W));
    a.byH = Divider(unsigned(a.H));
    a.byBlocks = Divider(unsigned(a.blocks));
    a.byKw = Divider(unsigned(a.kw));
    a.activation = int(op.activation);
    return launch<64, 256, 2, 2>(op.dataType == ML::TensorDataType::FLOAT16, a, s);
}

}  // namespace srx
