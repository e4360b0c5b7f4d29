// What the kernels of the convolution of 4-bit operands share (internal header; srx_conv_mx4.hip has the mathematics).
#pragma once

#include <optional>

#include "srx_mx4.h"

namespace srx {
namespace dev {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct ConvMxArgs
{
    const uint8_t *codes, *scales;    // [pixels][blocks][16], [pixels][blocks]
    const uint8_t *wCodes, *wScales;  // [O][total][16], [O][total]
    const void* bias;
    void* out;
    int pixels, H, W, O, kw, taps, padTop, padLeft;
    int blocks, total;                // blocks of a pixel, blocks of the whole reduction
    Divider byW, byH, byBlocks, byKw, byTilesO;
    int tilesO, tilesP;
    int activation;
    int stream;                       // the output passes by the caches
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
// 16 bytes a lane from memory to LDS, lane after lane from the address `lds` on, without registers.  The address goes by m0, an
// output, so that the compiler does not take what it wrote there for still there (an input, which the compiler would write,
// cost a tile kernel bound by its output 2 %).  The compiler does not count this load: whoever reads the data waits for it (vmcnt)
// and for the other waves (s_barrier) first.
__device__ __forceinline__ void loadToLds(i32x4 from, unsigned offset, unsigned lds)
{
    unsigned m0;
    asm volatile("s_mov_b32 %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds" : "=&{m0}"(m0) : "s"(lds), "v"(offset), "s"(from) : "memory");
}
// The same with 4 bytes a lane.
__device__ __forceinline__ void loadWordToLds(i32x4 from, unsigned offset, unsigned lds)
{
    unsigned m0;
    asm volatile("s_mov_b32 %0, %1\n\ts_nop 0\n\tbuffer_load_dword %2, %3, 0 offen lds" : "=&{m0}"(m0) : "s"(lds), "v"(offset), "s"(from) : "memory");
}
__device__ __forceinline__ unsigned loadByte(i32x4 from, unsigned offset)
{
    return __builtin_amdgcn_raw_buffer_load_b8(__builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uint64_t(unsigned(from[0])) | uint64_t(unsigned(from[1])) << 32), 0, from[2], from[3]), offset, 0, 0);
}

// Every sum starts with its channel's bias.
template <int FO, int FP>
__device__ __forceinline__ void startAt(f32x16 (&acc)[FO][FP], const float* bias, int h)
{
#pragma unroll
    for (int i = 0; i < FO; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
        {
            const f32x4 b = *reinterpret_cast<const f32x4*>(bias + 32 * i + 8 * g + 4 * h);
#pragma unroll
            for (int j = 0; j < FP; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[i][j][4 * g + k] = b[k];
        }
}

// Activation and stores of a wave's 32 * FO channels of 32 * FP pixels.  A lane holds, for its pixel, output channels
// 8 * (r >> 2) + 4 * h + (r & 3) of every 32; the wave turns 32 pixels at a time in its own part of LDS, so that whole
// rows of channels are stored.  place(j, to, count): where channel o0 of the first of the j-th 32 pixels goes, and how many
// of them exist (both the same for all lanes).
template <typename T, int FO, int FP, int ACT, typename Place>
__device__ __forceinline__ void finishAs(const ConvMxArgs& a, const f32x16 (&acc)[FO][FP], uint8_t* mine, int o0, int lane, Place&& place)
{
    constexpr int kOutRow = 32 * FO * int(sizeof(T)) + 16;
    constexpr int kN = 16 / int(sizeof(T)), kPerRow = 32 * FO / kN;   // elements of a store, stores of a pixel
    constexpr bool kEven = 64 % kPerRow == 0;
    constexpr int kPass = 64 / kPerRow, kStores = kPerRow / 2;        // pixels stored at a time (kEven), times for 32 pixels
    typedef T T4 __attribute__((ext_vector_type(4)));
    const int h = lane >> 5, l = lane & 31;
    int px = lane / kPerRow, part = lane % kPerRow, channels = a.O - o0 - part * kN;   // channels that exist from this lane's first on
    const unsigned lanes = unsigned(px) * unsigned(a.O) * unsigned(sizeof(T)) + part * 16, pass = unsigned(kPass) * unsigned(a.O) * unsigned(sizeof(T));
#pragma unroll
    for (int j = 0; j < FP; ++j)
    {
#pragma unroll
        for (int i = 0; i < FO; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g)
            {
                const int o = 32 * i + 8 * g + 4 * h;
                T4 v4;
#pragma unroll
                for (int k = 0; k < 4; ++k) v4[k] = (T)(ACT == 1 ? acc[i][j][4 * g + k] : activate(acc[i][j][4 * g + k], ACT));
                if (ACT == 1) v4 = __builtin_elementwise_maximum(v4, T4{0, 0, 0, 0});     // rounding keeps the sign: two at a time in fp16
                *reinterpret_cast<T4*>(mine + l * kOutRow + o * int(sizeof(T))) = v4;
            }
        __builtin_amdgcn_wave_barrier();
        uint8_t* to;
        int count;
        place(j, to, count);
#pragma unroll
        for (int u = 0; u < kStores; ++u)
        {
            if (!kEven)
            {
                px = (u * 64 + lane) / kPerRow;
                part = (u * 64 + lane) % kPerRow;
                channels = a.O - o0 - part * kN;
            }
            const int row = kEven ? u * kPass + px : px;
            const uint4 v = *reinterpret_cast<const uint4*>(mine + row * kOutRow + part * 16);
            if (row >= count) continue;
            uint8_t* dst = to + (kEven ? lanes + u * pass : unsigned(px) * unsigned(a.O) * unsigned(sizeof(T)) + part * 16);
            if (channels >= kN)
            {
                typedef unsigned u32x4_at __attribute__((ext_vector_type(4), aligned(2)));
                const u32x4_at w = {v.x, v.y, v.z, v.w};
                if (a.stream) __builtin_nontemporal_store(w, reinterpret_cast<u32x4_at*>(dst));
                else *reinterpret_cast<u32x4_at*>(dst) = w;
            }
            else
            {
                T e[kN];
                __builtin_memcpy(e, &v, 16);
#pragma unroll
                for (int k = 0; k < kN; ++k)
                    if (k < channels) reinterpret_cast<T*>(dst)[k] = e[k];
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}
template <typename T, int FO, int FP, typename Place>
__device__ __forceinline__ void finish(const ConvMxArgs& a, const f32x16 (&acc)[FO][FP], uint8_t* mine, int o0, int lane, Place&& place)
{
    if (a.activation == 0) finishAs<T, FO, FP, 0>(a, acc, mine, o0, lane, place);
    else if (a.activation == 1) finishAs<T, FO, FP, 1>(a, acc, mine, o0, lane, place);
    else finishAs<T, FO, FP, 2>(a, acc, mine, o0, lane, place);
}

// Tiles of the kernels that stage windows: pixels.
constexpr int kWinH = 8, kWinW = 32;

inline bool scalesInWords(const ConvMxArgs& a)
{
    return a.blocks % 4 == 0 && ((reinterpret_cast<uintptr_t>(a.scales) | reinterpret_cast<uintptr_t>(a.wScales)) & 3) == 0;
}

// What became of a launch; nothing where the kernel does not suit the sizes and none was tried.  (A launch that was tried and
// failed is an error, whatever its code: no other kernel may cover it up.)
typedef std::optional<hipError_t> Launched;

// ConvMxTapsKernel with tiles of 32, 64, 96 or 128 channels.  Nothing where the window does not fit half a CU's LDS, where the
// tiles at the images' edges are a quarter empty, or where there are too few.
Launched launchConvMxTaps(bool half, int channels, const ConvMxArgs& a, hipStream_t s);

}  // namespace dev
}  // namespace srx
