// gfx950 kernel of the convolution of 4-bit operands (srx_conv_mx4.hip) for filters of several taps.
#include "srx_conv_mx4.h"

namespace srx {

using namespace dev;

namespace {

// Filters of several taps: a tile's pixels are eight rows of 32, and the window that all its taps see is staged once, eight
// blocks of each pixel (a part) at a time, so that only the filters come from memory chunk by chunk (ConvMxKernel reads every pixel
// once for each tap, more than L2 delivers while tiles of 128 channels are multiplied).  A workgroup makes 32 * FO channels, a
// wave two rows of them; while one workgroup of a CU waits for its window, the others multiply.
struct TapsArgs
{
    int winW, winPixels;
    int scales;                       // place of the window's scales behind its codes
    int parts, last;                  // parts of a pixel's blocks, blocks of the last one
    int tilesX, tilesY;
    Divider byTilesX, byTilesY, byWinW, byLast;
};

template <typename T, int FO>
struct TapsLds
{
    static constexpr int kBO = 32 * FO, kStage = kBO * kRow + kThreads * 4;
    static constexpr int kOutRow = 32 * FO * int(sizeof(T)) + 16, kOut = kThreads / 64 * 32 * kOutRow;
    // two chunks of filters (codes, scales; the bias in the second one's place at first) and the window, later the turn of the results
    static int bytes(int window) { return 2 * kStage + window > kOut ? 2 * kStage + window : kOut; }
};

constexpr int kTapsLoads = 16;        // loads of a window's codes by a thread, at most

// WORDS: all parts are of four or eight blocks, whose scales are staged in words; otherwise byte by byte.  PARTS: more than one.
// As many waves a SIMD as the accumulators, and whole windows in LDS (PARTS), leave room for (96 -> 96 channels, 960x540: 8 %
// less time with three than with two).
template <typename T, int FO, bool WORDS, bool PARTS>
__global__ __launch_bounds__(kThreads, FO > 3 || PARTS ? 2 : FO > 2 ? 3 : 4) void ConvMxTapsKernel(const ConvMxArgs a, const TapsArgs w)
{
    using L = TapsLds<T, FO>;
    constexpr int kBO = L::kBO, kStage = L::kStage, kScales = kBO * kRow, kWindow = 2 * kStage, FP = 2, kPass = kThreads / 8, kWRows = kBO / kPass;
    extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l = lane & 31;
    const unsigned ldsAt = unsigned(uintptr_t((__attribute__((address_space(3))) uint8_t*)dyn));
    // as in ConvMxKernel
    const unsigned number = blockNumber(), turn = number >> 3, round = a.byTilesO(turn), tileP = round * 8 + (number & 7);
    if (tileP >= unsigned(a.tilesP)) return;
    const int o0 = int(turn - round * unsigned(a.tilesO)) * kBO;
    const unsigned tileY = w.byTilesX(tileP), n = w.byTilesY(tileY);
    const int x0 = int(tileP - tileY * unsigned(w.tilesX)) * kWinW, y0 = int(tileY - n * unsigned(w.tilesY)) * kWinH;
    const int r0 = 2 * wave;

    // Of the current part: its blocks, all of them in the reduction, division by its blocks (as Divider), and the place of a
    // pixel's block: block ^ (pixel >> down & mask), with which neighbouring 16 pixels lie in all banks.
    int part = 0, blocks, total;
    unsigned mul, shift, down, mask;
    const auto begin = [&]() {
        const bool last = !PARTS || part == w.parts - 1;
        blocks = last ? w.last : kChunk;
        total = a.taps * blocks;
        mul = last ? w.byLast.mul : 1u;
        shift = last ? w.byLast.shift : 3u;
        down = blocks == 8 ? 1 : blocks == 4 ? 2 : 3;
        mask = blocks == 8 ? 7 : blocks == 4 ? 3 : ~unsigned(blocks) & 1u;
    };
    const auto byBlocks = [&](unsigned n) { return (__umulhi(n, mul) + n) >> shift; };
    const auto place = [&](unsigned p, unsigned block) { return block ^ ((p >> down) & mask); };

    // The filters' next chunk of eight blocks of the part; beyond the last, nothing is read.
    const int sr = tid >> 3, sb = (tid & 7) ^ ((sr >> 1) & 7), zr = tid >> 1, zb = (tid & 1) * 4;
    i32x4 wd, vd;
    unsigned wOff[kWRows], off[kWRows], zOff = 0;
    uint8_t wz[kWRows];
#pragma unroll
    for (int i = 0; i < kWRows; ++i) wOff[i] = o0 + sr + kPass * i < a.O ? unsigned((sr + kPass * i) * a.total) * kMxBytes : kRange;
    const unsigned vOff = zr < kBO && o0 + zr < a.O ? unsigned(zr * a.total) : kRange;
    int next = 0;
    const auto prepare = [&]() {
        // number kb of the part is number kb + tap * (a pixel's other blocks) of a filter, from the part's first on
        const int64_t first = int64_t(o0) * a.total + part * kChunk + next;
        wd = descriptor(a.wCodes + first * kMxBytes, kRange);
        vd = descriptor(a.wScales + first, WORDS ? kRange : kRange >> 4);
        const unsigned others = PARTS ? unsigned(a.blocks - blocks) : 0u;
        const unsigned at = (byBlocks(unsigned(next + sb)) * others + unsigned(sb)) * kMxBytes, out = next + sb < total ? 0u : kRange;
#pragma unroll
        for (int i = 0; i < kWRows; ++i) off[i] = (wOff[i] + at) | out;
        if (WORDS) zOff = (vOff + byBlocks(unsigned(next + zb)) * others + unsigned(zb)) | (next + zb < total ? 0u : kRange);
        next += kChunk;
    };
    constexpr int kLoads = kWRows + (WORDS ? 1 : 0);
    const auto load = [&](int i, int stage) {
        if (i < kWRows) loadToLds(wd, off[i], ldsAt + stage + wave * 1024 + i * kThreads * 16);
        else loadWordToLds(vd, zOff, ldsAt + stage + kScales + wave * 256);
    };
    const auto loadBytes = [&]() {
#pragma unroll
        for (int i = 0; i < kWRows; ++i) wz[i] = uint8_t(loadByte(vd, off[i] / kMxBytes));
    };
    const auto settle = [&](int stage) {
#pragma unroll
        for (int i = 0; i < kWRows; ++i) dyn[stage + kScales + (sr + kPass * i) * kChunk + sb] = wz[i];
    };

    // Operands of step s of the current chunk: blocks s (lanes 0-31) and 4 + s (lanes 32-63).  Behind the last block the filters
    // are zeros, and the last block's pixels, which are in the sum anyway, stand in.
    int chunk = 0;
    uint4 wf[2][FO], xf[2][FP];
    unsigned ws[FO], oldW[FO], xs[2][FP], oldX[FP], xAt[FP];
    // window pixel, counted from the wave's own, that each half of the wave reads for blocks kb0 and kb1; first pixel of a lane
    const auto pixelOf = [&](int kb0, int kb1, int& b) {
        int at[2], block[2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
        {
            const int kb = min(k ? kb1 : kb0, total - 1), tap = int(byBlocks(unsigned(kb))), ky = int(a.byKw(unsigned(tap)));
            at[k] = ky * w.winW + tap - ky * a.kw;
            block[k] = kb - tap * blocks;
        }
        b = h ? block[1] : block[0];
        return r0 * w.winW + l + (h ? at[1] : at[0]);
    };
    const auto read = [&](int set, int stage, int s) {
#pragma unroll
        for (int i = 0; i < FO; ++i) wf[set][i] = *reinterpret_cast<const uint4*>(dyn + stage + slot(32 * i + l, 4 * h + s));
        int b;
        if (WORDS)
        {
            // a lane's four blocks are of one pixel: their places differ in two bits, and their scales are a word
            if (s == 0)
            {
                const int p0 = pixelOf(chunk * kChunk, chunk * kChunk + 4, b);
                b &= ~3;
#pragma unroll
                for (int j = 0; j < FP; ++j)
                {
                    const int p = p0 + j * w.winW;
                    xAt[j] = kWindow + (unsigned(p * blocks) + place(unsigned(p), unsigned(b))) * 16;
                    xs[0][j] = *reinterpret_cast<const unsigned*>(dyn + kWindow + w.scales + p * blocks + b);
                }
            }
#pragma unroll
            for (int j = 0; j < FP; ++j) xf[set][j] = *reinterpret_cast<const uint4*>(dyn + (xAt[j] ^ unsigned(s * 16)));
        }
        else
        {
            const int p0 = pixelOf(chunk * kChunk + s, chunk * kChunk + 4 + s, b);
#pragma unroll
            for (int j = 0; j < FP; ++j)
            {
                const int p = p0 + j * w.winW;
                xf[set][j] = *reinterpret_cast<const uint4*>(dyn + kWindow + (unsigned(p * blocks) + place(unsigned(p), unsigned(b))) * 16);
                xs[set][j] = dyn[kWindow + w.scales + p * blocks + b];
            }
        }
    };
    const auto readScales = [&](int stage) {
#pragma unroll
        for (int i = 0; i < FO; ++i) ws[i] = *reinterpret_cast<const unsigned*>(dyn + stage + kScales + (32 * i + l) * kChunk + 4 * h);
    };
#define SRX_STEP(S, SET, I, J, WS, XS)                                                                                 \
    acc[I][J] = WORDS ? __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(wf[SET][I]), widen(xf[SET][J]), acc[I][J], 4, 4, S, WS[I], S, XS[J])   \
                      : __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(wf[SET][I]), widen(xf[SET][J]), acc[I][J], 4, 4, S, WS[I], 0, xs[SET][J]);
#define SRX_MULTIPLY(S, SET)                                                                                           \
    _Pragma("unroll") for (int i = 0; i < FO; ++i)                                                                     \
        _Pragma("unroll") for (int j = 0; j < FP; ++j) { SRX_STEP(S, SET, i, j, ws, xs[0]) }

    f32x16 acc[FO][FP];
    for (;;)
    {
        begin();
        next = chunk = 0;
        prepare();
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(i, 0);
        if (!WORDS) loadBytes();
        // the window: codes unit by unit, scales in words or with their codes
        {
            const int pixelBytes = a.blocks * kMxBytes;
            const unsigned rowBytes = unsigned(a.W) * unsigned(pixelBytes);
            const int64_t first = ((int64_t(n) * a.H + y0 - a.padTop) * a.W + x0 - a.padLeft) * a.blocks + part * kChunk;
            const i32x4 xd = descriptor(a.codes + first * kMxBytes, kRange), zd = descriptor(a.scales + first, WORDS ? kRange : kRange >> 4);
            const auto offsetOf = [&](unsigned p) {                     // of a window's pixel, in codes; or kRange
                const unsigned row = w.byWinW(p), col = p - row * unsigned(w.winW);
                const bool in = unsigned(y0 - a.padTop + int(row)) < unsigned(a.H) && unsigned(x0 - a.padLeft + int(col)) < unsigned(a.W);
                return in && p < unsigned(w.winPixels) ? row * rowBytes + col * unsigned(pixelBytes) : kRange;
            };
            const int units = w.winPixels * blocks;
            // all loads first, or (PARTS: the sums are in registers meanwhile) four at a time
            constexpr int kBatch = PARTS ? 4 : kTapsLoads;
            uint8_t z[kBatch];
#pragma unroll 1
            for (int from = 0; from < kTapsLoads && from * kThreads < units; from += kBatch)
            {
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                {
                    const int at = (from + i) * kThreads;
                    if (at + wave * 64 >= units) continue;
                    const unsigned u = at + tid, p = byBlocks(u), o = offsetOf(p);
                    const unsigned off = o == kRange ? kRange : o + place(p, u - p * unsigned(blocks)) * kMxBytes;
                    loadToLds(xd, off, ldsAt + kWindow + (at + wave * 64) * 16);
                    if (!WORDS) z[i] = uint8_t(loadByte(zd, off / kMxBytes));
                }
                if (!WORDS)
                {
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                    {
                        const unsigned u = (from + i) * kThreads + tid, p = byBlocks(u);
                        if (u < unsigned(units)) dyn[kWindow + w.scales + p * unsigned(blocks) + place(p, u - p * unsigned(blocks))] = z[i];
                    }
                }
            }
            if (WORDS)
            {
#pragma unroll PARTS ? 1 : kTapsLoads / 4
                for (int i = 0; i < kTapsLoads / 4; ++i)
                {
                    if (i * kThreads + wave * 64 >= units / 4) continue;
                    const unsigned u = i * kThreads + tid, p = blocks == 8 ? u >> 1 : u, o = offsetOf(p);
                    loadWordToLds(zd, o == kRange ? kRange : o / kMxBytes + (blocks == 8 ? (u & 1) * 4 : 0), ldsAt + kWindow + w.scales + (i * kThreads + wave * 64) * 4);
                }
            }
            else settle(0);
        }
        float* const bias = reinterpret_cast<float*>(dyn + kStage);
        if ((!PARTS || part == 0) && tid < kBO) bias[tid] = a.bias && o0 + tid < a.O ? (float)static_cast<const T*>(a.bias)[o0 + tid] : 0.0f;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (!PARTS || part == 0)
        {
            startAt<FO, FP>(acc, bias, h);
            // the bias has been read by every wave: its place is the second chunk's
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        read(0, 0, 0);
        readScales(0);
        const int chunks = (total + kChunk - 1) / kChunk;
        if (chunks > 1)
        {
            prepare();
#pragma unroll
            for (int i = 0; i < kLoads; ++i) load(i, kStage);
            if (!WORDS) loadBytes();
        }
        int stage = 0;
        for (int c = 1; c < chunks; ++c)
        {
            // (no branch in here: the compiler would move the products behind it)
            read(1, stage, 1);
            __builtin_amdgcn_sched_barrier(0);
            SRX_MULTIPLY(0, 0)
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < FP; ++j) oldX[j] = xs[0][j];
            read(0, stage, 2);
            __builtin_amdgcn_sched_barrier(0);
            prepare();
            SRX_MULTIPLY(1, 1)
            __builtin_amdgcn_sched_barrier(0);
            read(1, stage, 3);
            __builtin_amdgcn_sched_barrier(0);
            SRX_MULTIPLY(2, 0)
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < FO; ++i) oldW[i] = ws[i];
            stage = kStage - stage;
            if (!WORDS) settle(stage);
            // after this the next chunk is there, and this one is in registers in every wave: its place is free
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            ++chunk;
            read(0, stage, 0);
            readScales(stage);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < FO; ++i)
#pragma unroll
                for (int j = 0; j < FP; ++j)
                {
                    SRX_STEP(3, 1, i, j, oldW, oldX)
                    __builtin_amdgcn_sched_barrier(0);
                    constexpr int kN = FO * FP;
#pragma unroll
                    for (int k = kLoads * (i * FP + j) / kN; k < kLoads * (i * FP + j + 1) / kN; ++k) load(k, kStage - stage);
                    __builtin_amdgcn_sched_barrier(0);
                }
            if (!WORDS) loadBytes();
            __builtin_amdgcn_sched_barrier(0);
        }
        const int left = total - chunk * kChunk;
        SRX_MULTIPLY(0, 0)
        if (left > 1)
        {
            read(1, stage, 1);
            SRX_MULTIPLY(1, 1)
            if (left > 2)
            {
                read(0, stage, 2);
                SRX_MULTIPLY(2, 0)
                if (left > 3)
                {
                    read(1, stage, 3);
                    SRX_MULTIPLY(3, 1)
                }
            }
        }
        // every wave has read this part's window and filters (and the loads behind the last chunk have written their zeros)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (!PARTS || ++part == w.parts) break;
    }
#undef SRX_MULTIPLY
#undef SRX_STEP
    finish<T, FO, FP>(a, acc, dyn + wave * 32 * L::kOutRow, o0, lane, [&](int j, uint8_t*& to, int& count) {
        to = static_cast<uint8_t*>(a.out) + (((int64_t(n) * a.H + y0 + r0 + j) * a.W + x0) * a.O + o0) * int64_t(sizeof(T));
        count = y0 + r0 + j < a.H ? min(32, a.W - x0) : 0;
    });
}

// Too few tiles: 96 -> 96 channels, 3x3, 200x200, 175 of them: 9.9 instead of 11.9 us; 180x180, 138: 9.6 instead of 8.3.
template <typename T, int FO>
Launched launchTaps(const ConvMxArgs& args, hipStream_t s)
{
    using L = TapsLds<T, FO>;
    ConvMxArgs a = args;
    TapsArgs w{};
    const int winH = kWinH + a.taps / a.kw - 1;
    if ((int64_t(winH) * a.W + a.kw + kWinW) * a.blocks * kMxBytes >= int64_t(kRange)) return {};
    w.tilesX = (a.W + kWinW - 1) / kWinW;
    w.tilesY = (a.H + kWinH - 1) / kWinH;
    a.tilesO = (a.O + L::kBO - 1) / L::kBO;
    a.tilesP = a.pixels / (a.H * a.W) * w.tilesX * w.tilesY;
    if (int64_t(a.tilesP) * a.tilesO < 160 || int64_t(a.tilesP) * (kWinW * kWinH * 4) > int64_t(a.pixels) * 5) return {};
    const bool words = scalesInWords(a);
    w.parts = (a.blocks + kChunk - 1) / kChunk;
    w.last = a.blocks - (w.parts - 1) * kChunk;
    w.winW = kWinW + a.kw - 1;
    w.winPixels = winH * w.winW;
    const int units = w.winPixels * (w.parts > 1 ? kChunk : w.last);
    w.scales = (units + 63) / 64 * 1024;
    const int lds = L::bytes(w.scales + (words ? (units / 4 + 63) / 64 * 256 : units)), most = 80 << 10;
    if (units > kTapsLoads * kThreads || lds > most) return {};
    w.byLast = Divider(unsigned(w.last));
    w.byTilesX = Divider(unsigned(w.tilesX));
    w.byTilesY = Divider(unsigned(w.tilesY));
    w.byWinW = Divider(unsigned(w.winW));
    a.byTilesO = Divider(unsigned(a.tilesO));
    const int64_t grid = int64_t(a.tilesO) * ((int64_t(a.tilesP) + 7) / 8 * 8);
    if (grid > INT32_MAX) return {};
    const auto launchAs = [&](auto kernel) -> Launched {
        const hipError_t e = dev::ensureDynamicLds(reinterpret_cast<const void*>(kernel), most);
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(kernel, gridOf(grid), dim3(kThreads), lds, s, a, w);
        return hipGetLastError();
    };
    if (w.parts > 1) return words ? launchAs(ConvMxTapsKernel<T, FO, true, true>) : launchAs(ConvMxTapsKernel<T, FO, false, true>);
    return words ? launchAs(ConvMxTapsKernel<T, FO, true, false>) : launchAs(ConvMxTapsKernel<T, FO, false, false>);
}
template <typename T>
Launched launchTaps(int channels, const ConvMxArgs& a, hipStream_t s)
{
    return channels == 128 ? launchTaps<T, 4>(a, s) : channels == 96 ? launchTaps<T, 3>(a, s) : channels == 64 ? launchTaps<T, 2>(a, s) : launchTaps<T, 1>(a, s);
}

}  // namespace

Launched dev::launchConvMxTaps(bool half, int channels, const ConvMxArgs& a, hipStream_t s)
{
    return half ? launchTaps<f16>(channels, a, s) : launchTaps<float>(channels, a, s);
}

}  // namespace srx
