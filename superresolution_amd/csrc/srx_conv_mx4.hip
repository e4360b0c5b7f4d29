// gfx950 kernel of the convolution whose input and filter are held in the 4-bit block form (srx_mx4.h).
//
//   out[pixel][o] = act(bias[o] + sum over taps (i, j) and channels c of in[pixel + (i - padTop, j - padLeft)][c] * w[o][i][j][c])
//
// as an implicit matrix product on v_mfma_scale_f32_32x32x64_f8f6f4: rows = output channels, columns = pixels, and a
// reduction over the blocks of 32 channels of every tap, numbered kb = tap * (blocks of a pixel) + block.  One
// instruction multiplies two blocks: lanes 0-31 hold one of them for 32 rows (or columns), lanes 32-63 the other, 16
// bytes and one scale byte each, so that the two blocks may come from different taps.  fp32 accumulation.
//
// Four kernels, chosen by LaunchConvMx4 (ConvMxTapsKernel is in srx_conv_mx4_taps.hip).  Times here and beside the rules are of the
// kernels themselves, back to back, with fp16 results and operands quantised from normal values; devices differ by 5 - 7 %, and
// operands of all bit patterns cost the wide layers 5 % more (the power limit).
//   ConvMxRowsKernel    few pixels; bound by the latency of one trip to memory and of the join, and up to 15 pixels by the 64 that
//                       its tile has room for where there are many channels.  One row times 4096 x 4096: 5.3 us (8.9 MB of filter:
//                       1.7 TB/s; 1.9 us at what reads alone reach); 16 rows 6.3, 64 rows 8.8.
//   ConvMxWindowKernel  up to 64 channels on large images; bound by the output's bytes.  64 -> 64 channels, 3x3, 1920x1080:
//                       75 - 79 us (336 MB: 4.3 - 4.5 TB/s; 2.0 PFLOP/s).
//   ConvMxTapsKernel    several taps.  512 -> 512 channels, 3x3, 256x256: 74 us, 4.2 PFLOP/s; 256 -> 256: 25, 3.1; 96 -> 96,
//                       960x540: 42 us (126 MB: 3.0 TB/s; 2.0 PFLOP/s), bound by the start and end of its tiles as much as by the
//                       products.
//   ConvMxKernel        everything else.  2048 -> 2048 channels, 1x1, 16384 pixels: 48 us, 2.8 PFLOP/s: one workgroup fits a CU, so
//                       nothing runs beside a tile's first load, its turn through LDS and its stores; 512 -> 512, 65536 pixels:
//                       23 us (103 MB: 4.5 TB/s).
// The matrix units alone reach 6.2 PFLOP/s on operands of all bit patterns held in registers (at the power limit; 7.7 on
// constants), 5.5 where every operand is read from LDS.  Of the 102 us that ConvMxKernel took for 512 -> 512, 3x3, on operands of all
// bit patterns, its loads from memory cost 36 and its reads from LDS 15: L2, LDS and power together bound the wide layers.
#include "srx_conv_mx4.h"

namespace srx {

using namespace dev;

namespace {

// LDS of a tile: the bias, and one or two chunks (rows of codes, words of scales), later the turn of the results.
template <typename T, int THREADS, int BO, int BP, int FO>
struct TileLds
{
    static constexpr int kXWords = (BP * 2 + THREADS - 1) / THREADS, kWWords = (BO * 2 + THREADS - 1) / THREADS;
    static constexpr int kCodes = (BO + BP) * kRow, kXScales = kCodes + kWWords * THREADS * 4, kStage = kXScales + kXWords * THREADS * 4;
    static constexpr int kOutRow = 32 * FO * int(sizeof(T)) + 16;     // bytes of a pixel in the epilogue, padded
    static constexpr int kOut = THREADS / 64 * 32 * kOutRow, kBias = (BO * 4 + 1023) / 1024 * 1024;
    static constexpr int bytes(int chunks) { return kBias + (chunks * kStage > kOut ? chunks * kStage : kOut); }
};

// A workgroup makes BO output channels of BP pixels; a wave makes 32 * FO channels of 32 * FP pixels.
// The reduction goes in chunks of eight blocks through two buffers in LDS: while one is multiplied, the next is on its
// way from memory to the other (one barrier a chunk).
//   WITHIN: no chunk crosses from one tap to the next (each tap's blocks are padded to whole chunks), so that a chunk's
//           tap is found once for all; otherwise blocks are numbered through and every thread finds its own tap.
//   WORDS:  the blocks of a pixel come in fours, so that scales are staged in words of four; otherwise byte by byte.
template <typename T, int THREADS, int BO, int BP, int FO, int FP, bool WITHIN, bool WORDS>
__global__ __launch_bounds__(THREADS, 2) void ConvMxKernel(const ConvMxArgs a)
{
    static_assert(BO * BP == THREADS / 64 * 32 * FO * 32 * FP, "the waves' tiles make the workgroup's");
    constexpr int kPass = THREADS / 8;                                // rows of codes that a pass of all threads stages
    constexpr int kXRows = BP / kPass, kWRows = BO / kPass;
    constexpr int kXWords = (BP * 2 + THREADS - 1) / THREADS, kWWords = (BO * 2 + THREADS - 1) / THREADS;
    using L = TileLds<T, THREADS, BO, BP, FO>;
    constexpr int kCodes = L::kCodes, kStage = L::kStage, kXScales = L::kXScales, kOutRow = L::kOutRow;
    extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
    uint8_t* const lds = dyn + L::kBias;
    float* const sBias = reinterpret_cast<float*>(dyn);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l = lane & 31;
    // Workgroups are dealt round-robin over the 8 XCDs.  Where there are enough pixel tiles, all channel tiles of the same
    // pixels go to one XCD and share its L2 (1x1, 2048 -> 2048 channels, 16384 pixels: 48 instead of 51 us; 512 -> 512, 65536
    // pixels: 22.5 instead of 24.3; 128 -> 512: 18.5 and 18.7); pixels are dealt out singly (one long run of them for each XCD:
    // 12.2 instead of 11.8 for 256 -> 256).
    const unsigned number = blockNumber();
    unsigned tileO, tileP;
    if (a.tilesP >= 64)
    {
        const unsigned turn = number >> 3, round = a.byTilesO(turn);
        tileO = turn - round * a.tilesO;
        tileP = round * 8 + (number & 7);
    }
    else
    {
        tileP = a.byTilesO(number);
        tileO = number - tileP * a.tilesO;
    }
    if (tileP >= unsigned(a.tilesP)) return;
    const int o0 = int(tileO) * BO;
    const int64_t m0 = int64_t(tileP) * BP;
    constexpr int kWavesO = BO / (32 * FO);
    const int wo = (wave % kWavesO) * 32 * FO, wp = (wave / kWavesO) * 32 * FP;
    const unsigned ldsAt = unsigned(uintptr_t((__attribute__((address_space(3))) uint8_t*)lds));

    // Staging.  Codes: eight threads a row; a thread's place in LDS is fixed, so the swizzle picks its block.
    // Scales: two threads a row, four blocks each (WORDS); else with the codes.
    const int sr = tid >> 3, sb = (tid & 7) ^ ((sr >> 1) & 7), zr = tid >> 1, zb = (tid & 1) * 4;
    const int pixelBytes = a.blocks * kMxBytes;
    const unsigned rowBytes = unsigned(a.W) * unsigned(pixelBytes);     // below 2^31 where it is used (!WITHIN)
    const auto place = [&](int64_t m, bool exists, int& y, int& x) {
        const unsigned row = a.byW(unsigned(m));
        x = int(unsigned(m) - row * unsigned(a.W)) - a.padLeft;
        y = exists && m < a.pixels ? int(row - a.byH(row) * unsigned(a.H)) - a.padTop : INT32_MIN / 2;   // never inside
    };
    int y[kXRows], x[kXRows], zy[kXWords], zx[kXWords];                 // of the window's first tap
    unsigned xOff[kXRows], wOff[kWRows], zOff[kXWords], vOff[kWWords];
#pragma unroll
    for (int i = 0; i < kXRows; ++i)
    {
        place(m0 + sr + kPass * i, true, y[i], x[i]);
        xOff[i] = unsigned((sr + kPass * i) * a.blocks + (WITHIN ? sb : 0)) * kMxBytes;
    }
#pragma unroll
    for (int i = 0; i < kWRows; ++i) wOff[i] = o0 + sr + kPass * i < a.O ? unsigned((sr + kPass * i) * a.total + sb) * kMxBytes : kRange;
    if (WORDS)
    {
#pragma unroll
        for (int i = 0; i < kXWords; ++i)
        {
            const int r = zr + THREADS / 2 * i;
            place(m0 + r, r < BP, zy[i], zx[i]);
            zOff[i] = unsigned(r * a.blocks + (WITHIN ? zb : 0));
        }
#pragma unroll
        for (int i = 0; i < kWWords; ++i)
        {
            const int r = zr + THREADS / 2 * i;
            vOff[i] = r < BO && o0 + r < a.O ? unsigned(r * a.total + zb) : kRange;
        }
    }
    const auto inside = [&](int yy, int xx) { return unsigned(yy) < unsigned(a.H) && unsigned(xx) < unsigned(a.W); };

    // The next chunk: tap and block of the pixel (WITHIN), or block of all.  Beyond the last, nothing is read.
    int tap = 0, c0 = 0;
    constexpr int kLoads = kWRows + kXRows + (WORDS ? kWWords + kXWords : 0);
    i32x4 xd, zd, wd, vd;
    unsigned off[kLoads];
    uint8_t xz[kXRows], wz[kWRows];
    // where the next chunk's data are
    const auto prepare = [&]() {
        // the pixels' descriptors start at the window's first tap (of the tile's first pixel) or at the chunk's tap
        int ky = 0, kx = 0;
        if (WITHIN) { ky = int(a.byKw(unsigned(tap))); kx = tap - ky * a.kw; }
        const int64_t first = m0 + int64_t(ky - a.padTop) * a.W + kx - a.padLeft;
        const int kb = WITHIN ? tap * a.blocks + c0 : c0;
        xd = descriptor(a.codes + (first * a.blocks + (WITHIN ? c0 : 0)) * kMxBytes, kRange);
        zd = descriptor(a.scales + first * a.blocks + (WITHIN ? c0 : 0), WORDS ? kRange : kRange >> 4);
        wd = descriptor(a.wCodes + (int64_t(o0) * a.total + kb) * kMxBytes, kRange);
        vd = descriptor(a.wScales + int64_t(o0) * a.total + kb, WORDS ? kRange : kRange >> 4);
        const int limit = WITHIN ? (tap < a.taps ? a.blocks : 0) : a.total;
        const unsigned out = c0 + sb < limit ? 0u : kRange;
        unsigned from = 0;
        if (!WITHIN)
        {
            const int t = int(a.byBlocks(unsigned(c0 + sb)));
            ky = int(a.byKw(unsigned(t)));
            kx = t - ky * a.kw;
            from = unsigned(ky) * rowBytes + unsigned(kx * pixelBytes + (c0 + sb - t * a.blocks) * kMxBytes);
        }
#pragma unroll
        for (int i = 0; i < kWRows; ++i) off[i] = wOff[i] | out;
#pragma unroll
        for (int i = 0; i < kXRows; ++i) off[kWRows + i] = (inside(y[i] + ky, x[i] + kx) ? xOff[i] + from : kRange) | out;
        if (WORDS)
        {
            const unsigned zOut = c0 + zb < limit ? 0u : kRange;
            if (!WITHIN)
            {
                const int t = int(a.byBlocks(unsigned(c0 + zb)));
                ky = int(a.byKw(unsigned(t)));
                kx = t - ky * a.kw;
                from = (unsigned(ky) * rowBytes + unsigned(kx * pixelBytes)) / kMxBytes + unsigned(c0 + zb - t * a.blocks);
            }
#pragma unroll
            for (int i = 0; i < kWWords; ++i) off[kWRows + kXRows + i] = vOff[i] | zOut;
#pragma unroll
            for (int i = 0; i < kXWords; ++i)
                off[kWRows + kXRows + kWWords + i] = (inside(zy[i] + ky, zx[i] + kx) ? zOff[i] + from : kRange) | zOut;
        }
        c0 += kChunk;
        if (WITHIN)
        {
            tap = c0 >= a.blocks ? tap + 1 : tap;
            c0 = c0 >= a.blocks ? 0 : c0;
        }
    };
    // load number i of the prepared chunk
    const auto load = [&](int i, int stage) {
        const unsigned at = ldsAt + stage + wave * 1024, zAt = ldsAt + stage + kCodes + wave * 256;
        if (i < kWRows) loadToLds(wd, off[i], at + i * THREADS * 16);
        else if (i < kWRows + kXRows) loadToLds(xd, off[i], at + BO * kRow + (i - kWRows) * THREADS * 16);
        else if (i < kWRows + kXRows + kWWords) loadWordToLds(vd, off[i], zAt + (i - kWRows - kXRows) * THREADS * 4);
        else loadWordToLds(zd, off[i], zAt + kXScales - kCodes + (i - kWRows - kXRows - kWWords) * THREADS * 4);
    };
    const auto loadBytes = [&]() {
#pragma unroll
        for (int i = 0; i < kWRows; ++i) wz[i] = loadByte(vd, off[i] / kMxBytes);
#pragma unroll
        for (int i = 0; i < kXRows; ++i) xz[i] = loadByte(zd, off[kWRows + i] / kMxBytes);
    };
    const auto loadAll = [&](int stage) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(i, stage);
        if (!WORDS) loadBytes();
    };
    // the bytes of loadBytes() to the chunk's place in LDS
    const auto settle = [&](int stage) {
#pragma unroll
        for (int i = 0; i < kWRows; ++i) lds[stage + kCodes + (sr + kPass * i) * kChunk + sb] = wz[i];
#pragma unroll
        for (int i = 0; i < kXRows; ++i) lds[stage + kXScales + (sr + kPass * i) * kChunk + sb] = xz[i];
    };


    // Step s multiplies the blocks s (lanes 0-31) and 4 + s (lanes 32-63) of the chunk: a lane's four scales are one word.
    uint4 wf[2][FO], xf[2][FP];
    unsigned ws[FO], xs[FP], oldW[FO], oldX[FP];
    const auto read = [&](int set, int stage, int s) {
#pragma unroll
        for (int i = 0; i < FO; ++i) wf[set][i] = *reinterpret_cast<const uint4*>(lds + stage + slot(wo + 32 * i + l, 4 * h + s));
#pragma unroll
        for (int j = 0; j < FP; ++j) xf[set][j] = *reinterpret_cast<const uint4*>(lds + stage + BO * kRow + slot(wp + 32 * j + l, 4 * h + s));
    };
    const auto readScales = [&](int stage) {
#pragma unroll
        for (int i = 0; i < FO; ++i) ws[i] = *reinterpret_cast<const unsigned*>(lds + stage + kCodes + (wo + 32 * i + l) * kChunk + 4 * h);
#pragma unroll
        for (int j = 0; j < FP; ++j) xs[j] = *reinterpret_cast<const unsigned*>(lds + stage + kXScales + (wp + 32 * j + l) * kChunk + 4 * h);
    };
#define SRX_MULTIPLY(S, SET, WS, XS)                                                                                   \
    _Pragma("unroll") for (int i = 0; i < FO; ++i)                                                                     \
        _Pragma("unroll") for (int j = 0; j < FP; ++j)                                                                 \
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(wf[SET][i]), widen(xf[SET][j]), acc[i][j], 4, 4, S, WS[i], S, XS[j]);

    const int chunks = WITHIN ? a.taps * ((a.blocks + kChunk - 1) / kChunk) : (a.total + kChunk - 1) / kChunk;
    prepare();
    loadAll(0);
    for (int o = tid; o < BO; o += THREADS)
        sBias[o] = a.bias && o0 + o < a.O ? (float)static_cast<const T*>(a.bias)[o0 + o] : 0.0f;
    if (!WORDS) settle(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    f32x16 acc[FO][FP];
    startAt<FO, FP>(acc, sBias + wo, h);
    read(0, 0, 0);
    readScales(0);
    if (chunks > 1)
    {
        prepare();
        loadAll(kStage);
    }
    int stage = 0;
    for (int c = 1; c < chunks; ++c)
    {
        // The first step's operands are in set 0; a step's operands are read while the one before is multiplied.
        read(1, stage, 1);
        __builtin_amdgcn_sched_barrier(0);
        SRX_MULTIPLY(0, 0, ws, xs)
        __builtin_amdgcn_sched_barrier(0);
        read(0, stage, 2);
        __builtin_amdgcn_sched_barrier(0);
        // the addresses of the chunk after the next, between the products
        prepare();
        SRX_MULTIPLY(1, 1, ws, xs)
#pragma unroll
        for (int i = 0; i < FO * FP; ++i)
        {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);            // one product,
            __builtin_amdgcn_sched_group_barrier(0x6, 96 / (FO * FP), 0);   // then scalar and vector arithmetic
        }
        __builtin_amdgcn_sched_barrier(0);
        read(1, stage, 3);
        __builtin_amdgcn_sched_barrier(0);
        SRX_MULTIPLY(2, 0, ws, xs)
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < FO; ++i) oldW[i] = ws[i];
#pragma unroll
        for (int j = 0; j < FP; ++j) oldX[j] = xs[j];
        stage = kStage - stage;
        if (!WORDS) settle(stage);
        // after this the next chunk is there, and this one is in registers in every wave: its place is free
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        read(0, stage, 0);
        readScales(stage);
        __builtin_amdgcn_sched_barrier(0);
        // the loads go out between the products
#pragma unroll
        for (int i = 0; i < FO; ++i)
#pragma unroll
            for (int j = 0; j < FP; ++j)
            {
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(wf[1][i]), widen(xf[1][j]), acc[i][j], 4, 4, 3, oldW[i], 3, oldX[j]);
                __builtin_amdgcn_sched_barrier(0);
                constexpr int kN = FO * FP;
#pragma unroll
                for (int k = kLoads * (i * FP + j) / kN; k < kLoads * (i * FP + j + 1) / kN; ++k) load(k, kStage - stage);
                __builtin_amdgcn_sched_barrier(0);
            }
        if (!WORDS) loadBytes();
        __builtin_amdgcn_sched_barrier(0);
    }
    // The last chunk: where three blocks or less are left, they lie in the first steps' lower lanes.
    const int last = WITHIN ? a.blocks - (a.blocks - 1) / kChunk * kChunk : a.total - (a.total - 1) / kChunk * kChunk;
    SRX_MULTIPLY(0, 0, ws, xs)
    if (last > 1)
    {
        read(1, stage, 1);
        SRX_MULTIPLY(1, 1, ws, xs)
        if (last > 2)
        {
            read(0, stage, 2);
            SRX_MULTIPLY(2, 0, ws, xs)
            if (last > 3)
            {
                read(1, stage, 3);
                SRX_MULTIPLY(3, 1, ws, xs)
            }
        }
    }
#undef SRX_MULTIPLY
    // (also the loads of the chunk after the last, which write zeros)
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    uint8_t* mine = lds + wave * 32 * kOutRow;
    finish<T, FO, FP>(a, acc, mine, o0 + wo, lane, [&](int j, uint8_t*& to, int& count) {
        const int64_t m = m0 + wp + 32 * j;
        to = static_cast<uint8_t*>(a.out) + (m * a.O + o0 + wo) * int64_t(sizeof(T));
        count = int(min(int64_t(32), a.pixels - m));
    });
}

// 16 bytes a lane, by the compiler's own count.
__device__ __forceinline__ uint4 loadCodes(i32x4 from, unsigned offset)
{
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(__builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uint64_t(unsigned(from[0])) | uint64_t(unsigned(from[1])) << 32), 0, from[2], from[3]), offset, 0, 0);
    return uint4{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ unsigned loadWord(i32x4 from, unsigned offset)
{
    return __builtin_amdgcn_raw_buffer_load_b32(__builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uint64_t(unsigned(from[0])) | uint64_t(unsigned(from[1])) << 32), 0, from[2], from[3]), offset, 0, 0);
}

// Few pixels: a workgroup makes 16 output channels of 16 * FP pixels on v_mfma_scale_f32_16x16x128_f8f6f4, and its waves
// share the reduction: wave w takes the chunks w, w + WAVES, .. of sixteen blocks, straight from memory into registers, and the
// partial sums are added up in LDS in the waves' order.  Lane l holds row (or column) l & 15; step s multiplies the
// blocks 4 * (l >> 4) + s, so that a lane's four scales are one word and its codes 64 bytes in a row.
template <typename T, int FP, bool WORDS, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void ConvMxRowsKernel(const ConvMxArgs a)
{
    __shared__ __attribute__((aligned(16))) f32x4 part[WAVES][FP][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), q = lane >> 4, l = lane & 15;
    const unsigned tileP = a.byTilesO(blockIdx.x);
    const int o0 = int(blockIdx.x - tileP * a.tilesO) * 16;
    const int64_t m0 = int64_t(tileP) * 16 * FP;
    const int pixelBytes = a.blocks * kMxBytes;
    const unsigned rowBytes = unsigned(a.W) * unsigned(pixelBytes);
    int y[FP], x[FP];
#pragma unroll
    for (int j = 0; j < FP; ++j)
    {
        const int64_t m = m0 + 16 * j + l;
        const unsigned row = a.byW(unsigned(m));
        x[j] = int(unsigned(m) - row * unsigned(a.W)) - a.padLeft;
        y[j] = m < a.pixels ? int(row - a.byH(row) * unsigned(a.H)) - a.padTop : INT32_MIN / 2;
    }
    const auto inside = [&](int yy, int xx) { return unsigned(yy) < unsigned(a.H) && unsigned(xx) < unsigned(a.W); };
    const int64_t first = m0 - int64_t(a.padTop) * a.W - a.padLeft;
    const i32x4 xd = descriptor(a.codes + first * pixelBytes, kRange), zd = descriptor(a.scales + first * a.blocks, kRange >> 4);
    const i32x4 wd = descriptor(a.wCodes + int64_t(o0) * a.total * kMxBytes, kRange), vd = descriptor(a.wScales + int64_t(o0) * a.total, kRange >> 4);
    const unsigned wRow = o0 + l < a.O ? unsigned(l * a.total) * kMxBytes : kRange;

    struct Operands
    {
        uint4 w[4], x[FP][4];
        unsigned ws, xs[FP];
    };
    const auto load = [&](Operands& to, int k0) {
        const int kb = k0 + 4 * q;
        unsigned off[FP];
        to.ws = 0;
#pragma unroll
        for (int j = 0; j < FP; ++j) to.xs[j] = 0;
#pragma unroll
        for (int s = 0; s < 4; ++s)
        {
            const unsigned out = kb + s < a.total ? 0u : kRange;
            const unsigned at = (wRow + unsigned(kb + s) * kMxBytes) | out;
            to.w[s] = loadCodes(wd, at);
            if (!WORDS) to.ws |= unsigned(loadByte(vd, at / kMxBytes)) << (8 * s);
            if (!WORDS || s == 0)
            {
                const int t = int(a.byBlocks(unsigned(kb + s))), ky = int(a.byKw(unsigned(t))), kx = t - ky * a.kw;
                const unsigned from = unsigned(ky) * rowBytes + unsigned(kx * pixelBytes + (kb + s - t * a.blocks) * kMxBytes);
#pragma unroll
                for (int j = 0; j < FP; ++j) off[j] = (inside(y[j] + ky, x[j] + kx) ? from + unsigned((16 * j + l) * pixelBytes) : kRange) | out;
            }
#pragma unroll
            for (int j = 0; j < FP; ++j)
            {
                to.x[j][s] = loadCodes(xd, WORDS ? off[j] + s * kMxBytes : off[j]);
                if (!WORDS) to.xs[j] |= unsigned(loadByte(zd, off[j] / kMxBytes)) << (8 * s);
            }
        }
        if (WORDS)
        {
            to.ws = loadWord(vd, ((wRow + unsigned(kb) * kMxBytes) | (kb < a.total ? 0u : kRange)) / kMxBytes);
#pragma unroll
            for (int j = 0; j < FP; ++j) to.xs[j] = loadWord(zd, off[j] / kMxBytes);
        }
    };
    f32x4 acc[FP];
#pragma unroll
    for (int j = 0; j < FP; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const auto multiply = [&](const Operands& o) {
#define SRX_STEP(S)                                                                                                    \
        _Pragma("unroll") for (int j = 0; j < FP; ++j)                                                                 \
            acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(widen(o.w[S]), widen(o.x[j][S]), acc[j], 4, 4, S, o.ws, S, o.xs[j]);
        SRX_STEP(0)
        SRX_STEP(1)
        SRX_STEP(2)
        SRX_STEP(3)
#undef SRX_STEP
    };
    // the next chunk's operands are asked for before the current one is multiplied
    int k0 = wave * 16;
    if (k0 < a.total)
    {
        Operands now, next;
        load(now, k0);
        for (k0 += WAVES * 16; k0 < a.total; k0 += WAVES * 16)
        {
            load(next, k0);
            multiply(now);
            now = next;
        }
        multiply(now);
    }
#pragma unroll
    for (int j = 0; j < FP; ++j) part[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave >= FP) return;
    // a lane holds, for its pixel, output channels 4 * (lane >> 4) ..
    f32x4 sum = part[0][wave][lane];
    const int waves = min(WAVES, (a.total + 15) / 16);
    for (int w = 1; w < waves; ++w) sum += part[w][wave][lane];
    const int64_t m = m0 + 16 * wave + l;
    if (m >= a.pixels) return;
    const int o = o0 + 4 * q;
    T* out = static_cast<T*>(a.out) + m * a.O + o;
    const T* bias = static_cast<const T*>(a.bias);
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (T)activate(sum[k] + (bias && o + k < a.O ? (float)bias[o + k] : 0.0f), a.activation);
    if (o + 4 <= a.O) __builtin_memcpy(out, &v, sizeof(v));
    else
    {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (o + k < a.O) out[k] = v[k];
    }
}

// Whether all taps of all pixels of a tile (of 256 pixels at most) lie within the range of one descriptor.
bool tapsInRange(const ConvMxArgs& a)
{
    return ((int64_t(a.taps / a.kw) * a.W + a.kw + 256) * a.blocks + a.total) * kMxBytes < int64_t(kRange);
}

template <typename T, int FP>
hipError_t launchRows(const ConvMxArgs& args, bool words, hipStream_t s)
{
    ConvMxArgs a = args;
    a.tilesO = (a.O + 15) / 16;
    a.byTilesO = Divider(unsigned(a.tilesO));
    const int64_t grid = int64_t(a.tilesO) * ((int64_t(a.pixels) + 16 * FP - 1) / (16 * FP));
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    const dim3 g(static_cast<unsigned>(grid));
    // Sixteen waves where eight would take several chunks each (1024 -> 1024 channels, 3x3, 8x8: 7.8 us), but for 64 pixels,
    // whose operands do not fit a sixteenth of the registers twice.
    if constexpr (FP < 4)
        if (a.total > 8 * 16)
        {
            if (words) hipLaunchKernelGGL((ConvMxRowsKernel<T, FP, true, 16>), g, dim3(1024), 0, s, a);
            else hipLaunchKernelGGL((ConvMxRowsKernel<T, FP, false, 16>), g, dim3(1024), 0, s, a);
            return hipGetLastError();
        }
    if (words) hipLaunchKernelGGL((ConvMxRowsKernel<T, FP, true, 8>), g, dim3(512), 0, s, a);
    else hipLaunchKernelGGL((ConvMxRowsKernel<T, FP, false, 8>), g, dim3(512), 0, s, a);
    return hipGetLastError();
}
template <int FP>
hipError_t launchRows(bool half, const ConvMxArgs& a, hipStream_t s)
{
    return half ? launchRows<f16, FP>(a, scalesInWords(a), s) : launchRows<float, FP>(a, scalesInWords(a), s);
}

// Up to two blocks a pixel: the tiles above would read every pixel once for each tap.  Here a workgroup
// keeps the filters of 32 * FO output channels in LDS, and walks over tiles of 8 rows of 32 pixels: the window that a tile's
// taps see is read once (NL loads of 16 bytes a thread), while the tile before it is multiplied.  A wave makes two rows.
// Block kb of the reduction (tap kb / blocks) of the filters lies at kb * 32 * FO + channel; of the window at pixel * blocks +
// block, with the two blocks of a pixel exchanged in every other eight columns: 16 neighbouring lanes then read all banks.
struct WindowArgs
{
    int winW, units;                  // window columns; window rows * columns * blocks
    int steps;                        // pairs of blocks of the reduction
    int swizzle;                      // two blocks a pixel: eight columns in sixteen have theirs exchanged
    int tilesX, tilesY, tiles, slots; // tiles of all images; workgroups for each channel tile
    Divider byTilesX, byTilesY, byWinRow;
};

template <typename T, int FO, int NL>
struct WindowLds
{
    static constexpr int kBO = 32 * FO, kUnits = NL * kThreads, kOutRow = 32 * FO * int(sizeof(T)) + 16;
    // places: two windows (codes, scales), the turn of the results, bias, table of the window's units, nothing, filters
    static constexpr int kWindow = kUnits * 17, kTurn = 2 * kWindow, kBias = kTurn + 4 * 32 * kOutRow, kTable = kBias + kBO * 4,
                         kNothing = kTable + kUnits * 4, kSteps = kNothing + 32;
    // then, for each step, the lanes' units (for the first wave) and the filters
    __host__ __device__ static constexpr int filters(int steps) { return kSteps + steps * 256; }
    static constexpr int bytes(int steps) { return filters(steps) + 2 * steps * kBO * 17; }
};

template <typename T, int FO, int NL>
__global__ __launch_bounds__(kThreads, 2) void ConvMxWindowKernel(const ConvMxArgs a, const WindowArgs w)
{
    using L = WindowLds<T, FO, NL>;
    constexpr int kBO = L::kBO, FP = 2;
    extern __shared__ __attribute__((aligned(1024))) uint8_t dyn[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, l = lane & 31;
    const unsigned ldsAt = unsigned(uintptr_t((__attribute__((address_space(3))) uint8_t*)dyn));
    // all channel tiles of a slot on one XCD, neighbouring slots on different ones
    const unsigned turn = blockIdx.x >> 3, round = a.byTilesO(turn);
    const int o0 = int(turn - round * a.tilesO) * kBO, slotNumber = int(round * 8 + (blockIdx.x & 7));
    const int pixelBytes = a.blocks * kMxBytes;
    const unsigned rowBytes = unsigned(a.W) * unsigned(pixelBytes);
    const int filters = L::filters(w.steps), filterScales = filters + 2 * w.steps * kBO * 16;

    // the filters, once
    {
        const i32x4 wd = descriptor(a.wCodes + int64_t(o0) * a.total * kMxBytes, kRange), vd = descriptor(a.wScales + int64_t(o0) * a.total, kRange >> 4);
        for (int u = wave * 64; u < 2 * w.steps * kBO; u += kThreads)
        {
            const int kb = (u + lane) / kBO, o = (u + lane) % kBO;
            const unsigned off = kb < a.total && o0 + o < a.O ? unsigned(o * a.total + kb) * kMxBytes : kRange;
            loadToLds(wd, off, ldsAt + filters + u * 16);
            dyn[filterScales + u + lane] = uint8_t(loadByte(vd, off / kMxBytes));
        }
        float* bias = reinterpret_cast<float*>(dyn + L::kBias);
        if (tid < kBO) bias[tid] = a.bias && o0 + tid < a.O ? (float)static_cast<const T*>(a.bias)[o0 + tid] : 0.0f;
        if (tid < 8) reinterpret_cast<unsigned*>(dyn + L::kNothing)[tid] = 0;
        // unit of the window: row, column, block (swizzled), or a row that no image has
        unsigned* table = reinterpret_cast<unsigned*>(dyn + L::kTable);
#pragma unroll
        for (int i = 0; i < NL; ++i)
        {
            const unsigned u = i * kThreads + tid, row = w.byWinRow(u), rest = u - row * unsigned(w.winW * a.blocks);
            const unsigned col = a.byBlocks(rest), block = (rest - col * unsigned(a.blocks)) ^ ((col >> 3) & unsigned(w.swizzle));
            table[u] = int(u) < w.units ? row | col << 8 | block << 16 : 0xffffffffu;
        }
        // Step s multiplies the blocks 2 s (lanes 0-31) and 2 s + 1 (lanes 32-63); an odd reduction's last half step has none.
        for (int u = tid; u < w.steps * 64; u += kThreads)
        {
            const int kb = (u >> 6) * 2 + ((u >> 5) & 1), tap = int(a.byBlocks(unsigned(kb))), ky = int(a.byKw(unsigned(tap)));
            const int px = (u & 31) + tap - ky * a.kw, block = (kb - tap * a.blocks) ^ ((px >> 3) & w.swizzle);
            reinterpret_cast<int*>(dyn + L::kSteps)[u] = kb < a.total ? (ky * w.winW + px) * a.blocks + block : -1;
        }
    }
    __syncthreads();

    uint8_t scale[NL];
    const auto fetch = [&](int tile, int window) {
        const unsigned q = w.byTilesX(unsigned(tile)), n = w.byTilesY(q);
        const int x0 = int(unsigned(tile) - q * unsigned(w.tilesX)) * kWinW - a.padLeft, y0 = int(q - n * unsigned(w.tilesY)) * kWinH - a.padTop;
        const int64_t first = (int64_t(n) * a.H + y0) * a.W + x0;
        const i32x4 xd = descriptor(a.codes + first * pixelBytes, kRange), zd = descriptor(a.scales + first * a.blocks, kRange >> 4);
        const unsigned* table = reinterpret_cast<const unsigned*>(dyn + L::kTable);
#pragma unroll
        for (int i = 0; i < NL; ++i)
        {
            const unsigned t = table[i * kThreads + tid], row = t & 255u, col = (t >> 8) & 255u, block = (t >> 16) & 255u;
            const bool in = int(t) >= 0 && unsigned(y0 + int(row)) < unsigned(a.H) && unsigned(x0 + int(col)) < unsigned(a.W);
            const unsigned off = in ? row * rowBytes + col * unsigned(pixelBytes) + block * kMxBytes : kRange;
            loadToLds(xd, off, ldsAt + window + (i * kThreads + wave * 64) * 16);
            scale[i] = uint8_t(loadByte(zd, off / kMxBytes));
        }
    };

    int window = 0;
    if (slotNumber < w.tiles) fetch(slotNumber, 0);
    for (int tile = slotNumber; tile < w.tiles; tile += w.slots)
    {
#pragma unroll
        for (int i = 0; i < NL; ++i) dyn[window + L::kUnits * 16 + i * kThreads + tid] = scale[i];
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (tile + w.slots < w.tiles) fetch(tile + w.slots, L::kWindow - window);

        f32x16 acc[FO][FP];
        startAt<FO, FP>(acc, reinterpret_cast<const float*>(dyn + L::kBias), h);

        // the next step's operands are read while one is multiplied
        uint4 wf[2][FO], xf[2][FP];
        unsigned ws[2][FO], xs[2][FP];
        const int rowUnits = w.winW * a.blocks;
        const uint8_t* stepAt = dyn + L::kSteps + lane * 4;
        const uint8_t* filterAt = dyn + filters + (h * kBO + l) * 16;
        const uint8_t* filterScaleAt = dyn + filterScales + h * kBO + l;
        const uint8_t* windowAt = dyn + window + 2 * wave * rowUnits * 16;
        const uint8_t* windowScaleAt = dyn + window + L::kUnits * 16 + 2 * wave * rowUnits;
        int unit = *reinterpret_cast<const int*>(stepAt);
        const auto read = [&](int set) {
#pragma unroll
            for (int i = 0; i < FO; ++i)
            {
                wf[set][i] = *reinterpret_cast<const uint4*>(filterAt + 512 * i);
                ws[set][i] = filterScaleAt[32 * i];
            }
            filterAt += 2 * kBO * 16;
            filterScaleAt += 2 * kBO;
#pragma unroll
            for (int j = 0; j < FP; ++j)
            {
                const int u = unit + j * rowUnits;
                xf[set][j] = *reinterpret_cast<const uint4*>(unit < 0 ? dyn + L::kNothing : windowAt + u * 16);
                xs[set][j] = unit < 0 ? dyn[L::kNothing] : windowScaleAt[u];
            }
            stepAt += 256;
            unit = *reinterpret_cast<const int*>(stepAt);               // (after the last step: of the filters, and not used)
        };
#define SRX_MULTIPLY(SET)                                                                                              \
    _Pragma("unroll") for (int i = 0; i < FO; ++i)                                                                     \
        _Pragma("unroll") for (int j = 0; j < FP; ++j)                                                                 \
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(widen(wf[SET][i]), widen(xf[SET][j]), acc[i][j], 4, 4, 0, ws[SET][i], 0, xs[SET][j]);
        read(0);
        int left = w.steps;
        for (; left > 2; left -= 2)
        {
            read(1);
            SRX_MULTIPLY(0)
            read(0);
            SRX_MULTIPLY(1)
        }
        if (left > 1)
        {
            read(1);
            SRX_MULTIPLY(0)
            SRX_MULTIPLY(1)
        }
        else { SRX_MULTIPLY(0) }
#undef SRX_MULTIPLY

        const unsigned q = w.byTilesX(unsigned(tile)), n = w.byTilesY(q);
        const int x0 = int(unsigned(tile) - q * unsigned(w.tilesX)) * kWinW, y0 = int(q - n * unsigned(w.tilesY)) * kWinH + 2 * wave;
        finish<T, FO, FP>(a, acc, dyn + L::kTurn + wave * 32 * L::kOutRow, o0, lane, [&](int j, uint8_t*& to, int& count) {
            to = static_cast<uint8_t*>(a.out) + (((int64_t(n) * a.H + y0 + j) * a.W + x0) * a.O + o0) * int64_t(sizeof(T));
            count = y0 + j < a.H ? min(32, a.W - x0) : 0;
        });
        window = L::kWindow - window;
    }
    // nothing is in flight: the last tile fetched no other
}

// Nothing where the filters or the window do not fit.
template <typename T, int FO, int NL>
Launched launchWindow(const ConvMxArgs& args, WindowArgs w, hipStream_t s)
{
    using L = WindowLds<T, FO, NL>;
    ConvMxArgs a = args;
    a.tilesO = (a.O + L::kBO - 1) / L::kBO;
    a.byTilesO = Divider(unsigned(a.tilesO));
    const void* kernel = reinterpret_cast<const void*>(ConvMxWindowKernel<T, FO, NL>);
    const int lds = L::bytes(w.steps), most = 160 << 10;
    if (lds > most) return {};
    const hipError_t e = dev::ensureDynamicLds(kernel, most);
    if (e != hipSuccess) return e;
    // as many workgroups as the device holds at a time, in eights
    const int perCu = FO == 2 ? 2 : 3;                                  // by registers
    const int resident = 256 * (most / lds < perCu ? most / lds : perCu);
    int slots = (resident / a.tilesO + 7) / 8 * 8;
    if (slots > (w.tiles + 7) / 8 * 8) slots = (w.tiles + 7) / 8 * 8;
    w.slots = slots;
    hipLaunchKernelGGL((ConvMxWindowKernel<T, FO, NL>), dim3(unsigned(slots * a.tilesO)), dim3(kThreads), lds, s, a, w);
    return hipGetLastError();
}
template <typename T, int FO>
Launched launchWindow(const ConvMxArgs& a, hipStream_t s)
{
    // (the rows of a window are eight more than the taps')
    if (a.blocks > 2 || (int64_t(a.taps / a.kw + kWinH) * a.W + a.kw + kWinW) * a.blocks * kMxBytes >= int64_t(kRange)) return {};
    WindowArgs w{};
    const int winH = kWinH + a.taps / a.kw - 1;
    w.winW = kWinW + a.kw - 1;
    w.units = winH * w.winW * a.blocks;
    w.steps = (a.total + 1) / 2;
    w.swizzle = a.blocks == 2 ? 1 : 0;
    w.tilesX = (a.W + kWinW - 1) / kWinW;
    w.tilesY = (a.H + kWinH - 1) / kWinH;
    w.tiles = a.pixels / (a.H * a.W) * w.tilesX * w.tilesY;
    w.byTilesX = Divider(unsigned(w.tilesX));
    w.byTilesY = Divider(unsigned(w.tilesY));
    w.byWinRow = Divider(unsigned(w.winW * a.blocks));
    if (w.units <= 2 * kThreads) return launchWindow<T, FO, 2>(a, w, s);
    if (w.units <= 4 * kThreads) return launchWindow<T, FO, 4>(a, w, s);
    if (w.units <= 7 * kThreads) return launchWindow<T, FO, 7>(a, w, s);
    return {};
}

template <typename T, int THREADS, int BO, int BP, int FO, int FP>
hipError_t launch(const ConvMxArgs& args, hipStream_t s)
{
    ConvMxArgs a = args;
    a.tilesO = (a.O + BO - 1) / BO;
    a.byTilesO = Divider(unsigned(a.tilesO));
    a.tilesP = int((int64_t(a.pixels) + BP - 1) / BP);
    const int64_t grid = int64_t(a.tilesO) * (a.tilesP >= 64 ? (a.tilesP + 7) / 8 * 8 : a.tilesP);
    if (grid > INT32_MAX) return hipErrorInvalidValue;
    const dim3 g = gridOf(grid), block(THREADS);
    const bool within = a.taps == 1 || a.blocks % kChunk == 0 || !tapsInRange(a), words = scalesInWords(a);
    // one chunk needs one buffer: more workgroups fit a CU (8 -> 416 channels, 1x7, 100500 pixels: 24 instead of 33 us)
    const int chunks = within ? a.taps * ((a.blocks + kChunk - 1) / kChunk) : (a.total + kChunk - 1) / kChunk;
    const int lds = TileLds<T, THREADS, BO, BP, FO>::bytes(chunks > 1 ? 2 : 1);
    const auto launchAs = [&](auto kernel) {
        const hipError_t e = dev::ensureDynamicLds(reinterpret_cast<const void*>(kernel), TileLds<T, THREADS, BO, BP, FO>::bytes(2));
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(kernel, g, block, lds, s, a);
        return hipGetLastError();
    };
    if (within && words) return launchAs(ConvMxKernel<T, THREADS, BO, BP, FO, FP, true, true>);
    if (within) return launchAs(ConvMxKernel<T, THREADS, BO, BP, FO, FP, true, false>);
    if (words) return launchAs(ConvMxKernel<T, THREADS, BO, BP, FO, FP, false, true>);
    return launchAs(ConvMxKernel<T, THREADS, BO, BP, FO, FP, false, false>);
}

template <int THREADS, int BO, int BP, int FO, int FP>
hipError_t launch(bool half, const ConvMxArgs& a, hipStream_t s)
{
    return half ? launch<f16, THREADS, BO, BP, FO, FP>(a, s) : launch<float, THREADS, BO, BP, FO, FP>(a, s);
}

}  // namespace

hipError_t LaunchConvMx4(const ML::Operator& op, const uint8_t* codes, const uint8_t* scales, const uint8_t* filterCodes,
                         const uint8_t* filterScales, const void* bias, void* out, hipStream_t s)
{
    if (op.kind != ML::Operator::Kind::CONVOLUTION_MX4 || !codes || !scales || !filterCodes || !filterScales || !out ||
        ((reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(filterCodes)) & 15))
        return hipErrorInvalidValue;
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
    a.stream = int64_t(a.pixels) * a.O * (op.dataType == ML::TensorDataType::FLOAT16 ? 2 : 4) > kStreamBytes;
    const bool half = op.dataType == ML::TensorDataType::FLOAT16;
    const auto tiles = [&](int64_t o, int64_t p) { return (a.O + o - 1) / o * ((a.pixels + p - 1) / p); };

    // Few pixels: the shared reduction (ConvMxRowsKernel), as wide as 256 workgroups allow, while what its workgroups read
    // (their number times 1 + FP rows of 16) takes less time than the chunks of a tile take one after the other.
    // 4096 -> 4096 channels, 1x1: 5.3 (1 pixel), 6.3 (16), 8.8 (64) us instead of 9.5, 9.7, 9.7 with tiles; 31 instead of 10.3
    // for 256 pixels.  256 -> 256 channels, 3x3, 16x16: 4.0 instead of 6.7; 1024 -> 1024, 3x3, 8x8: 8.0 instead of 18.
    // (256: the CUs of the device, here and in the thresholds below, which are those of the measured crossings.)
    const int rows = tiles(16, 64) >= 256 ? 4 : tiles(16, 32) >= 256 ? 2 : 1;
    if (tiles(16, 16 * rows) * (1 + rows) < 1560 && tapsInRange(a))
        return rows == 4 ? launchRows<4>(half, a, s) : rows == 2 ? launchRows<2>(half, a, s) : launchRows<1>(half, a, s);
    const auto padded = [&](int64_t o) { return (a.O + o - 1) / o * o; };
    // Up to 64 channels on large images: the window kernel.  64 -> 64 channels, 3x3: 79 us for 1920x1080 instead of 104 with
    // ConvMxTapsKernel, 14.5 and 14.0 for 640x360 (900 tiles); 1x1, 1920x1080: 63 instead of 88 with tiles.  32 -> 32, 3x3, 512x512:
    // 8.4 instead of 9.5, 32 -> 128: 18.4 instead of 19.5; with more channel tiles the window is read as often as the tiles read
    // it (64 -> 256, 3x3, 256x256: 14.7 and 15.9).  fp32 results leave room for 32 channels at a time only (960x540: 31 instead of
    // 33).
    if (a.blocks <= 2 && a.O <= 128 && (a.taps == 1 || padded(64) <= padded(96)) && a.W >= kWinW && a.H >= kWinH && tiles(64, 256) >= 768)
    {
        const Launched e = !half ? launchWindow<float, 1>(a, s) : a.O <= 32 ? launchWindow<f16, 1>(a, s) : launchWindow<f16, 2>(a, s);
        if (e) return *e;
    }
    // Several taps: the window staged once (launchConvMxTaps refuses where tiles are few or empty), with the tile that computes least
    // beyond what is needed; a tile of 96 channels takes a twentieth longer for a channel than one of 128, one of 64 a quarter, but
    // in short reductions, where the output takes the time, the smaller ones win (32 -> 384, 3x3, 512x512: 44 instead of 49 us;
    // 32 -> 300: 43 instead of 52).  3x3, instead of tiles that read every pixel for every tap: 96 -> 96, 960x540: 42 instead of 74
    // us; 128 -> 128, 512x512: 30 instead of 38; 96 -> 64: 17 instead of 26; 96 -> 32: 13.4 instead of 19; 160 -> 160, 256x256: 18
    // instead of 21; 256 -> 256: 25 instead of 28; 384 -> 384: 50 instead of 66; 512 -> 512: 74 instead of 80; 64 -> 96, 512x512:
    // 21 instead of 25 with the window kernel.
    if (a.taps > 1)
    {
        const bool brief = a.total <= 2 * kChunk;
        const int64_t by128 = padded(128) * 20, by96 = padded(96) * (brief ? 19 : 21), by64 = padded(64) * (brief ? 18 : 25);
        const Launched e = a.O <= 32                          ? launchConvMxTaps(half, 32, a, s)
                           : by128 <= by96 && by128 <= by64 ? launchConvMxTaps(half, 128, a, s)
                           : by96 <= by64                     ? launchConvMxTaps(half, 96, a, s)
                                                              : launchConvMxTaps(half, 64, a, s);
        if (e) return *e;
    }
    // The largest tile that leaves no CU without one: 256x256 reads half of what 128x128 does (2048 -> 2048 channels, 1x1,
    // 16384 pixels: 50 instead of 62 us), but 64 such tiles for 2048 pixels take 19 instead of 12.
    // 128x128: 13.0 instead of 15.3 us with 128x64 for 1024 -> 96, 1x1, 65536 pixels; 9.5 instead of 8.0 for half as many (256
    // tiles).  32x128: 27.5 instead of 29.4 with 64x64 for 1024 -> 32, 1x1, 262144 pixels; 42 instead of 54 for 288 -> 32, 3x3.
    // Channels that only fill up a tile count: 1024 -> 160, 1x1, 65536 pixels in 256: 18.4 instead of 21 us, but 8 -> 416, 1x7, one
    // row of 100500 pixels in 512: 34 instead of 24 (nothing but the output takes time there).
    const bool deep = a.total > 2 * kChunk;
    if (a.O > 128 && tiles(256, 256) >= 256 && padded(256) * 10 <= padded(64) * (deep ? 14 : 10)) return launch<512, 256, 256, 4, 2>(half, a, s);
    if (a.O > 64 && padded(128) * 10 <= padded(64) * (deep ? 14 : 10))
    {
        if (tiles(128, 128) >= 512) return launch<256, 128, 128, 2, 2>(half, a, s);
        if (tiles(128, 64) >= 512) return launch<256, 128, 64, 2, 1>(half, a, s);
    }
    if (a.O <= 32 && tiles(32, 128) >= 256) return launch<256, 32, 128, 1, 1>(half, a, s);
    if (tiles(64, 128) >= 1024) return launch<256, 64, 128, 1, 2>(half, a, s);
    return launch<256, 64, 64, 1, 1>(half, a, s);
}

}  // namespace srx
