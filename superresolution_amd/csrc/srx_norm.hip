// gfx950 kernels of the group normalisation layer and of the conversions to and from the 4-bit block form
// (srx_mx4.h).  Tensors are dense and channels last: {N, C, H, W} held as [N][H][W][C].
//
// Group normalisation of image n, group g (the C/G channels g*C/G ..):
//     mean = avg(x),  var = avg((x - mean)^2)  over the group's channels of every pixel
//     y = act((x - mean) / sqrt(var + epsilon) * scale[c] + bias[c])
// Statistics are kept as (mean, M2 = sum of squared deviations) of a part of the data and joined by
//     M2 = sum M2_i + sum n_i (mean_i - mean)^2,
// so nothing cancels when the mean is large against the deviation.  Everything is fp32, rounded once when stored, but for the
// statistics' sums of fp32 tensors and of groups wider than a workgroup, which are fp64 (NormStatsKernel).
//
// Times of the kernels themselves, and what bounds them (a large copy reaches 4.9 TB/s here, reads alone 6.4, writes 6.8):
//   NormSlabKernel       512 channels of 16x16 pixels, fp16, SiLU: 5.0 us; one trip to memory, two joins in LDS.
//   NormStatsKernel      64 channels of 1920x1080, fp16: 50 us, 5.3 TB/s of reads; fp32: 103 us, 5.2.  4096 channels of 64x64
//                        pixels in one group, fp16: 13.5 us, 2.5 TB/s (one load in flight a thread).
//   NormApplyKernel      the same: 89 us, 6.0 TB/s of reads (half of them still cached) and writes; fp32: 229.  256 channels of
//                        256x256 to 4 bits: 9.5 + 13.8 us, 3.5 TB/s and 3.1 from the last-level cache; the output's 18 vector
//                        instructions a value with SiLU take 71 % of the cycles that its CUs are busy.
//   QuantizeKernel, DequantizeKernel   133 M values in fp16: 62 us (5.4 TB/s) and 48 us (6.9 TB/s): memory.
#include "srx_mx4.h"

namespace srx {

using namespace dev;

namespace {

constexpr int kVec = 8;               // channels of one thread
constexpr int kTileC = kThreads * kVec;
constexpr int kJoin = 64;             // parts of an image that every workgroup of NormApplyKernel joins by itself

struct NormArgs
{
    const void *in, *scale, *bias;
    void* out;
    uint8_t *codes, *scales;
    float2* partial;                  // [N][G][chunks] (mean, M2)
    float2* joined;                   // [N][G] (mean, 1 / deviation), where chunks > kJoin
    int64_t pixels, values;           // H * W; N * H * W * C
    int C, G, groupC;                 // channels, groups, channels of a group
    int chunks, chunkPixels;          // statistics: parts of an image
    int tileGroups, tiles;            // whole groups per workgroup (statistics, slabs)
    int applyChunks, applyPixels, applyTiles;
    int groupsInAll;                  // N * G
    int blocks, first;                // workgroups, number of this launch's first one
    int slabRows;                     // pixels that the threads of a slab hold at a time
    Divider byTiles, byChunks, byGroupC, byVecs;
    float epsilon;
    int activation;
    int stream;                       // the output passes by the caches
};

// Eight values as they are held in memory: registers that wait for the statistics take half the room in fp16.
template <typename T> struct Held;
template <> struct Held<f16>
{
    f16x8 v;
    __device__ void load(const f16* p) { __builtin_memcpy(&v, p, 16); }
    __device__ void set(int i, float x) { v[i] = (f16)x; }
    __device__ float get(int i) const { return (float)v[i]; }
};
template <> struct Held<float>
{
    f32x4 a, b;
    __device__ void load(const float* p) { __builtin_memcpy(&a, p, 16); __builtin_memcpy(&b, p + 4, 16); }
    __device__ void set(int i, float x) { if (i < 4) a[i & 3] = x; else b[i & 3] = x; }
    __device__ float get(int i) const { return i < 4 ? a[i & 3] : b[i & 3]; }
};
// As loadUpTo8.
template <typename T>
__device__ __forceinline__ void loadHeld(const T* p, int count, const T* end, Held<T>& v)
{
    if (count >= kVec || (count > 0 && p + kVec <= end)) { v.load(p); return; }
#pragma unroll
    for (int i = 0; i < kVec; ++i) v.set(i, i < count ? (float)p[i] : 0.0f);
}

template <int CONTROL>
__device__ __forceinline__ float moved(float v)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CONTROL, 0xf, 0xf, true));
}
// Sum over the `lanes` (a power of two up to 64, the same in the whole wave) lanes of an aligned part of a wave, in each
// of them: neighbours, pairs, then mirrored halves of 8 and 16, and the exchanges of 16 and 32 lanes.
__device__ __forceinline__ float sumLanes(float v, int lanes)
{
    if (lanes > 1) v += moved<0xB1>(v);
    if (lanes > 2) v += moved<0x4E>(v);
    if (lanes > 4) v += moved<0x141>(v);
    if (lanes > 8) v += moved<0x140>(v);
    if (lanes > 16)
    {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if (lanes > 32)
    {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// Sum over a workgroup of kThreads, in each of its threads.  `waves` holds a value of each wave, of this call alone.
__device__ __forceinline__ double sumThreads(double v, double* waves)
{
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) v += __shfl_xor(v, i);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) v += waves[i];
    return v;
}

// What a thread's sums about a value of its own are held in.  fp32 values may lie so far apart that squares of 256 times the
// distance pass the range of fp32 while the sum of their squared deviations does not; fp16 values cannot.
template <typename T> struct SumOf { typedef double type; };
template <> struct SumOf<f16> { typedef float type; };

// Sum of squared deviations from sums about another point: rounding may leave it below zero, a NaN stays one.
template <typename S>
__device__ __forceinline__ float spread(S squares, S sum, S inverseCount)
{
    const S m2 = squares - sum * (sum * inverseCount);
    return m2 < S(0) ? 0.0f : float(m2);
}

// 1 / sqrt(v): the special function unit's estimate (one part in 2^22) and one Newton step.  An infinity, which stands for a
// variance past the range of fp32, gives NaN (the estimate is zero: normalised values would all be the bias).
__device__ __forceinline__ float inverseRoot(float v)
{
    const float r = __builtin_amdgcn_rsqf(v);
    return fmaf(0.5f * r, fmaf(-v * r, r, 1.0f), r);
}

// Threads that share one group's reduction when `threads` of them reduce `groups` groups.
__device__ __forceinline__ int lanesPerGroup(int groups, int threads)
{
    int lanes = 64;
    while (lanes > 1 && lanes * groups > threads) lanes >>= 1;
    return lanes;
}

// f(activation as a constant): the branch is taken once, not for every value.
template <int ACT> struct Constant { static constexpr int value = ACT; };
template <typename F>
__device__ __forceinline__ void forActivation(int activation, F&& f)
{
    if (activation == 0) f(Constant<0>{});
    else if (activation == 1) f(Constant<1>{});
    else f(Constant<2>{});
}

// What a thread needs to finish its eight channels, and the finish.
template <typename T>
struct Finish
{
    // y = (x - mean) * mul + add with mul = scale / deviation, add = bias.  (x * mul + (bias - mean * mul) would be an operation
    // less, but off by half a step of mean / deviation where x is near the mean.)
    float mean[kVec], mul[kVec], add[kVec];
    Held<T> scale, bias;
    // the parameters of m channels from c on: asked for early, used in prepare()
    __device__ __forceinline__ void load(const NormArgs& a, int m, int c)
    {
        if (a.scale) loadHeld(static_cast<const T*>(a.scale) + c, m, static_cast<const T*>(a.scale) + a.C, scale);
        if (a.bias) loadHeld(static_cast<const T*>(a.bias) + c, m, static_cast<const T*>(a.bias) + a.C, bias);
    }
    // stat: (mean, 1 / deviation) of group g0 and the following ones
    __device__ __forceinline__ void prepare(const NormArgs& a, const float2* stat, int g0, int m, int c)
    {
        int g = int(a.byGroupC(unsigned(min(c, a.C - 1)))), left = (g + 1) * a.groupC - c;
#pragma unroll
        for (int i = 0; i < kVec; ++i)
        {
            if (i == left && i < m) { ++g; left += a.groupC; }
            const float2 st = stat[g - g0];
            mul[i] = a.scale ? st.y * scale.get(i) : st.y;
            mean[i] = st.x;
            add[i] = a.bias ? bias.get(i) : 0.0f;
        }
    }
    // m channels exist
    template <bool MX4, int ACT>
    __device__ __forceinline__ void store(const NormArgs& a, const Held<T>& x, int m, T* out, uint8_t* codes, uint8_t* scaleOf) const
    {
        float v[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = activate(fmaf(x.get(i) - mean[i], mul[i], add[i]), ACT);
        if (MX4)
        {
            if (m < kVec)
            {
#pragma unroll
                for (int i = 0; i < kVec; ++i) v[i] = i < m ? v[i] : 0.0f;
            }
            unsigned s;
            *reinterpret_cast<unsigned*>(codes) = mxQuantise(v, s);
            if ((threadIdx.x & 3) == 0) *scaleOf = uint8_t(s);         // rows of threads are whole blocks
        }
        else if (a.stream && m == kVec) streamOut8(out, v);
        else storeUpTo8(out, m, v);
    }
};

// Where a thread's eight channels from c on of a pixel (counted over all images) go, and of the pixels `rows` further on.
template <typename T>
struct Target
{
    T* out;
    uint8_t *codes, *scales;
    int64_t step, blocks;
    __device__ __forceinline__ Target(const NormArgs& a, int64_t pixel, int c, int rows)
        : out(static_cast<T*>(a.out) + pixel * a.C + c), codes(a.codes + (pixel * mxBlocks(a.C) + (c >> 5)) * kMxBytes + ((c >> 1) & 12)),
          scales(a.scales + pixel * mxBlocks(a.C) + (c >> 5)), step(int64_t(rows) * a.C), blocks(rows * mxBlocks(a.C)) {}
    template <bool MX4, int ACT>
    __device__ __forceinline__ void store(const NormArgs& a, const Finish<T>& f, const Held<T>& x, int m, int u) const
    {
        f.template store<MX4, ACT>(a, x, m, out + u * step, codes + u * blocks * kMxBytes, scales + u * blocks);
    }
    __device__ __forceinline__ void advance(int u)
    {
        out += u * step;
        codes += u * blocks * kMxBytes;
        scales += u * blocks;
    }
};

// Threads of a row of `channels` channels; whole blocks of 32 take four threads each.
template <bool MX4>
__host__ __device__ __forceinline__ int vecsFor(int channels)
{
    return MX4 ? ((channels + 31) >> 5) << 2 : (channels + kVec - 1) / kVec;
}

// Small images: one workgroup holds a slab, all pixels of a range of whole groups of one image, in registers (R eighths
// a thread), takes mean and variance one after the other, and stores.  One launch, one trip to memory.
template <typename T, bool MX4, int THREADS, int R>
__global__ __launch_bounds__(THREADS) void NormSlabKernel(const NormArgs a)
{
    __shared__ __attribute__((aligned(16))) float sPart[THREADS * kVec];
    __shared__ float sTeam[THREADS];
    __shared__ float2 sStat[THREADS * kVec];
    const unsigned number = unsigned(a.first) + blockNumber();
    const int tid = threadIdx.x, n = int(a.byTiles(number)), tile = int(number) - n * a.tiles;
    const int g0 = tile * a.tileGroups, groups = min(a.tileGroups, a.G - g0);
    const int c0 = g0 * a.groupC, tileC = groups * a.groupC;
    // (the last tile may be narrower: its threads keep the others' places)
    const int vecs = int(a.byVecs.d), row = int(a.byVecs(unsigned(tid))), rows = a.slabRows, col = tid - row * vecs;
    const int m = row < rows ? max(0, min(kVec, tileC - col * kVec)) : 0;
    const int c = c0 + col * kVec, pixels = int(a.pixels);
    const T* in = static_cast<const T*>(a.in) + int64_t(n) * pixels * a.C + c;
    const T* end = static_cast<const T*>(a.in) + a.values;
    Held<T> x[R];
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (row + i * rows < pixels) loadHeld(in + int64_t(row + i * rows) * a.C, m, end, x[i]);
    Finish<T> f;
    f.load(a, m, c);

    const float inv = 1.0f / (float(pixels) * float(a.groupC));
    // put(g, sum of v over group g): by one thread for each group, seen by all afterwards.  One group: sums of waves.
    // Several: lanes x slices threads add up each group's values, then the slices are added up.
    const int lanes = lanesPerGroup(a.tileGroups, THREADS), lane = tid & (lanes - 1), team = tid / lanes;
    const int slices = max(1, THREADS / lanes / a.tileGroups), slice = slices > 1 ? team / a.tileGroups : 0;
    // Where a group is whole eighths, a thread adds up its eight channels first.
    const int per = a.groupC % kVec == 0 ? 1 : kVec;
    const int rowValues = vecs * per, groupValues = per == 1 ? a.groupC / kVec : a.groupC;
    const int first = slice * lanes + lane, step = slices * lanes;
    const int r0 = first / groupValues, k0 = first - r0 * groupValues, dr = step / groupValues, dk = step - dr * groupValues;
    const auto total = [&](const float (&v)[kVec], auto&& put) {
        const float own = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        if (a.tileGroups == 1)
        {
            const float w = sumLanes(own, 64);
            __syncthreads();                                            // (sTeam of the call before has been read)
            if ((tid & 63) == 0) sTeam[tid >> 6] = w;
            __syncthreads();
            float all = 0.0f;
#pragma unroll
            for (int i = 0; i < THREADS / 64; ++i) all += sTeam[i];
            if (tid == 0) put(0, all);
            __syncthreads();
            return;
        }
        if (row < rows)
        {
            if (per == 1) sPart[tid] = own;
            else
            {
#pragma unroll
                for (int i = 0; i < kVec; ++i) sPart[tid * kVec + i] = v[i];
            }
        }
        __syncthreads();
        if (slice < slices)
            for (int g = team - slice * a.tileGroups; g < groups; g += THREADS / lanes)
            {
                float sum = 0.0f;
                for (int r = r0, k = k0; r < rows;)
                {
                    sum += sPart[r * rowValues + g * groupValues + k];
                    k += dk;
                    r += dr;
                    if (k >= groupValues) { k -= groupValues; ++r; }
                }
                sum = sumLanes(sum, lanes);
                if (lane == 0 && slices == 1) put(g, sum);
                if (lane == 0 && slices > 1) sTeam[slice * a.tileGroups + g] = sum;
            }
        __syncthreads();
        if (slices > 1)
        {
            if (tid < groups)
            {
                float all = 0.0f;
                for (int i = 0; i < slices; ++i) all += sTeam[i * a.tileGroups + tid];
                put(tid, all);
            }
            __syncthreads();
        }
    };
    float s[kVec], mean[kVec];
#pragma unroll
    for (int k = 0; k < kVec; ++k) s[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (row + i * rows < pixels)
        {
#pragma unroll
            for (int k = 0; k < kVec; ++k) s[k] += k < m ? x[i].get(k) : 0.0f;
        }
    total(s, [&](int g, float sum) { sStat[g].x = sum * inv; });
    if (m > 0)
    {
        int g = int(a.byGroupC(unsigned(col * kVec))), left = (g + 1) * a.groupC - col * kVec;
#pragma unroll
        for (int k = 0; k < kVec; ++k)
        {
            if (k == left && k < m) { ++g; left += a.groupC; }
            mean[k] = sStat[g].x;
        }
    }
#pragma unroll
    for (int k = 0; k < kVec; ++k) s[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (row + i * rows < pixels)
        {
#pragma unroll
            for (int k = 0; k < kVec; ++k)
            {
                const float d = k < m ? x[i].get(k) - mean[k] : 0.0f;
                s[k] = fmaf(d, d, s[k]);
            }
        }
    total(s, [&](int g, float sum) { sStat[g].y = inverseRoot(fmaf(sum, inv, a.epsilon)); });
    // (in the last tile, whose threads may be more than its blocks', the others would write into the next pixel)
    if (row >= rows || col >= vecsFor<MX4>(tileC)) return;
    f.prepare(a, sStat, g0, m, c);
    const Target<T> to(a, int64_t(n) * pixels + row, c, rows);
    forActivation(a.activation, [&](auto act) {
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (row + i * rows < pixels) to.template store<MX4, act.value>(a, f, x[i], m, i);
    });
}

// Statistics of one part of one image for a range of whole groups.  A thread keeps eight channels and walks the
// part's pixels; sums are of x - (its first value of the channel), whose magnitude the part's own spread bounds.
// WHOLE: no group range and no pixel ends inside eight channels.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) void NormStatsKernel(const NormArgs a)
{
    __shared__ __attribute__((aligned(16))) float sMean[kTileC], sM2[kTileC];
    const unsigned number = unsigned(a.first) + blockNumber();
    const int b = int(a.byTiles(number)), tile = int(number) - b * a.tiles;
    const int n = int(a.byChunks(unsigned(b))), chunk = b - n * a.chunks;
    const int g0 = tile * a.tileGroups, groups = min(a.tileGroups, a.G - g0);
    const int c0 = g0 * a.groupC, tileC = groups * a.groupC;
    const int64_t p0 = int64_t(chunk) * a.chunkPixels;
    const int count = int(min(int64_t(a.chunkPixels), a.pixels - p0));
    const T* in = static_cast<const T*>(a.in) + (n * a.pixels + p0) * a.C + c0;
    const T* end = static_cast<const T*>(a.in) + a.values;
    float2* out = a.partial + (int64_t(n) * a.G + g0) * a.chunks + chunk;
    const int tid = threadIdx.x, vecs = (tileC + kVec - 1) / kVec;

    if (vecs > kThreads)
    {
        // One group wider than a workgroup: every value belongs to it, and a thread adds up thousands of them about its first one.
        // In 32 bits the rounding of those sums would drown the spread where the first value is far from the others.
        // (The sums are kept in halves, which do not wait for each other.)
        double k = 0.0, s[2] = {0.0, 0.0}, q[2] = {0.0, 0.0};
        int have = 0;
        for (int p = 0; p < count; ++p)
            for (int col = tid; col < vecs; col += kThreads)
            {
                float v[kVec];
                const int m = min(kVec, tileC - col * kVec);
                loadUpTo8(in + int64_t(p) * a.C + col * kVec, m, end, v);
                if (have == 0) k = v[0];
                have += m;
#pragma unroll
                for (int i = 0; i < kVec; ++i)
                {
                    const double d = i < m ? v[i] - k : 0.0;
                    s[i & 1] += d;
                    q[i & 1] = fma(d, d, q[i & 1]);
                }
            }
        // (vecs > kThreads: every thread has values)
        const double inverse = 1.0 / have, sum = s[0] + s[1], mean = k + sum * inverse;
        const double all = sumThreads(have * k + sum, reinterpret_cast<double*>(sMean)) / (double(count) * tileC), d = mean - all;
        const double m2 = sumThreads(double(spread(q[0] + q[1], sum, inverse)) + have * d * d, reinterpret_cast<double*>(sM2));
        if (tid == 0) out[0] = float2{float(all), float(m2)};
        return;
    }

    const int rows = kThreads / vecs, row = tid / vecs, col = tid - row * vecs;
    if (row < rows)
    {
        const int m = min(kVec, tileC - col * kVec);
        const T* src = in + col * kVec;
        typedef typename SumOf<T>::type Sum;
        float k[kVec];
        Sum s[kVec], q[kVec];
        // The odd pixels first, then whole batches, the next of which is asked for before the current one is summed up.
        constexpr int kFlight = 4;
        const int mine = row < count ? (count - row + rows - 1) / rows : 0, odd = mine % kFlight;
        const int64_t step = int64_t(rows) * a.C;
        const T* at = src + int64_t(row) * a.C;
        Held<T> first[kFlight - 1], v[kFlight];
        const auto load = [&](Held<T>& to, const T* from) {
            if (WHOLE) to.load(from);
            else loadHeld(from, m, end, to);
        };
        const auto sum = [&](const Held<T>& x) {
#pragma unroll
            for (int i = 0; i < kVec; ++i) { const Sum d = x.get(i) - k[i]; s[i] += d; q[i] = __builtin_elementwise_fma(d, d, q[i]); }
        };
#pragma unroll
        for (int u = 0; u < kFlight - 1; ++u)
            if (u < odd) load(first[u], at + u * step);
        at += odd * step;
        if (mine >= kFlight)
        {
#pragma unroll
            for (int u = 0; u < kFlight; ++u) load(v[u], at + u * step);
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) { k[i] = odd ? first[0].get(i) : (mine ? v[0].get(i) : 0.0f); s[i] = q[i] = 0; }
#pragma unroll
        for (int u = 0; u < kFlight - 1; ++u)
            if (u < odd) sum(first[u]);
        int batches = mine / kFlight;
        for (; batches > 1; --batches)
        {
            Held<T> next[kFlight];
            at += kFlight * step;
#pragma unroll
            for (int u = 0; u < kFlight; ++u) load(next[u], at + u * step);
#pragma unroll
            for (int u = 0; u < kFlight; ++u) sum(v[u]);
#pragma unroll
            for (int u = 0; u < kFlight; ++u) v[u] = next[u];
        }
        if (batches > 0)
        {
#pragma unroll
            for (int u = 0; u < kFlight; ++u) sum(v[u]);
        }
        const Sum inv = Sum(1) / Sum(max(1, mine));
#pragma unroll
        for (int i = 0; i < kVec; ++i)
        {
            sMean[(row * vecs + col) * kVec + i] = float(__builtin_elementwise_fma(s[i], inv, Sum(k[i])));
            sM2[(row * vecs + col) * kVec + i] = spread(q[i], s[i], inv);
        }
    }
    __syncthreads();
    // Join the rows and channels of each group: row r has `whole` pixels, and one more below `rest`.
    const int stride = vecs * kVec, whole = count / rows, rest = count - whole * rows, used = min(rows, count);
    const int lanes = lanesPerGroup(groups, kThreads), lane = tid & (lanes - 1);
    const int entries = used * a.groupC;
    for (int g = tid / lanes; g < groups; g += kThreads / lanes)
    {
        float mean = 0.0f, m2 = 0.0f;
        const auto each = [&](auto&& f) {
            for (int e0 = lane; e0 < entries; e0 += 4 * lanes)
            {
#pragma unroll
                for (int u = 0; u < 4; ++u)
                {
                    const int e = min(e0 + u * lanes, entries - 1), r = int(a.byGroupC(unsigned(e)));
                    const float n = e0 + u * lanes < entries ? float(whole + (r < rest ? 1 : 0)) : 0.0f;
                    f(n, r * stride + g * a.groupC + e - r * a.groupC);
                }
            }
        };
        each([&](float n, int at) { mean = fmaf(n, sMean[at], mean); });
        mean = sumLanes(mean, lanes) / (float(count) * float(a.groupC));
        each([&](float n, int at) { const float d = sMean[at] - mean; m2 += n > 0.0f ? fmaf(n * d, d, sM2[at]) : 0.0f; });
        m2 = sumLanes(m2, lanes);
        if (lane == 0) out[int64_t(g) * a.chunks] = float2{mean, m2};
    }
}

// The parts of one group of one image joined by `lanes` lanes: (mean, 1 / deviation).  PER parts of each lane are asked for
// at once and kept.  A lane has more where the output kernel's lanes share over 32 groups (64 parts over four lanes and less), and
// in NormJoinKernel from 1024 parts on (the least that images of over 2^18 pixels of 2048 channels, or 2^26 of 8, come in).
template <int PER>
__device__ __forceinline__ float2 joinParts(const NormArgs& a, const float2* partial, int lane, int lanes)
{
    const float last = float(a.pixels - int64_t(a.chunks - 1) * a.chunkPixels), each = float(a.chunkPixels), all = 1.0f / float(a.pixels);
    const auto pixels = [&](int k) { return k < a.chunks - 1 ? each : (k == a.chunks - 1 ? last : 0.0f); };
    float2 v[PER];
    float mean = 0.0f, m2 = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = lane + i * lanes < a.chunks ? partial[lane + i * lanes] : float2{0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < PER; ++i) mean = fmaf(pixels(lane + i * lanes), v[i].x, mean);
    for (int k = lane + PER * lanes; k < a.chunks; k += lanes) mean = fmaf(pixels(k), partial[k].x, mean);
    mean = sumLanes(mean, lanes) * all;
    const auto join = [&](int k, float2 p) {
        const float d = p.x - mean;
        m2 += k < a.chunks ? fmaf(pixels(k) * float(a.groupC), d * d, p.y) : 0.0f;
    };
#pragma unroll
    for (int i = 0; i < PER; ++i) join(lane + i * lanes, v[i]);
    for (int k = lane + PER * lanes; k < a.chunks; k += lanes) join(k, partial[k]);
    m2 = sumLanes(m2, lanes);
    return float2{mean, inverseRoot(fmaf(m2, all / float(a.groupC), a.epsilon))};
}

// One wave joins the parts of one group.
constexpr int kJoinPer = 16;
__global__ __launch_bounds__(64) void NormJoinKernel(const NormArgs a)
{
    const int group = blockIdx.x;
    const float2 v = joinParts<kJoinPer>(a, a.partial + int64_t(group) * a.chunks, threadIdx.x, 64);
    if (threadIdx.x == 0) a.joined[group] = v;
}

// Normalises, scales, activates and stores (MX4: as 4-bit blocks) a part of an image.
template <typename T, bool MX4, bool WHOLE>
__global__ __launch_bounds__(kThreads) void NormApplyKernel(const NormArgs a)
{
    __shared__ float2 sStat[kTileC];
    // from the last part to the first: the statistics kernel read the last ones last, so they are still cached
    const unsigned number = unsigned(a.first) + blockNumber();
    const int b0 = a.blocks - 1 - int(number), b = int(a.byTiles(unsigned(b0))), tile = b0 - b * a.tiles;
    const int n = int(a.byChunks(unsigned(b))), chunk = b - n * a.applyChunks;
    const int c0 = tile * kTileC, tileC = min(kTileC, a.C - c0);
    const int g0 = int(a.byGroupC(unsigned(c0))), groups = int(a.byGroupC(unsigned(c0 + tileC - 1))) + 1 - g0;
    const int64_t p0 = int64_t(chunk) * a.applyPixels;
    const int count = int(min(int64_t(a.applyPixels), a.pixels - p0));
    const int tid = threadIdx.x;

    const int vecs = vecsFor<MX4>(tileC), rows = kThreads / vecs, row = tid / vecs, col = tid - row * vecs;
    const int m = row < rows ? max(0, min(kVec, tileC - col * kVec)) : 0, c = c0 + col * kVec;
    const T* in = static_cast<const T*>(a.in) + (n * a.pixels + p0) * a.C + c;
    const T* end = static_cast<const T*>(a.in) + a.values;
    constexpr int kFlight = 2;
    Held<T> x[kFlight];
    const auto load = [&](Held<T>& to, const T* from) {
        if (WHOLE) to.load(from);
        else loadHeld(from, m, end, to);
    };
    const int64_t step = int64_t(rows) * a.C;
    const T* at = in + int64_t(row) * a.C;
    // neither the first loads nor those of the parameters wait for the statistics
    if (m > 0)
    {
#pragma unroll
        for (int u = 0; u < kFlight; ++u)
            if (row + u * rows < count) load(x[u], at + u * step);
    }
    Finish<T> f;
    f.load(a, m, c);

    if (a.chunks > kJoin)
    {
        for (int g = tid; g < groups; g += kThreads) sStat[g] = a.joined[int64_t(n) * a.G + g0 + g];
    }
    else
    {
        const int lanes = lanesPerGroup(groups, kThreads), lane = tid & (lanes - 1);
        for (int g = tid / lanes; g < groups; g += kThreads / lanes)
        {
            const float2 v = joinParts<8>(a, a.partial + (int64_t(n) * a.G + g0 + g) * a.chunks, lane, lanes);
            if (lane == 0) sStat[g] = v;
        }
    }
    __syncthreads();
    if (row >= rows) return;
    f.prepare(a, sStat, g0, m, c);
    Target<T> to(a, n * a.pixels + p0 + row, c, rows);
    forActivation(a.activation, [&](auto act) {
        int p = row;
        for (; p + (2 * kFlight - 1) * rows < count; p += kFlight * rows)
        {
            Held<T> next[kFlight];
            at += kFlight * step;
            if (m > 0)
            {
#pragma unroll
                for (int u = 0; u < kFlight; ++u) load(next[u], at + u * step);
            }
#pragma unroll
            for (int u = 0; u < kFlight; ++u) to.template store<MX4, act.value>(a, f, x[u], m, u);
            to.advance(kFlight);
#pragma unroll
            for (int u = 0; u < kFlight; ++u) x[u] = next[u];
        }
        for (; p < count; p += kFlight * rows)
        {
            Held<T> next[kFlight];
            at += kFlight * step;
#pragma unroll
            for (int u = 0; u < kFlight; ++u)
                if (m > 0 && p + (kFlight + u) * rows < count) load(next[u], at + u * step);
#pragma unroll
            for (int u = 0; u < kFlight; ++u)
                if (p + u * rows < count) to.template store<MX4, act.value>(a, f, x[u], m, u);
            to.advance(kFlight);
#pragma unroll
            for (int u = 0; u < kFlight; ++u) x[u] = next[u];
        }
    });
}

struct MxArgs
{
    const void* in;
    void* out;
    const uint8_t *codesIn, *scalesIn;
    uint8_t *codes, *scales;
    int64_t units;                    // rows x eighths of a row's blocks
    int64_t columns, values;          // values: rows * columns
    unsigned rowUnits;                // 4 * blocks of a row
    Divider byRow;
    int stream;                       // the unquantised side passes by the caches
};

constexpr int kUnits = 4;             // units per thread

// A thread makes the codes of eight values; four neighbours share a block.
// `row` and place of unit number `base + local` among the rows' units; local < 2^31, rem = base's place in its row.
struct Unit
{
    int64_t row;
    unsigned col;
    __device__ __forceinline__ Unit(const MxArgs& a, int64_t row0, unsigned rem, unsigned local)
    {
        const unsigned at = rem + local, r = a.byRow(at);
        row = row0 + r;
        col = at - r * a.rowUnits;
    }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void QuantizeKernel(const MxArgs a)
{
    const int64_t base = int64_t(blockNumber()) * (kThreads * kUnits);
    const int64_t row0 = base / a.rowUnits;
    const unsigned rem = unsigned(base - row0 * a.rowUnits);
    const T* in = static_cast<const T*>(a.in);
    float v[kUnits][kVec];
    // all loads first; units come in fours: a block's threads are there or not together
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
    {
        const unsigned local = u * kThreads + threadIdx.x;
        if (base + local >= a.units) break;
        const Unit unit(a, row0, rem, local);
        const int64_t c = int64_t(unit.col) * kVec;
        const int m = int(max(int64_t(0), min(int64_t(kVec), a.columns - c)));
        const T* p = in + unit.row * a.columns + c;
        if (m == kVec && a.stream) streamIn8(p, v[u]);
        else loadUpTo8(p, m, in + a.values, v[u]);
        if (m < kVec)
        {
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[u][i] = i < m ? v[u][i] : 0.0f;
        }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
    {
        const int64_t unit = base + u * kThreads + threadIdx.x;
        if (unit >= a.units) break;
        unsigned scale;
        const unsigned codes = mxQuantise(v[u], scale);
        *reinterpret_cast<unsigned*>(a.codes + unit * 4) = codes;
        if ((threadIdx.x & 3) == 0) a.scales[unit >> 2] = uint8_t(scale);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void DequantizeKernel(const MxArgs a)
{
    const int64_t base = int64_t(blockNumber()) * (kThreads * kUnits);
    const int64_t row0 = base / a.rowUnits;
    const unsigned rem = unsigned(base - row0 * a.rowUnits);
    unsigned codes[kUnits], scale[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
    {
        const int64_t unit = base + u * kThreads + threadIdx.x;
        if (unit >= a.units) break;
        codes[u] = *reinterpret_cast<const unsigned*>(a.codesIn + unit * 4);
        scale[u] = a.scalesIn[unit >> 2];
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
    {
        const unsigned local = u * kThreads + threadIdx.x;
        if (base + local >= a.units) break;
        const Unit unit(a, row0, rem, local);
        const int64_t c = int64_t(unit.col) * kVec;
        const int m = int(max(int64_t(0), min(int64_t(kVec), a.columns - c)));
        float v[kVec];
        mxValues8(codes[u], v);
        const float f = mxFactor(scale[u]);
#pragma unroll
        for (int i = 0; i < kVec; ++i)
        {
            v[i] *= f;
            asm("" : "+v"(v[i]));                       // else the rounding to fp16 becomes part of a fused product + 0: -0 would lose its sign
        }
        T* p = static_cast<T*>(a.out) + unit.row * a.columns + c;
        if (m == kVec && a.stream) streamOut8(p, v);
        else storeUpTo8(p, m, v);
    }
}

// How a normalisation is cut into workgroups.  Slabs (NormSlabKernel) where all pixels of the fewest whole groups fit
// one workgroup's registers; otherwise parts of images.
struct NormPlan
{
    NormArgs a{};
    int slabThreads = 0, slabHeld = 0;     // 0: no slabs
    int64_t images = 0;
};

NormPlan planNorm(const ML::Operator& op, bool mx4)
{
    NormPlan p;
    NormArgs& a = p.a;
    a.C = int(op.inputSizes[1]);
    a.G = int(op.groups);
    a.groupC = a.C / a.G;
    a.pixels = int64_t(op.inputSizes[2]) * op.inputSizes[3];
    a.values = a.pixels * a.C * op.inputSizes[0];
    a.epsilon = op.epsilon;
    a.activation = int(op.activation);
    p.images = op.inputSizes[0];
    const int64_t n = p.images;
    a.byGroupC = Divider(unsigned(a.groupC));
    a.groupsInAll = int(n * a.G);          // (the factory refuses more than 2^31 - 1)

    // Slabs of the fewest groups that are a whole number of 64-byte lines (of blocks of 32 channels), or of single groups.  A
    // slab has one CU's arithmetic: with SiLU 8192 values take 4.2 us, 32768 take 8.5, 131072 take 25, against 10 us for
    // the two kernels below on images up to 1 MB.  Single groups, whose pixels are pieces of lines: 32768 values take 15.6 us.
    const bool half = op.dataType == ML::TensorDataType::FLOAT16;
    const int64_t imageBytes = a.pixels * a.C * (half ? 2 : 4);
    const auto slab = [&](int groups, int most) {
        const int64_t vecs = mx4 ? vecsFor<true>(groups * a.groupC) : vecsFor<false>(groups * a.groupC);
        for (const int threads : {256, 1024})
        {
            if (vecs > threads || a.pixels > 1 << 20) continue;
            const int64_t rows = threads / vecs, held = (a.pixels + rows - 1) / rows;
            if (held > (threads == 256 ? 4 : most)) continue;
            p.slabThreads = threads;
            p.slabHeld = int(held);
            a.tileGroups = groups;
            a.tiles = (a.G + groups - 1) / groups;
            a.slabRows = int(rows);
            a.byTiles = Divider(unsigned(a.tiles));
            a.byVecs = Divider(unsigned(vecs));
            return n * a.tiles <= INT32_MAX;
        }
        return false;
    };
    const int unit = mx4 || half ? 32 : 16;
    int lines = 1;
    while (lines < a.G && (lines * a.groupC) % unit != 0) ++lines;
    // few slabs of whole lines: single groups make more of them (4 x 32x32 pixels of 128 channels: 7.8 instead of 10.9 us)
    if (!mx4 && n * ((a.G + lines - 1) / lines) < 32 && slab(1, 2)) return p;
    if (slab(lines, 4)) return p;
    p.slabThreads = 0;

    a.tileGroups = a.groupC >= kTileC ? 1 : (kTileC / a.groupC < a.G ? kTileC / a.groupC : a.G);
    a.tiles = (a.G + a.tileGroups - 1) / a.tileGroups;
    // Statistics: parts of 32 KB for small images, of 64 KB for others, about 1024 workgroups at most.  Up to kJoin parts of
    // an image spare the kernel that joins them (4.6 us), which pays while they stay below 192 KB.
    int64_t chunks = (imageBytes + (32 << 10) - 1) / (32 << 10);
    if (chunks > kJoin) chunks = imageBytes <= int64_t(kJoin) * (192 << 10) ? kJoin : (imageBytes + (64 << 10) - 1) / (64 << 10);
    const int64_t most = (1024 + n * a.tiles - 1) / (n * a.tiles);
    if (chunks > most) chunks = most;
    // No thread adds up more than 256 values of a channel (parts of 1 MB in fp16, if its rows fill the workgroup): the rounding of
    // its sums, about a first value that may be far from the others, grows with their number.  Threads of a group wider than the
    // workgroup add up all its channels, in 64 bits; their parts are cut to about the same size.
    const int64_t vecs = vecsFor<false>(a.tileGroups * a.groupC);
    const int64_t longest = vecs <= kThreads ? 256 * (kThreads / vecs) : 256 * kThreads / vecs;
    const int64_t least = longest > 1 ? (a.pixels + longest - 1) / longest : a.pixels;
    if (chunks < least) chunks = least;
    a.chunkPixels = int((a.pixels + chunks - 1) / chunks);
    a.chunks = int((a.pixels + a.chunkPixels - 1) / a.chunkPixels);
    // Output: about 1024 workgroups (256x256 pixels of 256 channels in 4 bits: 13.0 us; 2048: 14.6), four batches of pixels
    // for each thread at least.
    a.applyTiles = (a.C + kTileC - 1) / kTileC;
    const int rows = kTileC / (a.C < kTileC ? (a.C + 31) / 32 * 32 : kTileC);
    int64_t parts = (1024 + n * a.applyTiles - 1) / (n * a.applyTiles);
    const int64_t mostParts = (a.pixels + 4 * rows - 1) / (4 * rows);
    if (parts > mostParts) parts = mostParts;
    if (parts < (a.pixels + (1 << 22) - 1) >> 22) parts = (a.pixels + (1 << 22) - 1) >> 22;
    a.applyPixels = int((a.pixels + parts - 1) / parts);
    a.applyChunks = int((a.pixels + a.applyPixels - 1) / a.applyPixels);
    a.stream = n * imageBytes > kStreamBytes;
    return p;
}

size_t normWorkspace(const NormPlan& p)
{
    if (p.slabThreads) return 0;
    return size_t(p.images) * p.a.G * (p.a.chunks + (p.a.chunks > kJoin ? 1 : 0)) * sizeof(float2);
}

// f(grid, arguments) for all workgroups: whole rows of them (gridOf), and the rest in a launch of its own.  (One launch whose last
// workgroups leave at once would have every one of them wait for their number: 0.4 us of kernels of 6.)
template <typename F>
hipError_t inGrids(NormArgs a, int64_t blocks, F&& f)
{
    const int64_t rows = blocks / kGridRow, rest = blocks % kGridRow;
    a.blocks = int(blocks);
    a.first = 0;
    if (rows > 0) f(dim3(kGridRow, unsigned(rows)), a);
    a.first = int(rows * kGridRow);
    if (rest > 0) f(dim3(unsigned(rest)), a);
    return hipGetLastError();
}

template <typename T, bool MX4>
hipError_t launchNorm(const NormPlan& p, hipStream_t s)
{
    const NormArgs& a = p.a;
    if (p.slabThreads)
        return inGrids(a, p.images * a.tiles, [&](dim3 grid, const NormArgs& g) {
            if (p.slabThreads == 256 && p.slabHeld == 1) hipLaunchKernelGGL((NormSlabKernel<T, MX4, 256, 1>), grid, dim3(256), 0, s, g);
            else if (p.slabThreads == 256) hipLaunchKernelGGL((NormSlabKernel<T, MX4, 256, 4>), grid, dim3(256), 0, s, g);
            else if (p.slabHeld <= 2) hipLaunchKernelGGL((NormSlabKernel<T, MX4, 1024, 2>), grid, dim3(1024), 0, s, g);
            else hipLaunchKernelGGL((NormSlabKernel<T, MX4, 1024, 4>), grid, dim3(1024), 0, s, g);
        });
    const int64_t statsGrid = p.images * a.chunks * a.tiles, applyGrid = p.images * a.applyChunks * a.applyTiles;
    if (statsGrid > INT32_MAX || applyGrid > INT32_MAX || p.images * a.G > INT32_MAX) return hipErrorInvalidValue;
    const dim3 block(kThreads);
    NormArgs st = a, ap = a;
    st.byTiles = Divider(unsigned(a.tiles));
    st.byChunks = Divider(unsigned(a.chunks));
    ap.tiles = a.applyTiles;
    ap.byTiles = Divider(unsigned(a.applyTiles));
    ap.byChunks = Divider(unsigned(a.applyChunks));
    const bool whole = a.C % kVec == 0 && (a.tileGroups == a.G || (a.tileGroups * a.groupC) % kVec == 0);
    hipError_t e = inGrids(st, statsGrid, [&](dim3 grid, const NormArgs& g) {
        if (whole) hipLaunchKernelGGL((NormStatsKernel<T, true>), grid, block, 0, s, g);
        else hipLaunchKernelGGL((NormStatsKernel<T, false>), grid, block, 0, s, g);
    });
    if (e != hipSuccess) return e;
    if (a.chunks > kJoin)
    {
        hipLaunchKernelGGL(NormJoinKernel, dim3(unsigned(a.groupsInAll)), dim3(64), 0, s, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    return inGrids(ap, applyGrid, [&](dim3 grid, const NormArgs& g) {
        if (a.C % kVec == 0) hipLaunchKernelGGL((NormApplyKernel<T, MX4, true>), grid, block, 0, s, g);
        else hipLaunchKernelGGL((NormApplyKernel<T, MX4, false>), grid, block, 0, s, g);
    });
}

}  // namespace

size_t GroupNormWorkspace(const ML::Operator& op)
{
    if (op.kind != ML::Operator::Kind::GROUP_NORM) return 0;
    const size_t plain = normWorkspace(planNorm(op, false)), mx4 = normWorkspace(planNorm(op, true));
    return plain > mx4 ? plain : mx4;
}

hipError_t LaunchGroupNorm(const ML::Operator& op, const void* in, const void* scale, const void* bias, void* out,
                           uint8_t* codes, uint8_t* scales, void* workspace, size_t workspaceBytes, hipStream_t s)
{
    if (op.kind != ML::Operator::Kind::GROUP_NORM || !in || !codes != !scales || !out == !codes || (reinterpret_cast<uintptr_t>(codes) & 15))
        return hipErrorInvalidValue;
    NormPlan p = planNorm(op, codes != nullptr);
    const size_t need = normWorkspace(p);
    if (need && (!workspace || workspaceBytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7))) return hipErrorInvalidValue;
    NormArgs& a = p.a;
    a.in = in;
    a.scale = scale;
    a.bias = bias;
    a.out = out;
    a.codes = codes;
    a.scales = scales;
    a.partial = static_cast<float2*>(workspace);
    a.joined = a.partial + size_t(p.images) * a.G * a.chunks;
    const bool half = op.dataType == ML::TensorDataType::FLOAT16;
    if (half) return codes ? launchNorm<f16, true>(p, s) : launchNorm<f16, false>(p, s);
    return codes ? launchNorm<float, true>(p, s) : launchNorm<float, false>(p, s);
}

namespace {
bool planMx(int64_t rows, int64_t columns, int bytes, MxArgs& a, dim3& grid)
{
    if (rows < 1 || columns < 1 || columns > 1 << 20 || rows >= int64_t(1) << 40) return false;
    a.columns = columns;
    a.values = rows * columns;
    a.rowUnits = unsigned(4 * mxBlocks(columns));
    a.units = rows * a.rowUnits;
    a.byRow = Divider(a.rowUnits);
    a.stream = a.values * bytes > kStreamBytes;
    const int64_t blocks = (a.units + kThreads * kUnits - 1) / (kThreads * kUnits);
    grid = gridOf(blocks);
    return blocks <= INT32_MAX;
}
}  // namespace

hipError_t LaunchQuantizeMx4(ML::TensorDataType t, const void* in, int64_t rows, int64_t columns, uint8_t* codes,
                             uint8_t* scales, hipStream_t s)
{
    MxArgs a{};
    dim3 grid;
    if (!in || !codes || !scales || (reinterpret_cast<uintptr_t>(codes) & 15)) return hipErrorInvalidValue;
    if (!planMx(rows, columns, t == ML::TensorDataType::FLOAT16 ? 2 : 4, a, grid)) return hipErrorInvalidValue;
    a.in = in;
    a.codes = codes;
    a.scales = scales;
    if (t == ML::TensorDataType::FLOAT16) hipLaunchKernelGGL(QuantizeKernel<f16>, grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL(QuantizeKernel<float>, grid, dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

hipError_t LaunchDequantizeMx4(ML::TensorDataType t, const uint8_t* codes, const uint8_t* scales, int64_t rows,
                               int64_t columns, void* out, hipStream_t s)
{
    MxArgs a{};
    dim3 grid;
    if (!codes || !scales || !out || (reinterpret_cast<uintptr_t>(codes) & 15)) return hipErrorInvalidValue;
    if (!planMx(rows, columns, t == ML::TensorDataType::FLOAT16 ? 2 : 4, a, grid)) return hipErrorInvalidValue;
    a.codesIn = codes;
    a.scalesIn = scales;
    a.out = out;
    if (t == ML::TensorDataType::FLOAT16) hipLaunchKernelGGL(DequantizeKernel<f16>, grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL(DequantizeKernel<float>, grid, dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace srx
