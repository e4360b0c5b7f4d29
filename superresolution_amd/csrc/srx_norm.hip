// gfx950 kernels of the group normalisation layer and of the conversions to and from the 4-bit block form
// (srx_mx4.h).  Tensors are dense and channels last: {N, C, H, W} held as [N][H][W][C].
//
// Group normalisation of image n, group g (the C/G channels g*C/G ..):
//     mean = avg(x),  var = avg((x - mean)^2)  over the group's channels of every pixel
//     y = act((x - mean) / sqrt(var + epsilon) * scale[c] + bias[c])
// Statistics are kept as (mean, M2 = sum of squared deviations) of a part of the data and joined by
//     M2 = sum M2_i + sum n_i (mean_i - mean)^2,
// so nothing cancels when the mean is large against the deviation.  Everything is fp32, rounded once when stored.
#include "srx_mx4.h"

namespace srx {

using namespace dev;

namespace {

constexpr int kVec = 8;               // channels of one thread
constexpr int kTileC = kThreads * kVec;

struct NormArgs
{
    const void *in, *scale, *bias;
    void* out;
    uint8_t *codes, *scales;
    float2* partial;                  // [N][chunks][G] (mean, M2)
    int64_t pixels;                   // H * W
    int C, G, groupC;                 // channels, groups, channels of a group
    int chunks, chunkPixels;          // statistics: parts of an image
    int tileGroups, tiles;            // statistics: whole groups per workgroup
    int applyChunks, applyPixels, applyTiles;
    float epsilon;
    int activation;
};

// Sum over the `lanes` (a power of two up to 64) lanes of an aligned part of a wave.
__device__ __forceinline__ float sumLanes(float v, int lanes)
{
    for (int m = 1; m < lanes; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// Threads that share one group's reduction when a workgroup reduces `groups` of them.
__device__ __forceinline__ int lanesPerGroup(int groups)
{
    int lanes = 64;
    while (lanes > 1 && lanes * groups > kThreads) lanes >>= 1;
    return lanes;
}

// Statistics of one part of one image for a range of whole groups.  A thread keeps eight channels and walks the
// part's pixels; sums are of x - (its first value of the channel), whose magnitude the part's own spread bounds.
template <typename T>
__global__ __launch_bounds__(kThreads) void NormStatsKernel(const NormArgs a)
{
    __shared__ float sMean[kTileC], sM2[kTileC];
    int b = blockIdx.x;
    const int tile = b % a.tiles; b /= a.tiles;
    const int chunk = b % a.chunks, n = b / a.chunks;
    const int g0 = tile * a.tileGroups, groups = min(a.tileGroups, a.G - g0);
    const int c0 = g0 * a.groupC, tileC = groups * a.groupC;
    const int64_t p0 = int64_t(chunk) * a.chunkPixels;
    const int count = int(min(int64_t(a.chunkPixels), a.pixels - p0));
    const T* in = static_cast<const T*>(a.in) + (n * a.pixels + p0) * a.C + c0;
    float2* out = a.partial + (int64_t(n) * a.chunks + chunk) * a.G + g0;
    const int tid = threadIdx.x, vecs = (tileC + kVec - 1) / kVec;

    if (vecs > kThreads)
    {
        // one group wider than a workgroup: every value belongs to it
        float k = 0.0f, s = 0.0f, q = 0.0f;
        int have = 0;
        for (int p = 0; p < count; ++p)
            for (int col = tid; col < vecs; col += kThreads)
            {
                float v[kVec];
                const int m = min(kVec, tileC - col * kVec);
                loadUpTo8(in + int64_t(p) * a.C + col * kVec, m, v);
                if (have == 0) k = v[0];
                have += m;
#pragma unroll
                for (int i = 0; i < kVec; ++i)
                    if (i < m) { const float d = v[i] - k; s += d; q = fmaf(d, d, q); }
            }
        const float cnt = float(have), total = float(count) * float(tileC);
        const float mean = have ? k + s / cnt : 0.0f, m2 = have ? fmaxf(q - s * s / cnt, 0.0f) : 0.0f;
        sMean[tid] = cnt * mean;
        __syncthreads();
        float all = 0.0f;
        for (int i = 0; i < kThreads; ++i) all += sMean[i];
        all /= total;
        const float d = mean - all;
        sM2[tid] = m2 + cnt * d * d;
        __syncthreads();
        if (tid == 0)
        {
            float r = 0.0f;
            for (int i = 0; i < kThreads; ++i) r += sM2[i];
            out[0] = float2{all, r};
        }
        return;
    }

    const int rows = kThreads / vecs, row = tid / vecs, col = tid - row * vecs;
    if (row < rows)
    {
        const int m = min(kVec, tileC - col * kVec);
        const T* src = in + col * kVec;
        float k[kVec], s[kVec], q[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) k[i] = s[i] = q[i] = 0.0f;
        if (row < count) loadUpTo8(src + int64_t(row) * a.C, m, k);
#pragma unroll 4
        for (int p = row + rows; p < count; p += rows)
        {
            float v[kVec];
            loadUpTo8(src + int64_t(p) * a.C, m, v);
#pragma unroll
            for (int i = 0; i < kVec; ++i) { const float d = v[i] - k[i]; s[i] += d; q[i] = fmaf(d, d, q[i]); }
        }
        const float inv = 1.0f / float(max(1, (count - row + rows - 1) / rows));
#pragma unroll
        for (int i = 0; i < kVec; ++i)
        {
            sMean[(row * vecs + col) * kVec + i] = fmaf(s[i], inv, k[i]);
            sM2[(row * vecs + col) * kVec + i] = fmaxf(q[i] - s[i] * s[i] * inv, 0.0f);
        }
    }
    __syncthreads();
    // join the rows of each channel
    const int stride = vecs * kVec;
    for (int c = tid; c < tileC; c += kThreads)
    {
        float mean = 0.0f, m2 = 0.0f;
        for (int r = 0; r < rows && r < count; ++r) mean += float((count - r + rows - 1) / rows) * sMean[r * stride + c];
        mean /= float(count);
        for (int r = 0; r < rows && r < count; ++r)
        {
            const float d = sMean[r * stride + c] - mean;
            m2 += sM2[r * stride + c] + float((count - r + rows - 1) / rows) * d * d;
        }
        sMean[c] = mean;
        sM2[c] = m2;
    }
    __syncthreads();
    // join the channels of each group: equal counts
    const int lanes = lanesPerGroup(groups), lane = tid & (lanes - 1);
    for (int g = tid / lanes; g < groups; g += kThreads / lanes)
    {
        float mean = 0.0f, m2 = 0.0f;
        for (int c = lane; c < a.groupC; c += lanes) mean += sMean[g * a.groupC + c];
        mean = sumLanes(mean, lanes) / float(a.groupC);
        for (int c = lane; c < a.groupC; c += lanes)
        {
            const float d = sMean[g * a.groupC + c] - mean;
            m2 += sM2[g * a.groupC + c] + float(count) * d * d;
        }
        m2 = sumLanes(m2, lanes);
        if (lane == 0) out[g] = float2{mean, m2};
    }
}

// Normalises, scales, activates and stores (MX4: as 4-bit blocks) a part of an image; the parts' statistics are
// joined by every workgroup for the groups it needs.
template <typename T, bool MX4>
__global__ __launch_bounds__(kThreads) void NormApplyKernel(const NormArgs a)
{
    __shared__ float2 sStat[kTileC];
    int b = blockIdx.x;
    const int tile = b % a.applyTiles; b /= a.applyTiles;
    const int chunk = b % a.applyChunks, n = b / a.applyChunks;
    const int c0 = tile * kTileC, tileC = min(kTileC, a.C - c0);
    const int g0 = c0 / a.groupC, groups = (c0 + tileC - 1) / a.groupC + 1 - g0;
    const int64_t p0 = int64_t(chunk) * a.applyPixels;
    const int count = int(min(int64_t(a.applyPixels), a.pixels - p0));
    const int tid = threadIdx.x;

    {
        const int lanes = lanesPerGroup(groups), lane = tid & (lanes - 1);
        const float2* partial = a.partial + int64_t(n) * a.chunks * a.G + g0;
        const float lastPixels = float(a.pixels - int64_t(a.chunks - 1) * a.chunkPixels);
        for (int g = tid / lanes; g < groups; g += kThreads / lanes)
        {
            float mean = 0.0f, m2 = 0.0f;
            for (int k = lane; k < a.chunks; k += lanes)
                mean += (k == a.chunks - 1 ? lastPixels : float(a.chunkPixels)) * partial[int64_t(k) * a.G + g].x;
            mean = sumLanes(mean, lanes) / float(a.pixels);
            for (int k = lane; k < a.chunks; k += lanes)
            {
                const float2 v = partial[int64_t(k) * a.G + g];
                const float d = v.x - mean;
                m2 += v.y + (k == a.chunks - 1 ? lastPixels : float(a.chunkPixels)) * float(a.groupC) * d * d;
            }
            m2 = sumLanes(m2, lanes);
            if (lane == 0) sStat[g] = float2{mean, 1.0f / sqrtf(m2 / (float(a.pixels) * float(a.groupC)) + a.epsilon)};
        }
    }
    __syncthreads();

    int vecs = (tileC + kVec - 1) / kVec;
    if (MX4) vecs = (vecs + 3) & ~3;                    // whole blocks: four threads each
    const int rows = kThreads / vecs, row = tid / vecs, col = tid - row * vecs;
    if (row >= rows) return;
    const int m = max(0, min(kVec, tileC - col * kVec)), c = c0 + col * kVec;
    float mean[kVec], mul[kVec], add[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i)
    {
        const int ci = min(c + i, a.C - 1);
        const float2 st = sStat[ci / a.groupC - g0];
        mean[i] = st.x;
        mul[i] = st.y * (a.scale ? (float)static_cast<const T*>(a.scale)[ci] : 1.0f);
        add[i] = a.bias ? (float)static_cast<const T*>(a.bias)[ci] : 0.0f;
    }
    const T* in = static_cast<const T*>(a.in) + (n * a.pixels + p0) * a.C + c;
    const int64_t blocks = mxBlocks(a.C);
    for (int p = row; p < count; p += rows)
    {
        float v[kVec];
        loadUpTo8(in + int64_t(p) * a.C, m, v);
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] = activate(fmaf(v[i] - mean[i], mul[i], add[i]), a.activation);
        const int64_t pixel = n * a.pixels + p0 + p;
        if (MX4)
        {
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[i] = i < m ? v[i] : 0.0f;
            unsigned scale;
            const unsigned codes = mxQuantise(v, scale);
            const int64_t block = pixel * blocks + (c >> 5);
            *reinterpret_cast<unsigned*>(a.codes + block * kMxBytes + (col & 3) * 4) = codes;
            if ((col & 3) == 0) a.scales[block] = uint8_t(scale);
        }
        else storeUpTo8(static_cast<T*>(a.out) + pixel * a.C + c, m, v);
    }
}

struct MxArgs
{
    const void* in;
    void* out;
    const uint8_t *codesIn, *scalesIn;
    uint8_t *codes, *scales;
    int64_t units;                    // rows x eighths of a row's blocks
    int64_t columns;
    unsigned rowUnits;                // 4 * blocks of a row
};

constexpr int kUnits = 4;             // units per thread

// A thread makes the codes of eight values; four neighbours share a block.
template <typename T>
__global__ __launch_bounds__(kThreads) void QuantizeKernel(const MxArgs a)
{
    const int64_t base = int64_t(blockIdx.x) * (kThreads * kUnits);
    const int64_t row0 = base / a.rowUnits;
    const unsigned rem = unsigned(base - row0 * a.rowUnits);
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
    {
        const unsigned at = rem + u * kThreads + threadIdx.x;
        const int64_t unit = base + u * kThreads + threadIdx.x;
        if (unit >= a.units) break;                     // units come in fours: a block's threads leave together
        const unsigned r = at / a.rowUnits, col = at - r * a.rowUnits;
        const int64_t c = int64_t(col) * kVec;
        float v[kVec];
        loadUpTo8(static_cast<const T*>(a.in) + (row0 + r) * a.columns + c, int(max(int64_t(0), min(int64_t(kVec), a.columns - c))), v);
        unsigned scale;
        const unsigned codes = mxQuantise(v, scale);
        *reinterpret_cast<unsigned*>(a.codes + unit * 4) = codes;
        if ((threadIdx.x & 3) == 0) a.scales[unit >> 2] = uint8_t(scale);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void DequantizeKernel(const MxArgs a)
{
    const int64_t base = int64_t(blockIdx.x) * (kThreads * kUnits);
    const int64_t row0 = base / a.rowUnits;
    const unsigned rem = unsigned(base - row0 * a.rowUnits);
#pragma unroll
    for (int u = 0; u < kUnits; ++u)
    {
        const unsigned at = rem + u * kThreads + threadIdx.x;
        const int64_t unit = base + u * kThreads + threadIdx.x;
        if (unit >= a.units) break;
        const unsigned r = at / a.rowUnits, col = at - r * a.rowUnits;
        const int64_t c = int64_t(col) * kVec;
        float v[kVec];
        mxValues8(*reinterpret_cast<const unsigned*>(a.codesIn + unit * 4), v);
        const float f = mxFactor(a.scalesIn[unit >> 2]);
#pragma unroll
        for (int i = 0; i < kVec; ++i) v[i] *= f;
        storeUpTo8(static_cast<T*>(a.out) + (row0 + r) * a.columns + c, int(max(int64_t(0), min(int64_t(kVec), a.columns - c))), v);
    }
}

// How a normalisation is cut into workgroups.
void planNorm(const ML::Operator& op, NormArgs& a)
{
    a.C = int(op.inputSizes[1]);
    a.G = int(op.groups);
    a.groupC = a.C / a.G;
    a.pixels = int64_t(op.inputSizes[2]) * op.inputSizes[3];
    a.tileGroups = a.groupC >= kTileC ? 1 : (kTileC / a.groupC < a.G ? kTileC / a.groupC : a.G);
    a.tiles = (a.G + a.tileGroups - 1) / a.tileGroups;
    const int64_t n = op.inputSizes[0];
    // enough parts for the whole device, no part below 16 pixels
    int64_t chunks = (1024 + n * a.tiles - 1) / (n * a.tiles);
    const int64_t most = (a.pixels + 15) / 16;
    if (chunks > most) chunks = most;
    if (chunks < (a.pixels + (1 << 20) - 1) >> 20) chunks = (a.pixels + (1 << 20) - 1) >> 20;
    a.chunkPixels = int((a.pixels + chunks - 1) / chunks);
    a.chunks = int((a.pixels + a.chunkPixels - 1) / a.chunkPixels);
    a.applyTiles = (a.C + kTileC - 1) / kTileC;
    int64_t parts = (4096 + n * a.applyTiles - 1) / (n * a.applyTiles);
    if (parts > most) parts = most;
    if (parts < a.chunks) parts = a.chunks;
    a.applyPixels = int((a.pixels + parts - 1) / parts);
    a.applyChunks = int((a.pixels + a.applyPixels - 1) / a.applyPixels);
    a.epsilon = op.epsilon;
    a.activation = int(op.activation);
}

}  // namespace

size_t GroupNormWorkspace(const ML::Operator& op)
{
    NormArgs a{};
    planNorm(op, a);
    return size_t(op.inputSizes[0]) * a.chunks * a.G * sizeof(float2);
}

hipError_t LaunchGroupNorm(const ML::Operator& op, const void* in, const void* scale, const void* bias, void* out,
                           uint8_t* codes, uint8_t* scales, void* workspace, hipStream_t s)
{
    NormArgs a{};
    planNorm(op, a);
    a.in = in;
    a.scale = scale;
    a.bias = bias;
    a.out = out;
    a.codes = codes;
    a.scales = scales;
    a.partial = static_cast<float2*>(workspace);
    const int64_t n = op.inputSizes[0];
    const int64_t statsGrid = n * a.chunks * a.tiles, applyGrid = n * a.applyChunks * a.applyTiles;
    if (statsGrid > INT32_MAX || applyGrid > INT32_MAX) return hipErrorInvalidValue;
    const dim3 block(kThreads), g1(static_cast<unsigned>(statsGrid)), g2(static_cast<unsigned>(applyGrid));
    const bool half = op.dataType == ML::TensorDataType::FLOAT16;
    if (half) hipLaunchKernelGGL(NormStatsKernel<f16>, g1, block, 0, s, a);
    else hipLaunchKernelGGL(NormStatsKernel<float>, g1, block, 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (half && codes) hipLaunchKernelGGL((NormApplyKernel<f16, true>), g2, block, 0, s, a);
    else if (half) hipLaunchKernelGGL((NormApplyKernel<f16, false>), g2, block, 0, s, a);
    else if (codes) hipLaunchKernelGGL((NormApplyKernel<float, true>), g2, block, 0, s, a);
    else hipLaunchKernelGGL((NormApplyKernel<float, false>), g2, block, 0, s, a);
    return hipGetLastError();
}

namespace {
bool planMx(int64_t rows, int64_t columns, MxArgs& a, dim3& grid)
{
    a.columns = columns;
    a.rowUnits = unsigned(4 * mxBlocks(columns));
    a.units = rows * a.rowUnits;
    const int64_t blocks = (a.units + kThreads * kUnits - 1) / (kThreads * kUnits);
    grid = dim3(unsigned(blocks));
    return blocks <= INT32_MAX;
}
}  // namespace

hipError_t LaunchQuantizeMx4(ML::TensorDataType t, const void* in, int64_t rows, int64_t columns, uint8_t* codes,
                             uint8_t* scales, hipStream_t s)
{
    MxArgs a{};
    dim3 grid;
    if (!planMx(rows, columns, a, grid)) return hipErrorInvalidValue;
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
    if (!planMx(rows, columns, a, grid)) return hipErrorInvalidValue;
    a.codesIn = codes;
    a.scalesIn = scales;
    a.out = out;
    if (t == ML::TensorDataType::FLOAT16) hipLaunchKernelGGL(DequantizeKernel<f16>, grid, dim3(kThreads), 0, s, a);
    else hipLaunchKernelGGL(DequantizeKernel<float>, grid, dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace srx
