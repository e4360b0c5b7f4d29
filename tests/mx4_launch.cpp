// The host side of the normalisation and 4-bit layers, linked with a HIP runtime that launches nothing: it notes the kernels
// that are asked for, and the first launch leaves the error it is told to.
//
//   mx4_launch conv  dtype n c h w o kh kw error     LaunchConvMx4 on an operator of these sizes
//   mx4_launch norm  dtype n c h w groups mx4 error  LaunchGroupNorm
//   mx4_launch refusals                              calls that have to be refused: a line for each that was not
// Prints the status and then the launched kernels, one a line.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <cxxabi.h>
#include <map>
#include <string>

#include "srx_kernels.h"

namespace {
std::map<const void*, std::string>& names()
{
    static std::map<const void*, std::string> all;
    return all;
}
int g_launches = 0, g_error = 0;
hipError_t g_left = hipSuccess;
dim3 g_grid, g_block;
size_t g_lds = 0;
hipStream_t g_stream = nullptr;
}  // namespace

extern "C" {
void** __hipRegisterFatBinary(const void*)
{
    static void* module = nullptr;
    return &module;
}
void __hipUnregisterFatBinary(void**) {}
void __hipRegisterFunction(void**, const void* function, char*, const char* name, unsigned, void*, void*, void*, void*, int*)
{
    int status = 0;
    char* plain = abi::__cxa_demangle(name, nullptr, nullptr, &status);
    names()[function] = status == 0 ? plain : name;
    std::free(plain);
}
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t lds, hipStream_t stream)
{
    g_grid = grid, g_block = block, g_lds = lds, g_stream = stream;
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* lds, hipStream_t* stream)
{
    *grid = g_grid, *block = g_block, *lds = g_lds, *stream = g_stream;
    return hipSuccess;
}
hipError_t hipLaunchKernel(const void* function, dim3, dim3, void**, size_t, hipStream_t)
{
    std::printf("%s\n", names()[function].c_str());
    g_left = ++g_launches == 1 ? hipError_t(g_error) : hipSuccess;
    return g_left;
}
hipError_t hipGetLastError()
{
    const hipError_t e = g_left;
    g_left = hipSuccess;
    return e;
}
}

namespace srx {
namespace dev {
hipError_t ensureDynamicLds(const void*, int) { return hipSuccess; }
}  // namespace dev
}  // namespace srx

namespace {
using namespace srx;
using namespace srx::ML;

template <typename T> T* at(uintptr_t address) { return reinterpret_cast<T*>(address); }   // nothing looks there

int refusals()
{
    int taken = 0;
    const auto refuse = [&](const char* what, hipError_t e) {
        if (e == hipErrorInvalidValue && g_launches == 0) return;
        std::printf("taken: %s\n", what);
        ++taken;
        g_launches = 0;
    };
    const Util util(TensorDataType::FLOAT16, TensorLayout::NHWC), planar(TensorDataType::FLOAT16, TensorLayout::DEFAULT);
    const uint32_t sizes[4] = {1, 64, 300, 200}, filter[4] = {32, 64, 3, 3};
    uint32_t os[4];
    uint64_t ib = 0, ob = 0;
    Operator norm, conv, dense, none;
    if (!util.CreateGroupNormLayer(sizes, 8, 1e-5f, 0, norm) || !util.CreateConvolutionMx4Layer(sizes, filter, 0, conv) ||
        !util.CreateConvolutionLayer(sizes, filter, false, ib, ob, os, dense)) return 2;

    // what a factory refuses, it leaves alone
    const uint32_t wide[4] = {1, 64, 300, 200}, far[4] = {32, 64, 8, 3}, big[4] = {2, 64, 1u << 15, 1u << 15}, many[4] = {(1u << 20) + 1, 64, 1, 1};
    const auto untouched = [&](const char* what, bool made, const Operator& op) {
        if (made || op.kind != Operator::Kind::NONE) std::printf("taken: %s\n", what), ++taken;
    };
    Operator op;
    untouched("a filter of eight rows", util.CreateConvolutionMx4Layer(wide, far, 0, op), op);
    untouched("2^31 pixels", util.CreateConvolutionMx4Layer(big, filter, 0, op), op);
    untouched("2^20 + 1 filters", util.CreateConvolutionMx4Layer(wide, many, 0, op), op);
    untouched("planar tensors", planar.CreateConvolutionMx4Layer(wide, filter, 0, op), op);
    untouched("activation 3", util.CreateConvolutionMx4Layer(wide, filter, 3, op), op);
    untouched("groups of planar tensors", planar.CreateGroupNormLayer(wide, 8, 1e-5f, 0, op), op);
    untouched("seven groups of 64", util.CreateGroupNormLayer(wide, 7, 1e-5f, 0, op), op);

    void* const p = at<void>(1 << 20);
    uint8_t *const c = at<uint8_t>(2 << 20), *const odd = c + 8;
    const size_t need = GroupNormWorkspace(norm);
    if (need == 0 || GroupNormWorkspace(conv) || GroupNormWorkspace(none)) std::printf("taken: workspaces\n"), ++taken;
    for (const Operator* other : {&conv, &dense, &none})
        refuse("another operator's normalisation", LaunchGroupNorm(*other, p, nullptr, nullptr, p, nullptr, nullptr, p, need, nullptr));
    refuse("no input", LaunchGroupNorm(norm, nullptr, nullptr, nullptr, p, nullptr, nullptr, p, need, nullptr));
    refuse("no output", LaunchGroupNorm(norm, p, nullptr, nullptr, nullptr, nullptr, nullptr, p, need, nullptr));
    refuse("two outputs", LaunchGroupNorm(norm, p, nullptr, nullptr, p, c, c, p, need, nullptr));
    refuse("no scales", LaunchGroupNorm(norm, p, nullptr, nullptr, nullptr, c, nullptr, p, need, nullptr));
    refuse("no codes", LaunchGroupNorm(norm, p, nullptr, nullptr, nullptr, nullptr, c, p, need, nullptr));
    refuse("codes between blocks", LaunchGroupNorm(norm, p, nullptr, nullptr, nullptr, odd, c, p, need, nullptr));
    refuse("no workspace", LaunchGroupNorm(norm, p, nullptr, nullptr, p, nullptr, nullptr, nullptr, need, nullptr));
    refuse("a small workspace", LaunchGroupNorm(norm, p, nullptr, nullptr, p, nullptr, nullptr, p, 8, nullptr));
    refuse("a workspace between words", LaunchGroupNorm(norm, p, nullptr, nullptr, p, nullptr, nullptr, at<void>(4), need, nullptr));
    for (const Operator* other : {&norm, &dense, &none})
        refuse("another operator's convolution", LaunchConvMx4(*other, c, c, c, c, nullptr, p, nullptr));
    refuse("no input codes", LaunchConvMx4(conv, nullptr, c, c, c, nullptr, p, nullptr));
    refuse("no input scales", LaunchConvMx4(conv, c, nullptr, c, c, nullptr, p, nullptr));
    refuse("no filter codes", LaunchConvMx4(conv, c, c, nullptr, c, nullptr, p, nullptr));
    refuse("no filter scales", LaunchConvMx4(conv, c, c, c, nullptr, nullptr, p, nullptr));
    refuse("no result", LaunchConvMx4(conv, c, c, c, c, nullptr, nullptr, nullptr));
    refuse("input codes between blocks", LaunchConvMx4(conv, odd, c, c, c, nullptr, p, nullptr));
    refuse("filter codes between blocks", LaunchConvMx4(conv, c, c, odd, c, nullptr, p, nullptr));
    for (const Operator* other : {&norm, &conv, &none})
        refuse("an operator of other operands", DispatchOperator(*other, p, p, p, p, nullptr));
    const auto t = TensorDataType::FLOAT32;
    refuse("nothing to quantise", LaunchQuantizeMx4(t, nullptr, 1, 1, c, c, nullptr));
    refuse("quantised without codes", LaunchQuantizeMx4(t, p, 1, 1, nullptr, c, nullptr));
    refuse("quantised without scales", LaunchQuantizeMx4(t, p, 1, 1, c, nullptr, nullptr));
    refuse("quantised between blocks", LaunchQuantizeMx4(t, p, 1, 1, odd, c, nullptr));
    refuse("no rows", LaunchQuantizeMx4(t, p, 0, 1, c, c, nullptr));
    refuse("less than no columns", LaunchQuantizeMx4(t, p, 1, -1, c, c, nullptr));
    refuse("2^20 + 1 columns", LaunchQuantizeMx4(t, p, 1, (1 << 20) + 1, c, c, nullptr));
    refuse("values of no codes", LaunchDequantizeMx4(t, nullptr, c, 1, 1, p, nullptr));
    refuse("values of no scales", LaunchDequantizeMx4(t, c, nullptr, 1, 1, p, nullptr));
    refuse("values for nobody", LaunchDequantizeMx4(t, c, c, 1, 1, nullptr, nullptr));
    refuse("values between blocks", LaunchDequantizeMx4(t, odd, c, 1, 1, p, nullptr));
    std::printf("status %d\n", taken);
    return 0;
}
}  // namespace

int main(int argc, char** argv)
{
    if (argc == 2 && !std::strcmp(argv[1], "refusals")) return refusals();
    if (argc < 11 && !(argc == 10 && !std::strcmp(argv[1], "norm"))) return 2;
    uint32_t v[9] = {};
    for (int i = 2; i < argc; ++i) v[i - 2] = uint32_t(std::strtoul(argv[i], nullptr, 10));
    g_error = int(v[argc - 3]);
    const srx::ML::Util util(v[0] == 0 ? srx::ML::TensorDataType::FLOAT16 : srx::ML::TensorDataType::FLOAT32, srx::ML::TensorLayout::NHWC);
    const uint32_t sizes[4] = {v[1], v[2], v[3], v[4]};
    srx::ML::Operator op;
    uint8_t* const p = at<uint8_t>(1 << 20);
    hipError_t e = hipErrorInvalidValue;
    if (!std::strcmp(argv[1], "conv"))
    {
        const uint32_t filter[4] = {v[5], v[2], v[6], v[7]};
        if (util.CreateConvolutionMx4Layer(sizes, filter, 0, op)) e = srx::LaunchConvMx4(op, p, p, p, p, nullptr, p, nullptr);
    }
    else if (util.CreateGroupNormLayer(sizes, v[5], 1e-5f, 0, op))
        e = srx::LaunchGroupNorm(op, p, nullptr, nullptr, v[6] ? nullptr : p, v[6] ? p : nullptr, v[6] ? p : nullptr, p, size_t(1) << 30, nullptr);
    std::printf("status %d\n", int(e));
    return 0;
}
