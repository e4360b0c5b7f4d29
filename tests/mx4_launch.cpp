// The host side of the normalisation and 4-bit layers, linked with a HIP runtime that launches nothing: it notes the kernels
// that are asked for, and the first launch leaves the error it is told to.
//
//   mx4_launch conv  dtype n c h w o kh kw error     LaunchConvMx4 on an operator of these sizes
//   mx4_launch norm  dtype n c h w groups mx4 error  LaunchGroupNorm
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

int main(int argc, char** argv)
{
    if (argc < 11 && !(argc == 10 && !std::strcmp(argv[1], "norm"))) return 2;
    uint32_t v[9] = {};
    for (int i = 2; i < argc; ++i) v[i - 2] = uint32_t(std::strtoul(argv[i], nullptr, 10));
    g_error = int(v[argc - 3]);
    const srx::ML::Util util(v[0] == 0 ? srx::ML::TensorDataType::FLOAT16 : srx::ML::TensorDataType::FLOAT32, srx::ML::TensorLayout::NHWC);
    const uint32_t sizes[4] = {v[1], v[2], v[3], v[4]};
    srx::ML::Operator op;
    uint8_t* const at = reinterpret_cast<uint8_t*>(1 << 20);        // nothing looks there
    hipError_t e = hipErrorInvalidValue;
    if (!std::strcmp(argv[1], "conv"))
    {
        const uint32_t filter[4] = {v[5], v[2], v[6], v[7]};
        if (util.CreateConvolutionMx4Layer(sizes, filter, 0, op)) e = srx::LaunchConvMx4(op, at, at, at, at, nullptr, at, nullptr);
    }
    else if (util.CreateGroupNormLayer(sizes, v[5], 1e-5f, 0, op))
        e = srx::LaunchGroupNorm(op, at, nullptr, nullptr, v[6] ? nullptr : at, v[6] ? at : nullptr, v[6] ? at : nullptr, at, nullptr);
    std::printf("status %d\n", int(e));
    return 0;
}
