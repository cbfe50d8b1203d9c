// The library's host side without a GPU: its kernel launches are recorded -- the kernel's name, the grid, the block and the first
// argument's bytes -- and do nothing.  For programs linked with -rdynamic, whose symbols stand in for the HIP runtime's.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstring>
#include <map>
#include <string>
#include <vector>

#include "ascq.h"
#include "launch.h"

struct Launch {
    std::string kernel;  // mangled
    dim3 grid, block;
    uint8_t bytes[256];
    int64_t second;  // the second argument's first bytes, when there is one
    template <class T>
    T args() const
    {
        static_assert(sizeof(T) <= sizeof(bytes), "argument");
        T a;
        std::memcpy((void*)&a, bytes, sizeof(T));
        return a;
    }
    bool is(const char* name) const { return kernel.find(name) != std::string::npos; }
    uint64_t threads() const
    {
        return (uint64_t)grid.x * grid.y * grid.z * ((uint64_t)block.x * block.y * block.z);
    }
};
inline std::vector<Launch>& launches()
{
    static std::vector<Launch> v;
    return v;
}
inline std::map<const void*, std::string>& kernels()
{
    static std::map<const void*, std::string> m;
    return m;
}
// bytes that are kept of a kernel's first argument
inline size_t& first_argument()
{
    static size_t n = 0;
    return n;
}

inline size_t& second_argument()
{
    static size_t n = 0;
    return n;
}
inline Launch& configured()
{
    static Launch l{};
    return l;
}

extern "C" {
hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t, hipStream_t)
{
    configured().grid = grid;
    configured().block = block;
    return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* stream)
{
    *grid = configured().grid;
    *block = configured().block;
    *shared = 0;
    *stream = nullptr;
    return hipSuccess;
}
void __hipRegisterFunction(void**, const void* host, char*, const char* name, unsigned, void*, void*, void*, void*, int*)
{
    kernels()[host] = name;
}
hipError_t hipLaunchKernel(const void* host, dim3 grid, dim3 block, void** args, size_t, hipStream_t)
{
    Launch l{};
    l.kernel = kernels()[host];
    l.grid = grid;
    l.block = block;
    std::memcpy(l.bytes, args[0], first_argument() < sizeof(l.bytes) ? first_argument() : sizeof(l.bytes));
    if (second_argument()) std::memcpy(&l.second, args[1], second_argument());
    launches().push_back(l);
    return hipSuccess;
}
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipFuncSetAttribute(const void*, hipFuncAttribute, int) { return hipSuccess; }
hipError_t hipGetDevice(int* d)
{
    *d = 0;
    return hipSuccess;
}
}
