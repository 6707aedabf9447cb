// What the kernels over rows of 32- and 16-bit floats share: element types, and guards of the C entries.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "context.hpp"

namespace aeonb
{
    __device__ __forceinline__ float to_float(float v) { return v; }
    __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
    __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

    template <typename T>
    __device__ __forceinline__ T from_float(float v);
    template <>
    __device__ __forceinline__ float from_float<float>(float v)
    {
        return v;
    }
    template <>
    __device__ __forceinline__ __half from_float<__half>(float v)
    {
        return __float2half_rn(v);
    }
    template <>
    __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v)
    {
        return __float2bfloat16_rn(v);
    }

    // Makes a device current for a call and the caller's own one again afterwards.
    class device_scope
    {
    public:
        explicit device_scope(int device)
        {
            AEONB_CUDA(cudaGetDevice(&m_before));
            m_other = m_before != device;
            if (m_other)
                AEONB_CUDA(cudaSetDevice(device));
        }
        ~device_scope()
        {
            if (m_other)
                cudaSetDevice(m_before);
        }
        device_scope(const device_scope&) = delete;

    private:
        int  m_before = 0;
        bool m_other  = false;
    };

    inline int float_size(int dtype)
    {
        switch (dtype)
        {
        case AEONB_F32: return 4;
        case AEONB_F16:
        case AEONB_BF16: return 2;
        }
        throw std::invalid_argument("the type of the rows must be AEONB_F32, AEONB_F16 or AEONB_BF16");
    }

    inline bool aligned_to(const void* p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
}
