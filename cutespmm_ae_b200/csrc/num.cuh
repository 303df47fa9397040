// The storage types of the operators in pattern_ops.hpp (fp32, fp16, bf16) and 16-byte groups of them: values are held in fp32
// between a load and the one rounding of the store.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/cutespmm.h"

namespace cutespmm {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// V elements that one load brings: 16 bytes, or a single element where addresses or sizes do not allow that.
template <class T, int V> struct alignas(V * sizeof(T)) Pack {
    T x[V];
};
template <class T> constexpr int kVec = 16 / (int)sizeof(T);

template <class T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T *p)
{
    Pack<T, V> r;
    if constexpr (V * sizeof(T) == 16) {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p));
        r = *reinterpret_cast<const Pack<T, V> *>(&u);
    } else
        r.x[0] = p[0];
    return r;
}
template <class T, int V> __device__ __forceinline__ void store_pack(T *p, const float (&f)[V])
{
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.x[i] = from_f32<T>(f[i]);
    if constexpr (V * sizeof(T) == 16) __stcs(reinterpret_cast<uint4 *>(p), *reinterpret_cast<const uint4 *>(&r));
    else *p = r.x[0];
}

// fn<T>() for the element type a call names
template <class Fn> cudaError_t for_dtype(int dtype, Fn &&fn)
{
    switch (dtype) {
        case CUTESPMM_F32: return fn(float());
        case CUTESPMM_F16: return fn(__half());
        case CUTESPMM_BF16: return fn(__nv_bfloat16());
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace cutespmm
