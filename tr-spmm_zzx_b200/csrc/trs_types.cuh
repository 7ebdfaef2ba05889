// Elements of fp32, fp16 or bf16 rows, read and written in aligned pieces and computed with in fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "trs_common.cuh"

namespace trs {

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N neighbouring elements, one load or store of up to 16 bytes.
template <class T, int N>
struct alignas(sizeof(T) * N) Piece {
    T v[N];
};

inline int type_bytes(int type) { return type == TRS_TYPE_F32 ? 4 : 2; }
inline bool type_known(int type) { return type == TRS_TYPE_F32 || type == TRS_TYPE_F16 || type == TRS_TYPE_BF16; }

// fn(element of the type), for the type of a code.
template <class Fn>
int with_type(int type, Fn fn) {
    if (type == TRS_TYPE_F32) return fn(float());
    if (type == TRS_TYPE_F16) return fn(__half());
    return fn(__nv_bfloat16());
}

}  // namespace trs
