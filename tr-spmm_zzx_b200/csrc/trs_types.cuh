// Elements of fp32, fp16 or bf16 rows, read and written in aligned pieces and computed with in fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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

// A 16-byte piece as floats.
__device__ __forceinline__ void as_floats(const Piece<float, 4>& p, float (&v)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = p.v[k];
}
__device__ __forceinline__ void as_floats(const Piece<__half, 8>& p, float (&v)[8]) {
#pragma unroll
    for (int k = 0; k < 8; k += 2) {
        const float2 f = __half22float2(__halves2half2(p.v[k], p.v[k + 1]));
        v[k] = f.x;
        v[k + 1] = f.y;
    }
}
__device__ __forceinline__ void as_floats(const Piece<__nv_bfloat16, 8>& p, float (&v)[8]) {
    const uint4 w = *(const uint4*)&p;   // bf16 is the upper half of fp32
    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v[2 * k] = __uint_as_float(u[k] << 16);
        v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
    }
}

// Elements k and k + 1 of a piece.
template <class T, int N>
__device__ __forceinline__ float2 two_of(const Piece<T, N>& p, int k) {
    if constexpr (sizeof(T) == 4) return make_float2(p.v[k], p.v[k + 1]);
    else if constexpr (std::is_same<T, __half>::value) return __half22float2(__halves2half2(p.v[k], p.v[k + 1]));
    else return __bfloat1622float2(__halves2bfloat162(p.v[k], p.v[k + 1]));
}
template <class T, int N>
__device__ __forceinline__ void add_piece(float (&acc)[N], const Piece<T, N>& p) {
    if constexpr (N >= 2) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const float2 s = __fadd2_rn(make_float2(acc[k], acc[k + 1]), two_of(p, k));
            acc[k] = s.x;
            acc[k + 1] = s.y;
        }
    } else {
        acc[0] += as_float(p.v[0]);
    }
}

// x times a factor, in fp32, rounded once: pieces of N elements, two at a time.
template <class TO, class TI, int N>
__device__ __forceinline__ Piece<TO, N> scaled(const Piece<TI, N>& p, float mul) {
    Piece<TO, N> q;
    if constexpr (N >= 2) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            const float2 v = __fmul2_rn(two_of(p, k), make_float2(mul, mul));
            if constexpr (std::is_same<TO, __half>::value) *(__half2*)&q.v[k] = __float22half2_rn(v);
            else if constexpr (std::is_same<TO, __nv_bfloat16>::value) *(__nv_bfloat162*)&q.v[k] = __float22bfloat162_rn(v);
            else q.v[k] = v.x, q.v[k + 1] = v.y;
        }
    } else {
        q.v[0] = from_float<TO>(as_float(p.v[0]) * mul);
    }
    return q;
}

// Largest element of a piece (NaN where one is); 16-bit types two at a time.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_of(const Piece<float, 4>& p) { return max_nan(max_nan(p.v[0], p.v[1]), p.v[2], p.v[3]); }
__device__ __forceinline__ float max_of(const Piece<__half, 8>& p) {
    const __half2* h = (const __half2*)&p;
    const float2 f = __half22float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
    return max_nan(f.x, f.y);
}
__device__ __forceinline__ float max_of(const Piece<__nv_bfloat16, 8>& p) {
    const __nv_bfloat162* h = (const __nv_bfloat162*)&p;
    const float2 f = __bfloat1622float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
    return max_nan(f.x, f.y);
}

// -inf where the byte of the mask is 0: `bytes` has four of them, the first for element `from` of the piece.
__device__ __forceinline__ unsigned nonzero_bytes(unsigned bytes) {   // the top bit of every byte that is not 0 (the others as they come)
    return ((bytes & 0x7f7f7f7fu) + 0x7f7f7f7fu) | bytes;
}
__device__ __forceinline__ void mask_four(Piece<float, 4>& p, int from, unsigned bytes) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (!(bytes >> (8 * k) & 0xff)) p.v[from + k] = -INFINITY;
}
template <unsigned SELECT>
__device__ __forceinline__ unsigned spread(unsigned x) {   // prmt with the bytes' top bits repeated
    unsigned r;
    asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(x), "n"(SELECT));
    return r;
}
template <unsigned INF>
__device__ __forceinline__ void mask_four_16(unsigned* two, unsigned bytes) {
    const unsigned top = nonzero_bytes(bytes);
    const unsigned lo = spread<0x9988>(top), hi = spread<0xbbaa>(top);   // top bits spread over 16 bits each
    two[0] = (two[0] & lo) | (INF & ~lo);
    two[1] = (two[1] & hi) | (INF & ~hi);
}
__device__ __forceinline__ void mask_four(Piece<__half, 8>& p, int from, unsigned bytes) {
    mask_four_16<0xfc00fc00u>((unsigned*)&p + from / 2, bytes);
}
__device__ __forceinline__ void mask_four(Piece<__nv_bfloat16, 8>& p, int from, unsigned bytes) {
    mask_four_16<0xff80ff80u>((unsigned*)&p + from / 2, bytes);
}

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
