// Element types, 4-wide loads and stores and wave reductions shared by the score head's kernels (opal_head.hip: layer norm and
// softmax; opal_linear*.hip: matrix products).
#pragma once
#include "opal_internal.h"

namespace opal_head {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int WAVE = 64;

// four consecutive elements at the alignment of ONE element: rows start wherever the caller's row stride puts them, and gfx950
// takes 8- and 16-byte global accesses at any byte address, so one instruction serves every stride
template <class T> struct __attribute__((packed, aligned(sizeof(T)))) Quad { T v[4]; };

template <class T> __device__ __forceinline__ f32x4 load4(const T *p)
{
    const Quad<T> q = *reinterpret_cast<const Quad<T> *>(p);
    return f32x4{(float)q.v[0], (float)q.v[1], (float)q.v[2], (float)q.v[3]};
}

// float -> 16 bits rounds to the nearest, ties to even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32): the one rounding of a result
template <class T> __device__ __forceinline__ void store4(T *p, f32x4 v)
{
    Quad<T> q;
#pragma unroll
    for (int i = 0; i < 4; i++) q.v[i] = (T)v[i];
    *reinterpret_cast<Quad<T> *>(p) = q;
}

// the same for a matrix whose type is known at run time only (uniform over the launch: a scalar branch), with `m` of the four
// columns in range; columns out of range read as `fill` and are not written
__device__ __forceinline__ f32x4 load4_typed(const void *base, int type, uint64_t at, int m, float fill = 0.f)
{
    if (m >= 4) {
        if (type == OPAL_F32) return load4((const float *)base + at);
        if (type == OPAL_F16) return load4((const f16_t *)base + at);
        return load4((const bf16_t *)base + at);
    }
    f32x4 r = {fill, fill, fill, fill};
#pragma unroll
    for (int i = 0; i < 3; i++)
        if (i < m)
            r[i] = type == OPAL_F32 ? ((const float *)base)[at + i]
                 : type == OPAL_F16 ? (float)((const f16_t *)base)[at + i] : (float)((const bf16_t *)base)[at + i];
    return r;
}

__device__ __forceinline__ void store4_typed(void *base, int type, uint64_t at, int m, f32x4 v)
{
    if (m >= 4) {
        if (type == OPAL_F32) store4((float *)base + at, v);
        else if (type == OPAL_F16) store4((f16_t *)base + at, v);
        else store4((bf16_t *)base + at, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 3; i++)
        if (i < m) {
            if (type == OPAL_F32) ((float *)base)[at + i] = v[i];
            else if (type == OPAL_F16) ((f16_t *)base)[at + i] = (f16_t)v[i];
            else ((bf16_t *)base)[at + i] = (bf16_t)v[i];
        }
}

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, WAVE);
    return v;
}

// NaN never wins: a row's maximum is that of its numbers
__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, WAVE));
    return v;
}

// orders LDS accesses of one wave's lanes with each other (a wave's LDS operations complete in order; this keeps the compiler's)
__device__ __forceinline__ void wave_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

inline int type_bytes(int type) { return type == OPAL_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == OPAL_F32 || type == OPAL_F16 || type == OPAL_BF16; }

// makes the ctx's device current for a call and puts the caller's back
struct OnDevice {
    int before = -1;
    hipError_t err;
    explicit OnDevice(int device)
    {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;
    }
    ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};

}  // namespace opal_head
