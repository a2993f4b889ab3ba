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

// float -> 16 bits rounds to the nearest, ties to even (v_cvt_pk_bf16_f32 / v_cvt_f16_f32): the one rounding of a result.
// NT: past the caches' replacement order, for results that are larger than what the caches could keep for their reader
template <bool NT, class T> __device__ __forceinline__ void put4(T *p, f32x4 v)
{
    Quad<T> q;
#pragma unroll
    for (int i = 0; i < 4; i++) q.v[i] = (T)v[i];
    if constexpr (!NT) *reinterpret_cast<Quad<T> *>(p) = q;
    else {
        typedef uint32_t W __attribute__((ext_vector_type(sizeof(q) / 4)));
        typedef W Any __attribute__((aligned(sizeof(T))));
        __builtin_nontemporal_store(__builtin_bit_cast(W, q), reinterpret_cast<Any *>(p));
    }
}

template <class T> __device__ __forceinline__ void store4(T *p, f32x4 v) { put4<false>(p, v); }

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

template <bool NT = false> __device__ __forceinline__ void store4_typed(void *base, int type, uint64_t at, int m, f32x4 v)
{
    if (m >= 4) {
        if (type == OPAL_F32) put4<NT>((float *)base + at, v);
        else if (type == OPAL_F16) put4<NT>((f16_t *)base + at, v);
        else put4<NT>((bf16_t *)base + at, v);
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

// Four neighbouring elements as they lie in memory, so that loads can be started well before they are used (m of them in range;
// the others are zeros).
template <class T> struct RawOf { uint32_t w[sizeof(T)]; };
template <class T> __device__ __forceinline__ RawOf<T> load_raw_of(const T *p, int m)
{
    RawOf<T> r = {};
    if (m >= 4) {
        const Quad<T> q = *reinterpret_cast<const Quad<T> *>(p);
        r = __builtin_bit_cast(RawOf<T>, q);
    } else {
#pragma unroll
        for (int i = 0; i < 3; i++)
            if (i < m) {
                if constexpr (sizeof(T) == 4) r.w[i] = ((const uint32_t *)p)[i];
                else r.w[i / 2] |= (uint32_t)((const uint16_t *)p)[i] << (16 * (i & 1));
            }
    }
    return r;
}
template <class T> __device__ __forceinline__ f32x4 decode_of(const RawOf<T> &r)
{
    const Quad<T> q = __builtin_bit_cast(Quad<T>, r);
    return f32x4{(float)q.v[0], (float)q.v[1], (float)q.v[2], (float)q.v[3]};
}

// Sum and maximum over groups of WIDTH (16, 32, 64) lanes, in all of their lanes, without LDS: rotations within 16 lanes, then exchanges of
// 16 and of 32 lanes.  Both sides of an exchange add the same two numbers, so that all lanes get the same bits.
template <int ROTATE> __device__ __forceinline__ float rotated(float v)
{
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + ROTATE, 0xf, 0xf, true));
#else
    return v;
#endif
}
template <int WIDTH> struct Pair { float a, b; };
template <int LANES> __device__ __forceinline__ Pair<LANES> exchanged(float v)
{
#ifdef __HIP_DEVICE_COMPILE__
    const uint32_t x = __builtin_bit_cast(uint32_t, v);
    // (element by element into plain integers: a bit cast of a vector's element takes its first one)
    uint32_t lo, hi;
    if constexpr (LANES == 16) {
        const auto p = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        lo = p[0];
        hi = p[1];
    } else {
        const auto p = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        lo = p[0];
        hi = p[1];
    }
    return {__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
#else
    return {v, v};
#endif
}
template <int LANES> __device__ __forceinline__ float add_exchanged(float v)
{
    const auto p = exchanged<LANES>(v);
    return p.a + p.b;
}
template <int WIDTH = WAVE> __device__ __forceinline__ float wave_sum(float v)
{
    v += rotated<8>(v);
    v += rotated<4>(v);
    v += rotated<2>(v);
    v += rotated<1>(v);
    if constexpr (WIDTH >= 32) v = add_exchanged<16>(v);
    if constexpr (WIDTH >= 64) v = add_exchanged<32>(v);
    return v;
}

// NaN never wins: a row's maximum is that of its numbers
template <int WIDTH = WAVE> __device__ __forceinline__ float wave_max(float v)
{
    v = fmaxf(v, rotated<8>(v));
    v = fmaxf(v, rotated<4>(v));
    v = fmaxf(v, rotated<2>(v));
    v = fmaxf(v, rotated<1>(v));
    if constexpr (WIDTH >= 32) {
        const auto p = exchanged<16>(v);
        v = fmaxf(p.a, p.b);
    }
    if constexpr (WIDTH >= 64) {
        const auto p = exchanged<32>(v);
        v = fmaxf(p.a, p.b);
    }
    return v;
}

// orders LDS accesses of one wave's lanes with each other (a wave's LDS operations complete in order; this keeps the compiler's)
__device__ __forceinline__ void wave_order()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

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
