// Row access shared by the layer norm and the activation checkpoint kernels: E consecutive elements of a row at a
// time, fp32 / bf16 / fp16 in memory and fp32 in registers, and the 8-bit row quantiser of a checkpoint.
//
// E is the largest of {16 bytes, 2 elements, 1 element} that divides the row length and that every pointer and row
// stride of the call is aligned to (row_step below), so that no access needs a tail and none is misaligned.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include "quant_core.cuh"

namespace sgnn {

// element types of the entry points that take more than fp32
inline size_t elem_bytes(int dtype) { return dtype == SGNN_F32 ? 4 : 2; }
inline bool elem_known(int dtype) { return dtype == SGNN_F32 || dtype == SGNN_BF16 || dtype == SGNN_F16; }

// One operand of a row kernel: base, row stride in elements, bytes per element (nullptr: not there).
struct RowOperand {
    const void *p;
    int64_t ld;
    size_t bytes;
};

// Elements per access for rows of H elements: `wide` (16 bytes of the activation type), 2 or 1.
template <int N>
inline int row_step(int64_t H, int wide, const RowOperand (&ops)[N])
{
    for (int e : {wide, 2}) {
        bool ok = H % e == 0;
        for (const RowOperand &o : ops) {
            if (o.p == nullptr) continue;
            const size_t a = o.bytes * e < 16 ? o.bytes * e : 16;  // fp32 parameters of 8 elements: two 16-byte accesses
            ok = ok && reinterpret_cast<uintptr_t>(o.p) % a == 0 && (size_t)(o.ld * o.bytes) % a == 0;
        }
        if (ok) return e;
    }
    return 1;
}

#ifdef __CUDACC__

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// B bytes as one register type
template <int B>
struct Word;
template <>
struct Word<1> { using type = uint8_t; };
template <>
struct Word<2> { using type = unsigned short; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<16> { using type = uint4; };

// E elements at p (aligned to E * sizeof(T), at most 16 bytes), read once
template <class T, int E>
__device__ __forceinline__ void load_row(const T *p, float (&v)[E])
{
    union {
        typename Word<E * sizeof(T)>::type w;
        T e[E];
    } u;
    u.w = __ldcs(reinterpret_cast<const typename Word<E * sizeof(T)>::type *>(p));
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = to_f32<T>(u.e[i]);
}

template <class T, int E>
__device__ __forceinline__ void store_row(T *p, const float (&v)[E])
{
    union {
        typename Word<E * sizeof(T)>::type w;
        T e[E];
    } u;
#pragma unroll
    for (int i = 0; i < E; ++i) u.e[i] = from_f32<T>(v[i]);
    __stcs(reinterpret_cast<typename Word<E * sizeof(T)>::type *>(p), u.w);
}

// E entries of a parameter vector that is fp32 (`f32`) or of the activation type; `missing` where there is none
template <class T, int E>
__device__ __forceinline__ void load_param(const void *p, bool f32, int64_t c, float missing, float (&v)[E])
{
    if (p == nullptr) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = missing;
    } else if (f32) {
        if constexpr (E >= 4) {
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const float4 t = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(p) + c + i));
                v[i] = t.x, v[i + 1] = t.y, v[i + 2] = t.z, v[i + 3] = t.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = __ldg(static_cast<const float *>(p) + c + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = to_f32<T>(static_cast<const T *>(p)[c + i]);
    }
}

// ---- the 8-bit row quantiser ----
// zp = min, sc = (max - min) / 255, code = rne((x - zp) / sc), all IEEE fp32.  A range below 255 FLT_MIN counts as
// none (sc = 1, every code 0: the row comes back as its minimum), so that sc is never subnormal and no code passes 255.
// A row with a NaN or an infinity, or whose range is above FLT_MAX, gets NaN parameters: it comes back as NaN
// instead of as plausible numbers.
__device__ __forceinline__ RowQ row_quantiser(float mn, float mx, float poison)
{
    const float range = __fsub_rn(mx, mn);
    RowQ q;
    q.mn = mn;
    q.sc = __fdiv_rn(range, 255.0f);
    if (q.sc < FLT_MIN) q.sc = 1.0f;
    if (!(poison == 0.0f) || !(range <= FLT_MAX)) q.mn = q.sc = __int_as_float(0x7fffffff);
    q.rinv = __fdiv_rn(1.0f, q.sc);
    q.thr = q.sc * (0.5f * (1.0f - 1.0f / 4096.0f));
    return q;
}

// one code, by the same verified reciprocal as encode4: candidate, exact residual, division where it is not proved
__device__ __forceinline__ uint32_t encode1(float x, const RowQ q)
{
    const float d = __fsub_rn(x, q.mn);
    const float u = __fmaf_rn(d, q.rinv, 12582912.0f);
    const float res = __fmaf_rn(__fsub_rn(u, 12582912.0f), -q.sc, d);
    uint32_t b = __float_as_uint(u);
    if (!(fabsf(res) <= q.thr)) b = (uint32_t)code_of(x, q.mn, q.sc);
    return b & 0xFFu;
}

// E codes of one access, stored at p (aligned to E)
template <int E>
__device__ __forceinline__ void store_codes(uint8_t *p, const float (&v)[E], const RowQ q)
{
    if constexpr (E >= 4) {
#pragma unroll
        for (int i = 0; i < E; i += 4)
            __stcs(reinterpret_cast<uint32_t *>(p + i), encode4(make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]), q));
    } else if constexpr (E == 2) {
        __stcs(reinterpret_cast<unsigned short *>(p), (unsigned short)(encode1(v[0], q) | (encode1(v[1], q) << 8)));
    } else {
        __stcs(p, (uint8_t)encode1(v[0], q));
    }
}

// E codes at p (aligned to E) as fp32 integers
template <int E>
__device__ __forceinline__ void load_codes(const uint8_t *p, float (&v)[E])
{
    union {
        typename Word<E>::type w;
        uint8_t e[E];
    } u;
    u.w = __ldcs(reinterpret_cast<const typename Word<E>::type *>(p));
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = (float)u.e[i];
}

__device__ __forceinline__ float all_sum(float v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}

// The same over the LANES lanes that share a row, where a warp has several rows
template <int LANES>
__device__ __forceinline__ float row_sum(float v)
{
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
    return v;
}
template <int LANES>
__device__ __forceinline__ float row_min(float v)
{
    if constexpr (LANES == 32) {
        v = redux_min(v);
    } else {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(FULL, v, o));
    }
    return v;
}
template <int LANES>
__device__ __forceinline__ float row_max(float v)
{
    if constexpr (LANES == 32) {
        v = redux_max(v);
    } else {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
    }
    return v;
}

// Lanes for a row of H elements, at most eight elements a lane up to 256: narrow rows share a warp.  600000 rows of 16 fp32, layer
// norm in both directions: 53 us with four lanes a row, 78 with eight, 189 with 32; 64 in bf16 96 us against 298, 128 fp32 246
// against 275; checkpoint and back, 16 fp32: 28, 45 and 132 us.
inline int row_lanes(int64_t H) { return H <= 32 ? 4 : H <= 64 ? 8 : H <= 128 ? 16 : 32; }

#endif  // __CUDACC__
}  // namespace sgnn
