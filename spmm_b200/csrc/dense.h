// Shared by the dense operators around a sparse product (norm.cu, lora.cu): element access by type, argument checks.
#pragma once

#include <cstring>
#include <initializer_list>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "internal.h"

namespace tca {

tcaspmm_status cuda_fail(cudaError_t e, const char *what);

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Element i of an array whose type is known at run time (0 fp32, 1 fp16, 2 bf16): the same branch for every thread.
// 16-bit elements are loaded as integers: the header's own __ldg of a 16-bit float is an assembly statement without side
// effects, which the compiler may execute ahead of the branch that guards it (seen as a read through a NULL weight).
__device__ __forceinline__ float load_as(const void *p, int type, long long i)
{
    if (type == 0) return __ldg((const float *)p + i);
    if (type == 1) return __half2float(__ushort_as_half(__ldg((const unsigned short *)p + i)));
    return __bfloat162float(__ushort_as_bfloat16(__ldg((const unsigned short *)p + i)));
}
__device__ __forceinline__ void store_as(void *p, int type, long long i, float v)
{
    if (type == 0)
        ((float *)p)[i] = v;
    else if (type == 1)
        ((__half *)p)[i] = __float2half_rn(v);
    else
        ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
}

template <int BYTES> struct Bits;
template <> struct Bits<2> { using type = unsigned short; };
template <> struct Bits<4> { using type = unsigned; };
template <> struct Bits<8> { using type = uint2; };
template <> struct Bits<16> { using type = uint4; };

// VEC elements of type T as they lie in memory (at most 16 bytes).
template <typename T, int VEC>
struct Pack {
    typename Bits<sizeof(T) * VEC>::type bits;
    __device__ void load(const T *p) { bits = __ldg(reinterpret_cast<const decltype(bits) *>(p)); }
    __device__ void zero() { bits = {}; }
    // Element i as fp32 (i a constant of an unrolled loop).
    __device__ float get(int i) const
    {
        if constexpr (sizeof(T) == 4) {
            float v[VEC];
            memcpy(v, &bits, sizeof bits);
            return v[i];
        } else if constexpr (VEC == 1) {
            T v;
            memcpy(&v, &bits, sizeof v);
            return to_float(v);
        } else {
            unsigned w[VEC / 2];
            memcpy(w, &bits, sizeof bits);
            const unsigned two = w[i >> 1];
            if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(i & 1 ? two & 0xffff0000u : two << 16);
            return __half2float(__ushort_as_half((unsigned short)(i & 1 ? two >> 16 : two)));
        }
    }
};

// Type code of the kernels; TF32 is fp32 storage.
inline int type_code(tcaspmm_dtype dt) { return dt == TCASPMM_F16 ? 1 : dt == TCASPMM_BF16 ? 2 : 0; }

// Calls f(T{}) with the element type of code 0, 1 or 2.
template <typename F>
inline tcaspmm_status with_type(int code, F &&f)
{
    if (code == 0) return f(float{});
    if (code == 1) return f(__half{});
    return f(__nv_bfloat16{});
}

inline int size_of(int code) { return code == 0 ? 4 : 2; }

// Elements of the type of `code` may lie at p.
inline bool pointer_ok(const void *p, int code) { return (uintptr_t)p % size_of(code) == 0; }

// A matrix argument: an inner extent of `cols`, a leading dimension of `ld`, and a pointer unless it is empty.
inline bool matrix_ok(const void *p, int64_t rows, int64_t cols, int64_t ld, int code)
{
    return ld >= cols && (p != nullptr || rows == 0 || cols == 0) && pointer_ok(p, code);
}

// The memory of a matrix (or, with one row, of an array) that is passed as an argument.
struct Extent {
    const char *p;
    int64_t rows, bytes, pitch;  // of a row, and from one to the next
    Extent(const void *at, int64_t r, int64_t cols, int64_t ld, int size)
        : p((const char *)at), rows(at && cols > 0 ? r : 0), bytes(cols * size), pitch(ld * size)
    {
    }
    const char *end() const { return p + (rows - 1) * pitch + bytes; }
};

// Whether two share memory; of two windows of one wider matrix that lie side by side, none is shared.
inline bool overlap(const Extent &a, const Extent &b)
{
    if (a.rows <= 0 || b.rows <= 0 || a.end() <= b.p || b.end() <= a.p) return false;
    if (a.pitch != b.pitch || a.rows == 1 || b.rows == 1) return true;
    const int64_t d = ((b.p - a.p) % a.pitch + a.pitch) % a.pitch;
    return d < a.bytes || a.pitch - d < b.bytes;
}

// Whether an output shares memory with any of the other arguments.
inline bool overlaps_any(const Extent &out, std::initializer_list<Extent> others)
{
    for (const Extent &o : others)
        if (overlap(out, o)) return true;
    return false;
}

}  // namespace tca
