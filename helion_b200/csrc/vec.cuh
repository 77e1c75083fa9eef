// Element conversions and 16-byte vectors of bf16, fp16 and fp32 rows.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

namespace lce {

template <class T> struct Cvt;
template <> struct Cvt<__nv_bfloat16> {
    static __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
};
template <> struct Cvt<__half> {
    static __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
};
template <> struct Cvt<float> {
    static __device__ __forceinline__ float to_f(float x) { return x; }
    static __device__ __forceinline__ float from_f(float x) { return x; }
};

template <class T>
struct RmsTile {
    static constexpr int kVec = 16 / sizeof(T);
    static constexpr int kMaxVpt = 8;  // 256 threads x 8 vectors: 16384 16-bit or 8192 fp32 columns
};

// Columns c .. c + VEC of one row as a raw 16-byte vector; columns at or beyond H read as zero.
template <class T, bool VECTOR>
__device__ __forceinline__ uint4 rms_load(const T* __restrict__ row, int c, int H) {
    constexpr int VEC = RmsTile<T>::kVec;
    if (VECTOR) {
        return c < H ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0u, 0u, 0u, 0u);
    } else {
        alignas(16) T tmp[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) tmp[j] = (c + j < H) ? row[c + j] : Cvt<T>::from_f(0.f);
        return *reinterpret_cast<const uint4*>(tmp);
    }
}

// 16-byte vector <-> floats. The 16-bit forms convert two elements per instruction where the hardware
// can (bf16 -> fp32 is a shift or a mask of the packed word; fp32 -> 16-bit pairs is one cvt).
template <class T>
__device__ __forceinline__ void rms_unpack(const uint4& raw, float (&v)[RmsTile<T>::kVec]) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
        }
    }
}

template <class T>
__device__ __forceinline__ uint4 rms_pack(const float (&v)[RmsTile<T>::kVec]) {
    uint32_t w[4];
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = __float_as_uint(v[j]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <class T, bool VECTOR>
__device__ __forceinline__ void rms_store(T* __restrict__ row, int c, int H, const uint4& raw) {
    constexpr int VEC = RmsTile<T>::kVec;
    if (VECTOR) {
        if (c < H) *reinterpret_cast<uint4*>(row + c) = raw;
    } else {
        alignas(16) T tmp[VEC];
        *reinterpret_cast<uint4*>(tmp) = raw;
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (c + j < H) row[c + j] = tmp[j];
    }
}

// Two fp32 values that share an instruction where the hardware has one (multiply and fused multiply-add).
struct Pair {
    unsigned long long v;
};
__device__ __forceinline__ Pair pair(float lo, float hi) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
    return p;
}
__device__ __forceinline__ Pair both(float x) { return pair(x, x); }
__device__ __forceinline__ void split(Pair p, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p.v)); }
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}
__device__ __forceinline__ float sum(Pair p) {
    float lo, hi;
    split(p, lo, hi);
    return lo + hi;
}

template <class T>
__device__ __forceinline__ void unpack_pairs(const uint4& raw, Pair (&v)[RmsTile<T>::kVec / 2]) {
    float f[RmsTile<T>::kVec];
    rms_unpack<T>(raw, f);
#pragma unroll
    for (int j = 0; j < RmsTile<T>::kVec / 2; ++j) v[j] = pair(f[2 * j], f[2 * j + 1]);
}
template <class T>
__device__ __forceinline__ uint4 pack_pairs(const Pair (&v)[RmsTile<T>::kVec / 2]) {
    float f[RmsTile<T>::kVec];
#pragma unroll
    for (int j = 0; j < RmsTile<T>::kVec / 2; ++j) split(v[j], f[2 * j], f[2 * j + 1]);
    return rms_pack<T>(f);
}

}  // namespace lce
