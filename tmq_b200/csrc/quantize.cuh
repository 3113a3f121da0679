// Device pieces of the 8-bit row quantisation, shared by the row kernel and by the kernels that quantise on the fly.
//
// A vector is 16 bytes of a row (8 elements of two bytes, 4 of four).  Its largest magnitude is taken on the bit patterns:
// with the sign cleared they order like the numbers, infinities and NaN on top, so one integer maximum (two elements at a
// time for two-byte types) yields the row's maximum and whether the row is finite.  A code is the low byte of
// fma(x, 127 / amax, 1.5 * 2^23), whose rounding to an integer is round-half-even; the remainder of that rounding tells
// when the rounded quotient 127 / amax could have decided it, and only then the vector is redone with exact comparisons.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace tmq {

template <typename T>
struct QuantType;
template <>
struct QuantType<float> {
    static constexpr int V = 4;
    static constexpr uint32_t INF = 0x7f800000u;
    static __device__ __forceinline__ float get(const uint32_t (&w)[4], int i) { return __uint_as_float(w[i]); }
    static __device__ __forceinline__ uint32_t peak(uint32_t p, uint32_t w) { return max(p, w & 0x7fffffffu); }
    static __device__ __forceinline__ uint32_t fold(uint32_t p) { return p; }
    static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits); }
};
template <>
struct QuantType<__nv_bfloat16> {
    static constexpr int V = 8;
    static constexpr uint32_t INF = 0x7f80u;
    static __device__ __forceinline__ float get(const uint32_t (&w)[4], int i) {
        return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
    }
    static __device__ __forceinline__ uint32_t peak(uint32_t p, uint32_t w) { return __vmaxu2(p, w & 0x7fff7fffu); }
    static __device__ __forceinline__ uint32_t fold(uint32_t p) { return max(p & 0xffffu, p >> 16); }
    static __device__ __forceinline__ float value(uint32_t bits) { return __uint_as_float(bits << 16); }
};
template <>
struct QuantType<__half> {
    static constexpr int V = 8;
    static constexpr uint32_t INF = 0x7c00u;
    static __device__ __forceinline__ float get(const uint32_t (&w)[4], int i) {
        return __half2float(__ushort_as_half((unsigned short)((i & 1) ? (w[i >> 1] >> 16) : (w[i >> 1] & 0xffffu))));
    }
    static __device__ __forceinline__ uint32_t peak(uint32_t p, uint32_t w) { return __vmaxu2(p, w & 0x7fff7fffu); }
    static __device__ __forceinline__ uint32_t fold(uint32_t p) { return max(p & 0xffffu, p >> 16); }
    static __device__ __forceinline__ float value(uint32_t bits) { return __half2float(__ushort_as_half((unsigned short)bits)); }
};

// What a row's largest magnitude (its bit pattern, QuantType::fold) fixes.
template <typename T>
struct RowQuant {
    float scale, inv, amax, lift;
    bool dead;                           // all codes zero: an empty row or one with a NaN or an infinity
    bool tiny;                           // below 2^-100: lifted by 2^100 (exact) so that 127 / amax stays finite
    __device__ __forceinline__ explicit RowQuant(uint32_t bits) {
        const bool finite = bits < QuantType<T>::INF;
        const float peak = finite ? QuantType<T>::value(bits) : 0.0f;
        dead = peak == 0.0f;
        scale = finite ? __fdiv_rn(peak, 127.0f) : __int_as_float(0x7fffffff);
        tiny = peak < 7.888609e-31f;
        lift = tiny ? 1.2676506e30f : 1.0f;
        amax = peak * lift;
        inv = dead ? 0.0f : __fdiv_rn(127.0f, amax);
    }
    // 254 |x| against the border (2 n + 1) amax between the codes n and n + 1, both exact in 64 bits
    __device__ __forceinline__ int exact(float x) const {
        if (dead) return 0;
        const float xl = fabsf(x) * lift, n = floorf(xl * inv);
        // the quotient is off by less than 2e-5, so n is the lower neighbour unless it sits on an integer: step as needed
        int c = (int)n;
        const double have = 254.0 * (double)xl;
        if (have < (2.0 * c - 1.0) * (double)amax) c--;
        const double border = (2.0 * c + 1.0) * (double)amax;
        if (have > border || (have == border && (c & 1))) c++;
        return x < 0.0f ? -c : c;
    }
};

__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

template <typename T>
struct QuantVec {
    static constexpr int V = QuantType<T>::V;
    uint32_t w[4];
    // elements k .. k + V - 1 of a row, zero from K on; VLOAD: the row is 16-byte aligned
    template <bool VLOAD>
    __device__ __forceinline__ void load(const T *x, long long k, long long K) {
        if (VLOAD && k + V <= K) {
            const uint4 u = *reinterpret_cast<const uint4 *>(x + k);
            w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (sizeof(T) == 4) {
                w[i] = k + i < K ? reinterpret_cast<const uint32_t *>(x)[k + i] : 0u;
            } else {
                const uint16_t *h = reinterpret_cast<const uint16_t *>(x);
                const uint32_t lo = k + 2 * i < K ? h[k + 2 * i] : 0u, hi = k + 2 * i + 1 < K ? h[k + 2 * i + 1] : 0u;
                w[i] = lo | hi << 16;
            }
        }
    }
    __device__ __forceinline__ void peak(uint32_t &p) const {
#pragma unroll
        for (int i = 0; i < 4; i++) p = QuantType<T>::peak(p, w[i]);
    }
    // the V codes, four to a word
    __device__ __forceinline__ void codes(const RowQuant<T> &rq, uint32_t (&q)[V / 4]) const {
        const float magic = 12582912.0f;                 // 1.5 * 2^23
        float far = 0.0f;                                // largest remainder of the roundings
        uint32_t b[V];
        const uint64_t inv2 = pack2(rq.inv, rq.inv), magic2 = pack2(magic, magic), minus2 = pack2(-1.0f, -1.0f);
#pragma unroll
        for (int i = 0; i < V; i += 2) {                 // two elements per instruction
            const uint64_t x = pack2(QuantType<T>::get(w, i), QuantType<T>::get(w, i + 1));
            const uint64_t r = fma2(x, inv2, magic2);
            const uint64_t d = fma2(x, inv2, fma2(r, minus2, magic2));
            float lo, hi;
            unpack2(d, lo, hi);
            far = fmaxf(far, fmaxf(fabsf(lo), fabsf(hi)));
            b[i] = (uint32_t)r;
            b[i + 1] = (uint32_t)(r >> 32);
        }
        // the quotient is off by at most 127 * 2^-24, the remainder by as much again: 2e-5 covers both
        if (far > 0.49998f || rq.tiny) {
#pragma unroll
            for (int i = 0; i < V; i++) b[i] = (uint32_t)rq.exact(QuantType<T>::get(w, i));
        }
#pragma unroll
        for (int i = 0; i < V; i += 4)
            q[i / 4] = __byte_perm(__byte_perm(b[i], b[i + 1], 0x0040), __byte_perm(b[i + 2], b[i + 3], 0x0040), 0x5410);
    }
};

}  // namespace tmq
