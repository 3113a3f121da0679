// Device pieces of the 8-bit row quantisation, shared by the row kernel and by the kernels that quantise on the fly.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace tmq {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// What a row's maximum fixes: its scale and the quotient 127 / amax.  A row whose maximum is tiny is lifted by 2^100 first
// (exact), which keeps the quotient finite.  amax = infinity stands for "the row holds a NaN or an infinity".
struct RowQuant {
    float scale, inv, lift, amax;
    bool dead;                           // codes are all zero: empty row or a non-finite one
    __device__ __forceinline__ explicit RowQuant(float peak) {
        const bool finite = peak <= 3.402823466e38f;
        dead = !finite || peak == 0.0f;
        scale = finite ? __fdiv_rn(peak, 127.0f) : __int_as_float(0x7fffffff);
        lift = peak < 7.888609e-31f ? 1.2676506e30f : 1.0f;        // 2^-100, 2^100
        amax = peak * lift;
        inv = dead ? 0.0f : __fdiv_rn(127.0f, amax);
    }
    // round-half-even(127 x / amax).  The 32-bit product is off by at most 127 * 2^-23 < 2e-5; where that could decide
    // the rounding, 254 |x| is compared with the border (2 n + 1) amax, both exact in 64 bits.
    __device__ __forceinline__ int code(float x) const {
        if (dead) return 0;
        const float xl = x * lift, t = xl * inv;
        const float r = rintf(t);
        if (fabsf(t - r) < 0.4999f) return (int)r;
        const float n = floorf(fabsf(t));
        const double have = 254.0 * (double)fabsf(xl), border = (2.0 * (double)n + 1.0) * (double)amax;
        int c = (int)n;
        if (have > border || (have == border && (c & 1))) c++;
        return x < 0.0f ? -c : c;
    }
};

// VEC consecutive elements of a row, zero beyond K.  VEC > 1 means 16 bytes, read with one load where all of them exist.
template <typename T, int VEC>
struct QuantChunk {
    T v[VEC];
    __device__ __forceinline__ void load(const T *x, long long k, long long K) {
        if (VEC > 1 && k + VEC <= K) {
            const uint4 u = *reinterpret_cast<const uint4 *>(x + k);
            *reinterpret_cast<uint4 *>(v) = u;
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++) v[i] = k + i < K ? x[k + i] : T(0.0f);
        }
    }
    __device__ __forceinline__ void peak(float &amax, bool &bad) const {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const float f = fabsf(to_f32(v[i]));
            bad |= !(f <= 3.402823466e38f);
            amax = fmaxf(amax, f);
        }
    }
    __device__ __forceinline__ void store(int8_t *q, long long k, long long K, long long cols, const RowQuant &rq) const {
        if (k >= cols) return;
        if (VEC > 1) {                   // cols is a multiple of 16: the whole vector exists
            uint32_t w[(VEC + 3) / 4];
#pragma unroll
            for (int i = 0; i < VEC; i += 4) {
                w[i / 4] = 0;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (i + j < VEC) w[i / 4] |= (uint32_t)(rq.code(to_f32(v[(i + j) % VEC])) & 0xff) << (8 * j);
            }
            if (VEC == 8) *reinterpret_cast<uint2 *>(q + k) = make_uint2(w[0], w[(VEC + 3) / 4 - 1]);
            else *reinterpret_cast<uint32_t *>(q + k) = w[0];
        } else {
            q[k] = (int8_t)rq.code(to_f32(v[0]));
        }
    }
};

}  // namespace tmq
