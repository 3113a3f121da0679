// Rows of floating-point numbers -> 8-bit codes with one scale per row:
//   amax = max_k |x_k|,  scale = fl32(amax / 127),  q_k = round-half-even(127 x_k / amax)   (exact: no intermediate
//   rounding decides a code),  columns K .. cols - 1 zero.
// amax = 0: scale 0 and codes 0.  A NaN or an infinity in the row: scale NaN and codes 0, so every product of the row
// is NaN and no other row notices.
//
// Bound by HBM for many rows (one read, one write), by latency for one.  A row is held in registers between the two
// passes over it (maximum, then codes), so it is read once; a row too long for that is read a second time from L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "quantize.cuh"

namespace tmq {

struct QuantArgs {
    const void *X;
    int8_t *Q;
    float *scale;
    long long M, K, ldx, ldq, cols;        // cols >= K: columns written
};

// One row per TPR threads, 256 threads per block.  VEC: elements of one 16-byte load (1: the row is not 16-byte aligned
// and is read element by element).  CH: chunks of VEC elements a thread holds.
template <typename T, int TPR, int VEC, int CH>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantArgs a) {
    constexpr int ROWS = 256 / TPR;
    __shared__ float red[8];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int t = threadIdx.x % TPR;
    const long long m = (long long)blockIdx.x * ROWS + threadIdx.x / TPR;
    const bool live = m < a.M;
    const T *x = reinterpret_cast<const T *>(a.X) + (live ? m : 0) * a.ldx;
    const long long K = live ? a.K : 0;

    QuantChunk<T, VEC> held[CH];
    float amax = 0.0f;
    bool bad = false;
#pragma unroll
    for (int c = 0; c < CH; c++) held[c].load(x, ((long long)c * TPR + t) * VEC, K);
#pragma unroll
    for (int c = 0; c < CH; c++) held[c].peak(amax, bad);
    for (long long k = ((long long)CH * TPR + t) * VEC; k < K; k += (long long)TPR * VEC) {
        QuantChunk<T, VEC> v;
        v.load(x, k, K);
        v.peak(amax, bad);
    }
    if (bad) amax = __int_as_float(0x7f800000);          // one non-finite value marks the row
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (TPR > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) amax = fmaxf(amax, red[w]);
    }
    if (!live) return;
    const RowQuant rq(amax);
    if (t == 0) a.scale[m] = rq.scale;
    int8_t *q = a.Q + m * a.ldq;
#pragma unroll
    for (int c = 0; c < CH; c++) held[c].store(q, ((long long)c * TPR + t) * VEC, a.K, a.cols, rq);
    for (long long k = ((long long)CH * TPR + t) * VEC; k < a.cols; k += (long long)TPR * VEC) {
        QuantChunk<T, VEC> v;
        v.load(x, k, a.K);
        v.store(q, k, a.K, a.cols, rq);
    }
}

template <typename T, int TPR, int VEC, int CH>
static int launch_quantize(const QuantArgs &a, cudaStream_t st) {
    const long long rows = 256 / TPR, grid = (a.M + rows - 1) / rows;
    if (grid > 0x7FFFFFFF) return TMQ_ERR_UNSUPPORTED;
    return launch_chained(quantize_rows_kernel<T, TPR, VEC, CH>, a, (unsigned)grid, 256, 0, st);
}

template <typename T>
static int dispatch_quantize(const QuantArgs &a, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    const bool vec = aligned(a.X, 16) && (a.ldx * (long long)sizeof(T)) % 16 == 0 && aligned(a.Q, 16) && a.ldq % 16 == 0 &&
                     a.cols % 16 == 0;
    if (!vec) return launch_quantize<T, 256, 1, 8>(a, st);
    if (a.K <= 32 * V * 4 && a.M >= 8 * kNumSMs) return launch_quantize<T, 32, V, 4>(a, st);
    if (a.K <= 256 * V * 2) return launch_quantize<T, 256, V, 2>(a, st);
    return launch_quantize<T, 256, V, 8>(a, st);
}

}  // namespace tmq

using namespace tmq;

extern "C" int tmq_quantize_rows(const void *X, int x_type, int8_t *Q, float *scale, int64_t M, int64_t K, int64_t ldx,
                                 int64_t ldq, int64_t cols, void *stream) {
    if (M < 0 || K <= 0 || ldx < K || cols < K || ldq < cols || x_type < TMQ_TYPE_F32 || x_type > TMQ_TYPE_F16) return TMQ_ERR_ARG;
    if (M == 0) return TMQ_OK;
    if (!X || !Q || !scale) return TMQ_ERR_ARG;
    if (!aligned(X, x_type == TMQ_TYPE_F32 ? 4 : 2) || !aligned(scale, 4)) return TMQ_ERR_ALIGN;
    const QuantArgs a = {X, Q, scale, M, K, ldx, ldq, cols};
    if (x_type == TMQ_TYPE_F32) return dispatch_quantize<float>(a, (cudaStream_t)stream);
    if (x_type == TMQ_TYPE_BF16) return dispatch_quantize<__nv_bfloat16>(a, (cudaStream_t)stream);
    return dispatch_quantize<__half>(a, (cudaStream_t)stream);
}
