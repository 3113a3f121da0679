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
    int vstore;
};

// One row per TPR threads, 256 threads per block, CH vectors held per thread; the rest of a longer row is read twice.  Six
// blocks per SM where their registers allow it (8192 x 8192 bf16: 36.3 us, 5.5 TB/s, against 37.5 with five and 40 with seven),
// four for the others (1037 x 5003 fp32 rows without alignment: 7.6 us, 9.0 with more registers and fewer blocks).
template <typename T, bool VLOAD, int TPR, int CH>
__global__ void __launch_bounds__(256, VLOAD && CH <= 4 ? 6 : sizeof(T) == 2 && !VLOAD && CH > 4 ? 3 : 4) quantize_rows_kernel(const QuantArgs a) {
    constexpr int ROWS = 256 / TPR, V = QuantType<T>::V;
    __shared__ uint32_t red[8];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int t = threadIdx.x % TPR;
    const long long m = (long long)blockIdx.x * ROWS + threadIdx.x / TPR;
    const bool live = m < a.M;
    const T *x = reinterpret_cast<const T *>(a.X) + (live ? m : 0) * a.ldx;
    const long long K = live ? a.K : 0;

    QuantVec<T> held[CH];
    uint32_t peak = 0;
#pragma unroll
    for (int c = 0; c < CH; c++) held[c].template load<VLOAD>(x, (c * TPR + t) * V, K);
#pragma unroll
    for (int c = 0; c < CH; c++) held[c].peak(peak);
    for (long long k = (CH * TPR + t) * V; k < K; k += TPR * V) {
        QuantVec<T> v;
        v.template load<VLOAD>(x, k, K);
        v.peak(peak);
    }
    peak = __reduce_max_sync(0xffffffffu, QuantType<T>::fold(peak));
    if (TPR > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = peak;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) peak = max(peak, red[w]);
    }
    if (!live) return;
    const RowQuant<T> rq(peak);
    if (t == 0) a.scale[m] = rq.scale;
    int8_t *q = a.Q + m * a.ldq;
    auto put = [&](const QuantVec<T> &v, long long k) {
        if (k >= a.cols) return;
        uint32_t c[V / 4];
        v.codes(rq, c);
        if (a.vstore) {                                  // cols is a multiple of V: the whole vector exists
            if (V == 8) *reinterpret_cast<uint2 *>(q + k) = make_uint2(c[0], c[V / 4 - 1]);
            else *reinterpret_cast<uint32_t *>(q + k) = c[0];
        } else {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (k + i < a.cols) q[k + i] = (int8_t)(c[i / 4] >> (8 * (i & 3)));
        }
    };
#pragma unroll
    for (int c = 0; c < CH; c++) put(held[c], (c * TPR + t) * V);
    for (long long k = (CH * TPR + t) * V; k < a.cols; k += TPR * V) {
        QuantVec<T> v;
        v.template load<VLOAD>(x, k, a.K);
        put(v, k);
    }
}

template <typename T, bool VLOAD, int TPR, int CH>
static int launch_quantize(const QuantArgs &a, cudaStream_t st) {
    const long long rows = 256 / TPR, grid = (a.M + rows - 1) / rows;
    if (grid > 0x7FFFFFFF) return TMQ_ERR_UNSUPPORTED;
    return launch_chained(quantize_rows_kernel<T, VLOAD, TPR, CH>, a, (unsigned)grid, 256, 0, st);
}

template <typename T, bool VLOAD>
static int dispatch_width(const QuantArgs &a, cudaStream_t st) {
    constexpr int V = QuantType<T>::V;
    // short rows: one warp each when there are enough of them to fill the machine
    if (a.K <= 32 * V * 4 && a.M >= 8 * kNumSMs) return launch_quantize<T, VLOAD, 32, 4>(a, st);
    if (a.K <= 256 * V) return launch_quantize<T, VLOAD, 256, 1>(a, st);
    if (a.K <= 256 * V * 2) return launch_quantize<T, VLOAD, 256, 2>(a, st);
    if (a.K <= 256 * V * 4) return launch_quantize<T, VLOAD, 256, 4>(a, st);
    return launch_quantize<T, VLOAD, 256, 8>(a, st);
}

template <typename T>
static int dispatch_quantize(QuantArgs a, cudaStream_t st) {
    constexpr int V = QuantType<T>::V;
    a.vstore = aligned(a.Q, V) && a.ldq % V == 0 && a.cols % V == 0;
    if (aligned(a.X, 16) && (a.ldx * (long long)sizeof(T)) % 16 == 0) return dispatch_width<T, true>(a, st);
    return dispatch_width<T, false>(a, st);
}

}  // namespace tmq

using namespace tmq;

extern "C" int tmq_quantize_rows(const void *X, int x_type, int8_t *Q, float *scale, int64_t M, int64_t K, int64_t ldx,
                                 int64_t ldq, int64_t cols, void *stream) {
    if (M < 0 || K <= 0 || ldx < K || cols < K || ldq < cols || x_type < TMQ_TYPE_F32 || x_type > TMQ_TYPE_F16) return TMQ_ERR_ARG;
    if (M == 0) return TMQ_OK;
    if (!X || !Q || !scale) return TMQ_ERR_ARG;
    if (!aligned(X, x_type == TMQ_TYPE_F32 ? 4 : 2) || !aligned(scale, 4)) return TMQ_ERR_ALIGN;
    const QuantArgs a = {X, Q, scale, M, K, ldx, ldq, cols, 0};
    if (x_type == TMQ_TYPE_F32) return dispatch_quantize<float>(a, (cudaStream_t)stream);
    if (x_type == TMQ_TYPE_BF16) return dispatch_quantize<__nv_bfloat16>(a, (cudaStream_t)stream);
    return dispatch_quantize<__half>(a, (cudaStream_t)stream);
}
