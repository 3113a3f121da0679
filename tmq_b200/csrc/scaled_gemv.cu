// One to eight rows times a packed ternary matrix in 8 bits, quantisation included, in one launch:
//   Y[m][n] = (sum_k q[m][k] T[n][k]) * s[m] * scale[n] + bias[n],   (q, s) = quantised row m of X, or X and row_scale as given
//
// The decode step of a language model is a chain of such products, each a few microseconds long, so what counts is the
// number of launches and what a launch does before its first multiplication.  A CTA owns up to five groups of 16 channels
// and bulk-copies their packed rows (one contiguous run) into shared memory BEFORE it waits for its predecessor in the
// stream; after the wait every CTA reads the few rows of X (they sit in L2), finds their maxima and quantises them into
// shared memory for itself - 148 times the same 8 KB cost less than a second launch and its hand-over - and multiplies:
// byte dot products for one or two rows, warp-level int8 MMA (the rows as its eight columns) for more.  Sums are exact, so
// the order of the warps' slices does not show.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "decode.cuh"
#include "ptx.cuh"
#include "quantize.cuh"
#include "scaled_common.cuh"

namespace tmq {

constexpr int kSgWarps = 16;
constexpr int kSgGroups = 5;                 // channel groups per CTA at most
constexpr int kSgSmemMax = 200 * 1024;

struct ScaledGemvArgs {
    const void *X;
    const float *row_scale;                  // int8 X only
    const uint32_t *Wt;
    const float *scale, *bias;
    void *Y;
    long long M, N, K, KS, ldx, ldy;         // KS: row stride of the packed words
    int x_type, y_type;                      // x_type -1: int8 codes
    int vload;                               // rows of X are 16-byte aligned
    int ngroups, x_offset, x_pitch;          // shared memory: offset and row pitch of the codes, bytes
    int *status;
};

__device__ __forceinline__ void store_result(void *Y, int y_type, long long i, float f) {
    if (y_type == TMQ_TYPE_F32) reinterpret_cast<float *>(Y)[i] = f;
    else if (y_type == TMQ_TYPE_BF16) reinterpret_cast<__nv_bfloat16 *>(Y)[i] = __float2bfloat16_rn(f);
    else reinterpret_cast<__half *>(Y)[i] = __float2half_rn(f);
}

// Rows of X -> codes in shared memory (zero from K to the row pitch) and their scales.  16 / MP warps share a row.
template <typename T, int MP>
__device__ __forceinline__ void quantize_to_smem(const ScaledGemvArgs &a, uint8_t *xq, float *row_scale, uint32_t *red) {
    constexpr int WPR = kSgWarps / MP, V = QuantType<T>::V, STEP = WPR * 32 * V, CH = MP == 8 ? 8 : 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int m = warp / WPR, t = (warp % WPR) * 32 + lane;
    const bool live = m < a.M;
    const T *x = reinterpret_cast<const T *>(a.X) + (live ? m : 0) * a.ldx;
    const int K = live ? (int)a.K : 0;
    QuantVec<T> held[CH];
    uint32_t peak = 0;
    auto load = [&](QuantVec<T> &v, int k) {
        if (a.vload) v.template load<true>(x, k, K);
        else v.template load<false>(x, k, K);
    };
#pragma unroll
    for (int c = 0; c < CH; c++) load(held[c], c * STEP + t * V);
#pragma unroll
    for (int c = 0; c < CH; c++) held[c].peak(peak);
    for (int k = CH * STEP + t * V; k < K; k += STEP) {
        QuantVec<T> v;
        load(v, k);
        v.peak(peak);
    }
    peak = __reduce_max_sync(0xffffffffu, QuantType<T>::fold(peak));
    if (lane == 0) red[warp] = peak;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WPR; w++) peak = max(peak, red[warp / WPR * WPR + w]);
    if (!live) return;
    const RowQuant<T> rq(peak);
    if (t == 0) row_scale[m] = rq.scale;
    uint8_t *q = xq + m * a.x_pitch;
    auto put = [&](const QuantVec<T> &v, int k) {
        if (k >= a.x_pitch) return;
        uint32_t c[V / 4];
        v.codes(rq, c);
        if (V == 8) *reinterpret_cast<uint2 *>(q + k) = make_uint2(c[0], c[V / 4 - 1]);
        else *reinterpret_cast<uint32_t *>(q + k) = c[0];
    };
#pragma unroll
    for (int c = 0; c < CH; c++) put(held[c], c * STEP + t * V);
    for (int k = CH * STEP + t * V; k < a.x_pitch; k += STEP) {
        QuantVec<T> v;
        load(v, k);
        put(v, k);
    }
}

__device__ __forceinline__ void copy_codes(const ScaledGemvArgs &a, uint8_t *xq, float *row_scale) {
    const int per_row = a.x_pitch / 16;
    for (int i = threadIdx.x; i < (int)a.M * per_row; i += kSgWarps * 32) {
        const int m = i / per_row, k = (i - m * per_row) * 16;
        const int8_t *x = reinterpret_cast<const int8_t *>(a.X) + m * a.ldx;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k + 16 <= a.K) {
            v = *reinterpret_cast<const uint4 *>(x + k);
        } else if (k < a.K) {
            __align__(16) uint8_t b[16];
#pragma unroll
            for (int j = 0; j < 16; j++) b[j] = k + j < a.K ? (uint8_t)x[k + j] : 0;
            v = *reinterpret_cast<const uint4 *>(b);
        }
        *reinterpret_cast<uint4 *>(xq + m * a.x_pitch + k) = v;
    }
    if (threadIdx.x < a.M) row_scale[threadIdx.x] = a.row_scale ? a.row_scale[threadIdx.x] : 1.0f;
}

__device__ __forceinline__ uint4 lds_16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

// MP: rows rounded up to a power of two.  Lane (g, t) of a warp owns channels g and g + 8 of every group and 64 k of each
// 256-wide slice; warps take the slices round-robin.  Words a lane reads past the valid part of its row (row padding, the
// next row, the slack behind the last) meet codes that are zero, and any bits decode to finite numbers.
template <int MP>
__global__ void __launch_bounds__(kSgWarps * 32, MP <= 2 ? 2 : 1) scaled_gemv_kernel(const ScaledGemvArgs a) {
    constexpr bool DOT = MP <= 2;
    constexpr int RL = 2 * kSgGroups;                    // channels per lane
    constexpr int MC = DOT ? MP : 8;                     // accumulator columns
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bar;
    __shared__ float row_scale[8];
    __shared__ uint32_t red16[kSgWarps];
    uint8_t *xq = smem + a.x_offset;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int group0 = (int)((blockIdx.x * (unsigned)a.ngroups) / gridDim.x);
    const int G = (int)(((blockIdx.x + 1) * (unsigned)a.ngroups) / gridDim.x) - group0;
    if (threadIdx.x == 0) {
        long long rows = a.N - (long long)group0 * 16;
        if (rows > G * 16) rows = G * 16;
        const uint32_t bytes = (uint32_t)(rows * a.KS * 4);
        ptx::mbar_init(&bar, 1);
        ptx::fence_mbar_init();
        ptx::mbar_arrive_expect_tx(&bar, bytes);
        ptx::bulk_load(smem, a.Wt + (long long)group0 * 16 * a.KS, bytes, &bar);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const bool healthy = *reinterpret_cast<volatile int *>(a.status) == 0;
    if (a.x_type < 0) copy_codes(a, xq, row_scale);
    else if (a.x_type == TMQ_TYPE_F32) quantize_to_smem<float, MP>(a, xq, row_scale, red16);
    else if (a.x_type == TMQ_TYPE_BF16) quantize_to_smem<__nv_bfloat16, MP>(a, xq, row_scale, red16);
    else quantize_to_smem<__half, MP>(a, xq, row_scale, red16);
    __syncthreads();
    // the copy is waited for in any case: nobody may leave while it is on its way into this CTA's memory
    const bool ok = __syncthreads_and(ptx::mbar_wait_own(&bar, 0, a.status) && healthy);
    if (!ok) return;

    int acc[RL][DOT ? MP : 1];                           // DOT: channel i * 8 + g, row m
    int frag[kSgGroups][4];                              // MMA accumulators
#pragma unroll
    for (int i = 0; i < RL; i++)
#pragma unroll
        for (int m = 0; m < (DOT ? MP : 1); m++) acc[i][m] = 0;
#pragma unroll
    for (int i = 0; i < kSgGroups; i++)
#pragma unroll
        for (int m = 0; m < 4; m++) frag[i][m] = 0;

    const int nslices = (int)((a.K + 255) / 256);
    const uint32_t row8 = (uint32_t)a.KS * 32u;
    const uint32_t wbase = ptx::smem_u32(smem) + (uint32_t)g * ((uint32_t)a.KS * 4u) + 16u * t;
    const uint32_t xbase = ptx::smem_u32(xq) + 64u * t;
    for (int slice = warp; slice < nslices; slice += kSgWarps) {
        uint32_t xr[DOT ? MP : 1][16];
#pragma unroll
        for (int m = 0; m < (DOT ? MP : 1); m++) {
            const int row = DOT ? m : g;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (row < a.M) v = lds_16(xbase + (uint32_t)(row * a.x_pitch + slice * 256 + 16 * q));
                xr[m][4 * q] = v.x; xr[m][4 * q + 1] = v.y; xr[m][4 * q + 2] = v.z; xr[m][4 * q + 3] = v.w;
            }
        }
        const uint32_t w0 = wbase + 64u * (uint32_t)slice;
        if (DOT) {
#pragma unroll
            for (int i = 0; i < RL; i++) {
                if (i < 2 * G) {
                    const uint4 p = lds_16(w0 + (uint32_t)i * row8);
                    const uint32_t words[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        uint32_t d[4];
                        decode_word_i8_ptx(words[w], d);
#pragma unroll
                        for (int m = 0; m < (DOT ? MP : 1); m++)
#pragma unroll
                            for (int q = 0; q < 4; q++) acc[i][m] = __dp4a((int)d[q], (int)xr[m][4 * w + q], acc[i][m]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kSgGroups; i++) {
                if (i < G) {
                    const uint4 p = lds_16(w0 + (uint32_t)i * (2u * row8)), r = lds_16(w0 + (uint32_t)i * (2u * row8) + row8);
                    const uint32_t lo[4] = {p.x, p.y, p.z, p.w}, hi[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        uint32_t dl[4], dh[4];
                        decode_word_i8_ptx(lo[w], dl);
                        decode_word_i8_ptx(hi[w], dh);
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            asm volatile(
                                "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                                : "+r"(frag[i][0]), "+r"(frag[i][1]), "+r"(frag[i][2]), "+r"(frag[i][3])
                                : "r"(dl[2 * h]), "r"(dh[2 * h]), "r"(dl[2 * h + 1]), "r"(dh[2 * h + 1]),
                                  "r"(xr[0][4 * w + 2 * h]), "r"(xr[0][4 * w + 2 * h + 1]));
                    }
                }
            }
        }
    }
    if (DOT) {
#pragma unroll
        for (int i = 0; i < RL; i++)
#pragma unroll
            for (int m = 0; m < (DOT ? MP : 1); m++) {
                acc[i][m] += __shfl_xor_sync(0xffffffffu, acc[i][m], 1);
                acc[i][m] += __shfl_xor_sync(0xffffffffu, acc[i][m], 2);
            }
    }
    __syncthreads();                                     // the packed rows are read: their area takes the warps' sums
    int *red = reinterpret_cast<int *>(smem);            // [warp][channel of the CTA][MC]
    if (DOT) {
        if (t == 0)
#pragma unroll
            for (int i = 0; i < RL; i++)
                if (i < 2 * G)
#pragma unroll
                    for (int m = 0; m < (DOT ? MP : 1); m++) red[(warp * (RL * 8) + i * 8 + g) * MC + m] = acc[i][m];
    } else {
#pragma unroll
        for (int i = 0; i < kSgGroups; i++)
            if (i < G) {
                int *r = red + (warp * (RL * 8) + i * 16) * MC;
                r[g * MC + 2 * t] = frag[i][0];
                r[g * MC + 2 * t + 1] = frag[i][1];
                r[(g + 8) * MC + 2 * t] = frag[i][2];
                r[(g + 8) * MC + 2 * t + 1] = frag[i][3];
            }
    }
    __syncthreads();
    const int warps = nslices < kSgWarps ? nslices : kSgWarps;
    for (int o = threadIdx.x; o < G * 16 * (int)a.M; o += kSgWarps * 32) {
        const int m = o / (G * 16), c = o - m * (G * 16);
        const long long n = (long long)group0 * 16 + c;
        if (n < a.N) {
            int s = 0;
            for (int w = 0; w < warps; w++) s += red[(w * (RL * 8) + c) * MC + m];
            const float f = fmaf(__fmul_rn(__int2float_rn(s), row_scale[m]), a.scale ? a.scale[n] : 1.0f, a.bias ? a.bias[n] : 0.0f);
            store_result(a.Y, a.y_type, m * a.ldy + n, f);
        }
    }
}

template <int MP>
static int launch_scaled_gemv(const ScaledGemvArgs &a, unsigned grid, size_t smem, cudaStream_t st) {
    const int rc = ensure_dynamic_smem(scaled_gemv_kernel<MP>, kSgSmemMax, true);
    if (rc != TMQ_OK) return rc;
    return launch_chained(scaled_gemv_kernel<MP>, a, grid, kSgWarps * 32, smem, st);
}

int launch_token_product(const void *X, int x_type, int64_t ldx, const float *row_scale, const uint32_t *Wt, const float *scale,
                         const float *bias, void *Y, int y_type, int64_t M, int64_t N, int64_t K, int64_t ldy, int *status,
                         cudaStream_t stream) {
    if (M < 0 || N <= 0 || K <= 0 || ldx < K || ldy < N || x_type < -1 || x_type > TMQ_TYPE_F16 || y_type < TMQ_TYPE_F32 ||
        y_type > TMQ_TYPE_F16 || (x_type >= 0 && row_scale))
        return TMQ_ERR_ARG;
    if (M == 0) return TMQ_OK;
    if (!X || !Wt || !Y || !status) return TMQ_ERR_ARG;
    const int xe = x_type < 0 ? 1 : x_type == TMQ_TYPE_F32 ? 4 : 2;
    const bool vload = aligned(X, 16) && (M == 1 || (ldx * xe) % 16 == 0);
    if (!aligned(X, xe) || (x_type < 0 && !vload) || !aligned(Wt, 16) || !aligned(status, 4) || !aligned(row_scale, 4) ||
        !aligned(scale, 4) || !aligned(bias, 4) || !aligned(Y, y_type == TMQ_TYPE_F32 ? 4 : 2))
        return TMQ_ERR_ALIGN;
    const long long ngroups = (N + 15) / 16, grid = ngroups < kNumSMs ? ngroups : kNumSMs, G = (ngroups + grid - 1) / grid;
    if (M > 8 || K > 131071 || G > kSgGroups) return TMQ_ERR_UNSUPPORTED;
    const int mc = M <= 2 ? (int)M : 8;
    ScaledGemvArgs a = {X, row_scale, Wt, scale, bias, Y, M, N, K, prepack_row_words(K, 1), ldx, ldy, x_type, y_type, vload};
    a.ngroups = (int)ngroups;
    a.status = status;
    a.x_pitch = (int)((K + 255) / 256 * 256);
    // packed rows (64 bytes of slack: a lane reads up to 48 behind the last row), later the warps' sums; then the codes
    long long rows = G * 16 * a.KS * 4 + 64, red = (long long)kSgWarps * 2 * kSgGroups * 8 * mc * 4;
    if (rows < red) rows = red;
    a.x_offset = (int)((rows + 127) / 128 * 128);
    const long long smem = a.x_offset + M * a.x_pitch;
    if (smem > kSgSmemMax) return TMQ_ERR_UNSUPPORTED;
    if (M == 1) return launch_scaled_gemv<1>(a, (unsigned)grid, (size_t)smem, stream);
    if (M == 2) return launch_scaled_gemv<2>(a, (unsigned)grid, (size_t)smem, stream);
    if (M <= 4) return launch_scaled_gemv<4>(a, (unsigned)grid, (size_t)smem, stream);
    return launch_scaled_gemv<8>(a, (unsigned)grid, (size_t)smem, stream);
}

}  // namespace tmq
