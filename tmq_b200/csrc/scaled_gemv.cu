// One to eight rows times a packed ternary matrix in 8 bits, quantisation included, in one launch:
//   Y[m][n] = (sum_k q[m][k] T[n][k]) * s[m] * scale[n] + bias[n],   (q, s) = quantised row m of X, or X and row_scale as given
//
// The decode step of a language model is a chain of such products, each a few microseconds long, so what counts is the
// number of launches and what a launch does before its first multiplication.  A CTA owns up to five groups of 16 channels
// and asks for their packed rows (one contiguous run) to be brought into L2 BEFORE it waits for its predecessor in the stream -
// only that: L2 is where a predecessor's writes arrive, so weights it has just written are seen all the same - and copies them
// into shared memory after the wait, while every CTA reads the few rows of X, finds their maxima and quantises them into
// shared memory for itself: up to TMQ_A8_FUSED_ELEMS elements, 148 times the same 8 KB cost less than a second launch and its hand-over.
// Then it multiplies with warp-level int8 MMAs, the rows as their eight columns, for one row too: byte dot products took 5.9 us
// instead of 6.2 on 11008 x 4096 but 3.2 instead of 2.8 on 1024 x 2048, which does not pay for a second form.  (Now 6.4 us for the
// first, in a graph of such calls.)  Sums are exact, so the order of the warps' slices does not show.
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

// Rows of X -> codes in shared memory (zero from K to the row pitch) and their scales.  16 / MP warps share a row.
template <typename T, int MP>
__device__ __forceinline__ void quantize_to_smem(const ScaledGemvArgs &a, uint8_t *xq, float *row_scale, uint32_t *red) {
    constexpr int WPR = kSgWarps / MP, V = QuantType<T>::V, STEP = WPR * 32 * V, CH = 4;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int m = warp / WPR, t = (warp % WPR) * 32 + lane;
    const bool live = m < a.M;
    const T *x = reinterpret_cast<const T *>(a.X) + (live ? m : 0) * a.ldx;
    const int K = live ? (int)a.K : 0;
    QuantVec<T> held[CH];
    uint32_t peak = 0;
    // CH vectors at a time, all of them on their way before the first is looked at
    auto load = [&](int base) {
#pragma unroll
        for (int c = 0; c < CH; c++) {
            if (a.vload) held[c].template load<true>(x, base + c * STEP + t * V, K);
            else held[c].template load<false>(x, base + c * STEP + t * V, K);
        }
    };
    for (int base = 0; base == 0 || base < K; base += CH * STEP) {
        load(base);
#pragma unroll
        for (int c = 0; c < CH; c++) held[c].peak(peak);
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
    for (int base = 0; base < a.x_pitch; base += CH * STEP) {
        if (K > CH * STEP) load(base);                   // a row that fits the registers is still in them
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int k = base + c * STEP + t * V;
            if (k < a.x_pitch) {
                uint32_t d[V / 4];
                held[c].codes(rq, d);
                if (V == 8) *reinterpret_cast<uint2 *>(q + k) = make_uint2(d[0], d[V / 4 - 1]);
                else *reinterpret_cast<uint32_t *>(q + k) = d[0];
            }
        }
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

// MP: rows rounded up to a power of two.  Lane (g, t) of a warp owns channels g and g + 8 of every group and 64 k of each
// 256-wide slice; warps take the slices round-robin.  Words a lane reads past the valid part of its row (row padding, the
// next row, the slack behind the last) meet codes that are zero, and any bits decode to finite numbers.
template <int MP>
__global__ void __launch_bounds__(kSgWarps * 32, 1) scaled_gemv_kernel(const ScaledGemvArgs a) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t bar;
    __shared__ float row_scale[8];
    __shared__ uint32_t red16[kSgWarps];
    uint8_t *xq = smem + a.x_offset;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int group0 = (int)((blockIdx.x * (unsigned)a.ngroups) / gridDim.x);
    const int G = (int)(((blockIdx.x + 1) * (unsigned)a.ngroups) / gridDim.x) - group0;
    // this CTA's packed rows, one contiguous run of whole 64-byte blocks
    const uint32_t *rows = a.Wt + (long long)group0 * 16 * a.KS;
    const uint32_t bytes = (uint32_t)((a.N - (long long)group0 * 16 < G * 16 ? a.N - (long long)group0 * 16 : G * 16) * a.KS * 4);
    if (threadIdx.x == 0) {
        ptx::prefetch_l2(rows, bytes);
        ptx::mbar_init(&bar, 1);
        ptx::fence_mbar_init();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        ptx::mbar_arrive_expect_tx(&bar, bytes);
        ptx::bulk_load(smem, rows, bytes, &bar);
    }
    const bool healthy = *reinterpret_cast<volatile int *>(a.status) == 0;
    if (a.x_type < 0) copy_codes(a, xq, row_scale);
    else if (a.x_type == TMQ_TYPE_F32) quantize_to_smem<float, MP>(a, xq, row_scale, red16);
    else if (a.x_type == TMQ_TYPE_BF16) quantize_to_smem<__nv_bfloat16, MP>(a, xq, row_scale, red16);
    else quantize_to_smem<__half, MP>(a, xq, row_scale, red16);
    __syncthreads();
    // the copy is waited for in any case: nobody may leave while it is on its way into this CTA's memory
    const bool ok = __syncthreads_and(ptx::mbar_wait_own(&bar, 0, a.status) && healthy);
    if (!ok) return;

    int acc[kSgGroups][4];
#pragma unroll
    for (int i = 0; i < kSgGroups; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[i][j] = 0;

    const int nslices = (int)((a.K + 255) / 256);
    const uint32_t row8 = (uint32_t)a.KS * 32u;
    const uint32_t wbase = ptx::smem_u32(smem) + (uint32_t)g * ((uint32_t)a.KS * 4u) + 16u * t;
    const uint32_t xbase = ptx::smem_u32(xq) + (uint32_t)(g * a.x_pitch) + 64u * t;
    for (int slice = warp; slice < nslices; slice += kSgWarps) {
        uint32_t x[16];                                  // row g's 64 codes
#pragma unroll
        for (int q = 0; q < 4; q++) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (g < a.M) v = ptx::lds_v4(xbase + (uint32_t)(slice * 256 + 16 * q));
            x[4 * q] = v.x; x[4 * q + 1] = v.y; x[4 * q + 2] = v.z; x[4 * q + 3] = v.w;
        }
        const uint32_t w0 = wbase + 64u * (uint32_t)slice;
#pragma unroll
        for (int i = 0; i < kSgGroups; i++) {
            if (i < G) {
                const uint4 p = ptx::lds_v4(w0 + (uint32_t)i * (2u * row8)), r = ptx::lds_v4(w0 + (uint32_t)i * (2u * row8) + row8);
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
                            : "+r"(acc[i][0]), "+r"(acc[i][1]), "+r"(acc[i][2]), "+r"(acc[i][3])
                            : "r"(dl[2 * h]), "r"(dh[2 * h]), "r"(dl[2 * h + 1]), "r"(dh[2 * h + 1]), "r"(x[4 * w + 2 * h]),
                              "r"(x[4 * w + 2 * h + 1]));
                }
            }
        }
    }
    __syncthreads();                                     // the packed rows are read: their area takes the warps' sums
    int *red = reinterpret_cast<int *>(smem);            // [warp][channel of the CTA][8 rows]
#pragma unroll
    for (int i = 0; i < kSgGroups; i++)
        if (i < G) {
            int *r = red + (warp * (kSgGroups * 16) + i * 16) * 8 + 2 * t;
            r[g * 8] = acc[i][0];
            r[g * 8 + 1] = acc[i][1];
            r[(g + 8) * 8] = acc[i][2];
            r[(g + 8) * 8 + 1] = acc[i][3];
        }
    __syncthreads();
    const int warps = nslices < kSgWarps ? nslices : kSgWarps;
    for (int o = threadIdx.x; o < G * 16 * (int)a.M; o += kSgWarps * 32) {
        const int m = o / (G * 16), c = o - m * (G * 16);
        const long long n = (long long)group0 * 16 + c;
        if (n < a.N) {
            int s = 0;
            for (int w = 0; w < warps; w++) s += red[(w * (kSgGroups * 16) + c) * 8 + m];
            const float f = fmaf(__fmul_rn(__int2float_rn(s), row_scale[m]), a.scale ? a.scale[n] : 1.0f, a.bias ? a.bias[n] : 0.0f);
            store_one(a.Y, a.y_type, m * a.ldy + n, f);
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
    if (M > 8 || K > 131071 || G > kSgGroups || (x_type >= 0 && M * K > TMQ_A8_FUSED_ELEMS)) return TMQ_ERR_UNSUPPORTED;
    ScaledGemvArgs a = {X, row_scale, Wt, scale, bias, Y, M, N, K, prepack_row_words(K, 1), ldx, ldy, x_type, y_type, vload};
    a.ngroups = (int)ngroups;
    a.status = status;
    a.x_pitch = (int)((K + 255) / 256 * 256);
    // packed rows (64 bytes of slack: a lane reads up to 48 behind the last row), later the warps' sums; then the codes
    long long rows = G * 16 * a.KS * 4 + 64, red = (long long)kSgWarps * kSgGroups * 16 * 8 * 4;
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
