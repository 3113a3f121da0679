// What the kernels of the scaled and grouped products share: their arguments, the table of work units that the group
// boundaries make, element stores.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace tmq {

struct ScaledArgs {
    const float *row_scale;          // [M] or null (1)
    const float *scale, *bias;       // [groups][N] or null (1 / 0)
    void *Y;
    const void *offsets;             // [groups + 1] int32 or int64, null: one group of all rows
    long long M, N, K, ldy;
    int groups, offsets64, y_type, zero_rest;
    int *status;
    // by the launch:
    int unit_rows;                   // rows of a work unit
    int rows_first;                  // order of the work units (plain product only)
    int minors, majors;              // extents of the order: inner, outer (plain product; experts: the row tiles, on the device)
    int d_minor, d_major;            // step of a CTA's walk, gridDim.x units
    int first_mul;                   // x * first_mul >> 16 = x / minors for x < number of SMs
};

// A product as the C entry points describe it.
struct ScaledProblem {
    const void *X, *W;
    long long ldx, ldw;              // row strides of X (elements) and of 8-bit weights (bytes)
    ScaledArgs a;
};


// One to eight rows times a packed ternary matrix in one launch (scaled_gemv.cu); TMQ_ERR_UNSUPPORTED where an SM's share of
// the matrix exceeds its shared memory.
int launch_token_product(const void *X, int x_type, int64_t ldx, const float *row_scale, const uint32_t *Wt, const float *scale,
                         const float *bias, void *Y, int y_type, int64_t M, int64_t N, int64_t K, int64_t ldy, int *status,
                         cudaStream_t stream);

#ifdef __CUDACC__
// The units of a CTA, every gridDim.x-th.  A whole warp walks; per unit it costs two additions and, for the expert, one look at
// 32 table entries (a division and a search by one thread took up to 2800 cycles beside busy decode warps, more than the
// unit's k-blocks); its divisions are the host's.  Channel tiles run fastest, or row tiles (rows_first) where the weights are
// the larger operand: they are then read from memory once and the activations stay in L2.
struct Walk {
    int rt, nt, e;                           // row tile, channel tile, expert
    int d_major, d_minor, minors, majors;
    bool rows_first;
    // tiles[e]: row tiles before group e
    __device__ __forceinline__ Walk(const int *tiles, const ScaledArgs &a) {
        rows_first = a.rows_first != 0;
        minors = a.minors;
        majors = a.offsets ? tiles[a.groups] : a.majors;
        d_major = a.d_major;
        d_minor = a.d_minor;
        const int first = (int)((blockIdx.x * (unsigned)a.first_mul) >> 16);
        const int minor = (int)blockIdx.x - first * minors;
        rt = rows_first ? minor : first;
        nt = rows_first ? first : minor;
        e = 0;
    }
    __device__ __forceinline__ bool more() const { return (rows_first ? nt : rt) < majors; }
    __device__ __forceinline__ void next() {
        int &minor = rows_first ? rt : nt, &major = rows_first ? nt : rt;
        major += d_major;
        minor += d_minor;
        if (minor >= minors) {
            minor -= minors;
            major++;
        }
    }
};

// The unit a walk stands on: rows [row0, row0 + rows) of group e, channels [n0, n0 + tile_c).  begin[e]: first row of group e,
// begin[groups]: end of the last.  Whole converged warp.
struct Unit {
    int e, row0, rows, n0;
};
__device__ __forceinline__ Unit locate(Walk &w, const ScaledArgs &a, const int *begin, const int *tiles, int bn, int tile_c,
                                       int lane) {
    const int groups = a.groups;
    if (!a.offsets) {
        Unit q;
        q.e = 0;
        q.n0 = w.nt * tile_c;
        q.row0 = w.rt * bn;
        const int left = (int)a.M - q.row0;
        q.rows = left < bn ? left : bn;
        return q;
    }
    for (;;) {                               // tiles[] does not decrease: the entries at or below rt are a prefix
        const int i = w.e + 1 + lane;
        const int n = __popc(__ballot_sync(0xffffffffu, i <= groups && tiles[i] <= w.rt));
        w.e += n;
        if (n < 32) break;
    }
    Unit q;
    q.e = w.e;
    q.n0 = w.nt * tile_c;
    q.row0 = begin[w.e] + (w.rt - tiles[w.e]) * bn;
    const int left = begin[w.e + 1] - q.row0;
    q.rows = left < bn ? left : bn;
    return q;
}

// Executed by one warp: boundaries -> table.  Chunks of 32 boundaries, a running maximum and a running sum of tiles.
__device__ __forceinline__ void build_table(const ScaledArgs &a, int *begin, int *tiles, int bn, int lane) {
    int run = 0, sum = 0;                                       // running maximum of the boundaries, tiles so far
    for (int c = 0; c <= a.groups; c += 32) {
        const int i = c + lane;
        long long v = 0;
        if (i <= a.groups)
            v = a.offsets64 ? reinterpret_cast<const long long *>(a.offsets)[i] : reinterpret_cast<const int *>(a.offsets)[i];
        int b = (int)(v < 0 ? 0 : v > a.M ? a.M : v);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, b, o);
            if (lane >= o) b = max(b, x);
        }
        b = max(b, run);
        int prev = __shfl_up_sync(0xffffffffu, b, 1);
        if (lane == 0) prev = run;
        int t = (i == 0 || i > a.groups) ? 0 : (b - prev + bn - 1) / bn;      // tiles of group i - 1
        const int last = __shfl_sync(0xffffffffu, b, 31);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += x;
        }
        if (i <= a.groups) {
            begin[i] = b;
            tiles[i] = sum + t;
        }
        sum += __shfl_sync(0xffffffffu, t, 31);
        run = last;
    }
}

__device__ __forceinline__ void store_one(void *Y, int y_type, long long i, float f) {
    if (y_type == TMQ_TYPE_F32) reinterpret_cast<float *>(Y)[i] = f;
    else if (y_type == TMQ_TYPE_BF16) reinterpret_cast<__nv_bfloat16 *>(Y)[i] = __float2bfloat16_rn(f);
    else reinterpret_cast<__half *>(Y)[i] = __float2half_rn(f);
}


// Rows before the first and behind the last group of a fresh result, dealt over the CTAs and `threads` threads of each.
__device__ __forceinline__ void zero_rest_rows(const ScaledArgs &a, const int *begin, int thread, int threads) {
    const long long lead = begin[0], tail = begin[a.groups], total = lead + (a.M - tail);
    for (long long r = blockIdx.x; r < total; r += gridDim.x) {
        const long long m = r < lead ? r : tail + (r - lead);
        for (long long n = thread; n < a.N; n += threads) store_one(a.Y, a.y_type, m * a.ldy + n, 0.0f);
    }
}
#endif

}  // namespace tmq
