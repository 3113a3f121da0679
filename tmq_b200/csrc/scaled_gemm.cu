// Products with one scale per row and one per channel, plain or grouped by expert, on the 5th-generation tensor cores:
//   Y[m][n] = (sum_k X[m][k] * W_e[n][k]) * row_scale[m] * scale_e[n] + bias_e[n]       for offsets[e] <= m < offsets[e+1]
// X int8 against packed ternary or 8-bit weights (exact int32 sums), or bf16 against packed ternary weights (exact
// products, fp32 sums).  The plain product is the case of one group that holds every row.
//
//   * A work unit is (expert, up to BN of its rows, 128 channels).  The weight tile is the 128-row "A" operand, the rows
//     are the N side of the MMA, so a decoded weight tile serves up to BN rows, and the N of a unit's MMAs is its row
//     count rounded up to 32: an expert with three rows costs 32 columns of tensor work and 32 rows of operand traffic
//     whatever BN is.
//   * The group boundaries stay on the device.  Every CTA scans them into a table of tile counts in shared memory
//     (clamped to the rows that exist and made non-decreasing: bad boundaries give empty groups, never a bad address) and
//     walks the units u = CTA, CTA + grid, ... through it.
//   * Roles: warp 0 TMA of the activations (and 8-bit weights), warp 1 MMA issue, warp 2 TMA of the packed weights, then
//     eight decode warps (packed weights only) and four epilogue warps.  Decoded
//     weights go to tensor memory (the MMA reads its A operand there) except for int8 tiles of 256 rows, whose two
//     accumulators fill tensor memory: those are decoded into shared memory.  8-bit weights need no decode, TMA writes
//     them where the MMA reads them.
//   * Every wait is bounded (TMQ_ERR_TIMEOUT in the status word).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "decode.cuh"
#include "ptx.cuh"
#include "tma_host.cuh"

namespace tmq {

enum { W_TERNARY_BF16 = 0, W_TERNARY_I8 = 1, W_DENSE_I8 = 2 };

constexpr int kTileC = 128;          // channels of a unit (MMA M)
constexpr int kOpRow = 128;          // bytes of one operand row per k-block: 64 bf16 or 128 int8
constexpr int kRowStep = 32;         // granularity of a unit's MMA N
constexpr int kMaxGroups = TMQ_GROUPS_MAX;
constexpr int kDecodeWarps = 8;

struct ScaledArgs {
    const float *row_scale;          // [M] or null (1)
    const float *scale, *bias;       // [groups][N] or null (1 / 0)
    void *Y;
    const void *offsets;             // [groups + 1] int32 or int64, null: one group of all rows
    long long M, N, K, ldy;
    int groups, offsets64, y_type, zero_rest;
    int *status;
};

template <int WK, int BN>
struct ScaledCfg {
    static constexpr bool DENSE = WK == W_DENSE_I8, I8 = WK != W_TERNARY_BF16;
    static constexpr bool TA = WK == W_TERNARY_BF16 || (WK == W_TERNARY_I8 && BN <= 128);   // A operand in tensor memory
    static constexpr int BK = I8 ? 128 : 64;
    static constexpr int RAW_ROW = DENSE ? 0 : I8 ? 32 : 16;                  // packed bytes per channel and k-block
    // Packed words come RAWK k-blocks per box: a box costs the TMA unit about four cycles a row whatever its width (one
    // k-block per box measured 280 ns per k-block at any row count).  Rows of 128 / 64 bytes with the swizzle of that
    // width, so the decode warps' 16-byte reads meet no bank conflicts.
    static constexpr int RAWK = DENSE ? 1 : (TA ? 4 : 2);
    static constexpr int RAW_PITCH = RAWK * RAW_ROW;
    static constexpr int RAW_STAGES = DENSE ? 0 : !TA ? 2 : BN > 128 ? 2 : 4;
    static constexpr int STAGES = DENSE ? (BN > 128 ? 4 : BN > 64 ? 6 : 8) : BN > 128 ? (TA ? 6 : 4) : 8;
    static constexpr int A_BYTES = TA ? 0 : kTileC * kOpRow;
    static constexpr int B_BYTES = BN * kOpRow;
    static constexpr int RAW_BYTES = kTileC * RAW_PITCH;
    // activations arrive as one box of BN rows, or, for a unit of at most half of that, as one or two small boxes
    static constexpr int SMALL = BN > 128 ? 64 : 32;
    static constexpr int ACC_BUFS = (TA && BN > 128) ? 1 : 2;
    static constexpr int A_COLS = kOpRow / 4;
    static constexpr int A_BASE = ACC_BUFS * BN;
    static constexpr int TMEM_NEED = A_BASE + (TA ? STAGES * A_COLS : 0);
    static constexpr int TMEM_COLS = TMEM_NEED <= 128 ? 128 : TMEM_NEED <= 256 ? 256 : 512;
    static_assert(TMEM_NEED <= 512, "tensor memory exceeded");
    static constexpr int FIRST_EPI = DENSE ? 4 : 4 + kDecodeWarps;
    static constexpr int THREADS = (FIRST_EPI + 4) * 32;
    // shared memory
    static constexpr int A_OFF = 0;
    static constexpr int B_OFF = A_OFF + STAGES * A_BYTES;
    static constexpr int RAW_OFF = B_OFF + STAGES * B_BYTES;
    static constexpr int STAGE_OFF = RAW_OFF + RAW_STAGES * RAW_BYTES;            // 4 x 2 KB transposition areas
    static constexpr int RS_OFF = STAGE_OFF + 4 * 2048;                      // 4 x BN row scales
    static constexpr int BAR_OFF = RS_OFF + 4 * BN * 4;
    static constexpr int TAB_OFF = BAR_OFF + 512;                             // begin[groups + 1], tiles[groups + 1]
    static constexpr int bytes(int groups) { return TAB_OFF + 2 * 4 * (groups + 1) + 1024; }
    static_assert(TAB_OFF + 2 * 4 * (kMaxGroups + 1) + 1024 <= 227 * 1024, "shared memory exceeded");
};

// Unit u of the launch: rows [row0, row0 + rows) of group e, channels [n0, n0 + 128).
struct Unit {
    int e, row0, rows, n0;
};
// begin[e]: first row of group e, begin[groups]: end of the last; tiles[e]: row tiles before group e.  `e` only moves forward.
__device__ __forceinline__ Unit locate(int u, int &e, const int *begin, const int *tiles, int tiles_n, int bn) {
    const int rt = u / tiles_n;
    while (tiles[e + 1] <= rt) e++;
    Unit q;
    q.e = e;
    q.n0 = (u - rt * tiles_n) * kTileC;
    q.row0 = begin[e] + (rt - tiles[e]) * bn;
    const int left = begin[e + 1] - q.row0;
    q.rows = left < bn ? left : bn;
    return q;
}

// Executed by one warp: boundaries -> table.  Chunks of 32 boundaries, a running maximum and a running sum of tiles.
__device__ __forceinline__ void build_table(const ScaledArgs &a, int *begin, int *tiles, int bn, int lane) {
    if (!a.offsets) {
        if (lane == 0) {
            begin[0] = 0; begin[1] = (int)a.M;
            tiles[0] = 0; tiles[1] = (int)((a.M + bn - 1) / bn);
        }
        return;
    }
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

// 8 consecutive channels of one row, aligned for vector stores
__device__ __forceinline__ void store_eight(void *Y, int y_type, long long i, const float (&f)[8]) {
    if (y_type == TMQ_TYPE_F32) {
        float4 *p = reinterpret_cast<float4 *>(reinterpret_cast<float *>(Y) + i);
        p[0] = make_float4(f[0], f[1], f[2], f[3]);
        p[1] = make_float4(f[4], f[5], f[6], f[7]);
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (y_type == TMQ_TYPE_BF16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(Y) + i) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <int WK, int BN>
__global__ void __launch_bounds__(ScaledCfg<WK, BN>::THREADS, 1)
scaled_gemm_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_small,
                   const __grid_constant__ CUtensorMap tmap_w, const ScaledArgs a) {
    using C = ScaledCfg<WK, BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::BAR_OFF);         // TMA bytes landed
    uint64_t *ready = full + C::STAGES;                                       // weights decoded
    uint64_t *empty = ready + C::STAGES;
    uint64_t *raw_full = empty + C::STAGES;                                   // packed words landed
    uint64_t *raw_empty = raw_full + C::RAW_STAGES;
    uint64_t *acc_full = raw_empty + C::RAW_STAGES;                           // [2]
    uint64_t *acc_empty = acc_full + 2;                                       // [2]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
    int *begin = reinterpret_cast<int *>(smem + C::TAB_OFF);
    int *tiles = begin + a.groups + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nkb = (int)((a.K + C::BK - 1) / C::BK);
    const int tiles_n = (int)((a.N + kTileC - 1) / kTileC);

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; s++) {
            ptx::mbar_init(full + s, 1);
            ptx::mbar_init(ready + s, 4);
            ptx::mbar_init(empty + s, 1);
        }
        for (int s = 0; s < C::RAW_STAGES; s++) {
            ptx::mbar_init(raw_full + s, 1);
            ptx::mbar_init(raw_empty + s, kDecodeWarps);
        }
        for (int b = 0; b < 2; b++) {
            ptx::mbar_init(acc_full + b, 1);
            ptx::mbar_init(acc_empty + b, 4);
        }
        ptx::fence_mbar_init();
        ptx::prefetch_tensormap(&tmap_x);
        ptx::prefetch_tensormap(&tmap_small);
        ptx::prefetch_tensormap(&tmap_w);
    }
    if (warp == 1) {
        ptx::tmem_alloc(tmem_slot, C::TMEM_COLS);
        ptx::tmem_relinquish();
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");       // everything above is this CTA's own; below is the stream's
    if (warp == C::FIRST_EPI) build_table(a, begin, tiles, BN, lane);
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t *>(tmem_slot);
    const bool healthy = (*reinterpret_cast<volatile int *>(a.status) == 0);
    const int nunits = tiles[a.groups] * tiles_n;

    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer
        if (lane == 0 && healthy) {
            int it = 0, e = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < nunits && ok; u += gridDim.x) {
                const Unit q = locate(u, e, begin, tiles, tiles_n, BN);
                const bool whole = q.rows > BN / 2;
                const int rows = whole ? BN : q.rows > C::SMALL ? 2 * C::SMALL : C::SMALL;
                const int wrow = (int)(q.e * a.N) + q.n0;
                const uint32_t bytes = (uint32_t)(rows * kOpRow + (C::DENSE ? C::A_BYTES : 0));
                for (int kb = 0; kb < nkb; kb++, it++) {
                    const int s = it % C::STAGES;
                    const uint32_t ph = (uint32_t)(it / C::STAGES) & 1u;
                    ok = ptx::mbar_wait(empty + s, ph ^ 1u, a.status);
                    if (!ok) break;
                    ptx::mbar_arrive_expect_tx(full + s, bytes);
                    if (C::DENSE) ptx::tma_load_2d(smem + C::A_OFF + s * C::A_BYTES, &tmap_w, full + s, kb * C::BK, wrow);
                    uint8_t *dst = smem + C::B_OFF + s * C::B_BYTES;
                    ptx::tma_load_2d(dst, whole ? &tmap_x : &tmap_small, full + s, kb * C::BK, q.row0);
                    if (!whole && rows > C::SMALL)
                        ptx::tma_load_2d(dst + C::SMALL * kOpRow, &tmap_small, full + s, kb * C::BK, q.row0 + C::SMALL);
                }
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer (whole warp walks, one lane issues)
        if (healthy) {
            int it = 0, ti = 0, e = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < nunits && ok; u += gridDim.x, ti++) {
                const Unit q = locate(u, e, begin, tiles, tiles_n, BN);
                const uint32_t n_mma = (uint32_t)((q.rows + kRowStep - 1) / kRowStep * kRowStep);
                const uint32_t idesc = ((C::I8 ? 2u : 1u) << 4) | (1u << 7) | (1u << 10) | ((n_mma >> 3) << 17) | ((128u >> 4) << 24);
                const int buf = C::ACC_BUFS == 2 ? (ti & 1) : 0;
                const uint32_t use = (uint32_t)(C::ACC_BUFS == 2 ? (ti >> 1) : ti);
                ok = ptx::mbar_wait_warp(acc_empty + buf, (use & 1u) ^ 1u, a.status);
                if (!ok) break;
                ptx::tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + (uint32_t)(buf * BN);
                for (int kb = 0; kb < nkb; kb++, it++) {
                    const int s = it % C::STAGES;
                    const uint32_t ph = (uint32_t)(it / C::STAGES) & 1u;
                    if (!C::DENSE) ok = ptx::mbar_wait_warp(ready + s, ph, a.status);
                    // the activations were written by TMA: their barrier is waited on by this warp itself
                    ok = ok && ptx::mbar_wait_warp(full + s, ph, a.status);
                    if (!ok) break;
                    ptx::tc_fence_after_sync();
                    const uint64_t a_desc = ptx::umma_desc_sw128(ptx::smem_u32(smem + C::A_OFF + s * C::A_BYTES));
                    const uint64_t b_desc = ptx::umma_desc_sw128(ptx::smem_u32(smem + C::B_OFF + s * C::B_BYTES));
                    const uint32_t a_tmem = tmem_base + C::A_BASE + (uint32_t)(s * C::A_COLS);
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int k4 = 0; k4 < kOpRow / 32; k4++) {
                            const uint32_t accum = (kb > 0 || k4 > 0) ? 1u : 0u;
                            if (C::TA) {
                                if (C::I8) ptx::umma_i8_ts(d_tmem, a_tmem + 8 * k4, b_desc + 2 * k4, idesc, accum);
                                else ptx::umma_f16_ts(d_tmem, a_tmem + 8 * k4, b_desc + 2 * k4, idesc, accum);
                            } else {
                                ptx::umma_i8(d_tmem, a_desc + 2 * k4, b_desc + 2 * k4, idesc, accum);
                            }
                        }
                        ptx::umma_commit(empty + s);
                    }
                    __syncwarp();
                }
                if (ok && ptx::elect_one()) ptx::umma_commit(acc_full + buf);
                __syncwarp();
            }
        }
    } else if (warp == 2) {
        // ---------------------------------------------------------------- TMA producer of the packed words
        if (!C::DENSE && lane == 0 && healthy) {
            int rit = 0, e = 0;
            bool ok = true;
            for (int u = blockIdx.x; u < nunits && ok; u += gridDim.x) {
                const Unit q = locate(u, e, begin, tiles, tiles_n, BN);
                const int wrow = (int)(q.e * a.N) + q.n0;
                for (int kb = 0; kb < nkb; kb += C::RAWK, rit++) {
                    const int s = rit % (C::RAW_STAGES + C::DENSE);
                    const uint32_t ph = (uint32_t)(rit / (C::RAW_STAGES + C::DENSE)) & 1u;
                    ok = ptx::mbar_wait(raw_empty + s, ph ^ 1u, a.status);
                    if (!ok) break;
                    ptx::mbar_arrive_expect_tx(raw_full + s, (uint32_t)C::RAW_BYTES);
                    ptx::tma_load_2d(smem + C::RAW_OFF + s * C::RAW_BYTES, &tmap_w, raw_full + s, kb * (C::RAW_ROW / 4), wrow);
                }
            }
        }
    } else if (!C::DENSE && warp >= 4 && warp < C::FIRST_EPI) {
        // ---------------------------------------------------------------- decode: two sets of four warps, alternate k-blocks
        const int quarter = warp & 3, set = (warp - 4) >> 2;
        const int row = quarter * 32 + lane;
        bool ok = healthy;
        int it = 0, rit = 0;
        for (int u = blockIdx.x; u < nunits && ok; u += gridDim.x) {
            for (int kb0 = 0; kb0 < nkb && ok; kb0 += C::RAWK, rit++) {
                const int rs = rit % (C::RAW_STAGES + C::DENSE);
                ok = ptx::mbar_wait_warp(raw_full + rs, (uint32_t)(rit / (C::RAW_STAGES + C::DENSE)) & 1u, a.status);
                if (!ok) break;
                const uint8_t *raw = smem + C::RAW_OFF + rs * C::RAW_BYTES + row * C::RAW_PITCH;
                const int left = nkb - kb0 < C::RAWK ? nkb - kb0 : C::RAWK;
                for (int j = (it & 1) ^ set; j < left; j += 2) {
                    const int s = (it + j) % C::STAGES;
                    const uint32_t ph = (uint32_t)((it + j) / C::STAGES) & 1u;
                    uint4 p[C::I8 ? 2 : 1];
#pragma unroll
                    for (int h = 0; h < (C::I8 ? 2 : 1); h++) {
                        const int c = (C::I8 ? 2 * j : j) + h;
                        p[h] = *reinterpret_cast<const uint4 *>(raw + ((c ^ (C::RAW_PITCH == 128 ? row & 7 : (row >> 1) & 3)) << 4));
                    }
                    uint32_t cols[32];                   // the row's 128 operand bytes, K ascending
                    if (C::I8) {
                        const uint32_t words[8] = {p[0].x, p[0].y, p[0].z, p[0].w, p[C::I8].x, p[C::I8].y, p[C::I8].z, p[C::I8].w};
#pragma unroll
                        for (int wi = 0; wi < 8; wi++) {
                            uint32_t r[4];
                            decode_word_i8(words[wi], r);
#pragma unroll
                            for (int x = 0; x < 4; x++) cols[4 * wi + x] = r[x];
                        }
                    } else {
                        const uint32_t words[4] = {p[0].x, p[0].y, p[0].z, p[0].w};
#pragma unroll
                        for (int wi = 0; wi < 4; wi++) {
                            uint32_t r[8];
                            decode_word_bf16(words[wi], r);
#pragma unroll
                            for (int x = 0; x < 8; x++) cols[8 * wi + x] = r[x];
                        }
                    }
                    // the MMAs that read this operand slot last are done
                    ok = ptx::mbar_wait_warp(empty + s, ph ^ 1u, a.status);
                    if (!ok) break;
                    if (C::TA) {
                        ptx::tc_fence_after_sync();
                        ptx::tmem_st_x32(tmem_base + ((uint32_t)(quarter * 32) << 16) + C::A_BASE + (uint32_t)(s * C::A_COLS), cols);
                        ptx::tmem_st_wait();
                        ptx::tc_fence_before_sync();
                    } else {
                        uint8_t *arow = smem + C::A_OFF + s * C::A_BYTES + row * kOpRow;
#pragma unroll
                        for (int c = 0; c < 8; c++)
                            *reinterpret_cast<uint4 *>(arow + ((c ^ (row & 7)) << 4)) =
                                make_uint4(cols[4 * c], cols[4 * c + 1], cols[4 * c + 2], cols[4 * c + 3]);
                        ptx::fence_proxy_async_smem();
                    }
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ready + s);
                }
                it += left;
                __syncwarp();
                if (ok && lane == 0) ptx::mbar_arrive(raw_empty + rs);
            }
        }
    } else if (warp >= C::FIRST_EPI) {
        // ---------------------------------------------------------------- epilogue
        const int quarter = warp & 3;
        float *stage = reinterpret_cast<float *>(smem + C::STAGE_OFF) + (warp - C::FIRST_EPI) * 512;
        float *rs = reinterpret_cast<float *>(smem + C::RS_OFF) + (warp - C::FIRST_EPI) * BN;
        const bool vec_rows = ((a.ldy & 7) == 0) && ((reinterpret_cast<uintptr_t>(a.Y) & 15) == 0);
        bool ok = healthy;
        int ti = 0, e = 0;
        for (int u = blockIdx.x; u < nunits && ok; u += gridDim.x, ti++) {
            const Unit q = locate(u, e, begin, tiles, tiles_n, BN);
            const int n = q.n0 + quarter * 32 + lane;
            float sc = 1.0f, bi = 0.0f;
            if (n < a.N) {
                if (a.scale) sc = a.scale[(long long)q.e * a.N + n];
                if (a.bias) bi = a.bias[(long long)q.e * a.N + n];
            }
            if (!C::I8) sc *= 0.5f;                      // bf16 weights are carried as +-2
            __syncwarp();
            for (int r = lane; r < BN; r += 32) rs[r] = (a.row_scale && r < q.rows) ? a.row_scale[q.row0 + r] : 1.0f;
            __syncwarp();
            const int buf = C::ACC_BUFS == 2 ? (ti & 1) : 0;
            ok = ptx::mbar_wait_warp(acc_full + buf, (uint32_t)(C::ACC_BUFS == 2 ? (ti >> 1) : ti) & 1u, a.status);
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * BN);
#pragma unroll 1
            for (int c = 0; c < q.rows; c += 16) {
                uint32_t v[16];
                ptx::tmem_ld_x16(lane_addr + (uint32_t)c, v);
                ptx::tmem_ld_wait();
                if (c + 16 >= q.rows) {                  // last chunk read: the accumulator goes back to the MMA warp
                    ptx::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(acc_empty + buf);
                }
                float f[16];
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const float acc = C::I8 ? __int2float_rn((int)v[j]) : __uint_as_float(v[j]);
                    f[j] = fmaf(__fmul_rn(acc, rs[c + j]), sc, bi);
                }
                if (!vec_rows) {                         // rows that allow no vectors: a warp writes 32 neighbouring channels
                    if (n < a.N) {
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            if (c + j < q.rows) store_one(a.Y, a.y_type, (long long)(q.row0 + c + j) * a.ldy + n, f[j]);
                    }
                    continue;
                }
#pragma unroll
                for (int j = 0; j < 16; j++) stage[j * 32 + lane] = f[j];
                __syncwarp();
                const int cg = (lane & 3) * 8, nb = q.n0 + quarter * 32 + cg;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int p = h * 8 + (lane >> 2);
                    if (c + p < q.rows && nb < a.N) {
                        const float4 lo = *reinterpret_cast<const float4 *>(stage + p * 32 + cg);
                        const float4 hi = *reinterpret_cast<const float4 *>(stage + p * 32 + cg + 4);
                        const float o[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                        const long long i = (long long)(q.row0 + c + p) * a.ldy + nb;
                        if (nb + 8 <= a.N) store_eight(a.Y, a.y_type, i, o);
                        else
                            for (int x = 0; x < 8 && nb + x < a.N; x++) store_one(a.Y, a.y_type, i + x, o[x]);
                    }
                }
                __syncwarp();
            }
        }
        if (a.zero_rest && healthy) {
            // rows before the first and behind the last group of a fresh result
            const long long lead = begin[0], tail = begin[a.groups], total = lead + (a.M - tail);
            for (long long r = blockIdx.x; r < total; r += gridDim.x) {
                const long long m = r < lead ? r : tail + (r - lead);
                for (long long n = threadIdx.x - C::FIRST_EPI * 32; n < a.N; n += 128) store_one(a.Y, a.y_type, m * a.ldy + n, 0.0f);
            }
        }
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

// ---- host side --------------------------------------------------------------------------------------------------------

struct ScaledProblem {
    const void *X, *W;
    long long ldx, ldw;              // row strides of X (elements) and of 8-bit weights (bytes)
    ScaledArgs a;
};

template <int WK, int BN>
static int launch_scaled(const ScaledProblem &p, cudaStream_t st) {
    using C = ScaledCfg<WK, BN>;
    const ScaledArgs &a = p.a;
    CUtensorMap mx, ms, mw;
    const CUtensorMapDataType xt = C::I8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const uint64_t xpitch = (uint64_t)p.ldx * (C::I8 ? 1 : 2);
    const bool okx = make_map_2d(&mx, xt, p.X, (uint64_t)a.K, (uint64_t)a.M, xpitch, C::BK, BN, CU_TENSOR_MAP_SWIZZLE_128B) &&
                     make_map_2d(&ms, xt, p.X, (uint64_t)a.K, (uint64_t)a.M, xpitch, C::BK, C::SMALL, CU_TENSOR_MAP_SWIZZLE_128B);
    const uint64_t wrows = (uint64_t)a.groups * (uint64_t)a.N;
    const bool okw = C::DENSE
        ? make_map_2d(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, p.W, (uint64_t)a.K, wrows, (uint64_t)p.ldw, C::BK, kTileC,
                      CU_TENSOR_MAP_SWIZZLE_128B)
        : make_map_2d(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT32, p.W, (uint64_t)prepack_valid_words(a.K), wrows,
                      (uint64_t)prepack_row_words(a.K, C::I8 ? 1 : 0) * 4, C::DENSE ? 4 : C::RAW_PITCH / 4, kTileC,
                      C::RAW_PITCH == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
    if (!okx || !okw) return TMQ_ERR_LAUNCH;
    int rc = ensure_dynamic_smem(scaled_gemm_kernel<WK, BN>, C::bytes(kMaxGroups));
    if (rc != TMQ_OK) return rc;
    // at most (rows / BN + groups) row tiles; CTAs beyond the real count find nothing to do
    const long long units = ((a.M + BN - 1) / BN + a.groups - 1) * ((a.N + kTileC - 1) / kTileC);
    if (units > 0x7FFFFFFF) return TMQ_ERR_UNSUPPORTED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units < kNumSMs ? units : kNumSMs));
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = (size_t)C::bytes(a.groups);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, scaled_gemm_kernel<WK, BN>, mx, ms, mw, a));
}

template <int WK>
static int dispatch_scaled(const ScaledProblem &p, cudaStream_t st) {
    const long long per_group = (p.a.M + p.a.groups - 1) / p.a.groups;
    if (per_group > 128) return launch_scaled<WK, 256>(p, st);
    if (per_group > 64) return launch_scaled<WK, 128>(p, st);
    return launch_scaled<WK, 64>(p, st);
}

static int check_scaled(const ScaledProblem &p, int x_bytes, bool dense) {
    const ScaledArgs &a = p.a;
    if (a.M < 0 || a.N <= 0 || a.K <= 0 || a.groups < 1 || p.ldx < a.K || a.ldy < a.N) return TMQ_ERR_ARG;
    if (a.y_type < TMQ_TYPE_F32 || a.y_type > TMQ_TYPE_F16) return TMQ_ERR_ARG;
    if (a.M == 0) return TMQ_OK;
    if (!p.X || !p.W || !a.Y || !a.status || (dense && p.ldw < a.K)) return TMQ_ERR_ARG;
    if (a.M > 0x7FFFFFFF || a.K > 0x7FFFFFFF || a.groups > kMaxGroups || a.N * a.groups > 0x7FFFFFFF) return TMQ_ERR_UNSUPPORTED;
    // int32 sums of 8-bit products stay exact up to 2^31 / 2^14 of them
    if (x_bytes == 1 && a.K > 131071) return TMQ_ERR_UNSUPPORTED;
    if ((p.ldx * x_bytes) % 16 != 0 || (dense && p.ldw % 16 != 0)) return TMQ_ERR_UNSUPPORTED;
    if (!aligned(p.X, 16) || !aligned(p.W, 16) || !aligned(a.status, 4) || !aligned(a.offsets, a.offsets64 ? 8 : 4) ||
        !aligned(a.Y, a.y_type == TMQ_TYPE_F32 ? 4 : 2) || !aligned(a.row_scale, 4) || !aligned(a.scale, 4) || !aligned(a.bias, 4))
        return TMQ_ERR_ALIGN;
    return TMQ_OK;
}

}  // namespace tmq

using namespace tmq;

extern "C" int tmq_ternary_gemm_a8(const int8_t *X, int64_t ldx, const float *row_scale, const uint32_t *Wt, const float *scale,
                                   const float *bias, void *Y, int y_type, int64_t M, int64_t N, int64_t K, int64_t ldy,
                                   int *status, void *stream) {
    const ScaledProblem p = {X, Wt, ldx, 0, {row_scale, scale, bias, Y, nullptr, M, N, K, ldy, 1, 0, y_type, 0, status}};
    const int rc = check_scaled(p, 1, false);
    if (rc != TMQ_OK || M == 0) return rc;
    return dispatch_scaled<W_TERNARY_I8>(p, (cudaStream_t)stream);
}

extern "C" int tmq_gemm_i8(const int8_t *X, int64_t ldx, const float *row_scale, const int8_t *W, int64_t ldw,
                           const float *scale, const float *bias, void *Y, int y_type, int64_t M, int64_t N, int64_t K,
                           int64_t ldy, int *status, void *stream) {
    const ScaledProblem p = {X, W, ldx, ldw, {row_scale, scale, bias, Y, nullptr, M, N, K, ldy, 1, 0, y_type, 0, status}};
    const int rc = check_scaled(p, 1, true);
    if (rc != TMQ_OK || M == 0) return rc;
    return dispatch_scaled<W_DENSE_I8>(p, (cudaStream_t)stream);
}

extern "C" int tmq_ternary_gemm_grouped_bf16(const void *X, int64_t ldx, const uint32_t *Wt, const float *scale,
                                             const float *bias, const void *offsets, int offsets_bytes, int groups, void *Y,
                                             int y_type, int64_t M, int64_t N, int64_t K, int64_t ldy, int zero_rest,
                                             int *status, void *stream) {
    const ScaledProblem p = {X, Wt, ldx, 0,
                             {nullptr, scale, bias, Y, offsets, M, N, K, ldy, groups, offsets_bytes == 8, y_type, zero_rest != 0, status}};
    if (offsets_bytes != 4 && offsets_bytes != 8) return TMQ_ERR_ARG;
    const int rc = check_scaled(p, 2, false);
    if (rc != TMQ_OK || M == 0) return rc;
    if (!offsets) return TMQ_ERR_ARG;
    return dispatch_scaled<W_TERNARY_BF16>(p, (cudaStream_t)stream);
}

extern "C" int tmq_ternary_gemm_grouped_a8(const int8_t *X, int64_t ldx, const float *row_scale, const uint32_t *Wt,
                                           const float *scale, const float *bias, const void *offsets, int offsets_bytes,
                                           int groups, void *Y, int y_type, int64_t M, int64_t N, int64_t K, int64_t ldy,
                                           int zero_rest, int *status, void *stream) {
    const ScaledProblem p = {X, Wt, ldx, 0,
                             {row_scale, scale, bias, Y, offsets, M, N, K, ldy, groups, offsets_bytes == 8, y_type, zero_rest != 0, status}};
    if (offsets_bytes != 4 && offsets_bytes != 8) return TMQ_ERR_ARG;
    const int rc = check_scaled(p, 1, false);
    if (rc != TMQ_OK || M == 0) return rc;
    if (!offsets) return TMQ_ERR_ARG;
    return dispatch_scaled<W_TERNARY_I8>(p, (cudaStream_t)stream);
}

extern "C" int tmq_gemm_grouped_i8(const int8_t *X, int64_t ldx, const float *row_scale, const int8_t *W, int64_t ldw,
                                   const float *scale, const float *bias, const void *offsets, int offsets_bytes, int groups,
                                   void *Y, int y_type, int64_t M, int64_t N, int64_t K, int64_t ldy, int zero_rest,
                                   int *status, void *stream) {
    const ScaledProblem p = {X, W, ldx, ldw,
                             {row_scale, scale, bias, Y, offsets, M, N, K, ldy, groups, offsets_bytes == 8, y_type, zero_rest != 0, status}};
    if (offsets_bytes != 4 && offsets_bytes != 8) return TMQ_ERR_ARG;
    const int rc = check_scaled(p, 1, true);
    if (rc != TMQ_OK || M == 0) return rc;
    if (!offsets) return TMQ_ERR_ARG;
    return dispatch_scaled<W_DENSE_I8>(p, (cudaStream_t)stream);
}
