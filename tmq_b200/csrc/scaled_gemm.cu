// Products with one scale per row and one per channel, plain or grouped by expert, on the 5th-generation tensor cores:
//   Y[m][n] = (sum_k X[m][k] * W_e[n][k]) * row_scale[m] * scale_e[n] + bias_e[n]       for offsets[e] <= m < offsets[e+1]
// X int8 against packed ternary or 8-bit weights (exact int32 sums), or bf16 against packed ternary weights (exact
// products, fp32 sums).  The plain product is the case of one group that holds every row.
//
//   * A work unit is (expert, up to BN of its rows, 128 channels).  The weight tile is the 128-row "A" operand, the rows
//     are the N side of the MMA, so a decoded weight tile serves up to BN rows, and the N of a unit's MMAs is its row
//     count rounded up to 16.
//   * The group boundaries stay on the device.  Every CTA scans them into a table of tile counts in shared memory
//     (clamped to the rows that exist and made non-decreasing: bad boundaries give empty groups, never a bad address) and
//     takes every gridDim.x-th unit of it.
//   * Roles: warp 0 TMA of the activations (and 8-bit weights), warp 1 MMA issue, warp 2 TMA of the packed weights, then
//     decode warps (packed weights only) and epilogue warps.  Decoded weights go to tensor memory, where the MMA reads its A
//     operand without a byte through shared memory; 8-bit weights need no decode, TMA writes them where the MMA reads them.
//   * Every wait is bounded (TMQ_ERR_TIMEOUT in the status word).
//
// What bounds it: tall tiles the tensor pipe (bf16 256 rows: the 512 cycles per k-block that its MMAs take; int8 8192 x 28672 x
// 8192 in 1.28 ms = 3.0 Pop/s, 1.24 - 1.28 by box) and, with 8-bit weights, shared memory (96 KB per k-block); 8-bit weights and few rows memory
// (28672 x 8192, up to 32 rows: 41 us = 5.7 TB/s); ternary weights and few rows the decode warps' integer instructions: 140 ns
// per k-block, of which 104 remain without the decoding and 92 without its stores, where memory's 93 are; the int8 kernels of
// 32, 64 and 128 rows spill 32 / 32 / 44 bytes at the 80 registers that 24 warps leave each thread.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "decode.cuh"
#include "ptx.cuh"
#include "scaled_common.cuh"
#include "scaled_config.h"
#include "tma_host.cuh"

namespace tmq {

// Tensor maps of a launch.  A TMA instruction costs about 200 cycles of its unit whatever it brings (bf16 tiles of 32 rows
// with one box per k-block: 154 ns per k-block), so a box spans all k-blocks of a stage.  A row that ends inside a k-block has
// that last stage brought k-block by k-block through maps of the whole row, whose ends are filled with zeros (all stages that
// way: 32 x 4096 x 4080 ternary 9.7 us against 9.0).
// Activation boxes come in three heights (multiples of 8: the swizzle's period), a unit takes the lowest that holds its
// rows.  Rows of a box that lie outside the matrix cost about ten cycles each (one row of 11008 x 4096 8-bit weights: 12.8 us
// with a box of 32), so a plain product's last tile gets a box of its own height.
struct ScaledMaps {
    CUtensorMap x[3], w;             // boxes of a stage's k-blocks
    CUtensorMap x_end[3], w_end;     // ... of one
    int height[3];
};

// COUNT accumulator columns (rows of the result) of this lane's channel, scaled and rounded, to Y.  rs: their row scales (16-byte
// aligned).  TYPE fixed at compile time, addresses stepped.  FULL: all rows and channels exist.  PAIRS: two rows' 16-bit results
// make a word, and neighbouring lanes exchange halves (even lanes keep row j, odd lanes row j + 1), so a warp writes 4 bytes a
// lane, two 64-byte runs; otherwise one row's 32 channels at a time.  One warp per scheduler does this and is bound by its own
// instructions, 19 cycles a row; each step is made for all rows before the next, so that their latencies overlap (four rows at
// a time: 33 cycles a row; conversions by an addition of 1.5 * 2^23, or no stores at all, changed nothing).
template <bool I8, int TYPE, bool PAIRS, bool FULL, int COUNT>
__device__ __forceinline__ void store_rows(const uint32_t (&v)[COUNT], const float *rs, float sc, float bi, uint8_t *Y, long long row,
                                           long long ldy, int n, long long N, int left, int lane) {
    constexpr int ES = TYPE == TMQ_TYPE_F32 ? 4 : 2;
    const int odd = PAIRS ? lane & 1 : 0;
    const uint32_t pick = odd ? 0x3276u : 0x5410u;
    const int nb = n - odd;
    uint8_t *p = Y + ((row + odd) * ldy + nb) * ES;
    const long long step = ldy * ES;
    const int rows = nb < N ? left - odd : 0;
    const bool both = nb + 1 < N;
    float f[COUNT];
#pragma unroll
    for (int j = 0; j < COUNT; j += 4) {
        float4 r = make_float4(1.0f, 1.0f, 1.0f, 1.0f);
        if (I8) r = *reinterpret_cast<const float4 *>(rs + j);
        const float rj[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++)
            f[j + i] = fmaf(I8 ? __fmul_rn(__int2float_rn((int)v[j + i]), rj[i]) : __uint_as_float(v[j + i]), sc, bi);
    }
    if (PAIRS) {
        uint32_t w[COUNT / 2];
#pragma unroll
        for (int j = 0; j < COUNT / 2; j++) {
            if (TYPE == TMQ_TYPE_BF16) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __half2 h = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
                w[j] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
#pragma unroll
        for (int j = 0; j < COUNT / 2; j++) w[j] = __byte_perm(w[j], __shfl_xor_sync(0xffffffffu, w[j], 1), pick);
#pragma unroll
        for (int j = 0; j < COUNT / 2; j++) {
            if (FULL || 2 * j < rows) {
                if (FULL || both) *reinterpret_cast<uint32_t *>(p) = w[j];
                else *reinterpret_cast<uint16_t *>(p) = (uint16_t)w[j];
            }
            p += 2 * step;
        }
    } else {
#pragma unroll
        for (int j = 0; j < COUNT; j++) {
            if (FULL || j < rows) store_one(p, TYPE, 0, f[j]);
            p += step;
        }
    }
}

template <bool I8, int COUNT>
__device__ __forceinline__ void finish_rows(const uint32_t (&v)[COUNT], const float *rs, float sc, float bi, const ScaledArgs &a,
                                            bool pairs, long long row, int n, int left, int lane) {
    uint8_t *Y = reinterpret_cast<uint8_t *>(a.Y);
    const bool full = left >= COUNT && n - lane + 32 <= a.N;
#define TMQ_STORE(TYPE, PAIRS)                                                                            \
    (full ? store_rows<I8, TYPE, PAIRS, true, COUNT>(v, rs, sc, bi, Y, row, a.ldy, n, a.N, left, lane)    \
          : store_rows<I8, TYPE, PAIRS, false, COUNT>(v, rs, sc, bi, Y, row, a.ldy, n, a.N, left, lane))
    if (a.y_type == TMQ_TYPE_F32) TMQ_STORE(TMQ_TYPE_F32, false);
    else if (a.y_type == TMQ_TYPE_BF16) pairs ? TMQ_STORE(TMQ_TYPE_BF16, true) : TMQ_STORE(TMQ_TYPE_BF16, false);
    else pairs ? TMQ_STORE(TMQ_TYPE_F16, true) : TMQ_STORE(TMQ_TYPE_F16, false);
#undef TMQ_STORE
}

template <int WK, int BN>
__global__ void __launch_bounds__(ScaledCfg<WK, BN>::THREADS, 1)
scaled_gemm_kernel(const __grid_constant__ ScaledMaps maps, const ScaledArgs a) {
    using C = ScaledCfg<WK, BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::BAR_OFF);         // activations (and 8-bit weights) landed
    uint64_t *empty = full + C::NB;
    uint64_t *ready = empty + C::NB;                                          // weights decoded
    uint64_t *taken = ready + C::NA;                                          // ... and multiplied
    uint64_t *raw_full = taken + C::NA;                                   // packed words landed
    uint64_t *raw_empty = raw_full + C::RAW_STAGES;
    uint64_t *acc_full = raw_empty + C::RAW_STAGES;                           // [2]
    uint64_t *acc_empty = acc_full + 2;                                       // [2]
    uint64_t *drain = acc_empty + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    int *begin = reinterpret_cast<int *>(smem + C::TAB_OFF);
    int *tiles = begin + a.groups + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nkb = (int)((a.K + C::BK - 1) / C::BK), whole = (int)(a.K / C::BK);
    const int unit_rows = BN > 64 ? a.unit_rows : BN;        // (low tiles are never balanced)

    // Setting up.  Each copying warp makes the barriers it starts with; without a table of boundaries to wait for it finds its
    // first unit before the predecessor in the stream has ended and brings its first stage before the CTA has met (all of it
    // behind the meeting: 12.2 us instead of 11.6 for 48 rows of 11008 x 4096, one row of 8-bit weights 8.4 instead of 7.7).
    auto init = [&](uint64_t *bars, int n, uint32_t count) {
        for (int i = lane; i < n; i += 32) ptx::mbar_init(bars + i, count);
    };
    if (warp == 0) {
        init(full, 2 * C::NB, 1);
        init(acc_full, 2, 1);
        init(acc_empty, 2, C::EPI);
        init(drain, 1, 1);
        ptx::fence_mbar_init();
        if (lane < 4) ptx::prefetch_tensormap(lane < 3 ? maps.x + lane : &maps.w);
    } else if (!C::DENSE && warp == 2) {
        init(raw_full, C::RAW_STAGES, 1);
        init(raw_empty, C::RAW_STAGES, 8);
        init(ready, C::NA, 8);
        init(taken, C::NA, 1);
        ptx::fence_mbar_init();
    } else if (warp == 1) {
        ptx::tmem_alloc(tmem_slot, C::TMEM_COLS);
        ptx::tmem_relinquish();
        ptx::tc_fence_before_sync();
    }
    __syncwarp();
    // What precedes it is this CTA's own, what follows it the stream's.  A copying warp has found its first unit by then.
    auto enter_stream = []() { asm volatile("griddepcontrol.wait;" ::: "memory"); };
    bool met = a.offsets || (warp != 0 && (C::DENSE || warp != 2));
    if (met) enter_stream();
    if (warp == 3 && a.offsets) build_table(a, begin, tiles, BN, lane);
    __syncwarp();
    // The CTA meets.  The next launch may set itself up beside this one from then on: this CTA holds its tensor memory, so it
    // cannot be kept from it by a successor that waits for this grid.
    auto meet = [&]() {
        asm volatile("bar.sync 0;" ::: "memory");
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    };
    if (met) meet();
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = met ? *reinterpret_cast<volatile uint32_t *>(tmem_slot) : 0u;

    if (warp == 0) {
        // ---------------------------------------------------------------- TMA producer (whole warp walks, one lane issues)
        {
            int s = 0, round = 0;
            uint32_t ph = 1;
            bool ok = true;
            for (Walk w(tiles, a); w.more() && ok; w.next()) {
                const Unit q = locate(w, a, begin, tiles, unit_rows, kTileC, lane);
                const int box = q.rows > maps.height[1] ? 0 : q.rows > maps.height[2] ? 1 : 2, rows = maps.height[box];
                const CUtensorMap *mx = maps.x + box, *mx_end = maps.x_end + box;
                const int wrow = (int)(q.e * a.N) + q.n0;
                const uint32_t bytes = (uint32_t)(rows * kOpRow + (C::DENSE ? C::A_BYTES : 0));      // of one k-block
                for (int kb = 0; kb < nkb; kb += C::KB) {
                    const int n = nkb - kb < C::KB ? nkb - kb : C::KB;
                    ok = __all_sync(0xffffffffu, ptx::mbar_wait_idle(empty + s, ph, a.status) ? 1 : 0) != 0;
                    if (!ok) break;
                    if (!met) enter_stream();
                    if (ptx::elect_one()) {
                        uint8_t *wd = smem + C::A_OFF + s * C::KB * C::A_BYTES, *xd = smem + C::B_OFF + s * C::KB * C::B_BYTES;
                        const bool wide = whole == nkb || kb + C::KB <= whole;
                        ptx::mbar_arrive_expect_tx(full + s, bytes * (uint32_t)(wide ? C::KB : n));
                        if (wide) {                      // k-blocks beyond the row are filled with zeros, and counted
                            if (C::DENSE) ptx::tma_load_3d(wd, &maps.w, full + s, 0, wrow, kb);
                            ptx::tma_load_3d(xd, mx, full + s, 0, q.row0, kb);
                        } else {
                            for (int j = 0; j < n; j++) {
                                if (C::DENSE) ptx::tma_load_3d(wd + j * C::A_BYTES, &maps.w_end, full + s, (kb + j) * C::BK, wrow, 0);
                                ptx::tma_load_3d(xd + j * rows * kOpRow, mx_end, full + s, (kb + j) * C::BK, q.row0, 0);
                            }
                        }
                    }
                    __syncwarp();
                    if (!met) meet();
                    met = true;
                    if (++s == C::NB) { s = 0; ph ^= 1u; round = 1; }
                }
            }
            if (!met) meet();
            // no copy may be on its way when the CTA ends, whatever became of the others (ph: parity of the slots that this
            // round has yet to refill)
            for (int i = 0; i < C::NB; i++)
                if (round || i < s) ptx::mbar_wait_own(full + i, i < s ? ph ^ 1u : ph, a.status);
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------------- MMA issuer (whole warp walks, one lane issues)
        {
            int sa = 0, sb = 0, ti = 0;
            uint32_t pa = 0, pb = 0;
            bool ok = true, landed = false;
            // even lanes watch the weights' barrier, odd lanes the activations': one round for both
            const bool acts = C::DENSE || (lane & 1);
            for (Walk w(tiles, a); w.more() && ok; w.next(), ti++) {
                const Unit q = locate(w, a, begin, tiles, unit_rows, kTileC, lane);
                const uint32_t n_mma = (uint32_t)((q.rows + kRowStep - 1) / kRowStep * kRowStep);
                const int height = maps.height[q.rows > maps.height[1] ? 0 : q.rows > maps.height[2] ? 1 : 2];
                const uint32_t b_step = (uint32_t)(height * kOpRow) >> 4;
                const uint32_t idesc = ((C::I8 ? 2u : 1u) << 4) | (1u << 7) | (1u << 10) | ((n_mma >> 3) << 17) | ((128u >> 4) << 24);
                const int buf = C::ACC_BUFS == 2 ? (ti & 1) : 0;
                const uint32_t use = (uint32_t)(C::ACC_BUFS == 2 ? (ti >> 1) : ti);
                ok = ptx::mbar_wait_warp(acc_empty + buf, (use & 1u) ^ 1u, a.status);
                if (!ok) break;
                ptx::tc_fence_after_sync();
                const uint32_t d_tmem = tmem_base + (uint32_t)(buf * BN);
                for (int kb = 0; kb < nkb; kb += C::KB) {
                    if (!landed) ok = ptx::all_lanes(ptx::mbar_wait(acts ? full + sb : ready + sa, acts ? pb : pa, a.status));
                    if (!ok) break;
                    ptx::tc_fence_after_sync();
                    const uint64_t a_desc = ptx::umma_desc_sw128(ptx::smem_u32(smem + C::A_OFF + sb * C::KB * C::A_BYTES));
                    const uint64_t b_desc = ptx::umma_desc_sw128(ptx::smem_u32(smem + C::B_OFF + sb * C::KB * C::B_BYTES));
                    const uint32_t a_tmem = tmem_base + C::A_BASE + (uint32_t)(sa * C::KB * C::A_COLS);
                    uint64_t *const used_a = taken + sa, *const used_b = empty + sb;
                    if (++sb == C::NB) { sb = 0; pb ^= 1u; }
                    if (++sa >= C::NA) { sa = 0; pa ^= 1u; }
                    // the next stage is looked up while this one's MMAs are issued
                    const bool next = ptx::mbar_test_wait(acts ? full + sb : ready + sa, acts ? pb : pa);
                    if (ptx::elect_one()) {
#pragma unroll
                        for (int j = 0; j < C::KB; j++) {
                            if (j > 0 && kb + j >= nkb) break;
#pragma unroll
                            for (int k4 = 0; k4 < kOpRow / 32; k4++) {
                                const uint32_t accum = (kb > 0 || j > 0 || k4 > 0) ? 1u : 0u;
                                const uint64_t bd = b_desc + (uint64_t)(j * b_step + 2 * k4);
                                if (C::TA) {
                                    const uint32_t at = a_tmem + (uint32_t)(j * C::A_COLS + 8 * k4);
                                    if (C::I8) ptx::umma_i8_ts(d_tmem, at, bd, idesc, accum);
                                    else ptx::umma_f16_ts(d_tmem, at, bd, idesc, accum);
                                } else {
                                    ptx::umma_i8(d_tmem, a_desc + (uint64_t)(j * (C::A_BYTES >> 4) + 2 * k4), bd, idesc, accum);
                                }
                            }
                        }
                        ptx::umma_commit(used_b);
                        if (!C::DENSE) ptx::umma_commit(used_a);
                    }
                    landed = ptx::all_lanes(next);
                }
                if (ok && ptx::elect_one()) ptx::umma_commit(acc_full + buf);
                __syncwarp();
            }
            if (!ok) {                                   // gave up: the MMAs issued so far end before anything is freed
                if (ptx::elect_one()) ptx::umma_commit(drain);
                __syncwarp();
                ptx::mbar_wait_own(drain, 0, a.status);
                __syncwarp();
            }
        }
    } else if (warp == 2) {
        // ---------------------------------------------------------------- TMA producer of the packed words
        if (!C::DENSE) {
            int s = 0, round = 0;
            uint32_t ph = 1;
            bool ok = true;
            for (Walk w(tiles, a); w.more() && ok; w.next()) {
                const Unit q = locate(w, a, begin, tiles, unit_rows, kTileC, lane);
                const int wrow = (int)(q.e * a.N) + q.n0;
                for (int kb = 0; kb < nkb; kb += C::RAWK) {
                    ok = __all_sync(0xffffffffu, ptx::mbar_wait_idle(raw_empty + s, ph, a.status) ? 1 : 0) != 0;
                    if (!ok) break;
                    if (!met) enter_stream();
                    if (ptx::elect_one()) {
                        ptx::mbar_arrive_expect_tx(raw_full + s, (uint32_t)C::RAW_BYTES);
                        ptx::tma_load_2d(smem + C::RAW_OFF + s * C::RAW_BYTES, &maps.w, raw_full + s, kb * (C::RAW_ROW / 4), wrow);
                    }
                    __syncwarp();
                    if (!met) meet();
                    met = true;
                    if (++s == C::RAW_STAGES) { s = 0; ph ^= 1u; round = 1; }
                }
            }
            if (!met) meet();
            for (int i = 0; i < C::RAW_STAGES; i++)
                if (round || i < s) ptx::mbar_wait_own(raw_full + i, i < s ? ph ^ 1u : ph, a.status);
        }
    } else if (!C::DENSE && warp >= 4 && warp < C::FIRST_EPI) {
        // ---------------------------------------------------------------- decode
        const int quarter = warp & 3, pair = (warp - 4) >> 3, half = ((warp - 4) >> 2) & 1;
        const int row = quarter * 32 + lane;
        const uint32_t raw_row = ptx::smem_u32(smem + C::RAW_OFF) + (uint32_t)(row * C::RAW_PITCH);
        const uint32_t swz = (uint32_t)(C::RAW_PITCH == 128 ? row & 7 : (row >> 1) & 3) << 4;
        const uint32_t a_lane = tmem_base + ((uint32_t)(quarter * 32) << 16) + C::A_BASE;
        const uint32_t ready0 = ptx::smem_u32(ready), taken0 = ptx::smem_u32(taken), raw_full0 = ptx::smem_u32(raw_full),
                       raw_empty0 = ptx::smem_u32(raw_empty);
        bool ok = true;
        int s = 0, rs = 0, turn = 0;
        uint32_t ph = 1, rph = 0;                        // parities: slot taken by the MMAs, box landed
        for (Walk w(tiles, a); w.more() && ok; w.next()) {
            for (int left = nkb; left > 0; left -= C::RAWK) {
                if (C::SETS == 2 || turn == pair) {
#pragma unroll
                    for (int st = 0; st < C::RAWK; st += C::KB) {
                        if (st > 0 && st >= left) break;
                        // even lanes wait for the packed words, odd lanes for the slot; a set whose k-block lies beyond the
                        // unit waits (and reports) as well, or it would run a round ahead of the others
                        ok = ptx::mbar_wait_warp_at((lane & 1) ? taken0 + 8u * s : raw_full0 + 8u * rs, (lane & 1) ? ph : rph, a.status);
                        if (!ok) break;
                        ptx::tc_fence_after_sync();
#pragma unroll
                        for (int jj = 0; jj < (C::KB == 4 ? 2 : 1); jj++) {
                            // k-block of the box, and of the stage
                            const int j = C::KB == 4 ? half + 2 * jj : st + half, js = j - st;
                            if (j > 0 && j >= left) break;
                            const uint32_t words0 = raw_row + (uint32_t)(rs * C::RAW_BYTES);
                            uint32_t cols[32];           // the row's 128 operand bytes, K ascending
                            if (C::I8) {
                                const uint4 p = ptx::lds_v4(words0 + (((uint32_t)(2 * j) << 4) ^ swz));
                                const uint4 r = ptx::lds_v4(words0 + (((uint32_t)(2 * j + 1) << 4) ^ swz));
                                const uint32_t words[8] = {p.x, p.y, p.z, p.w, r.x, r.y, r.z, r.w};
#pragma unroll
                                for (int wi = 0; wi < 8; wi++) {
                                    uint32_t d[4];
                                    decode_word_i8_ptx(words[wi], d);
#pragma unroll
                                    for (int x = 0; x < 4; x++) cols[4 * wi + x] = d[x];
                                }
                            } else {
                                const uint4 p = ptx::lds_v4(words0 + (((uint32_t)j << 4) ^ swz));
                                const uint32_t words[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                                for (int wi = 0; wi < 4; wi++) {
                                    uint32_t d[8];
                                    decode_word_bf16(words[wi], d);
#pragma unroll
                                    for (int x = 0; x < 8; x++) cols[8 * wi + x] = d[x];
                                }
                            }
                            ptx::tmem_st_x32(a_lane + (uint32_t)((s * C::KB + js) * C::A_COLS), cols);
                        }
                        ptx::tmem_st_wait();
                        ptx::tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) ptx::mbar_arrive_at(ready0 + 8u * s);
                        if (++s == C::NA) { s = 0; ph ^= 1u; }
                    }
                    if (!ok) break;
                    __syncwarp();
                    if (ok && lane == 0) ptx::mbar_arrive_at(raw_empty0 + 8u * rs);
                } else {                                 // the other pair's box
                    s += left > C::RAWK - C::KB ? C::RAWK / C::KB : (left + C::KB - 1) / C::KB;
                    if (s >= C::NA) { s -= C::NA; ph ^= 1u; }
                }
                if (C::SETS == 4) turn ^= 1;
                if (++rs == C::RAW_STAGES) { rs = 0; rph ^= 1u; }
            }
        }
    } else if (warp >= C::FIRST_EPI) {
        // ---------------------------------------------------------------- epilogue
        // lane = channel, accumulator column = row: 32 rows at a time, what is left of a unit 8 at a time
        const int quarter = warp & 3, group = (warp - C::FIRST_EPI) >> 2;
        constexpr int kStep = 8 * C::EPI;                 // rows the epilogue warps of a quarter take per round
        float *rs = reinterpret_cast<float *>(smem + C::RS_OFF) + (warp - C::FIRST_EPI) * 32;
        const bool pairs = a.y_type != TMQ_TYPE_F32 && (a.ldy & 1) == 0 && (reinterpret_cast<uintptr_t>(a.Y) & 3) == 0;
        // A set status word means that results are not to be touched; it is read here, where its latency is hidden, and not
        // before the first copies (700 cycles of every launch).
        const bool healthy = (*reinterpret_cast<volatile int *>(a.status) == 0);
        bool ok = true;
        int ti = 0;
        for (Walk w(tiles, a); w.more() && ok; w.next(), ti++) {
            const Unit q = locate(w, a, begin, tiles, unit_rows, kTileC, lane);
            const int n = q.n0 + quarter * 32 + lane;
            float sc = 1.0f, bi = 0.0f, r = 1.0f;
            if (n < a.N) {
                if (a.scale) sc = a.scale[(long long)q.e * a.N + n];
                if (a.bias) bi = a.bias[(long long)q.e * a.N + n];
            }
            if (!C::I8) sc *= 0.5f;                      // bf16 weights are carried as +-2
            int c = 32 * group;
            if (C::I8 && a.row_scale && c + lane < q.rows) r = a.row_scale[q.row0 + c + lane];
            const int buf = C::ACC_BUFS == 2 ? (ti & 1) : 0;
            ok = ptx::mbar_wait_idle(acc_full + buf, (uint32_t)(C::ACC_BUFS == 2 ? (ti >> 1) : ti) & 1u, a.status);
            ok = __all_sync(0xffffffffu, ok ? 1 : 0) != 0;
            if (!ok) break;
            ptx::tc_fence_after_sync();
            const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * BN);
            auto release = [&]() {                       // everything read: the accumulator goes back to the MMA warp
                ptx::tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(acc_empty + buf);
            };
            if (c >= q.rows) release();
#pragma unroll 1
            for (; c < q.rows; c += kStep) {
                const int left = q.rows - c;
                if (C::I8) {
                    __syncwarp();
                    rs[lane] = r;
                    __syncwarp();
                    if (a.row_scale && c + kStep + lane < q.rows) r = a.row_scale[q.row0 + c + kStep + lane];
                }
                if (left >= 32) {
                    uint32_t v[32];
                    ptx::tmem_ld_x16(lane_addr + (uint32_t)c, reinterpret_cast<uint32_t(&)[16]>(v[0]));
                    ptx::tmem_ld_x16(lane_addr + (uint32_t)c + 16, reinterpret_cast<uint32_t(&)[16]>(v[16]));
                    ptx::tmem_ld_wait();
                    if (left <= kStep) release();
                    if (healthy) finish_rows<C::I8, 32>(v, rs, sc, bi, a, pairs, q.row0 + c, n, left, lane);
                } else {
#pragma unroll 1
                    for (int j = 0; j < left; j += 8) {
                        uint32_t v[8];
                        ptx::tmem_ld_x8(lane_addr + (uint32_t)(c + j), v);
                        ptx::tmem_ld_wait();
                        if (left - j <= 8) release();
                        if (healthy) finish_rows<C::I8, 8>(v, rs + j, sc, bi, a, pairs, q.row0 + c + j, n, left - j, lane);
                    }
                }
            }
        }
        if (a.zero_rest && healthy) zero_rest_rows(a, begin, (int)threadIdx.x - C::FIRST_EPI * 32, C::EPI * 32);
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem_base, C::TMEM_COLS);
    }
}

// ---- host side --------------------------------------------------------------------------------------------------------

template <int WK, int BN>
static int launch_scaled(const ScaledProblem &p, cudaStream_t st) {
    using C = ScaledCfg<WK, BN>;
    ScaledArgs a = p.a;
    ScaledMaps maps;
    const CUtensorMapDataType xt = C::I8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int xe = C::I8 ? 1 : 2;
    const int bn = a.unit_rows;
    const int last = (int)(a.M % bn + 7) / 8 * 8;         // rows of a plain product's last tile
    maps.height[1] = a.groups > 1 ? bn / 2 : last ? last : bn;
    maps.height[2] = a.groups > 1 ? bn / 4 : maps.height[1];
    maps.height[0] = a.groups == 1 && a.M < bn ? maps.height[1] : bn;        // a plain product without a full tile
    const long long whole = a.K / C::BK;                  // k-blocks that a row fills
    const bool wide = whole > 0, ended = a.K % C::BK != 0;
    const long long w_bytes = a.N * (C::DENSE ? p.ldw : prepack_row_words(a.K, C::I8 ? 1 : 0) * 4);
    // weights that do not stay in L2 between two row tiles (300 x 28672 x 8192 8-bit, 235 MB: 122 -> 82 us; up to 58 MB the two
    // orders are within 2 %)
    a.rows_first = a.groups == 1 && !a.offsets && w_bytes > (64ll << 20) && w_bytes > a.M * p.ldx * xe;
    for (int i = 0; i < 3; i++) {        // an encoding costs about half a microsecond: boxes of one height share it
        if (i > 0 && maps.height[i] == maps.height[i - 1]) {
            maps.x[i] = maps.x[i - 1];
            maps.x_end[i] = maps.x_end[i - 1];
            continue;
        }
        if (wide && !make_map_blocks(maps.x + i, xt, xe, p.X, whole * C::BK, a.M, p.ldx * xe, C::BK, maps.height[i], C::KB, true))
            return TMQ_ERR_LAUNCH;
        if (ended && !make_map_blocks(maps.x_end + i, xt, xe, p.X, a.K, a.M, p.ldx * xe, C::BK, maps.height[i], 1, false))
            return TMQ_ERR_LAUNCH;
        if (!wide) maps.x[i] = maps.x_end[i];
        if (!ended) maps.x_end[i] = maps.x[i];
    }
    const uint64_t wrows = (uint64_t)a.groups * (uint64_t)a.N;
    bool okw = true;
    if (C::DENSE) {
        okw = (!wide || make_map_blocks(&maps.w, xt, 1, p.W, whole * C::BK, wrows, p.ldw, C::BK, kTileC, C::KB, true)) &&
              (!ended || make_map_blocks(&maps.w_end, xt, 1, p.W, a.K, wrows, p.ldw, C::BK, kTileC, 1, false));
    } else {
        okw = make_map_2d(&maps.w, CU_TENSOR_MAP_DATA_TYPE_UINT32, p.W, (uint64_t)prepack_valid_words(a.K), wrows,
                          (uint64_t)prepack_row_words(a.K, C::I8 ? 1 : 0) * 4, C::DENSE ? 4 : C::RAW_PITCH / 4, kTileC,
                          C::RAW_PITCH == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
    }
    if (!okw) return TMQ_ERR_LAUNCH;
    if (C::DENSE && !wide) maps.w = maps.w_end;
    if (!C::DENSE || !ended) maps.w_end = maps.w;
    int rc = ensure_dynamic_smem(scaled_gemm_kernel<WK, BN>, C::bytes(kMaxGroups));
    if (rc != TMQ_OK) return rc;
    // at most (rows / bn + groups) row tiles; CTAs beyond the real count find nothing to do
    const long long row_tiles = (a.M + bn - 1) / bn, tiles_n = (a.N + kTileC - 1) / kTileC;
    const long long units = (row_tiles + a.groups - 1) * tiles_n;
    if (units > 0x7FFFFFFF) return TMQ_ERR_UNSUPPORTED;
    const int grid = (int)(units < kNumSMs ? units : kNumSMs);
    a.minors = (int)(a.rows_first ? row_tiles : tiles_n);
    a.majors = (int)(a.rows_first ? tiles_n : row_tiles);
    a.d_major = grid / a.minors;
    a.d_minor = grid % a.minors;
    a.first_mul = a.minors >= kNumSMs ? 0 : 65536 / a.minors + 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(C::THREADS);
    cfg.dynamicSmemBytes = (size_t)C::bytes(a.groups);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, scaled_gemm_kernel<WK, BN>, maps, a));
}

// Rows of a work unit.  Tall tiles use each decoded weight and each copied byte for more rows, low ones leave more units for
// the SMs and cost less to fill and drain.  Time = base + the first CTA's units * k-blocks * ns per k-block, with what full
// tiles measured: 155 / 160 / 240 / 352 ns for 32 / 64 / 128 / 256 rows (int8 and bf16 alike within a sixth) and straight
// lines between 64, 128 and 256, 0.6 us more to fill and drain per doubling.  The row tiles of experts are not known here: the
// even share plus 0.6 of a tile each.  Over 150 shapes (48 .. 2048 rows, 1 .. 128 experts with 1 .. 512 rows each on average)
// the choice costs 1 % on average against the best of the four tiles; e.g. 517 x 11008 x 4096 int8 52.9 / 35.6 / 28.3 / 29.0
// us, 64 experts (2816 x 2048) of 40 rows 54.9 / 45.5 / 47.8 / 61.2 us, of 512 rows 428 / 249 / 200 / 183 us.
// A plain product's rows are also dealt evenly, in tiles of any multiple of 16 rows, where the waves that whole tiles need
// leave SMs without work and that promises 4 % (less is lost again to the units' extra operand traffic): the same 517 rows in
// 24.6 us as three tiles of 176, 1089 x 2253 x 1223 12.1 -> 10.2 us, 4 % on average over 112 random products of 65 .. 4096 rows.
static int choose_unit_rows(const ScaledArgs &a, int bk) {
    static const double per_block[4] = {0.155, 0.160, 0.240, 0.352};
    const long long tiles_n = (a.N + kTileC - 1) / kTileC;
    const double blocks = (double)((a.K + bk - 1) / bk);
    int best = 32;
    double best_cost = 1e300;
    auto consider = [&](int i, int rows, double k_blocks) {
        const double cost = 0.6 * i + k_blocks * blocks;
        if (cost < best_cost) {
            best = rows;
            best_cost = cost;
        }
    };
    for (int i = 0, bn = 32; i < 4; i++, bn *= 2) {
        if (a.offsets) {
            const double partial = 0.6 * (double)(a.groups < a.M ? a.groups : a.M);
            const double waves = ((double)a.M / bn + partial) * (double)tiles_n / kNumSMs;
            consider(i, bn, (waves < 1.0 ? 1.0 : waves) * per_block[i]);
            continue;
        }
        // k-blocks' time of a unit of `rows` rows, and of the first CTA, which has the most units: `full` of them whole, the rest
        // of the last row tile
        auto block = [&](long long rows) {
            const double below = i > 0 ? per_block[i - 1] : per_block[0];
            return rows <= bn / 2 ? below : per_block[i] - (per_block[i] - below) * (double)(bn - rows) / (double)(bn / 2);
        };
        auto plain = [&](int rows) {
            const long long tiles = (a.M + rows - 1) / rows, last = a.M - (tiles - 1) * rows;
            const long long full = ((tiles - 1) * tiles_n + kNumSMs - 1) / kNumSMs, all = (tiles * tiles_n + kNumSMs - 1) / kNumSMs;
            consider(i, rows, ((double)full * block(rows) + (double)(all - full) * block(last)) * (rows < bn ? 1.04 : 1.0));
        };
        plain(bn);
        if (i >= 2) {
            const long long waves = ((a.M + bn - 1) / bn * tiles_n + kNumSMs - 1) / kNumSMs, tiles = waves * kNumSMs / tiles_n;
            const int rows = (int)(((a.M + tiles - 1) / tiles + kRowStep - 1) / kRowStep * kRowStep);
            if (rows > bn / 2) plain(rows);
        }
    }
    return best;
}

template <int WK>
static int dispatch_scaled(ScaledProblem p, cudaStream_t st) {
    const int rows = choose_unit_rows(p.a, WK == W_TERNARY_BF16 ? 64 : 128);
    p.a.unit_rows = rows;
    if (rows > 128) return launch_scaled<WK, 256>(p, st);
    if (rows > 64) return launch_scaled<WK, 128>(p, st);
    if (rows > 32) return launch_scaled<WK, 64>(p, st);
    return launch_scaled<WK, 32>(p, st);
}

static int check_scaled(const ScaledProblem &p, int x_bytes, bool dense) {
    const ScaledArgs &a = p.a;
    if (a.M < 0 || a.N <= 0 || a.K <= 0 || a.groups < 1 || p.ldx < a.K || a.ldy < a.N) return TMQ_ERR_ARG;
    if (a.y_type < TMQ_TYPE_F32 || a.y_type > TMQ_TYPE_F16) return TMQ_ERR_ARG;
    if (a.M == 0) return TMQ_OK;
    if (!p.X || !p.W || !a.Y || !a.status || (dense && p.ldw < a.K)) return TMQ_ERR_ARG;
    if (a.M > 0x7FFFFF00 || a.K > 0x7FFFFFFF || a.groups > kMaxGroups || a.N * a.groups > 0x7FFFFFFF) return TMQ_ERR_UNSUPPORTED;
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

// Scratch of a product whose activations arrive in floating point: their codes, then the scales.  Rows of codes start at
// multiples of 16 bytes at least, and of up to 128 where that lengthens them by an eighth at most: a copy's 128-byte rows then
// touch one line instead of two (2048 x 4096 x 4080, both operands: 45.1 us from multiples of 16, 31.8 of 32, 29.6 of 64, 27.1
// of 128).
static long long code_pitch(long long K) {
    const long long unit = K >= 1024 ? 128 : K >= 512 ? 64 : K >= 256 ? 32 : 16;
    return (K + unit - 1) / unit * unit;
}

extern "C" size_t tmq_a8_workspace_bytes(int x_type, int64_t M, int64_t K) {
    if (x_type < TMQ_TYPE_F32 || x_type > TMQ_TYPE_F16 || M <= 0 || K <= 0) return 0;
    return (size_t)(M * code_pitch(K) + 4 * M);
}

// Checks an 8-bit product's arguments and quantises floating-point activations into the workspace; p then describes the
// product of the codes.  Nothing is launched for a call that is refused.
static int prepare_a8(ScaledProblem &p, int x_type, bool dense, void *workspace, size_t workspace_bytes, cudaStream_t st) {
    ScaledArgs &a = p.a;
    if (x_type < 0) return check_scaled(p, 1, dense);
    const int xe = x_type == TMQ_TYPE_F32 ? 4 : 2;
    if (a.row_scale || a.K <= 0 || p.ldx < a.K || (a.M > 0 && !p.X)) return TMQ_ERR_ARG;
    ScaledProblem q = p;
    q.X = workspace;
    q.ldx = code_pitch(a.K);
    if (!workspace) q.X = reinterpret_cast<const void *>(uintptr_t(16));      // any aligned address: only the rest is looked at
    int rc = check_scaled(q, 1, dense);
    if (rc != TMQ_OK || a.M == 0) return rc;
    if (!aligned(p.X, xe)) return TMQ_ERR_ALIGN;
    if (!workspace || workspace_bytes < tmq_a8_workspace_bytes(x_type, a.M, a.K)) return TMQ_ERR_SCRATCH;
    int8_t *codes = reinterpret_cast<int8_t *>(workspace);
    float *scales = reinterpret_cast<float *>(codes + a.M * q.ldx);
    rc = tmq_quantize_rows(p.X, x_type, codes, scales, a.M, a.K, p.ldx, q.ldx, (a.K + 15) / 16 * 16, st);
    p.X = codes;
    p.ldx = q.ldx;
    a.row_scale = scales;
    return rc;
}

extern "C" int tmq_ternary_gemm_a8(const void *X, int x_type, int64_t ldx, const float *row_scale, const uint32_t *Wt,
                                   const float *scale, const float *bias, void *Y, int y_type, int64_t M, int64_t N, int64_t K,
                                   int64_t ldy, void *workspace, size_t workspace_bytes, int *status, void *stream) {
    if (x_type < -1 || x_type > TMQ_TYPE_F16) return TMQ_ERR_ARG;
    const cudaStream_t st = (cudaStream_t)stream;
    if (M <= 8) {                        // one launch
        const int rc = launch_token_product(X, x_type, ldx, row_scale, Wt, scale, bias, Y, y_type, M, N, K, ldy, status, st);
        if (rc != TMQ_ERR_UNSUPPORTED) return rc;
    }
    ScaledProblem p = {X, Wt, ldx, 0, {row_scale, scale, bias, Y, nullptr, M, N, K, ldy, 1, 0, y_type, 0, status}};
    int rc = prepare_a8(p, x_type, false, workspace, workspace_bytes, st);
    if (rc != TMQ_OK || M == 0) return rc;
    if (M <= 8 && x_type >= 0) {         // too many elements to quantise in every CTA, but few rows
        rc = launch_token_product(p.X, -1, p.ldx, p.a.row_scale, Wt, scale, bias, Y, y_type, M, N, K, ldy, status, st);
        if (rc != TMQ_ERR_UNSUPPORTED) return rc;
    }
    return dispatch_scaled<W_TERNARY_I8>(p, st);
}

extern "C" int tmq_gemm_i8(const void *X, int x_type, int64_t ldx, const float *row_scale, const int8_t *W, int64_t ldw,
                           const float *scale, const float *bias, void *Y, int y_type, int64_t M, int64_t N, int64_t K,
                           int64_t ldy, void *workspace, size_t workspace_bytes, int *status, void *stream) {
    if (x_type < -1 || x_type > TMQ_TYPE_F16) return TMQ_ERR_ARG;
    ScaledProblem p = {X, W, ldx, ldw, {row_scale, scale, bias, Y, nullptr, M, N, K, ldy, 1, 0, y_type, 0, status}};
    const int rc = prepare_a8(p, x_type, true, workspace, workspace_bytes, (cudaStream_t)stream);
    return rc != TMQ_OK || M == 0 ? rc : dispatch_scaled<W_DENSE_I8>(p, (cudaStream_t)stream);
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
