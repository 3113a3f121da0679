// Tiles, rings and shared memory of the scaled and grouped products' kernel (scaled_gemm.cu).  Plain C++: the host compiles it too.
#pragma once
#include "tmq_b200.h"

namespace tmq {

enum { W_TERNARY_BF16 = 0, W_TERNARY_I8 = 1, W_DENSE_I8 = 2 };

constexpr int kMaxGroups = TMQ_GROUPS_MAX;
constexpr int kTileC = 128;          // channels of a unit (MMA M)
constexpr int kOpRow = 128;          // bytes of one operand row per k-block: 64 bf16 or 128 int8
constexpr int kRowStep = 16;         // granularity of a unit's MMA N

template <int WK, int BN>
struct ScaledCfg {
    static constexpr bool DENSE = WK == W_DENSE_I8, I8 = WK != W_TERNARY_BF16;
    static constexpr bool TA = !DENSE;                                        // A operand in tensor memory
    static constexpr int BK = I8 ? 128 : 64;
    static constexpr int RAW_ROW = DENSE ? 0 : I8 ? 32 : 16;                  // packed bytes per channel and k-block
    // Packed words come RAWK k-blocks per box: a box costs the TMA unit about four cycles a row whatever its width (one
    // k-block per box measured 280 ns per k-block at any row count).  Rows of 128 / 64 bytes with the swizzle of that
    // width, so the decode warps' 16-byte reads meet no bank conflicts.  (Two k-blocks for int8 tiles of 256 rows, whose
    // activations take 192 KB.)
    static constexpr int RAWK = DENSE ? 1 : I8 && BN > 128 ? 2 : 4;
    static constexpr int RAW_PITCH = RAWK * RAW_ROW;
    // A pipeline stage is KB k-blocks: the MMA warp pays its barrier round (about 270 cycles of latency) once a stage, and
    // four MMAs of a k-block alone cover 170.  One k-block per stage measured 280 - 300 ns per k-block for every BN <= 128; two
    // instead of four for tiles of up to 64 rows 199 instead of 174 (32 rows, k-blocks of K = 16384 with fill and drain).
    static constexpr int KB = DENSE && BN > 128 ? 1 : !DENSE && BN <= 64 ? 4 : 2;
    // Three rings: decoded weights (NA stages of tensor memory), activations and
    // 8-bit weights (NB stages), packed words (RAW_STAGES boxes).  An activation box takes about 1250 cycles from L2, so its
    // ring is the one that must be deep: three stages of four k-blocks, shared with the weights, held bf16 tiles of 64 rows
    // at 154 ns per k-block.
    // A barrier's parity tells its last two phases apart, so whoever waits must have seen the phase before the one it waits for,
    // or know that it is over.  Copying and MMA warps see every phase.  Of the decode warps a pair of sets sees only its own boxes
    // (every second one where there are two pairs):
    //   packed words: boxes land in any order, so a slot's boxes must all be one pair's, hence an even RAW_STAGES;
    //   slots of decoded weights: MMAs end in order, so the slot a pair last waited for, at most RAWK / KB + 1 stages before, tells
    //   that all older ones are over too.  NA stages back from there must not be later than 2 NA stages back from now.
    static constexpr int NA = DENSE ? 0 : BN > 128 ? (I8 ? 4 : 3) : BN > 64 ? 4 : 3;
    static constexpr int NB = DENSE ? (BN > 128 ? 4 : BN > 64 ? 3 : BN > 32 ? 4 : 5) : BN > 128 ? 3 : BN > 64 ? (I8 ? 4 : 5) : BN > 32 ? 4 : 7;
    static constexpr int RAW_STAGES = DENSE ? 0 : BN > 128 ? 2 : 4;
    static constexpr int A_BYTES = TA ? 0 : kTileC * kOpRow;                  // of one k-block
    static constexpr int B_BYTES = BN * kOpRow;
    static constexpr int RAW_BYTES = kTileC * RAW_PITCH;
    // Two accumulators, so that one unit's results leave under the next unit's MMAs, but one where 256 rows and the decoded
    // weights fill tensor memory.  (int8 with two accumulators and the weights decoded into shared memory, 104 KB a k-block
    // through it: 8192 x 28672 x 8192 7 - 11 % slower.)
    static constexpr int ACC_BUFS = (TA && BN > 128) ? 1 : 2;
    static constexpr int A_COLS = kOpRow / 4;
    static constexpr int A_BASE = ACC_BUFS * BN;
    static constexpr int TMEM_NEED = A_BASE + (TA ? NA * KB * A_COLS : 0);
    static constexpr int TMEM_COLS = TMEM_NEED <= 128 ? 128 : TMEM_NEED <= 256 ? 256 : 512;
    static_assert(TMEM_NEED <= 512, "tensor memory exceeded");
    // Decode warps come in sets of four (one per lane quarter), a pair of sets takes a box of packed words: set i its k-blocks
    // i and i + 2.  Everything a round does besides decoding (waits, addresses, arrivals: about 100 integer instructions
    // against 72 for the codes of an int8 k-block) is paid once per box, and a second pair works on the next box meanwhile
    // where the MMAs of a k-block do not cover the decoding of one.
    static constexpr int SETS = BN > 128 ? 2 : 4;
    static_assert(RAW_STAGES % (SETS / 2) == 0, "a pair would wait for boxes it has not followed");
    static_assert(DENSE || SETS == 2 || RAWK / KB + 1 <= NA, "a pair would wait for slots it has not followed");
    static constexpr int DECODERS = DENSE ? 0 : 4 * SETS;
    static constexpr int FIRST_EPI = 4 + DECODERS;
    static constexpr int EPI = BN > 128 ? 8 : 4;                              // epilogue warps
    static constexpr int THREADS = (FIRST_EPI + EPI) * 32;
    // shared memory
    static constexpr int A_OFF = 0;
    static constexpr int B_OFF = A_OFF + NB * KB * A_BYTES;
    static constexpr int RAW_OFF = B_OFF + NB * KB * B_BYTES;
    static constexpr int RS_OFF = RAW_OFF + RAW_STAGES * RAW_BYTES;           // 32 row scales per epilogue warp
    static constexpr int BAR_OFF = RS_OFF + EPI * 128;
    static constexpr int TAB_OFF = BAR_OFF + 512;                             // begin[groups + 1], tiles[groups + 1]
    static constexpr int bytes(int groups) { return TAB_OFF + 2 * 4 * (groups + 1) + 1024; }
    static_assert(TAB_OFF + 2 * 4 * (kMaxGroups + 1) + 1024 <= 227 * 1024, "shared memory exceeded");
};

}  // namespace tmq
