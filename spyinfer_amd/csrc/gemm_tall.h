// The turns of blocks of 8 to 16 row tiles and 256 columns, one block a compute unit and one wave a SIMD, for operands of 16 bytes a lane:
// bfloat16 (gemm_rows_tall.hip, which has the design and what it measures) and 8-bit integers (gemm_q8_tall.hip).
#pragma once
#include "common.h"

// All turns of a block: n of them, of 256 bytes of K (128 bfloat16 or 256 8-bit integers).  OP: the operands' and the sums' registers, and two products of
// a row tile with two column tiles, the sums in accumulation registers (csrc/gemm_rows_tall.hip says why and what that asks of the code around it).  wres, w_lane, w_at, w_turn: W's buffer, this lane's bytes in a load, each column tile's place and a
// turn's bytes.  load_x(stage, i, c): asks for row tile i of turn c, straight into LDS (a wave 4 of its 16 rows).  Ends with nothing under way,
// the stages free and the sums fit to be read.  MT: 8 to 16.
template <typename OP, int MT, typename RES, typename X>
__device__ __forceinline__ void gr_tall_turns(typename OP::sums_t (&acc)[4][MT], RES wres, int w_lane, const int (&w_at)[4], int w_turn, int n, bf16_t* stage0, bf16_t* stage1,
                                              int lane, X load_x) {
    // (two arrays of their own: reads of a stage that the compiler cannot tell from the one that loads go to wait for these)
    typedef typename OP::operand_t operand_t;
    typedef typename OP::sums_t sums_t;
    static_assert(MT >= 8 && MT <= 16, "eight loads of W go between the row tiles of a step");
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = sums_t{0, 0, 0, 0};
    operand_t w[2][4][4];
    auto load_w = [&](int d, int s, int j, int c) {
        w[d][s][j] = __builtin_bit_cast(operand_t, __builtin_amdgcn_raw_buffer_load_b128(wres, w_lane, w_at[j] + c * w_turn + s * 1024, 0));
    };
    // The products of a turn with w[d].  Between them, one load a row tile: X of turn `next` into the other stage while step 0 runs; W of turn
    // `after` into the registers of steps 0 to 2 as soon as these are done; and, in step 1, W of turn `next` into the other set's
    // step 3, which the turn before had used to its end.  X's operands are read three ahead.
    auto products = [&](int d, const bf16_t* stage, bf16_t* other, int next, int after) {
        const bf16_t* xb = stage + r * 128;
        operand_t x[4];
#pragma unroll
        for (int q = 0; q < 3; ++q) x[q] = *reinterpret_cast<const operand_t*>(xb + (q % MT) * 2048 + ((4 * (q / MT) + g) ^ r) * 8);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_nop 1");
#pragma unroll
        for (int q = 0; q < 4 * MT; ++q) {
            const int s = q / MT, i = q % MT, ahead = q + 3;
            if (ahead < 4 * MT) x[ahead % 4] = *reinterpret_cast<const operand_t*>(xb + (ahead % MT) * 2048 + ((4 * (ahead / MT) + g) ^ r) * 8);
            OP::mfma2(acc[0][i], acc[1][i], w[d][s][0], w[d][s][1], x[q % 4]);
            __builtin_amdgcn_sched_barrier(0);
            if (s == 0) load_x(other, i, next);
            else if (i < 4) load_w(d, s - 1, i, after);
            else if (s == 1 && i < 8) load_w(1 - d, 3, i - 4, next);
            __builtin_amdgcn_sched_barrier(0);
            OP::mfma2(acc[2][i], acc[3][i], w[d][s][2], w[d][s][3], x[q % 4]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // A turn issues X's loads before its 16 loads of W, and loads return in order: at most 16 under way means that X is there
    auto turn = [&]() {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < MT; ++i) load_x(stage0, i, 0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) load_w(0, s, j, 0);
    turn();
#pragma unroll
    for (int s = 0; s < 3; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) load_w(1, s, j, min(1, n - 1));
    __builtin_amdgcn_sched_barrier(0);
    // (the last turns ask for the last turn's operands again: loads that a branch skips would make the compiler count fewer under way)
    int c = 0;
    for (; c + 1 < n; c += 2) {
        const int after = min(c + 2, n - 1);
        products(0, stage0, stage1, c + 1, after);
        turn();
        products(1, stage1, stage0, after, min(c + 3, n - 1));
        turn();
    }
    if (c < n) products(0, stage0, stage1, n - 1, n - 1);
    sums_settle(acc);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}
