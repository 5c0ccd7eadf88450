// Rows and matrices in 8-bit integers.
//
// Rows: int8 [rows][pitch], pitch = the width rounded up to 256 (what lies behind a row's last value may be anything: the matrix has zeros there), and a
// float32 scale for each row; a row stands for integers times its scale.
// Matrices: [K/256 chunks][N/16 tiles][4 steps][64 lanes][16 bytes], lane 16 g + r of step s of chunk c of tile t holding
// W[16 t + r][256 c + 64 s + 16 g ..]: a wave's operand of one 16 x 16 x 64 product is one load of 1 KiB in one piece.  K is filled up to 256 and N to 16
// with zeros (a gated matrix' gate rows and up rows each), and every row of W has a float32 scale.
#pragma once
#include "common.h"

#define Q8_CHUNK 256             // bytes of K in a chunk
#define Q8_STEP 64               // of K in one matrix instruction
typedef int q8_i32x4_t __attribute__((ext_vector_type(4)));

#define Q8_STORE 0               // C[M][N]
#define Q8_GATED 1               // W = [gate rows | up rows], C[M][N / 2] = act(gate) * up

// 16 x 16 x 64: d[column 4 g + e][row r] += sum over k of w[column][k] x[row][k]; lane 16 g + r brings 16 of K of row r of both
__device__ __forceinline__ q8_i32x4_t q8_mfma(q8_i32x4_t w, q8_i32x4_t x, q8_i32x4_t acc) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, acc, 0, 0, 0);
}
