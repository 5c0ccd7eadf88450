// What the products in 8-bit integers share.
#pragma once
#include "q8.h"

#define Q8_DIES 8

// The block at place v of the order of which every die takes a run: bands of `high` rows of blocks, one column of blocks of a band behind the other.  The 32 or more
// blocks that a die has at a time then read few rows of X and few columns of W.  (Whole columns, which read W into one L2 only, need many rows' X there at a time:
// blocks of 128 x 64, 3503 rows, 9728 -> 1024 78 us for 52, 1400 rows, 4096 -> 4096 45 for 42; of 256 x 256, 8192 rows, 4096 -> 4096 121 for 112, 4096 rows, 12288 ->
// 4096 152 for 148.  Bands of 8 and 16 of the former 51.5 and 57; of 4, 6 and 8 of 128 x 256, 4096 rows, 4096 -> 6144 100, 96.4 and 100, in one 120.)
__device__ __forceinline__ void q8_block_at(int v, int n_rows, int n_cols, int high, int& row, int& col) {
    int band = 0;
    if (n_rows > high) {
        band = v / (high * n_cols) * high;
        v -= band * n_cols;
        high = min(n_rows - band, high);
    } else high = n_rows;
    col = v / high;
    row = band + v % high;
}

// A row's scale as the results take it, a factor and a power of two for the end.  A sum is up to 2^31, so with a scale beyond 2^96 the first product of a sum,
// its row's and its column's scale may be no float32 though the result is one: 2^64 is then left to the end.  (The product before it is at
// least 2^32 times the column's scale, and so not below the normal numbers.)  Otherwise the power is one, and the result what it would be without.
// (Cost: nothing to 1 % of a product, 1.4 % of a gated one of many rows; a branch around it in the tall blocks' loop 1 to 3 %.)
__device__ __forceinline__ float2 q8_row_scale(float s) {
    const bool large = fabsf(s) > 0x1p96f;
    return float2{large ? s * 0x1p-64f : s, large ? 0x1p64f : 1.f};
}
// One result: a sum times its row's and its column's scale, in float32; gated, the activation of the gate's times the up rows'.
template <int EPI>
__device__ __forceinline__ float q8_value(const GateAct& act, int a, int up, float2 fx, float fw, float fu) {
    const float y = (float)a * fx.x * fw * fx.y;
    return EPI == Q8_GATED ? gated_value_short(act, y, (float)up * fx.x * fu * fx.y) : y;
}
// 16 bytes of results
__device__ __forceinline__ void q8_store_piece(bf16_t* o, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(o) = uint4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}
__device__ __forceinline__ void q8_store_piece(float* o, const float (&v)[4]) { *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]); }

// Blocks of MT (8 to 16) row tiles and 256 columns, one a compute unit (gemm_q8_tall.hip); M >= 16 MT
int q8_tall_launch(void* C, int c_dtype, const int8_t* X, const float* sx, const int8_t* W, const float* sw, int M, int N, int tiles, int chunks, int gated,
                   GateAct act, int MT, hipStream_t st);
