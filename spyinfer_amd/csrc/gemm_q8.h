// What the products in 8-bit integers share.
#pragma once
#include "q8.h"

#define Q8_DIES 8

// One result: a sum times its row's and its column's scale; gated, the activation of the gate's times the up rows'.
template <int EPI>
__device__ __forceinline__ float q8_value(const GateAct& act, int a, int up, float fx, float fw, float fu) {
    const float y = (float)a * fx * fw;
    return EPI == Q8_GATED ? gated_value_short(act, y, (float)up * fx * fu) : y;
}
// 16 bytes of results
__device__ __forceinline__ void q8_store_piece(bf16_t* o, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(o) = uint4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}
__device__ __forceinline__ void q8_store_piece(float* o, const float (&v)[4]) { *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]); }

// Blocks of MT (8 to 16) row tiles and 256 columns, one a compute unit (gemm_q8_tall.hip); M >= 16 MT
int q8_tall_launch(void* C, int c_dtype, const int8_t* X, const float* sx, const int8_t* W, const float* sw, int M, int N, int tiles, int chunks, int gated,
                   GateAct act, int MT, hipStream_t st);
