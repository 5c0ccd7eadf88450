// Products of many rows in 8-bit integers (q8.h) by blocks of 8 to 16 row tiles and 256 columns, one a compute unit (gemm_tall.h).
//
// A lane's 16 bytes are 16 integers where they are 8 bfloat16 there, and an instruction of the same 16 clocks multiplies twice as many; so the bfloat16
// products' turns stand as they are, of 256 bytes of K.  Measured: 4096 rows, 12288 -> 4096 145 to 156 us by box and clock (2.6 to 2.8 POP/s; the library's 8192 x 8192 x 8192 of
// integers 2.03, the first kernel here, whose waves took X's operands straight from memory, 1452 us), gated, 4096 -> 2 x 12288 322 to 348 us (2.4 to 2.6).
// What bounds it: by the counters the matrix units are busy for 68 % of all clocks and the clock is 1.97 GHz; with half of the compute units at work a turn takes
// 2.2 us, with all of them 3: the power.  Gated, the activations of a block's results cost 2 to 3 us of the 57 that it takes.  Operands read
// five or seven row tiles ahead in place of three change nothing.
#include "gemm_q8.h"
#include "gemm_tall.h"

// Two products of a row tile with two column tiles of W.  (The compiler does not see matrix instructions: gemm_rows_tall.hip has what follows from that.)
struct TallQ8 {
    typedef q8_i32x4_t operand_t;
    typedef q8_i32x4_t sums_t;
    static __device__ __forceinline__ void mfma2(sums_t& a, sums_t& b, operand_t w0, operand_t w1, operand_t x) {
        asm volatile("v_mfma_i32_16x16x64_i8 %0, %2, %4, %0\n\tv_mfma_i32_16x16x64_i8 %1, %3, %4, %1" : "+a"(a), "+a"(b) : "v"(w0), "v"(w1), "v"(x));
    }
};

// A block's results through its LDS stage, as many row tiles at a time as fit, in a part that a wave has to itself: the sums go there as they are, and a short loop reads
// pieces of rows, forms the values and stores whole lines.  A piece of four columns lies at place p ^ (row % 16).
// sx: the block's row scales (q8_row_scale) in LDS; sw: the column scales, those of the up rows `half` on; at: this wave's first column; columns: those that exist.
template <int MT, int EPI, typename TC>
__device__ __forceinline__ void q8_tall_results(q8_i32x4_t (&acc)[4][MT], bf16_t* stage, TC* out, int64_t ld, int columns, int at, const float2* sx, const float* sw,
                                                int half, const GateAct& act, int lane, int wave) {
    constexpr int CT = MT / 4, VEC = 16 / sizeof(TC), PIECES = (EPI == Q8_GATED ? 32 : 64) / VEC, ROWS = 64 / PIECES;
    int* mine = reinterpret_cast<int*>(stage) + wave * CT * 16 * 64;
    const int r = lane & 15, g = lane >> 4, q = (lane % PIECES) * (VEC / 4), column = at + q * 4;
    const bool whole = ld % VEC == 0 && (uintptr_t)out % 16 == 0;              // (a piece then exists whole or not at all)
    float fw[VEC], fu[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        fw[e] = column + e < columns ? sw[column + e] : 0.f;
        fu[e] = EPI == Q8_GATED && column + e < columns ? sw[half + column + e] : 0.f;
    }
#pragma unroll
    for (int i0 = 0; i0 < MT; i0 += CT) {
#pragma unroll
        for (int i = i0; i < i0 + CT && i < MT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<q8_i32x4_t*>(mine + ((i - i0) * 16 + r) * 64 + ((j * 4 + g) ^ r) * 4) = acc[j][i];
        __builtin_amdgcn_sched_barrier(0);
        const int here = 16 * min(CT, MT - i0);
        if (whole) {
#pragma unroll 2
            for (int row = lane / PIECES; row < here; row += ROWS) {
                const int* from = mine + row * 64;
                const float2 fx = sx[i0 * 16 + row];
                float v[VEC];
#pragma unroll
                for (int k = 0; k < VEC / 4; ++k) {
                    const q8_i32x4_t a = *reinterpret_cast<const q8_i32x4_t*>(from + ((q + k) ^ (row & 15)) * 4);
                    const q8_i32x4_t b = *reinterpret_cast<const q8_i32x4_t*>(from + ((q + k + (EPI == Q8_GATED ? 8 : 0)) ^ (row & 15)) * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[k * 4 + e] = q8_value<EPI>(act, a[e], b[e], fx, fw[k * 4 + e], fu[k * 4 + e]);
                }
                TC* o = out + (int64_t)(i0 * 16 + row) * ld + column;
                if (column < columns) q8_store_piece(o, v);
            }
        } else {
            // rows that begin anywhere: a lane has a column
            constexpr int WIDTH = EPI == Q8_GATED ? 32 : 64;
            const int c = lane % WIDTH, up = c + (EPI == Q8_GATED ? 32 : 0);
            const bool is = at + c < columns;
            const float cw = is ? sw[at + c] : 0.f, cu = EPI == Q8_GATED && is ? sw[half + at + c] : 0.f;
#pragma unroll 8
            for (int row = lane / WIDTH; row < here; row += 64 / WIDTH) {
                const int a = mine[row * 64 + ((c / 4) ^ (row & 15)) * 4 + c % 4], b = mine[row * 64 + ((up / 4) ^ (row & 15)) * 4 + up % 4];
                if (is) out[(int64_t)(i0 * 16 + row) * ld + at + c] = from_f32<TC>(q8_value<EPI>(act, a, b, sx[i0 * 16 + row], cw, cu));
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

template <int MT, int EPI, typename TC>
__global__ __launch_bounds__(256, 1) void gemm_q8_tall_kernel(TC* C, const int8_t* X, const float* sx, const int8_t* W, const float* sw, int M, int N,
                                                              int tiles, int chunks, int n_rows, int n_cols, GateAct act) {
    __shared__ __align__(1024) bf16_t stage0[MT * 16 * 128];
    __shared__ __align__(1024) bf16_t stage1[MT * 16 * 128];
    __shared__ float2 row_scales[MT * 16];
    // blocks go to the dies in turn: a die takes a run of the blocks
    const int blocks = n_rows * n_cols, per = (blocks + Q8_DIES - 1) / Q8_DIES, idx = blockIdx.x / Q8_DIES;
    const int v = (blockIdx.x % Q8_DIES) * per + idx;
    if (idx >= per || v >= blocks) return;
    const int pitch = chunks * Q8_CHUNK;
    int row_t, col_t;
    q8_block_at(v, n_rows, n_cols, 6, row_t, col_t);
    const int row0 = min(row_t * MT * 16, M - MT * 16);          // the last rows' tile ends with row M - 1 (what it shares with the one before, both form alike)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (threadIdx.x < MT * 16) row_scales[threadIdx.x] = q8_row_scale(sx[row0 + threadIdx.x]);              // (MT <= 16; behind the turns' barriers when it is read)
    const auto wres = __builtin_amdgcn_make_buffer_rsrc((void*)W, 0, tiles * chunks * 4096, 0x00020000);
    const auto xres = __builtin_amdgcn_make_buffer_rsrc((void*)(X + (size_t)row0 * pitch), 0, MT * 16 * pitch, 0x00020000);
    int w_at[4];                                       // this wave's column tiles; one that does not exist reads the last (nothing is stored)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int tile = EPI == Q8_GATED ? (j >> 1) * (tiles / 2) + min(col_t * 8 + wave * 2 + (j & 1), tiles / 2 - 1) : min(col_t * 16 + wave * 4 + j, tiles - 1);
        w_at[j] = __builtin_amdgcn_readfirstlane(tile * 4096);
    }
    // X: a wave's load brings 4 rows of 256 bytes; lane l has the piece that belongs to place l % 16 of row l / 16
    const int s_row = wave * 4 + (lane >> 4);
    const int x_lane = s_row * pitch + ((lane & 15) ^ s_row) * 16;
    q8_i32x4_t acc[4][MT];
    gr_tall_turns<TallQ8, MT>(acc, wres, lane * 16, w_at, tiles * 4096, chunks, stage0, stage1, lane, [&](bf16_t* stage, int i, int c) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xres, (__attribute__((address_space(3))) void*)(stage + (i * 4 + wave) * 512), 16, x_lane,
                                                 i * 16 * pitch + c * Q8_CHUNK, 0, 0);
    });
    constexpr int WAVE_COLUMNS = EPI == Q8_GATED ? 32 : 64;
    q8_tall_results<MT, EPI, TC>(acc, stage0, C + (size_t)row0 * N, N, N, (col_t * 4 + wave) * WAVE_COLUMNS, row_scales, sw, tiles * 8, act, lane, wave);
}

template <int MT>
static int tall_launch(void* C, int c_dtype, const int8_t* X, const float* sx, const int8_t* W, const float* sw, int M, int N, int tiles, int chunks, int gated,
                       GateAct act, hipStream_t st) {
    const int n_rows = (M + MT * 16 - 1) / (MT * 16), n_cols = gated ? (N + 127) / 128 : (N + 255) / 256;
    const int64_t blocks = (int64_t)n_rows * n_cols;
    SPY_REQUIRE(M >= MT * 16 && (blocks + Q8_DIES) * 256 < (1ll << 32), "spy_gemm_q8: %d rows in blocks of %d row tiles, %lld blocks", M, MT, (long long)blocks);
    const unsigned grid = (unsigned)((blocks + Q8_DIES - 1) / Q8_DIES * Q8_DIES);
#define TALL(EPI, TC) gemm_q8_tall_kernel<MT, EPI, TC><<<grid, 256, 0, st>>>((TC*)C, X, sx, W, sw, M, N, tiles, chunks, n_rows, n_cols, act)
    if (gated) TALL(Q8_GATED, bf16_t);
    else if (c_dtype == SPY_F32) TALL(Q8_STORE, float);
    else TALL(Q8_STORE, bf16_t);
#undef TALL
    SPY_CHECK_LAUNCH("spy_gemm_q8");
    return 0;
}

int q8_tall_launch(void* C, int c_dtype, const int8_t* X, const float* sx, const int8_t* W, const float* sw, int M, int N, int tiles, int chunks, int gated,
                   GateAct act, int MT, hipStream_t st) {
#define CASE(T) case T: return tall_launch<T>(C, c_dtype, X, sx, W, sw, M, N, tiles, chunks, gated, act, st)
    switch (MT) { CASE(8); CASE(10); CASE(12); CASE(14); CASE(16); }
#undef CASE
    return spy_fail("spy_gemm_q8: %d row tiles", MT);
}
