// Products of 8-bit integer rows with 8-bit integer matrices (q8.h has both forms), sums in 32-bit integers, which hold them exactly
// (K < 2^17):  y[m][n] = sum * row scale * column scale, rounded once; or the gated pair of such values.
#include "gemm_q8.h"

#define Q8_WAVES 4

// One block has 16 MT rows and one column tile (gated: the gate's and the up values' of the same columns); its waves share K by chunks
// and add through LDS.
template <int MT, int EPI, typename TC>
__global__ __launch_bounds__(Q8_WAVES * 64) void gemm_q8_kernel(TC* __restrict__ C, const int8_t* __restrict__ X, int64_t pitch, const float* __restrict__ sx,
                                                                const int8_t* __restrict__ W, const float* __restrict__ sw, int M, int N, int tiles, int chunks,
                                                                GateAct act) {
    constexpr int NT = EPI == Q8_GATED ? 2 : 1;
    __shared__ q8_i32x4_t red[Q8_WAVES - 1][NT][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
    const int tile = blockIdx.x, row0 = blockIdx.y * MT * 16;
    const int rows = min(M - row0, MT * 16);
    // what lies behind the last row reads as zeros; behind a row's end the matrix has zeros
    const auto xres = __builtin_amdgcn_make_buffer_rsrc((void*)(X + (size_t)row0 * pitch), 0, (int)(rows * pitch), 0x00020000);
    q8_i32x4_t acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = q8_i32x4_t{0, 0, 0, 0};
    for (int c = wave; c < chunks; c += Q8_WAVES) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            q8_i32x4_t w[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j)
                w[j] = *reinterpret_cast<const q8_i32x4_t*>(W + ((size_t)c * tiles + tile + j * (tiles / 2)) * 4096 + s * 1024 + lane * 16);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int at = (i * 16 + r) * (int)pitch + c * Q8_CHUNK + s * Q8_STEP + g * 16;
                const q8_i32x4_t x = __builtin_bit_cast(q8_i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(xres, at, 0, 0));
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[j][i] = q8_mfma(w[j], x, acc[j][i]);
            }
        }
    }
    if (wave) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < MT; ++i) red[wave - 1][j][i][lane] = acc[j][i];
    }
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
        for (int v = 0; v < Q8_WAVES - 1; ++v)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[j][i] += red[v][j][i][lane];
        const int m = row0 + i * 16 + r;
        if (m >= M) continue;
        const float fx = sx[m];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int n = tile * 16 + 4 * g + e;
            if (n >= N) continue;
            float y = (float)acc[0][i][e] * fx * sw[n];
            if (EPI == Q8_GATED) y = gated_value_short(act, y, (float)acc[NT - 1][i][e] * fx * sw[n + tiles * 8]);
            C[(size_t)m * N + n] = from_f32<TC>(y);
        }
    }
}

// C: bfloat16 or float32 [M, N].  X: rows of `pitch` bytes (a multiple of 16) and their scales; W: the matrix laid out, `tiles` column tiles (gated:
// of both halves) and `chunks` of K, and its scales [16 tiles].  Gated: C is bfloat16 [M, N], N one half's columns.
extern "C" int spy_gemm_q8(void* C, int c_dtype, const void* X, int64_t pitch, const float* sx, const void* W, const float* sw, int M, int N, int tiles, int chunks,
                           int gated, int act_code, hipStream_t st) {
    GateAct act = {1.f, 0.f};
    SPY_REQUIRE(M > 0 && N > 0 && tiles > 0 && chunks > 0, "spy_gemm_q8: empty operand");
    SPY_REQUIRE(pitch % 16 == 0 && pitch <= (int64_t)chunks * Q8_CHUNK && pitch > (int64_t)(chunks - 1) * Q8_CHUNK, "spy_gemm_q8: rows of %lld bytes for %d chunks of K", (long long)pitch, chunks);
    SPY_REQUIRE(chunks <= 511 && (int64_t)tiles * chunks * 4096 < (1ll << 31), "spy_gemm_q8: a matrix of %d x %d tiles is too large", tiles, chunks);
    SPY_REQUIRE(gated ? tiles % 2 == 0 && N <= tiles * 8 && N > tiles * 8 - 16 : N <= tiles * 16 && N > tiles * 16 - 16, "spy_gemm_q8: %d columns in %d tiles", N, tiles);
    SPY_REQUIRE((((uintptr_t)X | (uintptr_t)W) % 16) == 0, "spy_gemm_q8: operands must be 16-byte aligned");
    SPY_REQUIRE(!gated || (gate_act_of(act_code, &act) && c_dtype == SPY_BF16), "spy_gemm_q8: activation %d, result dtype %d", act_code, c_dtype);
    SPY_REQUIRE(M <= 65535 * 64, "spy_gemm_q8: too many rows");
    if (M > 512) return q8_tall_launch(C, c_dtype, (const int8_t*)X, pitch, sx, (const int8_t*)W, sw, M, N, tiles, chunks, gated, act, 16, st);
#define Q8(MT, EPI, TC) gemm_q8_kernel<MT, EPI, TC><<<dim3(EPI == Q8_GATED ? tiles / 2 : tiles, (M + 16 * MT - 1) / (16 * MT)), Q8_WAVES * 64, 0, st>>>( \
        (TC*)C, (const int8_t*)X, pitch, sx, (const int8_t*)W, sw, M, N, tiles, chunks, act)
    if (gated) { if (M <= 16) Q8(1, Q8_GATED, bf16_t); else Q8(4, Q8_GATED, bf16_t); }
    else if (c_dtype == SPY_F32) { if (M <= 16) Q8(1, Q8_STORE, float); else Q8(4, Q8_STORE, float); }
    else { if (M <= 16) Q8(1, Q8_STORE, bf16_t); else Q8(4, Q8_STORE, bf16_t); }
#undef Q8
    SPY_CHECK_LAUNCH("spy_gemm_q8");
    return 0;
}
