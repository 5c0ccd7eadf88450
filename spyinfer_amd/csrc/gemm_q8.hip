// Products of 8-bit integer rows with 8-bit integer matrices (q8.h has both forms), sums in 32-bit integers, which hold them exactly
// (K < 2^17):  y[m][n] = sum * row scale * column scale in float32 (three roundings), then rounded to the result's type; or the gated pair of such values.
//
// Few rows and some: a block has MT row tiles and NT column tiles (gated: the gate's and the up values' of the same columns).  Its four waves take units
// of S steps of 64 of K in turn, each all of the block's tiles, so that every byte is loaded by the one wave that multiplies it, and no wave
// waits for another before their sums are added, through LDS, at the end.  W goes from memory into operand registers, a kilobyte a load.  X goes through LDS, in a part that a
// wave has to itself: its loads there bring whole pieces of 64 S bytes of a row, its reads from there are the operands (16 rows straight from memory
// are 64 pieces of 16 bytes a load, which take the address unit 64 clocks: 64 rows, 12288 -> 4096 30.6 us for 20.7).  Piece p of row r of a tile
// lies at place p ^ (r S / 4), so that the reads meet in no bank.  A wave keeps two units under way; units behind the end are loads beyond their buffers, which ask
// the memory for nothing and bring zeros.
//
// What bounds it: few rows the matrix from memory (8 rows, 12288 -> 4096 9.6 us, 5.3 TB/s; 16 rows, gated, 4096 -> 2 x 12288 17.0 us, 5.9 TB/s) and a launch; 65 to
// 500 rows the way of X and W from the L2s into the compute units: 200 rows, 4096 -> 6144 12.3 us (14.3 with the matrix from memory), of which the matrix is 3.6 at the rate of a read and the
// products 5; each of 256 blocks brings 0.7 MB, and a block's way in and out is 2.3.  (In blocks of 128 x 64, of which there are 192, 12.9; without any loads but their
// issue those were 2.7 shorter, without those of X 2.7 more: four waves' loads of a kilobyte take the address unit 64 clocks.)  Loads one by one between the products
// of units of one step, whose pieces are half lines: 18.9 us for 16.6 (matrices from memory); between those of a unit's second step, whose operands are all in registers
// by then, not tried.
// 17 to 64 rows, with few columns: the blocks, of which there are as many as columns for all of K (2560 columns 160 of one column tile), leave compute units idle: 64 rows, 9728 -> 2560
// 13.3 us, the matrix 3.6.
// Blocks of one wave, which has all of K and adds nothing, for K up to 2048 (308 -> 4096, 735 rows 7.3 us; the best of four waves 10.8, tall 8.9): many lie on a compute unit,
// and K is over before four waves have shared it.
// Otherwise four waves a block: eight are slower, for all that they bring (16 rows, 12288 -> 4096 11.9 us for 11.6, 4096 -> 4096 6.4 for 6.1; 16 waves 11.8, 6.5), also
// where there are few blocks (16 rows, 12288 -> 256 8.9 for 8.5);
// so are units of one step of which two are under way (200 rows, 4096 -> 6144 19.6 for 17.2).
#include "gemm_q8.h"

// waits until at most N loads are under way (and for nothing else)
template <int N>
__device__ __forceinline__ void q8_wait_loads() {
    static_assert(N >= 0 && N <= 63, "the counter has six bits");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0f70);
    asm volatile("" ::: "memory");
}

// Two products of a row tile with two column tiles whose sums are held in accumulation registers: where a block's LDS leaves a SIMD one wave, the compiler
// keeps the sums there and moves every one of them to and fro (64 products, 192 moves).  It does not see matrix instructions here and leaves out the
// wait states behind an ordinary instruction that writes their operands, hence the first line, and those before the sums are read (the end of the loop).
__device__ __forceinline__ void q8_mfma2_held(q8_i32x4_t& a, q8_i32x4_t& b, q8_i32x4_t w0, q8_i32x4_t w1, q8_i32x4_t x) {
    asm volatile("s_nop 1\n\tv_mfma_i32_16x16x64_i8 %0, %2, %4, %0\n\tv_mfma_i32_16x16x64_i8 %1, %3, %4, %1" : "+a"(a), "+a"(b) : "v"(w0), "v"(w1), "v"(x));
}

__device__ __forceinline__ void q8_mfma_held(q8_i32x4_t& a, q8_i32x4_t w, q8_i32x4_t x) {
    asm volatile("s_nop 1\n\tv_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(a) : "v"(w), "v"(x));
}

// ONCE: W is read by one block only, and passes the caches by (up to 64 rows, matrices from memory: 16 rows, 4096 -> 2 x 12288 19.8 / 18.4 us).
template <int WAVES, int MT, int NT, int S, bool ONCE, int EPI, typename TC>
__device__ __forceinline__ void q8_staged_block(TC* C, const int8_t* X, const float* sx, const int8_t* W, const float* sw, int M, int N, int tiles, int chunks, int n_rows,
                                                int n_cols, const GateAct& act) {
    constexpr int PAIR = EPI == Q8_GATED ? 2 : 1, NO = NT / PAIR, PIECES = 4 * S, RPI = 16 / S;            // pieces of a row, rows that a load brings
    constexpr int D = 2, ITEMS = MT * NO, MOST = MT * S / PAIR, OPS = MT * S + NT * S;
    constexpr bool HELD = MT >= 6;
    static_assert((D - 1) * OPS <= 63, "a wait counts the loads issued after those that it waits for");
    // (arrays of their own: reads of one that the compiler cannot tell from another would wait for that one's loads)
    __shared__ __align__(1024) char stage0[WAVES * MT * S * 1024];
    __shared__ __align__(1024) char stage1[WAVES * MT * S * 1024];
    __shared__ float2 row_scales[MT * 16];
    __shared__ float col_scales[NT * 16];
    const int blocks = n_rows * n_cols, per = (blocks + Q8_DIES - 1) / Q8_DIES, idx = blockIdx.x / Q8_DIES;    // (a die takes a run of the blocks)
    const int v = (blockIdx.x % Q8_DIES) * per + idx;
    if (idx >= per || v >= blocks) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4, tid = threadIdx.x;
    int row_t, col_t;
    q8_block_at(v, n_rows, n_cols, 4, row_t, col_t);
    const int col0 = col_t * NO, row0 = row_t * MT * 16, rows = min(M - row0, MT * 16);
    constexpr int THREADS = WAVES * 64, SCALES = ((MT + NT) * 16 + THREADS - 1) / THREADS;
    float scale[SCALES];
#pragma unroll
    for (int q = 0; q < SCALES; ++q) {
        const int n = q * THREADS + tid - MT * 16;
        scale[q] = 0.f;
        if (n < 0) { if (n + MT * 16 < rows) scale[q] = sx[row0 + n + MT * 16]; }
        else if (n < NT * 16) {
            const int tile = col0 + n / 16 % NO;
            if (tile < tiles / PAIR) scale[q] = sw[(n / 16 / NO * (tiles / PAIR) + tile) * 16 + n % 16];
        }
    }
    const int w_bytes = tiles * chunks * 4096, pitch = chunks * Q8_CHUNK, n_units = chunks * 4 / S;
    const auto wres = __builtin_amdgcn_make_buffer_rsrc((void*)W, 0, w_bytes, 0x00020000);
    const auto xres = __builtin_amdgcn_make_buffer_rsrc((void*)(X + (size_t)row0 * pitch), 0, rows * pitch, 0x00020000);
    int w_at[NT], x_lane[S];
#pragma unroll
    for (int j = 0; j < NT; ++j) w_at[j] = min(col0 + j % NO, tiles / PAIR - 1) * 4096 + j / NO * (tiles / PAIR) * 4096;
#pragma unroll
    for (int q = 0; q < S; ++q) x_lane[q] = (q * RPI + lane / PIECES) * pitch + (lane % PIECES ^ (q * RPI + lane / PIECES) * S / 4) * 16;
    q8_i32x4_t acc[NT][MT], w[D][S][NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = q8_i32x4_t{0, 0, 0, 0};
    char* const mine[D] = {stage0 + wave * MT * S * 1024, stage1 + wave * MT * S * 1024};
    // A lane's own offset alone says whether a load lies in its buffer (the offset that all lanes share may not count): rows that do not exist, and whatever
    // belongs to a unit behind the end, lie beyond (2^30 is more than any block's rows, 2^31 more than any matrix)
    auto load = [&](int d, int unit) {
        const bool some = unit < n_units;
        const int wo = some ? (unit * S >> 2) * tiles * 4096 + (unit * S & 3) * 1024 : 0, xo = some ? unit * S * Q8_STEP : 0;
        const unsigned w_lane = some ? lane * 16 : 0x80000000u;
        const int x_skip = some ? 0 : 1 << 30;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int q = 0; q < S; ++q)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(xres, (__attribute__((address_space(3))) void*)(mine[d] + (i * S + q) * 1024), 16, x_lane[q] + (i * 16 * pitch + x_skip), xo, 0, 0);
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int j = 0; j < NT; ++j) w[d][s][j] = __builtin_bit_cast(q8_i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(wres, w_lane, w_at[j] + wo + s * 1024, ONCE ? 2 : 0));
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int d = 0; d < D; ++d) load(d, wave + d * WAVES);
    for (int u = wave; u < n_units; u += D * WAVES) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            // loads return in order: those of the D - 1 units behind this one may be under way
            __builtin_amdgcn_sched_barrier(0);
            q8_wait_loads<(D - 1) * OPS>();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < S; ++s) {
                q8_i32x4_t x[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) x[i] = *reinterpret_cast<const q8_i32x4_t*>(mine[d] + (i * 16 + r) * 64 * S + ((4 * s + g) ^ r * S / 4) * 16);
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; j += HELD ? 2 : 1) {
                        if constexpr (HELD && NT % 2) { if (j + 1 == NT) { q8_mfma_held(acc[j][i], w[d][s][j], x[i]); break; } }
                        if constexpr (HELD) q8_mfma2_held(acc[j][i], acc[j + 1][i], w[d][s][j], w[d][s][j + 1], x[i]);
                        else acc[j][i] = q8_mfma(w[d][s][j], x[i], acc[j][i]);
                    }
            }
            __builtin_amdgcn_sched_barrier(0);       // (the stage has been read: the products wait for the reads)
            load(d, u + (D + d) * WAVES);
        }
    }
#pragma unroll
    for (int q = 0; q < SCALES; ++q) {
        const int n = q * THREADS + tid - MT * 16;
        if (n < 0) row_scales[n + MT * 16] = q8_row_scale(scale[q]);
        else if (n < NT * 16) col_scales[n] = scale[q];
    }
    if constexpr (HELD) sums_settle(acc);
    // Nothing is under way into the stages when the sums go there, a wave's into the parts that it had to itself: tile t's at place t of the first, then of the
    // second, sum (row r, columns 4 g ..) at place r ^ (its lane in a row of readers) of the sixteen of g.  A row's results of a tile row are L readers' of V
    // neighbouring columns, so that a store is whole lines where the block has four column tiles (200 rows, 4096 -> 6144 15.5 us; tile by tile, 32 bytes of
    // a row, in two rounds of one stage: 16.7).
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    constexpr int V = NO == 1 ? 4 : 16 / (int)sizeof(TC), L = NO * 16 / V, TURN = 16 / L;
    static_assert(L * TURN <= 16 && ITEMS <= 2 * MOST, "readers of a row; tiles in two stages");
#pragma unroll
    for (int t = 0; t < ITEMS; ++t)
#pragma unroll
        for (int p = 0; p < PAIR; ++p)
            *reinterpret_cast<q8_i32x4_t*>(mine[t / MOST] + ((t % MOST * PAIR + p) * 64 + g * 16 + (r ^ (t % NO * 16 + 4 * g) / V * TURN)) * 16) = acc[p * NO + t % NO][t / NO];
    __syncthreads();
    // the sum of a row's places in the waves' parts, of column tile j from its column 4 q on
    auto from = [&](int row, int j, int q) {
        const int t = row / 16 * NO + j;
        return (t < MOST ? stage0 + t * PAIR * 1024 : stage1 + (t - MOST) * PAIR * 1024) + (q * 16 + (row % 16 ^ (j * 16 + 4 * q) / V * TURN)) * 16;
    };
    auto add = [&](const char* at, auto kind) {
        auto sum = *reinterpret_cast<const decltype(kind)*>(at);
#pragma unroll
        for (int o = 1; o < WAVES; ++o) sum += *reinterpret_cast<const decltype(kind)*>(at + o * MT * S * 1024);
        return sum;
    };
    const bool fours = N % 4 == 0 && (uintptr_t)C % (4 * sizeof(TC)) == 0, all = N % V == 0 && (uintptr_t)C % (V * sizeof(TC)) == 0;
    if (fours) {
#pragma unroll
        for (int u = 0; u < MT * 16 * L; u += WAVES * 64) {
            const int row = (u + tid) / L, c = (u + tid) % L, n = col0 * 16 + c * V;
            if (row >= rows) break;
            const char* const at = from(row, c * V / 16, c * V % 16 / 4);
            const float2 fx = row_scales[row];
            float y[V];
#pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                const q8_i32x4_t sum = add(at + h * 256, q8_i32x4_t{}), up = PAIR == 2 ? add(at + 1024 + h * 256, q8_i32x4_t{}) : sum;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[4 * h + e] = q8_value<EPI>(act, sum[e], up[e], fx, col_scales[c * V + 4 * h + e], col_scales[(NT - NO) * 16 + c * V + 4 * h + e]);
            }
            TC* const o = C + (size_t)(row0 + row) * N + n;
            if (V * sizeof(TC) == 16 && all) {
                if constexpr (V * sizeof(TC) == 16) if (n < N) q8_store_piece(o, y);
            } else
#pragma unroll
                for (int h = 0; h < V; h += 4)
                    if (n + h < N) Vec4<TC>::store(o + h, y + h);
        }
    } else {                                // a lane a column (200 rows, 2049 -> 4099 11.7 us; by readers of V columns, each stored by itself, 13.1)
#pragma unroll 4
        for (int u = tid; u < rows * NO * 16; u += WAVES * 64) {
            const int row = u / (NO * 16), c = u % (NO * 16), n = col0 * 16 + c;
            const char* const at = from(row, c / 16, c % 16 / 4) + c % 4 * 4;
            const int sum = add(at, 0), up = PAIR == 2 ? add(at + 1024, 0) : sum;
            if (n < N) C[(size_t)(row0 + row) * N + n] = from_f32<TC>(q8_value<EPI>(act, sum, up, row_scales[row], col_scales[c], col_scales[(NT - NO) * 16 + c]));
        }
    }
}

template <int WAVES, int MT, int NT, int S, bool ONCE, int EPI, typename TC>
__global__ __launch_bounds__(WAVES * 64, 2) void gemm_q8_kernel(TC* C, const int8_t* X, const float* sx, const int8_t* W, const float* sw, int M, int N,
                                                                    int tiles, int chunks, int n_rows, int n_cols, GateAct act) {
    q8_staged_block<WAVES, MT, NT, S, ONCE, EPI, TC>(C, X, sx, W, sw, M, N, tiles, chunks, n_rows, n_cols, act);
}

struct Q8Args {
    void* C; int c_dtype; const int8_t* X; const float* sx; const int8_t* W; const float* sw; int M, N, tiles, chunks, gated; GateAct act; hipStream_t st;
};

template <int MT, int NT, int S, int WAVES = 4>
static int split_launch(const Q8Args& a) {
    const int no = a.gated ? NT / 2 : NT, col_tiles = a.gated ? a.tiles / 2 : a.tiles;
    const int n_rows = (a.M + MT * 16 - 1) / (MT * 16), n_cols = (col_tiles + no - 1) / no;
    const int64_t blocks = (int64_t)n_rows * n_cols;
    SPY_REQUIRE((blocks + Q8_DIES) * WAVES * 64 < (1ll << 32), "spy_gemm_q8: %lld blocks are more than a launch holds", (long long)blocks);
    const unsigned grid = (unsigned)((blocks + Q8_DIES - 1) / Q8_DIES * Q8_DIES);
#define SPLIT_ARGS(TC) (TC*)a.C, a.X, a.sx, a.W, a.sw, a.M, a.N, a.tiles, a.chunks, n_rows, n_cols, a.act
#define SPLIT_BY(ONCE, EPI, TC) gemm_q8_kernel<WAVES, MT, NT, S, ONCE, EPI, TC><<<grid, WAVES * 64, 0, a.st>>>(SPLIT_ARGS(TC))
    // (more than four row tiles, or four column tiles, are for products of more rows)
#define SPLIT(EPI, TC) do { if (n_rows == 1 && MT <= 4 && NT <= 2) SPLIT_BY((MT <= 4 && NT <= 2), EPI, TC); else SPLIT_BY(false, EPI, TC); } while (0)
    if (a.gated) { if constexpr (NT % 2 == 0) SPLIT(Q8_GATED, bf16_t); else return spy_fail("spy_gemm_q8: a gated product by %d column tiles", NT); }
    else if (a.c_dtype == SPY_F32) SPLIT(Q8_STORE, float);
    else SPLIT(Q8_STORE, bf16_t);
#undef SPLIT
#undef SPLIT_BY
#undef SPLIT_ARGS
    SPY_CHECK_LAUNCH("spy_gemm_q8");
    return 0;
}

// Which blocks: those with the least estimated time, us, of c[0] + c[1] r k + c[2] r + c[3] b k + c[4] x, b the blocks over 256 compute units, r that rounded up,
// k the chunks of K; x: chunks of K that row tiles bring over the units, x k (tall blocks: b; blocks of one wave: k).  Fitted to 11000 products of 1 to 8192 rows, 16 to 24576
// columns and K of 16 to 17408, plain and gated, with ten matrices in turn, in every kind of block that might do (6 to 12 % rms, the short products' least exactly); what it
// takes is 0.7 % slower on average than the fastest kind, 5 % at the 95th percentile.  Most of those matrices fit the last cache, and no term has the bytes: where a matrix comes from
// memory the estimates are up to two fifths short (16 rows, gated, 4096 -> 2 x 12288 10.8 us, measured 17 to 18; 1 row, 17408 -> 17408 30, 57), and the
// choice is up to 6 % slower than the fastest kind (that row in blocks 201, 101 54 us; 64 rows, gated, 4096 -> 2 x 12288 in 404 27.1, 204 26.1).  (Without blocks of three column tiles and of five and seven row tiles 1.5 and 9 %
// from K = 512 on, with blocks of one column tile and two to four row tiles, of 2 x 6, 3 x 5 and 3 x 7 no better; without those of one wave 11 and 48 % up to there.)
// NT 100 + MT, 1000 more for one wave, or, tall, the row tiles alone.
struct Q8Cost { int plan; float c[5]; };
static const Q8Cost q8_costs[] = {
    {101, {2.66f, 0.0578f, 0.466f, 0.0347f, 0.f}}, {201, {2.78f, 0.0919f, 0.34f, 0.0535f, 0.f}}, {202, {2.84f, 0.11f, 0.473f, 0.0746f, 0.f}},
    {203, {2.88f, 0.139f, 0.668f, 0.0851f, 0.f}}, {204, {2.82f, 0.174f, 0.965f, 0.0928f, 0.f}}, {304, {3.26f, 0.212f, 1.14f, 0.115f, 0.f}},
    {306, {1.89f, 0.293f, 3.39f, 0.0819f, 0.00863f}}, {308, {1.79f, 0.36f, 4.27f, 0.0591f, 0.0123f}}, {404, {3.35f, 0.276f, 1.32f, 0.105f, 0.f}},
    {405, {1.69f, 0.33f, 3.68f, 0.132f, 0.f}}, {406, {1.67f, 0.332f, 3.94f, 0.165f, 0.f}}, {407, {1.68f, 0.38f, 4.49f, 0.129f, 0.00524f}},
    {408, {1.68f, 0.403f, 4.96f, 0.155f, 0.0032f}}, {1202, {2.94f, 0.0504f, 0.158f, 0.0781f, 0.281f}}, {1404, {3.88f, 0.f, 0.513f, 0.264f, 0.6f}},
    {8, {2.08f, 0.989f, 3.91f, 0.619f, 2.6f}}, {10, {1.92f, 1.17f, 5.07f, 0.667f, 2.73f}}, {12, {1.85f, 1.32f, 5.77f, 0.799f, 3.15f}},
    {14, {1.66f, 1.5f, 7.08f, 0.914f, 3.26f}}, {16, {1.43f, 1.74f, 7.64f, 0.978f, 3.84f}},
};

static int q8_plan(int M, int tiles, int chunks, int gated) {
    const int row_tiles = (M + 15) / 16, col_tiles = gated ? tiles / 2 : tiles;
    int best = 0;
    float least = INFINITY;
    for (const Q8Cost& p : q8_costs) {
        const bool tall = p.plan < 100, one = p.plan > 1000;
        const int MT = tall ? p.plan : p.plan % 100, NT = tall ? 16 : p.plan / 100 % 10, NO = gated ? NT / 2 : NT;
        // gate and up in pairs of column tiles; not many more row tiles than there are (four from 33 rows on, as many for more), tall blocks no more;
        // blocks of one wave, which has to walk all of K, up to K = 2048 (what was measured)
        if ((gated && NT % 2) || (one && chunks > 8) || (tall ? M < 16 * MT : MT == 4 ? row_tiles < 3 : row_tiles < MT)) continue;
        const int cols = (col_tiles + NO - 1) / NO;
        const float blocks = (float)((row_tiles + MT - 1) / MT) * (float)cols / 256.f, rounds = ceilf(blocks), k = (float)chunks;
        const float us = p.c[0] + p.c[1] * rounds * k + p.c[2] * rounds + p.c[3] * blocks * k + p.c[4] * (tall ? blocks : one ? k : (float)row_tiles * cols / 256.f * k);
        if (us < least) { least = us; best = p.plan; }
    }
    return best;
}

// C: bfloat16 or float32 [M, N].  X: rows of 256 bytes a chunk and their scales; W: the matrix laid out, `tiles` column tiles (gated:
// of both halves) and `chunks` of K, and its scales [16 tiles].  Gated: C is bfloat16 [M, N], N one half's columns.
// plan: 0, or the blocks by name (q8_costs).
extern "C" int spy_gemm_q8(void* C, int c_dtype, const void* X, const float* sx, const void* W, const float* sw, int M, int N, int tiles, int chunks,
                           int gated, int act_code, int plan, hipStream_t st) {
    GateAct act = {1.f, 0.f};
    SPY_REQUIRE(M > 0 && N > 0 && tiles > 0 && chunks > 0, "spy_gemm_q8: empty operand");
    SPY_REQUIRE(chunks <= 511 && (int64_t)tiles * chunks * 4096 < (1ll << 31), "spy_gemm_q8: a matrix of %d x %d tiles is too large", tiles, chunks);
    SPY_REQUIRE(gated ? tiles % 2 == 0 && N <= tiles * 8 && N > tiles * 8 - 16 : N <= tiles * 16 && N > tiles * 16 - 16, "spy_gemm_q8: %d columns in %d tiles", N, tiles);
    SPY_REQUIRE((((uintptr_t)X | (uintptr_t)W) % 16) == 0, "spy_gemm_q8: operands must be 16-byte aligned");
    SPY_REQUIRE(!gated || (gate_act_of(act_code, &act) && c_dtype == SPY_BF16), "spy_gemm_q8: activation %d, result dtype %d", act_code, c_dtype);
    const Q8Args a = {C, c_dtype, (const int8_t*)X, sx, (const int8_t*)W, sw, M, N, tiles, chunks, gated, act, st};
    if (!plan) plan = q8_plan(M, tiles, chunks, gated);
    if (plan >= 8 && plan <= 16) return q8_tall_launch(C, c_dtype, (const int8_t*)X, sx, (const int8_t*)W, sw, M, N, tiles, chunks, gated, act, plan, st);
    switch (plan) {
        case 101: return split_launch<1, 1, 4>(a);
        case 201: return split_launch<1, 2, 2>(a);
        case 202: return split_launch<2, 2, 2>(a);
        case 203: return split_launch<3, 2, 2>(a);
        case 204: return split_launch<4, 2, 2>(a);
        case 304: return split_launch<4, 3, 2>(a);
        case 306: return split_launch<6, 3, 2>(a);
        case 308: return split_launch<8, 3, 2>(a);
        case 404: return split_launch<4, 4, 2>(a);
        case 405: return split_launch<5, 4, 2>(a);
        case 406: return split_launch<6, 4, 2>(a);
        case 407: return split_launch<7, 4, 2>(a);
        case 408: return split_launch<8, 4, 2>(a);
        case 1202: return split_launch<2, 2, 2, 1>(a);
        case 1404: return split_launch<4, 4, 2, 1>(a);
    }
    return spy_fail("spy_gemm_q8: no blocks by the name of %d", plan);
}
