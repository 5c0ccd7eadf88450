// Rows brought to 8-bit integers with a scale for each row, and the RMS norm that hands its rows over so.
//
// z = a row's values (the norm: s * w, s the stream with the addend, the factor 1 / rms left out: it is positive and common to the row, so it
// does not enter the integers), a = max |z|:  q = 127 z / a rounded half to even, scale = a / 127 (the norm: a / (127 rms)).
// The quotient is formed in 64 bits, so that a row's integers are the same however and wherever it is computed: products of two float32 are
// exact there, and the maximum is one of them.
// A row of zeros: q 0, scale 0.  A row with a NaN or an infinity: q 0, scale NaN, so that all that is made of it is NaN.
#include "q8.h"

__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    const int nw = (blockDim.x + 63) >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.;
    for (int i = 0; i < nw; ++i) t += red[i];
    return t;
}
// the largest of the values' magnitudes as bits: a NaN is above an infinity, which is above all numbers
__device__ __forceinline__ unsigned long long block_max_bits(unsigned long long v, unsigned long long* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned long long)__shfl_xor(v, o, 64));
    const int nw = (blockDim.x + 63) >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned long long t = red[0];
    for (int i = 1; i < nw; ++i) t = max(t, red[i]);
    return t;
}
__device__ __forceinline__ unsigned long long magnitude_bits(double z) { return (unsigned long long)__double_as_longlong(z) & 0x7fffffffffffffffull; }

// One block a row.  NORM: x is the residual stream (float32, written with the addend), delta the addend (or null) and weight the norm's; else x are
// the rows, ldx apart.
template <typename TX, typename TD, typename TW, bool NORM>
__global__ __launch_bounds__(256) void rows_q8_kernel(int8_t* __restrict__ q, float* __restrict__ scales, TX* x, int64_t ldx, const TD* __restrict__ delta,
                                                      const TW* __restrict__ weight, float eps, int H, int64_t pitch) {
    __shared__ double red_sum[4];
    __shared__ unsigned long long red_max[4];
    const size_t row = blockIdx.x;
    TX* s = x + row * ldx;
    double ss = 0.;
    unsigned long long top = 0;
    for (int i = threadIdx.x; i < H; i += 256) {
        float v = to_f32<TX>(s[i]);
        double z = v;
        if (NORM) {
            if (delta) { v += to_f32<TD>(delta[row * H + i]); s[i] = from_f32<TX>(v); }
            ss = fma((double)v, (double)v, ss);
            z = (double)v * (double)to_f32<TW>(weight[i]);
        }
        top = max(top, magnitude_bits(z));
    }
    top = block_max_bits(top, red_max);
    const double a = __longlong_as_double((long long)top);
    double scale = a / 127.0;
    if (NORM) scale /= sqrt(block_sum_f64(ss, red_sum) / (double)H + (double)eps);
    const bool some = a > 0. && a < INFINITY;
    if (threadIdx.x == 0) scales[row] = a < INFINITY ? (a > 0. ? (float)scale : 0.f) : NAN;
    for (int i = threadIdx.x; i < H; i += 256) {
        double z = to_f32<TX>(s[i]);              // (this thread wrote it above)
        if (NORM) z *= (double)to_f32<TW>(weight[i]);
        q[row * pitch + i] = some ? (int8_t)(int)rint(z * 127.0 / a) : (int8_t)0;
    }
}

extern "C" int spy_add_rmsnorm_q8(void* q, float* scales, float* stream, const void* delta, int delta_dtype, const void* weight, int weight_dtype, float eps,
                                  int T, int H, int64_t pitch, hipStream_t st) {
    SPY_REQUIRE(T > 0 && H > 0 && pitch >= H, "spy_add_rmsnorm_q8: bad sizes %d x %d", T, H);
    SPY_DISPATCH(delta_dtype, TD, SPY_DISPATCH(weight_dtype, TW, rows_q8_kernel<float, TD, TW, true><<<T, 256, 0, st>>>(
        (int8_t*)q, scales, stream, (int64_t)H, (const TD*)delta, (const TW*)weight, eps, H, pitch)));
    SPY_CHECK_LAUNCH("spy_add_rmsnorm_q8");
    return 0;
}

extern "C" int spy_quantize_rows(void* q, float* scales, const void* x, int x_dtype, int64_t ldx, int T, int H, int64_t pitch, hipStream_t st) {
    SPY_REQUIRE(T > 0 && H > 0 && pitch >= H && ldx >= H, "spy_quantize_rows: bad sizes %d x %d", T, H);
    SPY_DISPATCH(x_dtype, TX, rows_q8_kernel<TX, float, float, false><<<T, 256, 0, st>>>((int8_t*)q, scales, (TX*)x, ldx, nullptr, nullptr, 0.f, H, pitch));
    SPY_CHECK_LAUNCH("spy_quantize_rows");
    return 0;
}
