// Rows brought to 8-bit integers with a scale for each row, and the RMS norm that hands its rows over so.
//
// z = a row's values (the norm: s * w, s the stream with the addend, the factor 1 / rms left out: it is positive and common to the row, so it
// does not enter the integers), a = max |z|:  q = 127 z / a rounded half to even, scale = a / 127 (the norm: a / (127 rms)).
// The quotient is formed in 64 bits, so that a row's integers are the same however and wherever it is computed: products of two float32 are
// exact there, and the maximum is one of them.
// A row of zeros: q 0, scale 0.  A row with a NaN or an infinity: q 0, scale NaN, so that all that is made of it is NaN.
//
// (The norm of zeros with eps 0 is no number, and its scale NaN.)
//
// Bound by memory: a block takes a row, reads it once, holds it in registers while the maximum (and the sum of squares) goes round, and writes it.
// 8192 x 4096 with a bfloat16 addend 66 us, 5.4 TB/s; rows of 2047 x 12288 bfloat16 16.2 (20.9 from memory).  Rows that a width or a place keeps from pieces of eight are bound by their
// narrow loads and stores: 2962 x 5667 bfloat16, a value a load and a byte a store, 30 us (10 at the rate of a copy), norms of 4096 x 1001 and 1000 17.7 and 12.6 (9).
#include "q8.h"
#include <type_traits>

// The bits of a value's magnitude: a NaN is above an infinity, which is above all numbers.
__device__ __forceinline__ unsigned long long magnitude(double z) { return (unsigned long long)__double_as_longlong(z) & 0x7fffffffffffffffull; }
__device__ __forceinline__ unsigned magnitude(float z) { return __float_as_uint(z) & 0x7fffffffu; }
__device__ __forceinline__ double value_of(unsigned long long m) { return __longlong_as_double((long long)m); }
__device__ __forceinline__ double value_of(unsigned m) { return (double)__uint_as_float(m); }

// A row's largest magnitude and its sum, over a block; every thread gets them.
template <int WAVES, bool SUM, typename BITS>
__device__ __forceinline__ void row_statistics(BITS& top, double& ss) {
    __shared__ BITS tops[WAVES];
    __shared__ double sums[WAVES];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        top = max(top, (BITS)__shfl_xor(top, o, 64));
        if (SUM) ss += __shfl_xor(ss, o, 64);
    }
    if (WAVES == 1) return;
    if ((threadIdx.x & 63) == 0) { tops[threadIdx.x >> 6] = top; if (SUM) sums[threadIdx.x >> 6] = ss; }
    __syncthreads();
    top = tops[0];
    if (SUM) ss = sums[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) { top = max(top, tops[i]); if (SUM) ss += sums[i]; }
}

// 127 z / a rounded half to even, z = x or x w.  In 32 bits the quotient is off by up to 4 2^-24 of 127 (the product, a, 127 / a and theirs), less than 2^-15; adding
// 1.5 2^23 leaves its nearest integer in the low bits, and only where what that leaves out is half an integer, but for 2^-15, is the quotient itself formed, in 64 bits (one value
// of 16 000, and ties).  Rows whose largest value is very large or small, for which 127 / a has no 32 bits, go by that altogether (inv NaN); rows
// whose integers are all 0 have inv 0.
template <bool NORM>
__device__ __forceinline__ int quotient(float x, float w, float inv, double a) {
    const float u = (NORM ? x * w : x) * inv, t = u + 12582912.f;
    if (__builtin_expect(!(fabsf(u - (t - 12582912.f)) <= 0.5f - 0x1p-15f), 0)) return (int)rint((NORM ? (double)x * (double)w : (double)x) * 127.0 / a);
    return (int)__float_as_uint(t);
}
__device__ __forceinline__ float inverse(double a) { return !(a < INFINITY) || a == 0. ? 0.f : a > 0x1p-90 && a < 0x1p120 ? 127.f / (float)a : NAN; }

// A row's scale from its largest magnitude and, for the norm, its sum of squares.
template <bool NORM>
__device__ __forceinline__ float row_scale(double a, double ss, float eps, int H) {
    if (!(a < INFINITY)) return NAN;
    return (float)(a / (NORM ? 127.0 * sqrt(ss / (double)H + (double)eps) : 127.0));
}

// VEC values of a row in one or two pieces, which are aligned so (VEC 8: 16 bytes each; 4: 16 or 8; 2: 8 or 4), or one value.
template <int VEC, typename T>
__device__ __forceinline__ void load_values(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) v[0] = to_f32<T>(*p);
    else if constexpr (VEC == 2 && sizeof(T) == 4) { const float2 t = *reinterpret_cast<const float2*>(p); v[0] = t.x; v[1] = t.y; }
    else if constexpr (VEC == 2) { const uint32_t t = *reinterpret_cast<const uint32_t*>(p); v[0] = __uint_as_float(t << 16); v[1] = __uint_as_float(t & 0xffff0000u); }
    else if constexpr (VEC == 4) Vec4<T>::load(p, v);
    else if constexpr (sizeof(T) == 4) { Vec4<float>::load(p, v); Vec4<float>::load(p + 4, v + 4); }
    else {
        const uint4 t = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[2 * e] = __uint_as_float(w[e] << 16); v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u); }
    }
}
// the stream's new values, and a row's integers
template <int VEC>
__device__ __forceinline__ void store_stream(float* p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) *p = v[0];
    else if constexpr (VEC == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    else {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) Vec4<float>::store(p + e, v + e);
    }
}
template <int VEC>
__device__ __forceinline__ void store_integers(int8_t* o, const int (&n)[VEC]) {
    if constexpr (VEC == 1) *o = (int8_t)n[0];
    else if constexpr (VEC == 2) *reinterpret_cast<uint16_t*>(o) = (uint16_t)((n[0] & 255) | (n[1] & 255) << 8);
    else {
        uint32_t b[VEC / 4];
#pragma unroll
        for (int h = 0; h < VEC / 4; ++h) b[h] = (n[4 * h] & 255) | (n[4 * h + 1] & 255) << 8 | (n[4 * h + 2] & 255) << 16 | (uint32_t)n[4 * h + 3] << 24;
        if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(o) = b[0];
        else *reinterpret_cast<uint2*>(o) = uint2{b[0], b[1]};
    }
}

// One block a row, held in registers: NP pieces of VEC values a thread.  NORM: x is the residual stream (float32, written with the addend), delta the
// addend (or null) and weight the norm's; else x are the rows, ldx apart.
template <typename TX, typename TD, typename TW, bool NORM, int VEC, int THREADS, int NP>
__global__ __launch_bounds__(THREADS) void rows_q8_kernel(int8_t* __restrict__ q, float* __restrict__ scales, TX* __restrict__ x, int64_t ldx, const TD* __restrict__ delta,
                                                          const TW* __restrict__ weight, float eps, int H, int64_t pitch) {
    const size_t row = blockIdx.x;
    TX* s = x + row * ldx;
    float v[NP][VEC], w[NP][VEC];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int i = (p * THREADS + threadIdx.x) * VEC;
        if (i < H) {
            load_values<VEC, TX>(s + i, v[p]);
            if (NORM) load_values<VEC, TW>(weight + i, w[p]);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[p][e] = w[p][e] = 0.f;
        }
    }
    if (NORM && delta) {
        float d[NP][VEC];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int i = (p * THREADS + threadIdx.x) * VEC;
            if (i < H) load_values<VEC, TD>(delta + row * H + i, d[p]);
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int i = (p * THREADS + threadIdx.x) * VEC;
            if (i < H) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[p][e] += d[p][e];
                store_stream<VEC>((float*)s + i, v[p]);
            }
        }
    }
    double ss = 0.;
    typename std::conditional<NORM, unsigned long long, unsigned>::type top = 0;
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            if constexpr (NORM) {
                const double z = (double)v[p][e];
                ss = fma(z, z, ss);
                top = max(top, magnitude(z * (double)w[p][e]));
            } else top = max(top, magnitude(v[p][e]));
        }
    row_statistics<THREADS / 64, NORM>(top, ss);
    const double a = value_of(top);
    const float inv = inverse(a);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const int i = (p * THREADS + threadIdx.x) * VEC;
        if (i >= H) continue;
        int n[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) n[e] = inv == 0.f ? 0 : quotient<NORM>(v[p][e], w[p][e], inv, a);
        store_integers<VEC>(q + row * pitch + i, n);
    }
    if (threadIdx.x == 0) scales[row] = row_scale<NORM>(a, ss, eps, H);
}

// The same for rows wider than a block's registers: read twice.
template <typename TX, typename TD, typename TW, bool NORM>
__global__ __launch_bounds__(1024) void wide_rows_q8_kernel(int8_t* __restrict__ q, float* __restrict__ scales, TX* x, int64_t ldx, const TD* __restrict__ delta,
                                                            const TW* __restrict__ weight, float eps, int H, int64_t pitch) {
    const size_t row = blockIdx.x;
    TX* s = x + row * ldx;
    double ss = 0.;
    typename std::conditional<NORM, unsigned long long, unsigned>::type top = 0;
    for (int i = threadIdx.x; i < H; i += 1024) {
        float v = to_f32<TX>(s[i]);
        if (NORM && delta) { v += to_f32<TD>(delta[row * H + i]); s[i] = from_f32<TX>(v); }
        if constexpr (NORM) {
            ss = fma((double)v, (double)v, ss);
            top = max(top, magnitude((double)v * (double)to_f32<TW>(weight[i])));
        } else top = max(top, magnitude(v));
    }
    row_statistics<16, NORM>(top, ss);
    const double a = value_of(top);
    const float inv = inverse(a);
    for (int i = threadIdx.x; i < H; i += 1024)                // (what a thread reads of the stream, it wrote itself)
        q[row * pitch + i] = inv == 0.f ? (int8_t)0 : (int8_t)quotient<NORM>(to_f32<TX>(s[i]), NORM ? to_f32<TW>(weight[i]) : 1.f, inv, a);
    if (threadIdx.x == 0) scales[row] = row_scale<NORM>(a, ss, eps, H);
}

template <typename TX, typename TD, typename TW, bool NORM>
static void rows_launch(int8_t* q, float* scales, TX* x, int64_t ldx, const TD* delta, const TW* weight, float eps, int T, int H, int64_t pitch, hipStream_t st) {
#define ROWS(VEC, THREADS, NP) rows_q8_kernel<TX, TD, TW, NORM, VEC, THREADS, NP><<<T, THREADS, 0, st>>>(q, scales, x, ldx, delta, weight, eps, H, pitch)
    // pieces of eight values where every row begins at a multiple of 16 bytes, of four or two where it begins at one of theirs
    const uintptr_t ends = (uintptr_t)x | (uintptr_t)delta | (uintptr_t)weight;
    const bool few = T <= 512;               // (as many threads as pieces; for more rows that is slower: a norm of 600 x 8192 21.3 us for 18.5)
    if (H % 8 == 0 && ldx % 8 == 0 && ends % 16 == 0 && H <= (NORM ? 16384 : 32768)) {
        if (H <= 512) ROWS(8, 64, 1);
        else if (H <= 2048) ROWS(8, 256, 1);
        else if (H <= 4096) ROWS(8, 512, 1);             // (256 threads with two pieces: a norm of 4096 x 4096 40.7 us for 36.9)
        else if (H <= 8192 && few) ROWS(8, 1024, 1);
        else if (H <= 6144) ROWS(8, 256, 3);
        else if (H <= 8192) ROWS(8, 512, 2);
        else if (H <= 16384 && few) ROWS(8, 1024, 2);
        else if (H <= 12288) ROWS(8, 512, 3);
        else if (H <= 16384) ROWS(8, 512, 4);
        else if constexpr (!NORM) { if (H <= 24576) ROWS(8, 1024, 3); else ROWS(8, 1024, 4); }       // (a norm's registers would not do)
    } else if (H % 4 == 0 && ldx % 4 == 0 && ends % 16 == 0 && H <= 16384) {
        if (H <= 1024) ROWS(4, 256, 1);
        else if (H <= 2048) ROWS(4, 256, 2);
        else if (H <= 4096) { if (few) ROWS(4, 1024, 1); else ROWS(4, 256, 4); }
        else if (H <= 8192) ROWS(4, 1024, 2);
        else ROWS(4, 1024, 4);
    } else if (H % 2 == 0 && ldx % 2 == 0 && ends % 8 == 0 && H <= 16384) {
        if (H <= 512) ROWS(2, 256, 1);
        else if (H <= 2048) ROWS(2, 256, 4);
        else if (H <= 4096) { if (few) ROWS(2, 1024, 2); else ROWS(2, 256, 8); }
        else ROWS(2, 1024, 8);
    }
    else if (H <= 256) ROWS(1, 256, 1);
    else if (H <= 1024) ROWS(1, 256, 4);
    else if (H <= 2048) ROWS(1, 256, 8);
    else if (H <= 4096) { if (few) ROWS(1, 1024, 4); else ROWS(1, 256, 16); }
    else if (H <= 8192) ROWS(1, 1024, 8);
    else if (H <= 16384) ROWS(1, 1024, 16);
    else wide_rows_q8_kernel<TX, TD, TW, NORM><<<T, 1024, 0, st>>>(q, scales, x, ldx, delta, weight, eps, H, pitch);
#undef ROWS
}

// rows in one launch: one of 2^32 threads or more is none
#define ROWS_AT_ONCE (1 << 21)

extern "C" int spy_add_rmsnorm_q8(void* q, float* scales, float* stream, const void* delta, int delta_dtype, const void* weight, int weight_dtype, float eps,
                                  int T, int H, int64_t pitch, hipStream_t st) {
    SPY_REQUIRE(T > 0 && H > 0 && pitch >= H && pitch % 16 == 0 && (uintptr_t)q % 16 == 0, "spy_add_rmsnorm_q8: bad sizes %d x %d", T, H);
    for (int64_t t = 0; t < T; t += ROWS_AT_ONCE) {
        const int n = (int)min((int64_t)ROWS_AT_ONCE, T - t);
        SPY_DISPATCH(delta_dtype, TD, SPY_DISPATCH(weight_dtype, TW, rows_launch<float, TD, TW, true>(
            (int8_t*)q + t * pitch, scales + t, stream + t * H, (int64_t)H, delta ? (const TD*)delta + t * H : nullptr, (const TW*)weight, eps, n, H, pitch, st)));
    }
    SPY_CHECK_LAUNCH("spy_add_rmsnorm_q8");
    return 0;
}

extern "C" int spy_quantize_rows(void* q, float* scales, const void* x, int x_dtype, int64_t ldx, int T, int H, int64_t pitch, hipStream_t st) {
    SPY_REQUIRE(T > 0 && H > 0 && pitch >= H && pitch % 16 == 0 && (uintptr_t)q % 16 == 0 && ldx >= H, "spy_quantize_rows: bad sizes %d x %d", T, H);
    for (int64_t t = 0; t < T; t += ROWS_AT_ONCE) {
        const int n = (int)min((int64_t)ROWS_AT_ONCE, T - t);
        SPY_DISPATCH(x_dtype, TX, rows_launch<TX, float, float, false>((int8_t*)q + t * pitch, scales + t, (TX*)x + t * ldx, ldx, nullptr, nullptr, 0.f, n, H, pitch, st));
    }
    SPY_CHECK_LAUNCH("spy_quantize_rows");
    return 0;
}
