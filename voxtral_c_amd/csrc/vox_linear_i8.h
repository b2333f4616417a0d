// vox_linear_i8.h — products in 8-bit integers: y = x_scale * w_scale * (xq . w), one scale per row of x and per output channel.
#pragma once
#include "vox_ops_common.h"

namespace vox {

// x / s rounded to the nearest whole number, ties to even, of the EXACT quotient.  q = rint(x * (1 / s)) is off by one at most, and only next
// to a border; r = x - q s is exact in f32 (it is a whole multiple of half an ulp of s and at most about s / 2 in size), so comparing 2 |r|
// with s settles it.  The exact form costs three instructions more and makes the 8-bit values the same on every implementation.
__device__ __forceinline__ float quant_i8(float x, float s, float inv) {
    const float q = rintf(x * inv);
    const float r = fmaf(-q, s, x), r2 = 2.f * fabsf(r);
    const bool odd = (int)q & 1;
    const bool fix = r2 > s || (r2 == s && odd);
    return fix ? q + copysignf(1.f, r) : q;
}
struct RowScale {
    float s, inv;
    bool broken;
};
// From the largest magnitude of a row, as the bits of |x| (NaN's are above infinity's).
__device__ __forceinline__ RowScale row_scale(unsigned amax_bits) {
    RowScale r;
    r.broken = amax_bits >= 0x7f800000u;
    r.s = fmaxf(__uint_as_float(r.broken ? 0u : amax_bits) / 127.f, 1.17549435e-38f);     // at least the smallest normal number
    r.inv = 1.f / r.s;
    return r;
}

// One workgroup per row: q [rows, ldq] (columns K .. ldq - 1 are zeros), scale [rows].  Bound by the row's two trips (the second one hits L2).
template <typename T> __global__ __launch_bounds__(256) void k_quant_rows_i8(const T *x, int64_t stride, int K, int ldq, int8_t *q, float *scale) {
    __shared__ unsigned red[4];
    const int64_t row = blockIdx.x;
    const T *xr = x + row * stride;
    int8_t *qr = q + row * ldq;
    unsigned m = 0;
    for (int k = threadIdx.x; k < K; k += 256) m = max(m, __float_as_uint((float)xr[k]) & 0x7fffffffu);
    m = wave_max_u(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    const RowScale r = row_scale(max(max(red[0], red[1]), max(red[2], red[3])));
    for (int k = threadIdx.x; k < ldq; k += 256) qr[k] = k < K && !r.broken ? (int8_t)quant_i8((float)xr[k], r.s, r.inv) : (int8_t)0;
    if (threadIdx.x == 0) scale[row] = r.broken ? NAN : r.s;
}

struct LinearI8Args {
    const int8_t *xq;            // [M, ldq], zeros behind K
    const float *xs;             // [M]
    const int8_t *w;
    int64_t w_stride;
    const float *ws;
    const void *bias;
    void *y;
    int64_t y_stride;
    int M, K, N, ldq;
};
// Three roundings of f32 (the sum's conversion and two products) and the one to the output's type; the sum itself is exact.
template <typename T> __device__ __forceinline__ T i8_out(int acc, float xs, float ws, const T *bias, int n) {
    float v = ((float)acc * ws) * xs;
    if (bias) v += (float)bias[n];
    return from_f32<T>(v);
}

// Any K, stride and alignment: 64 x 64 outputs per workgroup, slices of 64 bytes of K through LDS byte by byte, v_dot4 products.
template <typename T> __global__ __launch_bounds__(256) void k_linear_i8_bytes(LinearI8Args a) {
    __shared__ int xs[64][17], ws[64][17];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += 64) {
        for (int i = tid; i < 64 * 64; i += 256) {
            const int r = i >> 6, c = i & 63;
            reinterpret_cast<int8_t *>(&xs[r][0])[c] = m0 + r < a.M && k0 + c < a.ldq ? a.xq[(int64_t)(m0 + r) * a.ldq + k0 + c] : (int8_t)0;
            reinterpret_cast<int8_t *>(&ws[r][0])[c] = n0 + r < a.N && k0 + c < a.K ? a.w[(int64_t)(n0 + r) * a.w_stride + k0 + c] : (int8_t)0;
        }
        __syncthreads();
        for (int kk = 0; kk < 16; kk++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __builtin_amdgcn_sdot4(xs[ty * 4 + i][kk], ws[tx * 4 + j][kk], acc[i][j], false);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int m = m0 + ty * 4 + i, n = n0 + tx * 4 + j;
            if (m < a.M && n < a.N) ((T *)a.y)[m * a.y_stride + n] = i8_out<T>(acc[i][j], a.xs[m], a.ws[n], (const T *)a.bias, n);
        }
}

}  // namespace vox
