// vox_linear_i8.h — products in 8-bit integers: y = x_scale * w_scale * (xq . w), one scale per row of x and per output channel.
#pragma once
#include <type_traits>
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

// One workgroup per row: q [rows, ldq] (columns K .. ldq - 1 are zeros), scale [rows].  Bound by the row's two trips (the second one hits the
// caches; keeping the row in registers instead measured the same) and, for few rows, by their latency: as many threads as give each one load, up to 1024
// (25 x 5120 bf16: 3.9 us, with 256 threads 5.2).  4099 x 1280 bf16: 6.8 us on its own, 8.6 - 10 between products, for 15.7 MB.  N elements per load: K, stride and x allow it, and ldq % N = 0.
constexpr int I8_QUANT_THREADS = 1024;
template <typename T, int N> __global__ __launch_bounds__(I8_QUANT_THREADS) void k_quant_rows_i8(const T *x, int64_t stride, int K, int ldq, int8_t *q, float *scale) {
    __shared__ unsigned red[I8_QUANT_THREADS / 64];
    const int64_t row = blockIdx.x;
    const int threads = blockDim.x;
    const T *xr = x + row * stride;
    int8_t *qr = q + row * ldq;
    unsigned m = 0;
    for (int k = threadIdx.x * N; k < K; k += threads * N) {
        float v[N];
        load_vec<T, N>(v, xr + k);
#pragma unroll
        for (int i = 0; i < N; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    m = wave_max_u(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = red[0];
    for (int w = 1; w < threads >> 6; w++) m = max(m, red[w]);
    const RowScale r = row_scale(m);
    for (int k = threadIdx.x * N; k < ldq; k += threads * N) {
        typedef int8_t out __attribute__((ext_vector_type(N)));
        float v[N] = {};
        out o;
        if (k < K && !r.broken) load_vec<T, N>(v, xr + k);
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = (int8_t)(int)quant_i8(v[i], r.s, r.inv);
        *reinterpret_cast<out *>(qr + k) = o;
    }
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
    int *part;                   // [splits, padded rows, padded channels]: sums of a part of K each, where K is split
    int splits;
};
// Three roundings of f32 (the sum's conversion and two products) and the one to the output's type; the sum itself is exact.  Where the first product
// leaves f32's range the row's scale, which may be as small as 2^-126, goes first: if both orders overflow, so does the result.  The sum is at most 2^31:
// no weight scale up to I8_SAFE does that, and `LARGE` may be false.
constexpr float I8_SAFE = 0x1p96f;
template <bool LARGE = true> __device__ __forceinline__ float i8_scaled(int acc, float xs, float ws) {
    const float v = (float)acc, p = v * ws;
    return LARGE && __builtin_isinf(p) ? v * xs * ws : p * xs;
}
template <typename T> __device__ __forceinline__ T i8_out(int acc, float xs, float ws, const T *bias, int n) {
    float v = i8_scaled(acc, xs, ws);
    if (bias) v += (float)bias[n];
    return from_f32<T>(v);
}

// Any K, stride and alignment: 64 x 64 outputs per workgroup, slices of 64 bytes of K through LDS byte by byte, v_dot4 products.  Bound by the byte loads:
// 25 x 1283 x 6144 takes 123 us (K 1280: 9), 400 rows 153 (17).  It is there so that every layout is answered; a weight matrix laid out once can have
// rows of whole 16 bytes.
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


// ---- few rows: a read of the weights --------------------------------------------------------------------------------------------
// A workgroup makes 16 output channels of MT x 16 rows; its waves split K and their whole-number sums are added through LDS (exact in any order).
// v_mfma_i32_16x16x64_i8 with the weights as A operand: lane = (channel lane % 16, 16 bytes of K), loaded straight from the row-major matrix, 64 bytes of
// each of 16 rows per instruction and two neighbouring instructions per 128-byte line.  25 x 5120 x 1280: 8.6 us, 0.8 TB/s of weights (80 workgroups; operands
// four steps ahead changed nothing), 11.7 us a call with the quantiser's launch.
constexpr int I8_ROWS_WAVES = 8;
template <typename T, int MT> __global__ __launch_bounds__(64 * I8_ROWS_WAVES) void k_linear_i8_rows(LinearI8Args a) {
    __shared__ i32x4 part[I8_ROWS_WAVES][MT][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n16 = lane & 15, c = lane >> 4;
    static_assert(MT * 256 <= 64 * I8_ROWS_WAVES, "");
    const int n0 = blockIdx.x * 16;
    const int8_t *w = a.w + (int64_t)min(n0 + n16, a.N - 1) * a.w_stride + c * 16;
    const int8_t *x[MT];
#pragma unroll
    for (int t = 0; t < MT; t++) x[t] = a.xq + (int64_t)min(t * 16 + n16, a.M - 1) * a.ldq + c * 16;
    // this thread's output, its scales requested in front of the products
    const int ch = tid & 15, row = tid >> 4, n = n0 + ch;    // (the workgroup has a thread per output or more)
    const bool mine = tid < MT * 256 && row < a.M && n < a.N;
    const float out_xs = mine ? a.xs[row] : 0.f, out_ws = mine ? a.ws[n] : 0.f, out_bias = mine && a.bias ? (float)((const T *)a.bias)[n] : 0.f;
    i32x4 acc[MT] = {};
    for (int k = wave * 128; k < a.K; k += 128 * I8_ROWS_WAVES) {
        // (xq holds zeros from K to ldq, a multiple of 128: what stands in for weights behind K does not matter, so it is the row's first bytes)
        const i32x4 w0 = *reinterpret_cast<const i32x4 *>(w + (k + c * 16 < a.K ? k : -c * 16));
        const i32x4 w1 = *reinterpret_cast<const i32x4 *>(w + (k + 64 + c * 16 < a.K ? k + 64 : -c * 16));
#pragma unroll
        for (int t = 0; t < MT; t++) {
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, *reinterpret_cast<const i32x4 *>(x[t] + k), acc[t], 0, 0, 0);
            acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, *reinterpret_cast<const i32x4 *>(x[t] + k + 64), acc[t], 0, 0, 0);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; t++) part[wave][t][lane] = acc[t];
    __syncthreads();
    if (!mine) return;
    // channel ch of row: element (ch % 4) of lane (ch / 4) * 16 + row % 16
    int sum = 0;
#pragma unroll
    for (int v = 0; v < I8_ROWS_WAVES; v++) sum += reinterpret_cast<const int *>(&part[v][row >> 4][(ch >> 2) * 16 + (row & 15)])[ch & 3];
    ((T *)a.y)[row * a.y_stride + n] = from_f32<T>(i8_scaled(sum, out_xs, out_ws) + out_bias);
}

// The same in one launch for a few rows (single tokens): every workgroup quantises all of x into its LDS while its first weights are on their way.  Up
// to I8_FEW elements of x: 32 per thread, about a microsecond; a launch of its own costs 3 us (1 x 1280 x 6144,
// f32: 13.9 -> 10.9 us a call then; now 6.5 with weights from memory, 1.2 TB/s, and 5.8 with the same ones again and again).
constexpr int I8_FEW = 16384, I8_FEW_ROWS = 16, I8_FEW_AHEAD = 2;
template <typename T, int N> __global__ __launch_bounds__(64 * I8_ROWS_WAVES) void k_linear_i8_few(LinearI8Args a, const T *x, int64_t x_stride) {
    __shared__ i32x4 part[I8_ROWS_WAVES][64];
    __shared__ float xs[I8_FEW_ROWS];
    extern __shared__ __attribute__((aligned(128))) char lds[];                  // xq [M][ldq + 16]: rows start on different banks
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n16 = lane & 15, c = lane >> 4;
    const int n0 = blockIdx.x * 16, ld = a.ldq + 16;
    const int8_t *w = a.w + (int64_t)min(n0 + n16, a.N - 1) * a.w_stride + c * 16;
    auto weights = [&](int k) { return *reinterpret_cast<const i32x4 *>(w + (k + c * 16 < a.K ? k : -c * 16)); };       // (see above)
    const int ch = tid & 15, out_row = tid >> 4, n = n0 + ch;          // this thread's output, its scale requested here
    const bool mine = tid < 256 && out_row < a.M && n < a.N;
    const float out_ws = mine ? a.ws[n] : 0.f, out_bias = mine && a.bias ? (float)((const T *)a.bias)[n] : 0.f;
    i32x4 ahead[I8_FEW_AHEAD][2];
#pragma unroll
    for (int i = 0; i < I8_FEW_AHEAD; i++) {
        const int k = (wave + i * I8_ROWS_WAVES) * 128;
        if (k < a.K) { ahead[i][0] = weights(k); ahead[i][1] = weights(k + 64); }
    }
    for (int row = wave; row < a.M; row += I8_ROWS_WAVES) {
        const T *xr = x + row * x_stride;
        unsigned m = 0;
        for (int k = lane * N; k < a.K; k += 64 * N) {
            float v[N];
            load_vec<T, N>(v, xr + k);
#pragma unroll
            for (int i = 0; i < N; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        }
        const RowScale r = row_scale(wave_max_u(m));
        for (int k = lane * N; k < a.ldq; k += 64 * N) {
            typedef int8_t out __attribute__((ext_vector_type(N)));
            float v[N] = {};
            out o;
            if (k < a.K && !r.broken) load_vec<T, N>(v, xr + k);
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = (int8_t)(int)quant_i8(v[i], r.s, r.inv);
            *reinterpret_cast<out *>(lds + row * ld + k) = o;
        }
        if (lane == 0) xs[row] = r.broken ? NAN : r.s;
    }
    __syncthreads();
    const char *xq = lds + min(n16, a.M - 1) * ld + c * 16;
    i32x4 acc = {};
    auto step = [&](int k, i32x4 w0, i32x4 w1) {
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, *reinterpret_cast<const i32x4 *>(xq + k), acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, *reinterpret_cast<const i32x4 *>(xq + k + 64), acc, 0, 0, 0);
    };
#pragma unroll
    for (int i = 0; i < I8_FEW_AHEAD; i++) {
        const int k = (wave + i * I8_ROWS_WAVES) * 128;
        if (k < a.K) step(k, ahead[i][0], ahead[i][1]);
    }
    for (int k = (wave + I8_FEW_AHEAD * I8_ROWS_WAVES) * 128; k < a.K; k += 128 * I8_ROWS_WAVES) step(k, weights(k), weights(k + 64));
    part[wave][lane] = acc;
    __syncthreads();
    if (!mine) return;
    int sum = 0;
#pragma unroll
    for (int v = 0; v < I8_ROWS_WAVES; v++) sum += reinterpret_cast<const int *>(&part[v][(ch >> 2) * 16 + out_row])[ch & 3];
    ((T *)a.y)[out_row * a.y_stride + n] = from_f32<T>(i8_scaled(sum, xs[out_row], out_ws) + out_bias);
}

// ---- many rows: a matrix product ------------------------------------------------------------------------------------------------
// BM rows x 128 channels per workgroup of four waves (2 x 2, each BM / 2 rows x 64 channels) on v_mfma_i32_32x32x32_i8.  Slices of 128 bytes of K
// go from memory into LDS without registers (global_load_lds_dwordx4: a wave's instruction brings 128 bytes of each of 8 rows), STAGES of them in
// flight with one barrier per slice.  16-byte pieces of a row are stored at (piece ^ (row / 2 % 8)): of the MFMA operand reads (lane = row, one
// piece) 16 lanes at a time then touch every one of the 64 banks once (with row % 8 the counters show a conflict on every second cycle).  Outputs leave through LDS so that rows are written in whole lines.
// 4099 x 1280 x 10240 bf16: 82 - 86 us, 1.3 POP/s (31 % of the pipe's cycles; 84 MB of the output alone take 18 us; 96 in a run of
// 60 under the profiler); 8192^3: 1.6 POP/s.  What bounds it is neither LDS nor
// the depth of the pipeline: 256 x 128 tiles with slices of 64 bytes, three stages and a quarter less traffic per product took 107 us where these took 103,
// 256 x 128 with three stages and one workgroup per CU 119.
constexpr int I8_BN = 128, I8_BK = 128;
__device__ __forceinline__ int i8_swizzle(int row) { return (row >> 1) & 7; }
template <typename T, int BM, int STAGES> constexpr unsigned i8_tile_lds() {        // stages, later outputs; scales and bias behind them
    const unsigned stages = STAGES * (BM + I8_BN) * I8_BK, out = BM * (I8_BN * (unsigned)sizeof(T) + 16);
    return (stages > out ? stages : out) + (BM + 2 * I8_BN) * 4;
}
template <typename T, int BM, int STAGES> __global__ __launch_bounds__(256) void k_linear_i8_tile(LinearI8Args a, int tiles_m, int tiles_n) {
    typedef int i32x16 __attribute__((ext_vector_type(16)));
    constexpr int ROWS = BM + I8_BN, STAGE = ROWS * I8_BK, LOADS = ROWS / 32;      // LOADS: instructions per wave and slice
    constexpr int MI = BM / 64, NJ = 2;                                            // 32 x 32 blocks of a wave: rows, channels
    extern __shared__ __attribute__((aligned(128))) char lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
    // Each XCD (workgroup number mod 8) works through a range of tiles of its own in which the channels change fastest within bands of an
    // eighth of all channels: its L2 keeps the band's weights, and a row panel is read once per band.
    const int total = tiles_m * tiles_n * a.splits, per = (total + 7) / 8, all = (blockIdx.x & 7) * per + (blockIdx.x >> 3), split = all % a.splits, id = all / a.splits;
    if ((int)(blockIdx.x >> 3) >= per || all >= total) return;
    const int band_n = (tiles_n + 7) / 8, band = id / (tiles_m * band_n), in = id - band * tiles_m * band_n;
    const int width = min(band_n, tiles_n - band * band_n), tm = in / width, tn = band * band_n + in - tm * width;
    const int m0 = tm * BM, n0 = tn * I8_BN;

    // this lane's pieces: rows of x first, then rows of w; pieces behind K are the row's first one (x holds zeros there)
    const int piece = lane & 7;
    const int8_t *src[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const int row = (i * 4 + wave) * 8 + (lane >> 3), p = piece ^ i8_swizzle(row);
        src[i] = i * 32 >= BM ? a.w + (int64_t)min(n0 + row - BM, a.N - 1) * a.w_stride + p * 16 : a.xq + (int64_t)min(m0 + row, a.M - 1) * a.ldq + p * 16;
    }
    const int slices = a.ldq / I8_BK, s_begin = split * slices / a.splits, s_end = (split + 1) * slices / a.splits;
    // loads [from, to) of slice s
    auto issue = [&](int s, int from, int to) {
        const unsigned base = lds_addr(lds) + (s % STAGES) * STAGE;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            if (i < from || i >= to) continue;
            const int row = (i * 4 + wave) * 8 + (lane >> 3), p = (piece ^ i8_swizzle(row)) * 16;
            const bool past = i * 32 >= BM && s * I8_BK + p >= a.K;
            glds16(src[i] + (past ? -p : s * I8_BK), __builtin_amdgcn_readfirstlane(base + (i * 4 + wave) * 1024));
        }
    };
    i32x16 acc[NJ][MI] = {};
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++)
        if (s_begin + s < s_end) issue(s_begin + s, 0, LOADS);
    // scales and bias of the tile, f32 (read one by one behind the loop, they cost four times what the products do)
    float *sw = reinterpret_cast<float *>(lds + i8_tile_lds<T, BM, STAGES>()) - BM - 2 * I8_BN, *sb = sw + I8_BN, *sx = sb + I8_BN;
    if (tid < I8_BN) {
        const int n = min(n0 + tid, a.N - 1);
        sw[tid] = a.ws[n];
        sb[tid] = a.bias ? (float)((const T *)a.bias)[n] : 0.f;
    }
    for (int i = tid; i < BM; i += 256) sx[i] = a.xs[min(m0 + i, a.M - 1)];
    for (int s = s_begin; s < s_end; s++) {
        // slice s has landed when at most the younger slices' loads are in flight; behind the barrier everyone's has, and everyone is done with the
        // slice that the next loads overwrite
        // (this wave's own LDS reads of that slice have returned too: the compiler may place the products that use them behind the barrier)
        if (STAGES == 3 && s + 1 < s_end) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        // The operands of step k + 1 are read, and a quarter of the next loads requested, in front of step k's products.
        const char *buf = lds + (s % STAGES) * STAGE;
        const bool more = s + STAGES - 1 < s_end;
        i32x4 wf[2][NJ], xf[2][MI];
        auto read = [&](int k) {
            const int q = k * 2 + (lane >> 5);
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                const int row = BM + wn * 64 + j * 32 + (lane & 31);
                wf[k & 1][j] = *reinterpret_cast<const i32x4 *>(buf + row * I8_BK + ((q ^ i8_swizzle(row)) << 4));
            }
#pragma unroll
            for (int i = 0; i < MI; i++) {
                const int row = wm * (BM / 2) + i * 32 + (lane & 31);
                xf[k & 1][i] = *reinterpret_cast<const i32x4 *>(buf + row * I8_BK + ((q ^ i8_swizzle(row)) << 4));
            }
        };
        read(0);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            if (k < 3) read(k + 1);
            if (more) issue(s + STAGES - 1, k * LOADS / 4, (k + 1) * LOADS / 4);
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int i = 0; i < MI; i++) acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[k & 1][j], xf[k & 1][i], acc[j][i], 0, 0, 0);
        }
    }
    if (a.splits > 1) {
        const int64_t ld = (int64_t)tiles_n * I8_BN;
        int *part = a.part + ((int64_t)split * tiles_m * BM + m0) * ld + n0;
#pragma unroll
        for (int i = 0; i < MI; i++)
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const int row = wm * (BM / 2) + i * 32 + (lane & 31), ch = wn * 64 + j * 32 + g * 8 + (lane >> 5) * 4;
                    const i32x4 v = {acc[j][i][g * 4], acc[j][i][g * 4 + 1], acc[j][i][g * 4 + 2], acc[j][i][g * 4 + 3]};
                    *reinterpret_cast<i32x4 *>(part + row * ld + ch) = v;
                }
        return;
    }
    __syncthreads();
    // lane: row lane % 32 of a block, channels 8 g + 4 (lane / 32) + 0..3 in registers 4 g + 0..3
    constexpr int LD = I8_BN + 16 / sizeof(T);
    T *out = reinterpret_cast<T *>(lds);
    auto scale = [&](auto is_large) {                        // (the question asked for each output costs 4 % of the kernel's time)
        constexpr bool large = decltype(is_large)::value;
#pragma unroll
        for (int i = 0; i < MI; i++) {
            const int row = wm * (BM / 2) + i * 32 + (lane & 31);
            const float xs = sx[row];
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    typedef T out4 __attribute__((ext_vector_type(4)));
                    const int ch = wn * 64 + j * 32 + g * 8 + (lane >> 5) * 4;
                    const f32x4 ws = *reinterpret_cast<const f32x4 *>(sw + ch), bias = *reinterpret_cast<const f32x4 *>(sb + ch);
                    out4 v;
#pragma unroll
                    for (int r = 0; r < 4; r++) v[r] = from_f32<T>(i8_scaled<large>(acc[j][i][g * 4 + r], xs, ws[r]) + bias[r]);
                    *reinterpret_cast<out4 *>(out + row * LD + ch) = v;
                }
        }
    };
    if (__any(!(fabsf(sw[wn * 64 + lane]) <= I8_SAFE))) scale(std::true_type{});      // (the wave's 64 channels)
    else scale(std::false_type{});
    __syncthreads();
    const int rows = min(BM, a.M - m0), cols = min(I8_BN, a.N - n0);
    T *y = (T *)a.y + m0 * a.y_stride + n0;
    constexpr int V = 16 / sizeof(T);
    if (cols == I8_BN && ((reinterpret_cast<uintptr_t>(y) | (uintptr_t)(a.y_stride * sizeof(T))) & 15) == 0) {
        for (int i = tid; i < rows * (I8_BN / V); i += 256) {
            const int row = i / (I8_BN / V), ch = (i - row * (I8_BN / V)) * V;
            *reinterpret_cast<uint4 *>(y + row * a.y_stride + ch) = *reinterpret_cast<const uint4 *>(out + row * LD + ch);
        }
    } else {
        for (int i = tid; i < rows * I8_BN; i += 256) {
            const int row = i / I8_BN, ch = i - row * I8_BN;
            if (ch < cols) y[row * a.y_stride + ch] = out[row * LD + ch];
        }
    }
}


// Adds the parts (whole numbers: exact in any order) and scales: four channels per thread.  Bound by the launch (the parts are a few MB in the caches).
template <typename T> __global__ __launch_bounds__(256) void k_linear_i8_join(LinearI8Args a, int64_t ld, int64_t step) {
    const int groups = (a.N + 3) / 4;
    const int64_t total = (int64_t)a.M * groups;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / groups;
        const int n = (int)(i - m * groups) * 4;
        i32x4 sum = *reinterpret_cast<const i32x4 *>(a.part + m * ld + n);
        for (int s = 1; s < a.splits; s++) sum += *reinterpret_cast<const i32x4 *>(a.part + s * step + m * ld + n);
        const float xs = a.xs[m];
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (n + r < a.N) ((T *)a.y)[m * a.y_stride + n + r] = i8_out<T>(sum[r], xs, a.ws[n + r], (const T *)a.bias, n + r);
    }
}

}  // namespace vox
