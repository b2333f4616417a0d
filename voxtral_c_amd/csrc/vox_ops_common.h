// vox_ops_common.h — what the operators on device memory (vox_ops.hip) share: element types, vector access, wave reductions.
#pragma once
#include "vox_common.h"

namespace vox {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// One rounding to the storage type, to nearest even (the compiler's own conversion: v_cvt_pk_bf16_f32 / v_cvt_f16_f32).
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

// N consecutive elements as f32 from an address that is aligned to N * sizeof(T) (at most 16 bytes per load).
template <typename T, int N> __device__ __forceinline__ void load_vec(float (&o)[N], const T *p) {
    typedef T vec __attribute__((ext_vector_type(N)));
    const vec v = *reinterpret_cast<const vec *>(p);
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = (float)v[i];
}

// glds16 (vox_common.h) from a wave-uniform address and a 32-bit offset per lane.
__device__ __forceinline__ void glds16_at(const void *base, unsigned offset, unsigned lds_base) {
    unsigned keep;
    const uint64_t b = (uint64_t)base;
    const uint64_t u = ((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(b >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)b);
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(offset), "s"(u), "s"(lds_base) : "memory");
}

__device__ __forceinline__ int wave_sum_i(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ unsigned wave_max_u(unsigned v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (unsigned)__shfl_xor((int)v, o, 64));
    return v;
}

}  // namespace vox
