// dsp_ops.h -- what the kernels of a training step share (dsp_embed.hip, dsp_loss.hip, dsp_clip.hip, dsp_lstm_train.hip):
// element types, wide loads and stores, wave reductions, launch checks.
#ifndef DSP_OPS_H
#define DSP_OPS_H

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "dsp_amd.h"

extern "C" void dsp_set_error_(const char* msg);

namespace dsp {

typedef long long i64;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// N values of T as one memory access of N * sizeof(T) bytes
template <class T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };

// Every value is widened to 32 bits when it is read and rounded once, to nearest even, when it is written.
template <class T> __device__ __forceinline__ float to_f32(T x) { return (float)x; }
template <class T> __device__ __forceinline__ T from_f32(float x) { return (T)x; }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
template <class T> __device__ __forceinline__ T wave_sum(T x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

inline int refuse(const char* who, const char* what) {
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", who, what);
    dsp_set_error_(buf);
    return DSP_EINVAL;
}
// status of the launches made since the last check
inline int launched(const char* who) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return DSP_OK;
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: %s", who, hipGetErrorString(e));
    dsp_set_error_(buf);
    return DSP_EHIP;
}

// A launch of any number of workgroups (of at most 1,024 threads): a grid has fewer than 2^32 threads along each of its axes, so many
// workgroups go along two.  The last row of them may be surplus.
inline dim3 grid_of(long long blocks) {
    const long long x = blocks < (1 << 21) ? blocks : 1 << 21;
    return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
__device__ __forceinline__ i64 block_at() { return (i64)blockIdx.y * gridDim.x + blockIdx.x; }

inline i64 cdiv(i64 a, i64 b) { return (a + b - 1) / b; }
inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
// largest power of two of at most 16 bytes that divides `bytes` and every address given
inline int wide_bytes(size_t bytes, const void* a, const void* b) {
    const size_t all = bytes | (size_t)a | (size_t)b | 16;
    return (int)(all & (~all + 1));
}

}  // namespace dsp

#endif
