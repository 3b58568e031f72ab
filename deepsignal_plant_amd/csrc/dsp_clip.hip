// dsp_clip.hip -- the global norm of many gradients, and clipping by it (torch.nn.utils.clip_grad_norm_ as train.py:75-119
// uses it, with 0.5).
//
//   norm = sqrt(sum over all tensors and values of g^2)        k = min(1, max_norm / (norm + 1e-6))        out = k g
//
// Bound by memory: everything is read for the norm, and read again and written for the product.  Launches are few however
// many tensors there are: up to 128 of them are described in a launch's own arguments (4 KB) (no table to copy: the call can be
// captured), and a workgroup finds its tensor by bisection.  Squares and sums are held in 64 bits (no gradient overflows
// them, and the order of summation cannot be seen in the 32 bits of the answer); the product is rounded once.  (268,435,456 bf16 in 290
// tensors into fp32: 148 us for the squares = 3.6 TB/s, 371 for the product = 4.3 TB/s; the second reading in reverse or past the caches gains 2 %.)
#include "dsp_ops.h"

using namespace dsp;

namespace {

constexpr int kTensors = 128;
struct Table {
    const void* in[kTensors];
    void* out[kTensors];
    i64 n[kTensors];
    uint32_t first[kTensors + 1];   // first workgroup of a tensor
    uint8_t in_type[kTensors], out_type[kTensors];
    int count;
};
struct Clip { double sum, k; };   // what the launches hand on

__device__ __forceinline__ int tensor_of(const Table& t, uint32_t block) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= block) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// A tensor is taken as accesses of VEC values at addresses that are multiples of their size, `shift` values before its first;
// those at its ends value by value.  f(values, first of them, how many are inside)
template <class T, int VEC, class F> __device__ __forceinline__ void for_accesses(const T* x, i64 n, int shift, i64 from, i64 to, F f) {
    typedef Vec<T, VEC> V;
    for (i64 j = from + threadIdx.x; j < to; j += 4 * 256) {
        V v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const i64 at = (j + u * 256) * VEC - shift;
            if (j + u * 256 >= to) continue;
            if (at >= 0 && at + VEC <= n) v[u] = *(const V*)(x + at);
            else
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[u].v[e] = at + e >= 0 && at + e < n ? x[at + e] : T{};
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (j + u * 256 < to) f(v[u], (j + u * 256) * VEC - shift);
    }
}

template <class T> __device__ __forceinline__ double squares(const void* x, i64 n, i64 block, i64 chunk) {
    constexpr int VEC = 16 / sizeof(T);
    const int shift = (int)((size_t)x % 16 / sizeof(T));
    const i64 all = (n + shift + VEC - 1) / VEC, from = block * chunk, to = from + chunk < all ? from + chunk : all;
    double s = 0;
    for_accesses<T, VEC>((const T*)x, n, shift, from, to, [&](const Vec<T, VEC>& v, i64) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const double y = to_f32(v.v[e]);
            s = fma(y, y, s);
        }
    });
    return s;
}

__device__ __forceinline__ double block_sum(double s, double* scratch) {
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0;
    for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += scratch[i];
    return s;
}

__global__ __launch_bounds__(256) void clip_squares_kernel(Table t, i64 chunk, double* __restrict__ part) {
    __shared__ double scratch[4];
    const int i = tensor_of(t, blockIdx.x);
    const i64 block = blockIdx.x - t.first[i];
    double s;
    if (t.in_type[i] == DSP_FT_F32) s = squares<float>(t.in[i], t.n[i], block, chunk);
    else if (t.in_type[i] == DSP_FT_BF16) s = squares<__bf16>(t.in[i], t.n[i], block, chunk);
    else s = squares<_Float16>(t.in[i], t.n[i], block, chunk);
    s = block_sum(s, scratch);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ __launch_bounds__(1024) void clip_norm_kernel(i64 parts, const double* __restrict__ part, double max_norm, Clip* __restrict__ c,
                                                        float* __restrict__ norm) {
    __shared__ double scratch[16];
    double s = 0;
#pragma unroll 4
    for (i64 i = threadIdx.x; i < parts; i += 1024) s += part[i];
    s = block_sum(s, scratch);
    if (threadIdx.x) return;
    const double root = sqrt(s), k = max_norm / (root + 1e-6);
    c->k = k >= 1.0 ? 1.0 : k;   // NaN stays NaN: gradients that have no norm are not passed off as clipped ones
    *norm = (float)root;
}

template <class T, class O> __device__ __forceinline__ void scale(const void* in, void* out, i64 n, i64 block, i64 chunk, double k) {
    constexpr int VEC = 16 / sizeof(T);
    const int shift = (int)((size_t)in % 16 / sizeof(T));
    const i64 all = (n + shift + VEC - 1) / VEC, from = block * chunk, to = from + chunk < all ? from + chunk : all;
    // wide stores where input and output begin at the same place within 16 bytes
    const bool wide = ((size_t)out / sizeof(O) - (size_t)in / sizeof(T)) % (16 / sizeof(O) < VEC ? 16 / sizeof(O) : VEC) == 0;
    O* o = (O*)out;
    for_accesses<T, VEC>((const T*)in, n, shift, from, to, [&](const Vec<T, VEC>& v, i64 at) {
        constexpr int W = 16 / sizeof(O) < VEC ? 16 / sizeof(O) : VEC;   // values of one store
        O y[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) y[e] = from_f32<O>((float)(to_f32(v.v[e]) * k));
        if (wide && at >= 0 && at + VEC <= n) {
#pragma unroll
            for (int e = 0; e < VEC; e += W) {
                Vec<O, W> z;
#pragma unroll
                for (int i = 0; i < W; ++i) z.v[i] = y[e + i];
                *(Vec<O, W>*)(o + at + e) = z;
            }
        } else
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (at + e >= 0 && at + e < n) o[at + e] = y[e];
    });
}

__global__ __launch_bounds__(256) void clip_scale_kernel(Table t, i64 chunk, const Clip* __restrict__ c) {
    const double k = c->k;
    const int i = tensor_of(t, blockIdx.x);
    if (k == 1.0 && t.in[i] == t.out[i]) return;   // in place and nothing to clip
    const i64 block = blockIdx.x - t.first[i];
    const int a = t.in_type[i], b = t.out_type[i];
    if (a == DSP_FT_F32) scale<float, float>(t.in[i], t.out[i], t.n[i], block, chunk, k);
    else if (a == DSP_FT_BF16 && b == DSP_FT_BF16) scale<__bf16, __bf16>(t.in[i], t.out[i], t.n[i], block, chunk, k);
    else if (a == DSP_FT_BF16) scale<__bf16, float>(t.in[i], t.out[i], t.n[i], block, chunk, k);
    else if (b == DSP_FT_F16) scale<_Float16, _Float16>(t.in[i], t.out[i], t.n[i], block, chunk, k);
    else scale<_Float16, float>(t.in[i], t.out[i], t.n[i], block, chunk, k);
}

int size_of(int type) { return type == DSP_FT_F32 ? 4 : 2; }
bool known(int type) { return type == DSP_FT_F32 || type == DSP_FT_BF16 || type == DSP_FT_F16; }

// 16-byte accesses of one workgroup: about 16,384 workgroups in all, at least 1,024 accesses (16 KB) each.  (540 MB of bf16: 154 us for the
// squares and 377 for the product, 184 and 422 with 2,048 workgroups, which have too little under way.)
i64 chunk_of(i64 bytes) {
    const i64 c = cdiv(cdiv(bytes, 16), 16384);
    return c < 1024 ? 1024 : cdiv(c, 1024) * 1024;
}
i64 blocks_of(const void* x, i64 n, int type, i64 chunk) {
    const int vec = 16 / size_of(type);
    return cdiv(cdiv(n + (i64)((size_t)x % 16 / size_of(type)), vec), chunk);
}

}  // namespace

extern "C" {

int64_t dsp_clip_workspace(int32_t n_tensors, const int64_t* numels) {
    if (n_tensors < 0 || (n_tensors && !numels)) return refuse("dsp_clip_workspace", "bad argument");
    // as many workgroups as there could be: every tensor one more for its rest and one for its shift
    int64_t parts = 2ll * n_tensors + 32768;
    return 256 + parts * (int64_t)sizeof(double);
}

int32_t dsp_clip_grad_norm(void* stream, int32_t n_tensors, const void* const* grads, const int64_t* numels, const int32_t* dtypes, void* const* outs,
                           const int32_t* out_dtypes, double max_norm, float* norm, void* workspace, int64_t workspace_bytes) {
    const char* who = "dsp_clip_grad_norm";
    if (n_tensors < 0 || (n_tensors && (!grads || !numels || !dtypes)) || !norm || !workspace) return refuse(who, "NULL pointer or negative count");
    if (outs && !out_dtypes) return refuse(who, "outputs need their types");
    if (outs && !(max_norm >= 0)) return refuse(who, "max_norm must not be negative");
    if ((size_t)workspace & 255) return refuse(who, "the workspace must be aligned to 256 bytes");
    i64 bytes = 0;
    for (int i = 0; i < n_tensors; ++i) {
        if (numels[i] < 0) return refuse(who, "negative size");
        if (!known(dtypes[i]) || (outs && !known(out_dtypes[i]))) return refuse(who, "unknown element type");
        if (numels[i] && (!grads[i] || (outs && !outs[i]))) return refuse(who, "NULL tensor");
        if ((size_t)grads[i] % size_of(dtypes[i]) || (outs && (size_t)outs[i] % size_of(out_dtypes[i]))) return refuse(who, "a tensor is not aligned to its element type");
        if (outs && out_dtypes[i] != dtypes[i] && out_dtypes[i] != DSP_FT_F32) return refuse(who, "an output has its gradient's type or float32");
        bytes += numels[i] * size_of(dtypes[i]);
    }
    const i64 chunk = chunk_of(bytes);
    if (workspace_bytes < dsp_clip_workspace(n_tensors, numels)) return refuse(who, "workspace too small (dsp_clip_workspace)");
    Clip* c = (Clip*)workspace;
    double* part = (double*)((char*)workspace + 256);
    hipStream_t s = (hipStream_t)stream;
    i64 parts = 0;
    for (int step = 0; step < (outs ? 2 : 1); ++step) {
        Table t;
        t.count = 0;
        uint32_t blocks = 0;
        for (int i = 0; i <= n_tensors; ++i) {
            if (t.count && (i == n_tensors || t.count == kTensors)) {
                t.first[t.count] = blocks;
                if (step == 0) hipLaunchKernelGGL(clip_squares_kernel, dim3(blocks), dim3(256), 0, s, t, chunk, part + parts);
                else hipLaunchKernelGGL(clip_scale_kernel, dim3(blocks), dim3(256), 0, s, t, chunk, (const Clip*)c);
                parts += step == 0 ? blocks : 0;
                t.count = 0;
                blocks = 0;
            }
            if (i == n_tensors || numels[i] == 0) continue;
            const int k = t.count++;
            t.in[k] = grads[i];
            t.out[k] = outs ? outs[i] : nullptr;
            t.n[k] = numels[i];
            t.in_type[k] = (uint8_t)dtypes[i];
            t.out_type[k] = (uint8_t)(outs ? out_dtypes[i] : dtypes[i]);
            t.first[k] = blocks;
            blocks += (uint32_t)blocks_of(grads[i], numels[i], dtypes[i], chunk);
        }
        if (step == 0) hipLaunchKernelGGL(clip_norm_kernel, dim3(1), dim3(1024), 0, s, parts, part, max_norm, c, norm);
    }
    return launched(who);
}

}  // extern "C"
