// dsp_loss.hip -- weighted softmax cross entropy of a batch and its gradient (the loss of train.py:75-119:
// torch.nn.CrossEntropyLoss with a weight for each class).
//
//   l_n = w[y_n] (log sum_c exp x_nc - x_n,y_n)     loss = sum l_n / sum w[y_n]  (mean)  or  sum l_n  (sum)  or  l (none)
//   dx_nc = k_n (softmax(x_n)_c - [c = y_n]),       k_n = w[y_n] / sum w[y_m]  (mean)    or  w[y_n]
//
// Bound by memory: every logit is read once and every gradient written once; an exponential per logit is far below what the
// arithmetic could do meanwhile.  So a row is read into registers (it comes with its maximum and, of the values less the
// maximum, its sum), and its gradient is written from there at once, for an upstream gradient of 1; where the backward pass
// finds another one it computes the gradient from the logits again, so every gradient is rounded once.  Rows that do not
// fit a workgroup's registers are read twice, the second time from the caches.
// Rows whose label is ignore_index count for nothing and get a gradient of zeros, whatever they hold.  A label outside the
// classes makes its row's loss and gradient NaN.  Sums over rows are held in 64 bits, in an order that the sizes decide.
#include "dsp_ops.h"

using namespace dsp;

namespace {

struct Loss {   // what every kernel here is given
    const void* logits;      // [n][c], rows `stride` values apart
    const void* labels;
    const float* weight;     // [c] or NULL
    void* grad;              // [n][c] or NULL
    float* loss;             // [1], or [n] where reduction is none
    float2* stat;            // [n]: a row's maximum m and sum of exp(x - m)
    double* den;             // sum of the weights of all labels (mean)
    double2* part;           // per workgroup: sum of the rows' losses, sum of their weights
    const float* upstream;   // gradient of the loss: [1], or [n] where reduction is none
    i64 n, c, stride, ignore;
    int label_dtype, reduction, parts, skip_unit;
    double* weight_part;     // [weight_parts]: sums of labels' weights;  weight_parts 0: den holds their sum, if it is wanted
    int weight_parts;
    bool wide;               // 16 bytes of a gradient can be written where 16 bytes of logits are read
};

enum { kMean = DSP_REDUCE_MEAN, kSum = DSP_REDUCE_SUM, kNone = DSP_REDUCE_NONE };

__device__ __forceinline__ i64 label_at(const Loss& p, i64 r) {
    if (p.label_dtype == DSP_DT_I64) return ((const int64_t*)p.labels)[r];
    if (p.label_dtype == DSP_DT_I32) return ((const int32_t*)p.labels)[r];
    return ((const uint8_t*)p.labels)[r];
}
// weight of a row: 0 where it is ignored, NaN where its label is no class
__device__ __forceinline__ float weight_of(const Loss& p, i64 y) {
    if (y == p.ignore) return 0.0f;
    if (y < 0 || y >= p.c) return __builtin_nanf("");
    return p.weight ? p.weight[y] : 1.0f;
}
// The gradient comes from the maximum and the sum, not from their log sum exp: rounded to 32 bits that would shift every
// probability of a row by up to |lse| 2^-24.
// e^x as 2^(x log2 e), one hardware instruction: within 2 ulp of itself plus the rounding of the argument, |x| 2^-24
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }

// log sum exp of a row less its own class's logit: the difference of the logits first, where they are close it is exact
__device__ __forceinline__ float loss_of(float m, float z, float x) { return (m - x) + logf(z); }

// sum over the block's threads (a multiple of 64, at most 1,024), in every thread
template <class T> __device__ __forceinline__ T block_sum(T x, T* scratch) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    T s = scratch[0];
    for (int i = 1; i < (int)(blockDim.x >> 6); ++i) s += scratch[i];
    return s;
}
__device__ __forceinline__ float block_max(float x, float* scratch) {
    x = wave_max(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
    __syncthreads();
    float s = scratch[0];
    for (int i = 1; i < (int)(blockDim.x >> 6); ++i) s = fmaxf(s, scratch[i]);
    return s;
}

// the gradient's factor of a row; den: the sum of the labels' weights
__device__ __forceinline__ float factor_of(const Loss& p, float w, double den, i64 r) {
    double k = w;
    if (p.reduction == kMean) k /= den;
    if (p.upstream) k *= p.upstream[p.reduction == kNone ? r : 0];
    return (float)k;
}

// sum of the weights of all labels, where rows' gradients are to be written before all rows have been seen: at most kWeightParts
// sums, which every workgroup of the rows' launch adds for itself
constexpr int kWeightParts = 64;
__global__ __launch_bounds__(1024) void loss_weights_kernel(Loss p) {
    __shared__ double scratch[16];
    double s = 0;
#pragma unroll 4
    for (i64 r = (i64)blockIdx.x * 1024 + threadIdx.x; r < p.n; r += (i64)gridDim.x * 1024) s += weight_of(p, label_at(p, r));
    s = block_sum(s, scratch);
    if (threadIdx.x == 0) p.weight_part[blockIdx.x] = s;
}
// in every thread of a wave
__device__ __forceinline__ double weights_of(const Loss& p) {
    if (p.weight_parts == 0) return p.den ? *p.den : 1.0;
    return wave_sum((int)(threadIdx.x & 63) < p.weight_parts ? p.weight_part[threadIdx.x & 63] : 0.0);
}
// Many sums are joined by as many workgroups as fill the device, whose own sums another launch joins: one workgroup would need
// a microsecond for every few thousand
constexpr int kJoinParts = 256;
__global__ __launch_bounds__(1024) void loss_join_parts_kernel(Loss p, double2* __restrict__ out) {
    __shared__ double scratch[16];
    double a = 0, b = 0;
#pragma unroll 4
    for (i64 i = (i64)blockIdx.x * 1024 + threadIdx.x; i < p.parts; i += kJoinParts * 1024) {
        a += p.part[i].x;
        b += p.part[i].y;
    }
    a = block_sum(a, scratch);
    b = block_sum(b, scratch);
    if (threadIdx.x == 0) out[blockIdx.x] = make_double2(a, b);
}
__global__ __launch_bounds__(1024) void loss_join_kernel(Loss p) {
    __shared__ double scratch[16];
    double a = 0, b = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < p.parts; i += 1024) {
        a += p.part[i].x;
        b += p.part[i].y;
    }
    a = block_sum(a, scratch);
    b = p.weight_parts ? weights_of(p) : block_sum(b, scratch);   // what the gradients were made with
    if (threadIdx.x) return;
    if (p.reduction == kMean) *p.den = b;
    *p.loss = (float)(p.reduction == kMean ? a / b : a);
}

// ---- few classes: a group of lanes (a power of two, at most 64) per row, E values a lane -----------------------------------
// ONE: a single workgroup takes all rows, and the sums need no other launch (512 rows of 2 classes: 7 us in all, the loss, its gradient and what
// checks the upstream one).  Else labels, logits, what is kept of a row and its loss are all that is moved: 2^24 rows of 2 bf16 in 124 us.
template <class T, int E, bool BACKWARD, bool ONE>
__global__ __launch_bounds__(ONE ? 1024 : 256) void loss_few_kernel(Loss p, int log_lanes) {
    __shared__ double scratch[16];
    const int lanes = 1 << log_lanes, lane = threadIdx.x & (lanes - 1);
    const i64 groups = blockDim.x >> log_lanes;
    double num = 0, den = 0, all = 0;
    if (BACKWARD && p.skip_unit && p.reduction != kNone && *p.upstream == 1.0f) return;   // what the forward left is the gradient
    if (ONE) {
        for (i64 r = threadIdx.x; r < p.n; r += blockDim.x) all += weight_of(p, label_at(p, r));
        all = block_sum(all, scratch);
    } else if (p.grad)
        all = weights_of(p);
    for (i64 r = block_at() * groups + (threadIdx.x >> log_lanes); r < p.n; r += ONE ? groups : p.n) {
        const i64 y = label_at(p, r);
        const float w = weight_of(p, y);
        const T* row = (const T*)p.logits + r * p.stride;
        float x[E], m = -__builtin_inff(), z = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c = lane + (e << log_lanes);
            x[e] = c < p.c ? to_f32(row[c]) : -__builtin_inff();
            m = fmaxf(m, x[e]);
        }
        if (BACKWARD) {
            m = p.stat[r].x;
            z = p.stat[r].y;
        } else {
            for (int o = lanes >> 1; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
#pragma unroll
            for (int e = 0; e < E; ++e) z += lane + (e << log_lanes) < p.c ? fast_exp(x[e] - m) : 0.0f;
            for (int o = lanes >> 1; o; o >>= 1) z += __shfl_xor(z, o);
        }
        if (!BACKWARD && lane == 0) {
            p.stat[r] = make_float2(m, z);
            const float l = y != p.ignore ? w * loss_of(m, z, y >= 0 && y < p.c ? to_f32(row[y]) : 0.0f) : 0.0f;
            if (p.reduction == kNone) p.loss[r] = l;
            num += l;
            den += w;
        }
        if (p.grad) {
            const float k = factor_of(p, w, all, r), inv = 1.0f / z;
            T* out = (T*)p.grad + r * p.c;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int c = lane + (e << log_lanes);
                if (c < p.c) out[c] = from_f32<T>(y == p.ignore ? 0.0f : k * (fast_exp(x[e] - m) * inv - (c == y ? 1.0f : 0.0f)));
            }
        }
    }
    if (BACKWARD || p.reduction == kNone) return;
    num = block_sum(num, scratch);
    if (!ONE) den = block_sum(den, scratch);
    if (threadIdx.x) return;
    if (ONE) {
        if (p.reduction == kMean) *p.den = all;
        *p.loss = (float)(p.reduction == kMean ? num / all : num);
    } else if (block_at() < p.parts)
        p.part[block_at()] = make_double2(num, den);
}

// ---- many classes: lanes or a workgroup per row ----------------------------------------------------------------------------
// The row is taken as accesses of VEC values at addresses that are multiples of 16 bytes; those at its ends value by value, and so are all
// stores where the gradient's rows do not begin at the same place within 16 bytes as the logits'.
template <class T> struct RowOf {
    static constexpr int VEC = 16 / sizeof(T);
    typedef Vec<T, VEC> V;
    const T* row;
    T* out;
    int shift;   // values between the aligned address before the row and the row
    int c;
    bool wide;   // stores
    __device__ __forceinline__ RowOf(const Loss& p, i64 r)
        : row((const T*)p.logits + r * p.stride), out((T*)p.grad + r * p.c), shift((int)((size_t)row % 16 / sizeof(T))), c((int)p.c), wide(p.wide) {}
    __device__ __forceinline__ int accesses() const { return (c + shift + VEC - 1) / VEC; }
    __device__ __forceinline__ V load(int j) const {
        const int at = j * VEC - shift;
        if (at >= 0 && at + VEC <= c) return *(const V*)(row + at);
        V x;
#pragma unroll
        for (int e = 0; e < VEC; ++e) x.v[e] = at + e >= 0 && at + e < c ? row[at + e] : (T)(-__builtin_inff());
        return x;
    }
    __device__ __forceinline__ void store(int j, const V& x) const {
        const int at = j * VEC - shift;
        if (wide && at >= 0 && at + VEC <= c) {
            *(V*)(out + at) = x;
            return;
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (at + e >= 0 && at + e < c) out[at + e] = x.v[e];
    }
    __device__ __forceinline__ bool inside(int j, int e) const { return j * VEC - shift + e >= 0 && j * VEC - shift + e < c; }
};

// Rows of up to 512 accesses: a group of lanes (a power of two, at most 64) per row, R accesses a lane in registers; nothing passes through LDS
// but the workgroup's sums.  Rows come before their labels are known, ignored ones too: what such rows cost is waiting, not bytes.  (65,536 rows
// of 2,000 bf16: 62 us for the loss = 4.2 TB/s, 149 with the gradient; 1,048,576 of 300: 250 and 520, where a workgroup a row took 1,428 and 2,630.)
template <class T, int R, bool BACKWARD>
__global__ __launch_bounds__(256) void loss_group_kernel(Loss p, int log_lanes) {
    typedef typename RowOf<T>::V V;
    constexpr int VEC = RowOf<T>::VEC;
    __shared__ double scratch[4];
    if (BACKWARD && p.skip_unit && p.reduction != kNone && *p.upstream == 1.0f) return;
    const int lanes = 1 << log_lanes, lane = threadIdx.x & (lanes - 1);
    const double all = p.grad ? weights_of(p) : 1.0;
    const i64 r = block_at() * (256 >> log_lanes) + (threadIdx.x >> log_lanes);
    double num = 0, den = 0;
    if (r < p.n) {
        const i64 y = label_at(p, r);
        const float w = weight_of(p, y);
        const bool ignored = y == p.ignore;   // nothing to read then
        const RowOf<T> row(p, r);
        const int n = row.accesses();
        V x[R];
        float m = -__builtin_inff(), z = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (lane + (i << log_lanes) < n) x[i] = row.load(lane + (i << log_lanes));
        if (BACKWARD) {
            m = p.stat[r].x;
            z = p.stat[r].y;
        } else if (!ignored) {
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (lane + (i << log_lanes) < n)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) m = fmaxf(m, to_f32(x[i].v[e]));
            for (int o = lanes >> 1; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
#pragma unroll
            for (int i = 0; i < R; ++i)
                if (lane + (i << log_lanes) < n)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) z += row.inside(lane + (i << log_lanes), e) ? fast_exp(to_f32(x[i].v[e]) - m) : 0.0f;
            for (int o = lanes >> 1; o; o >>= 1) z += __shfl_xor(z, o);
        }
        if (!BACKWARD && lane == 0) {
            p.stat[r] = make_float2(m, z);
            const float l = ignored ? 0.0f : w * loss_of(m, z, y >= 0 && y < p.c ? to_f32(row.row[y]) : 0.0f);
            if (p.reduction == kNone) p.loss[r] = l;
            num = l;
            den = w;
        }
        if (p.grad) {
            const float k = factor_of(p, w, all, r), inv = 1.0f / z;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int j = lane + (i << log_lanes);
                if (j >= n) continue;
                V g;
#pragma unroll
                for (int e = 0; e < VEC; ++e)
                    g.v[e] = from_f32<T>(ignored ? 0.0f : k * (fast_exp(to_f32(x[i].v[e]) - m) * inv - (j * VEC - row.shift + e == y ? 1.0f : 0.0f)));
                row.store(j, g);
            }
        }
    }
    if (BACKWARD || p.reduction == kNone) return;
    num = block_sum(num, scratch);
    den = block_sum(den, scratch);
    if (threadIdx.x == 0 && block_at() < p.parts) p.part[block_at()] = make_double2(num, den);
}

// More: a workgroup per row.  R > 0: up to R accesses a thread, held in registers; R = 0: any number, read twice.  4 accesses a thread keep enough
// under way; more threads than that needs take the place of other rows (65,536 rows of 8,000 bf16 with their gradient: 438 us for 256 threads,
// 554 for 512), fewer registers than 8 accesses hide more (8,192 of 32,000: 234 us = 4.5 TB/s for 1,024 threads, 263 for 512, 286 for 256).
// EARLY: the row is on its way while its label is; where it is long and its time its bytes', rows that are ignored are not read instead.
template <class T, int R, bool EARLY, bool BACKWARD>
__global__ __launch_bounds__(1024) void loss_many_kernel(Loss p) {
    typedef typename RowOf<T>::V V;
    constexpr int VEC = RowOf<T>::VEC;
    __shared__ float scratch[16];
    if (BACKWARD && p.skip_unit && p.reduction != kNone && *p.upstream == 1.0f) return;
    const i64 r = block_at();
    if (r >= p.n) return;
    const int threads = blockDim.x;
    const RowOf<T> row(p, r);
    const int n = row.accesses();
    V x[R ? R : 1];
    auto load = [&]() {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int j = threadIdx.x + i * threads;
            if (j < n) x[i] = row.load(j);
        }
    };
    if (EARLY) load();
    const i64 y = label_at(p, r);
    const float w = weight_of(p, y);
    if (y == p.ignore) {   // nothing to read
        if (!BACKWARD && threadIdx.x == 0) {
            p.stat[r] = make_float2(0.0f, 1.0f);
            if (p.reduction == kNone) p.loss[r] = 0.0f;
            else p.part[r] = make_double2(0, 0);
        }
        V none;
#pragma unroll
        for (int e = 0; e < VEC; ++e) none.v[e] = T{};
        if (p.grad)
            for (int j = threadIdx.x; j < n; j += threads) row.store(j, none);
        return;
    }
    float m = -__builtin_inff(), z = 0.0f;
    if (!EARLY) load();
    if (BACKWARD) {
        m = p.stat[r].x;
        z = p.stat[r].y;
    } else {
        if (R) {
#pragma unroll
            for (int i = 0; i < R; ++i)
                if ((int)threadIdx.x + i * threads < n)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) m = fmaxf(m, to_f32(x[i].v[e]));
            m = block_max(m, scratch);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int j = threadIdx.x + i * threads;
                if (j < n)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) z += row.inside(j, e) ? fast_exp(to_f32(x[i].v[e]) - m) : 0.0f;
            }
        } else {
            // one pass with a running maximum: what was summed under the old one is scaled when it moves
            for (int j = threadIdx.x; j < n; j += threads) {
                const V v = row.load(j);
                float top = m;
#pragma unroll
                for (int e = 0; e < VEC; ++e) top = fmaxf(top, to_f32(v.v[e]));
                if (top > m) {
                    z *= fast_exp(m - top);   // m = -inf at first: 0
                    m = top;
                }
                if (m > -__builtin_inff())
#pragma unroll
                    for (int e = 0; e < VEC; ++e) z += row.inside(j, e) ? fast_exp(to_f32(v.v[e]) - m) : 0.0f;
                else
#pragma unroll
                    for (int e = 0; e < VEC; ++e) z += to_f32(v.v[e]) == m ? 0.0f : __builtin_nanf("");   // nothing but -inf so far, or a NaN
            }
            const float top = block_max(m, scratch);
            z = m == top ? z : z * fast_exp(m - top);
            m = top;
        }
        z = block_sum(z, scratch);
        if (m == -__builtin_inff()) z = __builtin_nanf("");   // no class is possible
        if (threadIdx.x == 0) {
            p.stat[r] = make_float2(m, z);
            const float l = w * loss_of(m, z, y >= 0 && y < p.c ? to_f32(row.row[y]) : 0.0f);
            if (p.reduction == kNone) p.loss[r] = l;
            else p.part[r] = make_double2(l, w);
        }
    }
    if (!p.grad) return;
    const float k = factor_of(p, w, weights_of(p), r), inv = 1.0f / z;
    auto gradient = [&](int j, V v) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            v.v[e] = from_f32<T>(k * (fast_exp(to_f32(v.v[e]) - m) * inv - (j * VEC - row.shift + e == y ? 1.0f : 0.0f)));
        row.store(j, v);
    };
    if (R) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int j = threadIdx.x + i * threads;
            if (j < n) gradient(j, x[i]);
        }
    } else
        for (int j = threadIdx.x; j < n; j += threads) gradient(j, row.load(j));
}

// ---- host -----------------------------------------------------------------------------------------------------------------
// Classes up to which a lane takes single values, 4 of them; many rows of more classes than one lane has are taken in accesses of 16 bytes
// instead (2^21 rows, loss alone: 32 bf16 classes 49 us, by single values 128; 8: 26 and 40; 4: 28 and 25)
constexpr i64 kFew = 256, kFewOfMany = 4;
// Accesses up to which a row is a group of lanes' (65,536 rows of bf16, loss alone: 112 us for 2,100 classes, 233 by a workgroup each; 65,536 of
// 4,100: 329 against 180)
constexpr i64 kGroupMost = 512;

constexpr i64 kOne = 4096;  // lanes' worth of rows up to which one workgroup takes them all: 2 launches less, 4 rows a group at most

int few_lanes(i64 c) {   // 4 values a lane
    int ll = 0;
    while ((4 << ll) < c) ++ll;
    return ll;
}
bool one_workgroup(i64 n, i64 c) { return c <= kFew && n << few_lanes(c) <= kOne; }

// notes in p how many sums there are to join
template <class T, bool BACKWARD> void launch_rows(hipStream_t s, Loss& p) {
    const bool one = one_workgroup(p.n, p.c);
    if (one || p.c <= kFewOfMany) {
        const int ll = few_lanes(p.c);
        if (!BACKWARD && one) {
            const i64 threads = cdiv(p.n << ll, 64) * 64;
            hipLaunchKernelGGL((loss_few_kernel<T, 4, false, true>), dim3(1), dim3((unsigned)(threads < 1024 ? threads : 1024)), 0, s, p, ll);
            return;
        }
        p.parts = (int)cdiv(p.n, 256 >> ll);
        hipLaunchKernelGGL((loss_few_kernel<T, 4, BACKWARD, false>), grid_of(p.parts), dim3(256), 0, s, p, ll);
        return;
    }
    p.wide = (size_t)p.logits % 16 == (size_t)p.grad % 16 && (p.n == 1 || (p.stride - p.c) * (i64)sizeof(T) % 16 == 0);
    const i64 accesses = cdiv(p.c, 16 / sizeof(T)) + 1;   // at most: whether or not there is a gradient to write, so that the sums are the same
    if (accesses <= kGroupMost) {
        int ll = 0;
        while ((4 << ll) < accesses && ll < 6) ++ll;
        p.parts = (int)cdiv(p.n, 256 >> ll);
        if (accesses <= 256) hipLaunchKernelGGL((loss_group_kernel<T, 4, BACKWARD>), grid_of(p.parts), dim3(256), 0, s, p, ll);
        else hipLaunchKernelGGL((loss_group_kernel<T, 8, BACKWARD>), grid_of(p.parts), dim3(256), 0, s, p, ll);
        return;
    }
    p.parts = (int)p.n;
    const int threads = accesses <= 1024 ? 256 : accesses <= 2048 ? 512 : 1024;
    const int per = (int)cdiv(accesses, threads);
    if (threads < 1024) hipLaunchKernelGGL((loss_many_kernel<T, 4, true, BACKWARD>), grid_of(p.n), dim3(threads), 0, s, p);
    else if (per <= 4) hipLaunchKernelGGL((loss_many_kernel<T, 4, false, BACKWARD>), grid_of(p.n), dim3(threads), 0, s, p);
    else if (per <= 8) hipLaunchKernelGGL((loss_many_kernel<T, 8, false, BACKWARD>), grid_of(p.n), dim3(threads), 0, s, p);
    else hipLaunchKernelGGL((loss_many_kernel<T, 0, false, BACKWARD>), grid_of(p.n), dim3(threads), 0, s, p);
}
template <bool BACKWARD> void launch_typed(hipStream_t s, Loss& p, int dtype) {
    if (dtype == DSP_FT_F32) launch_rows<float, BACKWARD>(s, p);
    else if (dtype == DSP_FT_BF16) launch_rows<__bf16, BACKWARD>(s, p);
    else launch_rows<_Float16, BACKWARD>(s, p);
}

const char* bad_loss(i64 n, i64 c, i64 stride, int dtype, int label_dtype, int reduction) {
    if (n < 0 || n > 0x7fffffffll) return "the number of rows must be within 0 .. 2^31 - 1";
    if (c < 1 || c > (1ll << 30)) return "the number of classes must be within 1 .. 2^30";
    if (stride < c && n > 1) return "rows overlap: the row stride is below the number of classes";
    if (dtype != DSP_FT_F32 && dtype != DSP_FT_BF16 && dtype != DSP_FT_F16) return "unknown element type";
    if (label_dtype != DSP_DT_I64 && label_dtype != DSP_DT_I32 && label_dtype != DSP_DT_U8) return "labels must be int64, int32 or uint8";
    if (reduction != kMean && reduction != kSum && reduction != kNone) return "unknown reduction";
    return nullptr;
}

}  // namespace

extern "C" {

uint64_t dsp_stream_capture_id(void* stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo((hipStream_t)stream, &status, &id) != hipSuccess) {
        (void)hipGetLastError();
        return 0;
    }
    return status == hipStreamCaptureStatusActive ? id : 0;
}

int64_t dsp_cross_entropy_workspace(int64_t n) { return n < 0 ? refuse("dsp_cross_entropy_workspace", "negative number of rows") : (int64_t)((n + kJoinParts) * sizeof(double2) + kWeightParts * sizeof(double)); }

int32_t dsp_cross_entropy_forward(void* stream, int64_t n, int64_t c, const void* logits, int32_t dtype, int64_t row_stride, const void* labels,
                                  int32_t label_dtype, const float* weight, int64_t ignore_index, int32_t reduction, float* loss, float* stat,
                                  double* weight_sum, void* grad, void* workspace, int64_t workspace_bytes) {
    const char* who = "dsp_cross_entropy_forward";
    if (const char* why = bad_loss(n, c, row_stride, dtype, label_dtype, reduction)) return refuse(who, why);
    if (!workspace || workspace_bytes < dsp_cross_entropy_workspace(n)) return refuse(who, "workspace too small (dsp_cross_entropy_workspace)");
    if (n && (!logits || !labels || !loss || !stat)) return refuse(who, "NULL pointer");
    if ((reduction != kNone && !loss) || (reduction == kMean && !weight_sum)) return refuse(who, "NULL pointer");
    if ((size_t)workspace & 255) return refuse(who, "the workspace must be aligned to 256 bytes");
    Loss p = {logits, labels, weight, grad, loss, (float2*)stat, weight_sum, (double2*)workspace, nullptr, n, c, row_stride, ignore_index, label_dtype, reduction, 0, 0,
              (double*)((double2*)workspace + n + kJoinParts), 0};
    hipStream_t s = (hipStream_t)stream;
    if (grad && reduction == kMean && n && !one_workgroup(n, c)) {
        p.weight_parts = (int)(cdiv(n, 1024) < kWeightParts ? cdiv(n, 1024) : kWeightParts);
        hipLaunchKernelGGL(loss_weights_kernel, dim3(p.weight_parts), dim3(1024), 0, s, p);
    }
    if (n) launch_typed<false>(s, p, dtype);
    if (reduction != kNone && p.parts > kJoinParts * 64) {   // up to 16,384 one workgroup takes no longer than another launch
        double2* joined = p.part + n;
        hipLaunchKernelGGL(loss_join_parts_kernel, dim3(kJoinParts), dim3(1024), 0, s, p, joined);
        p.part = joined;
        p.parts = kJoinParts;
    }
    if (reduction != kNone && (n == 0 || !one_workgroup(n, c))) hipLaunchKernelGGL(loss_join_kernel, dim3(1), dim3(1024), 0, s, p);
    return launched(who);
}

int32_t dsp_cross_entropy_backward(void* stream, int64_t n, int64_t c, const void* logits, int32_t dtype, int64_t row_stride, const void* labels,
                                   int32_t label_dtype, const float* weight, int64_t ignore_index, int32_t reduction, const float* stat,
                                   const double* weight_sum, const float* upstream, int32_t skip_unit, void* grad) {
    const char* who = "dsp_cross_entropy_backward";
    if (const char* why = bad_loss(n, c, row_stride, dtype, label_dtype, reduction)) return refuse(who, why);
    if (n == 0) return DSP_OK;
    if (!logits || !labels || !stat || !upstream || !grad || (reduction == kMean && !weight_sum)) return refuse(who, "NULL pointer");
    Loss p = {logits, labels, weight, grad, nullptr, (float2*)stat, (double*)weight_sum, nullptr, upstream, n, c, row_stride, ignore_index, label_dtype,
              reduction, 0, skip_unit, nullptr, 0};
    launch_typed<true>((hipStream_t)stream, p, dtype);
    return launched(who);
}

}  // extern "C"
