// dsp_lstm_train.hip -- an LSTM layer, one or both directions, with its gradient: the recurrence of models.py:137-157 as a
// training step needs it (torch.nn.LSTM's definition: gates i, f, g, o along 4H).
//
//   z_t = W_ih x_t + W_hh h_(t-1) + b_ih + b_hh      i, f, o = sigmoid(z)    g = tanh(z)
//   c_t = f c_(t-1) + i g                            h_t = o tanh(c_t)
//   backward, from the last step to the first:  dh_t = dy_t + W_hh^T dz_(t+1)     dc_t = dc_(t+1) f_(t+1) + dh_t o (1 - tanh^2 c_t)
//   dz = (dc g i (1 - i),  dc c_(t-1) f (1 - f),  dc i (1 - g^2),  dh tanh(c) o (1 - o))
//   dx_t = W_ih^T dz_t      dW_ih = sum dz_t x_t^T      dW_hh = sum dz_t h_(t-1)^T      db = sum dz_t
//
// All in 32 bits on the fp32 matrix instructions, which bound it where the batch is large: 2 x 4H (I + H) operations a step,
// sequence and direction, twice that again backward.  What does not wait for the recurrence (W_ih x of all steps, and dx, dW
// behind it) is done by one product over all steps; the recurrence is a launch per step for both directions, its product,
// the gates and the states in one kernel.  A launch ends before the next begins, so no workgroup waits for another.
//
// Layouts: x [B][T][I], y [B][T][dirs H], states [dirs][B][H], gates [dirs][T][B][4H] and cells [dirs][T][B][H] by the time in
// the sequence; a row of the products over all steps is m = t B + b.
#include "dsp_ops.h"

using namespace dsp;

namespace {

// ---- operands of a product C(m, n) = sum over k of A(m, k) B(n, k) -------------------------------------------------------
// kAlongK: values of a row lie along k (at(row) + k);  otherwise along the rows (at(k) + row).  NULL: zeros.
struct Plain {   // rows (or columns) `ld` apart
    const float* p[2];
    i64 ld;
    __device__ __forceinline__ const float* at(int d, int i) const { return p[d] + i * ld; }
};
struct Inputs {   // x by m = t B + b
    const float* x;
    int B, T, I;
    __device__ __forceinline__ const float* at(int, int m) const {
        const int t = m / B, b = m - t * B;
        return x + ((i64)b * T + t) * I;
    }
};
struct Before {   // h of the step before, by m = t B + b
    const float *y, *h0;
    int B, T, H, dirs;
    __device__ __forceinline__ const float* at(int d, int m) const {
        const int t = m / B, b = m - t * B, before = d ? t + 1 : t - 1;
        if (before < 0 || before >= T) return h0 ? h0 + ((i64)d * B + b) * H : nullptr;
        return y + (((i64)b * T + before) * dirs + d) * H;
    }
};

// ---- the product over all steps --------------------------------------------------------------------------------------------
// A workgroup of 4 waves makes a tile of TILE x TILE, a wave a quarter of it as 32 x 32 blocks of v_mfma_f32_32x32x2; 16 values
// of k are staged in LDS at a time, the next 16 on their way in registers meanwhile.  A lane's 4 values of k are consecutive
// (lane group q: k = 4q + j for instruction j): the order of k is the same for both operands, so any is right.
constexpr int kStep = 16;

template <bool ALONG_K, int TILE> struct Stage {
    static constexpr int kStride = ALONG_K ? kStep + 4 : TILE + 4;
    static constexpr int kFloats = ALONG_K ? TILE * kStride : kStep * kStride;
    static constexpr int kLoads = TILE * kStep / 4 / 256;
    f32x4 v[kLoads];
    // `rows`, `k_end`: bounds of the operand; row0, k0: the tile's
    template <class Op> __device__ __forceinline__ void fetch(const Op& op, int d, int row0, int rows, int k0, int k_end, bool wide) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int j = threadIdx.x + i * 256;
            const int a = ALONG_K ? row0 + j / (kStep / 4) : k0 + j / (TILE / 4);                     // which line
            const int b = ALONG_K ? k0 + j % (kStep / 4) * 4 : row0 + j % (TILE / 4) * 4;             // where on it
            const int lines = ALONG_K ? rows : k_end, most = ALONG_K ? k_end : rows;
            v[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            const float* p = a < lines ? op.at(d, a) : nullptr;
            if (!p) continue;
            if (wide && b + 4 <= most) v[i] = *(const f32x4*)(p + b);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (b + e < most) v[i][e] = p[b + e];
        }
    }
    __device__ __forceinline__ void put(float* lds) const {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int j = threadIdx.x + i * 256;
            const int at = ALONG_K ? j / (kStep / 4) * kStride + j % (kStep / 4) * 4 : j / (TILE / 4) * kStride + j % (TILE / 4) * 4;
            *(f32x4*)(lds + at) = v[i];
        }
    }
    // 4 consecutive values of k of one row
    static __device__ __forceinline__ f32x4 get(const float* lds, int row, int k) {
        if (ALONG_K) return *(const f32x4*)(lds + row * kStride + k);
        f32x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = lds[(k + e) * kStride + row];
        return r;
    }
};

// C tile += over k in [k0, k1) of direction d;  acc[i][j]: block (i, j) of the wave's quarter
template <bool A_ALONG_K, bool B_ALONG_K, int TILE, class A, class B>
__device__ __forceinline__ void product(const A& a, const B& b, int d, int m0, int M, int n0, int N, int k0, int k1, bool wide_a, bool wide_b,
                                        float* lds, f32x16 (&acc)[TILE / 64][TILE / 64]) {
    typedef Stage<A_ALONG_K, TILE> SA;
    typedef Stage<B_ALONG_K, TILE> SB;
    constexpr int R = TILE / 64;
    float *la = lds, *lb = lds + SA::kFloats;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = (wave >> 1) * (TILE / 2) + (lane & 31), wn = (wave & 1) * (TILE / 2) + (lane & 31), kq = (lane >> 5) * 4;
    SA sa;
    SB sb;
    sa.fetch(a, d, m0, M, k0, k1, wide_a);
    sb.fetch(b, d, n0, N, k0, k1, wide_b);
    for (int k = k0; k < k1; k += kStep) {
        __syncthreads();
        sa.put(la);
        sb.put(lb);
        __syncthreads();
        if (k + kStep < k1) {
            sa.fetch(a, d, m0, M, k + kStep, k1, wide_a);
            sb.fetch(b, d, n0, N, k + kStep, k1, wide_b);
        }
#pragma unroll
        for (int kk = 0; kk < kStep; kk += 8) {
            f32x4 fa[R], fb[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                fa[i] = SA::get(la, wm + i * 32, kk + kq);
                fb[i] = SB::get(lb, wn + i * 32, kk + kq);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int j = 0; j < R; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[i][e], fb[j][e], acc[i][j], 0, 0, 0);
        }
    }
}
// f(m, n, value) for every value of the tile that is inside
template <int TILE, class F> __device__ __forceinline__ void each(const f32x16 (&acc)[TILE / 64][TILE / 64], int m0, int M, int n0, int N, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < TILE / 64; ++i)
#pragma unroll
        for (int j = 0; j < TILE / 64; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + (wave >> 1) * (TILE / 2) + i * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
                const int n = n0 + (wave & 1) * (TILE / 2) + j * 32 + (lane & 31);
                if (m < M && n < N) f(m, n, acc[i][j][r]);
            }
}
template <bool A_ALONG_K, bool B_ALONG_K, int TILE> constexpr int lds_floats() { return Stage<A_ALONG_K, TILE>::kFloats + Stage<B_ALONG_K, TILE>::kFloats; }

struct Shape { int B, T, I, H, dirs, wide_x, wide_h, wide_wx; };   // wide_*: accesses of 16 bytes along I of x, along H, along I of W_ih
struct Weights { const float *w_ih[2], *w_hh[2], *b_ih[2], *b_hh[2]; };

// gates = W_ih x + b_ih + b_hh, all steps;  blockIdx.z: direction
template <int TILE> __global__ __launch_bounds__(256) void lstm_inputs_kernel(Shape s, const float* __restrict__ x, Weights w, float* __restrict__ gates) {
    __shared__ __attribute__((aligned(16))) float lds[lds_floats<true, true, TILE>()];
    const int d = blockIdx.z, m0 = blockIdx.x * TILE, n0 = blockIdx.y * TILE, M = s.B * s.T, N = 4 * s.H;
    const Inputs a = {x, s.B, s.T, s.I};
    const Plain b = {{w.w_ih[0], w.w_ih[1]}, s.I};
    f32x16 acc[TILE / 64][TILE / 64] = {};
    product<true, true, TILE>(a, b, d, m0, M, n0, N, 0, s.I, s.wide_x, s.wide_wx, lds, acc);
    float* out = gates + (i64)d * M * N;
    each<TILE>(acc, m0, M, n0, N, [&](int m, int n, float v) { out[(i64)m * N + n] = v + (w.b_ih[d][n] + w.b_hh[d][n]); });
}

// dx = sum over directions of dz W_ih
template <int TILE> __global__ __launch_bounds__(256) void lstm_input_grad_kernel(Shape s, const float* __restrict__ dz, Weights w, float* __restrict__ dx) {
    __shared__ __attribute__((aligned(16))) float lds[lds_floats<true, false, TILE>()];
    const int m0 = blockIdx.x * TILE, n0 = blockIdx.y * TILE, M = s.B * s.T, K = 4 * s.H;
    const Plain a = {{dz, dz + (i64)M * K}, K}, b = {{w.w_ih[0], w.w_ih[1]}, s.I};
    f32x16 acc[TILE / 64][TILE / 64] = {};
    for (int d = 0; d < s.dirs; ++d) product<true, false, TILE>(a, b, d, m0, M, n0, s.I, 0, K, true, s.wide_wx, lds, acc);
    each<TILE>(acc, m0, M, n0, s.I, [&](int m, int n, float v) {
        const int t = m / s.B, b = m - t * s.B;
        dx[((i64)b * s.T + t) * s.I + n] = v;
    });
}

// dW of both weights: tiles of [4H][I] first, tiles of [4H][H] behind them; blockIdx.z = direction x part of the sum over m.  Where
// there is one part it writes the gradients, else part[part][direction][4H][I + H] for lstm_join_kernel.
template <int TILE>
__global__ __launch_bounds__(256) void lstm_weight_grad_kernel(Shape s, const float* __restrict__ dz, const float* __restrict__ x, const float* __restrict__ y,
                                                               const float* __restrict__ h0, int parts, int per_part, int x_tiles, float* __restrict__ part,
                                                               float* dw_ih0, float* dw_ih1, float* dw_hh0, float* dw_hh1) {
    __shared__ __attribute__((aligned(16))) float lds[lds_floats<false, false, TILE>()];
    const int d = blockIdx.z / parts, q = blockIdx.z - d * parts, m0 = blockIdx.y * TILE, M = 4 * s.H, K = s.B * s.T;
    const bool of_x = (int)blockIdx.x < x_tiles;
    const int n0 = (of_x ? blockIdx.x : blockIdx.x - x_tiles) * TILE, N = of_x ? s.I : s.H;
    const int k0 = q * per_part, k1 = k0 + per_part < K ? k0 + per_part : K;
    const Plain a = {{dz, dz + (i64)M * K}, M};
    f32x16 acc[TILE / 64][TILE / 64] = {};
    if (of_x) {
        const Inputs b = {x, s.B, s.T, s.I};
        product<false, false, TILE>(a, b, d, m0, M, n0, N, k0, k1, true, s.wide_x, lds, acc);
    } else {
        const Before b = {y, h0, s.B, s.T, s.H, s.dirs};
        product<false, false, TILE>(a, b, d, m0, M, n0, N, k0, k1, true, s.wide_h, lds, acc);
    }
    if (parts == 1) {
        float* out = of_x ? (d ? dw_ih1 : dw_ih0) : (d ? dw_hh1 : dw_hh0);
        each<TILE>(acc, m0, M, n0, N, [&](int m, int n, float v) { out[(i64)m * N + n] = v; });
    } else {
        float* out = part + ((i64)q * s.dirs + d) * M * (s.I + s.H) + (of_x ? 0 : s.I);
        each<TILE>(acc, m0, M, n0, N, [&](int m, int n, float v) { out[(i64)m * (s.I + s.H) + n] = v; });
    }
}
// the parts in order, and both weights apart
__global__ __launch_bounds__(256) void lstm_join_kernel(Shape s, int parts, const float* __restrict__ part, float* dw_ih0, float* dw_ih1, float* dw_hh0, float* dw_hh1) {
    const i64 one = (i64)4 * s.H * (s.I + s.H), i = (i64)blockIdx.x * 256 + threadIdx.x;
    if (i >= one * s.dirs) return;
    float v = 0.0f;
    for (int q = 0; q < parts; ++q) v += part[q * one * s.dirs + i];
    const int d = i >= one;
    const i64 j = i - d * one, m = j / (s.I + s.H);
    const int n = (int)(j - m * (s.I + s.H));
    if (n < s.I) (d ? dw_ih1 : dw_ih0)[m * s.I + n] = v;
    else (d ? dw_hh1 : dw_hh0)[m * s.H + n - s.I] = v;
}

// db: sums of dz over m.  64 columns a workgroup, a quarter of its rows a wave; part[rows of workgroups][dirs][4H]
__global__ __launch_bounds__(256) void lstm_bias_grad_kernel(Shape s, const float* __restrict__ dz, int per_part, float* __restrict__ part) {
    __shared__ float sums[4][64];
    const int d = blockIdx.z, M = s.B * s.T, N = 4 * s.H, n = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
    const int from = blockIdx.y * per_part, to = from + per_part < M ? from + per_part : M;
    float v = 0.0f;
    if (n < N)
        for (int m = from + q; m < to; m += 4) v += dz[((i64)d * M + m) * N + n];
    sums[q][threadIdx.x & 63] = v;
    __syncthreads();
    if (q == 0 && n < N) part[((i64)blockIdx.y * s.dirs + d) * N + n] = (sums[0][threadIdx.x] + sums[1][threadIdx.x]) + (sums[2][threadIdx.x] + sums[3][threadIdx.x]);
}
__global__ __launch_bounds__(256) void lstm_bias_join_kernel(Shape s, int parts, const float* __restrict__ part, float* db0, float* db1, float* db2, float* db3) {
    const int N = 4 * s.H, i = blockIdx.x * 256 + threadIdx.x;
    if (i >= N * s.dirs) return;
    float v = 0.0f;
    for (int q = 0; q < parts; ++q) v += part[(i64)q * N * s.dirs + i];
    const int d = i >= N, n = i - d * N;
    (d ? db1 : db0)[n] = v;   // b_ih and b_hh are added to the same place
    (d ? db3 : db2)[n] = v;
}

// ---- the recurrence ----------------------------------------------------------------------------------------------------------
// sigmoid and tanh by one exponential each; both stay within a few 2^-24 of themselves near 1 and absolute elsewhere, and
// saturate without overflow: 2^(large) = inf and 1 / inf = 0
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f)); }
__device__ __forceinline__ float tanh_of(float x) {
    const float a = fabsf(x);
    if (a < 0.25f) {   // the quotient loses digits to cancellation here: the series of tanh to x^9 has an error below 2^-24 x
        const float q = x * x;
        return x + x * q * (-1.0f / 3 + q * (2.0f / 15 + q * (-17.0f / 315 + q * (62.0f / 2835))));
    }
    const float e = __builtin_amdgcn_exp2f(a * 2.88539008177792681472f);
    return copysignf(1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + e), x);
}

// A workgroup's tile: 64 sequences by 16 columns of each of G groups of columns (forward: the 4 gates of 16 units; backward:
// 16 units); a wave takes 16 sequences.  acc[g] += A [64][K] (rows by `row`, NULL = zeros) x W [columns][K], values along k in both,
// 32 values of k staged in LDS at a time.
constexpr int kSeqs = 64, kUnits = 16, kDepth = 32, kPad = kDepth + 4;

template <int G, class Row, class Col>
__device__ __forceinline__ void step_product(int K, bool wide, Row row, Col col, float* lds, f32x4 (&acc)[G]) {
    float *la = lds, *lw = lds + kSeqs * kPad;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int LA = kSeqs * kDepth / 4 / 256, LW = (G * kUnits * kDepth / 4 + 255) / 256;
    f32x4 va[LA], vw[LW];
    auto load = [&](const float* p, int k) {
        f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (!p) return v;
        if (wide && k + 4 <= K) return *(const f32x4*)(p + k);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k + e < K) v[e] = p[k + e];
        return v;
    };
    auto fetch = [&](int k) {
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            const int j = threadIdx.x + i * 256;
            va[i] = load(row(j / (kDepth / 4)), k + j % (kDepth / 4) * 4);
        }
#pragma unroll
        for (int i = 0; i < LW; ++i) {
            const int j = threadIdx.x + i * 256;
            if (j < G * kUnits * kDepth / 4) vw[i] = load(col(j / (kDepth / 4)), k + j % (kDepth / 4) * 4);
        }
    };
    fetch(0);
    for (int k = 0; k < K; k += kDepth) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LA; ++i) {
            const int j = threadIdx.x + i * 256;
            *(f32x4*)(la + j / (kDepth / 4) * kPad + j % (kDepth / 4) * 4) = va[i];
        }
#pragma unroll
        for (int i = 0; i < LW; ++i) {
            const int j = threadIdx.x + i * 256;
            if (j < G * kUnits * kDepth / 4) *(f32x4*)(lw + j / (kDepth / 4) * kPad + j % (kDepth / 4) * 4) = vw[i];
        }
        __syncthreads();
        if (k + kDepth < K) fetch(k + kDepth);
#pragma unroll
        for (int kk = 0; kk < kDepth; kk += 16) {
            const int at = kk + (lane >> 4) * 4;
            const f32x4 a = *(const f32x4*)(la + (wave * 16 + (lane & 15)) * kPad + at);
            f32x4 w[G];
#pragma unroll
            for (int g = 0; g < G; ++g) w[g] = *(const f32x4*)(lw + (g * kUnits + (lane & 15)) * kPad + at);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int g = 0; g < G; ++g) acc[g] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], w[g][e], acc[g], 0, 0, 0);
        }
    }
}

// gates: in W_ih x + b of all steps; out (save) i, f, g, o.  cells: c of all steps (save), else of two steps in turn
__global__ __launch_bounds__(256) void lstm_step_kernel(Shape s, int step, Weights w, const float* __restrict__ h0, const float* __restrict__ c0,
                                                        float* gates, float* cells, float* y, float* __restrict__ hn, float* __restrict__ cn, int save) {
    __shared__ __attribute__((aligned(16))) float lds[(kSeqs + 4 * kUnits) * kPad];
    const int d = blockIdx.z, B = s.B, T = s.T, H = s.H, t = d ? T - 1 - step : step, before = d ? t + 1 : t - 1;
    const int b0 = blockIdx.x * kSeqs, u0 = blockIdx.y * kUnits;
    f32x4 acc[4] = {};
    if (step > 0 || h0) {
        const float* w_hh = w.w_hh[d];
        step_product<4>(
            H, s.wide_h,
            [&](int i) -> const float* {
                const int b = b0 + i;
                if (b >= B) return nullptr;
                return step ? y + (((i64)b * T + before) * s.dirs + d) * H : h0 + ((i64)d * B + b) * H;
            },
            [&](int j) -> const float* {
                const int u = u0 + j % kUnits;
                return u < H ? w_hh + ((i64)(j / kUnits) * H + u) * H : nullptr;
            },
            lds, acc);
    }
    const int lane = threadIdx.x & 63, u = u0 + (lane & 15);
    if (u >= H) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int b = b0 + (threadIdx.x >> 6) * 16 + (lane >> 4) * 4 + r;
        if (b >= B) continue;
        float* z = gates + (((i64)d * T + t) * B + b) * 4 * H + u;
        const float i = sigmoid(z[0] + acc[0][r]), f = sigmoid(z[H] + acc[1][r]), g = tanh_of(z[2 * H] + acc[2][r]), o = sigmoid(z[3 * H] + acc[3][r]);
        float c = 0.0f;
        if (step) c = cells[(((i64)d * (save ? T : 2) + (save ? before : (step - 1) & 1)) * B + b) * H + u];
        else if (c0) c = c0[((i64)d * B + b) * H + u];
        c = f * c + i * g;
        const float h = o * tanh_of(c);
        if (save) {
            z[0] = i;
            z[H] = f;
            z[2 * H] = g;
            z[3 * H] = o;
        }
        cells[(((i64)d * (save ? T : 2) + (save ? t : step & 1)) * B + b) * H + u] = c;
        y[(((i64)b * T + t) * s.dirs + d) * H + u] = h;
        if (step == T - 1) {
            hn[((i64)d * B + b) * H + u] = h;
            cn[((i64)d * B + b) * H + u] = c;
        }
    }
}

// [4H][H] -> [H][4H] of both directions, so that the backward step reads along k
__global__ __launch_bounds__(256) void lstm_transpose_kernel(int H, Weights w, float* __restrict__ out) {
    __shared__ float tile[32][33];
    const int d = blockIdx.z, k0 = blockIdx.y * 32, u0 = blockIdx.x * 32, a = threadIdx.x & 31, b = threadIdx.x >> 5;
    for (int i = b; i < 32; i += 8)
        if (k0 + i < 4 * H && u0 + a < H) tile[i][a] = w.w_hh[d][(i64)(k0 + i) * H + u0 + a];
    __syncthreads();
    for (int i = b; i < 32; i += 8)
        if (u0 + i < H && k0 + a < 4 * H) out[((i64)d * H + u0 + i) * 4 * H + k0 + a] = tile[a][i];
}

// One step back; step = T - 1 .. 0, and -1 for the gradient of h0.  dc: gradient of the cell between steps, of c0 in the end.
__global__ __launch_bounds__(256) void lstm_step_back_kernel(Shape s, int step, const float* __restrict__ w_hh_t, const float* __restrict__ c0,
                                                             const float* __restrict__ gates, const float* __restrict__ cells, const float* __restrict__ gy,
                                                             const float* __restrict__ ghn, const float* __restrict__ gcn, float* dz, float* dc, float* dh0) {
    __shared__ __attribute__((aligned(16))) float lds[(kSeqs + kUnits) * kPad];
    const int d = blockIdx.z, B = s.B, T = s.T, H = s.H, t = d ? T - 1 - step : step, before = d ? t + 1 : t - 1, after = d ? t - 1 : t + 1;
    const int b0 = blockIdx.x * kSeqs, u0 = blockIdx.y * kUnits;
    f32x4 acc[1] = {};
    if (step < T - 1)
        step_product<1>(
            4 * H, true,
            [&](int i) -> const float* {
                const int b = b0 + i;
                return b < B ? dz + (((i64)d * T + after) * B + b) * 4 * H : nullptr;
            },
            [&](int j) -> const float* { return u0 + j < H ? w_hh_t + ((i64)d * H + u0 + j) * 4 * H : nullptr; }, lds, acc);
    const int lane = threadIdx.x & 63, u = u0 + (lane & 15);
    if (u >= H) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int b = b0 + (threadIdx.x >> 6) * 16 + (lane >> 4) * 4 + r;
        if (b >= B) continue;
        const i64 at = ((i64)d * B + b) * H + u;
        float dh = acc[0][r];
        if (step < 0) {
            dh0[at] = dh;
            continue;
        }
        if (step == T - 1 && ghn) dh += ghn[at];
        if (gy) dh += gy[(((i64)b * T + t) * s.dirs + d) * H + u];
        const i64 row = ((i64)d * T + t) * B + b;
        const float *a = gates + row * 4 * H + u, i = a[0], f = a[H], g = a[2 * H], o = a[3 * H];
        const float c = tanh_of(cells[row * H + u]);
        const float c_before = step ? cells[(((i64)d * T + before) * B + b) * H + u] : c0 ? c0[at] : 0.0f;
        float dct = step < T - 1 ? dc[at] : gcn ? gcn[at] : 0.0f;
        dct += dh * o * (1.0f - c * c);
        float* q = dz + row * 4 * H + u;
        q[0] = dct * g * i * (1.0f - i);
        q[H] = dct * c_before * f * (1.0f - f);
        q[2 * H] = dct * i * (1.0f - g * g);
        q[3 * H] = dh * c * o * (1.0f - o);
        dc[at] = dct * f;
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
const char* bad_lstm(i64 B, i64 T, i64 I, i64 H, int dirs) {
    if (dirs != 1 && dirs != 2) return "one direction or two";
    if (B < 0 || T < 1 || I < 1 || H < 1) return "sizes must be positive (the batch may be empty)";
    if (I > 65536 || H > 8192) return "at most 65,536 inputs and 8,192 units";
    if (B > (1 << 22) || T > (1 << 22) || B * T >= (1ll << 30)) return "at most 2^22 sequences, 2^22 steps and 2^30 of both";
    return nullptr;
}
// 128 x 128 tiles where they fill the device, else 64 x 64
bool big_tiles(i64 m, i64 n, i64 z) { return cdiv(m, 128) * cdiv(n, 128) * z >= 256; }
bool aligned(const void* p) { return (size_t)p % 16 == 0; }

struct Split { int tile, parts, per_part, bias_parts, bias_per; };
Split split_of(i64 B, i64 T, i64 I, i64 H, int dirs) {   // the sum over m of the weights' gradients, in parts
    Split q;
    const i64 M = 4 * H, K = B * T;
    q.tile = cdiv(M, 128) * (cdiv(I, 128) + cdiv(H, 128)) * dirs * cdiv(K, 512) >= 256 ? 128 : 64;
    const i64 tiles = cdiv(M, q.tile) * (cdiv(I, q.tile) + cdiv(H, q.tile)) * dirs;
    i64 parts = cdiv(512, tiles);   // about two workgroups a CU
    if (parts > cdiv(K, 256)) parts = cdiv(K, 256);
    if (parts < 1) parts = 1;
    q.per_part = (int)(cdiv(cdiv(K, parts), kStep) * kStep);
    if (q.per_part < kStep) q.per_part = kStep;
    q.parts = (int)cdiv(K, q.per_part);
    if (q.parts < 1) q.parts = 1;
    const i64 bias = cdiv(K, 256) < 64 ? cdiv(K, 256) : 64;
    q.bias_per = (int)cdiv(K, bias < 1 ? 1 : bias);
    if (q.bias_per < 1) q.bias_per = 1;
    q.bias_parts = (int)cdiv(K, q.bias_per);
    return q;
}

}  // namespace

extern "C" {

int32_t dsp_lstm_forward(void* stream, const dsp_lstm_layer* l, const float* x, const float* h0, const float* c0, float* y, float* hn, float* cn, float* gates,
                         float* cells, int32_t save) {
    const char* who = "dsp_lstm_forward";
    if (!l) return refuse(who, "NULL layer");
    if (const char* why = bad_lstm(l->batch, l->steps, l->input, l->hidden, l->directions)) return refuse(who, why);
    if (l->batch == 0) return DSP_OK;
    if (!x || !y || !hn || !cn || !gates || !cells) return refuse(who, "NULL pointer");
    Weights w = {};
    bool wide_h = l->hidden % 4 == 0 && aligned(y) && aligned(h0), wide_wx = l->input % 4 == 0;
    for (int d = 0; d < l->directions; ++d) {
        w.w_ih[d] = l->w_ih[d]; w.w_hh[d] = l->w_hh[d]; w.b_ih[d] = l->b_ih[d]; w.b_hh[d] = l->b_hh[d];
        if (!w.w_ih[d] || !w.w_hh[d] || !w.b_ih[d] || !w.b_hh[d]) return refuse(who, "NULL weight");
        wide_h = wide_h && aligned(w.w_hh[d]);
        wide_wx = wide_wx && aligned(w.w_ih[d]);
    }
    const Shape s = {(int)l->batch, (int)l->steps, (int)l->input, (int)l->hidden, l->directions, l->input % 4 == 0 && aligned(x), wide_h, wide_wx};
    hipStream_t q = (hipStream_t)stream;
    const i64 M = l->batch * l->steps, N = 4ll * s.H;
    if (big_tiles(M, N, s.dirs))
        hipLaunchKernelGGL(lstm_inputs_kernel<128>, dim3((unsigned)cdiv(M, 128), (unsigned)cdiv(N, 128), s.dirs), dim3(256), 0, q, s, x, w, gates);
    else
        hipLaunchKernelGGL(lstm_inputs_kernel<64>, dim3((unsigned)cdiv(M, 64), (unsigned)cdiv(N, 64), s.dirs), dim3(256), 0, q, s, x, w, gates);
    const dim3 grid((unsigned)cdiv(s.B, kSeqs), (unsigned)cdiv(s.H, kUnits), s.dirs);
    for (int step = 0; step < s.T; ++step)
        hipLaunchKernelGGL(lstm_step_kernel, grid, dim3(256), 0, q, s, step, w, h0, c0, gates, cells, y, hn, cn, save);
    return launched(who);
}

int64_t dsp_lstm_workspace(const dsp_lstm_layer* l) {
    const char* who = "dsp_lstm_workspace";
    if (!l) return refuse(who, "NULL layer");
    if (const char* why = bad_lstm(l->batch, l->steps, l->input, l->hidden, l->directions)) return refuse(who, why);
    const Split p = split_of(l->batch, l->steps, l->input, l->hidden, l->directions);
    size_t bytes = align256((size_t)l->directions * l->hidden * 4 * l->hidden * 4);                                     // W_hh transposed
    bytes += align256((size_t)l->directions * l->steps * l->batch * 4 * l->hidden * 4);                                 // dz
    if (p.parts > 1) bytes += align256((size_t)p.parts * l->directions * 4 * l->hidden * (l->input + l->hidden) * 4);   // parts of dW
    return (int64_t)(bytes + align256((size_t)p.bias_parts * l->directions * 4 * l->hidden * 4));                       // parts of db
}

int32_t dsp_lstm_backward(void* stream, const dsp_lstm_layer* l, const float* x, const float* h0, const float* c0, const float* y, const float* gates,
                          const float* cells, const float* gy, const float* ghn, const float* gcn, float* dx, float* dh0, float* dc0,
                          const dsp_lstm_grads* g, void* workspace, int64_t workspace_bytes) {
    const char* who = "dsp_lstm_backward";
    if (!l || !g) return refuse(who, "NULL layer");
    if (const char* why = bad_lstm(l->batch, l->steps, l->input, l->hidden, l->directions)) return refuse(who, why);
    const int dirs = l->directions;
    for (int d = 0; d < dirs; ++d)
        if (!l->w_ih[d] || !l->w_hh[d] || !g->w_ih[d] || !g->w_hh[d] || !g->b_ih[d] || !g->b_hh[d]) return refuse(who, "NULL weight or gradient");
    if (l->batch && (!x || !y || !gates || !cells || !dc0 || !workspace)) return refuse(who, "NULL pointer");
    if (workspace_bytes < dsp_lstm_workspace(l)) return refuse(who, "workspace too small (dsp_lstm_workspace)");
    if (!workspace || ((size_t)workspace & 255)) return refuse(who, "the workspace must be aligned to 256 bytes");
    Weights w = {};
    bool wide_wx = l->input % 4 == 0;
    for (int d = 0; d < dirs; ++d) {
        w.w_ih[d] = l->w_ih[d];
        w.w_hh[d] = l->w_hh[d];
        wide_wx = wide_wx && aligned(w.w_ih[d]);
    }
    const Shape s = {(int)l->batch, (int)l->steps, (int)l->input, (int)l->hidden, dirs, l->input % 4 == 0 && aligned(x),
                     l->hidden % 4 == 0 && aligned(y) && aligned(h0), wide_wx};
    const Split p = split_of(l->batch, l->steps, l->input, l->hidden, dirs);
    char* ws = (char*)workspace;
    float* wt = (float*)ws;
    ws += align256((size_t)dirs * s.H * 4 * s.H * 4);
    float* dz = (float*)ws;
    ws += align256((size_t)dirs * s.T * s.B * 4 * s.H * 4);
    float* dw_part = (float*)ws;
    if (p.parts > 1) ws += align256((size_t)p.parts * dirs * 4 * s.H * (s.I + s.H) * 4);
    float* db_part = (float*)ws;
    hipStream_t q = (hipStream_t)stream;
    const i64 M = (i64)s.B * s.T;
    if (s.B) {
        hipLaunchKernelGGL(lstm_transpose_kernel, dim3((unsigned)cdiv(s.H, 32), (unsigned)cdiv(4 * s.H, 32), dirs), dim3(256), 0, q, s.H, w, wt);
        const dim3 grid((unsigned)cdiv(s.B, kSeqs), (unsigned)cdiv(s.H, kUnits), dirs);
        for (int step = s.T - 1; step >= (dh0 ? -1 : 0); --step)
            hipLaunchKernelGGL(lstm_step_back_kernel, grid, dim3(256), 0, q, s, step, (const float*)wt, c0, gates, cells, gy, ghn, gcn, dz, dc0, dh0);
        if (dx) {
            if (big_tiles(M, s.I, 1))
                hipLaunchKernelGGL(lstm_input_grad_kernel<128>, dim3((unsigned)cdiv(M, 128), (unsigned)cdiv(s.I, 128)), dim3(256), 0, q, s, (const float*)dz, w, dx);
            else
                hipLaunchKernelGGL(lstm_input_grad_kernel<64>, dim3((unsigned)cdiv(M, 64), (unsigned)cdiv(s.I, 64)), dim3(256), 0, q, s, (const float*)dz, w, dx);
        }
    }
    const int x_tiles = (int)cdiv(s.I, p.tile);
    const dim3 grid((unsigned)(x_tiles + cdiv(s.H, p.tile)), (unsigned)cdiv(4 * s.H, p.tile), (unsigned)(dirs * p.parts));
    if (p.tile == 128)
        hipLaunchKernelGGL(lstm_weight_grad_kernel<128>, grid, dim3(256), 0, q, s, (const float*)dz, x, y, h0, p.parts, p.per_part, x_tiles, dw_part, g->w_ih[0],
                           g->w_ih[1], g->w_hh[0], g->w_hh[1]);
    else
        hipLaunchKernelGGL(lstm_weight_grad_kernel<64>, grid, dim3(256), 0, q, s, (const float*)dz, x, y, h0, p.parts, p.per_part, x_tiles, dw_part, g->w_ih[0],
                           g->w_ih[1], g->w_hh[0], g->w_hh[1]);
    if (p.parts > 1)
        hipLaunchKernelGGL(lstm_join_kernel, dim3((unsigned)cdiv((i64)dirs * 4 * s.H * (s.I + s.H), 256)), dim3(256), 0, q, s, p.parts, (const float*)dw_part,
                           g->w_ih[0], g->w_ih[1], g->w_hh[0], g->w_hh[1]);
    if (p.bias_parts)
        hipLaunchKernelGGL(lstm_bias_grad_kernel, dim3((unsigned)cdiv(4 * s.H, 64), (unsigned)p.bias_parts, dirs), dim3(256), 0, q, s, (const float*)dz, p.bias_per, db_part);
    hipLaunchKernelGGL(lstm_bias_join_kernel, dim3((unsigned)cdiv(4 * s.H * dirs, 256)), dim3(256), 0, q, s, p.bias_parts, (const float*)db_part, g->b_ih[0], g->b_ih[1],
                       g->b_hh[0], g->b_hh[1]);
    return launched(who);
}

}  // extern "C"
