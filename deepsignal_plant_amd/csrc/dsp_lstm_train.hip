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
// behind it) is done by one product over all steps (53,248 rows of 512 inputs, 256 units, two directions: the gates of x 122 TFLOP/s, dx 128,
// dW 126; the library's product of 4,096 x 4,096 x 4,096 132).  The recurrence is one launch for up to 128 units, else a launch per step for both
// directions, its product, the gates and the states in one kernel: no workgroup waits for another.
//
// Layouts: x [B][T][I], y [B][T][dirs H], states [dirs][B][H]; gates and their gradients [dirs][B][T][4H]; cells and the h before
// each step [dirs][B][T][H].  So the products over all steps are plain: a row is m = b T + t.
#include "dsp_products.h"

using namespace dsp;

namespace {

struct Shape { int B, T, I, H, dirs; };
struct Weights { const float *w_ih[2], *w_hh[2], *b_ih[2], *b_hh[2]; };

// gates = W_ih x + b_ih + b_hh, all steps.  (2^30 rows of both directions are more workgroups than one axis of a grid takes)
template <int TILE, bool FAST>
__global__ __launch_bounds__(256, 3) void lstm_inputs_kernel(Shape s, uint32_t tiles, const float* __restrict__ x, Weights w, float* __restrict__ gates) {
    __shared__ __attribute__((aligned(16))) float lds[2 * half_floats<true, true, TILE>()];
    if (block_at() >= tiles) return;
    const int M = s.B * s.T, N = 4 * s.H, n_tiles = (N + TILE - 1) / TILE;
    const uint32_t tile = tile_of((uint32_t)block_at(), tiles);
    const int n0 = tile % (n_tiles * s.dirs), d = n0 / n_tiles, at = (n0 - d * n_tiles) * TILE, m0 = tile / (n_tiles * s.dirs) * TILE;
    f32x16 acc[TILE / 64][TILE / 64] = {};
    product<true, true, TILE, FAST>({x, M, s.I}, {w.w_ih[d], N, s.I}, m0, at, 0, s.I, lds, acc, Nothing());
    float* out = gates + (i64)d * M * N;
    each<TILE>(acc, m0, M, at, N, [&](int m, int n, float v) { out[(i64)m * N + n] = v + (w.b_ih[d][n] + w.b_hh[d][n]); });
}

// dx = sum over directions of dz W_ih
template <int TILE, bool FAST> __global__ __launch_bounds__(256, 3) void lstm_input_grad_kernel(Shape s, const float* __restrict__ dz, Weights w, float* __restrict__ dx) {
    __shared__ __attribute__((aligned(16))) float lds[2 * half_floats<true, false, TILE>()];
    const int M = s.B * s.T, K = 4 * s.H, n_tiles = (s.I + TILE - 1) / TILE;
    const uint32_t tile = tile_of(blockIdx.x, gridDim.x);
    const int n0 = tile % n_tiles * TILE, m0 = tile / n_tiles * TILE;
    f32x16 acc[TILE / 64][TILE / 64] = {};
    for (int d = 0; d < s.dirs; ++d)
        product<true, false, TILE, FAST>({dz + (i64)d * M * K, M, K}, {w.w_ih[d], K, s.I}, m0, n0, 0, K, lds, acc, Nothing());
    each<TILE>(acc, m0, M, n0, s.I, [&](int m, int n, float v) { dx[(i64)m * s.I + n] = v; });
}

// dW of both weights and db: tiles of [4H][I] and [4H][H], the sum over m in parts;  part [parts][dirs][4H][I + H + 1]
template <int TILE, bool FAST>
__global__ __launch_bounds__(256) void lstm_weight_grad_kernel(Shape s, const float* __restrict__ dz, const float* __restrict__ x, const float* __restrict__ h_before,
                                                               int per_part, float* __restrict__ part) {
    __shared__ __attribute__((aligned(16))) float lds[2 * half_floats<false, false, TILE>()];
    const int M = 4 * s.H, K = s.B * s.T, m_tiles = (M + TILE - 1) / TILE, x_tiles = (s.I + TILE - 1) / TILE, n_tiles = x_tiles + (s.H + TILE - 1) / TILE;
    uint32_t tile = tile_of(blockIdx.x, gridDim.x);
    const int nt = tile % n_tiles;
    tile /= n_tiles;
    const int m0 = tile % m_tiles * TILE, dq = tile / m_tiles, d = dq % s.dirs, q = dq / s.dirs;
    const bool of_x = nt < x_tiles;
    const int n0 = (of_x ? nt : nt - x_tiles) * TILE, N = of_x ? s.I : s.H, cols = s.I + s.H + 1;
    const int k0 = q * per_part, k1 = k0 + per_part < K ? k0 + per_part : K;
    const Matrix a = {dz + (i64)d * K * M, K, M}, b = {of_x ? x : h_before + (i64)d * K * s.H, K, N};
    f32x16 acc[TILE / 64][TILE / 64] = {};
    float* out = part + (i64)dq * M * cols;
    if (nt == 0) {   // these see every dz of their rows once: db on the way
        RowSums<TILE> sums;
        product<false, false, TILE, FAST>(a, b, m0, n0, k0, k1, lds, acc, sums);
        sums.store(lds, [&](int row, float v) {
            if (m0 + row < M) out[(i64)(m0 + row) * cols + cols - 1] = v;
        });
    } else
        product<false, false, TILE, FAST>(a, b, m0, n0, k0, k1, lds, acc, Nothing());
    each<TILE>(acc, m0, M, n0, N, [&](int m, int n, float v) { out[(i64)m * cols + n + (of_x ? 0 : s.I)] = v; });
}
struct Grads { float *w_ih[2], *w_hh[2], *b_ih[2], *b_hh[2]; };
// the parts in order, and the gradients apart
__global__ __launch_bounds__(256) void lstm_join_kernel(Shape s, int parts, const float* __restrict__ part, Grads g) {
    const int cols = s.I + s.H + 1;
    const i64 one = (i64)4 * s.H * cols, i = (i64)blockIdx.x * 256 + threadIdx.x;
    if (i >= one * s.dirs) return;
    float v = 0.0f;
    for (int q = 0; q < parts; ++q) v += part[q * one * s.dirs + i];
    const int d = i >= one;
    const i64 j = i - d * one, m = j / cols;
    const int n = (int)(j - m * cols);
    if (n < s.I) g.w_ih[d][m * s.I + n] = v;
    else if (n < s.I + s.H) g.w_hh[d][m * s.H + n - s.I] = v;
    else {
        g.b_ih[d][m] = v;   // both biases are added to the same place
        g.b_hh[d][m] = v;
    }
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

// ---- the recurrence of up to 128 units: all steps in one launch --------------------------------------------------------------
// The recurrent weights of a direction fit a workgroup's registers then (256 KB of 512): a workgroup takes 4 sequences of one
// direction through all steps, h (forward) or dz (backward) passing through LDS from step to step.  v_mfma_f32_4x4x1 makes 4
// sequences by 64 columns of one k, the whole of its work useful where the 16 rows of the larger ones would be mostly padding: its
// 16 blocks all take the same 4 x 1 of A (broadcast from block `k mod 16`, so one register of A serves 16 k) and 4 columns of W
// each.  What bounds it is the matrix instructions' time (2,048 cycles a step at 128 units) and, behind them, one turn through LDS
// and the gates: 32 sequences of 128 units, 256 steps, both directions: 390 us forward and 372 back, 1.5 a step, of which the matrix
// instructions are 0.85 and the gates 0.16.  A launch per step (below) costs 4.5 us instead, at any size: 1.15 ms.
//
// N: 16s of units that the registers are for (8, 4 or 2); units beyond H have weights of zero.
constexpr int kWholeUnits = 128;

// acc[0] = sum over k of A[4][k] W[k][lane]; a: k x 4 in LDS, 16 N values of k
template <int N> __device__ __forceinline__ f32x4 whole_product(const float* a, const float (&w)[16 * N]) {
    const int lane = threadIdx.x & 63;
    f32x4 acc[4] = {};
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = a[i * 64 + lane];
#pragma unroll
    for (int i = 0; i < N; ++i) {
#define DSP_K(b) acc[b & 3] = __builtin_amdgcn_mfma_f32_4x4x1f32(v[i], w[i * 16 + b], acc[b & 3], 4, b, 0)
        DSP_K(0); DSP_K(1); DSP_K(2); DSP_K(3); DSP_K(4); DSP_K(5); DSP_K(6); DSP_K(7);
        DSP_K(8); DSP_K(9); DSP_K(10); DSP_K(11); DSP_K(12); DSP_K(13); DSP_K(14); DSP_K(15);
#undef DSP_K
    }
    return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}
// What has been loaded arrives here, before the stores that follow.  Loads and stores are counted together and in order: a wait behind stores, where the
// values are used, would be one for the stores as well, a turn to memory in every step.
template <class T> __device__ __forceinline__ void arrived(T& x) { asm volatile("" : "+v"(x)); }
// x[i] of 16-lane row r -> x[r] of row i: what a lane has for 4 sequences becomes what it has for 4 gates
__device__ __forceinline__ void turn(f32x4& x) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(x[i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {   // halves: rows 2 and 3 of v[i] against rows 0 and 1 of v[i + 2]
        const u32x2 y = __builtin_amdgcn_permlane32_swap(v[i], v[i + 2], false, false);
        v[i] = y[0];
        v[i + 2] = y[1];
    }
#pragma unroll
    for (int i = 0; i < 4; i += 2) {   // rows 1 and 3 of v[i] against rows 0 and 2 of v[i + 1]
        const u32x2 y = __builtin_amdgcn_permlane16_swap(v[i], v[i + 1], false, false);
        v[i] = y[0];
        v[i + 1] = y[1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(v[i]);
}

// A wave for every 16 units: in the product lane = gate x 16 + unit and 4 sequences a lane, then lane = sequence x 16 + unit and 4 gates.
template <int N>
__global__ __launch_bounds__(64 * N) void lstm_whole_kernel(Shape s, Weights weights, const float* __restrict__ h0, const float* __restrict__ c0, float* gates, float* cells,
                                                            float* h_before, float* __restrict__ y, float* __restrict__ hn, float* __restrict__ cn, int save) {
    __shared__ __attribute__((aligned(16))) float lds[N * 16 * 64 > 2 * N * 64 ? N * 16 * 64 : 2 * N * 64];
    const int B = s.B, T = s.T, H = s.H, d = blockIdx.x % s.dirs, b0 = blockIdx.x / s.dirs * 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, unit = wave * 16 + (lane & 15), part = lane >> 4;
    const bool real = unit < H;
    const int uc = real ? unit : H - 1;
    // the weights of column (gate part, unit): a row of W_hh, which other lanes load in whole lines
    float w[16 * N];
    {
        const float* w_hh = weights.w_hh[d];
        float* mine = lds + wave * 64 * 16;   // 64 rows of 16 values of k
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {   // 4 rows at a time
                const int row = j * 4 + (lane >> 4), k = i * 16 + (lane & 15), u = wave * 16 + (row & 15);
                mine[row * 16 + ((lane & 15) ^ (row & 15))] = u < H && k < H ? w_hh[((i64)(row >> 4) * H + u) * H + k] : 0.0f;
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int e = 0; e < 16; ++e) w[i * 16 + e] = mine[lane * 16 + (e ^ (lane & 15))];
            __builtin_amdgcn_wave_barrier();
        }
    }
    const i64 b = b0 + part < B ? b0 + part : B - 1;   // the lane's sequence behind the turn
    const i64 at = ((i64)d * B + b) * H + uc, first = ((i64)d * B + b) * T;
    const bool store = real && b0 + part < B;
    i64 in[4];   // rows of the 4 sequences in the product
#pragma unroll
    for (int r = 0; r < 4; ++r) in[r] = (((i64)d * B + (b0 + r < B ? b0 + r : B - 1)) * T * 4 + part) * H + uc;
    float c = c0 ? c0[at] : 0.0f, h = h0 ? h0[at] : 0.0f;
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * N * 64; i += blockDim.x) lds[i] = 0.0f;   // k beyond the units
    __syncthreads();
    lds[unit * 4 + part] = real ? h : 0.0f;
    f32x4 next;
    const int t0 = d ? T - 1 : 0, dt = d ? -1 : 1;
#pragma unroll
    for (int r = 0; r < 4; ++r) next[r] = gates[in[r] + (i64)t0 * 4 * H];
    float* gates_at = gates + (first + t0) * 4 * H + unit;
    float *cells_at = cells + (first + t0) * H + unit, *h_at = h_before + (first + t0) * H + unit, *y_at = y + ((b * T + t0) * s.dirs + d) * H + unit;
    const i64 move = (i64)dt * H;
    // A step's values are written while the next one's product is computed, where registers are left for them (389 us in place of 400)
    constexpr bool LATE = N == 8;
    float i, f, g, o, h_first = h;
    auto put = [&](int step) {   // what a step has computed; one at a time
        if (store) {
            *y_at = h;
            if (save) {
                if (step == 0) *h_at = h_first;
                gates_at[0] = i;
                gates_at[H] = f;
                gates_at[2 * H] = g;
                gates_at[3 * H] = o;
                *cells_at = c;
                if (step + 1 < T) h_at[move] = h;
            }
        }
        y_at += move * s.dirs;
        gates_at += move * 4;
        cells_at += move;
        h_at += move;
    };
    for (int step = 0; step < T; ++step) {
        const int t = t0 + step * dt;
        const f32x4 z0 = next;
        if (step + 1 < T)
#pragma unroll
            for (int r = 0; r < 4; ++r) next[r] = gates[in[r] + (i64)(t + dt) * 4 * H];
        __syncthreads();   // h of this step is there
        if (LATE && step) put(step - 1);
        f32x4 z = whole_product<N>(lds + (step & 1) * N * 64, w) + z0;
        turn(z);
        i = sigmoid(z[0]);
        f = sigmoid(z[1]);
        g = tanh_of(z[2]);
        o = sigmoid(z[3]);
        c = f * c + i * g;
        h = o * tanh_of(c);
        lds[((step & 1) ^ 1) * N * 64 + unit * 4 + part] = real ? h : 0.0f;   // its readers of the step before are behind this step's barrier
        arrived(next);
        if (!LATE) put(step);
    }
    if (LATE) put(T - 1);
    if (store) {
        hn[at] = h;
        cn[at] = c;
    }
}

// Backward: a wave for every gate and 64 units: it multiplies that gate's dz by its rows of W_hh; the 4 gates' sums meet in LDS, where a
// thread has one unit of one sequence.  M: 64s of units.
template <int N, int M>
__global__ __launch_bounds__(256 * M) void lstm_whole_back_kernel(Shape s, Weights weights, const float* __restrict__ c0, const float* __restrict__ gates,
                                                                  const float* __restrict__ cells, const float* __restrict__ gy, const float* __restrict__ ghn,
                                                                  const float* __restrict__ gcn, float* __restrict__ dz, float* __restrict__ dc0, float* __restrict__ dh0) {
    __shared__ float dz_lds[4 * N * 64], sums[4 * 4 * M * 64];   // [gate][k][sequence]; [gate][sequence][unit]
    const int B = s.B, T = s.T, H = s.H, d = blockIdx.x % s.dirs, b0 = blockIdx.x / s.dirs * 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, gate = wave & 3, column = (wave >> 2) * 64 + lane;
    float w[16 * N];
    {
        const float* w_hh = weights.w_hh[d] + (i64)gate * H * H;
#pragma unroll
        for (int k = 0; k < 16 * N; ++k) w[k] = k < H && column < H ? w_hh[(i64)k * H + column] : 0.0f;
    }
    const int unit = threadIdx.x % (64 * M), seq = threadIdx.x / (64 * M);
    const bool real = unit < H, store = real && b0 + seq < B;
    const int uc = real ? unit : H - 1;
    const i64 b = b0 + seq < B ? b0 + seq : B - 1, at = ((i64)d * B + b) * H + uc, first = ((i64)d * B + b) * T;
    const int t0 = d ? T - 1 : 0, dt = d ? -1 : 1;   // in time of the recurrence: step k is t0 + k dt
    for (int i = threadIdx.x; i < 4 * N * 64; i += 256 * M) dz_lds[i] = 0.0f;   // k beyond the units
    float dc = gcn ? gcn[at] : 0.0f, dh_end = ghn ? ghn[at] : 0.0f;
    float a[4], next[4], c_next = 0.0f, gy_next = 0.0f, c = cells[(first + t0 + (i64)(T - 1) * dt) * H + uc];
    const i64 last = first + t0 + (i64)(T - 1) * dt, move = (i64)dt * H;
    const float *gates_at = gates + last * 4 * H + uc, *cells_at = cells + (last - dt) * H + uc, *gy_at = gy ? gy + ((b * T + t0 + (i64)(T - 1) * dt) * s.dirs + d) * H + uc : nullptr;
    float* out = dz + last * 4 * H + unit;
    auto load = [&](int step) {   // gates, the cell before, gradient of y; from the last step down, one at a time
#pragma unroll
        for (int g = 0; g < 4; ++g) next[g] = gates_at[g * H];
        c_next = step ? *cells_at : c0 ? c0[at] : 0.0f;
        gy_next = gy ? *gy_at : 0.0f;
        gates_at -= move * 4;
        cells_at -= move;
        if (gy) gy_at -= move * s.dirs;
    };
    load(T - 1);
    for (int step = T - 1; step >= 0; --step) {
        const float c_before = c_next, gy_now = gy_next;
#pragma unroll
        for (int g = 0; g < 4; ++g) a[g] = next[g];
        if (step) load(step - 1);
        __syncthreads();   // dz of the step behind is there
        f32x4 p = {0.0f, 0.0f, 0.0f, 0.0f};
        if (step < T - 1) p = whole_product<N>(dz_lds + gate * N * 64, w);
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[(gate * 4 + r) * M * 64 + column] = p[r];
        __syncthreads();
        float dh = gy_now + dh_end;
        dh_end = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) dh += sums[(g * 4 + seq) * M * 64 + unit];
        const float tc = tanh_of(c), dcell = dc + dh * a[3] * (1.0f - tc * tc);
        float q[4];
        q[0] = dcell * a[2] * a[0] * (1.0f - a[0]);
        q[1] = dcell * c_before * a[1] * (1.0f - a[1]);
        q[2] = dcell * a[0] * (1.0f - a[2] * a[2]);
        q[3] = dh * tc * a[3] * (1.0f - a[3]);
        dc = dcell * a[1];
        c = c_before;
        if (real)
#pragma unroll
            for (int g = 0; g < 4; ++g) dz_lds[(g * N * 16 + unit) * 4 + seq] = q[g];
#pragma unroll
        for (int g = 0; g < 4; ++g) arrived(next[g]);
        arrived(c_next);
        arrived(gy_next);
        if (store)
#pragma unroll
            for (int g = 0; g < 4; ++g) out[g * H] = q[g];
        out -= move * 4;
    }
    if (dh0) {
        __syncthreads();
        const f32x4 p = whole_product<N>(dz_lds + gate * N * 64, w);
#pragma unroll
        for (int r = 0; r < 4; ++r) sums[(gate * 4 + r) * M * 64 + column] = p[r];
        __syncthreads();
        float dh = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) dh += sums[(g * 4 + seq) * M * 64 + unit];
        if (store) dh0[at] = dh;
    }
    if (store) dc0[at] = dc;
}

// ---- the recurrence of more units: a launch per step -------------------------------------------------------------------------
// By step_product: a workgroup has the 4 gates of 16 units forward, 16 units backward.  A step of both directions, 256 units: 512 sequences 11.4 us
// either way (47 TFLOP/s: a launch, its ramp and end are half of it).
// 16 units fastest, then sequences, then direction, a contiguous range for each die: with two directions it sees one of them, the states
// of its own sequences and whole lines of their gates
struct Place { int d, u0, b0; };
template <int S> __device__ __forceinline__ Place place_of(const Shape& s) {
    const uint32_t units = (s.H + 15) >> 4, seqs = (s.B + 16 * S - 1) / (16 * S);
    uint32_t i = tile_of(blockIdx.x, gridDim.x);
    Place p;
    p.u0 = i % units * 16;
    i /= units;
    p.b0 = i % seqs * (16 * S);
    p.d = i / seqs;
    return p;
}

// (One step of 16 sequences, 256 inputs and units, FUSED: 7.3 us for 4.4 MB, nearly all of them weights: a launch and two waits for memory.)
// gates: in W_ih x + b of all steps (FUSED: made here, from x); out (save) i, f, g, o.  cells: c of all steps (save), else of two steps
// in turn; h_before (save): h before each step
template <int S, bool WIDE, bool FUSED>
__global__ __launch_bounds__(256, 3) void lstm_step_kernel(Shape s, int step, Weights w, const float* __restrict__ x, const float* __restrict__ h0,
                                                        const float* __restrict__ c0, float* gates, float* cells, float* h_before, float* y,
                                                        float* __restrict__ hn, float* __restrict__ cn, int save) {
    __shared__ __attribute__((aligned(16))) float lds[step_floats<S, 4>()];
    const Place p = place_of<S>(s);
    const int d = p.d, B = s.B, T = s.T, H = s.H, t = d ? T - 1 - step : step, before = d ? t + 1 : t - 1, after = d ? t - 1 : t + 1;
    const int row = threadIdx.x >> 4, u = p.u0 + (threadIdx.x & 15);
    // what the gates need besides the product, on its way meanwhile
    float z[S][4], c[S];
    i64 at[S], m[S];
    const int uc = u < H ? u : H - 1;
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const i64 b = p.b0 + j * 16 + row < B ? p.b0 + j * 16 + row : B - 1;
        at[j] = ((i64)d * B + b) * H + uc;
        m[j] = ((i64)d * B + b) * T + t;
#pragma unroll
        for (int g = 0; g < 4; ++g) z[j][g] = FUSED ? w.b_ih[d][g * H + uc] + w.b_hh[d][g * H + uc] : gates[m[j] * 4 * H + g * H + uc];
        c[j] = 0.0f;
        if (step) c[j] = save ? cells[(m[j] + before - t) * H + uc] : cells[((step - 1) & 1) * (i64)s.dirs * B * H + at[j]];
        else if (c0) c[j] = c0[at[j]];
    }
    f32x4 acc[4][S] = {};
    auto sequence = [&](int i) -> i64 { return p.b0 + i < B ? p.b0 + i : B - 1; };   // rows behind the last: its values, which are not used
    auto column = [&](int i) -> uint32_t { return (i >> 4) * H + (p.u0 + (i & 15) < H ? p.u0 + (i & 15) : H - 1); };
    if (FUSED)
        step_product<S, 4, WIDE>(
            s.I, [&](int i) { return x + (sequence(i) * T + t) * s.I; }, w.w_ih[d], [&](int i) { return column(i) * (uint32_t)s.I * 4; }, lds, acc);
    if (step > 0 || h0)
        step_product<S, 4, WIDE>(
            H, [&](int i) { return step ? y + ((sequence(i) * T + before) * s.dirs + d) * H : h0 + ((i64)d * B + sequence(i)) * H; }, w.w_hh[d],
            [&](int i) { return column(i) * (uint32_t)H * 4; }, lds, acc);
    float sum[S][4];
    step_join<S, 4>(acc, lds, sum);
    if (u >= H) return;
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const i64 b = p.b0 + j * 16 + row;
        if (b >= B) continue;
        const float i = sigmoid(z[j][0] + sum[j][0]), f = sigmoid(z[j][1] + sum[j][1]), g = tanh_of(z[j][2] + sum[j][2]), o = sigmoid(z[j][3] + sum[j][3]);
        const float cell = f * c[j] + i * g, h = o * tanh_of(cell);
        if (save) {
            float* q = gates + m[j] * 4 * H + u;
            q[0] = i;
            q[H] = f;
            q[2 * H] = g;
            q[3 * H] = o;
            cells[m[j] * H + u] = cell;
            if (step == 0) h_before[m[j] * H + u] = h0 ? h0[at[j]] : 0.0f;
            if (step < T - 1) h_before[(m[j] + after - t) * H + u] = h;
        } else if (step < T - 1)
            cells[(step & 1) * (i64)s.dirs * B * H + at[j]] = cell;
        y[((b * T + t) * s.dirs + d) * H + u] = h;
        if (step == T - 1) {
            hn[at[j]] = h;
            cn[at[j]] = cell;
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
template <int S, bool WIDE>
__global__ __launch_bounds__(256, 3) void lstm_step_back_kernel(Shape s, int step, const float* __restrict__ w_hh_t, const float* __restrict__ c0,
                                                                const float* __restrict__ gates, const float* __restrict__ cells, const float* __restrict__ gy,
                                                                const float* __restrict__ ghn, const float* __restrict__ gcn, float* dz, float* dc, float* dh0) {
    __shared__ __attribute__((aligned(16))) float lds[step_floats<S, 1>()];
    const Place p = place_of<S>(s);
    const int d = p.d, B = s.B, T = s.T, H = s.H, t = d ? T - 1 - step : step, before = d ? t + 1 : t - 1, after = d ? t - 1 : t + 1;
    const int row = threadIdx.x >> 4, u = p.u0 + (threadIdx.x & 15), uc = u < H ? u : H - 1;
    float gate[S][4], c[S], c_before[S], dct[S], dh[S];
    i64 at[S], m[S];
#pragma unroll
    for (int j = 0; j < S; ++j) {
        const i64 b = p.b0 + j * 16 + row < B ? p.b0 + j * 16 + row : B - 1;
        at[j] = ((i64)d * B + b) * H + uc;
        m[j] = ((i64)d * B + b) * T + t;
        dh[j] = 0.0f;
        if (step < 0) continue;
#pragma unroll
        for (int g = 0; g < 4; ++g) gate[j][g] = gates[m[j] * 4 * H + g * H + uc];
        c[j] = cells[m[j] * H + uc];
        c_before[j] = step ? cells[(m[j] + before - t) * H + uc] : c0 ? c0[at[j]] : 0.0f;
        dct[j] = step < T - 1 ? dc[at[j]] : gcn ? gcn[at[j]] : 0.0f;
        if (step == T - 1 && ghn) dh[j] = ghn[at[j]];
        if (gy) dh[j] += gy[((b * T + t) * s.dirs + d) * H + uc];
    }
    f32x4 acc[1][S] = {};
    if (step < T - 1)
        step_product<S, 1, WIDE>(
            4 * H, [&](int i) { return dz + (((i64)d * B + (p.b0 + i < B ? p.b0 + i : B - 1)) * T + after) * 4 * H; }, w_hh_t + (i64)d * H * 4 * H,
            [&](int i) { return (uint32_t)(p.u0 + i < H ? p.u0 + i : H - 1) * 16 * H; }, lds, acc);
    float sum[S][1];
    step_join<S, 1>(acc, lds, sum);
    if (u >= H) return;
#pragma unroll
    for (int j = 0; j < S; ++j) {
        if (p.b0 + j * 16 + row >= B) continue;
        dh[j] += sum[j][0];
        if (step < 0) {
            dh0[at[j]] = dh[j];
            continue;
        }
        const float i = gate[j][0], f = gate[j][1], g = gate[j][2], o = gate[j][3], tc = tanh_of(c[j]);
        const float dcell = dct[j] + dh[j] * o * (1.0f - tc * tc);
        float* q = dz + m[j] * 4 * H + u;
        q[0] = dcell * g * i * (1.0f - i);
        q[H] = dcell * c_before[j] * f * (1.0f - f);
        q[2 * H] = dcell * i * (1.0f - g * g);
        q[3 * H] = dh[j] * tc * o * (1.0f - o);
        dc[at[j]] = dcell * f;
    }
}

// ---- the same of many sequences: tiles of 128 or 64 with both operands shared by the workgroup's waves --------------------------
// Bound by the matrix instructions and, before and behind them, by memory: gates, cells and states, 100 MB a step of 4,096 sequences of 256 units
// in both directions: 57 us forward (75 TFLOP/s, 1.8 TB/s) and 65 back, by the tiles above 71 and 68.
// Forward: 128 sequences by the 4 gates of 32 units; a wave has 32 sequences, a lane the 4 gates of one unit of 16 of them, so that the gates
// meet in registers.  They begin as what the product is added to.
__global__ __launch_bounds__(256, 2) void lstm_tile_step_kernel(Shape s, int step, Weights w, const float* __restrict__ h0, const float* __restrict__ c0, float* gates, float* cells,
                                                                float* h_before, float* y, float* __restrict__ hn, float* __restrict__ cn, int save) {
    __shared__ __attribute__((aligned(16))) float lds[2 * half_floats<true, true, 128>()];
    const int B = s.B, T = s.T, H = s.H, units = (H + 31) >> 5, seqs = (B + 127) >> 7;
    uint32_t tile = tile_of(blockIdx.x, gridDim.x);
    const int u0 = tile % units * 32;
    tile /= units;
    const int b0 = tile % seqs * 128, d = tile / seqs;
    const int t = d ? T - 1 - step : step, before = d ? t + 1 : t - 1, after = d ? t - 1 : t + 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, u = u0 + (lane & 31), uc = u < H ? u : H - 1;
    auto sequence = [&](int r) { return b0 + wave * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3); };
    f32x16 acc[1][4];
    float c[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const i64 b = sequence(r) < B ? sequence(r) : B - 1, at = ((i64)d * B + b) * H + uc, m = ((i64)d * B + b) * T + t;
#pragma unroll
        for (int g = 0; g < 4; ++g) acc[0][g][r] = gates[m * 4 * H + g * H + uc];
        c[r] = step ? save ? cells[(m + before - t) * H + uc] : cells[((step - 1) & 1) * (i64)s.dirs * B * H + at] : c0 ? c0[at] : 0.0f;
    }
    auto row_of_w = [&](int row) { return (row >> 5) * H + (row & 31); };   // a unit behind the last is another gate's or zeros, which are not used
    const Matrix wm = {w.w_hh[d], 4 * H, H};
    if (step) product<true, true, 128, true>(Matrix{y + ((i64)before * s.dirs + d) * H, B, T * s.dirs * H}, wm, b0, u0, 0, H, lds, acc, Nothing(), row_of_w);
    else if (h0) product<true, true, 128, true>(Matrix{h0 + (i64)d * B * H, B, H}, wm, b0, u0, 0, H, lds, acc, Nothing(), row_of_w);
    if (u >= H) return;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const i64 b = sequence(r);
        if (b >= B) continue;
        const i64 at = ((i64)d * B + b) * H + u, m = ((i64)d * B + b) * T + t;
        const float i = sigmoid(acc[0][0][r]), f = sigmoid(acc[0][1][r]), g = tanh_of(acc[0][2][r]), o = sigmoid(acc[0][3][r]);
        const float cell = f * c[r] + i * g, h = o * tanh_of(cell);
        if (save) {
            float* q = gates + m * 4 * H + u;
            q[0] = i;
            q[H] = f;
            q[2 * H] = g;
            q[3 * H] = o;
            cells[m * H + u] = cell;
            if (step == 0) h_before[m * H + u] = h0 ? h0[at] : 0.0f;
            if (step < T - 1) h_before[(m + after - t) * H + u] = h;
        } else if (step < T - 1)
            cells[(step & 1) * (i64)s.dirs * B * H + at] = cell;
        y[((b * T + t) * s.dirs + d) * H + u] = h;
        if (step == T - 1) {
            hn[at] = h;
            cn[at] = cell;
        }
    }
}

// Backward: 64 sequences by 64 units, a wave 32 by 32
__global__ __launch_bounds__(256, 4) void lstm_tile_back_kernel(Shape s, int step, const float* __restrict__ w_hh_t, const float* __restrict__ c0, const float* __restrict__ gates,
                                                                const float* __restrict__ cells, const float* __restrict__ gy, const float* __restrict__ ghn,
                                                                const float* __restrict__ gcn, float* dz, float* dc, float* dh0) {
    __shared__ __attribute__((aligned(16))) float lds[2 * half_floats<true, true, 64>()];
    const int B = s.B, T = s.T, H = s.H, units = (H + 63) >> 6, seqs = (B + 63) >> 6;
    uint32_t tile = tile_of(blockIdx.x, gridDim.x);
    const int u0 = tile % units * 64;
    tile /= units;
    const int b0 = tile % seqs * 64, d = tile / seqs;
    const int t = d ? T - 1 - step : step, before = d ? t + 1 : t - 1, after = d ? t - 1 : t + 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, u = u0 + (wave & 1) * 32 + (lane & 31);
    auto sequence = [&](int r) { return b0 + (wave >> 1) * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3); };
    f32x16 acc[1][1] = {};
    if (step < T - 1)
        product<true, true, 64, true>(Matrix{dz + ((i64)d * B * T + after) * 4 * H, B, T * 4 * H}, Matrix{w_hh_t + (i64)d * H * 4 * H, H, 4 * H}, b0, u0, 0, 4 * H, lds, acc, Nothing());
    if (u >= H) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {   // 4 rows at a time, the loads of one on their way together
        float a[4][4], c[4], c_before[4], dct[4], dh[4];
        i64 at[4], m[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const i64 b = sequence(q * 4 + e) < B ? sequence(q * 4 + e) : B - 1;
            at[e] = ((i64)d * B + b) * H + u;
            m[e] = ((i64)d * B + b) * T + t;
            dh[e] = 0.0f;
            if (step < 0) continue;
#pragma unroll
            for (int g = 0; g < 4; ++g) a[e][g] = gates[m[e] * 4 * H + g * H + u];
            c[e] = cells[m[e] * H + u];
            c_before[e] = step ? cells[(m[e] + before - t) * H + u] : c0 ? c0[at[e]] : 0.0f;
            dct[e] = step < T - 1 ? dc[at[e]] : gcn ? gcn[at[e]] : 0.0f;
            if (step == T - 1 && ghn) dh[e] = ghn[at[e]];
            if (gy) dh[e] += gy[((b * T + t) * s.dirs + d) * H + u];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (sequence(q * 4 + e) >= B) continue;
            dh[e] += acc[0][0][q * 4 + e];
            if (step < 0) {
                dh0[at[e]] = dh[e];
                continue;
            }
            const float i = a[e][0], f = a[e][1], g = a[e][2], o = a[e][3], tc = tanh_of(c[e]);
            const float dcell = dct[e] + dh[e] * o * (1.0f - tc * tc);
            float* z = dz + m[e] * 4 * H + u;
            z[0] = dcell * g * i * (1.0f - i);
            z[H] = dcell * c_before[e] * f * (1.0f - f);
            z[2 * H] = dcell * i * (1.0f - g * g);
            z[3 * H] = dh[e] * tc * o * (1.0f - o);
            dc[at[e]] = dcell * f;
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
const char* bad_lstm(i64 B, i64 T, i64 I, i64 H, int dirs) {
    if (dirs != 1 && dirs != 2) return "one direction or two";
    if (B < 0 || T < 1 || I < 1 || H < 1) return "sizes must be positive (the batch may be empty)";
    if (I > 16384 || H > 8192) return "at most 16,384 inputs and 8,192 units";
    if (B > (1 << 22) || T > (1 << 22) || B * T >= (1ll << 30)) return "at most 2^22 sequences, 2^22 steps and 2^30 of both";
    if (B * H >= (1ll << 31)) return "at most 2^31 - 1 values in a state";   // a step's launch: a thread for each, fewer than 2^32
    if (B * T * (H > I ? H : I) >= (1ll << 37)) return "the layer's activations would not fit any device";
    return nullptr;
}
// 16-sequence blocks of a step's workgroup: two where that leaves every CU a workgroup.  More would take registers and LDS from a third
// workgroup on a CU (4 blocks: 12.3 against 11.3 us at 512 sequences of 256 units, the same at 4,096)
int step_blocks(const Shape& s) { return cdiv(s.B, 32) * cdiv(s.H, 16) * s.dirs >= 256 ? 2 : 1; }

// Forward, many sequences of more than 64 units: 4 at a time pass a CU in so many turns that the step's larger tiles are faster, from 2,048 in
// both directions on (13 steps of training, whole and by steps: 128 units 1,536 sequences 178 and 176 us, 2,048: 228 and 232, 3,072: 336 and 302,
// 16,384: 1,797 and 1,220; 96 units 1,536: 146 and 147, 2,048: 197 and 165; 72 units 1,536: 132 and 133, 2,048: 172 and 164).
// Backward the whole form stays ahead (2,288 and 2,454 us at 16,384 of 128), and up to 64 units it does in both (530 and 564 forward at 16,384 of 64).
bool whole_forward(const Shape& s) { return s.H <= kWholeUnits && (s.H <= 64 || cdiv(s.B, 4) * s.dirs < 1024); }

// The forms of many sequences, where the tiles are a workgroup for every CU (forward, whose tiles are larger) or two.  13 steps of both directions, all
// that belongs to a pass: 2,048 sequences of 1,024 units forward 4,676 -> 3,854 us, back 9,395 -> 7,785; of 256 units, forward 256 tiles, 876 -> 837;
// 1,024 of 256, 128 tiles, 508 against 581, and 2,048 of 256 back, 256 tiles, 1,635 against 1,740.
bool tile_forward(const Shape& s) { return s.H % kStep == 0 && cdiv(s.B, 128) * cdiv(s.H, 32) * s.dirs >= 256 && 128ll * s.T * s.dirs * s.H < (1ll << 29); }
bool tile_backward(const Shape& s) { return s.H % 4 == 0 && cdiv(s.B, 64) * cdiv(s.H, 64) * s.dirs >= 512 && 64ll * s.T * 4 * s.H < (1ll << 29); }

// the sum over m of the weights' gradients
Split weight_split(const dsp_lstm_layer* l) { return split_of(l->batch * l->steps, 4 * l->hidden, l->input, l->hidden, l->directions); }

}  // namespace

extern "C" {

int32_t dsp_lstm_forward(void* stream, const dsp_lstm_layer* l, const float* x, const float* h0, const float* c0, float* y, float* hn, float* cn, float* gates,
                         float* cells, int32_t save) {
    const char* who = "dsp_lstm_forward";
    if (!l) return refuse(who, "NULL layer");
    if (const char* why = bad_lstm(l->batch, l->steps, l->input, l->hidden, l->directions)) return refuse(who, why);
    Weights w = {};
    bool hidden_wide = l->hidden % 4 == 0 && aligned16(y) && aligned16(h0), input_wide = l->input % 4 == 0 && aligned16(x);
    for (int d = 0; d < l->directions; ++d) {
        w.w_ih[d] = l->w_ih[d]; w.w_hh[d] = l->w_hh[d]; w.b_ih[d] = l->b_ih[d]; w.b_hh[d] = l->b_hh[d];
        if (!w.w_ih[d] || !w.w_hh[d] || !w.b_ih[d] || !w.b_hh[d]) return refuse(who, "NULL weight");
        hidden_wide = hidden_wide && aligned16(w.w_hh[d]);
        input_wide = input_wide && aligned16(w.w_ih[d]);
    }
    if (l->batch == 0) return DSP_OK;
    const Shape s = {(int)l->batch, (int)l->steps, (int)l->input, (int)l->hidden, l->directions};
    const bool fused = s.T == 1;   // a single step makes the gates of x itself: nothing is gained by a product of its own
    if (!x || !y || !hn || !cn || ((!gates || !cells) && (!fused || save))) return refuse(who, "NULL pointer");
    hipStream_t q = (hipStream_t)stream;
    const i64 M = l->batch * l->steps, N = 4ll * s.H, all = s.dirs * M * s.H;
    if (!fused) {
        const int tile = tile_for(M, N * s.dirs);
        const bool fast = input_wide && s.I % kStep == 0;   // a line's last 16 values are all its own
        const i64 tiles = cdiv(M, tile) * cdiv(N, tile) * s.dirs;
        DSP_TILES_ON(lstm_inputs_kernel, tile, fast, grid_of(tiles), q, s, (uint32_t)tiles, x, w, gates);
    }
    if (!fused && whole_forward(s)) {
        const dim3 grid((unsigned)(cdiv(s.B, 4) * s.dirs)), block(64 * (unsigned)cdiv(s.H, 16));
        if (s.H > 64) hipLaunchKernelGGL(lstm_whole_kernel<8>, grid, block, 0, q, s, w, h0, c0, gates, cells, cells + all, y, hn, cn, save);
        else if (s.H > 32) hipLaunchKernelGGL(lstm_whole_kernel<4>, grid, block, 0, q, s, w, h0, c0, gates, cells, cells + all, y, hn, cn, save);
        else hipLaunchKernelGGL(lstm_whole_kernel<2>, grid, block, 0, q, s, w, h0, c0, gates, cells, cells + all, y, hn, cn, save);
        return launched(who);
    }
    if (!fused && tile_forward(s) && hidden_wide) {
        const dim3 grid((unsigned)(cdiv(s.B, 128) * cdiv(s.H, 32) * s.dirs));
        for (int step = 0; step < s.T; ++step)
            hipLaunchKernelGGL(lstm_tile_step_kernel, grid, dim3(256), 0, q, s, step, w, h0, c0, gates, cells, cells + all, y, hn, cn, save);
        return launched(who);
    }
    const int S = step_blocks(s);
    const bool wide = hidden_wide && (!fused || input_wide);
    const dim3 grid((unsigned)(cdiv(s.B, 16 * S) * cdiv(s.H, 16) * s.dirs));
    for (int step = 0; step < s.T; ++step) {
#define DSP_STEP(S, W, F) hipLaunchKernelGGL((lstm_step_kernel<S, W, F>), grid, dim3(256), 0, q, s, step, w, x, h0, c0, gates, cells, cells + all, y, hn, cn, save)
#define DSP_STEP_OF(S)                                                                                       \
    do {                                                                                                     \
        if (fused) { if (wide) DSP_STEP(S, true, true); else DSP_STEP(S, false, true); }                     \
        else { if (wide) DSP_STEP(S, true, false); else DSP_STEP(S, false, false); }                         \
    } while (0)
        if (S == 2) DSP_STEP_OF(2);
        else DSP_STEP_OF(1);
#undef DSP_STEP_OF
#undef DSP_STEP
    }
    return launched(who);
}

int64_t dsp_lstm_workspace(const dsp_lstm_layer* l) {
    const char* who = "dsp_lstm_workspace";
    if (!l) return refuse(who, "NULL layer");
    if (const char* why = bad_lstm(l->batch, l->steps, l->input, l->hidden, l->directions)) return refuse(who, why);
    const Split p = weight_split(l);
    size_t bytes = align256((size_t)l->directions * l->hidden * 4 * l->hidden * 4);                                    // W_hh transposed
    bytes += align256((size_t)l->directions * l->steps * l->batch * 4 * l->hidden * 4);                                // dz
    return (int64_t)(bytes + align256((size_t)p.parts * l->directions * 4 * l->hidden * (l->input + l->hidden + 1) * 4));   // parts of dW and db
}

int32_t dsp_lstm_backward(void* stream, const dsp_lstm_layer* l, const float* x, const float* c0, const float* gates, const float* cells, const float* gy,
                          const float* ghn, const float* gcn, float* dx, float* dh0, float* dc0, const dsp_lstm_grads* g, void* workspace,
                          int64_t workspace_bytes) {
    const char* who = "dsp_lstm_backward";
    if (!l || !g) return refuse(who, "NULL layer");
    if (const char* why = bad_lstm(l->batch, l->steps, l->input, l->hidden, l->directions)) return refuse(who, why);
    const int dirs = l->directions;
    Weights w = {};
    Grads out = {};
    bool input_wide = l->input % 4 == 0 && aligned16(x);
    for (int d = 0; d < dirs; ++d) {
        w.w_ih[d] = l->w_ih[d];
        w.w_hh[d] = l->w_hh[d];
        out.w_ih[d] = g->w_ih[d]; out.w_hh[d] = g->w_hh[d]; out.b_ih[d] = g->b_ih[d]; out.b_hh[d] = g->b_hh[d];
        if (!w.w_ih[d] || !w.w_hh[d] || !out.w_ih[d] || !out.w_hh[d] || !out.b_ih[d] || !out.b_hh[d]) return refuse(who, "NULL weight or gradient");
        input_wide = input_wide && aligned16(w.w_ih[d]);
    }
    if (l->batch && (!x || !gates || !cells || !dc0)) return refuse(who, "NULL pointer");
    if (!workspace || workspace_bytes < dsp_lstm_workspace(l)) return refuse(who, "workspace too small (dsp_lstm_workspace)");
    if ((size_t)workspace & 255) return refuse(who, "the workspace must be aligned to 256 bytes");
    const Shape s = {(int)l->batch, (int)l->steps, (int)l->input, (int)l->hidden, dirs};
    const i64 M = (i64)s.B * s.T;
    const float* h_before = cells + dirs * M * s.H;
    const bool hidden_wide = s.H % 4 == 0 && aligned16(cells);
    const Split p = weight_split(l);
    char* ws = (char*)workspace;
    float* wt = (float*)ws;
    ws += align256((size_t)dirs * s.H * 4 * s.H * 4);
    float* dz = (float*)ws;
    ws += align256((size_t)dirs * s.T * s.B * 4 * s.H * 4);
    float* part = (float*)ws;
    hipStream_t q = (hipStream_t)stream;
    if (s.B) {
        if (s.H <= kWholeUnits) {
            const dim3 grid((unsigned)(cdiv(s.B, 4) * dirs));
            if (s.H > 64) hipLaunchKernelGGL((lstm_whole_back_kernel<8, 2>), grid, dim3(512), 0, q, s, w, c0, gates, cells, gy, ghn, gcn, dz, dc0, dh0);
            else if (s.H > 32) hipLaunchKernelGGL((lstm_whole_back_kernel<4, 1>), grid, dim3(256), 0, q, s, w, c0, gates, cells, gy, ghn, gcn, dz, dc0, dh0);
            else hipLaunchKernelGGL((lstm_whole_back_kernel<2, 1>), grid, dim3(256), 0, q, s, w, c0, gates, cells, gy, ghn, gcn, dz, dc0, dh0);
        } else {
            hipLaunchKernelGGL(lstm_transpose_kernel, dim3((unsigned)cdiv(s.H, 32), (unsigned)cdiv(4 * s.H, 32), dirs), dim3(256), 0, q, s.H, w, wt);
            const int S = step_blocks(s);
            const bool wide = s.H % 4 == 0;
            const bool tile = tile_backward(s);
            const dim3 tiles((unsigned)(cdiv(s.B, 64) * cdiv(s.H, 64) * dirs));
            const dim3 grid((unsigned)(cdiv(s.B, 16 * S) * cdiv(s.H, 16) * dirs));
            for (int step = s.T - 1; step >= (dh0 ? -1 : 0); --step) {
#define DSP_BACK(S, W) hipLaunchKernelGGL((lstm_step_back_kernel<S, W>), grid, dim3(256), 0, q, s, step, (const float*)wt, c0, gates, cells, gy, ghn, gcn, dz, dc0, dh0)
                if (tile) hipLaunchKernelGGL(lstm_tile_back_kernel, tiles, dim3(256), 0, q, s, step, (const float*)wt, c0, gates, cells, gy, ghn, gcn, dz, dc0, dh0);
                else if (S == 2) { if (wide) DSP_BACK(2, true); else DSP_BACK(2, false); }
                else { if (wide) DSP_BACK(1, true); else DSP_BACK(1, false); }
#undef DSP_BACK
            }
        }
        if (dx) {
            const int tile = tile_for(M, s.I);
            const bool fast = input_wide && s.H % 4 == 0;
            DSP_TILES(lstm_input_grad_kernel, tile, fast, cdiv(M, tile) * cdiv(s.I, tile), q, s, (const float*)dz, w, dx);
        }
    }
    const bool fast = input_wide && hidden_wide && (i64)p.per_part * 4 * (s.I > 4 * s.H ? s.I : 4 * s.H) < (1ll << 31);
    DSP_TILES(lstm_weight_grad_kernel, p.tile, fast, cdiv(4 * s.H, p.tile) * (cdiv(s.I, p.tile) + cdiv(s.H, p.tile)) * dirs * p.parts, q, s, (const float*)dz, x,
              h_before, p.per_part, part);
    hipLaunchKernelGGL(lstm_join_kernel, dim3((unsigned)cdiv((i64)dirs * 4 * s.H * (s.I + s.H + 1), 256)), dim3(256), 0, q, s, p.parts, (const float*)part, out);
    return launched(who);
}

}  // extern "C"
