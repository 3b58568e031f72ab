// dsp_linear.hip -- a fully connected layer with its gradient (fc_seq, fc_signal, fc1 and fc2 of models.py:147-161 in training).
//
//   y = x W^T + b          dx = dy W          dW = dy^T x          db = sum of dy over the rows
//
// Plain products, bound by the fp32 matrix instructions (dsp_products.h); db comes with dW: the workgroups that stage every dy once
// add it up on the way.  Where tiles are few, dW's sum over the rows and dx's over the outputs are split, and joined in order.
// (4,096 x 4,096 x 4,096: 126 TFLOP/s forward, the library's product 135; 53,248 x 512 x 256: 98 and 121; 16 x 4,096 x 4,096: 27 us, 2.5 TB/s of W)
#include "dsp_products.h"

using namespace dsp;

namespace {

struct Layer { int M, K, N; };   // rows, inputs, outputs

template <int TILE, bool FAST>
__global__ __launch_bounds__(256, 3) void linear_kernel(Layer l, const float* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b, float* __restrict__ y) {
    __shared__ __attribute__((aligned(16))) float lds[2 * half_floats<true, true, TILE>()];
    const int n_tiles = (l.N + TILE - 1) / TILE;
    const uint32_t tile = tile_of(blockIdx.x, gridDim.x);
    const int n0 = tile % n_tiles * TILE, m0 = tile / n_tiles * TILE;
    f32x16 acc[TILE / 64][TILE / 64] = {};
    product<true, true, TILE, FAST>({x, l.M, l.K}, {w, l.N, l.K}, m0, n0, 0, l.K, lds, acc, Nothing());
    each<TILE>(acc, m0, l.M, n0, l.N, [&](int m, int n, float v) { y[(i64)m * l.N + n] = v + (b ? b[n] : 0.0f); });
}

// Few tiles: smaller ones, whose 4 waves share k.  2^29 rows and more (of up to 16 outputs) are more workgroups than one axis of a grid takes
template <int S, int C, bool WIDE>
__global__ __launch_bounds__(256, 3) void linear_few_kernel(Layer l, uint32_t tiles, const float* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b,
                                                            float* __restrict__ y) {
    __shared__ __attribute__((aligned(16))) float lds[step_floats<S, C>()];
    if (block_at() >= tiles) return;
    const int n_tiles = (l.N + 16 * C - 1) / (16 * C);
    const uint32_t tile = tile_of((uint32_t)block_at(), tiles);
    const int n0 = tile % n_tiles * (16 * C), m0 = tile / n_tiles * (16 * S);
    f32x4 acc[C][S] = {};
    step_product<S, C, WIDE>(
        l.K, [&](int i) { return x + (i64)(m0 + i < l.M ? m0 + i : l.M - 1) * l.K; }, w,
        [&](int i) { return (uint32_t)(n0 + i < l.N ? n0 + i : l.N - 1) * (uint32_t)l.K * 4; }, lds, acc);
    float sum[S][C];
    step_join<S, C>(acc, lds, sum);
#pragma unroll
    for (int j = 0; j < S; ++j)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int m = m0 + j * 16 + (threadIdx.x >> 4), n = n0 + c * 16 + (threadIdx.x & 15);
            if (m < l.M && n < l.N) y[(i64)m * l.N + n] = sum[j][c] + (b ? b[n] : 0.0f);
        }
}

// dx, or with several parts of the sum over the outputs [parts][M][K]
template <int TILE, bool FAST>
__global__ __launch_bounds__(256, 3) void linear_input_grad_kernel(Layer l, const float* __restrict__ dy, const float* __restrict__ w, int per_part, float* __restrict__ dx) {
    __shared__ __attribute__((aligned(16))) float lds[2 * half_floats<true, false, TILE>()];
    const int m_tiles = (l.M + TILE - 1) / TILE, k_tiles = (l.K + TILE - 1) / TILE;
    uint32_t tile = tile_of(blockIdx.x, gridDim.x);
    const int k0 = tile % k_tiles * TILE;
    tile /= k_tiles;
    const int m0 = tile % m_tiles * TILE, q = tile / m_tiles, from = q * per_part, to = from + per_part < l.N ? from + per_part : l.N;
    dx += (i64)q * l.M * l.K;
    f32x16 acc[TILE / 64][TILE / 64] = {};
    product<true, false, TILE, FAST>({dy, l.M, l.N}, {w, l.N, l.K}, m0, k0, from, to, lds, acc, Nothing());
    each<TILE>(acc, m0, l.M, k0, l.K, [&](int m, int k, float v) { dx[(i64)m * l.K + k] = v; });
}

// The parts in order
__global__ __launch_bounds__(256) void linear_input_join_kernel(i64 n, int parts, const float* __restrict__ part, float* __restrict__ dx) {
    const i64 i = (i64)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float v = 0.0f;
    for (int q = 0; q < parts; ++q) v += part[q * n + i];
    dx[i] = v;
}

// One part: dW and db (or NULL).  Several: part [parts][N][K + 1], both of them
template <int TILE, bool FAST>
__global__ __launch_bounds__(256) void linear_weight_grad_kernel(Layer l, const float* __restrict__ dy, const float* __restrict__ x, int per_part, float* __restrict__ part, float* __restrict__ dw,
                                                                 float* __restrict__ db) {
    __shared__ __attribute__((aligned(16))) float lds[2 * half_floats<false, false, TILE>()];
    const int n_tiles = (l.N + TILE - 1) / TILE, k_tiles = (l.K + TILE - 1) / TILE, cols = part ? l.K + 1 : l.K;
    uint32_t tile = tile_of(blockIdx.x, gridDim.x);
    const int k0 = tile % k_tiles * TILE;
    tile /= k_tiles;
    const int n0 = tile % n_tiles * TILE, q = tile / n_tiles, from = q * per_part, to = from + per_part < l.M ? from + per_part : l.M;
    f32x16 acc[TILE / 64][TILE / 64] = {};
    float* out = part ? part + (i64)q * l.N * cols : dw;
    if (k0 == 0) {
        RowSums<TILE> sums;
        product<false, false, TILE, FAST>({dy, l.M, l.N}, {x, l.M, l.K}, n0, k0, from, to, lds, acc, sums);
        sums.store(lds, [&](int row, float v) {
            if (n0 + row >= l.N) return;
            if (part) out[(i64)(n0 + row) * cols + l.K] = v;
            else if (db) db[n0 + row] = v;
        });
    } else
        product<false, false, TILE, FAST>({dy, l.M, l.N}, {x, l.M, l.K}, n0, k0, from, to, lds, acc, Nothing());
    each<TILE>(acc, n0, l.N, k0, l.K, [&](int n, int k, float v) { out[(i64)n * cols + k] = v; });
}
__global__ __launch_bounds__(256) void linear_join_kernel(Layer l, int parts, const float* __restrict__ part, float* __restrict__ dw, float* __restrict__ db) {
    const int cols = l.K + 1;
    const i64 one = (i64)l.N * cols, i = (i64)blockIdx.x * 256 + threadIdx.x;
    if (i >= one) return;
    float v = 0.0f;
    for (int q = 0; q < parts; ++q) v += part[q * one + i];
    const int n = (int)(i / cols), k = (int)(i - (i64)n * cols);
    if (k < l.K) dw[(i64)n * l.K + k] = v;
    else if (db) db[n] = v;
}

const char* bad_linear(i64 m, i64 k, i64 n) {
    if (m < 0 || m >= (1ll << 30)) return "the number of rows must be within 0 .. 2^30 - 1";
    if (k < 1 || n < 1 || k > 16384 || n > 16384) return "inputs and outputs must be within 1 .. 16,384";
    return nullptr;
}

// the sum over the outputs in dx: in parts where its tiles are few, 128 of them each at least
Split input_split(i64 M, i64 K, i64 N) {
    Split q;
    q.tile = tile_for(M, K);
    i64 parts = cdiv(512, cdiv(M, q.tile) * cdiv(K, q.tile) + 1);
    if (parts > N / 128) parts = N / 128;
    if (parts < 1) parts = 1;
    q.per_part = (int)(cdiv(cdiv(N, parts), kStep) * kStep);
    q.parts = (int)cdiv(N, q.per_part);
    return q;
}
// The forward product by the form of few rows or columns: up to as many 64 x 64 tiles as there are CUs (1,000 x 1,000 x 1,000, 256 tiles: 30 us in
// place of 49; 8,192 x 512 x 256, 512 tiles: 39 and 27), or where a tile's columns would be mostly padding (65,536 x 256 x 2: 16 and 43)
bool few_tiles(const Layer& l) { return l.N <= 16 || cdiv(l.M, 64) * cdiv(l.N, 64) <= 256; }

struct Room { size_t weight, input; };   // of the workspace, which is never empty
Room room_of(i64 M, i64 K, i64 N) {
    const Split a = split_of(M, N, K, 0, 1), b = input_split(M, K, N);
    return Room{a.parts > 1 ? align256((size_t)a.parts * N * (K + 1) * 4) : 256, b.parts > 1 ? align256((size_t)b.parts * M * K * 4) : 0};
}

}  // namespace

extern "C" {

int32_t dsp_linear_forward(void* stream, int64_t rows, int64_t inputs, int64_t outputs, const float* x, const float* weight, const float* bias, float* y) {
    if (const char* why = bad_linear(rows, inputs, outputs)) return refuse("dsp_linear_forward", why);
    if (rows == 0) return DSP_OK;
    if (!x || !weight || !y) return refuse("dsp_linear_forward", "NULL pointer");
    const Layer l = {(int)rows, (int)inputs, (int)outputs};
    hipStream_t s = (hipStream_t)stream;
    if (few_tiles(l)) {
        const bool wide = l.K % 4 == 0 && aligned16(x) && aligned16(weight), narrow = l.N <= 16;
        const i64 across = narrow ? 1 : cdiv(l.N, 64);
        const int S = cdiv(l.M, 32) * across >= 256 ? 2 : 1;
#define DSP_FEW(S, C)                                                                                                                          \
    do {                                                                                                                                       \
        const uint32_t tiles = (uint32_t)(cdiv(l.M, 16 * S) * across);                                                                         \
        if (wide) hipLaunchKernelGGL((linear_few_kernel<S, C, true>), grid_of(tiles), dim3(256), 0, s, l, tiles, x, weight, bias, y);          \
        else hipLaunchKernelGGL((linear_few_kernel<S, C, false>), grid_of(tiles), dim3(256), 0, s, l, tiles, x, weight, bias, y);              \
    } while (0)
        if (narrow) { if (S == 2) DSP_FEW(2, 1); else DSP_FEW(1, 1); }
        else { if (S == 2) DSP_FEW(2, 4); else DSP_FEW(1, 4); }
#undef DSP_FEW
        return launched("dsp_linear_forward");
    }
    const int tile = tile_for(l.M, l.N);
    const bool fast = l.K % kStep == 0 && aligned16(x) && aligned16(weight);
    DSP_TILES(linear_kernel, tile, fast, cdiv(l.M, tile) * cdiv(l.N, tile), s, l, x, weight, bias, y);
    return launched("dsp_linear_forward");
}

int64_t dsp_linear_workspace(int64_t rows, int64_t inputs, int64_t outputs) {
    if (const char* why = bad_linear(rows, inputs, outputs)) return refuse("dsp_linear_workspace", why);
    const Room room = room_of(rows, inputs, outputs);
    return (int64_t)(room.weight + room.input);
}

int32_t dsp_linear_backward(void* stream, int64_t rows, int64_t inputs, int64_t outputs, const float* x, const float* weight, const float* grad_y, float* grad_x,
                            float* grad_weight, float* grad_bias, void* workspace, int64_t workspace_bytes) {
    const char* who = "dsp_linear_backward";
    if (const char* why = bad_linear(rows, inputs, outputs)) return refuse(who, why);
    if (!weight || !grad_weight || (rows && (!x || !grad_y))) return refuse(who, "NULL pointer");
    const Room room = room_of(rows, inputs, outputs);
    if (!workspace || workspace_bytes < (int64_t)(room.weight + room.input)) return refuse(who, "workspace too small (dsp_linear_workspace)");
    if ((size_t)workspace & 255) return refuse(who, "the workspace must be aligned to 256 bytes");
    const Layer l = {(int)rows, (int)inputs, (int)outputs};
    hipStream_t s = (hipStream_t)stream;
    if (grad_x && rows) {
        const Split p = input_split(l.M, l.K, l.N);
        const bool fast = l.N % kStep == 0 && l.K % 4 == 0 && aligned16(grad_y) && aligned16(weight);
        float* part = (float*)((char*)workspace + room.weight);
        DSP_TILES(linear_input_grad_kernel, p.tile, fast, cdiv(l.M, p.tile) * cdiv(l.K, p.tile) * p.parts, s, l, grad_y, weight, p.per_part, p.parts > 1 ? part : grad_x);
        if (p.parts > 1)
            hipLaunchKernelGGL(linear_input_join_kernel, dim3((unsigned)cdiv((i64)l.M * l.K, 256)), dim3(256), 0, s, (i64)l.M * l.K, p.parts, (const float*)part, grad_x);
    }
    const Split p = split_of(rows, outputs, inputs, 0, 1);
    const bool fast = l.N % 4 == 0 && l.K % 4 == 0 && aligned16(grad_y) && aligned16(x);
    float* part = p.parts > 1 ? (float*)workspace : nullptr;
    DSP_TILES(linear_weight_grad_kernel, p.tile, fast, cdiv(l.N, p.tile) * cdiv(l.K, p.tile) * p.parts, s, l, grad_y, x, p.per_part, part, grad_weight, grad_bias);
    if (part)
        hipLaunchKernelGGL(linear_join_kernel, dim3((unsigned)cdiv((i64)l.N * (l.K + 1), 256)), dim3(256), 0, s, l, p.parts, (const float*)part, grad_weight, grad_bias);
    return launched(who);
}

}  // extern "C"
