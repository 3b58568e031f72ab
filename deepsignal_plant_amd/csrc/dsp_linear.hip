// dsp_linear.hip -- a fully connected layer with its gradient (fc_seq, fc_signal, fc1 and fc2 of models.py:147-161 in training).
//
//   y = x W^T + b          dx = dy W          dW = dy^T x          db = sum of dy over the rows
//
// Plain products, bound by the fp32 matrix instructions (dsp_products.h); db comes with dW: the workgroups that stage every dy once
// add it up on the way.  dW's sum over the rows is split where its tiles are few, and joined in order.
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

template <int TILE, bool FAST>
__global__ __launch_bounds__(256, 3) void linear_input_grad_kernel(Layer l, const float* __restrict__ dy, const float* __restrict__ w, float* __restrict__ dx) {
    __shared__ __attribute__((aligned(16))) float lds[2 * half_floats<true, false, TILE>()];
    const int k_tiles = (l.K + TILE - 1) / TILE;
    const uint32_t tile = tile_of(blockIdx.x, gridDim.x);
    const int k0 = tile % k_tiles * TILE, m0 = tile / k_tiles * TILE;
    f32x16 acc[TILE / 64][TILE / 64] = {};
    product<true, false, TILE, FAST>({dy, l.M, l.N}, {w, l.N, l.K}, m0, k0, 0, l.N, lds, acc, Nothing());
    each<TILE>(acc, m0, l.M, k0, l.K, [&](int m, int k, float v) { dx[(i64)m * l.K + k] = v; });
}

// part [parts][N][K + 1]: dW and db
template <int TILE, bool FAST>
__global__ __launch_bounds__(256) void linear_weight_grad_kernel(Layer l, const float* __restrict__ dy, const float* __restrict__ x, int per_part, float* __restrict__ part) {
    __shared__ __attribute__((aligned(16))) float lds[2 * half_floats<false, false, TILE>()];
    const int n_tiles = (l.N + TILE - 1) / TILE, k_tiles = (l.K + TILE - 1) / TILE, cols = l.K + 1;
    uint32_t tile = tile_of(blockIdx.x, gridDim.x);
    const int k0 = tile % k_tiles * TILE;
    tile /= k_tiles;
    const int n0 = tile % n_tiles * TILE, q = tile / n_tiles, from = q * per_part, to = from + per_part < l.M ? from + per_part : l.M;
    f32x16 acc[TILE / 64][TILE / 64] = {};
    float* out = part + (i64)q * l.N * cols;
    if (k0 == 0) {
        RowSums<TILE> sums;
        product<false, false, TILE, FAST>({dy, l.M, l.N}, {x, l.M, l.K}, n0, k0, from, to, lds, acc, sums);
        sums.store(lds, [&](int row, float v) {
            if (n0 + row < l.N) out[(i64)(n0 + row) * cols + l.K] = v;
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

}  // namespace

extern "C" {

int32_t dsp_linear_forward(void* stream, int64_t rows, int64_t inputs, int64_t outputs, const float* x, const float* weight, const float* bias, float* y) {
    if (const char* why = bad_linear(rows, inputs, outputs)) return refuse("dsp_linear_forward", why);
    if (rows == 0) return DSP_OK;
    if (!x || !weight || !y) return refuse("dsp_linear_forward", "NULL pointer");
    const Layer l = {(int)rows, (int)inputs, (int)outputs};
    const int tile = tile_for(l.M, l.N);
    const bool fast = l.K % kStep == 0 && aligned16(x) && aligned16(weight);
    DSP_TILES(linear_kernel, tile, fast, cdiv(l.M, tile) * cdiv(l.N, tile), (hipStream_t)stream, l, x, weight, bias, y);
    return launched("dsp_linear_forward");
}

int64_t dsp_linear_workspace(int64_t rows, int64_t inputs, int64_t outputs) {
    if (const char* why = bad_linear(rows, inputs, outputs)) return refuse("dsp_linear_workspace", why);
    return (int64_t)align256((size_t)split_of(rows, outputs, inputs, 0, 1).parts * outputs * (inputs + 1) * 4);
}

int32_t dsp_linear_backward(void* stream, int64_t rows, int64_t inputs, int64_t outputs, const float* x, const float* weight, const float* grad_y, float* grad_x,
                            float* grad_weight, float* grad_bias, void* workspace, int64_t workspace_bytes) {
    const char* who = "dsp_linear_backward";
    if (const char* why = bad_linear(rows, inputs, outputs)) return refuse(who, why);
    if (!weight || !grad_weight || (rows && (!x || !grad_y))) return refuse(who, "NULL pointer");
    if (!workspace || workspace_bytes < dsp_linear_workspace(rows, inputs, outputs)) return refuse(who, "workspace too small (dsp_linear_workspace)");
    if ((size_t)workspace & 255) return refuse(who, "the workspace must be aligned to 256 bytes");
    const Layer l = {(int)rows, (int)inputs, (int)outputs};
    hipStream_t s = (hipStream_t)stream;
    if (grad_x && rows) {
        const int tile = tile_for(l.M, l.K);
        const bool fast = l.N % kStep == 0 && l.K % 4 == 0 && aligned16(grad_y) && aligned16(weight);
        DSP_TILES(linear_input_grad_kernel, tile, fast, cdiv(l.M, tile) * cdiv(l.K, tile), s, l, grad_y, weight, grad_x);
    }
    const Split p = split_of(rows, outputs, inputs, 0, 1);
    const bool fast = l.N % 4 == 0 && l.K % 4 == 0 && aligned16(grad_y) && aligned16(x);
    DSP_TILES(linear_weight_grad_kernel, p.tile, fast, cdiv(l.N, p.tile) * cdiv(l.K, p.tile) * p.parts, s, l, grad_y, x, p.per_part, (float*)workspace);
    hipLaunchKernelGGL(linear_join_kernel, dim3((unsigned)cdiv((i64)l.N * (l.K + 1), 256)), dim3(256), 0, s, l, p.parts, (const float*)workspace, grad_weight, grad_bias);
    return launched(who);
}

}  // extern "C"
