// dsp_products.h -- products of fp32 matrices on the fp32 matrix instructions, for the layers of a training step (dsp_lstm_train.hip:
// over all steps at once; dsp_linear.hip).
//
// C(m, n) = sum over k of A(m, k) B(n, k).  A workgroup of 4 waves makes a tile of TILE x TILE, a wave a quarter of it as 32 x 32
// blocks of v_mfma_f32_32x32x2.  16 values of k are staged in LDS at a time, the next 16 on their way in registers and the ones
// before them in the other half of LDS: one barrier per 16.  A lane's 4 values of k are consecutive (lane group q takes k =
// 4q + j for instruction j): the order of k is the same for both operands, so any is right.  (4,096 x 4,096 x 4,096: 126 TFLOP/s.)
//
// On this device vector instructions take their time from the fp32 matrix instructions, so the loop has next to none: where
// sizes and addresses allow (FAST), the operands come by buffer loads whose lane offsets are made once and whose descriptors
// end with the operand: what lies behind it reads as zeros.  Otherwise (an input size of 7) every value is guarded.
#ifndef DSP_PRODUCTS_H
#define DSP_PRODUCTS_H

#include "dsp_ops.h"

namespace dsp {

constexpr int kStep = 16;

struct Matrix {   // row-major, `lines` lines of `ld` values
    const float* p;
    int lines, ld;
};

struct AllLines { __device__ __forceinline__ int operator()(int row) const { return row; } };
// ALONG_K: a line is a row of the product, k along it.  Else a line is a k, the product's rows along it.  line_of (ALONG_K and FAST): the line
// that a row of the tile is, from row0
template <bool ALONG_K, int TILE, bool FAST> struct Stage {
    static constexpr int kStride = ALONG_K ? kStep + 4 : TILE + 4;
    static constexpr int kFloats = ALONG_K ? TILE * kStride : kStep * kStride;
    static constexpr int kLoads = TILE * kStep / 4 / 256, kAcross = ALONG_K ? kStep / 4 : TILE / 4;   // accesses of 4 along a line
    f32x4 v[kLoads];
    Matrix m;
    int row0, k_end;
    __amdgpu_buffer_rsrc_t rsrc;
    int lane_at[kLoads];
    uint32_t at, per_step;
    template <class Line = AllLines> __device__ __forceinline__ Stage(const Matrix& matrix, int row, int k0, int k1, Line line_of = {}) : m(matrix), row0(row), k_end(k1) {
        if (!FAST) return;
        const float* base = ALONG_K ? m.p + (i64)row0 * m.ld : m.p + (i64)k0 * m.ld + row0;
        const i64 bytes = ((i64)m.lines * m.ld - (base - m.p)) * 4;
        rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)(bytes > 0xfffffff0ll ? 0xfffffff0u : (uint32_t)bytes), 0x00020000);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int j = threadIdx.x + i * 256;
            lane_at[i] = (line_of(j / kAcross) * m.ld + j % kAcross * 4) * 4;
        }
        at = ALONG_K ? k0 * 4 : 0;
        per_step = ALONG_K ? kStep * 4 : (uint32_t)m.ld * kStep * 4;
    }
    __device__ __forceinline__ void fetch(int k) {
        if (FAST) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) v[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, lane_at[i], (int)at, 0));
            at += per_step;
            return;
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int j = threadIdx.x + i * 256;
            const int line = (ALONG_K ? row0 : k) + j / kAcross, on = (ALONG_K ? k : row0) + j % kAcross * 4;
            const int lines = ALONG_K ? m.lines : k_end, most = ALONG_K ? k_end : m.ld;
            const float* p = m.p + (i64)line * m.ld + on;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i][e] = line < lines && on + e < most ? p[e] : 0.0f;
        }
    }
    __device__ __forceinline__ void put(float* lds) const {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int j = threadIdx.x + i * 256;
            *(f32x4*)(lds + j / kAcross * kStride + j % kAcross * 4) = v[i];
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
template <bool A_ALONG_K, bool B_ALONG_K, int TILE> constexpr int half_floats() {
    return Stage<A_ALONG_K, TILE, false>::kFloats + Stage<B_ALONG_K, TILE, false>::kFloats;
}

// acc[i][j] (block (i, j) of the wave's part of the tile) += over k in [k0, k1).  f(values of A as they are staged) for every 16 of k.  The waves
// are 2 by 2, or (RM 1, RN 4 of a tile of 128) 4 by 1
template <bool A_ALONG_K, bool B_ALONG_K, int TILE, bool FAST, int RM, int RN, class F, class Line = AllLines>
__device__ __forceinline__ void product(const Matrix& a, const Matrix& b, int m0, int n0, int k0, int k1, float* lds, f32x16 (&acc)[RM][RN], F&& f, Line line_of_b = {}) {
    typedef Stage<A_ALONG_K, TILE, FAST> SA;
    typedef Stage<B_ALONG_K, TILE, FAST> SB;
    constexpr int HALF = SA::kFloats + SB::kFloats, ACROSS = TILE / 32 / RN;   // waves
    static_assert(RM * RN * 4 * 32 * 32 == TILE * TILE, "4 waves share the tile");
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / ACROSS * (RM * 32) + (lane & 31), wn = wave % ACROSS * (RN * 32) + (lane & 31), kq = (lane >> 5) * 4;
    if (k0 >= k1) return;
    SA sa(a, m0, k0, k1);
    SB sb(b, n0, k0, k1, line_of_b);
    auto step = [&](int half, int k) {   // 16 values of k from one half of LDS; the next 16 into the other
        const float *la = lds + half * HALF, *lb = la + SA::kFloats;
#pragma unroll
        for (int kk = 0; kk < kStep; kk += 8) {
            f32x4 fa[RM], fb[RN];
#pragma unroll
            for (int i = 0; i < RM; ++i) fa[i] = SA::get(la, wm + i * 32, kk + kq);
#pragma unroll
            for (int j = 0; j < RN; ++j) fb[j] = SB::get(lb, wn + j * 32, kk + kq);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int j = 0; j < RN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[i][e], fb[j][e], acc[i][j], 0, 0, 0);
        }
        if (k + kStep < k1) {
            float* next = lds + (half ^ 1) * HALF;
            f(sa.v);
            sa.put(next);
            sb.put(next + SA::kFloats);
            if (k + 2 * kStep < k1) {
                sa.fetch(k + 2 * kStep);
                sb.fetch(k + 2 * kStep);
            }
        }
        __syncthreads();
    };
    sa.fetch(k0);
    sb.fetch(k0);
    __syncthreads();   // what used LDS before is done
    f(sa.v);
    sa.put(lds);
    sb.put(lds + SA::kFloats);
    if (k0 + kStep < k1) {
        sa.fetch(k0 + kStep);
        sb.fetch(k0 + kStep);
    }
    __syncthreads();
    for (int k = k0; k < k1; k += 2 * kStep) {
        step(0, k);
        if (k + kStep < k1) step(1, k + kStep);
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
// Workgroups go to the 8 dies in turn, each with an L2 of its own: give each die a contiguous range of the tiles, so that tiles of the same
// rows (neighbours in it) find them there.
__device__ __forceinline__ uint32_t tile_of(uint32_t block, uint32_t tiles) {
    const uint32_t die = block & 7, per = tiles >> 3, more = tiles & 7;
    return die * per + (die < more ? die : more) + (block >> 3);
}
// What a workgroup of product<false, ...> has staged of A, summed over k: start from zeros, add in the product's f, store at the end
template <int TILE> struct RowSums {
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    template <class V> __device__ __forceinline__ void operator()(const V& v) {
        for (const f32x4& y : v) sum += y;
    }
    // f(row of the tile, sum).  A thread has summed 4 rows for the values of k that came to it: rows by access along a line, k by line
    template <class F> __device__ __forceinline__ void store(float* lds, F f) {
        constexpr int kAcross = TILE / 4, kLines = 256 / kAcross;
        f32x4* sums = (f32x4*)lds;
        __syncthreads();
        sums[threadIdx.x] = sum;
        __syncthreads();
        if (threadIdx.x >= kAcross) return;
        for (int i = 1; i < kLines; ++i) sum += sums[i * kAcross + threadIdx.x];
#pragma unroll
        for (int e = 0; e < 4; ++e) f((int)threadIdx.x * 4 + e, sum[e]);
    }
};
struct Nothing { template <class V> __device__ __forceinline__ void operator()(const V&) const {} };

// ---- products of few rows or columns ------------------------------------------------------------------------------------------
// A workgroup of 4 waves makes a tile of 16 S rows by C blocks of 16 columns (a recurrent step forward: the 4 gates of 16 units; backward: 16 units).
// Every wave takes a quarter of k and the whole tile, so that no value is loaded by two waves.  It loads lines of 128 bytes, 8 rows at a
// time, 32 values of k ahead, and turns them in LDS of its own into what v_mfma_f32_16x16x4 takes (a lane's 4 consecutive k of one
// row, as above).  Loaded in that form from memory they would cost the L1 an access for each 16 bytes: 16 neighbouring lanes are 16
// rows (90 us a step of 4,096 sequences instead of 70).  No wave waits for another until the quarters are joined, in order.
// WIDE: rows begin at multiples of 16 bytes and k is one of 4.
constexpr int kLine = 32;   // values of k at a time
// where 4 values of a row lie in LDS: the 8 places of a row change with the pair of rows, so that 16 rows read at once fall on all banks
__device__ __forceinline__ int spread(int row, int k) { return row * kLine + (((k >> 2) ^ (row >> 1)) & 7) * 4; }

// row_a(i): the tile's i-th row;  col_w(i): the tile's i-th column as its offset in bytes from w, below 2^32
template <int S, int C, bool WIDE, class RowA, class ColW>
__device__ __forceinline__ void step_product(int K, RowA row_a, const float* w, ColW col_w, float* lds, f32x4 (&acc)[C][S]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = lane >> 3, on = (lane & 7) * 4;
    const int lines = (K + kLine - 1) / kLine, per = (lines + 3) >> 2, from = wave * per, to = from + per < lines ? from + per : lines;
    if (from >= to) return;
    float *la = lds + wave * (S + C) * 16 * kLine, *lw = la + S * 16 * kLine;
    const float* pa[2 * S];
    uint32_t pw[2 * C];
#pragma unroll
    for (int i = 0; i < 2 * S; ++i) pa[i] = row_a(i * 8 + at) + on;
#pragma unroll
    for (int i = 0; i < 2 * C; ++i) pw[i] = col_w(i * 8 + at) + on * 4;
    f32x4 va[2 * S], vw[2 * C];
    auto fetch = [&](int line) {
        const int k = line * kLine;
        const char* wk = (const char*)(w + k);
        if (WIDE && k + kLine <= K) {
#pragma unroll
            for (int i = 0; i < 2 * S; ++i) va[i] = *(const f32x4*)(pa[i] + k);
#pragma unroll
            for (int i = 0; i < 2 * C; ++i) vw[i] = *(const f32x4*)(wk + pw[i]);
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = k + on + e < K;
#pragma unroll
            for (int i = 0; i < 2 * S; ++i) va[i][e] = in ? pa[i][k + e] : 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * C; ++i) vw[i][e] = in ? *(const float*)(wk + pw[i] + e * 4) : 0.0f;
        }
    };
    fetch(from);
    for (int line = from; line < to; ++line) {
        // one wave's accesses to LDS are carried out in order, and no other wave reads or writes here
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 2 * S; ++i) *(f32x4*)(la + spread(i * 8 + at, on)) = va[i];
#pragma unroll
        for (int i = 0; i < 2 * C; ++i) *(f32x4*)(lw + spread(i * 8 + at, on)) = vw[i];
        __builtin_amdgcn_wave_barrier();
        if (line + 1 < to) fetch(line + 1);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            f32x4 fa[S], fw[C];
            const int k = half * 16 + (lane >> 4) * 4;
#pragma unroll
            for (int j = 0; j < S; ++j) fa[j] = *(const f32x4*)(la + spread(j * 16 + (lane & 15), k));
#pragma unroll
            for (int c = 0; c < C; ++c) fw[c] = *(const f32x4*)(lw + spread(c * 16 + (lane & 15), k));
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int j = 0; j < S; ++j) acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[j][e], fw[c][e], acc[c][j], 0, 0, 0);
        }
    }
}
// the sums of the 4 waves: of the values of the tile at the thread's rows (16 apart) and column
constexpr int kRow = 17;   // floats of a row of 16 in LDS
template <int S, int C> constexpr int step_floats() {
    return 4 * (S + C) * 16 * kLine > 4 * C * S * 16 * kRow ? 4 * (S + C) * 16 * kLine : 4 * C * S * 16 * kRow;
}
template <int S, int C> __device__ __forceinline__ void step_join(const f32x4 (&acc)[C][S], float* lds, float (&sum)[S][C]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();   // the waves are done with their parts of LDS
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < S; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) lds[((wave * C + c) * S * 16 + j * 16 + (lane >> 4) * 4 + r) * kRow + (lane & 15)] = acc[c][j][r];
    __syncthreads();
    const int row = threadIdx.x >> 4, unit = threadIdx.x & 15;
#pragma unroll
    for (int j = 0; j < S; ++j)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            sum[j][c] = 0.0f;
#pragma unroll
            for (int v = 0; v < 4; ++v) sum[j][c] += lds[((v * C + c) * S * 16 + j * 16 + row) * kRow + unit];
        }
}

inline bool aligned16(const void* p) { return (size_t)p % 16 == 0; }

// tiles of 128 x 128 where they fill the device twice, else of 64 x 64
inline int tile_for(i64 m, i64 n) { return cdiv(m, 128) * cdiv(n, 128) >= 512 ? 128 : 64; }
#define DSP_TILES_ON(kernel, tile, fast, grid, s, ...)                                                                                  \
    do {                                                                                                                                \
        if (tile == 128 && fast) hipLaunchKernelGGL((kernel<128, true>), grid, dim3(256), 0, s, __VA_ARGS__);                           \
        else if (tile == 128) hipLaunchKernelGGL((kernel<128, false>), grid, dim3(256), 0, s, __VA_ARGS__);                             \
        else if (fast) hipLaunchKernelGGL((kernel<64, true>), grid, dim3(256), 0, s, __VA_ARGS__);                                      \
        else hipLaunchKernelGGL((kernel<64, false>), grid, dim3(256), 0, s, __VA_ARGS__);                                               \
    } while (0)
#define DSP_TILES(kernel, tile, fast, blocks, s, ...) DSP_TILES_ON(kernel, tile, fast, dim3((unsigned)(blocks)), s, __VA_ARGS__)

// A sum over K rows in parts: about 768 workgroups (3 a CU) of the tiles of M by (n0 | n1), and no more than 4,096 products in a row
struct Split { int tile, parts, per_part; };
inline Split split_of(i64 K, i64 M, i64 n0, i64 n1, int times) {
    Split q;
    q.tile = cdiv(M, 128) * (cdiv(n0, 128) + cdiv(n1, 128)) * times * cdiv(K, 512) >= 256 ? 128 : 64;
    const i64 tiles = cdiv(M, q.tile) * (cdiv(n0, q.tile) + cdiv(n1, q.tile)) * times;
    i64 parts = cdiv(768, tiles);
    if (parts > cdiv(K, 256)) parts = cdiv(K, 256);
    if (parts < cdiv(K, 4096)) parts = cdiv(K, 4096);
    if (parts < 1) parts = 1;
    q.per_part = (int)(cdiv(cdiv(K, parts), kStep) * kStep);
    if (q.per_part < kStep) q.per_part = kStep;
    q.parts = (int)cdiv(K, q.per_part);
    if (q.parts < 1) q.parts = 1;
    return q;
}

}  // namespace dsp

#endif
