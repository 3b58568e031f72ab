// dsp_embed.hip -- embedding lookup with scaling, and its gradient (the training side of the lookup at models.py:186).
//
//   out[n, :] = scale * W[t_n, :]                      dW[v, :] = scale * sum over { n : t_n = v } of g[n, :]
//
// Both are bound by memory: no product to speak of.  The forward reads a row and writes a row per token.
//
// The gradient needs the rows of g by token.  Atomic additions into dW would make the result depend on the order of
// arrival (and serialise where one token is frequent), so both forms below add in an order that the sizes alone decide:
//   * small tables of short rows (the model's 16 x 4) fit a workgroup's LDS many times over: every group of lanes keeps a private table
//     there and walks its own tokens, so the gradient is read once, in order; the tables are joined in a fixed order.
//   * larger tables: the token numbers are sorted (a stable radix sort, up to 10 bits a pass, carrying the positions; few tokens
//     by counting who comes before whom), then groups of lanes walk chunks of the sorted order, each run of equal tokens held in
//     registers.  A run inside a chunk is written to dW at once; a run that crosses chunks leaves one partial sum per chunk, and a
//     second launch joins those.
// Sums are held in 32 bits and rounded once to the table's type.
#include "dsp_ops.h"

using namespace dsp;

namespace {

constexpr int kBadToken = -1;

__device__ __forceinline__ int token_at(const void* __restrict__ tokens, int dt, i64 i, int vocab) {
    i64 t;
    if (dt == DSP_DT_U8) t = ((const uint8_t*)tokens)[i];
    else if (dt == DSP_DT_U16) t = ((const uint16_t*)tokens)[i];
    else if (dt == DSP_DT_I32) t = ((const int32_t*)tokens)[i];
    else if (dt == DSP_DT_I64) t = ((const int64_t*)tokens)[i];
    else {
        const float f = ((const float*)tokens)[i];
        t = f > -1.0f && f < 2147483648.0f ? (i64)f : -1;   // towards zero, as a cast does; NaN is no token
    }
    return t >= 0 && t < vocab ? (int)t : kBadToken;
}

// ---- forward ------------------------------------------------------------------------------------------------------------
// A group of `lanes` (a power of two, at most 64) takes a row, one access of VEC values a lane and step; 4 rows in flight per
// group.  No division: row and column come from the lane number.  (131,072 rows of 1,024 bf16: 78 us, 3.4 TB/s written and as much read from
// memory and the caches, 6.9 together.)
template <class T, int VEC>
__global__ __launch_bounds__(256) void embed_forward_kernel(i64 n, int vecs, int log_lanes, const void* __restrict__ tokens, int dt,
                                                            const T* __restrict__ w, int vocab, float scale, T* __restrict__ out) {
    typedef Vec<T, VEC> V;
    const int lane = threadIdx.x & ((1 << log_lanes) - 1);
    const i64 groups = 256 >> log_lanes;
    const i64 row0 = block_at() * groups * 4 + (threadIdx.x >> log_lanes);
    int t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const i64 r = row0 + k * groups;
        t[k] = r < n ? token_at(tokens, dt, r, vocab) : kBadToken;
    }
    for (int v = lane; v < vecs; v += 1 << log_lanes) {
        V x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (t[k] >= 0) x[k] = ((const V*)w)[(i64)t[k] * vecs + v];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const i64 r = row0 + k * groups;
            if (r >= n) continue;
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[k].v[e] = from_f32<T>(t[k] >= 0 ? to_f32(x[k].v[e]) * scale : __builtin_nanf(""));
            ((V*)out)[r * vecs + v] = x[k];
        }
    }
}

// cell[0 .. VEC) += x in accesses of up to 16 bytes
template <class T, int VEC> __device__ __forceinline__ void add_to(float* cell, const Vec<T, VEC>& x) {
    constexpr int N = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int e = 0; e < VEC; e += N) {
        Vec<float, N> c = *(Vec<float, N>*)(cell + e);
#pragma unroll
        for (int i = 0; i < N; ++i) c.v[i] += to_f32(x.v[e + i]);
        *(Vec<float, N>*)(cell + e) = c;
    }
}

// ---- gradient, small tables ----------------------------------------------------------------------------------------------
// LDS: table[v][group][dim] in 32 bits; the lanes of a group own its columns, so nothing is shared until the join.  What bounds it is the chain of
// additions to one place of LDS, so tokens go to as many groups as fit (851,968 tokens of 16 x 4: 10.7 us by 512 workgroups and 4.4 for their
// tables; 6,656: 14 us by one).
template <class T, int VEC>
__global__ __launch_bounds__(256) void embed_grad_small_kernel(i64 n, i64 per_block, int vecs, int log_lanes, const void* __restrict__ tokens,
                                                               int dt, const T* __restrict__ g, int vocab, int pad, float scale,
                                                               float* __restrict__ part, T* __restrict__ dw) {
    typedef Vec<T, VEC> V;
    extern __shared__ __attribute__((aligned(16))) float table[];
    const int dim = vecs * VEC, groups = blockDim.x >> log_lanes, cells = vocab * dim;
    const int lane = threadIdx.x & ((1 << log_lanes) - 1), group = threadIdx.x >> log_lanes;
    for (int i = threadIdx.x; i < cells * groups / 4; i += blockDim.x) ((f32x4*)table)[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (threadIdx.x < (cells * groups & 3)) table[cells * groups - 1 - threadIdx.x] = 0.0f;
    __syncthreads();
    const i64 from = (i64)blockIdx.x * per_block, to = from + per_block < n ? from + per_block : n;
    for (i64 r = from + group; r < to; r += 4 * groups) {
        int t[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            t[k] = r + k * groups < to ? token_at(tokens, dt, r + k * groups, vocab) : kBadToken;
            if (t[k] == pad) t[k] = kBadToken;
        }
        for (int v = lane; v < vecs; v += 1 << log_lanes) {
            V x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (t[k] >= 0) x[k] = ((const V*)g)[(r + k * groups) * vecs + v];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (t[k] >= 0) add_to<T, VEC>(table + ((i64)t[k] * groups + group) * dim + v * VEC, x[k]);
        }
    }
    __syncthreads();
    // the groups' tables joined: as many threads a cell as there are, each a range of the groups.  Rows begin in the same bank, so
    // every row starts at a group of its own.
    __shared__ float sums[256];
    const int each = cells < (int)blockDim.x ? blockDim.x / cells : 1, per = (groups + each - 1) / each;
    for (int i0 = 0; i0 < cells; i0 += blockDim.x) {
        const int i = i0 + threadIdx.x % cells, range = threadIdx.x / cells;   // cells >= blockDim: range 0
        float s = 0.0f;
        if (i < cells && range < each) {
            const int v = i / dim, to = (range + 1) * per < groups ? (range + 1) * per : groups;
            const float* row = table + (i64)v * groups * dim + i % dim;
#pragma unroll 8
            for (int k = range * per; k < to; ++k) s += row[((k + v) & (groups - 1)) * dim];
        }
        if (each > 1) {
            sums[threadIdx.x] = s;
            __syncthreads();
            s = 0.0f;
            if ((int)threadIdx.x < cells)
                for (int r = 0; r < each; ++r) s += sums[r * cells + threadIdx.x];
        }
        if (i >= cells || range) continue;
        if (part) part[(i64)blockIdx.x * cells + i] = s;
        else dw[i] = from_f32<T>(s * scale);
    }
}

// one wave per cell of the table: its lanes take the blocks' sums in turn, then join in a fixed order
template <class T>
__global__ __launch_bounds__(256) void embed_grad_small_join_kernel(int cells, int blocks, const float* __restrict__ part, float scale,
                                                                    T* __restrict__ dw) {
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= cells) return;
    float s = 0.0f;
    for (int b = threadIdx.x & 63; b < blocks; b += 64) s += part[(i64)b * cells + i];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) dw[i] = from_f32<T>(s * scale);
}

// ---- stable radix sort of (token, position) -----------------------------------------------------------------------------
// One pass: counts of every digit in every tile of 1,024 tokens, an exclusive scan of each digit's counts over the tiles, and
// the move.  A wave takes 256 consecutive tokens as 4 rows of 64; a token's place among equal digits of its row comes from one
// ballot per bit, the rows' and waves' counts from LDS: order within a digit is kept.  Tokens that are not to be counted
// (padding, outside the table) sort behind all others as `vocab`.  (131,072 tokens of 65,536: two passes of 8.8, 4.8 and 4.4 us: launches that
// wait for memory rather than use it.)
constexpr int kTile = 1024, kMaxBins = 1024;

struct Keys { const void* tokens; int dt; const uint32_t* key; int vocab, pad; };

__device__ __forceinline__ uint32_t key_at(const Keys& k, i64 i) {
    if (k.key) return k.key[i];
    const int t = token_at(k.tokens, k.dt, i, k.vocab);
    return t < 0 || t == k.pad ? (uint32_t)k.vocab : (uint32_t)t;
}

__global__ __launch_bounds__(256) void sort_count_kernel(i64 n, Keys keys, int shift, int bins, i64 tiles, uint32_t* __restrict__ count) {
    __shared__ uint32_t h[kMaxBins];
    for (int i = threadIdx.x; i < bins; i += 256) h[i] = 0;
    __syncthreads();
    for (int k = 0; k < kTile; k += 256) {
        const i64 i = (i64)blockIdx.x * kTile + k + threadIdx.x;
        if (i < n) atomicAdd(&h[(key_at(keys, i) >> shift) & (bins - 1)], 1u);   // whole numbers: the order does not matter
    }
    __syncthreads();
    for (int i = threadIdx.x; i < bins; i += 256) count[(i64)i * tiles + blockIdx.x] = h[i];
}

// exclusive prefix of x over the threads of a 256-thread block, and the block's sum
__device__ __forceinline__ uint32_t block_prefix(uint32_t x, uint32_t* wave_total, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(s, o);
        if (lane >= o) s += y;
    }
    __syncthreads();
    if (lane == 63) wave_total[wave] = s;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) before += wave_total[w];
        total += wave_total[w];
    }
    return before + s - x;
}

__global__ __launch_bounds__(256) void sort_scan_kernel(i64 tiles, uint32_t* __restrict__ count, uint32_t* __restrict__ digit_total) {
    __shared__ uint32_t wave_total[4];
    uint32_t* row = count + (i64)blockIdx.x * tiles;
    uint32_t base = 0;
    for (i64 at = 0; at < tiles; at += 256) {
        const i64 i = at + threadIdx.x;
        const uint32_t x = i < tiles ? row[i] : 0;
        uint32_t total;
        const uint32_t p = block_prefix(x, wave_total, total);
        if (i < tiles) row[i] = base + p;
        base += total;
    }
    if (threadIdx.x == 0) digit_total[blockIdx.x] = base;
}

__global__ __launch_bounds__(256) void sort_move_kernel(i64 n, Keys keys, const uint32_t* __restrict__ pos_in, int shift, int log_bins, i64 tiles,
                                                        const uint32_t* __restrict__ count, const uint32_t* __restrict__ digit_total,
                                                        uint32_t* __restrict__ key_out, uint32_t* __restrict__ pos_out) {
    __shared__ uint32_t seen[4][kMaxBins];   // per wave: tokens of a digit so far, then the place of the wave's first one
    __shared__ uint32_t wave_total[4];
    const int bins = 1 << log_bins, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < 4 * kMaxBins; i += 256) ((uint32_t*)seen)[i] = 0;
    __syncthreads();
    uint32_t key[4], rank[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const i64 i = (i64)blockIdx.x * kTile + wave * 256 + k * 64 + lane;
        const bool live = i < n;
        key[k] = live ? key_at(keys, i) : 0;
        const uint32_t d = (key[k] >> shift) & (bins - 1);
        uint64_t same = __ballot(live);
        for (int b = 0; b < log_bins; ++b) {
            const uint64_t m = __ballot(d >> b & 1);
            same &= d >> b & 1 ? m : ~m;
        }
        rank[k] = seen[wave][d] + __popcll(same & ((1ull << lane) - 1));
        __builtin_amdgcn_wave_barrier();   // every lane has read its digit's count before one of them moves it on
        if (live && lane == 63 - __clzll(same)) seen[wave][d] = rank[k] + 1;
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // first place of every digit (all digits before it), of this tile's tokens in it, and of every wave's
    uint32_t base = 0;
    for (int at = 0; at < bins; at += 256) {
        const int d = at + threadIdx.x;
        uint32_t total;
        const uint32_t before = block_prefix(d < bins ? digit_total[d] : 0, wave_total, total);
        if (d < bins) {
            uint32_t place = base + before + count[(i64)d * tiles + blockIdx.x];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t c = seen[w][d];
                seen[w][d] = place;
                place += c;
            }
        }
        base += total;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const i64 i = (i64)blockIdx.x * kTile + wave * 256 + k * 64 + lane;
        if (i >= n) continue;
        const uint32_t to = seen[wave][(key[k] >> shift) & (bins - 1)] + rank[k];
        key_out[to] = key[k];
        pos_out[to] = pos_in ? pos_in[i] : (uint32_t)i;
    }
}

// Few tokens: every one counts the tokens that come before it (a smaller key, or the same one earlier), one launch in place of three a pass.  A
// workgroup takes 64 tokens, a wave of it a quarter of what they are compared with.  The launch's other workgroups clear the gradient.
constexpr int kRanked = 4096;
template <class T>
__global__ __launch_bounds__(256) void sort_ranked_kernel(int n, Keys keys, uint32_t* __restrict__ key_out, uint32_t* __restrict__ pos_out, i64 cells, T* __restrict__ dw) {
    __shared__ __attribute__((aligned(16))) uint32_t k[kRanked];
    __shared__ int ranks[4][64];
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const int blocks = (n + 63) >> 6;
    if ((int)blockIdx.x >= blocks) {
        const i64 step = (i64)(gridDim.x - blocks) * 256;
        for (i64 i = (i64)(blockIdx.x - blocks) * 256 + threadIdx.x; i < cells; i += step) dw[i] = T{};
        return;
    }
    const int all = (n + 15) & ~15;
    for (int i = threadIdx.x; i < all; i += 256) k[i] = i < n ? key_at(keys, i) : 0xffffffffu;   // behind the last: before nothing
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = blockIdx.x * 64, i = first + lane, last = first + 64 < all ? first + 64 : all;
    const int from = wave * (all / 4), to = from + all / 4;
    const uint32_t mine = i < n ? k[i] : 0;
    int rank = 0;
    auto count = [&](int lo, int hi, uint32_t below) {   // lo, hi: multiples of 4
#pragma unroll 4
        for (int j = lo; j < hi; j += 4) {
            const u32x4 x = *(const u32x4*)(k + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) rank += x[e] < below;
        }
    };
    count(from, to < first ? to : first, mine + 1);
    for (int j = from > first ? from : first; j < (to < last ? to : last); ++j) rank += k[j] < mine + (j < i ? 1u : 0u);
    count(from > last ? from : last, to, mine);
    ranks[wave][lane] = rank;
    __syncthreads();
    if (wave || i >= n) return;
    rank = ranks[0][lane] + ranks[1][lane] + ranks[2][lane] + ranks[3][lane];
    key_out[rank] = mine;
    pos_out[rank] = (uint32_t)i;
}

// ---- gradient by sorted tokens ------------------------------------------------------------------------------------------
template <class T> __global__ __launch_bounds__(256) void embed_zero_kernel(i64 n, T* __restrict__ dw) {
    for (i64 i = (i64)blockIdx.x * 256 + threadIdx.x; i < n; i += (i64)gridDim.x * 256) dw[i] = T{};
}

// A group of lanes walks one chunk of the sorted order for the columns that its lanes hold (64 accesses of columns at most).
// part[chunk][0]: the sum of the run that reaches into the chunk from before; part[chunk][1]: of the run that begins here
// and goes on behind it.  Bound by memory: rows of the gradient in the order of their tokens, a row of dW for each token that occurs (131,072
// rows of 1,024 bf16 into 65,536: 100 us, 3.8 TB/s; with 16 rows ahead of their use in place of 8: 130, too few waves).
template <class T, int VEC>
__global__ __launch_bounds__(256) void embed_grad_walk_kernel(i64 n, int chunk, int vecs, int log_lanes, const uint32_t* __restrict__ key,
                                                              const uint32_t* __restrict__ pos, const T* __restrict__ g, int vocab, float scale,
                                                              float* __restrict__ part, T* __restrict__ dw) {
    typedef Vec<T, VEC> V;
    typedef Vec<float, VEC> F;
    const int slabs = (vecs + 63) >> 6;   // the parts of a row are neighbours, so that it is read at about one time
    const i64 c = (i64)(blockIdx.x / slabs) * (256 >> log_lanes) + (threadIdx.x >> log_lanes);
    const int v = blockIdx.x % slabs * 64 + (threadIdx.x & ((1 << log_lanes) - 1));
    const i64 from = c * chunk, to = from + chunk < n ? from + chunk : n;
    if (from >= n || v >= vecs) return;
    const int dim = vecs * VEC;
    uint32_t run = key[from];
    bool open = from > 0 && key[from - 1] == run;   // the run began before this chunk
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
    constexpr int AHEAD = 8;   // rows of the gradient on their way; which ones they are is read 8 rows before
    uint32_t k[AHEAD], next_k[AHEAD], next_p[AHEAD];
    auto read = [&](i64 i) {
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            next_k[j] = i + j < to ? key[i + j] : (uint32_t)vocab;
            next_p[j] = i + j < to ? pos[i + j] : 0;
        }
    };
    read(from);
    for (i64 i = from; i < to; i += AHEAD) {
        V x[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            k[j] = next_k[j];
            if (k[j] < (uint32_t)vocab) x[j] = ((const V*)g)[(i64)next_p[j] * vecs + v];
        }
        read(i + AHEAD);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            if (i + j >= to) break;
            if (k[j] != run) {
                if (run < (uint32_t)vocab) {   // a run ends inside the chunk
                    if (open) {
                        F f;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) f.v[e] = acc[e];
                        *(F*)(part + (c * 2) * dim + v * VEC) = f;
                    } else {
                        V y;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) y.v[e] = from_f32<T>(acc[e] * scale);
                        ((V*)dw)[(i64)run * vecs + v] = y;
                    }
                }
                run = k[j];
                open = false;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
            }
            if (k[j] < (uint32_t)vocab)
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += to_f32(x[j].v[e]);
        }
    }
    if (run >= (uint32_t)vocab) return;
    const bool goes_on = to < n && key[to] == run;
    if (open || goes_on) {
        F f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) f.v[e] = acc[e];
        *(F*)(part + (c * 2 + (open ? 0 : 1)) * dim + v * VEC) = f;
    } else {
        V y;
#pragma unroll
        for (int e = 0; e < VEC; ++e) y.v[e] = from_f32<T>(acc[e] * scale);
        ((V*)dw)[(i64)run * vecs + v] = y;
    }
}

// (2,048 chunks, 131,072 tokens: 14 us.)  A block per chunk in which a run begins that goes on behind it (the others end at once) and 64 x VEC columns: the run's last chunk is found
// by bisection; groups of lanes, VEC columns a lane, add a range of its partial sums each, then their sums are joined in order.
template <class T, int VEC>
__global__ __launch_bounds__(256) void embed_grad_join_kernel(i64 n, int chunk, i64 chunks, int vecs, int log_lanes, const uint32_t* __restrict__ key, int vocab,
                                                              float scale, const float* __restrict__ part, T* __restrict__ dw) {
    typedef Vec<float, VEC> F;
    __shared__ F sums[256];
    const i64 c = block_at(), from = c * chunk, to = from + chunk;
    if (to >= n) return;
    const uint32_t run = key[to], last = key[to - 1], start = key[from], before = from > 0 ? key[from - 1] : 0xffffffffu;
    if (run >= (uint32_t)vocab || last != run || (start == run && before == run)) return;   // no run goes on, or it began in an earlier chunk
    i64 lo = c + 1, hi = chunks;   // chunks lo - 1 and before begin with the run (or hold its beginning), hi and behind do not
    while (lo < hi) {
        const i64 mid = (lo + hi) >> 1;
        if (key[mid * chunk] == run) lo = mid + 1;
        else hi = mid;
    }
    const int lanes = 1 << log_lanes, groups = 256 >> log_lanes, group = threadIdx.x >> log_lanes, v = blockIdx.z * 64 + (threadIdx.x & (lanes - 1));
    const i64 count = lo - (c + 1), per = (count + groups - 1) / groups;   // partial sums behind the first
    F s;
#pragma unroll
    for (int e = 0; e < VEC; ++e) s.v[e] = 0.0f;
    if (v < vecs) {
        const F* p = (const F*)part + v;
        if (group == 0) s = p[(c * 2 + 1) * vecs];
        const i64 end = (group + 1) * per < count ? (group + 1) * per : count;
#pragma unroll 8
        for (i64 i = group * per; i < end; ++i) {
            const F x = p[(c + 1 + i) * 2 * vecs];
#pragma unroll
            for (int e = 0; e < VEC; ++e) s.v[e] += x.v[e];
        }
    }
    sums[threadIdx.x] = s;
    __syncthreads();
    if (group || v >= vecs) return;
    for (int g = 1; g < groups; ++g)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s.v[e] += sums[g * lanes + threadIdx.x].v[e];
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[(i64)run * vecs * VEC + v * VEC + e] = from_f32<T>(s.v[e] * scale);
}

// ---- host -----------------------------------------------------------------------------------------------------------------
int log2_lanes(int vecs) {
    int l = 0;
    while ((1 << l) < vecs && l < 6) ++l;
    return l;
}

constexpr size_t kSmallLds = 64 * 1024;   // two workgroups a CU
// groups of lanes (a power of two, `most` at first) whose tables fit a workgroup's LDS together
int groups_that_fit(i64 vocab, i64 dim, int most) {
    while (most > 1 && (size_t)vocab * dim * 4 * most > kSmallLds) most >>= 1;
    return most;
}
int few_lanes(i64 dim) { return log2_lanes((int)cdiv(dim, 4)); }
// Tables of up to 2 KB, of which 32 fit, and rows of up to 16 values, so that many tokens are walked at once.  (2^20 tokens: 64 rows of 8: 54 us,
// sorted 78; 32 of 16: 59 and 67; but 64 of 16: 91 and 71, 8 of 64: 123 and 90, 64 of 64: 424 and 94)
bool small_table(i64 vocab, i64 dim) { return dim <= 16 && vocab * dim <= 512; }
int type_size(int dt) { return dt == DSP_FT_F32 ? 4 : 2; }
// Few tokens: one workgroup, which needs no second launch and no workspace, where 64 of them are walked at once (6,656 x 16 x 4: 14 us on the GPU in
// place of 9, 78 in place of 84 us a step of forward and backward, which the host's side bounds; 8,000 of 64 x 8, 32 at once: 91 and 66)
constexpr i64 kSmallOne = 8192;
bool one_workgroup(i64 n, i64 vocab, i64 dim) { return n <= kSmallOne && groups_that_fit(vocab, dim, 256 >> few_lanes(dim)) >= 64; }
int key_bits(i64 vocab) {   // keys 0 .. vocab
    int b = 1;
    while (((i64)1 << b) <= vocab) ++b;
    return b;
}
i64 chunk_of(i64 n) { return n < 16384 ? 16 : 64; }

struct Plan {   // of the sorted form: places in the workspace
    i64 tiles, chunks;
    int passes, bits, chunk;
    size_t count, total, key[2], pos[2], part, bytes;
};
Plan plan_sorted(i64 n, i64 vocab, i64 dim) {
    Plan p;
    const int all = key_bits(vocab);
    p.passes = (all + 9) / 10;
    p.bits = (all + p.passes - 1) / p.passes;
    p.tiles = cdiv(n, kTile);
    p.chunk = (int)chunk_of(n);
    p.chunks = cdiv(n, p.chunk);
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t r = at; at += align256(bytes); return r; };
    p.count = take((size_t)p.tiles * ((size_t)4 << p.bits));
    p.total = take((size_t)4 << p.bits);
    for (int i = 0; i < 2; ++i) { p.key[i] = take((size_t)n * 4); p.pos[i] = take((size_t)n * 4); }
    p.part = take((size_t)p.chunks * 2 * dim * 4);
    p.bytes = at;
    return p;
}

template <class T, int VEC>
void forward_of(hipStream_t s, i64 n, int dim, const void* tokens, int dt, const void* w, int vocab, float scale, void* out) {
    const int vecs = dim / VEC;
    // fewer lanes in several turns where more than a third of them would have nothing (2^21 rows of 33 fp32: 158 us, 184 with 64 lanes; 9: 44 and 53;
    // 209,715 of 320 bf16: 31 and 37)
    int ll = log2_lanes(vecs);
    while (ll > 2 && ((((vecs - 1) >> ll) + 1) << ll) * 2 > vecs * 3) --ll;
    hipLaunchKernelGGL((embed_forward_kernel<T, VEC>), grid_of(cdiv(n, 4 * (256 >> ll))), dim3(256), 0, s, n, vecs, ll, tokens, dt,
                       (const T*)w, vocab, scale, (T*)out);
}

template <class T, int VEC>
void backward_of(hipStream_t s, i64 n, int dim, const void* tokens, int dt, const void* g, int vocab, int pad, float scale, void* dw, char* ws) {
    const int vecs = dim / VEC, ll = log2_lanes(vecs);
    if (small_table(vocab, dim)) {
        // several workgroups: of one wave until there are 512 of them (fewer tables to clear and to join a token), then of 4; 4 tokens a group at
        // least, the loads that it has under way at once
        const bool one = one_workgroup(n, vocab, dim);
        const int cells = vocab * dim, use = groups_that_fit(vocab, dim, (one || n > 512 * 4 * (64 >> ll) ? 256 : 64) >> ll);
        const i64 most = cdiv(n, (i64)use * 4), blocks = one || most < 1 ? 1 : most < 512 ? most : 512;
        float* part = blocks > 1 ? (float*)ws : nullptr;
        hipLaunchKernelGGL((embed_grad_small_kernel<T, VEC>), dim3((unsigned)blocks), dim3(use << ll), (size_t)cells * use * 4, s, n, cdiv(n, blocks), vecs, ll,
                           tokens, dt, (const T*)g, vocab, pad, scale, part, (T*)dw);
        if (part)
            hipLaunchKernelGGL((embed_grad_small_join_kernel<T>), dim3((unsigned)cdiv(cells, 4)), dim3(256), 0, s, cells, (int)blocks, part, scale, (T*)dw);
        return;
    }
    const i64 cells = (i64)vocab * dim, zero = cdiv(cells, 256) < 4096 ? cdiv(cells, 256) : 4096;
    const Plan p = plan_sorted(n, vocab, dim);
    const uint32_t *key = nullptr, *pos = nullptr;
    if (n > 0 && n <= kRanked) {
        key = (uint32_t*)(ws + p.key[0]);
        pos = (uint32_t*)(ws + p.pos[0]);
        hipLaunchKernelGGL((sort_ranked_kernel<T>), dim3((unsigned)(cdiv(n, 64) + zero)), dim3(256), 0, s, (int)n, (Keys{tokens, dt, nullptr, vocab, pad}),
                           (uint32_t*)(ws + p.key[0]), (uint32_t*)(ws + p.pos[0]), cells, (T*)dw);
    } else {
        hipLaunchKernelGGL((embed_zero_kernel<T>), dim3((unsigned)zero), dim3(256), 0, s, cells, (T*)dw);
        if (n == 0) return;
        uint32_t *count = (uint32_t*)(ws + p.count), *total = (uint32_t*)(ws + p.total);
        for (int k = 0; k < p.passes; ++k) {
            const Keys keys = {tokens, dt, key, vocab, pad};
            uint32_t *ko = (uint32_t*)(ws + p.key[k & 1]), *po = (uint32_t*)(ws + p.pos[k & 1]);
            hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)p.tiles), dim3(256), 0, s, n, keys, k * p.bits, 1 << p.bits, p.tiles, count);
            hipLaunchKernelGGL(sort_scan_kernel, dim3(1u << p.bits), dim3(256), 0, s, p.tiles, count, total);
            hipLaunchKernelGGL(sort_move_kernel, dim3((unsigned)p.tiles), dim3(256), 0, s, n, keys, pos, k * p.bits, p.bits, p.tiles, count, total, ko, po);
            key = ko;
            pos = po;
        }
    }
    float* part = (float*)(ws + p.part);
    hipLaunchKernelGGL((embed_grad_walk_kernel<T, VEC>), dim3((unsigned)(cdiv(p.chunks, 256 >> ll) * cdiv(vecs, 64))), dim3(256), 0, s, n, p.chunk, vecs,
                       ll, key, pos, (const T*)g, vocab, scale, part, (T*)dw);
    constexpr int JOIN = VEC < 4 ? VEC : 4;   // columns a lane
    const int jv = dim / JOIN;
    dim3 grid = grid_of(p.chunks);
    grid.z = (unsigned)cdiv(jv, 64);
    hipLaunchKernelGGL((embed_grad_join_kernel<T, JOIN>), grid, dim3(256), 0, s, n, p.chunk, p.chunks, jv, log2_lanes(jv),
                       key, vocab, scale, part, (T*)dw);
}

const char* bad_embedding(i64 n, i64 vocab, i64 dim, int dt, int ft) {
    if (n < 0 || n > 0x7fffffffll) return "the number of tokens must be within 0 .. 2^31 - 1";
    if (vocab < 1 || vocab >= 0x7fffffffll) return "the table must have 1 .. 2^31 - 2 rows";
    if (dim < 1 || dim > 65536) return "a row must have 1 .. 65,536 values";
    if (dt != DSP_DT_F32 && dt != DSP_DT_U8 && dt != DSP_DT_U16 && dt != DSP_DT_I32 && dt != DSP_DT_I64) return "unknown token type";
    if (ft != DSP_FT_F32 && ft != DSP_FT_BF16 && ft != DSP_FT_F16) return "unknown element type";
    return nullptr;
}

// f(T, VEC) for the element type and the widest access that rows and addresses allow
#define DSP_EMBED_DISPATCH(F, ft, wide, ...)                                   \
    do {                                                                       \
        if (ft == DSP_FT_F32) {                                                \
            if (wide == 16) F<float, 4>(__VA_ARGS__);                          \
            else if (wide == 8) F<float, 2>(__VA_ARGS__);                      \
            else F<float, 1>(__VA_ARGS__);                                     \
        } else if (ft == DSP_FT_BF16) {                                        \
            if (wide == 16) F<__bf16, 8>(__VA_ARGS__);                         \
            else if (wide == 8) F<__bf16, 4>(__VA_ARGS__);                     \
            else if (wide == 4) F<__bf16, 2>(__VA_ARGS__);                     \
            else F<__bf16, 1>(__VA_ARGS__);                                    \
        } else {                                                               \
            if (wide == 16) F<_Float16, 8>(__VA_ARGS__);                       \
            else if (wide == 8) F<_Float16, 4>(__VA_ARGS__);                   \
            else if (wide == 4) F<_Float16, 2>(__VA_ARGS__);                   \
            else F<_Float16, 1>(__VA_ARGS__);                                  \
        }                                                                      \
    } while (0)

}  // namespace

extern "C" {

int32_t dsp_embedding_forward(void* stream, int64_t n, const void* tokens, int32_t token_dtype, const void* weight, int64_t vocab, int64_t dim,
                              int32_t dtype, float scale, void* out) {
    if (const char* why = bad_embedding(n, vocab, dim, token_dtype, dtype)) return refuse("dsp_embedding_forward", why);
    if (n == 0) return DSP_OK;
    if (!tokens || !weight || !out) return refuse("dsp_embedding_forward", "NULL pointer");
    const int wide = wide_bytes((size_t)dim * type_size(dtype), weight, out);
    if (wide < type_size(dtype)) return refuse("dsp_embedding_forward", "an address is not aligned to its element type");
    DSP_EMBED_DISPATCH(forward_of, dtype, wide, (hipStream_t)stream, n, (int)dim, tokens, token_dtype, weight, (int)vocab, scale, out);
    return launched("dsp_embedding_forward");
}

int64_t dsp_embedding_workspace(int64_t n, int64_t vocab, int64_t dim) {
    if (const char* why = bad_embedding(n, vocab, dim, DSP_DT_U8, DSP_FT_F32)) return refuse("dsp_embedding_workspace", why);
    if (small_table(vocab, dim)) return one_workgroup(n, vocab, dim) ? 0 : (int64_t)align256((size_t)512 * vocab * dim * 4);
    return (int64_t)plan_sorted(n, vocab, dim).bytes;
}

int32_t dsp_embedding_backward(void* stream, int64_t n, const void* tokens, int32_t token_dtype, const void* grad, int64_t vocab, int64_t dim,
                               int32_t dtype, int64_t padding_idx, float scale, void* weight_grad, void* workspace, int64_t workspace_bytes) {
    if (const char* why = bad_embedding(n, vocab, dim, token_dtype, dtype)) return refuse("dsp_embedding_backward", why);
    if (padding_idx < -1 || padding_idx >= vocab) return refuse("dsp_embedding_backward", "padding_idx is not a row of the table");
    const int64_t need = dsp_embedding_workspace(n, vocab, dim);
    if (!weight_grad || (n && (!tokens || !grad || (need && !workspace)))) return refuse("dsp_embedding_backward", "NULL pointer");
    if (n && workspace_bytes < need) return refuse("dsp_embedding_backward", "workspace too small (dsp_embedding_workspace)");
    if ((size_t)workspace & 255) return refuse("dsp_embedding_backward", "the workspace must be aligned to 256 bytes");
    const int wide = wide_bytes((size_t)dim * type_size(dtype), grad, weight_grad);
    if (wide < type_size(dtype)) return refuse("dsp_embedding_backward", "an address is not aligned to its element type");
    // -2 stands for no padding row: no token has it
    DSP_EMBED_DISPATCH(backward_of, dtype, wide, (hipStream_t)stream, n, (int)dim, tokens, token_dtype, grad, (int)vocab,
                       padding_idx < 0 ? -2 : (int)padding_idx, scale, weight_grad, (char*)workspace);
    return launched("dsp_embedding_backward");
}

}  // extern "C"
