// Products of a layer's backward pass: gradients times codes.
//
//   dz = dy activation'(pre)                                  [M][N]
//   dx[m][k]  = s_k  sum_n dz[m][n] (b[k][n] - z_k)           where x lies inside its grid, else 0
//   dkernel[k][n] = s_in sum_m (a[m][k] - z_in) dz[m][n]      where the kernel does
//
// Codes minus their zero point are whole numbers of at most 8 bits: bfloat16 holds them exactly, so the matrix cores' bfloat16
// instructions multiply them without a rounding.  The gradient is the other operand.  It is the sum of two bfloat16 terms (16 bits)
// for 16-bit results, of three for float32 (24 bits, all that a float has), of fewer where those hold it (a bfloat16 gradient without an
// activation is one), and the product runs over the terms one after the other as over a longer depth.  Sums are float32 throughout.
//
// Both products run over the depth that is contiguous in both operands: dz is written straight and turned, the input's codes
// turned, the kernel's straight.  All are padded with zeros to whole tiles, so the product has no edges to look at but in its
// stores.
#include "layers_internal.h"

#include <algorithm>

namespace axc {
namespace {

// Four neighbouring values as `parts` terms, `pitch` elements from one term to the next.
__device__ __forceinline__ void store_terms(bf16 *p, int parts, int64_t pitch, float (&v)[4])
{
    for (int t = 0; t < parts; ++t) {
        bf16x4 b;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            b[j] = (bf16)v[j];
            v[j] = __fsub_rn(v[j], (float)b[j]);   // exact; of an infinity or NaN it is NaN, and so is the sum of the terms
        }
        *reinterpret_cast<bf16x4 *>(p + t * pitch) = b;
    }
}

// What a logit's sum says of its gradient: coefficient (softmax - one-hot).
template <typename I>
struct LogitTerms {
    Bracket<I> b;
    float scale;
    const GradSource &g;
    __device__ __forceinline__ explicit LogitTerms(const GradSource &source)
        : b(source.sums), scale(__fmul_rn(source.sums.grids->in.scale, source.sums.grids->kernel.scale)), g(source)
    {
    }
    struct Line {                        // of a row
        I term;
        float share, top, log_sum;
        int64_t target;
    };
    __device__ __forceinline__ Line line(int64_t r) const
    {
        return {b.row(g.sums.row_sums[r]), g.coefficient[r], g.top[r], g.log_sum[r], g.targets[r] - g.first_column};
    }
    __device__ __forceinline__ float bias(int64_t c) const { return g.bias ? load_any(g.bias, c, g.bias_type) : 0.0f; }
    __device__ __forceinline__ I column(int64_t c) const { return b.column(g.sums.column_sums[c]); }
    __device__ __forceinline__ float operator()(int32_t sum, const Line &l, I column, float bias, int64_t c) const
    {
        float z = __fmul_rn(Bracket<I>::value(sum, l.term, column), scale);
        if (g.bias)
            z = __fadd_rn(z, bias);
        const float p = __expf((z - l.top) - l.log_sum);
        // a row that does not count has no gradient, whatever its logits are
        return l.share == 0.0f ? 0.0f : l.share * (c == l.target ? p - 1.0f : p);
    }
};

// Gradient in front of the product, 64 x 64 of it a workgroup: into LDS, and from there out straight, turned, and summed by columns.
// SOURCE 0: dense; 1: logits' sums by rows, 2: turned.  `first`: the run's first row, in units of 64.
template <int SOURCE, typename I>
__device__ __forceinline__ void terms_tile(const GradSource &g, int tile_row, int tile_col, int64_t first, int64_t rows,
                                           int64_t rows_pad, int64_t cols, int64_t ld, int straight_parts,
                                           bf16 *__restrict__ straight, int turned_parts, bf16 *__restrict__ turned,
                                           float *__restrict__ column_partials, float (&tile)[64][65])
{
    const int64_t r0 = (int64_t)tile_row * 64, c0 = (int64_t)tile_col * 64;
    const int64_t cols_pad = product_pad(cols);
    const int quad = (threadIdx.x & 15) * 4, line = threadIdx.x / 16;
    if constexpr (SOURCE == 2) {         // a thread four rows of a column
        const LogitTerms<I> at(g);
        typename LogitTerms<I>::Line lines[4] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (r0 + quad + j < rows)
                lines[j] = at.line(r0 + quad + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t c = c0 + line + 16 * i;
            const bool there = c < cols && r0 + quad < rows;
            i32x4 sum = {};
            I column = 0;
            float bias = 0.0f;
            if (there) {
                sum = four_sums(g.sums.raw, r0 + quad, c);
                column = at.column(c);
                bias = at.bias(c);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                tile[quad + j][line + 16 * i] = there && r0 + quad + j < rows ? at(sum[j], lines[j], column, bias, c) : 0.0f;
        }
    } else {
        const int64_t c = c0 + quad;
        I column[4] = {};
        float bias[4] = {};
        if constexpr (SOURCE == 1) {
            const LogitTerms<I> at(g);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j < cols) {
                    column[j] = at.column(c + j);
                    bias[j] = at.bias(c + j);
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = r0 + line + 16 * i;
            float v[4] = {};
            if (r < rows && c < cols) {
                if constexpr (SOURCE == 1) {
                    const LogitTerms<I> at(g);
                    const typename LogitTerms<I>::Line l = at.line(r);
                    const i32x4 sum = four_sums(g.sums.raw, r, c);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[j] = c + j < cols ? at(sum[j], l, column[j], bias[j], c + j) : 0.0f;
                } else {
                    load_four_any(g.grad, r * ld + c, cols - c, g.type, v);
                    if (g.pre) {
                        float z[4];
                        load_four_any(g.pre, r * ld + c, cols - c, g.type, z);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (c + j < cols)
                                v[j] *= activation_slope(z[j], g.activation);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                tile[line + 16 * i][quad + j] = v[j];
        }
    }
    __syncthreads();
    const int64_t above = first * 64;    // rows of earlier runs
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = line + 16 * i;
        float v[4];
        if (straight) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = tile[at][quad + j];
            store_terms(straight + (above + r0 + at) * straight_parts * cols_pad + c0 + quad, straight_parts, cols_pad, v);
        }
        if (turned) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = tile[quad + j][at];
            store_terms(turned + (c0 + at) * turned_parts * rows_pad + above + r0 + quad, turned_parts, rows_pad, v);
        }
    }
    if (column_partials && threadIdx.x < 64) {
        float sum = 0.0f;
        for (int i = 0; i < 64; ++i)
            sum += tile[i][threadIdx.x];
        column_partials[(first + tile_row) * cols_pad + c0 + threadIdx.x] = sum;
    }
}

// Codes minus zero point of a tensor, straight or turned, a tile of 64 x 64; pads are zeros.
template <bool TURN>
__device__ __forceinline__ void centered_tile(const CenteredJob &job, const Grid &g, int tile_row, int tile_col, float (&tile)[64][65])
{
    const int64_t r0 = (int64_t)tile_row * 64, c0 = (int64_t)tile_col * 64;
    const int64_t rows_pad = product_pad(job.rows), cols_pad = product_pad(job.cols);
    const int quad = (threadIdx.x & 15) * 4, line = threadIdx.x / 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + line + 16 * i, c = c0 + quad;
        float v[4] = {};
        if (r < job.rows && c < job.cols) {
            load_four_any(job.values, r * job.ld + c, job.cols - c, job.type, v);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = c + j < job.cols ? (float)((int)code_of(v[j], g) - g.zero) : 0.0f;
        }
        if constexpr (TURN) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                tile[line + 16 * i][quad + j] = v[j];
        } else {
            bf16x4 b;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                b[j] = (bf16)v[j];
            *reinterpret_cast<bf16x4 *>(job.out + r * cols_pad + c) = b;
        }
    }
    if constexpr (TURN) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = line + 16 * i;
            bf16x4 b;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                b[j] = (bf16)tile[quad + j][col];
            *reinterpret_cast<bf16x4 *>(job.out + (c0 + col) * rows_pad + r0 + quad) = b;
        }
    }
}

__device__ __forceinline__ Grid own_grid(const RangeSource &range, float *ends)
{
    float lo, hi;
    fold(range, lo, hi, ends);
    return grid_of_range(lo, hi);
}

// Everything that stands in front of the products, in one launch: the gradient's tiles (in lines of term_cols), then those of the
// input's codes and of the kernel's.  With `ranges` the workgroups of codes make their grids out of the ranges' pairs themselves, and
// the first of all of them both for the launches behind.
template <int SOURCE, typename I>
__global__ void __launch_bounds__(256) grad_prep_kernel(GradSource g, int term_rows, int term_cols, int64_t first, int64_t rows,
                                                        int64_t rows_pad, int64_t cols, int64_t ld, int straight_parts,
                                                        bf16 *__restrict__ straight, int turned_parts, bf16 *__restrict__ turned,
                                                        float *__restrict__ column_partials, CenteredJob x, int x_rows, int x_cols,
                                                        CenteredJob k, int k_cols, RangeSource x_range, RangeSource k_range, int ranges,
                                                        Grids *grids)
{
    __shared__ float tile[64][65];
    __shared__ float ends[8];
    int block = (int)blockIdx.x;
    if (ranges && block == 0) {
        const Grid in = own_grid(x_range, ends), kernel = own_grid(k_range, ends);
        if (threadIdx.x == 0) {
            grids->in = in;
            grids->kernel = kernel;
        }
    }
    if (block < term_rows * term_cols) {
        terms_tile<SOURCE, I>(g, block / term_cols, block % term_cols, first, rows, rows_pad, cols, ld, straight_parts, straight,
                              turned_parts, turned, column_partials, tile);
        return;
    }
    block -= term_rows * term_cols;
    if (block < x_rows * x_cols) {
        const Grid of = ranges ? own_grid(x_range, ends) : grids->in;
        centered_tile<true>(x, of, block / x_cols, block % x_cols, tile);
        return;
    }
    block -= x_rows * x_cols;
    const Grid of = ranges ? own_grid(k_range, ends) : grids->kernel;
    centered_tile<false>(k, of, block / k_cols, block % k_cols, tile);
}

// Results that the product or the pass over its partial sums has, of type T, as the values that decide where there is a gradient.
template <typename T>
struct Results {
    typedef T four __attribute__((ext_vector_type(4)));
    T *out;
    const T *values;
    int64_t ld, values_ld;
    Grid grid;
    float scale;
    bool aligned;                        // every fourth column, in every row
    __device__ __forceinline__ explicit Results(const ProductOut &o)
        : out(static_cast<T *>(o.out)), values(static_cast<const T *>(o.values)), ld(o.ld), values_ld(o.values_ld), grid(*o.grid),
          scale(o.factor ? o.scale->scale * *o.factor : o.scale->scale)
    {
        aligned = ((ld | values_ld) & 3) == 0 && (((uintptr_t)out | (uintptr_t)values) & (4 * sizeof(T) - 1)) == 0;
    }
    __device__ __forceinline__ four values_at(int64_t r, int64_t c) const
    {
        return *reinterpret_cast<const four *>(values + r * values_ld + c);
    }
    __device__ __forceinline__ void store(int64_t r, int64_t c, const four &at, const f32x4 &v) const
    {
        four t;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            t[j] = (T)(inside((float)at[j], grid) ? v[j] * scale : 0.0f);
        *reinterpret_cast<four *>(out + r * ld + c) = t;
    }
    __device__ __forceinline__ void store_some(int64_t r, int64_t c, int64_t cols, const f32x4 &v) const
    {
        if (aligned && c + 4 <= cols) {
            store(r, c, values_at(r, c), v);
            return;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < cols)
                out[r * ld + c + j] = (T)(inside((float)values[r * values_ld + c + j], grid) ? v[j] * scale : 0.0f);
    }
};

constexpr int kStep = 64;   // of the depth
constexpr int product_lds(int groups) { return groups * 2 * 2 * kProductTile * kStep * 2; }

__device__ __forceinline__ void load_to_lds(const bf16 *from, bf16 *to)
{
    // 16 bytes a lane, to `to` of the wavefront plus 16 times the lane
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t *)from,
                                     (__attribute__((address_space(3))) uint32_t *)to, 16, 0, 0);
}

// Sums of the column partials, 64 columns a workgroup, in one order.
__device__ void column_sums(const ColumnJob &job, int block, float *red)
{
    const int column = threadIdx.x & 63, line = threadIdx.x / 64, lines = blockDim.x / 64;
    const int64_t c = (int64_t)block * 64 + column;
    float sum = 0.0f;
    if (c < job.cols)
#pragma unroll 8
        for (int64_t i = line; i < job.count; i += lines)
            sum += job.partials[i * job.pitch + c];
    red[line * 64 + column] = sum;
    __syncthreads();
    if (line == 0 && c < job.cols) {
        sum = 0.0f;
        for (int i = 0; i < lines; ++i)
            sum += red[i * 64 + column];
        store_any(job.out, c, job.type, job.factor ? sum * *job.factor : sum);
    }
}
__global__ void __launch_bounds__(512) column_sums_kernel(ColumnJob job)
{
    __shared__ float red[512];
    column_sums(job, (int)blockIdx.x, red);
}

// A tile of 128 x 128 by G groups of four wavefronts, each of which multiplies every G-th step of the depth, 64 x 64 a wavefront,
// and has two buffers of 64 of the depth in LDS, filled straight from memory while the other is multiplied.  Two wavefronts a SIMD, so
// that one reads while the other multiplies, are two workgroups of one group where there are tiles enough (one's end then goes on under
// the other's steps), else the two groups of one, which at the end exchange half of their sums each.
// In LDS a line of 64 elements is eight chunks of 16 bytes, chunk q of line r in place q ^ (r & 7): the 16 lanes that read
// neighbouring lines then meet different banks.  The loads write LDS in order, so it is their addresses that are exchanged.
// One launch makes both of a layer's products, and the column sums of `job` in workgroups behind their tiles: 78 us for 4096 rows,
// 1024 -> 4096, in bfloat16, 883 TFLOP/s (88 one after the other), 115 for a loss of 1024 rows, 512 -> 32 000 (144).
template <typename T, typename V>
__device__ __forceinline__ void store_tile(const Product &j, int row_tile, int col_tile, int64_t r0, int64_t c0, const V &sum)
{
    constexpr int R = sizeof(V) / sizeof(sum[0]);
    const Results<T> results(j.o);
    // What is read for the results is read all at once, where the tile has no edge: value by value it took as long as the product.
    if (results.aligned && (int64_t)(row_tile + 1) * kProductTile <= j.rows && (int64_t)(col_tile + 1) * kProductTile <= j.cols) {
        typename Results<T>::four at[R][4];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                at[i][k] = results.values_at(r0 + i * 16, c0 + k * 16);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                results.store(r0 + i * 16, c0 + k * 16, at[i][k], sum[i][k]);
        return;
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (r0 + i * 16 < j.rows && c0 + k * 16 < j.cols)
                results.store_some(r0 + i * 16, c0 + k * 16, j.cols, sum[i][k]);
}
template <int G>
__global__ void __launch_bounds__(G * 256) products_kernel(Product first_product, int first_tiles, Product second_product, int tiles,
                                                           ColumnJob job)
{
    extern __shared__ __align__(16) bf16 lds_raw[];
    int id = (int)blockIdx.x;
    if (id >= tiles) {
        column_sums(job, id - tiles, reinterpret_cast<float *>(lds_raw));
        return;
    }
    const Product &j = id < first_tiles ? first_product : second_product;
    const int row_tiles = (int)(product_pad(j.rows) / kProductTile), col_tiles = (int)(product_pad(j.cols) / kProductTile);
    // Workgroups go round the eight XCDs; each XCD gets a run of neighbouring tiles, in bands of eight row tiles, so that its L2
    // serves them.
    {
        const int own = id < first_tiles ? first_tiles : tiles - first_tiles;
        id -= id < first_tiles ? 0 : first_tiles;
        const int per = own / 8, more = own % 8, xcd = id % 8;
        id = xcd * per + (xcd < more ? xcd : more) + id / 8;
    }
    const int split = id / (row_tiles * col_tiles);
    id -= split * row_tiles * col_tiles;
    const int band = id / (8 * col_tiles), in_band = id - band * 8 * col_tiles;
    const int band_rows = row_tiles - band * 8 < 8 ? row_tiles - band * 8 : 8;
    const int row_tile = band * 8 + in_band % band_rows, col_tile = in_band / band_rows;
    const bf16 *const a = j.a, *const b = j.b;
    const int depth = j.depth, parts = j.parts, split_a = j.split_a, splits = j.splits;

    const int lane = threadIdx.x & 63, wave8 = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wave = wave8 & 3, part = wave8 >> 2;
    bf16(*const lds)[2][kProductTile * kStep] = reinterpret_cast<bf16(*)[2][kProductTile * kStep]>(lds_raw) + part * 2;
    const int per_part = depth / kStep, steps = per_part * parts;
    const int first = (int)((int64_t)steps * split / splits), last = (int)((int64_t)steps * (split + 1) / splits);
    const int64_t lda = split_a ? (int64_t)depth * parts : depth, ldb = split_a ? depth : (int64_t)depth * parts;
    const int line = wave * 32 + lane / 8, chunk = ((lane & 7) ^ (lane >> 3)) * 8;
    const bf16 *const pa = a + ((int64_t)row_tile * kProductTile + line) * lda + chunk;
    const bf16 *const pb = b + ((int64_t)col_tile * kProductTile + line) * ldb + chunk;

    auto fetch = [&](int step, int buffer) {
        const int wrapped = step % per_part;
        const int64_t ka = (int64_t)(split_a ? step : wrapped) * kStep, kb = (int64_t)(split_a ? wrapped : step) * kStep;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            load_to_lds(pa + ka + i * 8 * lda, &lds[buffer][0][(wave * 32 + i * 8) * kStep]);
            load_to_lds(pb + kb + i * 8 * ldb, &lds[buffer][1][(wave * 32 + i * 8) * kStep]);
        }
    };

    f32x4 acc[4][4] = {};
    const int wr = (wave >> 1) * 64, wc = (wave & 1) * 64, in_line = lane & 15, group = lane >> 4;
    const int rounds = (last - first + G - 1) / G;
    if (first + part < last)
        fetch(first + part, 0);
    for (int round = 0; round < rounds; ++round) {
        const int step = first + round * G + part, buffer = round & 1;
        // This buffer is full once the loads of all of its wavefronts have come (a barrier alone does not wait for loads into LDS), and
        // nobody reads the other any more.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (step + G < last)
            fetch(step + G, buffer ^ 1);
        if (step >= last)
            continue;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            bf16x8 fa[4], fb[4];
            const int place = ((kk * 4 + group) ^ (in_line & 7)) * 8;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                fa[i] = *reinterpret_cast<const bf16x8 *>(&lds[buffer][0][(wr + i * 16 + in_line) * kStep + place]);
                fb[i] = *reinterpret_cast<const bf16x8 *>(&lds[buffer][1][(wc + i * 16 + in_line) * kStep + place]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)   // b first: a lane's four results are neighbours in a row
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
        }
    }
    constexpr int R = 4 / G;             // of a wavefront's rows of four by 16 columns
    f32x4 sum[R][4];
    if constexpr (G == 2) {
        // the other group's half of the sums for this one's: rows 0 and 1 of four for the first group
        f32x4 *const give = reinterpret_cast<f32x4 *>(lds_raw) + (wave * 8) * 64 + lane;   // [wavefront][8][64], twice
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                give[part * 2048 + (i * 4 + k) * 64] = part == 0 ? acc[i + 2][k] : acc[i][k];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                sum[i][k] = (part == 0 ? acc[i][k] : acc[i + 2][k]) + give[(1 - part) * 2048 + (i * 4 + k) * 64];
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                sum[i][k] = acc[i][k];
    }
    const int64_t r0 = (int64_t)row_tile * kProductTile + wr + part * 32 + in_line, c0 = (int64_t)col_tile * kProductTile + wc + group * 4;
    if (j.partials) {
        const int64_t rows_pad = (int64_t)row_tiles * kProductTile, cols_pad = (int64_t)col_tiles * kProductTile;
        float *const to = j.partials + ((int64_t)split * rows_pad + r0) * cols_pad + c0;
        if (j.accumulate) {
            f32x4 was[R][4];
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    was[i][k] = *reinterpret_cast<const f32x4 *>(to + i * 16 * cols_pad + k * 16);
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    sum[i][k] += was[i][k];
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *reinterpret_cast<f32x4 *>(to + i * 16 * cols_pad + k * 16) = sum[i][k];
    } else if (j.o.type == AXC_F32) {
        store_tile<float>(j, row_tile, col_tile, r0, c0, sum);
    } else if (j.o.type == AXC_BF16) {
        store_tile<bf16>(j, row_tile, col_tile, r0, c0, sum);
    } else {
        store_tile<f16>(j, row_tile, col_tile, r0, c0, sum);
    }
}

template <typename T>
__device__ __forceinline__ void product_out(const Product &j, int block)
{
    const int64_t rows_pad = product_pad(j.rows), cols_pad = product_pad(j.cols);
    const int across = (int)((j.cols + 255) / 256);
    const int64_t c = ((int64_t)(block % across) * 64 + (threadIdx.x & 63)) * 4, r = (int64_t)(block / across) * 4 + threadIdx.x / 64;
    if (c >= j.cols || r >= j.rows)
        return;
    const Results<T> results(j.o);
    f32x4 sum = {};
#pragma unroll 8
    for (int s = 0; s < j.splits; ++s)
        sum += *reinterpret_cast<const f32x4 *>(j.partials + ((int64_t)s * rows_pad + r) * cols_pad + c);
    results.store_some(r, c, j.cols, sum);
}
__global__ void __launch_bounds__(256) products_out_kernel(Product first_product, int first_blocks, Product second_product)
{
    const bool first = (int)blockIdx.x < first_blocks;
    const Product &j = first ? first_product : second_product;
    const int block = first ? (int)blockIdx.x : (int)blockIdx.x - first_blocks;
    if (j.o.type == AXC_F32)
        product_out<float>(j, block);
    else if (j.o.type == AXC_BF16)
        product_out<bf16>(j, block);
    else
        product_out<f16>(j, block);
}

} // namespace

hipError_t launch_grad_prep(const GradSource &of_run, bool loss, int64_t first, int64_t run_rows, int64_t rows, int64_t cols,
                            int64_t ld, int straight_parts, bf16 *straight, int turned_parts, bf16 *turned, float *column_partials,
                            const CenteredJob &x, const CenteredJob &kernel, const RangeSource *ranges, Grids *grids,
                            hipStream_t stream)
{
    const int64_t rows_pad = product_pad(rows);
    // the last run makes the pad rows too
    const int64_t high = first + run_rows < rows ? run_rows : rows_pad - first;
    const int term_rows = (int)(high / 64), term_cols = (int)(product_pad(cols) / 64);
    auto tiles = [](int64_t n) { return (int)(product_pad(n) / 64); };
    const int x_rows = x.out ? tiles(x.rows) : 0, x_cols = x.out ? tiles(x.cols) : 1;
    const int k_rows = kernel.out ? tiles(kernel.rows) : 0, k_cols = kernel.out ? tiles(kernel.cols) : 1;
    const int64_t blocks = (int64_t)term_rows * term_cols + (int64_t)x_rows * x_cols + (int64_t)k_rows * k_cols;
    if (blocks >= (int64_t)1 << 31)
        return hipErrorInvalidConfiguration;
#define AXC_PREP(SOURCE, I)                                                                                                        \
    hipLaunchKernelGGL((grad_prep_kernel<SOURCE, I>), dim3((unsigned)blocks), dim3(256), 0, stream, of_run, term_rows, term_cols,  \
                       first / 64, run_rows, rows_pad, cols, ld, straight_parts, straight, turned_parts, turned, column_partials,  \
                       x, x_rows, x_cols, kernel, k_cols, ranges ? ranges[0] : RangeSource{}, ranges ? ranges[1] : RangeSource{},  \
                       ranges != nullptr, grids)
    const bool narrow = of_run.sums.K <= kNarrowDepth;
    if (!loss)
        AXC_PREP(0, uint32_t);
    else if (of_run.sums.raw.turned && narrow)
        AXC_PREP(2, uint32_t);
    else if (of_run.sums.raw.turned)
        AXC_PREP(2, int64_t);
    else if (narrow)
        AXC_PREP(1, uint32_t);
    else
        AXC_PREP(1, int64_t);
#undef AXC_PREP
    return hipGetLastError();
}

static int64_t product_tiles(int64_t rows, int64_t cols)
{
    return (product_pad(rows) / kProductTile) * (product_pad(cols) / kProductTile);
}
constexpr int64_t kManyTiles = 512;      // two workgroups a CU
void plan_products(const ProductShape *shapes, int count, ProductPlan *plans)
{
    int64_t tiles = 0, all = 0;
    for (int i = 0; i < count; ++i) {
        const int64_t t = product_tiles(shapes[i].rows, shapes[i].cols);
        tiles += t;
        all += t * (product_pad(shapes[i].depth) / kStep) * shapes[i].parts;
    }
    // steps of the depth that a workgroup takes, 4 at least
    const int64_t each = std::max<int64_t>(4, all / (tiles >= kManyTiles ? kManyTiles : kManyTiles / 2));
    for (int i = 0; i < count; ++i) {
        const ProductShape &s = shapes[i];
        const int64_t splits = std::max<int64_t>(1, product_pad(s.depth) / kStep * s.parts / each);
        plans[i] = {(int)splits, 0};
        if (splits > 1 || s.keep)
            plans[i].partial_bytes = (size_t)splits * product_pad(s.rows) * product_pad(s.cols) * sizeof(float);
    }
}

template <int G>
static hipError_t products(const Product *p, int count, int first_tiles, int tiles, const ColumnJob &job, hipStream_t stream)
{
    if (hipError_t e = set_max_dynamic_lds_once(reinterpret_cast<const void *>(&products_kernel<G>), product_lds(G)))
        return e;
    hipLaunchKernelGGL(products_kernel<G>, dim3((unsigned)(tiles + job.blocks())), dim3(G * 256), product_lds(G), stream, p[0],
                       first_tiles, p[count - 1], tiles, job);
    return hipGetLastError();
}
hipError_t launch_products(const Product *p, int count, const ColumnJob &job, hipStream_t stream)
{
    int64_t plain = 0, tiles[2] = {};
    for (int i = 0; i < count; ++i) {
        tiles[i] = product_tiles(p[i].rows, p[i].cols) * p[i].splits;
        plain += product_tiles(p[i].rows, p[i].cols);
    }
    return plain >= kManyTiles ? products<1>(p, count, (int)tiles[0], (int)(tiles[0] + tiles[1]), job, stream)
                               : products<2>(p, count, (int)tiles[0], (int)(tiles[0] + tiles[1]), job, stream);
}

hipError_t launch_products_out(const Product *p, int count, hipStream_t stream)
{
    int64_t blocks[2] = {};
    for (int i = 0; i < count; ++i)
        blocks[i] = (p[i].cols + 255) / 256 * ((p[i].rows + 3) / 4);
    hipLaunchKernelGGL(products_out_kernel, dim3((unsigned)(blocks[0] + blocks[1])), dim3(256), 0, stream, p[0], (int)blocks[0],
                       p[count - 1]);
    return hipGetLastError();
}

hipError_t launch_column_sums(const ColumnJob &job, hipStream_t stream)
{
    hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)job.blocks()), dim3(512), 0, stream, job);
    return hipGetLastError();
}

} // namespace axc
