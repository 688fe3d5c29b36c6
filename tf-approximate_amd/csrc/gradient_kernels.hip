// Products of a layer's backward pass: gradients times codes.
//
//   dz = dy activation'(pre)                                  [M][N]
//   dx[m][k]  = s_k  sum_n dz[m][n] (b[k][n] - z_k)           where x lies inside its grid, else 0
//   dkernel[k][n] = s_in sum_m (a[m][k] - z_in) dz[m][n]      where the kernel does
//
// Codes minus their zero point are whole numbers of at most 8 bits: bfloat16 holds them exactly, so the matrix cores' bfloat16
// instructions multiply them without a rounding.  The gradient is the other operand.  For a bfloat16 result it is rounded to
// bfloat16 itself; for float16 it is the sum of two bfloat16 terms (16 bits), for float32 of three (24 bits, all that a float
// has), and the product runs over the terms one after the other as over a longer depth.  Sums are float32 throughout.
//
// Both products run over the depth that is contiguous in both operands: dz is written straight and turned, the input's codes
// turned, the kernel's straight.  All are padded with zeros to whole tiles, so the product has no edges to look at but in its
// stores.
#include "layers_internal.h"

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
        float share, lse;
        int64_t target;
    };
    __device__ __forceinline__ Line line(int64_t r) const
    {
        return {b.row(g.sums.row_sums[r]), g.coefficient[r], g.lse[r], g.targets[r] - g.first_column};
    }
    __device__ __forceinline__ float bias(int64_t c) const { return g.bias ? load_any(g.bias, c, g.bias_type) : 0.0f; }
    __device__ __forceinline__ I column(int64_t c) const { return b.column(g.sums.column_sums[c]); }
    __device__ __forceinline__ float operator()(int32_t sum, const Line &l, I column, float bias, int64_t c) const
    {
        float z = __fmul_rn(Bracket<I>::value(sum, l.term, column), scale);
        if (g.bias)
            z = __fadd_rn(z, bias);
        const float p = __expf(z - l.lse);
        // a row that does not count has no gradient, whatever its logits are
        return l.share == 0.0f ? 0.0f : l.share * (c == l.target ? p - 1.0f : p);
    }
};

// Gradient in front of the product, 64 x 64 of it a workgroup: into LDS, and from there out straight, turned, and summed by columns.
// SOURCE 0: dense; 1: logits' sums by rows, 2: turned.  `first`: the run's first row, in units of 64.
template <int SOURCE, typename I>
__global__ void __launch_bounds__(256) grad_terms_kernel(GradSource g, int64_t first, int64_t rows, int64_t rows_pad, int64_t cols,
                                                         int64_t ld, int straight_parts, bf16 *__restrict__ straight,
                                                         int turned_parts, bf16 *__restrict__ turned,
                                                         float *__restrict__ column_partials)
{
    __shared__ float tile[64][65];
    const int64_t r0 = (int64_t)blockIdx.y * 64, c0 = (int64_t)blockIdx.x * 64;
    const int64_t cols_pad = (int64_t)gridDim.x * 64;
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
        column_partials[(first + blockIdx.y) * cols_pad + c0 + threadIdx.x] = sum;
    }
}

// Codes minus zero point of a tensor, straight or turned, 64 x 64 a workgroup; pads are zeros.
template <bool TURN>
__global__ void __launch_bounds__(256) centered_kernel(const void *values, int type, int64_t rows, int64_t cols, int64_t ld,
                                                       const Grid *grid, bf16 *__restrict__ out)
{
    __shared__ float tile[TURN ? 64 : 1][65];
    const int64_t r0 = (int64_t)blockIdx.y * 64, c0 = (int64_t)blockIdx.x * 64;
    const int quad = (threadIdx.x & 15) * 4, line = threadIdx.x / 16;
    const Grid g = *grid;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = r0 + line + 16 * i, c = c0 + quad;
        float v[4] = {};
        if (r < rows && c < cols) {
            load_four_any(values, r * ld + c, cols - c, type, v);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = c + j < cols ? (float)((int)code_of(v[j], g) - g.zero) : 0.0f;
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
            *reinterpret_cast<bf16x4 *>(out + r * ((int64_t)gridDim.x * 64) + c) = b;
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
            *reinterpret_cast<bf16x4 *>(out + (c0 + col) * ((int64_t)gridDim.y * 64) + r0 + quad) = b;
        }
    }
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
constexpr int kGroups = 2;  // of four wavefronts, which take the steps in turn
constexpr int kProductThreads = kGroups * 256;
constexpr int kProductLds = kGroups * 2 * 2 * kProductTile * kStep * 2;

__device__ __forceinline__ void load_to_lds(const bf16 *from, bf16 *to)
{
    // 16 bytes a lane, to `to` of the wavefront plus 16 times the lane
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t *)from,
                                     (__attribute__((address_space(3))) uint32_t *)to, 16, 0, 0);
}

// A tile of 128 x 128 by two groups of four wavefronts, each of which multiplies every other step of the depth, 64 x 64 a wavefront,
// and has two buffers of 64 of the depth in LDS, filled straight from memory while the other is multiplied: two wavefronts a SIMD, so
// that one reads while the other multiplies, where there are no more tiles than CUs.  At the end the groups exchange half of their
// sums each.
// In LDS a line of 64 elements is eight chunks of 16 bytes, chunk q of line r in place q ^ (r & 7): the 16 lanes that read
// neighbouring lines then meet different banks.  The loads write LDS in order, so it is their addresses that are exchanged.
// PARTIAL: sums go to `partials` (added to what is there with `accumulate`).
template <typename T, bool PARTIAL>
__global__ void __launch_bounds__(kProductThreads) product_kernel(const bf16 *__restrict__ a, const bf16 *__restrict__ b, int64_t rows,
                                                         int64_t cols, int row_tiles, int col_tiles, int depth, int parts,
                                                         int split_a, int splits, float *__restrict__ partials, int accumulate,
                                                         ProductOut o)
{
    extern __shared__ __align__(16) bf16 lds_raw[];
    // Workgroups go round the eight XCDs; each XCD gets a run of neighbouring tiles, in bands of eight row tiles, so that its L2
    // serves them.
    const int tiles = row_tiles * col_tiles * splits;
    int id = (int)blockIdx.x;
    {
        const int per = tiles / 8, more = tiles % 8, xcd = id % 8;
        id = xcd * per + (xcd < more ? xcd : more) + id / 8;
    }
    const int split = id / (row_tiles * col_tiles);
    id -= split * row_tiles * col_tiles;
    const int band = id / (8 * col_tiles), in_band = id - band * 8 * col_tiles;
    const int band_rows = row_tiles - band * 8 < 8 ? row_tiles - band * 8 : 8;
    const int row_tile = band * 8 + in_band % band_rows, col_tile = in_band / band_rows;

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
    const int rounds = (last - first + kGroups - 1) / kGroups;
    if (first + part < last)
        fetch(first + part, 0);
    for (int round = 0; round < rounds; ++round) {
        const int step = first + round * kGroups + part, buffer = round & 1;
        // This buffer is full once the loads of all of its wavefronts have come (a barrier alone does not wait for loads into LDS), and
        // nobody reads the other any more.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (step + kGroups < last)
            fetch(step + kGroups, buffer ^ 1);
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
    // the other group's half of the sums for this one's: rows 0 and 1 of four for the first group
    f32x4 *const give = reinterpret_cast<f32x4 *>(lds_raw) + (wave * 8) * 64 + lane;   // [wavefront][8][64], twice
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            give[part * 2048 + (i * 4 + j) * 64] = part == 0 ? acc[i + 2][j] : acc[i][j];
    __syncthreads();
    f32x4 sum[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            sum[i][j] = (part == 0 ? acc[i][j] : acc[i + 2][j]) + give[(1 - part) * 2048 + (i * 4 + j) * 64];
    // What is read for the results is read all at once, where the tile has no edge: value by value it took as long as the product.
    const int64_t r0 = (int64_t)row_tile * kProductTile + wr + part * 32 + in_line, c0 = (int64_t)col_tile * kProductTile + wc + group * 4;
    if constexpr (PARTIAL) {
        const int64_t rows_pad = (int64_t)row_tiles * kProductTile, cols_pad = (int64_t)col_tiles * kProductTile;
        float *const to = partials + ((int64_t)split * rows_pad + r0) * cols_pad + c0;
        if (accumulate) {
            f32x4 was[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    was[i][j] = *reinterpret_cast<const f32x4 *>(to + i * 16 * cols_pad + j * 16);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    sum[i][j] += was[i][j];
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<f32x4 *>(to + i * 16 * cols_pad + j * 16) = sum[i][j];
    } else {
        const Results<T> results(o);
        if (results.aligned && (int64_t)(row_tile + 1) * kProductTile <= rows && (int64_t)(col_tile + 1) * kProductTile <= cols) {
            typename Results<T>::four at[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    at[i][j] = results.values_at(r0 + i * 16, c0 + j * 16);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    results.store(r0 + i * 16, c0 + j * 16, at[i][j], sum[i][j]);
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (r0 + i * 16 < rows && c0 + j * 16 < cols)
                        results.store_some(r0 + i * 16, c0 + j * 16, cols, sum[i][j]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) product_out_kernel(const float *__restrict__ partials, int splits, int64_t rows, int64_t cols,
                                                          int64_t rows_pad, int64_t cols_pad, ProductOut o)
{
    const int64_t c = ((int64_t)blockIdx.x * 64 + (threadIdx.x & 63)) * 4;
    if (c >= cols)
        return;
    const Results<T> results(o);
    for (int64_t r = (int64_t)blockIdx.y * 4 + threadIdx.x / 64; r < rows; r += (int64_t)gridDim.y * 4) {
        f32x4 sum = {};
#pragma unroll 8
        for (int s = 0; s < splits; ++s)
            sum += *reinterpret_cast<const f32x4 *>(partials + ((int64_t)s * rows_pad + r) * cols_pad + c);
        results.store_some(r, c, cols, sum);
    }
}

// Sums of the column partials, 64 columns a workgroup, in one order.
__global__ void __launch_bounds__(256) column_sums_kernel(const float *__restrict__ partials, int64_t count, int64_t cols,
                                                          int64_t pitch, const float *factor, void *out, int type)
{
    __shared__ float red[4][64];
    const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    float sum = 0.0f;
    if (c < cols)
        for (int64_t i = threadIdx.x / 64; i < count; i += 4)
            sum += partials[i * pitch + c];
    red[threadIdx.x / 64][threadIdx.x & 63] = sum;
    __syncthreads();
    if (threadIdx.x < 64 && c < cols)
        store_any(out, c, type, ((red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x])) *
                                    (factor ? *factor : 1.0f));
}

} // namespace

hipError_t launch_grad_terms(const GradSource &of_run, bool loss, int64_t first, int64_t run_rows, int64_t rows, int64_t cols,
                             int64_t ld, int straight_parts, bf16 *straight, int turned_parts, bf16 *turned, float *column_partials,
                             hipStream_t stream)
{
    const int64_t rows_pad = product_pad(rows);
    // the last run makes the pad rows too
    const int64_t high = first + run_rows < rows ? run_rows : rows_pad - first;
    const dim3 grid((unsigned)(product_pad(cols) / 64), (unsigned)(high / 64));
#define AXC_TERMS(SOURCE, I)                                                                                                       \
    hipLaunchKernelGGL((grad_terms_kernel<SOURCE, I>), grid, dim3(256), 0, stream, of_run, first / 64, run_rows, rows_pad, cols, ld, \
                       straight_parts, straight, turned_parts, turned, column_partials)
    const bool narrow = of_run.sums.K <= kNarrowDepth;
    if (!loss)
        AXC_TERMS(0, uint32_t);
    else if (of_run.sums.raw.turned && narrow)
        AXC_TERMS(2, uint32_t);
    else if (of_run.sums.raw.turned)
        AXC_TERMS(2, int64_t);
    else if (narrow)
        AXC_TERMS(1, uint32_t);
    else
        AXC_TERMS(1, int64_t);
#undef AXC_TERMS
    return hipGetLastError();
}

hipError_t launch_centered(const void *v, int type, int64_t rows, int64_t cols, int64_t ld, const Grid *grid, bool turn, bf16 *out,
                           hipStream_t stream)
{
    const dim3 blocks((unsigned)(product_pad(cols) / 64), (unsigned)(product_pad(rows) / 64));
    if (turn)
        hipLaunchKernelGGL(centered_kernel<true>, blocks, dim3(256), 0, stream, v, type, rows, cols, ld, grid, out);
    else
        hipLaunchKernelGGL(centered_kernel<false>, blocks, dim3(256), 0, stream, v, type, rows, cols, ld, grid, out);
    return hipGetLastError();
}

ProductPlan plan_product(int64_t rows, int64_t cols, int64_t depth_pad, int parts, bool keep)
{
    const int64_t tiles = (product_pad(rows) / kProductTile) * (product_pad(cols) / kProductTile);
    const int64_t steps = depth_pad / kStep * parts;
    int64_t splits = tiles >= 256 ? 1 : 512 / tiles;
    if (splits > steps / 4)
        splits = steps / 4;
    if (splits < 1)
        splits = 1;
    ProductPlan plan = {(int)splits, 0};
    if (splits > 1 || keep)
        plan.partial_bytes = (size_t)splits * product_pad(rows) * product_pad(cols) * sizeof(float);
    return plan;
}

template <typename T, bool PARTIAL>
static hipError_t product(const bf16 *a, const bf16 *b, int64_t rows, int64_t cols, int64_t depth_pad, int parts, bool split_a,
                          int splits, float *partials, bool accumulate, const ProductOut &o, hipStream_t stream)
{
    const int row_tiles = (int)(product_pad(rows) / kProductTile), col_tiles = (int)(product_pad(cols) / kProductTile);
    if (hipError_t e = set_max_dynamic_lds_once(reinterpret_cast<const void *>(&product_kernel<T, PARTIAL>), kProductLds))
        return e;
    hipLaunchKernelGGL((product_kernel<T, PARTIAL>), dim3((unsigned)((int64_t)row_tiles * col_tiles * splits)), dim3(kProductThreads),
                       kProductLds,
                       stream, a, b, rows, cols, row_tiles, col_tiles, (int)depth_pad, parts, (int)split_a, splits, partials,
                       (int)accumulate, o);
    return hipGetLastError();
}

hipError_t launch_product(const bf16 *a, const bf16 *b, int64_t rows, int64_t cols, int64_t depth_pad, int parts, bool split_a,
                          const ProductPlan &plan, float *partials, bool keep, bool accumulate, const ProductOut &o,
                          hipStream_t stream)
{
    if (plan.splits > 1 || keep) {
        if (hipError_t e = product<float, true>(a, b, rows, cols, depth_pad, parts, split_a, plan.splits, partials, accumulate, o,
                                                stream))
            return e;
        return keep ? hipSuccess : launch_product_out(partials, plan.splits, rows, cols, o, stream);
    }
    if (o.type == AXC_F32)
        return product<float, false>(a, b, rows, cols, depth_pad, parts, split_a, 1, nullptr, false, o, stream);
    if (o.type == AXC_BF16)
        return product<bf16, false>(a, b, rows, cols, depth_pad, parts, split_a, 1, nullptr, false, o, stream);
    return product<f16, false>(a, b, rows, cols, depth_pad, parts, split_a, 1, nullptr, false, o, stream);
}

hipError_t launch_product_out(const float *partials, int splits, int64_t rows, int64_t cols, const ProductOut &o,
                              hipStream_t stream)
{
    const int64_t by = (rows + 3) / 4;
    const dim3 grid((unsigned)((cols + 255) / 256), (unsigned)(by > 16384 ? 16384 : by));
    const int64_t rows_pad = product_pad(rows), cols_pad = product_pad(cols);
    if (o.type == AXC_F32)
        hipLaunchKernelGGL(product_out_kernel<float>, grid, dim3(256), 0, stream, partials, splits, rows, cols, rows_pad, cols_pad, o);
    else if (o.type == AXC_BF16)
        hipLaunchKernelGGL(product_out_kernel<bf16>, grid, dim3(256), 0, stream, partials, splits, rows, cols, rows_pad, cols_pad, o);
    else
        hipLaunchKernelGGL(product_out_kernel<f16>, grid, dim3(256), 0, stream, partials, splits, rows, cols, rows_pad, cols_pad, o);
    return hipGetLastError();
}

hipError_t launch_column_sums(const float *partials, int64_t count, int64_t cols, int64_t pitch, const float *factor, void *out,
                              int type, hipStream_t stream)
{
    hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)((cols + 63) / 64)), dim3(256), 0, stream, partials, count, cols, pitch,
                       factor, out, type);
    return hipGetLastError();
}

} // namespace axc
