// Dense layers by table products: ranges, codes, the sums of few rows, and what is made of the sums.
//
//   product[m][n] = s_in s_k sum_k (T[a][b] - z_k a - z_in b + z_in z_k)
//                 = s_in s_k (sum_k T[a][b] - z_k sum_k a - z_in sum_k b + K z_in z_k)
//
// a, b: codes of the input and of the kernel, s, z: scale and zero point of their grids.  Everything in the brackets is a whole
// number and is computed as one, so a product is rounded three times: s_in s_k, the bracket, and the two multiplied.
//
// The sums of many rows are made by the kernels that make them for 1x1 convolutions (axc_conv2d_codes_acc_i32); those of few
// rows, where building rows for every filter element would cost more than the lookups, by few_rows_kernel.
#include "layers_internal.h"

namespace axc {
namespace {

// ---- ranges ----
// fminf and fmaxf pass over NaN, as the convolutions' range pass does.
template <typename T>
__device__ void range_of(const T *__restrict__ p, int64_t n, int64_t index, int64_t stride, float &lo, float &hi)
{
    constexpr int V = 16 / sizeof(T);
    int64_t done = 0;
    if (((uintptr_t)p & 15) == 0) {
        const int64_t nv = n / V;
#pragma unroll 4
        for (int64_t i = index; i < nv; i += stride) {
            float v[V];
            load_values<T, V>(p + i * V, V, true, 0.0f, v);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                lo = fminf(lo, v[j]);
                hi = fmaxf(hi, v[j]);
            }
        }
        done = nv * V;
    }
    for (int64_t i = done + index; i < n; i += stride) {
        lo = fminf(lo, (float)p[i]);
        hi = fmaxf(hi, (float)p[i]);
    }
}
__device__ void range_of_any(const void *p, int type, int64_t n, int64_t index, int64_t stride, float &lo, float &hi)
{
    if (type == AXC_F32)
        range_of(static_cast<const float *>(p), n, index, stride, lo, hi);
    else if (type == AXC_BF16)
        range_of(static_cast<const bf16 *>(p), n, index, stride, lo, hi);
    else
        range_of(static_cast<const f16 *>(p), n, index, stride, lo, hi);
}

// One pair per workgroup; the first x_blocks take the input, the others the kernel.  All of them clear `zeros`, into which a
// later launch adds.
__global__ void __launch_bounds__(1024) range_kernel(const void *x, int x_type, int64_t nx, int x_blocks, const void *kernel,
                                                     int kernel_type, int64_t nk, float *x_pairs, float *kernel_pairs,
                                                     int32_t *zeros, int64_t n_zeros)
{
    __shared__ float red[32];
    const bool second = (int)blockIdx.x >= x_blocks;
    const int block = second ? (int)blockIdx.x - x_blocks : (int)blockIdx.x;
    const int blocks = second ? (int)gridDim.x - x_blocks : x_blocks;
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < n_zeros; i += (int64_t)gridDim.x * 1024)
        zeros[i] = 0;
    float lo = INFINITY, hi = -INFINITY;
    range_of_any(second ? kernel : x, second ? kernel_type : x_type, second ? nk : nx, (int64_t)block * 1024 + threadIdx.x,
                 (int64_t)blocks * 1024, lo, hi);
    block_range(lo, hi, red);
    if (threadIdx.x == 0) {
        float *const to = second ? kernel_pairs : x_pairs;
        to[2 * block] = lo;
        to[2 * block + 1] = hi;
    }
}

__device__ void fold(const RangeSource &src, float &lo, float &hi, float *red)
{
    lo = src.lo;
    hi = src.hi;
    if (src.pairs) {
        lo = INFINITY;
        hi = -INFINITY;
        for (int i = threadIdx.x; i < src.count; i += blockDim.x) {
            const float2 p = reinterpret_cast<const float2 *>(src.pairs)[i];
            lo = fminf(lo, p.x);
            hi = fmaxf(hi, p.y);
        }
        block_range(lo, hi, red);
    }
}

__global__ void __launch_bounds__(256) grids_kernel(RangeSource in, RangeSource kernel, int has_in, int has_kernel, Grids *grids)
{
    __shared__ float red[8];
    float lo, hi;
    if (has_in) {
        fold(in, lo, hi, red);
        if (threadIdx.x == 0)
            grids->in = grid_of_range(lo, hi);
    }
    if (has_kernel) {
        fold(kernel, lo, hi, red);
        if (threadIdx.x == 0)
            grids->kernel = grid_of_range(lo, hi);
    }
}

// ---- codes ----
// Codes of one row by a group of `threads` threads, and this thread's part of their sum.  Behind the depth come pad codes, 0.
template <typename T>
__device__ int32_t row_codes(const T *__restrict__ x, int K, int Kp, bool whole, const Grid &g, uint8_t *__restrict__ codes,
                             int thread, int threads)
{
    int32_t sum = 0;
    for (int k = 4 * thread; k < Kp; k += 4 * threads) {
        float v[4];
        load_values<T, 4>(x + k, K - k, whole, 0.0f, v);
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t c = whole || k + j < K ? code_of(v[j], g) : 0u;
            word |= c << (8 * j);
            sum += (int32_t)c;
        }
        *reinterpret_cast<uint32_t *>(codes + k) = word;
    }
    return sum;
}
__device__ __forceinline__ int32_t row_codes_any(const void *x, int type, int64_t at, int K, int Kp, const Grid &g, uint8_t *codes,
                                                 int thread, int threads)
{
    // (a row's first value is aligned as the tensor's is where the depth is a multiple of four)
    const bool whole = (K & 3) == 0 && ((uintptr_t)x & (type == AXC_F32 ? 15 : 7)) == 0;
    if (type == AXC_F32)
        return row_codes(static_cast<const float *>(x) + at, K, Kp, whole, g, codes, thread, threads);
    if (type == AXC_BF16)
        return row_codes(static_cast<const bf16 *>(x) + at, K, Kp, whole, g, codes, thread, threads);
    return row_codes(static_cast<const f16 *>(x) + at, K, Kp, whole, g, codes, thread, threads);
}

// Few rows: every workgroup finds the range itself, of all rows, and then takes its own row.
__global__ void __launch_bounds__(512) few_codes_kernel(const void *x, int type, int rows, int K, int Kp, RangeSource src,
                                                        const Grid *kernel_grid, Grids *grids, uint8_t *codes, int32_t *row_sums)
{
    __shared__ float red[16];
    __shared__ int32_t sums[8];
    float lo, hi;
    if (!src.pairs && src.count < 0) {
        lo = INFINITY;
        hi = -INFINITY;
        range_of_any(x, type, (int64_t)rows * K, threadIdx.x, 512, lo, hi);
        block_range(lo, hi, red);
    } else {
        fold(src, lo, hi, red);
    }
    const Grid g = grid_of_range(lo, hi);
    const int64_t r = blockIdx.x;
    const int32_t part = wave_sum(row_codes_any(x, type, r * K, K, Kp, g, codes + r * Kp, (int)threadIdx.x, 512));
    if ((threadIdx.x & 63) == 0)
        sums[threadIdx.x / 64] = part;
    __syncthreads();
    if (threadIdx.x == 0) {
        int32_t sum = 0;
        for (int i = 0; i < 8; ++i)
            sum += sums[i];
        row_sums[r] = sum;
        if (r == 0) {
            grids->in = g;
            grids->kernel = *kernel_grid;
        }
    }
}

template <typename T>
__device__ void kernel_slab(const T *__restrict__ w, int K, int64_t N, const Pieces &pc, const Grid &g, uint8_t *__restrict__ codes,
                            int64_t c, int k0, int lines, int (&sum)[4])
{
    const int piece = (int)(c / pc.width);
    uint8_t *const to = codes + pc.offset(piece) + (c - pc.first(piece));
    const int pitch = pc.width_of(piece);
    const bool whole = c + 4 <= N && (N & 3) == 0 && ((uintptr_t)w & (4 * sizeof(T) - 1)) == 0;
#pragma unroll 4
    for (int i = 0; i < lines; ++i) {
        const int k = k0 + 4 * i;
        if (k >= pc.Kp)
            break;
        float v[4];
        uint32_t word = 0;
        if (k < K) {
            load_values<T, 4>(w + (int64_t)k * N + c, N - c, whole, 0.0f, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t q = c + j < N ? code_of(v[j], g) : 0u;
                word |= q << (8 * j);
                sum[j] += (int)q;
            }
        }
        *reinterpret_cast<uint32_t *>(to + (size_t)k * pitch) = word;
    }
}

// The first x_blocks workgroups take four rows of the input each, a wavefront a row (rows up to the next multiple of four are pad
// rows, of code 0).  The others take 256 columns of the kernel, four a lane, by 4 * lines of the depth, a wavefront every fourth;
// column sums are added to what the launch before cleared, as whole numbers, so in any order.  Every workgroup makes the grid it
// needs out of the range's pairs itself: a launch for that alone would be longer than folding 256 of them.
__global__ void __launch_bounds__(256) codes_kernel(CodesJob job, int x_blocks, int column_blocks, int lines)
{
    __shared__ float ends[8];
    __shared__ int32_t red[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    float lo, hi;
    if ((int)blockIdx.x < x_blocks) {
        fold(job.x_range, lo, hi, ends);
        const Grid g = grid_of_range(lo, hi);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            job.grids->in = g;
            if (!job.kernel)
                job.grids->kernel = *job.kernel_grid;
        }
        const int64_t r = (int64_t)blockIdx.x * 4 + wave;
        const int Kp = job.pieces.Kp;
        uint8_t *const codes = job.x_codes + r * Kp;
        int32_t sum = 0;
        if (r < job.rows)
            sum = row_codes_any(job.x, job.x_type, r * job.K, job.K, Kp, g, codes, lane, 64);
        else
            for (int k = 4 * lane; k < Kp; k += 256)
                *reinterpret_cast<uint32_t *>(codes + k) = 0u;
        sum = wave_sum(sum);
        if (lane == 0)
            job.row_sums[r] = sum;
        return;
    }
    fold(job.kernel_range, lo, hi, ends);
    const Grid g = grid_of_range(lo, hi);
    const int block = (int)blockIdx.x - x_blocks, slab = block / column_blocks;
    const int64_t first = (int64_t)(block - slab * column_blocks) * 256, c = first + 4 * lane;
    if (block == 0 && threadIdx.x == 0)
        job.grids->kernel = g;
    int sum[4] = {};
    if (c < job.pieces.Np) {
        const int k0 = slab * 4 * lines + wave;
        if (job.kernel_type == AXC_F32)
            kernel_slab(static_cast<const float *>(job.kernel), job.K, job.N, job.pieces, g, job.kernel_codes, c, k0, lines, sum);
        else if (job.kernel_type == AXC_BF16)
            kernel_slab(static_cast<const bf16 *>(job.kernel), job.K, job.N, job.pieces, g, job.kernel_codes, c, k0, lines, sum);
        else
            kernel_slab(static_cast<const f16 *>(job.kernel), job.K, job.N, job.pieces, g, job.kernel_codes, c, k0, lines, sum);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        red[wave][4 * lane + j] = sum[j];
    __syncthreads();
    const int64_t column = first + threadIdx.x;
    if (column < job.pieces.Np)
        atomicAdd(job.column_sums + column,
                  red[0][threadIdx.x] + red[1][threadIdx.x] + red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// ---- sums of few rows ----
// A pair of wavefronts takes MT rows, 1024 columns (eight a lane) and two elements of the depth at a time.  Each of the two turns the
// MT table rows that the rows' codes name at one of the elements into R[b] = entries of filter code b for all MT rows, in LDS; a lane
// then reads the entries of all MT rows for one weight with one access of 2 MT bytes.  Sums of two rows share a dword as they come:
// one register adds whole dwords modulo 2^32, another the upper halves, three instructions for two dwords.
// Eight pairs make a workgroup, which adds up their sums in LDS before it leaves them to the others' (parts of the depth).
// What bounds it for eight rows: lookups at random among 256 places of 16 bytes, 3 of 16 lanes on the busiest of 16 groups of banks
// (25 T/s), and the table rows out of the L2, 4 KiB for every element and 1024 columns.
constexpr int kFewGroups = 8;            // pairs of wavefronts
constexpr int kFewColumns = 1024;
constexpr int kFewRowsAtOnce = 4;        // whose sums are added up in LDS
template <int MT>
constexpr int few_lds_bytes()            // two buffers of table rows; then the sums of 16 wavefronts
{
    constexpr int table_rows = 2 * 2 * kFewGroups * 512 * MT, sums = 16 * 512 * 4 * (MT < kFewRowsAtOnce ? MT : kFewRowsAtOnce);
    return table_rows > sums ? table_rows : sums;
}

template <int MT>
__global__ void __launch_bounds__(1024) few_rows_kernel(const uint16_t *__restrict__ tableI, const uint8_t *__restrict__ x_codes,
                                                        int rows, int Kp, const uint8_t *__restrict__ kernel_codes, int width,
                                                        int32_t *__restrict__ acc)
{
    constexpr int H = (MT + 1) / 2;      // dwords of an entry
    constexpr int kRowBytes = 512 * MT;  // of R
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int group = wave >> 1, half = wave & 1;
    const int c = (int)blockIdx.x * kFewColumns + half * 512 + lane * 8;
    const int row0 = (int)blockIdx.z * MT;
    const int pairs = Kp / 2;
    const int first = (int)((int64_t)pairs * blockIdx.y / gridDim.y), last = (int)((int64_t)pairs * (blockIdx.y + 1) / gridDim.y);
    const int steps = (last - first + kFewGroups - 1) / kFewGroups;
    const bool in0 = c < width, in1 = c + 4 < width;

    uint2 t[MT];                         // table rows of this wavefront's element, four entries a lane
    uint32_t b[2][2];                    // weights of both elements, eight codes a lane
    auto load = [&](int step) {
        const int pair = first + step * kFewGroups + group;
        if (pair >= last)                // (uniform; what is there is not used)
            return;
        const int k = 2 * pair + half;
#pragma unroll
        for (int m = 0; m < MT; ++m) {   // (rows beyond the last repeat it; nobody stores them)
            const uint32_t four = *reinterpret_cast<const uint32_t *>(x_codes + (int64_t)min(row0 + m, rows - 1) * Kp + (k & ~3));
            t[m] = *reinterpret_cast<const uint2 *>(tableI + ((four >> (8 * (k & 3))) & 255u) * 256u + lane * 4);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint8_t *const p = kernel_codes + (size_t)(2 * pair + j) * width + c;
            b[j][0] = in0 ? *reinterpret_cast<const uint32_t *>(p) : 0u;
            b[j][1] = in1 ? *reinterpret_cast<const uint32_t *>(p + 4) : 0u;
        }
    };
    auto entry = [&](const unsigned char *R, uint32_t code, uint32_t (&e)[H]) {
        const unsigned char *const from = R + code * (2 * MT);
        if constexpr (MT == 1) {
            e[0] = *reinterpret_cast<const uint16_t *>(from);
        } else if constexpr (MT == 2) {
            e[0] = *reinterpret_cast<const uint32_t *>(from);
        } else if constexpr (MT == 4) {
            const uint2 v = *reinterpret_cast<const uint2 *>(from);
            e[0] = v.x;
            e[1] = v.y;
        } else {
            const uint4 v = *reinterpret_cast<const uint4 *>(from);
            e[0] = v.x;
            e[1] = v.y;
            e[2] = v.z;
            e[3] = v.w;
        }
    };

    uint32_t even[8][H] = {}, odd[8][H] = {};
    load(0);
    for (int step = 0; step < steps; ++step) {
        const bool there = first + step * kFewGroups + group < last;
        unsigned char *const R = lds + ((step & 1) * kFewGroups + group) * 2 * kRowBytes;
        if (there) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {   // filter code lane + 64 i
                const uint32_t sel = i & 1 ? 0x07060302u : 0x05040100u;
                uint32_t e[H];
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const uint32_t lo = i < 2 ? t[2 * h].x : t[2 * h].y;
                    const uint32_t hi = MT == 1 ? 0u : i < 2 ? t[(2 * h + 1) % MT].x : t[(2 * h + 1) % MT].y;
                    e[h] = __builtin_amdgcn_perm(hi, lo, sel);
                }
                unsigned char *const to = R + half * kRowBytes + (lane + 64 * i) * (2 * MT);
                if constexpr (MT == 1)
                    *reinterpret_cast<uint16_t *>(to) = (uint16_t)e[0];
                else if constexpr (MT == 2)
                    *reinterpret_cast<uint32_t *>(to) = e[0];
                else if constexpr (MT == 4)
                    *reinterpret_cast<uint2 *>(to) = make_uint2(e[0], e[1]);
                else
                    *reinterpret_cast<uint4 *>(to) = make_uint4(e[0], e[1], e[2], e[3]);
            }
        }
        uint32_t w[2][2] = {{b[0][0], b[0][1]}, {b[1][0], b[1][1]}};
        if (step + 1 < steps)
            load(step + 1);
        __syncthreads();   // both rows are there, and the other buffer's are no longer read
        if (there) {
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                uint32_t e0[H], e1[H];
                entry(R, (w[0][n / 4] >> (8 * (n & 3))) & 255u, e0);
                entry(R + kRowBytes, (w[1][n / 4] >> (8 * (n & 3))) & 255u, e1);
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    even[n][h] += e0[h] + e1[h];
                    if constexpr (MT > 1)
                        odd[n][h] += (e0[h] >> 16) + (e1[h] >> 16);
                }
            }
        }
    }
    // the pairs' sums, four rows at a time
    int32_t *const red = reinterpret_cast<int32_t *>(lds);
    constexpr int N = MT < kFewRowsAtOnce ? MT : kFewRowsAtOnce;
#pragma unroll
    for (int m0 = 0; m0 < MT; m0 += N) {
        __syncthreads();
#pragma unroll
        for (int m = 0; m < N; ++m)
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int of = m0 + m;
                const uint32_t v = of & 1 ? odd[n][of / 2] : even[n][of / 2] - (MT > 1 ? odd[n][of / 2] << 16 : 0u);
                red[(wave * N + m) * 512 + n * 64 + lane] = (int32_t)v;
            }
        __syncthreads();
        // column 8 l + n of a half stands at 64 n + l
        const int at = (threadIdx.x & 7) * 64 + (threadIdx.x & 511) / 8, of_half = threadIdx.x / 512;
        const int col = (int)blockIdx.x * kFewColumns + (int)threadIdx.x;
#pragma unroll
        for (int m = 0; m < N; ++m)
            if (row0 + m0 + m < rows && col < width) {
                int32_t sum = 0;
#pragma unroll
                for (int g = 0; g < kFewGroups; ++g)
                    sum += red[((2 * g + of_half) * N + m) * 512 + at];
                acc[((int64_t)blockIdx.y * rows + row0 + m0 + m) * width + col] = sum;
            }
    }
}

// ---- what is made of the sums ----
// residual + activation(product + bias), four neighbouring values of a row.  Products and everything behind them are in float32,
// rounded once to the output's type (`pre`, what the activation is given, once more).
template <typename T, typename I>
__device__ __forceinline__ void dense_four(const int32_t (&sum)[4], I row, const I (&column)[4], const float (&bias)[4], float scale,
                                           int64_t r, int c, int columns, bool whole, const DenseOut &o)
{
    float z[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        z[j] = __fmul_rn(Bracket<I>::value(sum[j], row, column[j]), scale);
        if (o.bias)
            z[j] = __fadd_rn(z[j], bias[j]);
    }
    activate_four(z, y, o.activation);
    const int64_t to = r * o.ld + c;
    if (o.pre)
        store_values<T, 4>(static_cast<T *>(o.pre) + to, columns - c, whole, z);
    if (o.residual) {
        float v[4];
        load_values<T, 4>(static_cast<const T *>(o.residual) + to, columns - c, whole, 0.0f, v);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            y[j] = __fadd_rn(y[j], v[j]);
    }
    store_values<T, 4>(static_cast<T *>(o.out) + to, columns - c, whole, y);
}
template <typename T>
__device__ __forceinline__ bool whole_fours(int c, int columns, const DenseOut &o)
{
    return c + 4 <= columns && (o.ld & 3) == 0 &&
           (((uintptr_t)o.out | (uintptr_t)o.residual | (uintptr_t)o.pre) & (4 * sizeof(T) - 1)) == 0;
}
template <typename I>
__device__ __forceinline__ void column_terms(const TableSums &s, const Bracket<I> &b, int c, int columns, const DenseOut &o,
                                             I (&column)[4], float (&bias)[4])
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool there = c + j < columns;
        column[j] = there ? b.column(s.column_sums[c + j]) : (I)0;
        bias[j] = there && o.bias ? load_any(o.bias, c + j, o.bias_type) : 0.0f;
    }
}

// Sums by rows: four columns a lane, a wavefront a row at a time.
template <typename T, typename I>
__global__ void __launch_bounds__(256) dense_out_kernel(TableSums s, int64_t rows, int columns, DenseOut o)
{
    const int c = ((int)blockIdx.x * 64 + (threadIdx.x & 63)) * 4;
    if (c >= columns)
        return;
    const float scale = __fmul_rn(s.grids->in.scale, s.grids->kernel.scale);
    const Bracket<I> b(s);
    const bool whole = whole_fours<T>(c, columns, o);
    I column[4];
    float bias[4];
    column_terms(s, b, c, columns, o, column, bias);
    for (int64_t r = (int64_t)blockIdx.y * 4 + threadIdx.x / 64; r < rows; r += (int64_t)gridDim.y * 4) {
        const i32x4 t = four_sums(s.raw, r, c);
        const int32_t sum[4] = {t[0], t[1], t[2], t[3]};
        dense_four<T, I>(sum, b.row(s.row_sums[r]), column, bias, scale, r, c, columns, whole, o);
    }
}

// Sums by rows of few rows, in many parts: the four wavefronts take a quarter of the parts each.
template <typename T, typename I>
__global__ void __launch_bounds__(256) dense_out_parts_kernel(TableSums s, int columns, DenseOut o)
{
    __shared__ i32x4 red[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const int c = ((int)blockIdx.x * 64 + lane) * 4;
    const int64_t r = blockIdx.y;
    i32x4 t = {};
    if (c < columns) {
        const int32_t *const p = s.raw.acc + r * s.raw.pitch + c;
#pragma unroll 8
        for (int i = wave; i < s.raw.splits; i += 4)
            t += *reinterpret_cast<const i32x4 *>(p + i * s.raw.split_stride);
    }
    red[wave][lane] = t;
    __syncthreads();
    if (wave != 0 || c >= columns)
        return;
    t = red[0][lane] + red[1][lane] + red[2][lane] + red[3][lane];
    const int32_t sum[4] = {t[0], t[1], t[2], t[3]};
    const Bracket<I> b(s);
    I column[4];
    float bias[4];
    column_terms(s, b, c, columns, o, column, bias);
    dense_four<T, I>(sum, b.row(s.row_sums[r]), column, bias, __fmul_rn(s.grids->in.scale, s.grids->kernel.scale), r, c, columns,
                     whole_fours<T>(c, columns, o), o);
}

// Turned sums: 64 rows by 64 columns through LDS.
template <typename T, typename I>
__global__ void __launch_bounds__(256) dense_out_turned_kernel(TableSums s, int64_t rows, int columns, DenseOut o)
{
    __shared__ int32_t tile[64][65];
    const int quad = (threadIdx.x & 15) * 4, line = threadIdx.x / 16;
    const int c0 = (int)blockIdx.x * 64;
    const int64_t r0 = (int64_t)blockIdx.y * 64;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = c0 + line + 16 * i;
        if (c < columns && r0 + quad < rows) {
            const i32x4 t = four_sums(s.raw, r0 + quad, c);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                tile[quad + j][line + 16 * i] = t[j];
        }
    }
    __syncthreads();
    const int c = c0 + quad;
    if (c >= columns)
        return;
    const float scale = __fmul_rn(s.grids->in.scale, s.grids->kernel.scale);
    const Bracket<I> b(s);
    const bool whole = whole_fours<T>(c, columns, o);
    I column[4];
    float bias[4];
    column_terms(s, b, c, columns, o, column, bias);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = line + 16 * i;
        if (r0 + at < rows) {
            const int32_t sum[4] = {tile[at][quad], tile[at][quad + 1], tile[at][quad + 2], tile[at][quad + 3]};
            dense_four<T, I>(sum, b.row(s.row_sums[r0 + at]), column, bias, scale, r0 + at, c, columns, whole, o);
        }
    }
}

__global__ void __launch_bounds__(256) zero_kernel(uint16_t *p, int64_t n)   // halfwords: what elements are multiples of
{
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        p[i] = 0;
}

} // namespace

hipError_t launch_zero(void *p, int64_t bytes, hipStream_t stream)
{
    const int64_t n = bytes / 2, blocks = (n + 255) / 256;
    if (n > 0)
        hipLaunchKernelGGL(zero_kernel, dim3((unsigned)(blocks > 4096 ? 4096 : blocks)), dim3(256), 0, stream,
                           static_cast<uint16_t *>(p), n);
    return hipGetLastError();
}

hipError_t launch_range(const void *x, int x_type, int64_t nx, const void *kernel, int kernel_type, int64_t nk, float *x_pairs,
                        float *kernel_pairs, int32_t *zeros, int64_t n_zeros, int *x_count, int *kernel_count, hipStream_t stream)
{
    auto blocks = [](int64_t n) {   // 16 values a thread and more
        const int64_t b = (n + 16383) / 16384;
        return (int)(b > kRangeBlocks ? kRangeBlocks : b);
    };
    const int bx = x ? blocks(nx) : 0, bk = kernel ? blocks(nk) : 0;
    *x_count = bx;
    *kernel_count = bk;
    const int total = bx + bk;
    if (total == 0)
        return hipSuccess;
    hipLaunchKernelGGL(range_kernel, dim3(total), dim3(1024), 0, stream, x, x_type, nx, bx, kernel, kernel_type, nk, x_pairs,
                       kernel_pairs, zeros, n_zeros);
    return hipGetLastError();
}

hipError_t launch_grids(const RangeSource &in, const RangeSource &kernel, bool has_in, bool has_kernel, Grids *grids,
                        hipStream_t stream)
{
    hipLaunchKernelGGL(grids_kernel, dim3(1), dim3(256), 0, stream, in, kernel, (int)has_in, (int)has_kernel, grids);
    return hipGetLastError();
}

hipError_t launch_few_codes(const void *x, int type, int rows, int K, int Kp, const RangeSource &src, const Grid *kernel_grid,
                            Grids *grids, uint8_t *codes, int32_t *row_sums, hipStream_t stream)
{
    hipLaunchKernelGGL(few_codes_kernel, dim3(rows), dim3(512), 0, stream, x, type, rows, K, Kp, src, kernel_grid, grids, codes,
                       row_sums);
    return hipGetLastError();
}

hipError_t launch_codes(const CodesJob &job, hipStream_t stream)
{
    const int x_blocks = job.x ? (int)((job.rows + 3) / 4) : 0;
    const int column_blocks = job.kernel ? (int)((job.pieces.Np + 255) / 256) : 1;
    // a wavefront 16 lines of the depth, fewer where that would leave CUs without work
    int lines = 16;
    auto slabs = [&] { return (job.pieces.Kp + 4 * lines - 1) / (4 * lines); };
    while (lines > 4 && (int64_t)slabs() * column_blocks < 1024)
        lines /= 2;
    const int64_t kernel_blocks = job.kernel ? (int64_t)slabs() * column_blocks : 0;
    hipLaunchKernelGGL(codes_kernel, dim3((unsigned)(x_blocks + kernel_blocks)), dim3(256), 0, stream, job, x_blocks, column_blocks,
                       lines);
    return hipGetLastError();
}

// A workgroup a CU, but at least two steps of the depth each.
int few_rows_splits(int64_t rows, int K, int width)
{
    const int64_t groups = (rows + kFewRows - 1) / kFewRows * ((width + kFewColumns - 1) / kFewColumns);
    const int64_t want = device_cus() / groups, most = (K + 3) / 4 * 2 / (2 * kFewGroups);
    const int64_t s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s);
}

template <int MT>
static hipError_t few_rows(const uint16_t *tableI, const uint8_t *x_codes, int rows, int Kp, const uint8_t *kernel_codes, int width,
                           int splits, int32_t *acc, hipStream_t stream)
{
    constexpr int bytes = few_lds_bytes<MT>();
    if (hipError_t e = set_max_dynamic_lds_once(reinterpret_cast<const void *>(&few_rows_kernel<MT>), bytes))
        return e;
    hipLaunchKernelGGL(few_rows_kernel<MT>,
                       dim3((unsigned)((width + kFewColumns - 1) / kFewColumns), (unsigned)splits, (unsigned)((rows + MT - 1) / MT)),
                       dim3(1024), bytes, stream, tableI, x_codes, rows, Kp, kernel_codes, width, acc);
    return hipGetLastError();
}

hipError_t launch_few_rows(const uint16_t *tableI, const uint8_t *x_codes, int rows, int Kp, const uint8_t *kernel_codes, int width,
                           int splits, int32_t *acc, hipStream_t stream)
{
    if (rows == 1)
        return few_rows<1>(tableI, x_codes, rows, Kp, kernel_codes, width, splits, acc, stream);
    if (rows == 2)
        return few_rows<2>(tableI, x_codes, rows, Kp, kernel_codes, width, splits, acc, stream);
    if (rows <= 4)
        return few_rows<4>(tableI, x_codes, rows, Kp, kernel_codes, width, splits, acc, stream);
    return few_rows<8>(tableI, x_codes, rows, Kp, kernel_codes, width, splits, acc, stream);
}

template <typename T, typename I>
static hipError_t dense_out(const TableSums &s, int64_t rows, int columns, const DenseOut &o, hipStream_t stream)
{
    if (s.raw.turned) {
        hipLaunchKernelGGL((dense_out_turned_kernel<T, I>), dim3((unsigned)((columns + 63) / 64), (unsigned)((rows + 63) / 64)),
                           dim3(256), 0, stream, s, rows, columns, o);
    } else if (s.raw.splits >= 8 && rows <= 64) {
        hipLaunchKernelGGL((dense_out_parts_kernel<T, I>), dim3((unsigned)((columns + 255) / 256), (unsigned)rows), dim3(256), 0,
                           stream, s, columns, o);
    } else {
        // several rows a wavefront, so that what belongs to the columns is loaded once for them
        const int64_t bx = (columns + 255) / 256, most = (4096 + bx - 1) / bx, by = (rows + 3) / 4;
        hipLaunchKernelGGL((dense_out_kernel<T, I>), dim3((unsigned)bx, (unsigned)(by > most ? most : by)), dim3(256), 0, stream, s,
                           rows, columns, o);
    }
    return hipGetLastError();
}
template <typename T>
static hipError_t dense_out(const TableSums &s, int64_t rows, int columns, const DenseOut &o, hipStream_t stream)
{
    return s.K > kNarrowDepth ? dense_out<T, int64_t>(s, rows, columns, o, stream)
                              : dense_out<T, uint32_t>(s, rows, columns, o, stream);
}

hipError_t launch_dense_out(const TableSums &s, int64_t rows, int columns, const DenseOut &o, hipStream_t stream)
{
    if (o.type == AXC_F32)
        return dense_out<float>(s, rows, columns, o, stream);
    if (o.type == AXC_BF16)
        return dense_out<bf16>(s, rows, columns, o, stream);
    return dense_out<f16>(s, rows, columns, o, stream);
}

} // namespace axc
