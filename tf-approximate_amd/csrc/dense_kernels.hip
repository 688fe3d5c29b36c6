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

// Few rows, in groups of eight: every workgroup finds the range itself, of all rows, and then takes its own row
// (of rows that are not there the codes are what the memory held: any byte is one, and nobody stores what comes of them).
template <typename T>
__device__ int32_t column_codes(const T *__restrict__ x, int K, int Kb, const Grid &g, uint8_t *__restrict__ codes)
{
    int32_t sum = 0;
#pragma unroll 4
    for (int k = threadIdx.x; k < Kb; k += 512) {
        const uint32_t c = k < K ? code_of((float)x[k], g) : 0u;
        codes[(int64_t)k * 8] = (uint8_t)c;
        sum += (int32_t)c;
    }
    return sum;
}
__global__ void __launch_bounds__(512) few_codes_kernel(const void *x, int type, int rows, int K, int Kb, RangeSource src,
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
    uint8_t *const to = codes + (r & ~7) * Kb + (r & 7);
    int32_t part = 0;
    if (type == AXC_F32)
        part = column_codes(static_cast<const float *>(x) + r * K, K, Kb, g, to);
    else if (type == AXC_BF16)
        part = column_codes(static_cast<const bf16 *>(x) + r * K, K, Kb, g, to);
    else
        part = column_codes(static_cast<const f16 *>(x) + r * K, K, Kb, g, to);
    part = wave_sum(part);
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
            if (kernel_grid)
                grids->kernel = *kernel_grid;
        }
    }
}

constexpr int kSlab = 64;   // most of the depth that a workgroup of codes_kernel takes

// tile: not null: the codes go there too, [element of the slab][column of the workgroup].
template <typename T>
__device__ void kernel_slab(const T *__restrict__ w, int K, int64_t N, const Pieces &pc, const Grid &g, uint8_t *__restrict__ codes,
                            uint32_t (*tile)[64], int64_t c, int first, int wave, int lines, int (&sum)[4])
{
    const int piece = (int)(c / pc.width);
    uint8_t *const to = codes + pc.offset(piece) + (c - pc.first(piece));
    const int pitch = pc.width_of(piece);
    const bool whole = c + 4 <= N && (N & 3) == 0 && ((uintptr_t)w & (4 * sizeof(T) - 1)) == 0;
#pragma unroll 4
    for (int i = 0; i < lines; ++i) {
        const int k = first + wave + 4 * i;
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
        if (codes && k < pc.Kp)
            *reinterpret_cast<uint32_t *>(to + (size_t)k * pitch) = word;
        if (tile)
            tile[wave + 4 * i][threadIdx.x & 63] = word;
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
    __shared__ uint32_t tile[kSlab][64];
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
    const int k0 = slab * 4 * lines;
    uint32_t(*const turn)[64] = job.kernel_blocks ? tile : nullptr;
    if (c < job.pieces.Np) {
        if (job.kernel_type == AXC_F32)
            kernel_slab(static_cast<const float *>(job.kernel), job.K, job.N, job.pieces, g, job.kernel_codes, turn, c, k0, wave,
                        lines, sum);
        else if (job.kernel_type == AXC_BF16)
            kernel_slab(static_cast<const bf16 *>(job.kernel), job.K, job.N, job.pieces, g, job.kernel_codes, turn, c, k0, wave,
                        lines, sum);
        else
            kernel_slab(static_cast<const f16 *>(job.kernel), job.K, job.N, job.pieces, g, job.kernel_codes, turn, c, k0, wave, lines,
                        sum);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        red[wave][4 * lane + j] = sum[j];
    __syncthreads();
    const int64_t column = first + threadIdx.x;
    if (column < job.pieces.Np)
        atomicAdd(job.column_sums + column,
                  red[0][threadIdx.x] + red[1][threadIdx.x] + red[2][threadIdx.x] + red[3][threadIdx.x]);
    if (!turn || column >= job.pieces.Np)
        return;
    // a column a thread: its codes of a block, begun at element n & 15
    const int piece = (int)(column / job.pieces.width), n = (int)(column - job.pieces.first(piece));
    uint8_t *const to = job.kernel_blocks + job.pieces.block_offset(piece) + (size_t)n * 16;
    const size_t pitch = (size_t)job.pieces.width_of(piece) * 16;
    for (int block_k = 0; block_k < 4 * lines && k0 + block_k < job.pieces.Kb; block_k += 16) {
        uint32_t word[4] = {};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t four = tile[block_k + ((n + i) & 15)][threadIdx.x / 4];
            word[i / 4] |= (four >> (8 * (threadIdx.x & 3)) & 255u) << (8 * (i & 3));
        }
        *reinterpret_cast<uint4 *>(to + (size_t)(k0 + block_k) / 16 * pitch) = make_uint4(word[0], word[1], word[2], word[3]);
    }
}

// ---- sums of few rows ----
// A workgroup takes MT rows, 1024 columns (one a lane) and 16 elements of the depth at a time.  For those elements it lays out in LDS
//   R[b][e] = entries of filter code b for all MT rows, at element e of the block: 16 places of 16 bytes, a row of 256 bytes,
// and every lane looks its column's 16 weights up in it, 2 MT bytes an access.  Which row that is, is anybody's guess, but the place
// in it decides the banks: at step s lane l takes element (l + s) & 15, so that any 16 lanes meet 16 different groups of banks,
// whatever their weights are (as all elements go into the same sum, their order does not matter; the codes are laid out in it).
// Building R takes 8 to 64 KiB of table rows for the block and 1024 columns, through a first-level cache that takes an address for
// every 64 neighbouring bytes a cycle: four neighbouring lanes read on in one table row, of one element, and the next four in
// another's (a different row for each lane, whose stores would meet no bank twice, took 64 addresses a load: 23.5 us instead of
// 15.8 for 8 rows by 4096 by 4096).  Sums of two rows share a dword as they come: one register adds whole dwords modulo 2^32, another the
// upper halves, three instructions for two dwords.
// RAW: the input comes as it is.  Every workgroup finds its range and its grid itself and makes the codes of its own part of the
// depth, into LDS; one of them the rows' sums and the grids for the launch behind this one.
constexpr int kFewColumns = 1024;
constexpr int kFewBlocks = 192;          // of the depth, a workgroup at most where it makes codes: 128 bytes of LDS each
constexpr int kFewLdsBytes = 2 * 65536;  // R twice: one is built while the other is read

template <int MT, bool RAW>
__global__ void __launch_bounds__(1024) few_rows_kernel(const uint16_t *__restrict__ tableI, const uint8_t *__restrict__ x_codes,
                                                        FewInput in, int rows, int Kb, const uint8_t *__restrict__ kernel_blocks,
                                                        int width, int32_t *__restrict__ acc)
{
    constexpr int H = (MT + 1) / 2;      // dwords of a place that are used
    constexpr int kOf = MT < 4 ? MT : 4; // rows that a wavefront takes table entries of
    constexpr int kEntries = MT == 8 ? 8 : 4;   // of neighbouring filter codes that a lane takes: eight rows are two wavefronts' work
    typedef uint32_t Words __attribute__((ext_vector_type(kEntries / 2)));
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const int c = (int)blockIdx.x * kFewColumns + (int)threadIdx.x;
    const int at = c < width ? c : width - 1;   // (lanes behind the columns repeat the last, at its place; nobody stores them)
    const int row0 = (int)blockIdx.z * 8;
    const int blocks = Kb / 16;
    const int first = (int)((int64_t)blocks * blockIdx.y / gridDim.y), last = (int)((int64_t)blocks * (blockIdx.y + 1) / gridDim.y);
    // this lane's part of R: filter codes b0 on, at element lane >> 2, rows `half` on
    const int half = MT == 8 ? (wave & 1) * 4 : 0;
    const int b0 = (MT == 8 ? (wave >> 1) * 32 : wave * 16) + (lane & 3) * kEntries;
    const uint8_t *const xs = x_codes + (int64_t)row0 * Kb + (lane >> 2) * 8 + half;

    uint32_t a;                          // the rows' codes at that element
    Words t[kOf];                        // table entries
    uint4 w;                             // the column's 16 weights
    unsigned char *const own_codes = lds + kFewLdsBytes;   // RAW: [element of this part][8 rows]
    auto load_codes = [&](int block) {
        if constexpr (RAW)
            a = *reinterpret_cast<const uint32_t *>(own_codes + (block - first) * 128 + (lane >> 2) * 8 + half);
        else
            a = *reinterpret_cast<const uint32_t *>(xs + (int64_t)block * 128);
    };
    auto load_entries = [&] {
#pragma unroll
        for (int m = 0; m < kOf; ++m)
            t[m] = *reinterpret_cast<const Words *>(tableI + ((a >> (8 * m)) & 255u) * 256u + b0);
    };
    auto load_weights = [&](int block) {
        w = *reinterpret_cast<const uint4 *>(kernel_blocks + ((int64_t)block * width + at) * 16);
    };
    uint32_t chunk[4];                   // where step 4 i + j reads in a row, in bytes: byte j of chunk[i]
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        chunk[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            chunk[i] |= (uint32_t)(((at + 4 * i + j) & 15) * 16) << (8 * j);
    }

    if (first < last)
        load_weights(first);
    if constexpr (RAW) {
        __shared__ float ends[32];
        __shared__ int32_t part[16][8];
        float lo, hi;
        if (!in.range.pairs && in.range.count < 0) {
            lo = INFINITY;
            hi = -INFINITY;
            range_of_any(in.x, in.type, (int64_t)rows * in.K, threadIdx.x, 1024, lo, hi);
            block_range(lo, hi, ends);
        } else {
            fold(in.range, lo, hi, ends);
        }
        const Grid g = grid_of_range(lo, hi);
        const int here = rows - row0 < 8 ? rows - row0 : 8, k0 = first * 16, many = (last - first) * 16;
        for (int i = (int)threadIdx.x; i < many * 8; i += 1024) {
            const int m = i & 7, k = k0 + (i >> 3);
            own_codes[i] = (unsigned char)(m < here && k < in.K
                                               ? code_of(load_any(in.x, (int64_t)(row0 + m) * in.K + k, in.type), g)
                                               : 0u);
        }
        if (blockIdx.x == 0 && blockIdx.y == 0) {
            int32_t sums[MT] = {};
            for (int k = 4 * (int)threadIdx.x; k < in.K; k += 4096)
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    float v[4] = {};
                    load_four_any(in.x, (int64_t)(row0 + (m < here ? m : 0)) * in.K + k, in.K - k, in.type, v);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        sums[m] += k + j < in.K ? (int32_t)code_of(v[j], g) : 0;
                }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                sums[m] = wave_sum(sums[m]);
                if (lane == 0)
                    part[wave][m] = sums[m];
            }
            __syncthreads();
            if ((int)threadIdx.x < here) {
                int32_t sum = 0;
                for (int i = 0; i < 16; ++i)
                    sum += part[i][threadIdx.x];
                in.row_sums[row0 + threadIdx.x] = sum;
            }
            if (blockIdx.z == 0 && threadIdx.x == 0) {
                in.grids->in = g;
                in.grids->kernel = *in.kernel_grid;
            }
        }
        __syncthreads();
    }
    uint32_t even[H] = {}, odd[H] = {};
    if (first < last) {
        load_codes(first);
        load_entries();
        if (first + 1 < last)
            load_codes(first + 1);
    }
    for (int block = first; block < last; ++block) {
        unsigned char *const R = lds + ((block - first) & 1) * 65536;
#pragma unroll
        for (int i = 0; i < kEntries; ++i) {
            const uint32_t sel = i & 1 ? 0x07060302u : 0x05040100u;
            uint32_t e[2] = {};
#pragma unroll
            for (int h = 0; h < (kOf + 1) / 2; ++h)
                e[h] = __builtin_amdgcn_perm(MT == 1 ? 0u : t[(2 * h + 1) % kOf][i / 2], t[2 * h][i / 2], sel);
            unsigned char *const to = R + (b0 + i) * 256 + (lane >> 2) * 16 + half * 2;
            if constexpr (H == 1)
                *reinterpret_cast<uint32_t *>(to) = e[0];
            else
                *reinterpret_cast<uint2 *>(to) = make_uint2(e[0], e[1]);
        }
        const uint32_t weights[4] = {w.x, w.y, w.z, w.w};
        if (block + 1 < last) {
            load_entries();
            load_weights(block + 1);
            if (block + 2 < last)
                load_codes(block + 2);
        }
        __syncthreads();   // R is whole, and the other one is no longer read
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t e[4][H];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // byte 1: the weight, byte 0: the place
                const unsigned char *const from = R + __builtin_amdgcn_perm(weights[i], chunk[i], 0x0c0c0400u + 0x0101u * j);
                if constexpr (H == 1) {
                    e[j][0] = *reinterpret_cast<const uint32_t *>(from);
                } else if constexpr (H == 2) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(from);
                    e[j][0] = v.x;
                    e[j][1] = v.y;
                } else {
                    const uint4 v = *reinterpret_cast<const uint4 *>(from);
                    e[j][0] = v.x;
                    e[j][1] = v.y;
                    e[j][2] = v.z;
                    e[j][3] = v.w;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j += 2)
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    even[h] += e[j][h] + e[j + 1][h];
                    if constexpr (MT > 1)
                        odd[h] += (e[j][h] >> 16) + (e[j + 1][h] >> 16);
                }
        }
    }
    if (c >= width)
        return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
        if (row0 + m < rows)
            acc[((int64_t)blockIdx.y * rows + row0 + m) * width + c] =
                (int32_t)(m & 1 ? odd[m / 2] : even[m / 2] - (MT > 1 ? odd[m / 2] << 16 : 0u));
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

// Turned sums: 64 rows by CT columns through LDS.
template <typename T, typename I, int CT>
__global__ void __launch_bounds__(256) dense_out_turned_kernel(TableSums s, int64_t rows, int columns, DenseOut o)
{
    __shared__ int32_t tile[64][CT + 1];
    const int c0 = (int)blockIdx.x * CT;
    const int64_t r0 = (int64_t)blockIdx.y * 64;
    {
        const int quad = (threadIdx.x & 15) * 4, line = threadIdx.x / 16;
#pragma unroll
        for (int i = 0; i < CT / 16; ++i) {
            const int c = c0 + line + 16 * i;
            if (c < columns && r0 + quad < rows) {
                const i32x4 t = four_sums(s.raw, r0 + quad, c);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    tile[quad + j][line + 16 * i] = t[j];
            }
        }
    }
    __syncthreads();
    const int quad = (int)threadIdx.x % (CT / 4) * 4, line = (int)threadIdx.x / (CT / 4);
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
    for (int i = 0; i < CT / 16; ++i) {
        const int at = line + 1024 / CT * i;
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

hipError_t launch_few_codes(const void *x, int type, int rows, int K, int Kb, const RangeSource &src, const Grid *kernel_grid,
                            Grids *grids, uint8_t *codes, int32_t *row_sums, hipStream_t stream)
{
    hipLaunchKernelGGL(few_codes_kernel, dim3(rows), dim3(512), 0, stream, x, type, rows, K, Kb, src, kernel_grid, grids, codes,
                       row_sums);
    return hipGetLastError();
}

hipError_t launch_codes(const CodesJob &job, hipStream_t stream)
{
    const int x_blocks = job.x ? (int)((job.rows + 3) / 4) : 0;
    const int column_blocks = job.kernel ? (int)((job.pieces.Np + 255) / 256) : 1;
    // a wavefront 16 lines of the depth, fewer where that would leave CUs without work
    int lines = kSlab / 4;
    const int depth = job.kernel_blocks ? job.pieces.Kb : job.pieces.Kp;
    auto slabs = [&] { return (depth + 4 * lines - 1) / (4 * lines); };
    while (lines > 4 && (int64_t)slabs() * column_blocks < 1024)
        lines /= 2;
    const int64_t kernel_blocks = job.kernel ? (int64_t)slabs() * column_blocks : 0;
    hipLaunchKernelGGL(codes_kernel, dim3((unsigned)(x_blocks + kernel_blocks)), dim3(256), 0, stream, job, x_blocks, column_blocks,
                       lines);
    return hipGetLastError();
}

// A workgroup a CU, but at least two blocks of the depth each, and at most kFewBlocks.
int few_rows_splits(int64_t rows, int Kb, int width)
{
    const int64_t groups = (rows + 7) / 8 * ((width + kFewColumns - 1) / kFewColumns);
    const int64_t want = device_cus() / groups, most = Kb / 32, least = (Kb / 16 + kFewBlocks - 1) / kFewBlocks;
    const int64_t s = want < most ? want : most;
    return (int)(s < least ? least : s);
}

template <int MT, bool RAW>
static hipError_t few_rows(const uint16_t *tableI, const uint8_t *x_codes, const FewInput &in, int rows, int Kb,
                           const uint8_t *kernel_blocks, int width, int splits, int32_t *acc, hipStream_t stream)
{
    const int bytes = kFewLdsBytes + (RAW ? kFewBlocks * 128 : 0);
    if (hipError_t e = set_max_dynamic_lds_once(reinterpret_cast<const void *>(&few_rows_kernel<MT, RAW>), bytes))
        return e;
    hipLaunchKernelGGL((few_rows_kernel<MT, RAW>),
                       dim3((unsigned)((width + kFewColumns - 1) / kFewColumns), (unsigned)splits, (unsigned)((rows + 7) / 8)),
                       dim3(1024), bytes, stream, tableI, x_codes, in, rows, Kb, kernel_blocks, width, acc);
    return hipGetLastError();
}

hipError_t launch_few_rows(const uint16_t *tableI, const uint8_t *x_codes, const FewInput *raw, int rows, int Kb,
                           const uint8_t *kernel_blocks, int width, int splits, int32_t *acc, hipStream_t stream)
{
    const FewInput in = raw ? *raw : FewInput{};
#define AXC_FEW(MT)                                                                                                         \
    return raw ? few_rows<MT, true>(tableI, x_codes, in, rows, Kb, kernel_blocks, width, splits, acc, stream)              \
               : few_rows<MT, false>(tableI, x_codes, in, rows, Kb, kernel_blocks, width, splits, acc, stream)
    if (rows == 1)
        AXC_FEW(1);
    if (rows == 2)
        AXC_FEW(2);
    if (rows <= 4)
        AXC_FEW(4);
    AXC_FEW(8);
#undef AXC_FEW
}

template <typename T, typename I>
static hipError_t dense_out(const TableSums &s, int64_t rows, int columns, const DenseOut &o, hipStream_t stream)
{
    if (s.raw.turned) {
        // tiles of fewer columns where those of 64 would leave CUs without work
        const unsigned by = (unsigned)((rows + 63) / 64);
        if ((int64_t)by * ((columns + 63) / 64) >= 1024)
            hipLaunchKernelGGL((dense_out_turned_kernel<T, I, 64>), dim3((unsigned)((columns + 63) / 64), by), dim3(256), 0, stream, s,
                               rows, columns, o);
        else
            hipLaunchKernelGGL((dense_out_turned_kernel<T, I, 16>), dim3((unsigned)((columns + 15) / 16), by), dim3(256), 0, stream, s,
                               rows, columns, o);
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
