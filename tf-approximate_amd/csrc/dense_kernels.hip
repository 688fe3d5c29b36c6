// Dense layers by table products: ranges, codes, the sums of few rows, and what is made of the sums.
//
//   product[m][n] = s_in s_k sum_k (T[a][b] - z_k a - z_in b + z_in z_k)
//                 = s_in s_k (sum_k T[a][b] - z_k sum_k a - z_in sum_k b + K z_in z_k)
//
// a, b: codes of the input and of the kernel, s, z: scale and zero point of their grids.  Everything in the brackets is a whole
// number and is computed as one, so a product is rounded three times: s_in s_k, the bracket, and the two multiplied.
//
// The sums of many rows are made by the kernels that make them for 1x1 convolutions (axc_conv2d_codes_acc_i32); those of few
// rows, where building rows for every filter element would cost more than the lookups, by few_rows_kernel; one row of up to
// 16 384 values, or two of up to 8192, are all token_kernel's.
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

// One pair per workgroup; the first x_blocks take the input (or one of them the pairs that a call before has reported of it: all that
// follows then reads one), the others the kernel.  All of them clear `zeros`, into which a later launch adds.
__global__ void __launch_bounds__(1024) range_kernel(const void *x, int x_type, int64_t nx, const float *reported, int x_blocks,
                                                     const void *kernel, int kernel_type, int64_t nk, float *x_pairs, float *kernel_pairs,
                                                     int32_t *zeros, int64_t n_zeros)
{
    __shared__ float red[32];
    const bool second = (int)blockIdx.x >= x_blocks;
    const int block = second ? (int)blockIdx.x - x_blocks : (int)blockIdx.x;
    const int blocks = second ? (int)gridDim.x - x_blocks : x_blocks;
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < n_zeros; i += (int64_t)gridDim.x * 1024)
        zeros[i] = 0;
    float lo = INFINITY, hi = -INFINITY;
    if (!second && reported) {
        fold({reported, kRangePairs, 0.0f, 0.0f}, lo, hi, red);
    } else {
        range_of_any(second ? kernel : x, second ? kernel_type : x_type, second ? nk : nx, (int64_t)block * 1024 + threadIdx.x,
                     (int64_t)blocks * 1024, lo, hi);
        block_range(lo, hi, red);
    }
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

// The grid of an input of few rows, found by one workgroup.  red: 2 * wavefronts floats of LDS.
__device__ __forceinline__ Grid few_grid(const FewInput &in, int rows, float *red)
{
    float lo, hi;
    if (!in.range.pairs && in.range.count < 0) {
        lo = INFINITY;
        hi = -INFINITY;
        range_of_any(in.x, in.type, (int64_t)rows * in.K, threadIdx.x, blockDim.x, lo, hi);
        block_range(lo, hi, red);
    } else {
        fold(in.range, lo, hi, red);
    }
    return grid_of_range(lo, hi);
}
// Few rows, in groups of eight: every workgroup finds the range itself, of all rows, and then takes its own row
// (of rows that are not there the codes are what the memory held: any byte is one, and nobody stores what comes of them).
__global__ void __launch_bounds__(512) few_codes_kernel(FewInput in, int rows, int Kb, Grids *grids, uint8_t *codes, int32_t *row_sums)
{
    __shared__ float red[16];
    __shared__ int32_t sums[8];
    const Grid g = few_grid(in, rows, red);
    const int64_t r = blockIdx.x;
    uint8_t *const to = codes + (r & ~7) * Kb + (r & 7);
    int32_t part = 0;
    for (int k = 4 * (int)threadIdx.x; k < Kb; k += 2048) {
        float v[4];
        load_four_any(in.x, r * in.K + k, in.K - k, in.type, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t c = k + j < in.K ? code_of(v[j], g) : 0u;
            to[(int64_t)(k + j) * 8] = (uint8_t)c;
            part += (int32_t)c;
        }
    }
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
            if (in.kernel_grid)
                grids->kernel = *in.kernel_grid;
        }
    }
}

constexpr int kSlab = 64;   // most of the depth that a workgroup of codes_kernel takes
constexpr int64_t kCodesBlocks = 1 << 20;   // workgroups for the input's rows, at most

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

// The first x_blocks workgroups take four rows of the input at a time, a wavefront a row (rows up to the next multiple of four are pad
// rows, of code 0).  The others take 256 columns of the kernel, four a lane, by 4 * lines of the depth, a wavefront every fourth;
// column sums are added to what the launch before cleared, as whole numbers, so in any order.  Every workgroup makes the grid it
// needs out of the range's pairs itself: a launch for that alone would be longer than folding 256 of them (or 4096, of a range that a
// call before has reported, against a packed kernel).
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
        const int Kp = job.pieces.Kp;
        const int64_t padded = (job.rows + 3) / 4 * 4;
        for (int64_t r = (int64_t)blockIdx.x * 4 + wave; r < padded; r += (int64_t)x_blocks * 4) {
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
        }
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
// A workgroup takes eight rows, 1024 columns and 16 elements of the depth at a time.  For those elements it lays out in LDS
//   R[b][e] = entries of filter code b for all eight rows, at element e of the block: 16 places of 16 bytes, a row of 256 bytes,
// and looks the columns' weights up in it, 16 bytes an access.  Which row that is, is anybody's guess, but the place in it decides the
// banks: a lane of column n takes the elements from n on, so that any 16 lanes meet 16 different groups of banks, whatever their
// weights are (as all elements go into the same sum, their order does not matter; the codes are laid out in it).
// The matrix cores add up what is found: a lane's 16 bytes are its column's line of the left operand, four lanes' blocks of the depth
// of 64, and the right operand, a one where byte and result agree, adds the bytes up one by one.  They are signed bytes there, so the
// table is the one whose bytes have their top bit flipped, 128 less each.  (The vector ALU would take three instructions
// for two dwords, six a lookup.)
// Building R takes 64 KiB of table rows for the block and 1024 columns, through a first-level cache that takes an address for
// every 64 neighbouring bytes a cycle: four neighbouring lanes read on in one table row, of one element, and the next four in
// another's (a different row for each lane, whose stores would meet no bank twice, took 64 addresses a load, and half as long again).
// So four lanes store to one place of four rows of R, which are the same banks: they store dwords, odd lanes the other of their two
// first (8 cycles a store; both at once took 24, twice as long as all reads together; with as many dwords as there are lanes, of loads
// half as wide, the stores took 2 and the loads more than they saved).
// MT: 4 where there are no more rows, 8 bytes a place then.  8 rows by 4096 by 4096, four blocks a workgroup, take 17 us: 5 until the
// first R is there (range, codes, table rows, one after the other), then 2 a block, 1.5 of them the LDS's accesses; 4 rows 15.
// RAW: the input comes as it is.  Every workgroup finds its range and its grid itself and makes the codes of its own part of the
// depth, into LDS, and their sums.
constexpr int kFewColumns = 1024;
constexpr int kFewBlocks = 192;          // of the depth, a workgroup at most where it makes codes: 128 bytes of LDS each
constexpr int kFewLdsBytes = 2 * 65536;  // R twice: one is built while the other is read

template <int MT, bool RAW>
__global__ void __launch_bounds__(1024) few_rows_kernel(FewJob job)
{
    constexpr int kEntries = MT;
    typedef uint32_t Words __attribute__((ext_vector_type(kEntries / 2)));
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int n = lane & 15, quarter = lane >> 4, width = job.width, Kb = job.Kb;
    const int column0 = (int)blockIdx.x * kFewColumns + wave * 64;
    const int row0 = (int)blockIdx.z * 8;
    const int blocks = Kb / 16;
    const int first = (int)((int64_t)blocks * blockIdx.y / gridDim.y), last = (int)((int64_t)blocks * (blockIdx.y + 1) / gridDim.y);
    // this lane's part of R: kEntries filter codes, b0 on, at element lane >> 2, four rows, `half` on
    const int half = MT == 8 ? (wave & 1) * 4 : 0;
    const int b0 = (MT == 8 ? (wave >> 1) * 32 : wave * 16) + (lane & 3) * kEntries;
    const int own_place = b0 * 256 + (lane >> 2) * 16 + half * 2, odd = (lane & 1) * 4;
    const uint8_t *const xs = job.x_codes + (int64_t)row0 * Kb + (lane >> 2) * 8 + half;

    uint32_t a;                          // the rows' codes at that element
    Words t[4];                          // table entries
    uint32_t w[4];                       // four weights of a column in each of four groups of 16
    unsigned char *const own_codes = lds + kFewLdsBytes;   // RAW: [element of this part][8 rows]
    auto load_codes = [&](int block) {
        if constexpr (RAW)
            a = *reinterpret_cast<const uint32_t *>(own_codes + (block - first) * 128 + (lane >> 2) * 8 + half);
        else
            a = *reinterpret_cast<const uint32_t *>(xs + (int64_t)block * 128);
    };
    auto load_entries = [&] {
#pragma unroll
        for (int m = 0; m < 4; ++m)
            t[m] = *reinterpret_cast<const Words *>(job.tableS + ((a >> (8 * m)) & 255u) * 256u + b0);
    };
    const uint8_t *from[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {        // (lanes behind the columns repeat the last; nobody stores them)
        const int c = column0 + q * 16 + n;
        from[q] = job.kernel_blocks + (int64_t)(c < width ? c : width - 1) * 16 + quarter * 4;
    }
    auto load_weights = [&](int block) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            w[q] = *reinterpret_cast<const uint32_t *>(from[q] + (int64_t)block * width * 16);
    };
    uint32_t places = 0;                 // of this lane's four elements, in bytes
#pragma unroll
    for (int i = 0; i < 4; ++i)
        places |= (uint32_t)(((n + 4 * quarter + i) & 15) * 16) << (8 * i);
    i32x4 one = {};                      // byte n of an element's 2 MT is 1
#pragma unroll
    for (int i = 0; i < 4; ++i)
        one[i] = n / 4 == i % (MT / 2) ? 1 << (8 * (n & 3)) : 0;

    if (first < last)
        load_weights(first);
    if constexpr (RAW) {
        __shared__ float ends[32];
        __shared__ int32_t part[8];
        if (threadIdx.x < 8)
            part[threadIdx.x] = 0;
        const int here = job.rows - row0 < 8 ? job.rows - row0 : 8, k0 = first * 16, many = (last - first) * 16;
        auto there = [&](int i) { return i < many * 8 && (i & 7) < here && k0 + (i >> 3) < job.in.K; };
        auto bits_at = [&](int i) {
            return there(i) ? load_bits(job.in.x, (int64_t)(row0 + (i & 7)) * job.in.K + k0 + (i >> 3), job.in.type) : 0u;
        };
        const uint32_t early = bits_at((int)threadIdx.x);   // (while the range is looked for)
        const Grid g = few_grid(job.in, job.rows, ends);
        __syncthreads();                 // (of a known range, nothing else waits for `part`)
        int32_t sum = 0;                 // of row threadIdx.x & 7
        for (int i = (int)threadIdx.x; i < many * 8; i += 1024) {
            const uint32_t bits = i < 1024 ? early : bits_at(i);
            const uint32_t c = there(i) ? code_of(value_of(bits, job.in.type), g) : 0u;
            own_codes[i] = (unsigned char)c;
            sum += (int32_t)c;
        }
        if (blockIdx.x == 0) {
            sum += __shfl_xor(sum, 8);
            sum += __shfl_xor(sum, 16);
            sum += __shfl_xor(sum, 32);
            if (lane < 8)
                atomicAdd(&part[lane], sum);   // whole numbers, in any order
        }
        if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
            job.grids->in = g;
            if (job.in.kernel_grid != &job.grids->kernel)
                job.grids->kernel = *job.in.kernel_grid;
        }
        __syncthreads();
        if (blockIdx.x == 0 && (int)threadIdx.x < here)
            job.acc[((int64_t)blockIdx.y * job.rows + row0 + threadIdx.x) * job.pitch + width] = part[threadIdx.x];
    }
    i32x4 sums[4] = {};
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
            const uint32_t e0 = __builtin_amdgcn_perm(t[1][i / 2], t[0][i / 2], sel);
            const uint32_t e1 = __builtin_amdgcn_perm(t[3][i / 2], t[2][i / 2], sel);
            unsigned char *const to = R + own_place + i * 256;
            *reinterpret_cast<uint32_t *>(to + odd) = odd ? e1 : e0;
            *reinterpret_cast<uint32_t *>(to + 4 - odd) = odd ? e0 : e1;
        }
        const uint32_t weights[4] = {w[0], w[1], w[2], w[3]};
        if (block + 1 < last) {
            load_entries();
            load_weights(block + 1);
            if (block + 2 < last)
                load_codes(block + 2);
        }
        __syncthreads();   // R is whole, and the other one is no longer read
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            // byte 1: the weight, byte 0: the place
            auto place = [&](int i) { return R + __builtin_amdgcn_perm(weights[q], places, 0x0c0c0400u + 0x0101u * i); };
            if constexpr (MT == 8) {
                i32x4 found[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    found[i] = *reinterpret_cast<const i32x4 *>(place(i));
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sums[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(found[i], one, sums[q], 0, 0, 0);
            } else {
                int2 found[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    found[i] = *reinterpret_cast<const int2 *>(place(i));
#pragma unroll
                for (int i = 0; i < 4; i += 2)
                    sums[q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(i32x4{found[i].x, found[i].y, found[i + 1].x, found[i + 1].y}, one,
                                                                    sums[q], 0, 0, 0);
            }
        }
    }
    // sums[q][r] is byte n of column 4 * quarter + r: rows n / 2, low and high byte in neighbouring lanes
    const int32_t flipped = (last - first) * 16 * (128 + 256 * 128);
    const bool high = n & 1;
    const int row = row0 + n / 2;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        i32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int32_t other = __builtin_amdgcn_update_dpp(0, sums[q][r], 0xb1, 0xf, 0xf, true);   // of lane ^ 1
            v[r] = (high ? other + 256 * sums[q][r] : sums[q][r] + 256 * other) + flipped;
        }
        const int c = column0 + q * 16 + quarter * 4;
        if ((q & 1) == (int)high && n < 2 * MT && row < job.rows && c < width)
            *reinterpret_cast<i32x4 *>(job.acc + ((int64_t)blockIdx.y * job.rows + row) * job.pitch + c) = v;
    }
}

// ---- one or two rows ----
// A workgroup holds the whole table in LDS and takes 16 columns, over all of the depth: nothing is left to be joined, and what is
// made of the sums is made here, in one launch.  A lane has one of the columns and every 64th block of 16 elements.
// A lookup is a read of two bytes from anywhere in LDS, 64 of which meet in the 64 banks as chance has it (about 10 a cycle and CU,
// a tenth of what few_rows_kernel finds once R is there), and chance is what is left to them: at step s the lane of column n takes
// element (n + s) & 15, so that lanes of one block have different input codes, and the table keeps T[a][b] at
//   [r(a)][b ^ r(a)], r(a) the bits of a turned round,
// so that neither codes around a mean, nor one input code throughout, make some banks busier than others.  Both bytes of such a place
// are pairs of bytes of the codes put together, two places at once.
// One row by 4096 by 4096 takes 11 us on its own, 4 until the input, the first weights and the table are there and 4.4 for the
// lookups; two rows 15, as many by few_rows_kernel and the launch behind it 18.  One row to 14336 columns: 25.
constexpr int kTokenTable = 131072;      // bytes of LDS
constexpr int kTokenCodes = 16384;       // of the input's codes
constexpr int kTokenColumns = 16;
constexpr int kTokenRows = 2;
constexpr int kTokenLds = kTokenTable + kTokenCodes + 2 * 16 * kTokenRows * kTokenColumns * 4 + 256;

__device__ __forceinline__ uint32_t twice_low(uint32_t pair)    // 2 * (pair & 0xffff) and 2 * (pair >> 16)
{
    uint32_t r;
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:WORD_0" : "=v"(r) : "s"(1), "v"(pair));
    return r;
}
__device__ __forceinline__ uint32_t twice_high(uint32_t pair)
{
    uint32_t r;
    asm("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:WORD_1" : "=v"(r) : "s"(1), "v"(pair));
    return r;
}

template <int MT>
__global__ void __launch_bounds__(1024) token_kernel(TokenJob job)
{
    constexpr int kDepth = kTokenCodes / MT, kRounds = kTokenCodes / 4096;   // four codes a thread and round
    extern __shared__ __align__(16) unsigned char lds[];
    unsigned char *const codes = lds + kTokenTable;                                // [row][kDepth]
    uint32_t *const red = reinterpret_cast<uint32_t *>(codes + kTokenCodes);       // [turn][wavefront][row][column]
    float *const ends = reinterpret_cast<float *>(red + 2 * 16 * MT * kTokenColumns);
    int32_t *const part = reinterpret_cast<int32_t *>(ends + 32);                  // [row][wavefront]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int n = lane & 15, own = wave * 4 + (lane >> 4);
    const int K = job.in.K, blocks = job.pieces.Kb / 16, steps = (blocks + 255) / 256;
    const int groups = (int)((job.columns + kTokenColumns - 1) / kTokenColumns);

    // the input first: it is waited for first
    float v[kRounds][4];
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
        const int at = (i * 1024 + (int)threadIdx.x) * 4, row = at / kDepth, k = at - row * kDepth;
        load_four_any(job.in.x, (int64_t)row * K + k, row < MT ? K - k : 0, job.in.type, v[i]);
    }
    auto load_weights = [&](int group, int step, uint4(&w)[4]) {
        const uint32_t c0 = (uint32_t)group * kTokenColumns;
        const int p = (int)(c0 / (uint32_t)job.pieces.width), width = job.pieces.width_of(p);
        int c = (int)(c0 - (uint32_t)job.pieces.first(p)) + n;
        c = c < width ? c : width - 1;   // (lanes behind the columns: nobody stores them)
        const uint8_t *const from = job.kernel_blocks + job.pieces.block_offset(p) + (size_t)c * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int block = step * 256 + i * 64 + own;
            w[i] = block < blocks ? *reinterpret_cast<const uint4 *>(from + (size_t)block * width * 16) : make_uint4(0, 0, 0, 0);
        }
    };
    int group = (int)blockIdx.x;
    uint4 w[4], next[4] = {};
    load_weights(group, 0, w);
#pragma unroll
    for (int i = 0; i < kTokenTable / 16384; ++i)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) uint32_t *)(reinterpret_cast<const unsigned char *>(job.tableL) +
                                                                 (i * 1024 + (int)threadIdx.x) * 16),
            (__attribute__((address_space(3))) uint32_t *)(lds + (i * 1024 + wave * 64) * 16), 16, 0, 0);
    float lo = INFINITY, hi = -INFINITY;
    if (!job.in.range.pairs && job.in.range.count < 0) {
#pragma unroll
        for (int i = 0; i < kRounds; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if ((i * 1024 + (int)threadIdx.x) * 4 % kDepth + j < K) {
                    lo = fminf(lo, v[i][j]);
                    hi = fmaxf(hi, v[i][j]);
                }
        block_range(lo, hi, ends);
    } else {
        fold(job.in.range, lo, hi, ends);
    }
    const Grid in_grid = grid_of_range(lo, hi), kernel_grid = *job.in.kernel_grid;
    int32_t row_part[MT] = {};
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
        const int at = (i * 1024 + (int)threadIdx.x) * 4, k = at % kDepth;
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t c = k + j < K ? code_of(v[i][j], in_grid) : 0u;
            word |= (__builtin_bitreverse32(c) >> 24) << (8 * j);
            row_part[i * 4096 / kDepth] += (int32_t)c;
        }
        *reinterpret_cast<uint32_t *>(codes + at) = word;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        row_part[m] = wave_sum(row_part[m]);
        if (lane == 0)
            part[m * 16 + wave] = row_part[m];
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // a barrier alone does not wait for loads into LDS
    __syncthreads();

    const uint32_t turned = (uint32_t)n & 3u;
    int order[4];                        // the dwords of a block's codes, this column's first one first
#pragma unroll
    for (int i = 0; i < 4; ++i)
        order[i] = (((n >> 2) + i) & 3) * 4;
    for (int turn = 0; group < groups; group += (int)gridDim.x, turn ^= 1) {
        // a thread a value at the end; what is read for it is read here
        const int64_t c = (int64_t)group * kTokenColumns + (threadIdx.x & 15);
        const int row = (int)threadIdx.x / 16;
        const bool mine = row < MT && c < job.columns;
        int32_t column_sum = 0;
        float bias = 0.0f, residual = 0.0f;
        if (mine) {
            column_sum = job.column_sums[c];
            bias = job.out.bias ? load_any(job.out.bias, c, job.out.bias_type) : 0.0f;
            residual = job.out.residual ? load_any(job.out.residual, row * job.out.ld + c, job.out.type) : 0.0f;
        }
        uint32_t sum[MT] = {};
        for (int s = 0; s < steps; ++s) {
            const bool end = s + 1 == steps;
            if (!end || group + (int)gridDim.x < groups)
                load_weights(end ? group + (int)gridDim.x : group, end ? 0 : s + 1, next);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int block = s * 256 + i * 64 + own;
                if (block >= blocks)
                    continue;
                const unsigned char *const x = codes + block * 16;
                const uint32_t weights[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    uint32_t d[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        d[q] = *reinterpret_cast<const uint32_t *>(x + m * kDepth + order[q]);
                    uint32_t found[16];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t a = __builtin_amdgcn_alignbyte(d[(q + 1) & 3], d[q], turned);
                        const uint32_t p = __builtin_amdgcn_perm(0u, a, 0x01010000u) ^ __builtin_amdgcn_perm(0u, weights[q], 0x0c010c00u);
                        const uint32_t t = __builtin_amdgcn_perm(0u, a, 0x03030202u) ^ __builtin_amdgcn_perm(0u, weights[q], 0x0c030c02u);
                        found[4 * q] = *reinterpret_cast<const uint16_t *>(lds + twice_low(p));
                        found[4 * q + 1] = *reinterpret_cast<const uint16_t *>(lds + twice_high(p));
                        found[4 * q + 2] = *reinterpret_cast<const uint16_t *>(lds + twice_low(t));
                        found[4 * q + 3] = *reinterpret_cast<const uint16_t *>(lds + twice_high(t));
                    }
#pragma unroll
                    for (int q = 0; q < 16; q += 2)
                        sum[m] += found[q] + found[q + 1];
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                w[i] = next[i];
        }
        // the four blocks of a wavefront; then, row by row, the wavefronts
        uint32_t stored = 0;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            sum[m] += (uint32_t)__shfl_xor((int)sum[m], 16);
            sum[m] += (uint32_t)__shfl_xor((int)sum[m], 32);
            stored = lane >> 4 == m ? sum[m] : stored;
        }
        uint32_t *const to = red + turn * 16 * MT * kTokenColumns;
        if (lane >> 4 < MT)
            to[wave * MT * kTokenColumns + lane] = stored;
        __syncthreads();
        if (!mine)
            continue;
        uint32_t all = 0;
        int32_t row_sum = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            all += to[i * MT * kTokenColumns + threadIdx.x];
            row_sum += part[row * 16 + i];
        }
        const int64_t zi = in_grid.zero, zk = kernel_grid.zero;
        const int64_t bracket = (int64_t)all + K * zi * zk - (int64_t)(job.pieces.Kb - K) * job.tableL[0] - zk * row_sum - zi * column_sum;
        float z = __fmul_rn((float)bracket, __fmul_rn(in_grid.scale, kernel_grid.scale));
        if (job.out.bias)
            z = __fadd_rn(z, bias);
        const int64_t at = row * job.out.ld + c;
        if (job.out.pre)
            store_any(job.out.pre, at, job.out.type, z);
        float y = activate(z, job.out.activation);
        if (job.out.residual)
            y = __fadd_rn(y, residual);
        store_any(job.out.out, at, job.out.type, y);
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
    int32_t row_sum = 0;
    if (s.row_sums) {
        row_sum = s.row_sums[r];
    } else {
        for (int i = lane; i < s.raw.splits; i += 64)
            row_sum += s.raw.acc[r * s.raw.pitch + s.sums_at + i * s.raw.split_stride];
        row_sum = wave_sum(row_sum);
    }
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
    dense_four<T, I>(sum, b.row(row_sum), column, bias, __fmul_rn(s.grids->in.scale, s.grids->kernel.scale), r, c, columns,
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

hipError_t launch_range(const void *x, int x_type, int64_t nx, const float *reported, const void *kernel, int kernel_type, int64_t nk,
                        float *x_pairs, float *kernel_pairs, int32_t *zeros, int64_t n_zeros, int *x_count, int *kernel_count,
                        hipStream_t stream)
{
    auto blocks = [](int64_t n) {   // 16 values a thread and more
        const int64_t b = (n + 16383) / 16384;
        return (int)(b > kRangeBlocks ? kRangeBlocks : b);
    };
    const int bx = x ? blocks(nx) : reported ? 1 : 0, bk = kernel ? blocks(nk) : 0;
    *x_count = bx;
    *kernel_count = bk;
    const int total = bx + bk;
    if (total == 0)
        return hipSuccess;
    hipLaunchKernelGGL(range_kernel, dim3(total), dim3(1024), 0, stream, x, x_type, nx, reported, bx, kernel, kernel_type, nk, x_pairs,
                       kernel_pairs, zeros, n_zeros);
    return hipGetLastError();
}

hipError_t launch_few_codes(const FewInput &in, int rows, int Kb, Grids *grids, uint8_t *codes, int32_t *row_sums, hipStream_t stream)
{
    hipLaunchKernelGGL(few_codes_kernel, dim3(rows), dim3(512), 0, stream, in, rows, Kb, grids, codes, row_sums);
    return hipGetLastError();
}

hipError_t launch_codes(const CodesJob &job, hipStream_t stream)
{
    // A launch has fewer than 2^32 threads, 2^24 of these workgroups; and where each reads a reported range, 32 KiB, four a CU go
    // over the rows (16 384 rows, 64 -> 64, packed: 34.4 us a call, 41.1 by one for every four rows).
    const int64_t most = job.x_range.count > kRangeBlocks ? 1024 : kCodesBlocks;
    const int x_blocks = job.x ? (int)((job.rows + 3) / 4 < most ? (job.rows + 3) / 4 : most) : 0;
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
static hipError_t few_rows(const FewJob &job, hipStream_t stream)
{
    const int bytes = kFewLdsBytes + (RAW ? kFewBlocks * 128 : 0);
    if (hipError_t e = set_max_dynamic_lds_once(reinterpret_cast<const void *>(&few_rows_kernel<MT, RAW>), bytes))
        return e;
    hipLaunchKernelGGL((few_rows_kernel<MT, RAW>),
                       dim3((unsigned)((job.width + kFewColumns - 1) / kFewColumns), (unsigned)job.splits, (unsigned)((job.rows + 7) / 8)),
                       dim3(1024), bytes, stream, job);
    return hipGetLastError();
}
hipError_t launch_few_rows(const FewJob &job, hipStream_t stream)
{
    if (job.rows <= 4)
        return job.in.x ? few_rows<4, true>(job, stream) : few_rows<4, false>(job, stream);
    return job.in.x ? few_rows<8, true>(job, stream) : few_rows<8, false>(job, stream);
}

bool token_fits(int64_t rows, int Kb)
{
    return rows <= kTokenRows && rows * Kb <= kTokenCodes;
}
template <int MT>
static hipError_t token(const TokenJob &job, hipStream_t stream)
{
    if (hipError_t e = set_max_dynamic_lds_once(reinterpret_cast<const void *>(&token_kernel<MT>), kTokenLds))
        return e;
    // a workgroup a CU, and as many columns in each
    const int64_t groups = (job.columns + kTokenColumns - 1) / kTokenColumns, each = (groups + device_cus() - 1) / device_cus();
    hipLaunchKernelGGL(token_kernel<MT>, dim3((unsigned)((groups + each - 1) / each)), dim3(1024), kTokenLds, stream, job);
    return hipGetLastError();
}
hipError_t launch_token(const TokenJob &job, hipStream_t stream)
{
    return job.rows == 1 ? token<1>(job, stream) : token<2>(job, stream);
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
    } else if (!s.row_sums || (s.raw.splits >= 8 && rows <= 64)) {
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
