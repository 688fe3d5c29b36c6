// Declarations shared by the translation units of the transformer layers: dense layers by table products, the loss over a
// vocabulary, residual norms.
#pragma once

#include "axconv_internal.h"

namespace axc {

// ---- element types ----
typedef __bf16 bf16;
typedef _Float16 f16;
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

__host__ __device__ inline int type_bytes(int type) { return type == AXC_F32 ? 4 : 2; }

// One value of a vector whose type is only known at run time (biases, weights of norms: few, and read through the caches).
__device__ __forceinline__ float load_any(const void *p, int64_t i, int type)
{
    if (type == AXC_F32)
        return static_cast<const float *>(p)[i];
    if (type == AXC_BF16)
        return (float)static_cast<const bf16 *>(p)[i];
    return (float)static_cast<const f16 *>(p)[i];
}
// The same in two steps: nothing waits for the first.
__device__ __forceinline__ uint32_t load_bits(const void *p, int64_t i, int type)
{
    return type == AXC_F32 ? static_cast<const uint32_t *>(p)[i] : static_cast<const uint16_t *>(p)[i];
}
__device__ __forceinline__ float value_of(uint32_t bits, int type)
{
    if (type == AXC_F32)
        return __builtin_bit_cast(float, bits);
    if (type == AXC_BF16)
        return __builtin_bit_cast(float, bits << 16);
    return (float)__builtin_bit_cast(f16, (uint16_t)bits);
}
__device__ __forceinline__ void store_any(void *p, int64_t i, int type, float v)
{
    if (type == AXC_F32)
        static_cast<float *>(p)[i] = v;
    else if (type == AXC_BF16)
        static_cast<bf16 *>(p)[i] = (bf16)v;
    else
        static_cast<f16 *>(p)[i] = (f16)v;
}

// V neighbouring values as floats: one access where `whole` says that all V are there and aligned, else value by value with
// `fill` in the place of those beyond n.
template <typename T, int V>
__device__ __forceinline__ void load_values(const T *p, int64_t n, bool whole, float fill, float (&v)[V])
{
    if constexpr (V > 1) {
        if (whole) {
            typedef T vector __attribute__((ext_vector_type(V)));
            const vector t = *reinterpret_cast<const vector *>(p);
#pragma unroll
            for (int i = 0; i < V; ++i)
                v[i] = (float)t[i];
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        v[i] = i < n ? (float)p[i] : fill;
}
template <typename T, int V>
__device__ __forceinline__ void store_values(T *p, int64_t n, bool whole, const float (&v)[V])
{
    if constexpr (V > 1) {
        if (whole) {
            typedef T vector __attribute__((ext_vector_type(V)));
            vector t;
#pragma unroll
            for (int i = 0; i < V; ++i)
                t[i] = (T)v[i];
            *reinterpret_cast<vector *>(p) = t;
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < n)
            p[i] = (T)v[i];
}

// Four neighbouring values of a tensor whose type is only known at run time, as many of them as there are (n).
__device__ __forceinline__ void load_four_any(const void *p, int64_t at, int64_t n, int type, float (&v)[4])
{
    if (type == AXC_F32) {
        const float *const q = static_cast<const float *>(p) + at;
        load_values<float, 4>(q, n, n >= 4 && ((uintptr_t)q & 15) == 0, 0.0f, v);
    } else if (type == AXC_BF16) {
        const bf16 *const q = static_cast<const bf16 *>(p) + at;
        load_values<bf16, 4>(q, n, n >= 4 && ((uintptr_t)q & 7) == 0, 0.0f, v);
    } else {
        const f16 *const q = static_cast<const f16 *>(p) + at;
        load_values<f16, 4>(q, n, n >= 4 && ((uintptr_t)q & 7) == 0, 0.0f, v);
    }
}
__device__ __forceinline__ void store_four_any(void *p, int64_t at, int64_t n, int type, const float (&v)[4])
{
    if (type == AXC_F32) {
        float *const q = static_cast<float *>(p) + at;
        store_values<float, 4>(q, n, n >= 4 && ((uintptr_t)q & 15) == 0, v);
    } else if (type == AXC_BF16) {
        bf16 *const q = static_cast<bf16 *>(p) + at;
        store_values<bf16, 4>(q, n, n >= 4 && ((uintptr_t)q & 7) == 0, v);
    } else {
        f16 *const q = static_cast<f16 *>(p) + at;
        store_values<f16, 4>(q, n, n >= 4 && ((uintptr_t)q & 7) == 0, v);
    }
}

// ---- the 8-bit grid of a tensor ----
// What fake quantization with a range gives (Nudge, tf2/src/approx_ops_types.h:29-49): value = scale * (code - zero).
struct Grid {
    float scale, inv_scale, low, high;   // low, high: the nudged range
    int32_t zero;                        // code of 0.0f
    int32_t pad[3];
};
struct Grids {                           // of a layer, in device memory
    Grid in, kernel;
};

// Every operation rounded on its own, as tensor_quant_device (prepass_kernels.hip) has it for the convolutions.
__device__ inline Grid grid_of_range(float mn, float mx)
{
    Grid g = {};
    if (mn == 0.0f && mx == 0.0f)
        return g;
    const float sc = __fdiv_rn(__fsub_rn(mx, mn), 255.0f);
    const float from_min = __fsub_rn(0.0f, __fdiv_rn(mn, sc));
    const int zp = from_min < 0.0f ? 0 : from_min > 255.0f ? 255 : from_min == from_min ? (int)roundf(from_min) : 0;
    g.scale = sc;
    g.inv_scale = __fdiv_rn(1.0f, sc);
    g.low = __fmul_rn(__fsub_rn(0.0f, (float)zp), sc);
    g.high = __fmul_rn(__fsub_rn(255.0f, (float)zp), sc);
    g.zero = zp;
    return g;
}
// The grid's code of a value: that of fake_quant_value followed by quantize_code, whose round trip through the grid's float
// changes no code (it is off by less than 2^-14 of a step).  NaN counts as the upper end, as there.
__device__ __forceinline__ uint32_t code_of(float v, const Grid &g)
{
    const float c = fmaxf(fminf(v, g.high), g.low);
    float t = floorf(__fadd_rn(__fmul_rn(__fsub_rn(c, g.low), g.inv_scale), 0.5f));
    t = t > 0.0f ? t : 0.0f;          // NaN (a grid of no width, or of no end) too
    return g.scale == 0.0f ? 0u : (uint32_t)(t < 255.0f ? t : 255.0f);
}
__device__ __forceinline__ bool inside(float v, const Grid &g) { return v >= g.low && v <= g.high; }

struct RangeSource {                     // where a tensor's smallest and largest value come from
    const float *pairs;                  // (smallest, largest) pairs, or null
    int count;                           // of the pairs; null and 0: lo and hi, known to the caller; null and -1: not known yet
    float lo, hi;
};

// ---- reductions ----
// Sum over a wavefront, in every lane: within rows of 16 lanes, then row to row, by the vector ALU's own lane moves, which take a
// few cycles each where a move through the LDS takes a hundred.
template <int CTRL, int ROWS>
__device__ __forceinline__ float add_moved(float v)
{
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ float row_of_lanes_sum(float v)   // in lane 15 of each row
{
    v = add_moved<0x111, 0xf>(v);   // from 1, 2, 4, 8 lanes before
    v = add_moved<0x112, 0xf>(v);
    v = add_moved<0x114, 0xf>(v);
    return add_moved<0x118, 0xf>(v);
}
__device__ __forceinline__ float wave_sum(float v)
{
    v = row_of_lanes_sum(v);
    v = add_moved<0x142, 0xa>(v);   // lane 15 to the next row, in rows 1 and 3
    v = add_moved<0x143, 0xc>(v);   // lane 31 to rows 2 and 3
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ int32_t wave_sum(int32_t v)
{
#pragma unroll
    for (int s = 32; s > 0; s >>= 1)
        v += __shfl_xor(v, s);
    return v;
}
// Smallest and largest, the same way: a lane that nothing moves to keeps its own.
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float v)
{
    const int i = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float wave_max(float v)
{
    v = fmaxf(v, moved<0x111, 0xf>(v));
    v = fmaxf(v, moved<0x112, 0xf>(v));
    v = fmaxf(v, moved<0x114, 0xf>(v));
    v = fmaxf(v, moved<0x118, 0xf>(v));
    v = fmaxf(v, moved<0x142, 0xa>(v));
    v = fmaxf(v, moved<0x143, 0xc>(v));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}
__device__ __forceinline__ float wave_min(float v) { return -wave_max(-v); }
// Smallest and largest over a workgroup, in every thread.  red: 2 * waves floats of LDS, free before and after.
__device__ __forceinline__ void block_range(float &lo, float &hi, float *red)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64, waves = blockDim.x / 64;
    lo = wave_min(lo);
    hi = wave_max(hi);
    if (lane == 0) {
        red[2 * wave] = lo;
        red[2 * wave + 1] = hi;
    }
    __syncthreads();
    const int of = lane < waves ? lane : 0;
    lo = wave_min(red[2 * of]);
    hi = wave_max(red[2 * of + 1]);
    __syncthreads();
}

// The range that a source stands for, in every thread.  red: 2 * waves floats of LDS, free before and after.
__device__ __forceinline__ void fold(const RangeSource &src, float &lo, float &hi, float *red)
{
    lo = src.lo;
    hi = src.hi;
    if (src.pairs) {
        lo = INFINITY;
        hi = -INFINITY;
#pragma unroll 4
        for (int i = threadIdx.x; i < src.count; i += blockDim.x) {
            const float2 p = reinterpret_cast<const float2 *>(src.pairs)[i];
            lo = fminf(lo, p.x);
            hi = fmaxf(hi, p.y);
        }
        block_range(lo, hi, red);
    }
}

// ---- activations ----
// Phi(z), the normal distribution, and its density phi(z).  Both tails come from one exponential, in the form of Abramowitz & Stegun,
// Handbook of Mathematical Functions, 7.1.26: erfc(x) = t P(t) exp(-x^2), t = 1 / (1 + p x), x >= 0.  Theirs, five coefficients, is off by
// 1.5e-7 of 1, but by 1e-2 of what is left of the tail at z = -8.  These eight are fitted to exp(x^2) erfc(x) / t by least squares, weights
// moved to where it is furthest off, up to x = 9.6, where exp(-x^2) ends: off by 1.1e-7 of the value itself, 4.9e-7 with their
// roundings; the exponential's argument adds 3 z^2 half steps.  The library's erff has two ranges, which a wavefront goes through both: an
// epilogue of 16.8 M values took 46 us with it and 64-bit whole numbers, more than its 100 MB.
__device__ __forceinline__ void normal(float z, float &cumulative, float &density)
{
    const float x = fabsf(z) * 0.70710678118654752f;
    const float e = __expf(-x * x);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.33f, x, 1.0f));
    float poly = fmaf(t, -0.13592872f, 0.46268788f);
    poly = fmaf(t, fmaf(t, poly, -0.355438352f), 0.412541091f);
    poly = fmaf(t, fmaf(t, poly, 0.0450109169f), 0.201923758f);
    poly = fmaf(t, fmaf(t, poly, 0.182837263f), 0.186366111f) * t;
    const float tail = 0.5f * poly * e;          // Phi(-|z|)
    cumulative = z > 0.0f ? 1.0f - tail : tail;
    density = 0.39894228040143268f * e;
}
__device__ __forceinline__ float gelu(float z)
{
    float c, d;
    normal(z, c, d);
    return z == -INFINITY ? -0.0f : z * c;
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }
__device__ __forceinline__ float activate(float z, int activation)
{
    switch (activation) {
    case AXC_ACT_RELU: return z > 0.0f ? z : z == z ? 0.0f : z;
    case AXC_ACT_GELU: return gelu(z);
    case AXC_ACT_GELU_TANH:   // 0.5 z (1 + tanh(u)) = z sigmoid(2u)
        return z == -INFINITY ? -0.0f : z * sigmoid(1.5957691216057308f * (z + 0.044715f * z * z * z));
    case AXC_ACT_SILU: return z == -INFINITY ? -0.0f : z * sigmoid(z);
    default: return z;
    }
}
// One look at which activation it is for four values.
__device__ __forceinline__ void activate_four(const float (&z)[4], float (&y)[4], int activation)
{
    switch (activation) {
#define AXC_FOUR(which)                  \
    case which:                          \
        _Pragma("unroll")                \
        for (int j = 0; j < 4; ++j)      \
            y[j] = activate(z[j], which); \
        break;
        AXC_FOUR(AXC_ACT_RELU)
        AXC_FOUR(AXC_ACT_GELU)
        AXC_FOUR(AXC_ACT_GELU_TANH)
        AXC_FOUR(AXC_ACT_SILU)
    default:
#pragma unroll
        for (int j = 0; j < 4; ++j)
            y[j] = z[j];
#undef AXC_FOUR
    }
}
__device__ __forceinline__ float activation_slope(float z, int activation)
{
    switch (activation) {
    case AXC_ACT_RELU: return z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    case AXC_ACT_GELU: {
        float c, d;
        normal(z, c, d);
        return fabsf(z) < 14.0f ? fmaf(z, d, c) : z > 0.0f ? 1.0f : z == z ? 0.0f : z;
    }
    case AXC_ACT_GELU_TANH: {
        if (fabsf(z) > 1e6f)
            return z > 0.0f ? 1.0f : 0.0f;
        const float s = sigmoid(1.5957691216057308f * (z + 0.044715f * z * z * z));
        return s + 2.0f * z * s * (1.0f - s) * 0.79788456080286536f * (1.0f + 0.134145f * z * z);
    }
    case AXC_ACT_SILU: {
        if (fabsf(z) > 1e6f)
            return z > 0.0f ? 1.0f : 0.0f;
        const float s = sigmoid(z);
        return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.0f;
    }
}

// ---- dense layers ----
// Operands as codes, padded: input [rows][Kp], Kp the depth in fours; kernel in pieces of columns, each [Kp][width], the columns
// in fours.  For few_rows_kernel the depth is padded to blocks of 16: input [groups of 8 rows][Kb][8]; kernel, in each piece,
// [block][width] of 16 codes, those of column n begun at element n & 15 of the block and gone on round it.
// Pad codes are 0: every pad element of the depth adds T[0][0] to a sum, which the epilogue takes away again.
struct Pieces {
    int64_t Np;            // columns, in fours
    int32_t Kp, Kb;
    int32_t width;         // of all pieces but the last
    int32_t count;
    __host__ __device__ int64_t first(int p) const { return (int64_t)p * width; }
    __host__ __device__ int width_of(int p) const { return p + 1 < count ? width : (int)(Np - (int64_t)(count - 1) * width); }
    __host__ __device__ size_t offset(int p) const { return (size_t)Kp * first(p); }   // of a piece's codes, in bytes
    __host__ __device__ size_t block_offset(int p) const { return (size_t)Kb * first(p); }
    size_t bytes() const { return (size_t)Kp * Np; }
    size_t block_bytes() const { return (size_t)Kb * Np; }
};

constexpr int kRangeBlocks = 256;        // pairs that the range pass leaves per tensor, at most

// Sums of table entries as a consumer finds them, of one piece and one run of rows.
struct TableSums {
    RawSums raw;                         // (every fourth row and column begins 16-byte aligned)
    const int32_t *row_sums;             // sums of the input's codes, of the run's first row on; null: a column behind the sums' last
    int sums_at;                         // (that column)
    const int32_t *column_sums;          // sums of the kernel's codes, of the piece's first column on
    const uint16_t *table;               // its first entry is T[0][0]
    const Grids *grids;
    int K, pad;                          // depth, and pad elements behind it
};

// A product in front of its scales, sum - z_k row_sums - z_in column_sums + K z_in z_k, without the pad elements: each of the K
// elements contributes between -65025 and 65535 + 65025.  Up to this depth it fits 32 bits, and so may be computed modulo 2^32
// whatever its parts are; in a longer one all of it is 64 bits wide.
constexpr int kNarrowDepth = 16384;      // 16384 * 130560 < 2^31
template <typename I>                    // uint32_t or int64_t
struct Bracket {
    I whole, zi, zk;
    __device__ __forceinline__ explicit Bracket(const TableSums &s)
        : zi((I)s.grids->in.zero), zk((I)s.grids->kernel.zero)
    {
        whole = (I)s.K * zi * zk - (I)s.pad * (I)s.table[0];
    }
    __device__ __forceinline__ I row(int32_t row_sum) const { return whole - zk * (I)row_sum; }
    __device__ __forceinline__ I column(int32_t column_sum) const { return zi * (I)column_sum; }
    // of the sum of table entries, which is 0 or more and below 2^31
    __device__ __forceinline__ static float value(int32_t sum, I row, I column)
    {
        if constexpr (sizeof(I) == 4)
            return (float)(int32_t)((I)sum + row - column);
        else
            return (float)((I)sum + row - column);
    }
};

// Four neighbouring sums, at (r, c) to (r, c + 3), or to (r + 3, c) where they are turned.
__device__ __forceinline__ i32x4 four_sums(const RawSums &s, int64_t r, int64_t c)
{
    const int32_t *const p = s.acc + (s.turned ? c * s.pitch + r : r * s.pitch + c);
    i32x4 t = {};
#pragma unroll 8
    for (int i = 0; i < s.splits; ++i)
        t += *reinterpret_cast<const i32x4 *>(p + i * s.split_stride);
    return t;
}

// reported: x is null, and this is what a call before has reported of it.
hipError_t launch_range(const void *x, int x_type, int64_t nx, const float *reported, const void *kernel, int kernel_type, int64_t nk,
                        float *x_pairs, float *kernel_pairs, int32_t *zeros, int64_t n_zeros, int *x_count, int *kernel_count,
                        hipStream_t stream);
// Codes of both operands and their sums, and the grids they are on.  x null: only the kernel's; kernel null: only the input's,
// and the kernel's grid is that of kernel_grid.
struct CodesJob {
    const void *x, *kernel;
    int x_type, kernel_type;
    int64_t rows, N;
    int K;
    RangeSource x_range, kernel_range;
    const Grid *kernel_grid;
    Pieces pieces;
    Grids *grids;
    uint8_t *x_codes, *kernel_codes;
    uint8_t *kernel_blocks;              // kernel_codes and kernel_blocks: the two layouts, either may be null
    int32_t *row_sums, *column_sums;     // (those of the columns are added to)
};
hipError_t launch_codes(const CodesJob &job, hipStream_t stream);
struct DenseOut {
    const void *bias, *residual;         // of the piece's / run's first element
    void *out, *pre;
    int bias_type, type, activation;
    int64_t ld;                          // columns of the layer
};
struct FewInput {                        // few rows of an input, and where its grid and the kernel's come from
    const void *x;
    int type, K;
    RangeSource range;
    const Grid *kernel_grid;
};
// Range (where it is not known), grid, codes and their sums of the input in one launch; a kernel_grid that is not null is copied
// next to it.
hipError_t launch_few_codes(const FewInput &in, int rows, int Kb, Grids *grids, uint8_t *codes, int32_t *row_sums, hipStream_t stream);
constexpr int kFewRowsAtOnce = 8;        // rows that a workgroup of few_rows_kernel takes
struct FewJob {
    const uint16_t *tableS;
    FewInput in;                         // x not null: the input as it is, its grid and the kernel's go to *grids, else:
    const uint8_t *x_codes;
    Grids *grids;
    const uint8_t *kernel_blocks;        // of a piece
    int rows, Kb, width, splits;
    int32_t *acc;                        // [splits][rows][pitch]; of an input as it is, the rows' sums are column `width`
    int pitch;
};
// Where every workgroup may read all of the input for its range: beyond that a launch of its own is as short (us a call without and
// with one, 4096 -> 4096: 8 rows 22 and 25).
constexpr int64_t kFewRawValues = 65536;
int few_rows_splits(int64_t rows, int Kb, int width);
hipError_t launch_few_rows(const FewJob &job, hipStream_t stream);

struct TokenJob {                        // one or two rows, and all that is made of them, in one launch
    const uint16_t *tableL;
    FewInput in;
    const uint8_t *kernel_blocks;
    const int32_t *column_sums;
    Pieces pieces;
    int rows;
    int64_t columns;
    DenseOut out;
};
bool token_fits(int64_t rows, int Kb);   // whether a workgroup has room for all of the input's codes
hipError_t launch_token(const TokenJob &job, hipStream_t stream);
hipError_t launch_zero(void *p, int64_t bytes, hipStream_t stream);   // a kernel: callers may capture it
hipError_t launch_dense_out(const TableSums &s, int64_t rows, int columns, const DenseOut &o, hipStream_t stream);

// ---- products of gradients with codes (gradient_kernels.hip) ----
// Operands in bfloat16, rows and depth padded to kProductTile.  Codes minus their zero point are whole numbers below 256 and
// exact in bfloat16; the other operand is split into `parts` terms of 8 bits each: three for float32 results, 24 bits, two for 16-bit
// ones, whose rounding (2^-16) is far below the result's own (2^-8, 2^-11), and fewer where fewer hold the gradient as it is (`exact`).
// One term of anything else for bfloat16 results is half the products, but as far off as the result's own rounding: the gradients of 4096
// rows, 1024 -> 4096, with Gelu were off from 64 bits by 2.3e-3 in 118 us, and are by 1.7e-3, the rounding's own, in 195.
constexpr int kProductTile = 128;
__host__ __device__ inline int64_t product_pad(int64_t n) { return (n + kProductTile - 1) / kProductTile * kProductTile; }
inline int parts_of(int result_type, int exact) { return result_type == AXC_F32 || exact < 2 ? exact : 2; }
// Terms that hold every gradient behind a dense layer's product: those of its type where nothing but 0 and 1 was multiplied into it.
inline int exact_terms(int type, int activation)
{
    if (activation != AXC_ACT_NONE && activation != AXC_ACT_RELU)
        return 3;
    return type == AXC_BF16 ? 1 : type == AXC_F16 ? 2 : 3;
}

struct GradSource {                      // where the gradient behind the product comes from
    const void *grad, *pre;              // dense: gradient of the output, what the activation was given (or null)
    int type, activation;
    // loss: sums of a piece, each row's largest logit and log of the sum of exponentials around it, its coefficient and target
    TableSums sums;
    const float *top, *log_sum, *coefficient;
    const int64_t *targets;
    const void *bias;
    int bias_type;
    int64_t first_column;
};
struct CenteredJob {                     // codes minus zero point of a tensor; out null: not wanted
    const void *values;
    int type;
    int64_t rows, cols, ld;
    bf16 *out;
};
// What stands in front of the products: of the gradient [rows_pad][parts][cols_pad], [cols_pad][parts][rows_pad] and per 64 rows the
// sums over them (each may be null), for the run of rows from `first` on (a multiple of kProductTile) out of `rows`, of_run describing
// its run_rows rows; of the input's codes [cols_pad][rows_pad], of the kernel's [rows_pad][cols_pad].  ranges (of input and kernel):
// the grids are not made yet, and this launch does.
hipError_t launch_grad_prep(const GradSource &of_run, bool loss, int64_t first, int64_t run_rows, int64_t rows, int64_t cols,
                            int64_t ld, int straight_parts, bf16 *straight, int turned_parts, bf16 *turned, float *column_partials,
                            const CenteredJob &x, const CenteredJob &kernel, const RangeSource *ranges, Grids *grids,
                            hipStream_t stream);
struct ColumnJob {                       // out[c] = sum over i of partials[i * pitch + c], times *factor
    const float *partials;
    int64_t count, cols, pitch;
    const float *factor;
    void *out;
    int type;
    int64_t blocks() const { return out ? (cols + 63) / 64 : 0; }
};
hipError_t launch_column_sums(const ColumnJob &job, hipStream_t stream);
struct ProductOut {
    void *out;                           // rows x cols, leading dimension ld
    int type;
    int64_t ld;
    const void *values;                  // like out, of its type: where they are outside `grid`, out gets 0
    int64_t values_ld;
    const Grid *grid, *scale;            // scale->scale times the sums
    const float *factor;                 // not null: times *factor
};
// out[r][c] = sum over parts and l of a[r][..l] * b[c][..l]; the operand with the parts is a where split_a, else b.
struct Product {
    const bf16 *a, *b;
    int64_t rows, cols;
    int depth, parts, split_a;           // depth in whole tiles
    int splits;                          // of the depth, by plan_products
    float *partials;                     // [splits][rows in tiles][cols in tiles]; null: not split, and not kept
    int accumulate;                      // add to the partial sums that are there
    ProductOut o;
};
struct ProductShape {
    int64_t rows, cols, depth;           // any; keep: its partial sums go on from launch to launch
    int parts, keep;
};
struct ProductPlan {
    int splits;
    size_t partial_bytes;
};
// Of one or two products that one launch makes.
void plan_products(const ProductShape *shapes, int count, ProductPlan *plans);
// job: column sums that the launch makes too.
hipError_t launch_products(const Product *products, int count, const ColumnJob &job, hipStream_t stream);
// What the partial sums of products give.
hipError_t launch_products_out(const Product *products, int count, hipStream_t stream);
// ---- loss (loss_kernels.hip) ----
// Columns at least that leave a maximum and a sum: fewer where few rows would leave CUs without work.
inline int loss_chunk(int64_t rows) { return rows >= 2048 ? 512 : rows >= 512 ? 256 : 64; }
struct LossState {
    float2 *parts;                       // [chunk][rows]: the largest logit and the sum of exponentials around it
    float *at;                           // per row: the target's logit
    float *top, *log_sum;                // the largest of all, and the log of the whole sum around it: not in one, whose rounding would be that
                                         // of what all logits have in common
    float *rows;                         // the row's loss
    float *coefficient, *factor;         // a row's gradient is multiplied by coefficient[row] * *factor
};
// Of a run of rows from `first_row` on, into parts from `chunk` on; returns how many chunks in *chunks.
hipError_t launch_loss_piece(const TableSums &s, int64_t first_row, int64_t run_rows, int64_t rows, int columns, int64_t first_column,
                             const void *bias, int bias_type, const int64_t *targets, int chunk, int *chunks, const LossState &st,
                             hipStream_t stream);
hipError_t launch_loss_rows(const LossState &st, const int64_t *targets, int64_t ignore, int64_t V, int64_t first_row, int64_t run_rows,
                            int64_t rows, int chunks, hipStream_t stream);
hipError_t launch_loss_out(const LossState &st, const int64_t *targets, int64_t ignore, int64_t V, int64_t rows, int reduction,
                           const float *grad_loss, float *loss, bool gradients, hipStream_t stream);

// ---- residual norms (norm_kernels.hip) ----
struct NormParams {
    int64_t rows, width, gate_groups;    // gate_groups: 0 = no gate; rows / gate_groups neighbouring rows share one
    int type, layer;                     // layer: 1 = LayerNorm, 0 = RMSNorm
    float eps;
    const void *x, *block, *weight, *bias, *gate, *scale, *post_weight;
    int vector_type;                     // of weight, bias, scale, post_weight
    void *h, *y;
    float *range;                        // kRangePairs pairs, or null
    // backwards: h is read; gradients in, gradients out (any may be null)
    const void *grad_h, *grad_y;
    void *dx, *dblock;
    void *dweight, *dbias, *dgate, *dscale, *dpost;
    float *partials;
};
constexpr int kNormMaxWidth = 32768;
hipError_t launch_norm(const NormParams &p, hipStream_t stream);
size_t norm_partial_bytes(const NormParams &p);
hipError_t launch_norm_gradients(const NormParams &p, hipStream_t stream);

} // namespace axc

// The table as its owner has it (axconv_api.hip).
struct axc_table {
    uint16_t *dev_tableT; // [257 filter code][256 input code]; row 256 is zero
    uint16_t *dev_tableF; // behind it in the same allocation: the same with the top bit of every byte flipped,
    uint16_t *dev_tableS; // and [257 input code][256 filter code], flipped too
    uint16_t *dev_tableL; // T[a][b] at [r][b ^ r], r the bits of a turned round, for single tokens
    int device;
};

namespace axc {
// What the entry points of axconv_api.hip use, for those of layers_api.hip.
int api_fail(int status, const char *msg);
int api_fail_hip(hipError_t e, const char *what);
int api_check_table(const axc_table *table);
// axc_conv2d_codes_acc_i32 without the pass that would put its sums in order; *raw is filled, unless there are no sums.
int api_codes_sums(const axc_table *table, const axc_conv2d_desc *desc, const uint8_t *input_codes, const uint8_t *filter_codes,
                   int32_t *acc, void *workspace, size_t workspace_bytes, void *stream, RawSums *raw);
class ApiTimer {   // brackets launches while the timers run
public:
    ApiTimer(const char *name, hipStream_t stream);
    ~ApiTimer();
    ApiTimer(const ApiTimer &) = delete;
    ApiTimer &operator=(const ApiTimer &) = delete;

private:
    void *scope_;
};
} // namespace axc
