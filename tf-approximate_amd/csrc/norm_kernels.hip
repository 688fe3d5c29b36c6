// Norms before and after a block of a residual network, with the block's gate and scale:
//
//   u = norm(block) post_weight (or block itself),  h = x + scale gate u,  y = norm(h) weight + bias
//   norm(v) = v / sqrt(mean(v^2) + eps), or (v - mean(v)) / sqrt(var(v) + eps)
//
// h is rounded to the tensors' type before it is normed, so that what the backward pass reads is what was normed.  A workgroup
// takes a row at a time; up to 8192 values, 4096 backwards, it keeps it in registers: everything is read once and written once, which is
// what bounds these kernels.  Wider rows are read again for every sum, by kernels of their own.
// Statistics are float32, the variance from the differences to the mean.
#include "layers_internal.h"

#include <algorithm>

namespace axc {
namespace {

constexpr int kMaxWaves = 16;
constexpr int V = 4;         // values of a vector

// Sums of N values over a workgroup, in every thread.  Two sets of LDS in turn: a set is written again only after the barrier of
// the reduction in between, which nobody passes before all have read it.
struct Reducer {
    float (*red)[kMaxWaves][4];
    int turn;
    template <int N>
    __device__ __forceinline__ void sum(float (&v)[N])
    {
        static_assert(N <= 4, "what a set holds");
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] = wave_sum(v[i]);
        const int waves = blockDim.x / 64;
        if (waves == 1)
            return;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i)
                red[turn][threadIdx.x / 64][i] = v[i];
        __syncthreads();
        const int lane = threadIdx.x & 15;   // a wavefront's sum each
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float part = red[turn][lane][i];
            v[i] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(
                                                 __builtin_bit_cast(int, row_of_lanes_sum(lane < waves ? part : 0.0f)), 15));
        }
    }
};

// A row in registers: NV vectors of four values a thread, vector j of thread t at (j * threads + t) * 4.  Rows of odd widths begin
// anywhere, so vectors are accessed as aligned as their elements are.
//
// Loads have no conditions: where a branch stands between a load and its use, the compiler waits for everything in flight, stores
// included.  In rows that are no whole aligned vectors (kOdd), a vector behind the row is loaded from the row's last four values
// and counts as zeros; the one that ends behind the row is loaded from there too, and moved.  Rows of less than four values (kTiny)
// are loaded one by one.
enum { kEven, kOdd, kTiny };
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ int place(int j) { return (j * (int)blockDim.x + (int)threadIdx.x) * V; }

template <typename T>
struct Vector {
    typedef T four __attribute__((ext_vector_type(4)));
    typedef four loose __attribute__((aligned(sizeof(T))));
};
template <int W, typename T>
__device__ __forceinline__ typename Vector<T>::four load_four(const T *p, int c, int width)
{
    if constexpr (W == kTiny) {
        typename Vector<T>::four t;
#pragma unroll
        for (int i = 0; i < V; ++i)
            t[i] = p[c + i < width ? c + i : width - 1];
        return t;
    } else {
        return *reinterpret_cast<const typename Vector<T>::loose *>(p + (c + V <= width ? c : width - V));
    }
}
// What load_four has loaded, as floats, in their places, with zeros behind the row.
template <int W, typename T>
__device__ __forceinline__ f32x4 in_place(const T &t, int c, int width)
{
    f32x4 v;
    if constexpr (W == kEven) {        // (zeros as loaded)
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[i] = (float)t[i];
    } else if constexpr (W == kTiny) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[i] = c + i < width ? (float)t[i] : 0.0f;
    } else {
        const int moved = c + V - width;   // 1 to 3 in the last vector
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float x = moved > 0 ? 0.0f : (float)t[i];
#pragma unroll
            for (int d = 1; d + i < V; ++d)
                x = moved == d ? (float)t[i + d] : x;
            v[i] = x;
        }
    }
    return v;
}
template <int W, typename T>
__device__ __forceinline__ void store_four(T *p, int c, int width, const float (&v)[V])
{
    if (W == kEven ? c < width : c + V <= width) {
        typename Vector<T>::four t;
#pragma unroll
        for (int i = 0; i < V; ++i)
            t[i] = (T)v[i];
        *reinterpret_cast<typename Vector<T>::loose *>(p + c) = t;
    } else if (W != kEven) {
#pragma unroll
        for (int i = 0; i < V - 1; ++i)
            if (c + i < width)
                p[c + i] = (T)v[i];
    }
}

// Rows of a tensor.  Aligned rows of whole vectors go through buffer descriptors, which give zeros for what lies behind a row (or
// for all of one that is not there, of no bytes) and drop stores there, so that neither needs a condition.
template <int W, typename T>
struct Rows {
    T *base;
    int width;
    bool there;
    __device__ __forceinline__ Rows(const void *p, int w) : base(static_cast<T *>(const_cast<void *>(p))), width(w), there(p != nullptr) {}
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t row(int64_t r) const
    {
        return __builtin_amdgcn_make_buffer_rsrc(base + r * width, 0, there ? width * (int)sizeof(T) : 0, 0x00020000);
    }
};

template <int NV>
struct Row {
    float v[NV][V];
};
template <typename T, int NV>
struct Raw {               // a row as it was loaded
    typename Vector<T>::four v[NV];
};
template <int W, typename T, int NV>
__device__ __forceinline__ void load_row(const Rows<W, T> &t, int64_t row, Raw<T, NV> &r)
{
    if constexpr (W == kEven) {
        const __amdgpu_buffer_rsrc_t from = t.row(row);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if constexpr (sizeof(T) == 4)
                r.v[j] = __builtin_bit_cast(typename Vector<T>::four,
                                            __builtin_amdgcn_raw_buffer_load_b128(from, place(j) * (int)sizeof(T), 0, 0));
            else
                r.v[j] = __builtin_bit_cast(typename Vector<T>::four,
                                            __builtin_amdgcn_raw_buffer_load_b64(from, place(j) * (int)sizeof(T), 0, 0));
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            r.v[j] = load_four<W>(t.base + row * t.width, place(j), t.width);
    }
}
template <int W, typename T, int NV>
__device__ __forceinline__ Row<NV> widen(const Raw<T, NV> &r, int width)
{
    Row<NV> w;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const f32x4 v = in_place<W>(r.v[j], place(j), width);
#pragma unroll
        for (int i = 0; i < V; ++i)
            w.v[j][i] = v[i];
    }
    return w;
}
template <int W, typename T, int NV>
__device__ __forceinline__ void store_row(const Rows<W, T> &t, int64_t row, const Row<NV> &r)
{
    if constexpr (W == kEven) {
        const __amdgpu_buffer_rsrc_t to = t.row(row);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            typename Vector<T>::four v;
#pragma unroll
            for (int i = 0; i < V; ++i)
                v[i] = (T)r.v[j][i];
            if constexpr (sizeof(T) == 4)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), to, place(j) * (int)sizeof(T), 0, 0);
            else
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v), to, place(j) * (int)sizeof(T), 0, 0);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            store_four<W>(t.base + row * t.width, place(j), t.width, r.v[j]);
    }
}
template <int NV>
__device__ __forceinline__ void scale_row(Row<NV> &r, float f)
{
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
            r.v[j][i] *= f;
}
template <int NV>
__device__ __forceinline__ float row_sum(const Row<NV> &r)
{
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
            s += r.v[j][i];
    return s;
}
template <int NV>
__device__ __forceinline__ float row_dot(const Row<NV> &a, const Row<NV> &b)
{
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
            s = fmaf(a.v[j][i], b.v[j][i], s);
    return s;
}
// Takes the mean from a row's values; what lies behind the row stays 0.
template <int W, int NV>
__device__ __forceinline__ void subtract(Row<NV> &r, float mean, int width)
{
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
            r.v[j][i] -= place(j) + (W == kEven ? 0 : i) < width ? mean : 0.0f;
}
__device__ __forceinline__ float root(float squares, int width, float eps) { return 1.0f / sqrtf(squares / (float)width + eps); }

// r becomes (v - mean) / sqrt(var + eps), mean 0 for RMS.
template <int W, int NV>
__device__ __forceinline__ void normalize(Row<NV> &r, const NormParams &p, Reducer &red)
{
    const int width = (int)p.width;
    float s[1];
    if (p.layer) {
        s[0] = row_sum(r);
        red.sum(s);
        subtract<W>(r, s[0] / (float)width, width);
    }
    s[0] = row_dot(r, r);
    red.sum(s);
    scale_row(r, root(s[0], width, p.eps));
}

// Four values of one of the layer's vectors, as floats; ones where it is not there.
template <int W>
__device__ __forceinline__ f32x4 load_vector(const void *p, int type, int c, int width)
{
    if (!p)
        return f32x4{1.0f, 1.0f, 1.0f, 1.0f};
    if (type == AXC_F32)
        return in_place<W>(load_four<W>(static_cast<const float *>(p), c, width), c, width);
    if (type == AXC_BF16)
        return in_place<W>(load_four<W>(static_cast<const bf16 *>(p), c, width), c, width);
    return in_place<W>(load_four<W>(static_cast<const f16 *>(p), c, width), c, width);
}

// The layer's vectors (weights and the like), as floats in LDS: each thread its own columns, so without a barrier.  Those that are not
// there are ones (rather than a branch where they are used, which took a tenth longer).
template <int W, int NV, int N>
struct Kept {
    f32x4 *lds;
    const void *vectors[N];
    int type, width;
    static int bytes(int threads) { return N * threads * NV * V * (int)sizeof(float); }
    __device__ __forceinline__ void fill()
    {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int j = 0; j < NV; ++j)
                lds[(k * NV + j) * (int)blockDim.x + (int)threadIdx.x] =
                    load_vector<W == kTiny ? kTiny : kOdd>(vectors[k], type, place(j), width);   // (may be aligned as their elements only)
    }
    __device__ __forceinline__ f32x4 get(int which, int j) const
    {
        return lds[(which * NV + j) * (int)blockDim.x + (int)threadIdx.x];
    }
};

enum { kWeight, kScale, kPost, kBias };

// A workgroup's pair of the range of y.
__device__ __forceinline__ void report_range(const NormParams &p, float lo, float hi, float *ends)
{
    if (!p.range)
        return;
    block_range(lo, hi, ends);
    if (threadIdx.x == 0)
        reinterpret_cast<float2 *>(p.range)[blockIdx.x] = make_float2(lo, hi);
    if (blockIdx.x == 0)   // pairs that nobody has
        for (int i = (int)gridDim.x + (int)threadIdx.x; i < kRangePairs; i += blockDim.x)
            reinterpret_cast<float2 *>(p.range)[i] = make_float2(INFINITY, -INFINITY);
}

template <typename T, int NV, int W>
__global__ void __launch_bounds__(512) norm_kernel(NormParams p)
{
    __shared__ float lds[2][kMaxWaves][4];
    __shared__ float ends[2 * kMaxWaves];
    extern __shared__ f32x4 kept_lds[];
    Reducer red = {lds, 0};
    const int width = (int)p.width;
    const int64_t group_rows = p.gate_groups ? p.rows / p.gate_groups : 1;
    Kept<W, NV, 4> kept = {kept_lds, {p.weight, p.scale, p.post_weight, p.bias}, p.vector_type, width};
    // (what is not there is loaded in any case, for nothing)
    const Rows<W, T> x(p.x, width), block(W == kEven || p.block ? p.block : p.x, width), gate(p.gate, width), hs(p.h, width),
        ys(p.y, width);
    float lo = INFINITY, hi = -INFINITY;
    // the gate group of the row that is loaded, and the row's place in it; a step of the loop further on
    int64_t group = (int64_t)blockIdx.x / group_rows, in_group = (int64_t)blockIdx.x - group * group_rows;
    const int64_t more_groups = (int64_t)gridDim.x / group_rows, more_rows = (int64_t)gridDim.x - more_groups * group_rows;
    Raw<T, NV> xr, br, gr = {};
    auto load = [&](int64_t r) {
        load_row(x, r, xr);
        load_row(block, p.block ? r : 0, br);
        if (p.gate)
            load_row(gate, group, gr);
        group += more_groups;
        in_group += more_rows;
        if (in_group >= group_rows) {
            in_group -= group_rows;
            ++group;
        }
    };
    load(blockIdx.x);
    kept.fill();
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        Row<NV> h = widen<W>(xr, width);
        Row<NV> u = widen<W>(br, width);
        const Raw<T, NV> ga = gr;
        if (r + gridDim.x < p.rows)
            load(r + gridDim.x);
        if (p.block) {
            if (p.post_weight)
                normalize<W>(u, p, red);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const f32x4 post = kept.get(kPost, j), scale = kept.get(kScale, j);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    u.v[j][i] *= post[i];
                if (p.gate) {
                    const f32x4 g = in_place<W>(ga.v[j], place(j), width);
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        u.v[j][i] *= g[i];
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float s = h.v[j][i] + u.v[j][i] * scale[i];
                    h.v[j][i] = place(j) + (W == kEven ? 0 : i) < width ? (float)(T)s : 0.0f;
                }
            }
            store_row(hs, r, h);
        }
        normalize<W>(h, p, red);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const f32x4 w = kept.get(kWeight, j);
#pragma unroll
            for (int i = 0; i < V; ++i)
                h.v[j][i] *= w[i];
            if (p.bias) {
                const f32x4 b = kept.get(kBias, j);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    h.v[j][i] += b[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float y = (float)(T)h.v[j][i];
                const bool there = place(j) + (W == kEven ? 0 : i) < width;
                lo = fminf(lo, there ? y : INFINITY);
                hi = fmaxf(hi, there ? y : -INFINITY);
            }
        }
        store_row(ys, r, h);
    }
    report_range(p, lo, hi, ends);
}

// Rows of more than 8192 values do not stay in registers: every sum goes over the row again, out of the caches, and other workgroups of
// the CU take the place of loads ahead.  16 384 values of bfloat16, 33.6 M altogether, take 76 us (216 in registers that spill).
template <typename T>
struct WideRow {                         // four values of a row, whatever its alignment
    const T *p;
    __device__ __forceinline__ WideRow(const void *base, int64_t row, int width)
        : p(base ? static_cast<const T *>(base) + row * width : nullptr)
    {
    }
    __device__ __forceinline__ f32x4 at(int c, int width) const
    {
        return p ? in_place<kOdd>(load_four<kOdd>(p, c, width), c, width) : f32x4{};
    }
};
template <typename T>
__global__ void __launch_bounds__(512) wide_norm_kernel(NormParams p)
{
    __shared__ float lds[2][kMaxWaves][4];
    __shared__ float ends[2 * kMaxWaves];
    Reducer red = {lds, 0};
    const int width = (int)p.width, step = (int)blockDim.x * V, c0 = (int)threadIdx.x * V;
    const int64_t group_rows = p.gate_groups ? p.rows / p.gate_groups : 1;
    float lo = INFINITY, hi = -INFINITY;
    auto squares = [&](const WideRow<T> &row, float mean) {
        float s[1] = {};
#pragma unroll 4
        for (int c = c0; c < width; c += step) {
            const f32x4 v = row.at(c, width);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = c + i < width ? v[i] - mean : 0.0f;
                s[0] = fmaf(d, d, s[0]);
            }
        }
        red.sum(s);
        return s[0];
    };
    auto mean_of = [&](const WideRow<T> &row) {
        float s[1] = {};
#pragma unroll 4
        for (int c = c0; c < width; c += step) {
            const f32x4 v = row.at(c, width);
            s[0] += v[0] + v[1] + v[2] + v[3];
        }
        red.sum(s);
        return s[0] / (float)width;
    };
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const WideRow<T> x(p.x, r, width), block(p.block, r, width), gate(p.gate, r / group_rows, width),
            h(p.block ? p.h : p.x, r, width);
        if (p.block) {
            float mean = 0.0f, factor = 1.0f;
            if (p.post_weight) {
                mean = p.layer ? mean_of(block) : 0.0f;
                factor = root(squares(block, mean), width, p.eps);
            }
#pragma unroll 2
            for (int c = c0; c < width; c += step) {
                const f32x4 v = x.at(c, width), b = block.at(c, width), post = load_vector<kOdd>(p.post_weight, p.vector_type, c, width),
                            scale = load_vector<kOdd>(p.scale, p.vector_type, c, width);
                const f32x4 g = p.gate ? gate.at(c, width) : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
                float t[V];
#pragma unroll
                for (int i = 0; i < V; ++i)
                    t[i] = v[i] + (b[i] - mean) * factor * post[i] * g[i] * scale[i];
                store_four<kOdd>(static_cast<T *>(p.h) + r * width, c, width, t);
            }
            // the row's last whole vector is read again by the thread of what is behind it
            __threadfence_block();
            __syncthreads();
        }
        const float mean = p.layer ? mean_of(h) : 0.0f, factor = root(squares(h, mean), width, p.eps);
#pragma unroll 2
        for (int c = c0; c < width; c += step) {
            const f32x4 v = h.at(c, width), w = load_vector<kOdd>(p.weight, p.vector_type, c, width);
            const f32x4 b = p.bias ? load_vector<kOdd>(p.bias, p.vector_type, c, width) : f32x4{};
            float t[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                t[i] = (v[i] - mean) * factor * w[i] + b[i];
                const float y = (float)(T)t[i];
                const bool there = c + i < width;
                lo = fminf(lo, there ? y : INFINITY);
                hi = fmaxf(hi, there ? y : -INFINITY);
            }
            store_four<kOdd>(static_cast<T *>(p.y) + r * width, c, width, t);
        }
    }
    report_range(p, lo, hi, ends);
}

// ---- backwards ----
//   n = norm(v), g the gradient of n:  dv = (g - n mean(g n) [- mean(g)]) / root
// With d = v - mean, n = d / root: mean(g n) is made of sum(g d), which needs no root and so goes into the same reduction as
// sum(d^2).  A row is two reductions, three for LayerNorm, and its successor is loaded ahead of them.
// A workgroup takes a run of neighbouring rows, all of one gate group or whole groups, and keeps the sums over rows (for the
// weights, the bias, the scale, the gate) in registers, a column in the same thread throughout; norm_column_kernel adds up what the
// runs leave, in one order.
struct NormRuns {
    int64_t run;            // rows of a workgroup
    int64_t per_group;      // workgroups of a gate group; 0: a workgroup takes whole groups, or there is no gate
    int64_t blocks;
};
constexpr int64_t kRunBlocks = 768;      // about as many workgroups, three a CU: what is resident
NormRuns norm_runs(int64_t rows, int64_t groups)
{
    NormRuns n = {};
    n.run = (rows + kRunBlocks - 1) / kRunBlocks;
    const int64_t group = groups ? rows / groups : 1;
    if (groups && group > n.run) {
        n.per_group = (group + n.run - 1) / n.run;
        n.run = (group + n.per_group - 1) / n.per_group;
        n.per_group = (group + n.run - 1) / n.run;
        n.blocks = n.per_group * groups;
    } else {
        n.run = (n.run + group - 1) / group * group;
        n.blocks = (rows + n.run - 1) / n.run;
    }
    return n;
}
enum { kSumWeight, kSumBias, kSumScale, kSumPost, kSumGate, kSums };

// Three wavefronts a SIMD are 168 registers each: rows of 16-bit values that are no whole vectors would take 171 (1283 of
// them, 33.6 M altogether: 177 us by two a SIMD, 133 by three); 32-bit ones would spill too many (181 us by two, 248 by three).
template <typename T, int NV, int W>
__global__ void __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(sizeof(T) == 2 ? 3 : 2))) norm_grad_kernel(NormParams p, NormRuns runs)
{
    __shared__ float lds[2][kMaxWaves][4];
    extern __shared__ f32x4 kept_lds[];
    Reducer red = {lds, 0};
    const int width = (int)p.width;
    const int64_t group_rows = p.gate_groups ? p.rows / p.gate_groups : 1;
    Kept<W, NV, 3> kept = {kept_lds, {p.weight, p.scale, p.post_weight}, p.vector_type, width};
    int64_t first, last, group, left;   // left: rows of the group behind the one at hand
    if (runs.per_group) {
        group = blockIdx.x / runs.per_group;
        first = group * group_rows + (blockIdx.x - group * runs.per_group) * runs.run;
        last = first + runs.run < (group + 1) * group_rows ? first + runs.run : (group + 1) * group_rows;
        left = (group + 1) * group_rows - first;
    } else {
        first = (int64_t)blockIdx.x * runs.run;
        last = first + runs.run < p.rows ? first + runs.run : p.rows;
        group = first / group_rows;
        left = group_rows;
    }
    // (what is not there is loaded in any case, as zeros or from h for nothing; a gate that is not there counts as ones)
    const void *const other = W == kEven ? nullptr : p.h;
    const Rows<W, T> hs(p.h, width), gys(p.grad_y ? p.grad_y : other, width), ghs(p.grad_h ? p.grad_h : other, width),
        blocks(p.block ? p.block : other, width), gates(p.gate, width), dxs(p.dx, width), dblocks(p.dblock, width),
        dgates(p.dgate, width);
    Raw<T, NV> hr, gyr, ghr, br, gr = {};
    auto load = [&](int64_t r, int64_t of) {
        load_row(hs, r, hr);
        load_row(gys, W == kEven && !p.grad_y ? 0 : r, gyr);
        load_row(ghs, W == kEven && !p.grad_h ? 0 : r, ghr);
        load_row(blocks, W == kEven && !p.block ? 0 : r, br);
        if (p.gate)
            load_row(gates, of, gr);
    };
    Row<NV> sw = {}, sb = {}, ss = {}, sp = {}, sg = {};
    if (first < last)
        load(first, group);
    kept.fill();
    for (int64_t r = first; r < last; ++r) {
        const bool ends = --left == 0;   // the group's last row
        const int64_t of = group;
        if (ends) {
            ++group;
            left = group_rows;
        }
        Row<NV> n = widen<W>(hr, width), b = widen<W>(br, width), dh = widen<W>(gyr, width), gh = widen<W>(ghr, width);
        const Raw<T, NV> gate = gr;
        if (r + 1 < last)              // ahead of all reductions
            load(r + 1, group);
        if constexpr (W != kEven)
            if (!p.grad_h)
                gh = {};
        if (p.layer) {
            float s[2] = {row_sum(n), row_sum(b)};
            red.sum(s);
            subtract<W>(n, s[0] / (float)width, width);
            if (p.post_weight)
                subtract<W>(b, s[1] / (float)width, width);
        }
        Row<NV> g = dh;                // the gradient of norm(h); dh that of y, until it is that of h itself
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const f32x4 w = kept.get(kWeight, j);
#pragma unroll
            for (int i = 0; i < V; ++i)
                g.v[j][i] *= w[i];
        }
        float s[4] = {row_dot(n, n), row_dot(g, n), row_sum(g), row_dot(b, b)};
        red.sum(s);
        const float rh = root(s[0], width, p.eps), rb = p.post_weight ? root(s[3], width, p.eps) : 1.0f;
        const float mgn = s[1] * rh / (float)width, mg = p.layer ? s[2] / (float)width : 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float at = n.v[j][i] * rh, gy = dh.v[j][i];
                sw.v[j][i] = fmaf(gy, at, sw.v[j][i]);
                sb.v[j][i] += gy;
                dh.v[j][i] = (g.v[j][i] - at * mgn - mg) * rh + gh.v[j][i];
            }
        if (!p.grad_y)                 // (rather than 0 times what may be infinite)
            dh = gh;
        store_row(dxs, r, dh);
        if (!p.block)
            continue;
        // du = dh scale gate; b is the block, normed where it is
        scale_row(b, rb);
        float t[2] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const f32x4 w = kept.get(kPost, j), sc = kept.get(kScale, j);
            f32x4 ga = {1.0f, 1.0f, 1.0f, 1.0f};
            if (p.gate)
                ga = in_place<W>(gate.v[j], place(j), width);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float hu = dh.v[j][i] * b.v[j][i] * w[i];   // dh u
                ss.v[j][i] = fmaf(hu, ga[i], ss.v[j][i]);
                sg.v[j][i] = fmaf(hu, sc[i], sg.v[j][i]);
                const float du = dh.v[j][i] * sc[i] * ga[i];
                sp.v[j][i] = fmaf(du, b.v[j][i], sp.v[j][i]);
                dh.v[j][i] = place(j) + (W == kEven ? 0 : i) < width ? du * w[i] : 0.0f;
                t[0] = fmaf(dh.v[j][i], b.v[j][i], t[0]);
                t[1] += dh.v[j][i];
            }
        }
        if (p.post_weight) {
            red.sum(t);
            const float mtn = t[0] / (float)width, mt = p.layer ? t[1] / (float)width : 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    dh.v[j][i] = (dh.v[j][i] - b.v[j][i] * mtn - mt) * rb;
        }
        store_row(dblocks, r, dh);
        if (p.dgate && !runs.per_group && ends) {
            store_row(dgates, of, sg);
            sg = {};
        }
    }
    if (!p.grad_y) {                   // what is not there was loaded for nothing, and 0 times an infinite h is no 0
        sw = {};
        sb = {};
    }
    const Rows<W, float> to(p.partials, width);
    const int64_t at = (int64_t)blockIdx.x * kSums;
    if (p.dweight)
        store_row(to, at + kSumWeight, sw);
    if (p.dbias)
        store_row(to, at + kSumBias, sb);
    if (p.dscale)
        store_row(to, at + kSumScale, ss);
    if (p.dpost)
        store_row(to, at + kSumPost, sp);
    if (p.dgate && runs.per_group)
        store_row(to, at + kSumGate, sg);
}

// Wide rows backwards, in two launches: nine rows of four vectors a thread are more than its registers (spilled, rows of 16 384 took
// 1630 us for 33.6 M values of bfloat16; 203 this way, rows of 8192 207 and 199; a norm of the block is a further pass, 349 and 326).
// The first leaves what a row's sums are, going over it from memory once for every dependent reduction; with that everything is value
// by value, and the second takes tiles of columns by runs of rows.
constexpr int kWideBackward = 4096;      // values that are not wide yet
struct RowStats {
    float mean, root, mgn, mg;           // of h: n = (h - mean) root; means of g n and of g
    float block_mean, block_root, mtn, mt;
};
template <typename T>
__global__ void __launch_bounds__(512) wide_stats_kernel(NormParams p, RowStats *__restrict__ stats)
{
    __shared__ float lds[2][kMaxWaves][4];
    Reducer red = {lds, 0};
    const int width = (int)p.width, step = (int)blockDim.x * V, c0 = (int)threadIdx.x * V;
    const int64_t group_rows = p.gate_groups ? p.rows / p.gate_groups : 1;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const WideRow<T> h(p.h, r, width), gy(p.grad_y, r, width), gh(p.grad_h, r, width),
            b(p.post_weight ? p.block : nullptr, r, width), gate(p.gate, r / group_rows, width);
        RowStats st = {};
        st.block_root = 1.0f;
        if (p.layer) {
            float s[2] = {};
            for (int c = c0; c < width; c += step) {
                const f32x4 x = h.at(c, width), y = b.at(c, width);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s[0] += x[i];
                    s[1] += y[i];
                }
            }
            red.sum(s);
            st.mean = s[0] / (float)width;
            if (p.post_weight)
                st.block_mean = s[1] / (float)width;
        }
        float s[4] = {};
#pragma unroll 2
        for (int c = c0; c < width; c += step) {
            const f32x4 x = h.at(c, width), y = b.at(c, width), w = load_vector<kOdd>(p.weight, p.vector_type, c, width), g = gy.at(c, width) * w;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool there = c + i < width;
                const float n = there ? x[i] - st.mean : 0.0f, m = there ? y[i] - st.block_mean : 0.0f;
                s[0] = fmaf(n, n, s[0]);
                s[1] = fmaf(g[i], n, s[1]);
                s[2] += g[i];
                s[3] = fmaf(m, m, s[3]);
            }
        }
        red.sum(s);
        st.root = root(s[0], width, p.eps);
        st.mgn = s[1] * st.root / (float)width;
        st.mg = p.layer ? s[2] / (float)width : 0.0f;
        if (p.post_weight) {
            st.block_root = root(s[3], width, p.eps);
            float t[2] = {};
#pragma unroll 2
            for (int c = c0; c < width; c += step) {
                const f32x4 x = h.at(c, width), y = b.at(c, width), w = load_vector<kOdd>(p.weight, p.vector_type, c, width),
                            g = gy.at(c, width) * w, other = gh.at(c, width), sc = load_vector<kOdd>(p.scale, p.vector_type, c, width),
                            post = load_vector<kOdd>(p.post_weight, p.vector_type, c, width);
                const f32x4 ga = p.gate ? gate.at(c, width) : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float at = (x[i] - st.mean) * st.root;
                    const float dh = p.grad_y ? (g[i] - at * st.mgn - st.mg) * st.root + other[i] : other[i];
                    const float du = c + i < width ? dh * sc[i] * ga[i] * post[i] : 0.0f;
                    t[0] = fmaf(du, (y[i] - st.block_mean) * st.block_root, t[0]);
                    t[1] += du;
                }
            }
            red.sum(t);
            st.mtn = t[0] / (float)width;
            st.mt = p.layer ? t[1] / (float)width : 0.0f;
        }
        if (threadIdx.x == 0)
            stats[r] = st;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) wide_grad_kernel(NormParams p, NormRuns runs, const RowStats *__restrict__ stats)
{
    const int width = (int)p.width, c = ((int)blockIdx.x * 256 + (int)threadIdx.x) * V;
    if (c >= width)
        return;
    const int64_t group_rows = p.gate_groups ? p.rows / p.gate_groups : 1, block = blockIdx.y;
    int64_t first, last, group, left;    // as in norm_grad_kernel
    if (runs.per_group) {
        group = block / runs.per_group;
        first = group * group_rows + (block - group * runs.per_group) * runs.run;
        last = first + runs.run < (group + 1) * group_rows ? first + runs.run : (group + 1) * group_rows;
        left = (group + 1) * group_rows - first;
    } else {
        first = block * runs.run;
        last = first + runs.run < p.rows ? first + runs.run : p.rows;
        group = first / group_rows;
        left = group_rows;
    }
    const f32x4 w = load_vector<kOdd>(p.weight, p.vector_type, c, width), sc = load_vector<kOdd>(p.scale, p.vector_type, c, width),
                post = load_vector<kOdd>(p.post_weight, p.vector_type, c, width), ones = {1.0f, 1.0f, 1.0f, 1.0f};
    auto gate_of = [&](int64_t of) { return p.gate ? WideRow<T>(p.gate, of, width).at(c, width) : ones; };
    f32x4 ga = gate_of(group < p.gate_groups ? group : 0), sw = {}, sb = {}, ss = {}, sp = {}, sg = {};
    auto put = [&](void *to, int64_t row, const float (&v)[V]) { store_four<kOdd>(static_cast<T *>(to) + row * width, c, width, v); };
#pragma unroll 2
    for (int64_t r = first; r < last; ++r) {
        const f32x4 x = WideRow<T>(p.h, r, width).at(c, width), gy = WideRow<T>(p.grad_y, r, width).at(c, width),
                    gh = WideRow<T>(p.grad_h, r, width).at(c, width), y = WideRow<T>(p.block, r, width).at(c, width);
        const RowStats st = stats[r];
        float dh[V], du[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float at = (x[i] - st.mean) * st.root;
            sw[i] = fmaf(gy[i], at, sw[i]);
            sb[i] += gy[i];
            dh[i] = p.grad_y ? (gy[i] * w[i] - at * st.mgn - st.mg) * st.root + gh[i] : gh[i];
            const float b = (y[i] - st.block_mean) * st.block_root, hu = dh[i] * b * post[i];   // dh u
            ss[i] = fmaf(hu, ga[i], ss[i]);
            sg[i] = fmaf(hu, sc[i], sg[i]);
            du[i] = dh[i] * sc[i] * ga[i];
            sp[i] = fmaf(du[i], b, sp[i]);
            du[i] *= post[i];
            if (p.post_weight)
                du[i] = (du[i] - b * st.mtn - st.mt) * st.block_root;
        }
        put(p.dx, r, dh);
        if (p.block)
            put(p.dblock, r, du);
        if (--left == 0) {               // the group's last row
            if (p.dgate && !runs.per_group) {
                const float v[V] = {sg[0], sg[1], sg[2], sg[3]};
                put(p.dgate, group, v);
                sg = {};
            }
            ++group;
            left = group_rows;
            if (r + 1 < last)
                ga = gate_of(group < p.gate_groups ? group : 0);
        }
    }
    auto leave = [&](void *wanted, int which, const f32x4 &v) {
        const float t[V] = {v[0], v[1], v[2], v[3]};
        if (wanted)
            store_four<kOdd>(p.partials + (block * kSums + which) * width, c, width, t);
    };
    leave(p.dweight, kSumWeight, p.grad_y ? sw : f32x4{});   // (0 times an infinite h is no 0)
    leave(p.dbias, kSumBias, sb);
    leave(p.dscale, kSumScale, ss);
    leave(p.dpost, kSumPost, sp);
    leave(runs.per_group ? p.dgate : nullptr, kSumGate, sg);
}

struct ColumnSums {
    void *out[kSums];
};
// Sums over the runs' partial sums, 64 columns a workgroup: blockIdx.y = which sum, or which group's gate.
template <typename T>
__global__ void __launch_bounds__(512) norm_column_kernel(const float *__restrict__ partials, int64_t width, NormRuns runs,
                                                          ColumnSums sums, int vector_type)
{
    __shared__ float red[8][64];
    const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const int which = (int)blockIdx.y < kSumGate ? (int)blockIdx.y : kSumGate;
    if (!sums.out[which])
        return;
    const int64_t group = (int64_t)blockIdx.y - kSumGate;
    const int64_t first = which == kSumGate ? group * runs.per_group : 0;
    const int64_t last = which == kSumGate ? first + runs.per_group : runs.blocks;
    float sum = 0.0f;
    if (c < width)
#pragma unroll 4
        for (int64_t i = first + threadIdx.x / 64; i < last; i += 8)
            sum += partials[(i * kSums + which) * width + c];
    red[threadIdx.x / 64][threadIdx.x & 63] = sum;
    __syncthreads();
    if (threadIdx.x >= 64 || c >= width)
        return;
    sum = 0.0f;
    for (int i = 0; i < 8; ++i)
        sum += red[i][threadIdx.x];
    if (which == kSumGate)
        static_cast<T *>(sums.out[kSumGate])[group * width + c] = (T)sum;
    else
        store_any(sums.out[which], c, vector_type, sum);
}

bool whole_vectors(const NormParams &p)
{
    const uintptr_t mask = (uintptr_t)(V * type_bytes(p.type) - 1);
    if (p.width % V)
        return false;
    for (const void *q : {p.x, p.block, p.gate, (const void *)p.h, (const void *)p.y, p.grad_h, p.grad_y, (const void *)p.dx,
                          (const void *)p.dblock, (const void *)p.dgate})
        if ((uintptr_t)q & mask)
            return false;
    return true;
}

// Two vectors a thread up to 4096 values, in steps of a wavefront; then four, and ("8") as many as there are.
template <template <typename, int, int> class Launch, typename T, int W>
hipError_t by_vectors(const NormParams &p, hipStream_t stream)
{
    const int vectors = (int)((p.width + V - 1) / V);
    auto threads = [&](int nv) { return ((vectors + nv - 1) / nv + 63) / 64 * 64; };
    if (vectors <= 128)
        return Launch<T, 1, W>::go(p, threads(1), stream);
    if (vectors <= 1024)
        return Launch<T, 2, W>::go(p, threads(2), stream);
    if (vectors <= 2048)
        return Launch<T, 4, W>::go(p, threads(4), stream);
    return Launch<T, 8, W>::go(p, threads(8), stream);
}
template <template <typename, int, int> class Launch, typename T>
hipError_t by_width(const NormParams &p, hipStream_t stream)
{
    if (p.width < V)
        return Launch<T, 1, kTiny>::go(p, 64, stream);
    return whole_vectors(p) ? by_vectors<Launch, T, kEven>(p, stream) : by_vectors<Launch, T, kOdd>(p, stream);
}
template <template <typename, int, int> class Launch>
hipError_t by_type(const NormParams &p, hipStream_t stream)
{
    if (p.type == AXC_F32)
        return by_width<Launch, float>(p, stream);
    if (p.type == AXC_BF16)
        return by_width<Launch, bf16>(p, stream);
    return by_width<Launch, f16>(p, stream);
}

template <typename T, int NV, int W>
struct Forward {
    static hipError_t go(const NormParams &p, int threads, hipStream_t stream)
    {
        int bytes = 0;
        void (*kernel)(NormParams);
        if constexpr (NV == 8) {
            threads = 512;
            kernel = wide_norm_kernel<T>;
        } else {
            bytes = Kept<W, NV, 4>::bytes(threads);
            kernel = norm_kernel<T, NV, W>;
            if (hipError_t e = set_max_dynamic_lds_once(reinterpret_cast<const void *>(kernel), bytes))
                return e;
        }
        // As many workgroups as are resident, each with its vectors in LDS and a row loaded ahead (rows of 8192 bfloat16, 33.6 M values:
        // 51 us by as many as have room for their threads alone, whose last begin when the others have ended, 45 this way).
        int64_t blocks = p.rows;
        if (blocks > device_cus()) {
            int a_cu = 0;
            if (hipError_t e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&a_cu, kernel, threads, bytes))
                return e;
            blocks = std::min<int64_t>({p.rows, kRangePairs, (int64_t)device_cus() * a_cu});   // (a pair of the range each)
        }
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(threads), bytes, stream, p);
        return hipGetLastError();
    }
};
size_t run_bytes(const NormParams &p)    // what the runs leave
{
    return ((size_t)norm_runs(p.rows, p.gate_groups).blocks * kSums * (size_t)p.width * sizeof(float) + 255) & ~(size_t)255;
}
template <typename T>
hipError_t column_sums(const NormParams &p, const NormRuns &runs, hipStream_t stream)
{
    ColumnSums sums = {{p.dweight, p.dbias, p.dscale, p.dpost, runs.per_group ? p.dgate : nullptr}};
    const unsigned ys = (unsigned)(kSumGate + (sums.out[kSumGate] ? p.gate_groups : 0));
    hipLaunchKernelGGL(norm_column_kernel<T>, dim3((unsigned)((p.width + 63) / 64), ys), dim3(512), 0, stream, p.partials, p.width,
                       runs, sums, p.vector_type);
    return hipGetLastError();
}
template <typename T, int NV, int W>
struct Backward {
    static hipError_t go(const NormParams &p, int threads, hipStream_t stream)
    {
        const NormRuns runs = norm_runs(p.rows, p.gate_groups);
        if constexpr (NV <= 2) {
            const int bytes = Kept<W, NV, 3>::bytes(threads);
            if (hipError_t e = set_max_dynamic_lds_once(reinterpret_cast<const void *>(&norm_grad_kernel<T, NV, W>), bytes))
                return e;
            hipLaunchKernelGGL((norm_grad_kernel<T, NV, W>), dim3((unsigned)runs.blocks), dim3(threads), bytes, stream, p, runs);
        } else {
            RowStats *const stats = reinterpret_cast<RowStats *>(reinterpret_cast<char *>(p.partials) + run_bytes(p));
            hipLaunchKernelGGL(wide_stats_kernel<T>, dim3((unsigned)(p.rows < 1024 ? p.rows : 1024)), dim3(512), 0, stream, p, stats);
            if (hipError_t e = hipGetLastError())
                return e;
            hipLaunchKernelGGL(wide_grad_kernel<T>, dim3((unsigned)((p.width + 1023) / 1024), (unsigned)runs.blocks), dim3(256), 0, stream,
                               p, runs, stats);
        }
        if (hipError_t e = hipGetLastError())
            return e;
        return column_sums<T>(p, runs, stream);
    }
};

} // namespace

hipError_t launch_norm(const NormParams &p, hipStream_t stream) { return by_type<Forward>(p, stream); }

size_t norm_partial_bytes(const NormParams &p)
{
    return run_bytes(p) + (p.width > kWideBackward ? (size_t)p.rows * sizeof(RowStats) : 0);
}

hipError_t launch_norm_gradients(const NormParams &p, hipStream_t stream) { return by_type<Backward>(p, stream); }

} // namespace axc
