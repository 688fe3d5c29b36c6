// Norms before and after a block of a residual network, with the block's gate and scale:
//
//   u = norm(block) post_weight (or block itself),  h = x + scale gate u,  y = norm(h) weight + bias
//   norm(v) = v / sqrt(mean(v^2) + eps), or (v - mean(v)) / sqrt(var(v) + eps)
//
// h is rounded to the tensors' type before it is normed, so that what the backward pass reads is what was normed.  A workgroup
// takes a row at a time and keeps it in registers: everything is read once and written once, which is what bounds these kernels.
// Statistics are float32, of the row as it stands in registers: the variance from the differences to the mean.
#include "layers_internal.h"

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

// The layer's vectors (weights and the like), as floats in LDS: each thread its own columns, so without a barrier.  Rows of eight
// vectors a thread have more of them than LDS holds, and load them again for every row.
template <int W, int NV, int N>
struct Kept {
    f32x4 *lds;
    const void *vectors[N];
    int type, width;
    static constexpr bool kKeep = NV <= 4;
    static int bytes(int threads) { return kKeep ? N * threads * NV * V * (int)sizeof(float) : 0; }
    __device__ __forceinline__ f32x4 load(int which, int j) const
    {
        const void *const p = vectors[which];
        const int c = place(j);
        constexpr int L = W == kTiny ? kTiny : kOdd;   // (may be aligned as their elements only)
        if (type == AXC_F32)
            return in_place<L>(load_four<L>(static_cast<const float *>(p), c, width), c, width);
        if (type == AXC_BF16)
            return in_place<L>(load_four<L>(static_cast<const bf16 *>(p), c, width), c, width);
        return in_place<L>(load_four<L>(static_cast<const f16 *>(p), c, width), c, width);
    }
    // Vectors that are not there are ones.
    __device__ __forceinline__ void fill()
    {
        if constexpr (!kKeep)
            return;
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int j = 0; j < NV; ++j)
                lds[(k * NV + j) * (int)blockDim.x + (int)threadIdx.x] = vectors[k] ? load(k, j) : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
    }
    __device__ __forceinline__ f32x4 get(int which, int j) const
    {
        if constexpr (kKeep)
            return lds[(which * NV + j) * (int)blockDim.x + (int)threadIdx.x];
        return vectors[which] ? load(which, j) : f32x4{1.0f, 1.0f, 1.0f, 1.0f};
    }
};

// Threads of a workgroup at most, by the vectors of a thread: 1024 threads have 128 registers each.
constexpr int most_threads(int NV) { return NV > 4 ? 1024 : 512; }

enum { kWeight, kScale, kPost, kBias };

template <typename T, int NV, int W>
__global__ void __launch_bounds__(most_threads(NV)) norm_kernel(NormParams p)
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
    if (!p.range)
        return;
    block_range(lo, hi, ends);
    if (threadIdx.x == 0)
        reinterpret_cast<float2 *>(p.range)[blockIdx.x] = make_float2(lo, hi);
    if (blockIdx.x == 0)   // pairs that nobody has
        for (int i = (int)gridDim.x + (int)threadIdx.x; i < kRangePairs; i += blockDim.x)
            reinterpret_cast<float2 *>(p.range)[i] = make_float2(INFINITY, -INFINITY);
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

template <typename T, int NV, int W>
__global__ void __launch_bounds__(most_threads(NV)) norm_grad_kernel(NormParams p, NormRuns runs)
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
    constexpr bool kAhead = NV <= 2;   // the next row's loads ahead of all reductions; of wider rows once registers are free
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
        if (kAhead && r + 1 < last)
            load(r + 1, group);
        if constexpr (W != kEven) {
            scale_row(dh, p.grad_y ? 1.0f : 0.0f);
            if (!p.grad_h)
                gh = {};
        }
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
        if (!kAhead && r + 1 < last)
            load(r + 1, group);
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

// Two vectors a thread up to 4096 values, in steps of a wavefront; then four, and eight of 1024 threads.
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
        // as many workgroups as are resident, each with its vectors in LDS, a row loaded ahead
        int64_t blocks = 256 * 2048 / threads;
        blocks = blocks < kRangePairs ? blocks : kRangePairs;   // a pair of the range each
        blocks = blocks < p.rows ? blocks : p.rows;
        const int bytes = Kept<W, NV, 4>::bytes(threads);
        if (hipError_t e = set_max_dynamic_lds_once(reinterpret_cast<const void *>(&norm_kernel<T, NV, W>), bytes))
            return e;
        hipLaunchKernelGGL((norm_kernel<T, NV, W>), dim3((unsigned)blocks), dim3(threads), bytes, stream, p);
        return hipGetLastError();
    }
};
template <typename T, int NV, int W>
struct Backward {
    static hipError_t go(const NormParams &p, int threads, hipStream_t stream)
    {
        const NormRuns runs = norm_runs(p.rows, p.gate_groups);
        const int bytes = Kept<W, NV, 3>::bytes(threads);
        if (hipError_t e = set_max_dynamic_lds_once(reinterpret_cast<const void *>(&norm_grad_kernel<T, NV, W>), bytes))
            return e;
        hipLaunchKernelGGL((norm_grad_kernel<T, NV, W>), dim3((unsigned)runs.blocks), dim3(threads), bytes, stream, p, runs);
        if (hipError_t e = hipGetLastError())
            return e;
        ColumnSums sums = {{p.dweight, p.dbias, p.dscale, p.dpost, runs.per_group ? p.dgate : nullptr}};
        const unsigned ys = (unsigned)(kSumGate + (sums.out[kSumGate] ? p.gate_groups : 0));
        hipLaunchKernelGGL(norm_column_kernel<T>, dim3((unsigned)((p.width + 63) / 64), ys), dim3(512), 0, stream, p.partials,
                           p.width, runs, sums, p.vector_type);
        return hipGetLastError();
    }
};

} // namespace

hipError_t launch_norm(const NormParams &p, hipStream_t stream) { return by_type<Forward>(p, stream); }

size_t norm_partial_bytes(const NormParams &p)
{
    return (size_t)norm_runs(p.rows, p.gate_groups).blocks * kSums * (size_t)p.width * sizeof(float);
}

hipError_t launch_norm_gradients(const NormParams &p, hipStream_t stream) { return by_type<Backward>(p, stream); }

} // namespace axc
