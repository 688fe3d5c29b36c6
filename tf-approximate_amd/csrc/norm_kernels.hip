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
// included.  A vector behind the row is loaded from the row's last four values and counts as zeros; the one that ends behind the
// row is loaded from there too, and moved.  So that rows of less than four values need no more than that, they take the place of
// the last four values of whatever is loaded one by one (kTiny).
enum { kEven, kOdd, kTiny };             // widths: a multiple of four, no multiple, less than four
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
    if constexpr (W == kEven) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[i] = c < width ? (float)t[i] : 0.0f;
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

template <int NV>
struct Row {
    float v[NV][V];
};
template <typename T, int NV>
struct Raw {               // a row as it was loaded
    typename Vector<T>::four v[NV];
};
template <int W, typename T, int NV>
__device__ __forceinline__ void load_row(const T *p, int width, Raw<T, NV> &r)
{
#pragma unroll
    for (int j = 0; j < NV; ++j)
        r.v[j] = load_four<W>(p, place(j), width);
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
__device__ __forceinline__ void store_row(T *p, int width, const Row<NV> &r)
{
#pragma unroll
    for (int j = 0; j < NV; ++j)
        store_four<W>(p, place(j), width, r.v[j]);
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
        if (type == AXC_F32)
            return in_place<W>(load_four<W>(static_cast<const float *>(p), c, width), c, width);
        if (type == AXC_BF16)
            return in_place<W>(load_four<W>(static_cast<const bf16 *>(p), c, width), c, width);
        return in_place<W>(load_four<W>(static_cast<const f16 *>(p), c, width), c, width);
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
    const T *const x = static_cast<const T *>(p.x);
    const T *const block = static_cast<const T *>(p.block ? p.block : p.x);   // (loaded in any case, for nothing without a block)
    const T *const gate = static_cast<const T *>(p.gate);
    float lo = INFINITY, hi = -INFINITY;
    // the gate group of the row that is loaded, and the row's place in it; a step of the loop further on
    int64_t group = (int64_t)blockIdx.x / group_rows, in_group = (int64_t)blockIdx.x - group * group_rows;
    const int64_t more_groups = (int64_t)gridDim.x / group_rows, more_rows = (int64_t)gridDim.x - more_groups * group_rows;
    Raw<T, NV> xr, br, gr = {};
    auto load = [&](int64_t r) {
        load_row<W>(x + r * width, width, xr);
        load_row<W>(block + r * width, width, br);
        if (gate)
            load_row<W>(gate + group * width, width, gr);
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
                if (gate) {
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
            store_row<W>(static_cast<T *>(p.h) + r * width, width, h);
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
        store_row<W>(static_cast<T *>(p.y) + r * width, width, h);
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
constexpr int64_t kRunBlocks = 1024;     // about as many workgroups, four a CU
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
    // (what is not there is loaded from h, for nothing, and counts as zeros, a gate as ones)
    const T *const hs = static_cast<const T *>(p.h);
    const T *const gys = p.grad_y ? static_cast<const T *>(p.grad_y) : hs, *const ghs = p.grad_h ? static_cast<const T *>(p.grad_h) : hs;
    const T *const blocks = p.block ? static_cast<const T *>(p.block) : hs, *const gates = static_cast<const T *>(p.gate);
    Raw<T, NV> hr, gyr, ghr, br, gr = {};
    auto load = [&](int64_t r, int64_t of) {
        load_row<W>(hs + r * width, width, hr);
        load_row<W>(gys + r * width, width, gyr);
        load_row<W>(ghs + r * width, width, ghr);
        load_row<W>(blocks + r * width, width, br);
        if (gates)
            load_row<W>(gates + of * width, width, gr);
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
        scale_row(dh, p.grad_y ? 1.0f : 0.0f);
        scale_row(gh, p.grad_h ? 1.0f : 0.0f);
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
        store_row<W>(static_cast<T *>(p.dx) + r * width, width, dh);
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
            if (gates)
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
        store_row<W>(static_cast<T *>(p.dblock) + r * width, width, dh);
        if (p.dgate && !runs.per_group && ends) {
            store_row<W>(static_cast<T *>(p.dgate) + of * width, width, sg);
            sg = {};
        }
    }
    float *const to = p.partials + (int64_t)blockIdx.x * kSums * width;
    if (p.dweight)
        store_row<W>(to + (int64_t)kSumWeight * width, width, sw);
    if (p.dbias)
        store_row<W>(to + (int64_t)kSumBias * width, width, sb);
    if (p.dscale)
        store_row<W>(to + (int64_t)kSumScale * width, width, ss);
    if (p.dpost)
        store_row<W>(to + (int64_t)kSumPost * width, width, sp);
    if (p.dgate && runs.per_group)
        store_row<W>(to + (int64_t)kSumGate * width, width, sg);
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
    return p.width % V ? by_vectors<Launch, T, kOdd>(p, stream) : by_vectors<Launch, T, kEven>(p, stream);
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
