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

// Sums of N values over a workgroup, in every thread.
template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float (*red)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] = wave_sum(v[i]);
    const int waves = blockDim.x / 64;
    if (waves == 1)
        return;
    __syncthreads();   // `red` is no longer read
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i)
            red[threadIdx.x / 64][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i)
        v[i] = 0.0f;
    for (int w = 0; w < waves; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] += red[w][i];
}

// A row in registers: NV vectors of V values a thread, vector j of thread t at (j * threads + t) * V.
template <int V, int NV>
struct Row {
    float v[NV][V];
};
template <int V>
__device__ __forceinline__ int place(int j) { return (j * (int)blockDim.x + (int)threadIdx.x) * V; }

template <typename T, int V, int NV>
__device__ __forceinline__ void load_row(const T *p, int width, Row<V, NV> &r)
{
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = place<V>(j);
        if (c < width)
            load_values<T, V>(p + c, V, V > 1, 0.0f, r.v[j]);
        else
#pragma unroll
            for (int i = 0; i < V; ++i)
                r.v[j][i] = 0.0f;
    }
}
template <typename T, int V, int NV>
__device__ __forceinline__ void store_row(T *p, int width, const Row<V, NV> &r)
{
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = place<V>(j);
        if (c < width)
            store_values<T, V>(p + c, V, V > 1, r.v[j]);
    }
}
// A vector of the layer (weights and the like), by columns as the row has them.
template <int V>
__device__ __forceinline__ void load_vector(const void *p, int type, int c, float (&v)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i)
        v[i] = load_any(p, c + i, type);
}

// r becomes (v - mean) / sqrt(var + eps) (mean 0 for RMS); returns the reciprocal of the root.
template <int V, int NV>
__device__ __forceinline__ float normalize(Row<V, NV> &r, int width, int layer, float eps, float (*red)[2])
{
    float s[2] = {};
    if (layer) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i)
                s[0] += r.v[j][i];
        block_sums<2>(s, red);
        const float mean = s[0] / (float)width;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (place<V>(j) < width)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    r.v[j][i] -= mean;
    }
    s[0] = s[1] = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
            s[0] = fmaf(r.v[j][i], r.v[j][i], s[0]);
    block_sums<2>(s, red);
    const float rs = 1.0f / sqrtf(s[0] / (float)width + eps);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
            r.v[j][i] *= rs;
    return rs;
}

template <typename T, int V, int NV>
__global__ void __launch_bounds__(NV * V > 16 ? 1024 : 512) norm_kernel(NormParams p)
{
    __shared__ float red[kMaxWaves][2];
    __shared__ float ends[2 * kMaxWaves];
    const int width = (int)p.width;
    const int64_t group_rows = p.gate_groups ? p.rows / p.gate_groups : 1;
    float lo = INFINITY, hi = -INFINITY;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        Row<V, NV> h;
        load_row<T, V, NV>(static_cast<const T *>(p.x) + r * width, width, h);
        if (p.block) {
            Row<V, NV> u;
            load_row<T, V, NV>(static_cast<const T *>(p.block) + r * width, width, u);
            if (p.post_weight)
                normalize<V, NV>(u, width, p.layer, p.eps, red);
            const T *const gate = p.gate ? static_cast<const T *>(p.gate) + r / group_rows * width : nullptr;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = place<V>(j);
                if (c >= width)
                    continue;
                float w[V];
                if (p.post_weight) {
                    load_vector<V>(p.post_weight, p.vector_type, c, w);
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        u.v[j][i] *= w[i];
                }
                if (gate) {
                    load_values<T, V>(gate + c, V, V > 1, 0.0f, w);
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        u.v[j][i] *= w[i];
                }
                if (p.scale) {
                    load_vector<V>(p.scale, p.vector_type, c, w);
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        u.v[j][i] *= w[i];
                }
#pragma unroll
                for (int i = 0; i < V; ++i)
                    h.v[j][i] = (float)(T)(h.v[j][i] + u.v[j][i]);
            }
            store_row<T, V, NV>(static_cast<T *>(p.h) + r * width, width, h);
        }
        normalize<V, NV>(h, width, p.layer, p.eps, red);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = place<V>(j);
            if (c >= width)
                continue;
            float w[V];
            load_vector<V>(p.weight, p.vector_type, c, w);
#pragma unroll
            for (int i = 0; i < V; ++i)
                h.v[j][i] *= w[i];
            if (p.bias) {
                load_vector<V>(p.bias, p.vector_type, c, w);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    h.v[j][i] += w[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h.v[j][i] = (float)(T)h.v[j][i];
                lo = fminf(lo, h.v[j][i]);
                hi = fmaxf(hi, h.v[j][i]);
            }
        }
        store_row<T, V, NV>(static_cast<T *>(p.y) + r * width, width, h);
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
//   norm(v) = n: dv = (g - n mean(g n) [- mean(g)]) / root, g the gradient of n
// A workgroup takes a run of neighbouring rows, all of one gate group or whole groups, and keeps the sums over rows (for the
// weights, the bias, the scale, the gate) in registers, a column in the same thread throughout; column_kernel adds up what the
// runs leave, in one order.
struct NormRuns {
    int64_t run;            // rows of a workgroup
    int64_t per_group;      // workgroups of a gate group; 0: a workgroup takes whole groups, or there is no gate
    int64_t blocks;
};
NormRuns norm_runs(int64_t rows, int64_t groups)
{
    // about 512 workgroups, two a CU, each with its own partial sums
    NormRuns n = {};
    n.run = (rows + 511) / 512;
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

template <typename T, int V, int NV>
__global__ void __launch_bounds__(NV * V > 16 ? 1024 : 512) norm_grad_kernel(NormParams p, NormRuns runs)
{
    __shared__ float red[kMaxWaves][2];
    const int width = (int)p.width;
    const int64_t group_rows = p.gate_groups ? p.rows / p.gate_groups : 1;
    int64_t first, last;
    if (runs.per_group) {
        const int64_t group = blockIdx.x / runs.per_group, part = blockIdx.x - group * runs.per_group;
        first = group * group_rows + part * runs.run;
        last = first + runs.run < (group + 1) * group_rows ? first + runs.run : (group + 1) * group_rows;
    } else {
        first = (int64_t)blockIdx.x * runs.run;
        last = first + runs.run < p.rows ? first + runs.run : p.rows;
    }
    Row<V, NV> sw = {}, sb = {}, ss = {}, sp = {}, sg = {};
    for (int64_t r = first; r < last; ++r) {
        Row<V, NV> n, dh;
        load_row<T, V, NV>(static_cast<const T *>(p.h) + r * width, width, n);
        if (p.grad_y) {
            load_row<T, V, NV>(static_cast<const T *>(p.grad_y) + r * width, width, dh);
            const float rs = normalize<V, NV>(n, width, p.layer, p.eps, red);
            float s[2] = {};
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = place<V>(j);
                if (c >= width)
                    continue;
                float w[V];
                load_vector<V>(p.weight, p.vector_type, c, w);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    sw.v[j][i] = fmaf(dh.v[j][i], n.v[j][i], sw.v[j][i]);
                    sb.v[j][i] += dh.v[j][i];
                    dh.v[j][i] *= w[i];
                    s[0] = fmaf(dh.v[j][i], n.v[j][i], s[0]);
                    s[1] += dh.v[j][i];
                }
            }
            block_sums<2>(s, red);
            const float mgn = s[0] / (float)width, mg = p.layer ? s[1] / (float)width : 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    dh.v[j][i] = (dh.v[j][i] - n.v[j][i] * mgn - mg) * rs;
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    dh.v[j][i] = 0.0f;
        }
        if (p.grad_h) {
            Row<V, NV> g;
            load_row<T, V, NV>(static_cast<const T *>(p.grad_h) + r * width, width, g);
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    dh.v[j][i] += g.v[j][i];
        }
        store_row<T, V, NV>(static_cast<T *>(p.dx) + r * width, width, dh);
        if (!p.block)
            continue;
        // du = dh scale gate; n is the block, normed where it is
        load_row<T, V, NV>(static_cast<const T *>(p.block) + r * width, width, n);
        float rs = 1.0f;
        if (p.post_weight)
            rs = normalize<V, NV>(n, width, p.layer, p.eps, red);
        const int64_t group = r / group_rows;
        const T *const gate = p.gate ? static_cast<const T *>(p.gate) + group * width : nullptr;
        float s[2] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = place<V>(j);
            if (c >= width)
                continue;
            float w[V], sc[V], ga[V];
#pragma unroll
            for (int i = 0; i < V; ++i)
                w[i] = sc[i] = ga[i] = 1.0f;
            if (p.post_weight)
                load_vector<V>(p.post_weight, p.vector_type, c, w);
            if (p.scale)
                load_vector<V>(p.scale, p.vector_type, c, sc);
            if (gate)
                load_values<T, V>(gate + c, V, V > 1, 0.0f, ga);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float hu = dh.v[j][i] * n.v[j][i] * w[i];   // dh u
                ss.v[j][i] = fmaf(hu, ga[i], ss.v[j][i]);
                sg.v[j][i] = fmaf(hu, sc[i], sg.v[j][i]);
                const float du = dh.v[j][i] * sc[i] * ga[i];
                sp.v[j][i] = fmaf(du, n.v[j][i], sp.v[j][i]);
                dh.v[j][i] = du * w[i];
                s[0] = fmaf(dh.v[j][i], n.v[j][i], s[0]);
                s[1] += dh.v[j][i];
            }
        }
        if (p.post_weight) {
            block_sums<2>(s, red);
            const float mgn = s[0] / (float)width, mg = p.layer ? s[1] / (float)width : 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    dh.v[j][i] = (dh.v[j][i] - n.v[j][i] * mgn - mg) * rs;
        }
        store_row<T, V, NV>(static_cast<T *>(p.dblock) + r * width, width, dh);
        if (p.dgate && !runs.per_group && (r + 1) % group_rows == 0) {   // the group's last row
            store_row<T, V, NV>(static_cast<T *>(p.dgate) + group * width, width, sg);
            sg = {};
        }
    }
    float *const to = p.partials + (int64_t)blockIdx.x * kSums * width;
    const bool want[kSums] = {p.dweight != nullptr, p.dbias != nullptr, p.dscale != nullptr, p.dpost != nullptr,
                              p.dgate != nullptr && runs.per_group != 0};
    const Row<V, NV> *const from[kSums] = {&sw, &sb, &ss, &sp, &sg};
#pragma unroll
    for (int k = 0; k < kSums; ++k)
        if (want[k])
            store_row<float, V, NV>(to + (int64_t)k * width, width, *from[k]);
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

// Rows in vectors of four where every row begins aligned, value by value where not; as many threads as have about two vectors
// each, in steps of a wavefront.
bool whole_vectors(const NormParams &p)
{
    const uintptr_t mask = (uintptr_t)(4 * type_bytes(p.type) - 1);
    if (p.width & 3)
        return false;
    for (const void *q : {p.x, p.block, p.gate, (const void *)p.h, (const void *)p.y, p.grad_h, p.grad_y, (const void *)p.dx,
                          (const void *)p.dblock, (const void *)p.dgate})
        if ((uintptr_t)q & mask)
            return false;
    return true;
}

template <template <typename, int, int> class Launch, typename T>
hipError_t by_width(const NormParams &p, hipStream_t stream)
{
    const bool whole = whole_vectors(p);
    const int64_t vectors = whole ? p.width / 4 : p.width;
    auto threads = [&](int nv, int most) {
        const int64_t t = ((vectors + nv - 1) / nv + 63) / 64 * 64;
        return (int)(t > most ? most : t);
    };
    if (whole) {
        if (vectors <= 512)
            return Launch<T, 4, 1>::go(p, threads(1, 512), stream);
        if (vectors <= 1024)
            return Launch<T, 4, 2>::go(p, threads(2, 512), stream);
        if (vectors <= 2048)
            return Launch<T, 4, 4>::go(p, threads(4, 512), stream);
        return Launch<T, 4, 8>::go(p, 1024, stream);
    }
    if (vectors <= 1024)
        return Launch<T, 1, 2>::go(p, threads(2, 512), stream);
    if (vectors <= 4096)
        return Launch<T, 1, 8>::go(p, threads(8, 512), stream);
    if (vectors <= 8192)
        return Launch<T, 1, 16>::go(p, 512, stream);
    return Launch<T, 1, 32>::go(p, 1024, stream);
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

template <typename T, int V, int NV>
struct Forward {
    static hipError_t go(const NormParams &p, int threads, hipStream_t stream)
    {
        const int64_t blocks = p.rows < kRangePairs ? p.rows : kRangePairs;
        hipLaunchKernelGGL((norm_kernel<T, V, NV>), dim3((unsigned)blocks), dim3(threads), 0, stream, p);
        return hipGetLastError();
    }
};
template <typename T, int V, int NV>
struct Backward {
    static hipError_t go(const NormParams &p, int threads, hipStream_t stream)
    {
        const NormRuns runs = norm_runs(p.rows, p.gate_groups);
        hipLaunchKernelGGL((norm_grad_kernel<T, V, NV>), dim3((unsigned)runs.blocks), dim3(threads), 0, stream, p, runs);
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
