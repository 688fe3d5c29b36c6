// Softmax cross entropy over a vocabulary whose logits are sums of table entries, a piece of the vocabulary at a time.
//
//   loss[m] = log sum_v exp(z[m][v]) - z[m][target[m]] = (t - z[m][target[m]]) + log s
//
// A chunk of columns leaves its largest logit t and s = sum exp(z - t), in float32; two of them make max(t, t') and
// s exp(t - max) + s' exp(t' - max).  t and log s stay apart to the end: what all of a row's logits have in common, however much, has no
// part in the loss or in a probability exp((z - t) - log s).  Chunks whose logits are all -infinity have t = -infinity and s = 0.
#include "layers_internal.h"

namespace axc {
namespace {

struct Exponentials {
    float top, sum;
    __device__ __forceinline__ Exponentials() : top(-INFINITY), sum(0.0f) {}
    __device__ __forceinline__ void join(float t, float s)
    {
        const float m = fmaxf(top, t);
        // (equal maxima, infinite ones among them, need no factor: infinity minus itself is NaN)
        sum = (top == m ? sum : sum * __expf(top - m)) + (t == m ? s : s * __expf(t - m));
        top = m;
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&z)[N])
    {
        float m = top;
#pragma unroll
        for (int j = 0; j < N; ++j)
            m = fmaxf(m, z[j]);
        if (fabsf(m) < INFINITY) {       // (a NaN, over which fmaxf has passed, is in the sum then)
            float s = sum * __expf(top - m);
#pragma unroll
            for (int j = 0; j < N; ++j)
                s += __expf(z[j] - m);
            sum = s;
            top = m;
        } else {                         // nothing but -infinity yet, or an infinite one
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (z[j] > -INFINITY)
                    join(z[j], 1.0f);
                else if (z[j] != z[j])
                    sum = z[j];
            }
        }
    }
};

// Sums by rows: a workgroup a row and kRowChunk columns, four neighbours a thread.
constexpr int kRowChunk = 2048;
template <typename I>
__global__ void __launch_bounds__(256) loss_piece_kernel(TableSums s, int64_t first_row, int64_t rows, int columns,
                                                         int64_t first_column, const void *bias, int bias_type,
                                                         const int64_t *__restrict__ targets, int chunk, LossState st)
{
    __shared__ float tops[4], sums[4];
    const int64_t r = blockIdx.x;
    const float scale = __fmul_rn(s.grids->in.scale, s.grids->kernel.scale);
    const Bracket<I> b(s);
    const I row = b.row(s.row_sums[r]);
    const int64_t target = targets[first_row + r] - first_column;
    Exponentials e;
#pragma unroll
    for (int i = 0; i < kRowChunk / 1024; ++i) {
        const int c = (int)blockIdx.y * kRowChunk + i * 1024 + 4 * (int)threadIdx.x;
        if (c >= columns)
            continue;
        const i32x4 t = four_sums(s.raw, r, c);
        float z[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            z[j] = -INFINITY;
            if (c + j < columns) {
                z[j] = __fmul_rn(Bracket<I>::value(t[j], row, b.column(s.column_sums[c + j])), scale);
                if (bias)
                    z[j] = __fadd_rn(z[j], load_any(bias, c + j, bias_type));
                if (c + j == target)
                    st.at[first_row + r] = z[j];
            }
        }
        e.add(z);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const float t = __shfl_xor(e.top, d), q = __shfl_xor(e.sum, d);
        e.join(t, q);
    }
    if ((threadIdx.x & 63) == 0) {
        tops[threadIdx.x / 64] = e.top;
        sums[threadIdx.x / 64] = e.sum;
    }
    __syncthreads();
    if (threadIdx.x != 0)
        return;
    for (int i = 1; i < 4; ++i)
        e.join(tops[i], sums[i]);
    st.parts[(chunk + blockIdx.y) * rows + first_row + r] = make_float2(e.top, e.sum);
}

// Turned sums: a workgroup 64 rows, a lane each, and `size` columns, a quarter for each wavefront.  A lane goes through its row's
// logits by itself; what belongs to a column is the same for all lanes.
template <typename I>
__global__ void __launch_bounds__(256) loss_turned_kernel(TableSums s, int64_t first_row, int64_t run_rows, int64_t rows, int columns,
                                                          int64_t first_column, const void *bias, int bias_type,
                                                          const int64_t *__restrict__ targets, int chunk, int size, LossState st)
{
    constexpr int N = 8;
    __shared__ float tops[4][64], sums[4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t at = (int64_t)blockIdx.y * 64 + lane;
    const int64_t r = at < run_rows ? at : run_rows - 1;   // (lanes behind the rows repeat the last; nobody stores them)
    const float scale = __fmul_rn(s.grids->in.scale, s.grids->kernel.scale);
    const Bracket<I> b(s);
    const I row = b.row(s.row_sums[r]);
    const int64_t target = targets[first_row + r] - first_column;
    const int c0 = (int)blockIdx.x * size + wave * (size / 4);
    const int end = c0 + size / 4 < columns ? c0 + size / 4 : columns;
    Exponentials e;
    for (int c = c0; c < end; c += N) {
        int32_t t[N] = {};
        for (int k = 0; k < s.raw.splits; ++k)
#pragma unroll
            for (int j = 0; j < N; ++j)
                t[j] += s.raw.acc[k * s.raw.split_stride + (int64_t)(c + j < end ? c + j : end - 1) * s.raw.pitch + r];
        float z[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int of = c + j < end ? c + j : end - 1;
            z[j] = __fmul_rn(Bracket<I>::value(t[j], row, b.column(s.column_sums[of])), scale);
            if (bias)
                z[j] = __fadd_rn(z[j], load_any(bias, of, bias_type));
            if (of == target)
                st.at[first_row + r] = z[j];
            z[j] = c + j < end ? z[j] : -INFINITY;
        }
        e.add(z);
    }
    tops[wave][lane] = e.top;
    sums[wave][lane] = e.sum;
    __syncthreads();
    if (wave != 0 || at >= run_rows)
        return;
    for (int i = 1; i < 4; ++i)
        e.join(tops[i][lane], sums[i][lane]);
    st.parts[(chunk + blockIdx.x) * rows + first_row + at] = make_float2(e.top, e.sum);
}

// 64 rows a workgroup, over what the chunks have left: a row a lane, every eighth chunk a wavefront.
constexpr int kRowWaves = 8;
__global__ void __launch_bounds__(64 * kRowWaves) loss_rows_kernel(LossState st, const int64_t *__restrict__ targets, int64_t ignore,
                                                                   int64_t V, int64_t first_row, int64_t run_rows, int64_t rows,
                                                                   int chunks)
{
    __shared__ float2 ends[kRowWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
    const int64_t i = (int64_t)blockIdx.x * 64 + lane, r = first_row + i;
    Exponentials e;
    if (i < run_rows)
#pragma unroll 4
        for (int c = wave; c < chunks; c += kRowWaves) {
            const float2 p = st.parts[c * rows + r];
            e.join(p.x, p.y);
        }
    ends[wave][lane] = make_float2(e.top, e.sum);
    __syncthreads();
    if (wave != 0 || i >= run_rows)
        return;
    for (int w = 1; w < kRowWaves; ++w)
        e.join(ends[w][lane].x, ends[w][lane].y);
    const float log_sum = logf(e.sum);
    const int64_t t = targets[r];
    st.top[r] = e.top;
    st.log_sum[r] = log_sum;
    // a target that is no column of the vocabulary has no loss
    st.rows[r] = t == ignore ? 0.0f : t >= 0 && t < V ? (e.top - st.at[r]) + log_sum : NAN;
}

// The loss out of the rows', in one order, and what each row's gradient is multiplied by.
__global__ void __launch_bounds__(1024) loss_out_kernel(LossState st, const int64_t *targets, int64_t ignore, int64_t V, int64_t rows,
                                                        int reduction, const float *grad_loss, float *loss, int gradients)
{
    __shared__ double part[16];
    __shared__ int64_t counts[16];
    double sum = 0.0;
    int64_t count = 0;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) {
        sum += (double)st.rows[r];
        count += targets[r] != ignore ? 1 : 0;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        sum += __shfl_xor(sum, d);
        count += __shfl_xor(count, d);
    }
    if ((threadIdx.x & 63) == 0) {
        part[threadIdx.x / 64] = sum;
        counts[threadIdx.x / 64] = count;
    }
    __syncthreads();
    sum = 0.0;
    count = 0;
    for (int i = 0; i < 16; ++i) {
        sum += part[i];
        count += counts[i];
    }
    if (reduction == AXC_LOSS_MEAN && count > 0)
        sum /= (double)count;
    if (reduction == AXC_LOSS_NONE) {
        for (int64_t r = threadIdx.x; r < rows; r += 1024)
            loss[r] = st.rows[r];
    } else if (threadIdx.x == 0) {
        loss[0] = (float)sum;
    }
    if (!gradients)
        return;
    // What all rows have in common goes behind the products: multiplied into softmax minus one-hot ahead of a rounding to terms of
    // bfloat16 it would round every row's largest part, minus the factor, off by the same amount.  What is each row's own stays
    // in front, and so does what is not finite: behind, rows that do not count would be 0 times infinity.
    float factor = reduction == AXC_LOSS_MEAN ? 1.0f / (float)(count > 0 ? count : 1) : 1.0f;
    bool own = reduction == AXC_LOSS_NONE;
    if (grad_loss && !own) {
        own = !(fabsf(grad_loss[0]) < INFINITY);
        factor *= own ? 1.0f : grad_loss[0];
    }
    if (threadIdx.x == 0)
        *st.factor = factor;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) {
        const float of = grad_loss ? grad_loss[reduction == AXC_LOSS_NONE ? r : 0] : 1.0f;
        const int64_t t = targets[r];
        st.coefficient[r] = t == ignore || of == 0.0f ? 0.0f : t >= 0 && t < V ? (own ? of : 1.0f) : NAN;
    }
}

} // namespace

hipError_t launch_loss_piece(const TableSums &s, int64_t first_row, int64_t run_rows, int64_t rows, int columns, int64_t first_column,
                             const void *bias, int bias_type, const int64_t *targets, int chunk, int *chunks, const LossState &st,
                             hipStream_t stream)
{
    const bool narrow = s.K <= kNarrowDepth;
    if (s.raw.turned) {
        const int size = loss_chunk(rows);
        *chunks = (columns + size - 1) / size;
        const dim3 grid((unsigned)*chunks, (unsigned)((run_rows + 63) / 64));
        if (narrow)
            hipLaunchKernelGGL(loss_turned_kernel<uint32_t>, grid, dim3(256), 0, stream, s, first_row, run_rows, rows, columns,
                               first_column, bias, bias_type, targets, chunk, size, st);
        else
            hipLaunchKernelGGL(loss_turned_kernel<int64_t>, grid, dim3(256), 0, stream, s, first_row, run_rows, rows, columns,
                               first_column, bias, bias_type, targets, chunk, size, st);
    } else {
        *chunks = (columns + kRowChunk - 1) / kRowChunk;
        const dim3 grid((unsigned)run_rows, (unsigned)*chunks);
        if (narrow)
            hipLaunchKernelGGL(loss_piece_kernel<uint32_t>, grid, dim3(256), 0, stream, s, first_row, rows, columns, first_column, bias,
                               bias_type, targets, chunk, st);
        else
            hipLaunchKernelGGL(loss_piece_kernel<int64_t>, grid, dim3(256), 0, stream, s, first_row, rows, columns, first_column, bias,
                               bias_type, targets, chunk, st);
    }
    return hipGetLastError();
}

hipError_t launch_loss_rows(const LossState &st, const int64_t *targets, int64_t ignore, int64_t V, int64_t first_row, int64_t run_rows,
                            int64_t rows, int chunks, hipStream_t stream)
{
    hipLaunchKernelGGL(loss_rows_kernel, dim3((unsigned)((run_rows + 63) / 64)), dim3(64 * kRowWaves), 0, stream, st, targets, ignore, V, first_row,
                       run_rows, rows, chunks);
    return hipGetLastError();
}

hipError_t launch_loss_out(const LossState &st, const int64_t *targets, int64_t ignore, int64_t V, int64_t rows, int reduction,
                           const float *grad_loss, float *loss, bool gradients, hipStream_t stream)
{
    hipLaunchKernelGGL(loss_out_kernel, dim3(1), dim3(1024), 0, stream, st, targets, ignore, V, rows, reduction, grad_loss, loss,
                       (int)gradients);
    return hipGetLastError();
}

} // namespace axc
