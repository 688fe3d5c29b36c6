// Softmax cross entropy over a vocabulary whose logits are sums of table entries, a piece of the vocabulary at a time.
//
//   loss[m] = log sum_v exp(z[m][v]) - z[m][target[m]]
//
// Per row a running maximum t and sum s of exp(z - t), in float32: a piece with maximum p makes them max(t, p) and
// s exp(t - max) + its own sum.  A row whose logits so far are all -infinity has s = 0 and t = -infinity.
#include "layers_internal.h"

namespace axc {
namespace {

// (t, s) and (p, q) together
__device__ __forceinline__ void join(float &t, float &s, float p, float q)
{
    const float m = fmaxf(t, p);
    // (equal maxima, infinite ones among them, need no factor: infinity minus itself is NaN)
    s = (t == m ? s : s * expf(t - m)) + (p == m ? q : q * expf(p - m));
    t = m;
}

// A workgroup a row: the piece's logits out of the sums, four at a time, joined with what earlier pieces left.
__global__ void __launch_bounds__(1024) loss_piece_kernel(TableSums s, int columns, int64_t first_column, const void *bias,
                                                          int bias_type, const int64_t *targets, int64_t ignore, int64_t V,
                                                          int first, int last, LossState st)
{
    __shared__ float tops[16], sums[16];
    const int64_t r = blockIdx.x;
    const float scale = __fmul_rn(s.grids->in.scale, s.grids->kernel.scale);
    const int64_t zi = s.grids->in.zero, row = row_term(s, r);
    const int64_t target = targets[r];
    const int32_t *const acc = s.acc + r * s.pitch;
    float top = -INFINITY, sum = 0.0f;
    bool undefined = false;
    for (int c = 4 * threadIdx.x; c < columns; c += 4 * blockDim.x) {
        int32_t t[4] = {};
        for (int k = 0; k < s.splits; ++k) {
            const i32x4 a = *reinterpret_cast<const i32x4 *>(acc + k * s.split_stride + c);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                t[j] += a[j];
        }
        float z[4], most = top;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            z[j] = -INFINITY;
            if (c + j < columns) {
                z[j] = __fmul_rn((float)((int64_t)t[j] + row - zi * s.column_sums[c + j]), scale);
                if (bias)
                    z[j] = __fadd_rn(z[j], load_any(bias, c + j, bias_type));
                if (first_column + c + j == target)
                    st.at[r] = z[j];
                undefined |= z[j] != z[j];
            }
            most = fmaxf(most, z[j]);
        }
        if (most > -INFINITY) {
            sum = top == most ? sum : sum * expf(top - most);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                sum += z[j] == most ? 1.0f : expf(z[j] - most);
            top = most;
        }
    }
    if (undefined)
        sum = NAN;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const float p = __shfl_xor(top, d), q = __shfl_xor(sum, d);
        join(top, sum, p, q);
    }
    if ((threadIdx.x & 63) == 0) {
        tops[threadIdx.x / 64] = top;
        sums[threadIdx.x / 64] = sum;
    }
    __syncthreads();   // (and what the thread with the target has stored is there to be read)
    if (threadIdx.x != 0)
        return;
    top = first ? -INFINITY : st.top[r];
    sum = first ? 0.0f : st.sum[r];
    for (int i = 0; i < (int)blockDim.x / 64; ++i)
        join(top, sum, tops[i], sums[i]);
    st.top[r] = top;
    st.sum[r] = sum;
    if (last) {
        const float lse = top + logf(sum);
        st.lse[r] = lse;
        // a target that is no column of the vocabulary has no loss
        st.rows[r] = target == ignore ? 0.0f : target >= 0 && target < V ? lse - st.at[r] : NAN;
    }
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
    // What all rows have in common goes behind the products: multiplied into softmax minus one-hot ahead of a rounding to
    // bfloat16 it would round every row's largest part, minus the factor, off by the same amount.
    float factor = reduction == AXC_LOSS_MEAN ? 1.0f / (float)(count > 0 ? count : 1) : 1.0f;
    float most = 1.0f;
    if (grad_loss) {
        most = 0.0f;
        if (reduction != AXC_LOSS_NONE)
            most = fabsf(grad_loss[0]);
        else
            for (int64_t r = threadIdx.x; r < rows; r += 1024)
                most = fmaxf(most, targets[r] == ignore ? 0.0f : fabsf(grad_loss[r]));
        float least = 0.0f;
        __shared__ float red[32];
        block_range(least, most, red);
        factor *= most;
    }
    if (threadIdx.x == 0)
        *st.factor = factor;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) {
        const float of = grad_loss ? grad_loss[reduction == AXC_LOSS_NONE ? r : 0] : 1.0f;
        const int64_t t = targets[r];
        st.coefficient[r] = t == ignore || of == 0.0f ? 0.0f : t >= 0 && t < V ? of / most : NAN;
    }
}

} // namespace

hipError_t launch_loss_piece(const TableSums &s, int64_t rows, int columns, int64_t first_column, const void *bias, int bias_type,
                             const int64_t *targets, int64_t ignore, int64_t V, bool first, bool last, const LossState &st,
                             hipStream_t stream)
{
    // many rows have wavefronts enough; few rows need theirs long
    hipLaunchKernelGGL(loss_piece_kernel, dim3((unsigned)rows), dim3(rows >= 1024 ? 256 : 1024), 0, stream, s, columns, first_column,
                       bias, bias_type, targets, ignore, V, (int)first, (int)last, st);
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
