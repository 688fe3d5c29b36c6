// C-ABI entry points of the transformer layers: checks, workspaces, launches.
#include "layers_internal.h"

#include <string.h>

#include <algorithm>

using namespace axc;

namespace {

#define AXC_HIP(call)                                \
    do {                                             \
        hipError_t e_ = (call);                      \
        if (e_ != hipSuccess)                        \
            return api_fail_hip(e_, #call);          \
    } while (0)

int64_t fours(int64_t n) { return (n + 3) & ~(int64_t)3; }

bool known_type(int type) { return type == AXC_F32 || type == AXC_BF16 || type == AXC_F16; }

int check_desc(const axc_dense_desc *d)
{
    if (!d)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    if (d->rows < 0 || d->columns < 0 || d->depth < 0)
        return api_fail(AXC_INVALID_ARGUMENT, "rows, depth and columns must not be negative");
    if (d->depth < 1)
        return api_fail(AXC_INVALID_ARGUMENT, "depth must be at least 1");
    if (fours(d->depth) >= 32768)   // 32768 * 65535 would overflow the int32 accumulator
        return api_fail(AXC_INVALID_ARGUMENT, "depth must be at most 32764 for int32 accumulation");
    const int64_t most = ((int64_t)1 << 31) - 256;
    if (d->rows > most || d->columns > most || d->rows * d->columns >= ((int64_t)1 << 40) ||
        d->columns * d->depth >= ((int64_t)1 << 40))
        return api_fail(AXC_INVALID_ARGUMENT, "tensor too large");
    if (!known_type(d->input_type) || !known_type(d->kernel_type) || !known_type(d->bias_type))
        return api_fail(AXC_INVALID_ARGUMENT, "unknown element type");
    if (d->activation < AXC_ACT_NONE || d->activation > AXC_ACT_SILU)
        return api_fail(AXC_INVALID_ARGUMENT, "unknown activation");
    return AXC_OK;
}
constexpr int64_t kMostGradientRows = 4194176;   // 65 534 tiles of 64: with those of the columns they are counted in 32 bits

// Hands out parts of a workspace; without one it only counts.
class Carver {
public:
    explicit Carver(void *base) : base_(static_cast<char *>(base)) {}
    template <typename T>
    T *take(size_t n)
    {
        T *const p = base_ ? reinterpret_cast<T *>(base_ + at_) : nullptr;
        at_ += (n * sizeof(T) + 255) & ~(size_t)255;
        return p;
    }
    size_t bytes() const { return at_; }

private:
    char *base_;
    size_t at_ = 0;
};

int check_workspace(const void *workspace, size_t have, size_t need)
{
    if (have < need || (!workspace && need))
        return api_fail(AXC_INVALID_ARGUMENT, "workspace too small (see the call's workspace query)");
    if (((uintptr_t)workspace & 255) != 0)
        return api_fail(AXC_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    return AXC_OK;
}

int check_aligned(const void *range, const void *packed)
{
    if (((uintptr_t)range & 7) != 0)
        return api_fail(AXC_INVALID_ARGUMENT, "ranges must be 8-byte aligned");
    if (((uintptr_t)packed & 255) != 0)
        return api_fail(AXC_INVALID_ARGUMENT, "a packed kernel must be 256-byte aligned");
    return AXC_OK;
}

const void *element(const void *p, int64_t i, int type) { return p ? static_cast<const char *>(p) + i * type_bytes(type) : nullptr; }
void *element(void *p, int64_t i, int type) { return p ? static_cast<char *>(p) + i * type_bytes(type) : nullptr; }

// Columns in pieces of about the same width, `most` at most.
Pieces pieces_of(int64_t depth, int64_t columns, int64_t most)
{
    Pieces p = {};
    p.Np = fours(columns);
    p.Kp = (int32_t)fours(depth);
    p.Kb = (int32_t)((depth + 15) & ~(int64_t)15);
    const int64_t count = std::max<int64_t>(1, (p.Np + most - 1) / most);
    const int64_t each = (p.Np + count - 1) / count;
    p.width = (int32_t)std::min<int64_t>(std::max<int64_t>(4, p.Np), (each + 63) / 64 * 64);
    p.count = (int32_t)std::max<int64_t>(1, (p.Np + p.width - 1) / p.width);
    return p;
}

// ---- sums of table entries: input codes by a piece of the kernel's ----
constexpr int64_t kRowRun = 16384;       // rows a LUT-GEMM call takes (its rows must be below 32768)
constexpr int64_t kSumsAtOnce = (int64_t)1 << 25;   // int32 sums in the workspace: 128 MiB, half the memory-side cache
// Up to here few_rows_kernel is the shorter one, by rows (us, packed 4096 -> 4096: 16 rows 29, 63 by the kernels of many rows, 32 rows
// 48 and 65, 64 rows about 85 and 72; 4096 -> 14336, 32 rows 131 and 141).
constexpr int64_t kFewRowsMost = 32;

bool few_rows(int64_t rows) { return rows <= kFewRowsMost; }

axc_conv2d_desc conv_desc(int64_t rows, int Kp, int width)
{
    axc_conv2d_desc c;
    memset(&c, 0, sizeof(c));
    c.input_shape[0] = c.input_shape[1] = 1;
    c.input_shape[2] = rows;
    c.input_shape[3] = Kp;
    c.filter_shape[0] = c.filter_shape[1] = 1;
    c.filter_shape[2] = Kp;
    c.filter_shape[3] = width;
    for (int i = 0; i < 4; ++i)
        c.strides[i] = c.dilations[i] = 1;
    c.padding = AXC_PAD_VALID;
    c.data_format = AXC_FORMAT_NHWC;
    c.num_bits = 8;
    return c;
}

// What the sums of a run of rows (kRowRun at most) and any piece need: int32 values of their own, and scratch bytes.  few: the call
// has few rows altogether.
int sums_workspace(bool few, int64_t rows, const Pieces &pc, size_t *count, size_t *bytes)
{
    for (const int width : {pc.width_of(0), pc.width_of(pc.count - 1)}) {
        if (few) {
            *count = std::max(*count, (size_t)few_rows_splits(rows, pc.Kb, width) * rows * (width + 4));
            continue;
        }
        const axc_conv2d_desc c = conv_desc(fours(rows), pc.Kp, width);
        size_t need = 0;
        if (int rc = axc_conv2d_workspace_bytes(&c, &need))
            return rc;
        *count = std::max(*count, (size_t)fours(rows) * width);
        *bytes = std::max(*bytes, need);
    }
    return AXC_OK;
}

// ---- operands ----
struct Operands {
    Grids *grids;
    float *x_pairs, *kernel_pairs;
    uint8_t *x_codes, *kernel_codes, *kernel_blocks;
    int32_t *row_sums, *column_sums;
    FewInput raw;                        // x not null: few_rows_kernel makes the input's codes itself
};

Operands carve_operands(Carver &c, const axc_dense_desc *d, const Pieces &pc, bool with_kernel, bool codes)
{
    Operands o = {};
    o.grids = c.take<Grids>(1);
    o.x_pairs = c.take<float>(2 * kRangeBlocks);
    o.kernel_pairs = c.take<float>(2 * kRangeBlocks);
    if (codes) {
        o.x_codes = few_rows(d->rows) ? c.take<uint8_t>((size_t)(d->rows + 7) / 8 * 8 * pc.Kb)
                                      : c.take<uint8_t>((size_t)fours(d->rows) * pc.Kp);
        o.row_sums = c.take<int32_t>((size_t)fours(d->rows));
    }
    if (codes && with_kernel) {
        if (few_rows(d->rows))
            o.kernel_blocks = c.take<uint8_t>(pc.block_bytes());
        else
            o.kernel_codes = c.take<uint8_t>(pc.bytes());
        o.column_sums = c.take<int32_t>((size_t)pc.Np);
    }
    return o;
}

RangeSource input_source(const axc_dense_desc *d, const void *range)
{
    if (d->range_known)
        return {nullptr, 0, d->input_min, d->input_max};
    if (range)
        return {static_cast<const float *>(range), kRangePairs, 0.0f, 0.0f};
    return {nullptr, -1, 0.0f, 0.0f};
}

// The ranges that have to be looked for, into pairs; clears the column sums of a kernel whose codes are to be made.  What a call before has
// reported of the input's, kRangePairs, becomes one pair on the way: each workgroup behind would read them all (16 384 rows, 64 -> 64:
// 39.5 us a call in place of 44.3).
int find_ranges(const axc_dense_desc *d, const void *input, const void *range, const void *kernel, float *x_pairs, float *kernel_pairs,
                int32_t *zeros, int64_t n_zeros, RangeSource *in, RangeSource *k, hipStream_t stream)
{
    *in = input ? input_source(d, range) : RangeSource{};
    const bool look = !in->pairs && in->count < 0;
    const float *const reported = kernel ? in->pairs : nullptr;
    int x_count = 0, k_count = 0;
    {
        ApiTimer t("layer_range", stream);
        AXC_HIP(launch_range(look ? input : nullptr, d->input_type, d->rows * d->depth, reported, kernel, d->kernel_type,
                             d->depth * d->columns, x_pairs, kernel_pairs, zeros, n_zeros, &x_count, &k_count, stream));
    }
    if (look || reported)
        *in = {x_pairs, x_count, 0.0f, 0.0f};
    *k = {kernel_pairs, k_count, 0.0f, 0.0f};
    return AXC_OK;
}

int make_codes(const axc_dense_desc *d, const void *input, const RangeSource &in, const void *kernel, const RangeSource &k,
               const Grid *kernel_grid, const Operands &o, const Pieces &pc, hipStream_t stream)
{
    CodesJob job = {};
    job.x = input;
    job.kernel = kernel;
    job.x_type = d->input_type;
    job.kernel_type = d->kernel_type;
    job.rows = d->rows;
    job.N = d->columns;
    job.K = (int)d->depth;
    job.x_range = in;
    job.kernel_range = k;
    job.kernel_grid = kernel_grid;
    job.pieces = pc;
    job.grids = o.grids;
    job.x_codes = o.x_codes;
    job.kernel_codes = o.kernel_codes;
    job.kernel_blocks = o.kernel_blocks;
    job.row_sums = o.row_sums;
    job.column_sums = o.column_sums;
    ApiTimer t("layer_codes", stream);
    AXC_HIP(launch_codes(job, stream));
    return AXC_OK;
}

// Few rows of the input, against a kernel whose grid is known (null: it stands in the grids already).
int make_few_codes(const axc_dense_desc *d, const void *input, const void *range, const Grid *kernel_grid, const Operands &o,
                   const Pieces &pc, hipStream_t stream)
{
    ApiTimer t("layer_codes", stream);
    const FewInput in = {input, d->input_type, (int)d->depth, input_source(d, range), kernel_grid};
    AXC_HIP(launch_few_codes(in, (int)d->rows, pc.Kb, o.grids, o.x_codes, o.row_sums, stream));
    return AXC_OK;
}

// The same of a kernel alone.
int make_kernel_codes(const axc_dense_desc *d, const void *kernel, const Operands &o, const Pieces &pc, hipStream_t stream)
{
    RangeSource in, k;
    if (int rc = find_ranges(d, nullptr, nullptr, kernel, nullptr, o.kernel_pairs, o.column_sums, pc.Np, &in, &k, stream))
        return rc;
    return make_codes(d, nullptr, in, kernel, k, nullptr, o, pc, stream);
}

// Ranges, grids, codes and their sums of both operands.
int find_codes(const axc_dense_desc *d, const void *input, const void *range, const void *kernel, const Operands &o, const Pieces &pc,
               hipStream_t stream)
{
    if (few_rows(d->rows)) {
        if (int rc = make_kernel_codes(d, kernel, o, pc, stream))
            return rc;
        return make_few_codes(d, input, range, nullptr, o, pc, stream);
    }
    RangeSource in, k;
    if (int rc = find_ranges(d, input, range, kernel, o.x_pairs, o.kernel_pairs, o.column_sums, pc.Np, &in, &k, stream))
        return rc;
    return make_codes(d, input, in, kernel, k, nullptr, o, pc, stream);
}

// Sums of the run of rows from r on and piece p, in acc or in the scratch, as their consumer is given them.
int table_sums(const axc_table *table, const axc_dense_desc *d, const Operands &o, const Pieces &pc, int p, int64_t r, int64_t rows,
               int32_t *acc, void *ws, size_t ws_bytes, hipStream_t stream, TableSums *out)
{
    const bool few = few_rows(d->rows);
    const int width = pc.width_of(p);
    *out = {};
    out->row_sums = o.row_sums + r;
    out->column_sums = o.column_sums + pc.first(p);
    out->table = table->dev_tableT;
    out->grids = o.grids;
    out->K = (int)d->depth;
    out->pad = (few ? pc.Kb : pc.Kp) - (int)d->depth;
    if (few) {
        const int splits = few_rows_splits(rows, pc.Kb, width);
        if (o.raw.x) {
            out->row_sums = nullptr;
            out->sums_at = width;
        }
        const FewJob job = {table->dev_tableS, o.raw, o.x_codes, o.grids, o.kernel_blocks + pc.block_offset(p), (int)rows, pc.Kb, width,
                            splits, acc, width + 4};
        out->raw = {acc, rows * job.pitch, splits, job.pitch, 0};
        ApiTimer t("few_rows", stream);
        AXC_HIP(launch_few_rows(job, stream));
        return AXC_OK;
    }
    const axc_conv2d_desc c = conv_desc(fours(rows), pc.Kp, width);
    return api_codes_sums(table, &c, o.x_codes + r * pc.Kp, o.kernel_codes + pc.offset(p), acc, ws, ws_bytes, stream, &out->raw);
}

// ---- dense ----
constexpr int64_t kDensePiece = 8192;    // columns; packed kernels are laid out by it, whatever rows they meet

struct Packed {                          // a packed kernel
    Grids *grids;
    float *pairs;
    int32_t *column_sums;
    uint8_t *codes, *blocks;             // for many rows, for few
    size_t bytes;
};
Packed packed_parts(const Pieces &pc, void *base)
{
    Carver c(base);
    Packed p = {};
    p.grids = c.take<Grids>(1);
    p.pairs = c.take<float>(2 * kRangeBlocks);
    p.column_sums = c.take<int32_t>((size_t)pc.Np);
    p.codes = c.take<uint8_t>(pc.bytes());
    p.blocks = c.take<uint8_t>(pc.block_bytes());
    p.bytes = c.bytes();
    return p;
}

int64_t dense_run(int64_t rows, const Pieces &pc)   // rows whose sums are in the workspace at a time
{
    const int64_t run = std::min(kRowRun, std::max<int64_t>(1024, kSumsAtOnce / pc.width & ~(int64_t)3));
    return std::min(rows, run);
}
// Sums and scratch of `rows` rows, a run at a time.
int runs_workspace(int64_t rows, int64_t run, const Pieces &pc, size_t *count, size_t *bytes)
{
    const bool few = few_rows(rows);
    *count = *bytes = 0;
    if (int rc = sums_workspace(few, run, pc, count, bytes))
        return rc;
    return rows % run ? sums_workspace(few, rows % run, pc, count, bytes) : AXC_OK;
}

struct DenseScratch {
    Operands o;
    int32_t *acc;
    char *lut;
    size_t lut_bytes, bytes;
};
int carve_dense(const axc_dense_desc *d, bool packed, void *base, DenseScratch *s)
{
    const Pieces pc = pieces_of(d->depth, d->columns, kDensePiece);
    Carver c(base);
    *s = {};
    if (packed && token_fits(d->rows, pc.Kb))
        return AXC_OK;                   // nothing is kept
    s->o = carve_operands(c, d, pc, !packed, true);
    size_t count = 0;
    if (int rc = runs_workspace(d->rows, dense_run(d->rows, pc), pc, &count, &s->lut_bytes))
        return rc;
    s->acc = c.take<int32_t>(count);
    s->lut = c.take<char>(s->lut_bytes);
    s->bytes = c.bytes();
    return AXC_OK;
}

// ---- gradients ----
// Rows whose gradient stands in front of the products at a time: 2^28 values of it, or of the input, are 512 MiB a term and copy.  (All rows
// at once took 12 GB for 65 536 rows, 4096 -> 14 336, in float32.  Kernels' gradients go on from run to run as partial sums: 16 384 of
// those rows, in bfloat16, take 4.21 ms at once, 4.42 in two runs.)
constexpr int64_t kGradValues = (int64_t)1 << 28;
int64_t grad_run(const axc_dense_desc *d)
{
    const int64_t run = kGradValues / product_pad(std::max(d->columns, d->depth)) / kProductTile * kProductTile;
    return std::min(d->rows, std::max<int64_t>(8 * kProductTile, run));
}
struct GradScratch {
    Operands o;
    bf16 *straight, *turned, *x_turned, *kernel;
    float *column_partials, *partials[2];
    ProductPlan plans[2];                // of the input's product and of the kernel's
};

} // namespace

extern "C" {

int axc_dense_packed_bytes(const axc_dense_desc *desc, size_t *bytes)
{
    if (int rc = check_desc(desc))
        return rc;
    if (!bytes)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    *bytes = packed_parts(pieces_of(desc->depth, desc->columns, kDensePiece), nullptr).bytes;
    return AXC_OK;
}

int axc_dense_pack(const axc_dense_desc *desc, const void *kernel, void *packed, void *stream_v)
{
    if (int rc = check_desc(desc))
        return rc;
    if (desc->columns == 0)
        return AXC_OK;
    if (!kernel || !packed)
        return api_fail(AXC_INVALID_ARGUMENT, "null tensor pointer");
    if (int rc = check_aligned(nullptr, packed))
        return rc;
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    const Pieces pc = pieces_of(desc->depth, desc->columns, kDensePiece);
    const Packed p = packed_parts(pc, packed);
    Operands o = {};
    o.grids = p.grids;
    o.kernel_pairs = p.pairs;
    o.kernel_codes = p.codes;
    o.kernel_blocks = p.blocks;
    o.column_sums = p.column_sums;
    return make_kernel_codes(desc, kernel, o, pc, stream);
}

int axc_fake_approx_dense_workspace_bytes(const axc_dense_desc *desc, int packed, size_t *bytes)
{
    if (int rc = check_desc(desc))
        return rc;
    if (!bytes)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    *bytes = 0;
    if (desc->rows == 0 || desc->columns == 0)
        return AXC_OK;
    DenseScratch s;
    if (int rc = carve_dense(desc, packed != 0, nullptr, &s))
        return rc;
    *bytes = s.bytes;
    return AXC_OK;
}

int axc_fake_approx_dense(const axc_table *table, const axc_dense_desc *desc, const void *input, const void *input_range,
                          const void *kernel, const void *packed, const void *bias, const void *residual, void *output, void *pre,
                          void *workspace, size_t workspace_bytes, void *stream_v)
{
    if (!table)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    if (int rc = check_desc(desc))
        return rc;
    if (int rc = api_check_table(table))
        return rc;
    if (desc->rows == 0 || desc->columns == 0)
        return AXC_OK;
    if (!input || !output || (!kernel && !packed))
        return api_fail(AXC_INVALID_ARGUMENT, "null tensor pointer");
    if (kernel && packed)
        return api_fail(AXC_INVALID_ARGUMENT, "either a kernel or a packed one");
    if (int rc = check_aligned(input_range, packed))
        return rc;
    const Pieces pc = pieces_of(desc->depth, desc->columns, kDensePiece);
    DenseScratch s;
    if (int rc = carve_dense(desc, packed != nullptr, workspace, &s))
        return rc;
    if (int rc = check_workspace(workspace, workspace_bytes, s.bytes))
        return rc;
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    Operands &o = s.o;
    const Grid *kernel_grid = nullptr;   // of a packed kernel
    if (packed) {
        const Packed p = packed_parts(pc, const_cast<void *>(packed));
        o.kernel_codes = p.codes;
        o.kernel_blocks = p.blocks;
        o.column_sums = p.column_sums;
        kernel_grid = &p.grids->kernel;
    }
    if (few_rows(desc->rows)) {
        if (!packed)
            if (int rc = make_kernel_codes(desc, kernel, o, pc, stream))
                return rc;
        const FewInput in = {input, desc->input_type, (int)desc->depth, input_source(desc, input_range),
                             packed ? kernel_grid : &o.grids->kernel};
        if (token_fits(desc->rows, pc.Kb)) {
            const TokenJob job = {table->dev_tableL, in, o.kernel_blocks, o.column_sums, pc, (int)desc->rows, desc->columns,
                                  {bias, residual, output, pre, desc->bias_type, desc->input_type, desc->activation, desc->columns}};
            ApiTimer t("token", stream);
            AXC_HIP(launch_token(job, stream));
            return AXC_OK;
        }
        if (desc->rows * desc->depth <= kFewRawValues || in.range.count >= 0)
            o.raw = in;
        else if (int rc = make_few_codes(desc, input, input_range, kernel_grid, o, pc, stream))
            return rc;
    } else if (packed) {
        RangeSource in, none;
        if (int rc = find_ranges(desc, input, input_range, nullptr, o.x_pairs, nullptr, nullptr, 0, &in, &none, stream))
            return rc;
        if (int rc = make_codes(desc, input, in, nullptr, none, kernel_grid, o, pc, stream))
            return rc;
    } else if (int rc = find_codes(desc, input, input_range, kernel, o, pc, stream)) {
        return rc;
    }
    const int64_t run = dense_run(desc->rows, pc);
    for (int p = 0; p < pc.count; ++p)
        for (int64_t r = 0; r < desc->rows; r += run) {
            const int64_t rows = std::min(run, desc->rows - r), c = pc.first(p);
            TableSums sums;
            if (int rc = table_sums(table, desc, o, pc, p, r, rows, s.acc, s.lut, s.lut_bytes, stream, &sums))
                return rc;
            const int64_t at = r * desc->columns + c;
            const DenseOut out = {element(bias, c, desc->bias_type), element(residual, at, desc->input_type),
                                  element(output, at, desc->input_type), element(pre, at, desc->input_type), desc->bias_type,
                                  desc->input_type, desc->activation, desc->columns};
            ApiTimer t("dense_out", stream);
            AXC_HIP(launch_dense_out(sums, rows, (int)std::min<int64_t>(pc.width_of(p), desc->columns - c), out, stream));
        }
    return AXC_OK;
}

// Operands and workspace of the gradients.
static int carve_gradients(const axc_dense_desc *d, void *base, GradScratch *s, size_t *bytes)
{
    if (d->rows > kMostGradientRows)
        return api_fail(AXC_UNIMPLEMENTED, "gradients of more than 4194176 rows");
    const Pieces pc = pieces_of(d->depth, d->columns, kDensePiece);
    const int64_t run = grad_run(d), M = product_pad(run), N = product_pad(d->columns), K = product_pad(d->depth);
    const int exact = exact_terms(d->input_type, d->activation);
    const int px = parts_of(d->input_type, exact), pk = parts_of(d->kernel_type, exact);
    Carver c(base);
    s->o = carve_operands(c, d, pc, false, false);
    s->straight = c.take<bf16>((size_t)M * N * px);
    s->turned = c.take<bf16>((size_t)M * N * pk);
    s->x_turned = c.take<bf16>((size_t)M * K);
    s->kernel = c.take<bf16>((size_t)K * N);
    s->column_partials = c.take<float>((size_t)(product_pad(d->rows) / 64) * N);
    const ProductShape shapes[2] = {{run, d->depth, d->columns, px, 0}, {d->depth, d->columns, run, pk, run < d->rows}};
    plan_products(shapes, 2, s->plans);
    for (int i = 0; i < 2; ++i)
        s->partials[i] = s->plans[i].partial_bytes ? reinterpret_cast<float *>(c.take<char>(s->plans[i].partial_bytes)) : nullptr;
    *bytes = c.bytes();
    return AXC_OK;
}

int axc_fake_approx_dense_gradients_workspace_bytes(const axc_dense_desc *desc, size_t *bytes)
{
    if (int rc = check_desc(desc))
        return rc;
    if (!bytes)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    *bytes = 0;
    if (desc->rows == 0 || desc->columns == 0)
        return AXC_OK;
    GradScratch s;
    return carve_gradients(desc, nullptr, &s, bytes);
}

// Products, then results of those whose partial sums are whole; column sums with them, or alone.
static int make_products(const Product *products, int count, const ColumnJob &job, hipStream_t stream)
{
    if (count == 0) {
        ApiTimer t("column_sums", stream);
        if (job.out)
            AXC_HIP(launch_column_sums(job, stream));
        return AXC_OK;
    }
    ApiTimer t("grad_product", stream);
    AXC_HIP(launch_products(products, count, job, stream));
    Product whole[2];
    int left = 0;
    for (int i = 0; i < count; ++i)
        if (products[i].partials && products[i].o.out)
            whole[left++] = products[i];
    if (left)
        AXC_HIP(launch_products_out(whole, left, stream));
    return AXC_OK;
}

static int fill_zero(void *p, int64_t n, int type, hipStream_t stream)
{
    if (!p || n == 0)
        return AXC_OK;
    AXC_HIP(launch_zero(p, n * type_bytes(type), stream));
    return AXC_OK;
}

int axc_fake_approx_dense_gradients(const axc_dense_desc *desc, const void *grad_output, const void *input,
                                    const void *input_range, const void *kernel, const void *pre, void *grad_input,
                                    void *grad_kernel, void *grad_bias, void *workspace, size_t workspace_bytes, void *stream_v)
{
    if (int rc = check_desc(desc))
        return rc;
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    if (desc->rows == 0 || desc->columns == 0) {   // empty sums
        if (int rc = fill_zero(grad_input, desc->rows * desc->depth, desc->input_type, stream))
            return rc;
        if (int rc = fill_zero(grad_kernel, desc->depth * desc->columns, desc->kernel_type, stream))
            return rc;
        return fill_zero(grad_bias, desc->columns, desc->kernel_type, stream);
    }
    if (!grad_output || !input || !kernel)
        return api_fail(AXC_INVALID_ARGUMENT, "null tensor pointer");
    if (int rc = check_aligned(input_range, nullptr))
        return rc;
    if (!pre && desc->activation != AXC_ACT_NONE)
        return api_fail(AXC_INVALID_ARGUMENT, "the gradient of an activation needs what the activation was given");
    GradScratch s;
    size_t need = 0;
    if (int rc = carve_gradients(desc, workspace, &s, &need))
        return rc;
    if (int rc = check_workspace(workspace, workspace_bytes, need))
        return rc;
    if (!grad_input && !grad_kernel && !grad_bias)
        return AXC_OK;
    const int64_t rows = desc->rows, K = desc->depth, N = desc->columns;
    const int exact = exact_terms(desc->input_type, desc->activation);
    const int px = parts_of(desc->input_type, exact), pk = parts_of(desc->kernel_type, exact);
    RangeSource ranges[2];
    if (int rc = find_ranges(desc, input, input_range, kernel, s.o.x_pairs, s.o.kernel_pairs, nullptr, 0, &ranges[0], &ranges[1],
                             stream))
        return rc;
    const int64_t run = grad_run(desc);
    for (int64_t r = 0; r < rows; r += run) {
        const int64_t n = std::min(run, rows - r);
        const bool first = r == 0, last = r + n == rows;
        const void *const x = element(input, r * K, desc->input_type);
        GradSource g = {};
        g.grad = element(grad_output, r * N, desc->input_type);
        g.pre = desc->activation == AXC_ACT_NONE ? nullptr : element(pre, r * N, desc->input_type);
        g.type = desc->input_type;
        g.activation = desc->activation;
        {
            ApiTimer t("grad_prep", stream);
            AXC_HIP(launch_grad_prep(g, false, 0, n, n, N, N, px, grad_input ? s.straight : nullptr, pk, grad_kernel ? s.turned : nullptr,
                                     grad_bias ? s.column_partials + r / 64 * product_pad(N) : nullptr,
                                     {x, desc->input_type, n, K, K, grad_kernel ? s.x_turned : nullptr},
                                     {kernel, desc->kernel_type, K, N, N, grad_input && first ? s.kernel : nullptr},
                                     first ? ranges : nullptr, s.o.grids, stream));
        }
        const ColumnJob job = {s.column_partials, product_pad(rows) / 64, N, product_pad(N), nullptr, last ? grad_bias : nullptr,
                               desc->kernel_type};
        Product products[2];
        int count = 0;
        if (grad_input)
            products[count++] = {s.straight, s.kernel, n, K, (int)product_pad(N), px, 1, s.plans[0].splits, s.partials[0], 0,
                                 {element(grad_input, r * K, desc->input_type), desc->input_type, K, x, K, &s.o.grids->in,
                                  &s.o.grids->kernel, nullptr}};
        if (grad_kernel)
            products[count++] = {s.x_turned, s.turned, K, N, (int)product_pad(n), pk, 0, s.plans[1].splits, s.partials[1], !first,
                                 {last ? grad_kernel : nullptr, desc->kernel_type, N, kernel, N, &s.o.grids->kernel, &s.o.grids->in,
                                  nullptr}};
        if (int rc = make_products(products, count, job, stream))
            return rc;
    }
    return AXC_OK;
}

// ---- loss ----
// Columns whose sums are in the workspace at a time, 256 MiB of them: the last piece's need not be made again for the gradients, and
// making them takes longer than reading them from beyond the memory-side cache.  The same without gradients, so that the loss is.
static Pieces loss_pieces(const axc_dense_desc *d)
{
    const int64_t most = 2 * kSumsAtOnce / fours(std::max<int64_t>(1, d->rows)) & ~(int64_t)255;
    const int64_t codes = ((int64_t)1 << 29) / fours(d->depth) & ~(int64_t)255;   // the LUT-GEMM's offsets have 32 bits
    return pieces_of(d->depth, d->columns, std::min(codes, std::min<int64_t>(65536, std::max<int64_t>(1024, most))));
}

// Products of a piece of so many columns; the input's is that of the first whatever the piece, as its partial sums go on.
struct LossPlan {
    ProductPlan input, kernel;
};
static LossPlan loss_plan(const axc_dense_desc *d, const Pieces &pc, int64_t columns)
{
    const int px = parts_of(d->input_type, 3), pk = parts_of(d->kernel_type, 3);
    const ProductShape first[2] = {{d->rows, d->depth, pc.width_of(0), px, 1}, {d->depth, pc.width_of(0), d->rows, pk, 0}};
    const ProductShape own[2] = {{d->rows, d->depth, columns, px, 1}, {d->depth, columns, d->rows, pk, 0}};
    ProductPlan a[2], b[2];
    plan_products(first, 2, a);
    plan_products(own, 2, b);
    return {a[0], b[1]};
}

struct LossScratch {
    Operands o;
    LossState st;
    int32_t *acc;
    char *lut;
    size_t lut_bytes, bytes;
    bf16 *straight, *turned, *x_turned, *kernel;
    float *column_partials, *kernel_partials, *input_partials;
};
static int carve_loss(const axc_dense_desc *d, bool gradients, void *base, LossScratch *s)
{
    if (d->rows > kMostGradientRows)
        return api_fail(AXC_UNIMPLEMENTED, "a loss of more than 4194176 rows");
    const Pieces pc = loss_pieces(d);
    Carver c(base);
    s->o = carve_operands(c, d, pc, true, true);
    float **const state[] = {&s->st.at, &s->st.top, &s->st.log_sum, &s->st.rows, &s->st.coefficient};
    for (float **p : state)
        *p = c.take<float>((size_t)d->rows);
    s->st.factor = c.take<float>(1);
    s->st.parts = c.take<float2>((size_t)pc.count * ((pc.width + loss_chunk(d->rows) - 1) / loss_chunk(d->rows)) * d->rows);
    size_t count = 0;
    if (int rc = runs_workspace(d->rows, std::min(d->rows, kRowRun), pc, &count, &s->lut_bytes))
        return rc;
    s->acc = c.take<int32_t>(count);
    s->lut = c.take<char>(s->lut_bytes);
    if (gradients) {
        const int64_t M = product_pad(d->rows), P = product_pad(pc.width), K = product_pad(d->depth);
        const int px = parts_of(d->input_type, 3), pk = parts_of(d->kernel_type, 3);
        s->straight = c.take<bf16>((size_t)M * P * px);
        s->turned = c.take<bf16>((size_t)M * P * pk);
        s->x_turned = c.take<bf16>((size_t)M * K);
        s->kernel = c.take<bf16>((size_t)K * P);
        s->column_partials = c.take<float>((size_t)(M / 64) * P);
        size_t most = 0;
        for (const int width : {pc.width_of(0), pc.width_of(pc.count - 1)})
            most = std::max(most, loss_plan(d, pc, width).kernel.partial_bytes);
        s->kernel_partials = reinterpret_cast<float *>(c.take<char>(most));
        s->input_partials = reinterpret_cast<float *>(c.take<char>(loss_plan(d, pc, pc.width_of(0)).input.partial_bytes));
    }
    s->bytes = c.bytes();
    return AXC_OK;
}

int axc_fake_approx_cross_entropy_workspace_bytes(const axc_dense_desc *desc, int gradients, size_t *bytes)
{
    if (int rc = check_desc(desc))
        return rc;
    if (!bytes)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    *bytes = 0;
    if (desc->rows == 0 || desc->columns == 0)
        return AXC_OK;
    LossScratch s;
    if (int rc = carve_loss(desc, gradients != 0, nullptr, &s))
        return rc;
    *bytes = s.bytes;
    return AXC_OK;
}

int axc_fake_approx_cross_entropy(const axc_table *table, const axc_dense_desc *desc, const void *input, const void *input_range,
                                  const void *kernel, const void *bias, const int64_t *targets, int64_t ignore_index,
                                  int reduction, const float *grad_loss, float *loss, void *grad_input, void *grad_kernel,
                                  void *grad_bias, void *workspace, size_t workspace_bytes, void *stream_v)
{
    if (!table)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    if (int rc = check_desc(desc))
        return rc;
    if (desc->activation != AXC_ACT_NONE)
        return api_fail(AXC_INVALID_ARGUMENT, "logits have no activation");
    if (reduction != AXC_LOSS_NONE && reduction != AXC_LOSS_SUM && reduction != AXC_LOSS_MEAN)
        return api_fail(AXC_INVALID_ARGUMENT, "unknown reduction");
    if (desc->columns == 0)
        return api_fail(AXC_INVALID_ARGUMENT, "a vocabulary must have at least one column");
    if (int rc = api_check_table(table))
        return rc;
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    const int64_t rows = desc->rows, K = desc->depth, V = desc->columns;
    if (!loss && !(rows == 0 && reduction == AXC_LOSS_NONE))
        return api_fail(AXC_INVALID_ARGUMENT, "null tensor pointer");
    if (rows == 0) {   // empty sums
        if (int rc = fill_zero(loss, reduction == AXC_LOSS_NONE ? 0 : 1, AXC_F32, stream))
            return rc;
        if (int rc = fill_zero(grad_kernel, K * V, desc->kernel_type, stream))
            return rc;
        return fill_zero(grad_bias, V, desc->kernel_type, stream);
    }
    if (!input || !kernel || !targets)
        return api_fail(AXC_INVALID_ARGUMENT, "null tensor pointer");
    if (int rc = check_aligned(input_range, nullptr))
        return rc;
    const bool gradients = grad_input || grad_kernel || grad_bias;
    const Pieces pc = loss_pieces(desc);
    LossScratch s;
    if (int rc = carve_loss(desc, gradients, workspace, &s))
        return rc;
    if (int rc = check_workspace(workspace, workspace_bytes, s.bytes))
        return rc;
    const Operands &o = s.o;
    if (int rc = find_codes(desc, input, input_range, kernel, o, pc, stream))
        return rc;

    const int64_t run = std::min(rows, kRowRun);
    TableSums sums;
    auto make_sums = [&](int p, int64_t r) {
        return table_sums(table, desc, o, pc, p, r, std::min(run, rows - r), s.acc, s.lut, s.lut_bytes, stream, &sums);
    };
    auto columns_of = [&](int p) { return std::min<int64_t>(pc.width_of(p), V - pc.first(p)); };
    for (int64_t r = 0; r < rows; r += run) {
        const int64_t run_rows = std::min(run, rows - r);
        int chunk = 0;
        for (int p = 0; p < pc.count; ++p) {
            if (int rc = make_sums(p, r))
                return rc;
            int more = 0;
            ApiTimer t("loss_piece", stream);
            AXC_HIP(launch_loss_piece(sums, r, run_rows, rows, (int)columns_of(p), pc.first(p),
                                      element(bias, pc.first(p), desc->bias_type), desc->bias_type, targets, chunk, &more, s.st,
                                      stream));
            chunk += more;
        }
        ApiTimer t("loss_rows", stream);
        AXC_HIP(launch_loss_rows(s.st, targets, ignore_index, V, r, run_rows, rows, chunk, stream));
    }
    {
        ApiTimer t("loss_out", stream);
        AXC_HIP(launch_loss_out(s.st, targets, ignore_index, V, rows, reduction, grad_loss, loss, gradients, stream));
    }
    if (!gradients)
        return AXC_OK;

    const int px = parts_of(desc->input_type, 3), pk = parts_of(desc->kernel_type, 3);
    const int64_t M = product_pad(rows);
    const ProductOut input_out = {grad_input, desc->input_type, K, input, K, &o.grids->in, &o.grids->kernel, s.st.factor};
    // from the last piece on, whose last run's sums are still there
    bool made = true;
    for (int p = pc.count - 1; p >= 0; --p) {
        const int64_t c = pc.first(p), n = columns_of(p), P = product_pad(n);
        for (int64_t r = (rows - 1) / run * run; r >= 0; r -= run) {
            if (!made)
                if (int rc = make_sums(p, r))
                    return rc;
            made = false;
            GradSource g = {};
            g.sums = sums;
            g.top = s.st.top + r;
            g.log_sum = s.st.log_sum + r;
            g.coefficient = s.st.coefficient + r;
            g.targets = targets + r;
            g.bias = element(bias, c, desc->bias_type);
            g.bias_type = desc->bias_type;
            g.first_column = c;
            // the kernel's codes of the piece, and once the input's, go with the first run
            const bool first_run = r == (rows - 1) / run * run;
            ApiTimer t("grad_prep", stream);
            AXC_HIP(launch_grad_prep(g, true, r, std::min(run, rows - r), rows, n, 0, px, grad_input ? s.straight : nullptr, pk,
                                     grad_kernel ? s.turned : nullptr, grad_bias ? s.column_partials : nullptr,
                                     {input, desc->input_type, rows, K, K,
                                      grad_kernel && first_run && p + 1 == pc.count ? s.x_turned : nullptr},
                                     {element(kernel, c, desc->kernel_type), desc->kernel_type, K, n, V,
                                      grad_input && first_run ? s.kernel : nullptr},
                                     nullptr, o.grids, stream));
        }
        ColumnJob job = {s.column_partials, M / 64, n, P, s.st.factor, element(grad_bias, c, desc->kernel_type), desc->kernel_type};
        const LossPlan plan = loss_plan(desc, pc, n);
        Product products[2];
        int count = 0;
        if (grad_input) {
            products[count] = {s.straight, s.kernel, rows, K, (int)P, px, 1, plan.input.splits, s.input_partials, p + 1 < pc.count,
                               input_out};
            if (p > 0)
                products[count].o.out = nullptr;   // not yet
            ++count;
        }
        if (grad_kernel)
            products[count++] = {s.x_turned, s.turned, K, n, (int)M, pk, 0, plan.kernel.splits,
                                 plan.kernel.partial_bytes ? s.kernel_partials : nullptr, 0,
                                 {element(grad_kernel, c, desc->kernel_type), desc->kernel_type, V,
                                  element(kernel, c, desc->kernel_type), V, &o.grids->kernel, &o.grids->in, s.st.factor}};
        if (int rc = make_products(products, count, job, stream))
            return rc;
    }
    return AXC_OK;
}

// ---- residual norms ----
static int check_norm(const axc_residual_norm_desc *d)
{
    if (!d)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    if (d->rows < 0 || d->width < 1 || d->gate_groups < 0)
        return api_fail(AXC_INVALID_ARGUMENT, "rows and gate groups must not be negative, the width at least 1");
    if (d->width > kNormMaxWidth)
        return api_fail(AXC_UNIMPLEMENTED, "norms of more than 32768 values");
    if (d->rows >= ((int64_t)1 << 40) / d->width)
        return api_fail(AXC_INVALID_ARGUMENT, "tensor too large");
    if (d->gate_groups > 0 && (d->gate_groups > d->rows || d->rows % d->gate_groups != 0) && d->rows > 0)
        return api_fail(AXC_INVALID_ARGUMENT, "the gate's groups must divide the rows");
    if (!known_type(d->type) || !known_type(d->vector_type))
        return api_fail(AXC_INVALID_ARGUMENT, "unknown element type");
    if (d->kind != AXC_NORM_RMS && d->kind != AXC_NORM_LAYER)
        return api_fail(AXC_INVALID_ARGUMENT, "unknown norm");
    if (!(d->eps >= 0.0f))
        return api_fail(AXC_INVALID_ARGUMENT, "eps must not be negative");
    return AXC_OK;
}

static int norm_params(const axc_residual_norm_desc *d, const axc_residual_norm_tensors *in, NormParams *p)
{
    if (!in)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    if (!in->weight)
        return api_fail(AXC_INVALID_ARGUMENT, "null tensor pointer");
    if (d->rows > 0 && !in->block && (in->gate || in->scale || in->post_weight))
        return api_fail(AXC_INVALID_ARGUMENT, "a gate, a scale and a weight of the block's norm need a block");
    if ((in->gate != nullptr) != (d->gate_groups > 0))
        return api_fail(AXC_INVALID_ARGUMENT, "a gate and its number of groups go together");
    *p = NormParams{};
    p->rows = d->rows;
    p->width = d->width;
    p->gate_groups = d->gate_groups;
    p->type = d->type;
    p->vector_type = d->vector_type;
    p->layer = d->kind == AXC_NORM_LAYER;
    p->eps = d->eps;
    p->x = in->x;
    p->block = in->block;
    p->weight = in->weight;
    p->bias = in->bias;
    p->gate = in->gate;
    p->scale = in->scale;
    p->post_weight = in->post_weight;
    return AXC_OK;
}

int axc_residual_norm(const axc_residual_norm_desc *desc, const axc_residual_norm_tensors *in, void *h, void *y,
                      void *output_range, void *stream_v)
{
    if (int rc = check_norm(desc))
        return rc;
    NormParams p;
    if (int rc = norm_params(desc, in, &p))
        return rc;
    if (desc->rows == 0) {
        if (output_range)
            return api_fail(AXC_INVALID_ARGUMENT, "no rows have no range");
        return AXC_OK;
    }
    if (!p.x || !y || (p.block && !h))
        return api_fail(AXC_INVALID_ARGUMENT, "null tensor pointer");
    if (int rc = check_aligned(output_range, nullptr))
        return rc;
    p.h = h;
    p.y = y;
    p.range = static_cast<float *>(output_range);
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    ApiTimer t("residual_norm", stream);
    AXC_HIP(launch_norm(p, stream));
    return AXC_OK;
}

int axc_residual_norm_gradients_workspace_bytes(const axc_residual_norm_desc *desc, size_t *bytes)
{
    if (int rc = check_norm(desc))
        return rc;
    if (!bytes)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    NormParams p = {};
    p.rows = desc->rows;
    p.width = desc->width;
    p.gate_groups = desc->gate_groups;
    *bytes = desc->rows ? norm_partial_bytes(p) : 0;
    return AXC_OK;
}

int axc_residual_norm_gradients(const axc_residual_norm_desc *desc, const axc_residual_norm_tensors *in, const void *h,
                                const void *grad_h, const void *grad_y, const axc_residual_norm_gradients_out *out,
                                void *workspace, size_t workspace_bytes, void *stream_v)
{
    if (int rc = check_norm(desc))
        return rc;
    NormParams p;
    if (int rc = norm_params(desc, in, &p))
        return rc;
    if (!out)
        return api_fail(AXC_INVALID_ARGUMENT, "null argument");
    if ((out->bias && !in->bias) || (out->gate && !in->gate) || (out->scale && !in->scale) ||
        (out->post_weight && !in->post_weight) || (out->block && !in->block))
        return api_fail(AXC_INVALID_ARGUMENT, "a gradient of what did not go in");
    hipStream_t stream = static_cast<hipStream_t>(stream_v);
    if (desc->rows == 0) {   // empty sums
        for (void *v : {out->weight, out->bias, out->scale, out->post_weight})
            if (int rc = fill_zero(v, desc->width, desc->vector_type, stream))
                return rc;
        return fill_zero(out->gate, desc->gate_groups * desc->width, desc->type, stream);
    }
    if (!h || (!grad_h && !grad_y) || !out->x || (p.block && !out->block))
        return api_fail(AXC_INVALID_ARGUMENT, "null tensor pointer");
    if (int rc = check_workspace(workspace, workspace_bytes, norm_partial_bytes(p)))
        return rc;
    p.x = nullptr;
    p.h = const_cast<void *>(h);
    p.grad_h = grad_h;
    p.grad_y = grad_y;
    p.dx = out->x;
    p.dblock = out->block;
    p.dweight = out->weight;
    p.dbias = out->bias;
    p.dgate = out->gate;
    p.dscale = out->scale;
    p.dpost = out->post_weight;
    p.partials = static_cast<float *>(workspace);
    ApiTimer t("residual_norm_gradients", stream);
    AXC_HIP(launch_norm_gradients(p, stream));
    return AXC_OK;
}

} // extern "C"
