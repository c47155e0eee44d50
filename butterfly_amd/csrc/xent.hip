// Entry points of the linear layer with softmax cross entropy (xent.hpp, of few rows xent_few.hpp): argument checks,
// workspace, launches.

#include "../../include/butterfly_hip.h"

#include <algorithm>

#include "error.hpp"
#include "xent.hpp"
#include "xent_few.hpp"

namespace {

using namespace bf;

int check_xent(const bf_linear_xent *p)
{
    if (!p) return fail(BF_ERR_INVALID, "loss descriptor is NULL");
    if (p->dtype != BF_F32 && p->dtype != BF_BF16) return fail(BF_ERR_INVALID, "dtype must be BF_F32 or BF_BF16");
    if (p->reduction != BF_XENT_NONE && p->reduction != BF_XENT_MEAN && p->reduction != BF_XENT_SUM)
        return fail(BF_ERR_INVALID, "reduction must be BF_XENT_NONE, BF_XENT_MEAN or BF_XENT_SUM");
    if (p->rows < 0 || p->features < 1 || p->vocab < 1) return fail(BF_ERR_INVALID, "rows must be >= 0, features and vocab >= 1");
    if (p->rows > (1 << 24) || p->features > (1 << 16) || p->vocab > (1 << 24))
        return fail(BF_ERR_UNSUPPORTED, "rows and vocab up to 2^24, features up to 2^16 are supported");
    if (p->hidden_stride < 0 || p->weight_stride < 0) return fail(BF_ERR_INVALID, "strides must be non-negative");
    return BF_OK;
}

size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// bfloat16 weights are read where they lie if 16-byte units divide their rows; others are laid out anew.
bool weight_in_place(const bf_linear_xent *p)
{
    return p->dtype == BF_BF16 && p->features % 8 == 0 && p->weight_stride % 8 == 0 && p->weight_stride >= p->features &&
           p->weight_stride <= (1 << 20);
}

struct Product {
    bool large = false, deep = false;   // tiles of 256 x 256, of 128 x 128 in four buffers
    int tiles_m = 0, tiles_n = 0, splits = 1;
    double time = 0;                    // estimate, microseconds
};

// The shape of tiles that takes less time by this estimate.  At a time the chip holds 256 tiles of 256 x 256 or 512 of
// 128 x 128; a k step of 64 takes them 1.75 and 1.05 us, a tile's end (exponentials, stores) 8 and 2 us (of two small
// tiles on a compute unit one computes meanwhile), sums that are split their bytes' way.  Measured, small and large: 8192
// rows, 1024 features, 32768 entries, bfloat16, forward and backward, 2311 and 1957 us (many tiles: the large ones read
// less); 572 x 2659 x 24269, float, 1237 and 1536 (285 large tiles are two rounds); 3300 x 70 x 74639, float, 1315 and
// 1667 (two k steps a tile); 1000 x 1000 x 8000, bfloat16, 121 and 219.
// Small tiles of which each compute unit has only one are made by eight wavefronts out of four buffers: 129 x 1731 x
// 1314, float, 157 us beside 194.
Product product(int64_t m, int64_t n, int64_t steps, int passes, bool may_split)
{
    const int64_t most = may_split ? std::min<int64_t>(std::max<int64_t>(steps / 8, 1), 512) : 1;
    auto ceil = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    auto of = [&](int64_t side, int64_t places, double step, double end) {
        Product r;
        r.large = side == 256;
        r.tiles_m = (int)ceil(m, side);
        r.tiles_n = (int)ceil(n, side);
        const int64_t tiles = std::max<int64_t>((int64_t)r.tiles_m * r.tiles_n, 1);
        auto time = [&](int64_t splits) {
            const double sums = splits > 1 ? 2 + splits * (double)m * n * 8 / 4.8e6 : 0;
            return ceil(tiles * splits, places) * (ceil(steps, splits) * passes * step + end) + sums;
        };
        const int64_t cut = std::max<int64_t>(1, std::min<int64_t>(most, places / tiles));
        r.splits = (int)(time(cut) < time(1) ? cut : 1);
        r.time = time(r.splits);
        return r;
    };
    Product small = of(128, 512, 1.05, 2), large = of(256, 256, 1.75, 8);
    if (large.time < small.time) return large;
    small.deep = (int64_t)small.tiles_m * small.tiles_n * small.splits <= 256;
    return small;
}

// As many as are at work at a time: one a compute unit for large tiles (128 KiB of LDS), two for small ones.
unsigned workgroups(const Product &r)
{
    return (unsigned)std::min<int64_t>((int64_t)r.tiles_m * r.tiles_n * r.splits, r.large || r.deep ? 256 : 512);
}

// d_l of a piece of the vocabulary (8192 rows, 1024 features, 32768 entries, bfloat16: 128 MiB 2161 us, 256 2055, 512 2045)
constexpr size_t kPieceBytes = (size_t)256 << 20;

struct XentPlan {
    int64_t features_up = 0, rows_up = 0;       // padded to k steps, to tiles
    size_t hidden_plane = 0, weight_plane = 0;  // bytes
    int planes = 1;
    Product logits;
    // backward
    int64_t piece = 0;                          // vocabulary entries of a piece, whole tiles
    Product to_hidden, to_weight;
    // offsets into what the forward call leaves for the backward one, and into the workspaces
    size_t scalars = 0, index = 0, position = 0, label = 0, lse = 0, hidden = 0, weight = 0, kept = 0;
    size_t picked = 0, losses = 0, partial = 0;
    size_t share = 0, shared = 0, d_l = 0, d_l_plane = 0, sums_hidden = 0, sums_weight = 0;
    size_t total = 0;
};

XentPlan plan(const bf_linear_xent *p, bool backward)
{
    XentPlan r;
    r.planes = p->dtype == BF_F32 ? 2 : 1;
    const int passes = p->dtype == BF_F32 ? 3 : 1;
    r.features_up = up_to(p->features, kMatK);
    r.rows_up = up_to(std::max<int64_t>(p->rows, 1), 256);
    r.hidden_plane = up256((size_t)r.rows_up * r.features_up * 2);
    r.weight_plane = up256((size_t)p->vocab * r.features_up * 2);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += up256(bytes);
        return here;
    };
    const size_t rows = (size_t)std::max<int64_t>(p->rows, 1);
    r.scalars = take(sizeof(XentScalars));
    r.index = take(rows * 4);
    r.position = take(rows * 4);
    r.label = take(rows * 4);
    r.lse = take(rows * 4);
    r.hidden = take(r.hidden_plane * r.planes);
    if (!weight_in_place(p)) r.weight = take(r.weight_plane * r.planes);
    r.kept = at;
    at = 0;
    if (!backward) {
        r.logits = product(p->vocab, p->rows, r.features_up / kMatK, passes, false);
        r.picked = take(rows * 4);
        r.losses = take(rows * 4);
        r.partial = take((size_t)2 * r.logits.tiles_m * rows * sizeof(float2));
    } else {
        const int64_t most = (int64_t)(kPieceBytes / ((size_t)r.rows_up * 2 * r.planes)) / 256 * 256;
        r.piece = std::min<int64_t>(up_to(p->vocab, 256), std::max<int64_t>(most, 2048));
        const int64_t pieces = (p->vocab + r.piece - 1) / r.piece;
        r.piece = std::min<int64_t>(up_to((p->vocab + pieces - 1) / pieces, 256), r.piece);
        r.logits = product(r.piece, p->rows, r.features_up / kMatK, passes, false);
        r.to_hidden = product(p->features, p->rows, r.piece / kMatK, passes, true);
        r.to_weight = product(p->features, r.piece, (p->rows + kMatK - 1) / kMatK, passes, true);
        r.share = take(rows * 4);
        if (p->dtype == BF_F32 && p->reduction == BF_XENT_NONE) r.shared = take(r.hidden_plane * r.planes);
        r.d_l_plane = up256((size_t)r.rows_up * r.piece * 2);
        r.d_l = take(r.d_l_plane * r.planes);
        r.sums_hidden = take((size_t)r.to_hidden.splits * rows * p->features * sizeof(float));
        if (r.to_weight.splits > 1) r.sums_weight = take((size_t)r.to_weight.splits * r.piece * p->features * sizeof(float));
    }
    r.total = at;
    return r;
}

// ---- few rows ----

// (the logits, which stay in memory, take no more room than float weights)
bool few_rows(const bf_linear_xent *p) { return p->rows > 0 && p->rows <= kFewRows && p->rows <= p->features; }

struct XentFewPlan {
    int tiles = 1, parts = 1, wide = 0;                     // of 16 rows; workgroups of the logits, those of 64 entries
    int64_t stride = 0, steps = 0;                          // of the logits' rows; of 32 entries
    int columns = 1, splits_hidden = 1, splits_weight = 1;  // parts of the columns, of the vocabulary
    size_t scalars = 0, index = 0, position = 0, label = 0, lse = 0, by_feature = 0, by_row = 0, logits = 0, kept = 0;
    size_t losses = 0, partial = 0, d_by_entry = 0, d_by_row = 0, sums = 0;
    size_t total = 0;
};

XentFewPlan few_plan(const bf_linear_xent *p, bool backward)
{
    const bool wide = p->dtype == BF_F32;
    const int64_t planes = wide ? 3 : 1, each = wide ? 4 : 8, chunk = wide ? 32 : 64, chunk_frags = wide ? 3 : 2;
    XentFewPlan r;
    r.tiles = p->rows <= 16 ? 1 : p->rows <= 32 ? 2 : 4;
    // Workgroups of 64 entries read hidden a quarter as often as those of 16 (60 rows, 1000 features, 30001 entries, float: 33 us
    // beside 44), which are work for all compute units where 64 are not (3 rows, 1390 features, 6879 entries: 9.9 us beside
    // 16).  The chip holds two or three of the former a compute unit; a last round that these would fill by less than
    // half is made by the latter.
    if (p->vocab >= 64 * 256) {
        const int64_t round = wide || r.tiles == 4 ? 512 : 768, all = p->vocab / 64;
        r.wide = (int)(all % round < round / 2 && all > round ? all / round * round : all);
    }
    r.parts = (int)(r.wide + (p->vocab - 64 * (int64_t)r.wide + 15) / 16);
    r.stride = up_to(p->vocab, 64);
    r.steps = (p->vocab + 31) / 32;
    r.columns = (int)((p->features + 16 * each - 1) / (16 * each));
    // Wavefronts for all compute units, of four steps or tiles and more; d_hidden's leave sums behind, of which 16 MiB are
    // enough: 60 rows, 4096 features, 65536 entries, bfloat16, forward and backward, 512 wavefronts 392 us, 2048 453; 33 x 1843 x
    // 67371 float, 512 607, 1024 509, 2048 518; 6 x 3185 x 32906 bfloat16, 512 198, 2048 180.
    const int64_t summing = std::min<int64_t>(2048, (16 << 20) / (r.tiles * 16 * 16 * each * 4));
    r.splits_hidden = (int)std::max<int64_t>(1, std::min<int64_t>(summing / r.columns, r.steps / 4));
    r.splits_weight = (int)std::max<int64_t>(1, std::min<int64_t>(4096 / r.columns, r.steps / 2));
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += up256(bytes);
        return here;
    };
    const size_t rows = (size_t)p->rows, row_steps = (size_t)(r.tiles + 1) / 2;
    r.scalars = take(sizeof(XentScalars));
    r.index = take(rows * 4);
    r.position = take(rows * 4);
    r.label = take(rows * 4);
    r.lse = take(rows * 4);
    r.by_feature = take((size_t)((p->features + chunk - 1) / chunk) * chunk_frags * r.tiles * 1024);
    r.by_row = take((size_t)r.columns * row_steps * planes * each * 1024);
    r.logits = take(rows * r.stride * 4);
    r.kept = at;
    at = 0;
    if (!backward) {
        r.losses = take(rows * 4);
        r.partial = take(rows * r.parts * sizeof(float2));
    } else {
        r.d_by_entry = take((size_t)r.steps * planes * r.tiles * 1024);
        r.d_by_row = take((size_t)r.steps * 2 * row_steps * planes * 1024);
        r.sums = take((size_t)r.splits_hidden * rows * p->features * 4);
    }
    r.total = at;
    return r;
}

size_t kept_bytes_of(const bf_linear_xent *p) { return few_rows(p) ? few_plan(p, false).kept : plan(p, false).kept; }
size_t workspace_bytes_of(const bf_linear_xent *p, bool backward)
{
    return few_rows(p) ? few_plan(p, backward).total : plan(p, backward).total;
}

template <typename Plan>
int check_memory(const Plan &r, const void *weight, const void *kept, size_t kept_bytes, const void *workspace, size_t bytes)
{
    if (!kept || kept_bytes < r.kept)
        return fail(BF_ERR_WORKSPACE, "room for %zu bytes of kept operands needed, %zu given", r.kept, kept ? kept_bytes : 0);
    if (reinterpret_cast<uintptr_t>(kept) & 255) return fail(BF_ERR_WORKSPACE, "the kept operands must be 256-byte aligned");
    if (reinterpret_cast<uintptr_t>(weight) & 15) return fail(BF_ERR_INVALID, "weight must be 16-byte aligned");
    if (!workspace || bytes < r.total)
        return fail(BF_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", r.total, workspace ? bytes : 0);
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return fail(BF_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    return BF_OK;
}

template <typename T>
T *part(void *workspace, size_t offset)
{
    return reinterpret_cast<T *>(static_cast<char *>(workspace) + offset);
}

void pack(const bf_linear_xent *p, const void *x, char *out, int64_t out_rows, int64_t rows, int64_t x_stride, int64_t stride,
          size_t plane, const int *index, XentScalars *scalars, int which, hipStream_t s)
{
    if (p->dtype == BF_F32 && rows > 0) {
        unsigned *largest = which ? &scalars->weight_max : &scalars->hidden_max;
        xent_largest_kernel<<<dim3((unsigned)std::min<int64_t>((rows * ((p->features + 7) / 8) + 1023) / 1024, 1024)), dim3(256), 0, s>>>(
            static_cast<const float *>(x), rows, p->features, x_stride, index, scalars, largest);
    }
    const XentPackArgs a = {x, out, out_rows, p->features, x_stride, stride, (int64_t)plane, index, scalars, which};
    const int64_t units = out_rows * (stride / 16);
    const dim3 grid((unsigned)std::min<int64_t>((units + 255) / 256, 8192));
    if (p->dtype == BF_F32) xent_pack_kernel<float><<<grid, dim3(256), 0, s>>>(a);
    else xent_pack_kernel<bf16><<<grid, dim3(256), 0, s>>>(a);
}

// Hidden and weight as the products read them: what prepare() made of them, or weight itself.
void operands(const bf_linear_xent *p, const XentPlan &r, const void *weight, void *kept, MatOperand &h, MatOperand &w)
{
    char *hp = part<char>(kept, r.hidden), *wp = part<char>(kept, r.weight);
    const int64_t stride = r.features_up * 2;
    h = {hp, (int64_t)r.hidden_plane, stride, r.rows_up * stride, kWholeTail};
    if (weight_in_place(p))
        w = {static_cast<const char *>(weight), 0, p->weight_stride * 2, ((p->vocab - 1) * p->weight_stride + p->features) * 2,
             p->features % kMatK ? (int)(p->features % kMatK) * 2 : kWholeTail};
    else
        w = {wp, (int64_t)r.weight_plane, stride, p->vocab * stride, kWholeTail};
}

// The counted rows, and both operands in that form, for both directions.
void prepare(const bf_linear_xent *p, const XentPlan &r, const void *hidden, const void *weight, const int64_t *target, void *kept,
             float *picked, hipStream_t s)
{
    XentScalars *scalars = part<XentScalars>(kept, r.scalars);
    const XentRowsArgs rows = {target, p->rows, p->vocab, p->ignore_index, scalars, part<int>(kept, r.index),
                               part<int>(kept, r.position), part<int>(kept, r.label), picked};
    xent_rows_kernel<<<dim3(1), dim3(kXentThreads), 0, s>>>(rows);
    const int64_t stride = r.features_up * 2;
    pack(p, hidden, part<char>(kept, r.hidden), r.rows_up, p->rows, p->hidden_stride, stride, r.hidden_plane,
         part<int>(kept, r.index), scalars, 0, s);
    if (!weight_in_place(p))
        pack(p, weight, part<char>(kept, r.weight), p->vocab, p->vocab, p->weight_stride, stride, r.weight_plane, nullptr, scalars, 1, s);
}

template <bool F16, bool BACKWARD>
void launch_logits(const Product &r, const XentTileArgs &a, hipStream_t s)
{
    const dim3 grid(workgroups(r)), threads(r.large ? mat_threads(256, 256, 2) : mat_threads(128, 128, r.deep ? 4 : 2));
    if (r.large) xent_logits_kernel<F16, 256, 256, 2, BACKWARD><<<grid, threads, 0, s>>>(a);
    else if (r.deep) xent_logits_kernel<F16, 128, 128, 4, BACKWARD><<<grid, threads, 0, s>>>(a);
    else xent_logits_kernel<F16, 128, 128, 2, BACKWARD><<<grid, threads, 0, s>>>(a);
}

template <typename T, MatLayout LB>
void launch_grad(const Product &r, const XentGradArgs &a, hipStream_t s)
{
    const dim3 grid(workgroups(r)), threads(r.large ? mat_threads(256, 256, 2) : mat_threads(128, 128, r.deep ? 4 : 2));
    if (r.large) xent_grad_kernel<T, LB, 256, 256, 2><<<grid, threads, 0, s>>>(a);
    else if (r.deep) xent_grad_kernel<T, LB, 128, 128, 4><<<grid, threads, 0, s>>>(a);
    else xent_grad_kernel<T, LB, 128, 128, 2><<<grid, threads, 0, s>>>(a);
}

template <MatLayout LB>
void launch_grad(const bf_linear_xent *p, const Product &r, const XentGradArgs &a, hipStream_t s)
{
    if (p->dtype == BF_F32) launch_grad<float, LB>(r, a, s);
    else launch_grad<bf16, LB>(r, a, s);
}

template <typename T, bool SCALED>
void gather_runs(const XentGatherArgs &a, hipStream_t s)
{
    const dim3 grid((unsigned)((a.m + 127) / 128), (unsigned)std::min<int64_t>(a.rows, 4096));
    xent_gather_runs_kernel<T, SCALED><<<grid, dim3(1024), 0, s>>>(a);
}

void gather(const bf_linear_xent *p, const XentGatherArgs &a, hipStream_t s)
{
    if (a.position && a.splits >= 16) {
        if (p->dtype == BF_F32) gather_runs<float, true>(a, s);
        else gather_runs<bf16, false>(a, s);
        return;
    }
    const int64_t units = a.rows * ((a.m + 7) / 8);
    const dim3 grid((unsigned)std::min<int64_t>((units + 255) / 256, 8192));
    if (p->dtype == BF_F32) xent_gather_kernel<float><<<grid, dim3(256), 0, s>>>(a);
    else xent_gather_kernel<bf16><<<grid, dim3(256), 0, s>>>(a);
}

template <typename T, int NT>
void few_fw(const bf_linear_xent *p, const XentFewPlan &r, const void *hidden, const void *weight, const int64_t *target, float *loss,
            void *kept, void *workspace, hipStream_t s)
{
    XentScalars *scalars = part<XentScalars>(kept, r.scalars);
    int *index = part<int>(kept, r.index), *position = part<int>(kept, r.position), *label = part<int>(kept, r.label);
    const XentFewPackArgs pack = {hidden, target, p->hidden_stride, (int)p->rows, r.tiles, (int)p->features, p->vocab, p->ignore_index,
                                  scalars, index, position, label, part<char>(kept, r.by_feature), part<char>(kept, r.by_row)};
    const size_t slots = (r.logits - r.by_feature) / 16;   // (an upper bound of the threads with work)
    xent_few_pack_kernel<T><<<dim3((unsigned)std::min<size_t>((slots + kFewThreads - 1) / kFewThreads, 1024)), dim3(kFewThreads), 0, s>>>(pack);
    float *logits = part<float>(kept, r.logits);
    float2 *partial = part<float2>(workspace, r.partial);
    const XentFewLogitsArgs l = {weight, p->weight_stride, p->vocab, (int)p->features, r.parts, r.wide, scalars,
                                 part<char>(kept, r.by_feature), logits, r.stride, partial};
    if (r.wide > 0) xent_few_logits_kernel<T, NT><<<dim3((unsigned)r.parts), dim3(kFewThreads), 0, s>>>(l);
    else xent_few_narrow_logits_kernel<T, NT><<<dim3((unsigned)r.parts), dim3(kFewThreads), 0, s>>>(l);
    float *losses = p->reduction == BF_XENT_NONE ? loss : part<float>(workspace, r.losses);
    const XentFewJoinArgs j = {partial, logits, r.stride, index, position, label, scalars, r.parts, part<float>(kept, r.lse), losses};
    xent_few_join_kernel<<<dim3((unsigned)p->rows), dim3(kFewThreads), 0, s>>>(j);
    if (p->reduction != BF_XENT_NONE)
        xent_total_kernel<<<dim3(1), dim3(kXentThreads), 0, s>>>(losses, p->rows, scalars, p->reduction == BF_XENT_MEAN, loss);
}

template <typename T, int NT>
void few_bw(const bf_linear_xent *p, const XentFewPlan &r, const void *weight, const float *grad, void *kept, void *d_hidden,
            void *d_weight, void *workspace, hipStream_t s)
{
    const XentScalars *scalars = part<XentScalars>(kept, r.scalars);
    const XentGrad gradient = {grad, p->reduction == BF_XENT_NONE, p->reduction == BF_XENT_MEAN};
    char *by_entry = d_hidden ? part<char>(workspace, r.d_by_entry) : nullptr, *by_row = d_weight ? part<char>(workspace, r.d_by_row) : nullptr;
    const XentFewDlArgs d = {part<float>(kept, r.logits), r.stride, p->vocab, part<float>(kept, r.lse), part<int>(kept, r.index),
                             part<int>(kept, r.label), scalars, gradient, by_entry, by_row};
    xent_few_dl_kernel<T, NT><<<dim3((unsigned)r.steps), dim3(64 * NT), 0, s>>>(d);
    XentFewGradArgs g = {};
    g.weight = weight;
    g.weight_stride = p->weight_stride;
    g.vocab = p->vocab;
    g.features = (int)p->features;
    g.rows = (int)p->rows;
    g.scalars = scalars;
    g.grad = gradient;
    g.by_entry = by_entry;
    g.by_row = by_row;
    g.hidden = part<char>(kept, r.by_row);
    g.parts = r.columns;
    g.splits_hidden = r.splits_hidden;
    g.splits_weight = r.splits_weight;
    g.blocks_hidden = d_hidden ? (r.columns * r.splits_hidden + 3) / 4 : 0;
    g.partial = part<float>(workspace, r.sums);
    g.d_weight = d_weight;
    const int blocks_weight = d_weight ? (r.columns * r.splits_weight + 3) / 4 : 0;
    xent_few_grad_kernel<T, NT><<<dim3((unsigned)(g.blocks_hidden + blocks_weight)), dim3(kFewThreads), 0, s>>>(g);
    if (!d_hidden) return;
    gather_runs<T, false>({g.partial, part<int>(kept, r.position), scalars, gradient, d_hidden, p->rows, p->rows, p->features, r.splits_hidden, 0,
                           nullptr}, s);
}

// f(the type, tiles of rows) of a call
template <typename Call>
void few_dispatch(const bf_linear_xent *p, const XentFewPlan &r, Call &&call)
{
    auto typed = [&](auto type) {
        if (r.tiles == 1) call(type, std::integral_constant<int, 1>());
        else if (r.tiles == 2) call(type, std::integral_constant<int, 2>());
        else call(type, std::integral_constant<int, 4>());
    };
    if (p->dtype == BF_F32) typed(float());
    else typed(bf16());
}

}  // namespace

extern "C" {

size_t bf_linear_xent_kept_bytes(const bf_linear_xent *p)
{
    return check_xent(p) ? BF_SIZE_INVALID : kept_bytes_of(p);
}

size_t bf_linear_xent_fw_workspace_bytes(const bf_linear_xent *p)
{
    return check_xent(p) ? BF_SIZE_INVALID : workspace_bytes_of(p, false);
}

size_t bf_linear_xent_bw_workspace_bytes(const bf_linear_xent *p)
{
    return check_xent(p) ? BF_SIZE_INVALID : workspace_bytes_of(p, true);
}

int bf_linear_xent_fw(const bf_linear_xent *p, const void *hidden, const void *weight, const int64_t *target, float *loss,
                      void *kept, size_t kept_bytes, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_xent(p);
    if (rc) return rc;
    if (p->rows > 0 && (!hidden || !target)) return fail(BF_ERR_INVALID, "hidden or target is NULL");
    if (!weight || (!loss && (p->rows > 0 || p->reduction != BF_XENT_NONE))) return fail(BF_ERR_INVALID, "weight or loss is NULL");
    if (p->rows == 0 && p->reduction == BF_XENT_NONE) return BF_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (few_rows(p)) {
        const XentFewPlan r = few_plan(p, false);
        if ((rc = check_memory(r, weight, kept, kept_bytes, workspace, workspace_bytes))) return rc;
        few_dispatch(p, r, [&](auto type, auto tiles) {
            few_fw<decltype(type), decltype(tiles)::value>(p, r, hidden, weight, target, loss, kept, workspace, s);
        });
        BF_HIP_CHECK(hipGetLastError());
        return BF_OK;
    }
    const XentPlan r = plan(p, false);
    if ((rc = check_memory(r, weight, kept, kept_bytes, workspace, workspace_bytes))) return rc;
    MatOperand h, w;
    float *picked = part<float>(workspace, r.picked);
    prepare(p, r, hidden, weight, target, kept, picked, s);
    operands(p, r, weight, kept, h, w);
    XentScalars *scalars = part<XentScalars>(kept, r.scalars);
    float *losses = p->reduction == BF_XENT_NONE ? loss : part<float>(workspace, r.losses);
    if (p->rows > 0) {
        XentTileArgs a = {};
        a.weight = w;
        a.hidden = h;
        a.scalars = scalars;
        a.label = part<int>(kept, r.label);
        a.rows = p->rows;
        a.vocab = p->vocab;
        a.features_steps = (int)(r.features_up / kMatK);
        a.tiles_m = r.logits.tiles_m;
        a.tiles_n = r.logits.tiles_n;
        a.partial = part<float2>(workspace, r.partial);
        a.picked = picked;
        if (p->dtype == BF_F32) launch_logits<true, false>(r.logits, a, s);
        else launch_logits<false, false>(r.logits, a, s);
        const XentJoinArgs j = {a.partial, picked, part<int>(kept, r.position), part<int>(kept, r.label), p->rows, 2 * r.logits.tiles_m,
                                part<float>(kept, r.lse), losses};
        xent_join_kernel<<<dim3((unsigned)((p->rows + 7) / 8)), dim3(1024), 0, s>>>(j);
    }
    if (p->reduction != BF_XENT_NONE)
        xent_total_kernel<<<dim3(1), dim3(kXentThreads), 0, s>>>(losses, p->rows, scalars, p->reduction == BF_XENT_MEAN, loss);
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

int bf_linear_xent_bw(const bf_linear_xent *p, const void *weight, const float *grad, void *kept, size_t kept_bytes, void *d_hidden,
                      void *d_weight, void *workspace, size_t workspace_bytes, void *stream)
{
    int rc = check_xent(p);
    if (rc) return rc;
    if (!weight || (!grad && (p->rows > 0 || p->reduction != BF_XENT_NONE))) return fail(BF_ERR_INVALID, "weight or grad is NULL");
    if (!d_hidden && !d_weight) return BF_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->rows == 0) {   // (the forward call has left nothing in `kept`)
        const int64_t count = p->vocab * p->features;
        const dim3 grid((unsigned)std::min<int64_t>((count + 255) / 256, 8192));
        if (d_weight && p->dtype == BF_F32) xent_zero_kernel<<<grid, dim3(256), 0, s>>>(static_cast<float *>(d_weight), count);
        else if (d_weight) xent_zero_kernel<<<grid, dim3(256), 0, s>>>(static_cast<bf16 *>(d_weight), count);
        BF_HIP_CHECK(hipGetLastError());
        return BF_OK;
    }
    if (few_rows(p)) {
        const XentFewPlan r = few_plan(p, true);
        if ((rc = check_memory(r, weight, kept, kept_bytes, workspace, workspace_bytes))) return rc;
        few_dispatch(p, r, [&](auto type, auto tiles) {
            few_bw<decltype(type), decltype(tiles)::value>(p, r, weight, grad, kept, d_hidden, d_weight, workspace, s);
        });
        BF_HIP_CHECK(hipGetLastError());
        return BF_OK;
    }
    const XentPlan r = plan(p, true);
    if ((rc = check_memory(r, weight, kept, kept_bytes, workspace, workspace_bytes))) return rc;
    MatOperand h, w;
    operands(p, r, weight, kept, h, w);
    XentScalars *scalars = part<XentScalars>(kept, r.scalars);
    const XentGrad gradient = {grad, p->reduction == BF_XENT_NONE, p->reduction == BF_XENT_MEAN};
    if (gradient.each)
        xent_share_kernel<<<dim3(1), dim3(kXentThreads), 0, s>>>(gradient, part<int>(kept, r.index), scalars,
                                                                 part<float>(workspace, r.share));
    const bool shared = gradient.each && p->dtype == BF_F32;
    MatOperand rows = h;   // hidden as d_weight's product takes it
    if (shared && d_weight) {
        rows.base = part<char>(workspace, r.shared);
        const XentSharedArgs a = {h.base, part<char>(workspace, r.shared), r.rows_up, h.stride, h.plane, part<float>(workspace, r.share), scalars};
        xent_shared_kernel<<<dim3((unsigned)std::min<int64_t>((r.rows_up * (h.stride / 16) + 255) / 256, 8192)), dim3(256), 0, s>>>(a);
    }
    const size_t elem = p->dtype == BF_F32 ? 4 : 2;
    char *d_l = part<char>(workspace, r.d_l);
    const int64_t d_l_stride = r.piece * 2;
    const MatOperand d_l_operand = {d_l, (int64_t)r.d_l_plane, d_l_stride, r.rows_up * d_l_stride, kWholeTail};
    for (int64_t first = 0; first < p->vocab; first += r.piece) {
        const int64_t entries = std::min<int64_t>(r.piece, p->vocab - first);
        MatOperand wp = w;
        wp.base += first * w.stride;
        wp.bytes -= first * w.stride;
        XentTileArgs a = {};
        a.weight = wp;
        a.hidden = h;
        a.scalars = scalars;
        a.label = part<int>(kept, r.label);
        a.rows = p->rows;
        a.vocab = entries;
        a.first = first;
        a.features_steps = (int)(r.features_up / kMatK);
        Product logits = r.logits;   // (a shorter last piece: fewer tiles of the same size)
        const int64_t side = logits.large ? 256 : 128;
        logits.tiles_m = (int)((entries + side - 1) / side);
        a.tiles_m = logits.tiles_m;
        a.tiles_n = logits.tiles_n;
        a.lse = part<float>(kept, r.lse);
        a.share = gradient.each ? part<float>(workspace, r.share) : nullptr;
        a.d_l = d_l;
        a.stride = d_l_stride;
        a.plane = (int64_t)r.d_l_plane;
        if (p->dtype == BF_F32) launch_logits<true, true>(logits, a, s);
        else launch_logits<false, true>(logits, a, s);
        if (d_hidden) {
            XentGradArgs g = {};
            g.a = wp;
            g.b = d_l_operand;
            g.scalars = scalars;
            g.grad = gradient;
            g.m = p->features;
            g.n = p->rows;
            g.tiles_m = r.to_hidden.tiles_m;
            g.tiles_n = r.to_hidden.tiles_n;
            g.steps = (int)((entries + kMatK - 1) / kMatK);
            g.splits = r.to_hidden.splits;
            g.add = first > 0;
            g.partial = part<float>(workspace, r.sums_hidden);
            launch_grad<kRows>(p, r.to_hidden, g, s);
        }
        if (d_weight) {
            XentGradArgs g = {};
            Product to_weight = r.to_weight;
            const int64_t t = to_weight.large ? 256 : 128;
            to_weight.tiles_n = (int)((entries + t - 1) / t);
            g.a = rows;
            g.b = d_l_operand;
            g.scalars = scalars;
            g.grad = gradient;
            g.m = p->features;
            g.n = entries;
            g.tiles_m = to_weight.tiles_m;
            g.tiles_n = to_weight.tiles_n;
            g.splits = to_weight.splits;
            char *out = static_cast<char *>(d_weight) + (size_t)first * p->features * elem;
            if (g.splits > 1) g.partial = part<float>(workspace, r.sums_weight);
            else g.out = out;
            launch_grad<kCols>(p, to_weight, g, s);
            if (g.splits > 1)
                gather(p, {g.partial, nullptr, scalars, gradient, out, entries, entries, p->features, g.splits, 1, nullptr}, s);
        }
    }
    if (d_hidden)
        gather(p, {part<float>(workspace, r.sums_hidden), part<int>(kept, r.position), scalars, gradient, d_hidden, p->rows, p->rows,
                   p->features, r.to_hidden.splits, 0, shared ? grad : nullptr}, s);
    BF_HIP_CHECK(hipGetLastError());
    return BF_OK;
}

}  // extern "C"
