// C-ABI of the norms around a block: argument validation, before any HIP call, and the launches.
#include "../../include/nmspmm.h"
#include "internal.h"

using namespace nmspmm;

namespace {

constexpr int kMaxFeatures = 16384;
constexpr long long kMaxRows = 1ll << 31;

bool is_type(int t) { return t == NMSPMM_F32 || t == NMSPMM_BF16 || t == NMSPMM_F16; }
size_t size_of(int t) { return t == NMSPMM_F32 ? 4 : 2; }
bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
bool is_kind(int k) { return k == NMSPMM_NORM_NONE || k == NMSPMM_NORM_RMS || k == NMSPMM_NORM_LAYER; }

int check(const nmspmm_block_norm* b, BlockNormArgs* a)
{
    if (!b)
        return NMSPMM_ERR_NULL_POINTER;
    if (!is_type(b->type) || (b->residual_type != b->type && b->residual_type != NMSPMM_F32) || !is_kind(b->post) || !is_kind(b->pre))
        return NMSPMM_ERR_BAD_PATTERN;
    if (b->rows < 0 || b->rows >= kMaxRows || b->features <= 0 || b->features > kMaxFeatures || !(b->eps >= 0.0f))
        return NMSPMM_ERR_BAD_SHAPE;
    if (b->gate && (b->gate_rows <= 0 || b->rows % b->gate_rows != 0))
        return NMSPMM_ERR_BAD_SHAPE;
    const long long D = b->features;
    if (b->ld_residual < D || (b->branch && (b->ld_branch < D || b->ld_sum < D)) || (b->out && b->ld_out < D))
        return NMSPMM_ERR_BAD_SHAPE;
    // what belongs to something that is not there
    if ((!b->branch && (b->gate || b->scale || b->post != NMSPMM_NORM_NONE)) ||
        (b->post == NMSPMM_NORM_NONE && (b->post_weight || b->post_bias)) ||
        (b->pre == NMSPMM_NORM_NONE && (b->pre_weight || b->pre_bias)) || (!b->out && b->pre != NMSPMM_NORM_NONE))
        return NMSPMM_ERR_BAD_PATTERN;
    if (b->rows > 0 && (!b->residual || (b->branch && !b->sum) || (!b->branch && !b->out)))
        return NMSPMM_ERR_NULL_POINTER;
    const size_t t = size_of(b->type), r = size_of(b->residual_type);
    if (!aligned(b->residual, r) || !aligned(b->sum, r) || !aligned(b->branch, t) || !aligned(b->out, t) || !aligned(b->stats, 16))
        return NMSPMM_ERR_ALIGNMENT;
    const void* const data[6] = {b->gate, b->scale, b->post_weight, b->post_bias, b->pre_weight, b->pre_bias};
    const int type[6] = {b->gate_type, b->scale_type, b->post_weight_type, b->post_bias_type, b->pre_weight_type, b->pre_bias_type};
    BlockNormVec* const to[6] = {&a->gate, &a->scale, &a->post_weight, &a->post_bias, &a->pre_weight, &a->pre_bias};
    for (int i = 0; i < 6; ++i) {
        if (data[i] && !is_type(type[i]))
            return NMSPMM_ERR_BAD_PATTERN;
        if (data[i] && !aligned(data[i], size_of(type[i])))
            return NMSPMM_ERR_ALIGNMENT;
        to[i]->data = data[i];
        to[i]->type = data[i] ? type[i] : NMSPMM_F32;
    }
    a->rows = (size_t)b->rows;
    a->D = b->features;
    a->residual = b->residual;
    a->branch = b->branch;
    a->sum = b->sum;
    a->out = b->out;
    a->stats = b->stats;
    a->ld_residual = (size_t)b->ld_residual;
    a->ld_branch = (size_t)b->ld_branch;
    a->ld_sum = (size_t)b->ld_sum;
    a->ld_out = (size_t)b->ld_out;
    a->gate_rows = (size_t)(b->gate ? b->gate_rows : b->rows > 0 ? b->rows : 1);
    a->factor = b->factor;
    a->eps = b->eps;
    a->weight_offset = b->weight_offset;
    a->post = b->post;
    a->pre = b->pre;
    return NMSPMM_OK;
}

} // namespace

extern "C" {

int nmspmm_block_norm_forward(const nmspmm_block_norm* b, void* stream)
{
    BlockNormArgs a;
    const int st = check(b, &a);
    if (st != NMSPMM_OK || b->rows == 0)
        return st;
    return launch_block_norm(a, b->type, b->residual_type, (hipStream_t)stream) == hipSuccess ? NMSPMM_OK : NMSPMM_ERR_HIP;
}

size_t nmspmm_block_norm_workspace_bytes(long long rows, long long gate_rows, int features)
{
    if (rows <= 0 || rows >= kMaxRows || gate_rows <= 0 || rows % gate_rows != 0 || features <= 0 || features > kMaxFeatures)
        return 0;
    return (size_t)block_norm_walk(rows, gate_rows, features).walkers * features * 6 * sizeof(float);
}

int nmspmm_block_norm_backward(const nmspmm_block_norm* b, const nmspmm_block_norm_grads* g, void* workspace,
                               size_t workspace_bytes, void* stream)
{
    BlockNormArgs a;
    if (!g)
        return NMSPMM_ERR_NULL_POINTER;
    // `sum` and `out` of the forward pass are not read: only whether there was an `out` counts
    const int st = check(b, &a);
    if (st != NMSPMM_OK)
        return st;
    const long long D = b->features;
    if (b->rows == 0 || (g->sum && g->ld_sum < D) || (g->out && g->ld_out < D) || (g->residual && g->ld_residual < D) ||
        (g->branch && g->ld_branch < D))
        return NMSPMM_ERR_BAD_SHAPE;
    if (!b->stats)
        return NMSPMM_ERR_NULL_POINTER;
    if ((g->out && !b->out) || (g->branch && !b->branch) || (g->gate && !b->gate) || (g->scale && !b->scale) ||
        (g->post_weight && !b->post_weight) || (g->post_bias && !b->post_bias) || (g->pre_weight && !b->pre_weight) ||
        (g->pre_bias && !b->pre_bias))
        return NMSPMM_ERR_BAD_PATTERN;
    const size_t t = size_of(b->type), r = size_of(b->residual_type);
    if (!aligned(g->sum, r) || !aligned(g->residual, r) || !aligned(g->out, t) || !aligned(g->branch, t) ||
        !aligned(g->gate, size_of(a.gate.type)) || !aligned(g->scale, size_of(a.scale.type)) ||
        !aligned(g->post_weight, size_of(a.post_weight.type)) || !aligned(g->post_bias, size_of(a.post_bias.type)) ||
        !aligned(g->pre_weight, size_of(a.pre_weight.type)) || !aligned(g->pre_bias, size_of(a.pre_bias.type)) || !aligned(workspace, 16))
        return NMSPMM_ERR_ALIGNMENT;
    if (!workspace || workspace_bytes < nmspmm_block_norm_workspace_bytes(b->rows, (long long)a.gate_rows, b->features))
        return NMSPMM_ERR_WORKSPACE;
    BlockNormGrads d = {};
    d.sum = g->sum;
    d.out = g->out;
    d.residual = g->residual;
    d.branch = g->branch;
    d.ld_sum = (size_t)g->ld_sum;
    d.ld_out = (size_t)g->ld_out;
    d.ld_residual = (size_t)g->ld_residual;
    d.ld_branch = (size_t)g->ld_branch;
    d.gate = g->gate;
    d.scale = g->scale;
    d.post_weight = g->post_weight;
    d.post_bias = g->post_bias;
    d.pre_weight = g->pre_weight;
    d.pre_bias = g->pre_bias;
    d.partial = (float*)workspace;
    return launch_block_norm_backward(a, d, b->type, b->residual_type, (hipStream_t)stream) == hipSuccess ? NMSPMM_OK : NMSPMM_ERR_HIP;
}

} // extern "C"
