// C-ABI of the 4-bit operands: argument validation, before any HIP call, and the launches.
#include "../../include/nmspmm.h"
#include "internal.h"

using namespace nmspmm;

namespace {

bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// The geometry of an operand, or the reason why there is none.
int q4_shape(int K, int N, int n, int m, int group, Q4Shape* p)
{
    if (group != 32 && group != 64 && group != 128)
        return NMSPMM_ERR_BAD_PATTERN;
    if (n <= 0 || m < n)
        return NMSPMM_ERR_BAD_PATTERN;
    if (n != m && ((n != 1 && n != 2 && n != 4 && n != 8) || (m != 2 * n && m != 4 * n && m != 8 * n)))
        return NMSPMM_ERR_BAD_PATTERN;
    if (K <= 0 || N <= 0 || K > (1 << 22) || N > (1 << 20))
        return NMSPMM_ERR_BAD_SHAPE;
    if (n != m && (K % m != 0 || N % 32 != 0))
        return NMSPMM_ERR_BAD_SHAPE;
    p->K = K;
    p->N = N;
    p->n = n == m ? 1 : n;
    p->m = n == m ? 1 : m;
    p->W = K / p->m * p->n;
    p->group = group;
    p->blocks = (p->W + 127) / 128;
    p->tiles = (N + 31) / 32 * 2;
    p->span = 32 * p->m / p->n;
    return NMSPMM_OK;
}

size_t q4_blocks(const Q4Shape& p) { return (size_t)p.tiles * p.blocks; }

int check_operand(const nmspmm_q4_operand* op, Q4Shape* p)
{
    if (!op)
        return NMSPMM_ERR_NULL_POINTER;
    const int st = q4_shape(op->K, op->N, op->n, op->m, op->group, p);
    if (st != NMSPMM_OK)
        return st;
    if (!op->codes || !op->meta || (p->m > 1 && !op->row_offsets))
        return NMSPMM_ERR_NULL_POINTER;
    if (!aligned(op->codes, 16) || !aligned(op->meta, 16) || !aligned(op->row_offsets, 16) || !aligned(op->bias, 4))
        return NMSPMM_ERR_ALIGNMENT;
    return NMSPMM_OK;
}

const uint8_t* offsets_of(const nmspmm_q4_operand* op, const Q4Shape& p)
{
    return p.m > 1 ? static_cast<const uint8_t*>(op->row_offsets) : nullptr;
}

} // namespace

extern "C" {

size_t nmspmm_q4_codes_bytes(int K, int N, int n, int m)
{
    Q4Shape p;
    return q4_shape(K, N, n, m, 128, &p) == NMSPMM_OK ? q4_blocks(p) * 1024 : 0;
}

size_t nmspmm_q4_meta_bytes(int K, int N, int n, int m, int group)
{
    Q4Shape p;
    return q4_shape(K, N, n, m, group, &p) == NMSPMM_OK ? q4_blocks(p) * 64 * (128 / group) : 0;
}

size_t nmspmm_q4_row_offsets_bytes(int K, int N, int n, int m)
{
    Q4Shape p;
    return q4_shape(K, N, n, m, 128, &p) == NMSPMM_OK && p.m > 1 ? (size_t)(N / 32) * p.blocks * 128 : 0;
}

size_t nmspmm_q4_workspace_bytes(int M, int K, int N, int n, int m, int type)
{
    Q4Shape p;
    if (M <= 0 || M > (1 << 24) || (type != NMSPMM_F32 && type != NMSPMM_BF16 && type != NMSPMM_F16) ||
        q4_shape(K, N, n, m, 32, &p) != NMSPMM_OK)     // (the group is not known here: groups of 32 take no less than larger ones)
        return 0;
    return q4_workspace_bytes(p, M, (ElementType)type);
}

int nmspmm_q4_quantize_device(const float* dBT, const int32_t* dDT, const nmspmm_q4_operand* op, unsigned flags, void* stream)
{
    Q4Shape p;
    const int st = check_operand(op, &p);
    if (st != NMSPMM_OK)
        return st;
    if (!dBT || (p.m > 1 && !dDT))
        return NMSPMM_ERR_NULL_POINTER;
    if (flags & ~NMSPMM_Q4_ASYMMETRIC)
        return NMSPMM_ERR_BAD_SHAPE;
    if (!aligned(dBT, 4) || !aligned(dDT, 4))
        return NMSPMM_ERR_ALIGNMENT;
    return launch_q4_pack(dBT, nullptr, nullptr, nullptr, p.m > 1 ? dDT : nullptr, p, (flags & NMSPMM_Q4_ASYMMETRIC) != 0,
                          (uint32_t*)op->codes, (uint32_t*)op->meta, (uint8_t*)op->row_offsets,
                          (hipStream_t)stream) == hipSuccess ? NMSPMM_OK : NMSPMM_ERR_HIP;
}

int nmspmm_q4_pack_device(const uint8_t* d_codes, const float* d_scales, const uint8_t* d_zeros, const int32_t* dDT,
                          const nmspmm_q4_operand* op, void* stream)
{
    Q4Shape p;
    const int st = check_operand(op, &p);
    if (st != NMSPMM_OK)
        return st;
    if (!d_codes || !d_scales || (p.m > 1 && !dDT))
        return NMSPMM_ERR_NULL_POINTER;
    if (!aligned(d_scales, 4) || !aligned(dDT, 4))
        return NMSPMM_ERR_ALIGNMENT;
    return launch_q4_pack(nullptr, d_codes, d_scales, d_zeros, p.m > 1 ? dDT : nullptr, p, false, (uint32_t*)op->codes,
                          (uint32_t*)op->meta, (uint8_t*)op->row_offsets,
                          (hipStream_t)stream) == hipSuccess ? NMSPMM_OK : NMSPMM_ERR_HIP;
}

int nmspmm_q4_expand_device(const nmspmm_q4_operand* op, float* dB, void* stream)
{
    Q4Shape p;
    const int st = check_operand(op, &p);
    if (st != NMSPMM_OK)
        return st;
    if (!dB)
        return NMSPMM_ERR_NULL_POINTER;
    if (!aligned(dB, 4))
        return NMSPMM_ERR_ALIGNMENT;
    return launch_q4_expand((const uint32_t*)op->codes, (const uint32_t*)op->meta, offsets_of(op, p), p, dB,
                            (hipStream_t)stream) == hipSuccess ? NMSPMM_OK : NMSPMM_ERR_HIP;
}

int nmspmm_q4_linear(const nmspmm_q4_operand* op, const void* x, long long ldx, void* y, long long ldy, int M, int type,
                     void* workspace, size_t workspace_bytes, void* stream)
{
    Q4Shape p;
    const int st = check_operand(op, &p);
    if (st != NMSPMM_OK)
        return st;
    if (type != NMSPMM_F32 && type != NMSPMM_BF16 && type != NMSPMM_F16)
        return NMSPMM_ERR_BAD_PATTERN;
    if (M < 0 || M > (1 << 24) || ldx < p.K || ldy < p.N || ldx > (1 << 24) || ldy > (1 << 24))
        return NMSPMM_ERR_BAD_SHAPE;
    if (M == 0)
        return NMSPMM_OK;
    if (!x || !y)
        return NMSPMM_ERR_NULL_POINTER;
    const size_t size = type == NMSPMM_F32 ? 4 : 2;
    if (!aligned(x, size) || !aligned(y, size))
        return NMSPMM_ERR_ALIGNMENT;
    const size_t need = q4_workspace_bytes(p, M, (ElementType)type);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return NMSPMM_ERR_WORKSPACE;
    if (need > 0 && !aligned(workspace, 16))
        return NMSPMM_ERR_ALIGNMENT;
    Q4LinearArgs a;
    a.x = x;
    a.codes = (const uint32_t*)op->codes;
    a.meta.words = (const uint32_t*)op->meta;
    a.meta.blocks = p.blocks;
    a.meta.per = 128 / p.group;
    a.meta.per_shift = p.group == 128 ? 0 : p.group == 64 ? 1 : 2;
    a.meta.group = p.group;
    a.meta.group_shift = p.group == 128 ? 7 : p.group == 64 ? 6 : 5;
    a.meta.last = (p.W - 1) / p.group;
    a.rows = offsets_of(op, p);
    a.bias = op->bias;
    a.y = y;
    a.ldx = (size_t)ldx;
    a.ldy = (size_t)ldy;
    a.M = M;
    a.p = p;
    a.stream = (hipStream_t)stream;
    return launch_q4_linear(a, (ElementType)type, workspace) == hipSuccess ? NMSPMM_OK : NMSPMM_ERR_HIP;
}

} // extern "C"
