// Compressed operands in 4 bits.  The kept values of an N:M-compressed operand B (W = K*n/m rows, N
// columns; n = m: an ordinary dense matrix) are whole numbers 0..15 with a scale and a zero point
// for each group of 32, 64 or 128 kept rows of a column:
//     b[r][c] = scale[j][c] * (code[r][c] - zero[j][c]),  j = r / group.
// A scale has 20 significant bits, so scale * (code - zero) is exact in fp32 (24 bits).
//
// Layout, made once when a layer is loaded (there is none in the reference, whose values are fp32):
// blocks of 128 kept rows x 16 columns, 1 KB each, ordered by column tile, then block.
//   codes [tile][block][lane][4] uint32: lane 16 kb + c holds column c, word s its rows
//         32 s + 8 kb + 0..7 (a k-step of 32 rows of a matrix instruction); nibble i of the word is row
//         2 i of the eight, nibble i + 4 row 2 i + 1, so that the words of the operand registers come
//         out of one shift and one mask-and-or each.
//   meta  [tile][block][16 columns][128 / group] uint32: the scale's fp32 bits with the zero point in
//         the low four.
//   rows  [N / 32][blocks * 128] uint8 (n < m only): the dense row of each kept row, counted from the
//         first row of the windows of its k-step (32 kept rows span 32 m / n <= 256 dense rows).
// Rows beyond W and columns beyond N are filled in (the group's zero point, meta 0, offset 0).
#include "internal.h"

namespace nmspmm {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ inline int dense_row(int kept, int n, int m, int local) { return kept / n * m + local; }

// One wave packs one block: lane 16 kb + c takes the 32 rows {32 s + 8 kb + e} of column c.
// FROM_VALUES: the codes are found here, otherwise they are given.  HBM-bound: a wave instruction reads
// four 64-byte row segments whose other half the neighbouring wave of the workgroup reads.
template <bool FROM_VALUES>
__global__ void __launch_bounds__(256)
q4_pack_kernel(const float* __restrict__ values, const uint8_t* __restrict__ given, const float* __restrict__ scales,
               const uint8_t* __restrict__ zeros, const int32_t* __restrict__ rows, Q4Shape p, bool asymmetric,
               uint32_t* __restrict__ codes, uint32_t* __restrict__ meta)
{
    const int lane = threadIdx.x & 63, c = lane & 15, kb = lane >> 4;
    const int tile = blockIdx.y * 4 + (threadIdx.x >> 6), block = blockIdx.x;
    if (tile >= p.tiles)
        return;
    const int col = tile * 16 + c;
    const bool column = col < p.N;
    const int per = 128 / p.group;      // groups of a block: 1, 2 or 4
    const int row0 = block * 128 + kb * 8;
    uint32_t word[4];
    uint32_t mt[4] = {0, 0, 0, 0};

    if (FROM_VALUES) {
        float v[4][8];
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = row0 + s * 32 + e;
                v[s][e] = column && r < p.W ? __builtin_nontemporal_load(values + (size_t)r * p.N + col) : 0.0f;
            }
        // largest and smallest of each step over its 32 rows, zero among them; a NaN or an infinity
        // anywhere makes the scale NaN (the whole group then expands to NaN)
        float top[4], low[4];
        bool bad[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            top[s] = low[s] = 0.0f;
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                top[s] = fmaxf(top[s], v[s][e]);
                low[s] = fminf(low[s], v[s][e]);
                odd |= (__float_as_uint(v[s][e]) & 0x7f800000u) == 0x7f800000u;
            }
#pragma unroll
            for (int mask = 16; mask < 64; mask <<= 1) {
                top[s] = fmaxf(top[s], __shfl_xor(top[s], mask, 64));
                low[s] = fminf(low[s], __shfl_xor(low[s], mask, 64));
                odd |= __shfl_xor((int)odd, mask, 64) != 0;
            }
            bad[s] = odd;
        }
        if (per <= 2)
#pragma unroll
            for (int s = 0; s < 4; s += 2) {
                top[s] = top[s + 1] = fmaxf(top[s], top[s + 1]);
                low[s] = low[s + 1] = fminf(low[s], low[s + 1]);
                bad[s] = bad[s + 1] = bad[s] || bad[s + 1];
            }
        if (per == 1) {
            top[0] = top[1] = top[2] = top[3] = fmaxf(top[0], top[2]);
            low[0] = low[1] = low[2] = low[3] = fminf(low[0], low[2]);
            bad[0] = bad[1] = bad[2] = bad[3] = bad[0] || bad[2];
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            // the smallest scale of 20 significant bits with steps * scale >= what has to be covered
            // (steps * scale has 24 bits at most: exact, and so is the comparison, in double)
            const double steps = asymmetric ? 15.0 : 7.0;
            const double need = asymmetric ? (double)top[s] - (double)low[s] : (double)fmaxf(top[s], -low[s]);
            uint32_t bits = __float_as_uint((float)(need / steps)) & ~15u;
            if (steps * (double)__uint_as_float(bits) < need)
                bits += 16;
            const float scale = __uint_as_float(bits);
            float zero = 8.0f;
            if (asymmetric)
                zero = scale > 0.0f ? fminf(fmaxf((float)rint(-(double)low[s] / (double)scale), 0.0f), 15.0f) : 0.0f;
            if (bad[s]) {
                bits = 0x7fc00000u;
                zero = 8.0f;
            }
            mt[s] = bits | (uint32_t)zero;
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                // nearest whole number to value / scale, ties to even: the quotient of two floats can
                // round onto a half that it only comes near, so the half is compared with the value
                // itself (fma: one rounding, the sign of the difference is right)
                float q = 0.0f;
                if (scale > 0.0f && !bad[s]) {
                    const float f = floorf(v[s][e] / scale);
                    const float over = fmaf(-(f + 0.5f), scale, v[s][e]);
                    q = over > 0.0f ? f + 1.0f : over < 0.0f ? f : 2.0f * rintf(0.5f * f + 0.25f);
                }
                q = row0 + s * 32 + e < p.W ? fminf(fmaxf(q + zero, 0.0f), 15.0f) : zero;
                w |= (uint32_t)q << (4 * ((e >> 1) + 4 * (e & 1)));
            }
            word[s] = w;
        }
        const uint32_t all[4] = {mt[0], mt[1], mt[2], mt[3]};
        if (per == 2)
            mt[1] = all[2];
    } else {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int j = block * per + g;
            if (g < per && column && (size_t)j * p.group < (size_t)p.W) {
                const uint32_t z = zeros ? zeros[(size_t)j * p.N + col] : 8u;
                // 20 significant bits, to the nearest (ties away from zero; 16-bit scales are exact)
                const uint32_t bits = __float_as_uint(scales[(size_t)j * p.N + col]);
                const bool odd = (bits & 0x7f800000u) == 0x7f800000u;
                mt[g] = ((odd ? 0x7fc00000u : bits + 8u) & ~15u) | (z & 15u);
            }
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint32_t z = mt[s * per / 4] & 15u;
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = row0 + s * 32 + e;
                uint32_t q = z;      // rows beyond W count as zero
                if (column && r < p.W) {
                    q = given[(size_t)r * p.N + col] & 15u;
                    if (rows) {     // a kept row outside its window counts as zero
                        const int local = rows[(size_t)r * (p.N / 32) + (col >> 5)];
                        if (local < 0 || local >= p.m)
                            q = z;
                    }
                }
                w |= q << (4 * ((e >> 1) + 4 * (e & 1)));
            }
            word[s] = w;
        }
    }
    if (FROM_VALUES && rows) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = row0 + s * 32 + e;
                if (column && r < p.W) {
                    const int local = rows[(size_t)r * (p.N / 32) + (col >> 5)];
                    const int at = 4 * ((e >> 1) + 4 * (e & 1));
                    if (local < 0 || local >= p.m)
                        word[s] = (word[s] & ~(15u << at)) | ((mt[s * per / 4] & 15u) << at);
                }
            }
    }
    const size_t at = (size_t)tile * p.blocks + block;
    *reinterpret_cast<u32x4*>(codes + (at * 64 + lane) * 4) = u32x4{word[0], word[1], word[2], word[3]};
    if (kb == 0)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (g < per)
                meta[(at * 16 + c) * per + g] = mt[g];
}

// rows[N/32][blocks*128]: one thread per entry, consecutive threads take consecutive vectors of a row
// of DT (the reads coalesce; the bytes are written once in a model's life).
__global__ void __launch_bounds__(256)
q4_rows_kernel(const int32_t* __restrict__ rows, Q4Shape p, uint8_t* __restrict__ out)
{
    const int Q = p.N / 32;
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int r = (int)(i / Q), v = (int)(i % Q);
    if (r >= p.blocks * 128)
        return;
    int offset = 0;
    if (r < p.W) {
        int local = rows[i];
        if (local < 0 || local >= p.m) {
            // its code is the zero point: any row that the window does not keep will do
            const int first = r / p.n * p.n;
            for (local = 0; local < p.m; ++local) {
                bool kept = false;
                for (int k = 0; k < p.n; ++k)
                    kept |= rows[(size_t)(first + k) * Q + v] == local;
                if (!kept)
                    break;
            }
        }
        offset = dense_row(r, p.n, p.m, local) - (r >> 5) * p.span;
    }
    out[(size_t)v * p.blocks * 128 + r] = (uint8_t)offset;
}

// Back to the dense fp32 matrix B[K][N].  One wave per block; a lane's eight rows of a step are whole
// windows (n divides 8), so it writes all their dense rows: the kept ones and the zeros between.
template <bool SPARSE>
__global__ void __launch_bounds__(256)
q4_expand_kernel(const uint32_t* __restrict__ codes, const uint32_t* __restrict__ meta, const uint8_t* __restrict__ rows,
                 Q4Shape p, float* __restrict__ B)
{
    const int lane = threadIdx.x & 63, c = lane & 15, kb = lane >> 4;
    const int tile = blockIdx.y * 4 + (threadIdx.x >> 6), block = blockIdx.x;
    const int col = tile * 16 + c;
    if (col >= p.N)
        return;
    const int per = 128 / p.group;
    const size_t at = (size_t)tile * p.blocks + block;
    const u32x4 word = *reinterpret_cast<const u32x4*>(codes + (at * 64 + lane) * 4);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const uint32_t mt = meta[(at * 16 + c) * per + s * per / 4];
        const float scale = __uint_as_float(mt & ~15u);
        const int zero = (int)(mt & 15u);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = scale * (float)((int)((word[s] >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u) - zero);
        const int r0 = block * 128 + s * 32 + kb * 8;
        if (!SPARSE) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (r0 + e < p.W)
                    __builtin_nontemporal_store(v[e], B + (size_t)(r0 + e) * p.N + col);
        } else {
            const uint2 offs = *reinterpret_cast<const uint2*>(rows + (size_t)(col >> 5) * p.blocks * 128 + r0);
            int at_row[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)   // from the first dense row of the lane's windows
                at_row[e] = r0 + e < p.W ? (int)(((e < 4 ? offs.x : offs.y) >> (8 * (e & 3))) & 255u) - kb * (p.span / 4) : -1;
            const int d0 = r0 / p.n * p.m;
            const int count = min(p.span / 4, p.K - d0);
            for (int d = 0; d < count; ++d) {
                float out = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    out = at_row[e] == d ? v[e] : out;
                __builtin_nontemporal_store(out, B + (size_t)(d0 + d) * p.N + col);
            }
        }
    }
}

} // namespace

hipError_t launch_q4_pack(const float* values, const uint8_t* given, const float* scales, const uint8_t* zeros,
                          const int32_t* rows, const Q4Shape& p, bool asymmetric, uint32_t* codes, uint32_t* meta,
                          uint8_t* row_offsets, hipStream_t stream)
{
    const dim3 grid(p.blocks, (p.tiles + 3) / 4);
    if (values)
        q4_pack_kernel<true><<<grid, 256, 0, stream>>>(values, nullptr, nullptr, nullptr, rows, p, asymmetric, codes, meta);
    else
        q4_pack_kernel<false><<<grid, 256, 0, stream>>>(nullptr, given, scales, zeros, rows, p, false, codes, meta);
    if (rows) {
        const size_t entries = (size_t)p.blocks * 128 * (p.N / 32);
        q4_rows_kernel<<<(unsigned)((entries + 255) / 256), 256, 0, stream>>>(rows, p, row_offsets);
    }
    return hipGetLastError();
}

hipError_t launch_q4_expand(const uint32_t* codes, const uint32_t* meta, const uint8_t* row_offsets, const Q4Shape& p,
                            float* B, hipStream_t stream)
{
    const dim3 grid(p.blocks, (p.tiles + 3) / 4);
    if (row_offsets)
        q4_expand_kernel<true><<<grid, 256, 0, stream>>>(codes, meta, row_offsets, p, B);
    else
        q4_expand_kernel<false><<<grid, 256, 0, stream>>>(codes, meta, row_offsets, p, B);
    return hipGetLastError();
}

} // namespace nmspmm
