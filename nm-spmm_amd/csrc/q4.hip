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
//         2 i of the eight, nibble i + 4 row 2 i + 1, and the whole is rotated left by three bits, so that the
//         operand registers come out of one shift (the first: none) and one mask-and-or each.
//   meta  [tile][block][16 columns][128 / group] uint32: the scale's fp32 bits with the zero point in
//         the low four.
//   rows  [N / 32][blocks * 128] uint8 (n < m only): the dense row of each kept row, counted from the
//         first row of the windows of its k-step (32 kept rows span 32 m / n <= 256 dense rows).
// Rows beyond W and columns beyond N are filled in (the group's zero point, meta 0, the dense row K).
#include "internal.h"

namespace nmspmm {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// Nearest whole number to x / scale, ties to even, for |x| <= 16 scale and a scale of 20 significant bits.  The product with the
// inverse gives it or its neighbour; what remains of x (exact: one fma, 23 bits at most) is compared with half a scale.
// Tiny scales are made normal together with x, so that the inverse exists.
struct Nearest {
    float factor, scale, inverse, half, below;
    __device__ explicit Nearest(float s)
    {
        factor = s < 0x1p-100f ? 0x1p100f : 1.0f;
        scale = s * factor;
        inverse = 1.0f / scale;
        half = 0.5f * scale;
        below = __uint_as_float(__float_as_uint(half) - 1);     // so that "more than it" is "half or more": an odd number does not keep a tie
    }
    __device__ float operator()(float x) const
    {
        x *= factor;
        const float q = rintf(x * inverse), rest = fmaf(-q, scale, x);
        const float most = ((int)q & 1) ? below : half;
        return q + (rest > most ? 1.0f : rest < -most ? -1.0f : 0.0f);
    }
};

// Where row e of a word's eight lies: its nibble's first bit.
__device__ constexpr int nibble(int e) { return 4 * ((e >> 1) + 4 * (e & 1)); }

// The dense rows of a lane's eight kept rows, counted from the first row of their step; `keep` bit e: row e is inside its
// window.  One that is not gets a row that its window does not keep (its code will be the zero point).
__device__ inline void row_offsets(const int (&local)[8], int r0, const Q4Shape& p, int (&offset)[8], uint32_t& keep)
{
    const int shift = __builtin_ctz(p.n);       // n is 1, 2, 4 or 8
    keep = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        keep |= local[e] >= 0 && local[e] < p.m ? 1u << e : 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        int at = local[e];
        if (!((keep >> e) & 1u)) {
            for (at = 0; at < p.m; ++at) {
                bool kept = false;
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    kept |= k >> shift == e >> shift && local[k] == at;
                if (!kept)
                    break;
            }
        }
        offset[e] = ((r0 + e) >> shift) * p.m + at - (r0 >> 5) * p.span;
    }
}

// A workgroup packs a block of 128 rows of 16 V columns, each of its four waves a step of 32 rows: lane 16 kb + c takes rows
// 8 kb + e of columns V c .. V c + V - 1.  FROM_VALUES: the codes are found here, otherwise they are given.  HBM-bound, with
// some 25 vector instructions a value to hide behind it: a wave holds a step and not a whole block (four columns and 128 rows
// a wave: 4096 x 4096 34 us, this way 24: 76 MB, 3.2 TB/s), a wave instruction reads four segments of 16 V values.
template <bool FROM_VALUES, int V, bool SPARSE>
__global__ void __launch_bounds__(256)
q4_pack_kernel(const float* __restrict__ values, const uint8_t* __restrict__ given, const float* __restrict__ scales,
               const uint8_t* __restrict__ zeros, const int32_t* __restrict__ rows, Q4Shape p, bool asymmetric,
               uint32_t* __restrict__ codes, uint32_t* __restrict__ meta, uint8_t* __restrict__ offsets)
{
    constexpr int Cols = 16 * V;
    __shared__ float tops[4][Cols], lows[4][Cols], odds[4][Cols];
    __shared__ uint32_t groups[4][Cols];
    __shared__ __attribute__((aligned(16))) uint32_t words[4 * Cols][4];    // [kb * Cols + column][step]
    const int lane = threadIdx.x & 63, c = lane & 15, kb = lane >> 4, s = threadIdx.x >> 6;
    const int block = blockIdx.y, first = blockIdx.x * Cols;    // neighbours run side by side: whole rows are in flight
    const int col = first + c * V;      // the first of the lane's columns
    const bool column = col < p.N;      // V divides N
    const int per = 128 / p.group;      // groups of a block: 1, 2 or 4
    const int g = per == 4 ? s : per == 2 ? s >> 1 : 0;     // this step's
    const int r0 = block * 128 + s * 32 + kb * 8;

    float v[8][V];
    uint32_t x[8];      // given codes, a byte a column
    if (FROM_VALUES) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            typedef float part __attribute__((ext_vector_type(V > 1 ? V : 2)));
            const float* const at = values + (size_t)(r0 + e) * p.N + col;
            const bool in = column && r0 + e < p.W;
            if (V > 1) {
                const part y = in ? __builtin_nontemporal_load(reinterpret_cast<const part*>(at)) : part(0.0f);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    v[e][i] = y[i % (V > 1 ? V : 2)];
            } else
                v[e][0] = in ? __builtin_nontemporal_load(at) : 0.0f;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint8_t* const at = given + (size_t)(r0 + e) * p.N + col;
            x[e] = 0;
            if (column && r0 + e < p.W)
                x[e] = V == 4 ? *reinterpret_cast<const uint32_t*>(at) : *at;
        }
    }
    // which of the kept rows lie inside their windows, and the offsets of all
    uint32_t keep = 255u;
    if (SPARSE) {
        const int Q = p.N / 32, vector = col >> 5;
        int local[8], offset[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            local[e] = column && r0 + e < p.W ? rows[(size_t)(r0 + e) * Q + vector] : e & (p.n - 1);
        row_offsets(local, r0, p, offset, keep);
        if (column && (col & 31) == 0) {
            uint2 eight = make_uint2(0, 0);
            // rows beyond W name the first element behind x's row, which reads as zero (a step that they share with others spans at most
            // 256 dense rows and is not whole: 255 at most)
            const int behind = max(p.K - (r0 >> 5) * p.span, 0);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t byte = (uint32_t)(r0 + e < p.W ? offset[e] : behind) & 255u;
                if (e < 4)
                    eight.x |= byte << (8 * (e & 3));
                else
                    eight.y |= byte << (8 * (e & 3));
            }
            *reinterpret_cast<uint2*>(offsets + (size_t)vector * p.blocks * 128 + r0) = eight;
        }
    }

    uint32_t mt[V];
    if (FROM_VALUES) {
        // largest and smallest of each step, zero among them; a NaN or an infinity anywhere makes the scale NaN (the
        // whole group then expands to NaN)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float top = 0.0f, low = 0.0f, odd = 0.0f;       // odd stays zero with finite numbers
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                top = fmaxf(top, v[e][i]);
                low = fminf(low, v[e][i]);
                odd = fmaf(v[e][i], 0.0f, odd);
            }
#pragma unroll
            for (int mask = 16; mask < 64; mask <<= 1) {
                top = fmaxf(top, __shfl_xor(top, mask, 64));
                low = fminf(low, __shfl_xor(low, mask, 64));
                odd += __shfl_xor(odd, mask, 64);
            }
            if (kb == 0) {
                tops[s][c * V + i] = top;
                lows[s][c * V + i] = low;
                odds[s][c * V + i] = odd;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float top = 0.0f, low = 0.0f, odd = 0.0f;
            for (int t = g * 4 / per; t < (g + 1) * 4 / per; ++t) {
                top = fmaxf(top, tops[t][c * V + i]);
                low = fminf(low, lows[t][c * V + i]);
                odd += odds[t][c * V + i];
            }
            // The smallest scale of 20 significant bits with steps * scale >= what has to be covered: the quotient (in double: a range may be
            // twice what a float holds) is near enough to be a step off at most (steps * scale has 24 bits: the comparison is exact).
            const double steps = asymmetric ? 15.0 : 7.0;
            const double need = asymmetric ? (double)top - (double)low : (double)fmaxf(top, -low);
            uint32_t bits = __float_as_uint((float)(need * (asymmetric ? 1.0 / 15.0 : 1.0 / 7.0))) & ~15u;
            if (steps * (double)__uint_as_float(bits) < need)
                bits += 16;
            else if (bits >= 16 && steps * (double)__uint_as_float(bits - 16) >= need)
                bits -= 16;
            const float scale = __uint_as_float(bits);
            float zero = 8.0f;
            if (asymmetric)
                zero = scale > 0.0f ? fminf(fmaxf(Nearest(scale)(-low), 0.0f), 15.0f) : 0.0f;
            mt[i] = odd != 0.0f ? 0x7fc00008u : bits | (uint32_t)zero;      // (odd is NaN)
        }
    } else {
        const int j = block * per + g;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            mt[i] = 0;
            if (column && (size_t)j * p.group < (size_t)p.W) {
                const uint32_t z = zeros ? zeros[(size_t)j * p.N + col + i] : 8u;
                // 20 significant bits, to the nearest (ties away from zero; 16-bit scales are exact), but never to infinity
                const uint32_t bits = __float_as_uint(scales[(size_t)j * p.N + col + i]);
                const bool odd = (bits & 0x7f800000u) == 0x7f800000u, last = (bits & 0x7ffffff0u) == 0x7f7ffff0u;
                mt[i] = ((odd ? 0x7fc00000u : last ? bits : bits + 8u) & ~15u) | (z & 15u);
            }
        }
    }
    uint32_t in = 0;        // the nibbles of rows that count: not beyond W, not outside their window
#pragma unroll
    for (int e = 0; e < 8; ++e)
        in |= column && r0 + e < p.W && ((keep >> e) & 1u) ? 15u << nibble(e) : 0u;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float scale = __uint_as_float(mt[i] & ~15u), zero = (float)(mt[i] & 15u);
        const Nearest nearest(scale);
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (FROM_VALUES)
                w |= (uint32_t)__builtin_amdgcn_fmed3f(nearest(v[e][i]) + zero, 0.0f, 15.0f) << nibble(e);
            else
                w |= ((x[e] >> (8 * i)) & 15u) << nibble(e);
        }
        const uint32_t mask = FROM_VALUES && !(scale > 0.0f) ? 0u : in;     // (nothing counts under a scale of 0 or NaN)
        w = (w & mask) | ((mt[i] & 15u) * 0x11111111u & ~mask);
        words[kb * Cols + c * V + i][s] = __builtin_amdgcn_alignbit(w, w, 29);
        if (kb == 0)
            groups[g][c * V + i] = mt[i];
    }
    __syncthreads();
    for (int n = threadIdx.x; n < 4 * Cols; n += 256) {
        const int part = n / Cols, at = first + n % Cols, tile = at >> 4;
        if (tile < p.tiles)
            *reinterpret_cast<u32x4*>(codes + (((size_t)tile * p.blocks + block) * 64 + part * 16 + (at & 15)) * 4) =
                *reinterpret_cast<const u32x4*>(words[n]);
    }
    for (int n = threadIdx.x; n < per * Cols; n += 256) {
        const int at = first + n / per, tile = at >> 4;
        if (tile < p.tiles)
            meta[(((size_t)tile * p.blocks + block) * 16 + (at & 15)) * per + n % per] = groups[n % per][n / per];
    }
}

// Back to the dense fp32 matrix B[K][N], with the same split.  A lane's eight rows of a step are whole windows (KEPT = n divides
// 8), so it writes all their dense rows: the kept ones and the zeros between.  KEPT 0: a dense operand.  HBM-bound by
// its writes: 4096 x 4096 14.4 us (76 MB, 5.3 TB/s), 11008 x 4096 2:8 37 (187 MB, 5.0 TB/s).
template <int KEPT, int V>
__global__ void __launch_bounds__(256)
q4_expand_kernel(const uint32_t* __restrict__ codes, const uint32_t* __restrict__ meta, const uint8_t* __restrict__ rows,
                 Q4Shape p, float* __restrict__ B)
{
    const int lane = threadIdx.x & 63, c = lane & 15, kb = lane >> 4;
    const int block = blockIdx.y;
    const int col = (blockIdx.x * 4 + (threadIdx.x >> 6)) * (16 * V) + c * V;
    if (col >= p.N)
        return;
    const int per = 128 / p.group;
    const size_t at = (size_t)(col >> 4) * p.blocks + block;
    const int place = col & 15;
    u32x4 word[V];
    uint32_t mt[V][4];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        word[i] = *reinterpret_cast<const u32x4*>(codes + (at * 64 + kb * 16 + place + i) * 4);
#pragma unroll
        for (int g = 0; g < 4; ++g)
            if (g < per)
                mt[i][g] = meta[(at * 16 + place + i) * per + g];
    }
    uint2 offs[4];
    if (KEPT)
#pragma unroll
        for (int s = 0; s < 4; ++s)
            offs[s] = *reinterpret_cast<const uint2*>(rows + (size_t)(col >> 5) * p.blocks * 128 + block * 128 + s * 32 + kb * 8);
    auto put = [&](int row, const float* x) {
        float* const to = B + (size_t)row * p.N + col;
        if (V == 4)
            __builtin_nontemporal_store(f32x4{x[0], x[1 % V], x[2 % V], x[3 % V]}, reinterpret_cast<f32x4*>(to));
        else
            __builtin_nontemporal_store(x[0], to);
    };
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        float v[8][V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const uint32_t m = per == 4 ? mt[i][s] : per == 2 ? mt[i][s >> 1] : mt[i][0];
            const float scale = __uint_as_float(m & ~15u);
            const int zero = (int)(m & 15u);
            const uint32_t packed = __builtin_amdgcn_alignbit(word[i][s], word[i][s], 3);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e][i] = scale * (float)((int)((packed >> nibble(e)) & 15u) - zero);
        }
        const int r0 = block * 128 + s * 32 + kb * 8;
        if (KEPT == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (r0 + e < p.W)
                    put(r0 + e, v[e]);
        } else {
            constexpr int n = KEPT ? KEPT : 1;
            const int d0 = r0 / n * p.m;
#pragma unroll
            for (int w = 0; w < 8 / n; ++w) {
                if (r0 + w * n >= p.W)
                    continue;
                int place_of[n];        // of the window's kept rows
#pragma unroll
                for (int k = 0; k < n; ++k) {
                    const int e = w * n + k;
                    place_of[k] = (int)(((e < 4 ? offs[s].x : offs[s].y) >> (8 * (e & 3))) & 255u) - (kb * (8 / n) + w) * p.m;
                }
                for (int d = 0; d < p.m; ++d) {
                    float out[V];
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        out[i] = 0.0f;
#pragma unroll
                    for (int k = 0; k < n; ++k)
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            out[i] = place_of[k] == d ? v[w * n + k][i] : out[i];
                    put(d0 + w * p.m + d, out);
                }
            }
        }
    }
}

} // namespace

hipError_t launch_q4_pack(const float* values, const uint8_t* given, const float* scales, const uint8_t* zeros,
                          const int32_t* rows, const Q4Shape& p, bool asymmetric, uint32_t* codes, uint32_t* meta,
                          uint8_t* row_offsets, hipStream_t stream)
{
    // four columns a lane where rows are whole pieces of four
    const bool four = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(values) & 15u) == 0 && (reinterpret_cast<uintptr_t>(given) & 3u) == 0;
    const dim3 grid(four ? (p.tiles + 3) / 4 : p.tiles, p.blocks);
#define NMSPMM_PACK(FROM, V, SPARSE)                                                                                          \
    q4_pack_kernel<FROM, V, SPARSE><<<grid, 256, 0, stream>>>(values, given, scales, zeros, rows, p, asymmetric, codes, meta, \
                                                              row_offsets)
    if (values) {
        if (rows)
            four ? NMSPMM_PACK(true, 4, true) : NMSPMM_PACK(true, 1, true);
        else
            four ? NMSPMM_PACK(true, 4, false) : NMSPMM_PACK(true, 1, false);
    } else {
        if (rows)
            four ? NMSPMM_PACK(false, 4, true) : NMSPMM_PACK(false, 1, true);
        else
            four ? NMSPMM_PACK(false, 4, false) : NMSPMM_PACK(false, 1, false);
    }
#undef NMSPMM_PACK
    return hipGetLastError();
}

hipError_t launch_q4_expand(const uint32_t* codes, const uint32_t* meta, const uint8_t* row_offsets, const Q4Shape& p,
                            float* B, hipStream_t stream)
{
    const bool four = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(B) & 15u) == 0;
    const dim3 grid(four ? (p.tiles + 15) / 16 : (p.tiles + 3) / 4, p.blocks);
#define NMSPMM_EXPAND(KEPT)                                                                                       \
    (four ? q4_expand_kernel<KEPT, 4><<<grid, 256, 0, stream>>>(codes, meta, row_offsets, p, B)                   \
          : q4_expand_kernel<KEPT, 1><<<grid, 256, 0, stream>>>(codes, meta, row_offsets, p, B))
    if (!row_offsets)
        NMSPMM_EXPAND(0);
    else if (p.n == 1)
        NMSPMM_EXPAND(1);
    else if (p.n == 2)
        NMSPMM_EXPAND(2);
    else if (p.n == 4)
        NMSPMM_EXPAND(4);
    else
        NMSPMM_EXPAND(8);
#undef NMSPMM_EXPAND
    return hipGetLastError();
}

} // namespace nmspmm
