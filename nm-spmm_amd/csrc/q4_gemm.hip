// y = x B for a B in 4 bits and many rows of x (the mathematics: q4_linear.hip; the layout: q4.hip).
//
// A workgroup computes 64 rows x 64 NC columns, each of its four waves all 64 rows of 16 NC columns: a code is
// widened once (a shift and a mask-and-or for two) and used for four row tiles.  The codes come straight from
// memory into the operand registers, their layout being that of the operands; x goes through LDS (64 rows x 128
// elements, two buffers, 16-byte pieces swapped by row so that the sixteen rows of a read lie in different
// banks).  The group sums of x, with which the offset of the widened codes is taken off, are made beforehand
// by the kernel that also cuts fp32 activations into their three bf16 pieces or copies rows that are not aligned.
// A sparse operand comes spread out, with code - zero in its places and zeros between, and for fp32 activations codes
// are widened to code - zero: there are no offsets then and no sums.
#include "internal.h"
#include "q4_device.h"

#include <algorithm>

namespace nmspmm {

namespace {

// ---- x: its pieces, and its sums over the dense rows of each group (at most 128 at a time) ---------------

// One wave per 512 elements of a row, eight each lane.  PLANES 0: only the sums.  Pieces: [row][plane][K filled up to 128].
// HBM-bound: 2000 rows of 4096 bf16 5.3 us (16 MB, 3.1 TB/s, launch and all).
template <ElementType T, int PLANES>
__global__ void __launch_bounds__(256)
q4_prepare_x_kernel(const void* __restrict__ x_, size_t ldx, int M, int K, int Kp, int unit, uint16_t* __restrict__ planes,
                    float* __restrict__ sums, size_t sums_ld)
{
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), k0 = blockIdx.y * 512 + lane * 8;
    if (row >= M)
        return;
    const bool whole = T == kF32 ? ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(x_) & 15u) == 0
                                 : ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(x_) & 15u) == 0;
    uint32_t v[8];      // fp32 bits, or 16 bits
    if (T == kF32) {
        const uint32_t* const x = static_cast<const uint32_t*>(x_) + (size_t)row * ldx;
        if (whole && k0 + 8 <= K) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(x + k0), b = *reinterpret_cast<const u32x4*>(x + k0 + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = e < 4 ? a[e & 3] : b[e & 3];
        } else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = k0 + e < K ? x[k0 + e] : 0u;
    } else {
        const uint16_t* const x = static_cast<const uint16_t*>(x_) + (size_t)row * ldx;
        if (whole && k0 + 8 <= K) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(x + k0);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = e & 1 ? a[e >> 1] >> 16 : a[e >> 1] & 0xffffu;
        } else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = k0 + e < K ? x[k0 + e] : 0u;
    }
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        sum += T == kF32 ? __uint_as_float(v[e]) : T == kBF16 ? __uint_as_float(v[e] << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)v[e]);
    for (int mask = 1; mask < unit / 8; mask <<= 1)
        sum += __shfl_xor(sum, mask, 64);
    if (sums && k0 < Kp && (lane & (unit / 8 - 1)) == 0)
        sums[(size_t)(k0 / unit) * sums_ld + row] = sum;
    if (PLANES == 0 || k0 >= Kp)
        return;
    if (PLANES == 1) {
        *reinterpret_cast<u32x4*>(planes + (size_t)row * Kp + k0) =
            u32x4{v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16};
    } else {
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = __builtin_amdgcn_perm(v[2 * e + 1], v[2 * e], 0x07060302u);
            *reinterpret_cast<u32x4*>(planes + ((size_t)row * 3 + q) * Kp + k0) = w;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = __float_as_uint(__uint_as_float(v[e]) - __uint_as_float(v[e] & 0xffff0000u));
        }
    }
}

// ---- a sparse operand's codes as a dense operand: a byte a row, zero where none was kept ------------------------

// The byte is an 8-bit float (e4m3) of code - zero: sign and magnitude, whose low numbers are evenly spaced (0 .. 15 stand for
// 0 .. 15 times 2^-9, exactly).  What x holds in a row that was not kept is multiplied by a zero: it leaves no rounding in the sums.
// (With the zero point's code there it did, of 31 times its size.)  Layout: [tile][block][half of the
// steps][lane][step][8 rows], so that a wave stores and reads 1 KB in a piece.
// Bound by its writes (four to sixteen times its reads); 4096 x 11008 2:4 29 us, 2:8 20, the price of a sparse operand at 33 rows and more.
template <int KEPT>     // kept rows that can lie among eight dense ones: those of their windows, or of the one they are part of; 0: dense
__global__ void __launch_bounds__(256)
q4_densify_kernel(const uint32_t* __restrict__ codes, const uint32_t* __restrict__ meta, const uint8_t* __restrict__ rows,
                  Q4Shape p, int dense_blocks, uint32_t* __restrict__ out)
{
    const int lane = threadIdx.x & 63, c = lane & 15, kb = lane >> 4;
    const int tile = blockIdx.y * 4 + (threadIdx.x >> 6), block = blockIdx.x;
    if (tile >= p.tiles)
        return;
    const int per = 128 / p.group;
    u32x4 word[2];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int d0 = min(block * 128 + s * 32 + kb * 8, (p.K - 1) & ~7);  // eight dense rows (of padding: anything, x is zero there)
        const int r0 = d0 / p.m * p.n;                                      // a multiple of KEPT: all in one word
        const size_t at = (size_t)tile * p.blocks + (r0 >> 7);
        const int zero = (int)(meta[(at * 16 + c) * per + ((r0 >> 5) & 3) * per / 4] & 15u);
        const uint32_t rotated = codes[(at * 64 + ((r0 >> 3) & 3) * 16 + c) * 4 + ((r0 >> 5) & 3)];
        const uint32_t packed = __builtin_amdgcn_alignbit(rotated, rotated, 3);
        uint2 eight = make_uint2(0, 0);
        if (KEPT)
            eight = *reinterpret_cast<const uint2*>(rows + (size_t)(tile >> 1) * p.blocks * 128 + (r0 & ~7));
        const int base = (r0 >> 5) * p.span - d0;
        uint32_t low = 0, high = 0;
#pragma unroll
        for (int i = 0; i < (KEPT ? KEPT : 8); ++i) {
            const int e = KEPT ? (r0 & 7) + i : i;
            const uint32_t off = ((e < 4 ? eight.x : eight.y) >> (8 * (e & 3))) & 255u;
            const uint32_t d = KEPT ? (uint32_t)(base + (int)off) : i;      // 0..7 if it is among the eight
            const int value = (int)((packed >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u) - zero;
            const uint32_t byte = (value < 0 ? 128u : 0u) | (uint32_t)abs(value);
            const uint32_t there = r0 + i < p.W ? byte << (8 * (d & 3)) : 0u;
            low |= d < 4u ? there : 0u;
            high |= d - 4u < 4u ? there : 0u;
        }
        word[s >> 1][(s & 1) * 2] = low;
        word[s >> 1][(s & 1) * 2 + 1] = high;
    }
    u32x4* const to = reinterpret_cast<u32x4*>(out) + ((size_t)tile * dense_blocks + block) * 128 + lane;
    to[0] = word[0];
    to[64] = word[1];
}

// ---- the product --------------------------------------------------------------------------------------------

typedef __attribute__((address_space(3))) uint32_t lds_u32;

struct GemmArgs {
    const uint16_t* x;      // rows ldx elements apart, their planes `plane`; 64 rows within 2 GiB
    size_t plane, ldx;
    const float* sums;      // [K / unit][sums_ld]
    size_t sums_ld;
    const uint32_t* codes;  // dense: 4 bits a row, or 8 (q4_densify_kernel)
    Q4Meta meta;
    const float* bias;
    void* y;
    size_t ldy;
    float* partial;         // [split][M][partial_ld] where K is split
    size_t partial_ld;
    int M, N;
    int blocks, unit;       // dense blocks of 128 rows; rows after which sums are scaled (32, 64, 128)
    int splits;
    int tiles, tiles_m, tiles_n;    // 16-column tiles of the operand; workgroups along rows and columns
};

// A workgroup computes 16 RT rows x 64 NC columns of a range of K.  A stage is 128 dense rows, or 64 with the three pieces of an fp32 x
// beside each other: a code is widened once for all of them.  STEPS: 32-row steps of a unit.
// 2000 rows of bf16, 4096 x 11008: 217 us, 830 TFLOP/s, where torch's product with bf16 weights takes 288.  The matrix cores are busy a
// third of the time; 5.8 vector instructions go with each of theirs (widening 1.3, scales and offsets 2), and a stage waits
// for its x in LDS.  Wider tiles (two column tiles a wave), offsets as one more product and x a stage further ahead were slower
// (227 to 249 us).  Groups of 64 / 32 scale two and four times as often: 290 / 480 us; three pieces of fp32 455 (groups of 32: 533).
// BYTES: a spread-out operand.  There, and with the pieces of an fp32 x, the operand's elements are code - zero exactly: sums start from
// zero and take none of x's.  (Pieces of 16 + code in one sum lost up to twice as much as an fp32 product does, and what x holds under a zero
// weight left its rounding; bf16 and fp16 rows of a dense operand, whose results are rounded far coarser, take the cheaper widening.)
template <ElementType T, int PLANES, ElementType OUT, bool BYTES, int RT, int NC, int STEPS>
__global__ void __launch_bounds__(256, 2)
q4_gemm_kernel(GemmArgs g)
{
    constexpr bool Exact = BYTES || PLANES == 3;
    constexpr int Words = BYTES ? 2 : 1;                                    // of a step
    constexpr int Rows = 16 * RT;
    constexpr int StageSteps = PLANES == 1 ? 4 : 2;                         // 32-row steps of a stage
    constexpr int Loops = StageSteps / STEPS;                               // units in a stage
    static_assert(STEPS <= StageSteps, "a unit lies within a stage");
    constexpr int Pieces = PLANES * StageSteps * 4;                         // 16-byte pieces of a row in a stage
    constexpr int RowBytes = Pieces * 16;
    constexpr int Mine = (Rows * Pieces + 255) / 256;                       // pieces that a thread brings
    __shared__ __attribute__((aligned(16))) unsigned char tile[2][Rows * RowBytes];
    __shared__ __attribute__((aligned(16))) float sums[2][Loops][Exact ? 4 : Rows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, kb = lane >> 4;

    // Workgroups of one die (ids 8 apart) walk through tiles that share rows of x and columns of B: groups of
    // eight row tiles, column by column.
    const int all = g.tiles_m * g.tiles_n;
    const int die = blockIdx.x & 7, place = blockIdx.x >> 3;
    const int share = all / 8, extra = all % 8;
    const int id = die * share + min(die, extra) + place;
    const int band = id / (8 * g.tiles_n), inside = id - band * 8 * g.tiles_n;
    const int height = min(8, g.tiles_m - band * 8);
    const int m0 = (band * 8 + inside % height) * Rows, tile0 = (inside / height) * (4 * NC) + wave * NC;
    const int rows_here = min(Rows, g.M - m0);
    const int first_block = (int)((long long)g.blocks * blockIdx.y / g.splits);
    const int end_block = (int)((long long)g.blocks * (blockIdx.y + 1) / g.splits);
    const int first = first_block * 4 / StageSteps, end = end_block * 4 / StageSteps;   // stages

    f32x4 acc[RT][NC], total[RT][NC];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int j = 0; j < NC; ++j)
            total[t][j] = f32x4{0, 0, 0, 0};

    // Where piece q of row r lies in a row of the tile: swapped so that the sixteen rows of a read start in different banks.
    auto place_of = [&](int r, int q) {
        return PLANES == 1 ? q ^ (r & 15) : (q & ~7) | ((q ^ (r >> 1)) & 7);
    };
    // A wave brings 1 KB at a time straight into LDS, where lane l's piece lands at place l: lane and place fix row and piece.
    uint32_t from[Mine];
#pragma unroll
    for (int i = 0; i < Mine; ++i) {
        const int n = (i * 4 + wave) * 64 + lane;
        const int r = n / Pieces, q = place_of(r, n % Pieces);     // (the swap is its own inverse)
        from[i] = (uint32_t)((q / (StageSteps * 4)) * g.plane * 2 + r * g.ldx * 2 + (q % (StageSteps * 4)) * 16);
        if (r >= rows_here)
            from[i] = 0x80000000u;      // read as zero
    }
    uint32_t sr = 0;
    const uint32_t one = PLANES == 3 ? sixteens<kF16>() : sixteens<T>();
    auto fetch_x = [&](int stage, unsigned char* to) {
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(g.x + (size_t)m0 * g.ldx + stage * (StageSteps * 32)), 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int i = 0; i < Mine; ++i)
            if (Rows * Pieces % 256 == 0 || (i * 4 + wave) * 64 < Rows * Pieces)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_u32*)(to + (i * 4 + wave) * 1024), 16, (int)from[i], 0, 0, 0);
    };
    auto fetch_sums = [&](int stage) {
        if (!Exact && wave < Loops) {
            const int unit = stage * Loops + wave;
            const float* const base = g.sums + (size_t)unit * g.sums_ld + m0;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, rows_here * 4, 0x00020000);
            sr = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, lane * 4, 0, 0);
        }
    };
    auto put_sums = [&](int half) {
        if (!Exact && wave < Loops && lane < Rows)
            sums[half][wave][lane] = __uint_as_float(sr);
    };
    uint32_t w[NC][StageSteps * Words], wn[NC][StageSteps * Words], mt[NC], mn[NC];
    auto fetch_codes = [&](int stage) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int t = min(tile0 + j, g.tiles - 1);      // beyond the last column: read, not used
            const int b = stage * StageSteps / 4;
            const uint32_t* const base = g.codes + ((size_t)t * g.blocks + b) * (256 * Words) +
                                         (PLANES == 1 ? 0 : (stage & 1) * (BYTES ? 256 : 2)) + lane * 4;
            if (PLANES == 1 || BYTES) {
#pragma unroll
                for (int h = 0; h < StageSteps * Words / 4; ++h) {
                    const u32x4 v = reinterpret_cast<const u32x4*>(base)[h * 64];
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        wn[j][h * 4 + s] = v[s];
                }
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(base);
                wn[j][0] = v.x;
                wn[j][1] = v.y;
            }
        }
    };
    auto fetch_meta = [&](int step) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
            mn[j] = g.meta.word(min(tile0 + j, g.tiles - 1), step * 32, c);
    };

    // Declared not to overlap, so that the reads of this stage's tile do not wait for the next one's arrival.
    auto multiply = [&](int stage, const unsigned char* __restrict__ now, const float* __restrict__ sums_now, unsigned char* __restrict__ next)
        __attribute__((always_inline)) {
        if (stage + 1 < end) {
            fetch_x(stage + 1, next);
            fetch_sums(stage + 1);
            fetch_codes(stage + 1);
            if (Loops == 1)
                fetch_meta((stage + 1) * StageSteps);
        }
#pragma clang loop unroll(disable)
        for (int u = 0; u < Loops; ++u) {       // (unrolled, smaller units would need more registers than there are)
            // the next unit's scales are on their way while this one's are used
            if (Loops > 1) {
#pragma unroll
                for (int j = 0; j < NC; ++j)
                    mt[j] = mn[j];
                if (u + 1 < Loops || stage + 1 < end)
                    fetch_meta(stage * StageSteps + (u + 1) * STEPS);
            }
            // a unit's sums start from what its offset takes off, - (16 + zero) times the sum of x (Exact: from zero)
            uint32_t offset[NC];
#pragma unroll
            for (int j = 0; j < NC; ++j)
                offset[j] = ((mt[j] & 15u) << 6 | 0xcc00u) * 0x10001u;     // - (16 + zero) in fp16, twice
            if (Exact) {
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int j = 0; j < NC; ++j)
                        acc[t][j] = f32x4{0, 0, 0, 0};
            } else {
                f32x4 xs[RT];
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    xs[t] = *reinterpret_cast<const f32x4*>(sums_now + u * Rows + t * 16 + kb * 4);
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    const float offset = -(16.0f + (float)(mt[j] & 15u));
#pragma unroll
                    for (int t = 0; t < RT; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            acc[t][j][e] = offset * xs[t][e];
                }
            }
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int s = u * STEPS + i;
                u32x4 wide[NC];
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    uint32_t word[Words];
#pragma unroll
                    for (int h = 0; h < Words; ++h) {
                        word[h] = w[j][i * Words + h];
#pragma unroll
                        for (int k = 1; k < Loops; ++k)
                            word[h] = u == k ? w[j][(k * STEPS + i) * Words + h] : word[h];
                    }
                    wide[j] = BYTES         ? from_bytes<T>(word[0], word[Words - 1])
                              : PLANES == 3 ? differences(word[0], one, offset[j])
                                            : widened<T>(word[0], one);
                }
#pragma unroll
                for (int q = 0; q < PLANES; ++q) {
                    u32x4 a[RT];
#pragma unroll
                    for (int t = 0; t < RT; ++t)
                        a[t] = *reinterpret_cast<const u32x4*>(now + (t * 16 + c) * RowBytes +
                                                               place_of(c, (q * StageSteps + s) * 4 + kb) * 16);
#pragma unroll
                    for (int j = 0; j < NC; ++j)
#pragma unroll
                        for (int t = 0; t < RT; ++t)
                            acc[t][j] = product<T>(a[t], wide[j], acc[t][j]);
                }
            }
            // and are scaled when it ends
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const float scale = __uint_as_float(mt[j] & ~15u);
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        total[t][j][e] = fmaf(scale, acc[t][j][e], total[t][j][e]);
            }
        }
    };

    if (first < end) {
        fetch_x(first, tile[0]);
        fetch_sums(first);
        fetch_codes(first);
        fetch_meta(first * StageSteps);
        put_sums(0);
    }
    for (int stage = first, half = 0; stage < end; ++stage, half ^= 1) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int s = 0; s < StageSteps * Words; ++s)
                w[j][s] = wn[j][s];
        if (Loops == 1)
#pragma unroll
            for (int j = 0; j < NC; ++j)
                mt[j] = mn[j];
        __builtin_amdgcn_s_waitcnt(0x0f70);     // vmcnt(0): this wave's part of the tile has landed
        __syncthreads();        // this stage's tile is whole, and nobody reads the other any more
        multiply(stage, tile[half], sums[half][0], tile[half ^ 1]);
        if (stage + 1 < end)
            put_sums(half ^ 1);
    }

    // rows beyond M and columns beyond N lie outside the descriptors
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int rows = min(16, rows_here - t * 16);
        if (rows <= 0)
            break;
        const size_t ld = g.splits > 1 ? g.partial_ld : g.ldy;
        const size_t size = g.splits > 1 || OUT == kF32 ? 4 : 2;
        char* const base = g.splits > 1 ? reinterpret_cast<char*>(g.partial + ((size_t)blockIdx.y * g.M + m0 + t * 16) * ld)
                                        : static_cast<char*>(g.y) + (size_t)(m0 + t * 16) * ld * size;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(base, 0, (int)(((rows - 1) * ld + g.N) * size), 0x00020000);
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int col = (tile0 + j) * 16 + c;
            const float bias = g.bias && g.splits == 1 && col < g.N ? g.bias[col] : 0.0f;
            const uint32_t at = col < g.N ? (uint32_t)((kb * 4 * ld + col) * size) : 0x80000000u;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (g.splits > 1)
                    store_bounded<kF32>(r, at + (uint32_t)(e * ld * size), total[t][j][e]);
                else
                    store_bounded<OUT>(r, at + (uint32_t)(e * ld * size), total[t][j][e] + bias);
            }
        }
    }
}

// The ranges of K added up in order.
template <ElementType OUT>
__global__ void __launch_bounds__(256)
q4_gemm_reduce_kernel(const float* __restrict__ partial, size_t partial_ld, int splits, const float* __restrict__ bias,
                      void* __restrict__ y, size_t ldy, int M, int N)
{
    const int col = (blockIdx.y * 256 + threadIdx.x) * 4, row = blockIdx.x;
    if (col >= N)
        return;
    f32x4 sum = {0, 0, 0, 0};
#pragma unroll 4
    for (int s = 0; s < splits; ++s)
        sum += *reinterpret_cast<const f32x4*>(partial + ((size_t)s * M + row) * partial_ld + col);
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (col + e < N)
            store_result<OUT>(y, (size_t)row * ldy + col + e, sum[e] + (bias ? bias[col + e] : 0.0f));
}

template <ElementType T, int PLANES, ElementType OUT, bool BYTES, int STEPS>
void run_steps(const GemmArgs& g, int row_tiles, int column_tiles, hipStream_t stream)
{
    const dim3 grid(g.tiles_m * g.tiles_n, g.splits);
    if (row_tiles == 1)
        q4_gemm_kernel<T, PLANES, OUT, BYTES, 1, 2, STEPS><<<grid, 256, 0, stream>>>(g);
    else if (row_tiles == 2)
        q4_gemm_kernel<T, PLANES, OUT, BYTES, 2, 2, STEPS><<<grid, 256, 0, stream>>>(g);
    else if (column_tiles == 2)
        q4_gemm_kernel<T, PLANES, OUT, BYTES, 4, 2, STEPS><<<grid, 256, 0, stream>>>(g);
    else
        q4_gemm_kernel<T, PLANES, OUT, BYTES, 4, 4, STEPS><<<grid, 256, 0, stream>>>(g);
}

// How a product is cut: a workgroup's row tiles and column tiles (of a wave), and the ranges of K.
struct GemmCut {
    int row_tiles, column_tiles, tiles_m, tiles_n, splits;
};
GemmCut gemm_cut(int M, int tiles, int blocks)
{
    GemmCut c;
    const int cus = machine().cus;
    c.row_tiles = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    c.tiles_m = (M + 16 * c.row_tiles - 1) / (16 * c.row_tiles);
    c.column_tiles = c.row_tiles == 4 && c.tiles_m * ((tiles + 15) / 16) >= 2 * cus ? 4 : 2;
    c.tiles_n = (tiles + 4 * c.column_tiles - 1) / (4 * c.column_tiles);
    // two workgroups to a compute unit, as long as each has two blocks of K
    const long long groups = (long long)c.tiles_m * c.tiles_n;
    long long splits = (2 * cus + groups - 1) / groups;
    if (splits > blocks / 2)
        splits = blocks / 2;
    c.splits = splits < 1 || groups >= 2 * cus ? 1 : (int)splits;
    return c;
}

template <ElementType T, int PLANES, ElementType OUT, bool BYTES>
void run_gemm(GemmArgs& g, const GemmCut& c, hipStream_t stream)
{
    g.tiles_m = c.tiles_m;
    g.tiles_n = c.tiles_n;
    g.splits = c.splits;
    if (PLANES == 1 && g.unit == 128)
        run_steps<T, PLANES, OUT, BYTES, PLANES == 1 ? 4 : 2>(g, c.row_tiles, c.column_tiles, stream);
    else if ((BYTES && PLANES == 1) || g.unit == 64)        // (32 kept rows are 64 dense ones and more)
        run_steps<T, PLANES, OUT, BYTES, 2>(g, c.row_tiles, c.column_tiles, stream);
    else
        run_steps<T, PLANES, OUT, BYTES && PLANES == 3, 1>(g, c.row_tiles, c.column_tiles, stream);
    if (c.splits > 1)
        q4_gemm_reduce_kernel<OUT><<<dim3(g.M, (g.N + 1023) / 1024), 256, 0, stream>>>(g.partial, g.partial_ld, g.splits, g.bias, g.y,
                                                                                       g.ldy, g.M, g.N);
}

size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

} // namespace

// What lies where in the workspace (bytes): the spread-out codes or the sums of x, the pieces of x, the ranges' results.
struct GemmSpace {
    size_t codes, sums, planes, partial, bytes;
};
static GemmSpace gemm_space(const Q4Shape& p, int M, ElementType type, bool codes, bool product)
{
    const size_t blocks = ((size_t)p.K + 127) / 128;
    GemmSpace s;
    s.codes = 0;
    s.sums = codes ? p.tiles * blocks * 2048 : 0;
    s.planes = s.sums;
    s.partial = s.sums;
    s.bytes = s.sums;
    if (product) {
        const GemmCut c = gemm_cut(M, p.tiles, (int)blocks);
        s.planes = s.sums + (codes || type == kF32 ? 0 : round_up(blocks * 4 * round_up(M, 4) * sizeof(float), 256));
        s.partial = s.planes + (type == kF32 ? 3 : 1) * (size_t)M * blocks * 256;
        s.bytes = s.partial + (c.splits > 1 ? (size_t)c.splits * M * round_up(p.N, 4) * sizeof(float) : 0);
    }
    return s;
}

// Rows of a sparse operand that are gathered (q4_linear.hip), sixteen to a launch.  32 rows, 4096 x 4096, us in two such launches / spread
// out: bf16 2:4 11.3 / 28.9, 2:8 12.9 / 26.4, 1:8 11.0 / 27.6; fp32 2:8 16.3 / 29.7, 1:8 11.7 / 31.2, 2:4 23.7 / 31.9; at 4096 x 11008
// in groups of 32, fp32 2:4 80 / 52.
int q4_gathered_rows(const Q4Shape& p, ElementType type) { return type != kF32 || p.m > 2 * p.n || p.group == 128 ? 32 : 16; }
// ... and fp32 rows for which the codes of a dense operand are widened by each workgroup, not spread out once (in groups of 128, us: 512
// rows of 4096 x 4096 67.3 / 72.7, 2000 rows of 4096 x 11008 506 / 459).
constexpr int kWidenedRows = 1000;
bool q4_densifies(const Q4Shape& p, int M, ElementType type)
{
    return p.m > 1 ? M > q4_gathered_rows(p, type) : type == kF32 && M > kWidenedRows;
}

size_t q4_workspace_bytes(const Q4Shape& p, int M, ElementType type)
{
    // (how 9 to 16 rows are aligned and grouped is not known here)
    return gemm_space(p, M, type, q4_densifies(p, M, type), M > (p.m > 1 ? q4_gathered_rows(p, type) : 8)).bytes;
}

hipError_t launch_q4_densify(const Q4LinearArgs& a, uint32_t* out)
{
    const int blocks = (a.p.K + 127) / 128;
    const dim3 grid(blocks, (a.p.tiles + 3) / 4);
    const int kept = a.p.m > 8 ? a.p.n : 8 / a.p.m * a.p.n;
    auto kernel = !a.rows     ? q4_densify_kernel<0>
                  : kept == 1 ? q4_densify_kernel<1>
                  : kept == 2 ? q4_densify_kernel<2>
                  : kept == 4 ? q4_densify_kernel<4>
                              : q4_densify_kernel<8>;
    kernel<<<grid, 256, 0, a.stream>>>(a.codes, a.meta.words, a.rows, a.p, blocks, out);
    return hipGetLastError();
}

// `a` is dense by now (q4_linear.hip).
hipError_t launch_q4_gemm(const Q4LinearArgs& a, ElementType type, bool densified, void* workspace)
{
    const GemmSpace s = gemm_space(a.p, a.M, type, densified, true);
    const GemmCut c = gemm_cut(a.M, a.p.tiles, a.p.blocks);
    char* const base = static_cast<char*>(workspace);
    const int Kp = a.p.blocks * 128;
    GemmArgs g;
    // (fp32: scaling twice as often costs less than sums over two stages, 2000 rows 4096 x 11008 469 against 495 us)
    g.unit = std::min(a.meta.group, type == kF32 ? 64 : 128);
    g.sums = reinterpret_cast<float*>(base + s.sums);
    g.sums_ld = round_up(a.M, 4);
    g.codes = a.codes;
    g.meta = a.meta;
    g.bias = a.bias;
    g.y = a.y;
    g.ldy = a.ldy;
    g.M = a.M;
    g.N = a.p.N;
    g.blocks = a.p.blocks;
    g.tiles = a.p.tiles;
    g.partial = reinterpret_cast<float*>(base + s.partial);
    g.partial_ld = round_up(a.p.N, 4);
    uint16_t* const planes = reinterpret_cast<uint16_t*>(base + s.planes);
    const dim3 grid((a.M + 3) / 4, (Kp + 511) / 512);
    // x as it is: 16-bit elements, rows of whole blocks on 16-byte boundaries, 64 of them within 1 GiB
    const bool as_is = type != kF32 && a.p.K == Kp && a.ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15u) == 0 &&
                       a.ldx < (1u << 23);
    float* const sums = densified || type == kF32 ? nullptr : const_cast<float*>(g.sums);
    if (as_is) {
        g.x = static_cast<const uint16_t*>(a.x);
        g.ldx = a.ldx;
        g.plane = 0;
    } else {
        g.x = planes;
        g.ldx = type == kF32 ? 3 * (size_t)Kp : Kp;
        g.plane = Kp;
    }
#define NMSPMM_PREPARE(T, PLANES) \
    q4_prepare_x_kernel<T, PLANES><<<grid, 256, 0, a.stream>>>(a.x, a.ldx, a.M, a.p.K, Kp, g.unit, planes, sums, g.sums_ld)
    if (!as_is)
        type == kF32 ? NMSPMM_PREPARE(kF32, 3) : type == kBF16 ? NMSPMM_PREPARE(kBF16, 1) : NMSPMM_PREPARE(kF16, 1);
    else if (sums)
        type == kBF16 ? NMSPMM_PREPARE(kBF16, 0) : NMSPMM_PREPARE(kF16, 0);
#undef NMSPMM_PREPARE
    if (type == kF32)
        densified ? run_gemm<kBF16, 3, kF32, true>(g, c, a.stream) : run_gemm<kBF16, 3, kF32, false>(g, c, a.stream);
    else if (type == kBF16)
        densified ? run_gemm<kBF16, 1, kBF16, true>(g, c, a.stream) : run_gemm<kBF16, 1, kBF16, false>(g, c, a.stream);
    else
        densified ? run_gemm<kF16, 1, kF16, true>(g, c, a.stream) : run_gemm<kF16, 1, kF16, false>(g, c, a.stream);
    return hipGetLastError();
}

} // namespace nmspmm
