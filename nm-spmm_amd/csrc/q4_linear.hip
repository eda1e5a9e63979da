// y = x B for a B in 4 bits (layout: q4.hip), x and y in fp32, bf16 or fp16.
//
// With u = 16 + code and the group sums over kept rows r of group j,
//     y[i][c] = sum_j scale[j][c] * ( sum_r x[i][row(r)] u[r][c]  -  (16 + zero[j][c]) sum_r x[i][row(r)] ).
// u is what a 4-bit code becomes by being put into the mantissa of 16.0: in bf16 (bits 3..6) and in fp16 (bits
// 6..9) it is exact and costs a shift and one mask-and-or for two codes.  Both sums run on the matrix cores with
// fp32 accumulators, the second as a product with ones; zero point and scale are applied once per group.
// bf16 and fp16 activations are operands as they are.  An fp32 activation is cut into three bf16 pieces by
// truncation, 8 + 8 + 8 bits, which is exact; the pieces are rows of the same product (rows 4 i .. 4 i + 2 of a
// tile for row i of x) and are added at the end, so no activation is rounded.
// An infinity or a NaN in a row of x makes that row of y NaN in the columns that keep it; what they do not keep is not read into them.
#include "internal.h"
#include "q4_device.h"

namespace nmspmm {

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kMaxWaves = 16;
constexpr size_t kMostLds = 163840;     // all of a compute unit's: sixteen waves of sixteen half-kept rows take 135 KB
constexpr int kRowPitch = 136;      // 16-bit elements between staged rows: 128 and 16 bytes, so that the sixteen
                                    // rows of a 128-bit LDS read start in different banks

// Of rows whose kept elements are half of them (m = 2 n) a block spans 256 elements.
constexpr int kSpan = 256;
constexpr int kSpanPitch = 264;     // between such rows in LDS: the sixteen lanes of a kept row read different banks

// How the activations reach the matrix operands: as they lie in memory (16-bit types, 16-byte aligned rows of whole
// blocks), or through the wave's own part of LDS: from consecutive elements, from elements gathered in memory, or from all elements that
// a block spans, gathered in LDS.
enum Source { kDirect, kStaged, kGathered, kSpanned };

__device__ inline __amdgpu_buffer_rsrc_t window(const void* base, size_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)(bytes < 0x7fffffffu ? bytes : 0x7fffffffu), 0x00020000);
}

// A workgroup takes NC 16-column tiles and at most RT row tiles; its waves take the blocks of 128 kept rows in turn
// and add up their sums in LDS at the end, in wave order.  A block costs about 60 vector instructions a tile, which is what bounds
// the kernel beside the launch: addresses are scalars, ends are left to the descriptors' bounds, groups are unrolled.
// Measured: one row, 4096 x 4096 in fp32 4.0 us (9 MB; the launch alone is over 2); 8192 x 8192 2:8 4.2; 8 rows of bf16, 11008 x 4096 9.8
// (24 MB, 2.4 TB/s: one workgroup of 16 waves per compute unit, a matrix instruction for half a tile of rows); 13 rows,
// 4096 x 14336 2:4 8.4 (17 MB).
// MX: rows of x the instance has registers for; UNITS: scaled groups in a block.
// What an instance needs registers for decides how many waves it runs with (us with sixteen waves, which spill, and eight: 13 rows of
// bf16, 4096 x 14336 in groups of 32 23.5 and 19.0; fp32, 8 rows, 2:4 in groups of 32 36.6 and 18.2).
constexpr int most_waves(Source SRC, int RT, int NC, int MX, int UNITS)
{
    return (MX > 8 && !(SRC == kSpanned && NC * UNITS < 8)) || (RT > 1 && MX == 1) ||
                   (UNITS == 4 && (RT > 1 || (NC == 2 && MX != 4))) || (UNITS == 2 && RT > 1 && SRC == kGathered)
               ? kMaxWaves / 2
               : kMaxWaves;
}

// Blocks under way at a time.  Many rows take many registers: there more waves hide more than more loads of one (13 rows, 4096 x 14336 2:4
// 11.2 us with two blocks and 180 registers, 8.4 with one and 92; 8 rows of fp32 14.8 and 12.7).  Gathered elements need two.
constexpr int depth_of(Source src, int RT, int NC, int MX, int UNITS)
{
    if ((src == kSpanned || src == kStaged) && MX >= 8)
        return 1;
    if (src == kDirect)
        return RT == 1 && NC == 1 && UNITS < 4 ? 3 : 2;
    return MX == 1 ? (NC == 1 ? 4 : UNITS < 4 ? 3 : 2) : MX == 4 && NC == 1 ? 3 : 2;
}

template <ElementType T, Source SRC, int RT, int NC, int MX, int UNITS>
__global__ void __launch_bounds__(most_waves(SRC, RT, NC, MX, UNITS) * 64)
q4_rows_product_kernel(const void* __restrict__ x_, size_t ldx, const uint32_t* __restrict__ codes, Q4Meta meta,
                       const uint8_t* __restrict__ rows, const float* __restrict__ bias, void* __restrict__ y, size_t ldy, int M,
                       Q4Shape p, bool pairs)
{
    constexpr int S = T == kF32 ? 3 : 1;              // staged rows per row of x
    constexpr int RowsPerTile = T == kF32 ? 4 : 16;
    constexpr int Chunk = RT * RowsPerTile;           // rows of x per workgroup
    constexpr int Steps = 4 / UNITS;                  // of 32 rows in a unit
    constexpr int Size = T == kF32 ? 4 : 2;
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int c = lane & 15, kb = lane >> 4;
    const int tile0 = blockIdx.x * NC;
    uint16_t* const stage = reinterpret_cast<uint16_t*>(lds) + (size_t)wave * (MX * S * (SRC == kSpanned ? kSpanPitch : kRowPitch));

    f32x4 total[RT][NC];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int j = 0; j < NC; ++j)
            total[t][j] = f32x4{0, 0, 0, 0};
    const uint32_t unit = T == kF16 ? 0x3c003c00u : 0x3f803f80u;
    const u32x4 unit8 = u32x4{unit, unit, unit, unit};
    const uint32_t sixteen = sixteens<T>();

    // this lane's place in x: its row and first element of a step, or its two kept rows of a block
    const __amdgpu_buffer_rsrc_t all = window(x_, ((size_t)(M - 1) * ldx + p.K) * Size);
    uint32_t at_row[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
        at_row[t] = (uint32_t)(min(t * 16 + c, M - 1) * (uint32_t)ldx + kb * 8) * 2;

    struct Block {
        u32x4 w[NC], x[SRC == kDirect ? RT : 1][4], span[MX / 2 + 1];
        u32x2 places[4];
        uint32_t mt[NC][UNITS], xs[MX][2], two;
    };
    auto load = [&](int b, Block& n) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            n.w[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(codes) + ((size_t)(tile0 + j) * p.blocks + b) * 64 + lane);
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
                n.mt[j][u] = meta.word(tile0 + j, b * 128 + u * (128 / UNITS), c);
        }
        if (SRC == kDirect) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    n.x[t][s] = __builtin_amdgcn_raw_buffer_load_b128(all, (int)(at_row[t] + s * 64), b * 256, 0);
        } else if (SRC == kStaged) {
#pragma unroll
            for (int i = 0; i < MX; ++i) {
                const __amdgpu_buffer_rsrc_t r = window(static_cast<const char*>(x_) + (size_t)min(i, M - 1) * ldx * Size, (size_t)p.K * Size);
                const int at = lane * 2 * Size, first = b * 128 * Size;     // elements beyond K read as zero
                if (T == kF32) {
                    if (pairs) {
                        const auto two = __builtin_amdgcn_raw_buffer_load_b64(r, at, first, 0);
                        n.xs[i][0] = two[0];
                        n.xs[i][1] = two[1];
                    } else {
                        n.xs[i][0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, first, 0);
                        n.xs[i][1] = __builtin_amdgcn_raw_buffer_load_b32(r, at + Size, first, 0);
                    }
                } else if (pairs)
                    n.xs[i][0] = __builtin_amdgcn_raw_buffer_load_b32(r, at, first, 0);
                else {
                    n.xs[i][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at, first, 0);
                    n.xs[i][1] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at + Size, first, 0);
                }
            }
        } else if (SRC == kSpanned) {
            const int e = b * kSpan + (lane & 31) * 8;
#pragma unroll
            for (int i = 0; i < MX / 2; ++i) {      // beyond K: zeros, by an offset that no window holds
                const uint32_t at = ((uint32_t)min(2 * i + (lane >> 5), M - 1) * (uint32_t)ldx + e) * 2;
                n.span[i] = __builtin_amdgcn_raw_buffer_load_b128(all, (int)(e < p.K ? at : 0x7fffffffu), 0, 0);
            }
            const u32x2* const from = reinterpret_cast<const u32x2*>(rows + ((size_t)(tile0 >> 1) * p.blocks + b) * 128);
#pragma unroll
            for (int s = 0; s < 4; ++s)
                n.places[s] = from[s * 4 + kb];
        } else
            n.two = reinterpret_cast<const uint16_t*>(rows + (size_t)(tile0 >> 1) * p.blocks * 128 + b * 128)[lane];
    };
    // gathered elements: their places were loaded a block earlier
    auto gather = [&](int b, Block& n) {
        const int first = (b * 4 + (lane >> 4)) * p.span;
        const int at0 = (first + (int)(n.two & 255u)) * Size, at1 = (first + (int)(n.two >> 8)) * Size;
#pragma unroll
        for (int i = 0; i < MX; ++i) {
            const __amdgpu_buffer_rsrc_t r = window(static_cast<const char*>(x_) + (size_t)min(i, M - 1) * ldx * Size, (size_t)p.K * Size);
            if (T == kF32) {
                n.xs[i][0] = __builtin_amdgcn_raw_buffer_load_b32(r, at0, 0, 0);
                n.xs[i][1] = __builtin_amdgcn_raw_buffer_load_b32(r, at1, 0, 0);
            } else {
                n.xs[i][0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at0, 0, 0);
                n.xs[i][1] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at1, 0, 0);
            }
        }
    };
    // x of one step as matrix operands
    auto operand = [&](const Block& n, int s, u32x4 (&xa)[RT]) {
#pragma unroll
        for (int t = 0; t < RT; ++t)
            if (SRC == kDirect)
                xa[t] = n.x[t][s];
            else if (SRC == kSpanned) {
                const uint16_t* const row = stage + min(c, MX - 1) * kSpanPitch + s * 64;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t two = n.places[s][i >> 1] >> (i & 1) * 16;
                    xa[t][i] = (uint32_t)row[two & 255u] | (uint32_t)row[two >> 8 & 255u] << 16;
                }
            } else {
                const int i = T == kF32 ? min(t * 4 + (c >> 2), MX - 1) * 3 + min(c & 3, 2) : min(t * 16 + c, MX - 1);
                xa[t] = *reinterpret_cast<const u32x4*>(stage + i * kRowPitch + s * 32 + kb * 8);
            }
    };
    auto multiply = [&](const Block& n) {
        if (SRC == kSpanned) {
#pragma unroll
            for (int i = 0; i < MX / 2; ++i)
                *reinterpret_cast<u32x4*>(stage + (2 * i + (lane >> 5)) * kSpanPitch + (lane & 31) * 8) = n.span[i];
        } else if (SRC != kDirect) {
#pragma unroll
            for (int i = 0; i < MX; ++i) {
                uint32_t* const to = reinterpret_cast<uint32_t*>(stage + i * S * kRowPitch) + lane;
                if (T == kF32) {
                    uint32_t part[2][3];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float v = __uint_as_float(n.xs[i][e]);
                        const float v1 = v - __uint_as_float(__float_as_uint(v) & 0xffff0000u);
                        const float v2 = v1 - __uint_as_float(__float_as_uint(v1) & 0xffff0000u);
                        part[e][0] = __float_as_uint(v);
                        part[e][1] = __float_as_uint(v1);
                        part[e][2] = __float_as_uint(v2);
                    }
#pragma unroll
                    for (int q = 0; q < 3; ++q)     // the upper halves of the two
                        to[q * kRowPitch / 2] = __builtin_amdgcn_perm(part[1][q], part[0][q], 0x07060302u);
                } else
                    to[0] = SRC == kStaged && pairs ? n.xs[i][0] : n.xs[i][0] | n.xs[i][1] << 16;
            }
        }
        if (SRC != kDirect) {
            // the lanes of this wave read what its other lanes wrote: LDS operations of one wave take
            // effect in order, only the compiler has to be kept from reordering them
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        u32x4 xa[2][RT];        // a step's operands are read while the step before is multiplied
        operand(n, 0, xa[0]);
        f32x4 ones[RT], acc[RT][NC];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int u = s / Steps, i = s % Steps;
            if (s < 3)
                operand(n, s + 1, xa[(s + 1) & 1]);
#pragma unroll
            for (int t = 0; t < RT; ++t)
                ones[t] = product<T>(xa[s & 1][t], unit8, i ? ones[t] : f32x4{0, 0, 0, 0});
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const u32x4 wide = widened<T>(n.w[j][s], sixteen);
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    acc[t][j] = product<T>(xa[s & 1][t], wide, i ? acc[t][j] : f32x4{0, 0, 0, 0});
            }
            if (i == Steps - 1)
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    const float scale = __uint_as_float(n.mt[j][u] & ~15u);
                    const float offset = -(16.0f + (float)(n.mt[j][u] & 15u));
#pragma unroll
                    for (int t = 0; t < RT; ++t)
#pragma unroll
                        for (int e = 0; e < (T == kF32 ? 3 : 4); ++e)
                            total[t][j][e] = fmaf(scale, fmaf(offset, ones[t][e], acc[t][j][e]), total[t][j][e]);
                }
            if (SRC == kSpanned)
                __builtin_amdgcn_sched_barrier(0);
        }
        if (SRC != kDirect) {
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    };

    // DEPTH blocks' loads are under way at any time (a gathered x one block behind its places)
    constexpr int DEPTH = depth_of(SRC, RT, NC, MX, UNITS);
    Block blocks[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (wave + d * waves < p.blocks)
            load(wave + d * waves, blocks[d]);
    if (SRC == kGathered && wave < p.blocks)
        gather(wave, blocks[0]);
    for (int first = wave; first < p.blocks; first += DEPTH * waves)
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int b = first + d * waves;
            if (b >= p.blocks)
                break;
            if (SRC == kGathered && b + waves < p.blocks)
                gather(b + waves, blocks[(d + 1) % DEPTH]);
            multiply(blocks[d]);
            if (b + DEPTH * waves < p.blocks)
                load(b + DEPTH * waves, blocks[d]);
        }

    // the waves' sums: [wave][row][column]; an fp32 row is the sum of its three pieces, smallest first
    float* const part = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            if (T == kF32)
                part[((size_t)wave * Chunk + t * 4 + kb) * (NC * 16) + j * 16 + c] =
                    (total[t][j][2] + total[t][j][1]) + total[t][j][0];
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    part[((size_t)wave * Chunk + t * 16 + kb * 4 + e) * (NC * 16) + j * 16 + c] = total[t][j][e];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < M * (NC * 16); i += blockDim.x) {
        const int col = tile0 * 16 + i % (NC * 16);
        float sum = 0.0f;
#pragma unroll 8
        for (int v = 0; v < waves; ++v)
            sum += part[(size_t)v * Chunk * (NC * 16) + i];
        if (col < p.N) {
            if (bias)
                sum += bias[col];
            store_result<T>(y, (size_t)(i / (NC * 16)) * ldy + col, sum);
        }
    }
}

template <ElementType T, Source SRC, int RT, int NC, int MX, int UNITS>
hipError_t launch_rows(const Q4LinearArgs& a, bool pairs)
{
    constexpr int Chunk = RT * (T == kF32 ? 4 : 16);
    // one workgroup to a compute unit: sixteen waves each; more workgroups than that: eight (measured, us with 8 / 16 waves:
    // 4096 x 14336 dense 8.7 / 9.3, 2:4 5.7 / 7.0 at one row; 8192 x 8192 9.9 / 8.4, 11008 x 4096 9.3 / 8.0)
    int most = a.p.tiles / NC > machine().cus ? kMaxWaves / 2 : kMaxWaves;
    if (most > most_waves(SRC, RT, NC, MX, UNITS))
        most = most_waves(SRC, RT, NC, MX, UNITS);
    const size_t staged = SRC == kDirect ? 0 : (size_t)MX * (T == kF32 ? 3 : 1) * (SRC == kSpanned ? kSpanPitch : kRowPitch) * 2;
    const size_t sums = (size_t)Chunk * NC * 16 * sizeof(float);
    const size_t each = staged > sums ? staged : sums;
    int waves = a.p.blocks < most ? a.p.blocks : most;
    if (each * waves > kMostLds)
        waves = kMostLds / each;
    const size_t lds = each * waves;
    auto kernel = q4_rows_product_kernel<T, SRC, RT, NC, MX, UNITS>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess)
            return e;
    }
    kernel<<<a.p.tiles / NC, waves * 64, lds, a.stream>>>(
        a.x, a.ldx, a.codes, a.meta, a.rows, a.bias, a.y, a.ldy, a.M, a.p, pairs);
    return hipGetLastError();
}

// From where on two column tiles share a workgroup's x: as soon as the compute units are covered (8192 x 8192 at one row: 9.2 -> 8.4 us,
// 4096 x 4096: 4.2 -> 5.0).
bool pair_columns(const Q4LinearArgs& a) { return a.p.tiles >= 2 * machine().cus; }

template <ElementType T, Source SRC, int RT, int MX, int UNITS>
hipError_t launch_columns(const Q4LinearArgs& a, bool pairs)
{
    // nine and more fp32 rows of small groups hold too much for two tiles (13 rows, 4096 x 14336, groups of 32: 78 us; the dense ones
    // of them are not taken here at all)
    constexpr bool both = !(T == kF32 && MX == 16 && UNITS > (SRC == kGathered ? 2 : 1));
    if constexpr (both)
        if (pair_columns(a))
            return launch_rows<T, SRC, RT, 2, MX, UNITS>(a, pairs);
    return launch_rows<T, SRC, RT, 1, MX, UNITS>(a, pairs);
}

template <ElementType T, Source SRC, int RT, int MX>
hipError_t launch_units(const Q4LinearArgs& a, bool pairs)
{
    return a.meta.group >= 128  ? launch_columns<T, SRC, RT, MX, 1>(a, pairs)
           : a.meta.group == 64 ? launch_columns<T, SRC, RT, MX, 2>(a, pairs)
                                : launch_columns<T, SRC, RT, MX, 4>(a, pairs);
}

template <ElementType T, Source SRC>
hipError_t launch_source(const Q4LinearArgs& a, bool pairs)
{
    if constexpr (SRC == kDirect)
        return a.M <= 16 ? launch_units<T, SRC, 1, 1>(a, pairs) : launch_units<T, SRC, 2, 1>(a, pairs);
    else {
        if constexpr (SRC != kSpanned) {
            if (a.M == 1)
                return launch_units<T, SRC, 1, 1>(a, pairs);
            if (a.M <= 4)
                return launch_units<T, SRC, 1, 4>(a, pairs);
        }
        if constexpr (T != kF32 && SRC == kStaged)      // (few_rows)
            return launch_units<T, SRC, 1, 8>(a, pairs);
        else
            return a.M <= 8 ? launch_units<T, SRC, T == kF32 ? 2 : 1, 8>(a, pairs) : launch_units<T, SRC, T == kF32 ? 4 : 1, 16>(a, pairs);
    }
}

// x can be read as matrix operands where it lies
bool direct(const Q4LinearArgs& a, ElementType type)
{
    return type != kF32 && !a.rows && a.p.K % 128 == 0 && a.ldx % 8 == 0 && a.ldx < (1u << 24) && (reinterpret_cast<uintptr_t>(a.x) & 15u) == 0;
}

// All elements that a block spans are read, in whole 16-byte pieces, where gathering would be what bounds the kernel (us, gathered
// in memory / in LDS: 4096 x 14336 2:4 at 13 rows 13.7 / 8.4, at 8 rows 8.0 / 6.8; 4096 x 4096 at 8 rows 4.8 / 4.5, at 4 rows 3.7 / 4.1).
bool spanned(const Q4LinearArgs& a)
{
    return a.M > 4 && a.p.m == 2 * a.p.n && a.p.K % 8 == 0 && a.ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15u) == 0;
}

// Whether the kernel above takes the rows.  Measured against the other one (q4_gemm.hip), us at 4096 x 4096: as they lie, 16 / 32
// rows 6.4 / 10.1 against 12 / 14.3 (11008 x 4096: 14 / 23.4 against 17.5 with 32); fp32, 8 / 16 rows 6.9 / 12.0 against 12.3 / 13.9;
// 16-bit rows that are not aligned, 16 of them 27.9 against 12; at 4096 x 14336 fp32, 13 against 17 rows, groups of 128 / 64 / 32
// 23.2 / 29.8 / 49.4 against 24.0 / 24.6 / 32.4.
bool few_rows(const Q4LinearArgs& a, ElementType type)
{
    if (direct(a, type))
        return a.M <= 16 || (a.M <= 32 && a.p.blocks <= 48);
    if (type == kF32 && !a.rows && a.meta.group < 128 && pair_columns(a))
        return a.M <= 8;
    return a.M <= (type == kF32 || a.rows ? 16 : 8);
}

} // namespace

hipError_t launch_q4_linear(const Q4LinearArgs& given, ElementType type, void* workspace)
{
    Q4LinearArgs a = given;
    const bool densified = q4_densifies(a.p, a.M, type);
    if (densified) {
        const hipError_t e = launch_q4_densify(a, static_cast<uint32_t*>(workspace));
        if (e != hipSuccess)
            return e;
        a.codes = static_cast<const uint32_t*>(workspace);
        a.meta.group = a.meta.group * a.p.m / a.p.n;
        while ((1 << a.meta.group_shift) < a.meta.group)
            ++a.meta.group_shift;
        a.rows = nullptr;
        a.p.W = a.p.K;
        a.p.blocks = (a.p.K + 127) / 128;
    }
    const size_t size = type == kF32 ? 4 : 2;
    if (a.rows && a.M > 16) {       // sixteen rows at a time (q4_gathered_rows)
        Q4LinearArgs part = a;
        for (int first = 0; first < a.M; first += 16) {
            part.M = a.M - first < 16 ? a.M - first : 16;
            part.x = static_cast<const char*>(a.x) + first * a.ldx * size;
            part.y = static_cast<char*>(a.y) + first * a.ldy * size;
            const hipError_t e = launch_q4_linear(part, type, nullptr);
            if (e != hipSuccess)
                return e;
        }
        return hipSuccess;
    }
    if (densified || !few_rows(a, type))
        return launch_q4_gemm(a, type, densified, workspace);
    const uintptr_t base = reinterpret_cast<uintptr_t>(a.x);
    // a lane's two neighbouring elements in one load
    const bool pairs = base % (2 * size) == 0 && a.ldx % 2 == 0 && a.p.K % 2 == 0;
    if (a.rows) {
        if (type == kF32)
            return launch_source<kF32, kGathered>(a, pairs);
        if (spanned(a))
            return type == kBF16 ? launch_source<kBF16, kSpanned>(a, pairs) : launch_source<kF16, kSpanned>(a, pairs);
        return type == kBF16 ? launch_source<kBF16, kGathered>(a, pairs) : launch_source<kF16, kGathered>(a, pairs);
    }
    if (type == kF32)
        return launch_source<kF32, kStaged>(a, pairs);
    if (direct(a, type))
        return type == kBF16 ? launch_source<kBF16, kDirect>(a, pairs) : launch_source<kF16, kDirect>(a, pairs);
    return type == kBF16 ? launch_source<kBF16, kStaged>(a, pairs) : launch_source<kF16, kStaged>(a, pairs);
}

} // namespace nmspmm
