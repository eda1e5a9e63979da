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
// An infinity or a NaN in a row of x makes that row of y NaN.
#include "internal.h"
#include "q4_device.h"

namespace nmspmm {

namespace {

constexpr int kMaxWaves = 16;
constexpr int kRowPitch = 136;      // 16-bit elements between staged rows: 128 and 16 bytes, so that the sixteen
                                    // rows of a 128-bit LDS read start in different banks

// How the activations reach the matrix operands: as they lie in memory (16-bit types, 16-byte aligned rows of whole
// 8-element pieces), or through the wave's own part of LDS, from consecutive or from gathered elements.
enum Source { kDirect, kStaged, kGathered };

// A workgroup takes NC 16-column tiles and at most RT row tiles; its waves take the blocks of 128 kept rows in turn
// and add up their sums in LDS at the end, in wave order.  MX: rows of x the instance has registers for.
template <ElementType T, Source SRC, int RT, int NC, int MX>
__global__ void __launch_bounds__(kMaxWaves * 64)
q4_rows_product_kernel(const void* __restrict__ x_, size_t ldx, const uint32_t* __restrict__ codes,
                       Q4Meta meta, const uint8_t* __restrict__ rows, const float* __restrict__ bias,
                       void* __restrict__ y, size_t ldy, int M, Q4Shape p, bool pairs)
{
    constexpr int S = T == kF32 ? 3 : 1;              // staged rows per row of x
    constexpr int RowsPerTile = T == kF32 ? 4 : 16;
    constexpr int Chunk = RT * RowsPerTile;           // rows of x per workgroup
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int c = lane & 15, kb = lane >> 4;
    const int tile0 = blockIdx.x * NC, m0 = blockIdx.y * Chunk;
    const int rows_here = min(Chunk, M - m0);
    // groups of 128 rows and more are scaled once a block, smaller ones when they end
    const int units = meta.group < 128 ? 128 / meta.group : 1, step_mask = 4 / units - 1, unit_shift = units == 4 ? 0 : units == 2 ? 1 : 2;
    uint16_t* const stage = reinterpret_cast<uint16_t*>(lds) + (size_t)wave * (MX * S * kRowPitch);

    f32x4 total[RT][NC], acc[RT][NC], ones[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        ones[t] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < NC; ++j)
            total[t][j] = acc[t][j] = f32x4{0, 0, 0, 0};
    }
    const uint32_t unit = T == kF16 ? 0x3c003c00u : 0x3f803f80u;
    const u32x4 unit8 = u32x4{unit, unit, unit, unit};

    u32x4 w[NC], mt[NC] = {}, xd[RT][4];
    uint32_t xs[MX][2];
    auto load = [&](int b) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const size_t at = (size_t)(tile0 + j) * p.blocks + b;
            w[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(codes) + at * 64 + lane);
#pragma unroll
            for (int g = 0; g < 4; ++g)
                if (g < units)
                    mt[j][g] = meta.word(tile0 + j, b * 128 + g * meta.group, c);
        }
        if (SRC == kDirect) {
            const uint16_t* const x = static_cast<const uint16_t*>(x_);
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int row = min(m0 + t * 16 + c, M - 1), k = b * 128 + s * 32 + kb * 8;
                    u32x4 v = *reinterpret_cast<const u32x4*>(x + (size_t)row * ldx + min(k, p.K - 8));
                    if (k >= p.K)
                        v = u32x4{0, 0, 0, 0};
                    xd[t][s] = v;
                }
        } else {
            const int r = b * 128 + lane * 2;       // this lane's two kept rows
            int k0 = r, k1 = r + 1;
            if (SRC == kGathered) {
                const uint32_t two = *reinterpret_cast<const uint16_t*>(rows + (size_t)(tile0 >> 1) * p.blocks * 128 + r);
                const int base = (r >> 5) * p.span;
                k0 = base + (int)(two & 255u);
                k1 = base + (int)(two >> 8);
            }
            const bool in0 = r < p.W && k0 < p.K, in1 = r + 1 < p.W && k1 < p.K;
            k0 = in0 ? k0 : 0;
            k1 = in1 ? k1 : 0;
#pragma unroll
            for (int i = 0; i < MX; ++i) {
                const size_t row = (size_t)min(m0 + i, M - 1) * ldx;
                if (T == kF32) {
                    const uint32_t* const x = static_cast<const uint32_t*>(x_) + row;
                    if (SRC == kStaged && pairs && in1) {
                        const uint2 two = *reinterpret_cast<const uint2*>(x + k0);
                        xs[i][0] = two.x;
                        xs[i][1] = two.y;
                    } else {
                        xs[i][0] = in0 ? x[k0] : 0u;
                        xs[i][1] = in1 ? x[k1] : 0u;
                    }
                } else {
                    const uint16_t* const x = static_cast<const uint16_t*>(x_) + row;
                    if (SRC == kStaged && pairs && in1)
                        xs[i][0] = *reinterpret_cast<const uint32_t*>(x + k0);
                    else
                        xs[i][0] = (in0 ? x[k0] : 0u) | (in1 ? (uint32_t)x[k1] << 16 : 0u);
                }
            }
        }
    };

    if (wave < p.blocks)
        load(wave);
    for (int b = wave; b < p.blocks; b += waves) {
        u32x4 wn[NC], mn[NC], xa[RT][4];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            wn[j] = w[j];
            mn[j] = mt[j];
        }
        if (SRC == kDirect) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    xa[t][s] = xd[t][s];
        } else {
#pragma unroll
            for (int i = 0; i < MX; ++i) {
                uint32_t* const to = reinterpret_cast<uint32_t*>(stage + (size_t)i * S * kRowPitch) + lane;
                if (T == kF32) {
                    uint32_t part[2][3];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float v = __uint_as_float(xs[i][e]);
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
                    to[0] = xs[i][0];
            }
            // the lanes of this wave read what its other lanes wrote: LDS operations of one wave take
            // effect in order, only the compiler has to be kept from reordering them
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const int i = T == kF32 ? min(t * 4 + (c >> 2), MX - 1) * 3 + min(c & 3, 2) : min(t * 16 + c, MX - 1);
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    xa[t][s] = *reinterpret_cast<const u32x4*>(stage + (size_t)i * kRowPitch + s * 32 + kb * 8);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        if (b + waves < p.blocks)
            load(b + waves);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
                ones[t] = product<T>(xa[t][s], unit8, ones[t]);
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const u32x4 u = widened<T>(wn[j][s]);
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    acc[t][j] = product<T>(xa[t][s], u, acc[t][j]);
            }
            if ((s & step_mask) == step_mask) {     // the group ends with this step
                const int g = s >> unit_shift;
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    const uint32_t word = g == 0 ? mn[j][0] : g == 1 ? mn[j][1] : g == 2 ? mn[j][2] : mn[j][3];
                    const float scale = __uint_as_float(word & ~15u);
                    const float offset = -(16.0f + (float)(word & 15u));
#pragma unroll
                    for (int t = 0; t < RT; ++t) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            total[t][j][e] = fmaf(scale, fmaf(offset, ones[t][e], acc[t][j][e]), total[t][j][e]);
                        acc[t][j] = f32x4{0, 0, 0, 0};
                    }
                }
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    ones[t] = f32x4{0, 0, 0, 0};
            }
        }
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
    for (int i = threadIdx.x; i < rows_here * (NC * 16); i += blockDim.x) {
        const int col = tile0 * 16 + i % (NC * 16);
        float sum = 0.0f;
#pragma unroll 8
        for (int v = 0; v < waves; ++v)
            sum += part[(size_t)v * Chunk * (NC * 16) + i];
        if (col < p.N) {
            if (bias)
                sum += bias[col];
            store_result<T>(y, (size_t)(m0 + i / (NC * 16)) * ldy + col, sum);
        }
    }
}

template <ElementType T, Source SRC, int RT, int NC, int MX>
hipError_t launch_rows(const Q4LinearArgs& a, bool pairs)
{
    constexpr int Chunk = RT * (T == kF32 ? 4 : 16);
    const int waves = a.p.blocks < kMaxWaves ? a.p.blocks : kMaxWaves;
    const size_t staged = SRC == kDirect ? 0 : (size_t)waves * MX * (T == kF32 ? 3 : 1) * kRowPitch * 2;
    const size_t sums = (size_t)waves * Chunk * NC * 16 * sizeof(float);
    const size_t lds = staged > sums ? staged : sums;
    auto kernel = q4_rows_product_kernel<T, SRC, RT, NC, MX>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess)
            return e;
    }
    const dim3 grid(a.p.tiles / NC, (a.M + Chunk - 1) / Chunk);
    kernel<<<grid, waves * 64, lds, a.stream>>>(a.x, a.ldx, a.codes, a.meta, a.rows, a.bias, a.y, a.ldy, a.M, a.p, pairs);
    return hipGetLastError();
}

template <ElementType T, Source SRC>
hipError_t launch_source(const Q4LinearArgs& a, bool pairs)
{
    if (SRC == kDirect) {
        if (a.M <= 16)
            return launch_rows<T, SRC, 1, 1, 1>(a, pairs);
        return a.M <= 32 ? launch_rows<T, SRC, 2, 1, 1>(a, pairs) : launch_rows<T, SRC, 4, 1, 1>(a, pairs);
    }
    if (a.M == 1)
        return launch_rows<T, SRC, 1, 1, 1>(a, pairs);
    return launch_rows<T, SRC, 1, 1, T == kF32 ? 4 : 16>(a, pairs);
}

} // namespace

hipError_t launch_q4_linear(const Q4LinearArgs& given, ElementType type, void* workspace)
{
    Q4LinearArgs a = given;
    const bool densified = q4_densifies(a.p, a.M);
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
    if (q4_uses_gemm(a.p, a.M))
        return launch_q4_gemm(a, type, densified, workspace);
    const size_t size = type == kF32 ? 4 : 2;
    const uintptr_t base = reinterpret_cast<uintptr_t>(a.x);
    // a lane's two neighbouring elements in one load
    const bool pairs = base % (2 * size) == 0 && a.ldx % 2 == 0;
    if (a.rows) {
        if (type == kF32)
            return launch_source<kF32, kGathered>(a, pairs);
        return type == kBF16 ? launch_source<kBF16, kGathered>(a, pairs) : launch_source<kF16, kGathered>(a, pairs);
    }
    if (type == kF32)
        return launch_source<kF32, kStaged>(a, pairs);
    if (base % 16 == 0 && a.ldx % 8 == 0 && a.p.K % 8 == 0)
        return type == kBF16 ? launch_source<kBF16, kDirect>(a, pairs) : launch_source<kF16, kDirect>(a, pairs);
    return type == kBF16 ? launch_source<kBF16, kStaged>(a, pairs) : launch_source<kF16, kStaged>(a, pairs);
}

} // namespace nmspmm
