// y = x B for a B in 4 bits and many rows of x (the mathematics: q4_linear.hip; the layout: q4.hip).
//
// A workgroup computes 64 rows x 64 NC columns, each of its four waves all 64 rows of 16 NC columns: a code is
// widened once (a shift and a mask-and-or for two) and used for four row tiles.  The codes come straight from
// memory into the operand registers, their layout being that of the operands; x goes through LDS (64 rows x 128
// elements, two buffers, 16-byte pieces swapped by row so that the sixteen rows of a read lie in different
// banks).  The group sums of x, with which the offset of the widened codes is taken off, are made beforehand
// by the kernel that also cuts fp32 activations into their three bf16 pieces or copies rows that are not aligned.
#include "internal.h"
#include "q4_device.h"

namespace nmspmm {

namespace {

constexpr int kRows = 64;               // rows of x per workgroup
constexpr int kTileBytes = kRows * 256; // a 64 x 128 tile of x

// ---- x: its pieces, and its sums over the dense rows of each group (at most 128 at a time) ---------------

// One wave per 512 elements of a row, eight each lane.  PLANES 0: only the sums.  Pieces: [plane][row][K filled up to 128].
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
    if (k0 < Kp && (lane & (unit / 8 - 1)) == 0)
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
            *reinterpret_cast<u32x4*>(planes + ((size_t)q * M + row) * Kp + k0) = w;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = __float_as_uint(__uint_as_float(v[e]) - __uint_as_float(v[e] & 0xffff0000u));
        }
    }
}

// ---- a sparse operand's codes as those of a dense one: the zero point where no row was kept ----------------

__global__ void __launch_bounds__(256)
q4_densify_kernel(const uint32_t* __restrict__ codes, const uint32_t* __restrict__ meta, const uint8_t* __restrict__ rows,
                  Q4Shape p, int dense_blocks, uint32_t* __restrict__ out)
{
    const int lane = threadIdx.x & 63, c = lane & 15, kb = lane >> 4;
    const int tile = blockIdx.y * 4 + (threadIdx.x >> 6), block = blockIdx.x;
    if (tile >= p.tiles)
        return;
    const int per = 128 / p.group;
    u32x4 word;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int d0 = block * 128 + s * 32 + kb * 8;       // eight dense rows
        // the kept rows that can lie among them: those of their windows, or of the one window they are a part of
        const int count = p.m > 8 ? p.n : 8 / p.m * p.n;
        const int r0 = d0 / p.m * p.n;                      // a multiple of count: all in one word
        const int b = r0 >> 7, step = (r0 >> 5) & 3, part = (r0 >> 3) & 3;
        uint32_t dense = 0x88888888u;
        if (d0 < p.K) {
            const size_t at = (size_t)tile * p.blocks + b;
            const uint32_t zero = meta[(at * 16 + c) * per + step * per / 4] & 15u;
            dense = zero * 0x11111111u;
            const uint32_t packed = codes[(at * 64 + part * 16 + c) * 4 + step];
            const uint8_t* const off = rows + (size_t)(tile >> 1) * p.blocks * 128 + r0;
            const int base = (r0 >> 5) * p.span - d0;
            for (int i = 0; i < count; ++i) {
                const int e = (r0 & 7) + i;
                const int d = base + off[i];                // 0..7 if it is among the eight
                const uint32_t q = (packed >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u;
                const int to = 4 * ((d >> 1) + 4 * (d & 1));
                if (d >= 0 && d < 8 && r0 + i < p.W)
                    dense = (dense & ~(15u << to)) | q << to;
            }
        }
        word[s] = dense;
    }
    *reinterpret_cast<u32x4*>(out + (((size_t)tile * dense_blocks + block) * 64 + lane) * 4) = word;
}

// ---- the product --------------------------------------------------------------------------------------------

struct GemmArgs {
    const uint16_t* x;      // [plane][M][ldx]
    size_t plane, ldx;
    const float* sums;      // [K / unit][sums_ld]
    size_t sums_ld;
    const uint32_t* codes;  // dense
    Q4Meta meta;
    const float* bias;
    void* y;
    size_t ldy;
    int M, N, Kx;           // Kx: elements of a row of x, a multiple of 128
    int blocks, unit;       // dense blocks of 128 rows; rows after which sums are scaled (32, 64, 128)
    int tiles, tiles_m, tiles_n;    // 16-column tiles of the operand; workgroups along rows and columns
};

// UNITS: how often in a block of 128 rows sums are scaled, 128 / unit.
template <ElementType T, int PLANES, ElementType OUT, int NC, int UNITS>
__global__ void __launch_bounds__(256, 2)
q4_gemm_kernel(GemmArgs g)
{
    __shared__ __attribute__((aligned(16))) unsigned char tile[2][kTileBytes];
    __shared__ __attribute__((aligned(16))) float sums[2][UNITS][kRows];
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
    const int m0 = (band * 8 + inside % height) * kRows, tile0 = (inside / height) * (4 * NC) + wave * NC;
    const int rows_here = min(kRows, g.M - m0);

    f32x4 acc[4][NC], total[4][NC];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < NC; ++j)
            acc[t][j] = total[t][j] = f32x4{0, 0, 0, 0};

    // this lane's 16-byte pieces of a tile of x: rows 16 wave + 4 i + lane / 16, the piece that belongs at place lane % 16
    uint32_t piece[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = wave * 16 + i * 4 + kb;
        piece[i] = (uint32_t)(row * g.ldx * 2) + ((c ^ (row & 15)) * 16);
    }
    // Through registers and not straight into LDS: behind such a load the compiler lets every LDS read wait for it.
    u32x4 xr[4];
    uint32_t sr = 0;
    auto fetch_x = [&](int b, int q) {
        const uint16_t* const base = g.x + q * g.plane + (size_t)m0 * g.ldx + b * 128;
        const uint32_t bytes = (uint32_t)(((size_t)(rows_here - 1) * g.ldx + (g.Kx - b * 128)) * 2);    // rows beyond M read as zero
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, (int)bytes, 0x00020000);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            xr[i] = __builtin_amdgcn_raw_buffer_load_b128(r, (int)piece[i], 0, 0);
    };
    auto put_x = [&](int half) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<u32x4*>(tile[half] + (wave * 16 + i * 4) * 256 + lane * 16) = xr[i];
    };
    auto fetch_sums = [&](int b) {
        if (wave < UNITS) {
            const float* const base = g.sums + (size_t)(b * UNITS + wave) * g.sums_ld + m0;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, rows_here * 4, 0x00020000);
            sr = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, lane * 4, 0, 0);
        }
    };
    auto put_sums = [&](int b) {
        if (wave < UNITS)
            sums[b & 1][wave][lane] = __uint_as_float(sr);
    };
    constexpr int Steps = 4 / UNITS;    // of 32 rows in a unit
    u32x4 w[NC], wn[NC];
    uint32_t mt[NC][UNITS];
    auto fetch_codes = [&](int b) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int t = min(tile0 + j, g.tiles - 1);      // beyond the last column: read, not used
            wn[j] = (reinterpret_cast<const u32x4*>(g.codes) + ((size_t)t * g.blocks + b) * 64)[lane];
        }
    };
    auto fetch_meta = [&](int b) {
#pragma unroll
        for (int j = 0; j < NC; ++j)
#pragma unroll
            for (int u = 0; u < UNITS; ++u)
                mt[j][u] = g.meta.word(min(tile0 + j, g.tiles - 1), b * 128 + u * (128 / UNITS), c);
    };

    fetch_x(0, 0);
    fetch_sums(0);
    fetch_codes(0);
    put_x(0);
    put_sums(0);
    const int stages = g.blocks * PLANES;
    for (int stage = 0, b = 0, q = 0; stage < stages; ++stage) {
        if (q == 0) {
#pragma unroll
            for (int j = 0; j < NC; ++j)
                w[j] = wn[j];
            fetch_meta(b);      // wanted when the first unit ends
        }
        __syncthreads();        // this stage's tile is whole, and nobody reads the other any more
        const int half = stage & 1;
        const int bq = b, qq = q;
        if (++q == PLANES) {
            q = 0;
            ++b;
        }
        if (stage + 1 < stages) {
            fetch_x(b, q);
            if (q == 0) {
                fetch_sums(b);
                fetch_codes(b);
            }
        }
        // the sums of a unit are scaled when it ends; the pieces of one fp32 x share the sum of x, which is taken off once
        const bool last = qq == PLANES - 1;
#pragma clang loop unroll(disable)
        for (int u = 0; u < UNITS; ++u) {       // (unrolled, smaller units would need more registers than there are)
#pragma unroll
            for (int i = 0; i < Steps; ++i) {
                const int s = u * Steps + i;
                u32x4 a[4];
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    a[t] = *reinterpret_cast<const u32x4*>(tile[half] + (t * 16 + c) * 256 + (((s * 4 + kb) ^ c) * 16));
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    const uint32_t word = UNITS == 1 ? w[j][i] : UNITS == 2 ? (u ? w[j][i + 2] : w[j][i])
                                                     : u == 0 ? w[j][0] : u == 1 ? w[j][1] : u == 2 ? w[j][2] : w[j][3];
                    const u32x4 wide = widened<T>(word);
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        acc[t][j] = product<T>(a[t], wide, acc[t][j]);
                }
            }
            if (last || UNITS > 1) {
                f32x4 xs[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    xs[t] = *reinterpret_cast<const f32x4*>(&sums[bq & 1][u][t * 16 + kb * 4]);
                    if (PLANES > 1 && !last)
                        xs[t] = f32x4{0, 0, 0, 0};
                }
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    const uint32_t word = UNITS == 1 ? mt[j][0] : UNITS == 2 ? (u ? mt[j][UNITS - 1] : mt[j][0])
                                                     : u == 0 ? mt[j][0] : u == 1 ? mt[j][1 % UNITS] : u == 2 ? mt[j][2 % UNITS] : mt[j][3 % UNITS];
                    const float scale = __uint_as_float(word & ~15u);
                    const float offset = -(16.0f + (float)(word & 15u));
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            total[t][j][e] = fmaf(scale, fmaf(offset, xs[t][e], acc[t][j][e]), total[t][j][e]);
                        acc[t][j] = f32x4{0, 0, 0, 0};
                    }
                }
            }
        }
        if (stage + 1 < stages) {
            put_x(half ^ 1);
            if (q == 0)
                put_sums(b);
        }
    }

#pragma unroll
    for (int j = 0; j < NC; ++j) {
        const int col = (tile0 + j) * 16 + c;
        if (col >= g.N)
            continue;
        const float bias = g.bias ? g.bias[col] : 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = t * 16 + kb * 4 + e;
                if (row < rows_here)
                    store_result<OUT>(g.y, (size_t)(m0 + row) * g.ldy + col, total[t][j][e] + bias);
            }
    }
}

template <ElementType T, int PLANES, ElementType OUT, int UNITS>
void run_units(GemmArgs& g, hipStream_t stream)
{
    g.tiles_m = (g.M + kRows - 1) / kRows;
    g.tiles_n = (g.tiles + 15) / 16;
    if (g.tiles_m * g.tiles_n >= 2 * machine().cus) {
        q4_gemm_kernel<T, PLANES, OUT, 4, UNITS><<<g.tiles_m * g.tiles_n, 256, 0, stream>>>(g);
    } else {
        g.tiles_n = (g.tiles + 7) / 8;
        q4_gemm_kernel<T, PLANES, OUT, 2, UNITS><<<g.tiles_m * g.tiles_n, 256, 0, stream>>>(g);
    }
}

template <ElementType T, int PLANES, ElementType OUT>
void run_gemm(GemmArgs& g, hipStream_t stream)
{
    if (g.unit == 128)
        run_units<T, PLANES, OUT, 1>(g, stream);
    else if (g.unit == 64)
        run_units<T, PLANES, OUT, 2>(g, stream);
    else
        run_units<T, PLANES, OUT, 4>(g, stream);
}

size_t round_up(size_t v, size_t to) { return (v + to - 1) / to * to; }

} // namespace

// What lies where in the workspace (bytes): the densified codes, the sums, the pieces of x.
struct GemmSpace {
    size_t codes, sums, planes, bytes;
};
static GemmSpace gemm_space(const Q4Shape& p, int M, ElementType type, bool codes, bool product, bool planes)
{
    const size_t blocks = ((size_t)p.K + 127) / 128;
    GemmSpace s;
    s.codes = 0;
    s.sums = codes ? p.tiles * blocks * 1024 : 0;
    s.planes = s.sums + (product ? round_up(blocks * 4 * round_up(M, 4) * sizeof(float), 256) : 0);
    s.bytes = s.planes + (product && planes ? (type == kF32 ? 3 : 1) * (size_t)M * blocks * 256 : 0);
    return s;
}

bool q4_uses_gemm(const Q4Shape&, int M) { return M > 64; }
bool q4_densifies(const Q4Shape& p, int M) { return p.m > 1 && M > 16; }

size_t q4_workspace_bytes(const Q4Shape& p, int M, ElementType type)
{
    return gemm_space(p, M, type, q4_densifies(p, M), q4_uses_gemm(p, M), true).bytes;
}

hipError_t launch_q4_densify(const Q4LinearArgs& a, uint32_t* out)
{
    const int blocks = (a.p.K + 127) / 128;
    q4_densify_kernel<<<dim3(blocks, (a.p.tiles + 3) / 4), 256, 0, a.stream>>>(a.codes, a.meta.words, a.rows, a.p, blocks, out);
    return hipGetLastError();
}

// `a` is dense by now (q4_linear.hip).
hipError_t launch_q4_gemm(const Q4LinearArgs& a, ElementType type, bool densified, void* workspace)
{
    const GemmSpace s = gemm_space(a.p, a.M, type, densified, true, true);
    char* const base = static_cast<char*>(workspace);
    const int Kp = a.p.blocks * 128;
    GemmArgs g;
    g.unit = a.meta.group < 128 ? a.meta.group : 128;
    g.sums = reinterpret_cast<float*>(base + s.sums);
    g.sums_ld = round_up(a.M, 4);
    g.codes = a.codes;
    g.meta = a.meta;
    g.bias = a.bias;
    g.y = a.y;
    g.ldy = a.ldy;
    g.M = a.M;
    g.N = a.p.N;
    g.Kx = Kp;
    g.blocks = a.p.blocks;
    g.tiles = a.p.tiles;
    uint16_t* const planes = reinterpret_cast<uint16_t*>(base + s.planes);
    const dim3 grid((a.M + 3) / 4, (Kp + 511) / 512);
    // x as it is: 16-bit elements, rows of whole blocks on 16-byte boundaries, 64 of them within 2 GiB
    const bool as_is = type != kF32 && a.p.K == Kp && a.ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15u) == 0 &&
                       a.ldx < (1u << 23);
    float* const sums = const_cast<float*>(g.sums);
    if (as_is) {
        g.x = static_cast<const uint16_t*>(a.x);
        g.ldx = a.ldx;
        g.plane = 0;
        if (type == kBF16)
            q4_prepare_x_kernel<kBF16, 0><<<grid, 256, 0, a.stream>>>(a.x, a.ldx, a.M, a.p.K, Kp, g.unit, nullptr, sums, g.sums_ld);
        else
            q4_prepare_x_kernel<kF16, 0><<<grid, 256, 0, a.stream>>>(a.x, a.ldx, a.M, a.p.K, Kp, g.unit, nullptr, sums, g.sums_ld);
    } else {
        g.x = planes;
        g.ldx = Kp;
        g.plane = (size_t)a.M * Kp;
        if (type == kF32)
            q4_prepare_x_kernel<kF32, 3><<<grid, 256, 0, a.stream>>>(a.x, a.ldx, a.M, a.p.K, Kp, g.unit, planes, sums, g.sums_ld);
        else if (type == kBF16)
            q4_prepare_x_kernel<kBF16, 1><<<grid, 256, 0, a.stream>>>(a.x, a.ldx, a.M, a.p.K, Kp, g.unit, planes, sums, g.sums_ld);
        else
            q4_prepare_x_kernel<kF16, 1><<<grid, 256, 0, a.stream>>>(a.x, a.ldx, a.M, a.p.K, Kp, g.unit, planes, sums, g.sums_ld);
    }
    if (type == kF32)
        run_gemm<kBF16, 3, kF32>(g, a.stream);
    else if (type == kBF16)
        run_gemm<kBF16, 1, kBF16>(g, a.stream);
    else
        run_gemm<kF16, 1, kF16>(g, a.stream);
    return hipGetLastError();
}

} // namespace nmspmm
