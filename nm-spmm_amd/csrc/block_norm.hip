// What stands between two blocks of a model, in one pass over the rows:
//     after = post(branch) w_post + b_post         (post: the RMS or the Layer norm of a row, or nothing)
//     sum   = residual * scale + after * gate
//     out   = pre(sum) w_pre + b_pre
// and its gradients.  With v^ = (v - mean) / deviation (mean 0 for the RMS norm) and D features,
//     d_sum'  = d_sum + (g - v^ mean(g v^) - mean(g)) / deviation,  g = d_out w_pre, v^ of sum (mean(g): Layer norm only)
//     d_residual = d_sum' scale;  d_branch: the same formula once more with g = d_sum' gate w_post, v^ of branch;
// the gradients of weights, biases, scale and gate are sums over rows of what stands next to them.
// HBM-bound: forward reads residual and branch and writes sum and out, once each; backward reads residual,
// branch, d_sum and d_out and writes d_residual and d_branch (sum is formed again: cheaper than to read its
// rounded value, and exact).  A row stays in the registers of its threads, 8 or 16 elements each; statistics
// and sums are fp32.  A thread keeps its columns' weights, and in the backward pass its columns' sums over
// rows, in registers while it walks through a contiguous range of rows; the ranges' sums go to the workspace and
// a second kernel adds them up in order, so that gradients repeat bit for bit.
#include "internal.h"

namespace nmspmm {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kMaxThreads = 1024;

__device__ inline float from_bits16(uint32_t bits, int type)
{
    if (type == kBF16)
        return __uint_as_float(bits << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}
__device__ inline uint32_t to_bits16(float v, int type)
{
    if (type == kBF16)
        return __builtin_bit_cast(uint16_t, (__bf16)v);
    return __builtin_bit_cast(uint16_t, (_Float16)v);
}

// The columns of a thread: eight consecutive ones, `stride` threads times eight between its groups of eight.  Where those reach
// beyond a row's end, the row's last eight (WIDE: rows of eight and more); what of them another thread has, or no one, does
// not count (owns).  So every access is 16 or 32 bytes, without a branch, and rows need no alignment beyond their elements'.
template <bool WIDE>
__device__ inline int column_of(int t, int stride, int v, int D)
{
    const int c = (t + v * stride) * 8;
    return WIDE ? min(c, D - 8) : c;
}
template <bool WIDE>
__device__ inline bool owns(int t, int stride, int v, int e, int D)
{
    const int c = column_of<WIDE>(t, stride, v, D) + e;
    return c >= (t + v * stride) * 8 && c < D;
}

// Eight elements as they lie in memory: loads of several tensors can be under way before the first is unpacked.
struct Raw {
    u32x4 a, b;
};
template <bool WIDE>
__device__ inline Raw load_raw(const void* p, int type, size_t row, int t, int stride, int v, int D)
{
    Raw r;
    const int c = column_of<WIDE>(t, stride, v, D);
    if (type == kF32) {
        const float* const q = static_cast<const float*>(p) + row;
        if (WIDE)
            __builtin_memcpy(&r, q + c, 32);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                (e < 4 ? r.a : r.b)[e & 3] = __float_as_uint(q[min(c + e, D - 1)]);
    } else {
        const uint16_t* const q = static_cast<const uint16_t*>(p) + row;
        if (WIDE)
            __builtin_memcpy(&r.a, q + c, 16);
        else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                r.a[e] = q[min(c + 2 * e, D - 1)] | (uint32_t)q[min(c + 2 * e + 1, D - 1)] << 16;
    }
    return r;
}
__device__ inline void unpack(const Raw& r, int type, float* out)
{
#pragma unroll
    for (int e = 0; e < 8; ++e)
        out[e] = type == kF32 ? __uint_as_float(e < 4 ? r.a[e & 3] : r.b[e & 3])
                              : from_bits16(e & 1 ? r.a[e >> 1] >> 16 : r.a[e >> 1] & 0xffffu, type);
}
template <bool WIDE>
__device__ inline void store8(void* p, int type, size_t row, int t, int stride, int v, int D, const float* x)
{
    const int c = (t + v * stride) * 8;
    const bool whole = c + 8 <= D;
    u32x4 w;
    if (type != kF32)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = to_bits16(x[2 * e], type) | to_bits16(x[2 * e + 1], type) << 16;
    if (whole) {
        if (type == kF32)
            __builtin_memcpy(static_cast<float*>(p) + row + c, x, 32);
        else
            __builtin_memcpy(static_cast<uint16_t*>(p) + row + c, &w, 16);
    } else if (c < D) {
        const int first = column_of<WIDE>(t, stride, v, D);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (owns<WIDE>(t, stride, v, e, D)) {
                if (type == kF32)
                    static_cast<float*>(p)[row + first + e] = x[e];
                else
                    static_cast<uint16_t*>(p)[row + first + e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            }
    }
}

// The sum over a row's lanes of a wave, in every one of them: neighbours, quads and rows of 16 by lane permutation within the vector unit, rows and halves by
// swapping them (an exchange through LDS takes ten times as long, and a row waits for six of them in turn).
template <int CTRL>
__device__ inline float exchanged(float v)
{
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
// Rows of 16 or 32 lanes share a wave: theirs stop there.
__device__ inline float lanes_sum(float v, int lanes)
{
    v += exchanged<0xb1>(v);        // lane ^ 1
    v += exchanged<0x4e>(v);        // lane ^ 2
    v += exchanged<0x141>(v);       // the other quad of eight
    v += exchanged<0x140>(v);       // the other half of sixteen
    if (lanes == 16)
        return v;
    const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
    if (lanes == 32)
        return v;
    const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
}

// Sums over the threads of a row: a wave, or the workgroup's waves through LDS (two halves used in turn: one barrier a sum).
struct RowSum {
    float (*slots)[2][kMaxThreads / 64];
    int half, waves, lanes;
    template <bool BOTH>
    __device__ void add(float& a, float& b)
    {
        a = lanes_sum(a, lanes);
        if (BOTH)
            b = lanes_sum(b, lanes);
        if (waves == 1)
            return;
        if ((threadIdx.x & 63) == 0) {
            slots[half][0][threadIdx.x >> 6] = a;
            if (BOTH)
                slots[half][1][threadIdx.x >> 6] = b;
        }
        __syncthreads();
        // (slots of waves that there are not hold zero)
        const float4* const from = reinterpret_cast<const float4*>(slots[half][0]);
        const float4 p = from[0], q = from[1], r = from[2], s = from[3];
        a = (((p.x + p.y) + (p.z + p.w)) + ((q.x + q.y) + (q.z + q.w))) + (((r.x + r.y) + (r.z + r.w)) + ((s.x + s.y) + (s.z + s.w)));
        if (BOTH) {
            const float4* const other = reinterpret_cast<const float4*>(slots[half][1]);
            const float4 t = other[0], u = other[1], v = other[2], w = other[3];
            b = (((t.x + t.y) + (t.z + t.w)) + ((u.x + u.y) + (u.z + u.w))) + (((v.x + v.y) + (v.z + v.w)) + ((w.x + w.y) + (w.z + w.w)));
        }
        half ^= 1;
    }
    __device__ void operator()(float& a)
    {
        float none = 0.0f;
        add<false>(a, none);
    }
    __device__ void operator()(float& a, float& b) { add<true>(a, b); }

    static __device__ void clear(float (*slots)[2][kMaxThreads / 64])
    {
        if (threadIdx.x < 4 * (kMaxThreads / 64))
            slots[0][0][threadIdx.x] = 0.0f;
        __syncthreads();
    }
};

// Mean (Layer norm) and 1 / deviation of the row whose elements the threads hold (zeros beyond D); v becomes v^.
template <int E>
__device__ inline void standardize(float* v, const bool* in, int kind, float inv_d, float eps, RowSum& sum, float& mean, float& inv)
{
    float a = 0.0f;
    mean = 0.0f;
    if (kind == kLayerNorm) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            a += v[e];
        sum(a);
        mean = a * inv_d;
#pragma unroll
        for (int e = 0; e < E; ++e)
            v[e] = in[e] ? v[e] - mean : 0.0f;
        a = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        a = fmaf(v[e], v[e], a);
    sum(a);
    inv = 1.0f / sqrtf(a * inv_d + eps);
#pragma unroll
    for (int e = 0; e < E; ++e)
        v[e] *= inv;
}

// The thread's columns of the parameters (1, 0 or the plain factor where there is none).
template <bool WIDE, int NV, bool BIAS>
struct Columns {
    float post_w[NV * 8], scale[NV * 8], pre_w[NV * 8], gate[NV * 8];
    float post_b[BIAS ? NV * 8 : 8], pre_b[BIAS ? NV * 8 : 8];

    // everything that does not change from row to row: all loads first, then their values
    __device__ void load(const BlockNormArgs& a, size_t gate_row, bool with_gate, int t, int stride)
    {
        Raw pw[NV], pb[NV], sc[NV], nw[NV], nb[NV], g[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (a.post_weight.data)
                pw[v] = load_raw<WIDE>(a.post_weight.data, a.post_weight.type, 0, t, stride, v, a.D);
            if (BIAS && a.post_bias.data)
                pb[v] = load_raw<WIDE>(a.post_bias.data, a.post_bias.type, 0, t, stride, v, a.D);
            if (a.scale.data)
                sc[v] = load_raw<WIDE>(a.scale.data, a.scale.type, 0, t, stride, v, a.D);
            if (a.pre_weight.data)
                nw[v] = load_raw<WIDE>(a.pre_weight.data, a.pre_weight.type, 0, t, stride, v, a.D);
            if (BIAS && a.pre_bias.data)
                nb[v] = load_raw<WIDE>(a.pre_bias.data, a.pre_bias.type, 0, t, stride, v, a.D);
            if (with_gate)
                g[v] = load_raw<WIDE>(a.gate.data, a.gate.type, gate_row * (size_t)a.D, t, stride, v, a.D);
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            value(a.post_weight, pw[v], 1.0f, a.weight_offset, post_w + v * 8);
            if (BIAS)
                value(a.post_bias, pb[v], 0.0f, 0.0f, post_b + v * 8);
            value(a.scale, sc[v], a.factor, 0.0f, scale + v * 8);
            value(a.pre_weight, nw[v], 1.0f, a.weight_offset, pre_w + v * 8);
            if (BIAS)
                value(a.pre_bias, nb[v], 0.0f, 0.0f, pre_b + v * 8);
            if (with_gate)
                unpack(g[v], a.gate.type, gate + v * 8);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    gate[v * 8 + e] = 1.0f;
        }
    }
    __device__ void load_gate(const BlockNormArgs& a, size_t gate_row, int t, int stride)
    {
#pragma unroll
        for (int v = 0; v < NV; ++v)
            unpack(load_raw<WIDE>(a.gate.data, a.gate.type, gate_row * (size_t)a.D, t, stride, v, a.D), a.gate.type, gate + v * 8);
    }

private:
    __device__ static void value(const BlockNormVec& p, const Raw& r, float missing, float offset, float* out)
    {
        if (p.data) {
            unpack(r, p.type, out);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                out[e] += offset;
        } else
#pragma unroll
            for (int e = 0; e < 8; ++e)
                out[e] = missing;
    }
};

// ---- forward ------------------------------------------------------------------------------------------
// 4096 rows of 8192 bf16: 57.5 us (268 MB, 4.7 TB/s, what a copy reaches); 1071 rows of 2049 fp32, whose accesses are not aligned: 22.5
// (44 MB, 2.0 TB/s); one row of 4096: 4.5, launch and two sums over 512 threads.

template <ElementType T, ElementType R, bool WIDE, int NV, int THREADS, bool BIAS>
__global__ void __launch_bounds__(THREADS)
block_norm_kernel(BlockNormArgs a, int row_threads, int walkers)
{
    __shared__ __attribute__((aligned(16))) float slots[2][2][kMaxThreads / 64];
    RowSum::clear(slots);
    constexpr int E = NV * 8;
    const int t = threadIdx.x % row_threads;
    const int walker = blockIdx.x * (blockDim.x / row_threads) + threadIdx.x / row_threads;
    if (walker >= walkers)      // only where a row is a wave or a part of one: no barrier is missed
        return;
    const size_t begin = (size_t)walker * a.rows / walkers, end = (size_t)(walker + 1) * a.rows / walkers;
    const int stride = row_threads;
    const float inv_d = 1.0f / (float)a.D;
    RowSum sum = {slots, 0, (row_threads + 63) / 64, min(row_threads, 64)};
    bool in[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
        in[e] = owns<WIDE>(t, stride, e / 8, e % 8, a.D);

    const bool branch = a.branch != nullptr, gated = branch && a.gate.data != nullptr;
    const bool each = gated && a.gate_rows == 1;        // a gate for every element comes with the row
    Raw rr[NV], yr[NV], gr[NV];
    auto load = [&](size_t row) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (each)
                gr[v] = load_raw<WIDE>(a.gate.data, a.gate.type, row * (size_t)a.D, t, stride, v, a.D);
            rr[v] = load_raw<WIDE>(a.residual, R, row * a.ld_residual, t, stride, v, a.D);
            if (branch)
                yr[v] = load_raw<WIDE>(a.branch, T, row * a.ld_branch, t, stride, v, a.D);
        }
    };
    if (begin < end)
        load(begin);
    Columns<WIDE, NV, BIAS> p;
    size_t gate_row = begin / a.gate_rows;
    p.load(a, gate_row, gated && !each, t, stride);

    for (size_t row = begin; row < end; ++row) {
        float s[E], mean, inv;
        float post_mean = 0.0f, post_inv = 1.0f, pre_mean = 0.0f, pre_inv = 1.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
            unpack(rr[v], R, s + v * 8);
        if (branch) {
            float y[E];
#pragma unroll
            for (int v = 0; v < NV; ++v)
                unpack(yr[v], T, y + v * 8);
            if (each)
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    unpack(gr[v], a.gate.type, p.gate + v * 8);
            else if (gated && row / a.gate_rows != gate_row) {
                gate_row = row / a.gate_rows;
                p.load_gate(a, gate_row, t, stride);
            }
            if (row + 1 < end)
                load(row + 1);
            if (a.post != kNoNorm) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    y[e] = in[e] ? y[e] : 0.0f;
                standardize<E>(y, in, a.post, inv_d, a.eps, sum, mean, inv);
                post_mean = mean;
                post_inv = inv;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    y[e] = BIAS ? fmaf(y[e], p.post_w[e], p.post_b[e]) : y[e] * p.post_w[e];
            }
#pragma unroll
            for (int e = 0; e < E; ++e)
                s[e] = fmaf(s[e], p.scale[e], y[e] * p.gate[e]);
#pragma unroll
            for (int v = 0; v < NV; ++v)
                store8<WIDE>(a.sum, R, row * a.ld_sum, t, stride, v, a.D, s + v * 8);
        } else if (row + 1 < end)
            load(row + 1);
        if (a.out) {
            // (what is not its own must not count)
#pragma unroll
            for (int e = 0; e < E; ++e)
                s[e] = in[e] ? s[e] : 0.0f;
            if (a.pre != kNoNorm) {
                standardize<E>(s, in, a.pre, inv_d, a.eps, sum, mean, inv);
                pre_mean = mean;
                pre_inv = inv;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    s[e] = BIAS ? fmaf(s[e], p.pre_w[e], p.pre_b[e]) : s[e] * p.pre_w[e];
            }
#pragma unroll
            for (int v = 0; v < NV; ++v)
                store8<WIDE>(a.out, T, row * a.ld_out, t, stride, v, a.D, s + v * 8);
        }
        if (a.stats && t == 0)
            *reinterpret_cast<float4*>(a.stats + row * 4) = make_float4(post_mean, post_inv, pre_mean, pre_inv);
    }
}

// ---- backward -----------------------------------------------------------------------------------------
// 4096 rows of 4096 bf16, all six parameters: 49 us (201 MB and 33.5 MB of walkers' sums, 4.8 TB/s) and 6.4 to add those up; 1505 rows of
// 1536 fp32: 18.5 (55 MB without the sums, 3.0 TB/s) and 4.8.  Above 4096 features registers do not suffice: 8192 spills some 200 of them, wider
// rows three to four times as many.

template <ElementType T, ElementType R, bool WIDE, int NV, int THREADS, bool BIAS>
__global__ void __launch_bounds__(THREADS)
block_norm_backward_kernel(BlockNormArgs a, BlockNormGrads d, int row_threads, int walkers, int per_gate, int gates_each)
{
    __shared__ __attribute__((aligned(16))) float slots[2][2][kMaxThreads / 64];
    RowSum::clear(slots);
    constexpr int E = NV * 8;
    const int t = threadIdx.x % row_threads;
    const int walker = blockIdx.x * (blockDim.x / row_threads) + threadIdx.x / row_threads;
    if (walker >= walkers)
        return;
    // a walker's rows: part `walker % per_gate` of a gate's rows, or those of `gates_each` whole gates
    const size_t gates = (a.rows + a.gate_rows - 1) / a.gate_rows;
    size_t begin, end;
    if (per_gate > 1) {
        const size_t g = walker / per_gate, part = walker % per_gate;
        begin = g * a.gate_rows + part * a.gate_rows / per_gate;
        end = g * a.gate_rows + (part + 1) * a.gate_rows / per_gate;
    } else {
        begin = (size_t)walker * gates_each * a.gate_rows;
        end = min(begin + (size_t)gates_each * a.gate_rows, gates * a.gate_rows);
    }
    const int stride = row_threads;
    const float inv_d = 1.0f / (float)a.D;
    RowSum sum = {slots, 0, (row_threads + 63) / 64, min(row_threads, 64)};
    const bool branch = a.branch != nullptr, gated = branch && a.gate.data != nullptr;
    bool in[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
        in[e] = owns<WIDE>(t, stride, e / 8, e % 8, a.D);

    const bool each = gated && a.gate_rows == 1;        // a gate for every element comes with the row
    Columns<WIDE, NV, BIAS> p;
    size_t gate_row = begin / a.gate_rows;
    p.load(a, gate_row, gated && !each, t, stride);
    float sum_post_w[E], sum_scale[E], sum_pre_w[E], sum_gate[E], sum_post_b[BIAS ? E : 8], sum_pre_b[BIAS ? E : 8];
#pragma unroll
    for (int e = 0; e < E; ++e)
    {
        sum_post_w[e] = sum_scale[e] = sum_pre_w[e] = sum_gate[e] = 0.0f;
        if (BIAS)
            sum_post_b[e] = sum_pre_b[e] = 0.0f;
    }

    auto after = [&](float y, int e) { return BIAS ? fmaf(y, p.post_w[e], p.post_b[e]) : y * p.post_w[e]; };

    // the next row is on its way while one is worked on
    Raw rr[NV], yr[NV], gs[NV], go[NV], gr[NV];
    float4 stats = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto load = [&](size_t row) {
        stats = *reinterpret_cast<const float4*>(a.stats + row * 4);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (each)
                gr[v] = load_raw<WIDE>(a.gate.data, a.gate.type, row * (size_t)a.D, t, stride, v, a.D);
            rr[v] = load_raw<WIDE>(a.residual, R, row * a.ld_residual, t, stride, v, a.D);
            if (branch)
                yr[v] = load_raw<WIDE>(a.branch, T, row * a.ld_branch, t, stride, v, a.D);
            if (d.sum)
                gs[v] = load_raw<WIDE>(d.sum, R, row * d.ld_sum, t, stride, v, a.D);
            if (d.out)
                go[v] = load_raw<WIDE>(d.out, T, row * d.ld_out, t, stride, v, a.D);
        }
    };
    if (begin < end)
        load(begin);
    for (size_t row = begin; row < end; ++row) {
        const float4 st = stats;
        if (gated && row / a.gate_rows != gate_row) {
            if (d.gate && per_gate == 1)
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    store8<WIDE>(d.gate, a.gate.type, gate_row * (size_t)a.D, t, stride, v, a.D, sum_gate + v * 8);
#pragma unroll
            for (int e = 0; e < E; ++e)
                sum_gate[e] = 0.0f;
            gate_row = row / a.gate_rows;
            if (!each)
                p.load_gate(a, gate_row, t, stride);
        }
        if (each)
#pragma unroll
            for (int v = 0; v < NV; ++v)
                unpack(gr[v], a.gate.type, p.gate + v * 8);
        float r[E], yn[E], s[E], ds[E], g[E];
#pragma unroll
        for (int v = 0; v < NV; ++v)
            unpack(rr[v], R, r + v * 8);
        if (branch) {
#pragma unroll
            for (int v = 0; v < NV; ++v)
                unpack(yr[v], T, yn + v * 8);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                yn[e] = (yn[e] - st.x) * st.y;      // mean 0 and 1 / deviation 1 where there is no norm
                s[e] = fmaf(r[e], p.scale[e], after(yn[e], e) * p.gate[e]);
            }
        } else
#pragma unroll
            for (int e = 0; e < E; ++e)
                s[e] = r[e];
        if (d.sum)
#pragma unroll
            for (int v = 0; v < NV; ++v)
                unpack(gs[v], R, ds + v * 8);
        else
#pragma unroll
            for (int e = 0; e < E; ++e)
                ds[e] = 0.0f;
        if (d.out)
#pragma unroll
            for (int v = 0; v < NV; ++v)
                unpack(go[v], T, g + v * 8);
        if (row + 1 < end)
            load(row + 1);
        if (d.out) {
            float with = 0.0f, plain = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                g[e] = in[e] ? g[e] : 0.0f;
                s[e] = (s[e] - st.z) * st.w;
                sum_pre_w[e] = fmaf(g[e], s[e], sum_pre_w[e]);
                if (BIAS)
                    sum_pre_b[e] += g[e];
                g[e] *= p.pre_w[e];
                with = fmaf(g[e], s[e], with);
                plain += g[e];
            }
            if (a.pre != kNoNorm) {
                sum(with, plain);
                with *= inv_d;
                plain = a.pre == kLayerNorm ? plain * inv_d : 0.0f;
            } else
                with = plain = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e)
                ds[e] = fmaf(st.w, g[e] - fmaf(s[e], with, plain), ds[e]);
        }
        if (!branch) {
            if (d.residual)
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    store8<WIDE>(d.residual, R, row * d.ld_residual, t, stride, v, a.D, ds + v * 8);
            continue;
        }
        float with = 0.0f, plain = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if (!in[e])
                ds[e] = 0.0f;
            sum_scale[e] = fmaf(ds[e], r[e], sum_scale[e]);
            sum_gate[e] = fmaf(ds[e], after(yn[e], e), sum_gate[e]);
            r[e] = ds[e] * p.scale[e];
            ds[e] *= p.gate[e];
            sum_post_w[e] = fmaf(ds[e], yn[e], sum_post_w[e]);
            if (BIAS)
                sum_post_b[e] += ds[e];
            ds[e] *= p.post_w[e];
            with = fmaf(ds[e], yn[e], with);
            plain += ds[e];
        }
        if (d.residual)
#pragma unroll
            for (int v = 0; v < NV; ++v)
                store8<WIDE>(d.residual, R, row * d.ld_residual, t, stride, v, a.D, r + v * 8);
        if (a.post != kNoNorm) {
            sum(with, plain);
            with *= inv_d;
            plain = a.post == kLayerNorm ? plain * inv_d : 0.0f;
        } else
            with = plain = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            ds[e] = st.y * (ds[e] - fmaf(yn[e], with, plain));
        if (d.branch)
#pragma unroll
            for (int v = 0; v < NV; ++v)
                store8<WIDE>(d.branch, T, row * d.ld_branch, t, stride, v, a.D, ds + v * 8);
    }

    if (gated && d.gate && per_gate == 1 && begin < end)
#pragma unroll
        for (int v = 0; v < NV; ++v)
            store8<WIDE>(d.gate, a.gate.type, gate_row * (size_t)a.D, t, stride, v, a.D, sum_gate + v * 8);
    // the walker's sums: [parameter][walker][column]
    auto leave = [&](int slot, const float* x) {
        if (slot >= 0)
#pragma unroll
            for (int v = 0; v < NV; ++v)
                store8<WIDE>(d.partial, kF32, ((size_t)slot * walkers + walker) * a.D, t, stride, v, a.D, x + v * 8);
    };
    leave(d.slot_post_weight, sum_post_w);
    if (BIAS)
        leave(d.slot_post_bias, sum_post_b);
    leave(d.slot_scale, sum_scale);
    leave(d.slot_pre_weight, sum_pre_w);
    if (BIAS)
        leave(d.slot_pre_bias, sum_pre_b);
    leave(d.slot_gate, sum_gate);
}

// Adds the walkers' sums up in order: 64 columns per workgroup, its 16 waves take the walkers in turn.
struct FinishArgs {
    const float* partial;
    void* out[6];
    int type[6], slot[6];
    int gate;           // the gate's place among the outputs, the last; -1 if it is not here
    int per_gate;
    int walkers, D;
};
__global__ void __launch_bounds__(1024)
block_norm_finish_kernel(FinishArgs f)
{
    __shared__ float part[16][64];
    const int x = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int col = blockIdx.x * 64 + x;
    int o = blockIdx.y, g = 0, first = 0, count = f.walkers;
    if (f.gate >= 0 && o >= f.gate) {
        g = o - f.gate;
        o = f.gate;
        first = g * f.per_gate;
        count = f.per_gate;
    }
    float sum = 0.0f;
    if (col < f.D) {
        const float* const p = f.partial + ((size_t)f.slot[o] * f.walkers + first) * f.D + col;
#pragma unroll 4
        for (int i = w; i < count; i += 16)
            sum += p[(size_t)i * f.D];
    }
    part[w][x] = sum;
    __syncthreads();
    if (w == 0 && col < f.D) {
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            sum += part[i][x];
        const size_t at = (size_t)g * f.D + col;
        if (f.type[o] == kF32)
            static_cast<float*>(f.out[o])[at] = sum;
        else
            static_cast<uint16_t*>(f.out[o])[at] = (uint16_t)to_bits16(sum, f.type[o]);
    }
}

// Threads of a row, 8 elements each up to 8192 features, 16 beyond: whole waves, or 16 or 32 lanes of one.
int row_threads_of(int D)
{
    if (D <= 256)
        return D <= 128 ? 16 : 32;
    const int each = D <= 8 * kMaxThreads ? 8 : 16;
    return (((D + each - 1) / each) + 63) / 64 * 64;
}

template <ElementType T, ElementType R>
void forward(const BlockNormArgs& a, hipStream_t stream)
{
    const int rt = row_threads_of(a.D), each = rt <= 64 ? 256 / rt : 1;
    // as many walkers as the GPU holds waves of this many registers (16 a compute unit)
    const size_t most = (size_t)machine().cus * 16 * 64 / rt;
    const size_t turns = (a.rows + most - 1) / most;       // rows of a walker, the same for nearly all
    const int walkers = (int)((a.rows + turns - 1) / turns);
    const dim3 grid((walkers + each - 1) / each), block(rt * each);
    const bool bias = a.post_bias.data || a.pre_bias.data;
#define NMSPMM_FORWARD(WIDE, NV, THREADS, BIAS) block_norm_kernel<T, R, WIDE, NV, THREADS, BIAS><<<grid, block, 0, stream>>>(a, rt, walkers)
    if (a.D < 8)
        NMSPMM_FORWARD(false, 1, 256, true);
    else if (bias && a.D <= 4096)
        NMSPMM_FORWARD(true, 1, 512, true);
    else if (a.D <= 8 * kMaxThreads)
        bias ? NMSPMM_FORWARD(true, 1, 1024, true) : NMSPMM_FORWARD(true, 1, 1024, false);
    else
        NMSPMM_FORWARD(true, 2, 1024, true);
#undef NMSPMM_FORWARD
}

template <ElementType T, ElementType R>
void backward(const BlockNormArgs& a, const BlockNormGrads& d, const BlockNormWalk& w, hipStream_t stream)
{
    const int rt = row_threads_of(a.D), each = rt <= 64 ? 256 / rt : 1;
    const dim3 grid((w.walkers + each - 1) / each), block(rt * each);
    const bool bias = a.post_bias.data || a.pre_bias.data;
#define NMSPMM_BACKWARD(WIDE, NV, THREADS, BIAS)                                                                         \
    block_norm_backward_kernel<T, R, WIDE, NV, THREADS, BIAS><<<grid, block, 0, stream>>>(a, d, rt, w.walkers, w.per_gate, \
                                                                                          w.gates_each)
    if (a.D < 8)
        NMSPMM_BACKWARD(false, 1, 256, true);
    else if (a.D <= 4096)
        bias ? NMSPMM_BACKWARD(true, 1, 512, true) : NMSPMM_BACKWARD(true, 1, 512, false);
    else if (a.D <= 8 * kMaxThreads)
        bias ? NMSPMM_BACKWARD(true, 1, 1024, true) : NMSPMM_BACKWARD(true, 1, 1024, false);
    else
        NMSPMM_BACKWARD(true, 2, 1024, true);
#undef NMSPMM_BACKWARD
}

} // namespace

hipError_t launch_block_norm(const BlockNormArgs& a, int type, int residual_type, hipStream_t stream)
{
#define NMSPMM_TYPES(T, R) forward<T, R>(a, stream)
    if (type == kF32)
        NMSPMM_TYPES(kF32, kF32);
    else if (type == kBF16)
        residual_type == kF32 ? NMSPMM_TYPES(kBF16, kF32) : NMSPMM_TYPES(kBF16, kBF16);
    else
        residual_type == kF32 ? NMSPMM_TYPES(kF16, kF32) : NMSPMM_TYPES(kF16, kF16);
#undef NMSPMM_TYPES
    return hipGetLastError();
}

// How the backward pass cuts the rows: about two workgroups per compute unit, at least four rows each, and no
// walker with a part of a gate's rows beside rows of another gate.
BlockNormWalk block_norm_walk(long long rows, long long gate_rows, int D)
{
    const int threads = row_threads_of(D);
    const long long most = (long long)machine().cus * 16 * 64 / (threads < 512 ? threads : 512);
    long long rows_each = (rows + most - 1) / most;
    if (rows_each < 4)
        rows_each = 4;
    const long long gates = (rows + gate_rows - 1) / gate_rows;
    BlockNormWalk w = {0, 1, 1};
    if (gate_rows > rows_each) {
        w.per_gate = (int)((gate_rows + rows_each - 1) / rows_each);
        w.walkers = (int)(gates * w.per_gate);
    } else {
        w.gates_each = (int)(rows_each / gate_rows);
        w.walkers = (int)((gates + w.gates_each - 1) / w.gates_each);
    }
    return w;
}

hipError_t launch_block_norm_backward(const BlockNormArgs& a, const BlockNormGrads& given, int type, int residual_type,
                                      hipStream_t stream)
{
    BlockNormGrads d = given;
    const BlockNormWalk w = block_norm_walk(a.rows, a.gate_rows, a.D);
    FinishArgs f = {};
    f.partial = d.partial;
    f.gate = -1;
    f.walkers = w.walkers;
    f.D = a.D;
    int slots = 0;
    auto column = [&](void* out, int out_type, int& slot) {
        slot = -1;
        if (!out)
            return;
        slot = slots;
        f.out[slots] = out;
        f.type[slots] = out_type;
        f.slot[slots] = slots;
        ++slots;
    };
    column(d.post_weight, a.post_weight.type, d.slot_post_weight);
    column(d.post_bias, a.post_bias.type, d.slot_post_bias);
    column(d.scale, a.scale.type, d.slot_scale);
    column(d.pre_weight, a.pre_weight.type, d.slot_pre_weight);
    column(d.pre_bias, a.pre_bias.type, d.slot_pre_bias);
    d.slot_gate = -1;
    int outputs = slots;
    if (d.gate && w.per_gate > 1) {
        f.gate = slots;
        f.per_gate = w.per_gate;
        column(d.gate, a.gate.type, d.slot_gate);
        outputs += (int)((a.rows + a.gate_rows - 1) / a.gate_rows);
    }
    if (a.rows > 0) {
#define NMSPMM_TYPES(T, R) backward<T, R>(a, d, w, stream)
        if (type == kF32)
            NMSPMM_TYPES(kF32, kF32);
        else if (type == kBF16)
            residual_type == kF32 ? NMSPMM_TYPES(kBF16, kF32) : NMSPMM_TYPES(kBF16, kBF16);
        else
            residual_type == kF32 ? NMSPMM_TYPES(kF16, kF32) : NMSPMM_TYPES(kF16, kF16);
#undef NMSPMM_TYPES
    }
    if (outputs > 0)
        block_norm_finish_kernel<<<dim3((a.D + 63) / 64, outputs), 1024, 0, stream>>>(f);
    return hipGetLastError();
}

} // namespace nmspmm
