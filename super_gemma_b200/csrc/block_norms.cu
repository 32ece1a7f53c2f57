// What stands between two blocks of a layer, row by row of the residual stream h (f16, bf16 or f32) and of the block's output y (f16):
//   n  = y / rms(y) * w_post   (post 1)   or y   (post 0)            rms(v) = sqrt(mean v^2 + eps)
//   h' = (h + g n) s                                                 g: nothing, one value a channel, a row, or one in all
//   x  = f16(h' / rms(h') * w_pre)                                   the next block's input
// and with post 2 the first norm of all, x = f16(h / rms(h) * w_pre) alone.  Both sums of squares, h' and everything between are f32; x is made of
// h' as it is before its own rounding.
//
// One pass over the bytes: a row stays in the registers of its lanes between the two sums, a unit being 16 bytes of h.  A row has eight or sixteen lanes of a warp
// (1, 2 or 4 if it has fewer units than eight) or whole warps, each lane up to eight units.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "sgb_common.cuh"
#include "sgb_kernels.h"

namespace sgb {

namespace {

struct NormsArgs {
    const __half* y;
    const void* h;
    const float *w_post, *gate, *w_pre;
    void* h_out;
    __half* x;
    uint32_t rows, hidden, lanes;  // lanes of a row: 2^k in a warp, or whole warps
    uint32_t post, gates;
    float plus, scale, eps;  // plus: 1 where weights are 1 + w
};
enum : uint32_t { POST_NONE = 0, POST_NORM = 1, FIRST_NORM = 2 };
enum : uint32_t { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_ROW = 2, GATE_ONE = 3 };
constexpr uint32_t MOST_WARPS = 16;  // of a row

// Rows of a CTA that come ahead and the one in use, and the shared memory for them.
constexpr uint32_t STAGES = 2;
constexpr size_t MOST_STAGED = 200 * 1024;
constexpr uint32_t MOST_STREAMED = 4;  // units of a lane of such a row
// Consecutive values of a unit: 16 bytes of R.
template <typename R>
constexpr int UNIT = 16 / sizeof(R);

// A unit of f16 as it is loaded, and as pairs of f32.
template <int U>
struct alignas(2 * U) RawHalf {
    uint32_t w[U / 2];
};
template <int U>
__device__ __forceinline__ RawHalf<U> load_f16(const __half* p)
{
    RawHalf<U> r;
    if constexpr (U == 8) {
        const uint4 u = ld_global(reinterpret_cast<const uint4*>(p));
        r.w[0] = u.x, r.w[1] = u.y, r.w[2] = u.z, r.w[3] = u.w;
    } else {
        const uint2 u = ld_global(reinterpret_cast<const uint2*>(p));
        r.w[0] = u.x, r.w[1] = u.y;
    }
    return r;
}
__device__ __forceinline__ float2 pair_of(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
template <int U>
__device__ __forceinline__ void store_f16(__half* p, const float2 (&v)[U / 2])
{
    uint32_t w[U / 2];
#pragma unroll
    for (int i = 0; i < U / 2; i++) w[i] = pack_half2(v[i].x, v[i].y);
    if constexpr (U == 8)
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}
template <typename R>
__device__ __forceinline__ void unpack(const uint4& u, float2 (&v)[UNIT<R> / 2])
{
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if constexpr (sizeof(R) == 4) {
        v[0] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
        v[1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (std::is_same_v<R, __half>)
                v[i] = pair_of(w[i]);
            else
                v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        }
    }
}
template <typename R>
__device__ __forceinline__ uint4 pack(const float2 (&v)[UNIT<R> / 2])
{
    uint32_t w[4];
    if constexpr (sizeof(R) == 4) {
        w[0] = __float_as_uint(v[0].x), w[1] = __float_as_uint(v[0].y), w[2] = __float_as_uint(v[1].x), w[3] = __float_as_uint(v[1].y);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (std::is_same_v<R, __half>) {
                w[i] = pack_half2(v[i].x, v[i].y);
            } else {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[i].x, v[i].y);
                w[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int U>
__device__ __forceinline__ void load_f32(const float* p, float2 (&v)[U / 2])
{
#pragma unroll
    for (int i = 0; i < U / 4; i++) {
        const float4 f = ld_global(reinterpret_cast<const float4*>(p) + i);
        v[2 * i] = make_float2(f.x, f.y);
        v[2 * i + 1] = make_float2(f.z, f.w);
    }
}

// The sum over a row's lanes: a butterfly in the warp, then over the row's warps in their order.  Everybody calls it.  A row of several warps has the CTA to itself, and
// `parts` is 0 for the warps up to the next multiple of four.
__device__ __forceinline__ float row_sum(float v, uint32_t lanes, float* parts)
{
    if (lanes >= 32) {
#pragma unroll
        for (uint32_t d = 1; d < 32; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    } else {
        for (uint32_t d = 1; d < lanes; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    }
    if (lanes <= 32) return v;
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (uint32_t i = 0; i < lanes / 32; i += 4) {
        const float4 f = reinterpret_cast<const float4*>(parts)[i / 4];
        v += (f.x + f.y) + (f.z + f.w);
    }
    return v;
}

// Where a thread stands: its row's place in the CTA, its first column.
struct Place {
    uint32_t in_cta, per_cta, col, step;  // `step` columns from unit to unit
};
template <int U>
__device__ __forceinline__ Place place_of(uint32_t lanes)
{
    if (lanes > 32) return Place{0, 1, threadIdx.x * U, lanes * U};
    const uint32_t shift = __ffs(lanes) - 1;
    return Place{threadIdx.x >> shift, blockDim.x >> shift, (threadIdx.x & (lanes - 1)) * U, lanes * U};
}

// h' = (h + y by w) s, in v (which holds h), and its sum of squares.
template <typename R, int N>
__device__ __forceinline__ void add_block(const NormsArgs& a, const RawHalf<UNIT<R>> (&y)[N], const float2 (&w)[N][UNIT<R> / 2], float by, float2 (&v)[N][UNIT<R> / 2])
{
    const float2 by2 = make_float2(by, by), scale2 = make_float2(a.scale, a.scale);
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < UNIT<R> / 2; j++) v[i][j] = mul2_rn(fma2_rn(mul2_rn(pair_of(y[i].w[j]), w[i][j]), by2, v[i][j]), scale2);
}
template <int N, int P>
__device__ __forceinline__ float squares(const float2 (&v)[N][P])
{
    float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < P; j++) ss = fma2_rn(v[i][j], v[i][j], ss);
    return ss.x + ss.y;
}
template <int N, int U>
__device__ __forceinline__ float squares(const RawHalf<U> (&y)[N])
{
    float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < U / 2; j++) {
            const float2 f = pair_of(y[i].w[j]);
            ss = fma2_rn(f, f, ss);
        }
    return ss.x + ss.y;
}
template <int U>
__device__ __forceinline__ void times_f32(const float* p, float2 (&w)[U / 2])
{
    float2 f[U / 2];
    load_f32<U>(p, f);
#pragma unroll
    for (int j = 0; j < U / 2; j++) w[j] = mul2_rn(w[j], f[j]);
}
template <typename R>
__device__ __forceinline__ void write_next(__half* x, const float2 (&v)[UNIT<R> / 2], const float2 (&w)[UNIT<R> / 2], float inv)
{
    float2 out[UNIT<R> / 2];
#pragma unroll
    for (int j = 0; j < UNIT<R> / 2; j++) out[j] = mul2_rn(mul2_rn(v[j], make_float2(inv, inv)), w[j]);
    store_f16<UNIT<R>>(x, out);
}

// One row a CTA (or a warp, or some of its lanes): nothing waits for anything that could have been asked for before it.  The block's weights come beside the row, the
// next ones beside the second sum.
// Three units of 16-bit values: two CTAs of twelve warps an SM, 80 registers instead of 98 (400 rows of 5376 4.6 us, else 5.7).
template <typename R, int N>
constexpr bool TIGHT = sizeof(R) == 2 && N == 3;
constexpr uint32_t TIGHT_LANES = 384;  // (norms_shape keeps to it)
template <typename R, int N>
__global__ void __launch_bounds__(TIGHT<R, N> ? TIGHT_LANES : 512, TIGHT<R, N> ? 2 : 0) block_norms_kernel(const __grid_constant__ NormsArgs a)
{
    constexpr int U = UNIT<R>, P = U / 2;
    __shared__ alignas(16) float parts[2][MOST_WARPS];
    pdl_wait();
    pdl_launch_dependents();
    const Place me = place_of<U>(a.lanes);
    const uint64_t row = (uint64_t)blockIdx.x * me.per_cta + me.in_cta;
    const size_t at = row * a.hidden + me.col;  // of the first unit
    const bool live = row < a.rows;
    const auto on = [&](int i) { return live && (i + 1 < N || me.col + i * me.step < a.hidden); };  // all units but the last are within the row
    RawHalf<U> y[N];
    uint4 raw[N];
    float2 w[N][P];
#pragma unroll
    for (int i = 0; i < N; i++) {
        y[i] = RawHalf<U>{};
        raw[i] = make_uint4(0, 0, 0, 0);
        if (on(i)) {
            if (a.post != FIRST_NORM) y[i] = load_f16<U>(a.y + at + i * me.step);
            raw[i] = ld_global(reinterpret_cast<const uint4*>(static_cast<const R*>(a.h) + at + i * me.step));
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
#pragma unroll
        for (int j = 0; j < P; j++) w[i][j] = make_float2(1.0f, 1.0f);
        if (a.post == POST_NORM && on(i)) load_f32<U>(a.w_post + me.col + i * me.step, w[i]);
    }
    float by = 1.0f;  // of the block's output
    if (a.gates == GATE_ROW && live) by = ld_global(a.gate + row);
    if (a.gates == GATE_ONE) by = ld_global(a.gate);
    if (a.lanes > 32) {
        if (threadIdx.x < MOST_WARPS) parts[0][threadIdx.x] = parts[1][threadIdx.x] = 0.0f;
        __syncthreads();  // the zeros come before the sums
    }
    const float inv_n = 1.0f / (float)a.hidden;
    const float2 plus2 = make_float2(a.plus, a.plus);
    if (a.post == POST_NORM) {
        by *= rsqrtf(row_sum(squares(y), a.lanes, parts[0]) * inv_n + a.eps);
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int j = 0; j < P; j++) w[i][j] = add2_rn(w[i][j], plus2);
    }
    float2 v[N][P];
#pragma unroll
    for (int i = 0; i < N; i++) unpack<R>(raw[i], v[i]);
    if (a.post != FIRST_NORM) {
        if (a.gates == GATE_CHANNEL) {
#pragma unroll
            for (int i = 0; i < N; i++)
                if (on(i)) times_f32<U>(a.gate + me.col + i * me.step, w[i]);
        }
        add_block<R, N>(a, y, w, by, v);
#pragma unroll
        for (int i = 0; i < N; i++)
            if (on(i)) *reinterpret_cast<uint4*>(static_cast<R*>(a.h_out) + at + i * me.step) = pack<R>(v[i]);
    }
#pragma unroll
    for (int i = 0; i < N; i++)
        if (on(i)) load_f32<U>(a.w_pre + me.col + i * me.step, w[i]);
    const float inv = rsqrtf(row_sum(squares(v), a.lanes, parts[1]) * inv_n + a.eps);
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (!on(i)) continue;
#pragma unroll
        for (int j = 0; j < P; j++) w[i][j] = add2_rn(w[i][j], plus2);
        write_next<R>(a.x + at + i * me.step, v[i], w[i], inv);
    }
}

// Many rows of f32, or of 16 bits that a warp holds: weights are asked for unit by unit where they are used, which leaves registers for more rows on an SM at a time.
// (Three units of f32 in 40 registers: 3 CTAs of fourteen warps an SM instead of 2, 8192 rows of 5376 99 -> 90 us; eight in 64 instead of 70: 2 CTAs, 2000 rows of 16384 113 -> 85.)
template <typename R, int N>
__global__ void __launch_bounds__(512, sizeof(R) == 4 ? (N <= 3 ? 3 : 2) : 0) block_norms_late_kernel(const __grid_constant__ NormsArgs a)
{
    constexpr int U = UNIT<R>, P = U / 2;
    __shared__ alignas(16) float parts[2][MOST_WARPS];
    pdl_wait();
    pdl_launch_dependents();
    const Place me = place_of<U>(a.lanes);
    const uint64_t row = (uint64_t)blockIdx.x * me.per_cta + me.in_cta;
    const size_t at = row * a.hidden + me.col;  // of the first unit
    const bool live = row < a.rows;
    const auto on = [&](int i) { return live && (i + 1 < N || me.col + i * me.step < a.hidden); };  // all units but the last are within the row
    RawHalf<U> y[N];
    uint4 raw[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        y[i] = RawHalf<U>{};
        raw[i] = make_uint4(0, 0, 0, 0);
        if (on(i)) {
            if (a.post != FIRST_NORM) y[i] = load_f16<U>(a.y + at + i * me.step);
            raw[i] = ld_global(reinterpret_cast<const uint4*>(static_cast<const R*>(a.h) + at + i * me.step));
        }
    }
    if (a.lanes > 32) {
        if (threadIdx.x < MOST_WARPS) parts[0][threadIdx.x] = parts[1][threadIdx.x] = 0.0f;
        __syncthreads();  // the zeros come before the sums
    }
    float by = 1.0f;  // of the block's output
    if (a.gates == GATE_ROW && live) by = ld_global(a.gate + row);
    if (a.gates == GATE_ONE) by = ld_global(a.gate);
    const float inv_n = 1.0f / (float)a.hidden;
    if (a.post == POST_NORM) by *= rsqrtf(row_sum(squares(y), a.lanes, parts[0]) * inv_n + a.eps);
    const float2 by2 = make_float2(by, by), scale2 = make_float2(a.scale, a.scale), plus2 = make_float2(a.plus, a.plus);
    float2 v[N][P];
#pragma unroll
    for (int i = 0; i < N; i++) {
        unpack<R>(raw[i], v[i]);
        if (a.post == FIRST_NORM || !on(i)) continue;
        float2 n[P], w[P];
#pragma unroll
        for (int j = 0; j < P; j++) n[j] = pair_of(y[i].w[j]);
        if (a.post == POST_NORM) {
            load_f32<U>(a.w_post + me.col + i * me.step, w);
#pragma unroll
            for (int j = 0; j < P; j++) n[j] = mul2_rn(n[j], add2_rn(w[j], plus2));
        }
        if (a.gates == GATE_CHANNEL) times_f32<U>(a.gate + me.col + i * me.step, n);
#pragma unroll
        for (int j = 0; j < P; j++) v[i][j] = mul2_rn(fma2_rn(n[j], by2, v[i][j]), scale2);
        *reinterpret_cast<uint4*>(static_cast<R*>(a.h_out) + at + i * me.step) = pack<R>(v[i]);
    }
    const float inv = rsqrtf(row_sum(squares(v), a.lanes, parts[1]) * inv_n + a.eps);
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (!on(i)) continue;
        float2 w[P];
        load_f32<U>(a.w_pre + me.col + i * me.step, w);
#pragma unroll
        for (int j = 0; j < P; j++) w[j] = add2_rn(w[j], plus2);
        write_next<R>(a.x + at + i * me.step, v[i], w, inv);
    }
}

// Many rows of 16 bits: CTAs that stay, with the weights of their columns in registers.  Rows come ahead of their turn into shared memory, STAGES - 1 of them on their way; a thread
// reads what it has copied itself, so that only its own copies are waited for, and a stage is written again one row after it was read.
template <typename R, int N>
__global__ void __launch_bounds__(512) block_norms_stream_kernel(const __grid_constant__ NormsArgs a)
{
    constexpr int U = UNIT<R>, P = U / 2;
    __shared__ alignas(16) float parts[3][MOST_WARPS];
    extern __shared__ uint4 stages[];
    pdl_wait();
    pdl_launch_dependents();
    const Place me = place_of<U>(a.lanes);
    const uint32_t stride = gridDim.x * me.per_cta;
    const uint64_t first = (uint64_t)blockIdx.x * me.per_cta;
    const auto on = [&](uint64_t row, int i) { return row < a.rows && (i + 1 < N || me.col + i * me.step < a.hidden); };
    const auto h_place = [&](uint32_t stage, int i) { return stages + (stage * N + i) * blockDim.x + threadIdx.x; };
    const auto y_place = [&](uint32_t stage, int i) {
        return reinterpret_cast<RawHalf<U>*>(stages + STAGES * N * blockDim.x) + (stage * N + i) * blockDim.x + threadIdx.x;
    };
    const auto ask = [&](uint64_t row, uint32_t stage) {
        const size_t at = row * a.hidden + me.col;
#pragma unroll
        for (int i = 0; i < N; i++) {
            copy_async_if(on(row, i) && a.post != FIRST_NORM, y_place(stage, i), a.y + at + i * me.step);
            copy_async_if(on(row, i), h_place(stage, i), static_cast<const R*>(a.h) + at + i * me.step);
        }
        copy_async_commit();
    };
#pragma unroll
    for (uint32_t j = 0; j + 1 < STAGES; j++) ask(first + me.in_cta + j * (uint64_t)stride, j);
    float2 w[N][P], next[N][P];  // what a column of the block and of the next input is multiplied by
    const float2 plus2 = make_float2(a.plus, a.plus);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t col = me.col + i * me.step;
#pragma unroll
        for (int j = 0; j < P; j++) w[i][j] = next[i][j] = make_float2(1.0f, 1.0f);
        if (col >= a.hidden) continue;
        if (a.post == POST_NORM) {
            load_f32<U>(a.w_post + col, w[i]);
#pragma unroll
            for (int j = 0; j < P; j++) w[i][j] = add2_rn(w[i][j], plus2);
        }
        if (a.gates == GATE_CHANNEL) times_f32<U>(a.gate + col, w[i]);
        load_f32<U>(a.w_pre + col, next[i]);
#pragma unroll
        for (int j = 0; j < P; j++) next[i][j] = add2_rn(next[i][j], plus2);
    }
    float one = 1.0f;
    if (a.gates == GATE_ONE) one = ld_global(a.gate);
    if (a.lanes > 32) {
        if (threadIdx.x < MOST_WARPS) parts[0][threadIdx.x] = parts[1][threadIdx.x] = parts[2][threadIdx.x] = 0.0f;
        __syncthreads();  // the zeros come before the sums
    }
    const float inv_n = 1.0f / (float)a.hidden;
    const auto gate_of = [&](uint64_t row) { return a.gates == GATE_ROW && row < a.rows ? ld_global(a.gate + row) : one; };
    float gate = gate_of(first + me.in_cta);
    uint32_t stage = 0, turn = 0;
    for (uint64_t row0 = first; row0 < a.rows; row0 += stride) {
        const uint64_t row = row0 + me.in_cta;
        const size_t at = row * a.hidden + me.col;
        float by = gate;
        gate = gate_of(row + stride);
        RawHalf<U> y[N];
        float2 v[N][P];
        copy_async_wait<STAGES - 2>();
#pragma unroll
        for (int i = 0; i < N; i++) {
            y[i] = RawHalf<U>{};
            uint4 raw = make_uint4(0, 0, 0, 0);
            if (on(row, i)) {
                if (a.post != FIRST_NORM) y[i] = *y_place(stage, i);
                raw = *h_place(stage, i);
            }
            unpack<R>(raw, v[i]);
        }
        ask(row + (STAGES - 1) * (uint64_t)stride, stage == 0 ? STAGES - 1 : stage - 1);
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        if (a.post == POST_NORM) by *= rsqrtf(row_sum(squares(y), a.lanes, parts[2]) * inv_n + a.eps);
        if (a.post != FIRST_NORM) {
            add_block<R, N>(a, y, w, by, v);
#pragma unroll
            for (int i = 0; i < N; i++)
                if (on(row, i)) *reinterpret_cast<uint4*>(static_cast<R*>(a.h_out) + at + i * me.step) = pack<R>(v[i]);
        }
        // a row's sums are read while the next one's are written where nothing is waited for in between (post 0 and 2): two places in turn
        const float inv = rsqrtf(row_sum(squares(v), a.lanes, parts[turn]) * inv_n + a.eps);
        turn ^= 1;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (on(row, i)) write_next<R>(a.x + at + i * me.step, v[i], next[i], inv);
    }
    copy_async_wait<0>();
}

struct PushNorms {
    uint32_t post, gates, plus_one;
    float scale, eps;
};

struct NormsShape {
    uint32_t lanes, each;  // of a row; units of a lane
};
// Eight lanes to sixteen warps a row and at most `most` units a lane, so that a row takes the fewest instructions: about 45 a unit, full or not, and 110 for the two sums.
template <typename R>
NormsShape norms_shape(uint32_t units, uint32_t most)
{
    NormsShape s{0, 0};
    uint32_t least = ~0u;
    const auto look = [&](uint32_t lanes) {
        const uint32_t each = (units + lanes - 1) / lanes, cost = lanes * (each * 45 + 110);
        if ((sizeof(R) == 2 && each == 3 && lanes > TIGHT_LANES) || each > most) return;
        if (cost < least) s = {lanes, each}, least = cost;
    };
    for (uint32_t lanes = units < 8 ? 1 : 8; lanes < 32; lanes *= 2) look(lanes);
    for (uint32_t warps = 1; warps <= MOST_WARPS; warps++) look(32 * warps);
    if (s.lanes == 0) s = {32 * MOST_WARPS, (units + 32 * MOST_WARPS - 1) / (32 * MOST_WARPS)};  // the widest rows
    return s;
}

uint32_t cta_threads(uint32_t lanes) { return lanes <= 32 ? 128 : lanes; }
template <typename R>
size_t staged_bytes(const NormsShape& s) { return (size_t)STAGES * s.each * cta_threads(s.lanes) * (16 + 2 * UNIT<R>); }

template <typename R, int N>
int launch_stream(const LaunchArgs& a, const NormsArgs& k, uint32_t threads, size_t smem)
{
    const auto kern = block_norms_stream_kernel<R, N>;
    static std::mutex mutex;
    static int registers[64] = {};  // of a thread, 0: not asked yet
    int regs = 0;
    {
        std::lock_guard<std::mutex> lock(mutex);
        if (a.device < 0 || a.device >= 64 || registers[a.device] == 0) {
            if (int r = check_cuda(a, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MOST_STAGED), "cudaFuncSetAttribute(block_norms)")) return r;
            cudaFuncAttributes at;
            if (int r = check_cuda(a, cudaFuncGetAttributes(&at, kern), "cudaFuncGetAttributes(block_norms)")) return r;
            regs = at.numRegs;
            if (a.device >= 0 && a.device < 64) registers[a.device] = regs;
        } else {
            regs = registers[a.device];
        }
    }
    // as many CTAs as the SMs hold at once: registers come in eights a thread, an SM has 65536 of them, 2048 threads and 228 KB, of which a CTA takes 1 KB more than it asks for
    const uint32_t by_regs = 65536 / ((regs + 7) / 8 * 8 * threads), by_smem = (uint32_t)(228 * 1024 / (smem + 2048)), by_threads = std::min(32u, 2048 / threads);
    const uint32_t resident = std::max(1u, std::min(by_regs, std::min(by_smem, by_threads)));
    const uint32_t per_cta = threads / k.lanes, ctas = (uint32_t)((k.rows + per_cta - 1ull) / per_cta);
    return check_cuda(a, launch_dependent(kern, dim3(std::min(ctas, resident * a.sm_count)), dim3(threads), smem, a.stream, k), "block_norms");
}

enum class Way { EARLY, LATE, STREAM };
template <typename R, int N>
int launch_norms(const LaunchArgs& a, const NormsArgs& k, Way way)
{
    const uint32_t threads = cta_threads(k.lanes), per_cta = threads / k.lanes;
    if constexpr (sizeof(R) == 2 && N <= MOST_STREAMED)
        if (way == Way::STREAM) return launch_stream<R, N>(a, k, threads, staged_bytes<R>({k.lanes, N}));
    auto kern = block_norms_kernel<R, N>;
    if constexpr (sizeof(R) == 4 || N >= 4)  // (rows of 16 bits that a warp holds have four units a lane and more)
        if (way == Way::LATE) kern = block_norms_late_kernel<R, N>;
    return check_cuda(a, launch_dependent(kern, dim3((unsigned)((k.rows + per_cta - 1ull) / per_cta)), dim3(threads), 0, a.stream, k), "block_norms");
}

}  // namespace

// block_norms_<residual>: y, h, w_post, gate, w_pre, h_out, x.  push {post, gate, plus_one, scale, eps}.  grid [hidden, rows].
template <typename R>
int launch_block_norms(const LaunchArgs& a)
{
    const PushNorms p = *(const PushNorms*)a.push;
    const uint32_t hidden = a.groups[0], rows = a.groups[1];
    constexpr uint32_t U = UNIT<R>;
    if (hidden == 0 || hidden % 8 || hidden > 16384) return fail_validation(a, "block_norms: groups[0] (hidden) must be a multiple of 8 up to 16384");
    if (rows == 0) return fail_validation(a, "block_norms: groups[1] (rows) must be > 0");
    if (p.post > FIRST_NORM) return fail_validation(a, "block_norms: post must be 0 (y as it is), 1 (normed) or 2 (no y)");
    if (p.gates > GATE_ONE) return fail_validation(a, "block_norms: gate must be 0 (none), 1 (a channel), 2 (a row) or 3 (one)");
    if (p.plus_one > 1) return fail_validation(a, "block_norms: plus_one must be 0 or 1");
    if (!std::isfinite(p.scale)) return fail_validation(a, "block_norms: scale must be finite");
    if (!(p.eps >= 0.0f) || !std::isfinite(p.eps)) return fail_validation(a, "block_norms: eps must be finite and not negative");
    if (p.post == FIRST_NORM && (p.gates != GATE_NONE || p.scale != 1.0f)) return fail_validation(a, "block_norms: post 2 has no gate and a scale of 1");
    const size_t n = (size_t)rows * hidden;
    const size_t gate = p.gates == GATE_CHANNEL ? hidden : p.gates == GATE_ROW ? rows : p.gates == GATE_ONE ? 1 : 0;
    const bool block = p.post != FIRST_NORM;
    if (block)
        if (int r = need_bytes(a, 0, 2 * n, "y")) return r;
    if (int r = need_bytes(a, 1, sizeof(R) * n, "h")) return r;
    if (p.post == POST_NORM)
        if (int r = need_bytes(a, 2, 4 * (size_t)hidden, "w_post")) return r;
    if (int r = need_bytes(a, 3, 4 * gate, "gate")) return r;
    if (int r = need_bytes(a, 4, 4 * (size_t)hidden, "w_pre")) return r;
    if (block)
        if (int r = need_bytes(a, 5, sizeof(R) * n, "h_out")) return r;
    if (int r = need_bytes(a, 6, 2 * n, "x")) return r;
    const uint32_t y_al = block ? 16 : 1, gate_al = p.gates == GATE_CHANNEL ? 16 : gate ? 4 : 1;
    if (int r = need_aligned(a, {y_al, 16, p.post == POST_NORM ? 16u : 1u, gate_al, 16, y_al, 16})) return r;
    const auto meet = [&](int i, size_t wi, int j, size_t wj) { return rows_meet(a.b[i].ptr, wi * hidden, wi * hidden, a.b[j].ptr, wj * hidden, wj * hidden, rows); };
    constexpr size_t R_BYTES = sizeof(R);
    if (block && a.b[1].ptr != a.b[5].ptr && meet(1, R_BYTES, 5, R_BYTES)) return fail_validation(a, "block_norms: h_out overlaps h and is not h");
    if (block && a.b[0].ptr != a.b[6].ptr && meet(0, 2, 6, 2)) return fail_validation(a, "block_norms: x overlaps y and is not y");
    if (meet(1, R_BYTES, 6, 2) || (block && (meet(0, 2, 5, R_BYTES) || meet(5, R_BYTES, 6, 2)))) return fail_validation(a, "block_norms: x or h_out overlaps another tensor");
    const Other w_post{2, p.post == POST_NORM ? 4 * (size_t)hidden : 0, "w_post"}, gates{3, 4 * gate, "gate"}, w_pre{4, 4 * (size_t)hidden, "w_pre"};
    if (block)
        if (int r = need_apart(a, "block_norms", 5, "h_out", sizeof(R) * n, sizeof(R) * n, 1, {w_post, gates, w_pre})) return r;
    if (int r = need_apart(a, "block_norms", 6, "x", 2 * n, 2 * n, 1, {w_post, gates, w_pre})) return r;
    const uint32_t units = hidden / U;
    NormsArgs k{(const __half*)a.b[0].ptr, a.b[1].ptr, (const float*)a.b[2].ptr, (const float*)a.b[3].ptr, (const float*)a.b[4].ptr, a.b[5].ptr, (__half*)a.b[6].ptr,
                rows, hidden, 1, p.post, p.gates, p.plus_one ? 1.0f : 0.0f, p.scale, p.eps};
    // Where all rows are on the GPU at once each has lanes enough for 2048 columns at a time and asks for its weights beside them; else lanes have as many units as registers
    // allow.  From 80 MB on rows of 16 bits come ahead of their turn, but for those that a warp holds.  Measured one launch after the other, us, early | late | ahead: f32, 8192 rows of 5376
    // 102.6 | 89 to 90 | 96.1, 30011 of 1096 70.7 | 68.0 | 74.5, 800 of 5376 13.7 | 14.0; bf16, 30011 of 1096 51.0 | 44.5 | 48.0; f16, 6000 of 5376 54.8 | 49.0 | 45.5, 100000 of 264 46.4 | 48.5 | 40.6, 3000 of 8192
    // 44.1 | 45.4 | 36.5.
    const bool many = (uint64_t)n * (4 + 2 * R_BYTES) >= 80ull << 20, warp_holds = units > 64 && units <= 192;
    NormsShape shape = norms_shape<R>(units, std::min(4u, (hidden + 2047) / 2048));
    Way way = Way::EARLY;
    if ((uint64_t)rows * shape.lanes > 1024ull * a.sm_count) {
        way = U == 4 || (many && warp_holds) ? Way::LATE : many ? Way::STREAM : Way::EARLY;
        shape = norms_shape<R>(units, U == 4 ? 3 : warp_holds ? 6 : MOST_STREAMED);
    }
    k.lanes = shape.lanes;
    int e = 0;
    switch (shape.each) {
        case 1: e = launch_norms<R, 1>(a, k, way); break;
        case 2: e = launch_norms<R, 2>(a, k, way); break;
        case 3: e = launch_norms<R, 3>(a, k, way); break;
        case 4: e = launch_norms<R, 4>(a, k, way); break;
        case 5: e = launch_norms<R, 5>(a, k, way); break;
        case 6: e = launch_norms<R, 6>(a, k, way); break;
        default:  // f32 rows of more than 12288
            if constexpr (U == 4) e = shape.each == 7 ? launch_norms<R, 7>(a, k, way) : launch_norms<R, 8>(a, k, way);
    }
    ++*a.launches;
    return e;
}
template int launch_block_norms<__half>(const LaunchArgs&);
template int launch_block_norms<__nv_bfloat16>(const LaunchArgs&);
template int launch_block_norms<float>(const LaunchArgs&);

}  // namespace sgb
