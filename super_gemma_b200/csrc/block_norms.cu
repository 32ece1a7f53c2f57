// What stands between two blocks of a layer, row by row of the residual stream h (f16, bf16 or f32) and of the block's output y (f16):
//   n  = y / rms(y) * w_post   (post 1)   or y   (post 0)            rms(v) = sqrt(mean v^2 + eps)
//   h' = (h + g n) s                                                 g: nothing, one value a channel, a row, or one in all
//   x  = f16(h' / rms(h') * w_pre)                                   the next block's input
// and with post 2 the first norm of all, x = f16(h / rms(h) * w_pre) alone.  Both sums of squares, h' and everything between are f32; x is made of
// h' as it is before its own rounding.
//
// One pass over the bytes: a row stays in the registers of its lanes between the two sums.  A row has 2^k lanes of a warp if one unit (16 bytes of h) a lane
// covers it, else whole warps with N units a lane.
#include <cuda_bf16.h>

#include <cmath>
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
constexpr uint32_t MOST_EACH = 8;   // units of a lane
enum : uint32_t { POST_NONE = 0, POST_NORM = 1, FIRST_NORM = 2 };
enum : uint32_t { GATE_NONE = 0, GATE_CHANNEL = 1, GATE_ROW = 2, GATE_ONE = 3 };
constexpr uint32_t MOST_WARPS = 16;  // of a row

// Consecutive values of a unit: 16 bytes of R.
template <typename R>
constexpr int UNIT = 16 / sizeof(R);

// A unit of f16 as it is loaded, and as pairs of f32.
template <int U>
struct RawHalf {
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

// The sum over a row's lanes: a butterfly in the warp, then over the row's warps in their order.  Everybody calls it.
__device__ __forceinline__ float row_sum(float v, uint32_t lanes, float* parts)
{
    if (lanes >= 32) {
#pragma unroll
        for (uint32_t d = 1; d < 32; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    } else {
        for (uint32_t d = 1; d < lanes; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    }
    if (lanes <= 32) return v;
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = v;  // (one row a CTA; those of warps that it has not are 0)
    __syncthreads();
    v = 0.0f;
    for (uint32_t i = 0; i < lanes / 32; i += 4) {
        const float4 f = reinterpret_cast<const float4*>(parts)[i / 4];
        v += (f.x + f.y) + (f.z + f.w);
    }
    return v;
}

template <typename R, int N>
__global__ void __launch_bounds__(32 * MOST_WARPS) block_norms_kernel(const __grid_constant__ NormsArgs a)
{
    constexpr int U = UNIT<R>, P = U / 2;
    __shared__ alignas(16) float parts[2][MOST_WARPS];
    if (a.lanes > 32 && threadIdx.x < 2 * MOST_WARPS) parts[threadIdx.x / MOST_WARPS][threadIdx.x % MOST_WARPS] = 0.0f;
    pdl_wait();
    pdl_launch_dependents();
    if (a.lanes > 32) __syncthreads();  // the zeros come before the sums
    const uint32_t shift = a.lanes <= 32 ? __ffs(a.lanes) - 1 : 31;  // a row of several warps has the CTA to itself
    const uint32_t lane = a.lanes <= 32 ? threadIdx.x & (a.lanes - 1) : threadIdx.x;
    const uint64_t row = a.lanes <= 32 ? (uint64_t)blockIdx.x * (blockDim.x >> shift) + (threadIdx.x >> shift) : blockIdx.x;
    const size_t at = row * a.hidden + lane * U;  // of the first unit
    const uint32_t step = a.lanes * U;
    const bool live = row < a.rows;
    const float inv_n = 1.0f / (float)a.hidden;
    // all units but the last are within the row
    const auto on = [&](int i) { return live && (i + 1 < N || lane * U + i * step < a.hidden); };
    RawHalf<U> y[N];
    uint4 raw[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        y[i] = RawHalf<U>{};
        raw[i] = make_uint4(0, 0, 0, 0);
        if (on(i)) {
            if (a.post != FIRST_NORM) y[i] = load_f16<U>(a.y + at + i * step);
            raw[i] = ld_global(reinterpret_cast<const uint4*>(static_cast<const R*>(a.h) + at + i * step));
        }
    }
    float by = 1.0f;  // of the block's output
    if (a.gates == GATE_ROW && live) by = ld_global(a.gate + row);
    if (a.gates == GATE_ONE) by = ld_global(a.gate);
    if (a.post == POST_NORM) {
        float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int j = 0; j < P; j++) {
                const float2 f = pair_of(y[i].w[j]);
                ss = fma2_rn(f, f, ss);
            }
        by *= rsqrtf(row_sum(ss.x + ss.y, a.lanes, parts[0]) * inv_n + a.eps);
    }
    const float2 by2 = make_float2(by, by), scale2 = make_float2(a.scale, a.scale), plus2 = make_float2(a.plus, a.plus);
    float2 ss = make_float2(0.0f, 0.0f), v[N][P];
#pragma unroll
    for (int i = 0; i < N; i++) {
        unpack<R>(raw[i], v[i]);
        if (a.post != FIRST_NORM && on(i)) {
            float2 n[P], w[P];
#pragma unroll
            for (int j = 0; j < P; j++) n[j] = pair_of(y[i].w[j]);
            if (a.post == POST_NORM) {
                load_f32<U>(a.w_post + lane * U + i * step, w);
#pragma unroll
                for (int j = 0; j < P; j++) n[j] = mul2_rn(n[j], add2_rn(w[j], plus2));
            }
            if (a.gates == GATE_CHANNEL) {
                load_f32<U>(a.gate + lane * U + i * step, w);
#pragma unroll
                for (int j = 0; j < P; j++) n[j] = mul2_rn(n[j], w[j]);
            }
#pragma unroll
            for (int j = 0; j < P; j++) v[i][j] = mul2_rn(fma2_rn(n[j], by2, v[i][j]), scale2);
            *reinterpret_cast<uint4*>(static_cast<R*>(a.h_out) + at + i * step) = pack<R>(v[i]);
        }
#pragma unroll
        for (int j = 0; j < P; j++) ss = fma2_rn(v[i][j], v[i][j], ss);
    }
    const float inv = rsqrtf(row_sum(ss.x + ss.y, a.lanes, parts[1]) * inv_n + a.eps);
    const float2 inv2 = make_float2(inv, inv);
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (!on(i)) continue;
        float2 w[P];
        load_f32<U>(a.w_pre + lane * U + i * step, w);
#pragma unroll
        for (int j = 0; j < P; j++) v[i][j] = mul2_rn(mul2_rn(v[i][j], inv2), add2_rn(w[j], plus2));
        store_f16<U>(a.x + at + i * step, v[i]);
    }
}

struct PushNorms {
    uint32_t post, gates, plus_one;
    float scale, eps;
};

template <typename R>
auto norms_kernel(uint32_t n)
{
    return n == 1 ? block_norms_kernel<R, 1> : n == 2 ? block_norms_kernel<R, 2> : n == 3 ? block_norms_kernel<R, 3> : n == 4 ? block_norms_kernel<R, 4>
         : n == 5 ? block_norms_kernel<R, 5> : n == 6 ? block_norms_kernel<R, 6> : n == 7 ? block_norms_kernel<R, 7> : block_norms_kernel<R, 8>;
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
    const uint32_t units = hidden / U;
    NormsArgs k{(const __half*)a.b[0].ptr, a.b[1].ptr, (const float*)a.b[2].ptr, (const float*)a.b[3].ptr, (const float*)a.b[4].ptr, a.b[5].ptr, (__half*)a.b[6].ptr,
                rows, hidden, 1, p.post, p.gates, p.plus_one ? 1.0f : 0.0f, p.scale, p.eps};
    // units a lane: eight at most
    uint32_t each = 1;
    if (units <= 32) {
        while (k.lanes < units) k.lanes <<= 1;
    } else {
        uint32_t warps = (units + 32 * MOST_EACH - 1) / (32 * MOST_EACH);
        each = (units + 32 * warps - 1) / (32 * warps);
        warps = (units + 32 * each - 1) / (32 * each);
        k.lanes = 32 * warps;
    }
    const uint32_t threads = k.lanes <= 32 ? 128 : k.lanes, per_cta = threads / k.lanes;
    const cudaError_t e = launch_dependent(norms_kernel<R>(each), dim3((unsigned)((rows + per_cta - 1ull) / per_cta)), dim3(threads), 0, a.stream, k);
    ++*a.launches;
    return check_cuda(a, e, "block_norms");
}
template int launch_block_norms<__half>(const LaunchArgs&);
template int launch_block_norms<__nv_bfloat16>(const LaunchArgs&);
template int launch_block_norms<float>(const LaunchArgs&);

}  // namespace sgb
