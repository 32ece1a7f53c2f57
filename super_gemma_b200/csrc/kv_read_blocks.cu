// The way back out of the 8-bit cache of blocks.cuh: tokens [from_r, from_r + n_r) of every request as packed f16 rows, n_r = starts[r + 1] - starts[r].
// value = e4m3 * 2^e is an f16 number for every tile that an append writes, so that nothing is rounded.
//
// One byte read and two written per value: bound by bytes (119690 tokens of 40 requests, 16 heads, pages of 16: 233 us, 0.96 of the copy rate;
// 1000 of one request 4.0).
#include "blocks.cuh"
#include "sgb_kernels.h"

namespace sgb {

namespace {

constexpr int THREADS = 256;
constexpr uint32_t ROWS = THREADS / 16;  // of a CTA
constexpr uint32_t AHEAD = 4;

struct ReadArgs {
    const uint8_t* pool[2];
    const int8_t* exps[2];
    const uint32_t *table, *from, *starts;
    __half* out[2];
    uint32_t n, tokens, n_kv, stride, page_shift, blocks;
    uint32_t* status;
};

// Pool row of packed row i, or NO_SLOT; half a warp looks for it together.
__device__ __forceinline__ uint32_t cached_row(const ReadArgs& a, uint32_t i)
{
    const uint32_t lane = threadIdx.x & 15, mask = 0xffffu << (threadIdx.x & 16);
    uint32_t lo = 0, left = a.n;  // the last request with starts <= i is one of these
    while (left > 1) {
        const uint32_t step = (left + 15) / 16, probe = (lane + 1) * step;
        const bool reached = probe < left && ld_global(a.starts + lo + min(probe, left - 1)) <= i;
        const uint32_t passed = __popc(__ballot_sync(mask, reached)) * step;  // less than `left`, whatever `starts` holds
        lo += passed;
        left = min(step, left - passed);
    }
    const uint32_t first = ld_global(a.starts + lo), end = ld_global(a.starts + lo + 1);
    if (i < first || i >= end) return NO_SLOT;
    const uint64_t pos = (uint64_t)ld_global(a.from + lo) + (i - first), page = pos >> a.page_shift;
    if (page >= a.stride) {
        report_error(a.status, DEV_ERR_BOUNDS, 641, lo, (uint32_t)pos);
        return NO_SLOT;
    }
    const uint64_t row = ((uint64_t)ld_global(a.table + (size_t)lo * a.stride + page) << a.page_shift) + (pos & ((1u << a.page_shift) - 1));
    if (row / TILE_TOK >= a.blocks) {
        report_error(a.status, DEV_ERR_BOUNDS, 642, lo, (uint32_t)(row >> a.page_shift));
        return NO_SLOT;
    }
    return (uint32_t)row;
}

// Two e4m3 numbers times 2^e as f16.  A tile of an append has e in [-15, 8] and the product is exact; others go through f32.
__device__ __forceinline__ uint32_t scaled(uint32_t two_bytes, int e)
{
    const __half2 q = as_half2(e4m3x2_to_f16x2(two_bytes));
    if (e >= -24 && e <= 15) return as_u32(__hmul2(q, power_of_two(e)));
    const float2 f = __half22float2(q);
    const float by = exp2_of(max(e, -126));  // 448 * 2^-126 is no f16 number either
    return pack_half2(f.x * by, f.y * by);
}

// A CTA has ROWS packed rows, half a warp each: eight bytes in and sixteen out a lane, so that both sides move whole sectors.  Sixteen rows are
// a tile's where a request's rows begin with one.  The heads of both sides go round, AHEAD of them asked for at a time (gridDim.y CTAs share
// them).  With one head at a time, or its place looked for by one thread a row, 40 requests took 289 and 231 us where they now take
// 226 (launches side by side).
__global__ void __launch_bounds__(THREADS) read_blocks_kernel(const __grid_constant__ ReadArgs a)
{
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t lane = threadIdx.x & 15, row = blockIdx.x * ROWS + threadIdx.x / 16;
    if (row >= a.tokens) return;
    const uint32_t at = cached_row(a, row);
    if (at == NO_SLOT) return;
    const size_t tile = (size_t)(at / TILE_TOK) * a.n_kv, in_tile = at % TILE_TOK * 128 + lane * 8, out = (size_t)row * a.n_kv * 128 + lane * 8;
    for (uint32_t u0 = blockIdx.y; u0 < 2 * a.n_kv; u0 += AHEAD * gridDim.y) {
        uint2 q[AHEAD];
        int e[AHEAD];
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; j++) {
            const uint32_t u = u0 + j * gridDim.y, side = u >= a.n_kv, head = side ? u - a.n_kv : u;
            const bool on = u < 2 * a.n_kv;
            q[j] = ld_global_if(on, reinterpret_cast<const uint2*>(a.pool[side] + (tile + head) * TILE_BYTES + in_tile));
            e[j] = ld_global_if(on, a.exps[side] + tile + head);
        }
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; j++) {
            const uint32_t u = u0 + j * gridDim.y, side = u >= a.n_kv, head = side ? u - a.n_kv : u;
            if (u >= 2 * a.n_kv) return;
            *reinterpret_cast<uint4*>(a.out[side] + out + (size_t)head * 128) =
                make_uint4(scaled(q[j].x & 0xffffu, e[j]), scaled(q[j].x >> 16, e[j]), scaled(q[j].y & 0xffffu, e[j]), scaled(q[j].y >> 16, e[j]));
        }
    }
}

struct PushRead {
    uint32_t page, stride;
};

}  // namespace

// kv_read_blocks_e4m3_d128: k pool, k exps, v pool, v exps, table, from, starts, k, v.  push {page, stride}.  grid [KV, requests, rows].
int launch_kv_read_blocks(const LaunchArgs& a)
{
    const PushRead p = *(const PushRead*)a.push;
    const uint32_t n_kv = a.groups[0], n = a.groups[1], tokens = a.groups[2];
    if (n_kv == 0 || n == 0 || tokens == 0) return fail_validation(a, "read_blocks: groups must be [kv heads, requests, rows]");
    if (n_kv > 1024) return fail_validation(a, "read_blocks: at most 1024 kv heads");
    if (n > MOST_REQUESTS) return fail_validation(a, "read_blocks: at most 65536 requests");
    if (tokens > 0x7fffffffu) return fail_validation(a, "read_blocks: less than 2^31 rows");
    if (p.page < (uint32_t)TILE_TOK || (p.page & (p.page - 1))) return fail_validation(a, "read_blocks: page must be a power of two, at least 16 tokens");
    if (p.stride == 0) return fail_validation(a, "read_blocks: the table's stride must be > 0");
    const size_t tile_row = (size_t)n_kv * TILE_BYTES, blocks = a.b[0].bytes / tile_row;
    if (blocks == 0 || a.b[2].bytes / tile_row != blocks)
        return fail_validation(a, "read_blocks: K and V pools must hold the same (non-zero) number of 16-token blocks");
    if (blocks > NO_SLOT / TILE_TOK) return fail_validation(a, "read_blocks: a pool holds less than 2^32 rows");
    if (int r = need_bytes(a, 1, blocks * n_kv, "k exponents")) return r;
    if (int r = need_bytes(a, 3, blocks * n_kv, "v exponents")) return r;
    if (int r = need_bytes(a, 4, 4 * (size_t)n * p.stride, "table")) return r;
    if (int r = need_bytes(a, 5, 4 * (size_t)n, "from")) return r;
    if (int r = need_bytes(a, 6, 4 * (size_t)n + 4, "starts")) return r;
    if (int r = need_bytes(a, 7, 256 * (size_t)tokens * n_kv, "k")) return r;
    if (int r = need_bytes(a, 8, 256 * (size_t)tokens * n_kv, "v")) return r;
    if (int r = need_aligned(a, {16, 1, 16, 1, 4, 4, 4, 16, 16})) return r;
    const size_t out = 256 * (size_t)tokens * n_kv;
    for (int i = 7; i < 9; i++)
        if (int r = need_apart(a, "read_blocks", i, i == 7 ? "k" : "v", out, out, 1,
                               {{0, blocks * tile_row, "k pool"}, {1, blocks * n_kv, "k exponents"}, {2, blocks * tile_row, "v pool"}, {3, blocks * n_kv, "v exponents"},
                                {4, 4 * (size_t)n * p.stride, "table"}, {5, 4 * (size_t)n, "from"}, {6, 4 * (size_t)n + 4, "starts"}, {8, i == 7 ? out : 0, "v"}}))
            return r;
    ReadArgs k{{(const uint8_t*)a.b[0].ptr, (const uint8_t*)a.b[2].ptr}, {(const int8_t*)a.b[1].ptr, (const int8_t*)a.b[3].ptr}, (const uint32_t*)a.b[4].ptr,
               (const uint32_t*)a.b[5].ptr, (const uint32_t*)a.b[6].ptr, {(__half*)a.b[7].ptr, (__half*)a.b[8].ptr}, n, tokens, n_kv, p.stride,
               (uint32_t)__builtin_ctz(p.page), (uint32_t)blocks, a.status};
    const uint32_t ctas = (tokens + ROWS - 1) / ROWS;
    uint32_t shares = 1;  // CTAs that have the same rows: as many as fill the GPU
    while (shares < 2 * n_kv && shares * (uint64_t)ctas < 4ull * a.sm_count) shares *= 2;
    const cudaError_t e = launch_dependent(read_blocks_kernel, dim3(ctas, shares), dim3(THREADS), 0, a.stream, k);
    ++*a.launches;
    return check_cuda(a, e, "kv_read_blocks_e4m3_d128");
}

}  // namespace sgb
