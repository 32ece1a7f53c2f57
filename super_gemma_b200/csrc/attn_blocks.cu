// Attention of a batch of requests over the 8-bit cache of blocks.cuh, head_dim 128.
//
// Request r brings n_r = starts[r + 1] - starts[r] query tokens, which are the last n_r of its lens[r] keys: query i stands at
// position lens[r] - n_r + i and sees the keys up to its own position, of those the last `window` if there is one.  A row that
// sees nothing (a request that was refused: its length is 0) is zero.  Output f16.
#include <cmath>

#include "blocks.cuh"
#include "sgb_kernels.h"

namespace sgb {

namespace {

// One CTA of four warps per (query token, query head); a warp takes every fourth tile, a lane four dims.
__global__ void __launch_bounds__(128) attn_blocks_simple_kernel(const BlocksAttn a)
{
    __shared__ float part[4][130];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x, qh = blockIdx.y, head = qh / a.group;
    uint32_t lo = 0, hi = a.req.n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (ld_global(a.req.starts + mid) <= t) lo = mid; else hi = mid;
    }
    const Request rq = request_at(a.req, lo);
    if (t - rq.first >= rq.n || rq.n * a.group <= FEW_ROWS) return;
    const int64_t pos = (int64_t)rq.len - rq.n + (t - rq.first);
    const int64_t from = a.req.window && pos + 1 > (int64_t)a.req.window ? pos + 1 - a.req.window : 0;
    const uint2 qw = ld_global(reinterpret_cast<const uint2*>(a.q + ((size_t)t * a.n_kv * a.group + qh) * 128 + 4 * lane));
    const float2 q0 = __half22float2(as_half2(qw.x)), q1 = __half22float2(as_half2(qw.y));
    const float scale2 = a.scale * 1.4426950408889634f;
    float m = NEG_SENTINEL, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t tile = from / TILE_TOK + warp; tile * TILE_TOK <= pos; tile += 4) {
        const size_t at = (size_t)block_at(a.req, lo, (uint32_t)tile) * a.n_kv + head;
        const float ks = __int_as_float((127 + *(volatile const int8_t*)(a.exps[0] + at)) << 23) * scale2;
        const float vs = __int_as_float((127 + *(volatile const int8_t*)(a.exps[1] + at)) << 23);
        for (int i = 0; i < TILE_TOK; i++) {
            const int64_t key = tile * TILE_TOK + i;
            if (key < from || key > pos) continue;
            const uint32_t kw = ld_global(reinterpret_cast<const uint32_t*>(a.pool[0] + at * TILE_BYTES + i * 128 + 4 * lane));
            const uint32_t vw = ld_global(reinterpret_cast<const uint32_t*>(a.pool[1] + at * TILE_BYTES + i * 128 + 4 * lane));
            const float2 k0 = __half22float2(as_half2(e4m3x2_to_f16x2(kw & 0xffffu))), k1 = __half22float2(as_half2(e4m3x2_to_f16x2(kw >> 16)));
            const float2 v0 = __half22float2(as_half2(e4m3x2_to_f16x2(vw & 0xffffu))), v1 = __half22float2(as_half2(e4m3x2_to_f16x2(vw >> 16)));
            float s = fmaf(q0.x, k0.x, fmaf(q0.y, k0.y, fmaf(q1.x, k1.x, q1.y * k1.y)));
#pragma unroll
            for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
            s *= ks;
            const float mn = fmaxf(m, s), c = ex2(m - mn), p = ex2(s - mn);
            m = mn;
            l = fmaf(l, c, p);
            const float pv = p * vs;
            o[0] = fmaf(o[0], c, pv * v0.x);
            o[1] = fmaf(o[1], c, pv * v0.y);
            o[2] = fmaf(o[2], c, pv * v1.x);
            o[3] = fmaf(o[3], c, pv * v1.y);
        }
    }
    for (int i = 0; i < 4; i++) part[warp][4 * lane + i] = o[i];
    if (lane == 0) part[warp][128] = m, part[warp][129] = l;
    __syncthreads();
    float big = NEG_SENTINEL, acc = 0.0f, den = 0.0f;
    for (int w = 0; w < 4; w++) big = fmaxf(big, part[w][128]);
    for (int w = 0; w < 4; w++) {
        const float f = part[w][129] > 0.0f ? ex2(part[w][128] - big) : 0.0f;
        acc = fmaf(f, part[w][threadIdx.x], acc);
        den = fmaf(f, part[w][129], den);
    }
    a.out[((size_t)t * a.n_kv * a.group + qh) * 128 + threadIdx.x] = __float2half_rn(den > 0.0f ? acc / den : 0.0f);
}

struct PushAttnBlocks {
    float scale;
    uint32_t page, stride, window, group, max_q;
};

}  // namespace

size_t attn_blocks_work_bytes(int sm_count, uint32_t n_kv, uint32_t group, uint32_t requests, uint32_t tokens, uint32_t max_q)
{
    return blocks_decode_work(sm_count, n_kv, group, requests, max_q);
}

// attn_blocks_e4m3_d128: q, k pool, k exps, v pool, v exps, table, lens, starts, out f16, work.
// push {scale, page, table stride, window, query heads per kv head, most query tokens of a request}.  grid [KV, requests, tokens].
int launch_attn_blocks(const LaunchArgs& a)
{
    const PushAttnBlocks p = *(const PushAttnBlocks*)a.push;
    const uint32_t n_kv = a.groups[0], n = a.groups[1], tokens = a.groups[2];
    if (n_kv == 0 || n == 0 || tokens == 0) return fail_validation(a, "attn_blocks: groups must be [kv heads, requests, query tokens]");
    if (n_kv > 1024) return fail_validation(a, "attn_blocks: at most 1024 kv heads");
    if (n > MOST_REQUESTS) return fail_validation(a, "attn_blocks: at most 65536 requests");
    if (p.group != 1 && p.group != 2 && p.group != 4 && p.group != 8) return fail_validation(a, "attn_blocks: query heads per kv head must be 1, 2, 4 or 8");
    if (p.page < (uint32_t)TILE_TOK || (p.page & (p.page - 1))) return fail_validation(a, "attn_blocks: page must be a power of two, at least 16 tokens");
    if (p.stride == 0 || p.max_q == 0) return fail_validation(a, "attn_blocks: the table's stride and the most query tokens must be > 0");
    if (!(p.scale > 0.0f) || !std::isfinite(p.scale)) return fail_validation(a, "attn_blocks: the softmax scale must be positive");
    const size_t tile_row = (size_t)n_kv * TILE_BYTES, rows = (size_t)tokens * n_kv * p.group;
    const size_t blocks = a.b[1].bytes / tile_row;
    if (blocks == 0 || a.b[3].bytes / tile_row != blocks)
        return fail_validation(a, "attn_blocks: K and V pools must hold the same (non-zero) number of 16-token blocks");
    if (blocks > NO_SLOT / TILE_TOK) return fail_validation(a, "attn_blocks: a pool holds less than 2^32 rows");
    if (blocks * n_kv >= 0x80000000ull) return fail_validation(a, "attn_blocks: a pool holds less than 2^31 tiles");
    if (blocks * TILE_TOK < p.page) return fail_validation(a, "attn_blocks: the pools hold no whole page");
    if (int r = need_bytes(a, 0, rows * 256, "q")) return r;
    if (int r = need_bytes(a, 2, blocks * n_kv, "k exponents")) return r;
    if (int r = need_bytes(a, 4, blocks * n_kv, "v exponents")) return r;
    if (int r = need_bytes(a, 5, 4 * (size_t)n * p.stride, "table")) return r;
    if (int r = need_bytes(a, 6, 4 * (size_t)n, "lens")) return r;
    if (int r = need_bytes(a, 7, 4 * ((size_t)n + 1), "starts")) return r;
    if (int r = need_bytes(a, 8, rows * 256, "out")) return r;
    if (int r = need_bytes(a, 9, attn_blocks_work_bytes(a.sm_count, n_kv, p.group, n, tokens, p.max_q), "work")) return r;
    if (int r = need_aligned(a, {16, 16, 1, 16, 1, 4, 4, 4, 16, 16})) return r;
    const uint32_t shift = (uint32_t)__builtin_ctz(p.page);
    const BlocksAttn k{{(const uint32_t*)a.b[5].ptr, (const uint32_t*)a.b[6].ptr, (const uint32_t*)a.b[7].ptr, n, p.stride, shift,
                        (uint32_t)(blocks >> (shift - 4)), tokens, p.max_q, p.window, a.status},
                       (const __half*)a.b[0].ptr, {(const uint8_t*)a.b[1].ptr, (const uint8_t*)a.b[3].ptr}, {(const int8_t*)a.b[2].ptr, (const int8_t*)a.b[4].ptr},
                       (__half*)a.b[8].ptr, (uint8_t*)a.b[9].ptr, n_kv, p.group, (uint32_t)(blocks * n_kv), p.scale};
    if (int r = launch_blocks_decode(a, k)) return r;
    if ((uint64_t)p.max_q * p.group <= FEW_ROWS) return 0;
    const cudaError_t e = launch_dependent(attn_blocks_simple_kernel, dim3(tokens, n_kv * p.group), dim3(128), 0, a.stream, k);
    ++*a.launches;
    return check_cuda(a, e, "attn_blocks_e4m3_d128");
}

}  // namespace sgb
