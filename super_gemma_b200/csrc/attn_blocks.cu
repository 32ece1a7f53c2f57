// Attention of a batch of requests over the 8-bit cache of blocks.cuh, head_dim 128.
//
// Request r brings n_r = starts[r + 1] - starts[r] query tokens, which are the last n_r of its lens[r] keys: query i stands at
// position lens[r] - n_r + i and sees the keys up to its own position, of those the last `window` if there is one.  A row that
// sees nothing (a request that was refused: its length is 0) is zero.  Output f16.
//
// Requests of few rows (query tokens x heads of a group) are decoded (attn_blocks_decode.cu), the others prefilled
// (attn_blocks_prefill.cu); a dispatch that names no request of more than 16 rows launches the decode alone.
#include <algorithm>

#include "blocks.cuh"
#include "blocks_work.cuh"
#include "sgb_kernels.h"

namespace sgb {

namespace {

struct PushAttnBlocks {
    float scale;
    uint32_t page, stride, window, group, max_q;
};

// Rows up to which a request is decoded: 8 or 16, as the most that the dispatch names need, and 8 beside prompts, for the single tokens' sake.
// (16 drafts of 2 to 4 tokens, four heads a group, up to 32768 keys: 99 us, as prompts 160; of two heads, 4 to 8 tokens 185 and 256.)
uint32_t rows_decoded(uint32_t group, uint32_t max_q)
{
    const uint64_t rows = (uint64_t)group * max_q;
    return rows <= 8 || rows > FEW_ROWS ? 8 : 16;
}

// A query with a key reaches 2^39 (128 products of f16 numbers), so below 2^-80 all scores lie within 2^-39 of each other and the weights are equal in f32
// whatever the scale: it is taken as that.  Times a tile's power of two a smaller one could become 0, and 0 times the -inf of a masked score is a NaN.
constexpr float LEAST_SCALE = 0x1p-80f, MOST_SCALE = 0x1p100f;

// What the grid and the push may say of heads and requests; the launcher names what it refuses.
constexpr uint32_t MOST_KV = 1024;
bool group_is_served(uint32_t group) { return group == 1 || group == 2 || group == 4 || group == 8; }

}  // namespace

size_t attn_blocks_work_bytes(int sm_count, uint32_t n_kv, uint32_t group, uint32_t requests, uint32_t tokens, uint32_t max_q)
{
    if (n_kv == 0 || n_kv > MOST_KV || !group_is_served(group) || requests == 0 || requests > MOST_REQUESTS || tokens == 0 || max_q == 0) return 0;
    const size_t few = blocks_decode_work(sm_count, n_kv, group, max_q);
    const size_t many = (uint64_t)max_q * group > FEW_ROWS ? blocks_prefill_work(sm_count) : 0;
    return blocks_work_header(requests, blocks_places(sm_count)) + (few > many ? few : many);
}

// attn_blocks_e4m3_d128: q, k pool, k exps, v pool, v exps, table, lens, starts, out f16, work.
// push {scale, page, table stride, window, query heads per kv head, most query tokens of a request}.  grid [KV, requests, tokens].
int launch_attn_blocks(const LaunchArgs& a)
{
    const PushAttnBlocks p = *(const PushAttnBlocks*)a.push;
    const uint32_t n_kv = a.groups[0], n = a.groups[1], tokens = a.groups[2];
    if (n_kv == 0 || n == 0 || tokens == 0) return fail_validation(a, "attn_blocks: groups must be [kv heads, requests, query tokens]");
    if (n_kv > MOST_KV) return fail_validation(a, "attn_blocks: at most 1024 kv heads");
    if (n > MOST_REQUESTS) return fail_validation(a, "attn_blocks: at most 65536 requests");
    if (!group_is_served(p.group)) return fail_validation(a, "attn_blocks: query heads per kv head must be 1, 2, 4 or 8");
    if (p.page < (uint32_t)TILE_TOK || (p.page & (p.page - 1))) return fail_validation(a, "attn_blocks: page must be a power of two, at least 16 tokens");
    if (p.stride == 0 || p.max_q == 0) return fail_validation(a, "attn_blocks: the table's stride and the most query tokens must be > 0");
    if (!(p.scale > 0.0f && p.scale <= MOST_SCALE)) return fail_validation(a, "attn_blocks: the softmax scale must be positive, and at most 2^100");
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
                       (__half*)a.b[8].ptr, n_kv, p.group, (uint32_t)__builtin_ctz(p.group), (uint32_t)(blocks * n_kv), rows_decoded(p.group, p.max_q) / p.group, std::max(p.scale, LEAST_SCALE)};
    const BlocksWork work = blocks_work_at((uint8_t*)a.b[9].ptr, n, blocks_places(a.sm_count));
    if (int r = launch_blocks_decode(a, k, work)) return r;
    return (uint64_t)p.max_q * p.group > FEW_ROWS ? launch_blocks_prefill(a, k, work) : 0;
}

}  // namespace sgb
