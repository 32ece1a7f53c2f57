// The work buffer of attn_blocks_e4m3_d128: what the first of its kernels leaves the others, and partial results.
//   u64 before[n + 2]        weight of the decoded requests before each (its 16-token tiles and one more), their total, the most stretches of a kv head
//   u32 order[2048][2]       the units of a kv head, request and number in it, those with the most keys first (only if there are no more than that)
//   u32 units_before[n + 1]  units (256 rows) of the prefilled requests before each, their total
//   u32 rest[places + 1]     tiles of 64 keys before each of the units that are cut, their total
//   u32 done[2 * places]     finished pieces of each unit that is cut, of either half of it
//   u32 queue, by_head       the prefill's next item; whether a head's units stand together
//   parts                    of the decode until they are merged, then of the prefill
#pragma once

#include "blocks.cuh"

namespace sgb {

constexpr uint32_t UNIT_ROWS = 256, UNIT_KEYS = 64;
// Weights are 2^(s - m), f16 in the second product.  m is found anew where a score exceeds it by GROWTH_T, and stands LIFT below the row's
// largest then, so that the largest weight is between 2^7 and 2^15.  f16's normal range thus reaches from 2^-21 of the largest on: V's powers of two are in
// the weights, and a tile of small values beside one of large ones keeps its digits (with m at the maximum, values whose scale was 2^-18 of the largest,
// in dims where the large tile holds nothing, were off by a tenth or more in a tenth of the results).
constexpr float LIFT = 7.0f, GROWTH_T = 15.0f;
constexpr uint32_t MOST_SORTED = 2048, MOST_PLACES = 256;

struct BlocksWork {
    uint64_t* before;
    uint32_t *units_before;
    uint2* order;
    uint32_t *rest, *done, *queue, *by_head;
    uint32_t places;
    uint8_t* parts;
};

// A unit of a prefilled request: its query tokens, and the keys that any of them sees.
struct Unit {
    uint32_t request, first_tok, toks;
    int first_pos, band_lo, tile0, n_tiles;  // position of the first query, first key, tiles of 64 keys
};
__device__ __forceinline__ Unit unit_at(const BlocksAttn& a, uint32_t request, uint32_t nth)
{
    const Request rq = request_at(a.req, request);
    const uint32_t per = UNIT_ROWS / a.group;
    uint32_t tok0 = nth * per;
    if (tok0 >= rq.n) tok0 = 0;  // only if starts that go back and forth, which are reported, made more units than a word counts
    Unit u;
    u.request = request;
    u.first_tok = rq.first + tok0;
    u.toks = min(per, rq.n - tok0);
    u.first_pos = (int)rq.len - (int)rq.n + (int)tok0;
    const int last_pos = u.first_pos + (int)u.toks - 1, window = a.req.window && a.req.window < MOST_KEYS ? (int)a.req.window : (int)MOST_KEYS;
    u.band_lo = max(u.first_pos + 1 - window, 0);
    u.tile0 = u.band_lo / (int)UNIT_KEYS;
    u.n_tiles = last_pos >= 0 ? last_pos / (int)UNIT_KEYS - u.tile0 + 1 : 0;
    return u;
}
// Item i of all units of all heads, `total` units a head: its head and its place in the order of units.
__device__ __forceinline__ void split_item(uint32_t i, uint32_t total, uint32_t n_kv, bool by_head, uint32_t& head, uint32_t& rank)
{
    head = by_head ? i / total : i % n_kv;
    rank = by_head ? i % total : i / n_kv;
}
// The first `whole` items go to the places one by one.  Those left over, fewer than there are places, are laid end to end and cut
// into equal stretches, one per place, of eight tiles at least unless that were fewer stretches than units: a unit has its start and its end to
// pay for (24 requests with three prompts: 87.6 us with fewer stretches than units, 80.3 so).
__device__ __forceinline__ uint32_t whole_items(uint32_t items, uint32_t places) { return items / places * places; }
__device__ __forceinline__ uint32_t rest_stretches(uint32_t tiles, uint32_t units, uint32_t places) { return min(max((tiles + 7) / 8, units), places); }

inline uint32_t blocks_places(int sm_count) { return (uint32_t)sm_count < MOST_PLACES ? (uint32_t)sm_count : MOST_PLACES; }
inline size_t blocks_work_header(uint32_t requests, uint32_t places)
{
    return ((size_t)(requests + 2) * 8 + ((size_t)requests + 1 + 2 * MOST_SORTED + 3 * places + 3) * 4 + 255) / 256 * 256;
}
inline BlocksWork blocks_work_at(uint8_t* p, uint32_t requests, uint32_t places)
{
    BlocksWork w;
    w.before = reinterpret_cast<uint64_t*>(p);
    w.order = reinterpret_cast<uint2*>(w.before + requests + 2);
    w.units_before = reinterpret_cast<uint32_t*>(w.order + MOST_SORTED);
    w.rest = w.units_before + requests + 1;
    w.done = w.rest + places + 1;
    w.queue = w.done + 2 * places;
    w.by_head = w.queue + 1;
    w.places = places;
    w.parts = p + blocks_work_header(requests, places);
    return w;
}

// attn_blocks_decode.cu
size_t blocks_decode_work(int sm_count, uint32_t n_kv, uint32_t group, uint32_t max_q);
int launch_blocks_decode(const LaunchArgs&, const BlocksAttn&, const BlocksWork&);
// attn_blocks_prefill.cu
size_t blocks_prefill_work(int sm_count);
int launch_blocks_prefill(const LaunchArgs&, const BlocksAttn&, const BlocksWork&);

}  // namespace sgb
