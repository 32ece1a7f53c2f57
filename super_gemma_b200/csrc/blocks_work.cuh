// The work buffer of attn_blocks_e4m3_d128: what the first of its kernels leaves the others, and partial results.
//   u64 before[n + 2]        16-token tiles of the decoded requests before each, their total, the number of stretches
//   u32 units_before[n + 1]  units (256 rows) of the prefilled requests before each, their total
//   u32 queue, done[2 * places]  the prefill's next item; finished pieces of each unit that is cut, of either half of it
//   parts                    of the decode until they are merged, then of the prefill
#pragma once

#include "blocks.cuh"

namespace sgb {

constexpr uint32_t UNIT_ROWS = 256;

struct BlocksWork {
    uint64_t* before;
    uint32_t *units_before, *queue, *done;
    uint32_t places;
    uint8_t* parts;
};
struct PrefillWork {
    const uint32_t* units_before;
    uint32_t *queue, *done;
    float4* acc;  // [slot][row][128]
    float2* ml;   // [slot][row]
    uint32_t slots;
};
inline size_t blocks_work_header(uint32_t requests, uint32_t places) { return ((size_t)(requests + 2) * 8 + (size_t)(requests + 2 + 2 * places) * 4 + 255) / 256 * 256; }
inline BlocksWork blocks_work_at(uint8_t* p, uint32_t requests, uint32_t places)
{
    BlocksWork w;
    w.before = reinterpret_cast<uint64_t*>(p);
    w.units_before = reinterpret_cast<uint32_t*>(w.before + requests + 2);
    w.queue = w.units_before + requests + 1;
    w.done = w.queue + 1;
    w.places = places;
    w.parts = p + blocks_work_header(requests, places);
    return w;
}

// attn_blocks_decode.cu
size_t blocks_decode_work(int sm_count, uint32_t n_kv, uint32_t group, uint32_t max_q);
int launch_blocks_decode(const LaunchArgs&, const BlocksAttn&, const BlocksWork&);
// attn_blocks_prefill.cu
size_t blocks_prefill_work(int sm_count, uint32_t n_kv, uint32_t group, uint32_t requests, uint32_t tokens);
int launch_blocks_prefill(const LaunchArgs&, const BlocksAttn&, const BlocksWork&);

}  // namespace sgb
