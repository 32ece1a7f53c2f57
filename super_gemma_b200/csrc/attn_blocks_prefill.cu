// Attention of requests with many queries (prompts, chunks of them, long drafts) over the 8-bit cache of blocks.cuh, on tcgen05.
//
// A unit is 256 rows of one request and kv head: 256 / group query tokens x the group's heads, so that a key is fetched and converted
// once for all of them.  They are two tiles of 128 rows, one softmax warpgroup each.  Per 64 keys and tile, as in the f16 flash
// kernel: S = Q K^T into one of two tensor-memory buffers, one thread per row for the online softmax (base 2, the maximum raised when it
// grows by more than 2^8, l from the unrounded weights), P back over S, O += P V.
// What differs is where K and V come from.  One warp copies the cache's bytes, 16 tokens of one head at a time through the block
// table, up to four tiles of keys ahead; four warps turn them into f16 in the swizzled operand tiles (16 bytes in, 32 out, one
// conversion a pair), so the cache is read once per unit at one byte a value and no f16 copy of it exists.  The powers of two go to the
// softmax, as in the decode: K's times the scores, V's into the exponent.
//
// One CTA per SM stays and takes units from a queue (the lengths are known on the device only); one warp fetches the next while the
// others work.  The units that are left when every CTA has had its whole ones are laid end to end and cut into equal stretches; the CTA
// that finishes the last piece of a unit merges them, in their order, so reruns give the same bits.
//
// Bound by shared memory's port, 192 KB = 1536 cycles per 64 keys and 256 rows (raw bytes in and out 32, f16 tiles 32, operands of Q K^T 96, of
// P V 32), of the 2000 or so that a tile takes; in long runs by the board's power.  1740 tokens of 65536 keys, 16 kv heads of two query heads:
// 1855 us, 0.99 PFLOP/s (the f16 kernel reaches 1.05 to 1.1 on cached f16 keys).  128 rows a CTA and two CTAs an SM would convert every key twice
// as often and need 256 KB of the port.
#include <mutex>

#include "blocks.cuh"
#include "blocks_work.cuh"
#include "sgb_kernels.h"

namespace sgb {

namespace {

constexpr int HD = 128;
constexpr int ROWS = 128, KEYS = 64;              // of a tile of queries, of keys
constexpr int THREADS = 512;                      // two softmax warpgroups, one that converts, one of single warps
constexpr int CONVERT_WARP = 8, MMA_WARP = 12, COPY_WARP = 13, QUEUE_WARP = 14, QUERY_WARP = 15;
constexpr int RAW = 4;                            // tiles of keys under way from the cache
constexpr int ITEMS = 2;                          // the item at work and the next: what a CTA takes early no other can take
constexpr int TILES_A_WAIT = 100000;              // fewer tiles of keys than go through in the time that a wait is bounded to (2000 cycles each)
constexpr int ITEM_READERS = 8 + 4 + 3;           // warps that give an item's place back
constexpr uint32_t HALF_TILE = 64 * 128;          // [64 rows][64 dims] f16
constexpr uint32_t Q_BYTES = 4 * HALF_TILE;       // of one tile of queries
constexpr uint32_t TMEM_COLS = 512, TMEM_O = 256; // S: [tile][buffer] of 64 columns, then O: [tile] of 128
// Registers: 512 threads are launched with 128 each; the warpgroups redistribute exactly those.
constexpr uint32_t LAUNCH_REGS = 128, SOFTMAX_REGS = 160, CONVERT_REGS = 96, ISSUE_REGS = 96;
static_assert(2 * SOFTMAX_REGS + CONVERT_REGS + ISSUE_REGS <= 4 * LAUNCH_REGS, "setmaxnreg draws on what the block was launched with");

struct Item {
    uint32_t valid, request, head, first_tok, toks, piece, pieces, slot, slot0, counter;  // slot, slot0: of this piece's part and of piece 0's
    int first_pos, band_lo, tile0;  // position of the first query, first key that any row sees, first tile of 64 keys
    int n_tiles[2];                 // of either tile of queries; the second has none, or as many as the unit
    uint32_t nan_met;               // the converting warps: a value that some rows see and others not may be a NaN, and counts as 0 in P V
    __device__ int unit_tiles() const { return max(n_tiles[0], n_tiles[1]); }
    __device__ int last_pos() const { return first_pos + (int)toks - 1; }
};

struct PrefillSmem {
    uint8_t q[2][2][2 * HALF_TILE];  // [tile][dim half][128 rows x 128 B]
    uint8_t k[2][2][HALF_TILE];      // [stage][dim half][64 keys x 128 B]
    uint8_t v[2][2][HALF_TILE];
    uint8_t raw[RAW][2][4][TILE_BYTES];  // [stage][K, V][block]: as cached
    uint64_t item_full[ITEMS], item_empty[ITEMS];
    uint64_t raw_full[RAW], raw_empty[RAW];
    uint64_t full_k[2], full_v[2];   // converting warps: the tile is there
    uint64_t k_free[2], v_free[2];   // MMA commit: both tiles of queries are done with it
    uint64_t s_ready[2][2];          // [tile][buffer] MMA commit: S holds Q K^T
    uint64_t p_ready[2][2];          // softmax threads: P is in tensor memory
    uint64_t pv_done[2][2];          // MMA commit: O += P V is complete
    uint64_t q_full, o_free[2];      // Q's copies; softmax threads: O of the last item has been read
    float4 exps[2 * RAW][2];         // [tile of keys % 8]: the powers of two of K, and the exponents of V, of its four blocks
    Item item[ITEMS];
    uint32_t tmem_base, last[2];
    uint32_t gave_up;                // a role has waited in vain
    uint4 rows[8][32][5];            // of each softmax warp: 32 dims of its 32 rows in f16 on their way out, 80 bytes a row
};
static_assert(sizeof(PrefillSmem) <= 227 * 1024, "shared memory of a CTA");

template <uint32_t N> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <uint32_t N> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Takes items from the queue; by a whole warp, which keeps what is left of its stretch.
struct Feed {
    uint32_t total, items, whole, stretches, rest_tiles;
    bool by_head, sorted, opened = false;
    uint32_t at = 0, end = 0, stretch = 0, next_unit = 0;  // of the stretch: tiles of the cut units that are still to do, the unit that they begin in
};
__device__ __forceinline__ uint32_t stretch_of_tile(const Feed& f, uint32_t tile) { return (uint32_t)((((uint64_t)tile + 1) * f.stretches - 1) / f.rest_tiles); }
__device__ __forceinline__ Feed open_feed(const BlocksAttn& a, const BlocksWork& w)
{
    Feed f;
    f.total = ld_global(w.units_before + a.req.n);  // units of a kv head
    f.items = f.total * a.n_kv;
    f.whole = whole_items(f.items, w.places);
    f.rest_tiles = ld_global(w.rest + w.places);
    f.stretches = rest_stretches(f.rest_tiles, f.items - f.whole, w.places);
    f.by_head = ld_global(w.by_head) != 0;
    f.sorted = f.total <= MOST_SORTED;
    return f;
}
__device__ __forceinline__ void fetch_item(const BlocksAttn& a, const BlocksWork& w, Feed& f, Item* out)
{
    const uint32_t lane = threadIdx.x & 31;
    Item it;
    it.valid = it.nan_met = 0;
    uint32_t i = 0, rest = 0, begin = 0, n = 0;  // the item; of one that is cut: its number among those, its first tile and its tiles
    it.piece = it.slot = it.slot0 = it.counter = 0;
    it.pieces = 1;
    const uint32_t cut = f.items - f.whole;
    for (;;) {
        if (f.at < f.end) {  // on with the stretch
            rest = f.next_unit;
            const uint32_t before = ld_global(w.rest + rest), after = rest + 1 < cut ? ld_global(w.rest + rest + 1) : f.rest_tiles;
            f.next_unit++;
            begin = f.at - before;
            n = min(after, f.end) - f.at;
            f.at += n;
            i = f.whole + rest;
            const uint32_t s0 = stretch_of_tile(f, before), s1 = stretch_of_tile(f, after - 1);
            it.pieces = s1 - s0 + 1;
            it.piece = f.stretch - s0;
            it.slot0 = 2 * s0 + 1;
            it.slot = it.piece ? 2 * f.stretch : it.slot0;
            it.counter = rest;
            break;
        }
        if (f.opened) {
            if (lane == 0) i = gridDim.x + atomicAdd(w.queue, 1u);
            i = __shfl_sync(0xffffffffu, i, 0);
        } else {  // every CTA's first is its own
            i = blockIdx.x;
            f.opened = true;
        }
        if (i < f.whole) break;
        i -= f.whole;
        if (i >= f.stretches) {
            if (lane == 0) *out = it;
            return;
        }
        f.stretch = i;
        f.at = (uint32_t)((uint64_t)f.rest_tiles * i / f.stretches);
        f.end = (uint32_t)((uint64_t)f.rest_tiles * (i + 1) / f.stretches);
        // the unit that tile `at` is of: the last one with rest <= at
        uint32_t lo = 0;
        for (uint32_t base = 0; base < cut; base += 32) {
            const bool le = base + lane < cut && ld_global(w.rest + base + lane) <= f.at;
            lo += __popc(__ballot_sync(0xffffffffu, le));
        }
        f.next_unit = lo - 1;
    }
    uint32_t head, rank;
    split_item(i, f.total, a.n_kv, f.by_head, head, rank);
    uint2 place;
    if (f.sorted) {
        place = ld_global(w.order + rank);
    } else {  // the request of a unit: the last one with units_before <= u
        const uint32_t u = f.total - 1 - rank;
        uint32_t lo = 0, left = a.req.n;
        while (left > 1) {
            const uint32_t step = (left + 31) / 32, probe = lo + lane * step;
            const bool at_or_before = lane * step < left && ld_global(w.units_before + probe) <= u;
            const uint32_t k = 31 - __clz(__ballot_sync(0xffffffffu, at_or_before));  // lane 0 always is
            lo += k * step;
            left = min(step, left - k * step);
        }
        place = make_uint2(lo, u - ld_global(w.units_before + lo));
    }
    const Unit unit = unit_at(a, place.x, place.y);
    it.valid = 1;
    it.request = place.x;
    it.head = head;
    it.first_tok = unit.first_tok;
    it.toks = unit.toks;
    it.first_pos = unit.first_pos;
    it.band_lo = unit.band_lo;
    const int mine = i < f.whole ? unit.n_tiles : min((int)n, unit.n_tiles), half = (ROWS >> (int)a.group_shift);
    it.tile0 = unit.tile0 + (int)begin;
    it.n_tiles[0] = mine;
    it.n_tiles[1] = 0;
    if ((int)it.toks > half) {  // the second tile of queries goes to the end, the first as far as its last query sees
        const int last_first = it.first_pos + half - 1;
        it.n_tiles[1] = mine;
        it.n_tiles[0] = last_first >= 0 ? min(mine, max(0, last_first / KEYS + 1 - it.tile0)) : 0;
    }
    if (lane == 0) *out = it;
}

// Keys of a tile of 64 that some rows of the unit see and others may not.
__device__ __forceinline__ bool crosses_edge(int key0, int first_pos, int last_lo) { return key0 + KEYS - 1 > first_pos || key0 < last_lo; }

// 16 cached bytes as 16 f16 numbers, into two 16-byte chunks of a row.
__device__ __forceinline__ void put_converted(uint32_t chunk0, uint32_t chunk1, const uint4& raw)
{
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t f[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f[2 * i] = e4m3x2_to_f16x2(w[i] & 0xffffu);
        f[2 * i + 1] = e4m3x2_to_f16x2(w[i] >> 16);
    }
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk0), "r"(f[0]), "r"(f[1]), "r"(f[2]), "r"(f[3]) : "memory");
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(chunk1), "r"(f[4]), "r"(f[5]), "r"(f[6]), "r"(f[7]) : "memory");
}

__global__ void __launch_bounds__(THREADS, 1)
    blocks_prefill_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ BlocksAttn a, const __grid_constant__ BlocksWork w, float4* acc_parts, float2* ml_parts)
{
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    PrefillSmem& sm = *reinterpret_cast<PrefillSmem*>(smem_raw);
    uint32_t* status = a.req.status;
    if ((smem_u32(smem_raw) & 1023u) != 0u) {  // the swizzled tiles need it; never seen, but never assumed
        if (threadIdx.x == 0) report_error(status, DEV_ERR_BOUNDS, 640, smem_u32(smem_raw), 0);
        return;
    }
    const int tid = threadIdx.x, warp = warp_uniform(tid >> 5);
    const uint32_t lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < ITEMS; i++) {
            mbar_init(&sm.item_full[i], 1);
            mbar_init(&sm.item_empty[i], ITEM_READERS);
        }
        for (int i = 0; i < RAW; i++) {
            mbar_init(&sm.raw_full[i], 2);  // the copies, and the exponents
            mbar_init(&sm.raw_empty[i], 4);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.full_k[i], 4);
            mbar_init(&sm.full_v[i], 4);
            mbar_init(&sm.k_free[i], 1);
            mbar_init(&sm.v_free[i], 1);
            for (int t = 0; t < 2; t++) {
                mbar_init(&sm.s_ready[t][i], 1);
                mbar_init(&sm.p_ready[t][i], 128);
                mbar_init(&sm.pv_done[t][i], 1);
            }
            mbar_init(&sm.o_free[i], 128);
        }
        mbar_init(&sm.q_full, 1);
        sm.gave_up = 0;
        mbar_fence_init();
    }
    pdl_wait();  // everything this kernel reads comes from earlier kernels of the stream, the cut of the units among it
    pdl_launch_dependents();
    if (warp == 0) {
        tmem_alloc(&sm.tmem_base, TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sm.tmem_base;
    bool failed = false;
    // The roles go through the items each at its own pace, the copies and conversions of the next one beside the end of this one.
    // Buffers are counted through: use u of a buffer of two is tile u of all, a barrier's phase u / 2.  Every wait is bounded, and a
    // role that has waited in vain leaves; the others then run into their own bounds.
    uint32_t nth = 0;
    auto next_item = [&]() -> const Item* {  // by whole warps; null at the end
        const Item& it = sm.item[nth % ITEMS];
        mbar_wait_warp(&sm.item_full[nth % ITEMS], (nth / ITEMS) & 1, status, 652, failed, 20);
        return !failed && it.valid ? &it : nullptr;
    };
    auto done_item = [&]() {  // what it said has been read
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.item_empty[nth % ITEMS]);
        nth++;
    };
    auto phase = [](uint32_t use) { return (use >> 1) & 1u; };

    if (warp >= MMA_WARP) {
        regs_down<ISSUE_REGS>();
        if (warp == MMA_WARP) {
            // ======================= MMA issue (the whole warp runs the loop, one lane issues) =======================
            // The tensor pipe runs ... PV_0(j) QK_0(j+2) PV_1(j) QK_1(j+2) ...: while one tile's softmax is at work the other's products run.
            const uint32_t one = elect_one(), tm = warp_uniform(tmem);
            constexpr uint32_t IDESC_QK = umma_idesc_f16(ROWS, KEYS, 0, 0), IDESC_PV = umma_idesc_f16(ROWS, HD, 0, 1);
            const uint64_t dq = umma_desc_sw128(smem_u32(sm.q[0][0]), 16, 1024), dk = umma_desc_sw128(smem_u32(sm.k[0][0]), 16, 1024),
                           dv = umma_desc_sw128(smem_u32(sm.v[0][0]), HALF_TILE, 1024);
            constexpr uint64_t Q_TILE = Q_BYTES >> 4, Q_HALF = 2 * HALF_TILE >> 4, K_HALF = HALF_TILE >> 4, STAGE = 2 * HALF_TILE >> 4;
            uint32_t nth_q = 0, items[2] = {0, 0};
            uint32_t key = 0, row[2] = {0, 0};  // tiles of keys, and of either tile of queries, before this item
            for (; const Item* it = next_item();) {
                const int n[2] = {warp_uniform(it->n_tiles[0]), warp_uniform(it->n_tiles[1])}, tiles = max(n[0], n[1]);
                done_item();
                if (tiles == 0) continue;
                const int last = n[1] ? 1 : 0;  // the tile of queries whose products come last
                auto issue_qk = [&](int t, int j) {
                    const uint32_t kb = (key + j) & 1, sb = (row[t] + j) & 1;
                    const uint64_t q0 = dq + t * Q_TILE, k0 = dk + kb * STAGE;
                    const uint32_t d = tm + (2 * t + sb) * KEYS;
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) umma_f16_ss(d, q0 + 2 * kk, k0 + 2 * kk, IDESC_QK, kk ? 1u : 0u, one);
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) umma_f16_ss(d, q0 + Q_HALF + 2 * kk, k0 + K_HALF + 2 * kk, IDESC_QK, 1u, one);
                    umma_commit(&sm.s_ready[t][sb], one);
                    if (t == last) umma_commit(&sm.k_free[kb], one);
                };
                auto keys = [&](int j) {  // waited for once, by the first tile that multiplies with them
                    mbar_wait_warp(&sm.full_k[(key + j) & 1], phase(key + j), status, 641, failed);
                    tc_fence_after_sync();
                };
                mbar_wait_warp(&sm.q_full, (nth_q++) & 1, status, 642, failed);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    if (j < tiles) keys(j);
#pragma unroll
                    for (int t = 0; t < 2; t++)
                        if (j < n[t] && !failed) issue_qk(t, j);
                }
                for (int j = 0; j < tiles && !failed; ++j) {
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        if (j >= n[t]) continue;
                        const uint32_t vb = (key + j) & 1, sb = (row[t] + j) & 1;
                        if (j == 0) mbar_wait_warp(&sm.o_free[t], (items[t]++ & 1) ^ 1, status, 653, failed);
                        mbar_wait_warp(&sm.p_ready[t][sb], phase(row[t] + j), status, 643, failed);
                        if (t == 0 || j >= n[0]) mbar_wait_warp(&sm.full_v[vb], phase(key + j), status, 644, failed);
                        if (failed) break;
                        tc_fence_after_sync();
                        const uint64_t v0 = dv + vb * STAGE;
                        const uint32_t pa = tm + (2 * t + sb) * KEYS, d = tm + TMEM_O + t * HD;
                        umma_f16_ts(d, pa, v0, IDESC_PV, j ? 1u : 0u, one);
#pragma unroll
                        for (int kk = 1; kk < 4; kk++) umma_f16_ts(d, pa + kk * 8, v0 + 128 * kk, IDESC_PV, 1u, one);
                        umma_commit(&sm.pv_done[t][sb], one);
                        if (t == last) umma_commit(&sm.v_free[vb], one);
                        if (j + 2 < n[t]) {  // S was read before P(j) was made
                            if (t == 0 || j + 2 >= n[0]) keys(j + 2);
                            if (failed) break;
                            issue_qk(t, j + 2);
                        }
                    }
                }
                key += (uint32_t)tiles;
                row[0] += (uint32_t)n[0];
                row[1] += (uint32_t)n[1];
            }
        } else if (warp == COPY_WARP) {
            // ======================= bytes out of the cache =======================
            // Lane l keeps what concerns one block of 16 tokens of a tile of keys, K's for l = 0..3, V's for l = 4..7: its page's number,
            // asked for two tiles ahead, its exponent, one ahead, and its copy of 2048 bytes.  Blocks that no query sees are not copied.
            const uint32_t side = (lane >> 2) & 1, blk = lane & 3;
            uint32_t stage = 0, round = 0;  // of the raw ring, over all items
            for (; const Item* it = next_item();) {
                const int tiles = it->unit_tiles(), tile0 = it->tile0, band_lo = it->band_lo, last_pos = it->last_pos();
                const uint32_t request = it->request, head = it->head;
                done_item();
                auto key_of = [&](int j) { return (tile0 + j) * KEYS + (int)blk * TILE_TOK; };
                auto seen = [&](int j) { return lane < 8 && j < tiles && key_of(j) <= last_pos && key_of(j) + TILE_TOK > band_lo; };
                auto look = [&](int j) { return ld_global_if(seen(j), page_at(a.req, request, (uint32_t)key_of(j) / TILE_TOK)); };
                auto tile_of = [&](int j, uint32_t page) { return seen(j) ? block_of_page(a.req, request, (uint32_t)key_of(j) / TILE_TOK, page) * a.n_kv + head : NO_SLOT; };
                uint32_t now = tile_of(0, look(0)), page = look(1);
                int e = ld_global_if(now != NO_SLOT, a.exps[side] + now);
                for (int j = 0; j < tiles; ++j) {
                    const uint32_t next = tile_of(j + 1, page);
                    page = look(j + 2);
                    mbar_wait_warp(&sm.raw_empty[stage], (round & 1) ^ 1, status, 650, failed, 50);
                    if (failed) break;
                    const uint32_t copied = __popc(__ballot_sync(0xffffffffu, now != NO_SLOT));
                    if (lane == 0) mbar_arrive_expect_tx(&sm.raw_full[stage], copied * TILE_BYTES);
                    __syncwarp();
                    if (now != NO_SLOT)
                        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                     ::"r"(smem_u32(sm.raw[stage][side][blk])), "l"(a.pool[side] + (size_t)now * TILE_BYTES), "r"(TILE_BYTES), "r"(smem_u32(&sm.raw_full[stage]))
                                     : "memory");
                    const int e_next = ld_global_if(next != NO_SLOT, a.exps[side] + next);
                    if (lane < 8) reinterpret_cast<float*>(sm.exps[stage + RAW * (round & 1)])[lane] = side ? (float)e : __int_as_float((127 + e) << 23);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.raw_full[stage]);
                    e = e_next;
                    now = next;
                    if (++stage == RAW) stage = 0, round++;
                }
            }
        } else if (warp == QUEUE_WARP) {
            Feed feed = open_feed(a, w);
            for (;; nth++) {
                // An item lasts as long as its keys: the bound here grows with the tiles of the one that is waited for.
                const int tiles = nth < ITEMS ? 0 : sm.item[nth % ITEMS].unit_tiles();
                for (int waited = 0; waited <= tiles; waited += TILES_A_WAIT) {
                    bool late = false;
                    mbar_wait_warp(&sm.item_empty[nth % ITEMS], ((nth / ITEMS) & 1) ^ 1, waited + TILES_A_WAIT <= tiles ? nullptr : status, 654, late, 200);
                    failed = late;
                    if (!late || *(volatile uint32_t*)&sm.gave_up) break;
                }
                if (failed) break;
                fetch_item(a, w, feed, &sm.item[nth % ITEMS]);
                __syncwarp();
                const bool valid = sm.item[nth % ITEMS].valid;
                if (lane == 0) mbar_arrive(&sm.item_full[nth % ITEMS]);
                if (!valid) break;
            }
        } else if (warp == QUERY_WARP) {
            // ======================= queries: once the item before has multiplied with its own for the last time =======================
            uint32_t key = 0;
            for (; const Item* it = next_item();) {
                const int tiles = it->unit_tiles(), column = (int)(it->head * a.group), row = (int)it->first_tok;
                const bool both = it->n_tiles[1] != 0;
                done_item();
                if (tiles == 0) continue;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sm.q_full, both ? 2 * Q_BYTES : Q_BYTES);
                    for (int t = 0; t < (both ? 2 : 1); t++) {
                        tma_load_3d(sm.q[t][0], &tm_q, &sm.q_full, 0, column, row + t * (ROWS >> a.group_shift));
                        tma_load_3d(sm.q[t][1], &tm_q, &sm.q_full, 64, column, row + t * (ROWS >> a.group_shift));
                    }
                }
                __syncwarp();
                // phase after phase: a parity tells the awaited one from the one before it, and from no other
                for (int j = 0; j < tiles && !failed; j++, key++) mbar_wait_warp(&sm.k_free[key & 1], phase(key), status, 655, failed, 100);
            }
        }
    } else if (warp >= CONVERT_WARP) {
        // ======================= bytes to f16 =======================
        regs_down<CONVERT_REGS>();
        // Its 16 bytes of every block: eight lanes read one half of a row and the other half of the next, so that neither their reads
        // nor their writes (the swizzle puts the even chunks of an even row where the odd row has its odd ones) meet a bank twice.
        const uint32_t cw = warp - CONVERT_WARP, odd = (lane >> 2) & 1, half = (cw & 1) ^ odd, tok = (cw >> 1) * 8 + (lane >> 2), c = 2 * (lane & 3);
        const uint32_t from = tok * 128 + half * 64 + (lane & 3) * 16;
        const uint32_t to = half * HALF_TILE + tok * 128, at0 = to + ((c ^ (tok & 7)) << 4), at1 = to + (((c + 1) ^ (tok & 7)) << 4);
        // Keys go two tiles ahead of values: Q K^T(j + 2) is issued right behind P V(j), so the order is K(0) K(1) V(0) K(2) V(1) K(3) ...
        // (in step, a tile's K behind the V before it, the tensor pipe waits for K: a chunk of 65536 keys 2055 us, 1905 this way).
        const int window = a.req.window && a.req.window < MOST_KEYS ? (int)a.req.window : (int)MOST_KEYS;
        uint32_t key = 0;  // tiles of keys before this item
        for (; const Item* it = next_item();) {
            const int tiles = it->unit_tiles(), tile0 = it->tile0, band_lo = it->band_lo, last_pos = it->last_pos(), first_pos = it->first_pos;
            const int last_lo = max(last_pos + 1 - window, 0);
            const uint32_t nan_met = smem_u32(&it->nan_met);  // (the softmax warps keep the item until they have read it)
            done_item();
            auto fetch = [&](int side, int j, uint4 (&d)[4]) {
                const uint32_t raw = smem_u32(sm.raw[(key + j) % RAW][side][0]) + from;
#pragma unroll
                for (int x = 0; x < 4; x++)
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(d[x].x), "=r"(d[x].y), "=r"(d[x].z), "=r"(d[x].w)
                                 : "r"(raw + x * TILE_BYTES)
                                 : "memory");
            };
            auto put = [&](int side, int j, const uint4 (&d)[4]) {
                const uint32_t out = smem_u32(side ? sm.v[(key + j) & 1][0] : sm.k[(key + j) & 1][0]);
#pragma unroll
                for (int x = 0; x < 4; x++) put_converted(out + at0 + x * 2048, out + at1 + x * 2048, d[x]);
            };
            auto done = [&](int side, int j) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(side ? &sm.full_v[(key + j) & 1] : &sm.full_k[(key + j) & 1]);
            };
            auto convert = [&](int side, int j) {
                uint4 d[4];
                fetch(side, j, d);
                put(side, j, d);
                done(side, j);
            };
            // Of values that not every row sees: those that none sees count as 0 (their weight is 0, but 0 times a NaN that stands there would not be), and so
            // do NaNs, which get into the rows that see them at their end.  (Keys need neither: a score that is masked is none, whatever it was.)
            auto convert_edge = [&](int j) {
                const int key0 = (tile0 + j) * KEYS + (int)tok;
                uint4 d[4];
                fetch(1, j, d);
                bool any = false;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    if (key0 + 16 * x > last_pos || key0 + 16 * x < band_lo) d[x] = make_uint4(0u, 0u, 0u, 0u);
                    any |= drop_nans(d[x]);
                }
                if (any) asm volatile("st.shared.u32 [%0], %1;" ::"r"(nan_met), "r"(1) : "memory");
                put(1, j, d);
                done(1, j);
            };
            auto keys = [&](int j) {
                mbar_wait_warp(&sm.raw_full[(key + j) % RAW], ((key + j) / RAW) & 1, status, 651, failed);
                if (key + j >= 2) mbar_wait_warp(&sm.k_free[(key + j) & 1], phase(key + j - 2), status, 645, failed, 20);
                if (!failed) convert(0, j);
            };
            if (tiles > 0) keys(0);
            if (tiles > 1 && !failed) keys(1);
            for (int j = 0; j < tiles && !failed; ++j) {
                if (key + j >= 2) mbar_wait_warp(&sm.v_free[(key + j) & 1], phase(key + j - 2), status, 646, failed, 20);
                if (failed) break;
                if (crosses_edge((tile0 + j) * KEYS, first_pos, last_lo)) convert_edge(j); else convert(1, j);
                if (lane == 0) mbar_arrive(&sm.raw_empty[(key + j) % RAW]);
                if (j + 2 < tiles) keys(j + 2);
            }
            key += (uint32_t)tiles;
        }
    } else {
        // ======================= softmax: row r of tile t <-> tensor-memory lane r <-> thread r of warpgroup t =======================
        regs_up<SOFTMAX_REGS>();
        const int r = tid & 127, t = warp >> 2;
        const float scale2 = a.scale * 1.4426950408889634f;  // > 0 (checked on the host)
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16), s_at = lane_addr + 2 * t * KEYS, o_at = lane_addr + TMEM_O + t * HD;
        const uint32_t tok = (uint32_t)t * (ROWS >> a.group_shift) + ((uint32_t)r >> a.group_shift);
        const int window = a.req.window && a.req.window < MOST_KEYS ? (int)a.req.window : (int)MOST_KEYS;
        uint32_t row = 0, key = 0;  // tiles of this warpgroup's, and of keys (for the exponents' ring), before this item
        for (;;) {
            const Item* at = next_item();
            if (named_barrier_or(1 + t, 128, failed)) {  // its warps leave together: they meet at barriers without a limit
                failed = true;
                break;
            }
            if (!at) break;
            const int tiles = at->n_tiles[t], unit_tiles = at->unit_tiles();
            const struct {
                uint32_t head, first_tok, toks, pieces, slot, slot0, counter;
                int first_pos, tile0, last_pos;
            } it = {at->head, at->first_tok, at->toks, at->pieces, at->slot, at->slot0, at->counter, at->first_pos, at->tile0, at->last_pos()};
            const int tile0 = it.tile0, pos = it.first_pos + (int)tok, row_lo = max(pos + 1 - window, 0);
            const int first_pos = it.first_pos + t * (ROWS >> a.group_shift), last_lo = max(it.last_pos + 1 - window, 0);
            float m_run = NEG_SENTINEL, l_run = 0.0f;
            for (int j = 0; j < tiles; ++j) {
                const int b = (int)((row + j) & 1), key0 = (tile0 + j) * KEYS;
                mbar_wait(&sm.s_ready[t][b], phase(row + j), status, 647, failed);
                tc_fence_after_sync();
                float v[64];
                {
                    uint32_t a0[32], a1[32];
                    tmem_ld_32x32b_x32(s_at + b * KEYS, a0);
                    tmem_ld_32x32b_x32(s_at + b * KEYS + 32, a1);
                    tc_wait_ld();
#pragma unroll
                    for (int x = 0; x < 32; x++) {
                        v[x] = __uint_as_float(a0[x]);
                        v[32 + x] = __uint_as_float(a1[x]);
                    }
                }
                if (key0 + KEYS - 1 > first_pos || key0 < last_lo) {  // the tile crosses an edge of the band: keys [lo, end) as a bit each
                    const int lo = min(max(row_lo - key0, 0), KEYS), end = min(max(pos + 1 - key0, 0), KEYS);
                    const uint64_t upto = end == KEYS ? ~0ull : (1ull << end) - 1, from = lo == KEYS ? 0ull : ~0ull << lo;
                    const uint32_t seen[2] = {(uint32_t)(upto & from), (uint32_t)((upto & from) >> 32)};
#pragma unroll
                    for (int x = 0; x < 64; x++)
                        if (((seen[x / 32] >> (x % 32)) & 1u) == 0) v[x] = -INFINITY;
                }
                // Block by block of 16 keys: scores times K's power of two, plus V's exponent (the weights carry V's scale, l does not).
                const float4 k4 = sm.exps[(key + j) & (2 * RAW - 1)][0], v4 = sm.exps[(key + j) & (2 * RAW - 1)][1];
                const float ks[4] = {k4.x * scale2, k4.y * scale2, k4.z * scale2, k4.w * scale2}, ve[4] = {v4.x, v4.y, v4.z, v4.w};
                float mx = -INFINITY;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    float m0 = max3(v[16 * x], v[16 * x + 1], v[16 * x + 2]), m1 = max3(v[16 * x + 3], v[16 * x + 4], v[16 * x + 5]);
#pragma unroll
                    for (int y = 6; y < 16; y += 5) {
                        m0 = max3(m0, v[16 * x + y], v[16 * x + y + 1]);
                        m1 = max3(m1, v[16 * x + y + 2], v[16 * x + y + 3]);
                        m0 = fmaxf(m0, v[16 * x + y + 4]);
                    }
                    mx = fmaxf(mx, fmaf(fmaxf(m0, m1), ks[x], ve[x]));
                }
                const bool grow = mx > m_run + GROWTH_T;
                float corr = 1.0f;
                if (grow) {
                    const float m = mx - LIFT;
                    corr = ex2(m_run - m);
                    m_run = m;
                    l_run *= corr;
                }
                uint32_t pk[32];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const float2 sc2 = make_float2(ks[x], ks[x]), neg_m = make_float2(ve[x] - m_run, ve[x] - m_run);
                    float2 ls[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                    for (int y = 8 * x; y < 8 * x + 8; y++) {
                        const float2 z = __ffma2_rn(make_float2(v[2 * y], v[2 * y + 1]), sc2, neg_m);
                        const float2 pp = make_float2(ex2(z.x), ex2(z.y));
                        ls[y & 1] = __fadd2_rn(ls[y & 1], pp);  // l from the unrounded weights
                        pk[y] = pack_half2(pp.x, pp.y);
                    }
                    l_run = fmaf((ls[0].x + ls[0].y) + (ls[1].x + ls[1].y), __int_as_float((127 - (int)ve[x]) << 23), l_run);
                }
                // O is scaled anew where a row's maximum moved, once P V of the tile before is complete.
                if (j > 0 && __any_sync(0xffffffffu, grow)) {
                    mbar_wait(&sm.pv_done[t][b ^ 1], phase(row + j - 1), status, 648, failed);
                    tc_fence_after_sync();
#pragma unroll 1
                    for (int c = 0; c < 4; c++) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(o_at + 32 * c, o);
                        tc_wait_ld();
#pragma unroll
                        for (int x = 0; x < 32; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * corr);
                        tmem_st_32x32b_x32(o_at + 32 * c, o);
                    }
                }
                tmem_st_32x32b_x32(s_at + b * KEYS, pk);
                tc_wait_st();
                tc_fence_before_sync();
                mbar_arrive(&sm.p_ready[t][b]);
            }
            if (tiles > 0) mbar_wait(&sm.pv_done[t][(row + tiles - 1) & 1], phase(row + tiles - 1), status, 649, failed);  // the last P V: all of them
            tc_fence_after_sync();

            // ---- out = O / l, or this piece's part ----
            const bool live = tok < it.toks, whole = it.pieces == 1;
            // A part is [32 groups of four dims][128 rows] and (m, l) of the rows: neighbouring threads write neighbouring 16 bytes.
            const auto part = [&](uint32_t s) { return acc_parts + (size_t)(2 * s + t) * (HD / 4) * ROWS + r; };
            const auto part_ml = [&](uint32_t s) { return ml_parts + (size_t)(2 * s + t) * ROWS + r; };
            const float mul = l_run != 0.0f ? 1.0f / l_run : 0.0f;
            const bool blank = __any_sync(0xffffffffu, l_run == 0.0f);
            __half* row_out[4];  // where this thread stores its sixteen bytes of other threads' rows
            bool row_live[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const uint32_t other = (uint32_t)(warp & 3) * 32 + 8 * x + (lane >> 2), tk = (uint32_t)t * (ROWS >> a.group_shift) + (other >> a.group_shift);
                row_live[x] = tk < it.toks;
                row_out[x] = a.out + ((size_t)(it.first_tok + tk) * (a.n_kv * a.group) + it.head * a.group + (other & (a.group - 1))) * HD + 8 * (lane & 3);
            }
#pragma unroll 1
            for (int c = 0; c < 4; c++) {
                uint32_t o[32];
                if (tiles > 0) {  // the same for all
                    tmem_ld_32x32b_x32(o_at + 32 * c, o);
                    tc_wait_ld();
                } else {
#pragma unroll
                    for (int x = 0; x < 32; x++) o[x] = 0u;
                }
                if (c == 3 && tiles > 0) {  // O may be overwritten
                    tc_fence_before_sync();
                    mbar_arrive(&sm.o_free[t]);
                }
                if (whole) {
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        uint4 h;
                        uint32_t* hw = reinterpret_cast<uint32_t*>(&h);
#pragma unroll
                        for (int y = 0; y < 4; y++) {
                            const float2 z = __fmul2_rn(make_float2(__uint_as_float(o[8 * x + 2 * y]), __uint_as_float(o[8 * x + 2 * y + 1])), make_float2(mul, mul));
                            hw[y] = pack_half2(z.x, z.y);
                        }
                        if (blank && l_run == 0.0f) h = make_uint4(0u, 0u, 0u, 0u);  // a row that saw nothing is 0, whatever stands in V
                        sm.rows[warp][lane][x] = h;
                    }
                    // 64 bytes of each of eight rows go out together (a thread's own row by itself would meet a line a thread)
                    __syncwarp();
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (row_live[x]) *reinterpret_cast<uint4*>(row_out[x] + 32 * c) = sm.rows[warp][8 * x + (lane >> 2)][lane & 3];
                    __syncwarp();
                } else if (live) {
#pragma unroll
                    for (int x = 0; x < 8; x++)
                        part(it.slot)[(8 * c + x) * ROWS] = make_float4(__uint_as_float(o[4 * x]), __uint_as_float(o[4 * x + 1]), __uint_as_float(o[4 * x + 2]), __uint_as_float(o[4 * x + 3]));
                }
            }
            // NaNs that the converting warps took out, at keys that this row sees: into what it has written (its row by other threads of the warp).
            if (live && *(const volatile uint32_t*)&at->nan_met) {
                const uint32_t request = at->request;
#pragma unroll 1
                for (int x = max(tile0 * KEYS, row_lo); x <= min((tile0 + tiles) * KEYS - 1, pos); x++) {
                    if (!crosses_edge(x / KEYS * KEYS, it.first_pos, last_lo)) continue;
                    const size_t block = block_of_page(a.req, request, (uint32_t)x / TILE_TOK, ld_global(page_at(a.req, request, (uint32_t)x / TILE_TOK)));
                    const uint8_t* v = a.pool[1] + (block * a.n_kv + it.head) * TILE_BYTES + x % TILE_TOK * HD;
#pragma unroll 1
                    for (uint32_t d = 0; d < (uint32_t)HD; d++) {
                        if ((*(const volatile uint8_t*)(v + d) & 0x7f) != 0x7f) continue;
                        if (whole) a.out[((size_t)(it.first_tok + tok) * (a.n_kv * a.group) + it.head * a.group + ((uint32_t)r & (a.group - 1))) * HD + d] = __ushort_as_half(0x7fff);
                        else reinterpret_cast<float*>(part(it.slot) + d / 4 * ROWS)[d % 4] = __int_as_float(0x7fffffff);
                    }
                }
            }
            if (!whole) {
                if (live) *part_ml(it.slot) = make_float2(m_run, l_run);
                __threadfence();
                named_barrier_sync(1 + t, 128);
                if (r == 0) {
                    const uint32_t before = atomicAdd(w.done + 2 * it.counter + t, 1u);
                    sm.last[t] = before + 1 == it.pieces;
                    __threadfence();
                }
                named_barrier_sync(1 + t, 128);
                if (sm.last[t]) {  // all pieces are written: merge them in their order
                    // Few rows are spread over all threads, every thread with a part of a row's dims; sixteen dims of four pieces are on their way at a time
                    // (a piece after another and a row a thread: 16 pieces of 32 rows took 13 us more).
                    const uint32_t in_tile = (uint32_t)t * (ROWS >> a.group_shift), rows = it.toks > in_tile ? min((it.toks - in_tile) << a.group_shift, (uint32_t)ROWS) : 0;
                    const uint32_t shares = rows <= ROWS / 4 ? 4 : rows <= ROWS / 2 ? 2 : 1, share_rows = ROWS / shares, at_row = (uint32_t)r & (share_rows - 1), share = (uint32_t)r / share_rows;
                    const float4* acc_at = acc_parts + (size_t)t * (HD / 4) * ROWS + at_row;
                    const float2* ml_at = ml_parts + (size_t)t * ROWS + at_row;
                    const auto slot = [&](uint32_t p) { return 2 * (size_t)(p ? it.slot0 - 1 + 2 * p : it.slot0); };
                    if (at_row < rows) {
                        float big = NEG_SENTINEL, den = 0.0f;
#pragma unroll 4
                        for (uint32_t p = 0; p < it.pieces; p++) big = fmaxf(big, __ldcg(ml_at + slot(p) * ROWS).x);
#pragma unroll 4
                        for (uint32_t p = 0; p < it.pieces; p++) {
                            const float2 ml = __ldcg(ml_at + slot(p) * ROWS);
                            den = fmaf(ex2(ml.x - big), ml.y, den);
                        }
                        const float inv = den != 0.0f ? 1.0f / den : 0.0f;
                        __half* to = a.out + ((size_t)(it.first_tok + in_tile + (at_row >> a.group_shift)) * (a.n_kv * a.group) + it.head * a.group + (at_row & (a.group - 1))) * HD;
#pragma unroll 1
                        for (uint32_t c = share; c < 8; c += shares) {
                            float4 acc[4] = {};
#pragma unroll 1
                            for (uint32_t p0 = 0; p0 < it.pieces; p0 += 4) {
                                float4 o[4][4];
                                float f[4];
#pragma unroll
                                for (uint32_t y = 0; y < 4; y++) {
                                    const size_t from = slot(min(p0 + y, it.pieces - 1));  // (those past the end are the last one again, and count nothing)
                                    f[y] = __ldcg(ml_at + from * ROWS).x;
#pragma unroll
                                    for (int x = 0; x < 4; x++) o[y][x] = __ldcg(acc_at + from * (HD / 4) * ROWS + (4 * c + x) * ROWS);
                                }
#pragma unroll
                                for (uint32_t y = 0; y < 4; y++) {
                                    const float w = p0 + y < it.pieces ? ex2(f[y] - big) * inv : 0.0f;
#pragma unroll
                                    for (int x = 0; x < 4; x++) {
                                        acc[x].x = fmaf(w, o[y][x].x, acc[x].x);
                                        acc[x].y = fmaf(w, o[y][x].y, acc[x].y);
                                        acc[x].z = fmaf(w, o[y][x].z, acc[x].z);
                                        acc[x].w = fmaf(w, o[y][x].w, acc[x].w);
                                    }
                                }
                            }
#pragma unroll
                            for (int x = 0; x < 2; x++)
                                *reinterpret_cast<uint4*>(to + 16 * c + 8 * x) = den == 0.0f ? make_uint4(0u, 0u, 0u, 0u) :
                                    make_uint4(pack_half2(acc[2 * x].x, acc[2 * x].y), pack_half2(acc[2 * x].z, acc[2 * x].w), pack_half2(acc[2 * x + 1].x, acc[2 * x + 1].y),
                                               pack_half2(acc[2 * x + 1].z, acc[2 * x + 1].w));
                        }
                    }
                }
            }
            key += (uint32_t)unit_tiles;
            row += (uint32_t)tiles;
            done_item();  // only now: the queue gives out the next but one behind it
        }
    }
    if (failed) sm.gave_up = 1;
    // A wait that ran out leaves MMAs (and Q's copy) in flight that nobody waits for: they get a bounded time to land.
    if (__syncthreads_or(failed)) {
        let_copies_land();
        __syncthreads();
    }
    if (warp == 0) tmem_dealloc(tmem, TMEM_COLS);
}

}  // namespace

// Two parts for every stretch: of the unit that it goes on with, and of the one that it begins and does not end.
size_t blocks_prefill_work(int sm_count) { return 2ull * blocks_places(sm_count) * UNIT_ROWS * (HD + 2) * 4; }

int launch_blocks_prefill(const LaunchArgs& a, const BlocksAttn& k, const BlocksWork& work)
{
    CUtensorMap tm_q;
    {
        const uint64_t heads = (uint64_t)k.n_kv * k.group;
        const uint64_t dims[3] = {HD, heads, k.req.tokens}, strides[2] = {HD * 2, heads * HD * 2};
        const uint32_t box[3] = {64, k.group, ROWS / k.group};
        if (int r = encode_tensor_map(a, &tm_q, 1, 3, const_cast<__half*>(k.q), dims, strides, box, 3)) return r;
    }
    const size_t smem = sizeof(PrefillSmem);
    {
        static std::mutex attr_mutex;
        static bool attr_set[64] = {};
        std::lock_guard<std::mutex> lock(attr_mutex);
        if (a.device < 0 || a.device >= 64 || !attr_set[a.device]) {
            if (int r = check_cuda(a, cudaFuncSetAttribute(blocks_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "cudaFuncSetAttribute(blocks_prefill)"))
                return r;
            cudaFuncAttributes at;
            if (int r = check_cuda(a, cudaFuncGetAttributes(&at, blocks_prefill_kernel), "cudaFuncGetAttributes(blocks_prefill)")) return r;
            if (at.numRegs < (int)LAUNCH_REGS) {  // setmaxnreg.inc would wait for registers that the block does not have
                if (a.err) *a.err = "blocks_prefill_kernel was built with fewer registers than it redistributes";
                return 4;
            }
            if (a.device >= 0 && a.device < 64) attr_set[a.device] = true;
        }
    }
    float4* acc = reinterpret_cast<float4*>(work.parts);
    float2* ml = reinterpret_cast<float2*>(acc + 2ull * work.places * UNIT_ROWS * (HD / 4));
    const cudaError_t e = launch_dependent(blocks_prefill_kernel, dim3(work.places), dim3(THREADS), smem, a.stream, tm_q, k, work, acc, ml);
    ++*a.launches;
    return check_cuda(a, e, "attn_blocks prefill");
}

}  // namespace sgb
