// Attention of many requests with few queries each over the 8-bit cache of blocks.cuh: decode, and the verification of short drafts.
//
// The work is the flat list of all requests' 16-token tiles, in their order, for every kv head.  The lengths are known on the device
// only, so the list is cut there: every warp that fits the GPU at once takes an equal stretch of one head's list, whatever
// the requests' lengths are, and walks it tile by tile through its own ring of TMA copies, which runs on across the ends of
// requests.  A request that lies in one stretch is finished by its warp; of one that several warps share each leaves (O, m, l), and a
// second kernel merges them in the list's order, so reruns give the same bits.  (The cut rests on all lengths, so a request's bits
// depend on its neighbours' lengths.)
//
// One tile: S = K Q^T with the 16 tokens as M and eight query rows (or twice eight) as N of mma.sync m16n8k16 (far below tcgen05's 64
// rows), e4m3 -> f16 exactly on the way from shared memory (ldmatrix, one conversion a pair), O^T += V^T P^T with 16 dims as M.
// The powers of two never touch the elements: K's multiplies the scores, V's goes into the exponent, P' = 2^(s + e_v - m),
// and out of the sum again, l += P' 2^-e_v.  P' goes into the second product as f16, 2^-11 of itself off at most in f16's normal range (LIFT says how far
// that reaches); l takes it unrounded.  Softmax in base 2 with a running maximum that is raised when it grows by more than 2^8:
// every lane compares its own scores with it, a row's maximum over the lanes is found only where one is that much larger (three shuffles
// a tile and row, and the wait for them: 64 requests 114 us, 107 without).
// Bound by the cache's bytes: 2 x 128 1/16 per token and kv head.  16 kv heads, two query heads each: 64 requests of 256 to 8192 keys 108 us
// (5.5 TB/s; 6.3 in this kernel, the merge is 7 to 8 us by itself), one of 131072 96 to 98 us, drafts of 2 to 4 tokens over up to 32768 keys in 16 requests
// 140 us (5.5 TB/s), one of 1000 keys 11.5 us.  Two blocks of rows are bound by their warps' own latency: drafts of 4 to 8 tokens 185 us (4.2 TB/s).
#include <mutex>
#include <type_traits>

#include "blocks.cuh"
#include "blocks_work.cuh"
#include "sgb_kernels.h"

namespace sgb {

namespace {

constexpr int HD = 128;
constexpr int WARPS = 4;
constexpr uint32_t LEAST_TILES = 2;  // of a stretch: fewer mean more to merge (one request of 1000 keys, 16 heads: 12.3 us with 4, 11.5 with 2, 11.1 with 1)
// A request weighs a tile more than it has: its queries to fetch, its result to write.  (256 requests of 17 to 2048 keys: without it
// the warps with many short ones end last, 61.9 us instead of 57.4.)
constexpr uint32_t REQUEST_WEIGHT = 1;
constexpr uint32_t STAGE_BYTES = 2 * TILE_BYTES;

// What the arithmetic needs of a request, left for it by the side that copies, which comes to it up to STAGES tiles earlier.
struct Met {
    uint32_t request, first, n, len, lo, tiles;
};
static_assert(REQUEST_WEIGHT == 1, "a stretch that begins within a request's own weight begins with it");

// What NB blocks of eight query rows take: O alone is 32 NB registers a thread, so three CTAs of 168 registers stand on an SM for two blocks.
// Their queries, another 32, are kept in shared memory, every lane's own beside each other.  (Four blocks: eight warps on an SM cannot hide
// their own latency; 16 drafts of 2 to 4 tokens of eight heads a group 187 us, as prompts 88.)
template <int NB> struct Shape {
    static constexpr int CTAS_PER_SM = NB == 1 ? 4 : 3, STAGES = 3;
    static constexpr int MET = 4;  // STAGES tiles under way are of three requests at most
    static constexpr bool Q_SHARED = NB > 1;
    static_assert(MET > STAGES, "a request is not overwritten before its last tile");
};
template <int NB>
struct __align__(1024) DecodeSmem {
    static constexpr int STAGES = Shape<NB>::STAGES, MET = Shape<NB>::MET;
    uint8_t k[WARPS][STAGES][TILE_BYTES];  // 128-byte swizzled by TMA
    uint8_t v[WARPS][STAGES][TILE_BYTES];
    uint64_t full[WARPS][STAGES];
    uint64_t sums[WARPS];
    Met met[WARPS][MET];  // the last requests that a warp's copies have come to
    uint32_t from[WARPS]; // weight of a stretch's first request that lies before it
    uint32_t begun[WARPS][2];  // requests that begin before a stretch, before its end
    uint2 q[Shape<NB>::Q_SHARED ? WARPS : 1][Shape<NB>::Q_SHARED ? 8 * NB : 1][32];
};

// Parts: (m, l) and O of [slot][kv head][row].  A stretch p has slot 2p for the request that it goes on with and 2p + 1 for
// one that it begins and does not end.
struct Work {
    BlocksWork head;
    float2* ml;
    float4* acc;
    uint32_t rows;
};
inline uint32_t part_rows(uint32_t most_rows, uint32_t group, uint32_t max_q)
{
    const uint32_t tokens = most_rows / group;
    return group * (max_q < tokens ? max_q : tokens);
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a)
{
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// Over the eight lanes that share lane % 4: the tokens of a tile.
__device__ __forceinline__ float tok_max(float v)
{
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float tok_sum(float v)
{
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// The tiles of a request that any of its queries sees: [lo, lo + n).  None of a request that is prefilled.
struct Tiles {
    uint32_t lo, n;
    __device__ uint32_t weight() const { return n ? n + REQUEST_WEIGHT : 0; }
};
__device__ __forceinline__ Tiles tiles_of(const BlocksAttn& a, const Request& q)
{
    if (q.n == 0 || q.n > a.few || q.len == 0) return Tiles{0, 0};
    const int64_t from = (int64_t)q.len - q.n + 1 - a.req.window;
    const uint32_t lo = a.req.window != 0 && from > 0 ? (uint32_t)from / TILE_TOK : 0;
    return Tiles{lo, (q.len + TILE_TOK - 1) / TILE_TOK - lo};
}
// `total` tiles in `n` stretches, the first `longer` of them of each + 1 tiles, the others of `each`.  (A division of 64 bits costs some
// hundred cycles, and this stands before the first copy: with one for every end of a stretch one request of 131072 keys took 102.5 us
// instead of 98.7.)
struct Stretches {
    uint64_t each;
    uint32_t n, longer;
    __device__ uint64_t begin(uint32_t p) const { return each * p + min(p, longer); }
    __device__ uint32_t of(uint64_t tile) const
    {
        const uint64_t in_longer = (each + 1) * longer;
        if (tile < in_longer) return tile >> 32 ? (uint32_t)(tile / (each + 1)) : (uint32_t)tile / ((uint32_t)each + 1);
        const uint64_t t = tile - in_longer;
        return longer + (t >> 32 ? (uint32_t)(t / each) : (uint32_t)t / (uint32_t)each);
    }
};
__device__ __forceinline__ Stretches stretches_for(uint64_t total, uint32_t most)
{
    Stretches s;
    const uint64_t n = (total + LEAST_TILES - 1) / LEAST_TILES;
    s.n = n < most ? (uint32_t)n : most;
    s.each = s.n == 0 ? 0 : total >> 32 ? total / s.n : (uint32_t)total / s.n;
    s.longer = (uint32_t)(total - s.each * s.n);
    return s;
}

// DRAFTS: a request may have more than one token.
template <int NB, bool DRAFTS>
__global__ void __launch_bounds__(WARPS * 32, Shape<NB>::CTAS_PER_SM)
    blocks_decode_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ BlocksAttn a, const __grid_constant__ Work work, uint32_t most)
{
    constexpr int STAGES = Shape<NB>::STAGES, MET = Shape<NB>::MET;
    constexpr bool Q_SHARED = Shape<NB>::Q_SHARED;
    extern __shared__ uint8_t smem_raw[];
    DecodeSmem<NB>& sm = *reinterpret_cast<DecodeSmem<NB>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    if (lane == 0) {
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
        for (int i = 0; i < STAGES; i++) mbar_init(&sm.full[warp][i], 1);
        mbar_fence_init();
    }
    pdl_wait();  // lengths, tables, queries and the cache come from earlier kernels of the stream
    pdl_launch_dependents();

    // ---- cut the list: every CTA sums up all requests' tiles and finds where its own warps begin ---------------------------------
    const uint32_t flat = blockIdx.x * WARPS + warp, head = flat % a.n_kv, part = flat / a.n_kv;
    const uint32_t per_thread = (a.req.n + WARPS * 32 - 1) / (WARPS * 32);
    const uint32_t r_begin = min(threadIdx.x * per_thread, a.req.n), r_end = min(r_begin + per_thread, a.req.n);
    Request rq{0, 0, 0};
    constexpr int COUNT_BITS = 17;  // of the sums: requests with tiles (at most MOST_REQUESTS) below, weights above
    uint64_t mine = 0;
    const auto add = [&](uint32_t, const Request& q) {
        rq = q;
        const Tiles tl = tiles_of(a, q);
        mine += (uint64_t)tl.weight() << COUNT_BITS | (tl.n ? 1 : 0);
    };
    if (per_thread == 1) {
        if (r_begin < r_end) add(r_begin, request_at(a.req, r_begin));
    } else {
        for_requests(a.req, r_begin, r_end, add);
    }
    uint64_t up_to = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint64_t t = __shfl_up_sync(0xffffffffu, up_to, off);
        if (lane >= (uint32_t)off) up_to += t;
    }
    if (lane == 31) sm.sums[warp] = up_to;
    __syncthreads();
    uint64_t all = 0, base = up_to - mine;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
        if (w < (int)warp) base += sm.sums[w];
        all += sm.sums[w];
    }
    const uint64_t total = all >> COUNT_BITS;
    const Stretches cut = stretches_for(total, most);
    if (total != 0) {
        uint64_t want[WARPS][2];  // where the warps' stretches begin and end
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const uint32_t p = (blockIdx.x * WARPS + w) / a.n_kv;
            want[w][0] = p < cut.n ? cut.begin(p) : ~0ull;
            want[w][1] = p < cut.n ? cut.begin(p + 1) : ~0ull;
        }
        uint64_t at = base >> COUNT_BITS;
        uint32_t nth = (uint32_t)base & ((1u << COUNT_BITS) - 1);
        const auto find = [&](uint32_t r, const Request& q) {
            const Tiles tiles = tiles_of(a, q);
            const uint64_t end = at + tiles.weight();
#pragma unroll
            for (int w = 0; w < WARPS; w++) {
                if (want[w][0] >= at && want[w][0] < end) {
                    sm.met[w][0] = Met{r, q.first, q.n, q.len, tiles.lo, tiles.n};
                    sm.from[w] = (uint32_t)(want[w][0] - at);
                }
#pragma unroll
                for (int i = 0; i < 2; i++)
                    if (want[w][i] >= at && want[w][i] < end) sm.begun[w][i] = nth + (want[w][i] > at ? 1 : 0);
            }
            if (blockIdx.x == 0) work.head.before[r] = at;
            at = end;
            nth += tiles.n ? 1 : 0;
        };
        if (per_thread == 1) {
            if (r_begin < r_end) find(r_begin, rq);
        } else {
            for_requests(a.req, r_begin, r_end, find);
        }
    } else if (blockIdx.x == 0) {
        for (uint32_t r = r_begin; r < r_end; r++) work.head.before[r] = 0;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        work.head.before[a.req.n] = total;
        work.head.before[a.req.n + 1] = most;
    }
    __syncthreads();
    if (part >= cut.n) return;
    // The tiles of the stretch are its weights less those of the requests that begin in it.
    const uint64_t part_end = cut.begin(part + 1);
    const uint32_t begun_end = part_end == total ? (uint32_t)all & ((1u << COUNT_BITS) - 1) : sm.begun[warp][1];
    const uint32_t n_iter = (uint32_t)(part_end - cut.begin(part)) - REQUEST_WEIGHT * (begun_end - sm.begun[warp][0]);
    if (n_iter == 0) return;
    const uint32_t passed = sm.from[warp] > REQUEST_WEIGHT ? sm.from[warp] - REQUEST_WEIGHT : 0;  // tiles of the first request that lie before

    // ---- the copies' side: STAGES tiles ahead of the arithmetic -------------------------------------------------------------------
    uint32_t to_r = sm.met[warp][0].request, to_nth = 0, to_tile = sm.met[warp][0].lo + passed, to_left = sm.met[warp][0].tiles - passed;
    // The first pages are asked for side by side, by a lane each.
    const uint32_t tile0 = to_tile, left0 = to_left;
    const uint32_t first_pages = ld_global_if(lane < STAGES && lane < left0 && lane < n_iter, page_at(a.req, to_r, to_tile + lane));
    auto next_tile = [&]() {
        to_tile++;
        if (--to_left == 0) {
            Tiles t{0, 0};
            Request q{0, 0, 0};
            while (t.n == 0 && ++to_r < a.req.n) {
                q = request_at(a.req, to_r);
                t = tiles_of(a, q);
            }
            to_tile = t.lo;
            to_left = t.n;
            to_nth++;
            if (lane == 0) sm.met[warp][to_nth % MET] = Met{to_r, q.first, q.n, q.len, t.lo, t.n};
        }
    };
    uint32_t to_page = 0;
    auto look = [&]() { to_page = ld_global(page_at(a.req, to_r, to_tile)); };
    // What is under way: which of the warp's requests, tile, and (lanes 0 and 1) the exponents of K and V.
    uint32_t way_r[STAGES], way_tile[STAGES];
    int way_exp[STAGES];
    const CUtensorMap* my_map = lane == 0 ? &tm_k : &tm_v;
    const uint32_t my_dst = lane == 0 ? smem_u32(sm.k[warp][0]) : smem_u32(sm.v[warp][0]);
    const int8_t* my_exps = a.exps[lane & 1];
    const uint32_t bar0 = smem_u32(&sm.full[warp][0]);
    auto issue = [&](uint32_t st, int& e) {
        const uint32_t bar = bar0 + st * 8, tile = block_of_page(a.req, to_r, to_tile, to_page) * a.n_kv + head;
        e = ld_global_if(lane < 2, my_exps + tile);
        if (lane < 2) {
            if (lane == 0) {
                fence_proxy_async_smem();  // the slot's previous contents were read through the generic proxy
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(STAGE_BYTES) : "memory");
            }
            asm volatile(
                "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                ::"r"(my_dst + st * TILE_BYTES), "l"(reinterpret_cast<uint64_t>(my_map)), "r"(bar), "r"(0), "r"(0), "r"((int)tile)
                : "memory");
        }
    };
    // ---- the arithmetic's side ------------------------------------------------------------------------------------------------------
    // Of every block of eight rows a lane supplies Q for row g (B operand) and owns the accumulators of rows 2 t4 and 2 t4 + 1.
    // Row = token * group + head.
    const uint32_t heads = a.n_kv * a.group;
    uint2 qb[Q_SHARED ? 1 : NB][8];
    float o[NB][8][4], m_run[NB][2], l_part[NB][2];
    uint32_t r_now = 0, rows = 0, first_tok = 0, tile_first = 0, tile_begin = 0, tile_end = 0;
    int pos0 = 0, len = 0, lo_all = 0, lo_any = 0;  // position of the first query; the first keys that all rows, that any row sees
    const int window = a.req.window && a.req.window < MOST_KEYS ? (int)a.req.window : (int)MOST_KEYS;
    auto begin_request = [&](uint32_t nth, uint32_t tile) {
        __syncwarp();  // lane 0 left it there
        const Met rq = sm.met[warp][nth % MET];
        r_now = nth;
        rows = rq.n * a.group;
        first_tok = rq.first;
        tile_first = tile;
        tile_begin = rq.lo;
        tile_end = rq.lo + rq.tiles;
#pragma unroll
        for (int n = 0; n < NB; n++) {
            const uint32_t row = 8 * n + g;
            const bool on = row < rows;
            const __half* qrow = a.q + ((size_t)(rq.first + (on ? row >> a.group_shift : 0)) * heads + head * a.group + (row & (a.group - 1))) * HD + 4 * t4;
#pragma unroll
            for (int c = 0; c < 8; c++) {
                if constexpr (Q_SHARED) {
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(&sm.q[warp][8 * n + c][lane])), "l"(qrow + 16 * c), "r"(on ? 8u : 0u) : "memory");
                } else {
                    qb[n][c] = make_uint2(0u, 0u);
                    if (on) qb[n][c] = ld_global(reinterpret_cast<const uint2*>(qrow + 16 * c));
                }
                o[n][c][0] = o[n][c][1] = o[n][c][2] = o[n][c][3] = 0.0f;
            }
            m_run[n][0] = m_run[n][1] = NEG_SENTINEL;
            l_part[n][0] = l_part[n][1] = 0.0f;
        }
        len = (int)rq.len;
        pos0 = len - (int)rq.n;
        lo_all = max(len - window, 0);
        lo_any = max(pos0 + 1 - window, 0);
    };
    auto end_request = [&](uint32_t tile_last) {
        const bool began = tile_first == tile_begin, ended = tile_last + 1 == tile_end;
#pragma unroll
        for (int n = 0; n < NB; n++) {
            if (NB > 1 && 8 * (uint32_t)n >= rows) break;
            const float l_row[2] = {tok_sum(l_part[n][0]), tok_sum(l_part[n][1])};
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t row = 8 * n + 2 * t4 + e;
                if (row >= rows) continue;
                if (began && ended) {
                    const bool saw = l_row[e] != 0.0f;  // a row that saw nothing is 0, whatever stands in V
                    const float f = 1.0f / l_row[e];
                    __half* dst = a.out + ((size_t)(first_tok + (row >> a.group_shift)) * heads + head * a.group + (row & (a.group - 1))) * HD + 2 * g;
#pragma unroll
                    for (int c = 0; c < 8; c++)
                        *reinterpret_cast<__half2*>(dst + 16 * c) = saw ? __floats2half2_rn(o[n][c][e] * f, o[n][c][2 + e] * f) : __float2half2_rn(0.0f);
                } else {
                    const size_t at = ((size_t)(2 * part + (began ? 1 : 0)) * a.n_kv + head) * work.rows + row;
                    float* dst = reinterpret_cast<float*>(work.acc + at * (HD / 4)) + 2 * g;
#pragma unroll
                    for (int c = 0; c < 8; c++) *reinterpret_cast<float2*>(dst + 16 * c) = make_float2(o[n][c][e], o[n][c][2 + e]);
                    if (g == 0) work.ml[at] = make_float2(m_run[n][e], l_row[e]);
                }
            }
        }
    };

    // Shared-memory offsets of a tile [16 tokens][128 B, swizzled]: one ldmatrix.x4 fetches 32 bytes of 16 tokens; lane l addresses row
    // (l & 7) of matrix (l >> 3) = (token half (l >> 3) & 1, 16-byte chunk 2b + (l >> 4)).
    const uint32_t lrow = lane & 7, lmat = lane >> 3;
    uint32_t off[4];
#pragma unroll
    for (int b = 0; b < 4; b++) off[b] = (8 * (lmat & 1) + lrow) * 128 + (((2 * b + (lmat >> 1)) ^ lrow) << 4);
    const float scale2 = a.scale * 1.4426950408889634f;
    bool failed = false;
    uint32_t tile_now = tile0;
    begin_request(0, tile0);  // its queries are on their way while the first pages are
#pragma unroll
    for (int i = 0; i < STAGES; i++) {
        way_r[i] = way_tile[i] = 0;
        way_exp[i] = 0;
        if ((uint32_t)i < n_iter) {
            if (i > 0) next_tile();
            if ((uint32_t)i < left0) to_page = __shfl_sync(0xffffffffu, first_pages, i); else look();
            way_r[i] = to_nth;
            way_tile[i] = to_tile;
            issue(i, way_exp[i]);
        }
    }
    if (STAGES < n_iter) {
        next_tile();
        look();
    }

    for (uint32_t it = 0; it < n_iter; ++it) {
        const uint32_t st = it % STAGES;
        if (way_r[0] != r_now) {
            end_request(tile_now);
            begin_request(way_r[0], way_tile[0]);
        }
        tile_now = way_tile[0];
        const int ek = __shfl_sync(0xffffffffu, way_exp[0], 0), ev = __shfl_sync(0xffffffffu, way_exp[0], 1);
        mbar_wait_warp(&sm.full[warp][st], (it / STAGES) & 1, a.req.status, 631, failed);
        if (failed) break;
        const int tok0 = (int)(tile_now * TILE_TOK);
        const uint32_t k_base = smem_u32(sm.k[warp][st]), v_base = smem_u32(sm.v[warp][st]);

        if (Q_SHARED) asm volatile("cp.async.wait_all;" ::: "memory");  // (of a lane's own queries)
        // S: s[n][2 th + e] = score of token g + 8 th against row 8 n + 2 t4 + e, of one block in two chains of four products
        float s[NB][4] = {}, s1[4] = {};
#pragma unroll
        for (int b = 0; b < 4; b++) {
            uint32_t x[4];
            ldsm_x4(k_base + off[b], x);
#pragma unroll
            for (int cc = 0; cc < 2; cc++) {
                const uint32_t f[4] = {e4m3x2_to_f16x2(x[2 * cc] & 0xffffu), e4m3x2_to_f16x2(x[2 * cc + 1] & 0xffffu), e4m3x2_to_f16x2(x[2 * cc] >> 16),
                                       e4m3x2_to_f16x2(x[2 * cc + 1] >> 16)};
#pragma unroll
                for (int n = 0; n < NB; n++) {
                    const uint2 q = Q_SHARED ? sm.q[Q_SHARED ? warp : 0][Q_SHARED ? 8 * n + 2 * b + cc : 0][lane] : qb[Q_SHARED ? 0 : n][2 * b + cc];
                    mma16816(NB == 1 && cc ? s1 : s[n], f, q.x, q.y);
                }
            }
        }
        const float ks = scale2 * __int_as_float((127 + ek) << 23), shift = (float)ev;
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[n][i] = fmaf(NB == 1 ? s[n][i] + s1[i] : s[n][i], ks, shift);
        if (tok0 < lo_all || tok0 + TILE_TOK - 1 > pos0) {
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = tok0 + (int)g + 8 * (i / 2), hi = min(pos0 + (int)((8 * n + 2 * t4 + i % 2) >> a.group_shift), len - 1);
                    if (t < max(hi + 1 - window, 0) || t > hi) s[n][i] = -INFINITY;
                }
        }
        bool grows = false;  // any row: a lane looks at its own scores, the rows' maxima are found only where one counts
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) grows |= fmaxf(s[n][e], s[n][2 + e]) > m_run[n][e] + GROWTH_T;
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float mx = tok_max(fmaxf(s[n][e], s[n][2 + e])), m = mx > m_run[n][e] + GROWTH_T ? mx - LIFT : m_run[n][e], corr = ex2(m_run[n][e] - m);
                    m_run[n][e] = m;
                    l_part[n][e] *= corr;
#pragma unroll
                    for (int c = 0; c < 8; c++) {
                        o[n][c][e] *= corr;
                        o[n][c][2 + e] *= corr;
                    }
                }
        }
        const float back = __int_as_float((127 - ev) << 23);
        uint32_t pt[NB][2];
#pragma unroll
        for (int n = 0; n < NB; n++) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) p[i] = ex2(s[n][i] - m_run[n][i % 2]);
            l_part[n][0] = fmaf(p[0] + p[2], back, l_part[n][0]);
            l_part[n][1] = fmaf(p[1] + p[3], back, l_part[n][1]);
            // P (tokens x rows) -> P^T fragments: lane (g, t4) gets row g, tokens 2 t4, 2 t4 + 1 and 8 + those
            pt[n][0] = movmatrix_trans(pack_half2(p[0], p[1]));
            pt[n][1] = movmatrix_trans(pack_half2(p[2], p[3]));
        }
        // Tokens that no row sees have P = 0, but 0 times a NaN that stands there would not be: they count as 0.
        // So do NaNs in tokens that some rows see and others not: the merge puts those into the rows that see them.
        if (tok0 < lo_all || tok0 + TILE_TOK - 1 > pos0) {
#pragma unroll 1
            for (int t = 0; t < TILE_TOK; t++)
                if (tok0 + t < lo_any || tok0 + t >= len) asm volatile("st.shared.u32 [%0], %1;" ::"r"(v_base + t * 128 + lane * 4), "r"(0) : "memory");
            if (DRAFTS && rows > a.group) {
                __syncwarp();
#pragma unroll 1
                for (int t = 0; t < TILE_TOK; t += 4) {
                    const uint32_t v_at = v_base + t * 128 + lane * 16;
                    uint4 v;
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(v_at) : "memory");
                    if (drop_nans(v)) asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(v_at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
                }
            }
            fence_proxy_async_smem();  // the slot's next copy comes behind these
            __syncwarp();
        }
#pragma unroll
        for (int b = 0; b < 4; b++) {
            uint32_t y[4];  // transposed: bytes V[8 th + 2 t4 (+1)][16c + 2g (+1)] for (th, c) = (0, 2b), (1, 2b), (0, 2b + 1), (1, 2b + 1)
            ldsm_x4_trans(v_base + off[b], y);
#pragma unroll
            for (int cc = 0; cc < 2; cc++) {
                const uint32_t y0 = __byte_perm(y[2 * cc], 0u, 0x3120), y1 = __byte_perm(y[2 * cc + 1], 0u, 0x3120);
                const uint32_t f[4] = {e4m3x2_to_f16x2(y0 & 0xffffu), e4m3x2_to_f16x2(y0 >> 16), e4m3x2_to_f16x2(y1 & 0xffffu), e4m3x2_to_f16x2(y1 >> 16)};
#pragma unroll
                for (int n = 0; n < NB; n++) mma16816(o[n][2 * b + cc], f, pt[n][0], pt[n][1]);
            }
        }
        __syncwarp();  // every lane is done with the slot
#pragma unroll
        for (int i = 0; i + 1 < STAGES; i++) {
            way_r[i] = way_r[i + 1];
            way_tile[i] = way_tile[i + 1];
            way_exp[i] = way_exp[i + 1];
        }
        if (it + STAGES < n_iter) {
            way_r[STAGES - 1] = to_nth;
            way_tile[STAGES - 1] = to_tile;
            issue(st, way_exp[STAGES - 1]);
            if (it + STAGES + 1 < n_iter) {  // its page is looked up while a tile is worked on
                next_tile();
                look();
            }
        }
    }
    if (failed) let_copies_land();
    end_request(tile_now);
}

constexpr uint32_t LISTED = 1024;  // requests whose first units the listing CTA keeps at hand
constexpr int MANY_CTAS_WARPS = 4;                                          // of the merge
constexpr int FEW_CTAS_WARPS = 16;

// What the prefill kernel takes its items from; by one CTA of the merge.  Units go out with the most keys first, so that what is left at
// the end is short (24 requests, three of them prompts of 841 to 1281 tokens: 110 us in the requests' order).  All heads of a unit
// follow each other while the keys and values of all prompts stay in about three quarters of the 126 MB L2; else a head's units do.
template <int MERGE_WARPS>
__device__ __forceinline__ void list_units(const BlocksAttn& a, const BlocksWork& w, uint32_t* shared)
{
    constexpr uint32_t N = MERGE_WARPS * 32;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // Exclusive prefix sum over the CTA.
    auto scan = [&](uint32_t mine, uint32_t& total) {
        uint32_t up_to = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, up_to, off);
            if (lane >= (uint32_t)off) up_to += t;
        }
        __syncthreads();
        uint32_t* sums = shared + MOST_SORTED + LISTED;
        if (lane == 31) sums[warp] = up_to;
        __syncthreads();
        uint32_t at = up_to - mine;
        total = 0;
#pragma unroll
        for (int i = 0; i < MERGE_WARPS; i++) {
            if (i < (int)warp) at += sums[i];
            total += sums[i];
        }
        return at;
    };
    const uint32_t per_thread = (a.req.n + N - 1) / N, r_begin = min(tid * per_thread, a.req.n), r_end = min(r_begin + per_thread, a.req.n);
    const auto units = [&](const Request& q) -> uint32_t { return q.n > a.few ? (uint32_t)(((uint64_t)q.n * a.group + UNIT_ROWS - 1) / UNIT_ROWS) : 0; };
    uint32_t mine = 0, kilokeys = 0, total, all_kilokeys;
    for_requests(a.req, r_begin, r_end, [&](uint32_t, const Request& q) {
        const uint32_t n = units(q);
        mine += n;
        if (n) kilokeys = min(kilokeys + q.len / 1024, 1u << 22);  // (no more than that it is much)
    });
    uint32_t at = scan(mine, total);
    scan(kilokeys, all_kilokeys);
    // At hand where the requests fit: what a unit's request is looked up in.
    uint32_t* firsts = shared + MOST_SORTED;
    const bool at_hand = a.req.n <= LISTED;
    const auto note = [&](uint32_t r, uint32_t n) {
        if (at_hand) firsts[r] = at;
        w.units_before[r] = at;
        at += n;
    };
    if (per_thread == 1) {
        if (r_begin < r_end) note(r_begin, mine);
    } else {
        for_requests(a.req, r_begin, r_end, [&](uint32_t r, const Request& q) { note(r, units(q)); });
    }
    const bool by_head = (uint64_t)all_kilokeys * 1024 * a.n_kv * 2 * HD > ((uint64_t)96 << 20);
    if (tid == 0) {
        w.units_before[a.req.n] = total;
        *w.queue = 0;
        *w.by_head = by_head;
    }
    for (uint32_t i = tid; i < 2 * w.places; i += N) w.done[i] = 0;
    __syncthreads();
    // The request of a unit, the last one with units_before <= u, and its number there.
    const auto locate = [&](uint32_t u) -> uint2 {
        uint32_t lo = 0, hi = a.req.n;
        const auto before = [&](uint32_t r) { return at_hand ? firsts[r] : ld_global(w.units_before + r); };
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (before(mid) <= u) lo = mid; else hi = mid;
        }
        return make_uint2(lo, u - before(lo));
    };
    const bool sorted = total <= MOST_SORTED;
    if (sorted) {  // bitonic, by tiles of keys and then by number: the same order every time
        uint32_t n = 1;
        while (n < total) n <<= 1;
        for (uint32_t u = tid; u < n; u += N) {
            const uint2 at = u < total ? locate(u) : make_uint2(0, 0);
            shared[u] = u < total ? (min((uint32_t)unit_at(a, at.x, at.y).n_tiles, (1u << 20) - 1) + 1) << 11 | u : 0;
        }
        for (uint32_t k = 2; k <= n; k <<= 1)
            for (uint32_t j = k >> 1; j > 0; j >>= 1) {
                __syncthreads();
                for (uint32_t i = tid; i < n; i += N) {
                    const uint32_t x = i ^ j;
                    if (x > i) {
                        const uint32_t p = shared[i], q = shared[x];
                        if (((i & k) == 0) == (p < q)) shared[i] = q, shared[x] = p;
                    }
                }
            }
        __syncthreads();
        for (uint32_t i = tid; i < total; i += N) w.order[i] = locate(shared[i] & (MOST_SORTED - 1));
    }
    const uint32_t items = total * a.n_kv, whole = whole_items(items, w.places);
    uint32_t all_tiles = 0;
    for (uint32_t base = 0; base < w.places; base += N) {  // fewer than places are left
        uint32_t tiles = 0, more;
        if (whole + base + tid < items) {
            uint32_t head, rank, u;
            split_item(whole + base + tid, total, a.n_kv, by_head, head, rank);
            u = total - 1 - rank;
            if (sorted) u = shared[rank] & (MOST_SORTED - 1), tiles = (shared[rank] >> 11) - 1;
            if (!sorted || tiles == (1u << 20) - 1) {
                const uint2 at = locate(u);
                tiles = (uint32_t)unit_at(a, at.x, at.y).n_tiles;
            }
            tiles = max(tiles, 1u);  // one without a key counts for its rows
        }
        const uint32_t before = all_tiles + scan(tiles, more);
        if (base + tid < w.places) w.rest[base + tid] = before;
        all_tiles += more;
    }
    if (tid == 0) w.rest[w.places] = all_tiles;
}

// One CTA per request, kv head and eight rows: nothing to do where one warp had all its tiles; zeros where it had none; else the warps' parts.
// Warp x of W takes parts x, x + W, ...  Row and part are spread over its lanes for (m, l), and over the E sums of four dims that a lane keeps
// for O, so that few rows go through several parts at a time; maxima and sums of the warps meet in shared memory, in a fixed order.
// SHIFT: rows up to this power of two in all requests, or -1: each request's own (a dispatch that has prompts as well knows no more than eight).
// DRAFTS: a request may have more than one token.
template <int E, int W, int SHIFT, bool DRAFTS>
__global__ void __launch_bounds__(W * 32, W == MANY_CTAS_WARPS ? (E == 8 ? 4 : 8) : SHIFT < 0 ? 2 : 1) blocks_merge_kernel(const __grid_constant__ BlocksAttn a, const __grid_constant__ Work work)
{
    constexpr int LEFT = SHIFT >= 0 ? 1 << SHIFT : E;  // sums that a lane leaves: one a row, where the rows are known beforehand
    __shared__ union {
        struct {
            float4 acc[W][LEFT][32];
            float big[W][8], den[W][8];
        } of;
        uint32_t sort[MOST_SORTED + LISTED + W];
    } sm;
    pdl_wait();
    pdl_launch_dependents();
    if (blockIdx.x == a.req.n) {  // there if a prefill follows
        if (blockIdx.y + blockIdx.z == 0) list_units<W>(a, work.head, sm.sort);
        return;
    }
    const uint32_t r = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t at = ld_global(work.head.before + r), end = ld_global(work.head.before + r + 1), total = ld_global(work.head.before + a.req.n);
    const uint32_t most = (uint32_t)ld_global(work.head.before + a.req.n + 1);
    const uint32_t first = ld_global(a.req.starts + r), last = ld_global(a.req.starts + r + 1);
    uint32_t p0 = 0, n = 0;
    if (end > at) {
        const Stretches cut = stretches_for(total, most);
        p0 = cut.of(at + REQUEST_WEIGHT);
        n = cut.of(end - 1) - p0 + 1;
        if (n == 1 && (!DRAFTS || last - first == 1)) return;
    }
    if (last <= first || last > a.req.tokens || last - first > a.few || last - first > a.req.max_q) return;
    const uint32_t row0 = SHIFT < 0 ? 8 * blockIdx.z : 0, all_rows = (last - first) * a.group;
    if (SHIFT < 0 && row0 >= all_rows) return;
    const uint32_t rows = SHIFT < 0 ? min(all_rows - row0, 8u) : all_rows;  // of this CTA
    const auto out = [&](uint32_t row) {
        row += row0;
        return reinterpret_cast<uint2*>(a.out + ((size_t)(first + (row >> a.group_shift)) * (a.n_kv * a.group) + head * a.group + (row & (a.group - 1))) * HD + 4 * lane);
    };
    if (n == 0) {
        for (uint32_t row = warp; row < rows; row += W) *out(row) = make_uint2(0u, 0u);
        return;
    }
    // NaNs of V that some of the request's rows see and others not, which the decode took for 0: into the rows that see them, in their dims.
    const auto put_nans = [&]() {
        const Request rq = request_at(a.req, r);
        const Tiles tiles = tiles_of(a, rq);
        const int len = (int)rq.len, pos0 = len - (int)rq.n, window = a.req.window && a.req.window < MOST_KEYS ? (int)a.req.window : (int)MOST_KEYS;
        // such are in the first tiles, up to the key from which on the last row sees all, and in those of the new tokens; one a warp at a time
        const uint32_t to = tiles.lo + tiles.n, mid = min((uint32_t)(max(len - window, 0) + TILE_TOK - 1) / TILE_TOK, to), passed = mid > tiles.lo ? mid - tiles.lo : 0;
        const uint32_t from = max((uint32_t)max(pos0 + 1, 0) / TILE_TOK, tiles.lo + passed);
        for (uint32_t i = warp; i < passed + (to - from); i += W) {
            const uint32_t tile = i < passed ? tiles.lo + i : from + (i - passed);
            const size_t block = block_of_page(a.req, r, tile, ld_global(page_at(a.req, r, tile)));
            const uint8_t* v = a.pool[1] + (block * a.n_kv + head) * TILE_BYTES + lane * 16;
            uint32_t nans = 0;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const uint4 y = ld_global(reinterpret_cast<const uint4*>(v + 512 * x));
                nans |= nan_bytes(y.x) | nan_bytes(y.y) | nan_bytes(y.z) | nan_bytes(y.w);
            }
            if (nans == 0) continue;
#pragma unroll 1
            for (uint32_t x = 0; x < 64; x++) {  // byte by byte: token 4 (x / 16) + lane / 8, dim 16 (lane % 8) + x % 16
                const int t = (int)(tile * TILE_TOK + 4 * (x / 16) + lane / 8);
                if ((*(const volatile uint8_t*)(v + 512 * (x / 16) + x % 16) & 0x7f) != 0x7f) continue;
#pragma unroll 1
                for (uint32_t row = 0; row < rows; row++) {
                    const int pos = pos0 + (int)((row0 + row) >> a.group_shift);
                    if (t <= pos && t > pos - window) *(reinterpret_cast<__half*>(out(row) - lane) + 16 * (lane % 8) + x % 16) = __ushort_as_half(0x7fff);
                }
            }
        }
    };
    if (DRAFTS && n == 1) {
        put_nans();
        return;
    }
    const uint32_t shift = SHIFT >= 0 ? SHIFT : rows <= 1 ? 0 : rows <= 2 ? 1 : rows <= 4 ? 2 : 3, mask = (1u << shift) - 1;  // rows up to a power of two
    const auto slot = [&](uint32_t j) { return ((size_t)(2 * (p0 + j) + (j == 0 ? 1 : 0)) * a.n_kv + head) * work.rows + row0; };
    const uint32_t batch = E >> shift, chunk = 32 >> shift;  // parts that a lane's sums go through at a time, parts whose (m, l) the lanes hold
    float4 v[E], acc[E];
    const auto fetch = [&](uint32_t k) {  // this warp's parts k ..
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = ld_global(work.acc + (slot(min(warp + (k + (e >> shift)) * W, n - 1)) + min(e & mask, rows - 1)) * (HD / 4) + lane);
    };
    const auto fetch_ml = [&](uint32_t k) { return ld_global(work.ml + slot(min(warp + (k + (lane >> shift)) * W, n - 1)) + min(lane & mask, rows - 1)); };
    float2 ml = fetch_ml(0);  // (parts past the end are the last one again)
    fetch(0);
    float big = ml.x, den = 0.0f;
    for (uint32_t k = chunk; warp + k * W < n; k += chunk) big = fmaxf(big, fetch_ml(k).x);
#pragma unroll
    for (uint32_t off = 16; off; off >>= 1)
        if (off > mask) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
    if (lane <= mask) sm.of.big[warp][lane] = big;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < W; x++) big = fmaxf(big, sm.of.big[x][lane & mask]);
#pragma unroll
    for (int e = 0; e < E; e++) acc[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t k0 = 0; warp + k0 * W < n; k0 += chunk) {
        if (k0) ml = fetch_ml(k0), fetch(k0);
        const float w = warp + (k0 + (lane >> shift)) * W < n ? ex2(ml.x - big) : 0.0f;
        den = fmaf(w, ml.y, den);
        for (uint32_t k = 0;; k += batch) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float f = __shfl_sync(0xffffffffu, w, ((k + (e >> shift)) << shift) + (e & mask));  // 0 past the end
                acc[e].x = fmaf(f, v[e].x, acc[e].x);
                acc[e].y = fmaf(f, v[e].y, acc[e].y);
                acc[e].z = fmaf(f, v[e].z, acc[e].z);
                acc[e].w = fmaf(f, v[e].w, acc[e].w);
            }
            if (k + batch >= chunk || warp + (k0 + k + batch) * W >= n) break;
            fetch(k0 + k + batch);
        }
    }
#pragma unroll
    for (uint32_t off = 16; off; off >>= 1)
        if (off > mask) den += __shfl_xor_sync(0xffffffffu, den, off);
    if (lane <= mask) sm.of.den[warp][lane] = den;
#pragma unroll
    for (int e = LEFT; e < E; e++) {
        float4& to = acc[e % LEFT];
        to.x += acc[e].x;
        to.y += acc[e].y;
        to.z += acc[e].z;
        to.w += acc[e].w;
    }
#pragma unroll
    for (int e = 0; e < LEFT; e++) sm.of.acc[warp][e][lane] = acc[e];
    __syncthreads();
    for (uint32_t row = warp; row < rows; row += W) {
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float l = 0.0f;
        for (int x = 0; x < W; x++) {
            l += sm.of.den[x][row];
            for (uint32_t e = row; e < LEFT; e += mask + 1) {
                const float4 o = sm.of.acc[x][e][lane];
                sum.x += o.x;
                sum.y += o.y;
                sum.z += o.z;
                sum.w += o.w;
            }
        }
        const float f = 1.0f / l;  // a row that saw nothing is 0, whatever stands in V
        *out(row) = l != 0.0f ? make_uint2(pack_half2(sum.x * f, sum.y * f), pack_half2(sum.z * f, sum.w * f)) : make_uint2(0u, 0u);
    }
    if (DRAFTS && last - first > 1) {
        __syncthreads();  // other warps wrote some of the rows
        put_nans();
    }
}

// Warps that fit the GPU at once, and what every kv head gets of them.
uint32_t grid_ctas(int sm_count, uint32_t n_kv, int ctas_per_sm)
{
    const uint32_t ctas = (uint32_t)(sm_count * ctas_per_sm), least = (n_kv + WARPS - 1) / WARPS;
    return ctas > least ? ctas : least;
}

template <int NB, bool DRAFTS>
int launch_decode(const LaunchArgs& a, const BlocksAttn& k, const CUtensorMap (&tm)[2], const Work& w, uint32_t ctas, uint32_t most)
{
    const size_t smem = sizeof(DecodeSmem<NB>) + 1024;
    static_assert((sizeof(DecodeSmem<NB>) + 2048) * Shape<NB>::CTAS_PER_SM <= 228 * 1024, "shared memory of an SM");
    {
        static std::mutex attr_mutex;
        static bool attr_set[64] = {};
        std::lock_guard<std::mutex> lock(attr_mutex);
        if (a.device < 0 || a.device >= 64 || !attr_set[a.device]) {
            if (int r = check_cuda(a, cudaFuncSetAttribute(blocks_decode_kernel<NB, DRAFTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                                   "cudaFuncSetAttribute(blocks_decode)"))
                return r;
            if (a.device >= 0 && a.device < 64) attr_set[a.device] = true;
        }
    }
    const cudaError_t e = launch_dependent(blocks_decode_kernel<NB, DRAFTS>, dim3(ctas), dim3(WARPS * 32), smem, a.stream, tm[0], tm[1], k, w, most);
    ++*a.launches;
    return check_cuda(a, e, "attn_blocks decode");
}
int ctas_per_sm(uint32_t most_rows) { return most_rows <= 8 ? Shape<1>::CTAS_PER_SM : Shape<2>::CTAS_PER_SM; }

}  // namespace

// (no less for fewer heads, nor for more query tokens of a request)
size_t blocks_decode_work(int sm_count, uint32_t n_kv, uint32_t group, uint32_t max_q)
{
    size_t parts = 0;
    for (uint32_t rows = 8; rows <= FEW_ROWS; rows *= 2) {
        if (rows > 8 && (uint64_t)group * max_q <= rows / 2) break;
        const size_t n = 2ull * grid_ctas(sm_count, n_kv, ctas_per_sm(rows)) * WARPS * part_rows(rows, group, max_q);
        parts = n > parts ? n : parts;
    }
    return parts * (HD + 2) * 4;
}

int launch_blocks_decode(const LaunchArgs& a, const BlocksAttn& k, const BlocksWork& head)
{
    CUtensorMap tm[2];
    for (int i = 0; i < 2; i++) {
        const uint64_t dims[3] = {128, TILE_TOK, k.tiles}, strides[2] = {128, TILE_BYTES};
        const uint32_t box[3] = {128, TILE_TOK, 1};
        if (int r = encode_tensor_map(a, &tm[i], 0, 3, const_cast<uint8_t*>(k.pool[i]), dims, strides, box, 3)) return r;
    }
    const uint32_t most_rows = k.few * k.group, ctas = grid_ctas(a.sm_count, k.n_kv, ctas_per_sm(most_rows)), most = ctas * WARPS / k.n_kv;
    Work w{head, nullptr, reinterpret_cast<float4*>(head.parts), part_rows(most_rows, k.group, k.req.max_q)};
    w.ml = reinterpret_cast<float2*>(w.acc + 2ull * most * k.n_kv * w.rows * (HD / 4));
    const bool drafts = k.req.max_q > 1;
    if (int r = most_rows > 8 ? launch_decode<2, true>(a, k, tm, w, ctas, most) : drafts ? launch_decode<1, true>(a, k, tm, w, ctas, most) : launch_decode<1, false>(a, k, tm, w, ctas, most))
        return r;
    // Few CTAs have many parts each (one request of 131072 keys: 148 of every head; 9.4 us with four warps a CTA).
    const uint32_t row_blocks = (w.rows + 7) / 8;
    const bool few = (uint64_t)k.req.n * k.n_kv * row_blocks <= 2u * (uint32_t)a.sm_count;
    const dim3 grid(k.req.n + (k.req.max_q > k.few ? 1 : 0), k.n_kv, row_blocks);
    const auto merge_of = [&](auto shift, auto with_drafts) {
        constexpr int SHIFT = decltype(shift)::value, WARPS_IF_FEW = SHIFT < 0 ? FEW_CTAS_WARPS / 2 : FEW_CTAS_WARPS;
        constexpr bool DRAFTS = decltype(with_drafts)::value;
        return few ? launch_dependent(blocks_merge_kernel<8, WARPS_IF_FEW, SHIFT, DRAFTS>, grid, dim3(WARPS_IF_FEW * 32), 0, a.stream, k, w)
                   : launch_dependent(blocks_merge_kernel<SHIFT < 0 ? 8 : 4, MANY_CTAS_WARPS, SHIFT, DRAFTS>, grid, dim3(MANY_CTAS_WARPS * 32), 0, a.stream, k, w);
    };
    const auto merge = [&](auto shift) { return drafts ? merge_of(shift, std::true_type()) : merge_of(shift, std::false_type()); };
    const cudaError_t e = w.rows <= 1 ? merge(std::integral_constant<int, 0>()) : w.rows <= 2 ? merge(std::integral_constant<int, 1>())
        : w.rows <= 4 ? merge(std::integral_constant<int, 2>()) : merge(std::integral_constant<int, -1>());
    ++*a.launches;
    return check_cuda(a, e, "attn_blocks merge");
}

}  // namespace sgb
