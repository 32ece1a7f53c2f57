// A serving step's bookkeeping and its writes into the 8-bit cache of blocks.cuh.
//
// kv_block_tables: from the lengths of all requests, which pages each keeps, gives back and takes, and where every new token goes.
// kv_append_blocks_e4m3_d128: new keys and values into their slots, with one power of two per tile of 16 tokens and head.
#include "blocks.cuh"
#include "sgb_kernels.h"

namespace sgb {

namespace {

// ---- block tables and slot maps ------------------------------------------------------------------------------------------------
// need_r = ceil((ctx_r + new_r) / page).  A request takes part if need_r <= stride and its tokens end within the step's `tokens`.
// Pages beyond need_r go to the end of the free list, in the order of requests and pages; then pages are taken from the list's
// end, in the same order, by every request whose wants the list still covers when all before it are counted.  The others are
// refused: they keep what they hold, their length is 0 and their tokens have no slot.
//
// Prefix sums over the requests and little else: bound by its own latency.  One CTA does the sums, of up to 1024 requests at a time, and
// moves the pages; it places the tokens too while there are few of them.  64 requests of one token take 4.1 us, 1024 of which an
// eighth ends and an eighth begins 12, 4000 with prompts 24 (one after the other in a stream).
constexpr uint32_t PLAN_THREADS = 1024, PLAN_WARPS = PLAN_THREADS / 32;
constexpr uint32_t PLACE_THREADS = 256;
constexpr uint32_t MOST_STRIDE = 1u << 21;
constexpr uint32_t SEARCHED = 4096;      // requests whose first tokens a CTA keeps at hand (16 KB)
constexpr uint32_t PLACED_HERE = 4096;   // tokens that the first CTA places itself (64 requests of one token: 8.2 us with a second kernel)

struct PlanArgs {
    const uint32_t *ctx, *add, *held, *count;
    uint32_t *free_list, *table, *held_out, *free_out, *starts, *lens, *slots, *at;
    uint32_t n, tokens, page_shift, stride, capacity;
    uint32_t* status;
};

// Exclusive prefix sums of N values over the CTA; `total` is everybody's.
template <int N>
__device__ __forceinline__ void block_scan(uint64_t (&v)[N], uint64_t (*warp_sums)[N], uint64_t (&total)[N])
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32;
    uint64_t x[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = v[i];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, x[i], off);
            if (lane >= (uint32_t)off) x[i] += t;
        }
    }
    __syncthreads();  // the last use of warp_sums is over
    if (lane == 31) {
#pragma unroll
        for (int i = 0; i < N; i++) warp_sums[warp][i] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint64_t mine = lane < warps ? warp_sums[lane][i] : 0;
        uint64_t s = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, s, off);
            if (lane >= (uint32_t)off) s += t;
        }
        total[i] = __shfl_sync(0xffffffffu, s, 31);
        v[i] = __shfl_sync(0xffffffffu, s - mine, warp) + x[i] - v[i];
    }
}

// Slot and position of token t of the step; `starts` is the requests' first tokens, at hand or in memory.
template <typename First>
__device__ __forceinline__ void place_token(const PlanArgs& a, uint32_t t, const First& starts)
{
    uint32_t lo = 0, hi = a.n;  // the request whose tokens t is among: the last one with starts <= t
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (starts(mid) <= t) lo = mid; else hi = mid;
    }
    uint32_t slot = NO_SLOT, pos = 0;
    if (t < starts(a.n)) {
        const uint32_t ctx = ld_global(a.ctx + lo), len = ld_global(a.lens + lo);
        pos = ctx + (t - starts(lo));
        if (len != 0) {
            const uint64_t row = ((uint64_t)ld_global(a.table + (size_t)lo * a.stride + (pos >> a.page_shift)) << a.page_shift) +
                                 (pos & ((1u << a.page_shift) - 1));
            if (row < NO_SLOT) slot = (uint32_t)row;
        }
    }
    a.slots[t] = slot;
    a.at[t] = pos;
}

// Moves of up to PLAN_THREADS requests: request r's words [0, n_r) by whichever thread comes to them, four of each on their way at a time.
// (A request's pages by one warp: a prompt of 32768 tokens in pages of 16 took 6 us of its own.)
struct Moves {
    uint32_t before[PLAN_THREADS + 1];  // words of the requests before each
    uint32_t first[PLAN_THREADS];       // where its words start in its row
};
template <typename From, typename To>
__device__ __forceinline__ void move_words(const Moves& mv, uint32_t requests, const From& from, const To& to)
{
    const uint32_t total = mv.before[requests];
    for (uint32_t j0 = threadIdx.x; j0 < total; j0 += 4 * blockDim.x) {
        uint32_t w[4], r[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            const uint32_t j = j0 + k * blockDim.x;
            uint32_t lo = 0, hi = requests;  // the last request with before <= j
            while (j < total && hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (mv.before[mid] <= j) lo = mid; else hi = mid;
            }
            r[k] = lo;
            w[k] = ld_global_if(j < total, from(lo, j - mv.before[lo], j));
        }
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            const uint32_t j = j0 + k * blockDim.x;
            if (j < total) to(r[k], j - mv.before[r[k]], j, w[k]);
        }
    }
}

// KEPT: all requests fit four rounds of the CTA's threads; what has been looked at stays in registers for the second pass.
constexpr uint32_t KEPT_ROUNDS = 4;
template <bool KEPT>
__global__ void __launch_bounds__(PLAN_THREADS) block_tables_kernel(const __grid_constant__ PlanArgs a, bool place_here)
{
    __shared__ uint64_t sums[PLAN_WARPS][1];
    __shared__ union {
        Moves moves;
        uint32_t firsts[SEARCHED + 1];
    } sm;
    __shared__ unsigned long long counted[3];  // pages taken, requests refused, tokens placed
    const uint32_t threads = blockDim.x;
    if (threadIdx.x < 3) counted[threadIdx.x] = 0;
    pdl_wait();
    pdl_launch_dependents();
    uint32_t count = ld_global(a.count);
    struct Mine {
        uint32_t held, add, ctx, need;
        bool fits;
        __device__ uint32_t back() const { return fits && held > need ? held - need : 0; }
        __device__ uint32_t want() const { return fits && need > held ? need - held : 0; }
    };
    auto load = [&](uint32_t r) {
        Mine m{0, 0, 0, 0, false};
        m.add = ld_global_if(r < a.n, a.add + r);
        m.ctx = ld_global_if(r < a.n, a.ctx + r);
        m.held = ld_global_if(r < a.n, a.held + r);
        return m;
    };
    // Where the request's tokens end, whether it takes part, how many pages it needs.
    auto look = [&](Mine& m, uint32_t r, uint64_t& carry) -> uint64_t {
        if (m.held > a.stride) {
            report_error(a.status, DEV_ERR_BOUNDS, 612, r, m.held);
            m.held = a.stride;
        }
        const uint64_t len = (uint64_t)m.ctx + m.add, need = (len + (1u << a.page_shift) - 1) >> a.page_shift;
        uint64_t before[1] = {m.add}, total[1];
        block_scan<1>(before, sums, total);
        const uint64_t end = carry + before[0] + m.add;
        carry += total[0];
        m.fits = r < a.n && need <= a.stride && end <= a.tokens && len < NO_SLOT;
        m.need = m.fits ? (uint32_t)need : 0;
        return end;
    };
    constexpr uint32_t ROUNDS = KEPT ? KEPT_ROUNDS : 1;
    Mine kept[ROUNDS];
    uint32_t kept_first[ROUNDS];
    uint64_t kept_before[ROUNDS], kept_total[ROUNDS];
    if (KEPT) {
#pragma unroll
        for (uint32_t k = 0; k < ROUNDS; k++) kept[k] = load(k * threads + threadIdx.x);
    }
    if (count > a.capacity) {
        if (threadIdx.x == 0) report_error(a.status, DEV_ERR_BOUNDS, 611, count, a.capacity);
        count = a.capacity;
    }

    // Pages given back, and where every request's tokens start.
    uint64_t ends = 0, given = 0;
    // Pages back (low half) and wanted (high half) before a request and of all of the round: 1024 rows of at most MOST_STRIDE fit a word.
    auto sum_up = [&](const Mine& m, uint64_t& total) -> uint64_t {
        uint64_t before[1] = {(uint64_t)m.want() << 32 | m.back()}, all[1];
        block_scan<1>(before, sums, all);
        total = all[0];
        return before[0];
    };
    auto first_pass = [&](Mine& m, uint32_t base, uint64_t& before, uint64_t& total) -> uint32_t {
        const uint32_t r = base + threadIdx.x;
        const uint32_t first = (uint32_t)min(look(m, r, ends), (uint64_t)a.tokens);
        before = sum_up(m, total);
        const uint32_t back_total = (uint32_t)total;
        if (r < a.n) {
            a.starts[r + 1] = first;
            if (r == 0) a.starts[0] = 0;
        }
        if (back_total != 0) {
            sm.moves.before[threadIdx.x] = (uint32_t)before;
            sm.moves.first[threadIdx.x] = m.need;
            if (threadIdx.x == 0) sm.moves.before[threads] = back_total;
            __syncthreads();
            const uint64_t to = count + given;
            move_words(sm.moves, threads, [&](uint32_t q, uint32_t j, uint32_t) { return a.table + (size_t)(base + q) * a.stride + sm.moves.first[q] + j; },
                       [&](uint32_t, uint32_t, uint32_t j, uint32_t page) {
                           if (to + j < a.capacity) a.free_list[to + j] = page;
                           else report_error(a.status, DEV_ERR_BOUNDS, 613, (uint32_t)(to + j), a.capacity);
                       });
            given += back_total;
            __syncthreads();
        }
        return first;
    };
    // Pages taken.
    uint64_t wanted = 0, used = 0, placed = 0, have = 0;
    uint32_t refused = 0;
    auto second_pass = [&](const Mine& m, uint32_t base, uint64_t both_before, uint64_t both_total) {
        const uint32_t r = base + threadIdx.x, want = m.want(), before = (uint32_t)(both_before >> 32), total = (uint32_t)(both_total >> 32);
        const bool granted = m.fits && (want == 0 || wanted + before + want <= have);
        if (r < a.n) {
            a.held_out[r] = granted ? m.need : m.held;
            a.lens[r] = granted ? m.ctx + m.add : 0;
            if (granted) used += want, placed += m.add; else refused++;
        }
        if (total != 0) {
            sm.moves.before[threadIdx.x] = before;
            sm.moves.first[threadIdx.x] = m.held;
            // those that are granted are the first of those that want any: the words up to the first one that is not
            const bool all = wanted + total <= have;
            if (threadIdx.x == 0) sm.moves.before[threads] = all ? total : 0;
            __syncthreads();
            if (!all) {
                if (granted && want) atomicMax(&sm.moves.before[threads], before + want);
                __syncthreads();
            }
            const uint32_t* last = a.free_list + (have - 1 - wanted);
            move_words(sm.moves, threads, [&](uint32_t, uint32_t, uint32_t j) { return last - j; },
                       [&](uint32_t q, uint32_t j, uint32_t, uint32_t page) { a.table[(size_t)(base + q) * a.stride + sm.moves.first[q] + j] = page; });
            __syncthreads();
        }
        wanted += total;
    };
    if (KEPT) {
#pragma unroll
        for (uint32_t k = 0; k < ROUNDS; k++)
            if (k * threads < a.n) kept_first[k] = first_pass(kept[k], k * threads, kept_before[k], kept_total[k]);
        have = min(count + given, (uint64_t)a.capacity);
#pragma unroll
        for (uint32_t k = 0; k < ROUNDS; k++)
            if (k * threads < a.n) second_pass(kept[k], k * threads, kept_before[k], kept_total[k]);
    } else {
        for (uint32_t base = 0; base < a.n; base += threads) {
            Mine m = load(base + threadIdx.x);
            uint64_t before, total;
            first_pass(m, base, before, total);
        }
        have = min(count + given, (uint64_t)a.capacity);
        ends = 0;
        for (uint32_t base = 0; base < a.n; base += threads) {
            Mine m = load(base + threadIdx.x);
            look(m, base + threadIdx.x, ends);
            uint64_t total;
            const uint64_t before = sum_up(m, total);
            second_pass(m, base, before, total);
        }
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) {
        used += __shfl_xor_sync(0xffffffffu, used, off);
        placed += __shfl_xor_sync(0xffffffffu, placed, off);
        refused += __shfl_xor_sync(0xffffffffu, refused, off);
    }
    if ((threadIdx.x & 31) == 0) {
        atomicAdd(&counted[0], (unsigned long long)used);
        atomicAdd(&counted[1], (unsigned long long)refused);
        atomicAdd(&counted[2], (unsigned long long)placed);
    }
    if (KEPT && place_here) {
#pragma unroll
        for (uint32_t k = 0; k < ROUNDS; k++)
            if (k * threads + threadIdx.x < a.n) sm.firsts[k * threads + threadIdx.x + 1] = kept_first[k];
        if (threadIdx.x == 0) sm.firsts[0] = 0;
    }
    __syncthreads();  // tables, lengths and starts are read from here on
    if (threadIdx.x == 0) {
        a.free_out[0] = (uint32_t)(have - counted[0]);
        a.free_out[1] = (uint32_t)counted[1];
        a.free_out[2] = (uint32_t)counted[2];
        a.free_out[3] = (uint32_t)counted[0];
    }
    if (!place_here) return;
    for (uint32_t t = threadIdx.x; t < a.tokens; t += threads) place_token(a, t, [&](uint32_t r) { return sm.firsts[r]; });
}

__global__ void __launch_bounds__(PLACE_THREADS) place_tokens_kernel(const __grid_constant__ PlanArgs a)
{
    __shared__ uint32_t firsts[SEARCHED + 1];
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t t = blockIdx.x * PLACE_THREADS + threadIdx.x;
    if (a.n <= SEARCHED) {
        for (uint32_t r = threadIdx.x; r <= a.n; r += PLACE_THREADS) firsts[r] = ld_global(a.starts + r);
        __syncthreads();
        if (t < a.tokens) place_token(a, t, [&](uint32_t r) { return firsts[r]; });
    } else if (t < a.tokens) {
        place_token(a, t, [&](uint32_t r) { return ld_global(a.starts + r); });
    }
}

// ---- append --------------------------------------------------------------------------------------------------------------------
// A run is a stretch of tokens with consecutive slots of one block; its first token leads it.  For every run, kv head and side one
// warp: A = max |x| over the run's rows, e = the least e >= -15 with A <= 448 * 2^e, no less than the tile's own exponent if
// the run does not begin the tile; if that grows, the rows before the run are rounded again (q * 2^(old - e)); then the run's rows
// are written as e4m3(x * 2^-e).  All products are by powers of two and exact in f16 wherever e4m3 does not round them to 0.
// Two bytes read and one written per value: bound by bytes.  17 prompts, 21078 tokens of 16 heads, take 47 us (5.5 TB/s), 64 single tokens
// 4.1, which is a launch and two loads one after the other.
constexpr int APPEND_THREADS = 256;

struct AppendArgs {
    const __half* src[2];
    const uint32_t* slots;
    uint8_t* pool[2];
    int8_t* exps[2];
    uint32_t n, n_kv, blocks;
    uint32_t* status;
};

// The least e >= LOWEST_EXP with a <= 448 * 2^e: a = f * 2^k, 1 <= f < 2, 448 = 1.75 * 2^8.
__device__ __forceinline__ int exponent_for(float a)
{
    const uint32_t bits = __float_as_uint(a);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, LOWEST_EXP);
}
// 2^e as f16 pair, e in [-24, 15].
__device__ __forceinline__ __half2 power_of_two(int e) { return __float2half2_rn(__int_as_float((e + 127) << 23)); }

// Eight f16 numbers as e4m3(x * f); 16 cached ones as e4m3(q * f).
__device__ __forceinline__ uint2 quantise(const uint4& x, __half2 f)
{
    const __half2 top = __float2half2_rn(61440.0f), low = __float2half2_rn(-61440.0f);
    const auto pair = [&](uint32_t w) { return f16x2_to_e4m3x2(as_u32(__hmul2(__hmax2_nan(__hmin2_nan(as_half2(w), top), low), f))); };
    return make_uint2(pair(x.x) | (pair(x.y) << 16), pair(x.z) | (pair(x.w) << 16));
}
__device__ __forceinline__ uint4 round_again(uint4 v, __half2 f)
{
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t lo = f16x2_to_e4m3x2(as_u32(__hmul2(as_half2(e4m3x2_to_f16x2(w[k] & 0xffffu)), f)));
        const uint32_t hi = f16x2_to_e4m3x2(as_u32(__hmul2(as_half2(e4m3x2_to_f16x2(w[k] >> 16)), f)));
        w[k] = lo | (hi << 16);
    }
    return v;
}
__device__ __forceinline__ __half2 largest(__half2 m, const uint4& x)  // a NaN loses against a number
{
    m = __hmax2(__hmax2(m, __habs2(as_half2(x.x))), __habs2(as_half2(x.y)));
    return __hmax2(__hmax2(m, __habs2(as_half2(x.z))), __habs2(as_half2(x.w)));
}

__device__ __forceinline__ void append_run(const AppendArgs& a, int side, uint32_t head, uint32_t t, uint32_t slot, uint32_t run)
{
    const uint32_t lane = threadIdx.x & 31, half = lane >> 4, c = lane & 15;
    const uint32_t block = slot / TILE_TOK, at = slot % TILE_TOK;
    const size_t tile = (size_t)block * a.n_kv + head;
    const __half* src = a.src[side] + ((size_t)t * a.n_kv + head) * 128 + c * 8;
    uint8_t* out = a.pool[side] + tile * TILE_BYTES;
    uint4 x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t j = 2 * i + half;
        x[i] = make_uint4(0, 0, 0, 0);
        if (j < run) x[i] = ld_global(reinterpret_cast<const uint4*>(src + (size_t)j * a.n_kv * 128));
    }
    int old = LOWEST_EXP;
    if (at != 0) old = *(volatile const int8_t*)(a.exps[side] + tile);
    __half2 m = __float2half2_rn(0.0f);
#pragma unroll
    for (int i = 0; i < 8; i++) m = largest(m, x[i]);
#pragma unroll
    for (int off = 16; off; off >>= 1) m = __hmax2(m, as_half2(__shfl_xor_sync(0xffffffffu, as_u32(m), off)));
    const float most = fminf(fmaxf(__low2float(m), __high2float(m)), 61440.0f);
    const int e = max(exponent_for(most), old);
    if (at != 0 && e > old) {
        const __half2 f = power_of_two(max(old - e, -24));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (4 * i + lane / 8 < at) {
                uint4* p = reinterpret_cast<uint4*>(out + i * 512 + lane * 16);
                *p = round_again(ld_global(p), f);
            }
        }
    }
    const __half2 f = power_of_two(-e);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t j = 2 * i + half;
        if (j < run)
            *reinterpret_cast<uint2*>(out + (at + j) * 128 + c * 8) =
                quantise(x[i], f);
    }
    if (lane == 0) a.exps[side][tile] = (int8_t)e;
}

// Runs of one token (a decode step's), up to 2 N of them at a time: half a warp for each, all their loads on their way together.
template <int N>
__device__ __forceinline__ void append_singles(const AppendArgs& a, int side, uint32_t head, uint32_t t0, uint32_t my_slot, uint32_t& todo)
{
    const uint32_t lane = threadIdx.x & 31, half = lane >> 4, c = lane & 15;
    uint4 x[N];
    uint32_t slot[N];
    int old[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int first = todo ? __ffs(todo) - 1 : 0;
        const bool has_first = todo != 0;
        todo &= todo - 1;
        const int second = todo ? __ffs(todo) - 1 : 0;
        const bool has_second = todo != 0;
        todo &= todo - 1;
        const uint32_t src = half ? second : first;
        const uint32_t s = __shfl_sync(0xffffffffu, my_slot, src);
        slot[i] = (half ? has_second : has_first) ? s : NO_SLOT;
        const bool on = slot[i] != NO_SLOT;
        x[i] = ld_global_if(on, reinterpret_cast<const uint4*>(a.src[side] + ((size_t)(t0 + src) * a.n_kv + head) * 128 + c * 8));
        old[i] = ld_global_if(on && slot[i] % TILE_TOK != 0, a.exps[side] + (size_t)(slot[i] / TILE_TOK) * a.n_kv + head);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        __half2 m = largest(__float2half2_rn(0.0f), x[i]);
#pragma unroll
        for (int off = 8; off; off >>= 1) m = __hmax2(m, as_half2(__shfl_xor_sync(0xffffffffu, as_u32(m), off)));
        if (slot[i] == NO_SLOT) continue;
        const uint32_t at = slot[i] % TILE_TOK;
        const size_t tile = (size_t)(slot[i] / TILE_TOK) * a.n_kv + head;
        uint8_t* out = a.pool[side] + tile * TILE_BYTES;
        const int least = at ? old[i] : LOWEST_EXP, e = max(exponent_for(fminf(fmaxf(__low2float(m), __high2float(m)), 61440.0f)), least);
        if (at != 0 && e > least) {
            const __half2 f = power_of_two(max(least - e, -24));
            for (uint32_t j = c / 8; j < at; j += 2) {
                uint4* p = reinterpret_cast<uint4*>(out + j * 128 + (c & 7) * 16);
                *p = round_again(ld_global(p), f);
            }
        }
        *reinterpret_cast<uint2*>(out + at * 128 + c * 8) = quantise(x[i], power_of_two(-e));
        if (c == 0) a.exps[side][tile] = (int8_t)e;
    }
}

// SPAN tokens of the slot map per warp, kv head and side.  A lane looks at one slot, of the SPAN tokens and of those that a run which one of
// them leads can go on with, so that the runs are known after one load.
template <int SPAN>
__global__ void __launch_bounds__(APPEND_THREADS) append_blocks_kernel(const __grid_constant__ AppendArgs a)
{
    static_assert(SPAN + TILE_TOK - 1 <= 32, "a lane a slot");
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t unit = (uint64_t)blockIdx.x * (APPEND_THREADS / 32) + threadIdx.x / 32;
    const int side = (int)(unit & 1);
    const uint32_t head = (uint32_t)((unit >> 1) % a.n_kv);
    const uint64_t t0 = (unit >> 1) / a.n_kv * SPAN;
    if (t0 >= a.n) return;
    uint32_t slot = NO_SLOT, first_before = NO_SLOT;
    if (t0 + lane < a.n) slot = ld_global(a.slots + t0 + lane);
    if (lane == 0 && t0 > 0) first_before = ld_global(a.slots + t0 - 1);
    uint32_t before = __shfl_up_sync(0xffffffffu, slot, 1);
    if (lane == 0) before = first_before;
    const bool follows = slot != NO_SLOT && before != NO_SLOT && before + 1 == slot && slot % TILE_TOK != 0;
    bool leads = false;
    if (lane < SPAN && slot != NO_SLOT) {
        if (slot / TILE_TOK >= a.blocks) {
            report_error(a.status, DEV_ERR_BOUNDS, 621, slot, a.blocks);
        } else if (before != NO_SLOT && before / TILE_TOK == slot / TILE_TOK && before + 1 != slot) {
            report_error(a.status, DEV_ERR_BOUNDS, 622, before, slot);  // a tile's tokens stand in its order
        } else {
            leads = !follows;
        }
    }
    const uint32_t chain = __ballot_sync(0xffffffffu, follows), leaders = __ballot_sync(0xffffffffu, leads);
    uint32_t singles = leaders & ~(chain >> 1);
    const uint32_t longer = leaders & ~singles;
    while (singles) append_singles<SPAN >= 8 ? 4 : SPAN / 2>(a, side, head, (uint32_t)t0, slot, singles);
    for (uint32_t todo = longer; todo; todo &= todo - 1) {
        const int src = __ffs(todo) - 1;
        const uint32_t more = src == 31 ? 0 : chain >> (src + 1);
        append_run(a, side, head, (uint32_t)t0 + src, __shfl_sync(0xffffffffu, slot, src), (uint32_t)__ffs(~more));
    }
}

struct PushPlan {
    uint32_t page, stride;
};

}  // namespace

// kv_block_tables: ctx, add, held, count, free list, table, held out, free out, starts, lens, slots, positions.
// push {page, table stride}.  grid [requests, tokens].
int launch_kv_block_tables(const LaunchArgs& a)
{
    const PushPlan p = *(const PushPlan*)a.push;
    const uint32_t n = a.groups[0], tokens = a.groups[1];
    if (n == 0 || n > MOST_REQUESTS) return fail_validation(a, "block_tables: groups[0] (requests) must be 1..65536");
    if (tokens == 0) return fail_validation(a, "block_tables: groups[1] (tokens of the step) must be > 0");
    if (p.page < (uint32_t)TILE_TOK || (p.page & (p.page - 1))) return fail_validation(a, "block_tables: page must be a power of two, at least 16 tokens");
    if (p.stride == 0 || p.stride > MOST_STRIDE) return fail_validation(a, "block_tables: the table's stride must be 1..2097152 pages");
    if (int r = need_aligned(a, {4, 4, 4, 4, 4, 4, 4, 4, 4, 4, 4, 4})) return r;
    const size_t per = 4 * (size_t)n;
    const char* names[12] = {"ctx", "new", "held", "count", "free list", "table", "held out", "free out", "starts", "lens", "slots", "positions"};
    const size_t bytes[12] = {per, per, per, 4, 4, per * p.stride, per, 16, per + 4, per, 4 * (size_t)tokens, 4 * (size_t)tokens};
    for (int i = 0; i < 12; i++)
        if (int r = need_bytes(a, i, bytes[i], names[i])) return r;
    const auto u = [&](int i) { return (uint32_t*)a.b[i].ptr; };
    const size_t capacity = a.b[4].bytes / 4;
    PlanArgs k{u(0), u(1), u(2), u(3), u(4), u(5), u(6), u(7), u(8), u(9), u(10), u(11), n, tokens, (uint32_t)__builtin_ctz(p.page), p.stride,
               (uint32_t)(capacity < NO_SLOT ? capacity : NO_SLOT), a.status};
    const bool place_here = n <= SEARCHED && tokens <= PLACED_HERE;
    const uint32_t work = !place_here && n < 256 ? 256 : place_here && tokens > n ? tokens : n, threads = work < PLAN_THREADS ? (work + 31) / 32 * 32 : PLAN_THREADS;
    cudaError_t e = launch_dependent(n <= KEPT_ROUNDS * threads ? block_tables_kernel<true> : block_tables_kernel<false>, dim3(1), dim3(threads), 0, a.stream, k, place_here);
    ++*a.launches;
    if (int r = check_cuda(a, e, "kv_block_tables")) return r;
    if (place_here) return 0;
    e = launch_dependent(place_tokens_kernel, dim3((unsigned)((tokens + PLACE_THREADS - 1ull) / PLACE_THREADS)), dim3(PLACE_THREADS), 0, a.stream, k);
    ++*a.launches;
    return check_cuda(a, e, "kv_block_tables tokens");
}

// kv_append_blocks_e4m3_d128: k, v f16 [n x KV x 128], slots, k pool, k exps, v pool, v exps.  grid [KV, n].
int launch_kv_append_blocks(const LaunchArgs& a)
{
    const uint32_t n_kv = a.groups[0], n = a.groups[1];
    if (n_kv == 0 || n == 0) return fail_validation(a, "append_blocks: groups must be [kv heads, tokens]");
    const size_t tile_row = (size_t)n_kv * TILE_BYTES, src = (size_t)n * n_kv * 256;
    const size_t blocks = a.b[3].bytes / tile_row;
    if (int r = need_bytes(a, 0, src, "k")) return r;
    if (int r = need_bytes(a, 1, src, "v")) return r;
    if (int r = need_bytes(a, 2, 4 * (size_t)n, "slots")) return r;
    if (blocks == 0 || a.b[5].bytes / tile_row != blocks)
        return fail_validation(a, "append_blocks: K and V pools must hold the same (non-zero) number of 16-token blocks");
    if (blocks > NO_SLOT / TILE_TOK) return fail_validation(a, "append_blocks: a pool holds less than 2^32 rows");
    if (int r = need_bytes(a, 4, blocks * n_kv, "k exponents")) return r;
    if (int r = need_bytes(a, 6, blocks * n_kv, "v exponents")) return r;
    if (int r = need_aligned(a, {16, 16, 4, 16, 1, 16, 1})) return r;
    AppendArgs k{{(const __half*)a.b[0].ptr, (const __half*)a.b[1].ptr}, (const uint32_t*)a.b[2].ptr, {(uint8_t*)a.b[3].ptr, (uint8_t*)a.b[5].ptr},
                 {(int8_t*)a.b[4].ptr, (int8_t*)a.b[6].ptr}, n, n_kv, (uint32_t)blocks, a.status};
    // Four tokens a warp while all warps are on the GPU at once, else sixteen (us, 16 kv heads, with 4 | with 16: 64 requests of one token 4.2 |
    // 6.2, 300 4.2 | 6.2, 1100 6.7 | 6.4, 4000 20.6 | 18.6; 17 prompts, 20300 tokens, 60.0 | 45.9; with one token a warp the last took 181).
    const uint64_t per_token = 2ull * n_kv;
    const bool few = per_token * ((n + 3ull) / 4) <= 64ull * a.sm_count;
    const uint64_t warps = per_token * (few ? (n + 3ull) / 4 : (n + 15ull) / 16);
    const unsigned ctas = (unsigned)((warps + APPEND_THREADS / 32 - 1) / (APPEND_THREADS / 32));
    const cudaError_t e = launch_dependent(few ? append_blocks_kernel<4> : append_blocks_kernel<16>, dim3(ctas), dim3(APPEND_THREADS), 0, a.stream, k);
    ++*a.launches;
    return check_cuda(a, e, "kv_append_blocks_e4m3_d128");
}

}  // namespace sgb
