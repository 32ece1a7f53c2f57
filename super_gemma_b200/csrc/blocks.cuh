// The 8-bit cache that many requests share: e4m3 numbers in tiles of 16 tokens of one kv head, one power of two per tile.
//
//   pool   u8 [block][kv head][16 tokens][128]    2048 consecutive bytes per (block, head); pool row = 16 * block + token in block
//   exps   i8 [block][kv head]                    value = e4m3 * 2^e, e in [-15, 8] as the append writes it
//   table  u32 [request][stride]                  token t of request r: row table[r][t / page] * page + t % page
//
// The scale is a power of two because e4m3 carries four significant bits whatever its scale: a free factor would buy nothing, and
// a power of two makes quantising, growing a tile's scale and undoing it exact but for e4m3's own rounding.  Magnitudes above
// 61440 count as 61440, the largest f16 of four significant bits, so that every cached value is an f16 number; 2^-15 is the least
// scale because f16's own grid is 2^-24 and e4m3's is 2^-9.
#pragma once

#include "sgb_common.cuh"

namespace sgb {

constexpr int TILE_TOK = 16;
constexpr uint32_t TILE_BYTES = TILE_TOK * 128;
constexpr uint32_t NO_SLOT = 0xffffffffu;
constexpr int LOWEST_EXP = -15;
constexpr uint32_t MOST_REQUESTS = 65536;
constexpr uint32_t MOST_KEYS = 0x3fffff00u;  // of one request: positions are signed words, and 256 requests' tiles of 64 keys fit one
constexpr uint32_t FEW_ROWS = 16;            // requests of at most so many rows (query tokens x heads of a group) can be decoded, the others are prefilled

// What a dispatch over the cache knows of its requests.
struct Requests {
    const uint32_t* table;   // [n][stride]
    const uint32_t* lens;    // [n] keys of each, this step's tokens among them
    const uint32_t* starts;  // [n + 1] first query token of each
    uint32_t n, stride, page_shift, pool_pages, tokens, max_q, window;
    uint32_t* status;
};
struct Request {
    uint32_t first, n, len;  // its query tokens, its keys
};
// Lengths come from the device: what does not fit the buffers is reported and taken as nothing (queries) or cut (keys).
__device__ __forceinline__ Request checked_request(const Requests& a, uint32_t r, uint32_t first, uint32_t end, uint32_t len)
{
    Request q{first, end - first, len};
    if (end < first || end > a.tokens || q.n > a.max_q) {
        report_error(a.status, DEV_ERR_BOUNDS, 601, r, end);
        q.n = 0;
    }
    const uint64_t most = min((uint64_t)a.stride << a.page_shift, (uint64_t)MOST_KEYS);
    if (q.len > most) {
        report_error(a.status, DEV_ERR_BOUNDS, 602, r, q.len);
        q.len = (uint32_t)most;
    }
    return q;
}
__device__ __forceinline__ Request request_at(const Requests& a, uint32_t r)
{
    const uint32_t first = ld_global(a.starts + r), end = ld_global(a.starts + r + 1), len = ld_global(a.lens + r);
    return checked_request(a, r, first, end, len);
}
// The pool's block that holds tokens 16 * tile .. of request r, in two steps, so that nothing waits for the table in between: its
// page's number, then the block.  A page that the pool does not have is reported and read as page 0.
__device__ __forceinline__ uint32_t block_of_page(const Requests& a, uint32_t r, uint32_t tile, uint32_t page)
{
    const uint32_t shift = a.page_shift - 4;
    if (page >= a.pool_pages) {
        report_error(a.status, DEV_ERR_BOUNDS, 604, r, page);
        page = 0;
    }
    return (page << shift) + (tile & ((1u << shift) - 1));
}
// `tile` lies within the request's keys, and those within its row of the table (request_at cuts them).
__device__ __forceinline__ const uint32_t* page_at(const Requests& a, uint32_t r, uint32_t tile) { return a.table + (size_t)r * a.stride + (tile >> (a.page_shift - 4)); }

// A dispatch of attn_blocks_e4m3_d128.
struct BlocksAttn {
    Requests req;
    const __half* q;
    const uint8_t* pool[2];
    const int8_t* exps[2];
    __half* out;
    uint32_t n_kv, group, group_shift, tiles;  // tiles of a pool: blocks x kv heads
    uint32_t few;                              // requests of at most so many query tokens are decoded
    float scale;
};
struct LaunchArgs;

// Loads that may be left out, as one instruction: a branch around the load would have its result moved behind it, and so waited for.
__device__ __forceinline__ uint4 ld_global_if(bool p, const uint4* at)
{
    uint4 v;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
        "@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
        : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
        : "l"(at), "r"((uint32_t)p));
    return v;
}
__device__ __forceinline__ uint2 ld_global_if(bool p, const uint2* at)
{
    uint2 v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %3, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\t@p ld.global.v2.b32 {%0, %1}, [%2];\n\t}"
                 : "=&r"(v.x), "=&r"(v.y)
                 : "l"(at), "r"((uint32_t)p));
    return v;
}
__device__ __forceinline__ uint32_t ld_global_if(bool p, const uint32_t* at)
{
    uint32_t v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.global.b32 %0, [%1];\n\t}" : "=&r"(v) : "l"(at), "r"((uint32_t)p));
    return v;
}
__device__ __forceinline__ int ld_global_if(bool p, const int8_t* at)
{
    int v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.global.s8 %0, [%1];\n\t}" : "=&r"(v) : "l"(at), "r"((uint32_t)p));
    return v;
}

// f(r, request) for r in [begin, end), four requests' words on their way at a time.
template <typename F>
__device__ __forceinline__ void for_requests(const Requests& a, uint32_t begin, uint32_t end, const F& f)
{
    for (uint32_t r0 = begin; r0 < end; r0 += 4) {
        uint32_t first[5], len[4];
#pragma unroll
        for (uint32_t k = 0; k < 5; k++) first[k] = ld_global_if(r0 + k <= end, a.starts + r0 + k);
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) len[k] = ld_global_if(r0 + k < end, a.lens + r0 + k);
#pragma unroll
        for (uint32_t k = 0; k < 4; k++)
            if (r0 + k < end) f(r0 + k, checked_request(a, r0 + k, first[k], first[k + 1], len[k]));
    }
}

// Two e4m3 bytes as two f16, exactly (one instruction at the rate of an integer one: 64 a clock and SM).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two_bytes)
{
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two_bytes));
    return r;
}
__device__ __forceinline__ uint32_t f16x2_to_e4m3x2(uint32_t x)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(x));
    return r;
}
// The bytes of four e4m3 numbers that are a NaN (0x7f, 0xff): 0x80 in each of those.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// Those of 16 numbers become 0: whether there are any.
__device__ __forceinline__ bool drop_nans(uint4& v)
{
    const uint32_t x = nan_bytes(v.x), y = nan_bytes(v.y), z = nan_bytes(v.z), w = nan_bytes(v.w);
    v = make_uint4(v.x & ~((x >> 7) * 0xffu), v.y & ~((y >> 7) * 0xffu), v.z & ~((z >> 7) * 0xffu), v.w & ~((w >> 7) * 0xffu));
    return (x | y | z | w) != 0;
}
__device__ __forceinline__ __half2 as_half2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
__device__ __forceinline__ uint32_t as_u32(__half2 x) { return *reinterpret_cast<const uint32_t*>(&x); }

// The least e >= LOWEST_EXP with a <= 448 * 2^e: a = f * 2^k, 1 <= f < 2, 448 = 1.75 * 2^8.
__device__ __forceinline__ int exponent_for(float a)
{
    const uint32_t bits = __float_as_uint(a);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, LOWEST_EXP);
}
// 2^e as f16 pair, e in [-24, 15].
__device__ __forceinline__ __half2 power_of_two(int e) { return __float2half2_rn(__int_as_float((e + 127) << 23)); }

// 2^e in f32, e in [-126, 127].
__device__ __forceinline__ float exp2_of(int e) { return __int_as_float((e + 127) << 23); }
// 16 cached numbers as e4m3(q * f).
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

}  // namespace sgb
