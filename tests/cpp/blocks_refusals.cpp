// Calls of the batched cache's launchers that have to be refused by their own checks.  Every call here differs from a good one in one
// thing; the launchers return SGB_ERR_VALIDATION (3) before they touch a device, so this runs on a machine without one.
#include <cstdio>
#include <cstring>
#include <functional>
#include <string>
#include <vector>

#include "sgb_kernels.h"

using namespace sgb;

static int failures = 0, calls = 0;

struct Call {
    std::vector<BufView> b;
    std::vector<uint32_t> push;
    uint32_t groups[3];
    LaunchFn fn;
    void expect(const char* what, const char* text)
    {
        std::string err;
        uint64_t launches = 0;
        LaunchArgs a{nullptr, b.data(), push.data(), {groups[0], groups[1], groups[2]}, nullptr, 148, 0, &err, &launches};
        const int r = fn(a);
        calls++;
        if (r != 3 || launches != 0 || err.find(text) == std::string::npos) {
            printf("%s: returned %d, %llu launches, \"%s\"\n", what, r, (unsigned long long)launches, err.c_str());
            failures++;
        }
    }
};

static uint32_t bits(float f)
{
    uint32_t u;
    memcpy(&u, &f, 4);
    return u;
}
static BufView at(size_t bytes) { return BufView{(void*)0x10000, bytes}; }

int main()
{
    // 3 requests, page 32, stride 4, 8 tokens
    const Call plan{{at(12), at(12), at(12), at(4), at(64), at(48), at(12), at(16), at(16), at(12), at(32), at(32)}, {32, 4}, {3, 8, 1}, launch_kv_block_tables};
    auto with = [](Call c, const std::function<void(Call&)>& change) { change(c); return c; };
    with(plan, [](Call& c) { c.groups[0] = 0; }).expect("no requests", "requests");
    with(plan, [](Call& c) { c.groups[0] = 65537; }).expect("too many requests", "requests");
    with(plan, [](Call& c) { c.groups[1] = 0; }).expect("no tokens", "tokens");
    for (uint32_t page : {0u, 8u, 48u}) with(plan, [=](Call& c) { c.push[0] = page; }).expect("page", "page");
    with(plan, [](Call& c) { c.push[1] = 0; }).expect("stride", "stride");
    for (size_t i = 0; i < plan.b.size(); i++) {
        if (i != 4) with(plan, [=](Call& c) { c.b[i].bytes -= 4; }).expect("short binding", "holds");
        with(plan, [=](Call& c) { c.b[i].ptr = (char*)c.b[i].ptr + 2; }).expect("misaligned", "aligned");
    }
    with(plan, [](Call& c) { c.b[4].bytes = 0; }).expect("empty list", "holds");
    with(plan, [](Call& c) { c.groups[0] = 65536; c.push[1] = 1u << 21; c.b[0].bytes = c.b[1].bytes = c.b[2].bytes = 1 << 18; }).expect("table beyond 2^32 bytes", "holds");
    with(plan, [](Call& c) { c.push[1] = (1u << 21) + 1; }).expect("stride", "stride");

    // 3 kv heads, 5 tokens, 4 blocks
    const size_t pool = 4 * 3 * 2048;
    const Call append{{at(5 * 768), at(5 * 768), at(20), at(pool), at(12), at(pool), at(12)}, {}, {3, 5, 1}, launch_kv_append_blocks};
    with(append, [](Call& c) { c.groups[0] = 0; }).expect("no heads", "groups");
    with(append, [](Call& c) { c.groups[1] = 0; }).expect("no tokens", "groups");
    for (size_t i : {0, 1, 2, 4, 6}) with(append, [=](Call& c) { c.b[i].bytes -= 1; }).expect("short binding", "holds");
    with(append, [](Call& c) { c.b[5].bytes -= 1; }).expect("V pool shorter", "same");
    with(append, [](Call& c) { c.b[3].bytes = c.b[5].bytes = 2048; }).expect("no block", "same");
    for (size_t i : {0, 1, 3, 5}) with(append, [=](Call& c) { c.b[i].ptr = (char*)c.b[i].ptr + 8; }).expect("misaligned", "aligned");
    with(append, [](Call& c) { c.b[2].ptr = (char*)c.b[2].ptr + 1; }).expect("misaligned", "aligned");

    // 3 kv heads, 2 query heads each, 2 requests, 5 tokens, page 16, stride 2
    const size_t work = attn_blocks_work_bytes(148, 3, 2, 2, 5, 4), rows = 5 * 6 * 256;
    const Call attend{{at(rows), at(pool), at(12), at(pool), at(12), at(16), at(8), at(12), at(rows), at(work)}, {bits(0.1f), 16, 2, 0, 2, 4}, {3, 2, 5}, launch_attn_blocks};
    for (int g = 0; g < 3; g++) with(attend, [=](Call& c) { c.groups[g] = 0; }).expect("empty grid", "groups");
    with(attend, [](Call& c) { c.groups[1] = 65537; }).expect("too many requests", "requests");
    for (uint32_t g : {0u, 3u, 16u}) with(attend, [=](Call& c) { c.push[4] = g; }).expect("group", "query heads");
    for (uint32_t page : {0u, 8u, 24u}) with(attend, [=](Call& c) { c.push[1] = page; }).expect("page", "page");
    with(attend, [](Call& c) { c.push[2] = 0; }).expect("stride", "stride");
    with(attend, [](Call& c) { c.push[5] = 0; }).expect("no query", "stride");
    for (float s : {0.0f, -1.0f, __builtin_nanf(""), __builtin_inff()}) with(attend, [=](Call& c) { c.push[0] = bits(s); }).expect("scale", "scale");
    for (size_t i : {0, 2, 4, 5, 6, 7, 8, 9}) with(attend, [=](Call& c) { c.b[i].bytes -= 1; }).expect("short binding", "holds");
    with(attend, [](Call& c) { c.b[3].bytes -= 1; }).expect("V pool shorter", "same");
    with(attend, [](Call& c) { c.push[1] = 128; }).expect("pool smaller than a page", "page");
    for (size_t i : {0, 1, 3, 8, 9}) with(attend, [=](Call& c) { c.b[i].ptr = (char*)c.b[i].ptr + 8; }).expect("misaligned", "aligned");
    for (size_t i : {5, 6, 7}) with(attend, [=](Call& c) { c.b[i].ptr = (char*)c.b[i].ptr + 2; }).expect("misaligned", "aligned");
    if (failures) return 1;
    printf("%d calls refused as they should be\n", calls);
    return 0;
}
