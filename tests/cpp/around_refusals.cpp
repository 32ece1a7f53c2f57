// Calls of the launchers around the batched attention that have to be refused by their own checks.  Every call here differs from a good one in
// one thing; the launchers return SGB_ERR_VALIDATION (3) before they touch a device, so this runs on a machine without one.
#include <cuda_bf16.h>

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
static size_t next = 0x100000;
static BufView at(size_t bytes)
{
    const size_t p = next;
    next += (bytes + 4095) / 4096 * 4096;
    return BufView{(void*)p, bytes};
}
static Call with(Call c, const std::function<void(Call&)>& change)
{
    change(c);
    return c;
}
static void short_and_misaligned(const Call& call, std::initializer_list<uint32_t> align, std::initializer_list<int> exact = {})
{
    size_t i = 0;
    for (const uint32_t n : align) {
        bool whole = true;
        for (int e : exact) whole = whole && (size_t)e != i;
        if (whole) with(call, [=](Call& c) { c.b[i].bytes -= 1; }).expect("short binding", "holds");
        if (n > 1) with(call, [=](Call& c) { c.b[i].ptr = (char*)c.b[i].ptr + n / 2; }).expect("misaligned", "aligned");
        i++;
    }
}

int main()
{
    const float inf = __builtin_inff(), nan = __builtin_nanf("");

    // 5 tokens, 48 dims that turn
    const Call angles{{at(24 * 8), at(20), at(5 * 48 * 4)}, {48, bits(1.0f)}, {5, 1, 1}, launch_rope_cos_sin};
    with(angles, [](Call& c) { c.groups[0] = 0; }).expect("no tokens", "tokens");
    for (uint32_t rot : {0u, 8u, 24u, 1040u}) with(angles, [=](Call& c) { c.push[0] = rot; }).expect("rot_dims", "rot_dims");
    for (float m : {0.0f, -1.0f, inf, nan}) with(angles, [=](Call& c) { c.push[1] = bits(m); }).expect("magnitude", "magnitude");
    short_and_misaligned(angles, {8, 4, 16});
    with(angles, [](Call& c) { c.groups[0] = 0xffffffffu; }).expect("2^32 tokens", "holds");

    // 5 tokens, 6 and 2 heads of 80 dims, 48 of them turn; q and k side by side in rows of 640
    const Call rotate{{at(5 * 640 * 2), at(4 * 640 * 2 + 320), at(5 * 48 * 4), at(5 * 480 * 2), at(5 * 160 * 2)}, {80, 48, 1, 640, 640, 0, 0}, {6, 2, 5}, launch_rope_qk_f16};
    with(rotate, [](Call& c) { c.groups[0] = 0; }).expect("no heads", "groups");
    with(rotate, [](Call& c) { c.groups[2] = 0; }).expect("no tokens", "groups");
    with(rotate, [](Call& c) { c.groups[0] = 4097; }).expect("heads", "heads");
    with(rotate, [](Call& c) { c.groups[1] = 0xffffffffu; }).expect("heads", "heads");
    for (uint32_t d : {0u, 8u, 72u, 1040u, 0xfffffff0u}) with(rotate, [=](Call& c) { c.push[0] = d; }).expect("head_dim", "head_dim");
    for (uint32_t d : {0u, 8u, 40u, 96u}) with(rotate, [=](Call& c) { c.push[1] = d; }).expect("rot_dims", "rot_dims");
    with(rotate, [](Call& c) { c.push[2] = 3; }).expect("layout", "layout");
    for (int i : {3, 4, 5, 6})
        for (uint32_t s : {8u, 644u}) with(rotate, [=](Call& c) { c.push[i] = s; }).expect("stride", "stride");
    with(rotate, [](Call& c) { c.b[0].bytes = (4 * 640 + 480) * 2 - 1; }).expect("short q", "holds");
    for (int i : {1, 2, 3, 4}) with(rotate, [=](Call& c) { c.b[i].bytes -= 1; }).expect("short binding", "holds");
    for (int i : {0, 1, 2, 3, 4}) with(rotate, [=](Call& c) { c.b[i].ptr = (char*)c.b[i].ptr + 8; }).expect("misaligned", "aligned");
    with(rotate, [](Call& c) { c.b[3].ptr = c.b[0].ptr; }).expect("q_out on q with another stride", "overlaps");
    with(rotate, [](Call& c) { c.b[3] = BufView{(char*)c.b[0].ptr + 32, 8000}; c.push[5] = 640; }).expect("q_out shifted on q", "overlaps");
    with(rotate, [](Call& c) { c.b[4] = BufView{(char*)c.b[0].ptr, 8000}; c.push[6] = 640; }).expect("k_out on q", "overlaps");
    with(rotate, [](Call& c) { c.b[3] = BufView{(char*)c.b[1].ptr, 8000}; c.push[5] = 640; }).expect("q_out on k", "overlaps");
    with(rotate, [](Call& c) { c.b[4].ptr = (char*)c.b[3].ptr + 64; }).expect("k_out on q_out", "overlap");
    with(rotate, [](Call& c) { c.groups[0] = 4096; c.groups[2] = 1u << 20; c.push[0] = 1024; c.push[1] = 1024; c.push[3] = 0; for (auto& b : c.b) b.bytes = 1ull << 45; c.push[4] = 0;
                               for (size_t i = 0; i < 5; i++) c.b[i].ptr = (void*)((i + 1) << 46); }).expect("2^42 values", "2^36");

    // 5 tokens, 6 and 3 heads, 4 blocks, rows of 12 * 128 side by side
    const size_t pool = 4 * 3 * 2048;
    const uint32_t row = 12 * 128;
    const Call pre{{at((4 * row + 768) * 2), at(512), at(5 * 6 * 256), at((4 * row + 384) * 2), at((4 * row + 384) * 2), at(512), at(5 * 64 * 4), at(20), at(pool), at(12), at(pool), at(12)},
                   {64, 0, 0, row, row, row, bits(1.0f)}, {6, 3, 5}, launch_qkv_norm_rope_append_blocks};
    for (int g = 0; g < 3; g++) with(pre, [=](Call& c) { c.groups[g] = 0; }).expect("empty grid", "groups");
    with(pre, [](Call& c) { c.groups[0] = 8193; }).expect("heads", "heads");
    with(pre, [](Call& c) { c.groups[1] = 1025; }).expect("heads", "heads");
    with(pre, [](Call& c) { c.groups[2] = (1u << 26) + 1; }).expect("tokens", "tokens");
    for (uint32_t d : {8u, 40u, 144u}) with(pre, [=](Call& c) { c.push[0] = d; }).expect("rot_dims", "rot_dims");
    with(pre, [](Call& c) { c.push[1] = 3; }).expect("layout", "layout");
    with(pre, [](Call& c) { c.push[2] = 2; }).expect("plus_one", "plus_one");
    for (int i : {3, 4, 5})
        for (uint32_t s : {8u, row + 4}) with(pre, [=](Call& c) { c.push[i] = s; }).expect("stride", "stride");
    for (float m : {0.0f, -1.0f, inf, nan, 65536.0f}) with(pre, [=](Call& c) { c.push[6] = bits(m); }).expect("magnitude", "magnitude");
    short_and_misaligned(pre, {16, 16, 16, 16, 16, 16, 16, 4, 16, 1, 16, 1}, {8, 10});
    with(pre, [](Call& c) { c.b[10].bytes -= 1; }).expect("V pool shorter", "same");
    with(pre, [](Call& c) { c.b[8].bytes = c.b[10].bytes = 2048; }).expect("no block", "same");
    with(pre, [](Call& c) { c.b[2].ptr = c.b[0].ptr; }).expect("q_out on strided q", "q_out overlaps q");
    with(pre, [](Call& c) { c.b[2].ptr = c.b[3].ptr; }).expect("q_out on k", "q_out overlaps k");
    with(pre, [](Call& c) { c.b[2].ptr = c.b[4].ptr; }).expect("q_out on v", "q_out overlaps v");

    // 5 rows of 40
    for (int type = 0; type < 3; type++) {
        const size_t n = 200, size = type == 2 ? 4 : 2;
        const Call norms{{at(2 * n), at(size * n), at(160), at(160), at(160), at(size * n), at(2 * n)}, {1, 1, 0, bits(0.5f), bits(1e-6f)}, {40, 5, 1},
                         type == 0 ? launch_block_norms<__half> : type == 1 ? launch_block_norms<__nv_bfloat16> : launch_block_norms<float>};
        for (uint32_t hidden : {0u, 4u, 44u, 16392u}) with(norms, [=](Call& c) { c.groups[0] = hidden; }).expect("hidden", "hidden");
        with(norms, [](Call& c) { c.groups[1] = 0; }).expect("no rows", "rows");
        with(norms, [](Call& c) { c.push[0] = 3; }).expect("post", "post");
        with(norms, [](Call& c) { c.push[1] = 4; }).expect("gate", "gate");
        with(norms, [](Call& c) { c.push[2] = 2; }).expect("plus_one", "plus_one");
        for (float s : {inf, nan}) with(norms, [=](Call& c) { c.push[3] = bits(s); }).expect("scale", "scale");
        for (float e : {inf, nan, -1e-6f}) with(norms, [=](Call& c) { c.push[4] = bits(e); }).expect("eps", "eps");
        with(norms, [](Call& c) { c.push[0] = 2; }).expect("a gate of nothing", "post 2");
        with(norms, [](Call& c) { c.push[0] = 2; c.push[1] = 0; }).expect("a scale of nothing", "post 2");
        short_and_misaligned(norms, {16, 16, 16, 16, 16, 16, 16});
        with(norms, [](Call& c) { c.push[1] = 2; c.b[3].bytes = 19; }).expect("gate of 5 rows", "holds");
        with(norms, [](Call& c) { c.push[1] = 3; c.b[3].bytes = 3; }).expect("one gate", "holds");
        with(norms, [](Call& c) { c.push[1] = 3; c.b[3].ptr = (char*)c.b[3].ptr + 2; }).expect("one gate", "aligned");
        with(norms, [](Call& c) { c.b[5].ptr = (char*)c.b[1].ptr + 16; }).expect("h_out shifted on h", "h_out overlaps");
        with(norms, [](Call& c) { c.b[6].ptr = (char*)c.b[0].ptr + 16; }).expect("x shifted on y", "x overlaps y");
        with(norms, [](Call& c) { c.b[6].ptr = c.b[1].ptr; }).expect("x on h", "overlaps");
        with(norms, [](Call& c) { c.b[6].ptr = c.b[5].ptr; }).expect("x on h_out", "overlaps");
        with(norms, [](Call& c) { c.b[5].ptr = c.b[0].ptr; }).expect("h_out on y", "overlaps");
    }

    // 3 kv heads, 2 requests, 5 rows, pages of 16, stride 2
    const Call read{{at(pool), at(12), at(pool), at(12), at(16), at(8), at(12), at(5 * 768), at(5 * 768)}, {16, 2}, {3, 2, 5}, launch_kv_read_blocks};
    for (int g = 0; g < 3; g++) with(read, [=](Call& c) { c.groups[g] = 0; }).expect("empty grid", "groups");
    with(read, [](Call& c) { c.groups[0] = 1025; }).expect("heads", "heads");
    with(read, [](Call& c) { c.groups[1] = 65537; }).expect("requests", "requests");
    with(read, [](Call& c) { c.groups[2] = 0x80000000u; }).expect("rows", "rows");
    for (uint32_t page : {0u, 8u, 24u}) with(read, [=](Call& c) { c.push[0] = page; }).expect("page", "page");
    with(read, [](Call& c) { c.push[1] = 0; }).expect("stride", "stride");
    with(read, [](Call& c) { c.push[1] = 0xffffffffu; }).expect("a table of 2^35 bytes", "holds");
    short_and_misaligned(read, {16, 1, 16, 1, 4, 4, 4, 16, 16}, {0, 2});
    with(read, [](Call& c) { c.b[2].bytes -= 1; }).expect("V pool shorter", "same");
    with(read, [](Call& c) { c.b[0].bytes = c.b[2].bytes = 2048; }).expect("no block", "same");
    if (failures) return 1;
    printf("%d calls refused as they should be\n", calls);
    return 0;
}
