// Calls of the launchers around the batched attention in which something that is written shares memory with something else.  The first part asks the comparison itself;
// every call behind it differs from a good one in the place of one binding and has to be refused (SGB_ERR_VALIDATION, 3) before a device is touched.  No good call is
// made: its tensors are no memory.
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
    // binding i moved onto the last byte of the `bytes` at binding j (down to a multiple of 16), and onto its first
    void refused(int i, int j, size_t bytes, const char* text) const
    {
        for (size_t off : {(bytes - 1) / 16 * 16, (size_t)0}) {
            Call c = *this;
            c.b[i].ptr = (char*)b[j].ptr + off;
            std::string err;
            uint64_t launches = 0;
            LaunchArgs a{nullptr, c.b.data(), c.push.data(), {groups[0], groups[1], groups[2]}, nullptr, 148, 0, &err, &launches};
            const int r = fn(a);
            calls++;
            if (r != 3 || launches != 0 || err.find("overlap") == std::string::npos || err.find(text) == std::string::npos) {
                printf("%d on %d: returned %d, %llu launches, \"%s\", not \"%s\"\n", i, j, r, (unsigned long long)launches, err.c_str(), text);
                failures++;
            }
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
    next += (bytes + 4095) / 4096 * 4096 * 4;
    return BufView{(void*)p, bytes};
}
static Call with(Call c, const std::function<void(Call&)>& change)
{
    change(c);
    return c;
}

static void comparison()
{
    // 3 rows of 32 bytes, 100 apart, against every stretch of 1, 7 or 150 bytes around them, byte by byte
    std::string err;
    for (size_t bytes : {0, 1, 7, 150})
        for (size_t p = 700; p < 1400; p++) {
            bool meets = false;
            for (size_t row = 0; row < 3; row++)
                for (size_t x = 1000 + 100 * row; x < 1032 + 100 * row; x++) meets = meets || (x >= p && x < p + bytes);
            const BufView b[2] = {{(void*)1000, 232}, {(void*)p, bytes}};
            LaunchArgs a{nullptr, b, nullptr, {1, 1, 1}, nullptr, 148, 0, &err, nullptr};
            calls++;
            if ((need_apart(a, "k", 0, "out", 100, 32, 3, {{1, bytes, "in"}}) != 0) != meets) failures++, printf("rows against %zu bytes at %zu\n", bytes, p);
            if (need_apart(a, "k", 0, "out", 100, 32, 0, {{1, bytes, "in"}}) != 0 || need_apart(a, "k", 0, "out", 100, 0, 3, {{1, bytes, "in"}}) != 0) failures++, printf("nothing overlaps\n");
        }
}

static void rope()
{
    // 5 tokens, 48 dims that turn
    const Call angles{{at(24 * 8), at(20), at(5 * 48 * 4)}, {48, bits(1.0f)}, {5, 1, 1}, launch_rope_cos_sin};
    angles.refused(2, 0, 24 * 8, "frequencies");
    angles.refused(2, 1, 20, "positions");
    angles.refused(0, 2, 5 * 48 * 4, "frequencies");
    angles.refused(1, 2, 5 * 48 * 4, "positions");

    // 5 tokens, 6 and 2 heads of 80 dims, 48 of them turn; outputs with room behind a token's heads, which cos_sin may not begin in either as it is longer
    const Call rotate{{at(5 * 640 * 2), at(4 * 640 * 2 + 320), at(5 * 48 * 4), at(5 * 500 * 2), at(5 * 168 * 2)}, {80, 48, 1, 640, 640, 488, 168}, {6, 2, 5}, launch_rope_qk_f16};
    rotate.refused(2, 3, (4 * 488 + 480) * 2, "q_out overlaps cos_sin");
    rotate.refused(2, 4, (4 * 168 + 160) * 2, "k_out overlaps cos_sin");
    rotate.refused(3, 2, 5 * 48 * 4, "q_out overlaps cos_sin");
    rotate.refused(4, 2, 5 * 48 * 4, "k_out overlaps cos_sin");
}

static void pre_attention()
{
    // 5 tokens, 6 and 3 heads, 4 blocks, rows of 12 * 128 side by side
    const size_t pool = 4 * 3 * 2048, q_out = 5 * 6 * 256;
    const uint32_t row = 12 * 128;
    const Call pre{{at((4 * row + 768) * 2), at(512), at(q_out), at((4 * row + 384) * 2), at((4 * row + 384) * 2), at(512), at(5 * 64 * 4), at(20), at(pool), at(12), at(pool), at(12)},
                   {64, 0, 0, row, row, row, bits(1.0f)}, {6, 3, 5}, launch_qkv_norm_rope_append_blocks};
    const size_t sizes[12] = {(4 * row + 768) * 2, 512, q_out, (4 * row + 384) * 2, (4 * row + 384) * 2, 512, 5 * 64 * 4, 20, pool, 12, pool, 12};
    const char* names[12] = {"q", "q_w", "q_out", "k", "v", "k_w", "cos_sin", "slots", "k pool", "k exponents", "v pool", "v exponents"};
    for (int out : {2, 8, 9, 10, 11})
        for (int in = 0; in < 12; in++) {
            if (in == out) continue;
            pre.refused(in, out, sizes[out], names[in]);
            // an output onto what is read, or onto another output; a 12-byte one may stand between the rows of q, k and v
            if (out != 9 && out != 11) pre.refused(out, in, sizes[in], names[out]);
        }
    // where nothing turns, cos_sin is not looked at: what is refused here is the overlap
    with(pre, [](Call& c) { c.push[0] = 0; c.b[6].ptr = (char*)c.b[6].ptr + 4; }).refused(1, 2, q_out, "q_w");
    with(pre, [&](Call& c) { c.push[0] = 0; c.b[6] = c.b[2]; }).refused(1, 2, q_out, "q_w");
}

static void norms()
{
    for (int type = 0; type < 3; type++) {
        // 5 rows of 40
        const size_t n = 200, size = type == 2 ? 4 : 2;
        const Call block{{at(2 * n), at(size * n), at(160), at(160), at(160), at(size * n), at(2 * n)}, {1, 1, 0, bits(0.5f), bits(1e-6f)}, {40, 5, 1},
                         type == 0 ? launch_block_norms<__half> : type == 1 ? launch_block_norms<__nv_bfloat16> : launch_block_norms<float>};
        for (int out : {5, 6})
            for (int w : {2, 3, 4}) {
                block.refused(w, out, out == 5 ? size * n : 2 * n, w == 2 ? "w_post" : w == 3 ? "gate" : "w_pre");
                block.refused(out, w, 160, out == 5 ? "h_out" : "x");
            }
        with(block, [](Call& c) { c.push[1] = 2; }).refused(3, 6, 2 * n, "gate");
        with(block, [](Call& c) { c.push[1] = 3; }).refused(3, 5, size * n, "gate");
        with(block, [](Call& c) { c.push[0] = 2; c.push[1] = 0; c.push[3] = bits(1.0f); }).refused(4, 6, 2 * n, "w_pre");
    }
}

static void read()
{
    // 3 kv heads, 2 requests, 5 rows, pages of 16, stride 2
    const size_t pool = 4 * 3 * 2048, sizes[9] = {pool, 12, pool, 12, 16, 8, 12, 5 * 768, 5 * 768};
    const Call back{{at(pool), at(12), at(pool), at(12), at(16), at(8), at(12), at(5 * 768), at(5 * 768)}, {16, 2}, {3, 2, 5}, launch_kv_read_blocks};
    const char* names[9] = {"k pool", "k exponents", "v pool", "v exponents", "table", "from", "starts", "k", "v"};
    for (int out : {7, 8})
        for (int in = 0; in < 9; in++) {
            if (in == out) continue;
            back.refused(in, out, sizes[out], names[in]);
            back.refused(out, in, sizes[in], names[out]);
        }
}

int main()
{
    comparison();
    rope();
    pre_attention();
    norms();
    read();
    if (failures) return 1;
    printf("%d comparisons and calls as they should be\n", calls);
    return 0;
}
