// Softmax scales that attn_blocks_e4m3_d128 refuses, on a machine without a device; the launcher returns SGB_ERR_VALIDATION (3) before it launches.
#include <cstdio>
#include <cstring>
#include <limits>
#include <string>

#include "sgb_kernels.h"

int main()
{
    const size_t pool = 4 * 3 * 2048, rows = 5 * 6 * 256;  // 3 kv heads, 2 query heads each, 2 requests, 5 tokens, page 16, stride 2
    int failures = 0;
    for (float scale : {0.0f, -1.0f, 0x1.000002p100f, std::numeric_limits<float>::max(), std::numeric_limits<float>::infinity(), std::numeric_limits<float>::quiet_NaN()}) {
        sgb::BufView b[10];
        const size_t bytes[10] = {rows, pool, 12, pool, 12, 16, 8, 12, rows, sgb::attn_blocks_work_bytes(148, 3, 2, 2, 5, 4)};
        for (int i = 0; i < 10; i++) b[i] = sgb::BufView{(void*)0x10000, bytes[i]};
        uint32_t push[6] = {0, 16, 2, 0, 2, 4};
        memcpy(push, &scale, 4);
        std::string err;
        uint64_t launches = 0;
        const sgb::LaunchArgs a{nullptr, b, push, {3, 2, 5}, nullptr, 148, 0, &err, &launches};
        const int r = sgb::launch_attn_blocks(a);
        if (r != 3 || launches != 0 || err.find("scale") == std::string::npos) {
            printf("scale %g: returned %d, \"%s\"\n", scale, r, err.c_str());
            failures++;
        }
    }
    return failures != 0;
}
