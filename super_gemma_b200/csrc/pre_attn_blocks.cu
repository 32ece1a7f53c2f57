// The step between the QKV projections and the attention over the 8-bit cache of blocks.cuh, for the packed tokens of a batch:
//   q: RMS norm per head (q_w), rotation, f16        k: RMS norm (k_w), rotation, e4m3 into its slot        v: weightless norm, e4m3
// in one pass.  All of it is f32 between the loaded f16 and the one rounding at the end.
//
// The exponent of a tile needs no look at its values: a normed row of 128 has a 2-norm of at most sqrt(128), so that with weights w and
// a rotation whose (cos, sin) have length m
//   |v_i| <= sqrt(128),     |k_i| <= sqrt(128) max|w| m,
// and e is the least >= -15 with that bound <= 448 * 2^e.  The bound is loose by 2 to 8 where values are spread evenly, which costs nothing: e4m3
// keeps its four significant bits down to 2^-6 2^e, for values 2^-11 below the rows' root mean square (|w| of one size), and what
// is smaller is off by at most 2^-10 2^e.  So every token is written by itself, where kv_append_blocks_e4m3_d128 has to see a tile's tokens together and to
// round the earlier ones again as the maximum grows.  Its tiles may stand in the same pool: a tile that this call continues keeps its exponent if that is
// larger; if it is smaller (a tile of the other append with small values), the rows before are rounded again, once.
//
// Three bytes a value of k and v and four of q move: bound by bytes when there are many tokens, by a launch and the chain slots -> exponents when few.
#include "blocks.cuh"
#include "rope_layout.cuh"
#include "sgb_kernels.h"

namespace sgb {

namespace {

constexpr float RMS_EPS = 1e-6f;
constexpr float ROW_REACH = 11.336f;  // sqrt(128) = 11.3137, and 0.2 % for the rounding of norm, weight and rotation
constexpr int THREADS = 128;
constexpr uint32_t ROW_LANES = 8;  // of a row: a lane has two octets that turn with each other

struct PreArgs {
    const __half *q, *k, *v;
    const float *q_w, *k_w;
    const float2* cos_sin;
    const uint32_t* slots;
    __half* q_out;
    uint8_t* pool[2];
    int8_t* exps[2];
    uint32_t q_stride, k_stride, v_stride;  // values from token to token
    uint32_t n_q, n_kv, tokens, blocks, pairs, layout, slot_bits;
    float magnitude;
    uint32_t* status;
};

// Sixteen normed values as e4m3 of x * 2^-e.  |x| 2^-e stays below 448 but where an exponent is at its upper end: magnitudes count up to
// 61440 (every cached value is an f16 number), which is 240 of an exponent of 8.
__device__ __forceinline__ uint32_t quantise4(float a, float b, float c, float d)
{
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
__device__ __forceinline__ void write_e4m3(uint8_t* row, const RopePiece& at, float (&x)[8], float (&y)[8], int e)
{
    const float f = exp2_of(-e);
    if (e > 7) {  // (NaN stays)
        const float most = 61440.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            x[i] = x[i] > most ? most : x[i] < -most ? -most : x[i];
            y[i] = y[i] > most ? most : y[i] < -most ? -most : y[i];
        }
    }
    *reinterpret_cast<uint2*>(row + at.lo) = make_uint2(quantise4(x[0] * f, x[1] * f, x[2] * f, x[3] * f), quantise4(x[4] * f, x[5] * f, x[6] * f, x[7] * f));
    *reinterpret_cast<uint2*>(row + at.hi) = make_uint2(quantise4(y[0] * f, y[1] * f, y[2] * f, y[3] * f), quantise4(y[4] * f, y[5] * f, y[6] * f, y[7] * f));
}

template <bool PLUS_ONE>
__global__ void __launch_bounds__(THREADS) pre_attn_blocks_kernel(const __grid_constant__ PreArgs a)
{
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t lane = threadIdx.x & (ROW_LANES - 1), group = blockIdx.x * (THREADS / ROW_LANES) + threadIdx.x / ROW_LANES;
    const uint32_t token = group >> a.slot_bits, rows = a.n_q + 2 * a.n_kv;
    // a warp's four groups may have different tokens; those behind the last one go along without rows
    const bool live = token < a.tokens;
    const RopePiece at = rope_piece(a.layout, lane, 128, a.pairs);
    // The slot, and those of the fifteen tokens before it: two a lane.
    uint32_t slot = NO_SLOT, before[2] = {NO_SLOT, NO_SLOT};
    if (live) {
        slot = ld_global(a.slots + token);
#pragma unroll
        for (uint32_t j = 0; j < 2; j++)
            if (token >= 1 + lane + 8 * j) before[j] = ld_global(a.slots + token - 1 - lane - 8 * j);
    }
    const uint32_t in_tile = slot % TILE_TOK, previous = __shfl_sync(0xffffffffu, before[0], 0, ROW_LANES);
    const uint32_t back = in_tile ? in_tile - 1 : 0;  // the token that would be the tile's first, counted from the one before this
    const uint32_t opener0 = __shfl_sync(0xffffffffu, before[0], back & 7, ROW_LANES), opener1 = __shfl_sync(0xffffffffu, before[1], back & 7, ROW_LANES);
    const bool fresh = in_tile == 0 || (back < 8 ? opener0 : opener1) == slot - in_tile;  // the tile begins with this run
    const bool follows = in_tile != 0 && previous != NO_SLOT && previous + 1 == slot;
    bool placed = slot != NO_SLOT;
    if (placed && slot / TILE_TOK >= a.blocks) {
        report_error(a.status, DEV_ERR_BOUNDS, 631, slot, a.blocks);
        placed = false;
    } else if (placed && previous != NO_SLOT && previous / TILE_TOK == slot / TILE_TOK && previous + 1 != slot) {
        report_error(a.status, DEV_ERR_BOUNDS, 632, previous, slot);  // a tile's tokens stand in its order
        placed = false;
    }
    const bool some = slot != NO_SLOT;
    float c[8], s[8];
    if (at.turns && some) load_cos_sin(a.cos_sin + (size_t)token * a.pairs + at.pair, c, s);
    for (uint32_t r0 = (blockIdx.y << a.slot_bits); r0 < rows; r0 += gridDim.y << a.slot_bits) {
        const uint32_t r = r0 + (group & ((1u << a.slot_bits) - 1));
        const bool is_q = r < a.n_q, is_v = r >= a.n_q + a.n_kv, on = some && r < rows;
        const uint32_t head = is_q ? r : is_v ? r - a.n_q - a.n_kv : r - a.n_q;
        const __half* src = (is_q ? a.q + (size_t)token * a.q_stride : is_v ? a.v + (size_t)token * a.v_stride : a.k + (size_t)token * a.k_stride) + (size_t)head * 128;
        const uint4 u = ld_global_if(on, reinterpret_cast<const uint4*>(src + at.lo)), w = ld_global_if(on, reinterpret_cast<const uint4*>(src + at.hi));
        const size_t tile = (size_t)(slot / TILE_TOK) * a.n_kv + head;
        const int old = ld_global_if(on && placed && !is_q && !fresh, a.exps[is_v] + tile);
        float x[8], y[8];
        unpack_f16x8(u, x);
        unpack_f16x8(w, y);
        float ss = 0.0f, more = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            ss = fmaf(x[i], x[i], ss);
            more = fmaf(y[i], y[i], more);
        }
        ss += more;
#pragma unroll
        for (uint32_t d = 1; d < ROW_LANES; d <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        const float inv = rsqrtf(ss / 128.0f + RMS_EPS);
        float most = 1.0f;
        if (!is_v) {
            const float* wt = is_q ? a.q_w : a.k_w;
            float wx[8], wy[8];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float4 f = ld_global(reinterpret_cast<const float4*>(wt + at.lo) + j), g = ld_global(reinterpret_cast<const float4*>(wt + at.hi) + j);
                wx[4 * j] = f.x, wx[4 * j + 1] = f.y, wx[4 * j + 2] = f.z, wx[4 * j + 3] = f.w;
                wy[4 * j] = g.x, wy[4 * j + 1] = g.y, wy[4 * j + 2] = g.z, wy[4 * j + 3] = g.w;
            }
            most = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (PLUS_ONE) wx[i] += 1.0f, wy[i] += 1.0f;
                x[i] *= inv * wx[i];
                y[i] *= inv * wy[i];
                most = max3(most, fabsf(wx[i]), fabsf(wy[i]));
            }
            if (at.turns) rope_turn(a.layout, x, y, c, s);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] *= inv, y[i] *= inv;
        }
        if (is_q && on) {
            __half* to = a.q_out + ((size_t)token * a.n_q + head) * 128;
            *reinterpret_cast<uint4*>(to + at.lo) = pack_f16x8(x);
            *reinterpret_cast<uint4*>(to + at.hi) = pack_f16x8(y);
        }
#pragma unroll
        for (uint32_t d = 1; d < ROW_LANES; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        if (is_q || !on || !placed) continue;
        const int least = exponent_for(fminf(is_v ? ROW_REACH : most * ROW_REACH * a.magnitude, 61440.0f));
        const int e = fresh ? least : max(least, old);
        uint8_t* to = a.pool[is_v] + tile * TILE_BYTES;
        if (!follows) {  // the run's first token: nobody else writes the rows before it, nor the exponent
            if (!fresh && least > old) {
                const __half2 f = power_of_two(max(old - least, -24));
                for (uint32_t j = 0; j < in_tile; j++) {
                    uint4* p = reinterpret_cast<uint4*>(to + j * 128 + lane * 16);
                    *p = round_again(ld_global(p), f);
                }
            }
            if (lane == 0) a.exps[is_v][tile] = (int8_t)e;
        }
        write_e4m3(to + in_tile * 128, at, x, y, e);
    }
}

struct PushPre {
    uint32_t rot_dims, layout, plus_one, q_stride, k_stride, v_stride;
    float magnitude;
};

}  // namespace

// qkv_norm_rope_append_blocks_e4m3_d128: q, q_w, q_out, k, v, k_w, cos_sin, slots, k pool, k exps, v pool, v exps.
// push {rot_dims, layout, plus_one, strides of q, k, v, magnitude}.  grid [q heads, kv heads, tokens].
int launch_qkv_norm_rope_append_blocks(const LaunchArgs& a)
{
    PushPre p = *(const PushPre*)a.push;
    const uint32_t n_q = a.groups[0], n_kv = a.groups[1], tokens = a.groups[2];
    if (n_q == 0 || n_kv == 0 || tokens == 0) return fail_validation(a, "qkv_append_blocks: groups must be [q heads, kv heads, tokens]");
    if (n_q > 8192 || n_kv > 1024) return fail_validation(a, "qkv_append_blocks: at most 8192 q heads and 1024 kv heads");
    if (tokens > 1u << 26) return fail_validation(a, "qkv_append_blocks: at most 2^26 tokens");
    if (p.rot_dims > 128 || p.rot_dims % 16) return fail_validation(a, "qkv_append_blocks: rot_dims must be a multiple of 16 up to 128");
    if (p.layout >= ROPE_LAYOUTS) return fail_validation(a, "qkv_append_blocks: layout must be 0 (i, i + 64), 1 (i, i + rot/2) or 2 (2i, 2i + 1)");
    if (p.plus_one > 1) return fail_validation(a, "qkv_append_blocks: plus_one must be 0 or 1");
    if (!(p.magnitude > 0.0f) || !(p.magnitude <= 65504.0f)) return fail_validation(a, "qkv_append_blocks: magnitude must be positive, that of cos_sin's rows");
    uint32_t* strides[3] = {&p.q_stride, &p.k_stride, &p.v_stride};
    const uint32_t heads[3] = {n_q, n_kv, n_kv};
    const int at[3] = {0, 3, 4};
    const char* names[3] = {"q", "k", "v"};
    for (int i = 0; i < 3; i++) {
        const uint32_t width = heads[i] * 128;
        if (*strides[i] == 0) *strides[i] = width;
        if (*strides[i] % 8 || *strides[i] < width) return fail_validation(a, std::string("qkv_append_blocks: a token's stride must be a multiple of 8 values that holds its heads (") + names[i] + ")");
        if (int r = need_bytes(a, at[i], 2 * ((size_t)(tokens - 1) * *strides[i] + width), names[i])) return r;
    }
    if (int r = need_bytes(a, 1, 512, "q_w")) return r;
    if (int r = need_bytes(a, 2, 256 * (size_t)tokens * n_q, "q_out")) return r;
    if (int r = need_bytes(a, 5, 512, "k_w")) return r;
    if (int r = need_bytes(a, 6, 4 * (size_t)tokens * p.rot_dims, "cos_sin")) return r;
    if (int r = need_bytes(a, 7, 4 * (size_t)tokens, "slots")) return r;
    for (int i = 0; i < 3; i++) {  // q_out may be q
        const size_t out = 256 * (size_t)n_q;
        if (i == 0 && a.b[0].ptr == a.b[2].ptr && 2 * (size_t)p.q_stride == out) continue;
        if (rows_meet(a.b[at[i]].ptr, 2 * (size_t)*strides[i], 256 * (size_t)heads[i], a.b[2].ptr, out, out, tokens))
            return fail_validation(a, std::string("qkv_append_blocks: q_out overlaps ") + names[i]);
    }
    const size_t tile_row = (size_t)n_kv * TILE_BYTES, blocks = a.b[8].bytes / tile_row;
    if (blocks == 0 || a.b[10].bytes / tile_row != blocks)
        return fail_validation(a, "qkv_append_blocks: K and V pools must hold the same (non-zero) number of 16-token blocks");
    if (blocks > NO_SLOT / TILE_TOK) return fail_validation(a, "qkv_append_blocks: a pool holds less than 2^32 rows");
    if (int r = need_bytes(a, 9, blocks * n_kv, "k exponents")) return r;
    if (int r = need_bytes(a, 11, blocks * n_kv, "v exponents")) return r;
    if (int r = need_aligned(a, {16, 16, 16, 16, 16, 16, 16, 4, 16, 1, 16, 1})) return r;
    const uint32_t rows = n_q + 2 * n_kv;
    PreArgs k{(const __half*)a.b[0].ptr, (const __half*)a.b[3].ptr, (const __half*)a.b[4].ptr, (const float*)a.b[1].ptr, (const float*)a.b[5].ptr, (const float2*)a.b[6].ptr,
              (const uint32_t*)a.b[7].ptr, (__half*)a.b[2].ptr, {(uint8_t*)a.b[8].ptr, (uint8_t*)a.b[10].ptr}, {(int8_t*)a.b[9].ptr, (int8_t*)a.b[11].ptr},
              p.q_stride, p.k_stride, p.v_stride, n_q, n_kv, tokens, (uint32_t)blocks, p.rot_dims / 2, p.layout, 0, p.magnitude, a.status};
    const uint64_t per_sm = ((uint64_t)tokens * rows + a.sm_count - 1) / a.sm_count;
    const uint32_t each = per_sm <= 64 ? 1 : per_sm <= 384 ? 2 : 4;  // rows of a group of lanes
    while ((1u << k.slot_bits) < 32 && (each << k.slot_bits) < rows) k.slot_bits++;
    const uint64_t groups = (uint64_t)tokens << k.slot_bits;  // < 2^31
    const uint32_t per_token = (rows + (1u << k.slot_bits) - 1) >> k.slot_bits;
    const dim3 grid((unsigned)((groups * ROW_LANES + THREADS - 1) / THREADS), each == 1 && per_token < 1024 ? per_token : 1);
    const cudaError_t e = launch_dependent(p.plus_one ? pre_attn_blocks_kernel<true> : pre_attn_blocks_kernel<false>, grid, dim3(THREADS), 0, a.stream, k);
    ++*a.launches;
    return check_cuda(a, e, "qkv_norm_rope_append_blocks_e4m3_d128");
}

}  // namespace sgb
