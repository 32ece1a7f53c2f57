// The step between the QKV projections and the attention over the 8-bit cache of blocks.cuh, for the packed tokens of a batch:
//   q: RMS norm per head (q_w), rotation, f16        k: RMS norm (k_w), rotation, e4m3 into its slot        v: weightless norm, e4m3
// in one pass.  All of it is f32 between the loaded f16 and the one rounding at the end.
//
// The exponent of a tile needs no look at its values: a normed row of 128 has a 2-norm of at most sqrt(128), so that with weights w and
// a rotation whose (cos, sin) have length m
//   |v_i| <= sqrt(128),     |k_i| <= sqrt(128) max|w| m   where dim i turns,     sqrt(128) max|w|   where it does not
// (so that m counts as 1 at least unless the whole head turns), and e is the least >= -15 with that bound <= 448 * 2^e.  The bound is loose by 2 to 8 where values are spread evenly, which costs nothing: e4m3
// keeps its four significant bits down to 2^-6 2^e, for values 2^-11 below the rows' root mean square (|w| of one size), and what
// is smaller is off by at most 2^-10 2^e.  So every token is written by itself, where kv_append_blocks_e4m3_d128 has to see a tile's tokens together and to
// round the earlier ones again as the maximum grows.  Its tiles may stand in the same pool: a tile that this call continues keeps its exponent if that is
// larger; if it is smaller (a tile of the other append with small values), the rows before are rounded again, once.
//
// Three bytes a value of k and v and four of q move: bound by bytes when there are many tokens, by a launch and the chain slots -> exponents when few.
#include <algorithm>

#include "blocks.cuh"
#include "rope_layout.cuh"
#include "sgb_kernels.h"

namespace sgb {

namespace {

constexpr float RMS_EPS = 1e-6f;
constexpr float ROW_REACH = 11.336f;  // sqrt(128) = 11.3137, and 0.2 % for the rounding of norm, weight and rotation
constexpr int THREADS = 128;
constexpr uint32_t SLOTS = 4;      // rows of a group on their way, and one in use
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
    uint32_t n_q, n_kv, tokens, blocks, pairs, layout;
    uint32_t share_bits, each, step;        // groups of a token, rows of a group, from row to row of it
    float plus, longest;  // plus: 1 where weights are 1 + w; longest: what a rotation, or a dim's staying, multiplies a row's bound by
    uint32_t* status;
};

// A lane's eight pairs, a[j] = (a_2j, a_2j+1) and b likewise: the two octets of its piece, or with NEXT (layout 2) their even and their odd
// dims.  Which register a value comes to is all that the layouts differ in.
struct Pairs {
    float2 a[4], b[4];
};
template <bool NEXT>
__device__ __forceinline__ Pairs unpack_pairs(const uint4& lo, const uint4& hi)
{
    const uint32_t x[4] = {lo.x, lo.y, lo.z, lo.w}, y[4] = {hi.x, hi.y, hi.z, hi.w};
    Pairs p;
    float2 f[4], g[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        f[j] = __half22float2(as_half2(x[j]));
        g[j] = __half22float2(as_half2(y[j]));
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2* from = j < 2 ? f + 2 * j : g + 2 * (j - 2);
        p.a[j] = NEXT ? make_float2(from[0].x, from[1].x) : f[j];
        p.b[j] = NEXT ? make_float2(from[0].y, from[1].y) : g[j];
    }
    return p;
}
template <bool NEXT>
__device__ __forceinline__ void write_f16(__half* row, const RopePiece& at, const Pairs& p)
{
    uint32_t x[4], y[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if constexpr (NEXT) {
            uint32_t* to = j < 2 ? x + 2 * j : y + 2 * (j - 2);
            to[0] = pack_half2(p.a[j].x, p.b[j].x);
            to[1] = pack_half2(p.a[j].y, p.b[j].y);
        } else {
            x[j] = pack_half2(p.a[j].x, p.a[j].y);
            y[j] = pack_half2(p.b[j].x, p.b[j].y);
        }
    }
    *reinterpret_cast<uint4*>(row + at.lo) = make_uint4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<uint4*>(row + at.hi) = make_uint4(y[0], y[1], y[2], y[3]);
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d)
{
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}
// Values times 2^-e already.
template <bool NEXT>
__device__ __forceinline__ void write_e4m3(uint8_t* row, const RopePiece& at, const Pairs& p)
{
    const float2 *a = p.a, *b = p.b;
    if constexpr (NEXT) {
        *reinterpret_cast<uint2*>(row + at.lo) = make_uint2(e4m3x4(a[0].x, b[0].x, a[0].y, b[0].y), e4m3x4(a[1].x, b[1].x, a[1].y, b[1].y));
        *reinterpret_cast<uint2*>(row + at.hi) = make_uint2(e4m3x4(a[2].x, b[2].x, a[2].y, b[2].y), e4m3x4(a[3].x, b[3].x, a[3].y, b[3].y));
    } else {
        *reinterpret_cast<uint2*>(row + at.lo) = make_uint2(e4m3x4(a[0].x, a[0].y, a[1].x, a[1].y), e4m3x4(a[2].x, a[2].y, a[3].x, a[3].y));
        *reinterpret_cast<uint2*>(row + at.hi) = make_uint2(e4m3x4(b[0].x, b[0].y, b[1].x, b[1].y), e4m3x4(b[2].x, b[2].y, b[3].x, b[3].y));
    }
}

// Weight and rotation of a token's heads in one: (a, b) -> (a A - b B, b C + a E) with A = w_a c, B = w_b s, C = w_b c, E = w_a s.
struct Turn {
    float2 A[4], minus_B[4], C[4], E[4];
};
__device__ __forceinline__ void apply(const Turn& t, bool turns, Pairs& p)
{
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 a = p.a[j], b = p.b[j];
        p.a[j] = mul2_rn(a, t.A[j]);
        p.b[j] = mul2_rn(b, t.C[j]);
        if (turns) {  // (a partner that is no number stays out of what does not turn)
            p.a[j] = fma2_rn(b, t.minus_B[j], p.a[j]);
            p.b[j] = fma2_rn(a, t.E[j], p.b[j]);
        }
    }
}

// 2^share_bits groups of eight lanes share the rows of a token (q heads, k heads, v heads in this order).  What is the same for
// a token's heads (the slot, the rotation with its weights, the exponents' bound) is made once a group.  Groups of a warp may have different rows to do, so that a
// group exchanges values within its own lanes only.  23931 tokens of 32 q and 16 kv heads (17 prompts) take 112 to 115 us, 6.2 TB/s, 0.94 of the copy rate (side by side
// with others of its kind 104.7); with rows asked for one ahead into registers 143, two ahead 131 (128 registers, four CTAs an SM), weights and rotation applied one after the other to every row 165.
template <bool NEXT>
__global__ void __launch_bounds__(THREADS, 4) pre_attn_blocks_kernel(const __grid_constant__ PreArgs a)
{
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t lane = threadIdx.x & (ROW_LANES - 1), group = blockIdx.x * (THREADS / ROW_LANES) + threadIdx.x / ROW_LANES;
    const uint32_t mask = 0xffu << (threadIdx.x & 24);
    const uint32_t token = group >> a.share_bits, share = group & ((1u << a.share_bits) - 1);
    if (token >= a.tokens) return;
    const RopePiece at = rope_piece(a.layout, lane, 128, a.pairs);
    // The slot, and those of the fifteen tokens before it: two a lane.
    const uint32_t slot = ld_global(a.slots + token);
    uint32_t before[2] = {NO_SLOT, NO_SLOT};
#pragma unroll
    for (uint32_t j = 0; j < 2; j++)
        if (token >= 1 + lane + 8 * j) before[j] = ld_global(a.slots + token - 1 - lane - 8 * j);
    const uint32_t end_q = a.n_q, end_k = a.n_q + a.n_kv, end = end_k + a.n_kv;
    uint32_t r = a.step == 1 ? share * a.each : share;
    const uint32_t stop = a.step == 1 ? min(end, r + a.each) : end;
    // Rows on their way: SLOTS places of 32 bytes a thread in shared memory, written and read by itself alone, so that nothing but its own copies is waited for.  A place
    // is written again when what was read from it has been used.
    __shared__ alignas(16) uint4 places[SLOTS][2][THREADS];
    const __half* const base_q = a.q + (size_t)token * a.q_stride + at.lo;
    const __half* const base_k = a.k + (size_t)token * a.k_stride + at.lo - (size_t)end_q * 128;  // (row 0 of all, were they keys)
    const __half* const base_v = a.v + (size_t)token * a.v_stride + at.lo - (size_t)end_k * 128;
    const uint32_t apart = at.hi - at.lo;
    uint32_t place = 0;
    const auto fetch = [&](uint32_t i, uint32_t to) {
        const __half* src = (i < end_q ? base_q : i < end_k ? base_k : base_v) + (size_t)i * 128;
        copy_async_if(i < stop, &places[to][0][threadIdx.x], src);
        copy_async_if(i < stop, &places[to][1][threadIdx.x], src + apart);
        copy_async_commit();
    };
#pragma unroll
    for (uint32_t j = 0; j + 1 < SLOTS; j++) fetch(r + j * a.step, j);
    const auto next = [&]() {  // row r
        copy_async_wait<SLOTS - 2>();
        const Pairs p = unpack_pairs<NEXT>(places[place][0][threadIdx.x], places[place][1][threadIdx.x]);
        fetch(r + (SLOTS - 1) * a.step, (place + SLOTS - 1) % SLOTS);
        place = (place + 1) % SLOTS;
        return p;
    };
    float c[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) c[i] = 1.0f, s[i] = 0.0f;
    if (at.turns && r < end_k) load_cos_sin(a.cos_sin + (size_t)token * a.pairs, at, c, s);
    float most = 0.0f;
    const auto turn_of = [&](const float* weights) {
        Turn t;
        float4 u[4];
#pragma unroll
        for (int j = 0; j < 4; j++) u[j] = ld_global(reinterpret_cast<const float4*>(weights + (j < 2 ? at.lo : at.hi)) + (j & 1));
        const float w[16] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w, u[2].x, u[2].y, u[2].z, u[2].w, u[3].x, u[3].y, u[3].z, u[3].w};
        most = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float2 wa = NEXT ? make_float2(w[4 * j], w[4 * j + 2]) : make_float2(w[2 * j], w[2 * j + 1]);
            float2 wb = NEXT ? make_float2(w[4 * j + 1], w[4 * j + 3]) : make_float2(w[8 + 2 * j], w[8 + 2 * j + 1]);
            wa = add2_rn(wa, make_float2(a.plus, a.plus));
            wb = add2_rn(wb, make_float2(a.plus, a.plus));
            most = max3(most, fmaxf(fabsf(wa.x), fabsf(wa.y)), fmaxf(fabsf(wb.x), fabsf(wb.y)));
            const float2 cc = make_float2(c[2 * j], c[2 * j + 1]), ss = make_float2(s[2 * j], s[2 * j + 1]);
            t.A[j] = mul2_rn(wa, cc);
            t.C[j] = mul2_rn(wb, cc);
            t.E[j] = mul2_rn(wa, ss);
            t.minus_B[j] = mul2_rn(wb, make_float2(-ss.x, -ss.y));
        }
        return t;
    };
    const auto inverse_rms = [&](const Pairs& p) {
        float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < 4; j++) ss = fma2_rn(p.b[j], p.b[j], fma2_rn(p.a[j], p.a[j], ss));
        float sum = ss.x + ss.y;
#pragma unroll
        for (uint32_t d = 1; d < ROW_LANES; d <<= 1) sum += __shfl_xor_sync(mask, sum, d);
        return rsqrtf(fmaf(sum, 1.0f / 128.0f, RMS_EPS));
    };
    const auto scale = [&](Pairs& p, float by) {
        const float2 f = make_float2(by, by);
#pragma unroll
        for (int j = 0; j < 4; j++) p.a[j] = mul2_rn(p.a[j], f), p.b[j] = mul2_rn(p.b[j], f);
    };
    Turn turn;
    if (r < end_q) turn = turn_of(a.q_w);

    if (slot == NO_SLOT) {
        copy_async_wait<0>();  // nothing lands in the memory of whoever comes next
        return;
    }
    const uint32_t in_tile = slot % TILE_TOK, previous = __shfl_sync(mask, before[0], 0, ROW_LANES);
    const uint32_t back = in_tile ? in_tile - 1 : 0;  // the token that would be the tile's first, counted from the one before this
    const uint32_t opener0 = __shfl_sync(mask, before[0], back & 7, ROW_LANES), opener1 = __shfl_sync(mask, before[1], back & 7, ROW_LANES);
    const bool fresh = in_tile == 0 || (back < 8 ? opener0 : opener1) == slot - in_tile;  // the tile begins with this run
    const bool follows = in_tile != 0 && previous != NO_SLOT && previous + 1 == slot;
    bool placed = true;
    if (slot / TILE_TOK >= a.blocks) {
        report_error(a.status, DEV_ERR_BOUNDS, 631, slot, a.blocks);
        placed = false;
    } else if (previous != NO_SLOT && previous / TILE_TOK == slot / TILE_TOK && previous + 1 != slot) {
        report_error(a.status, DEV_ERR_BOUNDS, 632, previous, slot);  // a tile's tokens stand in its order
        placed = false;
    }

    for (; r < min(end_q, stop); r += a.step) {
        Pairs p = next();
        const float inv = inverse_rms(p);
        apply(turn, at.turns, p);
        scale(p, inv);
        write_f16<NEXT>(a.q_out + ((size_t)token * a.n_q + r) * 128, at, p);
    }
    if (!placed) {
        copy_async_wait<0>();
        return;
    }

    // Rows [r, last) of one side into the cache; `least`: the exponent that holds them all.
    const size_t tile0 = (size_t)(slot / TILE_TOK) * a.n_kv;
    const auto append = [&](int side, uint32_t first, uint32_t last, int least, const auto& turned) {
        if (r >= last) return;
        uint8_t* const pool = a.pool[side] + tile0 * TILE_BYTES;
        int8_t* const exps = a.exps[side] + tile0;
        int old = ld_global_if(!fresh, exps + (r - first));
        for (; r < last; r += a.step) {
            Pairs p = next();
            const uint32_t head = r - first;
            const int had = old, e = fresh ? least : max(least, had);
            old = ld_global_if(!fresh && r + a.step < last, exps + head + a.step);
            const float inv = inverse_rms(p);
            turned(p);
            uint8_t* to = pool + (size_t)head * TILE_BYTES;
            if (!follows) {  // the run's first token: nobody else writes the rows before it, nor the exponent
                if (!fresh && least > had) {
                    const __half2 f = power_of_two(max(had - least, -24));
                    for (uint32_t j = 0; j < in_tile; j++) {
                        uint4* q = reinterpret_cast<uint4*>(to + j * 128 + lane * 16);
                        *q = round_again(ld_global(q), f);
                    }
                }
                if (lane == 0) exps[head] = (int8_t)e;
            }
            if (e > 7) {  // magnitudes count up to 61440, which is 240 of an exponent of 8 (NaN stays)
                scale(p, inv);
                const auto cut = [](float2& v) {
                    v.x = v.x > 61440.0f ? 61440.0f : v.x < -61440.0f ? -61440.0f : v.x;
                    v.y = v.y > 61440.0f ? 61440.0f : v.y < -61440.0f ? -61440.0f : v.y;
                };
#pragma unroll
                for (int j = 0; j < 4; j++) cut(p.a[j]), cut(p.b[j]);
                scale(p, exp2_of(-e));
            } else {
                scale(p, inv * exp2_of(-e));
            }
            write_e4m3<NEXT>(to + in_tile * 128, at, p);
        }
    };
    if (r < min(end_k, stop)) {
        turn = turn_of(a.k_w);
#pragma unroll
        for (uint32_t d = 1; d < ROW_LANES; d <<= 1) most = fmaxf(most, __shfl_xor_sync(mask, most, d));
        append(0, end_q, min(end_k, stop), exponent_for(fminf(most * ROW_REACH * a.longest, 61440.0f)), [&](Pairs& p) { apply(turn, at.turns, p); });
    }
    append(1, end_k, stop, exponent_for(ROW_REACH), [](Pairs&) {});
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
    if (int r = need_aligned(a, {16, 16, 16, 16, 16, 16, p.rot_dims ? 16u : 1u, 4, 16, 1, 16, 1})) return r;
    // nothing else that is written stands over anything else either
    const char* kernel = "qkv_append_blocks";
    const Other q_w{1, 512, "q_w"}, k_w{5, 512, "k_w"}, cos_sin{6, 4 * (size_t)tokens * p.rot_dims, "cos_sin"}, slots{7, 4 * (size_t)tokens, "slots"}, k_pool{8, blocks * tile_row, "k pool"},
        k_exps{9, blocks * n_kv, "k exponents"}, v_pool{10, blocks * tile_row, "v pool"}, v_exps{11, blocks * n_kv, "v exponents"};
    const auto dense = [&](const Other& out, std::initializer_list<Other> others) { return need_apart(a, kernel, out.binding, out.name, out.bytes, out.bytes, 1, others); };
    if (int r = dense({2, 256 * (size_t)tokens * n_q, "q_out"}, {q_w, k_w, cos_sin, slots, k_pool, k_exps, v_pool, v_exps})) return r;
    for (int i = 0; i < 3; i++)
        if (int r = need_apart(a, kernel, at[i], names[i], 2 * (size_t)*strides[i], 256 * (size_t)heads[i], tokens, {k_pool, k_exps, v_pool, v_exps})) return r;
    if (int r = dense(k_pool, {q_w, k_w, cos_sin, slots, k_exps, v_pool, v_exps})) return r;
    if (int r = dense(v_pool, {q_w, k_w, cos_sin, slots, k_exps, v_exps})) return r;
    if (int r = dense(k_exps, {q_w, k_w, cos_sin, slots, v_exps})) return r;
    if (int r = dense(v_exps, {q_w, k_w, cos_sin, slots})) return r;
    const uint32_t rows = n_q + 2 * n_kv;
    PreArgs k{(const __half*)a.b[0].ptr, (const __half*)a.b[3].ptr, (const __half*)a.b[4].ptr, (const float*)a.b[1].ptr, (const float*)a.b[5].ptr, (const float2*)a.b[6].ptr,
              (const uint32_t*)a.b[7].ptr, (__half*)a.b[2].ptr, {(uint8_t*)a.b[8].ptr, (uint8_t*)a.b[10].ptr}, {(int8_t*)a.b[9].ptr, (int8_t*)a.b[11].ptr},
              p.q_stride, p.k_stride, p.v_stride, n_q, n_kv, tokens, (uint32_t)blocks, p.rot_dims / 2, p.layout, 0, 0, 0, p.plus_one ? 1.0f : 0.0f,
              p.rot_dims == 128 ? p.magnitude : std::max(p.magnitude, 1.0f), a.status};
    // Groups of a token.  What a group makes for its token costs it as much as two rows, so that as few as give each SM 256 threads to do are best (us, one launch after the
    // other, at 128 | 256 | 512 threads: 512 tokens of 32 q and 16 kv heads 5.0 | 4.4 | 5.5, 440 of them 5.0 | 4.4 | 5.2, 200 3.3 | 3.5 | 4.4); but sixteen rows a group at
    // most: 23931 tokens take 122 with 8, 112 with 16, 116 with 32 of them, about 5000 tokens 31.5, 30.5, 34.7.
    while (k.share_bits < 10 && (1u << k.share_bits) < rows && (((uint64_t)tokens << k.share_bits) * ROW_LANES < 256ull * a.sm_count || rows > 16u << k.share_bits)) k.share_bits++;
    // An SM has 512 threads at a time; up to half as many again wait for two rounds, where shorter groups take three of half their length
    // (us, two | three: tokens of 8 q and 2 kv heads, floor 9.4 us of bytes 20.9 | 15.7, 11.3 us 20.5 | 16.9; of 32 and 16, 12.2 us 18.9 | 18.2; of 16 and 2, 10.6 us 16.3 | 17.2).
    const uint64_t threads = ((uint64_t)tokens << k.share_bits) * ROW_LANES;
    if (threads > 512ull * a.sm_count && threads <= 768ull * a.sm_count && rows > 8u << k.share_bits) k.share_bits++;
    // A group of few rows has them one after the other, most of them of one kind; with more, a warp's groups would read kilobytes apart at a time, and they take them in turn
    // (512 tokens, four rows each: 4.4 us, in turn 5.1; 23931 tokens, sixteen each: 202, in turn 112).
    k.each = (rows + (1u << k.share_bits) - 1) >> k.share_bits;
    k.step = k.each <= 4 ? 1 : 1u << k.share_bits;
    const uint64_t groups = (uint64_t)tokens << k.share_bits;
    const dim3 grid((unsigned)((groups * ROW_LANES + THREADS - 1) / THREADS));
    const cudaError_t e = launch_dependent(p.layout == 2 ? pre_attn_blocks_kernel<true> : pre_attn_blocks_kernel<false>, grid, dim3(THREADS), 0, a.stream, k);
    ++*a.launches;
    return check_cuda(a, e, "qkv_norm_rope_append_blocks_e4m3_d128");
}

}  // namespace sgb
