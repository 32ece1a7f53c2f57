// Rotary positions of the packed tokens of a step: rows of cosines and sines from the tokens' positions, once a step for all layers, and
// the rotation of queries and keys by those rows for heads that need no norm (with norms and the append: pre_attn_blocks.cu).
//
// rope_cos_sin:  row[t][i] = m * (cos a, sin a),  a = p_t * f_i       p: 32-bit whole numbers, a negative one turns back
// rope_qk_f16:   (x, y) -> (x c - y s, y c + x s)                     pair i of a head, coupled as `layout` says (rope_layout.cuh)
#include <cmath>

#include "../../include/sgattn.h"
#include "rope_layout.cuh"
#include "sgb_kernels.h"

namespace sgb {

namespace {

constexpr int ROW_THREADS = 256;
constexpr uint32_t MOST_ROT = 1024;

// ---- rows of cosines and sines ---------------------------------------------------------------------------------------------------
// Angles are counted in turns, as 64-bit fractions of one: F = f / 2 pi mod 1 in units of 2^-64, made of the f64 frequency and 1 / 2 pi in two f64 (hi + lo),
// so that the whole turns of p F fall off by themselves for every 32-bit p.  The nearest quarter turn goes into signs and an exchange of sine and cosine, the rest, an
// eighth of a turn at most, into their Taylor series up to x^9 and x^10 (cut off below 2 * 10^-9).  The rest becomes an f32 number with the digits of both of its words: the upper one alone is
// good to 2^-32 of a turn, which is 10^-3 of the sine of a slow pair (theta 1e6) in the first tokens.
// Integers instead of f64 sums and reductions: those kept the units that convert between formats busy, 5.8 us for 32768 rows of 64 pairs where these took 3.4 (launches side by side; 4.3 one after the
// other, 4.5 since the lower words count too).
// A thread makes two pairs (16 bytes) of ROWS tokens.
constexpr double INV_2PI_HI = 0.15915494309189535, INV_2PI_LO = -9.839338337591243e-18;

__device__ __forceinline__ uint64_t fraction_of_turn(double f)
{
    const double hi = f * INV_2PI_HI, lo = fma(f, INV_2PI_HI, -hi) + f * INV_2PI_LO, unit = 18446744073709551616.0;
    return (uint64_t)__double2ll_rn((hi - rint(hi)) * unit) + (uint64_t)__double2ll_rn(lo * unit);
}
// Cosines and sines of two angles of t 2^-64 turns each, times m.
__device__ __forceinline__ float4 cos_sin_of(uint64_t t0, uint64_t t1, float2 m)
{
    const uint32_t upper[2] = {(uint32_t)(t0 >> 32), (uint32_t)(t1 >> 32)};
    const uint32_t quarter[2] = {(upper[0] + 0x20000000u) >> 30, (upper[1] + 0x20000000u) >> 30};
    // what lies beyond the quarter, in 2^-32 turns: the upper word less 1, and 1 to 2 with the lower word's first 23 bits behind the point
    const float2 whole = make_float2((float)(int)(upper[0] - (quarter[0] << 30) - 1), (float)(int)(upper[1] - (quarter[1] << 30) - 1));
    const float2 part = make_float2(__uint_as_float(__funnelshift_r((uint32_t)t0, 0x7f, 9)), __uint_as_float(__funnelshift_r((uint32_t)t1, 0x7f, 9)));
    const float radian = 1.4629180792671596e-9f;  // 2 pi 2^-32
    const float2 x = mul2_rn(add2_rn(whole, part), make_float2(radian, radian)), z = mul2_rn(x, x);
    const auto both = [](float v) { return make_float2(v, v); };
    float2 c = both(-1.0f / 3628800.0f), s = both(1.0f / 362880.0f);
    c = fma2_rn(c, z, both(1.0f / 40320.0f));
    c = fma2_rn(c, z, both(-1.0f / 720.0f));
    c = fma2_rn(c, z, both(1.0f / 24.0f));
    c = fma2_rn(c, z, both(-0.5f));
    c = mul2_rn(fma2_rn(c, z, both(1.0f)), m);
    s = fma2_rn(s, z, both(-1.0f / 5040.0f));
    s = fma2_rn(s, z, both(1.0f / 120.0f));
    s = fma2_rn(s, z, both(-1.0f / 6.0f));
    s = mul2_rn(fma2_rn(mul2_rn(s, z), x, x), m);
    // a quarter turn on: (c, s) -> (-s, c)
    const auto place = [](uint32_t q, float c, float s) {
        const float a = q & 1 ? s : c, b = q & 1 ? c : s;
        return make_float2(__uint_as_float(__float_as_uint(a) ^ ((q + 1) >> 1 << 31)), __uint_as_float(__float_as_uint(b) ^ (q >> 1 << 31)));
    };
    const float2 first = place(quarter[0], c.x, s.x), second = place(quarter[1], c.y, s.y);
    return make_float4(first.x, first.y, second.x, second.y);
}

template <int ROWS>
__global__ void __launch_bounds__(ROW_THREADS) rope_cos_sin_kernel(const double* freqs, const int* positions, float4* __restrict__ cos_sin, float magnitude,
                                                                   uint32_t tokens, uint32_t per_row, uint32_t rows_here)
{
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t row = threadIdx.x / per_row, at = threadIdx.x - row * per_row;
    if (row >= rows_here) return;
    const uint64_t first = (uint64_t)blockIdx.x * (rows_here * ROWS) + row;
    const double f[2] = {ld_global(freqs + 2 * at), ld_global(freqs + 2 * at + 1)};
    uint32_t p[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        p[i] = 0;
        if (first + i * rows_here < tokens) p[i] = (uint32_t)ld_global(positions + first + i * rows_here);
    }
    const uint64_t turn[2] = {fraction_of_turn(f[0]), fraction_of_turn(f[1])};
    const float2 m = make_float2(magnitude + (float)(f[0] - f[0]), magnitude + (float)(f[1] - f[1]));  // a frequency that is no number gives rows that are none
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const uint64_t t = first + i * rows_here;
        if (t >= tokens) return;
        const uint64_t turns = (uint64_t)(int64_t)(int)p[i];  // a negative position's sign falls off above 2^64 too
        cos_sin[t * per_row + at] = cos_sin_of(turns * turn[0], turns * turn[1], m);
    }
}

struct PushCosSin {
    uint32_t rot_dims;
    float magnitude;
};

// ---- rotation --------------------------------------------------------------------------------------------------------------------
// A thread has one piece of 16 dims (two octets of a layout's pairs) of ROWS heads of a token, all of them asked for before the first
// is turned; the token's eight cosines and sines stay in its registers.  Two bytes read and two written per value: bound by bytes (8192
// tokens of 32 and 16 heads of 128, neighbours coupled, out of packed rows: 31.8 us, 6.5 TB/s).
struct RotateArgs {
    const __half* src[2];  // q, k
    __half* dst[2];
    uint32_t src_stride[2], dst_stride[2];  // values from token to token
    uint32_t heads[2];
    const float2* cos_sin;
    uint32_t tokens, head_dim, pairs, layout, pieces;  // pieces of a head that are touched
    uint32_t slots;                                    // threads of a token that share a piece's heads
};

template <int ROWS>
__global__ void __launch_bounds__(ROW_THREADS) rope_qk_kernel(const __grid_constant__ RotateArgs a)
{
    pdl_wait();
    pdl_launch_dependents();
    const uint32_t g = blockIdx.x * ROW_THREADS + threadIdx.x;  // the host checks that they fit
    const uint32_t per_token = a.pieces * a.slots, token = g / per_token;
    if (token >= a.tokens) return;
    const uint32_t in_token = g - token * per_token, slot = in_token / a.pieces, piece = in_token - slot * a.pieces;
    const RopePiece at = rope_piece(a.layout, piece, a.head_dim, a.pairs);
    const uint32_t all = a.heads[0] + a.heads[1];
    uint4 lo[ROWS], hi[ROWS];
    auto where = [&](uint32_t h, bool from) -> size_t {
        const bool k = h >= a.heads[0];
        return (size_t)token * (from ? a.src_stride[k] : a.dst_stride[k]) + (size_t)(k ? h - a.heads[0] : h) * a.head_dim;
    };
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const uint32_t h = slot + i * a.slots;
        lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
        if (h < all) {
            const __half* src = a.src[h >= a.heads[0]] + where(h, true);
            lo[i] = ld_global(reinterpret_cast<const uint4*>(src + at.lo));
            hi[i] = ld_global(reinterpret_cast<const uint4*>(src + at.hi));
        }
    }
    float c[8], s[8];
    if (at.turns) load_cos_sin(a.cos_sin + (size_t)token * a.pairs, at, c, s);
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const uint32_t h = slot + i * a.slots;
        if (h >= all) return;
        if (at.turns) {
            float x[8], y[8];
            unpack_f16x8(lo[i], x);
            unpack_f16x8(hi[i], y);
            rope_turn(a.layout, x, y, c, s);
            lo[i] = pack_f16x8(x);
            hi[i] = pack_f16x8(y);
        }
        __half* dst = a.dst[h >= a.heads[0]] + where(h, false);
        *reinterpret_cast<uint4*>(dst + at.lo) = lo[i];
        *reinterpret_cast<uint4*>(dst + at.hi) = hi[i];
    }
}

struct PushRotate {
    uint32_t head_dim, rot_dims, layout, stride[4];
};

}  // namespace

// Radians a position: f_i = theta^(-2 i / dims), and for contexts `factor` times the trained length a share of f_i / factor that grows
// from the pairs that turn often to those that turn rarely over that length.
int rope_frequencies(const sgb_rope_scaling& r, double* out, std::string* err)
{
    const auto bad = [&](const char* text) {
        *err = std::string("sgb_rope_frequencies: ") + text;
        return (int)SGB_ERR_VALIDATION;
    };
    const auto positive = [](double v) { return v > 0.0 && std::isfinite(v); };
    if (r.pairs == 0 || r.pairs > MOST_ROT / 2) return bad("pairs must be 1..512");
    if (r.dims < 2 * r.pairs) return bad("dims must be at least twice the pairs");
    if (!positive(r.theta) || r.theta <= 1.0) return bad("theta must be above 1");
    if (r.kind > SGB_ROPE_BY_PAIRS) return bad("kind must be one of SGB_ROPE_*");
    if (r.kind != SGB_ROPE_PLAIN && !positive(r.factor)) return bad("factor must be positive");
    const double turn = 2.0 * M_PI;
    double first = 0.0, last = 0.0;
    if (r.kind == SGB_ROPE_BY_TURNS || r.kind == SGB_ROPE_BY_PAIRS) {
        if (!positive(r.trained)) return bad("trained must be the length in tokens that the model was trained on");
        if (!positive(r.slow) || !positive(r.fast) || r.fast <= r.slow) return bad("turns must be 0 < slow < fast");
        const auto pair_of = [&](double turns) { return r.dims * std::log(r.trained / (turns * turn)) / (2.0 * std::log(r.theta)); };
        first = std::fmax(std::floor(pair_of(r.fast)), 0.0);
        last = std::fmin(std::ceil(pair_of(r.slow)), r.dims - 1.0);
    }
    for (uint32_t i = 0; i < r.pairs; i++) {
        const double f = std::pow(r.theta, -2.0 * i / r.dims);
        double keep = 1.0;  // the share that is not slowed down
        if (r.kind == SGB_ROPE_LINEAR) keep = 0.0;
        if (r.kind == SGB_ROPE_BY_TURNS) keep = (r.trained * f / turn - r.slow) / (r.fast - r.slow);
        if (r.kind == SGB_ROPE_BY_PAIRS) keep = last > first ? 1.0 - (i - first) / (last - first) : (i > first ? 0.0 : 1.0);
        keep = std::fmin(std::fmax(keep, 0.0), 1.0);
        out[i] = r.kind == SGB_ROPE_PLAIN ? f : keep * f + (1.0 - keep) * (f / r.factor);
    }
    return SGB_OK;
}

// rope_cos_sin: freqs f64 [rot / 2], positions i32 [N], cos_sin f32 [N x rot/2 x 2].  push {rot_dims, magnitude}.  grid [N].
int launch_rope_cos_sin(const LaunchArgs& a)
{
    const PushCosSin p = *(const PushCosSin*)a.push;
    const uint32_t tokens = a.groups[0];
    if (tokens == 0) return fail_validation(a, "rope_cos_sin: groups[0] (tokens) must be > 0");
    if (p.rot_dims == 0 || p.rot_dims % 16 || p.rot_dims > MOST_ROT) return fail_validation(a, "rope_cos_sin: rot_dims must be a multiple of 16 up to 1024");
    if (!(p.magnitude > 0.0f) || !std::isfinite(p.magnitude)) return fail_validation(a, "rope_cos_sin: magnitude must be positive");
    if (int r = need_bytes(a, 0, 4 * (size_t)p.rot_dims, "frequencies")) return r;
    if (int r = need_bytes(a, 1, 4 * (size_t)tokens, "positions")) return r;
    if (int r = need_bytes(a, 2, 4 * (size_t)tokens * p.rot_dims, "cos_sin")) return r;
    if (int r = need_aligned(a, {8, 4, 16})) return r;
    const size_t rows = 4 * (size_t)tokens * p.rot_dims;
    if (int r = need_apart(a, "rope_cos_sin", 2, "cos_sin", rows, rows, 1, {{0, 4 * (size_t)p.rot_dims, "frequencies"}, {1, 4 * (size_t)tokens, "positions"}})) return r;
    const uint32_t per_row = p.rot_dims / 4, rows_here = ROW_THREADS / per_row;
    const bool many = (uint64_t)tokens * per_row > 2048ull * a.sm_count;  // (ROWS 8 | 4 | 1, 20000 rows of 64 pairs: 4.4 | 3.7 us, 32768 4.5 | 4.2 | 6.2, 62500 7.5 | 7.9)
    const uint32_t each = rows_here * (many ? 8 : 1);
    const cudaError_t e = launch_dependent(many ? rope_cos_sin_kernel<8> : rope_cos_sin_kernel<1>, dim3((tokens + each - 1ull) / each), dim3(ROW_THREADS), 0, a.stream,
                                           (const double*)a.b[0].ptr, (const int*)a.b[1].ptr, (float4*)a.b[2].ptr, p.magnitude, tokens, per_row, rows_here);
    ++*a.launches;
    return check_cuda(a, e, "rope_cos_sin");
}

// rope_qk_f16: q, k, cos_sin, q_out, k_out.  push {head_dim, rot_dims, layout, strides of q, k, q_out, k_out}.  grid [q heads, kv heads, tokens].
int launch_rope_qk_f16(const LaunchArgs& a)
{
    PushRotate p = *(const PushRotate*)a.push;
    const uint32_t heads[2] = {a.groups[0], a.groups[1]}, tokens = a.groups[2];
    if (heads[0] == 0 || tokens == 0) return fail_validation(a, "rope_qk: groups must be [q heads > 0, kv heads, tokens > 0]");
    if (heads[0] > 4096 || heads[1] > 4096) return fail_validation(a, "rope_qk: at most 4096 heads");
    if (p.head_dim == 0 || p.head_dim % 16 || p.head_dim > MOST_ROT) return fail_validation(a, "rope_qk: head_dim must be a multiple of 16 up to 1024");
    if (p.rot_dims == 0 || p.rot_dims % 16 || p.rot_dims > p.head_dim) return fail_validation(a, "rope_qk: rot_dims must be a multiple of 16 up to head_dim");
    if (p.layout >= ROPE_LAYOUTS) return fail_validation(a, "rope_qk: layout must be 0 (i, i + head_dim/2), 1 (i, i + rot/2) or 2 (2i, 2i + 1)");
    const int at[4] = {0, 1, 3, 4};
    const char* names[4] = {"q", "k", "q_out", "k_out"};
    for (int i = 0; i < 4; i++) {
        const size_t width = (size_t)heads[i & 1] * p.head_dim;
        if (p.stride[i] == 0) p.stride[i] = (uint32_t)width;
        if (p.stride[i] % 8 || p.stride[i] < width) return fail_validation(a, std::string("rope_qk: a token's stride must be a multiple of 8 values that holds its heads (") + names[i] + ")");
        if (width == 0) continue;
        if (int r = need_bytes(a, at[i], 2 * ((size_t)(tokens - 1) * p.stride[i] + width), names[i])) return r;
    }
    if (int r = need_bytes(a, 2, 4 * (size_t)tokens * p.rot_dims, "cos_sin")) return r;
    const uint32_t k_al = heads[1] ? 16 : 1;
    if (int r = need_aligned(a, {16, k_al, 16, 16, k_al})) return r;
    // an output is its input, row for row, or shares nothing with what is read or written beside it
    const auto meet = [&](int i, int j) {
        return rows_meet(a.b[at[i]].ptr, 2 * (size_t)p.stride[i], 2 * (size_t)heads[i & 1] * p.head_dim, a.b[at[j]].ptr, 2 * (size_t)p.stride[j],
                         2 * (size_t)heads[j & 1] * p.head_dim, tokens);
    };
    bool in_place = true;
    for (int i = 0; i < 2; i++) {
        const bool same = a.b[at[i]].ptr == a.b[at[i + 2]].ptr && p.stride[i] == p.stride[i + 2];
        if ((!same && meet(i, i + 2)) || meet(i, 3 - i)) return fail_validation(a, std::string("rope_qk: ") + names[i] + " overlaps an output that is not its own");
        in_place = in_place && (same || heads[i] == 0);
    }
    if (meet(2, 3)) return fail_validation(a, "rope_qk: q_out and k_out overlap");
    for (int i = 2; i < 4; i++)
        if (int r = need_apart(a, "rope_qk", at[i], names[i], 2 * (size_t)p.stride[i], 2 * (size_t)heads[i & 1] * p.head_dim, tokens, {{2, 4 * (size_t)tokens * p.rot_dims, "cos_sin"}})) return r;
    RotateArgs k{{(const __half*)a.b[0].ptr, (const __half*)a.b[1].ptr}, {(__half*)a.b[3].ptr, (__half*)a.b[4].ptr}, {p.stride[0], p.stride[1]}, {p.stride[2], p.stride[3]},
                 {heads[0], heads[1]}, (const float2*)a.b[2].ptr, tokens, p.head_dim, p.rot_dims / 2, p.layout, 0, 0};
    k.pieces = (in_place ? p.rot_dims : p.head_dim) / 16;  // in place, what does not turn is not touched: a layout's turning pieces come first
    const uint32_t all = heads[0] + heads[1];
    const uint64_t rows = (uint64_t)tokens * all * k.pieces;
    // Heads of a thread: few threads start sooner, but one head of each is best while an SM has 256 or fewer.  Places that four heads leave empty cost where there are many
    // (us, one launch after the other, 1 | 2 | 4: 64 tokens of 32 and 16 heads of 128 1.71 | 1.88 | 2.23, 128 of them 2.13 | 1.89 | 2.23, 256 3.16 | 2.40 | 2.31, 1000 5.5 | 4.4 | 4.0, 5000
    // 23.5 | 20.1 | 20.4; 64 of 32 and 4 heads of 512, 64 pairs, 1.89 | 1.80 | 2.14; 2500 of 8 and 4 heads of 64 2.91 | 2.31 | 2.31; 10000 of 8 and 1 heads of 80 6.8 | 5.9 | 6.5).
    const bool empty_places = rows > 2048ull * a.sm_count && (all + 3) / 4 * 20 > all * 6;
    const uint32_t each = rows > 512ull * a.sm_count && !empty_places ? 4 : rows > 256ull * a.sm_count ? 2 : 1;
    k.slots = (all + each - 1) / each;
    const uint64_t threads = (uint64_t)tokens * k.pieces * k.slots;
    if (threads >= 1ull << 32) return fail_validation(a, "rope_qk: more values than one dispatch takes (2^36)");
    const auto kern = each == 4 ? rope_qk_kernel<4> : each == 2 ? rope_qk_kernel<2> : rope_qk_kernel<1>;
    const cudaError_t e = launch_dependent(kern, dim3((unsigned)((threads + ROW_THREADS - 1) / ROW_THREADS)), dim3(ROW_THREADS), 0, a.stream, k);
    ++*a.launches;
    return check_cuda(a, e, "rope_qk_f16");
}

}  // namespace sgb
