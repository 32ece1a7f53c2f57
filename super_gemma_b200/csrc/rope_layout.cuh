// Which dims of a head a rotary embedding couples, and their rotation.  pairs = rot_dims / 2, a multiple of 8:
//   layout 0   (i, i + head_dim / 2)   halves of the head; with rot_dims < head_dim the first pairs of each half turn
//   layout 1   (i, i + rot_dims / 2)   halves of the first rot_dims dims
//   layout 2   (2 i, 2 i + 1)          neighbours in the first rot_dims dims
// A head is cut into pieces of two octets of dims: of eight pairs, so that a rotation stays in a thread, or of octets that do not
// turn.  The pieces that turn come first; the first octets of consecutive pieces lie side by side, and so do the second ones (octets of a piece that lie side by
// side themselves leave half of a sector to each access: prompts through the pre-attention pass took 1.46 times the copy, now 1.05).
#pragma once

#include "sgb_common.cuh"

namespace sgb {

constexpr uint32_t ROPE_LAYOUTS = 3;

struct RopePiece {
    uint32_t lo, hi;      // first dims of its octets
    uint32_t pair[2];     // first pairs of its two fours
    bool turns;
};
__device__ __forceinline__ RopePiece rope_piece(uint32_t layout, uint32_t piece, uint32_t head_dim, uint32_t pairs)
{
    RopePiece p;
    const uint32_t turning = pairs / 8;
    p.turns = piece < turning;
    p.pair[0] = layout == 2 ? 4 * piece : 8 * piece;
    p.pair[1] = layout == 2 ? 4 * (turning + piece) : 8 * piece + 4;
    if (layout == 0) {
        p.lo = 8 * piece;
        p.hi = head_dim / 2 + 8 * piece;
    } else if (p.turns) {
        p.lo = 8 * piece;
        p.hi = pairs + 8 * piece;
    } else {
        p.lo = pairs + 8 * piece;  // 2 pairs + 8 (piece - turning)
        p.hi = head_dim / 2 + 8 * piece;
    }
    return p;
}

__device__ __forceinline__ void load_cos_sin(const float2* row, const RopePiece& at, float (&c)[8], float (&s)[8])  // row on 16 bytes
{
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float4 v = ld_global(reinterpret_cast<const float4*>(row + at.pair[j / 2]) + (j & 1));
        c[2 * j] = v.x;
        s[2 * j] = v.y;
        c[2 * j + 1] = v.z;
        s[2 * j + 1] = v.w;
    }
}

// The eight pairs of a piece's octets x, y, turned.
__device__ __forceinline__ void rope_turn(uint32_t layout, float (&x)[8], float (&y)[8], const float (&c)[8], const float (&s)[8])
{
    if (layout == 2) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float(&v)[8] = j < 4 ? x : y;
            const float a = v[2 * (j & 3)], b = v[2 * (j & 3) + 1];
            v[2 * (j & 3)] = a * c[j] - b * s[j];
            v[2 * (j & 3) + 1] = b * c[j] + a * s[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float a = x[j], b = y[j];
            x[j] = a * c[j] - b * s[j];
            y[j] = b * c[j] + a * s[j];
        }
    }
}

__device__ __forceinline__ void unpack_f16x8(const uint4& u, float (&v)[8])
{
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 f = __half22float2(h[j]);
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
    }
}
__device__ __forceinline__ uint4 pack_f16x8(const float (&v)[8])
{
    return make_uint4(pack_half2(v[0], v[1]), pack_half2(v[2], v[3]), pack_half2(v[4], v[5]), pack_half2(v[6], v[7]));
}

}  // namespace sgb
