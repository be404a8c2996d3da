// Layout of the paged 4-bit KV cache, shared by the kernels that write it (kv4_ops.cu) and the
// ones that attend over it (kv4_attn.cu).
//
// pages: uint8 [num_pages][Hkv][page bytes]. A (page, kv head) block is contiguous and holds
// page_size tokens in tiles of 16; a tile is 20 D bytes: key codes (8 D), value codes (8 D), key
// parameters (2 D), value parameters (2 D). A head vector is cut into groups of 32 dims, a group
// stores z = bf16(min) and s = bf16((max - z) / 15), and each dim a 4-bit code c that stands for
// s c + z: 5 bits a dim. A group that holds a NaN or an infinity stores s = z = NaN.
//
// The codes of a tile lie in the order in which a warp feeds them to mma.m16n8k16: with lane
// 4 r + t (r = 0..7, t = 0..3), key codes form the A operand of S^T = K Q^T (rows r, r + 8: the
// tile's tokens r, r + 8), value codes the A operand of O^T = V^T P^T (rows r, r + 8 of a 16-dim
// block, columns: tokens 2t, 2t + 1, 2t + 8, 2t + 9). Every 32-bit word holds four operand
// registers: nibble i of its low and high halves are the two elements of register i, so one shift
// and one logic operation make a register. Lane 4 r + t owns the 16 bytes at 16 (4 r + t) of each
// 512-byte block (64 dims):
//   keys    [token r: words of groups 2 blk, 2 blk + 1][token r + 8: the same]; nibble i, half e
//           of group w's word: dim 32 w + 16 (i / 2) + 8 (i % 2) + 2 t + e
//   values  [group 2 blk: words of tokens 0-7, 8-15][group 2 blk + 1: the same]; nibble i, half e
//           of group w's word h: dim 32 w + 16 (i / 2) + 8 (i % 2) + r, token 8 h + 2 t + e
// Parameters: (s, z) pairs, token order (t % 8, t / 8), groups inside: a lane's two tokens are
// adjacent. A byte holds codes of one token only, so tokens of a tile can be written by different
// threads without a race.
#pragma once

#include <stdint.h>

namespace pulsar {

constexpr int KV4_TILE = 16;     // tokens of a tile
constexpr int KV4_GROUP = 32;    // dims that share s and z
template <int HD>
struct Kv4Tile {
    static constexpr int NG = HD / KV4_GROUP;   // groups of a head vector
    static constexpr int V = 8 * HD;            // byte offset of the value codes
    static constexpr int KP = 16 * HD;          // of the key parameters
    static constexpr int VP = 18 * HD;          // of the value parameters
    static constexpr int BYTES = 20 * HD;
    static constexpr int BLK = 512;             // codes of 16 tokens x 64 dims
};

// Two fp32 lanes in one instruction.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 two(float a, float b) {
    f32x2 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void parts(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

}  // namespace pulsar
