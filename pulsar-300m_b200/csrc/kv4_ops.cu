// Writing and reading the paged 4-bit KV cache (layout: kv4.cuh): pulsar_op_kv4_append,
// pulsar_op_kv4_read.
//
// append, per token and head vector x of D dims (fp32 from bf16):
//   y = w x / sqrt(mean x^2 + eps)          queries and keys, when norm weights are given
//   (a, b) -> (a cos - b sin, b cos + a sin) on the first `rot` dims: pairs (i, i + rot/2), or
//                                           (2i, 2i + 1) when interleaved
//   queries: y gain[pos], rounded to bf16; keys and values: quantised in groups of 32 dims.
// Every operation is rounded on its own (no contraction), sums run over neighbours first and the
// square root and the divisions are the correctly rounded ones, so a plain fp32 evaluation in the
// same order stores the same codes: quantisation amplifies a last-bit difference at a tie into a
// whole step.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "capi_util.h"
#include "common.cuh"
#include "kv4.cuh"

using namespace pulsar;

namespace {

struct AppendArgs {
    const __nv_bfloat16 *q, *k, *v;
    int64_t qs, ks, vs, qh, kh, vh;   // element strides of tokens and heads
    const float *qw, *kw, *cs, *sn, *gain;
    const int64_t* slots;
    const int32_t* pos;
    uint8_t* pages;
    __nv_bfloat16* qo;
    int64_t num_slots, page_bytes;
    uint32_t n, warps;   // n (hq + 2 hkv) < 2^31
    int hq, hkv, page_shift, rot, max_pos, heads;
    float eps;
};

constexpr float WHOLE = 12582912.f;   // 1.5 2^23: adding it rounds to a whole number, ties to even

// A lane's 8 dims, two to a register pair: every packed operation rounds each half on its own.
struct Dims {
    f32x2 v[4];
    __device__ __forceinline__ void take(const uint4& u) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = two(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
    __device__ __forceinline__ uint4 bf16() const {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x, y;
            parts(v[i], x, y);
            const __nv_bfloat162 b = __floats2bfloat162_rn(x, y);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// How a call's queries and keys are turned: not at all; pairs (i, i + D/2) of the whole vector, whose
// halves a lane holds; neighbours; pairs (i, i + rot/2) of a part, which other lanes hold.
enum { TURN_NONE, TURN_WHOLE, TURN_NEIGHBOURS, TURN_PART };

__device__ __forceinline__ float min3(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// The largest, NaN where there is one.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void range(const Dims& x, float& mn, float& mx) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) parts(x.v[i], v[2 * i], v[2 * i + 1]);
    mn = min3(min3(min3(v[0], v[1], v[2]), v[3], v[4]), min3(v[5], v[6], v[7]), v[7]);
    mx = max3(max3(max3(v[0], v[1], v[2]), v[3], v[4]), max3(v[5], v[6], v[7]), v[7]);
}

// The 8 codes (nibble j = dim j) of a lane's quarter of a group with parameters par and inv = 1 / s, 0
// for a group of one value; a group of NaN has codes 0.
__device__ __forceinline__ uint32_t codes_of(const Dims& x, uint32_t par, float inv) {
    // (x - z) / s, correctly rounded: the reciprocal and one step of Markstein's division (IBM J. Res.
    // Dev. 34, 1990; s has a bf16 significand, which is none of the method's exceptions). At most
    // 15 (1 + 2^-8) since s is rounded, so no code passes 15; z is rounded too and may lie above x.
    const float s = __uint_as_float(par << 16), z = __uint_as_float(par & 0xffff0000u);
    const f32x2 z2 = two(-z, -z), s2 = two(-s, -s), i2 = two(inv, inv);
    float c[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2 d = add2(x.v[i], z2), q = mul2(d, i2), r = fma2(q, s2, d);
        float u, v;
        parts(fma2(r, i2, q), u, v);
        parts(add2(add2(two(fmaxf(u, 0.f), fmaxf(v, 0.f)), two(WHOLE, WHOLE)), two(-WHOLE, -WHOLE)), c[2 * i], c[2 * i + 1]);
    }
    // four codes at a time as the digits of one whole number
    uint32_t p[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        p[i] = __float_as_uint(__fmaf_rn(__fmaf_rn(__fmaf_rn(c[4 * i + 3], 16.f, c[4 * i + 2]), 16.f, c[4 * i + 1]),
                                         16.f, c[4 * i]) + 8388608.f);
    return __byte_perm(p[0], p[1], 0x5410);
}

// Codes and parameters (s, z above it) of the two groups of 32 dims of which the quad of lanes holds the
// quarters lo and hi. Even lanes look after the first group's parameters, odd lanes after the other's.
__device__ __forceinline__ void quantise(const Dims& lo, const Dims& hi, int lane, uint32_t* code, uint32_t* param) {
    const bool odd = lane & 1;
    float mn0, mx0, mn1, mx1;
    range(lo, mn0, mx0);
    range(hi, mn1, mx1);
    float mn = odd ? mn1 : mn0, mx = odd ? mx1 : mx0;
    const float mn_up = __shfl_xor_sync(0xffffffffu, odd ? mn0 : mn1, 1), mx_up = __shfl_xor_sync(0xffffffffu, odd ? mx0 : mx1, 1);
    const float mn2 = fminf(mn, mn_up), mx2 = max3(mx, mx_up, mx_up);
    mn = fminf(mn2, __shfl_xor_sync(0xffffffffu, mn2, 2));
    const float mx3 = __shfl_xor_sync(0xffffffffu, mx2, 2);
    mx = max3(mx2, mx3, mx3);
    const __nv_bfloat16 zb = __float2bfloat16(mn);
    const float z = __bfloat162float(zb);
    // (mx - z) / 15, correctly rounded in the same way
    const float span = __fsub_rn(mx, z), part = __fmul_rn(span, 1.f / 15.f);
    const __nv_bfloat16 sb = __float2bfloat16(__fmaf_rn(__fmaf_rn(part, -15.f, span), 1.f / 15.f, part));
    const float s = __bfloat162float(sb);
    uint32_t par = (uint32_t)__bfloat16_as_ushort(zb) << 16;
    float inv = 0.f;
    if (!(fabsf(z) < INFINITY && s < INFINITY)) {   // the whole group reads back as NaN
        par = 0x7fff7fffu;
    } else if (s >= 1.17549435e-38f) {   // else a group of one value (or a span below the normal range)
        par |= __bfloat16_as_ushort(sb);
        inv = __frcp_rn(s);
    }
    const uint32_t par_up = __shfl_xor_sync(0xffffffffu, par, 1);
    const float inv_up = __shfl_xor_sync(0xffffffffu, inv, 1);
    param[0] = odd ? par_up : par;
    param[1] = odd ? par : par_up;
    code[0] = codes_of(lo, param[0], odd ? inv_up : inv);
    code[1] = codes_of(hi, param[1], odd ? inv : inv_up);
}

// Byte j of each of the four lanes' words, for lane j of the quad.
__device__ __forceinline__ uint32_t quad_transpose(uint32_t p, int lane) {
    p = __byte_perm(p, __shfl_xor_sync(0xffffffffu, p, 2), lane & 2 ? 0x3276 : 0x5410);
    return __byte_perm(p, __shfl_xor_sync(0xffffffffu, p, 1), lane & 1 ? 0x3715 : 0x6240);
}
// Among the quad of lanes that holds a group: lane j = 2 b + n comes with the codes of dims
// 16 b + 8 n + x (nibble x) and leaves with the word of x = 2j, 2j + 1: half e = x % 2, byte b of the
// half, nibble n of the byte.
__device__ __forceinline__ uint32_t to_word(uint32_t p, int lane) {
    const uint32_t v = quad_transpose(p, lane), e0 = v & 0x0f0f0f0fu, e1 = (v >> 4) & 0x0f0f0f0fu;
    return __byte_perm(e0 | e0 >> 4, e1 | e1 >> 4, 0x6420);
}
__device__ __forceinline__ uint32_t from_word(uint32_t w, int lane) {
    const uint32_t a = __byte_perm(w, 0, 0x1100), b = __byte_perm(w, 0, 0x3322);
    return quad_transpose((a & 0x000f000fu) | ((a >> 4) & 0x0f000f00u) | ((b << 4) & 0x00f000f0u) | (b & 0xf000f000u), lane);
}

__device__ __forceinline__ void load4(const float* p, f32x2* x) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    x[0] = two(v.x, v.y);
    x[1] = two(v.z, v.w);
}
__device__ __forceinline__ void load8(const float* p, f32x2* x) {
    load4(p, x);
    load4(p + 4, x + 2);
}

// x = w x / sqrt(mean x^2 + eps) of the vector whose parts lo and hi this lane holds.
template <int HD>
__device__ __forceinline__ void norm(Dims& lo, Dims& hi, const f32x2* w, float eps, int lane) {
    constexpr int L = HD / 16;
    auto sum8 = [](const Dims& x) {
        float t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float u, v;
            parts(mul2(x.v[i], x.v[i]), u, v);
            t[i] = __fadd_rn(u, v);
        }
        return __fadd_rn(__fadd_rn(t[0], t[1]), __fadd_rn(t[2], t[3]));
    };
    // sums of neighbours first; even lanes add up the first half's, odd lanes the other's
    const bool odd = lane & 1;
    const float a = sum8(lo), b = sum8(hi);
    float ss = __fadd_rn(odd ? b : a, __shfl_xor_sync(0xffffffffu, odd ? a : b, 1));
#pragma unroll
    for (int o = 2; o < L; o <<= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, o));
    ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, 1));
    const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.f / HD), eps)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        lo.v[i] = mul2(w[i], mul2(lo.v[i], two(inv, inv)));
        hi.v[i] = mul2(w[4 + i], mul2(hi.v[i], two(inv, inv)));
    }
}

// What a token's vectors are turned by: cos in t[0..3] and sin in t[4..7] of a lane's 8 pairs. Pairs of
// neighbours: the first four pairs (of lo) in t[0..1] and t[4..5].
template <int HD, int TURN>
__device__ __forceinline__ void load_turn(const AppendArgs& a, int pos, int l, f32x2* t) {
    if (TURN != TURN_WHOLE && TURN != TURN_NEIGHBOURS) return;
    const int64_t row = (int64_t)pos * (a.rot >> 1);
    const float *cs = a.cs + row, *sn = a.sn + row;
    if (TURN == TURN_WHOLE) {
        load8(cs + 8 * l, t);
        load8(sn + 8 * l, t + 4);
    } else {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            const int p = hf * (HD / 4) + 4 * l;   // the first pair
            if (a.rot % 8 == 0) {   // rows of the tables are multiples of 16 bytes
                if (2 * p < a.rot) {
                    load4(cs + p, t + 2 * hf);
                    load4(sn + p, t + 4 + 2 * hf);
                }
            } else {
                float c[4], s[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool in = 2 * (p + j) < a.rot;
                    c[j] = in ? cs[p + j] : 1.f;
                    s[j] = in ? sn[p + j] : 0.f;
                }
                t[2 * hf] = two(c[0], c[1]);
                t[2 * hf + 1] = two(c[2], c[3]);
                t[4 + 2 * hf] = two(s[0], s[1]);
                t[5 + 2 * hf] = two(s[2], s[3]);
            }
        }
    }
}

// The products are taken in pairs; the sums are not, which would be contracted with them.
template <int HD, int TURN>
__device__ __forceinline__ void turn(const AppendArgs& a, Dims& lo, Dims& hi, const f32x2* t, int pos, int lane) {
    constexpr int L = HD / 16;
    const int l = lane % L;
    if (TURN == TURN_WHOLE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float u0, u1, v0, v1;
            parts(mul2(lo.v[i], t[i]), u0, u1);
            parts(mul2(hi.v[i], t[4 + i]), v0, v1);
            const f32x2 x = two(__fsub_rn(u0, v0), __fsub_rn(u1, v1));
            parts(mul2(hi.v[i], t[i]), u0, u1);
            parts(mul2(lo.v[i], t[4 + i]), v0, v1);
            hi.v[i] = two(__fadd_rn(u0, v0), __fadd_rn(u1, v1));
            lo.v[i] = x;
        }
    } else if (TURN == TURN_NEIGHBOURS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {   // (u c - v s, v c + u s)
            f32x2& x = j < 4 ? lo.v[j] : hi.v[j - 4];
            if ((j < 4 ? 0 : HD / 2) + 8 * l + 2 * (j & 3) >= a.rot) continue;
            float c[2], s[2], u, v, uc, vc, us, vs;
            parts(t[j / 2], c[0], c[1]);
            parts(t[4 + j / 2], s[0], s[1]);
            parts(x, u, v);
            parts(mul2(x, two(c[j & 1], c[j & 1])), uc, vc);
            parts(mul2(x, two(s[j & 1], s[j & 1])), us, vs);
            x = two(__fsub_rn(uc, vs), __fadd_rn(vc, us));
        }
    } else if (TURN == TURN_PART) {   // rot % 16 == 0: the partners of 8 dims are 8 of one lane
        const int hl = a.rot >> 4;
        const int64_t row = (int64_t)pos * (a.rot >> 1);
        const Dims x[2] = {lo, hi};
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
            if (hf * (HD / 2) >= a.rot) break;
            const int c = hf * L + l;   // which 8 dims
            const bool on = c < 2 * hl, first = c < hl;
            const int pc = on ? (first ? c + hl : c - hl) : 0, from = (lane - l) + pc % L;
            f32x2 o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                o[i] = __shfl_sync(0xffffffffu, x[0].v[i], from);
                if (a.rot > HD / 2) {
                    const f32x2 up = __shfl_sync(0xffffffffu, x[1].v[i], from);
                    if (pc >= L) o[i] = up;
                }
            }
            if (!on) continue;
            const int64_t at = row + 8 * (first ? c : c - hl);
            f32x2 cs[4], sn[4];
            load8(a.cs + at, cs);
            load8(a.sn + at, sn);
            const float sign = first ? -1.f : 1.f;   // x c - o s, or x c + o s
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float u0, u1, v0, v1;
                parts(mul2(x[hf].v[i], cs[i]), u0, u1);
                parts(mul2(o[i], mul2(sn[i], two(sign, sign))), v0, v1);
                (hf ? hi : lo).v[i] = two(__fadd_rn(u0, v0), __fadd_rn(u1, v1));
            }
        }
    }
}

// The tile of a slot (0 .. num_slots - 1) and kv head.
template <int HD>
__device__ __forceinline__ int64_t tile_at(int64_t slot, int h, int hkv, int page_shift, int64_t page_bytes) {
    return ((slot >> page_shift) * hkv + h) * page_bytes +
           (int64_t)((slot & ((1 << page_shift) - 1)) >> 4) * Kv4Tile<HD>::BYTES;
}

// Where the bytes of token t of a tile are: a lane's word of key codes, its two halves of a word of value
// codes (64 bytes apart), the parameters; of group g, lane j of the quad.
template <int HD>
__device__ __forceinline__ int key_at(int t, int g, int j) {
    return (g >> 1) * Kv4Tile<HD>::BLK + (4 * (t & 7) + j) * 16 + (t >> 3) * 8 + (g & 1) * 4;
}
template <int HD>
__device__ __forceinline__ int value_at(int t, int g, int j) {
    return Kv4Tile<HD>::V + (g >> 1) * Kv4Tile<HD>::BLK + (8 * j + ((t & 7) >> 1)) * 16 + (g & 1) * 8 + (t >> 3) * 4 + (t & 1) * 2;
}
template <int HD>
__device__ __forceinline__ int params_at(int t, int g) {
    return ((2 * (t & 7) + (t >> 3)) * Kv4Tile<HD>::NG + g) * 4;
}

// The words of a lane's two groups, `apart` bytes from each other: neighbours with heads of 64.
template <int HD>
__device__ __forceinline__ void store_two(uint8_t* p, int apart, uint32_t x, uint32_t y) {
    if (HD == 64) {
        *reinterpret_cast<uint2*>(p) = make_uint2(x, y);
    } else {
        *reinterpret_cast<uint32_t*>(p) = x;
        *reinterpret_cast<uint32_t*>(p + apart) = y;
    }
}
template <int HD>
__device__ __forceinline__ uint2 load_two(const uint8_t* p, int apart) {
    if (HD == 64) return *reinterpret_cast<const uint2*>(p);
    return make_uint2(*reinterpret_cast<const uint32_t*>(p), *reinterpret_cast<const uint32_t*>(p + apart));
}

// A warp's work: 512 / HD tokens (a lane holds dims 8 l .. and HD / 2 + 8 l .. of one's vector, l = lane %
// (HD / 16): both halves of the rotation's pairs, and quarters of two groups), and up to `heads` heads
// of one kind, one after the other: slots, positions and tables are looked up once for them.
struct Item {
    int64_t tok;
    int kind, h0, h1;   // 0 queries, 1 keys, 2 values; heads h0 .. h1 - 1
    bool live;
};
template <int HD>
__device__ __forceinline__ Item item_of(uint32_t w, uint32_t n, int hq, int hkv, int heads, int lane) {
    const uint32_t iq = (uint32_t)(hq + heads - 1) / heads, ik = (uint32_t)(hkv + heads - 1) / heads, per = iq + 2 * ik;
    const uint32_t grp = w / per;
    uint32_t i = w - grp * per;
    Item it;
    it.kind = i < iq ? 0 : i < iq + ik ? 1 : 2;
    i -= it.kind == 0 ? 0 : it.kind == 1 ? iq : iq + ik;
    it.h0 = (int)i * heads;
    const int all = it.kind == 0 ? hq : hkv;
    it.h1 = it.h0 + heads < all ? it.h0 + heads : all;
    it.tok = (int64_t)grp * (512 / HD) + lane / (HD / 16);
    it.live = it.tok < n;
    if (!it.live) it.tok = 0;   // any valid one, not stored
    return it;
}

// ONE: a head an item, no loop. 16384 tokens of 16 query and 4 kv heads of 64 take 26 us: 89 MB, 3.4 TB/s.
// One token: 2.3 us. What bounds it is the arithmetic (some 290 instructions for a lane's 16 dims, two a
// clock and SM) behind the chain slot, position, table, vector; 24 warps an SM (80 registers, a few spilled)
// hide that better than the 16 that fit without a bound: 32 us against 40. Two heads' work unrolled into one
// another: 29 -> 26 us. Inputs and queries pass the caches as used once: the stores' mark alone is worth 3 us
// here and a fifth of k_kv4_read's time. Tokens run along the warp so that neighbouring slots share sectors
// of a tile: a token's value codes are 2-byte pieces 64 bytes apart. Gathering whole tiles in shared memory
// to write them in 16-byte pieces gained nothing.
template <int HD, int TURN, bool ONE>
__global__ void __launch_bounds__(128, 6) k_kv4_append(const AppendArgs a) {
    constexpr int L = HD / 16, NG = Kv4Tile<HD>::NG;
    const int lane = threadIdx.x & 31, l = lane % L;
    const uint32_t w = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w >= a.warps) return;
    Item it = item_of<HD>(w, a.n, a.hq, a.hkv, ONE ? 1 : a.heads, lane);
    if (ONE) it.h1 = it.h0 + 1;
    const __nv_bfloat16* src = it.kind == 0 ? a.q + it.tok * a.qs + it.h0 * a.qh
                             : it.kind == 1 ? a.k + it.tok * a.ks + it.h0 * a.kh : a.v + it.tok * a.vs + it.h0 * a.vh;
    const int64_t next = it.kind == 0 ? a.qh : it.kind == 1 ? a.kh : a.vh;
    uint4 raw0 = __ldcs(reinterpret_cast<const uint4*>(src) + l), raw1 = __ldcs(reinterpret_cast<const uint4*>(src) + L + l);
    int pos = a.pos ? a.pos[it.tok] : 0;
    const bool ok = !a.pos || (pos >= 0 && pos < a.max_pos);
    if (!ok) pos = 0;
    const int64_t slot = it.kind ? a.slots[it.tok] : 0;
    f32x2 t[8] = {};
    if (it.kind != 2) load_turn<HD, TURN>(a, pos, l, t);
    const float* wn = it.kind == 0 ? a.qw : it.kind == 1 ? a.kw : nullptr;
    const float gain = it.kind == 0 && a.gain ? a.gain[pos] : 1.f;
    const bool put = it.live && ok && slot >= 0 && slot < a.num_slots;
    uint8_t* tile = a.pages + (put && it.kind ? tile_at<HD>(slot, it.h0, a.hkv, a.page_shift, a.page_bytes) : 0);
    __nv_bfloat16* dst = a.qo + (it.tok * a.hq + it.h0) * HD;
#pragma unroll 2
    for (int h = it.h0; h < it.h1; ++h) {
        f32x2 weight[8];
        if (wn) {
            load8(wn + h * HD + 8 * l, weight);
            load8(wn + h * HD + HD / 2 + 8 * l, weight + 4);
        }
        Dims lo, hi;
        lo.take(raw0);
        hi.take(raw1);
        src += next;
        if (h + 1 < it.h1) {
            raw0 = __ldcs(reinterpret_cast<const uint4*>(src) + l);
            raw1 = __ldcs(reinterpret_cast<const uint4*>(src) + L + l);
        }
        if (wn) norm<HD>(lo, hi, weight, a.eps, lane);
        if (it.kind != 2) turn<HD, TURN>(a, lo, hi, t, pos, lane);
        if (it.kind == 0) {
            if (a.gain) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    lo.v[i] = mul2(lo.v[i], two(gain, gain));
                    hi.v[i] = mul2(hi.v[i], two(gain, gain));
                }
            }
            if (it.live) {
                __stcs(reinterpret_cast<uint4*>(dst) + l, ok ? lo.bf16() : make_uint4(0, 0, 0, 0));
                __stcs(reinterpret_cast<uint4*>(dst) + L + l, ok ? hi.bf16() : make_uint4(0, 0, 0, 0));
            }
            dst += HD;
        } else {
            uint32_t code[2], param[2];
            quantise(lo, hi, lane, code, param);
            const uint32_t w0 = to_word(code[0], lane), w1 = to_word(code[1], lane);
            const int tt = (int)(slot & 15), g0 = l >> 2, g1 = g0 + NG / 2, j = l & 3;
            if (put) {
                if (it.kind == 1) {
                    store_two<HD>(tile + key_at<HD>(tt, g0, j), key_at<HD>(tt, g1, j) - key_at<HD>(tt, g0, j), w0, w1);
                } else {
                    uint8_t *v0 = tile + value_at<HD>(tt, g0, j), *v1 = tile + value_at<HD>(tt, g1, j);
                    *reinterpret_cast<uint16_t*>(v0) = (uint16_t)w0;
                    *reinterpret_cast<uint16_t*>(v0 + 64) = (uint16_t)(w0 >> 16);
                    *reinterpret_cast<uint16_t*>(v1) = (uint16_t)w1;
                    *reinterpret_cast<uint16_t*>(v1 + 64) = (uint16_t)(w1 >> 16);
                }
                if (j == 0) {
                    uint8_t* p = tile + (it.kind == 1 ? Kv4Tile<HD>::KP : Kv4Tile<HD>::VP);
                    store_two<HD>(p + params_at<HD>(tt, g0), params_at<HD>(tt, g1) - params_at<HD>(tt, g0), param[0], param[1]);
                }
            }
            tile += a.page_bytes;
        }
    }
}

// bf16(s c + z) of a lane's 8 dims, from its codes (nibble j = dim j).
__device__ __forceinline__ uint4 values_of(uint32_t p, uint32_t par) {
    const float s = __uint_as_float(par << 16), z = __uint_as_float(par & 0xffff0000u);
    const uint32_t even = p & 0x0f0f0f0fu, odd = (p >> 4) & 0x0f0f0f0fu;
    Dims x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        // a code under the exponent of 2^23 is 2^23 + c; s c is exact, so the sum is rounded once
        const f32x2 c = two(__uint_as_float(__byte_perm(even, 0x4b000000u, 0x7440 + i)),
                            __uint_as_float(__byte_perm(odd, 0x4b000000u, 0x7440 + i)));
        x.v[i] = fma2(add2(c, two(-8388608.f, -8388608.f)), two(s, s), two(z, z));
    }
    return x.bf16();
}

struct ReadArgs {
    const uint8_t* pages;
    const int64_t* slots;
    __nv_bfloat16 *k, *v;
    int64_t page_bytes, num_slots;
    uint32_t n, warps;   // 2 n hkv < 2^31
    int hkv, page_shift, heads;
};

// 32768 positions of 4 kv heads of 64: 44 MB in 9.6 us, 4.6 TB/s (16384 of 8 heads of 128: 88 MB in 19.2);
// 777 positions 2.4 us. Bound by the latency of the slot and then of its tile (long scoreboard 7.7 an issue at
// 1.8 instructions a clock and SM, 80 for a lane's 16 dims).
// Through shared memory in whole tiles it was a fifth slower; two heads' bytes asked for at a time cost
// more registers than waiting.
template <int HD>
__global__ void __launch_bounds__(128) k_kv4_read(const ReadArgs a) {
    constexpr int L = HD / 16, NG = Kv4Tile<HD>::NG;
    const int lane = threadIdx.x & 31, l = lane % L;
    const uint32_t w = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w >= a.warps) return;
    const Item it = item_of<HD>(w, a.n, 0, a.hkv, a.heads, lane);
    const int64_t slot = a.slots[it.tok];
    const bool ok = slot >= 0 && slot < a.num_slots;
    const uint8_t* tile = a.pages + (ok ? tile_at<HD>(slot, it.h0, a.hkv, a.page_shift, a.page_bytes) : 0);
    const int tt = (int)(slot & 15), g0 = l >> 2, g1 = g0 + NG / 2, j = l & 3;
    uint4* dst = reinterpret_cast<uint4*>((it.kind == 1 ? a.k : a.v) + (it.tok * a.hkv + it.h0) * HD);
#pragma unroll 1
    for (int h = it.h0; h < it.h1; ++h) {
        uint2 w = {}, par = {};
        if (ok) {
            if (it.kind == 1) {
                w = load_two<HD>(tile + key_at<HD>(tt, g0, j), key_at<HD>(tt, g1, j) - key_at<HD>(tt, g0, j));
            } else {
                const uint16_t *v0 = reinterpret_cast<const uint16_t*>(tile + value_at<HD>(tt, g0, j)),
                               *v1 = reinterpret_cast<const uint16_t*>(tile + value_at<HD>(tt, g1, j));
                w = make_uint2(v0[0] | (uint32_t)v0[32] << 16, v1[0] | (uint32_t)v1[32] << 16);
            }
            const uint8_t* p = tile + (it.kind == 1 ? Kv4Tile<HD>::KP : Kv4Tile<HD>::VP);
            par = load_two<HD>(p + params_at<HD>(tt, g0), params_at<HD>(tt, g1) - params_at<HD>(tt, g0));
        }
        const uint4 x0 = values_of(from_word(w.x, lane), par.x), x1 = values_of(from_word(w.y, lane), par.y);
        if (it.live) {
            __stcs(dst + l, x0);
            __stcs(dst + L + l, x1);
        }
        dst += HD / 8;
        tile += a.page_bytes;
    }
}

template <int HD, bool ONE>
auto append_kernel(int turn) {
    return turn == TURN_NONE ? k_kv4_append<HD, TURN_NONE, ONE> : turn == TURN_WHOLE ? k_kv4_append<HD, TURN_WHOLE, ONE>
         : turn == TURN_NEIGHBOURS ? k_kv4_append<HD, TURN_NEIGHBOURS, ONE> : k_kv4_append<HD, TURN_PART, ONE>;
}

// Heads of a warp's work, from the warps that one head each would take: four, which share the look-ups,
// once one each would fill the SMs (24 warps each) four times. Measured with 1 / 2 / 4 / 8 heads, append to
// 16 query and 4 kv heads of 64: 1024 tokens 3.2 / 5.1 / 6.6 / 7.2 us, 4096 (12288 warps) 8.8 / 9.1 / 8.5 / 9.6,
// 8192 16.9 / 16.4 / 14.4 / 18.6, 16384 31.7 / 28.7 / 25.8 / 27.8; 32 and 8 heads of 128, 1536 tokens (18432
// warps) 14.5 / 12.8 / 13.4 / 13.4, 8192 65 / 54 / 46 / 45; reading 8192 positions of 4 heads of 64 4.7 / 4.2 /
// 4.6 / 4.1, 16384 7.2 / 6.1 / 5.7 / 5.8.
constexpr int64_t HEADS_4 = 14208;
int heads_of(int64_t warps) { return warps < HEADS_4 ? 1 : 4; }

int page_geometry(const char* what, int64_t head_dim, int64_t page_size, int64_t num_pages, int64_t hkv,
                  const void* pages, int* shift, int64_t* page_bytes) {
    PULSAR_CHECK_ARG(head_dim == 64 || head_dim == 128, "%s: head_dim must be 64 or 128, got %lld", what,
                     (long long)head_dim);
    PULSAR_CHECK_ARG(page_size >= 16 && page_size <= 65536 && (page_size & (page_size - 1)) == 0,
                     "%s: page_size must be a power of two of at least 16, got %lld", what, (long long)page_size);
    PULSAR_CHECK_ARG(num_pages >= 0 && hkv >= 1 && hkv <= 1024, "%s: invalid cache shape", what);
    PULSAR_CHECK_ARG(pages && (reinterpret_cast<uintptr_t>(pages) & 15) == 0,
                     "%s: pages must be 16-byte aligned device memory", what);
    *shift = __builtin_ctzll((unsigned long long)page_size);
    *page_bytes = page_size / KV4_TILE * 20 * head_dim;
    return PULSAR_OK;
}

}  // namespace

extern "C" int pulsar_op_kv4_append(const void* q, const void* k, const void* v, const int64_t* strides, int64_t N,
                                    int64_t Hq, int64_t Hkv, int64_t head_dim, const float* q_norm,
                                    const float* k_norm, float eps, const float* cos, const float* sin, int64_t rot,
                                    int64_t max_pos, int interleaved, const float* q_gain, const int32_t* positions,
                                    const int64_t* slots, void* pages, int64_t num_pages, int64_t page_size,
                                    void* q_out, void* stream) {
    PULSAR_CHECK_ARG(N >= 0 && Hq >= 0 && Hq <= 65536 && Hkv >= 1 && Hkv <= 1024 && N <= INT32_MAX / (Hq + 2 * Hkv) - 64,
                     "kv4_append: invalid shape (%lld tokens)", (long long)N);
    int shift;
    int64_t pb;
    PULSAR_TRY(page_geometry("kv4_append", head_dim, page_size, num_pages, Hkv, pages, &shift, &pb));
    PULSAR_CHECK_ARG(rot >= 0 && rot <= head_dim && rot % (interleaved ? 2 : 16) == 0,
                     "kv4_append: rotated dims must be a multiple of %d up to head_dim, got %lld", interleaved ? 2 : 16,
                     (long long)rot);
    if (N == 0) return PULSAR_OK;
    PULSAR_CHECK_ARG(k && v && strides && slots && (Hq == 0 || (q && q_out)), "kv4_append: null pointer");
    PULSAR_CHECK_ARG(rot == 0 || (cos && sin), "kv4_append: null rotation table");
    PULSAR_CHECK_ARG((rot == 0 && !q_gain) || (positions && max_pos > 0 && max_pos < ((int64_t)1 << 31)),
                     "kv4_append: tables need positions and at least one row");
    for (int i = 0; i < 6; ++i)
        PULSAR_CHECK_ARG(strides[i] % 8 == 0, "kv4_append: token and head strides must be multiples of 8 elements");
    for (const void* p : {q, k, v, (const void*)q_out, (const void*)q_norm, (const void*)k_norm, (const void*)cos,
                          (const void*)sin})
        PULSAR_CHECK_ARG((reinterpret_cast<uintptr_t>(p) & 15) == 0,
                         "kv4_append: q, k, v, norm weights and tables must be 16-byte aligned");
    const int64_t groups = (N * head_dim + 511) / 512;
    const int heads = heads_of(groups * (Hq + 2 * Hkv));
    const int64_t warps = groups * ((Hq + heads - 1) / heads + 2 * ((Hkv + heads - 1) / heads));
    const int turn = rot == 0 ? TURN_NONE : interleaved ? TURN_NEIGHBOURS : rot == head_dim ? TURN_WHOLE : TURN_PART;
    const AppendArgs a{(const __nv_bfloat16*)q, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, strides[0], strides[2],
                       strides[4], strides[1], strides[3], strides[5], q_norm, k_norm, cos, sin, q_gain, slots,
                       (rot > 0 || q_gain) ? positions : nullptr, (uint8_t*)pages, (__nv_bfloat16*)q_out,
                       num_pages * page_size, pb, (uint32_t)N, (uint32_t)warps, (int)Hq, (int)Hkv, shift, (int)rot,
                       (int)max_pos, heads, eps};
    cudaStream_t st = (cudaStream_t)stream;
    const int grid = (int)((warps + 3) / 4);
    auto* kernel = heads == 1 ? (head_dim == 64 ? append_kernel<64, true>(turn) : append_kernel<128, true>(turn))
                              : (head_dim == 64 ? append_kernel<64, false>(turn) : append_kernel<128, false>(turn));
    kernel<<<grid, 128, 0, st>>>(a);
    PULSAR_LAUNCH_CHECK("k_kv4_append");
    return PULSAR_OK;
}

extern "C" int pulsar_op_kv4_read(const void* pages, int64_t num_pages, int64_t page_size, int64_t Hkv,
                                  int64_t head_dim, const int64_t* slots, int64_t N, void* k_out, void* v_out,
                                  void* stream) {
    PULSAR_CHECK_ARG(N >= 0, "kv4_read: invalid shape");
    int shift;
    int64_t pb;
    PULSAR_TRY(page_geometry("kv4_read", head_dim, page_size, num_pages, Hkv, pages, &shift, &pb));
    if (N == 0) return PULSAR_OK;
    PULSAR_CHECK_ARG(slots && k_out && v_out, "kv4_read: null pointer");
    for (const void* p : {(const void*)k_out, (const void*)v_out})
        PULSAR_CHECK_ARG((reinterpret_cast<uintptr_t>(p) & 15) == 0, "kv4_read: outputs must be 16-byte aligned");
    PULSAR_CHECK_ARG(N <= INT32_MAX / (2 * Hkv) - 64, "kv4_read: invalid shape (%lld positions)", (long long)N);
    const int64_t groups = (N * head_dim + 511) / 512;
    const int heads = heads_of(groups * 2 * Hkv);
    const int64_t warps = groups * 2 * ((Hkv + heads - 1) / heads);
    const ReadArgs a{(const uint8_t*)pages, slots, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, pb,
                     num_pages * page_size, (uint32_t)N, (uint32_t)warps, (int)Hkv, shift, heads};
    cudaStream_t st = (cudaStream_t)stream;
    const int grid = (int)((warps + 3) / 4);
    if (head_dim == 64)
        k_kv4_read<64><<<grid, 128, 0, st>>>(a);
    else
        k_kv4_read<128><<<grid, 128, 0, st>>>(a);
    PULSAR_LAUNCH_CHECK("k_kv4_read");
    return PULSAR_OK;
}
