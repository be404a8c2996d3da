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
    uint32_t n;   // n (hq + 2 hkv) < 2^31
    int hq, hkv, page_shift, rot, max_pos, interleaved;
    float eps;
};

// Sum of v over the L lanes of a vector, lane l ending with the sum that starts from neighbours.
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
    for (int o = 1; o < L; o <<= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

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

// Codes, s and z of the group of 32 dims whose 8-dim quarter this lane holds. Returns the lane's 8
// codes, nibble j = dim j.
__device__ __forceinline__ uint32_t quantise(const Dims& x, uint32_t& param) {
    float lo[8];
    f32x2 bad2 = two(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        parts(x.v[i], lo[2 * i], lo[2 * i + 1]);
        bad2 = fma2(x.v[i], two(0.f, 0.f), bad2);   // NaN once a value is none or infinite
    }
    float mn = fminf(fminf(fminf(lo[0], lo[1]), fminf(lo[2], lo[3])), fminf(fminf(lo[4], lo[5]), fminf(lo[6], lo[7])));
    float mx = fmaxf(fmaxf(fmaxf(lo[0], lo[1]), fmaxf(lo[2], lo[3])), fmaxf(fmaxf(lo[4], lo[5]), fmaxf(lo[6], lo[7])));
    float b0, b1;
    parts(bad2, b0, b1);
    if (!(b0 + b1 == 0.f)) mx = INFINITY;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    const __nv_bfloat16 zb = __float2bfloat16(mn);
    const float z = __bfloat162float(zb);
    const __nv_bfloat16 sb = __float2bfloat16(__fdiv_rn(__fsub_rn(mx, z), 15.f));
    const float s = __bfloat162float(sb);
    if (!(fabsf(z) < INFINITY && s < INFINITY)) {   // the whole group reads back as NaN
        param = 0x7fff7fffu;
        return 0u;
    }
    if (!(s >= 1.17549435e-38f)) {   // a constant group (or a span below the normal range)
        param = (uint32_t)__bfloat16_as_ushort(zb) << 16;
        return 0u;
    }
    param = (uint32_t)__bfloat16_as_ushort(zb) << 16 | __bfloat16_as_ushort(sb);
    // (x - z) / s, correctly rounded: the reciprocal and one step of Markstein's division (IBM J. Res.
    // Dev. 34, 1990; s has a bf16 significand, which is none of the method's exceptions). At most
    // 15 (1 + 2^-8) since s is rounded, so no code passes 15; z is rounded too and may lie above x.
    const float inv = __frcp_rn(s);
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

// Transpose among the quad of lanes that holds a group: lane j = 2 b + n comes with the codes of
// dims 16 b + 8 n + x (nibble x) and leaves with the word of x = 2j, 2j + 1: half e = x % 2, byte
// b of the half, nibble n of the byte.
__device__ __forceinline__ uint32_t quad_word(uint32_t p, int lane) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __shfl_sync(0xffffffffu, p, (lane & ~3) | i);
    const uint32_t j = lane & 3, sel = j | (4 + j) << 4;   // byte j of each of the four
    const uint32_t v = __byte_perm(__byte_perm(o[0], o[1], sel), __byte_perm(o[2], o[3], sel), 0x5410);
    const uint32_t e0 = v & 0x0f0f0f0fu, e1 = (v >> 4) & 0x0f0f0f0fu;
    return __byte_perm(e0 | e0 >> 4, e1 | e1 >> 4, 0x6420);
}

__device__ __forceinline__ void load4(const float* p, f32x2* x) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    x[0] = two(v.x, v.y);
    x[1] = two(v.z, v.w);
}

// x: the 8 dims (8 l ..) of a head vector that this lane holds, normed (weights w, or none) and
// turned. Every lane of the warp takes part.
template <int HD>
__device__ __forceinline__ void norm_rotate(const AppendArgs& a, const float* w, int pos, bool pos_ok, int lane, Dims& x) {
    constexpr int L = HD / 8;
    const int l = lane % L;
    if (w) {
        float t[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float u, v;
            parts(mul2(x.v[i], x.v[i]), u, v);
            t[i] = __fadd_rn(u, v);
        }
        const float ss = lanes_sum<L>(__fadd_rn(__fadd_rn(t[0], t[1]), __fadd_rn(t[2], t[3])));
        const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.f / HD), a.eps)));
        f32x2 wv[4];
        load4(w + 8 * l, wv);
        load4(w + 8 * l + 4, wv + 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[i] = mul2(wv[i], mul2(x.v[i], two(inv, inv)));
    }
    if (a.rot == 0) return;
    const int half = a.rot >> 1;
    const int64_t row = (int64_t)(pos_ok ? pos : 0) * half;
    const float *cs = a.cs + row, *sn = a.sn + row;
    const bool turn = 8 * l < a.rot;
    if (a.interleaved) {
        if (!turn) return;
        float c[4], s[4];
        if ((a.rot & 7) == 0) {   // rows of the tables are multiples of 16 bytes
            const float4 c4 = __ldg(reinterpret_cast<const float4*>(cs + 4 * l));
            const float4 s4 = __ldg(reinterpret_cast<const float4*>(sn + 4 * l));
            c[0] = c4.x; c[1] = c4.y; c[2] = c4.z; c[3] = c4.w;
            s[0] = s4.x; s[1] = s4.y; s[2] = s4.z; s[3] = s4.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bool in = 8 * l + 2 * j < a.rot;
                c[j] = in ? cs[4 * l + j] : 1.f;
                s[j] = in ? sn[4 * l + j] : 0.f;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (8 * l + 2 * j < a.rot) {   // (u c - v s, v c + u s)
                float u, v;
                parts(x.v[j], u, v);
                x.v[j] = two(__fsub_rn(__fmul_rn(u, c[j]), __fmul_rn(v, s[j])), __fadd_rn(__fmul_rn(v, c[j]), __fmul_rn(u, s[j])));
            }
        }
    } else {   // rot % 16 == 0: the partner's dims are the same 8 of another lane, rows multiples of 32 bytes
        const int hl = half >> 3;
        const bool first = l < hl;
        const int from = (lane - l) + (turn ? (first ? l + hl : l - hl) : l);
        f32x2 o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __shfl_sync(0xffffffffu, x.v[i], from);
        if (turn) {
            const int b = 8 * (first ? l : l - hl);
            f32x2 c[4], s[4];
            load4(cs + b, c);
            load4(cs + b + 4, c + 2);
            load4(sn + b, s);
            load4(sn + b + 4, s + 2);
            const float sign = first ? -1.f : 1.f;   // x c - o s, or x c + o s
#pragma unroll
            for (int i = 0; i < 4; ++i) {   // (the products in pairs; the sums not, which would be contracted with them)
                float u0, u1, v0, v1;
                parts(mul2(x.v[i], c[i]), u0, u1);
                parts(mul2(o[i], mul2(s[i], two(sign, sign))), v0, v1);
                x.v[i] = two(__fadd_rn(u0, v0), __fadd_rn(u1, v1));
            }
        }
    }
}

// N times the warp's 256 / HD query vectors from vb on (of the call's n hq). What they need from
// memory is asked for before any of it is used.
template <int HD, int N>
__device__ __forceinline__ void append_queries(const AppendArgs& a, uint32_t vb, int lane) {
    constexpr int L = HD / 8, VW = 256 / HD;
    const int l = lane % L;
    uint4 raw[N];
    int pos[N], head[N];
    const uint32_t first = vb + lane / L;
    int64_t tok = first / (uint32_t)a.hq;
    int h = (int)(first - (uint32_t)tok * a.hq);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (tok >= a.n) tok = 0;   // past the last vector: any valid one, not stored
        head[i] = h;
        raw[i] = __ldg(reinterpret_cast<const uint4*>(a.q + tok * a.qs + h * a.qh) + l);
        pos[i] = a.pos ? a.pos[tok] : 0;
        for (h += VW; h >= a.hq; h -= a.hq) ++tok;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t vi = first + i * VW;
        Dims x;
        x.take(raw[i]);
        const bool ok = !a.pos || (pos[i] >= 0 && pos[i] < a.max_pos);
        norm_rotate<HD>(a, a.qw ? a.qw + head[i] * HD : nullptr, pos[i], ok, lane, x);
        if (a.gain) {
            const float g = ok ? a.gain[pos[i]] : 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) x.v[j] = mul2(x.v[j], two(g, g));
        }
        if (vi < a.n * (uint32_t)a.hq)
            reinterpret_cast<uint4*>(a.qo)[(int64_t)vi * L + l] = ok ? x.bf16() : make_uint4(0, 0, 0, 0);
    }
}

// One (token, kv head) vector for each group of HD / 8 lanes: its codes and parameters, to those of
// the token's tile (in global or shared memory); t: the token's place in the tile.
template <int HD>
__device__ __forceinline__ void store_vector(const Dims& x, bool is_k, int t, bool put, uint8_t* codes, uint8_t* params,
                                             int lane) {
    using T = Kv4Tile<HD>;
    const int l = lane % (HD / 8), r = t & 7, hf = t >> 3, g = l >> 2, j = l & 3;
    uint32_t param;
    const uint32_t word = quad_word(quantise(x, param), lane);
    if (!put) return;
    if (is_k) {
        *reinterpret_cast<uint32_t*>(codes + (g >> 1) * T::BLK + (4 * r + j) * 16 + hf * 8 + (g & 1) * 4) = word;
    } else {
        uint8_t* p = codes + (g >> 1) * T::BLK + (8 * j + (r >> 1)) * 16 + (g & 1) * 8 + hf * 4 + (r & 1) * 2;
        *reinterpret_cast<uint16_t*>(p) = (uint16_t)word;
        *reinterpret_cast<uint16_t*>(p + 64) = (uint16_t)(word >> 16);
    }
    if (j == 0) *reinterpret_cast<uint32_t*>(params + ((2 * r + hf) * T::NG + g) * 4) = param;
}

// The tile of a slot (0 .. num_slots - 1) and kv head.
template <int HD>
__device__ __forceinline__ int64_t tile_at(int64_t slot, int h, int hkv, int page_shift, int64_t page_bytes) {
    return ((slot >> page_shift) * hkv + h) * page_bytes +
           (int64_t)((slot & ((1 << page_shift) - 1)) >> 4) * Kv4Tile<HD>::BYTES;
}

// Where the lane's 8 dims of a head vector of k or v are.
template <int HD>
__device__ __forceinline__ const uint4* kv_source(const AppendArgs& a, bool is_k, int64_t tok, int h, int lane) {
    return reinterpret_cast<const uint4*>(is_k ? a.k + tok * a.ks + h * a.kh : a.v + tok * a.vs + h * a.vh) +
           lane % (HD / 8);
}

// Few tokens: a warp per 32 / L head vectors of one kind (queries, keys or values), so that no warp
// quantises what it does not store.
template <int HD>
__global__ void __launch_bounds__(128) k_kv4_append(const AppendArgs a) {
    using T = Kv4Tile<HD>;
    constexpr int VW = 256 / HD;   // vectors a warp
    const int lane = threadIdx.x & 31;
    const uint32_t nq = (a.n * (uint32_t)a.hq + VW - 1) / VW, nk = (a.n * (uint32_t)a.hkv + VW - 1) / VW;
    const uint32_t w = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (w < nq) {
        append_queries<HD, 1>(a, w * VW, lane);
    } else if (w < nq + 2 * nk) {
        const bool is_k = w < nq + nk;
        const uint32_t vi = (w - nq - (is_k ? 0 : nk)) * VW + lane / (HD / 8);
        const bool live = vi < a.n * (uint32_t)a.hkv;
        const uint32_t tok = live ? vi / (uint32_t)a.hkv : 0u;
        const int h = live ? (int)(vi - tok * a.hkv) : 0;
        const uint4 raw = __ldg(kv_source<HD>(a, is_k, tok, h, lane));
        const int pos = a.pos ? a.pos[tok] : 0;
        const int64_t slot = a.slots[tok];
        const bool ok = !a.pos || (pos >= 0 && pos < a.max_pos), put = live && ok && slot >= 0 && slot < a.num_slots;
        Dims x;
        x.take(raw);
        if (is_k) norm_rotate<HD>(a, a.kw ? a.kw + h * HD : nullptr, pos, ok, lane, x);
        uint8_t* tile = a.pages + (put ? tile_at<HD>(slot, h, a.hkv, a.page_shift, a.page_bytes) : 0);
        store_vector<HD>(x, is_k, (int)(slot & 15), put, tile + (is_k ? 0 : T::V), tile + (is_k ? T::KP : T::VP), lane);
    }
}

// Many tokens: a warp per 16 tokens of one kv head's keys or values. Where they fill one tile of the
// cache, its codes and parameters are put together in shared memory and written in 16-byte pieces
// (value codes of a token are 2-byte pieces 64 bytes apart); others are written one by one. Groups
// of 16 start so that the first token's page lines up with them. Queries: 16 vectors a warp.
constexpr int BULK_WARPS = 8;
template <int HD>
__global__ void __launch_bounds__(BULK_WARPS * 32, 4) k_kv4_append_bulk(const AppendArgs a) {
    using T = Kv4Tile<HD>;
    constexpr int VW = 256 / HD, L = HD / 8;
    __shared__ __align__(16) uint8_t images[BULK_WARPS][10 * HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lead = (int)(a.slots[0] & 15);   // tokens of the first group that lie before token 0
    const uint32_t groups = (a.n + lead + 15) / 16, nkv = groups * 2 * a.hkv;
    const uint32_t nq = (a.n * (uint32_t)a.hq + 15) / 16, w = blockIdx.x * BULK_WARPS + warp;
    if (w >= nkv) {
        if (w < nkv + nq)
#pragma unroll 1
            for (int i = 0; i < 16; i += 4 * VW) append_queries<HD, 4>(a, (w - nkv) * 16 + i, lane);
    } else {
        const uint32_t grp = w / (2u * a.hkv);
        const int kh = (int)(w - grp * 2 * a.hkv);
        const bool is_k = kh < a.hkv;
        const int h = is_k ? kh : kh - a.hkv;
        const int64_t tok0 = (int64_t)grp * 16 - lead;
        constexpr int N = 4;   // vectors of a lane asked for at a time
        uint4 raw[N];
        auto ask = [&](int i0) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int64_t tk = tok0 + (i0 + i) * VW + lane / L;
                raw[i] = __ldg(kv_source<HD>(a, is_k, tk >= 0 && tk < a.n ? tk : 0, h, lane));
            }
        };
        ask(0);
        // lane t % 16 knows token t's slot and position. A whole tile: 16 tokens in the 16 consecutive
        // slots of one, all of them stored
        const int64_t mine = tok0 + (lane & 15);
        const bool in = mine >= 0 && mine < a.n;
        const int64_t my_slot = in ? a.slots[mine] : -1;
        const int my_pos = in && a.pos ? a.pos[mine] : 0;
        const bool my_ok = !a.pos || (my_pos >= 0 && my_pos < a.max_pos);
        const bool my_put = in && my_ok && my_slot >= 0 && my_slot < a.num_slots;
        const int64_t s0 = __shfl_sync(0xffffffffu, my_slot, 0);
        const bool whole = __all_sync(0xffffffffu, my_put && my_slot == s0 + (lane & 15) && (s0 & 15) == 0);
        const uint32_t puts = __ballot_sync(0xffffffffu, my_put), oks = __ballot_sync(0xffffffffu, my_ok);
        uint8_t* dst = a.pages + (whole ? tile_at<HD>(s0, h, a.hkv, a.page_shift, a.page_bytes) : 0);
#pragma unroll 1
        for (int i0 = 0; i0 < 16 / VW; i0 += N) {
          if (i0 > 0) ask(i0);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int t = (i0 + i) * VW + lane / L;
            const int pos = __shfl_sync(0xffffffffu, my_pos, t);
            const int64_t slot = __shfl_sync(0xffffffffu, my_slot, t);
            const bool put = puts >> t & 1;
            Dims x;
            x.take(raw[i]);
            if (is_k) norm_rotate<HD>(a, a.kw ? a.kw + h * HD : nullptr, pos, oks >> t & 1, lane, x);
            uint8_t *codes = images[warp], *params = images[warp] + 8 * HD;
            if (!whole) {
                codes = a.pages + (put ? tile_at<HD>(slot, h, a.hkv, a.page_shift, a.page_bytes) : 0);
                params = codes + (is_k ? T::KP : T::VP);
                codes += is_k ? 0 : T::V;
            }
            store_vector<HD>(x, is_k, (int)(slot & 15), put, codes, params, lane);
          }
        }
        if (whole) {
            __syncwarp();
            const uint4* src = reinterpret_cast<const uint4*>(images[warp]);
            uint4* codes = reinterpret_cast<uint4*>(dst + (is_k ? 0 : T::V));
            uint4* par = reinterpret_cast<uint4*>(dst + (is_k ? T::KP : T::VP));
#pragma unroll
            for (int i = lane; i < HD / 2; i += 32) codes[i] = src[i];
            if (lane < HD / 8) par[lane] = src[HD / 2 + lane];
        }
    }
}

// The inverse of quantise and quad_word: bf16(s c + z) of the lane's 8 dims of each group of lanes'
// head vector, from the codes and parameters of its tile (ok false: zeros).
template <int HD>
__device__ __forceinline__ uint4 fetch_vector(const uint8_t* codes, const uint8_t* params, bool is_k, int t, bool ok,
                                              int lane) {
    using T = Kv4Tile<HD>;
    const int l = lane % (HD / 8), g = l >> 2, j = l & 3, r = t & 7, hf = t >> 3;
    uint32_t word = 0, par = 0;
    if (ok) {
        if (is_k) {
            word = *reinterpret_cast<const uint32_t*>(codes + (g >> 1) * T::BLK + (4 * r + j) * 16 + hf * 8 + (g & 1) * 4);
        } else {
            const uint8_t* p = codes + (g >> 1) * T::BLK + (8 * j + (r >> 1)) * 16 + (g & 1) * 8 + hf * 4 + (r & 1) * 2;
            word = *reinterpret_cast<const uint16_t*>(p) | (uint32_t)*reinterpret_cast<const uint16_t*>(p + 64) << 16;
        }
        par = *reinterpret_cast<const uint32_t*>(params + ((2 * r + hf) * T::NG + g) * 4);
    }
    const float s = __uint_as_float(par << 16), z = __uint_as_float(par & 0xffff0000u);
    float x[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {   // dims 32 g + 8 j + 2 q, + 1: nibble (j / 2, j % 2) of quad lane q's word
        const uint32_t o = __shfl_sync(0xffffffffu, word, (lane & ~3) | q) >> (4 * j);
        // a code under the exponent of 2^23 is 2^23 + c; s c is exact, so the sum is rounded once
        x[2 * q] = fmaf(__uint_as_float((o & 15u) | 0x4b000000u) - 8388608.f, s, z);
        x[2 * q + 1] = fmaf(__uint_as_float(((o >> 16) & 15u) | 0x4b000000u) - 8388608.f, s, z);
    }
    return f32_to_bf16x8(x);
}

struct ReadArgs {
    const uint8_t* pages;
    const int64_t* slots;
    __nv_bfloat16 *k, *v;
    int64_t page_bytes, num_slots;
    uint32_t n;   // 2 n hkv < 2^31
    int hkv, page_shift;
};

// Few positions: a warp per 32 / L head vectors.
template <int HD>
__global__ void __launch_bounds__(128) k_kv4_read(const ReadArgs a) {
    using T = Kv4Tile<HD>;
    constexpr int L = HD / 8;
    const int lane = threadIdx.x & 31;
    const uint32_t vi = (blockIdx.x * 128 + threadIdx.x) / L;
    const bool live = vi < a.n * 2 * a.hkv;
    const uint32_t tok = live ? vi / (2u * a.hkv) : 0u;
    const int kh = live ? (int)(vi - tok * 2 * a.hkv) : 0;
    const bool is_k = kh < a.hkv;
    const int h = is_k ? kh : kh - a.hkv;
    const int64_t slot = a.slots[tok];
    const bool ok = slot >= 0 && slot < a.num_slots;
    const uint8_t* tile = a.pages + (ok ? tile_at<HD>(slot, h, a.hkv, a.page_shift, a.page_bytes) : 0);
    const uint4 x = fetch_vector<HD>(tile + (is_k ? 0 : T::V), tile + (is_k ? T::KP : T::VP), is_k, (int)(slot & 15), ok,
                                     lane);
    if (live) reinterpret_cast<uint4*>((is_k ? a.k : a.v) + ((int64_t)tok * a.hkv + h) * HD)[lane % L] = x;
}

// Many positions: a warp per 16 of one kv head's keys or values; where they are one whole tile, its
// bytes come through shared memory in 16-byte pieces. Groups of 16 start so that the first
// position's tile lines up with them.
template <int HD>
__global__ void __launch_bounds__(BULK_WARPS * 32) k_kv4_read_bulk(const ReadArgs a) {
    using T = Kv4Tile<HD>;
    constexpr int VW = 256 / HD, L = HD / 8;
    __shared__ __align__(16) uint8_t images[BULK_WARPS][10 * HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lead = (int)(a.slots[0] & 15);
    const uint32_t w = blockIdx.x * BULK_WARPS + warp;
    if (w >= (a.n + lead + 15) / 16 * 2 * a.hkv) return;
    const uint32_t grp = w / (2u * a.hkv);
    const int kh = (int)(w - grp * 2 * a.hkv);
    const bool is_k = kh < a.hkv;
    const int h = is_k ? kh : kh - a.hkv;
    const int64_t tok0 = (int64_t)grp * 16 - lead, mine = tok0 + (lane & 15);
    const int64_t s = mine >= 0 && mine < a.n ? a.slots[mine] : -1;
    const int64_t s0 = __shfl_sync(0xffffffffu, s, 0);
    const bool whole = __all_sync(0xffffffffu, s0 >= 0 && (s0 & 15) == 0 && s == s0 + (lane & 15) && s < a.num_slots);
    if (whole) {
        const uint8_t* src = a.pages + tile_at<HD>(s0, h, a.hkv, a.page_shift, a.page_bytes);
        const uint4* codes = reinterpret_cast<const uint4*>(src + (is_k ? 0 : T::V));
        const uint4* par = reinterpret_cast<const uint4*>(src + (is_k ? T::KP : T::VP));
        uint4* img = reinterpret_cast<uint4*>(images[warp]);
#pragma unroll
        for (int i = lane; i < HD / 2; i += 32) img[i] = __ldg(codes + i);
        if (lane < HD / 8) img[HD / 2 + lane] = __ldg(par + lane);
        __syncwarp();
    }
#pragma unroll 4
    for (int i = 0; i < 16; i += VW) {
        const int64_t slot = __shfl_sync(0xffffffffu, s, i + lane / L), tk = tok0 + i + lane / L;
        const bool ok = slot >= 0 && slot < a.num_slots;
        const uint8_t *codes = images[warp], *params = images[warp] + 8 * HD;
        if (!whole) {
            codes = a.pages + (ok ? tile_at<HD>(slot, h, a.hkv, a.page_shift, a.page_bytes) : 0);
            params = codes + (is_k ? T::KP : T::VP);
            codes += is_k ? 0 : T::V;
        }
        const uint4 x = fetch_vector<HD>(codes, params, is_k, (int)(slot & 15), ok, lane);
        if (tk >= 0 && tk < a.n) reinterpret_cast<uint4*>((is_k ? a.k : a.v) + (tk * a.hkv + h) * HD)[lane % L] = x;
    }
}

// From this many tokens on a warp takes 16 of them.
constexpr int64_t BULK_TOKENS = 1024;

int bulk_grid(int64_t warps) { return (int)((warps + BULK_WARPS - 1) / BULK_WARPS); }

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
    AppendArgs a{(const __nv_bfloat16*)q, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, strides[0], strides[2],
                 strides[4], strides[1], strides[3], strides[5], q_norm, k_norm, cos, sin, q_gain, slots,
                 (rot > 0 || q_gain) ? positions : nullptr, (uint8_t*)pages, (__nv_bfloat16*)q_out,
                 num_pages * page_size, pb, (uint32_t)N, (int)Hq, (int)Hkv, shift, (int)rot, (int)max_pos, interleaved, eps};
    cudaStream_t st = (cudaStream_t)stream;
    if (N >= BULK_TOKENS) {
        const int grid = bulk_grid((N + 30) / 16 * 2 * Hkv + (N * Hq + 15) / 16);
        if (head_dim == 64)
            k_kv4_append_bulk<64><<<grid, BULK_WARPS * 32, 0, st>>>(a);
        else
            k_kv4_append_bulk<128><<<grid, BULK_WARPS * 32, 0, st>>>(a);
    } else {
        const int64_t vw = 256 / head_dim, warps = (N * Hq + vw - 1) / vw + 2 * ((N * Hkv + vw - 1) / vw);
        const int grid = (int)((warps + 3) / 4);
        if (head_dim == 64)
            k_kv4_append<64><<<grid, 128, 0, st>>>(a);
        else
            k_kv4_append<128><<<grid, 128, 0, st>>>(a);
    }
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
    const ReadArgs a{(const uint8_t*)pages, slots, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, pb,
                     num_pages * page_size, (uint32_t)N, (int)Hkv, shift};
    cudaStream_t st = (cudaStream_t)stream;
    if (N >= BULK_TOKENS) {
        const int grid = bulk_grid((N + 30) / 16 * 2 * Hkv);
        if (head_dim == 64)
            k_kv4_read_bulk<64><<<grid, BULK_WARPS * 32, 0, st>>>(a);
        else
            k_kv4_read_bulk<128><<<grid, BULK_WARPS * 32, 0, st>>>(a);
    } else {
        const int grid = (int)((N * 2 * Hkv * (head_dim / 8) + 127) / 128);
        if (head_dim == 64)
            k_kv4_read<64><<<grid, 128, 0, st>>>(a);
        else
            k_kv4_read<128><<<grid, 128, 0, st>>>(a);
    }
    PULSAR_LAUNCH_CHECK("k_kv4_read");
    return PULSAR_OK;
}
