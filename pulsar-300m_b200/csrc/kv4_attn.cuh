// What the kernels of pulsar_op_kv4_attention share: the call's arguments, the rows of a sequence and
// how partial results are handed to the merge.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv4.cuh"

namespace pulsar {

constexpr float KV4_NEG = -1e30f;   // "no key yet": finite, so differences with it are defined

struct Kv4AttnArgs {
    const __nv_bfloat16* q;
    const uint8_t* pages;
    const int32_t *table, *kv_lens, *cu_q;
    __nv_bfloat16* out;
    // partials of split sp of (row, head) = at: part_o[(at nsplit + sp) HD ..], part_ml: the reference
    // exponent m (base 2) and the sum l of the weights relative to it
    float *part_o, *part_ml;
    int64_t q_row, q_head, page_bytes;
    int rows, hq, hkv, group, num_pages, width, page_shift, max_q, window, nsplit, split_len, unit_tile, step, cluster;
    float scale_log2;
};

// The part of sequence b that a unit tile (units u0 .. u0 + ut - 1) concerns. Everything stays inside
// the tensors whatever cu_q and kv_lens say.
struct Kv4Range {
    int row0, nq, units, ulast;   // the sequence's rows and units, the tile's last unit
    int len, first, last;         // keys; positions of the tile's first and last unit
    int kmin, kmax;               // keys that some unit of the tile sees: [kmin, kmax)
    int step0, steps, used;       // in steps of `step` keys from step0 on; splits that have some (at least 1)
};
__device__ __forceinline__ int kv4_low(const Kv4AttnArgs& a, int pos) {   // first key that position pos sees
    return a.window > 0 ? max(0, pos - a.window + 1) : 0;
}
__device__ __forceinline__ int kv4_row(const Kv4AttnArgs& a, int u) { return a.max_q == 1 ? 0 : u / a.group; }
__device__ __forceinline__ bool kv4_range(const Kv4AttnArgs& a, int b, int u0, int ut, int step, Kv4Range& r) {
    r.row0 = b;
    r.nq = 1;
    if (a.cu_q) {
        r.row0 = min(max(a.cu_q[b], 0), a.rows);
        r.nq = min(max(a.cu_q[b + 1] - r.row0, 0), min(a.max_q, a.rows - r.row0));
    }
    r.len = min(max(a.kv_lens[b], 0), a.width << a.page_shift);
    r.units = r.nq * a.group;
    if (u0 >= r.units) return false;
    r.ulast = min(u0 + ut, r.units) - 1;
    r.first = r.len - r.nq + kv4_row(a, u0);
    r.last = r.len - r.nq + kv4_row(a, r.ulast);
    r.kmin = kv4_low(a, r.first);
    r.kmax = max(r.last + 1, 0);
    r.step0 = r.kmin / step;
    r.steps = max((r.kmax + step - 1) / step - r.step0, 0);
    r.used = min(max((r.steps + a.split_len - 1) / a.split_len, 1), a.nsplit);
    return true;
}
// Steps [begin, end) of split sp < used, counted from step0: the last one takes what is left.
__device__ __forceinline__ void kv4_split(const Kv4AttnArgs& a, const Kv4Range& r, int sp, int& begin, int& end) {
    begin = sp * a.split_len;
    end = sp == r.used - 1 ? r.steps : min(r.steps, begin + a.split_len);
}

// Page of tile `tile` of sequence b (-1: none, or outside the cache).
__device__ __forceinline__ int kv4_page(const Kv4AttnArgs& a, int b, int tile) {
    const int col = tile >> (a.page_shift - 4);
    const int p = col < a.width ? a.table[(int64_t)b * a.width + col] : -1;
    return p >= 0 && p < a.num_pages ? p : -1;
}

__device__ __forceinline__ float kv4_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float kv4_s(uint32_t param) { return __uint_as_float(param << 16); }
__device__ __forceinline__ float kv4_z(uint32_t param) { return __uint_as_float(param & 0xffff0000u); }

// Weights in fp16, 2^(x - m) for a score x and a reference m of the unit: m moves when a sum of a few weights
// passes FULL (so each stays below 65504), and then lies ROOM below the largest score so far, so that weights
// down to 2^-21 of the largest keep their significand and what is lost below it is 2^-32 of the largest.
// (64 equal scores sum to 2^13, so scores may grow fourfold before m moves again.) m at the largest score itself
// gave 240 us instead of 243 for 2048 rows on 16384 keys, and lost a flat tail under one large weight.
constexpr float KV4_FULL = 32768.f, KV4_ROOM = 7.f;

// Operands in fp16 (values s c + z of 8-bit s, z and 4-bit c, rounded at 2^-12): fp16 has the significand but
// not the range, so powers of two are taken out of keys and values. What is far below the largest of its step
// falls under fp16's smallest numbers: the error is 2^-12 of a value or 2^-34 of that largest one.
__device__ __forceinline__ uint32_t kv4_half2(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ __half2 kv4_as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }

// The four operand registers of a code word as s c + z: codes under the exponent of 1024 (c, or 16 c).
__device__ __forceinline__ void kv4_unpack4(uint32_t w, uint32_t s, uint32_t z, uint32_t* r) {
    const uint32_t v = w >> 8;
    const __half2 one = __floats2half2_rn(1024.f, 1024.f), inv = __floats2half2_rn(0.0625f, 0.0625f),
                  sub = __floats2half2_rn(-64.f, -64.f);
    const __half2 c0 = __hsub2(kv4_as_half2((w & 0x000f000fu) | 0x64006400u), one);
    const __half2 c1 = __hfma2(kv4_as_half2((w & 0x00f000f0u) | 0x64006400u), inv, sub);
    const __half2 c2 = __hsub2(kv4_as_half2((v & 0x000f000fu) | 0x64006400u), one);
    const __half2 c3 = __hfma2(kv4_as_half2((v & 0x00f000f0u) | 0x64006400u), inv, sub);
    const __half2 x[4] = {__hfma2(c0, kv4_as_half2(s), kv4_as_half2(z)), __hfma2(c1, kv4_as_half2(s), kv4_as_half2(z)),
                          __hfma2(c2, kv4_as_half2(s), kv4_as_half2(z)), __hfma2(c3, kv4_as_half2(s), kv4_as_half2(z))};
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = *reinterpret_cast<const uint32_t*>(&x[i]);
}

// Power of two that brings a largest magnitude (float bits) to [2^9, 2^10): the exponent taken out of a step's
// keys or values. It reaches the largest numbers; at the lower end 2^-90 keeps sums of weights in range, and
// numbers down to 2^-100 their significand.
__device__ __forceinline__ int kv4_exponent_out(uint32_t bits) {
    return min(max((int)(bits >> 23) - 127 - 9, -90), 119);
}
// The same for a query row, to [2^3, 2^4).
__device__ __forceinline__ int kv4_query_exponent(uint32_t bits) {
    return min(max((int)(bits >> 23) - 127 - 3, -120), 124);
}
// 2^e, e from -126 to 127.
__device__ __forceinline__ float kv4_exp2i(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// Values of a step are operands 2^-ev V, O is kept in units of 2^er, and weights carry 2^(ev - er): er follows ev
// (O is rescaled) when it rises, or falls by more than SLACK, so that weights stay where fp16 is precise
// whatever sizes the values of other steps have. ev falls at most SPAN below the largest so far: O then stays in
// range, and values that far below lose precision. Where all are zero ev is er.
constexpr int KV4_SLACK = 6, KV4_SPAN = 80;
struct Kv4Unit {
    int ev = 0, er = 0, largest = -1000;
    __device__ __forceinline__ bool holds(int e) const { return (uint32_t)(e - er + KV4_SLACK) <= KV4_SLACK + 1; }
    // A step whose largest |value| is top (float bits). The factor for O, 1 where er stays.
    __device__ __forceinline__ float next(uint32_t top) {
        ev = kv4_exponent_out(top);
        if (holds(ev)) return 1.f;
        if (top == 0) {
            ev = er;
            return 1.f;
        }
        largest = max(largest, ev);
        ev = max(ev, largest - KV4_SPAN);
        const int old = er;
        if (!holds(ev)) er = ev;
        return kv4_ex2((float)(old - er));
    }
};

// Factor from sums of operand products to scores, from its query's and its keys' part. It stays above zero
// where both are tiny (queries and keys of zero, pages that are none): masked sums of -inf pass through it.
__device__ __forceinline__ float kv4_score_factor(float q, float k) { return fmaxf(q * k, 1.17549435e-38f); }

// The largest |value| that a parameter pair allows, as float bits (0 for NaN).
__device__ __forceinline__ uint32_t kv4_top(uint32_t param) {
    const float x = fmaxf(fabsf(kv4_z(param)), fabsf(fmaf(15.f, kv4_s(param), kv4_z(param))));
    return x == x ? __float_as_uint(x) : 0u;
}

// Many query rows (kv4_prefill.cu): units = query rows x heads of a group.
constexpr int kv4_pf_units(int head_dim) { return head_dim == 64 ? 512 : 256; }   // units of a CTA
constexpr int KV4_PF_STEP = 128;   // keys of a step
int kv4_prefill_launch(const Kv4AttnArgs& a, int head_dim, int64_t sequences, int utiles, cudaStream_t stream);

}  // namespace pulsar
