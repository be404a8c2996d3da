// Attention over the paged 4-bit KV cache (layout: kv4.cuh): pulsar_op_kv4_attention, and its kernel for
// few units a sequence and kv head (decoding, verify blocks, short prompts); more: kv4_prefill.cu.
//
// Row j of the n_b query rows of sequence b has position pos = len_b - n_b + j and sees the keys
// max(0, pos - window + 1) .. pos (window 0: all of 0 .. pos):
//   out = sum_k p_k v_k / sum_k p_k,  p_k = exp(scale q.k_k - m)
// with k = s c + z per group of 32 dims, so q.k = sum_g s_g (q.c)_g + z_g sum(q)_g: the codes enter
// the matrix instruction as they are (exact, see unpack) and s is applied in fp32 to its results;
// z meets the three bf16 terms of sum(q) in an instruction of its own. Values: O = sum_k (p_k s_kg) c
// + sum_k p_k z_kg: s goes into the weights, whose bf16 hi and lo halves (|x - hi - lo| <= 2^-17
// |x|) are both multiplied, and the second sum is a scalar per (row, group).
//
// A unit is a (query row, head of the kv head's group). CTA (split and unit tile, kv head,
// sequence): four warps, each walking every fourth pair of 16-token tiles of the split's range
// through a ring of its own (1-D bulk copies of whole tiles; each lane looks after every 32nd
// pair). Tokens are the M rows of S^T = K Q^T and units its N columns, so a tile's codes are
// unpacked once for all units, straight into operand registers; the weights pass through movmatrix
// into the B operand of O^T = V^T P^T. Up to four units the eight columns hold every unit twice and
// the copies carry the hi and the lo halves (256 sequences of 640 keys: 19.5 us, with both halves
// multiplied one after the other 20.0). Above eight units keys and values are unpacked to fp16 numbers
// instead (see wide_step): 64 x 5 rows of 4 heads on 1024 keys take 24 us, with codes as operands 38.
//
// The softmax keeps a maximum per unit that moves only when a sum of weights relative to it passes
// 2^LAZY (l and O use the same maximum, so the result does not depend on when it moves).
// Keys that a unit does not see get weight 0 by selection, not by multiplication: pages past a
// sequence's end may hold anything, NaN included. Tiles of a page outside the cache are skipped.
//
// Splits of the keys end in (m, l, O) partials, joined in split order: up to eight splits that fit the
// GPU at once are a cluster and read each other's shared memory, else k_kv4_merge follows.
//
// Time and what bounds it (4 kv heads of 64, 16 query heads): 4 x 32768 keys 18.2 us, 2.3 TB/s of cache;
// 256 x 513..767 20.2 us; 48 x 1..8191, 8 kv heads of 128, 71.6 us, 3.5 TB/s; 1 x 2048 6.5 us. The
// copies alone took 13.7, 13.3, 50 and 5.8 us. The rest are instructions, about 380 for a pair of tiles (heads
// of 128: 680) and 1000 a warp for its start and end, at 2 to 2.6 of 4 a clock and SM with 16 warps there.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "capi_util.h"
#include "common.cuh"
#include "kv4_attn.cuh"
#include "mega_ptx.cuh"

using namespace pulsar;

namespace {

// More than log2 of the keys of a row. Weights of 2^(LIFT + LAZY) times values stay in fp32 up to 2^37, and times
// codes 2^-133 down to values of 2^-50.
constexpr int LAZY = 30;
constexpr float NEG = KV4_NEG;

// d = a b + c (d and c may be the same registers)
__device__ __forceinline__ void mma16816(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, const float* c) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ void mma16816h(float* d, const uint32_t* a, uint32_t b0, uint32_t b1, const float* c) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Operand registers of a code word: its nibbles 0 and 1 of both halves are bf16 bit patterns as they
// stand, c 2^-133 and 16 c 2^-133 (bits 0..7 of a bf16 count in steps of 2^-133 across the border of
// the subnormal numbers, and the matrix instruction takes subnormal operands exactly); nibbles 2 and
// 3 need one shift for the two. No offset, no conversion.
__device__ __forceinline__ void unpack(uint32_t w, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    const uint32_t v = w >> 8;
    r0 = w & 0x000f000fu;
    r1 = w & 0x00f000f0u;
    r2 = v & 0x000f000fu;
    r3 = v & 0x00f000f0u;
}
constexpr int CODE_EXP = 133;   // a code c is the operand c 2^-133
constexpr int LIFT = 60;        // queries and weights are scaled by 2^60, so results are normal numbers
constexpr float pow2(int e) {   // 2^e (constant expressions only)
    float x = 1.f;
    for (; e > 0; --e) x *= 2.f;
    for (; e < 0; ++e) x *= 0.5f;
    return x;
}

__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo_of(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_of(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The pair at p of the cluster's CTA `rank`.
__device__ __forceinline__ float2 ld_cluster(const float* p, int rank) {
    uint32_t at;
    float2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}

// A stage holds two tiles (32 tokens): 10 KB in flight a warp.
template <int HD>
constexpr int stages() { return HD == 64 ? 4 : 2; }

// CTAs of four warps that an SM holds: 16 warps where the registers allow it.
constexpr int resident(int head_dim, int nt) { return nt == 1 ? 4 : nt == 2 && head_dim == 64 ? 3 : 2; }

template <int HD, int NT, bool DUP, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, resident(HD, NT) * 4 / WARPS) k_kv4_attn(const Kv4AttnArgs a) {
    using T = Kv4Tile<HD>;
    constexpr int NG = T::NG, NB = HD / 64, S = stages<HD>(), MT = HD / 16, TB = T::BYTES;
    constexpr int UT = DUP ? 4 : 8 * NT;
    constexpr bool WIDE = NT > 1;
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ uint64_t bars[WARPS][S];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % a.nsplit, u0 = blockIdx.x / a.nsplit * UT;
    const int h = blockIdx.y, b = blockIdx.z;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the merge may be set up meanwhile
    Kv4Range rg;
    if (!kv4_range(a, b, u0, UT, 32, rg) || (split >= rg.used && !a.cluster)) return;   // (the same for a cluster)
    const int row0 = rg.row0, units = rg.units, ulast = rg.ulast;
    // steps are pairs of tiles (32 tokens, aligned): the split's range, of which the warp takes every WARPS-th
    int s_begin, s_end;
    kv4_split(a, rg, split, s_begin, s_end);
    if (split >= rg.used) s_begin = s_end = 0;
    const int p_begin = rg.step0 + s_begin + warp, p_end = rg.step0 + s_end;
    const int mine = p_end > p_begin ? (p_end - p_begin + WARPS - 1) / WARPS : 0;

    if (lane == 0) {
        for (int i = 0; i < S; ++i) mbar_init(&bars[warp][i], 1);
        fence_mbar_init();
    }
    __syncwarp();

    // Lane i % 32 looks after the warp's i-th pair: it knows where the pair lies (null: no page) and
    // issues its copy. A page of 16 tokens holds one tile of the pair only.
    const bool two = a.page_shift == 4;
    unsigned char* ring = sm + warp * S * 2 * TB;
    struct Where {
        const uint8_t *t0, *t1;   // the pair's tiles
        uint32_t ok0, ok1;        // of the 32 pairs: which tiles are there
    };
    auto locate = [&](int i0) {   // pairs i0 .. i0 + 31
        Where w;
        const int tile = 2 * (p_begin + (i0 + lane) * WARPS);
        auto at = [&](int page, int tl) {
            return page < 0 ? nullptr
                            : a.pages + ((int64_t)page * a.hkv + h) * a.page_bytes +
                                  (int64_t)(tl & ((1 << (a.page_shift - 4)) - 1)) * TB;
        };
        w.t0 = w.t1 = nullptr;
        if (i0 + lane < mine) {
            const int page = kv4_page(a, b, tile);
            w.t0 = at(page, tile);
            w.t1 = two ? at(kv4_page(a, b, tile + 1), tile + 1) : page < 0 ? nullptr : w.t0 + TB;
        }
        w.ok0 = __ballot_sync(0xffffffffu, w.t0 != nullptr);
        w.ok1 = __ballot_sync(0xffffffffu, w.t1 != nullptr);
        return w;
    };
    auto issue = [&](int i, const Where& w) {   // one lane; a pair of no page completes its phase at once
        uint64_t* bar = &bars[warp][i % S];
        unsigned char* dst = ring + (i % S) * 2 * TB;
        if (w.t0 == nullptr && w.t1 == nullptr) {
            mbar_arrive(bar);
        } else if (!two) {
            mbar_arrive_expect_tx(bar, 2 * TB);
            tma_load_1d(dst, w.t0, 2 * TB, bar);
        } else {
            mbar_arrive_expect_tx(bar, (w.t0 ? TB : 0) + (w.t1 ? TB : 0));
            if (w.t0) tma_load_1d(dst, w.t0, TB, bar);
            if (w.t1) tma_load_1d(dst + TB, w.t1, TB, bar);
        }
    };
    Where here = locate(0), next = here;   // of the 32 pairs that hold the current one, the next one to issue
    // The first pair alone, the others of the ring once the queries are there: copies of an SM are served in
    // the order of issue, so every warp starts after a quarter of the rings instead of all of them
    // (4 x 32768: 19.3 -> 18.0 us).
    if (lane == 0 && mine > 0) issue(0, here);

    // queries: B operand of step j (dims 16 j ..): unit n = lane / 4, dims 2t, 2t + 1 and 8 further
    uint32_t qf[NT][2 * MT];
    // Sums of q over the groups, in the units of the scores: B operand that meets the keys' z, k = 2t and
    // 2t + 1 (and 8 further) groups 0 and 1 (2 and 3), the three bf16 terms of their sums on t = 0..2.
    uint32_t zq[NT][2] = {};
    float q_scale[NT][2];   // WIDE: scale times the power of two taken out of q
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int u = u0 + (DUP ? (r & 3) : nt * 8 + r);
        const bool ok = u < units;
        const int j = ok ? kv4_row(a, u) : 0, g = ok ? u - j * a.group : 0;
        const __nv_bfloat16* src = a.q + (row0 + j) * a.q_row + (h * a.group + g) * a.q_head;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) qf[nt][i] = ok ? *reinterpret_cast<const uint32_t*>(src + 8 * i + 2 * t) : 0u;
        if constexpr (WIDE) {   // q 2^-eq in fp16, its largest |dim| in [2^3, 2^4)
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i)
                top = max(top, max(qf[nt][i] << 16 & 0x7fffffffu, qf[nt][i] & 0x7fff0000u));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int eq = kv4_query_exponent(top);
            const float f = kv4_exp2i(-eq), s = fminf(a.scale_log2 * kv4_exp2i(eq), 3.4e38f);
            q_scale[nt][0] = __shfl_sync(0xffffffffu, s, 8 * t);
            q_scale[nt][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) qf[nt][i] = kv4_half2(lo_of(qf[nt][i]) * f, hi_of(qf[nt][i]) * f);
        } else {
#pragma unroll
            for (int g4 = 0; g4 < NG; ++g4) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) s += lo_of(qf[nt][4 * g4 + i]) + hi_of(qf[nt][4 * g4 + i]);
                s += __shfl_xor_sync(0xffffffffu, s, 1);
                s += __shfl_xor_sync(0xffffffffu, s, 2);
                s *= pow2(LIFT - CODE_EXP);
                const float s1 = s - lo_of(pack(s, s)), s2 = s1 - lo_of(pack(s1, s1));
                const uint32_t term = t == 0 ? pack(s, s) : t == 1 ? pack(s1, s1) : t == 2 ? pack(s2, s2) : 0u;
                zq[nt][g4 >> 1] = g4 & 1 ? __byte_perm(zq[nt][g4 >> 1], term, 0x5410) : term;
            }
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i) {   // odd registers meet 16 c
                const float f = i & 1 ? pow2(LIFT - 4) : pow2(LIFT);
                qf[nt][i] = pack(lo_of(qf[nt][i]) * f, hi_of(qf[nt][i]) * f);
            }
        }
    }
    int hi[NT][2], lo[NT][2];   // keys that the thread's columns see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int u = min(u0 + (DUP ? ((2 * t + c) & 3) : nt * 8 + 2 * t + c), units - 1);
            const int pos = rg.len - rg.nq + kv4_row(a, u);
            hi[nt][c] = pos + 1;
            lo[nt][c] = kv4_low(a, pos);
        }
    const int all_lo = kv4_low(a, rg.last), all_hi = rg.first + 1;   // keys in [all_lo, all_hi) are seen by every unit

    if (lane > 0 && lane < min(S, mine)) issue(lane, here);

    // Scores come in units of 2^(LIFT - CODE_EXP); m: their running maximum, nm = LIFT - scale m, so
    // that weights are 2^LIFT exp2(scale (s - m)). WIDE: m is the reference of the weights 2^(x - m), base 2
    float o[MT][NT][4], zacc[NT][NG][2], m[NT][2], nm[NT][2], l[NT][2];
    const float scale = a.scale_log2 * pow2(CODE_EXP - LIFT);
    const float unseen = WIDE ? NEG : fmaxf(NEG / scale, -1e38f);   // scale times it is finite, at any scale
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < MT; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) zacc[nt][g][0] = zacc[nt][g][1] = 0.f;
        m[nt][0] = m[nt][1] = unseen;
        nm[nt][0] = nm[nt][1] = -unseen * scale;
        l[nt][0] = l[nt][1] = 0.f;
    }
    const float minus_hi = t < 2 ? 0.f : -1.f;   // columns 4..7 of the doubled units (t >= 2) carry the lo halves
    uint32_t bad[NT][2] = {};   // WIDE: groups of V stored as NaN that the column sees
    Kv4Unit unit;   // WIDE: powers of two of the step's values and of O
    int failed = -1;   // the pair whose copy did not land within the bound

    // one pair of tiles; EDGE: some of its keys are not seen by some unit, or a page is missing
    auto pair_step = [&](auto edge_tag, const unsigned char* tp, int k0, bool ok0, bool ok1) {
        constexpr bool EDGE = decltype(edge_tag)::value;
        float sc[2][NT][4];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const unsigned char* kt = tp + x * TB;
            uint32_t kp[2][NG], kc[NB][4];
#pragma unroll
            for (int y = 0; y < NB; ++y)
                *reinterpret_cast<uint4*>(kc[y]) = *reinterpret_cast<const uint4*>(kt + y * T::BLK + lane * 16);
#pragma unroll
            for (int y = 0; y < 2 * NG; y += 4)
                *reinterpret_cast<uint4*>(&kp[0][0] + y) = *reinterpret_cast<const uint4*>(kt + T::KP + r * 8 * NG + y * 4);
            uint32_t az[4] = {};   // z of the keys
#pragma unroll
            for (int y = 0; y < NG; ++y) az[y] = __byte_perm(kp[y & 1][y & 2], kp[y & 1][(y & 2) + 1], 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                sc[x][nt][0] = sc[x][nt][1] = sc[x][nt][2] = sc[x][nt][3] = 0.f;
                mma16816(sc[x][nt], az, zq[nt][0], zq[nt][1], sc[x][nt]);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t a0[4], a1[4];
                unpack(kc[g >> 1][g & 1], a0[0], a0[2], a1[0], a1[2]);
                unpack(kc[g >> 1][2 + (g & 1)], a0[1], a0[3], a1[1], a1[3]);
                const float s0 = kv4_s(kp[0][g]), s8 = kv4_s(kp[1][g]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
                    mma16816(acc, a0, qf[nt][4 * g], qf[nt][4 * g + 1], acc);
                    mma16816(acc, a1, qf[nt][4 * g + 2], qf[nt][4 * g + 3], acc);
                    float* c = sc[x][nt];
                    c[0] = fmaf(s0, acc[0], c[0]);
                    c[1] = fmaf(s0, acc[1], c[1]);
                    c[2] = fmaf(s8, acc[2], c[2]);
                    c[3] = fmaf(s8, acc[3], c[3]);
                }
            }
        }
        bool see[2][NT][4], up = false;
        float p[2][NT][4], ls[NT][2];
        auto weigh = [&]() {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                ls[nt][0] = l[nt][0];
                ls[nt][1] = l[nt][1];
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[x][nt][e] = kv4_ex2(fmaf(sc[x][nt][e], scale, nm[nt][e & 1]));
                        ls[nt][e & 1] += p[x][nt][e];
                    }
            }
        };
        if (EDGE) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int k = k0 + 16 * x + r + (e < 2 ? 0 : 8);
                        see[x][nt][e] = (x ? ok1 : ok0) && k >= lo[nt][e & 1] && k < hi[nt][e & 1];
                        if (!see[x][nt][e]) sc[x][nt][e] = -INFINITY;
                    }
        }
        weigh();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) up |= ls[nt][0] > pow2(LIFT + LAZY) || ls[nt][1] > pow2(LIFT + LAZY);
        if (__any_sync(0xffffffffu, up)) {   // the sums would soon leave the range: move the maximum, weigh again
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float x = fmaxf(fmaxf(sc[0][nt][c], sc[0][nt][c + 2]), fmaxf(sc[1][nt][c], sc[1][nt][c + 2]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    x = fmaxf(x, m[nt][c]);
                    const float f = kv4_ex2((m[nt][c] - x) * scale);
                    m[nt][c] = x;
                    nm[nt][c] = fmaf(-x, scale, (float)LIFT);
                    l[nt][c] *= f;
#pragma unroll
                    for (int g = 0; g < NG; ++g) zacc[nt][g][c] *= f;
#pragma unroll
                    for (int y = 0; y < MT; ++y) {
                        o[y][nt][c] *= f;
                        o[y][nt][c + 2] *= f;
                    }
                }
            weigh();
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            l[nt][0] = ls[nt][0];
            l[nt][1] = ls[nt][1];
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const unsigned char* vt = tp + x * TB;
            uint32_t vp[2][NG], vc[NB][4];
#pragma unroll
            for (int y = 0; y < NB; ++y)
                *reinterpret_cast<uint4*>(vc[y]) = *reinterpret_cast<const uint4*>(vt + T::V + y * T::BLK + lane * 16);
#pragma unroll
            for (int y = 0; y < 2 * NG; y += 4)
                *reinterpret_cast<uint4*>(&vp[0][0] + y) = *reinterpret_cast<const uint4*>(vt + T::VP + r * 8 * NG + y * 4);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t a0[4], a1[4];
                unpack(vc[g >> 1][2 * (g & 1)], a0[0], a0[1], a1[0], a1[1]);
                unpack(vc[g >> 1][2 * (g & 1) + 1], a0[2], a0[3], a1[2], a1[3]);
                const float s0 = kv4_s(vp[0][g]), z0 = kv4_z(vp[0][g]), s8 = kv4_s(vp[1][g]), z8 = kv4_z(vp[1][g]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float* pp = p[x][nt];
                    float w[4] = {pp[0] * s0, pp[1] * s0, pp[2] * s8, pp[3] * s8};
                    float* za = zacc[nt][g];
                    if (EDGE) {   // what a unit does not see may hold anything: left out, not multiplied by 0
                        const bool* y = see[x][nt];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            w[e] = y[e] ? w[e] : 0.f;
                            za[e & 1] += y[e] ? pp[e] * (e < 2 ? z0 : z8) : 0.f;
                        }
                    } else {
                        za[0] = fmaf(pp[0], z0, fmaf(pp[2], z8, za[0]));
                        za[1] = fmaf(pp[1], z0, fmaf(pp[3], z8, za[1]));
                    }
                    uint32_t pa = pack(w[0], w[1]), pb = pack(w[2], w[3]);   // hi halves
                    const uint32_t ha = pa, hb = pb;
                    if (DUP) {   // of the columns that carry the lo halves: those
                        pa = pack(fmaf(lo_of(ha), minus_hi, w[0]), fmaf(hi_of(ha), minus_hi, w[1]));
                        pb = pack(fmaf(lo_of(hb), minus_hi, w[2]), fmaf(hi_of(hb), minus_hi, w[3]));
                    }
                    const uint32_t b0 = movmatrix(pa), b1 = movmatrix(pb);
                    mma16816(o[2 * g][nt], a0, b0, b1, o[2 * g][nt]);
                    mma16816(o[2 * g + 1][nt], a1, b0, b1, o[2 * g + 1][nt]);
                    if (!DUP) {
                        const uint32_t c0 = movmatrix(pack(w[0] - lo_of(ha), w[1] - hi_of(ha)));
                        const uint32_t c1 = movmatrix(pack(w[2] - lo_of(hb), w[3] - hi_of(hb)));
                        mma16816(o[2 * g][nt], a0, c0, c1, o[2 * g][nt]);
                        mma16816(o[2 * g + 1][nt], a1, c0, c1, o[2 * g + 1][nt]);
                    }
                }
            }
        }
    };

    // The same with keys and values unpacked to fp16 numbers, s and z applied: more work a tile and less
    // a unit (no s and z on scores, one operand of weights instead of two a group). 2^ek, 2^ev come
    // out of the pair's keys and values: x = 2^ek q.k scale, weights 2^(x + ev - er - m), l = sum 2^(er - ev) weight
    auto wide_step = [&](auto edge_tag, const unsigned char* tp, int k0, bool ok0, bool ok1) {
        constexpr bool EDGE = decltype(edge_tag)::value;
        auto known = [&](int x, int token) {   // some unit sees the token
            const int key = k0 + 16 * x + token;
            return !EDGE || ((x ? ok1 : ok0) && key >= rg.kmin && key < rg.kmax);
        };
        uint32_t topk = 0, topv = 0;
        bool nan_v = false;
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int y = 0; y < NB; ++y) {
                const int at = 32 * y + lane, slot = at / NG;
                const bool in = known(x, (slot >> 1) + 8 * (slot & 1));
                const uint32_t kw = *reinterpret_cast<const uint32_t*>(tp + x * TB + T::KP + 4 * at);
                const uint32_t vw = *reinterpret_cast<const uint32_t*>(tp + x * TB + T::VP + 4 * at);
                topk = max(topk, in ? kv4_top(kw) : 0u);
                topv = max(topv, in ? kv4_top(vw) : 0u);
                if (EDGE) nan_v |= in && !(kv4_z(vw) == kv4_z(vw));
            }
        topk = __reduce_max_sync(0xffffffffu, topk);
        topv = __reduce_max_sync(0xffffffffu, topv);
        if (EDGE) nan_v = __any_sync(0xffffffffu, nan_v);
        const int ek = kv4_exponent_out(topk);
        unit.ev = kv4_exponent_out(topv);
        const float fk = kv4_exp2i(-ek);
        float sc[2][NT][4], kq[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            kq[nt][0] = kv4_score_factor(q_scale[nt][0], kv4_exp2i(ek));
            kq[nt][1] = kv4_score_factor(q_scale[nt][1], kv4_exp2i(ek));
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const unsigned char* kt = tp + x * TB;
            uint32_t kp[2][NG], kc[NB][4];
#pragma unroll
            for (int y = 0; y < NB; ++y)
                *reinterpret_cast<uint4*>(kc[y]) = *reinterpret_cast<const uint4*>(kt + y * T::BLK + lane * 16);
#pragma unroll
            for (int y = 0; y < 2 * NG; y += 4)
                *reinterpret_cast<uint4*>(&kp[0][0] + y) = *reinterpret_cast<const uint4*>(kt + T::KP + r * 8 * NG + y * 4);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[x][nt][0] = sc[x][nt][1] = sc[x][nt][2] = sc[x][nt][3] = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t w0[4], w8[4];
                const float s0 = kv4_s(kp[0][g]) * fk, z0 = kv4_z(kp[0][g]) * fk, s8 = kv4_s(kp[1][g]) * fk,
                            z8 = kv4_z(kp[1][g]) * fk;
                kv4_unpack4(kc[g >> 1][g & 1], kv4_half2(s0, s0), kv4_half2(z0, z0), w0);
                kv4_unpack4(kc[g >> 1][2 + (g & 1)], kv4_half2(s8, s8), kv4_half2(z8, z8), w8);
                const uint32_t a0[4] = {w0[0], w8[0], w0[1], w8[1]}, a1[4] = {w0[2], w8[2], w0[3], w8[3]};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16816h(sc[x][nt], a0, qf[nt][4 * g], qf[nt][4 * g + 1], sc[x][nt]);
                    mma16816h(sc[x][nt], a1, qf[nt][4 * g + 2], qf[nt][4 * g + 3], sc[x][nt]);
                }
            }
        }
        if (EDGE) {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int k = k0 + 16 * x + r + (e < 2 ? 0 : 8);
                        const bool see = (x ? ok1 : ok0) && k >= lo[nt][e & 1] && k < hi[nt][e & 1];
                        if (!see) sc[x][nt][e] = -INFINITY;
                        if (nan_v && see) {   // rare
#pragma unroll
                            for (int g = 0; g < NG; ++g) {
                                const float z = kv4_z(*reinterpret_cast<const uint32_t*>(
                                    tp + x * TB + T::VP + ((2 * r + (e < 2 ? 0 : 1)) * NG + g) * 4));
                                if (!(z == z)) bad[nt][e & 1] |= 1u << g;
                            }
                        }
                    }
        }
        uint32_t p[2][NT][2];   // weights, fp16 pairs (token r; token r + 8)
        float ls[NT][2];
        auto weigh = [&]() {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                ls[nt][0] = ls[nt][1] = 0.f;
                const float b0 = (float)(unit.ev - unit.er) - m[nt][0], b1 = (float)(unit.ev - unit.er) - m[nt][1];
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float w0 = kv4_ex2(fmaf(sc[x][nt][2 * y], kq[nt][0], b0));
                        const float w1 = kv4_ex2(fmaf(sc[x][nt][2 * y + 1], kq[nt][1], b1));
                        ls[nt][0] += w0;
                        ls[nt][1] += w1;
                        p[x][nt][y] = kv4_half2(w0, w1);
                    }
            }
        };
        weigh();
        bool up = !unit.holds(unit.ev);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) up |= ls[nt][0] > KV4_FULL || ls[nt][1] > KV4_FULL;
        if (__any_sync(0xffffffffu, up)) {   // fp16 would soon be left: move the references, weigh again
            const float moved = unit.next(topv), shift = (float)(unit.ev - unit.er);   // O into a new unit
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float x = fmaxf(fmaxf(sc[0][nt][c], sc[0][nt][c + 2]), fmaxf(sc[1][nt][c], sc[1][nt][c + 2]));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    x = fmaxf(fmaf(x, kq[nt][c], shift) - KV4_ROOM, m[nt][c]);
                    const float f = kv4_ex2(m[nt][c] - x);
                    m[nt][c] = x;
                    l[nt][c] *= f;
#pragma unroll
                    for (int y = 0; y < MT; ++y) {
                        o[y][nt][c] *= f * moved;
                        o[y][nt][c + 2] *= f * moved;
                    }
                }
            weigh();
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            l[nt][0] = fmaf(ls[nt][0], kv4_exp2i(unit.er - unit.ev), l[nt][0]);
            l[nt][1] = fmaf(ls[nt][1], kv4_exp2i(unit.er - unit.ev), l[nt][1]);
        }
        const float fv = kv4_exp2i(-unit.ev);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const unsigned char* vt = tp + x * TB;
            uint32_t vp[4 * NG], vc[NB][4], b0[NT], b1[NT];
#pragma unroll
            for (int y = 0; y < NB; ++y)
                *reinterpret_cast<uint4*>(vc[y]) = *reinterpret_cast<const uint4*>(vt + T::V + y * T::BLK + lane * 16);
#pragma unroll
            for (int y = 0; y < 4 * NG; y += 4)   // tokens 2t, 2t + 8, 2t + 1, 2t + 9
                *reinterpret_cast<uint4*>(vp + y) = *reinterpret_cast<const uint4*>(vt + T::VP + t * 16 * NG + y * 4);
            if (EDGE) {   // what no unit sees, and NaN groups (in bad): zero
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int g = 0; g < NG; ++g)
                        if (!known(x, 2 * t + (y >> 1) + 8 * (y & 1)) || !(kv4_z(vp[y * NG + g]) == kv4_z(vp[y * NG + g])))
                            vp[y * NG + g] = 0u;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                b0[nt] = movmatrix(p[x][nt][0]);
                b1[nt] = movmatrix(p[x][nt][1]);
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t w[2][4];
#pragma unroll
                for (int y = 0; y < 2; ++y) {   // tokens 2t, 2t + 1 and 8 further
                    const uint32_t p0 = vp[y * NG + g], p1 = vp[(2 + y) * NG + g];
                    kv4_unpack4(vc[g >> 1][2 * (g & 1) + y], kv4_half2(kv4_s(p0) * fv, kv4_s(p1) * fv),
                                kv4_half2(kv4_z(p0) * fv, kv4_z(p1) * fv), w[y]);
                }
                const uint32_t a0[4] = {w[0][0], w[0][1], w[1][0], w[1][1]}, a1[4] = {w[0][2], w[0][3], w[1][2], w[1][3]};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma16816h(o[2 * g][nt], a0, b0[nt], b1[nt], o[2 * g][nt]);
                    mma16816h(o[2 * g + 1][nt], a1, b0[nt], b1[nt], o[2 * g + 1][nt]);
                }
            }
        }
    };
    auto step = [&](auto edge_tag, const unsigned char* tp, int k0, bool ok0, bool ok1) {
        if constexpr (WIDE)
            wide_step(edge_tag, tp, k0, ok0, ok1);
        else
            pair_step(edge_tag, tp, k0, ok0, ok1);
    };

    for (int i = 0; i < mine; ++i) {
        const int st = i % S;
        if (i > 0 && (i & 31) == 0) here = next;
        const bool ok0 = here.ok0 >> (i & 31) & 1, ok1 = here.ok1 >> (i & 31) & 1;
        if (!mbar_wait(&bars[warp][st], (i / S) & 1)) {
            failed = i;
            break;
        }
        const int k0 = (p_begin + i * WARPS) * 32;
        const unsigned char* tp = ring + st * 2 * TB;
        if (k0 >= all_lo && k0 + 32 <= all_hi && ok0 && ok1)
            step(std::false_type{}, tp, k0, true, true);
        else if (ok0 || ok1)
            step(std::true_type{}, tp, k0, ok0, ok1);
        __syncwarp();   // every lane has read the stage
        const int nx = i + S;
        if (nx < mine) {
            if ((nx & 31) == 0) next = locate(nx);
            if (lane == (nx & 31)) issue(nx, (nx >> 5) == (i >> 5) ? here : next);
        }
    }
    if (failed >= 0)   // let the copies in flight land (bounded again) and answer NaN
        for (int i = failed; i < min(mine, failed + S); ++i) mbar_wait(&bars[warp][i % S], (i / S) & 1);

    // join the warps: m, l and O of every unit through shared memory (the ring is drained)
    __syncthreads();
    float* wo = reinterpret_cast<float*>(sm) + warp * UT * (HD + 2);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int u = DUP ? ((2 * t + c) & 3) : nt * 8 + 2 * t + c;
            float s = l[nt][c];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
            if (failed >= 0) s = __int_as_float(0x7fffffff);
            if (r == 0 && (!DUP || t < 2)) {
                wo[u * (HD + 2) + HD] = WIDE ? m[nt][c] + (float)unit.er : m[nt][c] * scale;
                wo[u * (HD + 2) + HD + 1] = s * (WIDE ? kv4_exp2i(-unit.er) : pow2(-LIFT));
            }
            uint32_t none = bad[nt][c];
            if (WIDE) none = __reduce_or_sync(0x11111111u << t, none);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float z = zacc[nt][g][c];
                if (WIDE) {
                    z = none >> g & 1 ? __int_as_float(0x7fffffff) : 0.f;
                } else {
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) z += __shfl_xor_sync(0xffffffffu, z, x);
                    z *= pow2(-LIFT);
                }
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = o[2 * g + x][nt][c + 2 * e];
                        if (DUP) v += __shfl_xor_sync(0xffffffffu, v, 2);
                        if (!DUP || t < 2)
                            wo[u * (HD + 2) + 32 * g + 16 * x + 8 * e + r] =
                                fmaf(v, WIDE ? 1.f : pow2(CODE_EXP - LIFT - 4 * e), z);
                    }
            }
        }
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(sm);
    float* mine_o = reinterpret_cast<float*>(sm) + WARPS * UT * (HD + 2);   // cluster: the CTA's own, for the others
    const int items = (ulast - u0 + 1) * (HD / 2);   // two dims each
    auto place = [&](int u) {
        const int j = kv4_row(a, u0 + u), g = (u0 + u) - j * a.group;
        return (int64_t)(row0 + j) * a.hq + h * a.group + g;
    };
    auto answer = [&](int u, int d, float ll, float2 oo) {
        const __nv_bfloat162 v = ll == 0.f ? __floats2bfloat162_rn(0.f, 0.f) : __floats2bfloat162_rn(oo.x / ll, oo.y / ll);
        *reinterpret_cast<__nv_bfloat162*>(a.out + place(u) * HD + d) = v;
    };
    for (int i = tid; i < items; i += WARPS * 32) {
        const int u = i / (HD / 2), d = i % (HD / 2) * 2;
        float mm = NEG, ll = 0.f;
        float2 oo = make_float2(0.f, 0.f), ml[WARPS];
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            ml[w] = *reinterpret_cast<const float2*>(all + (w * UT + u) * (HD + 2) + HD);
            mm = fmaxf(mm, ml[w].x);
        }
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float f = kv4_ex2(ml[w].x - mm);
            const float2 p = *reinterpret_cast<const float2*>(all + (w * UT + u) * (HD + 2) + d);
            ll = fmaf(f, ml[w].y, ll);
            oo = make_float2(fmaf(f, p.x, oo.x), fmaf(f, p.y, oo.y));
        }
        if (a.cluster) {
            float* p = mine_o + u * (HD + 2);
            *reinterpret_cast<float2*>(p + d) = oo;
            if (d == 0) *reinterpret_cast<float2*>(p + HD) = make_float2(mm, ll);
        } else if (rg.used == 1) {
            answer(u, d, ll, oo);
        } else {
            const int64_t at = place(u) * a.nsplit + split;
            *reinterpret_cast<float2*>(a.part_o + at * HD + d) = oo;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(mm, ll);
        }
    }
    if (!a.cluster) return;
    // the splits are a cluster: each CTA joins a part of the dims from all of their shared memories
    cluster_sync();
    for (int i = split * WARPS * 32 + tid; i < items; i += a.nsplit * WARPS * 32) {
        const int u = i / (HD / 2), d = i % (HD / 2) * 2;
        const float* p = mine_o + u * (HD + 2);
        float mm = NEG, ll = 0.f;
        float2 oo = make_float2(0.f, 0.f);
        for (int sp = 0; sp < a.nsplit; ++sp) mm = fmaxf(mm, ld_cluster(p + HD, sp).x);
        for (int sp = 0; sp < a.nsplit; ++sp) {
            const float2 ml = ld_cluster(p + HD, sp), x = ld_cluster(p + d, sp);
            const float f = kv4_ex2(ml.x - mm);
            ll = fmaf(f, ml.y, ll);
            oo = make_float2(fmaf(f, x.x, oo.x), fmaf(f, x.y, oo.y));
        }
        answer(u, d, ll, oo);
    }
    cluster_sync();   // nobody leaves while its shared memory is read
}

// out of one (sequence row, head) from its splits' partials (where there is more than one): 128
// threads, HD / 4 to a partial; NG groups of these go through every NG-th split of one (row, head) and
// are joined in shared memory, the others of the block have rows of their own. Both orders are fixed.
template <int HD, int NG>
__global__ void __launch_bounds__(128) k_kv4_merge(const Kv4AttnArgs a) {
    constexpr int LN = HD / 4, PER = 128 / LN / NG;   // (row, head) pairs of a block
    __shared__ float4 os[NG > 1 ? NG : 1][LN];
    __shared__ float2 mls[NG];
    const int d = threadIdx.x % LN, g = threadIdx.x / LN % NG, b = blockIdx.y;
    const int jh = blockIdx.x * PER + threadIdx.x / (LN * NG), j = jh / a.hq, head = jh % a.hq;
    const int u = j * a.group + head % a.group;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the attention kernel's partials are there
    Kv4Range rg;
    if (!kv4_range(a, b, u - u % a.unit_tile, a.unit_tile, a.step, rg) || u >= rg.units || rg.used == 1) return;
    const int64_t at = (int64_t)(rg.row0 + j) * a.hq + head;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + at * a.nsplit;
    const float4* po = reinterpret_cast<const float4*>(a.part_o) + at * a.nsplit * LN + d;
    float m = NEG, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = g; s0 < rg.used; s0 += 4 * NG) {
        float2 x[4];
        float4 y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int s = s0 + i * NG;
            x[i] = s < rg.used ? ml[s] : make_float2(NEG, 0.f);
            y[i] = s < rg.used ? po[(int64_t)s * LN] : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const float top = fmaxf(fmaxf(fmaxf(x[0].x, x[1].x), fmaxf(x[2].x, x[3].x)), m);
        float f = kv4_ex2(m - top);
        m = top;
        l *= f;
        o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f = kv4_ex2(x[i].x - top);
            l = fmaf(f, x[i].y, l);
            o = make_float4(fmaf(f, y[i].x, o.x), fmaf(f, y[i].y, o.y), fmaf(f, y[i].z, o.z), fmaf(f, y[i].w, o.w));
        }
    }
    if (NG > 1) {   // (the block has one pair: all its threads are here)
        os[g][d] = o;
        if (d == 0) mls[g] = make_float2(m, l);
        __syncthreads();
        if (g > 0) return;
        float top = NEG;
#pragma unroll
        for (int i = 0; i < NG; ++i) top = fmaxf(top, mls[i].x);
        l = 0.f;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const float f = kv4_ex2(mls[i].x - top);
            const float4 y = os[i][d];
            l = fmaf(f, mls[i].y, l);
            o = make_float4(fmaf(f, y.x, o.x), fmaf(f, y.y, o.y), fmaf(f, y.z, o.z), fmaf(f, y.w, o.w));
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const __nv_bfloat162 lo2 = __floats2bfloat162_rn(o.x * inv, o.y * inv), hi2 = __floats2bfloat162_rn(o.z * inv, o.w * inv);
    uint2 v;
    v.x = *reinterpret_cast<const uint32_t*>(&lo2);
    v.y = *reinterpret_cast<const uint32_t*>(&hi2);
    *reinterpret_cast<uint2*>(a.out + at * HD + 4 * d) = v;
}

struct Plan {
    bool many;   // k_kv4_prefill
    int nt, dup, warps, unit_tile, utiles, step, nsplit, split_len, cluster;
};

// Splits of `steps` steps of the keys.
void split(Plan& p, int64_t steps, int64_t ns) {
    p.split_len = (int)((steps + ns - 1) / ns);
    if (p.split_len < 1) p.split_len = 1;
    p.nsplit = (int)((steps + p.split_len - 1) / p.split_len);
    if (p.nsplit < 1) p.nsplit = 1;
}
// The steps that a tile of ut units can need.
int64_t steps_of(int64_t ut, int64_t step, int64_t group, int64_t max_q, int64_t max_kv, int64_t window) {
    int64_t span = max_kv;
    if (window > 0) {
        const int64_t rows = (ut + group - 1) / group + 1;   // rows that a unit tile can touch
        const int64_t w = window + (rows < max_q ? rows : max_q) + step;
        if (w < span) span = w;
    }
    return (span + step - 1) / step;
}

// k_kv4_attn: the fewest columns that hold max_q rows of a group (four: both halves of the weights in one
// operand), at most 32 (heads of 128: 16, for the registers).
// Splits of the keys: as many as the SMs hold at once, of at least 8 pairs of tiles (two a warp); where
// there are many keys, of 32 to 64 pairs, so that sequences shorter than max_kv even out (the splits that
// they lack end at once). One that starts a second wave costs more than it evens out: 33 x 2000 keys with 2
// rows in 5 / 4 splits 18.4 / 12.0 us, with 5 rows in 3 / 2 34.9 / 22.6, 7 x 9000 in 22 / 21 14.6 / 11.8.
// Measured around it: 4 x 32768, 18 to 37 splits 19 to 19.6 us, 8 31, 74 23; 256 x 640, one 21.8, two 27;
// 48 x 1..8191 of heads of 128, 2 / 4 / 8 / 12 / 16 splits 93 / 81 / 77 / 81 / 83.
// Two warps instead of four where there is a CTA for every unit tile and each has few keys: what a CTA
// costs besides its keys is paid per warp (256 x 640: 21.8 us, with four 22.6).
// A cluster joins its splits through shared memory where there are at most eight and all clusters fit at
// once; each stays inside one of the GPU's eight parts, which hold 17 SMs or more. Measured against
// partials in memory and k_kv4_merge: 1 x 2048 6.2 / 6.5 us (on the host 12 / 22 a call: one launch and no
// workspace), 16 x 1024 6.7 / 7.7, 33 x 2000 with 2 rows 12.0 / 13.4, with 5 rows 22.9 / 25.3, heads of 128,
// 1 x 512 8.4 / 7.8; filling the SMs further: 96 clusters of 6 18.5 / 15.0, 80 of 7 27.5 / 22.3.
// cost: its time in us, for more than 32 units.
Plan plan_attn(int64_t B, int64_t Hkv, int64_t group, int head_dim, int64_t max_q, int64_t max_kv, int64_t window,
               double& cost) {
    Plan p{};
    const int64_t units = max_q * group, cap = head_dim == 64 ? 4 : 2;
    p.dup = units <= 4;
    p.nt = (int)(units > 8 * cap ? cap : (units + 7) / 8);
    p.unit_tile = p.dup ? 4 : 8 * p.nt;
    p.step = 32;
    p.utiles = (int)((units + p.unit_tile - 1) / p.unit_tile);
    const int64_t steps = steps_of(p.unit_tile, p.step, group, max_q, max_kv, window), ctas = B * Hkv * p.utiles;
    const int64_t fill = 148 * resident(head_dim, p.nt);   // CTAs that the GPU holds at once
    int64_t ns = fill / ctas;
    if (ns > steps / 8) ns = steps / 8;
    if (ctas * ((steps + 63) / 64) > fill && ns < (steps + 63) / 64) ns = (steps + 31) / 32;
    if (ns > 128) ns = 128;
    if (ns < 1) ns = 1;
    p.warps = p.nt == 1 && ns == 1 && ctas > 148 * 4 && steps <= 64 ? 2 : 4;
    split(p, steps, ns);
    p.cluster = p.nsplit > 1 && p.nsplit <= 8 && ctas <= 8 * (17 * resident(head_dim, p.nt) / p.nsplit);
    const double waves = (double)((ctas * p.nsplit + fill - 1) / fill), pairs = (p.split_len + 3) / 4;
    cost = 5 + waves * (head_dim == 64 ? 8 + pairs * (waves > 1 ? 2.0 : 1.45) : 6 + pairs * (waves > 1 ? 2.5 : 2.0)) +
           (p.nsplit > 1 && !p.cluster ? 3 : 0);
    return p;
}

// k_kv4_prefill: the splits that make the cost (us) least: the launch; for every wave of CTAs their start
// and end and their steps, by the tiles of 128 units that a CTA has; the partials' way through memory.
// 2048 rows on 16384 keys in 1 / 2 / 3 / 4 splits 441 / 241 / 321 / 254 us, on 2048 keys 69 / 53 / 51 / 61, 4096 rows
// with a window of 1024 52 / 85 / 104 / 102, 1500 with one of 1000 on 16384 keys 55 / 48 / 46 / 63, 33 rows on
// 16000 keys in 1 / 8 / 32 splits 350 / 57 / 28.
Plan plan_prefill(int64_t B, int64_t Hkv, int64_t group, int head_dim, int64_t max_q, int64_t max_kv, int64_t window,
                  double& cost) {
    Plan p{};
    const int64_t units = max_q * group;
    p.many = true;
    p.warps = 4;
    p.unit_tile = kv4_pf_units(head_dim);
    p.step = KV4_PF_STEP;
    p.utiles = (int)((units + p.unit_tile - 1) / p.unit_tile);
    const int64_t steps = steps_of(p.unit_tile, p.step, group, max_q, max_kv, window), ctas = B * Hkv * p.utiles;
    const double tiles = (double)(p.utiles > 1 ? p.unit_tile / 128 : (units + 127) / 128);
    const double ends = head_dim == 64 ? 1.5 + 3.5 * tiles : 10 * tiles, step = head_dim == 64 ? 1.2 + 0.55 * tiles : 1.4 + 0.8 * tiles;
    const int64_t most = steps / 2 < 64 ? steps / 2 : 64;
    int64_t ns = 1;
    cost = 1e30;
    for (int64_t s = 1; s <= most || s == 1; ++s) {
        const double waves = (double)((ctas * s + 147) / 148), len = (double)((steps + s - 1) / s);
        const double c = 6 + waves * (ends + len * step) +
                         (s > 1 ? 1 + (double)(B * Hkv * units) * s * (head_dim + 2) * 8 / 4e6 : 0);
        if (c < cost) {
            cost = c;
            ns = s;
        }
    }
    split(p, steps, ns);
    return p;
}

// How a call is cut. Up to 32 units a sequence k_kv4_attn; above, the kernel that costs less, which with
// few keys is k_kv4_attn up to some hundred units. Measured (k_kv4_attn / k_kv4_prefill, us), 4 kv heads of 64:
// 512 keys, 40 units 15.9 / 14.4, 256 16.4 / 18.6, 800 18 / 26; 4096 keys, 64 units 17.2 / 15.4, 512 25.9 / 30.8,
// 800 38.6 / 32.8; 16384 keys, 32 units 19.0 / 21.1, 128 28 / 24, 512 91 / 39; 8 x 4096, 64 units 25.7 / 30.8, 128
// 39 / 32; 64 x 2048, 32 units 38 / 86, 40 92 / 85; heads of 128: 512 keys, 256 units 16 / 29; 4096 keys, 256
// units 27 / 33, 512 44 / 34; 64 x 2048, 32 units 104 / 109, 40 144 / 110.
Plan make_plan(int64_t B, int64_t Hkv, int64_t group, int64_t head_dim, int64_t max_q, int64_t max_kv,
               int64_t window) {
    double cost, other;
    const Plan p = plan_attn(B, Hkv, group, (int)head_dim, max_q, max_kv, window, cost);
    if (max_q * group <= 32) return p;
    const Plan q = plan_prefill(B, Hkv, group, (int)head_dim, max_q, max_kv, window, other);
    return other < cost ? q : p;
}

template <int HD, int NT, bool DUP, int WARPS>
int launch(const Kv4AttnArgs& a, const Plan& p, int64_t B, cudaStream_t st) {
    constexpr int ring = WARPS * stages<HD>() * 2 * Kv4Tile<HD>::BYTES, merge = (WARPS + 1) * (DUP ? 4 : 8 * NT) * (HD + 2) * 4;
    constexpr int bytes = ring > merge ? ring : merge;
    PULSAR_TRY(ensure_smem_attr((const void*)k_kv4_attn<HD, NT, DUP, WARPS>, bytes, "k_kv4_attn shared memory"));
    const dim3 grid((unsigned)(p.utiles * p.nsplit), (unsigned)a.hkv, (unsigned)B);
    if (!p.cluster) {
        k_kv4_attn<HD, NT, DUP, WARPS><<<grid, WARPS * 32, bytes, st>>>(a);
        PULSAR_LAUNCH_CHECK("k_kv4_attn");
        return PULSAR_OK;
    }
    cudaLaunchAttribute splits{};
    splits.id = cudaLaunchAttributeClusterDimension;
    splits.val.clusterDim.x = (unsigned)p.nsplit;
    splits.val.clusterDim.y = splits.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = st;
    cfg.attrs = &splits;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, k_kv4_attn<HD, NT, DUP, WARPS>, a), "k_kv4_attn");
}

// The merge is launched under the attention kernel's end; it waits for that before it reads. Up to
// four splits a group of threads takes them all, above all groups of a block share those of one row:
// with one group / all, 64 x 2048 in 4 splits 18.9 / 20.4 us, 2048 rows on 16384 in 2 240 / 277,
// 4 x 32768 in 37 25.7 / 20.2, 8 splits even.
template <int HD>
int launch_merge(const Kv4AttnArgs& a, int64_t B, cudaStream_t st) {
    constexpr int ALL = 512 / HD;   // groups of a block
    const bool few = a.nsplit <= 4;
    const int64_t rows = (int64_t)a.max_q * a.hq;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(few ? (rows + ALL - 1) / ALL : rows), (unsigned)B);
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cuda_status(few ? cudaLaunchKernelEx(&cfg, k_kv4_merge<HD, 1>, a) : cudaLaunchKernelEx(&cfg, k_kv4_merge<HD, ALL>, a),
                       "k_kv4_merge");
}

int check_shape(int64_t N, int64_t Hq, int64_t Hkv, int64_t head_dim, int64_t B, int64_t max_q, int64_t max_kv,
                int64_t window) {
    PULSAR_CHECK_ARG(head_dim == 64 || head_dim == 128, "kv4_attention: head_dim must be 64 or 128, got %lld",
                     (long long)head_dim);
    PULSAR_CHECK_ARG(Hkv >= 1 && Hkv <= 1024 && Hq >= Hkv && Hq % Hkv == 0 && Hq / Hkv <= 1024,
                     "kv4_attention: %lld query heads over %lld kv heads", (long long)Hq, (long long)Hkv);
    PULSAR_CHECK_ARG(N >= 0 && N < (int64_t)1 << 31 && B >= 0 && B <= 65535, "kv4_attention: invalid batch");
    PULSAR_CHECK_ARG(max_q >= 1 && max_q * (Hq / Hkv) < (int64_t)1 << 30, "kv4_attention: max_q must be at least 1");
    PULSAR_CHECK_ARG(max_kv >= 1 && max_kv < (int64_t)1 << 30 && window >= 0 && window < (int64_t)1 << 30,
                     "kv4_attention: invalid max_kv or window");
    return PULSAR_OK;
}

}  // namespace

extern "C" int pulsar_op_kv4_attention_workspace(int64_t N, int64_t Hq, int64_t Hkv, int64_t head_dim, int64_t B,
                                                 int64_t max_q, int64_t max_kv, int64_t window, int64_t* bytes) {
    PULSAR_CHECK_ARG(bytes, "kv4_attention_workspace: null pointer");
    PULSAR_TRY(check_shape(N, Hq, Hkv, head_dim, B, max_q, max_kv, window));
    const Plan p = make_plan(B > 0 ? B : 1, Hkv, Hq / Hkv, head_dim, max_q, max_kv, window);
    *bytes = p.nsplit > 1 && !p.cluster ? N * Hq * p.nsplit * (head_dim + 2) * 4 : 0;
    return PULSAR_OK;
}

extern "C" int pulsar_op_kv4_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride, int64_t N,
                                       int64_t Hq, int64_t head_dim, const void* pages, int64_t num_pages,
                                       int64_t page_size, int64_t Hkv, const int32_t* block_table, int64_t B,
                                       int64_t width, const int32_t* kv_lens, const int32_t* cu_q, int64_t max_q,
                                       int64_t max_kv, float scale, int64_t window, void* workspace,
                                       int64_t workspace_bytes, void* out, void* stream) {
    PULSAR_TRY(check_shape(N, Hq, Hkv, head_dim, B, max_q, max_kv, window));
    PULSAR_CHECK_ARG(page_size >= 16 && page_size <= 65536 && (page_size & (page_size - 1)) == 0,
                     "kv4_attention: page_size must be a power of two of at least 16, got %lld", (long long)page_size);
    PULSAR_CHECK_ARG(num_pages >= 0 && num_pages < (int64_t)1 << 31 && width >= 0 && width * page_size < (int64_t)1 << 30,
                     "kv4_attention: invalid page table");
    PULSAR_CHECK_ARG(scale > 0.f && scale < INFINITY, "kv4_attention: scale must be positive and finite");
    // k_kv4_attn's scores up to 8 units are in units of 2^(LIFT - CODE_EXP)
    PULSAR_CHECK_ARG(scale <= pow2(50) || max_q * (Hq / Hkv) > 8, "kv4_attention: a scale past 2^50 needs more than 8 units");
    PULSAR_CHECK_ARG(cu_q || (N == B && max_q == 1), "kv4_attention: without cu_q every sequence has one row");
    if (N == 0 || B == 0) return PULSAR_OK;
    PULSAR_CHECK_ARG(q && pages && kv_lens && out && (block_table || width == 0), "kv4_attention: null pointer");
    PULSAR_CHECK_ARG((reinterpret_cast<uintptr_t>(q) & 3) == 0 && q_row_stride % 2 == 0 && q_head_stride % 2 == 0,
                     "kv4_attention: q must be 4-byte aligned with even strides");
    PULSAR_CHECK_ARG(((reinterpret_cast<uintptr_t>(pages) | reinterpret_cast<uintptr_t>(out) |
                       reinterpret_cast<uintptr_t>(workspace)) & 15) == 0,
                     "kv4_attention: pages, out and the workspace must be 16-byte aligned");
    const Plan p = make_plan(B, Hkv, Hq / Hkv, head_dim, max_q, max_kv, window);
    const int64_t need = p.nsplit > 1 && !p.cluster ? N * Hq * p.nsplit * (head_dim + 2) * 4 : 0;
    PULSAR_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                     "kv4_attention: workspace of %lld bytes needed, got %lld", (long long)need,
                     (long long)workspace_bytes);
    float* ws = (float*)workspace;
    Kv4AttnArgs a{(const __nv_bfloat16*)q, (const uint8_t*)pages, block_table, kv_lens, cu_q, (__nv_bfloat16*)out, ws,
               need > 0 ? ws + N * Hq * p.nsplit * head_dim : nullptr, q_row_stride, q_head_stride,
               page_size / KV4_TILE * 20 * head_dim, (int)N, (int)Hq, (int)Hkv, (int)(Hq / Hkv), (int)num_pages,
               (int)width, __builtin_ctzll((unsigned long long)page_size), (int)max_q, (int)window, p.nsplit,
               p.split_len, p.unit_tile, p.step, p.cluster, scale * 1.4426950408889634f};
    cudaStream_t st = (cudaStream_t)stream;
    int rc;
    if (p.many)
        rc = kv4_prefill_launch(a, (int)head_dim, B, p.utiles, st);
    else if (head_dim == 64 && p.warps == 2)
        rc = p.dup ? launch<64, 1, true, 2>(a, p, B, st) : launch<64, 1, false, 2>(a, p, B, st);
    else if (head_dim == 64)
        rc = p.dup ? launch<64, 1, true, 4>(a, p, B, st) : p.nt == 1 ? launch<64, 1, false, 4>(a, p, B, st)
           : p.nt == 2 ? launch<64, 2, false, 4>(a, p, B, st) : p.nt == 3 ? launch<64, 3, false, 4>(a, p, B, st)
           : launch<64, 4, false, 4>(a, p, B, st);
    else if (p.warps == 2)
        rc = p.dup ? launch<128, 1, true, 2>(a, p, B, st) : launch<128, 1, false, 2>(a, p, B, st);
    else
        rc = p.dup ? launch<128, 1, true, 4>(a, p, B, st) : p.nt == 1 ? launch<128, 1, false, 4>(a, p, B, st)
           : launch<128, 2, false, 4>(a, p, B, st);
    PULSAR_TRY(rc);
    if (need > 0) return head_dim == 64 ? launch_merge<64>(a, B, st) : launch_merge<128>(a, B, st);
    return PULSAR_OK;
}
