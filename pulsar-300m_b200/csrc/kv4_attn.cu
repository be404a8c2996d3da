// Attention over the paged 4-bit KV cache (layout: kv4.cuh): pulsar_op_kv4_attention.
//
// Row j of the n_b query rows of sequence b has position pos = len_b - n_b + j and sees the keys
// max(0, pos - window + 1) .. pos (window 0: all of 0 .. pos):
//   out = sum_k p_k v_k / sum_k p_k,  p_k = exp(scale q.k_k - m)
// with k = s c + z per group of 32 dims, so q.k = sum_g s_g (q.c)_g + z_g sum(q)_g: the codes enter
// the matrix instruction as small whole numbers (exact in bf16) and s, z are applied in fp32 to
// its results. Values: O = sum_k (p_k s_kg) (c - 8) + sum_k p_k (z_kg + 8 s_kg): s goes into the
// weights, whose bf16 hi and lo halves are both multiplied (|x - hi - lo| <= 2^-16 |x|), and the
// second sum is a scalar per (row, group).
//
// A unit is a (query row, head of the kv head's group). CTA (split and unit tile, kv head,
// sequence): four warps, each walking every fourth 16-token tile of the split's range through a
// ring of its own (1-D bulk copies of whole tiles, issued by its lane 0; page ids are prefetched
// 32 tiles at a time, one a lane). Tokens are the M rows of S^T = K Q^T and units its N columns, so
// a tile's codes are unpacked once for all units, straight into operand registers; the weights
// pass through movmatrix into the B operand of O^T = V^T P^T. Up to four units the eight columns
// hold every unit twice and the copies carry the hi and the lo halves.
//
// The softmax keeps a running maximum per unit that moves only when a score exceeds it by more
// than 2^LAZY (l and O use the same maximum, so the result does not depend on when it moves).
// Keys that a unit does not see get weight 0 by selection, not by multiplication: pages past a
// sequence's end may hold anything, NaN included. Tiles of a page outside the cache are skipped.
//
// Splits write (m, l, O) partials; k_kv4_merge joins them in split order.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "capi_util.h"
#include "common.cuh"
#include "kv4.cuh"
#include "mega_ptx.cuh"

using namespace pulsar;

namespace {

constexpr int WARPS = 4;
constexpr float LAZY = 8.f;
constexpr float NEG = -1e30f;   // "no key yet": finite, so differences with it are defined

struct AttnArgs {
    const __nv_bfloat16* q;
    const uint8_t* pages;
    const int32_t *table, *kv_lens, *cu_q;
    __nv_bfloat16* out;
    float *part_o, *part_ml;
    int64_t q_row, q_head, page_bytes;
    int rows, hq, hkv, group, num_pages, width, page_shift, max_q, window, nsplit, split_tiles;
    float scale_log2;
};

// The rows of sequence b, held inside q whatever cu_q says.
__device__ __forceinline__ void rows_of(const AttnArgs& a, int b, int& row0, int& nq) {
    row0 = b;
    nq = 1;
    if (a.cu_q) {
        row0 = min(max(a.cu_q[b], 0), a.rows);
        nq = min(max(a.cu_q[b + 1] - row0, 0), min(a.max_q, a.rows - row0));
    }
}

__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Operand register i of a code word: the bf16 pair 16 + c (the nibble goes to bits 3..6 of each
// half, where a bf16 in [16, 32) holds its whole part).
__device__ __forceinline__ uint32_t unpack(uint32_t w, int i) {
    return ((i == 0 ? w << 3 : w >> (4 * i - 3)) & 0x00780078u) | 0x41804180u;
}
// The same, less 24: c - 8, exact.
__device__ __forceinline__ uint32_t unpack8(uint32_t w, int i) {
    const uint32_t u = unpack(w, i);
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), __floats2bfloat162_rn(24.f, 24.f));
    return *reinterpret_cast<const uint32_t*>(&d);
}

__device__ __forceinline__ uint32_t pack(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo_of(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi_of(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }

template <int HD>
constexpr int stages() { return HD == 64 ? 8 : 4; }
template <int HD>
constexpr int ring_bytes() { return WARPS * stages<HD>() * Kv4Tile<HD>::BYTES; }

template <int HD, int NT, bool DUP>
__global__ void __launch_bounds__(WARPS * 32) k_kv4_attn(const AttnArgs a) {
    using T = Kv4Tile<HD>;
    constexpr int NG = T::NG, NB = HD / 64, S = stages<HD>(), MT = HD / 16;
    constexpr int UT = DUP ? 4 : 8 * NT;
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ uint64_t bars[WARPS][S];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % a.nsplit, u0 = blockIdx.x / a.nsplit * UT;
    const int h = blockIdx.y, b = blockIdx.z;

    int row0, nq;
    rows_of(a, b, row0, nq);
    const int units = nq * a.group;
    if (u0 >= units) return;
    const int len = min(max(a.kv_lens[b], 0), a.width << a.page_shift);
    const int ulast = min(u0 + UT, units) - 1;
    const int first = len - nq + u0 / a.group, last = len - nq + ulast / a.group;   // their positions
    auto low = [&](int pos) { return a.window > 0 ? max(0, pos - a.window + 1) : 0; };
    const int kmin = low(first), kmax = last + 1;   // keys that some unit sees: [kmin, kmax)
    const int tile0 = kmin / KV4_TILE, ntiles = kmax > 0 ? (kmax + KV4_TILE - 1) / KV4_TILE : 0;
    const int t_begin = tile0 + split * a.split_tiles;
    const int t_end = split == a.nsplit - 1 ? ntiles : min(ntiles, t_begin + a.split_tiles);
    const int mine = t_end > t_begin + warp ? (t_end - t_begin - warp + WARPS - 1) / WARPS : 0;

    if (lane == 0) {
        for (int i = 0; i < S; ++i) mbar_init(&bars[warp][i], 1);
        fence_mbar_init();
    }
    __syncwarp();

    // page of the warp's i-th tile: lane i % 32 holds it for the current 32
    int page_of = -1;
    auto fetch_pages = [&](int i0) {
        const int i = i0 + lane;
        page_of = -1;
        if (i < mine) {
            const int tl = t_begin + warp + i * WARPS;
            page_of = a.table[(int64_t)b * a.width + (tl >> (a.page_shift - 4))];
            if (page_of < 0 || page_of >= a.num_pages) page_of = -1;
        }
    };
    unsigned char* ring = sm + warp * S * T::BYTES;
    auto issue = [&](int i, int page) {   // lane 0; a tile of no page completes its phase at once
        uint64_t* bar = &bars[warp][i % S];
        if (page < 0) {
            mbar_arrive(bar);
            return;
        }
        const int tl = t_begin + warp + i * WARPS;
        const uint8_t* src = a.pages + ((int64_t)page * a.hkv + h) * a.page_bytes +
                             (int64_t)(tl & ((1 << (a.page_shift - 4)) - 1)) * T::BYTES;
        mbar_arrive_expect_tx(bar, T::BYTES);
        tma_load_1d(ring + (i % S) * T::BYTES, src, T::BYTES, bar);
    };
    fetch_pages(0);
    int next_pages = page_of;   // of the 32 tiles that hold the next one to issue
    for (int i = 0; i < min(S, mine); ++i) {
        const int p = __shfl_sync(0xffffffffu, page_of, i);
        if (lane == 0) issue(i, p);
    }

    // queries: B operand of step j (dims 16 j ..): unit n = lane / 4, dims 2t, 2t + 1 and 8 further
    uint32_t qf[NT][2 * MT];
    float nsum[NT][NG][2];   // -16 sum of q over the group, for the thread's two columns
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int u = u0 + (DUP ? (r & 3) : nt * 8 + r);
        const bool ok = u < units;
        const int j = ok ? u / a.group : 0, g = ok ? u - j * a.group : 0;
        const __nv_bfloat16* src = a.q + (row0 + j) * a.q_row + (h * a.group + g) * a.q_head;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) qf[nt][i] = ok ? *reinterpret_cast<const uint32_t*>(src + 8 * i + 2 * t) : 0u;
#pragma unroll
        for (int g4 = 0; g4 < NG; ++g4) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) s += lo_of(qf[nt][4 * g4 + i]) + hi_of(qf[nt][4 * g4 + i]);
            s += __shfl_xor_sync(0xffffffffu, s, 1);
            s += __shfl_xor_sync(0xffffffffu, s, 2);
            nsum[nt][g4][0] = -16.f * __shfl_sync(0xffffffffu, s, 8 * t);
            nsum[nt][g4][1] = -16.f * __shfl_sync(0xffffffffu, s, 8 * t + 4);
        }
    }
    int hi[NT][2], lo[NT][2];   // keys that the thread's columns see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int u = min(u0 + (DUP ? ((2 * t + c) & 3) : nt * 8 + 2 * t + c), units - 1);
            const int pos = len - nq + u / a.group;
            hi[nt][c] = pos + 1;
            lo[nt][c] = low(pos);
        }
    const int all_lo = low(last), all_hi = first + 1;   // keys in [all_lo, all_hi) are seen by every unit

    float o[MT][NT][4], zacc[NT][NG][2], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < MT; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) zacc[nt][g][0] = zacc[nt][g][1] = 0.f;
        m[nt][0] = m[nt][1] = NEG;
        l[nt][0] = l[nt][1] = 0.f;
    }
    int failed = -1;   // the tile whose copy did not land within the bound

    for (int i = 0; i < mine; ++i) {
        const int st = i % S;
        if (i > 0 && (i & 31) == 0) page_of = next_pages;
        const int page = __shfl_sync(0xffffffffu, page_of, i & 31);
        if (!mbar_wait(&bars[warp][st], (i / S) & 1)) {
            failed = i;
            break;
        }
        const unsigned char* tp = ring + st * T::BYTES;
        uint4 kc[NB], vc[NB];
        uint32_t kp[2][NG], vp[2][NG];
#pragma unroll
        for (int x = 0; x < NB; ++x) {
            kc[x] = *reinterpret_cast<const uint4*>(tp + x * T::BLK + lane * 16);
            vc[x] = *reinterpret_cast<const uint4*>(tp + T::V + x * T::BLK + lane * 16);
        }
#pragma unroll
        for (int x = 0; x < 2 * NG; x += 4) {
            *reinterpret_cast<uint4*>(&kp[0][0] + x) = *reinterpret_cast<const uint4*>(tp + T::KP + r * 8 * NG + x * 4);
            *reinterpret_cast<uint4*>(&vp[0][0] + x) = *reinterpret_cast<const uint4*>(tp + T::VP + r * 8 * NG + x * 4);
        }
        __syncwarp();   // every lane has read the stage
        const int nx = i + S;
        if (nx < mine) {
            if ((nx & 31) == 0) {
                const int keep = page_of;
                fetch_pages(nx);
                next_pages = page_of;
                page_of = keep;
            }
            const int p = __shfl_sync(0xffffffffu, (nx >> 5) == (i >> 5) ? page_of : next_pages, nx & 31);
            if (lane == 0) issue(nx, p);
        }
        if (page < 0) continue;

        // scores
        const int k0 = (t_begin + warp + i * WARPS) * KV4_TILE;
        float sc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const uint32_t wr = g & 1 ? kc[g >> 1].y : kc[g >> 1].x, w8 = g & 1 ? kc[g >> 1].w : kc[g >> 1].z;
            uint32_t af[2][4];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                af[x][0] = unpack(wr, 2 * x);
                af[x][1] = unpack(w8, 2 * x);
                af[x][2] = unpack(wr, 2 * x + 1);
                af[x][3] = unpack(w8, 2 * x + 1);
            }
            const float s0 = lo_of(kp[0][g]), z0 = hi_of(kp[0][g]) * -0.0625f;
            const float s8 = lo_of(kp[1][g]), z8 = hi_of(kp[1][g]) * -0.0625f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float n0 = nsum[nt][g][0], n1 = nsum[nt][g][1];
                float acc[4] = {n0, n1, n0, n1};
                mma16816(acc, af[0][0], af[0][1], af[0][2], af[0][3], qf[nt][4 * g], qf[nt][4 * g + 1]);
                mma16816(acc, af[1][0], af[1][1], af[1][2], af[1][3], qf[nt][4 * g + 2], qf[nt][4 * g + 3]);
                sc[nt][0] = fmaf(s0, acc[0], fmaf(z0, n0, sc[nt][0]));
                sc[nt][1] = fmaf(s0, acc[1], fmaf(z0, n1, sc[nt][1]));
                sc[nt][2] = fmaf(s8, acc[2], fmaf(z8, n0, sc[nt][2]));
                sc[nt][3] = fmaf(s8, acc[3], fmaf(z8, n1, sc[nt][3]));
            }
        }
        const bool edge = k0 < all_lo || k0 + KV4_TILE > all_hi;
        const int ka = k0 + r, kb = ka + 8;
        bool up = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = e & 1, k = e < 2 ? ka : kb;
                sc[nt][e] *= a.scale_log2;
                if (edge && (k < lo[nt][c] || k >= hi[nt][c])) sc[nt][e] = -INFINITY;
                up |= sc[nt][e] > m[nt][c] + LAZY;
            }
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float x = fmaxf(sc[nt][c], sc[nt][c + 2]);
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    x = fmaxf(x, m[nt][c]);
                    const float f = ex2(m[nt][c] - x);
                    m[nt][c] = x;
                    l[nt][c] *= f;
#pragma unroll
                    for (int g = 0; g < NG; ++g) zacc[nt][g][c] *= f;
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        o[x][nt][c] *= f;
                        o[x][nt][c + 2] *= f;
                    }
                }
        }
        bool see[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = e & 1, k = e < 2 ? ka : kb;
                see[nt][e] = !edge || (k >= lo[nt][c] && k < hi[nt][c]);
                sc[nt][e] = ex2(sc[nt][e] - m[nt][c]);
                l[nt][c] += sc[nt][e];
            }
        // values
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const float s0 = lo_of(vp[0][g]), s8 = lo_of(vp[1][g]);
            const float z0 = fmaf(8.f, s0, hi_of(vp[0][g])), z8 = fmaf(8.f, s8, hi_of(vp[1][g]));
            const uint32_t w0 = g & 1 ? vc[g >> 1].z : vc[g >> 1].x, w1 = g & 1 ? vc[g >> 1].w : vc[g >> 1].y;
            uint32_t af[2][4];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                af[x][0] = unpack8(w0, 2 * x);
                af[x][1] = unpack8(w0, 2 * x + 1);
                af[x][2] = unpack8(w1, 2 * x);
                af[x][3] = unpack8(w1, 2 * x + 1);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float w[4], z[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = see[nt][e] ? sc[nt][e] * (e < 2 ? s0 : s8) : 0.f;
                    z[e] = see[nt][e] ? sc[nt][e] * (e < 2 ? z0 : z8) : 0.f;
                }
                zacc[nt][g][0] += z[0] + z[2];
                zacc[nt][g][1] += z[1] + z[3];
                uint32_t pa = pack(w[0], w[1]), pb = pack(w[2], w[3]);
                const uint32_t la = pack(w[0] - lo_of(pa), w[1] - hi_of(pa)), lb = pack(w[2] - lo_of(pb), w[3] - hi_of(pb));
                if (DUP) {
                    const uint32_t b0 = movmatrix(t < 2 ? pa : la), b1 = movmatrix(t < 2 ? pb : lb);
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        mma16816(o[2 * g + x][nt], af[x][0], af[x][1], af[x][2], af[x][3], b0, b1);
                } else {
                    const uint32_t b0 = movmatrix(pa), b1 = movmatrix(pb), c0 = movmatrix(la), c1 = movmatrix(lb);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        mma16816(o[2 * g + x][nt], af[x][0], af[x][1], af[x][2], af[x][3], b0, b1);
                        mma16816(o[2 * g + x][nt], af[x][0], af[x][1], af[x][2], af[x][3], c0, c1);
                    }
                }
            }
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
                wo[u * (HD + 2) + HD] = m[nt][c];
                wo[u * (HD + 2) + HD + 1] = s;
            }
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                float z = zacc[nt][g][c];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) z += __shfl_xor_sync(0xffffffffu, z, x);
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = o[2 * g + x][nt][c + 2 * e];
                        if (DUP) v += __shfl_xor_sync(0xffffffffu, v, 2);
                        if (!DUP || t < 2) wo[u * (HD + 2) + 32 * g + 16 * x + 8 * e + r] = v + z;
                    }
            }
        }
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(sm);
    for (int i = tid; i < (ulast - u0 + 1) * HD; i += WARPS * 32) {
        const int u = i / HD, d = i % HD;
        float mm = NEG, ll = 0.f, oo = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, all[(w * UT + u) * (HD + 2) + HD]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float* p = all + (w * UT + u) * (HD + 2);
            const float f = ex2(p[HD] - mm);
            ll = fmaf(f, p[HD + 1], ll);
            oo = fmaf(f, p[d], oo);
        }
        const int j = (u0 + u) / a.group, g = (u0 + u) - j * a.group;
        const int64_t at = (int64_t)(row0 + j) * a.hq + h * a.group + g;
        if (a.nsplit == 1) {
            a.out[at * HD + d] = __float2bfloat16(ll == 0.f ? 0.f : oo / ll);
        } else {
            a.part_o[(at * a.nsplit + split) * HD + d] = oo;
            if (d == 0) {
                a.part_ml[(at * a.nsplit + split) * 2] = mm;
                a.part_ml[(at * a.nsplit + split) * 2 + 1] = ll;
            }
        }
    }
}

// out of one (sequence row, head) from its splits' partials, in split order: a block of HD threads.
template <int HD>
__global__ void __launch_bounds__(HD) k_kv4_merge(const AttnArgs a) {
    const int j = blockIdx.x / a.hq, b = blockIdx.y;
    int row0, nq;
    rows_of(a, b, row0, nq);
    if (j >= nq) return;
    const int64_t at = (int64_t)(row0 + j) * a.hq + blockIdx.x % a.hq;
    const float* ml = a.part_ml + at * a.nsplit * 2;
    float mm = NEG;
    for (int s = 0; s < a.nsplit; ++s) mm = fmaxf(mm, ml[2 * s]);
    float ll = 0.f, oo = 0.f;
    for (int s = 0; s < a.nsplit; ++s) {
        const float f = ex2(ml[2 * s] - mm);
        ll = fmaf(f, ml[2 * s + 1], ll);
        oo = fmaf(f, a.part_o[(at * a.nsplit + s) * HD + threadIdx.x], oo);
    }
    a.out[at * HD + threadIdx.x] = __float2bfloat16(ll == 0.f ? 0.f : oo / ll);
}

struct Plan {
    int nt, dup, utiles, nsplit, split_tiles;
};

// How a call is cut. Units: the fewest columns that hold max_q rows of a group (four: both halves
// of the weights in one operand), at most 32 (heads of 128: 16, for the registers). Splits: until
// about four CTAs an SM are there, of at least 16 tiles (four a warp) each.
Plan make_plan(int64_t B, int64_t Hkv, int64_t group, int64_t head_dim, int64_t max_q, int64_t max_kv,
               int64_t window) {
    Plan p{};
    const int64_t units = max_q * group, cap = head_dim == 64 ? 4 : 2;
    p.dup = units <= 4;
    p.nt = (int)(units > 8 * cap ? cap : (units + 7) / 8);
    const int64_t ut = p.dup ? 4 : 8 * p.nt;
    p.utiles = (int)((units + ut - 1) / ut);
    int64_t span = max_kv;
    if (window > 0) {
        const int64_t rows = (ut + group - 1) / group + 1;   // rows that a unit tile can touch
        const int64_t w = window + (rows < max_q ? rows : max_q) + KV4_TILE;
        if (w < span) span = w;
    }
    const int64_t tiles = (span + KV4_TILE - 1) / KV4_TILE;
    const int64_t ctas = B * Hkv * p.utiles;
    int64_t ns = (148 * 4 + ctas - 1) / ctas;
    if (ns > tiles / 16) ns = tiles / 16;
    if (ns > 64) ns = 64;
    if (ns < 1) ns = 1;
    p.split_tiles = (int)((tiles + ns - 1) / ns);
    if (p.split_tiles < 1) p.split_tiles = 1;
    p.nsplit = (int)((tiles + p.split_tiles - 1) / p.split_tiles);
    if (p.nsplit < 1) p.nsplit = 1;
    return p;
}

template <int HD, int NT, bool DUP>
int launch(const AttnArgs& a, const Plan& p, int64_t B, cudaStream_t st) {
    constexpr int merge = WARPS * (DUP ? 4 : 8 * NT) * (HD + 2) * 4;
    constexpr int bytes = ring_bytes<HD>() > merge ? ring_bytes<HD>() : merge;
    PULSAR_TRY(ensure_smem_attr((const void*)k_kv4_attn<HD, NT, DUP>, bytes, "k_kv4_attn shared memory"));
    const dim3 grid((unsigned)(p.utiles * p.nsplit), (unsigned)a.hkv, (unsigned)B);
    k_kv4_attn<HD, NT, DUP><<<grid, WARPS * 32, bytes, st>>>(a);
    PULSAR_LAUNCH_CHECK("k_kv4_attn");
    return PULSAR_OK;
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
    *bytes = p.nsplit > 1 ? N * Hq * p.nsplit * (head_dim + 2) * 4 : 0;
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
    PULSAR_CHECK_ARG(cu_q || (N == B && max_q == 1), "kv4_attention: without cu_q every sequence has one row");
    if (N == 0 || B == 0) return PULSAR_OK;
    PULSAR_CHECK_ARG(q && pages && kv_lens && out && (block_table || width == 0), "kv4_attention: null pointer");
    PULSAR_CHECK_ARG((reinterpret_cast<uintptr_t>(q) & 3) == 0 && q_row_stride % 2 == 0 && q_head_stride % 2 == 0,
                     "kv4_attention: q must be 4-byte aligned with even strides");
    PULSAR_CHECK_ARG((reinterpret_cast<uintptr_t>(pages) & 15) == 0, "kv4_attention: pages must be 16-byte aligned");
    const Plan p = make_plan(B, Hkv, Hq / Hkv, head_dim, max_q, max_kv, window);
    const int64_t need = p.nsplit > 1 ? N * Hq * p.nsplit * (head_dim + 2) * 4 : 0;
    PULSAR_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
                     "kv4_attention: workspace of %lld bytes needed, got %lld", (long long)need,
                     (long long)workspace_bytes);
    float* ws = (float*)workspace;
    AttnArgs a{(const __nv_bfloat16*)q, (const uint8_t*)pages, block_table, kv_lens, cu_q, (__nv_bfloat16*)out, ws,
               p.nsplit > 1 ? ws + N * Hq * p.nsplit * head_dim : nullptr, q_row_stride, q_head_stride,
               page_size / KV4_TILE * 20 * head_dim, (int)N, (int)Hq, (int)Hkv, (int)(Hq / Hkv), (int)num_pages,
               (int)width, __builtin_ctzll((unsigned long long)page_size), (int)max_q, (int)window, p.nsplit,
               p.split_tiles, scale * 1.4426950408889634f};
    cudaStream_t st = (cudaStream_t)stream;
    int rc;
    if (head_dim == 64)
        rc = p.dup ? launch<64, 1, true>(a, p, B, st) : p.nt == 1 ? launch<64, 1, false>(a, p, B, st)
           : p.nt == 2 ? launch<64, 2, false>(a, p, B, st) : p.nt == 3 ? launch<64, 3, false>(a, p, B, st)
           : launch<64, 4, false>(a, p, B, st);
    else
        rc = p.dup ? launch<128, 1, true>(a, p, B, st) : p.nt == 1 ? launch<128, 1, false>(a, p, B, st)
           : launch<128, 2, false>(a, p, B, st);
    PULSAR_TRY(rc);
    if (p.nsplit > 1) {
        const dim3 grid((unsigned)(max_q * Hq), (unsigned)B);
        if (head_dim == 64)
            k_kv4_merge<64><<<grid, 64, 0, st>>>(a);
        else
            k_kv4_merge<128><<<grid, 128, 0, st>>>(a);
        PULSAR_LAUNCH_CHECK("k_kv4_merge");
    }
    return PULSAR_OK;
}
