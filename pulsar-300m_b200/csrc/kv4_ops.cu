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
    int64_t n, num_slots, page_bytes;
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

// Codes, s and z of the group of 32 dims whose 8-dim quarter this lane holds (x: its values).
// Returns the lane's 8 codes, nibble j = dim j.
__device__ __forceinline__ uint32_t quantise(const float* x, uint32_t& param) {
    float mn = x[0], mx = x[0];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        mn = fminf(mn, x[j]);
        mx = fmaxf(mx, x[j]);
        bad |= !(fabsf(x[j]) < INFINITY);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, o) != 0;
    }
    const __nv_bfloat16 zb = __float2bfloat16(mn);
    const float z = __bfloat162float(zb);
    __nv_bfloat16 sb = __float2bfloat16(__fdiv_rn(__fsub_rn(mx, z), 15.f));
    float s = __bfloat162float(sb);
    bad |= !(fabsf(z) < INFINITY) || !(s < INFINITY);
    if (bad) {   // the whole group reads back as NaN
        param = 0x7fff7fffu;
        return 0u;
    }
    if (!(s >= 1.17549435e-38f)) {   // a constant group (or a span below the normal range)
        param = (uint32_t)__bfloat16_as_ushort(zb) << 16;
        return 0u;
    }
    param = (uint32_t)__bfloat16_as_ushort(zb) << 16 | __bfloat16_as_ushort(sb);
    uint32_t p = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float c = rintf(__fdiv_rn(__fsub_rn(x[j], z), s));
        p |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * j);
    }
    return p;
}

// Transpose among the quad of lanes that holds a group: lane j = 2 b + n comes with the codes of
// dims 16 b + 8 n + x (nibble x) and leaves with the word of x = 2j, 2j + 1: half e = x % 2, byte
// b of the half, nibble n of the byte.
__device__ __forceinline__ uint32_t quad_word(uint32_t p, int lane) {
    uint32_t w = 0;
    const int j = lane & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // byte j of the codes of lane (b, n) = (i / 2, i % 2)
        const uint32_t o = __shfl_sync(0xffffffffu, p, (lane & ~3) | i) >> (8 * j);
        w |= (o & 0xfu) << (8 * (i >> 1) + 4 * (i & 1)) | ((o >> 4) & 0xfu) << (16 + 8 * (i >> 1) + 4 * (i & 1));
    }
    return w;
}

// D / 8 lanes a head vector, 8 dims a lane.
template <int HD>
__global__ void __launch_bounds__(256) k_kv4_append(const AppendArgs a) {
    using T = Kv4Tile<HD>;
    constexpr int L = HD / 8;
    const int heads = a.hq + 2 * a.hkv;
    const int lane = threadIdx.x & 31, l = lane % L;
    const int64_t total = a.n * heads;
    const int64_t stride = (int64_t)gridDim.x * (blockDim.x / L);
    const int64_t v0 = ((int64_t)blockIdx.x * blockDim.x + (threadIdx.x & ~31)) / L;   // the warp's first vector
    for (int64_t vb = v0; vb < total; vb += stride) {
        const int64_t vi = vb + lane / L;
        const bool live = vi < total;
        const int64_t tok = live ? vi / heads : 0;
        const int h = live ? (int)(vi - tok * heads) : 0;
        const bool is_q = h < a.hq, is_k = !is_q && h < a.hq + a.hkv;
        const int hh = is_q ? h : is_k ? h - a.hq : h - a.hq - a.hkv;
        const __nv_bfloat16* src = is_q ? a.q + tok * a.qs + hh * a.qh
                                 : is_k ? a.k + tok * a.ks + hh * a.kh : a.v + tok * a.vs + hh * a.vh;
        float x[8];
        bf16x8_to_f32(__ldg(reinterpret_cast<const uint4*>(src) + l), x);
        const int pos = a.pos ? a.pos[tok] : 0;
        const bool pos_ok = !a.pos || (pos >= 0 && pos < a.max_pos);
        if (a.qw || a.kw) {   // (uniform: every lane takes part in the shuffles)
            const float* w = is_q ? a.qw : is_k ? a.kw : nullptr;
            float t[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) t[j] = __fmul_rn(x[j], x[j]);
            float ss = __fadd_rn(__fadd_rn(__fadd_rn(t[0], t[1]), __fadd_rn(t[2], t[3])),
                                 __fadd_rn(__fadd_rn(t[4], t[5]), __fadd_rn(t[6], t[7])));
            ss = lanes_sum<L>(ss);
            if (w) {
                const float inv = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.f / HD), a.eps)));
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(w[hh * HD + 8 * l + j], __fmul_rn(x[j], inv));
            }
        }
        __syncwarp();
        if (a.rot > 0) {
            const int half = a.rot >> 1;
            const float *cs = a.cs + (int64_t)(pos_ok ? pos : 0) * half, *sn = a.sn + (int64_t)(pos_ok ? pos : 0) * half;
            const bool turn = (is_q || is_k) && 8 * l < a.rot;
            if (a.interleaved) {
                if (turn) {
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        if (8 * l + j < a.rot) {
                            const float c = cs[4 * l + j / 2], s = sn[4 * l + j / 2];
                            const float u = x[j], v = x[j + 1];
                            x[j] = __fsub_rn(__fmul_rn(u, c), __fmul_rn(v, s));
                            x[j + 1] = __fadd_rn(__fmul_rn(v, c), __fmul_rn(u, s));
                        }
                    }
                }
            } else {   // rot % 16 == 0: the partner's dims are the same 8 of another lane
                const int hl = half >> 3;
                const bool first = l < hl;
                const int from = (lane - l) + (turn ? (first ? l + hl : l - hl) : l);
                float o[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) o[j] = __shfl_sync(0xffffffffu, x[j], from);
                if (turn) {
                    const int b = 8 * (first ? l : l - hl);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float c = cs[b + j], s = sn[b + j];
                        x[j] = first ? __fsub_rn(__fmul_rn(x[j], c), __fmul_rn(o[j], s))
                                     : __fadd_rn(__fmul_rn(x[j], c), __fmul_rn(o[j], s));
                    }
                }
            }
        }
        __syncwarp();
        uint32_t param;
        const uint32_t codes = quantise(x, param);
        const uint32_t word = quad_word(codes, lane);
        if (!live) continue;
        if (is_q) {
            if (a.gain) {
                const float g = pos_ok ? a.gain[pos] : 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = __fmul_rn(x[j], g);
            }
            if (!pos_ok) {
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = 0.f;
            }
            reinterpret_cast<uint4*>(a.qo + (tok * a.hq + hh) * HD)[l] = f32_to_bf16x8(x);
            continue;
        }
        const int64_t slot = a.slots[tok];
        if (slot < 0 || slot >= a.num_slots || !pos_ok) continue;
        const int64_t page = slot >> a.page_shift;
        const int off = (int)(slot & ((1 << a.page_shift) - 1));
        uint8_t* tile = a.pages + (page * a.hkv + hh) * a.page_bytes + (int64_t)(off >> 4) * T::BYTES;
        const int t = off & 15, r = t & 7, hf = t >> 3, g = l >> 2, j = l & 3;
        if (is_k) {
            *reinterpret_cast<uint32_t*>(tile + (g >> 1) * T::BLK + (4 * r + j) * 16 + hf * 8 + (g & 1) * 4) = word;
        } else {
            uint8_t* p = tile + T::V + (g >> 1) * T::BLK + (8 * j + (r >> 1)) * 16 + (g & 1) * 8 + hf * 4 + (r & 1) * 2;
            *reinterpret_cast<uint16_t*>(p) = (uint16_t)word;
            *reinterpret_cast<uint16_t*>(p + 64) = (uint16_t)(word >> 16);
        }
        if (j == 0)
            *reinterpret_cast<uint32_t*>(tile + (is_k ? T::KP : T::VP) + ((2 * r + hf) * T::NG + g) * 4) = param;
    }
}

// The inverse of quantise and quad_word: bf16(s c + z) of the positions asked for.
template <int HD>
__global__ void __launch_bounds__(256) k_kv4_read(const uint8_t* __restrict__ pages, const int64_t* __restrict__ slots,
                                                  int64_t n, int hkv, int page_shift, int64_t page_bytes,
                                                  int64_t num_slots, __nv_bfloat16* __restrict__ ko,
                                                  __nv_bfloat16* __restrict__ vo) {
    using T = Kv4Tile<HD>;
    constexpr int L = HD / 8;
    const int lane = threadIdx.x & 31, l = lane % L, g = l >> 2, j = l & 3;
    const int64_t total = n * 2 * hkv;
    const int64_t stride = (int64_t)gridDim.x * (blockDim.x / L);
    const int64_t v0 = ((int64_t)blockIdx.x * blockDim.x + (threadIdx.x & ~31)) / L;
    for (int64_t vb = v0; vb < total; vb += stride) {
        const int64_t vi = vb + lane / L;
        const bool live = vi < total;
        const int64_t tok = live ? vi / (2 * hkv) : 0;
        const int h = live ? (int)(vi - tok * 2 * hkv) : 0;
        const bool is_k = h < hkv;
        const int hh = is_k ? h : h - hkv;
        const int64_t slot = slots[tok];
        const bool ok = slot >= 0 && slot < num_slots;
        const int64_t page = ok ? slot >> page_shift : 0;
        const int off = ok ? (int)(slot & ((1 << page_shift) - 1)) : 0;
        const uint8_t* tile = pages + (page * hkv + hh) * page_bytes + (int64_t)(off >> 4) * T::BYTES;
        const int t = off & 15, r = t & 7, hf = t >> 3;
        uint32_t word = 0, par = 0;
        if (ok) {
            if (is_k) {
                word = *reinterpret_cast<const uint32_t*>(tile + (g >> 1) * T::BLK + (4 * r + j) * 16 + hf * 8 +
                                                          (g & 1) * 4);
            } else {
                const uint8_t* p = tile + T::V + (g >> 1) * T::BLK + (8 * j + (r >> 1)) * 16 + (g & 1) * 8 + hf * 4 +
                                   (r & 1) * 2;
                word = *reinterpret_cast<const uint16_t*>(p) |
                       (uint32_t)*reinterpret_cast<const uint16_t*>(p + 64) << 16;
            }
            par = *reinterpret_cast<const uint32_t*>(tile + (is_k ? T::KP : T::VP) + ((2 * r + hf) * T::NG + g) * 4);
        }
        const float s = __uint_as_float(par << 16), z = __uint_as_float(par & 0xffff0000u);
        float x[8];
        const int b = j >> 1, nb = j & 1;   // this lane's dims are 32 g + 16 b + 8 nb + x
#pragma unroll
        for (int i = 0; i < 4; ++i) {       // dims x = 2i, 2i + 1: word of quad lane i
            const uint32_t o = __shfl_sync(0xffffffffu, word, (lane & ~3) | i) >> (8 * b + 4 * nb);
            x[2 * i] = __fadd_rn(__fmul_rn((float)(o & 15u), s), z);
            x[2 * i + 1] = __fadd_rn(__fmul_rn((float)((o >> 16) & 15u), s), z);
        }
        if (live)
            reinterpret_cast<uint4*>((is_k ? ko : vo) + (tok * hkv + hh) * HD)[l] = f32_to_bf16x8(x);
    }
}

// Blocks of 256 threads for `vectors` head vectors of L lanes: at most eight resident blocks per
// SM's worth, the rest by the grid-stride loop.
int blocks_for(int64_t vectors, int lanes) {
    const int64_t g = (vectors * lanes + 255) / 256;
    return (int)(g < 148 * 8 ? g : 148 * 8);
}

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
    PULSAR_CHECK_ARG(N >= 0 && Hq >= 0 && Hq <= 65536, "kv4_append: invalid shape");
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
    for (const void* p : {q, k, v, (const void*)q_out})
        PULSAR_CHECK_ARG((reinterpret_cast<uintptr_t>(p) & 15) == 0, "kv4_append: q, k, v must be 16-byte aligned");
    AppendArgs a{(const __nv_bfloat16*)q, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, strides[0], strides[2],
                 strides[4], strides[1], strides[3], strides[5], q_norm, k_norm, cos, sin, q_gain, slots,
                 (rot > 0 || q_gain) ? positions : nullptr, (uint8_t*)pages, (__nv_bfloat16*)q_out, N,
                 num_pages * page_size, pb, (int)Hq, (int)Hkv, shift, (int)rot, (int)max_pos, interleaved, eps};
    const int grid = blocks_for(N * (Hq + 2 * Hkv), (int)head_dim / 8);
    if (head_dim == 64)
        k_kv4_append<64><<<grid, 256, 0, (cudaStream_t)stream>>>(a);
    else
        k_kv4_append<128><<<grid, 256, 0, (cudaStream_t)stream>>>(a);
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
    const int grid = blocks_for(N * 2 * Hkv, (int)head_dim / 8);
    if (head_dim == 64)
        k_kv4_read<64><<<grid, 256, 0, (cudaStream_t)stream>>>((const uint8_t*)pages, slots, N, (int)Hkv, shift, pb,
                                                               num_pages * page_size, (__nv_bfloat16*)k_out,
                                                               (__nv_bfloat16*)v_out);
    else
        k_kv4_read<128><<<grid, 256, 0, (cudaStream_t)stream>>>((const uint8_t*)pages, slots, N, (int)Hkv, shift, pb,
                                                                num_pages * page_size, (__nv_bfloat16*)k_out,
                                                                (__nv_bfloat16*)v_out);
    PULSAR_LAUNCH_CHECK("k_kv4_read");
    return PULSAR_OK;
}
