// What the kernels of pulsar_op_kv4_attention share: the call's arguments, the rows of a sequence and
// how partial results are handed to the merge.
#pragma once

#include <cuda_bf16.h>
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
    int rows, hq, hkv, group, num_pages, width, page_shift, max_q, window, nsplit, split_len;
    float scale_log2;
};

// The rows of sequence b, held inside q whatever cu_q says.
__device__ __forceinline__ void kv4_rows(const Kv4AttnArgs& a, int b, int& row0, int& nq) {
    row0 = b;
    nq = 1;
    if (a.cu_q) {
        row0 = min(max(a.cu_q[b], 0), a.rows);
        nq = min(max(a.cu_q[b + 1] - row0, 0), min(a.max_q, a.rows - row0));
    }
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

// Many query rows (kv4_prefill.cu): units = query rows x heads of a group.
constexpr int kv4_pf_units(int head_dim) { return head_dim == 64 ? 512 : 256; }   // units of a CTA
constexpr int KV4_PF_STEP = 128;   // keys of a step
int kv4_prefill_launch(const Kv4AttnArgs& a, int head_dim, int64_t sequences, int utiles, cudaStream_t stream);

}  // namespace pulsar
