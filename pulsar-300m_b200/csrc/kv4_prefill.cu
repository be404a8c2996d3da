// Attention of many query rows over the paged 4-bit KV cache (layout: kv4.cuh), the tensor-core
// half of pulsar_op_kv4_attention: prompts and chunks of prompts.
//
// CTA: 512 units (query rows x heads of one kv head's group; heads of 128: 256) of a sequence as
// tiles of 128, one TMEM lane a unit, over a range of its keys in chunks of 64, two to a step:
//   unpack    a warp takes tiles of 16 tokens through a ring of its own (1-D bulk copies, page ids
//             prefetched) to K^ [64 keys][HD] and V^T^ [HD][64 keys] in fp16, K-major SWIZZLE_128B:
//             the cache keeps codes so that a word's halves are neighbours in the operand's rows
//   S = Q K^  tcgen05.mma kind::f16, M 128, N 64, fp32 in TMEM (a warp for each tile of units)
//   softmax   a thread per unit (four warps a tile): weights in fp16 back to TMEM, over the scores
//   O += P V^ with P read from TMEM as the A operand, O in TMEM
// The exponentials (16 a clock and SM) take half of the time; what bounds the kernel is a tile's chain of MMA,
// scores, weights and MMA, which is longer, so four tiles are in flight at different places of it, each with a
// softmax warp on every scheduler (heads of 128: the two that TMEM holds; 2048 rows on 8192 keys 217 us).
// 2048 rows of 16 heads of 64 on 16384 keys (4 kv heads) take 239 us: 0.54 PFLOP/s of products, and
// 5 10^8 exponentials, which take 128 SMs (64 unit tiles x 2 splits) 130 us. Measured instead: three
// tiles with weights beside the scores 277, two threads a unit 322, chunks of 32 keys 300, a quarter
// of the exponentials as cubic polynomials 281.
//
// Exactness. fp16 has the significand for it (values s c + z of 8-bit s, z and 4-bit c are rounded
// at 2^-12, weights too) but not the range, so powers of two move out: queries by their row, keys and
// values by their step of 128 (2^eK, 2^eV from the largest |value| that s and z allow, over the keys that
// some unit sees). Score and weight: x = 2^eK 2^eq scale log2(e) S, P = 2^(x + eV - er - m); P V^ = 2^(x - er - m) V
// and l = sum 2^(er - eV) P, with 2^er the unit of O (Kv4Unit). The reference m of a unit moves when a chunk's
// sum of weights passes 2^15 (then the row of O is rescaled and the chunk's weights taken again), so P stays
// inside fp16 and no maximum is looked for in other chunks.
//
// Keys that a unit does not see get weight 0 by selection. V^ is 0 for keys that no unit sees (pages
// past the end may hold anything) and for groups stored as NaN; which (key, group) those were goes to
// the softmax threads, whose units that see the key answer NaN in the group's dims.
//
// Every wait is bounded; one that runs out raises the CTA's abort flag, which ends the others; MMAs
// and copies in flight are waited for (bounded again) and the rows answer NaN.
#include <type_traits>

#include "capi_util.h"
#include "kv4_attn.cuh"
#include "mega_ptx.cuh"

using namespace pulsar;

namespace {

template <int HD>
struct Lay {
    static constexpr int NT = HD == 64 ? 4 : 2;                              // tiles of 128 units
    static constexpr int UNITS = 128 * NT;
    static constexpr int SOFT = 4 * NT, UNPACK = HD == 64 ? 4 : 8, MMA = SOFT + UNPACK;   // warps; MMA + t: tile t
    static constexpr int THREADS = (MMA + 4) * 32;
    static constexpr int CK = 64, SK = KV4_PF_STEP, NG = HD / 32, NB = HD / 64;
    static constexpr int YT = 8 / UNPACK;                                    // tiles of a step an unpacking warp takes
    static constexpr int PS = HD == 64 ? 3 : 2, KS = HD == 64 ? 4 : 3;       // stages: packed steps, unpacked chunks
    static constexpr uint32_t QB = 128 * HD * 2, KB = CK * HD * 2;           // bytes of a Q tile, of K^ or V^
    static constexpr uint32_t TB = Kv4Tile<HD>::BYTES, PB = PS * YT * TB;    // of a warp's packed ring
    static constexpr uint32_t Q = 0, K = NT * QB, V = K + KS * KB, P = V + KS * KB, MISC = P + UNPACK * PB;
    static constexpr uint32_t BYTES = MISC + 2048;
    static constexpr uint32_t S_COL = 0, O_COL = NT * CK;   // TMEM columns of the tiles' scores and of O
    static_assert(O_COL + NT * HD <= 512 && MISC % 1024 == 0 && BYTES + 1024 <= 227 * 1024, "fits");
};

struct Misc {   // in shared memory after the operands
    uint64_t packed[8][3], kv_full[4], kv_empty[4], s_full[4], p_full[4], pv_done[4], drain[4];
    uint32_t stop[2][8];     // per step parity and unpacking warp: a wait has run out
    uint32_t top[2][8][2];   // largest |K|, |V| as float bits
    float kscale[4], shift[4], factor[4];   // per unpacked stage: 2^eK, eV - er, what O is rescaled by
    int er[4];
    uint32_t mark[4];        // a byte for each tile of 16 tokens: GONE, BAD, MOVED
    uint8_t bad_groups[4][64];
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(Misc) <= 2048, "Misc fits its space");

// A tile's page is none of the cache's; some group of V is NaN; the step's values have moved the unit of O.
constexpr uint32_t GONE = 0x01010101u, BAD = 0x02020202u, MOVED = 0x04040404u;

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
    if (mbar_try(bar, parity)) return true;
    const unsigned long long t0 = globaltimer();
    while (!mbar_try(bar, parity)) {
        if (*abort) return false;
        if (globaltimer() - t0 > WAIT_NS) {
            *abort = 1;
            return false;
        }
    }
    return true;
}

// K-major SWIZZLE_128B operand (rows of 128 bytes, atoms of 8 rows): the descriptor's upper word is a
// constant, the lower one the address.
constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc(uint32_t addr) { return ((addr >> 4) & 0x3FFF) | (1u << 16); }
// kind::f16: fp32 accumulator, fp16 operands, both K-major, M = 128.
constexpr uint32_t idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | (8u << 24); }

// The whole warp comes here with the same operands, which then sit in uniform registers; the elected
// lane (one nonzero) issues. (An MMA issued inside a branch on the lane takes about 70 cycles.)
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %0, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 x, {%2, %6};\n\tmov.b64 y, {%3, %6};\n\t"
        "@p tcgen05.mma.cta_group::1.kind::f16 [%1], x, y, %4, q;\n\t}" ::"r"(one),
        "r"(d), "r"(a), "r"(b), "r"(id), "r"(acc), "n"(DESC_HI)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d, uint32_t a, uint32_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %0, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "mov.b64 y, {%3, %6};\n\t"
        "@p tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], y, %4, q;\n\t}" ::"r"(one),
        "r"(d), "r"(a), "r"(b), "r"(id), "r"(acc), "n"(DESC_HI)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t one, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %0, 0;\n\t"
        "@p tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(one),
        "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ uint32_t elect() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 columns of the thread's TMEM lane (no wait) and 16 back.
__device__ __forceinline__ void ld32(uint32_t at, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void st16(uint32_t at, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(at),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void ld16(uint32_t at, uint32_t* r) {   // (waits)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(at)
        : "memory");
}
// Waits for the loads; the registers pass through it, so that nothing reads them earlier.
__device__ __forceinline__ void ld_wait(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void sts(uint32_t at, uint32_t v) {
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

template <int HD>
__global__ void __launch_bounds__(Lay<HD>::THREADS, 1) k_kv4_prefill(const Kv4AttnArgs a) {
    using L = Lay<HD>;
    using T = Kv4Tile<HD>;
    constexpr int CK = L::CK, SK = L::SK, NG = L::NG, NB = L::NB, PS = L::PS, KS = L::KS;
    extern __shared__ unsigned char raw[];
    unsigned char* sm = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const uint32_t sb = smem_u32(sm);
    Misc& ms = *reinterpret_cast<Misc*>(sm + L::MISC);
    volatile int* abort = &ms.abort;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // the last units first, which see the most keys (8192 rows on 8192 keys: 352 -> 314 us)
    const int split = blockIdx.x % a.nsplit, u0 = (gridDim.x / a.nsplit - 1 - blockIdx.x / a.nsplit) * L::UNITS;
    const int h = blockIdx.y, b = blockIdx.z;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the merge may be set up meanwhile
    Kv4Range rg;
    if (!kv4_range(a, b, u0, L::UNITS, SK, rg) || split >= rg.used) return;
    const int row0 = rg.row0, nq = rg.nq, units = rg.units, len = rg.len, kmin = rg.kmin, kmax = rg.kmax;
    const int tiles = (rg.ulast - u0) / 128 + 1;
    auto low = [&](int pos) { return kv4_low(a, pos); };
    int s_begin, s_end;
    kv4_split(a, rg, split, s_begin, s_end);
    const int step0 = rg.step0 + s_begin, base = step0 * SK, kend = min(kmax, (rg.step0 + s_end) * SK);
    const int n = kend > base ? (kend - base + CK - 1) / CK : 0, steps = (n + 1) / 2;   // chunks, steps

    if (tid == 0) {
        for (int i = 0; i < KS; ++i) {
            mbar_init(&ms.kv_full[i], 4);
            mbar_init(&ms.kv_empty[i], tiles);
        }
        for (int i = 0; i < L::NT; ++i) {
            mbar_init(&ms.s_full[i], 1);
            mbar_init(&ms.p_full[i], 4);
            mbar_init(&ms.pv_done[i], 1);
            mbar_init(&ms.drain[i], 1);
        }
        ms.abort = 0;
        fence_mbar_init();
    }
    if (warp == L::MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ms.tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // unpacking: warp w of four takes tile w of each chunk; with eight, warp 4 y + w of chunk y of the steps.
    // With heads of 64 its first copies are on their way while the others set up (2048 rows on 2048 keys
    // 53.0 -> 51.8 us); heads of 128 lost by it (246 -> 256 us on 8192 keys)
    constexpr int YT = L::YT;
    const int uw = warp >= L::SOFT && warp < L::MMA ? warp - L::SOFT : 0, y0 = uw >> 2, w = uw & 3;
    unsigned char* ring = sm + L::P + uw * L::PB;
    uint64_t* packed = ms.packed[uw];
    // pages of the warp's tiles, those of 32 steps at a time (lane i: step i)
    auto pages_of = [&](int c0, int* pg) {
#pragma unroll
        for (int y = 0; y < YT; ++y) pg[y] = c0 + lane < steps ? kv4_page(a, b, (step0 + c0 + lane) * 8 + 4 * (y0 + y) + w) : -1;
    };
    auto issue = [&](int c, const int* page) {   // lane 0
        uint64_t* bar = &packed[c % PS];
        uint32_t bytes = 0;
#pragma unroll
        for (int y = 0; y < YT; ++y) bytes += page[y] >= 0 ? L::TB : 0;
        if (bytes == 0) {
            mbar_arrive(bar);
            return;
        }
        mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
        for (int y = 0; y < YT; ++y)
            if (page[y] >= 0)
                tma_load_1d(ring + ((c % PS) * YT + y) * L::TB,
                            a.pages + ((int64_t)page[y] * a.hkv + h) * a.page_bytes +
                                (int64_t)(((step0 + c) * 8 + 4 * (y0 + y) + w) & ((1 << (a.page_shift - 4)) - 1)) * L::TB,
                            L::TB, bar);
    };
    int pg[YT], nextpg[YT];
    auto begin = [&]() {
        if (lane == 0) {
            for (int i = 0; i < PS; ++i) mbar_init(&packed[i], 1);
            fence_mbar_init();
        }
        __syncwarp();
        pages_of(0, pg);
#pragma unroll
        for (int y = 0; y < YT; ++y) nextpg[y] = pg[y];
        for (int c = 0; c < min(PS, steps); ++c) {
            int page[YT];
#pragma unroll
            for (int y = 0; y < YT; ++y) page[y] = __shfl_sync(0xffffffffu, pg[y], c);
            if (lane == 0) issue(c, page);
        }
    };
    if (HD == 64 && warp >= L::SOFT && warp < L::MMA) begin();
    float qscale = 0.f;
    // the tiles' queries, a thread a unit: q 2^-eq in fp16, its largest |dim| in [2^3, 2^4)
    if (warp < L::SOFT) {
        const int u = u0 + tid;
        const bool ok = u < units;
        const int j = ok ? u / a.group : 0, g = ok ? u - j * a.group : 0;
        const __nv_bfloat16* src = a.q + (row0 + j) * a.q_row + (h * a.group + g) * a.q_head;
        const bool wide = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
        auto dims = [&](int i, uint32_t* w) {   // 8 i ..
            const uint32_t* src2 = reinterpret_cast<const uint32_t*>(src) + 4 * i;
            if (!ok) {
                w[0] = w[1] = w[2] = w[3] = 0;
            } else if (wide) {
                *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(src2);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = src2[e];
            }
        };
        uint32_t top = 0, w[4];
#pragma unroll 4
        for (int i = 0; i < HD / 8; ++i) {
            dims(i, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, max(w[e] << 16 & 0x7fffffffu, w[e] & 0x7fff0000u));
        }
        const int eq = kv4_query_exponent(top);
        const float f = kv4_exp2i(-eq);
        qscale = fminf(a.scale_log2 * kv4_exp2i(eq), 3.4e38f);
        const int row = tid & 127;
        const uint32_t qt = sb + L::Q + (uint32_t)(tid >> 7) * L::QB + (row >> 3) * 1024 + (row & 7) * 128;
#pragma unroll 4
        for (int i = 0; i < HD / 8; ++i) {
            dims(i, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = kv4_half2(kv4_s(w[e]) * f, kv4_z(w[e]) * f);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(qt + (i >> 3) * (128 * 128) +
                                                                          (((i & 7) ^ (row & 7)) << 4)),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
        }
        fence_async();
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = ms.tmem;

    if (warp >= L::MMA) {
        const int t = warp - L::MMA;
        if (n > 0 && t < tiles) {
            const uint32_t one = elect(), tm = __shfl_sync(0xffffffffu, tmem, 0);
            auto ready = [&](uint64_t* bar, uint32_t parity) {
                const bool ok = __all_sync(0xffffffffu, wait(bar, parity, abort));
                fence_after();
                return ok;
            };
            const uint32_t qt = desc(sb + L::Q + t * L::QB);
            bool ok = ready(&ms.kv_full[0], 0);
            for (int c = 0; ok && c < n; ++c) {
                // scores, over the weights of chunk c - 1
                if (c > 0 && !(ok = ready(&ms.pv_done[t], (c - 1) & 1))) break;
                const uint32_t kt = desc(sb + L::K + (c % KS) * L::KB);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ++ks)
                    mma_ss(one, tm + L::S_COL + t * CK, qt + (((ks >> 2) * (128 * 128) + (ks & 3) * 32) >> 4),
                           kt + (((ks >> 2) * (CK * 128) + (ks & 3) * 32) >> 4), idesc(CK), ks > 0);
                commit(one, &ms.s_full[t]);
                // (the next chunk's operands are waited for here, off the way from weights to scores)
                if (c + 1 < n && !(ok = ready(&ms.kv_full[(c + 1) % KS], ((c + 1) / KS) & 1))) break;
                if (!(ok = ready(&ms.p_full[t], c & 1))) break;
                const uint32_t vt = desc(sb + L::V + (c % KS) * L::KB);
#pragma unroll
                for (int ks = 0; ks < CK / 16; ++ks)
                    mma_ts(one, tm + L::O_COL + t * HD, tm + L::S_COL + t * CK + ks * 8, vt + ks * 2, idesc(HD),
                           c > 0 || ks > 0);
                commit(one, &ms.pv_done[t]);
                commit(one, &ms.kv_empty[c % KS]);
            }
            commit(one, &ms.drain[t]);   // every MMA issued has completed
            mbar_wait(&ms.drain[t], 0);
        }
        __syncwarp();
    } else if (warp >= L::SOFT) {
        const int r = lane >> 2, t = lane & 3;
        if (HD != 64) begin();
        bool good = true;   // no wait of this warp has run out; the warps leave together
        Kv4Unit unit;       // (the same in all unpacking warps)
        int c = 0;
        for (; c < steps; ++c) {
            const int st = c % PS, sg = c & 1, k0 = base + c * SK;
            if (c > 0 && (c & 31) == 0)
#pragma unroll
                for (int y = 0; y < YT; ++y) pg[y] = nextpg[y];
            bool there[YT];
#pragma unroll
            for (int y = 0; y < YT; ++y) there[y] = __shfl_sync(0xffffffffu, pg[y], c & 31) >= 0;
            if (good) good = __all_sync(0xffffffffu, wait(&packed[st], (c / PS) & 1, abort));
            const unsigned char* pk = ring + st * YT * L::TB;
            // the largest magnitudes that the step's s and z allow, and the tiles' NaN groups of V
            uint32_t topk = 0, topv = 0;
            bool bad[YT][NB], any_bad[YT];
#pragma unroll
            for (int y = 0; y < YT; ++y) {
                const uint32_t* kp = reinterpret_cast<const uint32_t*>(pk + y * L::TB + T::KP);
                const uint32_t* vp = reinterpret_cast<const uint32_t*>(pk + y * L::TB + T::VP);
                any_bad[y] = false;
#pragma unroll
                for (int x = 0; x < NB; ++x) {
                    const int at = x * 32 + lane, slot = at / NG;
                    const int key = k0 + 16 * (4 * (y0 + y) + w) + (slot >> 1) + 8 * (slot & 1);
                    const bool in = there[y] && key >= kmin && key < kmax;
                    const uint32_t kw = kp[at], vw = vp[at];
                    topk = max(topk, in ? kv4_top(kw) : 0u);
                    topv = max(topv, in ? kv4_top(vw) : 0u);
                    bad[y][x] = in && !(kv4_z(vw) == kv4_z(vw));
                    any_bad[y] |= bad[y][x];
                }
                any_bad[y] = __any_sync(0xffffffffu, any_bad[y]);
            }
            topk = __reduce_max_sync(0xffffffffu, topk);
            topv = __reduce_max_sync(0xffffffffu, topv);
            if (lane == 0) {
                ms.top[sg][uw][0] = topk;
                ms.top[sg][uw][1] = topv;
                ms.stop[sg][uw] = !good;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(L::UNPACK * 32) : "memory");
            topk = __reduce_max_sync(0xffffffffu, ms.top[sg][lane % L::UNPACK][0]);
            topv = __reduce_max_sync(0xffffffffu, ms.top[sg][lane % L::UNPACK][1]);
            if (__any_sync(0xffffffffu, ms.stop[sg][lane % L::UNPACK] != 0)) break;
            const int ek = kv4_exponent_out(topk);
            const float factor = unit.next(topv);
            const float fk = kv4_exp2i(-ek), fv = kv4_exp2i(-unit.ev);
#pragma unroll
            for (int y = 0; y < YT; ++y) {
                const int ch = 2 * c + y0 + y, sk = ch % KS, tl = 4 * (y0 + y) + w;
                // the stage's readers: every tile's MMAs and softmax of chunk ch - KS
                if (good && ch < n && ch >= KS)
                    good = __all_sync(0xffffffffu, wait(&ms.kv_empty[sk], (ch / KS - 1) & 1, abort));
                if (!good || ch >= n) continue;
                if (any_bad[y]) {   // rare: which groups of which keys
#pragma unroll
                    for (int x = 0; x < NB; ++x) {
                        uint32_t bits = bad[y][x] ? 1u << (lane % NG) : 0u;
#pragma unroll
                        for (int o = 1; o < NG; o <<= 1) bits |= __shfl_xor_sync(0xffffffffu, bits, o);
                        const int slot = (x * 32 + lane) / NG;
                        if (lane % NG == 0) ms.bad_groups[sk][16 * w + (slot >> 1) + 8 * (slot & 1)] = (uint8_t)bits;
                    }
                }
                const uint32_t kt = sb + L::K + sk * L::KB, vt = sb + L::V + sk * L::KB;
                const unsigned char* tp = pk + y * L::TB;
                uint32_t code[NB][4], par[2 * NG];
#pragma unroll
                for (int x = 0; x < NB; ++x)
                    *reinterpret_cast<uint4*>(code[x]) = *reinterpret_cast<const uint4*>(tp + x * T::BLK + lane * 16);
#pragma unroll
                for (int x = 0; x < 2 * NG; x += 4)
                    *reinterpret_cast<uint4*>(par + x) = *reinterpret_cast<const uint4*>(tp + T::KP + r * 8 * NG + x * 4);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int key = k0 + 16 * tl + r + 8 * hf;
                    const bool in = there[y] && key >= kmin && key < kmax;
                    const uint32_t row = kt + (2 * w + hf) * 1024 + r * 128 + 4 * t;
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const float s = in ? kv4_s(par[hf * NG + g]) * fk : 0.f, z = in ? kv4_z(par[hf * NG + g]) * fk : 0.f;
                        uint32_t x[4];
                        kv4_unpack4(code[g >> 1][2 * hf + (g & 1)], kv4_half2(s, s), kv4_half2(z, z), x);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            sts(row + (g >> 1) * (CK * 128) + (((4 * (g & 1) + i) ^ r) << 4), x[i]);
                    }
                }
                uint32_t vpar[4 * NG];   // tokens 2t, 2t + 8, 2t + 1, 2t + 9
#pragma unroll
                for (int x = 0; x < NB; ++x)
                    *reinterpret_cast<uint4*>(code[x]) = *reinterpret_cast<const uint4*>(tp + T::V + x * T::BLK + lane * 16);
#pragma unroll
                for (int x = 0; x < 4 * NG; x += 4)
                    *reinterpret_cast<uint4*>(vpar + x) = *reinterpret_cast<const uint4*>(tp + T::VP + t * 16 * NG + x * 4);
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    const int key = k0 + 16 * tl + 2 * t + 8 * hf;
                    const bool in0 = there[y] && key >= kmin && key < kmax, in1 = there[y] && key + 1 >= kmin && key + 1 < kmax;
                    const uint32_t blk = vt + r * 128 + (((2 * w + hf) ^ r) << 4) + 4 * t;
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const uint32_t p0 = vpar[hf * NG + g], p1 = vpar[(2 + hf) * NG + g];
                        const bool ok0 = in0 && kv4_z(p0) == kv4_z(p0), ok1 = in1 && kv4_z(p1) == kv4_z(p1);
                        const uint32_t s = kv4_half2(ok0 ? kv4_s(p0) * fv : 0.f, ok1 ? kv4_s(p1) * fv : 0.f);
                        const uint32_t z = kv4_half2(ok0 ? kv4_z(p0) * fv : 0.f, ok1 ? kv4_z(p1) * fv : 0.f);
                        uint32_t x[4];
                        kv4_unpack4(code[g >> 1][2 * (g & 1) + hf], s, z, x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) sts(blk + (4 * g + i) * 1024, x[i]);
                    }
                }
                if (lane == 0) {
                    const bool moved = factor != 1.f && !(ch & 1);   // with the step's first chunk
                    reinterpret_cast<uint8_t*>(&ms.mark[sk])[w] =
                        (uint8_t)((there[y] ? 0u : GONE) | (any_bad[y] ? BAD : 0u) | (moved ? MOVED : 0u));
                    if (w == 0) {
                        ms.kscale[sk] = kv4_exp2i(ek);
                        ms.shift[sk] = (float)(unit.ev - unit.er);
                        ms.factor[sk] = factor;
                        ms.er[sk] = unit.er;
                    }
                }
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ms.kv_full[sk]);
            }
            __syncwarp();   // every lane has read the stage
            const int nx = c + PS;
            if (nx < steps) {
                if ((nx & 31) == 0) pages_of(nx, nextpg);
                int page[YT];
#pragma unroll
                for (int y = 0; y < YT; ++y)
                    page[y] = __shfl_sync(0xffffffffu, (nx >> 5) == (c >> 5) ? pg[y] : nextpg[y], nx & 31);
                if (lane == 0) issue(nx, page);
            }
        }
        // what was issued lands before the CTA ends
        for (int i = c; i < min(steps, c + PS); ++i) mbar_wait(&packed[i % PS], (i / PS) & 1);
    } else {
        // softmax: unit u, TMEM lane (warp % 4) 32 + lane of tile warp / 4
        const int tile = warp >> 2, u = u0 + tid;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + L::S_COL + tile * CK, o_at = tmem + lanes + L::O_COL + tile * HD;
        const int pos = len - nq + min(u, units - 1) / a.group;
        const int lo = low(pos), hi = pos + 1;
        // keys that every unit of the warp sees
        const int ua = min(u - lane, units - 1), ub = min(u - lane + 31, units - 1);
        const int all_lo = low(len - nq + ub / a.group), all_hi = len - nq + ua / a.group + 1;
        float m = KV4_NEG, l = 0.f;
        uint32_t bad = 0;
        // the chunk's scale of scores, eV - er and marks, taken while its scores are computed
        float kq = 0.f, shift = 0.f;
        uint32_t mark = 0;
        auto chunk = [&](int c) {
            const int sk = c % KS;
            const bool there = __all_sync(0xffffffffu, wait(&ms.kv_full[sk], (c / KS) & 1, abort));
            kq = kv4_score_factor(qscale, ms.kscale[sk]);
            shift = ms.shift[sk];
            mark = ms.mark[sk];
            return there;
        };
        bool ok = tile < tiles && n > 0;
        if (ok) ok = chunk(0);
        for (int c = 0; ok && c < n; ++c) {
            const int sk = c % KS, k0 = base + c * CK;
            ok = __all_sync(0xffffffffu, wait(&ms.s_full[tile], c & 1, abort));
            if (!ok) break;
            fence_after();
            const bool edge = k0 < all_lo || k0 + CK > all_hi || (mark & GONE);
            const int lo_c = lo - k0, hi_c = hi - k0;
            // scores of keys 32 q .. of the chunk; those that the unit does not see: -inf
            auto scores = [&](int q, uint32_t* v) {
                ld32(s_at + 32 * q, v);
                ld_wait(v);
                if (edge) {
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (32 * q + k < lo_c || 32 * q + k >= hi_c || (mark >> (8 * (2 * q + (k >> 4))) & 1)) v[k] = 0xff800000u;
                }
            };
            // weights with the reference m; their sum
            uint32_t p[CK / 2];
            auto weigh = [&]() {
                const f32x2 f2 = two(kq, kq), b2 = two(shift - m, shift - m);
                f32x2 sum = two(0.f, 0.f);
#pragma unroll
                for (int q = 0; q < CK / 32; ++q) {
                    uint32_t v[32];
                    scores(q, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float x, y;
                        parts(fma2(two(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), f2, b2), x, y);
                        x = kv4_ex2(x);
                        y = kv4_ex2(y);
                        sum = add2(sum, two(x, y));
                        p[16 * q + i] = kv4_half2(x, y);
                    }
                }
                float x, y;
                parts(sum, x, y);
                return x + y;
            };
            // m to the largest score so far less ROOM, the row of O with it and to its new unit (the scores say
            // that P V of the chunk before has completed)
            auto raise = [&]() {
                float top = -INFINITY;
#pragma unroll
                for (int q = 0; q < CK / 32; ++q) {
                    uint32_t v[32];
                    scores(q, v);
#pragma unroll
                    for (int k = 0; k < 32; ++k) top = fmaxf(top, fmaf(__uint_as_float(v[k]), kq, shift));
                }
                top = fmaxf(m, top - KV4_ROOM);
                float f = kv4_ex2(m - top);
                m = top;
                l *= f;
                if (mark & MOVED) f *= ms.factor[sk];
                if (c > 0) {
#pragma unroll
                    for (int q = 0; q < HD / 16; ++q) {
                        uint32_t o[16];
                        ld16(o_at + 16 * q, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        st16(o_at + 16 * q, o);
                    }
                }
            };
            float sum = 0.f;
            bool moved = c == 0 || (mark & MOVED);   // (the same for the warp)
            if (!moved) {
                sum = weigh();
                moved = __any_sync(0xffffffffu, sum > KV4_FULL);
            }
            if (moved) {
                raise();
                sum = weigh();
            }
            st16(s_at, p);
            st16(s_at + 16, p + 16);
            l = fmaf(sum, kv4_ex2(-shift), l);
            if (mark & BAD) {
                for (int k = max(lo_c, 0); k < min(hi_c, CK); ++k)
                    if (mark >> (8 * (k >> 4)) & 2) bad |= ms.bad_groups[sk][k];
            }
            st_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ms.p_full[tile]);
            if (c + 1 < n) ok = chunk(c + 1);
        }
        if (tile < tiles) {
            if (n == 0) ok = true;
            else if (ok) ok = wait(&ms.pv_done[tile], (n - 1) & 1, abort) && !*abort;
            ok = __all_sync(0xffffffffu, ok);
            fence_after();
            if (!ok) bad = 0xffu;
            const int er = n > 0 ? ms.er[(n - 1) % KS] : 0;
            l *= kv4_exp2i(-er);
            const bool row_ok = u < units;
            const int j = row_ok ? u / a.group : 0, g = row_ok ? u - j * a.group : 0;
            const int64_t at = (int64_t)(row0 + j) * a.hq + h * a.group + g;
            const float inv = rg.used > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int q = 0; q < HD / 16; ++q) {
                uint32_t v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = 0;
                if (ok && n > 0) ld16(o_at + 16 * q, v);
                if (!row_ok) continue;
                float x[16];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    x[i] = bad >> (q / 2) & 1 ? __int_as_float(0x7fffffff) : __uint_as_float(v[i]) * inv;
                if (rg.used > 1) {
                    float4* o = reinterpret_cast<float4*>(a.part_o + (at * a.nsplit + split) * HD + 16 * q);
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
                } else {
                    uint4* o = reinterpret_cast<uint4*>(a.out + at * HD + 16 * q);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        __nv_bfloat162 y[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = __floats2bfloat162_rn(x[8 * i + 2 * e], x[8 * i + 2 * e + 1]);
                        o[i] = *reinterpret_cast<uint4*>(y);
                    }
                }
            }
            if (row_ok && rg.used > 1) {
                a.part_ml[(at * a.nsplit + split) * 2] = m + (float)er;
                a.part_ml[(at * a.nsplit + split) * 2 + 1] = l;
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == L::MMA)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

}  // namespace

namespace pulsar {

int kv4_prefill_launch(const Kv4AttnArgs& a, int head_dim, int64_t sequences, int utiles, cudaStream_t stream) {
    const dim3 grid((unsigned)(utiles * a.nsplit), (unsigned)a.hkv, (unsigned)sequences);
    if (head_dim == 64) {
        constexpr int bytes = Lay<64>::BYTES + 1024;
        PULSAR_TRY(ensure_smem_attr((const void*)k_kv4_prefill<64>, bytes, "k_kv4_prefill shared memory"));
        k_kv4_prefill<64><<<grid, Lay<64>::THREADS, bytes, stream>>>(a);
    } else {
        constexpr int bytes = Lay<128>::BYTES + 1024;
        PULSAR_TRY(ensure_smem_attr((const void*)k_kv4_prefill<128>, bytes, "k_kv4_prefill shared memory"));
        k_kv4_prefill<128><<<grid, Lay<128>::THREADS, bytes, stream>>>(a);
    }
    PULSAR_LAUNCH_CHECK("k_kv4_prefill");
    return PULSAR_OK;
}

}  // namespace pulsar
