// Attention over pages of int8 codes for prompt portions, on the 5th-generation tensor cores.  Head sizes 64 and 128, bfloat16 queries.
// Formulas in attention_q8.cuh.
//
// A CTA owns up to 256 rows - (token, query head of one kv group) pairs, token-major - as two row tiles A and B of 128, and walks the keys
// its rows may see in tiles of 128.  Twenty warps in five groups, coupled by mbarriers:
//   warps 0-3, 4-7   softmax of A and of B: a thread owns a row, its 128 scores in registers; P goes back over S in TMEM as float16;
//   warp 8           one thread issues S_X = Q_X K^T and O_X += P_X V, tcgen05.mma M = 128, N = 128 (N = head size), in the order
//                    S_A S_B | PV_A S_A' PV_B S_B' | ..., so that one row tile is multiplied while the other is softmaxed;
//   warps 12-15      bring the codes of K from the cache, 16 bytes a lane, widen them to float16 and write them to shared memory in the
//                    swizzled layout of an operand, two stages ahead of the products at most; eight lanes of warp 12 bring the blocks'
//                    scales along;
//   warps 16-19      the same for V.
// A code is widened as the low byte of the float16 number 1024 + (c + 128), less 1152: a permutation for two codes and a subtraction of
// pairs.  Reading codes and not 16-bit numbers halves what a CTA fetches; the widening, 32,768 codes a key tile, takes some 1,800 of the
// four schedulers' issue slots, beside 4,100 of the softmax and 2,048 cycles of products at head size 128.
// The softmax groups hold 176 registers a thread, the others 40: what the 640 threads were launched with, dealt out again.  The roles share
// the SM's instruction caches, and the softmax is long, so the others are loops of a hundred instructions: with its eight products and their
// descriptors unrolled the issuing thread took 3,000 cycles for products of 64 each to have its code fetched.
//
// Scores enter the softmax as x = s * ck + lv with ck = (the key's scale) * (the row's), lv = log2 of the value's scale, both the same for
// 16 keys: the maximum is taken per block before the scales, and the exponent is one multiply-add as without them.  The sum of a block's
// weights is divided by its value's scale once.  The output accumulates in TMEM against a reference that moves only when a row's maximum
// has outgrown it by 8.  Codes are numbers whatever a stale page holds, so nothing has to be cleared.
//
// HALVES: a CTA with one row tile (up to 128 rows), whose even key tiles go to stream A and odd ones to B, over the same queries; the rows'
// two states are merged at the end.  Every wait is bounded.
//
// Bound by a row tile's chain: from its scores to its weights 2,900 cycles (4,000 where both streams' warps are at it), from there to the next
// scores 1,850, of which its products are 1,024; a pair of row tiles and a key tile take 4,850 cycles, where the products alone would take
// 2,048 at head size 128.  (At head size 64 TMEM has room for weights beside the scores, so that the next scores are there at once: 2 % faster
// at 8,192 tokens, 3 % slower or the same at 500, not kept.)  A CTA's beginning - queries, table, first codes - takes some 6,000.
// 32 / 8 heads of 128: a prompt of 2,048 tokens 57 us, 600 TFLOP/s, of 8,192 650 us, 850 TFLOP/s; 500 tokens behind 1,500 31 us, 470 TFLOP/s.
#include "attention_q8.cuh"
#include "tcgen05.cuh"

#include <math.h>

__device__ int g_q8t_error = 0;

namespace {

constexpr int THREADS = 640, BM = 128, BN = 128, BLOCKS = BN / Q8_BLOCK;
constexpr int SOFTMAX_REGS = 176, OTHER_REGS = 40;      // of 256 and of 384 threads: 60,416 in all; the launch has 640 x 96
constexpr uint32_t MAGIC = 0x64646464u;
constexpr float STEP = 8.0f;                            // log2 units by which a row's maximum may outgrow its reference

enum { Q_FULL = 0, K_FULL = 1, K_EMPTY = 3, V_FULL = 5, V_EMPTY = 7, S_FULL = 9, P_FULL = 11, PV_DONE = 13, SCALES_FULL = 15, BARS = 19 };

template <int HD, bool HALVES> struct Lay {
    static constexpr uint32_t PANEL = 128 * 128, PANELS = HD / 64, TILE = PANELS * PANEL;       // 128 rows of HD float16 numbers
    static constexpr uint32_t Q = 0, K = (HALVES ? 1 : 2) * TILE, V = K + 2 * TILE;             // Q_A (Q_B) | two stages of K | of V
    // codes on their way: two tiles of K and of V where there is room for them
    static constexpr int AHEAD = HD == 128 && !HALVES ? 0 : 2;
    static constexpr uint32_t CODES = V + 2 * TILE, RAW = 128 * HD, SCALES = CODES + 2 * AHEAD * RAW;
    static constexpr uint32_t ROWS = SCALES + 4 * BLOCKS * 16, BARRIERS = ROWS + 256 * 4, TMEM = BARRIERS + 8 * BARS, BYTES = TMEM + 16;
    static constexpr uint32_t TMEM_COLS = 512, O = 256;                                         // S_A S_B at 0 and 128, O_A O_B behind
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a) {             // - 1152 from both halves
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(0x64806480u));
    return d;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &lo, float &hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 32 consecutive TMEM columns of this thread's lane; ld_wait() before they are used
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// 16 packed words into 16 consecutive TMEM columns of this thread's lane
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D (TMEM) = or += A (TMEM, M x 16 packed two to a column) x B (shared memory)
__device__ __forceinline__ void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t at, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint4 ldg128(const int8_t *p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
// eight codes as eight float16 numbers
__device__ __forceinline__ uint4 widen(uint32_t a, uint32_t b) {
    a ^= 0x80808080u;
    b ^= 0x80808080u;
    return make_uint4(hsub2(__byte_perm(a, MAGIC, 0x4140)), hsub2(__byte_perm(a, MAGIC, 0x4342)),
                      hsub2(__byte_perm(b, MAGIC, 0x4140)), hsub2(__byte_perm(b, MAGIC, 0x4342)));
}

// One plane's widening, by four warps of which this is the w-th: key tiles of 128 into a ring of two stages at `ring`.  A warp's load is one
// unit: 512 bytes, 4 keys at head size 128 and 8 at 64.  Codes come by cp.async, two tiles ahead, every lane's into places that it alone
// reads.  Where shared memory has no room for them a warp has four units in flight in registers: once one is widened the load of the fourth
// after it starts, over the tiles' borders.  (32 / 8 heads of 128, 500 tokens behind 1,500 32 us, 38 through registers; 16 / 4 of 64, 2,048
// tokens 43 and 45; with one tile ahead, for which the larger layout has room, a prompt of 2,048 tokens of 32 / 8 heads of 128 59, 57
// through registers.)  A quarter-warp's stores of 16 bytes go to two keys and every other chunk, which the swizzle
// spreads over all banks.  Both planes' warps run the same instructions: with a copy for each, and all of a tile unrolled, the kernel
// waited for its code, and for what did not fit its registers.
template <int HD, bool HALVES>
__device__ __forceinline__ void convert(const Q8Params &p, const int *table, int kvh, const int8_t *plane, int w, bool scaled, int lane, int k_lo, int n_tiles,
                                        uint32_t base, uint32_t ring, uint32_t codes, int full0, int empty0, int error) {
    using L = Lay<HD, HALVES>;
    constexpr int KEYS = 512 / HD, MINE = BN / KEYS / 4, DEEP = 4;         // units of a tile that are this warp's: 8, or 4
    auto bar = [&](int i) { return base + L::BARRIERS + 8u * (uint32_t)i; };
    const int key = w * KEYS + (HD == 128 ? (lane >> 2) & 3 : lane >> 2);                   // among the keys of the four warps' units: 16, or 32
    const int chunk = HD == 128 ? (lane & 3) + 4 * (lane >> 4) : lane & 3;
    const uint32_t at0 = base + ring + (uint32_t)(chunk >> 2) * L::PANEL + swizzle128(key, 2 * (chunk & 3));
    const uint32_t at1 = base + ring + (uint32_t)(chunk >> 2) * L::PANEL + swizzle128(key, 2 * (chunk & 3) + 1);
    plane += (size_t)(key % Q8_BLOCK) * HD + 16 * chunk;
    // lane l (modulo 8) knows the cache row of a tile's l-th block
    auto rows_of = [&](int i) { return i < n_tiles ? q8_row_of(p, table, kvh, k_lo + i * BN + (lane & 7) * Q8_BLOCK) : 0; };
    auto load = [&](int rows, int u) {
        const int row = __shfl_sync(0xffffffffu, rows, HD == 128 ? u : 2 * u + (w >> 1));
        return plane + (size_t)row * HD;
    };
    // tile i's codes, asked for into this lane's own places of slot i % 2
    const uint32_t mine = base + codes + w * (MINE * 512) + lane * 16;
    auto fetch = [&](int i, int rows) {
        const uint32_t to = mine + (i & 1) * L::RAW;
        if (i < n_tiles) {
#pragma unroll
            for (int u = 0; u < MINE; ++u) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + u * 512), "l"(load(rows, u)) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int rows = rows_of(0), rows_next = rows_of(1), rows_after = L::AHEAD > 0 ? rows_of(2) : 0;
    uint4 q[DEEP];
    if constexpr (L::AHEAD > 0) {
        fetch(0, rows);
        fetch(1, rows_next);
    } else {
#pragma unroll
        for (int u = 0; u < DEEP; ++u) q[u] = ldg128(load(rows, u));
    }
#pragma unroll 1
    for (int i = 0; i < n_tiles; ++i) {
        const int b = i & 1;
        float sk = 0.f, sv = 0.f;
        if (scaled && lane < BLOCKS) sk = p.ks[rows / Q8_BLOCK], sv = p.vs[rows / Q8_BLOCK];
        const int rows_last = rows_of(i + (L::AHEAD > 0 ? 3 : 2));
        if constexpr (L::AHEAD > 0) asm volatile("cp.async.wait_group 1;" ::: "memory");
        if (!mbar_wait(bar(empty0 + b), (uint32_t)((i >> 1) + 1) & 1u)) { atomicExch(&g_q8t_error, error); break; }
#pragma unroll 1
        for (int h = 0; h < MINE; h += DEEP) {
#pragma unroll
            for (int u = 0; u < DEEP; ++u) {
                const uint32_t off = b * L::TILE + (uint32_t)(h + u) * (4 * KEYS * 128);
                if constexpr (L::AHEAD > 0) q[u] = lds128(mine + b * L::RAW + (h + u) * 512);
                sts128(at0 + off, widen(q[u].x, q[u].y));
                sts128(at1 + off, widen(q[u].z, q[u].w));
                // behind the last tile the rows are 0: a load that nothing waits for
                if constexpr (L::AHEAD == 0) q[u] = ldg128(h + DEEP < MINE ? load(rows, h + DEEP + u) : load(rows_next, u));
            }
        }
        if constexpr (L::AHEAD > 0) fetch(i + 2, rows_after);      // into the slot that was just read
        if (scaled) {
            // Slot i % 4 is free: tile i's stage was, so S(i - 2) is done, before which every thread was through with tile i - 4.
            // A scale that is no positive number becomes one that makes the sum of a row that sees the block no number, and no other's:
            // the weights of such a row come out as 2^0 against a reference that nothing else reaches, and 1 / s_v is NaN.
            const bool bad = !(sk >= 0.f && sk <= 3.4e38f && sv >= 0.f && sv <= 3.4e38f);
            const float k = bad ? Q8_LEAST_SCALE : fmaxf(sk, Q8_LEAST_SCALE), v = fmaxf(sv, Q8_LEAST_SCALE);
            if (lane < BLOCKS)
                sts128(base + L::SCALES + ((i & 3) * BLOCKS + lane) * 16, make_uint4(__float_as_uint(k), __float_as_uint(bad ? 3e4f : log2_fast(v)),
                                                                                     bad ? 0x7fc00000u : __float_as_uint(1.0f / v), 0));
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(SCALES_FULL + (i & 3)));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");     // these writes -> tensor-core reads
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(full0 + b));
        rows = rows_next;
        if (L::AHEAD > 0) {
            rows_next = rows_after;
            rows_after = rows_last;
        } else {
            rows_next = rows_last;
        }
    }
}

template <int HD, bool HALVES>
__global__ void __launch_bounds__(THREADS, 1) attention_q8_tc_kernel(const Q8Params p) {
    pdl_launch_dependents();
    using L = Lay<HD, HALVES>;
    // float16 x float16 -> float32, M = 128; S: both operands K-major, N = 128; PV: B is MN-major, N = head size
    constexpr uint32_t IDESC_S = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
    constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
    extern __shared__ uint8_t q8t_smem[];
    const uint32_t base = (smem_u32(q8t_smem) + 1023u) & ~1023u;
    uint8_t *aligned = q8t_smem + (base - smem_u32(q8t_smem));
    auto bar = [&](int i) { return base + L::BARRIERS + 8u * (uint32_t)i; };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (!p.described) pdl_wait();
    // late tiles, which see the most keys, come first - across all kv heads
    const int kvh = blockIdx.x % p.nkv, slice = blockIdx.z;
    Q8Tile t;
    if (!q8_find_tile(p, (int)(gridDim.x / p.nkv) - 1 - (int)(blockIdx.x / p.nkv), t)) { pdl_wait(); return; }

    if (tid == 0) {
        mbar_init(bar(Q_FULL), 8);
        for (int b = 0; b < 2; ++b) {
            mbar_init(bar(K_FULL + b), 4);  mbar_init(bar(K_EMPTY + b), 1);
            mbar_init(bar(V_FULL + b), 4);  mbar_init(bar(V_EMPTY + b), 1);
            mbar_init(bar(S_FULL + b), 1);  mbar_init(bar(P_FULL + b), 4);
            mbar_init(bar(PV_DONE + b), 1);
        }
        for (int b = 0; b < 4; ++b) mbar_init(bar(SCALES_FULL + b), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + L::TMEM), "r"(L::TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t *)(aligned + L::TMEM);
    pdl_wait();

    int k_first, k_hi;                                  // keys that this CTA's rows may see in its slice
    q8_slice(t, p.slices, slice, BN, k_first, k_hi);
    const int k_lo = k_first / BN * BN;
    const int n_tiles = k_hi > k_first ? (k_hi - k_lo + BN - 1) / BN : 0;
    // row tile A ends earlier: it skips the key tiles beyond its last row
    const int rows_a = min(t.rows, BM);
    const bool has_b = HALVES || t.rows > BM;
    const int k_hi_a = HALVES ? k_hi : min(t.pos_begin + (t.row0 + rows_a - 1) / t.G + 1, k_hi);
    const int n_tiles_a = HALVES ? (n_tiles + 1) / 2 : k_hi_a > k_lo ? min(n_tiles, (k_hi_a - k_lo + BN - 1) / BN) : 0;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(OTHER_REGS));
        if (warp >= 12) {
            const bool is_v = warp >= 16;
            if (n_tiles > 0)
                convert<HD, HALVES>(p, t.table, kvh, is_v ? p.v : p.k, warp & 3, warp == 12, lane, k_lo, n_tiles, base, is_v ? L::V : L::K,
                            L::CODES + (is_v ? L::AHEAD * L::RAW : 0), is_v ? V_FULL : K_FULL,
                            is_v ? V_EMPTY : K_EMPTY, is_v ? 4 : 3);
        } else if (warp == 8 && lane == 0 && n_tiles > 0) {
            // ---- issuer
            bool ok = mbar_wait(bar(Q_FULL), 0);
            if (!ok) atomicExch(&g_q8t_error, 5);
            const uint64_t q_desc = smem_desc(base + L::Q), k_desc = smem_desc(base + L::K), v_desc = smem_desc_mn_major(base + L::V, L::PANEL);
            auto issue_s = [&](int x, int i) {
                uint64_t dq = q_desc + (HALVES ? 0 : x * (L::TILE >> 4)), dk = k_desc + (i & 1) * (L::TILE >> 4);
#pragma unroll 1
                for (int pn = 0; pn < (int)L::PANELS; ++pn) {
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) tc_mma(tmem + x * 128, dq + 2 * ks, dk + 2 * ks, IDESC_S, (pn > 0 || ks > 0) ? 1u : 0u);      // 32 bytes on
                    dq += L::PANEL >> 4;
                    dk += L::PANEL >> 4;
                }
                tc_commit(bar(S_FULL + x));
            };
            auto issue_pv = [&](int x, int i) {
                if (!mbar_wait(bar(P_FULL + x), (uint32_t)(HALVES ? i >> 1 : i) & 1u)) { atomicExch(&g_q8t_error, 2); return false; }
                tc_fence_after();
                // A = P: keys 16 ks.. are columns 8 ks..; B = V: 16 keys down = 2 groups of 8 rows = 2,048 bytes
                uint64_t dv = v_desc + (i & 1) * (L::TILE >> 4);
                uint32_t pa = tmem + x * 128;
                const bool more = i > (HALVES ? 1 : 0);
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) mma_ts(tmem + L::O + x * 128, pa + 8 * ks, dv + 128 * ks, IDESC_PV, (more || h > 0 || ks > 0) ? 1u : 0u);
                    dv += 512;
                    pa += 32;
                }
                tc_commit(bar(PV_DONE + x));
                return true;
            };
            auto wait_k = [&](int i) {
                if (mbar_wait(bar(K_FULL + (i & 1)), (uint32_t)(i >> 1) & 1u)) { tc_fence_after(); return true; }
                atomicExch(&g_q8t_error, 1);
                return false;
            };
            auto wait_v = [&](int i) {
                if (mbar_wait(bar(V_FULL + (i & 1)), (uint32_t)(i >> 1) & 1u)) { tc_fence_after(); return true; }
                atomicExch(&g_q8t_error, 6);
                return false;
            };
            if (HALVES) {
                // per stream: S(i) | PV(i), S(i + 2); tile i is stream i % 2's step i / 2, and so is its stage
                for (int i = 0; i < min(2, n_tiles) && ok; ++i) {
                    if (!(ok = wait_k(i))) break;
                    issue_s(i, i);
                    tc_commit(bar(K_EMPTY + i));
                }
                for (int i = 0; i < n_tiles && ok; ++i) {
                    const int x = i & 1;
                    if (!(ok = wait_v(i)) || !(ok = issue_pv(x, i))) break;
                    tc_commit(bar(V_EMPTY + x));
                    if (i + 2 < n_tiles) {
                        if (!(ok = wait_k(i + 2))) break;
                        issue_s(x, i + 2);
                        tc_commit(bar(K_EMPTY + x));
                    }
                }
            } else {
                if (ok && (ok = wait_k(0))) {
                    if (n_tiles_a > 0) issue_s(0, 0);
                    if (has_b) issue_s(1, 0);
                    tc_commit(bar(K_EMPTY + 0));
                }
                for (int i = 0; i < n_tiles && ok; ++i) {
                    const bool next = i + 1 < n_tiles;
                    if (!(ok = wait_v(i))) break;
                    if (next && !(ok = wait_k(i + 1))) break;
                    // PV_A(i), S_A(i+1), PV_B(i), S_B(i+1): the products of one row tile fill the time the other's softmax takes
                    if (i < n_tiles_a && !(ok = issue_pv(0, i))) break;
                    if (next && i + 1 < n_tiles_a) issue_s(0, i + 1);
                    if (has_b && !(ok = issue_pv(1, i))) break;
                    if (next && has_b) issue_s(1, i + 1);
                    if (next) tc_commit(bar(K_EMPTY + ((i + 1) & 1)));
                    tc_commit(bar(V_EMPTY + (i & 1)));
                }
            }
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(SOFTMAX_REGS));
        // ---- softmax: thread r of a row tile owns row r (TMEM lane r)
        const int x = warp >> 2, r = tid & 127;
        float *row_up = reinterpret_cast<float *>(aligned + L::ROWS);
        {
            // Queries, in float16: a row is multiplied by the power of two that brings its largest number to [64, 128), so that a bfloat16
            // number keeps its bits down to 2^-21 of that, and the rest is off by 2^-31 of it.  LPR lanes hold a row, 8 numbers each.
            constexpr int LPR = HD / 8, RPT = LPR / 2;          // 256 threads take 512 / LPR .. rows of a tile each
            const int ld_c = tid % LPR, ld_r0 = tid / LPR * RPT;
#pragma unroll 1
            for (int xt = 0; xt < (HALVES ? 1 : 2); ++xt) {
                uint4 v[RPT];
                int tok = (t.row0 + xt * BM + ld_r0) / t.G, head = (t.row0 + xt * BM + ld_r0) - tok * t.G;
#pragma unroll
                for (int j = 0; j < RPT; ++j) {
                    v[j] = make_uint4(0, 0, 0, 0);
                    if (xt * BM + ld_r0 + j < t.rows)
                        v[j] = *reinterpret_cast<const uint4 *>((const __nv_bfloat16 *)p.q + ((size_t)(t.tok_begin + tok) * p.nq + kvh * t.G + head) * HD + 8 * ld_c);
                    if (++head == t.G) head = 0, ++tok;
                }
#pragma unroll
                for (int j = 0; j < RPT; ++j) {
                    const uint32_t u[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
                    uint32_t big = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) big = max(big, max(u[e] & 0x7fffu, (u[e] >> 16) & 0x7fffu));
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
                    const int e = (int)(big >> 7);              // biased exponent of the largest; 255: not finite, as it is
                    const int up = big == 0 || e == 255 ? 0 : 127 + 6 - max(e, 63);      // (below 2^-64 nothing weighs)
                    const float f = __uint_as_float((uint32_t)(127 + up) << 23);
                    uint32_t h[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) h[k] = pack_f16(__uint_as_float(u[k] << 16) * f, __uint_as_float(u[k] & 0xffff0000u) * f);
                    sts128(base + L::Q + xt * L::TILE + (ld_c >> 3) * L::PANEL + swizzle128(ld_r0 + j, ld_c & 7), make_uint4(h[0], h[1], h[2], h[3]));
                    if (ld_c == 0) row_up[xt * BM + ld_r0 + j] = __uint_as_float((uint32_t)(127 - up) << 23);
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(Q_FULL));
            asm volatile("bar.sync 1, 256;" ::: "memory");      // the rows' powers
        }
        const int tile_row = HALVES ? t.row0 : t.row0 + x * BM;
        const int rows_x = x == 0 || HALVES ? rows_a : t.rows - BM;                // rows of this row tile (<= 0: none)
        const int n_tiles_x = x == 0 ? n_tiles_a : HALVES ? n_tiles / 2 : (has_b ? n_tiles : 0);
        const int k_hi_x = x == 0 ? k_hi_a : k_hi;
        const bool row_ok = r < rows_x;
        const int my_pos = row_ok ? t.pos_begin + (tile_row + r) / t.G : -1;
        // the keys that this row sees in this slice: [see_lo, see_hi); a row that is not there sees all, which asks for no mask
        const int see_lo = row_ok ? max(k_first, p.window > 0 ? my_pos - p.window + 1 : 0) : 0, see_hi = row_ok ? min(my_pos + 1, k_hi_x) : 0x7fffffff;
        const float row_scale = fmaxf(row_up[HALVES ? r : x * BM + r] * p.scale * 1.4426950408889634f, Q8_LEAST_FACTOR);
        // warps none of whose 32 rows exist skip the arithmetic
        const bool warp_has_rows = 32 * (warp & 3) < rows_x;
        const uint32_t lane_base = ((uint32_t)(32 * (warp & 3))) << 16;
        const uint32_t s_addr = tmem + lane_base + x * 128, o_addr = tmem + lane_base + L::O + x * 128;
        float m_ref = -INFINITY, l_run = 0.f;       // the reference the output is accumulated against, and the row's sum
        bool ok = true;             // after a wait gave up the loop runs on without waiting, so that the warps still meet

        for (int step = 0; step < n_tiles_x; ++step) {
            const int i = HALVES ? 2 * step + x : step;
            const int kbase = k_lo + i * BN;
            // S_X(i) is done - and with it, in the issuer's order, O_X += P_X V of the step before
            if (ok && !mbar_wait(bar(S_FULL + x), (uint32_t)step & 1u)) { atomicExch(&g_q8t_error, 7); ok = false; }
            if (ok && !mbar_wait(bar(SCALES_FULL + (i & 3)), (uint32_t)(i >> 2) & 1u)) { atomicExch(&g_q8t_error, 10); ok = false; }
            tc_fence_after();
            if (warp_has_rows) {
                const uint4 *scales = reinterpret_cast<const uint4 *>(aligned + L::SCALES) + (i & 3) * BLOCKS;      // (s_k, log2 s_v, 1 / s_v)
                const bool whole = __all_sync(0xffffffffu, kbase >= see_lo && kbase + BN <= see_hi);
                uint32_t a[BN];
#pragma unroll
                for (int c = 0; c < BN; c += 32) ld32(s_addr + c, a + c);
                ld_wait();
                if (!whole) {
                    // keys this row may not see count as minus infinity
                    const int lo = see_lo - kbase, hi = see_hi - kbase;
#pragma unroll
                    for (int c = 0; c < BN; c += 32) {
                        const uint32_t from = lo <= c ? ~0u : lo >= c + 32 ? 0u : ~0u << (lo - c), upto = hi >= c + 32 ? ~0u : hi <= c ? 0u : ~(~0u << (hi - c));
                        const uint32_t seen = from & upto;
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (!(seen & 1u << j)) a[c + j] = 0xff800000u;
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) {
                    const uint4 sc = scales[b];
                    float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < 16; j += 4) {
                        m2[0] = max3(m2[0], __uint_as_float(a[16 * b + j]), __uint_as_float(a[16 * b + j + 1]));
                        m2[1] = max3(m2[1], __uint_as_float(a[16 * b + j + 2]), __uint_as_float(a[16 * b + j + 3]));
                    }
                    mx = fmaxf(mx, fmaf(fmaxf(m2[0], m2[1]), __uint_as_float(sc.x) * row_scale, __uint_as_float(sc.y)));
                }
                float alpha = 1.f;
                if (mx > m_ref + STEP || (m_ref == -INFINITY && mx > -INFINITY)) {
                    if (m_ref != -INFINITY) alpha = exp2_fast(m_ref - mx);
                    m_ref = mx;
                }
                l_run *= alpha;
                const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
                // P over this row's own scores; two blocks are stored while the next are computed
#pragma unroll
                for (int b = 0; b < BLOCKS; b += 2) {
                    uint32_t w[16];
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        const uint4 sc = scales[b + d];
                        const float ck = __uint_as_float(sc.x) * row_scale, shift = __uint_as_float(sc.y) - m_use;
                        const uint64_t scale2 = pack2(ck, ck), shift2 = pack2(shift, shift);
                        uint64_t l2[2] = {0ull, 0ull};
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            float x0, x1;
                            unpack2(fma2(pack2(__uint_as_float(a[16 * (b + d) + 2 * j]), __uint_as_float(a[16 * (b + d) + 2 * j + 1])), scale2, shift2), x0, x1);
                            const float e0 = exp2_fast(x0), e1 = exp2_fast(x1);
                            l2[j & 1] = add2(l2[j & 1], pack2(e0, e1));
                            w[8 * d + j] = pack_f16(e0, e1);
                        }
                        float a0, a1;
                        unpack2(add2(l2[0], l2[1]), a0, a1);
                        if (a0 + a1 != 0.f) l_run = fmaf(a0 + a1, __uint_as_float(sc.z), l_run);      // (nothing seen: whatever the scale is)
                    }
                    st16(s_addr + 8 * b, w);
                }
                if (__any_sync(0xffffffffu, alpha != 1.f)) {
                    // the whole warp walks its rows' outputs; rows whose reference stays are multiplied by one.  O_X is idle: its last
                    // product is done.
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        ld32(o_addr + c, a);
                        ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j) a[j] = __float_as_uint(__uint_as_float(a[j]) * alpha);
                        st16(o_addr + c, a);
                        st16(o_addr + c + 16, a + 16);
                    }
                }
                st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(P_FULL + x));
        }

        // the last product of this row tile
        if (n_tiles_x > 0 && ok && !mbar_wait(bar(PV_DONE + x), (uint32_t)(n_tiles_x - 1) & 1u)) { atomicExch(&g_q8t_error, 9); ok = false; }
        tc_fence_after();
        const bool write = row_ok && ok;
        const size_t qrow = write ? (size_t)(t.tok_begin + (tile_row + r) / t.G) * p.nq + kvh * t.G + (tile_row + r) % t.G : 0;
        // columns [c0, c0 + 32) of the row's output
        auto put = [&](int c0, const uint32_t *o, float inv) {
            if (p.slices > 1) {
                float *po = p.part_o + (qrow * p.slices + slice) * HD + c0;
#pragma unroll
                for (int j = 0; j < 32; j += 4) *reinterpret_cast<uint4 *>(po + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
            } else {
                __nv_bfloat16 *po = (__nv_bfloat16 *)p.out + qrow * HD + c0;
#pragma unroll
                for (int j = 0; j < 32; j += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const __nv_bfloat162 b2 = __floats2bfloat162_rn(__uint_as_float(o[j + 2 * k]) * inv, __uint_as_float(o[j + 2 * k + 1]) * inv);
                        w[k] = *reinterpret_cast<const uint32_t *>(&b2);
                    }
                    *reinterpret_cast<uint4 *>(po + j) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        };
        if (HALVES) {
            // both streams' last products, then the two states of a row as one: the threads of A take the first half of the columns
            const int n_other = x == 0 ? n_tiles / 2 : n_tiles_a;
            if (n_other > 0 && ok && !mbar_wait(bar(PV_DONE + (x ^ 1)), (uint32_t)(n_other - 1) & 1u)) { atomicExch(&g_q8t_error, 9); ok = false; }
            tc_fence_after();
            float m_a = -INFINITY, l_a = 0.f, m_b = -INFINITY, l_b = 0.f;
            if (n_tiles > 0) {
                float2 *meet = reinterpret_cast<float2 *>(aligned + L::Q);          // Q's memory: every product that read it is done
                meet[x * 128 + r] = make_float2(m_ref, l_run);
                asm volatile("bar.sync 1, 256;" ::: "memory");
                m_a = meet[r].x, l_a = meet[r].y, m_b = meet[128 + r].x, l_b = meet[128 + r].y;
            }
            const float m = fmaxf(m_a, m_b), f_a = m_a == -INFINITY ? 0.f : exp2_fast(m_a - m), f_b = m_b == -INFINITY ? 0.f : exp2_fast(m_b - m);
            // (a sum that is no number stays that)
            const float l = (f_a == 0.f && l_a == l_a ? 0.f : l_a * f_a) + (f_b == 0.f && l_b == l_b ? 0.f : l_b * f_b);
            if (warp_has_rows) {
#pragma unroll 1
                for (int c = 0; c < HD / 2; c += 32) {
                    const int c0 = x * (HD / 2) + c;
                    uint32_t oa[32], ob[32];
                    ld32(tmem + lane_base + L::O + c0, oa);             // warp-wide, whatever rows exist
                    ld32(tmem + lane_base + L::O + 128 + c0, ob);
                    ld_wait();
                    if (!write) continue;
                    // a stream without a tile has left its columns as they were: not a number, perhaps
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        oa[j] = __float_as_uint((n_tiles > 0 ? __uint_as_float(oa[j]) * f_a : 0.f) + (n_tiles > 1 ? __uint_as_float(ob[j]) * f_b : 0.f));
                    put(c0, oa, 1.0f / l);
                }
                if (write && p.slices > 1 && x == 0) *reinterpret_cast<float2 *>(p.part_ml + (qrow * p.slices + slice) * 2) = make_float2(m, l);
            }
        } else if (warp_has_rows) {
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                if (n_tiles_x > 0) {
                    ld32(o_addr + c, o);                // warp-wide, whatever rows exist
                    ld_wait();
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0u;
                }
                if (write) put(c, o, 1.0f / l_run);
            }
            if (write && p.slices > 1) *reinterpret_cast<float2 *>(p.part_ml + (qrow * p.slices + slice) * 2) = make_float2(m_ref, l_run);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::TMEM_COLS) : "memory");
    }
}

template <int HD, bool HALVES>
int launch_tc(const Q8Params &p, int tiles, cudaStream_t stream) {
    constexpr int smem = Lay<HD, HALVES>::BYTES + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    // the registers dealt out inside are those of the launch: with fewer the softmax groups would wait for the difference
    static const int regs = [] {
        cudaFuncAttributes a;
        return cudaFuncGetAttributes(&a, attention_q8_tc_kernel<HD, HALVES>) == cudaSuccess ? a.numRegs : 0;
    }();
    KESTREL_REQUIRE(regs * THREADS >= 256 * SOFTMAX_REGS + 384 * OTHER_REGS, "attention_q8: the kernel was built with %d registers a thread, %d are dealt out", regs,
                    (256 * SOFTMAX_REGS + 384 * OTHER_REGS) / THREADS);
    if (cudaFuncSetAttribute(attention_q8_tc_kernel<HD, HALVES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return kestrel_fail(-3, "attention_q8: cannot raise the shared-memory limit: %s", cudaGetErrorString(cudaGetLastError()));
    kestrel_launch(attention_q8_tc_kernel<HD, HALVES>, dim3((unsigned)tiles * p.nkv, 1, p.slices), dim3(THREADS), smem, stream, p);
    return kestrel_check_launch("attention_q8 tc");
}

}  // namespace

int q8_launch_tc(const Q8Params &p, int tiles, cudaStream_t stream) {
    if (p.rows_per_tile <= BM) return p.hd == 64 ? launch_tc<64, true>(p, tiles, stream) : launch_tc<128, true>(p, tiles, stream);
    return p.hd == 64 ? launch_tc<64, false>(p, tiles, stream) : launch_tc<128, false>(p, tiles, stream);
}

int q8_tc_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_q8t_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_q8t_error, &zero, sizeof(int));
    return v;
}
