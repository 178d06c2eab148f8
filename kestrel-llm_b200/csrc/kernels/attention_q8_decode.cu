// Attention over pages of int8 codes with few rows: single tokens, and the ragged ends of short portions.  Head sizes 64 and 128, bfloat16
// queries.  Formulas in attention_q8.cuh.
//
// A CTA takes up to 16 (token, query head) rows of one (request, kv head) and one slice of their keys.  A loader warp brings tiles of 64
// keys by TMA into a ring of stages, codes of K and V side by side, and the scales of their four blocks beside them; four consumer warps
// take one block of 16 keys each.  Codes go from shared memory straight into the fragments of mma.sync.m16n8k16 (float16, float32 sums):
// a code c is the low byte of the float16 number 1024 + (c + 128), made by a byte permutation and freed of 1152 by one subtraction of
// pairs.  The order of a product's inner index is free as long as both operands share it, which is used twice: a thread's 16 neighbouring
// dimensions of a key are one 16-byte load and four k-steps of the scores, and the columns of the scores stand for keys in an order that
// lets every load of a warp touch each bank once.  Bound by HBM: 2 hd bytes a key and kv head; about one instruction a code to widen it.
//
// Slices are merged through scratch by attention_q8_merge_kernel.
#include "attention_q8.cuh"
#include "tcgen05.cuh"

#include <math.h>

__device__ int g_q8d_error = 0;

namespace {

constexpr int THREADS = 160, BN = 64;       // four consumer warps and the loader; keys of a tile
constexpr uint32_t MAGIC = 0x64646464u;     // high byte of the float16 numbers 1024 .. 1279

template <int HD> struct Ring {
    static constexpr int STAGES = HD == 128 ? 6 : 8;
    static constexpr uint32_t PLANE = BN * HD, STAGE = 2 * PLANE;
    static constexpr uint32_t SCALES = STAGES * STAGE, BARS = SCALES + STAGES * 32, BYTES = BARS + 16 * STAGES;
    static constexpr int LDO = HD + 4;      // row of a warp's outputs, in floats, when the four warps meet
};

__device__ __forceinline__ uint32_t hsub2(uint32_t a) {             // - 1152 from both halves
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(0x64806480u));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma_f16(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}

// Key, among the eight of a column tile, that column n of the scores stands for.  A tile's lines of 128 bytes are swizzled as TMA writes
// them: 16-byte chunk c of line i lies at c ^ (i % 8).  Head size 128: a key is a line; eight lanes of a 16-byte load hold columns
// 2 i and 2 i + 1, whose keys are four lines apart, so that their chunks fall into different halves of the banks; the values' loads of
// sixteen lanes hold the even (or odd) columns, which are neighbouring keys.  Head size 64: a line is two keys.
template <int HD> __device__ __forceinline__ int key_of_column(int n) { return HD == 128 ? (n >> 1) + 4 * (n & 1) : n ^ ((n >> 1) & 1); }

// address of 16-byte chunk c (of HD / 16) of key k in a tile
template <int HD> __device__ __forceinline__ uint32_t chunk_at(uint32_t tile, int k, int c) {
    const int line = HD == 128 ? k : k >> 1, at = HD == 128 ? c : 4 * (k & 1) + c;
    return tile + line * 128 + ((at ^ (line & 7)) << 4);
}

template <int HD>
__global__ void __launch_bounds__(THREADS)
attention_q8_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Q8Params p) {
    pdl_launch_dependents();
    using R = Ring<HD>;
    constexpr int KS = HD / 16, HALVES = HD / 64, NT_O = HD / 8;
    extern __shared__ uint8_t q8d_smem[];
    const uint32_t base = (smem_u32(q8d_smem) + 1023u) & ~1023u;
    uint8_t *ring = q8d_smem + (base - smem_u32(q8d_smem));
    auto full_bar = [&](int s) { return base + R::BARS + 8u * s; };
    auto empty_bar = [&](int s) { return base + R::BARS + 8u * (R::STAGES + s); };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y, slice = blockIdx.z;
    if (tid == 0) {
        // a stage is full when its codes are there (the loader's bytes) and eight lanes' scales
        for (int s = 0; s < R::STAGES; ++s) { mbar_init(full_bar(s), 1 + 8); mbar_init(empty_bar(s), 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    Q8Tile t;
    // the step's description was on the device before the kernel in front of this one began
    if (!q8_find_tile(p, blockIdx.x, t)) { pdl_wait(); return; }
    int lo, hi;
    q8_slice(t, p.slices, slice, BN, lo, hi);
    const int kb0 = lo / BN * BN, n_tiles = hi > lo ? (hi - kb0 + BN - 1) / BN : 0;

    if (warp == 4) {
        // ---- loader: lane l brings the l-th box of a tile, K and V; lanes 0-3 (4-7) bring its blocks' scales of K (V)
        const int box = p.page_size % 64 == 0 ? 64 : p.page_size % 32 == 0 ? 32 : 16, boxes = BN / box;
        const float *scales = lane < 4 ? p.ks : p.vs;
        pdl_wait();
        for (int i = 0; i < n_tiles; ++i) {
            const int stage = i % R::STAGES, kb = kb0 + i * BN;
            const long long box_row = lane < boxes ? q8_row_of(p, t.table, kvh, kb + lane * box) : 0;
            const long long block_row = lane < 8 ? q8_row_of(p, t.table, kvh, kb + (lane & 3) * Q8_BLOCK) : 0;
            if (!mbar_wait(empty_bar(stage), (uint32_t)(i / R::STAGES + 1) & 1u)) { atomicExch(&g_q8d_error, 1); break; }
            if (lane == 0) mbar_expect_tx(full_bar(stage), R::STAGE);
            __syncwarp();
            if (lane < boxes) {
                const uint32_t dst = base + stage * R::STAGE + lane * box * HD;
                const int line = (int)(HD == 128 ? box_row : box_row >> 1);
                tma_load_2d(dst, &map_k, full_bar(stage), 0, line);
                tma_load_2d(dst + R::PLANE, &map_v, full_bar(stage), 0, line);
            }
            if (lane < 8) {
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(base + R::SCALES + stage * 32 + lane * 4), "l"(scales + block_row / Q8_BLOCK) : "memory");
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full_bar(stage)) : "memory");
            }
        }
        return;
    }

    // ---- consumers
    const int g = lane >> 2, c = lane & 3;              // rows g and g + 8; a quarter of the inner index
    pdl_wait();
    // Queries as fragments, in float16: a row is multiplied by the power of two that brings its largest number to [64, 128), so that a
    // bfloat16 number keeps its bits down to 2^-21 of that, and the rest is off by 2^-31 of it.
    uint32_t qa[KS][4];
    float row_scale[2];
    int pos[2], low[2], min_pos = 0x7fffffff;           // (of the rows that are there)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
        const bool live = r < t.rows;
        uint4 w[HALVES][2];
        uint32_t big = 0;
#pragma unroll
        for (int j = 0; j < HALVES; ++j) {
            w[j][0] = w[j][1] = make_uint4(0, 0, 0, 0);
            if (live) {
                const uint4 *src = reinterpret_cast<const uint4 *>((const __nv_bfloat16 *)p.q + q8_out_row(p, t, kvh, r) * HD + 64 * j + 16 * c);
                w[j][0] = src[0];
                w[j][1] = src[1];
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const uint32_t *u = reinterpret_cast<const uint32_t *>(&w[j][k]);
#pragma unroll
                for (int e = 0; e < 4; ++e) big = max(big, max(u[e] & 0x7fffu, (u[e] >> 16) & 0x7fffu));
            }
        }
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const int e = (int)(big >> 7);                  // biased exponent of the largest; 255: not finite, as it is
        const int up = big == 0 || e == 255 ? 0 : 127 + 6 - max(e, 27);
        const float f = __uint_as_float((uint32_t)(127 + up) << 23);
        row_scale[i] = __uint_as_float((uint32_t)(127 - up) << 23) * p.scale * 1.4426950408889634f;
#pragma unroll
        for (int j = 0; j < HALVES; ++j)
#pragma unroll
            for (int k = 0; k < 4; ++k) {               // k-step 4 j + k: dimensions 64 j + 16 c + 4 k ..
                const uint32_t a = reinterpret_cast<const uint32_t *>(&w[j][k >> 1])[2 * (k & 1)], b = reinterpret_cast<const uint32_t *>(&w[j][k >> 1])[2 * (k & 1) + 1];
                qa[4 * j + k][i] = pack_f16(__uint_as_float(a << 16) * f, __uint_as_float(a & 0xffff0000u) * f);
                qa[4 * j + k][2 + i] = pack_f16(__uint_as_float(b << 16) * f, __uint_as_float(b & 0xffff0000u) * f);
            }
        pos[i] = live ? t.pos_begin + (t.row0 + r) / t.G : -1;
        low[i] = p.window > 0 ? max(0, pos[i] - p.window + 1) : 0;
        if (live) min_pos = min(min_pos, pos[i]);
    }
    int max_low = max(low[0], low[1]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        min_pos = min(min_pos, __shfl_xor_sync(0xffffffffu, min_pos, o));
        max_low = max(max_low, __shfl_xor_sync(0xffffffffu, max_low, o));
    }
    float o[NT_O][4];
#pragma unroll
    for (int i = 0; i < NT_O; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    bool ok = true;             // after a wait gave up the loop runs on without waiting, so that the warps still meet below

    for (int i = 0; i < n_tiles; ++i) {
        const int stage = i % R::STAGES;
        if (ok && !mbar_wait(full_bar(stage), (uint32_t)(i / R::STAGES) & 1u)) { atomicExch(&g_q8d_error, 2); ok = false; }
        const int kbase = kb0 + i * BN + 16 * warp;     // this warp's block
        if (ok && kbase < hi && kbase + 16 > lo) {
            const uint32_t Kt = base + stage * R::STAGE, Vt = Kt + R::PLANE;
            float s[2][4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
                s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
                const int key = 16 * warp + 8 * nt + key_of_column<HD>(g);
#pragma unroll
                for (int j = 0; j < HALVES; ++j) {
                    const uint4 w = lds128(chunk_at<HD>(Kt, key, 4 * j + c));
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t x = u[k] ^ 0x80808080u;
                        mma_f16(s[nt], qa[4 * j + k], hsub2(__byte_perm(x, MAGIC, 0x4140)), hsub2(__byte_perm(x, MAGIC, 0x4342)));
                    }
                }
            }
            const float *sc = reinterpret_cast<const float *>(ring + R::SCALES + stage * 32);
            const float sk = sc[warp], sv = sc[4 + warp];
            const float lv = __log2f(sv), rv = 1.0f / sv;
            // scores with the value's scale in base-2 units, the mask where some row does not see the block whole, running reference
            const bool whole = kbase >= lo && kbase + 16 <= hi && kbase + 15 <= min_pos && kbase >= max_low;
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = fmaf(s[nt][e], sk * row_scale[e >> 1], lv);
                    if (!whole) {
                        const int key = kbase + 8 * nt + key_of_column<HD>(2 * c + (e & 1));
                        if (!(key <= pos[e >> 1] && key >= low[e >> 1] && key < hi && key >= lo)) x = -INFINITY;
                    }
                    s[nt][e] = x;
                    mx[e >> 1] = fmaxf(mx[e >> 1], x);
                }
            float use[2], alpha[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                alpha[r] = 1.f;
                // the reference moves once the maximum has outgrown it by 8: weights stay below 2^8
                if (mx[r] > m[r] + 8.f || (m[r] == -INFINITY && mx[r] > -INFINITY)) {
                    alpha[r] = m[r] == -INFINITY ? 0.f : exp2_fast(m[r] - mx[r]);
                    m[r] = mx[r];
                }
                use[r] = m[r] == -INFINITY ? 0.f : m[r];
            }
            if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
                l[0] *= alpha[0];
                l[1] *= alpha[1];
#pragma unroll
                for (int nt = 0; nt < NT_O; ++nt) {
                    o[nt][0] *= alpha[0]; o[nt][1] *= alpha[0];
                    o[nt][2] *= alpha[1]; o[nt][3] *= alpha[1];
                }
            }
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[nt][e] = exp2_fast(s[nt][e] - use[e >> 1]);
                    sum[e >> 1] += s[nt][e];
                }
            // a block of which a row sees nothing adds nothing to its sum, whatever its scale is; a maximum passes over what is no number
#pragma unroll
            for (int r = 0; r < 2; ++r)
                if (mx[r] > -INFINITY || sum[r] != sum[r]) l[r] = fmaf(sum[r], rv, l[r]);
            // out += w V: columns 2 c, 2 c + 1 of both score tiles are the four keys of this thread's fragments
            const uint32_t a[4] = {pack_f16(s[0][0], s[0][1]), pack_f16(s[0][2], s[0][3]), pack_f16(s[1][0], s[1][1]), pack_f16(s[1][2], s[1][3])};
            const int ka = 16 * warp + key_of_column<HD>(2 * c), kb = 16 * warp + key_of_column<HD>(2 * c + 1);
            uint32_t v[4][HD / 32];
            if (HD == 128) {
                const int ch = (g >> 1) + 4 * (g & 1);  // this thread's 16 dimensions: 16 ch ..
                *reinterpret_cast<uint4 *>(v[0]) = lds128(chunk_at<HD>(Vt, ka, ch));
                *reinterpret_cast<uint4 *>(v[1]) = lds128(chunk_at<HD>(Vt, kb, ch));
                *reinterpret_cast<uint4 *>(v[2]) = lds128(chunk_at<HD>(Vt, ka + 8, ch));
                *reinterpret_cast<uint4 *>(v[3]) = lds128(chunk_at<HD>(Vt, kb + 8, ch));
            } else {                                    // its 8 dimensions: 8 g ..
                *reinterpret_cast<uint2 *>(v[0]) = lds64(chunk_at<HD>(Vt, ka, g >> 1) + 8 * (g & 1));
                *reinterpret_cast<uint2 *>(v[1]) = lds64(chunk_at<HD>(Vt, kb, g >> 1) + 8 * (g & 1));
                *reinterpret_cast<uint2 *>(v[2]) = lds64(chunk_at<HD>(Vt, ka + 8, g >> 1) + 8 * (g & 1));
                *reinterpret_cast<uint2 *>(v[3]) = lds64(chunk_at<HD>(Vt, kb + 8, g >> 1) + 8 * (g & 1));
            }
#pragma unroll
            for (int k = 0; k < HD / 32; ++k) {         // output column tiles 4 k .. 4 k + 3: dimensions 4 k .. 4 k + 3 of the thread's
                const uint32_t p0 = __byte_perm(v[0][k], v[1][k], 0x5140) ^ 0x80808080u, p1 = __byte_perm(v[0][k], v[1][k], 0x7362) ^ 0x80808080u;
                const uint32_t p2 = __byte_perm(v[2][k], v[3][k], 0x5140) ^ 0x80808080u, p3 = __byte_perm(v[2][k], v[3][k], 0x7362) ^ 0x80808080u;
                mma_f16(o[4 * k], a, hsub2(__byte_perm(p0, MAGIC, 0x4140)), hsub2(__byte_perm(p2, MAGIC, 0x4140)));
                mma_f16(o[4 * k + 1], a, hsub2(__byte_perm(p0, MAGIC, 0x4342)), hsub2(__byte_perm(p2, MAGIC, 0x4342)));
                mma_f16(o[4 * k + 2], a, hsub2(__byte_perm(p1, MAGIC, 0x4140)), hsub2(__byte_perm(p3, MAGIC, 0x4140)));
                mma_f16(o[4 * k + 3], a, hsub2(__byte_perm(p1, MAGIC, 0x4342)), hsub2(__byte_perm(p3, MAGIC, 0x4342)));
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_bar(stage));
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }

    // the four warps' states, in warp order, in the ring's memory: every tile that was fetched has been consumed
    asm volatile("bar.sync 1, 128;" ::: "memory");
    float *mo = reinterpret_cast<float *>(ring);                // [4][16][LDO]
    float *mml = mo + 4 * 16 * R::LDO;                          // [4][16][2]
    // column n of output tile j is dimension j of thread n's: 2 c -> chunk c, 2 c + 1 -> chunk c + 4 (head size 64: 8 dimensions each)
    const int d0 = HD == 128 ? 16 * c : 16 * c, d1 = HD == 128 ? 64 + 16 * c : 16 * c + 8;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        float *row = mo + (warp * 16 + g + 8 * r) * R::LDO;
#pragma unroll
        for (int j = 0; j < NT_O; j += 4) {
            *reinterpret_cast<float4 *>(row + d0 + j) = make_float4(o[j][2 * r], o[j + 1][2 * r], o[j + 2][2 * r], o[j + 3][2 * r]);
            *reinterpret_cast<float4 *>(row + d1 + j) = make_float4(o[j][2 * r + 1], o[j + 1][2 * r + 1], o[j + 2][2 * r + 1], o[j + 3][2 * r + 1]);
        }
        if (c == 0) {
            mml[(warp * 16 + g + 8 * r) * 2] = m[r];
            mml[(warp * 16 + g + 8 * r) * 2 + 1] = l[r];
        }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    for (int idx = tid; idx < 16 * (HD / 8); idx += 128) {
        const int r = idx / (HD / 8), d = (idx % (HD / 8)) * 8;
        if (r >= t.rows) continue;
        float M = -INFINITY, L = 0.f, acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, mml[(w * 16 + r) * 2]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float mw = mml[(w * 16 + r) * 2], lw = mml[(w * 16 + r) * 2 + 1];
            const float f = mw == -INFINITY ? 0.f : exp2f(mw - M);
            if (f == 0.f && lw == lw) continue;         // (a sum that is no number stays that)
            L = fmaf(lw, f, L);
            const float4 a = *reinterpret_cast<const float4 *>(mo + (w * 16 + r) * R::LDO + d), b = *reinterpret_cast<const float4 *>(mo + (w * 16 + r) * R::LDO + d + 4);
            acc[0] = fmaf(a.x, f, acc[0]); acc[1] = fmaf(a.y, f, acc[1]); acc[2] = fmaf(a.z, f, acc[2]); acc[3] = fmaf(a.w, f, acc[3]);
            acc[4] = fmaf(b.x, f, acc[4]); acc[5] = fmaf(b.y, f, acc[5]); acc[6] = fmaf(b.z, f, acc[6]); acc[7] = fmaf(b.w, f, acc[7]);
        }
        if (!ok) continue;                              // a wait gave up: nothing is written
        const size_t row = q8_out_row(p, t, kvh, r);
        if (p.slices > 1) {
            float *po = p.part_o + (row * p.slices + slice) * HD + d;
            *reinterpret_cast<float4 *>(po) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            *reinterpret_cast<float4 *>(po + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
            if (d == 0) *reinterpret_cast<float2 *>(p.part_ml + (row * p.slices + slice) * 2) = make_float2(M, L);
        } else {
            const float inv = 1.0f / L;
            __nv_bfloat162 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __floats2bfloat162_rn(acc[2 * j] * inv, acc[2 * j + 1] * inv);
            *reinterpret_cast<uint4 *>((__nv_bfloat16 *)p.out + row * HD + d) = *reinterpret_cast<uint4 *>(w);
        }
    }
}

template <int HD> constexpr size_t decode_smem() { return Ring<HD>::BYTES + 1024; }

template <int HD>
int launch_decode(const Q8Params &p, int tiles, cudaStream_t stream) {
    CUtensorMap mk, mv;
    const long long lines = (long long)p.cache_pages * p.nkv * p.page_size * HD / 128;
    const int box = (p.page_size % 64 == 0 ? 64 : p.page_size % 32 == 0 ? 32 : 16) * HD / 128;
    // two codes as one 16-bit element: the copy moves lines of 128 bytes, whatever they hold
    int rc = kestrel_tensor_map_bf16(&mk, p.k, lines, 64, 64, box);
    if (rc == 0) rc = kestrel_tensor_map_bf16(&mv, p.v, lines, 64, 64, box);
    if (rc) return rc;
    if (cudaFuncSetAttribute(attention_q8_decode_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)decode_smem<HD>()) != cudaSuccess)
        return kestrel_fail(-3, "attention_q8: cannot raise the shared-memory limit: %s", cudaGetErrorString(cudaGetLastError()));
    kestrel_launch(attention_q8_decode_kernel<HD>, dim3(tiles, p.nkv, p.slices), dim3(THREADS), decode_smem<HD>(), stream, mk, mv, p);
    return kestrel_check_launch("attention_q8 decode");
}

}  // namespace

int q8_launch_decode(const Q8Params &p, int tiles, cudaStream_t stream) {
    return p.hd == 64 ? launch_decode<64>(p, tiles, stream) : launch_decode<128>(p, tiles, stream);
}

// CTAs that the SMs hold at once, by shared memory
int q8_decode_slots(int hd) {
    const size_t smem = hd == 64 ? decode_smem<64>() : decode_smem<128>();
    return kestrel_sms() * (int)((227 * 1024) / (smem + 1024));
}

int q8_decode_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_q8d_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_q8d_error, &zero, sizeof(int));
    return v;
}
