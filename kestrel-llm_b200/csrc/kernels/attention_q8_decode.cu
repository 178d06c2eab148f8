// Attention over pages of int8 codes with few rows: single tokens and short portions in bfloat16, and all of float32.  Head sizes 64 and 128.
// Formulas in attention_q8.cuh.
//
// The work is pairs - a kv head and up to 8 or 16 (token, query head) rows of a request - of key tiles of 64.  How CTAs take them
// (q8_decode_cluster has both sides' times):
//   - the CTAs of a cluster of up to 16 share one pair, evenly, and join their parts in each other's shared memory: few, short pairs;
//   - a CTA a pair, late rows first, more CTAs than there is room for: many pairs, none long;
//   - stretches: all key tiles of all pairs stand in one line, and every CTA takes as many of them as the next, whatever the requests' lengths.
//     A CTA walks its stretch pair by pair.  A pair that lies within one CTA's stretch is finished there; the others leave (maximum, sum,
//     outputs) of their parts in scratch, two parts a CTA at most, and the join kernel below adds them in the order of the keys.
//
// A loader warp brings tiles by cp.async into a ring of stages, codes of K and V side by side in lines of 128 bytes, swizzled so that lines
// meet in all banks, and the scales of their four blocks beside them, running ahead over the pairs' borders; four consumer warps take one
// block of 16 keys each.  (Tiles by TMA, a copy a page and plane, are no faster with pages of 64 and slower with pages of 16, whose copies
// are of 2,048 bytes: 256 requests behind 1,000 keys 102 us, 109 by TMA.)  Codes go from shared memory straight
// into the fragments of mma.sync.m16n8k16 (float16, float32 sums), as the operand of sixteen rows: 16 keys by 8 query rows of scores,
// 16 dimensions by 8 query rows of outputs, so that four heads a group leave half of a product unused and not three quarters, and a
// thread's softmax holds four scores.  The weights change places between the two products by transposing 8 by 8 tiles.  A code of V is the
// low byte of the float16 number 1024 + (c + 128), made by a byte permutation and freed of 1152 by one subtraction of pairs.  A code of K
// is the float16 number (c + 128) 2^-24, a subnormal one, which the permutation alone makes; the scores' sums begin with -128 2^-24 times
// the row's sum of queries instead of zero.  (The same for V would leave 128 times the weights' sum in the outputs, of which they are a
// hundredth where many keys weigh alike.)  The order of a product's inner index is free as long as both operands share it, which is used
// twice: a thread's 16 neighbouring dimensions of a key are one 16-byte load and four k-steps of the scores, and the columns of the scores
// stand for keys in an order that lets every load of a warp touch each bank once.
//
// float32: a query and a weight are two float16 parts each, which leave 2^-22 of it or, of a row's small ones, 2^-31 of the largest query and
// 2^-39 of the largest weight.  (A third part would leave less than float32 itself.  Outputs are off by 5.9e-8 of their norm with one key, 2.2e-7
// on random data and 3.5e-7 where scores reach tens; with three parts by 4.7e-8, 2.1e-7 and 2.1e-7, in PyTorch's float32 operations by 5.5e-7 on
// random data; and 64 requests behind 4,095 keys take 148 us, 168 with three parts, with heads of 64 105 and 111.)  Products with codes are exact.
// The matrix instructions cut their sums off instead of rounding them, so every k-step begins at zero, smaller part first, and is added in
// float32.  Codes of K are freed of their 1152 like those of V here.
//
// Bound by HBM with bfloat16: 2 hd bytes a key and kv head; some 0.6 instructions a code to widen it.  32 / 8 heads of 128: 64 requests
// behind up to 4,095 keys (407 MB) 80 us, 5.1 TB/s; two behind 65,535 (235 MB) 49 us, 4.8 TB/s; one behind 1,003 6.3 us, of which latency
// is nearly all; with a head size of 64, where a tile has half the bytes and the same softmax, 64 behind up to 4,095 55 us, 3.7 TB/s.
// float32: 64 behind 3,000 115 us, 3.5 TB/s, and 411 tokens of two requests, 16 / 4 heads, 20 us (CUDA cores: 39).
#include "attention_q8.cuh"
#include "tcgen05.cuh"

#include "device_table.h"

#include <cuda_fp16.h>
#include <math.h>
#include <type_traits>

__device__ int g_q8d_error = 0;

namespace {

constexpr int THREADS = 160, BN = 64, MAX_CLUSTER = 16;     // four consumer warps and the loader; keys of a tile
constexpr uint32_t MAGIC = 0x64646464u;     // high byte of the float16 numbers 1024 .. 1279

// NT: column tiles of eight rows.  One: three CTAs an SM; two, or one of float32: two.
template <int HD, int NT, typename T> struct Ring {
    static constexpr bool THREE = NT == 1 && sizeof(T) == 2;
    static constexpr int STAGES = (THREE ? 3 : 4) * (128 / HD), CTAS = THREE ? 3 : 2;
    static constexpr int LDO = HD + 4;      // row of a warp's outputs, in floats, when the four warps meet
    static constexpr uint32_t PLANE = BN * HD, STAGE = 2 * PLANE;
    static constexpr uint32_t SCALES = STAGES * STAGE, BARS = SCALES + STAGES * 32, MEET = BARS + 16 * STAGES, BYTES = MEET + 4 * 8 * NT * (LDO + 2) * 4;
};

template <typename T> constexpr int parts_of() { return sizeof(T) == 4 ? 2 : 1; }

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
__device__ __forceinline__ float log2_fast(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two numbers as pairs of float16 parts, the larger first: two of them leave 2^-22 of a number, or 2^-25
template <int PARTS>
__device__ __forceinline__ void split(float lo, float hi, uint32_t (&part)[PARTS]) {
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        part[i] = pack_f16(lo, hi);
        if (i + 1 == PARTS) break;
        const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&part[i]));
        lo -= x.x;
        hi -= x.y;
    }
}
__device__ __forceinline__ void mma_f16(float *d, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// shared memory of the rank-th CTA of this cluster at this one's address `at`
__device__ __forceinline__ uint32_t in_cluster(uint32_t at, int rank) {
    uint32_t remote;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(rank));
    return remote;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t at) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t at) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t transpose(uint32_t a) {        // of an 8 by 8 tile of 16-bit numbers
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
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

// Key, among the eight of a half tile, that row n of the scores stands for.  A tile's lines of 128 bytes are swizzled:
// 16-byte chunk c of line i lies at c ^ (i % 8).  Head size 128: a key is a line; eight lanes of a 16-byte load hold rows
// 2 i and 2 i + 1, whose keys are four lines apart, so that their chunks fall into different halves of the banks; the values' loads of
// sixteen lanes hold the even (or odd) rows, which are neighbouring keys.  Head size 64: a line is two keys.
template <int HD> __device__ __forceinline__ int key_of_row(int n) { return HD == 128 ? (n >> 1) + 4 * (n & 1) : n ^ ((n >> 1) & 1); }

// address of 16-byte chunk c (of HD / 16) of key k in a tile
template <int HD> __device__ __forceinline__ uint32_t chunk_at(int k, int c) {
    const int line = HD == 128 ? k : k >> 1, at = HD == 128 ? c : 4 * (k & 1) + c;
    return line * 128 + ((at ^ (line & 7)) << 4);
}

// a / b for a >= 0, b > 0: a division of 64 bits takes ten times one of 32
__device__ __forceinline__ long long over(long long a, long long b) { return (a | b) >> 32 ? a / b : (long long)((uint32_t)a / (uint32_t)b); }

// The line of key tiles: request i's pairs lie behind those of the requests before it, kv head by kv head and in these row tile by row tile: the
// first, the last, the second, the last but one, ..., so that neighbours, which see few keys of a prompt and many, weigh together like others.
// All pairs of a request have the tiles that its first or its last row sees.
struct Line {
    const Q8Params &p;

    // key tiles of a pair of request i; sets its row tiles
    __device__ __forceinline__ int tiles_of(int i, int &row_tiles) const {
        row_tiles = 0;
        if (i >= p.nseq) return 0;
        const int n = p.cu_seqlens[i + 1] - p.cu_seqlens[i], kv = p.kv_lens[i];
        const long long rows = (long long)n * (p.nq / p.nkv);
        if (rows <= p.rows_above || rows > p.rows_upto) return 0;
        const int first = p.window > 0 ? max(0, kv - n - p.window + 1) : 0;
        row_tiles = ((int)rows + p.rows_per_tile - 1) / p.rows_per_tile;
        return (kv + BN - 1) / BN - first / BN;
    }
    // of one kv head: below 2^31, which the host sees to
    __device__ __forceinline__ int place_of(int i) const {
        int rt;
        const int n = tiles_of(i, rt);
        return n * rt;
    }
    // all of it
    __device__ __forceinline__ long long length() const {
        int sum = 0;
        for (int i = threadIdx.x & 31; i < p.nseq; i += 32) sum += place_of(i);
        return (long long)__reduce_add_sync(0xffffffffu, sum) * p.nkv;
    }
    // the request in which tile `at` lies, and its first tile's place
    __device__ __forceinline__ int request_at(long long at, long long &begin) const {
        const int lane = threadIdx.x & 31;
        const int want = (int)over(at, p.nkv);      // on one kv head's line a request holds its place
        int before = 0;
        for (int base = 0; base < p.nseq; base += 32) {
            const int n = place_of(base + lane);
            int end = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, end, o);
                if (lane >= o) end += x;
            }
            const uint32_t behind = __ballot_sync(0xffffffffu, want < before + end);
            if (behind) {
                const int l = __ffs(behind) - 1;
                begin = (long long)(before + __shfl_sync(0xffffffffu, end - n, l)) * p.nkv;
                return base + l;
            }
            before += __shfl_sync(0xffffffffu, end, 31);
        }
        begin = 0;
        return -1;
    }
};

// Stretches that the line is cut into: one for every CTA, but of two tiles at least - a recorded launch may meet a shorter line than it was
// made for, and a CTA without tiles would leave its part of a pair unwritten
__device__ __forceinline__ int stretches(long long length, int ctas) { return (int)max(1ll, min((long long)ctas, length / 2)); }
// stretch u begins here; the stretch that holds tile `at`
__device__ __forceinline__ long long stretch(long long u, long long length, int ctas) { return over(u * length, ctas); }
__device__ __forceinline__ int holder(long long at, long long length, int ctas) { return (int)over((at + 1) * ctas - 1, length); }

// The k-th row tile of a request's kv head on the line, and a row tile's place there
__device__ __forceinline__ int nth_row_tile(int k, int row_tiles) { return k & 1 ? row_tiles - 1 - k / 2 : k / 2; }
__device__ __forceinline__ int place_of_row_tile(int rt, int row_tiles) { return 2 * rt < row_tiles ? 2 * rt : 2 * (row_tiles - 1 - rt) + 1; }

// One CTA's parts of pairs, one after the other
struct Walk {
    const Q8Params &p;
    long long at, end, begin;           // next tile, end of the stretch, place of the pair's first tile
    int seq, n, kvh, nth, row0;         // the pair; n: its tiles, nth: its row tile's place, row0: its first row among the request's
    // the part
    int G, row_tiles, all_rows, rows, tok_begin, pos_begin, k_first, k_end, from, to, seen_from, seen_to;
    const int *table;
    bool whole;

    // the rank-th of `ranks` equal parts of a pair
    __device__ __forceinline__ Walk(const Q8Params &p_, int pair, int rank, int ranks) : p(p_), at(0), end(0), begin(0), kvh(pair % p_.nkv) {
        G = p.nq / p.nkv;
        n = 0;
        seq = pair / p.nkv;
        row0 = 0;
        if (p.row_tiles > 1) {          // late row tiles, which see the most keys, come first
            Q8Tile t;
            if (!q8_find_tile(p, p.tiles - 1 - seq, t)) return;
            seq = t.seq;
            row0 = t.row0;
        }
        n = Line{p}.tiles_of(seq, row_tiles);
        if (n == 0) return;
        describe();
        see();
        from = seen_from + (int)((long long)(seen_to - seen_from) * rank / ranks);
        to = seen_from + (int)((long long)(seen_to - seen_from) * (rank + 1) / ranks);
        whole = ranks == 1;
    }
    __device__ __forceinline__ Walk(const Q8Params &p_, long long length) : p(p_), n(0) {
        const int cuts = stretches(length, gridDim.x);
        at = stretch(min((int)blockIdx.x, cuts), length, cuts);
        end = stretch(min((int)blockIdx.x + 1, cuts), length, cuts);
        G = p.nq / p.nkv;
        if (at >= end) return;
        const Line line{p};
        seq = line.request_at(at, begin);
        n = line.tiles_of(seq, row_tiles);
        const int pair = (int)over(at - begin, n);
        begin += (long long)pair * n;
        kvh = pair / row_tiles;
        nth = pair - kvh * row_tiles;
        describe();
    }
    __device__ __forceinline__ void describe() {
        tok_begin = p.cu_seqlens[seq];
        const int n_tok = p.cu_seqlens[seq + 1] - tok_begin;
        k_end = p.kv_lens[seq];
        pos_begin = k_end - n_tok;
        all_rows = n_tok * G;
        k_first = p.window > 0 ? max(0, pos_begin - p.window + 1) : 0;
        table = p.block_table + (size_t)seq * p.table_stride;
    }
    // the pair's rows, and the tiles that some of them see
    __device__ __forceinline__ void see() {
        rows = min(p.rows_per_tile, all_rows - row0);
        const int first = k_first / BN, last_pos = pos_begin + (row0 + rows - 1) / G;
        seen_from = p.window > 0 ? max(0, pos_begin + row0 / G - p.window + 1) / BN - first : 0;
        seen_to = last_pos / BN - first + 1;
    }
    // the next part: tiles [from, to) of the pair; false at the end of the stretch
    __device__ __forceinline__ bool next() {
        if (at >= end) return false;
        if (at >= begin + n) {
            begin += n;
            if (++nth == row_tiles) {
                nth = 0;
                if (++kvh == p.nkv) {
                    kvh = 0;
                    const Line line{p};
                    do n = line.tiles_of(++seq, row_tiles);
                    while (n == 0 && seq < p.nseq);
                    describe();
                }
            }
        }
        row0 = nth_row_tile(nth, row_tiles) * p.rows_per_tile;
        see();
        from = (int)(at - begin);
        to = (int)min((long long)n, end - begin);
        whole = from == 0 && to == n;
        at = begin + to;
        from = max(from, seen_from);
        to = min(to, seen_to);
        return true;
    }
    __device__ __forceinline__ size_t out_row(int r) const { return (size_t)(tok_begin + (row0 + r) / G) * p.nq + kvh * G + (row0 + r) % G; }
};

// Parts in scratch: 16 rows of HD outputs each, then 16 (maximum, sum) pairs each; a CTA's first part is its even one
template <int HD> __device__ __forceinline__ float *part_out(const Q8Params &p, long long part, int row) { return p.part_o + (part * 16 + row) * HD; }
__device__ __forceinline__ float2 *part_ml(const Q8Params &p, long long part, int row) { return reinterpret_cast<float2 *>(p.part_ml) + part * 16 + row; }

// A block's scores s - (key g, rows 2 c and 2 c + 1), (key g + 8, the same) - become weights; the rows' references, sums and outputs follow.
// sk: the keys' scale, lv and rv: log2 and reciprocal of the values', or of its power of two (WIDE).  MASKED: some row does not see the block whole.
template <int NT, bool MASKED, bool WIDE, int NO>
__device__ __forceinline__ void weigh(float (&s)[NT][4], float (&o)[NT][NO][4], float (&m)[NT][2], float (&l)[NT][2], const float (&row_scale)[NT][2], float sk,
                                      float lv, float rv, int kbase, int my_key, const int (&pos)[NT][2], const int (&low)[NT][2]) {
    float mx[NT][2], ck[NT][2];
    bool none[NT][2], grow = false;             // none: rows that see nothing of the block, whatever its scales are
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            none[nt][i] = MASKED && (kbase > pos[nt][i] || kbase + 15 < low[nt][i]);
            if (MASKED) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int key = kbase + my_key + 8 * h;
                    if (!(key <= pos[nt][i] && key >= low[nt][i])) s[nt][2 * h + i] = -INFINITY;
                }
            }
            ck[nt][i] = sk * row_scale[nt][i];
            // in base-2 units, with the value's scale: x = s * ck + lv
            mx[nt][i] = fmaf(fmaxf(s[nt][i], s[nt][2 + i]), ck[nt][i], lv);
            if (MASKED && none[nt][i]) mx[nt][i] = -INFINITY;
            grow |= mx[nt][i] > m[nt][i] + (WIDE ? 0.f : 8.f) || (m[nt][i] == -INFINITY && mx[nt][i] > -INFINITY);
        }
    // The reference moves once the maximum has outgrown it by 8: weights stay below 2^8.  (Float32: with the maximum.)
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) mx[nt][i] = fmaxf(mx[nt][i], __shfl_xor_sync(0xffffffffu, mx[nt][i], x));
                if (mx[nt][i] > m[nt][i]) {
                    const float alpha = m[nt][i] == -INFINITY ? 0.f : WIDE ? exp2f(m[nt][i] - mx[nt][i]) : exp2_fast(m[nt][i] - mx[nt][i]);
                    m[nt][i] = mx[nt][i];
                    l[nt][i] *= alpha;
#pragma unroll
                    for (int j = 0; j < NO; ++j) o[nt][j][i] *= alpha, o[nt][j][2 + i] *= alpha;
                }
            }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            // (float32: times 2^14, so that a weight with its scale's other factor stays below 2^15, and its parts leave no more than 2^-39 of the largest)
            const float shift = lv - (m[nt][i] == -INFINITY ? 0.f : m[nt][i]) + (WIDE ? 14.f : 0.f);
            float &a = s[nt][i], &b = s[nt][2 + i];
            a = WIDE ? exp2f(fmaf(a, ck[nt][i], shift)) : exp2_fast(fmaf(a, ck[nt][i], shift));
            b = WIDE ? exp2f(fmaf(b, ck[nt][i], shift)) : exp2_fast(fmaf(b, ck[nt][i], shift));
            if (MASKED && none[nt][i]) a = b = 0.f;
            else l[nt][i] = fmaf(a + b, rv, l[nt][i]);
        }
}

template <typename T, int HD, int NT, bool CLUSTER>
__global__ void __launch_bounds__(THREADS, Ring<HD, NT, T>::CTAS)
attention_q8_decode_kernel(const Q8Params p) {
    if (CLUSTER) pdl_launch_dependents();               // (stretches let the join kernel in at their end)
    using R = Ring<HD, NT, T>;
    constexpr int KS = HD / 16, HALVES = HD / 64, ROWS = 8 * NT, PARTS = parts_of<T>();
    constexpr bool WIDE = PARTS > 1;
    constexpr uint32_t FIN_ML = ROWS * HD * 4;
    extern __shared__ uint8_t q8d_smem[];
    const uint32_t base = (smem_u32(q8d_smem) + 1023u) & ~1023u;
    uint8_t *ring = q8d_smem + (base - smem_u32(q8d_smem));
    auto full_bar = [&](int s) { return base + R::BARS + 8u * s; };
    auto empty_bar = [&](int s) { return base + R::BARS + 8u * (R::STAGES + s); };
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        // a stage is full when what the loader's lanes have asked for is there
        for (int s = 0; s < R::STAGES; ++s) { mbar_init(full_bar(s), 32); mbar_init(empty_bar(s), 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (!p.described) pdl_wait();
    Walk w = CLUSTER ? Walk(p, (int)blockIdx.x / p.slices, (int)blockIdx.x % p.slices, p.slices) : Walk(p, Line{p}.length());
    int stage = 0;
    uint32_t phase = 0;
    pdl_wait();
    if (CLUSTER && w.n == 0) return;                    // another launch's request, or fewer rows than another's: all of the cluster
    bool more = true;
    auto next = [&] {
        if (!CLUSTER) return w.next();
        const bool now = more;
        more = false;
        return now;
    };

    // eight neighbouring numbers of an output row
    auto store = [&](size_t at, const float *acc, float L) {
        const float inv = 1.0f / L;
        if constexpr (WIDE) {
            *reinterpret_cast<float4 *>((float *)p.out + at) = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
            *reinterpret_cast<float4 *>((float *)p.out + at + 4) = make_float4(acc[4] * inv, acc[5] * inv, acc[6] * inv, acc[7] * inv);
        } else {
            __nv_bfloat162 b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = __floats2bfloat162_rn(acc[2 * j] * inv, acc[2 * j + 1] * inv);
            *reinterpret_cast<uint4 *>((__nv_bfloat16 *)p.out + at) = *reinterpret_cast<uint4 *>(b);
        }
    };

    if (warp == 4) {
        // ---- loader: 512 bytes at a time, sixteen a lane, to where the swizzle wants them; lanes 0-3 (4-7) bring the blocks' scales of K (V)
        constexpr int UNITS = 16 * HD / 512;            // of a block
        const float *scales = lane < 4 ? p.ks : p.vs;
        const int8_t *src_k = p.k + lane * 16, *src_v = p.v + lane * 16;
        const uint32_t to = base + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
        bool ok = true;
        while (ok && next()) {
            const int kb0 = w.k_first / BN * BN;
            for (int i = w.from; i < w.to; ++i) {
                const int kb = kb0 + i * BN;
                const int block_row = lane < 8 ? q8_row_of(p, w.table, w.kvh, kb + (lane & 3) * Q8_BLOCK) : 0;
                if (!mbar_wait(empty_bar(stage), phase ^ 1u)) { atomicExch(&g_q8d_error, 1); ok = false; break; }
#pragma unroll
                for (int b = 0; b < BN / Q8_BLOCK; ++b) {
                    const size_t row = (size_t)__shfl_sync(0xffffffffu, block_row, b) * HD;
#pragma unroll
                    for (int u = 0; u < UNITS; ++u) {
                        // (four lines further on the swizzle turns its third bit)
                        const uint32_t dst = (u & 1 ? to ^ 64u : to) + stage * R::STAGE + b * 16 * HD + u * 512;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src_k + row + u * 512) : "memory");
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + R::PLANE), "l"(src_v + row + u * 512) : "memory");
                    }
                }
                if (lane < 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(base + R::SCALES + stage * 32 + lane * 4), "l"(scales + block_row / Q8_BLOCK) : "memory");
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full_bar(stage)) : "memory");
                if (++stage == R::STAGES) stage = 0, phase ^= 1u;
            }
        }
    } else {

    // ---- consumers
    // a lane (g, c) holds rows g of the first operands, row g of the queries, and of a product keys g and g + 8 for rows 2 c and 2 c + 1
    const int g = lane >> 2, c = lane & 3;
    // where this thread's codes lie in a stage: of K for the block's first eight keys, and of V
    uint32_t k_off[HALVES], v_off[2];
#pragma unroll
    for (int j = 0; j < HALVES; ++j) k_off[j] = warp * 16 * HD + chunk_at<HD>(key_of_row<HD>(g), 4 * j + c);
#pragma unroll
    for (int j = 0; j < 2; ++j)
        v_off[j] = R::PLANE + warp * 16 * HD + chunk_at<HD>(key_of_row<HD>(2 * c + j), HD == 128 ? (g >> 1) + 4 * (g & 1) : g >> 1) + (HD == 64 ? 8 * (g & 1) : 0);
    // the other eight keys: 8 lines further at head size 128, which the swizzle repeats after, 4 at 64, which turn its third bit
    auto second = [](uint32_t at) { return HD == 128 ? at + 1024 : (at + 512) ^ 64u; };
    const int my_key = key_of_row<HD>(g);
    float *meet = reinterpret_cast<float *>(ring + R::MEET), *meet_ml = meet + 4 * ROWS * R::LDO;
    bool ok = true;             // after a wait gave up the loop runs on without waiting, so that the warps still meet below
    bool first_part = true;

    while (next()) {
        // Queries as fragments, in float16: a row is multiplied by the power of two that brings its largest number to [64, 128), so that
        // a bfloat16 number keeps its bits down to 2^-21 of that, and the rest is off by 2^-31 of it.
        // float32: two parts of a number.
        uint32_t qb[PARTS][NT][KS][2];
        float row_scale[NT][2], bias[NT][2];            // of rows 2 c and 2 c + 1
        int pos[NT][2], low[NT][2], min_pos = 0x7fffffff, max_low = 0;      // (the last two of the rows that are there)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = 8 * nt + g;
            constexpr int VECS = WIDE ? 4 : 2;
            uint4 q[HALVES][VECS];
            uint32_t big = 0;
#pragma unroll
            for (int j = 0; j < HALVES; ++j) {
#pragma unroll
                for (int k = 0; k < VECS; ++k) q[j][k] = make_uint4(0, 0, 0, 0);
                if (r < w.rows) {
                    const uint4 *src = reinterpret_cast<const uint4 *>((const T *)p.q + w.out_row(r) * HD + 64 * j + 16 * c);
#pragma unroll
                    for (int k = 0; k < VECS; ++k) q[j][k] = src[k];
                }
#pragma unroll
                for (int k = 0; k < VECS; ++k) {
                    const uint32_t *u = reinterpret_cast<const uint32_t *>(&q[j][k]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) big = max(big, WIDE ? u[e] & 0x7fffffffu : max(u[e] & 0x7fffu, (u[e] >> 16) & 0x7fffu));
                }
            }
            big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
            const int e = (int)(big >> (WIDE ? 23 : 7));         // biased exponent of the largest; 255: not finite, as it is
            const int up = big == 0 || e == 255 ? 0 : 127 + 6 - max(e, 63);      // (below 2^-64 nothing weighs)
            const float f = __uint_as_float((uint32_t)(127 + up) << 23);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < HALVES; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {           // k-step 4 j + k: dimensions 64 j + 16 c + 4 k ..
                    uint32_t x[PARTS], y[PARTS];
                    if constexpr (WIDE) {
                        split<PARTS>(__uint_as_float(q[j][k].x) * f, __uint_as_float(q[j][k].y) * f, x);
                        split<PARTS>(__uint_as_float(q[j][k].z) * f, __uint_as_float(q[j][k].w) * f, y);
                    } else {
                        const uint32_t a = reinterpret_cast<const uint32_t *>(&q[j][k >> 1])[2 * (k & 1)], b = reinterpret_cast<const uint32_t *>(&q[j][k >> 1])[2 * (k & 1) + 1];
                        x[0] = pack_f16(__uint_as_float(a << 16) * f, __uint_as_float(a & 0xffff0000u) * f);
                        y[0] = pack_f16(__uint_as_float(b << 16) * f, __uint_as_float(b & 0xffff0000u) * f);
                        const float2 fx = __half22float2(*reinterpret_cast<const __half2 *>(x)), fy = __half22float2(*reinterpret_cast<const __half2 *>(y));
                        sum += (fx.x + fx.y) + (fy.x + fy.y);
                    }
#pragma unroll
                    for (int i = 0; i < PARTS; ++i) {
                        qb[i][nt][4 * j + k][0] = x[i];
                        qb[i][nt][4 * j + k][1] = y[i];
                    }
                }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const float scale_g = fmaxf(__uint_as_float((uint32_t)(127 - up) << 23) * p.scale * (1.4426950408889634f * (WIDE ? 1.0f : 16777216.0f)), Q8_LEAST_FACTOR);
            const float bias_g = WIDE ? 0.f : sum * (-128.0f / 16777216.0f);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                row_scale[nt][i] = __shfl_sync(0xffffffffu, scale_g, 8 * c + 4 * i);
                bias[nt][i] = __shfl_sync(0xffffffffu, bias_g, 8 * c + 4 * i);
                const int row = 8 * nt + 2 * c + i;
                const bool live = row < w.rows;
                pos[nt][i] = live ? w.pos_begin + (w.row0 + row) / w.G : -1;
                low[nt][i] = p.window > 0 ? max(0, pos[nt][i] - p.window + 1) : 0;
                if (live) min_pos = min(min_pos, pos[nt][i]);
                max_low = max(max_low, low[nt][i]);
            }
        }
        min_pos = min(min_pos, __shfl_xor_sync(0xffffffffu, min_pos, 1));
        min_pos = min(min_pos, __shfl_xor_sync(0xffffffffu, min_pos, 2));
        max_low = max(max_low, __shfl_xor_sync(0xffffffffu, max_low, 1));
        max_low = max(max_low, __shfl_xor_sync(0xffffffffu, max_low, 2));
        float o[NT][HD / 16][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < HD / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }
        const int k_begin = w.k_first / BN * BN;

        for (int i = w.from; i < w.to; ++i) {
            if (ok && !mbar_wait(full_bar(stage), phase)) { atomicExch(&g_q8d_error, 2); ok = false; }
            const int kbase = k_begin + i * BN + 16 * warp;     // this warp's block
            if (ok && kbase < w.k_end && kbase + 16 > w.k_first) {
                const uint32_t at = base + stage * R::STAGE;
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    s[nt][0] = s[nt][2] = bias[nt][0];
                    s[nt][1] = s[nt][3] = bias[nt][1];
                }
#pragma unroll
                for (int j = 0; j < HALVES; ++j) {
                    const uint4 w0 = lds128(at + k_off[j]), w1 = lds128(at + second(k_off[j]));
                    const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t x0 = u0[k] ^ 0x80808080u, x1 = u1[k] ^ 0x80808080u;
                        if constexpr (WIDE) {
                            // small parts first, and every k-step from zero: the unit's sums are cut off rather than rounded
                            const uint32_t a[4] = {hsub2(__byte_perm(x0, MAGIC, 0x4140)), hsub2(__byte_perm(x1, MAGIC, 0x4140)),
                                                   hsub2(__byte_perm(x0, MAGIC, 0x4342)), hsub2(__byte_perm(x1, MAGIC, 0x4342))};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                                for (int i = PARTS - 1; i >= 0; --i) mma_f16(t, a, qb[i][nt][4 * j + k][0], qb[i][nt][4 * j + k][1]);
#pragma unroll
                                for (int i = 0; i < 4; ++i) s[nt][i] += t[i];
                            }
                        } else {
                            const uint32_t a[4] = {__byte_perm(x0, 0, 0x4140), __byte_perm(x1, 0, 0x4140), __byte_perm(x0, 0, 0x4342), __byte_perm(x1, 0, 0x4342)};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma_f16(s[nt], a, qb[0][nt][4 * j + k][0], qb[0][nt][4 * j + k][1]);
                        }
                    }
                }
                const float *sc = reinterpret_cast<const float *>(ring + R::SCALES + stage * 32);
                // (what is no number stays that)
                const float sk = sc[warp] < Q8_LEAST_SCALE ? Q8_LEAST_SCALE : sc[warp], sv = sc[4 + warp] < Q8_LEAST_SCALE ? Q8_LEAST_SCALE : sc[4 + warp];
                // float32: the values' scale is a power of two, which is exact as a logarithm, and a factor in [1, 2) on the weights
                const bool number = sv <= 3.4e38f;
                const float rv = WIDE ? 1.0f / __uint_as_float(__float_as_uint(sv) & 0x7f800000u) : rcp_fast(sv);
                const float lv = !WIDE ? log2_fast(sv) : number ? (float)((int)(__float_as_uint(sv) >> 23) - 127) : __uint_as_float(0x7fc00000u);
                if (kbase >= w.k_first && kbase + 16 <= w.k_end && kbase + 15 <= min_pos && kbase >= max_low) {
                    weigh<NT, false, WIDE>(s, o, m, l, row_scale, sk, lv, rv, kbase, my_key, pos, low);
                } else {
                    weigh<NT, true, WIDE>(s, o, m, l, row_scale, sk, lv, rv, kbase, my_key, pos, low);
                }
                // out += w V: the transposed weights' pairs are keys 2 c, 2 c + 1 of both halves
                uint32_t b[PARTS][NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float factor = WIDE && number ? sv * rv : 1.f;
                    uint32_t x[PARTS], y[PARTS];
                    split<PARTS>(s[nt][0] * factor, s[nt][1] * factor, x);
                    split<PARTS>(s[nt][2] * factor, s[nt][3] * factor, y);
#pragma unroll
                    for (int i = 0; i < PARTS; ++i) {
                        b[i][nt][0] = transpose(x[i]);
                        b[i][nt][1] = transpose(y[i]);
                    }
                }
                uint32_t v[4][HD / 32];
                if (HD == 128) {                            // this thread's 16 dimensions
                    *reinterpret_cast<uint4 *>(v[0]) = lds128(at + v_off[0]);
                    *reinterpret_cast<uint4 *>(v[1]) = lds128(at + v_off[1]);
                    *reinterpret_cast<uint4 *>(v[2]) = lds128(at + second(v_off[0]));
                    *reinterpret_cast<uint4 *>(v[3]) = lds128(at + second(v_off[1]));
                } else {                                    // its 8
                    *reinterpret_cast<uint2 *>(v[0]) = lds64(at + v_off[0]);
                    *reinterpret_cast<uint2 *>(v[1]) = lds64(at + v_off[1]);
                    *reinterpret_cast<uint2 *>(v[2]) = lds64(at + second(v_off[0]));
                    *reinterpret_cast<uint2 *>(v[3]) = lds64(at + second(v_off[1]));
                }
#pragma unroll
                for (int k = 0; k < HD / 32; ++k) {         // dimensions 4 k .. 4 k + 3 of the thread's, two to a product
                    const uint32_t p0 = __byte_perm(v[0][k], v[1][k], 0x5140) ^ 0x80808080u, p1 = __byte_perm(v[0][k], v[1][k], 0x7362) ^ 0x80808080u;
                    const uint32_t p2 = __byte_perm(v[2][k], v[3][k], 0x5140) ^ 0x80808080u, p3 = __byte_perm(v[2][k], v[3][k], 0x7362) ^ 0x80808080u;
                    const uint32_t a0[4] = {hsub2(__byte_perm(p0, MAGIC, 0x4140)), hsub2(__byte_perm(p0, MAGIC, 0x4342)),
                                            hsub2(__byte_perm(p2, MAGIC, 0x4140)), hsub2(__byte_perm(p2, MAGIC, 0x4342))};
                    const uint32_t a1[4] = {hsub2(__byte_perm(p1, MAGIC, 0x4140)), hsub2(__byte_perm(p1, MAGIC, 0x4342)),
                                            hsub2(__byte_perm(p3, MAGIC, 0x4140)), hsub2(__byte_perm(p3, MAGIC, 0x4342))};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if constexpr (WIDE) {
                            float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                            for (int i = PARTS - 1; i >= 0; --i) {
                                mma_f16(t0, a0, b[i][nt][0], b[i][nt][1]);
                                mma_f16(t1, a1, b[i][nt][0], b[i][nt][1]);
                            }
#pragma unroll
                            for (int i = 0; i < 4; ++i) o[nt][2 * k][i] += t0[i], o[nt][2 * k + 1][i] += t1[i];
                        } else {
                            mma_f16(o[nt][2 * k], a0, b[0][nt][0], b[0][nt][1]);
                            mma_f16(o[nt][2 * k + 1], a1, b[0][nt][0], b[0][nt][1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty_bar(stage));
            if (++stage == R::STAGES) stage = 0, phase ^= 1u;
        }

        // the four warps' states, in warp order
        asm volatile("bar.sync 1, 128;" ::: "memory");      // the part before has been read
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float sum = l[nt][i];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
                const int r = 8 * nt + 2 * c + i;
                // rows 2 c + i of this thread's dimensions: chunk (g >> 1) + 4 (g & 1) of 16, or 8 g ..
                float *row = meet + (warp * ROWS + r) * R::LDO + (HD == 128 ? 16 * ((g >> 1) + 4 * (g & 1)) : 8 * g);
#pragma unroll
                for (int k = 0; k < HD / 32; ++k)
                    *reinterpret_cast<float4 *>(row + 4 * k) = make_float4(o[nt][2 * k][i], o[nt][2 * k][2 + i], o[nt][2 * k + 1][i], o[nt][2 * k + 1][2 + i]);
                if (g == 0) {
                    meet_ml[(warp * ROWS + r) * 2] = m[nt][i];
                    meet_ml[(warp * ROWS + r) * 2 + 1] = sum;
                }
            }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const long long part = 2ll * blockIdx.x + (first_part ? 0 : 1);
        for (int idx = tid; idx < ROWS * (HD / 8); idx += 128) {
            const int r = idx / (HD / 8), d = (idx % (HD / 8)) * 8;
            if (r >= w.rows) break;
            float M = -INFINITY, L = 0.f, acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < 4; ++x) M = fmaxf(M, meet_ml[(x * ROWS + r) * 2]);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float mw = meet_ml[(x * ROWS + r) * 2], lw = meet_ml[(x * ROWS + r) * 2 + 1];
                const float f = mw == -INFINITY ? 0.f : exp2f(mw - M);
                if (f == 0.f && lw == lw) continue;         // (a sum that is no number stays that)
                L = fmaf(lw, f, L);
                const float *src = meet + (x * ROWS + r) * R::LDO + d;
                const float4 a = *reinterpret_cast<const float4 *>(src), b = *reinterpret_cast<const float4 *>(src + 4);
                acc[0] = fmaf(a.x, f, acc[0]); acc[1] = fmaf(a.y, f, acc[1]); acc[2] = fmaf(a.z, f, acc[2]); acc[3] = fmaf(a.w, f, acc[3]);
                acc[4] = fmaf(b.x, f, acc[4]); acc[5] = fmaf(b.y, f, acc[5]); acc[6] = fmaf(b.z, f, acc[6]); acc[7] = fmaf(b.w, f, acc[7]);
            }
            if (CLUSTER && !w.whole) {
                // this part's sums stay in the ring's memory, whose tiles have all been consumed, for the cluster
                float *fin = reinterpret_cast<float *>(ring) + r * HD + d;
                *reinterpret_cast<float4 *>(fin) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                *reinterpret_cast<float4 *>(fin + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
                if (d == 0) *reinterpret_cast<float2 *>(ring + FIN_ML + 8 * r) = make_float2(ok ? M : __uint_as_float(0x7fc00000u), L);
                continue;
            }
            if (!ok) continue;                              // a wait gave up: nothing is written
            if (w.whole) {
                store(w.out_row(r) * HD + d, acc, L);
            } else {
                float *po = part_out<HD>(p, part, r) + d;
                *reinterpret_cast<float4 *>(po) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                *reinterpret_cast<float4 *>(po + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
                if (d == 0) *part_ml(p, part, r) = make_float2(M, L);
            }
        }
        first_part = false;
    }
    }   // consumers
    // At the beginning this let the join kernel's CTAs, and those of the launch behind it, in a few at a time: 64 requests behind 4,095 keys,
    // heads of 64, took 83 us instead of 69.
    if (!CLUSTER) pdl_launch_dependents();

    if (CLUSTER && !w.whole) {
        // the parts of one pair, in ascending order of the keys; the rows are shared out among the CTAs.  Every thread takes part in the
        // barriers; no CTA leaves while its shared memory may still be read.
        const int rank = blockIdx.x % p.slices;
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        // MOST: parts at most, 8 or 16
        auto join = [&](auto most) {
            constexpr int MOST = most();
            for (int idx = tid; idx < ROWS * (HD / 8); idx += 128) {
                const int r = idx / (HD / 8), d = (idx % (HD / 8)) * 8;
                if (r >= w.rows) break;
                if (r % p.slices != rank) continue;
                // all parts' maxima and sums and eight parts' outputs in flight at once
                float2 ml[MOST];
#pragma unroll
                for (int s = 0; s < MOST; ++s) ml[s] = s < p.slices ? ld_cluster2(in_cluster(base + FIN_ML + 8 * r, s)) : make_float2(-INFINITY, 0.f);
                float M = -INFINITY, L = 0.f, acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                bool fine = true;
#pragma unroll
                for (int s0 = 0; s0 < MOST; s0 += 8) {
                    float4 x[8][2];
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        if (s0 + s >= p.slices) continue;
                        x[s][0] = ld_cluster4(in_cluster(base + (r * HD + d) * 4, s0 + s));
                        x[s][1] = ld_cluster4(in_cluster(base + (r * HD + d + 4) * 4, s0 + s));
                    }
                    if (s0 == 0) {
#pragma unroll
                        for (int s = 0; s < MOST; ++s) {
                            fine = fine && ml[s].x == ml[s].x;      // a wait gave up: nothing is written
                            M = fmaxf(M, ml[s].x);
                        }
                    }
#pragma unroll
                    for (int s = 0; s < 8; ++s) {
                        const float2 part = ml[s0 + s];
                        const float f = part.x == -INFINITY ? 0.f : exp2f(part.x - M);
                        if (s0 + s >= p.slices || (f == 0.f && part.y == part.y)) continue;     // (a sum that is no number stays that)
                        L = fmaf(part.y, f, L);
                        acc[0] = fmaf(x[s][0].x, f, acc[0]); acc[1] = fmaf(x[s][0].y, f, acc[1]); acc[2] = fmaf(x[s][0].z, f, acc[2]); acc[3] = fmaf(x[s][0].w, f, acc[3]);
                        acc[4] = fmaf(x[s][1].x, f, acc[4]); acc[5] = fmaf(x[s][1].y, f, acc[5]); acc[6] = fmaf(x[s][1].z, f, acc[6]); acc[7] = fmaf(x[s][1].w, f, acc[7]);
                    }
                }
                if (fine) store(w.out_row(r) * HD + d, acc, L);
            }
        };
        if (warp < 4) {
            if (p.slices <= 8) join(std::integral_constant<int, 8>());
            else join(std::integral_constant<int, MAX_CLUSTER>());
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

// Joins the parts of the pairs that lie in several CTAs' stretches: a warp a row, HD / 32 neighbouring dimensions a lane, eight parts'
// outputs in flight.  Bound by the latency of a few dependent loads: 3 to 4 us behind the stretches of 64 or two requests.
template <typename T, int HD>
__global__ void __launch_bounds__(256) attention_q8_join_kernel(const Q8Params p, int ctas) {
    pdl_launch_dependents();
    constexpr int DL = HD / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, seq = blockIdx.x / p.row_tiles, rt = blockIdx.x - seq * p.row_tiles, kvh = blockIdx.y, G = p.nq / p.nkv;
    const Line line{p};                 // (the description is there: every CTA of the stretches has waited for it before it let this kernel in)
    int before = 0, all = 0, row_tiles;
    for (int i = lane; i < p.nseq; i += 32) {
        const int n = line.place_of(i);
        all += n;
        if (i < seq) before += n;
    }
    const long long length = (long long)__reduce_add_sync(0xffffffffu, all) * p.nkv;
    const int n = line.tiles_of(seq, row_tiles);
    const long long begin = (long long)__reduce_add_sync(0xffffffffu, before) * p.nkv + ((long long)kvh * row_tiles + place_of_row_tile(rt, row_tiles)) * n;
    pdl_wait();
    if (n == 0 || rt >= row_tiles) return;
    ctas = stretches(length, ctas);
    const int u0 = holder(begin, length, ctas), u1 = holder(begin + n - 1, length, ctas);
    if (u0 == u1) return;
    const int tok_begin = p.cu_seqlens[seq], row0 = rt * p.rows_per_tile, rows = min(p.rows_per_tile, (p.cu_seqlens[seq + 1] - tok_begin) * G - row0);
    const long long first = 2ll * u0 + (begin > stretch(u0, length, ctas) ? 1 : 0);      // in its own CTA the pair's part is the last one
    auto part_of = [&](int k) { return k == 0 ? first : 2ll * (u0 + k); };
    const int parts = u1 - u0 + 1;
    for (int r = warp; r < rows; r += 8) {
        float M = -INFINITY;
        for (int k = lane; k < parts; k += 32) M = fmaxf(M, part_ml(p, part_of(k), r)->x);
        M = warp_max(M);
        float L = 0.f, acc[DL] = {};
        for (int k0 = 0; k0 < parts; k0 += 32) {
            const float2 ml = k0 + lane < parts ? *part_ml(p, part_of(k0 + lane), r) : make_float2(-INFINITY, 0.f);
            const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
            L += warp_sum(f == 0.f && ml.y == ml.y ? 0.f : ml.y * f);            // (a sum that is no number stays that)
            for (int k = 0; k < min(32, parts - k0); k += 8) {
                float x[8][DL];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k0 + k + j < parts) {
                        const float *src = part_out<HD>(p, part_of(k0 + k + j), r) + lane * DL;
                        if (DL == 4) *reinterpret_cast<float4 *>(x[j]) = *reinterpret_cast<const float4 *>(src);
                        else *reinterpret_cast<float2 *>(x[j]) = *reinterpret_cast<const float2 *>(src);
                    }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (k0 + k + j >= parts) break;
                    const float fs = __shfl_sync(0xffffffffu, f, k + j);
                    if (fs == 0.f) continue;
#pragma unroll
                    for (int d = 0; d < DL; ++d) acc[d] = fmaf(x[j][d], fs, acc[d]);
                }
            }
        }
        const float inv = 1.0f / L;
        T *out = (T *)p.out + ((size_t)(tok_begin + (row0 + r) / G) * p.nq + kvh * G + (row0 + r) % G) * HD + lane * DL;
#pragma unroll
        for (int d = 0; d < DL; d += 2) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float2 *>(out + d) = make_float2(acc[d] * inv, acc[d + 1] * inv);
            else *reinterpret_cast<__nv_bfloat162 *>(out + d) = __floats2bfloat162_rn(acc[d] * inv, acc[d + 1] * inv);
        }
    }
}

template <typename T, int HD, int NT> constexpr size_t decode_smem() { return Ring<HD, NT, T>::BYTES + 1024; }

// all but the grid and the stream of a launch in clusters
template <typename T, int HD, int NT>
int cluster_config(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, int size) {
    if (cudaFuncSetAttribute(attention_q8_decode_kernel<T, HD, NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)decode_smem<T, HD, NT>()) != cudaSuccess)
        return kestrel_fail(-3, "attention_q8: cannot raise the shared-memory limit: %s", cudaGetErrorString(cudaGetLastError()));
    // more than eight CTAs a cluster are not on every device; how many such clusters this one holds is asked below
    if (size > 8 && cudaFuncSetAttribute(attention_q8_decode_kernel<T, HD, NT, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return kestrel_fail(-3, "attention_q8: clusters of %d: %s", size, cudaGetErrorString(cudaGetLastError()));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = decode_smem<T, HD, NT>();
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return 0;
}

template <typename T, int HD, int NT>
int launch_decode(const Q8Params &p, int ctas, cudaStream_t stream) {
    int rc;
    if (p.slices > 0) {
        // a CTA, or a cluster of them, a pair
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[2];
        rc = cluster_config<T, HD, NT>(cfg, attr, p.slices);
        if (rc) return rc;
        cfg.gridDim = dim3((unsigned)p.tiles * p.nkv * p.slices);
        cfg.stream = stream;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = g_kestrel_pdl ? 2 : 1;
        cudaLaunchKernelEx(&cfg, attention_q8_decode_kernel<T, HD, NT, true>, p);
        return kestrel_check_launch("attention_q8 decode");
    }
    if (cudaFuncSetAttribute(attention_q8_decode_kernel<T, HD, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)decode_smem<T, HD, NT>()) != cudaSuccess)
        return kestrel_fail(-3, "attention_q8: cannot raise the shared-memory limit: %s", cudaGetErrorString(cudaGetLastError()));
    kestrel_launch(attention_q8_decode_kernel<T, HD, NT, false>, dim3(ctas), dim3(THREADS), decode_smem<T, HD, NT>(), stream, p);
    rc = kestrel_check_launch("attention_q8 decode");
    if (rc) return rc;
    kestrel_launch(attention_q8_join_kernel<T, HD>, dim3((unsigned)p.nseq * p.row_tiles, p.nkv), dim3(256), 0, stream, p, ctas);
    return kestrel_check_launch("attention_q8 join");
}

// Clusters of `size` CTAs that the current device holds at once.  A cluster lies within one GPC, so they are fewer than the CTAs' places
// divided by their size.  Asked of the runtime once a device, head size, rows and size.
template <typename T, int HD, int NT>
int resident_clusters(int size) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    if (cluster_config<T, HD, NT>(cfg, attr, size)) return 0;
    cfg.gridDim = dim3(size);
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, attention_q8_decode_kernel<T, HD, NT, true>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return n;
}

// calls f with the kernel's types and sizes: (T, head size, column tiles); float32 in tiles of 16 rows is for head size 64 alone
template <typename F>
auto with_form(Q8Form form, int hd, F f) {
    auto sized = [&](auto t, auto nt) { return hd == 64 ? f(t, std::integral_constant<int, 64>(), nt) : f(t, std::integral_constant<int, 128>(), nt); };
    using One = std::integral_constant<int, 1>;
    if (form == Q8_WIDE_SIXTEEN) return f(0.f, std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    return form == Q8_WIDE_EIGHT ? sized(0.f, One()) : form == Q8_EIGHT ? sized(__nv_bfloat16(), One()) : sized(__nv_bfloat16(), std::integral_constant<int, 2>());
}

}  // namespace

int q8_launch_decode(const Q8Params &p, Q8Form form, int ctas, cudaStream_t stream) {
    return with_form(form, p.hd, [&](auto t, auto hd, auto nt) { return launch_decode<decltype(t), hd(), nt()>(p, ctas, stream); });
}

// As many as are resident at once.  A stretch of fewer than two tiles costs more to begin and to join than it takes.
int q8_decode_ctas(long long tiles, int hd, Q8Form form) {
    const long long most = with_form(form, hd, [](auto t, auto h, auto nt) { return Ring<h(), nt(), decltype(t)>::CTAS; }) * (long long)kestrel_sms();
    return (int)(tiles / 2 < 1 ? 1 : tiles / 2 < most ? tiles / 2 : most);
}

// CTAs a pair, or 0 for stretches.  (Times in us; bfloat16, 32 / 8 heads of 128 | of 64 | float32 of 128 | of 64.)
// Where every pair can have its CTAs at once, as many as let every cluster be resident, up to 8, and two tiles each, or up to 16 where these have
// four; taken where the longest pair's share is no more than six tiles above a stretch, which is about what the join kernel takes:
//     1 request behind 1,003: 8 CTAs 6.2 | 5.5 | 6.6 | 5.9, stretches 7.8 | 7.1 | 8.6 | 7.9;   1 behind 4,095: 16 CTAs 10 | 8.3 | 11 | 9.2, 8 10 | 8.7 | 12.5 | 11
//     2 behind 8,000: 16 CTAs 15 | 12 | 28 | 24, 8 18 | 14 | 23 | 18, stretches 17 | 15 | 19 | 15 (float32 holds fewer such clusters: stretches)
//     8 behind 4,095: rule 18 | 14 | 24 | 20, stretches 20 | 17 | 28 | 22;   32 behind 500: one CTA 13 | 10 | 14 | 11, stretches 17 | 15 | 20 | 16
//     27 behind 4,000: two CTAs 40 | 30 | 78 | 62, stretches 45 | 39 | 67 | 49 (float32: taken);   55 behind 4,000: one 71 | 50 | 125 | 107, stretches 82 | 58 | 128 | 90
// Where only bounds are known (a recorded step, whose requests may be far shorter than the longest) a share is sixteen tiles at most: 8 requests
// behind 6,000, shares of 16, 23 | 17 | 46 | - against 25 | 21 | 36 in stretches, one behind 6,000 and seven behind 300 21 | 16 | 21 against 17 | 15 | 17, but
// one behind 16,000 and seven behind 300, shares of 42, 45 | 34 | 48 against 22 | 19 | 25.  Stretches follow the real lengths.
// (Recorded steps of like requests pay for that: 27 behind 4,000 45 instead of 40, 55 of them 82 instead of 70.)
// Where there are more pairs, one CTA, if the wait for the last one is worth what pairs cost a stretch: some five tiles' time each, and the join:
//     256 behind 300: one 45 | 35 | 69 | 55, stretches 71 | 51 | 93 | 66;   behind 2,000: 172 | 123 | 264 | 208 and 203 | 143 | 312 | 221
//     256 behind 20 to 1,805: 94 | 73 | 149 | 120 and 205 | 156 | 301 | 222;   one behind 4,000 and 255 behind 300: 52 | 40 | 73 and 73 | 52 | 96
//     64 behind 1,000: 35 | 26 | 44 | 34 and 38 | 29 | 52 | 37;   behind 4,095: 111 | 82 | 143 | 111 and 97 | 67 | 148 | 104;   one behind 1,500 and 63 behind 20: 19 | 16 | 24 and 14 | 11 | 19
//     411 float32 tokens of one request, 16 / 4 heads of 128: 25 and 35
int q8_decode_cluster(long long pairs, int longest_tiles, long long tiles, int hd, Q8Form form, bool exact) {
    static DeviceTable<8 * (MAX_CLUSTER + 1)> known;
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        dev = -1;
    }
    auto resident = [&](int size) {
        return known.get(dev, (2 * (int)form + (hd == 64)) * (MAX_CLUSTER + 1) + size, [&] {
            return with_form(form, hd, [&](auto t, auto h, auto nt) { return resident_clusters<decltype(t), h(), nt()>(size); });
        });
    };
    const long long ctas = q8_decode_ctas(tiles, hd, form), stretch = (tiles + ctas - 1) / ctas;
    const int most = longest_tiles >= 4 * MAX_CLUSTER ? MAX_CLUSTER : 8;
    for (int size = longest_tiles / 2 < most ? (longest_tiles < 2 ? 1 : longest_tiles / 2) : most; size >= 1; --size) {
        const int share = (longest_tiles + size - 1) / size;
        if (share > stretch + 6 || (!exact && share > 16)) break;
        if (pairs <= resident(size)) return size;
    }
    const int at_once = resident(1);
    return at_once > 0 && pairs > at_once && longest_tiles <= 25 * pairs / (2 * at_once) + 15 ? 1 : 0;
}

long long q8_decode_scratch(int ctas, int hd) { return 2ll * ctas * 16 * (hd + 2); }

int q8_decode_error() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_q8d_error, sizeof(int)) != cudaSuccess) return -1;
    if (v) cudaMemcpyToSymbol(g_q8d_error, &zero, sizeof(int));
    return v;
}
