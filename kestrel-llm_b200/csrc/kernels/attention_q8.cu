// Attention over pages of int8 codes: the kernel on the CUDA cores, for head sizes other than 64 and 128, the merge of key slices, and the
// entry point that decides which kernel takes which requests.  Formulas in attention_q8.cuh.
#include "attention_q8.cuh"

#include <algorithm>
#include <climits>
#include <math.h>

namespace {

// ---- CUDA cores ------------------------------------------------------------------------------------
// A CTA takes 32 rows and walks its keys in tiles of 64: codes are widened to float32 in shared memory, the keys' times their scale,
// scores and outputs are register tiles of 4 rows by 4 keys (by HDP / 16 dimensions), the softmax runs online with float32 statistics.
// The values' scales enter with the weights: the weight of a key that a row may not see is zero whatever its scale is, and a code is
// always a number, so that what is not finite stays with the rows that see it.  Products are pairs of float32 multiply-adds.  Bound by
// shared memory: of a 16-byte load by four rows or keys come eight such instructions, and a tile of 64 keys takes a CTA 6 us.
// 411 tokens of one request, 16 / 4 heads of 80: 51 us in float32 and bfloat16, 8.5 TFLOP/s; of 256 95 us, 14.6; eight single tokens behind 3,000
// keys, heads of 80, 64 us, of 256 144 us.
constexpr int BM = 32, BN = 64, THREADS = 128;

__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
    float2 d;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
    return d;
}
__device__ __forceinline__ void fma_pair(uint64_t &c, uint64_t a, uint64_t b) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(c) : "l"(a), "l"(b)); }
// code i of four: as the low byte of the number 2^23 + (c + 128), which a byte permutation makes (a conversion takes four times as long)
__device__ __forceinline__ float code(uint32_t biased, int i) { return __uint_as_float(__byte_perm(biased, 0x4b000000u, 0x7440 + i)) - 8388736.0f; }

template <int HDP> constexpr int lds_k() { return HDP + 4; }          // padded rows: sixteen lanes read sixteen keys without bank conflicts
template <int HDP> constexpr size_t plain_smem() { return sizeof(float) * ((size_t)BM * lds_k<HDP>() + 2 * (size_t)BN * lds_k<HDP>() + BM * (BN + 4) + BN); }

template <typename T, int HDP>
__global__ void __launch_bounds__(THREADS) attention_q8_plain_kernel(const Q8Params p) {
    pdl_launch_dependents();
    constexpr int LD = lds_k<HDP>(), DV = HDP / 16, LP = BN + 4;
    extern __shared__ __align__(16) float q8_smem[];
    float *Q = q8_smem, *K = Q + BM * LD, *V = K + BN * LD, *P = V + BN * LD, *sv_s = P + BM * LP;
    const int tid = threadIdx.x, kvh = blockIdx.y, slice = blockIdx.z;
    const int rg = tid >> 4, kg = tid & 15;             // rows 4 rg .. + 3; keys kg + 16 j, dimensions 4 kg + 64 j
    pdl_wait();
    Q8Tile t;
    if (!q8_find_tile(p, blockIdx.x, t)) return;
    int lo, hi;
    q8_slice(t, p.slices, slice, BN, lo, hi);
    // The four runs of a chunk of 16 dimensions lie a quarter of a row apart, so that the neighbours that hold a row's chunks write 16 bytes
    // side by side.
    auto place = [](int d, int run) { return run * (HDP / 4) + d / 4; };
    // the queries, sixteen numbers a thread and turn, all of them in flight
#pragma unroll
    for (int i = 0; i < (BM * (HDP / 16) + THREADS - 1) / THREADS; ++i) {
        const int r = (tid + i * THREADS) / (HDP / 16), d = (tid + i * THREADS) % (HDP / 16) * 16;
        if (r >= BM) break;
        const bool there = r < t.rows && d < p.hd;
        const T *src = (const T *)p.q + (there ? q8_out_row(p, t, kvh, r) * p.hd + d : 0);
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (there) {
                if (sizeof(T) == 4) {
                    x = *reinterpret_cast<const float4 *>(src + j);
                } else {
                    const uint2 u = *reinterpret_cast<const uint2 *>(src + j);
                    x = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xffff0000u));
                }
            }
            *reinterpret_cast<float4 *>(Q + r * LD + place(d, j / 4)) = x;
        }
    }
    float m[4], l[4];
    uint64_t o[4][DV / 2];
    int pos[4], low[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < DV / 2; ++d) o[i][d] = 0;
        const int r = 4 * rg + i;
        pos[i] = r < t.rows ? t.pos_begin + (t.row0 + r) / t.G : -1;
        low[i] = p.window > 0 ? max(0, pos[i] - p.window + 1) : 0;
    }
    const float scale_log2 = p.scale * 1.4426950408889634f;
    // sixteen codes a thread and load; those of the next tile are on their way while this one is worked on
    constexpr int LOADS = BN * (HDP / 16) / THREADS;
    uint4 kq[LOADS], vq[LOADS];
    float ks[LOADS], vs[LOADS];
    auto fetch = [&](int kb) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = (tid + i * THREADS) / (HDP / 16), d = (tid + i * THREADS) % (HDP / 16) * 16, key = kb + r;
            kq[i] = vq[i] = make_uint4(0, 0, 0, 0);         // keys outside the slice count as zero, whatever their page holds
            ks[i] = vs[i] = 0.f;
            if (key < lo || key >= hi || d >= p.hd) continue;
            const int row = q8_row_of(p, t.table, kvh, key);
            const size_t at = (size_t)(row + key % Q8_BLOCK) * p.hd + d;
            kq[i] = *reinterpret_cast<const uint4 *>(p.k + at);
            vq[i] = *reinterpret_cast<const uint4 *>(p.v + at);
            ks[i] = p.ks[row / Q8_BLOCK];
            vs[i] = p.vs[row / Q8_BLOCK];
        }
    };
    if (lo < hi) fetch(lo / BN * BN);
    for (int kb = lo / BN * BN; kb < hi; kb += BN) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = (tid + i * THREADS) / (HDP / 16), d = (tid + i * THREADS) % (HDP / 16) * 16;
            const uint32_t kw[4] = {kq[i].x, kq[i].y, kq[i].z, kq[i].w}, vw[4] = {vq[i].x, vq[i].y, vq[i].z, vq[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t k = kw[j] ^ 0x80808080u, v = vw[j] ^ 0x80808080u;
                *reinterpret_cast<float4 *>(K + r * LD + place(d, j)) = make_float4(code(k, 0) * ks[i], code(k, 1) * ks[i], code(k, 2) * ks[i], code(k, 3) * ks[i]);
                *reinterpret_cast<float4 *>(V + r * LD + place(d, j)) = make_float4(code(v, 0), code(v, 1), code(v, 2), code(v, 3));
            }
            if (d == 0) sv_s[r] = vs[i];
        }
        __syncthreads();
        if (kb + BN < hi) fetch(kb + BN);
        uint64_t s2[4][4] = {};             // even and odd dimensions' sums
#pragma unroll 4
        for (int d = 0; d < HDP; d += 4) {
            ulonglong2 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const ulonglong2 *>(Q + (4 * rg + i) * LD + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = *reinterpret_cast<const ulonglong2 *>(K + (kg + 16 * j) * LD + d);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    fma_pair(s2[i][j], a[i].x, b[j].x);
                    fma_pair(s2[i][j], a[i].y, b[j].y);
                }
        }
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = halves(s2[i][j]).x + halves(s2[i][j]).y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float mx = -INFINITY;
            bool seen[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = kb + kg + 16 * j;
                seen[j] = key >= lo && key < hi && key <= pos[i] && key >= low[i];
                s[i][j] = seen[j] ? s[i][j] * scale_log2 : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float mn = fmaxf(m[i], mx), use = mn == -INFINITY ? 0.f : mn;
            const float alpha = exp2f(m[i] - use);
            m[i] = mn;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = exp2f(s[i][j] - use);
                sum += s[i][j];
                P[(4 * rg + i) * LP + kg + 16 * j] = seen[j] ? s[i][j] * sv_s[kg + 16 * j] : 0.f;
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            l[i] = l[i] * alpha + sum;
#pragma unroll
            for (int d = 0; d < DV / 2; ++d) {
                const float2 x = halves(o[i][d]);
                o[i][d] = pair(x.x * alpha, x.y * alpha);
            }
        }
        __syncwarp();               // a row's probabilities are its own sixteen lanes'
#pragma unroll 2
        for (int j = 0; j < BN; j += 4) {
            float pr[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 x = *reinterpret_cast<const float4 *>(P + (4 * rg + i) * LP + j);
                pr[i][0] = x.x; pr[i][1] = x.y; pr[i][2] = x.z; pr[i][3] = x.w;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int d = 0; d < DV; d += 4) {
                    const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(V + (j + k) * LD + 4 * kg + 16 * d);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        fma_pair(o[i][d / 2], pair(pr[i][k], pr[i][k]), x.x);
                        fma_pair(o[i][d / 2 + 1], pair(pr[i][k], pr[i][k]), x.y);
                    }
                }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * rg + i;
        if (r >= t.rows) continue;
        const size_t row = q8_out_row(p, t, kvh, r);
        const float inv = p.slices > 1 ? 1.0f : 1.0f / l[i];
#pragma unroll
        for (int d = 0; d < DV; d += 4) {
            const int at = 4 * kg + 16 * d, dim = at % (HDP / 4) * 4 + at / (HDP / 4) * 4;      // four neighbours, and where they belong
            if (dim >= p.hd) continue;
            const float2 x = halves(o[i][d / 2]), y = halves(o[i][d / 2 + 1]);
            if (p.slices > 1) {
                *reinterpret_cast<float4 *>(p.part_o + (row * p.slices + slice) * p.hd + dim) = make_float4(x.x, x.y, y.x, y.y);
            } else if (sizeof(T) == 4) {
                *reinterpret_cast<float4 *>((T *)p.out + row * p.hd + dim) = make_float4(x.x * inv, x.y * inv, y.x * inv, y.y * inv);
            } else {
                const __nv_bfloat162 a = __floats2bfloat162_rn(x.x * inv, x.y * inv), b = __floats2bfloat162_rn(y.x * inv, y.y * inv);
                *reinterpret_cast<uint2 *>((T *)p.out + row * p.hd + dim) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
            }
        }
        if (p.slices > 1 && kg == 0) *reinterpret_cast<float2 *>(p.part_ml + (row * p.slices + slice) * 2) = make_float2(m[i], l[i]);
    }
}

// ---- merge -------------------------------------------------------------------------------------------
// A warp takes a row: lane s holds slice s's maximum and sum, the outputs are added in ascending order of the slices; a lane takes four
// neighbouring dimensions, four slices' in flight.  Bound by latency: 3 us behind a portion of 500 tokens, 16 heads of 64 in two slices.
template <typename T>
__global__ void __launch_bounds__(256) attention_q8_merge_kernel(const Q8Params p) {
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, kvh = blockIdx.y, r = blockIdx.z * 8 + (threadIdx.x >> 5);
    pdl_wait();
    Q8Tile t;
    if (!q8_find_tile(p, blockIdx.x, t) || r >= t.rows) return;
    const size_t row = q8_out_row(p, t, kvh, r);
    const float2 ml = lane < p.slices ? *reinterpret_cast<const float2 *>(p.part_ml + (row * p.slices + lane) * 2) : make_float2(-INFINITY, 0.f);
    const float M = warp_max(ml.x), f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
    const float inv = 1.0f / warp_sum(f == 0.f && ml.y == ml.y ? 0.f : ml.y * f);       // (a sum that is no number stays that)
    for (int d0 = 0; d0 < p.hd; d0 += 128) {
        const int d = d0 + 4 * lane;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s0 = 0; s0 < p.slices; s0 += 4) {
            float4 x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (s0 + j < p.slices && d < p.hd) x[j] = *reinterpret_cast<const float4 *>(p.part_o + (row * p.slices + s0 + j) * p.hd + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float fs = __shfl_sync(0xffffffffu, f, (s0 + j) & 31);
                if (s0 + j >= p.slices || d >= p.hd || fs == 0.f) continue;
                acc.x = fmaf(x[j].x, fs, acc.x); acc.y = fmaf(x[j].y, fs, acc.y); acc.z = fmaf(x[j].z, fs, acc.z); acc.w = fmaf(x[j].w, fs, acc.w);
            }
        }
        if (d < p.hd) {
            T *o = (T *)p.out + row * p.hd + d;
            o[0] = from_f32<T>(acc.x * inv); o[1] = from_f32<T>(acc.y * inv); o[2] = from_f32<T>(acc.z * inv); o[3] = from_f32<T>(acc.w * inv);
        }
    }
}

template <typename T, int HDP>
int launch_plain(const Q8Params &p, int tiles, cudaStream_t stream) {
    const size_t smem = plain_smem<HDP>();
    if (cudaFuncSetAttribute(attention_q8_plain_kernel<T, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return kestrel_fail(-3, "attention_q8: cannot raise the shared-memory limit: %s", cudaGetErrorString(cudaGetLastError()));
    kestrel_launch(attention_q8_plain_kernel<T, HDP>, dim3(tiles, p.nkv, p.slices), dim3(THREADS), smem, stream, p);
    return kestrel_check_launch("attention_q8");
}

}  // namespace

int q8_launch_plain(const Q8Params &p, int dtype, int tiles, cudaStream_t stream) {
    if (dtype == KESTREL_F32)
        return p.hd <= 64 ? launch_plain<float, 64>(p, tiles, stream) : p.hd <= 128 ? launch_plain<float, 128>(p, tiles, stream) : launch_plain<float, 256>(p, tiles, stream);
    return p.hd <= 64 ? launch_plain<__nv_bfloat16, 64>(p, tiles, stream)
                      : p.hd <= 128 ? launch_plain<__nv_bfloat16, 128>(p, tiles, stream) : launch_plain<__nv_bfloat16, 256>(p, tiles, stream);
}

int q8_launch_merge(const Q8Params &p, int dtype, int tiles, cudaStream_t stream) {
    const dim3 grid(tiles, p.nkv, (p.rows_per_tile + 7) / 8);
    if (dtype == KESTREL_F32) kestrel_launch(attention_q8_merge_kernel<float>, grid, dim3(256), 0, stream, p);
    else kestrel_launch(attention_q8_merge_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, p);
    return kestrel_check_launch("attention_q8 merge");
}

namespace {

constexpr int MAX_SLICES = 32;

// One launch of a step: the requests with rows_above < rows <= rows_upto, in tiles of rows_per_tile.
enum Kernel { CORES, DECODE, TC };
struct Part {
    Kernel kernel = CORES;
    Q8Form form = Q8_EIGHT;
    int rows_above = 0, rows_upto = 0, rows_per_tile = 0, slices = 1, longest = 0;
    long long tiles = 0;
    int ctas = 0, most_rows = 0, row_tiles = 0;
    long long scratch = 0;              // floats
    long long key_tiles = 0;             // of 64, over all requests and kv heads
};
struct Plan {
    Part part[2];
    int parts = 0;
};

int slices_for(long long ctas, int slots, int keys, int least) {
    if (ctas < 1 || keys < 1) return 1;
    return (int)std::max<long long>(1, std::min<long long>(std::min<long long>(slots / ctas, keys / least), MAX_SLICES));
}

// Rows follow from the host's copy of cu_seqlens; without it every request brings max_count tokens at most.
void make_plan(Plan &pl, const int *cu, const int *kv, int nseq, int max_count, int max_kv, int T, int nq, int nkv, int hd, int window, int dtype) {
    const int G = nq / nkv;
    auto seen_of = [&](int keys, long long rows) { return window > 0 ? (int)std::min<long long>(keys, window + (rows - 1) / G) : keys; };
    constexpr int FEW = 512;                // rows of a portion that may go to the decode kernel
    const bool cores = hd != 64 && hd != 128, wide = dtype != KESTREL_BF16;
    Part small, large;
    small.kernel = cores ? CORES : DECODE;
    small.rows_upto = cores || wide ? 0x7fffffff : 16;
    if (!cores && !wide && cu) {
        // Short portions go to the decode kernel, which reads a request's keys again for every 16 rows, if that leaves no portion to the other
        // kernel: where every pair has its CTAs at once and their work is little (32 / 8 heads of 128, one request, behind 500 keys: 16 tokens
        // 11.9 us against 14.8, 64 tokens 14.7 against 16.7, 128 tokens 17.7 against 17.8; 64 tokens behind 2,000 keys 27 against 19; four
        // requests of about 64 tokens behind 100, more pairs than CTAs, 19 against 11), and beside single tokens, which are a launch of the kernel
        // anyway, for three times that (requests of 2, 4, 6 and 8 tokens behind 2,000 keys 17 against 18, behind 8,000 36 against 54).
        // (32 / 8 heads of 64: 16 tokens behind 500 8.4 against 11.9, 64 11.6 and 13.1, 64 behind 2,000 21 and 15, four of 64 behind 100 14 and 8.3,
        // 2 to 8 behind 8,000 27 and 40; 24 / 8 of 128: 10.7 and 13.8, 14.4 and 16.4, 26 and 18, 18 and 10.6, 36 and 50.)
        long long tiles = 0;
        int most = 0, longest = 0;
        bool single = false, all = true;
        for (int i = 0; i < nseq; ++i) {
            const long long rows = (long long)(cu[i + 1] - cu[i]) * G;
            if (rows <= 0) continue;
            single |= rows <= 16;
            all &= rows <= FEW;
            if (!all) break;
            most = std::max(most, (int)rows);
            longest = std::max(longest, seen_of(kv[i], rows));
            tiles += (rows + 15) / 16 * nkv * ((seen_of(kv[i], rows) + 63) / 64);
        }
        const long long pairs = (long long)nseq * ((most + 15) / 16) * nkv;
        if (all && most > 16 && pairs <= 2ll * kestrel_sms() && tiles <= (single ? 24 : 8) * 2ll * kestrel_sms() &&
            (q8_decode_cluster(pairs, (longest + 63) / 64, tiles, hd, Q8_SIXTEEN, true) > 0 || (single && pairs <= q8_decode_ctas(tiles, hd, Q8_SIXTEEN))))
            small.rows_upto = FEW;
    }
    large.kernel = TC;
    large.rows_upto = 0x7fffffff;
    large.rows_per_tile = 256;
    if (!cores && !wide && cu) {
        // While tiles of 128 rows fit the SMs at once, a CTA may take one, and its key tiles go to the two streams in turn.  What a CTA has to do
        // is rows times keys of its slice, and slices cost their merge, as much as 128 rows' 380 keys; for as much to do, tiles of 128 take four
        // fifths of the time (32 / 8 heads of 128: 256 tokens 11 us in tiles of 128, 14 of 256; 500 behind 1,500 32 and 43, where only the latter
        // need slices; 300 behind 2,000 35 and 38; 500 behind 8,000 102 and 111).
        // (32 / 8 heads of 64: 256 tokens 8.1 and 10.8, 500 behind 1,500 27 and 36, 300 behind 2,000 28 and 30, 500 behind 8,000 86 and 94, 2,048 63 and 48;
        // 24 / 8 of 128: 10.5 and 14.4, 31 and 38, 30 and 34, 105 and 83, 60 and 52.  Where tiles of 128 just miss the SMs they would still be faster at times:
        // 16 / 4 of 64, 2,048 tokens 32 and 43; 24 / 8 of 128, 1,000 tokens 25 and 30.)
        // Single tokens beside portions come along where the SMs hold all of it at once and that takes no longer than a launch of the decode
        // kernel for them: what 128 rows' 400 keys take, and 55 more for every key tile of a CTA's (16 / 4 heads of 64, a window of 1,024: 500
        // tokens beside twelve single ones 20 us, in two launches 28; 32 / 8 heads of 128: 300 behind 2,000 beside six 35 and 51, 256 beside
        // eight behind 300 12 and 21, but beside one behind 3,000 31 and 22, 200 beside four behind 8,000 93 and 35).
        // (32 / 8 heads of 64: 29 and 37, 9.9 and 14.7, 27 and 16, 79 and 25; 24 / 8 of 128: 35 and 39 - not taken -, 12 and 18, 30 and 20, 57 and 32.)
        auto work = [&](int rows_above, int rows_per_tile) {
            long long tiles = 0;
            int longest = 0;
            for (int i = 0; i < nseq; ++i) {
                const long long rows = (long long)(cu[i + 1] - cu[i]) * G;
                if (rows <= rows_above) continue;
                tiles += (rows + rows_per_tile - 1) / rows_per_tile;
                longest = std::max(longest, seen_of(kv[i], rows));
            }
            const int slices = slices_for(tiles * nkv, kestrel_sms(), longest, 256);
            return tiles * nkv > kestrel_sms() ? LLONG_MAX : (long long)rows_per_tile * (longest / slices) + (slices > 1 ? 128 * 380 : 0);
        };
        long long halves = work(small.rows_upto, 128), whole = work(small.rows_upto, 256), singles = 0;
        bool portions = false;
        for (int i = 0; i < nseq; ++i) {
            const long long rows = (long long)(cu[i + 1] - cu[i]) * G;
            if (rows > small.rows_upto) portions = true;
            else if (rows > 0) singles += (seen_of(kv[i], rows) + 63) / 64 * (long long)nkv;
        }
        if (portions && singles && std::min(halves, whole) < LLONG_MAX) {
            const long long all_halves = work(0, 128), all_whole = work(0, 256);
            if (std::min(all_halves, all_whole) <= std::min(halves, whole) + 128 * (400 + 55 * singles / (3 * kestrel_sms()))) {
                small.rows_upto = 0;
                halves = all_halves;
                whole = all_whole;
            }
        }
        if (halves < LLONG_MAX && halves / 5 * 4 <= whole) large.rows_per_tile = 128;
    }
    // Recorded for no more than 128 rows a request (more than 16 query heads a kv head, single tokens): likewise (40 / 1 heads, ten requests behind
    // 1,000 keys 12.1 us in tiles of 128, 13.7 of 256; 64 of them 18.6 and 23.0; 72 / 2 heads, 32 behind 2,000 24 and 32).
    if (!cores && !wide && !cu && (long long)max_count * G <= 128) large.rows_per_tile = 128;
    large.rows_above = small.rows_upto;
    // float32: sixteen rows at head size 64, where they fit the registers (32 / 8 heads, 300 tokens behind 600 53 us, 64 in tiles of eight;
    // at 128, with spilled registers, 30 and 25 for 411 tokens)
    bool sixteen = !wide;
    if (wide && hd == 64) {
        if (!cu) sixteen = (long long)max_count * G > 8;
        else for (int i = 0; i < nseq; ++i) sixteen |= (long long)(cu[i + 1] - cu[i]) * G > 8;
    }
    small.rows_per_tile = cores ? BM : sixteen ? 16 : 8;
    auto count = [&](long long rows, int keys, int times) {
        if (rows <= 0) return;
        Part &p = rows <= small.rows_upto ? small : large;
        const int seen = seen_of(keys, rows);
        const long long each = (rows + p.rows_per_tile - 1) / p.rows_per_tile;
        // requests that may all bring so many rows still share the step's tokens
        p.tiles += times == 1 ? each : std::min(times * each, times + (long long)T * G / p.rows_per_tile);
        p.longest = std::max(p.longest, seen);
        p.most_rows = std::max(p.most_rows, (int)std::min<long long>(rows, p.rows_upto));
        p.key_tiles += times * each * nkv * ((seen + 63) / 64);
    };
    if (cu) {
        for (int i = 0; i < nseq; ++i) count((long long)(cu[i + 1] - cu[i]) * G, kv[i], 1);
    } else if ((long long)max_count * G <= small.rows_upto || G > small.rows_upto) {
        count((long long)max_count * G, max_kv, nseq);
    } else {                            // any request may be of either kind: both launches are made for all of them
        count(std::min<long long>(small.rows_upto, (long long)max_count * G), max_kv, nseq);
        count((long long)max_count * G, max_kv, nseq);
    }
    for (Part *p : {&small, &large}) {
        if (!p->tiles) continue;
        if (p->kernel == DECODE) {
            if (p->most_rows <= 8) p->rows_per_tile = 8;
            p->form = p->rows_per_tile == 8 ? (wide ? Q8_WIDE_EIGHT : Q8_EIGHT) : wide ? Q8_WIDE_SIXTEEN : Q8_SIXTEEN;
            p->ctas = q8_decode_ctas(p->key_tiles, hd, p->form);
            p->row_tiles = (p->most_rows + p->rows_per_tile - 1) / p->rows_per_tile;
            if (p->row_tiles == 1) p->tiles = nseq;
            p->slices = q8_decode_cluster(p->tiles * nkv, (p->longest + 63) / 64, p->key_tiles, hd, p->form, cu != nullptr);
            p->scratch = p->slices ? 0 : q8_decode_scratch(p->ctas, hd);
        } else {
            // The tensor cores: one CTA an SM, slices of two key tiles at least.  The CUDA cores: two CTAs an SM, which a key tile takes 6 us, the
            // merge 3: slices of one tile, and CTAs for two rounds (16 / 4 heads of 80: 8 tokens behind 400 keys 19 us, 45 with slices of 256
            // keys; 411 tokens 51 us, 63 with CTAs for one round).
            p->slices = p->kernel == TC ? slices_for(p->tiles * nkv, kestrel_sms(), p->longest, 256)
                                        : slices_for(p->tiles * nkv, kestrel_sms() * 4, p->longest, BN);
            p->scratch = p->slices > 1 ? (long long)T * nq * p->slices * (hd + 2) : 0;
        }
        pl.part[pl.parts++] = *p;
    }
}

}  // namespace

KESTREL_API long long kestrel_attention_q8_scratch(const int *cu_host, const int *kv_host, int nseq, int max_count, int max_kv, int T, int nq, int nkv, int hd,
                                                   int window, int dtype) {
    if (nseq <= 0 || T <= 0 || nq <= 0 || nkv <= 0 || nq % nkv) return 0;
    Plan pl;
    make_plan(pl, cu_host, kv_host, nseq, max_count, max_kv, T, nq, nkv, hd, window, dtype);
    long long most = 0;
    for (int i = 0; i < pl.parts; ++i) most = std::max(most, pl.part[i].scratch);
    return most;
}

KESTREL_API int kestrel_attention_q8(const void *q, const void *k_cache, const void *v_cache, const float *k_scale, const float *v_scale, void *out, float *scratch,
                                     long long scratch_floats, const int *cu_host, const int *kv_host, const int *cu_seqlens, const int *kv_lens,
                                     const int *block_table, int nseq, int max_count, int max_kv, int table_width, int table_stride, int page_size,
                                     int cache_pages, int T, int nq, int nkv, int hd, int window, float scale, int dtype, int described,
                                     kestrel_stream_t stream) {
    if (T == 0 || nseq == 0) return 0;
    KESTREL_REQUIRE(T > 0 && nseq > 0 && max_count > 0 && max_kv >= max_count, "attention_q8: a step of %d tokens of %d requests, %d at most, %d keys at most", T, nseq, max_count, max_kv);
    KESTREL_REQUIRE(dtype == KESTREL_F32 || dtype == KESTREL_BF16, "attention_q8: unknown dtype %d", dtype);
    KESTREL_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "attention_q8: %d query heads over %d kv heads", nq, nkv);
    KESTREL_REQUIRE(hd > 0 && hd % 16 == 0 && hd <= 256, "attention_q8: head size %d is no multiple of 16 up to 256", hd);
    KESTREL_REQUIRE(page_size > 0 && page_size % Q8_BLOCK == 0, "attention_q8: pages of %d tokens are no whole blocks of %d", page_size, Q8_BLOCK);
    KESTREL_REQUIRE(window >= 0 && scale > 0.f && isfinite(scale), "attention_q8: window %d, scale %g", window, scale);
    KESTREL_REQUIRE(cache_pages > 0 && (long long)cache_pages * nkv * page_size < (1ll << 31), "attention_q8: a cache of %d pages is beyond the 32-bit row coordinate", cache_pages);
    KESTREL_REQUIRE(table_width > 0 && table_stride >= table_width, "attention_q8: block table of %d entries a row, %d apart", table_width, table_stride);
    KESTREL_REQUIRE(nkv <= 65535 && nseq <= 0x7fffffff / nkv, "attention_q8: grid too large");
    KESTREL_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)scratch) & 15) == 0, "attention_q8: tensors must start on 16 bytes");
    Plan pl;
    make_plan(pl, cu_host, kv_host, nseq, max_count, max_kv, T, nq, nkv, hd, window, dtype);
    for (int i = 0; i < pl.parts; ++i) {
        const Part &part = pl.part[i];
        KESTREL_REQUIRE(part.tiles * nkv * std::max(part.slices, 1) < (1ll << 31) && (part.kernel != DECODE || (part.key_tiles / nkv < (1ll << 31) && (long long)nseq * part.row_tiles < (1ll << 31))),
                        "attention_q8: %lld row tiles and %lld key tiles of %d kv heads exceed the grid", part.tiles, part.key_tiles, nkv);
        if (part.scratch > 0 && (!scratch || part.scratch > scratch_floats))
            return kestrel_fail(-KESTREL_Q8_NEEDS_SCRATCH, "attention_q8: scratch of %lld floats is needed, %lld given", part.scratch, scratch_floats);
    }
    int launches = 0;
    for (int i = 0; i < pl.parts; ++i) {
        const Part &part = pl.part[i];
        Q8Params p = {};
        p.q = q; p.out = out; p.k = (const int8_t *)k_cache; p.v = (const int8_t *)v_cache; p.ks = k_scale; p.vs = v_scale;
        p.cu_seqlens = cu_seqlens; p.kv_lens = kv_lens; p.block_table = block_table;
        p.nseq = nseq; p.table_width = table_width; p.table_stride = table_stride; p.page_size = page_size; p.cache_pages = cache_pages;
        p.nq = nq; p.nkv = nkv; p.hd = hd; p.window = window; p.slices = part.slices; p.scale = scale; p.described = described;
        p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1;
        p.rows_above = part.rows_above; p.rows_upto = part.rows_upto; p.rows_per_tile = part.rows_per_tile; p.row_tiles = part.row_tiles;
        p.tiles = (int)part.tiles;
        p.part_o = scratch;
        int rc;
        if (part.kernel == DECODE) {
            p.part_ml = scratch ? scratch + 2ll * part.ctas * 16 * hd : nullptr;
            rc = q8_launch_decode(p, part.form, part.ctas, stream);
            launches += part.slices ? 1 : 2;
        } else {
            p.part_ml = scratch ? scratch + (long long)T * nq * part.slices * hd : nullptr;
            rc = part.kernel == TC ? q8_launch_tc(p, (int)part.tiles, stream) : q8_launch_plain(p, dtype, (int)part.tiles, stream);
            if (rc == 0 && part.slices > 1) rc = q8_launch_merge(p, dtype, (int)part.tiles, stream);
            launches += part.slices > 1 ? 2 : 1;
        }
        if (rc) return rc;
    }
    return launches;
}

// 1, 2: the decode kernel's loader and consumers; 100 and more: the portion kernel's wait
KESTREL_API int kestrel_attention_q8_error(void) {
    const int decode = q8_decode_error(), tc = q8_tc_error();
    return tc ? 100 + tc : decode;
}
