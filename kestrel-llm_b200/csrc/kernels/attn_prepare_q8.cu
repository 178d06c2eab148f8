// Appending to pages of int8 codes: a step's q, k, v product gets its bias, per-head norm and rotation; queries go to q_out, keys and
// values to their blocks of 16 tokens, coded against the block's scale.
//
// Two kinds of CTAs in one launch.  The first take one block of tokens of one (request, kv head): its keys and values stay in registers
// from the product to the codes, so that the block's largest magnitude is known before anything is rounded.  The others take one token's
// queries.  A block that earlier steps began and whose scale rises is read back and rounded again by the CTA that owns it: one owner a
// block, no atomics.  A row (one head of one token) belongs to LPR lanes that hold four neighbouring numbers each (NV times); the members
// of a rotation pair meet in shared memory.  Bound by the product's float32 bytes; at 2,048 tokens, 32 / 8 heads of 128, rotated and normed
// (71 MB), 18 us in a row of calls and 23 from cold caches, 3.9 and 3.1 TB/s, which instructions hold back: cosines, sums over a row, codes.
// 64 requests' tokens 4.0 us and one 3.7, from cold caches 6.2 and 8.0 (a product in 8 slices): latency.  The general form (heads other than 64 and
// 128, rotate-half pairs over part of a head) has pairs meet in shared memory: the same prompt with half of each head rotated 32 us, with heads of 80
// 32, 16 / 4 heads of 256 35.
//
// Angles are products of an int32 position and a float32 frequency, reduced in float64: a float32 product is off by 2^-24 of an angle that
// reaches 10^5 radians, 0.006 of one, by which every far key would be turned.
//
// A code is the whole number next to a float32 product with the scale's reciprocal, and the float32 product of a code with a ratio of scales where a
// scale has risen: within 1/2 + 2^-17 and 1/2 + 2^-16 of the quotient.  (Divisions instead: 2,048 tokens 18.8 us.  The number itself is off by
// some 2^-15 of a step.)
#include "attention_q8.cuh"

#include <math.h>

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_PAIRS = 128;          // of a head of 256

struct PrepParams {
    const float *partial, *bias, *q_w, *k_w, *inv_freq;
    size_t slice_stride;
    const int *positions, *cu, *table;
    int8_t *k, *v;
    float *ks, *vs;
    void *q_out;
    int S, nseq, table_width, table_stride, page_size, cache_pages, T, nq, nkv, hd, rot, rot_mode, units;
    int described;                  // positions, cu and table were on the device before the kernel in front of this one began
    float eps, rot_scale;
};

__device__ __forceinline__ float4 add4(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }

// Cosine and sine of position * frequency, times the encoding's scale.  What whole turns leave of the angle is off by its rounding to float32,
// 2^-23, and by what float64 loses: 2^-25 below position 2^28, 2^-22 at the largest; sincosf is within two units.
__device__ __forceinline__ float2 turn(int pos, float freq, float scale) {
    const double angle = (double)pos * (double)freq, turns = rint(angle * 0.15915494309189535);
    float s, c;
    sincosf((float)fma(turns, -6.283185307179586, angle), &s, &c);
    return make_float2(scale * c, scale * s);
}

template <int LPR, int NV>
struct Row {
    float4 x[NV];

    __device__ __forceinline__ static int dim(int sub, int v) { return 4 * sub + 4 * LPR * v; }

    __device__ __forceinline__ void load(const PrepParams &p, int t, int h, int sub, bool live) {
        const size_t at = ((size_t)t * (p.nq + 2 * p.nkv) + h) * p.hd;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            x[v] = make_float4(0.f, 0.f, 0.f, 0.f);
            const int d = dim(sub, v);
            if (!live || d >= p.hd) continue;
            for (int s = 0; s < p.S; ++s) x[v] = add4(x[v], *reinterpret_cast<const float4 *>(p.partial + (size_t)s * p.slice_stride + at + d));
            if (p.bias) x[v] = add4(x[v], *reinterpret_cast<const float4 *>(p.bias + (size_t)h * p.hd + d));
        }
    }

    __device__ __forceinline__ void norm(const PrepParams &p, const float *w, int sub) {
        float ss = 0.f;
#pragma unroll
        for (int v = 0; v < NV; ++v) ss += x[v].x * x[v].x + x[v].y * x[v].y + x[v].z * x[v].z + x[v].w * x[v].w;
#pragma unroll
        for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float rinv = 1.0f / sqrtf(ss / (float)p.hd + p.eps);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int d = dim(sub, v);
            if (d >= p.hd) continue;
            const float4 g = *reinterpret_cast<const float4 *>(w + d);
            x[v] = make_float4(x[v].x * rinv * g.x, x[v].y * rinv * g.y, x[v].z * rinv * g.z, x[v].w * rinv * g.w);
        }
    }

    // `stage`: this row's hd floats of shared memory; `cs`: (cosine, sine) of every pair of the token
    __device__ __forceinline__ void rotate(const PrepParams &p, float *stage, const float2 *cs, int sub) {
        const int half = p.rot >> 1;
        if (p.rot_mode == 0) {
            __syncwarp();
#pragma unroll
            for (int v = 0; v < NV; ++v)
                if (dim(sub, v) < p.rot) *reinterpret_cast<float4 *>(stage + dim(sub, v)) = x[v];
            __syncwarp();
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            float *e = reinterpret_cast<float *>(&x[v]);
            const int d = dim(sub, v);
            if (p.rot_mode == 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = d + i;
                    if (at >= p.rot) continue;
                    const bool first = at < half;
                    const float2 c = cs[first ? at : at - half];
                    const float other = stage[first ? at + half : at - half];
                    e[i] = first ? fmaf(e[i], c.x, -other * c.y) : fmaf(e[i], c.x, other * c.y);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    if (d + i >= p.rot) continue;
                    const float2 c = cs[(d + i) >> 1];
                    const float a = e[i], b = e[i + 1];
                    e[i] = fmaf(a, c.x, -b * c.y);
                    e[i + 1] = fmaf(b, c.x, a * c.y);
                }
            }
        }
    }

    // the bits of the largest magnitude: a number that is not finite compares above all others
    __device__ __forceinline__ unsigned largest() const {
        unsigned m = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            m = max(max(m, __float_as_uint(x[v].x) & 0x7fffffffu), __float_as_uint(x[v].y) & 0x7fffffffu);
            m = max(max(m, __float_as_uint(x[v].z) & 0x7fffffffu), __float_as_uint(x[v].w) & 0x7fffffffu);
        }
        return m;
    }
};

// Four codes as one word.  x / scale as a product with the reciprocal, which is off by 2^-24 of itself: 2^-17 of a step at most.  Added to 1.5 * 2^23 a number is
// rounded to a whole one, ties to even, whose two's complement is the low byte; no number is above the one that the scale came from.
__device__ __forceinline__ uint32_t codes_word(float a, float b, float c, float d, float inv) {
    constexpr float M = 12582912.0f;
    const uint32_t x = __float_as_uint(fmaf(a, inv, M)), y = __float_as_uint(fmaf(b, inv, M)), z = __float_as_uint(fmaf(c, inv, M)), w = __float_as_uint(fmaf(d, inv, M));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}

// A block's scale from the largest magnitude among the new tokens (its bits) and, where earlier steps began the block, its scale so far
__device__ __forceinline__ float block_scale(unsigned largest, bool begun, float before) {
    if (largest >= 0x7f800000u || (begun && !(before <= 3.4e38f))) return __uint_as_float(0x7fc00000u);
    const float s = fmaxf(__uint_as_float(largest) / 127.0f, 5.421010862427522e-20f);          // 2^-64
    return begun ? fmaxf(s, before) : s;
}

// The unit-th block of 16 positions among those that the step's requests touch
struct Block {
    int seq, t0, pos0, count;           // its request, first token, first position, tokens; seq -1: there are fewer
};
__device__ __forceinline__ Block find_block(const PrepParams &p, int unit) {
    const int lane = threadIdx.x & 31;
    Block r = {-1, 0, 0, 0};
    int left = unit;
    for (int base = 0; base < p.nseq && r.seq < 0; base += 32) {
        const int i = base + lane;
        int n = 0, first = 0, pos = 0, tokens = 0;
        if (i < p.nseq) {
            first = p.cu[i];
            tokens = p.cu[i + 1] - first;
            if (tokens > 0) {
                pos = p.positions[first];
                if (pos < 0) {                      // tokens in front of position 0 have no page
                    const int gone = pos > -tokens ? -pos : tokens;
                    first += gone;
                    tokens -= gone;
                    pos += gone;
                }
            }
            if (tokens > 0) {
                n = (pos + tokens - 1) / Q8_BLOCK - pos / Q8_BLOCK + 1;
            }
        }
        int end = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += x;
        }
        const unsigned behind = __ballot_sync(0xffffffffu, left < end);
        if (behind) {
            const int at = __ffs(behind) - 1;
            const int nth = left - __shfl_sync(0xffffffffu, end - n, at);            // among the request's blocks
            const int from = __shfl_sync(0xffffffffu, pos, at), cu = __shfl_sync(0xffffffffu, first, at), all = __shfl_sync(0xffffffffu, tokens, at);
            r.seq = base + at;
            r.pos0 = nth == 0 ? from : (from / Q8_BLOCK + nth) * Q8_BLOCK;
            r.t0 = cu + r.pos0 - from;
            r.count = min(from + all, (r.pos0 / Q8_BLOCK + 1) * Q8_BLOCK) - r.pos0;
        } else {
            left -= __shfl_sync(0xffffffffu, end, 31);
        }
    }
    return r;
}

// Codes that earlier steps left in a block, against a scale that has risen
__device__ __forceinline__ void round_again(int8_t *codes, int n, float ratio) {
    if (!(ratio < 1.0f)) return;                    // the same scale, or none
    char4 *c4 = reinterpret_cast<char4 *>(codes);
    for (int i = threadIdx.x; i < n / 4; i += THREADS) {
        const char4 c = c4[i];
        c4[i] = make_char4((signed char)__float2int_rn(c.x * ratio), (signed char)__float2int_rn(c.y * ratio), (signed char)__float2int_rn(c.z * ratio),
                           (signed char)__float2int_rn(c.w * ratio));
    }
}

// Head sizes 64 and 128 without rotation, with rotate-half pairs over the whole head (TURN 1) or neighbouring pairs (TURN 2).  Eight lanes
// hold a row, each the dimensions [n s, n s + n) and [HD / 2 + n s, ...) with n = HD / 16, so that both members of a pair are in one lane
// and a warp works on four rows: a third of the instructions of the general form, which is bound by them.
enum { TURN_NONE, TURN_HALF, TURN_NEXT };

// The same for steps with bfloat16 queries, their keys' codes included: __cosf and __sinf are off by 2^-21.2 and 2^-21.4 on [-pi, pi], so with the
// angle's 2^-22.7 a cosine is within 2^-20 of one, an absolute error, times the scale: 2^-12 of a code's step, and 2^-11 of a bfloat16 query's
// rounding.  Below position 2^28; 2^-19.8 at the largest.  (sincosf instead: 2,048 tokens 18.5 us, 17.9 so.)
__device__ __forceinline__ float2 turn_fast(int pos, float freq, float scale) {
    const double angle = (double)pos * (double)freq, turns = rint(angle * 0.15915494309189535);
    const float r = (float)fma(turns, -6.283185307179586, angle);
    return make_float2(scale * __cosf(r), scale * __sinf(r));
}

template <typename T, int HD, int TURN>
struct Eighth {
    static constexpr int N = HD / 16, N4 = N / 4;
    float x[2][N];                      // the two runs of dimensions

    __device__ __forceinline__ static int dim(int sub, int h) { return h * (HD / 2) + N * sub; }

    __device__ __forceinline__ void load(const PrepParams &p, int t, int h, int sub, bool live) {
        const float *at = p.partial + ((size_t)t * (p.nq + 2 * p.nkv) + h) * HD + N * sub;
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) x[i / N][i % N] = 0.f;
        if (!live) return;
        for (int s = 0; s < p.S; ++s, at += p.slice_stride) {
            float4 v[2][N4];
#pragma unroll
            for (int i = 0; i < 2 * N4; ++i) v[i / N4][i % N4] = __ldcs(reinterpret_cast<const float4 *>(at + (i / N4) * (HD / 2)) + i % N4);
#pragma unroll
            for (int i = 0; i < 2 * N; ++i) x[i / N][i % N] += reinterpret_cast<const float *>(&v[i / N][(i % N) / 4])[i % 4];
        }
        if (p.bias) {
#pragma unroll
            for (int i = 0; i < 2 * N; ++i) x[i / N][i % N] += p.bias[(size_t)h * HD + dim(sub, i / N) + i % N];
        }
    }
    __device__ __forceinline__ void norm(const PrepParams &p, const float *w, int sub) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) ss = fmaf(x[i / N][i % N], x[i / N][i % N], ss);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float rinv = 1.0f / sqrtf(ss * (1.0f / HD) + p.eps);
#pragma unroll
        for (int i = 0; i < 2 * N4; ++i) {
            const float4 g = *(reinterpret_cast<const float4 *>(w + dim(sub, i / N4)) + i % N4);
            float *e = &x[i / N4][4 * (i % N4)];
            e[0] *= rinv * g.x; e[1] *= rinv * g.y; e[2] *= rinv * g.z; e[3] *= rinv * g.w;
        }
    }
    // cs: (cosine, sine) of every pair of the token
    __device__ __forceinline__ void rotate(const PrepParams &p, const float2 *cs, int sub) {
        if (TURN == TURN_HALF) {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float4 c = *reinterpret_cast<const float4 *>(cs + N * sub + i);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float co = j ? c.z : c.x, si = j ? c.w : c.y, a = x[0][i + j], b = x[1][i + j];
                    x[0][i + j] = fmaf(a, co, -b * si);
                    x[1][i + j] = fmaf(b, co, a * si);
                }
            }
        } else if (TURN == TURN_NEXT) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < N; i += 2) {
                    const int d = dim(sub, h) + i;
                    if (d >= p.rot) continue;
                    const float2 c = cs[d >> 1];
                    const float a = x[h][i], b = x[h][i + 1];
                    x[h][i] = fmaf(a, c.x, -b * c.y);
                    x[h][i + 1] = fmaf(b, c.x, a * c.y);
                }
        }
    }
    __device__ __forceinline__ unsigned largest() const {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < 2 * N; ++i) m = max(m, __float_as_uint(x[i / N][i % N]) & 0x7fffffffu);
        return m;
    }
    __device__ __forceinline__ void put(T *o, int sub) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(o + dim(sub, h) + i) = make_float4(x[h][i], x[h][i + 1], x[h][i + 2], x[h][i + 3]);
            } else {
                __nv_bfloat162 w[N / 2];
#pragma unroll
                for (int i = 0; i < N / 2; ++i) w[i] = __floats2bfloat162_rn(x[h][2 * i], x[h][2 * i + 1]);
                if (N == 8) *reinterpret_cast<uint4 *>(o + dim(sub, h)) = *reinterpret_cast<uint4 *>(w);
                else *reinterpret_cast<uint2 *>(o + dim(sub, h)) = *reinterpret_cast<uint2 *>(w);
            }
        }
    }
    __device__ __forceinline__ void put_codes(int8_t *o, int sub, float inv) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t w[N4];
#pragma unroll
            for (int i = 0; i < N4; ++i) w[i] = codes_word(x[h][4 * i], x[h][4 * i + 1], x[h][4 * i + 2], x[h][4 * i + 3], inv);
            if (N == 8) *reinterpret_cast<uint2 *>(o + dim(sub, h)) = make_uint2(w[0], w[1 % N4]);
            else *reinterpret_cast<uint32_t *>(o + dim(sub, h)) = w[0];
        }
    }
};

template <typename T, int HD, int TURN>
__global__ void __launch_bounds__(THREADS) attn_prepare_q8_fast_kernel(const PrepParams p) {
    pdl_launch_dependents();
    __shared__ __align__(16) float2 cs[Q8_BLOCK][HD / 2];
    __shared__ unsigned big[WARPS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane & 7, mine = tid >> 3;
    const int half = TURN == TURN_NONE ? 0 : TURN == TURN_HALF ? HD / 2 : p.rot >> 1;
    const int kv_ctas = p.units * p.nkv;
    if (!p.described) pdl_wait();

    if ((int)blockIdx.x >= kv_ctas) {
        // ---- one token's queries, 32 heads at a time
        const int t = blockIdx.x - kv_ctas;
        if (t >= p.cu[p.nseq]) { pdl_wait(); return; }
        // in front of the wait, or while the product is on its way; half is no more than 64
        int pos = 0;
        float freq = 0.f;
        if (TURN != TURN_NONE && tid < half) pos = p.positions[t], freq = p.inv_freq[tid];
        auto angles = [&] {
            if (TURN != TURN_NONE && tid < half) cs[0][tid] = sizeof(T) == 4 ? turn(pos, freq, p.rot_scale) : turn_fast(pos, freq, p.rot_scale);
        };
        if (p.described) angles();
        pdl_wait();
        Eighth<T, HD, TURN> r;
        r.load(p, t, mine, sub, mine < p.nq);
        if (!p.described) angles();
        __syncthreads();
        for (int h0 = 0;;) {
            const int h = h0 + mine;
            if (p.q_w) r.norm(p, p.q_w, sub);
            r.rotate(p, cs[0], sub);
            if (h < p.nq) r.put((T *)p.q_out + ((size_t)t * p.nq + h) * HD, sub);
            h0 += THREADS / 8;
            if (h0 >= p.nq) break;
            r.load(p, t, h0 + mine, sub, h0 + mine < p.nq);
        }
        return;
    }

    // ---- one block of one (request, kv head): rows 0-15 are its tokens' keys, 16-31 their values
    const int kvh = blockIdx.x % p.nkv;
    const Block bl = find_block(p, blockIdx.x / p.nkv);
    if (bl.seq < 0) { pdl_wait(); return; }
    const int there = bl.pos0 % Q8_BLOCK;           // codes that earlier steps left in the block
    const int idx = bl.pos0 / p.page_size;
    const int page = idx < p.table_width ? p.table[(size_t)bl.seq * p.table_stride + idx] : -1;
    auto angles = [&] {
        if (TURN == TURN_NONE) return;
        for (int i = tid; i < bl.count * half; i += THREADS) {
            const int n = TURN == TURN_HALF ? i / (HD / 2) : i / half, j = i - n * half;
            cs[n][j] = sizeof(T) == 4 ? turn(bl.pos0 + n, p.inv_freq[j], p.rot_scale) : turn_fast(bl.pos0 + n, p.inv_freq[j], p.rot_scale);
        }
    };
    if (p.described) angles();
    pdl_wait();
    if (page < 0 || page >= p.cache_pages) return;  // no page to write to
    const size_t row0 = ((size_t)page * p.nkv + kvh) * p.page_size + (bl.pos0 - idx * p.page_size) - there;
    const bool is_k = warp < WARPS / 2;
    const int n = mine & (Q8_BLOCK - 1);
    float *scales = is_k ? p.ks : p.vs;
    int8_t *codes = (is_k ? p.k : p.v) + row0 * HD;
    const float k_before = there ? p.ks[row0 / Q8_BLOCK] : 0.f, v_before = there ? p.vs[row0 / Q8_BLOCK] : 0.f;
    Eighth<T, HD, TURN> r;
    r.load(p, bl.t0 + n, p.nq + (is_k ? 0 : p.nkv) + kvh, sub, n < bl.count);
    if (!p.described) angles();
    __syncthreads();                                // the cosines and sines
    if (is_k) {
        if (p.k_w) r.norm(p, p.k_w, sub);
        r.rotate(p, cs[n < bl.count ? n : 0], sub);
    }
    const unsigned m = __reduce_max_sync(0xffffffffu, n < bl.count ? r.largest() : 0u);
    if (lane == 0) big[warp] = m;
    __syncthreads();
    const unsigned k_big = max(max(big[0], big[1]), max(big[2], big[3])), v_big = max(max(big[4], big[5]), max(big[6], big[7]));
    const float k_s = block_scale(k_big, there > 0, k_before), v_s = block_scale(v_big, there > 0, v_before);
    if (n < bl.count) r.put_codes(codes + (size_t)(there + n) * HD, sub, 1.0f / (is_k ? k_s : v_s));
    if (there) {
        round_again(p.k + row0 * HD, there * HD, k_before / k_s);
        round_again(p.v + row0 * HD, there * HD, v_before / v_s);
    }
    if (tid == 0 || tid == THREADS / 2) scales[row0 / Q8_BLOCK] = is_k ? k_s : v_s;
}

template <typename T, int LPR, int NV>
__global__ void __launch_bounds__(THREADS) attn_prepare_q8_kernel(const PrepParams p) {
    pdl_launch_dependents();
    constexpr int RPW = 32 / LPR;                   // rows a warp holds at once
    constexpr int TOKENS = Q8_BLOCK / (WARPS * RPW) > 0 ? Q8_BLOCK / (WARPS * RPW) : 1;       // turns of a warp over a block's tokens
    __shared__ __align__(16) float stage[WARPS * RPW][4 * LPR * NV];
    __shared__ float2 cs[Q8_BLOCK][MAX_PAIRS];
    __shared__ unsigned big[2][WARPS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane % LPR, mine = warp * RPW + lane / LPR;
    const int half = p.rot >> 1;
    const int kv_ctas = p.units * p.nkv;
    if (!p.described) pdl_wait();
    const int n_tokens = p.cu[p.nseq];

    if ((int)blockIdx.x >= kv_ctas) {
        // ---- one token's queries
        const int t = blockIdx.x - kv_ctas;
        if (t >= n_tokens) { pdl_wait(); return; }
        const int pos = p.positions[t];
        for (int j = tid; j < half; j += THREADS) cs[0][j] = turn(pos, p.inv_freq[j], p.rot_scale);
        pdl_wait();
        __syncthreads();
        for (int h0 = 0; h0 < p.nq; h0 += WARPS * RPW) {
            const int h = h0 + mine;
            const bool live = h < p.nq;
            Row<LPR, NV> r;
            r.load(p, t, h, sub, live);
            if (p.q_w) r.norm(p, p.q_w, sub);
            if (p.rot) r.rotate(p, stage[mine], cs[0], sub);
            if (!live) continue;
            T *o = (T *)p.q_out + ((size_t)t * p.nq + h) * p.hd;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int d = r.dim(sub, v);
                if (d >= p.hd) continue;
                if (sizeof(T) == 4) {
                    *reinterpret_cast<float4 *>(o + d) = r.x[v];
                } else {
                    __nv_bfloat162 a = __floats2bfloat162_rn(r.x[v].x, r.x[v].y), b = __floats2bfloat162_rn(r.x[v].z, r.x[v].w);
                    *reinterpret_cast<uint2 *>(o + d) = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
                }
            }
        }
        return;
    }

    // ---- one block of one (request, kv head)
    const int kvh = blockIdx.x % p.nkv;
    const Block bl = find_block(p, blockIdx.x / p.nkv);
    const int seq = bl.seq, t0 = bl.t0, pos0 = bl.pos0, count = bl.count;
    if (seq < 0) { pdl_wait(); return; }
    const int there = pos0 % Q8_BLOCK;              // codes that earlier steps left in the block
    const int idx = pos0 / p.page_size;
    const int page = idx < p.table_width ? p.table[(size_t)seq * p.table_stride + idx] : -1;
    for (int i = tid; i < count * half; i += THREADS) cs[i / half][i % half] = turn(pos0 + i / half, p.inv_freq[i % half], p.rot_scale);
    pdl_wait();
    if (page < 0 || page >= p.cache_pages) return;  // no page to write to
    const size_t row0 = ((size_t)page * p.nkv + kvh) * p.page_size + (pos0 - idx * p.page_size) - there;
    const float k_before = there ? p.ks[row0 / Q8_BLOCK] : 0.f, v_before = there ? p.vs[row0 / Q8_BLOCK] : 0.f;
    Row<LPR, NV> k[TOKENS], v[TOKENS];
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
        const int n = mine + i * WARPS * RPW;
        k[i].load(p, t0 + n, p.nq + kvh, sub, n < count);
        v[i].load(p, t0 + n, p.nq + p.nkv + kvh, sub, n < count);
    }
    __syncthreads();                                // the cosines and sines
    unsigned k_big = 0, v_big = 0;
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
        const int n = mine + i * WARPS * RPW;
        if (p.k_w) k[i].norm(p, p.k_w, sub);
        if (p.rot) k[i].rotate(p, stage[mine], cs[min(n, Q8_BLOCK - 1)], sub);
        if (n < count) {
            k_big = max(k_big, k[i].largest());
            v_big = max(v_big, v[i].largest());
        }
    }
    k_big = __reduce_max_sync(0xffffffffu, k_big);
    v_big = __reduce_max_sync(0xffffffffu, v_big);
    if (lane == 0) big[0][warp] = k_big, big[1][warp] = v_big;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) k_big = max(k_big, big[0][w]), v_big = max(v_big, big[1][w]);
    const float k_s = block_scale(k_big, there > 0, k_before), v_s = block_scale(v_big, there > 0, v_before);
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
        const int n = mine + i * WARPS * RPW;
        if (n >= count) continue;
#pragma unroll
        for (int c = 0; c < NV; ++c) {
            const int d = k[i].dim(sub, c);
            if (d >= p.hd) continue;
            const size_t at = (row0 + there + n) * p.hd + d;
            *reinterpret_cast<uint32_t *>(p.k + at) = codes_word(k[i].x[c].x, k[i].x[c].y, k[i].x[c].z, k[i].x[c].w, 1.0f / k_s);
            *reinterpret_cast<uint32_t *>(p.v + at) = codes_word(v[i].x[c].x, v[i].x[c].y, v[i].x[c].z, v[i].x[c].w, 1.0f / v_s);
        }
    }
    round_again(p.k + row0 * p.hd, there * p.hd, k_before / k_s);
    round_again(p.v + row0 * p.hd, there * p.hd, v_before / v_s);
    if (tid == 0) p.ks[row0 / Q8_BLOCK] = k_s, p.vs[row0 / Q8_BLOCK] = v_s;
}

template <typename T, int HD>
int launch_fast(const PrepParams &p, unsigned ctas, cudaStream_t stream) {
    const dim3 grid(ctas), block(THREADS);
    if (p.rot == 0) kestrel_launch(attn_prepare_q8_fast_kernel<T, HD, TURN_NONE>, grid, block, 0, stream, p);
    else if (p.rot_mode == 0) kestrel_launch(attn_prepare_q8_fast_kernel<T, HD, TURN_HALF>, grid, block, 0, stream, p);
    else kestrel_launch(attn_prepare_q8_fast_kernel<T, HD, TURN_NEXT>, grid, block, 0, stream, p);
    return kestrel_check_launch("attn_prepare_q8");
}

template <typename T>
int launch(const PrepParams &p, unsigned ctas, cudaStream_t stream) {
    const bool whole = p.rot == 0 || p.rot_mode == 1 || p.rot == p.hd;
    if (whole && p.hd == 64) return launch_fast<T, 64>(p, ctas, stream);
    if (whole && p.hd == 128) return launch_fast<T, 128>(p, ctas, stream);
    if (p.hd <= 128) kestrel_launch(attn_prepare_q8_kernel<T, 32, 1>, dim3(ctas), dim3(THREADS), 0, stream, p);
    else kestrel_launch(attn_prepare_q8_kernel<T, 32, 2>, dim3(ctas), dim3(THREADS), 0, stream, p);
    return kestrel_check_launch("attn_prepare_q8");
}

}  // namespace

KESTREL_API int kestrel_attn_prepare_q8(const float *partial, int S, long long slice_stride, const float *bias, const float *q_norm_w, const float *k_norm_w,
                                        float norm_eps, const float *inv_freq, int rot, int rot_mode, float rot_scale, const int *positions,
                                        const int *cu_seqlens, int nseq, const int *block_table, int table_width, int table_stride, int page_size,
                                        int cache_pages, void *k_cache, void *v_cache, float *k_scale, float *v_scale, void *q_out, int dtype, int T, int nq,
                                        int nkv, int hd, int write_kv, int described, kestrel_stream_t stream) {
    if (T == 0 || nseq == 0) return 0;
    KESTREL_REQUIRE(T > 0 && nseq > 0 && S > 0 && nq > 0 && nkv > 0, "attn_prepare_q8: bad sizes");
    KESTREL_REQUIRE(dtype == KESTREL_F32 || dtype == KESTREL_BF16, "attn_prepare_q8: unknown dtype %d", dtype);
    KESTREL_REQUIRE(hd > 0 && hd % 16 == 0 && hd <= 256, "attn_prepare_q8: head size %d is no multiple of 16 up to 256", hd);
    KESTREL_REQUIRE(rot >= 0 && rot <= hd && rot % 2 == 0, "attn_prepare_q8: rotary size %d does not fit head size %d", rot, hd);
    KESTREL_REQUIRE(rot == 0 || inv_freq, "attn_prepare_q8: rotation asked for without frequencies");
    KESTREL_REQUIRE(rot_mode == 0 || rot_mode == 1, "attn_prepare_q8: rotation mode %d is neither 0 (rotate-half) nor 1 (interleaved)", rot_mode);
    KESTREL_REQUIRE(page_size > 0 && page_size % Q8_BLOCK == 0, "attn_prepare_q8: pages of %d tokens are no whole blocks of %d", page_size, Q8_BLOCK);
    KESTREL_REQUIRE(table_width > 0 && table_stride >= table_width && cache_pages > 0, "attn_prepare_q8: block table of %d entries a row, %d apart, %d pages", table_width, table_stride, cache_pages);
    KESTREL_REQUIRE(slice_stride % 4 == 0 && (((uintptr_t)partial | (uintptr_t)q_out | (uintptr_t)bias | (uintptr_t)q_norm_w | (uintptr_t)k_norm_w |
                     (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0, "attn_prepare_q8: tensors must start on 16 bytes");
    PrepParams p = {};
    p.partial = partial; p.bias = bias; p.q_w = q_norm_w; p.k_w = k_norm_w; p.inv_freq = inv_freq; p.slice_stride = (size_t)slice_stride;
    p.positions = positions; p.cu = cu_seqlens; p.table = block_table; p.k = (int8_t *)k_cache; p.v = (int8_t *)v_cache; p.ks = k_scale; p.vs = v_scale;
    p.q_out = q_out; p.S = S; p.nseq = nseq; p.table_width = table_width; p.table_stride = table_stride; p.page_size = page_size;
    p.cache_pages = cache_pages; p.T = T; p.nq = nq; p.nkv = nkv; p.hd = hd; p.rot = rot; p.rot_mode = rot_mode; p.eps = norm_eps; p.rot_scale = rot_scale; p.described = described;
    // n tokens touch at most (n + 14) / 16 + 1 blocks, and no more than n
    const long long units = write_kv ? (T < ((long long)T + 30ll * nseq) / 16 ? (long long)T : ((long long)T + 30ll * nseq) / 16) : 0;
    KESTREL_REQUIRE(units * nkv + T < (1ll << 31), "attn_prepare_q8: %d tokens of %d requests exceed the grid", T, nseq);
    p.units = (int)units;
    const unsigned ctas = (unsigned)(units * nkv + T);
    return dtype == KESTREL_F32 ? launch<float>(p, ctas, stream) : launch<__nv_bfloat16>(p, ctas, stream);
}
