// Attention over pages of int8 codes: what its kernels share (attention_q8.cu, attention_q8_decode.cu, attention_q8_tc.cu).
//
// A plane of the cache is codes [pages, kv heads, page size, head size], int8 in [-127, 127], and scales [pages, kv heads, page size / 16],
// float32: a value is code * scale, and the 16 tokens of a block share the scale of their head.  With s_k and s_v the scales of key j's
// block, the output of a query row is
//     o = sum_j p_j s_v(j) c_v(j),   p = softmax_j( scale * s_k(j) * (q . c_k(j)) )
// over the keys j that the row may see.  The tensor cores multiply codes, which are exact in float16; the scales enter with the scores.
// With x_j the score in base-2 units the tensor-core kernels hold
//     w_j = 2^(x_j + log2 s_v(j) - m),   out = sum_j w_j c_v(j),   l = sum_j w_j / s_v(j),
// so that w_j, rounded to float16 for the second product, lies in [0, 2^8] whatever the size of the values, one exponential serves both
// sums, and (m, l, out) of two key ranges merge as those of any online softmax.  o = out / l.  (float32: attention_q8_decode.cu.)
#pragma once
#include "common.cuh"

#define Q8_BLOCK KESTREL_Q8_BLOCK

// The tensor-core kernels mask a key by a score of minus infinity, which a product with zero would turn into no number.  So a block's scale
// counts as 2^-64 at least, which is what an append writes at least, and a row's factor as 2^-84: their product is a float32 number.  What
// that changes is a value of 2^-57 at most, and a score of 2^-63 times its block's scale at most.
constexpr float Q8_LEAST_SCALE = 5.421010862427522e-20f, Q8_LEAST_FACTOR = 5.169878828456423e-26f;

struct Q8Params {
    const void *q;                  // [T, nq * hd] float32 or bfloat16
    void *out;                      // [T, nq * hd], as q
    const int8_t *k, *v;            // [pages, nkv, page_size, hd]
    const float *ks, *vs;           // [pages, nkv, page_size / Q8_BLOCK]
    float *part_o;                  // [T * nq, slices, hd]   (slices > 1)
    float *part_ml;                 // [T * nq, slices, 2]
    const int *cu_seqlens;          // [nseq + 1] first token of each request in this step
    const int *kv_lens;             // [nseq] request length after this step
    const int *block_table;         // [nseq, table_stride], table_width entries of a row are read
    int nseq, table_width, table_stride, page_size, cache_pages, nq, nkv, hd, window, slices;
    int rows_above, rows_upto;      // this launch takes the requests with rows_above < (token, head) rows per kv head <= rows_upto
    int rows_per_tile, row_tiles;   // row_tiles: most of a request
    int tiles;                      // row tiles of all requests, or the requests where row_tiles is 1
    int page_shift;                 // log2 of the page size, or -1
    int described;                  // the step's description was on the device before the kernel in front of this one began
    float scale;
};

// What a CTA works on: rows [row0, row0 + rows) - (token, query head of the kv head's group) pairs, token-major - of one request.
struct Q8Tile {
    int seq, row0, rows, tok_begin, pos_begin, G;
    int k_first, k_end;             // keys that some row of the tile may see: [k_first, k_end)
    const int *table;
};

// The tile-th tile among those of the requests that this launch takes; false if there are fewer (a step with fewer requests than the grid
// was made for).  All lanes of a warp take part.
__device__ __forceinline__ bool q8_find_tile(const Q8Params &p, int tile, Q8Tile &t) {
    const int lane = threadIdx.x & 31, G = p.nq / p.nkv;
    int left = tile;
    for (int base = 0; base < p.nseq; base += 32) {
        const int i = base + lane;
        int n = 0;
        if (i < p.nseq) {
            const long long rows = (long long)(p.cu_seqlens[i + 1] - p.cu_seqlens[i]) * G;
            if (rows > p.rows_above && rows <= p.rows_upto) n = (int)((rows + p.rows_per_tile - 1) / p.rows_per_tile);
        }
        int end = n;                // tiles of the requests up to this lane's
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o) end += x;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, left < end);
        if (behind) {
            const int at = __ffs(behind) - 1;
            t.seq = base + at;
            t.row0 = (left - __shfl_sync(0xffffffffu, end - n, at)) * p.rows_per_tile;
            t.G = G;
            t.tok_begin = p.cu_seqlens[t.seq];
            const int n_tok = p.cu_seqlens[t.seq + 1] - t.tok_begin;
            t.pos_begin = p.kv_lens[t.seq] - n_tok;
            t.rows = min(p.rows_per_tile, n_tok * G - t.row0);
            t.table = p.block_table + (size_t)t.seq * p.table_stride;
            const int first_tok = t.row0 / G, last_tok = (t.row0 + t.rows - 1) / G;
            t.k_first = p.window > 0 ? max(0, t.pos_begin + first_tok - p.window + 1) : 0;
            t.k_end = t.pos_begin + last_tok + 1;
            return true;
        }
        left -= __shfl_sync(0xffffffffu, end, 31);
    }
    return false;
}

// The keys of one slice of a tile: its keys, from the first key tile of `align` keys that they touch, cut evenly.
__device__ __forceinline__ void q8_slice(const Q8Tile &t, int slices, int slice, int align, int &lo, int &hi) {
    const int from = t.k_first / align * align;
    const int per = ((t.k_end - from + slices - 1) / slices + align - 1) / align * align;
    lo = max(t.k_first, min(t.k_end, from + slice * per));
    hi = min(t.k_end, from + (slice + 1) * per);
}

// Row (in units of one token's codes of one head) of the first token of the block that holds position `pos`; a released or absent page,
// whose keys no row may see, stands for page 0.
__device__ __forceinline__ int q8_row_of(const Q8Params &p, const int *table, int kvh, int pos) {
    const int idx = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
    int page = idx < p.table_width ? table[idx] : 0;
    if (page < 0 || page >= p.cache_pages) page = 0;
    return (page * p.nkv + kvh) * p.page_size + (pos - idx * p.page_size) / Q8_BLOCK * Q8_BLOCK;       // below 2^31: checked on the host
}

__device__ __forceinline__ size_t q8_out_row(const Q8Params &p, const Q8Tile &t, int kvh, int r) {
    const int row = t.row0 + r;
    return (size_t)(t.tok_begin + row / t.G) * p.nq + kvh * t.G + row % t.G;
}

// attention_q8_decode.cu: requests of few rows and float32, head sizes 64 and 128; one or two kernels
enum Q8Form { Q8_EIGHT, Q8_SIXTEEN, Q8_WIDE_EIGHT, Q8_WIDE_SIXTEEN };      // tiles of 8 or 16 rows (Q8Params.rows_per_tile) of bfloat16, of float32
int q8_launch_decode(const Q8Params &p, Q8Form form, int ctas, cudaStream_t stream);
int q8_decode_ctas(long long tiles, int hd, Q8Form form);       // for so many (row tile, kv head, 64 keys)
// CTAs a pair (Q8Params.slices), or 0: ctas in stretches; exact: by the requests' own lengths, else by bounds of them
int q8_decode_cluster(long long pairs, int longest_tiles, long long tiles, int hd, Q8Form form, bool exact);
long long q8_decode_scratch(int ctas, int hd);          // floats: part_o, then part_ml
int q8_decode_error();                                  // its bounded waits' error word; synchronises
// attention_q8_tc.cu: tiles of up to 256 rows, head sizes 64 and 128, bfloat16
int q8_launch_tc(const Q8Params &p, int tiles, cudaStream_t stream);
int q8_tc_error();
// attention_q8.cu
int q8_launch_plain(const Q8Params &p, int dtype, int tiles, cudaStream_t stream);
int q8_launch_merge(const Q8Params &p, int dtype, int tiles, cudaStream_t stream);
