// Log probabilities of given tokens, the entropy, and the likeliest tokens of rows of logits.
//
// One pass over a row: every thread keeps the maximum m of its numbers, L = sum e^(x - m) and A = sum (x - m) e^(x - m), joined like any
// online softmax's states - the sums move to a larger maximum m' as L' = f L, A' = f (A + (m - m') L) with f = e^(m - m') - so that
//     log p(i) = (x_i - m) - log L,      entropy = log L - A / L,
// both without a difference of large numbers.  A row's distances, exponentials and sums are float32.
//
// The likeliest tokens come from the threads' maxima, which the pass has made anyway: a value T that at least `top` threads' maxima reach
// is at most the top-th largest number, so only threads whose maximum reaches T hold candidates.  T is the top-th largest among the two
// largest maxima of every warp: no more than its threads', and found in two steps.  A thread remembers the largest of its runs of 16 numbers, and the largest number outside that run:
// most candidates' threads read one run again, all at once, and the warps of the others all of their numbers.  Rows with very many equal
// numbers leave more candidates than there is room for; their warps keep the best, one a lane, in order.  Equal numbers go by index.
//
// A row is one block's, or a cluster's of up to 8; a cluster's blocks meet once, in the first block's shared memory.  Bound by the row's
// bytes; a number costs half a maximum, an add, a product, an exponential, an add, a bound and a multiply-add.  Rows of 151,936 numbers:
// 1,024 of them (622 MB) 112 us, 5.5 TB/s, 64 12 us, 3.3 TB/s, and one 9 us, which is the latency of a pass and of picking the likeliest.
#include "common.cuh"

#include <math.h>

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32, MOST = KESTREL_LOGPROBS_MAX_TOP, MAX_CLUSTER = 8;
constexpr int FLIGHT = 4;               // vectors of four numbers that a thread has in flight: a run
constexpr int ROOM = 512;               // candidates of a block
constexpr float LOG2E = 1.4426950408889634f;

struct State {
    float m, l, a;                      // m = -inf: nothing but -inf so far
    __device__ __forceinline__ void rise(float to) {
        if (to > m) {
            const float f = m == -INFINITY ? 0.f : exp2f((m - to) * LOG2E);
            a = f == 0.f ? 0.f : f * fmaf(m - to, l, a);
            l *= f;
            m = to;
        }
    }
    // the state against a maximum that is at least its own; sums that are no numbers stay that
    __device__ __forceinline__ void move(float to) {
        const float f = m == -INFINITY ? 0.f : exp2f((m - to) * LOG2E);
        a = f == 0.f && a == a ? 0.f : f * fmaf(m - to, l, a);
        l = f == 0.f && l == l ? 0.f : f * l;
        m = to;
    }
    // over the first n lanes of a warp, n a power of two: every lane has all of it
    __device__ __forceinline__ void over(int n) {
        float to = m;
        for (int o = n / 2; o > 0; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, o));
        move(to);
        for (int o = n / 2; o > 0; o >>= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, o);
            a += __shfl_xor_sync(0xffffffffu, a, o);
        }
    }
};

// order of the numbers as that of unsigned integers, never 0; what is no number counts as minus infinity, as the threads' maxima have it
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x == x ? x + 0.f : -INFINITY);       // -0 counts as 0
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return k ? k : 1u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// larger numbers first, equal ones by index
__device__ __forceinline__ uint64_t entry_of(float x, uint32_t i) { return (uint64_t)key_of(x) << 32 | (uint32_t)~i; }

__device__ __forceinline__ void add(State &s, float x, float m_use) {
    const float d = x - m_use;                                      // first the difference: the lowest number times anything is -inf
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * LOG2E));
    s.l += e;
    s.a = fmaf(e, fmaxf(d, -1e30f), s.a);                           // e is 0 where d is -inf
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t in_first(const void *p) {       // this address in the cluster's first block
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(0));
    return r;
}

// A warp's best `top` entries, one a lane, best first; e: a lane's new entry, 0 for none
__device__ __forceinline__ void keep(uint64_t &best, uint64_t e, int top, int lane) {
    const uint64_t last = __shfl_sync(0xffffffffu, best, top - 1);
    for (uint32_t rest = __ballot_sync(0xffffffffu, e > last); rest; rest &= rest - 1) {
        const uint64_t c = __shfl_sync(0xffffffffu, e, __ffs(rest) - 1);
        const int at = __popc(__ballot_sync(0xffffffffu, best > c));
        const uint64_t up = __shfl_up_sync(0xffffffffu, best, 1);
        if (lane == at) best = c;
        else if (lane > at) best = up;
    }
}

__global__ void __launch_bounds__(THREADS, 2)
token_logprobs_kernel(const float *__restrict__ logits, long long ld, int V, int cluster, const int *__restrict__ ids, int top, float *__restrict__ logprobs,
                      float *__restrict__ entropy, int *__restrict__ top_ids, float *__restrict__ top_logprobs) {
    pdl_launch_dependents();
    __shared__ State joined[MAX_CLUSTER], parts[WARPS];
    __shared__ uint64_t found[ROOM], block_best[MAX_CLUSTER * MOST];
    __shared__ int n_found, place[MAX_CLUSTER * MOST];
    __shared__ uint32_t maxima[2 * WARPS];
    static_assert(ROOM >= WARPS * MOST && ROOM == THREADS && 2 * WARPS == 32 && MOST == 32, "a thread an entry, room for what all warps keep, a lane a maximum");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x / cluster, rank = cluster > 1 ? (int)cluster_rank() : 0;
    const float *x = logits + (size_t)row * ld;
    // numbers in front of the first 16-byte boundary and behind the last vector go to single threads of the first and last block
    const int head = min(V, (int)((16 - ((uintptr_t)x & 15)) & 15) / 4), nv = (V - head) / 4;
    const float4 *xv = reinterpret_cast<const float4 *>(x + head);
    const int v0 = (int)((long long)nv * rank / cluster), v1 = (int)((long long)nv * (rank + 1) / cluster);
    int odd = -1;                       // index of this thread's number outside the vectors
    if (rank == 0 && tid < head) odd = tid;
    if (rank == cluster - 1 && tid >= 4 && tid - 4 < V - head - 4 * nv) odd = head + 4 * nv + tid - 4;
    if (tid == 0) n_found = 0;
    if (cluster > 1) cluster_arrive();  // the first block's shared memory may be written once every block has begun
    pdl_wait();
    float given = __uint_as_float(0x7fc00000u);
    if (ids && rank == 0 && tid == 0) {
        const int id = ids[row];
        if (id >= 0 && id < V) given = x[id];
    }

    State s = {-INFINITY, 0.f, 0.f};
    float big = -INFINITY, other = -INFINITY;       // this thread's largest number, and the largest outside its run
    int run = -1;                       // the run's first vector; -1: the number outside the vectors
    if (odd >= 0) {
        const float o = x[odd];
        big = fmaxf(big, o);
        s.rise(big);
        add(s, o, s.m == -INFINITY ? 0.f : s.m);
    }
    for (int v = v0 + tid; v < v1; v += FLIGHT * THREADS) {
        float4 q[FLIGHT];
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i)
            q[i] = v + i * THREADS < v1 ? __ldcs(xv + v + i * THREADS) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i) mx = fmaxf(fmaxf(fmaxf(mx, q[i].x), fmaxf(q[i].y, q[i].z)), q[i].w);
        if (mx > big) other = big, big = mx, run = v;
        else other = fmaxf(other, mx);
        s.rise(mx);
        const float m_use = s.m == -INFINITY ? 0.f : s.m;
#pragma unroll
        for (int i = 0; i < FLIGHT; ++i) {
            add(s, q[i].x, m_use);
            add(s, q[i].y, m_use);
            add(s, q[i].z, m_use);
            add(s, q[i].w, m_use);
        }
    }
    if (cluster > 1) cluster_wait();
    // the block's state
    State w = s;
    w.over(32);
    if (lane == 0) parts[warp] = w;

    if (top > 0) {
        // T: the top-th largest of the warps' two largest maxima each, which are as many threads'
        const bool some = odd >= 0 || v0 + tid < v1;
        const uint32_t mine = some ? key_of(big) : 0u;
        const uint32_t m1 = __reduce_max_sync(0xffffffffu, mine);
        const int at1 = __ffs(__ballot_sync(0xffffffffu, mine == m1)) - 1;
        const uint32_t m2 = __reduce_max_sync(0xffffffffu, lane == at1 ? 0u : mine);
        if (lane < 2) maxima[2 * warp + lane] = lane ? m2 : m1;
        __syncthreads();
        const uint32_t v = maxima[lane];
        int better = 0;
#pragma unroll 4
        for (int i = 0; i < 32; ++i) {
            const uint32_t u = __shfl_sync(0xffffffffu, v, i);
            better += u > v || (u == v && i < lane);
        }
        const uint32_t T = max(__shfl_sync(0xffffffffu, v, __ffs(__ballot_sync(0xffffffffu, better == top - 1)) - 1), 1u);
        auto offer = [&](float e, int i) {
            if (key_of(e) >= T) {
                const int at = atomicAdd(&n_found, 1);
                if (at < ROOM) found[at] = entry_of(e, i);
            }
        };
        if (mine >= T && odd >= 0) offer(x[odd], odd);
        const bool several = mine >= T && (key_of(other) >= T || run < 0);       // (numbers that are none have no run)
        if (mine >= T && !several) {
            float4 q[FLIGHT];
#pragma unroll
            for (int i = 0; i < FLIGHT; ++i)
                if (run + i * THREADS < v1) q[i] = xv[run + i * THREADS];
#pragma unroll
            for (int i = 0; i < FLIGHT; ++i) {
                const int at = run + i * THREADS;
                if (at >= v1) break;
                offer(q[i].x, head + 4 * at);
                offer(q[i].y, head + 4 * at + 1);
                offer(q[i].z, head + 4 * at + 2);
                offer(q[i].w, head + 4 * at + 3);
            }
        }
        // threads with candidates in several runs: their warp reads all of their numbers
        for (uint32_t rest = __ballot_sync(0xffffffffu, several); rest; rest &= rest - 1) {
            const int l = __ffs(rest) - 1;
            for (int at = v0 + 32 * warp + l + lane * THREADS; at < v1; at += 32 * THREADS) {
                const float4 q = xv[at];
                offer(q.x, head + 4 * at);
                offer(q.y, head + 4 * at + 1);
                offer(q.z, head + 4 * at + 2);
                offer(q.w, head + 4 * at + 3);
            }
        }
        __syncthreads();
        if (n_found > ROOM) {               // too many: every warp keeps the best of its threads'
            __syncthreads();
            if (tid == 0) n_found = 0;
            uint64_t best = 0;
            for (uint32_t rest = __ballot_sync(0xffffffffu, mine >= T); rest; rest &= rest - 1) {
                const int l = __ffs(rest) - 1;
                const int l_odd = __shfl_sync(0xffffffffu, odd, l);
                if (l_odd >= 0) keep(best, lane == 0 ? entry_of(x[l_odd], l_odd) : 0, top, lane);
                for (int v = v0 + 32 * warp + l; v < v1; v += 32 * THREADS) {
                    const int at = v + lane * THREADS;
                    float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (at < v1) q = xv[at];
                    const float e[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) keep(best, at < v1 && key_of(e[j]) >= T ? entry_of(e[j], head + 4 * at + j) : 0, top, lane);
                }
            }
            __syncthreads();
            if (best && lane < top) found[atomicAdd(&n_found, 1)] = best;
            __syncthreads();
        }
        // each goes to the place that the number of better ones gives it
        const int n = n_found;
        if (tid < n) {
            const uint64_t e = found[tid];
            int at = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) at += found[j] > e;
            if (at < top) {
                if (cluster > 1) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(in_first(block_best + rank * MOST + at)), "l"(e) : "memory");
                else block_best[at] = e;
            }
        }
        for (int i = n + tid; i < top; i += THREADS) {              // a block with fewer numbers than that
            if (cluster > 1) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(in_first(block_best + rank * MOST + i)), "l"(0ull) : "memory");
            else block_best[i] = 0;
        }
    }
    __syncthreads();
    if (warp == 0) {
        State b = parts[lane % WARPS];
        b.over(WARPS);
        if (lane == 0) {
            if (cluster > 1) {
                const uint32_t to = in_first(joined + rank);
                asm volatile("st.shared::cluster.f32 [%0], %1;\n\tst.shared::cluster.f32 [%0 + 4], %2;\n\tst.shared::cluster.f32 [%0 + 8], %3;"
                             ::"r"(to), "f"(b.m), "f"(b.l), "f"(b.a) : "memory");
            } else {
                joined[0] = b;
            }
        }
    }
    if (cluster > 1) {
        cluster_arrive();
        cluster_wait();
    } else {
        __syncthreads();
    }
    if (rank != 0) return;
    State r = joined[lane & (cluster - 1)];
    r.over(cluster);
    const float log_l = logf(r.l), m_use = r.m == -INFINITY ? 0.f : r.m;
    if (tid == 0) {
        if (entropy) entropy[row] = log_l - r.a / r.l;
        if (ids) logprobs[row] = (given - m_use) - log_l;
    }
    // An entry's place: its own in its block's list, and of every other list, which are in order, as many as a search by halves finds; a
    // thread a pair of entry and list.  (Rolled: what runs once a row costs what its code takes to arrive.)
    if (cluster > 1) {
        if (tid < MAX_CLUSTER * MOST) place[tid] = 0;
        __syncthreads();
#pragma unroll 1
        for (int j = tid; j < cluster * MOST * cluster; j += THREADS) {
            const int i = j / cluster, c = j & (cluster - 1);
            if (i % MOST >= top || i / MOST == c) continue;
            const uint64_t e = block_best[i], *list = block_best + c * MOST;
            int n = 0;
#pragma unroll 1
            for (int step = MOST; step > 0; step /= 2)
                if (n + step <= top && list[n + step - 1] > e) n += step;
            if (n) atomicAdd(&place[i], n);
        }
        __syncthreads();
    }
#pragma unroll 1
    for (int i = tid; i < cluster * MOST; i += THREADS) {
        const uint64_t e = block_best[i];
        const int at = i % MOST + (cluster > 1 ? place[i] : 0);
        if (i % MOST < top && e && at < top) {
            top_ids[(size_t)row * top + at] = (int)~(uint32_t)e;
            top_logprobs[(size_t)row * top + at] = (value_of((uint32_t)(e >> 32)) - m_use) - log_l;
        }
    }
}

}  // namespace

KESTREL_API int kestrel_token_logprobs(const float *logits, long long ld, int R, int V, const int *ids, int top, float *logprobs, float *entropy, int *top_ids,
                                       float *top_logprobs, kestrel_stream_t stream) {
    if (R == 0) return 0;
    KESTREL_REQUIRE(R > 0 && V > 0 && ld >= V, "token_logprobs: %d rows of %d logits, %lld apart", R, V, ld);
    KESTREL_REQUIRE(top >= 0 && top <= MOST && top <= V, "token_logprobs: the %d likeliest of %d; at most %d are picked", top, V, MOST);
    KESTREL_REQUIRE((!ids || logprobs) && (top == 0 || (top_ids && top_logprobs)), "token_logprobs: no place for the results");
    KESTREL_REQUIRE(((uintptr_t)logits & 3) == 0, "token_logprobs: logits must start on 4 bytes");
    // Blocks of a row: while twice as many would still be resident at once, two an SM.  (128 rows of 151,936, 20 likeliest: 17.5 us with clusters
    // of 2, 24.3 and 24.1 with 1 and 4; 64 rows 12.2 with 4, 15.8 and 24.4 with 2 and 8; 1,024 rows 116 with one block, 137 with clusters of
    // 2, although these leave the last round fuller.)
    int cluster = 1;
    while (cluster < MAX_CLUSTER && (long long)R * cluster * 2 <= 2ll * kestrel_sms() && V / (cluster * 2) >= 1024) cluster *= 2;
    KESTREL_REQUIRE((long long)R * cluster < (1ll << 31), "token_logprobs: %d rows exceed the grid", R);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)R * cluster);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_kestrel_pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, token_logprobs_kernel, logits, ld, V, cluster, ids, top, logprobs, entropy, top_ids, top_logprobs);
    return kestrel_check_launch("token_logprobs");
}
