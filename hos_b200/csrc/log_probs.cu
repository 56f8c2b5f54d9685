// Log probabilities of given tokens, the entropy, and the likeliest tokens, from rows of logits.
//
// Of a row l: M = max l, S = sum e^(l - M), U = sum e^(l - M) (l - M) (moments.cuh).  A thread keeps them of what it has seen and, when
// its maximum grows by d, takes S to S e^-d and U to (U - S d) e^-d, so the logits are read once.  All of it is held in 32 bits; a
// thread adds some hundred terms, trees the rest.
//
// The likeliest k tokens in the same pass.  A number and its token make a key of 64 bits, larger for larger numbers and, of equal
// ones, for lower tokens: keys are all different, so ties, rows ruled out (-inf) and rows that hold one number only need no path of
// their own.  The block keeps a threshold that at least k of its keys so far reach, and a list of those that do.  The first threshold
// is found by halving an interval of keys until between k and 2k of the THREADS' largest keys reach it; after that few numbers are
// anywhere near, and a tile costs a comparison a thread.  A list that grows is cut back by halving again; a tile that brings more
// keys than the list holds (numbers in rising order) gets a threshold of its own first.
//
// A row is one block's, or is cut over a cluster of 2 to 8 blocks whose first merges what they leave in shared memory: nothing is
// kept in device memory, and every sum has a fixed order.
#include "common.cuh"
#include "moments.cuh"

namespace hos {

constexpr int kMostTop = 32;                           // alternatives a row
constexpr int kEach = 32;                              // numbers that a thread holds of a tile
constexpr int kCompactAbove = 128;                     // keys in the list after which it is cut back
constexpr int kListRoom = kCompactAbove + 2 * kMostTop * kEach;

typedef unsigned long long Key;

// Larger numbers have larger keys, of equal numbers the one of the lower token; not-a-number counts as -inf.
__device__ __forceinline__ Key key_of(float v, int token) {
    v = v == v ? v + 0.f : -INFINITY;                  // (-0 and 0 are equal numbers)
    const uint32_t b = __float_as_uint(v);
    const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (Key)up << 32 | (uint32_t)~token;
}
__device__ __forceinline__ float key_number(Key k) {
    const uint32_t up = (uint32_t)(k >> 32);
    return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
// What a thread's largest number is compared with: no number that is less has a key that reaches k.
__device__ __forceinline__ float least_of(Key k) {
    const float v = key_number(k);
    return v == v ? v : -INFINITY;                     // (below every number's keys)
}
__device__ __forceinline__ int key_token(Key k) { return (int)~(uint32_t)k; }

struct LogProbArgs {
    const float* logits;
    long long stride;
    int vocab;
    const int* tokens;
    float* logprob;
    float* entropy;
    int top;
    int* top_ids;
    float* top_logprobs;
};

struct LogProbShared {
    Key list[kListRoom];
    Key best[kMostTop];              // a block's likeliest, sorted; in the end the first block's: all blocks'
    Key warp_key[32];
    Moments part[32];
    Moments all;
    Key threshold;
    int count;
};

__device__ __forceinline__ uint32_t cluster_address(const void* p, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ float cluster_float(uint32_t a) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ Key cluster_key(uint32_t a) {
    Key v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A key that between `top` and 2 top of the counted keys reach, or, where they cannot be told apart so (fewer keys than `top`), the
// lowest that they all do.  count_at(k): how many keys are >= k, the same answer to every thread, with a barrier inside.
template <typename Count>
__device__ __forceinline__ Key halved(Key lo, Key hi, int top, Count count_at) {
    while (hi - lo > 1) {                              // at least `top` keys reach lo (or all do), fewer reach hi
        const Key mid = lo + (hi - lo) / 2;
        const int n = count_at(mid);
        if (n >= top) {
            lo = mid;
            if (n <= 2 * top) break;
        } else {
            hi = mid;
        }
    }
    return lo;
}

template <int THREADS, bool TOP>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) log_probs_kernel(LogProbArgs a, int blocks) {
    __shared__ LogProbShared sh;
    pdl_enter();
    const int row = blockIdx.x / blocks, rank = blockIdx.x % blocks;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int WARPS = THREADS / 32;
    const int token = a.tokens[row];
    const bool padding = token < 0 || token >= a.vocab;          // the whole cluster's, like the row
    if (padding) {
        if (rank == 0) {
            if (tid == 0) a.logprob[row] = a.entropy[row] = 0.f;
            for (int i = tid; TOP && i < a.top; i += THREADS) {
                a.top_ids[(size_t)row * a.top + i] = -1;
                a.top_logprobs[(size_t)row * a.top + i] = 0.f;
            }
        }
        return;
    }
    const float* l = a.logits + (size_t)row * a.stride;
    // vectors of four on 16 bytes: the first begins up to three numbers before the row
    const int before = (int)(((uintptr_t)l & 15) >> 2);
    const int vectors = (a.vocab + before + 3) / 4;
    const int per_block = (vectors + blocks - 1) / blocks;
    const int v0 = rank * per_block, v1 = min(vectors, v0 + per_block);
    if (TOP && tid == 0) { sh.count = 0; sh.threshold = 0; }
    Moments mine{-INFINITY, 0.f, 0.f};
    if (TOP) __syncthreads();
    Key threshold = 0;
    float least = -INFINITY;                                     // the threshold's number: less than that is no candidate
    bool first = true;

    // the tiles are a block's in rising order of tokens; every thread of the block walks over all of them
    for (int base = v0; base < v1; base += THREADS * (kEach / 4)) {
        float x[kEach];
#pragma unroll
        for (int j = 0; j < kEach / 4; ++j) {
            const int v = base + j * THREADS + tid, i = 4 * v - before;
            if (v < v1 && i >= 0 && i + 4 <= a.vocab) {
                const float4 f = *reinterpret_cast<const float4*>(l + i);
                x[4 * j] = f.x; x[4 * j + 1] = f.y; x[4 * j + 2] = f.z; x[4 * j + 3] = f.w;
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) x[4 * j + c] = v < v1 && i + c >= 0 && i + c < a.vocab ? l[i + c] : -INFINITY;
            }
        }
        float most = x[0];
#pragma unroll
        for (int j = 1; j < kEach; ++j) most = fmaxf(most, x[j]);
        add_to(mine, x, most);
        if (!TOP) continue;

        // ---- candidates of this tile ----
        if (!__syncthreads_or(first || !(most < least))) continue;
        auto token_at = [&](int j) { return 4 * (base + (j >> 2) * THREADS + tid) - before + (j & 3); };
        auto inside = [&](int j) { return base + (j >> 2) * THREADS + tid < v1 && token_at(j) >= 0 && token_at(j) < a.vocab; };
        auto largest = [&]() {                                   // this thread's largest key of the tile
            Key k = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j)
                if (inside(j)) k = max(k, key_of(x[j], token_at(j)));
            return k;
        };
        auto from_maxima = [&]() {                               // a threshold by the threads' largest keys of this tile
            const Key k = largest();
            Key hi = k;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            if (lane == 0) sh.warp_key[warp] = hi;
            __syncthreads();
            hi = lane < WARPS ? sh.warp_key[lane] : 0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            return halved(0, hi + 1, a.top, [&](Key at) { return __syncthreads_count(k >= at); });
        };
        auto push = [&]() {
            if (!(most < least)) {
#pragma unroll
                for (int j = 0; j < kEach; ++j)
                    if (inside(j)) {
                        const Key k = key_of(x[j], token_at(j));
                        if (k >= threshold) {
                            const int at = atomicAdd(&sh.count, 1);
                            if (at < kListRoom) sh.list[at] = k;
                        }
                    }
            }
            __syncthreads();
        };
        if (first) {
            threshold = from_maxima();
            first = false;
            least = least_of(threshold);
        }
        const int held = sh.count;                               // (nobody adds to it before the barrier that is next)
        __syncthreads();
        push();
        if (sh.count > kListRoom) {                              // too many: no more than 2 top threads' numbers with this tile's own threshold
            __syncthreads();
            if (tid == 0) sh.count = held;
            threshold = max(threshold, from_maxima());
            least = least_of(threshold);
            __syncthreads();
            push();
        }
        if (sh.count > kCompactAbove) {
            const int n = sh.count;
            auto count_at = [&](Key at) {
                int c = 0;
                for (int i = tid; i < n; i += THREADS) c += sh.list[i] >= at;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
                __syncthreads();
                if (lane == 0) sh.warp_key[warp] = c;
                __syncthreads();
                c = 0;
                for (int w = 0; w < WARPS; ++w) c += (int)sh.warp_key[w];
                return c;
            };
            threshold = max(threshold, halved(threshold, ~0ull, a.top, count_at));
            least = least_of(threshold);
            // the keys that reach it, moved to the front: a round of threads at a time, read before any is written
            if (tid == 0) sh.count = 0;
            for (int i0 = 0; i0 < n; i0 += THREADS) {
                const Key k = i0 + tid < n ? sh.list[i0 + tid] : 0;
                __syncthreads();
                if (i0 + tid < n && k >= threshold) sh.list[atomicAdd(&sh.count, 1)] = k;
            }
            __syncthreads();
        }
    }

    // ---- the block's moments, and its likeliest in order ----
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        mine = joined(mine, Moments{__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o),
                                    __shfl_xor_sync(0xffffffffu, mine.u, o)});
    if (lane == 0) sh.part[warp] = mine;
    if (TOP && tid < kMostTop) sh.best[tid] = 0;
    __syncthreads();
    if (warp == 0) {
        mine = lane < WARPS ? sh.part[lane] : Moments{-INFINITY, 0.f, 0.f};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            mine = joined(mine, Moments{__shfl_xor_sync(0xffffffffu, mine.m, o), __shfl_xor_sync(0xffffffffu, mine.s, o),
                                        __shfl_xor_sync(0xffffffffu, mine.u, o)});
        if (lane == 0) sh.all = mine;
    }
    // a key's place is how many are larger
    auto sort_list = [&](const Key* from, int n, Key* to) {
        for (int i = tid; i < n; i += THREADS) {
            const Key k = from[i];
            int larger = 0;
            for (int j = 0; j < n; ++j) larger += from[j] > k;
            if (larger < a.top && k != 0) to[larger] = k;
        }
    };
    if (TOP) sort_list(sh.list, sh.count, sh.best);
    if (blocks > 1) {
        cluster_meet();
        if (rank == 0) {
            if (tid == 0) {
                Moments r = sh.all;
                for (int b = 1; b < blocks; ++b)
                    r = joined(r, Moments{cluster_float(cluster_address(&sh.all.m, b)), cluster_float(cluster_address(&sh.all.s, b)),
                                          cluster_float(cluster_address(&sh.all.u, b))});
                sh.all = r;
            }
            if (TOP) {
                for (int i = tid; i < blocks * kMostTop; i += THREADS) sh.list[i] = cluster_key(cluster_address(&sh.best[i % kMostTop], i / kMostTop));
                __syncthreads();
                if (tid < kMostTop) sh.best[tid] = 0;
                __syncthreads();
                sort_list(sh.list, blocks * kMostTop, sh.best);
            }
        }
        cluster_meet();                                          // nobody leaves while its memory is read
        if (rank != 0) return;
    }
    __syncthreads();
    const Moments r = sh.all;
    const float log_s = logf(r.s);
    if (tid == 0) {
        a.logprob[row] = (l[token] - r.m) - log_s;
        a.entropy[row] = log_s - r.u / r.s;
    }
    if (TOP && tid < a.top) {
        const Key k = sh.best[tid];
        a.top_ids[(size_t)row * a.top + tid] = k != 0 ? key_token(k) : -1;
        a.top_logprobs[(size_t)row * a.top + tid] = k != 0 ? (l[key_token(k)] - r.m) - log_s : 0.f;
    }
}

template <int THREADS, bool TOP>
static int launch_log_probs(const LogProbArgs& a, int rows, int blocks, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)rows * blocks);
    cfg.blockDim = dim3(THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, log_probs_kernel<THREADS, TOP>, a, blocks);
    return check_launch("log_probs");
}

}  // namespace hos

using namespace hos;

extern "C" const char* hos_last_error() { return error_buffer(); }

// Per row of float32 logits (`stride` numbers from row to row): the log probability of tokens[row] and the entropy; with `top`,
// the likeliest `top` tokens (of equal ones the lower first) and their log probabilities.  A row whose token is outside the vocabulary
// is padding: zeros, tokens -1.  `blocks` (1, 2, 4 or 8) of `threads` (256 or 1024) threads share a row.
extern "C" int hos_log_probs(const float* logits, long long stride, int rows, int vocab, const int* tokens, float* logprob,
                             float* entropy, int top, int* top_ids, float* top_logprobs, int threads, int blocks,
                             cudaStream_t stream) {
    if (rows <= 0) return 0;
    if (vocab < 1 || stride < vocab) HOS_REFUSE("log_probs: a vocabulary of %d in rows %lld numbers apart", vocab, stride);
    if (vocab > (1 << 30)) HOS_REFUSE("log_probs: a vocabulary of %d (at most 2^30)", vocab);
    if (top < 0 || top > kMostTop || top > vocab) HOS_REFUSE("log_probs: %d alternatives of %d tokens (at most %d)", top, vocab, kMostTop);
    if ((long long)rows * blocks > (1ll << 31) - 1) HOS_REFUSE("log_probs: %d rows", rows);
    if (blocks != 1 && blocks != 2 && blocks != 4 && blocks != 8) HOS_REFUSE("log_probs: %d blocks a row", blocks);
    const LogProbArgs a{logits, stride, vocab, tokens, logprob, entropy, top, top_ids, top_logprobs};
    if (threads == 1024) return top ? launch_log_probs<1024, true>(a, rows, blocks, stream) : launch_log_probs<1024, false>(a, rows, blocks, stream);
    if (threads == 256) return top ? launch_log_probs<256, true>(a, rows, blocks, stream) : launch_log_probs<256, false>(a, rows, blocks, stream);
    HOS_REFUSE("log_probs: blocks of %d threads", threads);
}
