// Log probabilities, entropy and the most probable entries from logits.
//
// One pass over a row: every thread keeps a running maximum m, the sum S of e^(x - m) and T of (x - m) e^(x - m);
// then lse = m + ln S, ln p = (x - m) - ln S, entropy = ln S - T / S (both terms are positive: nothing cancels).
// The most probable entries are 64-bit keys of (value, index) whose order is the wanted one, held by a warp, lane i
// the i-th best; lists are sorted and merged by bitonic networks across the warp.
//
// What bounds it: the logits' bytes (2048 rows of 32000: 44 us, 6.0 TB/s); with places, and for few rows, latency.  A row is cut into slices where there are fewer rows than blocks fit the
// device; up to sixteen slices are the blocks of a cluster, which joins them, more are joined by a second kernel.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "qk_common.h"

namespace {

constexpr uint32_t kMaxTop = 32, kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kMinSlice = 2048;   // entries a block takes at least
constexpr uint32_t kHeld = 8;          // vectors of four entries that a thread keeps in registers
constexpr uint32_t kCandidates = 512;  // places for entries that may be among the best of a slice
constexpr uint32_t kWantBlocks = 148 * 8;  // (two waves of the form with places)
constexpr size_t kResident = 148 * 2, kMaxCluster = 16, kMaxSlice = 16384;  // (longer slices than that are for more blocks than a cluster has)
constexpr float kLog2E = 1.4426950408889634f;

struct LogProbArgs {
    const float *logits;
    size_t stride;
    uint32_t n_tokens, vocab, n_top, n_slices, slice;
    const int32_t *targets;
    float *lse, *logprob, *entropy, *top_logprob;
    int32_t *top_ids;
    uint32_t clustered;  // the slices of a row are the blocks of a cluster, which join them; else a second launch does:
    float *stats;        // [n_tokens][n_slices][4]: m, S, T
    uint64_t *keys;      // [n_tokens][n_slices][32]; where n_top > 0
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// x, at least -10000 (where ex2 gives 0, and 0 times it is 0); a NaN stays.
__device__ __forceinline__ float floored(float x) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(x), "f"(-10000.f));
    return y;
}
// An order on (value, index) as one number: larger is better, the lowest index first among equals (0 and -0 are).
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return ((uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return 0xffffffffu - (uint32_t)key; }
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// Lane i keeps the larger (keep_max) or smaller of its and its partner's key.
__device__ __forceinline__ uint64_t exchanged(uint64_t key, int partner_bit, bool keep_max) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, key, partner_bit);
    return (key > other) == keep_max ? key : other;
}
// 32 keys in falling order over the lanes.
__device__ __forceinline__ uint64_t sorted(uint64_t key, uint32_t lane) {
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int bit = size / 2; bit > 0; bit /= 2)
            key = exchanged(key, bit, ((lane & bit) == 0) == ((lane & size) == 0 || size == 32));
    return key;
}
// The best 32 of two lists in falling order, in falling order: the larger of a and the reversed b is a bitonic sequence.
__device__ __forceinline__ uint64_t merged(uint64_t a, uint64_t b, uint32_t lane) {
    const uint64_t r = __shfl_xor_sync(0xffffffffu, b, 31);
    uint64_t key = a > r ? a : r;
#pragma unroll
    for (int bit = 16; bit > 0; bit /= 2) key = exchanged(key, bit, (lane & bit) == 0);
    return key;
}

struct Stats {  // m, S = sum e^(x - m), T = sum (x - m) e^(x - m)
    float m, s, t;
};
// Two disjoint parts of a row as one.
__device__ __forceinline__ Stats joined(Stats a, Stats b) {
    const float m = fmaxf(a.m, b.m);
    if (!(m > -INFINITY)) return {m, a.s + b.s, a.t + b.t};  // (nothing possible in either; a NaN stays)
    const float da = a.m - m, db = b.m - m, wa = ex2(da * kLog2E), wb = ex2(db * kLog2E);
    Stats r{m, a.s * wa + b.s * wb, 0.f};
    r.t = (wa > 0.f ? wa * (a.t + da * a.s) : 0.f) + (wb > 0.f ? wb * (b.t + db * b.s) : 0.f);
    return r;
}

// A row's results from its statistics and its best entries (held by the lanes of one warp).
__device__ __forceinline__ void finish(const LogProbArgs &a, uint32_t row, Stats st, uint64_t best, uint32_t lane) {
    const float *x = a.logits + row * a.stride;
    const float nan = __int_as_float(0x7fffffff);
    // (an infinity makes the sums NaN, a NaN too)
    const bool ok = st.m > -INFINITY && st.s < INFINITY && st.t > -INFINITY;
    const float ln = logf(st.s);
    if (lane == 0) {
        if (a.lse) a.lse[row] = ok ? st.m + ln : nan;
        if (a.entropy) a.entropy[row] = ok ? ln - st.t / st.s : nan;
        if (a.logprob) {
            const int32_t id = a.targets[row];
            a.logprob[row] = id < 0 ? 0.f : !ok || (uint32_t)id >= a.vocab ? nan : (x[id] - st.m) - ln;
        }
    }
    if (lane < a.n_top) {
        const size_t at = (size_t)row * a.n_top + lane;
        if (a.top_ids) a.top_ids[at] = ok ? (int32_t)key_index(best) : -1;
        if (a.top_logprob) a.top_logprob[at] = ok ? (key_value(best) - st.m) - ln : nan;
    }
}

// A thread's statistics of values in registers; the block's in shared memory.
__device__ __forceinline__ void share(Stats st, Stats *part) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
        st = joined(st, Stats{__shfl_xor_sync(0xffffffffu, st.m, off), __shfl_xor_sync(0xffffffffu, st.s, off),
                              __shfl_xor_sync(0xffffffffu, st.t, off)});
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = st;
}
__device__ __forceinline__ Stats of_block(const Stats *part) {
    Stats st = part[0];
    for (uint32_t w = 1; w < kWarps; ++w) st = joined(st, part[w]);
    return st;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A shared-memory address of this block in the cluster's block `rank`.
__device__ __forceinline__ uint32_t of_rank(const void *p, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ float load_float(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint64_t load_key(uint32_t addr) {
    uint64_t v;
    asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(addr));
    return v;
}
// The blocks of a cluster are the slices of a row: the first one joins their statistics and best entries (`best`, in
// lanes; kTop) through distributed shared memory.  All threads; st and best are those of the first warp.
template <bool kTop>
__device__ __forceinline__ void join_cluster(const LogProbArgs &a, uint32_t row, uint32_t slice, Stats st, uint64_t best,
                                             Stats *shared_stats, uint64_t (*lists)[32]) {
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (warp == 0) {
        if (lane == 0) *shared_stats = st;
        if constexpr (kTop) lists[0][lane] = best;
    }
    cluster_sync();
    if (slice == 0) {
        st = Stats{-INFINITY, 0.f, 0.f};
        if (warp == 0 && lane < a.n_slices) {
            const uint32_t from = of_rank(shared_stats, lane);
            st = Stats{load_float(from), load_float(from + 4), load_float(from + 8)};
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1)  // (every lane needs them)
            st = joined(st, Stats{__shfl_xor_sync(0xffffffffu, st.m, off), __shfl_xor_sync(0xffffffffu, st.s, off),
                                  __shfl_xor_sync(0xffffffffu, st.t, off)});
        best = 0;
        if constexpr (kTop) {
            for (uint32_t i = warp; i < a.n_slices; i += kWarps)
                best = merged(best, load_key(of_rank(&lists[0][lane], i)), lane);
#pragma unroll
            for (uint32_t half = kWarps / 2; half > 0; half /= 2) {
                if (warp >= half && warp < 2 * half) lists[warp][lane] = best;
                __syncthreads();
                if (warp < half) best = merged(best, lists[warp + half][lane], lane);
            }
        }
        if (warp == 0) finish(a, row, st, best, lane);
    }
    cluster_sync();  // (no block ends while the first one reads it)
}

// Where a slice's 16-byte vectors lie: up to three single entries in front, up to three behind.
struct Extent {
    uint32_t lo, hi, head, vectors, tail;
    __device__ __forceinline__ Extent(const float *x, const LogProbArgs &a, uint32_t slice) {
        lo = slice * a.slice, hi = min(a.vocab, lo + a.slice);
        head = min(hi - lo, (uint32_t)((16 - ((uintptr_t)(x + lo) & 15)) & 15) / 4);
        vectors = (hi - lo - head) / 4, tail = hi - lo - head - 4 * vectors;
    }
    // The single entry of this thread (threads 0 .. 2 and 8 .. 10), or none.
    __device__ __forceinline__ uint32_t single() const {
        return threadIdx.x < head ? lo + threadIdx.x
                                  : threadIdx.x >= 8 && threadIdx.x - 8 < tail ? hi - tail + threadIdx.x - 8 : 0xffffffffu;
    }
};

// Statistics alone: a slice of any length per block, streamed.  2048 rows of 32000: 44 us, 6.0 TB/s.
__global__ void __launch_bounds__(kThreads)
log_probs_kernel(LogProbArgs a) {
    qk::pdl_launch();
    qk::pdl_wait();
    __shared__ Stats part[kWarps];
    const uint32_t row = blockIdx.x / a.n_slices, slice = blockIdx.x % a.n_slices;
    const float *x = a.logits + row * a.stride;
    const Extent ext(x, a, slice);
    float m = -INFINITY, s = 0.f, t = 0.f;
    auto take = [&](float v0, float v1, float v2, float v3) {
        const float top = fmaxf(fmaxf(v0, v1), fmaxf(v2, v3));
        if (top > m) {
            if (m > -INFINITY) {
                const float d = m - top, w = ex2(d * kLog2E);
                t = w > 0.f ? w * fmaf(d, s, t) : 0.f;
                s *= w;
            }
            m = top;
        }
        const float base = m > -INFINITY ? m : 0.f;
        const float v[4] = {v0, v1, v2, v3};
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // (the difference first: its rounding counts for this entry alone)
            const float d = floored(v[e] - base), w = ex2(d * kLog2E);
            s += w;
            t = fmaf(d, w, t);
        }
    };
    const float4 *xv = reinterpret_cast<const float4 *>(x + ext.lo + ext.head);
    constexpr uint32_t kAhead = 4;
    uint32_t i = threadIdx.x;
    for (; i + (kAhead - 1) * kThreads < ext.vectors; i += kAhead * kThreads) {
        float4 v[kAhead];
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) v[u] = __ldg(xv + i + u * kThreads);
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) take(v[u].x, v[u].y, v[u].z, v[u].w);
    }
    for (; i < ext.vectors; i += kThreads) {
        const float4 v = __ldg(xv + i);
        take(v.x, v.y, v.z, v.w);
    }
    const uint32_t single = ext.single();
    if (single != 0xffffffffu) take(x[single], -INFINITY, -INFINITY, -INFINITY);
    share(Stats{m, s, t}, part);
    __syncthreads();
    if (a.clustered) {
        __shared__ Stats shared_stats;
        join_cluster<false>(a, row, slice, of_block(part), 0, &shared_stats, nullptr);
        return;
    }
    if (threadIdx.x >= 32) return;
    const Stats st = of_block(part);
    if (a.n_slices == 1) finish(a, row, st, 0, threadIdx.x);
    else if (threadIdx.x == 0) *reinterpret_cast<float4 *>(a.stats + (size_t)blockIdx.x * 4) = make_float4(st.m, st.s, st.t, 0.f);
}

// With the most probable entries: a slice of at most 32 entries a thread (and a single one) stays in registers.  The
// n_top-th of the largest values of 32 groups of eight threads is no better than the slice's n_top-th entry: what is as
// good as that, 30 to 110 entries of a slice of 8192 without ties, goes into a list whose places are found by counting.
// Where the list overflows because many entries equal the bound (masked vocabularies), those of the lowest indices are
// taken; where it overflows without them, the warps sort.
// 64 rows of 128256, 20 places: 15.7 us with the join (2.1 TB/s: chains of barriers in two waves of short blocks; 18.3
// with three blocks to an SM, whose 80 registers spill less, 17.1 with slices of 4096).  Whatever beats a running last
// place, sorted warp by warp, took 93 us; the bound from the 256 threads' best, sorted, and a sorted list 26.
__global__ void __launch_bounds__(kThreads, 4)
log_probs_top_kernel(LogProbArgs a) {
    qk::pdl_launch();
    qk::pdl_wait();
    __shared__ float2 part[kWarps];
    __shared__ float group_best[32], bound_value;
    __shared__ uint64_t candidates[kCandidates], best_of[kWarps][32];
    __shared__ uint32_t n_candidates, n_better, warp_count[kWarps];
    const uint32_t row = blockIdx.x / a.n_slices, slice = blockIdx.x % a.n_slices;
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const float *x = a.logits + row * a.stride;
    const Extent ext(x, a, slice);
    const float4 *xv = reinterpret_cast<const float4 *>(x + ext.lo + ext.head);
    const uint32_t first = ext.lo + ext.head, single = ext.single();
    if (threadIdx.x == 0) n_candidates = 0, n_better = 0;
    if (threadIdx.x < 32) best_of[0][threadIdx.x] = 0;
    float v[kHeld * 4 + 1];
#pragma unroll
    for (uint32_t u = 0; u < kHeld; ++u) {
        const uint32_t i = threadIdx.x + u * kThreads;
        const float4 w = i < ext.vectors ? __ldg(xv + i) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        v[4 * u] = w.x, v[4 * u + 1] = w.y, v[4 * u + 2] = w.z, v[4 * u + 3] = w.w;
    }
    v[kHeld * 4] = single != 0xffffffffu ? x[single] : -INFINITY;
    // (entries past the slice are -infinity too, but `there` tells them apart)
    auto index_of = [&](uint32_t i) { return i == kHeld * 4 ? single : first + 4 * (threadIdx.x + i / 4 * kThreads) + i % 4; };
    auto there = [&](uint32_t i) { return i == kHeld * 4 ? single != 0xffffffffu : threadIdx.x + i / 4 * kThreads < ext.vectors; };
    float m = -INFINITY;
#pragma unroll
    for (uint32_t i = 0; i <= kHeld * 4; ++i) m = fmaxf(m, v[i]);
    float top = m;
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (lane % 8 == 0) group_best[warp * 4 + lane / 8] = top;
    __syncthreads();
    float key = group_best[lane], m_block = key;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m_block = fmaxf(m_block, __shfl_xor_sync(0xffffffffu, m_block, off));
    if (warp == 0) {  // ---- the bound: the groups' values in falling order, the n_top-th of them
#pragma unroll
        for (int size = 2; size <= 32; size *= 2)
#pragma unroll
            for (int bit = size / 2; bit > 0; bit /= 2) {
                const float other = __shfl_xor_sync(0xffffffffu, key, bit);
                key = ((lane & bit) == 0) == ((lane & size) == 0 || size == 32) ? fmaxf(key, other) : fminf(key, other);
            }
        if (lane == a.n_top - 1) bound_value = key;
    }
    // ---- sums against the slice's maximum
    float s = 0.f, t = 0.f;
    const float base = m_block > -INFINITY ? m_block : 0.f;
#pragma unroll
    for (uint32_t i = 0; i <= kHeld * 4; ++i) {
        const float d = floored(v[i] - base), w = ex2(d * kLog2E);
        s += w;
        t = fmaf(d, w, t);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, off);
        t += __shfl_xor_sync(0xffffffffu, t, off);
    }
    if (lane == 0) part[warp] = make_float2(s, t);
    __syncthreads();
    const float bound = bound_value;
    auto push = [&](uint32_t i) {
        const uint32_t place = atomicAdd(&n_candidates, 1u);
        if (place < kCandidates) candidates[place] = rank_key(v[i], index_of(i));
    };
    if (m >= bound && bound > -INFINITY) {
#pragma unroll
        for (uint32_t i = 0; i <= kHeld * 4; ++i)
            if (v[i] >= bound) push(i);
    }
    __syncthreads();
    uint32_t n = n_candidates;
    uint64_t best = 0;
    if (n > kCandidates || bound == -INFINITY) {  // (the same for all threads)
        __syncthreads();
        if (threadIdx.x == 0) n_candidates = 0;
        __syncthreads();
        uint32_t better = 0;
#pragma unroll
        for (uint32_t i = 0; i <= kHeld * 4; ++i) {
            if (v[i] > bound) {
                push(i);
                ++better;
            }
        }
        if (better) atomicAdd(&n_better, better);
        __syncthreads();
        n = n_better;
        if (n <= kCandidates) {
            // entries equal to the bound, in the order of their indices: the single ones in front, the vectors' rounds, the
            // single ones behind; as many as there are places left
            uint32_t left = a.n_top > n ? a.n_top - n : 0;
#pragma unroll
            for (int round = -1; round <= (int)kHeld; ++round) {
                if (left == 0) break;
                const bool lone = round < 0 || round == (int)kHeld;
                auto equal = [&](uint32_t e) {
                    const uint32_t i = lone ? kHeld * 4 : 4 * round + e;
                    return there(i) && v[i] == bound && (!lone || ((threadIdx.x < ext.head) == (round < 0)));
                };
                uint32_t count = 0;
#pragma unroll
                for (uint32_t e = 0; e < (lone ? 1u : 4u); ++e) count += equal(e);
                uint32_t before = count;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const uint32_t o = __shfl_up_sync(0xffffffffu, before, off);
                    if (lane >= (uint32_t)off) before += o;
                }
                if (lane == 31) warp_count[warp] = before;
                __syncthreads();
                before -= count;
                uint32_t all = 0;
#pragma unroll
                for (uint32_t w = 0; w < kWarps; ++w) {
                    before += w < warp ? warp_count[w] : 0;
                    all += warp_count[w];
                }
#pragma unroll
                for (uint32_t e = 0; e < (lone ? 1u : 4u); ++e)
                    if (equal(e)) {
                        if (before < left) push(lone ? kHeld * 4 : 4 * round + e);
                        ++before;
                    }
                left -= min(left, all);
                __syncthreads();
            }
            n = min(n_candidates, kCandidates);
        } else {  // every warp sorts its own, then they join
            for (uint32_t i = 0; i <= kHeld * 4; ++i) {
                uint64_t key = 0;
#pragma unroll
                for (uint32_t e = 0; e <= kHeld * 4; ++e)
                    if (e == i && v[e] >= bound && there(e)) key = rank_key(v[e], index_of(e));
                if (__any_sync(0xffffffffu, key != 0)) best = merged(best, sorted(key, lane), lane);
            }
            best_of[warp][lane] = best;
            __syncthreads();
            if (warp == 0) {
                for (uint32_t w = 1; w < kWarps; ++w) best = merged(best, best_of[w][lane], lane);
                best_of[0][lane] = best;
            }
            n = 0;
        }
    }
    // ---- a candidate's place is the number of better ones
    for (uint32_t at = threadIdx.x; at < n; at += kThreads) {
        const uint64_t key = candidates[at];
        uint32_t place = 0;
        for (uint32_t i = 0; i < n; ++i) place += candidates[i] > key;
        if (place < 32) best_of[0][place] = key;
    }
    __syncthreads();
    if (warp != 0 && !a.clustered) return;
    best = best_of[0][lane];
    Stats st{m_block, 0.f, 0.f};
    for (uint32_t w = 0; w < kWarps; ++w) st.s += part[w].x, st.t += part[w].y;
    if (a.clustered) {
        __shared__ Stats shared_stats;
        __syncthreads();
        join_cluster<true>(a, row, slice, st, best, &shared_stats, best_of);
        return;
    }
    if (a.n_slices == 1) {
        finish(a, row, st, best, lane);
        return;
    }
    if (lane == 0) *reinterpret_cast<float4 *>(a.stats + (size_t)blockIdx.x * 4) = make_float4(st.m, st.s, st.t, 0.f);
    a.keys[(size_t)blockIdx.x * 32 + lane] = best;
}

// The slices of a row, one block each row.
template <bool kTop>
__global__ void __launch_bounds__(kThreads)
log_probs_join_kernel(LogProbArgs a) {
    qk::pdl_launch();
    qk::pdl_wait();
    __shared__ Stats part[kWarps];
    __shared__ uint64_t best_of[kTop ? kWarps : 1][32];
    const uint32_t row = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    Stats st{-INFINITY, 0.f, 0.f};
    for (uint32_t i = threadIdx.x; i < a.n_slices; i += kThreads) {
        const float4 v = *reinterpret_cast<const float4 *>(a.stats + ((size_t)row * a.n_slices + i) * 4);
        st = joined(st, Stats{v.x, v.y, v.z});
    }
    share(st, part);
    uint64_t best = 0;
    if constexpr (kTop) {
        for (uint32_t i = warp; i < a.n_slices; i += kWarps)
            best = merged(best, a.keys[((size_t)row * a.n_slices + i) * 32 + lane], lane);
        best_of[warp][lane] = best;
#pragma unroll
        for (uint32_t half = kWarps / 2; half > 0; half /= 2) {
            __syncthreads();
            if (warp < half) best_of[warp][lane] = best = merged(best, best_of[warp + half][lane], lane);
        }
    } else {
        __syncthreads();
    }
    if (warp != 0) return;
    st = of_block(part);
    finish(a, row, st, best, lane);
}

// How many slices a row is cut into, their length (a multiple of four entries), and whether a cluster joins them: while
// all blocks are resident at once.  (1 x 32768, 5 places: 24 -> 19 us a call.  Where blocks queue, clusters make them wait
// for one another: 64 x 128256, 20 places, 18 -> 30 us.)
bool slices(size_t n_tokens, size_t vocab, size_t n_top, uint32_t *n, uint32_t *length) {
    const size_t held = n_top ? kThreads * kHeld * 4 : SIZE_MAX;  // (what stays in registers)
    const size_t most = qk::ceil_div(vocab, kMinSlice), want = std::max<size_t>(1, kWantBlocks / std::max<size_t>(1, n_tokens));
    size_t count = std::min(most, want);
    if (count > kMaxCluster && n_tokens * kMaxCluster <= kResident && qk::ceil_div(vocab, kMaxCluster) <= std::min(held, kMaxSlice))
        count = kMaxCluster;
    const size_t len = std::min((qk::ceil_div(vocab, count) + 3) / 4 * 4, held);
    *length = (uint32_t)len;
    *n = (uint32_t)qk::ceil_div(vocab, len);
    return *n > 1 && *n <= kMaxCluster && n_tokens * *n <= kResident;
}

}  // namespace

extern "C" {

size_t qk_log_probs_scratch(size_t n_tokens, size_t vocab, size_t n_top) {
    if (!n_tokens || !vocab) return 0;
    uint32_t n, length;
    const bool clustered = slices(n_tokens, vocab, n_top, &n, &length);
    return n == 1 || clustered ? 0 : n_tokens * n * (16 + (n_top ? 256 : 0));
}

qk_status qk_log_probs(qk_ctx *ctx, const float *logits, size_t n_tokens, size_t vocab, size_t stride,
                       const int32_t *targets, size_t n_top, void *scratch, float *lse, float *logprob, float *entropy,
                       float *top_logprob, int32_t *top_ids) {
    if (vocab == 0 || vocab > 0x7fffffffull) return qk::fail(QK_ERR_VALUE, "vocab must lie in 1 .. 2^31 - 1, got %zu", vocab);
    if (stride < vocab) return qk::fail(QK_ERR_VALUE, "rows of %zu logits cannot be %zu apart", vocab, stride);
    if (n_top > kMaxTop || n_top > vocab)
        return qk::fail(QK_ERR_VALUE, "n_top must be at most %u and the vocabulary of %zu, got %zu", kMaxTop, vocab, n_top);
    if (n_tokens > (1u << 24)) return qk::fail(QK_ERR_VALUE, "%zu rows are more than one call takes", n_tokens);
    if (!logits) return qk::fail(QK_ERR_VALUE, "logits is null");
    if ((uintptr_t)logits % sizeof(float)) return qk::fail(QK_ERR_VALUE, "logits lie on no float boundary");
    if (logprob && !targets) return qk::fail(QK_ERR_VALUE, "logprob needs targets");
    for (const void *p : {(const void *)targets, (const void *)lse, (const void *)logprob, (const void *)entropy,
                          (const void *)top_logprob, (const void *)top_ids})
        if ((uintptr_t)p % 4) return qk::fail(QK_ERR_VALUE, "targets or an output lies on no boundary of its type");
    const size_t need = qk_log_probs_scratch(n_tokens, vocab, n_top);
    if (need && (!scratch || (uintptr_t)scratch % 16)) return qk::fail(QK_ERR_VALUE, "scratch is null or on no 16-byte boundary");
    if (n_tokens == 0) return QK_OK;
    qk_ctx *c;
    qk::DeviceGuard guard;
    qk_status st = qk::resolve_ctx(ctx, &c);
    if (st != QK_OK) return st;
    QK_CUDA(cudaSetDevice(c->device));
    std::lock_guard<std::mutex> lock(c->mu);
    LogProbArgs a{};
    a.logits = logits, a.stride = stride, a.n_tokens = (uint32_t)n_tokens, a.vocab = (uint32_t)vocab, a.n_top = (uint32_t)n_top;
    a.targets = targets, a.lse = lse, a.logprob = logprob, a.entropy = entropy, a.top_logprob = top_logprob, a.top_ids = top_ids;
    a.clustered = slices(n_tokens, vocab, n_top, &a.n_slices, &a.slice);
    a.keys = static_cast<uint64_t *>(scratch);
    a.stats = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + (n_top ? n_tokens * a.n_slices * 256 : 0));
    auto go = [&](auto kernel, unsigned blocks, unsigned cluster) -> qk_status {
        if (cluster > 8) QK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        (void)qk::launch_pdl_cluster(c->pdl, kernel, dim3(blocks), dim3(kThreads), cluster, 0, c->stream, a);
        QK_CUDA(cudaGetLastError());
        c->launches++;
        return QK_OK;
    };
    st = go(n_top ? log_probs_top_kernel : log_probs_kernel, (unsigned)(n_tokens * a.n_slices), a.clustered ? a.n_slices : 1);
    if (st != QK_OK || a.n_slices == 1 || a.clustered) return st;
    return go(n_top ? log_probs_join_kernel<true> : log_probs_join_kernel<false>, (unsigned)n_tokens, 1);
}

}  // extern "C"
