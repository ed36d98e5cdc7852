// Attention of many query rows over one slot's cache rows on tcgen05: a prompt's portion, and a prefix that a whole
// batch shares.  INT8 and bfloat16 caches, head sizes 64 and 128.
//
// The queries that read one kv head are the rows of one product: row r is query r / group, head r % group of the kv
// head, 128 rows to a CTA, which takes a range of keys 64 at a time.  Two units of four warps take the key blocks in
// turn, a thread owns a row (no shuffles): running maximum, sum and output in registers, the two units joined at the
// end.  While one unit is at its exponentials the tensor core works for the other; INT8 scores are formed three blocks
// ahead, and a block's output is read out when the maximum of the unit's next block is known.  The weights go back to
// tensor memory, over their scores, as the A operand; v is read as it lies (MN-major B).  Three warps bring the key blocks
// in, three the value blocks.
//
// Exactness.  INT8 rows: codes as float16 are exact (three warps convert them on their way into shared memory); q is
// two float16 terms after scaling by a power of two per row (22 bits), and so are the weights times the value scales,
// relative to a power of two at the scales' running maximum E (the bound stands at qk::scales_apart).  Where value scales
// lie too far apart for that, and in blocks that some row does not see whole, the weights are "wide": three bfloat16 terms
// times codes in bfloat16, in true units.  bfloat16 rows go in as they are; q and the weights are three bfloat16 terms.  A
// block's product with v starts from zero and is added to the row's output in registers, in float32: the tensor core
// truncates.
//
// What bounds it: a unit's chain for a block of 64 keys, 4200 cycles (waits, maxima, the output's turn, exponentials,
// weights and their terms), of which two run side by side, and 16000 cycles of a CTA before its first block (q) and behind
// its last (the units' exchange).  INT8, 2048 tokens from position 0, 32 / 8 heads of 128: 99.9 us, 0.34 PFLOP/s of the
// formula's operations.  64 x 32 / 8 heads behind 8192 bfloat16 rows: 35 us standing alone.  Slower, us for the INT8 portion:
// wide weights throughout (115 when two terms took 104), a branch on the form for every word that is converted (+ 7), the
// warp that issues the products waiting for what the units have waited for, and for the keys of later scores ahead of a
// product (104.8), 184 registers a thread for the units and 72 for the rest (103.6), 192 and 64 (111.5), 208 and 48 (113).
// Where the first value scale makes all weights wide: 131.  Faster by 1: scores four blocks ahead, which leaves no place for
// a third term.  bfloat16: 200 registers for the units
// (+ 1.4), scores three blocks ahead (+ 0.4).
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "qk_cache.h"
#include "qk_decoder_dev.cuh"
#include "qk_umma.cuh"

namespace {

using qk::CacheView;
using qk::TileArgs;

constexpr uint32_t kRows = 128, kKeys = 64;  // query rows of a CTA, keys of a block
constexpr uint32_t kThreads = 512, kLoaders = 96, kKeyWarp = 8, kValueWarp = 11, kScaleWarp = 14, kMmaWarp = 15;  // three warps a loader
constexpr int kLaunchRegs = 128;
constexpr uint32_t kTmemCols = 512;
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kWeightScale = 16384.f;  // float16 weights enter the product times this, their second terms times
constexpr uint32_t kLowBits = 11;        // 2^11 more (of wide weights too), which the product takes off again
constexpr float kKeyShrink = 0x1p-30f;   // of the second set of a block's key scales, see below
constexpr uint32_t kWaitLimit = 1u << 22;
constexpr uint32_t kSms = 148;
constexpr uint32_t kEdges = 4;  // causal: the blocks that some row of a tile does not see whole are among the last four

template <bool kI8, int D>
struct TileShape {
    static constexpr uint32_t kTerms = kI8 ? 2 : 3;                    // of q
    static constexpr int kUnitRegs = kI8 ? 200 : 184, kOtherRegs = kI8 ? 56 : 72;
    static_assert(256 * kUnitRegs + 256 * kOtherRegs <= (int)kThreads * kLaunchRegs, "setmaxnreg draws on the launch's registers");
    static constexpr uint32_t kChunks = D / 64;                        // of 64 channels, rows of 128 bytes
    static constexpr uint32_t kChunkBytes = kKeys * 128, kTileBytes = kChunks * kChunkBytes;
    static constexpr uint32_t kQChunkBytes = kRows * 128, kQTermBytes = kChunks * kQChunkBytes;
    static constexpr uint32_t kStages = kI8 || D == 64 ? 4 : 3;        // of the keys' ring, and of the values'
    // Of a block: key scales, value scales, key scales times kKeyShrink, E, whether its weights are wide.
    static constexpr uint32_t kScaleFloats = kI8 ? 3 * kKeys + 4 : 0;
    static constexpr uint32_t kRingBytes = 2 * kStages * kTileBytes;
    static constexpr uint32_t kSmem = 1024 + kTerms * kQTermBytes + kRingBytes + kStages * kScaleFloats * 4 + 512 + 512;
    static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
    // Tensor memory.  INT8: the scores of three blocks, over which the first two terms of their weights lie (16 columns of
    // scores become eight of either term), a third term's place for either unit, the units' outputs.  (Scores of four blocks:
    // 1 % faster.)  bfloat16, whose terms are three: a unit's scores, behind them the first two terms of its weights, the
    // third over scores that have been read, its output.
    static constexpr uint32_t kAhead = kI8 ? 3 : 2;  // blocks whose scores are formed ahead: block g's lie in place g % kAhead
    __device__ static constexpr uint32_t score_col(uint32_t g) { return (kI8 ? 64 : 256) * (g % kAhead); }
    __device__ static constexpr uint32_t out_col(uint32_t u) { return kI8 ? 256 + 128 * u : 256 * u + 128; }
    __device__ static constexpr uint32_t weight_col(uint32_t g, uint32_t term, uint32_t step) {  // of a step of 16 keys
        return !kI8 ? score_col(g) + (term == 2 ? 0 : 64 + 32 * term) + 8 * step
                    : term == 2 ? 192 + 32 * (g & 1) + 8 * step : score_col(g) + 16 * step + 8 * term;
    }
    static_assert(kRingBytes >= (D * kRows + 5 * kRows) * 4, "the units' exchange lies in the ring");
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(uint32_t magnitude_bits) {  // clamped to -110 .. 127
    return min(127, max(-110, (int)(magnitude_bits >> 23) - 127));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(v[0]),
                 "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
// M = 128, N = n, float32 accumulators; kind: 0 float16 operands, 1 bfloat16; b_mn: B is MN-major
__device__ __forceinline__ constexpr uint32_t instruction(uint32_t n, uint32_t b_mn, uint32_t kind) {
    return (1u << 4) | (kind << 7) | (kind << 10) | (b_mn << 16) | ((n >> 3) << 17) | ((kRows >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(ad), "l"(bd), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t at, uint64_t bd, uint32_t idesc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(at), "l"(bd), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
// The same where d counts for 2^-kLowBits of itself.
__device__ __forceinline__ void mma_ts_above(uint32_t d, uint32_t at, uint64_t bd, uint32_t idesc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.eq.b32 p, 0, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, %4;\n}" ::"r"(d),
        "r"(at), "l"(bd), "r"(idesc), "n"(kLowBits)
        : "memory");
}
// Barrier `id` of n threads; true when all of them say so.
template <int kId, int kN>
__device__ __forceinline__ bool vote(bool ok) {
    uint32_t all;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.and.pred q, %2, %3, p;\n selp.u32 %0, 1, 0, q;\n}"
        : "=r"(all)
        : "r"((uint32_t)ok), "n"(kId), "n"(kN)
        : "memory");
    return all != 0;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two values as their terms, t[0] the leading one: two of float16 or three of bfloat16, all but the first `times` larger.
__device__ __forceinline__ void terms_f16(float a, float b, float times, uint32_t *t) {
    t[0] = pack_f16x2(a, b);
    float2 r = __ffma2_rn(__half22float2(*reinterpret_cast<__half2 *>(&t[0])), make_float2(-1.f, -1.f), make_float2(a, b));
    r = __fmul2_rn(r, make_float2(times, times));
    t[1] = pack_f16x2(r.x, r.y);
}
__device__ __forceinline__ void terms_bf16(float a, float b, float times, uint32_t *t) {
    t[0] = bf16_pair(a, b);
    a = (a - __uint_as_float(t[0] << 16)) * times, b = (b - __uint_as_float(t[0] & 0xffff0000u)) * times;
    t[1] = bf16_pair(a, b);
    t[2] = bf16_pair(a - __uint_as_float(t[1] << 16), b - __uint_as_float(t[1] & 0xffff0000u));
}
// Four codes as float16: 1024 + u is the bit pattern 0x6400 | u, u = code + 128.
__device__ __forceinline__ void codes_to_f16(uint32_t codes, uint32_t &lo, uint32_t &hi) {
    const uint32_t u = codes ^ 0x80808080u;
    lo = __byte_perm(u, 0x64646464u, 0x4140);
    hi = __byte_perm(u, 0x64646464u, 0x4342);
    asm("{\n .reg .b32 c;\n mov.b32 c, 0x64806480;\n sub.rn.f16x2 %0, %0, c;\n sub.rn.f16x2 %1, %1, c;\n}" : "+r"(lo), "+r"(hi));
}
// Four codes as bfloat16: with the low seven bits u of a code 0x4300 | u is 128 + u, with its sign bit 0x4300 | 0x80 is 256
// and 0x4300 is 128; the code is the difference.
__device__ __forceinline__ void codes_to_bf16(uint32_t codes, uint32_t &lo, uint32_t &hi) {
    const uint32_t a = __byte_perm(codes, 0u, 0x4140), b = __byte_perm(codes, 0u, 0x4342);
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(lo) : "r"((a & 0x007f007fu) | 0x43004300u), "r"((a & 0x00800080u) | 0x43004300u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(hi) : "r"((b & 0x007f007fu) | 0x43004300u), "r"((b & 0x00800080u) | 0x43004300u));
}
// Waits for the loads of tensor memory, v's the last of them (which nothing may use before).
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                   "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :
                 : "memory");
}
// n times sixteen columns of tensor memory to use(i, values), each load under way while the values before are used.
template <int kN, typename Use>
__device__ __forceinline__ void each16(uint32_t taddr, Use use) {
    uint32_t v[2][16];
    tmem_ld16(taddr, v[0]);
#pragma unroll
    for (int i = 0; i < kN; ++i) {
        tmem_ld_wait(v[i % 2]);
        if (i + 1 < kN) tmem_ld16(taddr + 16 * (i + 1), v[(i + 1) % 2]);
        use(i, v[i % 2]);
    }
}
// Whether both barriers have completed their phases: the usual case of two waits, for the price of one.
__device__ __forceinline__ bool both_ready(uint64_t *bar1, uint32_t parity1, uint64_t *bar2, uint32_t parity2) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p, q;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n and.pred p, p, q;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(done)
        : "r"(smem_u32(bar1)), "r"(parity1), "r"(smem_u32(bar2)), "r"(parity2)
        : "memory");
    return __all_sync(0xffffffffu, done) != 0;
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Grid (kv heads x tiles of 128 rows, splits of the keys); late tiles see most keys: they go first.
template <bool kI8, int D>
__global__ void __launch_bounds__(kThreads, 1)
attend_tile_kernel(CacheView c, TileArgs a) {
    using S = TileShape<kI8, D>;
    constexpr uint32_t kTerms = S::kTerms, kChunks = S::kChunks, kStages = S::kStages, kAhead = S::kAhead;
    qk::pdl_launch();
    extern __shared__ __align__(1024) uint8_t raw_smem[];
    uint8_t *qs = raw_smem + (-smem_u32(raw_smem) & 1023u);  // (an offset: the compiler still sees shared memory)
    uint8_t *ring = qs + kTerms * S::kQTermBytes;
    uint8_t *v_ring = ring + kStages * S::kTileBytes;
    float *scales = reinterpret_cast<float *>(ring + S::kRingBytes);             // [stage of the values][kScaleFloats]
    float *row_factor = scales + kStages * S::kScaleFloats;                     // [128]
    uint64_t *q_full = reinterpret_cast<uint64_t *>(row_factor + 128);
    uint64_t *k_full = q_full + 1, *k_empty = k_full + kStages, *v_full = k_empty + kStages, *v_empty = v_full + kStages;
    uint64_t *s_full = v_empty + kStages, *p_full = s_full + kAhead, *o_full = p_full + 2;
    uint64_t *drain = o_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int *never = reinterpret_cast<volatile int *>(tmem_slot + 2);
    uint32_t *spoilt = tmem_slot + 3;  // [block from the last][2]: keys with an infinity or NaN among their values
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t kvh = blockIdx.x % c.n_kv, tile = gridDim.x / c.n_kv - 1 - blockIdx.x / c.n_kv, split = blockIdx.y;
    const uint32_t group = a.n_heads / c.n_kv, n_rows = a.n_queries * group;
    const uint32_t row0 = tile * kRows, rows = min(kRows, n_rows - row0);
    // keys of the tile: all of them, or up to its last query's own
    const uint32_t last_query = (row0 + rows - 1) / group;
    const uint32_t n_keys = a.causal ? a.first_row + last_query + 1 : a.n_keys;
    const uint32_t all_blocks = (n_keys + kKeys - 1) / kKeys, per_split = (all_blocks + a.n_splits - 1) / a.n_splits;
    const uint32_t block0 = min(all_blocks, split * per_split), n_blocks = min(all_blocks, block0 + per_split) - block0;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 8);
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(k_full + s, kLoaders / 32);
            mbar_init(k_empty + s, 1);
            mbar_init(v_full + s, kLoaders / 32 + (kI8 ? 1 : 0));
            mbar_init(v_empty + s, 1);
        }
        for (uint32_t i = 0; i < kAhead; ++i) mbar_init(s_full + i, 1);
        for (int u = 0; u < 2; ++u) {
            mbar_init(p_full + u, 4);
            mbar_init(o_full + u, 1);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        *never = 0;
        for (uint32_t i = 0; i < 2 * kEdges; ++i) spoilt[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    qk::pdl_wait();
    const uint32_t tmem = *tmem_slot;
    const size_t line0 = (a.seq * c.n_kv + kvh) * (size_t)c.rows + (size_t)block0 * kKeys;  // first key's row
    const uint32_t keys = n_blocks ? min(n_keys - block0 * kKeys, n_blocks * kKeys) : 0;    // of this CTA
    // keys that every row of the tile sees: the blocks past them (at the end) are edges
    const int seen0 = min((int)keys, a.causal ? (int)(a.first_row + row0 / group) + 1 - (int)(block0 * kKeys) : (int)keys);
    auto at_edge = [&](uint32_t g) { return (int)((g + 1) * kKeys) > seen0; };
    // INT8: whether block g's weights are wide, three bfloat16 terms (else two of float16): at an edge, where scales that some
    // row does not see must not count, and from the first block on up to which the value scales lie too far apart.  s0, s1:
    // the block's, two a lane; every warp that asks for all blocks in turn comes to the same answers.
    struct Scales {
        int e_max = -110;              // exponent of the largest so far
        uint32_t least = 0xffffffffu;  // bits, less one, of the smallest but zero
        bool wide = false;
    };
    auto look = [&](Scales &st, uint32_t g, float s0, float s1) {
        const uint32_t b0 = __float_as_uint(fabsf(s0)), b1 = __float_as_uint(fabsf(s1));
        const int e = max(st.e_max, exponent_of(__reduce_max_sync(0xffffffffu, max(b0, b1))));
        st.least = min(st.least, __reduce_min_sync(0xffffffffu, min(b0 - 1u, b1 - 1u)));
        st.wide = st.wide || at_edge(g) || qk::scales_apart(e, st.least);
        if (!st.wide) st.e_max = e;
    };

    if (warp >= kKeyWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kOtherRegs));
        if (warp < kScaleWarp) {
            // ---- key blocks into their ring, value blocks into theirs; rows past the end are zeros
            const bool is_v = warp >= kValueWarp;
            const uint32_t tid = threadIdx.x - (is_v ? kValueWarp : kKeyWarp) * 32;
            constexpr uint32_t kRowBytes = kI8 ? D : 2 * D, kPieces = kRowBytes / 16, kStep = kLoaders / kPieces;
            constexpr uint32_t kPasses = (kKeys + kStep - 1) / kStep;
            // A thread's piece, and its rows: first, first + kStep, ..  (INT8, head size 128: eight threads store two rows of
            // one chunk of 64 channels and meet no bank twice.)
            const uint32_t piece = kI8 && D == 128 ? tid / 8 % 2 * 4 + tid % 4 : tid % kPieces;
            const uint32_t first = kI8 && D == 128 ? tid / 16 * 2 + tid / 4 % 2 : tid / kPieces;
            const uint8_t *base = static_cast<const uint8_t *>(is_v ? c.v : c.k) + line0 * kRowBytes + piece * 16;
            uint8_t *tiles = is_v ? v_ring : ring;
            uint64_t *fulls = is_v ? v_full : k_full, *empties = is_v ? v_empty : k_empty;
            bool ok = true;
            auto hand_over = [&](uint64_t *bar) {
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            };
            if constexpr (kI8) {
                uint4 held[kPasses];  // the next block's, on their way while this one is converted
                float s0 = 0.f, s1 = 0.f;  // its value scales
                auto load = [&](uint32_t g) {
                    if (is_v) {
                        const uint32_t key = g * kKeys + lane;
                        s0 = key < keys ? c.v_scale[line0 + key] : 0.f, s1 = key + 32 < keys ? c.v_scale[line0 + key + 32] : 0.f;
                    }
#pragma unroll
                    for (uint32_t i = 0; i < kPasses; ++i) {
                        const uint32_t row = first + i * kStep, key = g * kKeys + row;
                        held[i] = row < kKeys && key < keys ? __ldg(reinterpret_cast<const uint4 *>(base + (size_t)key * kRowBytes))
                                                            : make_uint4(0u, 0u, 0u, 0u);
                    }
                };
                Scales st;
                load(0);
                for (uint32_t g = 0; g < n_blocks; ++g) {
                    const uint32_t s = g % kStages;
                    if (is_v) look(st, g, s0, s1);
                    ok = mbar_wait(empties + s, ((g / kStages) & 1) ^ 1, abort_flag, a.wait_limit);
                    if (!ok) break;
                    uint8_t *tile_at = tiles + s * S::kTileBytes + piece / 4 * S::kChunkBytes;
                    auto store = [&](auto convert) {
#pragma unroll
                        for (uint32_t i = 0; i < kPasses; ++i) {  // sixteen codes: two pieces of eight values
                            const uint32_t row = first + i * kStep;
                            if (row >= kKeys) break;
                            uint32_t w[8];
                            convert(held[i].x, w[0], w[1]);
                            convert(held[i].y, w[2], w[3]);
                            convert(held[i].z, w[4], w[5]);
                            convert(held[i].w, w[6], w[7]);
                            const uint32_t at = 2 * (piece % 4);
                            *reinterpret_cast<uint4 *>(tile_at + row * 128 + ((at ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                            *reinterpret_cast<uint4 *>(tile_at + row * 128 + (((at + 1) ^ (row & 7)) << 4)) =
                                make_uint4(w[4], w[5], w[6], w[7]);
                        }
                    };
                    if (st.wide) store([](uint32_t codes, uint32_t &lo, uint32_t &hi) { codes_to_bf16(codes, lo, hi); });
                    else store([](uint32_t codes, uint32_t &lo, uint32_t &hi) { codes_to_f16(codes, lo, hi); });
                    load(g + 1);
                    hand_over(fulls + s);
                }
            } else {
                // Values that some rows of the tile do not see: an infinity or NaN times their weight, zero, would reach them
                // all the same.  It becomes zero, and its key is noted for the rows that do see it.  (A thread looks at what it
                // copied itself.)
                auto clean = [&](uint32_t g) {
                    const uint32_t from_last = n_blocks - 1 - g;
                    if (!is_v || !a.causal || from_last >= kEdges) return;
                    uint8_t *tile_at = tiles + g % kStages * S::kTileBytes + piece / 8 * S::kChunkBytes;
#pragma unroll 1
                    for (uint32_t row = first; row < kKeys; row += kStep) {
                        uint32_t *w = reinterpret_cast<uint32_t *>(tile_at + row * 128 + (((piece % 8) ^ (row & 7)) << 4));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool lo = (w[i] & 0x7f80u) == 0x7f80u, hi = (w[i] & 0x7f800000u) == 0x7f800000u;
                            if (lo || hi) {
                                w[i] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0x0000ffffu : 0xffffffffu);
                                atomicOr(spoilt + 2 * from_last + row / 32, 1u << (row % 32));
                            }
                        }
                    }
                };
                for (uint32_t g = 0; g < n_blocks; ++g) {
                    const uint32_t s = g % kStages;
                    ok = mbar_wait(empties + s, ((g / kStages) & 1) ^ 1, abort_flag, a.wait_limit);
                    if (!ok) break;
                    uint8_t *tile_at = tiles + s * S::kTileBytes + piece / 8 * S::kChunkBytes;
#pragma unroll
                    for (uint32_t i = 0; i < kPasses; ++i) {
                        const uint32_t row = first + i * kStep, key = g * kKeys + row;
                        if (row >= kKeys) break;
                        const bool live = key < keys;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                                         smem_u32(tile_at + row * 128 + (((piece % 8) ^ (row & 7)) << 4))),
                                     "l"(base + (live ? (size_t)key * kRowBytes : 0)), "r"(live ? 16u : 0u)
                                     : "memory");
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (g) {  // (a block is handed over when the next one is under way)
                        asm volatile("cp.async.wait_group 1;" ::: "memory");
                        clean(g - 1);
                        hand_over(fulls + (g - 1) % kStages);
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                if (ok && n_blocks) {
                    clean(n_blocks - 1);
                    hand_over(fulls + (n_blocks - 1) % kStages);
                }
            }
            if (!ok) *abort_flag = 1;
        } else if (warp == kScaleWarp) {
            // ---- q of the tile that comes to an SM after this one (one CTA each is resident) on its way to L2
            if (blockIdx.x + kSms < gridDim.x) {
                const uint32_t next = blockIdx.x + kSms, kvh2 = next % c.n_kv, tile2 = gridDim.x / c.n_kv - 1 - next / c.n_kv;
                const uint32_t end = min(kRows, n_rows - tile2 * kRows) * (D / 32);  // lines of 128 bytes
                for (uint32_t i = lane; i < end; i += 32) {
                    const uint32_t which = tile2 * kRows + i / (D / 32);
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(a.q + which / group * a.q_stride +
                                                                  (size_t)(kvh2 * group + which % group) * D + i % (D / 32) * 32));
                }
            }
            // ---- INT8: the scales, those of the values relative to the running maximum's power of two, or (wide weights) as
            // they are, which is what relative to 2^13 would be
            if constexpr (kI8) {
                float sc[4];  // key and value scales of keys lane, lane + 32 of the next block
                auto load = [&](uint32_t g) {
#pragma unroll
                    for (uint32_t i = 0; i < 2; ++i) {
                        const uint32_t key = g * kKeys + lane + 32 * i;
                        sc[i] = key < keys ? c.k_scale[line0 + key] : 0.f, sc[2 + i] = key < keys ? c.v_scale[line0 + key] : 0.f;
                    }
                };
                Scales st;
                bool ok = true;
                load(0);
                for (uint32_t g = 0; g < n_blocks; ++g) {
                    const uint32_t s = g % kStages;
                    look(st, g, sc[2], sc[3]);
                    const int e = st.wide ? 13 : st.e_max;
                    const float mul = st.wide ? 1.f : pow2(-1 - e) * kWeightScale;
                    ok = mbar_wait(v_empty + s, ((g / kStages) & 1) ^ 1, abort_flag, a.wait_limit);
                    if (!ok) break;
                    float *dst = scales + s * S::kScaleFloats;
                    dst[lane] = sc[0], dst[32 + lane] = sc[1];
                    dst[2 * kKeys + lane] = sc[0] * kKeyShrink, dst[2 * kKeys + 32 + lane] = sc[1] * kKeyShrink;
                    dst[kKeys + lane] = sc[2] * mul, dst[kKeys + 32 + lane] = sc[3] * mul;
                    if (lane == 0) *reinterpret_cast<int2 *>(dst + 3 * kKeys) = make_int2(e, st.wide);
                    load(g + 1);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(v_full + s);
                }
                if (!ok) *abort_flag = 1;
            }
        } else {
            // ---- products
            constexpr uint32_t kind = kI8 ? 0 : 1;
            const uint32_t idesc_s = instruction(kKeys, 0, kind), idesc_o = instruction(D, 1, kind), idesc_wide = instruction(D, 1, 1);
            const uint64_t q_desc = umma_desc(smem_u32(qs)), k_desc = umma_desc(smem_u32(ring));
            // (MN-major: chunks of 64 channels kChunkBytes apart)
            const uint64_t v_desc = umma_desc(smem_u32(v_ring)) | ((uint64_t)(S::kChunkBytes >> 4) << 16);
            auto scores = [&](uint32_t g) {  // (one lane) small terms first
                const uint64_t kd = k_desc + (uint64_t)((g % kStages) * (S::kTileBytes >> 4));
                const uint32_t dst = tmem + S::score_col(g);
#pragma unroll
                for (uint32_t i = 0; i < kTerms; ++i)
#pragma unroll
                    for (uint32_t k = 0; k < 4 * kChunks; ++k) {
                        const uint64_t kk = kd + ((k / 4 * S::kChunkBytes + k % 4 * 32) >> 4);
                        mma_ss(dst, q_desc + (((kTerms - 1 - i) * S::kQTermBytes + k / 4 * S::kQChunkBytes + k % 4 * 32) >> 4), kk,
                               idesc_s, i + k != 0);
                    }
                umma_commit(k_empty + g % kStages);
                umma_commit(s_full + g % kAhead);
            };
            auto values = [&](uint32_t g, bool wide) {  // (one lane) small terms first
                const uint64_t vd = v_desc + (uint64_t)((g % kStages) * (S::kTileBytes >> 4));
                const uint32_t dst = tmem + S::out_col(g & 1), idesc = wide ? idesc_wide : idesc_o;
                if (wide)
#pragma unroll
                    for (uint32_t k = 0; k < kKeys / 16; ++k)
                        mma_ts(dst, tmem + S::weight_col(g, 2, k), vd + ((k * 2048) >> 4), idesc, k != 0);
#pragma unroll
                for (uint32_t k = 0; k < kKeys / 16; ++k)
                    mma_ts(dst, tmem + S::weight_col(g, 1, k), vd + ((k * 2048) >> 4), idesc, wide || k != 0);
                if constexpr (kI8) mma_ts_above(dst, tmem + S::weight_col(g, 0, 0), vd, idesc);
                else mma_ts(dst, tmem + S::weight_col(g, 0, 0), vd, idesc, true);
#pragma unroll
                for (uint32_t k = 1; k < kKeys / 16; ++k)
                    mma_ts(dst, tmem + S::weight_col(g, 0, k), vd + ((k * 2048) >> 4), idesc, true);
                umma_commit(v_empty + g % kStages);
                umma_commit(o_full + (g & 1));
            };
            bool ok = mbar_wait(q_full, 0, abort_flag, a.wait_limit);
            for (uint32_t g = 0; g < kAhead && g < n_blocks && ok; ++g) {
                ok = mbar_wait(k_full + g % kStages, (g / kStages) & 1, abort_flag, a.wait_limit);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) scores(g);
                __syncwarp();
            }
            uint32_t g = 0;
            auto issue = [&](auto wide_tag) {  // block g; false: the weights are of the other form, or a wait ran out
                constexpr bool kWide = decltype(wide_tag)::value;
                const bool more = g + kAhead < n_blocks;
                // (INT8: the units have waited for the values' stage, whose scales they need, before they gave the weights)
                if constexpr (!kI8) ok = mbar_wait(v_full + g % kStages, (g / kStages) & 1, abort_flag, a.wait_limit);
                if (ok) ok = mbar_wait(p_full + (g & 1), (g >> 1) & 1, abort_flag, a.wait_limit);
                if (!ok) return false;
                if constexpr (!kWide) {
                    const int wide = reinterpret_cast<const int *>(scales + (g % kStages) * S::kScaleFloats)[3 * kKeys + 1];
                    if (__any_sync(0xffffffffu, wide)) return false;
                }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) values(g, kWide);
                __syncwarp();
                if (more) {
                    ok = mbar_wait(k_full + (g + kAhead) % kStages, ((g + kAhead) / kStages) & 1, abort_flag, a.wait_limit);
                    if (!ok) return false;
                    if (elect_one()) scores(g + kAhead);  // (over columns whose weights the product before reads first)
                    __syncwarp();
                }
                ++g;
                return true;
            };
            if constexpr (kI8)
                while (g < n_blocks && ok && issue(std::false_type{})) {}
            while (g < n_blocks && ok && issue(std::true_type{})) {}
            if (!ok) *abort_flag = 1;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kUnitRegs));
        const uint32_t u = warp / 4, r = threadIdx.x % 128;
        const uint32_t query = min(row0 + r, n_rows - 1) / group;
        // q: a warp takes sixteen rows, D / 4 lanes a row
        {
            constexpr uint32_t kLanes = D / 4, kSide = 32 / kLanes;
            const uint32_t ch = 4 * (lane % kLanes);
            const float unit_scale = kLog2E / sqrtf((float)D);
            constexpr uint32_t kTurns = 16 / kSide;
            float4 held[kTurns];
            // (rows past the last repeat it)
            const uint32_t which = row0 + min(warp * 16 + lane % 16, rows - 1);
            const size_t where = which / group * a.q_stride + (size_t)(kvh * group + which % group) * D;  // of the row lane % 16
#pragma unroll
            for (uint32_t i = 0; i < kTurns; ++i)
                held[i] = __ldg(reinterpret_cast<const float4 *>(a.q + __shfl_sync(0xffffffffu, where, i * kSide + lane / kLanes) + ch));
#pragma unroll
            for (uint32_t i = 0; i < kTurns; ++i) {
                const uint32_t at = warp * 16 + i * kSide + lane / kLanes;
                // In log2 units from here on: what is left to do to a raw score is a power of two, so that its product with that
                // is exact and the largest score less the maximum is zero, however large it is.
                const float4 x = make_float4(held[i].x * unit_scale, held[i].y * unit_scale, held[i].z * unit_scale, held[i].w * unit_scale);
                float factor = 1.f, mul = 1.f;
                if constexpr (kI8) {
                    uint32_t top = max(max(__float_as_uint(fabsf(x.x)), __float_as_uint(fabsf(x.y))),
                                       max(__float_as_uint(fabsf(x.z)), __float_as_uint(fabsf(x.w))));
                    if constexpr (kLanes == 32) {
                        top = __reduce_max_sync(0xffffffffu, top);
                    } else {
#pragma unroll
                        for (uint32_t off = kLanes / 2; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
                    }
                    const int e = exponent_of(top);
                    mul = pow2(14 - e);
                    // (an infinity or NaN: the row is NaN)
                    factor = top < 0x7f800000u ? pow2(e - 14) : __int_as_float(0x7fffffff);
                }
                uint32_t t0[3], t1[3];
                if constexpr (kI8) {
                    terms_f16(x.x * mul, x.y * mul, 1.f, t0);
                    terms_f16(x.z * mul, x.w * mul, 1.f, t1);
                } else {
                    split3(x.x, x.y, t0);
                    split3(x.z, x.w, t1);
                }
                uint8_t *to = qs + ch / 64 * S::kQChunkBytes + at * 128 + (((ch % 64 / 8) ^ (at & 7)) << 4) + ch % 8 * 2;
#pragma unroll
                for (uint32_t n = 0; n < kTerms; ++n) *reinterpret_cast<uint2 *>(to + n * S::kQTermBytes) = make_uint2(t0[n], t1[n]);
                if (lane % kLanes == 0) row_factor[at] = factor;
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            asm volatile("bar.sync 3, 256;" ::: "memory");
        }
        const float f = kI8 ? row_factor[r] : 1.f;
        // A raw score is below 2^29, and times its key's scale it may leave float32's range although f brings it back: unless
        // f is so large that nothing comes back, scales are taken that are 2^30 smaller (what these lose of scales below 2^-96
        // is nothing after f).
        const bool large = f >= 0x1p46f;  // (a query of 2^60 or more)
        const uint32_t which_scales = large ? 0 : 2 * kKeys;
        const float to_log2 = !kI8 || large ? f : f * (1.f / kKeyShrink);
        const uint32_t outs = tmem + S::out_col(u) + (((warp % 4) * 32) << 16);
        // keys of this CTA that this row sees
        const int seen = a.causal ? (int)(a.first_row + query) + 1 - (int)(block0 * kKeys) : (int)keys;
        float m = -INFINITY, l = 0.f;
        int e_here = -110;
        float o[D];
#pragma unroll
        for (int i = 0; i < D; ++i) o[i] = 0.f;
        bool ok = true;
        float alpha = 1.f;  // of the block whose product has not joined the output yet
        // The product of the unit's block before joins the output (in registers: the sum is rounded, not truncated).
        auto take_output = [&](uint32_t done) {
            ok = mbar_wait(o_full + u, done & 1, abort_flag, a.wait_limit);
            if (!ok) return;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            each16<D / 16>(outs, [&](int part, const uint32_t (&w)[16]) {
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float2 x = __ffma2_rn(make_float2(o[16 * part + i], o[16 * part + i + 1]), make_float2(alpha, alpha),
                                                make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1])));
                    o[16 * part + i] = x.x, o[16 * part + i + 1] = x.y;
                }
            });
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        };
        uint32_t it = 0;
        for (uint32_t g = u; g < n_blocks; g += 2, ++it) {
            const int key0 = (int)(g * kKeys);
            const uint32_t lanes = tmem + (((warp % 4) * 32) << 16), cols = lanes + S::score_col(g);
            // (the scales come with the values, most often before the scores)
            if (!kI8 || !both_ready(v_full + g % kStages, (g / kStages) & 1, s_full + g % kAhead, (g / kAhead) & 1)) {
                if (kI8) ok = mbar_wait(v_full + g % kStages, (g / kStages) & 1, abort_flag, a.wait_limit);
                ok = ok && mbar_wait(s_full + g % kAhead, (g / kAhead) & 1, abort_flag, a.wait_limit);
            }
            if (!ok) break;  // (a warp at a time: the others' waits end with the flag below)
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const int limit = min(seen, (int)keys) - key0;  // keys of the block that this row sees
            const float *ks = scales + (g % kStages) * S::kScaleFloats, *vs = ks + kKeys;
            float alpha_new;
            float2 sum = make_float2(0.f, 0.f);
            // (kEdge in the type: a select per score would be paid in every block.  INT8: wide weights, at edges or not.)
            auto weights = [&](auto edge_tag) {
                constexpr bool kEdge = decltype(edge_tag)::value;
                constexpr uint32_t kOfWeights = kI8 && !kEdge ? 2 : 3;
                float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                each16<kKeys / 16>(cols, [&](int part, const uint32_t (&s)[16]) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const int at = 16 * part + e;
                        float4 x = make_float4(__uint_as_float(s[e]), __uint_as_float(s[e + 1]), __uint_as_float(s[e + 2]),
                                               __uint_as_float(s[e + 3]));
                        if constexpr (kI8) {
                            const float4 k4 = *reinterpret_cast<const float4 *>(ks + which_scales + at);
                            const float2 lo = __fmul2_rn(make_float2(x.x, x.y), make_float2(k4.x, k4.y));
                            const float2 hi = __fmul2_rn(make_float2(x.z, x.w), make_float2(k4.z, k4.w));
                            x = make_float4(lo.x, lo.y, hi.x, hi.y);
                        }
                        if constexpr (kEdge) {
                            x.x = at < limit ? x.x : -INFINITY;
                            x.y = at + 1 < limit ? x.y : -INFINITY;
                            x.z = at + 2 < limit ? x.z : -INFINITY;
                            x.w = at + 3 < limit ? x.w : -INFINITY;
                        }
                        t4[0] = fmaxf(t4[0], x.x), t4[1] = fmaxf(t4[1], x.y), t4[2] = fmaxf(t4[2], x.z), t4[3] = fmaxf(t4[3], x.w);
                    }
                });
                const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
                const float m_new = fmaxf(m, top * to_log2);
                const float base = m_new == -INFINITY ? 0.f : m_new;  // (nothing seen yet: every weight is zero)
                alpha_new = ex2(m - base);
                m = m_new;
                if (it) take_output(it - 1);
                if (!ok) return;
                const float2 f2 = make_float2(to_log2, to_log2), base2 = make_float2(-base, -base);
                each16<kKeys / 16>(cols, [&](int part, const uint32_t (&s)[16]) {
                    uint32_t t[kOfWeights][8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float2 x = make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
                        const int at = 16 * part + 2 * e;
                        // (to_log2 is a power of two: this is the difference of what the maximum was formed from)
                        if constexpr (kI8) x = __fmul2_rn(x, *reinterpret_cast<const float2 *>(ks + which_scales + at));
                        x = __ffma2_rn(x, f2, base2);
                        if constexpr (kEdge) {
                            x.x = at < limit ? x.x : -INFINITY;
                            x.y = at + 1 < limit ? x.y : -INFINITY;
                        }
                        x = make_float2(ex2(x.x), ex2(x.y));
                        sum = __fadd2_rn(sum, x);
                        if constexpr (kI8) {
                            x = __fmul2_rn(x, *reinterpret_cast<const float2 *>(vs + at));
                            if constexpr (kEdge) {  // (a key that this row does not see may have the scale NaN)
                                x.x = at < limit ? x.x : 0.f;
                                x.y = at + 1 < limit ? x.y : 0.f;
                            }
                        }
                        uint32_t w[3];
                        if constexpr (kOfWeights == 2) terms_f16(x.x, x.y, (float)(1 << kLowBits), w);
                        else terms_bf16(x.x, x.y, kI8 ? (float)(1 << kLowBits) : 1.f, w);
#pragma unroll
                        for (uint32_t n = 0; n < kOfWeights; ++n) t[n][e] = w[n];
                    }
#pragma unroll
                    for (uint32_t n = 0; n < kOfWeights; ++n) tmem_st8(lanes + S::weight_col(g, n, part), t[n]);
                });
            };
            const int2 form = kI8 ? *reinterpret_cast<const int2 *>(ks + 3 * kKeys) : make_int2(0, at_edge(g));  // E, wide
            if (form.y) weights(std::true_type{});
            else weights(std::false_type{});
            if (!ok) break;
            l = fmaf(l, alpha_new, sum.x + sum.y);
            alpha = alpha_new;
            if constexpr (kI8) {
                alpha *= pow2(max(-126, e_here - form.x));
                e_here = form.x;
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + u);
        }
        if (ok && it) take_output(it - 1);
        if constexpr (!kI8) {  // infinities and NaNs that the loaders took out, to the rows that see their keys
#pragma unroll 1
            for (uint32_t e = 0; ok && a.causal && e < min(kEdges, n_blocks); ++e) {
                const uint32_t g = n_blocks - 1 - e;
                if (g % 2 != u) continue;  // (the other unit's block)
#pragma unroll 1
                for (uint32_t half = 0; half < 2; ++half) {
                    uint32_t marked = spoilt[2 * e + half];
#pragma unroll 1
                    for (; marked; marked &= marked - 1) {
                        const uint32_t key = g * kKeys + 32 * half + __ffs(marked) - 1;
                        if ((int)key >= seen) break;
                        const uint4 *v = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(c.v) + (line0 + key) * (2 * D));
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) {
                            const uint4 w = __ldg(v + i);
                            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                if ((x[j] & 0x7f80u) == 0x7f80u) o[8 * i + 2 * j] += __uint_as_float(x[j] << 16);
                                if ((x[j] & 0x7f800000u) == 0x7f800000u) o[8 * i + 2 * j + 1] += __uint_as_float(x[j] & 0xffff0000u);
                            }
                        }
                    }
                }
            }
        }
        if (!ok) *abort_flag = 1;
        // ---- the units join: each finishes half of the channels and hands the others over, through the ring (every
        // product has been read out, every block consumed once both units are here)
        ok = vote<3, 256>(ok);
        if (ok) {
            constexpr int kHalf = D / 2;
            const float undo = kI8 ? pow2(e_here + 1) * (1.f / kWeightScale) : 1.f;
            float *swap = reinterpret_cast<float *>(ring), *stat = swap + 2 * kHalf * kRows;  // [unit][channel][128], [unit][m, l][128]
            float4 *mine = reinterpret_cast<float4 *>(swap + u * kHalf * kRows);  // [four channels][row]
#pragma unroll
            for (int i = 0; i < kHalf; i += 4)
                mine[i / 4 * kRows + r] = make_float4((u ? o[i] : o[kHalf + i]) * undo, (u ? o[i + 1] : o[kHalf + i + 1]) * undo,
                                                      (u ? o[i + 2] : o[kHalf + i + 2]) * undo, (u ? o[i + 3] : o[kHalf + i + 3]) * undo);
            stat[u * 256 + r] = m;
            stat[u * 256 + 128 + r] = l;
            asm volatile("bar.sync 3, 256;" ::: "memory");
            const float m2 = stat[(u ^ 1) * 256 + r], l2 = stat[(u ^ 1) * 256 + 128 + r];
            const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
            // (a unit without a key that the row sees has the sum 0; a NaN stays)
            const float w1 = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - base);
            const float w2 = m2 == -INFINITY ? (l2 == 0.f ? 0.f : 1.f) : ex2(m2 - base);
            const float sum = l * w1 + l2 * w2;
            const bool direct = a.n_slots == 1;
            const float inv = !direct ? 1.f : sum == 0.f ? 0.f : 1.f / sum;
            const float a1 = w1 * inv * undo, a2 = w2 * inv;
            const float4 *other = reinterpret_cast<const float4 *>(swap + (u ^ 1) * kHalf * kRows);
            // (through shared memory, where q has been, so that rows are written whole: pieces of 16 bytes, swizzled)
            if (u == 0) row_factor[r] = top, stat[512 + r] = sum;
            uint8_t *line = qs + r * (D * 4);
#pragma unroll
            for (int i = 0; i < kHalf; i += 4) {
                const float4 y = other[i / 4 * kRows + r];
                const float x[4] = {fmaf(u ? o[kHalf + i] : o[i], a1, y.x * a2), fmaf(u ? o[kHalf + i + 1] : o[i + 1], a1, y.y * a2),
                                    fmaf(u ? o[kHalf + i + 2] : o[i + 2], a1, y.z * a2),
                                    fmaf(u ? o[kHalf + i + 3] : o[i + 3], a1, y.w * a2)};
                *reinterpret_cast<float4 *>(line + (((u * kHalf + i) / 4 ^ (r & 7)) << 4)) = make_float4(x[0], x[1], x[2], x[3]);
            }
            asm volatile("bar.sync 3, 256;" ::: "memory");
            constexpr uint32_t kLanes = D / 4, kSide = 32 / kLanes;
            float2 *stats = reinterpret_cast<float2 *>(a.scratch + (size_t)a.n_queries * a.n_heads * a.n_slots * D);
            const uint32_t ch = lane % kLanes, which = row0 + min(warp * 16 + lane % 16, rows - 1);
            // where the row lane % 16 goes, and (lanes below 16) its sums
            const size_t head = (size_t)(which / group) * a.n_heads + kvh * group + which % group;
            const size_t at_slot = head * a.n_slots + a.slot0 + split;
            const size_t where = direct ? which / group * a.out_stride + (size_t)(kvh * group + which % group) * D : at_slot * D;
            if (!direct && lane < 16 && warp * 16 + lane < rows)
                stats[at_slot] = make_float2(row_factor[warp * 16 + lane], stat[512 + warp * 16 + lane]);
            float *base_out = direct ? a.out : a.scratch;
            const bool wide = ((uintptr_t)base_out & 15) == 0 && (!direct || a.out_stride % 4 == 0);
#pragma unroll 4
            for (uint32_t i = 0; i < 16; i += kSide) {
                const uint32_t at = warp * 16 + i + lane / kLanes;
                float *dst = base_out + __shfl_sync(0xffffffffu, where, i + lane / kLanes) + 4 * ch;
                if (at >= rows) continue;
                const float4 x = *reinterpret_cast<const float4 *>(qs + at * (D * 4) + ((ch ^ (at & 7)) << 4));
                if (wide) *reinterpret_cast<float4 *>(dst) = x;
                else dst[0] = x.x, dst[1] = x.y, dst[2] = x.z, dst[3] = x.w;
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == kMmaWarp && *abort_flag) {  // the products still in flight (whichever warp gave up)
        if (elect_one()) umma_commit(drain);
        __syncwarp();
        (void)mbar_wait(drain, 0, never, kWaitLimit);
    }
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    if (threadIdx.x == 0 && *abort_flag) atomicOr(a.error, 1);
}

template <bool kI8, int D>
qk_status launch_tile(qk_ctx *c, const CacheView &cache, const TileArgs &a) {
    qk_status st = qk::allow_smem(c, attend_tile_kernel<kI8, D>, TileShape<kI8, D>::kSmem);
    if (st != QK_OK) return st;
    const uint32_t tiles = (uint32_t)qk::ceil_div((size_t)a.n_queries * (a.n_heads / cache.n_kv), kRows);
    (void)qk::launch_pdl(c->pdl, attend_tile_kernel<kI8, D>, dim3(cache.n_kv * tiles, a.n_splits), dim3(kThreads),
                         (size_t)TileShape<kI8, D>::kSmem, c->stream, cache, a);
    QK_CUDA(cudaGetLastError());
    c->launches++;
    c->err_armed = true;
    return QK_OK;
}

}  // namespace

namespace qk {

qk_status attend_tiles(qk_ctx *c, const CacheView &cache, TileArgs a) {
    a.error = (int *)c->d_err.ptr;
    a.wait_limit = c->wait_limit ? c->wait_limit : kWaitLimit;
    if (cache.dtype == QK_I8) return cache.d == 128 ? launch_tile<true, 128>(c, cache, a) : launch_tile<true, 64>(c, cache, a);
    return cache.d == 128 ? launch_tile<false, 128>(c, cache, a) : launch_tile<false, 64>(c, cache, a);
}

}  // namespace qk
