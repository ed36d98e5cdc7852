// Attention of many query rows over one slot's cache rows on tcgen05: a prompt's portion, and a prefix that a whole
// batch shares.  INT8 and bfloat16 caches, head sizes 64 and 128.
//
// The queries that read one kv head are the rows of one product: row r is query r / group, head r % group of the kv
// head, 128 rows to a CTA, which takes a range of keys 64 at a time.  Two units of four warps take the key blocks in
// turn, a thread owns a row (no shuffles): running maximum, sum and output in registers, the two units joined at the
// end.  While one unit is at its exponentials the tensor core works for the other.  The weights go back to tensor
// memory as the A operand; v is read as it lies (MN-major B).  Three warps bring the key blocks in.
//
// Exactness.  INT8 rows: codes as float16 are exact (three warps convert them on their way into shared memory); q is
// two float16 terms after scaling by a power of two per row (22 bits), and so are the weights times the value scales,
// which are taken relative to a power of two at their running maximum E and scaled to 2^14.  bfloat16 rows go in as
// they are; q and the weights are three bfloat16 terms.  A block's product with v starts from zero and is added to the
// row's output in registers, in float32: the tensor core truncates.
//
// What bounds it: shared memory (the tensor core reads q anew for every block) and the instructions per score.
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
constexpr uint32_t kThreads = 384, kLoaders = 96, kFirstLoader = 8, kMmaWarp = 11;
constexpr int kUnitRegs = 208, kOtherRegs = 88, kLaunchRegs = 168;
static_assert(2 * 128 * kUnitRegs + 128 * kOtherRegs <= (int)kThreads * kLaunchRegs, "setmaxnreg draws on the launch's registers");
constexpr uint32_t kTmemCols = 512, kUnitCols = 256, kOutCol = 128;  // a unit's columns: scores, weights, outputs
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kWeightScale = 16384.f;
constexpr uint32_t kWaitLimit = 1u << 22;

template <bool kI8, int D>
struct TileShape {
    static constexpr uint32_t kTerms = kI8 ? 2 : 3;                    // of q and of the weights
    static constexpr uint32_t kChunks = D / 64;                        // of 64 channels, rows of 128 bytes
    static constexpr uint32_t kChunkBytes = kKeys * 128, kTileBytes = kChunks * kChunkBytes;
    static constexpr uint32_t kQChunkBytes = kRows * 128, kQTermBytes = kChunks * kQChunkBytes;
    static constexpr uint32_t kStages = kI8 || D == 64 ? 4 : 3, kStageBytes = 2 * kTileBytes;
    static constexpr uint32_t kScaleFloats = kI8 ? 2 * kKeys + 4 : 0;  // a stage's key and value scales, and E
    static constexpr uint32_t kSmem = 1024 + kTerms * kQTermBytes + kStages * kStageBytes + kStages * kScaleFloats * 4 + 1024 + 256;
    static_assert(kSmem <= 227 * 1024, "shared memory of a CTA");
    static_assert(kStages * kStageBytes >= (D * kRows + 4 * kRows) * 4, "the units' exchange lies in the ring");
    // Column of the weights' term n; the third lies over scores that have been read.
    __device__ static constexpr uint32_t weight_col(uint32_t n) { return n == 2 ? 0 : 64 + 32 * n; }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(uint32_t magnitude_bits) {  // clamped to -100 .. 125
    return min(125, max(-100, (int)(magnitude_bits >> 23) - 127));
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
// Two values as their terms, float16 or bfloat16 pairs; t[0] the leading one.
template <bool kI8>
__device__ __forceinline__ void terms_of(float a, float b, uint32_t *t) {
    if constexpr (kI8) {
        t[0] = pack_f16x2(a, b);
        const float2 h = __half22float2(*reinterpret_cast<__half2 *>(&t[0]));
        t[1] = pack_f16x2(a - h.x, b - h.y);
    } else {
        uint32_t w[3];
        split3(a, b, w);
        t[0] = w[0], t[1] = w[1], t[2] = w[2];
    }
}
// Four codes as float16: 1024 + u is the bit pattern 0x6400 | u, u = code + 128.
__device__ __forceinline__ void codes_to_f16(uint32_t codes, uint32_t &lo, uint32_t &hi) {
    const uint32_t u = codes ^ 0x80808080u;
    lo = __byte_perm(u, 0x64646464u, 0x4140);
    hi = __byte_perm(u, 0x64646464u, 0x4342);
    asm("{\n .reg .b32 c;\n mov.b32 c, 0x64806480;\n sub.rn.f16x2 %0, %0, c;\n sub.rn.f16x2 %1, %1, c;\n}" : "+r"(lo), "+r"(hi));
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Grid (kv heads x tiles of 128 rows, splits of the keys); late tiles see most keys: they go first.
template <bool kI8, int D>
__global__ void __launch_bounds__(kThreads, 1)
attend_tile_kernel(CacheView c, TileArgs a) {
    using S = TileShape<kI8, D>;
    constexpr uint32_t kTerms = S::kTerms, kChunks = S::kChunks, kStages = S::kStages;
    qk::pdl_launch();
    extern __shared__ __align__(1024) uint8_t raw_smem[];
    uint8_t *qs = raw_smem + (-smem_u32(raw_smem) & 1023u);  // (an offset: the compiler still sees shared memory)
    uint8_t *ring = qs + kTerms * S::kQTermBytes;
    float *scales = reinterpret_cast<float *>(ring + kStages * S::kStageBytes);  // [stage][kScaleFloats]
    float *row_peak = scales + kStages * S::kScaleFloats;                       // [2][128]
    uint64_t *q_full = reinterpret_cast<uint64_t *>(row_peak + 256);
    uint64_t *full = q_full + 1, *empty = full + kStages, *s_full = empty + kStages, *p_full = s_full + 2, *o_full = p_full + 2;
    uint64_t *drain = o_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int *never = reinterpret_cast<volatile int *>(tmem_slot + 2);
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
            mbar_init(full + s, kLoaders / 32);
            mbar_init(empty + s, 1);
        }
        for (int u = 0; u < 2; ++u) {
            mbar_init(s_full + u, 1);
            mbar_init(p_full + u, 4);
            mbar_init(o_full + u, 1);
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        *never = 0;
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

    if (warp >= kFirstLoader) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp != kMmaWarp) {
            // ---- key blocks into the ring; rows past the end are zeros
            const uint32_t tid = threadIdx.x - kFirstLoader * 32;
            constexpr uint32_t kRowBytes = kI8 ? D : 2 * D, kPieces = kRowBytes / 16, kStep = kLoaders / kPieces;
            constexpr uint32_t kPasses = (kKeys + kStep - 1) / kStep;
            const uint32_t piece = tid % kPieces, first = tid / kPieces;  // a thread's rows: first, first + kStep, ..
            const uint8_t *kb = static_cast<const uint8_t *>(c.k) + line0 * kRowBytes + piece * 16;
            const uint8_t *vb = static_cast<const uint8_t *>(c.v) + line0 * kRowBytes + piece * 16;
            bool ok = true;
            if constexpr (kI8) {
                uint4 held[kPasses];
                auto load = [&](const uint8_t *base, uint32_t g) {
#pragma unroll
                    for (uint32_t i = 0; i < kPasses; ++i) {
                        const uint32_t row = first + i * kStep, key = g * kKeys + row;
                        held[i] = row < kKeys && key < keys ? __ldg(reinterpret_cast<const uint4 *>(base + (size_t)key * kRowBytes))
                                                            : make_uint4(0u, 0u, 0u, 0u);
                    }
                };
                auto store = [&](uint8_t *to) {  // sixteen codes: two pieces of eight float16
#pragma unroll
                    for (uint32_t i = 0; i < kPasses; ++i) {
                        const uint32_t row = first + i * kStep;
                        if (row >= kKeys) break;
                        uint32_t w[8];
                        codes_to_f16(held[i].x, w[0], w[1]);
                        codes_to_f16(held[i].y, w[2], w[3]);
                        codes_to_f16(held[i].z, w[4], w[5]);
                        codes_to_f16(held[i].w, w[6], w[7]);
                        uint8_t *line = to + piece / 4 * S::kChunkBytes + row * 128;
                        const uint32_t at = 2 * (piece % 4), flip = piece / 4;  // (the two chunks in turn: no bank twice)
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            const bool second = (h ^ flip) != 0;
                            *reinterpret_cast<uint4 *>(line + (((at + (second ? 1 : 0)) ^ (row & 7)) << 4)) =
                                second ? make_uint4(w[4], w[5], w[6], w[7]) : make_uint4(w[0], w[1], w[2], w[3]);
                        }
                    }
                };
                int e_max = -100;
                load(kb, 0);
                for (uint32_t g = 0; g < n_blocks; ++g) {
                    const uint32_t s = g % kStages;
                    float sc[4] = {0.f, 0.f, 0.f, 0.f};  // (first warp) key and value scales of keys lane, lane + 32
                    if (warp == kFirstLoader) {
#pragma unroll
                        for (uint32_t i = 0; i < 2; ++i) {
                            const uint32_t key = g * kKeys + lane + 32 * i;
                            if (key < keys) sc[i] = c.k_scale[line0 + key], sc[2 + i] = c.v_scale[line0 + key];
                        }
                    }
                    ok = mbar_wait(empty + s, ((g / kStages) & 1) ^ 1, abort_flag, a.wait_limit);
                    if (!ok) break;
                    uint8_t *stage = ring + s * S::kStageBytes;
                    store(stage);
                    load(vb, g);
                    if (warp == kFirstLoader) {
                        const uint32_t top = __reduce_max_sync(
                            0xffffffffu, max(__float_as_uint(fabsf(sc[2])), __float_as_uint(fabsf(sc[3]))));
                        e_max = max(e_max, exponent_of(top));
                        const float mul = pow2(-1 - e_max);
                        float *dst = scales + s * S::kScaleFloats;
                        dst[lane] = sc[0], dst[32 + lane] = sc[1];
                        dst[kKeys + lane] = sc[2] * mul * kWeightScale, dst[kKeys + 32 + lane] = sc[3] * mul * kWeightScale;
                        if (lane == 0) reinterpret_cast<int *>(dst)[2 * kKeys] = e_max;
                    }
                    store(stage + S::kTileBytes);
                    if (g + 1 < n_blocks) load(kb, g + 1);
                    fence_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + s);
                }
            } else {
                auto copy = [&](const uint8_t *base, uint8_t *to, uint32_t g) {
#pragma unroll
                    for (uint32_t i = 0; i < kPasses; ++i) {
                        const uint32_t row = first + i * kStep, key = g * kKeys + row;
                        if (row >= kKeys) break;
                        const bool live = key < keys;
                        const uint32_t at = smem_u32(to + piece / 8 * S::kChunkBytes + row * 128 + (((piece % 8) ^ (row & 7)) << 4));
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at),
                                     "l"(base + (live ? (size_t)key * kRowBytes : 0)), "r"(live ? 16u : 0u)
                                     : "memory");
                    }
                };
                for (uint32_t g = 0; g < n_blocks + 1; ++g) {  // (a block is handed over when the next one is under way)
                    if (g < n_blocks) {
                        ok = mbar_wait(empty + g % kStages, ((g / kStages) & 1) ^ 1, abort_flag, a.wait_limit);
                        if (!ok) break;
                        uint8_t *stage = ring + g % kStages * S::kStageBytes;
                        copy(kb, stage, g);
                        copy(vb, stage + S::kTileBytes, g);
                    }
                    asm volatile("cp.async.commit_group;" ::: "memory");
                    if (g == 0) continue;
                    asm volatile("cp.async.wait_group 1;" ::: "memory");
                    fence_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + (g - 1) % kStages);
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
            }
            if (!ok) *abort_flag = 1;
        } else {
            // ---- products
            constexpr uint32_t kind = kI8 ? 0 : 1;
            const uint32_t idesc_s = instruction(kKeys, 0, kind), idesc_o = instruction(D, 1, kind);
            const uint64_t q_desc = umma_desc(smem_u32(qs)), k_desc = umma_desc(smem_u32(ring));
            // (MN-major: chunks of 64 channels kChunkBytes apart)
            const uint64_t v_desc = umma_desc(smem_u32(ring) + S::kTileBytes) | ((uint64_t)(S::kChunkBytes >> 4) << 16);
            auto scores = [&](uint32_t g) {  // (one lane) small terms first
                const uint64_t kd = k_desc + (uint64_t)((g % kStages) * (S::kStageBytes >> 4));
                const uint32_t dst = tmem + kUnitCols * (g & 1);
#pragma unroll
                for (uint32_t i = 0; i < kTerms; ++i)
#pragma unroll
                    for (uint32_t k = 0; k < 4 * kChunks; ++k)
                        mma_ss(dst, q_desc + (((kTerms - 1 - i) * S::kQTermBytes + k / 4 * S::kQChunkBytes + k % 4 * 32) >> 4),
                               kd + ((k / 4 * S::kChunkBytes + k % 4 * 32) >> 4), idesc_s, i + k != 0);
                umma_commit(s_full + (g & 1));
            };
            auto values = [&](uint32_t g) {  // (one lane)
                const uint64_t vd = v_desc + (uint64_t)((g % kStages) * (S::kStageBytes >> 4));
                const uint32_t unit = tmem + kUnitCols * (g & 1);
#pragma unroll
                for (uint32_t i = 0; i < kTerms; ++i)
#pragma unroll
                    for (uint32_t k = 0; k < kKeys / 16; ++k)
                        mma_ts(unit + kOutCol, unit + S::weight_col(kTerms - 1 - i) + k * 8, vd + ((k * 2048) >> 4), idesc_o,
                               i + k != 0);
                umma_commit(empty + g % kStages);
                umma_commit(o_full + (g & 1));
            };
            bool ok = mbar_wait(q_full, 0, abort_flag, a.wait_limit);
            for (uint32_t g = 0; g < 2 && g < n_blocks && ok; ++g) {
                ok = mbar_wait(full + g % kStages, 0, abort_flag, a.wait_limit);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) scores(g);
                __syncwarp();
            }
            for (uint32_t g = 0; g < n_blocks && ok; ++g) {
                ok = mbar_wait(p_full + (g & 1), (g >> 1) & 1, abort_flag, a.wait_limit);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) values(g);
                __syncwarp();
                if (g + 2 >= n_blocks) continue;
                ok = mbar_wait(full + (g + 2) % kStages, ((g + 2) / kStages) & 1, abort_flag, a.wait_limit);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (elect_one()) scores(g + 2);  // (over scores that the unit has read: it has handed in their weights)
                __syncwarp();
            }
            if (!ok) *abort_flag = 1;
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kUnitRegs));
        const uint32_t u = warp / 4, r = threadIdx.x % 128;
        const uint32_t row = min(row0 + r, n_rows - 1), query = row / group, head = kvh * group + row % group;
        // q: a unit takes one chunk of 64 channels, a thread its row
        float f = kLog2E / sqrtf((float)D);  // what turns a raw score into log2 units
        {
            const bool live = r < rows && u < kChunks;
            const float *src = a.q + query * a.q_stride + (size_t)head * D + u * 64;
            float x[64];
#pragma unroll
            for (int i = 0; i < 64; i += 4) {
                const float4 t = live ? *reinterpret_cast<const float4 *>(src + i) : make_float4(0.f, 0.f, 0.f, 0.f);
                x[i] = t.x, x[i + 1] = t.y, x[i + 2] = t.z, x[i + 3] = t.w;
            }
            float mul = 1.f;
            if constexpr (kI8) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < 64; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
                row_peak[u * 128 + r] = __uint_as_float(top);
                asm volatile("bar.sync 3, 256;" ::: "memory");
                top = max(top, __float_as_uint(row_peak[(u ^ 1) * 128 + r]));
                const int e = exponent_of(top);
                mul = pow2(14 - e);
                f = top < 0x7f800000u ? f * pow2(e - 14) : __int_as_float(0x7fffffff);  // (an infinity or NaN: the row is NaN)
            }
            if (u < kChunks) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint32_t t[4][3];
#pragma unroll
                    for (int e = 0; e < 4; ++e) terms_of<kI8>(x[8 * i + 2 * e] * mul, x[8 * i + 2 * e + 1] * mul, t[e]);
#pragma unroll
                    for (uint32_t n = 0; n < kTerms; ++n)
                        *reinterpret_cast<uint4 *>(qs + n * S::kQTermBytes + u * S::kQChunkBytes + r * 128 + ((i ^ (r & 7)) << 4)) =
                            make_uint4(t[0][n], t[1][n], t[2][n], t[3][n]);
                }
            }
            fence_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const uint32_t unit = tmem + kUnitCols * u + (((warp % 4) * 32) << 16);
        // keys of this CTA that this row sees, and its tile's first row
        const int base_key = (int)(block0 * kKeys);
        const int seen = a.causal ? (int)(a.first_row + query) + 1 - base_key : (int)keys;
        const int seen0 = a.causal ? (int)(a.first_row + row0 / group) + 1 - base_key : (int)keys;
        float m = -INFINITY, l = 0.f;
        int e_here = -100;
        float o[D];
#pragma unroll
        for (int i = 0; i < D; ++i) o[i] = 0.f;
        bool ok = true;
        for (uint32_t g = u, it = 0; g < n_blocks; g += 2, ++it) {
            const int key0 = (int)(g * kKeys);
            ok = mbar_wait(s_full + u, it & 1, abort_flag, a.wait_limit);
            // (the scales in the block's stage)
            if (kI8) ok = ok && mbar_wait(full + g % kStages, (g / kStages) & 1, abort_flag, a.wait_limit);
            ok = u ? vote<2, 128>(ok) : vote<1, 128>(ok);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const bool edge = key0 + (int)kKeys > min(seen0, (int)keys);  // some row of the tile does not see the whole block
            const int limit = min(seen, (int)keys) - key0;                // keys of the block that this row sees
            const float *ks = scales + (g % kStages) * S::kScaleFloats, *vs = ks + kKeys;
            float alpha;
            float2 sum = make_float2(0.f, 0.f);
            // (kEdge in the type: a select per score would be paid in every block)
            auto weights = [&](auto edge_tag) {
                constexpr bool kEdge = decltype(edge_tag)::value;
                float top = -INFINITY;
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    uint32_t s[32];
                    tmem_ld32(unit + 32 * part, s);
                    tmem_ld_wait();
                    float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float4 x = make_float4(__uint_as_float(s[e]), __uint_as_float(s[e + 1]), __uint_as_float(s[e + 2]),
                                               __uint_as_float(s[e + 3]));
                        if constexpr (kI8) {
                            const float4 k4 = *reinterpret_cast<const float4 *>(ks + 32 * part + e);
                            const float2 lo = __fmul2_rn(make_float2(x.x, x.y), make_float2(k4.x, k4.y));
                            const float2 hi = __fmul2_rn(make_float2(x.z, x.w), make_float2(k4.z, k4.w));
                            x = make_float4(lo.x, lo.y, hi.x, hi.y);
                        }
                        if constexpr (kEdge) {
                            x.x = 32 * part + e < limit ? x.x : -INFINITY;
                            x.y = 32 * part + e + 1 < limit ? x.y : -INFINITY;
                            x.z = 32 * part + e + 2 < limit ? x.z : -INFINITY;
                            x.w = 32 * part + e + 3 < limit ? x.w : -INFINITY;
                        }
                        t4[0] = fmaxf(t4[0], x.x), t4[1] = fmaxf(t4[1], x.y), t4[2] = fmaxf(t4[2], x.z), t4[3] = fmaxf(t4[3], x.w);
                    }
                    top = fmaxf(top, fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])));
                }
                const float m_new = fmaxf(m, top * f);
                const float base = m_new == -INFINITY ? 0.f : m_new;  // (nothing seen yet: every weight is zero)
                alpha = ex2(m - base);
                m = m_new;
                const float2 f2 = make_float2(f, f), base2 = make_float2(-base, -base);
#pragma unroll
                for (int part = 0; part < 4; ++part) {
                    uint32_t s[16], t[kTerms][8];
                    tmem_ld16(unit + 16 * part, s);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float2 x = make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1]));
                        const int at = 16 * part + 2 * e;
                        if constexpr (kI8) x = __fmul2_rn(x, *reinterpret_cast<const float2 *>(ks + at));
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
                        terms_of<kI8>(x.x, x.y, w);
#pragma unroll
                        for (uint32_t n = 0; n < kTerms; ++n) t[n][e] = w[n];
                    }
#pragma unroll
                    for (uint32_t n = 0; n < kTerms; ++n) tmem_st8(unit + S::weight_col(n) + 8 * part, t[n]);
                }
            };
            if (edge) weights(std::true_type{});
            else weights(std::false_type{});
            l = fmaf(l, alpha, sum.x + sum.y);
            if constexpr (kI8) {
                const int e_new = reinterpret_cast<const int *>(ks)[2 * kKeys];
                alpha *= pow2(max(-126, e_here - e_new));
                e_here = e_new;
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + u);
            // the block's product joins the output (in registers: the sum is rounded, not truncated)
            ok = mbar_wait(o_full + u, it & 1, abort_flag, a.wait_limit);
            ok = u ? vote<2, 128>(ok) : vote<1, 128>(ok);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
            for (int part = 0; part < D / 32; ++part) {
                uint32_t w[32];
                tmem_ld32(unit + kOutCol + 32 * part, w);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 x = __ffma2_rn(make_float2(o[32 * part + i], o[32 * part + i + 1]), make_float2(alpha, alpha),
                                                make_float2(__uint_as_float(w[i]), __uint_as_float(w[i + 1])));
                    o[32 * part + i] = x.x, o[32 * part + i + 1] = x.y;
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        }
        if (!ok) *abort_flag = 1;
        // ---- the units join: each finishes half of the channels and hands the others over, through the ring (every
        // product has been read out, every block consumed once both units are here)
        ok = vote<3, 256>(ok);
        if (ok) {
            constexpr int kHalf = D / 2;
            const float undo = kI8 ? pow2(e_here + 1) * (1.f / kWeightScale) : 1.f;
            float *swap = reinterpret_cast<float *>(ring), *stat = swap + 2 * kHalf * kRows;  // [unit][channel][128], [unit][m, l][128]
            float *mine = swap + u * kHalf * kRows;
#pragma unroll
            for (int i = 0; i < kHalf; ++i) mine[i * kRows + r] = (u ? o[i] : o[kHalf + i]) * undo;
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
            const float *other = swap + (u ^ 1) * kHalf * kRows;
            const size_t at_slot = ((size_t)query * a.n_heads + head) * a.n_slots + a.slot0 + split;
            float *dst = (direct ? a.out + query * a.out_stride + (size_t)head * D : a.scratch + at_slot * D) + u * kHalf;
            if (r < rows) {
                if (!direct && u == 0)
                    *reinterpret_cast<float2 *>(a.scratch + (size_t)a.n_queries * a.n_heads * a.n_slots * D + 2 * at_slot) =
                        make_float2(top, sum);
                const bool wide = ((uintptr_t)dst & 15) == 0;
#pragma unroll
                for (int i = 0; i < kHalf; i += 4) {
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[e] = fmaf(u ? o[kHalf + i + e] : o[i + e], a1, other[(i + e) * kRows + r] * a2);
                    if (wide) {
                        *reinterpret_cast<float4 *>(dst + i) = make_float4(x[0], x[1], x[2], x[3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) dst[i + e] = x[e];
                    }
                }
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
