// Attention of few query rows over INT8 and bfloat16 cache rows (a step of a batch; a prefix for small batches).
//
// Up to eight query rows that read the same kv head go through a span of keys together; four warps of a block
// take 16 keys at a time in turn, each through a ring of its own in shared memory (cp.async), with a running
// maximum and sum per row.  The keys are the M side of the scores' product and the channels that of the output's,
// (query row, term) the N side: a pair of accumulator columns is one row's leading and second term, so a thread
// (g, t) holds the scores of keys g and g + 8 for row t and, later, channels of the same row t; the weights turn
// into the second product's B fragment by one transposition of an 8 x 8 matrix (movmatrix).
//
// Exactness.  INT8: the codes are the A operand of the integer product as they lie; q is 23-bit fixed point in
// three 8-bit digits, so a score is exact but for q's rounding (2^-22 of its largest entry) and one float32
// rounding.  The weights times the value scales are two float16 terms, relative to a power of two at the scales' running
// maximum E (the bound stands at qk::scales_apart); codes as float16 are exact.  A block in whose span the value scales lie
// too far apart for that begins again with three bfloat16 terms, and codes in bfloat16, in true units.  bfloat16: q and the
// weights are three bfloat16 terms.  A step's output product starts from zero and is added to the running sum by float32
// arithmetic: the tensor core truncates.
//
// What bounds it: issue (0.59 of the slots: the codes' conversion to float16, legacy products) and the loads' latency, short
// of the cache's bytes.  INT8, 32 / 8 heads of 128: two sequences of 65536 rows 49.9 us (4.9 TB/s, join included), 64 of 1
// to 2048 rows 44.0 (4.8); the copy rate is 6.6.  Where every block begins again: 64 of 32 to 2048 rows 37 -> 69 us.
#pragma once

#include "qk_cache.h"
#include "qk_mma.cuh"

namespace {

using qk::CacheView;

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kWeightScale = 16384.f;  // weights enter the float16 product times this
constexpr float kLowScale = 2048.f;      // and their second terms times this too

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ int exponent_of(float magnitude) {  // clamped to -100 .. 127
    return min(127, max(-100, (int)(__float_as_uint(magnitude) >> 23) - 127));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {  // an 8 x 8 matrix of 16-bit values
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Products that begin from zero.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_s8_first(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ void copy4(void *smem, const void *gmem, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem),
                 "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16_to(uint32_t smem, const void *gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void copy16_some(uint32_t smem, const void *gmem, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(bytes) : "memory");
}
// {hi, lo 2^11} of a weight as two float16 in one word, hi below: lo loses nothing to float16's smallest numbers.
__device__ __forceinline__ uint32_t weight_terms(float w) {
    uint32_t hi, r;
    float back;
    asm("{\n .reg .b16 h;\n cvt.rn.f16.f32 h, %2;\n cvt.f32.f16 %1, h;\n mov.b32 %0, {h, h};\n}" : "=r"(hi), "=f"(back) : "f"(w));
    asm("{\n .reg .b16 l, h, x;\n mov.b32 {h, x}, %1;\n cvt.rn.f16.f32 l, %2;\n mov.b32 %0, {h, l};\n}"
        : "=r"(r)
        : "r"(hi), "f"((w - back) * kLowScale));
    return r;
}
// Codes of byte `i` of two words (biased by 128) as a pair of float16: 1024 + u is the bit pattern 0x6400 | u.
__device__ __forceinline__ uint32_t code_pair(uint32_t a, uint32_t b, int i) {
    uint32_t w = __byte_perm(a, b, (4 + i) << 4 | i);  // bytes 0 and 1; then 16 bits apart
    w = __byte_perm(w, 0x64646464u, 0x4140);
    uint32_t r;
    asm("{\n .reg .b32 c;\n mov.b32 c, 0x64806480;\n sub.rn.f16x2 %0, %1, c;\n}" : "=r"(r) : "r"(w));
    return r;
}
// The same as a pair of bfloat16, of codes as they are: with the low seven bits u of a code 0x4300 | u is 128 + u, with its
// sign bit 0x4300 | 0x80 is 256 and 0x4300 is 128; the code is the difference.
__device__ __forceinline__ uint32_t code_pair_bf16(uint32_t a, uint32_t b, int i) {
    const uint32_t w = __byte_perm(a, b, (4 + i) << 8 | i);
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"((w & 0x007f007fu) | 0x43004300u), "r"((w & 0x00800080u) | 0x43004300u));
    return r;
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A shared-memory address of this block in the cluster's block `rank`.
__device__ __forceinline__ uint32_t of_block(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float load_shared(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}

// What a block works on: its query rows and its span of keys.
struct Span {
    const void *k, *v;              // the kv head's rows, from row 0
    const float *k_scale, *v_scale;
    int begin, end;                 // rows
    uint32_t first_row, n_rows;     // query rows: row r is query (first_row + r) / group, head (first_row + r) % group of the kv head
    uint32_t slot;                  // where the partial result goes
};

template <bool kI8, int D>
struct AttendShape {
    static constexpr int kRowBytes = kI8 ? D : 2 * D, kPieces = kRowBytes / 16;
    static constexpr int kStageBytes = 2 * 16 * kRowBytes + (kI8 ? 128 : 0);
    static constexpr int kStages = kI8 ? (D == 64 ? 4 : 3) : D == 64 ? 3 : 2;
    static constexpr int kWarpBytes = kStages * kStageBytes;
    static constexpr int kQPitch = kRowBytes + 16;                     // bytes of one term of a query row
    static constexpr int kQBytes = 8 * 3 * kQPitch, kResultBytes = (8 * D + 16) * 4;  // (the block's results follow q's terms)
    static constexpr int kTermBytes = kQBytes > kResultBytes ? kQBytes : kResultBytes;
    static constexpr int kSmem = 4 * kWarpBytes + kTermBytes + 64;
    static_assert(kWarpBytes >= (8 * D + 16) * 4, "a warp's results lie in its ring");
    // (pieces of 16 bytes of a row change places so that fragment loads meet no bank twice)
    __device__ static uint32_t swizzle(uint32_t row, uint32_t piece) {
        return row * kRowBytes + ((piece ^ (kPieces >= 8 ? row & 7 : (row >> 1) & (kPieces - 1))) << 4);
    }
    // The i-th piece of a row that lane t feeds to the scores' product (any order of the channels will do).
    __device__ static uint32_t piece_of(uint32_t t, int i) {
        return kI8 ? (D == 128 ? 2 * t + i : t) : 2 * t + (i % 2) + 8 * (i / 2);
    }
};

// kTiles: column tiles of query rows, four rows each.  kWide: weights as three bfloat16 terms; else as two of float16, unless
// value scales of the block's lie too far apart for them, or a query is too small for its factor: then nothing is written,
// and the answer is false to all threads.
template <bool kI8, int D, int kTiles, bool kWide>
__device__ __forceinline__ bool attend_span(const Span s, const qk::AttendArgs &a, uint32_t kvh, uint32_t n_kv, uint32_t n_slots,
                                            uint32_t n_cluster, uint8_t *smem) {
    using Shape = AttendShape<kI8, D>;
    constexpr int kRowBytes = Shape::kRowBytes, kPieces = Shape::kPieces, kStages = Shape::kStages;
    constexpr int kQTiles = kTiles + 1;                              // column tiles of q: (first, second) term per row, then the thirds
    constexpr int kSteps = D / (kI8 ? 32 : 16);                      // of the scores' contraction
    constexpr int kOut = D / 16;                                     // channel tiles
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
    const uint32_t group = a.n_heads / n_kv;
    uint8_t *ring = smem + warp * Shape::kWarpBytes;
    const uint8_t *kb = static_cast<const uint8_t *>(s.k), *vb = static_cast<const uint8_t *>(s.v);

    // A step's rows lie one behind the other: a lane's pieces are 512 bytes apart, and their places in the stage are
    // two swizzled ones, eight rows apart.
    constexpr int kCopies = 16 * kPieces / 32, kFresh = kPieces / 4;
    uint32_t place[kFresh];
#pragma unroll
    for (int i = 0; i < kFresh; ++i) place[i] = smem_addr(ring) + Shape::swizzle((lane + 32 * i) / kPieces, lane % kPieces);
    const uint8_t *k_lane = kb + lane * 16, *v_lane = vb + lane * 16;
    const float *s_lane = kI8 ? (lane < 16 ? s.k_scale : s.v_scale) + lane % 16 : nullptr;
    auto fetch = [&](int j, int stage) {
        const uint32_t at = stage * Shape::kStageBytes;
        const uint8_t *ks = k_lane + (size_t)j * kRowBytes, *vs = v_lane + (size_t)j * kRowBytes;
        if (j + 16 <= s.end) {
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const uint32_t to = place[i % kFresh] + at + i / kFresh * 8 * kRowBytes;
                copy16_to(to, ks + i * 512);
                copy16_to(to + 16 * kRowBytes, vs + i * 512);
            }
            if (kI8) copy4(ring + at + 2 * 16 * kRowBytes + lane * 4, s_lane + j, 4u);
        } else {  // rows past the end are zeros
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const bool live = j + (int)((lane + 32 * i) / kPieces) < s.end;
                const uint32_t to = place[i % kFresh] + at + i / kFresh * 8 * kRowBytes;
                copy16_some(to, live ? ks + i * 512 : kb, live ? 16u : 0u);
                copy16_some(to + 16 * kRowBytes, live ? vs + i * 512 : vb, live ? 16u : 0u);
            }
            if (kI8) {
                const bool live = j + (int)(lane % 16) < s.end;
                copy4(ring + at + 2 * 16 * kRowBytes + lane * 4, live ? s_lane + j : s.k_scale, live ? 4u : 0u);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    constexpr int kStride = 64;
    const int j_first = s.begin + 16 * (int)warp;
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i)
        if (j_first + i * kStride < s.end) fetch(j_first + i * kStride, i);

    // ---- q's terms, a warp per row: lines of [row][term] in shared memory
    uint8_t *q_lines = smem + 4 * Shape::kWarpBytes;
    // What turns a row's sums into log2 units.  INT8, kWide: divided by a power of two that is given behind the eight factors,
    // for the smallest queries' own is below float32's range.
    float *q_factor = reinterpret_cast<float *>(q_lines + Shape::kTermBytes);
    bool tiny = false;  // INT8: a row has such a query
    const float unit = kLog2E / sqrtf((float)D);
    for (uint32_t r = warp; r < 4 * kTiles; r += 4) {
        constexpr uint32_t kLanes = D / 4;  // lanes with four channels each
        const uint32_t row = s.first_row + min(r, s.n_rows - 1), c = 4 * (lane % kLanes);
        float4 x = *reinterpret_cast<const float4 *>(a.q + (row / group) * a.q_stride +
                                                     (size_t)(kvh * group + row % group) * D + c);
        if (r >= s.n_rows) x = make_float4(0.f, 0.f, 0.f, 0.f);
        uint8_t *line = q_lines + r * 3 * Shape::kQPitch;
        if (kI8) {
            const uint32_t bits = max(max(__float_as_uint(fabsf(x.x)), __float_as_uint(fabsf(x.y))),
                                      max(__float_as_uint(fabsf(x.z)), __float_as_uint(fabsf(x.w))));
            const uint32_t peak = __reduce_max_sync(0xffffffffu, bits);  // (an infinity or NaN is larger than any number)
            const int e = exponent_of(__uint_as_float(peak));
            float mul = pow2(21 - e), more = 1.f;
            if constexpr (kWide) {
                const int down = (int)(peak >> 23) - 127 - e;  // (below zero for those alone)
                more = down < 0 && peak ? pow2(max(-26, down)) : 1.f;
                x.x /= more, x.y /= more, x.z /= more, x.w /= more;
            } else {
                tiny |= peak != 0 && (int)(peak >> 23) - 127 < e;
            }
            const float v4[4] = {x.x, x.y, x.z, x.w};
            uint32_t word[3] = {0, 0, 0};
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                // v = 65536 d2 + 256 d1 + d0, digits in -128 .. 127: the bytes of v + 0x8080, the lower two less 128
                const uint32_t v = (uint32_t)(__float2int_rn(v4[b] * mul) + 0x8080);
                word[0] |= (v >> 16 & 0xff) << (8 * b);
                word[1] |= ((v >> 8 & 0xff) ^ 0x80) << (8 * b);
                word[2] |= ((v & 0xff) ^ 0x80) << (8 * b);
            }
            if (lane < kLanes) {
#pragma unroll
                for (int term = 0; term < 3; ++term) *reinterpret_cast<uint32_t *>(line + term * Shape::kQPitch + c) = word[term];
            }
            if (lane == 0) {
                q_factor[r] = peak < 0x7f800000u ? pow2(e - 21) * unit : __int_as_float(0x7fffffff);
                if constexpr (kWide) q_factor[8 + r] = more;
            }
        } else {
            uint32_t w0[3], w1[3];
            split3(x.x, x.y, w0);
            split3(x.z, x.w, w1);
            if (lane < kLanes) {
#pragma unroll
                for (int term = 0; term < 3; ++term)
                    *reinterpret_cast<uint2 *>(line + term * Shape::kQPitch + 2 * c) = make_uint2(w0[term], w1[term]);
            }
            if (lane == 0) q_factor[r] = unit;
        }
    }
    __syncthreads();
    // ---- as B fragments.  Column g of tile n: tile n < kTiles: row 4 n + g / 2, term g % 2; the last: third terms of
    // rows g / 2 and 4 + g / 2 side by side
    uint32_t qf[kQTiles][kSteps][2];
    float f[kTiles], f_more[kTiles];
#pragma unroll
    for (int n = 0; n < kQTiles; ++n) {
        const uint32_t r = n >= kTiles ? 4 * (g % 2) + g / 2 : 4 * n + g / 2, term = n >= kTiles ? 2 : g % 2;
        const uint8_t *line = q_lines + (r * 3 + term) * Shape::kQPitch;
#pragma unroll
        for (int i = 0; i < kSteps / 2; ++i) {
            uint4 w = *reinterpret_cast<const uint4 *>(line + 16 * Shape::piece_of(t, i));
            if (kTiles == 1 && n == 1 && g % 2) w = make_uint4(0u, 0u, 0u, 0u);
            qf[n][2 * i][0] = w.x, qf[n][2 * i][1] = w.y;
            qf[n][2 * i + 1][0] = w.z, qf[n][2 * i + 1][1] = w.w;
        }
        if (n < kTiles) f[n < kTiles ? n : 0] = q_factor[4 * n + t], f_more[n < kTiles ? n : 0] = kI8 && kWide ? q_factor[8 + 4 * n + t] : 1.f;
    }

    float o[kTiles][kOut][2], m[kTiles], l[kTiles];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        m[n] = -INFINITY, l[n] = 0.f;
#pragma unroll
        for (int i = 0; i < kOut; ++i) o[n][i][0] = o[n][i][1] = 0.f;
    }
    int e_max = -100;              // exponent of the largest value scale so far
    uint32_t least = 0xffffffffu;  // bits, less one, of the smallest that is not zero (of this lane's)

    int stage = 0;
    for (int j = j_first; j < s.end; j += kStride, stage = stage + 1 == kStages ? 0 : stage + 1) {
        if (j + (kStages - 1) * kStride < s.end) {
            fetch(j + (kStages - 1) * kStride, (stage + kStages - 1) % kStages);
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        } else if (kStages > 3 && j + 2 * kStride < s.end) {
            asm volatile("cp.async.wait_group 2;" ::: "memory");
        } else if (j + kStride < s.end) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncwarp();
        const uint8_t *kt = ring + stage * Shape::kStageBytes, *vt = kt + 16 * kRowBytes;

        // ---- scores of keys g and g + 8
        float x[kTiles][2];
        float vs[2];
        if (kI8) {
            int acc[kQTiles][4];
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const uint32_t piece = Shape::piece_of(t, i);
                const uint4 lo = *reinterpret_cast<const uint4 *>(kt + Shape::swizzle(g, piece));
                const uint4 hi = *reinterpret_cast<const uint4 *>(kt + Shape::swizzle(g + 8, piece));
                const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
                for (int n = 0; n < kQTiles; ++n) {
                    if (i == 0) mma_s8_first(acc[n], a0, qf[n][0][0], qf[n][0][1]);
                    else mma_s8(acc[n], a0, qf[n][2 * i][0], qf[n][2 * i][1]);
                    mma_s8(acc[n], a1, qf[n][2 * i + 1][0], qf[n][2 * i + 1][1]);
                }
            }
            const float *sc = reinterpret_cast<const float *>(kt + 2 * 16 * kRowBytes);
            vs[0] = sc[16 + g], vs[1] = sc[24 + g];
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // (thirds: columns 2 t and 2 t + 1 of the last tile are rows t and 4 + t)
                    const int low = acc[n][2 * h + 1] * 256 + acc[kTiles][2 * h + n];
                    x[n][h] = fmaf((float)acc[n][2 * h], 65536.f, (float)low) * (f[n] * sc[8 * h + g]);
                    if constexpr (kWide) x[n][h] *= f_more[n];
                }
        } else {
            float acc[kQTiles][4];
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const uint32_t piece = Shape::piece_of(t, i);
                const uint4 lo = *reinterpret_cast<const uint4 *>(kt + Shape::swizzle(g, piece));
                const uint4 hi = *reinterpret_cast<const uint4 *>(kt + Shape::swizzle(g + 8, piece));
                const uint32_t a0[4] = {lo.x, hi.x, lo.y, hi.y}, a1[4] = {lo.z, hi.z, lo.w, hi.w};
#pragma unroll
                for (int n = 0; n < kQTiles; ++n) {
                    if (i == 0) mma_bf16_first(acc[n], a0, qf[n][0][0], qf[n][0][1]);
                    else mma16(acc[n], a0, qf[n][2 * i][0], qf[n][2 * i][1]);
                    mma16(acc[n], a1, qf[n][2 * i + 1][0], qf[n][2 * i + 1][1]);
                }
            }
            vs[0] = vs[1] = 1.f;
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    x[n][h] = (acc[n][2 * h] + (acc[n][2 * h + 1] + acc[kTiles][2 * h + n])) * f[n];
        }
        if (j + 16 > s.end) {
#pragma unroll
            for (int n = 0; n < kTiles; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (j + (int)g + 8 * h >= s.end) x[n][h] = -INFINITY;
        }
        // ---- the value scales' common power of two
        float shrink = 1.f;
        if constexpr (!kWide) {
            const uint32_t b0 = __float_as_uint(fabsf(vs[0])), b1 = __float_as_uint(fabsf(vs[1]));
            const int e_new = max(e_max, min(125, exponent_of(__uint_as_float(__reduce_max_sync(0xffffffffu, max(b0, b1))))));
            least = min(least, min(b0 - 1u, b1 - 1u));
            shrink = pow2(max(-126, e_max - e_new));
            e_max = e_new;
            const float vmul = pow2(-1 - e_new) * kWeightScale;
            vs[0] *= vmul, vs[1] *= vmul;
        }
        // ---- running maximum and sum, weights as terms
        uint32_t pf[kQTiles][2], last[kTiles];
        float alpha[kTiles];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
            float mx = fmaxf(x[n][0], x[n][1]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float m_new = fmaxf(m[n], mx), base = m_new == -INFINITY ? 0.f : m_new;
            alpha[n] = ex2(m[n] - base);
            m[n] = m_new;
            const float p0 = ex2(x[n][0] - base), p1 = ex2(x[n][1] - base);
            l[n] = fmaf(l[n], alpha[n], p0 + p1);
            alpha[n] *= shrink;
            if constexpr (kWide) {
                uint32_t w[3];
                split3(p0 * vs[0], p1 * vs[1], w);  // (key g below, key g + 8 above)
                pf[n][0] = transposed(__byte_perm(w[0], w[1], 0x5410));
                pf[n][1] = transposed(__byte_perm(w[0], w[1], 0x7632));
                last[n] = w[2];
            } else {
                pf[n][0] = transposed(weight_terms(p0 * vs[0]));
                pf[n][1] = transposed(weight_terms(p1 * vs[1]));
            }
        }
        if constexpr (kWide) {  // thirds of rows t and 4 + t side by side
            const uint32_t w0 = last[0], w1 = kTiles > 1 ? last[kTiles - 1] : 0u;
            pf[kTiles][0] = transposed(__byte_perm(w0, w1, 0x5410));
            pf[kTiles][1] = transposed(__byte_perm(w0, w1, 0x7632));
        }
        // A channel tile's product in three terms joins the output.
        auto add_wide = [&](int i, const uint32_t (&af)[4]) {
            float third[4];
            mma_bf16_first(third, af, pf[kTiles][0], pf[kTiles][1]);
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                float c[4];
                mma_bf16_first(c, af, pf[n][0], pf[n][1]);
                o[n][i][0] = fmaf(o[n][i][0], alpha[n], c[0] + (c[1] + third[n]));
                o[n][i][1] = fmaf(o[n][i][1], alpha[n], c[2] + (c[3] + third[2 + n]));
            }
        };
        // ---- output: channels are the M side
        if (kI8) {
            uint32_t vw[4][D / 32];  // keys 2t, 2t + 1, 2t + 8, 2t + 9: channels (D / 8) g ..
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t key = 2 * t + (r & 1) + 8 * (r >> 1);
                if constexpr (D == 128) {
                    const uint4 v4 = *reinterpret_cast<const uint4 *>(vt + Shape::swizzle(key, g));
                    vw[r][0] = v4.x, vw[r][1] = v4.y, vw[r][2] = v4.z, vw[r][3] = v4.w;
                } else {
                    const uint2 v2 = *reinterpret_cast<const uint2 *>(vt + Shape::swizzle(key, g / 2) + 8 * (g % 2));
                    vw[r][0] = v2.x, vw[r][1] = v2.y;
                }
            }
            if constexpr (!kWide)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) vw[r][i] ^= 0x80808080u;
#pragma unroll
            for (int i = 0; i < kOut; ++i) {  // rows g, g + 8 of tile i: channels (D / 8) g + 2 i, + 1
                const int w = i / 2, b = 2 * (i % 2);
                auto pair = [&](int r, int b) {
                    return kWide ? code_pair_bf16(vw[r][w], vw[r + 1][w], b) : code_pair(vw[r][w], vw[r + 1][w], b);
                };
                const uint32_t af[4] = {pair(0, b), pair(0, b + 1), pair(2, b), pair(2, b + 1)};
                if constexpr (kWide) {
                    add_wide(i, af);
                } else {
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) {
                        float c[4];
                        mma_f16_first(c, af, pf[n][0], pf[n][1]);
                        o[n][i][0] = fmaf(o[n][i][0], alpha[n], fmaf(c[1], 1.f / kLowScale, c[0]));
                        o[n][i][1] = fmaf(o[n][i][1], alpha[n], fmaf(c[3], 1.f / kLowScale, c[2]));
                    }
                }
            }
        } else {
            const uint32_t v_addr = (uint32_t)__cvta_generic_to_shared(vt);
#pragma unroll
            for (int i = 0; i < kOut; ++i) {  // rows g, g + 8 of tile i: channels 16 i + g, 16 i + 8 + g
                uint32_t af[4];
                const uint32_t key = (lane & 7) + 8 * (lane >> 4), piece = 2 * i + ((lane >> 3) & 1);
                ldsm4_trans(af, v_addr + Shape::swizzle(key, piece));
                add_wide(i, af);
            }
        }
        __syncwarp();  // the stage may be filled again
    }

    // ---- the block's warps join: [row][D] outputs, then maxima and sums, each in its warp's ring
    const float undo = kWide ? 1.f : pow2(e_max + 1) * (1.f / kWeightScale);
    float *mine = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 4);
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 8);
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 16);
        const uint32_t r = 4 * n + t;
        if (g == 0) mine[8 * D + r] = m[n], mine[8 * D + 8 + r] = l[n];
#pragma unroll
        for (int i = 0; i < kOut; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                mine[r * D + (kI8 ? (D / 8) * g + 2 * i + h : 16 * i + 8 * h + g)] = o[n][i][h] * undo;
    }
    if constexpr (kWide) {
        __syncthreads();
    } else if (__syncthreads_or(tiny || qk::scales_apart(e_max, __reduce_min_sync(0xffffffffu, least)))) {
        return false;
    }
    const bool alone = n_cluster == 1;
    float *result = reinterpret_cast<float *>(q_lines);  // [8][D] outputs, [8] maxima, [8] sums: for the cluster's blocks
    auto put = [&](uint32_t r, uint32_t c, float top, float sum, float val) {
        const uint32_t row = s.first_row + r, query = row / group, head = kvh * group + row % group;
        if (n_slots == 1) {
            a.out[query * a.out_stride + (size_t)head * D + c] = sum == 0.f ? 0.f : val / sum;
        } else {
            const size_t at_slot = ((size_t)query * a.n_heads + head) * n_slots + s.slot;
            a.scratch[at_slot * D + c] = val;
            if (c == 0)
                *reinterpret_cast<float2 *>(a.scratch + (size_t)a.n_queries * a.n_heads * n_slots * D + 2 * at_slot) =
                    make_float2(top, sum);
        }
    };
    // (a warp without keys has the sum 0; a NaN stays)
    auto share_of = [](float m, float l, float top) { return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2(m - top); };
    for (uint32_t at = threadIdx.x; at < s.n_rows * D; at += 128) {
        const uint32_t r = at / D, c = at % D;
        float mw[4], top = -INFINITY, sum = 0.f, val = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            mw[w] = reinterpret_cast<const float *>(smem + w * Shape::kWarpBytes)[8 * D + r];
            top = fmaxf(top, mw[w]);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float *src = reinterpret_cast<const float *>(smem + w * Shape::kWarpBytes);
            const float weight = share_of(mw[w], src[8 * D + 8 + r], top);
            sum = fmaf(src[8 * D + 8 + r], weight, sum);
            val = fmaf(src[r * D + c], weight, val);
        }
        if (alone) {
            put(r, c, top, sum, val);
        } else {
            result[r * D + c] = val;
            if (c == 0) result[8 * D + r] = top, result[8 * D + 8 + r] = sum;
        }
    }
    if (alone) return true;
    // ---- the splits of a cluster join through distributed shared memory, every block a part of the outputs
    cluster_sync();
    uint32_t rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const uint32_t here = smem_addr(result);
    for (uint32_t at = rank * 128 + threadIdx.x; at < s.n_rows * D; at += n_cluster * 128) {
        const uint32_t r = at / D, c = at % D;
        float m[8], l[8], v[8], top = -INFINITY, sum = 0.f, val = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            if (i >= n_cluster) break;
            const uint32_t there = of_block(here, i);
            v[i] = load_shared(there + (r * D + c) * 4);
            m[i] = load_shared(there + (8 * D + r) * 4);
            l[i] = load_shared(there + (8 * D + 8 + r) * 4);
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            if (i >= n_cluster) break;
            top = fmaxf(top, m[i]);
        }
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            if (i >= n_cluster) break;
            const float weight = share_of(m[i], l[i], top);
            sum = fmaf(l[i], weight, sum);
            val = fmaf(v[i], weight, val);
        }
        put(r, c, top, sum, val);
    }
    cluster_sync();  // (no block ends while another reads its results)
    return true;
}

}  // namespace
