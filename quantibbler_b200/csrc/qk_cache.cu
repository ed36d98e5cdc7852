// Key/value caches in float32, bfloat16 and INT8: appending with rotation and quantisation, reading back, the
// attention of a step and of a prompt's portion, both with rows in front that all sequences share.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <initializer_list>
#include <type_traits>

#include "qk_cache.h"
#include "qk_cache_attend.cuh"

namespace {

// ------------------------------------------------------------------ append
// Whether a later token of the call names the same row, as far as this thread looks: the block's threads share the
// tokens, four at a time where the lists lie on 16 bytes.
__device__ __forceinline__ bool named_again(const int32_t *__restrict__ positions, const int32_t *__restrict__ seq_index,
                                            uint32_t tok, int pos, int seq, uint32_t n_tokens) {
    bool later = false;
    if ((((uintptr_t)positions | (uintptr_t)seq_index) & 15) == 0) {
        const uint32_t whole = n_tokens / 4;
        const int4 *p4 = reinterpret_cast<const int4 *>(positions), *s4 = reinterpret_cast<const int4 *>(seq_index);
#pragma unroll 2
        for (uint32_t i = (tok + 1) / 4 + threadIdx.x; i < whole; i += blockDim.x) {
            const int4 p = p4[i], s = s4[i];
            const uint32_t t = 4 * i;
            later |= (p.x == pos && s.x == seq && t > tok) | (p.y == pos && s.y == seq && t + 1 > tok) |
                     (p.z == pos && s.z == seq && t + 2 > tok) | (p.w == pos && s.w == seq && t + 3 > tok);
        }
        const uint32_t i = 4 * whole + threadIdx.x;
        if (i < n_tokens) later |= positions[i] == pos && seq_index[i] == seq && i > tok;
    } else {
        for (uint32_t i = tok + 1 + threadIdx.x; i < n_tokens; i += blockDim.x) later |= positions[i] == pos && seq_index[i] == seq;
    }
    return later;
}

// The largest of the lanes' non-negative numbers (their bits are in their order).
__device__ __forceinline__ double warp_peak(double x) {
    const uint32_t hi = (uint32_t)__double2hiint(x), top = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t lo = __reduce_max_sync(0xffffffffu, hi == top ? (uint32_t)__double2loint(x) : 0u);
    return __hiloint2double((int)top, (int)lo);
}

// Four codes, clipped to -127 .. 127.
__device__ __forceinline__ uint32_t pack_codes(const int (&n)[4]) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) w |= (uint32_t)(min(127, max(-127, n[e])) & 0xff) << (8 * e);
    return w;
}

// n consecutive values.
template <int kN, typename T>
__device__ __forceinline__ void load_n(const T *p, T (&v)[kN]) {
    using V = std::conditional_t<kN * sizeof(T) == 16, uint4, std::conditional_t<kN * sizeof(T) == 8, uint2, uint32_t>>;
    *reinterpret_cast<V *>(v) = *reinterpret_cast<const V *>(p);
}

// Any even head size, addresses of any alignment: a warp per row (a head of q, k or v), a lane has the pairs (i, i + d/2),
// i = lane, lane + 32, ..
template <typename KV>  // float, uint16_t (bfloat16), int8_t
__global__ void __launch_bounds__(256)
append_kernel(CacheView c, const float *q, size_t q_stride, float *q_out, size_t q_out_stride, uint32_t n_heads,
              const float *__restrict__ k, size_t k_stride, const float *__restrict__ v, size_t v_stride,
              const float *__restrict__ cos_sin, uint32_t n_positions, const int32_t *__restrict__ positions,
              const int32_t *__restrict__ seq_index, uint32_t first_position, uint32_t n_tokens, int *__restrict__ error) {
    qk::pdl_launch();
    qk::pdl_wait();
    constexpr int kMine = 4;  // (head_dim <= 256)
    const uint32_t tok = blockIdx.x, d = c.d, half = d / 2, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t pos = positions[tok], seq = seq_index[tok], row = pos - (int64_t)first_position;
    if (row < 0 || row >= (int64_t)c.rows || pos >= (int64_t)n_positions || seq < 0 || seq >= (int64_t)c.n_seq) {
        if (threadIdx.x == 0) atomicOr(error, 4);
        return;
    }
    const float *cs = cos_sin + (size_t)pos * d;
    if (q)
        for (uint32_t h = warp; h < n_heads; h += 8) {
            const float *src = q + tok * q_stride + (size_t)h * d;
            float *dst = q_out + tok * q_out_stride + (size_t)h * d;
            for (uint32_t i = lane; i < half; i += 32) {
                const float a = src[i], b = src[half + i], co = cs[2 * i], si = cs[2 * i + 1];
                dst[i] = rope_first(a, b, co, si);
                dst[half + i] = rope_second(a, b, co, si);
            }
        }
    if (__syncthreads_or(named_again(positions, seq_index, tok, (int)pos, (int)seq, n_tokens))) return;  // (that one stays)
    for (uint32_t r = warp; r < 2 * c.n_kv; r += 8) {
        const bool is_k = r < c.n_kv;
        const uint32_t h = is_k ? r : r - c.n_kv;
        const float *src = (is_k ? k + tok * k_stride : v + tok * v_stride) + (size_t)h * d;
        const size_t line = ((size_t)seq * c.n_kv + h) * c.rows + (size_t)row;
        KV *dst = static_cast<KV *>(is_k ? c.k : c.v) + line * d;
        if constexpr (sizeof(KV) != 1) {
            for (uint32_t i = lane; i < half; i += 32) {
                const float a = src[i], b = src[half + i], co = cs[2 * i], si = cs[2 * i + 1];
                store_from_float<KV>(dst, i, is_k ? rope_first(a, b, co, si) : a);
                store_from_float<KV>(dst, half + i, is_k ? rope_second(a, b, co, si) : b);
            }
        } else {
            double x[2][kMine], peak = 0.0;  // in 64 bits, where products of two float32 are exact
            bool finite = true;
#pragma unroll
            for (int e = 0; e < kMine; ++e) {
                const uint32_t i = lane + 32 * e;
                x[0][e] = x[1][e] = 0.0;
                if (i >= half) continue;
                const double a = src[i], b = src[half + i], co = is_k ? cs[2 * i] : 1.0, si = is_k ? cs[2 * i + 1] : 0.0;
                x[0][e] = is_k ? fma(a, co, -(b * si)) : a;
                x[1][e] = is_k ? fma(b, co, a * si) : b;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    finite = finite && fabs(x[w][e]) <= (double)FLT_MAX;
                    peak = fmax(peak, fabs(x[w][e]));
                }
            }
            finite = __all_sync(0xffffffffu, finite);
            float scale = (float)(warp_peak(peak) / 127.0);
            if (scale == 0.f) scale = 1.f;
#pragma unroll
            for (int e = 0; e < kMine; ++e) {
                const uint32_t i = lane + 32 * e;
                if (i >= half) continue;
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    dst[w * half + i] =
                        (int8_t)(finite ? min(127, max(-127, __double2int_rn(x[w][e] / (double)scale))) : 0);
            }
            if (lane == 0) (is_k ? c.k_scale : c.v_scale)[line] = finite ? scale : __int_as_float(0x7fffffff);
        }
    }
}

// Head sizes 64 kGroups on 16-byte boundaries: eight lanes to a row, four rows to a warp at once (what a row
// costs beside its entries - the reductions, the division that gives the scale - is paid once for four), kGroups vectors
// of four pairs a lane.  2048 tokens, 32 / 8 heads of 128: 20 us, 4.4 TB/s (issue and the latency of one round of loads a
// block; 26 us with a row to a warp, most of it issue).
template <typename KV, int kGroups>
__global__ void __launch_bounds__(128, kGroups == 4 ? 4 : 8)
append_wide_kernel(CacheView c, const float *q, size_t q_stride, float *q_out, size_t q_out_stride, uint32_t n_heads,
                   const float *__restrict__ k, size_t k_stride, const float *__restrict__ v, size_t v_stride,
                   const float *__restrict__ cos_sin, uint32_t n_positions, const int32_t *__restrict__ positions,
                   const int32_t *__restrict__ seq_index, uint32_t first_position, uint32_t n_tokens, uint32_t kv_blocks,
                   int *__restrict__ error) {
    qk::pdl_launch();
    qk::pdl_wait();
    constexpr uint32_t d = 64 * kGroups, half = d / 2;
    constexpr int kMine = 4 * kGroups;  // pairs of a lane: 32 g + 4 (lane % 8) ..
    const uint32_t tok = blockIdx.x, lane = threadIdx.x % 32, i0 = 4 * (lane % 8);
    const bool is_q = blockIdx.y >= kv_blocks;
    const uint32_t r = (is_q ? blockIdx.y - kv_blocks : blockIdx.y) * 16 + threadIdx.x / 8;
    const bool is_k = r < c.n_kv, live = r < (is_q ? n_heads : 2 * c.n_kv);
    const uint32_t h = is_q || is_k ? r : r - c.n_kv;
    const int64_t pos = positions[tok], seq = seq_index[tok], row = pos - (int64_t)first_position;
    const float *src = (is_q ? q + tok * q_stride : is_k ? k + tok * k_stride : v + tok * v_stride) + h * d + i0;
    float a[kMine], b[kMine];
    if (live) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            *reinterpret_cast<float4 *>(a + 4 * g) = *reinterpret_cast<const float4 *>(src + 32 * g);
            *reinterpret_cast<float4 *>(b + 4 * g) = *reinterpret_cast<const float4 *>(src + half + 32 * g);
        }
    }
    if (row < 0 || row >= (int64_t)c.rows || pos >= (int64_t)n_positions || seq < 0 || seq >= (int64_t)c.n_seq) {
        if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(error, 4);
        return;
    }
    // (a later token of the call with the same row stays; its list is read while the row's entries are on their way)
    const bool later = !is_q && named_again(positions, seq_index, tok, (int)pos, (int)seq, n_tokens);
    const bool turned = is_q || is_k;
    float co[kMine], si[kMine];
    if (live && turned) {
        const float *cs = cos_sin + (size_t)pos * d + 2 * i0;
#pragma unroll
        for (int e = 0; e < kMine; e += 2) {
            const float4 t = *reinterpret_cast<const float4 *>(cs + e / 4 * 64 + e % 4 * 2);
            co[e] = t.x, si[e] = t.y, co[e + 1] = t.z, si[e + 1] = t.w;
        }
    }
    float p[2][kMine];
#pragma unroll
    for (int e = 0; e < kMine; ++e) {
        p[0][e] = !live ? 0.f : turned ? rope_first(a[e], b[e], co[e], si[e]) : a[e];
        p[1][e] = !live ? 0.f : turned ? rope_second(a[e], b[e], co[e], si[e]) : b[e];
    }
    if (is_q) {
        float *dst = q_out + tok * q_out_stride + h * d + i0;
        if (live)
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                *reinterpret_cast<float4 *>(dst + 32 * g) = *reinterpret_cast<const float4 *>(p[0] + 4 * g);
                *reinterpret_cast<float4 *>(dst + half + 32 * g) = *reinterpret_cast<const float4 *>(p[1] + 4 * g);
            }
        return;
    }
    if (__syncthreads_or(later)) return;
    const size_t line = ((size_t)seq * c.n_kv + h) * c.rows + (size_t)row;
    KV *dst = static_cast<KV *>(is_k ? c.k : c.v) + line * d + i0;
    if constexpr (sizeof(KV) == 4) {
        if (live)
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                *reinterpret_cast<float4 *>(dst + 32 * g) = *reinterpret_cast<const float4 *>(p[0] + 4 * g);
                *reinterpret_cast<float4 *>(dst + half + 32 * g) = *reinterpret_cast<const float4 *>(p[1] + 4 * g);
            }
    } else if constexpr (sizeof(KV) == 2) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                uint16_t x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = float_to_bf16_bits(p[w][4 * g + e]);
                if (live)
                    *reinterpret_cast<uint2 *>(dst + w * half + 32 * g) =
                        make_uint2((uint32_t)x[1] << 16 | x[0], (uint32_t)x[3] << 16 | x[2]);
            }
    } else {
        // The codes are those of 64-bit arithmetic (products of two float32 are exact there).  float32 gives an entry to
        // 2^-22 of the row's largest, 3e-5 of a code's width: the largest entry, and entries as near as 1e-3 to the border
        // between two codes, are formed again in 64 bits.
        auto exactly = [&](int e, int w) {
            // (seldom: read again, not kept)
            const uint32_t at = e / 4 * 32 + e % 4;
            if (!is_k) return (double)src[w * half + at];
            const float2 turn = *reinterpret_cast<const float2 *>(cos_sin + (size_t)pos * d + 2 * (i0 + at));
            const double x = src[at], y = src[half + at], co64 = turn.x, si64 = turn.y;
            return w ? fma(y, co64, x * si64) : fma(x, co64, -(y * si64));
        };
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < kMine; ++e)
            mine = max(mine, max(__float_as_uint(fabsf(p[0][e])), __float_as_uint(fabsf(p[1][e]))));
        uint32_t top = mine;
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
        const bool finite = top < 0x7f800000u;  // (an infinity or NaN is larger than any number)
        const float near_top = __uint_as_float(top) * (1.f - 0x1p-20f);
        double peak = (double)__uint_as_float(mine);
        if (is_k) {
            peak = 0.0;  // (unless another lane has the largest)
            if (live && __uint_as_float(mine) >= near_top) {
                int which = 0, several = 0;  // entries that may be the largest: nearly always one
#pragma unroll
                for (int e = 0; e < 2 * kMine; ++e)
                    if (fabsf(p[e / kMine][e % kMine]) >= near_top) which = e, ++several;
                if (several == 1)
                    peak = fabs(exactly(which % kMine, which / kMine));
                else
                    for (int e = 0; e < 2 * kMine; ++e) peak = fmax(peak, fabs(exactly(e % kMine, e / kMine)));
            }
        }
#pragma unroll
        for (int off = 4; off > 0; off >>= 1) peak = fmax(peak, __shfl_xor_sync(0xffffffffu, peak, off));
        float scale = (float)(peak / 127.0);
        if (scale == 0.f) scale = 1.f;
        const float inv = 1.f / scale;
        uint32_t codes[2][kGroups];
        float off_code = 0.f;
#pragma unroll
        for (int w = 0; w < 2; ++w)
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                uint32_t n[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // (1.5 2^23 more: the nearest integer, ties to even, in the low bits)
                    const float x = p[w][4 * g + e] * inv, more = x + 12582912.f;
                    off_code = fmaxf(off_code, fabsf(x - (more - 12582912.f)));
                    n[e] = __float_as_uint(more);
                }
                codes[w][g] = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
            }
        // (the smallest scales, whose reciprocal may be infinite and who may round by much, too)
        if (live && finite && (off_code > 0.499f || !(inv < 0x1p120f))) {
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    int n[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) n[e] = __double2int_rn(exactly(4 * g + e, w) / (double)scale);
                    codes[w][g] = pack_codes(n);
                }
        }
        if (!live) return;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            *reinterpret_cast<uint32_t *>(dst + 32 * g) = finite ? codes[0][g] : 0u;
            *reinterpret_cast<uint32_t *>(dst + half + 32 * g) = finite ? codes[1][g] : 0u;
        }
        if (lane % 8 == 0) (is_k ? c.k_scale : c.v_scale)[line] = finite ? scale : __int_as_float(0x7fffffff);
    }
}

// ------------------------------------------------------------------ reading back
template <typename KV> __device__ __forceinline__ float value_at(const KV *p, size_t i, float) {
    return load_as_float<KV>(p, i);
}
template <> __device__ __forceinline__ float value_at<int8_t>(const int8_t *p, size_t i, float scale) {
    return (float)p[i] * scale;
}

// A warp per row.  kVec: head sizes of whole groups of four values per lane, on 16-byte boundaries.  2048 INT8 tokens of 8
// heads of 128 as float32: 6.6 us, 3.2 TB/s (one round of loads a warp).
template <typename KV, typename Out, bool kVec>
__global__ void __launch_bounds__(256)
read_kernel(CacheView c, const int32_t *__restrict__ positions, const int32_t *__restrict__ seq_index, uint32_t first_position,
            uint32_t n_tokens, Out *__restrict__ k_out, Out *__restrict__ v_out, int *__restrict__ error) {
    qk::pdl_launch();
    qk::pdl_wait();
    const uint32_t lane = threadIdx.x % 32;
    const size_t r = (size_t)blockIdx.x * 8 + threadIdx.x / 32;  // (token, k or v, kv head)
    if (r >= (size_t)n_tokens * c.n_kv * 2) return;
    const uint32_t h = (uint32_t)(r % c.n_kv), tok = (uint32_t)(r / c.n_kv / 2);
    const bool is_v = r / c.n_kv % 2;
    const int64_t row = (int64_t)positions[tok] - (int64_t)first_position, seq = seq_index[tok];
    const bool there = row >= 0 && row < (int64_t)c.rows && seq >= 0 && seq < (int64_t)c.n_seq;
    if (!there && lane == 0) atomicOr(error, 4);
    const size_t line = there ? ((size_t)seq * c.n_kv + h) * c.rows + (size_t)row : 0;
    const KV *src = static_cast<const KV *>(is_v ? c.v : c.k) + line * c.d;
    const float scale = sizeof(KV) == 1 && there ? (is_v ? c.v_scale : c.k_scale)[line] : 1.f;
    Out *dst = (is_v ? v_out : k_out) + ((size_t)tok * c.n_kv + h) * c.d;
    if constexpr (kVec) {
        for (uint32_t i = 4 * lane; i < c.d; i += 128) {
            alignas(16) KV x[4];
            alignas(16) Out y[4];
            if (there) load_n<4>(src + i, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) store_from_float<Out>(y, e, there ? value_at<KV>(x, e, scale) : 0.f);
            if constexpr (sizeof(Out) == 4) *reinterpret_cast<uint4 *>(dst + i) = *reinterpret_cast<const uint4 *>(y);
            else *reinterpret_cast<uint2 *>(dst + i) = *reinterpret_cast<const uint2 *>(y);
        }
    } else {
        for (uint32_t i = lane; i < c.d; i += 32) store_from_float<Out>(dst, i, there ? value_at<KV>(src, i, scale) : 0.f);
    }
}

// ------------------------------------------------------------------ attention, plain form
// Any dtype and head size: a warp per (query row, head), the lanes share the channels, one pass with the running
// maximum and sum.  What the fast kernels cannot hold runs here, bound by the chain of a key: loads, the lanes' sum, two
// exponentials; keys are not split and rows not shared.  32 / 8 heads, float32 rows of 128: one sequence of 2048 rows
// 2180 us, 64 of 1 to 2048 4930, a portion of 2048 tokens 14800, 64 behind 8192 shared rows 12000.
template <typename KV>
__global__ void __launch_bounds__(128)
attend_plain_kernel(CacheView c, CacheView p, qk::AttendArgs a) {
    qk::pdl_launch();
    qk::pdl_wait();
    const size_t row = (size_t)blockIdx.x * 4 + threadIdx.x / 32;
    const uint32_t lane = threadIdx.x % 32, d = c.d;
    if (row >= (size_t)a.n_queries * a.n_heads) return;
    const uint32_t t = (uint32_t)(row / a.n_heads), head = (uint32_t)(row % a.n_heads), kvh = head / (a.n_heads / c.n_kv);
    const float *qr = a.q + t * a.q_stride + (size_t)head * d;
    const float scale = 1.0f / sqrtf((float)d);
    float qv[8], o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t i = lane + 32 * e;
        qv[e] = i < d ? qr[i] * scale : 0.f;
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    auto span = [&](const CacheView &s, size_t slot, uint32_t n) {
        const size_t line0 = (slot * s.n_kv + kvh) * s.rows;
        const KV *kb = static_cast<const KV *>(s.k) + line0 * d, *vb = static_cast<const KV *>(s.v) + line0 * d;
        for (uint32_t j = 0; j < n; ++j) {
            const float ks = sizeof(KV) == 1 ? s.k_scale[line0 + j] : 1.f, vs = sizeof(KV) == 1 ? s.v_scale[line0 + j] : 1.f;
            float dot = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t i = lane + 32 * e;
                if (i < d) dot = fmaf(qv[e], value_at<KV>(kb, (size_t)j * d + i, ks), dot);
            }
            for (int off = 16; off > 0; off >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, off);
            const float x = dot, m_new = fmaxf(m, x), alpha = m_new == -INFINITY ? 1.f : expf(m - m_new);
            const float w = x == -INFINITY ? 0.f : expf(x - m_new);
            l = l * alpha + w;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t i = lane + 32 * e;
                if (i < d) o[e] = o[e] * alpha + w * vs * value_at<KV>(vb, (size_t)j * d + i, 1.f);
            }
            m = m_new;
        }
    };
    if (a.prefix_len) span(p, a.prefix_seq, a.prefix_len);
    if (a.kv_len) span(c, t, (uint32_t)min(max(a.kv_len[t], 0), (int)c.rows));
    else span(c, a.seq, a.first_row + t + 1);
    float *dst = a.out + t * a.out_stride + (size_t)head * d;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t i = lane + 32 * e;
        if (i < d) dst[i] = l == 0.f ? 0.f : o[e] / l;
    }
}

// ------------------------------------------------------------------ attention of few query rows
// How a call is dealt out: blocks over the prefix first (all queries of a kv head in rows of eight, splits of the
// prefix), then blocks over the sequences' own rows.  A split of a sequence's rows is the same part of every
// sequence, so that unequal lengths keep all blocks at work.  The blocks of a cluster are neighbouring splits, whose
// results they join themselves.
struct Plan {
    uint32_t prefix_subs, prefix_splits, prefix_chunk, prefix_blocks;
    uint32_t own_subs, own_splits, own_rows;  // own_rows: query rows of a block
    uint32_t cluster;                         // blocks of a cluster; the splits are whole numbers of clusters
    uint32_t prefix_slots, n_slots;           // partial results per (query, head); n_slots 1: none, the output is written
};

// A block's work; its answer is attend_span's.  kMost: column tiles of four query rows that a block needs at most.
template <bool kI8, int D, int kMost, bool kWide>
__device__ __forceinline__ bool attend_block(const CacheView &c, const CacheView &p, const qk::AttendArgs &a, const Plan &pl,
                                             uint8_t *smem) {
    const uint32_t group = a.n_heads / c.n_kv, row_bytes = kI8 ? D : 2 * D;
    Span s;
    uint32_t id = blockIdx.x, kvh;
    const CacheView *src;
    size_t line;
    const uint32_t rank = id % pl.cluster;
    if (id < pl.prefix_blocks) {
        src = &p;
        id /= pl.cluster;
        const uint32_t sub = id % pl.prefix_subs, part = id / pl.prefix_subs % pl.prefix_slots;
        const uint32_t split = part * pl.cluster + rank;
        kvh = id / pl.prefix_subs / pl.prefix_slots;
        line = (a.prefix_seq * p.n_kv + kvh) * p.rows;
        s.begin = (int)min(a.prefix_len, split * pl.prefix_chunk);
        s.end = (int)min(a.prefix_len, (split + 1) * pl.prefix_chunk);
        s.first_row = sub * 8;
        s.n_rows = min(8u, a.n_queries * group - s.first_row);
        s.slot = part;
    } else {
        id = (id - pl.prefix_blocks) / pl.cluster;
        src = &c;
        const uint32_t sub = id % pl.own_subs, parts = pl.own_splits / pl.cluster;
        kvh = id / pl.own_subs % c.n_kv;
        const uint32_t part = id / pl.own_subs / c.n_kv % parts, b = id / pl.own_subs / c.n_kv / parts;
        const uint32_t split = part * pl.cluster + rank;
        line = ((a.kv_len ? b : a.seq) * c.n_kv + kvh) * c.rows;
        // (without lengths: the one query of a portion of one token)
        const uint32_t len = a.kv_len ? (uint32_t)min(max(a.kv_len[b], 0), (int)c.rows) : a.first_row + 1;
        const uint32_t chunk = ((len + pl.own_splits - 1) / pl.own_splits + 63) / 64 * 64;
        s.begin = (int)min(len, split * chunk);
        s.end = (int)min(len, (split + 1) * chunk);
        s.first_row = b * group + sub * pl.own_rows;
        s.n_rows = min(pl.own_rows, group - sub * pl.own_rows);
        s.slot = pl.prefix_slots + part;
    }
    s.k = static_cast<const uint8_t *>(src->k) + line * row_bytes;
    s.v = static_cast<const uint8_t *>(src->v) + line * row_bytes;
    s.k_scale = kI8 ? src->k_scale + line : nullptr;
    s.v_scale = kI8 ? src->v_scale + line : nullptr;
    if constexpr (kMost > 1) {
        if (s.n_rows > 4) return attend_span<kI8, D, 2, kWide>(s, a, kvh, c.n_kv, pl.n_slots, pl.cluster, smem);
    }
    return attend_span<kI8, D, 1, kWide>(s, a, kvh, c.n_kv, pl.n_slots, pl.cluster, smem);
}
template <int D, int kMost>
__device__ __noinline__ void attend_block_wide(const CacheView &c, const CacheView &p, const qk::AttendArgs &a, const Plan &pl,
                                               uint8_t *smem) {
    attend_block<true, D, kMost, true>(c, p, a, pl, smem);
}

template <bool kI8, int D, int kMost>
__global__ void __launch_bounds__(128, kI8 ? (kMost == 1 ? 4 : 3) : (kMost == 1 ? 3 : 2))
attend_rows_kernel(const __grid_constant__ CacheView c, const __grid_constant__ CacheView p,
                   const __grid_constant__ qk::AttendArgs a, const __grid_constant__ Plan pl) {
    qk::pdl_launch();
    qk::pdl_wait();
    extern __shared__ __align__(16) uint8_t attend_smem[];
    if constexpr (kI8) {
        // Value scales that lie too far apart are seldom, and told at the end: the block then begins again.  (With the other
        // form in the loop a look at every step costs a tenth of the time; inlined here, the registers that it takes do.)
        if (!attend_block<true, D, kMost, false>(c, p, a, pl, attend_smem)) attend_block_wide<D, kMost>(c, p, a, pl, attend_smem);
    } else {
        attend_block<false, D, kMost, true>(c, p, a, pl, attend_smem);
    }
}

// Partial results of a (query, head) joined: outputs [slot][D], then {maximum (log2 units), sum} [slot] of all rows.
// A block of four warps each; D / 4 lanes take a slot's output, four channels a lane.
constexpr uint32_t kMaxSlots = 256;

template <int D>
__global__ void __launch_bounds__(128)
join_kernel(qk::AttendArgs a, uint32_t n_slots) {
    qk::pdl_launch();
    qk::pdl_wait();
    __shared__ float weight[kMaxSlots], red[8];
    __shared__ __align__(16) float part[128 / (D / 4)][D];
    constexpr uint32_t kLanes = D / 4, kSide = 128 / kLanes;  // slots side by side
    const uint32_t query = blockIdx.x / a.n_heads, head = blockIdx.x % a.n_heads, warp = threadIdx.x / 32;
    const float *outs = a.scratch + (size_t)blockIdx.x * n_slots * D;
    const float2 *stats = reinterpret_cast<const float2 *>(a.scratch + (size_t)a.n_queries * a.n_heads * n_slots * D) +
                          (size_t)blockIdx.x * n_slots;
    float m[kMaxSlots / 128], l[kMaxSlots / 128], top = -INFINITY;
#pragma unroll
    for (uint32_t i = 0; i < kMaxSlots / 128; ++i) {
        const uint32_t s = threadIdx.x + 128 * i;
        const float2 st = s < n_slots ? stats[s] : make_float2(-INFINITY, 0.f);
        m[i] = st.x, l[i] = st.y;
        top = fmaxf(top, m[i]);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    if (threadIdx.x % 32 == 0) red[warp] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float sum = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < kMaxSlots / 128; ++i) {
        const uint32_t s = threadIdx.x + 128 * i;
        // (a span without keys has the sum 0; a NaN stays)
        const float w = m[i] == -INFINITY ? (l[i] == 0.f ? 0.f : 1.f) : ex2(m[i] - top);
        if (s < n_slots) weight[s] = w;
        sum = fmaf(l[i], w, sum);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (threadIdx.x % 32 == 0) red[4 + warp] = sum;
    __syncthreads();
    sum = (red[4] + red[5]) + (red[6] + red[7]);
    const uint32_t side = threadIdx.x / kLanes, c = 4 * (threadIdx.x % kLanes);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (uint32_t s = side; s < n_slots; s += kSide) {
        const float4 x = *reinterpret_cast<const float4 *>(outs + (size_t)s * D + c);
        const float w = weight[s];
        v.x = fmaf(x.x, w, v.x), v.y = fmaf(x.y, w, v.y), v.z = fmaf(x.z, w, v.z), v.w = fmaf(x.w, w, v.w);
    }
    *reinterpret_cast<float4 *>(&part[side][c]) = v;
    __syncthreads();
    if (threadIdx.x < D) {
        float x = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < kSide; ++i) x += part[i][threadIdx.x];
        a.out[query * a.out_stride + (size_t)head * D + threadIdx.x] = sum == 0.f ? 0.f : x / sum;
    }
}

// The same for up to 32 slots: a warp each, no barriers; the first outputs are on their way with the maxima and sums.
template <int D>
__global__ void __launch_bounds__(128)
join_few_kernel(qk::AttendArgs a, uint32_t n_slots) {
    qk::pdl_launch();
    qk::pdl_wait();
    using V = std::conditional_t<D == 128, float4, float2>;
    constexpr uint32_t kMine = D / 32, kAhead = 4;
    const uint32_t row = blockIdx.x * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
    if (row >= a.n_queries * a.n_heads) return;
    const V *outs = reinterpret_cast<const V *>(a.scratch + (size_t)row * n_slots * D) + lane;
    const float2 *stats = reinterpret_cast<const float2 *>(a.scratch + (size_t)a.n_queries * a.n_heads * n_slots * D) +
                          (size_t)row * n_slots;
    V x[kAhead];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) x[i] = outs[(size_t)min(i, n_slots - 1) * 32];
    const float2 st = lane < n_slots ? stats[lane] : make_float2(-INFINITY, 0.f);
    float top = st.x;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    // (a span without keys has the sum 0; a NaN stays)
    const float w = st.x == -INFINITY ? (st.y == 0.f ? 0.f : 1.f) : ex2(st.x - top);
    float sum = st.y * w, v[kMine] = {};
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    for (uint32_t s0 = 0; s0 < n_slots; s0 += kAhead) {
        V y[kAhead];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) y[i] = outs[(size_t)min(s0 + kAhead + i, n_slots - 1) * 32];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const float ws = __shfl_sync(0xffffffffu, w, (s0 + i) & 31);
            const float *xs = reinterpret_cast<const float *>(&x[i]);
            if (s0 + i < n_slots)
#pragma unroll
                for (uint32_t e = 0; e < kMine; ++e) v[e] = fmaf(xs[e], ws, v[e]);
            x[i] = y[i];
        }
    }
    float *dst = a.out + (size_t)(row / a.n_heads) * a.out_stride + (size_t)(row % a.n_heads) * D + lane * kMine;
#pragma unroll
    for (uint32_t e = 0; e < kMine; ++e) dst[e] = sum == 0.f ? 0.f : v[e] / sum;
}

// ------------------------------------------------------------------ host side
using qk::DeviceGuard;

bool on(size_t bytes, std::initializer_list<const void *> pointers) {  // all on boundaries of so many bytes
    return std::all_of(pointers.begin(), pointers.end(), [&](const void *p) { return (uintptr_t)p % bytes == 0; });
}

qk_status check_cache(const qk_kv_cache *c, const char *what) {
    if (!c) return qk::fail(QK_ERR_VALUE, "%s is null", what);
    if (c->dtype != QK_F32 && c->dtype != QK_BF16 && c->dtype != QK_I8)
        return qk::fail(QK_ERR_VALUE, "%s: dtype must be float32, bfloat16 or int8, got tag %d", what, c->dtype);
    if (c->n_seq == 0 || c->n_kv_heads == 0 || c->rows == 0 || c->head_dim == 0)
        return qk::fail(QK_ERR_VALUE, "%s is empty: %zu slots, %zu kv heads, %zu rows, head_dim %zu", what, c->n_seq,
                        c->n_kv_heads, c->rows, c->head_dim);
    if (c->head_dim > 256 || c->head_dim % 2)
        return qk::fail(QK_ERR_VALUE, "%s: head_dim must be even and at most 256, got %zu", what, c->head_dim);
    if (c->rows > 0x7fffffffull || c->n_seq > 0x7fffffffull || c->n_kv_heads > 65535)
        return qk::fail(QK_ERR_VALUE, "%s: at most 2^31 - 1 rows and slots and 65535 kv heads, got %zu, %zu, %zu", what, c->rows,
                        c->n_seq, c->n_kv_heads);
    if (!c->k || !c->v) return qk::fail(QK_ERR_VALUE, "%s: k or v is null", what);
    if (c->dtype == QK_I8 && (!c->k_scale || !c->v_scale))
        return qk::fail(QK_ERR_VALUE, "%s: an int8 cache needs k_scale and v_scale", what);
    if (!on(c->dtype == QK_F32 ? 4 : c->dtype == QK_BF16 ? 2 : 1, {c->k, c->v}) ||
        (c->dtype == QK_I8 && !on(4, {c->k_scale, c->v_scale})))
        return qk::fail(QK_ERR_VALUE, "%s: rows or scales lie on no boundary of their type", what);
    return QK_OK;
}

CacheView view(const qk_kv_cache *c) {
    CacheView v{};
    if (c) {
        v.k = c->k, v.v = c->v, v.k_scale = c->k_scale, v.v_scale = c->v_scale;
        v.rows = (uint32_t)c->rows, v.n_seq = (uint32_t)c->n_seq, v.n_kv = (uint32_t)c->n_kv_heads, v.d = (uint32_t)c->head_dim;
        v.dtype = c->dtype;
    }
    return v;
}

// The prefix of an attention call fits the cache it stands in front of.
qk_status check_prefix(const qk_kv_cache *c, const qk_kv_cache *p, size_t prefix_seq, size_t prefix_len) {
    if (prefix_len == 0) return QK_OK;
    qk_status st = check_cache(p, "prefix");
    if (st != QK_OK) return st;
    if (p->dtype != c->dtype || p->n_kv_heads != c->n_kv_heads || p->head_dim != c->head_dim)
        return qk::fail(QK_ERR_VALUE, "prefix and cache must agree in dtype, kv heads and head_dim: tags %d, %d; %zu, %zu; %zu, %zu",
                        p->dtype, c->dtype, p->n_kv_heads, c->n_kv_heads, p->head_dim, c->head_dim);
    if (prefix_seq >= p->n_seq || prefix_len > p->rows)
        return qk::fail(QK_ERR_VALUE, "prefix: %zu rows of slot %zu do not lie in %zu slots of %zu rows", prefix_len, prefix_seq,
                        p->n_seq, p->rows);
    return QK_OK;
}

qk_status check_heads(const qk_kv_cache *c, size_t n_heads, size_t n_tokens) {
    if (n_heads == 0 || n_heads % c->n_kv_heads != 0)
        return qk::fail(QK_ERR_VALUE, "n_kv_heads must divide n_heads: n_heads=%zu, n_kv_heads=%zu", n_heads, c->n_kv_heads);
    if (n_heads > 65535 || n_tokens > (1u << 24) || n_tokens * n_heads > 0x7fffffffull)
        return qk::fail(QK_ERR_VALUE, "%zu tokens of %zu heads are more than one call takes", n_tokens, n_heads);
    return QK_OK;
}

// A token's row of `width` values, `stride` to the next.
qk_status check_rows(const char *what, const void *p, size_t stride, size_t width) {
    if (!p) return qk::fail(QK_ERR_VALUE, "%s is null", what);
    if (!on(4, {p})) return qk::fail(QK_ERR_VALUE, "%s lies on no float boundary", what);
    if (stride < width) return qk::fail(QK_ERR_VALUE, "%s: rows of %zu values cannot be %zu apart", what, width, stride);
    return QK_OK;
}

qk_status check_scratch(const void *scratch, size_t need) {
    if (need && (!scratch || (uintptr_t)scratch % 16))
        return qk::fail(QK_ERR_VALUE, "scratch is null or on no 16-byte boundary (%zu bytes are needed)", need);
    return QK_OK;
}

qk_status enter(qk_ctx *ctx, qk_ctx **c) {
    qk_status st = qk::resolve_ctx(ctx, c);
    if (st != QK_OK) return st;
    QK_CUDA(cudaSetDevice((*c)->device));
    return QK_OK;
}

// The error word, which must exist before a capture begins.
qk_status ready_error_word(qk_ctx *c) {
    if (!c->d_err.ptr && qk::capturing(c))
        return qk::fail(QK_ERR_VALUE, "qk_cache_check has to be called on this context before a stream capture");
    return qk::error_word(c);
}

#define QK_PDL(c, kernel, grid, block, smem, ...) \
    (void)qk::launch_pdl((c)->pdl, kernel, grid, block, smem, (c)->stream, __VA_ARGS__)

// Whether attend_rows_kernel takes the shape.  (Rows on 16-byte boundaries are a matter of the pointers, below.)
bool takes_rows(const qk_kv_cache *c) { return c->dtype != QK_F32 && (c->head_dim == 64 || c->head_dim == 128); }
bool aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }
bool aligned_rows(const CacheView &v) { return aligned(v.k) && aligned(v.v); }

// Tokens of one launch of append, whose blocks each look through those after their own; a later launch's writes come last
// by the stream's order.  65536 INT8 tokens of 8 heads of 128: 990 us in one launch, 452 by 16384, 398 by 8192, 404 by 4096.
constexpr size_t kAppendTokens = 8192;
constexpr size_t kWantBlocks = 148 * 8, kMinChunk = 256, kResident = 148 * 2;

// The tile kernel takes 128 query rows to an SM: how often the keys (64 to a block, two blocks at a time) are split so
// that the SMs have work.
uint32_t tile_splits(size_t tiles, size_t keys) {
    const size_t pairs = qk::ceil_div(keys, 128);
    return (uint32_t)std::max<size_t>(1, std::min<size_t>({64, pairs, 148 / tiles}));
}
size_t tiles_of(const qk_kv_cache *c, size_t queries, size_t n_heads) {
    return qk::ceil_div(queries * (n_heads / c->n_kv_heads), 128) * c->n_kv_heads;
}
// Whether the query rows on a prefix go eight at a time through attend_rows_kernel, or 128 at a time through the tile
// kernel.  A block of the former costs the same for one row as for eight; one of the latter whatever its rows, and 10 us
// are spent before its first keys and behind its last.  Heads 32 / 8 of 128, by rows against by tiles, us: 8 sequences
// behind 6000 INT8 rows 22.7, 28.2; 12 behind 4000 22.1, 22.2; 16 behind 4000 29.1, 22.3; behind bfloat16 rows 16 and 1500
// 18.5, 19.3; 24 and 1300 22.0, 19.5; 40 and 800 25.5, 19.9.
bool prefix_by_rows(const qk_kv_cache *c, size_t rows, size_t prefix_len) {
    return rows <= 16 || qk::ceil_div(rows, 8) * prefix_len * c->n_kv_heads <= (c->dtype == QK_I8 ? 12u << 14 : 7u << 14);
}

// The most query rows that a block of the call has, and how many blocks of the kernel for it an SM holds.
uint32_t most_rows(const Plan &pl, bool prefix, size_t prefix_rows) {
    return prefix ? std::max(pl.own_rows, (uint32_t)std::min<size_t>(8, prefix_rows)) : pl.own_rows;
}
size_t blocks_an_sm(const qk_kv_cache *c, uint32_t rows) { return (c->dtype == QK_I8 ? 4 : 3) - (rows > 4); }

Plan plan_rows(const qk_kv_cache *c, size_t prefix_len, size_t batch, size_t n_heads) {
    Plan pl{};
    const size_t group = n_heads / c->n_kv_heads;
    auto splits = [](size_t blocks, size_t rows) {
        return std::max<size_t>(1, std::min({(size_t)128, qk::ceil_div(rows, kMinChunk), qk::ceil_div(kWantBlocks, blocks)}));
    };
    const bool by_rows = prefix_len && prefix_by_rows(c, batch * group, prefix_len);
    pl.own_rows = (uint32_t)std::min<size_t>(group, 8);
    pl.own_subs = (uint32_t)qk::ceil_div(group, pl.own_rows);
    pl.prefix_subs = (uint32_t)qk::ceil_div(batch * group, 8);
    const size_t own_blocks = batch * c->n_kv_heads * pl.own_subs, pre_blocks = by_rows ? pl.prefix_subs * c->n_kv_heads : 0;
    size_t own = splits(own_blocks, c->rows), pre = by_rows ? splits(pre_blocks, prefix_len) : 1;
    // Fewer splits where all blocks then fit the device at once and last no longer than two rounds would.  Eight sequences
    // behind 4001 INT8 rows: 19.5 -> 15.1 us; 14 of 2048 INT8 rows: 19.5 -> 17.4, 10 of bfloat16 22.8 -> 19.1.
    const size_t slots = 148 * blocks_an_sm(c, most_rows(pl, by_rows, batch * group));
    if (own_blocks * own + pre_blocks * pre > slots) {
        const size_t fit = by_rows ? (slots - std::min(slots, own_blocks * own)) / pre_blocks : slots / own_blocks;
        size_t &cut = by_rows ? pre : own;
        if (2 * fit > cut) cut = fit;
    }
    // While all blocks are resident at once, the splits are the blocks of a cluster (up to 32 of them become eight), and
    // there is no second launch: one sequence of 2048 INT8 rows, 32 heads: 14 -> 11.6 us a call on the host, the device's
    // time the same.  Where blocks queue, clusters make them wait for one another: 64 sequences 42 -> 47 us.
    pl.cluster = 1;
    const size_t most = std::max(own, pre);
    const size_t size = most > 4 ? 8 : most > 2 ? 4 : most;
    if (most <= 32 && (own_blocks + pre_blocks) * size <= kResident) {
        pl.cluster = (uint32_t)size;
        own = pre = size;
    }
    pl.own_splits = (uint32_t)(qk::ceil_div(own, pl.cluster) * pl.cluster);
    if (by_rows) {
        pl.prefix_splits = (uint32_t)(qk::ceil_div(pre, pl.cluster) * pl.cluster);
        pl.prefix_slots = pl.prefix_splits / pl.cluster;
        pl.prefix_chunk = (uint32_t)(qk::ceil_div(qk::ceil_div(prefix_len, pl.prefix_splits), 64) * 64);
        pl.prefix_blocks = (uint32_t)(pl.prefix_subs * pl.prefix_splits * c->n_kv_heads);
    } else if (prefix_len) {
        pl.prefix_slots = tile_splits(tiles_of(c, batch, n_heads), prefix_len);
    }
    pl.n_slots = pl.prefix_slots + pl.own_splits / pl.cluster;
    return pl;
}

struct PortionPlan {
    uint32_t prefix_splits, own_splits;
};
PortionPlan plan_portion(const qk_kv_cache *c, size_t first_row, size_t prefix_len, size_t tokens, size_t n_heads) {
    const size_t tiles = tiles_of(c, tokens, n_heads);
    return {prefix_len ? tile_splits(tiles, prefix_len) : 0, tile_splits(tiles, first_row + tokens)};
}

size_t partial_bytes(size_t queries, size_t n_heads, size_t slots, size_t d) {
    return slots > 1 ? queries * n_heads * slots * (d + 2) * sizeof(float) : 0;
}

qk_status join(qk_ctx *c, const qk::AttendArgs &a, uint32_t n_slots, uint32_t d) {
    if (n_slots == 1) return QK_OK;
    const dim3 grid(a.n_queries * a.n_heads), few((unsigned)qk::ceil_div((size_t)a.n_queries * a.n_heads, 4));
    if (n_slots <= 32 && d == 128) QK_PDL(c, join_few_kernel<128>, few, dim3(128), 0, a, n_slots);
    else if (n_slots <= 32) QK_PDL(c, join_few_kernel<64>, few, dim3(128), 0, a, n_slots);
    else if (d == 128) QK_PDL(c, join_kernel<128>, grid, dim3(128), 0, a, n_slots);
    else QK_PDL(c, join_kernel<64>, grid, dim3(128), 0, a, n_slots);
    QK_CUDA(cudaGetLastError());
    c->launches++;
    return QK_OK;
}

qk::TileArgs tile_args(const qk::AttendArgs &a, uint32_t n_splits, uint32_t slot0, uint32_t n_slots) {
    qk::TileArgs t{};
    t.q = a.q, t.q_stride = a.q_stride, t.out = a.out, t.out_stride = a.out_stride, t.scratch = a.scratch;
    t.n_queries = a.n_queries, t.n_heads = a.n_heads;
    t.n_splits = n_splits, t.slot0 = slot0, t.n_slots = n_slots;
    return t;
}
qk_status prefix_tiles(qk_ctx *c, const CacheView &pre, const qk::AttendArgs &a, uint32_t n_splits, uint32_t n_slots) {
    qk::TileArgs t = tile_args(a, n_splits, 0, n_slots);
    t.seq = a.prefix_seq, t.n_keys = a.prefix_len;
    return qk::attend_tiles(c, pre, t);
}

template <bool kI8, int D, int kMost>
qk_status launch_rows(qk_ctx *c, const CacheView &own, const CacheView &pre, const qk::AttendArgs &a, const Plan &pl) {
    constexpr size_t smem = AttendShape<kI8, D>::kSmem;
    qk_status st = qk::allow_smem(c, attend_rows_kernel<kI8, D, kMost>, smem);
    if (st != QK_OK) return st;
    const unsigned blocks = pl.prefix_blocks + a.n_queries * own.n_kv * pl.own_subs * pl.own_splits;
    (void)qk::launch_pdl_cluster(c->pdl, attend_rows_kernel<kI8, D, kMost>, dim3(blocks), dim3(128), pl.cluster, smem, c->stream,
                                 own, pre, a, pl);
    QK_CUDA(cudaGetLastError());
    c->launches++;
    return join(c, a, pl.n_slots, D);
}
template <bool kI8, int D>
qk_status launch_rows(qk_ctx *c, const CacheView &own, const CacheView &pre, const qk::AttendArgs &a, const Plan &pl) {
    if (a.prefix_len && !pl.prefix_blocks) {
        qk_status st = prefix_tiles(c, pre, a, pl.prefix_slots, pl.n_slots);
        if (st != QK_OK) return st;
    }
    return most_rows(pl, pl.prefix_blocks != 0, (size_t)a.n_queries * (a.n_heads / own.n_kv)) > 4
               ? launch_rows<kI8, D, 2>(c, own, pre, a, pl)
               : launch_rows<kI8, D, 1>(c, own, pre, a, pl);
}

qk_status attend(qk_ctx *ctx, const qk_kv_cache *cache, const qk_kv_cache *prefix, const qk::AttendArgs &a) {
    qk_ctx *c;
    DeviceGuard guard;
    qk_status st = enter(ctx, &c);
    if (st != QK_OK) return st;
    std::lock_guard<std::mutex> lock(c->mu);
    const CacheView own = view(cache), pre = view(a.prefix_len ? prefix : nullptr);
    if (takes_rows(cache) && aligned_rows(own) && aligned_rows(pre) && aligned(a.q) && a.q_stride % 4 == 0) {
        if ((st = ready_error_word(c)) != QK_OK) return st;
        if (!a.kv_len && a.n_queries > 1) {
            const PortionPlan pp = plan_portion(cache, a.first_row, a.prefix_len, a.n_queries, a.n_heads);
            const uint32_t slots = pp.prefix_splits + pp.own_splits;
            if (a.prefix_len && (st = prefix_tiles(c, pre, a, pp.prefix_splits, slots)) != QK_OK) return st;
            qk::TileArgs t = tile_args(a, pp.own_splits, pp.prefix_splits, slots);
            t.seq = a.seq, t.first_row = a.first_row, t.causal = 1;
            if ((st = qk::attend_tiles(c, own, t)) != QK_OK) return st;
            return join(c, a, slots, own.d);
        }
        const Plan pl = plan_rows(cache, a.prefix_len, a.n_queries, a.n_heads);
        if (own.dtype == QK_I8)
            return own.d == 128 ? launch_rows<true, 128>(c, own, pre, a, pl) : launch_rows<true, 64>(c, own, pre, a, pl);
        return own.d == 128 ? launch_rows<false, 128>(c, own, pre, a, pl) : launch_rows<false, 64>(c, own, pre, a, pl);
    }
    const unsigned blocks = (unsigned)qk::ceil_div((size_t)a.n_queries * a.n_heads, 4);
    if (own.dtype == QK_I8) QK_PDL(c, attend_plain_kernel<int8_t>, dim3(blocks), dim3(128), 0, own, pre, a);
    else if (own.dtype == QK_BF16) QK_PDL(c, attend_plain_kernel<uint16_t>, dim3(blocks), dim3(128), 0, own, pre, a);
    else QK_PDL(c, attend_plain_kernel<float>, dim3(blocks), dim3(128), 0, own, pre, a);
    QK_CUDA(cudaGetLastError());
    c->launches++;
    return QK_OK;
}

}  // namespace

extern "C" {

qk_status qk_cache_check(qk_ctx *ctx, const qk_kv_cache *cache) {
    qk_status st = check_cache(cache, "cache");
    if (st != QK_OK) return st;
    qk_ctx *c;
    DeviceGuard guard;
    if ((st = enter(ctx, &c)) != QK_OK) return st;
    std::lock_guard<std::mutex> lock(c->mu);
    return ready_error_word(c);
}

qk_status qk_cache_append(qk_ctx *ctx, const qk_kv_cache *cache, const float *q, size_t q_stride, float *q_out,
                          size_t q_out_stride, size_t n_heads, const float *k, size_t k_stride, const float *v,
                          size_t v_stride, const float *cos_sin, size_t n_positions, const int32_t *positions,
                          const int32_t *seq_index, size_t first_position, size_t n_tokens) {
    qk_status st = check_cache(cache, "cache");
    if (st != QK_OK) return st;
    const size_t d = cache->head_dim, kv_width = cache->n_kv_heads * d;
    if (q) {
        if ((st = check_heads(cache, n_heads, n_tokens)) != QK_OK) return st;
        if ((st = check_rows("q", q, q_stride, n_heads * d)) != QK_OK) return st;
        if ((st = check_rows("q_out", q_out, q_out_stride, n_heads * d)) != QK_OK) return st;
    } else if ((st = check_heads(cache, cache->n_kv_heads, n_tokens)) != QK_OK) {
        return st;
    }
    if ((st = check_rows("k", k, k_stride, kv_width)) != QK_OK) return st;
    if ((st = check_rows("v", v, v_stride, kv_width)) != QK_OK) return st;
    if (!cos_sin || !positions || !seq_index) return qk::fail(QK_ERR_VALUE, "cos_sin, positions or seq_index is null");
    if (!on(4, {cos_sin, positions, seq_index}))
        return qk::fail(QK_ERR_VALUE, "cos_sin, positions or seq_index lies on no boundary of its type");
    if (first_position > 0x7fffffffull || n_positions > 0x7fffffffull)
        return qk::fail(QK_ERR_VALUE, "positions are 32-bit: first_position %zu, n_positions %zu", first_position, n_positions);
    qk_ctx *c;
    DeviceGuard guard;
    if ((st = enter(ctx, &c)) != QK_OK) return st;
    if (n_tokens == 0) return QK_OK;
    std::lock_guard<std::mutex> lock(c->mu);
    if ((st = ready_error_word(c)) != QK_OK) return st;
    const CacheView cv = view(cache);
    int *err = (int *)c->d_err.ptr;
    // (a row's vectors lie on their boundaries where the tensors' addresses and strides do)
    const size_t mask = ((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)v | (uintptr_t)cv.k | (uintptr_t)cv.v) |
                        (q ? (q_stride | q_out_stride) * 4 : 0) | (k_stride | v_stride) * 4;
    const int groups = mask % 16 || (uintptr_t)cos_sin % 16 ? 0 : d == 64 ? 1 : d == 128 ? 2 : d == 256 ? 4 : 0;
#define QK_APPEND_ARGS                                                                                                    \
    cv, q, q_stride, q_out, q_out_stride, (uint32_t)n_heads, k, k_stride, v, v_stride, cos_sin, (uint32_t)n_positions, positions, \
        seq_index, (uint32_t)first_position, (uint32_t)n
#define QK_APPEND_WIDE(KV, N) QK_PDL(c, (append_wide_kernel<KV, N>), wide, dim3(128), 0, QK_APPEND_ARGS, wide_kv, err)
#define QK_APPEND(KV)                                                                                        \
    do {                                                                                                     \
        if (groups == 1) QK_APPEND_WIDE(KV, 1);                                                              \
        else if (groups == 2) QK_APPEND_WIDE(KV, 2);                                                         \
        else if (groups == 4) QK_APPEND_WIDE(KV, 4);                                                         \
        else QK_PDL(c, append_kernel<KV>, dim3((unsigned)n), dim3(256), 0, QK_APPEND_ARGS, err);      \
    } while (0)
    const uint32_t wide_kv = (uint32_t)qk::ceil_div(2 * cache->n_kv_heads, 16);
    for (size_t done = 0; done < n_tokens; done += kAppendTokens) {
        const size_t n = std::min(kAppendTokens, n_tokens - done);
        const dim3 wide((unsigned)n, wide_kv + (unsigned)(q ? qk::ceil_div(n_heads, 16) : 0));
        if (cv.dtype == QK_I8) QK_APPEND(int8_t);
        else if (cv.dtype == QK_BF16) QK_APPEND(uint16_t);
        else QK_APPEND(float);
        QK_CUDA(cudaGetLastError());
        c->launches++;
        c->err_armed = true;
        if (q) q += n * q_stride, q_out += n * q_out_stride;
        k += n * k_stride, v += n * v_stride, positions += n, seq_index += n;
    }
#undef QK_APPEND_WIDE
#undef QK_APPEND_ARGS
#undef QK_APPEND
    return QK_OK;
}

qk_status qk_cache_read(qk_ctx *ctx, const qk_kv_cache *cache, const int32_t *positions, const int32_t *seq_index,
                        size_t first_position, size_t n_tokens, int32_t out_dtype, void *k_out, void *v_out) {
    qk_status st = check_cache(cache, "cache");
    if (st != QK_OK) return st;
    if ((st = check_heads(cache, cache->n_kv_heads, n_tokens)) != QK_OK) return st;
    if (!positions || !seq_index || !k_out || !v_out)
        return qk::fail(QK_ERR_VALUE, "positions, seq_index, k_out or v_out is null");
    if (!on(4, {positions, seq_index}) || !on(out_dtype == QK_F32 ? 4 : 2, {k_out, v_out}))
        return qk::fail(QK_ERR_VALUE, "positions, seq_index, k_out or v_out lies on no boundary of its type");
    if (out_dtype != QK_F32 && out_dtype != QK_BF16)
        return qk::fail(QK_ERR_VALUE, "rows are read as float32 or bfloat16, got tag %d", out_dtype);
    if (first_position > 0x7fffffffull) return qk::fail(QK_ERR_VALUE, "positions are 32-bit: first_position %zu", first_position);
    qk_ctx *c;
    DeviceGuard guard;
    if ((st = enter(ctx, &c)) != QK_OK) return st;
    if (n_tokens == 0) return QK_OK;
    std::lock_guard<std::mutex> lock(c->mu);
    if ((st = ready_error_word(c)) != QK_OK) return st;
    const unsigned blocks = (unsigned)qk::ceil_div(n_tokens * cache->n_kv_heads * 2, 8);
    const CacheView cv = view(cache);
    int *err = (int *)c->d_err.ptr;
    const bool vec = cv.d % 4 == 0 && (((uintptr_t)cv.k | (uintptr_t)cv.v | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0;
#define QK_READ_V(KV, Out, V)                                                                                             \
    QK_PDL(c, (read_kernel<KV, Out, V>), dim3(blocks), dim3(256), 0, cv, positions, seq_index, (uint32_t)first_position, \
           (uint32_t)n_tokens, (Out *)k_out, (Out *)v_out, err)
#define QK_READ(KV, Out)                     \
    do {                                     \
        if (vec) QK_READ_V(KV, Out, true);   \
        else QK_READ_V(KV, Out, false);      \
    } while (0)
#define QK_READ_TO(Out)                                \
    do {                                               \
        if (cv.dtype == QK_I8) QK_READ(int8_t, Out);   \
        else if (cv.dtype == QK_BF16) QK_READ(uint16_t, Out); \
        else QK_READ(float, Out);                      \
    } while (0)
    if (out_dtype == QK_F32) QK_READ_TO(float);
    else QK_READ_TO(uint16_t);
#undef QK_READ_TO
#undef QK_READ
#undef QK_READ_V
    QK_CUDA(cudaGetLastError());
    c->launches++;
    c->err_armed = true;
    return QK_OK;
}

size_t qk_cache_attend_scratch(const qk_kv_cache *cache, size_t prefix_len, size_t batch, size_t n_heads) {
    if (!cache || cache->n_kv_heads == 0 || n_heads < cache->n_kv_heads || !batch || !takes_rows(cache)) return 0;
    return partial_bytes(batch, n_heads, plan_rows(cache, prefix_len, batch, n_heads).n_slots, cache->head_dim);
}

qk_status qk_cache_attend(qk_ctx *ctx, const qk_kv_cache *cache, const qk_kv_cache *prefix, size_t prefix_seq,
                          size_t prefix_len, const float *q, size_t q_stride, const int32_t *kv_len, size_t batch,
                          size_t n_heads, void *scratch, float *out, size_t out_stride) {
    qk_status st = check_cache(cache, "cache");
    if (st != QK_OK) return st;
    if ((st = check_prefix(cache, prefix, prefix_seq, prefix_len)) != QK_OK) return st;
    if ((st = check_heads(cache, n_heads, batch)) != QK_OK) return st;
    if (batch > cache->n_seq) return qk::fail(QK_ERR_VALUE, "%zu sequences, but the cache has %zu slots", batch, cache->n_seq);
    if ((st = check_rows("q", q, q_stride, n_heads * cache->head_dim)) != QK_OK) return st;
    if ((st = check_rows("out", out, out_stride, n_heads * cache->head_dim)) != QK_OK) return st;
    if (!kv_len) return qk::fail(QK_ERR_VALUE, "kv_len is null");
    if (!on(4, {kv_len})) return qk::fail(QK_ERR_VALUE, "kv_len lies on no boundary of its type");
    if ((st = check_scratch(scratch, qk_cache_attend_scratch(cache, prefix_len, batch, n_heads))) != QK_OK) return st;
    if (batch == 0) return QK_OK;
    qk::AttendArgs a{};
    a.q = q, a.q_stride = q_stride, a.out = out, a.out_stride = out_stride, a.kv_len = kv_len;
    a.n_queries = (uint32_t)batch, a.n_heads = (uint32_t)n_heads;
    a.prefix_len = (uint32_t)prefix_len, a.prefix_seq = prefix_seq;
    a.scratch = (float *)scratch;
    return attend(ctx, cache, prefix, a);
}

size_t qk_cache_portion_scratch(const qk_kv_cache *cache, size_t first_row, size_t prefix_len, size_t n_tokens,
                                size_t n_heads) {
    if (!cache || cache->n_kv_heads == 0 || n_heads < cache->n_kv_heads || !n_tokens || !takes_rows(cache)) return 0;
    if (n_tokens == 1) return qk_cache_attend_scratch(cache, prefix_len, 1, n_heads);
    const PortionPlan pp = plan_portion(cache, first_row, prefix_len, n_tokens, n_heads);
    return partial_bytes(n_tokens, n_heads, pp.prefix_splits + pp.own_splits, cache->head_dim);
}

qk_status qk_cache_portion(qk_ctx *ctx, const qk_kv_cache *cache, size_t seq, size_t first_row, const qk_kv_cache *prefix,
                           size_t prefix_seq, size_t prefix_len, const float *q, size_t q_stride, size_t n_tokens,
                           size_t n_heads, void *scratch, float *out, size_t out_stride) {
    qk_status st = check_cache(cache, "cache");
    if (st != QK_OK) return st;
    if ((st = check_prefix(cache, prefix, prefix_seq, prefix_len)) != QK_OK) return st;
    if ((st = check_heads(cache, n_heads, n_tokens)) != QK_OK) return st;
    if (seq >= cache->n_seq) return qk::fail(QK_ERR_VALUE, "slot %zu outside the cache of %zu slots", seq, cache->n_seq);
    if (first_row > cache->rows || n_tokens > cache->rows - first_row)
        return qk::fail(QK_ERR_VALUE, "%zu tokens from row %zu on do not fit the cache of %zu rows", n_tokens, first_row, cache->rows);
    if ((st = check_rows("q", q, q_stride, n_heads * cache->head_dim)) != QK_OK) return st;
    if ((st = check_rows("out", out, out_stride, n_heads * cache->head_dim)) != QK_OK) return st;
    if ((st = check_scratch(scratch, qk_cache_portion_scratch(cache, first_row, prefix_len, n_tokens, n_heads))) != QK_OK) return st;
    if (n_tokens == 0) return QK_OK;
    qk::AttendArgs a{};
    a.q = q, a.q_stride = q_stride, a.out = out, a.out_stride = out_stride;
    a.n_queries = (uint32_t)n_tokens, a.n_heads = (uint32_t)n_heads;
    a.seq = seq, a.first_row = (uint32_t)first_row;
    a.prefix_len = (uint32_t)prefix_len, a.prefix_seq = prefix_seq;
    a.scratch = (float *)scratch;
    return attend(ctx, cache, prefix, a);
}

}  // extern "C"
