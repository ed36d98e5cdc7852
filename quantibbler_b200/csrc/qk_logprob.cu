// Log probabilities, entropy and the most probable entries from logits.
#include <cmath>

#include "qk_common.h"

namespace {

constexpr uint32_t kMaxTop = 32;

struct LogProbArgs {
    const float *logits;
    size_t stride;
    uint32_t n_tokens, vocab, n_top;
    const int32_t *targets;
    float *lse, *logprob, *entropy, *top_logprob;
    int32_t *top_ids;
};

// An order on (value, index) as one number: larger is better, the lowest index first among equals (0 and -0 are).
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return ((uint64_t)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32) | (0xffffffffu - index);
}

__device__ __forceinline__ float block_reduce(float v, bool is_max, float *red) {
    for (int off = 16; off > 0; off >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, v, off);
        v = is_max ? fmaxf(v, o) : v + o;
    }
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
    __syncthreads();
    v = red[0];
    for (uint32_t w = 1; w < blockDim.x / 32; ++w) v = is_max ? fmaxf(v, red[w]) : v + red[w];
    __syncthreads();
    return v;
}

__global__ void __launch_bounds__(256)
log_probs_plain_kernel(LogProbArgs a) {
    qk::pdl_launch();
    qk::pdl_wait();
    __shared__ float red[8];
    __shared__ unsigned long long best;
    const uint32_t t = blockIdx.x;
    const float *x = a.logits + t * a.stride;
    float m = -INFINITY, bad = 0.f;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += 256) {
        m = fmaxf(m, x[i]);
        if (!(x[i] < INFINITY)) bad = 1.f;
    }
    m = block_reduce(m, true, red);
    bad = block_reduce(bad, true, red);
    float s = 0.f, w = 0.f;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += 256) {
        const float y = x[i] - m, e = expf(y);
        s += e;
        w += e == 0.f ? 0.f : y * e;
    }
    s = block_reduce(s, false, red);
    w = block_reduce(w, false, red);
    const float nan = __int_as_float(0x7fffffff);
    const bool ok = bad == 0.f && m > -INFINITY;
    const float ln = logf(s);
    if (threadIdx.x == 0) {
        if (a.lse) a.lse[t] = ok ? m + ln : nan;
        if (a.entropy) a.entropy[t] = ok ? ln - w / s : nan;
        if (a.logprob) {
            const int32_t id = a.targets ? a.targets[t] : -1;
            a.logprob[t] = id < 0 ? 0.f : !ok || (uint32_t)id >= a.vocab ? nan : (x[id] - m) - ln;
        }
    }
    uint64_t below = ~0ull;
    for (uint32_t j = 0; j < a.n_top; ++j) {
        if (threadIdx.x == 0) best = 0;
        __syncthreads();
        uint64_t mine = 0;
        for (uint32_t i = threadIdx.x; i < a.vocab; i += 256) {
            const uint64_t key = rank_key(x[i], i);
            if (key < below && key > mine) mine = key;
        }
        atomicMax(&best, (unsigned long long)mine);
        __syncthreads();
        below = best;
        if (threadIdx.x == 0) {
            const uint32_t id = 0xffffffffu - (uint32_t)below;
            if (a.top_ids) a.top_ids[(size_t)t * a.n_top + j] = ok ? (int32_t)id : -1;
            if (a.top_logprob) a.top_logprob[(size_t)t * a.n_top + j] = ok ? (x[id] - m) - ln : nan;
        }
        __syncthreads();
    }
}

}  // namespace

extern "C" {

size_t qk_log_probs_scratch(size_t n_tokens, size_t vocab, size_t n_top) {
    (void)n_tokens, (void)vocab, (void)n_top;
    return 0;
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
    if (logprob && !targets) return qk::fail(QK_ERR_VALUE, "logprob needs targets");
    if (!scratch && qk_log_probs_scratch(n_tokens, vocab, n_top)) return qk::fail(QK_ERR_VALUE, "scratch is null");
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
    (void)qk::launch_pdl(c->pdl, log_probs_plain_kernel, dim3((unsigned)n_tokens), dim3(256), 0, c->stream, a);
    QK_CUDA(cudaGetLastError());
    c->launches++;
    return QK_OK;
}

}  // extern "C"
