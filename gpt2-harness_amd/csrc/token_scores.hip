// Scores of given tokens under rows of logits (gfx950): log probability, entropy of
// the row, its most probable alternatives, and the gradient that these send back.
//
// With m = max_j x_j, z_j = x_j - m, e_j = exp(z_j) and
//     d = sum of e_j over all j but one that has x_j = m     (so sum e_j = 1 + d)
//     log p_j = z_j - log1p(d)
//     H       = log1p(d) - (sum_j e_j z_j) / (1 + d)
// (the reference's log_softmax in F.cross_entropy, model.py:591-597). d and not the sum
// is kept: 1 + d loses a d below 2^-24, which is the whole log probability of a
// token that the model is sure of; both terms of H are positive, so nothing cancels.
// A row that holds NaN or +inf, or nothing above -inf, has NaN scores, as torch's
// log_softmax. -inf elsewhere is a probability of 0 and adds nothing to H.
//
// Alternatives go by the logits: larger first, of equal ones the lower index; NaN
// stands above everything (as torch.topk).
//
// Gradient of (log p_t, H, log p of the alternatives a_i) weighted by g, h, g_i:
//     [j = t] g + sum_i [j = a_i] g_i - p_j (g + sum_i g_i + h (log p_j + H)),
// with 1 - p_j of a hot j from d / (1 + d) where x_j = m.
#include <algorithm>
#include <cmath>

#include "tiq_internal.hpp"

namespace tiq {
namespace {

constexpr int kMaxTop = 64;
constexpr int64_t kMaxVocab = 1 << 30;

__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const uint16_t* p) { return bf16_bits_to_f32(*p); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = f32_to_bf16_bits(v); }

// Order of logits as unsigned numbers: NaN on top, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// ... and of logits with their places: the lower place wins among equals.
__device__ __forceinline__ uint64_t place_key(float x, uint32_t j) {
    return (uint64_t)order_of(x) << 32 | (uint32_t)~j;
}

__device__ __forceinline__ uint64_t max_u64(uint64_t a, uint64_t b) { return a > b ? a : b; }

// Reductions over a workgroup of 256; every thread gets the result.
__device__ __forceinline__ uint64_t group_max(uint64_t v, uint64_t* red) {
#pragma unroll
    for (int off = 32; off; off >>= 1) v = max_u64(v, __shfl_xor(v, off, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return max_u64(max_u64(red[0], red[1]), max_u64(red[2], red[3]));
}
__device__ __forceinline__ float group_sum(float v, float* red) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

struct Scores {
    const int64_t* tokens;
    int64_t ignore;
    int top;
    float *logprob, *entropy, *stats;
    int64_t* top_ids;
    float* top_logprobs;
};

// z of a logit: finite values keep -inf away from e z = 0 (-inf).
__device__ __forceinline__ float weighted(float e, float z) { return e * fmaxf(z, -200.f); }

template <typename TX>
__global__ __launch_bounds__(256) void scores_simple(const TX* __restrict__ x, int64_t rows, int64_t sb, int64_t sr,
                                                     int V, Scores o) {
    __shared__ uint64_t red[4];
    __shared__ float redf[4];
    const int64_t row = blockIdx.x;
    const TX* xr = x + (row / rows) * sb + (row % rows) * sr;
    uint64_t best = 0;
    for (int j = threadIdx.x; j < V; j += 256) best = max_u64(best, place_key(logit(xr + j), j));
    best = group_max(best, red);
    const int at = (int)~(uint32_t)best;
    const float m = logit(xr + at);
    float d = 0.f, s1 = 0.f;
    for (int j = threadIdx.x; j < V; j += 256) {
        const float z = logit(xr + j) - m, e = expf(z);
        d += j == at && e == 1.f ? 0.f : e;
        s1 += weighted(e, z);
    }
    d = group_sum(d, redf);
    s1 = group_sum(s1, redf);
    const float L = log1pf(d), H = L - s1 / (1.f + d);
    if (threadIdx.x == 0) {
        const int64_t t = o.tokens[row];
        o.logprob[row] = t == o.ignore ? 0.f : t < 0 || t >= V ? __builtin_nanf("") : logit(xr + t) - m - L;
        o.entropy[row] = H;
        if (o.stats) {
            o.stats[2 * row] = m;
            o.stats[2 * row + 1] = d;
        }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < o.top; ++k) {
        uint64_t next = 0;
        for (int j = threadIdx.x; j < V; j += 256) {
            const uint64_t c = place_key(logit(xr + j), j);
            next = c < last ? max_u64(next, c) : next;
        }
        last = group_max(next, red);
        if (threadIdx.x == 0) {
            const uint32_t j = ~(uint32_t)last;
            o.top_ids[row * o.top + k] = j;
            o.top_logprobs[row * o.top + k] = logit(xr + j) - m - L;
        }
    }
}

struct Grads {
    const int64_t* tokens;
    int64_t ignore;
    int top;
    const float *stats, *entropy, *g_logprob, *g_entropy;
    const int64_t* top_ids;
    const float* g_top;
};

template <typename TX>
__global__ __launch_bounds__(256) void grad_simple(const TX* __restrict__ x, int64_t rows, int64_t sb, int64_t sr,
                                                   int V, Grads o, TX* __restrict__ grad) {
    const int64_t row = blockIdx.x;
    const TX* xr = x + (row / rows) * sb + (row % rows) * sr;
    TX* gr = grad + row * V;
    const float m = o.stats[2 * row], d = o.stats[2 * row + 1], s = 1.f + d, L = log1pf(d), H = o.entropy[row];
    const int64_t t = o.tokens[row];
    float gl = o.g_logprob && t != o.ignore ? o.g_logprob[row] : 0.f;
    if (t != o.ignore && (t < 0 || t >= V)) gl = __builtin_nanf("");
    const float gh = o.g_entropy ? o.g_entropy[row] : 0.f;
    float gt = 0.f;
    if (o.g_top)
        for (int k = 0; k < o.top; ++k) gt += o.g_top[row * o.top + k];
    for (int j = threadIdx.x; j < V; j += 256) {
        const float z = logit(xr + j) - m, e = expf(z), p = e / s;
        const float rest = e == 1.f ? d / s : 1.f - p;  // 1 - p
        float hot = j == t ? gl : 0.f;
        if (o.g_top)
            for (int k = 0; k < o.top; ++k) hot += o.top_ids[row * o.top + k] == j ? o.g_top[row * o.top + k] : 0.f;
        put(gr + j, hot * rest - p * ((gl + gt - hot) + gh * (fmaxf(z, -200.f) - L + H)));
    }
}

int check_rows(const void* logits, int dtype, int64_t batch, int64_t rows, int64_t vocab, const int64_t* tokens,
               int top) {
    if ((dtype != TIQ_F32 && dtype != TIQ_BF16) || batch < 0 || rows < 0 || vocab < 1 || top < 0) return TIQ_EINVAL;
    if (top > kMaxTop || top > vocab) return TIQ_EINVAL;
    if (vocab > kMaxVocab || (rows && batch > 0x7fffffffLL / rows)) return TIQ_EUNSUPPORTED;
    if (batch * rows == 0) return TIQ_OK;
    if (!logits || !tokens) return TIQ_EINVAL;
    if (!aligned(logits, dtype == TIQ_F32 ? 4 : 2) || !aligned(tokens, 8)) return TIQ_EALIGN;
    return TIQ_OK;
}

}  // namespace
}  // namespace tiq

using namespace tiq;

extern "C" size_t tiq_token_logprobs_workspace(int dtype, int64_t rows, int64_t vocab, int top) {
    (void)dtype, (void)rows, (void)vocab, (void)top;
    return 0;
}

extern "C" int tiq_token_logprobs(const void* logits, int dtype, int64_t batch, int64_t rows, int64_t stride_batch,
                                  int64_t stride_row, int64_t vocab, const int64_t* tokens, int64_t ignore_index,
                                  int top, float* logprob, float* entropy, float* stats, int64_t* top_ids,
                                  float* top_logprobs, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check_rows(logits, dtype, batch, rows, vocab, tokens, top);
    if (rc != TIQ_OK || batch * rows == 0) return rc;
    if (!logprob || !entropy || (top && (!top_ids || !top_logprobs))) return TIQ_EINVAL;
    (void)workspace, (void)workspace_bytes;
    const Scores o = {tokens, ignore_index, top, logprob, entropy, stats, top_ids, top_logprobs};
    const dim3 grid((unsigned)(batch * rows));
    if (dtype == TIQ_F32)
        hipLaunchKernelGGL(scores_simple<float>, grid, dim3(256), 0, as_stream(stream),
                           static_cast<const float*>(logits), rows, stride_batch, stride_row, (int)vocab, o);
    else
        hipLaunchKernelGGL(scores_simple<uint16_t>, grid, dim3(256), 0, as_stream(stream),
                           static_cast<const uint16_t*>(logits), rows, stride_batch, stride_row, (int)vocab, o);
    return launch_status();
}

extern "C" int tiq_token_logprobs_grad(const void* logits, int dtype, int64_t batch, int64_t rows,
                                       int64_t stride_batch, int64_t stride_row, int64_t vocab, const int64_t* tokens,
                                       int64_t ignore_index, const float* stats, const float* entropy,
                                       const float* g_logprob, const float* g_entropy, int top,
                                       const int64_t* top_ids, const float* g_top, void* grad, void* stream) {
    const int rc = check_rows(logits, dtype, batch, rows, vocab, tokens, top);
    if (rc != TIQ_OK || batch * rows == 0) return rc;
    if (!stats || !entropy || !grad || (g_top && (!top || !top_ids))) return TIQ_EINVAL;
    if (!aligned(grad, dtype == TIQ_F32 ? 4 : 2)) return TIQ_EALIGN;
    const Grads o = {tokens, ignore_index, top, stats, entropy, g_logprob, g_entropy, top_ids, g_top};
    const dim3 grid((unsigned)(batch * rows));
    if (dtype == TIQ_F32)
        hipLaunchKernelGGL(grad_simple<float>, grid, dim3(256), 0, as_stream(stream),
                           static_cast<const float*>(logits), rows, stride_batch, stride_row, (int)vocab, o,
                           static_cast<float*>(grad));
    else
        hipLaunchKernelGGL(grad_simple<uint16_t>, grid, dim3(256), 0, as_stream(stream),
                           static_cast<const uint16_t*>(logits), rows, stride_batch, stride_row, (int)vocab, o,
                           static_cast<uint16_t*>(grad));
    return launch_status();
}
