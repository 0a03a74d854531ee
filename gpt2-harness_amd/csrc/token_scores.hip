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
// The logit of a key's upper half.
__device__ __forceinline__ float of_order(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

// 16 bytes of logits, at a 16-byte boundary.
template <typename TX>
constexpr int kVec = 16 / (int)sizeof(TX);
__device__ __forceinline__ void load_vec(const float* p, float* v) {
    *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(p);
}
__device__ __forceinline__ void load_vec(const uint16_t* p, float* v) {
    const uint4 t = *reinterpret_cast<const uint4*>(p);
    v[0] = bf_lo(t.x), v[1] = bf_hi(t.x), v[2] = bf_lo(t.y), v[3] = bf_hi(t.y);
    v[4] = bf_lo(t.z), v[5] = bf_hi(t.z), v[6] = bf_lo(t.w), v[7] = bf_hi(t.w);
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;

// Running maximum, sum of e and sum of e z of some of a row's logits. m starts at the
// lowest finite number, so that -inf logits alone leave s = 0 and no inf - inf arises.
struct Sums {
    float m = kLowest, s = 0.f, s1 = 0.f;

    // (differences below -200 are probabilities of 0; the clamp keeps 0 (-inf) out of s1)
    __device__ __forceinline__ void rebase(float to) {
        const float dm = fmaxf(m - to, -200.f), r = __builtin_amdgcn_exp2f(dm * kLog2e);
        s1 = r * fmaf(dm, s, s1);
        s *= r;
        m = to;
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N]) {
        float g = m;
#pragma unroll
        for (int i = 0; i < N; ++i) g = fmaxf(g, v[i]);
        rebase(g);
        float t[2] = {}, t1[2] = {};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float z = v[i] - g, e = __builtin_amdgcn_exp2f(z * kLog2e);
            t[i & 1] += e;
            t1[i & 1] = fmaf(e, fmaxf(z, -200.f), t1[i & 1]);
        }
        s += t[0] + t[1];
        s1 += t1[0] + t1[1];
    }
};

constexpr int kThreads = 256;
constexpr int kCap = 1024;  // keys that the selection holds in LDS

// What a workgroup leaves of its segment of a row: d = -1 where nothing lies above -inf.
struct Part {
    float m, d, s1, pad;
};

struct Scores {
    const int64_t* tokens;
    int64_t ignore;
    int top;
    float *logprob, *entropy, *stats;
    int64_t* top_ids;
    float* top_logprobs;
};

// The scores of a row from its sums (one thread).
__device__ __forceinline__ float write_scores(const Scores& o, int64_t row, float m, float d, float s1, float xt,
                                              int64_t t, int V) {
    const bool any = 1.f + d > 0.f;  // else nothing above -inf, or NaN
    const float L = any ? log1pf(d) : __builtin_nanf("");
    o.logprob[row] = t == o.ignore ? 0.f : t < 0 || t >= V ? __builtin_nanf("") : xt - m - L;
    o.entropy[row] = L - s1 / (1.f + d);
    if (o.stats) {
        o.stats[2 * row] = m;
        o.stats[2 * row + 1] = any ? d : __builtin_nanf("");
    }
    return L;
}

// The `top` largest of the C <= kCap keys in LDS (C >= top, no two alike), each to
// its rank: key c goes where as many keys are larger.
template <typename Put>
__device__ __forceinline__ void select_keys(uint64_t* keys, int C, int top, Put put) {
    if (threadIdx.x == 0) keys[C] = 0;  // pairs below (the buffer holds kCap + 2)
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += kThreads) {
        const uint64_t mine = keys[c];
        int rank = 0;
        for (int i = 0; i < C; i += 2) {
            const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(keys + i);
            rank += (k.x > mine) + (k.y > mine);
        }
        if (rank < top) put(rank, mine);
    }
}

// One pass over a row, or over one of S segments of it (`per` vectors each): the sums
// go on with a running maximum, a thread's elements in batches of kBatch; every quad of
// threads has a maximum of its own by then, and the top-th largest of the 64 quads'
// is a bound that at least `top` logits reach. Only the threads whose own maximum
// reaches it look at their logits again (a few KB, out of L2), and so does the
// thread that holds the row's maximum, for d.
template <typename TX>
__global__ __launch_bounds__(kThreads) void scores_kernel(const TX* __restrict__ x, int64_t rows, int64_t sb, int64_t sr,
                                                          int V, int S, int per, Scores o, Part* __restrict__ parts,
                                                          uint64_t* __restrict__ part_keys) {
    constexpr int VEC = kVec<TX>;
    constexpr int B = 16 / VEC;  // vectors a batch
    __shared__ __attribute__((aligned(16))) uint64_t keys[kCap + 2];
    __shared__ float quad[64];
    __shared__ float wmax[4], wsum[4], wsum1[4], result[2];
    __shared__ int wowner[4], owners[kThreads], counts[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / (unsigned)S;
    const int seg = (int)(blockIdx.x - row * S);
    const TX* xr = x + (row / rows) * sb + (row % rows) * sr;
    // the row: `head` logits up to a 16-byte boundary, whole vectors, the rest
    const int head = min(V, (int)((16 - ((uintptr_t)xr & 15)) & 15) / (int)sizeof(TX));
    const int nvec = (V - head) / VEC, tail = V - head - nvec * VEC;
    const TX* xv = xr + head;
    const int v0 = seg * per, v1 = min(nvec, v0 + per);
    // the logit outside the vectors that thread t takes, or -1
    auto extra_of = [&](int t) {
        if (seg == 0 && t < head) return t;
        return seg == S - 1 && t >= VEC && t - VEC < tail ? V - tail + t - VEC : -1;
    };
    if (tid < 3) counts[tid] = 0;

    Sums a;
    {
        const int j = extra_of(tid);
        if (j >= 0) {
            const float v[1] = {logit(xr + j)};
            a.add(v);
        }
    }
    int v = v0 + tid;
    for (; v + kThreads * (B - 1) < v1; v += kThreads * B) {
        float t[16];
#pragma unroll
        for (int b = 0; b < B; ++b) load_vec(xv + (int64_t)(v + kThreads * b) * VEC, t + VEC * b);
        a.add(t);
    }
    for (; v < v1; v += kThreads) {
        float t[VEC];
        load_vec(xv + (int64_t)v * VEC, t);
        a.add(t);
    }

    // ---- the workgroup's sums
    const float qm = fmaxf(a.m, dpp_move<0xB1>(a.m));
    const float q4 = fmaxf(qm, dpp_move<0x4E>(qm));
    if ((tid & 3) == 0) quad[tid >> 2] = q4;
    const float wm = wave_max_dpp(a.m);
    const uint64_t at = __ballot(a.m == wm);
    if (lane == 0) wmax[wave] = wm, wowner[wave] = wave * 64 + __builtin_ctzll(at);
    __syncthreads();
    const float m = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    const int owner = wmax[0] == m ? wowner[0] : wmax[1] == m ? wowner[1] : wmax[2] == m ? wowner[2] : wowner[3];
    const float own_max = a.m;
    a.rebase(m);
    const float ws = wave_sum_dpp(tid == owner ? 0.f : a.s), ws1 = wave_sum_dpp(a.s1);
    if (lane == 0) wsum[wave] = ws, wsum1[wave] = ws1;
    // the owner's logits but one maximum (s of a thread that saw NaN is NaN already)
    float rest = 0.f;
    if (wave == 0) {
        int equal = 0;
        auto take = [&](float xj) {
            const float e = __builtin_amdgcn_exp2f((xj - m) * kLog2e);
            rest += xj == m ? xj - m : e;  // (+inf - +inf: NaN)
            equal += xj == m;
        };
        for (int w = v0 + owner + kThreads * lane; w < v1; w += kThreads * 64) {
            float t[VEC];
            load_vec(xv + (int64_t)w * VEC, t);
#pragma unroll
            for (int i = 0; i < VEC; ++i) take(t[i]);
        }
        const int j = extra_of(owner);
        if (lane == 0 && j >= 0) take(logit(xr + j));
        rest = wave_sum_dpp(rest) + (wave_sum_dpp((float)equal) - 1.f);  // nothing above -inf: -1
    }
    __syncthreads();
    const float others = (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]);
    const float s1 = (wsum1[0] + wsum1[1]) + (wsum1[2] + wsum1[3]);
    if (tid == 0) {
        const float d = others + rest;
        if (S > 1) {
            parts[blockIdx.x] = {m, d, s1, 0.f};
        } else {
            const int64_t t = o.tokens[row];
            const float xt = t >= 0 && t < V ? logit(xr + t) : 0.f;
            result[0] = write_scores(o, row, m, d, s1, xt, t, V);
        }
        result[1] = d;
    }
    const int top = o.top;
    if (!top) return;

    // ---- alternatives: the bound, and what reaches it
    float bound;
    {
        const float mine = quad[lane];
        int rank = 0;
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
            const float4 q = *reinterpret_cast<const float4*>(quad + i);
            rank += (q.x > mine || (q.x == mine && i < lane)) + (q.y > mine || (q.y == mine && i + 1 < lane)) +
                    (q.z > mine || (q.z == mine && i + 2 < lane)) + (q.w > mine || (q.w == mine && i + 3 < lane));
        }
        const uint64_t kth = __ballot(rank == top - 1);
        bound = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), __builtin_ctzll(kth)));
    }
    const bool low = bound <= kLowest;  // fewer than `top` quads saw more: every logit counts
    if (low || own_max >= bound) owners[atomicAdd(&counts[0], 1)] = tid;
    __syncthreads();
    const int nown = counts[0], slots = (max(v1 - v0, 0) + kThreads - 1) / kThreads + 1;
    const bool odd = !(result[1] == result[1]);  // NaN or +inf in the row
    auto each_again = [&](auto f) {  // f(logit, place) over the logits of the threads listed
        for (int i = tid; i < nown * slots; i += kThreads) {
            const int t = owners[i / slots], k = i % slots;
            if (k == slots - 1) {
                const int j = extra_of(t);
                if (j >= 0) f(logit(xr + j), j);
                continue;
            }
            const int w = v0 + t + kThreads * k;
            if (w >= v1) continue;
            float u[VEC];
            load_vec(xv + (int64_t)w * VEC, u);
#pragma unroll
            for (int e = 0; e < VEC; ++e) f(u[e], head + w * VEC + e);
        }
    };
    auto hold = [&](float xj, int j) {
        const int c = atomicAdd(&counts[1], 1);
        if (c < kCap) keys[c] = place_key(xj, j);
    };
    const int first = seg == 0 ? 0 : min(head + v0 * VEC, V - tail), last = seg == S - 1 ? V : head + v1 * VEC;  // the segment
    if (!odd) {
        each_again([&](float xj, int j) {
            if (low || xj >= bound) hold(xj, j);
        });
        __syncthreads();
        if (counts[1] > kCap) {
            // more ties than the buffer holds: what lies above the bound, then of
            // the equals the lowest places (and of -inf, where the bound is the
            // lowest number), a quarter of the segment a wavefront
            __syncthreads();
            if (tid == 0) counts[1] = 0;
            __syncthreads();
            each_again([&](float xj, int j) {
                if (xj > bound) hold(xj, j);
            });
            __syncthreads();
            if (counts[1] <= kCap / 2) {
                for (int pass = 0; pass < (low ? 2 : 1); ++pass) {
                    const float value = pass ? -__builtin_inff() : bound;
                    const int need = top - counts[1];
                    __syncthreads();
                    const int part = (last - first + 3) / 4, end = min(last, first + (wave + 1) * part);
                    int found = 0;
                    for (int j0 = first + wave * part; j0 < end && found < need; j0 += 512) {
                        float u[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) u[e] = logit(xr + min(j0 + 64 * e + lane, end - 1));
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int j = j0 + 64 * e + lane;
                            const bool hit = found < need && j < end && u[e] == value;
                            if (hit) hold(u[e], j);
                            found += __popcll(__ballot(hit));
                        }
                    }
                    __syncthreads();
                    if (counts[1] >= top) break;
                }
            }
        }
    }
    __syncthreads();
    int C = counts[1];
    if (odd || C > kCap) {
        // NaN among the logits, or large ones in a few threads' places only: the
        // largest key below the last, `top` times
        __syncthreads();
        uint64_t below = ~0ull;
        for (int k = 0; k < top; ++k) {
            uint64_t best = 0;
            for (int j = first + tid; j < last; j += kThreads) {
                const uint64_t c = place_key(logit(xr + j), j);
                best = c < below ? max_u64(best, c) : best;
            }
#pragma unroll
            for (int off = 32; off; off >>= 1) best = max_u64(best, __shfl_xor(best, off, 64));
            uint64_t* red = keys + kCap / 2;  // (the first `top` places hold the results)
            if (lane == 0) red[4 * (k & 1) + wave] = best;
            __syncthreads();
            red += 4 * (k & 1);
            below = max_u64(max_u64(red[0], red[1]), max_u64(red[2], red[3]));
            if (tid == 0) keys[k] = below;
        }
        C = top;
        __syncthreads();
        while (C > 0 && keys[C - 1] == 0) --C;  // a segment shorter than `top`
    }
    if (S > 1) {
        uint64_t* out = part_keys + (int64_t)blockIdx.x * top;
        for (int k = C + tid; k < top; k += kThreads) out[k] = 0;
        select_keys(keys, C, top, [&](int k, uint64_t key) { out[k] = key; });
    } else {
        const float L = result[0];
        select_keys(keys, C, top, [&](int k, uint64_t key) {
            o.top_ids[row * top + k] = (uint32_t)~(uint32_t)key;
            o.top_logprobs[row * top + k] = of_order(key >> 32) - m - L;
        });
    }
}

// The segments of a row joined (S <= kThreads, S top <= kCap).
template <typename TX>
__global__ __launch_bounds__(kThreads) void join_kernel(const TX* __restrict__ x, int64_t rows, int64_t sb, int64_t sr,
                                                        int V, int S, Scores o, const Part* __restrict__ parts,
                                                        const uint64_t* __restrict__ part_keys) {
    __shared__ __attribute__((aligned(16))) uint64_t keys[kCap + 2];
    __shared__ float wmax[4], wsum[4], wsum1[4], result[1];
    __shared__ int wowner[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const TX* xr = x + (row / rows) * sb + (row % rows) * sr;
    const int64_t t = o.tokens[row];
    const float xt = t >= 0 && t < V ? logit(xr + t) : 0.f;
    Part p = {kLowest, -1.f, 0.f, 0.f};
    if (tid < S) p = parts[row * S + tid];
    const int top = o.top;
    for (int i = tid; i < S * top; i += kThreads) keys[i] = part_keys[row * S * top + i];
    const float wm = wave_max_dpp(p.m);
    const uint64_t at = __ballot(p.m == wm);
    if (lane == 0) wmax[wave] = wm, wowner[wave] = wave * 64 + __builtin_ctzll(at);
    __syncthreads();
    const float m = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    const int owner = wmax[0] == m ? wowner[0] : wmax[1] == m ? wowner[1] : wmax[2] == m ? wowner[2] : wowner[3];
    Sums a;
    a.m = p.m;
    a.s = 1.f + p.d;
    a.s1 = p.s1;
    a.rebase(m);
    const float ws = wave_sum_dpp(tid == owner ? p.d : a.s), ws1 = wave_sum_dpp(a.s1);
    if (lane == 0) wsum[wave] = ws, wsum1[wave] = ws1;
    __syncthreads();
    if (tid == 0)
        result[0] = write_scores(o, row, m, (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]),
                                 (wsum1[0] + wsum1[1]) + (wsum1[2] + wsum1[3]), xt, t, V);
    if (!top) return;
    __syncthreads();
    const float L = result[0];
    select_keys(keys, S * top, top, [&](int k, uint64_t key) {
        o.top_ids[row * top + k] = (uint32_t)~(uint32_t)key;
        o.top_logprobs[row * top + k] = of_order(key >> 32) - m - L;
    });
}

// Segments of a row: enough workgroups for the chip where rows are few, each with a
// vector a thread at least, and as many keys as the join holds.
int segments(int dtype, int64_t rows, int64_t vocab, int top) {
    const int64_t vectors = vocab / (dtype == TIQ_F32 ? 4 : 8);
    int64_t S = std::min((vectors + kThreads - 1) / kThreads, (1024 + rows - 1) / rows);
    S = std::min<int64_t>(S, top ? kCap / top : kThreads);
    return (int)std::max<int64_t>(1, std::min<int64_t>(S, kThreads));
}

struct Grads {
    const int64_t* tokens;
    int64_t ignore;
    int top;
    const float *stats, *entropy, *g_logprob, *g_entropy;
    const int64_t* top_ids;
    const float* g_top;
};

// exp(z): fp32 rows with the argument's rounding made good (z log2e = t + r), which a
// gradient's own digits show; bf16 rows hold no such digits.
template <typename TX>
__device__ __forceinline__ float exp_of(float z) {
    const float t = z * kLog2e, e = __builtin_amdgcn_exp2f(t);
    if constexpr (sizeof(TX) == 2) return e;
    const float r = fmaf(z, 1.92596299e-8f, fmaf(z, kLog2e, -t));  // log2 e - float(log2 e)
    return t > -150.f ? fmaf(e * r, 0.693147181f, e) : e;
}

__device__ __forceinline__ void store_vec(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(v);
}
__device__ __forceinline__ void store_vec(uint16_t* p, const float* v) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7]));
}

// A read and a write of the logits: `per` vectors of a row a workgroup, aligned to the
// gradient's 16-byte boundaries (the logits' too, unless a caller's strides shift
// them). Every element as one that no token names; then the few that one does, anew.
template <typename TX>
__global__ __launch_bounds__(kThreads) void grad_kernel(const TX* __restrict__ x, int64_t rows, int64_t sb, int64_t sr,
                                                        int V, int chunks, int per, Grads o, TX* grad) {
    constexpr int VEC = kVec<TX>;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x / (unsigned)chunks;
    const int chunk = (int)(blockIdx.x - row * chunks);
    const TX* xr = x + (row / rows) * sb + (row % rows) * sr;
    TX* gr = grad + row * V;
    const int head = min(V, (int)((16 - ((uintptr_t)gr & 15)) & 15) / (int)sizeof(TX));
    const int nvec = (V - head) / VEC, tail = V - head - nvec * VEC;
    const int v0 = chunk * per, v1 = min(nvec, v0 + per);
    const float m = o.stats[2 * row], d = o.stats[2 * row + 1], s = 1.f + d, L = log1pf(d), H = o.entropy[row];
    const int64_t t = o.tokens[row];
    float gl = o.g_logprob && t != o.ignore ? o.g_logprob[row] : 0.f;
    if (o.g_logprob && t != o.ignore && (t < 0 || t >= V)) gl = __builtin_nanf("");
    const float gh = o.g_entropy ? o.g_entropy[row] : 0.f;
    float all = gl;
    if (o.g_top)
        for (int k = 0; k < o.top; ++k) all += o.g_top[row * o.top + k];
    const float c0 = fmaf(gh, H - L, all), inv = 1.f / s;
    auto plain = [&](float xj) {
        const float z = xj - m;
        return -(exp_of<TX>(z) * inv) * fmaf(gh, fmaxf(z, -200.f), c0);
    };
    // vectors through the row, `U` loads at a time
    const bool shifted = (uintptr_t)(xr + head) & 15;
    constexpr int U = 4;
    for (int v = v0 + tid; v < v1; v += kThreads * U) {
        float u[U][VEC];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const TX* src = xr + head + (int64_t)min(v + kThreads * i, v1 - 1) * VEC;
            if (!shifted) {
                load_vec(src, u[i]);
            } else {
#pragma unroll
                for (int e = 0; e < VEC; ++e) u[i][e] = logit(src + e);
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (v + kThreads * i >= v1) break;
#pragma unroll
            for (int e = 0; e < VEC; ++e) u[i][e] = plain(u[i][e]);
            store_vec(gr + head + (int64_t)(v + kThreads * i) * VEC, u[i]);
        }
    }
    if (chunk == 0) {
        const int j = tid < head ? tid : tid >= VEC && tid - VEC < tail ? V - tail + tid - VEC : -1;
        if (j >= 0) put(gr + j, plain(logit(xr + j)));
    }
    const int ids = o.g_top ? o.top : 0;
    if (!ids && (gl == 0.f || t < 0 || t >= V)) return;  // (alike in every thread)
    __syncthreads();
    if (tid > ids) return;
    int64_t j = t;
    float hot = gl;
    if (tid < ids) {
        j = o.top_ids[row * ids + tid];
        hot = o.g_top[row * ids + tid] + (j == t ? gl : 0.f);
    } else {
        for (int k = 0; k < ids; ++k)
            if (o.top_ids[row * ids + k] == t) return;
    }
    if (j < 0 || j >= V) return;
    const int home = j < head || j >= V - tail ? 0 : ((int)j - head) / VEC / per;
    if (home != chunk) return;
    const float z = logit(xr + j) - m, e = exp_of<TX>(z), p = e * inv;
    const float other = e == 1.f ? d * inv : 1.f - p;  // 1 - p
    put(gr + j, hot * other - p * fmaf(gh, fmaxf(z, -200.f) + (H - L), all - hot));
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

template <typename TX>
static int run_scores(const TX* x, int64_t count, int64_t rows, int64_t sb, int64_t sr, int V, int S, const Scores& o,
                      void* workspace, hipStream_t st) {
    const int vectors = V / kVec<TX>;
    Part* parts = static_cast<Part*>(workspace);
    uint64_t* keys = reinterpret_cast<uint64_t*>(parts + (S > 1 ? count * S : 0));
    hipLaunchKernelGGL(scores_kernel<TX>, dim3((unsigned)(count * S)), dim3(kThreads), 0, st, x, rows, sb, sr, V, S,
                       (vectors + S - 1) / S, o, parts, keys);
    if (S > 1)
        hipLaunchKernelGGL(join_kernel<TX>, dim3((unsigned)count), dim3(kThreads), 0, st, x, rows, sb, sr, V, S, o,
                           parts, keys);
    return launch_status();
}

extern "C" size_t tiq_token_logprobs_workspace(int dtype, int64_t rows, int64_t vocab, int top) {
    if (rows <= 0 || vocab <= 0 || top < 0 || top > kMaxTop || rows > 0x7fffffffLL) return 0;
    const int S = segments(dtype, rows, vocab, top);
    return S > 1 ? (size_t)rows * S * (sizeof(Part) + 8 * top) : 0;
}

extern "C" int tiq_token_logprobs(const void* logits, int dtype, int64_t batch, int64_t rows, int64_t stride_batch,
                                  int64_t stride_row, int64_t vocab, const int64_t* tokens, int64_t ignore_index,
                                  int top, float* logprob, float* entropy, float* stats, int64_t* top_ids,
                                  float* top_logprobs, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = check_rows(logits, dtype, batch, rows, vocab, tokens, top);
    if (rc != TIQ_OK || batch * rows == 0) return rc;
    if (!logprob || !entropy || (top && (!top_ids || !top_logprobs))) return TIQ_EINVAL;
    const int64_t count = batch * rows;
    const size_t need = tiq_token_logprobs_workspace(dtype, count, vocab, top);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return TIQ_EWORKSPACE;
    const int S = segments(dtype, count, vocab, top);
    const Scores o = {tokens, ignore_index, top, logprob, entropy, stats, top_ids, top_logprobs};
    if (dtype == TIQ_F32)
        return run_scores(static_cast<const float*>(logits), count, rows, stride_batch, stride_row, (int)vocab, S, o,
                          workspace, as_stream(stream));
    return run_scores(static_cast<const uint16_t*>(logits), count, rows, stride_batch, stride_row, (int)vocab, S, o,
                      workspace, as_stream(stream));
}

// Vectors a workgroup: 4 a thread, 16 where that leaves enough workgroups.
template <typename TX>
static int run_grad(const TX* x, int64_t count, int64_t rows, int64_t sb, int64_t sr, int V, const Grads& o, TX* grad,
                    hipStream_t st) {
    const int64_t vectors = std::max(1, V / kVec<TX>);
    int per = 4 * kThreads;
    int64_t chunks = (vectors + per - 1) / per;
    if (chunks * count > 0x7fffffffLL) per = (int)vectors, chunks = 1;
    hipLaunchKernelGGL(grad_kernel<TX>, dim3((unsigned)(count * chunks)), dim3(kThreads), 0, st, x, rows, sb, sr, V,
                       (int)chunks, per, o, grad);
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
    if (dtype == TIQ_F32)
        return run_grad(static_cast<const float*>(logits), batch * rows, rows, stride_batch, stride_row, (int)vocab, o,
                        static_cast<float*>(grad), as_stream(stream));
    return run_grad(static_cast<const uint16_t*>(logits), batch * rows, rows, stride_batch, stride_row, (int)vocab, o,
                    static_cast<uint16_t*>(grad), as_stream(stream));
}
