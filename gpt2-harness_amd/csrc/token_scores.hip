// Scores of given tokens under rows of logits (gfx950): log probability, entropy of
// the row, its most probable alternatives, and the gradient that these send back.
//
// With m = max_j x_j, z_j = x_j - m, e_j = exp(z_j) and
//     d = sum of e_j over all j but one that has x_j = m     (so sum e_j = 1 + d)
//     log p_j = z_j - log1p(d)
//     H       = log1p(d) - (sum_j e_j z_j) / (1 + d)
// (the reference's log_softmax in F.cross_entropy, model.py:593-598). d and not the sum
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
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;
constexpr float kFarRef = -3e38f;  // where a running maximum's ref starts
constexpr float kFarLogit = 2e38f;  // |m| from here on comes too near it

// Running maximum of some of a row's logits, the sum of 2^t and of 2^t t with t = x log2 e
// - ref. ref is the maximum times log2 e as a float, so t takes one instruction and one
// rounding; that ref is not m log2 e itself is made good once, at the end.
struct Sums {
    float m = kLowest, ref = kFarRef, s = 0.f, st = 0.f;

    // (t below -300 are probabilities of 0; the clamps keep 0 (-inf) out of st)
    __device__ __forceinline__ void rebase(float to) {
        const float next = fmaxf(to * kLog2e, kFarRef);
        const float dt = fmaxf(ref - next, -300.f), r = __builtin_amdgcn_exp2f(dt);
        st = r * fmaf(dt, s, st);
        s *= r;
        m = to;
        ref = next;
    }
    template <int N>
    __device__ __forceinline__ void add(const float (&v)[N]) {
        float g = m;
#pragma unroll
        for (int i = 0; i < N; ++i) g = fmaxf(g, v[i]);
        rebase(g);
        float a[2] = {}, b[2] = {};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = fmaf(v[i], kLog2e, -ref), e = __builtin_amdgcn_exp2f(t);
            a[i & 1] += e;
            b[i & 1] = fmaf(e, fmaxf(t, -300.f), b[i & 1]);
        }
        s += a[0] + a[1];
        st += b[0] + b[1];
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
template <int T, typename Put>
__device__ __forceinline__ void select_keys(uint64_t* keys, int C, int top, Put put) {
    if (threadIdx.x < 8) keys[C + threadIdx.x] = 0;  // eight at a time below (the buffer holds kCap + 8)
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += T) {
        const uint64_t mine = keys[c];
        int rank = 0;
        for (int i = 0; i < C; i += 8) {
            ulonglong2 k[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = *reinterpret_cast<const ulonglong2*>(keys + i + 2 * e);
#pragma unroll
            for (int e = 0; e < 4; ++e) rank += (k[e].x > mine) + (k[e].y > mine);
        }
        if (rank < top) put(rank, mine);
    }
}

// A key for the selection; past the buffer's end only counted.
__device__ __forceinline__ void hold(uint64_t* keys, int* count, float xj, int j) {
    const int c = atomicAdd(count, 1);
    if (c < kCap) keys[c] = place_key(xj, j);
}

// The top-th largest of 64 numbers in LDS, in every lane (any of them where one is NaN).
__device__ __forceinline__ float kth_of_64(const float* q, int top) {
    const int lane = threadIdx.x & 63;
    const float mine = q[lane];
    int rank = 0;
#pragma unroll
    for (int i = 0; i < 64; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(q + i);
        rank += (v.x > mine || (v.x == mine && i < lane)) + (v.y > mine || (v.y == mine && i + 1 < lane)) +
                (v.z > mine || (v.z == mine && i + 2 < lane)) + (v.w > mine || (v.w == mine && i + 3 < lane));
    }
    const uint64_t kth = __ballot(rank == top - 1);
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), kth ? __builtin_ctzll(kth) : 0));
}

// With every logit above `bound` of places first .. last - 1 held: of those equal to it
// the lowest places, up to `top` keys in all (`low`: the bound is the lowest number, and
// of -inf next). Each wavefront takes a part of the places in their order and stops
// when it has found enough.
template <int T, typename TX>
__device__ __forceinline__ void hold_ties(uint64_t* keys, int* count, const TX* xr, int first, int last, float bound,
                                          bool low, int top) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, W = T / 64;
    for (int pass = 0; pass < (low ? 2 : 1); ++pass) {
        const float value = pass ? -__builtin_inff() : bound;
        const int need = top - *count;
        __syncthreads();
        const int part = (last - first + W - 1) / W, end = min(last, first + (wave + 1) * part);
        int found = 0;
        for (int j0 = first + wave * part; j0 < end && found < need; j0 += 512) {
            float u[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] = logit(xr + min(j0 + 64 * e + lane, end - 1));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int j = j0 + 64 * e + lane;
                const bool hit = found < need && j < end && u[e] == value;
                const uint64_t hits = __ballot(hit);
                // (no more than `need` a wavefront: the first of them are the lowest)
                if (hit && found + __popcll(hits & ((1ull << lane) - 1)) < need) hold(keys, count, u[e], j);
                found += __popcll(hits);
            }
        }
        __syncthreads();
        if (*count >= top) break;
    }
}

// The `top` largest keys of places first .. last - 1 without a bound: the largest below
// the last one, `top` times. Returns how many there are.
template <int T, typename TX>
__device__ __forceinline__ int slow_keys(uint64_t* keys, const TX* xr, int first, int last, int top) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t* red = keys + kCap / 2;  // (the first `top` places hold the results)
    uint64_t below = ~0ull;
    __syncthreads();
    int C = 0;
    for (; C < top; ++C) {
        uint64_t best = 0;
        for (int j = first + (int)threadIdx.x; j < last; j += T) {
            const uint64_t c = place_key(logit(xr + j), j);
            best = c < below ? max_u64(best, c) : best;
        }
#pragma unroll
        for (int off = 32; off; off >>= 1) best = max_u64(best, __shfl_xor(best, off, 64));
        uint64_t* r = red + 16 * (C & 1);
        if (lane == 0) r[wave] = best;
        __syncthreads();
        below = 0;
#pragma unroll
        for (int w = 0; w < T / 64; ++w) below = max_u64(below, r[w]);
        if (!below) break;  // a segment shorter than `top`
        if (threadIdx.x == 0) keys[C] = below;
    }
    __syncthreads();
    return C;
}

// Row (b, r) of the logits, counted through (at most 2^31 - 1 of them).
template <typename TX>
__device__ __forceinline__ const TX* row_at(const TX* x, int64_t row, int64_t rows, int64_t sb, int64_t sr) {
    const unsigned b = (unsigned)row / (unsigned)rows, r = (unsigned)row - b * (unsigned)rows;
    return x + (int64_t)b * sb + (int64_t)r * sr;
}

// Where a row lies: logits up to a 16-byte boundary, whole vectors, the rest.
template <typename TX>
struct Row {
    const TX* x;
    int head, nvec, tail, V;
    __device__ __forceinline__ Row(const TX* x_, int V_) : x(x_), V(V_) {
        head = min(V, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(TX));
        nvec = (V - head) / kVec<TX>;
        tail = V - head - nvec * kVec<TX>;
    }
    __device__ __forceinline__ const TX* vec(int v) const { return x + head + (int64_t)v * kVec<TX>; }
    // the logit outside the vectors that thread t takes, or -1
    __device__ __forceinline__ int extra(int t, bool is_first, bool is_last) const {
        if (is_first && t < head) return t;
        return is_last && t >= kVec<TX> && t - kVec<TX> < tail ? V - tail + t - kVec<TX> : -1;
    }
};

// A row, or one of S segments of it (`per` vectors each), in one pass: the sums go on
// with a running maximum, a thread's logits in batches of B vectors. Each of 64 groups of
// threads has a maximum of its own by then, and the top-th largest of the 64 is a bound
// that at least `top` logits reach. Only the threads whose own maximum reaches it look
// at their logits again (a few KB, out of the cache), and so does the thread that holds
// the row's maximum, for d. ONE: a batch a thread is the whole of it, and the logits
// are looked at again in the registers.
// What bounds it: memory where the rows fill the chip (4096 x 50257 fp32 with 5
// alternatives 143 us, 5.7 TB/s; bf16 69 us, 6.0 TB/s: 9.6 vector instructions a logit, 54%
// of their units' time, so neither exps nor the second look show), and the chain of a
// launch, the vector units of the row's one CU, two barriers and the selection where they
// are few (one row of 50257: 9.5 us in a graph, 7.4 without alternatives; as long with half the
// bytes in bf16, and no shorter with 1024 threads, 10.7, or batches of 8 vectors, 9.6).
template <typename TX, int T, int B, bool ONE>
__global__ __launch_bounds__(T) void scores_kernel(const TX* __restrict__ x, int64_t row0, int64_t rows, int64_t sb,
                                                   int64_t sr, int V, int S, int per, Scores o, Part* __restrict__ parts,
                                                   uint64_t* __restrict__ part_keys) {
    constexpr int VEC = kVec<TX>, W = T / 64;
    __shared__ __attribute__((aligned(16))) uint64_t keys[kCap + 8];
    __shared__ __attribute__((aligned(16))) float group[64];
    __shared__ float wmax[W], wsum[W], wsum1[W], result[2];
    __shared__ int wowner[W], owners[ONE ? 1 : T], listed[1], count[1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const unsigned r0 = blockIdx.x / (unsigned)S;
    const int64_t row = row0 + r0;
    const int seg = (int)(blockIdx.x - r0 * S);
    const Row<TX> r(row_at(x, row, rows, sb, sr), V);
    const int v0 = seg * per, v1 = min(r.nvec, v0 + per);
    auto extra_of = [&](int t) { return r.extra(t, seg == 0, seg == S - 1); };
    if (tid == 0) listed[0] = count[0] = 0;
    // the row's token and its logit, two trips to memory, beside the logits' first
    int64_t token = 0;
    float xt = 0.f;
    if (S == 1 && tid == 0) {
        token = o.tokens[row];
        if (token >= 0 && token < V) xt = logit(r.x + token);
    }

    Sums a;
    int v = v0 + tid;
    if constexpr (!ONE) {
        for (; v + T * (B - 1) < v1; v += T * B) {
            uint4 raw[B];
#pragma unroll
            for (int b = 0; b < B; ++b) raw[b] = *reinterpret_cast<const uint4*>(r.vec(v + T * b));
            float t[VEC * B];
#pragma unroll
            for (int b = 0; b < B; ++b) load_vec(reinterpret_cast<const TX*>(&raw[b]), t + VEC * b);
            a.add(t);
        }
    }
    // the last batch, and the logits outside the vectors
    const int je = extra_of(tid);
    float u[VEC * B + 1];
    {
        constexpr uint32_t none = sizeof(TX) == 4 ? 0xff800000u : 0xff80ff80u;  // -inf
        uint4 raw[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            raw[b] = make_uint4(none, none, none, none);
            if (v + T * b < v1) raw[b] = *reinterpret_cast<const uint4*>(r.vec(v + T * b));
        }
        u[VEC * B] = je >= 0 ? logit(r.x + je) : -__builtin_inff();
#pragma unroll
        for (int b = 0; b < B; ++b) load_vec(reinterpret_cast<const TX*>(&raw[b]), u + VEC * b);
    }
    if constexpr (ONE) {
        a.add(u);
    } else {  // (wavefronts past the end leave vectors out)
#pragma unroll
        for (int b = 0; b < B; ++b) {
            if (v + T * b < v1) {
                float t[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) t[i] = u[VEC * b + i];
                a.add(t);
            }
        }
        if (je >= 0) {
            const float t[1] = {u[VEC * B]};
            a.add(t);
        }
    }

    // ---- the workgroup's sums
    const int top = o.top;
    if (top) {
        float q = a.m;
        if constexpr (W >= 2) q = fmaxf(q, dpp_move<0xB1>(q));
        if constexpr (W >= 4) q = fmaxf(q, dpp_move<0x4E>(q));
        if constexpr (W >= 8) q = fmaxf(q, dpp_move<0x141>(q));
        if constexpr (W >= 16) q = fmaxf(q, dpp_move<0x140>(q));
        if (tid % W == 0) group[tid / W] = q;
    }
    const float wm = wave_max_dpp(a.m);
    const uint64_t at = __ballot(a.m == wm);
    if (lane == 0) wmax[wave] = wm, wowner[wave] = wave * 64 + (at ? __builtin_ctzll(at) : 0);
    __syncthreads();
    float m = wmax[W - 1];
    int owner = wowner[W - 1];
#pragma unroll
    for (int w = W - 2; w >= 0; --w) {
        owner = wmax[w] >= m ? wowner[w] : owner;
        m = fmaxf(m, wmax[w]);
    }
    const float own_max = a.m;
    a.rebase(m);
    const float shift = fmaf(m, kLog2e, -a.ref), back = __builtin_amdgcn_exp2f(-shift);  // exp(x - m) = 2^t back
    const bool far = !(fabsf(m) < kFarLogit);  // a maximum that is infinite, or as low as a mask's
    // sums of e and e z; the owner's take its logits once more, without one maximum,
    // whose 1 would swallow what a sure row's others add
    float mine = tid == owner ? 0.f : a.s * back;
    float s1 = tid == owner ? 0.f : kLn2 * back * fmaf(-shift, a.s, a.st);
    float own = 0.f;
    int equal = 0;
    auto but_equal = [&](float xj) {  // e of a logit, but of those at the maximum, which are counted
        const float z = xj - m, e = xj == m ? z : __builtin_amdgcn_exp2f(z * kLog2e);  // (+inf - +inf: NaN)
        equal += xj == m;
        s1 = fmaf(e, fmaxf(z, -200.f), s1);
        return e;
    };
    if (far) {
        mine = s1 = 0.f;
        for (int w = v0 + tid; w < v1; w += T) {
            float t[VEC];
            load_vec(r.vec(w), t);
#pragma unroll
            for (int i = 0; i < VEC; ++i) mine += but_equal(t[i]);
        }
        if (je >= 0) mine += but_equal(u[VEC * B]);
        own = (float)equal - (tid == 0 ? 1.f : 0.f);  // nothing above -inf: -1
    } else if constexpr (ONE) {
        if (wave == owner >> 6) {
            const float others = s1;
#pragma unroll
            for (int i = 0; i < VEC * B + 1; ++i) own += but_equal(u[i]);
            own = tid == owner ? own + (float)(equal - 1) : 0.f;
            s1 = tid == owner ? s1 : others;
        }
    } else if (wave == 0) {
        for (int w = v0 + owner + T * lane; w < v1; w += T * 64) {
            float t[VEC];
            load_vec(r.vec(w), t);
#pragma unroll
            for (int i = 0; i < VEC; ++i) own += but_equal(t[i]);
        }
        const int j = extra_of(owner);
        if (lane == 0 && j >= 0) own += but_equal(logit(r.x + j));
        own = wave_sum_dpp(own) + (wave_sum_dpp((float)equal) - 1.f);
        own = lane == 0 ? own : 0.f;
    }
    const float ws = wave_sum_dpp(mine + own), ws1 = wave_sum_dpp(s1);
    if (lane == 0) wsum[wave] = ws, wsum1[wave] = ws1;
    // ---- alternatives: the bound, and the threads that reach it
    const float bound = top ? kth_of_64(group, top) : 0.f;
    const bool low = bound <= kLowest;  // fewer than `top` groups saw more: every logit counts
    const int first = seg == 0 ? 0 : min(r.head + v0 * VEC, V - r.tail), last = seg == S - 1 ? V : r.head + v1 * VEC;
    // ONE: the keys of a thread's own logits that a test takes
    auto hold_own = [&](auto takes) {
        uint64_t hits = 0;
#pragma unroll
        for (int i = 0; i < VEC * B + 1; ++i) hits |= (uint64_t)takes(u[i]) << i;
        if (je < 0) hits &= ~(1ull << VEC * B);
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (v + T * b >= v1) hits &= ~(((1ull << VEC) - 1) << VEC * b);
        while (hits) {
            const int i = __builtin_ctzll(hits);
            hits &= hits - 1;
            const int j = i == VEC * B ? je : r.head + (v + T * (i / VEC)) * VEC + i % VEC;
            hold(keys, count, logit(r.x + j), j);
        }
    };
    if (top) {
        if constexpr (ONE) {
            if (low || own_max >= bound) hold_own([&](float xj) { return low || xj >= bound; });
        } else {
            if (low || own_max >= bound) owners[atomicAdd(&listed[0], 1)] = tid;
        }
    }
    __syncthreads();
    if (tid == 0) {
        float d = 0.f, s1 = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) d += wsum[w], s1 += wsum1[w];
        if (S > 1) {
            parts[blockIdx.x] = {m, d, s1, 0.f};
        } else {
            result[0] = write_scores(o, row, m, d, s1, xt, token, V);
        }
        result[1] = d;
    }
    if (!top) return;
    const int nown = ONE ? 0 : listed[0], slots = (max(v1 - v0, 0) + T - 1) / T + 1;
    auto each_again = [&](auto f) {  // f(logit, place) over the logits of the threads listed
        for (int i = tid; i < nown * slots; i += T) {
            const int t = owners[i / slots], k = i % slots;
            if (k == slots - 1) {
                const int j = extra_of(t);
                if (j >= 0) f(logit(r.x + j), j);
                continue;
            }
            const int w = v0 + t + T * k;
            if (w >= v1) continue;
            float t8[VEC];
            load_vec(r.vec(w), t8);
#pragma unroll
            for (int e = 0; e < VEC; ++e) f(t8[e], r.head + w * VEC + e);
        }
    };
    if constexpr (!ONE) {
        each_again([&](float xj, int j) {
            if (low || xj >= bound) hold(keys, count, xj, j);
        });
    }
    __syncthreads();
    const bool odd = !(result[1] == result[1]);  // NaN or +inf in the row
    if (!odd && count[0] > kCap) {  // more ties than the buffer holds
        __syncthreads();
        if (tid == 0) count[0] = 0;
        __syncthreads();
        if constexpr (ONE) hold_own([&](float xj) { return xj > bound; });
        else each_again([&](float xj, int j) {
            if (xj > bound) hold(keys, count, xj, j);
        });
        __syncthreads();
        if (count[0] <= kCap / 2) hold_ties<T>(keys, count, r.x, first, last, bound, low, top);
    }
    int C = count[0];
    if (odd || C > kCap) C = slow_keys<T>(keys, r.x, first, last, top);
    if (S > 1) {
        uint64_t* out = part_keys + (int64_t)blockIdx.x * top;
        for (int k = C + tid; k < top; k += T) out[k] = 0;
        select_keys<T>(keys, C, top, [&](int k, uint64_t key) { out[k] = key; });
    } else {
        const float L = result[0];
        select_keys<T>(keys, C, top, [&](int k, uint64_t key) {
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
    __shared__ __attribute__((aligned(16))) uint64_t keys[kCap + 8];
    __shared__ float wmax[4], wsum[4], wsum1[4], result[1];
    __shared__ int wowner[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x;
    const TX* xr = row_at(x, row, rows, sb, sr);
    const int64_t t = o.tokens[row];
    const float xt = t >= 0 && t < V ? logit(xr + t) : 0.f;
    Part p = {kLowest, -1.f, 0.f, 0.f};
    if (tid < S) p = parts[row * S + tid];
    const int top = o.top;
    for (int i = tid; i < S * top; i += kThreads) keys[i] = part_keys[row * S * top + i];
    const float wm = wave_max_dpp(p.m);
    const uint64_t at = __ballot(p.m == wm);
    if (lane == 0) wmax[wave] = wm, wowner[wave] = wave * 64 + (at ? __builtin_ctzll(at) : 0);
    __syncthreads();
    const float m = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    const int owner = wmax[0] == m ? wowner[0] : wmax[1] == m ? wowner[1] : wmax[2] == m ? wowner[2] : wowner[3];
    // exp(p.m - m); segments that hold no more than the row's maximum keep NaN of theirs
    const float z = fmaxf(p.m - m, -200.f), e = __builtin_amdgcn_exp2f(z * kLog2e);
    const float ws = wave_sum_dpp(tid == owner ? p.d : (1.f + p.d) * e);
    const float ws1 = wave_sum_dpp(e * fmaf(z, 1.f + p.d, p.s1));
    if (lane == 0) wsum[wave] = ws, wsum1[wave] = ws1;
    __syncthreads();
    if (tid == 0)
        result[0] = write_scores(o, row, m, (wsum[0] + wsum[1]) + (wsum[2] + wsum[3]),
                                 (wsum1[0] + wsum1[1]) + (wsum1[2] + wsum1[3]), xt, t, V);
    if (!top) return;
    __syncthreads();
    const float L = result[0];
    select_keys<kThreads>(keys, S * top, top, [&](int k, uint64_t key) {
        o.top_ids[row * top + k] = (uint32_t)~(uint32_t)key;
        o.top_logprobs[row * top + k] = of_order(key >> 32) - m - L;
    });
}

// How rows of n vectors are taken. Up to 256 vectors, a wavefront a row; up to 1024, a
// workgroup of 256 with a batch a thread (5000 rows of 1003 bf16: 8.6 us against 15 with
// 256 threads a row); longer ones, 512 threads (4096 rows of 50257 fp32, 256 / 512 / 1024
// threads: 152 / 143 / 141 us; bf16 112 / 103 / 109). Only few and long rows are cut into
// segments, which a second launch joins: about 1024 workgroups, no more segments than keep
// the join's keys few (64 rows of 131071 with 20 alternatives, in 8 / 16: the join 3.9 /
// 7.5 us). Whole / cut, in a graph with 5 alternatives: one row of 50257 fp32 9.4 / 9.3 (an
// eager call 13.7 / 18.3, for the host's second launch), 131071 13.8 / 10.0, 262147 21.6 /
// 11.0; 256 rows of 131071 29.1 / 36.5.
struct Plan {
    int T, B;  // threads, vectors a batch
    bool one;  // a batch a thread
    int S, per;
};
Plan plan_of(int dtype, int64_t rows, int64_t vocab, int top) {
    const int64_t n = std::max<int64_t>(1, vocab / (dtype == TIQ_F32 ? 4 : 8));
    if (n <= 256) return {64, n <= 64 ? 1 : n <= 128 ? 2 : 4, true, 1, (int)n};
    if (n <= 1024) return {256, 4, true, 1, (int)n};
    if (n <= 16384 || rows >= 128) return {512, 4, false, 1, (int)n};
    int64_t S = std::min((n + 1023) / 1024, (1024 + rows - 1) / rows);
    S = std::min<int64_t>(S, top ? std::max(4, 160 / top) : kThreads);
    const int per = (int)((n + S - 1) / S);
    return {256, 4, per <= 1024, (int)S, per};
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

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4 packed(const float (&v)[4]) {
    return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
__device__ __forceinline__ u32x4 packed(const float (&v)[8]) {
    return u32x4{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3]), pk_bf16(v[4], v[5]), pk_bf16(v[6], v[7])};
}

// A read and a write of the logits: `per` vectors of a row a workgroup, aligned to the
// gradient's 16-byte boundaries (the logits' too, unless a caller's strides shift
// them). Every element as one that no token names; then the few that one does, anew.
// The last rows go first: they are what the scores' pass left in the 256 MB cache before
// memory; and a gradient that would not stay there (PAST) is stored past it, which
// spares whatever reads next the wait for its write-back. 4096 rows of 50257 bf16, the
// scores' pass and this one, again and again: 105 + 141 us; from the last row 98 + 136;
// past the cache too 69 + 136.
template <typename TX, bool PAST>
__global__ __launch_bounds__(kThreads) void grad_kernel(const TX* __restrict__ x, int64_t row0, int64_t rows, int64_t sb,
                                                        int64_t sr, int V, int chunks, int per, Grads o, TX* grad) {
    constexpr int VEC = kVec<TX>;
    const int tid = threadIdx.x;
    const unsigned id = gridDim.x - 1 - blockIdx.x;  // the last rows first
    const int64_t row = row0 + id / (unsigned)chunks;
    const int chunk = (int)(id % (unsigned)chunks);
    const TX* xr = row_at(x, row, rows, sb, sr);
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
            u32x4* dst = reinterpret_cast<u32x4*>(gr + head + (int64_t)(v + kThreads * i) * VEC);
            if constexpr (PAST) __builtin_nontemporal_store(packed(u[i]), dst);
            else *dst = packed(u[i]);
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

// Rows a launch: its threads are counted in 32 bits.
constexpr int64_t kLaunchRows = 1 << 22;

template <typename TX>
static int run_scores(const TX* x, int64_t count, int64_t rows, int64_t sb, int64_t sr, int V, const Plan& p,
                      const Scores& o, void* workspace, hipStream_t st) {
    Part* parts = static_cast<Part*>(workspace);
    uint64_t* keys = reinterpret_cast<uint64_t*>(parts + (p.S > 1 ? count * p.S : 0));
    for (int64_t r0 = 0; r0 < count; r0 += kLaunchRows) {  // (cut rows are few: one launch)
        const unsigned groups = (unsigned)(std::min(count - r0, kLaunchRows) * p.S);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(groups), dim3(p.T), 0, st, x, r0, rows, sb, sr, V, p.S, p.per, o, parts, keys);
        };
        if (p.T == 512) go(scores_kernel<TX, 512, 4, false>);
        else if (p.T == 256 && p.one) go(scores_kernel<TX, 256, 4, true>);
        else if (p.T == 256) go(scores_kernel<TX, 256, 4, false>);
        else if (p.B == 1) go(scores_kernel<TX, 64, 1, true>);
        else if (p.B == 2) go(scores_kernel<TX, 64, 2, true>);
        else go(scores_kernel<TX, 64, 4, true>);
        const int rc = launch_status();
        if (rc != TIQ_OK) return rc;
    }
    if (p.S > 1)
        hipLaunchKernelGGL(join_kernel<TX>, dim3((unsigned)count), dim3(kThreads), 0, st, x, rows, sb, sr, V, p.S, o,
                           parts, keys);
    return launch_status();
}

extern "C" size_t tiq_token_logprobs_workspace(int dtype, int64_t rows, int64_t vocab, int top) {
    if (rows <= 0 || vocab <= 0 || top < 0 || top > kMaxTop || rows > 0x7fffffffLL) return 0;
    const int S = plan_of(dtype, rows, vocab, top).S;
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
    const Plan p = plan_of(dtype, count, vocab, top);
    const Scores o = {tokens, ignore_index, top, logprob, entropy, stats, top_ids, top_logprobs};
    if (dtype == TIQ_F32)
        return run_scores(static_cast<const float*>(logits), count, rows, stride_batch, stride_row, (int)vocab, p, o,
                          workspace, as_stream(stream));
    return run_scores(static_cast<const uint16_t*>(logits), count, rows, stride_batch, stride_row, (int)vocab, p, o,
                      workspace, as_stream(stream));
}

// Four vectors a thread. The launches go from the last rows to the first, as each of them does.
template <typename TX>
static int run_grad(const TX* x, int64_t count, int64_t rows, int64_t sb, int64_t sr, int V, const Grads& o, TX* grad,
                    hipStream_t st) {
    const int64_t vectors = std::max(1, V / kVec<TX>);
    int per = 4 * kThreads;
    int64_t chunks = (vectors + per - 1) / per;
    const int64_t part = std::max<int64_t>(1, std::min(kLaunchRows, kLaunchRows / chunks));
    // logits and gradient together beyond the cache's 256 MB
    const bool past = count * V * (int64_t)sizeof(TX) > (128 << 20);
    for (int64_t r0 = (count - 1) / part * part; r0 >= 0; r0 -= part) {
        const int64_t n = std::min(count - r0, part);
        hipLaunchKernelGGL((past ? grad_kernel<TX, true> : grad_kernel<TX, false>), dim3((unsigned)(n * chunks)),
                           dim3(kThreads), 0, st, x, r0, rows, sb, sr, V, (int)chunks, per, o, grad);
        const int rc = launch_status();
        if (rc != TIQ_OK) return rc;
    }
    return TIQ_OK;
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
