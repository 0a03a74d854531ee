// Linear on int8 activations and int8 weights (gfx950): the tokens' rows are
// quantized when they arrive, one scale a row, and meet the weight's codes in
// an integer product:
//     y[m, n] = (sum_k qx[m, k] qw[n, k]) sx[m] sw[n] + bias[n].
// sx and qx are quantize_tensor's per-row scale and codes at 8 bits
// (quantization.py:78-116) of the fp32 or bf16 row. The sum is exact: |qx| <= 127,
// |qw| <= 128 and K <= kMaxK keep it below 2^31. It becomes a float once and
// takes sx, then sw and the bias in one fused step: three roundings to fp32 (and
// one more to bf16 outputs) an output.
//
// Both operands lie in 1 KB tiles of 32 rows x 32 columns, the order in which the
// matrix cores take them: byte 16 l + j of tile (t, u) is row 32 t + l % 32,
// column 32 u + 16 (l / 32) + j. Columns are padded with zeros to whole pairs of
// tiles and weight rows to whole tiles, so odd sizes cost no other path; token
// rows past M are whatever the workspace holds (their outputs are not stored).
#include <algorithm>

#include "tiq_internal.hpp"

namespace tiq {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// 2^31 / (127 128), rounded down to whole tiles
constexpr int64_t kMaxK = 131072;

int64_t units_of(int64_t K) { return (K + 63) / 64 * 2; }
int64_t tiles_of(int64_t rows) { return (rows + 31) / 32; }

// Place of column k of row r in the tiles.
__device__ __forceinline__ int64_t tile_byte(int64_t r, int64_t k, int64_t U) {
    return ((r >> 5) * U + (k >> 5)) * 1024 + ((k >> 4) & 1) * 512 + (r & 31) * 16 + (k & 15);
}

__device__ __forceinline__ float load_x(const float* p) { return *p; }
__device__ __forceinline__ float load_x(const uint16_t* p) { return bf16_bits_to_f32(*p); }

// A row a workgroup, read twice. TILES: the codes in tiles of U units a row (the
// padding columns zero), else row-major.
template <bool TILES, typename TX>
__global__ __launch_bounds__(256) void tokens_generic(const TX* __restrict__ x, int64_t ldx, int64_t K,
                                                      int8_t* __restrict__ q, int64_t ldq, int64_t U,
                                                      float* __restrict__ scale) {
    __shared__ uint32_t red[4];
    const int64_t row = blockIdx.x;
    const TX* xr = x + row * ldx;
    uint32_t m = 0;
    for (int64_t c = threadIdx.x; c < K; c += 256) m = max(m, abs_bits(load_x(xr + c)));
    m = wave_max_u32(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    m = max(max(red[0], red[1]), max(red[2], red[3]));
    const float s = scale_from_amax(__uint_as_float(m), 127.f);
    if (threadIdx.x == 0) scale[row] = s;
    const int64_t end = TILES ? 32 * U : K;
    for (int64_t c = threadIdx.x; c < end; c += 256) {
        const float v = c < K ? load_x(xr + c) : 0.f;
        const float t = __builtin_rintf(v / s);
        const int code = t != t ? 0 : (int)fminf(fmaxf(t, -128.f), 127.f);
        q[TILES ? tile_byte(row, c, U) : row * ldq + c] = (int8_t)code;
    }
}

// 16 bytes of a row at any alignment of its elements.
struct __attribute__((packed, aligned(4))) Bytes16F {
    float v[4];
};
struct __attribute__((packed, aligned(2))) Bytes16H {
    uint16_t v[8];
};
__device__ __forceinline__ void load_16(const float* p, float (&v)[4]) {
    const Bytes16F t = *reinterpret_cast<const Bytes16F*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = t.v[i];
}
__device__ __forceinline__ void load_16(const uint16_t* p, float (&v)[8]) {
    const Bytes16H t = *reinterpret_cast<const Bytes16H*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf16_bits_to_f32(t.v[i]);
}

// What is applied to a row before it is quantized.
enum Before { kAsIs, kLayerNorm, kGelu };
struct LnArgs {
    const float *w, *b;
    float eps;
};

// Sum over each 16-lane row of the wavefront, in every lane of the row.
__device__ __forceinline__ float row16_sum(float v) {
    v += dpp_move<0xB1>(v);
    v += dpp_move<0x4E>(v);
    v += dpp_move<0x141>(v);
    return v + dpp_move<0x140>(v);
}

// Four rows a workgroup, held in registers: 16 lanes of each wavefront on every row, so a
// load instruction reads 256 consecutive bytes of each and a store covers 64-byte pieces
// of the tiles. IT passes of TH / 4 lanes x 16 bytes a row; K >= 16 bytes of elements. A
// LayerNorm (mean and biased variance in two passes over the registers, as torch) or a
// GELU before costs no pass over memory. 8192 x 6400 fp32 rows: 50 us, 5.2 TB/s.
template <bool TILES, int IT, int TH, Before PRE, typename TX>
__global__ __launch_bounds__(TH) void tokens_kernel(const TX* __restrict__ x, int64_t ldx, int M, int K,
                                                    int8_t* __restrict__ q, int64_t ldq, int64_t U,
                                                    float* __restrict__ scale, LnArgs ln) {
    constexpr int VEC = 16 / (int)sizeof(TX), W = TH / 64, STEP = TH / 4 * VEC;
    __shared__ uint32_t red[W][4];
    __shared__ float sums[PRE == kLayerNorm ? 2 : 1][W][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * 4 + (lane >> 4);
    const int c0 = (wave * 16 + (lane & 15)) * VEC;
    const TX* xr = x + min(row, (int64_t)M - 1) * ldx;
    float v[IT][VEC];
#pragma unroll
    for (int i = 0; i < IT; ++i) load_16(xr + min(c0 + STEP * i, K - VEC), v[i]);
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = c0 + STEP * i;
        if (c > K - VEC) {  // past the row's last whole piece: its elements one by one
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i][e] = c + e < K ? load_x(xr + c + e) : 0.f;
        }
    }
    if constexpr (PRE == kLayerNorm) {
        auto row_sum = [&](float t, int slot) {
            t = row16_sum(t);
            if ((lane & 15) == 0) sums[slot][wave][lane >> 4] = t;
            __syncthreads();
            t = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) t += sums[slot][w][lane >> 4];
            return t;
        };
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) t += v[i][e];
        const float mu = row_sum(t, 0) / (float)K;
        t = 0.f;
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) t = c0 + STEP * i + e < K ? fmaf(v[i][e] - mu, v[i][e] - mu, t) : t;
        const float rstd = 1.0f / sqrtf(row_sum(t, 1) / (float)K + ln.eps);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            const int c = c0 + STEP * i;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int k = min(c + e, K - 1);
                v[i][e] = c + e < K ? fmaf((v[i][e] - mu) * rstd, ln.w[k], ln.b[k]) : 0.f;
            }
        }
    }
    if constexpr (PRE == kGelu) {
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i][e] = gelu_tanh(v[i][e]);
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) m = umax(m, abs_bits(v[i][e]));
    m = row16_max_u32(m);
    if ((lane & 15) == 0) red[wave][lane >> 4] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) m = umax(m, red[w][lane >> 4]);
    if (row >= M) return;
    const float s = scale_from_amax(__uint_as_float(m), 127.f), inv = 1.0f / s;
    if (c0 == 0) scale[row] = s;
    const int end = TILES ? (int)(32 * U) : K;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
        const int c = c0 + STEP * i;
        if (c >= end) break;
        uint32_t w[VEC / 4];
#pragma unroll
        for (int g = 0; g < VEC / 4; ++g) {
            int k[4];
            codes4(make_float4(v[i][4 * g], v[i][4 * g + 1], v[i][4 * g + 2], v[i][4 * g + 3]), s, inv, -128, 127, k);
            w[g] = (uint32_t)(k[0] & 0xff) | (uint32_t)(k[1] & 0xff) << 8 | (uint32_t)(k[2] & 0xff) << 16 |
                   (uint32_t)(k[3] & 0xff) << 24;
        }
        int8_t* dst = q + (TILES ? tile_byte(row, c, U) : row * ldq + c);
        if (TILES || (c + VEC <= K && ((uintptr_t)dst & 3) == 0)) {
            if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(dst) = w[0];
            else if constexpr (TILES) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
            else reinterpret_cast<uint32_t*>(dst)[0] = w[0], reinterpret_cast<uint32_t*>(dst)[1] = w[1];
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (c + e < K) dst[e] = (int8_t)(w[e >> 2] >> 8 * (e & 3));
        }
    }
}

// Weight codes (N, K) -> tiles, 16 bytes of them a thread at a time.
__global__ __launch_bounds__(256) void tile_weight_kernel(const int8_t* __restrict__ w, int64_t N, int64_t K,
                                                          int64_t ldw, int64_t U, int64_t chunks,
                                                          int8_t* __restrict__ tiles) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * 256) {
        const int64_t b = i >> 6, t = b / U, u = b - t * U;
        const int l = (int)(i & 63);
        const int64_t n = 32 * t + (l & 31), k = 32 * u + 16 * (l >> 5);
        int8_t c[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) c[j] = n < N && k + j < K ? w[n * ldw + k + j] : (int8_t)0;
        int4 v;
        __builtin_memcpy(&v, c, 16);
        *reinterpret_cast<int4*>(tiles + i * 16) = v;
    }
}

// Tiles -> codes (N, K), a code a thread at a time.
__global__ __launch_bounds__(256) void untile_weight_kernel(const int8_t* __restrict__ tiles, int64_t K, int64_t U,
                                                            int64_t count, int8_t* __restrict__ w) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256)
        w[i] = tiles[tile_byte(i / K, i % K, U)];
}

__device__ __forceinline__ void store_y(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_y(uint16_t* p, float v) { *p = f32_to_bf16_bits(v); }

__device__ __forceinline__ float finish(int sum, float sx, float sw, float b) {
    return fmaf((float)sum * sx, sw, b);
}

// Added to an output last (fp32 outputs): element (m, n) at res + m ldr + n; null: nothing.
struct Residual {
    const float* res = nullptr;
    int64_t ldr = 0;
    __device__ __forceinline__ float operator()(float v, int64_t m, int n) const {
        return res ? v + res[m * ldr + n] : v;
    }
};

// Scales and codes in LDS of a product's rows (few of them: rows_fused): the W wavefronts
// share a row where there are more of them than rows, else take rows in turn. Row m's
// codes lie at m * end, zero from K on.
constexpr int kSmallRows = 16, kFusedBytes = 32768;
template <int W, typename TX>
__device__ __forceinline__ void quantize_rows(const TX* __restrict__ x, int64_t ldx, int M, int K, int end,
                                              int8_t* __restrict__ codes, float* __restrict__ scale,
                                              uint32_t* __restrict__ red) {
    constexpr int VEC = 16 / (int)sizeof(TX);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per = M <= 1 ? W : M <= 2 ? W / 2 : M <= 4 ? W / 4 : M <= 8 ? W / 8 : max(1, W / 16);  // wavefronts a row
    const int c0 = ((wave % per) * 64 + lane) * VEC, step = per * 64 * VEC;
    for (int row = wave / per; row < kSmallRows; row += W / per) {
        if (row - wave / per >= M) break;  // (alike in every wavefront: no row left for any)
        const TX* xr = x + (int64_t)min(row, M - 1) * ldx;
        // `f` over the row's 16-byte pieces, past its end zeros
        auto pieces = [&](auto f) {
            for (int c = c0; c < end; c += 4 * step) {
                float v[4][VEC];
#pragma unroll
                for (int i = 0; i < 4; ++i) load_16(xr + min(c + step * i, K - VEC), v[i]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int ci = c + step * i;
                    if (ci >= end) break;
                    if (ci > K - VEC) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) v[i][e] = ci + e < K ? load_x(xr + ci + e) : 0.f;
                    }
                    f(ci, v[i]);
                }
            }
        };
        uint32_t m = 0;
        pieces([&](int, const float(&v)[VEC]) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) m = umax(m, abs_bits(v[e]));
        });
        m = wave_max_u32(m);
        if (per > 1) {  // then one turn is all
            if (lane == 0) red[wave] = m;
            __syncthreads();
            for (int w = 0; w < per; ++w) m = umax(m, red[wave / per * per + w]);
        }
        if (row >= M) continue;
        const float s = scale_from_amax(__uint_as_float(m), 127.f), inv = 1.0f / s;
        if (c0 == 0) scale[row] = s;
        pieces([&](int c, const float(&v)[VEC]) {
#pragma unroll
            for (int g = 0; g < VEC / 4; ++g) {
                int k[4];
                codes4(make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]), s, inv, -128, 127, k);
                *reinterpret_cast<uint32_t*>(codes + row * end + c + 4 * g) =
                    (uint32_t)(k[0] & 0xff) | (uint32_t)(k[1] & 0xff) << 8 | (uint32_t)(k[2] & 0xff) << 16 |
                    (uint32_t)(k[3] & 0xff) << 24;
            }
        });
    }
}

// The product of up to 16 rows: a workgroup of W wavefronts per 16 output columns, the K
// range dealt out to them in k64 blocks, their sums added through LDS. The weights are
// read once, by the wavefront that multiplies them, PF blocks on their way at a time.
// FUSE (few rows): the workgroup quantizes the rows itself, behind the first weights'
// loads, which spares a launch; else their tiles come from tokens_kernel. A launch's own
// cost and two trips to memory bound it (768 x 2304, one row: 3.6 us in a graph).
template <int W, bool FUSE, typename TX, typename TY>
__global__ __launch_bounds__(64 * W) void w8a8_small(const TX* __restrict__ x, int64_t ldx,
                                                     const int8_t* __restrict__ xt, const float* __restrict__ sx,
                                                     const int8_t* __restrict__ wt, const float* __restrict__ sw,
                                                     const float* __restrict__ bias, TY* y, int64_t ldy,
                                                     int M, int N, int K, int U, Residual res) {
    constexpr int PF = 4;
    __shared__ int part[W][256];
    __shared__ float scale[FUSE ? kSmallRows : 1];
    __shared__ uint32_t red[W];
    extern __shared__ __attribute__((aligned(16))) int8_t codes[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, c = lane >> 4, tn = blockIdx.x;
    const int nb = U / 2;  // k64 blocks; this wavefront's: wave, wave + W, ...
    const int place = (c >> 1) * 1024 + (c & 1) * 512 + r * 16;
    const int8_t* wp = wt + (int64_t)(tn >> 1) * U * 1024 + (tn & 1) * 256 + place;
    const int8_t* xp = FUSE ? nullptr : xt + place;
    i32x4 fw[PF], fx[PF];
    auto load = [&](int b0) {
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            const int b = min(b0 + W * i, nb - 1);
            fw[i] = *reinterpret_cast<const i32x4*>(wp + (int64_t)b * 2048);
            if constexpr (!FUSE) fx[i] = *reinterpret_cast<const i32x4*>(xp + (int64_t)b * 2048);
        }
    };
    load(wave);
    if constexpr (FUSE) {
        quantize_rows<W>(x, ldx, M, K, 32 * U, codes, scale, red);
        __syncthreads();
    }
    i32x4 acc = {};
    for (int b0 = wave; b0 < nb; b0 += W * PF) {
        i32x4 w[PF], a[PF];
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            w[i] = fw[i];
            if constexpr (FUSE)
                a[i] = *reinterpret_cast<const i32x4*>(codes + min(r, M - 1) * 32 * U + min(b0 + W * i, nb - 1) * 64 + 16 * c);
            else a[i] = fx[i];
        }
        if (b0 + W * PF < nb) load(b0 + W * PF);
#pragma unroll
        for (int i = 0; i < PF; ++i)
            if (b0 + W * i < nb) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], w[i], acc, 0, 0, 0);
    }
    // result register q of lane (r, c): row 4 c + q, column r
#pragma unroll
    for (int q = 0; q < 4; ++q) part[wave][(4 * c + q) * 16 + r] = acc[q];
    __syncthreads();
    const int m = tid >> 4, n = 16 * tn + (tid & 15);
    if (tid >= 256 || m >= M || n >= N) return;
    int s = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) s += part[w][tid];
    store_y(y + (int64_t)m * ldy + n, res(finish(s, FUSE ? scale[m] : sx[m], sw[n], bias ? bias[n] : 0.f), m, n));
}

// The product without a staging step: W wavefronts share the K range of an output tile of
// TM x TN 32 x 32 tiles, each with its own operand loads, PF units on their way at a
// time, and add their sums through LDS, a 32 x 32 tile after the other. No barrier until
// the sums: what bounds it is a trip to L2 a turn, then L2's rate (128 x 6400 x 1600: 11 us).
template <int W, int TM, int TN, int PF, typename TY>
__global__ __launch_bounds__(64 * W) void w8a8_direct(const int8_t* __restrict__ xt, const float* __restrict__ sx,
                                                      const int8_t* __restrict__ wt, const float* __restrict__ sw,
                                                      const float* __restrict__ bias, TY* y, int64_t ldy,
                                                      int M, int N, int U, int tiles_m, Residual res) {
    constexpr int G = TM * TN > 1 ? 2 : 1;  // sets of sums in LDS: one barrier a tile
    __shared__ int part[G][W][32 * 33];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, h = lane >> 5;
    const int tm = blockIdx.x % tiles_m, tn = blockIdx.x / tiles_m;  // a weight tile's workgroups side by side
    const int T = (M + 31) / 32, NT = (N + 31) / 32;
    const int8_t *xp[TM], *wp[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) xp[i] = xt + (int64_t)min(tm * TM + i, T - 1) * U * 1024 + lane * 16;
#pragma unroll
    for (int j = 0; j < TN; ++j) wp[j] = wt + (int64_t)min(tn * TN + j, NT - 1) * U * 1024 + lane * 16;
    i32x4 fa[PF][TM], fb[PF][TN];
    auto load = [&](int u0) {
#pragma unroll
        for (int p = 0; p < PF; ++p) {
            const int64_t o = (int64_t)min(u0 + W * p, U - 1) * 1024;
#pragma unroll
            for (int i = 0; i < TM; ++i) fa[p][i] = *reinterpret_cast<const i32x4*>(xp[i] + o);
#pragma unroll
            for (int j = 0; j < TN; ++j) fb[p][j] = *reinterpret_cast<const i32x4*>(wp[j] + o);
        }
    };
    load(wave);
    i32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = i32x16{};
    for (int u0 = wave; u0 < U; u0 += W * PF) {
        i32x4 a[PF][TM], b[PF][TN];
#pragma unroll
        for (int p = 0; p < PF; ++p) {
#pragma unroll
            for (int i = 0; i < TM; ++i) a[p][i] = fa[p][i];
#pragma unroll
            for (int j = 0; j < TN; ++j) b[p][j] = fb[p][j];
        }
        if (u0 + W * PF < U) load(u0 + W * PF);
#pragma unroll
        for (int p = 0; p < PF; ++p) {
            if (u0 + W * p >= U) break;
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[p][i], b[p][j], acc[i][j], 0, 0, 0);
        }
    }
    // result register q of lane (r, h): row 8 (q / 4) + 4 h + q % 4, column r
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            int(&set)[W][32 * 33] = part[(i * TN + j) % G];
#pragma unroll
            for (int q = 0; q < 16; ++q) set[wave][(8 * (q >> 2) + 4 * h + (q & 3)) * 33 + r] = acc[i][j][q];
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 1024 / (64 * W); ++e) {
                const int o = tid + 64 * W * e;
                const int m = 32 * (tm * TM + i) + (o >> 5), n = 32 * (tn * TN + j) + (o & 31);
                int s = 0;
#pragma unroll
                for (int w = 0; w < W; ++w) s += set[w][(o >> 5) * 33 + (o & 31)];
                if (m < M && n < N)
                    store_y(y + (int64_t)m * ldy + n, res(finish(s, sx[m], sw[n], bias ? bias[n] : 0.f), m, n));
            }
        }
}

// Tile index -> tile: eight contiguous ranges, one an XCD (workgroups go round the XCDs),
// each walked in groups of four row tiles, so that the workgroups of an XCD that run
// together share rows and weights in its L2 (groups of 8, 12 or 16, nearer to a square, are
// level or 1 to 5% slower: 4096 x 1600 x 4800 to bf16 45.1 / 46.6 / 47.3 / 47.3 us).
__device__ __forceinline__ void tile_of(int i, int tiles_m, int tiles_n, int& tm, int& tn) {
    constexpr int XCDS = 8, G = 4;
    const int total = tiles_m * tiles_n, q = total / XCDS, r = total % XCDS;
    const int xcd = i % XCDS, local = i / XCDS;
    const int id = min(xcd, r) * (q + 1) + max(xcd - r, 0) * q + local;
    const int group = id / (G * tiles_n), in = id % (G * tiles_n);
    const int gm = min(tiles_m - group * G, G);
    tm = group * G + in % gm;
    tn = in / gm;
}

// The product of many rows. A workgroup of four wavefronts side by side along N owns
// 32 TM rows x 128 TN columns, a wavefront all the rows and 32 TN columns. The rows' tiles
// pass through LDS (double buffered, one barrier a k64 step; loaded D - 1 steps before
// their LDS store), as all four wavefronts need them; the weights' go straight from
// memory into the registers of the one wavefront that needs them, WD - 1/2 steps ahead:
// 1 KB of consecutive memory an instruction either way, no bank conflicts, no swizzle.
// Beside each MFMA goes one of the step's other operations. Two workgroups a CU, so that
// one's epilogue runs beside the other's MFMAs.
// What bounds it: 8192 x 6400 x 1600 in 128 x 256 tiles takes 79 us (2.12 POP/s; the
// platform's int8 product 88), and 74 of them with every load left out: the MFMAs at the
// clock that the chip holds under them (on rows and codes of zeros 17 us less), and the
// two rounds that 1.75 tiles a CU make; over the launch the MFMAs are busy 0.48 of the cycles,
// at 2.0 GHz. 4096 x 1600 x 4800 to bf16 takes 35 us: 13 its launch and its outputs, the k-loop
// 20 without MFMAs, about as much without loads, 25 with both. Its epilogue took 25 us more when every scale was a load of its own and a
// store two bytes a lane. K split over two or four groups of wavefronts of a workgroup
// gained at 1024 x 6400 x 1600 only (27.4 us against 32.5) and lost 1 to 10 us elsewhere.
template <int TM, int TN, int D, int WD, typename TY>
__device__ __forceinline__ void staged_product(int8_t* smem, int t0, int tn, const int8_t* __restrict__ xt,
                                               const float* __restrict__ sx, const int8_t* __restrict__ wt,
                                               const float* __restrict__ sw, const float* __restrict__ bias, TY* y,
                                               int64_t ldy, int M, int N, int U, const Residual& res) {
    constexpr int STAGE = TM * 2048;             // bytes of a k64 step of rows
    constexpr int XL = STAGE / (256 * 16);       // staging loads a thread and step
    constexpr int NMF = TM * TN;                 // MFMAs a k32 block
    static_assert(STAGE % 4096 == 0, "whole loads a thread");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int T = (M + 31) / 32, NT = (N + 31) / 32, nk = U / 2;

    // rows' tile i of the workgroup: 2 KB a step; thread: 16 bytes of tile q (XL of them)
    const int8_t* xp[XL];
#pragma unroll
    for (int q = 0; q < XL; ++q) {
        const int o = q * 4096 + tid * 16;
        xp[q] = xt + (int64_t)min(t0 + o / 2048, T - 1) * U * 1024 + o % 2048;  // past the last: it again (not stored)
    }
    const int8_t* wp[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) wp[j] = wt + (int64_t)min((tn * 4 + wave) * TN + j, NT - 1) * U * 1024 + lane * 16;

    i32x4 st[D][XL], FW[WD][2][TN], FX[2][TM];
    auto gload = [&](int s, int p, int q) { st[p][q] = *reinterpret_cast<const i32x4*>(xp[q] + (int64_t)s * 2048); };
    auto wload = [&](int s, int p, int kk, int j) {
        FW[p][kk][j] = *reinterpret_cast<const i32x4*>(wp[j] + (int64_t)s * 2048 + kk * 1024);
    };
    auto lstore = [&](int buf, int p, int q) {
        *reinterpret_cast<i32x4*>(smem + buf * STAGE + q * 4096 + tid * 16) = st[p][q];
    };
    auto fread = [&](int buf, int kk, int set, int i) {
        FX[set][i] = *reinterpret_cast<const i32x4*>(smem + buf * STAGE + i * 2048 + kk * 1024 + lane * 16);
    };
    i32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = i32x16{};
    auto mfma = [&](int set, int p, int kk, int t) {
        const int i = t / TN, j = t % TN;
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(FX[set][i], FW[p][kk][j], acc[i][j], 0, 0, 0);
    };

#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int q = 0; q < XL; ++q) gload(min(d, nk - 1), d, q);
#pragma unroll
    for (int d = 0; d < WD; ++d)
#pragma unroll
        for (int kk = 0; kk < (d < WD - 1 ? 2 : 1); ++kk)
#pragma unroll
            for (int j = 0; j < TN; ++j) wload(min(d, nk - 1), d, kk, j);
#pragma unroll
    for (int q = 0; q < XL; ++q) lstore(0, 0, q);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TM; ++i) fread(0, 0, 0, i);

    // Step s (staging set p = s % D, weight set w = s % WD): the first k32 block's MFMAs
    // beside stage s + 1's LDS stores, the second block's row fragments and the
    // second block's weights of s + WD - 1; the barrier; the second block's beside the
    // next step's first row fragments, stage s + D's loads and the first block's weights
    // of s + WD. Past the last stage the loads repeat it.
    auto step = [&](int s, int p, int w) {
        const int cur = s & 1, nxt = cur ^ 1, pn = (p + 1) % D;
        const int s1 = min(s + WD - 1, nk - 1), s2 = min(s + WD, nk - 1), sd = min(s + D, nk - 1);
        constexpr int NOP = XL + TM + TN;
        // (the LDS stores first: done by the barrier)
#pragma unroll
        for (int t = 0; t < NMF; ++t) {
            mfma(0, w, 0, t);
#pragma unroll
            for (int k = t * NOP / NMF; k < (t + 1) * NOP / NMF; ++k) {
                if (k < XL) lstore(nxt, pn, k);
                else if (k < XL + TM) fread(cur, 1, 1, k - XL);
                else wload(s1, (w + WD - 1) % WD, 1, k - XL - TM);
            }
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NMF; ++t) {
            mfma(1, w, 1, t);
#pragma unroll
            for (int k = t * NOP / NMF; k < (t + 1) * NOP / NMF; ++k) {
                if (k < TM) fread(nxt, 0, 0, k);
                else if (k < TM + XL) gload(sd, p, k - TM);
                else wload(s2, w, 0, k - TM - XL);
            }
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr int P = D % 2 ? 2 * D : D;  // steps until the sets and the buffers come round
    static_assert(P % WD == 0, "weight sets");
    if ((tn * 4 + wave) * TN >= NT) {  // columns past the last: only its share of the staging
        int s = 0;
        for (; s < nk; s += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                if (s + d >= nk) break;
#pragma unroll
                for (int q = 0; q < XL; ++q) lstore((s + d + 1) & 1, (d + 1) % D, q);
                __syncthreads();
#pragma unroll
                for (int q = 0; q < XL; ++q) gload(min(s + d + D, nk - 1), d, q);
            }
        }
        return;
    }
    int s = 0;
    for (; s + P <= nk; s += P) {
#pragma unroll
        for (int d = 0; d < P; ++d) step(s + d, d % D, d % WD);
    }
#pragma unroll
    for (int d = 0; d < P - 1; ++d)
        if (s + d < nk) step(s + d, d % D, d % WD);

    // result register q of lane (r, h): row 8 (q / 4) + 4 h + q % 4, column r. The scales
    // are asked for all at once, whole tiles are stored without a test, and bf16
    // neighbours of two rows swap a value each, so that a store takes four bytes a lane. Past
    // the caches, as every workgroup of a round stores at once and the next one's operands are
    // read meanwhile (8192 x 6400 x 1600 fp32 126 us against 135, to bf16 115.5 against 117;
    // 1001 x 1024 x 4096 fp32 13.5 against 14.6; eight GPT-2-XL blocks over 4096 rows 2.64 ms
    // against 2.69).
    const int r = lane & 31, h = lane >> 5;
    const int m0 = t0 * 32 + 4 * h, n0 = (tn * 4 + wave) * TN * 32;
    float scw[TN], b[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int n = min(n0 + 32 * j + r, N - 1);
        scw[j] = sw[n];
        b[j] = bias ? bias[n] : 0.f;
    }
    float4 s4[TM][4];  // (the workspace holds whole tiles of scales)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            s4[i][g] = *reinterpret_cast<const float4*>(sx + min(t0 + i, T - 1) * 32 + 8 * g + 4 * h);
    auto value = [&](int i, int j, int g, int e) {
        const float sxe = e == 0 ? s4[i][g].x : e == 1 ? s4[i][g].y : e == 2 ? s4[i][g].z : s4[i][g].w;
        return finish(acc[i][j][4 * g + e], sxe, scw[j], b[j]);
    };
    const bool whole = (t0 + TM) * 32 <= M && n0 + 32 * TN <= N;
    if (whole && (sizeof(TY) == 4 || (((uintptr_t)y | (uint64_t)ldy * 2) & 3) == 0)) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                TY* dst = y + (int64_t)(m0 + 32 * i + 8 * g) * ldy + n0 + r;
                if constexpr (sizeof(TY) == 4) {
                    float add[4][TN];
                    if (res.res) {
                        const float* src = res.res + (int64_t)(m0 + 32 * i + 8 * g) * res.ldr + n0 + r;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int j = 0; j < TN; ++j) add[e][j] = src[(int64_t)e * res.ldr + 32 * j];
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int j = 0; j < TN; ++j) {
                            const float v = value(i, j, g, e);
                            __builtin_nontemporal_store(res.res ? v + add[e][j] : v, dst + (int64_t)e * ldy + 32 * j);
                        }
                } else {
                    const bool odd = r & 1;  // even lanes store row e, odd ones row e + 1
                    dst += odd ? ldy - 1 : 0;
#pragma unroll
                    for (int e = 0; e < 4; e += 2)
#pragma unroll
                        for (int j = 0; j < TN; ++j) {
                            const float v0 = value(i, j, g, e), v1 = value(i, j, g, e + 1);
                            const float got = dpp_move<0xB1>(odd ? v0 : v1);
                            __builtin_nontemporal_store(odd ? pk_bf16(got, v1) : pk_bf16(v0, got),
                                                        reinterpret_cast<uint32_t*>(dst + (int64_t)e * ldy + 32 * j));
                        }
                }
            }
        return;
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int m = m0 + 32 * i + 8 * g + e;
#pragma unroll
                for (int j = 0; j < TN; ++j)
                    if (m < M && n0 + 32 * j + r < N)
                        store_y(y + (int64_t)m * ldy + n0 + 32 * j + r, res(value(i, j, g, e), m, n0 + 32 * j + r));
            }
}

// A workgroup a tile (tile_of); TAIL: of each XCD's tiles the first `whole`, then the others
// in halves of TM / 2 (whole_of).
template <int TM, int TN, int D, int WD, int OCC, bool TAIL, typename TY>
__global__ __launch_bounds__(256, OCC) void w8a8_staged(const int8_t* __restrict__ xt, const float* __restrict__ sx,
                                                        const int8_t* __restrict__ wt, const float* __restrict__ sw,
                                                        const float* __restrict__ bias, TY* y, int64_t ldy, int M, int N,
                                                        int U, int tiles_m, int tiles_n, int whole, Residual res) {
    __shared__ __attribute__((aligned(1024))) int8_t smem[2 * TM * 2048];
    int tm, tn, i = blockIdx.x;
    if constexpr (TAIL) {
        if (i >= 8 * whole) {
            const int local = (i >> 3) - whole, half = local & 1;
            i = (whole + (local >> 1)) * 8 + (i & 7);
            if (i >= tiles_m * tiles_n) return;
            tile_of(i, tiles_m, tiles_n, tm, tn);
            if ((tm * TM + half * (TM / 2)) * 32 >= M) return;
            staged_product<TM / 2, TN, 4, 4>(smem, tm * TM + half * (TM / 2), tn, xt, sx, wt, sw, bias, y, ldy, M, N, U, res);
            return;
        }
    }
    tile_of(i, tiles_m, tiles_n, tm, tn);
    staged_product<TM, TN, D, WD>(smem, tm * TM, tn, xt, sx, wt, sw, bias, y, ldy, M, N, U, res);
}

// Workgroups of 256 for n pieces of work; each goes on to further ones past 2^20 of them.
unsigned groups_of(int64_t n) { return (unsigned)std::min<int64_t>((n + 255) / 256, 1 << 20); }

size_t round256(size_t b) { return (b + 255) / 256 * 256; }

// Rows a launch: its threads are counted in 32 bits.
constexpr int64_t kTokenRows = 1 << 22;

// Whether a row is held in registers while it is quantized: at most 32 passes of 256 threads
// over its columns, with the padding of the tiles.
template <bool TILES, typename TX>
int64_t token_passes(int64_t K) {
    constexpr int VEC = 16 / (int)sizeof(TX);
    return ((TILES ? 32 * units_of(K) : K) + 64 * VEC - 1) / (64 * VEC);
}
template <bool TILES, typename TX>
bool tokens_held(int64_t K) {
    return K >= 16 / (int64_t)sizeof(TX) && token_passes<TILES, TX>(K) <= 32;
}

template <bool TILES, Before PRE, typename TX>
int launch_tokens(const TX* x, int64_t rows, int64_t K, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                  hipStream_t st, const LnArgs& ln = {}) {
    const int64_t U = units_of(K), passes = token_passes<TILES, TX>(K);
    if (PRE != kAsIs && !tokens_held<TILES, TX>(K)) return TIQ_EUNSUPPORTED;
    for (int64_t r0 = 0; r0 < rows; r0 += kTokenRows) {
        const int n = (int)std::min(rows - r0, kTokenRows);
        const TX* xr = x + r0 * ldx;
        int8_t* qr = q + (TILES ? r0 / 32 * U * 1024 : r0 * ldq);
        auto held = [&](auto kernel, int threads) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)((n + 3) / 4)), dim3(threads), 0, st, xr, ldx, n, (int)K, qr, ldq, U,
                               scale + r0, ln);
        };
        if (!tokens_held<TILES, TX>(K))
            hipLaunchKernelGGL((tokens_generic<TILES, TX>), dim3((unsigned)n), dim3(256), 0, st, xr, ldx, K, qr, ldq, U,
                               scale + r0);
        else if (passes <= 2) held(tokens_kernel<TILES, 2, 256, PRE, TX>, 256);
        else if (passes <= 4) held(tokens_kernel<TILES, 4, 256, PRE, TX>, 256);
        else if (passes <= 8) held(tokens_kernel<TILES, 8, 256, PRE, TX>, 256);
        else if (passes <= 16) held(tokens_kernel<TILES, 4, 1024, PRE, TX>, 1024);
        else held(tokens_kernel<TILES, 8, 1024, PRE, TX>, 1024);
        const int rc = launch_status();
        if (rc != TIQ_OK) return rc;
    }
    return TIQ_OK;
}

// How a product over more than 16 rows is taken, by its 32 x 32 output tiles (rows' T,
// columns' NT); us with the rows' quantization, fp32, both sides:
//   few tiles: the direct product, whose wavefronts need no barrier on the way (T NT =
//     600, 384 x 1600 x 1600: 10.6 against 11.2 .. 12.2 staged; 1600, 1024 x 1600 x 1600:
//     17.1 against 12.4); 2 x 2 tiles a workgroup where K is long (512 x 6400 x 1600: 22.9
//     against 28.1);
//   128 x 256 staged tiles where those are many (152 of them, 1024 x 1600 x 4800: 21.6
//     against 22.9 with 64 x 256; 256, 2048 x 1024 x 4096: 22.4 against 22.0, to bf16 18.7
//     against 20.3; 128, 1001 x 1024 x 4096: 19.5 against 14.7);
//   64 x 256 where those are many (2048 x 1600 x 1600, 224 of them: 17.4 against 18.7 with
//     64 x 128; 1024 x 1600 x 1600, 112: 13.6 against 12.4), else 64 x 128.
// Whether the product quantizes its rows itself (then it takes no workspace): up to 8
// rows, up to 16 where they are short. (us in a graph, so / by a launch of their own before,
// which an eager call's host also waits 4 us for: 1 x 768 x 2304 3.6 / 5.3, 8 x 768 x 2304
// 4.3 / 5.3, 4 x 6400 x 1600 7.7 / 9.1, 8 x 4096 x 1024 7.5 / 6.9, 16 x 768 x 2304 5.9 / 5.3,
// 16 x 1600 x 6400 10.7 / 6.6.)
bool rows_fused(int x_dtype, int64_t M, int64_t K) {
    const int64_t bytes = M * 32 * units_of(K);  // of codes, in LDS
    return M <= kSmallRows && bytes <= (M <= 8 ? kFusedBytes : 12544) && K >= (x_dtype == TIQ_F32 ? 4 : 8);
}

enum Path { kDirect, kDirectLong, kStaged64x128, kStaged64x256, kStaged128x256 };

Path path_of(int64_t T, int64_t NT, int64_t K) {
    if (T * NT <= 400) return kDirect;
    if (K >= 3200 && T * NT <= 1200) return kDirectLong;
    if (T * NT <= 800) return kDirect;
    if ((T + 3) / 4 * ((NT + 7) / 8) >= 150) return kStaged128x256;
    return (T + 1) / 2 * ((NT + 7) / 8) >= 150 ? kStaged64x256 : kStaged64x128;
}

// 128 x 256 tiles: how many of an XCD's, which its 32 CUs take in rounds, are taken whole,
// the rest in halves, or -1: all of them whole. A last round of halves, one a CU at most,
// takes half the time (4096 x 1600 x 4800 fp32, 12 of 76 tiles an XCD: 47.6 us against 50.6;
// 4096 x 6400 x 2304, 4 of 36: 86.5 against 97.3); two a CU do not (8192 x 1600 x 1600, 24 of
// 56: 45.1 against 40.6).
int64_t whole_of(int64_t T, int64_t NT) {
    const int64_t tiles = ((T + 3) / 4 * ((NT + 7) / 8) + 7) / 8, whole = tiles / 32 * 32;
    return whole && tiles > whole && tiles - whole <= 16 ? whole : -1;
}

// What stands around a product: before its rows are quantized, after its sums.
struct Around {
    Before pre = kAsIs;
    LnArgs ln = {};
    Residual res = {};
};

template <typename TX, typename TY>
int run_w8a8(const TX* x, int64_t M, int64_t K, int64_t ldx, const int8_t* wt, const float* sw, const float* bias,
             int64_t N, TY* y, int64_t ldy, uint8_t* ws, hipStream_t st, const Around& o = {}) {
    const int64_t U = units_of(K), T = tiles_of(M), NT = tiles_of(N);
    int8_t* xt = reinterpret_cast<int8_t*>(ws);
    float* sx = reinterpret_cast<float*>(ws + T * U * 1024);
    auto small = [&](auto kernel, int W, size_t lds) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((N + 15) / 16)), dim3(64 * W), lds, st, x, ldx, xt, sx, wt, sw, bias,
                           y, ldy, (int)M, (int)N, (int)K, (int)U, o.res);
        return launch_status();
    };
    if (o.pre == kAsIs && rows_fused(sizeof(TX) == 4 ? TIQ_F32 : TIQ_BF16, M, K)) {
        const size_t lds = (size_t)(M * 32 * U);
        return K > 2048 ? small(w8a8_small<16, true, TX, TY>, 16, lds) : small(w8a8_small<8, true, TX, TY>, 8, lds);
    }
    int rc = TIQ_EUNSUPPORTED;
    if (o.pre == kAsIs) rc = launch_tokens<true, kAsIs>(x, M, K, ldx, xt, (int64_t)0, sx, st);
    if constexpr (sizeof(TX) == 4 && sizeof(TY) == 4) {
        if (o.pre == kLayerNorm) rc = launch_tokens<true, kLayerNorm>(x, M, K, ldx, xt, (int64_t)0, sx, st, o.ln);
        if (o.pre == kGelu) rc = launch_tokens<true, kGelu>(x, M, K, ldx, xt, (int64_t)0, sx, st);
    }
    if (rc != TIQ_OK) return rc;
    if (M <= kSmallRows) return K > 2048 ? small(w8a8_small<16, false, TX, TY>, 16, 0) : small(w8a8_small<8, false, TX, TY>, 8, 0);
    auto direct = [&](auto kernel, int TM, int TN) {
        const int64_t tm = (T + TM - 1) / TM, tn = (NT + TN - 1) / TN;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(tm * tn)), dim3(512), 0, st, xt, sx, wt, sw, bias, y, ldy, (int)M,
                           (int)N, (int)U, (int)tm, o.res);
        return launch_status();
    };
    auto staged = [&](auto kernel, int TM, int TN) {
        const int64_t tm = (T + TM - 1) / TM, tn = (NT + 4 * TN - 1) / (4 * TN);
        const int64_t whole = TM == 4 ? whole_of(T, NT) : -1;
        const int64_t groups = whole < 0 ? tm * tn : 8 * (2 * ((tm * tn + 7) / 8) - whole);
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, st, xt, sx, wt, sw, bias, y, ldy, (int)M,
                           (int)N, (int)U, (int)tm, (int)tn, (int)whole, o.res);
        return launch_status();
    };
    switch (path_of(T, NT, K)) {
        case kDirect: return direct(w8a8_direct<8, 1, 1, 4, TY>, 1, 1);
        case kDirectLong: return direct(w8a8_direct<8, 2, 2, 2, TY>, 2, 2);
        case kStaged64x128: return staged(w8a8_staged<2, 1, 4, 4, 2, false, TY>, 2, 1);
        case kStaged64x256: return staged(w8a8_staged<2, 2, 4, 4, 2, false, TY>, 2, 2);
        default:
            if (whole_of(T, NT) >= 0) return staged(w8a8_staged<4, 2, 3, 3, 2, true, TY>, 4, 2);
            return staged(w8a8_staged<4, 2, 3, 3, 2, false, TY>, 4, 2);
    }
}

size_t tiles_workspace(int64_t M, int64_t K) {
    return round256((size_t)(tiles_of(M) * (units_of(K) * 1024 + 128)));  // (scales of whole tiles)
}

// (threads of a launch are counted in 32 bits: 64 an output column, for few rows)
bool sizes_taken(int64_t M, int64_t K, int64_t N) {
    return K <= kMaxK && M <= 0x7fffffc0LL && N <= 1 << 25 && tiles_of(M) * tiles_of(N) <= 1 << 26;
}

bool known_dtype(int d) { return d == TIQ_F32 || d == TIQ_BF16; }

}  // namespace
}  // namespace tiq

using namespace tiq;

extern "C" int tiq_quantize_tokens(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t ldx, int8_t* q,
                                   int64_t ldq, float* scale, void* stream) {
    if (!known_dtype(x_dtype) || rows < 0 || cols < 0) return TIQ_EINVAL;
    if (rows == 0 || cols == 0) return TIQ_OK;
    if (!x || !q || !scale || ldx < cols || ldq < cols) return TIQ_EINVAL;
    if (!aligned(x, x_dtype == TIQ_F32 ? 4 : 2) || !aligned(scale, 4)) return TIQ_EALIGN;
    if (rows > 0x7fffffffLL) return TIQ_EUNSUPPORTED;
    if (x_dtype == TIQ_F32)
        return launch_tokens<false, kAsIs>(static_cast<const float*>(x), rows, cols, ldx, q, ldq, scale, as_stream(stream));
    return launch_tokens<false, kAsIs>(static_cast<const uint16_t*>(x), rows, cols, ldx, q, ldq, scale, as_stream(stream));
}

extern "C" size_t tiq_w8a8_tiles_bytes(int64_t N, int64_t K) {
    return N <= 0 || K <= 0 ? 0 : (size_t)(tiles_of(N) * units_of(K) * 1024);
}

extern "C" int tiq_w8a8_tile(const int8_t* q, int64_t N, int64_t K, int64_t ldq, int8_t* tiles, void* stream) {
    if (N < 0 || K < 0) return TIQ_EINVAL;
    if (N == 0 || K == 0) return TIQ_OK;
    if (!q || !tiles || ldq < K) return TIQ_EINVAL;
    if (!aligned(tiles, 16)) return TIQ_EALIGN;
    const int64_t U = units_of(K), chunks = tiles_of(N) * U * 64;
    hipLaunchKernelGGL(tile_weight_kernel, dim3(groups_of(chunks)), dim3(256), 0, as_stream(stream), q, N, K, ldq, U,
                       chunks, tiles);
    return launch_status();
}

extern "C" int tiq_w8a8_untile(const int8_t* tiles, int64_t N, int64_t K, int8_t* q, void* stream) {
    if (N < 0 || K < 0) return TIQ_EINVAL;
    if (N == 0 || K == 0) return TIQ_OK;
    if (!q || !tiles) return TIQ_EINVAL;
    hipLaunchKernelGGL(untile_weight_kernel, dim3(groups_of(N * K)), dim3(256), 0, as_stream(stream), tiles, K,
                       units_of(K), N * K, q);
    return launch_status();
}

extern "C" size_t tiq_linear_w8a8_workspace(int x_dtype, int64_t M, int64_t K, int64_t N) {
    if (!known_dtype(x_dtype) || M <= 0 || K <= 0 || N <= 0 || rows_fused(x_dtype, M, K)) return 0;
    return tiles_workspace(M, K);
}

extern "C" int tiq_linear_w8a8(const void* x, int x_dtype, int64_t M, int64_t K, int64_t ldx, const int8_t* w_tiles,
                               const float* scale, const float* bias, int64_t N, void* y, int y_dtype, int64_t ldy,
                               void* workspace, size_t workspace_bytes, void* stream) {
    if (!known_dtype(x_dtype) || !known_dtype(y_dtype) || M < 0 || K < 0 || N < 0) return TIQ_EINVAL;
    if (M == 0 || N == 0) return TIQ_OK;
    if (K == 0 || !x || !w_tiles || !scale || !y || ldx < K || ldy < N) return TIQ_EINVAL;
    if (!aligned(x, x_dtype == TIQ_F32 ? 4 : 2) || !aligned(y, y_dtype == TIQ_F32 ? 4 : 2) || !aligned(w_tiles, 16) ||
        !aligned(scale, 4) || !aligned(bias, 4))
        return TIQ_EALIGN;
    if (!sizes_taken(M, K, N)) return TIQ_EUNSUPPORTED;
    const size_t need = tiq_linear_w8a8_workspace(x_dtype, M, K, N);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16))) return TIQ_EWORKSPACE;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    hipStream_t st = as_stream(stream);
    if (x_dtype == TIQ_F32) {
        const float* xf = static_cast<const float*>(x);
        if (y_dtype == TIQ_F32) return run_w8a8(xf, M, K, ldx, w_tiles, scale, bias, N, static_cast<float*>(y), ldy, ws, st);
        return run_w8a8(xf, M, K, ldx, w_tiles, scale, bias, N, static_cast<uint16_t*>(y), ldy, ws, st);
    }
    const uint16_t* xb = static_cast<const uint16_t*>(x);
    if (y_dtype == TIQ_F32) return run_w8a8(xb, M, K, ldx, w_tiles, scale, bias, N, static_cast<float*>(y), ldy, ws, st);
    return run_w8a8(xb, M, K, ldx, w_tiles, scale, bias, N, static_cast<uint16_t*>(y), ldy, ws, st);
}

extern "C" size_t tiq_linear_w8a8_prefill_workspace(int64_t M, int64_t K, int64_t N) {
    if (M <= 0 || K <= 0 || N <= 0 || !tokens_held<true, float>(K) || !sizes_taken(M, K, N)) return 0;
    return tiles_workspace(M, K);
}

extern "C" int tiq_linear_w8a8_prefill(const float* x, int64_t M, int64_t K, int64_t ldx, const int8_t* w_tiles,
                                       const float* scale, const float* bias, int64_t N, float* y, int64_t ldy,
                                       const float* ln_weight, const float* ln_bias, float ln_eps, int gelu,
                                       const float* residual, int64_t ld_residual, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    if (M < 0 || K < 0 || N < 0 || (ln_weight == nullptr) != (ln_bias == nullptr) || (ln_weight && gelu))
        return TIQ_EINVAL;
    if (M == 0 || N == 0) return TIQ_OK;
    if (K == 0 || !x || !w_tiles || !scale || !y || ldx < K || ldy < N || (residual && ld_residual < N)) return TIQ_EINVAL;
    if (!aligned(x, 4) || !aligned(y, 4) || !aligned(w_tiles, 16) || !aligned(scale, 4) || !aligned(bias, 4) ||
        !aligned(residual, 4) || !aligned(ln_weight, 4) || !aligned(ln_bias, 4))
        return TIQ_EALIGN;
    const size_t need = tiq_linear_w8a8_prefill_workspace(M, K, N);
    if (!need) return TIQ_EUNSUPPORTED;
    if (!workspace || workspace_bytes < need || !aligned(workspace, 16)) return TIQ_EWORKSPACE;
    const Around o = {ln_weight ? kLayerNorm : gelu ? kGelu : kAsIs, {ln_weight, ln_bias, ln_eps}, {residual, ld_residual}};
    return run_w8a8(x, M, K, ldx, w_tiles, scale, bias, N, y, ldy, static_cast<uint8_t*>(workspace), as_stream(stream), o);
}
