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

// Weight codes (N, K) -> tiles, a thread per 16 bytes of them.
__global__ __launch_bounds__(256) void tile_weight_kernel(const int8_t* __restrict__ w, int64_t N, int64_t K,
                                                          int64_t ldw, int64_t U, int64_t chunks,
                                                          int8_t* __restrict__ tiles) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= chunks) return;
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

// Tiles -> codes (N, K), a thread per code.
__global__ __launch_bounds__(256) void untile_weight_kernel(const int8_t* __restrict__ tiles, int64_t K, int64_t U,
                                                            int64_t count, int8_t* __restrict__ w) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) w[i] = tiles[tile_byte(i / K, i % K, U)];
}

__device__ __forceinline__ void store_y(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_y(uint16_t* p, float v) { *p = f32_to_bf16_bits(v); }

__device__ __forceinline__ float finish(int sum, float sx, float sw, float b) {
    return fmaf((float)sum * sx, sw, b);
}

// The product without a staging step: W wavefronts share the K range of one 32 x 32
// output tile, each with its own operand loads (1 KB of consecutive memory an
// instruction), and add their sums through LDS.
template <int W, typename TY>
__global__ __launch_bounds__(64 * W) void w8a8_direct(const int8_t* __restrict__ xt, const float* __restrict__ sx,
                                                      const int8_t* __restrict__ wt, const float* __restrict__ sw,
                                                      const float* __restrict__ bias, TY* __restrict__ y, int64_t ldy,
                                                      int M, int N, int U, int tiles_n) {
    constexpr int LD = 36;  // a row of sums in LDS, padded to whole 16-byte chunks
    __shared__ __attribute__((aligned(16))) int part[W][32 * LD];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 31, h = lane >> 5;
    const int tm = blockIdx.x / tiles_n, tn = blockIdx.x % tiles_n;
    const int8_t* xp = xt + (int64_t)tm * U * 1024 + lane * 16;
    const int8_t* wp = wt + (int64_t)tn * U * 1024 + lane * 16;
    i32x16 acc = {};
    for (int u = wave; u < U; u += W) {
        const i32x4 a = *reinterpret_cast<const i32x4*>(xp + u * 1024);
        const i32x4 b = *reinterpret_cast<const i32x4*>(wp + u * 1024);
        acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, acc, 0, 0, 0);
    }
    // result register q of lane (r, h): row 8 (q / 4) + 4 h + q % 4, column r
#pragma unroll
    for (int q = 0; q < 16; ++q) part[wave][(8 * (q >> 2) + 4 * h + (q & 3)) * LD + r] = acc[q];
    __syncthreads();
    for (int i = threadIdx.x; i < 1024; i += 64 * W) {
        const int m = 32 * tm + (i >> 5), n = 32 * tn + (i & 31);
        if (m >= M || n >= N) continue;
        int s = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) s += part[w][(i >> 5) * LD + (i & 31)];
        store_y(y + (int64_t)m * ldy + n, finish(s, sx[m], sw[n], bias ? bias[n] : 0.f));
    }
}

size_t round256(size_t b) { return (b + 255) / 256 * 256; }

template <bool TILES, typename TX>
int launch_tokens(const TX* x, int64_t rows, int64_t K, int64_t ldx, int8_t* q, int64_t ldq, float* scale,
                  hipStream_t st) {
    hipLaunchKernelGGL((tokens_generic<TILES, TX>), dim3((unsigned)rows), dim3(256), 0, st, x, ldx, K, q, ldq,
                       units_of(K), scale);
    return launch_status();
}

template <typename TX, typename TY>
int run_w8a8(const TX* x, int64_t M, int64_t K, int64_t ldx, const int8_t* wt, const float* sw, const float* bias,
             int64_t N, TY* y, int64_t ldy, uint8_t* ws, hipStream_t st) {
    const int64_t U = units_of(K), TN = tiles_of(N);
    int8_t* xt = reinterpret_cast<int8_t*>(ws);
    float* sx = reinterpret_cast<float*>(ws + tiles_of(M) * U * 1024);
    const int rc = launch_tokens<true>(x, M, K, ldx, xt, (int64_t)0, sx, st);
    if (rc != TIQ_OK) return rc;
    hipLaunchKernelGGL((w8a8_direct<4, TY>), dim3((unsigned)(tiles_of(M) * TN)), dim3(256), 0, st, xt, sx, wt, sw,
                       bias, y, ldy, (int)M, (int)N, (int)U, (int)TN);
    return launch_status();
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
        return launch_tokens<false>(static_cast<const float*>(x), rows, cols, ldx, q, ldq, scale, as_stream(stream));
    return launch_tokens<false>(static_cast<const uint16_t*>(x), rows, cols, ldx, q, ldq, scale, as_stream(stream));
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
    if (chunks / 256 > 0x7fffffffLL) return TIQ_EUNSUPPORTED;
    hipLaunchKernelGGL(tile_weight_kernel, dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, as_stream(stream), q,
                       N, K, ldq, U, chunks, tiles);
    return launch_status();
}

extern "C" int tiq_w8a8_untile(const int8_t* tiles, int64_t N, int64_t K, int8_t* q, void* stream) {
    if (N < 0 || K < 0) return TIQ_EINVAL;
    if (N == 0 || K == 0) return TIQ_OK;
    if (!q || !tiles) return TIQ_EINVAL;
    if ((N * K + 255) / 256 > 0x7fffffffLL) return TIQ_EUNSUPPORTED;
    hipLaunchKernelGGL(untile_weight_kernel, dim3((unsigned)((N * K + 255) / 256)), dim3(256), 0, as_stream(stream),
                       tiles, K, units_of(K), N * K, q);
    return launch_status();
}

extern "C" size_t tiq_linear_w8a8_workspace(int64_t M, int64_t K, int64_t N) {
    if (M <= 0 || K <= 0 || N <= 0) return 0;
    return round256((size_t)(tiles_of(M) * units_of(K) * 1024 + 4 * M));
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
    if (K > kMaxK || M > 0x7fffffc0LL || N > 0x7fffffc0LL || tiles_of(M) * tiles_of(N) > 0x7fffffffLL)
        return TIQ_EUNSUPPORTED;
    if (!workspace || workspace_bytes < tiq_linear_w8a8_workspace(M, K, N) || !aligned(workspace, 16))
        return TIQ_EWORKSPACE;
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
