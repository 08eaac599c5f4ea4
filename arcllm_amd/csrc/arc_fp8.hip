// arc_fp8.hip -- products in 8-bit floating point (e4m3) with a scale for each block of
// 128: the rows' quantisation, y = x w^T, and the gate/up pair with its activation.
//
//   y[m][n] = sum_b xs[b][m] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k]
//
// The inner sums go through the matrix cores a block at a time, the outer ones are fused
// multiply-adds in fp32.
#include "arc_paged.hpp"

namespace arc {
namespace {

constexpr uint32_t kFpBlock = 128;
constexpr float kE4m3Max = 448.0f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

// ------------------------------------------------------------------ quantise
// A block's scale from the bits of its largest magnitude.
__device__ __forceinline__ float scale_of(uint32_t most)
{
    if (most >= 0x7f800000u) return __builtin_nanf("");
    return fmaxf(__builtin_bit_cast(float, most) / kE4m3Max, 0x1p-126f);
}

// The largest of 16 lanes (a DPP row), as bits of magnitudes.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v)
{
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ uint32_t row_max(uint32_t v)
{
    v = max(v, dpp_u<0xb1>(v));   // lanes ^ 1
    v = max(v, dpp_u<0x4e>(v));   // ^ 2
    v = max(v, dpp_u<0x141>(v));  // the other half of 8
    v = max(v, dpp_u<0x140>(v));  // the other half of 16
    return v;
}

struct Quantize {
    const void* x;
    uint8_t* q;
    float* scales;
    uint32_t rows, cols, ldx, ldq, lds;
};

// 16 lanes to a block, 8 values a lane; a wave has 4 blocks of a row, a workgroup those 4 of 32 rows, whose scales go
// out through LDS so that they are written in whole lines.
constexpr uint32_t kQuantRows = 32;
template <typename X>
__global__ __launch_bounds__(256) void k_fp8_quantize(Quantize a)
{
    __shared__ float scales[4][kQuantRows];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t col = blockIdx.x * 512 + lane * 8, row0 = blockIdx.y * kQuantRows;
    const bool in = col < a.cols;
    for (uint32_t i = wave; i < kQuantRows && row0 + i < a.rows; i += 4) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
        if (in) {
            const X* p = static_cast<const X*>(a.x) + uint64_t(row0 + i) * a.ldx + col;
            const vec8<X> r = *reinterpret_cast<const vec8<X>*>(p);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = static_cast<float>(r[j]);
        }
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = max(most, __builtin_bit_cast(uint32_t, v[j]) & 0x7fffffffu);
        const float s = scale_of(row_max(most));
        if ((lane & 15u) == 0) scales[lane >> 4][i] = s;
        if (in) {
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                w[j] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j] / s, v[4 * j + 1] / s, 0, false));
                w[j] = uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * j + 2] / s, v[4 * j + 3] / s, int(w[j]), true));
            }
            *reinterpret_cast<uint2*>(a.q + uint64_t(row0 + i) * a.ldq + col) = make_uint2(w[0], w[1]);
        }
    }
    __syncthreads();
    const uint32_t b = threadIdx.x / kQuantRows, r = threadIdx.x % kQuantRows;
    if (b < 4 && row0 + r < a.rows && (blockIdx.x * 4 + b) * kFpBlock < a.cols)
        a.scales[uint64_t(blockIdx.x * 4 + b) * a.lds + row0 + r] = scales[b][r];
}

// ------------------------------------------------------------------- product
struct Gemm {
    const uint8_t* w[2];
    const float* ws[2];
    const uint8_t* x;
    const float* xs;
    void* y;
    const void* res;
    uint32_t M, N, K, blocks;
    uint32_t ldw[2], ldws[2], ldx, ldxs, ldy, ldr;
    uint32_t wide;  // y and residual take 4 values at a time
};

// 4 neighbouring outputs of a row: the activation or the residual, rounded once.
__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }
template <typename Y>
__device__ __forceinline__ void store_out(const Gemm& a, uint32_t m, uint32_t n, f32x4 v)
{
    if (m >= a.M || n >= a.N) return;
    Y* p = static_cast<Y*>(a.y) + uint64_t(m) * a.ldy + n;
    const Y* r = static_cast<const Y*>(a.res) + uint64_t(m) * a.ldr + n;
    if (a.wide && n + 4 <= a.N) {
        if (a.res) {
            const vec4<Y> add = *reinterpret_cast<const vec4<Y>*>(r);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += static_cast<float>(add[i]);
        }
        vec4<Y> o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = static_cast<Y>(v[i]);
        *reinterpret_cast<vec4<Y>*>(p) = o;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < a.N) p[i] = static_cast<Y>(a.res ? v[i] + static_cast<float>(r[i]) : v[i]);
}

// A lane's 32 values of a row's block: 16 bytes from column c on and 16 from c + 64, zeros from column K on.
struct Frag {
    u32x4 lo, hi;
};
__device__ __forceinline__ Frag load_frag(const uint8_t* row, uint32_t c, uint32_t K)
{
    Frag f;
    f.lo = f.hi = u32x4{0, 0, 0, 0};
    if (c < K) f.lo = *reinterpret_cast<const u32x4*>(row + c);
    if (c + 64 < K) f.hi = *reinterpret_cast<const u32x4*>(row + c + 64);
    return f;
}
// 8 e4m3 values as fp16, which holds them all.
__device__ __forceinline__ h16x8 widen(uint32_t a, uint32_t b)
{
    const h16x2 x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false), y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    const h16x2 z = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false), w = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    return h16x8{x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}
struct Wide {
    h16x8 v[4];
};
__device__ __forceinline__ Wide widen(const Frag& f)
{
    return Wide{{widen(f.lo.x, f.lo.y), widen(f.lo.z, f.lo.w), widen(f.hi.x, f.hi.y), widen(f.hi.z, f.hi.w)}};
}
// A block's inner sums of 16 rows of w and 16 of x: lane -> row 4 (lane / 16) + i of w, row lane % 16 of x.  In which
// order the lanes hold a block's values does not matter, as it is the same for both.
__device__ __forceinline__ f32x4 block_sums(const Wide& w, const Wide& x)
{
    f32x4 p = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[i], x.v[i], p, 0, 0, 0);
    return p;
}

// 16 rows of w and 16 of x to a workgroup; its 8 waves take the blocks in turn, straight from memory, and add up in
// wave order through LDS.
constexpr uint32_t kFewWaves8 = 8;
template <typename Y, bool GATED>
__global__ __launch_bounds__(512) void k_fp8_few(Gemm a)
{
    constexpr int G = GATED ? 2 : 1;
    __shared__ f32x4 sums[kFewWaves8][G][64];
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
    const uint32_t wave = uint32_t(__builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)));
    const uint32_t n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
    const uint32_t n = min(n0 + r, a.N - 1), m = min(m0 + r, a.M - 1);
    const uint8_t* x = a.x + uint64_t(m) * a.ldx;
    f32x4 acc[G];
#pragma unroll
    for (int h = 0; h < G; ++h) acc[h] = f32x4{0, 0, 0, 0};
    for (uint32_t b = wave; b < a.blocks; b += kFewWaves8) {
        const uint32_t c = b * kFpBlock + g * 16;
        const Wide xf = widen(load_frag(x, c, a.K));
        const float xs = a.xs[uint64_t(b) * a.ldxs + m];
#pragma unroll
        for (int h = 0; h < G; ++h) {
            const Wide wf = widen(load_frag(a.w[h] + uint64_t(n) * a.ldw[h], c, a.K));
            const float s = xs * a.ws[h][uint64_t(n0 / kFpBlock) * a.ldws[h] + b];
            const f32x4 p = block_sums(wf, xf);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[h][i] = __builtin_fmaf(p[i], s, acc[h][i]);
        }
    }
#pragma unroll
    for (int h = 0; h < G; ++h) sums[wave][h][lane] = acc[h];
    __syncthreads();
    if (threadIdx.x >= 64) return;
    f32x4 t[G];
#pragma unroll
    for (int h = 0; h < G; ++h) {
        t[h] = sums[0][h][lane];
        for (uint32_t i = 1; i < kFewWaves8; ++i) t[h] += sums[i][h][lane];
    }
    if constexpr (GATED)
#pragma unroll
        for (int i = 0; i < 4; ++i) t[0][i] = silu(t[0][i]) * t[1][i];
    store_out<Y>(a, m0 + r, n0 + 4 * g, t[0]);
}

// ---------------------------------------------------------------------- host
constexpr uint32_t kMaxLd = 1u << 22;     // bytes from row to row of w and x
constexpr uint32_t kMaxRows = 1u << 24;

int check_matrix(const char* what, const void* p, const float* scales, uint32_t rows, uint32_t cols, uint32_t ld)
{
    if (!p || !scales) return set_error(ARC_ERR_INVALID_ARGUMENT, "%s: null values or scales", what);
    if (rows > kMaxRows || cols == 0 || cols % 16 || cols > kMaxLd)
        return set_error(ARC_ERR_UNSUPPORTED, "%s: %u x %u: at most 2^24 rows, columns a multiple of 16, at most 2^22", what, rows, cols);
    if (ld < cols || ld % 16 || ld > kMaxLd)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "%s: %u bytes from row to row: a multiple of 16, at least %u, at most 2^22", what, ld, cols);
    if (!aligned(p, 16) || !aligned(scales, 4))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "%s: values must be 16-byte, scales 4-byte aligned", what);
    return ARC_OK;
}
int check_rows(const arc_fp8_rows* x)
{
    if (!x) return set_error(ARC_ERR_INVALID_ARGUMENT, "null rows");
    if (int rc = check_matrix("rows", x->q, x->scales, x->rows, x->cols, x->ldq)) return rc;
    if (x->lds < x->rows) return set_error(ARC_ERR_INVALID_ARGUMENT, "rows: lds %u is less than %u rows", x->lds, x->rows);
    return ARC_OK;
}
int check_weights(const arc_fp8_weights* w, const arc_fp8_rows* x)
{
    if (!w) return set_error(ARC_ERR_INVALID_ARGUMENT, "null weights");
    if (int rc = check_matrix("weights", w->w, w->scales, w->rows, w->cols, w->ldw)) return rc;
    if (w->rows == 0) return set_error(ARC_ERR_INVALID_ARGUMENT, "weights: no rows");
    if (w->cols != x->cols) return set_error(ARC_ERR_INVALID_ARGUMENT, "weights of %u columns, rows of %u", w->cols, x->cols);
    if (w->lds < (w->cols + kFpBlock - 1) / kFpBlock)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "weights: lds %u is less than the blocks of %u columns", w->lds, w->cols);
    return ARC_OK;
}
uint32_t bytes_of(int dtype) { return dtype == ARC_F32 ? 4 : dtype == ARC_F16 || dtype == ARC_BF16 ? 2 : 0; }

template <typename Y, bool GATED>
hipError_t launch_few(const Gemm& a, hipStream_t st)
{
    hipLaunchKernelGGL((k_fp8_few<Y, GATED>), dim3((a.N + 15) / 16, (a.M + 15) / 16), dim3(64 * kFewWaves8), 0, st, a);
    return hipGetLastError();
}
template <typename Y>
hipError_t launch(const Gemm& a, bool gated, hipStream_t st)
{
    return gated ? launch_few<Y, true>(a, st) : launch_few<Y, false>(a, st);
}

int product(const arc_fp8_weights* w, const arc_fp8_weights* up, bool gated, const arc_fp8_rows* x, int y_dtype, void* y, uint32_t ldy,
            const void* residual, uint32_t ldr, void* workspace, hipStream_t st)
{
    int rc = check_rows(x);
    if (!rc) rc = check_weights(w, x);
    if (!rc && gated) rc = check_weights(up, x);
    if (rc) return rc;
    if (gated && up->rows != w->rows) return set_error(ARC_ERR_INVALID_ARGUMENT, "gate of %u rows, up of %u", w->rows, up->rows);
    const uint32_t size = bytes_of(y_dtype), N = w->rows;
    if (size == 0) return set_error(ARC_ERR_UNSUPPORTED, "y is ARC_F32, ARC_F16 or ARC_BF16 (dtype %d)", y_dtype);
    if (!y || !workspace) return set_error(ARC_ERR_INVALID_ARGUMENT, "null argument");
    if (ldy < N || (residual && ldr < N)) return set_error(ARC_ERR_INVALID_ARGUMENT, "ldy %u, ldr %u: at least %u", ldy, ldr, N);
    if (!aligned(y, size) || !aligned(residual, size)) return set_error(ARC_ERR_INVALID_ARGUMENT, "y and residual must be aligned to their type");
    if (!aligned(workspace, 256)) return set_error(ARC_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    const uint64_t row = uint64_t(N) * size;
    if (residual && !(residual == y && ldr == ldy) &&
        rows_overlap(y, row, uint64_t(ldy) * size, residual, row, uint64_t(ldr) * size, x->rows))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "y and residual share memory without being the same rows");
    if (rows_overlap(y, row, uint64_t(ldy) * size, x->q, x->cols, x->ldq, x->rows))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "y and the rows share memory");
    if (x->rows == 0) return ARC_OK;
    Gemm a{};
    a.w[0] = static_cast<const uint8_t*>(w->w);
    a.ws[0] = w->scales;
    a.ldw[0] = w->ldw;
    a.ldws[0] = w->lds;
    if (gated) {
        a.w[1] = static_cast<const uint8_t*>(up->w);
        a.ws[1] = up->scales;
        a.ldw[1] = up->ldw;
        a.ldws[1] = up->lds;
    }
    a.x = static_cast<const uint8_t*>(x->q);
    a.xs = x->scales;
    a.y = y;
    a.res = residual;
    a.M = x->rows;
    a.N = N;
    a.K = x->cols;
    a.blocks = (x->cols + kFpBlock - 1) / kFpBlock;
    a.ldx = x->ldq;
    a.ldxs = x->lds;
    a.ldy = ldy;
    a.ldr = ldr;
    a.wide = aligned(y, 4 * size) && ldy % 4 == 0 && (!residual || (aligned(residual, 4 * size) && ldr % 4 == 0));
    const hipError_t e = y_dtype == ARC_F32   ? launch<float>(a, gated, st)
                         : y_dtype == ARC_F16 ? launch<_Float16>(a, gated, st)
                                              : launch<bf16>(a, gated, st);
    return check_hip(e, "fp8 product");
}

}  // namespace
}  // namespace arc

using namespace arc;

extern "C" {

int arc_fp8_quantize(int x_dtype, const void* x, uint32_t ldx, const arc_fp8_rows* out, arc_stream_t stream)
{
    if (int rc = check_rows(out)) return rc;
    const uint32_t size = bytes_of(x_dtype);
    if (size == 0) return set_error(ARC_ERR_UNSUPPORTED, "x is ARC_F32, ARC_F16 or ARC_BF16 (dtype %d)", x_dtype);
    if (!x || !aligned(x, 16)) return set_error(ARC_ERR_INVALID_ARGUMENT, "x must be 16-byte aligned");
    if (ldx < out->cols || ldx % 8) return set_error(ARC_ERR_INVALID_ARGUMENT, "ldx %u: a multiple of 8, at least %u", ldx, out->cols);
    if (rows_overlap(x, uint64_t(out->cols) * size, uint64_t(ldx) * size, out->q, out->cols, out->ldq, out->rows))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "x and the rows share memory");
    if (out->rows == 0) return ARC_OK;
    const Quantize a{x, static_cast<uint8_t*>(out->q), out->scales, out->rows, out->cols, ldx, out->ldq, out->lds};
    const dim3 grid((out->cols + 511) / 512, (out->rows + kQuantRows - 1) / kQuantRows);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (x_dtype == ARC_F32) hipLaunchKernelGGL(k_fp8_quantize<float>, grid, dim3(256), 0, st, a);
    else if (x_dtype == ARC_F16) hipLaunchKernelGGL(k_fp8_quantize<_Float16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_fp8_quantize<bf16>, grid, dim3(256), 0, st, a);
    return check_hip(hipGetLastError(), "fp8 quantize");
}

size_t arc_fp8_gemm_workspace_bytes(uint32_t N, uint32_t K, uint32_t M, int gated)
{
    (void)gated;
    return N == 0 || N > kMaxRows || M > kMaxRows || K == 0 || K % 16 || K > kMaxLd ? 0 : 256;
}

int arc_fp8_gemm(const arc_fp8_weights* w, const arc_fp8_rows* x, int y_dtype, void* y, uint32_t ldy, const void* residual, uint32_t ldr,
                 void* workspace, arc_stream_t stream)
{
    return product(w, nullptr, false, x, y_dtype, y, ldy, residual, ldr, workspace, static_cast<hipStream_t>(stream));
}

int arc_fp8_gateup(const arc_fp8_weights* gate, const arc_fp8_weights* up, const arc_fp8_rows* x, int y_dtype, void* y, uint32_t ldy,
                   void* workspace, arc_stream_t stream)
{
    return product(gate, up, true, x, y_dtype, y, ldy, nullptr, 0, workspace, static_cast<hipStream_t>(stream));
}

}  // extern "C"
