// arc_paged_attn.hip -- attention of a serving step's new tokens over the pages of
// their requests (arc_paged.hpp), causal, with an optional sliding window whose
// first tokens stay visible.
#include "arc_paged.hpp"

#include <cmath>

namespace arc {
namespace {

struct PagedAttn {
    const void *q, *k, *v;
    void* out;
    const uint32_t *tables, *lens, *starts;
    uint64_t page_stride;
    uint32_t requests, rows, max_pages, num_pages, shift;
    uint32_t ldq, ldo, kv_heads, hpk, window, sinks;
    float scale;
};

__device__ __forceinline__ uint32_t request_of(const uint32_t* starts, uint32_t requests, uint32_t n)
{
    uint32_t lo = 0, hi = requests;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (starts[mid] <= n) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One wave per row and query head, 64 positions at a time: lane j scores position
// t0 + j, the wave's running maximum and sum are updated, then every lane adds the
// 64 weighted values of its own dims.  Reads K and V once per row and head.
template <typename T, int D>
__global__ __launch_bounds__(64) void k_paged_attn(PagedAttn a)
{
    constexpr int kPer = D / kWave;  // output dims per lane
    __shared__ float qs[D];
    const uint32_t n = blockIdx.x, h = blockIdx.y, g = h / a.hpk, lane = threadIdx.x;
    if (a.requests == 0 || n >= a.starts[a.requests]) return;
    const uint32_t b = request_of(a.starts, a.requests, n);
    const uint32_t behind = a.starts[b + 1] - n;  // this token and those after it
    const uint32_t len = uint32_t(min(uint64_t(a.lens[b]), uint64_t(a.max_pages) << a.shift));
    const int64_t pos = int64_t(len) - int64_t(behind);
    const T* q = static_cast<const T*>(a.q) + uint64_t(n) * a.ldq + h * D;
    for (int d = lane; d < D; d += kWave) qs[d] = static_cast<float>(q[d]) * a.scale;
    __syncthreads();
    const uint32_t* table = a.tables + uint64_t(b) * a.max_pages;
    const uint32_t kvd = a.kv_heads * D;
    float m = -INFINITY, l = 0.0f, o[kPer];
    for (int i = 0; i < kPer; ++i) o[i] = 0.0f;
    for (int64_t t0 = 0; t0 <= pos; t0 += kWave) {
        const int64_t j = t0 + lane;
        const bool seen = j <= pos && (a.window == 0 || pos - j < int64_t(a.window) || j < int64_t(a.sinks));
        const uint32_t page = seen ? table[j >> a.shift] : a.num_pages;
        const bool in = page < a.num_pages;
        const uint64_t at = in ? uint64_t(page) * a.page_stride + (uint64_t(j) & ((1u << a.shift) - 1u)) * kvd + g * D : 0;
        float s = -INFINITY;
        if (in) {
            const T* kp = static_cast<const T*>(a.k) + at;
            s = 0.0f;
            for (int d = 0; d < D; d += 8) {
                const vec8<T> kv = *reinterpret_cast<const vec8<T>*>(kp + d);
#pragma unroll
                for (int e = 0; e < 8; ++e) s = __builtin_fmaf(qs[d + e], static_cast<float>(kv[e]), s);
            }
        }
        const float mn = fmaxf(m, wave_max(s));
        if (mn == -INFINITY) continue;  // nothing seen yet
        const float w = expf(s - mn), al = expf(m - mn);
        l = l * al + group_sum<kWave>(w);
        m = mn;
        for (int i = 0; i < kPer; ++i) o[i] *= al;
        for (int t = 0; t < kWave; ++t) {
            if (!__shfl(int(in), t)) continue;
            const float wt = __shfl(w, t);
            const uint64_t vt = uint64_t(__shfl(static_cast<long long>(at), t));
            const T* vp = static_cast<const T*>(a.v) + vt + lane * kPer;
            for (int i = 0; i < kPer; ++i) o[i] = __builtin_fmaf(wt, static_cast<float>(vp[i]), o[i]);
        }
    }
    T* dst = static_cast<T*>(a.out) + uint64_t(n) * a.ldo + h * D + lane * kPer;
    for (int i = 0; i < kPer; ++i) dst[i] = static_cast<T>(l > 0.0f ? o[i] / l : 0.0f);
}

template <typename T>
hipError_t launch_paged(const PagedAttn& a, uint32_t dim, hipStream_t st)
{
    const dim3 grid(a.rows, a.kv_heads * a.hpk);
    if (dim == 64) hipLaunchKernelGGL((k_paged_attn<T, 64>), grid, dim3(64), 0, st, a);
    else hipLaunchKernelGGL((k_paged_attn<T, 128>), grid, dim3(64), 0, st, a);
    return hipGetLastError();
}

int check_sizes(const arc_kv_pages* pages, const arc_paged_batch* batch, uint32_t hpk)
{
    int rc = check_pages(pages);
    if (!rc) rc = check_batch_sizes(batch);
    if (rc) return rc;
    if (hpk == 0 || hpk > 64) return set_error(ARC_ERR_UNSUPPORTED, "hpk %u: 1..64 are supported", hpk);
    return ARC_OK;
}

}  // namespace
}  // namespace arc

using namespace arc;

extern "C" {

size_t arc_paged_attention_workspace_bytes(const arc_kv_pages* pages, const arc_paged_batch* batch, uint32_t hpk)
{
    return check_sizes(pages, batch, hpk) ? 0 : 256;
}

int arc_paged_attention(const arc_kv_pages* pages, const arc_paged_batch* batch, const void* q, uint32_t ldq,
                        uint32_t hpk, float scale, uint32_t window, uint32_t sinks, void* out, uint32_t ldo,
                        void* workspace, arc_stream_t stream)
{
    int rc = check_sizes(pages, batch, hpk);
    if (!rc) rc = check_tables(batch, pages->page_size);
    if (rc) return rc;
    if (!q || !out || !workspace) return set_error(ARC_ERR_INVALID_ARGUMENT, "null argument");
    const uint32_t width = pages->kv_heads * hpk * pages->head_dim;
    if (ldq < width || ldq % 8 || ldo < width || ldo % 8)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "ldq %u, ldo %u: multiples of 8, at least %u", ldq, ldo, width);
    if (!aligned(q, 16) || !aligned(out, 16)) return set_error(ARC_ERR_INVALID_ARGUMENT, "q and out must be 16-byte aligned");
    if (!aligned(workspace, 256)) return set_error(ARC_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    if (!std::isfinite(scale)) return set_error(ARC_ERR_INVALID_ARGUMENT, "scale must be finite");
    if (rows_overlap(q, uint64_t(width) * 2, uint64_t(ldq) * 2, out, uint64_t(width) * 2, uint64_t(ldo) * 2, batch->tokens))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "q and out share memory");
    if (batch->tokens == 0 || batch->requests == 0) return ARC_OK;
    PagedAttn a{};
    a.q = q;
    a.k = pages->k;
    a.v = pages->v;
    a.out = out;
    a.tables = batch->tables;
    a.lens = batch->lens;
    a.starts = batch->starts;
    a.page_stride = pages->page_stride;
    a.requests = batch->requests;
    a.rows = batch->tokens;
    a.max_pages = batch->max_pages;
    a.num_pages = pages->num_pages;
    a.shift = log2_of(pages->page_size);
    a.ldq = ldq;
    a.ldo = ldo;
    a.kv_heads = pages->kv_heads;
    a.hpk = hpk;
    a.window = window;
    a.sinks = sinks;
    a.scale = scale == 0.0f ? 1.0f / std::sqrt(float(pages->head_dim)) : scale;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = pages->dtype == ARC_F16 ? launch_paged<_Float16>(a, pages->head_dim, st)
                                                 : launch_paged<bf16>(a, pages->head_dim, st);
    return check_hip(e, "paged attention");
}

}  // extern "C"
