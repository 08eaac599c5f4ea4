// arc_paged.hpp -- what the paged-cache entry points share: the checks of their
// structs, element types and the address of a cached position.
#pragma once

#include "arc_device.hpp"
#include "../../include/arcllm_hip.h"

#include <utility>

namespace arc {

constexpr uint32_t kMaxRequests = 1u << 20;
constexpr uint32_t kMaxStepRows = 1u << 24;
constexpr uint64_t kMaxPositions = 1ull << 31;  // positions of a request stay below

typedef __bf16 bf16;
template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));
template <typename T>
using vec4 = T __attribute__((ext_vector_type(4)));

// v of the lane that a DPP row operation names, 0 where that is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(u)), CTRL, ROWS, 0xf, false));
    const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(u >> 32)), CTRL, ROWS, 0xf, false));
    return __builtin_bit_cast(double, (uint64_t(hi) << 32) | lo);
}
// Inclusive prefix sums over the wave: in each row of 16 lanes, then row 0's and 2's totals into rows 1
// and 3, then the lower half's into the upper.
__device__ __forceinline__ double wave_inclusive(double v)
{
    v += dpp_f64<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
    v += dpp_f64<0x112, 0xf>(v);
    v += dpp_f64<0x114, 0xf>(v);
    v += dpp_f64<0x118, 0xf>(v);
    v += dpp_f64<0x142, 0xa>(v);  // row_bcast 15
    v += dpp_f64<0x143, 0xc>(v);  // row_bcast 31
    return v;
}

inline bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Whether `rows` rows of `width` bytes, `stride` apart, at a and at b share memory:
// by columns where the strides agree, else by the ranges that they span.
inline bool rows_overlap(const void* a, uint64_t wa, uint64_t sa, const void* b, uint64_t wb, uint64_t sb, uint64_t rows)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    if (rows == 0 || x + (rows - 1) * sa + wa <= y || y + (rows - 1) * sb + wb <= x) return false;
    if (sa != sb) return true;
    const uint64_t d = (x > y ? x - y : y - x) % sa;  // b's columns behind a's, or a's behind b's
    const uint64_t first = x > y ? wb : wa, second = x > y ? wa : wb;
    return d < first || d + second > sa;
}

// `rows` rows of `width` bytes, `stride` apart.
struct Rows2d {
    const void* p;
    uint64_t rows, width, stride;
};
inline Rows2d bytes_at(const void* p, uint64_t bytes) { return Rows2d{p, bytes ? 1u : 0u, bytes, bytes}; }

// Whether two such arrays share memory, gaps between their rows left out: where both have gaps, the one of fewer rows is
// looked at row by row (of more than 2^15 rows each, by their spans).
inline bool overlap(Rows2d a, Rows2d b)
{
    if (!a.p || !b.p || !a.rows || !b.rows || !a.width || !b.width) return false;
    auto begin = [](const Rows2d& r) { return reinterpret_cast<uintptr_t>(r.p); };
    auto end = [&](const Rows2d& r) { return begin(r) + (r.rows - 1) * r.stride + r.width; };
    if (end(a) <= begin(b) || end(b) <= begin(a)) return false;
    if (a.rows > b.rows) std::swap(a, b);
    if (a.rows > 1 && a.width == a.stride) a = bytes_at(a.p, a.rows * a.stride);
    if (b.width >= b.stride) b = bytes_at(b.p, end(b) - begin(b));
    if (a.rows > 1u << 15) return true;
    for (uint64_t i = 0; i < a.rows; ++i) {
        const uintptr_t x0 = begin(a) + i * a.stride, x1 = x0 + a.width;
        // the first row of b that ends behind x0
        const uint64_t first = x0 < begin(b) + b.width ? 0 : (x0 - begin(b) - b.width) / b.stride + 1;
        if (first < b.rows && begin(b) + first * b.stride < x1) return true;
    }
    return false;
}

inline uint32_t log2_of(uint32_t pow2) { return uint32_t(__builtin_ctz(pow2)); }

inline int check_page_size(uint32_t page_size)
{
    if (page_size == 0 || page_size > 65536 || (page_size & (page_size - 1)))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "page_size %u must be a power of two, at most 65536", page_size);
    return ARC_OK;
}

inline int check_pages(const arc_kv_pages* p)
{
    if (!p || !p->k || !p->v) return set_error(ARC_ERR_INVALID_ARGUMENT, "null pages");
    if (int rc = check_page_size(p->page_size)) return rc;
    if (p->kv_heads == 0 || p->kv_heads > 256)
        return set_error(ARC_ERR_UNSUPPORTED, "kv_heads %u: 1..256 are supported", p->kv_heads);
    if (p->head_dim != 64 && p->head_dim != 128)
        return set_error(ARC_ERR_UNSUPPORTED, "head_dim %u: 64 and 128 are supported", p->head_dim);
    if (p->dtype != ARC_F16 && p->dtype != ARC_BF16)
        return set_error(ARC_ERR_UNSUPPORTED, "pages hold ARC_F16 or ARC_BF16 (dtype %d)", p->dtype);
    if (p->num_pages == 0 || uint64_t(p->num_pages) * p->page_size >= (1ull << 32))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "num_pages %u: at least 1, num_pages * page_size below 2^32",
                         p->num_pages);
    const uint64_t page = uint64_t(p->page_size) * p->kv_heads * p->head_dim;
    if (p->page_stride < page || p->page_stride % 8 || p->page_stride > (1ull << 40))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "page_stride %llu: a multiple of 8, at least %llu, at most 2^40",
                         static_cast<unsigned long long>(p->page_stride), static_cast<unsigned long long>(page));
    if (!aligned(p->k, 16) || !aligned(p->v, 16))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "k and v pages must be 16-byte aligned");
    return ARC_OK;
}

inline int check_batch_sizes(const arc_paged_batch* b)
{
    if (!b) return set_error(ARC_ERR_INVALID_ARGUMENT, "null batch");
    if (b->requests > kMaxRequests || b->tokens > kMaxStepRows)
        return set_error(ARC_ERR_UNSUPPORTED, "%u requests, %u rows: at most 2^20 and 2^24", b->requests, b->tokens);
    return ARC_OK;
}

inline int check_tables(const arc_paged_batch* b, uint32_t page_size)
{
    if (!b->tables || !b->lens || !b->starts) return set_error(ARC_ERR_INVALID_ARGUMENT, "null tables, lens or starts");
    if (b->max_pages == 0 || uint64_t(b->max_pages) * page_size > kMaxPositions)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "max_pages %u: at least 1, max_pages * page_size at most 2^31",
                         b->max_pages);
    return ARC_OK;
}

}  // namespace arc
