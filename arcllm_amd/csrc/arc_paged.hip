// arc_paged.hip -- a serving step over a paged KV cache: the step's plan (block
// tables, slots, positions from request lengths) and bias + rotary positions with
// the write into the pages.  The attention over the pages is arc_paged_attn.hip.
#include "arc_paged.hpp"

#include <cmath>

namespace arc {
namespace {

// -------------------------------------------------------------------- plan
struct PlanArgs {
    const uint32_t *old_lens, *new_lens;
    uint32_t* free_pages;
    const uint32_t* free_count;
    uint32_t *free_count_out, *status;
    uint32_t *tables, *lens, *starts, *positions, *slots;
    uint32_t requests, rows, max_pages, max_new, num_pages, shift;  // page_size = 1 << shift
};

// What one request contributes to the step: new tokens, pages it pops, pages it pushes.
// Whole numbers in doubles, which add up exactly where 32 bits would wrap.
struct PlanPart {
    double fresh, take, back;
};

__device__ __forceinline__ uint32_t pages_of(uint32_t len, uint32_t shift)
{
    return (len >> shift) + ((len & ((1u << shift) - 1u)) != 0u);
}

__device__ __forceinline__ PlanPart plan_part(uint32_t held, uint32_t fresh, uint32_t shift)
{
    if (fresh == ARC_PAGED_RELEASE) return PlanPart{0.0, 0.0, double(pages_of(held, shift))};
    return PlanPart{double(fresh), double(pages_of(held + fresh, shift) - pages_of(held, shift)), 0.0};
}

// The last i < n with at[i] <= x, for at ascending with at[0] <= x.
__device__ __forceinline__ uint32_t last_at_most(const uint32_t* at, uint32_t n, uint32_t x)
{
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The same over N entries in LDS, without branches: searches for several items run side by side.
template <uint32_t N>
__device__ __forceinline__ uint32_t last_at_most(const uint32_t (&at)[N], uint32_t x)
{
    static_assert((N & (N - 1)) == 0, "a power of two");
    uint32_t lo = 0;
#pragma unroll
    for (uint32_t step = N / 2; step; step >>= 1) lo += at[lo + step] <= x ? step : 0u;
    return lo;
}

// A block of NT requests, thread by thread: exclusive prefix sums of their parts.
template <int NT>
struct PlanBlock {
    double sums[3][NT / kWave];
    uint32_t bad[NT / kWave];
    uint32_t held[NT], fresh[NT], take[NT], back[NT];
};

// Prefix sums of p over the workgroup; `all` gets the sums, bad what any thread had.
template <int NT>
__device__ __forceinline__ PlanPart block_prefix(const PlanPart& p, PlanBlock<NT>& s, PlanPart& all, uint32_t& bad)
{
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const PlanPart inc{wave_inclusive(p.fresh), wave_inclusive(p.take), wave_inclusive(p.back)};
    const uint32_t any = (__ballot(bad & ARC_PLAN_MAX_NEW) ? ARC_PLAN_MAX_NEW : 0u) | (__ballot(bad & ARC_PLAN_TABLE) ? ARC_PLAN_TABLE : 0u);
    __syncthreads();  // the sums and prefixes before are read no more
    if (lane == 63) {
        s.sums[0][wave] = inc.fresh;
        s.sums[1][wave] = inc.take;
        s.sums[2][wave] = inc.back;
        s.bad[wave] = any;
    }
    __syncthreads();
    PlanPart before{inc.fresh - p.fresh, inc.take - p.take, inc.back - p.back};
    all = PlanPart{0.0, 0.0, 0.0};
#pragma unroll
    for (uint32_t i = 0; i < NT / kWave; ++i) {
        if (i < wave) {
            before.fresh += s.sums[0][i];
            before.take += s.sums[1][i];
            before.back += s.sums[2][i];
        }
        all.fresh += s.sums[0][i];
        all.take += s.sums[1][i];
        all.back += s.sums[2][i];
        bad |= s.bad[i];
    }
    return before;
}

// n items over the workgroup's threads, 4 at a time each: the loads of all four before the first store, so
// that their latencies are one.  get(k) reads item k, put(k, x) stores it.
template <int NT, typename Get, typename Put>
__device__ __forceinline__ void deal(uint32_t n, Get get, Put put)
{
    for (uint32_t k0 = threadIdx.x; k0 < n; k0 += 4 * NT) {
        uint2 x[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (k0 + i * NT < n) x[i] = get(k0 + i * NT);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (k0 + i * NT < n) put(k0 + i * NT, x[i]);
    }
}

// The plan by one workgroup: the requests in blocks of NT, a thread each.  First the step's totals and every
// check, before anything is written; then pages, table entries and rows are dealt out evenly over the
// threads from the prefix sums (a binary search in LDS finds an item's request), so that one long request costs
// no more than many short ones.  A row whose page is new takes it from the stack itself, as the table entry's
// writer does, so no row waits for a table entry.  ROWS: the rows too; else k_plan_rows writes them.
// Bound by the latency of three dependent loads (lengths, an ended request's entries, the stack) and
// the barriers: 24 requests 4.0 us, 700 with 60 prompts and 43000 rows 9.6 us and 3.9 us in
// k_plan_rows, of which an empty launch is 2.2.
template <int NT, bool ROWS>
__global__ __launch_bounds__(NT) void k_plan(PlanArgs a)
{
    __shared__ PlanBlock<NT> s;
    const uint32_t tid = threadIdx.x;
    const uint32_t blocks = (a.requests + NT - 1) / NT;
    const uint32_t count = *a.free_count;
    const uint64_t most = min(uint64_t(a.max_pages) << a.shift, uint64_t(0x7fffffffu));
    uint32_t bad = 0, len = 0, fresh = 0;
    PlanPart p{}, before{}, total{};
    auto read = [&](uint32_t block) {
        const uint32_t b = block * NT + tid;
        len = b < a.requests ? a.old_lens[b] : 0u;
        fresh = b < a.requests ? a.new_lens[b] : 0u;
    };
    for (uint32_t i = 0; i < blocks; ++i) {
        read(i);
        const bool ended = fresh == ARC_PAGED_RELEASE;
        const uint32_t bad_before = bad;
        if (!ended && fresh > a.max_new) bad |= ARC_PLAN_MAX_NEW;
        if (uint64_t(len) + (ended ? 0u : fresh) > most) bad |= ARC_PLAN_TABLE;
        p = bad == bad_before ? plan_part(len, fresh, a.shift) : PlanPart{};
        PlanPart all;
        before = block_prefix<NT>(p, s, all, bad);
        total.fresh += all.fresh;
        total.take += all.take;
        total.back += all.back;
    }
    double lacking = 0.0;
    if (!bad) {
        if (total.fresh > double(a.rows)) bad |= ARC_PLAN_TOKENS;
        if (count + total.back > double(a.num_pages)) bad |= ARC_PLAN_FREE_LIST;
        else if (total.take > count + total.back) {
            bad |= ARC_PLAN_NO_PAGES;
            lacking = total.take - (count + total.back);
        }
    }
    if (bad) {
        for (uint32_t b = tid; b < a.requests; b += NT) {
            a.lens[b] = a.old_lens[b];
            a.starts[b] = 0;
        }
        if (tid == 0) {
            a.starts[a.requests] = 0;
            *a.free_count_out = count;
            a.status[0] = bad;
            a.status[1] = uint32_t(fmin(lacking, 4294967295.0));
            a.status[2] = a.status[3] = 0;
        }
        if constexpr (ROWS)
            for (uint32_t n = tid; n < a.rows; n += NT) {
                a.positions[n] = 0;
                a.slots[n] = ARC_NO_SLOT;
            }
        return;
    }

    // every total fits 32 bits from here on
    const uint32_t top = count + uint32_t(total.back);
    auto publish = [&]() {  // this block's prefixes, for the searches
        s.held[tid] = len;
        s.fresh[tid] = uint32_t(before.fresh);
        s.take[tid] = uint32_t(before.take);
        s.back[tid] = uint32_t(before.back);
        __syncthreads();
    };
    auto block_of = [&](uint32_t i) {  // reads block i again, where there is more than one
        if (blocks == 1) return PlanPart{total.fresh, total.take, total.back};
        read(i);
        p = plan_part(len, fresh, a.shift);
        PlanPart all;
        uint32_t none = 0;
        before = block_prefix<NT>(p, s, all, none);
        return all;
    };
    if (blocks == 1) publish();
    // pages of ended requests onto the stack, before any are popped
    if (total.back > 0.0) {
        uint32_t done = 0;
        for (uint32_t i = 0; i < blocks; ++i) {
            const uint32_t pages = uint32_t(block_of(i).back);
            if (blocks > 1) publish();
            deal<NT>(
                pages,
                [&](uint32_t k) {
                    const uint32_t j = last_at_most(s.back, k);
                    return make_uint2(a.tables[uint64_t(i * NT + j) * a.max_pages + (k - s.back[j])], 0u);
                },
                [&](uint32_t k, uint2 x) { a.free_pages[count + done + k] = x.x; });
            done += pages;
        }
        __syncthreads();
    }
    uint32_t popped = 0, row = 0;
    for (uint32_t i = 0; i < blocks; ++i) {
        const PlanPart all = block_of(i);
        if (blocks > 1) publish();
        const uint32_t b = i * NT + tid, pages = uint32_t(all.take), rows = uint32_t(all.fresh);
        deal<NT>(
            pages, [&](uint32_t k) { return make_uint2(a.free_pages[top - 1u - popped - k], last_at_most(s.take, k)); },
            [&](uint32_t k, uint2 x) {
                a.tables[uint64_t(i * NT + x.y) * a.max_pages + pages_of(s.held[x.y], a.shift) + (k - s.take[x.y])] = x.x;
            });
        if (b < a.requests) {  // every read of old_lens is done: lens may be the same
            a.lens[b] = fresh == ARC_PAGED_RELEASE ? 0u : len + fresh;
            a.starts[b] = row + uint32_t(before.fresh);
        }
        if constexpr (ROWS)
            deal<NT>(
                rows,
                [&](uint32_t k) {
                    const uint32_t j = last_at_most(s.fresh, k), pos = s.held[j] + (k - s.fresh[j]);
                    const uint32_t entry = pos >> a.shift, had = pages_of(s.held[j], a.shift);
                    const uint32_t page = entry < had ? a.tables[uint64_t(i * NT + j) * a.max_pages + entry]
                                                      : a.free_pages[top - 1u - popped - s.take[j] - (entry - had)];
                    return make_uint2(page, pos);
                },
                [&](uint32_t k, uint2 x) {
                    a.positions[row + k] = x.y;
                    a.slots[row + k] = (x.x << a.shift) | (x.y & ((1u << a.shift) - 1u));
                });
        popped += pages;
        row += rows;
    }
    if (tid == 0) {
        a.starts[a.requests] = row;
        *a.free_count_out = top - popped;
        a.status[0] = a.status[1] = 0;
        a.status[2] = row;
        a.status[3] = popped;
    }
    if constexpr (ROWS)
        for (uint32_t n = row + tid; n < a.rows; n += NT) {
            a.positions[n] = 0;
            a.slots[n] = ARC_NO_SLOT;
        }
}

// The rows of a large step, one per thread, from the starts, lengths and tables that k_plan left.  IN_LDS: all
// starts, for the search, while they fit 16 KB: 700 requests, the call 11.2 us instead of 12.1; 1500, 19.0 and 19.4; at the
// limit their copy costs what it saves (4000: 30.8, from memory 29.1), and beyond more (8000: 54.4 and 49.0).
constexpr uint32_t kStartsInLds = 4096;
template <bool IN_LDS>
__global__ __launch_bounds__(256) void k_plan_rows(PlanArgs a)
{
    __shared__ uint32_t own[IN_LDS ? kStartsInLds : 1];
    const uint32_t n = blockIdx.x * 256 + threadIdx.x;
    if constexpr (IN_LDS) {
        for (uint32_t b = threadIdx.x; b <= a.requests; b += 256) own[b] = a.starts[b];
        __syncthreads();
    }
    const uint32_t* starts = IN_LDS ? own : a.starts;
    if (n >= a.rows) return;
    if (n >= starts[a.requests]) {
        a.positions[n] = 0;
        a.slots[n] = ARC_NO_SLOT;
        return;
    }
    const uint32_t b = last_at_most(starts, a.requests, n), pos = a.lens[b] - (starts[b + 1] - n);
    a.positions[n] = pos;
    a.slots[n] = (a.tables[uint64_t(b) * a.max_pages + (pos >> a.shift)] << a.shift) | (pos & ((1u << a.shift) - 1u));
}

// Rows that one workgroup writes itself; more go to a launch of their own.  24 requests, 1000, 4000 and 8000 rows: 7.3, 8.7
// and 10.2 us in one launch, 9.3 to 9.4 in two; one row a request: 3000 in 20.9 and 25.1, 6000 in 40.8 and 39.2.
constexpr uint32_t kPlanRowsInOne = 4096;

void launch_plan(const PlanArgs& a, hipStream_t st)
{
    if (a.rows > kPlanRowsInOne) hipLaunchKernelGGL((k_plan<1024, false>), dim3(1), dim3(1024), 0, st, a);
    // a small step: 4 waves, whose barriers cost less than 16 waves': 24 requests 4.7 us instead of 7.3, 256 5.0 instead
    // of 7.4, 900 rows 4.8 instead of 7.2; 512 requests are more than a thread's each (6.7 and 7.3), 1000 11.4 and 7.5
    else if (a.requests <= 256 && a.rows <= 1024) hipLaunchKernelGGL((k_plan<256, true>), dim3(1), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_plan<1024, true>), dim3(1), dim3(1024), 0, st, a);
}

// -------------------------------------------------------------------- rope
struct RopeArgs {
    const void* x;
    const float *qb, *kb, *vb;
    const uint64_t* phases;
    const uint32_t *positions, *slots;
    void *q, *k, *v;
    uint64_t page_stride;
    uint32_t rows, ldx, ldq, heads, kv_heads, dim, rot, half, shift, num_slots;
    float scale;
};

// The pair (x, y) turned by position * phase turns, times scale: the product modulo 2^64 is the angle's
// fraction of a turn exactly; its upper 32 bits, as a signed number, are in [-1/2, 1/2) and round to
// fp32 with an error of at most 2^-26 turns.
__device__ __forceinline__ void rotate(uint32_t pos, uint64_t phase, float scale, float& x, float& y)
{
    const float half_turns = float(int32_t((uint64_t(pos) * phase) >> 32)) * 0x1p-31f;
    float s, c;
    sincospif(half_turns, &s, &c);
    c *= scale;
    s *= scale;
    const float tx = x * c - y * s, ty = x * s + y * c;
    x = tx;
    y = ty;
}

template <typename X>
__device__ __forceinline__ void load4(const X* p, float* f)
{
    const vec4<X> v = *reinterpret_cast<const vec4<X>*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = static_cast<float>(v[i]);
}

// One lane: 8 values of one head of one row, as two groups of 4 that are loaded, rotated and stored together.
// Half layout: i .. i + 3 and their partners i + rot / 2 ..; values that are not rotated, and
// the interleaved layout, whose groups are 2 pairs each: a group of the head's first half and one of its
// second (of what is left of them), so that neighbouring lanes load neighbouring 16 bytes.  Every lane computes
// its own 4 angles: about 150 instructions against 48 bytes moved, which the memory time of a large
// step covers, and a small one waits for no barrier.  Bound by HBM: N (heads + 2 kv_heads) dim
// values read and written once; 8192 rows of 36 heads of 128, fp32 to fp16 (201 MB): 46 us with other inputs in each call,
// 4.4 TB/s, where a copy reaches 4.7 (35.6 us with one input over and over, part of which the last cache then holds).
template <typename X, typename T>
__device__ __forceinline__ void rope_unit(const RopeArgs& a, uint32_t n, uint32_t u, uint32_t slot, uint32_t pos)
{
    const uint32_t per = a.dim / 8, head = u / per, e = u - head * per;
    const bool is_v = head >= a.heads + a.kv_heads;
    const uint32_t rot = is_v ? 0u : a.rot;
    const bool halves = a.half && 8 * e < rot;
    const uint32_t skip = a.half && !halves ? rot : 0u;  // the half layout's rotated part, before the others
    const uint32_t i0 = skip + 4 * (e - skip / 8), i1 = i0 + (halves ? rot : a.dim - skip) / 2;

    const X* src = static_cast<const X*>(a.x) + uint64_t(n) * a.ldx + head * a.dim;
    float lo[4], hi[4];
    load4(src + i0, lo);
    load4(src + i1, hi);
    T* dst;
    const float* bias;
    uint32_t own = head;  // the head's index among q, k or v
    if (head < a.heads) {
        dst = static_cast<T*>(a.q) + uint64_t(n) * a.ldq + head * a.dim;
        bias = a.qb;
    } else {
        own -= is_v ? a.heads + a.kv_heads : a.heads;
        const uint64_t at = uint64_t(slot >> a.shift) * a.page_stride +
                            uint64_t(slot & ((1u << a.shift) - 1u)) * (a.kv_heads * a.dim) + own * a.dim;
        dst = static_cast<T*>(is_v ? a.v : a.k) + at;
        bias = is_v ? a.vb : a.kb;
    }
    if (bias) {
        float b0[4], b1[4];
        load4(bias + own * a.dim + i0, b0);
        load4(bias + own * a.dim + i1, b1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            lo[i] += b0[i];
            hi[i] += b1[i];
        }
    }
    if (halves) {
#pragma unroll
        for (int i = 0; i < 4; ++i) rotate(pos, a.phases[i0 + i], a.scale, lo[i], hi[i]);
    } else if (!a.half) {
        if (i0 < rot) {
            rotate(pos, a.phases[i0 / 2], a.scale, lo[0], lo[1]);
            rotate(pos, a.phases[i0 / 2 + 1], a.scale, lo[2], lo[3]);
        }
        if (i1 < rot) {
            rotate(pos, a.phases[i1 / 2], a.scale, hi[0], hi[1]);
            rotate(pos, a.phases[i1 / 2 + 1], a.scale, hi[2], hi[3]);
        }
    }
    vec4<T> o0, o1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o0[i] = static_cast<T>(lo[i]);
        o1[i] = static_cast<T>(hi[i]);
    }
    *reinterpret_cast<vec4<T>*>(dst + i0) = o0;
    *reinterpret_cast<vec4<T>*>(dst + i1) = o1;
}

template <typename X, typename T>
__global__ __launch_bounds__(256) void k_rope_append(RopeArgs a)
{
    const uint32_t units = (a.heads + 2 * a.kv_heads) * (a.dim / 8);
    const uint32_t u = blockIdx.x * blockDim.x + threadIdx.x;
    if (u >= units) return;
    for (uint32_t n = blockIdx.y; n < a.rows; n += gridDim.y) {
        const uint32_t slot = a.slots[n];
        if (slot < a.num_slots) rope_unit<X, T>(a, n, u, slot, a.positions[n]);
    }
}

constexpr uint32_t kRopeGridRows = 32768;  // a grid's second dimension holds 65535
constexpr uint32_t kCardWaves = 8192;      // that are resident at once: 8 for each of 1024 SIMDs

template <typename X>
void launch_rope_x(const RopeArgs& a, int dtype, hipStream_t st)
{
    const uint32_t units = (a.heads + 2 * a.kv_heads) * (a.dim / 8);
    // Threads: as many per workgroup as leave the fewest without a unit.  Rows: one per workgroup while the card
    // holds them all at once, then two (and more past the grid's limit), which halves the workgroups to start: 8192
    // rows of 36 heads of 128 53 -> 48.5 us, 16000 bf16 rows of 20 heads 75 -> 47.5, 1500 of 36 10.9 -> 10.2; three or
    // four rows: no better.
    uint32_t threads = 256;
    for (uint32_t t = 192; t >= 64; t -= 64)
        if ((units + t - 1) / t * t < (units + threads - 1) / threads * threads) threads = t;
    const uint64_t waves = uint64_t(a.rows) * ((units + 63) / 64);
    const uint32_t rows = waves <= kCardWaves ? a.rows : (a.rows + 1) / 2;
    const dim3 grid((units + threads - 1) / threads, rows < kRopeGridRows ? rows : kRopeGridRows);
    if (dtype == ARC_F16) hipLaunchKernelGGL((k_rope_append<X, _Float16>), grid, dim3(threads), 0, st, a);
    else hipLaunchKernelGGL((k_rope_append<X, bf16>), grid, dim3(threads), 0, st, a);
}

}  // namespace
}  // namespace arc

using namespace arc;

extern "C" {

int arc_paged_plan(const arc_paged_batch* batch, const uint32_t* old_lens, const uint32_t* new_lens,
                   uint32_t page_size, uint32_t* free_pages, uint32_t num_pages, const uint32_t* free_count,
                   uint32_t* free_count_out, uint32_t* status, arc_stream_t stream)
{
    int rc = check_batch_sizes(batch);
    if (!rc) rc = check_page_size(page_size);
    if (!rc) rc = check_tables(batch, page_size);
    if (rc) return rc;
    if (!old_lens || !new_lens || !free_pages || !free_count || !free_count_out || !status ||
        (batch->tokens && (!batch->positions || !batch->slots)))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "null argument");
    if (num_pages == 0 || uint64_t(num_pages) * page_size >= (1ull << 32))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "num_pages %u: at least 1, num_pages * page_size below 2^32", num_pages);
    if (batch->lens == new_lens) return set_error(ARC_ERR_INVALID_ARGUMENT, "lens may be old_lens, not new_lens");
    PlanArgs a{};
    a.old_lens = old_lens;
    a.new_lens = new_lens;
    a.free_pages = free_pages;
    a.free_count = free_count;
    a.free_count_out = free_count_out;
    a.status = status;
    a.tables = batch->tables;
    a.lens = batch->lens;
    a.starts = batch->starts;
    a.positions = batch->positions;
    a.slots = batch->slots;
    a.requests = batch->requests;
    a.rows = batch->tokens;
    a.max_pages = batch->max_pages;
    a.max_new = batch->max_new;
    a.num_pages = num_pages;
    a.shift = log2_of(page_size);
    hipStream_t st = static_cast<hipStream_t>(stream);
    launch_plan(a, st);
    if ((rc = check_hip(hipGetLastError(), "step plan")) || a.rows <= kPlanRowsInOne) return rc;
    const dim3 grid((a.rows + 255) / 256);
    if (a.requests < kStartsInLds) hipLaunchKernelGGL(k_plan_rows<true>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_plan_rows<false>, grid, dim3(256), 0, st, a);
    return check_hip(hipGetLastError(), "step rows");
}

int arc_rope_phases(uint32_t rot_dim, double theta, int scaling, double factor, uint32_t original_ctx,
                    double beta_fast, double beta_slow, const float* freq_factors, uint64_t* phases, float* scale)
{
    if (!phases || !scale) return set_error(ARC_ERR_INVALID_ARGUMENT, "null phases or scale");
    if (rot_dim == 0 || rot_dim % 8 || rot_dim > 128)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "rot_dim %u: a multiple of 8, at most 128", rot_dim);
    if (!(theta > 1.0) || !std::isfinite(theta)) return set_error(ARC_ERR_INVALID_ARGUMENT, "theta must be above 1");
    if (scaling != ARC_ROPE_PLAIN && scaling != ARC_ROPE_LINEAR && scaling != ARC_ROPE_YARN)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "scaling %d", scaling);
    if (scaling != ARC_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor)))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "factor must be at least 1");
    const uint32_t n = rot_dim / 2;
    const long double pi = 3.14159265358979323846264338L;
    long double low = 0.0, high = 0.0;
    if (scaling == ARC_ROPE_YARN) {
        if (beta_fast == 0.0) beta_fast = 32.0;
        if (beta_slow == 0.0) beta_slow = 1.0;
        if (original_ctx == 0 || !(beta_slow > 0.0) || !(beta_fast >= beta_slow) || !std::isfinite(beta_fast))
            return set_error(ARC_ERR_INVALID_ARGUMENT, "YaRN: original_ctx at least 1, 0 < beta_slow <= beta_fast");
        // the pair index that turns beta times within original_ctx positions
        auto at = [&](double beta) {
            return rot_dim * std::log(original_ctx / (beta * 2.0L * pi)) / (2.0L * std::log((long double)(theta)));
        };
        low = std::fmax(std::floor(at(beta_fast)), 0.0L);
        high = std::fmin(std::ceil(at(beta_slow)), (long double)(rot_dim) - 1.0L);
    }
    // in 64-bit mantissas: a double's 53 bits would cost the far positions
    for (uint32_t i = 0; i < n; ++i) {
        long double f = std::pow((long double)(theta), -2.0L * i / rot_dim);
        if (scaling == ARC_ROPE_LINEAR) f /= factor;
        if (scaling == ARC_ROPE_YARN) {
            const long double ramp = std::fmin(std::fmax((i - low) / std::fmax(high - low, 0.001L), 0.0L), 1.0L);
            f = f * (1.0L - ramp) + f / factor * ramp;
        }
        if (freq_factors) {
            if (!(freq_factors[i] > 0.0f) || !std::isfinite(freq_factors[i]))
                return set_error(ARC_ERR_INVALID_ARGUMENT, "freq_factors[%u] must be positive", i);
            f /= freq_factors[i];
        }
        long double t = f / (2.0L * pi);
        t = std::rint(std::ldexp(t - std::floor(t), 64));
        phases[i] = t < 0x1p64L ? uint64_t(t) : 0u;
    }
    *scale = scaling == ARC_ROPE_YARN ? float(0.1 * std::log(factor) + 1.0) : 1.0f;
    return ARC_OK;
}

int arc_rope_append(const arc_kv_pages* pages, const arc_paged_batch* batch, const arc_rope* rope, int x_dtype,
                    const void* x, uint32_t ldx, const float* q_bias, const float* k_bias, const float* v_bias,
                    uint32_t hpk, void* q, uint32_t ldq, arc_stream_t stream)
{
    int rc = check_pages(pages);
    if (!rc) rc = check_batch_sizes(batch);
    if (rc) return rc;
    if (!rope || !rope->phases || !x || !q || (batch->tokens && (!batch->positions || !batch->slots)))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "null argument");
    if (x_dtype != ARC_F32 && x_dtype != ARC_F16 && x_dtype != ARC_BF16)
        return set_error(ARC_ERR_UNSUPPORTED, "x is ARC_F32, ARC_F16 or ARC_BF16 (dtype %d)", x_dtype);
    if (hpk == 0 || hpk > 64) return set_error(ARC_ERR_UNSUPPORTED, "hpk %u: 1..64 are supported", hpk);
    if (rope->rot_dim == 0 || rope->rot_dim % 8 || rope->rot_dim > pages->head_dim)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "rot_dim %u: a multiple of 8, at most head_dim %u", rope->rot_dim,
                         pages->head_dim);
    if (rope->layout != ARC_ROPE_INTERLEAVED && rope->layout != ARC_ROPE_HALF)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "rope layout %d", rope->layout);
    const uint32_t heads = pages->kv_heads * hpk, dim = pages->head_dim;
    const uint32_t cols = (heads + 2 * pages->kv_heads) * dim;
    if (ldx < cols || ldx % 8) return set_error(ARC_ERR_INVALID_ARGUMENT, "ldx %u: a multiple of 8, at least %u", ldx, cols);
    if (ldq < heads * dim || ldq % 8)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "ldq %u: a multiple of 8, at least %u", ldq, heads * dim);
    if (!aligned(x, 16) || !aligned(q, 16) || !aligned(rope->phases, 8) || !aligned(q_bias, 16) || !aligned(k_bias, 16) ||
        !aligned(v_bias, 16))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "x, q and the biases must be 16-byte aligned, the phases 8-byte");
    const uint64_t xs = x_dtype == ARC_F32 ? 4 : 2;
    if (rows_overlap(x, cols * xs, ldx * xs, q, uint64_t(heads) * dim * 2, uint64_t(ldq) * 2, batch->tokens))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "x and q share memory");
    if (batch->tokens == 0) return ARC_OK;
    RopeArgs a{};
    a.x = x;
    a.qb = q_bias;
    a.kb = k_bias;
    a.vb = v_bias;
    a.phases = rope->phases;
    a.positions = batch->positions;
    a.slots = batch->slots;
    a.q = q;
    a.k = pages->k;
    a.v = pages->v;
    a.page_stride = pages->page_stride;
    a.rows = batch->tokens;
    a.ldx = ldx;
    a.ldq = ldq;
    a.heads = heads;
    a.kv_heads = pages->kv_heads;
    a.dim = dim;
    a.rot = rope->rot_dim;
    a.half = rope->layout == ARC_ROPE_HALF;
    a.shift = log2_of(pages->page_size);
    a.num_slots = pages->num_pages * pages->page_size;
    a.scale = rope->scale;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (x_dtype == ARC_F32) launch_rope_x<float>(a, pages->dtype, st);
    else if (x_dtype == ARC_F16) launch_rope_x<_Float16>(a, pages->dtype, st);
    else launch_rope_x<bf16>(a, pages->dtype, st);
    return check_hip(hipGetLastError(), "rope and cache write");
}

}  // extern "C"
