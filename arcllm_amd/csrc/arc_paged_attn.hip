// arc_paged_attn.hip -- attention of a serving step's new tokens over the pages of
// their requests (arc_paged.hpp), causal, with an optional sliding window whose
// first tokens stay visible.
//
// Rows.  The hpk query heads of a kv head read the same K and V, so the rows of a
// request and kv head g are its (token, head) pairs, token-major: row r is token
// r / hpk, head g * hpk + r % hpk.  A tile is up to 32 (few) or 32 for each wave (many) of
// them; it runs over the positions that any of them sees, a unit at a time.
//
// Work.  Requests differ in length by orders of magnitude, and the host does not know
// their lengths.  So the tiles of all requests and kv heads stand in one line, each
// with a cost that the device computes from starts and lens, and workgroup w of G takes
// the w-th of G equal parts of the line, cut wherever it falls, inside a tile too.  A
// tile in one part is written out; a part of one leaves its sums in the workspace
// (Piece) and k_paged_join adds the pieces of a tile in order, so results do not
// depend on timing.
//
// Trees (TREE).  A request's rows may be the nodes of a tree of drafted tokens: node i lies at place i behind the
// context, sees all of that (its window's part) and the nodes that its mask names, none of them behind itself.  So a
// tile runs over the same units as a causal one, and only those that reach behind the context look at masks.
#include "arc_paged.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace arc {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr uint32_t kFewRows = 32;      // rows of a few-rows tile
constexpr uint32_t kFewKeys = 32;      // positions of its unit, one wave's
constexpr uint32_t kFewWaves = 4;
constexpr uint32_t kManyKeys = 64;     // positions of a many-rows tile's unit
constexpr uint32_t kFewWgs = 512;      // most parts of the line
// Waves of a many-rows workgroup, 32 rows each, and workgroups that fill the card.  Heads of 128: 8 waves on a CU
// share each unit's copy, where two workgroups of 4 copied it twice: a chunk of 4096 tokens at 12288, 28 heads,
// 880 instead of 950 us (and 1.55 instead of 1.88 million cycles: the rest is the clock, which the matrix
// cores' power holds down).  Heads of 64 leave registers for 3 workgroups of 4 waves.
constexpr int many_waves(uint32_t dim) { return dim == 128 ? 8 : 4; }
constexpr uint32_t many_wgs(uint32_t dim) { return dim == 128 ? 256 : 768; }
// A tile's start and end (pages, first copy, stores), in positions: few rows 3 us, where a part's 32 take 0.5 (300
// requests of up to 1500, 28 heads: 72 us with 64 here, 64 with 192, 60 with 256 to 448; 64 of up to 8000: 57.6, 54.3,
// 54.6); many rows (bm of them) 7 us, where 64 take 1.9 and, with 4 waves, other workgroups of the CU have the time.
constexpr uint32_t tile_ends(bool few, uint32_t bm) { return few ? 256 : bm; }
constexpr float kLazy = 8.0f;          // see rescale
template <typename T>
constexpr float kLift = __is_same(T, _Float16) ? 7.0f : 0.0f;
// A tile in more pieces is joined in another way.  8 (16, 4): a chunk of 500 at 2500, 28 heads of 128, 40 us (42, 56); 700
// at 700, 64 of 64, 28 (30, 44); 100 at 8000, 28 of 128, 47 (51, 45); but 256 at 2000 50 (33, 45), 256 at 8000 70 (52, 65).
constexpr uint32_t kManyPieces = 8;

// What a part of a tile left in the workspace, one per slot; two slots per
// workgroup (its part may end one tile and begin another).
struct Piece {
    uint32_t n, idx;      // pieces of the tile (0: the slot is unused), this one's number
    uint32_t wg, slot;    // workgroup and slot of piece 0; piece i > 0 is in slot 2 (wg + i)
    uint32_t token, row0; // the request's first row of the step, the tile's first row
    uint32_t rows, g;
};

struct PagedAttn {
    const void *q, *k, *v;
    void* out;
    const uint32_t *tables, *lens, *starts;
    uint64_t page_stride;
    uint32_t requests, rows, max_pages, num_pages, shift;
    uint32_t ldq, ldo, kv_heads, hpk, window, sinks;
    uint32_t few_rows;   // requests of at most this many rows (per kv head) go to the few-rows kernel
    float scale;         // |scale| * log2(e)
    uint32_t neg;        // 0x80008000 where scale < 0: q's signs are flipped
    float *few_o, *many_o;    // [2 * workgroups][slot rows][D] sums of pieces
    float2 *few_ml, *many_ml; // [2 * workgroups][slot rows] reference score and sum
    Piece *few_p, *many_p;
    uint32_t few_slot, many_slot;  // rows of a slot
    uint32_t few_wgs, many_wgs;    // workgroups of this call's launches (0: not launched)
};
// Of the TREE kernels.  The others' arguments are 24 bytes and a cache line shorter: one request at 501 positions 11.1 us, not 11.2.
struct TreeAttn : PagedAttn {
    const uint32_t *masks, *positions;
    uint32_t words;
    uint32_t once;  // every tree is one tile: nothing of K and V is read twice
};
template <bool TREE>
using Attn = std::conditional_t<TREE, TreeAttn, PagedAttn>;
__device__ __forceinline__ const TreeAttn& of_tree(const PagedAttn& a) { return static_cast<const TreeAttn&>(a); }

// The kernel's arguments (its one parameter, a PagedAttn or a TreeAttn), read again: a phase that takes its own copy keeps
// none of it in scalar registers for the phases after it.
__device__ __forceinline__ const PagedAttn& arguments()
{
    typedef __attribute__((address_space(4))) const PagedAttn Arg;
    Arg* p = (Arg*)(__builtin_amdgcn_kernarg_segment_ptr());
    asm volatile("" : "+s"(p));
    return *(const PagedAttn*)(p);
}

// ------------------------------------------------------------------- tiles
// One request: its new rows and positions, and what its tiles cost.  Costs are whole
// numbers in doubles (the host keeps them below 2^52), exact and quicker than 64-bit
// integers here.
struct Request {
    uint32_t token;   // first row of the step
    uint32_t rows;    // (token, head) pairs per kv head
    int32_t base;     // position of its first new token (negative: rows without a position)
    uint32_t tiles;   // per kv head
    double first, cap;  // cost of tile 0; no tile costs more than cap
    double total;       // of a kv head's tiles
    // how many units its tiles count for, of a kv head, when a step is cut into parts of a unit (few rows: one for each wave):
    // about as many as they have and no fewer, but of trees fewer in the many-rows kernel (9 to 32 units a tile: a part
    // to several) and in the few-rows kernel as many as a workgroup takes in one turn, or more
    float units;
};

// Cost of tiles 0 .. t-1: tile t costs min(first + t * bm, cap), in positions times
// hpk; causal tiles grow by bm / hpk positions each.
__device__ __forceinline__ double cost_before(const Request& r, uint32_t t, double bm)
{
    const double n = double(t);
    const double k = fmin(n, r.first >= r.cap ? 0.0 : ceil((r.cap - r.first) * (1.0 / bm)));
    return k * r.first + bm * (k * (k - 1.0) * 0.5) + (n > k ? (n - k) * r.cap : 0.0);
}

// Whether a request's rows are a tree, not a chunk.
__device__ __forceinline__ bool is_tree(const PagedAttn& a, const Request& r) { return r.rows <= 32 * of_tree(a).words * a.hpk; }

template <bool TREE, bool FEW, uint32_t bm>
__device__ __forceinline__ Request request_of(const PagedAttn& a, uint32_t s0, uint32_t s1, uint32_t held)
{
    constexpr uint32_t keys = FEW ? kFewKeys : kManyKeys, ends = tile_ends(FEW, bm);
    Request r{};
    if (s1 <= s0 || s0 >= a.rows) return r;
    const uint32_t rows = (min(s1, a.rows) - s0) * a.hpk;
    if (FEW ? rows > a.few_rows : rows <= a.few_rows) return r;
    const uint64_t len = min(uint64_t(held), min(uint64_t(a.max_pages) << a.shift, uint64_t(0x7fffffffu)));
    const int64_t base = int64_t(len) - int64_t(s1 - s0);
    r.token = s0;
    r.rows = rows;
    r.base = int32_t(max(base, -(int64_t(1) << 25)));
    r.tiles = (rows + bm - 1) / bm;
    const bool tree = TREE && is_tree(a, r);  // a step of chunks alone is cut as paged attention cuts it
    // Trees over contexts that a workgroup takes in one turn cost the same, and a part (see below) is no less than one of their
    // tiles: parts then begin where tiles do.  64 of 3 nodes at 30 positions, 28 heads, 11.5 us; else in pieces, 38.
    constexpr uint32_t kTurn = FEW ? kFewWaves * kFewKeys : kManyKeys;
    const uint32_t old = uint32_t(max(r.base, 0));
    r.first = double(ends + (tree ? max(old, kTurn) : old)) * a.hpk + bm;
    r.cap = a.window ? (double(ends) + a.window + a.sinks) * a.hpk + 2 * bm : 0x1p60;
    if (tree && a.window) r.cap += rows;  // the tree lies behind the first node's window
    auto seen = [&] {
        const float all = float(a.window) + float(a.sinks);
        return tree ? all + float(rows / a.hpk) : all;
    };
    r.total = r.tiles == 1 ? fmin(r.first, r.cap) : cost_before(r, r.tiles, bm);
    const float spans = float(r.tiles) * ceilf(float(len) * (1.0f / keys));
    r.units = a.window ? fminf(spans, float(r.tiles) * (ceilf(seen() * (1.0f / keys)) + 2.0f)) : spans;
    if (tree && !FEW) {
        // up to 8 pieces of a tile are joined in the quicker way, worth some 3 units: 26 nodes at 501 positions, 28 heads on 4,
        // 15.2 us (a part to each unit 18.5); 60 nodes 19.6 (27.4); at 1700 18.4 (21.0); 32 heads of 64 on 8 at 1000 13.4 (18.1);
        // from 33 units on a unit a part is as quick or quicker
        const float each = r.units * __builtin_amdgcn_rcpf(float(r.tiles));
        if (each > 8.0f && each < 32.5f) r.units = float(r.tiles) * fmaxf(6.0f, ceilf(each * 0.25f - 0.01f));
    }
    if (tree && FEW) r.units = fmaxf(r.units, float(kFewWaves) * float(r.tiles));
    r.units = fmaxf(r.units, 1.0f);
    return r;
}

// A tile and the positions that it runs over: units of `keys` positions, first
// those of the sinks, then those from the first row's window on.
struct Tile {
    uint32_t row0, rows;
    int32_t pos0, pos1;       // first and last row's position
    uint32_t sink_units, low; // units of sinks before a gap; the first unit after it
    uint32_t units;
};

template <bool TREE>
__device__ __forceinline__ Tile tile_at(const PagedAttn& a, const Request& r, uint32_t t, uint32_t bm, uint32_t keys)
{
    Tile x;
    x.row0 = t * bm;
    x.rows = min(bm, r.rows - x.row0);
    x.pos0 = r.base + int32_t(x.row0 / a.hpk);
    if (TREE && is_tree(a, r)) x.pos0 = r.base - 1;  // what all rows see ends with the context, as do their windows
    x.pos1 = r.base + int32_t((x.row0 + x.rows - 1) / a.hpk);
    const uint32_t end = uint32_t(max(x.pos1 + 1, 0));
    const uint32_t all = (end + keys - 1) / keys;
    x.sink_units = x.low = 0;
    if (a.window && x.pos0 > 0 && uint32_t(x.pos0) >= a.window) {
        const uint32_t low = uint32_t(x.pos0) - a.window + 1;
        x.sink_units = uint32_t((uint64_t(min(a.sinks, low)) + keys - 1) / keys);
        x.low = low / keys;
        if (x.sink_units >= x.low) x.sink_units = x.low = 0;
    }
    x.units = max(1u, x.sink_units + all - x.low);
    return x;
}

__device__ __forceinline__ uint32_t unit_start(const Tile& x, uint32_t u, uint32_t keys)
{
    return (u < x.sink_units ? u : u - x.sink_units + x.low) * keys;
}

// ------------------------------------------------------------------ the line
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return uint32_t(__builtin_amdgcn_readfirstlane(int(v))); }
__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uniform(uint64_t v)
{
    return (uint64_t(uniform(uint32_t(v >> 32))) << 32) | uniform(uint32_t(v));
}
__device__ __forceinline__ double of_lane(double v, int lane)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(u)), lane));
    const uint32_t hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(u >> 32)), lane));
    return __builtin_bit_cast(double, (uint64_t(hi) << 32) | lo);
}
// A workgroup's place in the line and the segment of it that it works on, in LDS:
// wave 0 moves it on, the others read what they need, so that none of it is held in
// registers while a segment is computed.
struct Walk {
    double total, step;    // cost of all tiles, of a part
    double at, to;         // how far this part has come, its end
    double before;         // cost of the requests before b
    uint32_t parts, w, b;
    // the segment: units [u0, u1) of a tile
    uint32_t go;           // 0: the part is done
    uint32_t g, u0, u1, token, slot;
    uint32_t pieces;       // of the tile, 0: the segment is all of it
    int32_t base;
    Tile x;
};

// Boundary of part w, the same number wherever it is computed.  A tile costs far more than one for each unit that it counts
// for, so a part is never empty, though it may hold no whole unit.
__device__ __forceinline__ double part_at(const Walk& l, uint32_t w)
{
    return w >= l.parts ? l.total : floor(l.step * double(w));
}

// Quotients that only have to be near, or the same in every workgroup.
__device__ __forceinline__ float near_ratio(double x, double y) { return float(x) * __builtin_amdgcn_rcpf(float(y)); }

// Which of a tile's units lie before x: monotonic in x, the same for both neighbours
// of a cut (the same arithmetic on the same numbers).  The added 2^-8 keeps cuts that
// should fall on a unit's border on it.
__device__ __forceinline__ uint32_t units_before(double x, double begin, double end, uint32_t units)
{
    if (x <= begin) return 0;
    if (x >= end) return units;
    return min(units, uint32_t((x - begin) * double(near_ratio(units, end - begin)) + 0x1p-8));
}

// The part in which x lies, of the lower lanes' x and of the upper lanes', by the whole wave: near_ratio is off by
// one at most and the boundaries' rounding adds another, so 8 candidates hold it.
__device__ __forceinline__ void parts_of(const Walk& l, double x, uint32_t& lower, uint32_t& upper)
{
    const int32_t w0 = int32_t(min(l.parts - 1, uint32_t(near_ratio(x, l.step)))) - 4;
    const int32_t w = w0 + int32_t(threadIdx.x & 7u);
    const uint64_t from = __ballot(w <= 0 || (uint32_t(w) < l.parts && floor(l.step * double(w)) <= x));
    lower = uint32_t(__builtin_amdgcn_readlane(w0, 0) + __builtin_popcount(uint32_t(from) & 255u) - 1);
    upper = uint32_t(__builtin_amdgcn_readlane(w0, 32) + __builtin_popcount(uint32_t(from >> 32) & 255u) - 1);
}

// This workgroup's part, from the total: parts of a unit (few rows: one for each wave) or more.
// Workgroups go to the 8 XCDs in turn: an XCD's workgroups take neighbouring parts, which read the
// same K and V.
__device__ __forceinline__ void take_part(Walk& l, double total, float units)
{
    l.total = total;
    l.parts = total > 0.0 ? min(uint32_t(gridDim.x), uint32_t(fminf(fmaxf(units, 1.0f), 65536.0f))) : 0u;
    l.step = total * double(__builtin_amdgcn_rcpf(float(max(l.parts, 1u))));  // the last part has what that leaves
    l.w = blockIdx.x;
    l.at = l.to = 0.0;
    if (l.w >= l.parts) return;
    const uint32_t xcd = blockIdx.x & 7u, q = l.parts >> 3, rest = l.parts & 7u;
    l.w = xcd * q + min(xcd, rest) + (blockIdx.x >> 3);
    l.at = part_at(l, l.w);
    l.to = part_at(l, l.w + 1);
}

// The first 64 requests, read once.
struct Heads {
    uint32_t s0[64], s1[64], len[64];
};
template <bool TREE, bool FEW, uint32_t bm>
__device__ __forceinline__ Request request_at(const PagedAttn& a, const Heads& h, uint32_t b)
{
    if (a.requests <= 64) return request_of<TREE, FEW, bm>(a, h.s0[b], h.s1[b], h.len[b]);
    return request_of<TREE, FEW, bm>(a, a.starts[b], a.starts[b + 1], a.lens[b]);
}

// Wave 0: the segment of request r, b of the step, that lies at m.at, and the part's way on.  A cut tile gets its slot
// and its record for k_paged_join.  One wave's work that all others wait for, a chain of dependent steps: so
// searches are by 64 lanes at once, and what is needed twice (of a tile's ends, a part's ends) is computed in the lower
// and the upper lanes.
template <bool TREE, bool FEW, uint32_t bm>
__device__ __forceinline__ void cut_segment(const PagedAttn& a, Walk& m, const Request& r)
{
    constexpr uint32_t keys = FEW ? kFewKeys : kManyKeys;
    const uint32_t lane = threadIdx.x & 63u;
    const bool upper = lane >= 32;
    const double off = m.at - m.before;
    const int32_t g0 = int32_t(min(a.kv_heads - 1, uint32_t(near_ratio(off, r.total)))) - 2, gl = g0 + int32_t(lane & 3u);
    m.g = uint32_t(uniform(g0) + __builtin_popcount(uint32_t(__ballot(gl <= 0 || (uint32_t(gl) < a.kv_heads && gl * r.total <= off))) & 15u) - 1);
    const double start = m.before + m.g * r.total, in = m.at - start;
    uint32_t t = 0;
    double begin = start, end = start + r.total;
    if (r.tiles > 1) {
#pragma unroll 1
        for (uint32_t n = r.tiles; n > 1;) {  // the tile is one of n from t on
            const uint32_t each = (n + 63) / 64, c = lane * each;
            const uint32_t i = uint32_t(__builtin_popcountll(__ballot(c < n && cost_before(r, t + c, bm) <= in))) - 1;
            t += i * each;
            n = min(each, n - i * each);
        }
        const double ends = start + cost_before(r, t + (upper ? 1 : 0), bm);
        begin = of_lane(ends, 0);
        end = of_lane(ends, 32);
    }
    m.x = tile_at<TREE>(a, r, t, bm, keys);
    const uint32_t units = units_before(upper ? m.to : m.at, begin, end, m.x.units);
    m.u0 = uint32_t(__builtin_amdgcn_readlane(int(units), 0));
    m.u1 = uint32_t(__builtin_amdgcn_readlane(int(units), 32));
    m.token = r.token;
    m.base = r.base;
    m.pieces = 0;
    if (m.at > begin || end > m.to) {
        uint32_t w0, w1;
        parts_of(m, upper ? end - 1.0 : begin, w0, w1);
        const uint32_t first = 2 * w0 + (part_at(m, w0) < begin ? 1u : 0u);
        m.slot = m.w == w0 ? first : 2 * m.w;
        m.pieces = w1 - w0 + 1;
        if (lane == 0)
            (FEW ? a.few_p : a.many_p)[m.slot] = Piece{m.pieces, m.w - w0, w0, first, r.token, m.x.row0, m.x.rows, m.g};
    }
    m.at = fmin(end, m.to);
}

// Wave 0: the part's next segment after l's.
template <bool TREE, bool FEW, uint32_t bm>
__device__ __forceinline__ void next_segment(const PagedAttn& a, const Walk& l, Walk& to, const Heads& h)
{
    if (threadIdx.x >= 64) return;
    Walk m = l;
    m.go = m.at < m.to;
    if (m.go) {
        Request r = request_at<TREE, FEW, bm>(a, h, m.b);  // the request at m.at: this one, or one of those behind it
        while (m.at >= m.before + r.total * a.kv_heads) {
            m.before += r.total * a.kv_heads;
            const uint32_t next = ++m.b + threadIdx.x;
            if (next < a.requests) r = request_at<TREE, FEW, bm>(a, h, next);
            const double own = next < a.requests ? r.total * a.kv_heads : 0.0, inc = wave_inclusive(own);
            const uint64_t behind = __ballot(m.before + inc > m.at);
            if (behind == 0 && m.b + 64 >= a.requests) {  // starts or lens changed during the call
                m.go = 0;
                if (threadIdx.x == 0) to = m;
                return;
            }
            const int i = behind ? __builtin_ctzll(behind) : 63;
            m.b += uint32_t(i);
            m.before += of_lane(inc - own, i);
            r = request_at<TREE, FEW, bm>(a, h, m.b);
        }
        cut_segment<TREE, FEW, bm>(a, m, r);
    }
    if (threadIdx.x == 0) to = m;
}

// Adds up the requests, so that no launch has to come first, and finds the one in which the
// part begins and its first segment, `to`.  Up to 64 requests: wave 0 alone, one per lane.  More: thread t takes a run
// of them, l says where the part begins and next_segment, which wave 0 runs too, goes on from there.
template <bool TREE, bool FEW, uint32_t bm, int NT>
__device__ __forceinline__ void start_walk(const PagedAttn& a, Walk& l, Walk& to, Heads& h, double* red)
{
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    if (a.requests <= 64) {
        if (wave) return;
        Request r{};
        if (lane < a.requests) {
            const uint32_t s0 = a.starts[lane], s1 = a.starts[lane + 1], len = a.lens[lane];
            h.s0[lane] = s0;
            h.s1[lane] = s1;
            h.len[lane] = len;
            r = request_of<TREE, FEW, bm>(a, s0, s1, len);
        }
        const double own = r.total * a.kv_heads, inc = wave_inclusive(own);
        Walk m;
        take_part(m, of_lane(inc, 63), group_sum<kWave>(r.units) * a.kv_heads * (FEW ? 1.0f / kFewWaves : 1.0f));
        if (lane == 0) (FEW ? a.few_p : a.many_p)[2 * m.w].n = (FEW ? a.few_p : a.many_p)[2 * m.w + 1].n = 0;
        m.go = m.at < m.to;
        if (m.go) {
            const uint64_t behind = __ballot(inc > m.at);  // lanes from the part's first request on
            const int b = behind ? __builtin_ctzll(behind) : 0;
            m.b = uint32_t(b);
            m.before = of_lane(inc - own, b);
            const Request rb{uint32_t(__builtin_amdgcn_readlane(int(r.token), b)), uint32_t(__builtin_amdgcn_readlane(int(r.rows), b)),
                             __builtin_amdgcn_readlane(r.base, b), uint32_t(__builtin_amdgcn_readlane(int(r.tiles), b)),
                             of_lane(r.first, b), of_lane(r.cap, b), of_lane(r.total, b), 0.0f};
            cut_segment<TREE, FEW, bm>(a, m, rb);
        }
        if (lane == 0) to = m;
        return;
    }
    const uint32_t each = (a.requests + NT - 1) / NT;
    const uint32_t b0 = min(tid * each, a.requests), b1 = min(b0 + each, a.requests);
    double sum = 0.0;
    float units = 0.0f;
#pragma unroll 4
    for (uint32_t b = b0; b < b1; ++b) {
        const Request r = request_at<TREE, FEW, bm>(a, h, b);
        sum += r.total * a.kv_heads;
        units += r.units;
    }
    const double inc = wave_inclusive(sum);
    units = group_sum<kWave>(units);
    if (lane == 63) {
        red[wave] = inc;
        red[NT / kWave + wave] = double(units);
    }
    __syncthreads();
    double before = 0.0, total = 0.0, all = 0.0;
#pragma unroll
    for (int i = 0; i < NT / kWave; ++i) {
        const double r = red[i];
        if (uint32_t(i) < wave) before += r;
        total += r;
        all += red[NT / kWave + i];
    }
    Walk m;
    take_part(m, total, float(all) * a.kv_heads * (FEW ? 1.0f / kFewWaves : 1.0f));
    const double lo = before + inc - sum;
    if (tid == 0) {  // with no work, all there is
        m.b = 0;
        m.before = 0.0;
        l = m;
    }
    __syncthreads();
    if (lo <= m.at && m.at < lo + sum) {  // one thread, if there is any work
        double at = lo;
        uint32_t b = b0;
        for (; b + 1 < b1; ++b) {
            const double c = request_at<TREE, FEW, bm>(a, h, b).total * a.kv_heads;
            if (at + c > m.at) break;
            at += c;
        }
        l.b = b;
        l.before = at;
    }
    __syncthreads();
    if (tid == 0) (FEW ? a.few_p : a.many_p)[2 * m.w].n = (FEW ? a.few_p : a.many_p)[2 * m.w + 1].n = 0;
    next_segment<TREE, FEW, bm>(a, l, to, h);
}

// What every wave needs of the segment, in scalar registers.
struct Segment {
    uint32_t b, g, u0, u1, token, slot, pieces;
    int32_t base;
    Tile x;
};
__device__ __forceinline__ Segment read_segment(const Walk& l)
{
    Segment s;
    s.b = uniform(l.b);
    s.g = uniform(l.g);
    s.u0 = uniform(l.u0);
    s.u1 = uniform(l.u1);
    s.token = uniform(l.token);
    s.slot = uniform(l.slot);
    s.pieces = uniform(l.pieces);
    s.base = uniform(l.base);
    s.x.row0 = uniform(l.x.row0);
    s.x.rows = uniform(l.x.rows);
    s.x.pos0 = uniform(l.x.pos0);
    s.x.pos1 = uniform(l.x.pos1);
    s.x.sink_units = uniform(l.x.sink_units);
    s.x.low = uniform(l.x.low);
    s.x.units = 0;
    return s;
}

// ------------------------------------------------------------- rows of K and V
// What the segment's loop needs of the pool, the tables and the mask.
template <typename T>
struct Pool {
    const T *k, *v;  // at the kv head
    const uint32_t* table;
    uint64_t page_stride;
    uint32_t num_pages, shift, kvd, window, sinks;
    float scale;
};
template <typename T, int D>
__device__ __forceinline__ Pool<T> pool_of(const PagedAttn& a, const Segment& s)
{
    return Pool<T>{static_cast<const T*>(a.k) + s.g * D, static_cast<const T*>(a.v) + s.g * D,
                   a.tables + uint64_t(s.b) * a.max_pages, a.page_stride, a.num_pages, a.shift, a.kv_heads * D,
                   a.window, a.sinks, a.scale};
}

// The element offset of a position's row: its page's and its place's; 0 for a page that is none.
template <typename T>
__device__ __forceinline__ uint64_t row_offset(const Pool<T>& p, uint32_t page, uint32_t pos)
{
    const uint64_t at = uint64_t(page) * p.page_stride + uint64_t(pos & ((1u << p.shift) - 1u)) * p.kvd;
    return page < p.num_pages ? at : 0;
}

// A K or V row in LDS: D / 8 blocks of 16 bytes, block c of row r at place c ^ swizzle(r).  LDS serves 256
// bytes at a time from 64 banks: a read of K's 16-byte blocks takes 16 lanes, whose rows differ modulo 16; a
// transposing read of V takes 32 lanes, 4 rows of 4 blocks.  Each set falls on all 64 banks.
template <int D>
__device__ __forceinline__ uint32_t k_swizzle(uint32_t r)
{
    return D == 128 ? r & 15u : (r >> 1) & 7u;  // D = 64: two rows to 256 bytes
}
template <int D>
__device__ __forceinline__ uint32_t v_swizzle(uint32_t r)
{
    return D == 128 ? (r & 3u) << 2 : ((r >> 1) & 1u) << 2;
}

// 16 bytes per lane from memory straight into LDS, lane i's at lds + 16 i: from base (scalar) + off bytes, or
// from the lane's own address.  In assembly because the compiler waits for such a copy before
// the next read of LDS, whichever buffer that is from; there is no register for a load in
// flight to write, and nothing else here uses m0.  wait_loads and a barrier (a wave's own rows: wait_loads)
// come before the rows are read.
// ONCE: data that no other workgroup reads goes past the caches' keeping (nt): 2 contexts of 131071, 8 kv
// heads (732 MB): 13 % less time.
template <bool ONCE>
__device__ __forceinline__ void copy16(uint32_t lds, const void* base, uint32_t off)
{
    if constexpr (ONCE)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(off), "s"(base) : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
template <bool ONCE>
__device__ __forceinline__ void copy16(uint32_t lds, const void* from)
{
    if constexpr (ONCE)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds), "v"(from) : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(from) : "memory");
}

// N positions' rows of K and V, or one of them, from the pages straight into LDS, row i at kl, vl + i * D.
// `page`: lane first + i holds the page of row i's position pos0 + i.  Which 16 bytes a lane copies carries the swizzle, as
// LDS is written in lane order.  WIDE, pages of 16 and more: 16 aligned rows have one
// page, so the address is scalar and the lane's part of it the same for every unit.
template <bool K, bool V, bool ONCE, int N, bool WIDE, int D, typename T>
__device__ __forceinline__ void copy_rows(const Pool<T>& p, T* kl, T* vl, uint32_t page, uint32_t first, uint32_t pos0)
{
    constexpr uint32_t kAcross = D / 8, kRows = kWave / kAcross;  // lanes per row, rows per copy
    constexpr uint32_t kGroup = N < 16 ? N : 16;
    const uint32_t lane = threadIdx.x & 63u, r0 = lane / kAcross, c = lane % kAcross;
    typedef __attribute__((address_space(3))) void lptr;
    const uint32_t kto = uniform(uint32_t(reinterpret_cast<uintptr_t>((lptr*)(kl))));
    const uint32_t vto = uniform(uint32_t(reinterpret_cast<uintptr_t>((lptr*)(vl))));
#pragma unroll
    for (uint32_t part = 0; part < uint32_t(N); part += kGroup) {
        if constexpr (WIDE) {
            const uint64_t at = row_offset(p, uint32_t(__builtin_amdgcn_readlane(int(page), int(first + part))), pos0 + part);
            const T *kb = p.k + at, *vb = p.v + at;
#pragma unroll
            for (uint32_t i = 0; i < kGroup; i += kRows) {
                const uint32_t r = i + r0, row = first + part + r;
                if constexpr (K) copy16<ONCE>(kto + (part + i) * D * 2, kb, (r * p.kvd + ((c ^ k_swizzle<D>(row)) << 3)) * 2);
                if constexpr (V) copy16<ONCE>(vto + (part + i) * D * 2, vb, (r * p.kvd + ((c ^ v_swizzle<D>(row)) << 3)) * 2);
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kGroup; i += kRows) {
                const uint32_t r = part + i + r0;
                const uint64_t at = row_offset(p, uint32_t(__shfl(int(page), int(first + r))), pos0 + r);
                if constexpr (K) copy16<ONCE>(kto + (part + i) * D * 2, p.k + at + ((c ^ k_swizzle<D>(first + r)) << 3));
                if constexpr (V) copy16<ONCE>(vto + (part + i) * D * 2, p.v + at + ((c ^ v_swizzle<D>(first + r)) << 3));
            }
        }
    }
}

// Waits until every load and copy of this wave has arrived.
__device__ __forceinline__ void wait_loads()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    asm volatile("" ::: "memory");
}

// Waits until this wave's reads of LDS are done: a copy may then overwrite what they read.
__device__ __forceinline__ void wait_lds()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}

// ------------------------------------------------------------ matrix products
template <typename T>
__device__ __forceinline__ f32x16 mfma(vec8<T> x, vec8<T> y, f32x16 c)
{
    if constexpr (__is_same(T, _Float16)) return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
}

// Kinds of instructions for the scheduler, and how many LDS reads go ahead of the first product.
constexpr int kMfma = 0x008, kDsRead = 0x100, kAhead = 8;

// 8 consecutive values to 16 bits, round to nearest even.  The weights' one rounding, which the second product's
// 16-bit operands ask for; their sum l takes them unrounded.  Roundings of keys with different weights average out: the
// outputs' distance from 64 bits is a fifth to a third above the final rounding's own (2.0e-4 -> 2.6e-4 in fp16).  Many
// keys of one weight are all rounded alike, by half a step at most, as much as the output's own rounding.
template <typename T>
__device__ __forceinline__ vec8<T> narrow(const f32x16& p, int at)
{
    vec8<T> r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = static_cast<T>(p[at + j]);
    return r;
}

// V^T operand: dims 32 t + (lane & 31), keys 16 s + 8 (j / 4) + 4 (lane / 32) + j % 4 of rows in
// LDS, by two transposing reads (16 lanes read 4 rows of 16 values, each lane gets a column).
template <typename T, int D>
__device__ __forceinline__ vec8<T> load_vt(const T* rows, int s, int t)
{
    const uint32_t lane = threadIdx.x & 63u, i = lane & 15u;
    s16x4 part[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const uint32_t r = 16u * s + 8u * j + 4u * (lane >> 5) + (i >> 2);
        const uint32_t block = 4u * t + 2u * ((lane >> 4) & 1u) + ((i >> 1) & 1u);
        const T* p = rows + r * D + ((block ^ v_swizzle<D>(r)) << 3) + 4u * (i & 1u);
        part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
    }
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 both = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(vec8<T>, both);
}

// Nonzero where one of the two 16-bit values of w is infinite or NaN.
template <typename T>
__device__ __forceinline__ uint32_t nonfinite(uint32_t w)
{
    constexpr uint32_t kExp = __is_same(T, _Float16) ? 0x7c007c00u : 0x7f807f80u;
    const uint32_t x = ~w & kExp;  // a half that is zero here
    return (x - 0x00010001u) & ~x & 0x80008000u;
}
template <typename T>
__device__ __forceinline__ uint32_t without_nonfinite(uint32_t w)
{
    constexpr uint32_t kExp = __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    if ((w & kExp) == kExp) w &= 0xffff0000u;
    if (((w >> 16) & kExp) == kExp) w &= 0x0000ffffu;
    return w;
}

__device__ __forceinline__ bool sees(int32_t qpos, int32_t kpos, uint32_t window, uint32_t sinks)
{
    return kpos <= qpos && (window == 0 || uint32_t(qpos - kpos) < window || uint32_t(kpos) < sinks);
}

// Which of the 32 positions from k0 on a query at qpos sees, as bits.
__device__ __forceinline__ uint32_t seen_bits(int32_t qpos, int32_t k0, uint32_t window, uint32_t sinks)
{
    const int32_t n = qpos - k0;  // the last of them
    if (n < 0) return 0;
    uint32_t bits = n >= 31 ? ~0u : (2u << n) - 1u;
    if (window && uint32_t(n) >= window) {
        const uint32_t first = uint32_t(n) - window + 1u, sink = sinks > uint32_t(k0) ? sinks - uint32_t(k0) : 0u;
        bits &= (first > 31 ? 0u : ~0u << first) | (sink > 31 ? ~0u : (1u << sink) - 1u);
    }
    return bits;
}

// What a lane's query sees: its position in the cache, and, where its request's rows are a tree, its mask.
template <bool TREE>
struct Sight {
    int32_t qpos;
    __device__ __forceinline__ uint32_t bits(int32_t k0, uint32_t window, uint32_t sinks) const
    {
        return seen_bits(qpos, k0, window, sinks);
    }
    __device__ __forceinline__ bool at(int32_t kpos, uint32_t window, uint32_t sinks) const { return sees(qpos, kpos, window, sinks); }
};
template <>
struct Sight<true> {
    int32_t qpos;
    int32_t base;          // place of node 0
    int32_t depth;         // of the row's node
    uint32_t words;        // of its mask; 0: a chunk's row
    const uint32_t* mask;
    __device__ __forceinline__ uint32_t word(int32_t w) const { return uint32_t(w) < words ? mask[w] : 0; }
    // Of the nodes in `nodes`, from node `first` on, those that a window leaves: node j is as deep as the mask has
    // bits below j.
    __device__ __forceinline__ uint32_t in_window(uint32_t nodes, int32_t first, uint32_t window, uint32_t sinks) const
    {
        uint32_t left = 0;
        for (; nodes; nodes &= nodes - 1) {
            const uint32_t t = uint32_t(__builtin_ctz(nodes)), j = uint32_t(first + int32_t(t));
            int32_t d = __builtin_popcount(word(int32_t(j >> 5)) & ((1u << (j & 31u)) - 1u));
            for (uint32_t w = 0; w < (j >> 5); ++w) d += __builtin_popcount(word(int32_t(w)));
            if (uint32_t(max(depth - d, 0)) < window || uint32_t(max(base + d, 0)) < sinks) left |= 1u << t;
        }
        return left;
    }
    __device__ __forceinline__ uint32_t bits(int32_t k0, uint32_t window, uint32_t sinks) const
    {
        if (words == 0) return seen_bits(qpos, k0, window, sinks);
        const int32_t first = k0 - base;  // the node at k0
        const uint32_t context = first >= 0 ? 0u : first <= -32 ? ~0u : (1u << -first) - 1u;
        uint32_t seen = context ? context & seen_bits(base + depth, k0, window, sinks) : 0u;
        if (context != ~0u) {
            const int32_t w = first >> 5;
            uint32_t nodes = uint32_t(((uint64_t(word(w + 1)) << 32) | word(w)) >> (uint32_t(first) & 31u));
            nodes &= seen_bits(qpos, k0, 0, 0);
            if (window && uint32_t(depth) >= window) nodes = in_window(nodes, first, window, sinks);
            seen |= nodes;
        }
        return seen;
    }
    __device__ __forceinline__ bool at(int32_t kpos, uint32_t window, uint32_t sinks) const
    {
        return bits(kpos & ~31, window, sinks) >> (uint32_t(kpos) & 31u) & 1u;
    }
};
template <bool TREE>
__device__ __forceinline__ Sight<TREE> sight_of(const PagedAttn& a, const Segment& s, uint32_t row)
{
    const uint32_t i = (s.x.row0 + row) / a.hpk;
    Sight<TREE> v;
    v.qpos = s.base + int32_t(i);
    if constexpr (TREE) {
        v.base = s.base;
        const TreeAttn& t = of_tree(a);
        v.words = s.x.pos0 < s.base ? t.words : 0u;  // see tile_at
        v.mask = t.masks + uint64_t(s.token + i) * t.words;
        v.depth = a.window && v.words ? int32_t(t.positions[s.token + i]) - s.base : 0;
    }
    return v;
}

// The scores of a tile of 32 positions that its query does not see become -infinity.
__device__ __forceinline__ void hide(f32x16& sc, uint32_t bits)
{
    bits >>= 4u * ((threadIdx.x >> 5) & 1u);
#pragma unroll
    for (int i = 0; i < 16; ++i)
        sc[i] = int32_t(bits << (31 - 8 * (i >> 2) - (i & 3))) < 0 ? sc[i] : -INFINITY;
}

// Weights.  A score's weight is 2^(score * scale - R) with R = m * scale for a reference score m, about the largest
// so far.  Up to kLarge R is -c, rounded, and the exponent one fused multiply and add: what c's rounding adds to
// every exponent is in R too, so only the size of the weights knows of it (by 2^-13 powers of two at kLarge, 16 at 2^28,
// which no 16-bit weight survives).  Beyond, R is m * scale itself and the exponent (score - m) * scale, exact where it
// counts, for one instruction more a score: a branch that scores of models do not take, on a flag that changes with m.  It
// costs 0 to 2 % (64 requests of up to 8000 56.8 -> 57.0 us, a chunk of 4096 at 12288 897 -> 900); decided again in each unit
// 1.4 % (909).  The form of large scores for all would add an instruction to the seven that each score has.
constexpr float kLarge = 4096.0f;
__device__ __forceinline__ float offset_of(float m, float scale)
{
#pragma clang fp contract(off)  // the rounded product, wherever it goes
    return -(m * scale);
}
__device__ __forceinline__ bool is_large(float c) { return !(fabsf(c) <= kLarge); }

// The factor 2^(R - R') that takes sums with the reference m to the reference `to`, which is not -infinity; 0 for m =
// -infinity, sums of nothing.  R is m * scale and what its rounding adds, if it is rounded.
__device__ __forceinline__ float moved(float m, float to, float scale)
{
#pragma clang fp contract(off)
    auto rounding = [&](float r) {
        const float c = offset_of(r, scale);
        return is_large(c) ? 0.0f : -__builtin_fmaf(r, scale, c);
    };
    return __builtin_amdgcn_exp2f(__builtin_fmaf(m - to, scale, rounding(m) - rounding(to)));
}

// Running softmax of one query (a lane and its partner lane ^ 32, each with half of the
// keys): `m` is the reference score, `l` the lane's share of the sum of weights.
struct Running {
    float m = -INFINITY, l = 0.0f;
    float c = 0.0f;      // offset_of(m), of 0 while nothing is seen: all weights are 0 then
    bool large = false;  // is_large(c) in any lane
};
// m follows the maximum only when that has
// grown by more than kLazy powers of two, which saves nearly every rescaling of the output and costs no accuracy
// (relative rounding).  In fp16 it stays kLift powers of two below: the largest weight is 2^7 to 2^15, the upper part of the
// type's range, and weights keep all their bits down to 2^-21 of the largest and count down to 2^-32.  With the largest at 1 a
// context of 2^17 keys of 2^-24 each, one sharp key before them, was 0.5 % off.  bf16 has fp32's range.
template <typename T, int NO>
__device__ __forceinline__ void rescale(float mx, float scale, Running& s, f32x16 (&o)[NO])
{
    if (__ballot((mx - s.m) * scale > kLift<T> + kLazy) == 0) return;  // m = -inf: any score that is one
    // a scale so small that the lift is beyond 2^100 in scores takes less of it
    const float lift = kLift<T> > 0.0f ? fminf(kLift<T> * __builtin_amdgcn_rcpf(scale), 0x1p100f) : 0.0f;
    const float to = fmaxf(s.m, mx - lift);
    const float f = to == -INFINITY ? 1.0f : moved(s.m, to, scale);
    s.m = to;
    s.l *= f;
    s.c = to == -INFINITY ? 0.0f : offset_of(to, scale);
    s.large = __ballot(is_large(s.c)) != 0;
#pragma unroll
    for (int t = 0; t < NO; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] *= f;
}

// The k and c with which fma(score, k, c) is a score's exponent; large ones are exponents afterwards (k = 1, c = 0).
template <typename... Scores>
__device__ __forceinline__ void exponents(const Running& s, float& k, float& c, Scores&... sc)
{
    c = s.c;
    if (__builtin_expect(!s.large, 1)) return;
    auto each = [&](f32x16& x) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = is_large(s.c) ? (x[i] - s.m) * k : __builtin_fmaf(x[i], k, s.c);
    };
    (each(sc), ...);
    c = 0.0f;
    k = 1.0f;
}

// Value i of a score or output tile of 32: key, or dim, 8 (i / 4) + 4 (lane / 32) + i % 4.
__device__ __forceinline__ uint32_t tile_index(int i) { return 8u * (i >> 2) + 4u * ((threadIdx.x >> 5) & 1u) + (i & 3); }

// Where a slot holds 4 values of a row from dim d on.  Row by row, or, in blocks: 32 rows' same 8 dims side by
// side, as a wave of the many-rows kernel has them, so that its stores cover whole lines.
__device__ __forceinline__ uint32_t piece_place(bool blocks, uint32_t row, uint32_t dim, uint32_t d)
{
    return blocks ? (row & ~31u) * dim + (d & ~7u) * 32 + (row & 31u) * 8 + (d & 7u) : row * dim + d;
}

// Query operand of 32 rows: lane -> row lane & 31, dims 16 s + 8 (lane / 32) .. + 7; zeros for
// rows that the tile does not have.
template <typename T, int D>
__device__ __forceinline__ void load_q(const PagedAttn& a, uint32_t token, uint32_t row, bool in, uint32_t g, vec8<T> (&q)[D / 16])
{
    const uint32_t h2 = (threadIdx.x >> 5) & 1u;
    const uint32_t tok = row / a.hpk, h = row - tok * a.hpk;
    const T* p = static_cast<const T*>(a.q) + uint64_t(token + tok) * a.ldq + (g * a.hpk + h) * D + 8 * h2;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (in) w = *reinterpret_cast<const uint4*>(p + 16 * s);
        w.x ^= a.neg;
        w.y ^= a.neg;
        w.z ^= a.neg;
        w.w ^= a.neg;
        q[s] = __builtin_bit_cast(vec8<T>, w);
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, float x, float y, float z, float w)
{
    vec4<T> v;
    v[0] = static_cast<T>(x);
    v[1] = static_cast<T>(y);
    v[2] = static_cast<T>(z);
    v[3] = static_cast<T>(w);
    *reinterpret_cast<vec4<T>*>(p) = v;
}

template <typename T>
__device__ __forceinline__ T* out_row(const PagedAttn& a, uint32_t token, uint32_t row, uint32_t g, int dim)
{
    const uint32_t tok = row / a.hpk, h = row - tok * a.hpk;
    return static_cast<T*>(a.out) + uint64_t(token + tok) * a.ldo + (g * a.hpk + h) * dim;
}

// Whether every row of the tile sees all of `keys` positions from k0 on that have pages (valid).
template <typename T>
__device__ __forceinline__ bool all_seen(const Pool<T>& p, const Tile& x, int32_t k0, uint32_t keys, bool valid)
{
    return valid && k0 + int32_t(keys) - 1 <= x.pos0 &&
           (p.window == 0 || uint32_t(x.pos1 - k0) < p.window || uint32_t(k0) + keys <= p.sinks);
}

// Clears infinities and NaN of the 16 bytes at p, or all of them where the position is not in; whether there were
// infinities or NaN of one that is.
template <typename T>
__device__ __forceinline__ bool clean(T* p, bool in)
{
    uint4 w = *reinterpret_cast<const uint4*>(p);
    const bool any = (nonfinite<T>(w.x) | nonfinite<T>(w.y) | nonfinite<T>(w.z) | nonfinite<T>(w.w)) != 0;
    if (in && !any) return false;
    w = in ? make_uint4(without_nonfinite<T>(w.x), without_nonfinite<T>(w.y), without_nonfinite<T>(w.z), without_nonfinite<T>(w.w))
           : make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(p) = w;
    return in && any;
}

// What infinities and NaN of V at positions that only some of a tile's rows see have to add: their
// places in V were cleared for the product, where a weight of 0 would make NaN of them; here, after the
// segment's units, each row that sees such a position gets them.  Units that all rows see
// need none of it.  A slow pass over the wave's other units (from, from + step ..), for data that has any;
// first_of and page_of as in the kernels, `span` positions of each unit.
template <typename T, int D, bool TREE, typename First, typename Page>
__device__ __forceinline__ void add_nonfinite(const Pool<T>& p, f32x16 (&o)[D / 32], const Segment& s, uint32_t from, uint32_t step,
                                              uint32_t span, const Sight<TREE>& sight, First first_of, Page page_of)
{
#pragma unroll 1
    for (uint32_t u = from; u < s.u1; u += step) {
        const int32_t k0 = int32_t(first_of(u));
        const uint32_t page = page_of(u);
        if (all_seen(p, s.x, k0, span, __ballot(page < p.num_pages) == ~uint64_t(0))) continue;  // lanes beyond span repeat
#pragma unroll 1
        for (uint32_t j = 0; j < span; ++j) {
            const uint32_t pg = uint32_t(__builtin_amdgcn_readlane(int(page), int(j)));
            if (pg >= p.num_pages || !sight.at(k0 + int32_t(j), p.window, p.sinks)) continue;
            const T* row = p.v + row_offset(p, pg, uint32_t(k0) + j);
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    // all exponent bits set: the sum carries into the sign, which becomes a mask
                    const int32_t x = __builtin_bit_cast(int32_t, static_cast<float>(row[32 * t + tile_index(i)]));
                    const int32_t keep = int32_t((uint32_t(x) & 0x7f800000u) + 0x00800000u) >> 31;
                    o[t][i] += __builtin_bit_cast(float, x & keep);
                }
        }
    }
}

__device__ __forceinline__ void wave_fence()  // this wave's LDS accesses before it come before those after it
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// ------------------------------------------------------------------ few rows
// Tiles of up to 32 rows: decode, short chunks.  Bound by reading K and V once.  4
// waves, each on units of 32 positions with its own softmax, joined through LDS
// at the tile's end; nothing but that join needs a barrier.  K and V come straight into
// the wave's own LDS rows, in whole rows.  S^T = K Q^T (lane -> query), O^T = V^T P^T, P^T from the
// scores' registers.  The next unit's K is on its way as soon as this one's scores are done, its V
// after the output: with 8 waves a CU some 110 KB of 128 are in flight.  Measured, the call with its join: 64
// requests of up to 8000, 28 heads on 4 (271 MB) 57 us, 4.8 TB/s, of which 3 are the walk and 4 the join; 2 of
// 131071, 64 on 8 (732 MB) 123 us, 5.9 TB/s; plain reads of as much reach 6.2.  Pages of 1 to 8 positions: as long.
template <typename T, int D, bool WIDE, bool TREE>
__global__ __launch_bounds__(256, 2) void k_paged_few(Attn<TREE>)
{
    __shared__ struct {  // rows first: m0, which says where a copy goes, is used below 2^16 only
        __align__(16) float joined[4 * 32 * D];  // K and V rows of each wave, then the waves' outputs
        float mw[4][32], lw[4][32];
        double red[8];
        Walk walk[2];  // this segment and the next
        Heads heads;
    } lds;
    static_assert(sizeof(lds.joined) <= 65536, "rows below 2^16");
    auto& joined = lds.joined;
    auto &mw = lds.mw, &lw = lds.lw;
    auto& walk = lds.walk;
    Heads& heads = lds.heads;
    double* red = lds.red;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, l32 = lane & 31u, h2 = lane >> 5, wave = uniform(tid >> 6);
    start_walk<TREE, true, kFewRows, 256>(arguments(), walk[1], walk[0], heads, red);
    T* krows = reinterpret_cast<T*>(joined) + wave * (2 * 32 * D);
    T* vrows = krows + 32 * D;
    for (uint32_t turn = 0;; turn ^= 1u) {
        __syncthreads();
        if (uniform(walk[turn].go) == 0) break;
        const Segment s = read_segment(walk[turn]);
        const Pool<T> p = pool_of<T, D>(arguments(), s);
        const uint32_t row = min(l32, s.x.rows - 1);
        const Sight<TREE> sight = sight_of<TREE>(arguments(), s, row);
        f32x16 o[D / 32];
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
        Running run;
        bool odd = false;  // infinities or NaN cleared from V

        // the first position of unit u, the page of lane l32's
        auto first_of = [&](uint32_t u) { return unit_start(s.x, u, kFewKeys); };
        auto page_of = [&](uint32_t u) {
            const int32_t kp = int32_t(first_of(u) + l32);
            return kp <= s.x.pos1 ? p.table[uint32_t(kp) >> p.shift] : 0xffffffffu;
        };
        const uint32_t mine = s.u0 + wave;  // the waves take the units in turn
        if (mine < s.u1) {
            uint32_t page = page_of(mine);
            uint32_t npage = mine + kFewWaves < s.u1 ? page_of(mine + kFewWaves) : 0xffffffffu;
            vec8<T> q[D / 16];
            load_q<T, D>(arguments(), s.token, s.x.row0 + row, l32 < s.x.rows, s.g, q);
            copy_rows<true, true, true, 32, WIDE, D>(p, krows, vrows, page, 0, first_of(mine));
            next_segment<TREE, true, kFewRows>(arguments(), walk[turn], walk[turn ^ 1u], heads);  // while those are on their way
            for (uint32_t u = mine; u < s.u1; u += kFewWaves) {
                const int32_t k0 = int32_t(first_of(u));
                wait_loads();  // K, V of this unit, the next one's pages
                const bool more = u + kFewWaves < s.u1;
                f32x16 sc;
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const vec8<T> kf = *reinterpret_cast<const vec8<T>*>(&krows[l32 * D + (((2u * i + h2) ^ k_swizzle<D>(l32)) << 3)]);
                    sc = mfma<T>(kf, q[i], sc);
                }
                uint32_t far = 0xffffffffu;
                if (more) {
                    wait_lds();
                    copy_rows<true, false, true, 32, WIDE, D>(p, krows, krows, npage, 0, first_of(u + kFewWaves));
                    if (u + 2 * kFewWaves < s.u1) far = page_of(u + 2 * kFewWaves);
                }

                const bool in = page < p.num_pages;
                const uint32_t valid = uint32_t(__ballot(in));
                const bool whole = all_seen(p, s.x, k0, 32, valid == 0xffffffffu);
                if (!whole) {
                    for (uint32_t c = h2; c < D / 8; c += 2) odd |= clean(vrows + l32 * D + c * 8, in);
                    hide(sc, valid & sight.bits(k0, p.window, p.sinks));
                    wave_fence();
                }
                float mx = sc[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[i]);
                rescale<T>(xor_max<32>(mx), p.scale, run, o);
                float k = p.scale, c;
                exponents(run, k, c, sc);
                float sum = 0.0f;  // the unit's: a weight that would vanish beside l counts among its like
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sc[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], k, c));
                    sum += sc[i];
                }
                run.l += sum;
#pragma unroll
                for (int st = 0; st < 2; ++st) {
                    const vec8<T> w = narrow<T>(sc, 8 * st);
#pragma unroll
                    for (int t = 0; t < D / 32; ++t) o[t] = mfma<T>(load_vt<T, D>(vrows, st, t), w, o[t]);
                }
                if (more) {
                    wait_lds();
                    copy_rows<false, true, true, 32, WIDE, D>(p, vrows, vrows, npage, 0, first_of(u + kFewWaves));
                }
                page = npage;
                npage = far;
            }
            if (__ballot(odd)) add_nonfinite<T, D, TREE>(p, o, s, mine, kFewWaves, 32, sight, first_of, page_of);
        } else {
            next_segment<TREE, true, kFewRows>(arguments(), walk[turn], walk[turn ^ 1u], heads);
        }
        // the waves' states in wave order: out = sum_w f_w o_w / sum_w f_w l_w, f_w to the largest reference M
        __syncthreads();  // every wave is done with its V rows
        const float lsum = xor_sum<32>(run.l);
        if (l32 < s.x.rows) {
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4*>(&joined[(wave * 32 + l32) * D + 32 * t + tile_index(i)]) =
                        make_float4(o[t][i], o[t][i + 1], o[t][i + 2], o[t][i + 3]);
            if (lane < 32) {
                mw[wave][l32] = run.m;
                lw[wave][l32] = lsum;
            }
        }
        __syncthreads();
        const PagedAttn& e_ = arguments();
        for (uint32_t e = tid; e < s.x.rows * (D / 4); e += 256) {
            const uint32_t rr = e / (D / 4), d = 4 * (e % (D / 4));
            float M = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) M = fmaxf(M, mw[i][rr]);
            const float M0 = M == -INFINITY ? 0.0f : M;
            float L = 0.0f;
            float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = moved(mw[i][rr], M0, e_.scale);
                const float4 w = *reinterpret_cast<const float4*>(&joined[(i * 32 + rr) * D + d]);
                L = __builtin_fmaf(lw[i][rr], f, L);
                acc.x = __builtin_fmaf(w.x, f, acc.x);
                acc.y = __builtin_fmaf(w.y, f, acc.y);
                acc.z = __builtin_fmaf(w.z, f, acc.z);
                acc.w = __builtin_fmaf(w.w, f, acc.w);
            }
            if (s.pieces == 0) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // nothing seen: zeros
                store4<T>(out_row<T>(e_, s.token, s.x.row0 + rr, s.g, D) + d, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            } else {
                *reinterpret_cast<float4*>(e_.few_o + (uint64_t(s.slot) * e_.few_slot + rr) * D + d) = acc;
                if (d == 0) e_.few_ml[uint64_t(s.slot) * e_.few_slot + rr] = make_float2(M, L);
            }
        }
    }
}

// ----------------------------------------------------------------- many rows
// Tiles of NW * 32 rows: prompts and long chunks.  Bound by the matrix cores and the
// softmax's vector instructions.  Each wave holds 32 rows (Q, O in registers); the
// unit's 64 rows of K and V come straight into LDS, shared by the waves and double buffered:
// unit u + 1 is copied while unit u is computed; one barrier per unit.  Operands as in the
// few-rows kernel, K's read from LDS.  Measured: 4096 tokens at 12288, 28 heads of 128 on 4, 842 GFLOP that are
// seen: 850 to 910 us by the card, 0.93 to 0.99 PFLOP/s of the 1.23 that a large fp16 product reaches; with zeros for data 650 us, so the
// clock under the matrix cores' power is what is left.  3 x 2000 tokens in a window of 1024, heads of 64: 137 to
// 146 us, 0.5 PFLOP/s, bound by the softmax's vector instructions, as many per score as heads of 128 have for twice the
// products.
// Trees: 48 of up to 60 nodes at up to 8000, 28 heads of 128 on 4, 124 us; of up to 9 nodes 58.  A unit takes a wave 1.5 us
// however many of the waves have rows, so what bounds it is the units of tiles that are not full; waves without rows
// only copy.  Not quicker: tiles of 128 rows, two workgroups to a compute unit (133 us: each unit copied more often);
// two waves to 32 rows of a tile that is half empty, each with half a unit's positions (182 us: 59 registers too
// many).  One tree of 26 nodes at 501: 15.2 us, of which the join is 3.
template <typename T, int D, int NW, bool WIDE, bool TREE>
__global__ __launch_bounds__(NW * 64, D == 64 ? 3 : 2) void k_paged_many(Attn<TREE>)
{
    constexpr int NT = NW * 64;
    constexpr uint32_t kBm = NW * 32, kOwn = kManyKeys / NW;  // rows of K and V that a wave copies
    __shared__ struct {  // rows first: m0, which says where a copy goes, is used below 2^16 only
        __align__(16) T ks[2][kManyKeys * D];
        __align__(16) T vs[2][kManyKeys * D];
        double red[2 * NW];
        Walk walk[2];  // this segment and the next
        Heads heads;
        uint32_t odd;  // infinities or NaN cleared from V in this segment
    } lds;
    static_assert(sizeof(lds.ks) + sizeof(lds.vs) <= 65536, "rows below 2^16");
    auto &ks = lds.ks, &vs = lds.vs;
    auto& walk = lds.walk;
    Heads& heads = lds.heads;
    double* red = lds.red;
    uint32_t& odd = lds.odd;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, l32 = lane & 31u, h2 = lane >> 5, wave = uniform(tid >> 6);
    start_walk<TREE, false, kBm, NT>(arguments(), walk[1], walk[0], heads, red);
    for (uint32_t turn = 0;; turn ^= 1u) {
        __syncthreads();  // the tile before is done with LDS
        if (uniform(walk[turn].go) == 0) break;
        if (tid == 0) odd = 0;  // set after the first unit's barrier at the earliest
        const Segment s = read_segment(walk[turn]);
        const Pool<T> p = pool_of<T, D>(arguments(), s);
        const uint32_t trow = wave * 32 + l32;
        const uint32_t row = min(trow, s.x.rows - 1);
        const Sight<TREE> sight = sight_of<TREE>(arguments(), s, row);
        f32x16 o[D / 32];
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
        Running run;

        // trees are rarely a multiple of a tile's rows: waves without any only copy
        const bool rows_here = wave * 32 < s.x.rows;

        // the page of the lane's position in unit u
        auto page_of = [&](uint32_t u) {
            const int32_t kp = int32_t(unit_start(s.x, u, kManyKeys) + lane);
            return kp <= s.x.pos1 ? p.table[uint32_t(kp) >> p.shift] : 0xffffffffu;
        };
        auto copy_unit = [&](uint32_t u, uint32_t page, int buf) {
            const uint32_t at = wave * kOwn, pos = unit_start(s.x, u, kManyKeys) + at;
            // past the caches' keeping where no other tile reads it: 48 trees of up to 9 tokens at up to 8000, 28 heads, 58 us
            // instead of 66; with several tiles to a tree (16 of up to 250 at 4000) 3 % slower
            if (TREE && of_tree(arguments()).once) copy_rows<true, true, TREE, kOwn, WIDE, D>(p, &ks[buf][at * D], &vs[buf][at * D], page, at, pos);
            else copy_rows<true, true, false, kOwn, WIDE, D>(p, &ks[buf][at * D], &vs[buf][at * D], page, at, pos);
        };
        if (s.u0 < s.u1) {
            uint32_t page = page_of(s.u0);
            uint32_t npage = s.u0 + 1 < s.u1 ? page_of(s.u0 + 1) : 0xffffffffu;
            vec8<T> q[D / 16];
            load_q<T, D>(arguments(), s.token, s.x.row0 + row, trow < s.x.rows, s.g, q);
            copy_unit(s.u0, page, 0);
            next_segment<TREE, false, kBm>(arguments(), walk[turn], walk[turn ^ 1u], heads);  // while that is on its way
            int cur = 0;
            for (uint32_t u = s.u0; u < s.u1; ++u) {
                wait_loads();
                __syncthreads();  // this unit's rows are in LDS, the other buffer is read no more
                const int32_t k0 = int32_t(unit_start(s.x, u, kManyKeys));
                uint32_t far = 0xffffffffu;
                if (u + 1 < s.u1) {
                    copy_unit(u + 1, npage, cur ^ 1);
                    if (u + 2 < s.u1) far = page_of(u + 2);
                }
                const uint64_t valid = __ballot(page < p.num_pages);
                const bool whole = all_seen(p, s.x, k0, kManyKeys, valid == ~uint64_t(0));
                if (!whole) {
                    // positions without a page, infinities and NaN out of V
                    for (uint32_t e = tid; e < kManyKeys * (D / 8); e += NT) {
                        const uint32_t rr = e / (D / 8);
                        if (clean(&vs[cur][e * 8], (valid >> rr) & 1u)) odd = 1;
                    }
                    __syncthreads();
                }

                if (!TREE || rows_here) {
                    f32x16 sc[2];
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int i = 0; i < 16; ++i) sc[kt][i] = 0.0f;
                    // K's operands 4 steps ahead of their products: LDS answers in some 200 cycles
#pragma unroll
                    for (int st = 0; st < D / 16; ++st)
#pragma unroll
                        for (int kt = 0; kt < 2; ++kt) {
                            const uint32_t rr = 32u * kt + l32;
                            const vec8<T> kf =
                                *reinterpret_cast<const vec8<T>*>(&ks[cur][rr * D + (((2u * st + h2) ^ k_swizzle<D>(rr)) << 3)]);
                            sc[kt] = mfma<T>(kf, q[st], sc[kt]);
                        }
                    __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead, 0);
#pragma unroll
                    for (int i = 0; i < D / 8 - kAhead; ++i) {
                        __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
                    }
                    __builtin_amdgcn_sched_group_barrier(kMfma, kAhead, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    // V's operands a step ahead of theirs
                    vec8<T> vt[2][D / 32];
#pragma unroll
                    for (int t = 0; t < D / 32; ++t) vt[0][t] = load_vt<T, D>(vs[cur], 0, t);
                    if (!whole) {
                        hide(sc[0], uint32_t(valid) & sight.bits(k0, p.window, p.sinks));
                        hide(sc[1], uint32_t(valid >> 32) & sight.bits(k0 + 32, p.window, p.sinks));
                    }
                    float mx = sc[0][0];
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kt][i]);
                    rescale<T>(xor_max<32>(mx), p.scale, run, o);
                    float k = p.scale, c;
                    exponents(run, k, c, sc[0], sc[1]);
                    float sum = 0.0f;  // as in the few-rows kernel
                    auto weights = [&](int st) {  // the 16 positions of step st: their weights, rounded; sum adds the unrounded
                        f32x16& x = sc[st >> 1];
#pragma unroll
                        for (int i = 8 * (st & 1); i < 8 * (st & 1) + 8; ++i) {
                            x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], k, c));
                            sum += x[i];
                        }
                        return narrow<T>(x, 8 * (st & 1));
                    };
                    vec8<T> w = weights(0);
#pragma unroll
                    for (int st = 0; st < 4; ++st) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (st < 3)
#pragma unroll
                            for (int t = 0; t < D / 32; ++t) vt[(st + 1) & 1][t] = load_vt<T, D>(vs[cur], st + 1, t);
#pragma unroll
                        for (int t = 0; t < D / 32; ++t) o[t] = mfma<T>(vt[st & 1][t], w, o[t]);
                        if (st < 3) w = weights(st + 1);
                    }
                    run.l += sum;
                }
                cur ^= 1;
                page = npage;
                npage = far;
            }
            // set before the last unit's second barrier, if at all
            if (uniform(odd))
                add_nonfinite<T, D, TREE>(p, o, s, s.u0, 1, kManyKeys, sight, [&](uint32_t u) { return unit_start(s.x, u, kManyKeys); }, page_of);
        } else {
            next_segment<TREE, false, kBm>(arguments(), walk[turn], walk[turn ^ 1u], heads);
        }
        const float L = xor_sum<32>(run.l);
        const PagedAttn& e_ = arguments();
        if (trow < s.x.rows) {
            if (s.pieces == 0) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                T* dst = out_row<T>(e_, s.token, s.x.row0 + trow, s.g, D);
#pragma unroll
                for (int t = 0; t < D / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        store4<T>(dst + 32 * t + tile_index(i), o[t][i] * inv, o[t][i + 1] * inv, o[t][i + 2] * inv,
                                  o[t][i + 3] * inv);
            } else {
                float* dst = e_.many_o + uint64_t(s.slot) * e_.many_slot * D;
                const bool blocks = s.pieces <= kManyPieces;
#pragma unroll
                for (int t = 0; t < D / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<float4*>(dst + piece_place(blocks, trow, D, 32 * t + tile_index(i))) =
                            make_float4(o[t][i], o[t][i + 1], o[t][i + 2], o[t][i + 3]);
                if (h2 == 0) e_.many_ml[uint64_t(s.slot) * e_.many_slot + trow] = make_float2(run.m, L);
            }
        }
    }
}

// ---------------------------------------------------------------------- join
// Adds the pieces of the tiles that were cut, in order: out = sum_i f_i o_i / sum_i f_i l_i with f_i = 2^(R_i - R), to
// the largest reference.  A workgroup for each slot (many_split of them where tiles have many
// rows); the workgroups of a tile's n pieces share its rows.  D / 4 lanes span a row; few
// pieces (long rows of tiles cut once or twice): 256 / (D / 4) rows at once, each by its lanes
// alone; many (one long context): a row at a time, its pieces dealt out over the groups of lanes.
// What bounds it is the way to memory and back: the record, the sums, all of a row's pieces at once, and as few
// turns after that as the card has workgroups for.  Heads of 128, a chunk of 500 at 2500, 40 us the call with 8
// workgroups a slot: 3 more with 4, as long with 16; of 64, three chunks of 700, 49 us with 2: as long with 4, 6
// more with 8.
constexpr uint32_t many_split(uint32_t dim) { return dim == 128 ? 8 : 2; }

struct JoinRow {
    float L;
    float4 acc;
};
__device__ __forceinline__ void add_piece(JoinRow& r, float f, float l, const float4& o)
{
    r.L = __builtin_fmaf(l, f, r.L);
    r.acc.x = __builtin_fmaf(o.x, f, r.acc.x);
    r.acc.y = __builtin_fmaf(o.y, f, r.acc.y);
    r.acc.z = __builtin_fmaf(o.z, f, r.acc.z);
    r.acc.w = __builtin_fmaf(o.w, f, r.acc.w);
}
template <typename T>
__device__ __forceinline__ void store_row(T* p, const JoinRow& r)
{
    const float inv = r.L == 0.0f ? 0.0f : 1.0f / r.L;
    store4<T>(p, r.acc.x * inv, r.acc.y * inv, r.acc.z * inv, r.acc.w * inv);
}

template <typename T, int D>
__global__ __launch_bounds__(256) void k_paged_join(PagedAttn a)
{
    constexpr uint32_t kLanes = D / 4, kGroups = 256 / kLanes, kSplit = many_split(D);
    __shared__ __align__(16) float4 part[kGroups][kLanes];
    __shared__ float part_l[kGroups];
    const bool is_few = blockIdx.x < 2 * a.few_wgs;
    const uint32_t many = blockIdx.x - 2 * a.few_wgs;
    const Piece p = is_few ? a.few_p[blockIdx.x] : a.many_p[many / kSplit];
    if (p.n == 0) return;
    const uint32_t split = is_few ? 1 : kSplit, part_of_slot = is_few ? 0 : many % kSplit;
    const float* po = is_few ? a.few_o : a.many_o;
    const float2* pml = is_few ? a.few_ml : a.many_ml;
    const uint32_t srows = is_few ? a.few_slot : a.many_slot;
    const uint32_t tid = threadIdx.x;
    const bool blocks = !is_few && p.n <= kManyPieces;
    const uint32_t grp = blocks ? (tid >> 1) % kGroups : tid / kLanes;  // its row of kGroups
    const uint32_t d = 4 * (blocks ? 2 * (tid / (2 * kGroups)) + (tid & 1u) : tid % kLanes);
    auto slot = [&](uint32_t i) { return uint64_t(i ? 2 * (p.wg + i) : p.slot) * srows; };
    auto ml_at = [&](uint32_t i, uint32_t row) { return pml[slot(i) + row]; };
    auto o_at = [&](uint32_t i, uint32_t row) {
        return *reinterpret_cast<const float4*>(po + slot(i) * D + piece_place(blocks, row, D, d));
    };
    const uint32_t turn = p.idx * split + part_of_slot, turns = p.n * split;
    if (p.n <= kManyPieces) {
        for (uint32_t row = turn * kGroups + grp; row < p.rows; row += turns * kGroups) {
            float2 ml[kManyPieces];
            float4 o[kManyPieces];
#pragma unroll
            for (uint32_t i = 0; i < kManyPieces; ++i)  // all of them on their way at once
                if (i < p.n) {
                    ml[i] = ml_at(i, row);
                    o[i] = o_at(i, row);
                }
            float M = -INFINITY;
#pragma unroll
            for (uint32_t i = 0; i < kManyPieces; ++i)
                if (i < p.n) M = fmaxf(M, ml[i].x);
            const float M0 = M == -INFINITY ? 0.0f : M;
            JoinRow r{0.0f, make_float4(0, 0, 0, 0)};
#pragma unroll
            for (uint32_t i = 0; i < kManyPieces; ++i)
                if (i < p.n) add_piece(r, moved(ml[i].x, M0, a.scale), ml[i].y, o[i]);
            store_row(out_row<T>(a, p.token, p.row0 + row, p.g, D) + d, r);
        }
        return;
    }
    for (uint32_t row = turn; row < p.rows; row += turns) {
        float M = -INFINITY;
#pragma unroll 4
        for (uint32_t i = grp; i < p.n; i += kGroups) M = fmaxf(M, ml_at(i, row).x);
        __syncthreads();  // the row before is done with part and part_l
        if (d == 0) part_l[grp] = M;
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < kGroups; ++j) M = fmaxf(M, part_l[j]);
        const float M0 = M == -INFINITY ? 0.0f : M;
        JoinRow r{0.0f, make_float4(0, 0, 0, 0)};
#pragma unroll 4
        for (uint32_t i = grp; i < p.n; i += kGroups) {
            const float2 ml = ml_at(i, row);
            add_piece(r, moved(ml.x, M0, a.scale), ml.y, o_at(i, row));
        }
        __syncthreads();  // part_l is read
        part[grp][d / 4] = r.acc;
        if (d == 0) part_l[grp] = r.L;
        __syncthreads();
        if (grp == 0) {
            r = JoinRow{0.0f, make_float4(0, 0, 0, 0)};
#pragma unroll
            for (uint32_t j = 0; j < kGroups; ++j) add_piece(r, 1.0f, part_l[j], part[j][d / 4]);
            store_row(out_row<T>(a, p.token, p.row0 + row, p.g, D) + d, r);
        }
    }
}

// ---------------------------------------------------------------------- host
struct Space {
    size_t few_p, many_p, few_ml, many_ml, few_o, many_o, bytes;
    uint32_t few_slot, many_slot;
};

// Pieces of the two kernels: 2 slots per workgroup, of as many rows as a tile can have.
Space space_of(uint32_t dim, uint32_t hpk, uint32_t tokens)
{
    auto up = [](size_t b) { return (b + 255) / 256 * 256; };
    const uint64_t rows = uint64_t(tokens ? tokens : 1) * hpk;
    Space s{};
    s.few_slot = uint32_t(rows < kFewRows ? rows : kFewRows);
    const uint32_t bm = 32u * uint32_t(many_waves(dim)), wgs = many_wgs(dim);
    s.many_slot = uint32_t(rows <= kFewRows ? 0 : rows < bm ? (rows + 31) / 32 * 32 : bm);  // see piece_place
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += up(bytes);
        return here;
    };
    s.few_p = take(2 * kFewWgs * sizeof(Piece));
    s.many_p = take(2 * wgs * sizeof(Piece));
    s.few_ml = take(2 * kFewWgs * size_t(s.few_slot) * sizeof(float2));
    s.many_ml = take(2 * wgs * size_t(s.many_slot) * sizeof(float2));
    s.few_o = take(2 * kFewWgs * size_t(s.few_slot) * dim * sizeof(float));
    s.many_o = take(2 * wgs * size_t(s.many_slot) * dim * sizeof(float));
    s.bytes = at;
    return s;
}

template <typename T, int D, bool WIDE, bool TREE>
void launch_tiles(const TreeAttn& a, hipStream_t st)
{
    if (a.few_wgs) hipLaunchKernelGGL((k_paged_few<T, D, WIDE, TREE>), dim3(a.few_wgs), dim3(256), 0, st, a);
    if (a.many_wgs)
        hipLaunchKernelGGL((k_paged_many<T, D, many_waves(D), WIDE, TREE>), dim3(a.many_wgs), dim3(many_waves(D) * 64), 0, st, a);
}

template <typename T, int D, bool TREE>
hipError_t launch_paged(const TreeAttn& a, hipStream_t st)
{
    if (a.shift >= 4) launch_tiles<T, D, true, TREE>(a, st);
    else launch_tiles<T, D, false, TREE>(a, st);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL((k_paged_join<T, D>), dim3(2 * (a.few_wgs + many_split(D) * a.many_wgs)), dim3(256), 0, st, a);
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

template <bool TREE>
hipError_t launch_type(const TreeAttn& a, const arc_kv_pages* pages, hipStream_t st)
{
    const bool f16 = pages->dtype == ARC_F16;
    if (pages->head_dim == 64) return f16 ? launch_paged<_Float16, 64, TREE>(a, st) : launch_paged<bf16, 64, TREE>(a, st);
    return f16 ? launch_paged<_Float16, 128, TREE>(a, st) : launch_paged<bf16, 128, TREE>(a, st);
}

int attention(const arc_kv_pages* pages, const arc_paged_batch* batch, const arc_tree* tree, const void* q, uint32_t ldq, uint32_t hpk,
              float scale, uint32_t window, uint32_t sinks, void* out, uint32_t ldo, void* workspace, hipStream_t st)
{
    int rc = check_sizes(pages, batch, hpk);
    if (!rc) rc = check_tables(batch, pages->page_size);
    if (rc) return rc;
    if (tree && (!tree->masks || (window && !batch->positions)))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "null masks, or positions with a window");
    if (tree && (tree->mask_words == 0 || tree->mask_words > ARC_TREE_MAX_WORDS))
        return set_error(ARC_ERR_UNSUPPORTED, "mask_words %u: 1..%u are supported", tree->mask_words, uint32_t(ARC_TREE_MAX_WORDS));
    if (!q || !out || !workspace) return set_error(ARC_ERR_INVALID_ARGUMENT, "null argument");
    const uint32_t width = pages->kv_heads * hpk * pages->head_dim;
    if (ldq < width || ldq % 8 || ldo < width || ldo % 8)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "ldq %u, ldo %u: multiples of 8, at least %u", ldq, ldo, width);
    if (!aligned(q, 16) || !aligned(out, 16)) return set_error(ARC_ERR_INVALID_ARGUMENT, "q and out must be 16-byte aligned");
    if (!aligned(workspace, 256)) return set_error(ARC_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    const float s = scale == 0.0f ? 1.0f / std::sqrt(float(pages->head_dim)) : scale;
    const float s2 = std::fabs(s) * 1.44269504088896f;  // of powers of two
    if (!std::isfinite(s2)) return set_error(ARC_ERR_INVALID_ARGUMENT, "scale %g: finite, at most 2^127", double(scale));
    if (rows_overlap(q, uint64_t(width) * 2, uint64_t(ldq) * 2, out, uint64_t(width) * 2, uint64_t(ldo) * 2, batch->tokens))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "q and out share memory");
    // the line's costs (positions times hpk, over tiles and kv heads) stay below 2^52: times 1024 parts and
    // as doubles they are exact
    const unsigned __int128 most = (unsigned __int128)(uint64_t(batch->tokens) * hpk / kFewRows + batch->requests) *
                                   pages->kv_heads * hpk * (uint64_t(batch->max_pages) * pages->page_size + batch->tokens + 1024);
    if (most >> 52) return set_error(ARC_ERR_UNSUPPORTED, "tokens, heads and max_pages: more work than one call takes");
    if (batch->tokens == 0 || batch->requests == 0) return ARC_OK;
    const Space sp = space_of(pages->head_dim, hpk, batch->tokens);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    TreeAttn a{};
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
    a.scale = s2;
    a.neg = s < 0.0f ? 0x80008000u : 0u;
    if (tree) {
        a.masks = tree->masks;
        a.positions = batch->positions;
        a.words = tree->mask_words;
    }
    a.few_p = reinterpret_cast<Piece*>(ws + sp.few_p);
    a.many_p = reinterpret_cast<Piece*>(ws + sp.many_p);
    a.few_ml = reinterpret_cast<float2*>(ws + sp.few_ml);
    a.many_ml = reinterpret_cast<float2*>(ws + sp.many_ml);
    a.few_o = reinterpret_cast<float*>(ws + sp.few_o);
    a.many_o = reinterpret_cast<float*>(ws + sp.many_o);
    a.few_slot = sp.few_slot;
    a.many_slot = sp.many_slot;
    // which kernels can have work: with no request of more rows than a few-rows tile has, as max_new says, the
    // few-rows kernel takes them all; where tokens, if all are used, leave each request more, the many-rows
    // kernel does (either is right for any request)
    const uint64_t most_rows = uint64_t(batch->max_new < batch->tokens ? batch->max_new : batch->tokens) * hpk;
    const uint64_t others = uint64_t(batch->requests - 1) * batch->max_new;
    const bool many = most_rows > kFewRows;
    const bool few = !many || batch->tokens <= others || (batch->tokens - others) * hpk <= kFewRows;
    a.few_rows = !many ? ~0u : few ? kFewRows : 0u;
    a.few_wgs = few ? kFewWgs : 0;
    a.many_wgs = many ? many_wgs(pages->head_dim) : 0;
    if (tree && many) {
        // one launch where the rows say that trees are the rule: the many-rows kernel has the time for few rows too, as its
        // waves without rows only copy.  48 trees of up to 9 nodes at up to 8000, 32 heads on 8, 99 us (both kernels 106); 16 at
        // 2000 25 (47); but 64 single tokens at up to 8000 with two chunks of 64, 28 heads on 4, 105 (100)
        if (batch->tokens * uint64_t(hpk) >= kFewRows / 2 * uint64_t(batch->requests)) a.few_rows = a.few_wgs = 0;
        a.once = most_rows <= 32u * many_waves(pages->head_dim);
        // no more workgroups than there can be units
        const uint64_t tiles = uint64_t(batch->tokens) * hpk / (32u * many_waves(pages->head_dim)) + batch->requests;
        const uint64_t units = (uint64_t(batch->max_pages) * pages->page_size + kManyKeys - 1) / kManyKeys;
        a.many_wgs = uint32_t(std::min<uint64_t>(a.many_wgs, tiles * pages->kv_heads * units));
    }
    const hipError_t e = tree ? launch_type<true>(a, pages, st) : launch_type<false>(a, pages, st);
    return check_hip(e, tree ? "tree attention" : "paged attention");
}

}  // namespace
}  // namespace arc

using namespace arc;

extern "C" {

size_t arc_paged_attention_workspace_bytes(const arc_kv_pages* pages, const arc_paged_batch* batch, uint32_t hpk)
{
    return check_sizes(pages, batch, hpk) ? 0 : space_of(pages->head_dim, hpk, batch->tokens).bytes;
}

int arc_paged_attention(const arc_kv_pages* pages, const arc_paged_batch* batch, const void* q, uint32_t ldq,
                        uint32_t hpk, float scale, uint32_t window, uint32_t sinks, void* out, uint32_t ldo,
                        void* workspace, arc_stream_t stream)
{
    return attention(pages, batch, nullptr, q, ldq, hpk, scale, window, sinks, out, ldo, workspace, static_cast<hipStream_t>(stream));
}

size_t arc_tree_attention_workspace_bytes(const arc_kv_pages* pages, const arc_paged_batch* batch, uint32_t hpk)
{
    return check_sizes(pages, batch, hpk) ? 0 : space_of(pages->head_dim, hpk, batch->tokens).bytes;
}

int arc_tree_attention(const arc_kv_pages* pages, const arc_paged_batch* batch, const arc_tree* tree, const void* q, uint32_t ldq,
                       uint32_t hpk, float scale, uint32_t window, uint32_t sinks, void* out, uint32_t ldo, void* workspace,
                       arc_stream_t stream)
{
    if (!tree) return set_error(ARC_ERR_INVALID_ARGUMENT, "null tree");
    return attention(pages, batch, tree, q, ldq, hpk, scale, window, sinks, out, ldo, workspace, static_cast<hipStream_t>(stream));
}

}  // extern "C"
