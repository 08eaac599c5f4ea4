// arc_paged_attn.hip -- attention of a serving step's new tokens over the pages of
// their requests (arc_paged.hpp), causal, with an optional sliding window whose
// first tokens stay visible.
//
// Rows.  The hpk query heads of a kv head read the same K and V, so the rows of a
// request and kv head g are its (token, head) pairs, token-major: row r is token
// r / hpk, head g * hpk + r % hpk.  A tile is up to kFewRows (few) or NW * 32 (many) of
// them; it runs over the positions that any of them sees, a unit at a time.
//
// Work.  Requests differ in length by orders of magnitude, and the host does not know
// their lengths.  So the tiles of all requests and kv heads stand in one line, each
// with a cost that the device computes from starts and lens, and workgroup w of G takes
// the w-th of G equal parts of the line, cut wherever it falls, inside a tile too.  A
// tile in one part is written out; a part of one leaves its sums in the workspace
// (Piece) and k_paged_join adds the pieces of a tile in order, so results do not
// depend on timing.
#include "arc_paged.hpp"

#include <cmath>

namespace arc {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
template <typename T>
using vec2 = T __attribute__((ext_vector_type(2)));

constexpr uint32_t kFewRows = 32;      // rows of a few-rows tile
constexpr uint32_t kFewKeys = 128;     // positions of its unit, 32 for each wave
constexpr uint32_t kManyKeys = 64;     // positions of a many-rows tile's unit
constexpr uint32_t kFewWgs = 512;      // most parts of the line
constexpr uint32_t kManyWgs = 512;
constexpr int kManyWaves = 4;
constexpr uint32_t kTileKeys = 64;     // a tile's start and end cost about this many positions
constexpr float kLazy = 8.0f;          // see rescale

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
    float2 *few_ml, *many_ml; // [2 * workgroups][slot rows] running maximum (times scale) and sum
    Piece *few_p, *many_p;
    uint32_t few_slot, many_slot;  // rows of a slot
    uint32_t few_wgs, many_wgs;    // workgroups of this call's launches (0: not launched)
};

// ------------------------------------------------------------------- tiles
// One request: its new rows and positions.
struct Request {
    uint32_t token;   // first row of the step
    uint32_t rows;    // (token, head) pairs per kv head
    int32_t base;     // position of its first new token (negative: rows without a position)
    uint32_t tiles;   // per kv head
    uint64_t first, cap;  // cost of tile 0; no tile costs more than cap
    uint64_t total;       // of a kv head's tiles
};

// Cost of tiles 0 .. t-1: tile t costs min(first + t * bm, cap), in positions times
// hpk; causal tiles grow by bm / hpk positions each.
__device__ __forceinline__ uint64_t cost_before(const Request& r, uint32_t t, uint32_t bm)
{
    if (r.first + uint64_t(t) * bm <= r.cap) return t * r.first + uint64_t(bm) * (uint64_t(t) * (t - 1) / 2);  // t = 0: 0
    const uint64_t k = r.first >= r.cap ? 0 : (r.cap - r.first + bm - 1) / bm;
    return k * r.first + (k ? uint64_t(bm) * (k * (k - 1) / 2) : 0) + (t - k) * r.cap;
}

template <bool FEW>
__device__ __forceinline__ Request request_at(const PagedAttn& a, uint32_t b, uint32_t bm)
{
    Request r{};
    const uint32_t s0 = a.starts[b], s1 = a.starts[b + 1];
    if (s1 <= s0 || s0 >= a.rows) return r;
    const uint32_t fresh = min(s1, a.rows) - s0;
    const uint32_t rows = fresh * a.hpk;
    if (FEW ? rows > a.few_rows : rows <= a.few_rows) return r;
    const uint64_t len = min(uint64_t(a.lens[b]), uint64_t(a.max_pages) << a.shift);
    const int64_t base = int64_t(len) - int64_t(s1 - s0);
    r.token = s0;
    r.rows = rows;
    r.base = int32_t(max(base, -(int64_t(1) << 25)));
    r.tiles = (rows + bm - 1) / bm;
    r.first = uint64_t(kTileKeys + uint32_t(max(r.base, 0))) * a.hpk + bm;
    r.cap = a.window ? (uint64_t(kTileKeys) + a.window + a.sinks) * a.hpk + 2 * bm : ~uint64_t(0);
    r.total = cost_before(r, r.tiles, bm);
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

__device__ __forceinline__ Tile tile_at(const PagedAttn& a, const Request& r, uint32_t t, uint32_t bm, uint32_t keys)
{
    Tile x;
    x.row0 = t * bm;
    x.rows = min(bm, r.rows - x.row0);
    x.pos0 = r.base + int32_t(x.row0 / a.hpk);
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
__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d)
{
    const uint32_t lo = uint32_t(__shfl_up(int(uint32_t(v)), d)), hi = uint32_t(__shfl_up(int(uint32_t(v >> 32)), d));
    return (uint64_t(hi) << 32) | lo;
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return uint32_t(__builtin_amdgcn_readfirstlane(int(v))); }
__device__ __forceinline__ uint64_t uniform(uint64_t v)
{
    return (uint64_t(uniform(uint32_t(v >> 32))) << 32) | uniform(uint32_t(v));
}

struct Line {
    uint64_t total;     // cost of all tiles
    uint32_t parts, w;  // parts of the line, this workgroup's (w >= parts: it has none)
    uint64_t from, to;
    uint32_t b;       // the request in which it begins
    uint64_t before;  // cost of the requests before b
};

// Boundary of part w, the same number wherever it is computed; parts <= total, so no
// part is empty.
__device__ __forceinline__ uint64_t part_at(uint64_t total, uint32_t w, uint32_t parts)
{
    return w >= parts ? total : uint64_t(double(total) * double(w) / double(parts));
}

// Every workgroup adds up all requests (two loads each; thread t takes a run of
// them), so that no launch has to come first.  Workgroups go to the 8 XCDs in turn: an
// XCD's workgroups take neighbouring parts, which read the same K and V.
template <bool FEW, int NT>
__device__ __forceinline__ Line line_of(const PagedAttn& a, uint32_t bm, uint32_t keys, uint64_t* red)
{
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t each = (a.requests + NT - 1) / NT;
    const uint32_t b0 = min(tid * each, a.requests), b1 = min(b0 + each, a.requests);
    uint64_t sum = 0;
    for (uint32_t b = b0; b < b1; ++b) sum += request_at<FEW>(a, b, bm).total * a.kv_heads;
    uint64_t inc = sum;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const uint64_t o = shfl_up64(inc, d);
        if (lane >= uint32_t(d)) inc += o;
    }
    if (lane == 63) red[wave] = inc;
    __syncthreads();
    uint64_t before = 0, total = 0;
#pragma unroll
    for (int i = 0; i < NT / kWave; ++i) {
        const uint64_t r = red[i];
        if (uint32_t(i) < wave) before += r;
        total += r;
    }
    Line l;
    l.total = uniform(total);
    const uint64_t fit = l.total / (keys * a.hpk);
    l.parts = uniform(uint32_t(min(uint64_t(gridDim.x), max(fit, uint64_t(l.total != 0)))));
    l.w = blockIdx.x;
    l.from = l.to = 0;
    if (l.w >= l.parts) return l;
    const uint32_t xcd = blockIdx.x & 7u, q = l.parts >> 3, rest = l.parts & 7u;
    l.w = xcd * q + min(xcd, rest) + (blockIdx.x >> 3);
    l.from = part_at(l.total, l.w, l.parts);
    l.to = part_at(l.total, l.w + 1, l.parts);
    const uint64_t lo = before + inc - sum;
    if (lo <= l.from && l.from < lo + sum) {  // one thread, if there is any work
        uint64_t at = lo;
        uint32_t b = b0;
        for (; b < b1; ++b) {
            const uint64_t c = request_at<FEW>(a, b, bm).total * a.kv_heads;
            if (at + c > l.from) break;
            at += c;
        }
        red[NT / kWave] = b;
        red[NT / kWave + 1] = at;
    }
    __syncthreads();
    l.b = uniform(uint32_t(red[NT / kWave]));
    l.before = uniform(red[NT / kWave + 1]);
    return l;
}

// Part of a tile: units [u0, u1) of tile t of kv head g; where it stands in the line.
struct Segment {
    uint32_t g, t, u0, u1;
    uint64_t begin, end;  // the whole tile's
};

// Which of a tile's units lie before x: monotonic in x, the same for both neighbours
// of a cut (the same arithmetic on the same numbers).
__device__ __forceinline__ uint32_t units_before(uint64_t x, uint64_t begin, uint64_t end, uint32_t units)
{
    if (x <= begin) return 0;
    if (x >= end) return units;
    return min(units, uint32_t(double(x - begin) * double(units) / double(end - begin)));
}

__device__ __forceinline__ Segment segment_at(const PagedAttn& a, const Request& r, uint64_t before, uint64_t x, uint64_t to,
                                              uint32_t bm, uint32_t keys, Tile& tile)
{
    Segment s;
    const uint64_t off = x - before;
    uint32_t g = uint32_t(double(off) / double(r.total));
    while (g && uint64_t(g) * r.total > off) --g;
    while (uint64_t(g + 1) * r.total <= off) ++g;
    const uint64_t in = off - uint64_t(g) * r.total;
    uint32_t lo = 0, hi = r.tiles;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (cost_before(r, mid, bm) <= in) lo = mid;
        else hi = mid;
    }
    s.g = uniform(g);
    s.t = uniform(lo);
    tile = tile_at(a, r, s.t, bm, keys);
    s.begin = before + uint64_t(s.g) * r.total + cost_before(r, s.t, bm);
    s.end = before + uint64_t(s.g) * r.total + cost_before(r, s.t + 1, bm);
    s.u0 = units_before(x, s.begin, s.end, tile.units);
    s.u1 = units_before(to, s.begin, s.end, tile.units);
    s.u0 = uniform(s.u0);
    s.u1 = uniform(s.u1);
    return s;
}

// The workgroup in whose part x lies.
__device__ __forceinline__ uint32_t part_of(const Line& l, uint64_t x)
{
    uint32_t w = min(l.parts - 1, uint32_t(double(x) * double(l.parts) / double(l.total)));
    while (w && part_at(l.total, w, l.parts) > x) --w;
    while (w + 1 < l.parts && part_at(l.total, w + 1, l.parts) <= x) ++w;
    return w;
}

// ------------------------------------------------------------ matrix products
template <typename T>
__device__ __forceinline__ f32x16 mfma(vec8<T> x, vec8<T> y, f32x16 c)
{
    if constexpr (__is_same(T, _Float16)) return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
}

// 8 consecutive values to 16 bits, round to nearest even.
template <typename T>
__device__ __forceinline__ vec8<T> narrow(const f32x16& p, int at)
{
    vec8<T> r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = static_cast<T>(p[at + j]);
    return r;
}

// A K or V row in LDS: D / 8 blocks of 16 bytes, block c of row r at place
// c ^ swizzle(r), so that the 8 or 4 rows that a read touches at once lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t swizzle(uint32_t r)
{
    return D == 128 ? (r & 7u) << 1 : ((r >> 1) & 3u) << 1;
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
        const T* p = rows + r * D + ((block ^ swizzle<D>(r)) << 3) + 4u * (i & 1u);
        part[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
    }
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 both = __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(vec8<T>, both);
}

// Whether any of the two 16-bit values of w is infinite or NaN, and w without them.
template <typename T>
__device__ __forceinline__ bool drop_nonfinite(uint32_t& w)
{
    constexpr uint32_t kExp = __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
    const bool lo = (w & kExp) == kExp, hi = ((w >> 16) & kExp) == kExp;
    if (lo) w &= 0xffff0000u;
    if (hi) w &= 0x0000ffffu;
    return lo || hi;
}

__device__ __forceinline__ bool sees(int32_t qpos, int32_t kpos, uint32_t window, uint32_t sinks)
{
    return kpos <= qpos && (window == 0 || uint32_t(qpos - kpos) < window || uint32_t(kpos) < sinks);
}

// Running softmax of one query (a lane and its partner lane ^ 32, each with half of the
// keys): `m` is the reference that weights 2^(score - m) are relative to, `l` the lane's share of
// their sum.  m follows the maximum only when that has grown by more than kLazy: weights then
// reach 2^kLazy instead of 1, which costs no accuracy (relative rounding) and saves nearly
// every rescaling of the output.
template <int NO>
__device__ __forceinline__ void rescale(float mx, float& m, float& l, f32x16 (&o)[NO])
{
    if (__ballot(mx > m + kLazy) == 0) return;  // m = -inf: any score that is one
    const float to = fmaxf(m, mx);
    const float f = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
    m = to;
    l *= f;
#pragma unroll
    for (int t = 0; t < NO; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] *= f;
}

// Value i of a score or output tile of 32: key, or dim, 8 (i / 4) + 4 (lane / 32) + i % 4.
__device__ __forceinline__ uint32_t tile_index(int i) { return 8u * (i >> 2) + 4u * ((threadIdx.x >> 5) & 1u) + (i & 3); }

// What infinities and NaN of V at positions that only some of a tile's rows see have to
// add: their places in V were cleared for the product, where a weight of 0 would make NaN
// of them; here each row that sees the position gets them.  keys: bit k set where position k0 + k
// holds one; at: element offset of lane k's position (same for V and K).
template <typename T, int D>
__device__ __forceinline__ void add_nonfinite(f32x16 (&o)[D / 32], const T* v, uint64_t keys, int32_t k0, uint64_t at,
                                           int32_t qpos, uint32_t window, uint32_t sinks)
{
    while (keys) {
        const int k = __builtin_ctzll(keys);
        keys &= keys - 1;
        const uint64_t off = (uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(at >> 32)), k))) << 32) |
                             uint32_t(__builtin_amdgcn_readlane(int(uint32_t(at)), k));
        if (!sees(qpos, k0 + k, window, sinks)) continue;
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float x = static_cast<float>(v[off + 32 * t + tile_index(i)]);
                if (!(fabsf(x) < INFINITY)) o[t][i] += x;
            }
    }
}

// Query operand of 32 rows: lane -> row lane & 31, dims 16 s + 8 (lane / 32) .. + 7; zeros for
// rows that the tile does not have.
template <typename T, int D>
__device__ __forceinline__ void load_q(const PagedAttn& a, const Request& r, uint32_t row, bool in, uint32_t g, vec8<T> (&q)[D / 16])
{
    const uint32_t h2 = (threadIdx.x >> 5) & 1u;
    const uint32_t tok = row / a.hpk, h = row - tok * a.hpk;
    const T* p = static_cast<const T*>(a.q) + uint64_t(r.token + tok) * a.ldq + (g * a.hpk + h) * D + 8 * h2;
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

// The slot of a piece, and its record for k_paged_join.
__device__ __forceinline__ uint32_t write_piece(Piece* pieces, const Line& l, const Segment& s, const Request& r, const Tile& x)
{
    const uint32_t w0 = part_of(l, s.begin), w1 = part_of(l, s.end - 1);
    const uint32_t first = 2 * w0 + (part_at(l.total, w0, l.parts) < s.begin ? 1u : 0u);
    const uint32_t slot = l.w == w0 ? first : 2 * l.w;
    if (threadIdx.x == 0) pieces[slot] = Piece{w1 - w0 + 1, l.w - w0, w0, first, r.token, x.row0, x.rows, s.g};
    return slot;
}

// ------------------------------------------------------------------ few rows
// Tiles of up to 32 rows: decode, short chunks.  Bound by reading K and V once.  4
// waves, each on its own 32 positions of a unit with its own softmax, joined through LDS
// at the tile's end; nothing but that join needs a barrier.  Lane -> position
// lane & 31, half of the row's 16-byte blocks: one address serves K and V, and
// K's registers are the score product's operand as they come (S^T = K Q^T; lane -> query).
// V goes through LDS for its transposed operand (O^T = V^T P^T), P^T comes straight from the
// scores' registers.  The next unit's K and V are loaded while this one is computed.
template <typename T, int D>
struct KvRegs {
    uint4 k[D / 16], v[D / 16];
};

template <typename T, int D>
__device__ __forceinline__ void load_kv(KvRegs<T, D>& r, const T* k, const T* v, uint64_t at)
{
    const uint32_t h2 = (threadIdx.x >> 5) & 1u;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) r.k[s] = *reinterpret_cast<const uint4*>(k + at + 16 * s + 8 * h2);
#pragma unroll
    for (int s = 0; s < D / 16; ++s) r.v[s] = *reinterpret_cast<const uint4*>(v + at + 16 * s + 8 * h2);
}

template <typename T, int D>
struct FewState {
    vec8<T> q[D / 16];
    f32x16 o[D / 32];
    float m, l;
};

// One wave's 32 positions from k0 on.  `in`: the lane's position has a page.
template <typename T, int D>
__device__ __forceinline__ void few_unit(const PagedAttn& a, FewState<T, D>& st, KvRegs<T, D>& r, T* vrows, const T* v, int32_t k0,
                                         uint64_t at, bool in, const Tile& x, int32_t qpos)
{
    const uint32_t lane = threadIdx.x & 63u, l32 = lane & 31u, h2 = lane >> 5;
    const uint64_t valid = __ballot(in);
    const bool whole = uint32_t(valid) == 0xffffffffu && k0 + 31 <= x.pos0 &&
                       (a.window == 0 || uint32_t(x.pos1 - k0) < a.window || uint32_t(k0) + 32u <= a.sinks);
    uint64_t odd = 0;  // positions with infinities or NaN in V
    if (!whole) {
        bool any = false;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&r.v[s]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (!in) w[i] = 0;
                any |= drop_nonfinite<T>(w[i]);
            }
        }
        odd = __ballot(any);
        odd = (odd | (odd >> 32)) & 0xffffffffu;
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
        *reinterpret_cast<uint4*>(vrows + l32 * D + (((2u * s + h2) ^ swizzle<D>(l32)) << 3)) = r.v[s];
    f32x16 sc;
#pragma unroll
    for (int i = 0; i < 16; ++i) sc[i] = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) sc = mfma<T>(__builtin_bit_cast(vec8<T>, r.k[s]), st.q[s], sc);
    float mx = -INFINITY;
    if (whole) {
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t j = tile_index(i);
            const bool see = ((uint32_t(valid) >> j) & 1u) && sees(qpos, k0 + int32_t(j), a.window, a.sinks);
            sc[i] = see ? sc[i] : -INFINITY;
            mx = fmaxf(mx, sc[i]);
        }
    }
    mx = xor_max<32>(mx) * a.scale;
    rescale(mx, st.m, st.l, st.o);
    const float mr = st.m == -INFINITY ? 0.0f : st.m;  // nothing seen yet: all weights 0
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        sc[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], a.scale, -mr));
        sum += sc[i];
    }
    st.l += sum;
    // the wave's own V rows: its writes above come before these reads
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const vec8<T> p = narrow<T>(sc, 8 * s);
#pragma unroll
        for (int t = 0; t < D / 32; ++t) st.o[t] = mfma<T>(load_vt<T, D>(vrows, s, t), p, st.o[t]);
    }
    if (odd) add_nonfinite<T, D>(st.o, v, odd, k0, at, qpos, a.window, a.sinks);
    // the next unit's V overwrites these rows
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void k_paged_few(PagedAttn a)
{
    __shared__ uint64_t red[6];
    __shared__ __align__(16) float joined[4 * 32 * D];  // V rows of each wave, then the waves' outputs
    __shared__ float mw[4][32], lw[4][32];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, l32 = lane & 31u, wave = uniform(tid >> 6);
    const Line line = line_of<true, 256>(a, kFewRows, kFewKeys, red);
    if (tid < 2) a.few_p[2 * line.w + tid].n = 0;
    T* vrows = reinterpret_cast<T*>(joined) + wave * (32 * D);
    const T* k = static_cast<const T*>(a.k);
    const T* v = static_cast<const T*>(a.v);
    const uint32_t kvd = a.kv_heads * D, place = (1u << a.shift) - 1u;
    uint32_t b = line.b;
    uint64_t before = line.before;
    Request r{};
    for (uint64_t at = line.from; at < line.to;) {
        for (;; ++b) {  // the request at `at`
            r = request_at<true>(a, b, kFewRows);
            if (at < before + r.total * a.kv_heads) break;
            before += r.total * a.kv_heads;
        }
        Tile x;
        const Segment s = segment_at(a, r, before, at, line.to, kFewRows, kFewKeys, x);
        const uint32_t row = min(l32, x.rows - 1);
        const int32_t qpos = r.base + int32_t((x.row0 + row) / a.hpk);
        const uint32_t* table = a.tables + uint64_t(b) * a.max_pages;
        FewState<T, D> st;
        load_q<T, D>(a, r, x.row0 + row, l32 < x.rows, s.g, st.q);
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) st.o[t][i] = 0.0f;
        st.m = -INFINITY;
        st.l = 0.0f;

        // page of the lane's position in unit u: loaded a unit ahead of the K and V it points to
        auto key_of = [&](uint32_t u) { return int32_t(unit_start(x, u, kFewKeys) + 32u * wave + l32); };
        auto page_of = [&](uint32_t u) {
            const int32_t kp = key_of(u);
            return kp <= x.pos1 ? table[uint32_t(kp) >> a.shift] : 0xffffffffu;
        };
        auto offset_of = [&](uint32_t page, uint32_t u) {
            const uint32_t kp = uint32_t(key_of(u));
            return page < a.num_pages ? uint64_t(page) * a.page_stride + uint64_t(kp & place) * kvd + s.g * D : uint64_t(0);
        };
        if (s.u0 < s.u1) {
            KvRegs<T, D> cur, nxt;
            uint32_t page = page_of(s.u0);
            uint64_t off = offset_of(page, s.u0);
            load_kv(cur, k, v, off);
            uint32_t npage = s.u0 + 1 < s.u1 ? page_of(s.u0 + 1) : 0xffffffffu;
            for (uint32_t u = s.u0; u < s.u1; ++u) {
                uint64_t noff = 0;
                uint32_t far = 0xffffffffu;
                if (u + 1 < s.u1) {
                    noff = offset_of(npage, u + 1);
                    load_kv(nxt, k, v, noff);
                    if (u + 2 < s.u1) far = page_of(u + 2);
                }
                few_unit<T, D>(a, st, cur, vrows, v, int32_t(unit_start(x, u, kFewKeys) + 32u * wave), off, page < a.num_pages, x,
                               qpos);
                cur = nxt;
                off = noff;
                page = npage;
                npage = far;
            }
        }
        // the waves' states in wave order: out = sum_w 2^(m_w - M) o_w / sum_w 2^(m_w - M) l_w
        __syncthreads();  // every wave is done with its V rows
        const float l = xor_sum<32>(st.l);
        if (l32 < x.rows) {
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4*>(&joined[(wave * 32 + l32) * D + 32 * t + tile_index(i)]) =
                        make_float4(st.o[t][i], st.o[t][i + 1], st.o[t][i + 2], st.o[t][i + 3]);
            if (lane < 32) {
                mw[wave][l32] = st.m;
                lw[wave][l32] = l;
            }
        }
        __syncthreads();
        const bool complete = at <= s.begin && s.end <= line.to;
        uint32_t slot = 0;
        if (!complete) slot = write_piece(a.few_p, line, s, r, x);
        for (uint32_t e = tid; e < x.rows * (D / 4); e += 256) {
            const uint32_t rr = e / (D / 4), d = 4 * (e % (D / 4));
            float M = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) M = fmaxf(M, mw[i][rr]);
            const float M0 = M == -INFINITY ? 0.0f : M;
            float L = 0.0f;
            float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = __builtin_amdgcn_exp2f(mw[i][rr] - M0);
                const float4 o = *reinterpret_cast<const float4*>(&joined[(i * 32 + rr) * D + d]);
                L = __builtin_fmaf(lw[i][rr], f, L);
                acc.x = __builtin_fmaf(o.x, f, acc.x);
                acc.y = __builtin_fmaf(o.y, f, acc.y);
                acc.z = __builtin_fmaf(o.z, f, acc.z);
                acc.w = __builtin_fmaf(o.w, f, acc.w);
            }
            if (complete) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // nothing seen: zeros
                store4<T>(out_row<T>(a, r.token, x.row0 + rr, s.g, D) + d, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            } else {
                *reinterpret_cast<float4*>(a.few_o + (uint64_t(slot) * a.few_slot + rr) * D + d) = acc;
                if (d == 0) a.few_ml[uint64_t(slot) * a.few_slot + rr] = make_float2(M, L);
            }
        }
        __syncthreads();  // the next tile's V rows overwrite `joined`
        at = min(s.end, line.to);
    }
}

// ----------------------------------------------------------------- many rows
// Tiles of NW * 32 rows: prompts and long chunks.  Bound by the matrix cores and the
// softmax's vector instructions.  Each wave holds 32 rows (Q, O in registers); the
// unit's 64 rows of K and V come through LDS, shared by the waves and double buffered:
// while unit u is computed from one buffer, unit u + 1 is on its way to registers, and is
// written to the other buffer at the end; one barrier per unit.  Operands as in the
// few-rows kernel, K's read from LDS.
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, 2) void k_paged_many(PagedAttn a)
{
    constexpr int NT = NW * 64;
    constexpr uint32_t kBm = NW * 32;
    constexpr int kBlocks = D / 8;                       // 16-byte blocks of a row
    constexpr int kRows = NT / kBlocks;                  // rows staged at a time
    constexpr int kPass = kManyKeys / kRows;
    static_assert(kPass >= 1 && kPass * kRows == int(kManyKeys), "staging covers the unit");
    __shared__ uint64_t red[NW + 2];
    __shared__ __align__(16) T ks[2][kManyKeys * D];
    __shared__ __align__(16) T vs[2][kManyKeys * D];
    __shared__ uint32_t odd_bits[3][2];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, l32 = lane & 31u, h2 = lane >> 5, wave = uniform(tid >> 6);
    const Line line = line_of<false, NT>(a, kBm, kManyKeys, red);
    if (tid < 2) a.many_p[2 * line.w + tid].n = 0;
    const T* k = static_cast<const T*>(a.k);
    const T* v = static_cast<const T*>(a.v);
    const uint32_t kvd = a.kv_heads * D, place = (1u << a.shift) - 1u;
    const uint32_t sr = tid / kBlocks, sb = tid % kBlocks;  // staged row (of a pass) and block
    uint32_t b = line.b;
    uint64_t before = line.before;
    Request r{};
    for (uint64_t at = line.from; at < line.to;) {
        for (;; ++b) {
            r = request_at<false>(a, b, kBm);
            if (at < before + r.total * a.kv_heads) break;
            before += r.total * a.kv_heads;
        }
        Tile x;
        const Segment s = segment_at(a, r, before, at, line.to, kBm, kManyKeys, x);
        const uint32_t trow = wave * 32 + l32;
        const uint32_t row = min(trow, x.rows - 1);
        const int32_t qpos = r.base + int32_t((x.row0 + row) / a.hpk);
        const uint32_t* table = a.tables + uint64_t(b) * a.max_pages;
        vec8<T> q[D / 16];
        load_q<T, D>(a, r, x.row0 + row, trow < x.rows, s.g, q);
        f32x16 o[D / 32];
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
        float m = -INFINITY, l = 0.0f;

        // lane -> position lane of unit u: its page (loaded a unit ahead), then its element offset
        auto page_of = [&](uint32_t u) {
            const int32_t kp = int32_t(unit_start(x, u, kManyKeys) + lane);
            return kp <= x.pos1 ? table[uint32_t(kp) >> a.shift] : 0xffffffffu;
        };
        auto offset_of = [&](uint32_t page, uint32_t u) {
            const uint32_t kp = unit_start(x, u, kManyKeys) + lane;
            return page < a.num_pages ? uint64_t(page) * a.page_stride + uint64_t(kp & place) * kvd + s.g * D : uint64_t(0);
        };
        auto is_whole = [&](uint64_t valid, int32_t k0) {
            return valid == ~uint64_t(0) && k0 + int32_t(kManyKeys) - 1 <= x.pos0 &&
                   (a.window == 0 || uint32_t(x.pos1 - k0) < a.window || uint32_t(k0) + kManyKeys <= a.sinks);
        };
        uint4 sk[kPass], sv[kPass];
        auto fetch = [&](uint64_t off) {  // this thread's blocks of the unit whose positions lie at `off` (by lane)
#pragma unroll
            for (int i = 0; i < kPass; ++i) {
                const int src = int(sr + i * kRows);
                const uint64_t row_off = (uint64_t(uint32_t(__shfl(int(uint32_t(off >> 32)), src))) << 32) |
                                         uint32_t(__shfl(int(uint32_t(off)), src));
                sk[i] = *reinterpret_cast<const uint4*>(k + row_off + 8 * sb);
                sv[i] = *reinterpret_cast<const uint4*>(v + row_off + 8 * sb);
            }
        };
        auto stage = [&](int buf, int bits, uint64_t valid, bool whole) {
#pragma unroll
            for (int i = 0; i < kPass; ++i) {
                const uint32_t rr = sr + i * kRows;
                if (!whole) {
                    uint32_t* vw = reinterpret_cast<uint32_t*>(&sv[i]);
                    const bool in = (valid >> rr) & 1u;
                    bool any = false;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (!in) vw[j] = 0;
                        any |= drop_nonfinite<T>(vw[j]);
                    }
                    if (any) atomicOr(&odd_bits[bits][rr >> 5], 1u << (rr & 31u));
                }
                const uint32_t to = rr * D + ((sb ^ swizzle<D>(rr)) << 3);
                *reinterpret_cast<uint4*>(&ks[buf][to]) = sk[i];
                *reinterpret_cast<uint4*>(&vs[buf][to]) = sv[i];
            }
        };

        if (s.u0 < s.u1) {
            // bits of unit u in odd_bits[(u - u0) % 3]: cleared two units ahead
            if (tid < 6) odd_bits[tid >> 1][tid & 1u] = 0;
            uint32_t page = page_of(s.u0);
            uint64_t off = offset_of(page, s.u0);
            uint64_t valid = __ballot(page < a.num_pages);
            bool whole = is_whole(valid, int32_t(unit_start(x, s.u0, kManyKeys)));
            fetch(off);
            uint32_t npage = s.u0 + 1 < s.u1 ? page_of(s.u0 + 1) : 0xffffffffu;
            __syncthreads();
            stage(0, 0, valid, whole);
            __syncthreads();
            int cur = 0, bits = 0;
            for (uint32_t u = s.u0; u < s.u1; ++u) {
                const int32_t k0 = int32_t(unit_start(x, u, kManyKeys));
                uint64_t noff = 0, nvalid = 0;
                bool nwhole = true;
                const int nbits = bits == 2 ? 0 : bits + 1;
                if (u + 1 < s.u1) {
                    noff = offset_of(npage, u + 1);
                    nvalid = __ballot(npage < a.num_pages);
                    nwhole = is_whole(nvalid, int32_t(unit_start(x, u + 1, kManyKeys)));
                    fetch(noff);
                    npage = u + 2 < s.u1 ? page_of(u + 2) : 0xffffffffu;
                }
                if (tid < 2) odd_bits[nbits == 2 ? 0 : nbits + 1][tid] = 0;

                f32x16 sc[2];
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) sc[kt][i] = 0.0f;
#pragma unroll
                    for (int st = 0; st < D / 16; ++st) {
                        const uint32_t rr = 32u * kt + l32;
                        const vec8<T> kf =
                            *reinterpret_cast<const vec8<T>*>(&ks[cur][rr * D + (((2u * st + h2) ^ swizzle<D>(rr)) << 3)]);
                        sc[kt] = mfma<T>(kf, q[st], sc[kt]);
                    }
                }
                float mx = -INFINITY;
                if (!whole) {
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const uint32_t j = 32u * kt + tile_index(i);
                            const bool see = ((valid >> j) & 1u) && sees(qpos, k0 + int32_t(j), a.window, a.sinks);
                            sc[kt][i] = see ? sc[kt][i] : -INFINITY;
                        }
                }
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kt][i]);
                mx = xor_max<32>(mx) * a.scale;
                rescale(mx, m, l, o);
                const float mr = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        sc[kt][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kt][i], a.scale, -mr));
                        l += sc[kt][i];
                    }
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    const vec8<T> p = narrow<T>(sc[st >> 1], 8 * (st & 1));
#pragma unroll
                    for (int t = 0; t < D / 32; ++t) o[t] = mfma<T>(load_vt<T, D>(vs[cur], st, t), p, o[t]);
                }
                if (!whole) {
                    const uint64_t odd = (uint64_t(odd_bits[bits][1]) << 32) | odd_bits[bits][0];
                    if (odd) add_nonfinite<T, D>(o, v, uniform(odd), k0, off, qpos, a.window, a.sinks);
                }
                if (u + 1 < s.u1) stage(cur ^ 1, nbits, nvalid, nwhole);
                __syncthreads();
                cur ^= 1;
                bits = nbits;
                off = noff;
                valid = nvalid;
                whole = nwhole;
            }
        }
        const float L = xor_sum<32>(l);
        const bool complete = at <= s.begin && s.end <= line.to;
        uint32_t slot = 0;
        if (!complete) slot = write_piece(a.many_p, line, s, r, x);
        if (trow < x.rows) {
            if (complete) {
                const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                T* dst = out_row<T>(a, r.token, x.row0 + trow, s.g, D);
#pragma unroll
                for (int t = 0; t < D / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        store4<T>(dst + 32 * t + tile_index(i), o[t][i] * inv, o[t][i + 1] * inv, o[t][i + 2] * inv,
                                  o[t][i + 3] * inv);
            } else {
                float* dst = a.many_o + (uint64_t(slot) * a.many_slot + trow) * D;
#pragma unroll
                for (int t = 0; t < D / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        *reinterpret_cast<float4*>(dst + 32 * t + tile_index(i)) =
                            make_float4(o[t][i], o[t][i + 1], o[t][i + 2], o[t][i + 3]);
                if (h2 == 0) a.many_ml[uint64_t(slot) * a.many_slot + trow] = make_float2(m, L);
            }
        }
        at = min(s.end, line.to);
        __syncthreads();  // the next tile's first unit overwrites LDS
    }
}

// ---------------------------------------------------------------------- join
// Adds the pieces of the tiles that were cut, in order: out = sum_i 2^(m_i - M) o_i /
// sum_i 2^(m_i - M) l_i.  One group of workgroups per slot; the n workgroup groups of a tile's
// n pieces share its rows, a row at a time: D / 4 lanes across, 256 / (D / 4) pieces
// at once.
constexpr uint32_t kJoinSplit = 4;
template <typename T, int D>
__global__ __launch_bounds__(256) void k_paged_join(PagedAttn a)
{
    constexpr uint32_t kLanes = D / 4, kGroups = 256 / kLanes;
    __shared__ __align__(16) float4 part[kGroups][kLanes];
    __shared__ float part_l[kGroups];
    const uint32_t few = 2 * a.few_wgs;
    const bool is_few = blockIdx.x < few;
    const uint32_t own = is_few ? blockIdx.x : blockIdx.x - few;
    const Piece p = (is_few ? a.few_p : a.many_p)[own];
    if (p.n == 0) return;
    const float* po = is_few ? a.few_o : a.many_o;
    const float2* pml = is_few ? a.few_ml : a.many_ml;
    const uint32_t srows = is_few ? a.few_slot : a.many_slot;
    const uint32_t tid = threadIdx.x, grp = tid / kLanes, d = tid % kLanes;
    auto slot_of = [&](uint32_t i) { return uint64_t(i ? 2 * (p.wg + i) : p.slot); };
    for (uint32_t row = p.idx * kJoinSplit + blockIdx.y; row < p.rows; row += p.n * kJoinSplit) {
        float M = -INFINITY;
        for (uint32_t i = grp; i < p.n; i += kGroups) M = fmaxf(M, pml[slot_of(i) * srows + row].x);
        __syncthreads();  // the row before is done with part
        if (d == 0) part_l[grp] = M;
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < kGroups; ++j) M = fmaxf(M, part_l[j]);
        const float M0 = M == -INFINITY ? 0.0f : M;
        float L = 0.0f;
        float4 acc = make_float4(0, 0, 0, 0);
        for (uint32_t i = grp; i < p.n; i += kGroups) {
            const float2 ml = pml[slot_of(i) * srows + row];
            const float f = __builtin_amdgcn_exp2f(ml.x - M0);
            const float4 o = *reinterpret_cast<const float4*>(po + (slot_of(i) * srows + row) * D + 4 * d);
            L = __builtin_fmaf(ml.y, f, L);
            acc.x = __builtin_fmaf(o.x, f, acc.x);
            acc.y = __builtin_fmaf(o.y, f, acc.y);
            acc.z = __builtin_fmaf(o.z, f, acc.z);
            acc.w = __builtin_fmaf(o.w, f, acc.w);
        }
        __syncthreads();  // part_l is read
        part[grp][d] = acc;
        if (d == 0) part_l[grp] = L;
        __syncthreads();
        if (grp == 0) {
            L = 0.0f;
            acc = make_float4(0, 0, 0, 0);
#pragma unroll
            for (uint32_t j = 0; j < kGroups; ++j) {
                const float4 o = part[j][d];
                L += part_l[j];
                acc.x += o.x;
                acc.y += o.y;
                acc.z += o.z;
                acc.w += o.w;
            }
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            store4<T>(out_row<T>(a, p.token, p.row0 + row, p.g, D) + 4 * d, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
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
    s.many_slot = uint32_t(rows <= kFewRows ? 0 : rows < kManyWaves * 32 ? rows : kManyWaves * 32);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += up(bytes);
        return here;
    };
    s.few_p = take(2 * kFewWgs * sizeof(Piece));
    s.many_p = take(2 * kManyWgs * sizeof(Piece));
    s.few_ml = take(2 * kFewWgs * size_t(s.few_slot) * sizeof(float2));
    s.many_ml = take(2 * kManyWgs * size_t(s.many_slot) * sizeof(float2));
    s.few_o = take(2 * kFewWgs * size_t(s.few_slot) * dim * sizeof(float));
    s.many_o = take(2 * kManyWgs * size_t(s.many_slot) * dim * sizeof(float));
    s.bytes = at;
    return s;
}

template <typename T, int D>
hipError_t launch_paged(const PagedAttn& a, hipStream_t st)
{
    if (a.few_wgs) hipLaunchKernelGGL((k_paged_few<T, D>), dim3(a.few_wgs), dim3(256), 0, st, a);
    if (hipError_t e = hipGetLastError()) return e;
    if (a.many_wgs)
        hipLaunchKernelGGL((k_paged_many<T, D, kManyWaves>), dim3(a.many_wgs), dim3(kManyWaves * 64), 0, st, a);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL((k_paged_join<T, D>), dim3(2 * (a.few_wgs + a.many_wgs), kJoinSplit), dim3(256), 0, st, a);
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
    return check_sizes(pages, batch, hpk) ? 0 : space_of(pages->head_dim, hpk, batch->tokens).bytes;
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
    // the line's costs (positions times hpk, over tiles and kv heads) stay below 2^52: times 1024 parts and
    // as doubles they are exact
    const unsigned __int128 most = (unsigned __int128)(uint64_t(batch->tokens) * hpk / kFewRows + batch->requests) *
                                   pages->kv_heads * hpk * (uint64_t(batch->max_pages) * pages->page_size + 1024);
    if (most >> 52) return set_error(ARC_ERR_UNSUPPORTED, "tokens, heads and max_pages: more work than one call takes");
    if (batch->tokens == 0 || batch->requests == 0) return ARC_OK;
    const Space sp = space_of(pages->head_dim, hpk, batch->tokens);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
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
    const float s = scale == 0.0f ? 1.0f / std::sqrt(float(pages->head_dim)) : scale;
    a.scale = std::fabs(s) * 1.44269504088896f;
    a.neg = s < 0.0f ? 0x80008000u : 0u;
    a.few_p = reinterpret_cast<Piece*>(ws + sp.few_p);
    a.many_p = reinterpret_cast<Piece*>(ws + sp.many_p);
    a.few_ml = reinterpret_cast<float2*>(ws + sp.few_ml);
    a.many_ml = reinterpret_cast<float2*>(ws + sp.many_ml);
    a.few_o = reinterpret_cast<float*>(ws + sp.few_o);
    a.many_o = reinterpret_cast<float*>(ws + sp.many_o);
    a.few_slot = sp.few_slot;
    a.many_slot = sp.many_slot;
    // which kernels can have work: no request has more rows than max_new says, and then the few-rows
    // kernel takes them all; a single request with more goes to the many-rows kernel whatever it holds
    const uint64_t most_rows = uint64_t(batch->max_new < batch->tokens ? batch->max_new : batch->tokens) * hpk;
    const bool many = most_rows > kFewRows, few = !many || batch->requests > 1;
    a.few_rows = !many ? ~0u : few ? kFewRows : 0u;
    a.few_wgs = few ? kFewWgs : 0;
    a.many_wgs = many ? kManyWgs : 0;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const bool f16 = pages->dtype == ARC_F16;
    const hipError_t e = pages->head_dim == 64 ? (f16 ? launch_paged<_Float16, 64>(a, st) : launch_paged<bf16, 64>(a, st))
                                               : (f16 ? launch_paged<_Float16, 128>(a, st) : launch_paged<bf16, 128>(a, st));
    return check_hip(e, "paged attention");
}

}  // extern "C"
