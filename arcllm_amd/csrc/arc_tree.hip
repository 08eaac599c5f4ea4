// arc_tree.hip -- a step that verifies trees of drafted tokens: masks and positions from
// the parents, and the step's end (the target's tokens, the walk down each tree, the
// accepted rows' move in every layer's pages, the pages that go back).
//
// A request's rows are a tree if they are no more than 32 * mask_words, else a prompt's
// chunk.  Node i's parent is a node before it.
#include "arc_paged.hpp"

#include <algorithm>
#include <iterator>

namespace arc {
namespace {

constexpr uint32_t kMaxLogitRows = 1u << 20;
constexpr uint32_t kMaxNodes = 32 * ARC_TREE_MAX_WORDS;

// The rows of request b that the step has, and how many starts says; the context's length.
struct Rows {
    uint32_t first, n, all;
};
__device__ __forceinline__ Rows rows_of(const uint32_t* starts, uint32_t tokens, uint32_t b)
{
    const uint32_t s0 = starts[b], s1 = starts[b + 1], end = min(s1, tokens);
    return Rows{s0, s0 < end ? end - s0 : 0u, s1 > s0 ? s1 - s0 : 0u};
}
__device__ __forceinline__ uint32_t base_of(uint32_t len, const Rows& r) { return len > r.all ? len - r.all : 0u; }

// -------------------------------------------------------------------- plan
struct TreePlan {
    const uint32_t *lens, *starts, *parents;
    uint32_t *masks, *positions;
    uint32_t requests, tokens, words;
};

// A workgroup to a request, a lane to a node: it climbs from its node to the root, in LDS, and writes each word of its
// mask when it has left it behind.  A climb is a chain of LDS reads (some 60 ns each): the tree's depth bounds it.  One
// tree of 26 nodes 3.5 us, 500 of up to 60 nodes 3.8: the launch.
__global__ __launch_bounds__(256) void k_tree_plan(TreePlan a)
{
    __shared__ uint32_t parent[kMaxNodes];
    const uint32_t b = blockIdx.x, tid = threadIdx.x;
    const Rows r = rows_of(a.starts, a.tokens, b);
    if (r.n == 0) return;
    const uint32_t base = base_of(a.lens[b], r);
    if (r.n > 32 * a.words) {  // a chunk
        for (uint32_t i = tid; i < r.n; i += 256) a.positions[r.first + i] = base + i;
        return;
    }
    for (uint32_t i = tid; i < r.n; i += 256) parent[i] = a.parents[r.first + i];
    __syncthreads();
    for (uint32_t i = tid; i < r.n; i += 256) {
        uint32_t* out = a.masks + uint64_t(r.first + i) * a.words;
        uint32_t word = i >> 5, bits = 0, depth = 0, at = i;
        for (uint32_t w = word + 1; w < a.words; ++w) out[w] = 0;
        for (;;) {
            bits |= 1u << (at & 31u);
            const uint32_t up = parent[at];
            if (up >= at) break;  // none, or not a node before this one
            ++depth;
            if ((up >> 5) != word) {
                out[word] = bits;
                bits = 0;
                while (--word != (up >> 5)) out[word] = 0;
            }
            at = up;
        }
        out[word] = bits;
        while (word) out[--word] = 0;
        a.positions[r.first + i] = base + depth;
    }
}

// ------------------------------------------------------------ target tokens
struct Best {
    float val;
    uint32_t idx;
};
// The larger value, the lower index of equals; NaN is below all numbers.
__device__ __forceinline__ Best better(const Best& a, const Best& b)
{
    return b.val > a.val || (b.val == a.val && b.idx < a.idx) ? b : a;
}
template <typename T>
__device__ __forceinline__ void take(Best& best, T v, uint32_t i)
{
    const float f = static_cast<float>(v);
    if (f > best.val || (f == best.val && i < best.idx)) best = Best{f, i};
}
constexpr uint32_t kNoToken = 0xffffffffu;

struct Argmax {
    const void* logits;
    const uint32_t* starts;
    Best* parts;  // [tokens][splits]
    uint64_t ldl;
    uint32_t requests, tokens, vocab, splits;
};
// A workgroup to a part of a row; rows behind the last request are not read.  Bound by reading the logits: 16 bytes a lane
// from the first 16-byte border on, four at a time.  A step's end of 24 trees of up to 40 nodes with logits of 152064 in fp32: 70
// to 76 us in all, of which the logits, 365 MB, at 6.2 TB/s, would be 59.
template <typename T>
__global__ __launch_bounds__(256) void k_tree_argmax(Argmax a)
{
    constexpr uint32_t V = 16 / sizeof(T), kAhead = 4;
    typedef T wide __attribute__((ext_vector_type(16 / sizeof(T))));
    __shared__ Best waves[4];
    const uint32_t row = blockIdx.x / a.splits, split = blockIdx.x % a.splits, tid = threadIdx.x;
    if (row >= a.starts[a.requests]) return;
    const T* p = static_cast<const T*>(a.logits) + uint64_t(row) * a.ldl;
    // the row's values before its first border, its wide ones, those behind: the parts share the wide ones
    const uint32_t head = min(uint32_t(-reinterpret_cast<uintptr_t>(p) & 15u) / uint32_t(sizeof(T)), a.vocab);
    const uint32_t n = (a.vocab - head) / V, each = (n + a.splits - 1) / a.splits;
    const uint32_t v0 = min(split * each, n), v1 = min(v0 + each, n);
    const wide* w = reinterpret_cast<const wide*>(p + head);
    Best best{-INFINITY, kNoToken};
    if (split == 0 && tid < head) take(best, p[tid], tid);
    for (uint32_t v = v0 + tid; v < v1; v += kAhead * 256) {
        wide x[kAhead];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) x[i] = __builtin_nontemporal_load(w + min(v + i * 256, v1 - 1));
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i)
#pragma unroll
            for (uint32_t e = 0; e < V; ++e) take(best, x[i][e], head + min(v + i * 256, v1 - 1) * V + e);
    }
    if (split + 1 == a.splits && tid < a.vocab - head - n * V) take(best, p[head + n * V + tid], head + n * V + tid);
    for (int d = 32; d; d >>= 1) best = better(best, Best{__shfl_xor(best.val, d), uint32_t(__shfl_xor(int(best.idx), d))});
    if ((tid & 63u) == 0) waves[tid >> 6] = best;
    __syncthreads();
    if (tid == 0) {
        for (int i = 1; i < 4; ++i) best = better(best, waves[i]);
        a.parts[uint64_t(row) * a.splits + split] = best;
    }
}

// --------------------------------------------------------------------- walk
struct Walk {
    const uint32_t *lens, *starts, *parents, *drafts;
    uint32_t *targets, *lens_out, *counts, *tokens_out;
    uint32_t *path, *held;  // [tokens] the walk's rows; [requests] lens, which lens_out may take the place of
    const Best* parts;
    uint32_t requests, tokens, words, splits;
};

// Request b's target tokens, from the parts of its rows' logits if there are any, then wave 0's way from node 0 to the
// first child that holds the target's token, as long as there is one: 64 nodes a look.  The nodes on a tree's way, 0 for
// what is no tree; what the call gives is written where `writes`.
struct WalkSpace {
    uint32_t parent[kMaxNodes], draft[kMaxNodes], said[kMaxNodes], path[kMaxNodes];
    uint32_t kept;
};
__device__ __forceinline__ uint32_t walk(const Walk& a, uint32_t b, const Rows& r, uint32_t len, bool writes, WalkSpace& l)
{
    const uint32_t tid = threadIdx.x;
    // f(i, the target's token after row i), by one lane for each row: from targets, or as many lanes as a row's logits have
    // parts take one of them each
    auto said_after = [&](auto f) {
        if (!a.splits) {
            for (uint32_t i = tid; i < r.n; i += 256) f(i, a.targets[r.first + i]);
            return;
        }
        const uint32_t part = tid & (a.splits - 1);
        for (uint32_t i = tid / a.splits; i < r.n; i += 256 / a.splits) {
            Best best = a.parts[uint64_t(r.first + i) * a.splits + part];
            for (uint32_t d = a.splits >> 1; d; d >>= 1) best = better(best, Best{__shfl_xor(best.val, int(d)), uint32_t(__shfl_xor(int(best.idx), int(d)))});
            if (part) continue;
            const uint32_t token = best.idx == kNoToken ? 0u : best.idx;
            if (writes) a.targets[r.first + i] = token;
            f(i, token);
        }
    };
    if (r.n == 0 || r.n > 32 * a.words) {
        __syncthreads();  // everyone has read lens
        if (!writes) return 0;
        said_after([&](uint32_t i, uint32_t token) {
            if (i) a.tokens_out[r.first + i] = kNoToken;
            if (i + 1 == r.n) a.tokens_out[r.first] = token;
        });
        if (tid == 0) {
            a.counts[b] = r.n ? 1 : 0;
            a.lens_out[b] = len;
        }
        return 0;
    }
    for (uint32_t i = tid; i < r.n; i += 256) {
        l.parent[i] = a.parents[r.first + i];
        l.draft[i] = a.drafts[r.first + i];
    }
    said_after([&](uint32_t i, uint32_t token) { l.said[i] = token; });
    __syncthreads();
    if (tid < 64) {
        uint32_t node = 0, n = 0;
        for (;;) {
            if (tid == 0) l.path[n] = node;
            ++n;
            const uint32_t want = l.said[node];
            uint32_t next = kNoToken;
            for (uint32_t i = (node + 1) & ~63u; i < r.n; i += 64) {
                const uint32_t c = i + tid;
                const uint64_t fits = __ballot(c > node && c < r.n && l.parent[c] == node && l.draft[c] == want);
                if (fits) {
                    next = i + uint32_t(__builtin_ctzll(fits));
                    break;
                }
            }
            if (next == kNoToken) break;
            node = next;
        }
        if (tid == 0) l.kept = n;
    }
    __syncthreads();
    const uint32_t kept = l.kept;
    if (writes) {
        for (uint32_t i = tid; i < r.n; i += 256) a.tokens_out[r.first + i] = i < kept ? l.said[l.path[i]] : kNoToken;
        if (tid == 0) {
            a.counts[b] = kept;
            a.lens_out[b] = base_of(len, r) + kept;
        }
    }
    return kept;
}

// A workgroup to a request.  Bound by its launch and a chain of three round trips to memory, about 4 us.
__global__ __launch_bounds__(256) void k_tree_walk(Walk a)
{
    __shared__ WalkSpace l;
    const uint32_t b = blockIdx.x;
    const Rows r = rows_of(a.starts, a.tokens, b);
    const uint32_t len = a.lens[b], kept = walk(a, b, r, len, true, l);
    for (uint32_t i = threadIdx.x; i < kept; i += 256) a.path[r.first + i] = l.path[i];
    if (threadIdx.x == 0) a.held[b] = len;
}

// --------------------------------------------------------------------- move
struct Layers {
    void *k[ARC_MAX_LAYERS], *v[ARC_MAX_LAYERS];
};
struct Move {
    const uint32_t *tables, *held, *starts, *counts, *path;
    uint32_t *free_pages, *free_count_out;
    const uint32_t* free_count;
    uint64_t page_bytes;  // from page to page
    uint32_t requests, tokens, words, max_pages, num_pages, list_pages, shift, row_bytes, layers;
};

// The row of position pos in a pool, or none: a page that is none, a position past the table.
__device__ __forceinline__ bool place_of(const Move& a, uint32_t b, uint32_t pos, uint64_t& at)
{
    if ((pos >> a.shift) >= a.max_pages) return false;
    const uint32_t page = a.tables[uint64_t(b) * a.max_pages + (pos >> a.shift)];
    at = uint64_t(page) * a.page_bytes + uint64_t(pos & ((1u << a.shift) - 1u)) * a.row_bytes;
    return page < a.num_pages;
}

// A layer's move: row node(i) of the way, `kept` long, to place i behind base.  A few rows of some KB: a chain of round
// trips to memory (rows, walk, pages, values), so each is made for all rows at once.  Each thread has the same 16 bytes of
// every row and reads 8 rows before it writes any: a row is then read before its place is written, as node(i) >= i and both rise.
struct MoveSpace {
    uint64_t from[kMaxNodes], to[kMaxNodes];  // byte offsets; kNowhere: the row stays
};
template <typename Node>
__device__ __forceinline__ void move_rows(const Move& a, const Layers& layers, uint32_t layer, uint32_t b, uint32_t base, uint32_t kept,
                                          MoveSpace& l, Node node)
{
    constexpr uint32_t kBatch = 8;
    constexpr uint64_t kNowhere = ~0ull;
    const uint32_t tid = threadIdx.x, width = a.row_bytes / 16;
    for (uint32_t i = tid; i < kept; i += 256) {
        const uint32_t n = node(i);
        uint64_t to_at = 0, from_at = 0;
        const bool moves = n != i && place_of(a, b, base + i, to_at) && place_of(a, b, base + n, from_at);
        l.from[i] = moves ? from_at : kNowhere;
        l.to[i] = to_at;
    }
    __syncthreads();
    for (uint32_t c = tid; c < 2 * width; c += 256) {
        uint8_t* pool = static_cast<uint8_t*>(c < width ? layers.k[layer] : layers.v[layer]) + (c < width ? c : c - width) * 16;
        for (uint32_t i0 = 1; i0 < kept; i0 += kBatch) {
            uint4 v[kBatch];
#pragma unroll
            for (uint32_t i = 0; i < kBatch; ++i)
                if (i0 + i < kept && l.from[i0 + i] != kNowhere) v[i] = *reinterpret_cast<const uint4*>(pool + l.from[i0 + i]);
#pragma unroll
            for (uint32_t i = 0; i < kBatch; ++i)
                if (i0 + i < kept && l.from[i0 + i] != kNowhere) *reinterpret_cast<uint4*>(pool + l.to[i0 + i]) = v[i];
        }
    }
}
// Pages of a request, of len positions, that its accepted ones do not reach: the first, how many.
struct Spare {
    uint32_t low, n;
};
__device__ __forceinline__ Spare spare_of(const Move& a, const Rows& r, uint32_t len, uint32_t kept)
{
    if (r.n == 0 || r.n > 32 * a.words || len < r.all) return Spare{0, 0};
    const uint32_t size = 1u << a.shift;
    const uint32_t low = uint32_t((uint64_t(len - r.all + kept) + size - 1) >> a.shift);
    const uint32_t end = min(uint32_t((uint64_t(len) + size - 1) >> a.shift), a.max_pages);
    return Spare{low, end > low ? end - low : 0};
}

// A workgroup to a request and layer; that of one more layer number returns the pages, without table entries that are none.
__global__ __launch_bounds__(256) void k_tree_move(Move a, Layers layers)
{
    const uint32_t tid = threadIdx.x, layer = blockIdx.y;
    if (layer < a.layers) {
        __shared__ MoveSpace l;
        const uint32_t b = blockIdx.x;
        if (b >= a.requests) return;
        const Rows r = rows_of(a.starts, a.tokens, b);
        const uint32_t held = a.held[b], kept = a.counts[b];
        if (r.n == 0 || r.n > 32 * a.words || held < r.all || kept < 2) return;
        move_rows(a, layers, layer, b, held - r.all, kept, l, [&](uint32_t i) { return a.path[r.first + i]; });
        return;
    }
    if (blockIdx.x || !a.free_pages) return;
    __shared__ uint32_t sums[4];
    uint32_t count = *a.free_count;
    for (uint32_t b0 = 0; b0 < a.requests; b0 += 256) {
        const uint32_t b = b0 + tid;
        Spare spare{0, 0};
        if (b < a.requests) spare = spare_of(a, rows_of(a.starts, a.tokens, b), a.held[b], a.counts[b]);
        const uint32_t* pages = a.tables + uint64_t(b) * a.max_pages + spare.low;
        uint32_t back = 0;
        for (uint32_t i = 0; i < spare.n; ++i) back += pages[i] < a.num_pages;
        uint32_t inc = back;  // sums of the requests up to this one
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t v = uint32_t(__shfl_up(int(inc), d));
            if (int(tid & 63u) >= d) inc += v;
        }
        if ((tid & 63u) == 63) sums[tid >> 6] = inc;
        __syncthreads();
        uint32_t at = count + inc - back;
        for (uint32_t w = 0; w < 4; ++w) {
            if (w < (tid >> 6)) at += sums[w];
            count += sums[w];
        }
        for (uint32_t i = 0; i < spare.n; ++i) {
            const uint32_t page = pages[i];
            if (page >= a.num_pages) continue;
            if (at < a.list_pages) a.free_pages[at] = page;
            ++at;
        }
        __syncthreads();
    }
    if (tid == 0) *a.free_count_out = min(count, a.list_pages);
}

// The step's end of one request where lens_out is not lens, in one launch: each layer's workgroup walks for itself, the last one
// writes what the call gives and returns the pages.  28 layers after a tree of 26 nodes: 6.8 us, in two launches 9.8; in a
// graph 3.8 and 5.2.
__global__ __launch_bounds__(256) void k_tree_one(Walk w, Move a, Layers layers)
{
    __shared__ WalkSpace l;
    __shared__ MoveSpace at;
    const uint32_t tid = threadIdx.x, layer = blockIdx.x;
    const bool writes = layer == a.layers;
    const Rows r = rows_of(w.starts, w.tokens, 0);
    const uint32_t len = w.lens[0];
    uint32_t count = writes && a.free_pages ? *a.free_count : 0;
    const uint32_t kept = walk(w, 0, r, len, writes, l);  // a barrier in it: all have read the count
    if (!writes) {
        if (kept > 1 && len >= r.all) move_rows(a, layers, layer, 0, len - r.all, kept, at, [&](uint32_t i) { return l.path[i]; });
        return;
    }
    if (!a.free_pages) return;
    __shared__ uint32_t sums[4];
    const Spare spare = spare_of(a, r, len, kept);
    const uint32_t lane = tid & 63u, wave = tid >> 6;
    for (uint32_t i = 0; i < spare.n; i += 256) {
        const uint32_t page = i + tid < spare.n ? a.tables[spare.low + i + tid] : kNoToken;
        const uint64_t back = __ballot(page < a.num_pages);
        if (lane == 0) sums[wave] = uint32_t(__builtin_popcountll(back));
        __syncthreads();
        uint32_t place = count + uint32_t(__builtin_popcountll(back & ((1ull << lane) - 1u)));
        for (uint32_t w = 0; w < 4; ++w) {
            if (w < wave) place += sums[w];
            count += sums[w];
        }
        if (page < a.num_pages && place < a.list_pages) a.free_pages[place] = page;
        __syncthreads();
    }
    if (tid == 0) *a.free_count_out = min(count, a.list_pages);
}

// ---------------------------------------------------------------------- host
int check_tree(const arc_tree* t)
{
    if (!t || !t->parents) return set_error(ARC_ERR_INVALID_ARGUMENT, "null tree or parents");
    if (t->mask_words == 0 || t->mask_words > ARC_TREE_MAX_WORDS)
        return set_error(ARC_ERR_UNSUPPORTED, "mask_words %u: 1..%u are supported", t->mask_words, uint32_t(ARC_TREE_MAX_WORDS));
    return ARC_OK;
}

// Arrays of a call: what it writes must not share memory with what it reads or else writes; `same`: this array may be
// the input at the same address.
struct Array {
    Rows2d at;
    const void* same;
    Array(const void* p, uint64_t bytes, const void* same_ = nullptr) : at(bytes_at(p, bytes)), same(same_) {}
    explicit Array(const Rows2d& rows) : at(rows), same(nullptr) {}
};
bool share(const Array& a, const Array& b) { return !(a.same && a.same == b.at.p && a.at.p == b.at.p) && overlap(a.at, b.at); }
template <size_t W, size_t R>
bool shared(const Array (&written)[W], const Array (&read)[R])
{
    for (size_t i = 0; i < W; ++i) {
        for (size_t j = i + 1; j < W; ++j)
            if (share(written[i], written[j])) return true;
        for (size_t j = 0; j < R; ++j)
            if (share(written[i], read[j])) return true;
    }
    return false;
}

// The K and V of all layers: pools of one shape, whose pages may lie in turns.
class Pools {
public:
    Pools(const arc_kv_pages* layers, uint32_t num_layers)
        : n_(2 * num_layers), pages_(layers->num_pages), page_(uint64_t(layers->page_size) * layers->kv_heads * layers->head_dim * 2),
          stride_(layers->page_stride * 2), span_((pages_ - 1) * stride_ + page_)
    {
        for (uint32_t i = 0; i < num_layers; ++i) {
            at_[2 * i] = reinterpret_cast<uintptr_t>(layers[i].k);
            at_[2 * i + 1] = reinterpret_cast<uintptr_t>(layers[i].v);
        }
        std::sort(at_, at_ + n_);
        for (uint32_t i = 1; i < n_; ++i) apart_ &= at_[i] - at_[i - 1] >= span_;
    }
    bool twice() const { return std::adjacent_find(at_, at_ + n_) != at_ + n_; }
    // Whether two of them share memory.  Those whose ranges meet are told apart by their places in a stride, in one pass
    // over the sorted places; pairs are only looked at where that leaves a doubt.
    bool overlap() const
    {
        if (apart_) return false;
        uint64_t place[2 * ARC_MAX_LAYERS + 1];
        for (uint32_t i = 0; i < n_; ++i) place[i] = at_[i] % stride_;
        std::sort(place, place + n_);
        place[n_] = place[0] + stride_;
        bool clear = true;
        for (uint32_t i = 0; i < n_; ++i) clear &= place[i + 1] - place[i] >= page_;
        if (clear) return false;
        for (uint32_t i = 0; i < n_; ++i)
            for (uint32_t j = i + 1; j < n_ && at_[j] - at_[i] < span_; ++j)
                if (rows_overlap(pool(i), page_, stride_, pool(j), page_, stride_, pages_)) return true;
        return false;
    }
    // Whether rows share memory with one of them.
    bool hold(const Rows2d& rows) const
    {
        if (!rows.p || !rows.rows) return false;
        const uintptr_t lo = reinterpret_cast<uintptr_t>(rows.p), hi = lo + (rows.rows - 1) * rows.stride + rows.width;
        for (const uintptr_t* p = std::lower_bound(at_, at_ + n_, hi); p != at_; --p) {
            if (p[-1] + span_ <= lo) break;  // as those before it
            if (arc::overlap(rows, Rows2d{reinterpret_cast<const void*>(p[-1]), pages_, page_, stride_})) return true;
        }
        return false;
    }

private:
    const void* pool(uint32_t i) const { return reinterpret_cast<const void*>(at_[i]); }
    uintptr_t at_[2 * ARC_MAX_LAYERS];
    uint32_t n_;
    uint64_t pages_, page_, stride_, span_;  // bytes of a page, from page to page, of all
    bool apart_ = true;                      // their ranges do not meet
};

// Parts of a row of logits, a power of two: enough workgroups to fill the card, and a few KB or more to each.
uint32_t splits_of(uint32_t tokens)
{
    uint32_t s = 1;
    while (s < 64 && uint64_t(tokens) * s < 2048) s *= 2;
    return s;
}

// The most parts that logits of up to `tokens` rows are read in: rows of one number of parts end where 2048 are
// reached with half of it.
size_t most_parts(uint32_t tokens)
{
    size_t most = size_t(tokens) * splits_of(tokens);
    for (uint32_t s = 64; s > 1; s /= 2) {
        const uint32_t n = 4096 / s - 1;
        if (n <= tokens) most = std::max(most, size_t(n) * splits_of(n));
    }
    return most;
}

// Where a commit's workspace holds what: `bytes` of a step of these rows, `most` of any of fewer too.
struct Space {
    size_t held, parts, bytes, most;
};
Space space_of(const arc_paged_batch* b)
{
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    Space s;
    s.held = up(b->tokens * sizeof(uint32_t));
    s.parts = s.held + up(b->requests * sizeof(uint32_t));
    s.bytes = s.parts + up((size_t(b->tokens) * splits_of(b->tokens) + 1) * sizeof(Best));
    s.most = s.parts + up((most_parts(b->tokens) + 1) * sizeof(Best));
    return s;
}

}  // namespace
}  // namespace arc

using namespace arc;

extern "C" {

int arc_tree_plan(const arc_paged_batch* batch, const arc_tree* tree, arc_stream_t stream)
{
    int rc = check_batch_sizes(batch);
    if (!rc) rc = check_tree(tree);
    if (rc) return rc;
    if (!batch->lens || !batch->starts || !batch->positions || !tree->masks)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "null lens, starts, positions or masks");
    if (batch->requests == 0 || batch->tokens == 0) return ARC_OK;
    const uint64_t tokens = batch->tokens * 4ull, requests = batch->requests * 4ull;
    const Array written[] = {{tree->masks, tokens * tree->mask_words}, {batch->positions, tokens}};
    const Array read[] = {{tree->parents, tokens}, {batch->lens, requests}, {batch->starts, requests + 4}};
    if (shared(written, read)) return set_error(ARC_ERR_INVALID_ARGUMENT, "masks and positions share memory with each other or with what is read");
    const TreePlan a{batch->lens, batch->starts, tree->parents, tree->masks, batch->positions, batch->requests, batch->tokens, tree->mask_words};
    hipLaunchKernelGGL(k_tree_plan, dim3(batch->requests), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    return check_hip(hipGetLastError(), "tree plan");
}

size_t arc_tree_commit_workspace_bytes(const arc_paged_batch* batch)
{
    return check_batch_sizes(batch) ? 0 : space_of(batch).most;
}

int arc_tree_commit(const arc_kv_pages* layers, uint32_t num_layers, const arc_paged_batch* batch, const arc_tree* tree, int logits_dtype,
                    const void* logits, uint64_t ldl, uint32_t vocab, const uint32_t* drafts, uint32_t* targets, uint32_t* lens_out,
                    uint32_t* counts, uint32_t* tokens_out, uint32_t* free_pages, uint32_t num_pages, const uint32_t* free_count,
                    uint32_t* free_count_out, void* workspace, arc_stream_t stream)
{
    if (num_layers == 0 || num_layers > ARC_MAX_LAYERS)
        return set_error(ARC_ERR_UNSUPPORTED, "%u layers: 1..%u are supported", num_layers, uint32_t(ARC_MAX_LAYERS));
    if (!layers) return set_error(ARC_ERR_INVALID_ARGUMENT, "null pages");
    for (uint32_t i = 0; i < num_layers; ++i) {
        if (int rc = check_pages(layers + i)) return rc;
        const arc_kv_pages &p = layers[i], &q = layers[0];
        if (p.page_size != q.page_size || p.page_stride != q.page_stride || p.num_pages != q.num_pages || p.kv_heads != q.kv_heads ||
            p.head_dim != q.head_dim || p.dtype != q.dtype)
            return set_error(ARC_ERR_INVALID_ARGUMENT, "layer %u: pages of another shape than layer 0's", i);
    }
    int rc = check_batch_sizes(batch);
    if (!rc) rc = check_tables(batch, layers->page_size);
    if (!rc) rc = check_tree(tree);
    if (rc) return rc;
    if (!drafts || !targets || !lens_out || !counts || !tokens_out || !workspace)
        return set_error(ARC_ERR_INVALID_ARGUMENT, "null argument");
    if (!aligned(workspace, 256)) return set_error(ARC_ERR_INVALID_ARGUMENT, "workspace must be 256-byte aligned");
    if (free_pages && (!free_count || !free_count_out || num_pages == 0))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "a free list needs its counts and num_pages");
    if (logits) {
        const uint32_t size = logits_dtype == ARC_F32 ? 4 : logits_dtype == ARC_F16 || logits_dtype == ARC_BF16 ? 2 : 0;
        if (size == 0) return set_error(ARC_ERR_UNSUPPORTED, "logits are ARC_F32, ARC_F16 or ARC_BF16 (dtype %d)", logits_dtype);
        if (vocab == 0 || vocab > (1u << 24) || ldl < vocab)
            return set_error(ARC_ERR_INVALID_ARGUMENT, "vocab %u, ldl %llu: 1 .. 2^24, ldl at least vocab", vocab, static_cast<unsigned long long>(ldl));
        if (!aligned(logits, size)) return set_error(ARC_ERR_INVALID_ARGUMENT, "logits must be aligned to their type");
        if (batch->tokens > kMaxLogitRows) return set_error(ARC_ERR_UNSUPPORTED, "%u rows of logits: at most 2^20", batch->tokens);
    }
    const Pools pools(layers, num_layers);
    if (pools.twice()) return set_error(ARC_ERR_INVALID_ARGUMENT, "the same pages twice among the layers' k and v");
    if (pools.overlap()) return set_error(ARC_ERR_INVALID_ARGUMENT, "pages of two of the layers' k and v share memory");
    const Space sp = space_of(batch);
    const uint64_t tokens = batch->tokens * 4ull, requests = batch->requests * 4ull;
    const uint32_t logit_bytes = logits_dtype == ARC_F32 ? 4 : 2;
    const Array written[] = {{workspace, sp.bytes}, {tokens_out, tokens}, {counts, requests}, {lens_out, requests, batch->lens},
                             {free_pages, num_pages * 4ull}, {free_pages ? free_count_out : nullptr, 4, free_count},
                             {logits ? targets : nullptr, tokens}};
    const Array read[] = {{logits ? nullptr : targets, tokens}, {drafts, tokens}, {tree->parents, tokens}, {batch->lens, requests},
                          {batch->starts, requests + 4}, {batch->tables, requests * batch->max_pages},
                          {free_pages ? free_count : nullptr, 4},
                          Array(Rows2d{logits, batch->tokens, uint64_t(vocab) * logit_bytes, ldl * logit_bytes})};
    if (shared(written, read)) return set_error(ARC_ERR_INVALID_ARGUMENT, "an array that is written shares memory with another of the call");
    auto in_pools = [&](const Array& a) { return pools.hold(a.at); };
    if (std::any_of(std::begin(written), std::end(written), in_pools) || std::any_of(std::begin(read), std::end(read), in_pools))
        return set_error(ARC_ERR_INVALID_ARGUMENT, "an array of the call shares memory with the pages");
    hipStream_t st = static_cast<hipStream_t>(stream);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    uint32_t *path = reinterpret_cast<uint32_t*>(ws), *held = reinterpret_cast<uint32_t*>(ws + sp.held);
    Best* parts = reinterpret_cast<Best*>(ws + sp.parts);
    uint32_t splits = logits ? splits_of(batch->tokens) : 0;
    while (splits > 1 && vocab / splits < 4096) splits /= 2;
    if (splits && batch->requests && batch->tokens) {
        const Argmax a{logits, batch->starts, parts, ldl, batch->requests, batch->tokens, vocab, splits};
        const dim3 grid(batch->tokens * splits), block(256);
        if (logits_dtype == ARC_F32) hipLaunchKernelGGL(k_tree_argmax<float>, grid, block, 0, st, a);
        else if (logits_dtype == ARC_F16) hipLaunchKernelGGL(k_tree_argmax<_Float16>, grid, block, 0, st, a);
        else hipLaunchKernelGGL(k_tree_argmax<bf16>, grid, block, 0, st, a);
        if (hipError_t e = hipGetLastError()) return check_hip(e, "tree commit");
    }
    const Walk w{batch->lens, batch->starts, tree->parents, drafts, targets, lens_out, counts, tokens_out, path, held, parts,
                 batch->requests, batch->tokens, tree->mask_words, splits};
    const bool one = batch->requests == 1 && lens_out != batch->lens;
    if (batch->requests && !one) hipLaunchKernelGGL(k_tree_walk, dim3(batch->requests), dim3(256), 0, st, w);
    if (hipError_t e = hipGetLastError()) return check_hip(e, "tree commit");
    const uint32_t row_bytes = layers->kv_heads * layers->head_dim * 2;
    const Move m{batch->tables, held, batch->starts, counts, path, free_pages, free_count_out, free_count,
                 layers->page_stride * 2, batch->requests, batch->tokens, tree->mask_words, batch->max_pages, layers->num_pages,
                 num_pages, log2_of(layers->page_size), row_bytes, num_layers};
    Layers l{};
    for (uint32_t i = 0; i < num_layers; ++i) {
        l.k[i] = layers[i].k;
        l.v[i] = layers[i].v;
    }
    if (one) hipLaunchKernelGGL(k_tree_one, dim3(num_layers + 1), dim3(256), 0, st, w, m, l);
    else hipLaunchKernelGGL(k_tree_move, dim3(batch->requests ? batch->requests : 1, num_layers + (free_pages ? 1 : 0)), dim3(256), 0, st, m, l);
    return check_hip(hipGetLastError(), "tree commit");
}

}  // extern "C"
