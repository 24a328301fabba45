// bfft_attention_span.cuh -- what rows see beside the causal mask and the window: first
// tokens that stay visible, and prefixes that groups of sequences share; the token axis
// without what lies between, and the work of a call with groups cut into items.
// Included by bfft_attention.cuh.
#pragma once

namespace bfft {

// The kernels' forms: as the mask and the window say; with visible first tokens, cut by
// the host; with shared prefixes, cut into items on the device.
enum : int { kPlain = 0, kSinks = 1, kGroups = 2 };

struct SpanArgs {
    int sinks;              // first tokens that a window does not hide
    int n_groups;           // sequences groups[g] .. groups[g + 1] share shared[g] tokens
    const int32_t* groups;  // null: one group of all sequences
    const int32_t* shared;
};

// A row tile's piece of the axis.
struct Item {
    int table_row;          // of the block table
    int s0, s1;             // sequences that its rows are of
    int token, n;           // its first row, query tokens
    int part;               // of a token's heads
    int chunk, chunks;
    int from, to;           // tokens that it is about
    int pos, len;           // of a sequence: its first row's place, its tokens
    int prefix, shares;
    int spare[2];
};
static_assert(sizeof(Item) == 64, "four loads");

// One call with groups: row tiles of groups over their prefixes, then row tiles of
// sequences over their own tokens, each cut along the axis.  Item i and kv head h are
// block i * kv_heads + h; its parts are rows [block * rows of a tile, ...) of `parts`.
struct ItemArgs {
    int prefixes, own;      // which of them this launch takes
    int target;             // items a kv head that the axis is cut for
    int least;              // tokens of an item at least
    int unit;               // and a multiple of this
    int64_t most;           // items a kv head at most (the grid)
    const Item* list;       // where there are many units (see kFewUnits): the items, and how many
    const int* count;
    int4* own_of;           // [tokens] where a token's parts are: see ItemPlace
    int4* prefix_of;
};

// Of a token: the first item of its row tile, items along the axis, the row of its first
// head in the tile; parts of a head beyond the tile's rows lie `chunks` items further.
struct ItemPlace {
    int item, chunks, row, flags;
};
enum : int { kPlaceDone = 1, kPlacePrefix = 2 };  // written already; has a prefix's parts too

// What one query token sees: tokens [lo, hi), and those before `sinks`, none before `first`.
struct TokenSpan {
    int lo, hi, sinks;
};
__device__ __forceinline__ TokenSpan token_span(const AttentionArgs& a, const SpanArgs& p, int64_t pos, int64_t len,
                                                int64_t first, int64_t last) {
    const int64_t most = (int64_t)a.seq.max_pages << a.cache.page_log2;
    if (len > most) len = most;
    if (len > last) len = last;
    int64_t hi = a.causal && pos + 1 < len ? pos + 1 : len;
    if (hi < first) hi = first;
    int64_t lo = a.window > 0 ? pos - a.window + 1 : 0;
    if (lo < first) lo = first;
    if (lo > hi) lo = hi;
    int64_t sinks = a.window > 0 && p.sinks < hi ? p.sinks : hi;
    if (a.window <= 0 || sinks < first) sinks = first;
    return {(int)lo, (int)hi, (int)sinks};
}

// The axis that a row tile walks: the visible first tokens [first, first + head), rounded
// up to 16, then the tokens from `main` on; head is 0 where these follow on one another.
struct Axis {
    int first, head, main, total;
    int lo_any, hi_any, sinks_any;  // what some row sees, in places of the axis
    __device__ __forceinline__ int place(int token) const { return token - main + head; }
};
__device__ __forceinline__ Axis make_axis(int first, int lo_min, int hi_max, int sinks_max) {
    Axis x;
    x.first = first;
    x.head = 0;
    const bool none = lo_min >= hi_max;  // of the window's tokens
    const int up = first + ((sinks_max - first + 15) & ~15);
    if (none) {
        x.main = first;
        x.total = sinks_max - first;
        x.lo_any = x.hi_any = 0;
    } else {
        x.main = lo_min & ~15;
        if (sinks_max > first) {
            if (up >= x.main)
                x.main = first;
            else
                x.head = up - first;
        }
        x.total = x.place(hi_max > sinks_max ? hi_max : sinks_max);
        x.lo_any = x.place(lo_min);
        x.hi_any = x.place(hi_max);
    }
    x.sinks_any = sinks_max - first;
    return x;
}

// Tokens of the whole pages among n.
__device__ __forceinline__ int whole_pages(const AttentionArgs& a, int n) {
    n = min(n, a.seq.max_pages << a.cache.page_log2);  // 2^30 at most
    return n > 0 ? n >> a.cache.page_log2 << a.cache.page_log2 : 0;
}
// Sequences of group g.
__device__ __forceinline__ void group_sequences(const AttentionArgs& a, const SpanArgs& p, int g, int& s0, int& s1) {
    s0 = 0;
    s1 = a.seq.seqs;
    if (p.groups) {
        s0 = min(max(p.groups[g], 0), s1);
        s1 = min(max(p.groups[g + 1], s0), s1);
    }
}
// The group of sequence s, or -1: the largest g with groups[g] <= s, if s lies before its end.
__device__ __forceinline__ int group_of(const AttentionArgs& a, const SpanArgs& p, int s) {
    if (!p.groups) return 0;
    int lo = 0, n = p.n_groups;
    while (n > 1) {
        const int half = n >> 1;
        if (p.groups[lo + half] <= s) {
            lo += half;
            n -= half;
        } else {
            n = half;
        }
    }
    return p.groups[lo] <= s && s < p.groups[lo + 1] ? lo : -1;
}
// The rows [t0, t0 + n) that lie from starts' entry `from` to entry `to`.
__device__ __forceinline__ int rows_between(const AttentionArgs& a, int from, int to, int& t0) {
    t0 = from;
    if (to > a.seq.tokens) to = (int)a.seq.tokens;
    if (t0 < 0) t0 = to;
    return to > t0 ? to - t0 : 0;
}

// A group's or a sequence's row tiles (times parts), and the tokens that each walks.
struct Unit {
    int s0, s1, t0, rows, len;
    int shared;     // tokens that it is about (a group), or that come before them
    int tiles, length;
};
__device__ __forceinline__ Unit unit_of(const AttentionArgs& a, const SpanArgs& p, const ItemArgs& x, int u, int tile,
                                        int parts) {
    Unit v;
    const int groups = x.prefixes ? p.n_groups : 0;
    const bool prefix = u < groups;
    v.s0 = u - groups;
    v.s1 = v.s0 + 1;
    if (prefix) group_sequences(a, p, u, v.s0, v.s1);
    // the loads of what follows side by side: each waits for memory once
    const int t0 = a.seq.starts[v.s0], t1 = a.seq.starts[v.s1], len = a.seq.lens[v.s0 < a.seq.seqs ? v.s0 : 0];
    const int g = prefix ? u : group_of(a, p, v.s0);
    const int shared = g >= 0 ? p.shared[g] : 0;
    v.rows = rows_between(a, t0, t1, v.t0);
    v.shared = whole_pages(a, shared);
    v.len = prefix ? 0 : len;
    v.tiles = (int)((unsigned)(v.rows + tile - 1) / (unsigned)tile) * parts;
    // tokens up to the end, from the first that the first row (causal: the last row tile's) sees
    const int most = a.seq.max_pages << a.cache.page_log2;  // 2^30 at most
    const int end = prefix ? v.shared : min(v.len, most), first = prefix ? 0 : v.shared;
    int lo = first, sinks = 0;
    if (a.window > 0) {
        const int window = min(a.window, 1 << 30);
        lo = max(first, prefix ? end - window : v.len - (a.causal ? min(v.rows, tile) : v.rows) - window + 1);
        sinks = max(min(p.sinks, lo) - first, 0);
    }
    v.length = max(end - lo + sinks, 0);
    if (prefix && !v.length) v.tiles = 0;
    return v;
}

// Tokens of an item: those that all row tiles walk, `total`, shared out over x.target items.
// The grid has room for target + 2 items more than there are row tiles: a share goes up to
// the widest table (2^30 tokens), and what the sum rounds off is far under two shares.
__host__ __device__ __forceinline__ unsigned item_tokens(const ItemArgs& x, float total) {
    const int share = (int)fminf(total / (float)x.target, 1073741824.f) + 1;
    return max((unsigned)(share + x.unit - 1) / (unsigned)x.unit * x.unit, (unsigned)x.least);
}
__host__ __device__ __forceinline__ int pieces_of(const Unit& v, unsigned chunk) {
    return (unsigned)v.length > chunk ? (int)(((unsigned)v.length + chunk - 1) / chunk) : 1;
}
// Item `rest` of unit u.
__device__ __forceinline__ void fill_item(Item& f, const Unit& v, bool prefix, int rest, int pieces, int tile, int parts) {
    const unsigned at = (unsigned)rest / (unsigned)pieces, t = at / (unsigned)parts;
    f.prefix = prefix;
    f.table_row = f.s0 = v.s0;
    f.s1 = v.s1;
    f.chunks = pieces;
    f.chunk = rest - (int)at * pieces;
    f.part = (int)at - (int)t * parts;
    f.token = v.t0 + (int)t * tile;
    f.n = min(v.rows - (int)t * tile, tile);
    f.from = prefix ? 0 : v.shared;
    f.to = prefix ? v.shared : 0x7fffffff;
    f.shares = v.shared > 0;
    f.pos = v.len - v.rows + (int)t * tile;
    f.len = v.len;
}

// Units that a call's warps look at by themselves; more have their items listed first.  The
// list is a launch of its own (32 sequences over 2048 + 200 tokens 42 us with it, 32
// without), or free where a block of the row tiles makes it.
constexpr int kFewUnits = 128, kFewBesideTiles = 32;
__host__ __device__ inline int unit_count(const SpanArgs& p, const ItemArgs& x, int seqs) {
    return (x.prefixes ? p.n_groups : 0) + (x.own ? seqs : 0);
}

// Finds item i, each warp for itself.  With few units every warp makes the same sums over
// the sequences' tables, so that no launch has to come before (a block does this once, from
// a cold instruction cache: short code and few waits for memory are what counts).
__device__ __forceinline__ bool find_item(const AttentionArgs& a, const SpanArgs& p, const ItemArgs& x, int i, int tile,
                                          int parts, Item& it) {
    const int lane = threadIdx.x & 31;
    if (x.list) {
        const int count = *x.count;
        const int4* from = reinterpret_cast<const int4*>(x.list + i);
        int4* to = reinterpret_cast<int4*>(&it);
#pragma unroll
        for (int k = 0; k < 4; ++k) to[k] = from[k];
        return i < count;
    }
    const int groups = x.prefixes ? p.n_groups : 0, units = unit_count(p, x, a.seq.seqs);
    Unit v{};
    float total = 0.f;
#pragma unroll 1
    for (int u = lane; u < units; u += 32) {
        v = unit_of(a, p, x, u, tile, parts);
        total += (float)v.tiles * (float)v.length;
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
    const unsigned chunk = item_tokens(x, total);
    int before = 0;  // items of the units before these 32
#pragma unroll 1
    for (int u0 = 0; u0 < units; u0 += 32) {
        const int u = u0 + lane;
        if (units > 32) v = u < units ? unit_of(a, p, x, u, tile, parts) : Unit{};
        const int pieces = pieces_of(v, chunk);
        const int mine = v.tiles * pieces;
        int upto = mine;
#pragma unroll
        for (int w = 1; w < 32; w <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, w);
            if (lane >= w) upto += y;
        }
        const int rest = i - before - (upto - mine);
        const unsigned who = __ballot_sync(0xffffffffu, rest >= 0 && rest < mine);
        if (who) {
            Item f{};
            fill_item(f, v, u < groups, rest, pieces, tile, parts);
            const int* fields = reinterpret_cast<const int*>(&f);
            int* out = reinterpret_cast<int*>(&it);
#pragma unroll
            for (int k = 0; k < (int)(sizeof(Item) / 4); ++k) out[k] = __shfl_sync(0xffffffffu, fields[k], __ffs(who) - 1);
            return true;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

// Lists the items of more units, by one block: long pieces before short ones (in sixteen
// classes), as blocks start in the order of their items.  The order within a class is that
// of the atomics; a token's parts are joined in the order of its axis wherever they lie.
constexpr int kListThreads = 512;
struct ListArgs {
    ItemArgs items;
    int tile, parts;  // query tokens of a row tile, tiles of a token
    Item* list;       // null: nothing to list
    int* count;
};
__device__ __forceinline__ void list_items(const AttentionArgs& a, const SpanArgs& p, const ListArgs& l) {
    constexpr int WARPS = kListThreads / 32, CLASSES = 16;
    __shared__ float sums[WARPS];
    __shared__ int first[CLASSES];
    const ItemArgs& x = l.items;
    const int tile = l.tile, parts = l.parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int groups = x.prefixes ? p.n_groups : 0, units = unit_count(p, x, a.seq.seqs);
    if (tid < CLASSES) first[tid] = 0;
    float total = 0.f;
    unsigned chunk = 1;
    // three looks at every unit: the sum, the classes' counts, the items
#pragma unroll 1
    for (int look = 0; look < 3; ++look) {
#pragma unroll 1
        for (int u = tid; u < units; u += kListThreads) {
            const Unit v = unit_of(a, p, x, u, tile, parts);
            if (look == 0) {
                total += (float)v.tiles * (float)v.length;
                continue;
            }
            const int pieces = pieces_of(v, chunk), mine = v.tiles * pieces;
            const unsigned each = ((unsigned)v.length + pieces - 1) / pieces;
            const int of = CLASSES - 1 - (int)min(each * (float)CLASSES / (float)chunk, CLASSES - 1.f);
            const int at = mine ? atomicAdd(&first[of], mine) : 0;
            if (look == 1) continue;
            // a warp writes the items of its lanes' units, the many of a group side by side
            const unsigned active = __activemask();
            for (unsigned left = active; left; left &= left - 1) {
                const int from = __ffs(left) - 1;
                Unit w;
                const int* fields = reinterpret_cast<const int*>(&v);
                int* out = reinterpret_cast<int*>(&w);
#pragma unroll
                for (int k = 0; k < (int)(sizeof(Unit) / 4); ++k) out[k] = __shfl_sync(active, fields[k], from);
                const int n = __shfl_sync(active, mine, from), to = __shfl_sync(active, at, from),
                          each_of = __shfl_sync(active, pieces, from), prefix = __shfl_sync(active, (int)(u < groups), from);
                for (int k = __popc(active & ((1u << lane) - 1)); k < n && to + k < x.most; k += __popc(active))
                    fill_item(l.list[to + k], w, prefix, k, each_of, tile, parts);
            }
        }
        if (look == 0) {
#pragma unroll
            for (int w = 16; w; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
            if (lane == 0) sums[warp] = total;
            __syncthreads();
            total = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) total += sums[w];
            chunk = item_tokens(x, total);
        } else if (look == 1) {
            __syncthreads();
            if (tid == 0) {
                int sum = 0;
                for (int c = 0; c < CLASSES; ++c) {
                    const int n = first[c];
                    first[c] = sum;
                    sum += n;
                }
                *l.count = sum < x.most ? sum : (int)x.most;
            }
            __syncthreads();
        }
    }
}

// What the item's rows see of its tokens, a query token each, in shared memory, after a
// barrier behind which `spans` holds empty ones.  A group's rows are found from its sequences, a thread each:
// each row's own search of its sequence took 3900 clocks.
template <int THREADS>
__device__ __forceinline__ void item_spans(const AttentionArgs& a, const SpanArgs& p, const Item& it, TokenSpan* spans) {
    if (!it.prefix) {
        for (int t = threadIdx.x; t < it.n; t += THREADS)
            spans[t] = token_span(a, p, (int64_t)it.pos + t, it.len, it.from, it.to);
    } else {
        for (int s = it.s0 + (int)threadIdx.x; s < it.s1; s += THREADS) {
            int t0;
            const int from = a.seq.starts[s], to = a.seq.starts[s + 1], len = a.seq.lens[s];
            const int n = rows_between(a, from, to, t0);
            for (int t = max(t0, it.token); t < min(t0 + n, it.token + it.n); ++t)
                spans[t - it.token] = token_span(a, p, (int64_t)len - n + (t - t0), len, it.from, it.to);
        }
    }
    __syncthreads();
}

}  // namespace bfft
