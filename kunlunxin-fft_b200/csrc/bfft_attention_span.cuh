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

// One call with groups: row tiles of groups over their prefixes, then row tiles of
// sequences over their own tokens, each cut along the axis.  Item i and kv head h are
// block i * kv_heads + h; its parts are rows [block * rows of a tile, ...) of `parts`.
struct ItemArgs {
    int prefixes, own;      // which of them this launch takes
    int target;             // items a kv head that the axis is cut for
    int least;              // tokens of an item at least
    int unit;               // and a multiple of this
    int64_t most;           // items a kv head at most (the grid)
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

// Whole pages of the tokens that group g shares.
__device__ __forceinline__ int shared_tokens(const AttentionArgs& a, const SpanArgs& p, int g) {
    const int64_t most = (int64_t)a.seq.max_pages << a.cache.page_log2;
    int64_t n = p.shared[g];
    if (n > most) n = most;
    if (n > 0x7fffffff) n = 0x7fffffff;
    return n > 0 ? (int)(n >> a.cache.page_log2 << a.cache.page_log2) : 0;
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
// What sequence s shares: the largest g with groups[g] <= s.
__device__ __forceinline__ int sequence_shared(const AttentionArgs& a, const SpanArgs& p, int s) {
    if (!p.groups) return shared_tokens(a, p, 0);
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
    return p.groups[lo] <= s && s < p.groups[lo + 1] ? shared_tokens(a, p, lo) : 0;
}
// Rows of sequences [s0, s1).
__device__ __forceinline__ void rows_of(const AttentionArgs& a, int s0, int s1, int64_t& t0, int64_t& t1) {
    t0 = a.seq.starts[s0];
    t1 = a.seq.starts[s1];
    if (t1 > a.seq.tokens) t1 = a.seq.tokens;
    if (t0 < 0 || t1 < t0) t1 = t0 = 0;
}

// A row tile's piece of the axis.
struct Item {
    int table_row;          // of the block table
    int s0, s1;             // sequences that its rows are of
    int64_t token;          // its first row
    int n;                  // query tokens
    int part;               // of a token's heads
    int chunk, chunks;
    int from, to;           // tokens that it is about
    bool prefix, shares;
};

struct ItemScratch {
    long long sum[32];
    int chunk, found, rest, chunks;
};

// Row tiles (times parts) of unit u, groups before sequences, and tokens along the axis.
__device__ __forceinline__ void unit_shape(const AttentionArgs& a, const SpanArgs& p, const ItemArgs& x, int u, int tile,
                                           int parts, int64_t& tiles, int64_t& length) {
    const int groups = x.prefixes ? p.n_groups : 0;
    int64_t t0, t1;
    if (u < groups) {
        int s0, s1;
        group_sequences(a, p, u, s0, s1);
        rows_of(a, s0, s1, t0, t1);
        length = shared_tokens(a, p, u);
        if (a.window > 0 && length > (int64_t)a.window + p.sinks) length = (int64_t)a.window + p.sinks;
        tiles = length ? (t1 - t0 + tile - 1) / tile * parts : 0;
        return;
    }
    const int s = u - groups;
    rows_of(a, s, s + 1, t0, t1);
    const int64_t n = t1 - t0, len = a.seq.lens[s];
    const int first = sequence_shared(a, p, s);
    // the longest of the first and the last row tile
    length = 0;
    for (int k = 0; k < 2; ++k) {
        const int64_t at = k ? (n > tile ? n - tile : 0) : 0, end = k ? n : (n < tile ? n : tile);
        const TokenSpan lo = token_span(a, p, len - n + at, len, first, 0x7fffffff);
        const TokenSpan hi = token_span(a, p, len - n + end - 1, len, first, 0x7fffffff);
        const int64_t m = (int64_t)(hi.hi - lo.lo) + (hi.sinks < lo.lo ? hi.sinks - first : 0);
        if (m > length) length = m;
    }
    tiles = (n + tile - 1) / tile * parts;
}

// Tokens of a piece for items of x.target: what the rows' tokens come to, shared out.
__device__ __forceinline__ int64_t item_chunk(const ItemArgs& x, long long total) {
    int64_t c = (total + x.target - 1) / x.target;
    c = (c + x.unit - 1) / x.unit * x.unit;
    return c > x.least ? c : x.least;
}

// Finds item i by itself, block-wide: every block makes the same sums over the sequences'
// tables, so the items need no list in memory and no launch that makes one.
template <int THREADS>
__device__ __forceinline__ bool find_item(const AttentionArgs& a, const SpanArgs& p, const ItemArgs& x, int64_t i, int tile,
                                          int parts, ItemScratch& sh, Item& it) {
    constexpr int WARPS = THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int groups = x.prefixes ? p.n_groups : 0, units = groups + (x.own ? a.seq.seqs : 0);
    int64_t tiles = 0, length = 0;
    long long total = 0;
    for (int u = tid; u < units; u += THREADS) {
        unit_shape(a, p, x, u, tile, parts, tiles, length);
        total += tiles * length;
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
    if (lane == 0) sh.sum[warp] = total;
    if (tid == 0) sh.found = -1;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += sh.sum[w];
    const int64_t chunk = item_chunk(x, total);
    long long before = 0;  // items of the units before this round's
    for (int u0 = 0; u0 < units; u0 += THREADS) {
        const int u = u0 + tid;
        if (units > THREADS && u < units) unit_shape(a, p, x, u, tile, parts, tiles, length);
        const long long pieces = u < units ? (length > chunk ? (length + chunk - 1) / chunk : 1) : 0;
        const long long mine = u < units ? tiles * pieces : 0;
        long long upto = mine;
#pragma unroll
        for (int w = 1; w < 32; w <<= 1) {
            const long long v = __shfl_up_sync(0xffffffffu, upto, w);
            if (lane >= w) upto += v;
        }
        __syncthreads();
        if (lane == 31) sh.sum[warp] = upto;
        __syncthreads();
        long long all = 0, under = before;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) under += sh.sum[w];
            all += sh.sum[w];
        }
        const long long from = under + upto - mine;
        if (i >= from && i < from + mine) {
            sh.found = u;
            sh.rest = (int)(i - from);
            sh.chunks = (int)pieces;
        }
        before += all;
        if (i < before) break;
    }
    __syncthreads();
    const int u = sh.found;
    if (u < 0) return false;
    it.prefix = u < groups;
    if (it.prefix) {
        group_sequences(a, p, u, it.s0, it.s1);
        it.from = 0;
        it.to = shared_tokens(a, p, u);
        it.shares = true;
    } else {
        it.s0 = u - groups;
        it.s1 = it.s0 + 1;
        it.from = sequence_shared(a, p, it.s0);
        it.to = 0x7fffffff;
        it.shares = it.from > 0;
    }
    it.table_row = it.s0;
    it.chunks = sh.chunks;
    it.chunk = sh.rest % it.chunks;
    const int at = sh.rest / it.chunks;
    it.part = at % parts;
    int64_t t0, t1;
    rows_of(a, it.s0, it.s1, t0, t1);
    it.token = t0 + (int64_t)(at / parts) * tile;
    it.n = (int)(t1 - it.token < tile ? t1 - it.token : tile);
    return true;
}

// What row `token` sees of the item's tokens.
__device__ __forceinline__ TokenSpan item_span(const AttentionArgs& a, const SpanArgs& p, const Item& it, int64_t token) {
    int lo = it.s0, n = it.s1 - it.s0;
    while (n > 1) {  // the largest s with starts[s] <= token
        const int half = n >> 1;
        if (a.seq.starts[lo + half] <= token) {
            lo += half;
            n -= half;
        } else {
            n = half;
        }
    }
    int64_t t0, t1;
    rows_of(a, lo, lo + 1, t0, t1);
    return token_span(a, p, (int64_t)a.seq.lens[lo] - (t1 - t0) + (token - t0), a.seq.lens[lo], it.from, it.to);
}

}  // namespace bfft
