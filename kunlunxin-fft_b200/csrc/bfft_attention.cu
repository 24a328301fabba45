// bfft_attention.cu -- attention of ragged query rows over a paged 8-bit cache: entry
// points and plans, and the kernels' plain form (see bfft_attention.cuh).
#include "bfft_attention.cuh"

using namespace bfft;

namespace {

bfft_status check(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs, const bfft_attention_desc* d) {
    if (!cache || !seqs || !d || !d->q || !d->out) return fail(BFFT_ERR_VALUE, "null pointer");
    bfft_status st = check_cache(cache);
    if (st == BFFT_OK) st = check_sequences(seqs);
    if (st != BFFT_OK) return st;
    if (d->type != BFFT_F16 && d->type != BFFT_BF16)
        return fail(BFFT_ERR_UNSUPPORTED, "queries must be float16 or bfloat16, got type %lld", (long long)d->type);
    if (d->q_heads < 1 || d->q_heads % cache->kv_heads || d->q_heads > 0xffffff)
        return fail(BFFT_ERR_SHAPE, "%lld query heads are no multiple of %lld kv heads", (long long)d->q_heads,
                    (long long)cache->kv_heads);
    if (d->window < 0 || d->window > 0x7fffffffLL) return fail(BFFT_ERR_VALUE, "bad window %lld", (long long)d->window);
    if (!std::isfinite(d->softmax_scale)) return fail(BFFT_ERR_VALUE, "softmax_scale must be finite");
    if (!aligned(d->q, 2) || !aligned(d->out, 2) || !aligned(d->lse, 4)) return fail(BFFT_ERR_VALUE, "misaligned pointer");
    return BFFT_OK;
}

using EncodeTiledFn = PFN_cuTensorMapEncodeTiled_v12000;

EncodeTiledFn encoder() {
    static EncodeTiledFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}

}  // namespace

namespace bfft {

// The codes as [pages][kv_heads * page * dim / 128][128 bytes], boxes of 16 tokens,
// 128-byte swizzle (heads of 64, 128 or 256 elements: whole lines).
bool encode_codes(CUtensorMap* m, const void* codes, const bfft_cache_desc* c) {
    EncodeTiledFn enc = encoder();
    if (!enc) return false;
    const cuuint64_t lines = (cuuint64_t)(c->kv_heads * c->page * c->dim / 128);
    cuuint64_t dims[3] = {128, lines, (cuuint64_t)c->pages};
    cuuint64_t strides[2] = {128, 128 * lines};
    cuuint32_t box[3] = {128, (cuuint32_t)(c->dim / 8), 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(codes), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool encode_queries(CUtensorMap* m, const AttentionArgs& a, bool half, int tile_tokens) {
    EncodeTiledFn enc = encoder();
    const int64_t heads = a.q_heads, dim = a.cache.dim;
    // (the stride of a dimension of one is not used, and a map takes no zero)
    const int64_t head = heads > 1 ? a.qh : dim, token = a.seq.tokens > 1 ? a.qt : heads * dim;
    if (!enc || !a.q_packs || head <= 0 || token <= 0 || token >= (int64_t)1 << 38 || head >= (int64_t)1 << 38) return false;
    cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)a.seq.tokens};
    cuuint64_t strides[2] = {(cuuint64_t)head * 2, (cuuint64_t)token * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)tile_tokens};
    cuuint32_t estr[3] = {1, 1, 1};
    return enc(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(a.q), dims,
               strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace bfft

namespace {

int sm_count(int64_t device) {
    static std::atomic<int> counts[64];
    if (device < 0 || device >= 64) return 148;
    const int dev = (int)device;
    int n = counts[dev].load(std::memory_order_relaxed);
    if (!n) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
            cudaGetLastError();
            n = 148;
        }
        counts[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

// Tokens that a row tile of `tile` query tokens sees at most, `sinks` first ones among them.
int64_t seen_cover(const bfft_cache_desc* c, const bfft_sequence_desc* q, const bfft_attention_desc* d, int tile,
                   int align, int64_t sinks) {
    int64_t cover = q->max_pages * c->page;
    if (d->causal && d->window > 0) {
        const int64_t w = d->window + tile - 1 + align - 1 + (sinks + 15) / 16 * 16;
        if (w < cover) cover = w;
    }
    return cover;
}

SplitPlan plan_split(const bfft_cache_desc* c, const bfft_sequence_desc* q, const bfft_attention_desc* d, int sms,
                     int64_t sinks) {
    SplitPlan p;
    const int64_t group = d->q_heads / c->kv_heads;
    const int64_t each = q->tokens / q->seqs + (q->tokens % q->seqs != 0);  // rows of a sequence, about
    p.nt = each * group > 8 && c->dim <= 128 ? 2 : 1;
    const int64_t rows = 8 * p.nt;
    p.tile_tokens = group <= rows ? (int)(rows / group) : 1;
    p.token_tiles = group <= rows ? 1 : (int)((group + rows - 1) / rows);
    const int64_t runs = q->tokens / p.tile_tokens + q->seqs;
    p.by_token = q->tokens <= runs;
    p.slots = p.by_token ? q->tokens : runs;
    const int64_t cover = seen_cover(c, q, d, p.tile_tokens, 16, sinks);
    const int64_t tiles = (q->tokens + p.tile_tokens - 1) / p.tile_tokens;
    const int64_t units = tiles * p.token_tiles * c->kv_heads, resident = 3 * (int64_t)sms;
    // Where rows are many, chunks of 2048 tokens (512..4096 measure alike for 64 ragged
    // sequences).  Where they are few the table's width is shared out over a number of
    // CTAs that is counted as if three were resident on an SM (two are with 16 rows a
    // tile of heads over 64, one with heads over 128) and as if row tiles were full (those of sequences of
    // few rows are not: a tile's rows are one sequence's): "waves" times that many.  One
    // sequence of 131001 tokens, whose tiles are full: 71.6 us with 1, 75.8 with 2, 84.0
    // with 3, so 1, as a further wave's start costs more than it hides; 16 of 2000..8000
    // tokens, whose 4-row tiles are half full: 63.5, 59.4 and 69.6, so 2 for many
    // sequences.  The table's width is all that the host knows of the lengths: with a
    // table of 131072 tokens one row over 700 takes 18.4 us (12.3 with a table of 700,
    // timed with a cold L2), 8 over 4000 61.4 (32.8).
    const int64_t waves = q->seqs > 8 ? 2 : 1;
    int64_t chunks = units >= 2 * resident ? (cover + 2047) / 2048 : waves * resident / units;
    if (chunks < 1) chunks = 1;
    int64_t chunk = (cover + chunks - 1) / chunks;
    chunk = (chunk + 31) / 32 * 32;
    if (chunk < 256) chunk = 256;
    if (chunk > 4096) chunk = 4096;
    // Few rows over a short axis: eight chunks at most, one cluster that joins them
    // itself (8 row tiles over 704 tokens 10.1 us a call, by two launches 14.7; over 2000
    // tokens 12.3 by either, over 4000 15.4 and 12.7; 64 row tiles 28.7 and 22.6: a
    // cluster's CTAs keep their places until the last is done)
    const bool brief = units <= 32 && cover <= 2048;
    if (brief) {
        chunk = (cover + 7) / 8;
        chunk = (chunk + 31) / 32 * 32;
        if (chunk < 128) chunk = 128;
    }
    // The parts of many rows over a wide table (the plan knows the table's width, not the
    // lengths) are kept to 256 MB by longer chunks, as far as shared memory holds their
    // pages' scales (4.4 GB without: 512 sequences of 4 rows of 64 heads, 131072 tokens wide)
    const int64_t part = q->tokens * d->q_heads * (c->dim + 2) * 4, budget = (int64_t)256 << 20;
    // entries of a chunk beside its whole pages: its two ends; with first tokens the ends of
    // both of its pieces, and one where it is no whole pages (see open_segment)
    const int64_t ends = sinks ? 5 : 2;
    if (!brief && (cover + chunk - 1) / chunk * part > budget) {
        const int64_t n = part < budget ? budget / part : 1;
        const int64_t room = (kSplitSmemMost - split_smem((int)c->dim, 8 * p.nt, 0)) / (int64_t)(sizeof(BlockScale) + 4);
        int64_t most = (room - ends) * c->page;
        if (most > 1 << 20) most = 1 << 20;
        chunk = ((cover + n - 1) / n + 31) / 32 * 32;
        if (chunk > most) chunk = most / 32 * 32;
    }
    p.entries = (int)(chunk / c->page + ends);
    p.chunk = (int)chunk;
    const int64_t n = (cover + chunk - 1) / chunk;
    p.chunks = (int)n;
    p.cluster = brief && n > 1;
    p.ctas = p.slots * p.token_tiles * c->kv_heads * n;
    p.bytes = n > 1 && !p.cluster ? (size_t)(q->tokens * d->q_heads * n) * (size_t)(c->dim + 2) * 4 : 0;
    return p;
}

// Whether a call is one for the tensor-core tiles: with 48 rows or more to a kv
// head (16 rows of 32 heads over 16384 tokens: 31 us, split kernel 49; 8 rows: 33
// by either) and enough work to pay for a CTA's start and its 128-row halves, some
// 3 million (query head, token) pairs of 128 dimensions: 40 rows of 32 heads over
// 900 tokens 21 us by the split kernel and 29 by this; 128 rows, which the rule gives to
// this, 21 and 33 since the split kernel takes a tile's halves side by side.  The rows
// are the mean of the call's sequences, so one kernel takes a prompt and single tokens
// together: a prompt of 4096 rows with 255 single tokens of 4096, 32 heads, 1124 us
// (apart 205 and 337), of 512 rows over 512 520 (21 and 337).  Heads over 128 (S and O of two
// halves are more than tensor memory) and groups over 128 stay with the split kernel:
// 2 x 2048 rows of 16 heads of 256 over 8192 and 16384 tokens 8.6 ms, of 128 0.43.
bool use_tiles(const bfft_cache_desc* c, const bfft_sequence_desc* q, const bfft_attention_desc* d, int64_t sinks) {
    const int64_t group = d->q_heads / c->kv_heads, each = q->tokens / q->seqs;
    if (c->dim > 128 || group > 128 || each * group < 48) return false;
    const double pairs = (double)q->tokens * (double)d->q_heads * (double)seen_cover(c, q, d, 1, 1, sinks);
    return pairs * (double)c->dim >= 3.0e6 * 128;
}

TilePlan plan_tiles(const bfft_cache_desc* c, const bfft_sequence_desc* q, const bfft_attention_desc* d, int sms,
                    int64_t sinks) {
    TilePlan p;
    const int64_t group = d->q_heads / c->kv_heads;
    p.tile_tokens = (int)(256 / group);
    const int64_t runs = q->tokens / p.tile_tokens + q->seqs;
    p.by_token = q->tokens <= runs;
    p.slots = p.by_token ? q->tokens : runs;
    const int64_t cover = seen_cover(c, q, d, p.tile_tokens, sinks ? 16 : 128, sinks);
    const int64_t units = (q->tokens + p.tile_tokens - 1) / p.tile_tokens * c->kv_heads;
    int64_t chunks = units >= sms ? 1 : sms / units;
    int64_t chunk = (cover + chunks - 1) / chunks;
    if (chunk < 512) chunk = 512;
    chunk = (chunk + 127) / 128 * 128;
    if (chunk > 0x7fffff80LL) chunk = 0x7fffff80LL;
    p.chunk = (int)chunk;
    p.chunks = (int)((cover + chunk - 1) / chunk);
    p.ctas = p.slots * c->kv_heads * p.chunks;
    p.bytes = p.chunks > 1 ? (size_t)(q->tokens * d->q_heads * p.chunks) * (size_t)(c->dim + 2) * 4 : 0;
    return p;
}

// A call with groups: one launch for the prefixes and the sequences' own tokens where both
// go to one kernel, else two.
struct GroupLaunch {
    bool prefixes, own, tiles;
    SplitPlan split;      // nt, tile_tokens, token_tiles, entries, ctas
    TilePlan row_tiles;   // tile_tokens, ctas
    ItemArgs items;
    bool list;            // the items are listed first
    size_t list_at, parts_at;  // of the workspace
    int tile_tokens() const { return tiles ? row_tiles.tile_tokens : split.tile_tokens; }
    int token_tiles() const { return tiles ? 1 : split.token_tiles; }
    int rows() const { return tiles ? 256 : 8 * split.nt; }
    int64_t ctas() const { return tiles ? row_tiles.ctas : split.ctas; }
};
struct GroupPlan {
    GroupLaunch launch[2];
    int launches;
    size_t bytes;  // of the workspace: places of the tokens' parts, then per launch its list and parts
};

GroupPlan plan_groups(const bfft_cache_desc* c, const bfft_sequence_desc* q, const bfft_attention_desc* d,
                      const bfft_span_desc* w, int sms) {
    const int64_t group = d->q_heads / c->kv_heads, kv = c->kv_heads;
    const int64_t each = q->tokens / q->seqs + (q->tokens % q->seqs != 0), shared = q->tokens / w->n_groups;
    const bool own_tiles = use_tiles(c, q, d, w->sinks);
    // as use_tiles, for a group's rows
    const bool prefix_tiles =
        own_tiles || (c->dim <= 128 && group <= 128 && shared * group >= 48 &&
                      (double)q->tokens * (double)d->q_heads * (double)seen_cover(c, q, d, 1, 1, w->sinks) * (double)c->dim >=
                          3.0e6 * 128);
    // The few-row kernel's row tiles have 16 rows where a group's rows (a sequence's, where the
    // prefixes go to the row tiles) fill more than 8.  One launch takes prefixes and own tokens
    // then: two, with tiles of 8 rows for the sequences, are slower (8 sequences over 2048 + 200
    // tokens 16.4 us by one, 24.9 by two; 64 in 8 groups over 4096 + 300 82 and 92).
    auto tiles_of = [&](int64_t rows) { return rows * group > 8 && c->dim <= 128 ? 2 : 1; };
    const int prefix_nt = prefix_tiles ? 0 : tiles_of(shared);
    const int own_nt = own_tiles ? 0 : prefix_tiles ? tiles_of(each) : prefix_nt;
    GroupPlan p{};
    p.launches = prefix_nt == own_nt ? 1 : 2;
    size_t at = ((size_t)q->tokens * 2 * sizeof(int4) + 63) / 64 * 64;
    for (int k = 0; k < p.launches; ++k) {
        GroupLaunch& l = p.launch[k];
        l.prefixes = k == 0;
        l.own = k == p.launches - 1;
        const int nt = l.own ? own_nt : prefix_nt;
        l.tiles = nt == 0;
        if (l.tiles) {
            l.row_tiles.tile_tokens = (int)(256 / group);
        } else {
            l.split.nt = nt;
            const int64_t rows = 8 * nt;
            l.split.tile_tokens = group <= rows ? (int)(rows / group) : 1;
            l.split.token_tiles = group <= rows ? 1 : (int)((group + rows - 1) / rows);
            l.split.entries = 384;
        }
        // Items: of the row tiles one wave of CTAs' worth (64 sequences over a prefix of 16384 77
        // us, in two waves 98), of the few-row kernel two, one where there are few sequences, as
        // in plan_split (200 sequences of 16..2048 own tokens 445 us, in four waves 466).  A
        // piece costs a CTA's start, so none is short where there are row tiles for every
        // CTA's place (the 64 with 16..1024 tokens of their own: pieces of 256 on 77 us, of 512
        // 74, of 1024 75).  An SM holds three CTAs of 8-row tiles, two of 16-row ones (of 64-wide
        // heads three, counted as two); heads over 128 are counted as two too, though their rings leave room for one.  Counted as
        // one: 64 sequences over 8192 + 200 tokens, 8 kv heads of 256, 260 us for 277, 8 over
        // 32768 + 200 189 for 155, 32 of 2 kv heads over 2048 + 500 46 for 56.
        const int64_t units = ((l.prefixes ? q->tokens / l.tile_tokens() + w->n_groups : 0) +
                               (l.own ? q->tokens / l.tile_tokens() + q->seqs : 0)) * l.token_tiles();
        const int64_t places = (int64_t)sms * (l.tiles ? 1 : nt == 1 && c->dim <= 128 ? 3 : 2);
        const int64_t wanted = places * (!l.tiles && l.own && q->seqs > 8 ? 2 : 1) / kv;
        l.items.prefixes = l.prefixes;
        l.items.own = l.own;
        l.items.target = (int)(wanted > 0 ? wanted : 1);
        l.items.least = l.tiles || units * kv >= places ? 512 : 256;
        l.items.unit = l.tiles ? 128 : 32;
        l.items.most = l.items.target + 2 + units;  // every row tile may end with a piece that is not full
        (l.tiles ? l.row_tiles.ctas : l.split.ctas) = l.items.most * kv;
        SpanArgs counts{};
        counts.n_groups = (int)w->n_groups;
        l.list = unit_count(counts, l.items, (int)q->seqs) > (k == 1 && p.launch[0].tiles ? kFewBesideTiles : kFewUnits);
        l.list_at = at;
        at += l.list ? (size_t)(l.items.most + 1) * sizeof(Item) : 0;  // behind a count
        l.parts_at = at;
        at += ((size_t)l.ctas() * l.rows() * (size_t)(c->dim + 2) * 4 + 63) / 64 * 64;
    }
    p.bytes = at;
    return p;
}

// Sharing saves the bytes of a prefix for each sequence but the first of a group, and costs
// a second and a third launch.  The host knows the table's width, which is the prefix and
// what follows, and so the most that can be saved: under 24 MB (4 sequences over 2048 tokens
// of 8 kv heads of 128: 12.1 us alone, 14.6 shared; 8: 18.8 and 16.4) the call goes without.
// So it does where a sequence's rows fill the 128 of half a row tile by themselves (16
// sequences of 240 rows over 8192 tokens: 154 and 211), and where the parts, two or more of
// each row, would take more than 512 MB.
bool worth_sharing(const bfft_cache_desc* c, const bfft_sequence_desc* q, const bfft_attention_desc* d,
                   const bfft_span_desc* w) {
    if (q->tokens / q->seqs * (d->q_heads / c->kv_heads) > 128 || q->seqs > 0x3fffffffLL) return false;
    const double saved = (double)(q->seqs - w->n_groups) * (double)seen_cover(c, q, d, 1, 1, w->sinks) *
                         (double)(c->kv_heads * c->dim * 2);
    return saved >= 24.0e6 && plan_groups(c, q, d, w, sm_count(d->device)).bytes <= (size_t)512 << 20;
}

template <typename T>
cudaError_t run_groups(const AttentionArgs& a, const SpanArgs& w, const GroupPlan& p, const bfft_cache_desc* c, char* ws,
                       unsigned int* status, cudaStream_t s) {
    int4* places[2] = {reinterpret_cast<int4*>(ws), reinterpret_cast<int4*>(ws) + a.seq.tokens};  // own, prefixes
    JoinArgs join{a, {}};
    ListArgs lists[2]{};
    for (int k = 0; k < p.launches; ++k) {
        const GroupLaunch& l = p.launch[k];
        ItemArgs x = l.items;
        x.own_of = places[0];
        x.prefix_of = places[1];
        if (l.list) {
            x.count = reinterpret_cast<int*>(ws + l.list_at);
            x.list = reinterpret_cast<Item*>(ws + l.list_at) + 1;
        }
        lists[k] = ListArgs{x, l.tile_tokens(), l.token_tiles(), const_cast<Item*>(x.list), const_cast<int*>(x.count)};
    }
    cudaError_t e = cudaSuccess;
    const bool on_the_way = p.launches == 2 && p.launch[0].tiles && lists[1].list;  // a block of the row tiles lists
    for (int k = 0; k < p.launches && e == cudaSuccess; ++k)
        if (lists[k].list && !(k == 1 && on_the_way)) e = run_list(a, w, lists[k], s);
    for (int k = 0; k < p.launches && e == cudaSuccess; ++k) {
        const GroupLaunch& l = p.launch[k];
        float* parts = reinterpret_cast<float*>(ws + l.parts_at);
        float* stats = parts + l.ctas() * l.rows() * c->dim;
        for (int set = 0; set < 2; ++set)
            if (set ? l.prefixes : l.own) join.set[set] = JoinSet{parts, stats, places[set], l.rows(), l.ctas()};
        if (l.tiles) {
            TileArgs t{};
            t.a = a;
            t.parts = parts;
            t.stats = stats;
            t.tile_tokens = l.row_tiles.tile_tokens;
            t.status = status;
            t.span = w;
            t.items = lists[k].items;
            if (k == 0 && on_the_way) t.others = lists[1];
            e = run_tiles<T, kGroups>(t, l.row_tiles, c, s);
        } else {
            SplitArgs t{};
            t.a = a;
            t.parts = parts;
            t.stats = stats;
            t.tile_tokens = l.split.tile_tokens;
            t.token_tiles = l.split.token_tiles;
            t.entries = l.split.entries;
            t.status = status;
            t.span = w;
            t.items = lists[k].items;
            e = run_split<T, kGroups>(t, l.split, c, s);
        }
    }
    return e == cudaSuccess ? run_join_items<T>(join, s) : e;
}
int group_launches(const GroupPlan& p) {
    int n = p.launches + 1;
    for (int k = 0; k < p.launches; ++k) n += p.launch[k].list && !(k == 1 && p.launch[0].tiles);
    return n;
}

// The form of a call: sinks matter beside a window only.
bfft_status check_span(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs, const bfft_attention_desc* d,
                       const bfft_span_desc* w, int* form) {
    *form = kPlain;
    if (w->sinks < 0 || w->sinks > 0x3fffffffLL) return fail(BFFT_ERR_VALUE, "bad count of first tokens %lld", (long long)w->sinks);
    if (w->n_groups < 0 || w->n_groups > 0x3fffffffLL) return fail(BFFT_ERR_SHAPE, "bad group count %lld", (long long)w->n_groups);
    if (w->n_groups && (!w->shared || (!w->groups && w->n_groups > 1))) return fail(BFFT_ERR_VALUE, "null pointer");
    if (!aligned(w->groups, 4) || !aligned(w->shared, 4)) return fail(BFFT_ERR_VALUE, "misaligned pointer");
    if (!seqs->tokens) return BFFT_OK;
    if (w->n_groups && worth_sharing(cache, seqs, d, w))
        *form = kGroups;
    else if (w->sinks && d->window > 0)
        *form = kSinks;
    if (*form != kPlain && seqs->max_pages > 0x3fffffffLL / cache->page)
        return fail(BFFT_ERR_SHAPE, "tables of %lld pages of %lld tokens are too wide", (long long)seqs->max_pages,
                    (long long)cache->page);
    return BFFT_OK;
}

bfft_status workspace_call(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs, const bfft_attention_desc* d,
                           const bfft_span_desc* w, size_t* bytes) {
    if (!bytes) return fail(BFFT_ERR_VALUE, "null pointer");
    bfft_status st = check(cache, seqs, d);
    int form = kPlain;
    if (st == BFFT_OK && w) st = check_span(cache, seqs, d, w, &form);
    if (st != BFFT_OK) return st;
    const int64_t sinks = form == kSinks ? w->sinks : 0;
    const int sms = sm_count(d->device);
    if (!seqs->tokens)
        *bytes = 0;
    else if (form == kGroups)
        *bytes = plan_groups(cache, seqs, d, w, sms).bytes;
    else
        *bytes = use_tiles(cache, seqs, d, sinks) ? plan_tiles(cache, seqs, d, sms, sinks).bytes
                                                  : plan_split(cache, seqs, d, sms, sinks).bytes;
    return BFFT_OK;
}

template <int MODE>
cudaError_t run_plan(bool tiles, const TileArgs& ta, const TilePlan& tp, const SplitArgs& sa, const SplitPlan& sp, int64_t type,
                     const bfft_cache_desc* c, cudaStream_t s) {
    if (tiles)
        return type == BFFT_F16 ? run_tiles<__half, MODE>(ta, tp, c, s) : run_tiles<__nv_bfloat16, MODE>(ta, tp, c, s);
    return type == BFFT_F16 ? run_split<__half, MODE>(sa, sp, c, s) : run_split<__nv_bfloat16, MODE>(sa, sp, c, s);
}

bfft_status attention_call(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs, const bfft_attention_desc* d,
                           const bfft_span_desc* w, void* stream) {
    bfft_status st = check(cache, seqs, d);
    int form = kPlain;
    if (st == BFFT_OK && w) st = check_span(cache, seqs, d, w, &form);
    if (st != BFFT_OK) return st;
    if (seqs->tokens == 0) return BFFT_OK;
    AttentionArgs a;
    a.cache = cache_view(cache);
    a.seq = sequence_view(seqs);
    a.q = d->q;
    a.out = d->out;
    a.lse = static_cast<float*>(d->lse);
    a.qt = d->q_token, a.qh = d->q_head, a.ot = d->o_token, a.oh = d->o_head;
    a.q_heads = (int)d->q_heads;
    a.group = (int)(d->q_heads / cache->kv_heads);
    a.causal = d->causal != 0;
    a.window = (int)d->window;
    a.scale_log2 = (float)(d->softmax_scale * 1.4426950408889634);
    Device g(d->device);
    if (!g.ok) return fail(BFFT_ERR_CUDA, "cannot select device %lld", (long long)d->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    a.q_packs = aligned(d->q, 16) && d->q_token % 8 == 0 && d->q_head % 8 == 0;
    a.o_packs = aligned(d->out, 16) && d->o_token % 8 == 0 && d->o_head % 8 == 0;
    unsigned int* status;
    cudaError_t e = device_status_word(&status);
    if (e != cudaSuccess) return launched(e, "cache_attention");
    const int sms = sm_count(d->device);
    SpanArgs span{};
    if (form != kPlain) span.sinks = d->window > 0 ? (int)w->sinks : 0;
    auto room = [&](int64_t ctas, size_t bytes) {
        if (ctas > 0x7fffffffLL || seqs->tokens * d->q_heads > 0x7fffffffLL)
            return fail(BFFT_ERR_SHAPE, "too many rows: %lld", (long long)seqs->tokens);
        if (bytes && (!d->workspace || d->workspace_bytes < (int64_t)bytes))
            return fail(BFFT_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed", (long long)d->workspace_bytes,
                        (long long)bytes);
        if (bytes && !aligned(d->workspace, 16)) return fail(BFFT_ERR_WORKSPACE, "workspace must be 16-byte aligned");
        return BFFT_OK;
    };
    if (form == kGroups) {
        span.groups = static_cast<const int32_t*>(w->groups);
        span.shared = static_cast<const int32_t*>(w->shared);
        span.n_groups = (int)w->n_groups;
        const GroupPlan p = plan_groups(cache, seqs, d, w, sms);
        st = room(p.launch[p.launches - 1].ctas() > p.launch[0].ctas() ? p.launch[p.launches - 1].ctas() : p.launch[0].ctas(),
                  p.bytes);
        if (st != BFFT_OK) return st;
        count_launches(group_launches(p));
        char* ws = static_cast<char*>(d->workspace);
        return launched(d->type == BFFT_F16 ? run_groups<__half>(a, span, p, cache, ws, status, s)
                                            : run_groups<__nv_bfloat16>(a, span, p, cache, ws, status, s),
                        "cache_attention");
    }
    const bool tiles = use_tiles(cache, seqs, d, span.sinks);
    TilePlan tp{};
    SplitPlan sp{};
    if (tiles)
        tp = plan_tiles(cache, seqs, d, sms, span.sinks);
    else
        sp = plan_split(cache, seqs, d, sms, span.sinks);
    const int chunks = tiles ? tp.chunks : sp.chunks;
    st = room(tiles ? tp.ctas : sp.ctas, tiles ? tp.bytes : sp.bytes);
    if (st != BFFT_OK) return st;
    float* parts = static_cast<float*>(d->workspace);
    float* stats = parts ? parts + seqs->tokens * d->q_heads * chunks * cache->dim : nullptr;
    count_launches(chunks > 1 && !sp.cluster ? 2 : 1);
    const TileArgs ta{a,           parts,    stats,  tp.chunk, tp.chunks, tp.tile_tokens,
                      tp.by_token, tp.slots, status, 0,        span,      {},
                      {}};
    const SplitArgs sa{a,           parts,    stats,      sp.chunk,   sp.chunks, sp.tile_tokens, sp.token_tiles,
                       sp.by_token, sp.slots, sp.cluster, sp.entries, status,    span,           {}};
    e = form == kSinks ? run_plan<kSinks>(tiles, ta, tp, sa, sp, d->type, cache, s)
                       : run_plan<kPlain>(tiles, ta, tp, sa, sp, d->type, cache, s);
    return launched(e, "cache_attention");
}

}  // namespace

extern "C" bfft_status bfft_cache_attention_workspace(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs,
                                                      const bfft_attention_desc* d, size_t* bytes) {
    return workspace_call(cache, seqs, d, nullptr, bytes);
}

extern "C" bfft_status bfft_cache_attention_span_workspace(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs,
                                                           const bfft_attention_desc* d, const bfft_span_desc* w,
                                                           size_t* bytes) {
    if (!w) return fail(BFFT_ERR_VALUE, "null pointer");
    return workspace_call(cache, seqs, d, w, bytes);
}

extern "C" bfft_status bfft_cache_attention(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs,
                                            const bfft_attention_desc* d, void* stream) {
    return attention_call(cache, seqs, d, nullptr, stream);
}

extern "C" bfft_status bfft_cache_attention_span(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs,
                                                 const bfft_attention_desc* d, const bfft_span_desc* w, void* stream) {
    if (!w) return fail(BFFT_ERR_VALUE, "null pointer");
    return attention_call(cache, seqs, d, w, stream);
}
