// bfft_attention_split.cuh -- attention of few query rows over a long axis of
// 8-bit tokens (single tokens, drafted tokens).  Included by bfft_attention.cuh.
//
// Bound by the cache's bytes: with G query heads to a kv head a code (one byte)
// meets G products, far under the tensor rate, so the design is about keeping
// loads in flight and spending few instructions on a code:
//
// * The token axis is cut into chunks, one CTA per (row tile, kv head, chunk);
//   its four warps take 32-token tiles in turn, each with a ring of its own that
//   the copy engine fills (128-byte swizzled boxes for heads of 64, 128 and 256;
//   plain bulk copies for other widths), so no barrier joins the warps until the
//   chunk's end.  Up to eight chunks are a thread-block cluster and joined through
//   distributed shared memory; the parts of more by k_attention_join.
// * Products on m16n8k16 matrix instructions with tokens as rows and query heads
//   as columns, S^T = K Q^T and O^T = V^T P^T: eight heads fill a tile (rows of
//   queries would fill half of a 16-row one).  The order of the 16 products of an
//   instruction is free, so a lane takes 16 adjacent codes of a token (K) or of
//   each of four tokens (V) with one 16-byte load and widens them in registers;
//   both 8-bit types are exact in float16.
// * A block's key scale multiplies the scores.  Its value scale is folded into
//   the exponent: p' = 2^(z + log2 vs - m) with m the running maximum of z + log2
//   vs, so P' (float16) times codes is the weighted value, and the sum takes
//   p' / vs.  The largest p' is set to 2^14, near float16's top, so that weighted
//   values keep their bits down to 2^-28 of the largest; m is renewed when one
//   passes 2^15.5 (a vote instead of a reduction on most tiles).  A CTA that meets
//   a value scale under 2^-48 keeps its sum 2^36 times smaller (see SmallScales).
//
// * A tile's two 16-token halves go side by side through every step, dead ones masked
//   instead of skipped: with 8 or 12 warps to an SM the chain of a tile's products,
//   scores and exponentials is what a warp waits for (64 ragged sequences 399 us with the
//   halves one after the other and a branch between them, 357 so on that GPU).
//
// 64 sequences of 1024..32768 tokens, one row of 32 heads each (8 kv heads, 128
// dimensions): int8 357 to 362 us, 0.97 to 0.96 of the measured HBM rate; e4m3, whose
// codes take 2 instructions for 4 to widen instead of 5, 356.  One sequence of 131001 e4m3
// tokens, 64 heads: 55 us, the joining kernel's among them.
#pragma once

namespace bfft {

constexpr int kDeadBlock = 3;  // BlockScale::kind of tokens that nothing sees
// Value scale of a zero block: its codes must not count, its weights must.
constexpr float kZeroLog2 = -64.f;
// The sum takes p' / vs: up to 2^15.5 a token over a value scale of 2^-126, the least
// that is kept, and 2^20 tokens pass float32's 2^128 from 2^-91 on.  The joining
// kernel and the output take a sum in any unit that O shares, so where a CTA's tokens
// have a scale under 2^-48 its sum and, at the end, its O are held 2^36 times smaller
// (at most 2^126; large scales stay clear of 2^-126 up to 2^80).  There a zero block
// counts as 2^-126: as 2^-64 it would set the maximum by which the weights of such
// small values are rounded.  Looking for it costs 0.1 us of a short decode (8.4).
struct SmallScales {
    static constexpr float under_log2 = -48.f, zero_log2 = -126.f, shift = 36.f;
    static constexpr float factor = 1.f / 68719476736.f;                 // 2^-36
    static constexpr float inv_zero = 1237940039285380274899124224.f;   // 2^126 2^-36
};
constexpr float kTop = 14.f, kRenew = 15.5f;  // log2 of p' at the maximum, and where the maximum is renewed

struct SplitArgs {
    AttentionArgs a;
    float* parts;        // [tokens][q_heads][chunks][dim], then m and l as [..][chunks][2]
    float* stats;
    int chunk;           // tokens of a chunk, a multiple of 32
    int chunks;
    int tile_tokens;     // query tokens of a row tile (group <= rows of a tile), else 1
    int token_tiles;     // row tiles of a query token (group > rows of a tile), else 1
    int by_token;        // slots are tokens (else runs of tile_tokens, see slot_rows)
    int64_t slots;
    int cluster;         // the chunks of a row tile are one thread-block cluster, which joins them
    int entries;         // pages that a chunk can touch (kSinks, kGroups: that are held at a time)
    unsigned int* status;
    SpanArgs span;
    ItemArgs items;      // kGroups
};

constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = 32 * kSplitWarps;

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Shared memory at `local`'s place in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_address(const void* local, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 cluster_load2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Four codes of a word as two pairs of float16, exactly.  Int8: c + 128 in the
// low byte of 1024 (float16 holds integers to 2048), minus 1152.
template <int CODE>
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (CODE == kCodeInt8) {
        w ^= 0x80808080u;
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t l = __byte_perm(w, 0x64646464u, 0x4140), h = __byte_perm(w, 0x64646464u, 0x4342);
        __half2 l2 = __hsub2(*reinterpret_cast<const __half2*>(&l), bias);
        __half2 h2 = __hsub2(*reinterpret_cast<const __half2*>(&h), bias);
        lo = *reinterpret_cast<uint32_t*>(&l2);
        hi = *reinterpret_cast<uint32_t*>(&h2);
    } else {
        asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    }
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Power of two that brings a row's largest magnitude to [1, 2), in the last binades to
// [1, 4) (the power is a normal float), and its inverse, so that bfloat16 queries fit
// float16 (exactly, but for elements under 2^-14 of the row's largest, which lose bits
// under 2^-24 of it).  1 where the row is zero or not finite.
template <typename T>
__device__ __forceinline__ void row_power(float big, float& down, float& up) {
    down = up = 1.f;
    if constexpr (sizeof(T) == 2) {
        int e = (int)(__float_as_uint(big) >> 23) & 255;
        if (e > 0 && e < 255) {
            e = e < 253 ? e : 253;
            down = __uint_as_float((uint32_t)(254 - e) << 23);
            up = __uint_as_float((uint32_t)e << 23);
        }
    }
}
template <>
__device__ __forceinline__ void row_power<__half>(float, float& down, float& up) {
    down = up = 1.f;
}

// The value scale's part in the exponent, its inverse in the sum, and whether the
// block's values count (a zero scale, or one under 2^-126: the append keeps none) or
// spoil the rows that see it.
struct BlockScale {
    float key;
    float log2_value;
    float inv_value;
    int kind;  // 0 ordinary, 1 zero values, 2 values that are not finite, kDeadBlock
};
__device__ __forceinline__ BlockScale block_scale(float ks, float vs) {
    BlockScale b;
    b.key = ks;
    b.kind = vs >= 0.f && vs < 1.17549435e-38f ? 1 : (vs > 0.f && vs < INFINITY) ? 0 : 2;
    b.log2_value = b.kind == 0 ? log2f(vs) : kZeroLog2;
    b.inv_value = b.kind == 0 ? 1.f / vs : 18446744073709551616.f;
    return b;
}
__device__ __forceinline__ bool small_scale(const BlockScale& b) {
    return b.kind == 0 && b.log2_value < SmallScales::under_log2;
}
__device__ __forceinline__ void to_small(BlockScale& b) {
    b.inv_value = b.kind == 0 ? b.inv_value * SmallScales::factor : SmallScales::inv_zero;
    if (b.kind != 0) b.log2_value = SmallScales::zero_log2;
}

// The query tokens [first, first + n) of sequence s that slot i stands for, the
// first of them row `place` of the sequence's `rows`.
struct SlotRows {
    int s;
    int64_t first, place, rows;
    int n;
};
__device__ __forceinline__ bool slot_rows(const SequenceView& q, int64_t i, int tile, int by_token, SlotRows& r) {
    int s;
    if (by_token) {
        s = find_sequence(q.starts, q.seqs, i);
    } else {
        const int lane = threadIdx.x & 31;
        int lo = 0, n = q.seqs;
        while (n > 1) {
            const int step = (n + 31) >> 5, j = lane * step;
            const bool le = j < n && (int64_t)(q.starts[lo + j] / tile) + (lo + j) <= i;
            const int c = __popc(__ballot_sync(0xffffffffu, le));
            const int skip = (c > 0 ? c - 1 : 0) * step;
            lo += skip;
            n = n - skip < step ? n - skip : step;
        }
        s = lo;
    }
    const int64_t t0 = q.starts[s];
    int64_t t1 = q.starts[s + 1];
    if (t1 > q.tokens) t1 = q.tokens;
    if (t0 < 0 || t0 >= t1) return false;
    int64_t place;
    if (by_token) {
        if (i < t0 || i >= t1) return false;
        place = i - t0;
        if (place % tile) return false;
    } else {
        const int64_t j = i - (t0 / tile + s);
        if (j < 0) return false;
        place = j * tile;
        if (place >= t1 - t0) return false;
    }
    r.s = s;
    r.rows = t1 - t0;
    r.place = place;
    r.first = t0 + place;
    r.n = (int)(r.rows - place < tile ? r.rows - place : tile);
    return true;
}

// Tokens [lo, hi) that the row at `pos` sees.
__device__ __forceinline__ void seen_range(const AttentionArgs& a, int64_t pos, int64_t len, int64_t& lo, int64_t& hi) {
    hi = a.causal ? pos + 1 : len;
    if (hi > len) hi = len;
    lo = 0;
    if (a.window > 0 && pos - a.window + 1 > 0) lo = pos - a.window + 1;
}

// Shared memory: the warps' rings (a stage: keys of both 16-token halves, then values),
// in whose place the warps' parts and the CTA's for the cluster come, and the scale and
// number of each page.
constexpr int kSplitStages = 2;
constexpr int kSplitSmemMost = 226 * 1024;
__host__ __device__ constexpr int split_half_bytes(int dim) { return 16 * dim; }
__host__ __device__ constexpr int split_body_bytes(int dim, int rows) {
    const int ring = kSplitWarps * kSplitStages * 4 * split_half_bytes(dim), merge = (kSplitWarps + 1) * rows * (dim + 2) * 4;
    return ring > merge ? ring : merge;
}
__host__ __device__ constexpr int split_smem(int dim, int rows, int entries) {
    return 1024 + split_body_bytes(dim, rows) + entries * (int)(sizeof(BlockScale) + 4) + 64;
}

template <int DP, bool EXACT, int NT>
struct SplitGeo {
    static constexpr int STAGES = kSplitStages;
    static constexpr int ROWS = 8 * NT;
    static constexpr int KS = DP / 16;         // products of 16 along a head
    static constexpr int VW = DP / 32;         // words of a token's values in a lane
    __host__ __device__ static constexpr int half_bytes(int dim) { return split_half_bytes(dim); }
};

// Three CTAs an SM by their registers where that costs no spills: up to 168 for 8-row tiles and
// for 64-wide heads (with 176 to 204, two CTAs, 16-row tiles of these were slower: 64 sequences
// of 4 rows over 1000..9000 tokens 142 us for 129, 8 prompts of 100 rows with a window of 31
// tokens 39 for 30).
template <int DP, bool EXACT, int NT, typename T, int CODE, int MODE>
__global__ void __launch_bounds__(kSplitThreads, DP == 64 || (NT == 1 && DP == 128) ? 3 : 2)
    k_attention_split(SplitArgs p, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
    using G = SplitGeo<DP, EXACT, NT>;
    extern __shared__ unsigned char smem_raw[];
    const AttentionArgs& a = p.a;
    griddep_wait();
    const int dim = EXACT ? DP : a.cache.dim;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, q4 = lane & 3;
    unsigned char* ring = align_smem<1024>(smem_raw);
    BlockScale* scales = reinterpret_cast<BlockScale*>(ring + split_body_bytes(dim, G::ROWS));
    int* page_ids = reinterpret_cast<int*>(scales + p.entries);
    __shared__ uint64_t full[kSplitWarps * G::STAGES];

    // which rows and tokens
    int64_t i = blockIdx.x;
    int chunk = 0, kv, part;
    SlotRows sr{};
    Item it{};
    TokenSpan mine_span{0, 0, 0};  // kSinks, kGroups: of query token `lane` of the tile
    if constexpr (MODE == kGroups) {
        __shared__ TokenSpan spans[16];
        if (tid < 16) spans[tid] = TokenSpan{0, 0, 0};
        const unsigned item = blockIdx.x / (unsigned)a.cache.kv_heads;
        kv = (int)(blockIdx.x - item * a.cache.kv_heads);
        if (!find_item(a, p.span, p.items, (int)item, p.tile_tokens, p.token_tiles, it)) return;
        if (it.prefix) {
            __syncthreads();
            item_spans<kSplitThreads>(a, p.span, it, spans);
            if (lane < it.n) mine_span = spans[lane];
        } else if (lane < it.n) {
            mine_span = token_span(a, p.span, (int64_t)it.pos + lane, it.len, it.from, it.to);
        }
        part = it.part;
        chunk = it.chunk;
        sr.s = it.table_row;
        sr.first = it.token;
        sr.n = it.n;
    } else {
        chunk = (int)(i % p.chunks);
        i /= p.chunks;
        kv = (int)(i % a.cache.kv_heads);
        i /= a.cache.kv_heads;
        part = (int)(i % p.token_tiles);
    }
    if (tid == 0) {
        for (int b = 0; b < kSplitWarps * G::STAGES; ++b) mbar_init(&full[b], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if constexpr (MODE != kGroups)
        if (!slot_rows(a.seq, i / p.token_tiles, p.tile_tokens, p.by_token, sr)) return;
    const int head0 = part * G::ROWS;                       // of the group, where a token takes several tiles
    const int per_token = p.token_tiles > 1 ? min(a.group - head0, G::ROWS) : a.group;
    const int rows = sr.n * per_token;
    // [base, end) of the axis: kPlain counts sequence tokens, the others places of `axis`
    int64_t len = 0, pos0 = 0, base, end, lo_min = 0, hi_max, lo_max = 0, hi_min;
    Axis axis{};
    if constexpr (MODE == kPlain) {
        len = a.seq.lens[sr.s];
        const int64_t most = (int64_t)a.seq.max_pages << a.cache.page_log2;
        if (len > most) len = most;
        pos0 = (int64_t)a.seq.lens[sr.s] - sr.rows + sr.place;
        seen_range(a, pos0, len, lo_min, hi_min);
        seen_range(a, pos0 + sr.n - 1, len, lo_max, hi_max);
        base = (lo_min & ~(int64_t)15) + (int64_t)chunk * p.chunk;
        end = base + p.chunk;
        if (end > hi_max) end = hi_max;
    } else {
        int first = 0;
        if (MODE == kGroups) first = it.from;
        if (MODE == kSinks && lane < sr.n)
            mine_span = token_span(a, p.span, (int64_t)a.seq.lens[sr.s] - sr.rows + sr.place + lane, a.seq.lens[sr.s], 0,
                                   0x7fffffff);
        if (lane >= sr.n) mine_span.sinks = first;
        const bool some = mine_span.lo < mine_span.hi;
        axis = make_axis(first, __reduce_min_sync(0xffffffffu, some ? mine_span.lo : 0x7fffffff),
                         __reduce_max_sync(0xffffffffu, some ? mine_span.hi : 0),
                         __reduce_max_sync(0xffffffffu, mine_span.sinks));
        const int pieces = MODE == kGroups ? it.chunks : p.chunks;
        const int64_t each = ((axis.total + pieces - 1) / pieces + 31) & ~31;
        base = chunk * each;
        end = base + each;
        if (end > axis.total) end = axis.total;
    }
    const bool direct = MODE == kGroups && !it.prefix && !it.shares && it.chunks == 1;
    if constexpr (MODE == kGroups) {  // where the join finds the parts of the tile's tokens
        if (kv == 0 && part == 0 && chunk == 0 && tid < sr.n) {
            const int flags = (direct ? kPlaceDone : 0) | (!it.prefix && it.shares ? kPlacePrefix : 0);
            (it.prefix ? p.items.prefix_of : p.items.own_of)[sr.first + tid] =
                make_int4((int)(blockIdx.x / a.cache.kv_heads), it.chunks, p.token_tiles > 1 ? 0 : tid * a.group, flags);
        }
    }
    // row r of the tile: query token r / per_token, head r % per_token
    auto row_of = [&](int r, int64_t& token, int& head) {
        const int t = r / per_token;
        token = sr.first + t;
        head = kv * a.group + head0 + (r - t * per_token);
    };
    float* part_o = reinterpret_cast<float*>(ring);  // of the warps, at the end; then of the CTA
    float* part_ml = part_o + kSplitWarps * G::ROWS * dim;
    float* cta_o = part_ml + kSplitWarps * G::ROWS * 2;
    float* cta_ml = cta_o + G::ROWS * dim;
    if (base >= end) {  // nothing of the axis in this chunk
        if (tid < rows) {
            int64_t token;
            int head;
            row_of(tid, token, head);
            if (p.cluster) {
                cta_ml[tid * 2] = -INFINITY;
                cta_ml[tid * 2 + 1] = 0.f;
            } else if (MODE == kGroups ? !direct : p.chunks > 1) {
                const int64_t at = MODE == kGroups ? (int64_t)blockIdx.x * G::ROWS + tid
                                                   : (token * a.q_heads + head) * p.chunks + chunk;
                float* st = p.stats + at * 2;
                st[0] = -INFINITY;
                st[1] = 0.f;
            } else if (a.lse) {
                a.lse[token * a.q_heads + head] = -INFINITY;
            }
        }
        if (MODE == kGroups ? direct : p.chunks == 1)
            for (int e = tid; e < rows * dim; e += kSplitThreads) {
                int64_t token;
                int head;
                row_of(e / dim, token, head);
                static_cast<T*>(a.out)[token * a.ot + head * a.oh + e % dim] = from_f32<T>(0.f);
            }
        if (!p.cluster) return;
    } else {
    // The queries of this lane's rows, 16 adjacent elements by two loads, on their way while
    // the pages are looked up.
    auto query_of = [&](int r) -> const T* {
        if (r >= rows) return nullptr;
        int64_t token;
        int head;
        row_of(r, token, head);
        return static_cast<const T*>(a.q) + token * a.qt + head * a.qh;
    };
    Pack<T, 8> q_raw[NT][G::KS / 4][2];
    if (a.q_packs) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const T* x = query_of(nt * 8 + g);
#pragma unroll
            for (int c = 0; c < G::KS / 4; ++c) {
                const int d = 16 * (4 * c + q4);
                const bool has = x && (EXACT || d < dim);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    q_raw[nt][c][j] = has ? *reinterpret_cast<const Pack<T, 8>*>(x + d + 8 * j) : Pack<T, 8>{};
            }
        }
    }
    // From here on tokens are counted in 32 bits: kPlain from `base`, the others in places
    // of the axis.  A segment is what the table of pages holds: kPlain's chunks are one.
    const int lg = a.cache.page_log2, page_mask = (1 << lg) - 1;
    int64_t page0 = 0;
    int off = 0, span = 0, entries = 0;  // of kPlain: base's place in its page, tokens, pages
    int seg = 0, stop = 0, heads = 0, head_off = 0, main_off = 0, head_page = 0, main_page = 0;  // of the others: the segment
    // [seg, stop), its first tokens' pages, and the places of seg (of the window's first token) in theirs
    if constexpr (MODE == kPlain) {
        page0 = base >> lg;
        off = (int)(base & page_mask);
        span = (int)(end - base);
        entries = ((off + span - 1) >> lg) + 1;
        stop = span;
    }
    auto open_segment = [&](int from) {
        seg = from;
        const int room = (p.entries - 4) << lg;
        stop = (int)end - from > room ? from + room : (int)end;
        const int turn = axis.head < from ? from : axis.head < stop ? axis.head : stop;  // first tokens before it
        head_off = (axis.first + from) & page_mask;
        head_page = (axis.first + from) >> lg;
        heads = turn > from ? ((head_off + turn - from - 1) >> lg) + 1 : 0;
        const int at = axis.main + (turn - axis.head);
        main_off = (at & page_mask) - turn;
        main_page = at >> lg;
        entries = heads + (stop > turn ? ((main_off + stop - 1) >> lg) + 1 : 0);
    };
    // the table's entry of place t, and t's place in its page
    auto entry_of = [&](int t) {
        if constexpr (MODE == kPlain) return (off + t) >> lg;
        return t < axis.head ? (head_off + t - seg) >> lg : heads + ((main_off + t) >> lg);
    };
    auto slot_of = [&](int t) {
        if constexpr (MODE == kPlain) return (off + t) & page_mask;
        return (t < axis.head ? head_off + t - seg : main_off + t) & page_mask;
    };
    // The scales of the first entries are asked for with their pages: behind the tiles' copies
    // of all CTAs that start together (28 MB) they took 5300 clocks.
    float2 scale_raw = make_float2(0.f, 0.f);  // of this thread's first entry
    auto fetch_scale = [&](int id) {
        if (id < 0) return make_float2(0.f, 0.f);
        const int64_t b = (int64_t)id * a.cache.kv_heads + kv;
        return make_float2(a.cache.k_scale[b], a.cache.v_scale[b]);
    };
    auto load_pages = [&] {
#pragma unroll 1
        for (int e = tid; e < entries; e += kSplitThreads) {
            int64_t at = page0 + e;
            if (MODE != kPlain) at = e < heads ? head_page + e : main_page + e - heads;
            const int64_t id = a.seq.block_table[sr.s * a.seq.table_stride + at];
            page_ids[e] = id >= 0 && id < a.cache.pages ? (int)id : -1;
            if (e == tid) scale_raw = fetch_scale(page_ids[e]);
        }
    };
    auto load_scales = [&] {  // those behind scale_raw follow
        bool small = false;
#pragma unroll 1
        for (int e = tid; e < entries; e += kSplitThreads) {
            if (e != tid) scale_raw = fetch_scale(page_ids[e]);
            if (page_ids[e] >= 0) {
                scales[e] = block_scale(scale_raw.x, scale_raw.y);
                small |= small_scale(scales[e]);
            } else {
                scales[e] = BlockScale{0.f, 0.f, 0.f, kDeadBlock};
            }
        }
        return small;
    };
    auto rel = [&](int64_t t) { return (int)(t < base ? 0 : t - base > span ? span : t - base); };
    int lo_all, hi_all, lo_any, sinks_all = 0;
    if constexpr (MODE == kPlain) {
        lo_all = rel(lo_max);
        hi_all = rel(hi_min);
        lo_any = rel(lo_min);
    } else {
        open_segment((int)base);
        lo_any = axis.lo_any;
        const bool valid = lane < sr.n;
        lo_all = __reduce_max_sync(0xffffffffu, valid ? axis.place(mine_span.lo) : -0x7fffffff);
        hi_all = __reduce_min_sync(0xffffffffu, valid ? axis.place(mine_span.hi) : 0x7fffffff);
        sinks_all = __reduce_min_sync(0xffffffffu, valid ? mine_span.sinks - axis.first : 0x7fffffff);
    }
    load_pages();
    __syncthreads();

    // ring: tile t of this warp covers tokens [seg + 32 (t kSplitWarps + warp), + 32)
    int tiles = (stop - seg + 31) >> 5;
    unsigned char* mine = ring + warp * (G::STAGES * 4 * G::half_bytes(dim));
    uint64_t* bars = full + warp * G::STAGES;
    const int lines = EXACT ? DP / 8 : 1;  // 128-byte lines of 16 tokens
    auto fetch = [&](int t, int stage) {   // lanes 0..3: keys of half 0, 1, values of half 0, 1
        const int tok = seg + t * 32 + (lane & 1) * 16;
        int id = -1;
        if (lane < 4 && tok < stop) id = page_ids[entry_of(tok)];
        const unsigned any = __ballot_sync(0xffffffffu, id >= 0);
        if (lane == 0) mbar_arrive_expect_tx(&bars[stage], (uint32_t)(__popc(any) * G::half_bytes(dim)));
        __syncwarp();
        if (id >= 0) {
            unsigned char* dst = mine + (stage * 4 + lane) * G::half_bytes(dim);
            const int slot_in = slot_of(tok);
            if constexpr (EXACT) {
                tma_load_3d(dst, lane < 2 ? &kmap : &vmap, 0, ((kv << lg) + slot_in) / 16 * lines, id, &bars[stage]);
            } else {
                const uint8_t* src = (lane < 2 ? a.cache.k : a.cache.v) +
                                     ((((int64_t)id * a.cache.kv_heads + kv) << lg) + slot_in) * dim;
                bulk_load(dst, src, (uint32_t)G::half_bytes(dim), &bars[stage]);
            }
        }
    };
    int ahead = warp, fetched = 0;  // next tile to fetch, and how many were
    for (int s = 0; s < G::STAGES && ahead < tiles; ++s, ahead += kSplitWarps, ++fetched) fetch(ahead, s);
    // queries as B fragments: lane (g, q4) holds row g of each 8-row tile, dims 16 (4 i + q4) + 4 t ..
    uint32_t qf[NT][G::KS][2];
    float row_scale[NT][2];      // of rows 2 q4, 2 q4 + 1: softmax scale (log2) times the row's power
    int row_lo[NT][2], row_hi[NT][2], row_sinks[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 8 + g;
        float big = 0.f;
        const T* x = query_of(r);
        float e[G::KS][4];
        if (a.q_packs) {
#pragma unroll
            for (int c = 0; c < G::KS / 4; ++c)
#pragma unroll
                for (int j = 0; j < 16; ++j) e[4 * c + j / 4][j & 3] = to_f32(q_raw[nt][c][j >> 3].v[j & 7]);
        } else {
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int d = 16 * (4 * (ks >> 2) + q4) + 4 * (ks & 3) + j;
                    e[ks][j] = x && (EXACT || d < dim) ? to_f32(x[d]) : 0.f;
                }
        }
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
            for (int j = 0; j < 4; ++j) big = fmaxf(big, fabsf(e[ks][j]));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        float down, up;
        row_power<T>(big, down, up);
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks) {
            qf[nt][ks][0] = pack_f16(e[ks][0] * down, e[ks][1] * down);
            qf[nt][ks][1] = pack_f16(e[ks][2] * down, e[ks][3] * down);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            row_scale[nt][j] = __shfl_sync(0xffffffffu, up, (2 * q4 + j) * 4) * a.scale_log2;
            const int rr = nt * 8 + 2 * q4 + j;
            if constexpr (MODE == kPlain) {
                int64_t lo, hi;
                seen_range(a, pos0 + (rr < rows ? rr / per_token : 0), len, lo, hi);
                row_lo[nt][j] = rel(lo);
                row_hi[nt][j] = rel(hi);
                row_sinks[nt][j] = 0;
            } else {
                const int of = rr < rows ? rr / per_token : 0;
                row_lo[nt][j] = axis.place(__shfl_sync(0xffffffffu, mine_span.lo, of));
                row_hi[nt][j] = axis.place(__shfl_sync(0xffffffffu, mine_span.hi, of));
                row_sinks[nt][j] = __shfl_sync(0xffffffffu, mine_span.sinks, of) - axis.first;
            }
        }
    }
    bool any_small = load_scales();
    bool small = __syncthreads_or(any_small);  // a small value scale in the chunk (kPlain), or so far
    if (small) {
        for (int e = tid; e < entries; e += kSplitThreads) to_small(scales[e]);
        __syncthreads();
    }

    float o[NT][2 * G::VW][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int u = 0; u < 2 * G::VW; ++u)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[nt][u][c] = 0.f;
    }

    auto at = [&](int byte) { return EXACT ? byte ^ (((byte >> 7) & 7) << 4) : byte; };
    // token of fragment row r < 8: even rows in place, odd ones four apart, so that
    // the eight lanes of a 16-byte load phase meet eight different banks
    auto row_token = [](int r) { return (r & 1) ? r ^ 4 : r; };
    const int tk = row_token(g);

    bool ok = true;
    int used = 0;  // tiles that this warp has waited for
    for (;;) {     // segments
    for (int t = warp; t < tiles; t += kSplitWarps, ++used) {
        const int stage = used % G::STAGES;
        ok = mbar_wait_limited(&bars[stage], (uint32_t)((used / G::STAGES) & 1), p.status);
        if (__any_sync(0xffffffffu, !ok)) {
            ok = false;
            break;
        }
        const int tok0 = seg + t * 32;
        const unsigned char* buf = mine + stage * 4 * G::half_bytes(dim);
        // Both halves' tokens go through each step side by side, dead ones too (their scores
        // become -inf, their codes zeros): twice the products in flight, and no branches
        // between them.
        float z[2][NT][4];
        BlockScale bs[2];
        bool live[2], inside = true, whole = true;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int tok = tok0 + 16 * h;
            const int e = entry_of(tok);
            bs[h] = scales[e < entries ? e : entries - 1];
            live[h] = tok < stop && bs[h].kind != kDeadBlock;
            bool in = tok >= lo_all && tok + 16 <= hi_all;  // kPlain: hi_all is at most span
            if (MODE != kPlain) in = (in && tok + 16 <= stop) || tok + 16 <= sinks_all;
            inside = inside && in && live[h];
            in = tok >= lo_any && tok + 16 <= stop;
            if (MODE != kPlain) in = (in && tok + 16 <= axis.hi_any) || tok + 16 <= axis.sinks_any;
            whole = whole && in && live[h];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) z[h][nt][0] = z[h][nt][1] = z[h][nt][2] = z[h][nt][3] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < (DP + 63) / 64; ++c) {
            uint4 w[2][2];
            const int col = 16 * (4 * c + q4);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const unsigned char* kb = buf + h * G::half_bytes(dim);
                w[h][0] = w[h][1] = make_uint4(0, 0, 0, 0);
                if (EXACT || col < dim) {
                    w[h][0] = *reinterpret_cast<const uint4*>(kb + at(tk * dim + col));
                    w[h][1] = *reinterpret_cast<const uint4*>(kb + at((tk + 8) * dim + col));
                }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t u0 = s == 0 ? w[h][0].x : s == 1 ? w[h][0].y : s == 2 ? w[h][0].z : w[h][0].w;
                    const uint32_t u1 = s == 0 ? w[h][1].x : s == 1 ? w[h][1].y : s == 2 ? w[h][1].z : w[h][1].w;
                    uint32_t a0, a1, a2, a3;
                    widen<CODE>(u0, a0, a2);
                    widen<CODE>(u1, a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_f16(z[h][nt], a0, a1, a2, a3, qf[nt][c * 4 + s][0], qf[nt][c * 4 + s][1]);
                }
        }
        float worst = -INFINITY;  // largest z - m of this lane
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    z[h][nt][c] = z[h][nt][c] * (bs[h].key * row_scale[nt][c & 1]) + bs[h].log2_value;
        if (!inside) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const int j = tok0 + 16 * h + tk + (c >> 1) * 8;
                        bool hidden = j < row_lo[nt][c & 1] || j >= row_hi[nt][c & 1];
                        if (MODE != kPlain) hidden = hidden && j >= row_sinks[nt][c & 1];
                        if (hidden || !live[h]) z[h][nt][c] = -INFINITY;
                    }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const float v = z[h][nt][c];
                    worst = fmaxf(worst, v == -INFINITY ? v : v - m[nt][c & 1]);
                }
        if (__any_sync(0xffffffffu, worst > kRenew)) {  // a score far over a reference (or the first one): renew them
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = -INFINITY;
#pragma unroll
                    for (int h = 0; h < 2; ++h) top = fmaxf(top, fmaxf(z[h][nt][j], z[h][nt][2 + j]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                    const float now = fmaxf(m[nt][j], top - kTop);
                    const float f = now == -INFINITY ? 1.f : exp2_approx(m[nt][j] - now);
                    m[nt][j] = now;
                    l[nt][j] *= f;
#pragma unroll
                    for (int u = 0; u < 2 * G::VW; ++u) {
                        o[nt][u][j] *= f;
                        o[nt][u][2 + j] *= f;
                    }
                }
        }
        // values: tokens t0, t1, t0 + 8, t1 + 8 of this lane, dims 4 w .. 4 w + 3 of its columns
        const int t0 = row_token(2 * q4), t1 = row_token(2 * q4 + 1);
        const int toks[4] = {t0, t1, t0 + 8, t1 + 8};
        uint32_t w[2][4][G::VW];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned char* vb = buf + (2 + h) * G::half_bytes(dim);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (DP == 64) {
                    uint2 x = make_uint2(0, 0);
                    if (EXACT || 8 * g < dim) x = *reinterpret_cast<const uint2*>(vb + at(toks[k] * dim + 8 * g));
                    w[h][k][0] = x.x;
                    w[h][k][1] = x.y;
                } else {
#pragma unroll
                    for (int c = 0; c < DP / 128; ++c) {
                        uint4 x = make_uint4(0, 0, 0, 0);
                        const int col = 16 * g + 128 * c;
                        if (EXACT || col < dim) x = *reinterpret_cast<const uint4*>(vb + at(toks[k] * dim + col));
                        w[h][k][4 * c] = x.x;
                        w[h][k][4 * c + 1] = x.y;
                        w[h][k][4 * c + 2] = x.z;
                        w[h][k][4 * c + 3] = x.w;
                    }
                }
            }
        }
        if (!whole) {  // codes of slots that no row sees may be anything: 0 times NaN is NaN
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int j = tok0 + 16 * h + toks[k];
                    bool drop = j < lo_any || j >= stop;
                    if (MODE != kPlain) drop = (j < lo_any || j >= axis.hi_any) && j >= axis.sinks_any;
                    if (drop || !live[h])
#pragma unroll
                        for (int c = 0; c < G::VW; ++c) w[h][k][c] = 0;
                }
        }
        float e[2][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int c = 0; c < 4; ++c) e[h][nt][c] = exp2_approx(z[h][nt][c] - (c & 1 ? m1 : m0));
                l[nt][0] += (e[h][nt][0] + e[h][nt][2]) * bs[h].inv_value;
                l[nt][1] += (e[h][nt][1] + e[h][nt][3]) * bs[h].inv_value;
            }
        }
        if (bs[0].kind | bs[1].kind) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!bs[h].kind) continue;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if (bs[h].kind == 2) {  // values that are not finite spoil the rows that see one of them
                        int seen0 = z[h][nt][0] != -INFINITY || z[h][nt][2] != -INFINITY;
                        int seen1 = z[h][nt][1] != -INFINITY || z[h][nt][3] != -INFINITY;
#pragma unroll
                        for (int d = 4; d < 32; d <<= 1) {
                            seen0 |= __shfl_xor_sync(0xffffffffu, seen0, d);
                            seen1 |= __shfl_xor_sync(0xffffffffu, seen1, d);
                        }
#pragma unroll
                        for (int u = 0; u < 2 * G::VW; ++u) {
                            if (seen0) o[nt][u][0] = o[nt][u][2] = __int_as_float(0x7fffffff);
                            if (seen1) o[nt][u][1] = o[nt][u][3] = __int_as_float(0x7fffffff);
                        }
                    }
                    e[h][nt][0] = e[h][nt][1] = e[h][nt][2] = e[h][nt][3] = 0.f;
                }
            }
        }
        uint32_t pf[2][NT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                pf[h][nt][0] = movmatrix_trans(pack_f16(e[h][nt][0], e[h][nt][1]));
                pf[h][nt][1] = movmatrix_trans(pack_f16(e[h][nt][2], e[h][nt][3]));
            }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < G::VW; ++c)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint32_t sel = s ? 0x7362 : 0x5140;
                    uint32_t a0, a1, a2, a3;
                    widen<CODE>(__byte_perm(w[h][0][c], w[h][1][c], sel), a0, a1);
                    widen<CODE>(__byte_perm(w[h][2][c], w[h][3][c], sel), a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][2 * c + s], a0, a1, a2, a3, pf[h][nt][0], pf[h][nt][1]);
                }
        __syncwarp();
        if (ahead < tiles) {
            fetch(ahead, stage);
            ahead += kSplitWarps;
            ++fetched;
        }
    }
    if (!ok)  // status bit 0 is set; wait (bounded) for the copies that are still under way
        for (int b = used; b < used + G::STAGES; ++b)
            if (b < fetched) mbar_wait_limited(&bars[b % G::STAGES], (uint32_t)((b / G::STAGES) & 1), p.status);
    if (MODE == kPlain || stop >= (int)end) break;
    // the next pages, once every warp is done with these
    __syncthreads();
    open_segment(stop);
    load_pages();
    __syncthreads();
    tiles = ok ? (stop - seg + 31) >> 5 : 0;  // a warp whose wait expired does no more
    ahead = warp;
    for (int s = 0; s < G::STAGES && ahead < tiles; ++s, ahead += kSplitWarps, ++fetched)
        fetch(ahead, (used + s) % G::STAGES);
    any_small = load_scales();
    const bool now_small = __syncthreads_or(any_small) || small;
    if (now_small) {
        for (int e = tid; e < entries; e += kSplitThreads) to_small(scales[e]);
        if (!small) {  // the sums so far in the smaller unit
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                l[nt][0] *= SmallScales::factor;
                l[nt][1] *= SmallScales::factor;
            }
        }
        __syncthreads();
    }
    small = now_small;
    }

    griddep_launch_dependents();  // the joining kernel's CTAs may take their places and wait for this grid
    // join the warps: rows' m and l, then O, through the ring's memory
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
            l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
            l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
        }
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = nt * 8 + 2 * q4 + j;
            float* dst = part_o + (warp * G::ROWS + r) * dim;
#pragma unroll
            for (int c = 0; c < G::VW; ++c) {
                const int d = DP == 64 ? 8 * g + 4 * c : 128 * (c >> 2) + 16 * g + 4 * (c & 3);
                if (EXACT || d < dim)
                    *reinterpret_cast<float4*>(dst + d) = make_float4(o[nt][2 * c][j], o[nt][2 * c][2 + j],
                                                                      o[nt][2 * c + 1][j], o[nt][2 * c + 1][2 + j]);
            }
            if (g == 0) {
                part_ml[(warp * G::ROWS + r) * 2] = m[nt][j];
                part_ml[(warp * G::ROWS + r) * 2 + 1] = l[nt][j];
            }
        }
    __syncthreads();
    for (int e = tid; e < rows * (dim / 4); e += kSplitThreads) {
        const int r = e / (dim / 4), d = (e - r * (dim / 4)) * 4;
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) top = fmaxf(top, part_ml[(w * G::ROWS + r) * 2]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) {
            const float mw = part_ml[(w * G::ROWS + r) * 2];
            const float f = mw == -INFINITY ? (top == -INFINITY ? 1.f : 0.f) : exp2_approx(mw - top);
            const float4 x = *reinterpret_cast<const float4*>(part_o + (w * G::ROWS + r) * dim + d);
            sum += part_ml[(w * G::ROWS + r) * 2 + 1] * f;
            v.x += x.x * f;
            v.y += x.y * f;
            v.z += x.z * f;
            v.w += x.w * f;
        }
        if (small) {
            v.x *= SmallScales::factor;
            v.y *= SmallScales::factor;
            v.z *= SmallScales::factor;
            v.w *= SmallScales::factor;
            top += SmallScales::shift;
        }
        int64_t token;
        int head;
        row_of(r, token, head);
        if (p.cluster) {
            *reinterpret_cast<float4*>(cta_o + r * dim + d) = v;
            if (d == 0) {
                cta_ml[r * 2] = top;
                cta_ml[r * 2 + 1] = sum;
            }
        } else if (MODE == kGroups ? !direct : p.chunks > 1) {
            const int64_t at_part = MODE == kGroups ? (int64_t)blockIdx.x * G::ROWS + r
                                                    : (token * a.q_heads + head) * p.chunks + chunk;
            *reinterpret_cast<float4*>(p.parts + at_part * dim + d) = v;
            if (d == 0) {
                p.stats[at_part * 2] = top;
                p.stats[at_part * 2 + 1] = sum;
            }
        } else {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            T* y = static_cast<T*>(a.out) + token * a.ot + head * a.oh + d;
            y[0] = from_f32<T>(v.x * inv);
            y[1] = from_f32<T>(v.y * inv);
            y[2] = from_f32<T>(v.z * inv);
            y[3] = from_f32<T>(v.w * inv);
            if (d == 0 && a.lse)
                a.lse[token * a.q_heads + head] =
                    sum == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) + log2f(sum)) * 0.693147180559945309f;
        }
    }
    }
    if (!p.cluster) return;
    // the chunks' parts, each CTA a share of the tile's elements
    __syncthreads();
    cluster_sync();
    for (int e = tid + chunk * kSplitThreads; e < rows * (dim / 4); e += p.chunks * kSplitThreads) {
        const int r = e / (dim / 4), d = (e - r * (dim / 4)) * 4;
        float top = -INFINITY, sum = 0.f;
        float2 ml[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            ml[c] = c < p.chunks ? cluster_load2(cluster_address(cta_ml + r * 2, c)) : make_float2(-INFINITY, 0.f);
            top = fmaxf(top, ml[c].x);
        }
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            if (ml[c].y == 0.f) continue;  // nothing seen there, and no part
            const float f = ml[c].x == -INFINITY ? 1.f : exp2_approx(ml[c].x - top);
            const float4 x = cluster_load4(cluster_address(cta_o + r * dim + d, c));
            sum += ml[c].y * f;
            v.x += x.x * f;
            v.y += x.y * f;
            v.z += x.z * f;
            v.w += x.w * f;
        }
        int64_t token;
        int head;
        row_of(r, token, head);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T* y = static_cast<T*>(a.out) + token * a.ot + head * a.oh + d;
        y[0] = from_f32<T>(v.x * inv);
        y[1] = from_f32<T>(v.y * inv);
        y[2] = from_f32<T>(v.z * inv);
        y[3] = from_f32<T>(v.w * inv);
        if (d == 0 && a.lse)
            a.lse[token * a.q_heads + head] =
                sum == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) + log2f(sum)) * 0.693147180559945309f;
    }
    __syncthreads();
    cluster_sync();  // no CTA leaves while another reads its part
}

// Joins the chunks of a (row, head): a CTA each, its warps over the chunks, lanes
// over the dimensions.  A chunk in which the row saw nothing has l = 0 and no part.
// Bound by the latency of the parts' loads: 16 warps where there are many chunks (64
// rows of 103 chunks: 18.9 us with four).
constexpr int kJoinRun = 512;

template <typename T, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) k_attention_join(SplitArgs p) {
    __shared__ float weight[kJoinRun];
    __shared__ float red[2][WARPS];
    __shared__ float4 acc_s[WARPS][64];
    const AttentionArgs& a = p.a;
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dim = a.cache.dim;
    const int64_t i = blockIdx.x;
    const int64_t token = i / a.q_heads;
    const int head = (int)(i - token * a.q_heads);
    const int rows_from = a.seq.starts[0], rows_to = a.seq.starts[a.seq.seqs];
    if (token < rows_from || token >= rows_to) return;  // no sequence's row: it stays as it is
    const float2* st = reinterpret_cast<const float2*>(p.stats) + i * p.chunks;
    const float* parts = p.parts + i * p.chunks * dim;
    float top = -INFINITY;
    for (int c = tid; c < p.chunks; c += WARPS * 32) top = fmaxf(top, st[c].x);
#pragma unroll
    for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    if (lane == 0) red[0][warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, red[0][w]);
    float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    float sum = 0.f;
    for (int c0 = 0; c0 < p.chunks; c0 += kJoinRun) {
        const int n = min(kJoinRun, p.chunks - c0);
        __syncthreads();
        for (int c = tid; c < n; c += WARPS * 32) {
            const float2 v = st[c0 + c];
            // a NaN sum without a maximum keeps its weight: the row is NaN
            const float f = v.y == 0.f ? 0.f : v.x == -INFINITY ? 1.f : exp2_approx(v.x - top);
            weight[c] = f;
            sum += v.y * f;
        }
        __syncthreads();
#pragma unroll 8
        for (int c = warp; c < n; c += WARPS) {
            const float f = weight[c];
            const float4* o = reinterpret_cast<const float4*>(parts + (int64_t)(c0 + c) * dim);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (f != 0.f && (k * 32 + lane) * 4 < dim) {
                    const float4 x = o[k * 32 + lane];
                    acc[k].x += x.x * f;
                    acc[k].y += x.y * f;
                    acc[k].z += x.z * f;
                    acc[k].w += x.w * f;
                }
        }
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
    if (lane == 0) red[1][warp] = sum;
#pragma unroll
    for (int k = 0; k < 2; ++k) acc_s[warp][k * 32 + lane] = acc[k];
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) sum += red[1][w];
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* y = static_cast<T*>(a.out) + token * a.ot + head * a.oh;
    for (int d = tid; d < dim; d += WARPS * 32) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += reinterpret_cast<const float*>(acc_s[w])[d];
        y[d] = from_f32<T>(v * inv);
    }
    if (a.lse && tid == 0)
        a.lse[i] = sum == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) + log2f(sum)) * 0.693147180559945309f;
}

// Joins the parts of a call with groups: a CTA a (token, kv head), a warp a head in turn,
// lanes over the dimensions.  The parts of a token are those of its own row tile's items
// and of its group's.  What the places say is checked against the parts that there are:
// with tables that contradict themselves it may be anything.
constexpr int kJoinWarps = 4;  // (8 where a kv head has more than 4 heads)

struct JoinSet {
    const float *parts, *stats;
    const int4* place;
    int rows;        // of a tile
    int64_t blocks;  // item * kv_heads + head at most
};
struct JoinArgs {
    AttentionArgs a;
    JoinSet set[2];  // own tokens, prefixes
};

// Q: float4 of a row in a lane.  BATCH: parts in flight together, eight where there are few
// rows, as each waits for memory a few times over; four where there are many, for more CTAs
// on an SM (3696 CTAs of 8 warps: 42 us with 97 registers a thread).
template <typename T, int Q, int BATCH>
__global__ void __launch_bounds__(2 * kJoinWarps * 32, BATCH == 8 || Q == 2 ? 2 : 5) k_attention_join_items(JoinArgs p) {
    const AttentionArgs& a = p.a;
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, dim = a.cache.dim, kv_heads = a.cache.kv_heads;
    const int token = (int)(blockIdx.x / (unsigned)kv_heads), kv = (int)blockIdx.x - token * kv_heads;
    int4 at[2] = {p.set[0].place[token], p.set[1].place[token]};
    const int rows_from = a.seq.starts[0], rows_to = a.seq.starts[a.seq.seqs];
    if (token < rows_from || token >= rows_to || (at[0].w & kPlaceDone)) return;  // no sequence's row, or written
    if (!(at[0].w & kPlacePrefix)) at[1].y = 0;
    for (int h = warp; h < a.group; h += (int)(blockDim.x >> 5)) {
        int64_t first[2], step[2];  // row of the first piece's part, rows to the next
        int n[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const JoinSet& s = p.set[k];
            const int r = at[k].z + h, part = r / s.rows;
            const int64_t item = (int64_t)at[k].x + (int64_t)part * at[k].y;
            const bool fits = at[k].x >= 0 && at[k].y >= 0 && at[k].z >= 0 && at[k].z <= 255 &&
                              (item + at[k].y) * kv_heads <= s.blocks;
            n[k] = fits ? at[k].y : 0;
            first[k] = (item * kv_heads + kv) * s.rows + (r - part * s.rows);
            step[k] = (int64_t)kv_heads * s.rows;
        }
        const int all = n[0] + n[1];
        auto row_of = [&](int c) { return c < n[0] ? first[0] + c * step[0] : first[1] + (c - n[0]) * step[1]; };
        auto stat = [&](int c, int64_t row) {
            return reinterpret_cast<const float2*>(c < n[0] ? p.set[0].stats : p.set[1].stats)[row];
        };
        int64_t row = lane < all ? row_of(lane) : 0;  // of piece `lane`, then of those 32 behind
        float2 v = lane < all ? stat(lane, row) : make_float2(-INFINITY, 0.f);
        float top = v.x;
        for (int c = lane + 32; c < all; c += 32) top = fmaxf(top, stat(c, row_of(c)).x);
#pragma unroll
        for (int w = 16; w; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        float4 acc[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q) acc[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll 1
        for (int c0 = 0; c0 < all; c0 += 32) {
            const int c = c0 + lane;
            if (c0 && c < all) {
                row = row_of(c);
                v = stat(c, row);
            }
            // a NaN sum without a maximum keeps its weight: the row is NaN
            const float f = c >= all || v.y == 0.f ? 0.f : v.x == -INFINITY ? 1.f : exp2_approx(v.x - top);
            if (c < all) sum += v.y * f;
            const float* part = (c < n[0] ? p.set[0].parts : p.set[1].parts) + row * dim;
            // those that count, a batch in flight together (0 times what was not written may be NaN)
            unsigned left = __ballot_sync(0xffffffffu, f != 0.f);
            while (left) {
                float4 x[BATCH][Q];
                float g[BATCH];
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    g[j] = 0.f;
                    if (left) {
                        const int from = __ffs(left) - 1;
                        left &= left - 1;
                        g[j] = __shfl_sync(0xffffffffu, f, from);
                        const float4* o = reinterpret_cast<const float4*>(
                            __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(part), from));
#pragma unroll
                        for (int q = 0; q < Q; ++q)
                            if ((q * 32 + lane) * 4 < dim) x[j][q] = o[q * 32 + lane];
                    }
                }
#pragma unroll
                for (int j = 0; j < BATCH; ++j)
                    if (g[j] != 0.f)
#pragma unroll
                        for (int q = 0; q < Q; ++q) {
                            acc[q].x += x[j][q].x * g[j];
                            acc[q].y += x[j][q].y * g[j];
                            acc[q].z += x[j][q].z * g[j];
                            acc[q].w += x[j][q].w * g[j];
                        }
            }
        }
#pragma unroll
        for (int w = 16; w; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int head = kv * a.group + h;
        T* y = static_cast<T*>(a.out) + token * a.ot + head * a.oh;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int d = (q * 32 + lane) * 4;
            if (d < dim) {
                Pack<T, 4> w;
                w.v[0] = from_f32<T>(acc[q].x * inv);
                w.v[1] = from_f32<T>(acc[q].y * inv);
                w.v[2] = from_f32<T>(acc[q].z * inv);
                w.v[3] = from_f32<T>(acc[q].w * inv);
                if (a.o_packs) {
                    *reinterpret_cast<Pack<T, 4>*>(y + d) = w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) y[d + k] = w.v[k];
                }
            }
        }
        if (a.lse && lane == 0)
            a.lse[(int64_t)token * a.q_heads + head] =
                sum == 0.f ? -INFINITY : ((top == -INFINITY ? 0.f : top) + log2f(sum)) * 0.693147180559945309f;
    }
}

}  // namespace bfft
