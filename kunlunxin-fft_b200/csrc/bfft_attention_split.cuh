// bfft_attention_split.cuh -- attention of few query rows over a long axis of
// 8-bit tokens (single tokens, drafted tokens).  Included by bfft_attention.cu.
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
// 64 sequences of 1024..32768 tokens, one row of 32 heads each (8 kv heads, 128
// dimensions): int8 417 us, 5440 GB/s, 0.83 of the measured HBM rate (417 to 455, 0.76,
// on the GPUs that it was measured on; a GPU repeats itself within 1 %); e4m3, whose
// codes take 2 instructions for 4 to widen instead of 5, 386 us and 0.90.  One
// sequence of 131001 e4m3 tokens, 64 heads: 55 us, the joining kernel's among them.
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
    int entries;         // pages that a chunk can touch
    unsigned int* status;
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

template <int DP, bool EXACT, int NT, typename T, int CODE>
__global__ void __launch_bounds__(kSplitThreads, NT == 1 && DP <= 128 ? 3 : 2)
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
    const int chunk = (int)(i % p.chunks);
    i /= p.chunks;
    const int kv = (int)(i % a.cache.kv_heads);
    i /= a.cache.kv_heads;
    const int part = (int)(i % p.token_tiles);
    const int64_t slot = i / p.token_tiles;
    if (tid == 0) {
        for (int b = 0; b < kSplitWarps * G::STAGES; ++b) mbar_init(&full[b], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    SlotRows sr;
    if (!slot_rows(a.seq, slot, p.tile_tokens, p.by_token, sr)) return;
    const int head0 = part * G::ROWS;                       // of the group, where a token takes several tiles
    const int per_token = p.token_tiles > 1 ? min(a.group - head0, G::ROWS) : a.group;
    const int rows = sr.n * per_token;
    int64_t len = a.seq.lens[sr.s];
    const int64_t most = (int64_t)a.seq.max_pages << a.cache.page_log2;
    if (len > most) len = most;
    const int64_t pos0 = (int64_t)a.seq.lens[sr.s] - sr.rows + sr.place;
    int64_t lo_min, hi_max, lo_max, hi_min;
    seen_range(a, pos0, len, lo_min, hi_min);
    seen_range(a, pos0 + sr.n - 1, len, lo_max, hi_max);
    const int64_t base = (lo_min & ~(int64_t)15) + (int64_t)chunk * p.chunk;
    int64_t end = base + p.chunk;
    if (end > hi_max) end = hi_max;
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
            } else if (p.chunks > 1) {
                float* st = p.stats + ((token * a.q_heads + head) * p.chunks + chunk) * 2;
                st[0] = -INFINITY;
                st[1] = 0.f;
            } else if (a.lse) {
                a.lse[token * a.q_heads + head] = -INFINITY;
            }
        }
        if (p.chunks == 1)
            for (int e = tid; e < rows * dim; e += kSplitThreads) {
                int64_t token;
                int head;
                row_of(e / dim, token, head);
                static_cast<T*>(a.out)[token * a.ot + head * a.oh + e % dim] = from_f32<T>(0.f);
            }
        if (!p.cluster) return;
    } else {
    // from here on tokens are counted from `base`, in 32 bits
    const int lg = a.cache.page_log2;
    const int64_t page0 = base >> lg;
    const int off = (int)(base & (((int64_t)1 << lg) - 1)), span = (int)(end - base);
    const int entries = ((off + span - 1) >> lg) + 1;
    auto rel = [&](int64_t t) { return (int)(t < base ? 0 : t - base > span ? span : t - base); };
    const int lo_all = rel(lo_max), hi_all = rel(hi_min), lo_any = rel(lo_min);
    for (int e = tid; e < entries; e += kSplitThreads) {
        const int64_t id = a.seq.block_table[sr.s * a.seq.table_stride + page0 + e];
        page_ids[e] = id >= 0 && id < a.cache.pages ? (int)id : -1;
    }
    __syncthreads();

    // ring: tile t of this warp covers tokens [base + 32 (t kSplitWarps + warp), + 32)
    const int tiles = (span + 31) >> 5;
    unsigned char* mine = ring + warp * (G::STAGES * 4 * G::half_bytes(dim));
    uint64_t* bars = full + warp * G::STAGES;
    const int lines = EXACT ? DP / 8 : 1;  // 128-byte lines of 16 tokens
    auto fetch = [&](int t, int stage) {   // lanes 0..3: keys of half 0, 1, values of half 0, 1
        const int tok = t * 32 + (lane & 1) * 16;
        int id = -1;
        if (lane < 4 && tok < span) id = page_ids[(off + tok) >> lg];
        const unsigned any = __ballot_sync(0xffffffffu, id >= 0);
        if (lane == 0) mbar_arrive_expect_tx(&bars[stage], (uint32_t)(__popc(any) * G::half_bytes(dim)));
        __syncwarp();
        if (id >= 0) {
            unsigned char* dst = mine + (stage * 4 + lane) * G::half_bytes(dim);
            const int slot_in = (off + tok) & ((1 << lg) - 1);
            if constexpr (EXACT) {
                tma_load_3d(dst, lane < 2 ? &kmap : &vmap, 0, ((kv << lg) + slot_in) / 16 * lines, id, &bars[stage]);
            } else {
                const uint8_t* src = (lane < 2 ? a.cache.k : a.cache.v) +
                                     ((((int64_t)id * a.cache.kv_heads + kv) << lg) + slot_in) * dim;
                bulk_load(dst, src, (uint32_t)G::half_bytes(dim), &bars[stage]);
            }
        }
    };
    int ahead = warp;  // next tile to fetch
    for (int s = 0; s < G::STAGES && ahead < tiles; ++s, ahead += kSplitWarps) fetch(ahead, s);
    bool any_small = false;
    for (int e = tid; e < entries; e += kSplitThreads) {
        const int id = page_ids[e];
        if (id >= 0) {
            const int64_t b = (int64_t)id * a.cache.kv_heads + kv;
            scales[e] = block_scale(a.cache.k_scale[b], a.cache.v_scale[b]);
            any_small |= small_scale(scales[e]);
        } else {
            scales[e].kind = kDeadBlock;
        }
    }

    // queries as B fragments: lane (g, q4) holds row g of each 8-row tile, dims 16 (4 i + q4) + 4 t ..
    uint32_t qf[NT][G::KS][2];
    float row_scale[NT][2];      // of rows 2 q4, 2 q4 + 1: softmax scale (log2) times the row's power
    int row_lo[NT][2], row_hi[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 8 + g;
        float big = 0.f;
        const T* x = nullptr;
        if (r < rows) {
            int64_t token;
            int head;
            row_of(r, token, head);
            x = static_cast<const T*>(a.q) + token * a.qt + head * a.qh;
        }
        float e[G::KS][4];
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int d = 16 * (4 * (ks >> 2) + q4) + 4 * (ks & 3) + j;
                e[ks][j] = x && (EXACT || d < dim) ? to_f32(x[d]) : 0.f;
                big = fmaxf(big, fabsf(e[ks][j]));
            }
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
            int64_t lo, hi;
            seen_range(a, pos0 + (rr < rows ? rr / per_token : 0), len, lo, hi);
            row_lo[nt][j] = rel(lo);
            row_hi[nt][j] = rel(hi);
        }
    }
    const bool small = __syncthreads_or(any_small);  // a small value scale in the chunk
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
    int it = 0;
    for (int t = warp; t < tiles; t += kSplitWarps, ++it) {
        const int stage = it % G::STAGES;
        ok = mbar_wait_limited(&bars[stage], (uint32_t)((it / G::STAGES) & 1), p.status);
        if (__any_sync(0xffffffffu, !ok)) {
            ok = false;
            break;
        }
        const int tok0 = t * 32;
        const unsigned char* buf = mine + stage * 4 * G::half_bytes(dim);
        float z[2][NT][4];
        BlockScale bs[2];
        bool live[2];
        float worst = -INFINITY;  // largest z - m of this lane
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int tok = tok0 + 16 * h;
            const int e = (off + tok) >> lg;
            bs[h] = scales[e < entries ? e : entries - 1];
            live[h] = tok < span && bs[h].kind != kDeadBlock;
            if (!live[h]) continue;
            const unsigned char* kb = buf + h * G::half_bytes(dim);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) z[h][nt][0] = z[h][nt][1] = z[h][nt][2] = z[h][nt][3] = 0.f;
#pragma unroll
            for (int c = 0; c < (DP + 63) / 64; ++c) {
                uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
                const int col = 16 * (4 * c + q4);
                if (EXACT || col < dim) {
                    w0 = *reinterpret_cast<const uint4*>(kb + at(tk * dim + col));
                    w1 = *reinterpret_cast<const uint4*>(kb + at((tk + 8) * dim + col));
                }
                const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint32_t a0, a1, a2, a3;
                    widen<CODE>(u0[s], a0, a2);
                    widen<CODE>(u1[s], a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma_f16(z[h][nt], a0, a1, a2, a3, qf[nt][c * 4 + s][0], qf[nt][c * 4 + s][1]);
                }
            }
            const bool inside = tok >= lo_all && tok + 16 <= hi_all;  // hi_all is at most span
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float v = z[h][nt][c] * (bs[h].key * row_scale[nt][c & 1]) + bs[h].log2_value;
                    if (!inside) {
                        const int j = tok + tk + (c >> 1) * 8;
                        if (j < row_lo[nt][c & 1] || j >= row_hi[nt][c & 1]) v = -INFINITY;
                    }
                    z[h][nt][c] = v;
                    worst = fmaxf(worst, v == -INFINITY ? v : v - m[nt][c & 1]);
                }
        }
        if (__any_sync(0xffffffffu, worst > kRenew)) {  // a score far over a reference (or the first one): renew them
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float top = -INFINITY;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (live[h]) top = fmaxf(top, fmaxf(z[h][nt][j], z[h][nt][2 + j]));
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
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (!live[h]) continue;
            const int tok = tok0 + 16 * h;
            uint32_t pf[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
                float e0 = exp2_approx(z[h][nt][0] - m0), e1 = exp2_approx(z[h][nt][1] - m1);
                float e2 = exp2_approx(z[h][nt][2] - m0), e3 = exp2_approx(z[h][nt][3] - m1);
                l[nt][0] += (e0 + e2) * bs[h].inv_value;
                l[nt][1] += (e1 + e3) * bs[h].inv_value;
                if (bs[h].kind) {
                    if (bs[h].kind == 2) {  // values that are not finite spoil the rows that see one of them
                        int seen0 = z[h][nt][0] != -INFINITY || z[h][nt][2] != -INFINITY;
                        int seen1 = z[h][nt][1] != -INFINITY || z[h][nt][3] != -INFINITY;
#pragma unroll
                        for (int w = 4; w < 32; w <<= 1) {
                            seen0 |= __shfl_xor_sync(0xffffffffu, seen0, w);
                            seen1 |= __shfl_xor_sync(0xffffffffu, seen1, w);
                        }
#pragma unroll
                        for (int u = 0; u < 2 * G::VW; ++u) {
                            if (seen0) o[nt][u][0] = o[nt][u][2] = __int_as_float(0x7fffffff);
                            if (seen1) o[nt][u][1] = o[nt][u][3] = __int_as_float(0x7fffffff);
                        }
                    }
                    e0 = e1 = e2 = e3 = 0.f;
                }
                pf[nt][0] = movmatrix_trans(pack_f16(e0, e1));
                pf[nt][1] = movmatrix_trans(pack_f16(e2, e3));
            }
            // values: tokens t0, t1, t0 + 8, t1 + 8 of this lane, dims 4 w .. 4 w + 3 of its columns
            const unsigned char* vb = buf + (2 + h) * G::half_bytes(dim);
            const int t0 = row_token(2 * q4), t1 = row_token(2 * q4 + 1);
            const int toks[4] = {t0, t1, t0 + 8, t1 + 8};
            uint32_t w[4][G::VW];
            const bool whole = tok >= lo_any && tok + 16 <= span;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (DP == 64) {
                    uint2 x = make_uint2(0, 0);
                    if (EXACT || 8 * g < dim) x = *reinterpret_cast<const uint2*>(vb + at(toks[k] * dim + 8 * g));
                    w[k][0] = x.x;
                    w[k][1] = x.y;
                } else {
#pragma unroll
                    for (int c = 0; c < DP / 128; ++c) {
                        uint4 x = make_uint4(0, 0, 0, 0);
                        const int col = 16 * g + 128 * c;
                        if (EXACT || col < dim) x = *reinterpret_cast<const uint4*>(vb + at(toks[k] * dim + col));
                        w[k][4 * c] = x.x;
                        w[k][4 * c + 1] = x.y;
                        w[k][4 * c + 2] = x.z;
                        w[k][4 * c + 3] = x.w;
                    }
                }
                if (!whole) {  // codes of slots that no row sees may be anything: 0 times NaN is NaN
                    const int j = tok + toks[k];
                    if (j < lo_any || j >= span)
#pragma unroll
                        for (int c = 0; c < G::VW; ++c) w[k][c] = 0;
                }
            }
#pragma unroll
            for (int c = 0; c < G::VW; ++c)
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const uint32_t sel = s ? 0x7362 : 0x5140;
                    uint32_t a0, a1, a2, a3;
                    widen<CODE>(__byte_perm(w[0][c], w[1][c], sel), a0, a1);
                    widen<CODE>(__byte_perm(w[2][c], w[3][c], sel), a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][2 * c + s], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
                }
        }
        __syncwarp();
        if (ahead < tiles) {
            fetch(ahead, stage);
            ahead += kSplitWarps;
        }
    }
    if (!ok)  // status bit 0 is set; wait (bounded) for the copies that are still under way
        for (int t = warp + kSplitWarps * it; t < ahead; t += kSplitWarps, ++it)
            mbar_wait_limited(&bars[it % G::STAGES], (uint32_t)((it / G::STAGES) & 1), p.status);

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
        } else if (p.chunks > 1) {
            const int64_t at_part = (token * a.q_heads + head) * p.chunks + chunk;
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

}  // namespace bfft
