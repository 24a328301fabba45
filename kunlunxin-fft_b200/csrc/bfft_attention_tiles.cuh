// bfft_attention_tiles.cuh -- attention of many query rows (a prompt's chunk) over
// 8-bit tokens on the tensor cores (tcgen05).  Included by bfft_attention.cu.
//
// A CTA takes up to 256 rows of one kv head (query tokens times the group's heads,
// so all of them share the keys) and walks the tokens in tiles of 128:
//
//   loader warp    bulk copies of the 8-bit blocks, one ring for keys and values
//                  in the order of their use, and the tile's block scales
//   2 warps        look for a small value scale among the chunk's while the first
//                  tile loads
//   4 warps        widen codes to float16 (exact) in the layout of the matrix
//                  instructions: [token][64 dims] panels, 128-byte swizzle.  Keys
//                  (K-major) and values (N-major) share it
//   one thread     S = Q_h K^T into tensor memory, O_h += P V with P read from
//                  tensor memory, h = the two 128-row halves in turn, so that one
//                  half's products run under the other's exponentials
//   2 x 4 warps    a row each: S -> P (float16, in S's place), the row's maximum
//                  and sum; the maximum is renewed, and O rescaled, only where a
//                  score passes it by the room that float16 leaves
//
// Key and value scales enter in the exponent as in the split kernel:
// p' = 2^(s * ks + log2 vs - m), sum of p' / vs; a chunk with a small value scale
// (SmallScales) holds its sums 2^36 times smaller: the loader writes its scales so,
// and the rows take it back at their end (a flag that the rows' loop looked at cost
// 2 % of the two-prompt case).
//
// 2 x 2048 prompt rows of 32 heads (8 kv heads, 128 dimensions) over 8192 and 16384
// int8 tokens: 860 us (854 to 882 by the GPU), 880 TFLOP/s, 0.54 of the measured bf16
// rate.  Bound by the chain of a half's tile, not by one pipe: 4900 clocks a tile for
// 2048 of tensor work; and by the schedule: 512 CTAs of 65 to 113 tiles in the order
// of their slots end at 372 tile times where an even spread would be 318 (counted).
// Leaving a stage out (in a copy) gives, of 880 us: no widening 782, no
// exponentials 872, no maximum 862, half of the value products 832.  The special
// function pipe is 46 % busy, so exponentials by polynomials did not help; tiles of
// 64 tokens with two score buffers a half were slower (an M128 N64 product takes as
// long as N128 when the widening shares its shared memory); waits that poll without
// reading the clock, 975 us.
#pragma once

namespace bfft {

struct TileArgs {
    AttentionArgs a;
    float* parts;      // as in SplitArgs
    float* stats;
    int chunk;         // tokens of a chunk, a multiple of 128
    int chunks;
    int tile_tokens;   // query tokens of a CTA
    int by_token;
    int64_t slots;
    unsigned int* status;
};

template <int DP>
struct TileGeo {
    static constexpr int THREADS = 512;
    // registers a thread, by warpgroup: rows (2), codes, loads and products: 2 * 184 + 72 + 72 = 4 * 128 of the launch
    static constexpr int ROW_REGS = 184, CODE_REGS = 72, OTHER_REGS = 72;
    static constexpr int N = 128;                 // tokens of a tile
    static constexpr int PANELS = DP / 64;        // of 64 dims = 128 bytes
    static constexpr int Q_PANEL = 128 * 128;     // bytes: 128 rows
    static constexpr int PANEL = N * 128;         // bytes: a tile's rows
    static constexpr int Q_HALF = PANELS * Q_PANEL;
    static constexpr int T_BUF = PANELS * PANEL;  // widened keys or values
    static constexpr int T_RING = 3;
    static constexpr int RAW_BUF = N * DP;
    static constexpr int RAW_RING = 4;
    static constexpr int SLOTS = 8;              // tiles whose block scales are held
    static constexpr int GROUPS = N / 16;         // of 16 tokens
    static constexpr int BODY = 2 * Q_HALF + T_RING * T_BUF + RAW_RING * RAW_BUF;
    static constexpr int BARS = 2 * RAW_RING + 2 * T_RING + SLOTS + 2 + 2 * 2 + 1 + 2 + 1;
    // at least half of an SM's shared memory: a second CTA could not have its tensor memory
    static constexpr int SMEM_NEED = 1024 + BODY + SLOTS * GROUPS * 16 + BARS * 8 + 8 + SLOTS * 4 + 4;
    static constexpr int SMEM = SMEM_NEED > 118 * 1024 ? SMEM_NEED : 118 * 1024;
    static constexpr uint32_t TMEM = 512;
    static constexpr uint32_t S0 = 0, O0 = 256;   // columns: S_h at 128 h, O_h at 256 + 128 h
};

// As kTop and kRenew: a renewal costs a row's O one trip through registers, so the
// maximum leaves room for scores 32 times larger.
constexpr float kTileTop = 10.f, kTileRenew = 15.5f;

__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Descriptor of an operand with 128-byte swizzle: the low word holds the address (in
// 16 bytes) and the leading offset, the high word, the same for every step, the stride
// of eight rows, the version and the layout.  A step along the operand adds to the
// low word: one thread issues the products (2 x 2048 prompt rows 881 us with 64-bit
// descriptors built anew for each, 856 so on that GPU).
__device__ __forceinline__ uint32_t desc_low(uint32_t addr, uint32_t lbo) { return (addr >> 4) | ((lbo >> 4) << 16); }
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
// float16 operands, float32 accumulator, M = 128
__host__ __device__ constexpr uint32_t tile_idesc(int n, bool b_n_major) {
    return (1u << 4) | (b_n_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHigh)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}

// 32 columns of this warp's 32 rows, a row per lane; d holds them after tmem_arrived.
__device__ __forceinline__ void tmem_fetch(uint32_t addr, uint32_t* d) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]), "=r"(d[4]), "=r"(d[5]), "=r"(d[6]), "=r"(d[7]),
          "=r"(d[8]), "=r"(d[9]), "=r"(d[10]), "=r"(d[11]), "=r"(d[12]), "=r"(d[13]), "=r"(d[14]),
          "=r"(d[15]), "=r"(d[16]), "=r"(d[17]), "=r"(d[18]), "=r"(d[19]), "=r"(d[20]), "=r"(d[21]),
          "=r"(d[22]), "=r"(d[23]), "=r"(d[24]), "=r"(d[25]), "=r"(d[26]), "=r"(d[27]), "=r"(d[28]),
          "=r"(d[29]), "=r"(d[30]), "=r"(d[31])
        : "r"(addr)
        : "memory");
}
// Waits for this warp's fetches; naming d keeps its uses behind the wait.
__device__ __forceinline__ void tmem_arrived(uint32_t* d) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]), "+r"(d[4]), "+r"(d[5]), "+r"(d[6]), "+r"(d[7]),
                   "+r"(d[8]), "+r"(d[9]), "+r"(d[10]), "+r"(d[11]), "+r"(d[12]), "+r"(d[13]), "+r"(d[14]),
                   "+r"(d[15]), "+r"(d[16]), "+r"(d[17]), "+r"(d[18]), "+r"(d[19]), "+r"(d[20]), "+r"(d[21]),
                   "+r"(d[22]), "+r"(d[23]), "+r"(d[24]), "+r"(d[25]), "+r"(d[26]), "+r"(d[27]), "+r"(d[28]),
                   "+r"(d[29]), "+r"(d[30]), "+r"(d[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t addr, uint32_t (&d)[32]) {
    tmem_fetch(addr, d);
    tmem_arrived(d);
}
__device__ __forceinline__ void tmem_store(uint32_t addr, const uint32_t* d) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
        "r"(d[0]), "r"(d[1]), "r"(d[2]), "r"(d[3]), "r"(d[4]), "r"(d[5]), "r"(d[6]), "r"(d[7]), "r"(d[8]), "r"(d[9]),
        "r"(d[10]), "r"(d[11]), "r"(d[12]), "r"(d[13]), "r"(d[14]), "r"(d[15]), "r"(d[16]), "r"(d[17]), "r"(d[18]),
        "r"(d[19]), "r"(d[20]), "r"(d[21]), "r"(d[22]), "r"(d[23]), "r"(d[24]), "r"(d[25]), "r"(d[26]), "r"(d[27]),
        "r"(d[28]), "r"(d[29]), "r"(d[30]), "r"(d[31])
        : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&d)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(addr),
        "r"(d[0]), "r"(d[1]), "r"(d[2]), "r"(d[3]), "r"(d[4]), "r"(d[5]), "r"(d[6]), "r"(d[7]), "r"(d[8]), "r"(d[9]),
        "r"(d[10]), "r"(d[11]), "r"(d[12]), "r"(d[13]), "r"(d[14]), "r"(d[15])
        : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t addr, const uint32_t (&d)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(d[0]),
                 "r"(d[1]), "r"(d[2]), "r"(d[3]), "r"(d[4]), "r"(d[5]), "r"(d[6]), "r"(d[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t addr, uint32_t (&d)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];\n tcgen05.wait::ld.sync.aligned;"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]), "=r"(d[4]), "=r"(d[5]), "=r"(d[6]), "=r"(d[7]), "=r"(d[8]),
          "=r"(d[9]), "=r"(d[10]), "=r"(d[11]), "=r"(d[12]), "=r"(d[13]), "=r"(d[14]), "=r"(d[15])
        : "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int DP, typename T, int CODE>
__global__ void __launch_bounds__(TileGeo<DP>::THREADS, 1) k_attention_tiles(TileArgs p) {
    using G = TileGeo<DP>;
    extern __shared__ unsigned char smem_raw[];
    const AttentionArgs& a = p.a;
    griddep_wait();
    const int dim = a.cache.dim, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, lg = a.cache.page_log2;

    // which rows and tokens
    int64_t i = blockIdx.x;
    const int chunk = (int)(i % p.chunks);
    i /= p.chunks;
    const int kv = (int)(i % a.cache.kv_heads);
    const int64_t slot = i / a.cache.kv_heads;
    SlotRows sr;
    if (!slot_rows(a.seq, slot, p.tile_tokens, p.by_token, sr)) return;
    const int rows = sr.n * a.group;
    int64_t len = a.seq.lens[sr.s];
    const int64_t most = (int64_t)a.seq.max_pages << lg;
    if (len > most) len = most;
    const int64_t pos0 = (int64_t)a.seq.lens[sr.s] - sr.rows + sr.place;
    int64_t lo_min, hi_max, lo_max, hi_min;
    seen_range(a, pos0, len, lo_min, hi_min);
    seen_range(a, pos0 + sr.n - 1, len, lo_max, hi_max);
    const int64_t base = (lo_min & ~(int64_t)127) + (int64_t)chunk * p.chunk;
    int64_t end = base + p.chunk;
    if (end > hi_max) end = hi_max;
    auto row_of = [&](int r, int64_t& token, int& head) {
        const int t = r / a.group;
        token = sr.first + t;
        head = kv * a.group + (r - t * a.group);
    };
    if (base >= end) {  // nothing of the axis in this chunk
        for (int r = tid; r < rows; r += G::THREADS) {
            int64_t token;
            int head;
            row_of(r, token, head);
            if (p.chunks > 1) {
                float* st = p.stats + ((token * a.q_heads + head) * p.chunks + chunk) * 2;
                st[0] = -INFINITY;
                st[1] = 0.f;
            } else if (a.lse) {
                a.lse[token * a.q_heads + head] = -INFINITY;
            }
        }
        if (p.chunks == 1)
            for (int e = tid; e < rows * dim; e += G::THREADS) {
                int64_t token;
                int head;
                row_of(e / dim, token, head);
                static_cast<T*>(a.out)[token * a.ot + head * a.oh + e % dim] = from_f32<T>(0.f);
            }
        return;
    }
    const int tiles = (int)((end - base + G::N - 1) / G::N);
    const int halves = rows > 128 ? 2 : 1;

    unsigned char* q_s = align_smem<1024>(smem_raw);
    unsigned char* t_s = q_s + 2 * G::Q_HALF;
    unsigned char* raw_s = t_s + G::T_RING * G::T_BUF;
    BlockScale* scale_s = reinterpret_cast<BlockScale*>(raw_s + G::RAW_RING * G::RAW_BUF);
    uint64_t* bars = reinterpret_cast<uint64_t*>(scale_s + G::SLOTS * G::GROUPS);
    uint64_t *raw_full = bars, *raw_empty = raw_full + G::RAW_RING, *t_full = raw_empty + G::RAW_RING,
             *t_empty = t_full + G::T_RING, *scale_full = t_empty + G::T_RING, *s_full = scale_full + G::SLOTS,
             *p_half = s_full + 2, *p_full = p_half + 2, *q_full = p_full + 2, *o_full = q_full + 1, *drained = o_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + G::BARS);
    int* tile_kind = reinterpret_cast<int*>(bars + G::BARS + 1);  // of a tile: 0 where all its blocks are ordinary
    volatile int* small_s = tile_kind + G::SLOTS;                 // whether the chunk has a small value scale
    if (warp == 13) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(G::TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int b = 0; b < G::RAW_RING; ++b) {
            mbar_init(&raw_full[b], 1);
            mbar_init(&raw_empty[b], 128);
        }
        for (int b = 0; b < G::T_RING; ++b) {
            mbar_init(&t_full[b], 128);
            mbar_init(&t_empty[b], 1);
        }
        for (int b = 0; b < G::SLOTS; ++b) mbar_init(&scale_full[b], 1);
        for (int h = 0; h < 2; ++h) {
            mbar_init(&s_full[h], 1);
            mbar_init(&p_half[h], 128);
            mbar_init(&p_full[h], 128);
            mbar_init(&o_full[h], 1);
        }
        mbar_init(q_full, 256);
        mbar_init(drained, 1);
        *small_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto wait = [&](uint64_t* b, uint32_t parity) { return mbar_wait_limited(b, parity, p.status); };

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::ROW_REGS));
        // ------------------------------------------------------------ rows
        const int h = warp >> 2, r = tid;  // row r of the CTA is row r - 128 h of half h
        const bool mine = r < rows;
        int64_t token = 0;
        int head = 0;
        if (mine) row_of(r, token, head);
        float up = 1.f;
        {
            const T* x = static_cast<const T*>(a.q) + token * a.qt + head * a.qh;
            float big = 0.f, down;
            Pack<T, 8> w[DP / 8];  // the whole row in flight at once
#pragma unroll
            for (int c = 0; c < DP / 8; ++c) {
                if (!mine || 8 * c >= dim) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) w[c].v[k] = from_f32<T>(0.f);
                } else if (a.q_packs) {
                    w[c] = *reinterpret_cast<const Pack<T, 8>*>(x + 8 * c);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) w[c].v[k] = x[8 * c + k];
                }
            }
#pragma unroll
            for (int c = 0; c < DP / 8; ++c)
#pragma unroll
                for (int k = 0; k < 8; ++k) big = fmaxf(big, fabsf(to_f32(w[c].v[k])));
            row_power<T>(big, down, up);
            unsigned char* q_row = q_s + h * G::Q_HALF + (r & 127) * 128;
#pragma unroll
            for (int c = 0; c < DP / 8; ++c) {
                uint32_t e[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) e[k] = pack_f16(to_f32(w[c].v[2 * k]) * down, to_f32(w[c].v[2 * k + 1]) * down);
                *reinterpret_cast<uint4*>(q_row + (c >> 3) * G::Q_PANEL + (((c & 7) ^ (r & 7)) << 4)) =
                    make_uint4(e[0], e[1], e[2], e[3]);
            }
            fence_proxy_async_smem();
            mbar_arrive(q_full);
        }
        const float row_scale = up * a.scale_log2;
        const bool ordinary = a.scale_log2 >= 0.f;  // the largest product is the largest score
        int64_t row_lo, row_hi;
        seen_range(a, pos0 + (mine ? r / a.group : 0), len, row_lo, row_hi);
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + G::S0 + h * 128 + lanes, o_addr = tmem + G::O0 + h * 128 + lanes;
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        if (h < halves) {
            for (int j = 0; j < tiles; ++j) {
                ok = wait(&scale_full[j % G::SLOTS], (uint32_t)((j / G::SLOTS) & 1));
                // what the tile needs besides its scores, before they are there
                const int64_t tok0 = base + (int64_t)j * G::N;
                const bool inside = tok0 >= lo_max && tok0 + G::N <= hi_min;
                const BlockScale* bs = scale_s + (j % G::SLOTS) * G::GROUPS;
                const bool plain = inside && ordinary && tile_kind[j % G::SLOTS] == 0;
                ok = ok && wait(&s_full[h], (uint32_t)(j & 1));
                if (__any_sync(0xffffffffu, !ok)) {
                    ok = false;
                    break;
                }
                tmem_fence_after();
                uint32_t s[G::N];
#pragma unroll
                for (int c = 0; c < G::N / 32; ++c) tmem_fetch(s_addr + c * 32, s + c * 32);
#pragma unroll
                for (int c = 0; c < G::N / 32; ++c) tmem_arrived(s + c * 32);
                float top = -INFINITY;
                if (plain) {
                    // the largest exponent, from the blocks' largest scores
#pragma unroll
                    for (int g = 0; g < G::GROUPS; ++g) {
                        float x[5];
#pragma unroll
                        for (int k = 0; k < 5; ++k)
                            x[k] = max3(__uint_as_float(s[g * 16 + 3 * k]), __uint_as_float(s[g * 16 + 3 * k + 1]),
                                        __uint_as_float(s[g * 16 + 3 * k + 2]));
                        const float big =
                            fmaxf(max3(x[0], x[1], x[2]), max3(x[3], x[4], __uint_as_float(s[g * 16 + 15])));
                        const float2 b = *reinterpret_cast<const float2*>(&bs[g]);
                        top = fmaxf(top, fmaf(big, b.x * row_scale, b.y));
                    }
                } else {
                    // exponents in the scores' place, -inf where the row does not see the token
                    const int64_t lo = row_lo - tok0, hi = row_hi - tok0;
#pragma unroll
                    for (int g = 0; g < G::GROUPS; ++g) {
                        const BlockScale b = bs[g];
                        const bool dead = b.kind == kDeadBlock;
                        const float f = b.key * row_scale;
#pragma unroll
                        for (int k = g * 16; k < g * 16 + 16; ++k) {
                            const float z = !dead && k >= lo && k < hi ? fmaf(__uint_as_float(s[k]), f, b.log2_value)
                                                                       : -INFINITY;
                            top = fmaxf(top, z);
                            s[k] = __float_as_uint(z);
                        }
                    }
                }
                const bool renew = top > (m == -INFINITY ? -INFINITY : m + kTileRenew);
                if (__any_sync(0xffffffffu, renew)) {
                    float f = 1.f;
                    if (renew) {
                        const float now = top - kTileTop;
                        if (m != -INFINITY) f = exp2_approx(m - now);
                        m = now;
                        l *= f;
                    }
                    if (j > 0) {
                        // this half's products up to tile j - 1 are complete: s_full of tile j follows them
#pragma unroll 1
                        for (int c = 0; c < DP / 32; ++c) {
                            uint32_t o[32];
                            tmem_load(o_addr + c * 32, o);
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            tmem_store(o_addr + c * 32, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m;
                // P goes over scores that are in registers.  The products over the first 64
                // tokens start under the other exponentials
                auto written = [&](uint64_t* bar) {
                    tmem_store_wait();
                    tmem_fence_before();
                    mbar_arrive(bar);
                };
                if (plain) {
#pragma unroll
                    for (int g = 0; g < G::GROUPS; ++g) {
                        uint32_t pr[8];
                        const float4 b = *reinterpret_cast<const float4*>(&bs[g]);
                        const unsigned long long f2 = pack2(make_float2(b.x * row_scale, b.x * row_scale));
                        const unsigned long long off2 = pack2(make_float2(b.y - ref, b.y - ref));
                        unsigned long long part[2] = {0, 0};
#pragma unroll
                        for (int k = g * 8; k < g * 8 + 8; ++k) {
                            unsigned long long z;
                            asm("mov.b64 %0, {%1, %2};" : "=l"(z) : "r"(s[2 * k]), "r"(s[2 * k + 1]));
                            asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(z) : "l"(f2), "l"(off2));
                            const float2 x = unpack2(z);
                            const float2 e = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(part[k & 1]) : "l"(pack2(e)));
                            pr[k - g * 8] = pack_f16(e.x, e.y);
                        }
                        const float2 u = unpack2(part[0]), v = unpack2(part[1]);
                        l = fmaf((u.x + u.y) + (v.x + v.y), b.z, l);
                        tmem_store8(s_addr + g * 8, pr);
                        if (g == 3) written(&p_half[h]);
                    }
                } else {
#pragma unroll
                    for (int g = 0; g < G::GROUPS; ++g) {
                        uint32_t pr[8];
                        const int kind = bs[g].kind;
                        float part = 0.f;
#pragma unroll
                        for (int k = g * 8; k < g * 8 + 8; ++k) {
                            float e[2];
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const float z = __uint_as_float(s[2 * k + x]);
                                e[x] = exp2_approx(z - ref);
                                part += e[x];
                                // values that do not count, or spoil the row
                                if (kind == 1) e[x] = 0.f;
                                if (kind == 2 && z != -INFINITY) e[x] = __int_as_float(0x7fffffff);
                            }
                            pr[k - g * 8] = pack_f16(e[0], e[1]);
                        }
                        l = fmaf(part, bs[g].inv_value, l);
                        tmem_store8(s_addr + g * 8, pr);
                        if (g == 3) written(&p_half[h]);
                    }
                }
                written(&p_full[h]);
            }
            if (ok) ok = !__any_sync(0xffffffffu, !wait(&o_full[h], 0));
            if (ok) {
                tmem_fence_after();
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const bool small = *small_s;
                if (small) m += SmallScales::shift;
                const int64_t at = ((token * a.q_heads + head) * p.chunks + chunk);
                T* y = static_cast<T*>(a.out) + token * a.ot + head * a.oh;
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) {
                    uint32_t o[32];
                    tmem_load(o_addr + c * 32, o);
                    if (!mine) continue;
                    if (small) {
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * SmallScales::factor);
                    }
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {
                        const int d = c * 32 + k;
                        if (d >= dim) continue;
                        if (p.chunks > 1) {
#pragma unroll
                            for (int x = 0; x < 8; x += 4)
                                *reinterpret_cast<uint4*>(p.parts + at * dim + d + x) =
                                    make_uint4(o[k + x], o[k + x + 1], o[k + x + 2], o[k + x + 3]);
                        } else {
                            Pack<T, 8> w;
#pragma unroll
                            for (int x = 0; x < 8; ++x) w.v[x] = from_f32<T>(__uint_as_float(o[k + x]) * inv);
                            if (a.o_packs) {
                                *reinterpret_cast<Pack<T, 8>*>(y + d) = w;
                            } else {
#pragma unroll
                                for (int x = 0; x < 8; ++x) y[d + x] = w.v[x];
                            }
                        }
                    }
                }
                if (mine) {
                    if (p.chunks > 1) {
                        p.stats[at * 2] = m;
                        p.stats[at * 2 + 1] = l;
                    } else if (a.lse) {
                        a.lse[token * a.q_heads + head] =
                            l == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m) + log2f(l)) * 0.693147180559945309f;
                    }
                }
            }
        }
    } else if (warp < 12) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::CODE_REGS));
        // ------------------------------------------------------------ codes to float16
        // a thread takes 16-code column c of rows row0, row0 + STEP, ...; the panel and
        // the swizzle of its two 16-byte stores are the same for all of them.  Lanes of
        // the odd panels store their second half first: eight lanes, eight banks
        const int t = tid - 256;
        constexpr int COLS = DP / 16, STEP = 128 / COLS, PER = G::N / STEP;
        const int c = t % COLS, row0 = t / COLS;
        const bool inside_head = 16 * c < dim, swap = (c >> 2) & 1;
        const uint32_t first = (uint32_t)((((2 * c) & 7) ^ (row0 & 7)) << 4), second = first ^ 16u;
        const uint32_t to0 = (uint32_t)((c >> 2) * G::PANEL + row0 * 128) + (swap ? second : first);
        const uint32_t to1 = (uint32_t)((c >> 2) * G::PANEL + row0 * 128) + (swap ? first : second);
        static_assert(STEP % 8 == 0, "rows of a thread share the swizzle");
        for (int n = 0; n < 2 * tiles; ++n) {
            const int rb = n % G::RAW_RING, tb = n % G::T_RING;
            const int j = n >> 1;
            const bool value = n & 1;
            bool ok = wait(&raw_full[rb], (uint32_t)((n / G::RAW_RING) & 1));
            uint4 w[PER];
            const unsigned char* src = raw_s + rb * G::RAW_BUF + row0 * dim + c * 16;
#pragma unroll
            for (int k = 0; k < PER; ++k)
                w[k] = inside_head ? *reinterpret_cast<const uint4*>(src + k * STEP * dim) : make_uint4(0, 0, 0, 0);
            if (value) {
                // codes that no row sees may be anything: as values they become zeros (0 times NaN is NaN)
                const int64_t tok0 = base + (int64_t)j * G::N;
                const BlockScale* bs = scale_s + (j % G::SLOTS) * G::GROUPS;
                const bool whole = tok0 >= lo_min && tok0 + G::N <= hi_max;
#pragma unroll
                for (int k = 0; k < PER; ++k) {
                    const int row = row0 + k * STEP;
                    bool keep = bs[row >> 4].kind != kDeadBlock;
                    if (!whole) keep = keep && tok0 + row >= lo_min && tok0 + row < hi_max;
                    if (!keep) w[k] = make_uint4(0, 0, 0, 0);
                }
            }
            mbar_arrive(&raw_empty[rb]);
            ok = ok && wait(&t_empty[tb], (uint32_t)(((n / G::T_RING) & 1) ^ 1));
            if (__any_sync(0xffffffffu, !ok)) break;
            unsigned char* dst = t_s + tb * G::T_BUF;
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                uint4 u, v;
                widen<CODE>(w[k].x, u.x, u.y);
                widen<CODE>(w[k].y, u.z, u.w);
                widen<CODE>(w[k].z, v.x, v.y);
                widen<CODE>(w[k].w, v.z, v.w);
                *reinterpret_cast<uint4*>(dst + to0 + k * STEP * 128) = swap ? v : u;
                *reinterpret_cast<uint4*>(dst + to1 + k * STEP * 128) = swap ? u : v;
            }
            fence_proxy_async_smem();
            mbar_arrive(&t_full[tb]);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::OTHER_REGS));
        if (warp == 12) {
        // ------------------------------------------------------------ loads
        const int unit = 1 << lg, blocks = G::N / unit, per = unit / 16;  // tokens of a copy, copies of a tile
        auto page_at = [&](int64_t tok) -> int {
            if (tok >= end || tok + 15 < lo_min) return -1;
            const int64_t id = a.seq.block_table[sr.s * a.seq.table_stride + (tok >> lg)];
            return id >= 0 && id < a.cache.pages ? (int)id : -1;
        };
        // lanes 0..7: the 16-token groups of a tile; page numbers three tiles ahead of the copies, scales two
        auto group_tok = [&](int j) { return base + (int64_t)j * G::N + (lane & 7) * 16; };
        auto scale_at = [&](int id, float& ks, float& vs) {
            ks = vs = 0.f;
            if (id >= 0) {
                const int64_t b = (int64_t)id * a.cache.kv_heads + kv;
                ks = a.cache.k_scale[b];
                vs = a.cache.v_scale[b];
            }
        };
        // the sources of a tile's copies: lane b < blocks copies tokens [b unit, + unit).  The first of its groups
        // that has a page names it: the others may lie before what is seen
        auto copies_of = [&](int j, int id, int64_t& src) -> unsigned {
            const unsigned groups = __ballot_sync(0xffffffffu, lane < G::GROUPS && id >= 0);
            const unsigned mask = ((1u << per) - 1u) << ((lane * per) & 31);
            const bool copy = lane < blocks && (groups & mask);
            const int page = __shfl_sync(0xffffffffu, id, copy ? __ffs(groups & mask) - 1 : 0);
            const int64_t tok = base + (int64_t)j * G::N + lane * unit;
            src = ((((int64_t)page * a.cache.kv_heads + kv) << lg) + (tok & (((int64_t)1 << lg) - 1))) * dim;
            return __ballot_sync(0xffffffffu, copy);
        };
        int id0 = page_at(group_tok(0)), id1 = page_at(group_tok(1)), id2 = page_at(group_tok(2));
        float ks0, vs0, ks1, vs1;
        scale_at(id0, ks0, vs0);
        scale_at(id1, ks1, vs1);
        int64_t src = 0;  // the tile's copies: of its keys, then of its values
        unsigned who = 0;
        bool ok = true;
        int n = 0;
        for (; n < 2 * tiles; ++n) {
            const int j = n >> 1, rb = n % G::RAW_RING;
            const bool value = n & 1;
            if (!value) who = copies_of(j, id0, src);
            ok = !__any_sync(0xffffffffu, !wait(&raw_empty[rb], (uint32_t)(((n / G::RAW_RING) & 1) ^ 1)));
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(&raw_full[rb], (uint32_t)(__popc(who) * unit * dim));
            __syncwarp();
            if ((who >> lane) & 1)
                bulk_load(raw_s + rb * G::RAW_BUF + lane * unit * dim, (value ? a.cache.v : a.cache.k) + src,
                          (uint32_t)(unit * dim), &raw_full[rb]);
            if (!value) {
                BlockScale b = block_scale(ks0, vs0);
                const bool any = __any_sync(0xffffffffu, lane < G::GROUPS && (id0 < 0 || !(ks0 >= 0.f) || b.kind != 0));
                if (id0 < 0) {
                    b.kind = kDeadBlock;
                    b.key = 0.f;
                }
                if (n == 0) asm volatile("barrier.cta.sync 1, 96;" ::: "memory");  // *small_s is known
                if (*small_s) to_small(b);
                if (lane < G::GROUPS) scale_s[(j % G::SLOTS) * G::GROUPS + lane] = b;
                if (lane == 0) tile_kind[j % G::SLOTS] = any;
                __syncwarp();
                if (lane == 0) mbar_arrive(&scale_full[j % G::SLOTS]);
                id0 = id1;
                id1 = id2;
                ks0 = ks1;
                vs0 = vs1;
                scale_at(id1, ks1, vs1);
                id2 = page_at(group_tok(j + 3));
            }
        }
        if (!ok)  // an expired wait has set the status bit; wait (bounded) for the copies under way
            for (int b = n > G::RAW_RING ? n - G::RAW_RING : 0; b < n; ++b)
                wait(&raw_full[b % G::RAW_RING], (uint32_t)((b / G::RAW_RING) & 1));
    } else if (warp >= 14) {
        // ------------------------------------------------------------ value scales of the blocks that are seen
        const int64_t seen = base > lo_min ? base : lo_min;
        bool small = false;
        for (int64_t b = (seen >> lg) + (tid - 448); b <= (end - 1) >> lg; b += 64) {
            const int64_t id = a.seq.block_table[sr.s * a.seq.table_stride + b];
            if (id >= 0 && id < a.cache.pages) small |= small_scale(block_scale(0.f, a.cache.v_scale[id * a.cache.kv_heads + kv]));
        }
        if (small) *small_s = 1;
        __threadfence_block();
        asm volatile("barrier.cta.arrive 1, 96;" ::: "memory");
    } else if (lane == 0) {
        // ------------------------------------------------------------ products
        constexpr uint32_t qk = tile_idesc(G::N, false), pv = tile_idesc(DP, true);
        const uint32_t q_low = desc_low(smem_u32(q_s), 16), k_low = desc_low(smem_u32(t_s), 16),
                       v_low = desc_low(smem_u32(t_s), G::PANEL);
        auto scores = [&](int h, int j) {
            const int buf = 2 * j % G::T_RING;
            const uint32_t qa = q_low + (h ? G::Q_HALF >> 4 : 0), ka = k_low + buf * (G::T_BUF >> 4);
            const uint32_t d = tmem + G::S0 + h * 128;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k)
                mma_ss(d, qa + (((k >> 2) * G::Q_PANEL + (k & 3) * 32) >> 4),
                       ka + (((k >> 2) * G::PANEL + (k & 3) * 32) >> 4), qk, k > 0);
            mma_commit(&s_full[h]);
            if (h == halves - 1) mma_commit(&t_empty[buf]);
        };
        auto values = [&](int h, int j, int from) {  // over the first or the last 64 tokens
            const uint32_t va = v_low + ((2 * j + 1) % G::T_RING) * (G::T_BUF >> 4) + from * (2048 >> 4);
            const uint32_t d = tmem + G::O0 + h * 128, pa = tmem + G::S0 + h * 128 + from * 8;
            const uint32_t more = j > 0 || from > 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) mma_ts(d, pa + k * 8, va + k * (2048 >> 4), pv, k > 0 ? 1u : more);
        };
        auto ready = [&](int n) { return wait(&t_full[n % G::T_RING], (uint32_t)((n / G::T_RING) & 1)); };
        bool ok = wait(q_full, 0) && ready(0);
        if (ok) {
            tmem_fence_after();
            for (int h = 0; h < halves; ++h) scores(h, 0);
        }
        for (int j = 0; ok && j < tiles; ++j) {
            ok = ready(2 * j + 1);
            for (int h = 0; ok && h < halves; ++h) {
                ok = wait(&p_half[h], (uint32_t)(j & 1));
                if (!ok) break;
                tmem_fence_after();
                values(h, j, 0);
                ok = wait(&p_full[h], (uint32_t)(j & 1));
                if (!ok) break;
                tmem_fence_after();
                values(h, j, 4);
                if (h == halves - 1) mma_commit(&t_empty[(2 * j + 1) % G::T_RING]);
                if (j + 1 < tiles) {
                    if (h == 0) ok = ready(2 * j + 2);
                    if (!ok) break;
                    tmem_fence_after();
                    scores(h, j + 1);
                } else {
                    mma_commit(&o_full[h]);
                }
            }
        }
        if (!ok) {  // an expired wait has set the status bit: the products under way end before their memory goes
            mma_commit(drained);
            wait(drained, 0);
        }
    }
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == 13) {
        __syncwarp();
        tmem_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::TMEM) : "memory");
    }
}

}  // namespace bfft
