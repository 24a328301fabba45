// bfft_rotary.cu -- rotation by position, appending rotated keys (and values) to
// a paged 8-bit cache, and reading such a cache back.
//
// A rotation multiplies the pair (a, b) = a + ib of a head by a unit root of its
// position p, m e^{i p w_j} = c + is from a table made in float64 and rounded
// once (the form of the transforms' twiddle tables):
//     a' = a c - b s,   b' = a s + b c.
// The inverse direction conjugates the root; it is the adjoint, so it is also the
// gradient's rotation.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <string>

#include "../../include/bfft.h"
#include "bfft_cache.cuh"
#include "bfft_kernels.cuh"

using namespace bfft;

namespace bfft {

// A head's row is cut into units of 2 P elements, two packs of P each: P pairs
// that rotate (interleaved: neighbours; half: element j and j + rotated / 2), or
// 2 P elements behind the rotated part, which pass through.
struct RowShape {
    int rotated;
    int units;       // of a row
    int rot_units;   // of them, rotating
};

template <int P, int LAYOUT>
__device__ __forceinline__ void unit_offsets(const RowShape& r, int u, int& o0, int& o1) {
    if (u >= r.rot_units) {
        o0 = r.rotated + (u - r.rot_units) * 2 * P;
        o1 = o0 + P;
    } else if (LAYOUT == BFFT_PAIRS_HALF) {
        o0 = u * P;
        o1 = r.rotated / 2 + u * P;
    } else {
        o0 = u * 2 * P;
        o1 = o0 + P;
    }
}

template <typename T, int P>
struct Unit {
    Pack<T, P> a, b;
};

template <typename T, int P>
__device__ __forceinline__ Unit<T, P> load_unit(const T* row, int o0, int o1) {
    Unit<T, P> u;
    u.a = *reinterpret_cast<const Pack<T, P>*>(row + o0);
    u.b = *reinterpret_cast<const Pack<T, P>*>(row + o1);
    return u;
}
template <typename T, int P>
__device__ __forceinline__ void widen_unit(const Unit<T, P>& u, float (&e)[2 * P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
        e[i] = to_f32(u.a.v[i]);
        e[P + i] = to_f32(u.b.v[i]);
    }
}

template <typename T, int P>
__device__ __forceinline__ void store_unit(T* row, int o0, int o1, const float (&e)[2 * P]) {
    Pack<T, P> a, b;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        a.v[i] = from_f32<T>(e[i]);
        b.v[i] = from_f32<T>(e[P + i]);
    }
    *reinterpret_cast<Pack<T, P>*>(row + o0) = a;
    *reinterpret_cast<Pack<T, P>*>(row + o1) = b;
}

// Roots of unit u at position p; NaN where the table has no row p.
template <int P>
__device__ __forceinline__ void load_roots(const float2* __restrict__ table, int64_t rows, int pairs, int64_t p, int u,
                                           float (&c)[P], float (&s)[P]) {
    if (p >= 0 && p < rows) {
        const float2* t = table + p * pairs + u * P;
        if (P >= 2 && (reinterpret_cast<uintptr_t>(t) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < P; i += 2) {
                const float4 w = *reinterpret_cast<const float4*>(t + i);
                c[i] = w.x;
                s[i] = w.y;
                c[i + (P > 1)] = w.z;
                s[i + (P > 1)] = w.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 w = t[i];
                c[i] = w.x;
                s[i] = w.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < P; ++i) c[i] = s[i] = __int_as_float(0x7fffffff);
    }
}

// STEPS: every product and sum rounded by itself (no contraction), so that the
// 8-bit codes made from the result are those of the formula evaluated step by
// step in 32 bits; a contracted product moves one in some 10^5 to its neighbour.
template <int P, int LAYOUT, bool STEPS>
__device__ __forceinline__ void rotate_unit(float (&e)[2 * P], const float (&c)[P], const float (&s)[P]) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int ia = LAYOUT == BFFT_PAIRS_HALF ? i : 2 * i, ib = LAYOUT == BFFT_PAIRS_HALF ? P + i : 2 * i + 1;
        const float a = e[ia], b = e[ib];
        if constexpr (STEPS) {
            e[ia] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
            e[ib] = __fadd_rn(__fmul_rn(a, s[i]), __fmul_rn(b, c[i]));
        } else {
            e[ia] = a * c[i] - b * s[i];
            e[ib] = a * s[i] + b * c[i];
        }
    }
}

// ---------------------------------------------------------------- rotation
struct RotateArgs {
    const void* x;
    void* y;
    const void* positions;
    const float2* table;
    int64_t tokens, rows;  // rows = batch * tokens
    int64_t xb, xt, xh, yb, yt, yh, pb, pt;
    int64_t table_rows;
    RowShape shape;
    int heads, groups;     // a thread takes heads g, g + groups, ...
    int pos64;
    float sign;            // of the sine: -1 conjugates
};

// Heads g, g + step, ... of one token, unit (o0, o1) of each: the first head's loads
// are in flight beside the roots', which are loaded once for all heads.
// `roots` is called after the first loads (what it waits for runs beside them).
// y may be x: a thread writes only elements that it has read.  Bound by HBM: 16384
// tokens of 32 bf16 heads of 128 in 49 us, 5.7 TB/s, 0.87 of the measured rate (float32
// 0.93); two heads ahead took registers for nothing (57 us), four 70.
constexpr int kHeadsAhead = 1;
template <typename T, int P, int LAYOUT, typename Roots>
__device__ __forceinline__ void rotate_heads(const T* x, T* y, int64_t xh, int64_t yh, int heads, int g, int step, int o0,
                                             int o1, bool turns, float sign, Roots roots) {
    float c[P], s[P];
    bool have = false;
    for (int h0 = g; h0 < heads; h0 += kHeadsAhead * step) {
        Unit<T, P> w[kHeadsAhead];
#pragma unroll
        for (int k = 0; k < kHeadsAhead; ++k) {
            const int h = h0 + k * step;
            if (h < heads) w[k] = load_unit<T, P>(x + h * xh, o0, o1);
        }
        if (!have) {
            if (turns) {
                roots(c, s);
#pragma unroll
                for (int i = 0; i < P; ++i) s[i] *= sign;
            }
            have = true;
        }
#pragma unroll
        for (int k = 0; k < kHeadsAhead; ++k) {
            const int h = h0 + k * step;
            if (h >= heads) break;
            float e[2 * P];
            widen_unit<T, P>(w[k], e);
            if (turns) rotate_unit<P, LAYOUT, false>(e, c, s);
            store_unit<T, P>(y + h * yh, o0, o1, e);
        }
    }
}

template <typename T, int P, int LAYOUT>
__global__ void __launch_bounds__(256, 3) k_rotate(RotateArgs a) {
    griddep_wait();
    griddep_launch_dependents();
    const int u = threadIdx.x;
    const int64_t slot = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int64_t row = slot / a.groups;
    if (row >= a.rows) return;
    const int g = (int)(slot - row * a.groups);
    const int64_t b = row / a.tokens, t = row - b * a.tokens;
    int o0, o1;
    unit_offsets<P, LAYOUT>(a.shape, u, o0, o1);
    rotate_heads<T, P, LAYOUT>(static_cast<const T*>(a.x) + b * a.xb + t * a.xt, static_cast<T*>(a.y) + b * a.yb + t * a.yt,
                               a.xh, a.yh, a.heads, g, a.groups, o0, o1, u < a.shape.rot_units, a.sign,
                               [&](float (&c)[P], float (&s)[P]) {
                                   const int64_t at = b * a.pb + t * a.pt;
                                   const int64_t p = a.pos64 ? static_cast<const int64_t*>(a.positions)[at]
                                                             : (int64_t) static_cast<const int32_t*>(a.positions)[at];
                                   load_roots<P>(a.table, a.table_rows, a.shape.rotated / 2, p, u, c, s);
                               });
}

// ---------------------------------------------------------------- append
// One launch has a warp for each run and head and for each token's queries: the
// chain of dependent loads (sequence, page, scale) is the time, and many warps hide
// it (256 tokens of 32 + 8 + 8 heads of 128: 41 us with a block of 256 threads
// each).  A few long runs (a prompt) leave too few warps: they take two launches,
// the queries' rotation and a block for each run and group of heads.  Append and
// read back, 32 + 8 + 8 heads: 1024 tokens of one sequence 21.5 us by blocks, 30.8
// by warps; 64 sequences of 16 tokens 30.8 and 20.5; 16.9k tokens of 16 sequences
// 134 and 125.
struct AppendArgs {
    CacheView cache;
    SequenceView seq;        // lens: tokens held before the call
    const void *k, *v, *q;
    void* q_out;
    int64_t kt, kh, vt, vh, qt, qh, ot, oh;
    const void* positions;   // null: the place in the cache
    const float2* table;     // null: no rotation
    int64_t table_rows;
    RowShape k_shape, v_shape;
    int q_heads, pos64;
    int by_token;            // 1: a slot is a token, 0: a run of up to a page (see run_of_slot)
    int64_t slots;           // runs at most
};

// The run of new tokens that slot i stands for: tokens [first, first + n) of
// sequence s that go to one page, at place `at` of the sequence.  The runs of
// sequence s take the slots from starts[s] / page + 2 s on (a sequence of n
// tokens has at most n / page + 2 runs), so every slot finds its run by itself.
// By token: a slot is a token, and the first of each run stands for it.
struct Run {
    int s;
    int64_t first, n, at;
};
__device__ __forceinline__ bool run_of_slot(const AppendArgs& a, int64_t i, Run& r) {
    const SequenceView& q = a.seq;
    const int lg = a.cache.page_log2;
    const int64_t page = (int64_t)1 << lg;
    int s;
    if (a.by_token) {
        s = find_sequence(q.starts, q.seqs, i);
    } else {
        const int lane = threadIdx.x & 31;
        int lo = 0, n = q.seqs;
        while (n > 1) {
            const int step = (n + 31) >> 5;
            const int j = lane * step;
            const bool le = j < n && ((int64_t)q.starts[lo + j] >> lg) + 2 * (int64_t)(lo + j) <= i;
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
    const int64_t held = q.lens[s];
    if (t0 < 0 || t0 >= t1 || held < 0) return false;
    int64_t at;  // place of the run's first token
    if (a.by_token) {
        if (i < t0 || i >= t1) return false;
        at = held + (i - t0);
        if (i != t0 && (at & (page - 1))) return false;
    } else {
        const int64_t j = i - ((t0 >> lg) + 2 * (int64_t)s);
        if (j < 0) return false;
        at = j == 0 ? held : (((held >> lg) + j) << lg);
        if (at - held >= t1 - t0) return false;
    }
    r.s = s;
    r.at = at;
    r.first = t0 + (at - held);
    const int64_t room = page - (at & (page - 1)), left = t1 - r.first;
    r.n = room < left ? room : left;
    return true;
}

__device__ __forceinline__ int64_t token_position(const AppendArgs& a, int64_t token, int64_t place) {
    if (!a.positions) return place;
    return a.pos64 ? static_cast<const int64_t*>(a.positions)[token]
                   : (int64_t) static_cast<const int32_t*>(a.positions)[token];
}

constexpr int kAppendThreads = 256;  // of the kernel of short runs
constexpr int kRunThreads = 256;     // of the kernel of long runs: two units each of 64 rows of 128 elements

// max of |x| that keeps NaN
__device__ __forceinline__ float max_abs(float m, float x) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
    return r;
}

// Unit i of a run: its row and its packs' places.
struct Place {
    int row, u, o0, o1;
};
template <int P, int LAYOUT>
__device__ __forceinline__ Place place_of(const RowShape& shape, int i) {
    Place p;
    p.row = i / shape.units;
    p.u = i - p.row * shape.units;
    unit_offsets<P, LAYOUT>(shape, p.u, p.o0, p.o1);
    return p;
}

// What a thread holds of a run, the same for all heads: the places of HELD units and
// (keys) their roots.
template <int P, int HELD>
struct RunUnits {
    Place at[HELD];
    bool has[HELD], turns[HELD];
    float c[HELD][P], s[HELD][P];
};
template <int P, int LAYOUT, bool ROTATE, int HELD>
__device__ __forceinline__ void find_units(const AppendArgs& a, const Run& r, int tid, int threads, RunUnits<P, HELD>& m) {
    const RowShape& shape = ROTATE ? a.k_shape : a.v_shape;
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int i = tid + k * threads;
        m.has[k] = i < (int)r.n * shape.units;
        m.at[k] = place_of<P, LAYOUT>(shape, i);
        m.turns[k] = ROTATE && m.has[k] && m.at[k].u < shape.rot_units;
        if (m.turns[k])
            load_roots<P>(a.table, a.table_rows, shape.rotated / 2,
                          token_position(a, r.first + m.at[k].row, r.at + m.at[k].row), m.at[k].u, m.c[k], m.s[k]);
    }
}
template <typename T, int P, bool ROTATE, int HELD>
__device__ __forceinline__ void fetch_units(const AppendArgs& a, const Run& r, int head, const RunUnits<P, HELD>& m,
                                            Unit<T, P> (&raw)[HELD]) {
    const T* x = static_cast<const T*>(ROTATE ? a.k : a.v) + head * (ROTATE ? a.kh : a.vh);
    const int64_t xt = ROTATE ? a.kt : a.vt;
#pragma unroll
    for (int k = 0; k < HELD; ++k)
        if (m.has[k]) raw[k] = load_unit<T, P>(x + (r.first + m.at[k].row) * xt, m.at[k].o0, m.at[k].o1);
}

// One run's rows of one kv head, of the keys (ROTATE) or the values, by `threads`
// threads: the largest magnitude, the block's new scale, then the codes -- those
// that the page already held first, where the scale grew.  An infinity or a
// NaN survives the maximum: it makes the scale NaN, so that the block reads as NaN.
// The HELD units a thread of `raw` are rotated once and stay in registers; a longer
// run's others are read for the maximum and again for the codes.
template <typename T, int P, int LAYOUT, int CODE, bool ROTATE, int HELD, typename Most>
__device__ __forceinline__ void append_rows(const AppendArgs& a, const Run& r, int64_t page_id, int head,
                                            const RunUnits<P, HELD>& m, const Unit<T, P> (&raw)[HELD], int tid, int threads,
                                            Most most_of) {
    const RowShape& shape = ROTATE ? a.k_shape : a.v_shape;
    const T* x = static_cast<const T*>(ROTATE ? a.k : a.v) + head * (ROTATE ? a.kh : a.vh);
    const int64_t xt = ROTATE ? a.kt : a.vt;
    const int dim = a.cache.dim;
    const int old = (int)(r.at & (((int64_t)1 << a.cache.page_log2) - 1));
    const int total = (int)r.n * shape.units;
    const int64_t block = page_id * a.cache.kv_heads + head;
    uint8_t* codes = (ROTATE ? a.cache.k : a.cache.v) + ((block << a.cache.page_log2) * dim);
    float* scale = (ROTATE ? a.cache.k_scale : a.cache.v_scale) + block;
    const float before = old > 0 ? *scale : 0.f;

    auto value = [&](const Place& p, float (&e)[2 * P]) {
        widen_unit<T, P>(load_unit<T, P>(x + (r.first + p.row) * xt, p.o0, p.o1), e);
        if (ROTATE && p.u < shape.rot_units) {
            float c[P], s[P];
            load_roots<P>(a.table, a.table_rows, shape.rotated / 2, token_position(a, r.first + p.row, r.at + p.row), p.u, c,
                          s);
            rotate_unit<P, LAYOUT, true>(e, c, s);
        }
    };
    float held[HELD][2 * P];
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < HELD; ++k)
        if (m.has[k]) {
            widen_unit<T, P>(raw[k], held[k]);
            if (m.turns[k]) rotate_unit<P, LAYOUT, true>(held[k], m.c[k], m.s[k]);
#pragma unroll
            for (int j = 0; j < 2 * P; ++j) most = max_abs(most, held[k][j]);
        }
#pragma unroll 1
    for (int i = tid + HELD * threads; i < total; i += threads) {
        float e[2 * P];
        value(place_of<P, LAYOUT>(shape, i), e);
#pragma unroll
        for (int j = 0; j < 2 * P; ++j) most = max_abs(most, e[j]);
    }
    // the order of magnitudes' bits puts NaN over infinity over numbers; its barrier also orders the reads of the
    // scale before its write
    const uint32_t big = most_of(__float_as_uint(most) & 0x7fffffffu);
    // a block under 2^-126 * most is zero: no denormal scales
    float now = __uint_as_float(big) / CodeRange<CODE>::most;
    if (now < 1.17549435e-38f) now = 0.f;
    if (big >= 0x7f800000u) now = __int_as_float(0x7fffffff);
    now = __uint_as_float(max(__float_as_uint(now), __float_as_uint(before) & 0x7fffffffu));
    const float inv = now == 0.f ? 0.f : 1.f / now;
    if (old > 0 && now != before) {
        // codes times the ratio of the scales, in 64 bits: in 32 the three roundings of
        // a code of 127 (127 * 3 * 2^-24) could pass a value over the middle of two codes
        const double shrink = (double)before / (double)now;
#pragma unroll 1
        for (int i = tid; i < old * dim / 16; i += threads) {
            Pack<uint8_t, 16> c = reinterpret_cast<const Pack<uint8_t, 16>*>(codes)[i];
#pragma unroll 4
            for (int j = 0; j < 16; ++j) c.v[j] = to_code<CODE>((double)code_value<CODE>(c.v[j]) * shrink);
            reinterpret_cast<Pack<uint8_t, 16>*>(codes)[i] = c;
        }
    }
    if (tid == 0) *scale = now;
    auto write = [&](const Place& p, float (&e)[2 * P]) {
#pragma unroll
        for (int j = 0; j < 2 * P; ++j) e[j] = __fmul_rn(e[j], inv);
        uint8_t* to = codes + (old + p.row) * dim;
        *reinterpret_cast<Pack<uint8_t, P>*>(to + p.o0) = to_codes<CODE, P>(e);
        *reinterpret_cast<Pack<uint8_t, P>*>(to + p.o1) = to_codes<CODE, P>(e + P);
    };
#pragma unroll
    for (int k = 0; k < HELD; ++k)
        if (m.has[k]) write(m.at[k], held[k]);
#pragma unroll 1
    for (int i = tid + HELD * threads; i < total; i += threads) {
        const Place p = place_of<P, LAYOUT>(shape, i);
        float e[2 * P];
        value(p, e);
        write(p, e);
    }
}

// The run, its page and its roots are found once for the block's heads, and a
// head's rows load while the head before is coded.
template <typename T, int P, int LAYOUT, int CODE, bool ROTATE, int HELD>
__device__ __forceinline__ void append_heads(const AppendArgs& a, const Run& r, int first, int last,
                                             uint32_t (*shared_max)[kRunThreads / 32]) {
    RunUnits<P, HELD> m;
    Unit<T, P> raw[HELD], next[HELD];
    find_units<P, LAYOUT, ROTATE, HELD>(a, r, threadIdx.x, kRunThreads, m);
    fetch_units<T, P, ROTATE, HELD>(a, r, first, m, next);
    const int64_t page_id = page_of(a.seq, a.cache, r.s, r.at);
    if (page_id < 0) return;
    for (int head = first; head < last; ++head) {
#pragma unroll
        for (int k = 0; k < HELD; ++k) raw[k] = next[k];
        if (head + 1 < last) fetch_units<T, P, ROTATE, HELD>(a, r, head + 1, m, next);
        auto most_of = [&](uint32_t big) {
            big = __reduce_max_sync(0xffffffffu, big);
            if ((threadIdx.x & 31) == 0) shared_max[head & 1][threadIdx.x >> 5] = big;
            __syncthreads();
            return __reduce_max_sync(0xffffffffu, shared_max[head & 1][threadIdx.x & (kRunThreads / 32 - 1)]);
        };
        append_rows<T, P, LAYOUT, CODE, ROTATE, HELD>(a, r, page_id, head, m, raw, threadIdx.x, kRunThreads, most_of);
    }
}

template <typename T, int P, int LAYOUT, int CODE>
__global__ void __launch_bounds__(kRunThreads, 2) k_append_runs(AppendArgs a, int heads_per_block) {
    griddep_wait();
    griddep_launch_dependents();
    __shared__ uint32_t shared_max[2][kRunThreads / 32];
    const int heads = a.cache.kv_heads, parts = (heads + heads_per_block - 1) / heads_per_block;
    const int64_t slot = blockIdx.x / (2 * parts);
    const int which = (int)(blockIdx.x - slot * 2 * parts);
    Run r;
    if (!run_of_slot(a, slot, r)) return;
    const bool keys = which < parts;
    const int first = (keys ? which : which - parts) * heads_per_block;
    const int last = first + heads_per_block < heads ? first + heads_per_block : heads;
    constexpr int HELD = P >= 4 ? 2 : 4;
    if (keys)
        append_heads<T, P, LAYOUT, CODE, true, HELD>(a, r, first, last, shared_max);
    else
        append_heads<T, P, LAYOUT, CODE, false, HELD>(a, r, first, last, shared_max);
}

// A warp's run of one kv head.
template <typename T, int P, int LAYOUT, int CODE, bool ROTATE>
__device__ __forceinline__ void append_warp(const AppendArgs& a, const Run& r, int head, int lane) {
    RunUnits<P, 1> m;
    Unit<T, P> raw[1];
    find_units<P, LAYOUT, ROTATE, 1>(a, r, lane, 32, m);
    fetch_units<T, P, ROTATE, 1>(a, r, head, m, raw);
    const int64_t page_id = page_of(a.seq, a.cache, r.s, r.at);
    if (page_id < 0) return;
    append_rows<T, P, LAYOUT, CODE, ROTATE, 1>(a, r, page_id, head, m, raw, lane, 32, [](uint32_t big) {
        big = __reduce_max_sync(0xffffffffu, big);
        __syncwarp();  // the reduction alone does not order memory
        return big;
    });
}

// Position of a new token.
__device__ __forceinline__ int64_t new_position(const AppendArgs& a, int64_t token, int s) {
    return token_position(a, token, (int64_t)a.seq.lens[s] + (token - a.seq.starts[s]));
}

// Warps [0, slots * kv_heads * 2): a run's keys or values of one head.  The warps
// behind them rotate the queries, one token each.
template <typename T, int P, int LAYOUT, int CODE>
__global__ void __launch_bounds__(kAppendThreads, 3) k_append(AppendArgs a) {
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31;
    const int64_t per_slot = 2 * a.cache.kv_heads, runs = a.slots * per_slot;
    const int64_t i = (int64_t)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
    if (i < runs) {
        const int64_t slot = i / per_slot;
        const int which = (int)(i - slot * per_slot);
        Run r;
        if (!run_of_slot(a, slot, r)) return;
        if (which < a.cache.kv_heads)
            append_warp<T, P, LAYOUT, CODE, true>(a, r, which, lane);
        else
            append_warp<T, P, LAYOUT, CODE, false>(a, r, which - a.cache.kv_heads, lane);
        return;
    }
    const int64_t token = i - runs;
    if (!a.q || token >= a.seq.tokens) return;
    const int s = find_sequence(a.seq.starts, a.seq.seqs, token);
    const RowShape& shape = a.k_shape;
    const int64_t p = new_position(a, token, s);
    // the lanes over the units of one or several heads
    const int across = shape.units < 32 ? shape.units : 32, heads = 32 / across;
    for (int u = lane % across; u < shape.units && lane < across * heads; u += across) {
        int o0, o1;
        unit_offsets<P, LAYOUT>(shape, u, o0, o1);
        rotate_heads<T, P, LAYOUT>(static_cast<const T*>(a.q) + token * a.qt, static_cast<T*>(a.q_out) + token * a.ot, a.qh,
                                   a.oh, a.q_heads, lane / across, heads, o0, o1, u < shape.rot_units, 1.f,
                                   [&](float (&c)[P], float (&sn)[P]) {
                                       load_roots<P>(a.table, a.table_rows, shape.rotated / 2, p, u, c, sn);
                                   });
    }
}

// The queries of long runs: as k_rotate, the position from the token's sequence.
template <typename T, int P, int LAYOUT>
__global__ void __launch_bounds__(256, 3) k_rotate_new(AppendArgs a, int groups, int rows_per_block) {
    griddep_wait();
    griddep_launch_dependents();
    __shared__ int64_t position[256];
    const int units = a.k_shape.units;
    const int64_t token0 = (int64_t)blockIdx.x * rows_per_block;
    // a warp for each of the block's tokens in turn finds its position
    for (int r = threadIdx.x >> 5; r < rows_per_block; r += 8) {
        const int64_t token = token0 + r;
        if (token >= a.seq.tokens) break;
        const int s = find_sequence(a.seq.starts, a.seq.seqs, token);
        if ((threadIdx.x & 31) == 0) position[r] = new_position(a, token, s);
    }
    __syncthreads();
    const int per = units * groups, r = threadIdx.x / per, at = threadIdx.x - r * per;
    const int64_t token = token0 + r;
    if (r >= rows_per_block || token >= a.seq.tokens) return;
    const int g = at / units, u = at - g * units;
    int o0, o1;
    unit_offsets<P, LAYOUT>(a.k_shape, u, o0, o1);
    rotate_heads<T, P, LAYOUT>(static_cast<const T*>(a.q) + token * a.qt, static_cast<T*>(a.q_out) + token * a.ot, a.qh, a.oh,
                               a.q_heads, g, groups, o0, o1, u < a.k_shape.rot_units, 1.f,
                               [&](float (&c)[P], float (&sn)[P]) {
                                   load_roots<P>(a.table, a.table_rows, a.k_shape.rotated / 2, position[r], u, c, sn);
                               });
}

// ---------------------------------------------------------------- read
struct ReadArgs {
    CacheView cache;
    SequenceView seq;  // lens: the first token that is read of each sequence
    void *k, *v;       // [tokens][kv_heads][dim]
};

// A warp per token: its keys and values of all heads, 16 codes a lane and step
// (17.9k tokens of 8 + 8 heads of 128: 25 us, 4.4 TB/s).
// Tokens without a valid page read as NaN.
template <typename T, int CODE>
__global__ void __launch_bounds__(256) k_read(ReadArgs a) {
    griddep_wait();
    griddep_launch_dependents();
    const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (t >= a.seq.tokens) return;
    const int lane = threadIdx.x & 31, dim = a.cache.dim, heads = a.cache.kv_heads;
    const int s = find_sequence(a.seq.starts, a.seq.seqs, t);
    const int64_t at = (int64_t)a.seq.lens[s] + (t - a.seq.starts[s]);
    const int64_t page_id = t < a.seq.starts[s] ? -1 : page_of(a.seq, a.cache, s, at);
    const int slot = (int)(at & (((int64_t)1 << a.cache.page_log2) - 1));
    const int chunks = dim / 16, half = heads * chunks;
#pragma unroll 4
    for (int i = lane; i < 2 * half; i += 32) {
        const bool is_v = i >= half;
        const int j = is_v ? i - half : i;
        const int h = j / chunks, c = j - h * chunks;
        float scale = __int_as_float(0x7fffffff);
        Pack<uint8_t, 16> codes = {};
        if (page_id >= 0) {
            const int64_t block = page_id * heads + h;
            scale = (is_v ? a.cache.v_scale : a.cache.k_scale)[block];
            codes = *reinterpret_cast<const Pack<uint8_t, 16>*>((is_v ? a.cache.v : a.cache.k) +
                                                                ((block << a.cache.page_log2) + slot) * dim + c * 16);
        }
        constexpr int P = 16 / sizeof(T);
        T* to = static_cast<T*>(is_v ? a.v : a.k) + (t * heads + h) * dim + c * 16;
#pragma unroll
        for (int w = 0; w < 16 / P; ++w) {
            Pack<T, P> o;
#pragma unroll
            for (int b = 0; b < P; ++b) o.v[b] = from_f32<T>(code_value<CODE>(codes.v[w * P + b]) * scale);
            reinterpret_cast<Pack<T, P>*>(to)[w] = o;
        }
    }
}

}  // namespace bfft

// ---------------------------------------------------------------- host side
namespace {

int type_bytes(int64_t type) { return type == BFFT_F32 ? 4 : 2; }

// Largest pack of P elements (P * bytes <= 16) that divides every pointer's and
// stride's alignment and cuts the rotated and the passing part into whole units.
int pick_pack(int bytes, int layout, int64_t dim, int64_t rotated, const void* const* ptrs, int nptrs,
              const int64_t* strides, int nstrides) {
    for (int p = 16 / bytes; p > 1; p /= 2) {
        const int64_t rot = layout == BFFT_PAIRS_HALF ? rotated / 2 : rotated;
        bool ok = rot % (layout == BFFT_PAIRS_HALF ? p : 2 * p) == 0 && (dim - rotated) % (2 * p) == 0;
        for (int i = 0; ok && i < nptrs; ++i) ok = aligned(ptrs[i], p * bytes);
        for (int i = 0; ok && i < nstrides; ++i) ok = strides[i] % p == 0;
        if (ok) return p;
    }
    return 1;
}

RowShape row_shape(int64_t dim, int64_t rotated, int p) {
    RowShape r;
    r.rotated = (int)rotated;
    r.units = (int)(dim / (2 * p));
    r.rot_units = (int)(rotated / (2 * p));
    return r;
}

template <typename T, int P>
cudaError_t rotate_layout(int layout, const RotateArgs& a, dim3 grid, dim3 block, cudaStream_t s) {
    if (layout == BFFT_PAIRS_HALF) return launch_dependent(k_rotate<T, P, BFFT_PAIRS_HALF>, grid.x, block, 0, s, a);
    return launch_dependent(k_rotate<T, P, BFFT_PAIRS_INTERLEAVED>, grid.x, block, 0, s, a);
}
template <typename T>
cudaError_t rotate_pack(int p, int layout, const RotateArgs& a, dim3 grid, dim3 block, cudaStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (p == 8) return rotate_layout<T, 8>(layout, a, grid, block, s);
    if (p == 4) return rotate_layout<T, 4>(layout, a, grid, block, s);
    if (p == 2) return rotate_layout<T, 2>(layout, a, grid, block, s);
    return rotate_layout<T, 1>(layout, a, grid, block, s);
}

// Launches of one append; `runs`: by runs (see AppendArgs).
struct AppendPlan {
    bool runs;
    unsigned blocks;              // of the kernel of keys and values (and queries, where not by runs)
    int heads_per_block;          // kv heads, by runs
    int groups, rows_per_block;   // of the queries' rotation by runs
    unsigned q_blocks;
};

template <typename T, int P, int LAYOUT>
cudaError_t append_code(int code, const AppendArgs& a, const AppendPlan& p, cudaStream_t s) {
    if (!p.runs) {
        if (code == BFFT_CODE_INT8)
            return launch_dependent(k_append<T, P, LAYOUT, kCodeInt8>, p.blocks, kAppendThreads, 0, s, a);
        return launch_dependent(k_append<T, P, LAYOUT, kCodeE4m3>, p.blocks, kAppendThreads, 0, s, a);
    }
    if (p.q_blocks) {
        const cudaError_t e =
            launch_dependent(k_rotate_new<T, P, LAYOUT>, p.q_blocks, 256, 0, s, a, p.groups, p.rows_per_block);
        if (e != cudaSuccess) return e;
    }
    if (code == BFFT_CODE_INT8)
        return launch_dependent(k_append_runs<T, P, LAYOUT, kCodeInt8>, p.blocks, kRunThreads, 0, s, a, p.heads_per_block);
    return launch_dependent(k_append_runs<T, P, LAYOUT, kCodeE4m3>, p.blocks, kRunThreads, 0, s, a, p.heads_per_block);
}
template <typename T, int P>
cudaError_t append_layout(int layout, int code, const AppendArgs& a, const AppendPlan& p, cudaStream_t s) {
    if (layout == BFFT_PAIRS_HALF) return append_code<T, P, BFFT_PAIRS_HALF>(code, a, p, s);
    return append_code<T, P, BFFT_PAIRS_INTERLEAVED>(code, a, p, s);
}
template <typename T>
cudaError_t append_pack(int pack, int layout, int code, const AppendArgs& a, const AppendPlan& p, cudaStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (pack == 8) return append_layout<T, 8>(layout, code, a, p, s);
    if (pack == 4) return append_layout<T, 4>(layout, code, a, p, s);
    if (pack == 2) return append_layout<T, 2>(layout, code, a, p, s);
    return append_layout<T, 1>(layout, code, a, p, s);
}

template <typename T>
cudaError_t read_code(int code, const ReadArgs& a, dim3 grid, cudaStream_t s) {
    if (code == BFFT_CODE_INT8) return launch_dependent(k_read<T, kCodeInt8>, grid.x, 256, 0, s, a);
    return launch_dependent(k_read<T, kCodeE4m3>, grid.x, 256, 0, s, a);
}

}  // namespace

namespace bfft {

bfft_status fail(bfft_status st, const char* fmt, ...) {
    char buf[384];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_last_error(buf);  // reported by bfft_last_error()
    return st;
}

bfft_status launched(cudaError_t e, const char* call) {
    if (e == cudaSuccess) return BFFT_OK;
    cudaGetLastError();
    return fail(BFFT_ERR_CUDA, "%s: %s", call, cudaGetErrorString(e));
}

Device::Device(int64_t dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) ok = cudaSetDevice((int)dev) == cudaSuccess;
    changed = ok && prev != dev;
    if (!ok || prev < 0) cudaGetLastError();
}
Device::~Device() {
    if (changed && prev >= 0) cudaSetDevice(prev);
}

bfft_status check_cache(const bfft_cache_desc* c) {
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(BFFT_ERR_VALUE, "null cache pointer");
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return fail(BFFT_ERR_VALUE, "cache codes must be 16-byte aligned");
    if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return fail(BFFT_ERR_VALUE, "cache scales must be 4-byte aligned");
    if (c->code != BFFT_CODE_INT8 && c->code != BFFT_CODE_E4M3)
        return fail(BFFT_ERR_VALUE, "bad code %lld", (long long)c->code);
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
        return fail(BFFT_ERR_SHAPE, "page must be 16, 32, 64 or 128 tokens, got %lld", (long long)c->page);
    if (c->dim < 16 || c->dim > 256 || c->dim % 16)
        return fail(BFFT_ERR_SHAPE, "head dimension must be a multiple of 16 in [16, 256], got %lld",
                    (long long)c->dim);
    if (c->kv_heads < 1 || c->kv_heads > 65535 || c->pages < 1 || c->pages > 0x7fffffffLL)
        return fail(BFFT_ERR_SHAPE, "bad cache of %lld pages, %lld heads", (long long)c->pages,
                    (long long)c->kv_heads);
    return BFFT_OK;
}

bfft_status check_sequences(const bfft_sequence_desc* q) {
    if (!q->block_table || !q->lens || !q->starts) return fail(BFFT_ERR_VALUE, "null sequence pointer");
    if (!aligned(q->block_table, 4) || !aligned(q->lens, 4) || !aligned(q->starts, 4))
        return fail(BFFT_ERR_VALUE, "sequence tables must be 4-byte aligned");
    if (q->seqs < 1 || q->seqs > 0x7ffffffeLL || q->max_pages < 1 || q->max_pages > 0x7fffffffLL)
        return fail(BFFT_ERR_SHAPE, "bad table of %lld sequences, %lld pages each", (long long)q->seqs,
                    (long long)q->max_pages);
    if (q->tokens < 0 || q->tokens > 0x7fffffffLL) return fail(BFFT_ERR_SHAPE, "bad row count %lld", (long long)q->tokens);
    return BFFT_OK;
}

CacheView cache_view(const bfft_cache_desc* c) {
    CacheView v;
    v.k = static_cast<uint8_t*>(c->k);
    v.v = static_cast<uint8_t*>(c->v);
    v.k_scale = static_cast<float*>(c->k_scale);
    v.v_scale = static_cast<float*>(c->v_scale);
    v.pages = c->pages;
    v.kv_heads = (int)c->kv_heads;
    v.dim = (int)c->dim;
    v.page_log2 = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
    return v;
}

SequenceView sequence_view(const bfft_sequence_desc* q) {
    SequenceView v;
    v.block_table = static_cast<const int32_t*>(q->block_table);
    v.table_stride = q->table_stride;
    v.lens = static_cast<const int32_t*>(q->lens);
    v.starts = static_cast<const int32_t*>(q->starts);
    v.seqs = (int)q->seqs;
    v.max_pages = (int)q->max_pages;
    v.tokens = q->tokens;
    return v;
}

}  // namespace bfft

extern "C" bfft_status bfft_rotate_positions(const bfft_rotate_desc* d, const void* x, const void* positions,
                                             const void* table, void* y, void* stream) {
    if (!d || !x || !positions || !table || !y) return fail(BFFT_ERR_VALUE, "null pointer");
    if (d->type < BFFT_F32 || d->type > BFFT_BF16) return fail(BFFT_ERR_VALUE, "bad type %lld", (long long)d->type);
    if (d->layout != BFFT_PAIRS_HALF && d->layout != BFFT_PAIRS_INTERLEAVED)
        return fail(BFFT_ERR_VALUE, "bad layout %lld", (long long)d->layout);
    if (d->transform_direction != BFFT_FORWARD && d->transform_direction != BFFT_INVERSE)
        return fail(BFFT_ERR_VALUE, "bad transform_direction %lld", (long long)d->transform_direction);
    if (d->batch < 0 || d->tokens < 0 || d->heads < 0 || d->batch > 0x7fffffffLL || d->tokens > 0x7fffffffLL ||
        d->heads > 0x7fffffffLL)
        return fail(BFFT_ERR_SHAPE, "bad shape %lld x %lld x %lld", (long long)d->batch, (long long)d->tokens,
                    (long long)d->heads);
    if (d->dim < 2 || d->dim > 512 || d->dim % 2)
        return fail(BFFT_ERR_SHAPE, "head dimension must be even and in [2, 512], got %lld", (long long)d->dim);
    if (d->rotated < 2 || d->rotated > d->dim || d->rotated % 2)
        return fail(BFFT_ERR_SHAPE, "rotated part must be even and in [2, %lld], got %lld", (long long)d->dim,
                    (long long)d->rotated);
    const int bytes = type_bytes(d->type);
    if (!aligned(x, bytes) || !aligned(y, bytes) || !aligned(table, 8) || !aligned(positions, d->pos64 ? 8 : 4))
        return fail(BFFT_ERR_VALUE, "misaligned pointer");
    if (d->batch == 0 || d->tokens == 0 || d->heads == 0) return BFFT_OK;
    const void* ptrs[2] = {x, y};
    const int64_t strides[6] = {d->x_batch, d->x_token, d->x_head, d->y_batch, d->y_token, d->y_head};
    const int p = pick_pack(bytes, (int)d->layout, d->dim, d->rotated, ptrs, 2, strides, 6);
    RotateArgs a;
    a.x = x;
    a.y = y;
    a.positions = positions;
    a.table = static_cast<const float2*>(table);
    a.tokens = d->tokens;
    a.rows = d->batch * d->tokens;
    a.xb = d->x_batch, a.xt = d->x_token, a.xh = d->x_head;
    a.yb = d->y_batch, a.yt = d->y_token, a.yh = d->y_head;
    a.pb = d->pos_batch, a.pt = d->pos_token;
    a.table_rows = d->table_rows;
    a.shape = row_shape(d->dim, d->rotated, p);
    a.heads = (int)d->heads;
    // a thread takes eight heads of its token (the roots are loaded once for them),
    // fewer where that leaves the GPU without 1024 threads to an SM
    int per = 8;
    while (per > 1 && a.rows * ((a.heads + per - 1) / per) * a.shape.units < (int64_t)148 * 1024) per /= 2;
    a.groups = (a.heads + per - 1) / per;
    a.pos64 = d->pos64 != 0;
    a.sign = d->transform_direction == BFFT_INVERSE ? -1.f : 1.f;
    dim3 block((unsigned)a.shape.units, 1);
    while (block.x * block.y * 2 <= 256) block.y *= 2;
    const int64_t blocks = (a.rows * a.groups + block.y - 1) / block.y;
    if (blocks > 0x7fffffffLL) return fail(BFFT_ERR_SHAPE, "too many rows: %lld", (long long)a.rows);
    Device g(d->device);
    if (!g.ok) return fail(BFFT_ERR_CUDA, "cannot select device %lld", (long long)d->device);
    const dim3 grid((unsigned)blocks);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    count_launches(1);
    return launched(d->type == BFFT_F32   ? rotate_pack<float>(p, (int)d->layout, a, grid, block, s)
                    : d->type == BFFT_F16 ? rotate_pack<__half>(p, (int)d->layout, a, grid, block, s)
                                       : rotate_pack<__nv_bfloat16>(p, (int)d->layout, a, grid, block, s),
                    "rotate_positions");
}

extern "C" bfft_status bfft_cache_append(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs,
                                         const bfft_append_desc* d, void* stream) {
    if (!cache || !seqs || !d || !d->k || !d->v) return fail(BFFT_ERR_VALUE, "null pointer");
    bfft_status st = check_cache(cache);
    if (st == BFFT_OK) st = check_sequences(seqs);
    if (st != BFFT_OK) return st;
    if (d->type < BFFT_F32 || d->type > BFFT_BF16) return fail(BFFT_ERR_VALUE, "bad type %lld", (long long)d->type);
    if (d->layout != BFFT_PAIRS_HALF && d->layout != BFFT_PAIRS_INTERLEAVED)
        return fail(BFFT_ERR_VALUE, "bad layout %lld", (long long)d->layout);
    const int64_t rotated = d->table ? d->rotated : 0;
    if (rotated < 0 || rotated > cache->dim || rotated % 2 || (d->table && rotated < 2))
        return fail(BFFT_ERR_SHAPE, "rotated part must be even and in [2, %lld], got %lld", (long long)cache->dim,
                    (long long)d->rotated);
    if ((d->q == nullptr) != (d->q_out == nullptr)) return fail(BFFT_ERR_VALUE, "q and q_out go together");
    if (d->q && d->q_heads < 1) return fail(BFFT_ERR_SHAPE, "bad query head count %lld", (long long)d->q_heads);
    const int bytes = type_bytes(d->type);
    if (!aligned(d->k, bytes) || !aligned(d->v, bytes) || !aligned(d->q, bytes) || !aligned(d->q_out, bytes) ||
        !aligned(d->table, 8) || !aligned(d->positions, d->pos64 ? 8 : 4))
        return fail(BFFT_ERR_VALUE, "misaligned pointer");
    if (seqs->tokens == 0) return BFFT_OK;
    const void* ptrs[4] = {d->k, d->v, d->q, d->q_out};
    const int64_t strides[8] = {d->k_token, d->k_head, d->v_token, d->v_head,
                                d->q ? d->q_token : 0, d->q ? d->q_head : 0, d->q ? d->o_token : 0,
                                d->q ? d->o_head : 0};
    const int p = pick_pack(bytes, (int)d->layout, cache->dim, rotated, ptrs, 4, strides, 8);
    AppendArgs a;
    a.cache = cache_view(cache);
    a.seq = sequence_view(seqs);
    a.k = d->k, a.v = d->v, a.q = d->q, a.q_out = d->q_out;
    a.kt = d->k_token, a.kh = d->k_head, a.vt = d->v_token, a.vh = d->v_head;
    a.qt = d->q_token, a.qh = d->q_head, a.ot = d->o_token, a.oh = d->o_head;
    a.positions = d->positions;
    a.pos64 = d->pos64 != 0;
    a.table = static_cast<const float2*>(d->table);
    a.table_rows = d->table_rows;
    a.k_shape = row_shape(cache->dim, rotated, p);
    a.v_shape = row_shape(cache->dim, 0, p);
    a.q_heads = (int)d->q_heads;
    const int64_t runs = seqs->tokens / cache->page + 2 * seqs->seqs;
    a.by_token = seqs->tokens <= runs;
    a.slots = a.by_token ? seqs->tokens : runs;
    AppendPlan plan{};
    plan.runs = !a.by_token && seqs->tokens >= 48 * seqs->seqs && a.slots * 2 * cache->kv_heads < 4096;
    int64_t blocks = a.slots * 2 * cache->kv_heads, q_blocks = 0;
    if (plan.runs) {
        // four kv heads a block, fewer where that leaves less than four blocks to an SM
        plan.heads_per_block = 4;
        while (plan.heads_per_block > 1 &&
               a.slots * 2 * ((cache->kv_heads + plan.heads_per_block - 1) / plan.heads_per_block) < 4 * 148)
            plan.heads_per_block /= 2;
        blocks = a.slots * 2 * ((cache->kv_heads + plan.heads_per_block - 1) / plan.heads_per_block);
        // threads over the units of a group of heads, eight heads a thread at most
        const int units = a.k_shape.units;
        plan.groups = (int)((d->q_heads + 7) / 8);
        while (plan.groups > 1 && units * plan.groups > 256) plan.groups = (plan.groups + 1) / 2;
        plan.rows_per_block = 256 / (units * (plan.groups > 0 ? plan.groups : 1));
        if (d->q) q_blocks = (seqs->tokens + plan.rows_per_block - 1) / plan.rows_per_block;
    } else {
        blocks = (blocks + (d->q ? seqs->tokens : 0) + kAppendThreads / 32 - 1) / (kAppendThreads / 32);
    }
    if (blocks > 0x7fffffffLL) return fail(BFFT_ERR_SHAPE, "too many rows: %lld", (long long)seqs->tokens);
    plan.blocks = (unsigned)blocks;
    plan.q_blocks = (unsigned)q_blocks;
    Device g(d->device);
    if (!g.ok) return fail(BFFT_ERR_CUDA, "cannot select device %lld", (long long)d->device);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int layout = (int)d->layout, code = (int)cache->code;
    count_launches(q_blocks ? 2 : 1);
    return launched(d->type == BFFT_F32   ? append_pack<float>(p, layout, code, a, plan, s)
                    : d->type == BFFT_F16 ? append_pack<__half>(p, layout, code, a, plan, s)
                                       : append_pack<__nv_bfloat16>(p, layout, code, a, plan, s),
                    "cache_append");
}

extern "C" bfft_status bfft_cache_read(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs, int64_t type,
                                       void* k, void* v, int64_t device, void* stream) {
    if (!cache || !seqs || !k || !v) return fail(BFFT_ERR_VALUE, "null pointer");
    bfft_status st = check_cache(cache);
    if (st == BFFT_OK) st = check_sequences(seqs);
    if (st != BFFT_OK) return st;
    if (type < BFFT_F32 || type > BFFT_BF16) return fail(BFFT_ERR_VALUE, "bad type %lld", (long long)type);
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(BFFT_ERR_VALUE, "outputs must be 16-byte aligned");
    if (seqs->tokens == 0) return BFFT_OK;
    ReadArgs a;
    a.cache = cache_view(cache);
    a.seq = sequence_view(seqs);
    a.k = k;
    a.v = v;
    Device g(device);
    if (!g.ok) return fail(BFFT_ERR_CUDA, "cannot select device %lld", (long long)device);
    const dim3 grid((unsigned)((seqs->tokens + 7) / 8));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    count_launches(1);
    return launched(type == BFFT_F32   ? read_code<float>((int)cache->code, a, grid, s)
                    : type == BFFT_F16 ? read_code<__half>((int)cache->code, a, grid, s)
                                       : read_code<__nv_bfloat16>((int)cache->code, a, grid, s),
                    "cache_read");
}
