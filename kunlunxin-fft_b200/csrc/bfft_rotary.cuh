// bfft_rotary.cuh -- rotation by position, alone and on the way into a paged 8-bit
// cache: kernels and their launches by type, pack, layout and code.  Included by
// bfft_rotary.cu (one position a token) and bfft_rotary_axes.cu (positions of several
// axes), each of which instantiates launch_rotate and launch_append for its own.
//
// A rotation multiplies the pair (a, b) = a + ib of a head by a unit root of its
// position p, m e^{i p w_j} = c + is from a table made in float64 and rounded
// once (the form of the transforms' twiddle tables):
//     a' = a c - b s,   b' = a s + b c.
// The inverse direction conjugates the root; it is the adjoint, so it is also the
// gradient's rotation.
#pragma once

#include <cuda_runtime.h>

#include <type_traits>

#include "../../include/bfft.h"
#include "bfft_cache.cuh"
#include "bfft_kernels.cuh"

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

__device__ __forceinline__ int64_t position_at(const void* positions, int pos64, int64_t i) {
    return pos64 ? static_cast<const int64_t*>(positions)[i] : (int64_t) static_cast<const int32_t*>(positions)[i];
}

// Which rows of the table a token's pairs take.  OneAxis: all of them the row of its one
// position.  AxisMap: pair j that of position axis(j) among up to four (time, height,
// width), so that c_j + i s_j = table[p_axis(j)][j].
struct OneAxis {};
struct AxisMap {
    uint32_t of[16];  // two bits for each of up to 256 pairs
    int axes;
    int64_t stride;   // of the positions, from axis to axis
};

// Roots of unit u for the token whose first position is element `at`; NaN for the pairs of
// an axis whose row the table lacks.  A unit within one axis (runs of pairs) needs that
// axis's position and loads its roots as packs, as with one axis; another (pairs dealt in
// turn) loads the positions of all axes side by side and eight bytes a pair.
template <int P>
__device__ __forceinline__ void load_axis_roots(const float2* __restrict__ table, int64_t rows, int pairs, const AxisMap& m,
                                                const void* positions, int pos64, int64_t at, int u, float (&c)[P],
                                                float (&s)[P]) {
    constexpr uint32_t UNIT = (1u << 2 * P) - 1;
    const uint32_t which = (m.of[(u * P) >> 4] >> (2 * ((u * P) & 15))) & UNIT;
    if (which == ((which & 3) * 0x55555555u & UNIT)) {
        load_roots<P>(table, rows, pairs, position_at(positions, pos64, at + (which & 3) * m.stride), u, c, s);
        return;
    }
    int row[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        row[a] = -1;
        if (a < m.axes) {
            const int64_t p = position_at(positions, pos64, at + a * m.stride);
            if (p >= 0 && p < rows) row[a] = (int)p;
        }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const uint32_t a = (which >> (2 * i)) & 3;
        const int r = a < 2 ? (a ? row[1] : row[0]) : (a == 2 ? row[2] : row[3]);
        float2 w = make_float2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
        if (r >= 0) w = table[(int64_t)r * pairs + u * P + i];
        c[i] = w.x;
        s[i] = w.y;
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

// Root of pair j for the token whose first position is element `at`.
__device__ __forceinline__ float2 axis_root(const float2* __restrict__ table, int64_t rows, int pairs, const AxisMap& m,
                                            const void* positions, int pos64, int64_t at, int j) {
    const int64_t p = position_at(positions, pos64, at + ((m.of[j >> 4] >> (2 * (j & 15))) & 3) * m.stride);
    return p >= 0 && p < rows ? table[p * pairs + j] : make_float2(__int_as_float(0x7fffffff), __int_as_float(0x7fffffff));
}
// The roots of the tokens that a block rotates, in shared memory: neighbouring threads load
// neighbouring pairs, each once (16384 tokens of 32 heads, axes dealt in turn: 53 us where
// each thread loaded its own eight bytes at a time).

template <typename T, int P, int LAYOUT, typename Axes>
__global__ void __launch_bounds__(256, 3) k_rotate(RotateArgs a, const __grid_constant__ Axes axes) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr bool AXES = std::is_same_v<Axes, AxisMap>;
    const int u = threadIdx.x;
    const int64_t slot = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int64_t row = slot / a.groups;
    const int g = (int)(slot - row * a.groups);
    const int64_t b = row / a.tokens, t = row - b * a.tokens;
    const float2* mine = nullptr;  // this token's roots
    if constexpr (AXES) {
        extern __shared__ float2 roots[];
        const int pairs = a.shape.rotated / 2;
        const int64_t row0 = (int64_t)blockIdx.x * blockDim.y / a.groups;
        int64_t rows = ((int64_t)(blockIdx.x + 1) * blockDim.y - 1) / a.groups + 1;
        if (rows > a.rows) rows = a.rows;
        const int count = (int)(rows - row0) * pairs;
        for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < count; i += blockDim.x * blockDim.y) {
            const int r = i / pairs;
            const int64_t rb = (row0 + r) / a.tokens, rt = row0 + r - rb * a.tokens;
            const int j = i - r * pairs;  // pair j is the unit j / P's pair j % P: a unit's pairs lie rot_units apart
            roots[r * pairs + j % P * a.shape.rot_units + j / P] =
                axis_root(a.table, a.table_rows, pairs, axes, a.positions, a.pos64, rb * a.pb + rt * a.pt, j);
        }
        __syncthreads();
        mine = roots + (row - row0) * pairs + u;
    }
    if (row >= a.rows) return;
    int o0, o1;
    unit_offsets<P, LAYOUT>(a.shape, u, o0, o1);
    rotate_heads<T, P, LAYOUT>(static_cast<const T*>(a.x) + b * a.xb + t * a.xt, static_cast<T*>(a.y) + b * a.yb + t * a.yt,
                               a.xh, a.yh, a.heads, g, a.groups, o0, o1, u < a.shape.rot_units, a.sign,
                               [&](float (&c)[P], float (&s)[P]) {
                                   if constexpr (AXES) {
#pragma unroll
                                       for (int i = 0; i < P; ++i) {
                                           const float2 w = mine[i * a.shape.rot_units];
                                           c[i] = w.x;
                                           s[i] = w.y;
                                       }
                                   } else {
                                       load_roots<P>(a.table, a.table_rows, a.shape.rotated / 2,
                                                     position_at(a.positions, a.pos64, b * a.pb + t * a.pt), u, c, s);
                                   }
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
    return a.positions ? position_at(a.positions, a.pos64, token) : place;
}

// Roots of unit u of new token `token`, whose place in its sequence is `place`.
template <int P>
__device__ __forceinline__ void token_roots(const AppendArgs& a, const OneAxis&, int64_t token, int64_t place, int u,
                                            float (&c)[P], float (&s)[P]) {
    load_roots<P>(a.table, a.table_rows, a.k_shape.rotated / 2, token_position(a, token, place), u, c, s);
}
template <int P>
__device__ __forceinline__ void token_roots(const AppendArgs& a, const AxisMap& m, int64_t token, int64_t, int u,
                                            float (&c)[P], float (&s)[P]) {
    load_axis_roots<P>(a.table, a.table_rows, a.k_shape.rotated / 2, m, a.positions, a.pos64, token, u, c, s);
}
// The same for its queries, whose position is known (OneAxis): found between their first loads
// and these, it held the loads back (2900 tokens of 25 heads 17.7 -> 22.8 us).
template <int P>
__device__ __forceinline__ void query_roots(const AppendArgs& a, const OneAxis&, int64_t, int64_t position, int u,
                                            float (&c)[P], float (&s)[P]) {
    load_roots<P>(a.table, a.table_rows, a.k_shape.rotated / 2, position, u, c, s);
}
template <int P>
__device__ __forceinline__ void query_roots(const AppendArgs& a, const AxisMap& m, int64_t token, int64_t, int u,
                                            float (&c)[P], float (&s)[P]) {
    token_roots<P>(a, m, token, 0, u, c, s);
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
template <int P, int LAYOUT, bool ROTATE, int HELD, typename Axes>
__device__ __forceinline__ void find_units(const AppendArgs& a, const Axes& axes, const Run& r, int tid, int threads,
                                           RunUnits<P, HELD>& m) {
    const RowShape& shape = ROTATE ? a.k_shape : a.v_shape;
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
        const int i = tid + k * threads;
        m.has[k] = i < (int)r.n * shape.units;
        m.at[k] = place_of<P, LAYOUT>(shape, i);
        m.turns[k] = ROTATE && m.has[k] && m.at[k].u < shape.rot_units;
        if (m.turns[k])
            token_roots<P>(a, axes, r.first + m.at[k].row, r.at + m.at[k].row, m.at[k].u, m.c[k], m.s[k]);
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
template <typename T, int P, int LAYOUT, int CODE, bool ROTATE, int HELD, typename Axes, typename Most>
__device__ __forceinline__ void append_rows(const AppendArgs& a, const Axes& axes, const Run& r, int64_t page_id, int head,
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
            token_roots<P>(a, axes, r.first + p.row, r.at + p.row, p.u, c, s);
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
template <typename T, int P, int LAYOUT, int CODE, bool ROTATE, int HELD, typename Axes>
__device__ __forceinline__ void append_heads(const AppendArgs& a, const Axes& axes, const Run& r, int first, int last,
                                             uint32_t (*shared_max)[kRunThreads / 32]) {
    RunUnits<P, HELD> m;
    Unit<T, P> raw[HELD], next[HELD];
    find_units<P, LAYOUT, ROTATE, HELD>(a, axes, r, threadIdx.x, kRunThreads, m);
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
        append_rows<T, P, LAYOUT, CODE, ROTATE, HELD>(a, axes, r, page_id, head, m, raw, threadIdx.x, kRunThreads, most_of);
    }
}

template <typename T, int P, int LAYOUT, int CODE, typename Axes>
__global__ void __launch_bounds__(kRunThreads, 2) k_append_runs(AppendArgs a, const __grid_constant__ Axes axes,
                                                                int heads_per_block) {
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
        append_heads<T, P, LAYOUT, CODE, true, HELD>(a, axes, r, first, last, shared_max);
    else
        append_heads<T, P, LAYOUT, CODE, false, HELD>(a, axes, r, first, last, shared_max);
}

// A warp's run of one kv head.
template <typename T, int P, int LAYOUT, int CODE, bool ROTATE, typename Axes>
__device__ __forceinline__ void append_warp(const AppendArgs& a, const Axes& axes, const Run& r, int head, int lane) {
    RunUnits<P, 1> m;
    Unit<T, P> raw[1];
    find_units<P, LAYOUT, ROTATE, 1>(a, axes, r, lane, 32, m);
    fetch_units<T, P, ROTATE, 1>(a, r, head, m, raw);
    const int64_t page_id = page_of(a.seq, a.cache, r.s, r.at);
    if (page_id < 0) return;
    append_rows<T, P, LAYOUT, CODE, ROTATE, 1>(a, axes, r, page_id, head, m, raw, lane, 32, [](uint32_t big) {
        big = __reduce_max_sync(0xffffffffu, big);
        __syncwarp();  // the reduction alone does not order memory
        return big;
    });
}

// Position of a new token (of one axis).
__device__ __forceinline__ int64_t new_position(const AppendArgs& a, int64_t token, int s) {
    return token_position(a, token, (int64_t)a.seq.lens[s] + (token - a.seq.starts[s]));
}

// Warps [0, slots * kv_heads * 2): a run's keys or values of one head.  The warps
// behind them rotate the queries, one token each.
template <typename T, int P, int LAYOUT, int CODE, typename Axes>
__global__ void __launch_bounds__(kAppendThreads, 3) k_append(AppendArgs a, const __grid_constant__ Axes axes) {
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
            append_warp<T, P, LAYOUT, CODE, true>(a, axes, r, which, lane);
        else
            append_warp<T, P, LAYOUT, CODE, false>(a, axes, r, which - a.cache.kv_heads, lane);
        return;
    }
    const int64_t token = i - runs;
    if (!a.q || token >= a.seq.tokens) return;
    const RowShape& shape = a.k_shape;
    int64_t position = 0;
    if constexpr (!std::is_same_v<Axes, AxisMap>)
        position = new_position(a, token, find_sequence(a.seq.starts, a.seq.seqs, token));
    // the lanes over the units of one or several heads
    const int across = shape.units < 32 ? shape.units : 32, heads = 32 / across;
    for (int u = lane % across; u < shape.units && lane < across * heads; u += across) {
        int o0, o1;
        unit_offsets<P, LAYOUT>(shape, u, o0, o1);
        rotate_heads<T, P, LAYOUT>(static_cast<const T*>(a.q) + token * a.qt, static_cast<T*>(a.q_out) + token * a.ot, a.qh,
                                   a.oh, a.q_heads, lane / across, heads, o0, o1, u < shape.rot_units, 1.f,
                                   [&](float (&c)[P], float (&sn)[P]) {
                                       query_roots<P>(a, axes, token, position, u, c, sn);
                                   });
    }
}

// The queries of long runs: as k_rotate, the position (of one axis) from the token's sequence.
template <typename T, int P, int LAYOUT, typename Axes>
__global__ void __launch_bounds__(256, 3) k_rotate_new(AppendArgs a, const __grid_constant__ Axes axes, int groups,
                                                       int rows_per_block) {
    griddep_wait();
    griddep_launch_dependents();
    __shared__ int64_t position[256];
    const int units = a.k_shape.units;
    const int64_t token0 = (int64_t)blockIdx.x * rows_per_block;
    if constexpr (!std::is_same_v<Axes, AxisMap>) {
        // a warp for each of the block's tokens in turn finds its position
        for (int r = threadIdx.x >> 5; r < rows_per_block; r += 8) {
            const int64_t token = token0 + r;
            if (token >= a.seq.tokens) break;
            const int s = find_sequence(a.seq.starts, a.seq.seqs, token);
            if ((threadIdx.x & 31) == 0) position[r] = new_position(a, token, s);
        }
        __syncthreads();
    }
    const int per = units * groups, r = threadIdx.x / per, at = threadIdx.x - r * per;
    const int64_t token = token0 + r;
    if (r >= rows_per_block || token >= a.seq.tokens) return;
    const int g = at / units, u = at - g * units;
    int o0, o1;
    unit_offsets<P, LAYOUT>(a.k_shape, u, o0, o1);
    rotate_heads<T, P, LAYOUT>(static_cast<const T*>(a.q) + token * a.qt, static_cast<T*>(a.q_out) + token * a.ot, a.qh, a.oh,
                               a.q_heads, g, groups, o0, o1, u < a.k_shape.rot_units, 1.f,
                               [&](float (&c)[P], float (&sn)[P]) {
                                   query_roots<P>(a, axes, token, position[r], u, c, sn);
                               });
}

// ---------------------------------------------------------------- launches
template <typename T, int P, typename Axes>
cudaError_t rotate_layout(int layout, const RotateArgs& a, const Axes& x, dim3 grid, dim3 block, cudaStream_t s) {
    // the roots of a block's tokens (see k_rotate)
    const size_t smem = std::is_same_v<Axes, AxisMap> ? ((block.y - 1) / a.groups + 2) * (size_t)(a.shape.rotated / 2) * 8 : 0;
    if (layout == BFFT_PAIRS_HALF) return launch_dependent(k_rotate<T, P, BFFT_PAIRS_HALF, Axes>, grid.x, block, smem, s, a, x);
    return launch_dependent(k_rotate<T, P, BFFT_PAIRS_INTERLEAVED, Axes>, grid.x, block, smem, s, a, x);
}
template <typename T, typename Axes>
cudaError_t rotate_pack(int p, int layout, const RotateArgs& a, const Axes& x, dim3 grid, dim3 block, cudaStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (p == 8) return rotate_layout<T, 8>(layout, a, x, grid, block, s);
    if (p == 4) return rotate_layout<T, 4>(layout, a, x, grid, block, s);
    if (p == 2) return rotate_layout<T, 2>(layout, a, x, grid, block, s);
    return rotate_layout<T, 1>(layout, a, x, grid, block, s);
}

// Launches of one append; `runs`: by runs (see AppendArgs).
struct AppendPlan {
    bool runs;
    unsigned blocks;              // of the kernel of keys and values (and queries, where not by runs)
    int heads_per_block;          // kv heads, by runs
    int groups, rows_per_block;   // of the queries' rotation by runs
    unsigned q_blocks;
};

template <typename T, int P, int LAYOUT, typename Axes>
cudaError_t append_code(int code, const AppendArgs& a, const Axes& x, const AppendPlan& p, cudaStream_t s) {
    if (!p.runs) {
        if (code == BFFT_CODE_INT8)
            return launch_dependent(k_append<T, P, LAYOUT, kCodeInt8, Axes>, p.blocks, kAppendThreads, 0, s, a, x);
        return launch_dependent(k_append<T, P, LAYOUT, kCodeE4m3, Axes>, p.blocks, kAppendThreads, 0, s, a, x);
    }
    if (p.q_blocks) {
        const cudaError_t e =
            launch_dependent(k_rotate_new<T, P, LAYOUT, Axes>, p.q_blocks, 256, 0, s, a, x, p.groups, p.rows_per_block);
        if (e != cudaSuccess) return e;
    }
    if (code == BFFT_CODE_INT8)
        return launch_dependent(k_append_runs<T, P, LAYOUT, kCodeInt8, Axes>, p.blocks, kRunThreads, 0, s, a, x, p.heads_per_block);
    return launch_dependent(k_append_runs<T, P, LAYOUT, kCodeE4m3, Axes>, p.blocks, kRunThreads, 0, s, a, x, p.heads_per_block);
}
template <typename T, int P, typename Axes>
cudaError_t append_layout(int layout, int code, const AppendArgs& a, const Axes& x, const AppendPlan& p, cudaStream_t s) {
    if (layout == BFFT_PAIRS_HALF) return append_code<T, P, BFFT_PAIRS_HALF>(code, a, x, p, s);
    return append_code<T, P, BFFT_PAIRS_INTERLEAVED>(code, a, x, p, s);
}
template <typename T, typename Axes>
cudaError_t append_pack(int pack, int layout, int code, const AppendArgs& a, const Axes& x, const AppendPlan& p, cudaStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (pack == 8) return append_layout<T, 8>(layout, code, a, x, p, s);
    if (pack == 4) return append_layout<T, 4>(layout, code, a, x, p, s);
    if (pack == 2) return append_layout<T, 2>(layout, code, a, x, p, s);
    return append_layout<T, 1>(layout, code, a, x, p, s);
}

template <typename Axes>
cudaError_t launch_rotate(int64_t type, int pack, int layout, const RotateArgs& a, const Axes& x, dim3 grid, dim3 block,
                          cudaStream_t s) {
    return type == BFFT_F32   ? rotate_pack<float>(pack, layout, a, x, grid, block, s)
           : type == BFFT_F16 ? rotate_pack<__half>(pack, layout, a, x, grid, block, s)
                              : rotate_pack<__nv_bfloat16>(pack, layout, a, x, grid, block, s);
}
template <typename Axes>
cudaError_t launch_append(int64_t type, int pack, int layout, int code, const AppendArgs& a, const Axes& x,
                          const AppendPlan& p, cudaStream_t s) {
    return type == BFFT_F32   ? append_pack<float>(pack, layout, code, a, x, p, s)
           : type == BFFT_F16 ? append_pack<__half>(pack, layout, code, a, x, p, s)
                              : append_pack<__nv_bfloat16>(pack, layout, code, a, x, p, s);
}

// Compiled in bfft_rotary_axes.cu.
extern template cudaError_t launch_rotate(int64_t, int, int, const RotateArgs&, const AxisMap&, dim3, dim3, cudaStream_t);
extern template cudaError_t launch_append(int64_t, int, int, int, const AppendArgs&, const AxisMap&, const AppendPlan&,
                                          cudaStream_t);

}  // namespace bfft
