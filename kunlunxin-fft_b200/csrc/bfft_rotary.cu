// bfft_rotary.cu -- entry points of the rotation by position, of appending rotated keys
// (and values) to a paged 8-bit cache, and of reading such a cache back; the reading
// kernel, and the rotating ones (bfft_rotary.cuh) for one position a token.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <string>

#include "../../include/bfft.h"
#include "bfft_rotary.cuh"

using namespace bfft;

namespace bfft {

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

namespace {

// The axes of the pairs as the kernels take them.
bfft_status axis_map(const bfft_axes_desc* d, int64_t rotated, int64_t table_rows, AxisMap& m) {
    if (!d->axis) return fail(BFFT_ERR_VALUE, "null pointer");
    if (d->axes < 1 || d->axes > 4) return fail(BFFT_ERR_VALUE, "positions have 1 to 4 axes, got %lld", (long long)d->axes);
    if (table_rows > 0x7fffffffLL) return fail(BFFT_ERR_SHAPE, "bad table of %lld positions", (long long)table_rows);
    m = AxisMap{};
    m.axes = (int)d->axes;
    m.stride = d->pos_axis;
    const uint8_t* axis = static_cast<const uint8_t*>(d->axis);
    for (int64_t j = 0; j < rotated / 2; ++j) {
        if (axis[j] >= d->axes)
            return fail(BFFT_ERR_VALUE, "pair %lld is of axis %d, positions have %lld", (long long)j, (int)axis[j],
                        (long long)d->axes);
        m.of[j >> 4] |= (uint32_t)axis[j] << (2 * (j & 15));
    }
    return BFFT_OK;
}

bfft_status rotate_call(const bfft_rotate_desc* d, const bfft_axes_desc* axes, const void* x, const void* positions,
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
    AxisMap map;
    if (axes) {
        const bfft_status st = axis_map(axes, d->rotated, d->table_rows, map);
        if (st != BFFT_OK) return st;
    }
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
    return launched(axes ? launch_rotate(d->type, p, (int)d->layout, a, map, grid, block, s)
                         : launch_rotate(d->type, p, (int)d->layout, a, OneAxis{}, grid, block, s),
                    "rotate_positions");
}

bfft_status append_call(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs, const bfft_append_desc* d,
                        const bfft_axes_desc* axes, void* stream) {
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
    AxisMap map;
    if (axes) {
        if (!d->table || !d->positions) return fail(BFFT_ERR_VALUE, "axes need a table and positions");
        st = axis_map(axes, rotated, d->table_rows, map);
        if (st != BFFT_OK) return st;
    }
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
    return launched(axes ? launch_append(d->type, p, layout, code, a, map, plan, s)
                         : launch_append(d->type, p, layout, code, a, OneAxis{}, plan, s),
                    "cache_append");
}

}  // namespace

extern "C" bfft_status bfft_rotate_positions(const bfft_rotate_desc* d, const void* x, const void* positions,
                                             const void* table, void* y, void* stream) {
    return rotate_call(d, nullptr, x, positions, table, y, stream);
}

extern "C" bfft_status bfft_rotate_axes(const bfft_rotate_desc* d, const bfft_axes_desc* axes, const void* x,
                                        const void* positions, const void* table, void* y, void* stream) {
    if (!axes) return fail(BFFT_ERR_VALUE, "null pointer");
    return rotate_call(d, axes, x, positions, table, y, stream);
}

extern "C" bfft_status bfft_cache_append(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs,
                                         const bfft_append_desc* d, void* stream) {
    return append_call(cache, seqs, d, nullptr, stream);
}

extern "C" bfft_status bfft_cache_append_axes(const bfft_cache_desc* cache, const bfft_sequence_desc* seqs,
                                              const bfft_append_desc* d, const bfft_axes_desc* axes, void* stream) {
    if (!axes) return fail(BFFT_ERR_VALUE, "null pointer");
    return append_call(cache, seqs, d, axes, stream);
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
