// mi_cache.hip -- C ABI (include/mi_knn.h) of the 4-bit cache bank: argument checks, launch shapes, workspaces.
#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/mi_knn.h"
#include "cache_kernel.h"
#include "host_common.h"

namespace {

constexpr int64_t MAX_ROWS = (int64_t)1 << 30;

int width_of(int64_t dim)
{
    if (dim < 8 || dim > 256 || dim % 8) return 0;
    return dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
}

int check_cache(const mi_cache_t *c, const char *who)
{
    if (!c) return fail(MI_ERR_ARG, "%s: null cache", who);
    if (!c->key || !c->key_scale || !c->value || !c->value_scale || !c->weight || !c->position || !c->length || !c->seen)
        return fail(MI_ERR_ARG, "%s: null pointer in the cache", who);
    if (((uintptr_t)c->key | (uintptr_t)c->key_scale | (uintptr_t)c->value | (uintptr_t)c->value_scale | (uintptr_t)c->weight | (uintptr_t)c->position) & 15)
        return fail(MI_ERR_ARG, "%s: the cache's buffers must be 16-byte aligned", who);
    if (c->batch < 1 || c->heads < 1 || c->batch > (1 << 24) || c->heads > (1 << 24) || c->batch * c->heads > (1 << 24))
        return fail(MI_ERR_ARG, "%s: bad shape batch=%lld heads=%lld", who, (long long)c->batch, (long long)c->heads);
    if (!width_of(c->dim)) return fail(MI_ERR_UNSUPPORTED, "%s: dim=%lld must be a multiple of 8 in [8, 256]", who, (long long)c->dim);
    if (c->limit < 1 || c->rows < c->limit || c->rows % 64 || c->rows > MAX_ROWS)
        return fail(MI_ERR_ARG, "%s: bad capacity rows=%lld limit=%lld", who, (long long)c->rows, (long long)c->limit);
    return MI_OK;
}

mi::CacheView view(const mi_cache_t *c)
{
    mi::CacheView v{};
    v.key = c->key, v.key_scale = c->key_scale, v.value = c->value, v.value_scale = c->value_scale;
    v.weight = c->weight, v.position = c->position, v.length = c->length, v.seen = c->seen;
    v.batch = (int)c->batch, v.heads = (int)c->heads, v.dim = (int)c->dim, v.rows = (int)c->rows, v.limit = (int)c->limit;
    return v;
}

// Byte strides of a [sequence][head][row][dim] tensor; every row has to start on 16 bytes.
int check_rows(const char *who, const char *what, const void *p, const int64_t *strides, int dtype, long long (&out)[3])
{
    if (!p || !strides) return fail(MI_ERR_ARG, "%s: null %s", who, what);
    const int64_t es = dtype == MI_F32 ? 4 : 2;
    if ((uintptr_t)p & 15) return fail(MI_ERR_ARG, "%s: %s must be 16-byte aligned", who, what);
    for (int i = 0; i < 3; ++i) {
        if (strides[i] < 0 || strides[i] * es % 16) return fail(MI_ERR_ARG, "%s: strides of %s must be multiples of 16 bytes", who, what);
        out[i] = strides[i] * es;
    }
    return MI_OK;
}

#define MI_TRY(expr)            \
    do {                        \
        const int rc_ = (expr); \
        if (rc_) return rc_;    \
    } while (0)

int check_grid(const char *who, int64_t blocks)
{
    return blocks > INT32_MAX ? fail(MI_ERR_UNSUPPORTED, "%s: too many rows for one launch", who) : (int)MI_OK;
}

// Launch shape of the attention: tiles of 16 MT query rows, and pieces of the bank's rows so that the card is filled when
// there are few of them.
struct AttendPlan {
    int64_t R, mt, tiles, nsplit;
    bool tiled;                              // 32 `waves` query rows a workgroup through shared memory, not 16 mt straight from memory
    int waves;
    bool uneven;                             // tiled, causal, mostly its own rows: the first pieces are longer than the last
    int64_t chunks, rsplit;                  // weights: workgroups a (sequence, head) along the bank, and along the query rows
    bool scores;                             // weights: from scores left behind, not from a second product
    size_t off_ml, off_norm, off_scores, off_w, total;
};

// How long the tiled form takes, in tiles of 128 rows of the bank by 256 query rows, bf16 and 128 dims, on one compute unit (3.8 us),
// with `waves` waves a workgroup and the bank in `nsplit` pieces: the larger of an even share and the longest piece where pieces
// differ (causal, mostly its own rows), whole rounds of equal pieces otherwise.  Measured: other widths and types cost `work`
// (1.2 us a step of a workgroup of four waves at bf16 and 128 dims, 2.0 at 256, 1.9 / 2.5 for fp16 / fp32, 1.6 for fp32 at 64); four
// waves need 0.31 for a quarter of a tile alone on a unit, 0.2775 beside another workgroup, which fp32 and 256 dims leave no room for;
// getting started and leaving costs about 1.3; joining pieces one, and the writing and reading of their sums.
double tiled_cost(int64_t bh, int64_t R, int width, int dtype, int64_t span, double seen, bool uneven, int waves, int64_t nsplit)
{
    const int64_t tiles = ceil_div(R, 32 * waves), units = ceil_div(span, 16 * waves), per = ceil_div(units, nsplit), all = bh * tiles * nsplit;
    const bool pairs = waves == 4 && dtype != MI_F32 && width < 256;
    const double pieces = dtype == MI_BF16 ? 1 : dtype == MI_F16 ? 2 : 3, work = 0.37 + 0.63 * width / 128 * pieces;
    const double alone = (waves == 8 ? 1.0 : 0.31) * work, busy = pairs ? 0.2775 * work : alone, over = 1.3;
    const double share = seen / (double)span, groups = (double)(bh * tiles);
    const int64_t slots = pairs ? 512 : 256, turns = ceil_div(all, 256);
    double t;
    if (uneven) {
        const bool few = groups * ((double)nsplit * share + 0.5) <= 288;      // workgroups that have anything to do: hardly two on a unit
        t = std::max(groups * ((double)units * share * busy / 256 + over * std::max(1.0, (double)nsplit * share) / (double)slots),
                     (double)per * (few ? alone : pairs ? 1.6 * busy : busy) + over);
    }
    else t = (double)(turns * per) * (turns == 1 ? alone : busy) + (double)ceil_div(all, slots) * over;
    return t + (nsplit > 1 ? 1.0 + (double)(bh * R * nsplit) * width * 8 / (4.5e12 * 3.8e-6) : 0.0);
}

AttendPlan attend_plan(const mi_cache_t *c, int dtype, int64_t T, int64_t group, int64_t span, int causal, int accumulate)
{
    AttendPlan a{};
    a.R = T * group;
    a.mt = a.R <= 16 || width_of(c->dim) == 256 ? 1 : 2;         // 256 dims: the sums of two tiles do not fit two waves a SIMD
    const int64_t bh = c->batch * c->heads;
    span = span < 1 ? 1 : span > c->limit ? c->limit : span;
    a.tiled = a.R > 32;
    if (a.tiled) {
        const double seen = causal ? std::max((double)span * 0.5, (double)span - (double)T * 0.5) : (double)span;
        const int64_t most = std::min<int64_t>(ceil_div(span, 256), mi::CACHE_MAX_SPLIT);
        a.uneven = causal && 2 * T > span;
        double best = 1e300;
        for (int waves = dtype == MI_BF16 && width_of(c->dim) < 256 ? 8 : 4; waves >= 4; waves -= 4)
            for (int64_t ns = 1; ns <= most; ++ns) {
                const double t = tiled_cost(bh, a.R, width_of(c->dim), dtype, span, seen, a.uneven, waves, ns);
                if (t < best) best = t, a.waves = waves, a.nsplit = ns;
            }
        a.tiles = ceil_div(a.R, 32 * a.waves);
    } else {
        a.tiles = ceil_div(a.R, 16 * a.mt);
        const int64_t ns = ceil_div(512, bh * a.tiles), most = std::min<int64_t>(ceil_div(span, 512), mi::CACHE_MAX_SPLIT);
        a.nsplit = ns > most ? most : ns;
    }
    const int64_t rows = c->batch * c->heads * a.R;
    size_t at = 0;
    if (a.nsplit > 1) {
        at = (size_t)(a.nsplit * rows * width_of(c->dim) * 4);
        a.off_ml = at;
        at += (size_t)round_up(a.nsplit * rows * 8, 256);
    }
    a.off_norm = at;
    if (accumulate) at += (size_t)round_up(rows * 8, 256);
    // A slot's attention sum costs 8 R bytes if its scores are written and read again, or its key, W / 2 + W / 32 bytes, and the
    // product once more.  Scores are laid out by the capacity (a captured call may see longer sequences than `span`).
    const int64_t score_bytes = rows * c->rows * 4;
    a.scores = accumulate && a.mt == 1 && 8 * a.R <= width_of(c->dim) / 2 && score_bytes <= ((int64_t)1 << 30);
    a.chunks = ceil_div(span, a.scores ? 1024 : a.tiled ? 256 : 128);
    a.rsplit = 1;
    if (accumulate && a.tiled) {
        a.rsplit = std::min<int64_t>(std::max<int64_t>(1, 512 / (bh * a.chunks)), ceil_div(a.R, 256));
        while (a.rsplit > 1 && a.rsplit * bh * c->rows * 4 > ((int64_t)1 << 30)) --a.rsplit;
        a.off_w = at;
        if (a.rsplit > 1) at += (size_t)(a.rsplit * bh * c->rows * 4);
    }
    a.off_scores = at;
    if (a.scores) at += (size_t)score_bytes;
    a.total = at < 256 ? 256 : at;
    return a;
}

template <int DT, int NB, int WAVES>
hipError_t launch_tile(const mi::CacheAttendParams &p, dim3 grid, hipStream_t s)
{
    const size_t lds = (size_t)NB * WAVES * 4 * 1024;      // two tiles of 16 WAVES rows, keys and values in bf16
    static std::atomic<uint64_t> done{0};
    const hipError_t e = ensure_dynamic_lds(mi::cache_attend_tile_kernel<DT, NB, WAVES>, lds, done);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((mi::cache_attend_tile_kernel<DT, NB, WAVES>), grid, dim3(64 * WAVES), lds, s, p);
    return hipGetLastError();
}

template <int DT, int NB>
hipError_t launch_attend(const mi::CacheAttendParams &p, const AttendPlan &a, int accumulate, hipStream_t s)
{
    const int64_t bh = (int64_t)p.c.batch * p.c.heads;
    const dim3 grid((unsigned)(bh * a.tiles * a.nsplit));
    if (a.tiled) {
        hipError_t e;
        if constexpr (DT == mi::CACHE_BF16 && NB < 8) e = a.waves == 8 ? launch_tile<DT, NB, 8>(p, grid, s) : launch_tile<DT, NB, 4>(p, grid, s);
        else e = launch_tile<DT, NB, 4>(p, grid, s);
        if (e != hipSuccess) return e;
    } else if (a.mt == 1) hipLaunchKernelGGL((mi::cache_attend_kernel<DT, NB, 1>), grid, dim3(256), 0, s, p);
    if constexpr (NB < 8)
        if (!a.tiled && a.mt == 2) hipLaunchKernelGGL((mi::cache_attend_kernel<DT, NB, 2>), grid, dim3(256), 0, s, p);
    if (a.nsplit > 1 && a.nsplit <= mi::CACHE_FEW_SPLITS)
        hipLaunchKernelGGL((mi::cache_join_few_kernel<DT, 32 * NB>), dim3((unsigned)ceil_div(bh * a.R * (4 * NB), 256)), dim3(256), 0, s, p);
    else if (a.nsplit > 1)
        hipLaunchKernelGGL((mi::cache_join_kernel<DT, 32 * NB>), dim3((unsigned)(bh * a.R)), dim3(256), 0, s, p);
    if (a.scores) hipLaunchKernelGGL(mi::cache_weigh_scores_kernel, dim3((unsigned)(bh * a.chunks)), dim3(256), 0, s, p);
    else if (accumulate && a.tiled) {
        hipLaunchKernelGGL((mi::cache_weigh_tile_kernel<DT, NB>), dim3((unsigned)(bh * a.chunks * a.rsplit)), dim3(512), 0, s, p);
        if (a.rsplit > 1) hipLaunchKernelGGL(mi::cache_weigh_add_kernel, dim3((unsigned)(bh * a.chunks)), dim3(256), 0, s, p);
    } else if (accumulate) hipLaunchKernelGGL((mi::cache_weigh_kernel<DT, NB>), dim3((unsigned)(bh * a.chunks)), dim3(256), 0, s, p);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_attend_w(int width, const mi::CacheAttendParams &p, const AttendPlan &a, int accumulate, hipStream_t s)
{
    return width == 64 ? launch_attend<DT, 2>(p, a, accumulate, s) : width == 128 ? launch_attend<DT, 4>(p, a, accumulate, s)
                                                                                         : launch_attend<DT, 8>(p, a, accumulate, s);
}

template <int DT, int W>
void launch_push_w(const mi::PushParams &p, hipStream_t s)
{
    const int64_t lanes = (int64_t)p.c.heads * p.T * (W / 4);                    // of one sequence
    if (lanes <= 2048) {
        hipLaunchKernelGGL((mi::cache_push_kernel<DT, W, true>), dim3((unsigned)p.c.batch), dim3(256), 0, s, p);
        return;
    }
    const int64_t stretches = ceil_div(p.T, 1024 / (W / 4));                     // as the kernel cuts a head's rows
    hipLaunchKernelGGL((mi::cache_push_kernel<DT, W, false>), dim3((unsigned)((int64_t)p.c.batch * p.c.heads * stretches)), dim3(256), 0, s, p);
    hipLaunchKernelGGL(mi::cache_advance_kernel, dim3((unsigned)ceil_div(p.c.batch, 64)), dim3(64), 0, s, p);
}

template <int DT>
void launch_push(int width, const mi::PushParams &p, hipStream_t s)
{
    if (width == 64) launch_push_w<DT, 64>(p, s);
    else if (width == 128) launch_push_w<DT, 128>(p, s);
    else launch_push_w<DT, 256>(p, s);
}

bool known_dtype(int dtype) { return dtype == MI_F32 || dtype == MI_BF16 || dtype == MI_F16; }

}  // namespace

extern "C" {

int64_t mi_cache_width(int64_t dim) { return width_of(dim); }

int mi_cache_push(const mi_cache_t *cache, const void *key, const int64_t *key_strides, const void *value, const int64_t *value_strides,
                  int dtype, int64_t T, const int32_t *counts, void *held_key, void *held_value, mi_stream_t stream)
{
    MI_TRY(check_cache(cache, "mi_cache_push"));
    if (!known_dtype(dtype)) return fail(MI_ERR_ARG, "mi_cache_push: unknown dtype %d", dtype);
    if (T < 0 || T > MAX_ROWS) return fail(MI_ERR_ARG, "mi_cache_push: bad T=%lld", (long long)T);
    if (!held_key != !held_value) return fail(MI_ERR_ARG, "mi_cache_push: held_key and held_value go together");
    if (((uintptr_t)held_key | (uintptr_t)held_value) & 15) return fail(MI_ERR_ARG, "mi_cache_push: held rows must be 16-byte aligned");
    if (T == 0) return MI_OK;
    mi::PushParams p{};
    MI_TRY(check_rows("mi_cache_push", "key", key, key_strides, dtype, p.key_s));
    MI_TRY(check_rows("mi_cache_push", "value", value, value_strides, dtype, p.value_s));
    const int width = width_of(cache->dim);
    MI_TRY(check_grid("mi_cache_push", ceil_div(cache->batch * cache->heads * T * (width / 4), 256)));
    p.c = view(cache);
    p.key = (const char *)key, p.value = (const char *)value;
    p.counts = counts;
    p.T = (int)T;
    p.held_key = (char *)held_key, p.held_value = (char *)held_value;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MI_F32) launch_push<mi::CACHE_F32>(width, p, s);
    else if (dtype == MI_BF16) launch_push<mi::CACHE_BF16>(width, p, s);
    else launch_push<mi::CACHE_F16>(width, p, s);
    HIP_CHECK(hipGetLastError());
    return MI_OK;
}

int mi_cache_longest(const mi_cache_t *cache, const int32_t *counts, int64_t T, int32_t *out, mi_stream_t stream)
{
    MI_TRY(check_cache(cache, "mi_cache_longest"));
    if (!out) return fail(MI_ERR_ARG, "mi_cache_longest: null pointer");
    if (T < 0 || T > MAX_ROWS) return fail(MI_ERR_ARG, "mi_cache_longest: bad T=%lld", (long long)T);
    mi::PushParams p{};
    p.c = view(cache);
    p.counts = counts;
    p.T = (int)T;
    hipLaunchKernelGGL(mi::cache_longest_kernel, dim3(1), dim3(256), 0, (hipStream_t)stream, p, out);
    HIP_CHECK(hipGetLastError());
    return MI_OK;
}

int mi_cache_in_order(const mi_cache_t *cache, const int32_t *counts, int64_t T, int32_t *out, mi_stream_t stream)
{
    MI_TRY(check_cache(cache, "mi_cache_in_order"));
    if (!out) return fail(MI_ERR_ARG, "mi_cache_in_order: null pointer");
    if (T < 0 || T > MAX_ROWS) return fail(MI_ERR_ARG, "mi_cache_in_order: bad T=%lld", (long long)T);
    mi::PushParams p{};
    p.c = view(cache);
    p.counts = counts;
    p.T = (int)T;
    hipLaunchKernelGGL(mi::cache_order_start_kernel, dim3(1), dim3(1), 0, (hipStream_t)stream, out);
    hipLaunchKernelGGL(mi::cache_order_kernel, dim3((unsigned)(cache->batch * cache->heads)), dim3(256), 0, (hipStream_t)stream, p, out);
    HIP_CHECK(hipGetLastError());
    return MI_OK;
}

int mi_cache_trim(const mi_cache_t *cache, const int32_t *lengths, int64_t length, mi_stream_t stream)
{
    MI_TRY(check_cache(cache, "mi_cache_trim"));
    if (!lengths && (length < 0 || length > INT32_MAX)) return fail(MI_ERR_ARG, "mi_cache_trim: bad length %lld", (long long)length);
    hipLaunchKernelGGL(mi::cache_trim_kernel, dim3((unsigned)cache->batch), dim3(mi::TRIM_THREADS), 0, (hipStream_t)stream, view(cache), lengths, (int)length,
                       width_of(cache->dim));
    HIP_CHECK(hipGetLastError());
    return MI_OK;
}

int mi_cache_read(const mi_cache_t *cache, void *key, void *value, mi_stream_t stream)
{
    MI_TRY(check_cache(cache, "mi_cache_read"));
    if (!key || !value || (((uintptr_t)key | (uintptr_t)value) & 15)) return fail(MI_ERR_ARG, "mi_cache_read: key and value must be 16-byte aligned");
    const int width = width_of(cache->dim);
    const int64_t chunks = ceil_div(cache->limit, mi::CACHE_READ_TURNS * (1024 / width)), blocks = cache->batch * cache->heads * chunks;
    MI_TRY(check_grid("mi_cache_read", blocks));
    const dim3 grid((unsigned)blocks);
    hipStream_t s = (hipStream_t)stream;
    const mi::CacheView v = view(cache);
    if (width == 64) hipLaunchKernelGGL(mi::cache_read_kernel<64>, grid, dim3(256), 0, s, v, (uint4 *)key, (uint4 *)value, (int)chunks);
    else if (width == 128) hipLaunchKernelGGL(mi::cache_read_kernel<128>, grid, dim3(256), 0, s, v, (uint4 *)key, (uint4 *)value, (int)chunks);
    else hipLaunchKernelGGL(mi::cache_read_kernel<256>, grid, dim3(256), 0, s, v, (uint4 *)key, (uint4 *)value, (int)chunks);
    HIP_CHECK(hipGetLastError());
    return MI_OK;
}

size_t mi_cache_attend_workspace_bytes(const mi_cache_t *cache, int dtype, int64_t T, int64_t group, int64_t span, int causal, int accumulate)
{
    if (check_cache(cache, "mi_cache_attend_workspace_bytes") || !known_dtype(dtype) || T < 1 || group < 1 || group > 65536 || T > MAX_ROWS / group) return 0;
    return attend_plan(cache, dtype, T, group, span, causal, accumulate).total;
}

int mi_cache_attend(const mi_cache_t *cache, const void *query, const int64_t *query_strides, void *out, const int64_t *out_strides,
                    int dtype, int64_t T, int64_t group, const int32_t *counts, float scale, int causal, int accumulate, int64_t span,
                    void *workspace, size_t workspace_bytes, mi_stream_t stream)
{
    MI_TRY(check_cache(cache, "mi_cache_attend"));
    if (!known_dtype(dtype)) return fail(MI_ERR_ARG, "mi_cache_attend: unknown dtype %d", dtype);
    if (T < 0 || group < 1 || group > 65536 || T > MAX_ROWS / group) return fail(MI_ERR_ARG, "mi_cache_attend: bad shape T=%lld group=%lld", (long long)T, (long long)group);
    // a scale that the base 2 exponent cannot hold would make NaN of masked scores
    if (!(scale * mi::CACHE_LOG2E >= FLT_MIN) || !isfinite(scale * mi::CACHE_LOG2E)) return fail(MI_ERR_ARG, "mi_cache_attend: scale must be positive and finite, got %g", (double)scale);
    if (T == 0) return MI_OK;
    mi::CacheAttendParams p{};
    MI_TRY(check_rows("mi_cache_attend", "query", query, query_strides, dtype, p.q_s));
    MI_TRY(check_rows("mi_cache_attend", "out", out, out_strides, dtype, p.out_s));
    const AttendPlan a = attend_plan(cache, dtype, T, group, span, causal, accumulate);
    if (!workspace || ((uintptr_t)workspace & 15)) return fail(MI_ERR_ARG, "mi_cache_attend: workspace must be 16-byte aligned");
    if (workspace_bytes < a.total) return fail(MI_ERR_WORKSPACE, "mi_cache_attend: workspace %zu < required %zu", workspace_bytes, a.total);
    const int width = width_of(cache->dim);
    const int64_t bh = cache->batch * cache->heads;
    MI_TRY(check_grid("mi_cache_attend", bh * a.tiles * a.nsplit));
    MI_TRY(check_grid("mi_cache_attend", bh * a.R));
    MI_TRY(check_grid("mi_cache_attend", bh * a.chunks * a.rsplit));
    p.c = view(cache);
    p.q = (const char *)query;
    p.out = (char *)out;
    p.counts = counts;
    p.T = (int)T, p.G = (int)group, p.causal = causal ? 1 : 0;
    p.R = (int)a.R, p.tiles = (int)a.tiles, p.nsplit = (int)a.nsplit, p.mixed = a.uneven, p.chunks = (int)a.chunks;
    p.c2 = scale * mi::CACHE_LOG2E;
    p.part = (float *)workspace;
    p.part_ml = (float2 *)((char *)workspace + a.off_ml);
    p.rsplit = (int)a.rsplit;
    p.part_w = (float *)((char *)workspace + a.off_w);
    p.scores = a.scores ? (float *)((char *)workspace + a.off_scores) : nullptr;
    p.norm = accumulate ? (float2 *)((char *)workspace + a.off_norm) : nullptr;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MI_F32) HIP_CHECK(launch_attend_w<mi::CACHE_F32>(width, p, a, accumulate, s));
    else if (dtype == MI_BF16) HIP_CHECK(launch_attend_w<mi::CACHE_BF16>(width, p, a, accumulate, s));
    else HIP_CHECK(launch_attend_w<mi::CACHE_F16>(width, p, a, accumulate, s));
    return MI_OK;
}

size_t mi_cache_evict_workspace_bytes(const mi_cache_t *cache, int64_t keep)
{
    if (check_cache(cache, "mi_cache_evict_workspace_bytes") || keep < 1) return 0;
    return (size_t)(round_up(cache->batch * cache->heads * 4, 256) + cache->batch * cache->heads * keep * 8);
}

int mi_cache_evict(const mi_cache_t *cache, const mi_cache_t *into, int64_t keep, int64_t recent, int64_t span,
                   void *workspace, size_t workspace_bytes, mi_stream_t stream)
{
    MI_TRY(check_cache(cache, "mi_cache_evict"));
    if (into && into != cache) {
        MI_TRY(check_cache(into, "mi_cache_evict"));
        if (into->batch != cache->batch || into->heads != cache->heads || into->dim != cache->dim) return fail(MI_ERR_ARG, "mi_cache_evict: the two banks differ in batch, heads or dim");
        if (into->key == cache->key || into->length == cache->length) return fail(MI_ERR_ARG, "mi_cache_evict: the two banks share memory");
    } else into = cache;
    if (keep < 1 || keep > into->limit) return fail(MI_ERR_ARG, "mi_cache_evict: keep=%lld outside [1, %lld]", (long long)keep, (long long)into->limit);
    if (recent < 0 || recent > keep) return fail(MI_ERR_ARG, "mi_cache_evict: recent=%lld outside [0, keep=%lld]", (long long)recent, (long long)keep);
    if (!workspace || ((uintptr_t)workspace & 15)) return fail(MI_ERR_ARG, "mi_cache_evict: workspace must be 16-byte aligned");
    const size_t need = mi_cache_evict_workspace_bytes(cache, keep);
    if (workspace_bytes < need) return fail(MI_ERR_WORKSPACE, "mi_cache_evict: workspace %zu < required %zu", workspace_bytes, need);
    const int64_t bh = cache->batch * cache->heads;
    const int width = width_of(cache->dim);
    mi::EvictParams p{};
    p.c = view(cache), p.into = view(into);
    p.keep = (int)keep, p.recent = (int)recent, p.in_place = into == cache;
    p.count = (int *)workspace;
    p.pairs = (int2 *)((char *)workspace + round_up(bh * 4, 256));
    hipStream_t s = (hipStream_t)stream;
    const int64_t resident = std::min<int64_t>(round_up(span < 1 ? 1 : span > cache->limit ? cache->limit : span, 64), mi::EVICT_RESIDENT);
    static std::atomic<uint64_t> done{0};
    HIP_CHECK(ensure_dynamic_lds(mi::cache_select_kernel, (size_t)mi::EVICT_RESIDENT * 4, done));
    hipLaunchKernelGGL(mi::cache_select_kernel, dim3((unsigned)bh), dim3(mi::EVICT_THREADS), (size_t)resident * 4, s, p, (int)resident);
    HIP_CHECK(hipGetLastError());
    // a workgroup copies 2048 / width rows a turn; as many of them as the card holds at once are enough
    const int64_t turn = 2048 / width;
    int64_t chunks = ceil_div(keep, turn);
    const int64_t fill = ceil_div(4096, bh);
    if (chunks > fill) chunks = fill;
    const dim3 grid((unsigned)(bh * chunks));
    if (width == 64) hipLaunchKernelGGL(mi::cache_move_kernel<64>, grid, dim3(256), 0, s, p, (int)chunks);
    else if (width == 128) hipLaunchKernelGGL(mi::cache_move_kernel<128>, grid, dim3(256), 0, s, p, (int)chunks);
    else hipLaunchKernelGGL(mi::cache_move_kernel<256>, grid, dim3(256), 0, s, p, (int)chunks);
    HIP_CHECK(hipGetLastError());
    return MI_OK;
}

}  // extern "C"
