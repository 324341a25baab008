// Global gradient norm over a set of tensors, clipping by it, and the optimizer steps that take the factor from device
// memory.  Compiled with -fmad=false like rowops.cu: the steps round where znn_sgd_step and znn_adam_step do.
//
// Bound by HBM: 4 bytes per gradient for the norm, 20 (SGD with momentum) or 28 (Adam) for a step.  Measured on a B200 whose copies
// run at 6548 GB/s: norm of 98 million floats 61 us, 6.5 TB/s; Adam step on them 395 us, 6.8 TB/s of the 2.69 GB that cross HBM (the
// gradients that the norm read last come from L2); both as called 470 us.  Norm and SGD step of them 234 us, with momentum 355 (floors 180
// and 300); clipping them in place 125 us, 6.3 TB/s, with the norm 196 (180); norm and clipping of six tensors, 109 thousand floats, 6.4 us.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>
#include <new>
#include <utility>
#include <vector>

#include "overlap.cuh"

namespace cg = cooperative_groups;

namespace znn {

constexpr int kNormThreads = 512;
constexpr int kNormQuads = 4;                                  // 16-byte loads that a thread has under way
constexpr int kNormTile = 4 * kNormThreads * kNormQuads;       // floats of one tensor that a block takes at a time
constexpr int kNormHead = 4;                                   // floats of `result` before the partial sums (16-byte aligned doubles)
constexpr int kNormBlocks = (ZNN_GRAD_NORM_FLOATS - kNormHead) / 2;

// The tensors of one launch: they travel as a kernel argument (at most 32764 bytes).  Small sets take a small table, whose copy
// costs the launch less.
template <int Cap>
struct TensorTable {
    const float* data[Cap];
    long long count[Cap];
    int first_tile[Cap + 1];   // tiles before tensor i
    int n;
};
constexpr int kSmallTable = 16, kMiddleTable = 200, kLargeTable = 1000;

// The floats of one tile: whole 16-byte quads, kNormQuads per thread, and up to three floats before and after them, one each for
// a few threads, since a tensor may start at any float.
struct Tile {
    float* x;
    int n, head, quads;

    template <int Cap>
    __device__ __forceinline__ Tile(const TensorTable<Cap>& t, int tile)
    {
        int lo = 0, hi = t.n - 1;   // the last tensor whose first tile is not behind this one
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (t.first_tile[mid] <= tile) lo = mid;
            else hi = mid - 1;
        }
        const long long begin = (long long)(tile - t.first_tile[lo]) * kNormTile;
        x = const_cast<float*>(t.data[lo]) + begin;
        n = (int)min((long long)kNormTile, t.count[lo] - begin);
        head = min(n, (int)(0u - (unsigned)((uintptr_t)x >> 2)) & 3);
        quads = (n - head) >> 2;
    }
    __device__ __forceinline__ float4* quad(int q) const { return reinterpret_cast<float4*>(x + head) + q; }
    // the thread's float outside the quads, or -1
    __device__ __forceinline__ int extra() const
    {
        const int i = threadIdx.x, after = head + 4 * quads + i - 4;
        return i < head ? i : i >= 4 && after < n ? after : -1;
    }
};

// Squares of the tiles first, first + step, ...: fp64 from the first product on, so that no finite gradient overflows or vanishes
// and sums of any length keep their digits.  A conversion and a fused multiply-add per float cost nothing beside the loads (the
// schedulers issue in 37 % of the cycles); what counts is that the next tile's loads are under way meanwhile (24 layers of width
// 1000: 148 us without, 135 us with).
template <int Cap>
__device__ __forceinline__ double squares(const TensorTable<Cap>& t, int first, int step)
{
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    const int tiles = t.first_tile[t.n];
    float4 v[kNormQuads];
    float e = 0.0f;
    auto load = [&](int i) {
        const Tile tile(t, i);
#pragma unroll
        for (int k = 0; k < kNormQuads; k++) {
            const int q = threadIdx.x + k * kNormThreads;
            v[k] = q < tile.quads ? *tile.quad(q) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        const int c = tile.extra();
        e = c >= 0 ? tile.x[c] : 0.0f;
    };
    if (first < tiles) load(first);
    for (int i = first; i < tiles; i += step) {
        float4 u[kNormQuads];
#pragma unroll
        for (int k = 0; k < kNormQuads; k++) u[k] = v[k];
        const double f = e;
        if (i + step < tiles) load(i + step);   // under way while this tile's products are made
#pragma unroll
        for (int k = 0; k < kNormQuads; k++) {
            const double a = u[k].x, b = u[k].y, c = u[k].z, d = u[k].w;
            s[0] = fma(a, a, s[0]);
            s[1] = fma(b, b, s[1]);
            s[2] = fma(c, c, s[2]);
            s[3] = fma(d, d, s[3]);
        }
        s[0] = fma(f, f, s[0]);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

__device__ __forceinline__ void write_result(double sum, float grad_scale, float max_norm, float* result)
{
    const double norm = fabs((double)grad_scale) * sqrt(sum);
    result[0] = (float)norm;
    // (a factor that fp32 would round to 0 is its smallest number: 0 says that there is no finite norm)
    result[1] = !isfinite(norm) ? 0.0f : norm > (double)max_norm ? fmaxf((float)((double)max_norm / norm), 1.4e-45f) : 1.0f;
}

// partial[block] (+)= squares of the block's tiles
template <int Cap>
__global__ void __launch_bounds__(kNormThreads)
norm_partial_kernel(const __grid_constant__ TensorTable<Cap> t, double* __restrict__ partial, int add)
{
    __shared__ double sh[kNormThreads / 32];
    wait_for_previous_kernel();
    const double s = block_sum(squares(t, blockIdx.x, gridDim.x), sh);
    if (threadIdx.x == 0) partial[blockIdx.x] = add ? partial[blockIdx.x] + s : s;
}

__global__ void __launch_bounds__(kNormThreads)
norm_finish_kernel(const double* __restrict__ partial, int blocks, float grad_scale, float max_norm, float* __restrict__ result)
{
    __shared__ double sh[kNormThreads / 32];
    wait_for_previous_kernel();
    double s = 0.0;
    for (int i = threadIdx.x; i < blocks; i += kNormThreads) s += partial[i];
    s = block_sum(s, sh);
    if (threadIdx.x == 0) write_result(s, grad_scale, max_norm, result);
}

// A small set in one launch of one cluster of eight blocks.
template <int Cap>
__global__ void __launch_bounds__(kNormThreads) __cluster_dims__(8, 1, 1)
norm_small_kernel(const __grid_constant__ TensorTable<Cap> t, float grad_scale, float max_norm, float* __restrict__ result)
{
    __shared__ double sh[kNormThreads / 32], sh_all[8];
    cg::cluster_group cluster = cg::this_cluster();
    auto began = cluster.barrier_arrive();
    wait_for_previous_kernel();
    const double s = block_sum(squares(t, blockIdx.x, 8), sh);
    cluster.barrier_wait(std::move(began));   // the first block runs: its memory may be written to
    if (threadIdx.x == 0) *cluster.map_shared_rank(sh_all + blockIdx.x, 0) = s;
    auto written = cluster.barrier_arrive();
    if (blockIdx.x != 0) return;
    cluster.barrier_wait(std::move(written));
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int i = 0; i < 8; i++) sum += sh_all[i];
        write_result(sum, grad_scale, max_norm, result);
    }
}

template <int Cap>
__global__ void __launch_bounds__(kNormThreads)
clip_kernel(const __grid_constant__ TensorTable<Cap> t, const float* __restrict__ result)
{
    wait_for_previous_kernel();
    const float c = result[1];
    if (c == 1.0f || c == 0.0f) return;
    // from the last tile on: what the norm read last is still in L2
    for (int i = t.first_tile[t.n] - 1 - blockIdx.x; i >= 0; i -= gridDim.x) {
        const Tile tile(t, i);
        float4 v[kNormQuads];
#pragma unroll
        for (int k = 0; k < kNormQuads; k++) {
            const int q = threadIdx.x + k * kNormThreads;
            if (q < tile.quads) v[k] = *tile.quad(q);
        }
#pragma unroll
        for (int k = 0; k < kNormQuads; k++) {
            const int q = threadIdx.x + k * kNormThreads;
            if (q < tile.quads) *tile.quad(q) = make_float4(v[k].x * c, v[k].y * c, v[k].z * c, v[k].w * c);
        }
        const int e = tile.extra();
        if (e >= 0) tile.x[e] *= c;
    }
}

// ---- the steps: round where sgd_kernel and adam_kernel (rowops.cu) do --------------------------------------------------
struct SgdStep {
    float lr, momentum;
    template <bool Momentum>
    __device__ __forceinline__ void apply(float& w, float g, float& v) const
    {
        if (Momentum) {
            v = momentum * v + lr * g;
            w -= v;
        } else {
            w -= lr * g;
        }
    }
};

struct AdamStep {
    float lr_t, beta1, beta2, eps;
    __device__ __forceinline__ void apply(float& w, float g, float& m, float& v) const
    {
        m = beta1 * m + (1.0f - beta1) * g;
        v = beta2 * v + (1.0f - beta2) * g * g;
        w -= lr_t * m / (sqrtf(v) + eps);
    }
};

constexpr int kStepThreads = 256;

// Four floats of every array per thread where they are 16-byte aligned, one otherwise; one pass from the end: the gradients that
// the norm read last are still in L2 (everything else streams past it).
template <bool Momentum, bool Quads>
__global__ void __launch_bounds__(kStepThreads)
sgd_clipped_kernel(float* __restrict__ w, const float* __restrict__ g, float* __restrict__ v, SgdStep step, float grad_scale,
                   const float* __restrict__ result, size_t n)
{
    wait_for_previous_kernel();
    const float c = result[1];
    if (c == 0.0f) return;
    const float scale = grad_scale * c;
    const size_t unit = (size_t)(gridDim.x - 1 - blockIdx.x) * kStepThreads + threadIdx.x;
    float none = 0.0f;
    if (Quads && 4 * unit + 4 <= n) {
        float4 a = __ldcs(reinterpret_cast<const float4*>(w) + unit), d = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float4 b = reinterpret_cast<const float4*>(g)[unit];
        if (Momentum) d = __ldcs(reinterpret_cast<const float4*>(v) + unit);
        step.apply<Momentum>(a.x, b.x * scale, d.x);
        step.apply<Momentum>(a.y, b.y * scale, d.y);
        step.apply<Momentum>(a.z, b.z * scale, d.z);
        step.apply<Momentum>(a.w, b.w * scale, d.w);
        if (Momentum) __stcs(reinterpret_cast<float4*>(v) + unit, d);
        __stcs(reinterpret_cast<float4*>(w) + unit, a);
    } else {
        for (size_t i = Quads ? 4 * unit : unit; i < n && i < (Quads ? 4 * unit + 4 : unit + 1); i++)
            step.apply<Momentum>(w[i], g[i] * scale, Momentum ? v[i] : none);
    }
}

template <bool Quads>
__global__ void __launch_bounds__(kStepThreads)
adam_clipped_kernel(float* __restrict__ w, const float* __restrict__ g, float* __restrict__ m, float* __restrict__ v, AdamStep step,
                    float grad_scale, const float* __restrict__ result, size_t n)
{
    wait_for_previous_kernel();
    const float c = result[1];
    if (c == 0.0f) return;
    const float scale = grad_scale * c;
    const size_t unit = (size_t)(gridDim.x - 1 - blockIdx.x) * kStepThreads + threadIdx.x;
    if (Quads && 4 * unit + 4 <= n) {
        float4 a = __ldcs(reinterpret_cast<const float4*>(w) + unit), d = __ldcs(reinterpret_cast<const float4*>(m) + unit),
               e = __ldcs(reinterpret_cast<const float4*>(v) + unit);
        const float4 b = reinterpret_cast<const float4*>(g)[unit];
        step.apply(a.x, b.x * scale, d.x, e.x);
        step.apply(a.y, b.y * scale, d.y, e.y);
        step.apply(a.z, b.z * scale, d.z, e.z);
        step.apply(a.w, b.w * scale, d.w, e.w);
        __stcs(reinterpret_cast<float4*>(m) + unit, d);
        __stcs(reinterpret_cast<float4*>(v) + unit, e);
        __stcs(reinterpret_cast<float4*>(w) + unit, a);
    } else {
        for (size_t i = Quads ? 4 * unit : unit; i < n && i < (Quads ? 4 * unit + 4 : unit + 1); i++) step.apply(w[i], g[i] * scale, m[i], v[i]);
    }
}

}  // namespace znn

using namespace znn;

static int check_set(const void* grads, const size_t* counts, int n, const float* const* ptrs)
{
    ZNN_REQUIRE(n >= 0, "n is negative");
    ZNN_REQUIRE(n == 0 || (grads && counts), "NULL pointer");
    for (int i = 0; i < n; i++) {
        ZNN_REQUIRE(counts[i] == 0 || ptrs[i], "tensor %d is NULL", i);
        ZNN_REQUIRE(((uintptr_t)ptrs[i] & 3) == 0, "tensor %d is not aligned to 4 bytes", i);
        ZNN_REQUIRE(counts[i] <= (size_t)1 << 40, "tensor %d has an implausible size", i);
    }
    return ZNN_OK;
}

// The next up to Cap tensors as a table, advancing *at; false when none is left.
template <int Cap>
static bool next_table(const float* const* grads, const size_t* counts, int n, int* at, TensorTable<Cap>* t)
{
    long long tiles = 0;
    t->n = 0;
    while (*at < n && t->n < Cap) {
        const size_t c = counts[*at];
        const long long mine = (long long)((c + kNormTile - 1) / kNormTile);
        if (t->n > 0 && tiles + mine > 0x7ffffff) break;
        if (c) {
            t->data[t->n] = grads[*at];
            t->count[t->n] = (long long)c;
            t->first_tile[t->n] = (int)tiles;
            tiles += mine;
            t->n++;
        }
        ++*at;
    }
    t->first_tile[t->n] = (int)tiles;
    return t->n > 0;
}

template <int Cap>
static int grad_norm(const float* const* grads, const size_t* counts, int n, float grad_scale, float max_norm, float* result)
{
    double* partial = reinterpret_cast<double*>(result + kNormHead);
    const int blocks = std::min(kNormBlocks, sm_count() * 4);
    TensorTable<Cap> t;
    int at = 0, used = 0;
    while (next_table(grads, counts, n, &at, &t)) {
        const int tiles = t.first_tile[t.n];
        // one cluster where it has a few rounds at most: 645 thousand floats in six tensors take 10.1 us a call with it and 13.1 with two
        // launches, 1.5 million 16.7 and 13.4
        if (used == 0 && at == n && tiles <= 96) return launch_overlapped(norm_small_kernel<Cap>, "norm_small_kernel", 8, kNormThreads, 1, t, grad_scale, max_norm, result);
        // the first launch writes every partial sum that a later one adds to
        const int grid = (at < n || used) ? blocks : std::min(blocks, tiles);
        const int rc = launch_overlapped(norm_partial_kernel<Cap>, "norm_partial_kernel", grid, kNormThreads, 1, t, partial, used ? 1 : 0);
        if (rc != ZNN_OK) return rc;
        used = std::max(used, grid);
    }
    return launch_overlapped(norm_finish_kernel, "norm_finish_kernel", 1, kNormThreads, 1, (const double*)partial, used, grad_scale, max_norm, result);
}

template <int Cap>
static int clip_grads(float* const* grads, const size_t* counts, int n, const float* result)
{
    TensorTable<Cap> t;
    int at = 0;
    while (next_table(grads, counts, n, &at, &t)) {
        const int rc = launch_overlapped(clip_kernel<Cap>, "clip_kernel", std::min(t.first_tile[t.n], sm_count() * 4), kNormThreads, 1, t, result);
        if (rc != ZNN_OK) return rc;
    }
    return ZNN_OK;
}

// Whether no float belongs to two of the tensors: clipping would multiply it twice, or lose one of the two.
static bool apart(const float* const* grads, const size_t* counts, int n)
{
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    spans.reserve((size_t)n);
    for (int i = 0; i < n; i++)
        if (counts[i]) spans.emplace_back((uintptr_t)grads[i], (uintptr_t)grads[i] + 4 * counts[i]);
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); i++)
        if (spans[i].first < spans[i - 1].second) return false;
    return true;
}

static bool quads(const void* a, const void* b, const void* c, const void* d)
{
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 15) == 0;
}

// blocks of a step over n floats; 0 where they are more than a launch can have
static size_t step_blocks(size_t n, bool as_quads)
{
    const size_t units = as_quads ? (n + 3) / 4 : n, blocks = (units + kStepThreads - 1) / kStepThreads;
    return blocks <= 0x7fffffff ? blocks : 0;
}

extern "C" {

int znn_grad_norm(const float** grads, const size_t* counts, int n, float grad_scale, float max_norm, float* result)
{
    const int rc = check_set(grads, counts, n, grads);
    if (rc != ZNN_OK) return rc;
    ZNN_REQUIRE(result, "result is NULL");
    ZNN_REQUIRE(((uintptr_t)result & 15) == 0, "result is not aligned to 16 bytes");
    ZNN_REQUIRE(max_norm > 0.0f, "max_norm must be positive");
    ZNN_REQUIRE(isfinite(grad_scale), "grad_scale must be finite");
    ZNN_NEED_DEVICE();
    if (n <= kSmallTable) return grad_norm<kSmallTable>(grads, counts, n, grad_scale, max_norm, result);
    if (n <= kMiddleTable) return grad_norm<kMiddleTable>(grads, counts, n, grad_scale, max_norm, result);
    return grad_norm<kLargeTable>(grads, counts, n, grad_scale, max_norm, result);
}

int znn_clip_grads(float** grads, const size_t* counts, int n, const float* result)
{
    const int rc = check_set(grads, counts, n, grads);
    if (rc != ZNN_OK) return rc;
    ZNN_REQUIRE(result, "result is NULL");
    try {
        ZNN_REQUIRE(apart(grads, counts, n), "two of the tensors overlap");
    } catch (const std::bad_alloc&) {
        return fail(ZNN_ERR_NOMEM, "no host memory");
    }
    ZNN_NEED_DEVICE();
    if (n <= kSmallTable) return clip_grads<kSmallTable>(grads, counts, n, result);
    if (n <= kMiddleTable) return clip_grads<kMiddleTable>(grads, counts, n, result);
    return clip_grads<kLargeTable>(grads, counts, n, result);
}

int znn_sgd_step_clipped(float* w, const float* g, float* v, float lr, float momentum, float grad_scale, const float* result, size_t n)
{
    if (n == 0) return ZNN_OK;
    ZNN_REQUIRE(w && g && result, "NULL pointer");
    ZNN_REQUIRE(v || momentum == 0.0f, "momentum needs a velocity buffer");
    ZNN_NEED_DEVICE();
    const bool with_v = momentum > 0.0f, q = quads(w, g, with_v ? v : w, w);
    const size_t blocks = step_blocks(n, q);
    ZNN_REQUIRE(blocks, "n = %zu is too large", n);
    auto kernel = with_v ? (q ? sgd_clipped_kernel<true, true> : sgd_clipped_kernel<true, false>)
                         : (q ? sgd_clipped_kernel<false, true> : sgd_clipped_kernel<false, false>);
    return launch_overlapped(kernel, "sgd_clipped_kernel", blocks, kStepThreads, 1, w, g, v, SgdStep{lr, momentum}, grad_scale, result, n);
}

int znn_adam_step_clipped(float* w, const float* g, float* m, float* v, float lr, float beta1, float beta2, float eps, float t,
                          float grad_scale, const float* result, size_t n)
{
    if (n == 0) return ZNN_OK;
    ZNN_REQUIRE(w && g && m && v && result, "NULL pointer");
    ZNN_REQUIRE(t >= 1.0f, "t is the step count after the increment (>= 1)");
    ZNN_NEED_DEVICE();
    const float correction1 = 1.0f - powf(beta1, t);
    const float correction2 = 1.0f - powf(beta2, t);
    const float lr_t = lr * sqrtf(correction2) / correction1;   // as znn_adam_step
    const bool q = quads(w, g, m, v);
    const size_t blocks = step_blocks(n, q);
    ZNN_REQUIRE(blocks, "n = %zu is too large", n);
    return launch_overlapped(q ? adam_clipped_kernel<true> : adam_clipped_kernel<false>, "adam_clipped_kernel", blocks, kStepThreads, 1, w, g, m, v,
                  AdamStep{lr_t, beta1, beta2, eps}, grad_scale, result, n);
}

}  // extern "C"
