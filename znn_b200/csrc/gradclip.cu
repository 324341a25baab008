// Global gradient norm over a set of tensors, clipping by it, and the optimizer steps that take the factor from device
// memory.  Compiled with -fmad=false like rowops.cu: the steps round where znn_sgd_step and znn_adam_step do.
//
// Bound by HBM: 4 bytes per gradient for the norm, 20 (SGD with momentum) or 28 (Adam) for a step.
#include <math.h>

#include <algorithm>

#include "common.cuh"

namespace znn {

constexpr int kNormThreads = 512;
constexpr int kNormTile = 8192;      // floats of one tensor that a block takes at a time
constexpr int kNormTensors = 1000;   // tensors per launch: the table travels as a kernel argument (at most 32764 bytes)
constexpr int kNormHead = 4;         // floats of `result` before the partial sums (16-byte aligned doubles)
constexpr int kNormBlocks = (ZNN_GRAD_NORM_FLOATS - kNormHead) / 2;

struct TensorTable {
    const float* data[kNormTensors];
    long long count[kNormTensors];
    int first_tile[kNormTensors + 1];   // tiles before tensor i
    int n;
};

__device__ __forceinline__ double block_sum(double v, double* sh)
{
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) sh[w] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < nw; i++) t += sh[i];
    return t;
}

// the tensor that tile `tile` belongs to: the last one whose first tile is not behind it
__device__ __forceinline__ int find_tensor(const TensorTable& t, int tile)
{
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first_tile[mid] <= tile) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// partial[block] (+)= squares of the block's tiles, in fp64
__global__ void __launch_bounds__(kNormThreads)
norm_partial_kernel(const __grid_constant__ TensorTable t, double* __restrict__ partial, int add)
{
    __shared__ double sh[kNormThreads / 32];
    double s = 0.0;
    const int tiles = t.first_tile[t.n];
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int i = find_tensor(t, tile);
        const long long begin = (long long)(tile - t.first_tile[i]) * kNormTile;
        const int n = (int)min((long long)kNormTile, t.count[i] - begin);
        const float* x = t.data[i] + begin;
        for (int j = threadIdx.x; j < n; j += kNormThreads) {
            const double v = x[j];
            s = fma(v, v, s);
        }
    }
    s = block_sum(s, sh);
    if (threadIdx.x == 0) partial[blockIdx.x] = add ? partial[blockIdx.x] + s : s;
}

__global__ void __launch_bounds__(kNormThreads)
norm_finish_kernel(const double* __restrict__ partial, int blocks, float grad_scale, float max_norm, float* __restrict__ result)
{
    __shared__ double sh[kNormThreads / 32];
    double s = 0.0;
    for (int i = threadIdx.x; i < blocks; i += kNormThreads) s += partial[i];
    s = block_sum(s, sh);
    if (threadIdx.x == 0) {
        const double norm = fabs((double)grad_scale) * sqrt(s);
        result[0] = (float)norm;
        result[1] = !isfinite(norm) ? 0.0f : norm > (double)max_norm ? (float)((double)max_norm / norm) : 1.0f;
    }
}

__global__ void __launch_bounds__(kNormThreads)
clip_kernel(const __grid_constant__ TensorTable t, const float* __restrict__ result)
{
    const float c = result[1];
    if (c == 1.0f || c == 0.0f) return;
    const int tiles = t.first_tile[t.n];
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int i = find_tensor(t, tile);
        const long long begin = (long long)(tile - t.first_tile[i]) * kNormTile;
        const int n = (int)min((long long)kNormTile, t.count[i] - begin);
        float* x = const_cast<float*>(t.data[i]) + begin;
        for (int j = threadIdx.x; j < n; j += kNormThreads) x[j] *= c;
    }
}

// rounds where sgd_kernel and adam_kernel (rowops.cu) do
__global__ void sgd_clipped_kernel(float* __restrict__ w, const float* __restrict__ g, float* __restrict__ v, float lr,
                                   float momentum, float grad_scale, const float* __restrict__ result, size_t n)
{
    const float c = result[1];
    if (c == 0.0f) return;
    const float scale = grad_scale * c;
    const size_t tid = blockIdx.x * (size_t)blockDim.x + threadIdx.x, nth = (size_t)gridDim.x * blockDim.x;
    for (size_t i = tid; i < n; i += nth) {
        const float gi = g[i] * scale;
        if (v) {
            const float vel = momentum * v[i] + lr * gi;
            v[i] = vel;
            w[i] -= vel;
        } else {
            w[i] -= lr * gi;
        }
    }
}

__global__ void adam_clipped_kernel(float* __restrict__ w, const float* __restrict__ g, float* __restrict__ m, float* __restrict__ v,
                                    float lr_t, float beta1, float beta2, float eps, float grad_scale,
                                    const float* __restrict__ result, size_t n)
{
    const float c = result[1];
    if (c == 0.0f) return;
    const float scale = grad_scale * c, ob1 = 1.0f - beta1, ob2 = 1.0f - beta2;
    const size_t tid = blockIdx.x * (size_t)blockDim.x + threadIdx.x, nth = (size_t)gridDim.x * blockDim.x;
    for (size_t i = tid; i < n; i += nth) {
        const float gi = g[i] * scale;
        const float mi = beta1 * m[i] + ob1 * gi;
        const float vi = beta2 * v[i] + ob2 * gi * gi;
        m[i] = mi;
        v[i] = vi;
        w[i] -= lr_t * mi / (sqrtf(vi) + eps);
    }
}

}  // namespace znn

using namespace znn;

#define ZNN_NEED_DEVICE()                                                                                  \
    do {                                                                                                   \
        if (!stream()) return fail(ZNN_ERR_CUDA, "no CUDA device state; call znn_init (no CPU fallback)"); \
    } while (0)

static int step_blocks(size_t n)
{
    const size_t cap = (size_t)sm_count() * 32;
    return (int)std::max<size_t>(1, std::min(cap, (n + 1023) / 1024));
}

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

// The next up to kNormTensors tensors as a table, advancing *at; false when none is left.
static bool next_table(const float* const* grads, const size_t* counts, int n, int* at, TensorTable* t)
{
    long long tiles = 0;
    t->n = 0;
    while (*at < n && t->n < kNormTensors) {
        const size_t c = counts[*at];
        const long long mine = (long long)((c + kNormTile - 1) / kNormTile);
        if (t->n > 0 && tiles + mine > 0x7fffffff) break;
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
    double* partial = reinterpret_cast<double*>(result + kNormHead);
    const int blocks = std::min(kNormBlocks, sm_count() * 4);
    TensorTable t;
    int at = 0, used = 0;
    bool add = false;
    while (next_table(grads, counts, n, &at, &t)) {
        // the first launch writes every partial sum that a later one adds to
        const int grid = (at < n || add) ? blocks : std::min(blocks, t.first_tile[t.n]);
        norm_partial_kernel<<<grid, kNormThreads, 0, stream()>>>(t, partial, add ? 1 : 0);
        ZNN_LAUNCH_OK("norm_partial_kernel");
        add = true;
        used = std::max(used, grid);
    }
    norm_finish_kernel<<<1, kNormThreads, 0, stream()>>>(partial, used, grad_scale, max_norm, result);
    ZNN_LAUNCH_OK("norm_finish_kernel");
    return ZNN_OK;
}

int znn_clip_grads(float** grads, const size_t* counts, int n, const float* result)
{
    const int rc = check_set(grads, counts, n, grads);
    if (rc != ZNN_OK) return rc;
    ZNN_REQUIRE(result, "result is NULL");
    ZNN_NEED_DEVICE();
    TensorTable t;
    int at = 0;
    while (next_table(grads, counts, n, &at, &t)) {
        clip_kernel<<<std::min(t.first_tile[t.n], sm_count() * 4), kNormThreads, 0, stream()>>>(t, result);
        ZNN_LAUNCH_OK("clip_kernel");
    }
    return ZNN_OK;
}

int znn_sgd_step_clipped(float* w, const float* g, float* v, float lr, float momentum, float grad_scale, const float* result, size_t n)
{
    if (n == 0) return ZNN_OK;
    ZNN_REQUIRE(w && g && result, "NULL pointer");
    ZNN_REQUIRE(v || momentum == 0.0f, "momentum needs a velocity buffer");
    ZNN_NEED_DEVICE();
    sgd_clipped_kernel<<<step_blocks(n), 256, 0, stream()>>>(w, g, (momentum > 0.0f) ? v : nullptr, lr, momentum, grad_scale, result, n);
    ZNN_LAUNCH_OK("sgd_clipped_kernel");
    return ZNN_OK;
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
    adam_clipped_kernel<<<step_blocks(n), 256, 0, stream()>>>(w, g, m, v, lr_t, beta1, beta2, eps, grad_scale, result, n);
    ZNN_LAUNCH_OK("adam_clipped_kernel");
    return ZNN_OK;
}

}  // extern "C"
