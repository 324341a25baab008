// Fine-tuning losses on a language model's logits: token log-probabilities (forward, backward), the clipped policy loss
// with its gradient, the preference loss on pairs of sequences.  Formulas: include/znn_cuda.h.
//
// Every operator is bound by HBM: 10 to 20 operations per logit against 4 to 12 bytes.
#include <math.h>
#include <math_constants.h>

#include "common.cuh"

namespace znn {

// What a row of logits sums to, relative to the largest logit mx seen: s = sum exp(d), u = sum d exp(d) with
// d = it * (x - mx).  The entropy is log s - u / s.
struct RowSums {
    float mx, s, u;
};

// d for one logit: -inf stays -inf, and a row of -inf alone (mx = -inf) is measured from 0 so that no inf - inf arises
__device__ __forceinline__ float base_of(float mx) { return mx == -CUDART_INF_F ? 0.0f : mx; }

// sums of two disjoint parts of a row; an empty part (s = 0) changes nothing, a NaN stays
__device__ __forceinline__ RowSums join(const RowSums& a, const RowSums& b, float it)
{
    if (b.s == 0.0f) return a;
    if (a.s == 0.0f) return b;
    RowSums r;
    r.mx = fmaxf(a.mx, b.mx);
    const float da = (base_of(a.mx) - base_of(r.mx)) * it, db = (base_of(b.mx) - base_of(r.mx)) * it;
    const float fa = expf(da), fb = expf(db);
    r.s = a.s * fa + b.s * fb;
    // a part that is too far below to count adds nothing here, even where da * a.s overflows (logits of the type's lowest value)
    r.u = (fa > 0.0f ? fa * (a.u + da * a.s) : 0.0f) + (fb > 0.0f ? fb * (b.u + db * b.s) : 0.0f);
    return r;
}

__device__ __forceinline__ RowSums warp_join(RowSums v, float it)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        RowSums w;
        w.mx = __shfl_xor_sync(0xffffffffu, v.mx, o);
        w.s = __shfl_xor_sync(0xffffffffu, v.s, o);
        w.u = __shfl_xor_sync(0xffffffffu, v.u, o);
        // the lower lane's part comes first on both sides, so that both compute the same bits
        v = (threadIdx.x & o) ? join(w, v, it) : join(v, w, it);
    }
    return v;
}

// sum over a block of up to 1024 threads in a fixed order, valid in every thread
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

struct RowParams {
    const float* logits;
    long long ld;
    const int32_t* targets;
    float it;
    int M, N;
    float *logp, *entropy, *stats;
    // policy loss only
    const float *old_logp, *ref_logp, *advantages, *weights;
    float clip_low, clip_high, kl_coef, entropy_coef;
    const float* count;   // 1 / *count is the weight where weights is NULL
    float* token_loss;
    float* dlogits;
    long long ld_d;
    int* status;
};

// What a row's gradient is made of: dx_j = p_j * (a + b * (log p_j)) for j != t, and dx_t as it is.
struct RowGrad {
    float a, b, at_target;
};

// The scalars of one row from its sums (one thread): writes logp, entropy, stats, token_loss, returns the gradient's
// coefficients.  Log-probability, ratio and loss are computed in fp64 from the fp32 sums: a ratio is exp() of a difference of
// numbers around 10, which fp32 would leave with an error of 1e-6.
template <bool Policy>
__device__ __forceinline__ RowGrad row_scalars(const RowParams& p, int row, const RowSums& r, float x_t, float w)
{
    const bool empty = (r.s == 0.0f);
    const double log_s = log((double)r.s);
    const double logp = empty ? -CUDART_INF : (double)p.it * ((double)x_t - (double)base_of(r.mx)) - log_s;
    const double H = empty ? 0.0 : log_s - (double)r.u / (double)r.s;
    if (p.logp) p.logp[row] = (float)logp;
    if (p.entropy) p.entropy[row] = (float)H;
    if (p.stats) {
        p.stats[2 * (size_t)row] = r.mx;
        p.stats[2 * (size_t)row + 1] = r.s;
    }
    RowGrad g{0.0f, 0.0f, 0.0f};
    if (Policy) {
        const double A = p.advantages[row], ratio = exp(logp - (double)p.old_logp[row]);
        double loss = 0.0, slope = 0.0;
        if (A != 0.0) {
            const double lo = 1.0 - (double)p.clip_low, hi = 1.0 + (double)p.clip_high;
            // a gain counts up to the upper border, a loss down to the lower one
            const bool outside = A > 0.0 ? ratio > hi : ratio < lo;
            loss = -A * (outside ? (A > 0.0 ? hi : lo) : ratio);
            slope = outside ? 0.0 : loss;
        }
        if (p.kl_coef != 0.0f) {
            const double q = (double)p.ref_logp[row] - logp, e = expm1(q);
            loss += (double)p.kl_coef * (e - q);
            slope -= (double)p.kl_coef * e;
        }
        double h = 0.0;
        if (p.entropy_coef != 0.0f) {
            loss -= (double)p.entropy_coef * H;
            h = -(double)p.entropy_coef;
        }
        p.token_loss[row] = (float)loss;
        if (!empty) {
            const double G = (double)p.it * w * slope, E = (double)p.it * w * h;
            g.a = (float)(-G - E * H);
            g.b = (float)(-E);
            const double pt = exp(logp);
            g.at_target = (float)(-G * expm1(logp) - (pt > 0.0 ? E * pt * (logp + H) : 0.0));
        }
    }
    return g;
}

// a row that is left out (bad = false) or whose target is outside the vocabulary (bad = true)
template <bool Policy>
__device__ __forceinline__ void row_unused(const RowParams& p, int row, bool bad)
{
    const float v = bad ? CUDART_NAN_F : 0.0f;
    if (p.logp) p.logp[row] = v;
    if (p.entropy) p.entropy[row] = 0.0f;
    if (p.stats) {
        p.stats[2 * (size_t)row] = 0.0f;
        p.stats[2 * (size_t)row + 1] = 0.0f;
    }
    if (Policy) p.token_loss[row] = v;
    if (bad && p.status) atomicOr(p.status, ZNN_DEV_BAD_INDEX);
}

// One block per row, any length: the first walk over the row makes the sums, the second (policy loss with gradient) reads
// the logits again and writes the gradient.
template <bool Policy>
__global__ void __launch_bounds__(256) rows_walk_kernel(const RowParams p)
{
    __shared__ RowSums sh[8];
    __shared__ RowGrad sh_grad;
    const int row = blockIdx.x, tid = threadIdx.x;
    const int t = p.targets[row];
    float w = 1.0f;
    if (Policy && p.weights) w = p.weights[row];
    if (t < 0 || t >= p.N || w == 0.0f) {
        if (tid == 0) row_unused<Policy>(p, row, t >= p.N && w != 0.0f);
        if (Policy && p.dlogits)
            for (int j = tid; j < p.N; j += 256) p.dlogits[(size_t)row * p.ld_d + j] = 0.0f;
        return;
    }
    const float* x = p.logits + (size_t)row * p.ld;
    RowSums r{-CUDART_INF_F, 0.0f, 0.0f};
    for (int j0 = tid; j0 < p.N; j0 += 256 * 8) {
        float v[8];
        float mx = -CUDART_INF_F;
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int j = j0 + 256 * k;
            v[k] = j < p.N ? x[j] : -CUDART_INF_F;
            mx = fmaxf(mx, v[k]);
        }
        RowSums c{mx, 0.0f, 0.0f};
        const float base = base_of(mx);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float d = (v[k] - base) * p.it, e = expf(d);
            c.s += e;
            c.u += e > 0.0f ? d * e : 0.0f;
        }
        r = join(r, c, p.it);
    }
    r = warp_join(r, p.it);
    if ((tid & 31) == 0) sh[tid >> 5] = r;
    float x_t = 0.0f;
    if (tid == 0) x_t = x[t];   // before any gradient is written: dlogits may be the logits' own buffer
    __syncthreads();
    r = sh[0];
    for (int i = 1; i < 8; i++) r = join(r, sh[i], p.it);
    if (Policy && !p.weights) w = 1.0f / *p.count;
    if (tid == 0) sh_grad = row_scalars<Policy>(p, row, r, x_t, w);
    if (!Policy || !p.dlogits) return;
    __syncthreads();
    const RowGrad g = sh_grad;
    const float base = base_of(r.mx), inv_s = r.s == 0.0f ? 0.0f : 1.0f / r.s, log_s = logf(r.s);
    float* dx = p.dlogits + (size_t)row * p.ld_d;
    for (int j = tid; j < p.N; j += 256) {
        const float d = (x[j] - base) * p.it, e = expf(d);
        float o = e * inv_s * g.a;
        if (g.b != 0.0f && e != 0.0f) o = e * inv_s * (g.a + g.b * (d - log_s));
        dx[j] = j == t ? g.at_target : o;
    }
}

// dlogits of the log-probabilities from the forward's statistics: one block per row
template <bool Accumulate>
__global__ void __launch_bounds__(256)
logprob_bwd_kernel(const float* logits, long long ld, const int32_t* __restrict__ targets, float it,
                   const float* __restrict__ stats, const float* __restrict__ entropy, const float* __restrict__ dlogp,
                   const float* __restrict__ dentropy, float* dlogits, long long ld_d, int N)
{
    const int row = blockIdx.x, tid = threadIdx.x;
    const int t = targets[row];
    float* dx = dlogits + (size_t)row * ld_d;
    const float s = stats[2 * (size_t)row + 1];
    if (t < 0 || t >= N || s == 0.0f) {
        if (!Accumulate)
            for (int j = tid; j < N; j += 256) dx[j] = 0.0f;
        return;
    }
    const float* x = logits + (size_t)row * ld;
    const float base = base_of(stats[2 * (size_t)row]), inv_s = 1.0f / s;
    const float G = it * (dlogp ? dlogp[row] : 0.0f), E = it * (dentropy ? dentropy[row] : 0.0f);
    const float a = -G - (E != 0.0f ? E * entropy[row] : 0.0f), b = -E, log_s = logf(s);
    for (int j = tid; j < N; j += 256) {
        const float d = (x[j] - base) * it, e = expf(d);
        float o = e * inv_s * a;
        if (b != 0.0f && e != 0.0f) o = e * inv_s * (a + b * (d - log_s));
        if (j == t) o += G;
        dx[j] = Accumulate ? dx[j] + o : o;
    }
}

// loss[1] = rows in use; with_sum: loss[0] = sum of w_i token_loss_i as well.  One block, fixed order.
__global__ void __launch_bounds__(1024)
policy_total_kernel(const int32_t* __restrict__ targets, const float* __restrict__ weights, const float* __restrict__ token_loss,
                    float* __restrict__ loss, int M, int with_sum)
{
    __shared__ double sh[32];
    double count = 0.0, sum = 0.0;
    for (int i = threadIdx.x; i < M; i += 1024) {
        const float w = weights ? weights[i] : 1.0f;
        if (targets[i] < 0 || w == 0.0f) continue;
        count += 1.0;
        if (with_sum) sum += (double)w * (double)token_loss[i];
    }
    count = block_sum(count, sh);
    if (with_sum) sum = block_sum(sum, sh);
    if (threadIdx.x == 0) {
        loss[1] = (float)count;
        if (with_sum) loss[0] = (float)(weights ? sum : count > 0.0 ? sum / count : 0.0);
    }
}

// One block per pair: the two sums, the pair's loss, the gradient of its rows.
__global__ void __launch_bounds__(256)
preference_pair_kernel(const float* __restrict__ logp, const float* __restrict__ ref_logp, const int32_t* __restrict__ targets,
                       const int32_t* __restrict__ offsets, float beta, float smoothing, float margin, int by_length,
                       float* __restrict__ pair_loss, float* __restrict__ rewards, float* __restrict__ dlogp, int P, int M,
                       int* __restrict__ status)
{
    __shared__ double sh[8];
    const int pair = blockIdx.x;
    const int o[3] = {offsets[2 * pair], offsets[2 * pair + 1], offsets[2 * pair + 2]};
    if (o[0] < 0 || o[1] < o[0] || o[2] < o[1] || o[2] > M) {
        if (threadIdx.x == 0) {
            pair_loss[pair] = rewards[2 * pair] = rewards[2 * pair + 1] = CUDART_NAN_F;
            if (status) atomicOr(status, ZNN_DEV_BAD_INDEX);
        }
        return;
    }
    double reward[2], share[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        double sum = 0.0, n = 0.0;
        for (int i = o[k] + threadIdx.x; i < o[k + 1]; i += 256) {
            if (targets && targets[i] < 0) continue;
            sum += (double)logp[i] - (ref_logp ? (double)ref_logp[i] : 0.0);
            n += 1.0;
        }
        sum = block_sum(sum, sh);
        share[k] = beta;
        if (by_length) {
            n = block_sum(n, sh);
            share[k] = n > 0.0 ? (double)beta / n : 0.0;
        }
        reward[k] = share[k] * sum;
    }
    const double m = reward[0] - reward[1] - (double)margin, eps = smoothing;
    const double soft = log1p(exp(-fabs(m)));   // log(1 + exp(-|m|)): -log sigmoid(+-m) without overflow
    if (threadIdx.x == 0) {
        pair_loss[pair] = (float)((1.0 - eps) * (soft + fmax(-m, 0.0)) + eps * (soft + fmax(m, 0.0)));
        rewards[2 * pair] = (float)reward[0];
        rewards[2 * pair + 1] = (float)reward[1];
    }
    if (!dlogp) return;
    const double slope = (eps - 1.0 / (1.0 + exp(m))) / (double)P;   // -(1 - eps) sigmoid(-m) + eps sigmoid(m)
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const float g = (float)((k ? -slope : slope) * share[k]);
        for (int i = o[k] + threadIdx.x; i < o[k + 1]; i += 256) dlogp[i] = (targets && targets[i] < 0) ? 0.0f : g;
    }
}

__global__ void __launch_bounds__(1024) mean_kernel(const float* __restrict__ v, float* __restrict__ out, int n)
{
    __shared__ double sh[32];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) s += (double)v[i];
    s = block_sum(s, sh);
    if (threadIdx.x == 0) out[0] = (float)(s / (double)n);
}

}  // namespace znn

using namespace znn;

#define ZNN_NEED_DEVICE()                                                                                  \
    do {                                                                                                   \
        if (!stream()) return fail(ZNN_ERR_CUDA, "no CUDA device state; call znn_init (no CPU fallback)"); \
    } while (0)

static int check_rows(const float* logits, long long ld, const int32_t* targets, float inv_temp, int M, int N)
{
    ZNN_REQUIRE(M >= 0 && N > 0, "M must not be negative and N must be positive");
    ZNN_REQUIRE(M == 0 || (logits && targets), "NULL pointer");
    ZNN_REQUIRE(ld >= N, "ld = %lld is smaller than N = %d", ld, N);
    ZNN_REQUIRE(inv_temp > 0.0f && isfinite(inv_temp), "inv_temp must be positive and finite");
    return ZNN_OK;
}

extern "C" {

int znn_token_logprob_fwd(const float* logits, long long ld, const int32_t* targets, float inv_temp, float* logp, float* entropy,
                          float* stats, int M, int N)
{
    const int rc = check_rows(logits, ld, targets, inv_temp, M, N);
    if (rc != ZNN_OK) return rc;
    if (M == 0) return ZNN_OK;
    ZNN_REQUIRE(logp, "logp is NULL");
    ZNN_NEED_DEVICE();
    RowParams p{};
    p.logits = logits; p.ld = ld; p.targets = targets; p.it = inv_temp; p.M = M; p.N = N;
    p.logp = logp; p.entropy = entropy; p.stats = stats; p.status = device_status_word();
    rows_walk_kernel<false><<<M, 256, 0, stream()>>>(p);
    ZNN_LAUNCH_OK("rows_walk_kernel");
    return ZNN_OK;
}

int znn_token_logprob_bwd(const float* logits, long long ld, const int32_t* targets, float inv_temp, const float* stats,
                          const float* entropy, const float* dlogp, const float* dentropy, float* dlogits, long long ld_d,
                          int accumulate, int M, int N)
{
    const int rc = check_rows(logits, ld, targets, inv_temp, M, N);
    if (rc != ZNN_OK) return rc;
    if (M == 0) return ZNN_OK;
    ZNN_REQUIRE(stats && dlogits, "stats/dlogits is NULL");
    ZNN_REQUIRE(!dentropy || entropy, "dentropy needs the forward's entropy");
    ZNN_REQUIRE(ld_d >= N, "ld_d = %lld is smaller than N = %d", ld_d, N);
    ZNN_REQUIRE(dlogits != logits || (ld_d == ld && !accumulate), "dlogits may be the logits' own buffer only with ld_d == ld and accumulate = 0");
    ZNN_NEED_DEVICE();
    if (accumulate)
        logprob_bwd_kernel<true><<<M, 256, 0, stream()>>>(logits, ld, targets, inv_temp, stats, entropy, dlogp, dentropy, dlogits, ld_d, N);
    else
        logprob_bwd_kernel<false><<<M, 256, 0, stream()>>>(logits, ld, targets, inv_temp, stats, entropy, dlogp, dentropy, dlogits, ld_d, N);
    ZNN_LAUNCH_OK("logprob_bwd_kernel");
    return ZNN_OK;
}

int znn_policy_loss(const float* logits, long long ld, const int32_t* targets, float inv_temp, const float* old_logp,
                    const float* ref_logp, const float* advantages, const float* weights, float clip_low, float clip_high,
                    float kl_coef, float entropy_coef, float* loss, float* token_loss, float* logp, float* entropy,
                    float* dlogits, long long ld_d, int M, int N)
{
    const int rc = check_rows(logits, ld, targets, inv_temp, M, N);
    if (rc != ZNN_OK) return rc;
    ZNN_REQUIRE(M > 0, "M must be positive");
    ZNN_REQUIRE(old_logp && advantages && loss && token_loss, "NULL pointer");
    ZNN_REQUIRE(isfinite(kl_coef) && isfinite(entropy_coef), "kl_coef and entropy_coef must be finite");
    ZNN_REQUIRE(ref_logp || kl_coef == 0.0f, "kl_coef needs ref_logp");
    ZNN_REQUIRE(clip_low >= 0.0f && clip_low <= 1.0f && clip_high >= 0.0f && isfinite(clip_high),
                "clip_low must lie in [0, 1], clip_high must not be negative");
    ZNN_REQUIRE(!dlogits || ld_d >= N, "ld_d = %lld is smaller than N = %d", ld_d, N);
    ZNN_REQUIRE(dlogits != logits || ld_d == ld, "dlogits may be the logits' own buffer only with ld_d == ld");
    ZNN_NEED_DEVICE();
    RowParams p{};
    p.logits = logits; p.ld = ld; p.targets = targets; p.it = inv_temp; p.M = M; p.N = N;
    p.logp = logp; p.entropy = entropy; p.status = device_status_word();
    p.old_logp = old_logp; p.ref_logp = ref_logp; p.advantages = advantages; p.weights = weights;
    p.clip_low = clip_low; p.clip_high = clip_high; p.kl_coef = kl_coef; p.entropy_coef = entropy_coef;
    p.count = loss + 1; p.token_loss = token_loss; p.dlogits = dlogits; p.ld_d = ld_d;
    if (!weights) {   // the rows' weight 1 / count is needed before their gradients are written
        policy_total_kernel<<<1, 1024, 0, stream()>>>(targets, weights, token_loss, loss, M, 0);
        ZNN_LAUNCH_OK("policy_total_kernel");
    }
    rows_walk_kernel<true><<<M, 256, 0, stream()>>>(p);
    ZNN_LAUNCH_OK("rows_walk_kernel");
    policy_total_kernel<<<1, 1024, 0, stream()>>>(targets, weights, token_loss, loss, M, 1);
    ZNN_LAUNCH_OK("policy_total_kernel");
    return ZNN_OK;
}

int znn_preference_loss(const float* logp, const float* ref_logp, const int32_t* targets, const int32_t* seq_offsets, float beta,
                        float label_smoothing, float margin, int length_normalize, float* loss, float* pair_loss, float* rewards,
                        float* dlogp, int P, int M)
{
    ZNN_REQUIRE(P > 0 && M >= 0, "P must be positive and M must not be negative");
    ZNN_REQUIRE(P <= (1 << 30) - 1, "P = %d is too large for int32 offsets", P);
    ZNN_REQUIRE((M == 0 || logp) && seq_offsets && loss && pair_loss && rewards, "NULL pointer");
    ZNN_REQUIRE(isfinite(beta) && isfinite(margin), "beta and margin must be finite");
    ZNN_REQUIRE(label_smoothing >= 0.0f && label_smoothing < 1.0f, "label_smoothing must lie in [0, 1)");
    ZNN_NEED_DEVICE();
    preference_pair_kernel<<<P, 256, 0, stream()>>>(logp, ref_logp, targets, seq_offsets, beta, label_smoothing, margin,
                                                    length_normalize, pair_loss, rewards, dlogp, P, M, device_status_word());
    ZNN_LAUNCH_OK("preference_pair_kernel");
    mean_kernel<<<1, 1024, 0, stream()>>>(pair_loss, loss, P);
    ZNN_LAUNCH_OK("mean_kernel");
    return ZNN_OK;
}

}  // extern "C"
