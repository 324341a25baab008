// Fine-tuning losses on a language model's logits: token log-probabilities (forward, backward), the clipped policy loss
// with its gradient, the preference loss on pairs of sequences.  Formulas: include/znn_cuda.h.
//
// Bound by HBM where there is enough to do (10 to 20 operations per logit against 4 to 12 bytes), by launch and reduction latency
// where there is not.  Measured on B200s whose copies run at 6548 GB/s, the whole call, inputs in turn from three sets, on several devices:
//   log-probabilities and entropies 2045 x 50257, a fifth left out  57 - 62 us   5.3 - 5.7 TB/s   (floor 50 us)
//   their gradient with entropy term 8192 x 8192, a tenth left out  78 - 79 us   6.4 TB/s         (78 us)
//   policy loss 8192 x 8192, KL term                                94 - 96 us   5.7 TB/s         (82 us)
//   policy loss 2048 x 131000, KL and entropy, 0.15 left out       340 - 370 us  5.4 - 5.8 TB/s   (303 us)
//   preference loss 700 pairs, 1.4 million rows                     12 us                         (3.4 us: latency)
#include <math.h>
#include <math_constants.h>

#include <algorithm>

#include "overlap.cuh"
#include "tc_ptx.cuh"

namespace znn {

constexpr unsigned kAllLanes = 0xffffffffu;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Where exp2() is 0 in fp32 whatever comes after the point.  Exponents are clamped to it, so that no 0 * inf arises.
constexpr float kNothing = -150.0f;

// 2^x as the special-function unit gives it (relative error below 2^-22, subnormal results 0).  The exponentials of this file
// are 2^t with t = (x - xm) * inv_temp * log2(e): a subtraction, a product and this, where expf() would take twice as many
// operations after the same two roundings, and the kernels issue in half to two thirds of all cycles as it is.
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The same, for an exponential that is taken again rather than kept: the compiler does not see that it has been made already.
__device__ __forceinline__ float exp2_again(float x)
{
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// the larger of the two, and NaN where there is one (fmaxf() would drop it)
__device__ __forceinline__ float max_nan(float a, float b)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// What a row of logits (or a part of one) sums to, relative to the largest logit mx seen, with t = (x - mx) * inv_temp * log2(e):
// `ties` logits equal mx, s = sum of 2^t over the others, u = sum of t 2^t.  The row's sum is ties + s.  The ones are kept apart
// because a row that is nearly certain has s << 1, and its log-probability -log(1 + s) is only as exact as s is: 1 + s in fp32
// would leave an error of 6e-8 / s.
struct __align__(16) RowSums {
    float mx, ties, s, u;
};

// A row of -inf alone (mx = -inf) is measured from 0, so that no inf - inf arises: all its terms are 0.
__device__ __forceinline__ float base_of(float mx) { return mx == -CUDART_INF_F ? 0.0f : mx; }

// over the W lanes of a warp that `mask` names (W neighbours), in a fixed order, the result in each of them
template <int W = 32>
__device__ __forceinline__ float warp_max(float v, unsigned mask = kAllLanes)
{
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(mask, v, o));
    return v;
}

template <int W = 32>
__device__ __forceinline__ float warp_sum(float v, unsigned mask = kAllLanes)
{
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    return v;
}

// the sums of W lanes' disjoint parts, in each of them; an empty part (nothing but -inf) changes nothing, a NaN stays
template <int W = 32>
__device__ __forceinline__ RowSums join_lanes(const RowSums& v, float c, unsigned mask = kAllLanes)
{
    RowSums r;
    r.mx = warp_max<W>(v.mx, mask);
    const bool top = v.mx == r.mx;
    const float delta = top ? 0.0f : fmaxf((v.mx - r.mx) * c, kNothing), f = exp2_fast(delta);
    r.ties = warp_sum<W>(top ? v.ties : 0.0f, mask);
    r.s = warp_sum<W>(top ? v.s : (v.s + v.ties) * f, mask);
    r.u = warp_sum<W>(f * (v.u + delta * (v.s + v.ties)), mask);
    return r;
}

// log(ties + s) to about 4e-8, absolutely and (for sums near 1) relatively, with fp32's own logarithms: log1p() of s beside a
// single one, and elsewhere the logarithm of the mantissa beside an exact power of two.
__device__ __forceinline__ double log_of_sum(float ties, float s)
{
    if (ties == 1.0f && s < 1.0f) return (double)log1pf(s);
    const float total = ties + s;   // at least 1, or 0, or NaN
    const int bits = __float_as_int(total);
    if (total == 0.0f) return -CUDART_INF;
    return (double)((bits >> 23) - 127) * 0.693147180559945309417 + (double)logf(__int_as_float((bits & 0x007fffff) | 0x3f800000)) + (total - total);
}

// Every kernel here may begin while the one before it on the stream ends (overlap.cuh).  (Rows of a policy loss that began beside the
// kernel that counts them would save 2 us of 90, but nothing would promise that they see what ran before that one.)
struct RowParams {
    const float* logits;
    long long ld;
    const int32_t* targets;
    float it, c;   // inv_temp, inv_temp * log2(e)
    int M, N;
    float *logp, *entropy, *stats;
    // policy loss only
    const float *old_logp, *ref_logp, *advantages, *weights;
    float clip_low, clip_high, kl_coef, entropy_coef;
    const float* count;   // 1 / *count is the weight where weights is NULL; NULL: every group counts the (few) rows itself
    float* token_loss;
    float* dlogits;
    long long ld_d;
    int* status;
};

// What a row's gradient is made of: dx_j = 2^t * (a + b * t) for j != target, and dx at the target as it is.  t is measured
// from `mx`.
struct __align__(16) RowGrad {
    float a, b, at_target, mx;
};

// What decides whether a row is used: its target and (policy loss) its weight.  With them, in the thread that makes the row's
// scalars (`inputs`), the row's entries of the other inputs: they are on their way while the row is walked over, instead of behind it.
struct RowHead {
    int t;
    float w, old_logp, ref_logp, advantage;
    __device__ __forceinline__ bool used(int N) const { return t >= 0 && t < N && w != 0.0f; }
};

template <bool Policy>
__device__ __forceinline__ RowHead row_head(const RowParams& p, unsigned row, bool inputs)
{
    RowHead h{-1, 1.0f, 0.0f, 0.0f, 0.0f};
    if (row < (unsigned)p.M) {
        h.t = p.targets[row];
        if (Policy && p.weights) h.w = p.weights[row];
        if (Policy && inputs) {
            h.old_logp = p.old_logp[row];
            h.advantage = p.advantages[row];
            if (p.kl_coef != 0.0f) h.ref_logp = p.ref_logp[row];
        }
    }
    return h;
}

// The scalars of one row from its sums (one thread): writes logp, entropy, stats, token_loss (where `write`), returns the
// gradient's coefficients.  The log-probability, and the differences that ratio and
// KL term are made of, are fp64: fp32 would leave a ratio of two probabilities of e^-10 an error of 1e-6.  What follows from
// them is fp32: products, and the KL term, which is kept from cancelling.  (In short rows these few hundred operations of one lane are
// most of the work.)
template <bool Policy, bool Entropy>
__device__ __forceinline__ RowGrad row_scalars(const RowParams& p, int row, const RowSums& r, const RowHead& in, float x_t, int rows,
                                               bool write)
{
    const float total = r.ties + r.s, inv_total = 1.0f / total;
    const bool empty = total == 0.0f;
    const double log_s = log_of_sum(r.ties, r.s);
    const double logp = empty ? -CUDART_INF : (double)p.it * ((double)x_t - (double)base_of(r.mx)) - log_s;
    const float U = Entropy ? kLn2 * r.u * inv_total : 0.0f;   // sum of p_j (log p_j + log s)
    const float H = !Entropy || empty ? 0.0f : (float)(log_s - (double)U);
    if (write) {
        if (p.logp) p.logp[row] = (float)logp;
        if (Entropy && p.entropy) p.entropy[row] = H;
        if (p.stats) {
            p.stats[2 * (size_t)row] = r.mx;
            p.stats[2 * (size_t)row + 1] = total;
        }
    }
    RowGrad g{0.0f, 0.0f, 0.0f, r.mx};
    if (Policy) {
        const float A = in.advantage;
        float loss = 0.0f, slope = 0.0f;
        if (A != 0.0f) {
            const float ratio = expf((float)(logp - (double)in.old_logp));
            const float border = A > 0.0f ? 1.0f + p.clip_high : 1.0f - p.clip_low;
            // a gain counts up to the upper border, a loss down to the lower one
            const bool outside = A > 0.0f ? ratio > border : ratio < border;
            loss = -A * (outside ? border : ratio);
            slope = outside ? 0.0f : loss;
        }
        if (p.kl_coef != 0.0f) {
            const float q = (float)((double)in.ref_logp - logp);
            float e, rest;   // e^q - 1, e^q - 1 - q
            if (fabsf(q) < 0.5f) {
                // e - q would lose what e and q share: 63 halves of a step just above 1/32, 7 at 1/4.  The term comes from its series
                // q^2 (1/2! + q/3! + ... + q^7/9!), whose next member is below 2e-9 of it: 3 halves, as many as e - q has from 1/2 on.
                rest = q * q * (0.5f + q * (1.0f / 6 + q * (1.0f / 24 + q * (1.0f / 120 + q * (1.0f / 720 + q * (1.0f / 5040 + q * (1.0f / 40320 + q * (1.0f / 362880))))))));
                e = q + rest;
            } else {
                e = expm1f(q);
                rest = isinf(e) ? e : e - q;   // of q = +inf, e - q would leave NaN
            }
            loss += p.kl_coef * rest;
            slope -= p.kl_coef * e;
        }
        if (Entropy) loss -= p.entropy_coef * H;
        if (write) p.token_loss[row] = loss;
        if (!empty) {
            float w = in.w;
            if (!p.weights) w = 1.0f / (p.count ? *p.count : (float)rows);
            const float G = p.it * w * slope, E = Entropy ? -p.it * w * p.entropy_coef : 0.0f;
            // p_t, and 1 - p_t: where the target is the largest, what the others sum to; elsewhere p_t is at most 1/2
            const float top = base_of(r.mx), e_t = x_t == top ? 1.0f : exp2_fast(fmaxf((x_t - top) * p.c, kNothing));
            const float others = (x_t == top ? r.ties - 1.0f + r.s : total - e_t) * inv_total;
            g.at_target = (others == 0.0f ? 0.0f : G * others) - (Entropy && e_t > 0.0f ? E * e_t * inv_total * ((float)logp + H) : 0.0f);
            // p_j (-G - E (log p_j + H)),  p_j = 2^t / s,  log p_j + H = log(2) t - U
            g.a = inv_total * (-G + (Entropy ? E * U : 0.0f));
            g.b = Entropy ? -inv_total * E * kLn2 : 0.0f;
        }
    }
    return g;
}

// rows that are not left out, the share of one of `Lanes` neighbouring lanes: small calls count them on the way, where a kernel of
// its own would cost more than all the rest
template <int Lanes>
__device__ __forceinline__ int count_rows(const RowParams& p, int tid)
{
    int rows = 0;
#pragma unroll 4
    for (int i = tid; i < p.M; i += Lanes) rows += p.targets[i] >= 0 ? 1 : 0;
    return rows;
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

// ---- a row's columns among the threads ------------------------------------------------------------------------------
// Group threads take V 16-byte quads each of a row's part in a step: thread k the quads k, k + Group, ... of the step.  A part
// may start and end at any float: up to three columns lie before its first quad and after its last, one each for a few threads
// (`extra`), so that nothing stands between the quads' memory instructions.  Aligned: there are none of those.
template <int Group, int V, bool Aligned>
struct RowPart {
    float v[V][4];
    float extra;
    int n, head, quads;   // columns of the part, those before the first quad, quads
    int step;             // first quad of the step

    __device__ __forceinline__ void place(const float* x, int columns)
    {
        n = columns;
        head = Aligned ? 0 : min(n, (int)(0u - (unsigned)((uintptr_t)x >> 2)) & 3);
        quads = (n - head) >> 2;
        step = 0;
    }
    __device__ __forceinline__ bool has(int tid, int k) const { return step + tid + k * Group < quads; }
    __device__ __forceinline__ int column(int tid, int k) const { return head + 4 * (step + tid + k * Group); }
    // the thread's extra column: the first threads have those before the quads, from the fifth on those after them
    __device__ __forceinline__ int extra_column(int tid) const
    {
        if (Aligned || step > 0) return -1;
        const int after = head + 4 * quads + tid - 4;
        return tid < head ? tid : tid >= 4 && after < n ? after : -1;
    }

    // Last: nobody reads these logits again, so that they leave L2 before those that are read once more
    template <bool Last = false>
    __device__ __forceinline__ void load(const float* x, int tid)
    {
#pragma unroll
        for (int k = 0; k < V; k++) {
            float4 q = make_float4(-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F);
            const float4* from = reinterpret_cast<const float4*>(x + column(tid, k));
            if (has(tid, k)) q = Last ? __ldcs(from) : *from;
            v[k][0] = q.x; v[k][1] = q.y; v[k][2] = q.z; v[k][3] = q.w;
        }
        const int c = extra_column(tid);
        extra = c >= 0 ? x[c] : -CUDART_INF_F;
    }

    // whether the part's quads are quads of the row y as well
    __device__ __forceinline__ bool same_quads(const float* y) const { return Aligned || ((uintptr_t)(y + head) & 15) == 0; }

    // the same columns of a row of any alignment
    __device__ __forceinline__ void load_beside(const float* y, int tid, float (&o)[V][4], float& o_extra) const
    {
        const bool quad = same_quads(y);
#pragma unroll
        for (int k = 0; k < V; k++) {
            float4 q = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (has(tid, k)) {
                const float* from = y + column(tid, k);
                if (quad) q = __ldcs(reinterpret_cast<const float4*>(from));
                else q = make_float4(__ldcs(from), __ldcs(from + 1), __ldcs(from + 2), __ldcs(from + 3));
            }
            o[k][0] = q.x; o[k][1] = q.y; o[k][2] = q.z; o[k][3] = q.w;
        }
        const int c = extra_column(tid);
        o_extra = c >= 0 ? y[c] : 0.0f;
    }

    // whether this thread is the one that holds (and stores) column c in this step
    __device__ __forceinline__ bool owns(int c, int tid) const
    {
        if (c < 0 || c >= n) return false;
        if (!Aligned && (c < head || c >= head + 4 * quads)) return extra_column(tid) == c;
        const int q = ((c - head) >> 2) - step;
        return q >= 0 && q < Group * V && q % Group == tid;
    }

    // writes what the caller has put into v to a row of any alignment
    __device__ __forceinline__ void store(float* y, int tid) const
    {
        const bool quad = same_quads(y);
#pragma unroll
        for (int k = 0; k < V; k++) {
            if (!has(tid, k)) continue;
            float* to = y + column(tid, k);
            if (quad) {
                __stcs(reinterpret_cast<float4*>(to), make_float4(v[k][0], v[k][1], v[k][2], v[k][3]));
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) __stcs(to + i, v[k][i]);
            }
        }
        const int c = extra_column(tid);
        if (c >= 0) __stcs(y + c, extra);
    }

    // A row whose loss is +inf has an infinite coefficient: gradients of +-inf, and NaN (0 times it) where the column's probability is 0
    // and its gradient is to be 0.  This goes over what the thread has written to such a row y.  (The rows are few: a test per column in
    // the loops of all rows takes 1 to 6 % of their time.)
    __device__ __forceinline__ void clear_nan(float* y, int tid)
    {
        for (step = 0; step == 0 || step < quads; step += Group * V) {
#pragma unroll 1
            for (int k = 0; k < V; k++)
                if (has(tid, k))
                    for (int i = 0; i < 4; i++)
                        if (isnan(y[column(tid, k) + i])) y[column(tid, k) + i] = 0.0f;
            const int c = extra_column(tid);
            if (c >= 0 && isnan(y[c])) y[c] = 0.0f;
        }
    }

    // zeros for the whole part
    __device__ __forceinline__ static void clear(float* y, int columns, int tid)
    {
        const int before = Aligned ? 0 : min(columns, (int)(0u - (unsigned)((uintptr_t)y >> 2)) & 3), whole = (columns - before) >> 2;
        for (int q = tid; q < whole; q += Group) __stcs(reinterpret_cast<float4*>(y + before) + q, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        if (!Aligned) {
            if (tid < before) y[tid] = 0.0f;
            if (before + 4 * whole + tid < columns) y[before + 4 * whole + tid] = 0.0f;
        }
    }
};

// ---- what the blocks of a cluster tell one another -------------------------------------------------------------------
__device__ __forceinline__ int cluster_size()
{
    unsigned r;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return (int)r;
}
__device__ __forceinline__ int cluster_rank()
{
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return (int)r;
}

// (the barrier's own order is enough for mbarriers that are published by their fence: no memory fence on arrival)
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_store(double* place, int rank, double v)
{
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(mapa_shared(smem_u32(place), (uint32_t)rank)), "d"(v) : "memory");
}

// The sums of every block's part of a row, written by the blocks themselves.
struct RowWord {
    RowSums sums[8];
    unsigned long long bar;
};

// Sends this block's sums to every block of the cluster and waits for theirs; all lanes of one warp call it.  The stores count
// on the receiver's barrier as they land.
__device__ __forceinline__ void exchange(RowWord* word, const RowSums& mine, int ranks, int rank, int* status)
{
    const int lane = threadIdx.x & 31;
    const uint32_t bar = smem_u32(&word->bar), sums = smem_u32(&word->sums[rank]);
    if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(ranks * sizeof(RowSums)));
    if (lane < ranks) {
        const uint32_t there = mapa_shared(bar, lane);
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(mapa_shared(sums, lane)),
                     "f"(mine.mx), "f"(mine.ties), "f"(mine.s), "f"(mine.u), "r"(there)
                     : "memory");
    }
    // (every block of the cluster runs and comes here: the wait ends.  Its limit is there for what nobody foresees; the
    // row is then made of what has arrived, and the status word says so)
    if (!mbar_wait_bounded_cluster(bar, 0, kWaitLimitCycles) && status) atomicOr(status, ZNN_DEV_TMA_WAIT_EXPIRED);
    __syncwarp();
}

// Short rows: 8 lanes or a warp hold whole rows in registers from their load to the gradient's store, Rows of them at a time: lane k
// makes the scalars of the k-th, since those few hundred operations cost the same for one lane as for all.  The maximum comes first,
// so that every exponential is taken once, relative to it.  A row that is left out is one of nothing but -inf: its gradient is 0.
// Log-probabilities 65536 x 1000: 40 us, 6.5 TB/s, 65536 x 100: 6.9 us, 3.9 TB/s; policy loss with KL term 65536 x 1000: 95 us,
// 5.5 TB/s, 1000000 x 100: 283 us, 2.9 TB/s (369 with one row at a time): the rows' scalars and reductions show, the more the shorter
// the rows are.
template <bool Policy, bool Entropy, bool Aligned, int Group, int V, int Rows>
__global__ void __launch_bounds__(128) rows_held_kernel(const RowParams p)
{
    static_assert(Rows <= Group, "a lane makes the scalars of one row");
    const int tid = threadIdx.x % Group;
    const unsigned mask = Group < 32 ? ((1u << (Group & 31)) - 1) << (threadIdx.x & 31 & ~(Group - 1)) : kAllLanes;
    const unsigned row0 = (blockIdx.x * (128 / Group) + threadIdx.x / Group) * Rows, mine = row0 + tid;
    if (row0 >= (unsigned)p.M) return;
    wait_for_previous_kernel();
    const bool there = tid < Rows && mine < (unsigned)p.M;
    const RowHead in = row_head<Policy>(p, there ? mine : 0xffffffffu, true);
    const bool used = in.used(p.N);
    const float* x = p.logits + (size_t)row0 * p.ld;
    RowPart<Group, V, Aligned> r[Rows];
    int t[Rows];
#pragma unroll
    for (int k = 0; k < Rows; k++) {
        t[k] = __shfl_sync(mask, used ? in.t : -1, k, Group);
        r[k].place(x + k * p.ld, t[k] >= 0 ? p.N : 0);
        r[k].load(x + k * p.ld, tid);
    }
    const float x_t = used ? p.logits[(size_t)mine * p.ld + in.t] : 0.0f;   // before a gradient is written over it
    const int rows = Policy && !p.weights && !p.count ? __reduce_add_sync(mask, count_rows<Group>(p, tid)) : 0;
    RowSums own{};
#pragma unroll
    for (int k = 0; k < Rows; k++) {
        float top = r[k].extra;
#pragma unroll
        for (int q = 0; q < V; q++) top = fmaxf(fmaxf(top, fmaxf(r[k].v[q][0], r[k].v[q][1])), fmaxf(r[k].v[q][2], r[k].v[q][3]));
        RowSums sums{warp_max<Group>(top, mask), 0.0f, 0.0f, 0.0f};
        const float base = base_of(sums.mx);
        // with an entropy term t is clamped (0 * -inf is to be 0), and kept for the gradient, which takes 2^t again
        auto take = [&](float& x) {
            const float t2 = (x - base) * p.c, te = Entropy ? max_nan(t2, kNothing) : t2, e = exp2_fast(te);
            sums.s += e;
            if (Entropy) sums.u += te * e;
            x = Entropy ? te : e;
        };
#pragma unroll
        for (int q = 0; q < V; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) take(r[k].v[q][i]);
        if (!Aligned) take(r[k].extra);
        if (top == base) {   // the few threads that hold the largest logit tell its ones from the rest
            const float with_ones = sums.s;
            sums.s = 0.0f;
            auto add = [&](float x) {
                const float e = Entropy ? exp2_again(x) : x;
                if (!(e == 1.0f)) sums.s += e;
            };
#pragma unroll
            for (int q = 0; q < V; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) add(r[k].v[q][i]);
            if (!Aligned) add(r[k].extra);
            sums.ties = rintf(with_ones - sums.s);
        }
        sums.ties = warp_sum<Group>(sums.ties, mask);
        sums.s = warp_sum<Group>(sums.s, mask);
        if (Entropy) sums.u = warp_sum<Group>(sums.u, mask);
        if (tid == k) own = sums;
    }
    RowGrad g{};
    if (there) {
        if (used) g = row_scalars<Policy, Entropy>(p, mine, own, in, x_t, rows, true);
        else row_unused<Policy>(p, mine, in.t >= p.N && in.w != 0.0f);
    }
    if (!Policy || !p.dlogits) return;
    float* dx = p.dlogits + (size_t)row0 * p.ld_d;
#pragma unroll
    for (int k = 0; k < Rows; k++) {
        const float a = __shfl_sync(mask, g.a, k, Group), b = Entropy ? __shfl_sync(mask, g.b, k, Group) : 0.0f;
        const float at_target = __shfl_sync(mask, g.at_target, k, Group);
        auto slope = [&](float& x) { x = Entropy ? exp2_again(x) * (a + b * x) : x * a; };
#pragma unroll
        for (int q = 0; q < V; q++)
#pragma unroll
            for (int i = 0; i < 4; i++) slope(r[k].v[q][i]);
        if (!Aligned) slope(r[k].extra);
        r[k].place(x + k * p.ld, row0 + k < (unsigned)p.M ? p.N : 0);
        r[k].store(dx + k * p.ld_d, tid);
        if (r[k].owns(t[k], tid)) dx[k * p.ld_d + t[k]] = at_target;
    }
    if (__any_sync(mask, isinf(g.a)))
#pragma unroll
        for (int k = 0; k < Rows; k++)
            if (isinf(__shfl_sync(mask, g.a, k, Group))) r[k].clear_nan(dx + k * p.ld_d, tid);
}

// Longer rows: a block (or the blocks of a cluster, which take `part` columns each) walks over the row with running sums per thread,
// and for the gradient a second time, back from the end, through the L2 cache: 8 bytes per logit cross HBM, not 12 (2048 x 131000:
// 0.94 GB read, 1.02 GB written, 343 us under the profiler).  Small blocks with few registers are what makes it fast: a row's chain of loads,
// reductions and scalars takes microseconds, and enough other rows must be under way meanwhile.  Rows held in registers, by blocks
// of 256 or 512 threads and clusters of them, took 580 us for the same, since too few blocks per SM hid too little of that chain
// (copying the next row to shared memory ahead made it worse: 8192 x 8192 110 -> 138 us, where this form takes 94).
// Rows of some 30 to 60 thousand columns lie between one block a row and small parts, and their second pass misses L2 most often:
// 2000 x 50256 156 us (floor 123); 5 % more without the second pass's loads marked as the last, 9 % for 50257 columns.
template <bool Policy, bool Entropy, bool Aligned, int Threads, int kQuads>
__global__ void __launch_bounds__(Threads) rows_walk_kernel(const RowParams p, int part)
{
    constexpr int kWarps = Threads / 32;
    using Part = RowPart<Threads, kQuads, Aligned>;
    __shared__ RowSums sh_warps[kWarps];
    __shared__ int sh_rows[kWarps];
    __shared__ RowGrad sh_grad;
    __shared__ __align__(16) RowWord sh_word;
    const int ranks = cluster_size(), rank = cluster_rank(), tid = threadIdx.x;
    if (ranks > 1) {
        if (tid == 0) {
            mbar_init(smem_u32(&sh_word.bar), 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        cluster_arrive();   // waited for when the first walk is done: by then every block runs and has its barrier
    }
    wait_for_previous_kernel();
    const int row = blockIdx.x / ranks, first = rank * part, n = max(0, min(part, p.N - first));
    const float* x = p.logits + (size_t)row * p.ld + first;
    float* dx = Policy && p.dlogits ? p.dlogits + (size_t)row * p.ld_d + first : nullptr;
    const RowHead in = row_head<Policy>(p, row, tid == 0);
    const int at = in.t - first;
    if (!in.used(p.N)) {
        if (tid == 0 && rank == 0) row_unused<Policy>(p, row, in.t >= p.N && in.w != 0.0f);
        if (dx) Part::clear(dx, n, tid);
        return;
    }
    // before any gradient is written: dlogits may be the logits' own buffer
    float x_t = tid == 0 ? p.logits[(size_t)row * p.ld + in.t] : 0.0f;

    RowSums sums{-CUDART_INF_F, 0.0f, 0.0f, 0.0f};
    Part r;
    constexpr int kStep = Threads * kQuads;
    r.place(x, n);
#pragma unroll 1
    for (;;) {
        r.load(x, tid);
        float mx = fmaxf(sums.mx, r.extra);
#pragma unroll
        for (int k = 0; k < kQuads; k++)
            mx = fmaxf(fmaxf(mx, fmaxf(r.v[k][0], r.v[k][1])), fmaxf(r.v[k][2], r.v[k][3]));
        if (mx != sums.mx) {
            const float delta = fmaxf((sums.mx - mx) * p.c, kNothing), f = exp2_fast(delta);
            sums.u = f * (sums.u + delta * (sums.s + sums.ties));
            sums.s = f * (sums.s + sums.ties);
            sums.ties = 0.0f;
            sums.mx = mx;
        }
        const float base = base_of(mx);
        auto take = [&](float x) {
            const float t2 = (x - base) * p.c, te = Entropy ? max_nan(t2, kNothing) : t2, e = exp2_fast(te);
            if (e == 1.0f) sums.ties += 1.0f;
            else sums.s += e;
            if (Entropy) sums.u += te * e;
        };
#pragma unroll
        for (int k = 0; k < kQuads; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) take(r.v[k][i]);
        if (!Aligned) take(r.extra);
        if (r.step + kStep >= r.quads) break;
        r.step += kStep;
    }
    if (Policy && !p.weights && !p.count) {
        const int rows = __reduce_add_sync(kAllLanes, count_rows<Threads>(p, tid));
        if ((tid & 31) == 0) sh_rows[tid >> 5] = rows;
    }
    if (ranks > 1) cluster_wait();
    sums = join_lanes(sums, p.c);
    if ((tid & 31) == 0) sh_warps[tid >> 5] = sums;
    __syncthreads();
    if (tid < 32) {
        const RowSums none{-CUDART_INF_F, 0.0f, 0.0f, 0.0f};
        sums = join_lanes(tid < kWarps ? sh_warps[tid] : none, p.c);
        if (ranks > 1) {
            x_t = __shfl_sync(kAllLanes, x_t, 0);   // it has arrived before another block learns that it may write over it
            exchange(&sh_word, sums, ranks, rank, p.status);
            sums = join_lanes(tid < ranks ? sh_word.sums[tid] : none, p.c);
        }
        if (tid == 0) {
            int rows = 0;
            if (Policy && !p.weights && !p.count)
                for (int i = 0; i < kWarps; i++) rows += sh_rows[i];
            sh_grad = row_scalars<Policy, Entropy>(p, row, sums, in, x_t, rows, rank == 0);
        }
    }
    if (!dx) return;
    __syncthreads();
    const RowGrad g = sh_grad;
    const float base = base_of(g.mx);
    // back from the end: the last step's logits are still here, the ones before it in the nearest caches
#pragma unroll 1
    for (;;) {
        auto slope = [&](float& x) {
            const float te = max_nan((x - base) * p.c, kNothing);
            x = exp2_fast(te) * (g.a + g.b * te);
        };
#pragma unroll
        for (int k = 0; k < kQuads; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) slope(r.v[k][i]);
        if (!Aligned) slope(r.extra);
        r.store(dx, tid);
        if (r.owns(at, tid)) dx[at] = g.at_target;
        if (r.step == 0) break;
        r.step -= kStep;
        r.template load<true>(x, tid);
    }
    if (isinf(g.a)) r.clear_nan(dx, tid);
}

// Rows whose sum s is below this are nearly certain.  1 - p of the largest logit, and log s beside an entropy of the same size, are then
// what the others sum to: s in fp32 has the error of its 1 in them (3 halves of a step of 1: 99 of 1 - p at this limit, and nothing is
// left of 1 - p = 1e-8).  The others are summed up once more for that one column, which takes another walk over a row that is in more
// than one part: 8192 x 8192 79 us without such rows, 88 where half are, 4000 x 32003 153 and 200 where all are.
constexpr float kNearlyCertain = 1.03125f;

// the lanes of this thread's group (of up to a warp)
template <int Group>
__device__ __forceinline__ unsigned group_mask()
{
    return Group < 32 ? ((1u << (Group & 31)) - 1) << (threadIdx.x & 31 & ~(Group - 1)) : kAllLanes;
}

// the sum of v over a group's lanes, in each of them (once per block); all reads that v is made of are done then
template <int Group>
__device__ __forceinline__ float group_sum(float v, unsigned mask, float* sh)
{
    v = warp_sum<(Group < 32 ? Group : 32)>(v, mask);
    if (Group < 256) return v;
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < Group / 32; i++) v += sh[i];
    return v;
}

// what the logits of a row but the largest sum to, this thread's share
template <int Group>
__device__ __forceinline__ float others_of_row(const float* x, int N, float top, float c, int tid)
{
    constexpr int V = Group < 32 ? 2 : 4;
    RowPart<Group, V, false> r;
    float sum = 0.0f;
    r.place(x, N);
#pragma unroll 1
    for (;; r.step += V * Group) {
        r.load(x, tid);
        auto add = [&](float v) { sum += v == top ? 0.0f : exp2_fast((v - top) * c); };
#pragma unroll
        for (int k = 0; k < V; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) add(r.v[k][i]);
        add(r.extra);
        if (r.step + V * Group >= r.quads) return sum;
    }
}

// The gradient of a row's logit x_j without the target's own part, p_j (-G - E (log p_j + H)), with p_j = 2^t / s, log p_j = log(2) t - log s:
// 2^t (a + b t).  (Roundings are spelled out where two kernels' results are to be the same bits.)
struct BwdSlope {
    float base, c, a, b;
    __device__ __forceinline__ BwdSlope(float top, float it, float s, float G, float E, float H)
    {
        const float inv = 1.0f / s;
        base = base_of(top);
        c = it * kLog2e;
        a = __fmul_rn(inv, E != 0.0f ? __fmaf_rn(-E, H - logf(s), -G) : -G);
        b = -inv * E * kLn2;
    }
    __device__ __forceinline__ float operator()(float x) const
    {
        const float te = max_nan((x - base) * c, kNothing);
        return __fmul_rn(exp2_fast(te), __fmaf_rn(b, te, a));
    }
};

// The gradient of a nearly certain row's largest logit where it is the target and where it is not: 1 - p = others / (1 + others),
// log p = -log(1 + others).
struct LargestGrad {
    float target, other;
};
__device__ __forceinline__ LargestGrad largest_grad(float others, float G, float E, float H)
{
    const float p = __fdividef(1.0f, 1.0f + others), Gp = __fmul_rn(G, p), Ep = E != 0.0f ? __fmul_rn(E * p, H - log1pf(others)) : 0.0f;
    return {__fsub_rn(__fmul_rn(Gp, others), Ep), __fsub_rn(-Gp, Ep)};
}

// A nearly certain row over the logits' own buffer, in more than one part: one group has them all, since each is needed before any is
// written over.
template <int Group>
__device__ __noinline__ void bwd_certain_row_in_place(float* x, int N, int t, const BwdSlope slope, float G, float E, float H, float* sh)
{
    const int tid = Group < 256 ? threadIdx.x % Group : threadIdx.x;
    const LargestGrad largest = largest_grad(group_sum<Group>(others_of_row<Group>(x, N, slope.base, slope.c, tid), group_mask<Group>(), sh), G, E, H);
    RowPart<Group, 2, false> r;
    r.place(x, N);
#pragma unroll 1
    for (;; r.step += 2 * Group) {
        r.load(x, tid);
        auto make = [&](float& v, int column) {
            const bool target = column == t;
            v = v == slope.base ? (target ? largest.target : largest.other) : target ? __fadd_rn(slope(v), G) : slope(v);
        };
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) make(r.v[k][i], r.column(tid, k) + i);
        make(r.extra, r.extra_column(tid));
        r.store(x, tid);
        if (r.step + 2 * Group >= r.quads) return;
    }
}

// A part, from column `first` on, its logits loaded, of a row that may be nearly certain.  `mask`: the lanes of the warp that come here.
template <bool Accumulate, bool Aligned, int Group, int V>
__device__ __forceinline__ void bwd_certain_part(RowPart<Group, V, Aligned>& r, const float (&old)[V][4], float old_extra, const float* x, float* dx, int first,
                                                 int N, int parts, int t, const BwdSlope& slope, float G, float E, float H, bool certain, int tid, unsigned mask,
                                                 float* sh)
{
    const auto each = [&](auto&& f) {
#pragma unroll
        for (int k = 0; k < V; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) f(r.v[k][i], Accumulate ? old[k][i] : 0.0f, r.column(tid, k) + i);
        if (!Aligned) f(r.extra, old_extra, r.extra_column(tid));
    };
    const float top = certain ? slope.base : CUDART_NAN_F;   // equal to no logit where the row needs nothing
    const bool any = Group > 8 || __any_sync(mask, certain);
    float top_before = 0.0f;
    int top_at = -1;   // where the largest logit is, in the thread that has it
    LargestGrad largest{0.0f, 0.0f};
    if (any && parts == 1) {
        float others = 0.0f;
        each([&](float v, float, int) { others += v == top ? 0.0f : exp2_fast((v - slope.base) * slope.c); });
        largest = largest_grad(group_sum<Group>(others, mask, sh), G, E, H);
    }
    each([&](float& v, float before, int column) {
        float o = slope(v);
        if (column == t - first) o = __fadd_rn(o, G);
        if (v == top) {
            o = column == t - first ? largest.target : largest.other;
            top_at = column;
            top_before = before;
        }
        v = Accumulate ? before + o : o;
    });
    r.store(dx, tid);
    if (!any || parts == 1) return;
    // in more than one part: the part that has the largest logit makes it when all else is
    if (Group == 256) {
        if (!__syncthreads_or(top_at >= 0)) return;
    } else {
        const unsigned have = __ballot_sync(mask, top_at >= 0) & group_mask<Group>();
        mask = Group < 32 ? __ballot_sync(mask, have != 0) : kAllLanes;
        if (have == 0) return;
    }
    largest = largest_grad(group_sum<Group>(others_of_row<Group>(x - first, N, slope.base, slope.c, tid), mask, sh), G, E, H);
    if (top_at >= 0) dx[top_at] = top_before + (top_at == t - first ? largest.target : largest.other);
}

// a part of a nearly certain row from its load on; a call, so that what it needs is not in the way of the rows that are not
template <bool Accumulate, bool Aligned, int Group, int V>
__device__ __noinline__ void bwd_certain_row(const float* x, float* dx, int first, int n, int N, int parts, int t, const BwdSlope slope, float G, float E, float H,
                                             int tid, float* sh)
{
    RowPart<Group, V, Aligned> r;
    float old[V][4], old_extra = 0.0f;
    r.place(x, n);
    r.load(x, tid);
    if (Accumulate) r.load_beside(dx, tid, old, old_extra);
    bwd_certain_part<Accumulate, Aligned, Group, V>(r, old, old_extra, x, dx, first, N, parts, t, slope, G, E, H, true, tid, kAllLanes, sh);
}

// Blocks per SM that the rows that are not nearly certain have room for.  Without the bound the others' way takes registers from them:
// 4 to 14 % of their time.
constexpr int bwd_blocks(bool accumulate, bool aligned, int group, int quads)
{
    const int registers = accumulate ? (aligned ? (group == 256 ? 48 : quads == 4 ? 56 : 40) : (group == 256 ? 64 : quads == 4 ? 72 : quads == 2 ? 48 : 40))
                                     : (group == 256 || quads <= 2 ? 40 : quads == 4 ? (aligned ? 48 : 56) : (aligned ? 64 : 72));
    return 65536 / (registers * (group < 256 ? 128 : group));
}

// dlogits of the log-probabilities from the forward's statistics.  A group of threads takes 4 * Group * V columns of a row, one of its
// `parts`; every load of the logits, and of the gradient that is added to, is under way before the first result is made.  8192 x 8192:
// 78 us, 6.5 TB/s.
template <bool Accumulate, bool Aligned, int Group, int V>
__global__ void __launch_bounds__(Group < 256 ? 128 : Group, bwd_blocks(Accumulate, Aligned, Group, V))
logprob_bwd_kernel(const float* logits, long long ld, const int32_t* __restrict__ targets, float it,
                   const float* __restrict__ stats, const float* __restrict__ entropy, const float* __restrict__ dlogp,
                   const float* __restrict__ dentropy, float* dlogits, long long ld_d, int M, int N, int parts, int part)
{
    __shared__ float sh[Group < 256 ? 1 : Group / 32];
    const int tid = Group < 256 ? threadIdx.x % Group : threadIdx.x;
    const unsigned unit = Group < 256 ? blockIdx.x * (128 / Group) + threadIdx.x / Group : blockIdx.x;
    const int row = (int)(unit / (unsigned)parts), first = (int)(unit % (unsigned)parts) * part, n = min(part, N - first);
    if (Group > 8 && row >= M) return;
    wait_for_previous_kernel();
    const bool there = row < M;
    const float* x = logits + (size_t)row * ld + first;
    float* dx = dlogits + (size_t)row * ld_d + first;
    const int t = there ? targets[row] : -1;
    const float s = there ? stats[2 * (size_t)row + 1] : 0.0f;
    const bool used = t >= 0 && t < N && s != 0.0f, certain = s < kNearlyCertain, whole = certain && parts > 1 && !Accumulate && x == dx;
    const unsigned lanes = Group == 8 ? __ballot_sync(kAllLanes, used && !whole) : kAllLanes;
    if (!used) {
        if (!Accumulate && there) RowPart<Group, V, Aligned>::clear(dx, n, tid);
        return;
    }
    if (certain && (whole || Group > 8)) {
        const float G = it * (dlogp ? dlogp[row] : 0.0f), E = it * (dentropy ? dentropy[row] : 0.0f), H = E != 0.0f ? entropy[row] : 0.0f;
        const BwdSlope slope(stats[2 * (size_t)row], it, s, G, E, H);
        if (!whole) bwd_certain_row<Accumulate, Aligned, Group, V>(x, dx, first, n, N, parts, t, slope, G, E, H, tid, sh);
        else if (first == 0) bwd_certain_row_in_place<Group>(dx, N, t, slope, G, E, H, sh);
        return;
    }
    RowPart<Group, V, Aligned> r;
    float old[V][4], old_extra = 0.0f;
    r.place(x, n);
    r.load(x, tid);
    if (Accumulate) r.load_beside(dx, tid, old, old_extra);
    const float G = it * (dlogp ? dlogp[row] : 0.0f), E = it * (dentropy ? dentropy[row] : 0.0f);
    if (Group == 8) {
        // several rows share a warp: one way for all of them, and the target's part with the rest (adding it to what is stored takes a
        // trip to memory at each warp's end: 65536 x 30 8.9 us)
        const float H = E != 0.0f ? entropy[row] : 0.0f;
        const BwdSlope slope(stats[2 * (size_t)row], it, s, G, E, H);
        bwd_certain_part<Accumulate, Aligned, Group, V>(r, old, old_extra, x, dx, first, N, parts, t, slope, G, E, H, certain, tid, lanes, sh);
        return;
    }
    // as BwdSlope (which reads the entropy whether or not it is needed yet: 3 % of 8192 x 8192)
    const float base = base_of(stats[2 * (size_t)row]), c = it * kLog2e, inv = 1.0f / s;
    const float a = inv * (-G - (E != 0.0f ? E * (entropy[row] - logf(s)) : 0.0f)), b = -inv * E * kLn2;
    auto make = [&](float& x, float before) {
        const float te = max_nan((x - base) * c, kNothing), o = exp2_fast(te) * (a + b * te);
        x = Accumulate ? before + o : o;
    };
#pragma unroll
    for (int k = 0; k < V; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) make(r.v[k][i], Accumulate ? old[k][i] : 0.0f);
    if (!Aligned) make(r.extra, old_extra);
    r.store(dx, tid);
    if (r.owns(t - first, tid)) dx[t - first] += G;
}

// The number of rows that are not left out, and (with_sum) the sum of w_i token_loss_i; fixed order.  A cluster of blocks for
// many rows.
__global__ void __launch_bounds__(1024)
policy_total_kernel(const int32_t* __restrict__ targets, const float* __restrict__ weights, const float* __restrict__ token_loss,
                    float* __restrict__ loss, int M, int with_sum)
{
    __shared__ double sh[32], sh_all[2][8];
    const int ranks = cluster_size(), rank = cluster_rank();
    if (ranks > 1) cluster_sync_all();   // a block must run before another writes to its memory
    wait_for_previous_kernel();
    int rows = 0;
    double sum = 0.0;
#pragma unroll 8
    for (unsigned i = rank * 1024 + threadIdx.x; i < (unsigned)M; i += ranks * 1024) {   // no branch between the loads: all of a step's are under way at once
        const float w = weights ? weights[i] : 1.0f, l = with_sum ? token_loss[i] : 0.0f;
        const bool used = targets[i] >= 0 && w != 0.0f;
        rows += used ? 1 : 0;
        sum += used ? (double)w * (double)l : 0.0;
    }
    double count = block_sum((double)rows, sh);
    if (with_sum) sum = block_sum(sum, sh);
    if (ranks > 1) {
        if (threadIdx.x == 0) {
            cluster_store(&sh_all[0][rank], 0, count);
            cluster_store(&sh_all[1][rank], 0, sum);
        }
        cluster_sync_all();
        count = sum = 0.0;
        for (int i = 0; i < ranks; i++) {
            count += sh_all[0][i];
            sum += sh_all[1][i];
        }
    }
    if (threadIdx.x == 0 && rank == 0) {
        loss[1] = (float)count;
        if (with_sum) loss[0] = (float)(weights ? sum : count > 0.0 ? sum / count : 0.0);
    }
}

// What a pair's margin makes of it: its loss, and the slope of the mean loss by the margin.
struct PairTerms {
    double loss, slope;
};

__device__ __forceinline__ PairTerms pair_terms(double m, double eps, int P)
{
    const double e = exp(-fabs(m)), soft = log1p(e), inv = 1.0 / (1.0 + e);   // log(1 + e^-|m|), sigmoid(|m|): no overflow either way
    PairTerms t;
    t.loss = (1.0 - eps) * (soft + fmax(-m, 0.0));
    if (eps != 0.0) t.loss += eps * (soft + fmax(m, 0.0));   // (without smoothing an infinite margin costs nothing, where 0 * inf would be NaN)
    t.slope = (eps - (m >= 0.0 ? e * inv : inv)) / (double)P;   // -(1 - eps) sigmoid(-m) + eps sigmoid(m)
    return t;
}

// A block (or a cluster of blocks, for long sequences) per pair: the two sums, the pair's loss, the gradient of its rows.
// Small: one block has every pair, a warp each, and the mean as well.  The gradient is the same for all rows of a sequence, so the
// second walk reads nothing but which rows are left out.  Bound by HBM where there is enough: 12 to 16 bytes per row; 700 pairs of
// 2000 rows are a chain of loads, two sums, an exponential and a logarithm in fp64, and the mean's launch: 11.6 us (floor 3.4).
template <bool Small, int Threads>
__global__ void __launch_bounds__(Threads)
preference_pair_kernel(const float* __restrict__ logp, const float* __restrict__ ref_logp, const int32_t* __restrict__ targets,
                       const int32_t* __restrict__ offsets, float beta, float smoothing, float margin, int by_length,
                       float* __restrict__ loss, float* __restrict__ pair_loss, float* __restrict__ rewards, float* __restrict__ dlogp,
                       int P, int M, int* __restrict__ status)
{
    constexpr int kBatch = 8;   // rows per thread whose loads are under way at once
    __shared__ double sh[Threads / 32][4], sh_all[8][4];
    __shared__ float sh_slope[2];
    const int ranks = cluster_size(), rank = cluster_rank(), tid = Small ? threadIdx.x & 31 : threadIdx.x;
    if (ranks > 1) cluster_sync_all();   // a block must run before another writes to its memory
    wait_for_previous_kernel();
    const int pair = Small ? threadIdx.x >> 5 : blockIdx.x / ranks;
    const unsigned step = Small ? 32 : Threads * ranks, start = Small ? tid : rank * Threads + tid;
    int o[3];
    for (int k = 0; k < 3; k++) o[k] = offsets[2 * pair + k];
    const bool usable = o[0] >= 0 && o[1] >= o[0] && o[2] >= o[1] && o[2] <= M;   // the same in every block of the pair
    // of the ratios and of the rows, for both sequences: their rows lie one after the other, so one walk makes all four
    double sums[4] = {0.0, 0.0, 0.0, 0.0};
    // (an unusable pair's range is empty, whatever its offsets say)
    const unsigned begin = usable ? o[0] : 0, middle = usable ? o[1] : 0, end = usable ? o[2] : 0;
    int rows[2] = {0, 0};
    for (unsigned i0 = begin + start; i0 < end; i0 += kBatch * step) {
        float a[kBatch], b[kBatch];
        int t[kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; q++) {
            const unsigned i = i0 + q * step;
            const bool in = i < end;
            a[q] = in ? logp[i] : 0.0f;
            b[q] = in && ref_logp ? ref_logp[i] : 0.0f;
            t[q] = !in ? -1 : targets ? targets[i] : 0;
        }
#pragma unroll
        for (int q = 0; q < kBatch; q++) {
            const bool first = i0 + q * step < middle;
            const double d = t[q] >= 0 ? (double)a[q] - (double)b[q] : 0.0;
            const int one = t[q] >= 0 ? 1 : 0;
            if (first) {
                sums[0] += d;
                rows[0] += one;
            } else {
                sums[1] += d;
                rows[1] += one;
            }
        }
    }
    sums[2] = __reduce_add_sync(kAllLanes, rows[0]);
    sums[3] = __reduce_add_sync(kAllLanes, rows[1]);
#pragma unroll
    for (int l = 16; l > 0; l >>= 1)
#pragma unroll
        for (int k = 0; k < 2; k++) sums[k] += __shfl_xor_sync(kAllLanes, sums[k], l);
    if (!Small) {
        if ((tid & 31) == 0)
            for (int k = 0; k < 4; k++) sh[tid >> 5][k] = sums[k];
        __syncthreads();
        if (tid < 32) {
#pragma unroll
            for (int k = 0; k < 4; k++) sums[k] = tid < Threads / 32 ? sh[tid][k] : 0.0;
            sums[2] = __reduce_add_sync(kAllLanes, (int)sums[2]);
            sums[3] = __reduce_add_sync(kAllLanes, (int)sums[3]);
#pragma unroll
            for (int l = Threads / 64; l > 0; l >>= 1)
#pragma unroll
                for (int k = 0; k < 2; k++) sums[k] += __shfl_xor_sync(kAllLanes, sums[k], l);
        }
        if (ranks > 1) {
            if (tid < ranks)
                for (int k = 0; k < 4; k++) cluster_store(&sh_all[rank][k], tid, sums[k]);
            cluster_sync_all();
            if (tid == 0)
                for (int k = 0; k < 4; k++) {
                    sums[k] = 0.0;
                    for (int i = 0; i < ranks; i++) sums[k] += sh_all[i][k];
                }
        }
    }
    float slopes[2] = {0.0f, 0.0f};
    if (tid == 0) {
        double share[2], reward[2];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            share[k] = !by_length ? (double)beta : sums[2 + k] > 0.0 ? (double)beta / sums[2 + k] : 0.0;
            reward[k] = usable ? share[k] * sums[k] : CUDART_NAN;
        }
        const PairTerms t = pair_terms(reward[0] - reward[1] - (double)margin, (double)smoothing, P);
        slopes[0] = (float)(t.slope * share[0]);
        slopes[1] = (float)(-t.slope * share[1]);
        if (rank == 0) {
            pair_loss[pair] = (float)t.loss;
            if (!Small && P == 1) *loss = (float)t.loss;
            rewards[2 * pair] = (float)reward[0];
            rewards[2 * pair + 1] = (float)reward[1];
            if (!usable && status) atomicOr(status, ZNN_DEV_BAD_INDEX);
        }
        if (Small) sh[pair][0] = (double)(float)t.loss;   // the mean is that of the losses as rounded
        sh_slope[0] = slopes[0];
        sh_slope[1] = slopes[1];
    }
    __syncthreads();
    if (Small) {
        if (threadIdx.x == 0) {
            double sum = 0.0;
            for (int i = 0; i < P; i++) sum += sh[i][0];
            *loss = (float)(sum / (double)P);
        }
        slopes[0] = __shfl_sync(kAllLanes, slopes[0], 0);
        slopes[1] = __shfl_sync(kAllLanes, slopes[1], 0);
    } else {
        slopes[0] = sh_slope[0];
        slopes[1] = sh_slope[1];
    }
    if (!usable || !dlogp) return;
    for (unsigned i0 = begin + start; i0 < end; i0 += kBatch * step) {
        int t[kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; q++) {
            const unsigned i = i0 + q * step;
            t[q] = targets && i < end ? targets[i] : 0;
        }
#pragma unroll
        for (int q = 0; q < kBatch; q++) {
            const unsigned i = i0 + q * step;
            if (i < end) dlogp[i] = t[q] < 0 ? 0.0f : i < middle ? slopes[0] : slopes[1];
        }
    }
}

__global__ void __launch_bounds__(1024) mean_kernel(const float* __restrict__ v, float* __restrict__ out, int n)
{
    __shared__ double sh[32];
    wait_for_previous_kernel();
    double s = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += 1024) s += (double)v[i];
    s = block_sum(s, sh);
    if (threadIdx.x == 0) out[0] = (float)(s / (double)n);
}

}  // namespace znn

using namespace znn;

// ---- launches
template <bool Policy, bool Entropy, bool Aligned, int Group, int V, int Rows>
static int launch_held(const RowParams& p)
{
    constexpr int rows = 128 / Group * Rows;
    return launch_overlapped(rows_held_kernel<Policy, Entropy, Aligned, Group, V, Rows>, "rows_held_kernel", (p.M + (long long)rows - 1) / rows, 128, 1, p);
}

template <bool Policy, bool Entropy, bool Aligned, int Threads>
static int launch_walk(const RowParams& p, int ranks)
{
    const int part = (ceil_div(p.N, ranks) + 3) & ~3;   // parts start where the row's quads do
    if constexpr (Threads < 256) {
        // rows of a few steps: six quads a thread where those cover fewer columns that are not there (policy 60000 x 2100: 177 us with
        // six, 184 with eight; 60000 x 2000: 172 and 161; log-probabilities 65536 x 1100: 66 and 74)
        if (part <= 12288 && 6 * ceil_div(part, 24 * Threads) < 8 * ceil_div(part, 32 * Threads))
            return launch_overlapped(rows_walk_kernel<Policy, Entropy, Aligned, Threads, 6>, "rows_walk_kernel", (long long)p.M * ranks, Threads, ranks,
                          p, part);
    }
    return launch_overlapped(rows_walk_kernel<Policy, Entropy, Aligned, Threads, 8>, "rows_walk_kernel", (long long)p.M * ranks, Threads, ranks,
                  p, part);
}

// Which kernel: 8 lanes per row up to 256 columns, a warp up to 1024, then blocks that walk.  Rows held at a time (us, 1 / 2 / 4, policy
// loss of 65536 rows): 30 columns 22.3 / - / 19.0 (8: 21.7), 50 24.4 / 22.2 / 23.8, 100 29.0 / 27.6 / 30.3, 200 36.2 / 41.4 / -,
// 400 59.1 / 53.2 / 53.4, 1000 95 / 95 / -.  A walking block costs the same few reductions whatever its size, so the smallest one that
// a few steps suffice wins; the policy loss, which walks twice, wants its rows in flight to stay in L2 between the walks and so
// spreads long rows over clusters.  Measured (us, 32 / 64 / 128 / 256 threads):
//   policy   40000 x 2000: 111 / 125 / 183 / 339,  40000 x 2600: 145 / 156 / - / -,  20000 x 4096: 133 / 114 / 120 / 185,  10000 x 8192: - / 135 / 112 / 124,
//            4000 x 20000: - / - / 140 / 120;  256 threads in clusters of 1 / 2 / 4 / 8: 2500 x 32000: 133 / 117 / 139 / -,
//            1500 x 65536: 180 / 162 / 143 / 165,  700 x 131072: - / - / 152 / 136
//   logprob  40000 x 2000: 54 / 66 / 105 / 220,  20000 x 4099: 54 / 55 / 58 / 117,  20000 x 5000: 62 / 67 / - / -,  4000 x 20000: - / 59 / 54 / 59,
//            1000 x 100000: - / - / 66 / 67,  2045 x 50257 (1.7 times the blocks of 128 threads that are resident at once): - / 57 / 60 / 58
// The loss alone (no dlogits) goes by the same rule, although it walks once: 8192 x 8192 56 us, 2048 x 131000 215, 40000 x 2600 87, where
// the log-probabilities' sizes take 43, 164 and 73.
// Few rows are spread over clusters, as many as let all blocks run at once: 32 x 131072 takes 7.4 us with eight blocks per row, 8.7
// with four; policy 100 x 130000 31.4 and 27.5, 320 x 130000 73 and 77, 320 x 32000 27.3 with two and 24.2 with one.
template <bool Policy, bool Entropy, bool Aligned>
static int launch_rows_as(const RowParams& p)
{
    if (p.N <= 32) return launch_held<Policy, Entropy, Aligned, 8, 1, 4>(p);
    if (p.N <= 64) return launch_held<Policy, Entropy, Aligned, 8, 2, 2>(p);
    if (p.N <= 128) return launch_held<Policy, Entropy, Aligned, 8, 4, 2>(p);
    if (p.N <= 256) return launch_held<Policy, Entropy, Aligned, 8, 8, 1>(p);
    if (p.N <= 512) return launch_held<Policy, Entropy, Aligned, 32, 4, 2>(p);
    if (p.N <= 1024) return launch_held<Policy, Entropy, Aligned, 32, 8, 1>(p);
    if (p.M < (Policy ? 3 : 2) * sm_count() && p.N > 2048) {
        int ranks = Policy && p.N > 102400 && p.M >= sm_count() ? 8 : 1;
        while (ranks < 8 && p.N > 8192 * ranks && (long long)p.M * ranks < 2 * sm_count()) ranks *= 2;
        return launch_walk<Policy, Entropy, Aligned, 256>(p, ranks);
    }
    if (p.N <= (Policy ? 2816 : 5120)) return launch_walk<Policy, Entropy, Aligned, 32>(p, 1);
    if (p.N <= (Policy ? 5120 : 8192)) return launch_walk<Policy, Entropy, Aligned, 64>(p, 1);
    if constexpr (!Policy) {
        // long rows: where the blocks of a size smaller or larger are all resident at once, that size (an SM has 1024 threads of them)
        const int slots = sm_count() * (1024 / 64);
        if (p.M <= slots / 4) return launch_walk<Policy, Entropy, Aligned, 256>(p, 1);
        if (p.M > slots / 2 && p.M <= slots) return launch_walk<Policy, Entropy, Aligned, 64>(p, 1);
        return launch_walk<Policy, Entropy, Aligned, 128>(p, 1);
    }
    if (p.N <= 12288) return launch_walk<Policy, Entropy, Aligned, 128>(p, 1);
    return launch_walk<Policy, Entropy, Aligned, 256>(p, p.N <= 25600 ? 1 : p.N <= 51200 ? 2 : p.N <= 102400 ? 4 : 8);
}

// every row of the matrix starts with a 16-byte quad and has whole quads only
static bool rows_aligned(const float* m, long long ld, int N) { return ((uintptr_t)m & 15) == 0 && ld % 4 == 0 && N % 4 == 0; }

template <bool Policy>
static int launch_rows(const RowParams& p, bool entropy)
{
    if (rows_aligned(p.logits, p.ld, p.N) && (!p.dlogits || rows_aligned(p.dlogits, p.ld_d, p.N)))
        return entropy ? launch_rows_as<Policy, true, true>(p) : launch_rows_as<Policy, false, true>(p);
    return entropy ? launch_rows_as<Policy, true, false>(p) : launch_rows_as<Policy, false, false>(p);
}

struct BwdArgs {
    const float* logits;
    long long ld;
    const int32_t* targets;
    float it;
    const float *stats, *entropy, *dlogp, *dentropy;
    float* dlogits;
    long long ld_d;
    int M, N;
};

template <bool Accumulate, bool Aligned, int Group, int V>
static int launch_bwd(const BwdArgs& b)
{
    constexpr int rows = Group < 256 ? 128 / Group : 1;
    constexpr int fit = 4 * Group * V;
    const int part = (ceil_div(b.N, ceil_div(b.N, fit)) + 3) & ~3, parts = ceil_div(b.N, part);
    const long long units = (long long)b.M * parts;
    return launch_overlapped(logprob_bwd_kernel<Accumulate, Aligned, Group, V>, "logprob_bwd_kernel", (units + rows - 1) / rows, Group < 256 ? 128 : Group, 1,
                  b.logits, b.ld, b.targets, b.it, b.stats, b.entropy, b.dlogp, b.dentropy, b.dlogits, b.ld_d, b.M, b.N, parts, part);
}

// Pieces of a row for 8 lanes, a warp or a block: a piece must be nearly full and its loads all under way at once; those of a gradient
// that is added to are as many again.  Measured (us, stored / added to, 65536 rows: 30 columns by 8 lanes with one quad 6.4, with two 7.8,
// 200 columns by 8 lanes 20.3 / 26.6, by a warp 27.0 / 34.3,
// 400 37.0 / 47.8 and 35.9 / 46.4, 1100 by warps with 4 quads 95.9 / 124, with 8 93.1 / 140, by blocks 121 / 174; 30000 x 4101: 163 / 229,
// 149 / 245, 191 / 289; 20000 x 6200 with 4 quads 149, with 8 145, by blocks 154; 4000 x 32003: 160 / 215, 149 / 216, 150 / 210).
template <bool Accumulate, bool Aligned>
static int launch_bwd_as(const BwdArgs& b)
{
    if (b.N <= 32) return launch_bwd<Accumulate, Aligned, 8, 1>(b);
    if (b.N <= 64) return launch_bwd<Accumulate, Aligned, 8, 2>(b);
    if (b.N <= 384) return launch_bwd<Accumulate, Aligned, 8, 4>(b);
    if (b.N <= 512) return launch_bwd<Accumulate, Aligned, 32, 4>(b);
    if (b.N < 8192) return launch_bwd<Accumulate, Aligned, 32, Accumulate ? 4 : 8>(b);
    return launch_bwd<Accumulate, Aligned, 256, 4>(b);
}

static int check_rows(const float* logits, long long ld, const int32_t* targets, float inv_temp, int M, int N)
{
    ZNN_REQUIRE(M >= 0 && N > 0, "M must not be negative and N must be positive");
    ZNN_REQUIRE(M == 0 || (logits && targets), "NULL pointer");
    ZNN_REQUIRE(ld >= N, "ld = %lld is smaller than N = %d", ld, N);
    ZNN_REQUIRE(((uintptr_t)logits & 3) == 0, "logits are not aligned to 4 bytes");
    ZNN_REQUIRE(inv_temp > 0.0f && inv_temp < 1e38f, "inv_temp must be positive and finite (below 1e38)");
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
    p.logits = logits; p.ld = ld; p.targets = targets; p.it = inv_temp; p.c = (float)(inv_temp * 1.4426950408889634); p.M = M; p.N = N;
    p.logp = logp; p.entropy = entropy; p.stats = stats; p.status = device_status_word();
    return launch_rows<false>(p, entropy != nullptr);
}

int znn_token_logprob_bwd(const float* logits, long long ld, const int32_t* targets, float inv_temp, const float* stats,
                          const float* entropy, const float* dlogp, const float* dentropy, float* dlogits, long long ld_d,
                          int accumulate, int M, int N)
{
    const int rc = check_rows(logits, ld, targets, inv_temp, M, N);
    if (rc != ZNN_OK) return rc;
    if (M == 0) return ZNN_OK;
    ZNN_REQUIRE(stats && dlogits, "stats/dlogits is NULL");
    ZNN_REQUIRE(((uintptr_t)dlogits & 3) == 0, "dlogits are not aligned to 4 bytes");
    ZNN_REQUIRE(!dentropy || entropy, "dentropy needs the forward's entropy");
    ZNN_REQUIRE(ld_d >= N, "ld_d = %lld is smaller than N = %d", ld_d, N);
    ZNN_REQUIRE(dlogits != logits || (ld_d == ld && !accumulate), "dlogits may be the logits' own buffer only with ld_d == ld and accumulate = 0");
    ZNN_NEED_DEVICE();
    const BwdArgs b{logits, ld, targets, inv_temp, stats, entropy, dlogp, dentropy, dlogits, ld_d, M, N};
    if (rows_aligned(logits, ld, N) && rows_aligned(dlogits, ld_d, N)) return accumulate ? launch_bwd_as<true, true>(b) : launch_bwd_as<false, true>(b);
    return accumulate ? launch_bwd_as<true, false>(b) : launch_bwd_as<false, false>(b);
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
    ZNN_REQUIRE(((uintptr_t)dlogits & 3) == 0, "dlogits are not aligned to 4 bytes");
    ZNN_REQUIRE(isfinite(kl_coef) && isfinite(entropy_coef), "kl_coef and entropy_coef must be finite");
    ZNN_REQUIRE(ref_logp || kl_coef == 0.0f, "kl_coef needs ref_logp");
    ZNN_REQUIRE(clip_low >= 0.0f && clip_low <= 1.0f && clip_high >= 0.0f && isfinite(clip_high),
                "clip_low must lie in [0, 1], clip_high must not be negative");
    ZNN_REQUIRE(!dlogits || ld_d >= N, "ld_d = %lld is smaller than N = %d", ld_d, N);
    ZNN_REQUIRE(dlogits != logits || ld_d == ld, "dlogits may be the logits' own buffer only with ld_d == ld");
    ZNN_NEED_DEVICE();
    RowParams p{};
    p.logits = logits; p.ld = ld; p.targets = targets; p.it = inv_temp; p.c = (float)(inv_temp * 1.4426950408889634); p.M = M; p.N = N;
    p.logp = logp; p.entropy = entropy; p.status = device_status_word();
    p.old_logp = old_logp; p.ref_logp = ref_logp; p.advantages = advantages; p.weights = weights;
    p.clip_low = clip_low; p.clip_high = clip_high; p.kl_coef = kl_coef; p.entropy_coef = entropy_coef;
    p.token_loss = token_loss; p.dlogits = dlogits; p.ld_d = ld_d;
    const int total_ranks = M > 4096 ? 8 : 1;
    if (!weights && M > 512) {   // the rows' weight 1 / count is needed before their gradients are written
        p.count = loss + 1;
        const int counted = launch_overlapped(policy_total_kernel, "policy_total_kernel", total_ranks, 1024, total_ranks, targets, weights, token_loss, loss, M, 0);
        if (counted != ZNN_OK) return counted;
    }
    const int done = launch_rows<true>(p, entropy || entropy_coef != 0.0f);
    if (done != ZNN_OK) return done;
    return launch_overlapped(policy_total_kernel, "policy_total_kernel", total_ranks, 1024, total_ranks, targets, weights, token_loss, loss, M, 1);
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
#define ZNN_PAIRS(small, threads, blocks, used, ranks)                                                                                    \
    launch_overlapped(preference_pair_kernel<small, threads>, "preference_pair_kernel", blocks, used, ranks, logp, ref_logp, targets, seq_offsets, \
           beta, label_smoothing, margin, length_normalize, loss, pair_loss, rewards, dlogp, P, M, device_status_word())
    // A warp per pair in one launch for small calls: 32 pairs of 256 rows 5.2 us, 8 of 1024 5.5, where the next forms' two launches take 6.1
    // (32 x 260, 16 x 520).  (The limit counts the call's rows.  One to four pairs that fill it are slower this way: 4 x 2048 7.6 us, 2 x
    // 4096 13.3, 1 x 8192 24.7, against 6.1 for 4 x 4096 and 7.4 for 2 x 8192.)  Few pairs of long sequences: eight blocks each, where one
    // block's own bandwidth (about 100 GB/s) would be the limit.  Many short ones: small blocks.
    if (P <= 32 && M <= 8192) return ZNN_PAIRS(true, 1024, 1, 32 * P, 1);
    const int rows = M / P;
    const int rc = rows > 8192 && P <= 32              ? ZNN_PAIRS(false, 1024, 8LL * P, 1024, 8)
                   : rows > 8192 && P < 2 * sm_count() ? ZNN_PAIRS(false, 256, 8LL * P, 256, 8)
                   : rows > 1024                       ? ZNN_PAIRS(false, 256, P, 256, 1)
                                                       : ZNN_PAIRS(false, 64, P, 64, 1);
#undef ZNN_PAIRS
    if (rc != ZNN_OK || P == 1) return rc;   // (a single pair's loss is the mean)
    return launch_overlapped(mean_kernel, "mean_kernel", 1, 1024, 1, (const float*)pair_loss, loss, P);
}

}  // extern "C"
