// ml4tspbench_amd/csrc/policy_loss.hip -- losses on the step log-probabilities of tours
//
// Clipped policy loss, per kept step (or, ratio = tour, with x summed over a tour's kept steps):
//     x = lp - old,  r = exp x,  l = max(-r A, -clip(r, lo, hi) A),      d = ref - lp,  kl = exp d - 1 - d
// Preference loss over pairs (a, b) of one instance's tours, a the shorter, with s = beta sum(lp - ref):
//     l = -(1 - eps) log sigmoid(s_a - s_b) - eps log sigmoid(s_b - s_a)
// Both are averages; the gradients are recomputed from the same inputs in one pass.  Sums over steps and rows are
// kept in double and added in a fixed order: results do not depend on the schedule.  What is summed is a float: a step's
// or a pair's term carries a few 2^-24 of itself (a score difference z is rounded to float, and its sigmoid is off by
// |z| 2^-24 of itself for it), the precision that loss and gradient are given in.
//
// A row of steps is read by a group of G threads: 8 or 16 for short rows, a wave, or for long rows of few tours a whole
// workgroup.  Bound by memory where there is much (10000 x 1000 steps in float32 with reference and mask: 130 MB read in
// 39 us, 3.4 TB/s, and 170 MB moved by the gradient in 33 us, 5.2 TB/s), by the launches and the host's autograd where
// there is little: up to kOneBlock steps one workgroup does everything, sums and end, in one launch.
#include "learn_common.hpp"

#include <type_traits>

namespace t2o {

constexpr int kMaxBlocks = 2048;        // partial sums the finishing workgroup adds up
constexpr int kBlockRow = 1024;         // threads of a workgroup that has a row to itself
constexpr int64_t kOneBlock = 8192;     // steps that one workgroup of kOneThreads takes in one launch
constexpr int kOneThreads = 1024;
constexpr int kRatioTour = 1, kAverageTour = 2;

struct PolicyParams {
    const void *lp, *old, *ref;
    const float* adv;
    const uint8_t* mask;
    int64_t T, S;
    int32_t adv_per_step, mode;
    float lo, hi;
    double kl_coef, log_lo, log_hi;
    float *loss, *stats;    // stats: kl, clip fraction
    double* partial;        // [blocks][4]; with one block unused
    double* norm;           // 1 / what the averages divide by
    double2* rows;          // (T): gradient of the ratio term w.r.t. a whole tour's x; 1 / kept steps
    const float* g;
    void* grad;
};

// Terms are computed as float, and where that gives no finite number again as double: a term past the range of float
// may be in an average inside that range, and an advantage of 0 makes its own 0.  (All terms as double: 10000 x 1000
// steps 39 + 33 -> 42 + 35 us.)
// e^x as double: float's exponential, above 80 times e^80.  inf above 168, where no average of 2^62 steps is finite.
template <typename F>
__device__ __forceinline__ F exp_as(double x)
{
    if constexpr (sizeof(F) == 4) return expf((float)x);
    const bool far = x > 80.0;
    const double e = (double)expf((float)(far ? x - 80.0 : x));
    return (F)(far ? e * 5.54062238439351e34 : e);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < __builtin_inff(); }

// exp(d) - 1 - d.  Near 0 it is about d^2 / 2 and the subtraction would lose it: the series (to d^11, 2e-9 of the
// result at |d| = 1) instead.
template <typename F>
__device__ __forceinline__ F kl_term(float d)
{
    if (fabsf(d) > 1.0f) return (exp_as<F>((double)d) - (F)1) - (F)d;
    float s = 1.0f / 11.0f;
    s = fmaf(s * d, 0.1f, 0.1f);
    s = fmaf(s * d, 1.0f / 9.0f, 1.0f / 9.0f);
    s = fmaf(s * d, 1.0f / 8.0f, 1.0f / 8.0f);
    s = fmaf(s * d, 1.0f / 7.0f, 1.0f / 7.0f);
    s = fmaf(s * d, 1.0f / 6.0f, 1.0f / 6.0f);
    s = fmaf(s * d, 1.0f / 5.0f, 1.0f / 5.0f);
    s = fmaf(s * d, 1.0f / 4.0f, 1.0f / 4.0f);
    s = fmaf(s * d, 1.0f / 3.0f, 1.0f / 3.0f);
    s = fmaf(s * d, 1.0f / 2.0f, 1.0f / 2.0f);
    return (F)(s * d * d);
}

// The ratio term of one step or tour.  The gradient jumps where the ratio leaves [lo, hi]; the side is decided on x in
// double, where the difference of two floats is as good as exact.
__device__ __forceinline__ bool is_cut(const PolicyParams& p, float adv, double x)
{
    return (adv > 0.0f && x > p.log_hi) || (adv < 0.0f && x < p.log_lo);
}

// -adv e^x where it is not cut; 0 for an advantage of 0 and any x below inf (the steps of a long tour sum up to an e^x
// past every range, which would give 0 times inf).
template <typename F>
__device__ __forceinline__ F ratio_term(float adv, double x)
{
    if (sizeof(F) == 8 && adv == 0.0f && x < __builtin_inf()) return (F)0;
    return -(F)adv * exp_as<F>(x);
}

// Sum over a group of G threads (over the workgroup where G is more than a wave), in every thread of it.
template <int G, int N>
__device__ __forceinline__ void group_sum(double (&v)[N])
{
#pragma unroll
    for (int c = 0; c < N; ++c)
        for (int o = (G < 64 ? G : 64) / 2; o >= 1; o >>= 1) v[c] += __shfl_xor(v[c], o);
    if constexpr (G > 64) {
        __shared__ double part[G / 64][N];
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
            for (int c = 0; c < N; ++c) part[threadIdx.x >> 6][c] = v[c];
        __syncthreads();
        for (int c = 0; c < N; ++c) {
            double s = 0.0;
            for (int w = 0; w < (int)blockDim.x / 64; ++w) s += part[w][c];
            v[c] = s;
        }
    }
}

// The group of G threads that a thread belongs to, and how many there are.
template <int G>
struct Groups {
    int64_t first, count;
    int at;
    __device__ Groups()
    {
        const int64_t t = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
        first = t / G;
        count = (int64_t)gridDim.x * blockDim.x / G;
        at = (int)(t % G);
    }
};

// f(step) for the steps of a row that thread `at` of a group of G has: four at a time as long as there are, so that
// their loads are in flight together.  f<N>(first) does steps first, first + G, ..., N of them.
template <int G, typename F>
__device__ __forceinline__ void for_steps(int at, int64_t S, F f)
{
    int64_t s = at;
    for (; s + 3 * G < S; s += 4 * G) f(std::integral_constant<int, 4>(), s);
    for (; s + G < S; s += 2 * G) f(std::integral_constant<int, 2>(), s);
    if (s < S) f(std::integral_constant<int, 1>(), s);
}

// The values of steps i, i + G, ...: one branch an array, its loads together.
template <typename E, int N, int G>
__device__ __forceinline__ void load_steps(const void* from, int64_t i, bool there, float otherwise, float (&to)[N])
{
    if (there) {
#pragma unroll
        for (int u = 0; u < N; ++u) to[u] = widen(static_cast<const E*>(from)[i + u * G]);
    } else {
#pragma unroll
        for (int u = 0; u < N; ++u) to[u] = otherwise;
    }
}

template <int N, int G>
__device__ __forceinline__ void load_kept(const uint8_t* mask, int64_t i, uint8_t (&kept)[N])
{
    if (mask) {
#pragma unroll
        for (int u = 0; u < N; ++u) kept[u] = mask[i + u * G];
    } else {
#pragma unroll
        for (int u = 0; u < N; ++u) kept[u] = 1;
    }
}

__device__ __forceinline__ void policy_end(const PolicyParams& p, const double (&v)[4])
{
    const double inv = v[3] > 0.0 ? 1.0 / v[3] : 0.0, kl = v[1] * inv;
    p.norm[0] = inv;
    p.loss[0] = (float)(v[0] * inv + (p.kl_coef != 0.0 ? p.kl_coef * kl : 0.0));
    p.stats[0] = (float)kl;
    p.stats[1] = (float)(v[2] * inv);
}

__device__ __forceinline__ float cut_term(const PolicyParams& p, float adv) { return -adv * (adv > 0.0f ? p.hi : p.lo); }

// A thread's sums of a row again, of terms as double.
template <typename E, int G>
__device__ void far_sums(const PolicyParams& p, int64_t k, int at, float of_tour, double& ratio, double& kl)
{
    ratio = kl = 0.0;
    for (int64_t s = at; s < p.S; s += G) {
        const int64_t i = k * p.S + s;
        if (p.mask && !p.mask[i]) continue;
        const float lp = widen(static_cast<const E*>(p.lp)[i]);
        if (!(p.mode & kRatioTour)) {
            const float adv = p.adv_per_step ? p.adv[i] : of_tour;
            const double x = (double)lp - (double)widen(static_cast<const E*>(p.old)[i]);
            ratio += is_cut(p, adv, x) ? (double)cut_term(p, adv) : ratio_term<double>(adv, x);
        }
        if (p.ref) kl += kl_term<double>(widen(static_cast<const E*>(p.ref)[i]) - lp);
    }
}

template <typename E, int G>
__global__ __launch_bounds__(1024) void k_policy(PolicyParams p)
{
    const Groups<G> g;
    double sum[4] = {0.0, 0.0, 0.0, 0.0};               // ratio term, kl, clipped, weight
    for (int64_t k = g.first; k < p.T; k += g.count) {
        double v[5] = {0.0, 0.0, 0.0, 0.0, 0.0};        // ratio term, kl, clipped, steps, difference of the tour
        const float of_tour = p.adv_per_step ? 0.0f : p.adv[k];
        for_steps<G>(g.at, p.S, [&](auto many, int64_t first) {
            constexpr int N = decltype(many)::value;
            float lp[N], old[N], ref[N], adv[N];
            uint8_t kept[N];
            const int64_t i = k * p.S + first;
            load_steps<E, N, G>(p.lp, i, true, 0.0f, lp);
            load_steps<E, N, G>(p.old, i, true, 0.0f, old);
            load_steps<E, N, G>(p.ref, i, p.ref, 0.0f, ref);
            load_steps<float, N, G>(p.adv, i, p.adv_per_step, of_tour, adv);
            load_kept<N, G>(p.mask, i, kept);
#pragma unroll
            for (int u = 0; u < N; ++u) {
                if (!kept[u]) continue;
                const double x = (double)lp[u] - (double)old[u];
                v[3] += 1.0;
                if (p.mode & kRatioTour) {
                    v[4] += x;
                } else {
                    const bool cut = is_cut(p, adv[u], x);
                    v[0] += (double)(cut ? cut_term(p, adv[u]) : ratio_term<float>(adv[u], x));
                    v[2] += cut ? 1.0 : 0.0;
                }
                if (p.ref) v[1] += (double)kl_term<float>(ref[u] - lp[u]);
            }
        });
        if (!(fabs(v[0]) < __builtin_inf() && v[1] < __builtin_inf())) far_sums<E, G>(p, k, g.at, of_tour, v[0], v[1]);
        if (p.mode == 0) {
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] += v[c];
            continue;
        }
        group_sum<G>(v);
        const double inv = v[3] > 0.0 ? 1.0 / v[3] : 0.0;
        double c = 0.0;
        if (p.mode & kRatioTour) {
            const float adv = p.adv[k];
            const bool cut = is_cut(p, adv, v[4]);
            c = cut ? 0.0 : ratio_term<double>(adv, v[4]);
            v[0] = cut ? (double)cut_term(p, adv) : c;
            v[2] = cut ? 1.0 : 0.0;
        } else {
            v[0] *= inv;
            v[2] *= inv;
        }
        if (g.at == 0) {
            if (v[3] > 0.0) { sum[0] += v[0]; sum[1] += v[1] * inv; sum[2] += v[2]; sum[3] += 1.0; }
            p.rows[k] = make_double2(v[3] > 0.0 ? c : 0.0, inv);
        }
    }
    group_sum<1024>(sum);
    if (threadIdx.x != 0) return;
    if (gridDim.x == 1) policy_end(p, sum);
    else
        for (int c = 0; c < 4; ++c) p.partial[blockIdx.x * 4 + c] = sum[c];
}

__global__ __launch_bounds__(1024) void k_policy_end(PolicyParams p, int blocks)
{
    double v[4] = {0.0, 0.0, 0.0, 0.0};
    for (int b = threadIdx.x; b < blocks; b += 1024)
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] += p.partial[b * 4 + c];
    group_sum<1024>(v);
    if (threadIdx.x == 0) policy_end(p, v);
}

template <typename F>
__device__ __forceinline__ F step_grad(const PolicyParams& p, const double2& row, double scale, float lp, float old,
                                       float ref, float adv)
{
    F d;
    if (p.mode & kRatioTour) {
        d = (F)row.x;
    } else {
        const double x = (double)lp - (double)old;
        d = is_cut(p, adv, x) ? (F)0 : ratio_term<F>(adv, x) * (F)row.y;
    }
    if (p.ref && p.kl_coef != 0.0) {
        const float e = ref - lp;
        d -= (F)p.kl_coef * (F)row.y * (fabsf(e) > 1.0f ? exp_as<F>((double)e) - (F)1 : kl_term<F>(e) + (F)e);
    }
    return d * (F)scale;
}

template <typename E, int G>
__global__ __launch_bounds__(1024) void k_policy_grad(PolicyParams p)
{
    const Groups<G> g;
    const double scale = p.norm[0] * (double)p.g[0];
    for (int64_t k = g.first; k < p.T; k += g.count) {
        const double2 row = p.mode ? p.rows[k] : make_double2(0.0, 1.0);
        const float of_tour = p.adv_per_step ? 0.0f : p.adv[k];
        for_steps<G>(g.at, p.S, [&](auto many, int64_t first) {
            constexpr int N = decltype(many)::value;
            float lp[N], old[N], ref[N], adv[N];
            uint8_t kept[N];
            const int64_t i = k * p.S + first;
            load_steps<E, N, G>(p.lp, i, true, 0.0f, lp);
            load_steps<E, N, G>(p.old, i, !(p.mode & kRatioTour), 0.0f, old);
            load_steps<E, N, G>(p.ref, i, p.ref && p.kl_coef != 0.0, 0.0f, ref);
            load_steps<float, N, G>(p.adv, i, p.adv_per_step, of_tour, adv);
            load_kept<N, G>(p.mask, i, kept);
            float d[N], all = 0.0f;
#pragma unroll
            for (int u = 0; u < N; ++u) {
                d[u] = kept[u] ? step_grad<float>(p, row, scale, lp[u], old[u], ref[u], adv[u]) : 0.0f;
                all += d[u];
            }
            if (!finite(all)) {
#pragma unroll
                for (int u = 0; u < N; ++u)
                    if (!finite(d[u])) d[u] = (float)step_grad<double>(p, row, scale, lp[u], old[u], ref[u], adv[u]);
            }
#pragma unroll
            for (int u = 0; u < N; ++u) static_cast<E*>(p.grad)[i + u * G] = narrow<E>(d[u]);
        });
    }
}

struct PrefParams {
    const void *lp, *ref;
    const double* len;
    const uint8_t* mask;
    int64_t T, S;
    int32_t per, best, per_step;
    double beta;
    float eps;
    double* score;          // (T)
    float* scale;           // (T): beta, or beta / kept steps
    float* coef;            // (T): sum over the tour's pairs of dl / ds
    double* partial;        // [blocks][2]: loss, pairs
    double* norm;
    float* loss;
    int64_t* pairs;
    const float* g;
    void* grad;
};

template <typename E, int G>
__device__ __forceinline__ void pref_rows(const PrefParams& p)
{
    const Groups<G> g;
    for (int64_t k = g.first; k < p.T; k += g.count) {
        double v[2] = {0.0, 0.0};                       // sum, steps
        for_steps<G>(g.at, p.S, [&](auto many, int64_t first) {
            constexpr int N = decltype(many)::value;
            float lp[N], ref[N];
            uint8_t kept[N];
            const int64_t i = k * p.S + first;
            load_steps<E, N, G>(p.lp, i, true, 0.0f, lp);
            load_steps<E, N, G>(p.ref, i, p.ref, 0.0f, ref);
            load_kept<N, G>(p.mask, i, kept);
#pragma unroll
            for (int u = 0; u < N; ++u) {
                v[0] += kept[u] ? (double)lp[u] - (double)ref[u] : 0.0;
                v[1] += kept[u] ? 1.0 : 0.0;
            }
        });
        group_sum<G>(v);
        if (g.at == 0) {
            const double scale = p.per_step ? p.beta / fmax(v[1], 1.0) : p.beta;
            p.score[k] = v[0] * scale;
            p.scale[k] = (float)scale;
        }
    }
}

// W threads a tour a walk the other tours b of its instance; loss and pairs are added up at the winner.
template <int W>
__device__ __forceinline__ void pref_pairs(const PrefParams& p, double (&sum)[2])
{
    const Groups<W> g;
    for (int64_t k = g.first; k < p.T; k += g.count) {
        const int64_t base = k / p.per * p.per;
        const int a = (int)(k - base);
        const double sa = p.score[k], la = p.len[k];
        int first = -1;
        if (p.best) {                                   // the first of the shortest; NaN is none
            double least = 0.0;
            for (int b = g.at; b < p.per; b += W) {
                const double l = p.len[base + b];
                if (l == l && (first < 0 || l < least)) { first = b; least = l; }
            }
            for (int o = W / 2; o >= 1; o >>= 1) {
                const int other = __shfl_xor(first, o);
                const double l = __shfl_xor(least, o);
                if (other >= 0 && (first < 0 || l < least || (l == least && other < first))) { first = other; least = l; }
            }
        }
        double c[1] = {0.0};
        for (int b = g.at; b < p.per; b += W) {
            const double sb = p.score[base + b], lb = p.len[base + b];
            const bool wins = la < lb && (!p.best || a == first);
            const bool loses = lb < la && (!p.best || b == first);
            if (!wins && !loses) continue;
            const float z = (float)(wins ? sa - sb : sb - sa);
            const float e = expf(-fabsf(z));
            const float against = z >= 0.0f ? e / (1.0f + e) : 1.0f / (1.0f + e);       // sigmoid(-z)
            c[0] += (double)(wins ? p.eps - against : against - p.eps);
            if (wins) {
                sum[0] += (double)((1.0f - p.eps) * fmaxf(-z, 0.0f) + (p.eps != 0.0f ? p.eps * fmaxf(z, 0.0f) : 0.0f) +
                                   log1pf(e));
                sum[1] += 1.0;
            }
        }
        group_sum<W>(c);
        if (g.at == 0) p.coef[k] = (float)c[0];
    }
    group_sum<1024>(sum);
}

__device__ __forceinline__ void pref_end(const PrefParams& p, const double (&v)[2])
{
    const double inv = v[1] > 0.0 ? 1.0 / v[1] : 0.0;
    p.norm[0] = inv;
    p.loss[0] = (float)(v[0] * inv);
    p.pairs[0] = (int64_t)v[1];
}

template <typename E, int G>
__global__ __launch_bounds__(1024) void k_pref_rows(PrefParams p)
{
    pref_rows<E, G>(p);
}

template <int W>
__global__ __launch_bounds__(1024) void k_pref_pairs(PrefParams p)
{
    double sum[2] = {0.0, 0.0};
    pref_pairs<W>(p, sum);
    if (threadIdx.x < 2) p.partial[blockIdx.x * 2 + threadIdx.x] = sum[threadIdx.x];
}

__global__ __launch_bounds__(1024) void k_pref_end(PrefParams p, int blocks)
{
    double v[2] = {0.0, 0.0};
    for (int b = threadIdx.x; b < blocks; b += 1024) { v[0] += p.partial[2 * b]; v[1] += p.partial[2 * b + 1]; }
    group_sum<1024>(v);
    if (threadIdx.x == 0) pref_end(p, v);
}

// Everything in one workgroup: what little there is would otherwise take three launches.
template <typename E, int G>
__global__ __launch_bounds__(1024) void k_pref_one(PrefParams p)
{
    pref_rows<E, G>(p);
    __syncthreads();                                    // the scores are read by other threads of this workgroup
    double sum[2] = {0.0, 0.0};
    pref_pairs<8>(p, sum);
    if (threadIdx.x == 0) pref_end(p, sum);
}

template <typename E, int G>
__global__ __launch_bounds__(1024) void k_pref_grad(PrefParams p)
{
    const Groups<G> g;
    const double scale = p.norm[0] * (double)p.g[0];
    for (int64_t k = g.first; k < p.T; k += g.count) {
        const E d = narrow<E>((float)(scale * (double)p.coef[k] * (double)p.scale[k]));
        for (int64_t s = g.at; s < p.S; s += G) {
            const int64_t i = k * p.S + s;
            static_cast<E*>(p.grad)[i] = !p.mask || p.mask[i] ? d : narrow<E>(0.0f);
        }
    }
}

inline int64_t round256(int64_t bytes) { return (bytes + 255) & ~(int64_t)255; }
constexpr int64_t kPartialBytes = kMaxBlocks * 4 * 8 + 256;

int loss_check(int64_t T, int64_t S, int32_t dtype)
{
    if (T < 0 || S < 0) return fail(TSP2OPT_E_ARG, "bad size");
    if (!element_size(dtype)) return fail(TSP2OPT_E_ARG, "dtype must be float32, bfloat16 or float16");
    if (T > 0x7fffffffll || S > 0x7fffffffll) return fail(TSP2OPT_E_UNSUPPORTED, "too many tours or steps");
    return 0;
}

bool off(const void* ptr, size_t size) { return reinterpret_cast<uintptr_t>(ptr) % size != 0; }

// How rows of S steps are shared out: threads a row, threads a workgroup, workgroups.  Values and gradient in us, float32
// with reference and mask:            8 threads     16            64            1024
//   100000 tours x 10 steps           17.5 +  9     22.5 +  9     76.5 +  31
//    50000 x 24                       14   + 7.5    18   +  9     45   +  17
//    20000 x 150                      18   + 14     17.5 + 12     28   + 15.5
//    10000 x 499                      35   + 31     25   + 21     27   + 19
//     1500 x 3000 (ratio of tours)   129   + 94     68   + 49     23   + 17     74   + 16
//       16 x 10000 (ratio of tours)  414   + 245   208   + 120    42   + 32     16.5 + 6.5
// One workgroup alone, 160 x 100: 15 us in one launch against 6.6 + 5.3 us in two and 3.5 us more on the host.
struct Shape {
    int group, threads;
    unsigned grid;
};

Shape shape_of(int64_t T, int64_t S, bool one_block)
{
    Shape s;
    s.group = S <= 24 ? 8 : S <= 160 ? 16 : S > 2048 && T <= 256 ? kBlockRow : 64;
    s.threads = s.group == kBlockRow || one_block ? 1024 : 256;
    const int64_t grid = (T * s.group + s.threads - 1) / s.threads;
    s.grid = one_block ? 1u : (unsigned)(grid < kMaxBlocks ? grid : kMaxBlocks);
    return s;
}

#define T2O_BY_GROUP(group, CALL)                                  \
    switch (group) {                                               \
        case 8: { constexpr int G = 8; CALL; break; }              \
        case 16: { constexpr int G = 16; CALL; break; }            \
        case 64: { constexpr int G = 64; CALL; break; }            \
        default: { constexpr int G = kBlockRow; CALL; break; }     \
    }

int64_t policy_state_bytes(int64_t T) { return kPartialBytes + round256(16 * T); }

int64_t pref_state_bytes(int64_t T) { return kPartialBytes + round256(8 * T) + 2 * round256(4 * T); }

void pref_state(PrefParams& p, void* state)
{
    char* at = static_cast<char*>(state);
    p.norm = reinterpret_cast<double*>(at);
    p.partial = reinterpret_cast<double*>(at + 256);
    at += kPartialBytes;
    p.score = reinterpret_cast<double*>(at);
    at += round256(8 * p.T);
    p.scale = reinterpret_cast<float*>(at);
    p.coef = reinterpret_cast<float*>(at + round256(4 * p.T));
}

void policy_state(PolicyParams& p, void* state)
{
    char* at = static_cast<char*>(state);
    p.norm = reinterpret_cast<double*>(at);
    p.partial = reinterpret_cast<double*>(at + 256);
    p.rows = reinterpret_cast<double2*>(at + kPartialBytes);
}

int policy_fill(PolicyParams& p, const void* lp, const void* old, const void* ref, const float* adv,
                const uint8_t* mask, int64_t T, int64_t S, int32_t adv_per_step, int32_t ratio_of_tour,
                int32_t average_of_tours, double clip_low, double clip_high, double kl_coef, int32_t dtype,
                void* state, int64_t state_bytes)
{
    const int rc = loss_check(T, S, dtype);
    if (rc) return rc;
    if (!(clip_low >= 0.0 && clip_low < 1.0) || !(clip_high >= 0.0))
        return fail(TSP2OPT_E_ARG, "clip_low must be in [0, 1) and clip_high >= 0");
    if (!(kl_coef >= 0.0 && kl_coef < __builtin_inf()) || (kl_coef != 0.0 && !ref))
        return fail(TSP2OPT_E_ARG, "kl_coef must be >= 0 and finite, and 0 without reference log-probabilities");
    if (ratio_of_tour && (!average_of_tours || adv_per_step))
        return fail(TSP2OPT_E_ARG, "ratios of tours are averaged over tours and take one advantage a tour");
    if (!state) return fail(TSP2OPT_E_ARG, "null pointer");
    if (off(state, 256)) return fail(TSP2OPT_E_ARG, "state must be 256-byte aligned");
    if (state_bytes < policy_state_bytes(T)) return fail(TSP2OPT_E_WORKSPACE, "state_bytes too small");
    if (T * S > 0 && (!lp || !old || !adv)) return fail(TSP2OPT_E_ARG, "null pointer");
    if (T > 0 && !adv_per_step && !adv) return fail(TSP2OPT_E_ARG, "null pointer");      // read without steps too
    const size_t size = element_size(dtype);
    if (off(lp, size) || off(old, size) || off(ref, size) || off(adv, 4))
        return fail(TSP2OPT_E_ARG, "misaligned pointer (arrays must be aligned to their element size)");
    p.lp = lp; p.old = old; p.ref = ref; p.adv = adv; p.mask = mask; p.T = T; p.S = S; p.adv_per_step = adv_per_step;
    p.mode = (ratio_of_tour ? kRatioTour : 0) | (average_of_tours ? kAverageTour : 0);
    p.lo = (float)(1.0 - clip_low); p.hi = (float)(1.0 + clip_high); p.kl_coef = kl_coef;
    p.log_lo = log1p(-clip_low); p.log_hi = log1p(clip_high);
    policy_state(p, state);
    return 0;
}

}  // namespace t2o

using namespace t2o;

extern "C" int64_t tsp2opt_policy_loss_state_bytes(int64_t num_tours)
{
    const int rc = loss_check(num_tours, 0, TSP2OPT_DTYPE_F32);
    return rc ? rc : policy_state_bytes(num_tours);
}

extern "C" int64_t tsp2opt_preference_loss_state_bytes(int64_t num_tours)
{
    const int rc = loss_check(num_tours, 0, TSP2OPT_DTYPE_F32);
    return rc ? rc : pref_state_bytes(num_tours);
}

extern "C" int tsp2opt_policy_loss(const void* logp, const void* old_logp, const void* ref_logp,
                                   const float* advantages, const uint8_t* mask, float* loss_out, float* stats_out,
                                   void* state, int64_t state_bytes, int64_t num_tours, int64_t steps,
                                   int32_t adv_per_step, int32_t ratio_of_tour, int32_t average_of_tours,
                                   double clip_low, double clip_high, double kl_coef, int32_t dtype, int32_t device,
                                   void* hip_stream)
{
    PolicyParams p{};
    const int rc = policy_fill(p, logp, old_logp, ref_logp, advantages, mask, num_tours, steps, adv_per_step,
                               ratio_of_tour, average_of_tours, clip_low, clip_high, kl_coef, dtype, state, state_bytes);
    if (rc) return rc;
    if (!loss_out || !stats_out || off(loss_out, 4) || off(stats_out, 4))
        return fail(TSP2OPT_E_ARG, "null or misaligned output");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(TSP2OPT_E_HIP, "hipSetDevice failed");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    p.loss = loss_out;
    p.stats = stats_out;
    const Shape s = shape_of(num_tours, steps, num_tours * steps <= kOneBlock && num_tours <= kOneBlock / 8);
    T2O_BY_DTYPE(dtype, T2O_BY_GROUP(s.group, hipLaunchKernelGGL((k_policy<E, G>), dim3(s.grid), dim3(s.threads), 0,
                                                                 stream, p)));
    if (s.grid > 1) hipLaunchKernelGGL(k_policy_end, dim3(1), dim3(1024), 0, stream, p, (int)s.grid);
    HIP_TRY(hipGetLastError());
    return 0;
}

extern "C" int tsp2opt_policy_loss_grad(const void* logp, const void* old_logp, const void* ref_logp,
                                        const float* advantages, const uint8_t* mask, const void* state,
                                        int64_t state_bytes, const float* grad_loss, void* grad_out,
                                        int64_t num_tours, int64_t steps, int32_t adv_per_step, int32_t ratio_of_tour,
                                        int32_t average_of_tours, double clip_low, double clip_high, double kl_coef,
                                        int32_t dtype, int32_t device, void* hip_stream)
{
    PolicyParams p{};
    const int rc = policy_fill(p, logp, old_logp, ref_logp, advantages, mask, num_tours, steps, adv_per_step,
                               ratio_of_tour, average_of_tours, clip_low, clip_high, kl_coef, dtype,
                               const_cast<void*>(state), state_bytes);
    if (rc) return rc;
    if (num_tours == 0 || steps == 0) return 0;
    if (!grad_loss || !grad_out || off(grad_loss, 4) || off(grad_out, element_size(dtype)))
        return fail(TSP2OPT_E_ARG, "null or misaligned gradient");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(TSP2OPT_E_HIP, "hipSetDevice failed");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    p.g = grad_loss;
    p.grad = grad_out;
    const Shape s = shape_of(num_tours, steps, false);
    T2O_BY_DTYPE(dtype, T2O_BY_GROUP(s.group, hipLaunchKernelGGL((k_policy_grad<E, G>), dim3(s.grid), dim3(s.threads), 0,
                                                                 stream, p)));
    HIP_TRY(hipGetLastError());
    return 0;
}

extern "C" int tsp2opt_preference_loss(const void* logp, const void* ref_logp, const double* lengths,
                                       const uint8_t* mask, float* loss_out, int64_t* pairs_out, void* state,
                                       int64_t state_bytes, int64_t num_tours, int64_t steps,
                                       int32_t tours_per_instance, int32_t best_only, int32_t per_step, double beta,
                                       double label_smoothing, int32_t dtype, int32_t device, void* hip_stream)
{
    const int rc = loss_check(num_tours, steps, dtype);
    if (rc) return rc;
    if (tours_per_instance < 1 || num_tours % tours_per_instance)
        return fail(TSP2OPT_E_ARG, "num_tours % tours_per_instance != 0");
    if (!(label_smoothing >= 0.0 && label_smoothing < 0.5) || !(beta > 0.0 && beta < __builtin_inf()))
        return fail(TSP2OPT_E_ARG, "beta must be > 0 and finite and label_smoothing in [0, 0.5)");
    if (!loss_out || !pairs_out || !state) return fail(TSP2OPT_E_ARG, "null pointer");
    if (num_tours > 0 && (!lengths || (steps > 0 && !logp))) return fail(TSP2OPT_E_ARG, "null pointer");
    const size_t size = element_size(dtype);
    if (off(logp, size) || off(ref_logp, size) || off(lengths, 8) || off(loss_out, 4) || off(pairs_out, 8) ||
        off(state, 256))
        return fail(TSP2OPT_E_ARG, "misaligned pointer (arrays must be aligned to their element size, state to 256)");
    if (state_bytes < pref_state_bytes(num_tours)) return fail(TSP2OPT_E_WORKSPACE, "state_bytes too small");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(TSP2OPT_E_HIP, "hipSetDevice failed");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    PrefParams p{};
    p.lp = logp; p.ref = ref_logp; p.len = lengths; p.mask = mask; p.T = num_tours; p.S = steps;
    p.per = tours_per_instance; p.best = best_only; p.per_step = per_step; p.beta = beta; p.eps = (float)label_smoothing;
    p.loss = loss_out; p.pairs = pairs_out;
    pref_state(p, state);
    // one workgroup does all: it has 8 threads a tour, so the pairs of 512 tours take four turns of it.  No tours at all
    // are its too, whatever an instance would have of them: the other launches would have no workgroup
    if (num_tours == 0 || (num_tours * steps <= kOneBlock && num_tours <= 512 && tours_per_instance <= 64)) {
        const Shape s = shape_of(num_tours, steps, true);
        T2O_BY_DTYPE(dtype, T2O_BY_GROUP(s.group, hipLaunchKernelGGL((k_pref_one<E, G>), dim3(1), dim3(kOneThreads), 0,
                                                                     stream, p)));
    } else {
        const Shape s = shape_of(num_tours, steps, false);
        T2O_BY_DTYPE(dtype, T2O_BY_GROUP(s.group, hipLaunchKernelGGL((k_pref_rows<E, G>), dim3(s.grid), dim3(s.threads), 0,
                                                                     stream, p)));
        // us with 8 and with 64 threads a tour, instances x tours: 2000 x 16 6.5, 15.5; 500 x 64 13.5, 16.3; 250 x 128 21.7,
        // 23.8; 10 x 1000 78, 42.5
        const int w = tours_per_instance <= 64 ? 8 : 64;
        const int64_t need = (num_tours * w + 255) / 256;
        const unsigned blocks = (unsigned)(need < kMaxBlocks ? need : kMaxBlocks);
        if (w == 8) hipLaunchKernelGGL(k_pref_pairs<8>, dim3(blocks), dim3(256), 0, stream, p);
        else hipLaunchKernelGGL(k_pref_pairs<64>, dim3(blocks), dim3(256), 0, stream, p);
        hipLaunchKernelGGL(k_pref_end, dim3(1), dim3(1024), 0, stream, p, (int)blocks);
    }
    HIP_TRY(hipGetLastError());
    return 0;
}

extern "C" int tsp2opt_preference_loss_grad(const uint8_t* mask, const void* state, int64_t state_bytes,
                                            const float* grad_loss, void* grad_out, int64_t num_tours, int64_t steps,
                                            int32_t dtype, int32_t device, void* hip_stream)
{
    const int rc = loss_check(num_tours, steps, dtype);
    if (rc) return rc;
    if (num_tours == 0 || steps == 0) return 0;
    if (!state || !grad_loss || !grad_out) return fail(TSP2OPT_E_ARG, "null pointer");
    if (off(state, 256) || off(grad_loss, 4) || off(grad_out, element_size(dtype)))
        return fail(TSP2OPT_E_ARG, "misaligned pointer (arrays must be aligned to their element size, state to 256)");
    if (state_bytes < pref_state_bytes(num_tours)) return fail(TSP2OPT_E_WORKSPACE, "state_bytes too small");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(TSP2OPT_E_HIP, "hipSetDevice failed");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    PrefParams p{};
    p.mask = mask; p.T = num_tours; p.S = steps; p.g = grad_loss; p.grad = grad_out;
    pref_state(p, const_cast<void*>(state));
    const Shape s = shape_of(num_tours, steps, false);
    T2O_BY_DTYPE(dtype, T2O_BY_GROUP(s.group, hipLaunchKernelGGL((k_pref_grad<E, G>), dim3(s.grid), dim3(s.threads), 0,
                                                                 stream, p)));
    HIP_TRY(hipGetLastError());
    return 0;
}
