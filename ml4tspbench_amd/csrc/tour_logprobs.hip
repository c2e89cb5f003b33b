// ml4tspbench_amd/csrc/tour_logprobs.hip -- step log-probabilities of tours under heat maps / decoder logits
//
// A tour starts at tour[0] and step t = 0 .. n-2 chooses tour[t+1] among the nodes not visited yet, with the softmax
// of one row of logits over those nodes:
//     lp(t) = h[r, tour[t+1]] - log sum_{j : pos(j) > t} exp h[r, j],
// pos(j) = the step that visits j (the inverse permutation), r = tour[t] for heat maps, r = t for the rows that an
// autoregressive decoder wrote.  Gradient, with g(t) the gradient of lp(t):
//     dh[r, j] = sum over the tours that share the row of  g(t) ([j = tour[t+1]] - [pos(j) > t] softmax_j).
#include "learn_common.hpp"

namespace t2o {

constexpr float kInf = __builtin_inff();

struct LogpParams {
    const void* logits;
    const int64_t* tours;
    float* logp;            // (T, n - 1)
    float* pos;             // (T, n); -1 everywhere: the tour is no permutation
    float* top;             // (T, rows): largest open logit of the row
    float* total;           // (T, rows): sum of exp(h - top) over the open nodes
    const float* g;         // (T, n - 1)
    void* grad;             // (M, rows, n)
    int64_t maps, map_stride, row_stride;
    int32_t n, rows, per, by_step;
};

// Inverse permutation of every tour, one workgroup a tour; scattered in LDS so that the write is contiguous.
__global__ __launch_bounds__(256) void k_positions(const int64_t* tours, float* pos, float* logp, int n)
{
    extern __shared__ uint16_t at[];
    const int64_t k = blockIdx.x;
    const int64_t* t = tours + k * (int64_t)(n + 1);
    int bad = 0;
    for (int s = threadIdx.x; s < n; s += blockDim.x) {
        const int64_t j = t[s];
        if (j < 0 || j >= n) bad = 1;
        else at[j] = (uint16_t)s;
    }
    __syncthreads();
    for (int s = threadIdx.x; s < n; s += blockDim.x) {
        const int64_t j = t[s];
        if (j >= 0 && j < n && at[j] != (uint16_t)s) bad = 1;
    }
    bad = __syncthreads_or(bad);
    for (int j = threadIdx.x; j < n; j += blockDim.x) pos[k * n + j] = bad ? -1.0f : (float)at[j];
    if (bad)
        for (int s = threadIdx.x; s < n - 1; s += blockDim.x) logp[k * (n - 1) + s] = __builtin_nanf("");
}

// One wave a (tour, row): running maximum and sum over the open nodes.
template <typename E>
__global__ __launch_bounds__(256) void k_logp(LogpParams p)
{
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t k = w / p.rows;
    if (k >= p.maps * p.per) return;
    const int r = (int)(w - k * p.rows);
    const float* pos = p.pos + k * p.n;
    const float when = p.by_step ? (float)r : pos[r];
    const E* h = static_cast<const E*>(p.logits) + (k / p.per) * p.map_stride + (int64_t)r * p.row_stride;
    float top = -kInf, total = 0.0f;
    bool nan = false;
    for (int j = lane; j < p.n; j += 64) {
        if (!(pos[j] > when)) continue;
        const float x = widen(h[j]);
        nan |= x != x;
        const float m = fmaxf(top, x);
        if (m > -kInf) {
            total = total * expf(top - m) + expf(x - m);
            top = m;
        }
    }
    const float m = wave_max(top);
    total = wave_sum(top > -kInf ? total * expf(top - m) : 0.0f);
    if (__any(nan)) total = __builtin_nanf("");
    if (lane == 0) {
        p.top[w] = m;
        p.total[w] = total;
        const int t = (int)when;
        if (pos[0] >= 0.0f && t < p.n - 1) {
            const float x = widen(h[p.tours[k * (p.n + 1) + t + 1]]);
            p.logp[k * (p.n - 1) + t] = total == 0.0f ? -kInf : (x - m) - logf(total);
        }
    }
}

// One wave a row: the tours that share it are added up in their order.
template <typename E>
__global__ __launch_bounds__(256) void k_logp_grad(LogpParams p)
{
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t map = w / p.rows;
    if (map >= p.maps) return;
    const int r = (int)(w - map * p.rows);
    const E* h = static_cast<const E*>(p.logits) + map * p.map_stride + (int64_t)r * p.row_stride;
    E* out = static_cast<E*>(p.grad) + w * p.n;
    for (int j = lane; j < p.n; j += 64) {
        const float x = widen(h[j]);
        float d = 0.0f;
        for (int q = 0; q < p.per; ++q) {
            const int64_t k = map * p.per + q;
            const float* pos = p.pos + k * p.n;
            const float when = p.by_step ? (float)r : pos[r];
            const int t = (int)when;
            if (!(pos[j] > when) || t >= p.n - 1) continue;
            const float g = p.g[k * (p.n - 1) + t], total = p.total[k * p.rows + r];
            if (total == 0.0f || g == 0.0f) continue;
            d -= g * (expf(x - p.top[k * p.rows + r]) / total);
            if (pos[j] == when + 1.0f) d += g;
        }
        out[j] = narrow<E>(d);
    }
}

int logp_check(const void* logits, const int64_t* tours, const void* out, const void* state, int64_t num_tours, int32_t n,
               int32_t per, int32_t by_step, int64_t map_stride, int64_t row_stride, int32_t dtype,
               int out_size)
{
    if (num_tours < 0 || n < 1 || per < 1 || num_tours % per != 0) return fail(TSP2OPT_E_ARG, "bad size");
    if (n > TSP2OPT_MAX_N) return fail(TSP2OPT_E_UNSUPPORTED, "n > 65535 is not supported");
    if (by_step != 0 && by_step != 1) return fail(TSP2OPT_E_ARG, "rows must be 0 (one per node) or 1 (one per step)");
    if (by_step && per != 1) return fail(TSP2OPT_E_ARG, "rows of steps belong to one tour: tours_per_map must be 1");
    const int size = element_size(dtype);
    if (!size) return fail(TSP2OPT_E_ARG, "dtype must be float32, bfloat16 or float16");
    if (map_stride < 0 || row_stride < 0) return fail(TSP2OPT_E_ARG, "negative stride");
    if (num_tours > 0x7fffffffll || num_tours * (int64_t)n > (int64_t)1 << 32)
        return fail(TSP2OPT_E_UNSUPPORTED, "too many tours");
    if (num_tours == 0 || n == 1) return 0;
    if (!logits || !tours || !out || !state) return fail(TSP2OPT_E_ARG, "null pointer");
    if (reinterpret_cast<uintptr_t>(logits) % size || reinterpret_cast<uintptr_t>(tours) % 8 ||
        reinterpret_cast<uintptr_t>(out) % out_size || reinterpret_cast<uintptr_t>(state) % 256)
        return fail(TSP2OPT_E_ARG, "misaligned pointer (arrays must be aligned to their element size, state to 256)");
    return 0;
}

inline int64_t round256(int64_t bytes) { return (bytes + 255) & ~(int64_t)255; }

int64_t logp_state_bytes(int64_t num_tours, int32_t n) { return 3 * round256(4 * num_tours * n) + 256; }

LogpParams logp_params(const void* logits, const int64_t* tours, float* state, int64_t num_tours, int32_t n, int32_t per,
                       int32_t by_step, int64_t map_stride, int64_t row_stride)
{
    LogpParams p{};
    const int64_t one = round256(4 * num_tours * n) / 4;
    p.logits = logits; p.tours = tours; p.pos = state; p.top = state + one; p.total = state + 2 * one;
    p.maps = num_tours / per; p.map_stride = map_stride; p.row_stride = row_stride;
    p.n = n; p.rows = by_step ? n - 1 : n; p.per = per; p.by_step = by_step;
    return p;
}

}  // namespace t2o

using namespace t2o;

extern "C" int64_t tsp2opt_tour_logprobs_state_bytes(int64_t num_tours, int32_t n, int32_t tours_per_map, int32_t rows)
{
    const int rc = logp_check(nullptr, nullptr, nullptr, nullptr, 0, n, tours_per_map, rows, 0, 0, TSP2OPT_DTYPE_F32,
                              4);
    if (rc) return rc;
    if (num_tours < 0 || num_tours % tours_per_map) return fail(TSP2OPT_E_ARG, "bad size");
    return logp_state_bytes(num_tours, n);
}

extern "C" int tsp2opt_tour_logprobs(const void* logits, const int64_t* tours, float* logp_out, void* state,
                                     int64_t state_bytes, int64_t num_tours, int32_t n, int32_t tours_per_map,
                                     int32_t rows, int64_t map_stride, int64_t row_stride, int32_t dtype,
                                     int32_t device, void* hip_stream)
{
    const int rc = logp_check(logits, tours, logp_out, state, num_tours, n, tours_per_map, rows, map_stride, row_stride,
                              dtype, 4);
    if (rc) return rc;
    if (num_tours == 0 || n == 1) return 0;
    if (state_bytes < logp_state_bytes(num_tours, n)) return fail(TSP2OPT_E_WORKSPACE, "state_bytes too small");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(TSP2OPT_E_HIP, "hipSetDevice failed");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    LogpParams p = logp_params(logits, tours, static_cast<float*>(state), num_tours, n, tours_per_map, rows, map_stride,
                               row_stride);
    p.logp = logp_out;
    const size_t lds = 2 * (size_t)n;
    HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(k_positions), hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)lds));
    hipLaunchKernelGGL(k_positions, dim3((unsigned)num_tours), dim3(256), lds, stream, tours, p.pos, logp_out, n);
    const unsigned grid = (unsigned)((num_tours * p.rows + 3) / 4);
    T2O_BY_DTYPE(dtype, hipLaunchKernelGGL(k_logp<E>, dim3(grid), dim3(256), 0, stream, p));
    HIP_TRY(hipGetLastError());
    return 0;
}

extern "C" int tsp2opt_tour_logprobs_grad(const void* logits, const int64_t* tours, const void* state,
                                          int64_t state_bytes, const float* grad_logp, void* grad_out,
                                          int64_t num_tours, int32_t n, int32_t tours_per_map, int32_t rows,
                                          int64_t map_stride, int64_t row_stride, int32_t dtype, int32_t device,
                                          void* hip_stream)
{
    const int rc = logp_check(logits, tours, grad_out, state, num_tours, n, tours_per_map, rows, map_stride, row_stride,
                              dtype, dtype == TSP2OPT_DTYPE_F32 ? 4 : 2);
    if (rc) return rc;
    if (num_tours == 0 || n == 1) return 0;
    if (!grad_logp) return fail(TSP2OPT_E_ARG, "null pointer");
    if (reinterpret_cast<uintptr_t>(grad_logp) % 4)
        return fail(TSP2OPT_E_ARG, "misaligned pointer (arrays must be aligned to their element size)");
    if (state_bytes < logp_state_bytes(num_tours, n)) return fail(TSP2OPT_E_WORKSPACE, "state_bytes too small");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(TSP2OPT_E_HIP, "hipSetDevice failed");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    LogpParams p = logp_params(logits, tours, static_cast<float*>(const_cast<void*>(state)), num_tours, n,
                               tours_per_map, rows, map_stride, row_stride);
    p.g = grad_logp;
    p.grad = grad_out;
    const unsigned grid = (unsigned)((p.maps * p.rows + 3) / 4);
    T2O_BY_DTYPE(dtype, hipLaunchKernelGGL(k_logp_grad<E>, dim3(grid), dim3(256), 0, stream, p));
    HIP_TRY(hipGetLastError());
    return 0;
}
