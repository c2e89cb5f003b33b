// ml4tspbench_amd/csrc/tour_logprobs.hip -- step log-probabilities of tours under heat maps / decoder logits
//
// A tour starts at tour[0] and step t = 0 .. n-2 chooses tour[t+1] among the nodes not visited yet, with the softmax
// of one row of logits over those nodes:
//     lp(t) = h[r, tour[t+1]] - log sum_{j : pos(j) > t} exp h[r, j],
// pos(j) = the step that visits j (the inverse permutation), r = tour[t] for heat maps, r = t for the rows that an
// autoregressive decoder wrote.  Gradient, with g(t) the gradient of lp(t):
//     dh[r, j] = sum over the tours that share the row of  g(t) ([j = tour[t+1]] - [pos(j) > t] softmax_j).
//
// Every wave keeps (part of) its rows in registers: K entries of a row a lane, 64 K columns, loaded once.  Rows longer
// than 1024 entries are split into parts whose maxima and sums k_join puts together.
//
// Several tours a map (k_shared): e_j = exp(h_j - row maximum) does not depend on the tour, only which e_j are added
// does, and positions are whole numbers, so a masked addition is
//     S += min(max(pos_j - t, 0), 1) * e_j          (one v_sub with clamp, one v_fmac)
// instead of an exponential a tour.  That sum loses steps whose open entries all lie far below the row's maximum, so
// the exponentials are kept times 2^60, which spends the range of float above 1 too: what it flushes (below 2^-126,
// 65535 entries at most) is under 2^-30 of a sum above 2^-80, which is 2^-140 = e^-97 relative to the row's maximum.
// Steps below that (and those that are NaN) are redone alone, relative to their own maximum.
// One tour a row (k_single): the maximum is the open entries' own, nothing is ever lost.
#include "learn_common.hpp"

namespace t2o {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kSmall = 0x1p-80f, kScale = 0x1p60f;
constexpr int kWaves = 8, kRows = 4, kTile = 16;    // k_shared: waves a workgroup, rows a wave, tours a pass
constexpr int kSingleRows = 16;                     // k_single: rows a wave
constexpr int kMaxPer = 16;                         // entries of a row a lane holds at most

struct LogpParams {
    const void* logits;
    const int64_t* tours;
    float* logp;            // (T, n - 1)
    float* pos;             // (T, n); -1 everywhere: the tour is no permutation
    uint16_t* next;         // (T, n): the node after a node
    float* top;             // (M, rows) shared, (T, rows) single: what the exponentials are relative to
    float* total;           // (T, rows): sum of exp(h - top) over the open entries
    float* part_top;        // [parts](M or T, rows)
    float* part_total;      // [parts](T, rows)
    const float* g;         // (T, n - 1)
    void* grad;             // (M, rows, n)
    int64_t maps, map_stride, row_stride, groups;
    int32_t n, rows, per, by_step, parts, tile;
};

// Consecutive workgroups go to the eight dies in turn; this gives each die a contiguous range of the work instead, so
// that a map's tours, and the lines of logp that its rows write between them, stay in one L2.
__device__ __forceinline__ int64_t work_block()
{
    const int64_t n = gridDim.x, b = blockIdx.x, q = n / 8, rest = n % 8, die = b % 8;
    return die * q + (die < rest ? die : rest) + b / 8;
}

// Inverse permutation and successors of every tour, one workgroup a tour; scattered in LDS so that the writes are
// contiguous.
__global__ __launch_bounds__(1024) void k_positions(const int64_t* tours, float* pos, uint16_t* next, float* logp, int n)
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
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
        pos[k * n + j] = bad ? -1.0f : (float)at[j];
        next[k * n + j] = bad || at[j] + 1 >= n ? (uint16_t)0 : (uint16_t)t[at[j] + 1];
    }
    if (bad)
        for (int s = threadIdx.x; s < n - 1; s += blockDim.x) logp[k * (n - 1) + s] = __builtin_nanf("");
}

// ---- rows in registers: lane l holds entries c * 64 V + l V + v, V adjacent ones a load.  Rows of odd length start
// anywhere, so the loads are aligned to the element only, which the memory pipe takes at full width.
template <int K>
constexpr int kVec = K % 4 == 0 ? 4 : K % 2 == 0 ? 2 : 1;

template <typename E, int V>
struct Pack {
    typedef E type __attribute__((ext_vector_type(V), aligned(sizeof(E))));
};
template <typename E>
struct Pack<E, 1> {
    typedef E type;
};

// Loads are issued without a branch: a lane at or behind the end reads the row's last V entries instead (in front of a
// short last part there is the previous one) and end_row puts its entries in place.
template <typename E, int K>
struct Row {
    static constexpr int V = kVec<K>;
    typename Pack<E, V>::type x[K / V];
};

template <typename E, int K, int G = 64>
__device__ __forceinline__ void load_row(const E* row, int lane, int cols, Row<E, K>& raw)
{
    constexpr int V = kVec<K>;
    using P = typename Pack<E, V>::type;
#pragma unroll
    for (int c = 0; c < K / V; ++c) {
        const int j = c * G * V + lane * V;
        raw.x[c] = *reinterpret_cast<const P*>(row + min(j, cols - V));
    }
}

template <typename E, int K, int G = 64>
__device__ __forceinline__ void end_row(const Row<E, K>& raw, int lane, int cols, float (&h)[K])
{
    constexpr int V = kVec<K>;
#pragma unroll
    for (int c = 0; c < K / V; ++c) {
        const int j = c * G * V + lane * V;
        float x[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (V == 1) x[v] = widen(raw.x[c]);
            else x[v] = widen(raw.x[c][v]);
        }
        if ((c + 1) * G * V > cols) {
            const int shift = j - (cols - V);           // <= 0: the lane's own entries were read
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float y = -kInf;
#pragma unroll
                for (int w = V - 1; w > v; --w) y = shift == w - v ? x[w] : y;
                h[c * V + v] = shift <= 0 ? x[v] : y;
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) h[c * V + v] = x[v];
        }
    }
}

template <typename E, int K, int G = 64>
__device__ __forceinline__ void store_row(E* row, int lane, int cols, const float (&d)[K])
{
    constexpr int V = kVec<K>;
    using P = typename Pack<E, V>::type;
#pragma unroll
    for (int c = 0; c < K / V; ++c) {
        const int j = c * G * V + lane * V;
        P x;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (V == 1) x = narrow<E>(d[c]);
            else x[v] = narrow<E>(d[c * V + v]);
        }
        if (j + V <= cols) *reinterpret_cast<P*>(row + j) = x;
        if constexpr (V > 1) {
            if ((c + 1) * G * V > cols && cols % V) {
#pragma unroll
                for (int v = 0; v < V - 1; ++v)
                    if (j + V > cols && j + v < cols) row[j + v] = x[v];
            }
        }
    }
}

// The column of register i of this lane.
template <int K, int G = 64>
__device__ __forceinline__ int column(int i, int lane)
{
    constexpr int V = kVec<K>;
    return (i / V) * G * V + lane * V + i % V;
}

// ---- sums over the 64 lanes, four values at a time
template <int CTRL>
__device__ __forceinline__ float dpp(float x)
{
    const int i = __float_as_int(x);
    return __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false));
}

// a[0..3] -> value (lane & 3) summed over the 16 lanes of this lane's row, in every lane of that row
__device__ __forceinline__ float quad_sum(const float (&a)[4], bool odd, bool high)
{
    const float u = (odd ? a[1] : a[0]) + dpp<0xB1>(odd ? a[0] : a[1]);         // quad_perm [1,0,3,2]
    const float v = (odd ? a[3] : a[2]) + dpp<0xB1>(odd ? a[2] : a[3]);
    float w = (high ? v : u) + dpp<0x4E>(high ? u : v);                         // quad_perm [2,3,0,1]
    w += dpp<0x124>(w);                                                         // row_ror:4
    return w + dpp<0x128>(w);                                                   // row_ror:8
}

// z0..z3 -> z(lane >> 4) summed over the four rows of 16 lanes
__device__ __forceinline__ float rows_sum(float z0, float z1, float z2, float z3)
{
    auto swap16 = [](float a, float b) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
        return __uint_as_float(r[0]) + __uint_as_float(r[1]);
    };
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(swap16(z0, z1)), __float_as_uint(swap16(z2, z3)),
                                                    false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ float row_max(float m)
{
    m = fmaxf(m, dpp<0xB1>(m));
    m = fmaxf(m, dpp<0x4E>(m));
    m = fmaxf(m, dpp<0x141>(m));                                                // row_half_mirror
    m = fmaxf(m, dpp<0x140>(m));                                                // row_mirror
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
    m = fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(m)));
}

__device__ __forceinline__ float lane_value(float x, int lane)
{
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// What the exponentials are relative to: an empty row's maximum is -inf, which no entry may be subtracted from.
__device__ __forceinline__ float base_of(float top) { return top == -kInf ? 0.0f : top; }

__device__ __forceinline__ float sum64(float v)
{
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    v += dpp<0x140>(v);
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// exp(x) 2^60 of a difference x <= 0.  Far below 0 the scale goes into the argument, where float does not flush yet.
__device__ __forceinline__ float scaled_exp(float x)
{
    x *= kLog2e;
    const bool far = x < -40.0f;
    return __builtin_amdgcn_exp2f(far ? x + 60.0f : x) * (far ? 1.0f : kScale);
}

// Maximum and sum over a row's open entries by the whole wave: the steps that k_shared cannot see.
template <typename E, int K>
__device__ void open_sum(const E* row, const float* pos, float when, int n, int lane, float& top, float& total)
{
    top = -kInf;
    total = 0.0f;
    for (int c = 0; c < n; c += 64 * K) {
        const int cols = min(64 * K, n - c);
        Row<E, K> raw;
        Row<float, K> raw_pos;
        load_row<E, K>(row + c, lane, cols, raw);
        load_row<float, K>(pos + c, lane, cols, raw_pos);
        float h[K], at[K], m = -kInf, s = 0.0f;
        end_row<E, K>(raw, lane, cols, h);
        end_row<float, K>(raw_pos, lane, cols, at);
#pragma unroll
        for (int x = 0; x < K; ++x) {
            h[x] = at[x] > when ? h[x] : -kInf;
            m = fmaxf(m, h[x]);
        }
        const float now = fmaxf(top, row_max(m)), from = base_of(now);
#pragma unroll
        for (int x = 0; x < K; ++x) s += __builtin_amdgcn_exp2f((h[x] - from) * kLog2e);
        if (total != 0.0f) total *= __builtin_amdgcn_exp2f((top - from) * kLog2e);
        total += sum64(s);
        top = now;
    }
}

// Ends the steps of the lanes with `valid`: (tour k, row r, step `when`).  `total` is 2^60 times the sum where it is
// shared.  Steps of which a shared sum says nothing are redone one after the other by the whole wave: all lanes have to
// be here.
template <typename E, int K, bool SHARED>
__device__ void end_steps(const LogpParams& p, bool valid, int64_t map, int64_t k, int r, float when, float top,
                          float total, int lane)
{
    const E* base = static_cast<const E*>(p.logits);
    const E* row = base + map * p.map_stride + (int64_t)r * p.row_stride;
    const int t = (int)when;
    float chosen = 0.0f;
    if (valid) chosen = widen(row[p.by_step ? (int)p.tours[k * (p.n + 1) + t + 1] : (int)p.next[k * p.n + r]]);
    // log(total) and not of total 2^-60 where that would leave the range of float
    float log_total = logf(!SHARED ? total : total >= 0x1p-60f ? total * (1.0f / kScale) : total);
    if (SHARED && total < 0x1p-60f) log_total -= 60.0f / kLog2e;
    if constexpr (SHARED) {
        uint64_t redo = __ballot(valid && !(total >= kSmall));
        while (redo) {
            const int l = __ffsll((unsigned long long)redo) - 1;
            redo &= redo - 1;
            const int64_t kk = ((int64_t)__builtin_amdgcn_readlane((int)(k >> 32), l) << 32) |
                               (unsigned)__builtin_amdgcn_readlane((int)k, l);
            const int64_t mm = ((int64_t)__builtin_amdgcn_readlane((int)(map >> 32), l) << 32) |
                               (unsigned)__builtin_amdgcn_readlane((int)map, l);
            const int rr = __builtin_amdgcn_readlane(r, l);
            float m, s;
            open_sum<E, K>(base + mm * p.map_stride + (int64_t)rr * p.row_stride, p.pos + kk * p.n, lane_value(when, l),
                           p.n, lane, m, s);
            if (lane == l) { top = m; total = s; log_total = logf(s); }
        }
    }
    if (valid) p.logp[k * (p.n - 1) + t] = total == 0.0f ? -kInf : (chosen - base_of(top)) - log_total;
}

// The positions of a pass's tours in LDS, a wave a tour.
template <int K>
__device__ __forceinline__ void stage(float* tile, const float* pos, int count, int n, int col0, int cols, int wave, int lane)
{
    constexpr int V = kVec<K>, per_wave = kTile / kWaves;
    Row<float, K> raw[per_wave];
#pragma unroll
    for (int a = 0; a < per_wave; ++a) {
        const int q = min(a * kWaves + wave, count - 1);
        load_row<float, K>(pos + (int64_t)q * n + col0, lane, cols, raw[a]);
    }
#pragma unroll
    for (int a = 0; a < per_wave; ++a) {
        const int q = a * kWaves + wave;
        if (q >= count) break;
        float at[K];
        end_row<float, K>(raw[a], lane, cols, at);      // behind the end: -inf, which no step comes before
#pragma unroll
        for (int c = 0; c < K / V; ++c)
#pragma unroll
            for (int v = 0; v < V; ++v) tile[q * 64 * K + c * 64 * V + lane * V + v] = fmaxf(at[c * V + v], -1.0f);
    }
}

template <typename E, int K>
__global__ __launch_bounds__(64 * kWaves) void k_shared(LogpParams p)
{
    extern __shared__ float tile[];                     // [tours of a pass][64 K] positions
    __shared__ float4 when[kWaves][kTile];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t b = work_block();
    const int part = (int)(b % p.parts);
    const int64_t group = b / p.parts, map = group / p.groups;
    const int r0 = (int)(group % p.groups) * (kWaves * kRows) + wave * kRows;
    const int col0 = part * 64 * K, cols = min(64 * K, p.n - col0);
    const bool odd = lane & 1, high = lane & 2;
    const E* row0 = static_cast<const E*>(p.logits) + map * p.map_stride + col0;

    float e[kRows][K], top[kRows];
    Row<E, K> raw[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) load_row<E, K>(row0 + (int64_t)min(r0 + r, p.n - 1) * p.row_stride, lane, cols, raw[r]);
    stage<K>(tile, p.pos + map * p.per * (int64_t)p.n, min(kTile, p.per), p.n, col0, cols, wave, lane);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        end_row<E, K>(raw[r], lane, cols, e[r]);
        const int self = r0 + r - col0;                 // the diagonal is never open: it must not set the maximum
        if (self >= 0 && self < cols) {
#pragma unroll
            for (int x = 0; x < K; ++x)
                if (column<K>(x, lane) == self) e[r][x] = -kInf;
        }
        float m = e[r][0];
#pragma unroll
        for (int x = 1; x < K; ++x) m = fmaxf(m, e[r][x]);
        top[r] = row_max(m);
        const float from = base_of(top[r]);
#pragma unroll
        for (int x = 0; x < K; ++x) e[r][x] = scaled_exp(e[r][x] - from);
    }
    const float mine = (lane & 2) ? ((lane & 1) ? top[3] : top[2]) : ((lane & 1) ? top[1] : top[0]);
    const int i = r0 + (lane & 3);
    if (lane < kRows && i < p.n) (p.parts == 1 ? p.top : p.part_top + (int64_t)part * p.maps * p.n)[map * p.n + i] = mine;

    for (int q0 = 0; q0 < p.per; q0 += kTile) {
        const int count = min(kTile, p.per - q0);
        const float* pos = p.pos + (map * p.per + q0) * (int64_t)p.n;
        if (q0) {
            __syncthreads();
            stage<K>(tile, pos, count, p.n, col0, cols, wave, lane);
        }
        // lane = (tour q0 + lane / 4, row lane % 4): the step at which the tour leaves the row's node
        const int q = lane >> 2;
        const bool in = q < count && i < p.n;
        const float t = in ? pos[(int64_t)q * p.n + i] : 65536.0f;
        reinterpret_cast<float*>(when[wave])[lane] = t;
        __syncthreads();
        float z0 = 0.0f, z1 = 0.0f, z2 = 0.0f, z3 = 0.0f;
        for (int a = 0; a < kTile / 4; ++a) {
            z0 = z1; z1 = z2; z2 = z3; z3 = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int qq = 4 * a + c;
                if (qq >= count) continue;
                const float4 tt = when[wave][qq];
                const float* at = tile + qq * 64 * K;
                float s[kRows] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < K; ++x) {
                    const float y = at[column<K>(x, lane)];
                    s[0] = fmaf(__builtin_amdgcn_fmed3f(y - tt.x, 0.0f, 1.0f), e[0][x], s[0]);
                    s[1] = fmaf(__builtin_amdgcn_fmed3f(y - tt.y, 0.0f, 1.0f), e[1][x], s[1]);
                    s[2] = fmaf(__builtin_amdgcn_fmed3f(y - tt.z, 0.0f, 1.0f), e[2][x], s[2]);
                    s[3] = fmaf(__builtin_amdgcn_fmed3f(y - tt.w, 0.0f, 1.0f), e[3][x], s[3]);
                }
                const float w = quad_sum(s, odd, high);
                z3 = ((lane >> 2) & 3) == c ? w : z3;
            }
        }
        const float total = rows_sum(z0, z1, z2, z3);
        const int64_t k = map * p.per + q0 + q;
        if (in) (p.parts == 1 ? p.total : p.part_total + (int64_t)part * p.maps * p.per * p.n)[k * p.n + i] = total;
        if (p.parts == 1)
            end_steps<E, K, true>(p, in && t >= 0.0f && t < (float)(p.n - 1), map, k, i, t, mine, total, lane);
    }
}

template <typename E, int K>
__global__ __launch_bounds__(64 * kWaves) void k_shared_grad(LogpParams p)
{
    extern __shared__ float tile[];                     // [tours of a pass][64 K] positions; in the end [waves][64 K]
    __shared__ float4 when[kWaves][kTile], weight[kWaves][kTile];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float* hits = tile + wave * 64 * K;
    const int64_t b = work_block();
    const int part = (int)(b % p.parts);
    const int64_t group = b / p.parts, map = group / p.groups;
    const int r0 = (int)(group % p.groups) * (kWaves * kRows) + wave * kRows;
    const int col0 = part * 64 * K, cols = min(64 * K, p.n - col0);
    const E* row0 = static_cast<const E*>(p.logits) + map * p.map_stride + col0;
    const int i = r0 + (lane & 3);

    float sum[kRows][K];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int x = 0; x < K; ++x) sum[r][x] = 0.0f;
    bool any_redo = false;
    for (int q0 = 0; q0 < p.per; q0 += kTile) {
        const int count = min(kTile, p.per - q0);
        const float* pos = p.pos + (map * p.per + q0) * (int64_t)p.n;
        if (q0) __syncthreads();
        stage<K>(tile, pos, count, p.n, col0, cols, wave, lane);
        const int q = lane >> 2;
        const bool in = q < count && i < p.n;
        const int64_t k = map * p.per + q0 + q;
        const float t = in ? pos[(int64_t)q * p.n + i] : 65536.0f;
        float w = 0.0f;
        if (in && t >= 0.0f && t < (float)(p.n - 1)) {
            const float g = p.g[k * (p.n - 1) + (int)t], total = p.total[k * p.n + i];
            if (g != 0.0f) {
                w = g / total;
                if (!(total >= kSmall) || !(fabsf(w) < kInf)) { w = 0.0f; any_redo = true; }
            }
        }
        reinterpret_cast<float*>(when[wave])[lane] = t;
        reinterpret_cast<float*>(weight[wave])[lane] = w;
        __syncthreads();
        for (int qq = 0; qq < count; ++qq) {
            const float4 tt = when[wave][qq], ww = weight[wave][qq];
            const float* at = tile + qq * 64 * K;
#pragma unroll
            for (int x = 0; x < K; ++x) {
                const float y = at[column<K>(x, lane)];
                sum[0][x] = fmaf(__builtin_amdgcn_fmed3f(y - tt.x, 0.0f, 1.0f), ww.x, sum[0][x]);
                sum[1][x] = fmaf(__builtin_amdgcn_fmed3f(y - tt.y, 0.0f, 1.0f), ww.y, sum[1][x]);
                sum[2][x] = fmaf(__builtin_amdgcn_fmed3f(y - tt.z, 0.0f, 1.0f), ww.z, sum[2][x]);
                sum[3][x] = fmaf(__builtin_amdgcn_fmed3f(y - tt.w, 0.0f, 1.0f), ww.w, sum[3][x]);
            }
        }
    }
    const uint64_t redo = __ballot(any_redo);
    __syncthreads();
    Row<E, K> raw[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) load_row<E, K>(row0 + (int64_t)min(r0 + r, p.n - 1) * p.row_stride, lane, cols, raw[r]);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int ii = r0 + r;
        if (ii >= p.n) break;
        const E* row = row0 + (int64_t)ii * p.row_stride;
        float h[K], d[K];
        end_row<E, K>(raw[r], lane, cols, h);
        const float from = base_of(p.top[map * p.n + ii]);
        // an entry that no tour had open may hold anything: its weight is 0, and so is its gradient
#pragma unroll
        for (int x = 0; x < K; ++x)
            d[x] = sum[r][x] != 0.0f ? -sum[r][x] * scaled_exp(h[x] - from) : 0.0f;
        // + g at the chosen entries.  Tours of one map often choose the same one: they are added one after the other,
        // in their order, by one lane at a time.
#pragma unroll
        for (int x = 0; x < K; ++x) hits[column<K>(x, lane)] = 0.0f;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");      // the lanes of a wave write each other's columns
        const bool row_redo = redo & (0x1111111111111111ull << r);
        for (int q0 = 0; q0 < p.per; q0 += 64) {
            const int q = q0 + lane;
            const int64_t k = map * p.per + q;
            float g = 0.0f;
            int to = -1;
            bool again = false;
            float t = 0.0f;
            if (q < p.per) {
                t = p.pos[k * p.n + ii];
                if (t >= 0.0f && t < (float)(p.n - 1)) {
                    g = p.g[k * (p.n - 1) + (int)t];
                    const float total = p.total[k * p.n + ii];
                    again = g != 0.0f && (!(total >= kSmall) || !(fabsf(g / total) < kInf));
                    to = (int)p.next[k * p.n + ii] - col0;
                }
            }
            if (row_redo) {
                uint64_t todo = __ballot(again);
                while (todo) {
                    const int l = __ffsll((unsigned long long)todo) - 1;
                    todo &= todo - 1;
                    const int64_t kk = map * p.per + q0 + l;
                    const float tt = lane_value(t, l), gg = lane_value(g, l);
                    float m, s;
                    open_sum<E, K>(row - col0, p.pos + kk * p.n, tt, p.n, lane, m, s);
                    if (s == 0.0f) {                    // nothing was open: no choice, no gradient
                        if (lane == l) to = -1;
                        continue;
                    }
                    const float ws = gg / s;
#pragma unroll
                    for (int x = 0; x < K; ++x) {
                        const int j = column<K>(x, lane);
                        if (j < cols && p.pos[kk * p.n + col0 + j] > tt)
                            d[x] -= ws * __builtin_amdgcn_exp2f((h[x] - base_of(m)) * kLog2e);
                    }
                }
            }
            uint64_t chosen = __ballot(g != 0.0f && to >= 0 && to < cols);
            while (chosen) {
                const int l = __ffsll((unsigned long long)chosen) - 1;
                chosen &= chosen - 1;
                if (lane == l) __hip_atomic_fetch_add(&hits[to], g, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int x = 0; x < K; ++x) d[x] += hits[column<K>(x, lane)];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        store_row<E, K>(static_cast<E*>(p.grad) + (map * p.n + ii) * (int64_t)p.n + col0, lane, cols, d);
    }
}

// ---- one tour a row
template <typename E, int K>
__global__ __launch_bounds__(256) void k_single(LogpParams p)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t w = work_block() * 4 + wave;
    const int part = (int)(w % p.parts);
    const int64_t group = w / p.parts, k = group / p.groups;
    if (k >= p.maps) return;
    const int r0 = (int)(group % p.groups) * kSingleRows;
    const int col0 = part * 64 * K, cols = min(64 * K, p.n - col0);
    const bool odd = lane & 1, high = lane & 2;
    float pos[K];
#pragma unroll
    for (int x = 0; x < K; ++x) {
        const int j = column<K>(x, lane);
        pos[x] = j < cols ? p.pos[k * p.n + col0 + j] : -1.0f;
    }
    const int count = min(kSingleRows, p.rows - r0);
    const int mine = 4 * (lane >> 4) + (lane & 3);      // the row whose results this lane ends up with
    const int r_mine = r0 + min(mine, count - 1);
    const float when = p.by_step ? (float)r_mine : p.pos[k * p.n + r_mine];
    const E* row0 = static_cast<const E*>(p.logits) + k * p.map_stride + col0;
    float z0 = 0.0f, z1 = 0.0f, z2 = 0.0f, z3 = 0.0f, top = -kInf;
    for (int a = 0; a < kSingleRows / 4; ++a) {
        z0 = z1; z1 = z2; z2 = z3; z3 = 0.0f;
        if (4 * a >= count) continue;
        float h[4][K], s[4], tt[4];
        Row<E, K> raw[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = min(4 * a + r, count - 1);
            load_row<E, K>(row0 + (int64_t)(r0 + i) * p.row_stride, lane, cols, raw[r]);
            tt[r] = lane_value(when, 16 * (i >> 2) + (i & 3));
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float m = -kInf;
            end_row<E, K>(raw[r], lane, cols, h[r]);
#pragma unroll
            for (int x = 0; x < K; ++x) {
                h[r][x] = pos[x] > tt[r] ? h[r][x] : -kInf;
                m = fmaxf(m, h[r][x]);
            }
            m = row_max(m);
            const float from = base_of(m);
            float sum = 0.0f;
#pragma unroll
            for (int x = 0; x < K; ++x) sum += __builtin_amdgcn_exp2f((h[r][x] - from) * kLog2e);
            s[r] = sum;
            top = mine == 4 * a + r ? m : top;
        }
        z3 = quad_sum(s, odd, high);
    }
    const float total = rows_sum(z0, z1, z2, z3);
    const bool writes = mine < count && ((lane >> 2) & 3) == 0;
    const int64_t at = k * p.rows + r0 + mine;
    if (writes) {
        (p.parts == 1 ? p.top : p.part_top + (int64_t)part * p.maps * p.rows)[at] = top;
        (p.parts == 1 ? p.total : p.part_total + (int64_t)part * p.maps * p.rows)[at] = total;
    }
    if (p.parts == 1)
        end_steps<E, K, false>(p, writes && p.pos[k * p.n] >= 0.0f && when < (float)(p.n - 1), k, k, r0 + mine, when, top,
                            total, lane);
}

template <typename E, int K>
__global__ __launch_bounds__(256) void k_single_grad(LogpParams p)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t w = work_block() * 4 + wave;
    const int part = (int)(w % p.parts);
    const int64_t group = w / p.parts, k = group / p.groups;
    if (k >= p.maps) return;
    const int r0 = (int)(group % p.groups) * kSingleRows;
    const int col0 = part * 64 * K, cols = min(64 * K, p.n - col0);
    float pos[K];
#pragma unroll
    for (int x = 0; x < K; ++x) {
        const int j = column<K>(x, lane);
        pos[x] = j < cols ? p.pos[k * p.n + col0 + j] : -1.0f;
    }
    const int count = min(kSingleRows, p.rows - r0);
    float when = 0.0f, from = 0.0f, weight = 0.0f, g = 0.0f;        // of row r0 + lane
    if (lane < count) {
        const int64_t at = k * p.rows + r0 + lane;
        when = p.by_step ? (float)(r0 + lane) : p.pos[k * p.n + r0 + lane];
        from = base_of(p.top[at]);
        const float total = p.total[at];
        if (p.pos[k * p.n] >= 0.0f && when < (float)(p.n - 1) && total != 0.0f) {
            g = p.g[k * (p.n - 1) + (int)when];
            weight = g / total;
        }
    }
    const E* row0 = static_cast<const E*>(p.logits) + k * p.map_stride + r0 * p.row_stride + col0;
    E* out0 = static_cast<E*>(p.grad) + (k * p.rows + r0) * (int64_t)p.n + col0;
    for (int r0 = 0; r0 < count; r0 += 2) {             // two rows in flight
        Row<E, K> raw[2];
#pragma unroll
        for (int a = 0; a < 2; ++a) load_row<E, K>(row0 + (int64_t)min(r0 + a, count - 1) * p.row_stride, lane, cols, raw[a]);
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            const int r = r0 + a;
            if (r >= count) break;
            const float tt = lane_value(when, r), ff = lane_value(from, r), ww = lane_value(weight, r), gg = lane_value(g, r);
            float d[K];
            end_row<E, K>(raw[a], lane, cols, d);
            if (gg == 0.0f) {                           // whatever the row holds
#pragma unroll
                for (int x = 0; x < K; ++x) d[x] = 0.0f;
            } else {
#pragma unroll
                for (int x = 0; x < K; ++x) {
                    const float y = -ww * __builtin_amdgcn_exp2f((d[x] - ff) * kLog2e);
                    d[x] = pos[x] > tt ? (pos[x] == tt + 1.0f ? y + gg : y) : 0.0f;
                }
            }
            store_row<E, K>(out0 + (int64_t)r * p.n, lane, cols, d);
        }
    }
}

// Puts the parts of long rows together and ends their steps: one lane a (tour, row).
template <typename E, bool SHARED>
__global__ __launch_bounds__(256) void k_join(LogpParams p)
{
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x, all = p.maps * p.per * p.rows;
    const bool in = w < all;
    const int64_t k = in ? w / p.rows : 0;
    const int r = in ? (int)(w - k * p.rows) : 0;
    const int64_t row = SHARED ? k / p.per * p.rows + r : w;
    float top = -kInf, total = 0.0f;
    if (in) {
        for (int c = 0; c < p.parts; ++c) top = fmaxf(top, p.part_top[c * p.maps * p.rows + row]);
        for (int c = 0; c < p.parts; ++c) {
            const float m = base_of(p.part_top[c * p.maps * p.rows + row]), s = p.part_total[c * all + w];
            const float x = (m - base_of(top)) * kLog2e;
            if (s == 0.0f) continue;
            // a shared sum is up to 2^76 and counts down to 2^-80: its factor must not be flushed before it is applied
            total += SHARED && x < -40.0f ? s * __builtin_amdgcn_exp2f(x + 60.0f) * (1.0f / kScale)
                                          : s * __builtin_amdgcn_exp2f(x);
        }
        p.total[w] = total;
        if (!SHARED || k % p.per == 0) p.top[row] = top;
    }
    const float when = in ? (p.by_step ? (float)r : p.pos[k * p.n + r]) : 0.0f;
    end_steps<E, kMaxPer, SHARED>(p, in && p.pos[k * p.n] >= 0.0f && when < (float)(p.n - 1), SHARED ? k / p.per : k, k, r, when,
                         top, total, lane);
}

// Columns of a wave: the fewest registers a lane that hold the row, or an even part of a long one.
inline int parts_of(int n) { return (n + 64 * kMaxPer - 1) / (64 * kMaxPer); }

inline int held(int n)
{
    const int parts = parts_of(n), need = ((n + parts - 1) / parts + 63) / 64;
    for (int k : {1, 2, 4, 6, 8, 12})
        if (need <= k) return k;
    return kMaxPer;
}

#define T2O_BY_HELD(k, CALL)                                \
    switch (k) {                                            \
        case 1: { constexpr int K = 1; CALL; break; }       \
        case 2: { constexpr int K = 2; CALL; break; }       \
        case 4: { constexpr int K = 4; CALL; break; }       \
        case 6: { constexpr int K = 6; CALL; break; }       \
        case 8: { constexpr int K = 8; CALL; break; }       \
        case 12: { constexpr int K = 12; CALL; break; }     \
        default: { constexpr int K = 16; CALL; break; }     \
    }

template <typename Kernel>
int shared_launch(Kernel kern, LogpParams p, unsigned grid, size_t lds, hipStream_t stream)
{
    if (lds > 48 * 1024)
        HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)lds));
    hipLaunchKernelGGL(kern, dim3(grid), dim3(64 * kWaves), lds, stream, p);
    return 0;
}

template <typename E>
int logp_launch(LogpParams p, bool grad, hipStream_t stream)
{
    const bool shared = p.per > 1;
    const int k = held(p.n), per_block = shared ? kWaves * kRows : kSingleRows;
    p.parts = parts_of(p.n);
    p.groups = (p.rows + per_block - 1) / per_block;
    p.tile = p.per < kTile ? p.per : kTile;
    const int64_t units = p.maps * p.groups * p.parts, grid = shared ? units : (units + 3) / 4;
    if (grid > 0x7fffffffll) return fail(TSP2OPT_E_UNSUPPORTED, "too many rows");
    int rc = 0;
    if (shared) {
        const size_t lds = sizeof(float) * 64 * k * (grad && p.tile < kWaves ? kWaves : p.tile);
        if (grad) T2O_BY_HELD(k, (rc = shared_launch(k_shared_grad<E, K>, p, (unsigned)grid, lds, stream)))
        else T2O_BY_HELD(k, (rc = shared_launch(k_shared<E, K>, p, (unsigned)grid, lds, stream)))
    } else {
        if (grad) T2O_BY_HELD(k, hipLaunchKernelGGL((k_single_grad<E, K>), dim3((unsigned)grid), dim3(256), 0, stream, p))
        else T2O_BY_HELD(k, hipLaunchKernelGGL((k_single<E, K>), dim3((unsigned)grid), dim3(256), 0, stream, p))
    }
    if (rc) return rc;
    if (!grad && p.parts > 1) {
        const unsigned blocks = (unsigned)((p.maps * p.per * p.rows + 255) / 256);
        if (shared) hipLaunchKernelGGL((k_join<E, true>), dim3(blocks), dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((k_join<E, false>), dim3(blocks), dim3(256), 0, stream, p);
    }
    HIP_TRY(hipGetLastError());
    return 0;
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

// Offsets of the state's arrays and its size: positions, successors, row maxima, sums, and for long rows the parts.
struct LogpState {
    int64_t pos, next, top, total, part_top, part_total, bytes;
    LogpState(int64_t T, int32_t n, int32_t per, int32_t by_step)
    {
        const int64_t rows = by_step ? n - 1 : n, parts = parts_of(n), many = parts > 1 ? parts : 0;
        int64_t at = 0;
        auto take = [&](int64_t bytes) { const int64_t a = at; at += round256(bytes); return a; };
        pos = take(4 * T * n);
        next = take(2 * T * n);
        top = take(4 * (T / per) * rows);
        total = take(4 * T * rows);
        part_top = take(4 * many * (T / per) * rows);
        part_total = take(4 * many * T * rows);
        bytes = at + 256;
    }
};

LogpParams logp_params(const void* logits, const int64_t* tours, void* state, int64_t num_tours, int32_t n, int32_t per,
                       int32_t by_step, int64_t map_stride, int64_t row_stride)
{
    LogpParams p{};
    const LogpState s(num_tours, n, per, by_step);
    char* at = static_cast<char*>(state);
    p.logits = logits; p.tours = tours;
    p.pos = reinterpret_cast<float*>(at + s.pos); p.next = reinterpret_cast<uint16_t*>(at + s.next);
    p.top = reinterpret_cast<float*>(at + s.top); p.total = reinterpret_cast<float*>(at + s.total);
    p.part_top = reinterpret_cast<float*>(at + s.part_top); p.part_total = reinterpret_cast<float*>(at + s.part_total);
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
    return LogpState(num_tours, n, tours_per_map, rows).bytes;
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
    if (state_bytes < LogpState(num_tours, n, tours_per_map, rows).bytes) return fail(TSP2OPT_E_WORKSPACE, "state_bytes too small");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(TSP2OPT_E_HIP, "hipSetDevice failed");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    LogpParams p = logp_params(logits, tours, state, num_tours, n, tours_per_map, rows, map_stride, row_stride);
    p.logp = logp_out;
    const size_t lds = 2 * (size_t)n;
    if (lds > 48 * 1024)
        HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(k_positions),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    const unsigned threads = n <= 64 ? 64 : n <= 128 ? 128 : n <= 1024 ? 256 : 1024;
    hipLaunchKernelGGL(k_positions, dim3((unsigned)num_tours), dim3(threads), lds, stream, tours, p.pos, p.next, logp_out,
                       n);
    int result = 0;
    T2O_BY_DTYPE(dtype, result = logp_launch<E>(p, false, stream));
    return result;
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
    if (state_bytes < LogpState(num_tours, n, tours_per_map, rows).bytes) return fail(TSP2OPT_E_WORKSPACE, "state_bytes too small");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(TSP2OPT_E_HIP, "hipSetDevice failed");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    LogpParams p = logp_params(logits, tours, const_cast<void*>(state), num_tours, n, tours_per_map, rows, map_stride,
                               row_stride);
    p.g = grad_logp;
    p.grad = grad_out;
    int result = 0;
    T2O_BY_DTYPE(dtype, result = logp_launch<E>(p, true, stream));
    return result;
}
