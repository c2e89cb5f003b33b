// ml4tspbench_amd/csrc/tour_logprobs.hip -- step log-probabilities of tours under heat maps / decoder logits
//
// A tour starts at tour[0] and step t = 0 .. n-2 chooses tour[t+1] among the nodes not visited yet, with the softmax
// of one row of logits over those nodes:
//     lp(t) = h[r, tour[t+1]] - log sum_{j : pos(j) > t} exp h[r, j],
// pos(j) = the step that visits j (the inverse permutation), r = tour[t] for heat maps, r = t for the rows that an
// autoregressive decoder wrote.  Gradient, with g(t) the gradient of lp(t):
//     dh[r, j] = sum over the tours that share the row of  g(t) ([j = tour[t+1]] - [pos(j) > t] softmax_j).
//
// Rows are kept in registers, K entries a lane, loaded once.  A row of up to 256 entries takes G = 16 lanes (four rows
// side by side in a wave: sums over 16 lanes need no cross-row steps), longer ones G = 64; rows of more than 1024 are
// split into parts whose maxima and sums k_join puts together.  Values + gradient in us with 16 and with 64 lanes:
// 250 maps x 20 tours of 200 nodes 55 + 66 and 57 + 77, 2000 x 1 of 200 92 + 110 and 101 + 121, 1000 x 16 of 128
// 46 + 64 and 92 + 116 (float32).
//
// Several tours a map (k_shared): e_j = exp(h_j - row maximum) does not depend on the tour, only which e_j are added
// does, and positions are whole numbers, so a masked addition is
//     S += min(max(pos_j - t, 0), 1) * e_j
// instead of an exponential a tour: a subtraction with clamp and a fused multiply-add.  Up to 2048 nodes, where half
// floats hold every position and difference exactly, the subtraction takes two entries at a time (v_pk_add_f16 clamp)
// and v_fma_mix_f32 widens the 0 or 1 on its way into the float sum.
// That sum loses steps whose open entries all lie far below the row's maximum, so the exponentials are kept times 2^60,
// which spends the range of float above 1 too: what it flushes (below 2^-126, 65535 entries at most) is under 2^-30 of a
// sum above 2^-80, which is 2^-140 = e^-97 relative to the row's maximum.  Steps below that (and those that are NaN) are
// redone alone, relative to their own maximum.  The others are rounded at their distance from the row's maximum and not
// from their own: 2^-24 of up to 97, the price of one exponential for all tours.  On 16 TSP-500 maps exp(-distance / tau)
// with 256 sampled tours the largest error of a log-probability is 7.6e-6 and their root mean square 1.9e-7; with every
// step's own maximum (k_single) 9.7e-7 and 8.6e-8.
// One tour a row (k_single): the maximum is the open entries' own, nothing is ever lost.
#include "learn_common.hpp"

#include <type_traits>

namespace t2o {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kSmall = 0x1p-80f, kScale = 0x1p60f;
constexpr float kDead = -1.0f;                      // k_shared's total of a step with no open entry
constexpr int kRows = 4, kTile = 16;                // k_shared: rows of a group of lanes, tours a pass
constexpr int kSingleRows = 16;                     // k_single: rows a wave
constexpr int kMaxPer = 16;                         // entries of a row a lane holds at most
constexpr int kShortRow = 256;                      // longest row of a group of 16 lanes
constexpr int kHalfRow = 2048;                      // up to here half floats hold every position and difference exactly

struct LogpParams {
    const void* logits;
    const int64_t* tours;
    float* logp;            // (T, n - 1)
    float* pos;             // (T, n); -1 everywhere: the tour is no permutation
    uint16_t* next;         // (T, n): the node after a node
    float* top;             // (M, rows) shared, (T, rows) single: what the exponentials are relative to
    float* total;           // (T, rows): sum of exp(h - top) over the open entries (shared: times 2^60)
    float* part_top;        // [parts](M or T, rows)
    float* part_total;      // [parts](T, rows)
    const float* g;         // (T, n - 1)
    void* grad;             // (M, rows, n)
    int64_t maps, map_stride, row_stride, groups;
    int32_t n, rows, per, by_step, parts;
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

// ---- rows in registers: lane l of a group of G holds entries c G V + l V + v, V adjacent ones a load.  Rows of odd
// length start anywhere, so the loads are aligned to the element only, which the memory pipe takes at full width.
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

// V adjacent entries of a row in LDS, aligned to their size: one access of 8 or 16 bytes a lane.  (Two of 4 bytes would
// leave every other bank idle.)
template <typename E, int V>
struct Aligned {
    typedef E type __attribute__((ext_vector_type(V)));
};
template <typename E>
struct Aligned<E, 1> {
    typedef E type;
};

// Loads are issued without a branch: a lane at or behind the end reads the row's last V entries instead (in front of a
// short last part there is the previous one) and end_row puts its entries in place.
template <typename E, int K>
struct Row {
    typename Pack<E, kVec<K>>::type x[K / kVec<K>];
};

template <typename E, int K, int G>
__device__ __forceinline__ void load_row(const E* row, int l, int cols, Row<E, K>& raw)
{
    constexpr int V = kVec<K>;
    using P = typename Pack<E, V>::type;
#pragma unroll
    for (int c = 0; c < K / V; ++c) raw.x[c] = *reinterpret_cast<const P*>(row + min(c * G * V + l * V, cols - V));
}

template <typename E, int K, int G>
__device__ __forceinline__ void end_row(const Row<E, K>& raw, int l, int cols, float (&h)[K])
{
    constexpr int V = kVec<K>;
#pragma unroll
    for (int c = 0; c < K / V; ++c) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (V == 1) h[c] = widen(raw.x[c]);
            else h[c * V + v] = widen(raw.x[c][v]);
        }
        if ((c + 1) * G * V <= cols) continue;
        const int shift = c * G * V + l * V - (cols - V);       // <= 0: the lane's own entries were read
        if (cols % V == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) h[c * V + v] = shift <= 0 ? h[c * V + v] : -kInf;
        } else {
            float x[V];
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = h[c * V + v];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float y = -kInf;
#pragma unroll
                for (int w = V - 1; w > v; --w) y = shift == w - v ? x[w] : y;
                h[c * V + v] = shift <= 0 ? x[v] : y;
            }
        }
    }
}

template <typename E, int K, int G>
__device__ __forceinline__ void store_row(E* row, int l, int cols, const float (&d)[K])
{
    constexpr int V = kVec<K>;
    using P = typename Pack<E, V>::type;
#pragma unroll
    for (int c = 0; c < K / V; ++c) {
        const int j = c * G * V + l * V;
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

// The column of register i of lane l.
template <int K, int G>
__device__ __forceinline__ int column(int i, int l)
{
    constexpr int V = kVec<K>;
    return (i / V) * G * V + l * V + i % V;
}

// ---- sums and maxima over the G lanes of a group
template <int CTRL>
__device__ __forceinline__ float dpp(float x)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// fmaxf quiets its operands first; these are one instruction.  A NaN operand is left out, as fmaxf leaves it out.
__device__ __forceinline__ float vmax(float a, float b)
{
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
    return r;
}

__device__ __forceinline__ float vmax3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

template <int K>
__device__ __forceinline__ float max_of(const float (&h)[K])
{
    if constexpr (K == 1) return h[0];
    float m = vmax(h[0], h[1]);
#pragma unroll
    for (int x = 2; x + 1 < K; x += 2) m = vmax3(m, h[x], h[x + 1]);
    return m;                                           // K is 1 or even
}

template <typename F>
__device__ __forceinline__ float swap16(float a, float b, F f)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <typename F>
__device__ __forceinline__ float swap32(float a, float b, F f)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

struct Add {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
    __device__ __forceinline__ float operator()(float a, float b) const { return vmax(a, b); }
};

template <int G, typename F>
__device__ __forceinline__ float all(float v, F f)
{
    v = f(v, dpp<0xB1>(v));                             // quad_perm [1,0,3,2]
    v = f(v, dpp<0x4E>(v));                             // quad_perm [2,3,0,1]
    v = f(v, dpp<0x141>(v));                            // row_half_mirror
    v = f(v, dpp<0x140>(v));                            // row_mirror
    if constexpr (G == 64) v = swap32(swap16(v, v, f), swap16(v, v, f), f);
    return v;
}

// a[0..3] -> value (lane & 3) over the 16 lanes of this lane's row, in every lane of that row
template <typename F>
__device__ __forceinline__ float quads(const float (&a)[4], bool odd, bool high, F f)
{
    const float u = f(odd ? a[1] : a[0], dpp<0xB1>(odd ? a[0] : a[1]));
    const float v = f(odd ? a[3] : a[2], dpp<0xB1>(odd ? a[2] : a[3]));
    float w = f(high ? v : u, dpp<0x4E>(high ? u : v));
    w = f(w, dpp<0x124>(w));                            // row_ror:4
    return f(w, dpp<0x128>(w));                         // row_ror:8
}

// z0..z3 -> z(lane >> 4) summed over the four rows of 16 lanes
__device__ __forceinline__ float rows_sum(float z0, float z1, float z2, float z3)
{
    return swap32(swap16(z0, z1, Add()), swap16(z2, z3, Add()), Add());
}

__device__ __forceinline__ float lane_value(float x, int lane)
{
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane));
}

// What the exponentials are relative to: an empty row's maximum is -inf, which no entry may be subtracted from.
__device__ __forceinline__ float base_of(float top) { return top == -kInf ? 0.0f : top; }

// exp(x) 2^60 of a difference x <= 0, down to where exp(x) 2^60 itself is flushed: as the square of exp(x / 2) 2^30.
__device__ __forceinline__ float scaled_exp(float x)
{
    const float y = __builtin_amdgcn_exp2f(x * (0.5f * kLog2e)) * 0x1p30f;
    return y * y;
}

__device__ __forceinline__ float plain_exp(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// The steps that k_shared cannot see, by a group of lanes: h becomes exp(h - top) of the open entries (positions `at`),
// 0 of the others; top and the sum.
template <int K, int G>
__device__ __forceinline__ void open_terms(float (&h)[K], const float (&at)[K], float when, float& top, float& total)
{
#pragma unroll
    for (int x = 0; x < K; ++x) h[x] = at[x] > when ? h[x] : -kInf;
    top = all<G>(max_of(h), Max());
    const float from = base_of(top);
    float s = 0.0f;
#pragma unroll
    for (int x = 0; x < K; ++x) s += h[x] = plain_exp(h[x] - from);
    total = all<G>(s, Add());
}

// The same for a row of any length, from memory.
template <typename E, int KK, int G>
__device__ void open_sum(const E* row, const float* pos, float when, int n, int l, float& top, float& total)
{
    constexpr int K = KK > 8 ? 8 : KK;                  // fewer registers than the rows that wait meanwhile
    top = -kInf;
    total = 0.0f;
    for (int c = 0; c < n; c += G * K) {
        const int cols = min(G * K, n - c);
        Row<E, K> raw;
        Row<float, K> raw_pos;
        load_row<E, K, G>(row + c, l, cols, raw);
        load_row<float, K, G>(pos + c, l, cols, raw_pos);
        float h[K], at[K], m, s;
        end_row<E, K, G>(raw, l, cols, h);
        end_row<float, K, G>(raw_pos, l, cols, at);
        open_terms<K, G>(h, at, when, m, s);
        const float now = vmax(top, m), from = base_of(now);
        if (total != 0.0f) total *= plain_exp(top - from);
        if (s != 0.0f) total += s * plain_exp(m - from);
        top = now;
    }
}

// The group's lanes with `todo`, one after the other: the lane whose turn it is, or -1 when the group is through.
template <int G>
struct Turns {
    uint64_t mask;
    int first;
    __device__ Turns(bool todo, int lane) : mask(__ballot(todo)), first(lane & ~(G - 1))
    {
        if constexpr (G < 64) mask = (mask >> first) & ((1ull << G) - 1);
    }
    __device__ bool more() const { return __any(mask != 0); }
    __device__ int take()
    {
        const int at = __ffsll((unsigned long long)mask) - 1;
        mask &= mask - 1;
        return at < 0 ? -1 : first + at;
    }
};

__device__ __forceinline__ int64_t shfl64(int64_t x, int src)
{
    return ((int64_t)__shfl((int)(x >> 32), src) << 32) | (unsigned)__shfl((int)x, src);
}

// Ends the steps of the lanes with `valid`: (tour k, row r, step `when`, node `next` chosen).  A shared total is 2^60 times
// the sum; steps of which it says nothing are redone one after the other by their group of lanes: all lanes have to be
// here.  redo(lane, top, total) redoes the step of one of a group's lanes (-1: none).  Returns what the gradient needs
// to know.
template <typename E, int G, bool SHARED, typename Redo>
__device__ __forceinline__ float end_steps(const LogpParams& p, bool valid, int64_t map, int64_t k, int r, float when,
                                           int next, float top, float total, int lane, Redo redo)
{
    const E* row = static_cast<const E*>(p.logits) + map * p.map_stride + (int64_t)r * p.row_stride;
    float chosen = 0.0f, keep = total;
    if (valid) chosen = widen(row[next]);
    // log(total) and not of total 2^-60 where that would leave the range of float
    float log_total = logf(!SHARED ? total : total >= 0x1p-60f ? total * (1.0f / kScale) : total);
    if (SHARED && total < 0x1p-60f) log_total -= 60.0f / kLog2e;
    if constexpr (SHARED) {
        for (Turns<G> turns(valid && !(total >= kSmall), lane); turns.more();) {
            const int turn = turns.take();
            float m = 0.0f, s = 0.0f;
            redo(turn, m, s);
            if (lane == turn) {
                top = m;
                total = s;
                log_total = logf(s);
                if (s == 0.0f) keep = kDead;
            }
        }
    }
    if (valid) p.logp[k * (p.n - 1) + (int)when] = total == 0.0f ? -kInf : (chosen - base_of(top)) - log_total;
    return keep;
}

// ---- several tours a map
template <int G>
constexpr int kWaves = G == 64 ? 8 : 4;
template <int G>
constexpr int kWaveRows = kRows * 64 / G;               // rows of a wave

using half2 = _Float16 __attribute__((ext_vector_type(2)));

// The steps at which a tour leaves the kRows rows of a group of lanes, as the masks take them.
template <typename Q>
struct Leaves {
    float t[kRows];
    __device__ __forceinline__ explicit Leaves(const float4& x) : t{x.x, x.y, x.z, x.w} {}
};
template <>
struct Leaves<_Float16> {
    half2 t[kRows];
    __device__ __forceinline__ explicit Leaves(const float4& x)
        : t{__builtin_bit_cast(half2, x.x), __builtin_bit_cast(half2, x.y), __builtin_bit_cast(half2, x.z),
            __builtin_bit_cast(half2, x.w)} {}
};

template <typename Q>
__device__ __forceinline__ float pack_step(float t)
{
    if constexpr (sizeof(Q) == 4) return t;
    const half2 both = {(_Float16)t, (_Float16)t};
    return __builtin_bit_cast(float, both);
}

template <typename Q>
__device__ __forceinline__ float unpack_step(float x)
{
    if constexpr (sizeof(Q) == 4) return x;
    return (float)__builtin_bit_cast(half2, x)[0];
}

constexpr float kNever = 4096.0f;                       // a step that no position comes after (n <= kHalfRow)
constexpr float kNeverFloat = 65536.0f;

// f(row, register, mask) for the K entries of a lane and the kRows rows: mask = 1 where the entry's position `at` is behind
// the step at which the tour leaves the row, else 0.
template <int K, int G, typename Q, typename F>
__device__ __forceinline__ void open_masks(const Q* at, int l, const Leaves<Q>& leaves, F f)
{
    constexpr int V = kVec<K>;
    if constexpr (V == 1) {                             // half floats always: one entry a lane is a row of up to 16
        const Q y = at[l];
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            f(r, 0, (float)__builtin_elementwise_min(
                        __builtin_elementwise_max((_Float16)(y - leaves.t[r][0]), (_Float16)0), (_Float16)1));
    } else {
#pragma unroll
        for (int c = 0; c < K; c += V) {
            const auto y = *reinterpret_cast<const typename Aligned<Q, V>::type*>(at + column<K, G>(c, l));
            if constexpr (sizeof(Q) == 4) {
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int r = 0; r < kRows; ++r) f(r, c + v, __builtin_amdgcn_fmed3f(y[v] - leaves.t[r], 0.0f, 1.0f));
            } else {
#pragma unroll
                for (int v = 0; v < V; v += 2) {
                    const half2 two = {y[v], y[v + 1]};
#pragma unroll
                    for (int r = 0; r < kRows; ++r) {
                        const half2 m = __builtin_elementwise_min(__builtin_elementwise_max(two - leaves.t[r], (half2)0),
                                                                  (half2)1);
                        f(r, c + v, (float)m[0]);
                        f(r, c + v + 1, (float)m[1]);
                    }
                }
            }
        }
    }
}

// The positions of a pass's tours in LDS, a group of 64 lanes a tour; behind the end of a row: -inf, which is never open.
template <int K, int G, typename Q>
__device__ __forceinline__ void stage(Q* tile, const float* pos, int count, int n, int col0, int cols, int wave, int lane)
{
    constexpr int per_wave = kTile / kWaves<G>, C = G * K;
    if constexpr (G == 64) {
        constexpr int V = kVec<K>;
        Row<float, K> raw[per_wave];
#pragma unroll
        for (int a = 0; a < per_wave; ++a) {
            const int q = min(a * kWaves<G> + wave, count - 1);
            load_row<float, K, 64>(pos + (int64_t)q * n + col0, lane, cols, raw[a]);
        }
#pragma unroll
        for (int a = 0; a < per_wave; ++a) {
            const int q = a * kWaves<G> + wave;
            if (q >= count) break;
            float at[K];
            end_row<float, K, 64>(raw[a], lane, cols, at);
#pragma unroll
            for (int c = 0; c < K / V; ++c) {
                typename Aligned<Q, V>::type y;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if constexpr (V == 1) y = (Q)at[c];
                    else y[v] = (Q)at[c * V + v];
                }
                *reinterpret_cast<typename Aligned<Q, V>::type*>(tile + q * C + c * 64 * V + lane * V) = y;
            }
        }
    } else {
        constexpr int steps = (C + 63) / 64;
        float x[per_wave][steps];
#pragma unroll
        for (int a = 0; a < per_wave; ++a)
#pragma unroll
            for (int c = 0; c < steps; ++c)
                x[a][c] = pos[(int64_t)min(a * kWaves<G> + wave, count - 1) * n + min(c * 64 + lane, cols - 1)];
#pragma unroll
        for (int a = 0; a < per_wave; ++a)
#pragma unroll
            for (int c = 0; c < steps; ++c) {
                const int q = a * kWaves<G> + wave, j = c * 64 + lane;
                if (q < count && j < C) tile[q * C + j] = (Q)(j < cols ? x[a][c] : -kInf);
            }
    }
}

// The same from the tours themselves, for rows that fit a workgroup's tile whole (G = 16): k_positions for a pass's
// tours, a wave a tour, with the successors.  A map's first workgroup also writes them down for the gradient.
template <int K, typename Q>
__device__ __forceinline__ void stage_tours(const LogpParams& p, Q* tile, uint16_t* after, int64_t k0, int count,
                                            bool writes, int wave, int lane)
{
    constexpr int C = 16 * K, steps = (C + 63) / 64, per_wave = kTile / kWaves<16>;
    for (int a = 0; a < per_wave; ++a) {
        const int q = a * kWaves<16> + wave;
        if (q >= count) break;
        const int64_t k = k0 + q;
        const int64_t* t = p.tours + k * (p.n + 1);
        int node[steps], then[steps];
#pragma unroll
        for (int c = 0; c < steps; ++c) {
            const int s = min(c * 64 + lane, p.n - 1);
            const int64_t j = t[s], i = t[min(s + 1, p.n - 1)];         // nothing is chosen after the last node
            node[c] = j >= 0 && j < p.n ? (int)j : -1;
            then[c] = (int)i;
        }
        bool bad = false;
#pragma unroll
        for (int c = 0; c < steps; ++c) {
            const int s = c * 64 + lane;
            if (s >= p.n) continue;
            if (node[c] < 0) bad = true;
            else tile[q * C + node[c]] = (Q)(float)s;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int c = 0; c < steps; ++c) {
            const int s = c * 64 + lane;
            if (s < p.n && node[c] >= 0) {
                bad |= (float)tile[q * C + node[c]] != (float)s;       // two steps at one node: one sees the other's
                after[q * C + node[c]] = (uint16_t)then[c];
            }
        }
        bad = __any(bad);
#pragma unroll
        for (int c = 0; c < steps; ++c) {
            const int j = c * 64 + lane;
            if (j < C && (bad || j >= p.n)) tile[q * C + j] = (Q)(j < p.n ? -1.0f : -kInf);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (!writes) continue;
#pragma unroll
        for (int c = 0; c < steps; ++c) {
            const int j = c * 64 + lane;
            if (j >= p.n) continue;
            p.pos[k * p.n + j] = (float)tile[q * C + j];
            p.next[k * p.n + j] = bad ? (uint16_t)0 : after[q * C + j];
            if (bad && j < p.n - 1) p.logp[k * (p.n - 1) + j] = __builtin_nanf("");
        }
    }
}

// Where a wave's work lies.
template <int K, int G>
struct SharedWork {
    int lane, wave, l, group, part, r0, mine, col0, cols;       // mine: first row of this lane's group of lanes
    int64_t map;
    bool first;                                                 // the map's first workgroup
    __device__ explicit SharedWork(const LogpParams& p)
    {
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        l = lane & (G - 1);
        group = lane / G;
        const int64_t b = work_block(), block = b / p.parts;
        part = (int)(b % p.parts);
        map = block / p.groups;
        first = block % p.groups == 0;
        r0 = (int)(block % p.groups) * (kWaves<G> * kWaveRows<G>) + wave * kWaveRows<G>;
        mine = r0 + group * kRows;
        col0 = part * G * K;
        cols = min(G * K, p.n - col0);
    }
};

// Reads the rows once and adds kRows rows up for a tour with every position that it reads from LDS.  128 maps x 16 tours of
// 500 nodes: 60 us in float32, 50 us in bfloat16 under the profiler, where every launch ends by itself (in a stream of
// passes 57 and 49 us, the 7 us of k_positions included).  Of the 60, reading and exponentiating the rows alone takes 32 us
// (128 MB, the rate of any large read here), the masked additions 22 and the ends of the steps 6: the workgroups of a unit
// run their phases side by side and overlap little.  Measured and left out: 6 instead of 4 waves a SIMD by limiting the
// registers (the same), workgroups of four waves (53 and 65 us), several blocks of rows in a workgroup with the next one's
// rows in flight (62 and 70 us: its registers halve the waves), sums over the lanes by v_mfma_f32_16x16x4 with a unit
// matrix (64 us in bfloat16 against 51: the matrix and vector instructions of these kernels do not run side by side),
// positions kept in memory as half floats in the order of the tile (62 and 54 us: nothing waits for them).
template <typename E, int K, int G, typename Q>
__global__ __launch_bounds__(64 * kWaves<G>) void k_shared(LogpParams p)
{
    extern __shared__ __align__(16) float lds[];
    Q* const tile = reinterpret_cast<Q*>(lds);          // [tours of a pass][G K] positions
    __shared__ float4 when[kWaves<G>][kTile][64 / G];   // the steps at which the tours leave a wave's rows
    __shared__ uint16_t after[G == 16 ? kTile * 16 * K : 1];
    const SharedWork<K, G> w(p);
    const int lane = w.lane, l = w.l;
    const bool odd = lane & 1, high = lane & 2;
    const E* row0 = static_cast<const E*>(p.logits) + w.map * p.map_stride + w.col0;

    float e[kRows][K], top[kRows];
    Row<E, K> raw[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
        load_row<E, K, G>(row0 + (int64_t)min(w.mine + r, p.n - 1) * p.row_stride, l, w.cols, raw[r]);
    auto stage_pass = [&](int q0, int count) {
        if constexpr (G == 16)
            stage_tours<K, Q>(p, tile, after, w.map * p.per + q0, count, w.first, w.wave, lane);
        else
            stage<K, G, Q>(tile, p.pos + (w.map * p.per + q0) * (int64_t)p.n, count, p.n, w.col0, w.cols, w.wave, lane);
    };
    stage_pass(0, min(kTile, p.per));
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        end_row<E, K, G>(raw[r], l, w.cols, e[r]);
        // the diagonal is never open: it must not set the maximum
        const int self = w.mine + r - w.col0;
#pragma unroll
        for (int c = 0; c < K; c += kVec<K>) {
            const int first = column<K, G>(c, 0);
            if (w.r0 + kWaveRows<G> <= w.col0 + first || w.r0 >= w.col0 + first + G * kVec<K>) continue;
#pragma unroll
            for (int v = 0; v < kVec<K>; ++v) e[r][c + v] = column<K, G>(c + v, l) == self ? -kInf : e[r][c + v];
        }
        top[r] = max_of(e[r]);
    }
    float mine = quads(top, odd, high, Max());          // of row lane & 3 of the group
    if constexpr (G == 64) mine = swap32(swap16(mine, mine, Max()), swap16(mine, mine, Max()), Max());
    top[0] = dpp<0x00>(mine);                           // quad_perm [r,r,r,r]
    top[1] = dpp<0x55>(mine);
    top[2] = dpp<0xAA>(mine);
    top[3] = dpp<0xFF>(mine);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const float from = base_of(top[r]);
#pragma unroll
        for (int x = 0; x < K; ++x) e[r][x] = scaled_exp(e[r][x] - from);
    }
    const int i = w.mine + (lane & 3);
    if (l < kRows && i < p.n)
        (p.parts == 1 ? p.top : p.part_top + (int64_t)w.part * p.maps * p.n)[w.map * p.n + i] = mine;

    float* const when_of = reinterpret_cast<float*>(when[w.wave]);      // [tour][row of the wave]
    // lane (tour, row i): its step, and its sum where this is the only part
    auto finish = [&](int q0, int q, int count, float total) {
        const float t = unpack_step<Q>(when_of[q * kWaveRows<G> + w.group * kRows + (lane & 3)]);
        const bool in = q < count && i < p.n;
        const int64_t k = w.map * p.per + q0 + q;
        if (p.parts == 1) {
            const bool valid = in && t >= 0.0f && t < (float)(p.n - 1);
            int next = 0;
            if (valid) {
                if constexpr (G == 16) next = after[q * G * K + i];
                else next = p.next[k * p.n + i];
            }
            total = end_steps<E, G, true>(p, valid, w.map, k, i, t, next, mine, total, lane,
                                          [&](int turn, float& m, float& s) {
                const int src = max(turn, 0), qq = __shfl(q, src);      // its positions are in LDS still
                const float tt = __shfl(t, src);
                Row<E, K> one;
                load_row<E, K, G>(row0 + (int64_t)min(w.mine + (src & 3), p.n - 1) * p.row_stride, l, w.cols, one);
                float h[K], at[K];
                end_row<E, K, G>(one, l, w.cols, h);
#pragma unroll
                for (int x = 0; x < K; ++x) at[x] = (float)tile[qq * G * K + column<K, G>(x, l)];
                open_terms<K, G>(h, at, tt, m, s);
            });
        }
        if (in) (p.parts == 1 ? p.total : p.part_total + (int64_t)w.part * p.maps * p.per * p.n)[k * p.n + i] = total;
    };

    for (int q0 = 0; q0 < p.per; q0 += kTile) {
        const int count = min(kTile, p.per - q0);
        const float* pos = p.pos + (w.map * p.per + q0) * (int64_t)p.n;
        if (q0) {
            __syncthreads();
            stage_pass(q0, count);
        }
        if constexpr (G == 16) __syncthreads();
#pragma unroll
        for (int x = lane; x < kTile * kWaveRows<G>; x += 64) {
            const int q = x / kWaveRows<G>, r = w.r0 + x % kWaveRows<G>;
            float t = sizeof(Q) == 4 ? kNeverFloat : kNever;
            if (q < count && r < p.n) {
                if constexpr (G == 16) t = (float)tile[q * G * K + r];
                else t = pos[(int64_t)q * p.n + r];
            }
            when_of[x] = pack_step<Q>(t);
        }
        if constexpr (G == 16) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        else __syncthreads();
        float z0 = 0.0f, z1 = 0.0f, z2 = 0.0f, z3 = 0.0f;
        for (int a = 0; a < kTile / 4; ++a) {
            z0 = z1; z1 = z2; z2 = z3; z3 = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int q = 4 * a + c;
                if (q >= count) continue;
                const Leaves<Q> leaves(when[w.wave][q][w.group]);
                float s[kRows] = {0.0f, 0.0f, 0.0f, 0.0f};
                open_masks<K, G, Q>(tile + q * G * K, l, leaves,
                                    [&](int r, int x, float m) { s[r] = fmaf(m, e[r][x], s[r]); });
                const float sum = quads(s, odd, high, Add());
                z3 = ((lane >> 2) & 3) == c ? sum : z3;
            }
            if constexpr (G == 16) {
                if (4 * a < count) finish(q0, 4 * a + ((lane >> 2) & 3), count, z3);
            }
        }
        if constexpr (G == 64) finish(q0, lane >> 2, count, rows_sum(z0, z1, z2, z3));
    }
}

// Equal targets among 16 lanes: their values are added up, nearest first, in the last lane of them; the others get -1.
__device__ __forceinline__ void join_equal(int& to, float& g)
{
    bool later = false;
    float sum = g;
    auto step = [&](auto shift) {
        constexpr int D = decltype(shift)::value;
        const int before = __builtin_amdgcn_update_dpp(-2, to, 0x110 + D, 0xf, 0xf, false);         // row_shr
        const int behind = __builtin_amdgcn_update_dpp(-2, to, 0x100 + D, 0xf, 0xf, false);         // row_shl
        const float x = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(g), 0x110 + D, 0xf, 0xf, false));
        sum += before == to ? x : 0.0f;
        later |= behind == to;
    };
    step(std::integral_constant<int, 1>()); step(std::integral_constant<int, 2>());
    step(std::integral_constant<int, 3>()); step(std::integral_constant<int, 4>());
    step(std::integral_constant<int, 5>()); step(std::integral_constant<int, 6>());
    step(std::integral_constant<int, 7>()); step(std::integral_constant<int, 8>());
    step(std::integral_constant<int, 9>()); step(std::integral_constant<int, 10>());
    step(std::integral_constant<int, 11>()); step(std::integral_constant<int, 12>());
    step(std::integral_constant<int, 13>()); step(std::integral_constant<int, 14>());
    step(std::integral_constant<int, 15>());
    g = sum;
    if (later) to = -1;
}

// sum_q g_q / S_q [open in tour q] for every entry of a row by the same masked additions, times its exponential, plus g
// at the chosen entries.  128 maps x 16 tours of 500 nodes in bfloat16: 66 us for 128 MB (27 us at the rate of a large
// copy), of which 20 are the masked additions and 7 the choices (copies without them take so much less); the rest is
// reading positions, steps and rows one after the other.
template <typename E, int K, int G, typename Q>
__global__ __launch_bounds__(64 * kWaves<G>) void k_shared_grad(LogpParams p)
{
    extern __shared__ __align__(16) float lds[];
    Q* const tile = reinterpret_cast<Q*>(lds);          // [tours of a pass][G K] positions, then [waves][64 K] floats
    __shared__ float4 when[kWaves<G>][kTile][64 / G], weight[kWaves<G>][kTile][64 / G];
    // of the steps: gradient; entry, bit 20: to be redone
    __shared__ float2 choice[G == 64 ? kWaves<G> : 1][kTile * kRows];
    const SharedWork<K, G> w(p);
    const int lane = w.lane, l = w.l;
    const bool once = G == 64 && p.per <= kTile;        // 16 lanes a row: the four rows' choices at one go
    const E* row0 = static_cast<const E*>(p.logits) + w.map * p.map_stride + w.col0;
    // what the gradient of tour q's step that leaves row i takes; g = 0: nothing
    struct Step {
        float t, g, total;
        int to;
    };
    auto step_of = [&](int q, int i, bool want_to) {
        Step s{sizeof(Q) == 4 ? kNeverFloat : kNever, 0.0f, 0.0f, -1};
        if (q >= p.per || i >= p.n) return s;
        const int64_t k = w.map * p.per + q;
        s.t = p.pos[k * p.n + i];
        if (!(s.t >= 0.0f && s.t < (float)(p.n - 1))) return s;
        s.total = p.total[k * p.n + i];
        if (s.total != kDead) s.g = p.g[k * (p.n - 1) + (int)s.t];
        if (want_to && s.g != 0.0f) s.to = (int)p.next[k * p.n + i];
        return s;
    };
    // g over the sum itself, without its 2^60: small gradients keep their digits
    auto weight_of = [](const Step& s) { return (s.g * 0x1p30f) / (s.total * 0x1p-30f); };
    auto unseen = [&](const Step& s) { return s.g != 0.0f && (!(s.total >= kSmall) || !(fabsf(weight_of(s)) < 0x1p100f)); };

    float sum[kRows][K];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int x = 0; x < K; ++x) sum[r][x] = 0.0f;
    bool any_redo = false;
    for (int q0 = 0; q0 < p.per; q0 += kTile) {
        const int count = min(kTile, p.per - q0);
        if (q0) __syncthreads();
        stage<K, G, Q>(tile, p.pos + (w.map * p.per + q0) * (int64_t)p.n, count, p.n, w.col0, w.cols, w.wave, lane);
#pragma unroll
        for (int x = lane; x < kTile * kWaveRows<G>; x += 64) {
            const Step s = step_of(q0 + x / kWaveRows<G>, w.r0 + x % kWaveRows<G>, once);
            const bool redo = unseen(s);
            any_redo |= redo;
            if (once) choice[w.wave][x] = make_float2(s.g, __int_as_float(redo ? s.to | 1 << 20 : s.to));
            reinterpret_cast<float*>(when[w.wave])[x] = pack_step<Q>(s.t);
            reinterpret_cast<float*>(weight[w.wave])[x] = redo || s.g == 0.0f ? 0.0f : weight_of(s);
        }
        __syncthreads();
        for (int q = 0; q < count; ++q) {
            const Leaves<Q> leaves(when[w.wave][q][w.group]);
            const float4 ww = weight[w.wave][q][w.group];
            const float weights[kRows] = {ww.x, ww.y, ww.z, ww.w};
            open_masks<K, G, Q>(tile + q * G * K, l, leaves,
                                [&](int r, int x, float m) { sum[r][x] = fmaf(m, weights[r], sum[r][x]); });
        }
    }
    Row<E, K> raw[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
        load_row<E, K, G>(row0 + (int64_t)min(w.mine + r, p.n - 1) * p.row_stride, l, w.cols, raw[r]);
    // + g at the chosen entries, through LDS: a row of zeros, the choices of 16 tours added with equal ones joined first
    // (all lanes then write different entries), further tours after them in their order.
    Step mine{};
    float g_mine = 0.0f;
    bool redo_mine = false;
    if (once) {
        const int x = (lane & 15) * kRows + (lane >> 4);
        const float2 c = choice[w.wave][x];
        mine.t = unpack_step<Q>(reinterpret_cast<const float*>(when[w.wave])[x]);
        g_mine = mine.g = c.x;
        mine.to = __float_as_int(c.y);
        redo_mine = mine.to >= 0 && (mine.to & 1 << 20);
        if (mine.to >= 0) mine.to &= (1 << 20) - 1;
        join_equal(mine.to, mine.g);
    }
    const bool redo_any = __any(any_redo);
    constexpr int V = kVec<K>;
    using Hits = typename Aligned<float, V>::type;
    float* const hits = reinterpret_cast<float*>(tile + min(kTile, p.per) * G * K) + (w.wave * (64 / G) + w.group) * G * K;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int i = w.mine + r;
        if (G == 64 && i >= p.n) break;
        float h[K], d[K];
        end_row<E, K, G>(raw[r], l, w.cols, h);
        const float from = base_of(p.top[w.map * p.n + min(i, p.n - 1)]);
        // an entry that no tour had open may hold anything: its weight is 0, and so is its gradient
#pragma unroll
        for (int x = 0; x < K; ++x) {
            const float y = plain_exp(0.5f * (h[x] - from));        // the square would be flushed too soon
            d[x] = sum[r][x] != 0.0f ? -(sum[r][x] * y) * y : 0.0f;
        }
#pragma unroll
        for (int x = 0; x < K; x += V) *reinterpret_cast<Hits*>(hits + column<K, G>(x, l)) = Hits(0.0f);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the lanes of a group write each other's columns
        constexpr int at_once = G == 64 ? 64 : 16;
        for (int q0 = 0; q0 < p.per; q0 += at_once) {
            Step s;
            if (once) {
                s = mine;
                if ((lane >> 4) != r) s.to = -1;
            } else {
                s = step_of(q0 + (G == 64 ? lane : l), i, true);
            }
            if (redo_any) {
                const bool todo = once ? redo_mine && (lane >> 4) == r : unseen(s);
                const float t_own = once ? mine.t : s.t, g_own = once ? g_mine : s.g;
                for (Turns<G> turns(todo, lane); turns.more();) {
                    const int turn = turns.take(), src = max(turn, 0);
                    const int q = q0 + (once || G == 16 ? src & 15 : src);
                    const float tt = __shfl(t_own, src), gg = __shfl(g_own, src);
                    float m, total, ex[K], at[K];
                    const float* pos = p.pos + (w.map * p.per + q) * (int64_t)p.n;
                    if (p.per <= kTile) {               // the tile holds all tours still
#pragma unroll
                        for (int x = 0; x < K; ++x) at[x] = (float)tile[q * G * K + column<K, G>(x, l)];
                    } else {
                        Row<float, K> raw_pos;
                        load_row<float, K, G>(pos + w.col0, l, w.cols, raw_pos);
                        end_row<float, K, G>(raw_pos, l, w.cols, at);
                    }
                    if (p.parts == 1) {
#pragma unroll
                        for (int x = 0; x < K; ++x) ex[x] = h[x];
                        open_terms<K, G>(ex, at, tt, m, total);
                    } else {
                        open_sum<E, K, G>(row0 - w.col0 + (int64_t)i * p.row_stride, pos, tt, p.n, l, m, total);
#pragma unroll
                        for (int x = 0; x < K; ++x) ex[x] = at[x] > tt ? plain_exp(h[x] - base_of(m)) : 0.0f;
                    }
                    const float ws = turn < 0 ? 0.0f : gg / total;
#pragma unroll
                    for (int x = 0; x < K; ++x) d[x] -= at[x] > tt && turn >= 0 ? ws * ex[x] : 0.0f;
                }
            }
            if (!once) join_equal(s.to, s.g);
            const int at = s.to - w.col0;
            const bool hit = at >= 0 && at < w.cols;
#pragma unroll
            for (int c = 0; c < (G == 64 ? 4 : 1); ++c)
                if (hit && (G == 16 || (lane >> 4) == c))
                    __hip_atomic_fetch_add(&hits[at], s.g, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int x = 0; x < K; x += V) {
            const Hits y = *reinterpret_cast<const Hits*>(hits + column<K, G>(x, l));
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if constexpr (V == 1) d[x] += y;
                else d[x + v] += y[v];
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (G == 64 || i < p.n)
            store_row<E, K, G>(static_cast<E*>(p.grad) + (w.map * p.n + i) * (int64_t)p.n + w.col0, l, w.cols, d);
    }
}

__device__ __forceinline__ int successor(const LogpParams& p, int64_t k, int r, float when)
{
    return p.by_step ? (int)p.tours[k * (p.n + 1) + (int)when + 1] : (int)p.next[k * p.n + r];
}

// ---- one tour a row: a wave has kSingleRows rows of a tour, 64 / G side by side
template <int K, int G>
struct SingleWork {
    int lane, l, group, part, r0, count, col0, cols;
    int64_t k;
    __device__ explicit SingleWork(const LogpParams& p)
    {
        lane = threadIdx.x & 63;
        l = lane & (G - 1);
        group = lane / G;
        const int64_t w = work_block() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), block = w / p.parts;
        part = (int)(w % p.parts);
        k = block / p.groups;
        r0 = (int)(block % p.groups) * kSingleRows;
        count = min(kSingleRows, p.rows - r0);
        col0 = part * G * K;
        cols = min(G * K, p.n - col0);
    }
};

// Bound by memory: 16 maps of 10000 nodes in float32 (6.4 GB) 1.07 ms, 6.0 TB/s; 10000 decoders' rows of TSP-100 in
// bfloat16 (198 MB) 63 us, 3.1 TB/s.  Four rows are in flight a wave, 16 share its positions.
template <typename E, int K, int G>
__global__ __launch_bounds__(256) void k_single(LogpParams p)
{
    const SingleWork<K, G> w(p);
    if (w.k >= p.maps) return;
    const int lane = w.lane, l = w.l;
    const bool odd = lane & 1, high = lane & 2;
    const float* const at = p.pos + w.k * p.n;
    const E* row0 = static_cast<const E*>(p.logits) + w.k * p.map_stride + (int64_t)w.r0 * p.row_stride + w.col0;
    Row<float, K> raw_pos;
    load_row<float, K, G>(at + w.col0, l, w.cols, raw_pos);
    // the row whose results this lane ends up with, of four lanes each
    const int mine = G == 64 ? 4 * (lane >> 4) + (lane & 3) : 4 * (lane & 3) + (lane >> 4);
    const bool writes = mine < w.count && ((lane >> 2) & 3) == 0;
    const int r_mine = w.r0 + min(mine, w.count - 1);
    const float when = p.by_step ? (float)r_mine : at[r_mine];
    float pos[K], top = -kInf, total = 0.0f;
    end_row<float, K, G>(raw_pos, l, w.cols, pos);
    if constexpr (G == 64) {
        float z0 = 0.0f, z1 = 0.0f, z2 = 0.0f, z3 = 0.0f;
        for (int a = 0; a < kSingleRows / 4; ++a) {
            z0 = z1; z1 = z2; z2 = z3; z3 = 0.0f;
            if (4 * a >= w.count) continue;
            float h[4][K], s[4];
            Row<E, K> raw[4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                load_row<E, K, G>(row0 + (int64_t)min(4 * a + r, w.count - 1) * p.row_stride, l, w.cols, raw[r]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float tt = lane_value(when, 16 * a + r);
                end_row<E, K, G>(raw[r], l, w.cols, h[r]);
#pragma unroll
                for (int x = 0; x < K; ++x) h[r][x] = pos[x] > tt ? h[r][x] : -kInf;
                s[r] = max_of(h[r]);
            }
            float m = quads(s, odd, high, Max());
            m = swap32(swap16(m, m, Max()), swap16(m, m, Max()), Max());
            top = (lane >> 4) == a ? m : top;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float from = base_of(lane_value(m, r));
                s[r] = 0.0f;
#pragma unroll
                for (int x = 0; x < K; ++x) s[r] += plain_exp(h[r][x] - from);
            }
            z3 = quads(s, odd, high, Add());
        }
        total = rows_sum(z0, z1, z2, z3);
    } else {
        constexpr int U = K > 8 ? 2 : 4;                // rows of a group in flight
#pragma unroll
        for (int a0 = 0; a0 < 4; a0 += U) {
            Row<E, K> raw[U];
            float tt[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = min(4 * (a0 + u) + w.group, w.count - 1);
                load_row<E, K, G>(row0 + (int64_t)r * p.row_stride, l, w.cols, raw[u]);
                tt[u] = p.by_step ? (float)(w.r0 + r) : at[w.r0 + r];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float h[K], s = 0.0f;
                end_row<E, K, G>(raw[u], l, w.cols, h);
#pragma unroll
                for (int x = 0; x < K; ++x) h[x] = pos[x] > tt[u] ? h[x] : -kInf;
                const float m = all<G>(max_of(h), Max()), from = base_of(m);
#pragma unroll
                for (int x = 0; x < K; ++x) s += plain_exp(h[x] - from);
                s = all<G>(s, Add());
                const bool own = (lane & 3) == a0 + u;
                top = own ? m : top;
                total = own ? s : total;
            }
        }
    }
    const int64_t to = w.k * p.rows + w.r0 + mine;
    if (writes) {
        (p.parts == 1 ? p.top : p.part_top + (int64_t)w.part * p.maps * p.rows)[to] = top;
        (p.parts == 1 ? p.total : p.part_total + (int64_t)w.part * p.maps * p.rows)[to] = total;
    }
    if (p.parts == 1) {
        const bool valid = writes && at[0] >= 0.0f && when < (float)(p.n - 1);
        end_steps<E, G, false>(p, valid, w.k, w.k, w.r0 + mine, when,
                               valid ? successor(p, w.k, w.r0 + mine, when) : 0, top, total, lane,
                               [](int, float&, float&) {});
    }
}

// Bound by memory: 16 maps of 10000 nodes in float32 (12.8 GB read and written) 2.47 ms, 5.2 TB/s; the decoders' rows above
// (396 MB) 87 us, 4.6 TB/s.
template <typename E, int K, int G>
__global__ __launch_bounds__(256) void k_single_grad(LogpParams p)
{
    const SingleWork<K, G> w(p);
    if (w.k >= p.maps) return;
    const int lane = w.lane, l = w.l;
    const float* const at = p.pos + w.k * p.n;
    const E* row0 = static_cast<const E*>(p.logits) + w.k * p.map_stride + (int64_t)w.r0 * p.row_stride + w.col0;
    E* out0 = static_cast<E*>(p.grad) + (w.k * p.rows + w.r0) * (int64_t)p.n + w.col0;
    Row<float, K> raw_pos;
    load_row<float, K, G>(at + w.col0, l, w.cols, raw_pos);
    float when = 0.0f, from = 0.0f, weight = 0.0f, g = 0.0f;        // of row r0 + lane
    if (lane < w.count) {
        const int64_t row = w.k * p.rows + w.r0 + lane;
        when = p.by_step ? (float)(w.r0 + lane) : at[w.r0 + lane];
        from = base_of(p.top[row]);
        const float total = p.total[row];
        if (at[0] >= 0.0f && when < (float)(p.n - 1) && total != 0.0f) {
            g = p.g[w.k * (p.n - 1) + (int)when];
            weight = -g / total;
        }
    }
    float pos[K];
    end_row<float, K, G>(raw_pos, l, w.cols, pos);
    constexpr int side = 64 / G, U = G == 64 ? 2 : K > 8 ? 2 : 4;   // rows side by side, and in flight of each
    for (int a = 0; a < w.count; a += side * U) {
        Row<E, K> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            load_row<E, K, G>(row0 + (int64_t)min(a + u * side + w.group, w.count - 1) * p.row_stride, l, w.cols, raw[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = a + u * side + w.group;
            if (a + u * side >= w.count) break;
            float tt, ff, ww, gg, d[K];
            if constexpr (G == 64) {
                tt = lane_value(when, r); ff = lane_value(from, r); ww = lane_value(weight, r); gg = lane_value(g, r);
            } else {
                tt = __shfl(when, r); ff = __shfl(from, r); ww = __shfl(weight, r); gg = __shfl(g, r);
            }
            end_row<E, K, G>(raw[u], l, w.cols, d);
            const bool none = gg == 0.0f;               // then whatever the row holds
            tt = none ? 65536.0f : tt;
            const float chosen = tt + 1.0f;
#pragma unroll
            for (int x = 0; x < K; ++x) {
                const float y = ww * plain_exp(d[x] - ff);
                d[x] = pos[x] > tt ? (pos[x] == chosen ? y + gg : y) : 0.0f;
            }
            if (G == 64 || r < w.count) store_row<E, K, G>(out0 + (int64_t)r * p.n, l, w.cols, d);
        }
    }
}

// Puts the parts of long rows together and ends their steps: one lane a (tour, row).  Where steps may have to be redone,
// one after the other in a wave, a wave has 16 of them: 7 maps x 3 tours of 1704 nodes with 10 neighbours 40 -> 23 us.
template <typename E, bool SHARED>
__global__ __launch_bounds__(256) void k_join(LogpParams p)
{
    constexpr int per_wave = SHARED ? 16 : 64;
    const int lane = threadIdx.x & 63;
    const int64_t w = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * per_wave + lane, every = p.maps * p.per * p.rows;
    const bool in = lane < per_wave && w < every;
    const int64_t k = in ? w / p.rows : 0, map = SHARED ? k / p.per : k;
    const int r = in ? (int)(w - k * p.rows) : 0;
    const int64_t row = map * p.rows + r;
    float top = -kInf, total = 0.0f;
    if (in) {
        for (int c = 0; c < p.parts; ++c) top = vmax(top, p.part_top[c * p.maps * p.rows + row]);
        for (int c = 0; c < p.parts; ++c) {
            const float m = base_of(p.part_top[c * p.maps * p.rows + row]), s = p.part_total[c * every + w];
            const float x = (m - base_of(top)) * kLog2e;
            if (s == 0.0f) continue;
            // a shared sum is up to 2^76 and counts down to 2^-80: its factor must not be flushed before it is applied
            total += SHARED && x < -40.0f ? s * __builtin_amdgcn_exp2f(x + 60.0f) * (1.0f / kScale)
                                          : s * __builtin_amdgcn_exp2f(x);
        }
        if (!SHARED || k % p.per == 0) p.top[row] = top;
    }
    const float when = in ? (p.by_step ? (float)r : p.pos[k * p.n + r]) : 0.0f;
    const bool valid = in && p.pos[k * p.n] >= 0.0f && when < (float)(p.n - 1);
    total = end_steps<E, 64, SHARED>(p, valid, map, k, r, when, valid ? successor(p, k, r, when) : 0, top, total, lane,
                                     [&](int turn, float& m, float& s) {
        const int src = max(turn, 0);
        const int64_t kk = shfl64(k, src), mm = shfl64(map, src);
        open_sum<E, kMaxPer, 64>(static_cast<const E*>(p.logits) + mm * p.map_stride + (int64_t)__shfl(r, src) * p.row_stride,
                                 p.pos + kk * p.n, __shfl(when, src), p.n, lane, m, s);
    });
    if (in) p.total[w] = total;
}

// Columns of a group of lanes: the fewest registers a lane that hold the row, or an even part of a long one.
inline int parts_of(int n) { return (n + 64 * kMaxPer - 1) / (64 * kMaxPer); }

inline int held(int n)
{
    const int lanes = n <= kShortRow ? 16 : 64, parts = parts_of(n);
    const int need = ((n + parts - 1) / parts + lanes - 1) / lanes;
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

// Launch shape of the kernels of one call, and whether a launch takes it: a grid of 2^32 threads or more starts nothing.
struct LogpShape {
    int k, parts, tours, position_threads;
    int64_t groups, rows_grid, rows_threads, join_grid;
    bool fits;
    LogpShape(int64_t T, int n, int rows, int per)
    {
        k = held(n);
        parts = parts_of(n);
        tours = per < kTile ? per : kTile;
        // us of k_positions with 64, 128, 256, 512, 1024 threads: 20000 tours of 50 nodes 11, 15.5, 24, 42, 71; 10000 of 100
        // 9.4, 10.2, 15, 25, 42; 2048 of 500 10.7, 7.6, 6.5, 7.8, 11.6; 128 of 1000 15, 8.7, 5.8, 4.8, 4.8; 16 of 10000
        // 131, 68, 36, 20, 14
        position_threads = n <= 128 ? 64 : n <= 512 ? 256 : n <= 1024 ? 512 : 1024;
        const int64_t maps = T / per;
        if (per > 1) {
            const int block = n <= kShortRow ? kWaves<16> * kWaveRows<16> : kWaves<64> * kWaveRows<64>;
            rows_threads = 64 * (n <= kShortRow ? kWaves<16> : kWaves<64>);
            groups = (rows + block - 1) / block;
            rows_grid = maps * groups * parts;
        } else {
            rows_threads = 256;
            groups = (rows + kSingleRows - 1) / kSingleRows;
            rows_grid = (maps * groups * parts + 3) / 4;
        }
        const int64_t items = per > 1 ? 64 : 256;
        join_grid = parts > 1 ? (T * rows + items - 1) / items : 0;
        fits = T * position_threads < (int64_t)1 << 32 && rows_grid * rows_threads < (int64_t)1 << 32 &&
               join_grid * 256 < (int64_t)1 << 32;
    }
};

template <typename Kernel>
int logp_start(Kernel kern, const LogpParams& p, int64_t grid, int64_t threads, size_t lds, hipStream_t stream)
{
    if (lds > 48 * 1024)
        HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)lds));
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3((unsigned)threads), lds, stream, p);
    return 0;
}

template <typename E, int K, int G>
int logp_rows(const LogpParams& p, const LogpShape& s, bool grad, hipStream_t stream)
{
    if (p.per > 1) {
        auto start = [&](auto position) {
            using Q = decltype(position);
            return logp_start(grad ? k_shared_grad<E, K, G, Q> : k_shared<E, K, G, Q>, p, s.rows_grid, s.rows_threads,
                              (sizeof(Q) * G * s.tours + (grad ? 256 * kWaves<G> : 0)) * K, stream);
        };
        if constexpr (G == 64 && K >= 12) {             // fewer entries a lane only hold shorter rows
            if (p.n > kHalfRow) return start(float());
        }
        return start(_Float16());
    }
    return logp_start(grad ? k_single_grad<E, K, G> : k_single<E, K, G>, p, s.rows_grid, s.rows_threads, 0, stream);
}

template <typename E>
int logp_launch(LogpParams p, const LogpShape& s, bool grad, hipStream_t stream)
{
    p.parts = s.parts;
    p.groups = s.groups;
    int rc = 0;
    if (p.n <= kShortRow) T2O_BY_HELD(s.k, (rc = logp_rows<E, K, 16>(p, s, grad, stream)))
    else T2O_BY_HELD(s.k, (rc = logp_rows<E, K < 6 ? 6 : K, 64>(p, s, grad, stream)))
    if (rc) return rc;
    if (!grad && p.parts > 1) {
        rc = logp_start(p.per > 1 ? k_join<E, true> : k_join<E, false>, p, s.join_grid, 256, 0, stream);
        if (rc) return rc;
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
    if (num_tours > 0x7fffffffll || !LogpShape(num_tours, n, by_step ? n - 1 : n, per).fits)
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
    if (num_tours > 0x7fffffffll) return fail(TSP2OPT_E_UNSUPPORTED, "too many tours");
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
    if (state_bytes < LogpState(num_tours, n, tours_per_map, rows).bytes)
        return fail(TSP2OPT_E_WORKSPACE, "state_bytes too small");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(TSP2OPT_E_HIP, "hipSetDevice failed");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    LogpParams p = logp_params(logits, tours, state, num_tours, n, tours_per_map, rows, map_stride, row_stride);
    p.logp = logp_out;
    const LogpShape shape(num_tours, n, p.rows, tours_per_map);
    if (tours_per_map == 1 || n > kShortRow) {          // otherwise k_shared makes them itself
        const size_t lds = 2 * (size_t)n;
        if (lds > 48 * 1024)
            HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(k_positions),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
        hipLaunchKernelGGL(k_positions, dim3((unsigned)num_tours), dim3(shape.position_threads), lds, stream, tours, p.pos,
                           p.next, logp_out, n);
    }
    int result = 0;
    T2O_BY_DTYPE(dtype, result = logp_launch<E>(p, shape, false, stream));
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
    if (state_bytes < LogpState(num_tours, n, tours_per_map, rows).bytes)
        return fail(TSP2OPT_E_WORKSPACE, "state_bytes too small");
    DeviceGuard guard(device);
    if (!guard.ok) return fail(TSP2OPT_E_HIP, "hipSetDevice failed");
    hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    LogpParams p = logp_params(logits, tours, const_cast<void*>(state), num_tours, n, tours_per_map, rows, map_stride,
                               row_stride);
    p.g = grad_logp;
    p.grad = grad_out;
    int result = 0;
    T2O_BY_DTYPE(dtype, result = logp_launch<E>(p, LogpShape(num_tours, n, p.rows, tours_per_map), true, stream));
    return result;
}
