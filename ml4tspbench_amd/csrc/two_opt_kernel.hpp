// ml4tspbench_amd/csrc/two_opt_kernel.hpp -- filter sweep, incremental sweeps, argmin selection, reversal, cluster exchange, k_two_opt
// Part of the single translation unit tsp2opt.hip (design notes at its top).
#pragma once

namespace t2o {

// ------------------------------------------------------------------------------------------
// filter sweep
// ------------------------------------------------------------------------------------------
// Window geometry of one lane group gp: stream A walks diagonals 2+8gp .. 5+8gp, stream B the next
// four, so the B operand of a column is the A operand 4 positions later = the .y half of the same
// LDS entry.  Rows advance 4 per macro step; two macro steps (row parities PAR = 0, 1 of an 8-row
// block rq) make one TILE of 8 rows x 8 diagonals = 64 pairs, the unit of the minimum cache.
//
// load_block<PAR>(b): per stream C[u] = P[8b + 4 PAR + 2 + u], E[u] = e[8b + 4 PAR + 1 + u]
template <int Q, int PAR>
__device__ __forceinline__ void load_block(const v2f* Xq, const v2f* Yq, const v2f* Eq, int b,
                                           v2f (&CX)[4], v2f (&CY)[4], v2f (&E)[4])
{
    if constexpr (PAR == 0) {
        CX[0] = Xq[2 * Q + b]; CX[1] = Xq[3 * Q + b]; CX[2] = Xq[4 * Q + b]; CX[3] = Xq[5 * Q + b];
        CY[0] = Yq[2 * Q + b]; CY[1] = Yq[3 * Q + b]; CY[2] = Yq[4 * Q + b]; CY[3] = Yq[5 * Q + b];
        E[0] = Eq[Q + b]; E[1] = Eq[2 * Q + b]; E[2] = Eq[3 * Q + b]; E[3] = Eq[4 * Q + b];
    } else {
        CX[0] = Xq[6 * Q + b]; CX[1] = Xq[7 * Q + b]; CX[2] = Xq[b + 1]; CX[3] = Xq[Q + b + 1];
        CY[0] = Yq[6 * Q + b]; CY[1] = Yq[7 * Q + b]; CY[2] = Yq[b + 1]; CY[3] = Yq[Q + b + 1];
        E[0] = Eq[5 * Q + b]; E[1] = Eq[6 * Q + b]; E[2] = Eq[7 * Q + b]; E[3] = Eq[b + 1];
    }
}

// One macro step: rows r0..r0+3, r0 = 8*rq + 4*PAR, x the lane's 2 x 4 diagonals, 32 pairs.
// cb = rq + gp.  Per stream, with c0 = r0 + 2 + 8*gp:
//   Cold[u] = P[c0+u], Cnew[u] = P[c0+4+u], Eold[u] = e[c0-1+u], Enew[u] = e[c0+3+u],
//   Dc[q] = D(r0, c0+q) on entry and D(r0+4, c0+4+q) on exit.
template <int Q, int PAR>
__device__ __forceinline__ float macro_step(const v2f* Xq, const v2f* Yq, const v2f* Eq,
                                            int rq, int cb,
                                            const v2f (&CXo)[4], const v2f (&CYo)[4], v2f (&CXn)[4],
                                            v2f (&CYn)[4], const v2f (&Eo)[4], v2f (&En)[4],
                                            v2f (&Dc)[4])
{
    load_block<Q, 1 - PAR>(Xq, Yq, Eq, cb + PAR, CXn, CYn, En);
    float rx[4], ry[4], er[4];
    if constexpr (PAR == 0) {
        rx[0] = Xq[Q + rq].x;     ry[0] = Yq[Q + rq].x;             // P[r0+1]
        rx[1] = Xq[2 * Q + rq].x; ry[1] = Yq[2 * Q + rq].x;
        rx[2] = Xq[3 * Q + rq].x; ry[2] = Yq[3 * Q + rq].x;
        rx[3] = Xq[4 * Q + rq].x; ry[3] = Yq[4 * Q + rq].x;         // P[r0+4]
        er[0] = Eq[rq].x;                                           // e[r0]
        er[1] = Eq[Q + rq].x;
        er[2] = Eq[2 * Q + rq].x;
        er[3] = Eq[3 * Q + rq].x;
    } else {
        rx[0] = Xq[5 * Q + rq].x; ry[0] = Yq[5 * Q + rq].x;
        rx[1] = Xq[6 * Q + rq].x; ry[1] = Yq[6 * Q + rq].x;
        rx[2] = Xq[7 * Q + rq].x; ry[2] = Yq[7 * Q + rq].x;
        rx[3] = Xq[rq + 1].x;     ry[3] = Yq[rq + 1].x;
        er[0] = Eq[4 * Q + rq].x;
        er[1] = Eq[5 * Q + rq].x;
        er[2] = Eq[6 * Q + rq].x;
        er[3] = Eq[7 * Q + rq].x;
    }
    float mm = INFINITY;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        v2f t[4], Dn[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int vp = a + q + 1;                   // column point c0 + vp
            Dn[q] = dist32x2(rx[a], ry[a], vp < 4 ? CXo[vp] : CXn[vp - 4],
                             vp < 4 ? CYo[vp] : CYn[vp - 4]);       // D(r0+a+1, c0+a+q+1)
            const int ve = a + q;                       // column edge c0 + ve
            t[q] = (Dc[q] + Dn[q]) - (ve < 3 ? Eo[ve + 1] : En[ve - 3]);
        }
        float m = __builtin_fminf(__builtin_fminf(t[0].x, t[0].y), t[1].x);
        m = __builtin_fminf(__builtin_fminf(m, t[1].y), t[2].x);
        m = __builtin_fminf(__builtin_fminf(m, t[2].y), t[3].x);
        m = __builtin_fminf(m, t[3].y) - er[a];
        mm = __builtin_fminf(mm, m);
#pragma unroll
        for (int q = 0; q < 4; ++q) Dc[q] = Dn[q];
    }
    return mm;
}

// The same with the row parity of the macro step in a register (Geo::half: units start at any macro row, so the
// lanes of a wave differ in parity).  Window position w sits in sub-array w & 7 at index w >> 3: moving 4
// positions on (par = 1) moves sub-arrays 0..3 to 4..7 (+4Q entries: oa) and 4..7 to 0..3 of the next index
// (+1 - 4Q entries: ob), so every operand keeps a compile-time offset from one of two lane bases.
template <int Q>
__device__ __forceinline__ void load_block_rt(const v2f* Xq, const v2f* Yq, const v2f* Eq, int b, int par,
                                              v2f (&CX)[4], v2f (&CY)[4], v2f (&E)[4])
{
    const int oa = b + par * (4 * Q), ob = b + par * (1 - 4 * Q);
    CX[0] = Xq[2 * Q + oa]; CX[1] = Xq[3 * Q + oa]; CX[2] = Xq[4 * Q + ob]; CX[3] = Xq[5 * Q + ob];
    CY[0] = Yq[2 * Q + oa]; CY[1] = Yq[3 * Q + oa]; CY[2] = Yq[4 * Q + ob]; CY[3] = Yq[5 * Q + ob];
    E[0] = Eq[Q + oa]; E[1] = Eq[2 * Q + oa]; E[2] = Eq[3 * Q + oa]; E[3] = Eq[4 * Q + ob];
}

template <int Q>
__device__ __forceinline__ float macro_step_rt(const v2f* Xq, const v2f* Yq, const v2f* Eq,
                                               int rq, int cb, int par,
                                               const v2f (&CXo)[4], const v2f (&CYo)[4], v2f (&CXn)[4],
                                               v2f (&CYn)[4], const v2f (&Eo)[4], v2f (&En)[4],
                                               v2f (&Dc)[4])
{
    load_block_rt<Q>(Xq, Yq, Eq, cb + par, 1 - par, CXn, CYn, En);
    const int oa = rq + par * (4 * Q), ob = rq + par * (1 - 4 * Q);
    float rx[4], ry[4], er[4];
    rx[0] = Xq[Q + oa].x;     ry[0] = Yq[Q + oa].x;             // P[r0+1], r0 = 8 rq + 4 par
    rx[1] = Xq[2 * Q + oa].x; ry[1] = Yq[2 * Q + oa].x;
    rx[2] = Xq[3 * Q + oa].x; ry[2] = Yq[3 * Q + oa].x;
    rx[3] = Xq[4 * Q + ob].x; ry[3] = Yq[4 * Q + ob].x;         // P[r0+4]
    er[0] = Eq[oa].x;                                           // e[r0]
    er[1] = Eq[Q + oa].x;
    er[2] = Eq[2 * Q + oa].x;
    er[3] = Eq[3 * Q + oa].x;
    float mm = INFINITY;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
        v2f t[4], Dn[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int vp = a + q + 1;
            Dn[q] = dist32x2(rx[a], ry[a], vp < 4 ? CXo[vp] : CXn[vp - 4],
                             vp < 4 ? CYo[vp] : CYn[vp - 4]);
            const int ve = a + q;
            t[q] = (Dc[q] + Dn[q]) - (ve < 3 ? Eo[ve + 1] : En[ve - 3]);
        }
        float m = __builtin_fminf(__builtin_fminf(t[0].x, t[0].y), t[1].x);
        m = __builtin_fminf(__builtin_fminf(m, t[1].y), t[2].x);
        m = __builtin_fminf(__builtin_fminf(m, t[2].y), t[3].x);
        m = __builtin_fminf(m, t[3].y) - er[a];
        mm = __builtin_fminf(mm, m);
#pragma unroll
        for (int q = 0; q < 4; ++q) Dc[q] = Dn[q];
    }
    return mm;
}

__device__ __forceinline__ void track(float mm, unsigned id, float& a1, float& a2, unsigned& chunk)
{
    a2 = __builtin_amdgcn_fmed3f(a1, mm, a2);   // runner-up (a1 <= a2 invariant)
    chunk = mm < a1 ? id : chunk;
    a1 = fminf(a1, mm);
}

// Tile ids: id = (rq << 8) | gpl, rq = 8-row block of the whole window (segment s of unit
// u = s * GPl + gpl covers rq = s*MS/2 .. (s+1)*MS/2 - 1), gpl = this workgroup's lane group (< 256,
// global lane group gp = wc + CS * gpl); the cached minimum of the tile sits at Mc[rq * GPl + gpl].
// Full sweep: every lane walks its own unit; the tile minima go to the cache when there is one.
template <int Q, bool CL>
__device__ __forceinline__ void filter_sweep(const v2f* Xq, const v2f* Yq, const v2f* Eq, float* Mc,
                                             const Geo& g, int tid, float& a1, float& a2,
                                             unsigned& chunk)
{
    a1 = INFINITY;
    a2 = INFINITY;
    chunk = 0;
    const int units = g.GPl * g.NS, MS2 = g.MS >> 1;
    if constexpr (!CL) {
        if (g.half) {       // (uniform) macro-step units: chunk id = (macro row << 8) | lane group
            for (int u = tid; u < units; u += g.nt) {
                const int s = div_gpl(g, u), gpl = u - s * g.GPl;
                const int m0 = s * g.MS;
                int par = m0 & 1, rq = m0 >> 1, cb = rq + gpl;
                v2f CX0[4], CY0[4], CX1[4], CY1[4], E0[4], E1[4], Dc[4];
                load_block_rt<Q>(Xq, Yq, Eq, cb, par, CX0, CY0, E0);
                const float ax = Xq[rq + par * (4 * Q)].x, ay = Yq[rq + par * (4 * Q)].x;      // P[r0]
#pragma unroll
                for (int q = 0; q < 4; ++q) Dc[q] = dist32x2(ax, ay, CX0[q], CY0[q]);
                unsigned id = ((unsigned)m0 << 8) | (unsigned)gpl;
                int k = 0;
                for (; k + 1 < g.MS; k += 2) {
                    float mm = macro_step_rt<Q>(Xq, Yq, Eq, rq, cb, par, CX0, CY0, CX1, CY1, E0, E1, Dc);
                    track(mm, id, a1, a2, chunk);
                    id += 256u; rq += par; cb += par; par ^= 1;
                    mm = macro_step_rt<Q>(Xq, Yq, Eq, rq, cb, par, CX1, CY1, CX0, CY0, E1, E0, Dc);
                    track(mm, id, a1, a2, chunk);
                    id += 256u; rq += par; cb += par; par ^= 1;
                }
                if (k < g.MS) {
                    const float mm = macro_step_rt<Q>(Xq, Yq, Eq, rq, cb, par, CX0, CY0, CX1, CY1, E0, E1, Dc);
                    track(mm, id, a1, a2, chunk);
                }
            }
            return;
        }
    }
    for (int u = tid; u < units; u += g.nt) {
        const int s = div_gpl(g, u), gpl = u - s * g.GPl;
        const int gp = CL ? g.wc + g.CS * gpl : gpl;
        if constexpr (CL) {
            if (gp >= g.GP) continue;                       // padding of the last workgroups
        }
        int rq = s * MS2;
        int cb = rq + gp;
        v2f CX0[4], CY0[4], CX1[4], CY1[4], E0[4], E1[4], Dc[4];
        load_block<Q, 0>(Xq, Yq, Eq, cb, CX0, CY0, E0);
        const float ax = Xq[rq].x, ay = Yq[rq].x;           // P[r0]
#pragma unroll
        for (int q = 0; q < 4; ++q) Dc[q] = dist32x2(ax, ay, CX0[q], CY0[q]);
        unsigned id = ((unsigned)rq << 8) | (unsigned)gpl;
        float* mc = Mc ? Mc + rq * g.GPl + gpl : nullptr;
        for (int m2 = 0; m2 < MS2; ++m2) {
            float mm = macro_step<Q, 0>(Xq, Yq, Eq, rq, cb, CX0, CY0, CX1, CY1, E0, E1, Dc);
            mm = __builtin_fminf(mm, macro_step<Q, 1>(Xq, Yq, Eq, rq, cb, CX1, CY1, CX0, CY0, E1, E0, Dc));
            if (mc) { *mc = mm; mc += g.GPl; }
            track(mm, id, a1, a2, chunk);
            ++rq; ++cb; id += 256u;
        }
    }
}

// filter minimum of one tile, from scratch (incremental sweeps)
template <int Q>
__device__ __forceinline__ float tile_min(const v2f* Xq, const v2f* Yq, const v2f* Eq, int rq, int gp)
{
    const int cb = rq + gp;
    v2f CX0[4], CY0[4], CX1[4], CY1[4], E0[4], E1[4], Dc[4];
    load_block<Q, 0>(Xq, Yq, Eq, cb, CX0, CY0, E0);
    const float ax = Xq[rq].x, ay = Yq[rq].x;
#pragma unroll
    for (int q = 0; q < 4; ++q) Dc[q] = dist32x2(ax, ay, CX0[q], CY0[q]);
    float mm = macro_step<Q, 0>(Xq, Yq, Eq, rq, cb, CX0, CY0, CX1, CY1, E0, E1, Dc);
    return __builtin_fminf(mm, macro_step<Q, 1>(Xq, Yq, Eq, rq, cb, CX1, CY1, CX0, CY0, E1, E0, Dc));
}

// bits [a, b] of a 64-bit mask, clipped to [0, M-1]
__device__ __forceinline__ unsigned long long bit_range(int a, int b, int M)
{
    a = a < 0 ? 0 : a;
    b = b > M - 1 ? M - 1 : b;
    if (a > b) return 0ull;
    return (~0ull >> (63 - b)) & (~0ull << a);
}

// bits [a, b] of a 32-bit mask, clipped to [0, M-1] (M <= 32)
__device__ __forceinline__ unsigned bit_range32(int a, int b, int M)
{
    a = a < 0 ? 0 : a;
    b = b > M - 1 ? M - 1 : b;
    if (a > b) return 0u;
    return (~0u >> (31 - b)) & (~0u << a);
}

struct Unit {               // the lane's own unit, fixed for the whole kernel
    int gp;                 // lane group (of the whole tour), or -1 when the lane owns no unit
    int gpl;                // its index among this workgroup's lane groups
    int rq0;                // first 8-row block of its row segment
};

// Recomputed where it is needed rather than carried through the iteration loop: the kernel sits at
// the VGPR limit and loop-carried registers are the ones that get spilled.
template <bool CL>
__device__ __forceinline__ Unit lane_unit(const Geo& g, int tid)
{
    Unit un{-1, 0, 0};
    if (tid >= 0 && tid < g.GPl * g.NS) {
        const int s = div_gpl(g, tid);
        un.gpl = tid - s * g.GPl;
        un.rq0 = s * (g.MS >> 1);
        const int gp = CL ? g.wc + g.CS * un.gpl : un.gpl;
        if (!CL || gp < g.GP) un.gp = gp;
    }
    return un;
}

// Filter sweep of one iteration for geometries WITHOUT the tile cache: every lane walks its whole unit.
template <int Q, bool CL, typename T>
__device__ __forceinline__ void sweep(const View<T>& v, const Geo& g, int tid,
                                      float& a1, float& a2, unsigned& chunk, Prof& pf)
{
    FINE_START(pf);
    __builtin_amdgcn_s_setprio(0);
    filter_sweep<Q, CL>(v.Xq, v.Yq, v.Eq, nullptr, g, tid, a1, a2, chunk);
    __builtin_amdgcn_s_setprio(3);
    FINE(pf, 3);                                            // full sweep
}

// ------------------------------------------------------------------------------------------
// cached path (g.inc): tile minima Mc + per-unit minima Mu, three barriers per iteration
// ------------------------------------------------------------------------------------------
// One iteration with the tile cache is three phases, each closed by ONE workgroup barrier:
//   A  apply the chosen reversal to the LDS copies AND mark the tiles it touches (closed form per
//      lane): the lane resets its unit's minimum Mu[u] to the minimum of its UNTOUCHED tiles and the
//      touched tile ids are compacted into a list;
//   B  the listed tiles are recomputed evenly by all lanes (or, on list overflow, every lane re-walks
//      its whole unit): Mc[tile] = value, Mu[unit] = min(Mu[unit], value) with an LDS atomic;
//   C  ONE wave (it rotates; in a cluster every wave, redundantly): scan Mu for the workgroup minimum m,
//      find the units and then the tiles inside the window m + 2 eps, re-evaluate those tiles pair by
//      pair in fp32 and decide (unique far-enough pair: certain move / window above the threshold:
//      converged / else the exact stage, cooperatively); the verdict reaches the other waves through LDS
//      at the phase's barrier (select_cached).
// Mu holds order-preserving unsigned keys of the float minima so that ds_min_u32 can merge them.
__device__ __forceinline__ unsigned fkey(float f)
{
    const unsigned b = __float_as_uint(f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float funkey(unsigned k)
{
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// full sweep of the lane's own unit: every tile minimum to Mc, the unit minimum to Mu
template <int Q, bool CL, typename T>
__device__ __forceinline__ void filter_sweep_cached(const View<T>& v, const Geo& g, int tid)
{
    tid -= g.u0;                                        // the lane's unit number
    const Unit un = lane_unit<CL>(g, tid);
    if (un.gp < 0) return;
    const int MS2 = g.MS >> 1;
    int rq = un.rq0;
    int cb = rq + un.gp;
    v2f CX0[4], CY0[4], CX1[4], CY1[4], E0[4], E1[4], Dc[4];
    load_block<Q, 0>(v.Xq, v.Yq, v.Eq, cb, CX0, CY0, E0);
    const float ax = v.Xq[rq].x, ay = v.Yq[rq].x;           // P[r0]
#pragma unroll
    for (int q = 0; q < 4; ++q) Dc[q] = dist32x2(ax, ay, CX0[q], CY0[q]);
    unsigned* mc = v.Mc + rq * g.GPl + un.gpl;
    float um = INFINITY;
    for (int m2 = 0; m2 < MS2; ++m2) {
        float mm = macro_step<Q, 0>(v.Xq, v.Yq, v.Eq, rq, cb, CX0, CY0, CX1, CY1, E0, E1, Dc);
        mm = __builtin_fminf(mm, macro_step<Q, 1>(v.Xq, v.Yq, v.Eq, rq, cb, CX1, CY1, CX0, CY0, E1, E0, Dc));
        *mc = fkey(mm);
        mc += g.GPl;
        um = __builtin_fminf(um, mm);
        ++rq; ++cb;
    }
    v.Mu[tid] = fkey(um);
}

// phase A, second half: mark the tiles the reversal of LDS positions lo0 .. lo0 + len - 1 (mod n) touches
// (those coordinates and the edges lo0 - 1 .. lo0 + len - 1, in every cyclic copy of the window), reset the
// unit minimum to its untouched tiles, queue the touched tile ids
template <bool CL, typename T>
__device__ __forceinline__ void mark_touched(const View<T>& v, const Geo& g, int tid, int lo0, int len)
{
    const int ut = tid - g.u0;                          // the lane's unit number
    const Unit un = lane_unit<CL>(g, ut);
    const int MS2 = g.MS >> 1;
    int i = lo0 - 1, j = lo0 + len - 1;                 // window positions [i, j] (+ k n) read changed values
    if (j >= g.n) { i -= g.n; j -= g.n; }               // (uniform) the earliest copy that reaches the window
    unsigned mask = 0u;                                 // touched tiles of the lane's unit (MS2 <= 32)
    if (un.gp >= 0) {
        // (two to four copies.  The counter is opaque to the compiler, which otherwise computes the trip count up front:
        //  a division by n through a reciprocal that it keeps in scratch memory -- a scratch load per iteration)
        for (int lo = i, hi = j; lo < g.W; lo += g.n, hi += g.n) {
            asm volatile("" : "+v"(lo));
            mask |= bit_range32((lo >> 3) - un.rq0, (hi >> 3) - un.rq0, MS2);                              // rows
            mask |= bit_range32(((lo - 9) >> 3) - un.gp - un.rq0, ((hi - 2) >> 3) - un.gp - un.rq0, MS2);  // columns
        }
    }
    if (mask) {
        // minimum of the unit's UNTOUCHED tiles; eight cached minima per LDS round trip (a plain loop
        // would wait for every single read)
        const unsigned* mc = v.Mc + un.rq0 * g.GPl + un.gpl;
        const unsigned skip = MS2 >= 32 ? mask : (mask | (~0u << MS2));     // touched, or beyond the unit
        unsigned km = 0xffffffffu;
        for (int m0 = 0; m0 < MS2; m0 += 8) {
            unsigned c[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int m2 = m0 + k < MS2 ? m0 + k : MS2 - 1;             // always a valid address
                c[k] = mc[m2 * g.GPl];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) km = ((skip >> (m0 + k)) & 1u) ? km : (c[k] < km ? c[k] : km);
        }
        v.Mu[ut] = km;
    }
    // compaction: prefix sum of the lanes' counts -> one atomic per wave -> every lane writes its run
    const unsigned cnt = (unsigned)__popc(mask);
    const unsigned incl = wave_scan_add(cnt);
    const unsigned wtotal = (unsigned)__builtin_amdgcn_readlane((int)incl, 63);
    if (wtotal) {
        unsigned base = 0;
        if ((tid & 63) == 0) base = atomicAdd(&v.ctl->nlist, wtotal);
        unsigned pos = (unsigned)__builtin_amdgcn_readfirstlane((int)base) + incl - cnt;
        const unsigned id0 = ((unsigned)un.rq0 << 8) | (unsigned)un.gpl;
        while (mask) {
            const unsigned b = (unsigned)__builtin_ctz(mask);
            mask &= mask - 1u;
            if (pos < (unsigned)g.lcap) v.list[pos] = (uint16_t)(id0 + (b << 8));
            ++pos;
        }
    }
}

// Filter value of the reference pair (0, n-1): cyclically adjacent edges, on no walked diagonal.  Its operands
// are R[0], R[1], R[n-1] and the edges between them, wherever the frame has put them.
template <int Q, typename T>
__device__ __forceinline__ float special_pair_filter(const View<T>& v, int n)
{
    const int p0 = v.fo, p1 = wrapn(v.fo + v.fs, n), pm = wrapn(v.fo - v.fs, n);
    const int e0 = v.fs > 0 ? p0 : p1, em = v.fs > 0 ? pm : p0;         // LDS edges (R0,R1) and (R[n-1],R0)
    const int s0 = slot<Q>(p0), s1 = slot<Q>(p1), sm = slot<Q>(pm);
    const float x0 = v.Xq[s0].x, y0 = v.Yq[s0].x;
    const float d0 = dist32(x0, y0, v.Xq[sm].x, v.Yq[sm].x);
    const float d1 = dist32(v.Xq[s1].x, v.Yq[s1].x, x0, y0);
    return ((d0 + d1) - v.Eq[slot<Q>(em)].x) - v.Eq[slot<Q>(e0)].x;
}

// phase B: bring Mc / Mu up to date after reversal `last` (kFullSweep: everything)
template <int Q, bool CL, typename T>
__device__ __forceinline__ void refresh_cached(const View<T>& v, const Geo& g, int tid, unsigned last, Prof& pf)
{
    Ctl* ctl = v.ctl;
    FINE_START_G(pf, 0x000e);
    const unsigned nl = ctl->nlist;
    // (the lane's first list entry is read before nl is known -- one LDS round trip instead of two on the chain;
    //  whatever an unused slot holds is never looked at)
    __builtin_amdgcn_s_setprio(0);
    if (last == kFullSweep || nl > (unsigned)g.lcap) {      // (uniform) first sweep, or most of the tour moved
        filter_sweep_cached<Q, CL>(v, g, tid);
        FINE(pf, 3);
    } else {
        const float inv_ms2 = 1.0f / (float)(g.MS >> 1);
        unsigned id_next = (unsigned)tid < nl ? v.list[tid] : 0u;
        for (unsigned t = (unsigned)tid; t < nl; t += (unsigned)g.nt) {
            const unsigned id = id_next;
            if (t + (unsigned)g.nt < nl) id_next = v.list[t + (unsigned)g.nt];     // in flight during tile_min
            const int rq = (int)(id >> 8), gpl = (int)(id & 255u);
            const float val = tile_min<Q>(v.Xq, v.Yq, v.Eq, rq, g.wc + g.CS * gpl);
            const unsigned kv = fkey(val);
            v.Mc[rq * g.GPl + gpl] = kv;
            const int seg = (int)(((float)rq + 0.5f) * inv_ms2);         // rq / MS2 (exact: rq <= 255, MS2 <= 32)
            atomicMin(&v.Mu[seg * g.GPl + gpl], kv);
        }
        FINE(pf, 1);
    }
    __builtin_amdgcn_s_setprio(3);
    if (tid == 0) {     // the pair (0, n-1): cyclically adjacent, not on any walked diagonal
        const int n = g.n;
        // (its operands R[1], R[n-1] and the two edges change only when the reversal starts at reference
        //  position 1 or ends at n-1, whatever the frame)
        if (last == kFullSweep || (last >> 16) == 0u || (last & 0xffffu) == (unsigned)(n - 1))
            ctl->spd = special_pair_filter<Q>(v, n);
    }
}

// window position -> tour position; window positions are below 3n (make_plan guarantees W < 3n)
__device__ __forceinline__ int wrap3(int w, int n)
{
    w -= w >= n ? n : 0;
    w -= w >= n ? n : 0;
    return w;
}

// window positions (row, column) of pair `pr` (0..63: row 0..7, diagonal 0..7) of tile `id`
// (Geo::half: the chunk is a macro step, id >> 8 its macro row: pairs 0..31; pairs 32..63 are the next macro
//  step's, valid pairs of the window too, which the callers leave out)
__device__ __forceinline__ void tile_pair(const Geo& g, unsigned id, int pr, int& rw, int& cw)
{
    rw = (g.half ? 4 : 8) * (int)(id >> 8) + (pr >> 3);
    cw = rw + 2 + 8 * (g.wc + g.CS * (int)(id & 255u)) + (pr & 7);
}

// Reference index (two_opt.py:37-38: i, j of the flat argmin) of the pair of LDS edges r and c (edge q joins
// LDS positions q and q + 1): LDS position p is reference position fs * (p - fo) mod n, and with fs = -1 the
// edge's first reference position is that of its SECOND LDS position.  Returns packed (i << 16 | j), i < j.
template <typename T>
__device__ __forceinline__ unsigned pair_index(const View<T>& v, int n, int r, int c)
{
    const int er = v.fs > 0 ? wrapn(r - v.fo, n) : wrapn(v.fo - 1 - r, n);
    const int ec = v.fs > 0 ? wrapn(c - v.fo, n) : wrapn(v.fo - 1 - c, n);
    const int i = er < ec ? er : ec, j = er < ec ? ec : er;
    return ((unsigned)i << 16) | (unsigned)j;
}

// exact value of pair `pr` of tile `id`; returns packed index
template <typename T>
__device__ __forceinline__ void eval_chunk_pair(const View<T>& v, const Geo& g, unsigned id, int pr,
                                                double& e, unsigned& idx)
{
    int rw, cw;
    tile_pair(g, id, pr, rw, cw);
    idx = pair_index(v, g.n, wrap3(rw, g.n), wrap3(cw, g.n));
    e = exact_delta(v, g.n, (int)(idx >> 16), (int)(idx & 0xffffu));
}

// fp32 (filter) value of pair `pr` of tile `id`, recomputed from the LDS window exactly as the
// sweep computes it, with the pair's packed index
template <int Q, typename T>
__device__ __forceinline__ void filter_chunk_pair(const View<T>& v, const Geo& g, unsigned id, int pr,
                                                  float& d, unsigned& idx)
{
    int rw, cw;
    tile_pair(g, id, pr, rw, cw);
    const int sr = slot<Q>(rw), sr1 = slot<Q>(rw + 1), sc = slot<Q>(cw), sc1 = slot<Q>(cw + 1);
    const float d0 = dist32(v.Xq[sr].x, v.Yq[sr].x, v.Xq[sc].x, v.Yq[sc].x);
    const float d1 = dist32(v.Xq[sr1].x, v.Yq[sr1].x, v.Xq[sc1].x, v.Yq[sc1].x);
    d = ((d0 + d1) - v.Eq[sc].x) - v.Eq[sr].x;
    idx = pair_index(v, g.n, wrap3(rw, g.n), wrap3(cw, g.n));
}

// filter_chunk_pair with every LDS read issued before the first use (one round trip instead of six)
template <int Q, typename T>
__device__ __forceinline__ void filter_chunk_pair_b(const View<T>& v, const Geo& g, unsigned id, int pr,
                                                    float& d, unsigned& idx)
{
    int rw, cw;
    tile_pair(g, id, pr, rw, cw);
    const int sr = slot<Q>(rw), sr1 = slot<Q>(rw + 1), sc = slot<Q>(cw), sc1 = slot<Q>(cw + 1);
    const float xr = v.Xq[sr].x, yr = v.Yq[sr].x, xc = v.Xq[sc].x, yc = v.Yq[sc].x;
    const float xr1 = v.Xq[sr1].x, yr1 = v.Yq[sr1].x, xc1 = v.Xq[sc1].x, yc1 = v.Yq[sc1].x;
    const float ec = v.Eq[sc].x, er = v.Eq[sr].x;
    asm volatile("" ::"v"(xr), "v"(yr), "v"(xc), "v"(yc), "v"(xr1), "v"(yr1), "v"(xc1), "v"(yc1), "v"(ec), "v"(er));
    const float d0 = dist32(xr, yr, xc, yc);
    const float d1 = dist32(xr1, yr1, xc1, yc1);
    d = ((d0 + d1) - ec) - er;
    idx = pair_index(v, g.n, wrap3(rw, g.n), wrap3(cw, g.n));
}

// The margin of the fp32 decisions (eps2 = 2 eps; 25 % extra), recomputed WHERE IT IS USED: left alone the compiler
// hoists the loop-invariant product (and its double) out of the improvement loop and, the kernel being at its
// register limit, keeps them in scratch memory -- two scratch loads on every iteration's decision chain.
__device__ __forceinline__ float decision_eps(const Geo& g)
{
    float e2 = g.eps2;
    asm volatile("" : "+v"(e2));
    return 0.625f * e2;
}

// One full argmin (the reference's per-tour torch.min / torch.argmin, two_opt.py:35-38) for geometries
// WITHOUT the tile cache (tiny tours with one tile per lane; N where the cache does not fit) and the
// exact-only kernel (Q = 0); select_cached below is the same decision on top of the cache.
// Returns in every thread: e = min(0, min valid delta), idx = packed (i,j) or kNoMove.
// `need_exact_sign`: the caller needs the exact sign of a non-improving minimum (coupled-mode
// continuation); otherwise a minimum proven >= -1e-6 by the filter alone ends the search.
// CL (several workgroups per tour): this workgroup's tiles only, always exact (the result is compared
// with the other workgroups' results), no fp32-only shortcut.
// ctl->spd (thread 0 only): cached filter value of the pair (0, n-1); its operands P[1], P[n-1], e[0],
// e[n-1] change only when the last reversal started at position 1 or ended at position n-1.  (In
// LDS, not in a register: the kernel sits at the VGPR limit and loop-carried registers get spilled.)
template <typename T, int Q, bool CL>
__device__ void find_best(const View<T>& v, const Geo& g, int tid, bool need_exact_sign,
                          unsigned last, double& e, unsigned& idx, Prof& pf)
{
    Ctl* ctl = v.ctl;
    unsigned long long t0 = 0;
    if (pf.on) t0 = clock64();
    if constexpr (Q == 0) {
        exact_sweep(v, g.n, tid, g.nt, e, idx);
        block_best(ctl, tid, g.nt, e, idx);
        return;
    } else {
        float a1, a2;
        unsigned chunk;
        // everything outside the sweep arithmetic is a latency chain that idles most of the
        // workgroup: it runs at high issue priority (set inside sweep()) so that the other
        // workgroups' sweeps on this SIMD do not stretch it
        sweep<Q, CL>(v, g, tid, a1, a2, chunk, pf);
        if (pf.on) { const unsigned long long t1 = clock64(); pf.sweep += t1 - t0; t0 = t1; }
        const int nw = g.nt >> 6, lane = tid & 63, wv = tid >> 6;
        const float wm = wave_min_ordered(a1);       // (filter values are never NaN: scaled coordinates are finite)
        float m = wm;
        if (nw > 1) {                                       // one-wave workgroups need no LDS round trip
            if (lane == 0) ctl->wmin[wv] = wm;
            __syncthreads();
            m = ctl->wmin[0];
            for (int w = 1; w < nw; ++w) m = fminf(m, ctl->wmin[w]);
        }
        float thr = m + g.eps2;
        if constexpr (CL) {
            // This workgroup sees only its own tiles, whose minimum may be far above the tour's.  Only
            // moves below -1e-6 are ever applied (independent termination), so pairs whose filter value
            // proves delta >= -1e-6 need no exact evaluation: without this clamp a workgroup whose tiles
            // hold no improving move would chase near-ties among its non-improving minima.
            thr = fminf(thr, -ctl->tsc + decision_eps(g));
        }
        const unsigned long long cmask0 = __ballot(a1 <= thr);
        int amb = __ballot(a2 <= thr) != 0ull || __popcll(cmask0) > 8;
        FINE(pf, 4);                                        // workgroup minimum of the filter

        if constexpr (CL) {
            if (lane == 0) ctl->pAmb[wv] = amb;
            __syncthreads();
            int fl = 0;
            for (int w = 0; w < nw; ++w) fl |= ctl->pAmb[w];
            amb = fl & 1;
        } else {
            // ---- stage 1, fp32 only.  Every pair whose exact delta can be the argmin has a filter
            // value <= m + 2 eps and sits in a candidate macro step.  Re-evaluate those steps pair by
            // pair (lanes 0..31) in fp32: if exactly ONE pair of the whole tour is inside the window it
            // IS the reference's argmin, and if its value is below -1e-6 by more than eps the move is
            // certain without any exact arithmetic.  Likewise a window that lies above -1e-6 + eps
            // proves convergence.  Anything else falls through to the exact stage.
            const float thr_scale = ctl->tsc;
            float fd = INFINITY;
            unsigned fidx = 0xffffffffu;
            bool multi = false;
            if (!amb) {
                unsigned long long cm = cmask0;
                while (cm) {
                    const int src = __builtin_amdgcn_readfirstlane(__ffsll((long long)cm) - 1);
                    cm &= cm - 1;
                    const unsigned id = (unsigned)__builtin_amdgcn_readlane((int)chunk, src);
                    float d;
                    unsigned di;
                    filter_chunk_pair_b<Q>(v, g, id, lane, d, di);
                    if (g.half && lane >= 32) d = INFINITY;         // a macro step has 32 pairs
                    if (d <= thr) {
                        multi = multi || (fidx != 0xffffffffu && fidx != di);
                        if (d < fd || (d == fd && di < fidx)) { fd = d; fidx = di; }
                    }
                }
                if (tid == 0) {     // the pair (0, n-1): cyclically adjacent, not on any walked diagonal
                    const int n = g.n;
                    if (last == kFullSweep || (last >> 16) == 0u || (last & 0xffffu) == (unsigned)(n - 1))
                        ctl->spd = special_pair_filter<Q>(v, n);
                    const float d = ctl->spd;
                    const unsigned di = (unsigned)(n - 1);
                    if (d <= thr) {
                        multi = multi || (fidx != 0xffffffffu && fidx != di);
                        if (d < fd || (d == fd && di < fidx)) { fd = d; fidx = di; }
                    }
                }
            }
            FINE(pf, 5);                                    // fp32 re-evaluation of the candidate tiles
            // wave result: the minimum value and, when every in-window pair of the wave is the same
            // pair, that pair (otherwise the index is not used: `wother` sends the search to stage 2)
            const unsigned long long hm = __ballot(fidx != 0xffffffffu);
            double wd = (double)wave_min_ordered(fd);
            unsigned widx = 0xffffffffu;
            if (hm) widx = (unsigned)__builtin_amdgcn_readlane((int)fidx, __ffsll((long long)hm) - 1);
            const bool wother = __ballot(multi || (fidx != 0xffffffffu && fidx != widx)) != 0ull;
            double bd = wd;
            unsigned bi = widx;
            int fl = amb | (wother ? 2 : 0);
            bool unique = true;
            if (nw > 1) {
                if (lane == 0) {
                    ctl->pE[wv] = wd;
                    ctl->pIdx[wv] = widx;
                    ctl->pAmb[wv] = fl;
                }
                __syncthreads();
                bd = ctl->pE[0];
                bi = ctl->pIdx[0];
                fl = ctl->pAmb[0];
            }
            for (int w = 1; w < nw; ++w) {
                const double od = ctl->pE[w];
                const unsigned oi = ctl->pIdx[w];
                fl |= ctl->pAmb[w];
                if (oi != 0xffffffffu && bi != 0xffffffffu && oi != bi) unique = false;
                if (better(od, oi, bd, bi)) { bd = od; bi = oi; }
            }
            amb = fl & 1;
            unique = unique && !(fl & 2) && bi != 0xffffffffu;
            FINE(pf, 6);                                    // wave + workgroup reduction of the fp32 stage
            if (!amb) {
                const float eps = decision_eps(g);
                if (unique && (float)bd < -thr_scale - eps) {           // certain improving move
                    e = ((double)(float)bd + (double)eps) * ctl->isc;   // an upper bound, < -1e-6
                    idx = bi;
                    if (pf.on) pf.select += clock64() - t0;
                    return;
                }
                if (!need_exact_sign && m > -thr_scale + eps && (bi == 0xffffffffu || (float)bd > -thr_scale + eps)) {
                    e = 0.0;                                            // proven: no delta below -1e-6
                    idx = kNoMove;
                    if (pf.on) pf.select += clock64() - t0;
                    return;
                }
            }
        }
        __syncthreads();        // partials are rewritten below
        if (pf.on) { pf.cands += 1; pf.amb += amb ? 1 : 0; }

        // ---- stage 2, exact: each wave re-evaluates its candidate macro steps in the reference's
        // dtype and operation order (lanes 0..31 = the 32 pairs)
        e = 0.0;
        idx = kNoMove;
        if (!amb) {
            unsigned long long cm = cmask0;
            while (cm) {
                const int src = __builtin_amdgcn_readfirstlane(__ffsll((long long)cm) - 1);
                cm &= cm - 1;
                const unsigned id = (unsigned)__builtin_amdgcn_readlane((int)chunk, src);
                double d;
                unsigned di;
                eval_chunk_pair(v, g, id, lane, d, di);
                if (!(g.half && lane >= 32) && better(d, di, e, idx)) { e = d; idx = di; }
            }
            if (tid == 0) {
                const double d = exact_delta(v, g.n, 0, g.n - 1);
                if (better(d, (unsigned)(g.n - 1), e, idx)) { e = d; idx = (unsigned)(g.n - 1); }
            }
            wave_best(e, idx);
        }
        if (lane == 0) { ctl->pE[wv] = e; ctl->pIdx[wv] = idx; }
        __syncthreads();
        e = ctl->pE[0];
        idx = ctl->pIdx[0];
        for (int w = 1; w < nw; ++w) {
            const double oe = ctl->pE[w];
            const unsigned oi = ctl->pIdx[w];
            if (better(oe, oi, e, idx)) { e = oe; idx = oi; }
        }
        if (amb) {
            // A lane holds two tiles inside the window (or a wave more than 8 candidates): the per-lane
            // best/runner-up no longer names every candidate and there is no tile cache to list them
            // from: the whole tour is swept exactly.
            __syncthreads();
            exact_sweep(v, g.n, tid, g.nt, e, idx);
            block_best(ctl, tid, g.nt, e, idx);
        }
        FINE(pf, 7);                                        // exact stage
        if (pf.on) pf.select += clock64() - t0;
    }
}

// The unit minima of this workgroup, held by a wave: lane l keeps units 256c + 4l .. 256c + 4l + 3 of
// chunk c (one 16-byte LDS read per chunk; Mu is padded to a multiple of 4 with "+inf" keys).
struct UnitMinima {
    uint4 k[4];             // up to 1024 units
    int nch;
};

template <typename T>
__device__ __forceinline__ UnitMinima load_unit_minima(const View<T>& v, const Geo& g, int lane)
{
    UnitMinima um;
    const int units = g.GPl * g.NS;
    um.nch = (units + 255) >> 8;
    const uint4 inf = make_uint4(0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        um.k[c] = inf;
        if (c < um.nch && 256 * c + 4 * lane < units)
            um.k[c] = *reinterpret_cast<const uint4*>(v.Mu + 256 * c + 4 * lane);
    }
    return um;
}

__device__ __forceinline__ unsigned unit_minimum(const UnitMinima& um)
{
    unsigned km = 0xffffffffu;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (c < um.nch) {
            const unsigned a = um.k[c].x < um.k[c].y ? um.k[c].x : um.k[c].y;
            const unsigned b = um.k[c].z < um.k[c].w ? um.k[c].z : um.k[c].w;
            const unsigned m = a < b ? a : b;
            km = m < km ? m : km;
        }
    }
    return wave_min_u32(km);
}

// Visit every tile of this workgroup whose cached minimum is <= thr: a wave-uniform loop, f(id) runs
// with all 64 lanes.  Returns the number of tiles visited, or -1 as soon as more than max_tiles are
// inside the window (heavy ties; the caller falls back to the cooperative listing).
template <typename T, typename F>
__device__ __forceinline__ int for_each_candidate_tile(const View<T>& v, const Geo& g, int lane, float thr,
                                                       const UnitMinima& um, int max_tiles, F&& f)
{
    const int MS2 = g.MS >> 1;
    const unsigned kthr = fkey(thr);
    int count = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (c >= um.nch) break;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned key = k == 0 ? um.k[c].x : k == 1 ? um.k[c].y : k == 2 ? um.k[c].z : um.k[c].w;
            unsigned long long ub = __ballot(key <= kthr);
            while (ub) {
                const int u = 256 * c + 4 * __builtin_amdgcn_readfirstlane(__ffsll((long long)ub) - 1) + k;
                ub &= ub - 1;
                const int s = div_gpl(g, u), gpl = u - s * g.GPl;
                const int rq0 = s * MS2;
                const unsigned cm = v.Mc[(rq0 + (lane < MS2 ? lane : MS2 - 1)) * g.GPl + gpl];
                unsigned long long tb = __ballot(lane < MS2 && cm <= kthr);
                while (tb) {
                    const int m2 = __builtin_amdgcn_readfirstlane(__ffsll((long long)tb) - 1);
                    tb &= tb - 1;
                    if (count >= max_tiles) return -1;
                    ++count;
                    f(((unsigned)(rq0 + m2) << 8) | (unsigned)gpl);
                }
            }
        }
    }
    return count;
}

constexpr int kStage1Tiles = 8;     // more candidate tiles than this: heavy ties, cooperative path

// window of the filter values that can hold the argmin, from the unit minima (every lane of a wave)
template <bool CL>
__device__ __forceinline__ float window_threshold(const UnitMinima& um, const Geo& g, float thr_scale, float& m)
{
    m = funkey(unit_minimum(um));
    float thr = m + g.eps2;
    // CL: this workgroup sees only its own tiles, whose minimum may be far above the tour's.  Only moves
    // below -1e-6 are ever applied (independent termination), so pairs whose filter value proves
    // delta >= -1e-6 need no exact evaluation.
    if constexpr (CL) thr = fminf(thr, -thr_scale + decision_eps(g));
    return thr;
}

// Phase C of the cached path: the argmin decision from Mu / Mc / the window (see the header of this
// section).  One workgroup per tour: ONE wave (rotating with `round`) decides and posts the result in
// LDS; the barrier that follows both publishes it and marks the end of all reads of the window, so
// the reversal may start right after it.  CL: every wave decides redundantly (clusters run at low
// occupancy, the redundancy is free) and the cluster exchange's barrier plays that role.
// Same contract as find_best: in every thread e = min(0, min valid delta) (or a certified upper bound
// below -1e-6 for a certain move), idx = packed (i,j) or kNoMove.  CL: this workgroup's tiles only,
// always exact (the result is compared across workgroups).
template <typename T, int Q, bool CL>
__device__ void select_cached(const View<T>& v, const Geo& g, int tid, bool need_exact_sign, int turn,
                              double& e, unsigned& idx, Prof& pf)
{
    Ctl* ctl = v.ctl;
    const int nw = g.nt >> 6, lane = tid & 63, wv = tid >> 6;
    const bool mine = CL || nw == 1 || wv == turn;      // turn = iteration mod waves (kept by the caller: no division)
    int code = 0;                                       // 0: (e, idx) final, 1: exact stage, 2: heavy ties
    e = 0.0;
    idx = kNoMove;
    FINE_START_G(pf, 0x02f0);
    if (mine) {
        const UnitMinima um = load_unit_minima(v, g, lane);     // one LDS round trip together with sc / spd
        const double iscale = ctl->isc;
        const float spd = ctl->spd;
        const float thr_scale = ctl->tsc;
        float m;
        const float thr = window_threshold<CL>(um, g, thr_scale, m);
        FINE(pf, 4);                                    // workgroup minimum of the filter
        if constexpr (CL) {
            const int nct = for_each_candidate_tile(v, g, lane, thr, um, kStage1Tiles, [&](unsigned id) {
                double d;
                unsigned di;
                eval_chunk_pair(v, g, id, lane, d, di);
                if (better(d, di, e, idx)) { e = d; idx = di; }
            });
            if (nct >= 0) {
                // the pair (0, n-1): its filter value gates the exact evaluation exactly like a tile's minimum
                if (spd <= thr) {                       // (uniform)
                    const double d = exact_delta(v, g.n, 0, g.n - 1);
                    if (better(d, (unsigned)(g.n - 1), e, idx)) { e = d; idx = (unsigned)(g.n - 1); }
                }
                wave_best(e, idx);
            } else {
                code = 2;
            }
        } else {
            // ---- stage 1, fp32 only.  Every pair whose exact delta can be the argmin has a filter value
            // <= m + 2 eps and sits in a tile whose cached minimum is inside that window.  Re-evaluate those
            // tiles pair by pair in fp32 (lane = pair): if exactly ONE pair of the whole tour is inside the
            // window it IS the reference's argmin, and if its value is below -1e-6 by more than eps the move
            // is certain without any exact arithmetic.  Likewise a window that lies above -1e-6 + eps proves
            // convergence.  Anything else goes to the exact stage.
            //
            // Fast path, straight-line (the usual case once the tour is nearly converged, where this serial
            // chain of one wave IS the iteration's critical path): exactly one unit, one tile of it and one
            // pair of that tile inside the window.  Same decision as the general code below for that case.
            bool fast = false;
#ifndef TSP2OPT_NO_FASTC
            {
                const unsigned kthr = fkey(thr);
                // (per-lane counters under wave-uniform chunk guards: three VALU instructions a key)
                int cnt = 0, first = 0;
#pragma unroll
                for (int c = 3; c >= 0; --c) {
                    if (c < um.nch) {                                   // (uniform)
#pragma unroll
                        for (int k = 3; k >= 0; --k) {
                            const unsigned key = k == 0 ? um.k[c].x : k == 1 ? um.k[c].y : k == 2 ? um.k[c].z : um.k[c].w;
                            const bool hit = key <= kthr;
                            cnt += hit ? 1 : 0;
                            first = hit ? 4 * c + k : first;
                        }
                    }
                }
                const unsigned long long ub = __ballot(cnt != 0);
                int c1 = 0, u = 0;
                if (__popcll(ub) == 1) {
                    const int src = __ffsll((long long)ub) - 1;
                    const int f1 = __builtin_amdgcn_readlane(first, src);
                    c1 = __builtin_amdgcn_readlane(cnt, src);
                    u = 256 * (f1 >> 2) + 4 * src + (f1 & 3);
                }
                {
                    if (c1 == 1) {
                        const int MS2 = g.MS >> 1;
                        const int s = div_gpl(g, u), gpl = u - s * g.GPl;
                        const int rq0 = s * MS2;
                        const unsigned cm = v.Mc[(rq0 + (lane < MS2 ? lane : MS2 - 1)) * g.GPl + gpl];
                        const unsigned long long tb = __ballot(lane < MS2 && cm <= kthr);
                        if (__popcll(tb) == 1) {
                            const int m2 = __ffsll((long long)tb) - 1;
                            float d;
                            unsigned di;
                            filter_chunk_pair_b<Q>(v, g, ((unsigned)(rq0 + m2) << 8) | (unsigned)gpl, lane, d, di);
                            const bool sp = spd <= thr;                 // the pair (0, n-1), (uniform)
                            const unsigned long long wb = __ballot(d <= thr);
                            if (__popcll(wb) + (sp ? 1 : 0) == 1) {
                                FINE(pf, 5);
                                float wd = spd;
                                unsigned widx = (unsigned)(g.n - 1);
                                if (!sp) {
                                    const int wl = __ffsll((long long)wb) - 1;
                                    wd = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, d), wl));
                                    widx = (unsigned)__builtin_amdgcn_readlane((int)di, wl);
                                }
                                code = 1;
                                const float eps = decision_eps(g);
                                if (wd < -thr_scale - eps) {                            // certain improving move
                                    e = ((double)wd + (double)eps) * iscale;
                                    idx = widx;
                                    code = 0;
                                } else if (!need_exact_sign && m > -thr_scale + eps && wd > -thr_scale + eps) {
                                    e = 0.0;
                                    idx = kNoMove;
                                    code = 0;
                                }
                                FINE(pf, 6);
                                fast = true;
                            }
                        }
                    }
                }
            }
#endif
            if (!fast) {
            float fd = INFINITY;
            unsigned fidx = 0xffffffffu;
            bool multi = false;
            const int nct = for_each_candidate_tile(v, g, lane, thr, um, kStage1Tiles, [&](unsigned id) {
                float d;
                unsigned di;
                filter_chunk_pair_b<Q>(v, g, id, lane, d, di);
                if (d <= thr) {
                    multi = multi || (fidx != 0xffffffffu && fidx != di);
                    if (d < fd || (d == fd && di < fidx)) { fd = d; fidx = di; }
                }
            });
            if (nct < 0) {
                code = 2;
            } else {
                if (lane == 0) {
                    const unsigned di = (unsigned)(g.n - 1);
                    if (spd <= thr) {
                        multi = multi || (fidx != 0xffffffffu && fidx != di);
                        if (spd < fd || (spd == fd && di < fidx)) { fd = spd; fidx = di; }
                    }
                }
                FINE(pf, 5);                            // fp32 re-evaluation of the candidate tiles
                const unsigned long long hm = __ballot(fidx != 0xffffffffu);
                const float wd = wave_min_ordered(fd);
                unsigned widx = 0xffffffffu;
                if (hm) widx = (unsigned)__builtin_amdgcn_readlane((int)fidx, __ffsll((long long)hm) - 1);
                const bool wother = __ballot(multi || (fidx != 0xffffffffu && fidx != widx)) != 0ull;
                const bool unique = !wother && widx != 0xffffffffu;
                code = 1;
                const float eps = decision_eps(g);
                if (unique && wd < -thr_scale - eps) {                  // certain improving move
                    e = ((double)wd + (double)eps) * iscale;            // an upper bound, < -1e-6
                    idx = widx;
                    code = 0;
                } else if (!need_exact_sign && m > -thr_scale + eps &&
                           (widx == 0xffffffffu || wd > -thr_scale + eps)) {
                    e = 0.0;                                            // proven: no delta below -1e-6
                    idx = kNoMove;
                    code = 0;
                }
                FINE(pf, 6);
            }
            }   // !fast
        }
    }
    if constexpr (!CL) {
        if (nw > 1) {
            if (mine && lane == 0) { ctl->bestE = e; ctl->bestIdx = idx; ctl->ambiguous = code; }
            __syncthreads();            // the decision is out AND nobody reads the window any more
            e = ctl->bestE;
            idx = ctl->bestIdx;
            code = ctl->ambiguous;
            FINE(pf, 9);
        }
    }
    if (code == 0) return;              // (uniform: CL waves all computed the same code)

    // ---- exact stage, cooperative: every wave rebuilds the window from the same LDS words
    const bool heavy = code == 2;
    if (pf.on) { pf.cands += 1; pf.amb += heavy ? 1 : 0; }
    const UnitMinima um = load_unit_minima(v, g, lane);
    float m;
    const float thr = window_threshold<CL>(um, g, ctl->tsc, m);
    e = 0.0;
    idx = kNoMove;
    if (!heavy) {
        // each wave takes every nw-th candidate tile, reference dtype and operation order (lane = pair)
        int c = 0;
        for_each_candidate_tile(v, g, lane, thr, um, 1 << 30, [&](unsigned id) {
            if (c++ % nw == wv) {
                double d;
                unsigned di;
                eval_chunk_pair(v, g, id, lane, d, di);
                if (better(d, di, e, idx)) { e = d; idx = di; }
            }
        });
        if (tid == 0) {
            const double d = exact_delta(v, g.n, 0, g.n - 1);
            if (better(d, (unsigned)(g.n - 1), e, idx)) { e = d; idx = (unsigned)(g.n - 1); }
        }
        block_best(ctl, tid, g.nt, e, idx);
    } else {
        // heavy ties (regular grids): list every tile inside the window cooperatively and evaluate the
        // list exactly, one tile per wave at a time; if even the list overflows, sweep the tour exactly
        __syncthreads();                                // nlist was zeroed after the phase B barrier
        bool listed = false;
        const int tiles = g.GPl * g.NS * (g.MS >> 1);
        const unsigned kthr = fkey(thr);
        for (int t = tid; t < tiles; t += g.nt) {
            const int gpl = t % g.GPl;
            if (g.wc + g.CS * gpl < g.GP && v.Mc[t] <= kthr) {
                const unsigned pos = atomicAdd(&ctl->nlist, 1u);
                if (pos < (unsigned)g.lcap) v.list[pos] = (uint16_t)(((unsigned)(t / g.GPl) << 8) | (unsigned)gpl);
            }
        }
        __syncthreads();
        const unsigned nl = ctl->nlist;
        __syncthreads();
        if (tid == 0) ctl->nlist = 0;
        if (nl <= (unsigned)g.lcap) {
            listed = true;
            for (unsigned c = (unsigned)wv; c < nl; c += (unsigned)nw) {
                double d;
                unsigned di;
                eval_chunk_pair(v, g, v.list[c], lane, d, di);
                if (better(d, di, e, idx)) { e = d; idx = di; }
            }
            if (tid == 0) {
                const double d = exact_delta(v, g.n, 0, g.n - 1);
                if (better(d, (unsigned)(g.n - 1), e, idx)) { e = d; idx = (unsigned)(g.n - 1); }
            }
            block_best(ctl, tid, g.nt, e, idx);
        }
        if (!listed) {
            exact_sweep(v, g.n, tid, g.nt, e, idx);
            block_best(ctl, tid, g.nt, e, idx);
        }
    }
    FINE(pf, 7);                                        // exact stage
}

// write the filter copy of position p: every window index w = p (mod n) is the A value of entry
// slot(w) and the B value of entry slot(w - 4)
template <int Q, typename T>
__device__ __forceinline__ void put_xy(const View<T>& v, const Geo& g, int p, float x, float y)
{
    if (g.W + 4 <= 2 * g.n) {       // (uniform) at most two window copies: w = p and w = p + n
        const int s0 = slot<Q>(p), w1 = p + g.n;
        v.Xq[s0].x = x;
        v.Yq[s0].x = y;
        if (p >= 4) {
            const int sb = slot<Q>(p - 4);
            v.Xq[sb].y = x;
            v.Yq[sb].y = y;
        }
        if (w1 < g.W + 4) {
            const int sb = slot<Q>(w1 - 4);
            v.Xq[sb].y = x;
            v.Yq[sb].y = y;
            if (w1 < g.W) {
                const int s1 = slot<Q>(w1);
                v.Xq[s1].x = x;
                v.Yq[s1].x = y;
            }
        }
        return;
    }
    for (int w = p; w < g.W + 4; w += g.n) {
        if (w < g.W) {
            const int s = slot<Q>(w);
            v.Xq[s].x = x;
            v.Yq[s].x = y;
        }
        if (w >= 4) {
            const int sb = slot<Q>(w - 4);
            v.Xq[sb].y = x;
            v.Yq[sb].y = y;
        }
    }
}

template <int Q, typename T>
__device__ __forceinline__ void put_e(const View<T>& v, const Geo& g, int p, float e)
{
    if (g.W + 4 <= 2 * g.n) {
        const int w1 = p + g.n;
        v.Eq[slot<Q>(p)].x = e;
        if (p >= 4) v.Eq[slot<Q>(p - 4)].y = e;
        if (w1 < g.W + 4) {
            v.Eq[slot<Q>(w1 - 4)].y = e;
            if (w1 < g.W) v.Eq[slot<Q>(w1)].x = e;
        }
        return;
    }
    for (int w = p; w < g.W + 4; w += g.n) {
        if (w < g.W) v.Eq[slot<Q>(w)].x = e;
        if (w >= 4) v.Eq[slot<Q>(w - 4)].y = e;
    }
}

// reverse tour[i+1..j] (two_opt.py:42) and keep the filter window consistent.  Every lane first loads
// everything its swap needs (two positions with their coordinates, two interior edges) and only then
// writes, so the LDS round trips of the phase overlap; the caller closes the phase with a barrier.
// The reversal of R[i+1..j] (two_opt.py:42) as a reversal of the LDS copy: LDS positions lo0 .. lo0 + len - 1
// (mod n).  A segment longer than half the tour is replaced by its complement -- reversing either side of a
// cycle gives the same cycle, with the opposite orientation -- and the frame (fo, fs) records how the
// reference's array reads the LDS copy afterwards: with lo, hi the segment's LDS ends and q a position of the
// complement, new[q] = old[lo + hi - q], so R'[k] = old'[lo + hi - (fo + fs k)]: fo' = lo + hi - fo, fs' = -fs.
// At most n / 2 positions move (instead of up to n - 2), and with them the tiles the sweep has to recompute:
// at most 3/4 of the pairs read a moved position (1 - (1 - L/n)^2 with L <= n / 2) instead of up to all.
// The whole-tour reversal (0, n-1) that converged tours of a coupled group keep applying becomes a flip of fs.
// Q == 0 (exact kernel, no filter window to save on): never folded, the frame stays the identity.
template <int Q, typename T>
__device__ __forceinline__ void resolve_move(View<T>& v, int n, unsigned idx, int& lo0, int& len)
{
    const unsigned u = (unsigned)__builtin_amdgcn_readfirstlane((int)idx);      // (uniform: scalar registers)
    const int i = (int)(u >> 16), j = (int)(u & 0xffffu);
    const int L = j - i;
    int lo = v.fs > 0 ? v.fo + i + 1 : v.fo - j;        // LDS position of the segment's first entry, in (-n, 2n)
    lo = wrapn(lo, n);
    lo0 = lo;
    len = L;
    if constexpr (Q != 0) {
        if (2 * L > n) {
            lo0 = wrapn(lo + L - n, n);                 // the complement starts right behind the segment
            len = n - L;
            int fo = v.fs > 0 ? v.fo + i + j + 1 : v.fo - i - j - 1;    // lo + hi - fo, in (-2n, 3n)
            fo += fo < 0 ? n : 0;
            fo -= fo >= n ? n : 0;
            v.fo = wrapn(fo, n);
            v.fs = -v.fs;
        }
    }
}

// reverse the LDS copy's positions lo0 .. lo0 + len - 1 (mod n) and keep the filter window consistent
template <typename T, int Q, bool SPLIT = true>
__device__ __forceinline__ void apply_move(const View<T>& v, const Geo& g, int tid, int lo0, int len, Prof& pf)
{
    const int n = g.n;
    FINE_START_G(pf, 0x0100);
    const int h = len >> 1;                     // position swaps
    const int he = (len - 1) >> 1;              // the interior edges are mirrored (he <= h)
    if constexpr (Q != 0 && SPLIT) {
        // Short reversals (at most 31 swaps: nearly all of a tour's late iterations, every one of a 50- or 100-city
        // tour): FOUR lanes of wave 0 per swap up to 15 swaps -- the two coordinate copies and the two mirrored edges --,
        // two lanes (one per side, coordinates and edge) up to 31, and two more lanes for the new boundary edges.  A
        // lane then writes one position's window copies (8 stores) and / or one edge's (4) instead of all 26 of its
        // swap, and the wave runs the two store shapes once each: about half the instructions of the one-lane-per-swap
        // loop below, on the chain of every late iteration.  All lanes sit in one wave and read before they write, so
        // the swaps need no barrier between them, as below.
        // (Not where unit-less waves apply the reversal beside the marking -- u0 > 0, and the cluster kernel, which is
        //  compiled without this path: there the reversal is off the chain.)
        if (g.u0 == 0 && h >= 1 && h <= 31) {   // (uniform)
            const int lsh = h <= 15 ? 2 : 1;    // log2 of the lanes per swap
            int dxy = -1, de = -1;              // position whose coordinates / edge this lane writes
            float vx = 0.f, vy = 0.f, ve = 0.f;
            uint16_t tv = 0;
            if (tid < 64) {
                const int k = tid >> lsh, q = tid & ((1 << lsh) - 1);
                if (k < h) {
                    int p = lo0 + k, p2 = lo0 + len - 1 - k;
                    p -= p >= n ? n : 0;
                    p2 -= p2 >= n ? n : 0;
                    const int p2m = p2 == 0 ? n - 1 : p2 - 1;           // the edge in front of p2
                    const bool side = (q & 1) != 0;                     // false: writes at p, true: at p2 / p2m
                    if (lsh == 1 || q < 2) {
                        const int ss = slot<Q>(side ? p : p2);
                        dxy = side ? p2 : p;
                        vx = v.Xq[ss].x; vy = v.Yq[ss].x;
                        tv = v.tour[side ? p : p2];
                    }
                    if ((lsh == 1 || q >= 2) && k < he) {
                        de = side ? p2m : p;
                        ve = v.Eq[slot<Q>(side ? p : p2m)].x;
                    }
                } else if (tid < (h << lsh) + 2) {      // the two new boundary edges (the ends' neighbours outside)
                    int p = lo0, p2 = lo0 + len - 1;
                    p2 -= p2 >= n ? n : 0;
                    const int pl = p == 0 ? n - 1 : p - 1, pr = p2 == n - 1 ? 0 : p2 + 1;
                    const bool left = tid == (h << lsh);
                    const int sa = slot<Q>(left ? pl : p), sb = slot<Q>(left ? p2 : pr);
                    const float x1 = v.Xq[sa].x, y1 = v.Yq[sa].x, x2 = v.Xq[sb].x, y2 = v.Yq[sb].x;
                    ve = dist32(x1, y1, x2, y2);        // (pl, new p = old p2) or (new p2 = old p, pr)
                    de = left ? pl : p2;
                }
            }
            if (dxy >= 0) {
                v.tour[dxy] = tv;
                put_xy<Q>(v, g, dxy, vx, vy);
            }
            if (de >= 0) put_e<Q>(v, g, de, ve);
            FINE(pf, 8);
            return;
        }
    }
    for (int k = tid; k < h; k += g.nt) {
        int p = lo0 + k, p2 = lo0 + len - 1 - k;
        p -= p >= n ? n : 0;
        p2 -= p2 >= n ? n : 0;
        const uint16_t ta = v.tour[p], tb = v.tour[p2];
        if constexpr (Q != 0) {
            const int p2m = p2 == 0 ? n - 1 : p2 - 1;       // the edge in front of p2
            const int sp = slot<Q>(p), sp2 = slot<Q>(p2);
            const float ax = v.Xq[sp].x, ay = v.Yq[sp].x, bx = v.Xq[sp2].x, by = v.Yq[sp2].x;
            const bool ed = k < he;
            float ea = 0.f, eb = 0.f, lx = 0.f, ly = 0.f, rx = 0.f, ry = 0.f;
            int pl = 0;
            if (ed) { ea = v.Eq[sp].x; eb = v.Eq[slot<Q>(p2m)].x; }
            if (k == 0) {                       // p, p2 are the ends: the neighbours outside the segment
                pl = p == 0 ? n - 1 : p - 1;
                const int pr = p2 == n - 1 ? 0 : p2 + 1;
                lx = v.Xq[slot<Q>(pl)].x; ly = v.Yq[slot<Q>(pl)].x;
                rx = v.Xq[slot<Q>(pr)].x; ry = v.Yq[slot<Q>(pr)].x;
            }
            v.tour[p] = tb;
            v.tour[p2] = ta;
            put_xy<Q>(v, g, p, bx, by);
            put_xy<Q>(v, g, p2, ax, ay);
            if (ed) {
                put_e<Q>(v, g, p, eb);
                put_e<Q>(v, g, p2m, ea);
            }
            if (k == 0) {                       // the two new boundary edges
                put_e<Q>(v, g, pl, dist32(lx, ly, bx, by));
                put_e<Q>(v, g, p2, dist32(ax, ay, rx, ry));
            }
        } else {
            v.tour[p] = tb;
            v.tour[p2] = ta;
        }
    }
    FINE(pf, 8);                                // positions + coordinates + edges
}

// ------------------------------------------------------------------------------------------
// cluster barrier + best-move exchange (several workgroups per tour, both cluster kernels)
// ------------------------------------------------------------------------------------------
constexpr unsigned kSpinLimit = 1u << 26;       // bounded wait (about 10 s): never hang the GPU
constexpr int kSlotDw = 8;                      // three tagged 64-bit words per slot (+ one of padding)

// The exchange of one iteration: publish this workgroup's (e, idx, flags), wait until every workgroup of the cluster
// has published its own, reduce all of them (the same lexicographic rule everywhere, so all workgroups and all waves
// arrive at the same move).  Returns false on abort (a workgroup of the cluster is missing: spin limit hit), uniformly
// for the whole workgroup.
//
// Every 64-bit word of a slot carries the exchange's number in its upper half (epoch + 1: the area starts zeroed,
// and a cluster's exchanges are numbered through all of its tours): delta low half, delta high half, index (+ the stop
// flag in the tag's top bit).  A word is written by ONE 64-bit store and read by one 64-bit load, so a reader that sees
// the tag sees the value: no release / acquire pair, no arrival counter -- publishing is three stores that nobody
// waits for, and the wait is a poll of the slots themselves by wave 0 (lane = slot; agent-scope loads bypass the
// CU's vector cache), which reduces them and hands the winner to the other waves through LDS at the barrier.
// (Measured at TSP-1000 x 128: every wave polling for itself 13.8 -> 14.8 ms, wave 0 alone 13.5 -> 12.7 ms.)  The counter scheme it replaces cost four trips to the L2 per exchange (data, release + counter
// increment, the poll that sees the count, the slots) where this costs two.  Slots alternate between two sets by the
// exchange's parity: nobody can be two exchanges ahead of a workgroup that has not read the previous one.
// The one barrier inside also separates the waves' reads of the filter window (move selection) from the writes of
// the reversal that follows.  CS <= 64.
__device__ bool cluster_exchange_w(Ctl* ctl, unsigned* cs, int CS, int wc, unsigned epoch, int tid,
                                   unsigned flags_in, double& e, unsigned& idx, unsigned& flags_out)
{
    const unsigned ep = epoch + 1u;
    unsigned long long* set = reinterpret_cast<unsigned long long*>(cs + 16) +
                              (size_t)((epoch & 1u) * (unsigned)CS) * (kSlotDw / 2);
    if (tid == 0) {
        unsigned long long* s = set + (size_t)wc * (kSlotDw / 2);
        const unsigned long long tag = (unsigned long long)ep << 32;
        __hip_atomic_store(s + 0, tag | (unsigned)__double2loint(e), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(s + 1, tag | (unsigned)__double2hiint(e), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(s + 2, ((unsigned long long)(ep | (flags_in ? 0x80000000u : 0u)) << 32) | idx,
                           __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // wave 0 polls (lane = slot), reduces and hands the result to the other waves through LDS
    const int lane = tid & 63;
    if (tid < 64) {
        const unsigned long long* s = set + (size_t)(lane < CS ? lane : 0) * (kSlotDw / 2);
        unsigned long long w0 = 0, w1 = 0, w2 = 0;
        bool ok = true;
        for (unsigned spins = 0;; ++spins) {
            w0 = __hip_atomic_load(s + 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            w1 = __hip_atomic_load(s + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            w2 = __hip_atomic_load(s + 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            const bool have = (unsigned)(w0 >> 32) == ep && (unsigned)(w1 >> 32) == ep &&
                              ((unsigned)(w2 >> 32) & 0x7fffffffu) == ep;
            if (__ballot(!have) == 0ull) break;
            if (spins > kSpinLimit || __hip_atomic_load(cs + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0u) {
                __hip_atomic_store(cs + 1, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                ok = false;
                break;
            }
            __builtin_amdgcn_s_sleep(1);
        }
        double we = 0.0;
        unsigned wi = kNoMove;
        bool fl = false;
        if (ok && lane < CS) {
            we = __hiloint2double((int)(unsigned)w1, (int)(unsigned)w0);
            wi = (unsigned)w2;
            fl = (w2 >> 63) != 0ull;
        }
        wave_best(we, wi);
        const unsigned fo = __ballot(fl) != 0ull ? 1u : 0u;
        if (lane == 0) { ctl->xE = we; ctl->xIdx = wi; ctl->xok = ok ? 1 : 0; ctl->xfl = (int)fo; }
    }
    __syncthreads();
    e = ctl->xE;
    idx = ctl->xIdx;
    flags_out = (unsigned)ctl->xfl;
    return ctl->xok != 0;
}

constexpr unsigned kFlagStop = 1u;      // published by workgroup 0: wall-clock limit reached

// ------------------------------------------------------------------------------------------
// the persistent kernel
// ------------------------------------------------------------------------------------------
__host__ __device__ inline size_t align16(size_t x) { return (x + 15) & ~(size_t)15; }

// CL = several workgroups per tour ("full-window cluster", N up to the fast path's LDS limit): every
// workgroup of a cluster holds the whole tour and the whole filter window and applies every reversal,
// but sweeps only the lane groups gp = wc (mod CS) -- interleaved, so all workgroups see the same mix
// of short and long diagonals and the same share of the tiles a reversal touches.  Per iteration each
// finds the exact best move of its tiles, the cluster meets at cluster_exchange and everybody applies
// the winner.  Clusters take tours statically (cluster, cluster + num_clusters, ...); the host
// launches at most one workgroup per CU so that a cluster is co-resident.  Independent termination only.
// Threads per workgroup by filter class.  Class 256 (N about 670..1340) fills a CU's LDS with one
// workgroup of 512 threads = 2 waves per SIMD: bounding the launch at 512 gives the compiler 256 VGPRs
// instead of 128 (no spills); the other classes need the 128-VGPR budget for their occupancy
// (4 workgroups of 256 threads per CU at class 128) or run 1024 threads (class 512, exact kernel).
template <int Q>
constexpr int kMaxThreads = Q == 256 ? 512 : 1024;

template <typename T, int Q, bool CL>
__global__ void __launch_bounds__(kMaxThreads<Q>) k_two_opt(Params p)
{
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    Geo g = p.g;
    int64_t tk_next = 0;
    unsigned* cs = nullptr;
    unsigned epoch = 0;                         // barriers passed by this cluster so far
    if constexpr (CL) {
        g.wc = (int)(blockIdx.x % (unsigned)g.CS);
        tk_next = blockIdx.x / (unsigned)g.CS;
        cs = p.csync + (size_t)tk_next * (size_t)p.cstride;
    } else {                                    // compile-time constants for the one-workgroup kernel
        g.CS = 1;
        g.wc = 0;
        g.GPl = g.GP;
    }
    const int n = g.n, tid = threadIdx.x, nt = g.nt;
    View<T> v;
    v.ctl = reinterpret_cast<Ctl*>(smem);
    size_t off = align16(sizeof(Ctl));
    v.tour = reinterpret_cast<uint16_t*>(smem + off);
    off += align16(sizeof(uint16_t) * (size_t)(n + 1));
    v.Xq = reinterpret_cast<v2f*>(smem + off);
    off += sizeof(v2f) * 8 * (size_t)Q;
    v.Yq = reinterpret_cast<v2f*>(smem + off);
    off += sizeof(v2f) * 8 * (size_t)Q;
    v.Eq = reinterpret_cast<v2f*>(smem + off);
    off += sizeof(v2f) * 8 * (size_t)Q;
    v.Mc = nullptr;
    v.list = nullptr;
    v.Mu = nullptr;
    if (g.inc) {
        const size_t tiles = (size_t)g.GPl * g.NS * (g.MS >> 1);
        v.Mc = reinterpret_cast<unsigned*>(smem + off);
        off += align16(sizeof(float) * tiles);
        v.list = reinterpret_cast<uint16_t*>(smem + off);
        off += align16(sizeof(uint16_t) * (size_t)g.lcap);
        v.Mu = reinterpret_cast<unsigned*>(smem + off);
        off += align16(sizeof(unsigned) * (size_t)(g.GPl * g.NS));    // (padded to a multiple of 4 entries)
    }
    T* xl = reinterpret_cast<T*>(smem + off);
    Ctl* ctl = v.ctl;
    for (;;) {
        __syncthreads();
        int64_t tk;
        if constexpr (CL) {
            if (tid == 0) ctl->nlist = 0;
            tk = tk_next;
            tk_next += p.num_clusters;
        } else {
            if (tid == 0) { ctl->tour_id = (int)atomicAdd(p.queue, 1u); ctl->nlist = 0; }
            __syncthreads();
            tk = ctl->tour_id;
        }
        if (tk >= p.num_tours) break;          // uniform exit: every wave leaves here

        const int64_t grp = tk / p.group_size;
        Prof pf = make_prof(p.stamps);
        const unsigned long long t_tour = pf.on ? clock64() : 0;
        int it = 0, target = 0;
        if (p.mode == kModeForced) {
            it = p.iters[tk];
            target = p.target[grp];
            const int st = p.status ? p.status[tk] : 0;
            if (it >= target || (st & (TSP2OPT_ST_BAD_INDEX | TSP2OPT_ST_NOT_CLOSED |
                                       TSP2OPT_ST_NONFINITE | TSP2OPT_ST_RANGE)))
                continue;
        }
        const T* X = reinterpret_cast<const T*>(p.points) + (size_t)(tk / p.tpi) * (size_t)n * 2;
        int64_t* gt = p.tours + (size_t)tk * (size_t)(n + 1);

        // ---- stage the tour, validate it (no out-of-range index may reach a gather) --------
        int bad = 0;
        for (int k = tid; k <= n; k += nt) {
            const int64_t t = gt[k];
            if (t < 0 || t >= n) { bad |= TSP2OPT_ST_BAD_INDEX; v.tour[k] = 0; }
            else v.tour[k] = (uint16_t)t;
        }
        if (tid == 0 && gt[0] != gt[n]) bad |= TSP2OPT_ST_NOT_CLOSED;
        // ---- bounding box of the instance (for centring/scaling the filter copy) -----------
        double mnx = INFINITY, mxx = -INFINITY, mny = INFINITY, mxy = -INFINITY;
        for (int k = tid; k < n; k += nt) {
            const T x = X[2 * k], y = X[2 * k + 1];
            if (g.xlds) { xl[2 * k] = x; xl[2 * k + 1] = y; }
            const double dx = (double)x, dy = (double)y;
            if (!(fabs(dx) <= 1.0e150) || !(fabs(dy) <= 1.0e150))
                bad |= (dx != dx || dy != dy || fabs(dx) == INFINITY || fabs(dy) == INFINITY)
                           ? TSP2OPT_ST_NONFINITE : TSP2OPT_ST_RANGE;
            mnx = fmin(mnx, dx); mxx = fmax(mxx, dx);
            mny = fmin(mny, dy); mxy = fmax(mxy, dy);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            mnx = fmin(mnx, __shfl_xor(mnx, o)); mxx = fmax(mxx, __shfl_xor(mxx, o));
            mny = fmin(mny, __shfl_xor(mny, o)); mxy = fmax(mxy, __shfl_xor(mxy, o));
            bad |= __shfl_xor(bad, o);
        }
        if ((tid & 63) == 0) {
            const int w = tid >> 6;
            ctl->redd[4 * w] = mnx; ctl->redd[4 * w + 1] = mxx;
            ctl->redd[4 * w + 2] = mny; ctl->redd[4 * w + 3] = mxy;
            ctl->pIdx[w] = (unsigned)bad;
        }
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < (nt >> 6); ++w) {
                mnx = fmin(mnx, ctl->redd[4 * w]); mxx = fmax(mxx, ctl->redd[4 * w + 1]);
                mny = fmin(mny, ctl->redd[4 * w + 2]); mxy = fmax(mxy, ctl->redd[4 * w + 3]);
                bad |= (int)ctl->pIdx[w];
            }
            ctl->flags = bad;
            ctl->cx = 0.5 * (mnx + mxx);
            ctl->cy = 0.5 * (mny + mxy);
            const double half = fmax(0.5 * (mxx - mnx), 0.5 * (mxy - mny));
            int ex = 0;
            double sc = 1.0;
            double isc = 1.0;
            if (half > 0.0 && half < INFINITY) { (void)frexp(half, &ex); sc = ldexp(1.0, -ex); isc = ldexp(1.0, ex); }
            ctl->sc = sc;                       // half * sc in [0.5, 1)
            ctl->tsc = (float)(1.0e-6 * sc);
            ctl->isc = isc;
        }
        __syncthreads();
        const int flags = ctl->flags;
        v.X = g.xlds ? xl : X;
        v.fo = 0;                               // the staged copy IS the reference's array
        v.fs = 1;
        if (flags != 0) {                       // invalid input: tour untouched (uniform branch)
            if (tid == 0 && g.wc == 0) {
                if (p.status) p.status[tk] = flags;
                if (p.mode == kModeIndep) p.iters[tk] = 0;
            }
            continue;
        }
        if (p.mode == kModeValidate) {          // (uniform branch)
            if (tid == 0) { p.iters[tk] = 0; if (p.status) p.status[tk] = 0; }
            continue;
        }
        if constexpr (Q != 0) {
            const double cx = ctl->cx, cy = ctl->cy, sc = ctl->sc;
            for (int w = tid; w < 8 * Q; w += nt) {
                const int na = v.tour[w % n], nb = v.tour[(w + 4) % n];
                const double xa = (double)v.X[2 * na], ya = (double)v.X[2 * na + 1];
                const double xb = (double)v.X[2 * nb], yb = (double)v.X[2 * nb + 1];
                v.Xq[slot<Q>(w)] = (v2f){(float)((xa - cx) * sc), (float)((xb - cx) * sc)};
                v.Yq[slot<Q>(w)] = (v2f){(float)((ya - cy) * sc), (float)((yb - cy) * sc)};
            }
            __syncthreads();
            for (int w = tid; w < 8 * Q; w += nt) {
                const int s0 = slot<Q>(w), s1 = slot<Q>(w + 1 < 8 * Q ? w + 1 : w);
                const v2f x0 = v.Xq[s0], y0 = v.Yq[s0], x1 = v.Xq[s1], y1 = v.Yq[s1];
                v.Eq[s0] = (v2f){dist32(x0.x, y0.x, x1.x, y1.x), dist32(x0.y, y0.y, x1.y, y1.y)};
            }
            if (g.inc)          // units without a lane group (cluster padding) never get a minimum
                for (int u = tid; u < ((g.GPl * g.NS + 3) & ~3); u += nt) v.Mu[u] = 0xffffffffu;
        }
        __syncthreads();

        // ---- improvement loop ----------------------------------------------------------------
        if (pf.on && tid == 0) atomicAdd(&p.stamps[3], clock64() - t_tour);
        const long long t_start = p.time_limit_ticks ? wall_clock64() : 0;
        int sweeps = 0, st = 0, turn = 0;       // turn: which wave decides this iteration (rotates)
        double e;
        unsigned idx;
        if constexpr (Q != 0) {
            if (p.dbg_sweeps > 0) {     // diagnostic: pure filter-sweep throughput, no selection/reversal
                float acc = 0.f;
                for (int k = 0; k < p.dbg_sweeps; ++k) {
                    float a1, a2;
                    unsigned chunk;
                    filter_sweep<Q, CL>(v.Xq, v.Yq, v.Eq, nullptr, g, tid, a1, a2, chunk);
                    acc += a1 + a2 + (float)chunk;
                    asm volatile("" ::: "memory");
                }
                if (acc == 12345.678f) p.iters[tk] = 1;      // keeps the sweeps live
                if (tid == 0) { p.iters[tk] = p.dbg_sweeps; if (p.status) p.status[tk] = 0; }
                continue;
            }
        }
        // One loop for both modes (a single inlined copy of the sweep keeps the hot code small).
        //   independent: stop on the tour's own minimum (two_opt.py:40) or the cap (:47).
        //   forced (coupled mode, continuation): the group keeps iterating until `target`; this tour
        //   applies its own strictly negative argmin every iteration (two_opt.py:41-42).  A fixed
        //   point (no negative delta) or a proven 2-cycle (the same reversal twice in a row) fixes
        //   the rest of the trajectory without sweeping; otherwise one more sweep at `target` tells
        //   whether the tour is still active there (then the group is not finished: k_group_lockstep).
        const bool forced = p.mode == kModeForced;
        bool have_prev = false, prev_active = false, active_at_target = false;
        unsigned prev_idx = kNoMove;
        unsigned last = kFullSweep;             // reversal applied since the previous sweep
        const int tid_fixed = tid;
        for (;;) {
            // The kernel sits at its VGPR limit.  Left alone, the compiler hoists everything that is
            // derived from the thread index (unit, LDS addresses, conversion constants) out of this loop
            // and then spills it to scratch, paying a memory round trip per use; an opaque copy of the
            // index per iteration makes those values loop-variant, i.e. recomputed where they are used.
            int tid = tid_fixed;
            asm volatile("" : "+v"(tid));
            const bool check_only = forced && it >= target;
            if (check_only && target >= p.max_iter) break;
            bool cached = false;
            if constexpr (Q != 0) cached = g.inc != 0;          // (uniform)
            if constexpr (Q != 0) {
                if (cached) {
                    unsigned long long t0 = 0;
                    if (COARSE(pf)) t0 = clock64();
                    refresh_cached<Q, CL>(v, g, tid, last, pf);                 // phase B
                    __syncthreads();
                    FINE(pf, 2);                                                // barrier after the refresh
                    if (tid == 0) ctl->nlist = 0;
                    if (COARSE(pf)) { const unsigned long long t1 = clock64(); pf.sweep += t1 - t0; t0 = t1; }
                    select_cached<T, Q, CL>(v, g, tid, forced, turn, e, idx, pf);      // phase C
                    turn = turn + 1 == (g.nt >> 6) ? 0 : turn + 1;
                    if (COARSE(pf)) pf.select += clock64() - t0;
                }
            }
            if (!cached) find_best<T, Q, CL>(v, g, tid, forced, last, e, idx, pf);
            ++sweeps;
            unsigned xfl = 0;
            if constexpr (CL) {
                unsigned myflags = 0;
                if (g.wc == 0 && p.time_limit_ticks && wall_clock64() - t_start > p.time_limit_ticks)
                    myflags |= kFlagStop;
                if (!cluster_exchange_w(ctl, cs, g.CS, g.wc, epoch, tid, myflags, e, idx, xfl)) {
                    st = TSP2OPT_ST_INTERNAL;
                    break;
                }
                ++epoch;
            }
            const bool active = e < -1.0e-6;
            bool stop_after = false;
            if (!forced) {
                if (!active) break;                                         // two_opt.py:40
            } else {
                if (check_only) { active_at_target = active; break; }
                if (!(e < 0.0)) { it = target; break; }                     // fixed point: inactive forever
                if (have_prev && idx == prev_idx) {                         // 2-cycle A -> B -> A
                    const int rem = target - it;
                    it = target;
                    if (!(rem & 1)) { active_at_target = active; break; }
                    active_at_target = prev_active;
                    stop_after = true;                                      // one more reversal: back to A
                }
                have_prev = true; prev_idx = idx; prev_active = active;
            }
            unsigned long long ta = 0;
            if (COARSE(pf)) ta = clock64();
            // (cached path: select_cached / the cluster exchange ended with the barrier after which nobody
            //  reads the window any more)
            FINE_START_G(pf, 0x0501);
            int lo0, len;
            resolve_move<Q>(v, n, idx, lo0, len);               // which side of the cycle; frame update
            apply_move<T, Q, !CL>(v, g, tid, lo0, len, pf);     // phase A
            if constexpr (Q != 0) {
                if (cached) mark_touched<CL>(v, g, tid, lo0, len);
            }
            FINE(pf, 0);                                        // marking + compaction
            __syncthreads();
            FINE(pf, 10);                                       // closing barrier
            last = idx;
            if (COARSE(pf)) pf.apply += clock64() - ta;
            if (stop_after) break;
            ++it;
            if (!forced) {
                if (it >= p.max_iter) { st |= TSP2OPT_ST_CAPPED; break; }   // two_opt.py:47
                if (CL ? (xfl & kFlagStop) != 0u
                       : (p.time_limit_ticks && wall_clock64() - t_start > p.time_limit_ticks)) {
                    st |= TSP2OPT_ST_TIME;                                  // plugin two_opt.py:63-65
                    break;
                }
            }
        }
        if (forced && active_at_target && target < p.max_iter && tid == 0)
            atomicOr(&p.group_flag[grp], 1);

        // ---- write back ------------------------------------------------------------------------
        __builtin_amdgcn_s_setprio(0);
        if (CL && st == TSP2OPT_ST_INTERNAL) {
            // cluster broken (a workgroup is missing): this tour and every later tour of the cluster stay
            // untouched and are flagged, by whichever workgroups got here (same values: idempotent)
            if (tid == 0)
                for (int64_t t = tk; t < p.num_tours; t += p.num_clusters) {
                    if (p.status) p.status[t] = st;
                    p.iters[t] = 0;
                }
            return;
        }
        if (CL && g.wc != 0) continue;          // every workgroup holds the same tour; the first writes it
        for (int k = tid; k <= n; k += nt) gt[k] = (int64_t)v.tour[ipos(v, n, k)];     // R[k], through the frame
        if (tid == 0) {
            p.iters[tk] = it;
            if (p.work_sweeps) p.work_sweeps[tk] += sweeps;
            if (p.status && p.mode == kModeIndep) p.status[tk] = st;
            if (pf.on) {
                atomicAdd(&p.stamps[0], pf.sweep);
                atomicAdd(&p.stamps[1], pf.select);
                atomicAdd(&p.stamps[2], pf.apply);
                atomicAdd(&p.stamps[4], clock64() - t_tour);
                atomicAdd(&p.stamps[5], (unsigned long long)pf.amb);
                atomicAdd(&p.stamps[6], (unsigned long long)pf.cands);
                atomicAdd(&p.stamps[7], pf.candcyc);
#ifdef TSP2OPT_FINE
                for (int k = 0; k < 16; ++k) atomicAdd(&p.stamps[8 + k], pf.fine[k]);
#endif
            }
        }
    }
}

}  // namespace t2o
