// nm_scan.hip -- the gated linear recurrence along sequences and its gradient (C ABI: nm_scan_*).
//
//   h_i = r_i h_{i-1} + u_i      plain: r = a, u = x;   blend: r = 1 - a, u = a x  (alpha compositing, a = opacity, far to near)
//   backward, f_i = r_i lambda_i:  lambda_i = g_i + f_{i+1} (+ g_last at a sequence's last step, where f_{i+1} is dropped)
//     dx = lambda (blend: a lambda),   da = lambda h_{i-1} (blend: lambda (x - h_{i-1})),   dh0 = f at the first step
//
// Bound: HBM.  A step of a channel costs two multiply-adds and 6 .. 20 bytes, so what counts is to touch every operand once, in whole lines.
//
// Split.  All sequences lie one after the other on ONE axis of L steps; a sequence's first step starts anew (a flag, never a product with zero:
// an infinity in one sequence must not reach the next).  A workgroup takes a range of steps and a block of channels, a tile at a time:
// CL lanes side by side hold VEC channels each, TL = 256 / CL lanes follow each other in time with SEG consecutive steps each.  A
// thread reduces its steps to one affine map (A, H, flag), the maps are scanned by lane exchanges within a wave and through LDS between the four
// waves, and the thread then runs its steps again from its true initial state -- from registers, nothing is loaded twice.
//   - many short sequences: ranges are whole sequences, no state crosses a workgroup;
//   - few long ones, or packed ones of any length: ranges are cut anywhere.  A first launch reduces every range to its map, reading it from its LAST
//     sequence start on only; a small launch scans the maps; the main launch starts every range from its carried state.
// The backward pass walks the tiles from the last to the first with the same decomposition of f, and recomputes h_{i-1} in fp32 from the
// states that the forward pass kept at every tile's start: 4 bytes per channel and tile instead of a second read of rounded states.
// States, maps and sums are fp32; outputs are rounded once.  Every sum has a fixed order.
#include "nm_error.h"
#include "nm_num.h"
#include "nm_scan_index.h"

struct NmScanArgs {
    const void* gate;
    const void* x;
    const float* h0;                     // [S, D] or NULL
    const int* seg;                      // packed: sequence of every row (-1: none); NULL: row / T
    const int* cu;                       // packed: [S + 1]
    long long L, S, chunk;               // chunk: steps of one workgroup
    unsigned T;
    int D, reverse, blend, cl_log2, blocks, map_only;
    void* states;                        // [L, D] or NULL
    float* last;                         // [S, D]
    float* keep;                         // states at the tile starts, [chunks][tiles per chunk][D], or NULL
    float* map_a; float* map_h; int* map_f;     // [chunks, D] x 2, [chunks]
    const float* carry;                  // [chunks, D] or NULL
    // backward
    const void* g;                       // [L, D] or NULL
    const float* g_last;                 // [S, D] or NULL
    void* dgate; void* dx; float* dh0;   // each may be NULL
    float* dgate_part;                   // shared gate over several channel blocks: [blocks, L]
};

template <int DT, int VEC> struct NmVec { typename NmType<DT>::elem e[VEC]; };

template <int DT, int VEC>
__device__ __forceinline__ NmVec<DT, VEC> nm_s_load(const typename NmType<DT>::elem* p) {
    NmVec<DT, VEC> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <int DT, int VEC>
__device__ __forceinline__ void nm_s_store(typename NmType<DT>::elem* p, const float (&f)[VEC]) {
    NmVec<DT, VEC> v;
#pragma unroll
    for (int k = 0; k < VEC; ++k) v.e[k] = (typename NmType<DT>::elem)f[k];
    __builtin_memcpy(p, &v, sizeof(v));
}

// the affine map h -> A h + H of a stretch of steps; F: it starts anew, whatever came before
template <int VEC> struct NmMap { float a[VEC], h[VEC]; int f; };

// `m` applied after the state `s`
template <int VEC>
__device__ __forceinline__ void nm_s_apply(const NmMap<VEC>& m, float (&s)[VEC]) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) s[k] = m.f ? m.h[k] : fmaf(m.a[k], s[k], m.h[k]);
}

// exclusive scan of the lanes' maps in time order within a wave (DIR = 1: lower lanes come first, -1: higher lanes); the wave's total is left in the
// last lane's `m`.  Lanes of one time are neighbours: exchanges go over multiples of cl.
template <int VEC, int DIR>
__device__ __forceinline__ void nm_s_wave_scan(NmMap<VEC>& m, NmMap<VEC>& before, int lane, int cl) {
    for (int o = cl; o < 64; o <<= 1) {
        NmMap<VEC> p;
        const int src = lane - DIR * o;
        const bool has = src >= 0 && src < 64;
        p.f = __shfl(m.f, src & 63);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            p.a[k] = __shfl(m.a[k], src & 63);
            p.h[k] = __shfl(m.h[k], src & 63);
        }
        if (has && !m.f) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                m.h[k] = fmaf(m.a[k], p.h[k], m.h[k]);
                m.a[k] *= p.a[k];
            }
            m.f = p.f;
        }
    }
    const int src = lane - DIR * cl;
    const bool has = src >= 0 && src < 64;
    before.f = __shfl(m.f, src & 63);
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        before.a[k] = __shfl(m.a[k], src & 63);
        before.h[k] = __shfl(m.h[k], src & 63);
        if (!has) { before.a[k] = 1.f; before.h[k] = 0.f; }
    }
    if (!has) before.f = 0;
}

// which sequence the thread's steps belong to: index (-1: none), bit s of first / final: the step is its sequence's first / last
template <int SEG> struct NmSteps { int seq[SEG]; unsigned first, final; int n; };

template <int SEG>
__device__ __forceinline__ NmSteps<SEG> nm_s_steps(const NmScanArgs& p, long long c0, long long c1, long long i0, unsigned pos0, long long q0) {
    NmSteps<SEG> t;
    t.first = t.final = 0u;
    const long long left = c1 - i0;
    t.n = left >= SEG ? SEG : left > 0 ? (int)left : 0;
    if (p.seg) {
        int before = -2;
        if (t.n > 0 && i0 > 0) before = p.seg[p.reverse ? p.L - i0 : i0 - 1];
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            t.seq[s] = -1;
            if (s < t.n) t.seq[s] = p.seg[p.reverse ? p.L - 1 - (i0 + s) : i0 + s];
        }
        int after = -2;
        if (t.n == SEG && i0 + SEG < p.L) after = p.seg[p.reverse ? p.L - 1 - (i0 + SEG) : i0 + SEG];
        else if (t.n > 0 && t.n < SEG && i0 + t.n < p.L) after = p.seg[p.reverse ? p.L - 1 - (i0 + t.n) : i0 + t.n];
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            const int prev = s == 0 ? before : t.seq[s > 0 ? s - 1 : 0], next = s + 1 < t.n ? t.seq[s + 1 < SEG ? s + 1 : s] : after;
            if (prev != t.seq[s] || t.seq[s] < 0) t.first |= 1u << s;
            if (next != t.seq[s] || t.seq[s] < 0) t.final |= 1u << s;
        }
    } else {
        const unsigned off = (unsigned)(i0 - c0) + pos0, q = off / p.T;
        unsigned pos = off - q * p.T;
        int b = (int)(q0 + q);
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            t.seq[s] = p.reverse ? (int)(p.S - 1) - b : b;
            if (pos == 0) t.first |= 1u << s;
            if (pos + 1 == p.T) {
                t.final |= 1u << s;
                pos = 0;
                ++b;
            } else {
                ++pos;
            }
        }
    }
    return t;
}

#define NM_S_THREADS 256

template <int DX, int DG, int VEC, int SEG, bool SHARED>
__global__ __launch_bounds__(NM_S_THREADS) void nm_scan_forward_kernel(NmScanArgs p) {
    typedef typename NmType<DX>::elem TX;
    typedef typename NmType<DG>::elem TG;
    constexpr int GV = SHARED ? 1 : VEC;
    __shared__ float sh_a[2][4][64 * VEC], sh_h[2][4][64 * VEC];
    __shared__ int sh_f[2][4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, cl = 1 << p.cl_log2, cx = t & (cl - 1), tl = t >> p.cl_log2;
    const int tile = (NM_S_THREADS >> p.cl_log2) * SEG;
    const long long c = blockIdx.x / p.blocks;
    const int blk = (int)(blockIdx.x % p.blocks);
    const long long c0 = c * p.chunk, c1 = c0 + p.chunk < p.L ? c0 + p.chunk : p.L;
    // (channels that would end beyond D are the last VEC: computed twice, written twice with the same value)
    int ch = (blk * cl + cx) * VEC;
    if (ch + VEC > p.D) ch = p.D - VEC;
    const long long step = p.reverse ? -1 : 1;
    const long long q0 = p.seg ? 0 : c0 / p.T;
    const unsigned pos0 = p.seg ? 0u : (unsigned)(c0 - q0 * p.T);
    const long long tiles_per_chunk = (p.chunk + tile - 1) / tile;

    NmMap<VEC> total;                    // map_only: everything before the current tile
    float state[VEC];                    // otherwise: the state before the current tile
    total.f = 0;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        total.a[k] = 1.f;
        total.h[k] = 0.f;
        state[k] = p.carry ? p.carry[c * p.D + ch + k] : 0.f;
    }
    long long b0 = c0;
    if (p.map_only) {                    // what comes before the range's last sequence start does not matter
        const long long s0 = p.seg ? nm_scan_reduce_from(p.cu, p.seg[p.reverse ? p.L - c1 : c1 - 1], p.reverse, p.L, c0, c1) : (c1 - 1) / p.T * p.T;
        if (s0 > c0) b0 = c0 + (s0 - c0) / tile * tile;
    }
    int buf = 0;
    for (long long b = b0; b < c1; b += tile, buf ^= 1) {
        const long long i0 = b + tl * SEG;
        const long long row0 = p.reverse ? p.L - 1 - i0 : i0;
        const TX* px = (const TX*)p.x + row0 * p.D + ch;
        const TG* pg = (const TG*)p.gate + (SHARED ? row0 : row0 * p.D + ch);
        const long long gs = SHARED ? step : step * p.D;
        NmVec<DX, VEC> xv[SEG];
        NmVec<DG, GV> gv[SEG];
        if (b + tile <= c1) {
#pragma unroll
            for (int s = 0; s < SEG; ++s) {
                gv[s] = nm_s_load<DG, GV>(pg + s * gs);
                xv[s] = nm_s_load<DX, VEC>(px + s * step * p.D);
            }
        } else {
#pragma unroll
            for (int s = 0; s < SEG; ++s) {
                gv[s] = {};
                xv[s] = {};
                if (i0 + s < c1) {
                    gv[s] = nm_s_load<DG, GV>(pg + s * gs);
                    xv[s] = nm_s_load<DX, VEC>(px + s * step * p.D);
                }
            }
        }
        const NmSteps<SEG> st = nm_s_steps<SEG>(p, c0, c1, i0, pos0, q0);
        // one step: state h -> r h + u
        auto advance = [&](int s, float (&h)[VEC]) {
            if (((st.first >> s) & 1) != 0) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) h[k] = p.h0 && st.seq[s] >= 0 ? p.h0[(long long)st.seq[s] * p.D + ch + k] : 0.f;
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float a = (float)gv[s].e[SHARED ? 0 : k], x = (float)xv[s].e[k];
                h[k] = p.blend ? fmaf(1.0f - a, h[k], a * x) : fmaf(a, h[k], x);
                if (st.seq[s] < 0) h[k] = 0.f;
            }
        };
        NmMap<VEC> m, before;
        m.f = 0;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            m.a[k] = 1.f;
            m.h[k] = 0.f;
        }
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            if (s >= st.n) break;
            if ((st.first >> s) & 1) m.f = 1;
            advance(s, m.h);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float a = (float)gv[s].e[SHARED ? 0 : k];
                m.a[k] *= p.blend ? 1.0f - a : a;
            }
        }
        nm_s_wave_scan<VEC, 1>(m, before, lane, cl);
        if (lane >= 64 - cl) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                sh_a[buf][wave][cx * VEC + k] = m.a[k];
                sh_h[buf][wave][cx * VEC + k] = m.h[k];
            }
            if (lane == 63) sh_f[buf][wave] = m.f;
        }
        __syncthreads();                 // (two buffers: a wave that is a tile ahead writes the other one)
        if (!p.map_only && p.keep && tl == 0) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) p.keep[(c * tiles_per_chunk + (b - c0) / tile) * p.D + ch + k] = state[k];
        }
        float h[VEC];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            NmMap<VEC> mw;
            mw.f = sh_f[buf][w];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                mw.a[k] = sh_a[buf][w][cx * VEC + k];
                mw.h[k] = sh_h[buf][w][cx * VEC + k];
                if (w == wave) h[k] = state[k];
            }
            nm_s_apply(mw, state);
            if (p.map_only) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) total.a[k] = total.f || mw.f ? 0.f : total.a[k] * mw.a[k];
                total.f |= mw.f;
            }
        }
        if (p.map_only) continue;
        nm_s_apply(before, h);
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            if (s >= st.n) break;
            advance(s, h);
            if (p.states) nm_s_store<DX, VEC>((TX*)p.states + (row0 + s * step) * p.D + ch, h);
            if (((st.final >> s) & 1) && st.seq[s] >= 0) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) p.last[(long long)st.seq[s] * p.D + ch + k] = h[k];
            }
        }
    }
    if (p.map_only && tl == 0) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            p.map_a[c * p.D + ch + k] = total.a[k];
            p.map_h[c * p.D + ch + k] = state[k];
        }
        if (blk == 0 && cx == 0) p.map_f[c] = total.f || b0 > c0;
    }
}

template <int DX, int DG, int VEC, int SEG, bool SHARED>
__global__ __launch_bounds__(NM_S_THREADS) void nm_scan_backward_kernel(NmScanArgs p) {
    typedef typename NmType<DX>::elem TX;
    typedef typename NmType<DG>::elem TG;
    constexpr int GV = SHARED ? 1 : VEC;
    __shared__ float sh_a[2][4][64 * VEC], sh_h[2][4][64 * VEC], sh_b[2][4][64 * VEC], sh_r[2][4][64 * VEC];
    __shared__ int sh_f[2][4], sh_e[2][4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, cl = 1 << p.cl_log2, cx = t & (cl - 1), tl = t >> p.cl_log2;
    const int tile = (NM_S_THREADS >> p.cl_log2) * SEG;
    const long long c = blockIdx.x / p.blocks;
    const int blk = (int)(blockIdx.x % p.blocks);
    const long long c0 = c * p.chunk, c1 = c0 + p.chunk < p.L ? c0 + p.chunk : p.L;
    const int own = (blk * cl + cx) * VEC;                   // first channel that is this thread's own (see the forward kernel)
    int ch = own;
    if (ch + VEC > p.D) ch = p.D - VEC;
    const long long step = p.reverse ? -1 : 1;
    const long long q0 = p.seg ? 0 : c0 / p.T;
    const unsigned pos0 = p.seg ? 0u : (unsigned)(c0 - q0 * p.T);
    const long long tiles_per_chunk = (p.chunk + tile - 1) / tile;

    NmMap<VEC> total;                    // map_only: everything after the current tile
    float flow[VEC];                     // f of the step after the current tile
    total.f = 0;
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        total.a[k] = 1.f;
        flow[k] = p.carry ? p.carry[c * p.D + ch + k] : 0.f;
    }
    long long tiles = (c1 - c0 + tile - 1) / tile;
    bool cut = false;
    if (p.map_only) {                    // what comes after the range's first sequence end does not matter
        const long long e = p.seg ? nm_scan_reduce_to(p.cu, p.seg[p.reverse ? p.L - 1 - c0 : c0], p.reverse, p.L, c0, c1) : c0 / p.T * p.T + p.T - 1;
        if (e < c1) {
            const long long need = (e - c0) / tile + 1;
            cut = need < tiles;
            tiles = need;
        }
    }
    int buf = 0;
    for (long long j = tiles - 1; j >= 0; --j, buf ^= 1) {
        const long long b = c0 + j * tile, i0 = b + tl * SEG;
        const long long row0 = p.reverse ? p.L - 1 - i0 : i0;
        const long long gs = SHARED ? step : step * p.D;
        const TX* px = (const TX*)p.x + row0 * p.D + ch;
        const TX* pc = (const TX*)p.g + row0 * p.D + ch;
        const TG* pg = (const TG*)p.gate + (SHARED ? row0 : row0 * p.D + ch);
        NmVec<DX, VEC> xv[SEG], cv[SEG];
        NmVec<DG, GV> gv[SEG];
        const bool inside = b + tile <= c1, want_x = !p.map_only && (p.dgate || p.dgate_part);
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            gv[s] = {};
            xv[s] = {};
            cv[s] = {};
        }
        if (inside) {
#pragma unroll
            for (int s = 0; s < SEG; ++s) {
                gv[s] = nm_s_load<DG, GV>(pg + s * gs);
                if (p.g) cv[s] = nm_s_load<DX, VEC>(pc + s * step * p.D);
                if (want_x) xv[s] = nm_s_load<DX, VEC>(px + s * step * p.D);
            }
        } else {
#pragma unroll
            for (int s = 0; s < SEG; ++s)
                if (i0 + s < c1) {
                    gv[s] = nm_s_load<DG, GV>(pg + s * gs);
                    if (p.g) cv[s] = nm_s_load<DX, VEC>(pc + s * step * p.D);
                    if (want_x) xv[s] = nm_s_load<DX, VEC>(px + s * step * p.D);
                }
        }
        const NmSteps<SEG> st = nm_s_steps<SEG>(p, c0, c1, i0, pos0, q0);
        auto enter = [&](int s, float (&h)[VEC]) {           // state before step s, where it is a sequence's first
            if ((st.first >> s) & 1) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) h[k] = p.h0 && st.seq[s] >= 0 ? p.h0[(long long)st.seq[s] * p.D + ch + k] : 0.f;
            }
        };
        auto advance = [&](int s, float (&h)[VEC]) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float a = (float)gv[s].e[SHARED ? 0 : k], x = (float)xv[s].e[k];
                h[k] = p.blend ? fmaf(1.0f - a, h[k], a * x) : fmaf(a, h[k], x);
                if (st.seq[s] < 0) h[k] = 0.f;
            }
        };
        auto retreat = [&](int s, float (&f)[VEC], float (&lam)[VEC]) {     // f of the step after s -> lambda and f of s
            const bool end = (st.final >> s) & 1;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float a = (float)gv[s].e[SHARED ? 0 : k], r = p.blend ? 1.0f - a : a;
                float v = end ? 0.f : f[k];
                if (end && p.g_last && st.seq[s] >= 0) v = p.g_last[(long long)st.seq[s] * p.D + ch + k];
                lam[k] = (float)cv[s].e[k] + v;
                f[k] = r * lam[k];
                if (st.seq[s] < 0) lam[k] = f[k] = 0.f;
            }
        };
        NmMap<VEC> mf, mr, bf, br;
        mf.f = mr.f = 0;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            mf.a[k] = 1.f;
            mf.h[k] = mr.h[k] = 0.f;
        }
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            if (s >= st.n) break;
            if (want_x) {
                if ((st.first >> s) & 1) mf.f = 1;
                enter(s, mf.h);
                advance(s, mf.h);
            }
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float a = (float)gv[s].e[SHARED ? 0 : k];
                mf.a[k] *= p.blend ? 1.0f - a : a;
            }
        }
#pragma unroll
        for (int s = SEG - 1; s >= 0; --s) {
            if (s >= st.n) continue;
            float lam[VEC];
            if ((st.final >> s) & 1) mr.f = 1;
            retreat(s, mr.h, lam);
        }
#pragma unroll
        for (int k = 0; k < VEC; ++k) mr.a[k] = mf.a[k];
        if (want_x) nm_s_wave_scan<VEC, 1>(mf, bf, lane, cl);
        nm_s_wave_scan<VEC, -1>(mr, br, lane, cl);
        if (want_x && lane >= 64 - cl) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                sh_a[buf][wave][cx * VEC + k] = mf.a[k];
                sh_h[buf][wave][cx * VEC + k] = mf.h[k];
            }
            if (lane == 63) sh_f[buf][wave] = mf.f;
        }
        if (lane < cl) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                sh_b[buf][wave][cx * VEC + k] = mr.a[k];
                sh_r[buf][wave][cx * VEC + k] = mr.h[k];
            }
            if (lane == 0) sh_e[buf][wave] = mr.f;
        }
        __syncthreads();
        float f[VEC], hp[SEG][VEC];
#pragma unroll
        for (int w = 3; w >= 0; --w) {
            NmMap<VEC> mw;
            mw.f = sh_e[buf][w];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                mw.a[k] = sh_b[buf][w][cx * VEC + k];
                mw.h[k] = sh_r[buf][w][cx * VEC + k];
                if (w == wave) f[k] = flow[k];
            }
            nm_s_apply(mw, flow);
            if (p.map_only) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) total.a[k] = total.f || mw.f ? 0.f : total.a[k] * mw.a[k];
                total.f |= mw.f;
            }
        }
        if (p.map_only) continue;
        nm_s_apply(br, f);
        if (want_x) {
            float h[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) h[k] = p.keep[(c * tiles_per_chunk + j) * p.D + ch + k];
#pragma unroll
            for (int w = 0; w < 3; ++w) {
                NmMap<VEC> mw;
                mw.f = sh_f[buf][w];
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    mw.a[k] = sh_a[buf][w][cx * VEC + k];
                    mw.h[k] = sh_h[buf][w][cx * VEC + k];
                }
                if (w < wave) nm_s_apply(mw, h);
            }
            nm_s_apply(bf, h);
#pragma unroll
            for (int s = 0; s < SEG; ++s) {
                if (s >= st.n) break;
                enter(s, h);
#pragma unroll
                for (int k = 0; k < VEC; ++k) hp[s][k] = h[k];
                advance(s, h);
            }
        }
#pragma unroll
        for (int s = SEG - 1; s >= 0; --s) {
            if (s >= st.n) continue;
            float lam[VEC], o[VEC];
            retreat(s, f, lam);
            if (p.dx) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) o[k] = p.blend ? (float)gv[s].e[SHARED ? 0 : k] * lam[k] : lam[k];
                if (st.seq[s] < 0) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) o[k] = 0.f;
                }
                nm_s_store<DX, VEC>((TX*)p.dx + (row0 + s * step) * p.D + ch, o);
            }
            if (want_x) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    o[k] = lam[k] * (p.blend ? (float)xv[s].e[k] - hp[s][k] : hp[s][k]);
                    if (st.seq[s] < 0) o[k] = 0.f;
                }
                if constexpr (SHARED) {
                    float sum = 0.f;
#pragma unroll
                    for (int k = 0; k < VEC; ++k) sum += ch + k >= own ? o[k] : 0.f;     // (own channels only)
                    hp[s][0] = sum;
                } else {
                    nm_s_store<DG, VEC>((TG*)p.dgate + (row0 + s * step) * p.D + ch, o);
                }
            }
            if (p.dh0 && ((st.first >> s) & 1) && st.seq[s] >= 0) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) p.dh0[(long long)st.seq[s] * p.D + ch + k] = f[k];
            }
        }
        if constexpr (SHARED) {
            if (want_x) {                // sum over the channel lanes (all lanes of the wave take part)
#pragma unroll
                for (int s = 0; s < SEG; ++s) {
                    float sum = s < st.n ? hp[s][0] : 0.f;
                    for (int o = 1; o < cl; o <<= 1) sum += __shfl_xor(sum, o);
                    if (s < st.n && cx == 0) {
                        if (p.dgate_part) p.dgate_part[(long long)blk * p.L + row0 + s * step] = sum;
                        else ((TG*)p.dgate)[row0 + s * step] = (TG)sum;
                    }
                }
            }
        }
    }
    if (p.map_only && tl == 0) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            p.map_a[c * p.D + ch + k] = total.a[k];
            p.map_h[c * p.D + ch + k] = flow[k];
        }
        if (blk == 0 && cx == 0) p.map_f[c] = total.f || cut;
    }
}

// maps of the ranges -> the state before every range (DIR = 1), or the flow after it (-1).  8 channels x 32 lanes in time, 16 ranges each.
template <int DIR>
__global__ __launch_bounds__(NM_S_THREADS) void nm_scan_carry_kernel(const float* __restrict__ map_a, const float* __restrict__ map_h, const int* __restrict__ map_f, long long n,
                                                                     int D, float* __restrict__ carry) {
    __shared__ float sh_a[2][4][8], sh_h[2][4][8];
    __shared__ int sh_f[2][4];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, cx = t & 7, tl = t >> 3;
    int ch = blockIdx.x * 8 + cx;
    if (ch >= D) ch = D - 1;
    float state = 0.f;
    int buf = 0;
    for (long long b = 0; b < n; b += 512, buf ^= 1) {
        NmMap<1> m, before, v[16];
        m.a[0] = 1.f; m.h[0] = 0.f; m.f = 0;
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            const long long i = b + tl * 16 + s, c = DIR > 0 ? i : n - 1 - i;
            v[s].a[0] = 1.f; v[s].h[0] = 0.f; v[s].f = 0;
            if (i < n) { v[s].a[0] = map_a[c * D + ch]; v[s].h[0] = map_h[c * D + ch]; v[s].f = map_f[c]; }
        }
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            nm_s_apply(v[s], m.h);
            m.a[0] *= v[s].a[0];
            m.f |= v[s].f;
        }
        nm_s_wave_scan<1, 1>(m, before, lane, 8);
        if (lane >= 56) {
            sh_a[buf][wave][cx] = m.a[0];
            sh_h[buf][wave][cx] = m.h[0];
            if (lane == 63) sh_f[buf][wave] = m.f;
        }
        __syncthreads();
        float h[1] = {0.f}, all[1] = {state};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w == wave) h[0] = all[0];
            NmMap<1> mw;
            mw.a[0] = sh_a[buf][w][cx]; mw.h[0] = sh_h[buf][w][cx]; mw.f = sh_f[buf][w];
            nm_s_apply(mw, all);
        }
        state = all[0];
        nm_s_apply(before, h);
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            const long long i = b + tl * 16 + s, c = DIR > 0 ? i : n - 1 - i;
            if (i < n) carry[c * D + ch] = h[0];
            nm_s_apply(v[s], h);
        }
    }
}

// packed sequences: the sequence of every row (-1: none), and the result of empty sequences (their state / their cotangent passes through).
__global__ __launch_bounds__(256) void nm_scan_rows_kernel(const int* __restrict__ cu, long long S, long long L, int D, const float* __restrict__ src, float* __restrict__ dst,
                                                           int* __restrict__ seg) {
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    if (t < L) seg[t] = nm_scan_sequence(cu, S, t);
    if (dst && t < S * D) {
        const long long s = t / D;
        if (cu[s + 1] <= cu[s]) dst[t] = src ? src[t] : 0.f;
    }
}

// what passes through a batch without a single step
__global__ __launch_bounds__(256) void nm_scan_pass_kernel(const float* __restrict__ src, float* __restrict__ dst, long long n) {
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    if (t < n) dst[t] = src ? src[t] : 0.f;
}

// shared gate over several channel blocks: sum of the blocks' parts, in order
template <int DG>
__global__ __launch_bounds__(256) void nm_scan_gate_sum_kernel(const float* __restrict__ part, int blocks, long long L, typename NmType<DG>::elem* __restrict__ dgate) {
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    if (t >= L) return;
    float s = 0.f;
    for (int b = 0; b < blocks; ++b) s += part[(long long)b * L + t];
    dgate[t] = (typename NmType<DG>::elem)s;
}

// ------------------------------------------------------------------------------------------------ plans and launches
static inline long long nm_s_up(long long a, long long b) { return (a + b - 1) / b; }
static inline size_t nm_s_align(size_t x) { return (x + 255) & ~(size_t)255; }

struct NmScanPlan {
    int vec, seg, cl_log2, blocks;
    bool split;                          // ranges cut sequences: maps and carried states
    long long tile, chunk, chunks, tiles_per_chunk;
    size_t off_seg, off_a, off_h, off_f, off_carry, off_part, bytes;
};

#define NM_S_FILL 1024       // workgroups that fill the chip

static NmScanPlan nm_s_plan(long long L, long long S, int D, int dtype, bool packed, bool part) {
    NmScanPlan p;
    p.vec = D >= 4 ? 4 : dtype == NM_F32 && D == 3 ? 3 : 1;
    p.seg = p.vec == 4 ? 4 : 8;
    const int groups = (int)nm_s_up(D, p.vec);
    p.cl_log2 = 0;
    while ((1 << p.cl_log2) < groups && p.cl_log2 < 6) ++p.cl_log2;
    p.blocks = (int)nm_s_up(groups, 1 << p.cl_log2);
    p.tile = (NM_S_THREADS >> p.cl_log2) * p.seg;
    const long long T = packed || S == 0 ? 0 : L / S;
    p.split = true;
    if (!packed) {
        const long long whole = T >= p.tile ? T : p.tile / (T > 0 ? T : 1) * T;       // steps of the sequences that fit a tile, or of one
        if (T <= p.tile || nm_s_up(L, whole) * p.blocks >= NM_S_FILL / 2) {
            p.split = false;
            p.chunk = whole;
        }
    }
    if (p.split) p.chunk = nm_s_up(nm_s_up(L, p.tile) * p.blocks, NM_S_FILL) * p.tile;
    if (p.chunk < 1) p.chunk = 1;
    p.chunks = nm_s_up(L, p.chunk);
    if (p.chunks <= 1) p.split = false;
    p.tiles_per_chunk = nm_s_up(p.chunk, p.tile);
    size_t off = 0;
    p.off_seg = off;
    if (packed) off += nm_s_align((size_t)L * 4);
    p.off_a = off;
    const size_t map = p.split ? nm_s_align((size_t)p.chunks * D * 4) : 0;
    off += map;
    p.off_h = off;
    off += map;
    p.off_carry = off;
    off += map;
    p.off_f = off;
    if (p.split) off += nm_s_align((size_t)p.chunks * 4);
    p.off_part = off;
    if (part && p.blocks > 1) off += nm_s_align((size_t)p.blocks * L * 4);
    p.bytes = off;
    return p;
}

#define NM_S_LAUNCH(KERNEL, DX, DG, VEC, SEG)                                                                                     \
    do {                                                                                                                          \
        if (shared) hipLaunchKernelGGL((KERNEL<DX, DG, VEC, SEG, true>), grid, dim3(NM_S_THREADS), 0, stream, a);                  \
        else hipLaunchKernelGGL((KERNEL<DX, DG, VEC, SEG, false>), grid, dim3(NM_S_THREADS), 0, stream, a);                        \
    } while (0)
#define NM_S_PICK_VEC(KERNEL, DX, DG)                                                                                             \
    do {                                                                                                                          \
        if (pl.vec == 4) NM_S_LAUNCH(KERNEL, DX, DG, 4, 4);                                                                       \
        else NM_S_LAUNCH(KERNEL, DX, DG, 1, 8);                                                                                   \
    } while (0)
#define NM_S_PICK(KERNEL)                                                                                                         \
    do {                                                                                                                          \
        if (dtype == NM_F32 && pl.vec == 3) NM_S_LAUNCH(KERNEL, NM_F32, NM_F32, 3, 8);                                            \
        else if (dtype == NM_F32) NM_S_PICK_VEC(KERNEL, NM_F32, NM_F32);                                                          \
        else if (dtype == NM_F16 && gate_dtype == NM_F32) NM_S_PICK_VEC(KERNEL, NM_F16, NM_F32);                                  \
        else if (dtype == NM_F16) NM_S_PICK_VEC(KERNEL, NM_F16, NM_F16);                                                          \
        else if (gate_dtype == NM_F32) NM_S_PICK_VEC(KERNEL, NM_BF16, NM_F32);                                                    \
        else NM_S_PICK_VEC(KERNEL, NM_BF16, NM_BF16);                                                                             \
    } while (0)

static int nm_s_check(const char* who, int64_t L, int64_t S, int64_t D, int dtype, int gate_dtype, bool packed) {
    if (!nm_dtype_ok(dtype) || (gate_dtype != dtype && gate_dtype != NM_F32)) return nm_fail("%s: unknown element types %d / %d (the gate is fp32 or of the values' type)", who, dtype, gate_dtype);
    if (L < 0 || S < 0 || D < 0 || L > 0x7fffffffLL || S > 0x7fffffffLL || D > (1 << 20)) return nm_fail("%s: bad sizes L=%lld S=%lld D=%lld", who, (long long)L, (long long)S, (long long)D);
    if (!packed && (S == 0 ? L != 0 : L % S != 0)) return nm_fail("%s: %lld steps are not %lld sequences of equal length", who, (long long)L, (long long)S);
    return 0;
}

static void nm_s_fill(NmScanArgs& a, const NmScanPlan& pl, const void* gate, const void* x, const float* h0, const int* cu, int64_t L, int64_t S, int64_t D, int reverse,
                      int blend, char* ws) {
    a.gate = gate; a.x = x; a.h0 = h0; a.cu = cu;
    a.seg = cu ? (const int*)(ws + pl.off_seg) : nullptr;
    a.L = L; a.S = S; a.chunk = pl.chunk; a.T = cu || S == 0 ? 1u : (unsigned)(L / S); a.D = (int)D;
    a.reverse = reverse ? 1 : 0; a.blend = blend ? 1 : 0; a.cl_log2 = pl.cl_log2; a.blocks = pl.blocks;
    if (pl.split) {
        a.map_a = (float*)(ws + pl.off_a); a.map_h = (float*)(ws + pl.off_h); a.map_f = (int*)(ws + pl.off_f);
    }
}

extern "C" {

int64_t nm_scan_workspace_bytes(int64_t L, int64_t S, int64_t D, int dtype, int packed, int backward) {
    if (nm_s_check("nm_scan_workspace_bytes", L, S, D, dtype, dtype, packed != 0)) return -1;
    return L == 0 || D == 0 ? 0 : (int64_t)nm_s_plan(L, S, (int)D, dtype, packed != 0, backward != 0).bytes;
}

int64_t nm_scan_keep_elems(int64_t L, int64_t S, int64_t D, int dtype, int packed) {
    if (nm_s_check("nm_scan_keep_elems", L, S, D, dtype, dtype, packed != 0)) return -1;
    if (L == 0 || D == 0) return 0;
    const NmScanPlan pl = nm_s_plan(L, S, (int)D, dtype, packed != 0, false);
    return pl.chunks * pl.tiles_per_chunk * D;
}

int nm_scan_forward(const void* gate, int gate_dtype, int shared_gate, const void* x, int dtype, const float* h0, const int32_t* cu_seqlens, int64_t L, int64_t S, int64_t D,
                    int reverse, int blend, void* states, float* last, float* keep, void* workspace, int64_t workspace_bytes, nm_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    const bool packed = cu_seqlens != nullptr, shared = shared_gate != 0;
    if (nm_s_check("nm_scan_forward", L, S, D, dtype, gate_dtype, packed)) return 1;
    if (D == 0 || (L == 0 && S == 0)) return 0;
    if ((L > 0 && (!gate || !x)) || (S > 0 && !last)) return nm_fail("nm_scan_forward: NULL argument");
    if (L == 0) {                        // every sequence is empty: its state passes through
        hipLaunchKernelGGL(nm_scan_pass_kernel, dim3((unsigned)nm_s_up(S * D, 256)), dim3(256), 0, stream, h0, last, (long long)(S * D));
        NM_LAUNCH_CHECK();
        return 0;
    }
    const NmScanPlan pl = nm_s_plan(L, S, (int)D, dtype, packed, false);
    if ((size_t)(workspace_bytes < 0 ? 0 : workspace_bytes) < pl.bytes || (pl.bytes > 0 && !workspace)) return nm_fail("nm_scan_forward: workspace too small");
    if (pl.chunks * pl.blocks > 0x7fffffffLL) return nm_fail("nm_scan_forward: %lld steps x %lld channels exceed one launch", (long long)L, (long long)D);
    char* ws = (char*)workspace;
    if (packed) {
        const long long n = L > S * D ? L : S * D;
        hipLaunchKernelGGL(nm_scan_rows_kernel, dim3((unsigned)nm_s_up(n, 256)), dim3(256), 0, stream, cu_seqlens, (long long)S, (long long)L, (int)D, h0, last, (int*)(ws + pl.off_seg));
    }
    NmScanArgs a = {};
    nm_s_fill(a, pl, gate, x, h0, cu_seqlens, L, S, D, reverse, blend, ws);
    a.states = states; a.last = last; a.keep = keep;
    const dim3 grid((unsigned)(pl.chunks * pl.blocks));
    if (pl.split) {
        float* carry = (float*)(ws + pl.off_carry);
        a.map_only = 1;
        NM_S_PICK(nm_scan_forward_kernel);
        hipLaunchKernelGGL(nm_scan_carry_kernel<1>, dim3((unsigned)nm_s_up(D, 8)), dim3(NM_S_THREADS), 0, stream, a.map_a, a.map_h, a.map_f, pl.chunks, (int)D, carry);
        a.map_only = 0;
        a.carry = carry;
    }
    NM_S_PICK(nm_scan_forward_kernel);
    NM_LAUNCH_CHECK();
    return 0;
}

int nm_scan_backward(const void* gate, int gate_dtype, int shared_gate, const void* x, int dtype, const float* h0, const int32_t* cu_seqlens, int64_t L, int64_t S, int64_t D,
                     int reverse, int blend, const float* keep, const void* g_states, const float* g_last, void* dgate, void* dx, float* dh0, void* workspace,
                     int64_t workspace_bytes, nm_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    const bool packed = cu_seqlens != nullptr, shared = shared_gate != 0;
    if (nm_s_check("nm_scan_backward", L, S, D, dtype, gate_dtype, packed)) return 1;
    if (D == 0 || (L == 0 && S == 0) || (!dgate && !dx && !dh0)) return 0;
    if (L > 0 && (!gate || (dgate && (!x || !keep)))) return nm_fail("nm_scan_backward: NULL argument");
    if (L == 0) {
        if (!dh0) return 0;
        hipLaunchKernelGGL(nm_scan_pass_kernel, dim3((unsigned)nm_s_up(S * D, 256)), dim3(256), 0, stream, g_last, dh0, (long long)(S * D));
        NM_LAUNCH_CHECK();
        return 0;
    }
    const NmScanPlan pl = nm_s_plan(L, S, (int)D, dtype, packed, true);
    if ((size_t)(workspace_bytes < 0 ? 0 : workspace_bytes) < pl.bytes || (pl.bytes > 0 && !workspace)) return nm_fail("nm_scan_backward: workspace too small");
    if (pl.chunks * pl.blocks > 0x7fffffffLL) return nm_fail("nm_scan_backward: %lld steps x %lld channels exceed one launch", (long long)L, (long long)D);
    char* ws = (char*)workspace;
    if (packed) {
        const long long n = L > S * D ? L : S * D;
        hipLaunchKernelGGL(nm_scan_rows_kernel, dim3((unsigned)nm_s_up(n, 256)), dim3(256), 0, stream, cu_seqlens, (long long)S, (long long)L, (int)D, g_last, dh0, (int*)(ws + pl.off_seg));
    }
    NmScanArgs a = {};
    nm_s_fill(a, pl, gate, x, h0, cu_seqlens, L, S, D, reverse, blend, ws);
    a.keep = const_cast<float*>(keep); a.g = g_states; a.g_last = g_last; a.dgate = dgate; a.dx = dx; a.dh0 = dh0;
    const bool parts = shared && dgate && pl.blocks > 1;
    if (parts) a.dgate_part = (float*)(ws + pl.off_part);
    const dim3 grid((unsigned)(pl.chunks * pl.blocks));
    if (pl.split) {
        float* carry = (float*)(ws + pl.off_carry);
        a.map_only = 1;
        NM_S_PICK(nm_scan_backward_kernel);
        hipLaunchKernelGGL(nm_scan_carry_kernel<-1>, dim3((unsigned)nm_s_up(D, 8)), dim3(NM_S_THREADS), 0, stream, a.map_a, a.map_h, a.map_f, pl.chunks, (int)D, carry);
        a.map_only = 0;
        a.carry = carry;
    }
    NM_S_PICK(nm_scan_backward_kernel);
    if (parts) {
        const dim3 g2((unsigned)nm_s_up(L, 256));
        if (gate_dtype == NM_F32) hipLaunchKernelGGL(nm_scan_gate_sum_kernel<NM_F32>, g2, dim3(256), 0, stream, a.dgate_part, pl.blocks, (long long)L, (float*)dgate);
        else if (gate_dtype == NM_F16) hipLaunchKernelGGL(nm_scan_gate_sum_kernel<NM_F16>, g2, dim3(256), 0, stream, a.dgate_part, pl.blocks, (long long)L, (_Float16*)dgate);
        else hipLaunchKernelGGL(nm_scan_gate_sum_kernel<NM_BF16>, g2, dim3(256), 0, stream, a.dgate_part, pl.blocks, (long long)L, (__bf16*)dgate);
    }
    NM_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
