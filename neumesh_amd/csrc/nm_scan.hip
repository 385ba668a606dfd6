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
// states that the forward pass kept at every tile's start: 4 bytes per channel and tile instead of a second read of rounded states; sequences that fit a
// tile keep none.  Sequences of one step (a state carried from call to call) have a kernel of their own, nm_scan_step_kernel.
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
    int D, reverse, blend, cl_log2, blocks;
    void* states;                        // [L, D] or NULL
    float* last;                         // [S, D]
    float* keep; int keep_steps;         // states before every keep_steps-th step, [chunks][pieces][D] counted from a range's start, or (keep_seq)
    int pieces;                          // kept states per range or sequence
    int keep_seq;                        // [S][pieces][D] from a sequence's start, in the order of the recurrence; or NULL
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

// Where a thread's steps lie: step s is row `row` + `lane` + s, or - s.  `row` is uniform over the workgroup and `lane` within the tile, so that an address is
// a scalar base and a 32-bit offset (tile x D elements stay below 2^30).
struct NmPlace {
    long long row;
    unsigned lane;
    int reverse;
};
template <typename T> struct NmRow {
    char* base; long long stride; unsigned off;
    __device__ __forceinline__ T* at(int s) const { return (T*)(base + s * stride + (size_t)off); }
};
template <typename T>
__device__ __forceinline__ NmRow<T> nm_s_rows(T* base, const NmPlace& w, int D, unsigned ch) {
    return {(char*)(base + w.row * D), (w.reverse ? -1LL : 1LL) * D * (long long)sizeof(T), (w.lane * (unsigned)D + ch) * (unsigned)sizeof(T)};
}
// A thread's n <= SEG consecutive steps of VEC channels, a vector per row.
template <int DT, int VEC, int SEG>
__device__ __forceinline__ void nm_s_load_steps(const typename NmType<DT>::elem* base, const NmPlace& w, int D, int ch, int n, NmVec<DT, VEC> (&v)[SEG]) {
    const NmRow<const typename NmType<DT>::elem> r = nm_s_rows(base, w, D, ch);
    if (n == SEG) {
#pragma unroll
        for (int s = 0; s < SEG; ++s) v[s] = nm_s_load<DT, VEC>(r.at(s));
    } else {
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            v[s] = {};
            if (s < n) v[s] = nm_s_load<DT, VEC>(r.at(s));
        }
    }
}
// The same where a row has exactly VEC elements, so that the steps are one stretch of memory: read as such, in descending order if the recurrence runs
// backwards.
template <int DT, int VEC, int SEG>
__device__ __forceinline__ void nm_s_load_whole(const typename NmType<DT>::elem* base, const NmPlace& at, int n, NmVec<DT, VEC> (&v)[SEG]) {
    if (n < SEG) {
        nm_s_load_steps<DT, VEC, SEG>(base, at, VEC, 0, n, v);
        return;
    }
    NmVec<DT, VEC * SEG> w;
    __builtin_memcpy(&w, nm_s_rows(base, at, VEC, 0).at(at.reverse ? SEG - 1 : 0), sizeof(w));
    if (at.reverse) {                    // (uniform)
#pragma unroll
        for (int s = 0; s < SEG; ++s)
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[s].e[k] = w.e[(SEG - 1 - s) * VEC + k];
    } else {
#pragma unroll
        for (int s = 0; s < SEG; ++s)
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[s].e[k] = w.e[s * VEC + k];
    }
}
// ... by the whole workgroup: a tile of 256 SEG steps from step b on is one stretch of memory, read in 16-byte pieces side by side and dealt out through
// LDS (PIECES per thread, at an odd stride from three on: four workgroups per CU).  Pieces beyond the array's ends are left out; what lies beyond the workgroup's range is not used.
template <int DT, int VEC, int SEG> struct NmStage {
    static constexpr int PIECES = SEG * VEC * (int)sizeof(typename NmType<DT>::elem) / 16, STRIDE = PIECES < 3 ? PIECES : PIECES | 1;
    static_assert(SEG * VEC * sizeof(typename NmType<DT>::elem) % 16 == 0, "whole pieces per thread");
};
template <int DT, int VEC, int SEG>
__device__ __forceinline__ void nm_s_stage(const typename NmType<DT>::elem* base, long long b, long long L, int reverse, uint4* lds, int t) {
    typedef typename NmType<DT>::elem T;
    typedef NmStage<DT, VEC, SEG> G;
    constexpr int E = 16 / (int)sizeof(T);
    const long long first = (reverse ? L - b - 256LL * SEG : b) * VEC, end = L * VEC;      // element of memory that piece 0 starts with
#pragma unroll
    for (int i = 0; i < G::PIECES; ++i) {
        const int j = t + 256 * i;
        const long long e0 = first + (long long)j * E;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (e0 >= 0 && e0 + E <= end) {
            __builtin_memcpy(&v, base + e0, 16);
        } else if (e0 > -E && e0 < end) {
            T x[E];
#pragma unroll
            for (int k = 0; k < E; ++k) x[k] = e0 + k >= 0 && e0 + k < end ? base[e0 + k] : (T)0.f;
            __builtin_memcpy(&v, x, 16);
        }
        lds[j / G::PIECES * G::STRIDE + j % G::PIECES] = v;
    }
}
template <int DT, int VEC, int SEG>
__device__ __forceinline__ void nm_s_unstage(const uint4* lds, int reverse, int t, NmVec<DT, VEC> (&v)[SEG]) {
    typedef NmStage<DT, VEC, SEG> G;
    NmVec<DT, VEC * SEG> w;
    __builtin_memcpy(&w, lds + (reverse ? 255 - t : t) * G::STRIDE, sizeof(w));
    if (reverse) {                       // (uniform)
#pragma unroll
        for (int s = 0; s < SEG; ++s)
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[s].e[k] = w.e[(SEG - 1 - s) * VEC + k];
    } else {
#pragma unroll
        for (int s = 0; s < SEG; ++s)
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[s].e[k] = w.e[s * VEC + k];
    }
}
template <int DT, int VEC, int SEG>
__device__ __forceinline__ void nm_s_store_whole(typename NmType<DT>::elem* base, const NmPlace& at, int n, const float (&f)[SEG][VEC]) {
    typedef typename NmType<DT>::elem T;
    if (n == SEG) {
        NmVec<DT, VEC * SEG> w;
#pragma unroll
        for (int s = 0; s < SEG; ++s)
#pragma unroll
            for (int k = 0; k < VEC; ++k) w.e[s * VEC + k] = (T)(at.reverse ? f[SEG - 1 - s][k] : f[s][k]);
        __builtin_memcpy(nm_s_rows(base, at, VEC, 0).at(at.reverse ? SEG - 1 : 0), &w, sizeof(w));
    } else {
#pragma unroll
        for (int s = 0; s < SEG; ++s)
            if (s < n) nm_s_store<DT, VEC>(nm_s_rows(base, at, VEC, 0).at(s), f[s]);
    }
}

// the affine map h -> A h + H of a stretch of steps; F: it starts anew, whatever came before.  AV: a shared gate's factor is one for all channels.
template <int VEC, int AV> struct NmMap { float a[AV], h[VEC]; int f; };

template <int VEC, int AV>
__device__ __forceinline__ void nm_s_identity(NmMap<VEC, AV>& m) {
#pragma unroll
    for (int k = 0; k < AV; ++k) m.a[k] = 1.f;
#pragma unroll
    for (int k = 0; k < VEC; ++k) m.h[k] = 0.f;
    m.f = 0;
}
// `m` applied after the state `s`
template <int VEC, int AV>
__device__ __forceinline__ void nm_s_apply(const NmMap<VEC, AV>& m, float (&s)[VEC]) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) s[k] = m.f ? m.h[k] : fmaf(m.a[AV == 1 ? 0 : k], s[k], m.h[k]);
}
// the map `m` followed by `n`, in m
template <int VEC, int AV>
__device__ __forceinline__ void nm_s_then(NmMap<VEC, AV>& m, const NmMap<VEC, AV>& n) {
    nm_s_apply(n, m.h);
#pragma unroll
    for (int k = 0; k < AV; ++k) m.a[k] = n.f ? 0.f : m.a[k] * n.a[k];
    m.f |= n.f;
}
template <int VEC, int AV>
__device__ __forceinline__ void nm_s_from_lane(const NmMap<VEC, AV>& m, int src, NmMap<VEC, AV>& p) {
    p.f = __shfl(m.f, src);
#pragma unroll
    for (int k = 0; k < AV; ++k) p.a[k] = __shfl(m.a[k], src);
#pragma unroll
    for (int k = 0; k < VEC; ++k) p.h[k] = __shfl(m.h[k], src);
}

// exclusive scan of the lanes' maps in time order within a wave (DIR = 1: lower lanes come first, -1: higher lanes); the wave's total is left in the
// last lane's `m`.  Lanes of one time are neighbours: exchanges go over multiples of cl.
template <int VEC, int AV, int DIR>
__device__ __forceinline__ void nm_s_wave_scan(NmMap<VEC, AV>& m, NmMap<VEC, AV>& before, int lane, int cl) {
    for (int o = cl; o < 64; o <<= 1) {
        NmMap<VEC, AV> p;
        const int src = lane - DIR * o;
        nm_s_from_lane(m, src & 63, p);
        if (src >= 0 && src < 64 && !m.f) {                  // p followed by m
#pragma unroll
            for (int k = 0; k < VEC; ++k) m.h[k] = fmaf(m.a[AV == 1 ? 0 : k], p.h[k], m.h[k]);
#pragma unroll
            for (int k = 0; k < AV; ++k) m.a[k] *= p.a[k];
            m.f = p.f;
        }
    }
    const int src = lane - DIR * cl;
    nm_s_from_lane(m, src & 63, before);
    if (src < 0 || src >= 64) nm_s_identity(before);
}

// the maps of the four waves, per channel lane
// (fewer than four channels: one lane holds a whole row)
template <int VEC, int AV> struct NmShared { float a[4][(VEC < 4 ? 1 : 64) * AV], h[4][(VEC < 4 ? 1 : 64) * VEC]; int f[4]; };

template <int VEC, int AV>
__device__ __forceinline__ void nm_s_put(NmShared<VEC, AV>& sh, int wave, int cx, const NmMap<VEC, AV>& m) {
#pragma unroll
    for (int k = 0; k < AV; ++k) sh.a[wave][cx * AV + k] = m.a[k];
#pragma unroll
    for (int k = 0; k < VEC; ++k) sh.h[wave][cx * VEC + k] = m.h[k];
    if (cx == 0) sh.f[wave] = m.f;
}
template <int VEC, int AV>
__device__ __forceinline__ void nm_s_get(const NmShared<VEC, AV>& sh, int wave, int cx, NmMap<VEC, AV>& m) {
#pragma unroll
    for (int k = 0; k < AV; ++k) m.a[k] = sh.a[wave][cx * AV + k];
#pragma unroll
    for (int k = 0; k < VEC; ++k) m.h[k] = sh.h[wave][cx * VEC + k];
    m.f = sh.f[wave];
}

// What a thread knows of its steps: bit s of first / final: the step is its sequence's first / last; none: it belongs to no sequence.
struct NmSteps {
    unsigned first, final, none;
    int n, q;                            // n: steps of this thread; q, pos: sequence of step 0 in the order of the recurrence, and its place in it
    unsigned pos;                        // (equal lengths)
    int q_first, q_final;                // sequence of the first bit of first / final whose step belongs to one
};
// packed: the sequences of a thread's steps and of its neighbours.  Asked for before the operands, so that start values can be asked for while those come
template <int SEG> struct NmSeqs { NmVec<NM_F32, 1> v[SEG]; int prev, next; };      // (bits of the sequence numbers)

template <int SEG>
__device__ __forceinline__ void nm_s_seqs(const NmScanArgs& p, const NmPlace& at, int n, long long i0, NmSeqs<SEG>& w) {
    w.prev = w.next = -2;
#pragma unroll
    for (int s = 0; s < SEG; ++s) w.v[s] = {};
    if (!p.seg || n == 0) return;
    nm_s_load_whole<NM_F32, 1, SEG>((const float*)p.seg, at, n, w.v);
    if (i0 > 0) w.prev = p.seg[p.reverse ? p.L - i0 : i0 - 1];
    if (i0 + n < p.L) w.next = p.seg[p.reverse ? p.L - 1 - (i0 + n) : i0 + n];
}

template <int SEG>
__device__ __forceinline__ NmSteps nm_s_steps(const NmScanArgs& p, const NmSeqs<SEG>& w, int n, unsigned off, int q0) {
    NmSteps t;
    t.first = t.final = t.none = 0u;
    t.n = n;
    t.q = t.q_first = t.q_final = 0;
    t.pos = 0;
    if (p.seg) {
        if (n == 0) return t;
        int prev = w.prev;
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            if (s >= n) continue;
            const int q = __float_as_int(w.v[s].e[0]), after = s + 1 < n ? __float_as_int(w.v[s + 1 < SEG ? s + 1 : s].e[0]) : w.next;
            if (prev != q || q < 0) {
                if (!(t.first & ~t.none)) t.q_first = q;
                t.first |= 1u << s;
            }
            if (after != q || q < 0) {
                if (!(t.final & ~t.none)) t.q_final = q;
                t.final |= 1u << s;
            }
            if (q < 0) t.none |= 1u << s;
            prev = q;
        }
        return t;
    }
    const unsigned valid = (1u << n) - 1u;
    const unsigned q = off / p.T, pos = off - q * p.T;       // off: steps since the start of sequence q0
    t.q = q0 + (int)q;
    t.pos = pos;
    t.q_final = p.reverse ? (int)p.S - 1 - t.q : t.q;
    t.q_first = t.q_final + (pos == 0 ? 0 : p.reverse ? -1 : 1);
    if (p.T >= SEG) {                    // one border at most
        const unsigned k = p.T - pos;    // steps up to it
        t.first = (pos == 0 ? 1u : 0u) | (k < SEG ? 1u << k : 0u);
        t.final = k <= SEG ? 1u << (k - 1) : 0u;
    } else {
        unsigned at = pos;
        for (int s = 0; s < SEG; ++s) {
            if (at == 0) t.first |= 1u << s;
            if (++at == p.T) {
                t.final |= 1u << s;
                at = 0;
            }
        }
    }
    t.first &= valid;
    t.final &= valid;
    return t;
}
// sequence of step s, which is a bit of `border` (first or final); `q`: that of the first such bit.  Threads with more of them look the others up.
__device__ __forceinline__ long long nm_s_sequence(const NmScanArgs& p, const NmSteps& t, unsigned border, int q, long long i0, int s) {
    if (!(border & ~t.none & ((1u << s) - 1u))) return q;
    if (p.seg) return p.seg[p.reverse ? p.L - 1 - (i0 + s) : i0 + s];
    const int b = t.q + __popc(t.first & ((2u << s) - 2u));
    return p.reverse ? p.S - 1 - b : b;
}

// the value (src [S, D], NULL: 0) with which the sequence of a thread's first border starts
template <int VEC>
__device__ __forceinline__ void nm_s_start(const NmScanArgs& p, const float* src, const NmSteps& t, unsigned border, int q, int ch, float (&v)[VEC]) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = 0.f;
    if (src && (border & ~t.none)) {
        const NmVec<NM_F32, VEC> f = nm_s_load<NM_F32, VEC>(src + (long long)q * p.D + ch);
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = f.e[k];
    }
}
// where bit s of `border` is set: the start value instead of v
template <int VEC>
__device__ __forceinline__ void nm_s_enter(const NmScanArgs& p, const float* src, const NmSteps& t, unsigned border, int q, const float (&start)[VEC], long long i0, int s, int ch,
                                           float (&v)[VEC]) {
    const unsigned bit = 1u << s, own = border & ~t.none;
#pragma unroll
    for (int k = 0; k < VEC; ++k) v[k] = border & bit ? (t.none & bit ? 0.f : start[k]) : v[k];
    if (src && (own & bit) && (own & (bit - 1u))) {          // a later border of the same thread
        const float* from = src + nm_s_sequence(p, t, border, q, i0, s) * p.D + ch;
#pragma unroll
        for (int k = 0; k < VEC; ++k) v[k] = from[k];
    }
}

// r and w of a gate a: plain a and 1, blend 1 - a and a
template <int DG>
__device__ __forceinline__ float nm_s_factor(typename NmType<DG>::elem e, int blend) {
    return fmaf(nm_to_float<DG>(e), blend ? -1.0f : 1.0f, blend ? 1.0f : 0.0f);
}
// h -> r h + w x
template <int DX, int DG, int VEC, int AV>
__device__ __forceinline__ void nm_s_step(const NmVec<DG, AV>& g, const NmVec<DX, VEC>& x, int blend, float (&h)[VEC]) {
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        const float a = nm_to_float<DG>(g.e[AV == 1 ? 0 : k]), v = nm_to_float<DX>(x.e[k]);
        h[k] = fmaf(nm_s_factor<DG>(g.e[AV == 1 ? 0 : k], blend), h[k], blend ? a * v : v);
    }
}
// steps beyond a thread's n: gates that leave the state as it is (the other operands are 0 there), so that no later pass has to ask
template <int DG, int AV, int SEG>
__device__ __forceinline__ void nm_s_pad(NmVec<DG, AV> (&g)[SEG], int n, int blend) {
#pragma unroll
    for (int s = 0; s < SEG; ++s)
#pragma unroll
        for (int k = 0; k < AV; ++k) g[s].e[k] = s < n ? g[s].e[k] : nm_from_float<DG>(blend ? 0.f : 1.f);
}

// Operands between two passes over them: what the first pass derived from them (factors, converted values) is not to wait in registers for the second one.
template <typename T, int SEG>
__device__ __forceinline__ void nm_s_forget(T (&v)[SEG]) {
    constexpr int N = (int)sizeof(v) / 4;
    static_assert(sizeof(v) % 4 == 0, "whole registers");
    unsigned w[N];
    __builtin_memcpy(w, &v, sizeof(v));
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(w[i]));
    __builtin_memcpy(&v, w, sizeof(v));
}

#define NM_S_THREADS 256
#define NM_S_MAX_GROUPS (0xffffffffLL / NM_S_THREADS)    // of one launch: its threads are counted in 32 bits
// Steps of a thread.  Forward: as many as 32 .. 64 registers of operands allow (the scan's own instructions are per thread; with 4 steps they bound
// short sequences at 2.4 TB/s).  Backward: three operands and the recomputed states.
template <int VEC, bool SHARED> struct NmSeg {
    static constexpr int F = VEC == 8 ? (SHARED ? 8 : 4) : 8;
    static constexpr int B = VEC == 4 ? 4 : 8;
};

// MAP: only the range's map, from its last sequence start on.
// Measured, main launch: 4 x 16384 x 512 bf16 44 us (201 MB: 4.6 TB/s; maps 25 us, carries 9), 8192 packed sequences of 96 x 32 fp32 60 us (302 MB: 5.0 TB/s;
// maps 20), 32768 x 127 x 3 fp32, last state only, 26 us (67 MB: 2.5 TB/s: two rounds of workgroups of one tile, 38 % of the time instructions and
// the rest latency of loads, lane exchanges and barriers).
template <int DX, int DG, int VEC, bool SHARED, bool MAP>
__global__ __launch_bounds__(NM_S_THREADS) void nm_scan_forward_kernel(NmScanArgs p) {
    typedef typename NmType<DX>::elem TX;
    typedef typename NmType<DG>::elem TG;
    constexpr int AV = SHARED ? 1 : VEC, SEG = NmSeg<VEC, SHARED>::F;
    constexpr bool WHOLE = VEC < 4;
    __shared__ NmShared<VEC, AV> sh[2];
    __shared__ uint4 lds_g[WHOLE ? 256 * NmStage<DG, AV, SEG>::STRIDE : 1], lds_x[WHOLE ? 256 * NmStage<DX, VEC, SEG>::STRIDE : 1];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, cl = 1 << p.cl_log2, cx = t & (cl - 1), tl = t >> p.cl_log2;
    const int tile = (NM_S_THREADS >> p.cl_log2) * SEG;
    const unsigned blk_c = blockIdx.x / (unsigned)p.blocks;
    const long long c = blk_c;
    const int blk = (int)(blockIdx.x - blk_c * (unsigned)p.blocks);
    const long long c0 = c * p.chunk, c1 = c0 + p.chunk < p.L ? c0 + p.chunk : p.L;
    // (channels that would end beyond D are the last VEC: computed twice, written twice with the same value)
    int ch = (blk * cl + cx) * VEC;
    if (ch + VEC > p.D) ch = p.D - VEC;
    const unsigned q0 = p.seg ? 0u : (unsigned)c0 / p.T, pos0 = (unsigned)c0 - q0 * p.T;      // (L < 2^31)

    NmMap<VEC, AV> total;                // MAP: everything before the current tile
    float state[VEC];                    // otherwise: the state before the current tile
    nm_s_identity(total);
#pragma unroll
    for (int k = 0; k < VEC; ++k) state[k] = !MAP && p.carry ? p.carry[c * p.D + ch + k] : 0.f;
    long long b0 = c0;
    if constexpr (MAP) {                 // what comes before the range's last sequence start does not matter
        const long long s0 = p.seg ? nm_scan_reduce_from(p.cu, p.seg[p.reverse ? p.L - c1 : c1 - 1], p.reverse, p.L, c0, c1) : (long long)((unsigned)(c1 - 1) / p.T * p.T);
        if (s0 > c0) b0 = s0;
    }
    int buf = 0;
    for (long long b = b0; b < c1; b += tile, buf ^= 1) {
        const long long i0 = b + tl * SEG;
        const NmPlace at = {p.reverse ? p.L - b - tile : b, (unsigned)(p.reverse ? tile - 1 - tl * SEG : tl * SEG), p.reverse};
        const int n = c1 - i0 >= SEG ? SEG : c1 > i0 ? (int)(c1 - i0) : 0;
        NmVec<DX, VEC> xv[SEG];
        NmVec<DG, AV> gv[SEG];
        NmSeqs<SEG> sq;
        nm_s_seqs(p, at, n, i0, sq);
        if constexpr (WHOLE) {
            __syncthreads();             // (everybody has read the tile before)
            nm_s_stage<DG, AV, SEG>((const TG*)p.gate, b, p.L, p.reverse, lds_g, t);
            nm_s_stage<DX, VEC, SEG>((const TX*)p.x, b, p.L, p.reverse, lds_x, t);
            __syncthreads();
            nm_s_unstage<DG, AV, SEG>(lds_g, p.reverse, t, gv);
            nm_s_unstage<DX, VEC, SEG>(lds_x, p.reverse, t, xv);
        } else {
            if constexpr (SHARED) nm_s_load_whole<DG, 1, SEG>((const TG*)p.gate, at, n, gv);
            else nm_s_load_steps<DG, AV, SEG>((const TG*)p.gate, at, p.D, ch, n, gv);
            nm_s_load_steps<DX, VEC, SEG>((const TX*)p.x, at, p.D, ch, n, xv);
        }
        const NmSteps st = nm_s_steps<SEG>(p, sq, n, (unsigned)(i0 - c0) + pos0, (int)q0);
        if (p.seg && __any(st.none != 0)) {                  // rows of no sequence: operands of 0 keep their states and gradients 0
#pragma unroll
            for (int s = 0; s < SEG; ++s)
                if ((st.none >> s) & 1) {
                    gv[s] = {};
                    xv[s] = {};
                }
        }
        if (n < SEG) {
            nm_s_pad<DG, AV, SEG>(gv, n, p.blend);
            if constexpr (WHOLE) {       // (staged rows beyond the range)
#pragma unroll
                for (int s = 0; s < SEG; ++s)
                    if (s >= n) xv[s] = {};
            }
        }
        float start[VEC];
        nm_s_start(p, p.h0, st, st.first, st.q_first, ch, start);
        // one step: state h -> r h + u
        auto advance = [&](int s, float (&h)[VEC]) {
            nm_s_enter(p, p.h0, st, st.first, st.q_first, start, i0, s, ch, h);
            nm_s_step<DX, DG, VEC, AV>(gv[s], xv[s], p.blend, h);
        };
        NmMap<VEC, AV> m, before;
        nm_s_identity(m);
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            advance(s, m.h);
#pragma unroll
            for (int k = 0; k < AV; ++k) m.a[k] *= nm_s_factor<DG>(gv[s].e[k], p.blend);
        }
        m.f = st.first ? 1 : 0;
        nm_s_wave_scan<VEC, AV, 1>(m, before, lane, cl);
        if (lane >= 64 - cl) nm_s_put(sh[buf], wave, cx, m);
        __syncthreads();                 // (two buffers: a wave that is a tile ahead writes the other one)
        float h[VEC];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            NmMap<VEC, AV> mw;
            nm_s_get(sh[buf], w, cx, mw);
            if constexpr (MAP) {
                nm_s_then(total, mw);
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    if (w == wave) h[k] = state[k];
                nm_s_apply(mw, state);
            }
            __builtin_amdgcn_sched_barrier(0);               // (one wave's map in registers at a time)
        }
        if constexpr (!MAP) {
            nm_s_forget(gv);
            nm_s_forget(xv);
            nm_s_forget(start);
            nm_s_apply(before, h);
            if (p.keep && !p.keep_seq && n > 0 && ((unsigned)(i0 - c0) & (unsigned)(p.keep_steps - 1)) == 0) {
                float* dst = p.keep + (c * p.pieces + (unsigned)(i0 - c0) / (unsigned)p.keep_steps) * p.D + ch;
#pragma unroll
                for (int k = 0; k < VEC; ++k) dst[k] = h[k];
            }
            if (p.states || p.keep_seq || __any(st.final != 0)) {
                float out[WHOLE ? SEG : 1][VEC];
                const NmRow<TX> so = nm_s_rows((TX*)p.states, at, p.D, ch);
#pragma unroll
                for (int s = 0; s < SEG; ++s) {
                    if (p.keep_seq && s < n) {               // (sequences longer than keep_steps: one border in these steps at most)
                        const unsigned left = p.T - st.pos, at_s = (unsigned)s < left ? st.pos + s : s - left;
                        if (at_s > 0 && (at_s & (unsigned)(p.keep_steps - 1)) == 0) {
                            const long long piece = (st.q + ((unsigned)s < left ? 0 : 1)) * (long long)p.pieces + at_s / (unsigned)p.keep_steps;
#pragma unroll
                            for (int k = 0; k < VEC; ++k) p.keep[piece * p.D + ch + k] = h[k];
                        }
                    }
                    advance(s, h);
                    if constexpr (WHOLE) {
#pragma unroll
                        for (int k = 0; k < VEC; ++k) out[s][k] = h[k];
                    } else {
                        if (p.states && s < n) nm_s_store<DX, VEC>(so.at(s), h);
                    }
                    if (((st.final & ~st.none) >> s) & 1) {
                        float* dst = p.last + nm_s_sequence(p, st, st.final, st.q_final, i0, s) * p.D + ch;
#pragma unroll
                        for (int k = 0; k < VEC; ++k) dst[k] = h[k];
                    }
                }
                if constexpr (WHOLE) {
                    if (p.states) nm_s_store_whole<DX, VEC, SEG>((TX*)p.states, at, n, out);
                }
            }
        }
    }
    if (MAP && tl == 0) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            p.map_a[c * p.D + ch + k] = total.a[SHARED ? 0 : k];
            p.map_h[c * p.D + ch + k] = total.h[k];
        }
        if (blk == 0 && cx == 0) p.map_f[c] = total.f || b0 > c0;
    }
}

// MAP: only the range's map of the flow, up to its first sequence end.
// Measured, main launch: 8192 packed sequences of 96 x 32 fp32 with h0 118 us (503 MB: 4.3 TB/s; maps 23), 1 x 32768 x 256 bf16 27 us (84 MB: 3.0 TB/s), 2048 x
// 127 x 32 bf16 with a shared gate 27 us (51 MB: 1.9 TB/s).  Bound by two or three workgroups per CU (163 .. 193 registers): a bound of three for
// all of them spills and costs 35 us instead of 27 for the second.
template <int DX, int DG, int VEC, bool SHARED, bool MAP>
__global__ __launch_bounds__(NM_S_THREADS) void nm_scan_backward_kernel(NmScanArgs p) {
    typedef typename NmType<DX>::elem TX;
    typedef typename NmType<DG>::elem TG;
    constexpr int AV = SHARED ? 1 : VEC, SEG = NmSeg<VEC, SHARED>::B;
    constexpr bool WHOLE = VEC < 4;
    __shared__ NmShared<VEC, AV> sh_r[2], sh_h[MAP ? 1 : 2];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, cl = 1 << p.cl_log2, cx = t & (cl - 1), tl = t >> p.cl_log2;
    const int tile = (NM_S_THREADS >> p.cl_log2) * SEG;
    const unsigned blk_c = blockIdx.x / (unsigned)p.blocks;
    const long long c = blk_c;
    const int blk = (int)(blockIdx.x - blk_c * (unsigned)p.blocks);
    const long long c0 = c * p.chunk;
    long long c1 = c0 + p.chunk < p.L ? c0 + p.chunk : p.L;
    const int own = (blk * cl + cx) * VEC;                   // first channel that is this thread's own (see the forward kernel)
    int ch = own;
    if (ch + VEC > p.D) ch = p.D - VEC;
    const unsigned q0 = p.seg ? 0u : (unsigned)c0 / p.T, pos0 = (unsigned)c0 - q0 * p.T;      // (L < 2^31)

    NmMap<VEC, AV> total;                // MAP: everything after the current tile
    float flow[VEC];                     // otherwise: f of the step after the current tile
    nm_s_identity(total);
#pragma unroll
    for (int k = 0; k < VEC; ++k) flow[k] = !MAP && p.carry ? p.carry[c * p.D + ch + k] : 0.f;
    bool cut = false;
    if constexpr (MAP) {                 // what comes after the range's first sequence end does not matter
        const long long e = p.seg ? nm_scan_reduce_to(p.cu, p.seg[p.reverse ? p.L - 1 - c0 : c0], p.reverse, p.L, c0, c1) : (long long)q0 * p.T + p.T - 1;
        if (e + 1 < c1) {
            cut = true;
            c1 = e + 1;
        }
    }
    const int tiles = (int)((unsigned)(c1 - c0 + tile - 1) / (unsigned)tile);
    const bool want_x = !MAP && (p.dgate || p.dgate_part);
    int buf = 0;
    for (int j = tiles - 1; j >= 0; --j, buf ^= 1) {
        const long long b = c0 + (long long)j * tile, i0 = b + tl * SEG;
        const NmPlace at = {p.reverse ? p.L - b - tile : b, (unsigned)(p.reverse ? tile - 1 - tl * SEG : tl * SEG), p.reverse};
        const int n = c1 - i0 >= SEG ? SEG : c1 > i0 ? (int)(c1 - i0) : 0;
        NmVec<DX, VEC> xv[SEG], cv[SEG];
        NmVec<DG, AV> gv[SEG];
        NmSeqs<SEG> sq;
        nm_s_seqs(p, at, n, i0, sq);
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            xv[s] = {};
            cv[s] = {};
        }
        if constexpr (SHARED || WHOLE) nm_s_load_whole<DG, AV, SEG>((const TG*)p.gate, at, n, gv);
        else nm_s_load_steps<DG, AV, SEG>((const TG*)p.gate, at, p.D, ch, n, gv);
        if constexpr (WHOLE) {
            if (p.g) nm_s_load_whole<DX, VEC, SEG>((const TX*)p.g, at, n, cv);
            if (want_x) nm_s_load_whole<DX, VEC, SEG>((const TX*)p.x, at, n, xv);
        } else {
            if (p.g) nm_s_load_steps<DX, VEC, SEG>((const TX*)p.g, at, p.D, ch, n, cv);
            if (want_x) nm_s_load_steps<DX, VEC, SEG>((const TX*)p.x, at, p.D, ch, n, xv);
        }
        const NmSteps st = nm_s_steps<SEG>(p, sq, n, (unsigned)(i0 - c0) + pos0, (int)q0);
        if (p.seg && __any(st.none != 0)) {                  // rows of no sequence: operands of 0 keep their states and gradients 0
#pragma unroll
            for (int s = 0; s < SEG; ++s)
                if ((st.none >> s) & 1) {
                    gv[s] = {};
                    xv[s] = {};
                    cv[s] = {};
                }
        }
        float start[VEC], end[VEC];
        nm_s_start(p, want_x ? p.h0 : nullptr, st, st.first, st.q_first, ch, start);
        nm_s_start(p, p.g_last, st, st.final, st.q_final, ch, end);
        auto enter = [&](int s, float (&h)[VEC]) { nm_s_enter(p, p.h0, st, st.first, st.q_first, start, i0, s, ch, h); };
        if (n < SEG) nm_s_pad<DG, AV, SEG>(gv, n, p.blend);
        auto advance = [&](int s, float (&h)[VEC]) { nm_s_step<DX, DG, VEC, AV>(gv[s], xv[s], p.blend, h); };
        auto retreat = [&](int s, float (&f)[VEC], float (&lam)[VEC]) {     // f of the step after s -> lambda and f of s
            nm_s_enter(p, p.g_last, st, st.final, st.q_final, end, i0, s, ch, f);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                lam[k] = nm_to_float<DX>(cv[s].e[k]) + f[k];
                f[k] = nm_s_factor<DG>(gv[s].e[AV == 1 ? 0 : k], p.blend) * lam[k];
            }
        };
        NmMap<VEC, AV> mf, mr, bf, br;
        nm_s_identity(mf);
        nm_s_identity(mr);
#pragma unroll
        for (int s = 0; s < SEG; ++s) {
            if (want_x) {
                enter(s, mf.h);
                advance(s, mf.h);
            }
#pragma unroll
            for (int k = 0; k < AV; ++k) mf.a[k] *= nm_s_factor<DG>(gv[s].e[k], p.blend);
        }
#pragma unroll
        for (int k = 0; k < AV; ++k) mr.a[k] = mf.a[k];
        mf.f = st.first ? 1 : 0;
        mr.f = st.final ? 1 : 0;
        if (want_x) {
            nm_s_wave_scan<VEC, AV, 1>(mf, bf, lane, cl);
            if (lane >= 64 - cl) nm_s_put(sh_h[MAP ? 0 : buf], wave, cx, mf);
        }
#pragma unroll
        for (int s = SEG - 1; s >= 0; --s) {
            float lam[VEC];
            retreat(s, mr.h, lam);
        }
        nm_s_wave_scan<VEC, AV, -1>(mr, br, lane, cl);
        if (lane < cl) nm_s_put(sh_r[buf], wave, cx, mr);
        __syncthreads();
        float f[VEC];
#pragma unroll
        for (int w = 3; w >= 0; --w) {
            NmMap<VEC, AV> mw;
            nm_s_get(sh_r[buf], w, cx, mw);
            if constexpr (MAP) {
                nm_s_then(total, mw);
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k)
                    if (w == wave) f[k] = flow[k];
                nm_s_apply(mw, flow);
            }
            __builtin_amdgcn_sched_barrier(0);               // (one wave's map in registers at a time)
        }
        if constexpr (!MAP) {
            nm_s_forget(gv);
            nm_s_forget(xv);
            nm_s_forget(cv);
            nm_s_forget(start);
            nm_s_forget(end);
            nm_s_apply(br, f);
            float hp[SEG][VEC];          // states before the steps, then the gradient of the gate
            if (want_x) {
                float h[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) h[k] = p.keep ? p.keep[(c * p.pieces + j) * p.D + ch + k] : 0.f;
#pragma unroll
                for (int w = 0; w < 3; ++w) {
                    NmMap<VEC, AV> mw;
                    nm_s_get(sh_h[buf], w, cx, mw);
                    if (w < wave) nm_s_apply(mw, h);
                    __builtin_amdgcn_sched_barrier(0);
                }
                nm_s_apply(bf, h);
#pragma unroll
                for (int s = 0; s < SEG; ++s) {
                    enter(s, h);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) hp[s][k] = h[k];
                    advance(s, h);
                }
            }
            float ox[WHOLE ? SEG : 1][VEC];
            const NmRow<TX> rx = nm_s_rows((TX*)p.dx, at, p.D, ch);
            const NmRow<TG> rg = nm_s_rows((TG*)p.dgate, at, SHARED ? 1 : p.D, SHARED ? 0 : ch);
#pragma unroll
            for (int s = SEG - 1; s >= 0; --s) {
                float lam[VEC], o[VEC];
                retreat(s, f, lam);
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    o[k] = p.blend ? nm_to_float<DG>(gv[s].e[SHARED ? 0 : k]) * lam[k] : lam[k];
                    if constexpr (WHOLE) ox[s][k] = o[k];
                }
                if constexpr (!WHOLE) {
                    if (p.dx && s < n) nm_s_store<DX, VEC>(rx.at(s), o);
                }
                if (want_x) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k) hp[s][k] = lam[k] * (p.blend ? nm_to_float<DX>(xv[s].e[k]) - hp[s][k] : hp[s][k]);
                    if constexpr (!SHARED && !WHOLE)
                        if (s < n) nm_s_store<DG, VEC>(rg.at(s), hp[s]);
                }
                if (p.dh0 && (((st.first & ~st.none) >> s) & 1)) {
                    float* dst = p.dh0 + nm_s_sequence(p, st, st.first, st.q_first, i0, s) * p.D + ch;
#pragma unroll
                    for (int k = 0; k < VEC; ++k) dst[k] = f[k];
                }
            }
            if constexpr (WHOLE) {
                if (p.dx) nm_s_store_whole<DX, VEC, SEG>((TX*)p.dx, at, n, ox);
                if constexpr (!SHARED) {
                    if (want_x) nm_s_store_whole<DG, VEC, SEG>((TG*)p.dgate, at, n, hp);
                }
            }
            if constexpr (SHARED) {
                if (want_x) {            // sum over the channels: own ones only, then the channel lanes (all lanes of the wave take part)
                    float sum[SEG][1];
#pragma unroll
                    for (int s = 0; s < SEG; ++s) {
                        sum[s][0] = 0.f;
#pragma unroll
                        for (int k = 0; k < VEC; ++k) sum[s][0] += ch + k >= own ? hp[s][k] : 0.f;
                        for (int o = 1; o < cl; o <<= 1) sum[s][0] += __shfl_xor(sum[s][0], o);
                    }
                    if (cx == 0) {
                        if (p.dgate_part) nm_s_store_whole<NM_F32, 1, SEG>(p.dgate_part + (long long)blk * p.L, at, n, sum);
                        else nm_s_store_whole<DG, 1, SEG>((TG*)p.dgate, at, n, sum);
                    }
                }
            }
        }
    }
    if (MAP && tl == 0) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            p.map_a[c * p.D + ch + k] = total.a[SHARED ? 0 : k];
            p.map_h[c * p.D + ch + k] = total.h[k];
        }
        if (blk == 0 && cx == 0) p.map_f[c] = total.f || cut;
    }
}

// maps of the ranges -> the state before every range (DIR = 1), or the flow after it (-1).  8 channels x 128 lanes in time, 16 ranges each: one round for
// all the ranges of a launch (nm_s_plan makes some NM_S_FILL_PACKED at most, so that offsets stay far below 2^32), for what a round costs is its latency (9 us for 1537 ranges of 32 channels).
#define NM_S_CARRY 1024
template <int DIR>
__global__ __launch_bounds__(NM_S_CARRY) void nm_scan_carry_kernel(const float* __restrict__ map_a, const float* __restrict__ map_h, const int* __restrict__ map_f, int n, int D,
                                                                   float* __restrict__ carry) {
    constexpr int WAVES = NM_S_CARRY / 64;
    __shared__ float sh_a[2][WAVES][8], sh_h[2][WAVES][8];
    __shared__ int sh_f[2][WAVES];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, cx = t & 7, tl = t >> 3;
    unsigned ch = blockIdx.x * 8u + cx;
    if (ch >= (unsigned)D) ch = D - 1;
    float state = 0.f;
    int buf = 0;
    for (int b = 0; b < n; b += NM_S_CARRY * 2, buf ^= 1) {
        const int i0 = b + tl * 16;
        float a[16], h[16];
        unsigned fresh = 0u;
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            const bool in = i0 + s < n;
            const unsigned c = in ? (unsigned)(DIR > 0 ? i0 + s : n - 1 - i0 - s) : 0u;
            a[s] = in ? map_a[c * (unsigned)D + ch] : 1.f;
            h[s] = in ? map_h[c * (unsigned)D + ch] : 0.f;
            if (in && map_f[c]) fresh |= 1u << s;
        }
        auto step = [&](int s, float& v) { v = (fresh >> s) & 1 ? h[s] : fmaf(a[s], v, h[s]); };
        NmMap<1, 1> m, before;
        nm_s_identity(m);
        m.f = fresh ? 1 : 0;
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            step(s, m.h[0]);
            m.a[0] *= a[s];
        }
        nm_s_wave_scan<1, 1, 1>(m, before, lane, 8);
        if (lane >= 56) {
            sh_a[buf][wave][cx] = m.a[0];
            sh_h[buf][wave][cx] = m.h[0];
            if (lane == 63) sh_f[buf][wave] = m.f;
        }
        __syncthreads();
        float v[1] = {0.f}, all[1] = {state};
#pragma unroll 4
        for (int w = 0; w < WAVES; ++w) {
            if (w == wave) v[0] = all[0];
            NmMap<1, 1> mw;
            mw.a[0] = sh_a[buf][w][cx]; mw.h[0] = sh_h[buf][w][cx]; mw.f = sh_f[buf][w];
            nm_s_apply(mw, all);
        }
        state = all[0];
        nm_s_apply(before, v);
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            if (i0 + s < n) carry[(unsigned)(DIR > 0 ? i0 + s : n - 1 - i0 - s) * (unsigned)D + ch] = v[0];
            step(s, v[0]);
        }
    }
}

// packed sequences: the sequence of every row (-1: none), and the result of empty sequences (their state / their cotangent passes through).
// (Launches have 2^31 threads at most, nm_s_threads: S x D may be more.)
__global__ __launch_bounds__(256) void nm_scan_rows_kernel(const int* __restrict__ cu, long long S, long long L, int D, const float* __restrict__ src, float* __restrict__ dst,
                                                           int* __restrict__ seg) {
    const long long t0 = (long long)blockIdx.x * 256 + threadIdx.x;
    if (seg && t0 < L) seg[t0] = nm_scan_sequence(cu, S, t0);
    if (!dst) return;
    for (long long t = t0; t < S * D; t += (long long)gridDim.x * 256) {
        const long long s = t / D;
        if (cu[s + 1] <= cu[s]) dst[t] = src ? src[t] : 0.f;
    }
}

// what passes through a batch without a single step
__global__ __launch_bounds__(256) void nm_scan_pass_kernel(const float* __restrict__ src, float* __restrict__ dst, long long n) {
    for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < n; t += (long long)gridDim.x * 256) dst[t] = src ? src[t] : 0.f;
}

// Sequences of one step, the form of a state carried from call to call: no order among the rows, so one thread per VEC channels, without tiles, scans and
// borders (512 x 256 fp32: 2.8 us, 10.1 in the kernel for sequences; 65536 x 512 bf16: 83 and 104).
template <int DX, int DG, int VEC>
__global__ __launch_bounds__(256) void nm_scan_step_kernel(NmScanArgs p, int shared, unsigned groups, unsigned n) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i >= n) return;
    const unsigned s = i / groups, ch = (i - s * groups) * VEC;
    const long long e = (long long)s * p.D + ch;
    NmVec<DG, VEC> g;
    const typename NmType<DG>::elem* gate = (const typename NmType<DG>::elem*)p.gate;
    if (shared) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) g.e[k] = gate[s];
    } else {
        g = nm_s_load<DG, VEC>(gate + e);
    }
    const NmVec<DX, VEC> x = nm_s_load<DX, VEC>((const typename NmType<DX>::elem*)p.x + e);
    float h[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) h[k] = 0.f;
    if (p.h0) {
        const NmVec<NM_F32, VEC> v = nm_s_load<NM_F32, VEC>(p.h0 + e);
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[k] = v.e[k];
    }
    nm_s_step<DX, DG, VEC, VEC>(g, x, p.blend, h);
    if (p.states) nm_s_store<DX, VEC>((typename NmType<DX>::elem*)p.states + e, h);
    nm_s_store<NM_F32, VEC>(p.last + e, h);
}

// shared gate over several channel blocks: sum of the blocks' parts, in order (no block: 0)
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
// workgroups of 256 threads for n threads, 2^31 threads at most (a launch of 2^32 is refused by the runtime; L < 2^31)
static inline dim3 nm_s_threads(long long n) { return dim3((unsigned)(n < 0x80000000LL ? nm_s_up(n, 256) : 0x800000LL)); }

struct NmScanShape { int vec, cl_log2, blocks, tile; };      // of one direction: channels and channel lanes, tile in steps
struct NmScanPlan {
    NmScanShape f, b;
    bool split;                          // ranges cut sequences: maps and carried states
    long long chunk_f, chunks_f, chunk_b, chunks_b, keep_elems;
    bool keep_seq;                       // kept states are counted from the sequences' starts (needed by those longer than a backward tile)
    long long keep_rows;                 // packed: words of `keep` (and of the workspace) that hold the sequence of every row
    size_t off_seg, off_a, off_h, off_f, off_carry, off_part, bytes;
};

// Workgroups of a launch over ranges that cut sequences.  Packed ones twice as many: their maps end at the first border, so that more ranges cost them
// little, and the longest waits less for its tiles (8192 sequences of 96 steps x 32 channels fp32, backward: 117 us instead of 138).  Equal lengths read all
// operands for the maps either way (4 x 16384 x 512 bf16: 69 us for maps and states with either number).
#define NM_S_FILL 1024
#define NM_S_FILL_PACKED 2048

static NmScanShape nm_s_shape(int D, int vec, int seg) {
    NmScanShape s;
    s.vec = vec;
    const int groups = (int)nm_s_up(D, vec);
    s.cl_log2 = 0;
    while ((1 << s.cl_log2) < groups && s.cl_log2 < 6) ++s.cl_log2;
    s.blocks = (int)nm_s_up(groups, 1 << s.cl_log2);
    s.tile = (NM_S_THREADS >> s.cl_log2) * seg;
    return s;
}

static NmScanPlan nm_s_plan(long long L, long long S, int D, int dtype, bool shared, bool packed) {
    NmScanPlan p;
    const int vb = D >= 4 ? 4 : D, vf = dtype != NM_F32 && D >= 8 ? 8 : vb;
    const int seg_f = vf == 8 ? (shared ? NmSeg<8, true>::F : NmSeg<8, false>::F) : vf == 4 ? NmSeg<4, true>::F : NmSeg<1, true>::F;
    const int seg_b = vb == 4 ? NmSeg<4, true>::B : NmSeg<1, true>::B;
    p.f = nm_s_shape(D, vf, seg_f);
    p.b = nm_s_shape(D, vb, seg_b);
    // ranges: whole tiles of both directions (powers of two of the same), or whole sequences
    const long long tile = p.f.tile > p.b.tile ? p.f.tile : p.b.tile;
    const int blocks = p.f.blocks < p.b.blocks ? p.f.blocks : p.b.blocks;
    const long long T = packed || S == 0 ? 0 : L / S;
    p.split = packed || (T > tile && S * blocks < NM_S_FILL / 2);
    if (p.split) {
        p.chunk_f = p.chunk_b = nm_s_up(nm_s_up(L, tile) * blocks, packed ? NM_S_FILL_PACKED : NM_S_FILL) * tile;
        p.keep_elems = nm_s_up(L, p.chunk_b) * (p.chunk_b / p.b.tile) * D;
        if (p.chunk_f >= L) p.split = false;                 // (one range)
        p.keep_seq = false;
    } else {
        const long long t = T > 0 ? T : 1;
        p.chunk_f = t >= p.f.tile ? t : p.f.tile / t * t;    // the sequences that fit a tile, or one
        p.chunk_b = t >= p.b.tile ? t : p.b.tile / t * t;
        p.keep_seq = t > p.b.tile;
        p.keep_elems = p.keep_seq ? S * nm_s_up(t, p.b.tile) * D : 0;
    }
    p.chunks_f = nm_s_up(L, p.chunk_f);
    p.chunks_b = nm_s_up(L, p.chunk_b);
    p.keep_rows = packed ? nm_s_up(L, 64) * 64 : 0;
    size_t off = 0;
    p.off_seg = off;
    off += (size_t)p.keep_rows * 4;
    p.off_a = off;
    const size_t map = p.split ? nm_s_align((size_t)p.chunks_f * D * 4) : 0;
    off += map;
    p.off_h = off;
    off += map;
    p.off_carry = off;
    off += map;
    p.off_f = off;
    if (p.split) off += nm_s_align((size_t)p.chunks_f * 4);
    p.off_part = off;
    if (shared && p.b.blocks > 1) off += nm_s_align((size_t)p.b.blocks * L * 4);
    p.bytes = off;
    return p;
}

#define NM_S_LAUNCH(KERNEL, DX, DG, VEC, MAP)                                                                                     \
    do {                                                                                                                          \
        if (shared) hipLaunchKernelGGL((KERNEL<DX, DG, VEC, true, MAP>), grid, dim3(NM_S_THREADS), 0, stream, a);                  \
        else hipLaunchKernelGGL((KERNEL<DX, DG, VEC, false, MAP>), grid, dim3(NM_S_THREADS), 0, stream, a);                        \
    } while (0)
#define NM_S_PICK_VEC(KERNEL, DX, DG, MAP, WIDE)                                                                                  \
    do {                                                                                                                          \
        if (shape.vec == 8) { if constexpr (WIDE) NM_S_LAUNCH(KERNEL, DX, DG, 8, MAP); }                                          \
        else if (shape.vec == 4) NM_S_LAUNCH(KERNEL, DX, DG, 4, MAP);                                                             \
        else if (shape.vec == 3) NM_S_LAUNCH(KERNEL, DX, DG, 3, MAP);                                                             \
        else if (shape.vec == 2) NM_S_LAUNCH(KERNEL, DX, DG, 2, MAP);                                                             \
        else NM_S_LAUNCH(KERNEL, DX, DG, 1, MAP);                                                                                 \
    } while (0)
#define NM_S_PICK(KERNEL, MAP, WIDE)                                                                                              \
    do {                                                                                                                          \
        if (dtype == NM_F32) NM_S_PICK_VEC(KERNEL, NM_F32, NM_F32, MAP, false);                                                   \
        else if (dtype == NM_F16 && gate_dtype == NM_F32) NM_S_PICK_VEC(KERNEL, NM_F16, NM_F32, MAP, WIDE);                       \
        else if (dtype == NM_F16) NM_S_PICK_VEC(KERNEL, NM_F16, NM_F16, MAP, WIDE);                                               \
        else if (gate_dtype == NM_F32) NM_S_PICK_VEC(KERNEL, NM_BF16, NM_F32, MAP, WIDE);                                         \
        else NM_S_PICK_VEC(KERNEL, NM_BF16, NM_BF16, MAP, WIDE);                                                                  \
    } while (0)

static int nm_s_check(const char* who, int64_t L, int64_t S, int64_t D, int dtype, int gate_dtype, bool packed) {
    if (!nm_dtype_ok(dtype) || (gate_dtype != dtype && gate_dtype != NM_F32)) return nm_fail("%s: unknown element types %d / %d (the gate is fp32 or of the values' type)", who, dtype, gate_dtype);
    if (L < 0 || S < 0 || D < 0 || L > 0x7fffffffLL || S > 0x7fffffffLL || D > (1 << 20)) return nm_fail("%s: bad sizes L=%lld S=%lld D=%lld", who, (long long)L, (long long)S, (long long)D);
    if (!packed && (S == 0 ? L != 0 : L % S != 0)) return nm_fail("%s: %lld steps are not %lld sequences of equal length", who, (long long)L, (long long)S);
    return 0;
}

static void nm_s_fill(NmScanArgs& a, const NmScanPlan& pl, const NmScanShape& shape, const void* gate, const void* x, const float* h0, const int* cu, int64_t L, int64_t S, int64_t D, int reverse,
                      int blend, char* ws, int* rows) {
    a.gate = gate; a.x = x; a.h0 = h0; a.cu = cu;
    a.seg = cu ? rows : nullptr;
    a.L = L; a.S = S; a.chunk = &shape == &pl.f ? pl.chunk_f : pl.chunk_b; a.T = cu || S == 0 ? 1u : (unsigned)(L / S); a.D = (int)D;
    a.reverse = reverse ? 1 : 0; a.blend = blend ? 1 : 0; a.cl_log2 = shape.cl_log2; a.blocks = shape.blocks;
    a.keep_steps = pl.b.tile;
    a.pieces = (int)nm_s_up(pl.chunk_b, pl.b.tile);
    if (pl.split) {
        a.map_a = (float*)(ws + pl.off_a); a.map_h = (float*)(ws + pl.off_h); a.map_f = (int*)(ws + pl.off_f);
    }
}

static void nm_s_gate_sum(const float* part, int blocks, long long L, void* dgate, int gate_dtype, hipStream_t stream) {
    const dim3 grid = nm_s_threads(L);
    if (gate_dtype == NM_F32) hipLaunchKernelGGL(nm_scan_gate_sum_kernel<NM_F32>, grid, dim3(256), 0, stream, part, blocks, L, (float*)dgate);
    else if (gate_dtype == NM_F16) hipLaunchKernelGGL(nm_scan_gate_sum_kernel<NM_F16>, grid, dim3(256), 0, stream, part, blocks, L, (_Float16*)dgate);
    else hipLaunchKernelGGL(nm_scan_gate_sum_kernel<NM_BF16>, grid, dim3(256), 0, stream, part, blocks, L, (__bf16*)dgate);
}

extern "C" {

int64_t nm_scan_workspace_bytes(int64_t L, int64_t S, int64_t D, int dtype, int shared_gate, int packed) {
    if (nm_s_check("nm_scan_workspace_bytes", L, S, D, dtype, dtype, packed != 0)) return -1;
    return L == 0 || D == 0 ? 0 : (int64_t)nm_s_plan(L, S, (int)D, dtype, shared_gate != 0, packed != 0).bytes;
}

int64_t nm_scan_keep_elems(int64_t L, int64_t S, int64_t D, int dtype, int shared_gate, int packed) {
    if (nm_s_check("nm_scan_keep_elems", L, S, D, dtype, dtype, packed != 0)) return -1;
    if (L == 0 || D == 0) return 0;
    const NmScanPlan pl = nm_s_plan(L, S, (int)D, dtype, shared_gate != 0, packed != 0);
    return pl.keep_rows + pl.keep_elems;
}

int nm_scan_forward(const void* gate, int gate_dtype, int shared_gate, const void* x, int dtype, const float* h0, const int32_t* cu_seqlens, int64_t L, int64_t S, int64_t D,
                    int reverse, int blend, void* states, float* last, float* keep, void* workspace, int64_t workspace_bytes, nm_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    const bool packed = cu_seqlens != nullptr, shared = shared_gate != 0;
    if (nm_s_check("nm_scan_forward", L, S, D, dtype, gate_dtype, packed)) return 1;
    if (D == 0 || (L == 0 && S == 0)) return 0;
    if ((L > 0 && (!gate || !x)) || (S > 0 && !last)) return nm_fail("nm_scan_forward: NULL argument");
    if (L == 0) {                        // every sequence is empty: its state passes through
        hipLaunchKernelGGL(nm_scan_pass_kernel, nm_s_threads(S * D), dim3(256), 0, stream, h0, last, (long long)(S * D));
        NM_LAUNCH_CHECK();
        return 0;
    }
    const NmScanPlan pl = nm_s_plan(L, S, (int)D, dtype, shared, packed);
    const NmScanShape& shape = pl.f;
    if ((size_t)(workspace_bytes < 0 ? 0 : workspace_bytes) < pl.bytes || (pl.bytes > 0 && !workspace)) return nm_fail("nm_scan_forward: workspace too small");
    if (pl.chunks_f * shape.blocks > NM_S_MAX_GROUPS) return nm_fail("nm_scan_forward: %lld steps x %lld channels exceed one launch", (long long)L, (long long)D);
    char* ws = (char*)workspace;
    int* rows = packed ? keep ? (int*)keep : (int*)(ws + pl.off_seg) : nullptr;
    if (packed) {
        const long long n = L > S * D ? L : S * D;
        hipLaunchKernelGGL(nm_scan_rows_kernel, nm_s_threads(n), dim3(256), 0, stream, cu_seqlens, (long long)S, (long long)L, (int)D, h0, last, rows);
        NM_LAUNCH_CHECK();               // (the main launch indexes with these rows)
    }
    NmScanArgs a = {};
    nm_s_fill(a, pl, shape, gate, x, h0, cu_seqlens, L, S, D, reverse, blend, ws, rows);
    a.states = states; a.last = last; a.keep = keep && pl.keep_elems > 0 ? keep + pl.keep_rows : nullptr;
    a.keep_seq = a.keep && pl.keep_seq;
    if (!packed && L == S && L * D <= 0xffffff00LL) {        // (thread numbers are 32 bits)
        const unsigned vec = D % 4 == 0 ? 4u : 1u, groups = (unsigned)(D / vec), n = (unsigned)(S * groups);
        const dim3 steps((unsigned)nm_s_up(n, 256)), block(256);
#define NM_S_STEP(DX, DG)                                                                                              \
    do {                                                                                                               \
        if (vec == 4) hipLaunchKernelGGL((nm_scan_step_kernel<DX, DG, 4>), steps, block, 0, stream, a, (int)shared, groups, n); \
        else hipLaunchKernelGGL((nm_scan_step_kernel<DX, DG, 1>), steps, block, 0, stream, a, (int)shared, groups, n);          \
    } while (0)
        if (dtype == NM_F32) NM_S_STEP(NM_F32, NM_F32);
        else if (dtype == NM_F16 && gate_dtype == NM_F32) NM_S_STEP(NM_F16, NM_F32);
        else if (dtype == NM_F16) NM_S_STEP(NM_F16, NM_F16);
        else if (gate_dtype == NM_F32) NM_S_STEP(NM_BF16, NM_F32);
        else NM_S_STEP(NM_BF16, NM_BF16);
        NM_LAUNCH_CHECK();
        return 0;
    }
    const dim3 grid((unsigned)(pl.chunks_f * shape.blocks));
    if (pl.split) {
        float* carry = (float*)(ws + pl.off_carry);
        NM_S_PICK(nm_scan_forward_kernel, true, true);
        hipLaunchKernelGGL(nm_scan_carry_kernel<1>, dim3((unsigned)nm_s_up(D, 8)), dim3(NM_S_CARRY), 0, stream, a.map_a, a.map_h, a.map_f, (int)pl.chunks_f, (int)D, carry);
        a.carry = carry;
    }
    NM_S_PICK(nm_scan_forward_kernel, false, true);
    NM_LAUNCH_CHECK();
    return 0;
}

int nm_scan_backward(const void* gate, int gate_dtype, int shared_gate, const void* x, int dtype, const float* h0, const int32_t* cu_seqlens, int64_t L, int64_t S, int64_t D,
                     int reverse, int blend, const float* keep, const void* g_states, const float* g_last, void* dgate, void* dx, float* dh0, void* workspace,
                     int64_t workspace_bytes, nm_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    const bool packed = cu_seqlens != nullptr, shared = shared_gate != 0;
    if (nm_s_check("nm_scan_backward", L, S, D, dtype, gate_dtype, packed)) return 1;
    if ((L == 0 && S == 0) || (!dgate && !dx && !dh0)) return 0;
    if (D == 0) {                        // no channels: nothing but a shared gate's gradient, a sum over none of them
        if (dgate && shared && L > 0) nm_s_gate_sum(nullptr, 0, L, dgate, gate_dtype, stream);
        NM_LAUNCH_CHECK();
        return 0;
    }
    if (L > 0 && (!gate || (dgate && (!x || (!keep && nm_scan_keep_elems(L, S, D, dtype, shared_gate, packed) > 0))))) return nm_fail("nm_scan_backward: NULL argument");
    if (L == 0) {
        if (!dh0) return 0;
        hipLaunchKernelGGL(nm_scan_pass_kernel, nm_s_threads(S * D), dim3(256), 0, stream, g_last, dh0, (long long)(S * D));
        NM_LAUNCH_CHECK();
        return 0;
    }
    const NmScanPlan pl = nm_s_plan(L, S, (int)D, dtype, shared, packed);
    const NmScanShape& shape = pl.b;
    if ((size_t)(workspace_bytes < 0 ? 0 : workspace_bytes) < pl.bytes || (pl.bytes > 0 && !workspace)) return nm_fail("nm_scan_backward: workspace too small");
    if (pl.chunks_b * shape.blocks > NM_S_MAX_GROUPS) return nm_fail("nm_scan_backward: %lld steps x %lld channels exceed one launch", (long long)L, (long long)D);
    char* ws = (char*)workspace;
    int* rows = packed ? keep ? (int*)const_cast<float*>(keep) : (int*)(ws + pl.off_seg) : nullptr;
    if (packed && (!keep || dh0)) {      // (the rows' sequences are kept from the forward pass)
        const long long n = keep ? S * D : L > S * D ? L : S * D;
        hipLaunchKernelGGL(nm_scan_rows_kernel, nm_s_threads(n), dim3(256), 0, stream, cu_seqlens, (long long)S, (long long)L, (int)D, g_last, dh0, keep ? nullptr : rows);
        NM_LAUNCH_CHECK();
    }
    NmScanArgs a = {};
    nm_s_fill(a, pl, shape, gate, x, h0, cu_seqlens, L, S, D, reverse, blend, ws, rows);
    a.keep = keep && pl.keep_elems > 0 ? const_cast<float*>(keep) + pl.keep_rows : nullptr; a.g = g_states; a.g_last = g_last; a.dgate = dgate; a.dx = dx; a.dh0 = dh0;
    const bool parts = shared && dgate && shape.blocks > 1;
    if (parts) a.dgate_part = (float*)(ws + pl.off_part);
    const dim3 grid((unsigned)(pl.chunks_b * shape.blocks));
    if (pl.split) {
        float* carry = (float*)(ws + pl.off_carry);
        NM_S_PICK(nm_scan_backward_kernel, true, false);
        hipLaunchKernelGGL(nm_scan_carry_kernel<-1>, dim3((unsigned)nm_s_up(D, 8)), dim3(NM_S_CARRY), 0, stream, a.map_a, a.map_h, a.map_f, (int)pl.chunks_b, (int)D, carry);
        a.carry = carry;
    }
    NM_S_PICK(nm_scan_backward_kernel, false, false);
    if (parts) nm_s_gate_sum(a.dgate_part, shape.blocks, L, dgate, gate_dtype, stream);
    NM_LAUNCH_CHECK();
    return 0;
}

}  // extern "C"
