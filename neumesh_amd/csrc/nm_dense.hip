// nm_dense.hip -- dense layers: y = act(x W^T + b) + r and its gradient (C ABI: nm_dense_*), on the matrix pipe.
//
//   z = x W^T + b,   y = act(z) + r          x [M,K], W [N,K], b [N], r and y [M,N]
//   dz = g * act'(z);  dx = dz W;  dW = dz^T x;  db = sum over the rows of dz;  dr = g
//
// Three products:
//   forward and dx: rows x a weight matrix, contraction along the rows' contiguous axis: nm_dense_tile_kernel (16-bit forward, enough outputs to
//                        fill the chip with 256 x 256 tiles), nm_dense_resident_kernel (weights that fit in LDS), nm_dense_stream_kernel (the rest)
//   nm_dense_grad_kernel  dW and db: contraction over the rows, split over workgroups; nm_dense_sum_kernel adds the partial sums in a
//                        fixed order (the same bits from run to run)
// nm_dense_few_kernel serves 1 .. 8 rows (a probe, a picked point).
//
// Arithmetic.  16-bit inputs: one product per pair on the f16 / bf16 pipe, fp32 accumulation, fp32 epilogue, one rounding at the end.  The forward pass
// keeps act'(z) for the backward pass (NmFactor).  dz = g act'(z) enters the products as TWO bf16 pieces (value + residual: 16 bits over fp32's whole
// range, an error of 1/32 (fp16) and 1/256 (bf16) of the result's own rounding): a single rounded piece put an error as large as that rounding on dx and
// dW, and fp16 pieces lost what lies below 2^-13 (g of a mean over many outputs) and beyond 65504 (g near the maximum times act' = 1.13).  Beside fp16
// rows the other operand is cut into two bf16 pieces as well, exactly, and three piece products are taken (10007 x 177 -> 131 forward and backward 123 us,
// 126 with two products of fp16 pieces).  fp32 inputs: every operand cut into three bf16 pieces (nm_d_cut8), six piece products, fp32 accumulation.  A
// product of several pieces with a non-finite operand is NaN where IEEE arithmetic may give an infinity.
#include "nm_error.h"
#include "nm_num.h"

#include <utility>

#define NM_D_MAX_DIM (1 << 20)   // columns and contraction lengths fit 32-bit arithmetic with room
#define NM_D_MAX_LD (1 << 24)    // 64 rows of any stride stay below 2^32 bytes
#define NM_D_MAX_THREADS 0xffffffffLL    // of one launch

// ------------------------------------------------------------------------------------------------ kept derivatives
// act'(z) of [R, C] outputs, contiguous, from the forward to the backward pass.  Beside fp32 rows: fp32.  Beside 16-bit rows: the upper 24 bits of the
// fp32 value, rounded: 16 significant bits, as many as dz has in the products, and fp32's exponent, so that a unit deep in the tail of its activation keeps
// its gradient (fp16 had steps of 2^-24: sigmoid' 3 % off at -15 and 0 at -18).  Two planes: upper halves [R, C], 16 bits each, then the third
// bytes [R, C].  Three bytes and not four because the buffer is written once and read twice, in layers that are bound by memory.
template <int DT> struct NmFactor {                          // a row (or any place) of the planes
    const char* hi; const char* lo;
    static constexpr int E = DT == NM_F32 ? 4 : 2;           // bytes per element of the first plane
    __device__ __forceinline__ NmFactor at(long long i) const { return {hi + i * E, DT == NM_F32 ? nullptr : lo + i}; }
};
template <int DT> struct NmFactorOct { uint4 hi[DT == NM_F32 ? 2 : 1]; uint2 lo; };       // eight of them

// the planes that start at `base`, n elements
template <int DT>
__host__ __device__ __forceinline__ NmFactor<DT> nm_d_planes(const void* base, long long n) { return {(const char*)base, DT == NM_F32 || !base ? nullptr : (const char*)base + 2 * n}; }

// upper half (h = 0, 1) of a word of the first plane and byte k of a word of the second -> the value
template <int H, int K>
__device__ __forceinline__ float nm_d_join(unsigned hi, unsigned lo) {
    return __uint_as_float(__builtin_amdgcn_perm(hi, lo, (unsigned)(5 + 2 * H) << 24 | (unsigned)(4 + 2 * H) << 16 | (unsigned)K << 8 | 0x0cu));
}
__device__ __forceinline__ unsigned nm_d_round24(float d) { return d != d ? 0x7fc00000u : __float_as_uint(d) + 0x80u; }

template <int DT>
__device__ __forceinline__ void nm_d_factors(const NmFactorOct<DT>& o, float (&f)[8]) {
    if constexpr (DT == NM_F32) {
        __builtin_memcpy(f, &o, 32);
    } else {
        unsigned w[4];
        __builtin_memcpy(w, &o, 16);
        f[0] = nm_d_join<0, 0>(w[0], o.lo.x); f[1] = nm_d_join<1, 1>(w[0], o.lo.x); f[2] = nm_d_join<0, 2>(w[1], o.lo.x); f[3] = nm_d_join<1, 3>(w[1], o.lo.x);
        f[4] = nm_d_join<0, 0>(w[2], o.lo.y); f[5] = nm_d_join<1, 1>(w[2], o.lo.y); f[6] = nm_d_join<0, 2>(w[3], o.lo.y); f[7] = nm_d_join<1, 3>(w[3], o.lo.y);
    }
}
// eight from place q of a row of Q on, by the rule of nm_d_fetch: rows of eight or more in one whole load that ends at Q at the latest
template <int DT>
__device__ __forceinline__ NmFactorOct<DT> nm_d_fetch_factors(const NmFactor<DT>& row, int q, int Q) {
    NmFactorOct<DT> o;
    if (Q >= 8) {                                            // (uniform)
        const NmFactor<DT> from = row.at(q + 8 <= Q ? q : Q - 8);
        __builtin_memcpy(&o.hi, from.hi, sizeof(o.hi));
        if constexpr (DT != NM_F32) __builtin_memcpy(&o.lo, from.lo, 8);
        return o;
    }
    const int n = q == 0 ? Q : 0;
    __builtin_memset(&o, 0, sizeof(o));
    if constexpr (DT == NM_F32) {
        const NmOct<NM_F32> v = nm_oct_load_short<NM_F32>((const float*)row.hi, n);
        __builtin_memcpy(&o.hi, &v, sizeof(v));
    } else {
        o.hi[0] = nm_oct_load_short<NM_F16>((const _Float16*)row.hi, n).v[0];
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            const unsigned b = (unsigned char)row.lo[i];
            o.lo.x |= i < 4 ? b << (8 * i) : 0u;
            o.lo.y |= i < 4 ? 0u : b << (8 * (i - 4));
        }
    }
    return o;
}
// its first `sh` cleared (upper halves are enough: what is left is below 2^-133, and goes with an operand that is cleared)
template <int DT>
__device__ __forceinline__ NmFactorOct<DT> nm_d_clear_factors(NmFactorOct<DT> o, int sh) {
    NmOct<DT> h;
    __builtin_memcpy(&h, &o.hi, sizeof(h));
    h = nm_oct_clear_first<DT>(h, sh);
    __builtin_memcpy(&o.hi, &h, sizeof(h));
    return o;
}

// ------------------------------------------------------------------------------------------------ activations
// Exponentials and reciprocals from the hardware's approximations; F32 (fp32 outputs) corrects them to the last place (library exponential and division:
// 70 instructions per element, 34 us of a 65536 x 256 layer), 16-bit outputs take them as they are (errors of 1e-6 are far below their rounding).
template <bool F32>
__device__ __forceinline__ float nm_d_exp(float x) {         // x <= 0
    const float t = x * 1.44269504088896341f;
    if (!F32) return __builtin_amdgcn_exp2f(t);
    // what the rounded product t leaves of x log2(e), as a first-order factor: 1 + r ln 2
    const float r = fmaf(x, 1.92596299112661746e-8f, fmaf(x, 1.44269504088896341f, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return x < -104.0f ? 0.0f : fmaf(e, r * 0.693147180559945309f, e);
}
template <bool F32>
__device__ __forceinline__ float nm_d_rcp(float x) {         // 1 <= x <= 3
    const float r = __builtin_amdgcn_rcpf(x);
    return F32 ? fmaf(r, fmaf(-x, r, 1.0f), r) : r;          // one Newton step
}

// log(1 + e) for e in [0, 1]: 2 atanh(e / (2 + e)), series in s^2 <= 1/9 (truncation 1.4e-8 relative)
template <bool F32>
__device__ __forceinline__ float nm_d_log1p(float e) {
    const float s = e * nm_d_rcp<F32>(2.0f + e), q = s * s;
    float p = fmaf(q, 1.0f / 13.0f, 1.0f / 11.0f);
    p = fmaf(q, p, 1.0f / 9.0f);
    p = fmaf(q, p, 1.0f / 7.0f);
    p = fmaf(q, p, 1.0f / 5.0f);
    p = fmaf(q, p, 1.0f / 3.0f);
    return 2.0f * fmaf(s * q, p, s);
}

// values z -> act(z) in place, derivatives -> d.  sigmoid, SiLU and GELU are one form, z or 1 times sigmoid(c1 z + c3 z^3); the tests are on the
// launch's activation, once per group.
template <bool F32, int N>
__device__ __forceinline__ void nm_d_act(int act, float beta, float ibeta, bool want, float (&z)[N], float (&d)[N]) {
    if (act == NM_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = 1.f;
    } else if (act == NM_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            d[i] = z[i] > 0.f ? 1.f : 0.f;
            z[i] = z[i] <= 0.f ? 0.f : z[i];                 // NaN stays NaN
        }
    } else if (act == NM_ACT_SOFTPLUS) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float u = beta * z[i], e = nm_d_exp<F32>(-fabsf(u));
            // 16 bits: the hardware's logarithm, off by 1e-7 near 1, so that a small e has its series (the next term is e^2 / 3 < 6e-6 of it)
            const float l = F32 ? nm_d_log1p<F32>(e) : e < 0x1p-8f ? fmaf(-0.5f * e, e, e) : 0.693147180559945309f * __builtin_amdgcn_logf(1.0f + e);
            z[i] = fmaf(l, ibeta, fmaxf(z[i], 0.f));
            if (want) {
                const float r = nm_d_rcp<F32>(1.0f + e);
                d[i] = u >= 0.f ? r : e * r;
            }
        }
    } else {
        const float c1 = act == NM_ACT_GELU_TANH ? 1.59576912160573071f : 1.0f;      // 2 sqrt(2 / pi)
        const float c3 = act == NM_ACT_GELU_TANH ? 0.044715f : 0.0f;
        const bool gate_only = act == NM_ACT_SIGMOID;
        if constexpr (!F32) {            // 16 bits: one exponential of either sign; where it is infinite q is 0, and so is what it multiplies
            const float k1 = -1.44269504088896341f * c1;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float x = z[i], e = __builtin_amdgcn_exp2f(k1 * x * fmaf(c3, fminf(x * x, 1e8f), 1.0f)), q = __builtin_amdgcn_rcpf(1.0f + e);
                if (want) {
                    const float t = fminf(fmaxf(x, -1e4f), 1e4f), q1 = fminf(e, 3e38f) * q;      // (beyond, q or q1 is 0: no infinity times zero)
                    d[i] = gate_only ? q * q1 : fmaf(t * q, q1 * (c1 * fmaf(3.0f * c3, t * t, 1.0f)), q);
                }
                z[i] = gate_only ? q : x * q;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = fminf(fmaxf(z[i], -1e4f), 1e4f), t2 = t * t;             // (beyond, q or q1 is 0: no infinity times zero)
            const float u = c1 * t * fmaf(c3, t2, 1.0f);
            const float e = nm_d_exp<F32>(-fabsf(u)), r = nm_d_rcp<F32>(1.0f + e), er = e * r;
            const float q = z[i] != z[i] ? z[i] : u >= 0.f ? r : er, q1 = u >= 0.f ? er : r;
            if (want) d[i] = gate_only ? q * q1 : fmaf(t * q, q1 * (c1 * fmaf(3.0f * c3, t2, 1.0f)), q);
            z[i] = gate_only ? q : z[i] * q;
        }
    }
}

// ------------------------------------------------------------------------------------------------ operand pieces
__device__ __forceinline__ unsigned nm_d_pair(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }   // upper halves

// eight fp32 values -> fragments (16 bytes: eight 16-bit pieces per plane): three bf16 pieces each, a = p0 + p1 + p2 exactly.  The first two are rounded to
// nearest, so that |p1| <= 2^-8 and |p2| <= 2^-17 of a's power of two, of either sign (cut off instead, pieces have the sign of a and are twice as
// large: the piece products that are left out were up to 2^-21 of every product, all in one direction).  What would round to an infinity takes the largest bf16.
__device__ __forceinline__ void nm_d_cut8(const float (&f)[8], uint4 (&p)[3]) {
    __bf16 b[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        b[0][e] = (__bf16)__builtin_amdgcn_fmed3f(f[e], -0x1.fep127f, 0x1.fep127f);
        const float r = f[e] - (float)b[0][e];
        b[1][e] = (__bf16)r;
        b[2][e] = (__bf16)(r - (float)b[1][e]);
    }
    __builtin_memcpy(p, b, sizeof(b));
}
// value + residual in bf16: 16 bits of any fp32 value, all of an fp16 one (no residual of an infinity)
__device__ __forceinline__ void nm_d_two8(const float (&f)[8], uint4 (&p)[2]) {
    __bf16 hi[8], lo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        hi[e] = (__bf16)f[e];
        const float b = (float)hi[e];
        lo[e] = (__bf16)(fabsf(b) < __builtin_inff() ? f[e] - b : 0.f);
    }
    __builtin_memcpy(&p[0], hi, 16);
    __builtin_memcpy(&p[1], lo, 16);
}

// Pieces of the operands of a product, and the 16-bit type that the matrix pipe sees.  PROD: one operand (the rows, or dz of the weight gradient) is g * act'(z).
template <int DT, bool PROD> struct NmPieces {
    static constexpr int PLAIN = DT == NM_F32 ? 3 : DT == NM_F16 && PROD ? 2 : 1;        // the other operand
    static constexpr int ROWS = DT == NM_F32 ? 3 : PROD ? 2 : 1;
    static constexpr int MF = DT == NM_F16 && !PROD ? (int)NM_F16 : (int)NM_BF16;
};
static inline int nm_d_pieces(int dt, bool prod) { return dt == NM_F32 ? 3 : dt == NM_F16 && prod ? 2 : 1; }      // (PLAIN)

// one matrix instruction: V = nm_v16f: 32 x 32 outputs, 16 deep;  nm_v4f: 16 x 16 outputs, 32 deep
template <int DT, typename V>
__device__ __forceinline__ V nm_d_mfma(const uint4& a, const uint4& b, V c) {
    constexpr bool WIDE = sizeof(V) == 64;
    if constexpr (DT == NM_F16) {
        nm_v8h x, y;
        __builtin_memcpy(&x, &a, 16);
        __builtin_memcpy(&y, &b, 16);
        if constexpr (WIDE) return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
    } else {
        nm_v8b x, y;
        __builtin_memcpy(&x, &a, 16);
        __builtin_memcpy(&y, &b, 16);
        if constexpr (WIDE) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
    }
}

// all piece products of one pair of fragments, small terms first.  Planes: PA of a, PB of b.
template <int DT, int PA, int PB, typename V>
__device__ __forceinline__ V nm_d_products(const uint4 (&a)[PA], const uint4 (&b)[PB], V c) {
    if constexpr (PA == 3 && PB == 3) {      // dropped: a1 b2 + a2 b1 + a2 b2 < 2^-23 |a||b|, of either sign
        c = nm_d_mfma<DT>(a[1], b[1], c);
        c = nm_d_mfma<DT>(a[0], b[2], c);
        c = nm_d_mfma<DT>(a[2], b[0], c);
        c = nm_d_mfma<DT>(a[0], b[1], c);
        c = nm_d_mfma<DT>(a[1], b[0], c);
        return nm_d_mfma<DT>(a[0], b[0], c);
    } else if constexpr (PA == 2 && PB == 2) {               // dropped: a1 b1 <= 2^-16 |a||b|, of either sign
        c = nm_d_mfma<DT>(a[1], b[0], c);
        c = nm_d_mfma<DT>(a[0], b[1], c);
        return nm_d_mfma<DT>(a[0], b[0], c);
    } else {
        static_assert(PA == 1 || PB == 1, "two pieces against one");
#pragma unroll
        for (int i = PA - 1; i >= 0; --i)
#pragma unroll
            for (int j = PB - 1; j >= 0; --j) c = nm_d_mfma<DT>(a[i], b[j], c);
        return c;
    }
}

// ------------------------------------------------------------------------------------------------ weights in fragment order
// Column operand of the products rows x weights: element (c, q), output column c, contraction q.  Fragment (step q / 32, tile of 16 columns): lane
// (i, h), i = lane % 16, holds q = 32 step + 8 h .. + 7 of the column at position i.  An output tile of the matrix pipe gives lane (j, h) the positions
// 4 h .. 4 h + 3 of row j.  16-bit outputs: a pair of tiles is 32 columns, positions ordered so that the lane's eight values of the pair are
// columns 8 h .. 8 h + 7 -- 16 bytes, and the four lanes of a row 64 bytes on end; fp32 outputs: columns in order, the lane's four values are
// 16 bytes.  (32 x 32 tiles leave a row to two lanes: pieces of 16 bytes 32 apart made the stores three quarters of a memory-bound layer's time.)
template <int DT>
__host__ __device__ __forceinline__ int nm_d_column(int tile, int i) {
    return DT == NM_F32 ? 16 * tile + i : 32 * (tile >> 1) + 8 * (i >> 2) + 4 * (tile & 1) + (i & 3);
}

// Eight consecutive contraction elements always come as ONE whole load: the piece that would end beyond Q starts at Q - 8 instead, and what it
// repeats is zero on the packed side (and cleared on the rows' side, where it may be an infinity).  Q < 8: element by element from 0.
__host__ __device__ __forceinline__ long long nm_d_window(long long q0, long long Q) { return Q < 8 || q0 + 8 <= Q ? q0 : Q - 8; }

// eight weights in PW pieces -> their place in each plane
template <int DT, int PW>
__device__ __forceinline__ void nm_d_put_weights(const NmOct<DT>& o, uint4* d) {
    if constexpr (PW == 1) {
        *d = o.v[0];
    } else {
        float f[8];
        uint4 x[PW];
        nm_oct_to_float<DT>(o, f);
        if constexpr (PW == 3) nm_d_cut8(f, x);
        else nm_d_two8(f, x);
#pragma unroll
        for (int q = 0; q < PW; ++q) d[q * 64] = x[q];
    }
}

// The streaming kernel's weights: dst [steps][tiles][plane][lane], zero beyond C and Q
template <int DT, int PW>
__global__ __launch_bounds__(256) void nm_dense_pack_kernel(const typename NmType<DT>::elem* __restrict__ w, long long ldw, int trans, int C, int Q, int tiles,
                                                            int steps, uint4* __restrict__ dst) {
    typedef typename NmType<DT>::elem T;
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    const int lane = (int)(t & 63), h = lane >> 4;
    const long long frag = t >> 6;
    const int tile = (int)(frag % tiles);
    const long long step = frag / tiles;
    if (step >= steps) return;
    const int c = nm_d_column<DT>(tile, lane & 15);
    const long long q0 = 32 * step + 8 * h, s0 = nm_d_window(q0, Q);
    NmOct<DT> o = nm_oct_zero<DT>();
    if (!trans) {
        if (c < C) {
            const T* row = w + (long long)c * ldw;
            if (Q < 8) { if (q0 == 0) o = nm_oct_load_short<DT>(row, Q); }
            else o = nm_oct_clear_first<DT>(nm_oct_load<DT>(row + s0), (int)(q0 - s0 < 8 ? q0 - s0 : 8));
        }
    } else {
        T e[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = c < C && s0 + k < Q && s0 + k >= q0 ? w[(s0 + k) * ldw + c] : (T)0.f;
        __builtin_memcpy(&o, e, sizeof(o));
    }
    nm_d_put_weights<DT, PW>(o, dst + ((step * tiles + tile) * PW) * 64 + lane);
}

// ------------------------------------------------------------------------------------------------ rows x weights
struct NmDenseArgs {
    const void* A; long long lda;        // rows [R, Q]
    const void* D;                       // PROD: factor of every element of A (kept derivatives), contiguous [R, Q]
    const void* W; long long ldw;        // column operand as it is: [C, Q], or (trans) [Q, C]
    const uint4* P; int tiles;           // ... in fragment order (streaming kernel)
    const void* bias;                    // [C] or NULL
    int trans, bias_f32;
    const void* res; long long ldr;      // added after the activation, [R, C] or NULL
    void* Y; long long ldy;              // [R, C]
    void* DV;                            // act'(z) (kept derivatives), contiguous [R, C], or NULL
    long long R;
    int Q, C, act;
    float beta;
    unsigned col_blocks;
};

// a piece of a row (times its factor) -> fragments
template <int DT, bool PROD, int PX>
__device__ __forceinline__ void nm_d_operand(const NmOct<DT>& a, const NmFactorOct<DT>& d, uint4 (&x)[PX]) {
    if constexpr (DT != NM_F32 && !PROD) {
        x[0] = a.v[0];
    } else {
        float f[8];
        nm_oct_to_float<DT>(a, f);
        if constexpr (PROD) {
            float g[8];
            nm_d_factors<DT>(d, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] *= g[e];
        }
        if constexpr (DT == NM_F32) nm_d_cut8(f, x);
        else nm_d_two8(f, x);
    }
}

// piece q .. q + 7 of a row of Q (its window, nm_d_window); rows shorter than eight: from the first lane group alone
template <int DT>
__device__ __forceinline__ NmOct<DT> nm_d_fetch(const typename NmType<DT>::elem* row, int q, int Q) {
    if (Q >= 8) return nm_oct_load<DT>(row + (q + 8 <= Q ? q : Q - 8));      // (uniform)
    return nm_oct_load_short<DT>(row, q == 0 ? Q : 0);
}

// Eight columns of one row as the matrix pipe leaves them to a lane: 16-bit: on end; fp32: two quads, 16 columns apart.
template <int DT>
__device__ __forceinline__ NmOct<DT> nm_d_load_cols(const typename NmType<DT>::elem* row, int c, int C) {
    if constexpr (DT != NM_F32) {
        return nm_oct_load_row<DT>(row, c, C);
    } else {
        NmOct<DT> o;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int at = c + 16 * k;
            o.v[k] = make_uint4(0, 0, 0, 0);
            if (at + 4 <= C) __builtin_memcpy(&o.v[k], row + at, 16);
            else if (at < C) o.v[k] = nm_oct_load_short<DT>(row + at, C - at).v[0];
        }
        return o;
    }
}
template <int DT>
__device__ __forceinline__ void nm_d_store_cols(typename NmType<DT>::elem* row, const float (&f)[8], int c, int C) {
    if constexpr (DT != NM_F32) {
        if (c < C) nm_oct_store_n<DT>(row + c, f, C - c);
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int at = c + 16 * k;
            if (at + 4 <= C) __builtin_memcpy(row + at, f + 4 * k, 16);
            else {
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (at + i < C) row[at + i] = f[4 * k + i];
            }
        }
    }
}

// ... of kept derivatives
template <int DT>
__device__ __forceinline__ void nm_d_store_factors(void* base, long long R, int C, long long m, const float (&f)[8], int c) {
    if constexpr (DT == NM_F32) {
        nm_d_store_cols<DT>((float*)base + m * C, f, c, C);
    } else {
        if (c >= C) return;
        const NmFactor<DT> at = nm_d_planes<DT>(base, R * C).at(m * C + c);
        char *hi = const_cast<char*>(at.hi), *lo = const_cast<char*>(at.lo);
        unsigned u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = nm_d_round24(f[i]);
        uint4 h = make_uint4(nm_d_pair(u[0], u[1]), nm_d_pair(u[2], u[3]), nm_d_pair(u[4], u[5]), nm_d_pair(u[6], u[7]));
        uint2 l;
        l.x = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0501u) | __builtin_amdgcn_perm(u[3], u[2], 0x05010c0cu);
        l.y = __builtin_amdgcn_perm(u[5], u[4], 0x0c0c0501u) | __builtin_amdgcn_perm(u[7], u[6], 0x05010c0cu);
        if (c + 8 <= C) {
            __builtin_memcpy(hi, &h, 16);
            __builtin_memcpy(lo, &l, 8);
            return;
        }
#pragma unroll 1
        for (int i = 0; i < C - c; ++i) {
            const unsigned short e = (unsigned short)h.x;
            __builtin_memcpy(hi + 2 * i, &e, 2);
            lo[i] = (char)l.x;
            h.x = h.x >> 16 | h.y << 16;
            h.y = h.y >> 16 | h.z << 16;
            h.z = h.z >> 16 | h.w << 16;
            h.w >>= 16;
            l.x = l.x >> 8 | l.y << 24;
            l.y >>= 8;
        }
    }
}

template <typename F, int... K>
__device__ __forceinline__ void nm_d_each(F f, std::integer_sequence<int, K...>) { (f(std::integral_constant<int, K>{}), ...); }

// accumulators of 16 RT rows x 32 NP columns -> bias (in LDS), activation, residual, stores.  A load waits for every store before it: a bias read from
// global memory here, piece by piece, cost a 131072 x 256 layer 8 of 52 us.  So the residual (RES) of eight pieces is in flight before the first store, and
// column blocks with one that stay resident have no more than eight pieces per wave (256 x 256 tiles: six ahead, eight would spill).  The scheduling barriers keep the pieces apart, and the opaque column makes its tests, biases and
// addresses HERE: mixed together or hoisted out of a loop over row tiles they cost 100 registers and spills.
template <int DT, bool PROD, bool RES, int RT, int NP, bool KEEP = !PROD>
__device__ __forceinline__ void nm_d_epilogue(const NmDenseArgs& p, const nm_v4f (&acc)[RT][2 * NP], const float* bias, long long m0, int cb,
                                              int lane) {
    typedef typename NmType<DT>::elem T;
    constexpr int PIECES = RT * NP, AHEAD = RT == 8 ? 6 : PIECES < 8 ? PIECES : 8;
    const float ibeta = 1.0f / p.beta;
    const int cw = cb * (32 * NP) + (DT == NM_F32 ? 4 : 8) * (lane >> 4);
    NmOct<DT> rs[AHEAD];
    auto row_of = [&](int piece) { return m0 + 16 * (piece / NP) + (lane & 15); };
    auto fetch = [&](int piece) {
        if (!RES || !p.res || piece >= PIECES) return;
        long long m = row_of(piece);
        m = m < p.R ? m : p.R - 1;
        int c = cw + 32 * (piece % NP);
        asm volatile("" : "+v"(c));
        rs[piece % AHEAD] = nm_d_load_cols<DT>((const T*)p.res + m * p.ldr, c, p.C);
    };
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) fetch(k);
    // (written out by a template: `#pragma unroll` gives up on pieces of this size, which leaves the accumulators in scratch memory)
    nm_d_each([&](auto piece) __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        constexpr int k = decltype(piece)::value, r = k / NP, n = k % NP;
        const long long m = row_of(k);
        int c = cw + 32 * n;
        asm volatile("" : "+v"(c));
        float z[8], dv[8], q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = acc[r][2 * n + (i >> 2)][i & 3];
        if (!PROD && p.bias) {
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] += bias[c - cb * (32 * NP) + (DT == NM_F32 ? 16 * (i >> 2) + (i & 3) : i)];
        }
        if (RES && p.res) {
            nm_oct_to_float<DT>(rs[k % AHEAD], q);
            fetch(k + AHEAD);
        }
        if constexpr (!PROD) nm_d_act<DT == NM_F32>(p.act, p.beta, ibeta, KEEP && p.DV, z, dv);
        if (m >= p.R) return;
        if constexpr (!PROD) {
            if (KEEP && p.DV) nm_d_store_factors<DT>(p.DV, p.R, p.C, m, dv, c);
            if (RES && p.res) {
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] += q[i];
            }
        }
        nm_d_store_cols<DT>((T*)p.Y + m * p.ldy, z, c, p.C);
    }, std::make_integer_sequence<int, PIECES>{});
}

template <int DT>
__device__ __forceinline__ float nm_d_bias(const NmDenseArgs& p, int c) {
    return c >= p.C ? 0.f : p.bias_f32 ? ((const float*)p.bias)[c] : (float)((const typename NmType<DT>::elem*)p.bias)[c];
}

// a weight block -> LDS in fragment order, [step][tile][plane][lane], by 512 threads; zero beyond C and Q
template <int DT, int PW, int NP>
__device__ __forceinline__ void nm_d_load_block(const NmDenseArgs& p, int cb, int steps, uint4* lds, int t) {
    typedef typename NmType<DT>::elem T;
    const T* w = (const T*)p.W;
    if (!p.trans) {                                          // a lane's eight contraction elements lie on end: one piece each
        const int n = steps * 2 * NP * 64;
#pragma unroll 8
        for (int i = t; i < n; i += 512) {
            const int lane = i & 63, tile = (i >> 6) % (2 * NP), s = (i >> 6) / (2 * NP);
            const int c = cb * (32 * NP) + nm_d_column<DT>(tile, lane & 15), q0 = 32 * s + 8 * (lane >> 4);
            NmOct<DT> o = nm_d_fetch<DT>(w + (long long)(c < p.C ? c : p.C - 1) * p.ldw, q0, p.Q);
            const int sh = c >= p.C ? 8 : p.Q < 8 || q0 + 8 <= p.Q ? 0 : q0 + 8 - p.Q;
            nm_d_put_weights<DT, PW>(nm_oct_clear_first<DT>(o, sh), lds + (i >> 6) * (PW * 64) + lane);
        }
        return;
    }
    // transposed: eight rows x eight columns per thread, columns side by side over the threads
    const int n = steps * 4 * (4 * NP);                      // groups of eight rows x groups of eight columns
    for (int i = t; i < n; i += 512) {
        const int g = i % (4 * NP), qg = i / (4 * NP);
        const int c = cb * (32 * NP) + 8 * g, q0 = 8 * qg, s0 = (int)nm_d_window(q0, p.Q);
        NmOct<DT> v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int q = s0 + e;
            v[e] = nm_oct_zero<DT>();
            if (q >= q0 && q < p.Q) v[e] = nm_oct_load_row<DT>(w + (long long)q * p.ldw, c, p.C);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // tile and position of column 8 g + e of the block
            const int tile = DT == NM_F32 ? g >> 1 : 2 * (g >> 2) + (e >> 2), pos = DT == NM_F32 ? 8 * (g & 1) + e : 4 * (g & 3) + (e & 3);
            uint4* d = lds + ((qg >> 2) * (2 * NP) + tile) * (PW * 64) + 16 * (qg & 3) + pos;
            NmOct<DT> o;
            if constexpr (DT == NM_F32) {
                float f[8], a[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    nm_oct_to_float<DT>(v[k], a);
                    f[k] = a[e];
                }
                __builtin_memcpy(&o, f, sizeof(o));
            } else {
                const unsigned sel = (e & 1) ? 0x07060302u : 0x05040100u;
                unsigned r[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) r[k] = (e >> 1) == 0 ? v[k].v[0].x : (e >> 1) == 1 ? v[k].v[0].y : (e >> 1) == 2 ? v[k].v[0].z : v[k].v[0].w;
                o.v[0] = make_uint4(__builtin_amdgcn_perm(r[1], r[0], sel), __builtin_amdgcn_perm(r[3], r[2], sel), __builtin_amdgcn_perm(r[5], r[4], sel),
                                    __builtin_amdgcn_perm(r[7], r[6], sel));
            }
            nm_d_put_weights<DT, PW>(o, d);
        }
    }
}

// Many rows against a weight block that FITS in LDS (32-deep steps x 16-column tiles x pieces <= NM_D_RESIDENT KB): one persistent workgroup per CU loads
// it once, and its eight waves then walk over tiles of 32 rows, each for itself, without another barrier.  A wave owns whole rows: their elements
// go from global memory straight into fragments (a lane's 8 consecutive elements of one row ARE a fragment), RING steps ahead of their use
// and across the end of a tile: the next tile's rows are in flight while this one's results are stored.
// Measured (counters: profiles/ops_counters.txt): 65536 x 256 -> 256 fp32 with softplus 83 us (51.5 G multiplications and additions as six bf16 products: 620 TFLOP/s;
// the rows are cut into pieces once per column block, the vector unit is busy 56 % of the time, the matrix pipe 27 %) and its dx 90 us (570 TFLOP/s; address units busy
// 73 %); dx of 131072 x 256 -> 256 bf16 65 us (234 MB with the kept derivatives: 3.6 TB/s, address units 62 %).
#define NM_D_RESIDENT 144

template <int DT, bool PROD, int NP>
__global__ __launch_bounds__(512, 2) void nm_dense_resident_kernel(NmDenseArgs p) {
    typedef typename NmType<DT>::elem T;
    constexpr int PW = NmPieces<DT, PROD>::PLAIN, PX = NmPieces<DT, PROD>::ROWS, MF = NmPieces<DT, PROD>::MF;
    constexpr int RING = DT == NM_F32 || (PROD && NP == 8) ? 2 : 4;
    __shared__ uint4 lds[NM_D_RESIDENT * 64];
    __shared__ float bias[32 * NP];
    const int t = threadIdx.x, lane = t & 63, li = lane & 15, h = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // consecutive workgroup numbers go to the eight XCDs in turn: the column blocks of one share of the rows sit on one XCD and read them together
    const unsigned id = blockIdx.x, turn = id >> 3;
    const int cb = (int)(turn % p.col_blocks);
    const long long slot = (long long)(turn / p.col_blocks) * 8 + (id & 7), slots = gridDim.x / p.col_blocks;
    const int steps = (p.Q + 31) / 32;
    const long long tiles = (p.R + 31) / 32;
    const T* arow[2];
    const NmFactor<DT> planes = nm_d_planes<DT>(p.D, p.R * p.Q);
    NmFactor<DT> drow[2];
    auto rows_of = [&](long long tile) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            long long m = tile * 32 + 16 * r + li;
            m = m < p.R ? m : p.R - 1;
            arow[r] = (const T*)p.A + m * p.lda;
            if constexpr (PROD) drow[r] = planes.at(m * p.Q);
        }
    };
    NmOct<DT> xa[RING][2];
    NmFactorOct<DT> xd[RING][2];
    auto fetch = [&](int s, NmOct<DT> (&a)[2], NmFactorOct<DT> (&d)[2]) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            a[r] = nm_d_fetch<DT>(arow[r], 32 * s + 8 * h, p.Q);
            if constexpr (PROD) d[r] = nm_d_fetch_factors<DT>(drow[r], 32 * s + 8 * h, p.Q);
        }
    };
    long long tile = slot * 8 + wave;
    if (tile < tiles) {
        rows_of(tile);
#pragma unroll
        for (int u = 0; u < RING; ++u)
            if (u < steps) fetch(u, xa[u], xd[u]);
    }
    nm_d_load_block<DT, PW, NP>(p, cb, steps, lds, t);
    if (!PROD && p.bias && t < 32 * NP) bias[t] = nm_d_bias<DT>(p, cb * (32 * NP) + t);
    __syncthreads();
    for (; tile < tiles; tile += slots * 8) {
        nm_v4f acc[2][2 * NP];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int n = 0; n < 2 * NP; ++n) acc[r][n] = nm_v4f{0.f, 0.f, 0.f, 0.f};
        const bool more = tile + slots * 8 < tiles;
        for (int b = 0; b < steps; b += RING) {
#pragma unroll
            for (int u = 0; u < RING; ++u) {
                const int s = b + u;
                if (s >= steps) break;                       // (uniform)
                __builtin_amdgcn_sched_barrier(0);           // (one step's pieces at a time)
                uint4 x[2][PX];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    NmOct<DT> a = xa[u][r];
                    NmFactorOct<DT> d = xd[u][r];
                    if (32 * s + 32 > p.Q && p.Q >= 8) {     // what the last whole load repeated
                        const int q = 32 * s + 8 * h, sh = q + 8 <= p.Q ? 0 : q + 8 - p.Q;
                        a = nm_oct_clear_first<DT>(a, sh);
                        if constexpr (PROD) d = nm_d_clear_factors<DT>(d, sh);
                    }
                    nm_d_operand<DT, PROD>(a, d, x[r]);
                }
                if (s + RING < steps) {
                    fetch(s + RING, xa[u], xd[u]);
                } else if (more) {                           // the first use of this place in the next tile
                    if (s == (steps > RING ? steps - RING : 0)) rows_of(tile + slots * 8);
                    fetch(u, xa[u], xd[u]);
                }
#pragma unroll
                for (int n = 0; n < 2 * NP; ++n) {
                    uint4 w[PW];
#pragma unroll
                    for (int q = 0; q < PW; ++q) w[q] = lds[((s * (2 * NP) + n) * PW + q) * 64 + lane];
#pragma unroll
                    for (int r = 0; r < 2; ++r) acc[r][n] = nm_d_products<MF>(w, x[r], acc[r][n]);
                }
            }
        }
        nm_d_epilogue<DT, PROD, !PROD && NP <= 4, 2, NP>(p, acc, bias, tile * 32, cb, lane);
    }
}

// Large 16-bit layers, W as it lies: 256 rows x 256 columns per workgroup of eight waves (128 x 64 each).  Both operands come in panels of 64
// contraction elements as whole 128-byte lines, eight lanes a line -- the kernel above reads rows straight into fragments, sixteen rows side by side, which keeps
// the address units busy for 62 .. 73 % of its time, this one for 22 .. 28 % -- and go through LDS, in two buffers, with one barrier per panel and
// the next panel in flight in registers.  The eight 16-byte pieces of an LDS row are exchanged by the row's number, so that the sixteen rows of a fragment
// lie in different banks.
// Measured: 16384 x 1024 -> 1024 bf16 with GELU and residual 55 us (34.4 GFLOP: 630 TFLOP/s); 65536 x 207 -> 256 with ReLU 24 us (60.8 MB: 2.5 TB/s); 131072 x
// 256 -> 256 with softplus, residual and kept derivatives 105 us (302 MB: 2.9 TB/s).  Waves wait 43 .. 58 % of their time: load, product, activation and store add
// up, since the one workgroup of a CU has all its waves in the same phase.  Results and residual through LDS, in whole lines, changed nothing.
// KEEP: with kept derivatives.  One kernel for both has 81 KB of instructions, and calls without derivatives paid for them (the second layer: 28.6 us a call instead of 21.5).
template <int DT, bool KEEP>
__global__ __launch_bounds__(512, 2) void nm_dense_tile_kernel(NmDenseArgs p) {
    typedef typename NmType<DT>::elem T;
    __shared__ uint4 lds[2][2][256 * 8];                     // [buffer][rows, columns][row][piece]
    __shared__ float bias[256];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, li = lane & 15, h = lane >> 4, wr = wave >> 2, wc = wave & 3;
    const unsigned id = blockIdx.x, turn = id >> 3;          // (XCDs: see above)
    const long long rb = (long long)(turn / p.col_blocks) * 8 + (id & 7);
    const int cb = (int)(turn % p.col_blocks);
    if (rb * 256 >= p.R) return;
    const int panels = (p.Q + 63) / 64, piece = t & 7;
    // this thread's pieces: rows t / 8 + 64 i of both sides (LDS row n of the columns' side: the column that nm_d_column puts there)
    const T* src[2][4];
    int dst[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = (t >> 3) + 64 * i;
        const long long m = rb * 256 + n;
        const int c = cb * 256 + nm_d_column<DT>(n >> 4, n & 15);
        src[0][i] = (const T*)p.A + (m < p.R ? m : p.R - 1) * p.lda;
        src[1][i] = (const T*)p.W + (long long)(c < p.C ? c : p.C - 1) * p.ldw;
        dst[i] = n * 8 + (piece ^ ((n >> 1) & 7));
    }
    NmOct<DT> v[2][4];
    auto load = [&](int panel) {
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[o][i] = nm_d_fetch<DT>(src[o][i], panel * 64 + 8 * piece, p.Q);
    };
    auto store = [&](int panel) {
        if ((panel + 1) * 64 > p.Q && p.Q >= 8) {            // what the last whole load repeated
            const int q = panel * 64 + 8 * piece, sh = q + 8 <= p.Q ? 0 : q + 8 - p.Q;
#pragma unroll
            for (int o = 0; o < 2; ++o)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[o][i] = nm_oct_clear_first<DT>(v[o][i], sh < 8 ? sh : 8);
        }
#pragma unroll
        for (int o = 0; o < 2; ++o)
#pragma unroll
            for (int i = 0; i < 4; ++i) lds[panel & 1][o][dst[i]] = v[o][i].v[0];
    };
    nm_v4f acc[8][4];
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[r][n] = nm_v4f{0.f, 0.f, 0.f, 0.f};

    if (p.bias && t < 256) bias[t] = nm_d_bias<DT>(p, cb * 256 + t);
    load(0);
    store(0);
    __syncthreads();
    const int at = li * 8 + (h ^ (li >> 1));                 // piece h of a fragment's row; the panel's second half: ^ 4
    for (int k = 0; k < panels; ++k) {
        // (a wave that is a panel ahead fills the OTHER buffer; nobody is two panels ahead)
        if (k + 1 < panels) load(k + 1);
        const uint4 *x = lds[k & 1][0] + wr * 1024, *w = lds[k & 1][1] + wc * 512;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint4 b[4][1];
#pragma unroll
            for (int n = 0; n < 4; ++n) b[n][0] = w[n * 128 + (at ^ (4 * s))];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                uint4 a[1] = {x[r * 128 + (at ^ (4 * s))]};
#pragma unroll
                for (int n = 0; n < 4; ++n) acc[r][n] = nm_d_products<DT>(b[n], a, acc[r][n]);
            }
        }
        if (k + 1 < panels) store(k + 1);
        __syncthreads();
    }
    nm_d_epilogue<DT, false, true, 8, 2, KEEP>(p, acc, bias + wc * 64, rb * 256 + wr * 128, cb * 4 + wc, lane);
}

// Otherwise: one workgroup: 4 waves, 64 RT rows x 32 NP columns, both sides streamed.  The rows as above; the column operand is shared by the four waves
// through LDS, PS steps at a time in two buffers, one barrier per panel, both sides' next panel in flight in registers meanwhile.
// Measured: 4096 x 1024 -> 1024 bf16 with GELU 43 us, 16384 x 520 -> 300 25 us; bound by latency: one workgroup of four waves per CU, waiting 63 % of their time.
template <int DT, bool PROD, int RT, int NP, int PS>
__global__ __launch_bounds__(256, 2) void nm_dense_stream_kernel(NmDenseArgs p) {
    typedef typename NmType<DT>::elem T;
    constexpr int PW = NmPieces<DT, PROD>::PLAIN, PX = NmPieces<DT, PROD>::ROWS, MF = NmPieces<DT, PROD>::MF;
    constexpr int STEP = 2 * NP * PW * 64, PANEL = PS * STEP, WV = PANEL / 256;      // uint4
    static_assert(PANEL % 256 == 0, "a panel is whole 16-byte pieces per thread");
    __shared__ uint4 lds[2][PANEL];
    __shared__ float bias[32 * NP];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, li = lane & 15, h = lane >> 4;
    const unsigned id = blockIdx.x, turn = id >> 3;          // (XCDs: see above)
    const long long rb = (long long)(turn / p.col_blocks) * 8 + (id & 7);
    const int cb = (int)(turn % p.col_blocks);
    const long long m0 = rb * (64 * RT) + wave * (16 * RT);
    if (rb * (64 * RT) >= p.R) return;
    const int steps = (p.Q + 31) / 32, panels = (steps + PS - 1) / PS;
    const T* arow[RT];
    const NmFactor<DT> planes = nm_d_planes<DT>(p.D, p.R * p.Q);
    NmFactor<DT> drow[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        long long m = m0 + 16 * r + li;
        m = m < p.R ? m : p.R - 1;
        arow[r] = (const T*)p.A + m * p.lda;
        if constexpr (PROD) drow[r] = planes.at(m * p.Q);
    }
    nm_v4f acc[RT][2 * NP];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < 2 * NP; ++n) acc[r][n] = nm_v4f{0.f, 0.f, 0.f, 0.f};

    uint4 wv[WV];
    NmOct<DT> xa[PS][RT];
    NmFactorOct<DT> xd[PS][RT];
    auto load_w = [&](int panel) {
#pragma unroll
        for (int i = 0; i < WV; ++i) {
            const int e = i * 256 + t;
            wv[i] = p.P[((long long)(panel * PS + e / STEP) * p.tiles + cb * (2 * NP)) * (PW * 64) + e % STEP];
        }
    };
    auto store_w = [&](int buf) {
#pragma unroll
        for (int i = 0; i < WV; ++i) lds[buf][i * 256 + t] = wv[i];
    };
    auto load_x = [&](int panel, NmOct<DT> (&a)[PS][RT], NmFactorOct<DT> (&d)[PS][RT]) {
#pragma unroll
        for (int s = 0; s < PS; ++s)
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                a[s][r] = nm_d_fetch<DT>(arow[r], (panel * PS + s) * 32 + 8 * h, p.Q);
                if constexpr (PROD) d[s][r] = nm_d_fetch_factors<DT>(drow[r], (panel * PS + s) * 32 + 8 * h, p.Q);
            }
    };
    // the last panel: clear what a whole load repeated or brought beyond the row
    auto trim = [&](int panel, NmOct<DT> (&a)[PS][RT], NmFactorOct<DT> (&d)[PS][RT]) {
        if ((panel + 1) * (32 * PS) <= p.Q || p.Q < 8) return;
#pragma unroll
        for (int s = 0; s < PS; ++s) {
            const int q = (panel * PS + s) * 32 + 8 * h, sh = q + 8 <= p.Q ? 0 : q + 8 - p.Q;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                a[s][r] = nm_oct_clear_first<DT>(a[s][r], sh);
                if constexpr (PROD) d[s][r] = nm_d_clear_factors<DT>(d[s][r], sh);
            }
        }
    };
    auto compute = [&](int buf, const NmOct<DT> (&a)[PS][RT], const NmFactorOct<DT> (&d)[PS][RT]) {
#pragma unroll
        for (int s = 0; s < PS; ++s) {
            __builtin_amdgcn_sched_barrier(0);               // (one step's pieces at a time)
            uint4 x[RT][PX];
#pragma unroll
            for (int r = 0; r < RT; ++r) nm_d_operand<DT, PROD>(a[s][r], d[s][r], x[r]);
#pragma unroll
            for (int n = 0; n < 2 * NP; ++n) {
                uint4 w[PW];
#pragma unroll
                for (int q = 0; q < PW; ++q) w[q] = lds[buf][((s * (2 * NP) + n) * PW + q) * 64 + lane];
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[r][n] = nm_d_products<MF>(w, x[r], acc[r][n]);
            }
        }
    };

    if (!PROD && p.bias && t < 32 * NP) bias[t] = nm_d_bias<DT>(p, cb * (32 * NP) + t);
    if (panels > 0) {
        load_w(0);
        load_x(0, xa, xd);
        store_w(0);
    }
    __syncthreads();
    for (int k = 0; k < panels; ++k) {
        // (a wave that is a panel ahead fills the OTHER buffer; nobody is two panels ahead: one barrier per panel)
        NmOct<DT> na[PS][RT];
        NmFactorOct<DT> nd[PS][RT];
        if (k + 1 < panels) {
            load_w(k + 1);
            load_x(k + 1, na, nd);
        }
        trim(k, xa, xd);
        compute(k & 1, xa, xd);
        if (k + 1 < panels) store_w((k + 1) & 1);
        __syncthreads();
#pragma unroll
        for (int s = 0; s < PS; ++s)
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                xa[s][r] = na[s][r];
                if constexpr (PROD) xd[s][r] = nd[s][r];
            }
    }
    nm_d_epilogue<DT, PROD, !PROD, RT, NP>(p, acc, bias, m0, cb, lane);
}

// ------------------------------------------------------------------------------------------------ a few rows
// 1 .. MR rows: bound by the read of the weights and by latency.  16 lanes share a column (8 elements each per round), so W is read once, in its own
// layout, with whole 16-byte pieces, and the partial sums meet in four lane exchanges; plain fp32 multiply-adds.  1 x 256 -> 256 fp16: 3.5 us, the latency of a launch and two loads.
template <int DT, int MR>
__global__ __launch_bounds__(256) void nm_dense_few_kernel(const typename NmType<DT>::elem* __restrict__ x, long long ldx,
                                                           const typename NmType<DT>::elem* __restrict__ w, long long ldw, const void* __restrict__ bias, int bias_f32,
                                                           const typename NmType<DT>::elem* __restrict__ res, long long ldr, int M, int K, int N, int act, float beta,
                                                           typename NmType<DT>::elem* __restrict__ y, long long ldy, void* __restrict__ dv) {
    typedef typename NmType<DT>::elem T;
    const int sub = threadIdx.x & 15, n = blockIdx.x * 16 + (threadIdx.x >> 4);
    float acc[MR];
#pragma unroll
    for (int m = 0; m < MR; ++m) acc[m] = 0.f;
    if (n < N) {
        for (int k = sub * 8; k < K; k += 128) {
            float a[8];
            nm_oct_to_float<DT>(nm_oct_load_row<DT>(w + (long long)n * ldw, k, K), a);
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                float b[8];
                nm_oct_to_float<DT>(nm_oct_load_row<DT>(x + (long long)(m < M ? m : M - 1) * ldx, k, K), b);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[m] = fmaf(a[e], b[e], acc[m]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) acc[m] += __shfl_xor(acc[m], o);
    }
    float z = acc[0];
#pragma unroll
    for (int m = 1; m < MR; ++m) z = sub == m ? acc[m] : z;
    if (n >= N || sub >= M) return;
    if (bias) z += bias_f32 ? ((const float*)bias)[n] : (float)((const T*)bias)[n];
    float hv[1] = {z}, d[1];
    nm_d_act<DT == NM_F32>(act, beta, 1.0f / beta, dv != nullptr, hv, d);
    float h = hv[0];
    if (res) h += (float)res[sub * ldr + n];
    y[sub * ldy + n] = (T)h;
    if (!dv) return;
    const long long at = (long long)sub * N + n;
    if constexpr (DT == NM_F32) {
        ((float*)dv)[at] = d[0];
    } else {
        const unsigned u = nm_d_round24(d[0]);
        ((unsigned short*)dv)[at] = (unsigned short)(u >> 16);
        ((unsigned char*)dv)[2LL * M * N + at] = (unsigned char)(u >> 8);
    }
}

// ------------------------------------------------------------------------------------------------ weight and bias gradient
// dW = dz^T x, contraction over the rows.  One workgroup: a 128 x 128 tile of dW over a range of rows, in blocks of 64 (fp32: 32); 4 waves of 64 x 64.
// The contraction is the SLOW axis of both operands.  A thread loads eight rows x CG columns of each (8-byte pieces, whole lines per row) and
// transposes them in its own registers (one byte permute per two elements, or on the way through the product's fp32): it then holds, for each of its
// columns, eight consecutive rows -- a fragment -- and writes it to LDS in the order in which the waves read fragments.  Every wave brings its share of
// dz (from g and act'(z), in two pieces or three) AND of x: the conversions, which cost as much as the products, are spread over the four
// SIMDs.  The next block's rows are in flight while this one is multiplied.
// Measured: 256 x 256 weights, 131072 rows bf16 68 us (234 MB with the kept derivatives: 3.5 TB/s), 65536 rows fp32 65 us (51.5 G as six products: 790 TFLOP/s).
struct NmDenseGradArgs {
    const void* G; long long ldg; const void* D;   // dz = G * D (D contiguous [R, N], kept derivatives, or NULL)
    const void* X; long long ldx;
    long long R;
    int N, K, n_tiles, k_tiles, splits;
    long long rows;                      // rows per workgroup (a multiple of 64)
    float* part;                         // [splits][n_tiles * k_tiles][16384] in the order of the accumulators; one split: NULL, straight to
    void* dw; void* db; int db_f32;      // dW [N, K] (or NULL) and db [N] (or NULL)
    float* bias_part;                    // [splits][128 n_tiles], or NULL: db is not wanted, or one split
};

template <int DT> struct NmGroup { static constexpr int C = DT == NM_F32 ? 2 : 4; };    // columns of a thread: 8 bytes
// Position i of the matrix pipe's tile t -> the thread group (of columns) and its column.  Lanes that follow each other sit at consecutive positions: whole
// 256 bytes per 16 lanes go into LDS.
template <int DT>
__host__ __device__ __forceinline__ void nm_d_place(int t, int i, int& group, int& e) {
    if (DT == NM_F32) { group = i + 32 * (t & 1); e = t >> 1; }
    else { group = i; e = t; }
}
// first column of the group that belongs at c: a group that would end beyond the row is the row's last one (nm_dense_sum_kernel takes the columns that
// are its own)
template <int DT>
__host__ __device__ __forceinline__ int nm_d_group(int c, int n) { return n < NmGroup<DT>::C ? 0 : c + NmGroup<DT>::C <= n ? c : n - NmGroup<DT>::C; }

// The thread's eight rows 8 rg .. of a block of `rows` <= full rows at row `base`, a piece V of columns col .. (ncol: of the array).  An address is a uniform base and a
// 32-bit offset of the lane (strides are below 2^24): 24 addresses of 64 bits per lane cost more registers than the data.  All three forms are
// straight code without branches per lane; rows beyond the block read its last row and are cleared.
template <typename T, typename V>
__device__ __forceinline__ void nm_d_load_rows(const T* src, long long ld, int ncol, int col, long long base, int rows, int full, int rg, V (&v)[8]) {
    constexpr unsigned E = sizeof(T), G = sizeof(V) / E;
    const char* at = (const char*)(src + base * ld);
    if (ncol >= (int)G && rows == full) {                    // (uniform)
        const unsigned off = (unsigned)(rg * 8 * (unsigned)ld + col) * E;
#pragma unroll
        for (int r = 0; r < 8; ++r) __builtin_memcpy(&v[r], (const T*)(at + r * ld * E + off), sizeof(V));
        return;
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const int m = rg * 8 + r < rows ? rg * 8 + r : rows - 1;
        const unsigned off = ((unsigned)m * (unsigned)ld + col) * E;
        v[r] = V{};
        if (ncol >= (int)G) {
            __builtin_memcpy(&v[r], (const T*)(at + off), sizeof(V));
        } else if (ncol > 0) {                               // fewer columns than a group: one by one, the last one again
            T x[G];
#pragma unroll
            for (int e = 0; e < (int)G; ++e) x[e] = *(const T*)(at + off + (e < ncol ? e : ncol - 1) * E);
            __builtin_memcpy(&v[r], x, sizeof(V));
        }
        if (rg * 8 + r >= rows) v[r] = V{};
    }
}
template <int DT>
__device__ __forceinline__ float nm_d_element(const uint2& v, int e) {
    typename NmType<DT>::elem x[8 / sizeof(typename NmType<DT>::elem)];
    __builtin_memcpy(x, &v, 8);
    return nm_to_float<DT>(x[e]);
}
// column e of a piece of kept derivatives
template <int DT>
__device__ __forceinline__ float nm_d_factor(const uint2& hi, unsigned lo, int e) {
    if constexpr (DT == NM_F32) return __uint_as_float(e ? hi.y : hi.x);
    else return e == 0 ? nm_d_join<0, 0>(hi.x, lo) : e == 1 ? nm_d_join<1, 1>(hi.x, lo) : e == 2 ? nm_d_join<0, 2>(hi.y, lo) : nm_d_join<1, 3>(hi.y, lo);
}
// 16-bit elements: column e of eight rows
__device__ __forceinline__ uint4 nm_d_column16(const uint2 (&r)[8], int e) {
    const unsigned sel = (e & 1) ? 0x07060302u : 0x05040100u;
    unsigned w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = e < 2 ? r[j].x : r[j].y;
    return make_uint4(__builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[3], w[2], sel), __builtin_amdgcn_perm(w[5], w[4], sel),
                      __builtin_amdgcn_perm(w[7], w[6], sel));
}

// four values of a lane's accumulators (rows 8 rq + 4 (lane / 32) .. of tile `ti`, position lane % 32 of tile `tj`) -> dW
template <int DT>
__device__ __forceinline__ void nm_d_put_grad(typename NmType<DT>::elem* dw, int N, int K, int tn, int tk, int ti, int tj, int lane, int rq, const float4& s) {
    constexpr int CG = NmGroup<DT>::C;
    int gr, e;
    nm_d_place<DT>(tj, lane & 31, gr, e);
    const int gk = tk * 128 + gr * CG, k = nm_d_group<DT>(gk, K) + e;
    if (k < gk || k >= K) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        nm_d_place<DT>(ti, q + 8 * rq + 4 * (lane >> 5), gr, e);
        const int gn = tn * 128 + gr * CG, n = nm_d_group<DT>(gn, N) + e;
        if (n >= gn && n < N) dw[(long long)n * K + k] = (typename NmType<DT>::elem)(q == 0 ? s.x : q == 1 ? s.y : q == 2 ? s.z : s.w);
    }
}

template <int DT, bool PROD>
__global__ __launch_bounds__(256, 2) void nm_dense_grad_kernel(NmDenseGradArgs p) {
    typedef typename NmType<DT>::elem T;
    typedef typename std::conditional<DT == NM_F32, float, unsigned short>::type TD;
    constexpr int CG = NmGroup<DT>::C;
    constexpr int PZ = NmPieces<DT, PROD>::ROWS, PX = NmPieces<DT, PROD>::PLAIN, MF = NmPieces<DT, PROD>::MF;
    constexpr int LANES = 128 / CG;                          // lanes side by side
    constexpr int ROWS = 8 * 4 * (64 / LANES), STEPS = ROWS / 16;
    __shared__ uint4 lds[(PZ + PX) * STEPS * 256];           // [plane][step][tile 4][lane 64], dz then x
    constexpr int LZ = PZ * STEPS * 256;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // the tiles of one range of rows on one XCD, at the same time: they read the same rows
    const unsigned turn = blockIdx.x >> 3, tile = turn % (p.n_tiles * p.k_tiles), split = turn / (p.n_tiles * p.k_tiles) * 8 + (blockIdx.x & 7);
    if ((int)split >= p.splits) return;
    const int tn = (int)(tile / p.k_tiles), tk = (int)(tile % p.k_tiles);
    const long long r0 = (long long)split * p.rows, r1 = r0 + p.rows < p.R ? r0 + p.rows : p.R;
    const int cg = t % LANES, rg = t / LANES;                // group of columns, group of eight rows
    const int coln = nm_d_group<DT>(tn * 128 + cg * CG, p.N), colk = nm_d_group<DT>(tk * 128 + cg * CG, p.K);
    const bool want_bias = (p.bias_part || p.db) && tk == 0;
    float bsum[CG];
#pragma unroll
    for (int e = 0; e < CG; ++e) bsum[e] = 0.f;
    nm_v16f acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    const NmFactor<DT> planes = nm_d_planes<DT>(p.D, p.R * p.N);
    uint2 vg[8], vd[8], vx[8];
    unsigned vl[8];
    auto load = [&](long long base) {
        const int rows = r1 - base < ROWS ? (int)(r1 - base) : ROWS;
        nm_d_load_rows((const T*)p.G, p.ldg, p.N, coln, base, rows, ROWS, rg, vg);
        if constexpr (PROD) nm_d_load_rows((const TD*)planes.hi, p.N, p.N, coln, base, rows, ROWS, rg, vd);
        if constexpr (PROD && DT != NM_F32) nm_d_load_rows((const unsigned char*)planes.lo, p.N, p.N, coln, base, rows, ROWS, rg, vl);
        nm_d_load_rows((const T*)p.X, p.ldx, p.K, colk, base, rows, ROWS, rg, vx);
    };
    // a fragment of this thread -> LDS: its column e, rows 8 rg ..
    auto put = [&](uint4* base, const uint4& c, int e) {
        const int tt = DT == NM_F32 ? 2 * e + (cg >> 5) : e;
        base[(rg >> 1) * 256 + tt * 64 + (rg & 1) * 32 + (cg & 31)] = c;
    };
    auto stash = [&]() {
#pragma unroll
        for (int e = 0; e < CG; ++e) {                       // one column: eight rows -> a fragment per plane
            __builtin_amdgcn_sched_barrier(0);               // (one column's temporaries at a time)
            float f[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                f[r] = nm_d_element<DT>(vg[r], e);
                if constexpr (PROD) f[r] *= nm_d_factor<DT>(vd[r], vl[r], e);
                if (want_bias) bsum[e] += f[r];
            }
            if constexpr (DT == NM_F32) {
                uint4 c[3];
                nm_d_cut8(f, c);
#pragma unroll
                for (int q = 0; q < 3; ++q) put(lds + q * STEPS * 256, c[q], e);
#pragma unroll
                for (int r = 0; r < 8; ++r) f[r] = nm_d_element<DT>(vx[r], e);
                nm_d_cut8(f, c);
#pragma unroll
                for (int q = 0; q < 3; ++q) put(lds + LZ + q * STEPS * 256, c[q], e);
            } else {
                if constexpr (PROD) {
                    uint4 c[2];
                    nm_d_two8(f, c);
                    put(lds, c[0], e);
                    put(lds + STEPS * 256, c[1], e);
                } else {
                    put(lds, nm_d_column16(vg, e), e);
                }
                if constexpr (PX == 2) {
                    uint4 c[2];
#pragma unroll
                    for (int r = 0; r < 8; ++r) f[r] = nm_d_element<DT>(vx[r], e);
                    nm_d_two8(f, c);
                    put(lds + LZ, c[0], e);
                    put(lds + LZ + STEPS * 256, c[1], e);
                } else {
                    put(lds + LZ, nm_d_column16(vx, e), e);
                }
            }
        }
    };

    const int wn = wave & 1, wk = wave >> 1;
    if (r0 < r1) load(r0);
    for (long long b = r0; b < r1; b += ROWS) {
        stash();
        if (b + ROWS < r1) load(b + ROWS);
        __syncthreads();
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if (s % 2 == 0) __builtin_amdgcn_sched_barrier(0);
            uint4 z[2][PZ], x[2][PX];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int q = 0; q < PZ; ++q) z[i][q] = lds[(q * STEPS + s) * 256 + (2 * wn + i) * 64 + lane];
#pragma unroll
                for (int q = 0; q < PX; ++q) x[i][q] = lds[LZ + (q * STEPS + s) * 256 + (2 * wk + i) * 64 + lane];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = nm_d_products<MF>(z[i], x[j], acc[i][j]);
        }
        __syncthreads();
    }
    if (p.part) {
        float* out = p.part + ((long long)split * (p.n_tiles * p.k_tiles) + tile) * 16384 + wave * 4096;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<float4*>(out + ((i * 2 + j) * 4 + (r >> 2)) * 256 + lane * 4) =
                        make_float4(acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]);
    } else if (p.dw) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    nm_d_put_grad<DT>((T*)p.dw, p.N, p.K, tn, tk, 2 * wn + i, 2 * wk + j, lane, r >> 2,
                                      make_float4(acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]));
    }
    if (!want_bias) return;                                  // (uniform over the workgroup)
    float* sh = reinterpret_cast<float*>(lds);               // [row group][128]
#pragma unroll
    for (int e = 0; e < CG; ++e) sh[rg * 128 + cg * CG + e] = bsum[e];
    __syncthreads();
    if (t < 128) {
        float b = 0.f;
#pragma unroll
        for (int g = 0; g < ROWS / 8; ++g) b += sh[g * 128 + t];
        if (p.bias_part) {
            p.bias_part[((long long)split * p.n_tiles + tn) * 128 + t] = b;
        } else {
            const int gn = tn * 128 + t / CG * CG, n = nm_d_group<DT>(gn, p.N) + t % CG;
            if (n >= gn && n < p.N) {
                if (p.db_f32) ((float*)p.db)[n] = b;
                else ((T*)p.db)[n] = (T)b;
            }
        }
    }
}

// partial sums -> dW [N, K], db [N].  Eight groups of threads take the splits s, s + 8, .. of the same 64 pieces, and their sums are added in order
// (what 128 partial sums of a 256 x 256 weight cost is latency: 8.9 us, and 15 with four groups and the bias left to one of them).
template <int DT>
__global__ __launch_bounds__(512) void nm_dense_sum_kernel(const float* __restrict__ part, const float* __restrict__ bias_part, int splits, int N, int K, int n_tiles,
                                                           int k_tiles, typename NmType<DT>::elem* __restrict__ dw, void* __restrict__ db, int db_f32) {
    typedef typename NmType<DT>::elem T;
    constexpr int CG = NmGroup<DT>::C;
    __shared__ float4 sh[7][64];
    __shared__ float sh_b[7][64];
    const int g = threadIdx.x >> 6;
    const long long t = (long long)blockIdx.x * 64 + (threadIdx.x & 63), tiles = (long long)n_tiles * k_tiles;
    const bool in = t < tiles * 4096;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (dw && in) {
        const float* src = part + t * 4;
#pragma unroll 8
        for (int c = g; c < splits; c += 8) {
            const float4 v = *reinterpret_cast<const float4*>(src + (long long)c * tiles * 16384);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
    }
    float b = 0.f;
    if (db && t < N) {
        const int gn = (int)t / CG * CG, e = (int)t - nm_d_group<DT>(gn, N);
#pragma unroll 8
        for (int c = g; c < splits; c += 8) b += bias_part[(long long)c * n_tiles * 128 + gn + e];
    }
    if (g > 0) {
        sh[g - 1][threadIdx.x & 63] = s;
        sh_b[g - 1][threadIdx.x & 63] = b;
    }
    __syncthreads();
    if (g > 0) return;
#pragma unroll
    for (int o = 0; o < 7; ++o) {
        const float4 v = sh[o][threadIdx.x];
        s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        b += sh_b[o][threadIdx.x];
    }
    if (db && t < N) {
        if (db_f32) ((float*)db)[t] = b;
        else ((T*)db)[t] = (T)b;
    }
    if (!dw || !in) return;
    const int tile = (int)(t >> 12), e4 = (int)(t & 4095), wave = e4 >> 10, sub = (e4 >> 6) & 15;
    nm_d_put_grad<DT>(dw, N, K, tile / k_tiles, tile % k_tiles, 2 * (wave & 1) + (sub >> 3), 2 * (wave >> 1) + ((sub >> 2) & 1), e4 & 63, sub & 3, s);
}

// ------------------------------------------------------------------------------------------------ launch plans
static inline long long nm_d_up(long long a, long long b) { return (a + b - 1) / b; }
static inline long long nm_d_align(long long b) { return nm_d_up(b, 256) * 256; }

struct NmDensePlan { bool resident, tile; int np, tiles, col_blocks, rt; long long steps, bytes; };

// columns C, contraction Q, rows R: which kernel, and its column blocks of 32 np columns
static NmDensePlan nm_d_plan(int dt, bool prod, bool res, bool trans, long long R, long long C, long long Q) {
    NmDensePlan p;
    const int pieces = nm_d_pieces(dt, prod);
    const long long steps = nm_d_up(Q, 32);
    p.np = C > 128 ? 8 : C > 64 ? 4 : C > 32 ? 2 : 1;
    int fit = pieces == 3 && p.np == 8 ? 4 : p.np;           // (three pieces of sixteen tiles leave no registers)
    if (res && fit == 8) fit = 4;                            // (the residual of eight pieces is in flight at once)
    while (fit > 0 && 2 * steps * pieces * fit > NM_D_RESIDENT) fit >>= 1;
    p.resident = fit > 0 && nm_d_up(C, 32 * fit) <= 4;
    // 256 x 256 tiles: one per CU and round, so what counts is the share of the rounds' 2^24 outputs that is there.  Measured in bf16 with GELU, us
    // (tiles / otherwise).  Against streaming: share 1: 50 / 85 (16384 x 1024 -> 1024), 0.63: 86 / 131 (16384 x 1024 -> 1280), 0.38: 43 / 56, 0.25: 42 / 43
    // (6144 and 4096 x 1024 -> 1024).  Against resident weights: share 1: 51 / 81 (65536 x 1024 -> 256), 25 / 31 (65536 x 256 -> 256), 44 / 47 (65536 x
    // 256 -> 512), 0.59: 51 / 50 (65536 x 300 -> 300), 0.5: 43 / 45 (32768 x 1024 -> 256).
    const double rounds = (double)nm_d_up(nm_d_up(R, 256) * nm_d_up(C, 256), 256), share = (double)R * (double)C / (rounds * 16777216.0);
    p.tile = dt != NM_F32 && !prod && !trans && Q > 0 && R > 0 && share >= (p.resident ? 0.75 : 0.3);
    if (p.tile) p.resident = false;
    p.np = p.resident ? fit : p.np > 4 ? 4 : p.np;
    // few rows: narrower column blocks until every wave has a tile (streaming: every CU a workgroup)
    while (p.np > 1 && (p.resident ? nm_d_up(R, 32) * nm_d_up(C, 32 * p.np) < 1024 : nm_d_up(R, 128) * nm_d_up(C, 32 * p.np) < 256)) p.np >>= 1;
    // streaming many rows: 64 rows per wave, so that a read of the weights serves twice the products
    p.rt = !p.resident && p.np == 4 && dt != NM_F32 && !prod && nm_d_up(R, 256) * nm_d_up(C, 128) >= 256 ? 4 : 2;
    const int ps = dt != NM_F32 || p.np == 1 ? 2 : 1;
    p.tiles = (int)(nm_d_up(C, 32 * p.np) * p.np * 2);
    p.col_blocks = p.tiles / (2 * p.np);
    p.steps = p.resident ? steps : nm_d_up(steps, ps) * ps;
    if (p.tile) p.col_blocks = (int)nm_d_up(C, 256);
    p.bytes = p.resident || p.tile ? 0 : nm_d_align(p.steps * p.tiles * pieces * 1024);
    return p;
}

struct NmDenseGradPlan { int n_tiles, k_tiles, splits; long long rows, bytes_part, bytes; };
static NmDenseGradPlan nm_d_grad_plan(long long M, long long N, long long K) {
    NmDenseGradPlan p;
    p.n_tiles = (int)nm_d_up(N > 0 ? N : 1, 128);
    p.k_tiles = (int)nm_d_up(K > 0 ? K : 1, 128);
    const long long tiles = (long long)p.n_tiles * p.k_tiles;
    long long splits = nm_d_up(512, tiles);                  // two workgroups per CU
    const long long most = nm_d_up(M, 256);
    if (splits > most) splits = most < 1 ? 1 : most;
    p.rows = nm_d_up(nm_d_up(M, splits), 64) * 64;
    p.splits = (int)(M > 0 ? nm_d_up(M, p.rows) : 1);
    p.bytes_part = p.splits > 1 ? nm_d_align((long long)p.splits * tiles * 16384 * 4) : 0;
    p.bytes = p.splits > 1 ? p.bytes_part + nm_d_align((long long)p.splits * p.n_tiles * 128 * 4) : 0;
    return p;
}

template <int DT, bool PROD>
static int nm_d_launch(const NmDensePlan& pl, NmDenseArgs a, hipStream_t stream) {
    a.tiles = pl.tiles;
    a.col_blocks = (unsigned)pl.col_blocks;
    constexpr bool F = DT == NM_F32;
    if (pl.resident) {
        // eight waves per workgroup, one tile of 32 rows each at least; one workgroup per CU
        long long slots = nm_d_up(nm_d_up(nm_d_up(a.R, 32), 8), 8) * 8;
        const long long most = 256 / pl.col_blocks / 8 * 8;
        if (slots > most) slots = most;
        const dim3 grid((unsigned)(slots * pl.col_blocks)), block(512);
        switch (pl.np) {
            case 8:
                if constexpr (!F) hipLaunchKernelGGL((nm_dense_resident_kernel<DT, PROD, 8>), grid, block, 0, stream, a);
                break;
            case 4: hipLaunchKernelGGL((nm_dense_resident_kernel<DT, PROD, 4>), grid, block, 0, stream, a); break;
            case 2: hipLaunchKernelGGL((nm_dense_resident_kernel<DT, PROD, 2>), grid, block, 0, stream, a); break;
            default: hipLaunchKernelGGL((nm_dense_resident_kernel<DT, PROD, 1>), grid, block, 0, stream, a); break;
        }
        NM_LAUNCH_CHECK();
        return 0;
    }
    const long long groups = nm_d_up(nm_d_up(a.R, pl.tile ? 256 : 64 * pl.rt), 8) * 8 * pl.col_blocks;
    if (groups * (pl.tile ? 512 : 256) > NM_D_MAX_THREADS) return nm_fail("nm_dense: %lld rows x %d columns exceed one launch", a.R, a.C);
    const dim3 grid((unsigned)groups), block(256);
    if (pl.tile) {
        if constexpr (!F && !PROD) {
            if (a.DV) hipLaunchKernelGGL((nm_dense_tile_kernel<DT, true>), grid, dim3(512), 0, stream, a);
            else hipLaunchKernelGGL((nm_dense_tile_kernel<DT, false>), grid, dim3(512), 0, stream, a);
        }
    } else if (pl.rt == 4) {
        if constexpr (!F && !PROD) hipLaunchKernelGGL((nm_dense_stream_kernel<DT, PROD, 4, 4, 2>), grid, block, 0, stream, a);
    } else {
        switch (pl.np) {
            case 4: hipLaunchKernelGGL((nm_dense_stream_kernel<DT, PROD, 2, 4, F ? 1 : 2>), grid, block, 0, stream, a); break;
            case 2: hipLaunchKernelGGL((nm_dense_stream_kernel<DT, PROD, 2, 2, F ? 1 : 2>), grid, block, 0, stream, a); break;
            default: hipLaunchKernelGGL((nm_dense_stream_kernel<DT, PROD, 2, 1, 2>), grid, block, 0, stream, a); break;
        }
    }
    NM_LAUNCH_CHECK();
    return 0;
}

template <int DT, bool PROD>
static int nm_d_pack(const NmDensePlan& pl, const NmDenseArgs& a, char* ws, hipStream_t stream) {
    if (pl.resident || pl.tile || pl.steps == 0) return 0;
    hipLaunchKernelGGL((nm_dense_pack_kernel<DT, NmPieces<DT, PROD>::PLAIN>), dim3((unsigned)nm_d_up(pl.steps * pl.tiles * 64, 256)), dim3(256), 0, stream, (const typename NmType<DT>::elem*)a.W,
                       a.ldw, a.trans, a.C, a.Q, pl.tiles, (int)pl.steps, (uint4*)ws);
    NM_LAUNCH_CHECK();
    return 0;
}

#define NM_D_FEW 8     // rows served by nm_dense_few_kernel

template <int DT>
static int nm_d_forward(const void* x, long long ldx, const void* w, long long ldw, const void* bias, int bias_dt, const void* res, long long ldr, long long M, int K,
                        int N, int act, float beta, void* y, long long ldy, void* deriv, char* ws, hipStream_t stream) {
    typedef typename NmType<DT>::elem T;
    if (M <= NM_D_FEW) {
        const dim3 grid((unsigned)nm_d_up(N, 16)), block(256);
#define NM_D_FEW_LAUNCH(MR)                                                                                                                                    \
    hipLaunchKernelGGL((nm_dense_few_kernel<DT, MR>), grid, block, 0, stream, (const T*)x, ldx, (const T*)w, ldw, bias, bias_dt == NM_F32, (const T*)res, ldr, \
                       (int)M, K, N, act, beta, (T*)y, ldy, deriv)
        if (M == 1) NM_D_FEW_LAUNCH(1);
        else if (M <= 2) NM_D_FEW_LAUNCH(2);
        else if (M <= 4) NM_D_FEW_LAUNCH(4);
        else NM_D_FEW_LAUNCH(8);
        NM_LAUNCH_CHECK();
        return 0;
    }
    const NmDensePlan pl = nm_d_plan(DT, false, res != nullptr, false, M, N, K);
    NmDenseArgs a = {};
    a.A = x; a.lda = ldx; a.W = w; a.ldw = ldw; a.P = (const uint4*)ws; a.bias = bias; a.bias_f32 = bias_dt == NM_F32;
    a.res = res; a.ldr = ldr; a.Y = y; a.ldy = ldy; a.DV = deriv; a.R = M; a.Q = K; a.C = N; a.act = act; a.beta = beta;
    if (nm_d_pack<DT, false>(pl, a, ws, stream)) return 1;
    return nm_d_launch<DT, false>(pl, a, stream);
}

template <int DT>
static int nm_d_backward(const void* g, long long ldg, const void* deriv, const void* x, long long ldx, const void* w, long long ldw, long long M, int K, int N, void* dx,
                         long long lddx, void* dw, void* db, int bias_dt, char* ws, hipStream_t stream) {
    typedef typename NmType<DT>::elem T;
    if (dx) {
        const NmDensePlan pl = nm_d_plan(DT, deriv != nullptr, false, true, M, K, N);
        NmDenseArgs a = {};
        a.A = g; a.lda = ldg; a.D = deriv; a.W = w; a.ldw = ldw; a.trans = 1; a.P = (const uint4*)ws; a.Y = dx; a.ldy = lddx; a.R = M; a.Q = N; a.C = K; a.act = NM_ACT_NONE; a.beta = 1.f;
        if (deriv ? nm_d_pack<DT, true>(pl, a, ws, stream) : nm_d_pack<DT, false>(pl, a, ws, stream)) return 1;
        if (deriv ? nm_d_launch<DT, true>(pl, a, stream) : nm_d_launch<DT, false>(pl, a, stream)) return 1;
        ws += pl.bytes;
    }
    if (!dw && !db) return 0;
    const NmDenseGradPlan pl = nm_d_grad_plan(M, N, dw ? K : 1);      // (db alone: no columns of x)
    NmDenseGradArgs a = {};
    a.G = g; a.ldg = ldg; a.D = deriv; a.X = x; a.ldx = ldx; a.R = M; a.N = N; a.K = dw ? K : 0; a.n_tiles = pl.n_tiles; a.k_tiles = pl.k_tiles; a.rows = pl.rows;
    if (pl.splits > 1) {
        a.part = (float*)ws;
        a.bias_part = db ? (float*)(ws + pl.bytes_part) : nullptr;
    } else {
        a.dw = dw; a.db = db; a.db_f32 = bias_dt == NM_F32;
    }
    const long long tiles = (long long)pl.n_tiles * pl.k_tiles;
    const long long groups = tiles * nm_d_up(pl.splits, 8) * 8;
    a.splits = pl.splits;
    if (groups * 256 > NM_D_MAX_THREADS) return nm_fail("nm_dense_backward: %d x %d weights exceed one launch", N, K);
    const dim3 grid((unsigned)groups), block(256);
    if (deriv) hipLaunchKernelGGL((nm_dense_grad_kernel<DT, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((nm_dense_grad_kernel<DT, false>), grid, block, 0, stream, a);
    if (pl.splits == 1) {
        NM_LAUNCH_CHECK();
        return 0;
    }
    const long long pieces = tiles * 4096 > N ? tiles * 4096 : N;
    hipLaunchKernelGGL((nm_dense_sum_kernel<DT>), dim3((unsigned)nm_d_up(pieces, 64)), dim3(512), 0, stream, a.part, a.bias_part, pl.splits, N, a.K, pl.n_tiles,
                       pl.k_tiles, (T*)dw, db, bias_dt == NM_F32);
    NM_LAUNCH_CHECK();
    return 0;
}

// ------------------------------------------------------------------------------------------------ C ABI
static int nm_d_check(const char* who, int64_t M, int64_t K, int64_t N, int dtype, int bias_dtype) {
    if (!nm_dtype_ok(dtype)) return nm_fail("%s: unknown element type %d", who, dtype);
    if (bias_dtype != dtype && bias_dtype != NM_F32) return nm_fail("%s: the bias is fp32 or of the rows' type", who);
    if (M < 0 || K < 0 || N < 0 || K > NM_D_MAX_DIM || N > NM_D_MAX_DIM) return nm_fail("%s: bad sizes M=%lld K=%lld N=%lld", who, (long long)M, (long long)K, (long long)N);
    return 0;
}

extern "C" {

int64_t nm_dense_workspace_bytes(int64_t M, int64_t K, int64_t N, int dtype, int backward) {
    if (nm_d_check("nm_dense_workspace_bytes", M, K, N, dtype, dtype)) return -1;
    if (!backward) {
        if (M <= NM_D_FEW) return 0;
        const long long with = nm_d_plan(dtype, false, true, false, M, N, K).bytes, without = nm_d_plan(dtype, false, false, false, M, N, K).bytes;
        return with > without ? with : without;
    }
    // (the bias gradient alone is a plan of its own: one block of columns, more splits)
    const long long both = nm_d_grad_plan(M, N, K).bytes, bias = nm_d_grad_plan(M, N, 1).bytes;
    const long long plain = nm_d_plan(dtype, false, false, true, M, K, N).bytes, prod = nm_d_plan(dtype, true, false, true, M, K, N).bytes;      // (deriv given or not)
    return (plain > prod ? plain : prod) + (both > bias ? both : bias);
}

int nm_dense_forward(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, int bias_dtype, const void* residual, int64_t ldr, int64_t M,
                     int64_t K, int64_t N, int dtype, int act, float beta, void* y, int64_t ldy, void* deriv, void* workspace, int64_t workspace_bytes,
                     nm_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    if (nm_d_check("nm_dense_forward", M, K, N, dtype, bias_dtype)) return 1;
    if (act < NM_ACT_NONE || act > NM_ACT_GELU_TANH) return nm_fail("nm_dense_forward: unknown activation %d", act);
    if (act == NM_ACT_SOFTPLUS && !(beta >= 0x1p-126f && beta <= 0x1p126f)) return nm_fail("nm_dense_forward: softplus needs beta in [2^-126, 2^126]");
    if (M == 0 || N == 0) return 0;
    if ((K > 0 && (!x || !weight)) || !y) return nm_fail("nm_dense_forward: NULL argument");
    if (ldx > NM_D_MAX_LD || ldw > NM_D_MAX_LD || ldy > NM_D_MAX_LD || ldr > NM_D_MAX_LD) return nm_fail("nm_dense_forward: row stride beyond 2^24");
    if (ldx < K || ldw < K || ldy < N || (residual && ldr < N)) return nm_fail("nm_dense_forward: row stride shorter than a row");
    if (workspace_bytes < nm_dense_workspace_bytes(M, K, N, dtype, 0)) return nm_fail("nm_dense_forward: workspace too small");
    if (workspace_bytes > 0 && !workspace) return nm_fail("nm_dense_forward: NULL workspace");
    if (act == NM_ACT_NONE) deriv = nullptr;      // act' = 1: backward takes NULL
    if (act != NM_ACT_SOFTPLUS) beta = 1.f;
    const int k = (int)K, n = (int)N;
    if (dtype == NM_F32) return nm_d_forward<NM_F32>(x, ldx, weight, ldw, bias, bias_dtype, residual, ldr, M, k, n, act, beta, y, ldy, deriv, (char*)workspace, stream);
    if (dtype == NM_F16) return nm_d_forward<NM_F16>(x, ldx, weight, ldw, bias, bias_dtype, residual, ldr, M, k, n, act, beta, y, ldy, deriv, (char*)workspace, stream);
    return nm_d_forward<NM_BF16>(x, ldx, weight, ldw, bias, bias_dtype, residual, ldr, M, k, n, act, beta, y, ldy, deriv, (char*)workspace, stream);
}

int nm_dense_backward(const void* g, int64_t ldg, const void* deriv, const void* x, int64_t ldx, const void* weight, int64_t ldw, int64_t M, int64_t K, int64_t N,
                      int dtype, void* dx, int64_t lddx, void* dweight, void* dbias, int bias_dtype, void* workspace, int64_t workspace_bytes, nm_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    if (nm_d_check("nm_dense_backward", M, K, N, dtype, bias_dtype)) return 1;
    if (K == 0) { dx = nullptr; dweight = nullptr; }
    if (N == 0) { dweight = nullptr; dbias = nullptr; }
    if (M == 0) dx = nullptr;
    if (!dx && !dweight && !dbias) return 0;
    if ((M > 0 && N > 0 && !g) || (dx && N > 0 && !weight) || (dweight && M > 0 && !x)) return nm_fail("nm_dense_backward: NULL argument");
    if (ldg > NM_D_MAX_LD || ldx > NM_D_MAX_LD || ldw > NM_D_MAX_LD || lddx > NM_D_MAX_LD) return nm_fail("nm_dense_backward: row stride beyond 2^24");
    if (ldg < N || (dx && (ldw < K || lddx < K)) || (dweight && ldx < K)) return nm_fail("nm_dense_backward: row stride shorter than a row");
    if (workspace_bytes < nm_dense_workspace_bytes(M, K, N, dtype, 1) || (workspace_bytes > 0 && !workspace)) return nm_fail("nm_dense_backward: workspace too small");
    const int k = (int)K, n = (int)N;
    char* ws = (char*)workspace;
    if (dtype == NM_F32) return nm_d_backward<NM_F32>(g, ldg, deriv, x, ldx, weight, ldw, M, k, n, dx, lddx, dweight, dbias, bias_dtype, ws, stream);
    if (dtype == NM_F16) return nm_d_backward<NM_F16>(g, ldg, deriv, x, ldx, weight, ldw, M, k, n, dx, lddx, dweight, dbias, bias_dtype, ws, stream);
    return nm_d_backward<NM_BF16>(g, ldg, deriv, x, ldx, weight, ldw, M, k, n, dx, lddx, dweight, dbias, bias_dtype, ws, stream);
}

}  // extern "C"
