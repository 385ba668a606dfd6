// nm_dense.hip -- dense layers: y = act(x W^T + b) + r and its gradient (C ABI: nm_dense_*), on the matrix pipe.
//
//   z = x W^T + b,   y = act(z) + r          x [M,K], W [N,K], b [N], r and y [M,N]
//   dz = g * act'(z);  dx = dz W;  dW = dz^T x;  db = sum over the rows of dz;  dr = g
//
// Three products, two kernels:
//   nm_dense_kernel      forward and dx: rows x a weight matrix, contraction along the rows' contiguous axis
//   nm_dense_grad_kernel dW and db: contraction over the rows, split over workgroups; nm_dense_sum_kernel adds the partial sums in a
//                        fixed order (the same bits from run to run)
// nm_dense_few_kernel serves 1 .. 8 rows (a probe, a picked point) without the layout step of the weights.
//
// Arithmetic.  16-bit inputs: one product per pair on the f16 / bf16 pipe, fp32 accumulation, fp32 epilogue, one rounding at the end.  The
// forward pass keeps act'(z) for the backward pass as fp16 (of either 16-bit type: its values lie in [-0.2, 1.2], where fp16 has 11 bits
// and bf16 8); dz = g act'(z) enters the products as TWO 16-bit pieces (value + residual): a single rounded piece put an error as
// large as the output's own rounding on dx and dW.  fp32 inputs: every operand cut into three bf16 pieces (nm_gemm.h: exact), six
// piece products, fp32 accumulation; act'(z) is kept in fp32.  An fp32 product with a non-finite operand is NaN where IEEE
// arithmetic may give an infinity.
#include "nm_error.h"
#include "nm_num.h"

#define NM_D_MAX_DIM (1 << 20)   // columns and contraction lengths fit 32-bit arithmetic with room

// ------------------------------------------------------------------------------------------------ activations
// F32: the accurate exponential and division (fp32 outputs); otherwise the hardware approximations (16-bit outputs: errors of 1e-6 are far below
// their rounding)
template <bool F32>
__device__ __forceinline__ float nm_d_exp(float x) {
    return F32 ? expf(x) : __builtin_amdgcn_exp2f(x * 1.44269504088896341f);
}
template <bool F32>
__device__ __forceinline__ float nm_d_rcp(float x) {
    return F32 ? 1.0f / x : __builtin_amdgcn_rcpf(x);
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
__device__ __forceinline__ void nm_d_act(int act, float beta, float ibeta, float (&z)[N], float (&d)[N]) {
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
            const float u = beta * z[i], e = nm_d_exp<F32>(-fabsf(u)), r = nm_d_rcp<F32>(1.0f + e);
            z[i] = fmaf(nm_d_log1p<F32>(e), ibeta, fmaxf(z[i], 0.f));
            d[i] = u >= 0.f ? r : e * r;
        }
    } else {
        const float c1 = act == NM_ACT_GELU_TANH ? 1.59576912160573071f : 1.0f;      // 2 sqrt(2 / pi)
        const float c3 = act == NM_ACT_GELU_TANH ? 0.044715f : 0.0f;
        const bool gate_only = act == NM_ACT_SIGMOID;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float t = fminf(fmaxf(z[i], -1e4f), 1e4f), t2 = t * t;             // (beyond, q or q1 is 0: no infinity times zero)
            const float u = c1 * t * fmaf(c3, t2, 1.0f);
            const float e = nm_d_exp<F32>(-fabsf(u)), r = nm_d_rcp<F32>(1.0f + e), er = e * r;
            const float q = z[i] != z[i] ? z[i] : u >= 0.f ? r : er, q1 = u >= 0.f ? er : r;
            d[i] = gate_only ? q * q1 : fmaf(t * q, q1 * (c1 * fmaf(3.0f * c3, t2, 1.0f)), q);
            z[i] = gate_only ? q : z[i] * q;
        }
    }
}

// ------------------------------------------------------------------------------------------------ operand pieces
// fp32 -> three bf16 pieces by truncation, a = p0 + p1 + p2 exactly
__device__ __forceinline__ void nm_d_cut(float a, unsigned& b0, unsigned& b1, unsigned& b2) {
    b0 = __float_as_uint(a) & 0xffff0000u;
    const float r = a - __uint_as_float(b0);
    b1 = __float_as_uint(r) & 0xffff0000u;
    b2 = __float_as_uint(r - __uint_as_float(b1));
}
__device__ __forceinline__ unsigned nm_d_pair(unsigned lo, unsigned hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }   // upper halves

// eight values -> fragments (16 bytes: eight 16-bit pieces per plane)
__device__ __forceinline__ void nm_d_cut8(const float (&f)[8], uint4 (&p)[3]) {
    unsigned b[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) nm_d_cut(f[e], b[0][e], b[1][e], b[2][e]);
#pragma unroll
    for (int q = 0; q < 3; ++q)
        p[q] = make_uint4(nm_d_pair(b[q][0], b[q][1]), nm_d_pair(b[q][2], b[q][3]), nm_d_pair(b[q][4], b[q][5]), nm_d_pair(b[q][6], b[q][7]));
}
// value + residual in the 16-bit type (no residual of an infinity)
template <int DT>
__device__ __forceinline__ void nm_d_two8(const float (&f)[8], uint4 (&p)[2]) {
    typedef typename NmType<DT>::elem T;
    T hi[8], lo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        hi[e] = (T)f[e];
        const float b = (float)hi[e];
        lo[e] = (T)(fabsf(b) < __builtin_inff() ? f[e] - b : 0.f);
    }
    __builtin_memcpy(&p[0], hi, 16);
    __builtin_memcpy(&p[1], lo, 16);
}

template <int DT>
__device__ __forceinline__ nm_v16f nm_d_mfma(const uint4& a, const uint4& b, nm_v16f c) {
    if constexpr (DT == NM_F16) {
        nm_v8h x, y;
        __builtin_memcpy(&x, &a, 16);
        __builtin_memcpy(&y, &b, 16);
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
    } else {
        nm_v8b x, y;
        __builtin_memcpy(&x, &a, 16);
        __builtin_memcpy(&y, &b, 16);
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
    }
}

// all piece products of one pair of fragments, small terms first.  Planes: PA of a, PB of b.
template <int DT, int PA, int PB>
__device__ __forceinline__ nm_v16f nm_d_products(const uint4 (&a)[PA], const uint4 (&b)[PB], nm_v16f c) {
    if constexpr (PA == 3 && PB == 3) {      // dropped: a1 b2 + a2 b1 + a2 b2 < 2^-21 |a||b|
        c = nm_d_mfma<DT>(a[1], b[1], c);
        c = nm_d_mfma<DT>(a[0], b[2], c);
        c = nm_d_mfma<DT>(a[2], b[0], c);
        c = nm_d_mfma<DT>(a[0], b[1], c);
        c = nm_d_mfma<DT>(a[1], b[0], c);
        return nm_d_mfma<DT>(a[0], b[0], c);
    } else {
        static_assert(PA == 1 || PB == 1, "16-bit products: at most one operand in two pieces");
#pragma unroll
        for (int i = PA - 1; i >= 0; --i)
#pragma unroll
            for (int j = PB - 1; j >= 0; --j) c = nm_d_mfma<DT>(a[i], b[j], c);
        return c;
    }
}

// ------------------------------------------------------------------------------------------------ weights in fragment order
// Column operand of nm_dense_kernel: element (c, q), output column c, contraction q.  Fragment (step q / 16, column tile c / 32): lane (i, h) holds
// q = 16 step + 8 h .. + 7 of column 32 tile + nm_d_col(i).  An output tile of the matrix pipe gives a lane the rows (r & 3) + 8 (r >> 2) + 4 h of
// the first operand: with this order of the columns they are 16 consecutive ones, which the epilogue stores as whole 16-byte pieces.
__host__ __device__ __forceinline__ int nm_d_col(int i) { return 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3); }

// Eight consecutive contraction elements always come as ONE whole load: the piece that would end beyond Q starts at Q - 8 instead, and what it
// repeats is zero on the packed side (and cleared on the rows' side, where it may be an infinity).  Q < 8: element by element from 0.
__host__ __device__ __forceinline__ long long nm_d_window(long long q0, long long Q) { return Q < 8 || q0 + 8 <= Q ? q0 : Q - 8; }

// pieces per weight element
template <int DT> struct NmPlanes { static constexpr int W = DT == NM_F32 ? 3 : 1; };

// dst [steps][tiles][plane][lane] (zero beyond C and Q); bias -> fp32 [32 tiles]
template <int DT>
__global__ __launch_bounds__(256) void nm_dense_pack_kernel(const typename NmType<DT>::elem* __restrict__ w, long long ldw, int trans, int C, int Q, int tiles,
                                                            int steps, uint4* __restrict__ dst, const void* __restrict__ bias, int bias_f32,
                                                            float* __restrict__ bias_out) {
    typedef typename NmType<DT>::elem T;
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    if (bias && t < 32LL * tiles) bias_out[t] = t >= C ? 0.f : bias_f32 ? ((const float*)bias)[t] : (float)((const T*)bias)[t];
    const int lane = (int)(t & 63), i = lane & 31, h = lane >> 5;
    const long long frag = t >> 6;
    const int tile = (int)(frag % tiles);
    const long long step = frag / tiles;
    if (step >= steps) return;
    const int c = 32 * tile + nm_d_col(i);
    const long long q0 = 16 * step + 8 * h, s0 = nm_d_window(q0, Q);
    T e[8];
    if (!trans) {
        NmOct<DT> o = nm_oct_zero<DT>();
        if (c < C) {
            const T* row = w + (long long)c * ldw;
            if (Q < 8) { if (q0 == 0) o = nm_oct_load_short<DT>(row, Q); }
            else o = nm_oct_clear_first<DT>(nm_oct_load<DT>(row + s0), (int)(q0 - s0 < 8 ? q0 - s0 : 8));
        }
        __builtin_memcpy(e, &o, sizeof(o));
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) e[k] = c < C && s0 + k < Q && s0 + k >= q0 ? w[(s0 + k) * ldw + c] : (T)0.f;
    }
    uint4* d = dst + ((step * tiles + tile) * NmPlanes<DT>::W) * 64 + lane;
    if constexpr (DT == NM_F32) {
        float f[8];
        uint4 p[3];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = e[k];
        nm_d_cut8(f, p);
#pragma unroll
        for (int q = 0; q < 3; ++q) d[q * 64] = p[q];
    } else {
        uint4 p;
        __builtin_memcpy(&p, e, 16);
        *d = p;
    }
}

// ------------------------------------------------------------------------------------------------ rows x weights
struct NmDenseArgs {
    const void* A; long long lda;        // rows [R, Q]
    const void* D;                       // PROD: factor of every element of A, contiguous [R, Q] (fp16 beside 16-bit rows, else fp32)
    const uint4* W; int tiles;           // packed column operand
    const float* bias;                   // [32 tiles] or NULL
    const void* res; long long ldr;      // added after the activation, [R, C] or NULL
    void* Y; long long ldy;              // [R, C]
    void* DV;                            // act'(z), contiguous [R, C] (fp16 / fp32) or NULL
    long long R;
    int Q, C, act;
    float beta;
    unsigned col_blocks;
};

// One workgroup: 4 waves, 128 RT rows x 32 NT columns.  A wave owns 32 RT whole rows: their elements go from global memory straight into fragments
// (a lane's 8 consecutive elements of one row ARE a fragment), so the rows need no shared memory and are read once per column block; the column
// operand is shared by the four waves through LDS, PS steps of 16 at a time in two buffers, one barrier per panel, both sides' next
// panel in flight in registers meanwhile.
template <int DT, bool PROD, int RT, int NT, int PS>
__global__ __launch_bounds__(256, 2) void nm_dense_kernel(NmDenseArgs p) {
    typedef typename NmType<DT>::elem T;
    constexpr int PW = NmPlanes<DT>::W, PX = DT == NM_F32 ? 3 : PROD ? 2 : 1;
    constexpr int DD = DT == NM_F32 ? NM_F32 : NM_F16;       // type of the factor
    constexpr int PANEL = PS * NT * PW * 64;                 // uint4
    constexpr int WV = PANEL / 256;
    static_assert(PANEL % 256 == 0, "a panel is whole 16-byte pieces per thread");
    __shared__ uint4 lds[2][PANEL];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, li = lane & 31, h = lane >> 5;
    // consecutive workgroup numbers go to the eight XCDs in turn: the column blocks of one row block follow each other on ONE of them
    const unsigned id = blockIdx.x, xcd = id & 7, slot = id >> 3;
    const long long rb = (long long)(slot / p.col_blocks) * 8 + xcd;
    const int cb = (int)(slot % p.col_blocks);
    const long long m0 = rb * (128 * RT) + wave * (32 * RT);
    if (rb * (128 * RT) >= p.R) return;
    const int steps = (p.Q + 15) / 16, panels = (steps + PS - 1) / PS;
    const T* arow[RT];
    const typename NmType<DD>::elem* drow[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        long long m = m0 + 32 * r + li;
        m = m < p.R ? m : p.R - 1;
        arow[r] = (const T*)p.A + m * p.lda;
        drow[r] = PROD ? (const typename NmType<DD>::elem*)p.D + m * p.Q : nullptr;
    }
    nm_v16f acc[RT][NT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[r][n][i] = 0.f;

    uint4 wv[WV];
    NmOct<DT> xa[2][RT][PS];
    NmOct<DD> xd[2][RT][PS];
    auto load_w = [&](int panel) {
#pragma unroll
        for (int i = 0; i < WV; ++i) {
            const int e = i * 256 + t, s = e / (NT * PW * 64), o = e % (NT * PW * 64);
            wv[i] = p.W[((long long)(panel * PS + s) * p.tiles + cb * NT) * (PW * 64) + o];
        }
    };
    auto store_w = [&](int buf) {
#pragma unroll
        for (int i = 0; i < WV; ++i) lds[buf][i * 256 + t] = wv[i];
    };
    auto load_x = [&](int panel, NmOct<DT> (&a)[RT][PS], NmOct<DD> (&d)[RT][PS]) {
        if (p.Q >= 8) {
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int s = 0; s < PS; ++s) {
                    const int q = panel * (16 * PS) + 16 * s + 8 * h, w = q + 8 <= p.Q ? q : p.Q - 8;
                    a[r][s] = nm_oct_load<DT>(arow[r] + w);
                    if constexpr (PROD) d[r][s] = nm_oct_load<DD>(drow[r] + w);
                }
        } else {                                             // (one step; lanes of the upper half have nothing)
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int s = 0; s < PS; ++s) {
                    a[r][s] = nm_oct_zero<DT>();
                    if constexpr (PROD) d[r][s] = nm_oct_zero<DD>();
                    if (s == 0 && h == 0) {
                        a[r][s] = nm_oct_load_short<DT>(arow[r], p.Q);
                        if constexpr (PROD) d[r][s] = nm_oct_load_short<DD>(drow[r], p.Q);
                    }
                }
        }
    };
    // the last panel: clear what a whole load repeated or brought beyond the row
    auto trim = [&](int panel, NmOct<DT> (&a)[RT][PS], NmOct<DD> (&d)[RT][PS]) {
        if ((panel + 1) * (16 * PS) <= p.Q || p.Q < 8) return;
#pragma unroll
        for (int s = 0; s < PS; ++s) {
            const int q = panel * (16 * PS) + 16 * s + 8 * h, sh = q + 8 <= p.Q ? 0 : q + 8 - p.Q;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                a[r][s] = nm_oct_clear_first<DT>(a[r][s], sh);
                if constexpr (PROD) d[r][s] = nm_oct_clear_first<DD>(d[r][s], sh);
            }
        }
    };
    auto compute = [&](int buf, const NmOct<DT> (&a)[RT][PS], const NmOct<DD> (&d)[RT][PS]) {
#pragma unroll
        for (int s = 0; s < PS; ++s) {
            uint4 x[RT][PX];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                if constexpr (DT != NM_F32 && !PROD) {
                    x[r][0] = a[r][s].v[0];
                } else {
                    float f[8];
                    nm_oct_to_float<DT>(a[r][s], f);
                    if constexpr (PROD) {
                        float g[8];
                        nm_oct_to_float<DD>(d[r][s], g);
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] *= g[e];
                    }
                    if constexpr (DT == NM_F32) nm_d_cut8(f, x[r]);
                    else nm_d_two8<DT>(f, x[r]);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint4 w[PW];
#pragma unroll
                for (int q = 0; q < PW; ++q) w[q] = lds[buf][((s * NT + n) * PW + q) * 64 + lane];
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[r][n] = nm_d_products<DT>(w, x[r], acc[r][n]);
            }
        }
    };

    if (panels > 0) {
        load_w(0);
        load_x(0, xa[0], xd[0]);
        store_w(0);
    }
    __syncthreads();
    for (int k = 0; k < panels; k += 2) {
        // (a wave that is a panel ahead fills the OTHER buffer; nobody is two panels ahead: one barrier per panel)
        if (k + 1 < panels) {
            load_w(k + 1);
            load_x(k + 1, xa[1], xd[1]);
        }
        trim(k, xa[0], xd[0]);
        compute(0, xa[0], xd[0]);
        if (k + 1 >= panels) break;
        store_w(1);
        __syncthreads();
        if (k + 2 < panels) {
            load_w(k + 2);
            load_x(k + 2, xa[0], xd[0]);
        }
        trim(k + 1, xa[1], xd[1]);
        compute(1, xa[1], xd[1]);
        if (k + 2 < panels) store_w(0);
        __syncthreads();
    }

    const float ibeta = 1.0f / p.beta;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const long long m = m0 + 32 * r + li;
        if (m >= p.R) continue;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int c0 = (cb * NT + n) * 32 + 16 * h;
            if (c0 >= p.C) continue;
            float z[16], dv[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) z[i] = acc[r][n][i];
            if (!PROD && p.bias) {
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] += p.bias[c0 + i];
            }
            if constexpr (!PROD) nm_d_act<DT == NM_F32>(p.act, p.beta, ibeta, z, dv);
#pragma unroll
            for (int o = 0; o < 16; o += 8) {
                const long long left = p.C - c0 - o;
                if (left <= 0) break;
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = z[o + i];
                if (!PROD && p.res) {
                    float q[8];
                    nm_oct_to_float<DT>(nm_oct_load_row<DT>((const T*)p.res + m * p.ldr, c0 + o, p.C), q);
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] += q[i];
                }
                nm_oct_store_n<DT>((T*)p.Y + m * p.ldy + c0 + o, f, left);
                if (!PROD && p.DV) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) f[i] = dv[o + i];
                    nm_oct_store_n<DD>((typename NmType<DD>::elem*)p.DV + m * p.C + c0 + o, f, left);
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ a few rows
// 1 .. MR rows: bound by the read of the weights and by latency.  16 lanes share a column (8 elements each per round), so W is read once, in its own
// layout, with whole 16-byte pieces, and the partial sums meet in four lane exchanges; plain fp32 multiply-adds.
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
    nm_d_act<DT == NM_F32>(act, beta, 1.0f / beta, hv, d);
    float h = hv[0];
    if (res) h += (float)res[sub * ldr + n];
    y[sub * ldy + n] = (T)h;
    if (dv) {
        if (DT == NM_F32) ((float*)dv)[(long long)sub * N + n] = d[0];
        else ((_Float16*)dv)[(long long)sub * N + n] = (_Float16)d[0];
    }
}

// ------------------------------------------------------------------------------------------------ weight and bias gradient
// dW = dz^T x, contraction over the rows.  One workgroup: a 128 x 128 tile of dW over a range of rows, 64 rows at a time; 4 waves of 64 x 64.
// The contraction is the SLOW axis of both operands.  A thread loads eight rows x eight columns (16-byte pieces, whole lines per row) and
// transposes them in its own registers (one byte permute per two elements, or on the way through the product's fp32): it then holds, for each of its columns, eight consecutive rows --
// a fragment -- and writes it to LDS in the order in which the waves read fragments.  Tile t, position i of the matrix pipe is column
// 8 (i % 16) + 2 t + i / 16 of the 128.  Two waves bring dz (from g and act'(z), in two pieces or three), two bring x.
__host__ __device__ __forceinline__ int nm_d_group(int c, int n) { return n < 8 || c + 8 <= n ? c : n - 8; }   // first column of the group at c

struct NmDenseGradArgs {
    const void* G; long long ldg; const void* D;   // dz = G * D (D contiguous [R, N] fp16 / fp32, or NULL)
    const void* X; long long ldx;
    long long R;
    int N, K, n_tiles, k_tiles;
    long long rows;                      // rows per workgroup (a multiple of 64)
    float* part;                         // [splits][n_tiles * k_tiles][16384] in the order of the accumulators
    float* bias_part;                    // [splits][128 n_tiles] or NULL
};

// 16-bit elements: column e of eight rows
template <int DT>
__device__ __forceinline__ uint4 nm_d_column16(const NmOct<DT> (&r)[8], int e) {
    const unsigned sel = (e & 1) ? 0x07060302u : 0x05040100u;
    unsigned w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = (e >> 1) == 0 ? r[j].v[0].x : (e >> 1) == 1 ? r[j].v[0].y : (e >> 1) == 2 ? r[j].v[0].z : r[j].v[0].w;
    return make_uint4(__builtin_amdgcn_perm(w[1], w[0], sel), __builtin_amdgcn_perm(w[3], w[2], sel), __builtin_amdgcn_perm(w[5], w[4], sel),
                      __builtin_amdgcn_perm(w[7], w[6], sel));
}
template <int DT>
__device__ __forceinline__ float nm_d_element(const NmOct<DT>& o, int e) {
    float f[8];
    nm_oct_to_float<DT>(o, f);
    return f[e];
}

template <int DT, bool PROD>
__global__ __launch_bounds__(256, 2) void nm_dense_grad_kernel(NmDenseGradArgs p) {
    typedef typename NmType<DT>::elem T;
    constexpr int DD = DT == NM_F32 ? NM_F32 : NM_F16;
    constexpr int PZ = DT == NM_F32 ? 3 : PROD ? 2 : 1, PX = DT == NM_F32 ? 3 : 1;
    constexpr int STEPS = DT == NM_F32 ? 2 : 4;              // steps of 16 rows in a block
    constexpr int ROWS = 16 * STEPS;
    constexpr int LZ = PZ * STEPS * 256, LX = PX * STEPS * 256;   // uint4: [plane][step][tile 4][lane 64]
    __shared__ uint4 lds[LZ + LX];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const unsigned tile = blockIdx.x % (p.n_tiles * p.k_tiles), split = blockIdx.x / (p.n_tiles * p.k_tiles);
    const int tn = (int)(tile / p.k_tiles), tk = (int)(tile % p.k_tiles);
    const long long r0 = (long long)split * p.rows, r1 = r0 + p.rows < p.R ? r0 + p.rows : p.R;
    const bool isz = wave < 2;                               // (wave-uniform)
    // a thread's share of a block: columns 8 cg .. + 7 of eight rows; four row groups per wave.  16-bit: two waves bring 64 rows.  fp32: a block
    // is 32 rows (three planes of 64 would leave one workgroup per CU): one wave of the two brings them.
    const int cg = lane & 15, rg = (lane >> 4) + 4 * (wave & 1);
    const bool active = rg * 8 < ROWS;
    // (a group of columns that would end beyond the row is the row's last eight: nm_dense_sum_kernel takes the columns that are its own)
    const int ncol = isz ? p.N : p.K, col = nm_d_group((isz ? tn : tk) * 128 + cg * 8, ncol);
    const bool want_bias = isz && p.bias_part && tk == 0;
    float bsum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) bsum[e] = 0.f;
    nm_v16f acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    NmOct<DT> va[8];
    NmOct<DD> vd[8];
    auto load = [&](long long base) {
        const T* src = isz ? (const T*)p.G : (const T*)p.X;
        const long long ld = isz ? p.ldg : p.ldx;
        const typename NmType<DD>::elem* fac = (const typename NmType<DD>::elem*)p.D;
        if (base + ROWS <= r1 && ncol >= 8) {                // (uniform over the wave)
            if (active) {
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const long long m = base + rg * 8 + r;
                    va[r] = nm_oct_load<DT>(src + m * ld + col);
                    if constexpr (PROD)
                        if (isz) vd[r] = nm_oct_load<DD>(fac + m * p.N + col);
                }
            }
            return;
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const long long m = base + rg * 8 + r;
            va[r] = nm_oct_zero<DT>();
            if constexpr (PROD) vd[r] = nm_oct_zero<DD>();
            if (m < r1 && active && ncol > 0) {
                if (ncol >= 8) {
                    va[r] = nm_oct_load<DT>(src + m * ld + col);
                    if constexpr (PROD)
                        if (isz) vd[r] = nm_oct_load<DD>(fac + m * p.N + col);
                } else if (col == 0) {
                    va[r] = nm_oct_load_short<DT>(src + m * ld, ncol);
                    if constexpr (PROD)
                        if (isz) vd[r] = nm_oct_load_short<DD>(fac + m * p.N, ncol);
                }
            }
        }
    };
    // a fragment of this thread -> LDS: column e of its eight is position 16 (e & 1) + cg of tile e >> 1
    auto put = [&](uint4* base, const uint4& c, int e) { base[(rg >> 1) * 256 + (e >> 1) * 64 + (rg & 1) * 32 + (e & 1) * 16 + cg] = c; };
    auto stash = [&]() {
        if (!active) return;
        uint4* base = isz ? lds : lds + LZ;
#pragma unroll
        for (int e = 0; e < 8; ++e) {                        // one column: eight rows -> a fragment per plane
            if (DT != NM_F32 && !(isz && (PROD || want_bias))) {
                if constexpr (DT != NM_F32) put(base, nm_d_column16<DT>(va, e), e);
                continue;
            }
            float f[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                f[r] = nm_d_element<DT>(va[r], e);
                if constexpr (PROD)
                    if (isz) f[r] *= nm_d_element<DD>(vd[r], e);
                if (want_bias) bsum[e] += f[r];
            }
            if constexpr (DT == NM_F32) {
                uint4 c[3];
                nm_d_cut8(f, c);
#pragma unroll
                for (int q = 0; q < 3; ++q) put(base + q * STEPS * 256, c[q], e);
            } else if constexpr (PROD) {
                uint4 c[2];
                nm_d_two8<DT>(f, c);
                put(base, c[0], e);
                put(base + STEPS * 256, c[1], e);
            } else {
                put(base, nm_d_column16<DT>(va, e), e);
            }
        }
    };

    const int wn = wave & 1, wk = wave >> 1;
    if (r0 < r1) load(r0);
    for (long long b = r0; b < r1; b += ROWS) {
        stash();
        __syncthreads();
        if (b + ROWS < r1) load(b + ROWS);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
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
                for (int j = 0; j < 2; ++j) acc[i][j] = nm_d_products<DT>(z[i], x[j], acc[i][j]);
        }
        __syncthreads();
    }
    float* out = p.part + ((long long)split * (p.n_tiles * p.k_tiles) + tile) * 16384 + wave * 4096;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<float4*>(out + ((i * 2 + j) * 4 + (r >> 2)) * 256 + lane * 4) =
                    make_float4(acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]);
    if (!p.bias_part || tk != 0) return;                      // (uniform over the workgroup)
    float* sh = reinterpret_cast<float*>(lds);
    if (isz) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            bsum[e] += __shfl_xor(bsum[e], 16);
            bsum[e] += __shfl_xor(bsum[e], 32);
            if (lane < 16) sh[wave * 128 + cg * 8 + e] = bsum[e];
        }
    }
    __syncthreads();
    if (t < 128) p.bias_part[((long long)split * p.n_tiles + tn) * 128 + t] = sh[t] + sh[128 + t];
}

// partial sums -> dW [N, K], db [N], over the splits in order
template <int DT>
__global__ __launch_bounds__(256) void nm_dense_sum_kernel(const float* __restrict__ part, const float* __restrict__ bias_part, int splits, int N, int K, int n_tiles,
                                                           int k_tiles, typename NmType<DT>::elem* __restrict__ dw, void* __restrict__ db, int db_f32) {
    typedef typename NmType<DT>::elem T;
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long tiles = (long long)n_tiles * k_tiles;
    if (t < tiles * 4096) {
        const int tile = (int)(t >> 12), e4 = (int)(t & 4095);
        const int wave = e4 >> 10, sub = (e4 >> 6) & 15, lane = e4 & 63, li = lane & 31, h = lane >> 5;
        const int i = sub >> 3, j = (sub >> 2) & 1, rq = sub & 3;
        // position of the matrix pipe -> group of eight columns and column of the group
        const int gk = (tile % k_tiles) * 128 + 8 * (li & 15), k = nm_d_group(gk, K) + 2 * (2 * (wave >> 1) + j) + (li >> 4);
        if (dw && k >= gk && k < K) {
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
            const float* src = part + t * 4;
            for (int c = 0; c < splits; ++c) {
                const float4 v = *reinterpret_cast<const float4*>(src + (long long)c * tiles * 16384);
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int pn = q + 8 * rq + 4 * h;
                const int gn = (tile / k_tiles) * 128 + 8 * (pn & 15), n = nm_d_group(gn, N) + 2 * (2 * (wave & 1) + i) + (pn >> 4);
                if (n >= gn && n < N) dw[(long long)n * K + k] = (T)(q == 0 ? s.x : q == 1 ? s.y : q == 2 ? s.z : s.w);
            }
        }
    }
    if (db && t < N) {
        const int gn = (int)t & ~7, e = (int)t - nm_d_group(gn, N);
        float s = 0.f;
        for (int c = 0; c < splits; ++c) s += bias_part[(long long)c * n_tiles * 128 + gn + e];
        if (db_f32) ((float*)db)[t] = s;
        else ((T*)db)[t] = (T)s;
    }
}

// ------------------------------------------------------------------------------------------------ launch plans
static inline long long nm_d_up(long long a, long long b) { return (a + b - 1) / b; }
static inline long long nm_d_align(long long b) { return nm_d_up(b, 256) * 256; }

struct NmDensePlan { int nt, ps, tiles, col_blocks; long long steps, bytes_w, bytes; };

// columns C, contraction Q, rows R.  Panels: PS steps x NT tiles.
static NmDensePlan nm_d_plan(int dt, long long R, long long C, long long Q) {
    NmDensePlan p;
    p.nt = C > 128 ? 8 : C > 64 ? 4 : C > 32 ? 2 : 1;
    const long long rb = nm_d_up(R, 128);
    while (p.nt > 1 && rb * nm_d_up(C, 32 * p.nt) < 256) p.nt >>= 1;     // few rows: narrower column blocks until the chip is filled
    p.ps = dt != NM_F32 ? (p.nt == 8 ? 2 : 4) : p.nt == 8 ? 1 : p.nt == 1 ? 4 : 2;
    p.tiles = (int)(nm_d_up(C, 32 * p.nt) * p.nt);
    p.col_blocks = p.tiles / p.nt;
    p.steps = nm_d_up(nm_d_up(Q, 16), p.ps) * p.ps;
    p.bytes_w = nm_d_align(p.steps * p.tiles * (dt == NM_F32 ? 3 : 1) * 1024);
    p.bytes = p.bytes_w + nm_d_align(32LL * p.tiles * 4);
    return p;
}

struct NmDenseGradPlan { int n_tiles, k_tiles, splits; long long rows, bytes_part, bytes; };
static NmDenseGradPlan nm_d_grad_plan(long long M, long long N, long long K) {
    NmDenseGradPlan p;
    p.n_tiles = (int)nm_d_up(N > 0 ? N : 1, 128);
    p.k_tiles = (int)nm_d_up(K > 0 ? K : 1, 128);
    const long long tiles = (long long)p.n_tiles * p.k_tiles;
    long long splits = nm_d_up(256, tiles);
    const long long most = nm_d_up(M, 256);
    if (splits > most) splits = most < 1 ? 1 : most;
    p.rows = nm_d_up(nm_d_up(M, splits), 64) * 64;
    p.splits = (int)(M > 0 ? nm_d_up(M, p.rows) : 1);
    p.bytes_part = nm_d_align((long long)p.splits * tiles * 16384 * 4);
    p.bytes = p.bytes_part + nm_d_align((long long)p.splits * p.n_tiles * 128 * 4);
    return p;
}

template <int DT, bool PROD>
static int nm_d_launch(const NmDensePlan& pl, NmDenseArgs a, hipStream_t stream) {
    a.tiles = pl.tiles;
    a.col_blocks = (unsigned)pl.col_blocks;
    const long long groups = nm_d_up(nm_d_up(a.R, 128), 8) * 8 * pl.col_blocks;
    if (groups > 0x7fffffffLL) return nm_fail("nm_dense: %lld rows x %d columns exceed one launch", a.R, a.C);
    const dim3 grid((unsigned)groups), block(256);
    constexpr bool F = DT == NM_F32;
    switch (pl.nt) {
        case 8: hipLaunchKernelGGL((nm_dense_kernel<DT, PROD, 1, 8, F ? 1 : 2>), grid, block, 0, stream, a); break;
        case 4: hipLaunchKernelGGL((nm_dense_kernel<DT, PROD, 1, 4, F ? 2 : 4>), grid, block, 0, stream, a); break;
        case 2: hipLaunchKernelGGL((nm_dense_kernel<DT, PROD, 1, 2, F ? 2 : 4>), grid, block, 0, stream, a); break;
        default: hipLaunchKernelGGL((nm_dense_kernel<DT, PROD, 1, 1, 4>), grid, block, 0, stream, a); break;
    }
    NM_LAUNCH_CHECK();
    return 0;
}

template <int DT>
static int nm_d_pack(const NmDensePlan& pl, const void* w, long long ldw, int trans, int C, int Q, const void* bias, int bias_dt, char* ws, hipStream_t stream) {
    const long long threads = pl.steps * pl.tiles * 64 > 32LL * pl.tiles ? pl.steps * pl.tiles * 64 : 32LL * pl.tiles;
    hipLaunchKernelGGL((nm_dense_pack_kernel<DT>), dim3((unsigned)nm_d_up(threads, 256)), dim3(256), 0, stream, (const typename NmType<DT>::elem*)w, ldw, trans, C, Q,
                       pl.tiles, (int)pl.steps, (uint4*)ws, bias, bias_dt == NM_F32, (float*)(ws + pl.bytes_w));
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
    const NmDensePlan pl = nm_d_plan(DT, M, N, K);
    if (nm_d_pack<DT>(pl, w, ldw, 0, N, K, bias, bias_dt, ws, stream)) return 1;
    NmDenseArgs a = {};
    a.A = x; a.lda = ldx; a.W = (const uint4*)ws; a.bias = bias ? (const float*)(ws + pl.bytes_w) : nullptr;
    a.res = res; a.ldr = ldr; a.Y = y; a.ldy = ldy; a.DV = deriv; a.R = M; a.Q = K; a.C = N; a.act = act; a.beta = beta;
    return nm_d_launch<DT, false>(pl, a, stream);
}

template <int DT>
static int nm_d_backward(const void* g, long long ldg, const void* deriv, const void* x, long long ldx, const void* w, long long ldw, long long M, int K, int N, void* dx,
                         long long lddx, void* dw, void* db, int bias_dt, char* ws, hipStream_t stream) {
    typedef typename NmType<DT>::elem T;
    if (dx) {
        const NmDensePlan pl = nm_d_plan(DT, M, K, N);
        if (nm_d_pack<DT>(pl, w, ldw, 1, K, N, nullptr, NM_F32, ws, stream)) return 1;
        NmDenseArgs a = {};
        a.A = g; a.lda = ldg; a.D = deriv; a.W = (const uint4*)ws; a.Y = dx; a.ldy = lddx; a.R = M; a.Q = N; a.C = K; a.act = NM_ACT_NONE; a.beta = 1.f;
        if (deriv ? nm_d_launch<DT, true>(pl, a, stream) : nm_d_launch<DT, false>(pl, a, stream)) return 1;
        ws += pl.bytes;
    }
    if (!dw && !db) return 0;
    const NmDenseGradPlan pl = nm_d_grad_plan(M, N, dw ? K : 1);      // (db alone: no columns of x)
    NmDenseGradArgs a = {};
    a.G = g; a.ldg = ldg; a.D = deriv; a.X = x; a.ldx = ldx; a.R = M; a.N = N; a.K = dw ? K : 0; a.n_tiles = pl.n_tiles; a.k_tiles = pl.k_tiles; a.rows = pl.rows;
    a.part = (float*)ws; a.bias_part = db ? (float*)(ws + pl.bytes_part) : nullptr;
    const long long tiles = (long long)pl.n_tiles * pl.k_tiles;
    if (tiles * pl.splits > 0x7fffffffLL) return nm_fail("nm_dense_backward: %d x %d weights exceed one launch", N, K);
    const dim3 grid((unsigned)(tiles * pl.splits)), block(256);
    if (deriv) hipLaunchKernelGGL((nm_dense_grad_kernel<DT, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((nm_dense_grad_kernel<DT, false>), grid, block, 0, stream, a);
    const long long threads = tiles * 4096 > N ? tiles * 4096 : N;
    hipLaunchKernelGGL((nm_dense_sum_kernel<DT>), dim3((unsigned)nm_d_up(threads, 256)), dim3(256), 0, stream, a.part, a.bias_part, pl.splits, N, a.K, pl.n_tiles,
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
    if (!backward) return M <= NM_D_FEW ? 0 : nm_d_plan(dtype, M, N, K).bytes;
    // (the bias gradient alone is a plan of its own: one block of columns, more splits)
    const long long both = nm_d_grad_plan(M, N, K).bytes, bias = nm_d_grad_plan(M, N, 1).bytes;
    return nm_d_plan(dtype, M, K, N).bytes + (both > bias ? both : bias);
}

int nm_dense_forward(const void* x, int64_t ldx, const void* weight, int64_t ldw, const void* bias, int bias_dtype, const void* residual, int64_t ldr, int64_t M,
                     int64_t K, int64_t N, int dtype, int act, float beta, void* y, int64_t ldy, void* deriv, void* workspace, int64_t workspace_bytes,
                     nm_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    if (nm_d_check("nm_dense_forward", M, K, N, dtype, bias_dtype)) return 1;
    if (act < NM_ACT_NONE || act > NM_ACT_GELU_TANH) return nm_fail("nm_dense_forward: unknown activation %d", act);
    if (act == NM_ACT_SOFTPLUS && !(beta > 0.f)) return nm_fail("nm_dense_forward: softplus needs beta > 0");
    if (M == 0 || N == 0) return 0;
    if ((K > 0 && (!x || !weight)) || !y) return nm_fail("nm_dense_forward: NULL argument");
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
    if (ldg < N || (dx && (ldw < K || lddx < K)) || (dweight && ldx < K)) return nm_fail("nm_dense_backward: row stride shorter than a row");
    if (!workspace || workspace_bytes < nm_dense_workspace_bytes(M, K, N, dtype, 1)) return nm_fail("nm_dense_backward: workspace too small");
    const int k = (int)K, n = (int)N;
    char* ws = (char*)workspace;
    if (dtype == NM_F32) return nm_d_backward<NM_F32>(g, ldg, deriv, x, ldx, weight, ldw, M, k, n, dx, lddx, dweight, dbias, bias_dtype, ws, stream);
    if (dtype == NM_F16) return nm_d_backward<NM_F16>(g, ldg, deriv, x, ldx, weight, ldw, M, k, n, dx, lddx, dweight, dbias, bias_dtype, ws, stream);
    return nm_d_backward<NM_BF16>(g, ldg, deriv, x, ldx, weight, ldw, M, k, n, dx, lddx, dweight, dbias, bias_dtype, ws, stream);
}

}  // extern "C"
