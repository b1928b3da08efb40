// gated_feed_forward: y = (act(x Wg^T + bg) * (x Wv^T + bv)) Wo^T + bo, forward and backward (gfx950).
//
// Every product is C[m, n] = sum_k A(m, k) B(n, k) with operands of any strides.  The gate and the value projection are one product
// whose output tile holds 32 gate columns next to the 32 value columns of the same hidden units, so that act(a) * v is formed from the
// accumulators; the backward pass forms da = dh v act'(a) and dv = dh act(a) in the same way from the accumulators of dh = dy Wo, which
// is never stored.
#include "cg_vec.h"
#include <type_traits>

namespace {

inline int grp_n(const cg_group* g) { return g && g->n > 1 ? g->n : 1; }
inline size_t grp_stride(const cg_group* g) { return g && g->n > 1 ? (size_t)g->stride : 0; }

// element (row, k) of operand z: p[z * zs + row * rs + k * ks]
template <typename T> struct Mat { const T* p; size_t zs, rs, ks; };

enum { EPI_STORE = 0, EPI_GATE_FWD = 1, EPI_GATE_BWD = 2 };

template <typename T> struct Gemm {
    Mat<T> A[2], B[2];        // EPI_STORE: nseg pairs, summed; EPI_GATE_FWD: B[0] gate, B[1] value weights
    int nseg;
    size_t M, K;
    int N;                    // EPI_GATE_FWD: hidden units
    int gate;
    T* c; size_t cz;          // EPI_STORE: C[m * N + n]
    int accumulate;
    const T* bias[2]; size_t bz;
    T *o0, *o1, *o2;          // EPI_GATE_FWD: h, a, v; EPI_GATE_BWD: da, dv
    const T *i0, *i1;         // EPI_GATE_BWD: a, v
    size_t oz;
};

__device__ __forceinline__ void gate_fn(float a, int gate, float& u, float& du) {
    if (gate == CG_GATE_GELU) {
        const float cdf = 0.5f * erfcf(-a * 0.70710678118654752f);
        u = a * cdf;
        du = cdf + a * expf(-0.5f * a * a) * 0.39894228040143268f;
    } else {
        const float s = 1.f / (1.f + expf(-a));
        u = gate == CG_GATE_SILU ? a * s : s;
        du = gate == CG_GATE_SILU ? s + u * (1.f - s) : s * (1.f - s);
    }
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int TM = 64, TN = 64, TK = 16, LD = 68;

// 64 x 64 tile, four waves of 16 rows, exact fp32 products on v_mfma_f32_16x16x4_f32 for every type
template <typename T, int EPI>
__global__ __launch_bounds__(256) void gemm_kernel(Gemm<T> g) {
    __shared__ float As[TK][LD], Bs[TK][LD];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const size_t z = blockIdx.z;
    const size_t m0 = (size_t)blockIdx.x * TM;
    const int n0 = blockIdx.y * (EPI == EPI_GATE_FWD ? TN / 2 : TN);
    f32x4 acc[4] = {};
    for (int s = 0; s < g.nseg; ++s) {
        for (size_t k0 = 0; k0 < g.K; k0 += TK) {
            __syncthreads();
#pragma unroll
            for (int q = 0; q < TM * TK / 256; ++q) {
                const int e = q * 256 + tid;
                // the faster index of the load follows the unit stride of the operand
                const Mat<T>& a = g.A[s];
                const int ar = a.ks == 1 ? e / TK : e % TM, ak = a.ks == 1 ? e % TK : e / TM;
                As[ak][ar] = m0 + ar < g.M && k0 + ak < g.K ? (float)a.p[z * a.zs + (m0 + ar) * a.rs + (k0 + ak) * a.ks] : 0.f;
                const int second = EPI == EPI_GATE_FWD ? 1 : s;
                const int ks1 = g.B[second].ks == 1;
                const int br = ks1 ? e / TK : e % TN, bk = ks1 ? e % TK : e / TN;
                const Mat<T>& b = EPI == EPI_GATE_FWD ? g.B[br >> 5] : g.B[s];
                const int n = EPI == EPI_GATE_FWD ? n0 + (br & 31) : n0 + br;
                Bs[bk][br] = n < g.N && k0 + bk < g.K ? (float)b.p[z * b.zs + (size_t)n * b.rs + (k0 + bk) * b.ks] : 0.f;
            }
            __syncthreads();
#pragma unroll
            for (int kk = 0; kk < TK; kk += 4) {
                const float av = As[kk + (lane >> 4)][wid * 16 + (lane & 15)];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(av, Bs[kk + (lane >> 4)][j * 16 + (lane & 15)], acc[j], 0, 0, 0);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const size_t m = m0 + wid * 16 + 4 * (lane >> 4) + r;
        if (m >= g.M) continue;
#pragma unroll
        for (int j = 0; j < (EPI == EPI_GATE_FWD ? 2 : 4); ++j) {
            const int n = n0 + j * 16 + (lane & 15);
            if (n >= g.N) continue;
            const size_t o = m * g.N + n;
            if (EPI == EPI_STORE) {
                float v = acc[j][r] + (g.bias[0] ? (float)g.bias[0][z * g.bz + n] : 0.f);
                T* c = g.c + z * g.cz + o;
                *c = (T)(g.accumulate ? (float)*c + v : v);
            } else if (EPI == EPI_GATE_FWD) {
                const T a = (T)(acc[j][r] + (g.bias[0] ? (float)g.bias[0][z * g.bz + n] : 0.f));
                const T v = (T)(acc[j + 2][r] + (g.bias[1] ? (float)g.bias[1][z * g.bz + n] : 0.f));
                float u, du;
                // act(a) v from the rounded a, v that the backward pass differentiates
                gate_fn((float)a, g.gate, u, du);
                g.o0[z * g.oz + o] = (T)(u * (float)v);
                if (g.o1) {
                    g.o1[z * g.oz + o] = a;
                    g.o2[z * g.oz + o] = v;
                }
            } else {
                float u, du;
                gate_fn((float)g.i0[z * g.oz + o], g.gate, u, du);
                const float d = acc[j][r];
                g.o0[z * g.oz + o] = (T)(d * (float)g.i1[z * g.oz + o] * du);
                g.o1[z * g.oz + o] = (T)(d * u);
            }
        }
    }
}

template <typename T, int EPI> void gemm(const Gemm<T>& g, int nz, hipStream_t st) {
    if (!g.M || !g.N) return;
    gemm_kernel<T, EPI><<<dim3(cg_div_up(g.M, TM), cg_div_up(g.N, EPI == EPI_GATE_FWD ? TN / 2 : TN), nz), 256, 0, st>>>(g);
}

// da, dv from a stored gradient of h (no output projection)
template <typename T>
__global__ __launch_bounds__(256) void gate_bwd_kernel(const T* __restrict__ dh, const T* __restrict__ a, const T* __restrict__ v,
                                                       T* __restrict__ da, T* __restrict__ dv, size_t n, int gate) {
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        float u, du;
        gate_fn((float)a[i], gate, u, du);
        const float d = (float)dh[i];
        da[i] = (T)(d * (float)v[i] * du);
        dv[i] = (T)(d * u);
    }
}

// out[z * zs + c] (+)= sum over the member's rows of p[r * C + c]
template <typename T>
__global__ __launch_bounds__(256) void colsum_kernel(const T* __restrict__ p, T* __restrict__ out, size_t rows, int C, size_t zs,
                                                     int accumulate) {
    __shared__ float sm[4][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
    const size_t z = blockIdx.y;
    float s = 0.f;
    if (c < C)
        for (size_t r = w; r < rows; r += 4) s += (float)p[(z * rows + r) * C + c];
    sm[w][threadIdx.x & 63] = s;
    __syncthreads();
    if (w == 0 && c < C) {
        s = sm[0][threadIdx.x] + sm[1][threadIdx.x] + sm[2][threadIdx.x] + sm[3][threadIdx.x];
        T* o = out + z * zs + c;
        *o = (T)(accumulate ? (float)*o + s : s);
    }
}

bool dims_ok(const cg_gated_dims* d, const cg_group* grp) {
    return d && d->rows >= 0 && d->rows % grp_n(grp) == 0 && d->D > 0 && d->F > 0 && d->O >= 0 &&
           (d->dtype == CG_DT_F32 || d->dtype == CG_DT_F16 || d->dtype == CG_DT_BF16) && d->gate >= 0 && d->gate <= CG_GATE_SIGMOID &&
           (grp_n(grp) == 1 || d->dtype == CG_DT_F32);
}

inline size_t esize(int dt) { return dt == CG_DT_F32 ? 4 : 2; }
inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

template <typename T>
void fwd(const cg_gated_dims* d, const cg_group* grp, const T* x, const T* wg, const T* wv, const T* wo, const T* bg, const T* bv,
         const T* bo, T* h, T* a, T* v, T* y, hipStream_t st) {
    const int nz = grp_n(grp);
    const size_t M = d->rows / nz, gs = grp_stride(grp);
    const size_t D = d->D, F = d->F;
    Gemm<T> g = {};
    g.nseg = 1;
    g.A[0] = {x, M * D, D, 1};
    g.B[0] = {wg, gs, D, 1};
    g.B[1] = {wv, gs, D, 1};
    g.M = M, g.K = D, g.N = d->F, g.gate = d->gate;
    g.bias[0] = bg, g.bias[1] = bv, g.bz = gs;
    g.o0 = h, g.o1 = a, g.o2 = v, g.oz = M * F;
    gemm<T, EPI_GATE_FWD>(g, nz, st);
    if (d->O) {
        Gemm<T> p = {};
        p.nseg = 1;
        p.A[0] = {h, M * F, F, 1};
        p.B[0] = {wo, gs, F, 1};
        p.M = M, p.K = F, p.N = d->O;
        p.bias[0] = bo, p.bz = gs;
        p.c = y, p.cz = M * d->O;
        gemm<T, EPI_STORE>(p, nz, st);
    }
}

template <typename T>
void bwd(const cg_gated_dims* d, const cg_group* grp, const T* dy, const T* x, const T* wg, const T* wv, const T* wo, const T* h,
         const T* a, const T* v, T* dx, T* dwg, T* dwv, T* dwo, T* dbg, T* dbv, T* dbo, int acc, T* da, T* dv, hipStream_t st) {
    const int nz = grp_n(grp);
    const size_t M = d->rows / nz, gs = grp_stride(grp);
    const size_t D = d->D, F = d->F, O = d->O;
    if (dx || dwg || dwv || dbg || dbv) {
        if (O) {
            Gemm<T> g = {};
            g.nseg = 1;
            g.A[0] = {dy, M * O, O, 1};
            g.B[0] = {wo, gs, 1, F};
            g.M = M, g.K = O, g.N = d->F, g.gate = d->gate;
            g.o0 = da, g.o1 = dv, g.i0 = a, g.i1 = v, g.oz = M * F;
            gemm<T, EPI_GATE_BWD>(g, nz, st);
        } else if (M) {
            const size_t n = (size_t)d->rows * F, nb = (n + 255) / 256;
            gate_bwd_kernel<T><<<(unsigned)(nb < 16384 ? nb : 16384), 256, 0, st>>>(dy, a, v, da, dv, n, d->gate);
        }
    }
    if (dx) {
        Gemm<T> g = {};
        g.nseg = 2;
        g.A[0] = {da, M * F, F, 1}, g.A[1] = {dv, M * F, F, 1};
        g.B[0] = {wg, gs, 1, D}, g.B[1] = {wv, gs, 1, D};
        g.M = M, g.K = F, g.N = d->D;
        g.c = dx, g.cz = M * D;
        gemm<T, EPI_STORE>(g, nz, st);
    }
    auto wgrad = [&](const T* p, size_t P, const T* q, size_t Q, T* dw, int bit) {
        if (!dw) return;
        Gemm<T> g = {};
        g.nseg = 1;
        g.A[0] = {p, M * P, 1, P};
        g.B[0] = {q, M * Q, 1, Q};
        g.M = P, g.K = M, g.N = (int)Q;
        g.c = dw, g.cz = gs, g.accumulate = acc >> bit & 1;
        gemm<T, EPI_STORE>(g, nz, st);
    };
    wgrad(da, F, x, D, dwg, 0);
    wgrad(dv, F, x, D, dwv, 1);
    if (O) wgrad(dy, O, h, F, dwo, 2);
    auto bgrad = [&](const T* p, int C, T* db, int bit) {
        if (db) colsum_kernel<T><<<dim3(cg_div_up(C, 64), nz), 256, 0, st>>>(p, db, M, C, gs, acc >> bit & 1);
    };
    bgrad(da, d->F, dbg, 3);
    bgrad(dv, d->F, dbv, 4);
    if (O) bgrad(dy, d->O, dbo, 5);
}

}  // namespace

extern "C" size_t cg_gated_ff_fwd_workspace(const cg_gated_dims* d, const cg_group* grp) {
    (void)d, (void)grp;
    return 0;
}

extern "C" int cg_gated_ff_fwd(const cg_gated_dims* d, const cg_group* grp, const void* x, const void* wg, const void* wv, const void* wo,
                               const void* bg, const void* bv, const void* bo, void* h, void* a, void* v, void* y, void* ws,
                               size_t ws_bytes, cg_stream_t stream) {
    CG_CHECK_ARG(dims_ok(d, grp) && wg && wv && !a == !v && (!d->O || wo) && (!d->rows || (x && h && (!d->O || y))), "cg_gated_ff_fwd: bad args");
    if (ws_bytes < cg_gated_ff_fwd_workspace(d, grp) || (!ws && cg_gated_ff_fwd_workspace(d, grp)))
        return cg_set_error(CG_ERR_WORKSPACE, "cg_gated_ff_fwd: workspace too small");
    if (!d->rows) return CG_OK;
    CG_DISPATCH_DT(d->dtype, T, (fwd<T>(d, grp, (const T*)x, (const T*)wg, (const T*)wv, (const T*)wo, (const T*)bg, (const T*)bv,
                                        (const T*)bo, (T*)h, (T*)a, (T*)v, (T*)y, cg_s(stream))));
    CG_LAUNCH_CHECK("cg_gated_ff_fwd");
    return CG_OK;
}

extern "C" size_t cg_gated_ff_bwd_workspace(const cg_gated_dims* d, const cg_group* grp) {
    (void)grp;
    return dims_ok(d, nullptr) ? 2 * up256((size_t)d->rows * d->F * esize(d->dtype)) : 0;
}

extern "C" int cg_gated_ff_bwd(const cg_gated_dims* d, const cg_group* grp, const void* dy, const void* x, const void* wg,
                               const void* wv, const void* wo, const void* h, const void* a, const void* v, void* dx, void* dwg,
                               void* dwv, void* dwo, void* dbg, void* dbv, void* dbo, int accumulate, void* ws, size_t ws_bytes,
                               cg_stream_t stream) {
    CG_CHECK_ARG(dims_ok(d, grp) && wg && wv && (!d->O || wo) &&
                     (!d->rows || (dy && x && a && v && (!d->O || h))), "cg_gated_ff_bwd: bad args");
    const size_t need = cg_gated_ff_bwd_workspace(d, grp);
    if (ws_bytes < need || (!ws && need)) return cg_set_error(CG_ERR_WORKSPACE, "cg_gated_ff_bwd: workspace too small");
    CG_DISPATCH_DT(d->dtype, T, {
        T* da = (T*)ws;
        T* dv = (T*)((char*)ws + need / 2);
        bwd<T>(d, grp, (const T*)dy, (const T*)x, (const T*)wg, (const T*)wv, (const T*)wo, (const T*)h, (const T*)a, (const T*)v, (T*)dx,
               (T*)dwg, (T*)dwv, (T*)dwo, (T*)dbg, (T*)dbv, (T*)dbo, accumulate, da, dv, cg_s(stream));
    });
    CG_LAUNCH_CHECK("cg_gated_ff_bwd");
    return CG_OK;
}
