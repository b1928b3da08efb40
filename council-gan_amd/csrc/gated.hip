// gated_feed_forward: y = (act(x Wg^T + bg) * (x Wv^T + bv)) Wo^T + bo, forward and backward (gfx950).
//
// Every product is C[m, n] = sum_k A(m, k) B(n, k).  The gate and the value projection are one product
// whose output tile holds 32 gate columns next to the 32 value columns of the same hidden units, so that act(a) * v is formed from the
// accumulators; the backward pass forms da = dh v act'(a) and dv = dh act(a) in the same way from the accumulators of dh = dy Wo, which
// is never stored.
#include "cg_vec.h"
#include <type_traits>

namespace {

inline int grp_n(const cg_group* g) { return g && g->n > 1 ? g->n : 1; }
inline size_t grp_stride(const cg_group* g) { return g && g->n > 1 ? (size_t)g->stride : 0; }

constexpr int MAX_ROWS = 1 << 30;       // a step past the last row is still an int
constexpr int MAX_WIDTH = 1 << 21;      // a tile's offsets stay below 2^31 bytes

enum { EPI_STORE = 0, EPI_GATE_FWD = 1, EPI_GATE_BWD = 2 };

// C[m, n] = sum_k A(m, k) B(n, k).  Operands are "K-contiguous" (A(m, k) = A[m * ld + k]) or "row-contiguous" (A(m, k) = A[k * ld + m]).
template <typename T> struct Gemm {
    const T *A[2], *B[2];     // nseg pairs are summed; nsel results share B[0] (sel picks A and C); EPI_GATE_FWD: B = gate, value weights
    size_t az, bz, lda, ldb;  // member strides, leading dimensions
    int nseg, nsel;
    size_t M, K;
    int N;                    // EPI_GATE_FWD: hidden units
    T* c[2];                  // EPI_STORE: C[m * N + n]
    size_t cz;
    int accumulate;           // bit sel
    const T* bias[2];
    size_t biasz;
    int gate;
    T *o0, *o1, *o2;          // EPI_GATE_FWD: h and, for the backward pass, u = act(a) and p = v act'(a); EPI_GATE_BWD: da, dv (few rows: float)
    const T *i0, *i1;         // EPI_GATE_BWD: u, p
    unsigned short* low;      // 16 bit: the third bytes of u and p (keep)
    int ld0, ldf;             // pitch of h; of u, p, da, dv.  A pitch beyond N is a multiple of 8 and its columns get zeros
    float* sums;              // EPI_GATE_BWD, or NULL: column sums of da and dv over a wave's rows, [member][2][strips][N]
    int strips;
    float* part;              // splits > 1: partial sums [split][member * nsel + sel][M][planes][NP]
    int splits, tiles_m, tiles_n;
};

// u = act(a), du = act'(a).  The epilogues evaluate this for every hidden unit, where the library's expf, division and erfcf took 16 of the
// 39 us of a 777 x 2816 gate product: exponentials are one v_exp_f32 (of 2^x), reciprocals one v_rcp_f32, each good to an ulp.
//   fp32: the argument's product with log2 e is carried in two parts (its rounding alone would cost |a| half ulps of the result).  Beyond
//   -88.72 the exponential is infinite and the gate 0 (a clamp that kept it finite would leave silu a multiple of a); from -87.34 on its
//   reciprocal is below the normal numbers, which v_rcp_f32 gives as 0 (off by 1e-38, silu by 1e-36);
//   16 bit: one part -- the error stays below 2^-17 for every |a| that does not end in 0 or 1.
// gelu, 16 bit: erfc(z) = t exp(-z^2 + P(t)), t = 1 / (1 + z / 2), with the degree-9 Chebyshev fit of Press et al., Numerical Recipes,
// section 6.2 (relative error 1.2e-7 everywhere); fp32: the library's erfcf.
template <bool FP32> __device__ __forceinline__ float exp_neg(float a) {       // exp(-a)
    constexpr float L = 1.44269504f, L_LO = 1.92596299e-8f;                     // log2 e
    if (!FP32) return __builtin_amdgcn_exp2f(-a * L);
    const float c = __builtin_amdgcn_fmed3f(a, -104.f, 104.f), h = -c * L, l = -(__builtin_fmaf(c, L, h) + c * L_LO);
    const float e = __builtin_amdgcn_exp2f(h);
    return h < 128.f ? __builtin_fmaf(e, l * 0.69314718f, e) : e;      // from 2^128 on e is infinite, and inf l + inf NaN where l < 0
}
template <bool FP32> __device__ __forceinline__ void gate_fn(float a, int gate, float& u, float& du) {
    if (gate == CG_GATE_GELU) {
        if (FP32) {
            const float cdf = 0.5f * erfcf(-a * 0.70710678f);
            u = a * cdf;
            du = cdf + a * exp_neg<true>(0.5f * a * a) * 0.39894228f;
        } else {
            const float z = fabsf(a) * 0.70710678f, t = __builtin_amdgcn_rcpf(1.f + 0.5f * z), g = exp_neg<false>(0.5f * a * a);
            float q = 0.17087277f;
            q = __builtin_fmaf(q, t, -0.82215223f);
            q = __builtin_fmaf(q, t, 1.48851587f);
            q = __builtin_fmaf(q, t, -1.13520398f);
            q = __builtin_fmaf(q, t, 0.27886807f);
            q = __builtin_fmaf(q, t, -0.18628806f);
            q = __builtin_fmaf(q, t, 0.09678418f);
            q = __builtin_fmaf(q, t, 0.37409196f);
            q = __builtin_fmaf(q, t, 1.00002368f);
            q = __builtin_fmaf(q, t, -1.26551223f);
            const float tail = 0.5f * t * g * exp_neg<false>(-q), cdf = a > 0.f ? 1.f - tail : tail;      // 0.5 erfc(|z|)
            u = a * cdf;
            du = cdf + a * g * 0.39894228f;
        }
    } else {
        float s = __builtin_amdgcn_rcpf(1.f + exp_neg<FP32>(a));
        if (FP32) s = a != a ? a : s;       // the clamped exponential hides a NaN
        u = gate == CG_GATE_SILU ? a * s : s;
        du = gate == CG_GATE_SILU ? s + u * (1.f - s) : s * (1.f - s);
    }
}

// 16-bit types keep u and p for the backward pass as the upper 24 bits of their fp32 values: a plane of upper halves each, and one of both
// third bytes.  Rounded to 16 bits they would put another full rounding into da and dv (the gradients 1.7 output roundings off instead
// of 1.4); the third plane is 0.37 of the 2.9 GB and some 50 of the 3045 us of 16384 x 2048 x 5632 bf16.  Cutting off is below 2^-15.
__device__ __forceinline__ unsigned bits(float x) { return __builtin_bit_cast(unsigned, x); }
__device__ __forceinline__ float from(unsigned x) { return __builtin_bit_cast(float, x); }
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void keep(const float (&u)[8], const float (&p)[8], u32x4& hu, u32x4& hp, u32x4& low) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const unsigned u0 = bits(u[2 * k]), u1 = bits(u[2 * k + 1]), p0 = bits(p[2 * k]), p1 = bits(p[2 * k + 1]);
        hu[k] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
        hp[k] = __builtin_amdgcn_perm(p1, p0, 0x07060302u);
        low[k] = __builtin_amdgcn_perm(p0, u0, 0x0c0c0501u) | __builtin_amdgcn_perm(p1, u1, 0x05010c0cu);
    }
}
__device__ __forceinline__ void recall(float (&u)[8], float (&p)[8], const u32x4& hu, const u32x4& hp, const u32x4& low) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        u[2 * k] = from(__builtin_amdgcn_perm(hu[k], low[k], 0x0504000cu));
        u[2 * k + 1] = from(__builtin_amdgcn_perm(hu[k], low[k], 0x0706020cu));
        p[2 * k] = from(__builtin_amdgcn_perm(hp[k], low[k], 0x0504010cu));
        p[2 * k + 1] = from(__builtin_amdgcn_perm(hp[k], low[k], 0x0706030cu));
    }
}

// ------------------------------------------------------------------------------------------
// epilogue of 8 consecutive columns: v = the sums (EPI_GATE_FWD: of the gate, w of the value projection).  What it reads is fetched
// ahead: the biases of its columns once, the rest of a row (`Row`) while earlier rows are on their way out.
// ------------------------------------------------------------------------------------------
template <typename T> struct Chunk { typename CgT<T>::V q[8 / CgT<T>::N]; };
template <typename T> __device__ __forceinline__ void get(Chunk<T>& c, const T* p, int left) {
    constexpr int W = CgT<T>::N;
    if (left >= 8) {
#pragma unroll
        for (int i = 0; i < 8 / W; ++i) c.q[i] = *(const typename CgT<T>::V*)(p + i * W);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) c.q[i / W][i % W] = i < left ? p[i] : (T)0.f;
    }
}
template <typename T> struct Row { Chunk<T> x, y, z; };
template <typename T, int EPI> __device__ __forceinline__ void fetch_row(const Gemm<T>& g, size_t z, int sel, size_t m, int n, Row<T>& r) {
    const int left = m < g.M ? g.N - n : 0;
    if (EPI == EPI_STORE && (g.accumulate >> sel & 1)) get<T>(r.x, g.c[sel] + z * g.cz + m * g.N + n, left);
    if (EPI == EPI_GATE_BWD) {
        const size_t o = (z * g.M + m) * g.ldf + n;
        get<T>(r.x, g.i0 + o, m < g.M ? g.ldf - n : 0);
        get<T>(r.y, g.i1 + o, m < g.M ? g.ldf - n : 0);
        if (sizeof(T) == 2) get<T>(r.z, (const T*)g.low + o, m < g.M ? g.ldf - n : 0);
    }
}
struct Bias { float x[8], y[8]; };
template <typename T, int EPI> __device__ __forceinline__ void fetch_bias(const Gemm<T>& g, size_t z, int n, Bias& b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b.x[i] = b.y[i] = 0.f;
    if (EPI != EPI_GATE_BWD && g.bias[0]) cg_load<T, 8>(g.bias[0] + z * g.biasz + n, g.N - n, b.x);
    if (EPI == EPI_GATE_FWD && g.bias[1]) cg_load<T, 8>(g.bias[1] + z * g.biasz + n, g.N - n, b.y);
}

template <typename T, int EPI>
__device__ __forceinline__ void emit(const Gemm<T>& g, size_t z, int sel, size_t m, int n, float (&v)[8], float (&w)[8], const Bias& b,
                                     const Row<T>& row, float (&sx)[8], float (&sy)[8]) {
    constexpr int W = CgT<T>::N;
    const int left = g.N - n;
    if (EPI == EPI_STORE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] += b.x[i];
            if (g.accumulate >> sel & 1) v[i] += (float)row.x.q[i / W][i % W];
        }
        cg_store<T, 8>(g.c[sel] + z * g.cz + m * g.N + n, left, v);
        return;
    }
    const size_t of = (z * g.M + m) * g.ldf + n;
    if (EPI == EPI_GATE_FWD) {
        float h[8], u, du;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // formed in fp32 from the sums; 16 bit: h, da and dv are rounded as operands of further 16-bit products.  With u and p, and not a
            // and v, in memory no rounding goes through the gate, and the backward pass evaluates none.
            w[i] += b.y[i];
            gate_fn<sizeof(T) == 4>(v[i] + b.x[i], g.gate, u, du);
            h[i] = i < left ? u * w[i] : 0.f;
            v[i] = u;
            w[i] *= du;
        }
        cg_store<T, 8>(g.o0 + (z * g.M + m) * g.ld0 + n, g.ld0 - n, h);
        if (g.o1) {
            if constexpr (sizeof(T) == 2) {
                typedef typename CgT<T>::V V;
                u32x4 hu, hp, low;
                keep(v, w, hu, hp, low);
                *(V*)(g.o1 + of) = __builtin_bit_cast(V, hu);
                *(V*)(g.o2 + of) = __builtin_bit_cast(V, hp);
                *(V*)((T*)g.low + of) = __builtin_bit_cast(V, low);
            } else {
                cg_store<T, 8>(g.o1 + of, 8, v);
                cg_store<T, 8>(g.o2 + of, 8, w);
            }
        }
    } else {
        float u[8], p[8];
        if constexpr (sizeof(T) == 2) {
            recall(u, p, __builtin_bit_cast(u32x4, row.x.q[0]), __builtin_bit_cast(u32x4, row.y.q[0]), __builtin_bit_cast(u32x4, row.z.q[0]));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) u[i] = row.x.q[i / W][i % W], p[i] = row.y.q[i / W][i % W];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = i < left ? v[i] * u[i] : 0.f;
            v[i] = i < left ? v[i] * p[i] : 0.f;
            sx[i] += v[i];
            sy[i] += w[i];
        }
        cg_store<T, 8>(g.o0 + of, g.ldf - n, v);
        cg_store<T, 8>(g.o1 + of, g.ldf - n, w);
    }
}

template <int EPI> constexpr int planes() { return EPI == EPI_GATE_FWD ? 2 : 1; }
__host__ __device__ __forceinline__ size_t pad8(int n) { return (size_t)((n + 7) & ~7); }

// ------------------------------------------------------------------------------------------
// Products of fp32 operands on v_mfma_f32_32x32x16_bf16: 128 x 128 tiles, 4 waves of 64 x 64; 64 x 64 tiles, 2 waves of 32 x 64.
//
// The operands are split exactly into three bf16 values on their way to LDS, x = h + m + l (round to nearest even, 8 + 8 + 8
// significant bits), and a product is the six terms hh, hm, mh, hl, mm, lh: what is left out is below 2^-23 of |x y|, half a
// rounding of an fp32 product.  Six products on the 16-bit matrix pipe take less than half the time of one fp32 product on the fp32 one.
//
// LDS: a K-contiguous operand lies as [row][K-step] with its 16-byte chunks xor-swizzled by the row, so that the 16 rows that one
// pass of ds_read_b128 reads (a chunk of each) cover all 64 banks once; a row-contiguous one lies as [k][row], its chunks xor-swizzled by
// the depth, and is transposed by the read (ds_read_b64_tr_b16: inside 16 lanes, lane s names the address of 4 values X[s][0..3] and lane
// i gets X[4 j + i / 4][i % 4]; the four depths that they gather lie 64 bytes apart).
// ------------------------------------------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((__vector_size__(4 * sizeof(short))));

template <typename E> struct V8 { typedef E V __attribute__((ext_vector_type(8))); };
__device__ __forceinline__ f32x16 mfma(typename V8<cg_h16>::V a, typename V8<cg_h16>::V b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(typename V8<cg_b16>::V a, typename V8<cg_b16>::V b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// One operand of a tile: global -> registers -> LDS, and the fragments of one 16-deep step
template <int ROWS, int NT, bool KC, bool GATE> struct Operand {
    typedef float T;
    typedef cg_b16 E;
    typedef V8<E>::V Frag;
    typedef CgT<T>::V Raw;
    static constexpr int P = 3, BK = 32, W = CgT<T>::N;
    static constexpr int CPR = KC ? BK / W : ROWS / W;             // chunks of W elements per LDS row
    static constexpr int CH = (KC ? ROWS : BK) * CPR / NT;
    static constexpr int PITCH = KC ? BK * 2 : ROWS * 2;           // bytes
    static constexpr int PLANE = (KC ? ROWS : BK) * PITCH;
    static constexpr int BYTES = P * PLANE;
    static_assert(CH >= 1 && ((KC ? ROWS : BK) * CPR) % NT == 0, "every thread has the same number of chunks");

    struct Regs { Raw q[CH]; };
    unsigned off[CH];    // bytes from the tile's origin: of the row (K-contiguous), of the chunk (row-contiguous); below 2^31 (MAX_WIDTH)
    int tid, col, shift; // row-contiguous: first row of the thread's chunk, and how far it was moved back to end with the operand

    static __device__ __forceinline__ int lrow(int tid, int i) { return (tid + i * NT) / CPR; }
    static __device__ __forceinline__ int lch(int tid) { return tid % CPR; }
    static_assert(NT % CPR == 0, "a thread keeps its chunk column");

    // Every chunk is loaded whole from inside the operand (of at least W in the contiguous direction), without a branch: rows past the end
    // come from a row that exists (what they give is never stored), a chunk that would cross the end is moved back, and `store` puts that
    // right where it matters -- so the loads of two steps stay in flight together.
    __device__ __forceinline__ void init(int t, size_t row0, size_t rows, size_t ld) {
        tid = t;
        if (KC) {
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                int j = lrow(tid, i);
                if (GATE) j = (j >> 6) * 32 + (j & 31);
                const size_t r = row0 + j;
                off[i] = (unsigned)(((r < rows ? r : rows - 1) - row0) * ld * sizeof(T));
            }
        } else {
            const long long r = (long long)row0 + lch(tid) * W, most = (long long)rows - W;
            col = (int)(r < most ? r : most);
            shift = (int)(r - col < W ? r - col : 0);
#pragma unroll
            for (int i = 0; i < CH; ++i) off[i] = (unsigned)((lrow(tid, i) * ld + col) * sizeof(T));
        }
    }
    // p0, p1: the operands (K-contiguous: from the tile's first row on)
    __device__ __forceinline__ void load(Regs& raw, const T* p0, const T* p1, int k0, int K, size_t ld) const {
        auto at = [](const T* p, unsigned o) { return (const Raw*)((const char*)p + o); };
        if (KC) {
            const int k = k0 + lch(tid) * W;
            const unsigned kc = (unsigned)(k < K - W ? k : K - W) * (unsigned)sizeof(T);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                const bool second = GATE && (i * (NT / CPR) >> 5 & 1);       // rows 32 .. 63 of 64; a thread's first row is below 32
                raw.q[i] = *at(second ? p1 : p0, off[i] + kc);
            }
        } else {
            unsigned o[CH];
#pragma unroll
            for (int i = 0; i < CH; ++i) o[i] = off[i];
            if (k0 + BK > K)
#pragma unroll
                for (int i = 0; i < CH; ++i) {
                    const int r = lrow(tid, i), last = K - 1 - k0;
                    o[i] = (unsigned)(((r < last ? r : last) * ld + col) * sizeof(T));
                }
#pragma unroll
            for (int i = 0; i < CH; ++i) raw.q[i] = *at(p0 + (size_t)k0 * ld, o[i]);
        }
    }
    // the elements of a chunk moved down by s, zeros behind (s >= W: all zero)
    static __device__ __forceinline__ Raw moved(Raw v, int s) {
        if (s & 2) v = Raw{v[2], v[3], 0, 0};
        if (s & 1) v = Raw{v[1], v[2], v[3], 0};
        if (s >= W) v = Raw{0, 0, 0, 0};
        return v;
    }
    // what step k0 loaded, with zeros past K
    __device__ __forceinline__ void fix(Regs& raw, int k0, int K, size_t row0, size_t rows) const {
        const bool tail = k0 + BK > K;
        if (KC && tail) {
            const int k = k0 + lch(tid) * W, s = k - (K - W) > 0 ? k - (K - W) : 0;
#pragma unroll
            for (int i = 0; i < CH; ++i) raw.q[i] = moved(raw.q[i], s);
        }
        if (!KC && (tail || (rows % W && row0 + ROWS > rows))) {
#pragma unroll
            for (int i = 0; i < CH; ++i) raw.q[i] = moved(raw.q[i], k0 + lrow(tid, i) < K ? shift : W);
        }
    }
    // where 16-byte chunk `chunk` of LDS row `row` lies in it (a row-contiguous operand's LDS rows are its depths)
    static __device__ __forceinline__ unsigned swz(int row, int chunk) {
        if (!KC) return (unsigned)(chunk ^ (ROWS >= 128 ? (row & 3) << 2 : (row >> 1 & 1) << 2));
        return (unsigned)(chunk ^ ((row >> 2) & 3));
    }
    // FLIP: rows 32 .. 63 of every 64 with the other sign (gemm_kernel)
    template <bool FLIP> __device__ __forceinline__ void store(char* lds, const Regs& raw) const {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            typedef E E4 __attribute__((ext_vector_type(4)));
            const int r = lrow(tid, i), c = lch(tid);
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = FLIP && (i * (NT / CPR) >> 5 & 1) ? -raw.q[i][e] : raw.q[i][e];
            char* d = lds + r * PITCH + swz(r, c >> 1) * 16 + (c & 1) * 8;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                E4 h;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    h[e] = (E)x[e];
                    x[e] -= (float)h[e];
                }
                *(E4*)(d + p * PLANE) = h;
            }
        }
    }
    // rows r0 .. r0 + 31, K-step ks: lane l holds row r0 + l % 32, k = 16 ks + 8 (l / 32) .. + 7
    static __device__ __forceinline__ Frag frag(const char* lds, int lane, int r0, int ks, int p) {
        if constexpr (KC) {
            const int r = r0 + (lane & 31);
            return *(const Frag*)(lds + p * PLANE + r * PITCH + swz(r, 2 * ks + (lane >> 5)) * 16);
        } else {
            typedef __attribute__((address_space(3))) s16x4* Q;
            const int sl = lane & 15;
            // depths k and k + 4 have the same swizzle
            const int k = ks * 16 + (lane >> 5) * 8 + (sl >> 2), c = r0 / 8 + 2 * ((lane >> 4) & 1) + ((sl & 3) >> 1);
            const int at = p * PLANE + k * PITCH + swz(k, c) * 16 + (sl & 1) * 8;
            const Q q = (Q)((const __attribute__((address_space(3))) char*)lds + at);
            struct { s16x4 a, b; } f;
            f.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(q);
            f.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(q + 4 * PITCH / 8);
            return __builtin_bit_cast(Frag, f);
        }
    }
};

// Blocks go to the 8 XCDs in turn: each XCD takes a run of neighbouring tiles, in panels of 8 tile rows, so that what its L2 holds is
// read again.
template <int BM, int BN> __device__ __forceinline__ void tile_origin(int tiles_m, int tiles_n, size_t& m0, int& n0) {
    const unsigned nt = gridDim.x, xcd = blockIdx.x & 7, q = nt / 8, rem = nt % 8;
    const unsigned t = xcd * q + (xcd < rem ? xcd : rem) + (blockIdx.x >> 3);
    const unsigned panel = 8 * tiles_n, pm = t / panel * 8, pr = t % panel, ph = tiles_m - pm < 8 ? tiles_m - pm : 8;
    m0 = (size_t)(pm + pr % ph) * BM;
    n0 = (int)(pr / ph) * BN;
}

// A wave's accumulators (TM x TN blocks of 32 x 32; TN = 2) go through its own 32 x 68 floats of LDS, 32 rows at a time, so that every
// lane stores 8 consecutive columns.  EPI_GATE_FWD: the left 32 columns are the gate, the right ones the value projection.
template <typename T, int EPI, int TM, int TN>
__device__ __forceinline__ void store_tile(const Gemm<T>& g, const f32x16 (&acc)[TM][TN], float* ep, int lane, size_t mw, int nw,
                                           size_t z, int sel, int split, int zs) {
    constexpr int EP = TN * 32 + 4, LPR = EPI == EPI_GATE_FWD ? 4 : 8, RPP = 64 / LPR, PASSES = 32 / RPP;
    static_assert(TN == 2, "a wave's 64 columns are 32 gate and 32 value columns");
    const int n = nw + lane % LPR * 8;
    const size_t ml = mw + lane / LPR;
    const bool whole = g.splits == 1;
    Bias bias;
    float sx[8] = {}, sy[8] = {};
    // the fp32 rows of the gate's backward pass take 64 registers: one set of them, or the tiles lose their third block on a CU (1386 us
    // instead of 1368 for the backward pass of 65536 x 256 x 1024)
    constexpr int SETS = EPI == EPI_GATE_BWD && sizeof(T) == 4 ? 1 : 2;
    Row<T> row[SETS][PASSES];
    auto fetch = [&](int i) {
#pragma unroll
        for (int pass = 0; pass < PASSES; ++pass) fetch_row<T, EPI>(g, z, sel, ml + i * 32 + pass * RPP, n, row[i % SETS][pass]);
    };
    if (whole) {
        fetch_bias<T, EPI>(g, z, n, bias);
        fetch(0);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) ep[(8 * (r >> 2) + 4 * (lane >> 5) + (r & 3)) * EP + j * 32 + (lane & 31)] = acc[i][j][r];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        if (SETS == 2 && whole && i + 1 < TM) fetch(i + 1);
#pragma unroll
        for (int pass = 0; pass < PASSES; ++pass) {
            const int at = (pass * RPP + lane / LPR) * EP + lane % LPR * 8;
            const size_t m = ml + i * 32 + pass * RPP;
            float v[8], w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = ep[at + e];
                if (EPI == EPI_GATE_FWD) w[e] = ep[at + 32 + e];
            }
            if (m < g.M && n < g.N) {
                if (whole) {
                    emit<T, EPI>(g, z, sel, m, n, v, w, bias, row[i % SETS][pass], sx, sy);
                } else {
                    const size_t np = pad8(g.N);
                    float* p = g.part + (((size_t)split * (gridDim.z / g.splits) + zs) * g.M + m) * planes<EPI>() * np + n;
                    cg_store<float, 8>(p, 8, v);
                    if (EPI == EPI_GATE_FWD) cg_store<float, 8>(p + np, 8, w);
                }
            }
        }
        if (SETS == 1 && whole && i + 1 < TM) fetch(i + 1);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
    }
    if (EPI == EPI_GATE_BWD && whole && g.sums) {
        // lanes of the same columns, then one strip of TM x 32 rows for every wave
#pragma unroll
        for (int o = LPR; o < 64; o <<= 1)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sx[e] += __shfl_xor(sx[e], o, 64);
                sy[e] += __shfl_xor(sy[e], o, 64);
            }
        if (lane < LPR && n < g.N) {
            float* p = g.sums + (z * 2 * g.strips + mw / (TM * 32)) * g.N + n;
            cg_store<float, 8>(p, g.N - n, sx);
            cg_store<float, 8>(p + (size_t)g.strips * g.N, g.N - n, sy);
        }
    }
}

// The matrix pipe cuts its sums off downwards a few bits below fp32, so every result is low by some 1e-7 of its size, and a sum of 65536
// of them (a bias gradient) by 1.4e-6, where its random errors come to 4e-7.  So half of A's rows go through with the other sign: the
// errors of neighbouring row blocks cancel in any sum over rows (no time is lost by it).
// One LDS buffer, loads one K-step ahead in registers, and three blocks on a CU: 510 us instead of 577 for the gate product of
// 65536 x 256 x 1024 with two blocks and two steps ahead.
template <int BM, int BN, int WM, int WN, bool KA, bool KB, int EPI>
__global__ __launch_bounds__((BM / WM) * (BN / WN) * 64, BM == 128 ? 3 : 2) void gemm_kernel(Gemm<float> g) {
    typedef float T;
    constexpr int NW = (BM / WM) * (BN / WN), NT = NW * 64, TM = WM / 32, TN = WN / 32;
    typedef Operand<BM, NT, KA, false> OA;
    typedef Operand<BN, NT, KB, EPI == EPI_GATE_FWD> OB;
    constexpr int P = OA::P, BK = OA::BK, EP = WN + 4, BUF = OA::BYTES + OB::BYTES;
    constexpr int SMEM = BUF > NW * 32 * EP * 4 ? BUF : NW * 32 * EP * 4;
    __shared__ __attribute__((aligned(16))) char smem[SMEM];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;

    size_t m0;
    int n0;
    tile_origin<BM, EPI == EPI_GATE_FWD ? BN / 2 : BN>(g.tiles_m, g.tiles_n, m0, n0);
    const int split = blockIdx.z % g.splits, zs = blockIdx.z / g.splits, sel = zs % g.nsel;
    const size_t z = zs / g.nsel;

    f32x16 acc[TM][TN] = {};
    const int wm = wid / (BN / WN) * WM, wn = wid % (BN / WN) * WN;
    const int kt = (int)((g.K + BK - 1) / BK), all = kt * g.nseg;
    const int k_begin = (int)((long long)all * split / g.splits), k_end = (int)((long long)all * (split + 1) / g.splits);
    OA a;
    OB b;
    a.init(tid, m0, g.M, g.lda);
    b.init(tid, n0, g.N, g.ldb);
    typename OA::Regs ra;
    typename OB::Regs rb;
    auto load = [&](int step) {      // behind the end: the last step again
        step = step < k_end ? step : k_end - 1;
        const int s = g.nseg == 2 && step >= kt ? 1 : 0, k = step - s * kt;
        const T* pa = g.nseg == 2 ? (s ? g.A[1] : g.A[0]) : (sel ? g.A[1] : g.A[0]);
        const T* pb = s ? g.B[1] : g.B[0];
        a.load(ra, pa + z * g.az + (KA ? m0 * g.lda : 0), nullptr, k * BK, (int)g.K, g.lda);
        const size_t ob = z * g.bz + (KB ? n0 * g.ldb : 0);
        b.load(rb, pb + ob, EPI == EPI_GATE_FWD ? g.B[1] + ob : nullptr, k * BK, (int)g.K, g.ldb);
    };
    auto store = [&](int step) {
        const int k0 = (g.nseg == 2 && step >= kt ? step - kt : step) * BK;
        a.fix(ra, k0, (int)g.K, m0, g.M);
        b.fix(rb, k0, (int)g.K, n0, g.N);
        a.template store<KA>(smem, ra);
        b.template store<false>(smem + OA::BYTES, rb);
    };
    auto compute = [&](const char* from) {
#pragma unroll
        for (int ks = 0; ks < BK / 16; ++ks) {
            typename OA::Frag fa[TM][P], fb[TN][P];
#pragma unroll
            for (int p = 0; p < P; ++p) {
#pragma unroll
                for (int i = 0; i < TM; ++i) fa[i][p] = OA::frag(from, lane, wm + i * 32, ks, p);
#pragma unroll
                for (int j = 0; j < TN; ++j) fb[j][p] = OB::frag(from + OA::BYTES, lane, wn + j * 32, ks, p);
            }
            // the smaller terms first
#pragma unroll
            for (int d = P - 1; d >= 0; --d)
#pragma unroll
                for (int p = 0; p <= d; ++p)
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j) acc[i][j] = mfma(fa[i][p], fb[j][d - p], acc[i][j]);
        }
    };
    if (k_begin < k_end) {
        load(k_begin);
        for (int step = k_begin; step < k_end; ++step) {
            __syncthreads();
            store(step);
            __syncthreads();
            load(step + 1);
            compute(smem);
        }
    }

    if (KA)
#pragma unroll
        for (int i = 0; i < TM; ++i)
            if ((wm / 32 + i) & 1)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = -acc[i][j];
    // the accumulators leave through LDS
    __syncthreads();
    store_tile<T, EPI, TM, TN>(g, acc, (float*)smem + wid * 32 * EP, lane, m0 + wm, n0 + (EPI == EPI_GATE_FWD ? wn / 2 : wn), z, sel,
                               split, zs);
}

// ------------------------------------------------------------------------------------------
// The same product of 16-bit operands, whose rows start on 16 bytes and end in zeros where they are longer than K: 256 x 256 tiles, 8 waves
// of 128 x 64, one block a CU; 128 x 128 tiles, 4 waves of 64 x 64, two blocks a CU.
//
// The tiles come straight from memory into LDS (buffer_load_dwordx4 ... lds: 64 lanes x 16 bytes to consecutive LDS addresses, no
// registers on the way), so the swizzle is in the address that each lane fetches: chunk c of row r of a K-contiguous tile lies at
// c ^ (r / 2 & 7); chunk c of depth k of a row-contiguous tile at c ^ 4 (k & 3), which puts the four depths that 16 lanes of a transposing
// read gather 64 bytes apart.  What lies outside the operand reads as zero (buffer bounds).
// A K-contiguous row gives a whole 128-byte line (64 K-steps) to a load: with 64 bytes of a line at a time a piece of 1 KB takes 20 ns
// instead of 9 (the other half has left the 32 KB L1 when its turn comes).
// What bounds the loop is the time from a load to its data, more than a microsecond where it is the first to touch a line, against one
// microsecond of products per 64-deep step.  All 160 KB of LDS hold tiles on their way: three of A and two of B, so A is requested
// almost two steps ahead and B, first of all after a buffer has become free, one step.  The fragments of a 16-deep step are read while the
// step before it is on the matrix pipe, across the change of tiles too: before the last step of a tile every wave has its fragments in
// registers, waits for its own loads of the next tiles, and meets the others.
// The loads are issued from inline assembly because the compiler takes the builtin for a store to all of LDS and would wait for it before
// every read; the waits are therefore by hand.
// ------------------------------------------------------------------------------------------
typedef int rsrc4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void dma16(rsrc4 rsrc, unsigned lds, unsigned off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(lds), "v"(off), "s"(rsrc) : "memory", "m0");
}

constexpr unsigned OUTSIDE = 0x80000000u, MOST = 0x7fffff00u;      // an offset past every bound; the largest bound

template <typename T, int ROWS, bool KC> struct WideOperand {
    typedef typename V8<T>::V Frag;
    static constexpr int BK = 64, PIECES = 4, BYTES = ROWS * BK * 2;      // ROWS / 32 waves
    static constexpr int PITCH = ROWS * 2, LANES = ROWS / 8;               // row-contiguous: bytes and lanes of a depth
    unsigned off[PIECES];
    int k_of[2];     // K-contiguous: first k of the lane's chunk in even and odd pieces
    // the tile to fill next: its address, the bytes and the K-steps from there to the operand's end, the bytes to the next tile
    unsigned long long at;
    long long left, step;
    int room;

    // wave w fills LDS rows w * 32 + 8 i .. (K-contiguous) or its share of the 64 depths, 64 / LANES at a time (row-contiguous)
    __device__ __forceinline__ void init(int w, int lane, size_t ld) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if (KC) {
                const int row = lane >> 3, c = (lane & 7) ^ (((i * 8 + row) >> 1) & 7);
                k_of[i & 1] = c * 8;
                off[i] = (unsigned)((w * 32 + i * 8 + row) * ld * 2) + c * 16;
            } else {
                const int k = (w * PIECES + i) * (64 / LANES) + lane / LANES, c = lane % LANES ^ ((k & 3) << 2);
                off[i] = (unsigned)(k * ld * 2) + c * 16;
            }
        }
    }
    // gate / value weights: wave w's rows come from the gate (w even) or the value (w odd) weights, 32 rows of each in turn
    __device__ __forceinline__ void init_gate(int w, int lane, size_t ld) {
        init(w, lane, ld);
#pragma unroll
        for (int i = 0; i < PIECES; ++i) off[i] -= (unsigned)((w * 32 - (w >> 1) * 32) * ld * 2);
    }
    // p: the operand; row0, k0: the tile's origin; rows, K: the operand's extent
    __device__ __forceinline__ void aim(const T* p, size_t ld, size_t row0, size_t rows, size_t k0, size_t K) {
        const size_t o = (KC ? row0 * ld + k0 : k0 * ld + row0) * 2;
        at = (unsigned long long)p + o;
        left = (long long)((KC ? rows : K) * ld * 2) - (long long)o;
        step = (KC ? BK : BK * (long long)ld) * 2;
        room = K - k0 < 0x40000000 ? (int)(K - k0) : 0x40000000;
    }
    __device__ __forceinline__ void next() {
        at += step;
        left -= step;
        room -= BK;
    }
    __device__ __forceinline__ rsrc4 window() const {
        rsrc4 r;
        r[0] = (int)(unsigned)at;
        r[1] = (int)((unsigned)(at >> 32) & 0xffffu);
        r[2] = left <= 0 ? 0 : left < (long long)MOST ? (int)left : (int)MOST;
        r[3] = 0x00020000;
        return r;
    }
    __device__ __forceinline__ void fill(rsrc4 r, int i, unsigned lds, int w) const {
        dma16(r, lds + (w * PIECES + i) * 1024, KC && k_of[i & 1] >= room ? OUTSIDE : off[i]);
    }
    static __device__ __forceinline__ Frag lds_at(unsigned a) { return *(const __attribute__((address_space(3))) Frag*)(size_t)a; }
    // address of the fragment of rows r0 + 32 j (r0 a multiple of 64) at step 0; frag() adds the step
    static __device__ __forceinline__ unsigned addr(int lane, int r0, int j) {
        if (KC) return (r0 + j * 32 + (lane & 31)) * 128 + (((lane >> 5) ^ ((lane >> 1) & 7)) << 4);
        const int sl = lane & 15, c = (r0 + j * 32) / 8 + ((lane >> 4) & 1) * 2 + ((sl & 3) >> 1);
        return ((lane >> 5) * 8 + (sl >> 2)) * PITCH + ((c ^ ((sl >> 2) << 2)) << 4) + (sl & 1) * 8;
    }
    static __device__ __forceinline__ Frag frag(unsigned base, unsigned a, int ks) {
        if constexpr (KC) {
            return lds_at(base + (a ^ (ks << 5)));
        } else {
            typedef __attribute__((address_space(3))) s16x4* Q;
            struct { s16x4 a, b; } f;
            f.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Q)(size_t)(base + a + ks * 16 * PITCH));
            f.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Q)(size_t)(base + a + ks * 16 * PITCH + 4 * PITCH));
            return __builtin_bit_cast(Frag, f);
        }
    }
};

template <typename T, int TILE, bool KA, bool KB, int EPI> __global__ __launch_bounds__(TILE * 2, 2) void gemm_wide_kernel(Gemm<T> g) {
    typedef WideOperand<T, TILE, KA> OA;
    typedef WideOperand<T, TILE, KB> OB;
    constexpr int TM = TILE / 64, TN = 2, WN = TILE / 64, BK = OA::BK, A_BUFS = 3, LDS_B = A_BUFS * OA::BYTES;
    __shared__ __attribute__((aligned(1024))) char smem[A_BUFS * OA::BYTES + 2 * OB::BYTES];
    const unsigned lds = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    size_t m0;
    int n0;
    tile_origin<TILE, EPI == EPI_GATE_FWD ? TILE / 2 : TILE>(g.tiles_m, g.tiles_n, m0, n0);
    const int split = blockIdx.z % g.splits, zs = blockIdx.z / g.splits, sel = zs % g.nsel;
    const size_t z = zs / g.nsel;
    const int wm = wid / WN * (TILE / 2), wn = wid % WN * 64;

    f32x16 acc[TM][TN] = {};
    const int kt = (int)((g.K + BK - 1) / BK), all = kt * g.nseg;
    const int k_begin = (int)((long long)all * split / g.splits), k_end = (int)((long long)all * (split + 1) / g.splits);
    OA a;
    OB b;
    a.init(wid, lane, g.lda);
    if (EPI == EPI_GATE_FWD) b.init_gate(wid, lane, g.ldb);
    else b.init(wid, lane, g.ldb);
    // the tile to fetch next of either operand: K-step k of segment s, nothing behind k_end
    auto aim_a = [&](int step) {
        const int s = g.nseg == 2 && step >= kt ? 1 : 0;
        const T* p = g.nseg == 2 ? (s ? g.A[1] : g.A[0]) : (sel ? g.A[1] : g.A[0]);
        a.aim(p + z * g.az, g.lda, m0, g.M, (size_t)(step - s * kt) * BK, g.K);
    };
    auto aim_b = [&](int step) {
        const int s = g.nseg == 2 && step >= kt ? 1 : 0;
        const T* p = EPI == EPI_GATE_FWD ? (wid & 1 ? g.B[1] : g.B[0]) : s ? g.B[1] : g.B[0];
        b.aim(p + z * g.bz, g.ldb, n0, g.N, (size_t)(step - s * kt) * BK, g.K);
    };
    int next_a = k_begin, next_b = k_begin;
    const int second = g.nseg == 2 && k_begin < kt ? kt : -1;      // the step at which the second segment begins
    auto advance_a = [&]() {
        a.next();
        if (++next_a == second) aim_a(next_a);
        if (next_a >= k_end) a.left = 0;
    };
    auto advance_b = [&]() {
        b.next();
        if (++next_b == second) aim_b(next_b);
        if (next_b >= k_end) b.left = 0;
    };
    unsigned aa[TM], ba[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) aa[i] = OA::addr(lane, wm, i);
#pragma unroll
    for (int j = 0; j < TN; ++j) ba[j] = OB::addr(lane, wn, j);
    typename OA::Frag fa[2][TM];
    typename OB::Frag fb[2][TN];
    auto read = [&](unsigned la, unsigned lb, int ks, int f) {
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[f][j] = OB::frag(lb, ba[j], ks);
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[f][i] = OA::frag(la, aa[i], ks);
    };
    auto multiply = [&](int f, int half) {       // half of the row blocks
#pragma unroll
        for (int i = half * TM / 2; i < (half + 1) * TM / 2; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = mfma(fa[f][i], fb[f][j], acc[i][j]);
    };
    constexpr int READS = TM * (KA ? 1 : 2) + TN * (KB ? 1 : 2), PER = (READS + TM - 1) / TM;
    auto interleave = [&]() {       // the reads of the next step spread between the first TM (half the) products of this one
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if (k_begin < k_end) {
        aim_a(k_begin);
        aim_b(k_begin);
        auto fill_a = [&](rsrc4 r, int i, unsigned to) { a.fill(r, i, to, wid); };
        unsigned a0 = lds, a1 = a0 + OA::BYTES, a2 = a1 + OA::BYTES, b0 = lds + LDS_B, b1 = b0 + OB::BYTES;
        // tiles 0 of both, then B of step 1 and A of step 1 -- the order that the loop keeps: B of the next step, A of the one after it
#pragma unroll
        for (int i = 0; i < 4; ++i) fill_a(a.window(), i, a0);
#pragma unroll
        for (int i = 0; i < 4; ++i) b.fill(b.window(), i, b0, wid);
        advance_a();
        advance_b();
#pragma unroll
        for (int i = 0; i < 4; ++i) fill_a(a.window(), i, a1);
        asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        {
            const rsrc4 rb = b.window();
#pragma unroll
            for (int i = 0; i < 4; ++i) b.fill(rb, i, b1, wid);
        }
        read(a0, b0, 0, 0);
        for (int step = k_begin; step < k_end; ++step) {
            advance_a();
            advance_b();
            const rsrc4 ra = a.window(), rb = b.window();
            read(a0, b0, 1, 1), multiply(0, 0), interleave();
            fill_a(ra, 0, a2);
            multiply(0, 1);
            fill_a(ra, 1, a2);
            read(a0, b0, 2, 0), multiply(1, 0), interleave();
            fill_a(ra, 2, a2);
            multiply(1, 1);
            fill_a(ra, 3, a2);
            read(a0, b0, 3, 1), multiply(0, 0), interleave(), multiply(0, 1);
            // all but the newest four loads (A of the step after the next) have landed
            asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            b.fill(rb, 0, b0, wid);
            b.fill(rb, 1, b0, wid);
            read(a1, b1, 0, 0), multiply(1, 0), interleave();
            b.fill(rb, 2, b0, wid);
            b.fill(rb, 3, b0, wid);
            multiply(1, 1);
            const unsigned ta = a0, tb = b0;
            a0 = a1, a1 = a2, a2 = ta, b0 = b1, b1 = tb;
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    store_tile<T, EPI, TM, TN>(g, acc, (float*)smem + wid * 32 * 68, lane, m0 + wm, n0 + (EPI == EPI_GATE_FWD ? wn / 2 : wn), z, sel, split,
                               zs);
}

// joins the partial sums of a split product, in the order of the splits
template <typename T, int EPI> __global__ __launch_bounds__(256) void join_kernel(Gemm<T> g, int nz) {
    const size_t np = pad8(g.N), per = g.M * (np / 8), total = per * nz, plane = (size_t)nz * g.M * planes<EPI>() * np;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        const int zs = (int)(i / per), n = (int)(i % (np / 8)) * 8;
        const size_t m = i % per / (np / 8);
        const float* p = g.part + ((size_t)zs * g.M + m) * planes<EPI>() * np + n;
        float v[8] = {}, w[8] = {}, x[8];
        for (int s = 0; s < g.splits; ++s, p += plane) {
            cg_load<float, 8>(p, 8, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += x[e];
            if (EPI == EPI_GATE_FWD) {
                cg_load<float, 8>(p + np, 8, x);
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] += x[e];
            }
        }
        Bias bias;
        Row<T> row;
        fetch_bias<T, EPI>(g, zs / g.nsel, n, bias);
        fetch_row<T, EPI>(g, zs / g.nsel, zs % g.nsel, m, n, row);
        float sx[8] = {}, sy[8] = {};
        emit<T, EPI>(g, zs / g.nsel, zs % g.nsel, m, n, v, w, bias, row, sx, sy);
    }
}

// Operands narrower than one 16-byte chunk (fewer than 4 or 8 channels or hidden units): one output per thread, or per block where K is long.
template <typename T, int EPI> __device__ __forceinline__ void emit1(const Gemm<T>& g, size_t z, int sel, size_t m, int n, float v, float w) {
    const size_t o = (z * g.M + m) * g.ldf + n;
    if (EPI == EPI_STORE) {
        T* c = g.c[sel] + z * g.cz + m * g.N + n;
        v += g.bias[0] ? (float)g.bias[0][z * g.biasz + n] : 0.f;
        *c = (T)(g.accumulate >> sel & 1 ? (float)*c + v : v);
    } else if (EPI == EPI_GATE_FWD) {
        float u, du;
        w += g.bias[1] ? (float)g.bias[1][z * g.biasz + n] : 0.f;
        gate_fn<sizeof(T) == 4>(v + (g.bias[0] ? (float)g.bias[0][z * g.biasz + n] : 0.f), g.gate, u, du);
        g.o0[(z * g.M + m) * g.ld0 + n] = (T)(u * w);
        if (!g.o1) return;
        if constexpr (sizeof(T) == 2) {
            const unsigned x = bits(u), y = bits(w * du);
            ((unsigned short*)g.o1)[o] = (unsigned short)(x >> 16);
            ((unsigned short*)g.o2)[o] = (unsigned short)(y >> 16);
            g.low[o] = (unsigned short)((x >> 8 & 0xff) | (y & 0xff00));
        } else {
            g.o1[o] = u, g.o2[o] = w * du;
        }
    } else {
        float u, p;
        if constexpr (sizeof(T) == 2) {
            const unsigned low = g.low[o];
            u = from((unsigned)((const unsigned short*)g.i0)[o] << 16 | (low & 0xff) << 8);
            p = from((unsigned)((const unsigned short*)g.i1)[o] << 16 | (low & 0xff00));
        } else {
            u = g.i0[o], p = g.i1[o];
        }
        ((float*)g.o0)[o] = v * p;      // few rows multiply in fp32: da and dv are not rounded (narrow_kernel's T is float)
        ((float*)g.o1)[o] = v * u;
    }
}
template <typename T, bool KA, bool KB, int EPI, bool BLOCK> __global__ __launch_bounds__(256) void narrow_kernel(Gemm<T> g) {
    __shared__ float sm[2][4];
    const int sel = blockIdx.z % g.nsel;
    const size_t z = blockIdx.z / g.nsel, total = g.M * g.N, per = BLOCK ? 1 : 256;
    for (size_t o0 = blockIdx.x * per; o0 < total; o0 += gridDim.x * per) {
        const size_t o = BLOCK ? o0 : o0 + threadIdx.x, m = o / g.N;
        const int n = (int)(o % g.N);
        float v = 0.f, w = 0.f;
        if (o < total)
            for (int s = 0; s < g.nseg; ++s) {
                const T* a = (g.nseg == 2 ? g.A[s] : g.A[sel]) + z * g.az + (KA ? m * g.lda : m);
                const T* b = g.B[EPI == EPI_GATE_FWD ? 0 : s] + z * g.bz + (KB ? n * g.ldb : n);
                const T* b1 = g.B[1] + z * g.bz + n * g.ldb;
                for (size_t k = BLOCK ? threadIdx.x : 0; k < g.K; k += BLOCK ? 256 : 1) {
                    const float x = (float)a[KA ? k : k * g.lda];
                    v += x * (float)b[KB ? k : k * g.ldb];
                    if (EPI == EPI_GATE_FWD) w += x * (float)b1[k];
                }
            }
        if (BLOCK) {
            v = wave_sum(v);
            w = wave_sum(w);
            __syncthreads();
            if ((threadIdx.x & 63) == 0) sm[0][threadIdx.x >> 6] = v, sm[1][threadIdx.x >> 6] = w;
            __syncthreads();
            v = sm[0][0] + sm[0][1] + sm[0][2] + sm[0][3];
            w = sm[1][0] + sm[1][1] + sm[1][2] + sm[1][3];
        }
        if (o < total && (!BLOCK || threadIdx.x == 0)) emit1<T, EPI>(g, z, sel, m, n, v, w);
    }
}

// ------------------------------------------------------------------------------------------
// Few rows (at most FEW_ROWS): every product is one launch and reads its weights once, straight into registers -- bound by the weights'
// bytes and, below a few MB, by the launches.  A block owns 16 or 32 columns of the result, its 16 waves share K, and their sums are
// joined through LDS in wave order.  v_mfma_f32_16x16x4_f32 takes 16 columns x 4 K-steps of the weights against 16 rows x 4 K-steps of
// the rows, one value a lane (lane l: column or row l % 16, K-step l / 16): with weights that are K-contiguous a lane loads 16 bytes of
// its row and the K-steps of a product are whichever the lanes hold; row-contiguous weights need no transposition at all.  Every type is
// multiplied in fp32 (16-bit K-contiguous operands on v_mfma_f32_16x16x32, which takes the 16 bytes as they are), and da and dv stay fp32.
// h is rounded to the type: as two 16-bit parts it would cost 8 % of a call of 1 x 1024 x 2816 bf16 and 24 % of 32 x 2048 x 5632.
// FEW_ROWS: as many rows as a block's join has threads for (16 rows x 2 blocks x 2 tiles).  us of these kernels against the tiles, in replayed
// graphs, serving and training: 16 x 256 x 1024 fp32 10 / 33 against 27 / 68, 32 rows 13 / 40 against 29 / 70; 32 x 1024 x 4096 fp32 37 / 135
// against 44 / 123; bf16 16 x 1024 x 2816 13 / 61 against 24 / 75, 32 rows 16 / 105 against 25 / 82; 16 x 2048 x 5632 28 / 127 against
// 35 / 114, 32 rows 37 / 227 against 34 / 115.  Of wide layers the tiles would be the better backward pass from some 17 rows on.
// ------------------------------------------------------------------------------------------
constexpr int FEW_ROWS = 32, FEW_WAVES = 16;

__device__ __forceinline__ f32x4 mfma16(typename V8<cg_h16>::V a, typename V8<cg_h16>::V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(typename V8<cg_b16>::V a, typename V8<cg_b16>::V b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// MT: blocks of 16 rows; KB: the weights are K-contiguous
template <typename T, int MT, bool KB, int EPI> __global__ __launch_bounds__(FEW_WAVES * 64) void few_kernel(Gemm<T> g) {
    constexpr int W = CgT<T>::N, NT = EPI == EPI_GATE_FWD || !KB ? 2 : 1;       // 16-column tiles: gate and value, or even and odd columns
    constexpr int REGS = MT * NT * 4;
    typedef typename CgT<T>::V V;
    typedef std::conditional_t<EPI == EPI_STORE && !KB, float, T> TX;       // the rows: da and dv are fp32
    typedef TX VX __attribute__((ext_vector_type(W), aligned(sizeof(TX))));
    __shared__ float sm[FEW_WAVES * REGS * 64];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, l16 = lane & 15, lk = lane >> 4;
    const size_t z = blockIdx.y;
    const int n0 = blockIdx.x * (KB ? 16 : 32), K = (int)g.K;
    f32x4 acc[MT][NT] = {};
    for (int s = 0; s < g.nseg; ++s) {
        const TX* x[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const size_t m = i * 16 + l16;
            x[i] = (const TX*)g.A[s] + z * g.az + (m < g.M ? m : g.M - 1) * g.lda;
        }
        if constexpr (KB) {
            const size_t n = n0 + l16 < g.N ? n0 + l16 : g.N - 1;
            const T* b[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j] = g.B[j] + z * g.bz + n * g.ldb;
            constexpr int U = 2, STEP = U * 4 * W;      // a wave takes whole 128-byte lines of its rows
            auto multiply = [&](const V(&xa)[MT], const V(&ba)[NT]) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        if constexpr (sizeof(T) == 2) {
                            typedef typename V8<T>::V F;
                            acc[i][j] = mfma16(__builtin_bit_cast(F, ba[j]), __builtin_bit_cast(F, xa[i]), acc[i][j]);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(ba[j][e], xa[i][e], acc[i][j], 0, 0, 0);
                        }
                    }
            };
            int k0 = wid * STEP;
#pragma unroll 2
            for (; k0 + STEP <= K; k0 += FEW_WAVES * STEP) {
                V xa[U][MT], ba[U][NT];
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    const int k = k0 + (q * 4 + lk) * W;
#pragma unroll
                    for (int j = 0; j < NT; ++j) ba[q][j] = *(const V*)(b[j] + k);
#pragma unroll
                    for (int i = 0; i < MT; ++i) xa[q][i] = *(const V*)(x[i] + k);
                }
#pragma unroll
                for (int q = 0; q < U; ++q) multiply(xa[q], ba[q]);
            }
            if (k0 < K) {
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    const int k = k0 + (q * 4 + lk) * W;
                    V xa[MT], ba[NT];
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        const bool in = k + e < K;
#pragma unroll
                        for (int j = 0; j < NT; ++j) ba[j][e] = in ? b[j][k + e] : (T)0.f;
#pragma unroll
                        for (int i = 0; i < MT; ++i) xa[i][e] = in ? x[i][k + e] : (T)0.f;
                    }
                    multiply(xa, ba);
                }
            }
        } else {
            // lane: columns n0 + 2 l16, + 1 of K-step lk; a pair is one load (moved back inside the row where it would cross its end: what the
            // columns past the end get is never stored).  U K-steps are in flight at a time: a block's chain of loads is what takes the time.
            const int n = n0 + 2 * l16, cb = n + 1 < g.N ? n : g.N > 1 ? g.N - 2 : 0;
            const bool odd = n > cb;
            const T* b = g.B[s] + z * g.bz + cb;
            typedef T V2 __attribute__((ext_vector_type(2), aligned(sizeof(T))));
            // K-step e of a chunk of 4 W is k0 + W lk + e in lane group lk: the rows' values are one 16-byte load a lane
            constexpr int U = (MT == 1 ? 64 : 32) / (4 * W);
            for (int k0 = wid * 4 * W * U; k0 < K; k0 += FEW_WAVES * 4 * W * U) {
                V2 ba[U][W];
                VX xa[U][MT];
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    const int k = k0 + (q * 4 + lk) * W;
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        const T* r = b + (size_t)(k + e < K ? k + e : K - 1) * g.ldb;
                        if (g.N > 1) ba[q][e] = *(const V2*)r;
                        else ba[q][e][0] = ba[q][e][1] = *r;
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        if (k + W <= K) {
                            xa[q][i] = *(const VX*)(x[i] + k);
                        } else {
#pragma unroll
                            for (int e = 0; e < W; ++e) xa[q][i][e] = k + e < K ? x[i][k + e] : (TX)0.f;
                        }
                    }
                }
#pragma unroll
                for (int q = 0; q < U; ++q)
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        const bool in = k0 + (q * 4 + lk) * W + e < K;
                        const float w0 = in ? (float)(odd ? ba[q][e][1] : ba[q][e][0]) : 0.f, w1 = in ? (float)ba[q][e][1] : 0.f;
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            acc[i][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(w0, (float)xa[q][i][e], acc[i][0], 0, 0, 0);
                            acc[i][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(w1, (float)xa[q][i][e], acc[i][1], 0, 0, 0);
                        }
                    }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sm[(wid * REGS + (i * NT + j) * 4 + r) * 64 + lane] = acc[i][j][r];
    __syncthreads();
    if (tid < REGS * 64) {
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < FEW_WAVES; ++q) v += sm[q * REGS * 64 + tid];
        sm[tid] = v;        // its own column of the array: nobody else reads it before the barrier
    }
    __syncthreads();
    // column c of the block, row m: tile and register of column (KB: c; else c / 2 of tile c % 2), lane 16 (column / 4) + m % 16
    constexpr int COLS = KB ? 16 : 32;
    if (tid < MT * 16 * COLS) {
        const int m = tid / COLS, c = tid % COLS, i = m >> 4, t = KB ? c : c >> 1, j = KB ? 0 : c & 1;
        const int at = ((i * NT + j) * 4 + (t & 3)) * 64 + (t >> 2) * 16 + (m & 15);
        if ((size_t)m < g.M && n0 + c < g.N) emit1<T, EPI>(g, z, 0, m, n0 + c, sm[at], EPI == EPI_GATE_FWD ? sm[at + 4 * 64] : 0.f);
    }
}

template <typename T, bool KB, int EPI> void few(const Gemm<T>& g, int members, hipStream_t st) {
    if (!g.M || !g.N) return;
    const dim3 grid(cg_div_up(g.N, KB ? 16 : 32), members);
    if (g.M <= 16) few_kernel<T, 1, KB, EPI><<<grid, FEW_WAVES * 64, 0, st>>>(g);
    else few_kernel<T, 2, KB, EPI><<<grid, FEW_WAVES * 64, 0, st>>>(g);
}

// All parameter gradients of few rows in one launch: dW = P^T Q in tiles of 64 x 64 (4 waves of 16 x 64), db = column sums of P.
template <typename T> struct FewGrads {
    struct { const void* p; const T* q; T *dw, *db; int P, Q, ldp, ldq, tiles_q, first, add_w, add_b, p32; } o[3];      // p32: p is fp32
    int n, M;
    size_t gs;
};
template <typename T> __global__ __launch_bounds__(256) void few_grads_kernel(FewGrads<T> g) {
    int i = 0;
    while (i + 1 < g.n && (int)blockIdx.x >= g.o[i + 1].first) ++i;
    const auto& o = g.o[i];
    const int tile = blockIdx.x - o.first, lane = threadIdx.x & 63, l16 = lane & 15, lk = lane >> 4;
    const size_t z = blockIdx.y;
    const int p0 = tile / o.tiles_q * 64 + (threadIdx.x >> 6) * 16, q0 = tile % o.tiles_q * 64;
    const size_t zp = z * g.M * o.ldp;
    const T* q = o.q + z * g.M * o.ldq;
    const int pc = p0 + l16 < o.P ? p0 + l16 : o.P - 1;
    int qc[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) qc[j] = q0 + j * 16 + l16 < o.Q ? q0 + j * 16 + l16 : o.Q - 1;
    f32x4 acc[4] = {};
    float sum = 0.f;
    for (int m0 = 0; m0 < g.M; m0 += 8) {
        float a[2], b[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int m = m0 + h * 4 + lk;
            const bool in = m < g.M;
            const size_t at = zp + (size_t)m * o.ldp + pc;
            a[h] = !in ? 0.f : o.p32 ? ((const float*)o.p)[at] : (float)((const T*)o.p)[at];
            sum += a[h];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[h][j] = in ? (float)q[(size_t)m * o.ldq + qc[j]] : 0.f;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[h], b[h][j], acc[j], 0, 0, 0);
    }
    if (o.dw) {
        T* dw = o.dw + z * g.gs;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = p0 + 4 * lk + r;
            if (row >= o.P) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = q0 + j * 16 + l16;
                if (c >= o.Q) continue;
                T* d = dw + (size_t)row * o.Q + c;
                *d = (T)(o.add_w ? (float)*d + acc[j][r] : acc[j][r]);
            }
        }
    }
    if (o.db && tile % o.tiles_q == 0) {
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (lk == 0 && p0 + l16 < o.P) {
            T* d = o.db + z * g.gs + p0 + l16;
            *d = (T)(o.add_b ? (float)*d + sum : sum);
        }
    }
}

// Tile and number of K splits: 256 x 256 or 128 x 128 (16 bit), 128 x 128 or 64 x 64 (fp32; 4 waves of 64 x 64, 2 of 32 x 64).  The pair with
// the least time by this account is taken: tiles run in rounds of as many as fit the chip, the last one with what is left; a tile takes
// its K-steps, longer where tiles share a CU, and its epilogue; joining splits costs a launch, the lost fusions of the epilogue, and the
// partial sums' way out and back at about 5 TB/s.  A split takes at least 4 K-steps.  The figures below are measured (us).  The number of
// members is left out: a member's results do not depend on how many run beside it.
struct Plan { int tile, splits; };
Plan plan(size_t M, size_t N, size_t K, int nsel, int esz) {
    const size_t bk = esz == 4 ? 32 : 64, steps = (K + bk - 1) / bk, most = steps / 4 > 1 ? steps / 4 : 1;
    Plan p = {128, 1};
    if (!M || !N) return p;
    double best = 1e30;
    for (int c = 0; c < 2; ++c) {
        const int tile = esz == 2 ? 256 >> c : 128 >> c;
        const size_t t = (size_t)cg_div_up(M, tile) * cg_div_up(N, tile) * nsel;
        const size_t slots = esz == 2 ? (tile == 256 ? 256 : 512) : tile == 128 ? 768 : 1024;      // what the chip holds
        const double epilogue = esz == 2 ? (tile == 256 ? 8 : 4) : tile == 128 ? 5 : 2;
        auto step = [&](size_t n) {       // a K-step where n tiles are at work
            if (esz == 2) return tile == 256 ? 1.0 : n > 256 ? 0.9 : 0.7;
            return tile == 128 ? (n > 512 ? 2.2 : n > 256 ? 1.6 : 1.4) : 1.4;
        };
        for (size_t s = 1; s <= most && s <= 64; ++s) {
            const size_t n = t * s, k = (steps + s - 1) / s;
            const double us = n / slots * (k * step(slots) + epilogue) + (n % slots ? k * step(n % slots) + epilogue : 0) +
                              (s > 1 ? 8.0 + 2.0 * 4 * s * M * N * nsel / 5e6 : 0);
            if (us < best) best = us, p = {tile, (int)s};
        }
    }
    return p;
}
size_t part_bytes(size_t M, size_t N, size_t K, int members, int nsel, int esz, int np) {      // N: columns of the product
    const Plan p = plan(M, N, K, nsel, esz);
    return p.splits > 1 ? (size_t)p.splits * members * nsel * M * np * pad8((int)(N / np)) * 4 : 0;
}

template <typename T, bool KA, bool KB, int EPI> void gemm(Gemm<T>& g, int members, float* part, hipStream_t st) {
    if (!g.M || !g.N) return;
    const int nz = members * g.nsel;
    const size_t N = (size_t)g.N * planes<EPI>();
    if constexpr (sizeof(T) == 4) {
        constexpr size_t W = CgT<T>::N;
        if ((KA ? g.K : g.M) < W || (KB ? g.K : (size_t)g.N) < W) {
            g.sums = nullptr;
            if (!g.K || g.K > 64) narrow_kernel<T, KA, KB, EPI, true><<<dim3((unsigned)(g.M * g.N < 65536 ? g.M * g.N : 65536), 1, nz), 256, 0, st>>>(g);
            else narrow_kernel<T, KA, KB, EPI, false><<<dim3((unsigned)(g.M * g.N < 1 << 24 ? (g.M * g.N + 255) / 256 : 65536), 1, nz), 256, 0, st>>>(g);
            return;
        }
    }
    const Plan p = plan(g.M, N, g.K * g.nseg, g.nsel, sizeof(T));
    g.part = part, g.splits = p.splits;
    g.tiles_m = cg_div_up(g.M, p.tile), g.tiles_n = cg_div_up(N, p.tile);
    g.strips = 2 * g.tiles_m;
    if (p.splits > 1) g.sums = nullptr;
    const dim3 grid((unsigned)g.tiles_m * g.tiles_n, 1, nz * p.splits);
    if constexpr (sizeof(T) == 2) {
        if (p.tile == 256) gemm_wide_kernel<T, 256, KA, KB, EPI><<<grid, 512, 0, st>>>(g);
        else gemm_wide_kernel<T, 128, KA, KB, EPI><<<grid, 256, 0, st>>>(g);
    } else {
        if (p.tile == 128) gemm_kernel<128, 128, 64, 64, KA, KB, EPI><<<grid, 256, 0, st>>>(g);
        else gemm_kernel<64, 64, 32, 64, KA, KB, EPI><<<grid, 128, 0, st>>>(g);
    }
    if (p.splits > 1) {
        const size_t nb = (g.M * (pad8(g.N) / 8) * nz + 255) / 256;
        join_kernel<T, EPI><<<(unsigned)(nb < 4096 ? nb : 4096), 256, 0, st>>>(g, nz);
    }
}

// da, dv from a stored gradient of h (no output projection)
template <typename T> struct GateBwd { const T *dh, *u, *p; const unsigned short* low; void *da, *dv; size_t rows; int F, ldf; };
template <typename T, typename TO> __global__ __launch_bounds__(256) void gate_bwd_kernel(GateBwd<T> g) {
    const size_t per = g.ldf / 8;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < g.rows * per; i += (size_t)gridDim.x * 256) {
        const size_t m = i / per;
        const int n = (int)(i % per) * 8;
        float d[8], u[8], p[8];
        cg_load<T, 8>(g.dh + m * g.F + n, g.F - n, d);       // zeros behind F: da and dv end in zeros
        if constexpr (sizeof(T) == 2) {
            typedef typename CgT<T>::V V;
            auto at = [&](const void* q) { return __builtin_bit_cast(u32x4, *(const V*)((const T*)q + m * g.ldf + n)); };
            recall(u, p, at(g.u), at(g.p), at(g.low));
        } else {
            cg_load<T, 8>(g.u + m * g.ldf + n, 8, u);
            cg_load<T, 8>(g.p + m * g.ldf + n, 8, p);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            p[e] = n + e < g.F ? p[e] * d[e] : 0.f;
            u[e] = n + e < g.F ? u[e] * d[e] : 0.f;
        }
        cg_store<TO, 8>((TO*)g.da + m * g.ldf + n, 8, p);
        cg_store<TO, 8>((TO*)g.dv + m * g.ldf + n, 8, u);
    }
}

// Column sums of one or two [rows][C] tensors (bias gradients): strips of rows, then the strips in turn.
constexpr int STRIP_ROWS = 32, MAX_STRIPS = 512;
inline int strips_of(size_t rows) {
    const size_t s = (rows + STRIP_ROWS - 1) / STRIP_ROWS;
    return (int)(s < 1 ? 1 : s > MAX_STRIPS ? MAX_STRIPS : s);
}
template <typename T> struct ColSum { const T* p[2]; T* out[2]; size_t rows, zs; int C, ld, strips, accumulate; float* part; };

template <typename T> __global__ __launch_bounds__(256) void colsum_part_kernel(ColSum<T> g) {
    constexpr int N = CgT<T>::N;
    __shared__ float sm[3][64 * N];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, c = (blockIdx.x * 64 + lane) * N;
    const size_t z = blockIdx.z >> 1, per = (g.rows + g.strips - 1) / g.strips, r0 = blockIdx.y * per;
    const size_t r1 = r0 + per < g.rows ? r0 + per : g.rows;
    const T* p = g.p[blockIdx.z & 1];
    float s[N] = {}, v[N];
    if (p && c < g.C)
#pragma unroll 8
        for (size_t r = r0 + w; r < r1; r += 4) {
            cg_load<T>(p + (z * g.rows + r) * g.ld + c, g.C - c, v);
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] += v[i];
        }
    if (w) {
#pragma unroll
        for (int i = 0; i < N; ++i) sm[w - 1][i * 64 + lane] = s[i];
    }
    __syncthreads();
    if (!w && p && c < g.C) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] += sm[0][i * 64 + lane] + sm[1][i * 64 + lane] + sm[2][i * 64 + lane];
        cg_store<float, N>(g.part + ((size_t)blockIdx.z * g.strips + blockIdx.y) * g.C + c, g.C - c, s);
    }
}
// the strips: 32 columns a block, 32 threads a column, each with its share of the strips in order
template <typename T> __global__ __launch_bounds__(1024) void colsum_join_kernel(ColSum<T> g) {
    __shared__ float sm[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5, sel = blockIdx.z & 1;
    if (!g.out[sel]) return;
    float s = 0.f;
    if (c < g.C) {
        const float* p = g.part + (size_t)blockIdx.z * g.strips * g.C + c;
#pragma unroll 8
        for (int i = k; i < g.strips; i += 32) s += p[(size_t)i * g.C];
    }
    sm[k][threadIdx.x & 31] = s;
    __syncthreads();
    if (k || c >= g.C) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sm[i][threadIdx.x];
    T* o = g.out[sel] + (blockIdx.z >> 1) * g.zs + c;
    *o = (T)(g.accumulate >> sel & 1 ? (float)*o + s : s);
}

bool dims_ok(const cg_gated_dims* d, const cg_group* grp) {
    return d && d->rows >= 0 && d->rows <= MAX_ROWS && d->rows % grp_n(grp) == 0 && d->D > 0 && d->F > 0 && d->O >= 0 &&
           d->D <= MAX_WIDTH && d->F <= MAX_WIDTH && d->O <= MAX_WIDTH &&
           (d->dtype == CG_DT_F32 || d->dtype == CG_DT_F16 || d->dtype == CG_DT_BF16) && d->gate >= 0 && d->gate <= CG_GATE_SIGMOID &&
           (grp_n(grp) == 1 || d->dtype == CG_DT_F32);
}

// what the kernels read 16 bytes at a time without a copy: the caller's buffers between the passes
inline bool aligned16(const void* a, const void* b, const void* c, const void* d) {
    return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c | (uintptr_t)d) & 15) == 0;
}
inline size_t esize(int dt) { return dt == CG_DT_F32 ? 4 : 2; }
inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// Copies of 16-bit operands whose rows do not start on 16 bytes (an odd width, a shifted tensor): rows of a multiple of 8 elements that end
// in zeros.  The tiles are fetched 16 bytes at a time straight into LDS; a copy reads and writes an operand once, where the product
// reads it once for every 256 rows or columns of the result.
template <typename T> struct Pack {
    struct { const T* src; T* dst; size_t first, end; int cols, chunks; } o[4];      // chunks [first, end) of the launch, `chunks` a row
    int n;
};
template <typename T> __global__ __launch_bounds__(256) void pack_kernel(Pack<T> g) {
    const size_t total = g.o[g.n - 1].end;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (size_t)gridDim.x * 256) {
        int j = 0;
        while (i >= g.o[j].end) ++j;
        const size_t c = i - g.o[j].first, r = c / g.o[j].chunks;
        const int k = (int)(c % g.o[j].chunks) * 8;
        float v[8];
        cg_load<T, 8>(g.o[j].src + r * g.o[j].cols + k, g.o[j].cols - k, v);
        cg_store<T, 8>(g.o[j].dst + c * 8, 8, v);
    }
}

// Operands as the products read them: pointer and pitch, packed or in place
template <typename T> struct Operands { const T *x, *wg, *wv, *wo; size_t ldx, ldw, ldo; };
bool packs(const cg_gated_dims* d, const cg_group* grp, const void* p, size_t cols) {
    return d->dtype != CG_DT_F32 && (size_t)d->rows / grp_n(grp) > FEW_ROWS && (cols % 8 != 0 || (uintptr_t)p % 16 != 0);
}
size_t pack_bytes(const cg_gated_dims* d, const cg_group* grp, const void* x, const void* wg, const void* wv, const void* wo) {
    size_t n = 0;
    auto add = [&](const void* p, size_t rows, size_t cols) { n += packs(d, grp, p, cols) ? up256(rows * pad8((int)cols) * 2) : 0; };
    add(x, d->rows, d->D);
    // the two projections share a pitch
    if (packs(d, grp, wg, d->D) || packs(d, grp, wv, d->D)) n += 2 * up256((size_t)d->F * pad8(d->D) * 2);
    if (d->O) add(wo, d->O, d->F);
    return n;
}
// where the operands are once `pack` is filled; run: fill it
template <typename T>
Operands<T> operands(const cg_gated_dims* d, const cg_group* grp, const T* x, const T* wg, const T* wv, const T* wo, void* pack, bool run,
                     hipStream_t st) {
    const size_t D = d->D, F = d->F, dp = pad8(d->D), fp = pad8(d->F);
    Operands<T> r = {x, wg, wv, wo, D, D, F};
    char* at = (char*)pack;
    Pack<T> g = {};
    auto add = [&](const T*& p, size_t rows, size_t cols, size_t pitch) {
        const size_t first = g.n ? g.o[g.n - 1].end : 0;
        auto& o = g.o[g.n++];
        o.src = p, o.dst = (T*)at, o.first = first, o.end = first + rows * (pitch / 8), o.cols = (int)cols, o.chunks = (int)(pitch / 8);
        p = (const T*)at;
        at += up256(rows * pitch * 2);
    };
    if (packs(d, grp, x, D)) add(r.x, d->rows, D, dp), r.ldx = dp;
    if (packs(d, grp, wg, D) || packs(d, grp, wv, D)) add(r.wg, F, D, dp), add(r.wv, F, D, dp), r.ldw = dp;
    if (d->O && packs(d, grp, wo, F)) add(r.wo, d->O, F, fp), r.ldo = fp;
    if (g.n && run) {
        const size_t nb = (g.o[g.n - 1].end + 255) / 256;
        pack_kernel<T><<<(unsigned)(nb < 8192 ? nb : 8192), 256, 0, st>>>(g);
    }
    return r;
}

// scratch of the forward and the backward pass: both use it for one product or sum after the other
size_t fwd_part(const cg_gated_dims* d, const cg_group* grp) {
    const int nz = grp_n(grp), e = (int)esize(d->dtype);
    const size_t M = d->rows / nz;
    if (M <= FEW_ROWS) return 0;
    const size_t p = part_bytes(M, 2 * (size_t)d->F, d->D, nz, 1, e, 2);
    const size_t q = d->O ? part_bytes(M, d->O, d->F, nz, 1, e, 1) : 0;
    return p > q ? p : q;
}
size_t bwd_part(const cg_gated_dims* d, const cg_group* grp) {
    const int nz = grp_n(grp), e = (int)esize(d->dtype);
    const size_t M = d->rows / nz, F = d->F, D = d->D, O = d->O;
    if (M <= FEW_ROWS) return 0;
    const size_t n[] = {O ? part_bytes(M, F, O, nz, 1, e, 1) : 0, part_bytes(M, D, 2 * F, nz, 1, e, 1), part_bytes(F, D, M, nz, 1, e, 1),
                        part_bytes(F, D, M, nz, 2, e, 1), O ? part_bytes(O, F, M, nz, 1, e, 1) : 0,
                        (size_t)2 * nz * strips_of(M) * (F > O ? F : O) * 4, (size_t)4 * nz * cg_div_up(M, 64) * F * 4};
    size_t most = 0;
    for (size_t v : n) most = v > most ? v : most;
    return up256(most);
}

// pitch of u, p, da, dv, and of h where it is not the result: rows on 16 bytes
inline int ldf_of(const cg_gated_dims* d) { return (int)pad8(d->F); }

template <typename T>
void fwd(const cg_gated_dims* d, const cg_group* grp, const T* x, const T* wg, const T* wv, const T* wo, const T* bg, const T* bv,
         const T* bo, T* h, T* kept, T* y, void* pack, float* part, hipStream_t st) {
    const int nz = grp_n(grp), ldf = ldf_of(d);
    const size_t M = d->rows / nz, gs = grp_stride(grp);
    const bool small = M <= FEW_ROWS;
    const Operands<T> op = operands<T>(d, grp, x, wg, wv, wo, pack, true, st);
    Gemm<T> g = {};
    g.nseg = g.nsel = 1;
    g.A[0] = op.x, g.az = M * op.ldx, g.lda = op.ldx;
    g.B[0] = op.wg, g.B[1] = op.wv, g.bz = gs, g.ldb = op.ldw;
    g.M = M, g.K = d->D, g.N = d->F, g.gate = d->gate;
    g.bias[0] = bg, g.bias[1] = bv, g.biasz = gs;
    g.o0 = h, g.o1 = kept, g.o2 = kept ? kept + d->rows * ldf : nullptr, g.low = kept ? (unsigned short*)(kept + 2 * d->rows * ldf) : nullptr,
     g.ld0 = d->O ? ldf : d->F, g.ldf = ldf;
    if (small) few<T, true, EPI_GATE_FWD>(g, nz, st);
    else gemm<T, true, true, EPI_GATE_FWD>(g, nz, part, st);
    if (!d->O) return;
    Gemm<T> o = {};
    o.nseg = o.nsel = 1;
    o.A[0] = h, o.az = M * ldf, o.lda = ldf;
    o.B[0] = op.wo, o.bz = gs, o.ldb = op.ldo;
    o.M = M, o.K = d->F, o.N = d->O;
    o.bias[0] = bo, o.biasz = gs;
    o.c[0] = y, o.cz = M * d->O;
    if (small) few<T, true, EPI_STORE>(o, nz, st);
    else gemm<T, true, true, EPI_STORE>(o, nz, part, st);
}

template <typename T>
void bwd(const cg_gated_dims* d, const cg_group* grp, const T* dy, const T* x, const T* wg, const T* wv, const T* wo, const T* h,
         const T* kept, T* dx, T* dwg, T* dwv, T* dwo, T* dbg, T* dbv, T* dbo, int acc, void* pack, T* da, T* dv, T* dyp,
         float* part, hipStream_t st) {
    const int nz = grp_n(grp), ldf = ldf_of(d);
    const size_t M = d->rows / nz, gs = grp_stride(grp), D = d->D, F = d->F, O = d->O;
    const bool small = M <= FEW_ROWS;
    const Operands<T> op = operands<T>(d, grp, x, wg, wv, wo, pack, false, st);
    const T *u = kept, *p = kept + d->rows * ldf;
    unsigned short* low = (unsigned short*)(kept + 2 * d->rows * ldf);
    size_t ldy = O;
    if (O && packs(d, grp, dy, O)) {
        Pack<T> g = {};
        g.n = 1, ldy = pad8(d->O);
        g.o[0].src = dy, g.o[0].dst = dyp, g.o[0].end = d->rows * (ldy / 8), g.o[0].cols = d->O, g.o[0].chunks = (int)(ldy / 8);
        const size_t nb = (g.o[0].end + 255) / 256;
        pack_kernel<T><<<(unsigned)(nb < 8192 ? nb : 8192), 256, 0, st>>>(g);
        dy = dyp;
    }
    if (dx || dwg || dwv || dbg || dbv) {
        if (O) {
            Gemm<T> g = {};
            g.nseg = g.nsel = 1;
            g.A[0] = dy, g.az = M * ldy, g.lda = ldy;
            g.B[0] = op.wo, g.bz = gs, g.ldb = op.ldo;
            g.M = M, g.K = O, g.N = d->F;
            g.o0 = da, g.o1 = dv, g.i0 = u, g.i1 = p, g.low = low, g.ldf = ldf;
            if ((dbg || dbv) && !small) g.sums = part;
            if (small) few<T, false, EPI_GATE_BWD>(g, nz, st);
            else gemm<T, true, false, EPI_GATE_BWD>(g, nz, part, st);
            if (g.sums && M) {
                ColSum<T> c = {{da, dv}, {dbg, dbv}, M, gs, d->F, ldf, g.strips, acc >> 3 & 3, part};
                colsum_join_kernel<T><<<dim3(cg_div_up(F, 32), 1, 2 * nz), 1024, 0, st>>>(c);
                dbg = dbv = nullptr;
            }
        } else if (M) {
            const size_t nb = ((size_t)d->rows * (ldf / 8) + 255) / 256;
            const unsigned blocks = (unsigned)(nb < 16384 ? nb : 16384);
            const GateBwd<T> g = {dy, u, p, low, da, dv, (size_t)d->rows, d->F, ldf};
            if (small) gate_bwd_kernel<T, float><<<blocks, 256, 0, st>>>(g);
            else gate_bwd_kernel<T, T><<<blocks, 256, 0, st>>>(g);
        }
    }
    if (dx) {
        Gemm<T> g = {};
        g.nseg = 2, g.nsel = 1;
        g.A[0] = da, g.A[1] = dv, g.az = M * ldf, g.lda = ldf;
        g.B[0] = op.wg, g.B[1] = op.wv, g.bz = gs, g.ldb = op.ldw;
        g.M = M, g.K = F, g.N = d->D;
        g.c[0] = dx, g.cz = M * D;
        if (small) few<T, false, EPI_STORE>(g, nz, st);
        else gemm<T, true, false, EPI_STORE>(g, nz, part, st);
    }
    if (small) {
        FewGrads<T> g = {};
        g.M = (int)M, g.gs = gs;
        int first = 0;
        auto add = [&](const T* p, int p32, size_t P, size_t ldp, const T* q, size_t Q, size_t ldq, T* dw, T* db, int bit) {
            if (!dw && !db) return;
            auto& o = g.o[g.n++];
            o.p = p, o.p32 = p32, o.q = q, o.dw = dw, o.db = db, o.P = (int)P, o.Q = (int)Q, o.ldp = (int)ldp, o.ldq = (int)ldq;
            o.tiles_q = dw ? (int)cg_div_up(Q, 64) : 1, o.first = first;
            o.add_w = acc >> bit & 1, o.add_b = acc >> (bit + 3) & 1;
            first += (int)cg_div_up(P, 64) * o.tiles_q;
        };
        add(da, 1, F, ldf, x, D, D, dwg, dbg, 0);
        add(dv, 1, F, ldf, x, D, D, dwv, dbv, 1);
        if (O) add(dy, sizeof(T) == 4, O, O, h, F, ldf, dwo, dbo, 2);
        if (g.n) few_grads_kernel<T><<<dim3(first, nz), 256, 0, st>>>(g);
        return;
    }
    auto wgrad = [&](const T* p0, const T* p1, size_t P, size_t ldp, const T* q, size_t Q, size_t ldq, T* dw0, T* dw1, int accumulate) {
        if (!dw0 && !dw1) return;
        Gemm<T> g = {};
        g.nseg = 1, g.nsel = dw0 && dw1 ? 2 : 1;
        g.A[0] = dw0 ? p0 : p1, g.A[1] = p1, g.az = M * ldp, g.lda = ldp;
        g.B[0] = q, g.bz = M * ldq, g.ldb = ldq;
        g.M = P, g.K = M, g.N = (int)Q;
        g.c[0] = dw0 ? dw0 : dw1, g.c[1] = dw1, g.cz = gs, g.accumulate = dw0 ? accumulate : accumulate >> 1;
        gemm<T, false, false, EPI_STORE>(g, nz, part, st);
    };
    wgrad(da, dv, F, ldf, op.x, D, op.ldx, dwg, dwv, acc & 3);
    if (O) wgrad(dy, nullptr, O, ldy, h, F, ldf, dwo, nullptr, acc >> 2 & 1);
    auto bgrad = [&](const T* p0, const T* p1, int C, size_t ld, T* db0, T* db1, int accumulate) {
        if (!db0 && !db1) return;
        ColSum<T> g = {{db0 ? p0 : nullptr, db1 ? p1 : nullptr}, {db0, db1}, M, gs, C, (int)ld, strips_of(M), accumulate, part};
        colsum_part_kernel<T><<<dim3(cg_div_up(C, 64 * CgT<T>::N), g.strips, 2 * nz), 256, 0, st>>>(g);
        colsum_join_kernel<T><<<dim3(cg_div_up(C, 32), 1, 2 * nz), 1024, 0, st>>>(g);
    };
    bgrad(da, dv, d->F, ldf, dbg, dbv, acc >> 3 & 3);
    if (O) bgrad(dy, nullptr, d->O, ldy, dbo, nullptr, acc >> 5 & 1);
}

}  // namespace

extern "C" size_t cg_gated_ff_pack_bytes(const cg_gated_dims* d, const cg_group* grp, const void* x, const void* wg, const void* wv,
                                         const void* wo) {
    return dims_ok(d, grp) ? pack_bytes(d, grp, x, wg, wv, wo) : 0;
}

extern "C" size_t cg_gated_ff_fwd_workspace(const cg_gated_dims* d, const cg_group* grp) { return dims_ok(d, grp) ? fwd_part(d, grp) : 0; }

extern "C" int cg_gated_ff_fwd(const cg_gated_dims* d, const cg_group* grp, const void* x, const void* wg, const void* wv, const void* wo,
                               const void* bg, const void* bv, const void* bo, void* h, void* kept, void* y, void* pack, void* ws,
                               size_t ws_bytes, cg_stream_t stream) {
    CG_CHECK_ARG(dims_ok(d, grp) && wg && wv && (!d->O || wo) && (!d->rows || (x && h && (!d->O || y))) &&
                     aligned16(d->O ? h : nullptr, kept, pack, ws),
                 "cg_gated_ff_fwd: bad args");
    const size_t need = fwd_part(d, grp);
    if (ws_bytes < need || (!ws && need) || (!pack && pack_bytes(d, grp, x, wg, wv, wo)))
        return cg_set_error(CG_ERR_WORKSPACE, "cg_gated_ff_fwd: workspace too small");
    if (!d->rows) return CG_OK;
    CG_DISPATCH_DT(d->dtype, T, (fwd<T>(d, grp, (const T*)x, (const T*)wg, (const T*)wv, (const T*)wo, (const T*)bg, (const T*)bv,
                                        (const T*)bo, (T*)h, (T*)kept, (T*)y, pack, (float*)ws, cg_s(stream))));
    CG_LAUNCH_CHECK("cg_gated_ff_fwd");
    return CG_OK;
}

// da or dv: fp32 for few rows
static size_t bwd_hidden(const cg_gated_dims* d, const cg_group* grp) {
    return up256((size_t)d->rows * ldf_of(d) * (d->rows / grp_n(grp) <= FEW_ROWS ? 4 : esize(d->dtype)));
}
static size_t bwd_dy(const cg_gated_dims* d) { return d->dtype == CG_DT_F32 ? 0 : up256((size_t)d->rows * pad8(d->O) * 2); }

extern "C" size_t cg_gated_ff_bwd_workspace(const cg_gated_dims* d, const cg_group* grp) {
    return dims_ok(d, grp) ? 2 * bwd_hidden(d, grp) + bwd_dy(d) + bwd_part(d, grp) : 0;
}

extern "C" int cg_gated_ff_bwd(const cg_gated_dims* d, const cg_group* grp, const void* dy, const void* x, const void* wg,
                               const void* wv, const void* wo, const void* h, const void* kept, void* dx, void* dwg,
                               void* dwv, void* dwo, void* dbg, void* dbv, void* dbo, int accumulate, const void* pack, void* ws,
                               size_t ws_bytes, cg_stream_t stream) {
    CG_CHECK_ARG(dims_ok(d, grp) && wg && wv && (!d->O || wo) && (!d->rows || (dy && x && kept && (!d->O || h))) &&
                     aligned16(d->O ? h : nullptr, kept, pack, ws),
                 "cg_gated_ff_bwd: bad args");
    const size_t need = cg_gated_ff_bwd_workspace(d, grp);
    if (ws_bytes < need || (!ws && need) || (!pack && pack_bytes(d, grp, x, wg, wv, wo)))
        return cg_set_error(CG_ERR_WORKSPACE, "cg_gated_ff_bwd: workspace too small");
    CG_DISPATCH_DT(d->dtype, T, {
        char* w = (char*)ws;
        T *da = (T*)w, *dv = (T*)(w + bwd_hidden(d, grp)), *dyp = (T*)(w + 2 * bwd_hidden(d, grp));
        float* part = (float*)(w + 2 * bwd_hidden(d, grp) + bwd_dy(d));
        bwd<T>(d, grp, (const T*)dy, (const T*)x, (const T*)wg, (const T*)wv, (const T*)wo, (const T*)h, (const T*)kept, (T*)dx,
               (T*)dwg, (T*)dwv, (T*)dwo, (T*)dbg, (T*)dbv, (T*)dbo, accumulate, (void*)pack, da, dv, dyp, part, cg_s(stream));
    });
    CG_LAUNCH_CHECK("cg_gated_ff_bwd");
    return CG_OK;
}
