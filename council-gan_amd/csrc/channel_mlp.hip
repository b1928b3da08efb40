// channel_norm and dropout: the memory-bound operators of the channel MLP (gfx950).
#include "cg_vec.h"

namespace {

inline bool dt_ok(int dt) { return dt == CG_DT_F32 || dt == CG_DT_F16 || dt == CG_DT_BF16; }
inline int grp_n(const cg_group* g) { return g && g->n > 1 ? g->n : 1; }
inline size_t grp_stride(const cg_group* g) { return g && g->n > 1 ? (size_t)g->stride : 0; }

// ------------------------------------------------------------------------------------------
// channel_norm: y = (x - mean) rstd w + b per row, rstd = 1 / sqrt(var + eps), biased variance.
// One row per block; the row is read for the mean, again for the centred squares (no cancellation) and again for the output.
// ------------------------------------------------------------------------------------------
constexpr int NT = 256;

__device__ __forceinline__ float block_sum(float v, float* sm) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) s += sm[i];
    return s;
}

template <typename T, typename W>
__global__ __launch_bounds__(NT) void channel_norm_fwd_kernel(const T* __restrict__ x, const W* __restrict__ w, const W* __restrict__ b,
                                                              T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                                                              size_t rows, int C, float eps, size_t gstride) {
    __shared__ float sm[NT / 64];
    constexpr int N = CgT<T>::N;
    w += blockIdx.y * gstride;
    if (b) b += blockIdx.y * gstride;
    for (size_t i = blockIdx.x; i < rows; i += gridDim.x) {
        const size_t r = blockIdx.y * rows + i;
        const T* xr = x + r * C;
        float s = 0.f, q = 0.f, v[N], wv[N], bv[N];
        for (int c = threadIdx.x * N; c < C; c += NT * N) {
            cg_load<T>(xr + c, C - c, v);
#pragma unroll
            for (int k = 0; k < N; ++k) s += v[k];
        }
        const float m = block_sum(s, sm) / (float)C;
        for (int c = threadIdx.x * N; c < C; c += NT * N) {
            cg_load<T>(xr + c, C - c, v);
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (c + k < C) q += (v[k] - m) * (v[k] - m);
        }
        const float rs = 1.f / sqrtf(block_sum(q, sm) / (float)C + eps);
        for (int c = threadIdx.x * N; c < C; c += NT * N) {
            cg_load<T>(xr + c, C - c, v);
            cg_load<W, N>(w + c, C - c, wv);
            if (b) cg_load<W, N>(b + c, C - c, bv);
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = (v[k] - m) * rs * wv[k] + (b ? bv[k] : 0.f);
            cg_store<T>(y + r * C + c, C - c, v);
        }
        if (threadIdx.x == 0 && mean) {
            mean[r] = m;
            rstd[r] = rs;
        }
    }
}

// dx = rstd (g - mean(g) - xh mean(g xh)), g = dy w
template <typename T, typename W>
__global__ __launch_bounds__(NT) void channel_norm_dx_kernel(const T* __restrict__ dy, const T* __restrict__ x, const W* __restrict__ w,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd,
                                                             T* __restrict__ dx, size_t rows, int C, size_t gstride) {
    __shared__ float sm[NT / 64];
    constexpr int N = CgT<T>::N;
    w += blockIdx.y * gstride;
    for (size_t i = blockIdx.x; i < rows; i += gridDim.x) {
        const size_t r = blockIdx.y * rows + i;
        const float m = mean[r], rs = rstd[r];
        float s1 = 0.f, s2 = 0.f, v[N], d[N], wv[N];
        for (int c = threadIdx.x * N; c < C; c += NT * N) {
            cg_load<T>(x + r * C + c, C - c, v);
            cg_load<T>(dy + r * C + c, C - c, d);
            cg_load<W, N>(w + c, C - c, wv);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const float g = d[k] * wv[k];
                s1 += g;
                s2 += g * ((v[k] - m) * rs);
            }
        }
        s1 = block_sum(s1, sm) / (float)C;
        s2 = block_sum(s2, sm) / (float)C;
        for (int c = threadIdx.x * N; c < C; c += NT * N) {
            cg_load<T>(x + r * C + c, C - c, v);
            cg_load<T>(dy + r * C + c, C - c, d);
            cg_load<W, N>(w + c, C - c, wv);
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = rs * (d[k] * wv[k] - s1 - (v[k] - m) * rs * s2);
            cg_store<T>(dx + r * C + c, C - c, v);
        }
    }
}

// partial sums over a strip of rows: part[strip][0][c] = sum dy xh, part[strip][1][c] = sum dy
template <typename T>
__global__ __launch_bounds__(NT) void channel_norm_dw_part_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                  const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                  float* __restrict__ part, size_t rows, int C) {
    const int c = blockIdx.x * NT + threadIdx.x;
    if (c >= C) return;
    const size_t strips = gridDim.z, per = (rows + strips - 1) / strips;
    const size_t r0 = blockIdx.z * per, r1 = r0 + per < rows ? r0 + per : rows;
    float sw = 0.f, sb = 0.f;
    for (size_t i = r0; i < r1; ++i) {
        const size_t r = blockIdx.y * rows + i;
        const float d = (float)dy[r * C + c];
        sw += d * (((float)x[r * C + c] - mean[r]) * rstd[r]);
        sb += d;
    }
    float* p = part + ((size_t)blockIdx.y * strips + blockIdx.z) * 2 * C;
    p[c] = sw;
    p[C + c] = sb;
}

template <typename W>
__global__ __launch_bounds__(NT) void channel_norm_dw_sum_kernel(const float* __restrict__ part, W* __restrict__ dw, W* __restrict__ db,
                                                                 int strips, int C, int accumulate, size_t gstride) {
    const int c = blockIdx.x * NT + threadIdx.x;
    if (c >= 2 * C) return;
    W* out = c < C ? dw : db;
    if (!out) return;
    float s = 0.f;
    for (int i = 0; i < strips; ++i) s += part[((size_t)blockIdx.y * strips + i) * 2 * C + c];
    out += blockIdx.y * gstride + (c < C ? c : c - C);
    *out = (W)(accumulate ? (float)*out + s : s);
}

inline int norm_strips(size_t rows) { return (int)(rows < 1 ? 1 : (rows + 63) / 64 > 256 ? 256 : (rows + 63) / 64); }

// ------------------------------------------------------------------------------------------
// dropout.  Philox4x32-10 (J. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011): a bijection of a 128-bit counter
// under a 64-bit key, so the draw of an element is a function of (key, position) alone and the backward pass computes the mask again
// instead of reading one.  A block of 8 elements shares a counter: 128 bits = 8 draws of 16.
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)c[0] * 0xD2511F53u, p1 = (uint64_t)c[2] * 0xCD9E8D57u;
        const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c[1] ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
        c[1] = (uint32_t)p1;
        c[3] = (uint32_t)p0;
        c[0] = n0;
        c[2] = n2;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

template <typename T, bool RES>
__global__ __launch_bounds__(NT) void dropout_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y, size_t n,
                                                     uint32_t threshold, float scale, const uint64_t* __restrict__ key) {
    const uint64_t seed = key[0], step = key[1];
    const size_t blocks = (n + 7) / 8;
    for (size_t b = (size_t)blockIdx.x * NT + threadIdx.x; b < blocks; b += (size_t)gridDim.x * NT) {
        uint32_t c[4] = {(uint32_t)b, (uint32_t)(b >> 32), (uint32_t)step, (uint32_t)(step >> 32)};
        const size_t e = b * 8;
        const int left = n - e < 8 ? (int)(n - e) : 8;
        float v[8], r[8];
        cg_load<T, 8>(x + e, left, v);
        if (RES) cg_load<T, 8>(res + e, left, r);
        philox(c, (uint32_t)seed, (uint32_t)(seed >> 32));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t d = (i & 1) ? c[i >> 1] >> 16 : c[i >> 1] & 0xffffu;
            v[i] = d >= threshold ? v[i] * scale : 0.f;      // a dropped infinity or NaN is dropped
            if (RES) v[i] = r[i] + v[i];
        }
        cg_store<T, 8>(y + e, left, v);
    }
}

// key = state; state's step + 1: one thread, on the caller's stream, so captured graphs draw anew on every replay
__global__ void dropout_key_kernel(uint64_t* state, uint64_t* key) {
    const uint64_t s = state[0], t = state[1];
    key[0] = s;
    key[1] = t;
    state[1] = t + 1;
}

}  // namespace

extern "C" int cg_channel_norm_fwd(const cg_group* grp, const void* x, const void* weight, const void* bias, void* y, float* mean,
                                   float* rstd, size_t rows, int C, int dtype, int wdtype, float eps, cg_stream_t stream) {
    CG_CHECK_ARG((!rows || (x && y)) && weight && C > 0 && dt_ok(dtype) && (wdtype == dtype || wdtype == CG_DT_F32) && eps >= 0.f &&
                     !mean == !rstd && rows % grp_n(grp) == 0, "cg_channel_norm_fwd: bad args");
    if (!rows) return CG_OK;
    rows /= grp_n(grp);
    const dim3 grid((unsigned)(rows < 65536 ? rows : 65536), grp_n(grp));
    CG_DISPATCH_DT(dtype, T, CG_DISPATCH_DT(wdtype, W, {
        if constexpr (std::is_same_v<W, T> || std::is_same_v<W, float>)
            channel_norm_fwd_kernel<T, W><<<grid, NT, 0, cg_s(stream)>>>((const T*)x, (const W*)weight, (const W*)bias, (T*)y, mean,
                                                                         rstd, rows, C, eps, grp_stride(grp));
    }));
    CG_LAUNCH_CHECK("cg_channel_norm_fwd");
    return CG_OK;
}

extern "C" size_t cg_channel_norm_bwd_workspace(const cg_group* grp, size_t rows, int C) {
    return (size_t)grp_n(grp) * norm_strips(rows / grp_n(grp)) * 2 * (size_t)(C > 0 ? C : 0) * sizeof(float);
}

extern "C" int cg_channel_norm_bwd(const cg_group* grp, const void* dy, const void* x, const void* weight, const float* mean,
                                   const float* rstd, void* dx, void* dweight, void* dbias, int accumulate, size_t rows, int C,
                                   int dtype, int wdtype, void* ws, size_t ws_bytes, cg_stream_t stream) {
    CG_CHECK_ARG((!rows || (dy && x && mean && rstd)) && weight && C > 0 && dt_ok(dtype) && (wdtype == dtype || wdtype == CG_DT_F32) &&
                     rows % grp_n(grp) == 0, "cg_channel_norm_bwd: bad args");
    const int n = grp_n(grp);
    if ((dweight || dbias) && (!ws || ws_bytes < cg_channel_norm_bwd_workspace(grp, rows, C)))
        return cg_set_error(CG_ERR_WORKSPACE, "cg_channel_norm_bwd: workspace too small");
    rows /= n;
    if (dx && rows) {
        const dim3 grid((unsigned)(rows < 65536 ? rows : 65536), n);
        CG_DISPATCH_DT(dtype, T, CG_DISPATCH_DT(wdtype, W, {
            if constexpr (std::is_same_v<W, T> || std::is_same_v<W, float>)
                channel_norm_dx_kernel<T, W><<<grid, NT, 0, cg_s(stream)>>>((const T*)dy, (const T*)x, (const W*)weight, mean, rstd,
                                                                            (T*)dx, rows, C, grp_stride(grp));
        }));
        CG_LAUNCH_CHECK("cg_channel_norm_bwd");
    }
    if (dweight || dbias) {
        const int strips = norm_strips(rows);
        CG_DISPATCH_DT(dtype, T, (channel_norm_dw_part_kernel<T><<<dim3(cg_div_up(C, NT), n, strips), NT, 0, cg_s(stream)>>>(
                                     (const T*)dy, (const T*)x, mean, rstd, (float*)ws, rows, C)));
        CG_DISPATCH_DT(wdtype, W, (channel_norm_dw_sum_kernel<W><<<dim3(cg_div_up(2 * (size_t)C, NT), n), NT, 0, cg_s(stream)>>>(
                                      (const float*)ws, (W*)dweight, (W*)dbias, strips, C, accumulate, grp_stride(grp))));
        CG_LAUNCH_CHECK("cg_channel_norm_bwd");
    }
    return CG_OK;
}

extern "C" int cg_dropout_key(void* state, void* key, cg_stream_t stream) {
    CG_CHECK_ARG(state && key && state != key, "cg_dropout_key: bad args");
    dropout_key_kernel<<<1, 1, 0, cg_s(stream)>>>((uint64_t*)state, (uint64_t*)key);
    CG_LAUNCH_CHECK("cg_dropout_key");
    return CG_OK;
}

extern "C" int cg_dropout(const void* x, const void* residual, void* y, size_t n, int threshold, const void* key, int dtype,
                          cg_stream_t stream) {
    CG_CHECK_ARG((!n || (x && y)) && key && dt_ok(dtype) && threshold >= 0 && threshold < 65536, "cg_dropout: bad args");
    if (!n) return CG_OK;
    const float scale = 65536.f / (float)(65536 - threshold);
    const size_t nb = ((n + 7) / 8 + NT - 1) / NT;
    const unsigned grid = (unsigned)(nb < 65536 ? nb : 65536);
    CG_DISPATCH_DT(dtype, T, {
        if (residual)
            dropout_kernel<T, true><<<grid, NT, 0, cg_s(stream)>>>((const T*)x, (const T*)residual, (T*)y, n, threshold, scale,
                                                                   (const uint64_t*)key);
        else
            dropout_kernel<T, false><<<grid, NT, 0, cg_s(stream)>>>((const T*)x, nullptr, (T*)y, n, threshold, scale,
                                                                    (const uint64_t*)key);
    });
    CG_LAUNCH_CHECK("cg_dropout");
    return CG_OK;
}
