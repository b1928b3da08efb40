// channel_norm and dropout: the memory-bound operators of the channel MLP (gfx950).
#include "cg_vec.h"
#include <type_traits>

namespace {

inline bool dt_ok(int dt) { return dt == CG_DT_F32 || dt == CG_DT_F16 || dt == CG_DT_BF16; }
inline int grp_n(const cg_group* g) { return g && g->n > 1 ? g->n : 1; }
inline size_t grp_stride(const cg_group* g) { return g && g->n > 1 ? (size_t)g->stride : 0; }

// ------------------------------------------------------------------------------------------
// channel_norm: y = (x - mean) rstd w + b per row, rstd = 1 / sqrt(var + eps), biased variance.
//
// A row is read once and stays in registers: TPR threads hold NV chunks of W elements each, the mean and then the centred squares
// (no cancellation) are summed across them, and the output leaves from the same registers.  The backward pass keeps x and dy of a row
// in the same way and adds dy xh and dy to sums of its own columns over all the rows that it visits, so that dx, dweight and dbias cost
// one reading of x and dy; the blocks' sums are then joined in block order (the same result on every run).
// Rows of any width: the last chunk of a row is moved back to end with the row; the elements that it shares with its neighbour are
// masked out of the sums, and both lanes store the same value for them.
// Bound by memory: 65536 x 256 fp32 forward 22 us (6.0 TB/s), backward 35 us (5.8 TB/s) and 4 us to join; 16384 x 4096 bf16 46 us
// (5.9 TB/s), 85 us (4.7 TB/s) and 5 us.
// ------------------------------------------------------------------------------------------
constexpr int NT = 256;
constexpr int MAX_CHANNELS = 1 << 29;       // column indices, also of both sums next to each other (2 C), are ints

// Every kernel of this file takes its arguments as one struct: the runtime looks up each pointer among a launch's arguments, 4 to 7 us
// for the forward pass's seven pointers when the launching thread changes (the backward pass runs on autograd's own).
template <typename T, typename W> struct Norm {
    const T *dy, *x;
    const W *w, *b;
    T *y, *dx;
    float *mean, *rstd, *part;
    W *dw, *db;
    size_t rows, gstride;
    int C, accumulate, blocks;
    float eps;
};

// sums over the TPR threads of a row
template <int TPR, int K> __device__ __forceinline__ void row_sum(float (&v)[K], float* sm) {
#pragma unroll
    for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], o, 64);
    if constexpr (TPR > 64) {
        constexpr int NWV = TPR / 64;
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; ++k) sm[k * NWV + (threadIdx.x >> 6)] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            v[k] = 0.f;
#pragma unroll
            for (int i = 0; i < NWV; ++i) v[k] += sm[k * NWV + i];
        }
    }
}

// the columns of one thread: chunk j starts at at[j], its elements below first[j] belong to the neighbour (or to nobody)
template <typename T, int TPR, int NV> struct Columns {
    static constexpr int W = CgT<T>::N;
    int at[NV], first[NV];
    __device__ __forceinline__ Columns(int t, int C) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * TPR + t) * W;
            at[j] = c < C - W ? c : C - W;
            first[j] = c - at[j];
        }
    }
    __device__ __forceinline__ bool mine(int j, int e) const { return e >= first[j]; }
    __device__ __forceinline__ bool any(int j) const { return first[j] < W; }
    __device__ __forceinline__ bool shares(int j) const { return first[j] > 0 && first[j] < W; }
};

template <typename T, typename W_, int TPR, int NV>
__global__ __launch_bounds__(NT) void channel_norm_fwd_kernel(Norm<T, W_> n) {
    const T* __restrict__ x = n.x;
    T* __restrict__ y = n.y;
    const W_ *w = n.w + blockIdx.y * n.gstride, *b = n.b ? n.b + blockIdx.y * n.gstride : nullptr;
    const size_t rows = n.rows;
    const int C = n.C;
    constexpr int W = CgT<T>::N, RPB = NT / TPR;
    typedef typename CgT<T>::V V;
    __shared__ float sm[NT / 64];
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    const Columns<T, TPR, NV> col(t, C);
    const float inv = 1.f / (float)C;
    const size_t row0 = blockIdx.y * rows, step = (size_t)gridDim.x * RPB;
    V nx[NV];
    auto fetch = [&](size_t i) {
        const T* xr = x + (row0 + (i < rows ? i : rows - 1)) * C;
#pragma unroll
        for (int j = 0; j < NV; ++j) nx[j] = *(const V*)(xr + col.at[j]);
    };
    fetch((size_t)blockIdx.x * RPB + g);
    float wv[NV][W], bv[NV][W];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        cg_load<W_, W>(w + col.at[j], W, wv[j]);
        if (b) cg_load<W_, W>(b + col.at[j], W, bv[j]);
    }
    for (size_t i0 = (size_t)blockIdx.x * RPB; i0 < rows; i0 += step) {      // the whole block, so that its barriers meet
        const size_t i = i0 + g;
        float v[NV][W], s[1] = {0.f}, q[1] = {0.f};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                v[j][e] = (float)nx[j][e];
                s[0] += col.mine(j, e) ? v[j][e] : 0.f;
            }
        if (i0 + step < rows) fetch(i + step);
        row_sum<TPR, 1>(s, sm);
        const float m = s[0] / (float)C;      // the mean of equal values is that value
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                v[j][e] -= m;
                q[0] += col.mine(j, e) ? v[j][e] * v[j][e] : 0.f;
            }
        row_sum<TPR, 1>(q, sm);
        const float rs = 1.f / sqrtf(q[0] * inv + n.eps);
        if (i < rows) {
            const size_t r = row0 + i;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
#pragma unroll
                for (int e = 0; e < W; ++e) v[j][e] = v[j][e] * rs * wv[j][e] + (b ? bv[j][e] : 0.f);
                if (col.any(j)) cg_store<T>(y + r * C + col.at[j], W, v[j]);
            }
            if (t == 0 && n.mean) {
                n.mean[r] = m;
                n.rstd[r] = rs;
            }
        }
    }
}

// dx = rstd (g - mean(g) - xh mean(g xh)), g = dy w; part[block][0][c] = sum dy xh, part[block][1][c] = sum dy over the block's rows
// (written to dw / db themselves when one block sees all rows)
template <typename T, typename W_, int TPR, int NV>
__global__ __launch_bounds__(NT) void channel_norm_bwd_kernel(Norm<T, W_> n) {
    const T* __restrict__ dy = n.dy;
    const T* __restrict__ x = n.x;
    T* __restrict__ dx = n.dx;
    const W_* w = n.w + blockIdx.y * n.gstride;
    W_ *dw = n.dw, *db = n.db;
    const size_t rows = n.rows, gstride = n.gstride;
    const int C = n.C, accumulate = n.accumulate;
    constexpr int W = CgT<T>::N, RPB = NT / TPR;
    typedef typename CgT<T>::V V;
    __shared__ float sm[2 * NT / 64];
    __shared__ float cols[RPB > 1 ? 2 * TPR * NV * W : 1];
    const int t = threadIdx.x % TPR, g = threadIdx.x / TPR;
    const Columns<T, TPR, NV> col(t, C);
    const float inv = 1.f / (float)C;
    const size_t row0 = blockIdx.y * rows, step = (size_t)gridDim.x * RPB;
    V nx[NV], nd[NV];
    float nm = 0.f, nr = 0.f;
    auto fetch = [&](size_t i) {
        const size_t r = row0 + (i < rows ? i : rows - 1);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            nx[j] = *(const V*)(x + r * C + col.at[j]);
            nd[j] = *(const V*)(dy + r * C + col.at[j]);
        }
        nm = n.mean[r];
        nr = n.rstd[r];
    };
    if (rows) fetch((size_t)blockIdx.x * RPB + g);
    // dy goes into the sums with zeros in the elements that are not the thread's own (a mask on the raw chunk: the sums themselves take no
    // selects, which were half of the loop's instructions), and as it is into the dx that a shared chunk stores
    typedef unsigned Bits __attribute__((ext_vector_type(4)));
    float wv[NV][W], sw[NV][W] = {}, sb[NV][W] = {};
    Bits own[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        cg_load<W_, W>(w + col.at[j], W, wv[j]);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            own[j][k] = W == 4 ? (col.mine(j, k) ? ~0u : 0u) : (col.mine(j, 2 * k) ? 0xffffu : 0u) | (col.mine(j, 2 * k + 1) ? 0xffff0000u : 0u);
    }
    for (size_t i0 = (size_t)blockIdx.x * RPB; i0 < rows; i0 += step) {
        const size_t i = i0 + g;
        const bool live = i < rows;
        const float m = nm, rs = nr;
        float v[NV][W], d[NV][W], s[2] = {0.f, 0.f};
        V raw[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            raw[j] = nd[j];
            if (!live) raw[j] = V{};
            const V md = __builtin_bit_cast(V, __builtin_bit_cast(Bits, raw[j]) & own[j]);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                v[j][e] = ((float)nx[j][e] - m) * rs;
                d[j][e] = (float)md[e];
                sw[j][e] += d[j][e] * v[j][e];
                sb[j][e] += d[j][e];
                d[j][e] *= wv[j][e];
                s[0] += d[j][e];
                s[1] += d[j][e] * v[j][e];
            }
        }
        if (i0 + step < rows) fetch(i + step);
        if (dx) {
            row_sum<TPR, 2>(s, sm);
            const float s1 = s[0] * inv, s2 = s[1] * inv;
            if (live)
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    if (col.shares(j))
#pragma unroll
                        for (int e = 0; e < W; ++e) d[j][e] = (float)raw[j][e] * wv[j][e];
#pragma unroll
                    for (int e = 0; e < W; ++e) d[j][e] = rs * (d[j][e] - s1 - v[j][e] * s2);
                    if (col.any(j)) cg_store<T>(dx + (row0 + i) * C + col.at[j], W, d[j]);
                }
        }
    }
    if (!n.part && !dw && !db) return;
    // the row groups of the block, one after the other
    if constexpr (RPB > 1) {
        for (int k = 1; k < RPB; ++k) {
            __syncthreads();
            if (g == k)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        cols[((j * W + e) * 2) * TPR + t] = sw[j][e];
                        cols[((j * W + e) * 2 + 1) * TPR + t] = sb[j][e];
                    }
            __syncthreads();
            if (g == 0)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        sw[j][e] += cols[((j * W + e) * 2) * TPR + t];
                        sb[j][e] += cols[((j * W + e) * 2 + 1) * TPR + t];
                    }
        }
        if (g) return;
    }
    float* p = n.part ? n.part + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * C : nullptr;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const int c = col.at[j] + e;
            if (!col.mine(j, e)) continue;
            if (p) {
                p[c] = sw[j][e];
                p[C + c] = sb[j][e];
            } else {
                if (dw) dw[blockIdx.y * gstride + c] = (W_)(accumulate & 1 ? (float)dw[blockIdx.y * gstride + c] + sw[j][e] : sw[j][e]);
                if (db) db[blockIdx.y * gstride + c] = (W_)(accumulate & 2 ? (float)db[blockIdx.y * gstride + c] + sb[j][e] : sb[j][e]);
            }
        }
}

// joins the blocks' sums: 32 columns a block, 32 threads a column, each with its share of the blocks in order
template <typename T, typename W> __global__ __launch_bounds__(1024) void channel_norm_join_kernel(Norm<T, W> n) {
    const int C = n.C, blocks = n.blocks;
    __shared__ float sm[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    const float* __restrict__ part = n.part + (size_t)blockIdx.y * blocks * 2 * C;
    float s = 0.f;
    if (c < 2 * C)
#pragma unroll 8
        for (int i = k; i < blocks; i += 32) s += part[(size_t)i * 2 * C + c];
    sm[k][threadIdx.x & 31] = s;
    __syncthreads();
    if (k || c >= 2 * C) return;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sm[i][threadIdx.x];
    W* out = c < C ? n.dw : n.db;
    if (!out) return;
    out += blockIdx.y * n.gstride + (c < C ? c : c - C);
    *out = (W)(n.accumulate & (c < C ? 1 : 2) ? (float)*out + s : s);
}

// Rows that do not fit a block's registers, or are shorter than one chunk: one row per block, read again for every sum.
__device__ __forceinline__ float block_sum(float v, float* sm) {
    float a[1] = {v};
    row_sum<NT, 1>(a, sm);
    return a[0];
}

template <typename T, typename W>
__global__ __launch_bounds__(NT) void channel_norm_long_fwd_kernel(Norm<T, W> n) {
    __shared__ float sm[NT / 64];
    constexpr int N = CgT<T>::N;
    const W *w = n.w + blockIdx.y * n.gstride, *b = n.b ? n.b + blockIdx.y * n.gstride : nullptr;
    const int C = n.C;
    for (size_t i = blockIdx.x; i < n.rows; i += gridDim.x) {
        const size_t r = blockIdx.y * n.rows + i;
        const T* xr = n.x + r * C;
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
        const float rs = 1.f / sqrtf(block_sum(q, sm) / (float)C + n.eps);
        for (int c = threadIdx.x * N; c < C; c += NT * N) {
            cg_load<T>(xr + c, C - c, v);
            cg_load<W, N>(w + c, C - c, wv);
            if (b) cg_load<W, N>(b + c, C - c, bv);
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = (v[k] - m) * rs * wv[k] + (b ? bv[k] : 0.f);
            cg_store<T>(n.y + r * C + c, C - c, v);
        }
        if (threadIdx.x == 0 && n.mean) {
            n.mean[r] = m;
            n.rstd[r] = rs;
        }
    }
}

template <typename T, typename W> __global__ __launch_bounds__(NT) void channel_norm_long_dx_kernel(Norm<T, W> n) {
    __shared__ float sm[NT / 64];
    constexpr int N = CgT<T>::N;
    const T* __restrict__ dy = n.dy;
    const T* __restrict__ x = n.x;
    const W* w = n.w + blockIdx.y * n.gstride;
    const size_t rows = n.rows;
    const int C = n.C;
    for (size_t i = blockIdx.x; i < rows; i += gridDim.x) {
        const size_t r = blockIdx.y * rows + i;
        const float m = n.mean[r], rs = n.rstd[r];
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
            cg_store<T>(n.dx + r * C + c, C - c, v);
        }
    }
}

template <typename T, typename W> __global__ __launch_bounds__(NT) void channel_norm_long_dw_kernel(Norm<T, W> n) {
    const int C = n.C, c = blockIdx.x * NT + threadIdx.x;
    if (c >= C) return;
    const size_t strips = gridDim.z, per = (n.rows + strips - 1) / strips;
    const size_t r0 = blockIdx.z * per, r1 = r0 + per < n.rows ? r0 + per : n.rows;
    float sw = 0.f, sb = 0.f;
    for (size_t i = r0; i < r1; ++i) {
        const size_t r = blockIdx.y * n.rows + i;
        const float d = (float)n.dy[r * C + c];
        sw += d * (((float)n.x[r * C + c] - n.mean[r]) * n.rstd[r]);
        sb += d;
    }
    float* p = n.part + ((size_t)blockIdx.y * strips + blockIdx.z) * 2 * C;
    p[c] = sw;
    p[C + c] = sb;
}

// Which kernel a row width gets (both passes): the narrowest group of threads that holds the row in at most 4 chunks a thread -- short
// rows share a wave, since a wave's sum needs no barrier.
struct NormKind { int tpr, nv; };       // tpr 0: the long-row kernels
NormKind norm_kind(int C, int esz) {
    const int W = 16 / esz;
    if (C < W) return {0, 0};
    const int ch = (C + W - 1) / W;
    if (ch <= 16) return {16, 1};
    if (ch <= 32) return {32, 1};
    if (ch <= 64) return {64, 1};
    if (ch <= 128) return {64, 2};
    if (ch <= 256) return {64, 4};
    if (ch <= 512) return {256, 2};
    if (ch <= 1024) return {256, 4};
    return {0, 0};
}
// blocks of the backward pass = partial sums to join: at least 4 rows for every row group, and no more blocks than the chip holds at once
// (the more chunks a thread has, the fewer): 16384 x 8192 bf16, 4 chunks, 156 us with 256 blocks, 171 with 512, 195 with 1024; 40000 x 2048
// fp32, 2 chunks, 180 with 512, 259 with 256, 196 with 1024; 65536 x 256 fp32, 1 chunk, both passes 64 with 1024, 86 with 256.
int norm_blocks(size_t rows, int C, int esz) {
    const NormKind k = norm_kind(C, esz);
    if (!k.tpr) return (int)(rows < 1 ? 1 : (rows + 63) / 64 > 256 ? 256 : (rows + 63) / 64);
    const size_t b = (rows + NT / k.tpr * 4 - 1) / (NT / k.tpr * 4);
    const size_t most = 1024 / k.nv;
    return (int)(b < 1 ? 1 : b > most ? most : b);
}

template <typename T, typename W, int TPR, int NV> void norm_fwd(const Norm<T, W>& g, int members, hipStream_t st) {
    const size_t nb = (g.rows + NT / TPR - 1) / (NT / TPR);
    channel_norm_fwd_kernel<T, W, TPR, NV><<<dim3((unsigned)(nb < 2048 ? nb : 2048), members), NT, 0, st>>>(g);
}
template <typename T, typename W, int TPR, int NV> void norm_bwd(const Norm<T, W>& g, int members, hipStream_t st) {
    channel_norm_bwd_kernel<T, W, TPR, NV><<<dim3(g.blocks, members), NT, 0, st>>>(g);
}
#define CG_NORM_KIND(kind, F, ...)                             \
    do {                                                       \
        if ((kind).tpr == 16) F<T, W, 16, 1>(__VA_ARGS__);     \
        else if ((kind).tpr == 32) F<T, W, 32, 1>(__VA_ARGS__); \
        else if ((kind).tpr == 64) {                           \
            if ((kind).nv == 1) F<T, W, 64, 1>(__VA_ARGS__);   \
            else if ((kind).nv == 2) F<T, W, 64, 2>(__VA_ARGS__); \
            else F<T, W, 64, 4>(__VA_ARGS__);                  \
        } else if ((kind).nv == 2) F<T, W, 256, 2>(__VA_ARGS__); \
        else F<T, W, 256, 4>(__VA_ARGS__);                     \
    } while (0)

// ------------------------------------------------------------------------------------------
// dropout.  Philox4x32-10 (J. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", SC 2011): a bijection of a 128-bit counter
// under a 64-bit key, so the draw of an element is a function of (key, position) alone and the backward pass computes the mask again
// instead of reading one.  A block of 8 elements shares a counter: 128 bits = 8 draws of 16, so p counts in steps of 2^-16, and the ten
// rounds (40 multiplications for 8 elements) stay behind the memory: 16384 x 4096 bf16 48 us (5.6 TB/s), with a residual 73 us (5.5 TB/s).
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

struct Dropout { const void *x, *res; void* y; const uint64_t* key; size_t n; uint32_t threshold; float scale; };

template <typename T, bool RES> __global__ __launch_bounds__(NT) void dropout_kernel(Dropout g) {
    const T* __restrict__ x = (const T*)g.x;
    const T* __restrict__ res = (const T*)g.res;
    T* __restrict__ y = (T*)g.y;
    const uint64_t seed = g.key[0], step = g.key[1];
    const size_t n = g.n, blocks = (n + 7) / 8;
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
            v[i] = d >= g.threshold ? v[i] * g.scale : 0.f;      // a dropped infinity or NaN is dropped
            if (RES) v[i] = r[i] + v[i];
        }
        cg_store<T, 8>(y + e, left, v);
    }
}

struct KeyArgs { uint64_t *state, *key; };
// key = state; state's step + 1: one thread, on the caller's stream, so captured graphs draw anew on every replay
__global__ void dropout_key_kernel(KeyArgs g) {
    const uint64_t s = g.state[0], t = g.state[1];
    g.key[0] = s;
    g.key[1] = t;
    g.state[1] = t + 1;
}

}  // namespace

extern "C" int cg_channel_norm_fwd(const cg_group* grp, const void* x, const void* weight, const void* bias, void* y, float* mean,
                                   float* rstd, size_t rows, int C, int dtype, int wdtype, float eps, cg_stream_t stream) {
    CG_CHECK_ARG((!rows || (x && y)) && weight && C > 0 && C <= MAX_CHANNELS && dt_ok(dtype) &&
                     (wdtype == dtype || wdtype == CG_DT_F32) && eps >= 0.f && !mean == !rstd && rows % grp_n(grp) == 0,
                 "cg_channel_norm_fwd: bad args");
    if (!rows) return CG_OK;
    const int n = grp_n(grp);
    rows /= n;
    const NormKind kind = norm_kind(C, dtype == CG_DT_F32 ? 4 : 2);
    CG_DISPATCH_DT(dtype, T, CG_DISPATCH_DT(wdtype, W, {
        if constexpr (std::is_same_v<W, T> || std::is_same_v<W, float>) {
            Norm<T, W> g = {};
            g.x = (const T*)x, g.w = (const W*)weight, g.b = (const W*)bias, g.y = (T*)y, g.mean = mean, g.rstd = rstd;
            g.rows = rows, g.gstride = grp_stride(grp), g.C = C, g.eps = eps;
            if (kind.tpr) CG_NORM_KIND(kind, norm_fwd, g, n, cg_s(stream));
            else channel_norm_long_fwd_kernel<T, W><<<dim3((unsigned)(rows < 65536 ? rows : 65536), n), NT, 0, cg_s(stream)>>>(g);
        }
    }));
    CG_LAUNCH_CHECK("cg_channel_norm_fwd");
    return CG_OK;
}

extern "C" size_t cg_channel_norm_bwd_workspace(const cg_group* grp, size_t rows, int C, int dtype) {
    if (C <= 0 || C > MAX_CHANNELS || !dt_ok(dtype)) return 0;
    const int n = grp_n(grp), blocks = norm_blocks(rows / n, C, dtype == CG_DT_F32 ? 4 : 2);
    return blocks == 1 && norm_kind(C, dtype == CG_DT_F32 ? 4 : 2).tpr ? 0 : (size_t)n * blocks * 2 * C * sizeof(float);
}

extern "C" int cg_channel_norm_bwd(const cg_group* grp, const void* dy, const void* x, const void* weight, const float* mean,
                                   const float* rstd, void* dx, void* dweight, void* dbias, int accumulate, size_t rows, int C,
                                   int dtype, int wdtype, void* ws, size_t ws_bytes, cg_stream_t stream) {
    CG_CHECK_ARG((!rows || (dy && x && mean && rstd)) && weight && C > 0 && C <= MAX_CHANNELS && dt_ok(dtype) &&
                     (wdtype == dtype || wdtype == CG_DT_F32) && rows % grp_n(grp) == 0, "cg_channel_norm_bwd: bad args");
    const int n = grp_n(grp);
    const size_t need = cg_channel_norm_bwd_workspace(grp, rows, C, dtype);
    const bool params = dweight || dbias;
    if (params && need && (!ws || ws_bytes < need)) return cg_set_error(CG_ERR_WORKSPACE, "cg_channel_norm_bwd: workspace too small");
    rows /= n;
    const NormKind kind = norm_kind(C, dtype == CG_DT_F32 ? 4 : 2);
    CG_DISPATCH_DT(dtype, T, CG_DISPATCH_DT(wdtype, W, {
        if constexpr (std::is_same_v<W, T> || std::is_same_v<W, float>) {
            Norm<T, W> g = {};
            g.dy = (const T*)dy, g.x = (const T*)x, g.w = (const W*)weight, g.mean = (float*)mean, g.rstd = (float*)rstd;
            g.dx = rows ? (T*)dx : nullptr, g.dw = (W*)dweight, g.db = (W*)dbias, g.part = params && need ? (float*)ws : nullptr;
            g.rows = rows, g.gstride = grp_stride(grp), g.C = C, g.accumulate = accumulate;
            g.blocks = norm_blocks(rows, C, dtype == CG_DT_F32 ? 4 : 2);
            if (kind.tpr) {
                CG_NORM_KIND(kind, norm_bwd, g, n, cg_s(stream));
            } else {
                if (g.dx) channel_norm_long_dx_kernel<T, W><<<dim3((unsigned)(rows < 65536 ? rows : 65536), n), NT, 0, cg_s(stream)>>>(g);
                if (params) channel_norm_long_dw_kernel<T, W><<<dim3(cg_div_up(C, NT), n, g.blocks), NT, 0, cg_s(stream)>>>(g);
            }
            if (g.part) channel_norm_join_kernel<T, W><<<dim3(cg_div_up(2 * (size_t)C, 32), n), 1024, 0, cg_s(stream)>>>(g);
        }
    }));
    CG_LAUNCH_CHECK("cg_channel_norm_bwd");
    return CG_OK;
}

extern "C" int cg_dropout_key(void* state, void* key, cg_stream_t stream) {
    CG_CHECK_ARG(state && key && state != key, "cg_dropout_key: bad args");
    dropout_key_kernel<<<1, 1, 0, cg_s(stream)>>>(KeyArgs{(uint64_t*)state, (uint64_t*)key});
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
    const Dropout g = {x, residual, y, (const uint64_t*)key, n, (uint32_t)threshold, scale};
    CG_DISPATCH_DT(dtype, T, {
        if (residual) dropout_kernel<T, true><<<grid, NT, 0, cg_s(stream)>>>(g);
        else dropout_kernel<T, false><<<grid, NT, 0, cg_s(stream)>>>(g);
    });
    CG_LAUNCH_CHECK("cg_dropout");
    return CG_OK;
}
