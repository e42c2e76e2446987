// Layer normalisation and its gradient.
//
// Per item n of a (features, items) matrix, in fp32:
//
//     mean_n = sum_f x_fn / F        rstd_n = 1 / sqrt(sum_f (x_fn - mean_n)^2 / F + eps)
//     h_fn   = (x_fn - mean_n) rstd_n                y_fn = h_fn gamma_f + beta_f
//
// and, from the error e_fn at the output, with g_fn = e_fn gamma_f,
//
//     delta_fn = rstd_n (g_fn - sum_f g_fn / F - h_fn sum_f (g_fn h_fn) / F)
//     grad_gamma_f = sum_n e_fn h_fn                 grad_beta_f = sum_n e_fn
//
// The variance is the centred one (a second walk over the item, not E[x^2] - mean^2), so items
// with a mean far from zero keep their digits.  Every sum is fp32 and in a fixed order.

#include "nn_common.cuh"

using namespace nn;

namespace {

struct LnP {
    u64 x, e, out, gamma, beta, mean, rstd;          // e, out: error and delta, or unused and y
    i64 x0, x1, e0, e1, o0, o1;                      // element strides along features and items
    int dt, pdt;                                     // element types of the matrices and of gamma / beta
    i64 F, N;
    float eps;
};

struct LnGradP {
    u64 x, e, mean, rstd, ggamma, gbeta;
    i64 x0, x1, e0, e1;
    int dt, pdt;
    i64 F, N;
};

// ---- any strides: a block per item, one element per thread and step
__global__ void __launch_bounds__(256) ln_fprop_any(const __grid_constant__ LnP p) {
    __shared__ float s[32];
    const float inv = 1.f / (float)p.F;
    for (i64 n = blockIdx.x; n < p.N; n += gridDim.x) {
        float a = 0.f;
        for (i64 f = threadIdx.x; f < p.F; f += blockDim.x) a += ld_any(p.x, f * p.x0 + n * p.x1, p.dt);
        const float mean = block_sum(a, s) * inv;
        a = 0.f;
        for (i64 f = threadIdx.x; f < p.F; f += blockDim.x) {
            const float d = ld_any(p.x, f * p.x0 + n * p.x1, p.dt) - mean;
            a += d * d;
        }
        const float rstd = 1.f / sqrtf(block_sum(a, s) * inv + p.eps);
        for (i64 f = threadIdx.x; f < p.F; f += blockDim.x) {
            float v = (ld_any(p.x, f * p.x0 + n * p.x1, p.dt) - mean) * rstd;
            if (p.gamma) v *= ld_any(p.gamma, f, p.pdt);
            if (p.beta) v += ld_any(p.beta, f, p.pdt);
            st_any(p.out, f * p.o0 + n * p.o1, p.dt, v);
        }
        if (threadIdx.x == 0) {
            if (p.mean) reinterpret_cast<float*>(p.mean)[n] = mean;
            if (p.rstd) reinterpret_cast<float*>(p.rstd)[n] = rstd;
        }
    }
}

__global__ void __launch_bounds__(256) ln_delta_any(const __grid_constant__ LnP p) {
    __shared__ float s[32];
    const float inv = 1.f / (float)p.F;
    for (i64 n = blockIdx.x; n < p.N; n += gridDim.x) {
        const float mean = reinterpret_cast<const float*>(p.mean)[n], rstd = reinterpret_cast<const float*>(p.rstd)[n];
        float a = 0.f, b = 0.f;
        for (i64 f = threadIdx.x; f < p.F; f += blockDim.x) {
            const float g = ld_any(p.e, f * p.e0 + n * p.e1, p.dt) * (p.gamma ? ld_any(p.gamma, f, p.pdt) : 1.f);
            a += g;
            b += g * ((ld_any(p.x, f * p.x0 + n * p.x1, p.dt) - mean) * rstd);
        }
        a = block_sum(a, s) * inv;
        b = block_sum(b, s) * inv;
        for (i64 f = threadIdx.x; f < p.F; f += blockDim.x) {
            const float g = ld_any(p.e, f * p.e0 + n * p.e1, p.dt) * (p.gamma ? ld_any(p.gamma, f, p.pdt) : 1.f);
            const float h = (ld_any(p.x, f * p.x0 + n * p.x1, p.dt) - mean) * rstd;
            st_any(p.out, f * p.o0 + n * p.o1, p.dt, rstd * (g - a - h * b));
        }
    }
}

// a block per feature
__global__ void __launch_bounds__(256) ln_grads_any(const __grid_constant__ LnGradP p) {
    __shared__ float s[32];
    for (i64 f = blockIdx.x; f < p.F; f += gridDim.x) {
        float a = 0.f, b = 0.f;
        for (i64 n = threadIdx.x; n < p.N; n += blockDim.x) {
            const float e = ld_any(p.e, f * p.e0 + n * p.e1, p.dt);
            const float h = (ld_any(p.x, f * p.x0 + n * p.x1, p.dt) - reinterpret_cast<const float*>(p.mean)[n])
                            * reinterpret_cast<const float*>(p.rstd)[n];
            a += e * h;
            b += e;
        }
        a = block_sum(a, s);
        b = block_sum(b, s);
        if (threadIdx.x == 0) {
            if (p.ggamma) st_any(p.ggamma, f, p.pdt, a);
            if (p.gbeta) st_any(p.gbeta, f, p.pdt, b);
        }
    }
}

// ---- features of an item next to each other (their stride is 1)
//
// An item lives in registers: every thread holds NV vectors of V elements of it, so x is read
// once for the mean, the centred variance and the result.  Blocks are persistent: gamma and beta
// (and, backwards, the sums for their gradients) stay in registers from item to item, and the
// next item is loaded while this one is worked on.  WARP: a warp per item instead of a block, for
// items that fit into the registers of one.
template <int DT, int V, int NV> struct Slice {
    static constexpr int W = (dt_size<DT>::value * V + 3) / 4;
    u32 w[NV][W];
    DEV void load(u64 base, i64 at, int me, int T, int F) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int f = (j * T + me) * V;
            if (f < F) ld_w<DT, V, false>(base, at + f, w[j]);
        }
    }
    DEV void get(int j, float* v) const { cvt_in<DT, V>(w[j], v); }
};

template <int V, int NV> DEV void load_params(u64 base, int dt, float fill, int me, int T, int F, float (&v)[NV][V]) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int f = (j * T + me) * V + i;
            v[j][i] = base && f < F ? ld_any(base, f, dt) : fill;
        }
}

template <bool WARP> DEV float item_sum(float v, float* s, int& turn) {
    if constexpr (WARP) return warp_sum(v);
    else return block_sum_turn(v, s, turn);
}
template <bool WARP> DEV float2 item_sum2(float a, float b, float2* s, int& turn) {
    if constexpr (WARP) return make_float2(warp_sum(a), warp_sum(b));
    else return block_sum2_turn(a, b, s, turn);
}

template <int DT, int V, int NV, bool WARP, int MAXT>
__global__ void __launch_bounds__(MAXT) ln_fprop_rows(const __grid_constant__ LnP p) {
    __shared__ float s[64];
    const int T = WARP ? 32 : blockDim.x, me = WARP ? threadIdx.x & 31 : threadIdx.x, F = (int)p.F;
    const i64 step = WARP ? (i64)gridDim.x * 8 : gridDim.x;
    i64 n = WARP ? (i64)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (n >= p.N) return;                              // whole warps, or whole blocks
    const float inv = 1.f / (float)F;
    int turn = 0;
    Slice<DT, V, NV> cur, next;
    cur.load(p.x, n * p.x1, me, T, F);
    float gamma[NV][V], beta[NV][V];
    load_params<V, NV>(p.gamma, p.pdt, 1.f, me, T, F, gamma);
    load_params<V, NV>(p.beta, p.pdt, 0.f, me, T, F, beta);
    for (; n < p.N; n += step) {
        if (n + step < p.N) next.load(p.x, (n + step) * p.x1, me, T, F);
        float x[NV][V], a = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            cur.get(j, x[j]);
            if ((j * T + me) * V < F) {
#pragma unroll
                for (int i = 0; i < V; ++i) a += x[j][i];
            }
        }
        const float mean = item_sum<WARP>(a, s, turn) * inv;
        a = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if ((j * T + me) * V < F) {
#pragma unroll
                for (int i = 0; i < V; ++i) { x[j][i] -= mean; a = fmaf(x[j][i], x[j][i], a); }
            }
        const float rstd = 1.f / sqrtf(item_sum<WARP>(a, s, turn) * inv + p.eps);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int f = (j * T + me) * V;
            if (f >= F) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) x[j][i] = fmaf(x[j][i] * rstd, gamma[j][i], beta[j][i]);
            st_f<DT, V>(p.out, n * p.o1 + f, x[j]);
        }
        if (me == 0) {
            if (p.mean) reinterpret_cast<float*>(p.mean)[n] = mean;
            if (p.rstd) reinterpret_cast<float*>(p.rstd)[n] = rstd;
        }
        cur = next;
    }
}

// part[block][0][F]: the block's share of grad_gamma, part[block][1][F]: of grad_beta
template <int DT, int V, int NV, bool WARP, int MAXT>
__global__ void __launch_bounds__(MAXT) ln_bprop_rows(const __grid_constant__ LnP p, float* part) {
    __shared__ float2 s[64];
    const int T = WARP ? 32 : blockDim.x, me = WARP ? threadIdx.x & 31 : threadIdx.x, F = (int)p.F;
    const i64 step = WARP ? (i64)gridDim.x * 8 : gridDim.x;
    i64 n = WARP ? (i64)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    const float inv = 1.f / (float)F;
    int turn = 0;
    Slice<DT, V, NV> x, e, nx, ne;
    float mean = 0.f, rstd = 0.f;
    if (n < p.N) {
        x.load(p.x, n * p.x1, me, T, F);
        e.load(p.e, n * p.e1, me, T, F);
        mean = reinterpret_cast<const float*>(p.mean)[n];
        rstd = reinterpret_cast<const float*>(p.rstd)[n];
    }
    float gamma[NV][V], gg[NV][V], gb[NV][V];
    load_params<V, NV>(p.gamma, p.pdt, 1.f, me, T, F, gamma);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) gg[j][i] = gb[j][i] = 0.f;
    for (; n < p.N; n += step) {
        float nmean = 0.f, nrstd = 0.f;
        if (n + step < p.N) {
            nx.load(p.x, (n + step) * p.x1, me, T, F);
            ne.load(p.e, (n + step) * p.e1, me, T, F);
            nmean = reinterpret_cast<const float*>(p.mean)[n + step];
            nrstd = reinterpret_cast<const float*>(p.rstd)[n + step];
        }
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if ((j * T + me) * V >= F) continue;
            float h[V], g[V];
            x.get(j, h);
            e.get(j, g);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[i] = (h[i] - mean) * rstd;
                gg[j][i] = fmaf(g[i], h[i], gg[j][i]);
                gb[j][i] += g[i];
                g[i] *= gamma[j][i];
                a += g[i];
                b = fmaf(g[i], h[i], b);
            }
        }
        const float2 ab = item_sum2<WARP>(a, b, s, turn);
        a = ab.x * inv;
        b = ab.y * inv;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int f = (j * T + me) * V;
            if (f >= F) continue;
            float h[V], g[V];
            x.get(j, h);
            e.get(j, g);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                h[i] = (h[i] - mean) * rstd;
                g[i] = rstd * (g[i] * gamma[j][i] - a - h[i] * b);
            }
            st_f<DT, V>(p.out, n * p.o1 + f, g);
        }
        x = nx; e = ne; mean = nmean; rstd = nrstd;
    }
    if (!part) return;
    if constexpr (WARP) {
        // the warps of a block one after the other, in shared memory
        extern __shared__ float acc[];                 // [2][F]
        for (int w = 0; w < 8; ++w) {
            if ((threadIdx.x >> 5) == w) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const int f = (j * T + me) * V + i;
                        if (f >= F) continue;
                        acc[f] = (w ? acc[f] : 0.f) + gg[j][i];
                        acc[F + f] = (w ? acc[F + f] : 0.f) + gb[j][i];
                    }
            }
            __syncthreads();
        }
        for (int f = threadIdx.x; f < 2 * F; f += 256) part[(i64)blockIdx.x * 2 * F + f] = acc[f];
    } else {
        float* to = part + (i64)blockIdx.x * 2 * F;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int f = (j * T + me) * V + i;
                if (f < F) { to[f] = gg[j][i]; to[F + f] = gb[j][i]; }
            }
    }
}

// The sum of the blocks' shares, in the order of the blocks within each of 32 rows of threads.
__global__ void __launch_bounds__(1024) ln_sum_parts(const float* part, int blocks, i64 F, u64 ggamma, u64 gbeta, int pdt) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const i64 c = (i64)blockIdx.x * 32 + lane;          // column of [grad_gamma | grad_beta]
    float a = 0.f;
    if (c < 2 * F)
        for (int b = row; b < blocks; b += 32) a += part[(i64)b * 2 * F + c];
    s[row][lane] = a;
    __syncthreads();
    a = warp_sum(s[lane][row]);
    const i64 out = (i64)blockIdx.x * 32 + row;
    if (lane == 0 && out < 2 * F) {
        const u64 to = out < F ? ggamma : gbeta;
        if (to) st_any(to, out < F ? out : out - F, pdt, a);
    }
}

// Which of the register kernels an item of F features takes: T threads with NV vectors of V
// elements each; a warp where `most` elements per lane hold an item.
struct Rows { int V, NV, T; bool warp; };
enum { kMaxRow = 16384 };

inline bool rows_plan(i64 F, int V, int most, Rows& r) {
    if (F > kMaxRow) return false;
    const int nvec = (int)((F + V - 1) / V);
    r.V = V;
    for (int nv = 1; nv * V <= most; nv *= 2)
        if (nvec <= 32 * nv) { r.NV = nv; r.T = 32; r.warp = true; return true; }
    r.warp = false;
    for (r.NV = 1; r.NV * V <= 16; r.NV *= 2) {
        r.T = ((nvec + r.NV - 1) / r.NV + 31) / 32 * 32;
        if (r.T <= 512 || (r.NV * V == 16 && r.T <= 1024)) return true;
    }
    return false;
}

template <int DT, int V, int NV> cudaError_t launch_fprop(const LnP& p, const Rows& r, cudaStream_t s) {
    const i64 want = r.warp ? (p.N + 7) / 8 : p.N;
    auto go = [&](auto k, int threads) {
        const i64 most = resident_blocks(k, threads, 0);
        k<<<(unsigned)(want < most ? want : most), threads, 0, s>>>(p);
        return cudaGetLastError();
    };
    if (r.warp) return go(ln_fprop_rows<DT, V, NV, true, 256>, 256);
    if (r.T <= 512) return go(ln_fprop_rows<DT, V, NV, false, 512>, r.T);
    if constexpr (V * NV == 16) return go(ln_fprop_rows<DT, V, NV, false, 1024>, r.T);
    return cudaErrorInvalidValue;
}
template <int DT, int V> cudaError_t launch_fprop_v(const LnP& p, const Rows& r, cudaStream_t s) {
    if (r.NV == 1) return launch_fprop<DT, V, 1>(p, r, s);
    if (r.NV == 2) return launch_fprop<DT, V, 2>(p, r, s);
    if constexpr (V <= 4) { if (r.NV == 4) return launch_fprop<DT, V, 4>(p, r, s); }
    if constexpr (V == 1) {
        if (r.NV == 8) return launch_fprop<DT, V, 8>(p, r, s);
        if (r.NV == 16) return launch_fprop<DT, V, 16>(p, r, s);
    }
    return cudaErrorInvalidValue;
}

// Most blocks whose shares of the parameters' gradients fit into 32 MB.
inline i64 most_parts(i64 F) {
    const i64 fit = (32ll << 20) / (8 * F);
    return fit < 1 ? 1 : fit > 2048 ? 2048 : fit;
}

template <int DT, int V, int NV> cudaError_t launch_bprop(const LnP& p, const Rows& r, float* part, int& blocks, cudaStream_t s) {
    const i64 want = r.warp ? (p.N + 7) / 8 : p.N;
    const int smem = r.warp ? (int)(8 * p.F) : 0;
    auto go = [&](auto k, int threads) {
        i64 most = resident_blocks(k, threads, smem);
        if (part && most > most_parts(p.F)) most = most_parts(p.F);
        blocks = (int)(want < most ? want : most);
        k<<<blocks, threads, smem, s>>>(p, part);
        return cudaGetLastError();
    };
    if (r.warp) return go(ln_bprop_rows<DT, V, NV, true, 256>, 256);
    if (r.T <= 512) return go(ln_bprop_rows<DT, V, NV, false, 512>, r.T);
    if constexpr (V * NV == 16) return go(ln_bprop_rows<DT, V, NV, false, 1024>, r.T);
    return cudaErrorInvalidValue;
}
template <int DT, int V> cudaError_t launch_bprop_v(const LnP& p, const Rows& r, float* part, int& blocks, cudaStream_t s) {
    if (r.NV == 1) return launch_bprop<DT, V, 1>(p, r, part, blocks, s);
    if (r.NV == 2) return launch_bprop<DT, V, 2>(p, r, part, blocks, s);
    if constexpr (V <= 4) { if (r.NV == 4) return launch_bprop<DT, V, 4>(p, r, part, blocks, s); }
    if constexpr (V == 1) {
        if (r.NV == 8) return launch_bprop<DT, V, 8>(p, r, part, blocks, s);
        if (r.NV == 16) return launch_bprop<DT, V, 16>(p, r, part, blocks, s);
    }
    return cudaErrorInvalidValue;
}

// Whether every item of the matrices starts on a 16-byte boundary and is a whole number of
// vectors of V elements long.
inline bool vectors(const b200_matrix& m, i64 F, int V) {
    return m.ptr % 16 == 0 && m.s1 % V == 0 && F % V == 0;
}
inline bool is_rows(const b200_matrix& m, i64 F) { return m.s0 == 1 || F == 1; }

unsigned blocks_for(i64 n) { return (unsigned)(n < 65536 ? n : 65536); }

// Checks that the matrices and vectors of either direction have in common.
int32_t check_sizes(const char* where, i64 F, i64 N) {
    if (F < 1 || F > 0x7fffffff) return refuse(where, "between 1 and 2^31 - 1 features");
    if (N < 0 || N > 0x7fffffff) return refuse(where, "between 0 and 2^31 - 1 items");
    return B200_OK;
}
b200_matrix vec(uint64_t ptr, int dt) { b200_matrix m; m.ptr = ptr; m.s0 = 1; m.s1 = 1; m.dtype = dt; m.reserved = 0; return m; }

}  // namespace

extern "C" b200_status b200_ln_fprop(const b200_matrix* x, const b200_matrix* y, uint64_t gamma, uint64_t beta,
                                     int32_t param_dtype, uint64_t mean, uint64_t rstd, int64_t features,
                                     int64_t items, float eps, uint64_t stream, int32_t* launches) {
    const char* where = "b200_ln_fprop";
    if (launches) *launches = 0;
    if (!x || !y) return refuse(where, "null matrix");
    if (int32_t st = check_sizes(where, features, items)) return st;
    if (!is_float(x->dtype) || y->dtype != x->dtype || !is_float(param_dtype))
        return refuse(where, "only f32, f16 and bf16, the same for x and y", B200_ERR_UNSUPPORTED);
    if (!(eps >= 0.f)) return refuse(where, "eps must not be negative");
    if (items == 0) return B200_OK;
    if (!x->ptr || !y->ptr) return refuse(where, "null device pointer");
    if (!same(*x, *y) && meet(*x, features, items, *y, features, items))
        return refuse(where, "y may be x itself or apart from it, not a shifted view of it");
    if (!aligned(x->ptr, x->dtype) || !aligned(y->ptr, y->dtype) || !aligned(gamma | beta, param_dtype) ||
        !aligned(mean | rstd, B200_F32)) return refuse(where, "misaligned pointer");
    const b200_matrix vecs[4] = {vec(gamma, param_dtype), vec(beta, param_dtype), vec(mean, B200_F32), vec(rstd, B200_F32)};
    for (int i = 0; i < 4; ++i) {
        const i64 n = i < 2 ? features : items;
        if (!vecs[i].ptr) continue;
        if (meet(*y, features, items, vecs[i], n, 1)) return refuse(where, "y shares memory with gamma, beta, mean or rstd");
        if (i >= 2) {
            if (meet(*x, features, items, vecs[i], n, 1)) return refuse(where, "mean or rstd shares memory with x");
            for (int j = 0; j < i; ++j)
                if (vecs[j].ptr && meet(vecs[j], j < 2 ? features : items, 1, vecs[i], n, 1))
                    return refuse(where, "mean, rstd, gamma and beta must not share memory");
        }
    }
    DeviceScope scope;
    if (scope.error() != cudaSuccess) return cuda_status(where, scope.error());
    cudaStream_t s = static_cast<cudaStream_t>(b200_detail_stream(stream));
    LnP p;
    p.x = x->ptr; p.e = 0; p.out = y->ptr; p.gamma = gamma; p.beta = beta; p.mean = mean; p.rstd = rstd;
    p.x0 = x->s0; p.x1 = x->s1; p.e0 = p.e1 = 0; p.o0 = y->s0; p.o1 = y->s1;
    p.dt = x->dtype; p.pdt = param_dtype; p.F = features; p.N = items; p.eps = eps;
    cudaError_t e = cudaSuccess;
    Rows r;
    const int V = 16 / (int)esize(x->dtype);
    const bool rows = is_rows(*x, features) && is_rows(*y, features);
    if (rows && vectors(*x, features, V) && vectors(*y, features, V) && rows_plan(features, V, 16, r)) {
        if (x->dtype == B200_F32) e = launch_fprop_v<F32, 4>(p, r, s);
        else if (x->dtype == B200_F16) e = launch_fprop_v<F16, 8>(p, r, s);
        else e = launch_fprop_v<BF16, 8>(p, r, s);
    } else if (rows && rows_plan(features, 1, 16, r)) {
        if (x->dtype == B200_F32) e = launch_fprop_v<F32, 1>(p, r, s);
        else if (x->dtype == B200_F16) e = launch_fprop_v<F16, 1>(p, r, s);
        else e = launch_fprop_v<BF16, 1>(p, r, s);
    } else {
        ln_fprop_any<<<blocks_for(items), 256, 0, s>>>(p);
        e = cudaGetLastError();
    }
    if (launches) *launches = 1;
    return cuda_status(where, e);
}

extern "C" uint64_t b200_ln_bprop_scratch_bytes(int64_t features, int64_t items) {
    if (features < 1 || items < 1 || features > kMaxRow) return 0;
    const i64 parts = most_parts(features);
    return (uint64_t)((items < parts ? items : parts) * 8 * features);
}

extern "C" b200_status b200_ln_bprop(const b200_matrix* delta, const b200_matrix* error, const b200_matrix* x,
                                     uint64_t mean, uint64_t rstd, uint64_t gamma, uint64_t grad_gamma,
                                     uint64_t grad_beta, int32_t param_dtype, int64_t features, int64_t items,
                                     uint64_t scratch, uint64_t scratch_bytes, uint64_t stream, int32_t* launches) {
    const char* where = "b200_ln_bprop";
    if (launches) *launches = 0;
    if (!delta || !error || !x) return refuse(where, "null matrix");
    if (int32_t st = check_sizes(where, features, items)) return st;
    if (!is_float(x->dtype) || error->dtype != x->dtype || delta->dtype != x->dtype || !is_float(param_dtype))
        return refuse(where, "only f32, f16 and bf16, the same for x, error and delta", B200_ERR_UNSUPPORTED);
    const uint64_t need = b200_ln_bprop_scratch_bytes(features, items);
    if (scratch_bytes < need || (need && (!scratch || scratch % 256))) return refuse(where, "scratch too small or misaligned");
    if (items && (!delta->ptr || !error->ptr || !x->ptr || !mean || !rstd)) return refuse(where, "null device pointer");
    if (!aligned(x->ptr | error->ptr | delta->ptr, x->dtype) || !aligned(gamma | grad_gamma | grad_beta, param_dtype) ||
        !aligned(mean | rstd, B200_F32)) return refuse(where, "misaligned pointer");
    for (const b200_matrix* in : {error, x})
        if (!same(*in, *delta) && meet(*in, features, items, *delta, features, items))
            return refuse(where, "delta may be x or the error itself or apart from them, not a shifted view");
    const b200_matrix vecs[5] = {vec(gamma, param_dtype), vec(mean, B200_F32), vec(rstd, B200_F32),
                                 vec(grad_gamma, param_dtype), vec(grad_beta, param_dtype)};
    for (int i = 0; i < 5; ++i) {
        const i64 n = i == 1 || i == 2 ? items : features;
        if (!vecs[i].ptr) continue;
        if (meet(*delta, features, items, vecs[i], n, 1))
            return refuse(where, "delta shares memory with a vector of the call");
        if (i < 3) continue;
        if (meet(*x, features, items, vecs[i], n, 1) || meet(*error, features, items, vecs[i], n, 1))
            return refuse(where, "a gradient shares memory with x or the error");
        for (int j = 0; j < i; ++j)
            if (vecs[j].ptr && meet(vecs[j], j == 1 || j == 2 ? items : features, 1, vecs[i], n, 1))
                return refuse(where, "a gradient shares memory with another vector of the call");
    }
    DeviceScope scope;
    if (scope.error() != cudaSuccess) return cuda_status(where, scope.error());
    cudaStream_t s = static_cast<cudaStream_t>(b200_detail_stream(stream));
    cudaError_t err = cudaSuccess;
    if (items == 0) {                                  // sums over nothing
        for (uint64_t g : {grad_gamma, grad_beta})
            if (g && err == cudaSuccess) err = cudaMemsetAsync(reinterpret_cast<void*>(g), 0, (size_t)(features * esize(param_dtype)), s);
        return cuda_status(where, err);
    }
    LnP p;
    p.x = x->ptr; p.e = error->ptr; p.out = delta->ptr; p.gamma = gamma; p.beta = 0; p.mean = mean; p.rstd = rstd;
    p.x0 = x->s0; p.x1 = x->s1; p.e0 = error->s0; p.e1 = error->s1; p.o0 = delta->s0; p.o1 = delta->s1;
    p.dt = x->dtype; p.pdt = param_dtype; p.F = features; p.N = items; p.eps = 0.f;
    int count = 1;
    Rows r;
    const int V = 16 / (int)esize(x->dtype);
    const bool rows = is_rows(*x, features) && is_rows(*error, features) && is_rows(*delta, features);
    const bool wide = rows && vectors(*x, features, V) && vectors(*error, features, V) && vectors(*delta, features, V)
                      && rows_plan(features, V, 8, r);
    if (wide || (rows && rows_plan(features, 1, 8, r))) {
        float* part = grad_gamma || grad_beta ? reinterpret_cast<float*>(scratch) : nullptr;
        int blocks = 0;
        if (wide) {
            if (x->dtype == B200_F32) err = launch_bprop_v<F32, 4>(p, r, part, blocks, s);
            else if (x->dtype == B200_F16) err = launch_bprop_v<F16, 8>(p, r, part, blocks, s);
            else err = launch_bprop_v<BF16, 8>(p, r, part, blocks, s);
        } else {
            if (x->dtype == B200_F32) err = launch_bprop_v<F32, 1>(p, r, part, blocks, s);
            else if (x->dtype == B200_F16) err = launch_bprop_v<F16, 1>(p, r, part, blocks, s);
            else err = launch_bprop_v<BF16, 1>(p, r, part, blocks, s);
        }
        if (part && err == cudaSuccess) {
            ln_sum_parts<<<(unsigned)((2 * features + 31) / 32), 1024, 0, s>>>(part, blocks, features, grad_gamma, grad_beta, param_dtype);
            err = cudaGetLastError();
            ++count;
        }
    } else {
        if (grad_gamma || grad_beta) {                 // before delta, which may overwrite x or the error
            LnGradP q;
            q.x = x->ptr; q.e = error->ptr; q.mean = mean; q.rstd = rstd; q.ggamma = grad_gamma; q.gbeta = grad_beta;
            q.x0 = x->s0; q.x1 = x->s1; q.e0 = error->s0; q.e1 = error->s1;
            q.dt = x->dtype; q.pdt = param_dtype; q.F = features; q.N = items;
            ln_grads_any<<<blocks_for(features), 256, 0, s>>>(q);
            ++count;
        }
        ln_delta_any<<<blocks_for(items), 256, 0, s>>>(p);
        err = cudaGetLastError();
    }
    if (launches) *launches = count;
    return cuda_status(where, err);
}
