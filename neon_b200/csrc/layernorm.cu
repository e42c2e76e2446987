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
    ln_fprop_any<<<blocks_for(items), 256, 0, s>>>(p);
    if (launches) *launches = 1;
    return cuda_status(where, cudaGetLastError());
}

extern "C" uint64_t b200_ln_bprop_scratch_bytes(int64_t features, int64_t items) {
    (void)features; (void)items;
    return 0;
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
    if (scratch_bytes < b200_ln_bprop_scratch_bytes(features, items)) return refuse(where, "scratch too small");
    DeviceScope scope;
    if (scope.error() != cudaSuccess) return cuda_status(where, scope.error());
    cudaStream_t s = static_cast<cudaStream_t>(b200_detail_stream(stream));
    if (items == 0) {                                  // sums over nothing
        cudaError_t e = cudaSuccess;
        for (uint64_t g : {grad_gamma, grad_beta})
            if (g && e == cudaSuccess) e = cudaMemsetAsync(reinterpret_cast<void*>(g), 0, (size_t)(features * esize(param_dtype)), s);
        return cuda_status(where, e);
    }
    if (!delta->ptr || !error->ptr || !x->ptr || !mean || !rstd) return refuse(where, "null device pointer");
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
    int count = 0;
    if (grad_gamma || grad_beta) {                     // before delta, which may overwrite x or the error
        LnGradP q;
        q.x = x->ptr; q.e = error->ptr; q.mean = mean; q.rstd = rstd; q.ggamma = grad_gamma; q.gbeta = grad_beta;
        q.x0 = x->s0; q.x1 = x->s1; q.e0 = error->s0; q.e1 = error->s1;
        q.dt = x->dtype; q.pdt = param_dtype; q.F = features; q.N = items;
        ln_grads_any<<<blocks_for(features), 256, 0, s>>>(q);
        ++count;
    }
    LnP p;
    p.x = x->ptr; p.e = error->ptr; p.out = delta->ptr; p.gamma = gamma; p.beta = 0; p.mean = mean; p.rstd = rstd;
    p.x0 = x->s0; p.x1 = x->s1; p.e0 = error->s0; p.e1 = error->s1; p.o0 = delta->s0; p.o1 = delta->s1;
    p.dt = x->dtype; p.pdt = param_dtype; p.F = features; p.N = items; p.eps = 0.f;
    ln_delta_any<<<blocks_for(items), 256, 0, s>>>(p);
    if (launches) *launches = count + 1;
    return cuda_status(where, cudaGetLastError());
}
