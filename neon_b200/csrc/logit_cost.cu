// Two costs on a (vocabulary, items) matrix of logits, each with its gradient.
//
// Distillation from a teacher's K largest logits t_k at the words i_k, at temperature T:
//
//     p = softmax over k of t_k / T        q = softmax over v of z_v / T
//     cost  = w T^2 sum_k p_k (ln p_k - ln q_{i_k})
//     delta_v = w T (q_v - sum_{k: i_k = v} p_k)
//
// Clipped policy cost with a KL term for the word a that was chosen:
//
//     l = z_a - ln sum_v exp z_v     r = exp(l - old)     d = ref - l
//     cost  = w (kl (exp(d) - d - 1) - min(r A, clip(r, 1 - lo, 1 + hi) A))
//     delta_v = s ([v = a] - q_v)    s = w (kl (1 - exp(d)) - r A [r A is the smaller one])
//
// Both read every logit for the softmax and then touch K (or one) of them again.  The softmax is
// kept in base 2: with c = log2(e) / T and M = fl(c max z), s = sum 2^(z c - M) uses the same
// rounded M as the gradient's 2^(z c - M) / s, so that M's rounding cancels there, and
// ln sum exp(z / T) = max z / T + ln s - ln 2 (c max z - M) takes it out of the cost.
//
// An item of weight 0, an item whose word lies outside the vocabulary and a teacher's list
// without a usable entry (words outside, or logits of -inf) give cost 0 and delta 0, whatever
// the logits hold.  The delta may overwrite the logits.

#include "nn_common.cuh"

#include <cmath>

using namespace nn;

namespace {

enum { kMaxTop = B200_DISTILL_MAX_TOP };

struct CostP {
    u64 z, d;                            // logits; delta or 0
    i64 z0, z1, d0, d1;                  // element strides along the vocabulary and the items
    int dt;
    int V;
    i64 N;
    u64 weights, cost;
    float c, temp, inv_temp;             // log2(e) / T, T, 1 / T
    // distillation
    u64 ids, top;
    i64 i0, i1, t0, t1;
    int tdt, K;
    // policy
    u64 actions, old, ref, adv, logp;
    float lo, hi, kl;
};

// What an item's gradient needs besides the logits: delta_v = scale 2^(z_v c - M) for the words
// without an entry of their own.
struct Item { float M, scale; bool dead; };

// Shared memory of one item: the word numbers, probabilities and finished gradients of its entries.
struct Entries { int* id; float* p; float* g; float* red; };

DEV float weight_of(const CostP& p, i64 n) { return p.weights ? reinterpret_cast<const float*>(p.weights)[n] : 1.f; }

// Items that need not be looked at: their cost and delta are zero.
DEV bool skipped(const CostP& p, i64 n, bool policy) {
    if (weight_of(p, n) == 0.f && !(policy && p.logp)) return true;
    if (policy) {
        const int a = reinterpret_cast<const int*>(p.actions)[n];
        return a < 0 || a >= p.V;
    }
    return false;
}

// The entries of one item, by all threads of its block, once the logits' maximum and sum are known.
DEV Item distill_entries(const CostP& p, i64 n, float zmax, float s, const Entries& e) {
    const int tid = threadIdx.x, nt = blockDim.x;
    Item it;
    it.M = zmax * p.c;
    const float w = weight_of(p, n);
    const float ln_s = logf(s) - fmaf(zmax, p.c, -it.M) * 0.693147182464599609375f;
    float m = -INFINITY;
    for (int k = tid; k < p.K; k += nt) {
        const int id = *(reinterpret_cast<const int*>(p.ids) + k * p.i0 + n * p.i1);
        float t = ld_any(p.top, k * p.t0 + n * p.t1, p.tdt);
        const bool used = id >= 0 && id < p.V && t != -INFINITY;
        e.id[k] = used ? id : -1;
        e.p[k] = t;
        if (used) m = fmaxf(m, t);
    }
    // a NaN among the teacher's logits reaches the sum below whatever the maximum says
    m = block_max(m, e.red);
    float sum = 0.f;
    int used = 0;
    for (int k = tid; k < p.K; k += nt) {
        if (e.id[k] < 0) { e.p[k] = 0.f; continue; }
        used = 1;
        e.p[k] = (e.p[k] - m) * p.inv_temp;
        sum += expf(e.p[k]);
    }
    sum = block_sum(sum, e.red);
    const bool any = __syncthreads_or(used);
    it.dead = w == 0.f || !any;
    it.scale = w * p.temp / s;
    const float ln_sum = logf(sum);
    float cost = 0.f;
    for (int k = tid; k < p.K; k += nt) {
        float zk = 0.f;
        if (e.id[k] >= 0) {
            zk = ld_any(p.z, (i64)e.id[k] * p.z0 + n * p.z1, p.dt);
            const float lp = e.p[k] - ln_sum, pk = expf(lp);
            e.p[k] = pk;
            if (pk != 0.f) cost += pk * (lp - ((zk - zmax) * p.inv_temp - ln_s));
        }
        e.g[k] = zk;
    }
    cost = block_sum(cost, e.red);
    if (tid == 0) reinterpret_cast<float*>(p.cost)[n] = it.dead ? 0.f : w * p.temp * p.temp * cost;
    if (p.d) {
        // a word listed more than once: all of its entries hold (and later write) the same value
        __syncthreads();
        for (int k = tid; k < p.K; k += nt) {
            const int id = e.id[k];
            if (id < 0) continue;
            float mass = 0.f;
            for (int j = 0; j < p.K; ++j) mass += e.id[j] == id ? e.p[j] : 0.f;
            e.g[k] = it.scale * exp2f(fmaf(e.g[k], p.c, -it.M)) - w * p.temp * mass;
        }
        __syncthreads();
    }
    return it;
}

DEV Item policy_entry(const CostP& p, i64 n, float zmax, float s, const Entries& e) {
    Item it;
    it.M = zmax * p.c;
    const float w = weight_of(p, n);
    const int a = reinterpret_cast<const int*>(p.actions)[n];
    const float za = ld_any(p.z, (i64)a * p.z0 + n * p.z1, p.dt);
    const float ln_s = logf(s) - fmaf(zmax, p.c, -it.M) * 0.693147182464599609375f;
    const float l = (za - zmax) - ln_s;
    const float adv = reinterpret_cast<const float*>(p.adv)[n];
    const float r = expf(l - reinterpret_cast<const float*>(p.old)[n]);
    const float free = r * adv, held = fminf(fmaxf(r, 1.f - p.lo), 1.f + p.hi) * adv;
    const bool is_free = !(held < free);
    float cost = -(is_free ? free : held), slope = is_free ? -free : 0.f;
    if (p.ref) {
        const float d = reinterpret_cast<const float*>(p.ref)[n] - l, m1 = expm1f(d);
        cost += p.kl * (m1 - d);
        slope -= p.kl * m1;
    }
    slope *= w;
    it.dead = w == 0.f;
    it.scale = -slope / s;
    if (threadIdx.x == 0) {
        reinterpret_cast<float*>(p.cost)[n] = it.dead ? 0.f : w * cost;
        if (p.logp) reinterpret_cast<float*>(p.logp)[n] = l;
        e.id[0] = a;
        e.g[0] = fmaf(it.scale, exp2f(fmaf(za, p.c, -it.M)), slope);
    }
    __syncthreads();
    return it;
}

// ---- any strides: a block per item, one logit per thread and step
template <bool POLICY>
__global__ void __launch_bounds__(256) cost_any(const __grid_constant__ CostP p) {
    __shared__ float red[32];
    __shared__ int ids[POLICY ? 1 : kMaxTop];
    __shared__ float probs[POLICY ? 1 : kMaxTop], grads[POLICY ? 1 : kMaxTop];
    const Entries e = {ids, probs, grads, red};
    const int entries = POLICY ? 1 : p.K;
    for (i64 n = blockIdx.x; n < p.N; n += gridDim.x) {
        __syncthreads();                               // the entries of the previous item are written
        Item it;
        it.dead = skipped(p, n, POLICY);
        if (it.dead) {
            if (threadIdx.x == 0) {
                reinterpret_cast<float*>(p.cost)[n] = 0.f;
                if (POLICY && p.logp) reinterpret_cast<float*>(p.logp)[n] = 0.f;
            }
        } else {
            float m = -INFINITY;
            for (int v = threadIdx.x; v < p.V; v += blockDim.x) m = fmaxf(m, ld_any(p.z, v * p.z0 + n * p.z1, p.dt));
            m = block_max(m, red);
            const float M = m * p.c;
            float s = 0.f;
            for (int v = threadIdx.x; v < p.V; v += blockDim.x) s += exp2f(fmaf(ld_any(p.z, v * p.z0 + n * p.z1, p.dt), p.c, -M));
            s = block_sum(s, red);
            it = POLICY ? policy_entry(p, n, m, s, e) : distill_entries(p, n, m, s, e);
        }
        if (!p.d) continue;
        for (int v = threadIdx.x; v < p.V; v += blockDim.x) {
            const float z = ld_any(p.z, v * p.z0 + n * p.z1, p.dt);
            st_any(p.d, v * p.d0 + n * p.d1, p.dt, it.dead ? 0.f : it.scale * exp2f(fmaf(z, p.c, -it.M)));
        }
        if (it.dead) continue;
        __syncthreads();
        for (int k = threadIdx.x; k < entries; k += blockDim.x)
            if (e.id[k] >= 0)
                st_any(p.d, (i64)e.id[k] * p.d0 + n * p.d1, p.dt, e.g[k]);
    }
}

unsigned blocks_for(i64 n) { return (unsigned)(n < 65536 ? n : 65536); }

b200_matrix vec(uint64_t ptr, int dt) { b200_matrix m; m.ptr = ptr; m.s0 = 1; m.s1 = 1; m.dtype = dt; m.reserved = 0; return m; }

// Sizes, types and overlaps that the two costs check alike; `in` are vectors of one value per
// item that are read, `out` those that are written (cost first).
int32_t check(const char* where, const b200_matrix* z, const b200_matrix* d, i64 V, i64 N, const b200_matrix* in, int n_in,
              const b200_matrix* out, int n_out) {
    if (V < 1 || V > 0x7fffffff) return refuse(where, "between 1 and 2^31 - 1 words");
    if (N < 0 || N > 0x7fffffff) return refuse(where, "between 0 and 2^31 - 1 items");
    if (!is_float(z->dtype) || (d->ptr && d->dtype != z->dtype))
        return refuse(where, "only f32, f16 and bf16, the same for logits and delta", B200_ERR_UNSUPPORTED);
    if (N == 0) return B200_OK;
    if (!z->ptr || !out[0].ptr) return refuse(where, "null device pointer");
    if (!aligned(z->ptr | d->ptr, z->dtype)) return refuse(where, "misaligned pointer");
    if (d->ptr && !same(*z, *d) && meet(*z, V, N, *d, V, N))
        return refuse(where, "delta may be the logits themselves or apart from them, not a shifted view");
    for (int i = 0; i < n_in; ++i) {
        if (!in[i].ptr) continue;
        if (!aligned(in[i].ptr, in[i].dtype)) return refuse(where, "misaligned pointer");
        if (d->ptr && meet(*d, V, N, in[i], N, 1)) return refuse(where, "delta shares memory with an input");
    }
    for (int i = 0; i < n_out; ++i) {
        if (!out[i].ptr) continue;
        if (!aligned(out[i].ptr, out[i].dtype)) return refuse(where, "misaligned pointer");
        if (meet(*z, V, N, out[i], N, 1) || (d->ptr && meet(*d, V, N, out[i], N, 1)))
            return refuse(where, "the cost shares memory with logits or delta");
        for (int j = 0; j < n_in; ++j)
            if (in[j].ptr && meet(in[j], N, 1, out[i], N, 1)) return refuse(where, "the cost shares memory with an input");
        for (int j = 0; j < i; ++j)
            if (out[j].ptr && meet(out[j], N, 1, out[i], N, 1)) return refuse(where, "two outputs share memory");
    }
    return B200_OK;
}

template <bool POLICY>
int32_t run(const char* where, CostP& p, uint64_t stream, int32_t* launches) {
    DeviceScope scope;
    if (scope.error() != cudaSuccess) return cuda_status(where, scope.error());
    cudaStream_t s = static_cast<cudaStream_t>(b200_detail_stream(stream));
    cost_any<POLICY><<<blocks_for(p.N), 256, 0, s>>>(p);
    if (launches) *launches = 1;
    return cuda_status(where, cudaGetLastError());
}

void set_logits(CostP& p, const b200_matrix* z, const b200_matrix* d, i64 V, i64 N, uint64_t weights, uint64_t cost) {
    p = CostP();
    p.z = z->ptr; p.z0 = z->s0; p.z1 = z->s1; p.dt = z->dtype;
    p.d = d->ptr; p.d0 = d->s0; p.d1 = d->s1;
    p.V = (int)V; p.N = N; p.weights = weights; p.cost = cost;
}

}  // namespace

extern "C" b200_status b200_distill(const b200_matrix* logits, const b200_matrix* delta, const b200_matrix* top_ids,
                                    const b200_matrix* top_logits, uint64_t weights, uint64_t cost, int64_t words,
                                    int64_t items, int64_t top, float temperature, uint64_t stream, int32_t* launches) {
    const char* where = "b200_distill";
    if (launches) *launches = 0;
    if (!logits || !top_ids || !top_logits) return refuse(where, "null matrix");
    const b200_matrix none = vec(0, logits->dtype), *d = delta ? delta : &none;
    const b200_matrix in[1] = {vec(weights, B200_F32)}, out[1] = {vec(cost, B200_F32)};
    if (!(temperature > 0.f) || !std::isfinite(temperature) || !std::isfinite(1.f / temperature))
        return refuse(where, "the temperature must be positive and finite");
    if (top < 1 || top > kMaxTop) return refuse(where, "between 1 and 1024 entries per item");
    if (int32_t st = check(where, logits, d, words, items, in, 1, out, 1)) return st;
    if (top_ids->dtype != B200_I32) return refuse(where, "word numbers must be int32", B200_ERR_UNSUPPORTED);
    if (!is_float(top_logits->dtype)) return refuse(where, "teacher's logits must be f32, f16 or bf16", B200_ERR_UNSUPPORTED);
    if (items == 0) return B200_OK;
    if (!top_ids->ptr || !top_logits->ptr) return refuse(where, "null device pointer");
    for (const b200_matrix* m : {top_ids, top_logits}) {
        if (!aligned(m->ptr, m->dtype)) return refuse(where, "misaligned pointer");
        if ((d->ptr && meet(*d, words, items, *m, top, items)) || meet(out[0], items, 1, *m, top, items))
            return refuse(where, "an output shares memory with the teacher's entries");
    }
    CostP p;
    set_logits(p, logits, d, words, items, weights, cost);
    p.temp = temperature; p.inv_temp = 1.f / temperature; p.c = (float)(1.4426950408889634 / (double)temperature);
    p.ids = top_ids->ptr; p.i0 = top_ids->s0; p.i1 = top_ids->s1;
    p.top = top_logits->ptr; p.t0 = top_logits->s0; p.t1 = top_logits->s1; p.tdt = top_logits->dtype;
    p.K = (int)top;
    return run<false>(where, p, stream, launches);
}

extern "C" b200_status b200_policy(const b200_matrix* logits, const b200_matrix* delta, uint64_t actions,
                                   uint64_t old_logp, uint64_t ref_logp, uint64_t advantages, uint64_t weights,
                                   uint64_t cost, uint64_t logp, int64_t words, int64_t items, float clip_low,
                                   float clip_high, float kl_coef, uint64_t stream, int32_t* launches) {
    const char* where = "b200_policy";
    if (launches) *launches = 0;
    if (!logits) return refuse(where, "null matrix");
    const b200_matrix none = vec(0, logits->dtype), *d = delta ? delta : &none;
    const b200_matrix in[5] = {vec(actions, B200_I32), vec(old_logp, B200_F32), vec(ref_logp, B200_F32),
                               vec(advantages, B200_F32), vec(weights, B200_F32)};
    const b200_matrix out[2] = {vec(cost, B200_F32), vec(logp, B200_F32)};
    if (!(clip_low >= 0.f) || !(clip_high >= 0.f)) return refuse(where, "the clip range must not be negative");
    if (!std::isfinite(kl_coef)) return refuse(where, "the KL coefficient must be finite");
    if (int32_t st = check(where, logits, d, words, items, in, 5, out, 2)) return st;
    if (items == 0) return B200_OK;
    if (!actions || !old_logp || !advantages) return refuse(where, "null device pointer");
    if (kl_coef != 0.f && !ref_logp) return refuse(where, "a KL term needs the reference's log-probabilities");
    CostP p;
    set_logits(p, logits, d, words, items, weights, cost);
    p.temp = p.inv_temp = 1.f; p.c = 1.44269502162933349609375f;
    p.K = 1; p.actions = actions; p.old = old_logp; p.ref = kl_coef != 0.f ? ref_logp : 0; p.adv = advantages; p.logp = logp;
    p.lo = clip_low; p.hi = clip_high; p.kl = kl_coef;
    return run<true>(where, p, stream, launches);
}
