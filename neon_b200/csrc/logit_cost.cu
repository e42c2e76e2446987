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
// Both read every logit for the softmax and then touch K (or one) of them again.  Exponentials are
// taken in base 2 of differences to the largest logit m, 2^((z_v - m) c) with c = log2(e) / T, so
// nothing overflows whatever the logits' offset; s is their sum, q_v = 2^((z_v - m) c) / s.
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

// What an item's gradient needs besides the logits: delta_v = scale 2^((z_v - m) c) for the words
// without an entry of their own; 0 for all if dead.
struct Item { float m, scale; int dead; };

// One item's entries: word, log-probability at the teacher's (-inf: no entry), student's logit.
struct Entries { int* id; float* lp; float* z; };

DEV float weight_of(const CostP& p, i64 n) { return p.weights ? reinterpret_cast<const float*>(p.weights)[n] : 1.f; }

// Items that need not be looked at: their cost and delta are zero.
template <bool POLICY> DEV bool skipped(const CostP& p, i64 n) {
    if (weight_of(p, n) == 0.f && !(POLICY && p.logp)) return true;
    if (POLICY) {
        const int a = reinterpret_cast<const int*>(p.actions)[n];
        return a < 0 || a >= p.V;
    }
    return false;
}
template <bool POLICY> DEV void put_skipped(const CostP& p, i64 n) {
    reinterpret_cast<float*>(p.cost)[n] = 0.f;
    if (POLICY && p.logp) reinterpret_cast<float*>(p.logp)[n] = 0.f;
}

// The maximum of a running softmax as the exponentials use it: items (or parts of one) that hold
// nothing but -inf so far take differences to 0, which leaves their exponentials at 0 and a NaN a NaN.
DEV float usable(float m) { return m == -INFINITY ? 0.f : m; }
DEV float exp_of(float z, float m, float c) { return ex2_approx((z - m) * c); }
// Teacher's entries of one item, by one warp: words, log-probabilities, and the student's logits
// there.  Nothing here needs the student's softmax.
DEV void read_entries(const CostP& p, i64 n, const Entries& e) {
    const int lane = threadIdx.x & 31;
    float top = -INFINITY;
    for (int k = lane; k < p.K; k += 32) {
        const int id = *(reinterpret_cast<const int*>(p.ids) + k * p.i0 + n * p.i1);
        const float t = ld_any(p.top, k * p.t0 + n * p.t1, p.tdt);
        const bool used = id >= 0 && id < p.V && t != -INFINITY;
        e.id[k] = used ? id : -1;
        e.lp[k] = t;
        e.z[k] = used ? ld_any(p.z, (i64)id * p.z0 + n * p.z1, p.dt) : 0.f;
        if (used) top = fmaxf(top, t);
    }
    top = usable(warp_max(top));                       // (a NaN reaches the sum whatever the maximum says)
    float sum = 0.f;
    for (int k = lane; k < p.K; k += 32)
        if (e.id[k] >= 0) sum += expf((e.lp[k] - top) * p.inv_temp);
    const float ln_sum = logf(warp_sum(sum));
    for (int k = lane; k < p.K; k += 32) e.lp[k] = e.id[k] >= 0 ? (e.lp[k] - top) * p.inv_temp - ln_sum : -INFINITY;
}

// The item's cost, by one warp (all lanes), from its entries and its logits' maximum and sum.
DEV Item distill_item(const CostP& p, i64 n, float m, float s, const Entries& e) {
    const float w = weight_of(p, n), ln_s = logf(s);
    float cost = 0.f;
    int any = 0;
    for (int k = threadIdx.x & 31; k < p.K; k += 32) {
        if (e.id[k] < 0) continue;
        any = 1;
        const float lp = e.lp[k], pk = expf(lp);
        if (pk != 0.f) cost += pk * (lp - ((e.z[k] - m) * p.inv_temp - ln_s));
    }
    cost = warp_sum(cost);
    any = __any_sync(0xffffffffu, any);
    Item it;
    it.m = usable(m);
    it.dead = w == 0.f || !any;
    it.scale = w * p.temp / s;
    if ((threadIdx.x & 31) == 0) reinterpret_cast<float*>(p.cost)[n] = it.dead ? 0.f : w * p.temp * p.temp * cost;
    return it;
}
// The gradient at an entry's word: a word listed more than once collects all its entries, so each
// of them holds the same value.
DEV float entry_delta(const CostP& p, const Item& it, float w, const Entries& e, int k) {
    const int id = e.id[k];
    float mass = 0.f;
    for (int j = 0; j < p.K; ++j) if (e.id[j] == id) mass += expf(e.lp[j]);
    return it.scale * exp_of(e.z[k], it.m, p.c) - w * p.temp * mass;
}

// Policy: cost and log-probability of one item; `at_word`: the gradient at the word chosen.
DEV Item policy_item(const CostP& p, i64 n, float m, float s, float za, bool put, float& at_word) {
    const float w = weight_of(p, n), l = (za - m) - logf(s);
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
    Item it;
    it.m = usable(m);
    it.dead = w == 0.f;
    it.scale = -slope / s;
    at_word = fmaf(it.scale, exp_of(za, it.m, p.c), slope);
    if (put) {
        reinterpret_cast<float*>(p.cost)[n] = it.dead ? 0.f : w * cost;
        if (p.logp) reinterpret_cast<float*>(p.logp)[n] = l;
    }
    return it;
}

// ---- any strides, and words next to each other (their stride is 1)
//
// A block per item, items from a persistent grid.  The first walk over the logits keeps a running
// maximum and sum per thread (rescaled when a group of vectors holds a larger logit, which is rare
// after the first), the second writes the gradient.  The second read comes from L2: the rows under
// way, at most 512 KB times the blocks that fit on the GPU, stay there, so HBM sees one read and
// one write.  Meanwhile one warp reads the teacher's entries.  DT >= 0: 16-byte vectors, the first of which starts at
// the boundary at or before the row; DT < 0: one logit at a time with any strides.
template <int DT> struct Words {                       // loads and stores of one vector of a row
    static constexpr int V = 16 / dt_size<DT>::value;
    u32 w[4];
    DEV void load(const CostP& p, i64 row, int f) {
        ld_w<DT, V, false>(p.z, row + f, w);
        if (f < 0 || f + V > p.V) {                    // -inf where there is no word
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if ((unsigned)(f + i) < (unsigned)p.V) continue;
                if constexpr (DT == F32) w[i] = 0xff800000u;
                else {
                    const u32 low = DT == F16 ? 0xfc00u : 0xff80u;
                    w[i >> 1] = i & 1 ? (w[i >> 1] & 0xffffu) | low << 16 : (w[i >> 1] & 0xffff0000u) | low;
                }
            }
        }
    }
};
// the largest of four vectors' elements (NaN is passed over)
DEV u32 max_pair(u32 a, u32 b, int dt) {
    u32 r;
    if (dt == F16) asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <int DT, int U> DEV float top_of(const Words<DT> (&x)[U]) {
    if constexpr (DT == F32) {
        float m = __uint_as_float(x[0].w[0]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) m = fmaxf(m, __uint_as_float(x[u].w[i]));
        return m;
    } else {
        u32 m = x[0].w[0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) m = max_pair(m, x[u].w[i], DT);
        float lo, hi;
        split(get2<DT>(&m, 0), lo, hi);
        return fmaxf(lo, hi);
    }
}

template <bool POLICY, int DT>
__global__ void __launch_bounds__(512) cost_rows(const __grid_constant__ CostP p) {
    constexpr bool VEC = DT >= 0;
    constexpr int D = VEC ? DT : 0, V = VEC ? 16 / dt_size<D>::value : 1, U = 4;
    // [2][3][K], and below [2][32]: an item's are read and written while others use the last one's;
    // the barrier of the item in between keeps two uses of one half apart
    extern __shared__ float entries[];
    __shared__ float2 red[64];
    const int tid = threadIdx.x, T = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = T >> 5;
    int turn = 0;
    for (i64 n = blockIdx.x; n < p.N; n += gridDim.x) {
        const bool skip = skipped<POLICY>(p, n);
        Item it;
        float za = 0.f, at_word = 0.f;
        const i64 row = n * p.z1, drow = n * p.d1;
        int mis = 0, nvec = p.V;
        if constexpr (VEC) {
            mis = (int)((p.z / dt_size<D>::value + (u64)row) % V);
            nvec = (p.V + mis + V - 1) / V;
        }
        Entries e;
        e.id = reinterpret_cast<int*>(entries) + turn * 3 * p.K;
        e.lp = entries + (turn * 3 + 1) * p.K;
        e.z = entries + (turn * 3 + 2) * p.K;
        if (skip) {
            it.dead = 1;
            if (tid == 0) put_skipped<POLICY>(p, n);
        } else {
            if (POLICY) za = ld_any(p.z, reinterpret_cast<const int*>(p.actions)[n] * p.z0 + row, p.dt);
            else if (warp == 0) read_entries(p, n, e);
            float m = -INFINITY, s = 0.f;
            if constexpr (VEC) {
                f32x2 sum = 0;
                const f32x2 c2 = pair(p.c, p.c);
                for (int k0 = tid; k0 < nvec; k0 += T * U) {
                    Words<D> x[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (k0 + u * T < nvec) x[u].load(p, row, (k0 + u * T) * V - mis);
                        else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) x[u].w[i] = D == F32 ? 0xff800000u : D == F16 ? 0xfc00fc00u : 0xff80ff80u;
                        }
                    }
                    const float top = top_of<D, U>(x);
                    if (top > m) {
                        const float f = exp_of(m, top, p.c);
                        sum = mul2(sum, pair(f, f));
                        m = top;
                    }
                    const float t = usable(m);
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int i = 0; i < V / 2; ++i) {
                            float lo, hi;
                            split(mul2(less2<D>(x[u].w, i, t), c2), lo, hi);
                            sum = add2(sum, pair(ex2_approx(lo), ex2_approx(hi)));
                        }
                }
                s = both(sum);
            } else {
                for (int v = tid; v < p.V; v += T) {
                    const float z = ld_any(p.z, v * p.z0 + row, p.dt);
                    if (z > m) { s *= exp_of(m, z, p.c); m = z; }
                    s += exp_of(z, usable(m), p.c);
                }
            }
            // one maximum and sum for the block
            const float top = warp_max(m);
            s = warp_sum(s * exp_of(m, usable(top), p.c));
            if (lane == 0) red[turn * 32 + warp] = make_float2(top, s);
            __syncthreads();
            const float2 part = lane < warps ? red[turn * 32 + lane] : make_float2(-INFINITY, 0.f);
            m = warp_max(part.x);
            s = warp_sum(part.y * exp_of(part.x, usable(m), p.c));
            turn ^= 1;
            if (POLICY) it = policy_item(p, n, m, s, za, tid == 0, at_word);
            else {
                if (warp == 0) it = distill_item(p, n, m, s, e);
                if (p.d) {
                    // what all need for the gradient, without waiting for the cost
                    const float w = weight_of(p, n);
                    int any = 0;
                    for (int k = lane; k < p.K; k += 32) any |= e.id[k] >= 0;
                    it.m = usable(m);
                    it.dead = w == 0.f || !__any_sync(0xffffffffu, any);
                    it.scale = w * p.temp / s;
                }
            }
        }
        if (!p.d) continue;
        if constexpr (VEC) {
            const f32x2 c2 = pair(p.c, p.c), scale = pair(it.scale, it.scale);
            for (int k0 = tid; k0 < nvec; k0 += T * U) {
                Words<D> x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (k0 + u * T >= nvec || it.dead) x[u].w[0] = x[u].w[1] = x[u].w[2] = x[u].w[3] = 0;
                    else ld_w<D, V, false>(p.z, row + (k0 + u * T) * V - mis, x[u].w);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (k0 + u * T >= nvec) break;
                    if (!it.dead) {
#pragma unroll
                        for (int i = 0; i < V / 2; ++i) {
                            float lo, hi;
                            split(mul2(less2<D>(x[u].w, i, it.m), c2), lo, hi);
                            set2<D>(x[u].w, i, mul2(scale, pair(ex2_approx(lo), ex2_approx(hi))));
                        }
                    }
                    put_part<D, V>(p.d, drow, (k0 + u * T) * V - mis, p.V, x[u].w);
                }
            }
        } else {
            for (int v = tid; v < p.V; v += T)
                st_any(p.d, v * p.d0 + drow, p.dt, it.dead ? 0.f : it.scale * exp_of(ld_any(p.z, v * p.z0 + row, p.dt), it.m, p.c));
        }
        __syncthreads();                               // the entries' words have been written with the others
        if (it.dead) continue;
        if (POLICY) {
            if (tid == 0) st_any(p.d, reinterpret_cast<const int*>(p.actions)[n] * p.d0 + drow, p.dt, at_word);
        } else {
            const float w = weight_of(p, n);
            for (int k = tid; k < p.K; k += T)
                if (e.id[k] >= 0) st_any(p.d, e.id[k] * p.d0 + drow, p.dt, entry_delta(p, it, w, e, k));
        }
    }
}

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

template <bool POLICY, int DT> cudaError_t launch_rows(const CostP& p, cudaStream_t s) {
    constexpr int V = DT >= 0 ? 16 / dt_size<DT >= 0 ? DT : 0>::value : 1;
    // as many threads as have two vectors each, up to 512
    const i64 pairs = ((i64)p.V + 2 * V - 1) / (2 * V);
    const int T = pairs >= 512 ? 512 : (int)(pairs + 31) / 32 * 32, smem = POLICY ? 0 : 6 * p.K * 4;
    const i64 most = resident_blocks(cost_rows<POLICY, DT>, T, smem);
    if (!most) return cudaErrorInvalidConfiguration;
    cost_rows<POLICY, DT><<<(unsigned)(p.N < most ? p.N : most), T, smem, s>>>(p);
    return cudaGetLastError();
}

template <bool POLICY>
int32_t run(const char* where, CostP& p, uint64_t stream, int32_t* launches) {
    DeviceScope scope;
    if (scope.error() != cudaSuccess) return cuda_status(where, scope.error());
    cudaStream_t s = static_cast<cudaStream_t>(b200_detail_stream(stream));
    // vectors: words next to each other, and logits and delta alike to the 16-byte boundaries
    const int V = 16 / (int)esize(p.dt);
    const bool rows = (p.z0 == 1 || p.V == 1) &&
        (!p.d || ((p.d0 == 1 || p.V == 1) && (p.z - p.d) % 16 == 0 && (p.z1 - p.d1) % V == 0));
    cudaError_t e;
    if (!rows) e = launch_rows<POLICY, -1>(p, s);
    else if (p.dt == B200_F32) e = launch_rows<POLICY, F32>(p, s);
    else if (p.dt == B200_F16) e = launch_rows<POLICY, F16>(p, s);
    else e = launch_rows<POLICY, BF16>(p, s);
    if (launches) *launches = 1;
    return cuda_status(where, e);
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
