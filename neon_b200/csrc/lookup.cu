// Embedding lookup and its gradient.
//
//     out_fn = scale W_{i_n, f}
//     dW_vf  = beta dW_vf + alpha sum_{n: i_n = v} error_fn
//
// A word number outside the table looks up zeros and collects nothing; the padding word
// (pad_idx) collects nothing.
//
// The gradient is gathered, not scattered: the word numbers are sorted (a stable radix sort of
// (word, position) pairs), and the errors of one word, now neighbours in sorted order, are added
// up by one owner.  No floating-point atomics, so two runs give the same bits, and every element
// of the error is read once and every element of dW written once.  Frequent words of a text hold
// a large share of all positions, so the work is cut into equal chunks of sorted positions, not
// into words: a word inside one chunk is finished there, a word that crosses a border leaves one
// partial sum per chunk, which the last kernel adds in the order of the chunks.

#include "nn_common.cuh"

using namespace nn;

namespace {

enum { kDigitBits = 9, kDigits = 1 << kDigitBits, kTile = 4096, kSortThreads = 256, kSortWarps = kSortThreads / 32,
       kPerWarp = kTile / kSortWarps };

struct LutP {
    u64 ids, w, out;
    i64 w0, w1, o0, o1;
    int dt, V;
    i64 F, N;
    float scale;
};

__global__ void __launch_bounds__(256) lut_fprop_any(const __grid_constant__ LutP p) {
    for (i64 n = blockIdx.x; n < p.N; n += gridDim.x) {
        const int id = reinterpret_cast<const int*>(p.ids)[n];
        const bool in = id >= 0 && id < p.V;
        for (i64 f = threadIdx.x; f < p.F; f += blockDim.x)
            st_any(p.out, f * p.o0 + n * p.o1, p.dt, in ? ld_any(p.w, id * p.w0 + f * p.w1, p.dt) * p.scale : 0.f);
    }
}

// ------------------------------------------------------------------ sort of (word, position)
struct SortP {
    const int *ids;                       // first pass: the word numbers as given
    const int *key_in, *pos_in;           // later passes
    int *key_out, *pos_out, *hist;        // hist[digit][tile]
    int N, V, pad, tiles, shift, first;
};

// The sort key of a word number: itself, or V for one that collects nothing.
DEV int sort_key(const SortP& p, int i) {
    if (!p.first) return p.key_in[i];
    const int id = p.ids[i];
    return id < 0 || id >= p.V || id == p.pad ? p.V : id;
}

__global__ void __launch_bounds__(kSortThreads) sort_count(const __grid_constant__ SortP p) {
    __shared__ int c[kDigits];
    for (int i = threadIdx.x; i < kDigits; i += kSortThreads) c[i] = 0;
    __syncthreads();
    const int base = blockIdx.x * kTile;
    for (int i = base + threadIdx.x; i < base + kTile && i < p.N; i += kSortThreads)
        atomicAdd(&c[(sort_key(p, i) >> p.shift) & (kDigits - 1)], 1);
    __syncthreads();
    for (int i = threadIdx.x; i < kDigits; i += kSortThreads) p.hist[i * p.tiles + blockIdx.x] = c[i];
}

// Exclusive prefix sums of `count` numbers, in place, by one block.
__global__ void __launch_bounds__(1024) sort_scan(int* a, int count) {
    __shared__ int s[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per = (count + 1023) / 1024, lo = min((int)threadIdx.x * per, count), hi = min(lo + per, count);
    int sum = 0;
    for (int i = lo; i < hi; ++i) sum += a[i];
    int x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) s[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int y = s[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += t;
        }
        s[lane] = y;
    }
    __syncthreads();
    int at = x - sum + (warp ? s[warp - 1] : 0);
    for (int i = lo; i < hi; ++i) { const int v = a[i]; a[i] = at; at += v; }
}

// Moves a tile to its places.  A warp takes 512 neighbouring pairs, 32 at a time in their order;
// lanes with the same digit find each other with match_any, so equal digits keep their order.
__global__ void __launch_bounds__(kSortThreads) sort_move(const __grid_constant__ SortP p) {
    __shared__ int c[kSortWarps][kDigits];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&c[0][0])[i] = 0;
    __syncthreads();
    constexpr int R = kPerWarp / 32;
    int key[R], rank[R];
    const int base = blockIdx.x * kTile + warp * kPerWarp;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = base + r * 32 + lane;
        const bool in = i < p.N;
        key[r] = in ? sort_key(p, i) : 0;
        const int d = in ? (key[r] >> p.shift) & (kDigits - 1) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        const int leader = __ffs(peers) - 1;
        int before = 0;
        if (lane == leader && in) {
            before = c[warp][d];
            c[warp][d] = before + __popc(peers);
        }
        before = __shfl_sync(0xffffffffu, before, leader);
        rank[r] = before + __popc(peers & ((1u << lane) - 1));
        __syncwarp();
    }
    __syncthreads();
    for (int d = threadIdx.x; d < kDigits; d += kSortThreads) {
        int at = p.hist[d * p.tiles + blockIdx.x];
#pragma unroll
        for (int w = 0; w < kSortWarps; ++w) { const int v = c[w][d]; c[w][d] = at; at += v; }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = base + r * 32 + lane;
        if (i >= p.N) continue;
        const int to = c[warp][(key[r] >> p.shift) & (kDigits - 1)] + rank[r];
        p.key_out[to] = key[r];
        p.pos_out[to] = p.first ? i : p.pos_in[i];
    }
}

// start[v] = first sorted place whose word is at least v, for v in 0 .. V
__global__ void __launch_bounds__(256) sort_starts(const int* key, int N, int* start, int V) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v > V) return;
    int lo = 0, hi = N;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (key[mid] < v) lo = mid + 1; else hi = mid;
    }
    start[v] = lo;
}

// ------------------------------------------------------------------ sums
struct SumP {
    const int *key, *pos, *start;
    u64 e, w;
    i64 e0, e1, w0, w1;
    int edt, wdt, V;
    i64 F, L;                             // L sorted places per chunk
    float* part;                          // [chunk][2][F]: 0 continues an earlier chunk, 1 begins here and goes on
    float alpha, beta;
};

DEV void put_dw(const SumP& p, int v, i64 f, float sum) {
    const i64 at = v * p.w0 + f * p.w1;
    float r = p.alpha * sum;
    if (p.beta != 0.f) r += p.beta * ld_any(p.w, at, p.wdt);
    st_any(p.w, at, p.wdt, r);
}

__global__ void __launch_bounds__(256) lut_chunks_any(const __grid_constant__ SumP p) {
    const int used = p.start[p.V];
    const i64 f = (i64)blockIdx.y * 256 + threadIdx.x;
    const i64 lo = (i64)blockIdx.x * p.L;
    const i64 hi = lo + p.L < used ? lo + p.L : used;
    if (lo >= used || f >= p.F) return;
    float sum = 0.f;
    int v = p.key[lo];
    for (i64 i = lo; i < hi; ++i) {
        sum += ld_any(p.e, f * p.e0 + p.pos[i] * p.e1, p.edt);
        const int next = i + 1 < hi ? p.key[i + 1] : -1;
        if (next == v) continue;
        const bool from_before = p.start[v] < lo, goes_on = p.start[v + 1] > hi;
        if (from_before || goes_on) p.part[((i64)blockIdx.x * 2 + (from_before ? 0 : 1)) * p.F + f] = sum;
        else put_dw(p, v, f, sum);
        sum = 0.f;
        v = next;
    }
}

// Words without a position, and words that cross a border between chunks.
__global__ void __launch_bounds__(256) lut_finish_any(const __grid_constant__ SumP p) {
    for (i64 v = blockIdx.x; v < p.V; v += gridDim.x) {
        const int lo = p.start[v], hi = p.start[v + 1];
        if (lo == hi) {
            if (p.beta != 1.f)
                for (i64 f = threadIdx.x; f < p.F; f += 256) {
                    const i64 at = v * p.w0 + f * p.w1;
                    st_any(p.w, at, p.wdt, p.beta == 0.f ? 0.f : p.beta * ld_any(p.w, at, p.wdt));
                }
            continue;
        }
        const i64 c0 = lo / p.L, c1 = (hi - 1) / p.L;
        if (c0 == c1) continue;
        for (i64 f = threadIdx.x; f < p.F; f += 256) {
            float sum = p.part[(c0 * 2 + 1) * p.F + f];
            for (i64 c = c0 + 1; c <= c1; ++c) sum += p.part[c * 2 * p.F + f];
            put_dw(p, (int)v, f, sum);
        }
    }
}

unsigned blocks_for(i64 n) { return (unsigned)(n < 65536 ? n : 65536); }

// Where the pieces of the gradient's scratch lie.
struct Plan {
    i64 tiles, chunks, L, passes, key[2], pos[2], hist, start, part, bytes;
};
enum : i64 { kPartBytes = 32ll << 20 };       // partial sums are held to about this much

Plan plan(i64 V, i64 F, i64 N) {
    Plan q;
    q.tiles = (N + kTile - 1) / kTile;
    q.passes = 1;
    while ((V >> (kDigitBits * q.passes)) != 0) ++q.passes;
    // chunks of 64 places (512 bytes of partials per column against 64 elements read), longer
    // where the partial sums would outgrow their share of the scratch
    q.L = 64;
    while ((N + q.L - 1) / q.L * 8 * F > kPartBytes && q.L < N) q.L *= 2;
    q.chunks = (N + q.L - 1) / q.L;
    i64 at = 0;
    auto take = [&at](i64 bytes) { const i64 r = at; at += (bytes + 255) & ~255ll; return r; };
    for (int k = 0; k < 2; ++k) { q.key[k] = take(4 * N); q.pos[k] = take(4 * N); }
    q.hist = take(4 * kDigits * q.tiles);
    q.start = take(4 * (V + 1));
    q.part = take(8 * F * q.chunks);
    q.bytes = at;
    return q;
}

int32_t check_sizes(const char* where, i64 V, i64 F, i64 N) {
    if (V < 1 || V >= 0x7fffffff) return refuse(where, "between 1 and 2^31 - 2 words");
    if (F < 1 || F > 65535 * 256) return refuse(where, "between 1 and 65535 * 256 features");
    if (N < 0 || N > 0x7fffffff - kTile) return refuse(where, "fewer than 2^31 - 4096 positions");
    return B200_OK;
}
b200_matrix vec(uint64_t ptr, int dt) { b200_matrix m; m.ptr = ptr; m.s0 = 1; m.s1 = 1; m.dtype = dt; m.reserved = 0; return m; }

}  // namespace

extern "C" b200_status b200_lut_fprop(uint64_t ids, const b200_matrix* table, const b200_matrix* out, int64_t words,
                                      int64_t features, int64_t positions, float scale, uint64_t stream) {
    const char* where = "b200_lut_fprop";
    if (!table || !out) return refuse(where, "null matrix");
    if (int32_t st = check_sizes(where, words, features, positions)) return st;
    if (!is_float(table->dtype) || out->dtype != table->dtype)
        return refuse(where, "only f32, f16 and bf16, the same for table and result", B200_ERR_UNSUPPORTED);
    if (positions == 0) return B200_OK;
    if (!ids || !table->ptr || !out->ptr) return refuse(where, "null device pointer");
    if (!aligned(table->ptr | out->ptr, table->dtype) || !aligned(ids, B200_I32)) return refuse(where, "misaligned pointer");
    if (meet(*out, features, positions, *table, words, features) || meet(*out, features, positions, vec(ids, B200_I32), positions, 1))
        return refuse(where, "the result shares memory with the table or the word numbers");
    DeviceScope scope;
    if (scope.error() != cudaSuccess) return cuda_status(where, scope.error());
    cudaStream_t s = static_cast<cudaStream_t>(b200_detail_stream(stream));
    LutP p;
    p.ids = ids; p.w = table->ptr; p.out = out->ptr;
    p.w0 = table->s0; p.w1 = table->s1; p.o0 = out->s0; p.o1 = out->s1;
    p.dt = table->dtype; p.V = (int)words; p.F = features; p.N = positions; p.scale = scale;
    lut_fprop_any<<<blocks_for(positions), 256, 0, s>>>(p);
    return cuda_status(where, cudaGetLastError());
}

extern "C" uint64_t b200_lut_bprop_scratch_bytes(int64_t words, int64_t features, int64_t positions) {
    if (words < 1 || features < 1 || positions < 1) return 0;
    return (uint64_t)plan(words, features, positions).bytes;
}

extern "C" b200_status b200_lut_bprop(uint64_t ids, const b200_matrix* error, const b200_matrix* dtable, int64_t words,
                                      int64_t features, int64_t positions, int64_t pad_idx, float alpha, float beta,
                                      uint64_t scratch, uint64_t scratch_bytes, uint64_t stream, int32_t* launches) {
    const char* where = "b200_lut_bprop";
    if (launches) *launches = 0;
    if (!error || !dtable) return refuse(where, "null matrix");
    if (int32_t st = check_sizes(where, words, features, positions)) return st;
    if (!is_float(error->dtype) || !is_float(dtable->dtype)) return refuse(where, "only f32, f16 and bf16", B200_ERR_UNSUPPORTED);
    if (!dtable->ptr || (positions && (!ids || !error->ptr))) return refuse(where, "null device pointer");
    if (!aligned(dtable->ptr, dtable->dtype) || !aligned(error->ptr, error->dtype) || !aligned(ids, B200_I32))
        return refuse(where, "misaligned pointer");
    if (positions && (meet(*dtable, words, features, *error, features, positions) ||
                      meet(*dtable, words, features, vec(ids, B200_I32), positions, 1)))
        return refuse(where, "the gradient shares memory with the error or the word numbers");
    const Plan q = plan(words, features, positions);
    if (!scratch || scratch % 256 || scratch_bytes < (uint64_t)q.bytes) return refuse(where, "scratch too small or misaligned");
    DeviceScope scope;
    if (scope.error() != cudaSuccess) return cuda_status(where, scope.error());
    cudaStream_t s = static_cast<cudaStream_t>(b200_detail_stream(stream));
    char* base = reinterpret_cast<char*>(scratch);
    auto ints = [base](i64 off) { return reinterpret_cast<int*>(base + off); };
    int count = 0, from = 0;
    SortP t;
    t.ids = reinterpret_cast<const int*>(ids); t.hist = ints(q.hist);
    t.N = (int)positions; t.V = (int)words; t.tiles = (int)q.tiles;
    t.pad = pad_idx < 0 || pad_idx >= words ? -1 : (int)pad_idx;
    for (int k = 0; positions && k < q.passes; ++k) {
        t.first = k == 0; t.shift = k * kDigitBits;
        t.key_in = ints(q.key[from]); t.pos_in = ints(q.pos[from]);
        t.key_out = ints(q.key[1 - from]); t.pos_out = ints(q.pos[1 - from]);
        sort_count<<<(unsigned)q.tiles, kSortThreads, 0, s>>>(t);
        sort_scan<<<1, 1024, 0, s>>>(t.hist, (int)(kDigits * q.tiles));
        sort_move<<<(unsigned)q.tiles, kSortThreads, 0, s>>>(t);
        from = 1 - from;
        count += 3;
    }
    SumP p;
    p.key = ints(q.key[from]); p.pos = ints(q.pos[from]); p.start = ints(q.start);
    p.e = error->ptr; p.e0 = error->s0; p.e1 = error->s1; p.edt = error->dtype;
    p.w = dtable->ptr; p.w0 = dtable->s0; p.w1 = dtable->s1; p.wdt = dtable->dtype;
    p.V = (int)words; p.L = q.L; p.F = features; p.part = reinterpret_cast<float*>(base + q.part);
    p.alpha = alpha; p.beta = beta;
    sort_starts<<<(unsigned)((words + 256) / 256), 256, 0, s>>>(p.key, (int)positions, ints(q.start), (int)words);
    ++count;
    if (positions) {
        lut_chunks_any<<<dim3((unsigned)q.chunks, (unsigned)((features + 255) / 256)), 256, 0, s>>>(p);
        ++count;
    }
    lut_finish_any<<<blocks_for(words), 256, 0, s>>>(p);
    if (launches) *launches = count + 1;
    return cuda_status(where, cudaGetLastError());
}
