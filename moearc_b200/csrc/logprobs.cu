// logprobs.cu — log probabilities of given tokens under rows of logits, with each row's entropy and
// its k likeliest tokens, in one pass over the logits.
//
// With x = scale logit, M = max x, L = sum e^(x - M) and S = sum e^(x - M) (x - M):
//
//   logprob(t) = (x_t - M) - log L,      entropy = log L - S / L,
//
// Measured: 2047 rows of 100003 bf16, k 5, 432 MB of logits: 86 us (5.0 TB/s; 62 at the measured copy
// rate); 64 rows of 200019 f32, k 20: 18.9 us, of which the stream is 8; one row of 131072 f32, k 8: 7 us.
//
// Both results come from running (M, L, S) triples, joined as S' = f (S + (m - M) L) with f = e^(m - M) when the
// maximum moves from m to M. The pass reads each logit once and is bound by HBM; for 16-bit logits the
// exponentials (16 a clock and SM) come close behind.
//
// A row is one CTA, or a cluster of up to 16 where there are too few rows to fill the GPU; the
// cluster's CTAs write what they found into the first one's shared memory, so there is no second
// kernel and no workspace, and the order of the sums depends on the sizes alone.
//
// The k likeliest: a thread's running maximum is the largest of the elements it read, so the k-th
// largest of a CTA's thread maxima is a bound that k elements reach. Only the elements of threads
// at or above it (about k of 256 threads) are read again, from L2, all at once, and those that
// reach the bound are ranked by counting. Should more reach it than the list holds (equal values), the k-th of the
// listed ones becomes the next bound. A key is the value's bits in order, then the complement of
// the index: no two are equal, and ties go to the lowest index.
#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>

#include "kvcache.cuh"

namespace cg = cooperative_groups;
using namespace moearc;

namespace {

constexpr int MAX_K = MAX_TOPK, LIST = 512;
// Threads a CTA: 128 where there are more rows than SMs hold such CTAs (about 8 an SM) and they are
// short, so that what follows a row's pass is hidden by more rows; else 256, for a row's own speed.
// 3000 rows of 8000 f32: 44 us with 256, 29 with 128; 600 of 32000 bf16: 17 and 24; 2047 of 100003
// bf16: 83 and 91.
constexpr size_t SHORT_ROW = 100 << 10;
constexpr float LOG2E = 1.4426950408889634f;

typedef unsigned long long u64;

struct lp_args {
    const void *logits;
    const unsigned *tokens;
    size_t row_stride;
    unsigned n_vocab, k;
    float scale;
    float *logprob, *entropy, *top_lp;
    unsigned *top_id;
};

// 2^x, subnormal results as 0.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

struct triple {
    float m, l, s;
};
// a and b joined; the smaller maximum's sums are moved to the larger. An empty side (m -inf, l 0)
// adds nothing; a NaN sum stays.
__device__ __forceinline__ triple join(triple a, triple b) {
    triple r;
    r.m = fmaxf(a.m, b.m);
    if (r.m == -INFINITY) return triple{-INFINITY, a.l + b.l, a.s + b.s};
    const float da = fmaxf(a.m - r.m, -200.f), db = fmaxf(b.m - r.m, -200.f);
    const float fa = ex2(da * LOG2E), fb = ex2(db * LOG2E);
    r.l = a.l * fa + b.l * fb;
    r.s = fa * fmaf(da, a.l, a.s) + fb * fmaf(db, b.l, b.s);
    return r;
}

// Values in order as unsigned bits; a NaN ranks with -inf, -0 with +0.
__device__ __forceinline__ u64 key_of(float x, unsigned i) {
    const float v = x != x ? -INFINITY : x + 0.f;
    const unsigned b = __float_as_uint(v);
    return (u64)(b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u)) << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float value_of(u64 key) {
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}

template <typename T>
struct vec {
    static constexpr int N = 16 / sizeof(T);
    float v[N];
};
__device__ __forceinline__ uint4 ld16(const void *p) {
    uint4 u;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
    return u;
}
template <typename T>
__device__ __forceinline__ void unpack(uint4 u, float *v) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        } else {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ float one(const float *p) { return *p; }
__device__ __forceinline__ float one(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ float one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mul.rn.f32x2 z, x, y; mov.b64 {%0, %1}, z; }" : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ void fma2(float2 &d, float2 a, float2 b) {
    asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%0, %1}; fma.rn.f32x2 z, x, y, z; mov.b64 {%0, %1}, z; }"
        : "+f"(d.x), "+f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
}

// N logits, unscaled, into a running triple of unscaled m and s: one look at the maximum for all of
// them, then two at a time. scale2: scale x log2(e).
template <int N>
__device__ __forceinline__ void take(triple &r, const float (&x)[N], float scale2) {
    float b = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) b = fmaxf(b, x[i]);
    if (b > r.m) {
        if (r.m != -INFINITY) {
            const float d = fmaxf(r.m - b, -FLT_MAX), f = ex2(d * scale2);
            r.s = f * r.s + (f * d) * r.l;
            r.l *= f;
        }
        r.m = b;
    }
    const float base = r.m == -INFINITY ? 0.f : r.m;
    const float2 mb = make_float2(-base, -base), sc = make_float2(scale2, scale2);
    float2 l = make_float2(0.f, 0.f), t = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) {
        // the floor keeps 0 x -inf out of S: a weight that far down is 0 at any scale allowed
        float2 d = add2(make_float2(x[i], x[i + 1]), mb);
        d.x = max_nan(d.x, -FLT_MAX);
        d.y = max_nan(d.y, -FLT_MAX);
        float2 e = mul2(d, sc);
        e.x = ex2(e.x);
        e.y = ex2(e.y);
        l = add2(l, e);
        fma2(t, e, d);
    }
    if constexpr (N & 1) {
        const float d = max_nan(x[N - 1] - base, -FLT_MAX), e = ex2(d * scale2);
        l.x += e;
        t.x = fmaf(e, d, t.x);
    }
    r.l += l.x + l.y;
    r.s += t.x + t.y;
}

// The CTA's run [c0, c1) of a row: single elements up to a 16-byte boundary, whole vectors, the
// rest. Thread t reads element t of the first and last, vectors t, t + TH, ...
template <typename T>
struct run {
    const T *row;
    unsigned c0, head, nv, c1;
    __device__ run(const T *r, unsigned a, unsigned b) : row(r), c0(a), c1(b) {
        constexpr int V = vec<T>::N;
        const unsigned off = (unsigned)(reinterpret_cast<uintptr_t>(r + a) & 15) / sizeof(T);
        head = min((V - off) % V, c1 - c0);
        nv = (c1 - c0 - head) / V;
    }
    __device__ unsigned body() const { return c0 + head; }
    __device__ unsigned tail() const { return body() + nv * vec<T>::N; }
};

template <int TH>
struct shared_lists {
    static constexpr int WARPS = TH / 32;
    triple part[WARPS];
    float warp_bound[WARPS];
    __align__(16) float max_v[TH];
    unsigned max_t[TH], sub[TH];
    unsigned n_max, n_sub, n_list;
    float bound;
    __align__(16) u64 list[LIST + 2];
    // what the cluster's CTAs found, in the first one's copy: keys largest first, 0 past the last
    triple whole[16];
    __align__(16) u64 top[16][MAX_K];
    u64 best[MAX_K];
};

// The largest k of list[0, n) in order into top, 0 past the last; rank by counting. n is even (a
// 0 fills up an odd one).
template <int TH>
__device__ void rank_list(const u64 *list, unsigned n, unsigned k, u64 *top) {
    const auto *two = reinterpret_cast<const ulonglong2 *>(list);
    for (unsigned i = threadIdx.x; i < n; i += TH) {
        const u64 key = list[i];
        unsigned rank = 0;
#pragma unroll 4
        for (unsigned j = 0; j < n / 2; ++j) {
            const ulonglong2 v = two[j];
            rank += (v.x > key) + (v.y > key);
        }
        if (rank < k && key) top[rank] = key;
    }
}

// The largest min(k, elements) keys of the CTA's run, in order, into top, 0 past the last; m: the
// thread's maximum, scaled.
template <int TH, typename T>
__device__ void top_of_run(const run<T> &R, float m, float scale, unsigned k, shared_lists<TH> &sh, u64 *top) {
    constexpr int V = vec<T>::N, WARPS = TH / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // a first bound: each warp has ceil(k / WARPS) lanes at or above its own, so k threads of the
    // CTA are at or above the least of them (as ordered bits, for the warp's maximum in one step)
    unsigned v = (unsigned)(key_of(m, 0) >> 32), last = v;
    for (unsigned q = 0; q < (k + WARPS - 1) / WARPS; ++q) {
        last = __reduce_max_sync(0xffffffffu, v);
        const unsigned who = __ballot_sync(0xffffffffu, v == last);
        if (lane == __ffs(who) - 1) v = 0;
    }
    if (lane == 0) sh.warp_bound[warp] = value_of((u64)last << 32);
    if (threadIdx.x == 0) sh.n_max = sh.n_sub = 0;
    sh.max_v[threadIdx.x] = -INFINITY;
    __syncthreads();
    float bound = sh.warp_bound[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) bound = fminf(bound, sh.warp_bound[w]);
    if (m >= bound) {
        const unsigned i = atomicAdd(&sh.n_max, 1u);
        sh.max_v[i] = m;
        sh.max_t[i] = threadIdx.x;
    }
    __syncthreads();
    // the k-th largest of the listed maxima: fewer than k above it, at least k at or above
    const unsigned n_max = sh.n_max;
    if (threadIdx.x < n_max) {
        const float mine = sh.max_v[threadIdx.x];
        unsigned above = 0, at = 0;
#pragma unroll 4
        for (unsigned j = 0; j < (n_max + 3) / 4; ++j) {
            const float4 o = reinterpret_cast<const float4 *>(sh.max_v)[j];
            above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
            at += (o.x == mine) + (o.y == mine) + (o.z == mine) + (o.w == mine);
        }
        if (above < k && above + at >= k) sh.bound = mine;
    }
    __syncthreads();
    bound = sh.bound;
    if (m >= bound) sh.sub[atomicAdd(&sh.n_sub, 1u)] = threadIdx.x;
    u64 least = key_of(bound, 0xffffffffu);
    const unsigned per = (R.nv + TH - 1) / TH;  // vectors a thread, at most
    for (;;) {
        if (threadIdx.x == 0) sh.n_list = 0;
        if (threadIdx.x < MAX_K) top[threadIdx.x] = 0;
        __syncthreads();
        auto see = [&](float x, unsigned i) {
            const u64 key = key_of(x, i);
            if (key >= least) {
                const unsigned at = atomicAdd(&sh.n_list, 1u);
                if (at < LIST) sh.list[at] = key;
            }
        };
        const unsigned n_sub = sh.n_sub, n_vec = n_sub * per;
        for (unsigned q = threadIdx.x; q < n_sub; q += TH) {
            const unsigned t = sh.sub[q];
            if (t < R.head) see(one(R.row + R.c0 + t) * scale, R.c0 + t);
            if (R.tail() + t < R.c1) see(one(R.row + R.tail() + t) * scale, R.tail() + t);
        }
        for (unsigned q = threadIdx.x; q < n_vec; q += 2 * TH) {
            uint4 u[2];
            unsigned j[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const unsigned qe = q + e * TH, w = qe / per;
                j[e] = qe < n_vec ? sh.sub[w] + (qe - w * per) * TH : R.nv;
                if (j[e] < R.nv) u[e] = ld16(R.row + R.body() + (size_t)j[e] * V);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (j[e] < R.nv) {
                    float x[V];
                    unpack<T>(u[e], x);
#pragma unroll
                    for (int i = 0; i < V; ++i) see(x[i] * scale, R.body() + j[e] * V + i);
                }
        }
        __syncthreads();
        const bool over = sh.n_list > LIST;
        unsigned n = min(sh.n_list, (unsigned)LIST);
        if ((n & 1) && threadIdx.x == 0) sh.list[n] = 0;
        n += n & 1;
        __syncthreads();
        rank_list<TH>(sh.list, n, k, top);
        __syncthreads();
        if (!over) return;
        least = top[k - 1];  // k listed elements reach it: the next bound, above the last
        __syncthreads();
    }
}

template <int TH, typename T>
__global__ void __launch_bounds__(TH, (sizeof(T) == 4 ? 4 : 5) * 256 / TH) k_logprobs(const lp_args a) {
    constexpr int V = vec<T>::N, WARPS = TH / 32;
    __shared__ shared_lists<TH> sh;
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned size = cluster.num_blocks(), rank = cluster.block_rank();
    const unsigned row = blockIdx.x / size;
    if (size > 1) cluster.barrier_arrive();  // waited for before the first one's memory is written
    pdl_trigger();
    pdl_wait();
    const T *p = static_cast<const T *>(a.logits) + (size_t)row * a.row_stride;
    const unsigned share = ((a.n_vocab + size - 1) / size + V - 1) / V * V;
    const unsigned c0 = min(rank * share, a.n_vocab), c1 = min(c0 + share, a.n_vocab);
    const run<T> R(p, c0, c1);
    // the given token's logit, asked for before the pass
    unsigned token = 0;
    float given = 0.f;
    if (a.logprob && rank == 0 && threadIdx.x == 0) {
        token = a.tokens[row];
        if (token < a.n_vocab) given = one(p + token);
    }
    const float scale = a.scale, scale2 = a.scale * LOG2E;

    // 16-byte loads: 32 f32 or 16 16-bit logits a look, as registers for four or five CTAs an SM allow
    constexpr int UNROLL = sizeof(T) == 4 ? 8 : 2;
    triple r{-INFINITY, 0.f, 0.f};
    unsigned j = threadIdx.x;
    for (; j + (UNROLL - 1) * TH < R.nv; j += UNROLL * TH) {
        uint4 u[UNROLL];
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) u[i] = ld16(R.row + R.body() + (size_t)(j + i * TH) * V);
        float x[UNROLL * V];
#pragma unroll
        for (int i = 0; i < UNROLL; ++i) unpack<T>(u[i], x + i * V);
        take(r, x, scale2);
    }
    for (; j < R.nv; j += TH) {
        float x[V];
        unpack<T>(ld16(R.row + R.body() + (size_t)j * V), x);
        take(r, x, scale2);
    }
    if (threadIdx.x < R.head) {
        const float x[1] = {one(R.row + R.c0 + threadIdx.x)};
        take(r, x, scale2);
    }
    if (R.tail() + threadIdx.x < R.c1) {
        const float x[1] = {one(R.row + R.tail() + threadIdx.x)};
        take(r, x, scale2);
    }
    r.m *= scale;  // rounding keeps the order: this is the largest of the rounded products
    r.s *= scale;
    // every product -inf: nothing here has a weight (the unscaled logits may be finite, a mask's lowest
    // value, and equal); a sum that is NaN stays
    if (r.m == -INFINITY) r.l = r.s = r.l * 0.f;
    const float mine = r.m;

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const triple b{__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.l, o), __shfl_xor_sync(0xffffffffu, r.s, o)};
        r = join(r, b);
    }
    if (lane == 0) sh.part[warp] = r;
    if (a.k) top_of_run(R, mine, scale, a.k, sh, size > 1 ? sh.best : sh.top[0]);
    else __syncthreads();
    if (size > 1) cluster.barrier_wait();
    shared_lists<TH> &first = size > 1 ? *cluster.map_shared_rank(&sh, 0) : sh;
    if (threadIdx.x == 0) {
        r = sh.part[0];
        for (int w = 1; w < WARPS; ++w) r = join(r, sh.part[w]);
        first.whole[rank] = r;
    }
    if (size > 1) {
        if (threadIdx.x < MAX_K && a.k) first.top[rank][threadIdx.x] = sh.best[threadIdx.x];
        cluster.sync();
        if (rank != 0) return;
    } else {
        __syncthreads();
    }
    // the cluster's triples, joined in pairs by every warp
    r = lane < (int)size ? sh.whole[lane] : triple{-INFINITY, 0.f, 0.f};
    for (unsigned o = size >> 1; o > 0; o >>= 1) {
        const triple b{__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.l, o), __shfl_xor_sync(0xffffffffu, r.s, o)};
        r = join(r, b);
    }
    r.m = __shfl_sync(0xffffffffu, r.m, 0);
    r.l = __shfl_sync(0xffffffffu, r.l, 0);
    r.s = __shfl_sync(0xffffffffu, r.s, 0);
    const float log_l = logf(r.l);
    const bool none = r.m == -INFINITY && r.l == 0.f;  // every logit -inf
    if (threadIdx.x == 0) {
        if (a.entropy) a.entropy[row] = none ? 0.f : log_l - r.s / r.l;
        if (a.logprob) a.logprob[row] = token >= a.n_vocab ? 0.f : none ? -INFINITY : (given * scale - r.m) - log_l;
    }
    if (a.k) {
        if (size > 1) {
            // a key's rank: its place in its own list, and in each other list the keys above it
            for (unsigned i = threadIdx.x; i < size * a.k; i += TH) {
                const unsigned c = i / a.k, e = i - c * a.k;
                const u64 key = sh.top[c][e];
                unsigned place = e;
                for (unsigned o = 0; o < size; ++o) {
                    if (o == c) continue;
                    unsigned n = 0;  // lists fall, their unused ends are 0
#pragma unroll
                    for (unsigned w = MAX_K / 2; w > 0; w >>= 1)
                        if (sh.top[o][n + w - 1] > key) n += w;
                    if (sh.top[o][n] > key) ++n;
                    place += n;
                }
                if (key && place < a.k) sh.best[place] = key;
            }
            __syncthreads();
        }
        if (threadIdx.x < a.k) {
            const u64 key = size > 1 ? sh.best[threadIdx.x] : sh.top[0][threadIdx.x];
            const float v = value_of(key);
            a.top_id[(size_t)row * a.k + threadIdx.x] = 0xffffffffu - (unsigned)key;
            a.top_lp[(size_t)row * a.k + threadIdx.x] = none ? -INFINITY : (v - r.m) - log_l;
        }
    }
}

template <int TH, typename T>
cudaError_t launch_with(moearc_ctx *c, const lp_args &a, unsigned n_rows) {
    static std::atomic<bool> done[MOEARC_MAX_DEVICES];
    cudaError_t e = once_per_device(done, [] {
        return cudaFuncSetAttribute(k_logprobs<TH, T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    if (e != cudaSuccess) return e;
    // CTAs for twice the SMs, but at least 16 vectors a thread of each; clusters of 16 only where they
    // are few enough to run at once (16 rows of 131072 f32: 20 us with 16 CTAs a row, 11 with 8)
    const unsigned most = std::max(1u, a.n_vocab / (TH * 16 * (unsigned)vec<T>::N));
    unsigned size = 1;
    while (size < 16 && n_rows * size < (unsigned)c->sm_count * 2 && size * 2 <= most && (size < 8 || n_rows * 16 <= (unsigned)c->sm_count)) size *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_rows * size);
    cfg.blockDim = dim3(TH);
    cfg.stream = c->stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = size;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, k_logprobs<TH, T>, a);
}

template <typename T>
cudaError_t launch(moearc_ctx *c, const lp_args &a, unsigned n_rows) {
    return n_rows > (unsigned)c->sm_count * 8 && (size_t)a.n_vocab * sizeof(T) <= SHORT_ROW ? launch_with<128, T>(c, a, n_rows) : launch_with<256, T>(c, a, n_rows);
}

}  // namespace

extern "C" {

int moearc_x_token_logprobs(moearc_ctx *c, const void *logits, unsigned int type, unsigned long row_stride, unsigned int n_rows,
                            unsigned int n_vocab, float scale, const unsigned int *tokens, float *logprob, float *entropy,
                            unsigned int k, unsigned int *top_ids, float *top_logprobs) {
    if (!c || !logits || (!tokens) != (!logprob)) return ERR;
    if (k && (!top_ids || !top_logprobs)) return ERR;
    if (!kv_elem_bytes(type)) return ERR_ARG;
    if (n_vocab == 0 || n_vocab > (1u << 30) || row_stride < n_vocab || k > MAX_TOPK || k > n_vocab || n_rows > (1u << 26)) return ERR_ARG;
    if (!(scale >= 1e-30f && scale <= 1e30f)) return ERR_ARG;
    if (!aligned(logits, kv_elem_bytes(type)) || !aligned(tokens, 4) || !aligned(logprob, 4) || !aligned(entropy, 4)) return ERR_ARG;
    if (k && (!aligned(top_ids, 4) || !aligned(top_logprobs, 4))) return ERR_ARG;
    if (n_rows == 0) return OK;
    const lp_args a{logits, tokens, row_stride, n_vocab, k, scale, logprob, entropy, top_logprobs, top_ids};
    device_guard g(c->device);
    if (!g.ok) return ERR;
    launch_scope ls(c, "token_logprobs", n_rows, n_vocab);
    const cudaError_t e = type == T_F32   ? launch<float>(c, a, n_rows)
                          : type == T_F16 ? launch<__half>(c, a, n_rows)
                                          : launch<__nv_bfloat16>(c, a, n_rows);
    if (e != cudaSuccess) cudaGetLastError();  // the failed launch's error, not left for an unrelated later check
    const int rc = ls.finish();
    return e != cudaSuccess ? ERR : rc;
}

}  // extern "C"
