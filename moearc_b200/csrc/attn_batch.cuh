// attn_batch.cuh — what the kernels of decode attention over the paged cache share: their arguments,
// the cut of the work into equal runs, the 16-bit terms of f32 values, and the join of rows that
// several CTAs had a part of.
#pragma once

#include "kvcache.cuh"

namespace moearc {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MAX_SMEM = 227 * 1024;
// A row's weights are taken against a reference m that follows its maximum only once that is this much
// above (in powers of two): most tiles then rescale nothing. A weight, in the sums and the records of
// parts, is 2^(s - m - LAZY): one at most, so that no sum leaves the range before n times the largest value does.
constexpr float LAZY = 4.f, DOWN = 1.f / 16;  // DOWN: 2^-LAZY

struct attn_args {
    float *out;
    const float *q, *k_new, *v_new, *sinks;
    uint8_t *k, *v;  // the layer's pools
    const unsigned *tables, *n_kv, *begin;
    unsigned *status;
    size_t q_stride, new_stride, token_bytes, head_bytes;  // bytes: n_kv_heads x head_dim elements, head_dim elements
    unsigned n_seq, max_pages, n_pages, pt, pt_inv, cap;  // pt_inv: floor(2^32 / pt), at most 2^32 - 1
    unsigned unit;  // bytes of one copy: 16 where rows start on 16-byte boundaries, else 4 or 2
    int one_page;   // tiles never cross a page
    const unsigned *rows;  // the batch rows' cache rows, or null: row i is i
    int n_heads, group, D, subs;  // subs: virtual heads a kv head (its query heads by GP)
    int hg, rsplit, nhg;          // virtual heads a CTA, warps a head, head groups
    float scale2;  // scale x log2(e): scores are kept in powers of two
    float *part;   // [CTA][2][hg][GP][D + 2]
    int4 *notes;   // [CTA] what is to join: batch row, first virtual head, parts (0: nothing), the first part's record
};

// The keys [lo, hi) of batch row i in cache row `row`, hi cut to the table.
__device__ __forceinline__ void span_of(const attn_args &a, unsigned i, unsigned &row, unsigned &lo, unsigned &hi) {
    row = a.rows ? a.rows[i] : i;
    hi = min(a.n_kv[row], a.cap);
    lo = a.begin ? min(a.begin[i], hi) : 0;
}

// Token j's table entry and slot: j / pt by its inverse, one short at most.
__device__ __forceinline__ void place_of(const attn_args &a, unsigned j, unsigned &entry, unsigned &slot) {
    entry = __umulhi(j, a.pt_inv);
    slot = j - entry * a.pt;
    if (slot >= a.pt) {
        ++entry;
        slot -= a.pt;
    }
}

// The line's tiles over `ctas` CTAs: each takes `each` of them, the first `more` one more.
struct runs {
    int each, more;
    __device__ __forceinline__ runs(int total, int ctas) : each(total / ctas), more(total - total / ctas * ctas) {}
    __device__ __forceinline__ int start(int c) const { return each * c + min(c, more); }
    __device__ __forceinline__ int owner(int g) const {
        const int cut = more * (each + 1);
        return g < cut ? g / (each + 1) : more + (g - cut) / each;
    }
};

// CTA c's note for the join: its run begins inside the unit [u0, u1) of batch row `row` and is the
// first to do so.
__device__ __forceinline__ int4 note_of(const runs &r, int c, int row, int vh, int u0, int u1) {
    const bool joins = c > 0 && r.start(c) > u0 && r.start(c - 1) <= u0;
    return make_int4(row, vh, joins ? r.owner(u1 - 1) - c + 2 : 0, c > 0 && r.start(c - 1) == u0 ? 0 : 1);
}

// 2^x, subnormal results as 0.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <bool BF>
__device__ __forceinline__ uint16_t to16(float v) {
    if constexpr (BF) return f32_to_bf16_bits(v);
    else return __half_as_ushort(__float2half_rn(v));
}
template <bool BF>
__device__ __forceinline__ float from16(uint16_t b) {
    if constexpr (BF) return bf16_bits_to_f32(b);
    else return f16_bits_to_f32(b);
}
// Two values rounded to 16 bits and packed, and a packed pair's values.
template <bool BF>
__device__ __forceinline__ uint32_t pack(float x, float y) {
    if constexpr (BF) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&v);
    } else {
        const __half2 v = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
}
template <bool BF>
__device__ __forceinline__ float2 unpack(uint32_t u) {
    if constexpr (BF) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
// Two values as packed pairs of 16-bit terms: x = t0 + t1 + t2, each term the rounding of what
// the ones before it leave (the largest finite values' to a finite bf16).
template <bool BF>
__device__ __forceinline__ void terms(float x, float y, uint32_t &t0, uint32_t &t1, uint32_t &t2) {
    const float most = __uint_as_float(0x7f7f0000u);
    t0 = BF ? pack<BF>(fminf(fmaxf(x, -most), most), fminf(fmaxf(y, -most), most)) : pack<BF>(x, y);
    const float2 a = unpack<BF>(t0);
    t1 = pack<BF>(x - a.x, y - a.y);
    const float2 b = unpack<BF>(t1);
    t2 = pack<BF>(x - a.x - b.x, y - a.y - b.y);
}
// What the first term a of x leaves for the next. A weight's bf16 terms go on as they are: x = t0 + t1 + t2. f16 ends at
// 2^-24, where plain terms of a small x would lose its bits and then x itself: each is 2^11 times as fine as
// the one before, x = t0 + FINE (t1 + FINE t2), which keeps 22 bits of x <= 2^15 down to 2^-24 and ends at 2^-46.
// (A fourth term ended at 2^-57 and cost 2 to 11% more where rows are short.)
constexpr float FINE = 1.f / 2048;
template <bool BF>
__device__ __forceinline__ float rest(float x, float a) {
    if constexpr (BF) return x - a;
    else return fmaf(a, -1.f / FINE, x * (1.f / FINE));  // exactly
}

// 16 (or 4) bytes global -> shared, zeros in their place where the source is not to be read.
__device__ __forceinline__ void cp_async16(unsigned dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16z(unsigned dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4z(unsigned dst, const void *src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }
__device__ __forceinline__ unsigned smem_u32(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }

// Joins the parts of a row that the runs of several CTAs cut up, in tile order: CTA (c, virtual head
// of the group, share of the channels) joins the row that run c begins inside, where the note says so.
// Four threads take a quarter of the parts each for four channels of a head. The parts are in L2: bound by
// the latency of note, maxima and sums, about 2 us behind the kernel before it (7 us from cold caches).
constexpr int JOIN_THREADS = 256, JOIN_PARTS = 4, JOIN_OUT = JOIN_THREADS / JOIN_PARTS * 4;
template <int GP>
static __global__ void __launch_bounds__(JOIN_THREADS, 4) k_attn_join(const __grid_constant__ attn_args a) {
    extern __shared__ float wgt[];  // [GP][parts]
    __shared__ float inv[GP];
    __shared__ float4 sums[JOIN_PARTS][JOIN_THREADS / JOIN_PARTS];
    pdl_trigger();
    pdl_wait();
    const int c = blockIdx.x + 1, hs = blockIdx.y;
    const int4 at = a.notes[c];
    const int n = at.z;
    if (n == 0) return;
    const int D = a.D, HG = a.hg, vh = at.y + hs, kvh = vh / a.subs, sub = vh - kvh * a.subs;
    const int h0 = kvh * a.group + sub * GP, heads = min(GP, a.group - sub * GP);
    // the first part is CTA c - 1's, in its first or second record; the others' parts are their first
    const size_t rec = (size_t)GP * (D + 2), step = (size_t)2 * HG * rec;
    const float *rest = a.part + (size_t)c * step + hs * rec, *part0 = rest - step + (size_t)at.w * HG * rec;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q = threadIdx.x & (JOIN_THREADS / JOIN_PARTS - 1), grp = threadIdx.x / (JOIN_THREADS / JOIN_PARTS);
    const int k0 = n * grp / JOIN_PARTS, k1 = n * (grp + 1) / JOIN_PARTS;
    auto part_at = [&](int k) { return k ? rest + (size_t)(k - 1) * step : part0; };
    // this thread's first parts of its first channels, asked for before the weights are worked out
    constexpr int AHEAD = 4;
    float4 ahead[AHEAD];
    const int e0 = blockIdx.z * JOIN_OUT + 4 * q;
    const bool quads = D % 4 == 0;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
        if (quads && e0 < heads * D && k0 + i < k1) ahead[i] = *reinterpret_cast<const float4 *>(part_at(k0 + i) + e0);
    for (int hd = warp; hd < heads; hd += JOIN_THREADS / 32) {
        const float sk = a.sinks ? a.sinks[h0 + hd] * LOG2E : -INFINITY;
        const size_t ml = (size_t)GP * D + 2 * hd;  // even: max and sum are read together
        // up to 32 parts are in registers, more are read again for the sum
        float2 mine = make_float2(-INFINITY, 0.f);
        float M = sk;
        for (int k = lane; k < n; k += 32) {
            const float2 v = *reinterpret_cast<const float2 *>(part_at(k) + ml);
            if (k < 32) mine = v;
            M = fmaxf(M, v.x);
        }
        M = warp_max(M);
        float sum = 0.f;
        for (int k = lane; k < n; k += 32) {
            const float2 v = k < 32 ? mine : *reinterpret_cast<const float2 *>(part_at(k) + ml);
            const float f = v.x == -INFINITY ? 0.f : ex2(v.x - M);
            wgt[hd * n + k] = f;
            sum += v.y * f;
        }
        sum = warp_sum(sum);
        if (lane == 0) {
            sum += sk == -INFINITY ? 0.f : ex2(sk - M) * DOWN;
            inv[hd] = sum == 0.f ? 0.f : 1.f / sum;
        }
    }
    __syncthreads();
    float *out = a.out + ((size_t)at.x * a.n_heads + h0) * D;
    for (int b = blockIdx.z * JOIN_OUT; b < heads * D; b += gridDim.z * JOIN_OUT) {
        const int e = b + 4 * q;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        // channels of one head where head_dim is a multiple of four; else each channel has its own
        const float *w0 = wgt + min(e, heads * D - 1) / D * n;
        if (e < heads * D) {
            if (quads) {
                auto add = [&](float4 x, float w) {
                    v[0] = fmaf(x.x, w, v[0]);
                    v[1] = fmaf(x.y, w, v[1]);
                    v[2] = fmaf(x.z, w, v[2]);
                    v[3] = fmaf(x.w, w, v[3]);
                };
                int k = k0;
                if (e == e0) {
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i)
                        if (k0 + i < k1) add(ahead[i], w0[k0 + i]);
                    k += AHEAD;
                }
#pragma unroll 4
                for (; k < k1; ++k) add(*reinterpret_cast<const float4 *>(part_at(k) + e), w0[k]);
            } else {
                for (int k = k0; k < k1; ++k) {
                    const float *p = part_at(k);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (e + i < heads * D) v[i] = fmaf(p[e + i], wgt[(e + i) / D * n + k], v[i]);
                }
            }
        }
        sums[grp][q] = make_float4(v[0], v[1], v[2], v[3]);
        __syncthreads();
        if (grp == 0) {
#pragma unroll
            for (int g = 1; g < JOIN_PARTS; ++g) {
                const float4 x = sums[g][q];
                v[0] += x.x;
                v[1] += x.y;
                v[2] += x.z;
                v[3] += x.w;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e + i < heads * D) out[e + i] = v[i] * inv[(e + i) / D];
        }
        __syncthreads();
    }
}

// After the kernel that wrote the notes; its grid was `grid`.
template <int GP>
static cudaError_t attn_join_launch(moearc_ctx *c, int grid, const attn_args &a) {
    if (grid < 2) return cudaSuccess;
    // the join's few KB under the same split of L1 and shared memory as the kernel before it
    static std::atomic<bool> done[MOEARC_MAX_DEVICES];
    const cudaError_t e = once_per_device(done, [] { return set_smem(k_attn_join<GP>, 40 * 1024); });
    if (e != cudaSuccess) return e;
    return launch_pdl(k_attn_join<GP>, dim3((unsigned)grid - 1, (unsigned)a.hg, (unsigned)(GP * a.D + JOIN_OUT - 1) / JOIN_OUT),
                      dim3(JOIN_THREADS), (size_t)GP * grid * 4, c->stream, a);
}

// How a shape is cut: virtual heads and warps per CTA, stages, shared memory and the grid.
struct attn_plan {
    int gp, keys, subs, hg, rsplit, nhg, warps, ns, smem, grid;
};

// The tcgen05 kernel (attn_tc.cu), for 16-bit caches of head_dim 40 to 256, a multiple of 8, with fewer
// than 2^31 tokens: its cut, and its launch.
void attn_tc_plan(attn_plan &p, int n_heads, int n_kv, int D, int sms);
cudaError_t attn_tc_launch(moearc_ctx *c, const attn_plan &p, unsigned kv_type, const attn_args &a);

}  // namespace moearc
