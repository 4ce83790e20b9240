// attn_batch.cu — decode attention of one new token for every row of a ragged batch over the
// paged cache of kvcache.cu.
//
//   out[i, h] = sum_j softmax_j(scale q[i, h] . k_j  [, sink_h]) v_j,   begin_i <= j < n_kv_i,
//
// over the keys whose table entry is a page; zeros where there are none. GQA: the `group` query
// heads of a kv head share its keys. The row's newest token may come with the call (k_new, v_new):
// it is rounded to the cache's type, attended as such and stored in its slot.
//
// The operator reads each live key and value once, 2 n_kv_heads head_dim elements a token, and
// does 4 group flops for each: it is bound by HBM. So:
//
// - Work is split evenly whatever the lengths are. The keys of all rows form one line of tiles; each
//   CTA of a grid that just fills the GPU takes an equal run of it, found from a prefix sum over the
//   lengths that every CTA computes. A run that ends inside a row leaves a partial (max, sum,
//   accumulator) behind, at most two a CTA, and a second kernel joins them in tile order; so
//   results do not depend on timing, and partials do not grow with the batch.
// - A warp is one kv head (with up to 8 of its query heads) of the CTA's tile, so that the CTA's
//   warps together read whole rows of a page; where a model has fewer heads than warps, several
//   warps share a head, taking alternate tiles. A warp streams its K and V tiles through a ring of
//   cp.async stages of its own, which runs on across rows: no barrier in the loop, and the next
//   row's keys are on their way before this row is finished. The tensor-core tiles' copies are issued by
//   other warps (one for two), which hand stages over and back at mbarriers with a limit to every wait:
//   the addresses of a tile's copies were a third of a computing warp's instructions. The CUDA cores' tile
//   has 16 warps that hide them.
// - 16-bit caches of 40 to 256 channels, a multiple of 8, have a kernel of their own on tcgen05
//   (attn_tc.cu). Here, on the same line of tiles: f32 caches of 36 to 256 channels, a multiple of 4,
//   on mma.sync with tf32 terms (tcgen05's tf32 would want keys and values taken apart in shared
//   memory, three times the bytes there); every other size, and pools off a 16-byte boundary, on CUDA cores.
// - f32 keys and values keep all 24 bits there, as three tf32 terms; q and the softmax weights are two
//   rounded ones (23 bits, a last place more than f32's own rounding of a product). A tile's P V is
//   summed from zero and added to the f32 accumulator by an ordinary add: the
//   tensor core's own accumulation truncates, which a long context would show.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "attn_batch.cuh"
#include "tc.cuh"

using namespace moearc;

namespace moearc {
size_t kv_page_work_bytes(unsigned n_pages);
}

namespace {

// ---- the tensor-core tile of f32 caches ---------------------------------------------------------
//
// head_dim up to D_, a multiple of 4. mma.sync m16n8k8 on tf32 terms: a key or value is cut into 11, 11 and
// 2 bits (three MMAs), q and the weights are two rounded terms on rows 0-7 and 8-15 of the A operand.
// Which channel (or key) stands for which k of an MMA is free as long as both
// operands agree: k = j and j + 4 are channels 2 j and 2 j + 1 of an eight, read as one 8-byte load,
// and keys 2 j and 2 j + 1, as the scores come out. Rows are 8 (keys) and 4 (values) words off a
// multiple of 32, so that these reads meet 32 banks.
//
// 30 rows of up to 6000 tokens: 8 kv heads of 64 with 8 query heads each 107 us (318 on CUDA cores),
// 4 heads of 128 with 8 each 125 (317), 1 of 256 with 16 159 (369; two passes over the keys), where the
// bytes alone take 74, 74 and 37. Bound by the instructions around the MMAs (three a side, each operand
// taken apart as it leaves shared memory) and, at one CTA an SM, by their latency. Keys and values in two terms
// (23 bits: a row of one key did not return its value, and the largest finite values became
// infinite) took 98, 110 and 140; the third as bf16 in MMAs of twice the k 105, 139 (its registers spill) and 177.

__device__ __forceinline__ uint32_t tf32(float x) {
    uint32_t u;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(u) : "f"(x));
    return u;
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x rounded to 11 bits, the largest finite values to a finite one.
__device__ __forceinline__ uint32_t tf32_finite(float x) {
    return __float_as_uint(fminf(fmaxf(__uint_as_float(tf32(x)), __uint_as_float(0xff7fe000u)), __uint_as_float(0x7f7fe000u)));
}
// All 24 bits of x as tf32 terms of 11, 11 and 2 bits, cut rather than rounded: the largest finite values keep
// finite terms.
__device__ __forceinline__ void thirds(float x, uint32_t (&t)[3]) {
    t[0] = __float_as_uint(x) & 0xffffe000u;
    const float r = x - __uint_as_float(t[0]);
    t[1] = __float_as_uint(r) & 0xffffe000u;
    t[2] = __float_as_uint(r - __uint_as_float(t[1]));
}

template <int D_, int KEYS_>
struct tf32_tile {
    static constexpr int KEYS = KEYS_, NB = KEYS / 8, GP = 8, D = D_, WARPS = D_ > 128 ? 4 : 8;
    static constexpr bool SPLIT = true;
    static constexpr int KROW = (D + 31) / 32 * 32 + 8, VROW = (D + 31) / 32 * 32 + 4;  // words
    static constexpr bool QREG = D <= 128;  // q's terms in registers, else in shared memory

    uint32_t qa[QREG ? D / 8 : 1][4];
    float o[D / 8][2], m, l;
    static __host__ __device__ int stage_bytes(int) { return KEYS * (KROW + VROW) * 4; }
    static __host__ __device__ bool padded(int d) { return d < D; }
    static __host__ __device__ int extra_bytes(int) { return QREG ? 0 : D / 8 * 512; }
    static __device__ __forceinline__ int key_row(int r) { return r * KROW * 4; }
    static __device__ __forceinline__ int value_row(int r) { return (KEYS * KROW + r * VROW) * 4; }

    __device__ __forceinline__ void init(const float *q, int heads, const attn_args &a, uint8_t *extra, int lane) {
        const int hr = lane >> 2, qd = lane & 3;
        const bool live = hr < heads;
        const float *p = q + (size_t)(live ? hr : 0) * a.D;
        if constexpr (!QREG) __syncwarp();
        // whole where q's terms are registers: an index known at run time puts the tile in local memory
#pragma unroll(QREG ? D / 8 : 4)
        for (int kk = 0; kk < D / 8; ++kk) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = 8 * kk + 2 * qd + e;
                const float x = live && d < a.D ? p[d] : 0.f;
                w[2 * e] = tf32_finite(x);
                w[2 * e + 1] = tf32(x - __uint_as_float(w[2 * e]));
            }
            if constexpr (QREG) {
#pragma unroll
                for (int e = 0; e < 4; ++e) qa[kk][e] = w[e];
            } else {
                reinterpret_cast<uint4 *>(extra)[kk * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        if constexpr (!QREG) __syncwarp();
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = 0.f;
        m = -INFINITY;
        l = 0.f;
    }
    // copy(row, chunk) for every 16-byte chunk of the tile's rows
    template <typename F>
    static __device__ __forceinline__ void chunks(const attn_args &a, int lane, F &&copy) {
        constexpr int CH = D / 4;
        if (a.D == D) {
#pragma unroll
            for (int i = 0; i < KEYS * CH / 32; ++i) copy((lane + 32 * i) / CH, (lane + 32 * i) % CH, true);
        } else {
#pragma unroll 4
            for (int i = 0; i < KEYS * CH / 32; ++i) copy((lane + 32 * i) / CH, (lane + 32 * i) % CH, (lane + 32 * i) % CH < a.D / 4);
        }
    }
    static __device__ __forceinline__ void load_run(uint8_t *stage, const uint8_t *src, long long to_v, const attn_args &a, int lane) {
        const unsigned s0 = smem_u32(stage);
        chunks(a, lane, [&](int r, int ch, bool on) {
            const uint8_t *p = src + (size_t)r * a.token_bytes + ch * 16;
            if (on) {
                cp_async16(s0 + key_row(r) + ch * 16, p);
                cp_async16(s0 + value_row(r) + ch * 16, p + to_v);
            }
        });
    }
    static __device__ __forceinline__ void load_rows(uint8_t *stage, long long off, const attn_args &a, int lane) {
        const unsigned s0 = smem_u32(stage);
        chunks(a, lane, [&](int r, int ch, bool on) {
            const long long b = __shfl_sync(0xffffffffu, off, r);
            const size_t src = (b < 0 ? 0 : (size_t)b) + ch * 16;
            if (on) {
                cp_async16z(s0 + key_row(r) + ch * 16, a.k + src, b >= 0);
                cp_async16z(s0 + value_row(r) + ch * 16, a.v + src, b >= 0);
            }
        });
    }
    static __device__ __forceinline__ void round_row(const float *x, uint8_t *stage, int r, uint8_t *slot, const attn_args &a, int lane) {
        auto *row = reinterpret_cast<float *>(stage + (r < KEYS ? key_row(r) : value_row(r - KEYS)));
        for (int d = lane; d < a.D; d += 32) {
            row[d] = x[d];
            if (slot) reinterpret_cast<float *>(slot)[d] = x[d];
        }
    }
    __device__ __forceinline__ void step(const uint8_t *stage, unsigned live, const attn_args &a, uint8_t *extra, int lane) {
        const int g = lane >> 2, qd = lane & 3;
        float c0[2][4] = {}, c1[2][4] = {};  // of each eight keys, or of one and every other eight channels
        const float *ks = reinterpret_cast<const float *>(stage + key_row(g)) + 2 * qd;
#pragma unroll
        for (int kk = 0; kk < D / 8; ++kk) {
            uint32_t w[4];
            if constexpr (QREG) {
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = qa[kk][e];
            } else {
                const uint4 u = reinterpret_cast<const uint4 *>(extra)[kk * 32 + lane];
                w[0] = u.x;
                w[1] = u.y;
                w[2] = u.z;
                w[3] = u.w;
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const float2 k = *reinterpret_cast<const float2 *>(ks + n * 8 * KROW + 8 * kk);
                uint32_t x[3], y[3];
                thirds(k.x, x);
                thirds(k.y, y);
                mma_tf32(c0[NB == 2 ? n : kk & 1], w, x[0], y[0]);
                mma_tf32(c1[NB == 2 ? n : kk & 1], w, x[1], y[1]);
                mma_tf32(c1[NB == 2 ? n : kk & 1], w, x[2], y[2]);
            }
        }
        // scores (in powers of two) of head lane / 4 for keys 2 qd, 2 qd + 1 (and 8 + 2 qd, 9 + 2 qd)
        float s[2 * NB], mt = -INFINITY;
        const unsigned in = live >> (2 * qd);
        if constexpr (NB == 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c0[0][e] += c0[1][e];
                c1[0][e] += c1[1][e];
            }
        }
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float x = (c0[n][e] + (c0[n][e + 2] + (c1[n][e] + c1[n][e + 2]))) * a.scale2;
                s[2 * n + e] = in >> (8 * n + e) & 1 ? x : -INFINITY;
                mt = fmaxf(mt, s[2 * n + e]);
            }
        if (__any_sync(0xffffffffu, mt - m > LAZY)) {
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
            const float mn = fmaxf(m, mt), corr = ex2(m - (mn == -INFINITY ? 0.f : mn));
            l *= corr;
            m = mn;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                o[i][0] *= corr;
                o[i][1] *= corr;
            }
        }
        const float base = m == -INFINITY ? 0.f : m;
        uint32_t pa[NB][4];
#pragma unroll
        for (int e = 0; e < 2 * NB; ++e) {
            const float p = ex2(s[e] - base) * DOWN;
            l += p;
            pa[e >> 1][2 * (e & 1)] = tf32(p);
            pa[e >> 1][2 * (e & 1) + 1] = tf32(p - __uint_as_float(pa[e >> 1][2 * (e & 1)]));
        }
        const float *vs = reinterpret_cast<const float *>(stage + value_row(2 * qd)) + g;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            float c[4] = {}, d[4] = {};
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                uint32_t x[3], y[3];
                thirds(vs[n * 8 * VROW + 8 * i], x);
                thirds(vs[(n * 8 + 1) * VROW + 8 * i], y);
                mma_tf32(c, pa[n], x[0], y[0]);
                mma_tf32(d, pa[n], x[1], y[1]);
                mma_tf32(d, pa[n], x[2], y[2]);
            }
            o[i][0] += c[0] + (c[2] + (d[0] + d[2]));
            o[i][1] += c[1] + (c[3] + (d[1] + d[3]));
        }
    }
    __device__ __forceinline__ void close(int) {
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
    }
    template <typename F, typename G>
    __device__ __forceinline__ void each(int lane, const attn_args &a, F &&f, G &&one) {
        const int hr = lane >> 2, qd = lane & 3;
        one(hr, m, l, qd == 0);
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (8 * i + 2 * qd + e < a.D) f(hr, 8 * i + 2 * qd + e, o[i][e]);
    }
};

// ---- the CUDA-core tile (any head size, any alignment) -----------------------------------------
//
// Eight keys a tile. Scores: lane (key, quarter) sums over every fourth group of four channels for
// all GP heads, and the quarters are added so that each lane ends with GP / 4 heads of its key.
// Values: a lane owns groups of four channels (lane + 32 i) of all GP heads, the weights come from
// shared memory, each twice over: channels are multiplied in pairs (fma.rn.f32x2), which halves the
// instructions, and those are what bounds it: 64 query heads over 8 of 64, f32, 30 rows of up to 6000
// tokens 318 us, three times the tensor cores' tile.

// d += a b, two values at once.
__device__ __forceinline__ void fma2(float2 &d, float2 a, float2 b) {
    asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%0, %1}; fma.rn.f32x2 z, x, y, z; mov.b64 {%0, %1}, z; }"
        : "+f"(d.x), "+f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
}

template <typename T>
__device__ __forceinline__ float4 four(const T *p) {
    if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const float4 *>(p);
    } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        if constexpr (std::is_same<T, __half>::value) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&u.x)), y = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
            return make_float4(x.x, x.y, y.x, y.y);
        } else {
            return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                               __uint_as_float(u.y & 0xffff0000u));
        }
    }
}
__device__ __forceinline__ void round_to(float v, float &d) { d = v; }
__device__ __forceinline__ void round_to(float v, __half &d) { d = __float2half_rn(v); }
__device__ __forceinline__ void round_to(float v, __nv_bfloat16 &d) { d = __float2bfloat16_rn(v); }

template <typename T, int NQ, int GP_>
struct core_tile {
    static constexpr int KEYS = 8, GP = GP_, WARPS = NQ == 1 ? 16 : 8;
    static constexpr bool SPLIT = false;
    float2 acc[NQ][GP][2];
    float m[GP / 4], l[GP / 4];

    // A row in shared memory: an odd number of 16-byte chunks, so that eight keys meet eight bank
    // groups; its tail past head_dim is zero.
    static __host__ __device__ int row_bytes(int D) { return (((D * (int)sizeof(T) + 15) / 16) | 1) * 16; }
    static __host__ __device__ int stage_bytes(int D) { return 2 * KEYS * row_bytes(D); }
    static __host__ __device__ bool padded(int D) { return D * (int)sizeof(T) % 16 != 0; }
    static __host__ __device__ int dpad(int D) { return (D + 3) & ~3; }
    // per warp beside the stages: q, the tile's weights, the heads' corrections
    static __host__ __device__ int extra_bytes(int D) { return (GP * dpad(D) + 2 * KEYS * GP + GP) * 4; }

    __device__ __forceinline__ void init(const float *q, int heads, const attn_args &a, uint8_t *extra, int lane) {
        // q as [four channels][head][4], so that a lane's loop has fixed offsets
        auto *qs = reinterpret_cast<float *>(extra);
        __syncwarp();
        for (int d = lane; d < dpad(a.D); d += 32)
#pragma unroll
            for (int h = 0; h < GP; ++h) qs[(d >> 2) * (4 * GP) + h * 4 + (d & 3)] = h < heads && d < a.D ? q[(size_t)h * a.D + d] : 0.f;
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int h = 0; h < GP; ++h) acc[i][h][0] = acc[i][h][1] = make_float2(0.f, 0.f);
#pragma unroll
        for (int h = 0; h < GP / 4; ++h) {
            m[h] = -INFINITY;
            l[h] = 0.f;
        }
        __syncwarp();
    }
    static __device__ __forceinline__ void load_run(uint8_t *stage, const uint8_t *src, long long to_v, const attn_args &a, int lane) {
        const int rb = row_bytes(a.D);
        const unsigned s0 = smem_u32(stage);
        for (unsigned c = lane * 16; c < a.head_bytes; c += 512) {
            const uint8_t *p = src + c;
#pragma unroll
            for (int r = 0; r < KEYS; ++r, p += a.token_bytes) {
                cp_async16(s0 + r * rb + c, p);
                cp_async16(s0 + (KEYS + r) * rb + c, p + to_v);
            }
        }
    }
    static __device__ __forceinline__ void load_rows(uint8_t *stage, long long off, const attn_args &a, int lane) {
        const int rb = row_bytes(a.D);
        const unsigned s0 = smem_u32(stage);
        if (a.unit == 16) {
            for (unsigned c = lane * 16; c - lane * 16 < a.head_bytes; c += 512) {
                const bool on = c < a.head_bytes;
#pragma unroll
                for (int r = 0; r < KEYS; ++r) {
                    const long long b = __shfl_sync(0xffffffffu, off, r);
                    const size_t src = (b < 0 ? 0 : (size_t)b) + c;
                    if (on) {
                        cp_async16z(s0 + r * rb + c, a.k + src, b >= 0);
                        cp_async16z(s0 + (KEYS + r) * rb + c, a.v + src, b >= 0);
                    }
                }
            }
            return;
        }
#pragma unroll 1
        for (int r = 0; r < KEYS; ++r) {  // rows off a 16-byte boundary
            const long long b = __shfl_sync(0xffffffffu, off, r);
            const size_t src = b < 0 ? 0 : (size_t)b;
            uint8_t *kr = stage + r * rb, *vr = kr + KEYS * rb;
            if (a.unit == 4) {
                for (unsigned c = lane * 4; c < a.head_bytes; c += 128) {
                    cp_async4z(smem_u32(kr + c), a.k + src + c, b >= 0);
                    cp_async4z(smem_u32(vr + c), a.v + src + c, b >= 0);
                }
            } else {
                for (unsigned c = lane * 2; c < a.head_bytes; c += 64) {
                    *reinterpret_cast<uint16_t *>(kr + c) = b >= 0 ? *reinterpret_cast<const uint16_t *>(a.k + src + c) : uint16_t(0);
                    *reinterpret_cast<uint16_t *>(vr + c) = b >= 0 ? *reinterpret_cast<const uint16_t *>(a.v + src + c) : uint16_t(0);
                }
            }
        }
    }
    static __device__ __forceinline__ void round_row(const float *x, uint8_t *stage, int r, uint8_t *slot, const attn_args &a, int lane) {
        for (int d = lane; d < a.D; d += 32) {
            T v;
            round_to(x[d], v);
            reinterpret_cast<T *>(stage + r * row_bytes(a.D))[d] = v;
            if (slot) reinterpret_cast<T *>(slot)[d] = v;
        }
    }
    __device__ __forceinline__ void step(const uint8_t *stage, unsigned live, const attn_args &a, uint8_t *extra, int lane) {
        const int D = a.D, dp = dpad(D), rb = row_bytes(D);
        auto *qs = reinterpret_cast<float *>(extra), *ps = qs + GP * dp, *cs = ps + 2 * KEYS * GP;
        const int key = lane >> 2, cl = lane & 3;
        const T *kr = reinterpret_cast<const T *>(stage + key * rb);
        float2 s2[GP];
#pragma unroll
        for (int h = 0; h < GP; ++h) s2[h] = make_float2(0.f, 0.f);
        const float *qc = qs + 4 * cl * GP;
#pragma unroll 2
        for (int c = 4 * cl; c < dp; c += 16, qc += 16 * GP) {
            const float4 kv = four(kr + c);
#pragma unroll
            for (int h = 0; h < GP; ++h) {
                const float4 qv = *reinterpret_cast<const float4 *>(qc + 4 * h);
                fma2(s2[h], make_float2(qv.x, qv.y), make_float2(kv.x, kv.y));
                fma2(s2[h], make_float2(qv.z, qv.w), make_float2(kv.z, kv.w));
            }
        }
        float s[GP];
#pragma unroll
        for (int h = 0; h < GP; ++h) s[h] = s2[h].x + s2[h].y;
        // heads cl GP / 4 + (0 .. GP / 4 - 1) of the key, summed over the quarters
        float t[GP / 2], x[GP / 4];
#pragma unroll
        for (int h = 0; h < GP / 2; ++h) {
            const float mine = cl & 2 ? s[h + GP / 2] : s[h], other = cl & 2 ? s[h] : s[h + GP / 2];
            t[h] = mine + __shfl_xor_sync(0xffffffffu, other, 2);
        }
#pragma unroll
        for (int h = 0; h < GP / 4; ++h) {
            const float mine = cl & 1 ? t[h + GP / 4] : t[h], other = cl & 1 ? t[h] : t[h + GP / 4];
            x[h] = mine + __shfl_xor_sync(0xffffffffu, other, 1);
        }
        const bool in = live >> key & 1;
        bool up = false;
#pragma unroll
        for (int h = 0; h < GP / 4; ++h) {
            x[h] = in ? x[h] * a.scale2 : -INFINITY;
            up |= x[h] - m[h] > LAZY;
        }
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
            for (int h = 0; h < GP / 4; ++h) {
                float mt = x[h];
                mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 4));
                mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 8));
                mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 16));
                const float mn = fmaxf(m[h], mt), corr = ex2(m[h] - (mn == -INFINITY ? 0.f : mn));
                l[h] *= corr;
                m[h] = mn;
                if (key == 0) cs[cl * (GP / 4) + h] = corr;
            }
            __syncwarp();
#pragma unroll
            for (int h = 0; h < GP; ++h) {
                const float corr = cs[h];
#pragma unroll
                for (int i = 0; i < NQ; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        acc[i][h][e].x *= corr;
                        acc[i][h][e].y *= corr;
                    }
            }
        }
#pragma unroll
        for (int h = 0; h < GP / 4; ++h) {
            const float p = ex2(x[h] - (m[h] == -INFINITY ? 0.f : m[h])) * DOWN;
            l[h] += p;
            *reinterpret_cast<float2 *>(ps + 2 * (key * GP + cl * (GP / 4) + h)) = make_float2(p, p);
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < KEYS; ++k) {
            const T *vr = reinterpret_cast<const T *>(stage + (KEYS + k) * rb);
            float4 p[GP / 2];  // the weights of two heads, each twice
#pragma unroll
            for (int h = 0; h < GP / 2; ++h) p[h] = *reinterpret_cast<const float4 *>(ps + 2 * k * GP + 4 * h);
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                const int c = 4 * (lane + 32 * i);
                if (c < dp) {
                    const float4 v = four(vr + c);
#pragma unroll
                    for (int h = 0; h < GP; ++h) {
                        const float2 w = h & 1 ? make_float2(p[h / 2].z, p[h / 2].w) : make_float2(p[h / 2].x, p[h / 2].y);
                        fma2(acc[i][h][0], w, make_float2(v.x, v.y));
                        fma2(acc[i][h][1], w, make_float2(v.z, v.w));
                    }
                }
            }
        }
        __syncwarp();
    }
    __device__ __forceinline__ void close(int) {
#pragma unroll
        for (int h = 0; h < GP / 4; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
        }
    }
    template <typename F, typename G>
    __device__ __forceinline__ void each(int lane, const attn_args &a, F &&f, G &&one) {
#pragma unroll
        for (int h = 0; h < GP / 4; ++h) one((lane & 3) * (GP / 4) + h, m[h], l[h], lane < 4);
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int h = 0; h < GP; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int d = 4 * (lane + 32 * i) + e;
                    if (d < a.D) f(h, d, e & 1 ? acc[i][h][e / 2].y : acc[i][h][e / 2].x);
                }
    }
};

// ---- the kernel over the line of tiles --------------------------------------------------------

// Shared memory: scan words and the tile prefix, then per warp its stages (KEYS rows of K, KEYS of V), then per
// warp the stages' live masks and the new token's place, the heads' sums and what the tile keeps (q), then the
// accumulators that warps of one head add.
constexpr int MAX_NS = 4;  // masks, places and barriers kept a warp
constexpr int WARP_HEAD = MAX_NS * 28;
struct smem_layout {
    int ring, warp, warp_bytes, merge, total;
};
__host__ __device__ inline smem_layout layout_of(int n_seq, int warps, int ns, int stage, int extra, int gp, int merge_warps, int D) {
    smem_layout s;
    s.ring = (128 + (((n_seq + 31) & ~31) + 1) * 4 + 511) & ~511;  // rows of up to 512 bytes start on a multiple of their size
    s.warp = s.ring + warps * ns * stage;
    s.warp_bytes = (WARP_HEAD + 3 * gp * 4 + extra + 15) & ~15;
    s.merge = s.warp + warps * s.warp_bytes;
    s.total = s.merge + merge_warps * gp * D * 4;
    return s;
}

template <class Tile>
__global__ void __launch_bounds__(Tile::WARPS * (Tile::SPLIT ? 48 : 32), 1)
    k_attn_batch(const __grid_constant__ attn_args a, int ns) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int KEYS = Tile::KEYS, GP = Tile::GP;
    constexpr bool SPLIT = Tile::SPLIT;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = a.D, HG = a.hg, R = a.rsplit, hs = warp % HG, r = warp / HG, warps = HG * R;
    const int stage_bytes = Tile::stage_bytes(D);
    const smem_layout S = layout_of((int)a.n_seq, warps, ns, stage_bytes, Tile::extra_bytes(D), GP, warps - HG, D);
    int *sums = reinterpret_cast<int *>(smem), *pre = sums + 32;
    volatile int *abort = sums + 31;  // past what the scan's warps use
    // a computing warp's: the new token's place in a pool, where its tile is; SPLIT: its stages' barriers;
    // the stages' live keys
    auto ring_of = [&](int w) { return smem + S.ring + w * ns * stage_bytes; };
    auto slots_of = [&](int w) { return reinterpret_cast<long long *>(smem + S.warp + w * S.warp_bytes); };
    auto full_of = [&](int w) { return reinterpret_cast<uint64_t *>(slots_of(w) + MAX_NS); };
    auto empty_of = [&](int w) { return full_of(w) + MAX_NS; };
    auto masks_of = [&](int w) { return reinterpret_cast<unsigned *>(empty_of(w) + MAX_NS); };
    auto warp_heads = [&](int w) { return reinterpret_cast<float *>(smem + S.warp + w * S.warp_bytes + WARP_HEAD); };
    float *hm = warp_heads(warp), *hl = hm + GP, *ff = hl + GP;
    uint8_t *extra = reinterpret_cast<uint8_t *>(ff + GP);
    if (SPLIT && warp < warps && lane == 0) {
        for (int i = 0; i < ns; ++i) {
            tc::bar_init(full_of(warp) + i, 33);  // a lane's copies each, and the note
            tc::bar_init(empty_of(warp) + i, 1);
        }
        tc::bar_init_fence();
    }
    // rows' tails past head_dim hold zeros: no copy writes there
    if (Tile::padded(D))
        for (int i = threadIdx.x * 16; i < warps * ns * stage_bytes; i += blockDim.x * 16)
            *reinterpret_cast<uint4 *>(smem + S.ring + i) = make_uint4(0, 0, 0, 0);
    pdl_trigger();
    pdl_wait();

    // The line of tiles: R x KEYS keys each, from a multiple of KEYS on, rows in batch order, the head groups one after another.
    int run = 0;
    for (unsigned b = 0; b < a.n_seq; b += blockDim.x) {
        const unsigned i = b + threadIdx.x;
        unsigned row, lo = 0, hi = 0;
        if (i < a.n_seq) span_of(a, i, row, lo, hi);
        int total;
        const int upto = block_scan(lo < hi ? (int)((hi - lo / KEYS * KEYS + R * KEYS - 1) / (R * KEYS)) : 0, sums, &total);
        if (i < a.n_seq) pre[i + 1] = run + upto;
        run += total;
    }
    if (threadIdx.x == 0) {
        pre[0] = 0;
        *abort = 0;
    }
    __syncthreads();
    const int line = run, T = line * a.nhg;  // below 2^31: the host has seen to it
    const int ctas = min((int)gridDim.x, max(1, T));
    // rows without keys are zero
    for (int i = blockIdx.x; i < (int)a.n_seq; i += gridDim.x)
        if (pre[i] == pre[i + 1])
            for (int e = threadIdx.x; e < a.n_heads * D; e += blockDim.x) a.out[(size_t)i * a.n_heads * D + e] = 0.f;
    if ((int)blockIdx.x >= ctas || T == 0) {
        if (threadIdx.x == 0) a.notes[blockIdx.x] = make_int4(0, 0, 0, 0);
        return;
    }
    const runs parts(T, ctas);
    const int g0 = parts.start((int)blockIdx.x), g1 = parts.start((int)blockIdx.x + 1);

    int s0;
    {
        const int x = g0 % line;
        int lo = 0, hi = (int)a.n_seq;  // pre[lo] <= x < pre[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (pre[mid] <= x) lo = mid;
            else hi = mid;
        }
        s0 = lo;
    }
    const int h0g = g0 / line;
    if (threadIdx.x == 0) a.notes[blockIdx.x] = note_of(parts, (int)blockIdx.x, s0, h0g * HG, h0g * line + pre[s0], h0g * line + pre[s0 + 1]);
    auto next_row = [&](int &s, int &h) {
        do {
            if (++s == (int)a.n_seq) {
                s = 0;
                ++h;
            }
        } while (pre[s + 1] == pre[s]);
    };

    // The loading side runs ns - 1 tiles ahead of the computing side, across rows: the same warp, or
    // (SPLIT) a warp of its own for every two computing ones.
    constexpr int SERVED = SPLIT ? 2 : 1;
    const int apart = SPLIT ? (int)(blockDim.x >> 5) - warps : 0, first_w = SPLIT ? warp - warps : warp;
    int lg = g0, lend, ls = s0, lh = h0g, lstage = 0;
    unsigned lrow, llo, lhi, lnew, lslot[SERVED] = {}, lpage[SERVED], lj[SERVED] = {};
    const unsigned *ltab;
    auto enter = [&]() {
        span_of(a, (unsigned)ls, lrow, llo, lhi);
        ltab = a.tables + (size_t)lrow * a.max_pages;
        lend = lh * line + pre[ls + 1];
        lnew = a.k_new ? a.n_kv[lrow] - 1 : 0xffffffffu;
    };
    // the table entry of the next tile's key `lane`, asked for one tile early
    const long long to_v = a.v - a.k;
    auto look_up = [&]() {
        const unsigned t = (unsigned)(lg - lh * line - pre[ls]);
#pragma unroll
        for (int q = 0; q < SERVED; ++q) {
            lj[q] = llo / KEYS * KEYS + (t * R + (first_w + q * apart) / HG) * KEYS + lane;
            lpage[q] = NO_PAGE;
            if (lane < KEYS && lj[q] >= llo && lj[q] < lhi) {
                unsigned e;
                place_of(a, lj[q], e, lslot[q]);
                lpage[q] = ltab[e];
            }
        }
    };
    auto copy_tile = [&](int q, int w) {
        const bool in = lpage[q] < a.n_pages;
        const size_t head = (size_t)((lh * HG + w % HG) / a.subs) * a.head_bytes;
        const long long off = in ? (long long)(((size_t)lpage[q] * a.pt + lslot[q]) * a.token_bytes + head) : -1;
        const unsigned mask = __ballot_sync(0xffffffffu, in);
        uint8_t *stage = ring_of(w) + lstage * stage_bytes;
        if (lane == 0) masks_of(w)[lstage] = mask;
        if (in && lj[q] == lnew) slots_of(w)[lstage] = off;
        if (a.one_page && mask == (1u << KEYS) - 1) Tile::load_run(stage, a.k + __shfl_sync(0xffffffffu, off, 0), to_v, a, lane);
        else Tile::load_rows(stage, off, a, lane);
    };
    auto advance = [&]() {
        lstage = lstage + 1 == ns ? 0 : lstage + 1;
        if (++lg < g1) {
            if (lg == lend) {
                next_row(ls, lh);
                enter();
            }
            look_up();
        }
    };
    auto issue = [&]() {
        if (lg < g1) {
            copy_tile(0, first_w);
            advance();
        }
        cp_commit();
    };
    int *status = reinterpret_cast<int *>(a.status);
    constexpr int WAIT = (int)MOEARC_X_KV_WAIT;
    if (SPLIT && warp >= warps) {
        enter();
        look_up();
        for (unsigned phase = 1; lg < g1; advance()) {  // the first round waits for nothing
#pragma unroll
            for (int q = 0; q < SERVED; ++q) {
                const int w = first_w + q * apart;
                if (w >= warps) break;
                const bool ok = lg - g0 < ns || tc::bar_wait(empty_of(w) + lstage, phase, abort, status, WAIT);
                if (!__all_sync(0xffffffffu, ok)) {
                    cp_commit();
                    cp_wait<0>();
                    return;
                }
                copy_tile(q, w);
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full_of(w) + lstage)) : "memory");
                __syncwarp();
                if (lane == 0) tc::bar_arrive(full_of(w) + lstage);
            }
            if (lstage == ns - 1) phase ^= 1;
        }
        cp_commit();
        cp_wait<0>();
        return;
    }
    if constexpr (!SPLIT) {
        enter();
        look_up();
    }

    auto compute_sync = [&]() { asm volatile("barrier.cta.sync 1, %0;" ::"r"(warps * 32) : "memory"); };
    Tile tile;
    int s = s0, h = h0g, cstage = 0, ahead = ns - 1;
    unsigned cphase = 0;
    for (int g = g0; g < g1; next_row(s, h)) {
        const int u0 = h * line + pre[s], u1 = h * line + pre[s + 1], first = g, end = min(u1, g1);
        unsigned row, lo, hi;
        span_of(a, (unsigned)s, row, lo, hi);
        const int vh = h * HG + hs, kvh = vh / a.subs, sub = vh - kvh * a.subs;
        const int h0 = kvh * a.group + sub * GP, heads = min(GP, a.group - sub * GP);
        const unsigned newest = a.k_new ? a.n_kv[row] - 1 : 0xffffffffu;
        tile.init(a.q + (size_t)s * a.q_stride + (size_t)h0 * D, heads, a, extra, lane);
        for (; g < end; ++g) {
            bool ok = true;
            if constexpr (SPLIT) {
                ok = __all_sync(0xffffffffu, tc::bar_wait(full_of(warp) + cstage, cphase, abort, status, WAIT));
            } else {
                for (; ahead >= 0; --ahead) issue();  // one a tile, ns before the first
                ahead = 0;
                if (ns == 3) cp_wait<2>();
                else cp_wait<1>();
                __syncwarp();
            }
            uint8_t *stage = ring_of(warp) + cstage * stage_bytes;
            const unsigned live = ok ? masks_of(warp)[cstage] : 0, j0 = lo / KEYS * KEYS + ((unsigned)(g - u0) * R + r) * KEYS;
            if (newest >= j0 && newest - j0 < KEYS && (live >> (newest - j0) & 1)) {
                const unsigned at = newest - j0;
                const size_t dst = (size_t)slots_of(warp)[cstage];
                const size_t src = (size_t)s * a.new_stride + (size_t)kvh * D;
                Tile::round_row(a.k_new + src, stage, (int)at, sub == 0 ? a.k + dst : nullptr, a, lane);
                Tile::round_row(a.v_new + src, stage, (int)(KEYS + at), sub == 0 ? a.v + dst : nullptr, a, lane);
                __syncwarp();
            }
            if (live) tile.step(stage, live, a, extra, lane);
            __syncwarp();
            if (SPLIT && lane == 0) tc::bar_arrive(empty_of(warp) + cstage);
            if (++cstage == ns) {
                cstage = 0;
                cphase ^= 1;
            }
        }

        // Close the row or its part: the head's warps are added into its first, which writes.
        tile.close(lane);
        tile.each(lane, a, [](int, int, float &) {}, [&](int hd, float m, float l, bool mine) {
            if (mine) {
                hm[hd] = m;
                hl[hd] = l;
            }
        });
        __syncwarp();
        auto merge_of = [&](int rr) { return reinterpret_cast<float *>(smem + S.merge) + ((size_t)(rr - 1) * HG + hs) * GP * D; };
        if (R > 1) {
            if (r > 0) {
                float *b = merge_of(r);
                tile.each(lane, a, [&](int hd, int d, float &o) { b[hd * D + d] = o; }, [](int, float, float, bool) {});
            }
            compute_sync();
            if (r == 0) {
                if (lane < GP) {
                    float M = -INFINITY, sum = 0.f;
                    for (int w = 0; w < R; ++w) M = fmaxf(M, warp_heads(w * HG + hs)[lane]);
                    for (int w = 0; w < R; ++w) {
                        float *o = warp_heads(w * HG + hs);
                        const float f = o[lane] == -INFINITY ? 0.f : ex2(o[lane] - M);
                        sum += o[GP + lane] * f;
                        o[2 * GP + lane] = f;
                    }
                    hm[lane] = M;
                    hl[lane] = sum;
                }
                __syncwarp();
                tile.each(lane, a, [&](int hd, int d, float &o) {
                    float v = o * ff[hd];
#pragma unroll 1
                    for (int w = 1; w < R; ++w) v = fmaf(merge_of(w)[hd * D + d], warp_heads(w * HG + hs)[2 * GP + hd], v);
                    o = v;
                }, [](int, float, float, bool) {});
                __syncwarp();
            }
        }
        if (r == 0) {
            const bool whole = first == u0 && end == u1;
            float *part = nullptr;
            if (whole) {
                if (lane < heads) {
                    float M = hm[lane], sum = hl[lane], f = 1.f;
                    if (a.sinks) {
                        const float sk = a.sinks[h0 + lane] * LOG2E, top = fmaxf(M, sk);
                        f = M == -INFINITY ? 0.f : ex2(M - top);
                        sum = sum * f + (sk == -INFINITY ? 0.f : ex2(sk - top) * DOWN);
                    }
                    ff[lane] = sum == 0.f ? 0.f : f / sum;
                }
            } else {
                part = a.part + (((size_t)blockIdx.x * 2 + (first == g0 ? 0 : 1)) * HG + hs) * GP * (D + 2);
                if (lane < GP) {
                    part[GP * D + 2 * lane] = hm[lane];
                    part[GP * D + 2 * lane + 1] = hl[lane];
                }
            }
            __syncwarp();
            float *out = a.out + ((size_t)s * a.n_heads + h0) * D;
            tile.each(lane, a, [&](int hd, int d, float &o) {
                if (!whole) part[hd * D + d] = o;
                else if (hd < heads) out[(size_t)hd * D + d] = o * ff[hd];
            }, [](int, float, float, bool) {});
        }
        if (R > 1) compute_sync();  // the sums and accumulators are free for the next row
        else __syncwarp();
    }
}

// The rows of a listed batch into the work buffer: by value into a launch of their own, so that the
// launches that have none to pass stay short.
template <int N>
struct seq_list {
    unsigned row[N];
};
template <int N>
__global__ void __launch_bounds__(KV_LIST) k_attn_rows(const __grid_constant__ seq_list<N> L, unsigned n, unsigned *rows) {
    pdl_trigger();
    pdl_wait();
    if (threadIdx.x < n) rows[threadIdx.x] = L.row[threadIdx.x];
}
template <typename F>
cudaError_t with_list(const unsigned *rows, unsigned n, F &&f) {
    auto fill = [&](auto &L) {
        std::copy(rows, rows + n, L.row);
        return f(L);
    };
    if (n <= 64) {
        seq_list<64> L;
        return fill(L);
    }
    seq_list<KV_LIST> L;
    return fill(L);
}

// ---- host side --------------------------------------------------------------------------------

// Whether the tensor cores serve a shape, where the pools' rows are 16-byte aligned: multiples of 8
// channels of 16 bits and of 4 channels of f32, from the size at which half of the smallest tile is
// used on. CUDA cores have the rest. f32 heads without a group go the same way: they leave seven of eight rows of an
// MMA empty and are level with CUDA cores or ahead of them (30 rows to 6000 and 200 to 500 tokens: 8 heads of 64 105
// and 81 us, 156 and 120 on CUDA cores; 7 of 72 158 and 118, 154 and 122).
bool tensor_dim(unsigned D, unsigned kv_type) { return D > 32 && D <= 256 && D % (kv_type == T_F32 ? 4 : 8) == 0; }
// Of the latter, up to 128 channels whose kv heads serve four query heads at most take half the
// arithmetic with tiles of four heads.
bool few_heads(unsigned D, int group) { return D <= 128 && group <= 4; }

template <class Tile>
bool cut(attn_plan &p, int warps, int ns, int n_heads, int n_kv, int D, int n_seq, int sms) {
    p.gp = Tile::GP;
    p.keys = Tile::KEYS;
    const int group = n_heads / n_kv;
    p.subs = (group + p.gp - 1) / p.gp;
    const int V = n_kv * p.subs;
    p.hg = 1;
    for (int d = 2; d <= warps; ++d)
        if (V % d == 0) p.hg = d;
    p.rsplit = warps / p.hg;
    p.nhg = V / p.hg;
    p.warps = p.hg * p.rsplit;
    p.ns = ns;
    p.smem = layout_of(n_seq, p.warps, ns, Tile::stage_bytes(D), Tile::extra_bytes(D), p.gp, p.warps - p.hg, D).total;
    if (p.smem > MAX_SMEM - 512) return false;
    p.grid = sms;
    return true;
}

// Three stages where the tile's warps have them, else two, else fewer warps.
template <class Tile>
bool cut_any(attn_plan &p, int n_heads, int n_kv, int D, int n_seq, int sms) {
    for (int warps = Tile::WARPS; warps >= 1; warps /= 2)
        for (int ns = 3; ns >= 2; --ns)
            if (cut<Tile>(p, warps, ns, n_heads, n_kv, D, n_seq, sms)) return true;
    return false;
}

// f(a null pointer to the tile) for the tile that serves a shape.
template <typename F>
auto with_tile(bool mma, unsigned kv_type, unsigned D, int group, F &&f) {
    if (mma) {  // f32: attn_tc.cu has the 16-bit ones
        // 16 keys a tile take fewer instructions a key, 8 let twice the warps' stages fit. So 8 above 128
        // channels (16 query heads over 1 of 256, 30 rows of up to 6000: 159 us, 278 with 16), and above 80
        // where each kv head is one unit (32 over 8 of 128: 217 and 260; 48 over 3, two units a kv head: 212
        // and 188, its second unit's keys coming from L2); 16 below (64 over 8 of 64: 107, 155 with 8).
        if (D <= 64) return f((tf32_tile<64, 16> *)nullptr);
        if (D <= 80) return f((tf32_tile<80, 16> *)nullptr);
        if (D <= 128) return group > 8 ? f((tf32_tile<128, 16> *)nullptr) : f((tf32_tile<128, 8> *)nullptr);
        return f((tf32_tile<256, 8> *)nullptr);
    }
#define CORE_CASE(T)                                                                                  \
    if (few_heads(D, group)) return f((core_tile<T, 1, 4> *)nullptr); \
    if (D <= 128) return f((core_tile<T, 1, 8> *)nullptr);          \
    if (D <= 256) return f((core_tile<T, 2, 8> *)nullptr);          \
    if (D <= 512) return f((core_tile<T, 4, 4> *)nullptr);          \
    return f((core_tile<T, 8, 4> *)nullptr);
    if (kv_type == T_F32) {
        CORE_CASE(float)
    } else if (kv_type == T_F16) {
        CORE_CASE(__half)
    }
    CORE_CASE(__nv_bfloat16)
#undef CORE_CASE
}

bool plan_of(attn_plan &p, bool mma, unsigned kv_type, int n_heads, int n_kv, int D, int n_seq, int sms) {
    return with_tile(mma, kv_type, (unsigned)D, n_heads / n_kv, [&](auto *t) {
        using Tile = std::remove_pointer_t<decltype(t)>;
        return cut_any<Tile>(p, n_heads, n_kv, D, n_seq, sms);
    });
}

// The work buffer: the rows' list, a note a CTA, then the parts.
size_t attn_bytes(const attn_plan &p, int D) {
    return KV_LIST * 4 + (size_t)p.grid * 16 + (size_t)p.grid * 2 * p.hg * p.gp * (D + 2) * 4;
}
// Most query heads that an SM's CTA works on at once, hg x gp: 16 x 8 (CUDA cores) up to 128 channels,
// 8 warps of 8 or of 4 heads above; attn_tc.cu's two CTAs of one head group are fewer.
int heads_of_sm(unsigned D) { return D <= 128 ? 128 : D <= 256 ? 64 : 32; }

template <class Tile>
cudaError_t launch(moearc_ctx *c, const attn_plan &p, const attn_args &a) {
    static std::atomic<bool> done[MOEARC_MAX_DEVICES];
    cudaError_t e = once_per_device(done, [] {
        return set_smem(k_attn_batch<Tile>, MAX_SMEM - 512);
    });
    if (e == cudaSuccess)
        e = launch_pdl(k_attn_batch<Tile>, dim3((unsigned)p.grid), dim3((unsigned)(p.warps + (Tile::SPLIT ? (p.warps + 1) / 2 : 0)) * 32), (size_t)p.smem, c->stream, a, p.ns);
    if (e == cudaSuccess) e = attn_join_launch<Tile::GP>(c, p.grid, a);
    return e;
}

}  // namespace

extern "C" {

unsigned long moearc_x_kv_work_bytes(moearc_ctx *c, const moearc_x_kv_cache *kv, unsigned int n_heads) {
    if (!c || !kv || !kv_shape_ok(*kv)) return 0;
    size_t need = kv_page_work_bytes(kv->n_pages);
    if (n_heads) {
        if (n_heads > 65535 || n_heads % kv->n_kv_heads) return 0;
        // the cut goes by the batch, the heads and the pools' alignment: the most that any takes
        const int D = (int)kv->head_dim;
        attn_plan p;
        if (!plan_of(p, false, kv->kv_type, (int)n_heads, (int)kv->n_kv_heads, D, (int)KV_LIST, c->sm_count)) return 0;
        need = std::max(need, KV_LIST * 4 + (size_t)c->sm_count * (2 * 16 + 2 * (size_t)heads_of_sm(kv->head_dim) * (D + 2) * 4));
    }
    return need;
}

int moearc_x_attn_decode_batch(moearc_ctx *c, const moearc_x_kv_cache *kv, unsigned int layer, float *out, const float *q,
                               unsigned long q_stride, const float *k_new, const float *v_new, unsigned long new_stride,
                               const unsigned int *seqs, const unsigned int *kv_begin, const float *sinks, unsigned int n_seq,
                               unsigned int n_heads, float scale) {
    const int rc = kv_check(c, kv);
    if (rc) return rc;
    if (!out || !q || (!k_new) != (!v_new)) return ERR;
    for (const void *p : {static_cast<const void *>(out), static_cast<const void *>(q), static_cast<const void *>(k_new),
                          static_cast<const void *>(v_new), static_cast<const void *>(kv_begin), static_cast<const void *>(sinks)})
        if (!aligned(p, 4)) return ERR_ARG;
    if (layer >= kv->n_layer || n_heads == 0 || n_heads > 65535 || n_heads % kv->n_kv_heads || n_seq > KV_LIST) return ERR_ARG;
    if (n_seq == 0) return OK;
    const size_t D = kv->head_dim;
    if (q_stride < n_heads * D || (k_new && new_stride < kv->n_kv_heads * D)) return ERR_ARG;
    if (!(scale == scale) || scale - scale != 0.f) return ERR_ARG;
    if (seqs) {
        kv_rows_seen seen(kv->max_seq);
        for (unsigned i = 0; i < n_seq; ++i)
            if (!seen.add(seqs[i], kv->max_seq)) return ERR_ARG;
    } else if (n_seq > kv->max_seq) {
        return ERR_ARG;
    }
    const uintptr_t align = reinterpret_cast<uintptr_t>(kv->k_pages[layer]) | reinterpret_cast<uintptr_t>(kv->v_pages[layer]);
    const bool mma = tensor_dim(kv->head_dim, kv->kv_type) && (align & 15) == 0, tc = mma && kv->kv_type != T_F32;
    // tokens are numbered in 32 bits there; more of them than that would not fit the memory
    if (tc && (unsigned long long)kv->n_pages * kv->page_tokens >= (1ull << 31)) return ERR_ARG;
    attn_plan p = {};
    if (tc) attn_tc_plan(p, (int)n_heads, (int)kv->n_kv_heads, (int)D, c->sm_count);
    else if (!plan_of(p, mma, kv->kv_type, (int)n_heads, (int)kv->n_kv_heads, (int)D, (int)n_seq, c->sm_count)) return ERR_ARG;
    if (kv->work_bytes < attn_bytes(p, (int)D)) return ERR_ARG;
    const unsigned cap = kv->max_pages * kv->page_tokens;
    if ((unsigned long long)n_seq * (cap / (unsigned)(p.keys * p.rsplit) + 2) * p.nhg * p.hg >= (1ull << 31)) return ERR_ARG;

    attn_args a;
    a.out = out;
    a.q = q;
    a.k_new = k_new;
    a.v_new = v_new;
    a.sinks = sinks;
    a.k = static_cast<uint8_t *>(kv->k_pages[layer]);
    a.v = static_cast<uint8_t *>(kv->v_pages[layer]);
    a.tables = kv->tables;
    a.n_kv = kv->n_kv;
    a.begin = kv_begin;
    a.q_stride = q_stride;
    a.new_stride = new_stride;
    a.token_bytes = (size_t)kv->n_kv_heads * D * kv_elem_bytes(kv->kv_type);
    a.head_bytes = D * kv_elem_bytes(kv->kv_type);
    a.n_seq = n_seq;
    a.max_pages = kv->max_pages;
    a.n_pages = kv->n_pages;
    a.pt = kv->page_tokens;
    a.pt_inv = (unsigned)std::min(0xffffffffull, (1ull << 32) / kv->page_tokens);
    a.cap = cap;
    const uintptr_t rows = align | a.head_bytes;
    a.unit = (rows & 15) == 0 ? 16 : (rows & 3) == 0 ? 4 : 2;
    a.one_page = a.unit == 16 && kv->page_tokens % (unsigned)p.keys == 0;
    a.n_heads = (int)n_heads;
    a.group = (int)(n_heads / kv->n_kv_heads);
    a.D = (int)D;
    a.subs = p.subs;
    a.hg = p.hg;
    a.rsplit = p.rsplit;
    a.nhg = p.nhg;
    a.scale2 = scale * LOG2E;
    a.status = kv->status;
    a.rows = seqs ? static_cast<unsigned *>(kv->work) : nullptr;
    a.notes = reinterpret_cast<int4 *>(static_cast<uint8_t *>(kv->work) + KV_LIST * 4);
    a.part = reinterpret_cast<float *>(a.notes + p.grid);
    device_guard g(c->device);
    if (!g.ok) return ERR;
    launch_scope ls(c, "attn_decode_batch", n_seq, n_heads);
    cudaError_t e = cudaSuccess;
    if (seqs)
        e = with_list(seqs, n_seq, [&](auto &L) {
            constexpr int N = (int)(sizeof(L.row) / sizeof(unsigned));
            return launch_pdl(k_attn_rows<N>, dim3(1), dim3(KV_LIST), 0, c->stream, L, n_seq, static_cast<unsigned *>(kv->work));
        });
    if (e == cudaSuccess) e = tc ? attn_tc_launch(c, p, kv->kv_type, a) : with_tile(mma, kv->kv_type, kv->head_dim, a.group, [&](auto *t) {
        return launch<std::remove_pointer_t<decltype(t)>>(c, p, a);
    });
    if (e != cudaSuccess) cudaGetLastError();  // the failed launch's error, not left for an unrelated later check
    const int rc2 = ls.finish();
    return e != cudaSuccess ? ERR : rc2;
}

}  // extern "C"
