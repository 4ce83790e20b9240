// attn_tc.cu — decode attention of a ragged batch over the paged cache on the fifth-generation
// tensor cores: 16-bit caches of up to 256 channels, a multiple of 8 above 32 (attn_batch.cu serves
// the rest; the formula, the equal runs and the join are the same).
//
// A unit is a batch row and a kv head (with up to eight of its query heads); its keys are cut into
// tiles of 128, and each CTA takes an equal run of all units' tiles. Per tile:
//
//   S [128 keys x 32] = K Q'     K as the A operand from shared memory, K-major
//   p = 2^(S - m), thread = key  eight heads a thread, from tensor memory
//   O [channels x 32] = V' P     V as it was loaded (channel-major) as the A operand, P from the threads
//
// Measured: 3 rows of up to 100001 tokens, 8 heads of 128, f16, 1.08 GB: 172 us, 6.3 TB/s of a measured 6.56
// (164 us); 64 rows of up to 4096, 4 heads of 128, bf16, 362 MB: 71 us (55), of which about 12 are the start
// (lengths, tables, the first tile's way through the roles) and the join; 120 rows of 128 tokens, 8 heads
// of 64: 19 us (5). The tensor pipe is 9% busy: HBM bounds long rows, the chain from load to weights to
// output short ones. On mma.sync the first two took 193 and 93 us.
//
// The 32 columns are the 16-bit terms of eight heads, three each of q and of p. f16's range is short: p's second
// and third terms are 2^11 and 2^22 times as fine, so that a weight has 22 bits down to 2^-35 of its row's
// largest (24 natural units of score) and the last of them at 2^-57; a row whose largest weights have
// values of zero is made of the small ones. (200 rows of up to 500, 64/8 x 64, f16: 57 us, 54 with two plain
// terms.) The tensor core sums a tile (8 MMAs) and the threads, now one a channel, add the columns of a
// head to f32 registers, since its sums truncate and a long row's would show it.
//
// Two tiles are in flight or in use (one of 256 channels, its keys loaded again while its weights are
// worked out: 16 heads over 1 of 256 channels, 30 rows of up to 6000, 50 us, 94 on mma.sync). They are loaded by 16-byte asynchronous copies, two warps a
// stage: any page size, and as many bytes under way as the stages hold. (TMA boxes of 128-byte rows
// brought 3.5 TB/s and untiled bulk copies of a row 4, where these bring 6.2: one head of a token is
// 128 or 256 bytes in a row of thousands.) Roles, each a warp or more that meet at mbarriers: loads; MMA issue; four warps of
// softmax; two warps that split the next unit's queries into terms ahead of its first tile. Keys are
// given back for loading as soon as S is computed, values once O is. Every wait has a limit
// (tc.cuh): one that runs out raises MOEARC_X_KV_WAIT and ends the kernel.
#include <algorithm>

#include "attn_batch.cuh"
#include "tc.cuh"

using namespace moearc;

namespace {

constexpr int KEYS = 128, GP = 8, NT = 32;
// Warps: softmax 0-3, MMA of S 4, loads 5-8 (two a stage, or all four for the one), queries 9-10, MMA of O 11.
constexpr int THREADS = 384, LOAD_THREADS = 128;
constexpr int FIRST = 1, LAST = 2, WHOLE = 4, SECOND = 8;

struct tile_meta {
    int flags, row, vh;
    unsigned live[4];
};

template <int D>
struct tc_smem {
    // Stages of K and V: two, or one where two do not fit (a tile of 256 channels is 128 KB; its keys'
    // half is loaded again while the weights are worked out). S, the weights, O and q are in two places either way.
    static constexpr int NS = D <= 128 ? 2 : 1, LOADERS = LOAD_THREADS / NS;
    static constexpr int TMEM = D <= 128 ? 128 : 256;  // columns: two of S, then two of O for each 128 channels
    static constexpr int MAT = KEYS * D * 2;       // a tile's keys (or values)
    static constexpr int Q = NT * D * 2, P = KEYS * NT * 2;
    static constexpr int STAGE = 2 * MAT;
    static constexpr int at_q = NS * STAGE, at_p = at_q + 2 * Q, at_bar = at_p + 2 * P;
    static constexpr int at_meta = at_bar + 24 * 8, at_scale = at_meta + 2 * (int)sizeof(tile_meta), at_red = at_scale + 8 * 2 * GP * 4;
    static constexpr int at_max = at_red + 2 * 4 * GP * 4, at_tok = at_max + 2 * 4 * GP * 4;
    static constexpr int at_scan = at_tok + NS * KEYS * 4, at_pre = at_scan + 128 + 16;
    // the tile prefix, then each row's first key and end (bit 31: the end was cut to the table); 1024:
    // room to align the stages
    static constexpr int total(int n_seq) { return at_pre + (3 * n_seq + 1) * 4 + 1024; }
};

// Descriptor of an operand whose M (or N) index is contiguous, K rows one after another: V in rows
// of 128 bytes (128-byte swizzle; `lbo` bytes from 64 channels to the next 64, 1024 from 8 keys to the
// next 8), P in rows of 64 bytes (64-byte swizzle; 512 from 8 keys to the next 8).
__device__ __forceinline__ uint64_t desc_v(uint32_t addr, uint32_t lbo) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)((lbo >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t desc_p(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)(512 >> 4) << 16 | (uint64_t)(512 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)4 << 61;
}
// 32 consecutive f32 columns of this thread's tensor memory lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
        "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// A 16-byte copy where `on`, zeros in its place where not `valid`.
__device__ __forceinline__ void cp_async16p(unsigned dst, const void *src, bool valid, bool on) {
    asm volatile(
        "{ .reg .pred p; setp.ne.s32 p, %3, 0; @p cp.async.cg.shared.global [%0], [%1], 16, %2; }" ::"r"(dst),
        "l"(src), "r"(valid ? 16 : 0), "r"((int)on)
        : "memory");
}
// Eight values a lane over the warp, by op: 9 exchanges, each step leaving a lane half as many. The
// result of value (lane / 4) is in lanes 4 (lane / 4) ...
template <typename Op>
__device__ __forceinline__ float reduce8(const float (&v)[8], int lane, Op op) {
    float a[4], b[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float keep = lane & 16 ? v[i + 4] : v[i], give = lane & 16 ? v[i] : v[i + 4];
        a[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, 16));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float keep = lane & 8 ? a[i + 2] : a[i], give = lane & 8 ? a[i] : a[i + 2];
        b[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, 8));
    }
    float c = op(lane & 4 ? b[1] : b[0], __shfl_xor_sync(0xffffffffu, lane & 4 ? b[0] : b[1], 4));
    c = op(c, __shfl_xor_sync(0xffffffffu, c, 2));
    return op(c, __shfl_xor_sync(0xffffffffu, c, 1));
}
// Barriers of a stage's load warps, then of the four softmax warps, and with it whether any thread's `x` holds.
template <int N>
__device__ __forceinline__ void load_sync(int st) {
    if (st) asm volatile("barrier.cta.sync 3, %0;" ::"n"(N) : "memory");
    else asm volatile("barrier.cta.sync 2, %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void soft_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool soft_any(bool x) {
    int r;
    asm volatile(
        "{ .reg .pred p, q; setp.ne.s32 p, %1, 0; barrier.cta.red.or.pred q, 1, 128, p; selp.s32 %0, 1, 0, q; }"
        : "=r"(r)
        : "r"((int)x)
        : "memory");
    return r != 0;
}

// DP: the channels that tiles have room for, 64, 128 or 256; head_dim is that (FULL) or less.
template <int DP, bool FULL, bool BF>
__global__ void __launch_bounds__(THREADS, DP == 64 ? 2 : 1)
    k_attn_tc(const __grid_constant__ attn_args a) {
    using S = tc_smem<DP>;
    const int D = FULL ? DP : a.D;
    constexpr int CH = DP / 8, TERMS = 3, NS = S::NS, LOADERS = S::LOADERS, MH = DP <= 128 ? 1 : DP / 128;
    constexpr float PSCALE = BF ? 1.f : 32768.f;  // of the weights' terms
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (((tc::sa(smem_raw) + 1023u) & ~1023u) - tc::sa(smem_raw));
    auto *bars = reinterpret_cast<uint64_t *>(smem + S::at_bar);
    uint64_t *kfull = bars, *vfull = bars + 2, *empty = bars + 4, *qfull = bars + 6, *qempty = bars + 8, *sfull = bars + 10,
             *pfull = bars + 12, *ofull = bars + 14, *qready = bars + 16, *done = bars + 20;
    auto *meta = reinterpret_cast<volatile tile_meta *>(smem + S::at_meta);
    // of eight units: a unit's are read until its close, when the queries may be four units ahead
    auto *scales = reinterpret_cast<float *>(smem + S::at_scale);
    auto *scan = reinterpret_cast<int *>(smem + S::at_scan);
    volatile int *abort = scan + 32;
    auto *tslot = reinterpret_cast<uint32_t *>(scan + 33);
    int *pre = reinterpret_cast<int *>(smem + S::at_pre);
    unsigned *first_key = reinterpret_cast<unsigned *>(pre + a.n_seq + 1), *end_key = first_key + a.n_seq;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int *status = reinterpret_cast<int *>(a.status);
    constexpr int WAIT = (int)MOEARC_X_KV_WAIT;

    // channels past head_dim are zeros in the keys and in q, and never written again
    if (D < DP)
        for (int i = threadIdx.x * 16; i < S::at_p; i += THREADS * 16) *reinterpret_cast<uint4 *>(smem + i) = make_uint4(0, 0, 0, 0);
    fence_async();
    if (warp == 4) tc::tmem_alloc(tslot, S::TMEM);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            tc::bar_init(kfull + i, LOADERS);
            tc::bar_init(vfull + i, LOADERS);
            tc::bar_init(empty + i, 1);
            tc::bar_init(qfull + i, 64);
            tc::bar_init(qempty + i, 1);
            tc::bar_init(sfull + i, 1);
            tc::bar_init(pfull + i, 128);
            tc::bar_init(ofull + i, 1);
        }
        for (int i = 0; i < 4; ++i) tc::bar_init(qready + i, 64);
        tc::bar_init(done, 2);
        tc::bar_init_fence();
        *abort = 0;
    }
    // The kernel after this one may start once every CTA here has its tensor memory: one that
    // allocates its own early can then not be what a CTA of this kernel waits for.
    __syncthreads();
    pdl_trigger();
    pdl_wait();

    // The line of tiles: rows in batch order, within a row its virtual heads, within those 128 keys each.
    int run = 0;
    for (unsigned b = 0; b < a.n_seq; b += blockDim.x) {
        const unsigned i = b + threadIdx.x;
        unsigned row = 0, lo = 0, hi = 0;
        if (i < a.n_seq) span_of(a, i, row, lo, hi);
        int total;
        const int upto = block_scan(lo < hi ? (int)((hi - lo + KEYS - 1) / KEYS) : 0, scan, &total);
        if (i < a.n_seq) {
            pre[i + 1] = run + upto;
            first_key[i] = lo;
            end_key[i] = hi | (hi < a.n_kv[row] ? 1u << 31 : 0);
        }
        run += total;
    }
    if (threadIdx.x == 0) pre[0] = 0;
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tslot;
    const int V = a.nhg, T = run * V;  // V: virtual heads; below 2^31: the host has seen to it
    const int ctas = min((int)gridDim.x, max(1, T));
    for (int i = blockIdx.x; i < (int)a.n_seq; i += gridDim.x)
        if (pre[i] == pre[i + 1])
            for (int e = threadIdx.x; e < a.n_heads * D; e += blockDim.x) a.out[(size_t)i * a.n_heads * D + e] = 0.f;

    if ((int)blockIdx.x < ctas && T > 0) {
        const runs parts(T, ctas);
        const int g0 = parts.start((int)blockIdx.x), g1 = parts.start((int)blockIdx.x + 1);
        int s0;
        {
            const int x = g0 / V;
            int lo = 0, hi = (int)a.n_seq;  // pre[lo] <= x < pre[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (pre[mid] <= x) lo = mid;
                else hi = mid;
            }
            s0 = lo;
        }
        const int vh0 = (g0 - V * pre[s0]) / (pre[s0 + 1] - pre[s0]);
        auto unit_start = [&](int s, int vh) { return V * pre[s] + vh * (pre[s + 1] - pre[s]); };
        auto next_unit = [&](int &s, int &vh) {
            if (++vh < V) return;
            vh = 0;
            do ++s;
            while (s < (int)a.n_seq && pre[s + 1] == pre[s]);
        };
        if (threadIdx.x == 0) {
            const int u0 = unit_start(s0, vh0);
            a.notes[blockIdx.x] = note_of(parts, (int)blockIdx.x, s0, vh0, u0, u0 + pre[s0 + 1] - pre[s0]);
        }
        const int n_tiles = g1 - g0;

        if (warp >= 5 && warp < 9) {
            // ---- loads: this group's tiles, every NS-th ------------------------------------------
            const int st = NS == 2 ? (warp - 5) >> 1 : 0, t = threadIdx.x - 160 - st * LOADERS;
            auto *tok = reinterpret_cast<int *>(smem + S::at_tok) + st * KEYS;
            int s = s0, vh = vh0, u0 = unit_start(s, vh), u1 = u0 + pre[s + 1] - pre[s], was = -1;
            constexpr int R = KEYS / LOADERS;  // keys a thread looks up
            unsigned lo = 0, hi = 0, newest = 0, page[R], slot[R];
            const unsigned *tab = nullptr;
            auto look_up = [&](int g) {  // keys t, LOADERS + t ... of tile g, one of the group's tiles early
                while (g >= u1) {
                    next_unit(s, vh);
                    u0 = u1;
                    u1 = u0 + pre[s + 1] - pre[s];
                }
                if (s != was) {
                    was = s;
                    lo = first_key[s];
                    hi = end_key[s] & 0x7fffffffu;
                    tab = a.tables + (size_t)(a.rows ? a.rows[s] : (unsigned)s) * a.max_pages;
                    newest = a.k_new && !(end_key[s] >> 31) ? hi - 1 : 0xffffffffu;
                }
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const unsigned j = lo + (unsigned)(g - u0) * KEYS + r * LOADERS + t;
                    page[r] = NO_PAGE;
                    if (j < hi) {
                        unsigned e;
                        place_of(a, j, e, slot[r]);
                        page[r] = tab[e];
                    }
                }
            };
            if (st < n_tiles) look_up(g0 + st);
            const int ch = t % CH, r0 = t / CH;
            const bool used = ch * 8 < D;
            uint8_t *stage = smem + st * S::STAGE;
            const unsigned d0 = smem_u32(stage) + (ch >> 3) * KEYS * 128;
            constexpr int RW = LOADERS / CH, BATCH = 8;  // rows a step; steps whose rows are looked at together
            auto copy = [&](const uint8_t *pool, unsigned dst) {  // every row but the new token's
#pragma unroll 1
                for (int r = r0; r < KEYS; r += RW * BATCH) {
                    int at[BATCH];
#pragma unroll
                    for (int e = 0; e < BATCH; ++e) at[e] = tok[r + e * RW];
#pragma unroll
                    for (int e = 0; e < BATCH; ++e) {
                        const int q = r + e * RW;
                        cp_async16p(dst + q * 128 + (((ch & 7) ^ (q & 7)) << 4), pool + (size_t)(unsigned)max(at[e], 0) * a.token_bytes, at[e] >= 0, used && at[e] > -2);
                    }
                }
                cp_commit();
            };
            // channel d of the new token's row, rounded, into the tile and its slot
            auto put = [&](int mat, int r, int d, float x, uint8_t *slot_row) {
                const uint16_t b = to16<BF>(x);
                *reinterpret_cast<uint16_t *>(stage + mat * S::MAT + (d >> 6) * KEYS * 128 + r * 128 + (((d >> 3 & 7) ^ (r & 7)) << 4) + (d & 7) * 2) = b;
                if (slot_row) reinterpret_cast<uint16_t *>(slot_row)[d] = b;
            };
            int i = st;
            for (; i < n_tiles; i += NS) {
                const int g = g0 + i;
                // the keys' place is free once S is computed, the values' once O is
                const int was_in = i - NS;  // the stage's last tile
                bool ok = i < NS || tc::bar_wait(sfull + (was_in & 1), (was_in >> 1) & 1, abort, status, WAIT);
                if (!__all_sync(0xffffffffu, ok)) break;
                const unsigned j0 = lo + (unsigned)(g - u0) * KEYS;
                const int kvh = vh / a.subs, at_new = newest >= j0 && newest - j0 < KEYS ? (int)(newest - j0) : -1;
                const int flags = (g == g0 || g == u0 ? FIRST : 0) | (g == g1 - 1 || g == u1 - 1 ? LAST : 0) |
                                  (u0 >= g0 && u1 <= g1 ? WHOLE : 0) | (u0 > g0 ? SECOND : 0);
                const bool stores = vh == kvh * a.subs;
                const int row_i = s, vh_i = vh;
                unsigned m[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const bool in = page[r] < a.n_pages;
                    const int id = in ? (int)(page[r] * a.pt + slot[r]) : -1;
                    m[r] = __ballot_sync(0xffffffffu, in);
                    tok[r * LOADERS + t] = in && r * LOADERS + t == at_new ? -2 - id : id;
                }
                load_sync<LOADERS>(st);
                const size_t head = (size_t)kvh * a.head_bytes;
                copy(a.k + head + ch * 16, d0);
                ok = i < NS || tc::bar_wait(empty + (was_in & 1), (was_in >> 1) & 1, abort, status, WAIT);
                auto &note = meta[i & 1];
                if (lane == 0)
#pragma unroll
                    for (int r = 0; r < R; ++r) note.live[(r * LOADERS + t) >> 5] = m[r];
                if (t == 0) {
                    note.flags = flags;
                    note.row = row_i;
                    note.vh = vh_i;
                }
                copy(a.v + head + ch * 16, d0 + S::MAT);
                constexpr int EACH = DP / LOADERS;
                float kn[EACH], vn[EACH];
                uint8_t *slot_k = nullptr, *slot_v = nullptr;
                const bool fresh = at_new >= 0 && tok[at_new] < -1;
                if (fresh) {
                    const size_t src = (size_t)row_i * a.new_stride + (size_t)kvh * D + t, dst = (size_t)(-2 - tok[at_new]) * a.token_bytes + head;
#pragma unroll
                    for (int e = 0; e < EACH; ++e)
                        if (t + e * LOADERS < D) {
                            kn[e] = a.k_new[src + e * LOADERS];
                            vn[e] = a.v_new[src + e * LOADERS];
                        }
                    if (stores) {
                        slot_k = a.k + dst;
                        slot_v = a.v + dst;
                    }
                }
                if (i + NS < n_tiles) look_up(g + NS);
                cp_wait<1>();
                if (fresh)
#pragma unroll
                    for (int e = 0; e < EACH; ++e)
                        if (t + e * LOADERS < D) put(0, at_new, t + e * LOADERS, kn[e], slot_k);
                fence_async();  // what the copies wrote, before the tensor core reads it
                tc::bar_arrive(kfull + st);
                cp_wait<0>();
                if (fresh)
#pragma unroll
                    for (int e = 0; e < EACH; ++e)
                        if (t + e * LOADERS < D) put(1, at_new, t + e * LOADERS, vn[e], slot_v);
                fence_async();
                tc::bar_arrive(vfull + st);
                if (!__all_sync(0xffffffffu, ok)) break;
            }
            // the MMA's last arrival, before the CTA ends
            if (i >= NS && *abort == 0) tc::bar_drain(empty + ((i - NS) & 1), ((i - NS) >> 1) & 1);
        } else if (warp == 4) {
            // ---- S = K Q' ------------------------------------------------------------------------
            // (apart from O = V' P: with one warp for both, a tile's O would wait for the next tile's keys)
            constexpr uint32_t kind = BF ? tc::idesc_bf16_f32(128, NT) : tc::idesc_f16_f32(128, NT);
            const uint32_t base = tc::sa(smem);
            int u = 0;
            for (int i = 0; i < n_tiles; ++i) {
                const int st = i % NS;
                bool ok = tc::bar_wait(kfull + st, (i / NS) & 1, abort, status, WAIT);
                if (ok && i >= 2) ok = tc::bar_wait(pfull + (i & 1), ((i >> 1) - 1) & 1, abort, status, WAIT);  // tile i - 2's S has been read
                const int flags = meta[i & 1].flags;
                if (ok && (flags & FIRST)) ok = tc::bar_wait(qfull + (u & 1), (u >> 1) & 1, abort, status, WAIT);
                if (!__all_sync(0xffffffffu, ok)) break;
                __syncwarp();
                tc::fence_after_sync();
                if (lane == 0) {
#pragma unroll
                    for (int kk = 0; kk < DP / 16; ++kk)
                        if (16 * kk < D)
                            tc::mma_bf16(tmem + (i & 1) * 32, tc::desc_k_sw128(base + st * S::STAGE + (kk >> 2) * KEYS * 128 + (kk & 3) * 32),
                                     tc::desc_k_sw128(base + S::at_q + (u & 1) * S::Q + (kk >> 2) * NT * 128 + (kk & 3) * 32), kind, kk > 0);
                    tc::mma_commit(sfull + (i & 1));
                    if (flags & LAST) tc::mma_commit(qempty + (u & 1));
                }
                if (flags & LAST) ++u;
                __syncwarp();
            }
            // nothing issued is under way when tensor memory is given back
            if (lane == 0) tc::mma_commit(done);
            tc::bar_drain(done, 0);
        } else if (warp == 11) {
            // ---- O = V' P ------------------------------------------------------------------------
            constexpr uint32_t kind = (BF ? tc::idesc_bf16_f32(128, NT) : tc::idesc_f16_f32(128, NT)) | 1u << 15 | 1u << 16;
            const uint32_t base = tc::sa(smem);
            for (int i = 0; i < n_tiles; ++i) {
                const int st = i % NS, at = i & 1;
                bool ok = tc::bar_wait(vfull + st, (i / NS) & 1, abort, status, WAIT);
                if (ok) ok = tc::bar_wait(pfull + at, (i >> 1) & 1, abort, status, WAIT);
                if (!__all_sync(0xffffffffu, ok)) break;
                tc::fence_after_sync();
                if (lane == 0) {
                    const uint32_t v = base + st * S::STAGE + S::MAT, p = base + S::at_p + at * S::P;
#pragma unroll
                    for (int h = 0; h < MH; ++h)  // 128 channels each
#pragma unroll
                        for (int kk = 0; kk < KEYS / 16; ++kk)
                            tc::mma_bf16(tmem + 64 + (h * 2 + at) * 32, desc_v(v + h * 2 * KEYS * 128 + kk * 2048, DP >= 128 ? KEYS * 128 : 0),
                                         desc_p(p + kk * 1024), kind, kk > 0);
                    tc::mma_commit(ofull + at);
                    tc::mma_commit(empty + at);
                }
                __syncwarp();
            }
            if (lane == 0) tc::mma_commit(done);
            tc::bar_drain(done, 0);
        } else if (warp >= 9) {
            // ---- the next units' queries ---------------------------------------------------------
            const int t = threadIdx.x - 288;
            int s = s0, vh = vh0, u = 0;
            bool ok = true;
            for (int us = unit_start(s, vh); ok && us < g1; ++u) {
                const int tiles = pre[s + 1] - pre[s];
                if (u >= 2) ok = tc::bar_wait(qempty + (u & 1), ((u >> 1) - 1) & 1, abort, status, WAIT);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const int kvh = vh / a.subs, sub = vh - kvh * a.subs;
                const int h0 = kvh * a.group + sub * GP, heads = min(GP, a.group - sub * GP);
                const float *q = a.q + (size_t)s * a.q_stride + (size_t)h0 * D;
                uint8_t *qs = smem + S::at_q + (u & 1) * S::Q;
                for (int c = t; c < GP * CH; c += 64) {  // eight channels of a head a thread
                    const int h = c / CH, ch = c % CH;
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = h < heads && ch * 8 < D ? q[(size_t)h * D + ch * 8 + e] : 0.f;
                    float f = 1.f;
                    if constexpr (!BF) {  // the head's largest magnitude to [2^12, 2^13)
                        float mx = 0.f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
#pragma unroll
                        for (int o = 1; o < CH; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        if (mx > 0.f) f = exp2f((float)min(100, 12 - ilogbf(mx)));
                    }
                    uint32_t w[3][4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) terms<BF>(x[2 * e] * f, x[2 * e + 1] * f, w[0][e], w[1][e], w[2][e]);
#pragma unroll
                    for (int r = 0; r < TERMS; ++r)
                        *reinterpret_cast<uint4 *>(qs + (ch >> 3) * NT * 128 + (r * 8 + h) * 128 + (((ch & 7) ^ h) << 4)) =
                            make_uint4(w[r][0], w[r][1], w[r][2], w[r][3]);
                    if (ch == 0) {
                        scales[(u & 7) * 2 * GP + h] = a.scale2 / f;
                        scales[((u & 7) * 2 + 1) * GP + h] = a.sinks && h < heads ? a.sinks[h0 + h] * LOG2E : -INFINITY;
                    }
                }
                fence_async();
                tc::bar_arrive(qfull + (u & 1));
                tc::bar_arrive(qready + (u & 3));
                us += tiles;
                next_unit(s, vh);
            }
            for (int w = max(0, u - 2); w < u; ++w)
                if (*abort == 0) tc::bar_drain(qempty + (w & 1), (w >> 1) & 1);
        } else {
            // ---- softmax: thread = key of S, then channel of O ----------------------------------
            const int t = threadIdx.x;
            float O[MH][GP], l[GP], m[GP], sc[GP];
            int u = 0;
            bool ok = true;
            auto *red = reinterpret_cast<float *>(smem + S::at_red);
            auto *mxs = reinterpret_cast<float *>(smem + S::at_max);
            const uint32_t lanes = (uint32_t)(warp * 32) << 16;
            auto flush = [&](int i) {  // O takes tile i's sums
                if (!__all_sync(0xffffffffu, tc::bar_wait(ofull + (i & 1), (i >> 1) & 1, abort, status, WAIT))) return false;
                tc::fence_after_sync();
#pragma unroll
                for (int b = 0; b < MH; ++b) {
                    float c[32];
                    tmem_ld32(tmem + 64 + (b * 2 + (i & 1)) * 32 + lanes, c);
#pragma unroll
                    for (int h = 0; h < GP; ++h)
                        O[b][h] += BF ? c[h] + (c[8 + h] + c[16 + h]) : fmaf(fmaf(c[16 + h], FINE, c[8 + h]), FINE, c[h]);
                }
                return true;
            };
            bool pending = false;
            for (int i = 0; i < n_tiles; ++i) {
                const int st = i & 1;
                ok = ok && tc::bar_wait(kfull + i % NS, (i / NS) & 1, abort, status, WAIT) && tc::bar_wait(sfull + st, (i >> 1) & 1, abort, status, WAIT);
                const int flags = meta[st].flags;
                if (ok && (flags & FIRST)) ok = tc::bar_wait(qready + (u & 3), (u >> 2) & 1, abort, status, WAIT);
                if (soft_any(!ok)) break;  // the four warps leave together: they meet at barriers
                if (flags & FIRST) {
#pragma unroll
                    for (int h = 0; h < GP; ++h) {
                        for (int b = 0; b < MH; ++b) O[b][h] = 0.f;
                        l[h] = 0.f;
                        m[h] = -INFINITY;
                        sc[h] = scales[(u & 7) * 2 * GP + h];
                    }
                    pending = false;
                }
                // the note is the loads' again once this tile's weights are handed over
                const bool live = meta[st].live[warp] >> lane & 1;
                const int row = meta[st].row, vh = meta[st].vh;
                tc::fence_after_sync();
                float s[GP];
                {
                    float c[32];
                    tmem_ld32(tmem + st * 32 + lanes, c);
#pragma unroll
                    for (int h = 0; h < GP; ++h) s[h] = live ? (c[h] + (c[8 + h] + c[16 + h])) * sc[h] : -INFINITY;
                }
                bool up = false;
#pragma unroll
                for (int h = 0; h < GP; ++h) up |= s[h] - m[h] > LAZY;
                if (soft_any(up)) {
                    if (pending) {
                        ok = flush(i - 1) && ok;
                        pending = false;
                    }
                    const float top = reduce8(s, lane, [](float x, float y) { return fmaxf(x, y); });
                    if ((lane & 3) == 0) mxs[(st * 4 + warp) * GP + (lane >> 2)] = top;
                    soft_sync();
#pragma unroll
                    for (int h = 0; h < GP; ++h) {
                        const float *x = mxs + st * 4 * GP + h;
                        const float mn = fmaxf(fmaxf(fmaxf(m[h], x[0]), fmaxf(x[GP], x[2 * GP])), x[3 * GP]);
                        const float corr = ex2(m[h] - (mn == -INFINITY ? 0.f : mn));
                        l[h] *= corr;
                        for (int b = 0; b < MH; ++b) O[b][h] *= corr;
                        m[h] = mn;
                    }
                }
#pragma unroll
                for (int h = 0; h < GP; ++h) {
                    const float p = ex2(s[h] - (m[h] == -INFINITY ? 0.f : m[h]));
                    l[h] += p;
                    s[h] = p * (PSCALE * DOWN);
                }
                uint8_t *prow = smem + S::at_p + st * S::P + t * 64;
#pragma unroll
                for (int r = 0; r < TERMS; ++r) {  // a term of every head, then what it leaves
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        w[e] = pack<BF>(s[2 * e], s[2 * e + 1]);
                        const float2 a = unpack<BF>(w[e]);
                        s[2 * e] = rest<BF>(s[2 * e], a.x);
                        s[2 * e + 1] = rest<BF>(s[2 * e + 1], a.y);
                    }
                    *reinterpret_cast<uint4 *>(prow + ((r ^ (t >> 1 & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                fence_async();
                tc::fence_before_sync();
                tc::bar_arrive(pfull + st);
                if (pending) ok = ok && flush(i - 1);
                pending = true;
                if (flags & LAST) {
                    const float part_l = reduce8(l, lane, [](float x, float y) { return x + y; });
                    if ((lane & 3) == 0) red[((u & 1) * 4 + warp) * GP + (lane >> 2)] = part_l;
                    ok = ok && flush(i);
                    soft_sync();
                    const int kvh = vh / a.subs, sub = vh - kvh * a.subs;
                    const int h0 = kvh * a.group + sub * GP, heads = min(GP, a.group - sub * GP);
                    const float *x = red + (u & 1) * 4 * GP;
#pragma unroll
                    for (int h = 0; h < GP; ++h) {
                        l[h] = ((x[h] + x[GP + h]) + (x[2 * GP + h] + x[3 * GP + h])) * DOWN;
                        for (int b = 0; b < MH; ++b) O[b][h] *= 1.f / PSCALE;
                    }
                    if (flags & WHOLE) {
                        float *out = a.out + ((size_t)row * a.n_heads + h0) * D;
#pragma unroll
                        for (int h = 0; h < GP; ++h) {
                            if (h >= heads) break;
                            float sum = l[h], f = 1.f;
                            const float sk = scales[((u & 7) * 2 + 1) * GP + h];
                            if (sk != -INFINITY) {
                                const float top = fmaxf(m[h], sk);
                                f = m[h] == -INFINITY ? 0.f : ex2(m[h] - top);
                                sum = sum * f + ex2(sk - top) * DOWN;
                            }
                            f = sum == 0.f ? 0.f : f / sum;
#pragma unroll
                            for (int b = 0; b < MH; ++b)
                                if (b * 128 + t < D) out[h * D + b * 128 + t] = O[b][h] * f;
                        }
                    } else {
                        float *part = a.part + ((size_t)blockIdx.x * 2 + (flags & SECOND ? 1 : 0)) * GP * (D + 2);
#pragma unroll
                        for (int h = 0; h < GP; ++h) {
#pragma unroll
                            for (int b = 0; b < MH; ++b)
                                if (b * 128 + t < D) part[h * D + b * 128 + t] = O[b][h];
                            if (t == h) {
                                part[GP * D + 2 * h] = m[h];
                                part[GP * D + 2 * h + 1] = l[h];
                            }
                        }
                    }
                    ++u;
                }
            }
        }
    } else if (threadIdx.x == 0) {
        a.notes[blockIdx.x] = make_int4(0, 0, 0, 0);
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    if (warp == 4) tc::tmem_dealloc(tmem, S::TMEM);
}

template <int DP, bool FULL, bool BF>
cudaError_t launch_tile(moearc_ctx *c, int grid, const attn_args &a) {
    static std::atomic<bool> done[MOEARC_MAX_DEVICES];
    cudaError_t e = once_per_device(done, [] { return set_smem(k_attn_tc<DP, FULL, BF>, tc_smem<DP>::total((int)KV_LIST)); });
    if (e == cudaSuccess)
        e = launch_pdl(k_attn_tc<DP, FULL, BF>, dim3((unsigned)grid), dim3(THREADS), (size_t)tc_smem<DP>::total((int)a.n_seq), c->stream, a);
    return e != cudaSuccess ? e : attn_join_launch<GP>(c, grid, a);
}
template <bool BF>
cudaError_t launch(moearc_ctx *c, int grid, const attn_args &a) {
    if (a.D <= 64) return a.D == 64 ? launch_tile<64, true, BF>(c, grid, a) : launch_tile<64, false, BF>(c, grid, a);
    if (a.D <= 128) return a.D == 128 ? launch_tile<128, true, BF>(c, grid, a) : launch_tile<128, false, BF>(c, grid, a);
    return a.D == 256 ? launch_tile<256, true, BF>(c, grid, a) : launch_tile<256, false, BF>(c, grid, a);
}

}  // namespace

namespace moearc {

void attn_tc_plan(attn_plan &p, int n_heads, int n_kv, int D, int sms) {
    p.gp = GP;
    p.keys = KEYS;
    p.subs = (n_heads / n_kv + GP - 1) / GP;
    p.hg = p.rsplit = 1;
    p.nhg = n_kv * p.subs;
    p.grid = D <= 64 ? 2 * sms : sms;
}

cudaError_t attn_tc_launch(moearc_ctx *c, const attn_plan &p, unsigned kv_type, const attn_args &a) {
    return kv_type == T_BF16 ? launch<true>(c, p.grid, a) : launch<false>(c, p.grid, a);
}

}  // namespace moearc
