// kvcache.cu — the pages of a paged KV cache shared by many sequences: growing, forking, cutting
// and compacting rows, with tables, lengths and reference counts on the device.
//
// A page is free when no row holds it (refs 0), and new pages are the free ones of lowest id in
// list order, so every result is a function of the state alone. Each call is two launches: a plan
// kernel of one CTA decides everything (rows in a prefix sum, free pages in an ascending sweep of
// refs) and writes the list of page moves into `work`; a copy kernel over all SMs then moves the
// pages in every pool. Freeing moves nothing and is one launch.
//
// A page move reads and writes page_bytes per pool: the copy kernel is bound by HBM (3.08 GB read and
// written for deep forks in 36 layers: 497 us, 6.2 TB/s; a compaction's 2.0 GB: 326 us). The plan is
// bound by the latency of its few dependent loads (10 us for a compaction of 6001 pages).
#include "kvcache.cuh"

using namespace moearc;

namespace {

constexpr int PLAN_THREADS = 1024;
static_assert(PLAN_THREADS == KV_LIST, "one plan thread a list entry");
constexpr int SWEEP = 16;  // refs a plan thread reads at once: four 16-byte loads in flight

// Lists go into a launch by value; short ones in a shorter argument (a launch with 10 KB of them
// held up the next one by 10 us; 256 rows cut back and grown again: 15.6 us with 2 KB, 17.4 with 8).
constexpr int SHORT_LIST = 64, MID_LIST = 256, SHORT_POOLS = 16;
template <int N>
struct row_list {
    unsigned a[N], b[N];  // grow: row, add; fork: src, dst; free: row, keep
    unsigned n;
};
template <int N>
struct pool_list {
    void *p[N];
    unsigned n;
};
struct cache_view {
    unsigned *tables, *n_kv, *refs, *status;
    unsigned n_pages, pt, max_pages, max_seq;
};

// The work buffer: a header, each list entry's first new page, the new pages, the moves and (for
// compaction) where every page goes.
struct plan_head {
    unsigned ok, n_moves, n_live, n;
    unsigned off[KV_LIST], src[KV_LIST], dst[KV_LIST];  // a fork's list for the kernel after the plan
};
struct work_view {
    plan_head *head;
    unsigned *ids;   // [n_pages] new pages in list order; compaction: the new id of every page
    uint2 *moves;    // [n_pages] (from, to)
};
__host__ __device__ inline size_t pages16(unsigned n_pages) { return ((size_t)n_pages + 15) & ~size_t(15); }
inline size_t kv_plan_bytes(unsigned n_pages) { return ((sizeof(plan_head) + 15) & ~size_t(15)) + pages16(n_pages) * 12; }
inline work_view work_of(void *work, unsigned n_pages) {
    auto *b = static_cast<uint8_t *>(work);
    work_view w;
    w.head = reinterpret_cast<plan_head *>(b);
    w.moves = reinterpret_cast<uint2 *>(b + ((sizeof(plan_head) + 15) & ~size_t(15)));
    w.ids = reinterpret_cast<unsigned *>(w.moves + pages16(n_pages));
    return w;
}

// SWEEP refs from page p on as a mask of which are 0 (pages at or past n_pages count as held).
__device__ __forceinline__ unsigned free_mask(const unsigned *refs, unsigned p, unsigned n_pages, bool vec) {
    unsigned m = 0;
    if (vec && p + SWEEP <= n_pages) {
        const uint4 *r = reinterpret_cast<const uint4 *>(refs + p);
        uint4 v[SWEEP / 4];
#pragma unroll
        for (int i = 0; i < SWEEP / 4; ++i) v[i] = r[i];
#pragma unroll
        for (int i = 0; i < SWEEP / 4; ++i)
            m |= (unsigned)((v[i].x == 0) | (v[i].y == 0) << 1 | (v[i].z == 0) << 2 | (v[i].w == 0) << 3) << (4 * i);
    } else {
        for (int i = 0; i < SWEEP; ++i)
            if (p + i < n_pages && refs[p + i] == 0) m |= 1u << i;
    }
    return m;
}

// The first `want` free pages in ascending order into ids; false when there are fewer.
__device__ bool find_free(const cache_view &k, unsigned *ids, unsigned want, unsigned *warp_sums) {
    const bool vec = (reinterpret_cast<uintptr_t>(k.refs) & 15) == 0;
    unsigned have = 0;
    for (unsigned base = 0; base < k.n_pages && have < want; base += PLAN_THREADS * SWEEP) {
        const unsigned p = base + threadIdx.x * SWEEP;
        unsigned m = p < k.n_pages ? free_mask(k.refs, p, k.n_pages, vec) : 0, total;
        unsigned at = have + block_scan((unsigned)__popc(m), warp_sums, &total) - __popc(m);
        for (; m && at < want; m &= m - 1, ++at) ids[at] = p + __ffs(m) - 1;
        have += total;
    }
    return have >= want;
}

// The list entry that new page m belongs to: the last i with off[i] <= m (entries without pages
// share the next one's offset and are passed over).
__device__ __forceinline__ unsigned entry_of(const unsigned *off, unsigned n, unsigned m) {
    unsigned lo = 0, hi = n;
    while (hi - lo > 1) {
        const unsigned mid = (lo + hi) >> 1;
        if (off[mid] <= m) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Plan of a grow (FORK false) or fork (true): the pages each entry needs, the free pages handed
// out, the moves; a grow's tables, counts and lengths too. All or nothing.
template <bool FORK, int N>
__global__ void __launch_bounds__(PLAN_THREADS) k_kv_plan(const __grid_constant__ row_list<N> L, cache_view k, work_view w, int deep) {
    __shared__ unsigned long long sums64[32];
    __shared__ unsigned sums[32], off[KV_LIST + 1], bad, n_moves;
    const unsigned i = threadIdx.x;
    if (i == 0) bad = n_moves = 0;
    pdl_trigger();
    pdl_wait();
    __syncthreads();
    unsigned cur = 0, add = 0, need = 0, flag = 0, row = 0;
    bool cow = false;
    if (i < L.n) {
        row = L.a[i];
        cur = k.n_kv[row];
        const unsigned tail = cur / k.pt;
        if ((unsigned long long)cur > (unsigned long long)k.max_pages * k.pt) flag = MOEARC_X_KV_LONG;  // not a length of ours
        else if (FORK) {
            if (k.n_kv[L.b[i]] != 0) flag = MOEARC_X_KV_TAKEN;
            if (deep) need = (cur + k.pt - 1) / k.pt;
            else if (cur % k.pt) need = k.tables[(size_t)row * k.max_pages + tail] < k.n_pages;
        } else {
            add = L.b[i];
            const unsigned long long want = (unsigned long long)cur + add;
            if (want > (unsigned long long)k.max_pages * k.pt) flag = MOEARC_X_KV_LONG;
            else if (add) {
                if (cur % k.pt) {
                    const unsigned p = k.tables[(size_t)row * k.max_pages + tail];
                    cow = p < k.n_pages && k.refs[p] > 1;
                }
                need = cow + (unsigned)((want + k.pt - 1) / k.pt) - (cur + k.pt - 1) / k.pt;
            }
        }
    }
    if (flag) atomicOr(&bad, flag);
    unsigned long long total;
    const unsigned long long end = block_scan((unsigned long long)need, sums64, &total);
    const unsigned flags = bad;  // every flag is in before the scan's barriers
    bool ok = flags == 0 && total <= k.n_pages;
    if (ok && total) {
        off[i] = (unsigned)(end - need);
        if (i == 0) off[KV_LIST] = (unsigned)total;
        ok = find_free(k, w.ids, (unsigned)total, sums);
    }
    __syncthreads();
    if (ok && total) {
        for (unsigned m = i; m < (unsigned)total; m += PLAN_THREADS) {
            const unsigned e = entry_of(off, L.n, m), r = m - off[e], id = w.ids[m];
            const unsigned s = L.a[e], len = k.n_kv[s];
            unsigned *t = k.tables + (size_t)s * k.max_pages;
            if (FORK) {
                const unsigned p = t[deep ? r : len / k.pt];
                if (p < k.n_pages) {
                    k.refs[id] = 1;
                    w.moves[atomicAdd(&n_moves, 1u)] = make_uint2(p, id);
                }
            } else {
                const unsigned first = (len + k.pt - 1) / k.pt;
                const unsigned news = (unsigned)(((unsigned long long)len + L.b[e] + k.pt - 1) / k.pt) - first;
                const unsigned copies = off[e + 1 < L.n ? e + 1 : KV_LIST] - off[e] - news;  // 1: the shared last page
                k.refs[id] = 1;
                if (r < copies) {
                    const unsigned p = t[first - 1];
                    atomicSub(k.refs + p, 1u);
                    w.moves[atomicAdd(&n_moves, 1u)] = make_uint2(p, id);
                    t[first - 1] = id;
                } else {
                    t[first + r - copies] = id;
                }
            }
        }
        __syncthreads();
    }
    if (!FORK && ok && i < L.n) k.n_kv[row] = cur + add;
    if (FORK && ok && i < L.n) {
        w.head->off[i] = total ? off[i] : 0;
        w.head->src[i] = row;
        w.head->dst[i] = L.b[i];
    }
    if (i == 0) {
        w.head->ok = ok;
        w.head->n = L.n;
        w.head->n_moves = ok ? n_moves : 0;
        if (!ok) atomicOr(k.status, flags ? flags : MOEARC_X_KV_FULL);
    }
}

// Copy the planned pages in every pool: 256-thread CTAs over chunks of CHUNK elements of V.
constexpr int COPY_THREADS = 256, COPY_UNROLL = 4, COPY_CHUNK = COPY_THREADS * COPY_UNROLL;

template <typename V, int NP>
__device__ void copy_pages(const uint2 *moves, unsigned n_moves, const pool_list<NP> &P, unsigned page_v) {
    const unsigned cpp = (page_v + COPY_CHUNK - 1) / COPY_CHUNK;  // chunks a page
    const unsigned long long items = (unsigned long long)n_moves * P.n * cpp;
    for (unsigned long long it = blockIdx.x; it < items; it += gridDim.x) {
        const unsigned long long mp = it / cpp;
        const unsigned c0 = (unsigned)(it - mp * cpp) * COPY_CHUNK + threadIdx.x;
        const unsigned m = (unsigned)(mp / P.n), pool = (unsigned)(mp - (unsigned long long)m * P.n);
        const uint2 mv = moves[m];
        const V *src = static_cast<const V *>(P.p[pool]) + (size_t)mv.x * page_v;
        V *dst = static_cast<V *>(P.p[pool]) + (size_t)mv.y * page_v;
        V v[COPY_UNROLL];
#pragma unroll
        for (int u = 0; u < COPY_UNROLL; ++u)
            if (c0 + u * COPY_THREADS < page_v) v[u] = src[c0 + u * COPY_THREADS];
#pragma unroll
        for (int u = 0; u < COPY_UNROLL; ++u)
            if (c0 + u * COPY_THREADS < page_v) dst[c0 + u * COPY_THREADS] = v[u];
    }
}

template <typename V, int NP>
__global__ void __launch_bounds__(COPY_THREADS) k_kv_copy(const __grid_constant__ pool_list<NP> P, work_view w, unsigned page_v) {
    pdl_trigger();
    pdl_wait();
    copy_pages<V>(w.moves, w.head->n_moves, P, page_v);
}

// A fork's rows: dst's table from src's, its own pages in place, one more reference on each
// shared page; then the copies. CTAs stride over the list.
template <typename V, int NP>
__global__ void __launch_bounds__(COPY_THREADS) k_kv_fork(const __grid_constant__ pool_list<NP> P, cache_view k, work_view w,
                                                          unsigned page_v, int deep) {
    pdl_trigger();
    pdl_wait();
    if (!w.head->ok) return;
    for (unsigned e = blockIdx.x; e < w.head->n; e += gridDim.x) {
        const unsigned len = k.n_kv[w.head->src[e]], np = (len + k.pt - 1) / k.pt;
        const unsigned first = deep ? 0 : len / k.pt;  // pages from here on are the row's own
        const unsigned *src = k.tables + (size_t)w.head->src[e] * k.max_pages;
        unsigned *dst = k.tables + (size_t)w.head->dst[e] * k.max_pages;
        for (unsigned j = threadIdx.x; j < np; j += COPY_THREADS) {
            unsigned p = src[j];
            if (p < k.n_pages) {
                if (j >= first) p = w.ids[w.head->off[e] + j - first];
                else atomicAdd(k.refs + p, 1u);
            }
            dst[j] = p;
        }
        if (threadIdx.x == 0) k.n_kv[w.head->dst[e]] = len;
    }
    copy_pages<V>(w.moves, w.head->n_moves, P, page_v);
}

template <int N>
__global__ void __launch_bounds__(256) k_kv_free(const __grid_constant__ row_list<N> L, cache_view k) {
    pdl_trigger();
    pdl_wait();
    const unsigned s = L.a[blockIdx.x], cur = k.n_kv[s], keep = min(cur, L.b[blockIdx.x]);
    unsigned *t = k.tables + (size_t)s * k.max_pages;
    const unsigned j1 = min((unsigned)(((unsigned long long)cur + k.pt - 1) / k.pt), k.max_pages);
    for (unsigned j = (unsigned)(((unsigned long long)keep + k.pt - 1) / k.pt) + threadIdx.x; j < j1; j += 256) {
        const unsigned p = t[j];
        if (p < k.n_pages) atomicSub(k.refs + p, 1u);
        t[j] = NO_PAGE;
    }
    __syncthreads();
    if (threadIdx.x == 0) k.n_kv[s] = keep;
}

// Plan of a compaction: n_live, then free pages below it and live pages from it on, both ascending
// and equally many, paired into moves; ids[p] for p >= n_live is where page p goes.
__global__ void __launch_bounds__(PLAN_THREADS) k_kv_compact_plan(cache_view k, work_view w) {
    __shared__ unsigned sums[32];
    pdl_trigger();
    pdl_wait();
    const bool vec = (reinterpret_cast<uintptr_t>(k.refs) & 15) == 0;
    unsigned live = 0, total;
    for (unsigned p = threadIdx.x * SWEEP; p < k.n_pages; p += PLAN_THREADS * SWEEP) {
        const unsigned in = min((unsigned)SWEEP, k.n_pages - p);
        live += in - __popc(free_mask(k.refs, p, k.n_pages, vec));
    }
    block_scan(live, sums, &total);
    const unsigned n_live = total;
    unsigned holes = 0, tails = 0;
    for (unsigned base = 0; base < k.n_pages; base += PLAN_THREADS * SWEEP) {
        const unsigned p = base + threadIdx.x * SWEEP;
        const unsigned in = p < k.n_pages ? min((unsigned)SWEEP, k.n_pages - p) : 0;
        const unsigned fr = in ? free_mask(k.refs, p, k.n_pages, vec) : 0;
        const unsigned all = (1u << in) - 1;
        const unsigned below = p >= n_live ? 0 : n_live - p >= SWEEP ? all : all & ((1u << (n_live - p)) - 1);
        unsigned h = fr & below, t = ~fr & all & ~below;
        // holes and tails scanned together, 16 bits each: a chunk holds 16384 pages at most
        const unsigned mine = __popc(h) | (unsigned)__popc(t) << 16;
        const unsigned upto = block_scan(mine, sums, &total) - mine;
        unsigned ho = holes + (upto & 0xffff), to = tails + (upto >> 16);
        for (; h; h &= h - 1) w.moves[ho++].y = p + __ffs(h) - 1;
        for (unsigned q = 0; q < in; ++q)
            if (!(below >> q & 1) && !(t >> q & 1)) w.ids[p + q] = NO_PAGE;
        for (; t; t &= t - 1) w.moves[to++].x = p + __ffs(t) - 1;
        holes += total & 0xffff;
        tails += total >> 16;
    }
    __syncthreads();
    for (unsigned m = threadIdx.x; m < tails; m += PLAN_THREADS) {
        const uint2 mv = w.moves[m];
        w.ids[mv.x] = mv.y;
    }
    if (threadIdx.x == 0) {
        w.head->ok = 1;
        w.head->n_moves = tails;
        w.head->n_live = n_live;
    }
}

// A compaction's copies, tables and counts. In place as well: a hole's count is written with its
// page's, and every other element is written with what it holds or holds already.
template <typename V, int NP>
__global__ void __launch_bounds__(COPY_THREADS) k_kv_compact(const __grid_constant__ pool_list<NP> P, cache_view k, work_view w,
                                                             unsigned page_v, unsigned *tables_out, unsigned *refs_out,
                                                             unsigned *n_live_out) {
    pdl_trigger();
    pdl_wait();
    const unsigned n_live = w.head->n_live, n_moves = w.head->n_moves;
    const size_t me = (size_t)blockIdx.x * COPY_THREADS + threadIdx.x, all = (size_t)gridDim.x * COPY_THREADS;
    if (me == 0 && n_live_out) *n_live_out = n_live;
    for (size_t t = me; t < (size_t)k.max_seq * k.max_pages; t += all) {
        const unsigned p = k.tables[t];
        const unsigned q = p < n_live ? p : p < k.n_pages ? w.ids[p] : p;
        if (tables_out != k.tables || q != p) tables_out[t] = q;
    }
    for (size_t p = me; p < k.n_pages; p += all)
        if (refs_out != k.refs) {
            const unsigned r = k.refs[p];
            if (p < n_live ? r != 0 : r == 0) refs_out[p] = r;
        }
    for (size_t m = me; m < n_moves; m += all) {
        const uint2 mv = w.moves[m];
        refs_out[mv.y] = k.refs[mv.x];
        refs_out[mv.x] = 0;
    }
    copy_pages<V>(w.moves, n_moves, P, page_v);
}

cache_view view_of(const moearc_x_kv_cache &k) {
    return cache_view{k.tables, k.n_kv, k.refs, k.status, k.n_pages, k.page_tokens, k.max_pages, k.max_seq};
}

// The widest element (16, 4 or 2 bytes) that every page of every pool starts on and is a whole number of.
unsigned copy_width(const moearc_x_kv_cache &k, size_t &page_bytes) {
    page_bytes = (size_t)k.page_tokens * k.n_kv_heads * k.head_dim * kv_elem_bytes(k.kv_type);
    uintptr_t a = page_bytes;
    for (unsigned l = 0; l < k.n_layer; ++l) a |= reinterpret_cast<uintptr_t>(k.k_pages[l]) | reinterpret_cast<uintptr_t>(k.v_pages[l]);
    return (a & 15) == 0 ? 16 : (a & 3) == 0 ? 4 : 2;
}

// f(V, pools, elements a page): the copy's element type and the pools in an argument of their size.
template <typename F>
cudaError_t with_pools(const moearc_x_kv_cache &k, F &&f) {
    size_t page_bytes;
    const unsigned width = copy_width(k, page_bytes), page_v = (unsigned)(page_bytes / width);
    auto by_width = [&](auto &P) {
        P.n = 2 * k.n_layer;
        for (unsigned l = 0; l < k.n_layer; ++l) {
            P.p[2 * l] = k.k_pages[l];
            P.p[2 * l + 1] = k.v_pages[l];
        }
        return width == 16 ? f(uint4(), P, page_v) : width == 4 ? f(uint32_t(), P, page_v) : f(uint16_t(), P, page_v);
    };
    if (2 * k.n_layer <= SHORT_POOLS) {
        pool_list<SHORT_POOLS> P;
        return by_width(P);
    }
    pool_list<2 * KV_LAYERS> P;
    return by_width(P);
}
// f(list): the rows in an argument of their size.
template <typename F>
cudaError_t with_rows(const unsigned *a, const unsigned *b, unsigned n, F &&f) {
    auto fill = [&](auto &L) {
        L.n = n;
        for (unsigned i = 0; i < n; ++i) {
            L.a[i] = a[i];
            L.b[i] = b ? b[i] : 0;
        }
        return f(L);
    };
    if (n <= SHORT_LIST) {
        row_list<SHORT_LIST> L;
        return fill(L);
    }
    if (n <= MID_LIST) {
        row_list<MID_LIST> L;
        return fill(L);
    }
    row_list<KV_LIST> L;
    return fill(L);
}

// Eight CTAs an SM: 3 GB of pages in 503 us, against 562 with two.
dim3 copy_grid(const moearc_ctx *c) { return dim3((unsigned)c->sm_count * 8); }

int finish(moearc_ctx *c, cudaError_t e) {
    if (e != cudaSuccess) {
        cudaGetLastError();  // the failed launch's error, not left for an unrelated later check
        return ERR;
    }
    return c->sync_each && cudaStreamSynchronize(c->stream) != cudaSuccess ? ERR : OK;
}

// kv_check and the work buffer's size.
int page_call_check(moearc_ctx *c, const moearc_x_kv_cache *kv) {
    const int rc = kv_check(c, kv);
    if (rc) return rc;
    return kv->work_bytes < kv_plan_bytes(kv->n_pages) ? ERR_ARG : OK;
}

}  // namespace

namespace moearc {
size_t kv_page_work_bytes(unsigned n_pages) { return kv_plan_bytes(n_pages); }
}  // namespace moearc

extern "C" {

int moearc_x_kv_reset(moearc_ctx *c, const moearc_x_kv_cache *kv) {
    const int rc = kv_check(c, kv);
    if (rc) return rc;
    device_guard g(c->device);
    if (!g.ok) return ERR;
    cudaError_t e = cudaMemsetAsync(kv->tables, 0xFF, (size_t)kv->max_seq * kv->max_pages * 4, c->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(kv->n_kv, 0, (size_t)kv->max_seq * 4, c->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(kv->refs, 0, (size_t)kv->n_pages * 4, c->stream);
    if (e == cudaSuccess) e = cudaMemsetAsync(kv->status, 0, 4, c->stream);
    return finish(c, e);
}

int moearc_x_kv_grow(moearc_ctx *c, const moearc_x_kv_cache *kv, const unsigned int *seqs, const unsigned int *add, unsigned int n) {
    const int rc = page_call_check(c, kv);
    if (rc) return rc;
    if (n == 0) return OK;
    if (!seqs || !add) return ERR;
    if (n > KV_LIST) return ERR_ARG;
    kv_rows_seen seen(kv->max_seq);
    for (unsigned i = 0; i < n; ++i)
        if (!seen.add(seqs[i], kv->max_seq)) return ERR_ARG;
    device_guard g(c->device);
    if (!g.ok) return ERR;
    const work_view w = work_of(kv->work, kv->n_pages);
    launch_scope ls(c, "kv_grow", n, kv->n_layer);
    cudaError_t e = with_rows(seqs, add, n, [&](auto &L) {
        constexpr int N = (int)(sizeof(L.a) / sizeof(unsigned));
        return launch_pdl(k_kv_plan<false, N>, dim3(1), dim3(PLAN_THREADS), 0, c->stream, L, view_of(*kv), w, 0);
    });
    if (e == cudaSuccess)
        e = with_pools(*kv, [&](auto v, auto &P, unsigned page_v) {
            constexpr int NP = (int)(sizeof(P.p) / sizeof(void *));
            return launch_pdl(k_kv_copy<decltype(v), NP>, copy_grid(c), dim3(COPY_THREADS), 0, c->stream, P, w, page_v);
        });
    const int rc2 = ls.finish();
    return e != cudaSuccess ? finish(c, e) : rc2;
}

int moearc_x_kv_fork(moearc_ctx *c, const moearc_x_kv_cache *kv, const unsigned int *src, const unsigned int *dst, unsigned int n,
                     int deep) {
    const int rc = page_call_check(c, kv);
    if (rc) return rc;
    if (n == 0) return OK;
    if (!src || !dst) return ERR;
    if (n > KV_LIST) return ERR_ARG;
    kv_rows_seen seen(kv->max_seq);
    for (unsigned i = 0; i < n; ++i)
        if (!seen.add(dst[i], kv->max_seq)) return ERR_ARG;
    for (unsigned i = 0; i < n; ++i)
        if (src[i] >= kv->max_seq || seen.has(src[i])) return ERR_ARG;
    device_guard g(c->device);
    if (!g.ok) return ERR;
    const work_view w = work_of(kv->work, kv->n_pages);
    const cache_view k = view_of(*kv);
    launch_scope ls(c, "kv_fork", n, kv->n_layer);
    cudaError_t e = with_rows(src, dst, n, [&](auto &L) {
        constexpr int N = (int)(sizeof(L.a) / sizeof(unsigned));
        return launch_pdl(k_kv_plan<true, N>, dim3(1), dim3(PLAN_THREADS), 0, c->stream, L, k, w, deep);
    });
    if (e == cudaSuccess)
        e = with_pools(*kv, [&](auto v, auto &P, unsigned page_v) {
            constexpr int NP = (int)(sizeof(P.p) / sizeof(void *));
            return launch_pdl(k_kv_fork<decltype(v), NP>, copy_grid(c), dim3(COPY_THREADS), 0, c->stream, P, k, w, page_v, deep);
        });
    const int rc2 = ls.finish();
    return e != cudaSuccess ? finish(c, e) : rc2;
}

int moearc_x_kv_free(moearc_ctx *c, const moearc_x_kv_cache *kv, const unsigned int *seqs, const unsigned int *keep, unsigned int n) {
    const int rc = page_call_check(c, kv);
    if (rc) return rc;
    if (n == 0) return OK;
    if (!seqs) return ERR;
    if (n > KV_LIST) return ERR_ARG;
    kv_rows_seen seen(kv->max_seq);
    for (unsigned i = 0; i < n; ++i)
        if (!seen.add(seqs[i], kv->max_seq)) return ERR_ARG;
    device_guard g(c->device);
    if (!g.ok) return ERR;
    launch_scope ls(c, "kv_free", n, 1);
    const cudaError_t e = with_rows(seqs, keep, n, [&](auto &L) {
        constexpr int N = (int)(sizeof(L.a) / sizeof(unsigned));
        return launch_pdl(k_kv_free<N>, dim3(n), dim3(256), 0, c->stream, L, view_of(*kv));
    });
    const int rc2 = ls.finish();
    return e != cudaSuccess ? finish(c, e) : rc2;
}

int moearc_x_kv_compact(moearc_ctx *c, const moearc_x_kv_cache *kv, unsigned int *tables_out, unsigned int *refs_out,
                        unsigned int *n_live) {
    const int rc = page_call_check(c, kv);
    if (rc) return rc;
    if (!tables_out || !refs_out) return ERR;
    if (!aligned(tables_out, 4) || !aligned(refs_out, 4) || !aligned(n_live, 4)) return ERR_ARG;
    if ((tables_out == kv->tables) != (refs_out == kv->refs)) return ERR_ARG;  // counts that do not go with the tables
    device_guard g(c->device);
    if (!g.ok) return ERR;
    const work_view w = work_of(kv->work, kv->n_pages);
    const cache_view k = view_of(*kv);
    launch_scope ls(c, "kv_compact", kv->n_pages, kv->n_layer);
    cudaError_t e = launch_pdl(k_kv_compact_plan, dim3(1), dim3(PLAN_THREADS), 0, c->stream, k, w);
    if (e == cudaSuccess)
        e = with_pools(*kv, [&](auto v, auto &P, unsigned page_v) {
            constexpr int NP = (int)(sizeof(P.p) / sizeof(void *));
            return launch_pdl(k_kv_compact<decltype(v), NP>, copy_grid(c), dim3(COPY_THREADS), 0, c->stream, P, k, w, page_v, tables_out,
                              refs_out, n_live);
        });
    const int rc2 = ls.finish();
    return e != cudaSuccess ? finish(c, e) : rc2;
}

int moearc_x_kv_status(moearc_ctx *c, const moearc_x_kv_cache *kv) {
    const int rc = kv_check(c, kv);
    if (rc) return rc;
    device_guard g(c->device);
    unsigned v = 0;
    if (!g.ok || cudaMemcpyAsync(&v, kv->status, 4, cudaMemcpyDeviceToHost, c->stream) != cudaSuccess ||
        cudaMemsetAsync(kv->status, 0, 4, c->stream) != cudaSuccess || cudaStreamSynchronize(c->stream) != cudaSuccess)
        return ERR;
    return (int)v;
}

}  // extern "C"
