// kvcache.cuh — what the calls on a paged cache of many sequences share: the checks of
// moearc_x_kv_cache, row lists passed by value, the device guard and a block-wide scan.
#pragma once

#include <cstring>

#include "common.cuh"

namespace moearc {

constexpr unsigned NO_PAGE = MOEARC_X_NO_PAGE;
constexpr unsigned KV_LIST = MOEARC_X_KV_LIST;
constexpr unsigned KV_LAYERS = MOEARC_X_KV_LAYERS;
constexpr unsigned KV_MAX_SEQ = 65536;

inline unsigned kv_elem_bytes(unsigned t) { return t == T_F32 ? 4 : (t == T_F16 || t == T_BF16) ? 2 : 0; }

// Ranges of the plain numbers in a cache's description.
inline bool kv_shape_ok(const moearc_x_kv_cache &k) {
    return k.n_layer >= 1 && k.n_layer <= KV_LAYERS && k.n_pages >= 1 && k.n_pages <= (1u << 28) && k.page_tokens >= 1 &&
           k.n_kv_heads >= 1 && k.n_kv_heads <= 65535 && k.head_dim >= 1 && k.head_dim <= 1024 && kv_elem_bytes(k.kv_type) &&
           k.max_seq >= 1 && k.max_seq <= KV_MAX_SEQ && k.max_pages >= 1 && k.max_pages <= (1u << 24) &&
           (unsigned long long)k.max_pages * k.page_tokens < (1ull << 31) &&
           (unsigned long long)k.page_tokens * k.n_kv_heads < (1ull << 31) / k.head_dim;  // a page's elements, for 32-bit indexes
}

// Whether an address is a whole number of `each` bytes (2 or 4); NULL is.
inline bool aligned(const void *p, unsigned each) { return (reinterpret_cast<uintptr_t>(p) & (each - 1)) == 0; }

// 0 when every pointer is there and every number in range; else the code to return.
inline int kv_check(const moearc_ctx *c, const moearc_x_kv_cache *k) {
    if (!c || !k || !k->k_pages || !k->v_pages || !k->tables || !k->n_kv || !k->refs || !k->status || !k->work) return ERR;
    if (!kv_shape_ok(*k)) return ERR_ARG;
    for (unsigned l = 0; l < k->n_layer; ++l)
        if (!k->k_pages[l] || !k->v_pages[l]) return ERR;
    const unsigned each = kv_elem_bytes(k->kv_type);
    for (unsigned l = 0; l < k->n_layer; ++l)
        if (!aligned(k->k_pages[l], each) || !aligned(k->v_pages[l], each)) return ERR_ARG;
    if (!aligned(k->tables, 4) || !aligned(k->n_kv, 4) || !aligned(k->refs, 4) || !aligned(k->status, 4)) return ERR_ARG;
    if (reinterpret_cast<uintptr_t>(k->work) & 15) return ERR_ARG;
    return OK;
}

// The rows of one list: below max_seq and distinct, none of them already marked in `seen`
// (one bit a row).
struct kv_rows_seen {
    unsigned bits[KV_MAX_SEQ / 32];
    explicit kv_rows_seen(unsigned max_seq) { std::memset(bits, 0, (max_seq + 31) / 32 * 4); }
    bool has(unsigned s) const { return bits[s >> 5] >> (s & 31) & 1; }
    bool add(unsigned s, unsigned max_seq) {
        if (s >= max_seq || has(s)) return false;
        bits[s >> 5] |= 1u << (s & 31);
        return true;
    }
};

// The context's device made current for a call, and the caller's put back.
struct device_guard {
    int prev = -1, dev;
    bool ok;
    explicit device_guard(int d) : dev(d) {
        ok = cudaGetDevice(&prev) == cudaSuccess && (prev == dev || cudaSetDevice(dev) == cudaSuccess);
    }
    ~device_guard() {
        if (ok && prev != dev) cudaSetDevice(prev);
    }
};

// Inclusive sum over the CTA (blockDim.x a multiple of 32, <= 1024); warp_sums: 32 words of
// shared memory, free again after the call's last barrier. *total gets the CTA's sum.
template <typename T>
__device__ __forceinline__ T block_scan(T v, T *warp_sums, T *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        T w = lane < nw ? warp_sums[lane] : T(0);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const T u = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += u;
        }
        if (lane < nw) warp_sums[lane] = w;
    }
    __syncthreads();
    if (warp > 0) v += warp_sums[warp - 1];
    *total = warp_sums[nw - 1];
    __syncthreads();
    return v;
}

}  // namespace moearc
