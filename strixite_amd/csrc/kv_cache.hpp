// Host checks of a paged key / value cache (sx_kv_cache) and of packed head rows (sx_head_rows), shared by the calls
// that read and write them.
#pragma once
#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <utility>

namespace sx {

// Whether rows of dim values at these (count, element stride) steps share no memory: each stride passes what the
// smaller ones cover. Asked of what a kernel writes; what it reads may be expanded.
inline bool rows_apart(int64_t dim, std::initializer_list<std::pair<int64_t, int64_t>> steps) {
    std::pair<int64_t, int64_t> s[4];
    const int n = (int)(std::copy_if(steps.begin(), steps.end(), s, [](const auto &x) { return x.first > 1; }) - s);
    std::sort(s, s + n, [](const auto &x, const auto &y) { return x.second < y.second; });
    __int128 covered = dim;
    for (int i = 0; i < n; ++i) {
        if (s[i].second < covered) return false;
        covered += (__int128)(s[i].first - 1) * s[i].second;
    }
    return true;
}

inline int kv_bytes(const sx_kv_cache &c) { return c.dtype == SX_KV_E4M3 ? 1 : 2; }

// Why a cache is not one that the kernels take; empty where it is. Pages hold whole 16-token tiles, rows are loaded
// 16 bytes at a time, and a page's tokens are addressed by 31-bit offsets (the pages themselves by 64-bit ones).
inline std::string kv_cache_error(const sx_kv_cache &c) {
    if (c.k == nullptr || c.v == nullptr || c.table == nullptr || c.lens == nullptr) return "null pointer in the cache";
    if (c.dtype != SX_KV_BF16 && c.dtype != SX_KV_E4M3) return cat("unsupported cache dtype ", c.dtype);
    const int e = kv_bytes(c);
    if (c.page_size < 16 || c.page_size > 65536 || (c.page_size & (c.page_size - 1)) != 0)
        return cat("page_size = ", c.page_size, ", expected a power of two, 16..65536");
    if (c.pages < 1 || c.pages > 0x7fffffff) return cat("pages = ", c.pages);
    if (c.heads < 1 || c.heads > 4096 || c.dim < 8 || c.dim > 1024 || c.dim % 8 != 0) return cat("heads = ", c.heads, ", dim = ", c.dim);
    if (c.batch < 1 || c.batch > 65535) return cat("batch = ", c.batch, ", expected 1..65535");
    if (c.pages_per_seq < 1 || c.pages_per_seq * c.page_size > 0x7fffffff - 65536)
        return cat("pages_per_seq = ", c.pages_per_seq, " of ", c.page_size, " tokens");
    if (c.table_ld < c.pages_per_seq) return cat("table_ld = ", c.table_ld, " < pages_per_seq = ", c.pages_per_seq);
    if (c.layers < 1 || c.layers > 65535) return cat("layers = ", c.layers);
    const int64_t s[8] = {c.k_page, c.v_page, c.k_token, c.v_token, c.k_head, c.v_head, c.k_layer, c.v_layer};
    for (int i = 0; i < 8; ++i)
        if (s[i] < 0 || s[i] > ((int64_t)1 << 40) || (s[i] * e) % 16 != 0)
            return cat("cache strides must be multiples of 16 bytes (", s[i], " elements)");
    if (!aligned(c.k, 16) || !aligned(c.v, 16)) return "the cache must be 16-byte aligned";
    if (c.k_token * e * c.page_size > 0x7fffffff || c.v_token * e * c.page_size > 0x7fffffff)
        return "a page spans more than 2^31 bytes";
    if (c.dtype == SX_KV_E4M3 && !(std::isfinite(c.k_scale) && c.k_scale > 0.f && std::isfinite(c.v_scale) && c.v_scale > 0.f))
        return cat("k_scale = ", c.k_scale, ", v_scale = ", c.v_scale, ", expected positive");
    return "";
}

inline std::string head_rows_error(const sx_head_rows &r, const char *name, int64_t heads, int64_t dim) {
    if (!aligned(r.p, 16)) return cat(name, " must be 16-byte aligned");
    if (r.token < 0 || r.head < 0 || r.token > ((int64_t)1 << 40) || r.head > ((int64_t)1 << 40) || r.token % 8 != 0 || r.head % 8 != 0)
        return cat(name, ": strides must be multiples of 8 elements (token ", r.token, ", head ", r.head, ")");
    if (heads > 1 && r.head < dim) return cat(name, ": heads overlap (stride ", r.head, ", dim ", dim, ")");
    return "";
}

inline int64_t head_rows_bytes(const sx_head_rows &r, int64_t T, int64_t heads, int64_t dim) {
    return 2 * ((T - 1) * r.token + (heads - 1) * r.head + dim);
}

}  // namespace sx
