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

// `bytes` bytes at p, again at each of up to four (count, byte stride) steps.
struct Strided {
    const void *p;
    int64_t bytes;
    std::pair<int64_t, int64_t> steps[4];
};

// Whether two such blocks surely share no memory: some of the steps that they have in common (number i of both, of equal
// count and stride) repeat a piece that holds one block's span and, behind it, the other's. None of them: the whole spans
// are apart. Interleaved keys and values and slabs of pages and rows are told apart that way.
inline bool strided_apart(Strided a, Strided b) {
    auto pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
    if (pa > pb) std::swap(a, b), std::swap(pa, pb);
    for (int common = 0; common < 16; ++common) {
        __int128 la = a.bytes, lb = b.bytes;
        std::pair<int64_t, int64_t> outer[4];
        bool both = true;
        for (int i = 0; i < 4; ++i) {
            outer[i] = {1, 0};
            if (common >> i & 1) {
                both &= a.steps[i] == b.steps[i] && a.steps[i].first > 1;
                outer[i] = a.steps[i];
            } else {
                la += (__int128)std::max<int64_t>(a.steps[i].first - 1, 0) * a.steps[i].second;
                lb += (__int128)std::max<int64_t>(b.steps[i].first - 1, 0) * b.steps[i].second;
            }
        }
        const __int128 d = (__int128)pb - pa, piece = d + lb;
        if (both && la <= d && (common == 0 || (piece < ((__int128)1 << 62) && rows_apart((int64_t)piece, {outer[0], outer[1], outer[2], outer[3]})))) return true;
    }
    return false;
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
    // inside them the reciprocals, and the products with a softmax's terms, stay in FP32's range
    if (c.dtype == SX_KV_E4M3 && !(c.k_scale >= 0x1p-100f && c.k_scale <= 0x1p100f && c.v_scale >= 0x1p-100f && c.v_scale <= 0x1p100f))
        return cat("k_scale = ", c.k_scale, ", v_scale = ", c.v_scale, ", expected 2^-100..2^100");
    return "";
}

inline std::string head_rows_error(const sx_head_rows &r, const char *name, int64_t heads, int64_t dim) {
    if (!aligned(r.p, 16)) return cat(name, " must be 16-byte aligned");
    if (r.token < 0 || r.head < 0 || r.token > ((int64_t)1 << 40) || r.head > ((int64_t)1 << 40) || r.token % 8 != 0 || r.head % 8 != 0)
        return cat(name, ": strides must be multiples of 8 elements (token ", r.token, ", head ", r.head, ")");
    if (heads > 1 && r.head < dim) return cat(name, ": heads overlap (stride ", r.head, ", dim ", dim, ")");
    return "";
}

inline Strided rows_block(const sx_head_rows &r, int64_t T, int64_t heads, int64_t dim, int64_t layers = 1) {
    return {r.p, dim * 2, {{layers, r.layer * 2}, {1, 0}, {T, r.token * 2}, {heads, r.head * 2}}};
}

inline int64_t head_rows_bytes(const sx_head_rows &r, int64_t T, int64_t heads, int64_t dim) {
    return 2 * ((T - 1) * r.token + (heads - 1) * r.head + dim);
}

// What a cache of all its layers holds for keys (values).
inline Strided kv_block(const sx_kv_cache &c, bool values) {
    const int64_t e = kv_bytes(c);
    if (values) return {c.v, c.dim * e, {{c.layers, c.v_layer * e}, {c.pages, c.v_page * e}, {c.page_size, c.v_token * e}, {c.heads, c.v_head * e}}};
    return {c.k, c.dim * e, {{c.layers, c.k_layer * e}, {c.pages, c.k_page * e}, {c.page_size, c.k_token * e}, {c.heads, c.k_head * e}}};
}

}  // namespace sx
