// The accepted tokens of a verify into the paged cache of every layer, one launch.
//
// Token i < count[b] of sequence b is drafted row starts[b] + path[b, i] and goes to position lens[b] + i: page
// table[b, position / page], row position % page, for keys and values of each layer; an FP8 cache takes e4m3(x / scale).
// It moves 2 layers tokens Hkv D values and computes nothing, so the kernel is a copy in 16-byte pieces of the source
// whose only care is that the chain ahead of the first store is short: lengths, counts and path are one round trip,
// the page and the source rows the second. 48 sequences, 24 layers, 8 heads of 128 into FP8: 17.4 us, the VALU busy 0.79 of
// it (the pieces' addresses, divisions and conversions; counters); one sequence, 48 layers: 3.3.
#include "kv_cache.hpp"

namespace sx {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kPieces = 4;

struct Args {
    const uint16_t *kn, *vn;
    uint8_t *kc, *vc;
    const int32_t *table, *lens, *starts, *count, *path;
    int32_t *lens_out;
    uint32_t *err;
    int64_t kn_l, kn_t, kn_h, vn_l, vn_t, vn_h;                                  // element strides: layer, token, head
    int64_t kc_l, kc_p, kc_t, kc_h, vc_l, vc_p, vc_t, vc_h;                      // byte strides: layer, page, token, head
    int64_t table_ld, path_ld;
    int32_t B, T, P, pages, page_shift, heads, dim8, per_token;  // per_token: 16-byte pieces of a token over all layers
    int32_t max_count;
    float k_scale, v_scale;
};

// Two values to e4m3, saturating at +-448 (NaN stays NaN).
__device__ __forceinline__ uint32_t pack2_e4m3(float a, float b, uint32_t old, bool hi) {
    a = a != a ? a : fminf(fmaxf(a, -448.f), 448.f);
    b = b != b ? b : fminf(fmaxf(b, -448.f), 448.f);
    return hi ? (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)old, true) : (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, (int)old, false);
}

template <bool F8>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const Args a) {
    const int b = blockIdx.z, i = blockIdx.y;
    const int t0 = a.starts[b], t1 = a.starts[b + 1], len = a.lens[b], cnt = a.count[b];
    if (i > 0 && i >= cnt) return;
    // every block of a sequence looks all of its words over, so that they agree: it is appended to as asked or not at all
    const bool odd = t0 < 0 || t1 < t0 || t1 > a.T || len < 0 || cnt < 0 || cnt > a.max_count ||
                     (int64_t)len + cnt > ((int64_t)a.P << a.page_shift);
    uint32_t word = (uint32_t)cnt;
    bool bad = odd;
    if (!odd)
        for (int j = threadIdx.x; j < cnt; j += kThreads) {
            const int node = a.path != nullptr ? a.path[b * a.path_ld + j] : j;
            const int page = a.table[b * a.table_ld + ((len + j) >> a.page_shift)];
            if ((uint32_t)page >= (uint32_t)a.pages) bad = true, word = (uint32_t)page;
            else if (node < 0 || node >= t1 - t0) bad = true, word = (uint32_t)node;
        }
    const bool any_bad = __syncthreads_or(bad);
    if (blockIdx.x == 0 && i == 0) {
        if (bad) report(a.err, word, (uint32_t)b);
        if (threadIdx.x == 0 && a.lens_out != nullptr) a.lens_out[b] = any_bad ? len : len + cnt;
    }
    if (any_bad || i >= cnt) return;
    const int node = a.path != nullptr ? a.path[b * a.path_ld + i] : i;
    const int pos = len + i, page = a.table[b * a.table_ld + (pos >> a.page_shift)];
    const int64_t tok = t0 + node, row = pos & ((1 << a.page_shift) - 1);
    // kPieces pieces a thread, all read before the first is written
    u32x4 w[kPieces];
    uint8_t *dst[kPieces];
    float unit[kPieces];
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
        const int u = min((int)(blockIdx.x * kPieces + j) * kThreads + (int)threadIdx.x, a.per_token - 1);  // past the end: the last again
        const int d = u % a.dim8, r = u / a.dim8, h = r % a.heads, r2 = r / a.heads, layer = r2 >> 1;
        const bool is_v = r2 & 1;
        w[j] = *reinterpret_cast<const u32x4 *>((is_v ? a.vn + layer * a.vn_l + tok * a.vn_t + h * a.vn_h : a.kn + layer * a.kn_l + tok * a.kn_t + h * a.kn_h) + d * 8);
        dst[j] = (is_v ? a.vc + layer * a.vc_l + page * a.vc_p + row * a.vc_t + h * a.vc_h
                       : a.kc + layer * a.kc_l + page * a.kc_p + row * a.kc_t + h * a.kc_h) + d * (F8 ? 8 : 16);
        unit[j] = is_v ? a.v_scale : a.k_scale;
    }
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
        if ((int)(blockIdx.x * kPieces + j) * kThreads + (int)threadIdx.x >= a.per_token) break;
        if constexpr (!F8) {
            *reinterpret_cast<u32x4 *>(dst[j]) = w[j];
        } else {
            uint32_t o[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 4; ++k)
                o[k >> 1] = pack2_e4m3(bf16_to_f32(w[j][k] & 0xFFFFu) / unit[j], __uint_as_float(w[j][k] & 0xFFFF0000u) / unit[j], o[k >> 1], k & 1);
            *reinterpret_cast<uint2 *>(dst[j]) = uint2{o[0], o[1]};
        }
    }
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" int sx_kv_append(const sx_head_rows *k_new, const sx_head_rows *v_new, int64_t T, const sx_kv_cache *cache,
                            const int32_t *starts, const int32_t *count, int64_t max_count, const int32_t *path,
                            int64_t path_ld, int32_t *lens_out, uint32_t *err, sx_stream stream) {
    SX_CHECK(k_new != nullptr && v_new != nullptr && cache != nullptr && k_new->p != nullptr && v_new->p != nullptr &&
                 starts != nullptr && count != nullptr,
             "null pointer");
    std::string why = kv_cache_error(*cache);
    SX_CHECK(why.empty(), why);
    why = head_rows_error(*k_new, "k_new", cache->heads, cache->dim);
    if (why.empty()) why = head_rows_error(*v_new, "v_new", cache->heads, cache->dim);
    SX_CHECK(why.empty(), why);
    SX_CHECK(k_new->layer >= 0 && v_new->layer >= 0 && k_new->layer % 8 == 0 && v_new->layer % 8 == 0,
             "layer strides must be multiples of 8 elements (", k_new->layer, ", ", v_new->layer, ")");
    SX_CHECK(T >= 1 && T <= 0x7fffffff, "T = ", T);
    const sx_kv_cache &c = *cache;
    SX_CHECK(rows_apart(c.dim, {{c.layers, c.k_layer}, {c.pages, c.k_page}, {c.page_size, c.k_token}, {c.heads, c.k_head}}) &&
                 rows_apart(c.dim, {{c.layers, c.v_layer}, {c.pages, c.v_page}, {c.page_size, c.v_token}, {c.heads, c.v_head}}),
             "rows of the cache share memory");
    SX_CHECK(max_count >= 1 && max_count <= 65535, "max_count = ", max_count, ", expected 1..65535");
    SX_CHECK(path == nullptr || path_ld >= max_count, "path_ld = ", path_ld, " < max_count = ", max_count);
    // one block writes a sequence's lens_out while its others still read these
    const int64_t n4 = cache->batch * 4;
    SX_CHECK(lens_out == nullptr ||
                 (apart(lens_out, n4, cache->lens, n4) && apart(lens_out, n4, starts, n4 + 4) && apart(lens_out, n4, count, n4) &&
                  apart(lens_out, n4, cache->table, 4 * ((cache->batch - 1) * cache->table_ld + cache->pages_per_seq)) &&
                  (path == nullptr || apart(lens_out, n4, path, 4 * ((cache->batch - 1) * path_ld + max_count)))),
             "lens_out overlaps lens, starts, count, path or the table");
    SX_CHECK(cache->layers * cache->heads * cache->dim <= 0x3fffffff, "layers * heads * dim too large");
    SX_CHECK(strided_apart(kv_block(c, false), kv_block(c, true)), "the caches of keys and values share memory");
    for (const bool values : {false, true})  // rows are read while others are written
        SX_CHECK(strided_apart(rows_block(*k_new, T, c.heads, c.dim, c.layers), kv_block(c, values)) &&
                     strided_apart(rows_block(*v_new, T, c.heads, c.dim, c.layers), kv_block(c, values)),
                 "k_new or v_new lies in the cache that is written");
    SX_CHECK(aligned(starts, 4) && aligned(count, 4) && aligned(path, 4) && aligned(lens_out, 4) && aligned(c.lens, 4) && aligned(c.table, 4) &&
                 aligned(err, 4),
             "starts, count, path, lens, the table, lens_out and err must be 4-byte aligned");
    const int e = kv_bytes(*cache);
    Args a;
    a.kn = static_cast<const uint16_t *>(k_new->p), a.kn_l = k_new->layer, a.kn_t = k_new->token, a.kn_h = k_new->head;
    a.vn = static_cast<const uint16_t *>(v_new->p), a.vn_l = v_new->layer, a.vn_t = v_new->token, a.vn_h = v_new->head;
    a.kc = static_cast<uint8_t *>(cache->k), a.vc = static_cast<uint8_t *>(cache->v);
    a.kc_l = cache->k_layer * e, a.kc_p = cache->k_page * e, a.kc_t = cache->k_token * e, a.kc_h = cache->k_head * e;
    a.vc_l = cache->v_layer * e, a.vc_p = cache->v_page * e, a.vc_t = cache->v_token * e, a.vc_h = cache->v_head * e;
    a.table = cache->table, a.table_ld = cache->table_ld, a.lens = cache->lens, a.starts = starts, a.count = count;
    a.path = path, a.path_ld = path_ld, a.lens_out = lens_out, a.err = err;
    a.B = (int32_t)cache->batch, a.T = (int32_t)T, a.P = (int32_t)cache->pages_per_seq, a.pages = (int32_t)cache->pages;
    a.page_shift = __builtin_ctzll((uint64_t)cache->page_size), a.heads = (int32_t)cache->heads;
    a.dim8 = (int32_t)(cache->dim / 8), a.per_token = (int32_t)(2 * cache->layers * cache->heads * a.dim8);
    a.max_count = (int32_t)max_count, a.k_scale = cache->k_scale, a.v_scale = cache->v_scale;
    const dim3 grid((unsigned)((a.per_token + kThreads * kPieces - 1) / (kThreads * kPieces)), (unsigned)max_count, (unsigned)cache->batch);
    if (cache->dtype == SX_KV_E4M3) kv_append_kernel<true><<<grid, kThreads, 0, stream_of(stream)>>>(a);
    else kv_append_kernel<false><<<grid, kThreads, 0, stream_of(stream)>>>(a);
    SX_LAUNCHED("kv_append B=", cache->batch, " layers=", cache->layers);
    return SX_OK;
}
