// Routing by scores: s = sigmoid(logit) or softmax over the experts, choice c = s + bias (a balance bias moves the
// choice, never the weight), optionally only inside the best top_groups of `groups` equal runs of experts (a group is
// worth the sum of its best one or two choices), the k best choices, coefficients s, optionally divided by their sum,
// times a factor.
//
// The work is tiny and the answer is discrete: two choices may lie closer than FP32 tells apart, so scores and choices
// are FP64 (a few exponentials a lane), compared as 64-bit keys; ties go to the lower index. One wave a token. Group gi
// belongs to P = 64 / ceil_pow2(groups) neighbouring lanes (one group: all 64), lane `sub` of them holding experts gi *
// per + sub + P i, so a group's best two are a butterfly over P lanes. The top k as in the plain router: a threshold
// that k lanes' maxima reach, by a search over the keys' high words, then the few keys above it ranked against each
// other. 8.4 us for 6 tokens and for 2048: one wave's chain, not the amount of work.
#include "common.hpp"
#include "route_impl.hpp"

#include <climits>
#include <cmath>

namespace sx {
namespace {

struct Args {
    const void *logits, *shared;
    const float *bias;
    int32_t *ids;
    float *coef;
    uint32_t *err;
    int64_t ld, shared_ld;
    int32_t M, E, k, A, shared_id, groups, per, lanes, top_groups, group_best;  // lanes: P
    int32_t softmax, renorm;
    float factor;
};

// Larger first as unsigned: a double's bits made monotone (-0 as +0).
__device__ __forceinline__ uint64_t order_key(double v) {
    const uint64_t b = v == 0.0 ? 0ull : (uint64_t)__double_as_longlong(v);
    return (b >> 63) ? ~b : b | 0x8000000000000000ull;
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int d) {
    return (uint64_t)__shfl_xor((unsigned long long)v, d);
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) {  // lane: uniform
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ double key_double(uint64_t key) {
    return __longlong_as_double((long long)((key >> 63) ? key & 0x7FFFFFFFFFFFFFFFull : ~key));
}

template <typename T, int NV>
__global__ void __launch_bounds__(64) router_scored_kernel(const Args a) {
    __shared__ uint64_t cand_key[64];
    __shared__ int cand_id[64];
    const int lane = threadIdx.x, P = a.lanes, gi = lane / P, sub = lane % P;
    const int64_t m = blockIdx.x;
    const T *row = static_cast<const T *>(a.logits) + m * a.ld;
    int32_t *ids = a.ids + m * a.A;
    float *coef = a.coef + m * a.A;
    const float sl = a.shared != nullptr ? load_act(static_cast<const T *>(a.shared), m * a.shared_ld) : 0.f;
    auto expert = [&](int j) { return gi < a.groups && sub + P * j < a.per ? gi * a.per + sub + P * j : -1; };

    float v[NV];
    double s[NV];
    int bad = INT_MAX;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = load_act(row, max(expert(j), 0));
#pragma unroll
    for (int j = 0; j < NV; ++j) s[j] = a.bias != nullptr ? (double)a.bias[max(expert(j), 0)] : 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int e = expert(j);
        if (e >= 0 && (!isfinite(v[j]) || !isfinite(s[j]))) bad = min(bad, e);
        if (e >= 0) top = fmaxf(top, v[j]);
    }
    if (a.shared != nullptr && !isfinite(sl)) bad = min(bad, a.E);
    if (__ballot(bad != INT_MAX)) {
        bad = (int)routing::wave_min_u32((uint32_t)bad);
        if (lane == 0) report(a.err, (uint32_t)m, (uint32_t)bad);
        if (lane < a.A) ids[lane] = -1, coef[lane] = qnan();
        return;
    }
    double scale = 0.0, sum = 1.0;  // softmax: the maximum and the sum over all experts
    if (a.softmax) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
        scale = (double)top;
        double part = 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (expert(j) >= 0) part += exp((double)v[j] - scale);
        sum = wave_sum_f64(part);
    }
    auto score = [&](float x) { return a.softmax ? exp((double)x - scale) / sum : 1.0 / (1.0 + exp(-(double)x)); };
    uint64_t key[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) key[j] = expert(j) >= 0 ? order_key(score(v[j]) + s[j]) : 0ull;

    if (a.groups > 1) {
        uint64_t b1 = 0, b2 = 0;  // the group's best two
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const uint64_t lo = min(b1, key[j]);
            b1 = max(b1, key[j]), b2 = max(b2, lo);
        }
        for (int d = 1; d < P; d <<= 1) {
            const uint64_t o1 = shfl_xor64(b1, d), o2 = shfl_xor64(b2, d), lo = min(b1, o1);
            b1 = max(b1, o1), b2 = max(max(b2, o2), lo);
        }
        double worth = key_double(b1);
        if (a.group_best == 2) worth += key_double(b2);
        const uint64_t mine = order_key(worth);
        int rank = 0;
        for (int g = 0; g < a.groups; ++g) {
            const uint64_t o = lane_value(mine, g * P);
            rank += o > mine || (o == mine && g < gi) ? 1 : 0;
        }
        if (rank >= a.top_groups) {
#pragma unroll
            for (int j = 0; j < NV; ++j) key[j] = 0ull;
        }
    }

    // T: k lanes hold a key whose high word reaches it (24 bits of it searched), so every one of the top k does; where
    // fewer than k lanes hold open experts it is 1, which all of those reach
    uint32_t lm = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) lm = max(lm, (uint32_t)(key[j] >> 32));
    uint32_t Th = 0u;
    for (int b = 30; b >= 8; b -= 2) {
        const uint32_t t1 = Th | (1u << b), t2 = Th | (2u << b), t3 = Th | (3u << b);
        const int c1 = __popcll(__ballot(lm >= t1)), c2 = __popcll(__ballot(lm >= t2)), c3 = __popcll(__ballot(lm >= t3));
        Th = c3 >= a.k ? t3 : c2 >= a.k ? t2 : c1 >= a.k ? t1 : Th;
    }
    Th = max(Th, 1u);
    int C = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const bool in = (uint32_t)(key[j] >> 32) >= Th;
        const uint64_t bal = __ballot(in);
        const int pos = C + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(bal >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)bal, 0u));
        if (in && pos < 64) cand_key[pos] = key[j], cand_id[pos] = expert(j);
        C += __popcll(bal);
    }
    int my_id = -1;
    if (C <= 64) {
        __syncthreads();
        const uint64_t mine = lane < C ? cand_key[lane] : 0ull;
        const int id = lane < C ? cand_id[lane] : INT_MAX;
        int rank = lane < C ? 0 : lane;
        if (lane < C)
            for (int c = 0; c < C; ++c) {
                const uint64_t o = cand_key[c];
                rank += o > mine || (o == mine && cand_id[c] < id) ? 1 : 0;
            }
        my_id = __builtin_amdgcn_ds_permute(rank * 4, id);
    } else {  // many equal high words: k rounds of the wave's largest key
        for (int r = 0; r < a.k; ++r) {
            uint64_t best = 0;
#pragma unroll
            for (int j = 0; j < NV; ++j) best = max(best, key[j]);
            const uint32_t hi = routing::wave_max_u32((uint32_t)(best >> 32));
            const uint32_t lo = routing::wave_max_u32((uint32_t)(best >> 32) == hi ? (uint32_t)best : 0u);
            const uint64_t w = ((uint64_t)hi << 32) | lo;
            uint32_t e = 0xFFFFFFFFu;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (key[j] == w) e = min(e, (uint32_t)expert(j));
            e = routing::wave_min_u32(e);
            if (lane == r) my_id = (int)e;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (expert(j) == (int)e) key[j] = 0ull;
        }
    }
    double c = lane < a.k ? score(load_act(row, my_id)) : 0.0;
    if (a.renorm) {
        const double total = wave_sum_f64(c);
        c = total > 0.0 ? c / total : c;
    }
    if (lane < a.k) ids[lane] = my_id, coef[lane] = (float)(c * (double)a.factor);
    if (a.shared != nullptr && lane == 0) ids[a.k] = a.shared_id, coef[a.k] = 1.0f / (1.0f + expf(-sl));
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" int sx_moe_router_scored(const void *logits, int64_t ld, int64_t M, int64_t E, int64_t k, int score, const float *bias,
                                    int64_t groups, int64_t top_groups, int64_t group_best, int renorm, float factor,
                                    const void *shared_logit, int64_t shared_ld, int32_t shared_id, int32_t *ids, float *coef,
                                    int act, uint32_t *err, sx_stream stream) {
    SX_CHECK(logits != nullptr && ids != nullptr && coef != nullptr, "null pointer");
    SX_CHECK(M >= 1 && M <= 0x7fffffff, "M = ", M, " tokens, expected 1..", 0x7fffffff);
    SX_CHECK(E >= 1 && E <= 1024, "E = ", E, " experts, expected 1..1024");
    SX_CHECK(k >= 1 && k <= E && k <= 32, "k = ", k, ", expected 1..min(E = ", E, ", 32)");
    SX_CHECK(ld >= E, "logits row stride ld = ", ld, " < E = ", E);
    SX_CHECK(score == SX_SCORE_SIGMOID || score == SX_SCORE_SOFTMAX, "unknown score ", score);
    SX_CHECK(groups >= 1 && groups <= 64 && E % groups == 0, "groups = ", groups, ", expected 1..64, a divisor of E = ", E);
    SX_CHECK(top_groups >= 1 && top_groups <= groups, "top_groups = ", top_groups, " of ", groups);
    SX_CHECK(top_groups * (E / groups) >= k, "k = ", k, " of ", top_groups * (E / groups), " experts in the chosen groups");
    SX_CHECK(group_best == 1 || (group_best == 2 && E / groups >= 2), "group_best = ", group_best, ", expected 1 or 2, groups of ", E / groups);
    SX_CHECK(std::isfinite(factor), "factor = ", factor);
    if (shared_logit != nullptr) {
        SX_CHECK(shared_ld >= 1, "shared_ld = ", shared_ld, ", expected >= 1");
        SX_CHECK(shared_id >= 0, "shared_id = ", shared_id, ", expected >= 0 (its expert row block)");
    }
    SX_CHECK(act == SX_ACT_F32 || act == SX_ACT_BF16, "unsupported activation dtype ", act);
    const int64_t slots = 4 * M * (k + (shared_logit != nullptr ? 1 : 0)), read = ((M - 1) * ld + E) * act_bytes(act);
    SX_CHECK(apart(ids, slots, coef, slots), "ids and coef are the same buffer or overlap");
    SX_CHECK(apart(ids, slots, logits, read) && apart(coef, slots, logits, read), "ids or coef overlap the logits");
    SX_CHECK(bias == nullptr || (apart(ids, slots, bias, 4 * E) && apart(coef, slots, bias, 4 * E)), "ids or coef overlap the bias");
    const int64_t shared_read = ((M - 1) * shared_ld + 1) * act_bytes(act);
    SX_CHECK(shared_logit == nullptr || (apart(ids, slots, shared_logit, shared_read) && apart(coef, slots, shared_logit, shared_read)),
             "ids or coef overlap the shared logits");
    SX_CHECK(aligned(ids, 4) && aligned(coef, 4) && aligned(bias, 4) && aligned(err, 4) && aligned(logits, act_bytes(act)) &&
                 aligned(shared_logit, act_bytes(act)),
             "ids, coef, bias and err must be 4-byte aligned, the logits to their elements");
    int P = 64;
    while (P * groups > 64) P >>= 1;
    const int per = (int)(E / groups), need = (per + P - 1) / P;
    const Args a{logits, shared_logit, bias, ids, coef, err, ld, shared_ld, (int32_t)M, (int32_t)E, (int32_t)k,
                 (int32_t)(k + (shared_logit != nullptr ? 1 : 0)), shared_id, (int32_t)groups, per, P, (int32_t)top_groups,
                 (int32_t)group_best, score == SX_SCORE_SOFTMAX ? 1 : 0, renorm ? 1 : 0, factor};
    auto go = [&](auto tag, auto nv) {
        router_scored_kernel<decltype(tag), decltype(nv)::value><<<(unsigned)M, 64, 0, stream_of(stream)>>>(a);
    };
    auto by_nv = [&](auto tag) {
        if (need <= 2) go(tag, std::integral_constant<int, 2>{});
        else if (need <= 4) go(tag, std::integral_constant<int, 4>{});
        else if (need <= 8) go(tag, std::integral_constant<int, 8>{});
        else if (need <= 16) go(tag, std::integral_constant<int, 16>{});
        else go(tag, std::integral_constant<int, 32>{});
    };
    if (act == SX_ACT_F32) by_nv(float{});
    else by_nv(uint16_t{});
    SX_LAUNCHED("moe_router_scored M=", M, " E=", E, " k=", k);
    return SX_OK;
}
