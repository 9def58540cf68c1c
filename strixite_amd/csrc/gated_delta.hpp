// What the gated delta rule's kernels share: their arguments, a sequence's words and their checks, gates, and the exact
// split of FP32 values into BF16 operands.
#pragma once
#include "common.hpp"

namespace sx {
namespace delta {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kMaxSeqs = 1024;
constexpr float kNormEps = 1e-6f;

struct Args {
    const uint16_t *q, *k, *v;
    const void *a, *b;
    const float *A_log, *dt_bias;
    float *state;
    const int32_t *slot, *starts;
    uint16_t *out;
    uint32_t *err;
    int64_t q_t, q_h, k_t, k_h, v_t, v_h, a_t, b_t, o_t, o_h, s_slot;  // element strides: token, head; of a state
    int32_t T, Hk, Hv, rep, Dv, B, slots, max_len;
    float scale;
    bool f32_gates, normalize;
};

// A sequence's rows t0 .. t0 + n - 1 and its state. run false: its words are impossible, nothing of it is touched. ok
// false: its rows are NaN and its state stays as it is. Starts that fall make every sequence from the falling one on impossible: what
// lies behind could be another's rows, and two blocks that write one row, or two sequences' chunks in one place of a prompt's
// workspace, would race.
struct Seq {
    int t0, n, slot;
    bool run, ok;
};

// Every lane of a wave calls this with the same b. alone: the state will be written, so no other sequence with tokens may
// have it (one with the same slot is refused, as is this one).
__device__ __forceinline__ Seq sequence(const int32_t *starts, const int32_t *slots, int b, int B, int T, int max_len, int states, bool alone) {
    const int t0 = starts[b], t1 = starts[b + 1];
    const int slot = slots != nullptr ? slots[b] : b;
    Seq s{t0, (int)((uint32_t)t1 - (uint32_t)t0), slot, t0 >= 0 && t1 >= t0 && t1 <= T && t1 - t0 <= max_len, slot >= 0 && slot < states};
    const bool others = alone && slots != nullptr;
    bool twice = false, falls = false;
    for (int j = threadIdx.x & 63; j < (others ? B : b); j += 64) {
        const int at = starts[j], next = starts[j + 1];
        if (j < b && next < at) falls = true;
        if (others && j != b && slots[j] == slot && next > at) twice = true;
    }
    if (__any(falls)) s.run = false;
    if (__any(twice)) s.ok = false;
    if (!s.run) s.n = 0;
    return s;
}

// The words of an unusable sequence, by one thread of the launch for each.
__device__ __forceinline__ void tell(const Seq &s, int b, uint32_t *err) {
    if (!s.run) report(err, (uint32_t)s.t0, (uint32_t)b);
    else if (s.n > 0 && !s.ok) report(err, (uint32_t)s.slot, (uint32_t)b);
}

// The logarithm of token t's decay for head h, and the share of its correction that is written. A decay of -1e4 and less, -inf too,
// is a full reset: e to it is 0, and sums and differences of it stay numbers.
__device__ __forceinline__ void gates(const Args &a, int64_t t, int h, float &g, float &beta) {
    const float x = a.f32_gates ? static_cast<const float *>(a.a)[t * a.a_t + h] : bf16_to_f32(static_cast<const uint16_t *>(a.a)[t * a.a_t + h]);
    const float y = a.f32_gates ? static_cast<const float *>(a.b)[t * a.b_t + h] : bf16_to_f32(static_cast<const uint16_t *>(a.b)[t * a.b_t + h]);
    g = x, beta = y;
    if (a.A_log != nullptr) {
        const float z = x + a.dt_bias[h];
        g = -expf(a.A_log[h]) * (z > 20.f ? z : log1pf(expf(z)));
        beta = 1.f / (1.f + expf(-y));
    }
    g = g < -1e4f ? -1e4f : g;
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// The factors that scale a key and a query, from their sums of squares. A key whose squares overflow has no length in FP32 and its
// products with others none either: it is no number, in every form. So is a query that is to be divided by its length.
__device__ __forceinline__ float key_scale(const Args &a, float kk) { return !finite(kk) ? qnan() : a.normalize ? 1.f / sqrtf(kk + kNormEps) : 1.f; }
__device__ __forceinline__ float query_scale(const Args &a, float qq) {
    return (!a.normalize ? 1.f : finite(qq) ? 1.f / sqrtf(qq + kNormEps) : qnan()) * a.scale;
}

__device__ __forceinline__ void unpack8(u32x4 u, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
}

// Sums over lanes l, l ^ 16 (and l ^ 32), in all of them.
__device__ __forceinline__ float sum_rows(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Lane (l & 15) + 16 G's value, in all of l's four lanes.
template <int G>
__device__ __forceinline__ float of_row(float x) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const uint32_t h = b[G >> 1];
    const auto a = __builtin_amdgcn_permlane16_swap(h, h, false, false);
    return __uint_as_float(a[G & 1]);
}

// The upper halves of two words as one.
__device__ __forceinline__ uint32_t tops(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302); }

// Eight FP32 values as N BF16 operands: each takes the next eight leading bits, so three of them are the value itself
// (24 bits; what is left after each is exact). Products of such operands with BF16 values are exact, their sums FP32:
// a state meets the matrix unit without being rounded, for corrections and outputs alike. Of a product of two FP32 values the six
// largest of nine products are taken.
template <int N>
__device__ __forceinline__ void split(const float (&x)[8], bf16x8 (&o)[N]) {
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
    for (int s = 0; s < N; ++s) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = tops(__float_as_uint(r[2 * i]), __float_as_uint(r[2 * i + 1]));
        o[s] = __builtin_bit_cast(bf16x8, w);
        if (s + 1 < N) {
#pragma unroll
            for (int i = 0; i < 8; ++i) r[i] -= __uint_as_float(__float_as_uint(r[i]) & 0xFFFF0000u);
        }
    }
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Host: what prefill needs (gated_delta_prefill.hip).
size_t prefill_bytes(int64_t T, int64_t B, int64_t Hk, int64_t Hv, int64_t Dk);
void prefill(const Args &a, int Dk, void *ws, hipStream_t s);

}  // namespace delta
}  // namespace sx
