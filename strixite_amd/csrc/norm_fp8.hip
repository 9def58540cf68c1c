// RMS norm with the residual's addition and an FP8 output: r = x + residual (rounded to the activations' type, as the
// stream keeps it), y = r / sqrt(mean(r^2) + eps) * (w + w_add), and for each run of 128 features of a row e4m3 codes
// with one FP32 scale, amax(|y|) / 448 - the form sx_linear_fp8 takes its activations in.
//
// It has to move its bytes (BF16: 9 a feature and the scales), so a row is read once into registers (8 features a
// 16-byte load), reduced, and written from there. At 2048 rows of 2560 features the VALU is busy all of the time (counters: 431
// instructions a wave on average, an exact division a code among them), so it runs at 3.3 TB/s, 0.63 of a copy. 16 neighbouring lanes hold a run of 128: its maximum is a reduction
// inside a DPP row. Since the row's 1 / rms cancels in y / scale, the codes come from t = r * w alone: code =
// e4m3(448 t / amax(|t|)), one division from exact operands (BF16 r and w: t is exact), so a code is the nearest one.
#include "common.hpp"

#include <cmath>

namespace sx {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Args {
    const void *x, *residual, *weight;
    void *residual_out, *y;
    uint8_t *q;
    float *scale;
    int64_t M, ldx;
    int32_t K;
    float eps, w_add;
};

__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load8(const uint16_t *p, float (&v)[8]) {
    const u32x4 u = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
}
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
    *reinterpret_cast<float4 *>(p) = float4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<float4 *>(p + 4) = float4{v[4], v[5], v[6], v[7]};
}
__device__ __forceinline__ void store8(uint16_t *p, const float (&v)[8]) {
    u32x4 u;
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = f32_to_bf16(v[2 * i]) | (f32_to_bf16(v[2 * i + 1]) << 16);
    *reinterpret_cast<u32x4 *>(p) = u;
}

// The largest of 16 neighbouring lanes (a DPP row), in every one of them.
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// TPR threads a row (whole waves), NV runs of 8 features a thread. A block holds 256 / TPR rows, one where TPR > 256.
template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) norm_fp8_kernel(const Args a) {
    constexpr int kRows = TPR < 256 ? 256 / TPR : 1, kRowWaves = TPR / 64;
    __shared__ float part[kRows][kRowWaves];
    const int tid = threadIdx.x % TPR, sub = threadIdx.x / TPR;
    const int64_t m = (int64_t)blockIdx.x * kRows + sub;
    const bool on = m < a.M;  // whole waves; a row past the last joins the barrier only
    const int n8 = a.K / 8;
    const T *x = static_cast<const T *>(a.x) + m * a.ldx, *w = static_cast<const T *>(a.weight);
    float r[NV][8], wt[NV][8];
    float ss = 0.f;
    if (on) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = tid + j * TPR;
            if (i < n8) {
                load8(x + i * 8, r[j]);
                load8(w + i * 8, wt[j]);
            }
        }
        if (a.residual != nullptr) {
            const T *res = static_cast<const T *>(a.residual) + m * a.K;
            T *out = static_cast<T *>(a.residual_out) + m * a.K;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int i = tid + j * TPR;
                if (i < n8) {
                    float v[8];
                    load8(res + i * 8, v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) r[j][k] = as_stored(r[j][k] + v[k], (const T *)nullptr);
                    store8(out + i * 8, r[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (tid + j * TPR < n8) {
#pragma unroll
                for (int k = 0; k < 8; ++k) ss = fmaf(r[j][k], r[j][k], ss);
            }
    }
    ss = wave_sum(ss);
    if constexpr (kRowWaves > 1) {
        if ((tid & 63) == 0) part[sub][tid >> 6] = ss;
        __syncthreads();
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < kRowWaves; ++i) ss += part[sub][i];
    }
    if (!on) return;
    const float inv = 1.0f / sqrtf(ss / (float)a.K + a.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = tid + j * TPR;
        if (i >= n8) continue;  // whole runs of 128: the 16 lanes of a run are on together
        float t[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) wt[j][k] += a.w_add;
        if (a.y != nullptr) {
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = r[j][k] * inv * wt[j][k];
            store8(static_cast<T *>(a.y) + m * a.K + i * 8, t);
        }
        if (a.q == nullptr) continue;
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            t[k] = r[j][k] * wt[j][k];
            top = max(top, __float_as_uint(t[k]) & 0x7FFFFFFFu);  // as integers: a NaN is the largest
        }
        const float amax = __uint_as_float(row16_max(top));
        // 448 t / amax as (7/8 t) / (amax / 512): neither side leaves the range; runs below 2^-60 are lifted first
        const float lift = amax < 0x1p-60f ? 0x1p64f : 1.0f;
        const float den = amax * lift * 0x1p-9f, num = 0.875f * lift;
        uint32_t o[2] = {0u, 0u};
        if (amax != 0.f) {
            float c[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                c[k] = t[k] * num / den;
                c[k] = c[k] != c[k] ? c[k] : fminf(fmaxf(c[k], -448.f), 448.f);
            }
            o[0] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
            o[0] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], (int)o[0], true);
            o[1] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[4], c[5], 0, false);
            o[1] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c[6], c[7], (int)o[1], true);
        }
        *reinterpret_cast<uint2 *>(a.q + m * a.K + i * 8) = uint2{o[0], o[1]};
        if ((i & 15) == 0) a.scale[m * (a.K / 128) + i / 16] = amax * inv / 448.0f;
    }
}

template <typename T, int TPR, int NV>
void go(const Args &a, hipStream_t s) {
    constexpr int rows = TPR < 256 ? 256 / TPR : 1;
    norm_fp8_kernel<T, TPR, NV><<<(unsigned)((a.M + rows - 1) / rows), TPR < 256 ? 256 : TPR, 0, s>>>(a);
}

// One run of 8 a thread, so that a row's loads are all in flight at once, up to 8192 features; rows of few features share
// a block. (2048 rows of 2560 in us: a wave a row and five runs a lane 16.9, 256 threads 15.0, 512 14.7; 6 of 4096: 512
// threads 4.1, 256 and two runs 5.2.)
template <typename T>
void launch(const Args &a, hipStream_t s) {
    const int n8 = a.K / 8;
    if (n8 <= 64) go<T, 64, 1>(a, s);
    else if (n8 <= 128) go<T, 128, 1>(a, s);
    else if (n8 <= 256) go<T, 256, 1>(a, s);
    else if (n8 <= 512) go<T, 512, 1>(a, s);
    else if (n8 <= 1024) go<T, 1024, 1>(a, s);
    else if (n8 <= 2048) go<T, 1024, 2>(a, s);
    else go<T, 1024, 4>(a, s);
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" int sx_add_rms_norm_fp8(const void *x, int64_t ldx, const void *residual, const void *weight, int64_t M, int64_t K,
                                   float eps, float w_add, void *residual_out, void *y, uint8_t *q, float *scale, int act,
                                   sx_stream stream) {
    SX_CHECK(x != nullptr && weight != nullptr, "null pointer");
    SX_CHECK(q != nullptr || y != nullptr, "no output: q and y are null");
    SX_CHECK((q == nullptr) == (scale == nullptr), "q and scale go together");
    SX_CHECK((residual == nullptr) == (residual_out == nullptr), "residual and residual_out go together");
    SX_CHECK(act == SX_ACT_F32 || act == SX_ACT_BF16, "unsupported activation dtype ", act);
    SX_CHECK(M >= 1 && M <= 0x7fffffff, "M = ", M);
    SX_CHECK(K >= 128 && K % 128 == 0 && K <= 32768, "K = ", K, ", expected a multiple of 128, 128..32768");
    SX_CHECK(ldx >= K && ldx % 8 == 0, "ldx = ", ldx, ", expected a multiple of 8, >= K = ", K);
    SX_CHECK(std::isfinite(eps) && eps >= 0.f && std::isfinite(w_add), "eps = ", eps, ", w_add = ", w_add);
    SX_CHECK(aligned(x, 16) && aligned(residual, 16) && aligned(weight, 16) && aligned(residual_out, 16) && aligned(y, 16) && aligned(q, 8),
             "x, residual, weight, residual_out and y must be 16-byte and q 8-byte aligned");
    const int e = act_bytes(act);
    const int64_t xb = ((M - 1) * ldx + K) * e, rb = M * K * e, sb = M * (K / 128) * 4;
    // a row is read before it is written: y may be x or the residual, and residual_out the residual or x, row for row
    const bool same_x = ldx == K;
    auto in_place = [&](const void *o, const void *in, int64_t in_bytes, bool rows_match) {
        return o == nullptr || in == nullptr || (o == in && rows_match) || apart(o, rb, in, in_bytes);
    };
    SX_CHECK(in_place(y, x, xb, same_x) && in_place(residual_out, x, xb, same_x) && in_place(y, residual, rb, true) &&
                 in_place(residual_out, residual, rb, true),
             "an output overlaps an input at other rows");
    SX_CHECK(y == nullptr || residual_out == nullptr || apart(y, rb, residual_out, rb), "y overlaps residual_out");
    auto clear = [&](const void *o, int64_t n) {
        return o == nullptr || (apart(o, n, x, xb) && apart(o, n, weight, K * e) && (residual == nullptr || (apart(o, n, residual, rb) && apart(o, n, residual_out, rb))) &&
                                (y == nullptr || apart(o, n, y, rb)));
    };
    SX_CHECK(clear(q, M * K) && clear(scale, sb) && (q == nullptr || apart(q, M * K, scale, sb)), "q or scale overlaps another argument");
    SX_CHECK((y == nullptr || apart(y, rb, weight, K * e)) && (residual_out == nullptr || apart(residual_out, rb, weight, K * e)), "an output overlaps the weight");
    const Args a{x, residual, weight, residual_out, y, q, scale, M, ldx, (int32_t)K, eps, w_add};
    if (act == SX_ACT_F32) launch<float>(a, stream_of(stream));
    else launch<uint16_t>(a, stream_of(stream));
    SX_LAUNCHED("add_rms_norm_fp8 M=", M, " K=", K);
    return SX_OK;
}
