// FP8 linear with a scale for each block of 128: y[m, n] = sum_b sx[m, b] * sw[n / 128, b] * sum_{k in block b} x[m, k]
// w[n, k], x and w e4m3 codes, the scales FP32, sums over the blocks in FP32, one rounding at the store.
//
// One v_mfma_f32_16x16x128_f8f6f4 is exactly one block of 16 rows x 16 tokens: its result is scaled by sx * sw as it
// is added to the running sum (four FMAs for 32768 products). W is the A operand and x the B operand, so a lane holds
// one token (its sx) and four weight rows, and 16 rows of W share one sw.
#include "common.hpp"

namespace sx {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct Args {
    const uint8_t *x, *w;
    const float *xs, *ws;
    void *y;
    int64_t N;
    int32_t M, K, kb;  // kb = K / 128
};

// 32 codes of a row as an operand of the 128-wide product: lane group g holds codes 32 g .. 32 g + 31 of the block.
__device__ __forceinline__ i32x8 load32(const uint8_t *p) {
    const i32x4 a = *reinterpret_cast<const i32x4 *>(p), b = *reinterpret_cast<const i32x4 *>(p + 16);
    return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

__device__ __forceinline__ bf16x8 as_bf16x8(int lo, int hi) {
    const auto pair = [](int w, bool up) {
        return __builtin_bit_cast(uint32_t, up ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                                               : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    };
    return __builtin_bit_cast(bf16x8, u32x4{pair(lo, false), pair(lo, true), pair(hi, false), pair(hi, true)});
}

// A block's products of 16 rows and 16 tokens. The FP8 instructions keep fewer bits than FP32 of the products of one
// block (1.4e-5 of the result, root mean square, on random codes): a hundredth of a BF16 output's rounding, but far
// over an FP32 output's. FP32 outputs take the codes as BF16, exact there, whose products are summed in FP32 (a quarter
// of the rate; they are logits of few tokens, bound by the weight's bytes).
template <bool F32>
__device__ __forceinline__ f32x4 block_products(i32x8 a, i32x8 b) {
    f32x4 d = {0.f, 0.f, 0.f, 0.f};
    if constexpr (!F32) {
        d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, d, 0, 0, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a[i], a[i + 1]), as_bf16x8(b[i], b[i + 1]), d, 0, 0, 0);
    }
    return d;
}

// ---------------- few tokens: the weight's bytes are the cost ----------------
// A block takes 16 weight rows and 16 MT tokens; its 8 waves split K block by block, and their sums meet in LDS in
// wave order.
constexpr int kRowWaves = 8;

template <typename TY, int MT>
__global__ void __launch_bounds__(64 * kRowWaves) fp8_rows_kernel(const Args a) {
    __shared__ f32x4 part[kRowWaves][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int m0 = blockIdx.y * 16 * MT;
    const uint8_t *w = a.w + min(n0 + n16, a.N - 1) * a.K + g * 32;
    const float *ws = a.ws + n0 / 128 * a.kb;
    const uint8_t *x[MT];
    const float *xs[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t m = min(m0 + t * 16 + n16, a.M - 1);
        x[t] = a.x + m * a.K + g * 32, xs[t] = a.xs + m * a.kb;
    }
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int b = wave; b < a.kb; b += kRowWaves) {
        const i32x8 A = load32(w + b * 128);
        const float sw = ws[b];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const f32x4 d = block_products<sizeof(TY) == 4>(A, load32(x[t] + b * 128));
            const float s = sw * xs[t][b];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(d[i], s, acc[t][i]);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    const float *p = reinterpret_cast<const float *>(part);
    TY *y = static_cast<TY *>(a.y);
    for (int i = threadIdx.x; i < MT * 256; i += 64 * kRowWaves) {
        const int n = i & 15, m = i >> 4;  // token m of the block, row n: lane (m % 16) + 16 (n / 4), value n % 4
        const int at = ((m >> 4) * 64 + (m & 15) + 16 * (n >> 2)) * 4 + (n & 3);
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < kRowWaves; ++v) sum += p[v * MT * 256 + at];
        if (m0 + m < a.M && n0 + n < a.N) store_act(y, (m0 + m) * a.N + n0 + n, sum);
    }
}

template <typename TY>
void launch(const Args &a, hipStream_t s) {
    const unsigned gx = (unsigned)((a.N + 15) / 16);
    if (a.M <= 16) fp8_rows_kernel<TY, 1><<<dim3(gx, 1), 64 * kRowWaves, 0, s>>>(a);
    else if (a.M <= 32) fp8_rows_kernel<TY, 2><<<dim3(gx, 1), 64 * kRowWaves, 0, s>>>(a);
    else fp8_rows_kernel<TY, 4><<<dim3(gx, (unsigned)((a.M + 63) / 64)), 64 * kRowWaves, 0, s>>>(a);
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" int sx_linear_fp8(const uint8_t *x, const float *x_scale, const sx_fp8_view *w, void *y, int64_t M, int out_act,
                             sx_stream stream) {
    SX_CHECK(x != nullptr && x_scale != nullptr && w != nullptr && w->q != nullptr && w->scale != nullptr && y != nullptr,
             "null pointer");
    const int64_t N = w->N, K = w->K;
    SX_CHECK(N >= 1 && N <= 0x7ffffff0 && K >= 128 && K % 128 == 0 && K <= 65536, "weight [", N, ", ", K, "]: K a multiple of 128, 128..65536");
    SX_CHECK(M >= 1 && M <= 4194240, "M = ", M, ", expected 1..4194240");
    SX_CHECK(out_act == SX_ACT_F32 || out_act == SX_ACT_BF16, "unsupported output dtype ", out_act);
    SX_CHECK(aligned(x, 16) && aligned(w->q, 16) && aligned(x_scale, 4) && aligned(w->scale, 4) && aligned(y, act_bytes(out_act)),
             "x and w must be 16-byte aligned, the scales 4-byte, y to its elements");
    const int64_t yb = M * N * act_bytes(out_act);
    SX_CHECK(apart(y, yb, x, M * K) && apart(y, yb, x_scale, M * (K / 128) * 4) && apart(y, yb, w->q, N * K) &&
                 apart(y, yb, w->scale, (N + 127) / 128 * (K / 128) * 4),
             "y overlaps an input");
    const Args a{x, w->q, x_scale, w->scale, y, N, (int32_t)M, (int32_t)K, (int32_t)(K / 128)};
    if (out_act == SX_ACT_F32) launch<float>(a, stream_of(stream));
    else launch<uint16_t>(a, stream_of(stream));
    SX_LAUNCHED("linear_fp8 M=", M, " N=", N, " K=", K);
    return SX_OK;
}
