// The norms around a block with its gate, residual and 8-bit output, one row of K features at a time:
//   h = x / sqrt(mean(x^2) + eps) * (post + w_add)      (over the row or each run of `group` features; post null: h = x)
//   h = h * act(gate)                                   (gate null: left out)
//   r = residual_scale residual + branch_scale h        (with a residual rounded to the activations' type, as the stream keeps it)
//   y = r / sqrt(mean(r^2) + eps) * (pre + w_add)       (pre null: y = r)
// and y as int8 codes with one FP32 scale a row, amax(|y|) / 127: the form sx_linear_int8 takes its activations in.
//
// A row is read once into registers (8 features a 16-byte load) and written from there. A code is a whole number that a border
// decides, so it has to be that of the exact value: all is computed in FP64, which runs at FP32's rate here. Where a product of BF16
// values lies on the border itself, the rounding of x / root decides, so mean, root and quotient are FP64's nearest and the code is
// the formula's in 64 bits, but for silu and sigmoid, which are good to 6e-15 (40 instructions of 744 a wave; with a reciprocal root
// three calls in a hundred, without a residual, had a code on the border's other side). The second norm's root cancels in the codes,
// which come from t = r (pre + w_add) alone. The VALU's work bounds it where there is a gate (2048 rows of 4096, heads of 128: 24.8 us a
// call; a launch by itself 28.2, 0.74 of the VALU's cycles). In FP32 with a bound on what that is off, and FP64 for what the bound
// leaves open (one code in two thousand, the row's largest value), it was as slow: 820 instructions.
#include "common.hpp"

#include <cmath>

namespace sx {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct Args {
    const void *x, *post, *gate, *residual, *pre;
    void *residual_out, *y;
    int8_t *q;
    float *scale;
    int64_t M, ldx, ldg;
    int32_t K, group, post_wrap;  // group: 0, the row; post_wrap: post has that many values
    int32_t gate_act;
    double eps, w_add, rs, bs, over_k, over_group;
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
    for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)v[2 * i], (__bf16)v[2 * i + 1]});
    *reinterpret_cast<u32x4 *>(p) = u;
}

// 1 / (1 + e^-z) of eight values in FP64: e^-|z| as 2^n times the power series of e^r, |r| <= ln(2) / 2, to the eleventh power (6e-15 is
// left), the reciprocal by a Newton step (2^-48 is left of the instruction's 2^-24). The coefficients are held in scalar registers: as
// literals each took two moves a value.
__device__ __forceinline__ double held(double c) {
    asm("" : "+s"(c));
    return c;
}
__device__ __forceinline__ void sigmoid8(const float (&z)[8], double (&s)[8]) {
    const double c[12] = {1.0, 1.0, 0.5, held(1.0 / 6.0), held(1.0 / 24.0), held(1.0 / 120.0), held(1.0 / 720.0), held(1.0 / 5040.0), held(1.0 / 40320.0),
                          held(1.0 / 362880.0), held(1.0 / 3628800.0), held(1.0 / 39916800.0)};
    const double log2e = held(1.4426950408889634), ln2 = held(-0.6931467056274414), rest = held(-4.7493250390316726e-07);  // 21 bits, whose multiples are exact, and the rest
    const double least = held(-800.0);  // e^-800 is 0
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const double y = fmax(-fabs((double)z[k]), least), n = rint(y * log2e), r = fma(n, rest, fma(n, ln2, y));
        double p = fma(c[11], r, c[10]);
#pragma unroll
        for (int i = 9; i >= 0; --i) p = fma(p, r, c[i]);
        const double e = ldexp(p, (int)n), d = 1.0 + e;
        double q = __builtin_amdgcn_rcp(d);
        q = fma(fma(-d, q, 1.0), q, q);
        s[k] = z[k] < 0.f ? e * q : q;
    }
}

// 1 / sqrt(x): the instruction's 2^-24 and two Newton steps (x zero: infinity; no number: none).
__device__ __forceinline__ double over_root(double x) {
    double q = __builtin_amdgcn_rsq(x);
    if (!(q < INFINITY) || q == 0.0) return q;
    const double half = -0.5 * x;
    q = fma(fma(half * q, q, 0.5), q, q);
    return fma(fma(half * q, q, 0.5), q, q);
}

// sqrt(mean + eps), its reciprocal and, for the quotients' correction, its negative (0 where it is infinite: x / infinity is 0).
struct Root {
    double inv, neg;
};
__device__ __forceinline__ Root root_of(double sum, double over, double eps) {
#pragma clang fp contract(off)
    const double mean = sum * over, root = sqrt(mean + eps);  // two roundings, as the formula has them
    return {1.0 / root, root < INFINITY ? -root : 0.0};
}
// x / root: the product's error, computed exactly, put right in one step.
__device__ __forceinline__ double divided(double x, Root r) {
    const double q = x * r.inv;
    return fma(fma(q, r.neg, x), r.inv, q);
}

struct Sum {
    __device__ static double of(double a, double b) { return a + b; }
};
struct Top {
    __device__ static double of(double a, double b) { return a > b ? a : b; }
};

// A lane's value of the same row of 16: neighbours (0xB1), pairs (0x4E), halves and the row mirrored (0x141, 0x140).
template <int CTRL>
__device__ __forceinline__ double across(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}

// Over the group / 8 lanes that hold a run of `group` features.
__device__ __forceinline__ double group_sum(double v, int group) {
    if (group > 8) v += across<0xB1>(v);
    if (group > 16) v += across<0x4E>(v);
    if (group > 32) v += across<0x141>(v);
    if (group > 64) v += across<0x140>(v);
    if (group > 128) v += __shfl_xor(v, 16);
    if (group > 256) v += __shfl_xor(v, 32);
    return v;
}

// Over the TPR threads of a row, in all of them. Every thread of the block calls it.
template <typename Op, int TPR>
__device__ __forceinline__ double row_reduce(double v, double *part) {
    v = Op::of(v, across<0xB1>(v)), v = Op::of(v, across<0x4E>(v));
    v = Op::of(v, across<0x141>(v)), v = Op::of(v, across<0x140>(v));
    v = Op::of(v, __shfl_xor(v, 16)), v = Op::of(v, __shfl_xor(v, 32));
    if constexpr (TPR > 64) {
        const int wave = threadIdx.x >> 6, first = wave / (TPR / 64) * (TPR / 64);
        if ((threadIdx.x & 63) == 0) part[wave] = v;
        __syncthreads();
        v = part[first];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) v = Op::of(v, part[first + i]);
    }
    return v;
}

template <typename T, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) block_norm_kernel(const Args a) {
    constexpr int kRows = TPR < 256 ? 256 / TPR : 1;
    __shared__ double part[3][TPR < 256 ? 4 : TPR / 64];
    const int tid = threadIdx.x % TPR;
    const int64_t m = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
    const bool row = m < a.M;  // whole waves; a row past the last joins the barriers only
    const int n8 = a.K / 8;
    float x[NV][8];
    double h[NV][8];
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = tid + j * TPR;
        const bool on = row && i < n8;
        if (on) load8(static_cast<const T *>(a.x) + m * a.ldx + i * 8, x[j]);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (!on) x[j][k] = 0.f;
            h[j][k] = (double)x[j][k];
        }
    }
    if (a.post != nullptr) {
        Root whole{};
        if (a.group == 0) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int k = 0; k < 8; ++k) ss = fma(h[j][k], h[j][k], ss);
            whole = root_of(row_reduce<Sum, TPR>(ss, part[0]), a.over_k, a.eps);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = tid + j * TPR;
            Root root = whole;
            if (a.group != 0) {
                double sum = 0.0;
#pragma unroll
                for (int k = 0; k < 8; ++k) sum = fma(h[j][k], h[j][k], sum);
                root = root_of(group_sum(sum, a.group), a.over_group, a.eps);
            }
            if (row && i < n8) {
                float w[8];
                load8(static_cast<const T *>(a.post) + (a.post_wrap == a.K ? i * 8 : i * 8 & (a.post_wrap - 1)), w);
#pragma unroll
                for (int k = 0; k < 8; ++k) h[j][k] = divided(h[j][k], root) * (a.w_add == 0.0 ? (double)w[k] : (double)w[k] + a.w_add);
            }
        }
    }
    if (a.gate != nullptr) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = tid + j * TPR;
            if (row && i < n8) {
                float z[8];
                load8(static_cast<const T *>(a.gate) + m * a.ldg + i * 8, z);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (a.gate_act != SX_GATE_SIGMOID) h[j][k] *= (double)z[k];
                if (a.gate_act != SX_GATE_NONE) {
                    double g[8];
                    sigmoid8(z, g);
#pragma unroll
                    for (int k = 0; k < 8; ++k) h[j][k] *= g[k];
                    if (a.gate_act == SX_GATE_SIGMOID) {
#pragma unroll
                        for (int k = 0; k < 8; ++k) h[j][k] = z[k] == z[k] ? h[j][k] : (double)z[k];
                    }
                }
            }
        }
    }
    double s2 = 0.0, top = 0.0;
    double odd = 0.0;  // no number where something is none, or too large for one
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = tid + j * TPR;
        const bool on = row && i < n8;
        if (a.bs != 1.0) {
#pragma unroll
            for (int k = 0; k < 8; ++k) h[j][k] *= a.bs;
        }
        if (on && a.residual != nullptr) {
            float v[8];
            load8(static_cast<const T *>(a.residual) + m * a.K + i * 8, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = as_stored((float)fma(a.rs, (double)v[k], h[j][k]), (const T *)nullptr);
            store8(static_cast<T *>(a.residual_out) + m * a.K + i * 8, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) h[j][k] = (double)v[k];
        }
        if (a.pre != nullptr) {
            float w[8] = {};
            if (on) load8(static_cast<const T *>(a.pre) + i * 8, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                s2 = fma(h[j][k], h[j][k], s2);
                h[j][k] *= (double)w[k] + a.w_add;
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmax(top, fabs(h[j][k])), odd = fma(h[j][k], 0.0, odd);
    }
    double inv = 1.0;
    if (a.pre != nullptr) inv = over_root(fma(row_reduce<Sum, TPR>(s2, part[1]), a.over_k, a.eps));
    if (a.q != nullptr) top = row_reduce<Top, TPR>(odd == 0.0 ? top : INFINITY, part[2]);
    const bool fine = top < INFINITY;
    const double mul = 127.0 / top;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int i = tid + j * TPR;
        if (!row || i >= n8) continue;
        if (a.y != nullptr) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = (float)(a.pre != nullptr ? h[j][k] * inv : h[j][k]);
            store8(static_cast<T *>(a.y) + m * a.K + i * 8, v);
        }
        if (a.q == nullptr) continue;
        uint32_t o[2] = {0u, 0u};
        if (fine && top > 0.0) {
            double n[8];
            double far = 0.0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const double c = h[j][k] * mul;
                n[k] = rint(c);
                far = fmax(far, fabs(c - n[k]));
            }
            if (far > 0.5 - 1e-9) {  // beside a border the quotient itself says which side, and a tie that it is one
#pragma unroll
                for (int k = 0; k < 8; ++k) n[k] = rint(h[j][k] * 127.0 / top);
            }
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
                const uint32_t lo = __builtin_amdgcn_perm((uint32_t)(int)n[k + 1], (uint32_t)(int)n[k], 0x0C0C0400);
                const uint32_t hi = __builtin_amdgcn_perm((uint32_t)(int)n[k + 3], (uint32_t)(int)n[k + 2], 0x04000C0C);
                o[k / 4] = lo | hi;
            }
        }
        *reinterpret_cast<uint2 *>(a.q + m * a.K + i * 8) = uint2{o[0], o[1]};
        if (i == 0) a.scale[m] = fine ? (float)(top * inv / 127.0) : qnan();
    }
}

template <typename T, int TPR, int NV>
void go(const Args &a, hipStream_t s) {
    constexpr int rows = TPR < 256 ? 256 / TPR : 1;
    block_norm_kernel<T, TPR, NV><<<(unsigned)((a.M + rows - 1) / rows), TPR < 256 ? 256 : TPR, 0, s>>>(a);
}

// One run of 8 a thread, so that a row's loads are all in flight at once, up to 8192 features; rows of few features share a block.
template <typename T>
void launch(const Args &a, hipStream_t s) {
    const int n8 = a.K / 8;
    if (n8 <= 64) go<T, 64, 1>(a, s);
    else if (n8 <= 128) go<T, 128, 1>(a, s);
    else if (n8 <= 256) go<T, 256, 1>(a, s);
    else if (n8 <= 512) go<T, 512, 1>(a, s);
    else if (n8 <= 1024) go<T, 1024, 1>(a, s);
    else go<T, 1024, 2>(a, s);
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" int sx_block_norm_int8(const sx_block_norm *p, int64_t M, int64_t K, int act, sx_stream stream) {
    SX_CHECK(p != nullptr && p->x != nullptr, "null pointer");
    const sx_block_norm &n = *p;
    SX_CHECK(n.q != nullptr || n.y != nullptr || n.residual_out != nullptr, "no output: q, y and residual_out are null");
    SX_CHECK((n.q == nullptr) == (n.scale == nullptr), "q and scale go together");
    SX_CHECK((n.residual == nullptr) == (n.residual_out == nullptr), "residual and residual_out go together");
    SX_CHECK(act == SX_ACT_F32 || act == SX_ACT_BF16, "unsupported activation dtype ", act);
    SX_CHECK(M >= 1 && M <= 0x7fffffff, "M = ", M);
    SX_CHECK(K >= 8 && K % 8 == 0 && K <= 16384, "K = ", K, ", expected a multiple of 8, 8..16384");
    SX_CHECK(n.ldx >= K && n.ldx % 8 == 0, "ldx = ", n.ldx, ", expected a multiple of 8, >= K = ", K);
    SX_CHECK(n.gate == nullptr || ((n.ld_gate == 0 || n.ld_gate >= K) && n.ld_gate % 8 == 0), "ld_gate = ", n.ld_gate, ", expected 0 or a multiple of 8, >= K = ", K);
    SX_CHECK(n.gate == nullptr || (n.gate_act >= SX_GATE_NONE && n.gate_act <= SX_GATE_SIGMOID), "unsupported gate activation ", n.gate_act);
    const int64_t g = n.group;
    SX_CHECK(g == 0 || g == K || (g >= 8 && g <= 512 && (g & (g - 1)) == 0 && K % g == 0), "group = ", g, ", expected 0, K or a power of two, 8..512, that divides K = ", K);
    SX_CHECK(n.post_len == 0 || n.post_len == K || n.post_len == g, "post_len = ", n.post_len, ", expected K or the group");
    SX_CHECK(std::isfinite(n.eps) && n.eps >= 0.0 && std::isfinite(n.w_add) && std::isfinite(n.residual_scale) && std::isfinite(n.branch_scale),
             "eps = ", n.eps, ", w_add = ", n.w_add, ", residual_scale = ", n.residual_scale, ", branch_scale = ", n.branch_scale);
    SX_CHECK(aligned(n.x, 16) && aligned(n.post, 16) && aligned(n.gate, 16) && aligned(n.residual, 16) && aligned(n.pre, 16) && aligned(n.residual_out, 16) &&
                 aligned(n.y, 16) && aligned(n.q, 8) && aligned(n.scale, 4),
             "activations and weights must be 16-byte, q 8-byte and scale 4-byte aligned");
    const int64_t e = act_bytes(act), xb = ((M - 1) * n.ldx + K) * e, rb = M * K * e, gb = ((M - 1) * n.ld_gate + K) * e, wb = K * e;
    const int64_t pb = (n.post_len != 0 ? n.post_len : K) * e;
    struct Span {
        const void *p;
        int64_t n;
        bool rows;  // [M, K] dense: a row is read whole before it is written, so an output may be it
    };
    const Span in[5] = {{n.x, xb, n.ldx == K}, {n.residual, rb, true}, {n.gate, gb, n.ld_gate == K}, {n.post, pb, false}, {n.pre, wb, false}};
    const Span outs[4] = {{n.residual_out, rb, true}, {n.y, rb, true}, {n.q, M * K, false}, {n.scale, M * 4, false}};
    for (int o = 0; o < 4; ++o) {
        if (outs[o].p == nullptr) continue;
        for (const Span &i : in)
            SX_CHECK(i.p == nullptr || (i.p == outs[o].p && i.rows && outs[o].rows) || apart(i.p, i.n, outs[o].p, outs[o].n), "output ", o, " overlaps an input at other rows");
        for (int k = 0; k < o; ++k) SX_CHECK(outs[k].p == nullptr || apart(outs[k].p, outs[k].n, outs[o].p, outs[o].n), "outputs ", k, " and ", o, " overlap");
    }
    const Args a{n.x, n.post, n.gate, n.residual, n.pre, n.residual_out, n.y, n.q, n.scale, M, n.ldx, n.ld_gate, (int32_t)K, (int32_t)(g == K ? 0 : g),
                 (int32_t)(n.post_len != 0 ? n.post_len : K), n.gate_act, n.eps, n.w_add, n.residual_scale, n.branch_scale,
                 1.0 / (double)K, g == 0 ? 0.0 : 1.0 / (double)g};
    if (act == SX_ACT_F32) launch<float>(a, stream_of(stream));
    else launch<uint16_t>(a, stream_of(stream));
    SX_LAUNCHED("block_norm_int8 M=", M, " K=", K);
    return SX_OK;
}
