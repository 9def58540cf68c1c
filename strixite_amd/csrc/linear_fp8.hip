// FP8 linear with a scale for each block of 128: y[m, n] = sum_b sx[m, b] * sw[n / 128, b] * sum_{k in block b} x[m, k]
// w[n, k], x and w e4m3 codes, the scales FP32, sums over the blocks in FP32, one rounding at the store.
//
// One v_mfma_f32_16x16x128_f8f6f4 is exactly one block of 16 rows x 16 tokens: its result is scaled by sx * sw as it
// is added to the running sum (four FMAs for 32768 products). W is the A operand and x the B operand, so a lane holds
// one token (its sx) and four weight rows, and 16 rows of W share one sw.
#include "common.hpp"

#include <algorithm>

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
    bool by16;         // rows of y are whole 16-byte pieces
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

// A block's products of 16 rows and 16 tokens. The FP8 instruction keeps fewer bits than FP32: the products of eight
// neighbouring codes are cut, toward zero, at 2^-13 of the largest one's power of two (2^(ex + ew), codes under 2^-6 counted
// as 2^-6), so a block is off by 2^-10 of its sum of |products| at most, by 1.4e-5 of its result (root mean square) on random
// codes: a hundredth of a BF16 output's rounding there, but more where large products cancel, and far over an FP32 output's
// rounding. FP32 outputs take the codes as BF16, exact there, whose products are summed in FP32 (half the rate: a K block
// of the tiles takes 1.5 to 1.6 times as long; these are logits of few tokens, bound by the weight's bytes).
template <bool F32>
__device__ __forceinline__ f32x4 block_products(i32x8 a, i32x8 b) {
    f32x4 d = {0.f, 0.f, 0.f, 0.f};
    if constexpr (!F32) {
        d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, d, 0, 0, 0, 0x7F7F7F7F, 0, 0x7F7F7F7F);  // scales of one
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a[i], a[i + 1]), as_bf16x8(b[i], b[i + 1]), d, 0, 0, 0);
    }
    return d;
}

// ---------------- few tokens: the weight's bytes are the cost ----------------
// A block takes 16 NT weight rows and 16 MT tokens; its 8 waves split K block by block, straight from memory into the
// operands, and their sums meet in LDS in wave order. 12288 x 4096, M = 6: 14.0 us, 3.6 TB/s with the launch.
__device__ __forceinline__ void store4(float *p, f32x4 v) { *reinterpret_cast<f32x4 *>(p) = v; }
__device__ __forceinline__ void store4(uint16_t *p, f32x4 v) {
    *reinterpret_cast<uint2 *>(p) = uint2{f32_to_bf16(v[0]) | (f32_to_bf16(v[1]) << 16), f32_to_bf16(v[2]) | (f32_to_bf16(v[3]) << 16)};
}

constexpr int kRowWaves = 8;

template <typename TY, int NT, int MT>
__global__ void __launch_bounds__(64 * kRowWaves) fp8_rows_kernel(const Args a) {
    constexpr bool F32 = sizeof(TY) == 4;
    __shared__ f32x4 part[kRowWaves][NT][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16 * NT;
    const int m0 = blockIdx.y * 16 * MT;
    const uint8_t *w[NT], *x[MT];
    const float *xs[MT], *ws = a.ws + n0 / 128 * a.kb;  // the block's rows lie in one row of tiles
#pragma unroll
    for (int r = 0; r < NT; ++r) w[r] = a.w + min(n0 + r * 16 + n16, a.N - 1) * a.K + g * 32;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t m = min(m0 + t * 16 + n16, a.M - 1);
        x[t] = a.x + m * a.K + g * 32, xs[t] = a.xs + m * a.kb;
    }
    f32x4 acc[NT][MT];
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // kAhead K blocks of this wave at a time, all requested before the first is used (past the end the last one again,
    // not used)
    constexpr int kAhead = NT == 1 && MT <= 2 ? 4 : 2;
    for (int b0 = wave; b0 < a.kb; b0 += kRowWaves * kAhead) {
        i32x8 A[kAhead][NT];
        float sw[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int at = min(b0 + j * kRowWaves, a.kb - 1);
#pragma unroll
            for (int r = 0; r < NT; ++r) A[j][r] = load32(w[r] + at * 128);
            sw[j] = ws[at];
        }
        i32x8 B[kAhead][MT];
        float sx[kAhead][MT];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int at = min(b0 + j * kRowWaves, a.kb - 1);
                B[j][t] = load32(x[t] + at * 128), sx[j][t] = xs[t][at];
            }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (b0 + j * kRowWaves < a.kb) {
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int r = 0; r < NT; ++r) {
                        const f32x4 d = block_products<F32>(A[j][r], B[j][t]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[r][t][i] = fmaf(d[i], sw[j] * sx[j][t], acc[r][t][i]);
                    }
            }
    }
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) part[wave][r][t][lane] = acc[r][t];
    __syncthreads();
    const float *p = reinterpret_cast<const float *>(part);
    TY *y = static_cast<TY *>(a.y);
    for (int i = threadIdx.x; i < NT * MT * 256; i += 64 * kRowWaves) {
        const int n = i % (16 * NT), m = i / (16 * NT);  // lane (m % 16) + 16 (n % 16 / 4), value n % 4
        const int at = (((n >> 4) * MT + (m >> 4)) * 64 + (m & 15) + 16 * ((n & 15) >> 2)) * 4 + (n & 3);
        float sum = 0.f;
#pragma unroll
        for (int v = 0; v < kRowWaves; ++v) sum += p[v * NT * MT * 256 + at];
        if (m0 + m < a.M && n0 + n < a.N) store_act(y, (m0 + m) * a.N + n0 + n, sum);
    }
}

// ---------------- many tokens: the products are the cost ----------------
// A block takes BN weight rows and BM tokens. A K block of both (128 bytes a row) is a stage in LDS, two deep; the one
// after next is already in registers or on its way there, so a load has two K blocks' time to arrive. (Loads straight into
// LDS, one or two blocks ahead, measured 2-10 % slower.) A 16-byte chunk c of row r lies at c ^ (r & 7), so that the
// operand reads of 16 rows spread over all banks. Eight waves, two a SIMD (one's scaling FMAs beside the other's
// products): four along the rows, two along the tokens. Whatever the staging's depth, a compute unit took in 40 bytes a
// nanosecond, so the time a product falls with the tile's size. 7680 x 2560, M = 1531: no unit is full (counters: MFMA 0.31, VALU
// 0.37 and LDS 0.27 of their cycles, L2 hits 0.81); the waves wait 0.37 of their time, and 0.31 to issue.
constexpr int kTileWaves = 8, kWn = 4, kWm = 2;

template <typename TY, int BN, int BM>
__global__ void __launch_bounds__(64 * kTileWaves) fp8_tiles_kernel(const Args a, int m_tiles, int tiles) {
    constexpr bool F32 = sizeof(TY) == 4;
    constexpr int NT = BN / kWn / 16, MT = BM / kWm / 16, kScales = BM + 64;
    constexpr int kLoadW = BN / 8 / kTileWaves, kLoadX = BM / 8 / kTileWaves;  // 8 rows a load
    static_assert(BN % 128 == 0 && kLoadX * 8 * kTileWaves == BM && BM / 64 < kTileWaves);
    __shared__ __attribute__((aligned(16))) uint8_t w0[BN * 128], w1[BN * 128], x0[BM * 128], x1[BM * 128];
    __shared__ float s0[kScales], s1[kScales];  // sx of the tokens, then sw of the row tiles
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g = lane >> 4;
    const int wn = wave % kWn, wm = wave / kWn;
    // Block i runs on XCD i % 8: each XCD takes a run of the tiles, all token tiles of a row tile together, so that its
    // L2 reads a row tile's weights once.
    const int per = (tiles + 7) / 8, tile = (blockIdx.x % 8) * per + blockIdx.x / 8;
    if (tile >= tiles) return;
    const int64_t n0 = (int64_t)(tile / m_tiles) * BN;
    const int m0 = tile % m_tiles * BM;

    const int r8 = lane >> 3, chunk = ((lane & 7) ^ r8) * 16;
    // a tile's rows span at most 256 x 65,536 bytes: one uniform base each and 32-bit offsets
    const uint8_t *wbase = a.w + n0 * a.K, *xbase = a.x + (int64_t)m0 * a.K;
    const int wrows = (int)min<int64_t>(a.N - n0, BN), xrows = min(a.M - m0, BM);
    uint32_t wo[kLoadW], xo[kLoadX];
#pragma unroll
    for (int i = 0; i < kLoadW; ++i) wo[i] = (uint32_t)(min((wave * kLoadW + i) * 8 + r8, wrows - 1) * a.K + chunk);
#pragma unroll
    for (int i = 0; i < kLoadX; ++i) xo[i] = (uint32_t)(min((wave * kLoadX + i) * 8 + r8, xrows - 1) * a.K + chunk);
    // waves 0 .. BM / 64 - 1 bring the tokens' scales, the next one the row tiles'
    const float *sp = wave < BM / 64 ? a.xs + (int64_t)min(m0 + wave * 64 + lane, a.M - 1) * a.kb
                                     : a.ws + min(n0 / 128 + min(lane, BN / 128 - 1), (a.N - 1) / 128) * a.kb;
    i32x4 rw[kLoadW], rx[kLoadX];
    float rs = 0.f;
    auto fetch = [&](int b) __attribute__((always_inline)) {  // past the end: the last block again, not used
        const int at = min(b, a.kb - 1);
#pragma unroll
        for (int i = 0; i < kLoadW; ++i) rw[i] = *reinterpret_cast<const i32x4 *>(wbase + at * 128 + wo[i]);
#pragma unroll
        for (int i = 0; i < kLoadX; ++i) rx[i] = *reinterpret_cast<const i32x4 *>(xbase + at * 128 + xo[i]);
        if (wave <= BM / 64) rs = sp[at];
    };
    auto put = [&](uint8_t *wb, uint8_t *xb, float *sb) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kLoadW; ++i) *reinterpret_cast<i32x4 *>(wb + (wave * kLoadW + i) * 1024 + lane * 16) = rw[i];
#pragma unroll
        for (int i = 0; i < kLoadX; ++i) *reinterpret_cast<i32x4 *>(xb + (wave * kLoadX + i) * 1024 + lane * 16) = rx[i];
        if (wave <= BM / 64) sb[wave * 64 + lane] = rs;
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // lane group g's codes of a block: chunks g and g + 4 (of x and w alike). With chunks 2 g and 2 g + 1 the lanes that a
    // 16-byte read serves together met in pairs on the same banks (46 % of the LDS cycles).
    const int c0 = (g ^ (n16 & 7)) * 16, c1 = ((g + 4) ^ (n16 & 7)) * 16;
    auto operand = [&](const uint8_t *row) __attribute__((always_inline)) {
        const i32x4 p = *reinterpret_cast<const i32x4 *>(row + c0), q = *reinterpret_cast<const i32x4 *>(row + c1);
        return i32x8{p[0], p[1], p[2], p[3], q[0], q[1], q[2], q[3]};
    };
    // A product is scaled and added while the two after it run, and the next token tile's operand is read meanwhile.
    auto multiply = [&](const uint8_t *wb, const uint8_t *xb, const float *sb) __attribute__((always_inline)) {
        const uint8_t *wrow = wb + (wn * (BN / kWn) + n16) * 128, *xrow = xb + (wm * (BM / kWm) + n16) * 128;
        const float *srow = sb + wm * (BM / kWm) + n16;
        i32x8 A[NT], B[2];
        float scale[2];
        f32x4 d[3];
        B[0] = operand(xrow);
#pragma unroll
        for (int r = 0; r < NT; ++r) A[r] = operand(wrow + r * 2048);
        const float sw = sb[BM + wn * (BN / kWn) / 128];
        scale[0] = srow[0] * sw;
#pragma unroll
        for (int i = 0; i < NT * MT + 2; ++i) {
            const int t = i / NT, r = i % NT;
            if (r == 0 && t + 1 < MT) B[(t + 1) & 1] = operand(xrow + (t + 1) * 2048);
            if (i < NT * MT) d[i % 3] = block_products<F32>(A[r], B[t & 1]);
            if (i >= 2) {
                const int pt = (i - 2) / NT, pr = (i - 2) % NT;
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[pr][pt][j] = fmaf(d[(i - 2) % 3][j], scale[pt & 1], acc[pr][pt][j]);
            }
            if (r == NT - 1 && t + 1 < MT) scale[(t + 1) & 1] = srow[(t + 1) * 16] * sw;
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // The barrier at the top of a K block makes the block's stage visible and says that the stage before has been read;
    // that one takes the next block from the registers, which the block after it is fetched into.
    auto step = [&](int b, const uint8_t *wb, const uint8_t *xb, const float *sb, uint8_t *wn_, uint8_t *xn_, float *sn_) __attribute__((always_inline)) {
        lds_barrier();
        put(wn_, xn_, sn_);
        fetch(b + 2);
        multiply(wb, xb, sb);
    };
    fetch(0);
    put(w0, x0, s0);
    fetch(1);
    for (int b = 0; b < a.kb; b += 2) {
        step(b, w0, x0, s0, w1, x1, s1);
        if (b + 1 < a.kb) step(b + 1, w1, x1, s1, w0, x0, s0);
    }
    // A lane holds rows 4 g .. 4 g + 3 of each row tile for one token: 8 or 16 bytes of the output's row. 16 tokens at a
    // time go through the wave's own piece of LDS and leave as whole lines (straight from the lanes 512 x 4096 took 5 us
    // longer).
    constexpr int kRowBytes = NT * 16 * (int)sizeof(TY), kPitch = kRowBytes + (F32 ? 0 : 16), kLanes = kRowBytes / 16, kPass = 64 / kLanes;
    static_assert(kTileWaves * 16 * kPitch <= BN * 128);
    __syncthreads();  // every wave has read the last block
    uint8_t *piece = w0 + wave * 16 * kPitch;
    TY *y = static_cast<TY *>(a.y);
    const int64_t n = n0 + wn * (BN / kWn) + (lane % kLanes) * (16 / (int)sizeof(TY));
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int r = 0; r < NT; ++r) store4(reinterpret_cast<TY *>(piece + n16 * kPitch) + r * 16 + 4 * g, acc[r][t]);
        // one wave's LDS accesses take effect in program order: these reads follow the writes above
#pragma unroll
        for (int j = 0; j < 16; j += kPass) {
            const int row = j + lane / kLanes;
            const int64_t m = m0 + wm * (BM / kWm) + t * 16 + row;
            const u32x4 v = *reinterpret_cast<const u32x4 *>(piece + row * kPitch + (lane % kLanes) * 16);
            if (m >= a.M || n >= a.N) continue;
            if (a.by16) {
                *reinterpret_cast<u32x4 *>(y + m * a.N + n) = v;
            } else {
                constexpr int kEach = 16 / (int)sizeof(TY);
#pragma unroll
                for (int i = 0; i < kEach; ++i)
                    if (n + i < a.N) {
                        if constexpr (F32) y[m * a.N + n + i] = __uint_as_float(v[i]);
                        else y[m * a.N + n + i] = (uint16_t)(v[i / 2] >> (16 * (i & 1)));
                    }
            }
        }
    }
}

template <typename TY, int BN, int BM>
void launch_tiles(const Args &a, hipStream_t s) {
    const int m_tiles = (a.M + BM - 1) / BM;
    const int64_t tiles = (a.N + BN - 1) / BN * m_tiles;
    fp8_tiles_kernel<TY, BN, BM><<<(unsigned)((tiles + 7) / 8 * 8), 64 * kTileWaves, 0, s>>>(a, m_tiles, (int)tiles);
}

template <typename TY, int NT, int MT>
void launch_rows(const Args &a, hipStream_t s) {
    const dim3 grid((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
    fp8_rows_kernel<TY, NT, MT><<<grid, 64 * kRowWaves, 0, s>>>(a);
}

// Up to 16 tokens: 16 weight rows a block, whose waves read nothing twice. Up to 32, and up to 64 where two passes still
// are at most two blocks a compute unit: 32 rows x 32 tokens a block (M = 24: 8192 x 2560 8.7 us, 15.7 on the smallest
// tile; M = 48: 4096 x 4096 12.4 / 17.7, 12288 x 4096 past that limit 28.5 / 25.0). Above, the tile with the least
// rounds of blocks over the compute units times the time of a K block, measured with the chip full: 0.48, 0.87, 1.37 and
// 1.75 us for 128 x 64, 128 x 128, 256 x 128 and 256 x 192 (rows x tokens); 0.72, 1.4 and 2.2 us with FP32 outputs, whose
// 256 x 192 does not fit the registers. 12288 x 4096 in us for the four tiles: M = 256 36.2 / 33.5 / 47.1 / 59.1, 512
// 55.4 / 61.6 / 47.9 / 61.0; 7680 x 2560 M = 1531 59.6 / 58.8 / 61.9 / 43.4.
template <typename TY>
void launch(const Args &a, hipStream_t s) {
    constexpr bool F32 = sizeof(TY) == 4;
    const int64_t cus = device_cus();
    if (a.M <= 16) return launch_rows<TY, 1, 1>(a, s);
    if (a.M <= 32 || (a.M <= 64 && (a.N + 31) / 32 * 2 <= 2 * cus)) return launch_rows<TY, 2, 2>(a, s);
    auto cost = [&](int bn, int bm, double each) {
        const int64_t tiles = (a.N + bn - 1) / bn * ((a.M + bm - 1) / bm);
        return (double)((tiles + cus - 1) / cus) * each;
    };
    const double c[4] = {cost(128, 64, F32 ? 0.72 : 0.48), cost(128, 128, F32 ? 1.4 : 0.87), cost(256, 128, F32 ? 2.2 : 1.37),
                         cost(256, 192, 1.75)};
    switch ((int)(std::min_element(c, c + (F32 ? 3 : 4)) - c)) {
    case 0: return launch_tiles<TY, 128, 64>(a, s);
    case 1: return launch_tiles<TY, 128, 128>(a, s);
    case 2: return launch_tiles<TY, 256, 128>(a, s);
    default:
        if constexpr (!F32) return launch_tiles<TY, 256, 192>(a, s);
    }
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
    SX_CHECK(M >= 1 && M <= 1 << 22, "M = ", M, ", expected 1..", 1 << 22);
    SX_CHECK((N + 127) / 128 * ((M + 63) / 64) <= 0x7ffffff0, "N = ", N, " with M = ", M, ": too many tiles");
    SX_CHECK(out_act == SX_ACT_F32 || out_act == SX_ACT_BF16, "unsupported output dtype ", out_act);
    SX_CHECK(aligned(x, 16) && aligned(w->q, 16) && aligned(x_scale, 4) && aligned(w->scale, 4) && aligned(y, act_bytes(out_act)),
             "x and w must be 16-byte aligned, the scales 4-byte, y to its elements");
    const int64_t yb = M * N * act_bytes(out_act);
    SX_CHECK(apart(y, yb, x, M * K) && apart(y, yb, x_scale, M * (K / 128) * 4) && apart(y, yb, w->q, N * K) &&
                 apart(y, yb, w->scale, (N + 127) / 128 * (K / 128) * 4),
             "y overlaps an input");
    const Args a{x, w->q, x_scale, w->scale, y, N, (int32_t)M, (int32_t)K, (int32_t)(K / 128), N * act_bytes(out_act) % 16 == 0 && aligned(y, 16)};
    if (out_act == SX_ACT_F32) launch<float>(a, stream_of(stream));
    else launch<uint16_t>(a, stream_of(stream));
    SX_LAUNCHED("linear_fp8 M=", M, " N=", N, " K=", K);
    return SX_OK;
}
