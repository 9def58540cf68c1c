// Linear in 8-bit integers with a scale for each token and channel: y[m, n] = sx[m] * sw[n] * sum_k x[m, k] w[n, k], x and w
// int8 codes, the sum in 32-bit integers (exact: K is at most 131056, 128 * 128 * K under 2^31), then two FP32 products and one
// rounding at the store.
//
// One v_mfma_i32_16x16x64_i8 takes 16 rows x 16 tokens x 64 codes and adds to its accumulator, so nothing happens between the
// products of a row. W is the A operand and x the B operand: a lane holds one token and four weight rows of a tile. K is gone
// through in blocks of 128 codes (a line of memory a row); which 16 of a block a lane group brings is free as long as x and w
// agree. A last block that is not full takes zeros for w.
#include "common.hpp"

#include <algorithm>

namespace sx {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Args {
    const int8_t *x, *w;
    const float *xs, *ws;
    void *y;
    int64_t N;
    int32_t M, K, kb;  // kb = ceil(K / 128)
    bool by16;         // rows of y are whole 16-byte pieces
};

__device__ __forceinline__ i32x4 load16(const int8_t *p) { return *reinterpret_cast<const i32x4 *>(p); }
__device__ __forceinline__ i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }

__device__ __forceinline__ void store4(float *p, f32x4 v) { *reinterpret_cast<f32x4 *>(p) = v; }
__device__ __forceinline__ void store4(uint16_t *p, f32x4 v) {
    *reinterpret_cast<uint2 *>(p) = uint2{f32_to_bf16(v[0]) | (f32_to_bf16(v[1]) << 16), f32_to_bf16(v[2]) | (f32_to_bf16(v[3]) << 16)};
}

// ---------------- few tokens: the weight's bytes are the cost ----------------
// A block takes 16 NT weight rows and 16 MT tokens; its 8 waves split K block by block, straight from memory into the
// operands, and their sums meet in LDS.
constexpr int kRowWaves = 8;

template <typename TY, int NT, int MT>
__global__ void __launch_bounds__(64 * kRowWaves) int8_rows_kernel(const Args a) {
    __shared__ i32x4 part[kRowWaves][NT][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16 * NT;
    const int m0 = blockIdx.y * 16 * MT;
    const int8_t *w[NT], *x[MT];
#pragma unroll
    for (int r = 0; r < NT; ++r) w[r] = a.w + min(n0 + r * 16 + n16, a.N - 1) * a.K;
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = a.x + (int64_t)min(m0 + t * 16 + n16, a.M - 1) * a.K;
    i32x4 acc[NT][MT];
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[r][t] = i32x4{0, 0, 0, 0};
    // kAhead K blocks of this wave at a time, all requested before the first is used (past the end zeros meet the last codes)
    constexpr int kAhead = NT == 1 && MT <= 2 ? 4 : 2;
    const i32x4 none = {0, 0, 0, 0};
    for (int b0 = wave; b0 < a.kb; b0 += kRowWaves * kAhead) {
        i32x4 A[kAhead][NT][2], B[kAhead][MT][2];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int in = min((b0 + j * kRowWaves) * 128 + c * 64 + g * 16, a.K - 16);
#pragma unroll
                for (int r = 0; r < NT; ++r) A[j][r][c] = load16(w[r] + in);
            }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int in = min((b0 + j * kRowWaves) * 128 + c * 64 + g * 16, a.K - 16);
#pragma unroll
                for (int t = 0; t < MT; ++t) B[j][t][c] = load16(x[t] + in);
            }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const bool past = (b0 + j * kRowWaves) * 128 + c * 64 + g * 16 >= a.K;  // asked here: at the loads it would wait for them
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int r = 0; r < NT; ++r) acc[r][t] = mfma(past ? none : A[j][r][c], B[j][t][c], acc[r][t]);
            }
    }
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) part[wave][r][t][lane] = acc[r][t];
    __syncthreads();
    const int *p = reinterpret_cast<const int *>(part);
    TY *y = static_cast<TY *>(a.y);
    for (int i = threadIdx.x; i < NT * MT * 256; i += 64 * kRowWaves) {
        const int n = i % (16 * NT), m = i / (16 * NT);  // lane (m % 16) + 16 (n % 16 / 4), value n % 4
        const int at = (((n >> 4) * MT + (m >> 4)) * 64 + (m & 15) + 16 * ((n & 15) >> 2)) * 4 + (n & 3);
        int sum = 0;
#pragma unroll
        for (int v = 0; v < kRowWaves; ++v) sum += p[v * NT * MT * 256 + at];
        if (m0 + m < a.M && n0 + n < a.N) store_act(y, (m0 + m) * a.N + n0 + n, (float)sum * a.xs[m0 + m] * a.ws[n0 + n]);
    }
}

// ---------------- many tokens: the products are the cost ----------------
// A block takes BN weight rows and BM tokens. A K block of both (128 bytes a row) is a stage in LDS, two deep; the one
// after next is already in registers or on its way there, so a load has two K blocks' time to arrive. A 16-byte chunk c of
// row r lies at c ^ (r & 7), so that the operand reads of 16 rows spread over all banks. Eight waves, two a SIMD: four along
// the rows, two along the tokens.
constexpr int kTileWaves = 8, kWn = 4, kWm = 2;

template <typename TY, int BN, int BM>
__global__ void __launch_bounds__(64 * kTileWaves) int8_tiles_kernel(const Args a, int m_tiles, int tiles) {
    constexpr bool F32 = sizeof(TY) == 4;
    constexpr int NT = BN / kWn / 16, MT = BM / kWm / 16;
    constexpr int kLoadW = BN / 8 / kTileWaves, kLoadX = BM / 8 / kTileWaves;  // 8 rows a load
    static_assert(kLoadW * 8 * kTileWaves == BN && kLoadX * 8 * kTileWaves == BM);
    __shared__ __attribute__((aligned(16))) uint8_t w0[BN * 128], w1[BN * 128], x0[BM * 128], x1[BM * 128];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g = lane >> 4;
    const int wn = wave % kWn, wm = wave / kWn;
    // Block i runs on XCD i % 8: each XCD takes a run of the tiles, all token tiles of a row tile together, so that its
    // L2 reads a row tile's weights once.
    const int per = (tiles + 7) / 8, tile = (blockIdx.x % 8) * per + blockIdx.x / 8;
    if (tile >= tiles) return;
    const int64_t n0 = (int64_t)(tile / m_tiles) * BN;
    const int m0 = tile % m_tiles * BM;

    const int r8 = lane >> 3, chunk = ((lane & 7) ^ r8) * 16;
    // a tile's rows span at most 384 x 131,056 bytes: one uniform base each and 32-bit offsets
    const int8_t *wbase = a.w + n0 * a.K, *xbase = a.x + (int64_t)m0 * a.K;
    const int wrows = (int)min<int64_t>(a.N - n0, BN), xrows = min(a.M - m0, BM);
    uint32_t wo[kLoadW], xo[kLoadX];
#pragma unroll
    for (int i = 0; i < kLoadW; ++i) wo[i] = (uint32_t)(min((wave * kLoadW + i) * 8 + r8, wrows - 1) * a.K);
#pragma unroll
    for (int i = 0; i < kLoadX; ++i) xo[i] = (uint32_t)(min((wave * kLoadX + i) * 8 + r8, xrows - 1) * a.K);
    i32x4 rw[kLoadW], rx[kLoadX];
    const i32x4 none = {0, 0, 0, 0};
    auto fetch = [&](int b) __attribute__((always_inline)) {  // past the end: the last codes again
        const int in = min(min(b, a.kb - 1) * 128 + chunk, a.K - 16);
#pragma unroll
        for (int i = 0; i < kLoadW; ++i) rw[i] = load16(wbase + wo[i] + in);
#pragma unroll
        for (int i = 0; i < kLoadX; ++i) rx[i] = load16(xbase + xo[i] + in);
    };
    // Block b in the registers: zeros for w past the end of K (at the loads they would wait for them).
    auto clear_past = [&](int b) __attribute__((always_inline)) {
        if (b * 128 + 128 > a.K && b * 128 + chunk >= a.K) {
#pragma unroll
            for (int i = 0; i < kLoadW; ++i) rw[i] = none;
        }
    };
    auto put = [&](int b, uint8_t *wb, uint8_t *xb) __attribute__((always_inline)) {
        clear_past(b);
#pragma unroll
        for (int i = 0; i < kLoadW; ++i) *reinterpret_cast<i32x4 *>(wb + (wave * kLoadW + i) * 1024 + lane * 16) = rw[i];
#pragma unroll
        for (int i = 0; i < kLoadX; ++i) *reinterpret_cast<i32x4 *>(xb + (wave * kLoadX + i) * 1024 + lane * 16) = rx[i];
    };
    i32x4 acc[NT][MT];
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[r][t] = none;
    auto multiply = [&](const uint8_t *wb, const uint8_t *xb) __attribute__((always_inline)) {
        const uint8_t *wrow = wb + (wn * (BN / kWn) + n16) * 128, *xrow = xb + (wm * (BM / kWm) + n16) * 128;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int at = ((g + 4 * c) ^ (n16 & 7)) * 16;
            i32x4 A[NT], B[MT];
#pragma unroll
            for (int r = 0; r < NT; ++r) A[r] = *reinterpret_cast<const i32x4 *>(wrow + r * 2048 + at);
#pragma unroll
            for (int t = 0; t < MT; ++t) B[t] = *reinterpret_cast<const i32x4 *>(xrow + t * 2048 + at);
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int r = 0; r < NT; ++r) acc[r][t] = mfma(A[r], B[t], acc[r][t]);
        }
    };
    // The barrier at the top of a K block makes the block's stage visible and says that the stage before has been read; that one takes
    // the next block from the registers, which the block after it is then fetched into. kSpread: operands are read, and the next
    // block's pieces moved and requested, between the products (sched_barrier holds them there): 256 x 192 1.42 -> 1.28 us a K block
    // with one round of 32; 384 x 192 has no registers left for it, the smaller tiles gain nothing.
    constexpr bool kSpread = BN == 256;
    constexpr int kPieces = kLoadW + kLoadX, kSlots = 2 * MT, kEach = (kPieces + kSlots - 1) / kSlots, kA = (NT + MT - 1) / MT;
    auto spread_step = [&](int b, const uint8_t *wb, const uint8_t *xb, uint8_t *wn_, uint8_t *xn_) __attribute__((always_inline)) {
        const uint8_t *wrow = wb + (wn * (BN / kWn) + n16) * 128, *xrow = xb + (wm * (BM / kWm) + n16) * 128;
        const int at[2] = {(g ^ (n16 & 7)) * 16, ((g + 4) ^ (n16 & 7)) * 16};
        const int off = min(min(b + 2, a.kb - 1) * 128 + chunk, a.K - 16);  // past the end: the last codes again
        clear_past(b + 1);
        i32x4 A[2][NT], B[2];
        lds_barrier();
#pragma unroll
        for (int r = 0; r < NT; ++r) A[0][r] = *reinterpret_cast<const i32x4 *>(wrow + r * 2048 + at[0]);
        B[0] = *reinterpret_cast<const i32x4 *>(xrow + at[0]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            const int c = i / MT, t = i % MT;
            if (i + 1 < kSlots) B[(i + 1) & 1] = *reinterpret_cast<const i32x4 *>(xrow + (i + 1) % MT * 2048 + at[(i + 1) / MT]);
            if (c == 0) {
#pragma unroll
                for (int r = t * kA; r < t * kA + kA && r < NT; ++r) A[1][r] = *reinterpret_cast<const i32x4 *>(wrow + r * 2048 + at[1]);
            }
#pragma unroll
            for (int k = i * kEach; k < i * kEach + kEach && k < kPieces; ++k) {
                if (k < kLoadW) {
                    *reinterpret_cast<i32x4 *>(wn_ + (wave * kLoadW + k) * 1024 + lane * 16) = rw[k];
                    rw[k] = load16(wbase + wo[k] + off);
                } else {
                    *reinterpret_cast<i32x4 *>(xn_ + (wave * kLoadX + k - kLoadW) * 1024 + lane * 16) = rx[k - kLoadW];
                    rx[k - kLoadW] = load16(xbase + xo[k - kLoadW] + off);
                }
            }
#pragma unroll
            for (int r = 0; r < NT; ++r) acc[r][t] = mfma(A[c][r], B[i & 1], acc[r][t]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto plain_step = [&](int b, const uint8_t *wb, const uint8_t *xb, uint8_t *wn_, uint8_t *xn_) __attribute__((always_inline)) {
        lds_barrier();
        put(b + 1, wn_, xn_);
        fetch(b + 2);
        multiply(wb, xb);
    };
    auto step = [&](int b, const uint8_t *wb, const uint8_t *xb, uint8_t *wn_, uint8_t *xn_) __attribute__((always_inline)) {
        if constexpr (kSpread) spread_step(b, wb, xb, wn_, xn_);
        else plain_step(b, wb, xb, wn_, xn_);
    };
    fetch(0);
    put(0, w0, x0);
    fetch(1);
    for (int b = 0; b < a.kb; b += 2) {
        step(b, w0, x0, w1, x1);
        if (b + 1 < a.kb) step(b + 1, w1, x1, w0, x0);
    }
    // A lane holds rows 4 g .. 4 g + 3 of each row tile for one token: 8 or 16 bytes of the output's row. 16 tokens at a
    // time go through the wave's own piece of LDS and leave as whole lines.
    constexpr int kRowBytes = NT * 16 * (int)sizeof(TY), kPitch = kRowBytes + (F32 ? 0 : 16), kLanes = kRowBytes / 16;
    constexpr int kPass = 64 / kLanes;  // rows a pass; lanes past a whole number of them idle
    static_assert(kTileWaves * 16 * kPitch <= BN * 128);
    __syncthreads();  // every wave has read the last block
    uint8_t *piece = w0 + wave * 16 * kPitch;
    TY *y = static_cast<TY *>(a.y);
    const int64_t nb = n0 + wn * (BN / kWn);
    const int64_t n = nb + (lane % kLanes) * (16 / (int)sizeof(TY));
    f32x4 sw[NT];
#pragma unroll
    for (int r = 0; r < NT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) sw[r][i] = a.ws[min(nb + r * 16 + 4 * g + i, a.N - 1)];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const float sx = a.xs[min(m0 + wm * (BM / kWm) + t * 16 + n16, a.M - 1)];
#pragma unroll
        for (int r = 0; r < NT; ++r) {
            f32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (float)acc[r][t][i] * sx * sw[r][i];
            store4(reinterpret_cast<TY *>(piece + n16 * kPitch) + r * 16 + 4 * g, v);
        }
        // one wave's LDS accesses take effect in program order: these reads follow the writes above
#pragma unroll
        for (int j = 0; j < 16; j += kPass) {
            const int row = j + lane / kLanes;
            if (lane >= kPass * kLanes || row >= 16) continue;
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
    int8_tiles_kernel<TY, BN, BM><<<(unsigned)((tiles + 7) / 8 * 8), 64 * kTileWaves, 0, s>>>(a, m_tiles, (int)tiles);
}

template <typename TY, int NT, int MT>
void launch_rows(const Args &a, hipStream_t s) {
    const dim3 grid((unsigned)((a.N + 16 * NT - 1) / (16 * NT)), (unsigned)((a.M + 16 * MT - 1) / (16 * MT)));
    int8_rows_kernel<TY, NT, MT><<<grid, 64 * kRowWaves, 0, s>>>(a);
}

// Up to 16 tokens: 16 weight rows a block, whose waves read nothing twice (12288 x 4096, M = 6: 12.3 us, 4.1 TB/s). Up to 32, and up to
// 64 where two passes still are at most two blocks a compute unit: 32 rows x 32 tokens a block. Above, the tile with the least rounds of
// blocks over the compute units times the time of a K block of 128, measured with the chip full: 0.41, 0.65, 1.19, 1.5 and 2.27 us for
// 128 x 64, 128 x 128, 256 x 128, 256 x 192 and 384 x 192 (rows x tokens). In us for the five tiles: 12288 x 4096, M = 1531 116 / 105 / 108 /
// 95 / 75, 512 41 / 43 / 38 / 47 / 66, 256 26 / 24 / 33 / 43 / 65; 4096 x 4096, M = 2048 53 / 44 / 41 / 48 / 67; 7680 x 2560, M = 1531 50 / 44 /
// 50 / 37 / 49. 75 us are 2.07 POP/s; the library's product of 8192 x 8192 x 8192 8-bit integers reaches 2.08 on the same card.
template <typename TY>
void launch(const Args &a, hipStream_t s) {
    const int64_t cus = device_cus();
    if (a.M <= 16) return launch_rows<TY, 1, 1>(a, s);
    if (a.M <= 32 || (a.M <= 64 && (a.N + 31) / 32 * 2 <= 2 * cus)) return launch_rows<TY, 2, 2>(a, s);
    auto cost = [&](int bn, int bm, double each) {
        const int64_t tiles = (a.N + bn - 1) / bn * ((a.M + bm - 1) / bm);
        return (double)((tiles + cus - 1) / cus) * each;
    };
    const double c[5] = {cost(128, 64, 0.41), cost(128, 128, 0.65), cost(256, 128, 1.19), cost(256, 192, 1.5), cost(384, 192, 2.27)};
    switch ((int)(std::min_element(c, c + 5) - c)) {
    case 0: return launch_tiles<TY, 128, 64>(a, s);
    case 1: return launch_tiles<TY, 128, 128>(a, s);
    case 2: return launch_tiles<TY, 256, 128>(a, s);
    case 3: return launch_tiles<TY, 256, 192>(a, s);
    default: return launch_tiles<TY, 384, 192>(a, s);
    }
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" int sx_linear_int8(const int8_t *x, const float *x_scale, const sx_int8_view *w, void *y, int64_t M, int out_act,
                              sx_stream stream) {
    SX_CHECK(x != nullptr && x_scale != nullptr && w != nullptr && w->q != nullptr && w->scale != nullptr && y != nullptr,
             "null pointer");
    const int64_t N = w->N, K = w->K;
    SX_CHECK(N >= 1 && N <= 0x7ffffff0 && K >= 16 && K % 16 == 0 && K <= 131056, "weight [", N, ", ", K, "]: K a multiple of 16, 16..131056");
    SX_CHECK(M >= 1 && M <= 1 << 22, "M = ", M, ", expected 1..", 1 << 22);
    SX_CHECK((N + 127) / 128 * ((M + 63) / 64) <= 0x7ffffff0, "N = ", N, " with M = ", M, ": too many tiles");
    SX_CHECK(out_act == SX_ACT_F32 || out_act == SX_ACT_BF16, "unsupported output dtype ", out_act);
    SX_CHECK(aligned(x, 16) && aligned(w->q, 16) && aligned(x_scale, 4) && aligned(w->scale, 4) && aligned(y, act_bytes(out_act)),
             "x and w must be 16-byte aligned, the scales 4-byte, y to its elements");
    const int64_t yb = M * N * act_bytes(out_act);
    SX_CHECK(apart(y, yb, x, M * K) && apart(y, yb, x_scale, M * 4) && apart(y, yb, w->q, N * K) && apart(y, yb, w->scale, N * 4), "y overlaps an input");
    const Args a{x, w->q, x_scale, w->scale, y, N, (int32_t)M, (int32_t)K, (int32_t)((K + 127) / 128), N * act_bytes(out_act) % 16 == 0 && aligned(y, 16)};
    if (out_act == SX_ACT_F32) launch<float>(a, stream_of(stream));
    else launch<uint16_t>(a, stream_of(stream));
    SX_LAUNCHED("linear_int8 M=", M, " N=", N, " K=", K);
    return SX_OK;
}
