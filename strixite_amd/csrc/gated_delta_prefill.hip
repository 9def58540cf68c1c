// The gated delta rule over prompts: sequences in chunks of 64 tokens. Inside a chunk (G the running sum of g from its first
// token on, k and q of length one, q times the scale)
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j (j < i),  T = (I + A)^-1 diag(beta),  P_ij = e^(G_i - G_j) q_i . k_j (j <= i),
//   U = T (V - e^G K S),  O = e^G Q S + P U,  S <- e^(G_C) S + (e^(G_C - G) K)^T U.
//
// T and P do not need the state: the first launch makes them for all chunks and heads at once. The second goes through the
// chunks in order. A state's columns do not need each other, so a block has 16 columns of one (256 blocks for one sequence of
// 32 heads of 128) and its four waves share a chunk: wave w holds a quarter of the state's rows in registers, multiplies K
// and Q with them for all 64 tokens, and has a quarter of the tokens after that. What passes between the waves (sums of K S
// and Q S, V - e^G K S, U) goes through LDS, three barriers a chunk. The latency of that chain is what bounds one
// sequence.
//
// Operands: a result of the matrix unit has four consecutive rows a lane, an operand eight consecutive values of a row. The
// rows of two result tiles are dealt out so that a lane's four of the one and four of the other are eight consecutive
// ones: row 4 g + r of tile s stands for 8 g + 4 s + r. So the state, V - e^G K S and U become operands where they are.
// FP32 values enter as three BF16 terms, which together are the value (P U, which only the BF16 output sees: two).
//
// Tokens that are no numbers: a triangular product would carry them to the tokens before them in the chunk. They are taken
// out and everything from them on (a value's: in its column) is NaN, as the rule has it.
#include "gated_delta.hpp"

namespace sx {
namespace delta {
namespace {

constexpr int kC = 64, kPitch = kC + 4;
constexpr int kBlocksT = 6;  // (row tile, pair of column tiles) with anything in it: 1, 1, 2, 2
constexpr int64_t kTBytes = kBlocksT * 3 * 1024, kPBytes = kBlocksT * 2 * 1024, kHeadBytes = kTBytes + kPBytes + 1024;

__host__ __device__ constexpr int block_of(int ti, int p) { return ti < 2 ? ti : 2 * (ti - 1) + p; }

// What a chunk and head leave for the scan beside T and P.
struct Words {
    float in[kC];    // e^G / |k|: of K S
    float out[kC];   // scale e^G / |q|: of Q S
    float keep[kC];  // e^(G_C - G) / |k|: of U in the new state
    float fade;      // e^(G_C)
    int32_t bad;     // the first token that is no number, kC: none
    uint64_t use;    // the tokens that count
};
static_assert(sizeof(Words) <= 1024);

struct Work {
    uint8_t *heads;  // [chunk slots][Hv] kHeadBytes: T, P, Words
    uint8_t *keys;   // [chunk slots][Hk] K^T as operands: [Dk / 16][2][64 lanes][8]
};

// A sequence's chunks take slots starts[b] / 64 + b on: enough for a last chunk that is not full.
__device__ __forceinline__ int64_t first_slot(int t0, int b) { return t0 / kC + b; }

// The token that result row 4 g + r of tile ti stands for, and that of operand row m.
__device__ __forceinline__ constexpr int token_of(int ti, int g, int r) { return 32 * (ti >> 1) + 8 * g + 4 * (ti & 1) + r; }
__device__ __forceinline__ int token_at(int ti, int m) { return token_of(ti, m >> 2, m & 3); }

template <int DK>
__global__ void __launch_bounds__(256) delta_prepare_kernel(const Args a, const Work w) {
    constexpr int KS = DK / 32;
    __shared__ __attribute__((aligned(16))) float At[kC * kPitch], P[kC * kPitch], Tm[kC * kPitch];
    __shared__ double path[kC];
    __shared__ float rk[kC], rq[kC], beta[kC];
    __shared__ uint64_t use_mask;
    __shared__ int found;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g4 = lane >> 4;
    const int64_t slot = blockIdx.x / a.Hv;
    const int h = blockIdx.x % a.Hv, hk = h / a.rep;
    // the sequence whose chunk this is: at most one (of possible starts)
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    for (int b = threadIdx.x; b < a.B; b += 256) {
        const int t0 = a.starts[b], t1 = a.starts[b + 1];
        if (t0 < 0 || t1 <= t0 || t1 > a.T || t1 - t0 > a.max_len) continue;
        const int64_t f = first_slot(t0, b);
        if (slot >= f && slot < f + (t1 - t0 + kC - 1) / kC) found = b;
    }
    __syncthreads();
    const int b = found;
    if (b < 0) return;
    const int t0 = a.starts[b], first = (int)(slot - first_slot(t0, b)) * kC, n = min(a.starts[b + 1] - t0 - first, kC);
    const int64_t row0 = (int64_t)t0 + first;
    const u32x4 none = {0u, 0u, 0u, 0u};
    bf16x8 K[4][KS], Q[KS];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        if (t > wave) continue;
        const int i = t * 16 + n16;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const u32x4 x = *reinterpret_cast<const u32x4 *>(a.k + (row0 + min(i, n - 1)) * a.k_t + hk * a.k_h + ks * 32 + g4 * 8);
            K[t][ks] = __builtin_bit_cast(bf16x8, i < n ? x : none);
        }
    }
    bf16x8 mine[KS];  // of this wave's tile
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int i = wave * 16 + n16;
        const u32x4 x = *reinterpret_cast<const u32x4 *>(a.q + (row0 + min(i, n - 1)) * a.q_t + hk * a.q_h + ks * 32 + g4 * 8);
        Q[ks] = __builtin_bit_cast(bf16x8, i < n ? x : none);
        mine[ks] = wave == 0 ? K[0][ks] : wave == 1 ? K[1][ks] : wave == 2 ? K[2][ks] : K[3][ks];
    }
    float kk = 0.f, qq = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        float x[8], y[8];
        unpack8(__builtin_bit_cast(u32x4, mine[ks]), x);
        unpack8(__builtin_bit_cast(u32x4, Q[ks]), y);
#pragma unroll
        for (int j = 0; j < 8; ++j) kk = fmaf(x[j], x[j], kk), qq = fmaf(y[j], y[j], qq);
    }
    kk = sum_rows(kk), qq = sum_rows(qq);
    if (g4 == 0) {
        // a key that is no number has no length
        rk[wave * 16 + n16] = !finite(kk) ? qnan() : a.normalize ? 1.f / sqrtf(kk + kNormEps) : 1.f;
        rq[wave * 16 + n16] = (a.normalize ? 1.f / sqrtf(qq + kNormEps) : 1.f) * a.scale;
    }
    __syncthreads();
    if (wave == 0) {
        float g = 0.f, be = 0.f;
        if (lane < n) gates(a, row0 + lane, h, g, be);
        const bool num = finite(rk[lane]) && finite(g) && finite(be), use = lane < n && num;
        if (!use) g = 0.f, be = 0.f, rk[lane] = 0.f;
        const uint64_t um = __ballot(use), bm = __ballot(lane < n && !num);
        double G = (double)g;  // in 64 bits: differences of long sums lose bits in 32
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double x = __shfl_up(G, d);
            if (lane >= d) G += x;
        }
        const double all = __shfl(G, 63);
        path[lane] = G, beta[lane] = be;
        Words *o = reinterpret_cast<Words *>(w.heads + (slot * a.Hv + h) * kHeadBytes + kTBytes + kPBytes);
        o->in[lane] = expf((float)G) * rk[lane];
        o->out[lane] = expf((float)G) * rq[lane];
        o->keep[lane] = expf((float)(all - G)) * rk[lane];
        if (lane == 0) o->fade = expf((float)all), o->bad = bm != 0 ? __builtin_ctzll(bm) : kC, o->use = um, use_mask = um;
    }
    __syncthreads();
    const uint64_t use = use_mask;
#pragma unroll
    for (int tj = 0; tj < 4; ++tj) {
        f32x4 kp = {0.f, 0.f, 0.f, 0.f}, qp = kp;
        if (tj <= wave) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) kp = mfma(mine[ks], K[tj][ks], kp), qp = mfma(Q[ks], K[tj][ks], qp);
        }
        const int j = tj * 16 + n16, i0 = wave * 16 + g4 * 4;
        const bool uj = use >> j & 1;
        f32x4 left;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + r;
            const float fade = uj && j <= i ? expf((float)(path[i] - path[j])) * rk[j] : 0.f;
            left[r] = uj && j < i && (use >> i & 1) ? beta[i] * rk[i] * fade * kp[r] : 0.f;
            P[i * kPitch + j] = uj && j <= i ? rq[i] * fade * qp[r] : 0.f;
        }
        *reinterpret_cast<f32x4 *>(&At[j * kPitch + i0]) = left;
    }
    __syncthreads();
    // Wave w solves (I + A) T = diag(beta) for its 16 columns: T's rows come out one after the other.
    f32x4 U[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) U[t][r] = t == wave && g4 * 4 + r == n16 ? beta[t * 16 + n16] : 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        if (t < wave) continue;
        auto take = [&](int i, float u) __attribute__((always_inline)) {
#pragma unroll
            for (int x = t; x < 4; ++x) {
                const f32x4 c = *reinterpret_cast<const f32x4 *>(&At[i * kPitch + x * 16 + g4 * 4]);
#pragma unroll
                for (int r = 0; r < 4; ++r) U[x][r] = fmaf(-c[r], u, U[x][r]);
            }
        };
#pragma unroll
        for (int r = 0; r < 4; ++r) take(t * 16 + r, of_row<0>(U[t][r]));
#pragma unroll
        for (int r = 0; r < 4; ++r) take(t * 16 + 4 + r, of_row<1>(U[t][r]));
#pragma unroll
        for (int r = 0; r < 4; ++r) take(t * 16 + 8 + r, of_row<2>(U[t][r]));
#pragma unroll
        for (int r = 0; r < 4; ++r) take(t * 16 + 12 + r, of_row<3>(U[t][r]));
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) Tm[(t * 16 + g4 * 4 + r) * kPitch + wave * 16 + n16] = U[t][r];
    __syncthreads();
    uint8_t *head = w.heads + (slot * a.Hv + h) * kHeadBytes;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        if (p > wave >> 1) continue;
        const int at = token_at(wave, n16) * kPitch + 32 * p + 8 * g4, blk = block_of(wave, p);
        float t8[8], p8[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t8[j] = Tm[at + j], p8[j] = P[at + j];
        bf16x8 ts[3], ps[2];
        split(t8, ts);
        split(p8, ps);
#pragma unroll
        for (int s = 0; s < 3; ++s) *reinterpret_cast<bf16x8 *>(head + (blk * 3 + s) * 1024 + lane * 16) = ts[s];
#pragma unroll
        for (int s = 0; s < 2; ++s) *reinterpret_cast<bf16x8 *>(head + kTBytes + (blk * 2 + s) * 1024 + lane * 16) = ps[s];
    }
    if (h % a.rep != 0) return;
    // the key head's K^T: row dk, eight tokens a lane
    static_assert(DK * kPitch * 2 <= sizeof(At));
    uint16_t *kt = reinterpret_cast<uint16_t *>(At);
    const bool count = use >> (wave * 16 + n16) & 1;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const u32x4 x = __builtin_bit_cast(u32x4, mine[ks]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            kt[(ks * 32 + g4 * 8 + j) * kPitch + wave * 16 + n16] = count ? (uint16_t)(x[j / 2] >> (16 * (j & 1))) : (uint16_t)0;
    }
    __syncthreads();
    uint8_t *keys = w.keys + (slot * a.Hk + hk) * (DK / 16 * 2048);
    constexpr int TS = DK / 64;
#pragma unroll
    for (int s = 0; s < TS; ++s)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int dk = 16 * TS * wave + 4 * TS * (n16 >> 2) + 4 * s + (n16 & 3);
            const u32x2 *src = reinterpret_cast<const u32x2 *>(&kt[dk * kPitch + 32 * p + 8 * g4]);
            const u32x2 lo = src[0], hi = src[1];
            *reinterpret_cast<u32x4 *>(keys + ((wave * TS + s) * 2 + p) * 1024 + lane * 16) = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
}

// What a wave needs of a chunk from memory.
template <int TS>
struct Chunk {
    bf16x8 K[4], Q[4];       // 4 TS of a token's values
    bf16x8 T[2][3], P[2][2];
    bf16x8 KT[TS][2];
    f32x4 in, out, keep;     // of the wave's four tokens a lane
    uint16_t v[4];
    float fade;
    int32_t bad;
    uint64_t use;
};

template <int DK>
__global__ void __launch_bounds__(256, 1) delta_scan_kernel(const Args a, const Work w, int pairs8) {
    constexpr int TS = DK / 64;  // tiles of the state's rows a wave has
    __shared__ __attribute__((aligned(16))) f32x4 xs[4][4][64], ys[4][4][64];  // [wave][tile]
    __shared__ __attribute__((aligned(16))) u32x2 rs[3][4][64], us[2][4][64], ks[3][4][64];
    __shared__ int poison[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g4 = lane >> 4;
    const int pair = blockIdx.x % pairs8, b = pair / a.Hv, h = pair % a.Hv, hk = h / a.rep;
    if (b >= a.B) return;
    const int col = (int)(blockIdx.x / pairs8) * 16 + n16;
    const Seq s = sequence(a.starts, a.slot, b, a.B, a.T, a.max_len, a.slots, true);
    if (blockIdx.x / pairs8 == 0 && h == 0 && threadIdx.x == 0) tell(s, b, a.err);
    if (s.n == 0) return;
    if (!s.ok) {
        for (int i = threadIdx.x >> 4; i < s.n; i += 16) a.out[(int64_t)(s.t0 + i) * a.o_t + h * a.o_h + col] = 0x7fc0;
        return;
    }
    if (threadIdx.x < 16) poison[threadIdx.x] = 0x7fffffff;
    float *state = a.state + s.slot * a.s_slot + ((int64_t)h * DK + 16 * TS * wave + 4 * TS * g4) * a.Dv + col;
    f32x4 S[TS];
#pragma unroll
    for (int t = 0; t < TS; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[t][r] = state[(int64_t)(4 * t + r) * a.Dv];
    const int chunks = (s.n + kC - 1) / kC;
    const int64_t slot0 = first_slot(s.t0, b);
    const uint16_t *kp = a.k + s.t0 * a.k_t + hk * a.k_h + 16 * TS * wave + 4 * TS * g4, *qp = a.q + s.t0 * a.q_t + hk * a.q_h + 16 * TS * wave + 4 * TS * g4;
    const uint16_t *vp = a.v + s.t0 * a.v_t + h * a.v_h + col;
    auto fetch = [&](int c, Chunk<TS> &o) __attribute__((always_inline)) {  // past the last one: the last one again, not used
        c = min(c, chunks - 1);
        const uint8_t *head = w.heads + ((slot0 + c) * a.Hv + h) * kHeadBytes, *keys = w.keys + ((slot0 + c) * a.Hk + hk) * (DK / 16 * 2048);
        const Words *words = reinterpret_cast<const Words *>(head + kTBytes + kPBytes);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int64_t at = min(c * kC + token_at(t, n16), s.n - 1);
            if constexpr (TS == 2) {
                o.K[t] = *reinterpret_cast<const bf16x8 *>(kp + at * a.k_t);
                o.Q[t] = *reinterpret_cast<const bf16x8 *>(qp + at * a.q_t);
            } else {
                const u32x2 x = *reinterpret_cast<const u32x2 *>(kp + at * a.k_t), y = *reinterpret_cast<const u32x2 *>(qp + at * a.q_t);
                o.K[t] = __builtin_bit_cast(bf16x8, u32x4{x[0], x[1], 0u, 0u}), o.Q[t] = __builtin_bit_cast(bf16x8, u32x4{y[0], y[1], 0u, 0u});
            }
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            if (p <= wave >> 1) {
                const int blk = block_of(wave, p);
#pragma unroll
                for (int i = 0; i < 3; ++i) o.T[p][i] = *reinterpret_cast<const bf16x8 *>(head + (blk * 3 + i) * 1024 + lane * 16);
#pragma unroll
                for (int i = 0; i < 2; ++i) o.P[p][i] = *reinterpret_cast<const bf16x8 *>(head + kTBytes + (blk * 2 + i) * 1024 + lane * 16);
            }
#pragma unroll
            for (int t = 0; t < TS; ++t) o.KT[t][p] = *reinterpret_cast<const bf16x8 *>(keys + ((wave * TS + t) * 2 + p) * 1024 + lane * 16);
        }
        const int at = token_of(wave, g4, 0);
        o.in = *reinterpret_cast<const f32x4 *>(&words->in[at]);
        o.out = *reinterpret_cast<const f32x4 *>(&words->out[at]);
        o.keep = *reinterpret_cast<const f32x4 *>(&words->keep[at]);
        o.fade = words->fade, o.bad = words->bad, o.use = words->use;
#pragma unroll
        for (int r = 0; r < 4; ++r) o.v[r] = vp[(int64_t)min(c * kC + at + r, s.n - 1) * a.v_t];
    };
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    auto put3 = [&](u32x2 (*to)[4][64], const f32x4 &x) __attribute__((always_inline)) {
        float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            to[i][wave][lane] = u32x2{tops(__float_as_uint(r[0]), __float_as_uint(r[1])), tops(__float_as_uint(r[2]), __float_as_uint(r[3]))};
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] -= __uint_as_float(__float_as_uint(r[j]) & 0xFFFF0000u);
        }
    };
    auto get = [&](const u32x2 (*from)[64], int p) __attribute__((always_inline)) {
        const u32x2 x = from[2 * p][lane], y = from[2 * p + 1][lane];
        return __builtin_bit_cast(bf16x8, u32x4{x[0], x[1], y[0], y[1]});
    };
    auto chunk = [&](int c, Chunk<TS> &now, Chunk<TS> &next) __attribute__((always_inline)) {
        fetch(c + 1, next);
        if (now.use != ~0ull) {
            const u32x4 none = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (!(now.use >> token_at(t, n16) & 1)) now.K[t] = __builtin_bit_cast(bf16x8, none);
        }
        // K S and Q S over this wave's rows of the state
        float s8[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) s8[j] = S[0][j], s8[4 + j] = TS == 2 ? S[TS - 1][j] : 0.f;
        bf16x8 so[3];
        split(s8, so);
        f32x4 X[4], Y[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) X[t] = mfma(now.K[t], so[2], zero);
#pragma unroll
        for (int t = 0; t < 4; ++t) X[t] = mfma(now.K[t], so[1], X[t]);
#pragma unroll
        for (int t = 0; t < 4; ++t) X[t] = mfma(now.K[t], so[0], X[t]);
#pragma unroll
        for (int t = 0; t < 4; ++t) Y[t] = mfma(now.Q[t], so[1], zero);
#pragma unroll
        for (int t = 0; t < 4; ++t) Y[t] = mfma(now.Q[t], so[0], Y[t]);
#pragma unroll
        for (int t = 0; t < 4; ++t) xs[wave][t][lane] = X[t], ys[wave][t][lane] = Y[t];
        lds_barrier();
        // this wave's 16 tokens: what the state does not explain of them
        f32x4 x = xs[0][wave][lane] + xs[1][wave][lane] + xs[2][wave][lane] + xs[3][wave][lane];
        const f32x4 y = ys[0][wave][lane] + ys[1][wave][lane] + ys[2][wave][lane] + ys[3][wave][lane];
        bool odd = now.bad < kC;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int at = token_of(wave, g4, r);
            float v = bf16_to_f32(now.v[r]);
            const bool use = now.use >> at & 1, num = finite(v);
            odd |= use && !num;
            x[r] = use && num ? v - now.in[r] * x[r] : use ? -now.in[r] * x[r] : 0.f;
        }
        if (__any(odd)) {
            int at = now.bad;
#pragma unroll
            for (int r = 3; r >= 0; --r) {
                const int i = token_of(wave, g4, r);
                if ((now.use >> i & 1) && !finite(bf16_to_f32(now.v[r]))) at = min(at, i);
            }
            if (at < kC) atomicMin(&poison[n16], c * kC + at);
        }
        put3(rs, x);
        lds_barrier();
        // U = T x
        f32x4 u = zero;
#pragma unroll
        for (int p = 0; p < 2; ++p)
            if (p <= wave >> 1) {
                const bf16x8 r0 = get(rs[0], p), r1 = get(rs[1], p), r2 = get(rs[2], p);
                u = mfma(now.T[p][2], r0, u);
                u = mfma(now.T[p][1], r1, u);
                u = mfma(now.T[p][0], r2, u);
                u = mfma(now.T[p][1], r0, u);
                u = mfma(now.T[p][0], r1, u);
                u = mfma(now.T[p][0], r0, u);
            }
        f32x4 uk = u;
#pragma unroll
        for (int r = 0; r < 4; ++r) uk[r] *= now.keep[r];
        put3(ks, uk);
        float lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[j] = u[j] - __uint_as_float(__float_as_uint(u[j]) & 0xFFFF0000u);
        us[0][wave][lane] = u32x2{tops(__float_as_uint(u[0]), __float_as_uint(u[1])), tops(__float_as_uint(u[2]), __float_as_uint(u[3]))};
        us[1][wave][lane] = u32x2{tops(__float_as_uint(lo[0]), __float_as_uint(lo[1])), tops(__float_as_uint(lo[2]), __float_as_uint(lo[3]))};
        lds_barrier();
#pragma unroll
        for (int t = 0; t < TS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[t][r] *= now.fade;
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int i = 2; i >= 0; --i) {
                const bf16x8 o = get(ks[i], p);
#pragma unroll
                for (int t = 0; t < TS; ++t) S[t] = mfma(now.KT[t][p], o, S[t]);
            }
        f32x4 O;
#pragma unroll
        for (int r = 0; r < 4; ++r) O[r] = now.out[r] * y[r];
#pragma unroll
        for (int p = 0; p < 2; ++p)
            if (p <= wave >> 1) {
                const bf16x8 u0 = get(us[0], p), u1 = get(us[1], p);
                O = mfma(now.P[p][1], u0, O);
                O = mfma(now.P[p][0], u1, O);
                O = mfma(now.P[p][0], u0, O);
            }
        const int from = poison[n16];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = c * kC + token_of(wave, g4, r);
            if (i < s.n) a.out[(int64_t)(s.t0 + i) * a.o_t + h * a.o_h + col] = i >= from ? (uint16_t)0x7fc0 : (uint16_t)f32_to_bf16(O[r]);
        }
    };
    Chunk<TS> even, other;
    fetch(0, even);
    __syncthreads();  // poison
    for (int c = 0; c < chunks; c += 2) {
        chunk(c, even, other);
        if (c + 1 < chunks) chunk(c + 1, other, even);
    }
    const bool lost = poison[n16] != 0x7fffffff;
#pragma unroll
    for (int t = 0; t < TS; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) state[(int64_t)(4 * t + r) * a.Dv] = lost ? qnan() : S[t][r];
}

}  // namespace

size_t prefill_bytes(int64_t T, int64_t B, int64_t Hk, int64_t Hv, int64_t Dk) {
    return (size_t)((T / kC + B) * (Hv * kHeadBytes + Hk * (Dk / 16 * 2048)));
}

void prefill(const Args &a, int Dk, void *ws, hipStream_t s) {
    const int64_t slots = a.T / kC + a.B;
    const Work w{static_cast<uint8_t *>(ws), static_cast<uint8_t *>(ws) + slots * a.Hv * kHeadBytes};
    // the blocks of one head's columns run on one XCD (block i: i % 8), whose L2 then has the chunk's T, P and K once
    const int pairs8 = (a.B * a.Hv + 7) / 8 * 8;
    const unsigned prep = (unsigned)(a.Hv * slots);
    if (Dk == 64) {
        delta_prepare_kernel<64><<<prep, 256, 0, s>>>(a, w);
        delta_scan_kernel<64><<<(unsigned)(pairs8 * (a.Dv / 16)), 256, 0, s>>>(a, w, pairs8);
    } else {
        delta_prepare_kernel<128><<<prep, 256, 0, s>>>(a, w);
        delta_scan_kernel<128><<<(unsigned)(pairs8 * (a.Dv / 16)), 256, 0, s>>>(a, w, pairs8);
    }
}

}  // namespace delta
}  // namespace sx
