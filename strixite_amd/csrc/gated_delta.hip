// The gated delta rule: a state S [Dk, Dv] for each value head, and for each token
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = S^T q,
// k and q scaled to length one (q times `scale` too). Steps of a few tokens, the verify of drafted tokens and the commit of
// those that were accepted; prompts are in gated_delta_prefill.hip.
//
// Step: the cost is the state, read and written once (2 x 64 KB a head at 128 x 128), so it goes through registers: a wave
// has 16 columns of one state, a lane four of them in Dk / 16 rows. Columns do not need each other, so waves never meet. Both
// sums over Dk, S^T k and S^T q, are taken of the state before the token (o = e^g S^T q + (k . q) u), one reduction. One token each
// of 48 sequences, 32 heads of 128: 44 us, 4.6 TB/s; of one sequence: 6.
//
// Verify: the drafted tokens are a tree, the state must not change before the accepted path is known, and token i needs
// the state behind its ancestors only. With G the sum of g along a token's path and A_ij = beta_i e^(G_i - G_j) k_i . k_j for
// the ancestors j of i,
//   (I + A) U = beta (V - e^G K S),   o_i = e^G_i S^T q_i + sum_j e^(G_i - G_j) (q_i . k_j) u_j   (j: ancestors and i),
// so the state is read once for all tokens, by the matrix unit, and no token's state is ever formed. U is what is left to
// write: the commit adds k_j u_j^T along the accepted path to the state, for all layers in one launch. 32 heads of 128: 24 trees of
// up to 24 26 us (a block's chain: waits 0.45 of its time, VALU 0.53) and 20 for the commit (5.1 TB/s, the states both ways); one
// chain of 6: 9.0 and 6.6.
#include "gated_delta.hpp"

#include "kv_cache.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace sx {
namespace {

using namespace delta;

// The four columns' sums over a wave's 16 row groups (lanes 4 apart), in all of them.
__device__ __forceinline__ float sum_slices(float x) {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x124, 0xF, 0xF, false));
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, false));
    return sum_rows(x);
}

// R consecutive BF16 values.
template <int R>
__device__ __forceinline__ void load_rows(const uint16_t *p, float (&v)[R]) {
    if constexpr (R == 8) {
        unpack8(*reinterpret_cast<const u32x4 *>(p), v);
    } else {
        const u32x2 u = *reinterpret_cast<const u32x2 *>(p);
        v[0] = __uint_as_float(u[0] << 16), v[1] = __uint_as_float(u[0] & 0xFFFF0000u);
        v[2] = __uint_as_float(u[1] << 16), v[3] = __uint_as_float(u[1] & 0xFFFF0000u);
    }
}

__device__ __forceinline__ void store_bf16x4(uint16_t *p, const float (&o)[4]) {
    *reinterpret_cast<u32x2 *>(p) = u32x2{f32_to_bf16(o[0]) | (f32_to_bf16(o[1]) << 16), f32_to_bf16(o[2]) | (f32_to_bf16(o[3]) << 16)};
}

template <int DK>
__global__ void __launch_bounds__(256) delta_step_kernel(const Args a) {
    constexpr int R = DK / 16;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = a.Dv / 16;
    const int64_t id = (int64_t)blockIdx.x * (blockDim.x >> 6) + wave;
    const int b = (int)(id / ((int64_t)tiles * a.Hv));
    if (b >= a.B) return;
    const int in = (int)(id - (int64_t)b * tiles * a.Hv), h = in / tiles, col = in % tiles * 16 + (lane & 3) * 4, row = (lane >> 2) * R;
    const int hk = h / a.rep;
    const Seq s = sequence(a.starts, a.slot, b, a.B, a.T, a.max_len, a.slots, true);
    if (in == 0 && lane == 0) tell(s, b, a.err);
    if (s.n == 0) return;
    if (!s.ok) {
        if (row == 0) {
            const float nan4[4] = {qnan(), qnan(), qnan(), qnan()};
            for (int i = 0; i < s.n; ++i) store_bf16x4(a.out + (s.t0 + i) * a.o_t + h * a.o_h + col, nan4);
        }
        return;
    }
    float *state = a.state + s.slot * a.s_slot + ((int64_t)h * DK + row) * a.Dv + col;
    f32x4 S[R];
#pragma unroll
    for (int r = 0; r < R; ++r) S[r] = *reinterpret_cast<const f32x4 *>(state + (int64_t)r * a.Dv);
    for (int i = 0; i < s.n; ++i) {
        const int64_t t = s.t0 + i;
        float k[R], q[R], v[4], g, beta;
        load_rows<R>(a.k + t * a.k_t + hk * a.k_h + row, k);
        load_rows<R>(a.q + t * a.q_t + hk * a.q_h + row, q);
        load_rows<4>(a.v + t * a.v_t + h * a.v_h + col, v);
        gates(a, t, h, g, beta);
        float kk = 0.f, qq = 0.f, kq = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) kk = fmaf(k[r], k[r], kk), qq = fmaf(q[r], q[r], qq), kq = fmaf(k[r], q[r], kq);
        f32x4 sk = {0.f, 0.f, 0.f, 0.f}, sq = sk;
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) sk[c] = fmaf(S[r][c], k[r], sk[c]), sq[c] = fmaf(S[r][c], q[r], sq[c]);
        kk = sum_slices(kk), qq = sum_slices(qq), kq = sum_slices(kq);
        const float rk = key_scale(a, kk), rq = query_scale(a, qq);
        const float fade = expf(g);
        float o[4];
        f32x4 u;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            u[c] = beta * (v[c] - fade * rk * sum_slices(sk[c]));
            o[c] = fade * rq * sum_slices(sq[c]) + kq * rk * rq * u[c];
            u[c] *= rk;
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) S[r][c] = fmaf(k[r], u[c], fade * S[r][c]);
        if (row == 0) store_bf16x4(a.out + t * a.o_t + h * a.o_h + col, o);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) *reinterpret_cast<f32x4 *>(state + (int64_t)r * a.Dv) = S[r];
}

// ---------------- verify ----------------

// Over the C neighbouring lanes (8 or 16) that hold a row.
template <int C>
__device__ __forceinline__ float sum_chunks(float x) {
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0xB1, 0xF, 0xF, false));
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x4E, 0xF, 0xF, false));
    x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x141, 0xF, 0xF, false));
    if constexpr (C == 16) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x140, 0xF, 0xF, false));
    return x;
}

constexpr int kMaxNew = 64;

struct VerifyArgs {
    Args d;
    const uint64_t *mask;
    int64_t mask_ld;
    float *u, *decay;
};

// NT tiles of 16 tokens, W waves of 16 columns each, which share the tokens' keys and queries and their products in LDS. All operand
// orders are natural: a lane (n16, g4) of a 32-deep product has values 8 g4 .. 8 g4 + 7 of row n16, of a result column n16 and rows
// 4 g4 .. 4 g4 + 3. A row's 16-byte chunk c lies at c ^ row, so that 16 rows' reads spread over all banks.
template <int DK, int NT, int W>
__global__ void __launch_bounds__(64 * W) delta_verify_kernel(const VerifyArgs va) {
    constexpr int N = 16 * NT, KS = DK / 32, kPitch = N + 4, kRow = DK / 8;  // chunks a row
    const Args &a = va.d;
    __shared__ u32x4 keys[N * kRow], queries[N * kRow];
    __shared__ __attribute__((aligned(16))) float At[N * kPitch];  // [j][i]: of token j in row i's system
    __shared__ __attribute__((aligned(16))) float P[N * kPitch];   // [i][j]
    __shared__ double path[N];                                     // G
    __shared__ uint64_t sees[N];
    __shared__ float rk[N], rq[N], beta[N], grow[N];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g4 = lane >> 4;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / a.rep;
    const int col = ((int)blockIdx.x * W + wave) * 16 + n16;
    const bool on = col < a.Dv;  // whole waves
    const Seq s = sequence(a.starts, a.slot, b, a.B, a.T, a.max_len, a.slots, false);
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) tell(s, b, a.err);
    if (s.n == 0) return;
    if (!s.ok) {
        if (on)
            for (int i = g4; i < s.n; i += 4) {
                a.out[(s.t0 + i) * a.o_t + h * a.o_h + col] = 0x7fc0;
                va.u[((int64_t)(s.t0 + i) * a.Hv + h) * a.Dv + col] = qnan();
                if (blockIdx.x == 0 && wave == 0 && n16 == 0) va.decay[(int64_t)(s.t0 + i) * a.Hv + h] = qnan();
            }
        return;
    }
    // everything from memory is requested before anything is used
    constexpr int kPieces = (N * kRow + 64 * W - 1) / (64 * W);
    u32x4 kp[kPieces], qp[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        const int id = threadIdx.x + i * 64 * W;
        const int64_t at = s.t0 + min(id / kRow, s.n - 1);
        kp[i] = *reinterpret_cast<const u32x4 *>(a.k + at * a.k_t + hk * a.k_h + id % kRow * 8);
        qp[i] = *reinterpret_cast<const u32x4 *>(a.q + at * a.q_t + hk * a.q_h + id % kRow * 8);
    }
    float g = 0.f, be = 0.f;
    uint64_t word = 0;
    if (wave == 0 && lane < s.n) {
        gates(a, s.t0 + lane, h, g, be);
        word = (va.mask[(s.t0 + lane) * va.mask_ld] & ((1ull << lane) - 1)) | 1ull << lane;
    }
    float st[KS][8];
    if (on) {
        const float *state = a.state + s.slot * a.s_slot + (int64_t)h * DK * a.Dv + col;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) st[ks][j] = state[(int64_t)(ks * 32 + g4 * 8 + j) * a.Dv];
    }
    uint16_t v[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[t][r] = a.v[(s.t0 + min(t * 16 + g4 * 4 + r, s.n - 1)) * a.v_t + h * a.v_h + (on ? col : 0)];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
        if (threadIdx.x + i * 64 * W >= N * kRow) break;
        const int id = threadIdx.x + i * 64 * W, row = id / kRow, c = (id % kRow) ^ (row & (kRow - 1));
        const u32x4 none = {0u, 0u, 0u, 0u};
        if (row >= s.n) kp[i] = none, qp[i] = none;
        keys[row * kRow + c] = kp[i], queries[row * kRow + c] = qp[i];
        float x[8], y[8], kk = 0.f, qq = 0.f;
        unpack8(kp[i], x);
        unpack8(qp[i], y);
#pragma unroll
        for (int j = 0; j < 8; ++j) kk = fmaf(x[j], x[j], kk), qq = fmaf(y[j], y[j], qq);
        kk = sum_chunks<kRow>(kk), qq = sum_chunks<kRow>(qq);
        if (id % kRow == 0) {
            rk[row] = key_scale(a, kk), rq[row] = query_scale(a, qq);
        }
    }
    if (wave == 0) {
        // token `lane`'s path, its sum in 64 bits: differences of long paths lose bits in 32
        double G = 0.0;
        for (int j = 0; j < s.n; ++j) {
            const float gj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), j));
            G += word >> j & 1 ? (double)gj : 0.0;
        }
        if (lane < N) path[lane] = G, sees[lane] = word, beta[lane] = be, grow[lane] = expf((float)G);
        if (blockIdx.x == 0 && lane < s.n) va.decay[(int64_t)(s.t0 + lane) * a.Hv + h] = g;
    }
    __syncthreads();
    auto operand = [&](const u32x4 *rows, int t, int ks) __attribute__((always_inline)) {
        const int row = t * 16 + n16;
        return __builtin_bit_cast(bf16x8, rows[row * kRow + ((ks * 4 + g4) ^ (row & (kRow - 1)))]);
    };
    // Products of tokens. An unseen pair is -0.0, which no seen one is: what it would meet is left out, NaN too.
#pragma unroll
    for (int ti = 0; ti < NT; ++ti)
#pragma unroll
        for (int tj = 0; tj < NT; ++tj) {
            if ((ti * NT + tj) % W != wave) continue;
            f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = kk;
            if (tj <= ti) {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const bf16x8 other = operand(keys, tj, ks);
                    kk = mfma(operand(keys, ti, ks), other, kk), qk = mfma(operand(queries, ti, ks), other, qk);
                }
            }
            const int j = tj * 16 + n16, i0 = ti * 16 + g4 * 4;
            const float rj = rk[j];
            const double Gj = path[j];
            f32x4 left;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = i0 + r;
                const bool seen = tj <= ti && (sees[i] >> j & 1);
                const float fade = seen ? expf((float)(path[i] - Gj)) * rj : 0.f;
                left[r] = seen && j < i ? beta[i] * rk[i] * fade * kk[r] + 0.f : -0.f;
                P[i * kPitch + j] = seen ? rq[i] * fade * qk[r] + 0.f : -0.f;
            }
            *reinterpret_cast<f32x4 *>(&At[j * kPitch + i0]) = left;
        }
    __syncthreads();
    if (!on) return;
    f32x4 X[NT], Y[NT], U[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) X[t] = Y[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        bf16x8 o[3], K[NT], Q[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) K[t] = operand(keys, t, ks), Q[t] = operand(queries, t, ks);
        split(st[ks], o);
#pragma unroll
        for (int p = 2; p >= 0; --p)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                X[t] = mfma(K[t], o[p], X[t]);
                Y[t] = mfma(Q[t], o[p], Y[t]);
            }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = t * 16 + g4 * 4 + r;
            U[t][r] = i < s.n ? beta[i] * (bf16_to_f32(v[t][r]) - grow[i] * rk[i] * X[t][r]) : 0.f;
        }
    // Forward substitution: token i's u is ready once those before it have been taken off its row, and then taken off all rows behind
    // it. GUARD leaves unseen pairs out; without it they are zeros, which is as good while all is finite.
    auto solve = [&](auto guard) __attribute__((always_inline)) {
        constexpr bool GUARD = decltype(guard)::value;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            auto take = [&](int i, float u) __attribute__((always_inline)) {
#pragma unroll
                for (int x = t; x < NT; ++x) {
                    const f32x4 c = *reinterpret_cast<const f32x4 *>(&At[i * kPitch + x * 16 + g4 * 4]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) U[x][r] = GUARD && __float_as_uint(c[r]) == 0x80000000u ? U[x][r] : fmaf(-c[r], u, U[x][r]);
                }
            };
            if (t * 16 < s.n) {
#pragma unroll
                for (int r = 0; r < 4; ++r) take(t * 16 + r, of_row<0>(U[t][r]));
            }
            if (t * 16 + 4 < s.n) {
#pragma unroll
                for (int r = 0; r < 4; ++r) take(t * 16 + 4 + r, of_row<1>(U[t][r]));
            }
            if (t * 16 + 8 < s.n) {
#pragma unroll
                for (int r = 0; r < 4; ++r) take(t * 16 + 8 + r, of_row<2>(U[t][r]));
            }
            if (t * 16 + 12 < s.n) {
#pragma unroll
                for (int r = 0; r < 4; ++r) take(t * 16 + 12 + r, of_row<3>(U[t][r]));
            }
        }
    };
    f32x4 before[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) before[t] = U[t];
    solve(std::false_type{});
    bool fine = true;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) fine &= finite(U[t][r]);
    const bool all_fine = !__any(!fine);
    if (!all_fine) {
#pragma unroll
        for (int t = 0; t < NT; ++t) U[t] = before[t];
        solve(std::true_type{});
    }
    f32x4 O[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = t * 16 + g4 * 4 + r;
            O[t][r] = grow[i] * rq[i] * Y[t][r];
        }
    if (all_fine) {
        // P U with both in three BF16 terms, of whose products the six largest are taken (what is left is under 2^-22), one of 32
        // tokens a pair of tiles
#pragma unroll
        for (int p = 0; p < (NT + 1) / 2; ++p) {
            float u8[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) u8[j] = U[2 * p][j], u8[4 + j] = 2 * p + 1 < NT ? U[(2 * p + 1) % NT][j] : 0.f;
            bf16x8 ub[3];
            split(u8, ub);
#pragma unroll
            for (int t = 2 * p; t < NT; ++t) {
                const float *prow = &P[(t * 16 + n16) * kPitch + p * 32 + g4 * 4];
                const f32x4 lo = *reinterpret_cast<const f32x4 *>(prow);
                f32x4 hi = {0.f, 0.f, 0.f, 0.f};
                if (2 * p + 1 < NT) hi = *reinterpret_cast<const f32x4 *>(prow + 16);
                const float p8[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                bf16x8 pb[3];
                split(p8, pb);
                O[t] = mfma(pb[2], ub[0], O[t]);
                O[t] = mfma(pb[1], ub[1], O[t]);
                O[t] = mfma(pb[0], ub[2], O[t]);
                O[t] = mfma(pb[1], ub[0], O[t]);
                O[t] = mfma(pb[0], ub[1], O[t]);
                O[t] = mfma(pb[0], ub[0], O[t]);
            }
        }
    } else {  // a token that is no number, or too large for one, meets only those that see it
        for (int j = 0; j < s.n; ++j) {
            float mine = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) mine = j == t * 16 + g4 * 4 + r ? U[t][r] : mine;
            const float uj = __shfl(mine, n16 + 16 * ((j >> 2) & 3));
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float c = P[(t * 16 + g4 * 4 + r) * kPitch + j];
                    O[t][r] = __float_as_uint(c) == 0x80000000u ? O[t][r] : fmaf(c, uj, O[t][r]);
                }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = t * 16 + g4 * 4 + r;
            if (i >= s.n) continue;
            a.out[(s.t0 + i) * a.o_t + h * a.o_h + col] = __builtin_bit_cast(uint16_t, (__bf16)O[t][r]);
            va.u[((int64_t)(s.t0 + i) * a.Hv + h) * a.Dv + col] = rk[i] * U[t][r];
        }
}

// ---------------- commit ----------------

struct CommitArgs {
    const uint16_t *k;
    const float *u, *decay;
    float *state;
    const int32_t *slot, *starts, *count, *path;
    uint32_t *err;
    int64_t k_l, k_t, k_h, u_l, g_l, s_l, s_slot, path_ld;
    int32_t T, Hv, rep, Dv, B, slots, max_count, layers;
};

// A wave has 16 columns of a state, as in a step. Lane i has path entry i's decay; the weights are e to the sums behind.
template <int DK>
__global__ void __launch_bounds__(256) delta_commit_kernel(const CommitArgs a) {
    constexpr int R = DK / 16, kAhead = 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles = a.Dv / 16;
    const int64_t id = (int64_t)blockIdx.x * 4 + wave;
    const int64_t pair = id / ((int64_t)tiles * a.Hv);
    const int layer = (int)(pair / a.B), b = (int)(pair % a.B);
    if (layer >= a.layers) return;
    const int in = (int)(id - pair * tiles * a.Hv), h = in / tiles, col = in % tiles * 16 + (lane & 3) * 4, row = (lane >> 2) * R;
    const Seq s = sequence(a.starts, a.slot, b, a.B, a.T, kMaxNew, a.slots, true);
    const int cnt = a.count[b];
    // every wave of a sequence looks all of its words over, so that they agree: it is committed as asked or not at all
    bool bad = !s.run || (!s.ok && s.n > 0) || cnt < 0 || cnt > a.max_count || cnt > s.n;
    uint32_t word = !s.run ? (uint32_t)s.t0 : !s.ok ? (uint32_t)s.slot : (uint32_t)cnt;
    int node = lane;
    if (!bad && lane < cnt) {
        if (a.path != nullptr) node = a.path[b * a.path_ld + lane];
        if (node < 0 || node >= s.n) bad = true, word = (uint32_t)node;
    }
    if (in == 0 && layer == 0 && bad) report(a.err, word, (uint32_t)b);
    if (__any(bad) || cnt == 0) return;
    const int64_t t0 = s.t0;
    float g = lane < cnt ? a.decay[layer * a.g_l + (t0 + node) * a.Hv + h] : 0.f;
    double behind = g;  // the sum of lane .. 63
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double x = __shfl_down(behind, d);
        if (lane + d < 64) behind += x;
    }
    const float all = expf((float)__shfl(behind, 0)), weight = expf((float)(behind - (double)g));
    float *state = a.state + layer * a.s_l + s.slot * a.s_slot + ((int64_t)h * DK + row) * a.Dv + col;
    f32x4 S[R];
#pragma unroll
    for (int r = 0; r < R; ++r) S[r] = all * *reinterpret_cast<const f32x4 *>(state + (int64_t)r * a.Dv);
    const uint16_t *kp = a.k + layer * a.k_l + (h / a.rep) * a.k_h + row;
    const float *up = a.u + layer * a.u_l + (int64_t)h * a.Dv + col;
    for (int i0 = 0; i0 < cnt; i0 += kAhead) {
        float k[kAhead][R], w[kAhead];
        f32x4 u[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = min(i0 + j, cnt - 1), at = __builtin_amdgcn_readfirstlane(__shfl(node, i));
            w[j] = __shfl(weight, i);
            load_rows<R>(kp + (t0 + at) * a.k_t, k[j]);
            u[j] = *reinterpret_cast<const f32x4 *>(up + (t0 + at) * a.Hv * a.Dv);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (i0 + j < cnt) {
                u[j] *= w[j];
#pragma unroll
                for (int r = 0; r < R; ++r)
#pragma unroll
                    for (int c = 0; c < 4; ++c) S[r][c] = fmaf(k[j][r], u[j][c], S[r][c]);
            }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) *reinterpret_cast<f32x4 *>(state + (int64_t)r * a.Dv) = S[r];
}

}  // namespace
}  // namespace sx

using namespace sx;

namespace {

// Why an sx_delta is not one that the kernels take; empty where it is.
std::string delta_error(const sx_delta &d) {
    if (d.q.p == nullptr || d.k.p == nullptr || d.v.p == nullptr || d.a == nullptr || d.b == nullptr || d.state == nullptr || d.starts == nullptr)
        return "null pointer";
    if ((d.A_log == nullptr) != (d.dt_bias == nullptr)) return "A_log and dt_bias go together";
    if (d.gate_act != SX_ACT_F32 && d.gate_act != SX_ACT_BF16) return cat("unsupported gate dtype ", d.gate_act);
    if (d.T < 1 || d.T > 0x3fffffff) return cat("T = ", d.T);
    if (d.batch < 1 || d.batch > delta::kMaxSeqs) return cat("batch = ", d.batch, ", expected 1..", delta::kMaxSeqs);
    if (d.key_heads < 1 || d.heads < d.key_heads || d.heads > 1024 || d.heads % d.key_heads != 0)
        return cat("heads = ", d.heads, ", expected a multiple of the key heads ", d.key_heads, ", up to 1024");
    if (d.key_dim != 64 && d.key_dim != 128) return cat("key_dim = ", d.key_dim, ", expected 64 or 128");
    if (d.dim < 16 || d.dim > 1024 || d.dim % 16 != 0) return cat("dim = ", d.dim, ", expected a multiple of 16, 16..1024");
    if (d.slots < 1 || d.slots > 0x7fffffff || (d.slot == nullptr && d.slots < d.batch)) return cat("slots = ", d.slots, " for batch = ", d.batch);
    if (d.state_slot < d.heads * d.key_dim * d.dim || d.state_slot % 4 != 0 || d.state_slot > (int64_t)1 << 40)
        return cat("state_slot = ", d.state_slot, ", expected a multiple of 4, at least heads key_dim dim");
    if (!aligned(d.state, 16) || !aligned(d.q.p, 16) || !aligned(d.k.p, 16) || !aligned(d.v.p, 16)) return "q, k, v and state must be 16-byte aligned";
    if (!aligned(d.starts, 4) || !aligned(d.slot, 4) || !aligned(d.A_log, 4) || !aligned(d.dt_bias, 4) ||
        !aligned(d.a, act_bytes(d.gate_act)) || !aligned(d.b, act_bytes(d.gate_act)))
        return "starts, slot and the gates must be aligned to their elements";
    // a chunk's rows are addressed by 32-bit offsets, heads by 64-bit ones
    const int64_t t[3] = {d.q.token, d.k.token, d.v.token}, h[3] = {d.q.head, d.k.head, d.v.head};
    for (int i = 0; i < 3; ++i)
        if (t[i] < 0 || t[i] > (int64_t)1 << 24 || t[i] % 8 != 0 || h[i] < 0 || h[i] > (int64_t)1 << 40 || h[i] % 8 != 0)
            return cat("strides of q, k and v must be multiples of 8, of tokens up to 2^24 (", t[i], ", ", h[i], ")");
    if (d.a_token < 0 || d.b_token < 0 || d.a_token > (int64_t)1 << 32 || d.b_token > (int64_t)1 << 32) return cat("gate strides ", d.a_token, ", ", d.b_token);
    if (!std::isfinite(d.scale)) return cat("scale = ", d.scale);
    return "";
}

int64_t span(const sx_head_rows &r, int64_t T, int64_t H, int64_t D) { return 2 * ((T - 1) * r.token + (H - 1) * r.head + D); }
int64_t state_bytes(const sx_delta &d) { return 4 * ((d.slots - 1) * d.state_slot + d.heads * d.key_dim * d.dim); }

// Why out, or another output of n bytes, cannot be written; empty where it can.
std::string output_error(const sx_delta &d, const void *o, int64_t n) {
    const int64_t e = act_bytes(d.gate_act);
    if (!apart(o, n, d.q.p, span(d.q, d.T, d.key_heads, d.key_dim)) || !apart(o, n, d.k.p, span(d.k, d.T, d.key_heads, d.key_dim)) ||
        !apart(o, n, d.v.p, span(d.v, d.T, d.heads, d.dim)))
        return "overlaps q, k or v";
    if (!apart(o, n, d.a, ((d.T - 1) * d.a_token + d.heads) * e) || !apart(o, n, d.b, ((d.T - 1) * d.b_token + d.heads) * e)) return "overlaps the gates";
    if (!apart(o, n, d.starts, 4 * (d.batch + 1)) || (d.slot != nullptr && !apart(o, n, d.slot, 4 * d.batch)) ||
        (d.A_log != nullptr && (!apart(o, n, d.A_log, 4 * d.heads) || !apart(o, n, d.dt_bias, 4 * d.heads))))
        return "overlaps starts, slot, A_log or dt_bias";
    return "";
}

std::string out_error(const sx_delta &d, const sx_head_rows &o) {
    if (o.p == nullptr) return "null pointer";
    if (!aligned(o.p, 8) || o.token < 0 || o.head < 0 || o.token % 4 != 0 || o.head % 4 != 0 || o.token > (int64_t)1 << 24 || o.head > (int64_t)1 << 40)
        return cat("must be 8-byte aligned with strides that are multiples of 4, of tokens up to 2^24 (", o.token, ", ", o.head, ")");
    if (!rows_apart(d.dim, {{d.T, o.token}, {d.heads, o.head}})) return "has heads that overlap";
    const std::string e = output_error(d, o.p, span(o, d.T, d.heads, d.dim));
    if (!e.empty()) return e;
    return apart(o.p, span(o, d.T, d.heads, d.dim), d.state, state_bytes(d)) ? "" : "overlaps the states";
}

delta::Args args_of(const sx_delta &d, const sx_head_rows *out, int64_t max_len, uint32_t *err) {
    const auto h = [](const sx_head_rows &r) { return static_cast<const uint16_t *>(r.p); };
    return {h(d.q), h(d.k), h(d.v), d.a, d.b, d.A_log, d.dt_bias, d.state, d.slot, d.starts, static_cast<uint16_t *>(out->p), err,
            d.q.token, d.q.head, d.k.token, d.k.head, d.v.token, d.v.head, d.a_token, d.b_token, d.T > 1 ? out->token : d.dim, out->head, d.state_slot,
            (int32_t)d.T, (int32_t)d.key_heads, (int32_t)d.heads, (int32_t)(d.heads / d.key_heads), (int32_t)d.dim, (int32_t)d.batch,
            (int32_t)d.slots, (int32_t)max_len, d.scale, d.gate_act == SX_ACT_F32, d.normalize != 0};
}

// Up to this many tokens a sequence go one by one.
constexpr int64_t kStepTokens = 16;

template <int DK, int NT>
void launch_verify(const VerifyArgs &v, hipStream_t s) {
    const Args &a = v.d;
    const int64_t waves = (int64_t)a.Dv / 16 * a.Hv * a.B;
    if (waves > 2 * device_cus()) delta_verify_kernel<DK, NT, 4><<<dim3((unsigned)((a.Dv + 63) / 64), (unsigned)a.Hv, (unsigned)a.B), 256, 0, s>>>(v);
    else delta_verify_kernel<DK, NT, 1><<<dim3((unsigned)(a.Dv / 16), (unsigned)a.Hv, (unsigned)a.B), 64, 0, s>>>(v);
}

template <int DK>
void launch_verify(const VerifyArgs &v, hipStream_t s) {
    if (v.d.max_len <= 16) return launch_verify<DK, 1>(v, s);
    if (v.d.max_len <= 32) return launch_verify<DK, 2>(v, s);
    launch_verify<DK, 4>(v, s);
}

}  // namespace

extern "C" int sx_gated_delta_workspace_bytes(int64_t T, int64_t B, int64_t Hk, int64_t Hv, int64_t Dk, int64_t max_len, size_t *bytes) {
    SX_CHECK(bytes != nullptr, "null pointer");
    SX_CHECK(T >= 1 && T <= 0x3fffffff && B >= 1 && B <= delta::kMaxSeqs && Hk >= 1 && Hv >= Hk && Hv <= 1024 && Hv % Hk == 0 && (Dk == 64 || Dk == 128) && max_len >= 1,
             "T = ", T, ", batch = ", B, ", heads = ", Hk, ", ", Hv, ", key_dim = ", Dk, ", max_len = ", max_len);
    *bytes = max_len <= kStepTokens ? 0 : delta::prefill_bytes(T, B, Hk, Hv, Dk);
    return SX_OK;
}

extern "C" int sx_gated_delta(const sx_delta *d, int64_t max_len, const sx_head_rows *out, void *ws, size_t ws_bytes, uint32_t *err, sx_stream stream) {
    SX_CHECK(d != nullptr && out != nullptr, "null pointer");
    const std::string e = delta_error(*d);
    SX_CHECK(e.empty(), e);
    SX_CHECK(max_len >= 1 && max_len <= 0x3fffffff, "max_len = ", max_len);
    const std::string o = out_error(*d, *out);
    SX_CHECK(o.empty(), "out ", o);
    const std::string st = output_error(*d, d->state, state_bytes(*d));
    SX_CHECK(st.empty(), "state ", st);
    const Args a = args_of(*d, out, max_len, err);
    if (max_len <= kStepTokens) {
        const int64_t waves = d->dim / 16 * d->heads * d->batch;
        // four waves a block; one where that leaves compute units without any (a step of one sequence of 32 heads)
        const int per = waves >= 16 * device_cus() ? 4 : 1;
        const unsigned blocks = (unsigned)((waves + per - 1) / per);
        if (d->key_dim == 64) delta_step_kernel<64><<<blocks, 64 * per, 0, stream_of(stream)>>>(a);
        else delta_step_kernel<128><<<blocks, 64 * per, 0, stream_of(stream)>>>(a);
    } else {
        const size_t need = delta::prefill_bytes(d->T, d->batch, d->key_heads, d->heads, d->key_dim);
        SX_CHECK(ws != nullptr && ws_bytes >= need, "a workspace of ", ws_bytes, " bytes, expected ", need);
        SX_CHECK(aligned(ws, 16), "the workspace must be 16-byte aligned");
        const std::string w = output_error(*d, ws, (int64_t)need);
        SX_CHECK(w.empty() && apart(ws, (int64_t)need, d->state, state_bytes(*d)) && apart(ws, (int64_t)need, out->p, span(*out, d->T, d->heads, d->dim)),
                 "the workspace overlaps another argument");
        SX_CHECK((d->T / 64 + d->batch) * d->heads <= 0x7fffffff && (d->batch * d->heads + 8) * (d->dim / 16) <= 0x7fffffff, "T = ", d->T, " of ", d->heads, " heads: too many chunks");
        delta::prefill(a, (int)d->key_dim, ws, stream_of(stream));
    }
    SX_LAUNCHED("gated_delta T=", d->T, " batch=", d->batch);
    return SX_OK;
}

extern "C" int sx_gated_delta_verify(const sx_delta *d, int64_t max_new, const uint64_t *mask, int64_t mask_ld, const sx_head_rows *out, float *u,
                                     float *decay, uint32_t *err, sx_stream stream) {
    SX_CHECK(d != nullptr && out != nullptr && mask != nullptr && u != nullptr && decay != nullptr, "null pointer");
    const std::string e = delta_error(*d);
    SX_CHECK(e.empty(), e);
    SX_CHECK(max_new >= 1 && max_new <= kMaxNew, "max_new = ", max_new, ", expected 1..", kMaxNew);
    SX_CHECK(mask_ld >= 1 && mask_ld <= (int64_t)1 << 32 && aligned(mask, 8), "mask_ld = ", mask_ld, ", or a misaligned mask");
    const std::string o = out_error(*d, *out);
    SX_CHECK(o.empty(), "out ", o);
    SX_CHECK(aligned(u, 16) && aligned(decay, 4), "u must be 16-byte and decay 4-byte aligned");
    const int64_t ub = 4 * d->T * d->heads * d->dim, gb = 4 * d->T * d->heads, ob = span(*out, d->T, d->heads, d->dim), mb = 8 * ((d->T - 1) * mask_ld + 1);
    const std::string eu = output_error(*d, u, ub), eg = output_error(*d, decay, gb);
    SX_CHECK(eu.empty(), "u ", eu);
    SX_CHECK(eg.empty(), "decay ", eg);
    SX_CHECK(apart(u, ub, decay, gb) && apart(u, ub, out->p, ob) && apart(decay, gb, out->p, ob) && apart(u, ub, d->state, state_bytes(*d)) &&
                 apart(decay, gb, d->state, state_bytes(*d)) && apart(u, ub, mask, mb) && apart(decay, gb, mask, mb) && apart(out->p, ob, mask, mb),
             "u, decay, out, mask and the states overlap");
    const VerifyArgs v{args_of(*d, out, max_new, err), mask, mask_ld, u, decay};
    if (d->key_dim == 64) launch_verify<64>(v, stream_of(stream));
    else launch_verify<128>(v, stream_of(stream));
    SX_LAUNCHED("gated_delta_verify T=", d->T, " batch=", d->batch);
    return SX_OK;
}

extern "C" int sx_gated_delta_commit(const sx_head_rows *k, const float *u, const float *decay, int64_t layers, int64_t T, int64_t Hk, int64_t Hv,
                                     int64_t Dk, int64_t Dv, float *state, int64_t state_layer, int64_t state_slot, int64_t slots, const int32_t *slot,
                                     const int32_t *starts, int64_t batch, const int32_t *count, int64_t max_count, const int32_t *path,
                                     int64_t path_ld, uint32_t *err, sx_stream stream) {
    SX_CHECK(k != nullptr && k->p != nullptr && u != nullptr && decay != nullptr && state != nullptr && starts != nullptr && count != nullptr, "null pointer");
    SX_CHECK(layers >= 1 && layers <= 65535 && T >= 1 && T <= 0x3fffffff, "layers = ", layers, ", T = ", T);
    SX_CHECK(batch >= 1 && batch <= delta::kMaxSeqs, "batch = ", batch, ", expected 1..", delta::kMaxSeqs);
    SX_CHECK(Hk >= 1 && Hv >= Hk && Hv <= 1024 && Hv % Hk == 0, "heads = ", Hv, ", expected a multiple of the key heads ", Hk, ", up to 1024");
    SX_CHECK((Dk == 64 || Dk == 128) && Dv >= 16 && Dv <= 1024 && Dv % 16 == 0, "key_dim = ", Dk, " (64 or 128), dim = ", Dv, " (a multiple of 16, up to 1024)");
    SX_CHECK(max_count >= 1 && max_count <= kMaxNew, "max_count = ", max_count, ", expected 1..", kMaxNew);
    SX_CHECK(path == nullptr || path_ld >= max_count, "path_ld = ", path_ld, " < max_count = ", max_count);
    SX_CHECK(slots >= 1 && slots <= 0x7fffffff && (slot != nullptr || slots >= batch), "slots = ", slots, " for batch = ", batch);
    SX_CHECK(k->token >= 0 && k->head >= 0 && k->layer >= 0 && k->token % 8 == 0 && k->head % 8 == 0 && k->layer % 8 == 0 && k->token <= (int64_t)1 << 32 &&
                 k->head <= (int64_t)1 << 32 && k->layer <= (int64_t)1 << 40,
             "strides of k must be multiples of 8");
    const int64_t one = Hv * Dk * Dv;
    SX_CHECK(state_slot >= one && state_slot % 4 == 0 && state_layer % 4 == 0 && state_slot <= (int64_t)1 << 40 && state_layer >= 0 && state_layer <= (int64_t)1 << 44,
             "state strides ", state_layer, ", ", state_slot);
    SX_CHECK(rows_apart(one, {{layers, state_layer}, {slots, state_slot}}), "states overlap");
    SX_CHECK(aligned(k->p, 16) && aligned(u, 16) && aligned(state, 16) && aligned(decay, 4) && aligned(starts, 4) && aligned(count, 4) && aligned(path, 4) && aligned(slot, 4),
             "k, u and state must be 16-byte aligned, the others 4-byte");
    const int64_t sb = 4 * ((layers - 1) * state_layer + (slots - 1) * state_slot + one);
    SX_CHECK(apart(state, sb, k->p, 2 * ((layers - 1) * k->layer) + span(*k, T, Hk, Dk)) && apart(state, sb, u, 4 * layers * T * Hv * Dv) &&
                 apart(state, sb, decay, 4 * layers * T * Hv) && apart(state, sb, starts, 4 * (batch + 1)) && apart(state, sb, count, 4 * batch) &&
                 (path == nullptr || apart(state, sb, path, 4 * ((batch - 1) * path_ld + max_count))) && (slot == nullptr || apart(state, sb, slot, 4 * batch)),
             "the states overlap another argument");
    const int64_t waves = Dv / 16 * Hv * batch * layers, blocks = (waves + 3) / 4;
    SX_CHECK(blocks <= 0x7fffffff, "layers = ", layers, " of batch = ", batch, ": too many states");
    const CommitArgs a{static_cast<const uint16_t *>(k->p), u, decay, state, slot, starts, count, path, err, k->layer, k->token, k->head, T * Hv * Dv,
                       T * Hv, state_layer, state_slot, path_ld, (int32_t)T, (int32_t)Hv, (int32_t)(Hv / Hk), (int32_t)Dv, (int32_t)batch, (int32_t)slots,
                       (int32_t)max_count, (int32_t)layers};
    if (Dk == 64) delta_commit_kernel<64><<<(unsigned)blocks, 256, 0, stream_of(stream)>>>(a);
    else delta_commit_kernel<128><<<(unsigned)blocks, 256, 0, stream_of(stream)>>>(a);
    SX_LAUNCHED("gated_delta_commit T=", T, " batch=", batch);
    return SX_OK;
}
