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
// sequence: 8192 tokens, 32 heads of 128: 99 + 259 us, 2.0 us a chunk (the matrix unit busy 0.18 of it; 1.2 us without any loads,
// which are 100 KB a chunk and compute unit).
//
// Operands: a result of the matrix unit has four consecutive rows a lane, an operand eight consecutive values of a row. The
// rows of two result tiles are dealt out so that a lane's four of the one and four of the other are eight consecutive
// ones: row 4 g + r of tile s stands for 8 g + 4 s + r. So the state, V - e^G K S and U become operands where they are.
// FP32 values enter as three BF16 terms, which together are the value; of a product of two such values the six largest of the nine
// products are taken (what is left is under 2^-22 of it).
//
// Tokens that are no numbers, and corrections too large for one: a triangular product would carry them to the tokens before them in
// the chunk. They are taken out and everything from them on (a value's or a correction's: in its column) is NaN, as the rule has it.
#include "gated_delta.hpp"

#include <type_traits>

namespace sx {
namespace delta {
namespace {

constexpr int kC = 64, kPitch = kC + 4;
constexpr int kBlocksT = 6;  // (row tile, pair of column tiles) with anything in it: 1, 1, 2, 2
constexpr int64_t kTBytes = kBlocksT * 3 * 1024 /* BF16 terms */, kPBytes = kBlocksT * 2 * 1024, kHeadBytes = kTBytes + kPBytes + 1024;

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
    uint8_t *keys;   // [chunk slots][Hk] 3 Dk 128: K^T, K and Q as operands: K^T [Dk / 16][2][64 lanes][8], K and Q [4 tiles][4][64 lanes][Dk / 16]
};
template <int DK>
constexpr int kKeyBytes = DK * kC * 2;  // of one of the three

// A sequence's chunks take slots starts[b] / 64 + b on: enough for a last chunk that is not full, where starts rise.
__device__ __forceinline__ int64_t first_slot(int t0, int b) { return t0 / kC + b; }

// The token that result row 4 g + r of tile ti stands for, and that of operand row m.
__device__ __forceinline__ constexpr int token_of(int ti, int g, int r) { return 32 * (ti >> 1) + 8 * g + 4 * (ti & 1) + r; }
__device__ __forceinline__ int token_at(int ti, int m) { return token_of(ti, m >> 2, m & 3); }

template <int DK>
__global__ void __launch_bounds__(256, 4) delta_prepare_kernel(const Args a, const Work w) {
    constexpr int KS = DK / 32;
    // At becomes T, P the keys' transpose, once they have been read: four blocks a compute unit
    __shared__ __attribute__((aligned(16))) float At[kC * kPitch], P[kC * kPitch];
    float *const Tm = At;
    __shared__ double path[kC];
    __shared__ float rk[kC], rq[kC], beta[kC];
    __shared__ uint64_t use_mask, key_mask;  // tokens that count; those whose key does, whatever this head's gates are
    __shared__ int found, falls;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g4 = lane >> 4;
    const int64_t slot = blockIdx.x / a.Hv;
    const int h = blockIdx.x % a.Hv, hk = h / a.rep;
    // the sequence whose chunk this is: the lowest whose words say so, if starts have not fallen before it. Up to there they only
    // rise, so it is the only one; sequences behind a falling start are impossible (sequence())
    int b = 0, t0 = 0, n = 0;
    auto mine_is = [&](int i) {
        t0 = a.starts[i];
        const int t1 = a.starts[i + 1];
        const int64_t f = first_slot(t0, i);
        if (t0 < 0 || t1 <= t0 || t1 > a.T || t1 - t0 > a.max_len || slot < f) return false;
        n = t1 - t0 - (int)(slot - f) * kC;
        return n > 0;
    };
    if (a.B == 1) {
        if (!mine_is(0)) return;
    } else {
        if (threadIdx.x == 0) found = falls = a.B;
        __syncthreads();
        for (int i = threadIdx.x; i < a.B; i += 256) {
            if (a.starts[i + 1] < a.starts[i]) atomicMin(&falls, i);
            if (mine_is(i)) atomicMin(&found, i);
        }
        __syncthreads();
        b = found;
        if (b >= falls) return;
        mine_is(b);
    }
    const int64_t row0 = t0 + (slot - first_slot(t0, b)) * kC;
    n = min(n, kC);
    float g = 0.f, be = 0.f;  // requested before anything is waited for
    if (wave == 0 && lane < n) gates(a, row0 + lane, h, g, be);
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
        rk[wave * 16 + n16] = key_scale(a, kk);
        rq[wave * 16 + n16] = query_scale(a, qq);
    }
    __syncthreads();
    if (wave == 0) {
        const uint64_t km = __ballot(lane < n && finite(rk[lane]));
        if (lane == 0) key_mask = km;
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
    __syncthreads();  // every wave has read At
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
        bf16x8 ts[3];
        split(t8, ts);
#pragma unroll
        for (int s = 0; s < 3; ++s) *reinterpret_cast<bf16x8 *>(head + (blk * 3 + s) * 1024 + lane * 16) = ts[s];
#pragma unroll
        for (int s = 0; s < 2; ++s)
            *reinterpret_cast<f32x4 *>(head + kTBytes + (blk * 2 + s) * 1024 + lane * 16) = f32x4{p8[4 * s], p8[4 * s + 1], p8[4 * s + 2], p8[4 * s + 3]};
    }
    if (h % a.rep != 0) return;
    // The key head's K and Q, their rows in the order of the tiles, and K^T: row dk, eight tokens a lane. (Read from the caller's rows,
    // half a line of each, they cost the scan 45 us of a prompt of 8192 tokens.)
    uint8_t *keys = w.keys + (slot * a.Hk + hk) * (3 * kKeyBytes<DK>);
    {
        const int i = wave * 16 + n16, at = 2 * (i >> 5) + (i >> 2 & 1), m = 4 * (i >> 3 & 3) + (i & 3);  // tile and row of token i
        const bool in = key_mask >> i & 1;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const u32x4 kx = in ? __builtin_bit_cast(u32x4, mine[ks]) : none, qx = __builtin_bit_cast(u32x4, Q[ks]);
            if constexpr (DK == 128) {
                const int to = ((at * 4 + ks) * 64 + m + 16 * g4) * 16;
                *reinterpret_cast<u32x4 *>(keys + kKeyBytes<DK> + to) = kx;
                *reinterpret_cast<u32x4 *>(keys + 2 * kKeyBytes<DK> + to) = qx;
            } else {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int to = ((at * 4 + 2 * ks + (g4 >> 1)) * 64 + m + 16 * ((g4 & 1) * 2 + half)) * 8;
                    *reinterpret_cast<u32x2 *>(keys + kKeyBytes<DK> + to) = u32x2{kx[2 * half], kx[2 * half + 1]};
                    *reinterpret_cast<u32x2 *>(keys + 2 * kKeyBytes<DK> + to) = u32x2{qx[2 * half], qx[2 * half + 1]};
                }
            }
        }
    }
    static_assert(DK * kPitch * 2 <= sizeof(P));
    uint16_t *kt = reinterpret_cast<uint16_t *>(P);
    __syncthreads();  // every wave has read P
    const bool count = key_mask >> (wave * 16 + n16) & 1;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const u32x4 x = __builtin_bit_cast(u32x4, mine[ks]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            kt[(ks * 32 + g4 * 8 + j) * kPitch + wave * 16 + n16] = count ? (uint16_t)(x[j / 2] >> (16 * (j & 1))) : (uint16_t)0;
    }
    __syncthreads();
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

// What a state wave needs of a chunk from memory.
template <int TS>
struct StateChunk {
    bf16x8 K[4];             // 4 TS values of a token
    bf16x8 T[2][3];
    bf16x8 KT[TS][2];
    f32x4 in, keep;          // of the wave's four tokens a lane
    uint16_t v[4];
    float fade;
    int32_t bad;
    uint64_t use;
};
// And an output wave.
struct OutChunk {
    bf16x8 Q[4];
    f32x4 P[2][2];  // FP32: as three terms they are half as many bytes again, and the scan of 8192 tokens took 274 us for 255
    f32x4 out;
};

__device__ __forceinline__ u32x4 load16(const void *base, uint32_t off) { return *reinterpret_cast<const u32x4 *>(static_cast<const uint8_t *>(base) + off); }
__device__ __forceinline__ u32x2 load8(const void *base, uint32_t off) { return *reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(base) + off); }
template <int TS>
__device__ __forceinline__ bf16x8 load_piece(const void *base, uint32_t off) {  // 4 TS values, the rest zero
    if constexpr (TS == 2) {
        return __builtin_bit_cast(bf16x8, load16(base, off));
    } else {
        const u32x2 x = load8(base, off);
        return __builtin_bit_cast(bf16x8, u32x4{x[0], x[1], 0u, 0u});
    }
}

// Eight tokens of a column from two tiles of four, as an operand.
__device__ __forceinline__ bf16x8 pair_of(const u32x2 (*from)[64], int p) {
    const u32x2 x = from[2 * p][threadIdx.x & 63], y = from[2 * p + 1][threadIdx.x & 63];
    return __builtin_bit_cast(bf16x8, u32x4{x[0], x[1], y[0], y[1]});
}

// Waves 0 to 3 carry the state, waves 4 to 7 make the outputs from what those leave in LDS, a chunk's products of Q and P beside
// the next one's of K: alone on its SIMD a wave that did both took twice as long for a chunk.
template <int DK>
__global__ void __launch_bounds__(512) delta_scan_kernel(const Args a, const Work w, int pairs8) {
    constexpr int TS = DK / 64;  // tiles of the state's rows a state wave has
    __shared__ __attribute__((aligned(16))) f32x4 xs[4][4][64];  // [wave][tile]: K S over the wave's rows
    __shared__ __attribute__((aligned(16))) u32x4 ss[4][3][64];  // the state's rows of each wave as operands
    __shared__ __attribute__((aligned(16))) u32x2 rs[3][4][64], us[3][4][64], ks[3][4][64];
    __shared__ int poison[16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wt = wave & 3, n16 = lane & 15, g4 = lane >> 4;
    const int pair = blockIdx.x % pairs8, b = pair / a.Hv, h = pair % a.Hv, hk = h / a.rep;
    if (b >= a.B) return;
    const int col = (int)(blockIdx.x / pairs8) * 16 + n16;
    const Seq s = sequence(a.starts, a.slot, b, a.B, a.T, a.max_len, a.slots, true);
    if (blockIdx.x / pairs8 == 0 && h == 0 && threadIdx.x == 0) tell(s, b, a.err);
    if (s.n == 0) return;
    uint16_t *const op = a.out + s.t0 * a.o_t + h * a.o_h;
    if (!s.ok) {
        for (int i = threadIdx.x >> 4; i < s.n; i += 32) op[i * a.o_t + col] = 0x7fc0;
        return;
    }
    if (threadIdx.x < 16) poison[threadIdx.x] = 0x7fffffff;
    const int chunks = (s.n + kC - 1) / kC;
    const int64_t slot0 = first_slot(s.t0, b);
    const uint8_t *const heads = w.heads + (slot0 * a.Hv + h) * kHeadBytes, *const keys = w.keys + (slot0 * a.Hk + hk) * (3 * kKeyBytes<DK>);
    const uint16_t *const vp = a.v + s.t0 * a.v_t + h * a.v_h;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const uint32_t at16 = lane * 16;
    const int mine = token_of(wt, g4, 0);  // the first of this lane's four tokens
    __syncthreads();                        // poison
    // The barriers of a chunk, which all eight waves pass: behind the first xs and ss are there, behind the second rs, behind the
    // third us and ks. What they hold is read before the next barrier but one, and written again behind it.
    // PAIRS: of column tiles in the wave's rows of T and P. Each piece of a chunk is requested as soon as the one two chunks before
    // it has been used, into its registers: one chunk ahead, the loads' latency was on the way of every chunk.
    auto carry = [&](auto count) __attribute__((always_inline)) {
        constexpr int PAIRS = decltype(count)::value;
        float *state = a.state + s.slot * a.s_slot + ((int64_t)h * DK + 16 * TS * wave + 4 * TS * g4) * a.Dv + col;
        f32x4 S[TS];
#pragma unroll
        for (int t = 0; t < TS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) S[t][r] = state[(int64_t)(4 * t + r) * a.Dv];
        // byte offsets of a whole chunk's values from its first
        const uint32_t vstep = (uint32_t)a.v_t * 2, vcol = col * 2;
        uint32_t vo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) vo[i] = (mine + i) * vstep + vcol;
        StateChunk<TS> now;
        // past the last chunk: the last one again, not used
        auto fetch_k = [&](int c, StateChunk<TS> &o) __attribute__((always_inline)) {
            c = min(c, chunks - 1);
            const uint8_t *key = keys + (int64_t)c * a.Hk * (3 * kKeyBytes<DK>) + kKeyBytes<DK> + wave * (512 * TS);
#pragma unroll
            for (int i = 0; i < 4; ++i) o.K[i] = load_piece<TS>(key + i * (2048 * TS), lane * (8 * TS));
        };
        auto fetch_v = [&](int c, StateChunk<TS> &o) __attribute__((always_inline)) {
            c = min(c, chunks - 1);
            const uint8_t *vc = reinterpret_cast<const uint8_t *>(vp + (int64_t)c * kC * a.v_t);
            const int left = s.n - 1 - c * kC;
            if (left >= kC - 1) {
#pragma unroll
                for (int i = 0; i < 4; ++i) o.v[i] = *reinterpret_cast<const uint16_t *>(vc + vo[i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) o.v[i] = *reinterpret_cast<const uint16_t *>(vc + min(mine + i, left) * vstep + vcol);
            }
            const Words *words = reinterpret_cast<const Words *>(heads + (int64_t)c * a.Hv * kHeadBytes + kTBytes + kPBytes);
            o.in = __builtin_bit_cast(f32x4, load16(words->in, mine * 4));
            o.keep = __builtin_bit_cast(f32x4, load16(words->keep, mine * 4));
            o.fade = words->fade, o.bad = words->bad, o.use = words->use;
        };
        auto fetch_t = [&](int c, StateChunk<TS> &o) __attribute__((always_inline)) {
            c = min(c, chunks - 1);
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) {
                const uint8_t *blk = heads + (int64_t)c * a.Hv * kHeadBytes + block_of(wave, p) * (3 * 1024);
#pragma unroll
                for (int i = 0; i < 3; ++i) o.T[p][i] = __builtin_bit_cast(bf16x8, load16(blk, at16 + i * 1024));
            }
        };
        auto fetch_kt = [&](int c, StateChunk<TS> &o) __attribute__((always_inline)) {
            c = min(c, chunks - 1);
            const uint8_t *key = keys + (int64_t)c * a.Hk * (3 * kKeyBytes<DK>) + wave * TS * 2048;
#pragma unroll
            for (int t = 0; t < TS; ++t)
#pragma unroll
                for (int p = 0; p < 2; ++p) o.KT[t][p] = __builtin_bit_cast(bf16x8, load16(key + t * 2048, at16 + p * 1024));
        };
        auto put = [&](u32x2 (*to)[4][64], int i, float (&r)[4]) __attribute__((always_inline)) {  // the leading bits; r: what is left
            to[i][wave][lane] = u32x2{tops(__float_as_uint(r[0]), __float_as_uint(r[1])), tops(__float_as_uint(r[2]), __float_as_uint(r[3]))};
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] -= __uint_as_float(__float_as_uint(r[j]) & 0xFFFF0000u);
        };
        auto chunk = [&](int c, StateChunk<TS> &now) __attribute__((always_inline)) {
            float s8[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) s8[j] = S[0][j], s8[4 + j] = TS == 2 ? S[TS - 1][j] : 0.f;
            bf16x8 so[3];
            split(s8, so);
#pragma unroll
            for (int i = 0; i < 3; ++i) ss[wave][i][lane] = __builtin_bit_cast(u32x4, so[i]);
            f32x4 X[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) X[t] = mfma(now.K[t], so[2], zero);
#pragma unroll
            for (int t = 0; t < 4; ++t) X[t] = mfma(now.K[t], so[1], X[t]);
#pragma unroll
            for (int t = 0; t < 4; ++t) X[t] = mfma(now.K[t], so[0], X[t]);
            fetch_k(c + 1, now);
#pragma unroll
            for (int t = 0; t < 4; ++t) xs[wave][t][lane] = X[t];
            lds_barrier();
            // this wave's 16 tokens: what the state does not explain of them
            const f32x4 x = (xs[0][wave][lane] + xs[1][wave][lane]) + (xs[2][wave][lane] + xs[3][wave][lane]);
            float r[4];
            bool odd = now.bad < kC;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                r[j] = bf16_to_f32(now.v[j]) - now.in[j] * x[j];
                odd |= !finite(r[j]);
            }
            if (now.use != ~0ull || __any(odd)) {
                int at = now.bad;
#pragma unroll
                for (int j = 3; j >= 0; --j) {
                    const bool use = now.use >> (mine + j) & 1;
                    if (use && !finite(r[j])) at = min(at, mine + j);
                    r[j] = use && finite(r[j]) ? r[j] : 0.f;
                }
                if (at < kC) atomicMin(&poison[n16], c * kC + at);
            }
            const float fade = now.fade;
            const f32x4 keep = now.keep;
            fetch_v(c + 1, now);
#pragma unroll
            for (int i = 0; i < 3; ++i) put(rs, i, r);
            lds_barrier();
            // U = T r
            f32x4 u = zero, u2 = zero;
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) {
                const bf16x8 r0 = pair_of(rs[0], p), r1 = pair_of(rs[1], p), r2 = pair_of(rs[2], p);
                u2 = mfma(now.T[p][2], r0, u2), u = mfma(now.T[p][1], r0, u);
                u2 = mfma(now.T[p][1], r1, u2), u = mfma(now.T[p][0], r1, u);
                u2 = mfma(now.T[p][0], r2, u2), u = mfma(now.T[p][0], r0, u);
            }
            fetch_t(c + 1, now);
            u += u2;
            float uu[4], uk[4];
            odd = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) uu[j] = u[j], uk[j] = u[j] * keep[j], odd |= !finite(uu[j]);
            if (__any(odd)) {  // too large for FP32
#pragma unroll
                for (int j = 3; j >= 0; --j) {
                    if (finite(uu[j])) continue;
                    atomicMin(&poison[n16], c * kC + mine + j);
                    uu[j] = uk[j] = 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < 3; ++i) put(ks, i, uk);
#pragma unroll
            for (int i = 0; i < 3; ++i) put(us, i, uu);
            lds_barrier();
#pragma unroll
            for (int t = 0; t < TS; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) S[t][j] *= fade;
#pragma unroll
            for (int i = 2; i >= 0; --i)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const bf16x8 o = pair_of(ks[i], p);
#pragma unroll
                    for (int t = 0; t < TS; ++t) S[t] = mfma(now.KT[t][p], o, S[t]);
                }
            fetch_kt(c + 1, now);
        };
        auto fetch = [&](int c, StateChunk<TS> &o) __attribute__((always_inline)) { fetch_k(c, o), fetch_v(c, o), fetch_t(c, o), fetch_kt(c, o); };
        fetch(0, now);
        for (int c = 0; c < chunks; ++c) chunk(c, now);
        const bool lost = poison[n16] != 0x7fffffff;
#pragma unroll
        for (int t = 0; t < TS; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) state[(int64_t)(4 * t + r) * a.Dv] = lost ? qnan() : S[t][r];
    };
    auto output = [&](auto count) __attribute__((always_inline)) {
        constexpr int PAIRS = decltype(count)::value;
        const uint32_t ostep = (uint32_t)a.o_t * 2;
        uint32_t oo[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) oo[r] = (mine + r) * ostep + col * 2;
        OutChunk now;
        auto fetch_q = [&](int c, OutChunk &o) __attribute__((always_inline)) {
            c = min(c, chunks - 1);
            const uint8_t *key = keys + (int64_t)c * a.Hk * (3 * kKeyBytes<DK>) + 2 * kKeyBytes<DK> + wt * (2048 * TS);
#pragma unroll
            for (int i = 0; i < 4; ++i) o.Q[i] = load_piece<TS>(key + i * (512 * TS), lane * (8 * TS));
            o.out = __builtin_bit_cast(f32x4, load16(reinterpret_cast<const Words *>(heads + (int64_t)c * a.Hv * kHeadBytes + kTBytes + kPBytes)->out, mine * 4));
        };
        auto fetch_p = [&](int c, OutChunk &o) __attribute__((always_inline)) {
            c = min(c, chunks - 1);
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) {
                const uint8_t *blk = heads + (int64_t)c * a.Hv * kHeadBytes + kTBytes + block_of(wt, p) * 2048;
#pragma unroll
                for (int i = 0; i < 2; ++i) o.P[p][i] = __builtin_bit_cast(f32x4, load16(blk, at16 + i * 1024));
            }
        };
        auto chunk = [&](int c, OutChunk &now) __attribute__((always_inline)) {
            lds_barrier();
            f32x4 Y = zero, Y2 = zero;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                Y2 = mfma(now.Q[i], __builtin_bit_cast(bf16x8, ss[i][2][lane]), Y2);
                Y2 = mfma(now.Q[i], __builtin_bit_cast(bf16x8, ss[i][1][lane]), Y2);
                Y = mfma(now.Q[i], __builtin_bit_cast(bf16x8, ss[i][0][lane]), Y);
            }
            lds_barrier();
            f32x4 O, O2 = zero;
#pragma unroll
            for (int r = 0; r < 4; ++r) O[r] = now.out[r] * (Y[r] + Y2[r]);
            fetch_q(c + 1, now);
            bf16x8 P[PAIRS][3];
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) {
                float p8[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) p8[j] = now.P[p][0][j], p8[4 + j] = now.P[p][1][j];
                split(p8, P[p]);
            }
            lds_barrier();
            const int from = poison[n16] - c * kC, left = s.n - c * kC;
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) {
                const bf16x8 u0 = pair_of(us[0], p), u1 = pair_of(us[1], p), u2 = pair_of(us[2], p);
                O2 = mfma(P[p][2], u0, O2), O = mfma(P[p][1], u0, O);
                O2 = mfma(P[p][1], u1, O2), O = mfma(P[p][0], u1, O);
                O2 = mfma(P[p][0], u2, O2), O = mfma(P[p][0], u0, O);
            }
            fetch_p(c + 1, now);
            uint8_t *oc = reinterpret_cast<uint8_t *>(op + (int64_t)c * kC * a.o_t);
            // Always four stores, of rows past the sequence's end too, which the buffer's size leaves out: stores that a branch skips
            // would make the next chunk's Q wait for all that is in flight.
            const auto rows = __builtin_amdgcn_make_buffer_rsrc(oc, 0, (int)((uint32_t)min(left, kC) * ostep), 0x00020000);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float o = mine + r >= from ? qnan() : O[r] + O2[r];
                __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, (__bf16)o), rows, (int)oo[r], 0, 0);
            }
        };
        fetch_q(0, now), fetch_p(0, now);
        for (int c = 0; c < chunks; ++c) chunk(c, now);
    };
    if (wave < 2) carry(std::integral_constant<int, 1>{});
    else if (wave < 4) carry(std::integral_constant<int, 2>{});
    else if (wave < 6) output(std::integral_constant<int, 1>{});
    else output(std::integral_constant<int, 2>{});
}

}  // namespace

size_t prefill_bytes(int64_t T, int64_t B, int64_t Hk, int64_t Hv, int64_t Dk) {
    return (size_t)((T / kC + B) * (Hv * kHeadBytes + Hk * (3 * Dk * kC * 2)));
}

void prefill(const Args &a, int Dk, void *ws, hipStream_t s) {
    const int64_t slots = a.T / kC + a.B;
    const Work w{static_cast<uint8_t *>(ws), static_cast<uint8_t *>(ws) + slots * a.Hv * kHeadBytes};
    // the blocks of one head's columns run on one XCD (block i: i % 8), whose L2 then has the chunk's T, P and K once
    const int pairs8 = (a.B * a.Hv + 7) / 8 * 8;
    const unsigned prep = (unsigned)(a.Hv * slots);
    if (Dk == 64) {
        delta_prepare_kernel<64><<<prep, 256, 0, s>>>(a, w);
        delta_scan_kernel<64><<<(unsigned)(pairs8 * (a.Dv / 16)), 512, 0, s>>>(a, w, pairs8);
    } else {
        delta_prepare_kernel<128><<<prep, 256, 0, s>>>(a, w);
        delta_scan_kernel<128><<<(unsigned)(pairs8 * (a.Dv / 16)), 512, 0, s>>>(a, w, pairs8);
    }
}

}  // namespace delta
}  // namespace sx
