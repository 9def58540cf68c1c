// Attention of a tree of drafted tokens over a paged cache (the attention of a verify step).
//
// Row r = (drafted token t of sequence b, query head h) attends the L_b cached tokens of its sequence, all of them, and
// the drafted tokens of the same sequence that its mask names: o = sum_j p_j v_j, p = softmax_j(scale * q . k_j).
// A plain decode step is a tree of one token.
//
// The cost is the cache: 2 L Hkv D values read once, against 4 R L D flops for the R = tokens * (query heads a key
// head) rows that share them. A block therefore takes all rows of a sequence and key head (up to its tile of rows) and
// streams stages of keys and values (32 KB each; 16 KB where two blocks share a compute unit) through LDS, two deep: the loads of the next stage are
// asynchronous and in flight, without registers, for as long as this stage is worked on.
//   S^T = K Q^T: 16 keys are the A operand, Q^T stays in registers as the B operand; a lane gets 4 keys of a 16-key
//   tile for one row.
//   O^T += V^T P^T: those 2 x 4 keys of a 32-key step are, with the keys of the product permuted alike on both sides,
//   already the B operand, so P never moves between lanes. V^T needs 8 keys of one dim a lane: a lane reads the same
//   D / 16 dims of its 8 keys and pairs the keys with one v_perm a dword.
// The waves of a block split a stage's 32-key steps (WK ways) and the rows (WR ways). Scores, maxima, sums
// and O are FP32; how P enters the matrix unit is said at as_operand.
//
// Work: a unit is one stage of a sequence's cached keys, or its drafted tokens, for one row group (16 NT WR rows); the
// units of all sequences form one list that the blocks of a key head share in equal runs, whatever the lengths are
// (they are on the device: a captured graph replays with other ones). A block whose run covers a pair of sequence and
// row group whole writes its rows; else it leaves a partial (at most two a block: its run's first and last pair) that
// tree_attn_join_kernel adds up in the order of the list, so the result does not depend on the schedule.
//
// Measured (both kernels): 131,072 keys, 8 key heads of 128, 4 rows each: 112 to 115 us, 4.7 TB/s; 65,536 keys: 65 us, so
// 5.4 to 5.8 TB/s beyond them and 15 to 19 us that do not grow with the keys. Up to 64 rows the time hardly moves (71 us for
// 65,536 keys), above it grows with the rows (96: 79 us; 256: 123 us, 0.56 PFLOP/s).
#include "common.hpp"
#include "kv_cache.hpp"
#include "route_impl.hpp"

#include <algorithm>
#include <cmath>

namespace sx {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 32, kMaxSeqs = 1024, kMaxNew = 256, kJoinThreads = 256;
constexpr float kNegInf = -INFINITY;

struct Args {
    const uint16_t *q, *kn, *vn;
    const uint8_t *kc, *vc;
    const int32_t *table, *lens, *starts;
    const uint64_t *mask;
    uint16_t *out;
    float *lse;
    float *part_o, *part_ml;  // [Hkv][2 nb] partials: O [rows, D], then (m, l) [rows, 2]
    uint32_t *prefix;         // [B + 1]: units ahead of each sequence
    uint32_t *err;
    int64_t q_t, q_h, kn_t, kn_h, vn_t, vn_h;  // element strides: token, head
    int64_t kc_p, vc_p;                        // byte strides of the caches: page,
    int64_t kc_h, vc_h;                        // head,
    int32_t kc_t, vc_t;                        // token (a page's span fits 31 bits)
    int64_t out_t, out_h, lse_t, table_ld, mask_ld;
    int32_t B, T, G, P, pages, page_shift, max_new, nb, heads;
    float scale, k_scale, v_scale;  // scale: softmax scale * log2(e)
};

// How a cache row of D values lies in a stage and in the operands.
template <int D, bool F8, int HS>  // HS: bytes of keys (of values) a stage
struct Lay {
    static constexpr int E = F8 ? 1 : 2, RB = D * E;                       // bytes of a value, of a row
    static constexpr int KEYS = HS / RB < 256 ? HS / RB : 256;  // keys a stage
    static constexpr int CH = RB / 16;                                     // 16-byte chunks a row
    static constexpr int VEC = D / 16, PE = F8 ? VEC : (VEC < 8 ? VEC : 8);  // dims a lane of a value row; in one piece
    static constexpr int VB = PE * E;                                      // bytes of a piece: 4, 8 or 16
    // keys: chunk c of row r lies at c ^ swz(r), so that the 16 rows of an operand read use all banks
    __device__ static constexpr int swz(int r) { return CH >= 16 ? r & 15 : (r / (16 / CH)) & (CH - 1); }
    // the dim of element e of value-operand row x (0..15)
    __device__ static constexpr int dim(int x, int e) { return e / PE * 16 * PE + x * PE + e % PE; }
    // the dims of a key row that lane group g brings to product step kk: an FP8 chunk is two steps
    __device__ static constexpr int k_dim(int kk, int g) { return F8 ? (kk >> 1) * 64 + g * 16 + (kk & 1) * 8 : kk * 32 + g * 8; }
};

// What a sequence asks for. A sequence whose words contradict the call (lengths past its table, token runs outside
// the packed rows) has no units and is reported.
struct Seq {
    int t0, n, L, rgs, chunks;
    bool bad;
};

template <int ROWS, int KEYS, int FRESH>
__device__ __forceinline__ Seq seq_of(const Args &a, int b) {
    Seq s;
    const int t0 = a.starts[b], t1 = a.starts[b + 1], L = a.lens[b];
    s.bad = t0 < 0 || t1 < t0 || t1 > a.T || t1 - t0 > a.max_new || L < 0 || ((int64_t)L > ((int64_t)a.P << a.page_shift));
    s.t0 = t0, s.n = s.bad ? 0 : t1 - t0, s.L = s.bad ? 0 : L;
    s.rgs = (s.n * a.G + ROWS - 1) / ROWS;
    s.chunks = s.n == 0 ? 0 : (s.n + FRESH - 1) / FRESH + (s.L + KEYS - 1) / KEYS;  // drafted stages, then cached ones
    return s;
}

__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, bool hi) {  // two e4m3 codes as two BF16
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
}

__device__ __forceinline__ uint32_t fp8_pair_f16(uint32_t w, bool hi) {  // as two FP16 (exact)
    return hi ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))
              : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
}

// The lane's number, made anew where it is asked for (no register held for it).
__device__ __forceinline__ int lane_anew() {
    int l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(l));
    return l;
}

// N dwords (1, 2, or a multiple of 4) from memory or LDS.
template <int N, typename P>
__device__ __forceinline__ void load_words(P p, uint32_t *w) {
    if constexpr (N == 1) {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else if constexpr (N == 2) {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        w[0] = u.x, w[1] = u.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 u = *reinterpret_cast<const u32x4 *>(p + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i + j] = u[j];
        }
    }
}

__device__ __forceinline__ void dma16(const void *src, void *lds) {
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

// The four lane groups' maximum or sum, in all of them.
__device__ __forceinline__ float over_g(float x, bool mx) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = mx ? fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])) : __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return mx ? fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1])) : __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A wave's rows: column n16 of NT tiles. l: this lane's share of the sum.
template <int D, int NT>
struct Acc {
    f32x4 o[NT][D / 16];
    float m[NT], l[NT];
};

// s: raw scores (-inf where a row does not see the key) of keys {4g + i, 16 + 4g + i}; leaves p = 2^(s ks - m) in s. m is
// a row's maximum, less kLift, at the last time that a p went over 2^kTop: sums and O grow by that factor at most, far
// inside FP32, and O is rescaled a few times a run and not at every new maximum. Where P becomes FP16 (F16) the lift puts
// the largest p at FP16's upper end: FP16 takes 2^-25 at most from a key, against a sum of 2^7 and more, so many keys far
// under a row's maximum count down to 2^-32 of it (65,536 keys a wave: 2^-16 of the largest value is lost at most).
template <int D, int NT, bool F16>
__device__ __forceinline__ void softmax_step(Acc<D, NT> &acc, float (&s)[NT][8], float ks) {
    constexpr float kLift = F16 ? 7.f : 0.f, kTop = F16 ? 15.f : 8.f;
    float mx[NT];
    bool up = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        mx[t] = fmaxf(fmaxf(fmaxf(s[t][0], s[t][1]), fmaxf(s[t][2], s[t][3])), fmaxf(fmaxf(s[t][4], s[t][5]), fmaxf(s[t][6], s[t][7])));
        up |= mx[t] * ks > acc.m[t] + kTop;
    }
    if (__any(up)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const float m = fmaxf(acc.m[t], over_g(mx[t], true) * ks - kLift);
            const float c = __builtin_amdgcn_exp2f(acc.m[t] - (m == kNegInf ? 0.f : m));
            acc.l[t] *= c, acc.m[t] = m;
#pragma unroll
            for (int e = 0; e < D / 16; ++e) acc.o[t][e] *= c;
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const float base = acc.m[t] == kNegInf ? 0.f : acc.m[t];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], ks, -base));
            sum += s[t][i];
        }
        acc.l[t] += sum;
    }
}

// Where O and Q leave few registers the operand reads are held two steps ahead of their products, not further: left to
// itself the scheduler brings a whole step's operands in at once and spills (a spill's wait counts the stage's loads too).
template <int D, int NT>
constexpr bool kTight = D * NT > 256;

// S^T of two 16-key tiles; frag(kt, kk): the key operand.
template <int D, int NT, typename F>
__device__ __forceinline__ void scores(F frag, const bf16x8 (&q)[NT][D / 32], float (&s)[NT][8]) {
    f32x4 c[2][NT];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int t = 0; t < NT; ++t) c[kt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int kAhead = 2, kSteps = D / 32;
    bf16x8 A[kSteps][2];
    if constexpr (kTight<D, NT>) {
#pragma unroll
        for (int kk = 0; kk < kAhead; ++kk) A[kk][0] = frag(0, kk), A[kk][1] = frag(1, kk);
    }
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) {
        if constexpr (kTight<D, NT>) {
            if (kk + kAhead < kSteps) A[kk + kAhead][0] = frag(0, kk + kAhead), A[kk + kAhead][1] = frag(1, kk + kAhead);
        } else {
            A[kk][0] = frag(0, kk), A[kk][1] = frag(1, kk);
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int t = 0; t < NT; ++t) c[kt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A[kk][kt], q[t][kk], c[kt][t], 0, 0, 0);
        if constexpr (kTight<D, NT>) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) s[t][i] = c[i >> 2][t][i & 3];
}

// P as the B operand. BF16 values: TERMS BF16 numbers that add up to p (one: 2^-9 of it is lost, two: 2^-17). E4M3 values
// are exact in FP16 too, so there one FP16 number does (2^-12; small ones: see softmax_step).
template <int NT, int TERMS, bool F16>
__device__ __forceinline__ void as_operand(const float (&p)[NT][8], float factor, bool scaled, u32x4 (&b)[TERMS][NT]) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if constexpr (F16) {
            f16x8 h;
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = (_Float16)p[t][i];
            b[0][t] = __builtin_bit_cast(u32x4, h);
        } else {
            bf16x8 hi, lo;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = scaled ? p[t][i] * factor : p[t][i];
                hi[i] = (__bf16)v;
                if constexpr (TERMS == 2) lo[i] = (__bf16)(v - (float)hi[i]);
            }
            b[0][t] = __builtin_bit_cast(u32x4, hi);
            if constexpr (TERMS == 2) b[1][t] = __builtin_bit_cast(u32x4, lo);
        }
    }
}

// O^T += V^T P^T for dims e, e + 1 of the lane's piece: w[j] holds them for key slot j.
template <int D, int NT, int TERMS, bool F16>
__device__ __forceinline__ void values_pair(Acc<D, NT> &acc, int e, const uint32_t (&w)[8], const u32x4 (&p)[TERMS][NT]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        u32x4 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], u ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int x = TERMS - 1; x >= 0; --x)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f32x4 &o = acc.o[t][e + u];
                if constexpr (F16) o = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, f), __builtin_bit_cast(f16x8, p[x][t]), o, 0, 0, 0);
                else o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, f), __builtin_bit_cast(bf16x8, p[x][t]), o, 0, 0, 0);
            }
    }
}

// The drafted tokens' values of one piece of dims that are not finite: a row that does not see such a token must not
// meet it (0 * inf is NaN in the matrix unit), so it leaves the operand and is added row by row. Rare: one ballot a key
// slot says so. x: the piece (PE BF16 dims) of key slot j in dwords.
template <int D, int NT, int PE, typename DimOf>
__device__ __forceinline__ void odd_values(Acc<D, NT> &acc, int e0, uint32_t (&x)[8][PE / 2], const float (&p)[NT][8],
                                           const uint32_t (&seen)[NT], float factor, const uint16_t *v_step, int64_t v_t, int count, DimOf dim) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < PE / 2; ++i) odd |= (x[j][i] & 0x7F80u) == 0x7F80u || (x[j][i] & 0x7F800000u) == 0x7F800000u;
        const uint64_t who = __ballot(odd);
        if (who == 0) continue;
        if ((who >> (16 * g)) & 0xFFFFu) {
#pragma unroll
            for (int i = 0; i < PE / 2; ++i) x[j][i] = 0;
        }
        for (int gg = 0; gg < 4; ++gg) {
            const int key = (j < 4 ? 0 : 16) + 4 * gg + (j & 3);
            if (!((who >> (16 * gg)) & 0xFFFFu) || key >= count) continue;  // uniform
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const float pk = __shfl(p[t][j], 16 * gg + (lane & 15)) * factor;
                if ((seen[t] >> key) & 1u) {
                    const uint16_t *row = v_step + key * v_t;
#pragma unroll
                    for (int e = 0; e < PE; ++e)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc.o[t][e0 + e][i] = fmaf(pk, bf16_to_f32(row[dim(4 * g + i, e0 + e)]), acc.o[t][e0 + e][i]);
                }
            }
        }
    }
}

// The natural logarithm of a row's sum of exp(score).
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? kNegInf : 0.6931471805599453f * m + logf(l); }

// The block's list of units: prefix sums over the sequences, and what the sequences ask for, in LDS.
struct List {
    uint32_t pre[kMaxSeqs + 1], wave_tot[8];
    int t0[kMaxSeqs], len[kMaxSeqs];
    uint16_t n[kMaxSeqs];
};

template <int ROWS, int KEYS, int FRESH, int THREADS>
__device__ __forceinline__ void scan_units(const Args &a, List &ls) {
    constexpr int kPer = kMaxSeqs / THREADS;
    const int tid = threadIdx.x, per = (a.B + THREADS - 1) / THREADS, b0 = tid * per, b1 = min(b0 + per, a.B);
    const bool first = blockIdx.x == 0 && blockIdx.y == 0;
    uint32_t units[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        units[i] = 0;
        if (b0 + i < b1) {
            const Seq s = seq_of<ROWS, KEYS, FRESH>(a, b0 + i);
            units[i] = (uint32_t)(s.rgs * s.chunks);
            ls.t0[b0 + i] = s.t0, ls.len[b0 + i] = s.L, ls.n[b0 + i] = (uint16_t)s.n;
            if (s.bad && first) report(a.err, (uint32_t)a.lens[b0 + i], (uint32_t)(b0 + i));
        }
        sum += units[i];
    }
    const uint32_t incl = routing::wave_incl_scan_u32(sum);
    if ((tid & 63) == 63) ls.wave_tot[tid >> 6] = incl;
    __syncthreads();
    uint32_t at = incl - sum;
    for (int w = 0; w < (tid >> 6); ++w) at += ls.wave_tot[w];
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (b0 + i < b1) {
            ls.pre[b0 + i] = at;
            if (first) a.prefix[b0 + i] = at;
            at += units[i];
            if (b0 + i == a.B - 1) {
                ls.pre[a.B] = at;
                if (first) a.prefix[a.B] = at;
            }
        }
    __syncthreads();
}

__device__ __forceinline__ int seq_at(const uint32_t *pre, int B, uint32_t u) {  // the b with pre[b] <= u < pre[b + 1]
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (pre[mid + 1] <= u) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

template <int D, int NT, int WR, int WK, int HS, bool F8>
__global__ void __launch_bounds__(64 * WR * WK, HS < 32768 || WR * WK > 4 ? 2 : 1) tree_attn_kernel(const Args a) {
    using C_ = Lay<D, F8, HS>;     // cached stages
    using N_ = Lay<D, false, HS>;  // drafted stages
    // BF16 values meet P in two terms where there are few rows and products to spare (at 16 rows and 65,536 keys the time
    // is the same), else in one, rounded as the values are: the output's error is its own rounding, or 1.4 times that (two
    // above 64 rows too: 8 to 23 % slower, 96 rows 78.7 -> 92 us)
    constexpr int kWaves = WR * WK, ROWS = 16 * NT * WR, KEYS = C_::KEYS, FRESH = N_::KEYS, VEC = D / 16, BF16_TERMS = ROWS <= 64 ? 2 : 1;
    static_assert(WK / 2 * WR <= 4, "an array for each pair of waves that meet");
    // one array a stage and operand, so that the wait-count pass tells a stage's loads apart from the other's
    __shared__ __attribute__((aligned(1024))) uint8_t k0[HS], k1[HS], v0[HS], v1[HS];
    __shared__ List ls;
    __shared__ float merge_ml[kWaves][16 * NT][2];
    scan_units<ROWS, KEYS, FRESH, 64 * kWaves>(a, ls);

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n16 = lane & 15, g = lane >> 4;
    const int wr = wave % WR, wk = wave / WR;
    const int kvh = blockIdx.y, page_mask = (1 << a.page_shift) - 1;
    const uint32_t U = ls.pre[a.B], nb = min((uint32_t)a.nb, U);  // as many runs as there are units to deal out: none is empty
    if (blockIdx.x >= nb) return;
    const uint32_t lo = (uint32_t)((uint64_t)U * blockIdx.x / nb), hi = (uint32_t)((uint64_t)U * (blockIdx.x + 1) / nb);

    for (uint32_t u = lo; u < hi;) {
        const int b = __builtin_amdgcn_readfirstlane(seq_at(ls.pre, a.B, u));
        const int L = __builtin_amdgcn_readfirstlane(ls.len[b]), n = __builtin_amdgcn_readfirstlane((int)ls.n[b]);
        const int t0 = __builtin_amdgcn_readfirstlane(ls.t0[b]);
        const int fresh = (n + FRESH - 1) / FRESH, chunks = fresh + (L + KEYS - 1) / KEYS;
        const int item = u - __builtin_amdgcn_readfirstlane((int)ls.pre[b]);
        const int rg = item / chunks, c0 = item % chunks, c1 = (int)min((uint32_t)chunks, c0 + (hi - u));
        const int R = n * a.G, row0 = rg * ROWS + wr * 16 * NT;
        const int s0 = max(c0 - fresh, 0), stages = max(c1 - fresh, 0) - s0;  // cached stages s0 .. s0 + stages - 1
        const bool mine = row0 < R;  // a wave with no rows of its own only loads
        bool bad_page = false;
        int odd_page = 0;

        Acc<D, NT> acc;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            acc.m[t] = kNegInf, acc.l[t] = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc.o[t][e] = f32x4{0.f, 0.f, 0.f, 0.f};
        }

        const int32_t *table = a.table + b * a.table_ld;
        const int last_tile = max(L - 1, 0) >> 4;
        // lane i: the page of the stage's 16-key tile i (a page holds whole tiles), clamped to the last tile with keys
        auto pages_of = [&](int c) __attribute__((always_inline)) {
            return table[(min(c * (KEYS / 16) + (lane & (KEYS / 16 - 1)), last_tile) << 4) >> a.page_shift];
        };
        // This wave's share of a stage's loads. tile_at(i): keys and values of its 16-key tile i, the row it starts at, and
        // how many rows further there are any. Rows past the last repeat it.
        auto issue = [&](auto lay, auto tile_at, int k_t, int v_t, uint8_t *kb, uint8_t *vb) __attribute__((always_inline)) {
            using L_ = decltype(lay);
            constexpr int kDma = L_::KEYS * L_::RB / 1024 / kWaves, RPI = 64 / L_::CH;  // loads a wave, rows a load
            static_assert(kDma >= 1 && 16 % RPI == 0, "a load's rows lie in one 16-key tile");
            const int ln = kTight<D, NT> ? lane_anew() : lane;  // addresses are made anew, not kept across stages
#pragma unroll
            for (int i = 0; i < kDma; ++i) {
                const int at = wave * kDma + i, r = (at * RPI) % 16 + ln / L_::CH, chunk = ln % L_::CH;
                const uint8_t *kp, *vp;
                int first, most;
                tile_at(at * RPI / 16, kp, vp, first, most);
                dma16(kp + (uint32_t)((first + min(r, most)) * k_t + (chunk ^ L_::swz(r)) * 16), kb + at * 1024);
                // values: LDS row 4 j + g holds key 4 g + j, so that an operand read takes four rows in a row
                const int key = (r & 3) * 4 + (r >> 2);
                dma16(vp + (uint32_t)((first + min(key, most)) * v_t + chunk * 16), vb + at * 1024);
            }
        };
        auto issue_cached = [&](int c, int pg, uint8_t *kb, uint8_t *vb) __attribute__((always_inline)) {
            if ((uint32_t)pg >= (uint32_t)a.pages) bad_page = true, odd_page = pg, pg = 0;
            issue(C_{}, [&](int tile, const uint8_t *&kp, const uint8_t *&vp, int &first, int &most) __attribute__((always_inline)) {
                const int64_t page = __builtin_amdgcn_readlane(pg, tile);
                const int gt = min(c * (KEYS / 16) + tile, last_tile);
                kp = a.kc + kvh * a.kc_h + page * a.kc_p, vp = a.vc + kvh * a.vc_h + page * a.vc_p;
                first = (gt << 4) & page_mask, most = L - 1 - gt * 16;
            }, a.kc_t, a.vc_t, kb, vb);
        };
        auto issue_fresh = [&](int c, uint8_t *kb, uint8_t *vb) __attribute__((always_inline)) {
            issue(N_{}, [&](int tile, const uint8_t *&kp, const uint8_t *&vp, int &first, int &most) __attribute__((always_inline)) {
                const int gt = min(c * (FRESH / 16) + tile, (n - 1) >> 4);
                kp = reinterpret_cast<const uint8_t *>(a.kn + t0 * a.kn_t + kvh * a.kn_h);
                vp = reinterpret_cast<const uint8_t *>(a.vn + t0 * a.vn_t + kvh * a.vn_h);
                first = gt << 4, most = n - 1 - gt * 16;
            }, (int)a.kn_t * 2, (int)a.vn_t * 2, kb, vb);
        };
        // with an FP8 cache O is kept in units of v_scale
        const float ks = F8 ? a.scale * a.k_scale : a.scale, v_unit = F8 ? a.v_scale : 1.f, inv_v = 1.f / v_unit;
        int pg = 0;
        if (c0 < fresh) issue_fresh(c0, k1, v1);
        if (stages > 0) {
            issue_cached(s0, pages_of(s0), k0, v0);
            pg = pages_of(s0 + 1);
        }
        // this wave's rows: Q^T as the B operand (rows past the last repeat it)
        bf16x8 q[NT][D / 32];
        const uint64_t *row_mask[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = min(row0 + t * 16 + n16, R - 1), tok = t0 + r / a.G, h = kvh * a.G + r % a.G;
            const uint16_t *qr = a.q + tok * a.q_t + h * a.q_h;
            row_mask[t] = a.mask + tok * a.mask_ld;
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) q[t][kk] = *reinterpret_cast<const bf16x8 *>(qr + C_::k_dim(kk, g));
        }
        // Q is waited for here, once, and not at every step behind the loads of the next stage
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) asm volatile("" : "+v"(q[t][kk]));
        // Stage c in kb, vb (keys first .. of `total`): this wave's 32-key steps. Drafted stages go by the rows' masks.
        auto work = [&](auto lay, auto drafted, int c, int total, float ks, const uint8_t *kb, const uint8_t *vb) __attribute__((always_inline)) {
            using L_ = decltype(lay);
            constexpr bool NEW = decltype(drafted)::value, E4 = F8 && !NEW;
#pragma unroll 1
            for (int st = wk; st < L_::KEYS / kStep; st += WK) {
                const int key0 = c * L_::KEYS + st * kStep;
                if (key0 >= total) break;
                const int ln = kTight<D, NT> ? lane_anew() : lane, n16_ = ln & 15, g_ = ln >> 4;  // nor LDS addresses across steps
                float s[NT][8];
                scores<D, NT>([&](int kt, int kk) __attribute__((always_inline)) {
                    const uint8_t *row = kb + (st * kStep + kt * 16 + n16_) * L_::RB;
                    if constexpr (!E4) {  // the dims of Q's operand, wherever the row keeps them
                        return *reinterpret_cast<const bf16x8 *>(row + ((C_::k_dim(kk, g_) / 8) ^ L_::swz(n16_)) * 16);
                    } else {
                        uint32_t w[2];
                        load_words<2>(row + (((kk >> 1) * 4 + g_) ^ L_::swz(n16_)) * 16 + (kk & 1) * 8, w);
                        return __builtin_bit_cast(bf16x8, u32x4{fp8_pair(w[0], false), fp8_pair(w[0], true), fp8_pair(w[1], false), fp8_pair(w[1], true)});
                    }
                }, q, s);
                uint32_t seen[NT];
                const int count = total - key0;
                if constexpr (NEW) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        seen[t] = (uint32_t)(row_mask[t][key0 >> 6] >> (key0 & 63));
                        if (count < kStep) seen[t] &= (1u << count) - 1u;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (!((seen[t] >> ((i >> 2) * 16 + 4 * g_ + (i & 3))) & 1u)) s[t][i] = kNegInf;
                    }
                } else if (count < kStep) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if ((i >> 2) * 16 + 4 * g_ + (i & 3) >= count) {
#pragma unroll
                            for (int t = 0; t < NT; ++t) s[t][i] = kNegInf;
                        }
                }
                softmax_step<D, NT, F8>(acc, s, ks);
                constexpr int TERMS = E4 ? 1 : BF16_TERMS;
                u32x4 p[TERMS][NT];
                as_operand<NT, TERMS, E4>(s, inv_v, F8 && NEW, p);
                // a lane's piece of a value row: with a BF16 row under an FP8 layout's dims, as many BF16 values
                constexpr int P0 = kTight<D, NT> && C_::PE > 4 ? C_::PE / 2 : C_::PE, W0 = P0 * L_::E / 4;
#pragma unroll
                for (int e0 = 0; e0 < VEC; e0 += P0) {
                    uint32_t x[8][W0];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        load_words<W0>(vb + (st * kStep + (j >> 2) * 16 + (j & 3) * 4 + g_) * L_::RB + C_::dim(n16_, e0) * L_::E, x[j]);
                    if constexpr (NEW)
                        odd_values<D, NT, P0>(acc, e0, x, s, seen, inv_v, a.vn + (t0 + key0) * a.vn_t + kvh * a.vn_h, a.vn_t, count,
                                              [](int r, int e) { return C_::dim(r, e); });
#pragma unroll
                    for (int e = 0; e < P0; e += 2) {
                        uint32_t w[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[j] = E4 ? fp8_pair_f16(x[j][e / 4], e & 2) : x[j][e / 2];
                        values_pair<D, NT, TERMS, E4>(acc, e0 + e, w, p);
                    }
                    if constexpr (kTight<D, NT>) __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        // Every wave waits for its own loads, and the barrier makes all of them visible; it also says that what the next
        // loads overwrite has been read.
        auto arrived = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
        for (int c = c0; c < min(c1, fresh); ++c) {  // more than one only for trees past a stage
            if (c > c0) {
                __syncthreads();
                issue_fresh(c, k1, v1);
            }
            arrived();
            if (mine) work(N_{}, std::true_type{}, c, n, a.scale, k1, v1);
        }
        auto stage = [&](int i, const uint8_t *kb, const uint8_t *vb, uint8_t *kn, uint8_t *vn) __attribute__((always_inline)) {
            arrived();
            if (i + 1 < stages) {
                issue_cached(s0 + i + 1, pg, kn, vn);
                if (i + 2 < stages) pg = pages_of(s0 + i + 2);
            }
            if (mine) work(C_{}, std::false_type{}, s0 + i, L, ks, kb, vb);
        };
        for (int i = 0; i < stages; i += 2) {
            stage(i, k0, v0, k1, v1);
            if (i + 1 < stages) stage(i + 1, k1, v1, k0, v0);
        }
        if (const uint64_t who = __ballot(bad_page)) {  // every wave has looked at every page of its stages
            if (bad_page && lane == __builtin_ctzll(who)) report(a.err, (uint32_t)odd_page, (uint32_t)b);
            bad_page = true;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            acc.l[t] = over_g(acc.l[t], false);
            if (bad_page) acc.l[t] = qnan();
        }

        // ---- the key groups' results into group 0's: the upper half of the groups into the lower, until one is left.
        // The stages' arrays hold them (every wave is past its last stage once all pass the barrier). ----
#pragma unroll
        for (int half = WK / 2; half >= 1; half >>= 1) {
            const bool gives = wk >= half && wk < 2 * half, takes = wk < half;
            const int place = (gives ? wk - half : wk) * WR + wr;  // whose array: one for each pair of waves
            float *at = reinterpret_cast<float *>(place == 0 ? k0 : place == 1 ? k1 : place == 2 ? v0 : v1);
            float f1[NT], f2[NT];
            if (gives && g == 0) {
#pragma unroll
                for (int t = 0; t < NT; ++t) merge_ml[wave][t * 16 + n16][0] = acc.m[t], merge_ml[wave][t * 16 + n16][1] = acc.l[t];
            }
            constexpr int kParts = (16 * NT * D * 4 + HS - 1) / HS, kEach = VEC / kParts;  // O in as many parts as arrays hold
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                __syncthreads();
                if (gives) {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int e = 0; e < kEach; ++e)
                            *reinterpret_cast<f32x4 *>(at + ((t * kEach + e) * 64 + lane) * 4) = acc.o[t][part * kEach + e];
                }
                __syncthreads();
                if (!takes) continue;
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    if (part == 0) {
                        const float m2 = merge_ml[wave + half * WR][t * 16 + n16][0], l2 = merge_ml[wave + half * WR][t * 16 + n16][1];
                        const float m = fmaxf(acc.m[t], m2), base = m == kNegInf ? 0.f : m;
                        f1[t] = __builtin_amdgcn_exp2f(acc.m[t] - base), f2[t] = __builtin_amdgcn_exp2f(m2 - base);
                        acc.m[t] = m, acc.l[t] = acc.l[t] * f1[t] + l2 * f2[t];
                    }
#pragma unroll
                    for (int e = 0; e < kEach; ++e)
                        acc.o[t][part * kEach + e] = acc.o[t][part * kEach + e] * f1[t] +
                                                     *reinterpret_cast<const f32x4 *>(at + ((t * kEach + e) * 64 + lane) * 4) * f2[t];
                }
            }
        }
        __syncthreads();  // the arrays are free for the next pair's loads
        if (wk == 0 && mine) {
            constexpr int PE = C_::PE;
            const bool whole = c0 == 0 && c1 == chunks;
            const int64_t slot = ((int64_t)kvh * a.nb + blockIdx.x) * 2 + (u == lo ? 0 : 1);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const int in = wr * 16 * NT + t * 16 + n16, r = rg * ROWS + in;
                if (r >= R) continue;
                if (whole) {
                    const int tok = t0 + r / a.G, head = kvh * a.G + r % a.G;
                    const float inv = acc.l[t] == 0.f ? 0.f : v_unit / acc.l[t];  // nothing seen: zeros
                    uint16_t *row = a.out + tok * a.out_t + head * a.out_h;
#pragma unroll
                    for (int e0 = 0; e0 < VEC; e0 += PE) {
                        uint32_t w[2 * PE];  // dims dim(4 g, e0) ..: 4 runs of PE, one after the other
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < PE; e += 2)
                                w[(i * PE + e) / 2] = f32_to_bf16(acc.o[t][e0 + e][i] * inv) | (f32_to_bf16(acc.o[t][e0 + e + 1][i] * inv) << 16);
#pragma unroll
                        for (int i = 0; i < 2 * PE; i += 4)
                            *reinterpret_cast<u32x4 *>(row + C_::dim(4 * g, e0) + 2 * i) = u32x4{w[i], w[i + 1], w[i + 2], w[i + 3]};
                    }
                    if (a.lse != nullptr && g == 0) a.lse[tok * a.lse_t + head] = log_sum(acc.m[t], acc.l[t]);
                } else {
                    float *po = a.part_o + (slot * ROWS + in) * D;
#pragma unroll
                    for (int e0 = 0; e0 < VEC; e0 += PE)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < PE; e += 4)
                                *reinterpret_cast<f32x4 *>(po + C_::dim(4 * g + i, e0 + e)) =
                                    f32x4{acc.o[t][e0 + e][i], acc.o[t][e0 + e + 1][i], acc.o[t][e0 + e + 2][i], acc.o[t][e0 + e + 3][i]} * v_unit;
                    if (g == 0) {
                        float *ml = a.part_ml + (slot * ROWS + in) * 2;
                        ml[0] = acc.m[t], ml[1] = acc.l[t];
                    }
                }
            }
        }
        u += c1 - c0;
    }
}

// The partials of a row, and the rows of sequences that could not be read (NaN). D / 4 lanes hold four dims each of one
// row. With few partials a row (many short sequences) every such group of lanes takes a row of its own, heads side by
// side; with many, all groups of a block take one row's partials in turn and meet in LDS in order (SHARE).
template <int D, int ROWS, int KEYS, int FRESH, bool SHARE>
__global__ void __launch_bounds__(kJoinThreads) tree_attn_join_kernel(const Args a) {
    constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes, kStride = SHARE ? kGroups : 1;
    __shared__ f32x4 sums[SHARE ? kGroups : 1][kLanes];
    __shared__ float ml[SHARE ? kGroups : 1][2];
    const int ln = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
    const int tok = blockIdx.x, head = SHARE ? blockIdx.y : blockIdx.y * kGroups + grp, kvh = head / a.G, h = head % a.G;
    int lo = 0, hi = a.B - 1;
    while (lo < hi) {  // the sequence of this token
        const int mid = (lo + hi) >> 1;
        if (a.starts[mid + 1] <= tok) lo = mid + 1;
        else hi = mid;
    }
    const int b = lo;
    if (head >= a.heads || tok < a.starts[b] || tok >= a.starts[b + 1]) return;  // a row behind the last sequence
    const Seq sq = seq_of<ROWS, KEYS, FRESH>(a, b);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = kNegInf, l = 0.f;
    if (!sq.bad) {
        const uint32_t U = a.prefix[a.B], nb = min((uint32_t)a.nb, U);
        const int r = (tok - sq.t0) * a.G + h, rg = r / ROWS;
        const uint32_t u0 = a.prefix[b] + (uint32_t)(rg * sq.chunks), u1 = u0 + sq.chunks;
        const int i0 = (int)((((uint64_t)u0 + 1) * nb - 1) / U), i1 = (int)(((uint64_t)u1 * nb - 1) / U);
        if (i0 == i1) return;  // written whole
#pragma unroll 4
        for (int i = i0 + (SHARE ? grp : 0); i <= i1; i += kStride) {
            // only the first block of the pair can hold it as its run's last one
            const bool second = i == i0 && (uint32_t)((uint64_t)U * i / nb) < u0;
            const int64_t row = (((int64_t)kvh * a.nb + i) * 2 + (second ? 1 : 0)) * ROWS + (r - rg * ROWS);
            const float m2 = a.part_ml[row * 2], l2 = a.part_ml[row * 2 + 1];
            const f32x4 v = *reinterpret_cast<const f32x4 *>(a.part_o + row * D + ln * 4);
            const float mx = fmaxf(m, m2), base = mx == kNegInf ? 0.f : mx;
            const float f1 = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
            o = o * f1 + v * f2, l = l * f1 + l2 * f2, m = mx;
        }
    } else {
        l = qnan();
    }
    if constexpr (SHARE) {
        sums[grp][ln] = o;
        if (ln == 0) ml[grp][0] = m, ml[grp][1] = l;
        __syncthreads();
        if (grp != 0) return;
        for (int i = 1; i < kGroups; ++i) {
            const float m2 = ml[i][0], l2 = ml[i][1], mx = fmaxf(m, m2), base = mx == kNegInf ? 0.f : mx;
            const float f1 = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
            o = o * f1 + sums[i][ln] * f2, l = l * f1 + l2 * f2, m = mx;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    *reinterpret_cast<uint2 *>(a.out + tok * a.out_t + head * a.out_h + ln * 4) =
        uint2{f32_to_bf16(o[0] * inv) | (f32_to_bf16(o[1] * inv) << 16), f32_to_bf16(o[2] * inv) | (f32_to_bf16(o[3] * inv) << 16)};
    if (a.lse != nullptr && ln == 0) a.lse[tok * a.lse_t + head] = log_sum(m, l);
}

// The rows a block holds - NT tiles of 16 a wave, WR waves side by side on the same keys - and the blocks a key head. The
// smallest tile that takes all rows of a sequence is taken, so that the cache is read once; a call with more rows than
// the largest tile takes further row groups, which read the cache again.
// Up to 32 rows a block of four waves a compute unit keeps 64 KB of loads in flight and has little else to do. Above, a
// step's chain of products and exponentials is as long as its loads, and two blocks of four waves with half the stage a
// compute unit, out of step with each other, beat one of eight (65,536 keys, 8 key heads of 128, us: 48 rows 67.4 / 74.2,
// 64 68.4 / 75.9, 96 78.5 / 82.8, 128 83.2 / 89.2, 192 alike; FP8 at 131,072: 48 rows 81 / 96, 128 121 / 134). 256 rows, and
// more than 64 at D = 256, take a block of eight waves (D = 256, 128 rows: 103 / 114).
struct Plan {
    int nt, wr, nb, hs;  // hs: bytes of keys (of values) a stage
    int64_t rows() const { return 16 * nt * wr; }
    // units of a sequence's row group, stages as Lay deals them
    int64_t units(int64_t D, int e, int64_t cached, int64_t max_new) const {
        const int64_t keys = std::min<int64_t>(hs / (D * e), 256), fresh = std::min<int64_t>(hs / (2 * D), 256);
        return (cached + keys - 1) / keys + (max_new + fresh - 1) / fresh;
    }
};
Plan plan_of(int64_t D, int64_t G, int64_t Hkv, int64_t max_new) {
    Plan p;
    const int64_t rows = max_new * G;
    if (D == 256) {  // a BF16 stage has two 32-key steps: two waves on keys at most
        p.nt = rows <= 64 ? 1 : 2, p.wr = rows <= 32 ? 2 : rows <= 128 ? 4 : 8;
    } else if (rows <= 32) {
        p.nt = rows <= 16 ? 1 : 2, p.wr = 1;
    } else {
        p.nt = rows <= 64 ? 2 : rows <= 96 ? 3 : rows <= 128 ? 2 : rows <= 192 ? 3 : 2, p.wr = rows <= 96 ? 2 : rows <= 192 ? 4 : 8;
    }
    const int per_cu = D == 256 ? (p.wr == 4 && p.nt == 1 ? 2 : 1) : p.wr == 2 || p.wr == 4 ? 2 : 1;
    p.nb = (int)std::max<int64_t>(1, (int64_t)device_cus() * per_cu / Hkv);
    p.hs = per_cu == 2 ? 16384 : 32768;
    return p;
}

const char *shape_error(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new) {
    if (D != 64 && D != 128 && D != 256) return "head dimension: 64, 128 or 256";
    if (Hkv < 1 || Hkv > 4096 || Hq < Hkv || Hq > 65535 || Hq % Hkv != 0) return "query heads: a multiple of the key heads";
    if (max_new < 1 || max_new > kMaxNew) return "max_new: 1..256";
    if (B < 1 || B > kMaxSeqs) return "sequences: 1..1024";
    return nullptr;
}

struct Space {
    int64_t o, ml, prefix, bytes;
};
Space space_of(const Plan &p, int64_t B, int64_t Hkv, int64_t D) {
    Space s;
    const int64_t rows = Hkv * p.nb * 2 * p.rows();
    s.o = 0, s.ml = rows * D * 4, s.prefix = s.ml + rows * 8, s.bytes = s.prefix + (B + 1) * 4;
    return s;
}

template <int D, int NT, int WR, int WK, int HS, bool F8>
void launch_type(const Args &a, int64_t Hkv, hipStream_t stream) {
    constexpr int ROWS = 16 * NT * WR, KEYS = Lay<D, F8, HS>::KEYS, FRESH = Lay<D, false, HS>::KEYS, kGroups = kJoinThreads / (D / 4);
    tree_attn_kernel<D, NT, WR, WK, HS, F8><<<dim3((unsigned)a.nb, (unsigned)Hkv), 64 * WR * WK, 0, stream>>>(a);
    // about nb / B + 1 partials a row (32 sequences, 64 blocks a head, 361 x 32 rows: 23.4 us shared, 8.0 not)
    if (a.nb > 8 * a.B) tree_attn_join_kernel<D, ROWS, KEYS, FRESH, true><<<dim3((unsigned)a.T, (unsigned)a.heads), kJoinThreads, 0, stream>>>(a);
    else tree_attn_join_kernel<D, ROWS, KEYS, FRESH, false><<<dim3((unsigned)a.T, (unsigned)((a.heads + kGroups - 1) / kGroups)), kJoinThreads, 0, stream>>>(a);
}

template <int D, int NT, int WR, int WK, int HS = 32768>
void launch(const Args &a, int64_t Hkv, bool f8, hipStream_t stream) {
    f8 ? launch_type<D, NT, WR, WK, HS, true>(a, Hkv, stream) : launch_type<D, NT, WR, WK, HS, false>(a, Hkv, stream);
}

template <int D>
void launch_rows(const Plan &p, const Args &a, int64_t Hkv, bool f8, hipStream_t s) {
    if constexpr (D == 256) {
        if (p.wr == 2) launch<D, 1, 2, 2>(a, Hkv, f8, s);
        else if (p.wr == 4) p.nt == 1 ? launch<D, 1, 4, 1, 16384>(a, Hkv, f8, s) : launch<D, 2, 4, 2>(a, Hkv, f8, s);
        else launch<D, 2, 8, 1>(a, Hkv, f8, s);
    } else {
        if (p.wr == 1) p.nt == 1 ? launch<D, 1, 1, 4>(a, Hkv, f8, s) : launch<D, 2, 1, 4>(a, Hkv, f8, s);
        else if (p.wr == 2) p.nt == 2 ? launch<D, 2, 2, 2, 16384>(a, Hkv, f8, s) : launch<D, 3, 2, 2, 16384>(a, Hkv, f8, s);
        else if (p.wr == 4) p.nt == 2 ? launch<D, 2, 4, 1, 16384>(a, Hkv, f8, s) : launch<D, 3, 4, 1, 16384>(a, Hkv, f8, s);
        else launch<D, 2, 8, 1>(a, Hkv, f8, s);
    }
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" {

int sx_tree_attention_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t max_new, size_t *bytes) {
    SX_CHECK(bytes != nullptr, "null pointer");
    const char *why = shape_error(B, Hq, Hkv, D, max_new);
    SX_CHECK(why == nullptr, why, " (B = ", B, ", Hq = ", Hq, ", Hkv = ", Hkv, ", D = ", D, ", max_new = ", max_new, ")");
    *bytes = (size_t)space_of(plan_of(D, Hq / Hkv, Hkv, max_new), B, Hkv, D).bytes;
    return SX_OK;
}

int sx_tree_attention(const sx_head_rows *q, const sx_head_rows *k_new, const sx_head_rows *v_new, int64_t T, int64_t Hq,
                      const sx_kv_cache *cache, const int32_t *starts, int64_t max_new, const uint64_t *mask,
                      int64_t mask_ld, float scale, const sx_head_rows *out, float *lse, void *ws, size_t ws_bytes,
                      uint32_t *err, sx_stream stream) {
    SX_CHECK(q != nullptr && k_new != nullptr && v_new != nullptr && cache != nullptr && out != nullptr && q->p != nullptr &&
                 k_new->p != nullptr && v_new->p != nullptr && out->p != nullptr && starts != nullptr && mask != nullptr &&
                 ws != nullptr,
             "null pointer");
    std::string why = kv_cache_error(*cache);
    SX_CHECK(why.empty(), why);
    const int64_t B = cache->batch, Hkv = cache->heads, D = cache->dim;
    const char *bad = shape_error(B, Hq, Hkv, D, max_new);
    SX_CHECK(bad == nullptr, bad, " (B = ", B, ", Hq = ", Hq, ", Hkv = ", Hkv, ", D = ", D, ", max_new = ", max_new, ")");
    SX_CHECK(cache->layers == 1, "layers = ", cache->layers, ": attention takes one layer's cache");
    // a launch has fewer than 2^32 threads a dimension: the join's is T blocks (the sequences' own are 2^18 rows at most)
    SX_CHECK(T >= 1 && T < ((int64_t)1 << 32) / kJoinThreads, "T = ", T, " rows of drafted tokens, expected 1..", ((int64_t)1 << 32) / kJoinThreads - 1);
    SX_CHECK(k_new->token <= (1 << 21) && v_new->token <= (1 << 21), "token strides of k_new and v_new up to 2^21 elements (", k_new->token, ", ", v_new->token, ")");
    SX_CHECK(mask_ld >= (max_new + 63) / 64, "mask_ld = ", mask_ld, " words a token for max_new = ", max_new);
    const float scale2 = scale * 1.4426950408889634f;  // the kernels work in powers of two
    SX_CHECK(scale > 0.f && std::isnormal(scale2) && (cache->dtype != SX_KV_E4M3 || std::isnormal(scale2 * cache->k_scale)),
             "scale = ", scale, ", expected positive and, times k_scale, a normal number");
    why = head_rows_error(*q, "q", Hq, D);
    if (why.empty()) why = head_rows_error(*k_new, "k_new", Hkv, D);
    if (why.empty()) why = head_rows_error(*v_new, "v_new", Hkv, D);
    if (why.empty()) why = head_rows_error(*out, "out", Hq, D);
    SX_CHECK(why.empty(), why);
    SX_CHECK(rows_apart(D, {{T, out->token}, {Hq, out->head}}), "rows of out share memory (strides: token ", out->token, ", head ", out->head, ")");
    SX_CHECK(aligned(mask, 8) && aligned(ws, 16), "mask must be 8-byte and the workspace 16-byte aligned");
    const int64_t out_bytes = head_rows_bytes(*out, T, Hq, D);
    const Strided rows[3] = {rows_block(*q, T, Hq, D), rows_block(*k_new, T, Hkv, D), rows_block(*v_new, T, Hkv, D)}, o = rows_block(*out, T, Hq, D);
    SX_CHECK(strided_apart(o, rows[0]) && strided_apart(o, rows[1]) && strided_apart(o, rows[2]), "out overlaps q, k_new or v_new");
    const Plan p = plan_of(D, Hq / Hkv, Hkv, max_new);
    const Space sp = space_of(p, B, Hkv, D);
    SX_CHECK(ws_bytes >= (size_t)sp.bytes, "workspace of ", ws_bytes, " bytes, needs ", sp.bytes);
    SX_CHECK(apart(ws, sp.bytes, out->p, out_bytes) && (lse == nullptr || (apart(lse, 4 * T * Hq, ws, sp.bytes) && apart(lse, 4 * T * Hq, out->p, out_bytes))),
             "out, lse and the workspace overlap");
    const int64_t most = p.units(D, kv_bytes(*cache), cache->pages_per_seq * cache->page_size, max_new);
    const int64_t groups = (max_new * (Hq / Hkv) + p.rows() - 1) / p.rows();
    SX_CHECK(B * groups * most < ((int64_t)1 << 31), "more than 2^31 units of work (B = ", B, ", pages a sequence ", cache->pages_per_seq, ")");
    // blocks read all of these until the call's last one ends
    const Strided reads[9] = {rows[0], rows[1], rows[2], kv_block(*cache, false), kv_block(*cache, true),
                              {mask, (max_new + 63) / 64 * 8, {{1, 0}, {1, 0}, {T, mask_ld * 8}, {1, 0}}},
                              {starts, 4 * (B + 1), {}}, {cache->lens, 4 * B, {}},
                              {cache->table, 4 * cache->pages_per_seq, {{1, 0}, {1, 0}, {B, cache->table_ld * 4}, {1, 0}}}};
    for (const Strided &r : reads)
        SX_CHECK(strided_apart(o, r) && strided_apart({ws, sp.bytes, {}}, r) && (lse == nullptr || strided_apart({lse, 4 * T * Hq, {}}, r)),
                 "out, lse or the workspace overlaps the inputs, the cache or its words");
    SX_CHECK(aligned(starts, 4) && aligned(cache->lens, 4) && aligned(cache->table, 4) && aligned(lse, 4) && aligned(err, 4),
             "starts, lens, table, lse and err must be 4-byte aligned");

    Args a;
    const int e = kv_bytes(*cache);
    a.q = static_cast<const uint16_t *>(q->p), a.q_t = q->token, a.q_h = q->head;
    a.kn = static_cast<const uint16_t *>(k_new->p), a.kn_t = k_new->token, a.kn_h = k_new->head;
    a.vn = static_cast<const uint16_t *>(v_new->p), a.vn_t = v_new->token, a.vn_h = v_new->head;
    a.out = static_cast<uint16_t *>(out->p), a.out_t = out->token, a.out_h = out->head;
    a.kc = static_cast<const uint8_t *>(cache->k), a.vc = static_cast<const uint8_t *>(cache->v);
    a.kc_p = cache->k_page * e, a.kc_t = (int32_t)(cache->k_token * e), a.kc_h = cache->k_head * e;
    a.vc_p = cache->v_page * e, a.vc_t = (int32_t)(cache->v_token * e), a.vc_h = cache->v_head * e;
    a.table = cache->table, a.table_ld = cache->table_ld, a.lens = cache->lens, a.starts = starts;
    a.mask = mask, a.mask_ld = mask_ld, a.lse = lse, a.lse_t = Hq, a.err = err;
    uint8_t *w = static_cast<uint8_t *>(ws);
    a.part_o = reinterpret_cast<float *>(w + sp.o), a.part_ml = reinterpret_cast<float *>(w + sp.ml);
    a.prefix = reinterpret_cast<uint32_t *>(w + sp.prefix);
    a.B = (int32_t)B, a.T = (int32_t)T, a.G = (int32_t)(Hq / Hkv), a.P = (int32_t)cache->pages_per_seq;
    a.pages = (int32_t)cache->pages, a.page_shift = __builtin_ctzll((uint64_t)cache->page_size);
    a.max_new = (int32_t)max_new, a.nb = p.nb, a.heads = (int32_t)Hq;
    a.scale = scale2, a.k_scale = cache->k_scale, a.v_scale = cache->v_scale;
    const bool f8 = cache->dtype == SX_KV_E4M3;
    hipStream_t s = stream_of(stream);
    if (D == 64) launch_rows<64>(p, a, Hkv, f8, s);
    else if (D == 128) launch_rows<128>(p, a, Hkv, f8, s);
    else launch_rows<256>(p, a, Hkv, f8, s);
    SX_LAUNCHED("tree_attention T=", T, " B=", B, " Hq=", Hq, " Hkv=", Hkv, " D=", D);
    return SX_OK;
}

}  // extern "C"
