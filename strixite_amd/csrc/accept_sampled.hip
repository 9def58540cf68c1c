// Acceptance of drafted tokens against the target's probabilities (rejection sampling): with p the softmax of a row's logits over
// a temperature and q that of the draft's, draft d stays where u q(d) < p(d); the first that does not is replaced by a token
// from max(p - q, 0), and behind the last draft comes one from p. What comes out has the target's distribution. Without draft
// logits q is all on the draft (a head that proposes its best token).
//
// The results are whole numbers that a border decides, and a token is picked out of sums over a vocabulary: probabilities and sums
// are FP64 (exponentials good to 6e-15). All logits are read once, by as many blocks as they need: rows in chunks of 4096, a chunk's
// largest value, its place and its sum of exponentials. Then a wave combines a row's chunks, the rows of a sequence at once, which tells
// the last row that counts; that one's chunks of max(p - q, 0) are summed where there are draft logits, and one block a sequence finds the chunk,
// and in it the token, at which the running sum passes u times the total (second launch). Sums are taken in one order, whatever
// the schedule. 16 sequences of up to 6 rows of 151,936 logits with draft logits: 25 + 5.6 + 17 us, the first the VALU's (an FP64
// exponential a logit, 0.66 of its cycles); one sequence without: 5.5 + 8.7, latencies.
#include "common.hpp"

#include <cmath>

namespace sx {
namespace {

constexpr int kChunk = 4096, kThreads = 256, kEach = kChunk / kThreads, kDrawThreads = 512, kDrawEach = kChunk / kDrawThreads, kMaxRows = 256, kMaxSeqs = 1024;

struct Part {
    double sum;  // of exp((x - top) / temperature)
    float top;
    int32_t at;  // its lowest place; -1: the chunk holds a NaN
};

// What a sequence's rows come to.
struct Verdict {
    double m, z, mq, zq;  // of the row a token is drawn from: largest logit and 1 / sum, the target's and the draft's
    int32_t kept;         // drafts that stay
    int32_t status;
    int32_t kind;         // below
    int32_t best;         // the row's largest logit's place
    int32_t t0, draft;    // the sequence's first row; the row's draft
    double draw;          // the row's second number
};
enum { kNone, kTarget, kHole, kRest, kGreedy };  // nothing; from p; from p without the draft; from max(p - q, 0); the best

struct Args {
    const void *logits, *draft_logits;
    const int32_t *drafts, *starts;
    const double *u;
    const float *temperature;
    int32_t *tokens, *count, *status;
    Part *parts, *draft_parts;  // [T][chunks]
    double *rest;               // [B][chunks]
    int32_t *arrived;           // [B]: blocks whose sum is there
    Verdict *verdicts;          // [B]
    int64_t ld, draft_ld;
    int32_t T, V, Vd, B, max_rows, chunks, draft_chunks;
};

__device__ __forceinline__ float load(const float *p) { return *p; }
__device__ __forceinline__ float load(const uint16_t *p) { return bf16_to_f32(*p); }

// N neighbouring logits in 16-byte loads; rows start at any element. Places from `left` on are -inf.
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8), aligned(2)));
template <int N>
__device__ __forceinline__ void load_run(const float *p, int left, float (&x)[N]) {
    if (left >= N) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4 *>(p + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[i + j] = v[j];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i < left ? p[i] : -INFINITY;
    }
}
template <int N>
__device__ __forceinline__ void load_run(const uint16_t *p, int left, float (&x)[N]) {
    if (left >= N) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const u16x8 v = *reinterpret_cast<const u16x8 *>(p + i);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i + j] = bf16_to_f32(v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i < left ? bf16_to_f32(p[i]) : -INFINITY;
    }
}

// Sequence b's own words. Where starts fall, that sequence and all behind it are impossible too: their rows could be another's,
// whose temperature a row's sums are taken at.
__device__ __forceinline__ bool usable(const Args &a, int b, int &t0, int &n) {
    t0 = a.starts[b];
    n = (int)((uint32_t)a.starts[b + 1] - (uint32_t)t0);
    return t0 >= 0 && n >= 0 && (int64_t)t0 + n <= a.T && n <= a.max_rows;
}

// Across a wave, the result in all lanes: neighbours by DPP, then halves of 32 and of 64 lanes.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false); }
template <int STEP>
__device__ __forceinline__ uint32_t other(uint32_t v) {
    if constexpr (STEP == 0) return dpp<0xB1>(v);
    else if constexpr (STEP == 1) return dpp<0x4E>(v);
    else if constexpr (STEP == 2) return dpp<0x141>(v);
    else if constexpr (STEP == 3) return dpp<0x140>(v);
    else {
        const bool up = threadIdx.x & (STEP == 4 ? 16 : 32);
        const auto x = STEP == 4 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return up ? x[0] : x[1];
    }
}
template <int STEP>
__device__ __forceinline__ double other(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)other<STEP>((uint32_t)(u >> 32)) << 32 | other<STEP>((uint32_t)u)));
}
__device__ __forceinline__ double wave_sum(double v) {
    v += other<0>(v), v += other<1>(v), v += other<2>(v);
    v += other<3>(v), v += other<4>(v);
    return v + other<5>(v);
}
// The largest value and its lowest place.
template <int STEP>
__device__ __forceinline__ void best_step(float &top, int &at) {
    const float o = __uint_as_float(other<STEP>(__float_as_uint(top)));
    const int oa = (int)other<STEP>((uint32_t)at);
    if (o > top || (o == top && oa < at)) top = o, at = oa;
}
__device__ __forceinline__ void wave_best(float &top, int &at) {
    best_step<0>(top, at), best_step<1>(top, at), best_step<2>(top, at);
    best_step<3>(top, at), best_step<4>(top, at), best_step<5>(top, at);
}

// exp(y) for y <= 0 (-inf: 0) in FP64: 2^n times the power series of e^r, |r| <= ln(2) / 2, to the eleventh power (6e-15 is left).
// The library's takes more instructions for ranges that a softmax does not reach; of these a chunk's launch consists.
__device__ __forceinline__ double weight(double y) {
    y = fmax(y, -800.0);  // 0 from there on
    const double n = rint(y * 1.4426950408889634);
    const double r = fma(n, -4.7493250390316726e-07, fma(n, -0.6931467056274414, y));  // ln(2): 21 bits, whose multiples are exact, and the rest
    double p = 1.0 / 39916800.0;
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) accept_parts_kernel(const Args a) {
    __shared__ float tops[4];
    __shared__ int ats[4], owners[4], fallen[4];
    __shared__ double sums[4];
    const int chunk = blockIdx.x, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.y % a.T;
    const bool draft = blockIdx.y >= (unsigned)a.T;
    if (chunk >= (draft ? a.draft_chunks : a.chunks)) return;
    const int V = draft ? a.Vd : a.V, first = chunk * kChunk;
    const T *p = static_cast<const T *>(draft ? a.draft_logits : a.logits) + row * (draft ? a.draft_ld : a.ld) + first;
    float x[kEach];
#pragma unroll
    for (int i = 0; i < kEach / 8; ++i) {
        const int k = ((int)threadIdx.x + i * kThreads) * 8;
        float run[8];
        load_run<8>(p + min(k, V - 1 - first), V - first - k, run);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[8 * i + j] = run[j];
    }
    // the row's sequence (a last row has no draft): the lowest whose words say so, if starts have not fallen before it
    int owner = a.B, falls = a.B;
    for (int b0 = threadIdx.x & ~63; b0 < a.B; b0 += kThreads) {
        const int b = b0 + (threadIdx.x & 63);
        bool has = false, down = false;
        if (b < a.B) {
            int t0, n;
            has = usable(a, b, t0, n) && row >= t0 && row < t0 + n - (draft ? 1 : 0);
            down = a.starts[b + 1] < t0;
        }
        const uint64_t h = __ballot(has), d = __ballot(down);
        if (h != 0 && owner == a.B) owner = b0 + __builtin_ctzll(h);
        if (d != 0 && falls == a.B) falls = b0 + __builtin_ctzll(d);
    }
    float top = -INFINITY;
    int at = 0x7fffffff;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        nan |= x[i] != x[i];
        if (x[i] > top) top = x[i], at = first + ((int)threadIdx.x + i / 8 * kThreads) * 8 + i % 8;
    }
    wave_best(top, at);
    if ((threadIdx.x & 63) == 0) tops[wave] = top, ats[wave] = at, owners[wave] = owner, fallen[wave] = falls;
    nan = __syncthreads_or(nan);
    top = tops[0], at = ats[0], owner = min(min(owners[0], owners[1]), min(owners[2], owners[3]));
    if (owner >= min(min(fallen[0], fallen[1]), min(fallen[2], fallen[3]))) return;
#pragma unroll
    for (int w = 1; w < 4; ++w)
        if (tops[w] > top || (tops[w] == top && ats[w] < at)) top = tops[w], at = ats[w];
    const float temp = a.temperature[owner];
    double sum = 0.0;
    if (temp > 0.f && top > -INFINITY && top < INFINITY) {
        const double over_t = 1.0 / (double)temp;
#pragma unroll
        for (int i = 0; i < kEach; ++i) sum += weight(((double)x[i] - (double)top) * over_t);
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
        (draft ? a.draft_parts + row * a.draft_chunks : a.parts + row * a.chunks)[chunk] = Part{(sums[0] + sums[1]) + (sums[2] + sums[3]), top, nan ? -1 : at};
}

// A row's largest logit, its place (-1: a NaN) and its sum, by one wave, in all lanes.
struct Row {
    float m;
    int at;
    double z;
};
// `mine`: the lane's first part, requested before. One copy in the code: a launch of few blocks waits for its instructions more than
// for its data.
__device__ __attribute__((noinline)) Row row_stats(const Part *parts, int chunks, Part mine, double over_t) {
    const int lane = threadIdx.x & 63;
    Row r{-INFINITY, 0x7fffffff, 0.0};
    bool nan = false;
    for (int c = lane; c < chunks; c += 64) {
        const Part x = c < 64 ? mine : parts[c];
        nan |= x.at < 0;
        if (x.top > r.m || (x.top == r.m && x.at < r.at)) r.m = x.top, r.at = x.at;
    }
    wave_best(r.m, r.at);
    if (__any(nan)) r.at = -1;
    if (fabsf(r.m) < INFINITY)
#pragma unroll 1
        for (int c = lane; c < chunks; c += 64) {
            const Part x = c < 64 ? mine : parts[c];
            r.z += x.sum * weight(((double)x.top - (double)r.m) * over_t);
        }
    r.z = wave_sum(r.z);
    return r;
}

// What a block knows of its sequence's rows.
struct Rows {
    double stats[5 * kMaxRows];
    uint8_t fate[kMaxRows];
};

// Every thread of the block calls it; the verdict is in `v` (LDS) for all of them.
template <typename T>
__device__ __forceinline__ void decide(const Args &a, int b, Verdict &v, Rows &rows) {
    int t0, n;
    bool falls = false;
    for (int j = threadIdx.x; j < b; j += kDrawThreads) falls |= a.starts[j + 1] < a.starts[j];
    falls = b > 0 && __syncthreads_or(falls);
    const bool ok = usable(a, b, t0, n) && !falls;
    if (!ok || n == 0) {
        if (threadIdx.x == 0) v = Verdict{0, 0, 0, 0, 0, ok ? 0 : -1, kNone, 0, 0, 0, 0};
        __syncthreads();
        return;
    }
    const float temp = a.temperature[b];
    const bool greedy = temp <= 0.f;
    const double over_t = greedy ? 0.0 : 1.0 / (double)temp;
    const int wave = threadIdx.x >> 6;
    for (int i = wave; i < n; i += kDrawThreads / 64) {
        const int64_t t = t0 + i;
        const bool drafted = i + 1 < n, both = drafted && a.draft_logits != nullptr && !greedy;
        const int lane = threadIdx.x & 63;
        const Part p = a.parts[t * a.chunks + min(lane, a.chunks - 1)], pq = both ? a.draft_parts[t * a.draft_chunks + min(lane, a.draft_chunks - 1)] : Part{};
        const int d = a.drafts[t];
        const bool inside = d >= 0 && d < a.V;
        const double u = a.u[2 * t];
        const float x = load(static_cast<const T *>(a.logits) + t * a.ld + (inside ? d : 0));
        const float xq = both && inside && d < a.Vd ? load(static_cast<const T *>(a.draft_logits) + t * a.draft_ld + d) : -INFINITY;
        const Row r = row_stats(a.parts + t * a.chunks, a.chunks, p, over_t);
        Row rq{0.f, 0, 1.0};
        bool bad = r.at < 0 || !(fabsf(r.m) < INFINITY) || !(fabsf(temp) < INFINITY) || (drafted && !inside), stays = false;
        if (drafted && !bad) {
            if (greedy) {
                stays = d == r.at;
            } else {
                double q = 1.0;
                if (both) {
                    rq = row_stats(a.draft_parts + t * a.draft_chunks, a.draft_chunks, pq, over_t);
                    bad = rq.at < 0 || !(fabsf(rq.m) < INFINITY);
                    q = weight(((double)xq - (double)rq.m) * over_t) / rq.z;
                }
                stays = u * q < weight(((double)x - (double)r.m) * over_t) / r.z;
            }
        }
        if ((threadIdx.x & 63) == 0) {
            rows.fate[i] = bad ? 2 : stays ? 1 : 0;
            double *s = rows.stats + 5 * i;
            s[0] = r.m, s[1] = 1.0 / r.z, s[2] = rq.m, s[3] = 1.0 / rq.z, s[4] = r.at;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int j = 0;
        while (rows.fate[j] == 1) ++j;  // the last row has no draft: it is 0 or 2
        const double *s = rows.stats + 5 * j;
        const bool last = j + 1 == n;
        v = Verdict{s[0], s[1], s[2], s[3], j, rows.fate[j] == 2 ? 1 + j : 0,
                    rows.fate[j] == 2 ? kNone : greedy ? kGreedy : last ? kTarget : a.draft_logits != nullptr ? kRest : kHole, (int)s[4], t0,
                    a.drafts[t0 + j], a.u[2 * (int64_t)(t0 + j) + 1]};
    }
    __syncthreads();
}

__device__ __forceinline__ double block_sum(double v, double *part) {
    v = wave_sum(v);
    __syncthreads();  // part may still be read
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads) accept_decide_kernel(const Args a) {
    __shared__ Verdict v;
    __shared__ Rows rows;
    decide<T>(a, blockIdx.x, v, rows);
    if (threadIdx.x == 0) a.verdicts[blockIdx.x] = v, a.arrived[blockIdx.x] = 0;
}

// Grid (1, B) without draft logits; with them (chunks, B) behind accept_decide_kernel: then a block also sums its chunk of
// max(p - q, 0), and the last block of a sequence to get there draws. (Without the launch between, all of these blocks deciding for
// themselves, it is as fast: 22.6 us for 5.6 + 17.2 with 16 sequences of up to 6 rows of 38 chunks, calls of 256 rows 118 to 189 us for
// 121 to 192. So a row's chunks are combined once, and not by every block of its sequence.)
template <typename T, bool DRAFT>
__global__ void __launch_bounds__(kDrawThreads) accept_draw_kernel(const Args a) {
    __shared__ Verdict v;
    __shared__ double part[8], ends[8];
    __shared__ int chosen, last, firsts[8], lasts[8];
    const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double over_t = 1.0 / (double)a.temperature[b];
    if constexpr (DRAFT) {
        if (threadIdx.x == 0) v = a.verdicts[b];
        __syncthreads();
    } else {
        __shared__ Rows rows;
        decide<T>(a, b, v, rows);
    }
    const int64_t row = (int64_t)v.t0 + v.kept;
    const int draft = v.draft;
    if (DRAFT && v.kind != kRest && blockIdx.x != 0) return;
    int token = v.kind == kGreedy ? v.best : -1;
    if (v.kind == kTarget || v.kind == kHole || v.kind == kRest) {
        int kind = v.kind;
        const int per = (a.chunks + kDrawThreads - 1) / kDrawThreads, c0 = min((int)threadIdx.x * per, a.chunks), c1 = min(c0 + per, a.chunks);
        const int hole = kind == kHole ? draft / kChunk : -1;
        double hole_sum = 0.0, upto = 0.0, mine = 0.0, total = 0.0, goal = 0.0, run0 = 0.0;
        // Running sums of all threads' values: upto ends with this thread's.
        auto scan = [&]() {
            upto = mine;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const double x = __shfl_up(upto, d);
                if (lane >= d) upto += x;
            }
            __syncthreads();  // ends may still be read
            if (lane == 63) ends[wave] = upto;
            __syncthreads();
            double before = 0.0;
            total = 0.0;
#pragma unroll
            for (int w = 0; w < kDrawThreads / 64; ++w) {
                if (w == wave) before = total;
                total += ends[w];
            }
            upto += before;
        };
        // The first thread's candidate (threads hold rising ones); where rounding left none, the last one's fallback.
        auto first_of = [&](int candidate, int fallback) {
            const uint64_t c = __ballot(candidate >= 0), f = __ballot(fallback >= 0);
            candidate = c != 0 ? __shfl(candidate, __builtin_ctzll(c)) : -1;
            fallback = f != 0 ? __shfl(fallback, 63 - __builtin_clzll(f)) : -1;
            __syncthreads();  // they may still be read
            if (lane == 0) firsts[wave] = candidate, lasts[wave] = fallback;
            __syncthreads();
            int got = -1;
#pragma unroll
            for (int w = 0; w < kDrawThreads / 64; ++w) got = lasts[w] >= 0 ? lasts[w] : got;
#pragma unroll
            for (int w = kDrawThreads / 64 - 1; w >= 0; --w) got = firsts[w] >= 0 ? firsts[w] : got;
            return got;
        };
        auto of_chunk = [&](int c) {
            if (kind == kRest) return __hip_atomic_load(&a.rest[(int64_t)b * a.chunks + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (kind == kHole && c == hole) return hole_sum;
            const Part p = a.parts[row * a.chunks + c];
            return p.top > -INFINITY ? p.sum * weight(((double)p.top - v.m) * over_t) : 0.0;
        };
        // A chunk's places, kDrawEach neighbouring ones a thread: first the chunk of this block's sum (of the hole: by taking the draft
        // off its chunk's sum, what is left would be noise), then the one that the token is in. The same code for both.
        int at_chunk = kind == kRest ? (int)blockIdx.x : hole;
        bool found = false;
#pragma unroll 1
        for (;;) {
            double w[kDrawEach];
            mine = 0.0;
            if (at_chunk >= 0) {
                const int at0 = at_chunk * kChunk + threadIdx.x * kDrawEach;
                float x[kDrawEach], xq[kDrawEach];
                load_run<kDrawEach>(static_cast<const T *>(a.logits) + row * a.ld + min(at0, a.V - 1), a.V - at0, x);
                if (DRAFT && kind == kRest) load_run<kDrawEach>(static_cast<const T *>(a.draft_logits) + row * a.draft_ld + min(at0, a.Vd - 1), a.Vd - at0, xq);
#pragma unroll
                for (int i = 0; i < kDrawEach; ++i) {
                    w[i] = weight(((double)x[i] - v.m) * over_t);
                    if (DRAFT && kind == kRest) w[i] = fmax(w[i] * v.z - weight(((double)xq[i] - v.mq) * over_t) * v.zq, 0.0);
                    if (kind == kHole && at0 + i == draft) w[i] = 0.0;
                    mine += w[i];
                }
            }
            if (found) {
                scan();
                double run = run0 + (upto - mine);
                int pass = -1, some = -1;
#pragma unroll
                for (int i = 0; i < kDrawEach; ++i) {
                    run += w[i];
                    const int at = at_chunk * kChunk + threadIdx.x * kDrawEach + i;
                    if (w[i] > 0.0) {
                        some = at;
                        if (pass < 0 && run > goal) pass = at;
                    }
                }
                token = first_of(pass, some);
                break;
            }
            if (at_chunk >= 0) hole_sum = block_sum(mine, part);
            if (DRAFT && kind == kRest) {
                if (threadIdx.x == 0) {
                    // written through to where all XCDs see it, and counted once it is there
                    __hip_atomic_store(&a.rest[(int64_t)b * a.chunks + blockIdx.x], hole_sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    last = __hip_atomic_fetch_add(&a.arrived[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int)gridDim.x - 1;
                }
                __syncthreads();
                if (!last) return;
            }
            // the weights of this thread's run of chunks; a row that has nothing left over the draft's is drawn from p
            for (;;) {
                mine = 0.0;
#pragma unroll 1
                for (int c = c0; c < c1; ++c) mine += of_chunk(c);
                scan();
                if (total > 0.0 || kind == kTarget) break;
                kind = kTarget;
            }
            goal = v.draw * total;
            const int run_of = first_of(mine > 0.0 && upto > goal ? (int)threadIdx.x : -1, mine > 0.0 ? (int)threadIdx.x : -1);
            if ((int)threadIdx.x == run_of) {
                double run = upto - mine, some_run = run;
                int some = c0;
                if (per > 1)
#pragma unroll 1
                    for (int c = c0; c < c1; ++c) {
                        const double x = of_chunk(c);
                        if (x > 0.0) some = c, some_run = run;
                        if (x > 0.0 && run + x > goal) break;
                        run += x;
                    }
                chosen = some, part[0] = some_run;
            }
            __syncthreads();
            at_chunk = chosen, run0 = part[0], found = true;
            __syncthreads();  // both are written again
        }
    }
    const int kept = v.kept;
    for (int i = threadIdx.x; i < a.max_rows; i += kDrawThreads)
        a.tokens[(int64_t)b * a.max_rows + i] = i < kept ? a.drafts[v.t0 + i] : i == kept ? token : -1;
    if (threadIdx.x == 0) a.count[b] = v.kind == kNone ? kept : kept + 1, a.status[b] = v.status;
}

struct Sizes {
    int64_t chunks, draft_chunks, parts, draft_parts, rest, bytes;
};
Sizes sizes(int64_t T, int64_t B, int64_t V, int64_t Vd) {
    Sizes s;
    s.chunks = (V + kChunk - 1) / kChunk, s.draft_chunks = (Vd + kChunk - 1) / kChunk;
    s.parts = T * s.chunks * (int64_t)sizeof(Part), s.draft_parts = T * s.draft_chunks * (int64_t)sizeof(Part);
    s.rest = Vd > 0 ? B * s.chunks * 8 : 0;
    s.bytes = s.parts + s.draft_parts + s.rest + (Vd > 0 ? B * ((int64_t)sizeof(Verdict) + 4) : 0);
    return s;
}

template <typename T>
void launch(const Args &a, hipStream_t s) {
    const bool drafted = a.draft_logits != nullptr;
    accept_parts_kernel<T><<<dim3((unsigned)std::max(a.chunks, a.draft_chunks), (unsigned)(drafted ? 2 * a.T : a.T)), kThreads, 0, s>>>(a);
    if (drafted) accept_decide_kernel<T><<<(unsigned)a.B, kDrawThreads, 0, s>>>(a);
    if (drafted) accept_draw_kernel<T, true><<<dim3((unsigned)a.chunks, (unsigned)a.B), kDrawThreads, 0, s>>>(a);
    else accept_draw_kernel<T, false><<<dim3(1, (unsigned)a.B), kDrawThreads, 0, s>>>(a);
}

bool sizes_ok(int64_t T, int64_t B, int64_t V, int64_t Vd) {
    return T >= 1 && T <= 32767 && B >= 1 && B <= kMaxSeqs && V >= 1 && V <= 1 << 24 && Vd >= 0 && Vd <= V;
}

}  // namespace
}  // namespace sx

using namespace sx;

extern "C" int sx_mtp_accept_sampled_workspace_bytes(int64_t T, int64_t B, int64_t V, int64_t Vd, size_t *bytes) {
    SX_CHECK(bytes != nullptr, "null pointer");
    SX_CHECK(sizes_ok(T, B, V, Vd), "T = ", T, ", batch = ", B, ", n_valid = ", V, ", n_draft = ", Vd);
    *bytes = (size_t)sizes(T, B, V, Vd).bytes;
    return SX_OK;
}

extern "C" int sx_mtp_accept_sampled(const void *logits, int64_t ld, int64_t T, int64_t V, const void *draft_logits, int64_t draft_ld, int64_t Vd,
                                     int act, const int32_t *drafts, const int32_t *starts, int64_t B, int64_t max_rows, const double *u,
                                     const float *temperature, int32_t *tokens, int32_t *count, int32_t *status, void *ws, size_t ws_bytes,
                                     sx_stream stream) {
    SX_CHECK(logits != nullptr && drafts != nullptr && starts != nullptr && u != nullptr && temperature != nullptr && tokens != nullptr &&
                 count != nullptr && status != nullptr && ws != nullptr,
             "null pointer");
    SX_CHECK(act == SX_ACT_F32 || act == SX_ACT_BF16, "unsupported logit dtype ", act);
    SX_CHECK(T >= 1 && T <= 32767, "T = ", T, ", expected 1..32767");
    SX_CHECK(B >= 1 && B <= kMaxSeqs, "batch = ", B, ", expected 1..", kMaxSeqs);
    SX_CHECK(V >= 1 && V <= 1 << 24 && ld >= V && ld <= (int64_t)1 << 32, "n_valid = ", V, ", ld = ", ld);
    SX_CHECK((draft_logits == nullptr) == (Vd == 0), "draft_logits and n_draft go together");
    SX_CHECK(Vd >= 0 && Vd <= V && (Vd == 0 || (draft_ld >= Vd && draft_ld <= (int64_t)1 << 32)), "n_draft = ", Vd, ", draft_ld = ", draft_ld, " for n_valid = ", V);
    SX_CHECK(max_rows >= 1 && max_rows <= kMaxRows, "max_rows = ", max_rows, ", expected 1..", kMaxRows);
    const Sizes z = sizes(T, B, V, Vd);
    SX_CHECK((int64_t)ws_bytes >= z.bytes, "a workspace of ", ws_bytes, " bytes, expected ", z.bytes);
    const int e = act_bytes(act);
    SX_CHECK(aligned(logits, e) && aligned(draft_logits, e) && aligned(drafts, 4) && aligned(starts, 4) && aligned(u, 8) && aligned(temperature, 4) &&
                 aligned(tokens, 4) && aligned(count, 4) && aligned(status, 4) && aligned(ws, 16),
             "the workspace must be 16-byte aligned, the others to their elements");
    struct Span {
        const void *p;
        int64_t n;
    };
    const Span in[6] = {{logits, ((T - 1) * ld + V) * e}, {draft_logits, Vd > 0 ? ((T - 1) * draft_ld + Vd) * e : 0}, {drafts, 4 * T}, {starts, 4 * (B + 1)},
                        {u, 16 * T}, {temperature, 4 * B}};
    const Span outs[4] = {{tokens, 4 * B * max_rows}, {count, 4 * B}, {status, 4 * B}, {ws, z.bytes}};
    for (int o = 0; o < 4; ++o) {
        for (const Span &i : in) SX_CHECK(i.n == 0 || apart(i.p, i.n, outs[o].p, outs[o].n), "output ", o, " (tokens, count, status, workspace) overlaps an input");
        for (int k = 0; k < o; ++k) SX_CHECK(apart(outs[k].p, outs[k].n, outs[o].p, outs[o].n), "outputs ", k, " and ", o, " overlap");
    }
    uint8_t *w = static_cast<uint8_t *>(ws);
    const Args a{logits, draft_logits, drafts, starts, u, temperature, tokens, count, status, reinterpret_cast<Part *>(w),
                 reinterpret_cast<Part *>(w + z.parts), reinterpret_cast<double *>(w + z.parts + z.draft_parts),
                 reinterpret_cast<int32_t *>(w + z.parts + z.draft_parts + z.rest + B * (int64_t)sizeof(Verdict)),
                 reinterpret_cast<Verdict *>(w + z.parts + z.draft_parts + z.rest), ld, draft_ld, (int32_t)T, (int32_t)V, (int32_t)Vd, (int32_t)B,
                 (int32_t)max_rows, (int32_t)z.chunks, (int32_t)z.draft_chunks};
    if (act == SX_ACT_F32) launch<float>(a, stream_of(stream));
    else launch<uint16_t>(a, stream_of(stream));
    SX_LAUNCHED("mtp_accept_sampled T=", T, " batch=", B);
    return SX_OK;
}
