// Acceptance of drafted tokens against the target's probabilities (rejection sampling): with p the softmax of a row's logits over
// a temperature and q that of the draft's, draft d stays where u q(d) < p(d); the first that does not is replaced by a token
// from max(p - q, 0), and behind the last draft comes one from p. What comes out has the target's distribution. Without draft
// logits q is all on the draft (a head that proposes its best token).
//
// The results are whole numbers that a border decides, and a token is picked out of sums over a vocabulary: probabilities and sums
// are FP64. All logits are read once, by as many blocks as they need: rows in chunks of 2048, a chunk's largest value, its
// place and its sum of exponentials. Then a wave combines a row's chunks, the rows of a sequence at once, which tells the last row that
// counts; that one's chunks of max(p - q, 0) are summed (second launch, with draft logits only), and one block a sequence
// finds the chunk, and in it the token, at which the running sum passes u times the total. Sums are taken in one order, whatever
// the schedule.
#include "common.hpp"

#include <cmath>

namespace sx {
namespace {

constexpr int kChunk = 2048, kThreads = 256, kEach = kChunk / kThreads, kMaxRows = 256, kMaxSeqs = 1024;

struct Part {
    double sum;  // of exp((x - top) / temperature)
    float top;
    int32_t at;  // its lowest place; -1: the chunk holds a NaN
};

// What a sequence's rows come to.
struct Verdict {
    double m, z, mq, zq;  // of the row a token is drawn from: largest logit and sum, the target's and the draft's
    int32_t kept;         // drafts that stay
    int32_t status;
    int32_t kind;         // below
    int32_t best;         // the row's largest logit's place
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
    Verdict *verdicts;          // [B]
    int64_t ld, draft_ld;
    int32_t T, V, Vd, B, max_rows, chunks, draft_chunks;
};

__device__ __forceinline__ float load(const float *p) { return *p; }
__device__ __forceinline__ float load(const uint16_t *p) { return bf16_to_f32(*p); }

__device__ __forceinline__ bool usable(const Args &a, int b, int &t0, int &n) {
    t0 = a.starts[b];
    n = a.starts[b + 1] - t0;
    return t0 >= 0 && n >= 0 && (int64_t)t0 + n <= a.T && n <= a.max_rows;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// exp(x / t) for x <= 0 (x -inf: 0).
__device__ __forceinline__ double weight(double x, double over_t) { return exp(x * over_t); }

template <typename T>
__global__ void __launch_bounds__(kThreads) accept_parts_kernel(const Args a) {
    __shared__ int found;
    __shared__ float tops[4];
    __shared__ int ats[4];
    __shared__ double sums[4];
    const int chunk = blockIdx.x;
    const int64_t row = blockIdx.y % a.T;
    const bool draft = blockIdx.y >= (unsigned)a.T;
    if (chunk >= (draft ? a.draft_chunks : a.chunks)) return;
    if (threadIdx.x == 0) found = -1;
    __syncthreads();
    for (int b = threadIdx.x; b < a.B; b += kThreads) {
        int t0, n;
        if (usable(a, b, t0, n) && row >= t0 && row < t0 + n - (draft ? 1 : 0)) found = b;  // a last row has no draft
    }
    __syncthreads();
    if (found < 0) return;
    const float temp = a.temperature[found];
    const int V = draft ? a.Vd : a.V, first = chunk * kChunk;
    const T *p = static_cast<const T *>(draft ? a.draft_logits : a.logits) + row * (draft ? a.draft_ld : a.ld) + first;
    float x[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int at = threadIdx.x + i * kThreads;
        x[i] = first + at < V ? load(p + at) : -INFINITY;
    }
    float top = -INFINITY;
    int at = 0x7fffffff;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        nan |= x[i] != x[i];
        if (x[i] > top) top = x[i], at = first + threadIdx.x + i * kThreads;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float o = __shfl_xor(top, d);
        const int oa = __shfl_xor(at, d);
        if (o > top || (o == top && oa < at)) top = o, at = oa;
    }
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top, ats[threadIdx.x >> 6] = at;
    nan = __syncthreads_or(nan);
    top = tops[0], at = ats[0];
#pragma unroll
    for (int w = 1; w < 4; ++w)
        if (tops[w] > top || (tops[w] == top && ats[w] < at)) top = tops[w], at = ats[w];
    double sum = 0.0;
    if (temp > 0.f && top > -INFINITY && top < INFINITY) {
        const double over_t = 1.0 / (double)temp;
#pragma unroll
        for (int i = 0; i < kEach; ++i) sum += weight((double)x[i] - (double)top, over_t);
    }
    sum = wave_sum(sum);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0)
        (draft ? a.draft_parts + row * a.draft_chunks : a.parts + row * a.chunks)[chunk] = Part{(sums[0] + sums[1]) + (sums[2] + sums[3]), top, nan ? -1 : at};
}

// A row's largest logit, its place (-1: a NaN) and its sum, by one wave, in all lanes.
__device__ __forceinline__ void row_stats(const Part *parts, int chunks, double over_t, float &m, int &at, double &z) {
    const int lane = threadIdx.x & 63;
    float top = -INFINITY;
    at = 0x7fffffff;
    bool nan = false;
    for (int c = lane; c < chunks; c += 64) {
        const Part p = parts[c];
        nan |= p.at < 0;
        if (p.top > top) top = p.top, at = p.at;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float o = __shfl_xor(top, d);
        const int oa = __shfl_xor(at, d);
        if (o > top || (o == top && oa < at)) top = o, at = oa;
    }
    if (__any(nan)) at = -1;
    m = top;
    double sum = 0.0;
    if (top > -INFINITY && top < INFINITY)
        for (int c = lane; c < chunks; c += 64) {
            const Part p = parts[c];
            if (p.top > -INFINITY) sum += p.sum * weight((double)p.top - (double)top, over_t);
        }
    z = wave_sum(sum);
}

// Every thread of the block calls it; the verdict is in `v` (LDS) for all of them.
template <typename T>
__device__ __forceinline__ void decide(const Args &a, int b, Verdict &v, uint8_t *fate, double *stats) {
    int t0, n;
    const bool ok = usable(a, b, t0, n);
    if (!ok || n == 0) {
        if (threadIdx.x == 0) v = Verdict{0, 0, 0, 0, 0, ok ? 0 : -1, kNone, 0};
        __syncthreads();
        return;
    }
    const float temp = a.temperature[b];
    const bool greedy = temp <= 0.f;
    const double over_t = greedy ? 0.0 : 1.0 / (double)temp;
    const int wave = threadIdx.x >> 6;
    for (int i = wave; i < n; i += kThreads / 64) {
        const int64_t t = t0 + i;
        float m, mq = 0.f;
        int at, atq = 0;
        double z, zq = 1.0;
        row_stats(a.parts + t * a.chunks, a.chunks, over_t, m, at, z);
        bool bad = at < 0 || !(fabsf(m) < INFINITY) || !(fabsf(temp) < INFINITY), stays = false;
        if (i + 1 < n) {
            const int d = a.drafts[t];
            if (d < 0 || d >= a.V) {
                bad = true;
            } else if (greedy) {
                stays = d == at;
            } else if (!bad) {
                double q = 1.0;
                if (a.draft_logits != nullptr) {
                    row_stats(a.draft_parts + t * a.draft_chunks, a.draft_chunks, over_t, mq, atq, zq);
                    bad = atq < 0 || !(fabsf(mq) < INFINITY);
                    q = d < a.Vd ? weight((double)load(static_cast<const T *>(a.draft_logits) + t * a.draft_ld + d) - (double)mq, over_t) / zq : 0.0;
                }
                const double p = weight((double)load(static_cast<const T *>(a.logits) + t * a.ld + d) - (double)m, over_t) / z;
                stays = a.u[2 * t] * q < p;
            }
        }
        if ((threadIdx.x & 63) == 0) {
            fate[i] = bad ? 2 : stays ? 1 : 0;
            double *s = stats + 5 * i;
            s[0] = m, s[1] = z, s[2] = mq, s[3] = zq, s[4] = at;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int j = 0;
        while (fate[j] == 1) ++j;  // the last row has no draft: it is 0 or 2
        const double *s = stats + 5 * j;
        const bool last = j + 1 == n;
        v = Verdict{s[0], s[1], s[2], s[3], j, fate[j] == 2 ? 1 + j : 0,
                    fate[j] == 2 ? kNone : greedy ? kGreedy : last ? kTarget : a.draft_logits != nullptr ? kRest : kHole, (int)s[4]};
    }
    __syncthreads();
}

// Place i's weight in the row a token is drawn from. Only ratios to the row's total count: kTarget and kHole leave z out.
template <typename T>
__device__ __forceinline__ double place(const Args &a, const Verdict &v, int64_t row, double over_t, int i, int kind) {
    const double p = weight((double)load(static_cast<const T *>(a.logits) + row * a.ld + i) - v.m, over_t);
    if (kind == kTarget) return p;
    if (kind == kHole) return i == a.drafts[row] ? 0.0 : p;
    const double q = i < a.Vd ? weight((double)load(static_cast<const T *>(a.draft_logits) + row * a.draft_ld + i) - v.mq, over_t) / v.zq : 0.0;
    return fmax(p / v.z - q, 0.0);
}

__device__ __forceinline__ double block_sum(double v, double *part) {
    v = wave_sum(v);
    __syncthreads();  // part may still be read
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) accept_rest_kernel(const Args a) {
    __shared__ Verdict v;
    __shared__ uint8_t fate[kMaxRows];
    __shared__ double stats[5 * kMaxRows], part[4];
    const int b = blockIdx.y, chunk = blockIdx.x;
    decide<T>(a, b, v, fate, stats);
    if (chunk == 0 && threadIdx.x == 0) a.verdicts[b] = v;
    if (v.kind != kRest) return;
    const int64_t row = a.starts[b] + v.kept;
    const double over_t = 1.0 / (double)a.temperature[b];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int at = chunk * kChunk + i * kThreads + threadIdx.x;
        if (at < a.V) sum += place<T>(a, v, row, over_t, at, kRest);
    }
    sum = block_sum(sum, part);
    if (threadIdx.x == 0) a.rest[(int64_t)b * a.chunks + chunk] = sum;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) accept_pick_kernel(const Args a) {
    __shared__ Verdict v;
    __shared__ uint8_t fate[kMaxRows];
    __shared__ double stats[5 * kMaxRows], part[4], before[kThreads];
    __shared__ int chosen;
    const int b = blockIdx.x;
    if (a.draft_logits == nullptr) {
        decide<T>(a, b, v, fate, stats);
    } else {
        if (threadIdx.x == 0) v = a.verdicts[b];
        __syncthreads();
    }
    int t0, n;
    usable(a, b, t0, n);
    const int64_t row = (int64_t)t0 + v.kept;
    int token = -1;
    if (v.kind == kGreedy) token = v.best;
    if (v.kind == kTarget || v.kind == kHole || v.kind == kRest) {
        const double over_t = 1.0 / (double)a.temperature[b];
        int kind = v.kind;
        // weights of thread t's run of chunks; a row that has nothing left over the draft's is drawn from p
        const int per = (a.chunks + kThreads - 1) / kThreads, c0 = min((int)threadIdx.x * per, a.chunks), c1 = min(c0 + per, a.chunks);
        const int hole = kind == kHole ? a.drafts[row] / kChunk : -1;
        auto of_chunk = [&](int c) {
            if (kind == kRest) return a.rest[(int64_t)b * a.chunks + c];
            const Part p = a.parts[row * a.chunks + c];
            return p.top > -INFINITY ? p.sum * weight((double)p.top - v.m, over_t) : 0.0;
        };
        double hole_sum = 0.0, mine = 0.0, total = 0.0;
        for (int pass = 0; pass < 2; ++pass) {
            if (kind == kHole) {  // the draft's chunk without it: by taking it off, what is left would be noise
                double s = 0.0;
                for (int i = threadIdx.x; i < kChunk; i += kThreads)
                    if (hole * kChunk + i < a.V) s += place<T>(a, v, row, over_t, hole * kChunk + i, kHole);
                hole_sum = block_sum(s, part);
            }
            mine = 0.0;
            for (int c = c0; c < c1; ++c) mine += kind == kHole && c == hole ? hole_sum : of_chunk(c);
            total = block_sum(mine, part);
            if (total > 0.0 || kind == kTarget) break;
            kind = kTarget;
        }
        const double goal = a.u[2 * row + 1] * total;
        if (threadIdx.x == 0) chosen = -1;
        before[threadIdx.x] = mine;
        __syncthreads();
        if (threadIdx.x == 0) {  // the chunk in which the running sum passes the goal (rounding left it out: the last with anything)
            double run = 0.0;
            int last = 0;
            double last_run = 0.0;
            for (int t = 0; t < kThreads && chosen < 0; ++t) {
                if (t * per >= a.chunks) break;
                if (before[t] > 0.0 && run + before[t] > goal) {
                    for (int c = t * per; c < min((t + 1) * per, a.chunks); ++c) {
                        const double w = kind == kHole && c == hole ? hole_sum : of_chunk(c);
                        if (w > 0.0) last = c, last_run = run;
                        if (run + w > goal) {
                            chosen = c, part[0] = run;
                            break;
                        }
                        run += w;
                    }
                } else {
                    if (before[t] > 0.0)
                        for (int c = t * per; c < min((t + 1) * per, a.chunks); ++c) {
                            const double w = kind == kHole && c == hole ? hole_sum : of_chunk(c);
                            if (w > 0.0) last = c, last_run = run;
                            run += w;
                        }
                }
            }
            if (chosen < 0) chosen = last, part[0] = last_run;
        }
        __syncthreads();
        const int first = chosen * kChunk;
        const double run0 = part[0];
        // in the chunk: eight neighbouring places a thread
        double w[kEach], own = 0.0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int at = first + threadIdx.x * kEach + i;
            w[i] = at < a.V ? place<T>(a, v, row, over_t, at, kind) : 0.0;
            own += w[i];
        }
        __syncthreads();
        double run = own;  // of the wave's lanes up to this one
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double x = __shfl_up(run, d);
            if ((threadIdx.x & 63) >= d) run += x;
        }
        if ((threadIdx.x & 63) == 63) before[threadIdx.x >> 6] = run;
        if (threadIdx.x == 0) chosen = 0x7fffffff;
        __syncthreads();
        run += run0 - own;
        for (int w2 = 0; w2 < (int)(threadIdx.x >> 6); ++w2) run += before[w2];
        int pass = 0x7fffffff, some = -1;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            run += w[i];
            const int at = first + threadIdx.x * kEach + i;
            if (w[i] > 0.0) {
                some = at;
                if (run > goal) pass = min(pass, at);
            }
        }
        atomicMin(&chosen, pass);
        __syncthreads();
        token = chosen;
        if (token == 0x7fffffff) {  // rounding between the chunk's sum and its places: the last place with anything
            __syncthreads();
            if (threadIdx.x == 0) chosen = -1;
            __syncthreads();
            atomicMax(&chosen, some);
            __syncthreads();
            token = chosen;
        }
    }
    const int kept = v.kept;
    for (int i = threadIdx.x; i < a.max_rows; i += kThreads)
        a.tokens[(int64_t)b * a.max_rows + i] = i < kept ? a.drafts[t0 + i] : i == kept ? token : -1;
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
    s.bytes = s.parts + s.draft_parts + s.rest + (Vd > 0 ? B * (int64_t)sizeof(Verdict) : 0);
    return s;
}

template <typename T>
void launch(const Args &a, hipStream_t s) {
    const bool drafted = a.draft_logits != nullptr;
    accept_parts_kernel<T><<<dim3((unsigned)std::max(a.chunks, a.draft_chunks), (unsigned)(drafted ? 2 * a.T : a.T)), kThreads, 0, s>>>(a);
    if (drafted) accept_rest_kernel<T><<<dim3((unsigned)a.chunks, (unsigned)a.B), kThreads, 0, s>>>(a);
    accept_pick_kernel<T><<<(unsigned)a.B, kThreads, 0, s>>>(a);
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
                 reinterpret_cast<Verdict *>(w + z.parts + z.draft_parts + z.rest), ld, draft_ld, (int32_t)T, (int32_t)V, (int32_t)Vd, (int32_t)B,
                 (int32_t)max_rows, (int32_t)z.chunks, (int32_t)z.draft_chunks};
    if (act == SX_ACT_F32) launch<float>(a, stream_of(stream));
    else launch<uint16_t>(a, stream_of(stream));
    SX_LAUNCHED("mtp_accept_sampled T=", T, " batch=", B);
    return SX_OK;
}
