// Beam search's selection: of all beams x vocabulary continuations of a request the k with the greatest
//   total(w, i) = score[w] + log softmax(logits[w])[i] = score[w] + ((x - max) - log sum exp(x - max))
// in descending order; ties: the lowest beam, then the greater logit, then the lowest token.
// Stands beside tensor.argmax-f32 (the greedy choice).
//
// Launch 1 reads every logit once: a warp takes a segment of a row (1024 logits, fewer where a request has few) and leaves its maximum
// and its sum of exp(x - max).  That is all it does, so it runs at the memory's rate: no warp waits for another.
// Launch 2, one CTA per request, joins the sums, and looks for the k best among the segments' maxima: a segment whose maximum is
// behind k others cannot hold one of the k best, so about k segments are read again (from L2) and give the few candidates, which are
// ranked by comparing them with each other.  Keeping k candidates per segment in launch 1 instead cost twice its time (45 against
// 23 us for 32 x 8 rows of 128000 f32, 5.6 TB/s): almost all of them lose to another segment.
// Candidates of different beams can lie closer together than a total in f32 resolves, so the joined sums and the totals are f64; what
// they can tell apart is limited by the segments' sums in f32, below 2^-19 of themselves.  Segments are counted from a row's start
// whatever its alignment, so equal rows have equal sums and their ties are ties.
#include <math.h>

#include "catena_math.cuh"
#include "paged.cuh"

namespace catena {
namespace beam {

using paged::pdl_trigger;
using paged::pdl_wait;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPer = 32;                              // logits per lane of a whole segment
constexpr uint32_t kMaxK = 64, kMaxBeams = 64;
constexpr uint32_t kRoom = 256;                       // candidates that are ranked by mutual comparison
constexpr float kLog2e = 1.44269504f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float exp_of(float x) { return ex2(__fmul_rn(x, kLog2e)); }
__device__ __forceinline__ float take(float x) {      // NaN: never chosen; +inf: the greatest finite value, so that totals are numbers
    return x != x ? -INFINITY : fminf(x, 3.402823466e38f);
}
__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);     // -0 as +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t bits) { return __uint_as_float(bits & 0x80000000u ? bits & 0x7FFFFFFFu : ~bits); }

template <class T> struct Piece;                      // 16 bytes of logits
template <> struct Piece<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void load(const float* p, float* x) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p));
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <> struct Piece<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* x) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
};

// the rows of logits and how they are cut
template <class T> struct Rows {
    const T* logits;
    uint64_t pitch;
    uint32_t vocab, segs;     // segments of a row
    uint32_t pieces;          // 16-byte pieces per lane of a segment
    uint32_t vec;             // rows start on 16-byte boundaries

    static constexpr int N = Piece<T>::kN;
    __device__ __forceinline__ uint32_t index(uint32_t seg, int u, uint32_t lane) const {
        return seg * (pieces * 32 * N) + (u / N * 32 + lane) * N + u % N;
    }
    // a lane's logits of a segment; behind the row's or the segment's end: -inf
    __device__ __forceinline__ void load(uint32_t row, uint32_t seg, uint32_t lane, float (&x)[kPer]) const {
        const T* p = logits + (size_t)row * pitch;
#pragma unroll
        for (int u = 0; u < kPer; u += N) {
            const uint32_t at = index(seg, u, lane);
            const bool mine = (uint32_t)u / N < pieces;
            if (vec && mine && at + N <= vocab) {
                Piece<T>::load(p + at, x + u);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) x[u + e] = mine && at + e < vocab ? Piece<T>::one(p + at + e) : -INFINITY;
            }
        }
    }
};

// ---------------------------------------------------------------- launch 1
__device__ __forceinline__ float warp_max(float x) { return value_of(__reduce_max_sync(0xFFFFFFFFu, order_bits(x))); }
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) x = __fadd_rn(x, __shfl_xor_sync(0xFFFFFFFFu, x, off));
    return x;
}

template <class T>
__global__ void __launch_bounds__(kThreads) beam_stats_kernel(Rows<T> rows, uint64_t n, float2* __restrict__ stats) {
    pdl_trigger();
    pdl_wait();
    const uint64_t at = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);       // (row, segment)
    if (at >= n) return;
    const uint32_t lane = threadIdx.x & 31;
    float x[kPer];
    rows.load((uint32_t)(at / rows.segs), (uint32_t)(at % rows.segs), lane, x);
    float top = x[0];
#pragma unroll
    for (int u = 1; u + 1 < kPer; u += 2) top = cmath::max3(top, x[u], x[u + 1]);
    top = fmaxf(top, x[kPer - 1]);
    float m = warp_max(top), sum;
    {
        // sum of 2^(x log2 e - r), r = m log2 e rounded; the factor takes the rounding of r out again.  Two values per instruction.
        const float r = __fmul_rn(m, kLog2e), off = __fmaf_rn(m, kLog2e, -r);
        const uint64_t l2 = cmath::pk2f(kLog2e, kLog2e), r2 = cmath::pk2f(-r, -r);
        uint64_t s2 = 0;
#pragma unroll
        for (int u = 0; u < kPer; u += 2) {
            if ((uint32_t)u / Rows<T>::N >= rows.pieces) break;
            float a, b;
            cmath::unpk2f(cmath::fma2(cmath::pk2f(x[u], x[u + 1]), l2, r2), a, b);
            s2 = cmath::add2(s2, cmath::pk2f(ex2(a), ex2(b)));
        }
        float a, b;
        cmath::unpk2f(s2, a, b);
        sum = __fmul_rn(warp_sum(__fadd_rn(a, b)), __fmaf_rn(off, -0.693147181f, 1.0f));
    }
    if (sum != sum || fabsf(m) > 1e37f) {                 // a NaN, an infinity, nothing but -inf, or m log2 e overflows; whole warp
        top = -INFINITY;
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            x[u] = take(x[u]);
            top = fmaxf(top, x[u]);
        }
        m = warp_max(top);
        sum = 0.0f;
        if (m != -INFINITY) {
#pragma unroll
            for (int u = 0; u < kPer; ++u) sum = __fadd_rn(sum, exp_of(__fsub_rn(x[u], m)));
            sum = warp_sum(sum);
        }
    }
    if (lane == 0) stats[at] = make_float2(m, sum);
}

// ---------------------------------------------------------------- launch 2
constexpr int kPickThreads = 1024;
constexpr int kPickWarps = kPickThreads / 32;
constexpr int kBests = 2 * kMaxK + kPickWarps;        // values among which the limit is looked for

struct Total {
    uint64_t total;       // order-preserving bits of the f64 total; 0: none
    uint64_t key;         // order-preserving bits of the logit << 32 | ~token
    uint64_t beam;
};
__device__ __forceinline__ bool ahead(const Total& a, const Total& b) {
    return a.total > b.total || (a.total == b.total && (a.beam < b.beam || (a.beam == b.beam && a.key > b.key)));
}
__device__ __forceinline__ uint64_t order_bits64(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double value_of64(uint64_t bits) {
    return __longlong_as_double((long long)(bits >> 63 ? bits & ~(1ull << 63) : ~bits));
}
struct Beams {
    double top[kMaxBeams], log_sum[kMaxBeams], score[kMaxBeams];
    float off[kMaxBeams];            // score - top - log_sum in f32; -inf for a beam that goes nowhere
    // (x - max) first: a row of the lowest value throughout is uniform, not of probability 1
    __device__ __forceinline__ uint64_t total(uint32_t w, float x) const {
        double t = x == -INFINITY ? -INFINITY : score[w] + (((double)x - top[w]) - log_sum[w]);
        if (t != t) t = -INFINITY;
        return order_bits64(t);
    }
};
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) { return (uint64_t)order_bits(x) << 32 | (uint32_t)~token; }

// the best of the threads' values, to all; whole CTA
__device__ __forceinline__ Total block_best(Total mine, Total* per_warp) {
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        Total o;
        o.total = __shfl_xor_sync(0xFFFFFFFFu, mine.total, off);
        o.key = __shfl_xor_sync(0xFFFFFFFFu, mine.key, off);
        o.beam = __shfl_xor_sync(0xFFFFFFFFu, mine.beam, off);
        if (ahead(o, mine)) mine = o;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) per_warp[threadIdx.x >> 5] = mine;
    __syncthreads();
    mine = per_warp[0];
    for (int w = 1; w < kPickWarps; ++w)
        if (ahead(per_warp[w], mine)) mine = per_warp[w];
    return mine;
}

// The search for candidates is in f32: a(x) = x + off[beam], off by at most 2^-23 of |off| and of itself.  The k-th best of some of the
// segments' maxima is a limit that the true k-th best total is not below by more than those errors, so with a margin of 2^-20 of the
// magnitudes nothing that belongs to the answer is lost; what is gained too much is sorted out in f64.
template <class T>
__global__ void __launch_bounds__(kPickThreads) beam_pick_kernel(Rows<T> rows, const float2* __restrict__ stats, const float* __restrict__ scores,
                                                                 uint32_t beams, uint32_t k, float* __restrict__ out_scores,
                                                                 int32_t* __restrict__ out_parents, int32_t* __restrict__ out_tokens) {
    __shared__ Beams s_beam;
    __shared__ float s_least[kMaxBeams];
    __shared__ Total cand[kRoom], per_warp[kPickWarps];
    __shared__ __align__(16) uint32_t s_best[kBests];
    __shared__ uint32_t s_n, s_lists, s_lim, s_first, s_off, s_list[kRoom];
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, req = blockIdx.x;
    const uint32_t row0 = req * beams, segs = rows.segs, n_segs = beams * segs;
    const float2* st = stats + (size_t)row0 * segs;
    // a warp's segments are spread over all beams, which may be of very different merit
    const uint32_t seg0 = lane * kPickWarps + warp;
    const float x0 = seg0 < n_segs ? st[seg0].x : -INFINITY;
    for (uint32_t w = warp; w < beams; w += kPickWarps) {         // a warp joins a beam's sums
        const float score = scores[row0 + w];
        float top = -INFINITY;
        for (uint32_t i = lane; i < segs; i += 32) top = fmaxf(top, st[(size_t)w * segs + i].x);
        top = warp_max(top);
        double sum = 0.0;
        if (top != -INFINITY)
            for (uint32_t i = lane; i < segs; i += 32) {
                const float2 ms = st[(size_t)w * segs + i];
                sum += (double)ms.y * (double)exp_of(__fsub_rn(ms.x, top));
            }
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, off);
        if (lane == 0) {
            const double log_sum = log(sum);
            const float off = (float)((double)score - (double)top - log_sum);
            s_beam.top[w] = top;
            s_beam.log_sum[w] = log_sum;
            s_beam.score[w] = score;
            s_beam.off[w] = top == -INFINITY || off != off ? -INFINITY : off;
        }
    }
    if (tid == 0) {
        s_n = s_lists = 0;
    }
    __syncthreads();

    // Candidates: first a limit from the segments' maxima; if the segments that reach it hold too many logits that do (few segments,
    // or one beam far ahead of the others), a second one from the logits of these segments.
    const uint32_t width = rows.pieces * 32 * Rows<T>::N;
#pragma unroll 1
    for (int attempt = 0; attempt < 2; ++attempt) {
        uint32_t best = 0, best_beam = 0, n = attempt == 0 ? n_segs : s_lists * width;      // of what a thread looks at; its beam
        for (uint32_t i = attempt == 0 ? seg0 : tid; i < n; i += kPickThreads) {
            uint32_t w;
            float x;
            if (attempt == 0) {
                w = i / segs;
                x = i == seg0 ? x0 : st[i].x;
            } else {
                const uint32_t nth = i / s_lists, at = s_list[i - nth * s_lists];        // neighbours look at different segments
                w = at / segs;
                const uint32_t token = (at - w * segs) * width + nth;
                if (token >= rows.vocab) continue;
                x = take(Piece<T>::one(rows.logits + (size_t)(row0 + w) * rows.pitch + token));
            }
            const uint32_t v = order_bits(__fadd_rn(x, s_beam.off[w]));
            if (v > best) { best = v; best_beam = w; }
        }
        // the limit: of every warp's `share` best, 2 k or more in all, the k-th best
        const uint32_t active = min((attempt == 0 ? n : (n + 31) / 32), (uint32_t)kPickWarps);
        const uint32_t share = min(32u, (2 * k + active - 1) / active), bests = (active * share + 3) / 4 * 4;
        for (uint32_t i = tid; i < kBests; i += kPickThreads) s_best[i] = 0;
        __syncthreads();
        if (tid == 0) {
            s_first = s_off = s_n = 0;
            s_lim = 0xFFFFFFFFu;
        }
        uint32_t v = best;
        for (uint32_t i = 0; i < share && warp < active; ++i) {
            const uint32_t nth = __reduce_max_sync(0xFFFFFFFFu, v);
            const uint32_t holders = __ballot_sync(0xFFFFFFFFu, v == nth);
            if (lane == (uint32_t)__ffs(holders) - 1) {
                v = 0;
                s_best[warp * share + i] = nth;
            }
        }
        __syncthreads();
        if (tid < bests) {
            const uint32_t mine = s_best[tid];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < bests; j += 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(s_best + j);
                rank += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
            }
            if (rank < k) atomicMin(&s_lim, mine);                // 0 when there are fewer than k: no limit
            if (rank == 0) s_first = mine;
        }
        __syncthreads();
        const uint32_t lim = s_lim;
        if (best >= lim && best) atomicMax(&s_off, __float_as_uint(fabsf(s_beam.off[best_beam])));
        __syncthreads();
        // the least logit of each beam that can be a candidate
        if (tid < beams) {
            const double l = value_of(lim), top = value_of(s_first), off = s_beam.off[tid], most = __uint_as_float(s_off);
            const double least = l - off - 0x1p-20 * (fabs(l) + fabs(top) + fabs(off) + most);
            s_least[tid] = lim && least == least ? __double2float_rd(least) : -INFINITY;
        }
        __syncthreads();
        if (attempt == 0) {
            for (uint32_t i = seg0; i < n_segs; i += kPickThreads) {
                if ((i == seg0 ? x0 : st[i].x) < s_least[i / segs]) continue;
                const uint32_t at = atomicAdd(&s_lists, 1u);
                if (at < kRoom) s_list[at] = i;
            }
            __syncthreads();
            if (s_lists > kRoom) break;
        }
        for (uint32_t i = warp; i < s_lists; i += kPickWarps) {
            const uint32_t w = s_list[i] / segs, seg = s_list[i] - w * segs;
            const float least = s_least[w];
            float x[kPer];
            rows.load(row0 + w, seg, lane, x);
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                const float v = take(x[u]);
                if (v < least) continue;
                const uint32_t token = rows.index(seg, u, lane);
                if ((uint32_t)u / Rows<T>::N >= rows.pieces || token >= rows.vocab) continue;
                const uint32_t at = atomicAdd(&s_n, 1u);
                if (at < kRoom) cand[at] = {0, key_of(v, token), w};
            }
        }
        __syncthreads();
        if (s_n <= kRoom) break;
    }
    const uint32_t n = s_n;
    if (s_lists <= kRoom && n <= kRoom) {
        if (tid < n) cand[tid].total = s_beam.total((uint32_t)cand[tid].beam, value_of((uint32_t)(cand[tid].key >> 32)));
        __syncthreads();
        for (uint32_t i = warp; i < n; i += kPickWarps) {         // a warp ranks a candidate
            const Total mine = cand[i];
            uint32_t place = 0;
            for (uint32_t j = lane; j < n; j += 32) place += ahead(cand[j], mine);
            place = __reduce_add_sync(0xFFFFFFFFu, place);
            if (place < k && lane == 0) {
                const size_t o = (size_t)req * k + place;
                out_scores[o] = (float)value_of64(mine.total);
                out_parents[o] = (int32_t)mine.beam;
                out_tokens[o] = (int32_t)~(uint32_t)mine.key;
            }
        }
        return;
    }
    // Many equal totals: the k best segments one after the other (equal maxima: the lower segment has the lower tokens), then the
    // k best of their logits one after the other.
    Total last = {~0ull, ~0ull, 0};
    uint32_t lists = 0;
    for (; lists < k; ++lists) {
        Total mine = {0, 0, 0};
        for (uint32_t i = tid; i < n_segs; i += kPickThreads) {
            const uint32_t w = i / segs;
            const Total t = {s_beam.total(w, st[i].x), key_of(st[i].x, i - w * segs), w};
            if (ahead(last, t) && ahead(t, mine)) mine = t;
        }
        last = block_best(mine, per_warp);
        if (last.total == 0) break;
        if (tid == 0) s_list[lists] = (uint32_t)last.beam * segs + ~(uint32_t)last.key;
    }
    __syncthreads();
    last = {~0ull, ~0ull, 0};
    for (uint32_t place = 0; place < k; ++place) {
        Total mine = {0, 0, 0};
        for (uint32_t i = tid; i < lists * width; i += kPickThreads) {
            const uint32_t w = s_list[i / width] / segs, token = s_list[i / width] % segs * width + i % width;
            if (token >= rows.vocab) continue;
            const float v = take(Piece<T>::one(rows.logits + (size_t)(row0 + w) * rows.pitch + token));
            const Total t = {s_beam.total(w, v), key_of(v, token), w};
            if (ahead(last, t) && ahead(t, mine)) mine = t;
        }
        last = block_best(mine, per_warp);
        if (tid == 0) {
            const size_t o = (size_t)req * k + place;
            out_scores[o] = (float)value_of64(last.total);
            out_parents[o] = (int32_t)last.beam;
            out_tokens[o] = (int32_t)~(uint32_t)last.key;
        }
    }
}

// ---------------------------------------------------------------- host side
static catena_status_t check_sizes(uint64_t batch, uint64_t beams, uint64_t vocab, uint64_t k) {
    if (!beams || !vocab || !k) return fail(CATENA_E_BAD_ARG, "beam_select: no beams, vocabulary or places");
    if (beams > kMaxBeams || k > kMaxK) return fail(CATENA_E_UNSUPPORTED, "beam_select: at most 64 beams and 64 places");
    if (vocab > (1ull << 24) || batch > 0xFFFFull) return fail(CATENA_E_TOO_LARGE, "beam_select: at most 2^24 tokens and 65535 requests");
    if (k > beams * vocab) return fail(CATENA_E_BAD_ARG, "beam_select: fewer continuations than places");
    return CATENA_OK;
}
// Segments of 1024 logits, halved (down to one 16-byte piece per lane) until a request has 512 of them, because few segments make a poor
// limit (62 x 16 x 6574 f32: 16 us with segments of 512, 28 with 1024), or until the call has 48 warps for every SM, because a warp costs
// about the same whatever its segment holds (52 x 4 x 29213 f32: 14 us with segments of 512, 31 with 128).
static uint32_t pieces_for(uint64_t batch, uint64_t beams, uint64_t vocab, uint32_t per_piece) {
    const uint64_t sms = tls().sm_count > 0 ? tls().sm_count : 148;
    uint32_t pieces = kPer / per_piece;
    for (; pieces > 1; pieces /= 2) {
        const uint64_t segs = beams * ceil_div_u64(vocab, (uint64_t)pieces * 32 * per_piece);
        if (segs >= 512 || batch * segs >= sms * 48) break;
    }
    return pieces;
}

template <class T>
static catena_status_t select_into(const T* logits, uint64_t pitch, const float* scores, uint64_t batch, uint64_t beams, uint64_t vocab, uint64_t k,
                                   float* out_scores, int32_t* out_parents, int32_t* out_tokens, void* workspace, uint64_t workspace_bytes) {
    CATENA_TRY(check_sizes(batch, beams, vocab, k));
    if (!batch) return CATENA_OK;
    if (!logits || !scores || !out_scores || !out_parents || !out_tokens || !workspace) return fail(CATENA_E_BAD_ARG, "beam_select: null argument");
    if (((uintptr_t)logits % sizeof(T)) || !paged::aligned4(scores) || !paged::aligned4(out_scores) || !paged::aligned4(out_parents) ||
        !paged::aligned4(out_tokens) || ((uintptr_t)workspace & 255))
        return fail(CATENA_E_BAD_ARG, "beam_select: misaligned argument (the workspace is 256-byte aligned)");
    if (pitch < vocab) return fail(CATENA_E_BAD_ARG, "beam_select: rows of logits overlap");
    if (workspace_bytes < catena_b200_beam_select_workspace_bytes(batch, beams, vocab, k)) return fail(CATENA_E_BAD_ARG, "beam_select: workspace too small");
    uint32_t* err;
    CATENA_TRY(paged::begin(&err));
    Rows<T> rows = {logits, pitch, (uint32_t)vocab, 0, pieces_for(batch, beams, vocab, Piece<T>::kN), 0};
    rows.segs = (uint32_t)ceil_div_u64(vocab, rows.pieces * 32 * Piece<T>::kN);
    rows.vec = paged::aligned16(logits) && pitch * sizeof(T) % 16 == 0;
    const uint64_t n = batch * beams * rows.segs;
    if (ceil_div_u64(n, kWarps) > 0x7FFFFFFFull) return fail(CATENA_E_TOO_LARGE, "beam_select: more logits than the kernels index");
    float2* stats = static_cast<float2*>(workspace);
    CATENA_TRY(paged::launch("beam_stats_kernel", beam_stats_kernel<T>, dim3((unsigned)ceil_div_u64(n, kWarps)), dim3(kThreads), 0, rows, n, stats));
    CATENA_TRY(paged::launch("beam_pick_kernel", beam_pick_kernel<T>, dim3((unsigned)batch), dim3(kPickThreads), 0, rows, stats, scores, (uint32_t)beams,
                             (uint32_t)k, out_scores, out_parents, out_tokens));
    return paged::end();
}

}  // namespace beam

extern "C" {

uint64_t catena_b200_beam_select_workspace_bytes(uint64_t batch, uint64_t beams, uint64_t vocab, uint64_t k) {
    if (!batch || beam::check_sizes(batch, beams, vocab, k) != CATENA_OK) return 0;
    // (maximum, sum) of every segment; f32's are never longer than bf16's
    return batch * beams * ceil_div_u64(vocab, (uint64_t)beam::pieces_for(batch, beams, vocab, 4) * 32 * 4) * sizeof(float2);
}
catena_status_t catena_b200_beam_select_f32_into(const float* logits, uint64_t pitch, const float* scores, uint64_t batch, uint64_t beams,
                                                 uint64_t vocab, uint64_t k, float* out_scores, int32_t* out_parents, int32_t* out_tokens,
                                                 void* workspace, uint64_t workspace_bytes) {
    return beam::select_into<float>(logits, pitch, scores, batch, beams, vocab, k, out_scores, out_parents, out_tokens, workspace, workspace_bytes);
}
catena_status_t catena_b200_beam_select_bf16_into(const void* logits, uint64_t pitch, const float* scores, uint64_t batch, uint64_t beams,
                                                  uint64_t vocab, uint64_t k, float* out_scores, int32_t* out_parents, int32_t* out_tokens,
                                                  void* workspace, uint64_t workspace_bytes) {
    return beam::select_into<__nv_bfloat16>((const __nv_bfloat16*)logits, pitch, scores, batch, beams, vocab, k, out_scores, out_parents,
                                            out_tokens, workspace, workspace_bytes);
}

}  // extern "C"

}  // namespace catena
