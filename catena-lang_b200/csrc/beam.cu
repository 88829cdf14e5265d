// Beam search's selection: of all beams x vocabulary continuations of a request the k with the greatest
//   total(w, i) = score[w] + log softmax(logits[w])[i] = score[w] + ((x - max) - log sum exp(x - max))
// in descending order; ties: the lowest beam, then the greater logit, then the lowest token.  Stands beside tensor.argmax-f32 (the greedy choice).
//
// One pass over the logits.  Launch 1: a CTA takes a chunk of one beam's row and leaves the chunk's maximum, its sum of
// exp(x - max) and its k greatest logits in order.  Launch 2: one CTA per request joins the sums and picks the k best totals.
// Candidates of different beams can lie closer together than f32 resolves, so the joined sums and the totals are f64 (a few thousand of them);
// within a beam the order is the logits' own.
// Bound: HBM, every logit is read once.
//
// The k greatest of n values without sorting them: every thread knows the greatest of its own values; the k-th greatest of those
// maxima is a limit below which nothing can be among the k greatest, and few values reach it.  Keys (value, lowest index first)
// are unique, so at most k threads hold such values and the survivors fit a buffer of fixed size, whatever the data are.
#include <math.h>

#include "paged.cuh"

namespace catena {
namespace beam {

using paged::pdl_trigger;
using paged::pdl_wait;

constexpr int kThreads = 256;
constexpr int kPer = 16;                              // logits per thread and step
constexpr int kStep = kThreads * kPer;
constexpr uint32_t kMaxK = 64, kMaxBeams = 64;
constexpr uint32_t kMaxLists = kThreads;              // chunks of one request: one per thread of the second launch

// what a chunk leaves: its maximum and sum, and its k greatest logits as (order-preserving bits << 32 | ~token), descending;
// fewer than k are followed by zeros
struct Chunk {
    float2* stats;        // [rows][splits]
    uint64_t* keys;       // [rows][splits][k]
};

__device__ __forceinline__ float take(float x) {      // NaN: never chosen; +inf: the greatest finite value, so that totals are numbers
    return x != x ? -INFINITY : fminf(x, 3.402823466e38f);
}
__device__ __forceinline__ uint32_t order_bits(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);     // -0 as +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t bits) { return __uint_as_float(bits & 0x80000000u ? bits & 0x7FFFFFFFu : ~bits); }

// the k-th greatest of the threads' maxima (0 when fewer than k threads hold anything); whole CTA
__device__ __forceinline__ uint64_t limit_of(uint64_t mine, uint32_t k, uint64_t* tops, uint64_t* limit) {
    tops[threadIdx.x] = mine;
    if (threadIdx.x == 0) *limit = 0;
    __syncthreads();
    if (mine) {
        uint32_t rank = 0;
        for (int j = 0; j < kThreads; ++j) rank += tops[j] > mine;
        if (rank == k - 1) *limit = mine;
    }
    __syncthreads();
    return *limit;
}

template <class T> __device__ __forceinline__ void load_logits(const T* __restrict__ row, uint32_t at, uint32_t end, bool vec, float (&x)[kPer]);
template <> __device__ __forceinline__ void load_logits<float>(const float* __restrict__ row, uint32_t at, uint32_t end, bool vec, float (&x)[kPer]) {
    if (vec && at + kPer <= end) {
#pragma unroll
        for (int u = 0; u < kPer / 4; ++u) {
            const float4 v = __ldg(reinterpret_cast<const float4*>(row + at) + u);
            x[4 * u] = v.x; x[4 * u + 1] = v.y; x[4 * u + 2] = v.z; x[4 * u + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int u = 0; u < kPer; ++u) x[u] = at + u < end ? row[at + u] : 0.0f;
    }
}
template <> __device__ __forceinline__ void load_logits<__nv_bfloat16>(const __nv_bfloat16* __restrict__ row, uint32_t at, uint32_t end, bool vec, float (&x)[kPer]) {
    if (vec && at + kPer <= end) {
#pragma unroll
        for (int u = 0; u < kPer / 8; ++u) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + at) + u);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[8 * u + 2 * e] = __uint_as_float(w[e] << 16);
                x[8 * u + 2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
            }
        }
    } else {
#pragma unroll
        for (int u = 0; u < kPer; ++u) x[u] = at + u < end ? __bfloat162float(row[at + u]) : 0.0f;
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) beam_chunk_kernel(const T* __restrict__ logits, uint64_t pitch, uint32_t vocab, uint32_t k, uint32_t chunk,
                                                              uint32_t vec, Chunk out) {
    __shared__ uint64_t cand[kMaxK + kMaxK * kPer];       // the k kept so far, and what a step adds
    __shared__ uint64_t best[kMaxK];
    __shared__ uint64_t tops[kThreads];
    __shared__ uint64_t s_limit;
    __shared__ uint32_t s_n;
    __shared__ float2 warp_ml[kThreads / 32];
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x, row = blockIdx.y, split = blockIdx.x;
    const uint32_t begin = split * chunk, end = min(vocab, begin + chunk);
    const T* x_row = logits + (size_t)row * pitch;
    float m = -INFINITY, sum = 0.0f;
    for (uint32_t i = tid; i < k; i += kThreads) best[i] = 0;
    for (uint32_t s0 = begin; s0 < end; s0 += kStep) {
        const uint32_t at = s0 + tid * kPer;
        float x[kPer];
        load_logits<T>(x_row, at, end, vec != 0, x);
        float top = -INFINITY;
        uint64_t mine = 0;
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            x[u] = take(x[u]);
            if (at + u < end) {
                if (!mine || x[u] > top) mine = ((uint64_t)order_bits(x[u]) << 32) | (uint32_t)~(at + u);
                top = fmaxf(top, x[u]);
            }
        }
        if (top > m) {
            sum = __fmul_rn(sum, __expf(__fsub_rn(m, top)));
            m = top;
        }
        if (m != -INFINITY) {
#pragma unroll
            for (int u = 0; u < kPer; ++u)
                if (at + u < end) sum = __fadd_rn(sum, __expf(__fsub_rn(x[u], m)));
        }
        __syncthreads();                                  // `best` of the last step is complete, `cand` is free
        const uint64_t kth = best[k - 1];                 // a key below it is not among the k greatest
        const uint64_t limit = max(limit_of(mine > kth ? mine : 0, k, tops, &s_limit), kth + 1);
        for (uint32_t i = tid; i < k; i += kThreads) cand[i] = best[i];
        if (tid == 0) s_n = 0;
        __syncthreads();
        if (mine >= limit) {
#pragma unroll
            for (int u = 0; u < kPer; ++u) {
                const uint64_t key = ((uint64_t)order_bits(x[u]) << 32) | (uint32_t)~(at + u);
                if (at + u < end && key >= limit) cand[k + atomicAdd(&s_n, 1u)] = key;
            }
        }
        __syncthreads();
        const uint32_t n = s_n;
        if (n) {
            // zeros in the part kept so far rank behind every key; equal keys (zeros only) are not written
            for (uint32_t i = tid; i < k + n; i += kThreads) {
                const uint64_t key = cand[i];
                uint32_t rank = 0;
                for (uint32_t j = 0; j < k + n; ++j) rank += cand[j] > key;
                if (key && rank < k) best[rank] = key;
            }
        }
    }
    // the chunk's maximum and sum
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
        const float m2 = __shfl_xor_sync(0xFFFFFFFFu, m, off), s2 = __shfl_xor_sync(0xFFFFFFFFu, sum, off);
        const float top = fmaxf(m, m2);
        sum = top == -INFINITY ? 0.0f : __fadd_rn(__fmul_rn(sum, __expf(__fsub_rn(m, top))), __fmul_rn(s2, __expf(__fsub_rn(m2, top))));
        m = top;
    }
    if ((tid & 31) == 0) warp_ml[tid >> 5] = make_float2(m, sum);
    __syncthreads();
    const size_t at_out = (size_t)row * gridDim.x + split;
    if (tid == 0) {
        float top = -INFINITY, s = 0.0f;
        for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, warp_ml[w].x);
        if (top != -INFINITY)
            for (int w = 0; w < kThreads / 32; ++w) s = __fadd_rn(s, __fmul_rn(warp_ml[w].y, __expf(__fsub_rn(warp_ml[w].x, top))));
        out.stats[at_out] = make_float2(top, s);
    }
    for (uint32_t i = tid; i < k; i += kThreads) out.keys[at_out * k + i] = best[i];
}

struct Total {
    uint64_t total;       // order-preserving bits of the f64 total
    uint64_t key;         // (logit, token) as in Chunk
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
// (logit - max) first: a row of the lowest value throughout is uniform, not of probability 1
__device__ __forceinline__ Total total_of(uint64_t key, uint32_t beam, float score, double top, double log_sum) {
    const float x = value_of((uint32_t)(key >> 32));
    double t = x == -INFINITY ? -INFINITY : (double)score + (((double)x - top) - log_sum);
    if (t != t) t = -INFINITY;
    return {order_bits64(t), key, beam};
}

// One CTA per request; thread i < beams * splits looks after chunk i.  The limit is the k-th best of the chunks' first entries, so
// at most k chunks hold survivors, k each.
__global__ void __launch_bounds__(kThreads) beam_pick_kernel(Chunk in, const float* __restrict__ scores, uint32_t beams, uint32_t splits, uint32_t k,
                                                             float* __restrict__ out_scores, int32_t* __restrict__ out_parents,
                                                             int32_t* __restrict__ out_tokens) {
    extern __shared__ __align__(16) uint8_t smem[];
    Total* cand = reinterpret_cast<Total*>(smem);                 // [k * k]
    __shared__ Total tops[kThreads];
    __shared__ double s_top[kMaxBeams], s_log[kMaxBeams];
    __shared__ Total s_limit;
    __shared__ uint32_t s_n, s_bounded;
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x, req = blockIdx.x, lists = beams * splits;
    const size_t first = (size_t)req * lists;
    if (tid < beams) {
        const float2* st = in.stats + first + (size_t)tid * splits;
        float top = -INFINITY;
        for (uint32_t i = 0; i < splits; ++i) top = fmaxf(top, st[i].x);
        double sum = 0.0;
        if (top != -INFINITY)
            for (uint32_t i = 0; i < splits; ++i) sum += (double)st[i].y * exp((double)st[i].x - (double)top);
        s_top[tid] = top;
        s_log[tid] = log(sum);
    }
    if (tid == 0) { s_n = 0; s_bounded = 0; }
    __syncthreads();
    const uint32_t beam = tid / splits;
    const uint64_t* keys = in.keys + (first + tid) * k;
    Total head = {0, 0, 0};
    float score = 0.0f;
    double top = 0.0, log_sum = 0.0;
    if (tid < lists) {
        score = scores[(size_t)req * beams + beam];
        top = s_top[beam];
        log_sum = s_log[beam];
        if (keys[0]) head = total_of(keys[0], beam, score, top, log_sum);
    }
    tops[tid] = head;
    __syncthreads();
    if (head.total) {
        uint32_t rank = 0;
        for (uint32_t j = 0; j < lists; ++j) rank += ahead(tops[j], head);
        if (rank == k - 1) { s_limit = head; s_bounded = 1; }
    }
    __syncthreads();
    if (head.total) {
        const bool bounded = s_bounded != 0;
        const Total limit = s_limit;
        for (uint32_t i = 0; i < k; ++i) {
            const uint64_t key = keys[i];
            if (!key) break;
            const Total t = total_of(key, beam, score, top, log_sum);
            if (bounded && ahead(limit, t)) break;
            cand[atomicAdd(&s_n, 1u)] = t;
        }
    }
    __syncthreads();
    const uint32_t n = s_n;
    for (uint32_t i = tid; i < n; i += kThreads) {
        const Total mine = cand[i];
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n; ++j) rank += ahead(cand[j], mine);
        if (rank < k) {
            const size_t o = (size_t)req * k + rank;
            out_scores[o] = (float)value_of64(mine.total);
            out_parents[o] = (int32_t)mine.beam;
            out_tokens[o] = (int32_t)~(uint32_t)mine.key;
        }
    }
}

// ---------------------------------------------------------------- host side
struct Plan {
    uint32_t splits, chunk;
    uint64_t keys, bytes;
};
static Plan plan_for(uint64_t batch, uint64_t beams, uint64_t vocab, uint64_t k) {
    Plan p = {};
    const uint64_t rows = batch * beams;
    const int sms = tls().sm_count > 0 ? tls().sm_count : 148;
    // chunks of one step, unless that makes more CTAs than four waves or more chunks than a request may have
    uint64_t splits = ceil_div_u64(vocab, kStep);
    const uint64_t fit = ceil_div_u64((uint64_t)sms * 4 * 4, rows), most = kMaxLists / beams;
    if (splits > fit) splits = fit;
    if (splits > most) splits = most;
    const uint64_t chunk = ceil_div_u64(ceil_div_u64(vocab, splits), kPer) * kPer;
    p.chunk = (uint32_t)chunk;
    p.splits = (uint32_t)ceil_div_u64(vocab, chunk);
    p.keys = (rows * p.splits * sizeof(float2) + 255) & ~255ull;
    p.bytes = p.keys + rows * p.splits * k * sizeof(uint64_t);
    return p;
}
static catena_status_t check_sizes(uint64_t batch, uint64_t beams, uint64_t vocab, uint64_t k) {
    if (!beams || !vocab || !k) return fail(CATENA_E_BAD_ARG, "beam_select: no beams, vocabulary or places");
    if (beams > kMaxBeams || k > kMaxK) return fail(CATENA_E_UNSUPPORTED, "beam_select: at most 64 beams and 64 places");
    if (vocab > 0x7FFFFFFFull - kStep || batch > 0xFFFFull || batch * beams > 0xFFFFull) return fail(CATENA_E_TOO_LARGE, "beam_select: more rows or tokens than the kernels index");
    if (k > beams * vocab) return fail(CATENA_E_BAD_ARG, "beam_select: fewer continuations than places");
    return CATENA_OK;
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
    uint32_t* err;
    CATENA_TRY(paged::begin(&err));
    const Plan p = plan_for(batch, beams, vocab, k);
    if (workspace_bytes < p.bytes) return fail(CATENA_E_BAD_ARG, "beam_select: workspace too small");
    const Chunk chunks = {(float2*)workspace, (uint64_t*)((uint8_t*)workspace + p.keys)};
    const uint32_t vec = paged::aligned16(logits) && pitch * sizeof(T) % 16 == 0;
    CATENA_TRY(paged::launch("beam_chunk_kernel", beam_chunk_kernel<T>, dim3(p.splits, (unsigned)(batch * beams)), dim3(kThreads), 0, logits, pitch,
                             (uint32_t)vocab, (uint32_t)k, p.chunk, vec, chunks));
    const size_t smem = k * k * sizeof(Total);
    if (smem > 32768) CATENA_CUDA(cudaFuncSetAttribute(beam_pick_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxK * kMaxK * sizeof(Total)));
    CATENA_TRY(paged::launch("beam_pick_kernel", beam_pick_kernel, dim3((unsigned)batch), dim3(kThreads), smem, chunks, scores, (uint32_t)beams,
                             p.splits, (uint32_t)k, out_scores, out_parents, out_tokens));
    return paged::end();
}

}  // namespace beam

extern "C" {

uint64_t catena_b200_beam_select_workspace_bytes(uint64_t batch, uint64_t beams, uint64_t vocab, uint64_t k) {
    if (!batch || beam::check_sizes(batch, beams, vocab, k) != CATENA_OK) return 0;
    return beam::plan_for(batch, beams, vocab, k).bytes;
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
