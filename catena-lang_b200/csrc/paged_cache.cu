// A key/value cache in pages: rotation and append of ragged tokens, eviction by accumulated attention weight, and the hand-over
// of pages between the beams of a beam search.  (The attention that reads the pages: attn_decode_paged.cu.)
// The reference has no cache; layouts follow this library's contiguous caches [batch, n_kv_heads, rows, head_dim].
#include <cooperative_groups.h>

#include "catena_math.cuh"
#include "paged.cuh"

namespace cg = cooperative_groups;

namespace catena {
namespace paged {

// ---------------------------------------------------------------- host side shared by the paged operators
static thread_local uint32_t* g_err[kMaxDevices] = {nullptr};

catena_status_t begin(uint32_t** err) {
    CATENA_TRY(ensure_device());
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    CATENA_CUDA(cudaStreamIsCapturing(tls().stream, &cap));
    if (cap != cudaStreamCaptureStatusNone && tls().blocking)
        return fail(CATENA_E_BAD_ARG, "a captured call cannot wait for the stream: catena_b200_set_blocking(0) first");
    uint32_t*& word = g_err[tls().device];
    if (!word) {
        if (cap != cudaStreamCaptureStatusNone)
            return fail(CATENA_E_UNSUPPORTED, "the first call of a thread on a device allocates its error word: make it before the capture");
        CATENA_CUDA(cudaMalloc(&word, sizeof(uint32_t)));
        CATENA_CUDA(cudaMemset(word, 0, sizeof(uint32_t)));
        CATENA_CUDA(cudaStreamSynchronize(0));
    }
    *err = word;
    return CATENA_OK;
}

catena_status_t check_errors() {
    if (tls().device < 0 || !g_err[tls().device]) return CATENA_OK;
    CATENA_TRY(ensure_device());
    uint32_t* word = g_err[tls().device];
    uint32_t h = 0;
    CATENA_CUDA(cudaMemcpyAsync(&h, word, sizeof(h), cudaMemcpyDeviceToHost, tls().stream));
    CATENA_CUDA(cudaStreamSynchronize(tls().stream));
    if (!h) return CATENA_OK;
    CATENA_CUDA(cudaMemsetAsync(word, 0, sizeof(uint32_t), tls().stream));
    if (h & kErrTable) return fail(CATENA_E_ASSERT, "paged cache: a page id outside the pool");
    if (h & kErrLength) return fail(CATENA_E_ASSERT, "paged cache: a length outside what the page table can hold");
    if (h & kErrPosition) return fail(CATENA_E_ASSERT, "paged cache: a position outside the table of angles");
    return fail(CATENA_E_ASSERT, "beam search: a parent outside its group of beams");
}

catena_status_t end() {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail_cuda(e, "paged cache");
    if (!tls().blocking) return CATENA_OK;
    CATENA_CUDA(cudaStreamSynchronize(tls().stream));
    return check_errors();
}

catena_status_t check_cache(const catena_paged_cache_t* c, const char* what, View* view) {
    if (!c || !c->k_pages || !c->v_pages || !c->table || !c->lengths) return fail(CATENA_E_BAD_ARG, what);
    if (!aligned16(c->k_pages) || !aligned16(c->v_pages) || !aligned4(c->table) || !aligned4(c->lengths))
        return fail(CATENA_E_BAD_ARG, "paged cache: pages must be 16-byte aligned, table and lengths 4-byte");
    if (c->head_dim != 64 && c->head_dim != 128) return fail(CATENA_E_UNSUPPORTED, "paged cache: head_dim must be 64 or 128");
    if (!c->n_pages || !c->page_size || !c->max_pages || !c->n_kv_heads) return fail(CATENA_E_BAD_ARG, "paged cache: empty dimension");
    // rows of a pool and of a sequence are 32-bit in the kernels (byte offsets are 64-bit)
    const uint64_t lim = 0xFFFFFFFFull, lim31 = 0x7FFFFFFFull;
    if (c->n_pages > lim31 || c->page_size > lim31 || c->max_pages > lim31 || c->n_kv_heads > 0xFFFFull || c->n_seqs > 0xFFFFFull ||
        c->max_pages * c->page_size > lim31 || c->n_kv_heads * c->page_size >= lim || c->n_pages * (c->n_kv_heads * c->page_size) >= lim)
        return fail(CATENA_E_TOO_LARGE, "paged cache: more pages, rows or sequences than the kernels index");
    view->k = (__nv_bfloat16*)c->k_pages;
    view->v = (__nv_bfloat16*)c->v_pages;
    view->table = c->table;
    view->lengths = c->lengths;
    view->n_pages = (uint32_t)c->n_pages;
    view->page_size = (uint32_t)c->page_size;
    view->n_seqs = (uint32_t)c->n_seqs;
    view->max_pages = (uint32_t)c->max_pages;
    view->hkv = (uint32_t)c->n_kv_heads;
    view->err = nullptr;
    return CATENA_OK;
}

// ---------------------------------------------------------------- angles
struct InvFreq { float f[64]; };
__global__ void rope_angles_kernel(InvFreq inv, float2* __restrict__ out, uint32_t pos0, uint64_t n, uint32_t half) {
    pdl_trigger();
    pdl_wait();
    const uint64_t idx = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (idx >= n * half) return;
    // the functions and roundings of the Llama block's rotation (llama.cu): the same bits
    const float angle = cmath::mul(cmath::u32_to_f32(pos0 + (uint32_t)(idx / half)), inv.f[idx % half]);
    out[idx] = make_float2(cmath::sin_full(cmath::add(angle, cmath::from_bits(0x3FC90FDBu))), cmath::sin_full(angle));
}

// ---------------------------------------------------------------- rotation + append
// Token t of sequence b (token_start[b] <= t < token_start[b + 1]) is the (t - token_start[b])-th of the sequence's new rows, which
// are its last: row = length - new + nth, position = positions[b] + nth.  Rotation (rotate half, products and sum rounded
// separately as in llama.cu): (x1 c - x2 s, x2 c + x1 s).
// A CTA has a token: a thread 8 pairs of every 16th (d = 128) or 32nd head, so the angles and the row's place are found once for all
// of them, and three heads' loads are on their way at once.  Few tokens: the heads over several CTAs.  The sequence of a token is found
// by a whole warp at once, 32 boundaries per step.
// Bound: HBM, every element is read and written once (9219 tokens of 16 + 32 heads of 128: 38.7 us,
// 5.3 TB/s; with a thread per head and pair group, which looks everything up for itself, 45 us).
__device__ __forceinline__ uint32_t find_seq(const int32_t* __restrict__ start, uint32_t n, int64_t t) {
    // the largest b with start[b] <= t, for start[0] <= t; whole warp
    uint32_t lo = 0, width = n + 1;                    // boundaries lo .. lo + width - 1 can still be it
    const uint32_t lane = threadIdx.x & 31;
    while (width > 1) {
        const uint32_t step = (width + 31) / 32, at = lane * step;
        const bool le = at < width && (int64_t)start[lo + at] <= t;
        const uint32_t votes = __ballot_sync(0xFFFFFFFFu, le);
        // lane 0's boundary is <= t whenever the first one is; the last lane that says so holds the block
        const uint32_t last = votes ? 31 - __clz(votes) : 0;
        lo += last * step;
        width = min(step, width - last * step);
    }
    return lo;
}

template <int D>
__global__ void __launch_bounds__(128) rope_append_paged_kernel(View c, const __nv_bfloat16* __restrict__ qkv, uint64_t pitch,
                                                                const int32_t* __restrict__ token_start, const int32_t* __restrict__ positions,
                                                                const float4* __restrict__ angles, uint32_t n_angles, uint32_t hq,
                                                                __nv_bfloat16* __restrict__ q_out) {
    constexpr uint32_t kPieces = D / 16;               // 8 pairs each
    constexpr uint32_t kHeads = 128 / kPieces;
    constexpr int kAtOnce = 3;
    pdl_trigger();
    pdl_wait();
    const uint32_t t = blockIdx.x;
    uint32_t b = t, nth = 0, fresh = 1;
    if (token_start) {
        if (token_start[0] > (int64_t)t) return;
        b = find_seq(token_start, c.n_seqs, t);
        if (b >= c.n_seqs) return;                     // behind the last sequence: left alone
        nth = t - (uint32_t)token_start[b];
        fresh = (uint32_t)(token_start[b + 1] - token_start[b]);
    }
    const uint32_t n = c.length(b);
    if (fresh > n) {
        atomicOr(c.err, kErrLength);
        return;
    }
    const uint32_t r = n - fresh + nth, i0 = threadIdx.x % kPieces * 8;
    const int64_t pos = (positions ? (int64_t)positions[b] : (int64_t)(n - fresh)) + nth;
    const uint32_t row0 = c.row(b, 0, r);              // that of kv head 0; a head's are page_size rows on
    if (pos < 0 || pos >= (int64_t)n_angles) {
        atomicOr(c.err, kErrPosition);
        return;
    }
    float4 cs[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) cs[e] = angles[((size_t)pos * (D / 2) + i0) / 2 + e];
    const uint32_t heads = hq + 2 * c.hkv, step = kHeads * gridDim.y;
    for (uint32_t h0 = blockIdx.y * kHeads + threadIdx.x / kPieces; h0 < heads; h0 += kAtOnce * step) {
        uint4 lo[kAtOnce], hi[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const uint32_t head = h0 + u * step;
            if (head >= heads) break;
            const __nv_bfloat16* src = qkv + (size_t)t * pitch + head * D + i0;
            lo[u] = *reinterpret_cast<const uint4*>(src);
            hi[u] = *reinterpret_cast<const uint4*>(src + D / 2);
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const uint32_t head = h0 + u * step;
            if (head >= heads) break;
            if (head >= hq && row0 == kNoRow) continue;
            __nv_bfloat16* dst;
            if (head < hq) dst = q_out + ((size_t)t * hq + head) * D;
            else if (head < hq + c.hkv) dst = c.k + (size_t)(row0 + (head - hq) * c.page_size) * D;
            else dst = c.v + (size_t)(row0 + (head - hq - c.hkv) * c.page_size) * D;
            if (head < hq + c.hkv) {
                const uint32_t lw[4] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w}, hw[4] = {hi[u].x, hi[u].y, hi[u].z, hi[u].w};
                uint32_t r1[4], r2[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 a = cs[e];
                    const float x10 = __uint_as_float(lw[e] << 16), x11 = __uint_as_float(lw[e] & 0xFFFF0000u);
                    const float x20 = __uint_as_float(hw[e] << 16), x21 = __uint_as_float(hw[e] & 0xFFFF0000u);
                    const __nv_bfloat162 o1 = __floats2bfloat162_rn(cmath::sub(cmath::mul(x10, a.x), cmath::mul(x20, a.y)),
                                                                    cmath::sub(cmath::mul(x11, a.z), cmath::mul(x21, a.w)));
                    const __nv_bfloat162 o2 = __floats2bfloat162_rn(cmath::add(cmath::mul(x20, a.x), cmath::mul(x10, a.y)),
                                                                    cmath::add(cmath::mul(x21, a.z), cmath::mul(x11, a.w)));
                    r1[e] = *reinterpret_cast<const uint32_t*>(&o1);
                    r2[e] = *reinterpret_cast<const uint32_t*>(&o2);
                }
                lo[u] = make_uint4(r1[0], r1[1], r1[2], r1[3]);
                hi[u] = make_uint4(r2[0], r2[1], r2[2], r2[3]);
            }
            *reinterpret_cast<uint4*>(dst + i0) = lo[u];
            *reinterpret_cast<uint4*>(dst + D / 2 + i0) = hi[u];
        }
    }
}

// ---------------------------------------------------------------- eviction: which rows stay
// A cluster of CTAs per (sequence, kv head), each with a stretch of the rows, whose weights it keeps in shared memory.  Rows
// 0 .. n - recent - 1 compete by weight for budget - recent places; the limit is found by a radix select over the weights'
// order-preserving bits, 2048 bins between the least and the greatest of a sample, which every CTA takes alike (weights spread over
// few octaves: bins cut from the top bits would hold thousands each), every CTA adding up all CTAs' bins for itself.  One pass usually
// leaves a bin of at most 256 rows, which are ranked by comparing them with each other; ties at the limit go to the lowest rows.
// A NaN counts as -inf and -0 as +0, so the order is total.  What stays is then written in order: every warp counts in its part
// of the stretch and writes once it knows how many stay before it.
constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kBinsPer = kBins / kSelThreads;
constexpr uint32_t kRanked = 256;
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kSelRoom = 49152;                   // weights a CTA can hold (192 KB)
constexpr uint32_t kSelAlone = 116 * 1024;             // more than half of an SM's shared memory

__device__ __forceinline__ uint32_t order_bits(float w) {
    if (w != w) return 0x007FFFFFu;                    // -inf
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// exclusive prefix sum over the CTA of one value per thread
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, off);
        if (lane >= (uint32_t)off) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    const uint32_t before = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? warp_sums[lane] : 0u);
    __syncthreads();
    return before + x - v;
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(View c, const float* __restrict__ weights, uint32_t budget, uint32_t recent,
                                                                   int32_t* __restrict__ lengths_out, float* __restrict__ weights_out,
                                                                   uint32_t cap_out, int32_t* __restrict__ kept, int32_t* __restrict__ rows_ws,
                                                                   uint32_t room) {
    extern __shared__ uint32_t sel_smem[];             // [room] the stretch's weights, [room / 32] who stays
    __shared__ __align__(8) uint32_t hist[kBins];
    __shared__ uint64_t cand[kRanked], all[kRanked];
    __shared__ uint32_t warp_sums[32], s_lo, s_hi, s_digit, s_left, s_count, s_n, s_equal, s_stay;
    __shared__ uint64_t s_limit;
    pdl_wait();
    pdl_trigger();                                     // only now: the copies below begin before this kernel is done
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t unit = blockIdx.x / ctas, b = unit / c.hkv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t n = c.length(b);
    const uint32_t stay = min(n, budget);
    const float* w = weights + (size_t)unit * c.cap();
    float* w_out = weights_out + (size_t)unit * cap_out;
    int32_t* rows = rows_ws + (size_t)unit * budget;
    int32_t* kept_row = kept ? kept + (size_t)unit * budget : nullptr;
    if (unit % c.hkv == 0 && rank == 0 && tid == 0) lengths_out[b] = (int32_t)stay;
    for (uint32_t i = stay + rank * kSelThreads + tid; i < cap_out; i += ctas * kSelThreads) w_out[i] = 0.0f;
    if (n <= budget) {
        for (uint32_t i = rank * kSelThreads + tid; i < n; i += ctas * kSelThreads) {
            rows[i] = (int32_t)i;
            if (kept_row) kept_row[i] = (int32_t)i;
            w_out[i] = w[i];
        }
        return;
    }
    const uint32_t m = n - recent, want = budget - recent;         // want < m
    const uint32_t part = (n + ctas * kSelWarps * 32 - 1) / (ctas * kSelWarps * 32) * 32;      // rows of a warp
    const uint32_t r0 = min(n, rank * kSelWarps * part), r1 = min(n, r0 + kSelWarps * part), c1 = min(r1, max(m, r0));
    float* own = reinterpret_cast<float*>(sel_smem);
    uint32_t* words = sel_smem + room;
    const bool held = kSelWarps * part <= room;                    // else the weights are read again in every pass
    auto weight = [&](uint32_t i) { return held ? own[i - r0] : w[i]; };
    auto key = [&](uint32_t i) { return order_bits(weight(i)); };
    // a value of every CTA of the cluster, lane q that of CTA q (0 behind the last)
    auto of_all = [&](uint32_t* mine) { return lane < ctas ? *cluster.map_shared_rank(mine, lane) : 0u; };

    if (tid == 0) { s_lo = 0xFFFFFFFFu; s_hi = 0; s_n = s_equal = 0; }
    for (uint32_t i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
    const uint32_t sample = order_bits(w[(uint32_t)((uint64_t)tid * m / kSelThreads)]);
    if (held) {
#pragma unroll 4
        for (uint32_t i = r0 + tid; i < r1; i += kSelThreads) own[i - r0] = w[i];
    }
    __syncthreads();
    {
        const uint32_t lo = __reduce_min_sync(0xFFFFFFFFu, sample), hi = __reduce_max_sync(0xFFFFFFFFu, sample);
        if (lane == 0) {
            atomicMin(&s_lo, lo);
            atomicMax(&s_hi, hi);
        }
    }
    __syncthreads();
    uint64_t limit = ~0ull;                                        // a row stays when (bits, lowest row first) reaches it
    if (want) {
        // Keys from lo on in bins of 2^shift, the last bin open above; in the first pass those below lo are in the first bin, and
        // afterwards all that can hold the limit, the left-th greatest of them, are lo .. lo + span.
        uint32_t lo = s_lo, span = s_hi - lo, left = want, count;
        int shift = max(0, 21 - __clz(span));                      // span >> shift < 2048 (clz(0) is 32)
        bool first = true;
        while (true) {
#pragma unroll 4
            for (uint32_t i = r0 + tid; i < c1; i += kSelThreads) {
                const uint32_t u = key(i);
                if (first) atomicAdd(&hist[u < lo ? 0u : min((u - lo) >> shift, kBins - 1)], 1u);
                else if (u - lo <= span) atomicAdd(&hist[(u - lo) >> shift], 1u);
            }
            cluster.sync();
            // the bin of the left-th greatest: sums from the top
            uint32_t h[kBinsPer], sum = 0;
            const uint32_t top = kBins - kBinsPer * (tid + 1);
#pragma unroll
            for (uint32_t e = 0; e < kBinsPer; ++e) h[e] = 0;
            for (uint32_t q = 0; q < ctas; ++q) {
                const uint2* bins = cluster.map_shared_rank(reinterpret_cast<uint2*>(hist + top), q);
#pragma unroll
                for (uint32_t e = 0; e < kBinsPer; e += 2) {
                    const uint2 v = bins[kBinsPer / 2 - 1 - e / 2];
                    h[e] += v.y;
                    h[e + 1] += v.x;
                }
            }
#pragma unroll
            for (uint32_t e = 0; e < kBinsPer; ++e) sum += h[e];
            uint32_t above = block_scan(sum, warp_sums);
#pragma unroll
            for (uint32_t e = 0; e < kBinsPer; ++e) {
                if (above < left && left <= above + h[e]) { s_digit = top + kBinsPer - 1 - e; s_left = left - above; s_count = h[e]; }
                above += h[e];
            }
            __syncthreads();
            const uint32_t base = lo, end = lo + span;
            lo += s_digit << shift;
            span = (1u << shift) - 1;
            if (first && s_digit == 0) {
                span += base;
                lo = 0;
            } else if (first && s_digit == kBins - 1) {
                span = ~0u - lo;
            } else if (!first) {
                span = min(span, end - lo);                        // the last bin may reach past what is left
            }
            first = false;
            left = s_left;
            count = s_count;
            if (count <= kRanked || span == 0) break;
            shift = max(0, 21 - __clz(span));
            cluster.sync();                                        // everyone has read the bins
            for (uint32_t i = tid; i < kBins; i += kSelThreads) hist[i] = 0;
            __syncthreads();
        }
        if (count <= kRanked) {
#pragma unroll 4
            for (uint32_t i = r0 + tid; i < c1; i += kSelThreads) {
                const uint32_t u = key(i);
                if (u - lo <= span) cand[atomicAdd(&s_n, 1u)] = (uint64_t)u << 32 | (uint32_t)~i;
            }
            cluster.sync();
            const uint32_t sizes = of_all(&s_n);
            uint32_t at = 0;
            for (uint32_t q = 0; q < ctas; ++q) {
                const uint32_t size = __shfl_sync(0xFFFFFFFFu, sizes, q);
                if (tid < size) all[at + tid] = cluster.map_shared_rank(cand, q)[tid];
                at += size;
            }
            __syncthreads();
            if (tid < count) {
                const uint64_t mine = all[tid];
                uint32_t before = 0;
                for (uint32_t j = 0; j < count; ++j) before += all[j] > mine;
                if (before == left - 1) s_limit = mine;
            }
        } else {
            // more than 256 rows of one weight: the left-th lowest of them
            uint32_t mine = 0;
            const uint32_t i0 = r0 + warp * part;
            for (uint32_t i = i0; i < i0 + part; i += 32) mine += __popc(__ballot_sync(0xFFFFFFFFu, i + lane < c1 && key(i + lane) == lo));
            if (lane == 0) {
                warp_sums[warp] = mine;
                atomicAdd(&s_equal, mine);
            }
            cluster.sync();
            const uint32_t equal = of_all(&s_equal);
            uint32_t before = __reduce_add_sync(0xFFFFFFFFu, (lane < rank ? equal : 0u) + (lane < warp ? warp_sums[lane] : 0u));
            if (before < left && left <= before + mine)
                for (uint32_t i = i0; i < i0 + part; i += 32) {
                    const bool eq = i + lane < c1 && key(i + lane) == lo;
                    const uint32_t votes = __ballot_sync(0xFFFFFFFFu, eq);
                    if (eq && before + __popc(votes & ((1u << lane) - 1)) == left - 1)
                        for (uint32_t q = 0; q < ctas; ++q) *cluster.map_shared_rank(&s_limit, q) = (uint64_t)lo << 32 | (uint32_t)~(i + lane);
                    before += __popc(votes);
                }
            cluster.sync();
        }
        __syncthreads();
        limit = s_limit;
    }
    __syncthreads();                                               // warp_sums of the tie search has been read
    auto stays = [&](uint32_t i) { return i < r1 && (i >= m || ((uint64_t)key(i) << 32 | (uint32_t)~i) >= limit); };
    const uint32_t i0 = r0 + warp * part;
    uint32_t mine = 0;
#pragma unroll 4
    for (uint32_t i = i0; i < i0 + part; i += 32) {
        const uint32_t votes = __ballot_sync(0xFFFFFFFFu, stays(i + lane));
        if (held && lane == 0) words[(i - r0) / 32] = votes;
        mine += __popc(votes);
    }
    if (lane == 0) warp_sums[warp] = mine;
    __syncthreads();
    uint32_t at = __reduce_add_sync(0xFFFFFFFFu, lane < warp ? warp_sums[lane] : 0u);
    if (warp == kSelWarps - 1 && lane == 0) s_stay = at + mine;
    cluster.sync();
    const uint32_t staying = of_all(&s_stay);
    at += __reduce_add_sync(0xFFFFFFFFu, lane < rank ? staying : 0u);
    cluster.sync();                                                // no CTA leaves while another reads from it
#pragma unroll 4
    for (uint32_t i = i0; i < i0 + part; i += 32) {
        const uint32_t votes = held ? words[(i - r0) / 32] : __ballot_sync(0xFFFFFFFFu, stays(i + lane));
        if (votes >> lane & 1) {
            const uint32_t to = at + __popc(votes & ((1u << lane) - 1));
            rows[to] = (int32_t)(i + lane);
            if (kept_row) kept_row[to] = (int32_t)(i + lane);
            w_out[to] = weight(i + lane);
        }
        at += __popc(votes);
    }
}

// ---------------------------------------------------------------- eviction: the rows that stay, into their new pages
// The recent rows stay whatever the weights are, and all rows of a sequence within its budget: CTAs that have only such rows copy
// while the selection still runs (which starts them only once everything before it is done).  Bound by the chain row number -> page
// -> data: two rows per thread on 64 warps per SM took 29.6 us with the selection (4 x 16384 rows), four on 32 warps 30.8.
constexpr int kCopySteps = 2;
template <int D>
__global__ void __launch_bounds__(256, 8) evict_copy_kernel(View c, const int32_t* rows_ws, uint32_t budget, uint32_t recent,
                                                         const int32_t* __restrict__ table_out, uint32_t max_pages_out) {
    constexpr uint32_t kLanes = D / 8;                 // 16-byte pieces of a row
    constexpr uint32_t kRows = 256 / kLanes;           // rows of a CTA's step
    constexpr int kSteps = kCopySteps;
    pdl_trigger();
    const uint32_t unit = blockIdx.y, b = unit / c.hkv, h = unit % c.hkv;
    const uint32_t n = c.length(b), stay = min(n, budget), chosen = n <= budget ? 0 : stay - recent;     // rows the selection has to name
    const uint32_t piece = threadIdx.x % kLanes, first = blockIdx.x * (kSteps * kRows), i0 = first + threadIdx.x / kLanes;
    const bool early = first >= chosen;
    if (!early || first >= stay) pdl_wait();
    if (first >= stay) return;
    uint32_t src[kSteps], dst[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
        const uint32_t i = i0 + u * kRows;
        src[u] = i >= stay ? kNoRow : i >= chosen ? i + (n - stay) : (uint32_t)rows_ws[(size_t)unit * budget + i];
    }
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
        dst[u] = src[u] == kNoRow ? kNoRow : c.row(table_out, max_pages_out, b, h, i0 + u * kRows);
        src[u] = dst[u] == kNoRow ? kNoRow : c.row(b, h, src[u]);
    }
    uint4 k[kSteps], v[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u)
        if (src[u] != kNoRow) {
            k[u] = reinterpret_cast<const uint4*>(c.k)[(size_t)src[u] * kLanes + piece];
            v[u] = reinterpret_cast<const uint4*>(c.v)[(size_t)src[u] * kLanes + piece];
        }
#pragma unroll
    for (int u = 0; u < kSteps; ++u)
        if (src[u] != kNoRow) {
            reinterpret_cast<uint4*>(c.k)[(size_t)dst[u] * kLanes + piece] = k[u];
            reinterpret_cast<uint4*>(c.v)[(size_t)dst[u] * kLanes + piece] = v[u];
        }
    if (early) pdl_wait();                             // this kernel is not done before the selection is
}

// ---------------------------------------------------------------- beams take over their parents' pages
// Full pages are shared: the child's table names the parent's.  The page that is still being filled is copied into the child's
// fresh page, because parent and child write different rows behind it.  grid.y < hkv: keys, values and weights of a head; the
// last grid.y: table and length.
template <int D>
__global__ void __launch_bounds__(128) beam_reorder_kernel(View c, const int32_t* __restrict__ parents, uint32_t beams,
                                                           const int32_t* __restrict__ fresh, int32_t* __restrict__ table_out,
                                                           int32_t* __restrict__ lengths_out, const float* __restrict__ weights,
                                                           float* __restrict__ weights_out) {
    pdl_trigger();
    pdl_wait();
    const uint32_t s = blockIdx.x, tid = threadIdx.x;
    const uint32_t parent = (uint32_t)parents[s];
    if (parent >= beams) {
        if (tid == 0) atomicOr(c.err, kErrParent);
        return;
    }
    const uint32_t p = s / beams * beams + parent;
    const uint32_t n = c.length(p), full = n / c.page_size, rest = n - full * c.page_size;
    if (blockIdx.y == c.hkv) {
        for (uint32_t j = tid; j < full; j += 128) table_out[(size_t)s * c.max_pages + j] = c.table[(size_t)p * c.max_pages + j];
        if (tid == 0) {
            if (rest) table_out[(size_t)s * c.max_pages + full] = fresh[s];
            lengths_out[s] = (int32_t)n;
        }
        return;
    }
    const uint32_t h = blockIdx.y;
    if (rest) {
        const uint32_t from = (uint32_t)c.table[(size_t)p * c.max_pages + full], to = (uint32_t)fresh[s];
        if (from >= c.n_pages || to >= c.n_pages) {
            if (tid == 0) atomicOr(c.err, kErrTable);
        } else {
            const size_t src = ((size_t)from * c.hkv + h) * c.page_size * (D / 8), dst = ((size_t)to * c.hkv + h) * c.page_size * (D / 8);
#pragma unroll 4
            for (uint32_t i = tid; i < rest * (D / 8); i += 128) {
                const uint4 k = reinterpret_cast<const uint4*>(c.k)[src + i], v = reinterpret_cast<const uint4*>(c.v)[src + i];
                reinterpret_cast<uint4*>(c.k)[dst + i] = k;
                reinterpret_cast<uint4*>(c.v)[dst + i] = v;
            }
        }
    }
    if (weights) {
        const float* w = weights + ((size_t)p * c.hkv + h) * c.cap();
        float* o = weights_out + ((size_t)s * c.hkv + h) * c.cap();
#pragma unroll 8
        for (uint32_t i = tid; i < c.cap(); i += 128) o[i] = i < n ? w[i] : 0.0f;
    }
}

}  // namespace paged

using namespace paged;

extern "C" {

catena_status_t catena_b200_rope_angles_f32_into(float base, uint64_t pos0, uint64_t count, uint64_t head_dim, void* angles) {
    if (head_dim != 64 && head_dim != 128) return fail(CATENA_E_UNSUPPORTED, "rope_angles: head_dim must be 64 or 128");
    if (!(base > 0.0f) || base - base != 0.0f) return fail(CATENA_E_BAD_ARG, "rope_angles: base must be positive and finite");
    if (count > 0x7FFFFFFFull || pos0 > 0x7FFFFFFFull) return fail(CATENA_E_TOO_LARGE, "rope_angles: positions are below 2^31");
    if (!count) return CATENA_OK;
    if (!angles || !aligned16(angles)) return fail(CATENA_E_BAD_ARG, "rope_angles: null or misaligned output");
    uint32_t* err;
    CATENA_TRY(begin(&err));
    InvFreq inv;
    const uint32_t half = (uint32_t)head_dim / 2;
    for (uint32_t i = 0; i < 64; ++i) inv.f[i] = i < half ? cmath::powf_approx(base, -cmath::div(cmath::u32_to_f32(2 * i), cmath::u32_to_f32((uint32_t)head_dim))) : 0.0f;
    CATENA_TRY(launch("rope_angles_kernel", rope_angles_kernel, dim3((unsigned)ceil_div_u64(count * half, 256)), dim3(256), 0, inv,
                      (float2*)angles, (uint32_t)pos0, count, half));
    return end();
}

catena_status_t catena_b200_rope_append_paged_bf16_into(const catena_paged_cache_t* cache, const void* qkv, uint64_t qkv_pitch,
                                                        const int32_t* token_start, uint64_t tokens, const int32_t* positions,
                                                        const void* angles, uint64_t n_angles, uint64_t n_heads, void* q_out) {
    View c;
    CATENA_TRY(check_cache(cache, "rope_append_paged: null cache", &c));
    if (!tokens || !c.n_seqs) return CATENA_OK;
    if (!qkv || !angles || (n_heads && !q_out)) return fail(CATENA_E_BAD_ARG, "rope_append_paged: null argument");
    if (!aligned16(qkv) || !aligned16(angles) || !aligned16(q_out) || qkv_pitch % 8)
        return fail(CATENA_E_BAD_ARG, "rope_append_paged: qkv, its rows, angles and q_out must be 16-byte aligned");
    if (!aligned4(token_start) || !aligned4(positions)) return fail(CATENA_E_BAD_ARG, "rope_append_paged: misaligned token_start or positions");
    if (n_heads > 0xFFFFull || tokens > 0x7FFFFFFFull || n_angles > 0x7FFFFFFFull) return fail(CATENA_E_TOO_LARGE, "rope_append_paged: more tokens or heads than the kernel indexes");
    if (qkv_pitch < (n_heads + 2 * c.hkv) * cache->head_dim) return fail(CATENA_E_BAD_ARG, "rope_append_paged: rows of qkv overlap");
    if (!token_start && tokens != c.n_seqs) return fail(CATENA_E_BAD_ARG, "rope_append_paged: without token_start there is one token per sequence");
    CATENA_TRY(begin(&c.err));
    const bool wide = cache->head_dim == 128;
    // CTAs of all heads of a token, or of a part of them until there are some for every SM
    const uint64_t sms = tls().sm_count > 0 ? tls().sm_count : 148, steps = ceil_div_u64((n_heads + 2 * c.hkv) * (cache->head_dim / 16), 128);
    const uint64_t parts = ceil_div_u64(sms * 4, tokens);
    const dim3 grid((unsigned)tokens, (unsigned)(parts < steps ? parts : steps));
    CATENA_TRY(launch("rope_append_paged_kernel", wide ? rope_append_paged_kernel<128> : rope_append_paged_kernel<64>, grid, dim3(128), 0, c,
                      (const __nv_bfloat16*)qkv, qkv_pitch, token_start, positions, (const float4*)angles, (uint32_t)n_angles, (uint32_t)n_heads,
                      (__nv_bfloat16*)q_out));
    return end();
}

uint64_t catena_b200_kv_evict_paged_workspace_bytes(const catena_paged_cache_t* cache, uint64_t budget) {
    View c;
    if (check_cache(cache, "kv_evict_paged: null cache", &c) != CATENA_OK || budget > 0x7FFFFFFFull || (uint64_t)c.n_seqs * c.hkv > 65535) return 0;
    return (uint64_t)c.n_seqs * c.hkv * budget * sizeof(int32_t);
}

catena_status_t catena_b200_kv_evict_paged_bf16_into(const catena_paged_cache_t* cache, const float* weights, uint64_t budget, uint64_t recent,
                                                     const int32_t* table_out, uint64_t max_pages_out, int32_t* lengths_out,
                                                     float* weights_out, int32_t* kept, void* workspace, uint64_t workspace_bytes) {
    View c;
    CATENA_TRY(check_cache(cache, "kv_evict_paged: null cache", &c));
    if (!c.n_seqs) return CATENA_OK;
    if (!weights || !table_out || !lengths_out || !weights_out || !workspace) return fail(CATENA_E_BAD_ARG, "kv_evict_paged: null argument");
    if (!aligned4(weights) || !aligned4(table_out) || !aligned4(lengths_out) || !aligned4(weights_out) || !aligned4(kept) || !aligned16(workspace))
        return fail(CATENA_E_BAD_ARG, "kv_evict_paged: misaligned argument");
    if (budget == 0 || recent > budget) return fail(CATENA_E_BAD_ARG, "kv_evict_paged: budget must be positive and hold the recent rows");
    if (max_pages_out == 0 || max_pages_out > 0x7FFFFFFFull || budget > 0x7FFFFFFFull || max_pages_out * c.page_size > 0x7FFFFFFFull)
        return fail(CATENA_E_TOO_LARGE, "kv_evict_paged: more rows than the kernels index");
    if (budget > max_pages_out * c.page_size) return fail(CATENA_E_BAD_ARG, "kv_evict_paged: table_out holds fewer rows than the budget");
    if (table_out == cache->table || lengths_out == cache->lengths || weights_out == weights)
        return fail(CATENA_E_BAD_ARG, "kv_evict_paged: rows move into other pages, lengths and weights into other buffers");
    const uint64_t units = (uint64_t)c.n_seqs * c.hkv;
    if (units > 65535) return fail(CATENA_E_TOO_LARGE, "kv_evict_paged: more than 65535 (sequence, kv head) pairs");
    if (workspace_bytes < catena_b200_kv_evict_paged_workspace_bytes(cache, budget)) return fail(CATENA_E_BAD_ARG, "kv_evict_paged: workspace too small");
    CATENA_TRY(begin(&c.err));
    // A CTA per 2048 rows that a sequence may have, up to eight and as long as every CTA has an SM of its own.  (Clusters of small
    // CTAs are packed onto few SMs: 256 CTAs took 21 us where 128 with an SM each take 16.)  The shared memory that keeps a second CTA
    // off the SM is asked for whether it is filled or not.
    const uint64_t sms = tls().sm_count > 0 ? tls().sm_count : 148;
    uint32_t ctas = 1;
    while (ctas < kMaxCluster && c.cap() > 2048u * ctas && units * ctas * 2 <= sms) ctas *= 2;
    const uint64_t stretch = ceil_div_u64(c.cap(), ctas * kSelWarps * 32) * (kSelWarps * 32);
    const uint32_t room = stretch > kSelRoom ? 0u : (uint32_t)stretch;
    size_t smem = (size_t)room * 4 + room / 8;
    if (ctas > 1 && smem < kSelAlone) smem = kSelAlone;
    static thread_local uint32_t told = 0;
    CATENA_TRY(allow_smem(evict_select_kernel, kSelRoom * 4 + kSelRoom / 8, &told));
    How how;
    how.cluster = ctas;
    CATENA_TRY(launch_as(how, "evict_select_kernel", evict_select_kernel, dim3((unsigned)units * ctas), dim3(kSelThreads), smem, c, weights,
                              (uint32_t)budget, (uint32_t)recent, lengths_out, weights_out, (uint32_t)(max_pages_out * c.page_size), kept,
                              (int32_t*)workspace, room));
    const uint64_t rows_per_cta = kCopySteps * (256 / (cache->head_dim / 8));
    const dim3 grid((unsigned)ceil_div_u64(budget, rows_per_cta), (unsigned)units);
    CATENA_TRY(launch("evict_copy_kernel", cache->head_dim == 128 ? evict_copy_kernel<128> : evict_copy_kernel<64>, grid, dim3(256), 0, c,
                      (const int32_t*)workspace, (uint32_t)budget, (uint32_t)recent, table_out, (uint32_t)max_pages_out));
    return end();
}

catena_status_t catena_b200_beam_reorder_paged_bf16_into(const catena_paged_cache_t* cache, const int32_t* parents, uint64_t beams,
                                                         const int32_t* fresh_pages, int32_t* table_out, int32_t* lengths_out,
                                                         const float* weights, float* weights_out) {
    View c;
    CATENA_TRY(check_cache(cache, "beam_reorder_paged: null cache", &c));
    if (!c.n_seqs) return CATENA_OK;
    if (!parents || !fresh_pages || !table_out || !lengths_out || (!weights) != (!weights_out))
        return fail(CATENA_E_BAD_ARG, "beam_reorder_paged: null argument");
    if (!aligned4(parents) || !aligned4(fresh_pages) || !aligned4(table_out) || !aligned4(lengths_out) || !aligned4(weights) || !aligned4(weights_out))
        return fail(CATENA_E_BAD_ARG, "beam_reorder_paged: misaligned argument");
    if (beams == 0 || beams > c.n_seqs || c.n_seqs % beams) return fail(CATENA_E_BAD_ARG, "beam_reorder_paged: sequences must be whole groups of beams");
    if (table_out == cache->table || lengths_out == cache->lengths || (weights && weights_out == weights))
        return fail(CATENA_E_BAD_ARG, "beam_reorder_paged: outputs must be other buffers than the inputs");
    if (c.hkv >= 65535) return fail(CATENA_E_TOO_LARGE, "beam_reorder_paged: too many heads");
    CATENA_TRY(begin(&c.err));
    CATENA_TRY(launch("beam_reorder_kernel", cache->head_dim == 128 ? beam_reorder_kernel<128> : beam_reorder_kernel<64>, dim3(c.n_seqs, c.hkv + 1),
                      dim3(128), 0, c, parents, (uint32_t)beams, fresh_pages, table_out, lengths_out, weights, weights_out));
    return end();
}

}  // extern "C"

}  // namespace catena
