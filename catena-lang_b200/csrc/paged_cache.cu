// A key/value cache in pages: rotation and append of ragged tokens, eviction by accumulated attention weight, and the hand-over
// of pages between the beams of a beam search.  (The attention that reads the pages: attn_decode_paged.cu.)
// The reference has no cache; layouts follow this library's contiguous caches [batch, n_kv_heads, rows, head_dim].
#include <string.h>

#include "catena_math.cuh"
#include "paged.cuh"

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
// One thread per (token, head, 8 pairs).  The sequence of a token is found by a whole warp at once, 32 boundaries per step.
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
                                                                const float2* __restrict__ angles, uint32_t n_angles, uint32_t hq,
                                                                __nv_bfloat16* __restrict__ q_out) {
    constexpr uint32_t kPieces = D / 16;               // 8 pairs each
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
    const uint32_t idx = blockIdx.y * 128 + threadIdx.x, head = idx / kPieces, i0 = idx % kPieces * 8;
    const uint32_t heads = hq + 2 * c.hkv;
    if (head >= heads) return;
    const uint32_t n = c.length(b);
    if (fresh > n) {
        atomicOr(c.err, kErrLength);
        return;
    }
    uint32_t dst_row = 0;
    if (head >= hq) {
        dst_row = c.row(b, (head - hq) % c.hkv, n - fresh + nth);
        if (dst_row == kNoRow) return;
    }
    const __nv_bfloat16* src = qkv + (size_t)t * pitch + head * D;
    const uint4 lo = *reinterpret_cast<const uint4*>(src + i0), hi = *reinterpret_cast<const uint4*>(src + D / 2 + i0);
    __nv_bfloat16* dst;
    uint4 out_lo = lo, out_hi = hi;
    if (head >= hq + c.hkv) {
        dst = c.v + (size_t)dst_row * D;
    } else {
        const int64_t pos = (positions ? (int64_t)positions[b] : (int64_t)(n - fresh)) + nth;
        if (pos < 0 || pos >= (int64_t)n_angles) {
            atomicOr(c.err, kErrPosition);
            return;
        }
        const float4* cs = reinterpret_cast<const float4*>(angles + (size_t)pos * (D / 2) + i0);
        const uint32_t lw[4] = {lo.x, lo.y, lo.z, lo.w}, hw[4] = {hi.x, hi.y, hi.z, hi.w};
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
        out_lo = make_uint4(r1[0], r1[1], r1[2], r1[3]);
        out_hi = make_uint4(r2[0], r2[1], r2[2], r2[3]);
        dst = head < hq ? q_out + ((size_t)t * hq + head) * D : c.k + (size_t)dst_row * D;
    }
    *reinterpret_cast<uint4*>(dst + i0) = out_lo;
    *reinterpret_cast<uint4*>(dst + D / 2 + i0) = out_hi;
}

// ---------------------------------------------------------------- eviction: which rows stay
// One CTA per (sequence, kv head).  Rows 0 .. n - recent - 1 compete by weight for budget - recent places; the place's limit is
// found by a radix select over the weights' order-preserving bits (11 + 11 + 10), ties at the limit go to the lowest rows.
// A NaN counts as -inf and -0 as +0, so the order is total.
constexpr int kSelThreads = 1024;

__device__ __forceinline__ uint32_t order_bits(float w) {
    if (w != w) return 0x007FFFFFu;                    // -inf
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// exclusive prefix sum over the CTA of one value per thread; the total in *total
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* warp_sums, uint32_t* total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, off);
        if (lane >= (uint32_t)off) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        uint32_t s = warp_sums[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, s, off);
            if (lane >= (uint32_t)off) s += y;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    const uint32_t base = warp ? warp_sums[warp - 1] : 0;
    *total = warp_sums[31];
    __syncthreads();
    return base + x - v;
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(View c, const float* __restrict__ weights, uint32_t budget, uint32_t recent,
                                                                   int32_t* __restrict__ lengths_out, float* __restrict__ weights_out,
                                                                   uint32_t cap_out, int32_t* __restrict__ kept, int32_t* __restrict__ rows_ws) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t warp_sums[32];
    __shared__ uint32_t s_digit, s_left;
    pdl_trigger();
    pdl_wait();
    const uint32_t unit = blockIdx.x, b = unit / c.hkv, tid = threadIdx.x;
    const uint32_t n = c.length(b);
    const uint32_t stay = min(n, budget);
    const float* w = weights + (size_t)unit * c.cap();
    float* w_out = weights_out + (size_t)unit * cap_out;
    int32_t* rows = rows_ws + (size_t)unit * budget;
    int32_t* kept_row = kept ? kept + (size_t)unit * budget : nullptr;
    if (unit % c.hkv == 0 && tid == 0) lengths_out[b] = (int32_t)stay;
    if (n <= budget) {
        for (uint32_t i = tid; i < n; i += kSelThreads) {
            rows[i] = (int32_t)i;
            if (kept_row) kept_row[i] = (int32_t)i;
            w_out[i] = w[i];
        }
    } else {
        const uint32_t m = n - recent, want = budget - recent;     // want < m
        uint32_t limit = 0xFFFFFFFFu, left = 0;                    // rows above `limit` stay, and the first `left` that equal it
        if (want) {
            uint32_t prefix = 0, prefix_bits = 0;
            left = want;
            for (int pass = 0; pass < 3; ++pass) {
                const uint32_t bits = pass == 2 ? 10 : 11, shift = 32 - prefix_bits - bits;
                for (uint32_t i = tid; i < 2048; i += kSelThreads) hist[i] = 0;
                __syncthreads();
                for (uint32_t i = tid; i < m; i += kSelThreads) {
                    const uint32_t u = order_bits(w[i]);
                    if (prefix_bits == 0 || (u >> (32 - prefix_bits)) == prefix) atomicAdd(&hist[(u >> shift) & ((1u << bits) - 1)], 1u);
                }
                __syncthreads();
                // the digit whose bin holds the left-th largest: suffix sums, two bins per thread, largest digit first
                const uint32_t nb = 1u << bits, d1 = nb - 1 - 2 * tid, d0 = nb - 2 - 2 * tid;
                const bool mine = 2 * tid < nb;
                const uint32_t h1 = mine ? hist[d1] : 0, h0 = mine ? hist[d0] : 0;
                uint32_t total;
                const uint32_t above = block_scan(h1 + h0, warp_sums, &total);
                if (mine && above < left && left <= above + h1) { s_digit = d1; s_left = left - above; }
                if (mine && above + h1 < left && left <= above + h1 + h0) { s_digit = d0; s_left = left - above - h1; }
                __syncthreads();
                left = s_left;
                prefix = (prefix << bits) | s_digit;
                prefix_bits += bits;
                __syncthreads();
            }
            limit = prefix;
        }
        uint32_t out0 = 0, eq0 = 0;                                // rows and ties taken by earlier blocks of rows
        for (uint32_t i0 = 0; i0 < n; i0 += kSelThreads) {
            const uint32_t i = i0 + tid;
            uint32_t u = 0;
            if (want && i < m) u = order_bits(w[i]);
            const uint32_t eq = want && i < m && u == limit ? 1u : 0u;
            uint32_t n_eq, n_out;
            const uint32_t eq_before = eq0 + block_scan(eq, warp_sums, &n_eq);
            const bool keep = (i < n && i >= m) || (want && i < m && (u > limit || (eq && eq_before < left)));
            const uint32_t at = out0 + block_scan(keep ? 1u : 0u, warp_sums, &n_out);
            if (keep) {
                rows[at] = (int32_t)i;
                if (kept_row) kept_row[at] = (int32_t)i;
                w_out[at] = w[i];
            }
            eq0 += n_eq;
            out0 += n_out;
        }
    }
    for (uint32_t i = stay + tid; i < cap_out; i += kSelThreads) w_out[i] = 0.0f;
}

// ---------------------------------------------------------------- eviction: the rows that stay, into their new pages
template <int D>
__global__ void __launch_bounds__(256) evict_copy_kernel(View c, const int32_t* __restrict__ rows_ws, uint32_t budget,
                                                         const int32_t* __restrict__ table_out, uint32_t max_pages_out) {
    constexpr uint32_t kLanes = D / 8;                 // 16-byte pieces of a row
    constexpr uint32_t kRows = 256 / kLanes;           // rows of a CTA's step
    pdl_trigger();
    pdl_wait();
    const uint32_t unit = blockIdx.y, b = unit / c.hkv, h = unit % c.hkv;
    const uint32_t stay = min(c.length(b), budget);
    const uint32_t piece = threadIdx.x % kLanes;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t i = (blockIdx.x * 4 + u) * kRows + threadIdx.x / kLanes;
        if (i >= stay) return;
        const uint32_t src = c.row(b, h, (uint32_t)rows_ws[(size_t)unit * budget + i]);
        const uint32_t dst = c.row(table_out, max_pages_out, b, h, i);
        if (src == kNoRow || dst == kNoRow) continue;
        const uint4 k = reinterpret_cast<const uint4*>(c.k)[(size_t)src * kLanes + piece];
        const uint4 v = reinterpret_cast<const uint4*>(c.v)[(size_t)src * kLanes + piece];
        reinterpret_cast<uint4*>(c.k)[(size_t)dst * kLanes + piece] = k;
        reinterpret_cast<uint4*>(c.v)[(size_t)dst * kLanes + piece] = v;
    }
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
    const uint64_t work = (n_heads + 2 * c.hkv) * (cache->head_dim / 16);
    const dim3 grid((unsigned)tokens, (unsigned)ceil_div_u64(work, 128));
    CATENA_TRY(launch("rope_append_paged_kernel", wide ? rope_append_paged_kernel<128> : rope_append_paged_kernel<64>, grid, dim3(128), 0, c,
                      (const __nv_bfloat16*)qkv, qkv_pitch, token_start, positions, (const float2*)angles, (uint32_t)n_angles, (uint32_t)n_heads,
                      (__nv_bfloat16*)q_out));
    return end();
}

uint64_t catena_b200_kv_evict_paged_workspace_bytes(const catena_paged_cache_t* cache, uint64_t budget) {
    View c;
    if (check_cache(cache, "kv_evict_paged: null cache", &c) != CATENA_OK || budget > 0x7FFFFFFFull) return 0;
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
    if (workspace_bytes < catena_b200_kv_evict_paged_workspace_bytes(cache, budget)) return fail(CATENA_E_BAD_ARG, "kv_evict_paged: workspace too small");
    const uint64_t units = (uint64_t)c.n_seqs * c.hkv;
    if (units > 65535) return fail(CATENA_E_TOO_LARGE, "kv_evict_paged: more than 65535 (sequence, kv head) pairs");
    CATENA_TRY(begin(&c.err));
    CATENA_TRY(launch("evict_select_kernel", evict_select_kernel, dim3((unsigned)units), dim3(kSelThreads), 0, c, weights, (uint32_t)budget,
                      (uint32_t)recent, lengths_out, weights_out, (uint32_t)(max_pages_out * c.page_size), kept, (int32_t*)workspace));
    const uint64_t rows_per_cta = 4 * (256 / (cache->head_dim / 8));
    const dim3 grid((unsigned)ceil_div_u64(budget, rows_per_cta), (unsigned)units);
    CATENA_TRY(launch("evict_copy_kernel", cache->head_dim == 128 ? evict_copy_kernel<128> : evict_copy_kernel<64>, grid, dim3(256), 0, c,
                      (const int32_t*)workspace, (uint32_t)budget, table_out, (uint32_t)max_pages_out));
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
