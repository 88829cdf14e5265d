// Attention of one new token per sequence over a paged key/value cache, sequences of any lengths.
//   s_j = scale * (q . k_j)     o = sum_j p_j v_j / sum_j p_j     p_j = exp(s_j - max s)
// and, when asked for, weights_out[j] = weights_in[j] + sum over the group's query heads of p_j / sum p.
// The exponential is the true one (ex2.approx in base 2), not math.exp-approx: that polynomial is not multiplicative, so it would
// need the row's maximum before the first probability and with it a second pass over the scores.  Here one pass carries a running
// maximum and sum.  q, k, v are bf16; scores, maxima, sums and outputs are f32 until the one rounding of o.  A probability enters
// the second product as a bf16 pair (p rounded, and what the rounding left): with a single bf16 every p would be off by up to 2^-8
// of itself, which for a row that looks at few keys is as much as the rounding of o.
//
// Bound: HBM.  A row costs 4 d bytes and 4 d flops per query head of the group, so even 16 heads (64 flops per 4 bytes) stay far
// under the tensor rate; mma.sync on 16-row pieces feeds from a buffer that each warp fills for itself with cp.async, and no warp
// waits for another while it streams.  A warp has one tile, keys and values apart: 12 such warps per SM keep 14 MB in flight, which
// is enough; rings of two and three tiles on 8 warps per SM (19, 28 MB) only make the queues longer and the SMs' shares less equal
// (4 x 131072 rows of 8 heads: 323 us, 6.65 TB/s, against 321 and 340; 64 x 2048 on average: 91 against 96 and 98).
//
// Split: all (sequence, kv head) units' rows are cut into tiles of 64 (d = 128) or 128 (d = 64) keys, and the list of all tiles into
// equal ranges, one per CTA; the lengths need not be known on the host.  A unit that lies inside one range is finished there; of a
// unit cut by range boundaries every CTA leaves (max, sum, unnormalised output), joined in ascending order by the second launch.
// The ranges depend on the lengths and the number of SMs only: equal calls give equal bits.
// (Ranges of falling sizes, taken as CTAs become free — by the block scheduler, or by clusterlaunchcontrol within running CTAs —
// cost more in additional parts than their balance gave, with the ring of three tiles: 357 / 358 against 348 us and 102 / 106
// against 96 us for the same two cases.  Ranges that end inside a tile, for equal shares to the last 16 keys: 100 against 91 us for
// the second, whose partial tiles leave warps without rows.)
#include "catena_math.cuh"
#include "paged.cuh"

namespace catena {
namespace paged {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr uint32_t kWarpBytes = 8192;           // a warp's buffer: its keys and its values of one tile
// resident CTAs by 8-head tiles of the group: what registers allow
constexpr int ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }
constexpr float kLazy = 8.0f;                   // probabilities may reach 2^8 before the running maximum is raised

template <int D> struct Shape {
    static constexpr int kKeys = D == 128 ? 16 : 32;          // keys per warp and tile
    static constexpr int kTile = kKeys * kWarps;
    static constexpr int kPitch = D + 4;                      // floats per head of the merge buffer: conflict-free for (8 d, 4 heads)
    static constexpr uint32_t kRing = kWarps * kWarpBytes;
    static constexpr uint32_t kMerge = kWarps * 8 * kPitch * 4;
    static constexpr uint32_t kSmem = kRing + kMerge;
};

// The tiles in `ranges` ranges, of which the first `tiles` have one each when there are fewer.  start(k) = k tiles / n, in 32 bits.
struct Ranges {
    uint32_t tiles, n, each, more;
    __device__ __forceinline__ Ranges(uint32_t tiles_, uint32_t ranges) : tiles(tiles_), n(max(1u, min(tiles_, ranges))) {
        each = tiles / n;
        more = tiles - each * n;
    }
    __device__ __forceinline__ uint32_t start(uint32_t k) const { return k < n ? k * each + k * more / n : tiles; }
    // the range that holds tile t: the greatest k with k tiles / n < t + 1
    __device__ __forceinline__ uint32_t holder(uint32_t t) const { return (uint32_t)((((uint64_t)t + 1) * n + tiles - 1) / tiles - 1); }
};

// What the ranges leave behind.  Slot 2 k + 1 holds range k's part of a unit that it began and did not finish, slot 2 k its part of
// a unit begun by an earlier range.  first[k].x: the last range that holds a part of the unit in slot 2 k + 1 (0: that slot is
// empty), .y: the unit.  With weights: split[unit] = (k, last) of a unit that is cut, (1, 0) of one that is not.
struct Partials {
    uint2* first;       // [ranges]
    float2* ml;         // [ranges][2][16]   (max in base 2, sum)
    float* o;           // [ranges][2][hq / hkv][D]
    uint2* split;       // [units]
    float2* stats;      // [n_seqs][hq]      (max in base 2, sum) of units that are not cut
    float* scores;      // [n_seqs][hq][pitch] in base 2
    uint32_t pitch;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16u : 0u) : "memory");
}

// tiles of one head of all sequences; every warp for itself
template <int TILE>
__device__ __forceinline__ uint32_t count_tiles(const View& c) {
    uint32_t mine = 0;
#pragma unroll 4
    for (uint32_t b = threadIdx.x & 31; b < c.n_seqs; b += 32) mine += (c.length(b) + TILE - 1) / TILE;
    return __reduce_add_sync(0xFFFFFFFFu, mine);
}

// a position in the list of all tiles: unit (b, h), tile of the unit, rows of the sequence
template <int TILE>
struct Cursor {
    uint32_t b, h, tile, n;
    __device__ __forceinline__ uint32_t tiles() const { return (n + TILE - 1) / TILE; }
    // whole warp, and only where the range goes on: sequences without rows are passed over 32 at a time
    __device__ __forceinline__ void next(const View& c) {
        if (++tile < tiles()) return;
        tile = 0;
        if (++h < c.hkv) return;
        h = 0;
        for (++b; b < c.n_seqs; b += 32) {
            const uint32_t at = b + (threadIdx.x & 31), mine = at < c.n_seqs ? c.length(at) : 0u;
            const uint32_t some = __ballot_sync(0xFFFFFFFFu, mine != 0);
            if (some == 0) continue;
            n = __shfl_sync(0xFFFFFFFFu, mine, __ffs(some) - 1);
            b += __ffs(some) - 1;
            return;
        }
        n = 1;
    }
};

// four elements of an output: sum / L, zeros where no row has any weight
__device__ __forceinline__ void store_o(__nv_bfloat16* o, const float4& sum, float L) {
    const float r = __frcp_rn(L);
    __nv_bfloat162 lo = __floats2bfloat162_rn(__fmul_rn(sum.x, r), __fmul_rn(sum.y, r)), hi = __floats2bfloat162_rn(__fmul_rn(sum.z, r), __fmul_rn(sum.w, r));
    if (L == 0.0f) lo = hi = __floats2bfloat162_rn(0.0f, 0.0f);
    *reinterpret_cast<uint2*>(o) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

template <int D, int NT, bool WEIGHTS>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(NT)) attn_decode_paged_kernel(View c, const __nv_bfloat16* __restrict__ q, __nv_bfloat16* __restrict__ o,
                                                                                 uint32_t hq, float scale_log2, Partials part) {
    using S = Shape<D>;
    constexpr int KEYS = S::kKeys, TILE = S::kTile, SUB = KEYS / 16, CH = D / 8;     // CH: 16-byte pieces of a row
    extern __shared__ __align__(128) uint8_t smem[];
    float* merge = reinterpret_cast<float*>(smem + S::kRing);
    // the maxima are written before a segment's first barrier, while a slow warp may still read the last segment's: two of them in turn
    __shared__ float merge_ms[2][kWarps][NT * 8], merge_l[kWarps][NT * 8];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const uint32_t group = hq / c.hkv, range = blockIdx.x;
    pdl_trigger();
    pdl_wait();

    const Ranges ranges(count_tiles<TILE>(c) * c.hkv, gridDim.x);
    const uint32_t t0 = ranges.start(range), t1 = ranges.start(range + 1);
    // sequences without rows: zeros, written while the first tiles are on their way
    auto write_zeros = [&] {
        for (uint32_t b = range; b < c.n_seqs; b += gridDim.x) {
            if (c.length(b) != 0) continue;
            for (uint32_t i = tid; i < hq * D / 8; i += kThreads) reinterpret_cast<uint4*>(o + (size_t)b * hq * D)[i] = make_uint4(0, 0, 0, 0);
        }
    };
    if (t0 == t1) {
        if (tid == 0) part.first[range] = make_uint2(0, 0);
        write_zeros();
        return;
    }
    Cursor<TILE> look;                                             // the tile whose rows are looked up next
    {
        // the sequence that holds tile t0: warps look at 32 sequences at a time
        uint32_t before = 0, b0 = 0, found = 0;
        for (; b0 < c.n_seqs; b0 += 32) {
            const uint32_t b = b0 + lane;
            uint32_t mine = b < c.n_seqs ? (c.length(b) + TILE - 1) / TILE : 0u, x = mine;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const uint32_t y = __shfl_up_sync(0xFFFFFFFFu, x, off);
                if (lane >= (uint32_t)off) x += y;
            }
            const uint32_t hit = __ballot_sync(0xFFFFFFFFu, (before + x) * c.hkv > t0);
            if (hit) {
                found = __ffs(hit) - 1;
                before += __shfl_sync(0xFFFFFFFFu, x - mine, found);
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, x, 31);
        }
        look.b = b0 + found;
        look.n = c.length(look.b);
        const uint32_t rest = t0 - before * c.hkv;
        look.h = rest / look.tiles();
        look.tile = rest - look.h * look.tiles();
    }
    Cursor<TILE> at = look;                                        // the tile that is computed next
    uint32_t to_look = t1 - t0;
    const uint32_t kbase = smem_u32(smem) + warp * kWarpBytes, vbase = kbase + kWarpBytes / 2;

    // A lane's row of a tile lies in the page that the table names, which has to be known before the tile can be asked for: the
    // table is read a tile ahead, and nothing looks at the entry until then.  Rows behind the sequence's end: kNoRow.
    uint32_t next_page = 0, next_within = kNoRow;
    auto look_up = [&] {
        next_within = kNoRow;
        if (!to_look) return;
        --to_look;
        const uint32_t r = look.tile * TILE + warp * KEYS + lane;
        if (lane < KEYS && r < look.n) {
            const uint32_t j = r / c.page_size;
            next_page = (uint32_t)c.table[(size_t)look.b * c.max_pages + j];
            next_within = look.h * c.page_size + (r - j * c.page_size);
        }
        if (to_look) look.next(c);
    };
    auto next_row = [&]() -> uint32_t {
        if (next_within == kNoRow) return kNoRow;
        if (next_page < c.n_pages) return next_page * (c.hkv * c.page_size) + next_within;
        atomicOr(c.err, kErrTable);
        return kNoRow;
    };
    // the warp's rows of a tile from a pool; rows that are none are zeros and read nothing
    auto issue = [&](const __nv_bfloat16* pool, uint32_t row, uint32_t base) {
#pragma unroll
        for (int j = 0; j < KEYS * CH / 32; ++j) {
            const uint32_t i = j * 32 + lane, rr = i / CH, ch = i % CH;
            const uint32_t ri = __shfl_sync(0xFFFFFFFFu, row, rr);
            const bool live = ri != kNoRow;
            cp16(base + rr * (D * 2) + ((ch ^ (rr & 7)) << 4), pool + ((size_t)(live ? ri : 0u) * D + ch * 8), live);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    uint32_t qf[NT][D / 16][2];
    float acc[NT][D / 16][4], m[NT][2], l[NT][2];
    // the group's queries for a segment, as the second operand of the products with the keys
    auto load_q = [&](uint32_t b, uint32_t h) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t head = nt * 8 + g;
            const uint32_t* qr = reinterpret_cast<const uint32_t*>(q + ((size_t)b * hq + h * group + (head < group ? head : 0)) * D);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                qf[nt][kk][0] = head < group ? qr[kk * 8 + t4] : 0u;
                qf[nt][kk][1] = head < group ? qr[kk * 8 + 4 + t4] : 0u;
            }
        }
    };
    look_up();
    load_q(at.b, at.h);
    uint32_t row = next_row();
    issue(c.k, row, kbase);
    issue(c.v, row, vbase);
    look_up();
    write_zeros();

    uint32_t seg_first = 0;
    uint32_t turn = 0;
    bool fresh = true;                                             // the next tile begins a segment
    for (uint32_t t = t0; t < t1; ++t) {
        if (fresh) {
            fresh = false;
            seg_first = at.tile;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int mt = 0; mt < D / 16; ++mt) acc[nt][mt][0] = acc[nt][mt][1] = acc[nt][mt][2] = acc[nt][mt][3] = 0.0f;
                m[nt][0] = m[nt][1] = -INFINITY;
                l[nt][0] = l[nt][1] = 0.0f;
            }
        }
        const uint32_t r0 = at.tile * TILE + warp * KEYS;
        // The keys' half of the buffer is refilled as soon as the scores are known, the values' half at the end of the tile, so
        // that one of them is always on its way.
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        float s[SUB][NT][4];
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[sub][nt][0] = s[sub][nt][1] = s[sub][nt][2] = s[sub][nt][3] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                // keys on M: lanes 0-7 / 8-15 address keys 0-7 / 8-15 of the first 8 elements, 16-31 the same of the next 8
                uint32_t a[4];
                const uint32_t rr = sub * 16 + (lane & 15), ch = kk * 2 + (lane >> 4);
                ldsm_x4(kbase + rr * (D * 2) + ((ch ^ (rr & 7)) << 4), a);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma(s[sub][nt], a, qf[nt][kk][0], qf[nt][kk][1]);
            }
        }
        __syncwarp();
        row = next_row();
        issue(c.k, row, kbase);
        look_up();
        const Cursor<TILE> now = at;
        const bool last = t + 1 == t1;
        if (!last) at.next(c);
        if (!last && at.tile == 0) load_q(at.b, at.h);             // the next segment's, while this one is finished
        // thread: keys g, g + 8 of every 16 (rows of s), heads 2 t4, 2 t4 + 1 of each n-tile
        bool raise = false;
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) {
            const uint32_t key = r0 + sub * 16 + g;
            const bool live0 = key < now.n, live1 = key + 8 < now.n;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& s0 = s[sub][nt][e];
                    float& s1 = s[sub][nt][2 + e];
                    s0 = live0 ? __fmul_rn(s0, scale_log2) : -INFINITY;
                    s1 = live1 ? __fmul_rn(s1, scale_log2) : -INFINITY;
                    raise |= s0 > __fadd_rn(m[nt][e], kLazy) || s1 > __fadd_rn(m[nt][e], kLazy);
                    if (WEIGHTS) {
                        const uint32_t head = nt * 8 + 2 * t4 + e;
                        if (head < group) {
                            float* dst = part.scores + ((size_t)now.b * hq + now.h * group + head) * part.pitch;
                            if (live0) dst[key] = s0;
                            if (live1) dst[key + 8] = s1;
                        }
                    }
                }
            }
        }
        if (__any_sync(0xFFFFFFFFu, raise)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = m[nt][e];
#pragma unroll
                    for (int sub = 0; sub < SUB; ++sub) top = fmaxf(top, fmaxf(s[sub][nt][e], s[sub][nt][2 + e]));
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, off));
                    const float f = top == m[nt][e] ? 1.0f : ex2(__fsub_rn(m[nt][e], top));
                    m[nt][e] = top;
                    l[nt][e] = __fmul_rn(l[nt][e], f);
#pragma unroll
                    for (int mt = 0; mt < D / 16; ++mt) {
                        acc[nt][mt][e] = __fmul_rn(acc[nt][mt][e], f);
                        acc[nt][mt][2 + e] = __fmul_rn(acc[nt][mt][2 + e], f);
                    }
                }
            }
        }
        uint32_t hi[SUB][NT][2], lo[SUB][NT][2];
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                // a maximum of -inf (nothing but -inf so far) must not turn -inf - -inf into a NaN
                const float b0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0], b1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1];
                const float p00 = ex2(__fsub_rn(s[sub][nt][0], b0)), p01 = ex2(__fsub_rn(s[sub][nt][1], b1));
                const float p10 = ex2(__fsub_rn(s[sub][nt][2], b0)), p11 = ex2(__fsub_rn(s[sub][nt][3], b1));
                l[nt][0] = __fadd_rn(l[nt][0], __fadd_rn(p00, p10));
                l[nt][1] = __fadd_rn(l[nt][1], __fadd_rn(p01, p11));
                const __nv_bfloat162 h0 = __floats2bfloat162_rn(p00, p01), h1 = __floats2bfloat162_rn(p10, p11);
                const __nv_bfloat162 e0 = __floats2bfloat162_rn(__fsub_rn(p00, __low2float(h0)), __fsub_rn(p01, __high2float(h0)));
                const __nv_bfloat162 e1 = __floats2bfloat162_rn(__fsub_rn(p10, __low2float(h1)), __fsub_rn(p11, __high2float(h1)));
                hi[sub][nt][0] = transpose8(*reinterpret_cast<const uint32_t*>(&h0));
                hi[sub][nt][1] = transpose8(*reinterpret_cast<const uint32_t*>(&h1));
                lo[sub][nt][0] = transpose8(*reinterpret_cast<const uint32_t*>(&e0));
                lo[sub][nt][1] = transpose8(*reinterpret_cast<const uint32_t*>(&e1));
            }
        }
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
#pragma unroll
        for (int sub = 0; sub < SUB; ++sub) {
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt) {
                // head dimension on M, keys on K: lanes 0-7 keys 0-7 of d 0-7, 8-15 keys 0-7 of d 8-15, 16-31 the same of keys 8-15
                uint32_t a[4];
                const uint32_t rr = sub * 16 + (lane & 7) + ((lane >> 4) << 3), ch = mt * 2 + ((lane >> 3) & 1);
                ldsm_x4_trans(vbase + rr * (D * 2) + ((ch ^ (rr & 7)) << 4), a);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma(acc[nt][mt], a, hi[sub][nt][0], hi[sub][nt][1]);
                    mma(acc[nt][mt], a, lo[sub][nt][0], lo[sub][nt][1]);
                }
            }
        }
        __syncwarp();
        issue(c.v, row, vbase);

        const uint32_t unit_tiles = now.tiles(), b = now.b, h = now.h, tile = now.tile;
        if (!last && at.tile != 0) continue;
        // ---- the segment [seg_first, tile] of unit (b, h) is done: join the warps
        fresh = true;
        const bool whole = seg_first == 0 && tile + 1 == unit_tiles;
        const uint32_t slot = range * 2 + (seg_first == 0 ? 1u : 0u);
        float (&merge_m)[kWarps][NT * 8] = merge_ms[turn];
        turn ^= 1;
        // first the common maximum, then every warp's part at that scale, then sums of four: the exponentials are taken once
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) l[nt][e] = __fadd_rn(l[nt][e], __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], off));
                if (g == 0) merge_m[warp][nt * 8 + 2 * t4 + e] = m[nt][e];
            }
        }
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t j = nt * 8 + 2 * t4 + e;
                const float M = fmaxf(fmaxf(merge_m[0][j], merge_m[1][j]), fmaxf(merge_m[2][j], merge_m[3][j]));
                const float f = m[nt][e] == M ? 1.0f : ex2(__fsub_rn(m[nt][e], M));
                if (g == 0) merge_l[warp][j] = __fmul_rn(l[nt][e], f);
                float* dst = merge + (warp * 8 + 2 * t4 + e) * S::kPitch + g;
#pragma unroll
                for (int mt = 0; mt < D / 16; ++mt) {
                    dst[mt * 16] = __fmul_rn(acc[nt][mt][e], f);
                    dst[mt * 16 + 8] = __fmul_rn(acc[nt][mt][2 + e], f);
                }
            }
            __syncthreads();
            for (uint32_t i = tid; i < 8 * (D / 4); i += kThreads) {
                const uint32_t head = nt * 8 + i / (D / 4), d4 = i % (D / 4);
                if (head >= group) break;
                const float L = __fadd_rn(__fadd_rn(merge_l[0][head], merge_l[1][head]), __fadd_rn(merge_l[2][head], merge_l[3][head]));
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(merge + (w * 8 + i / (D / 4)) * S::kPitch + d4 * 4);
                    sum.x = __fadd_rn(sum.x, v.x);
                    sum.y = __fadd_rn(sum.y, v.y);
                    sum.z = __fadd_rn(sum.z, v.z);
                    sum.w = __fadd_rn(sum.w, v.w);
                }
                const float M = fmaxf(fmaxf(merge_m[0][head], merge_m[1][head]), fmaxf(merge_m[2][head], merge_m[3][head]));
                const size_t out_head = (size_t)b * hq + h * group + head;
                if (whole) {
                    store_o(o + out_head * D + d4 * 4, sum, L);
                    if (WEIGHTS && d4 == 0) part.stats[out_head] = make_float2(M, L);
                } else {
                    reinterpret_cast<float4*>(part.o)[((size_t)slot * group + head) * (D / 4) + d4] = sum;
                    if (d4 == 0) part.ml[slot * 16 + head] = make_float2(M, L);
                }
            }
            if (nt + 1 < NT) __syncthreads();
        }
        if (tid == 0) {
            const bool begun = !whole && seg_first == 0;               // then this is the range's last tile
            uint2 f = make_uint2(0, 0);
            if (begun) f = make_uint2(ranges.holder(t + (unit_tiles - tile - 1)), b * c.hkv + h);
            if (t + 1 == t1) part.first[range] = f;
            if (WEIGHTS && seg_first == 0) part.split[b * c.hkv + h] = begun ? make_uint2(range, f.x) : make_uint2(1, 0);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// The first ranges * ceil(group / heads_each) CTAs join the parts of a unit that was cut, for heads_each of its heads: that of
// range k does it for the unit that range k began and did not finish.  (heads_each is small where units are cut into many parts:
// one CTA for 16 heads of a unit in 296 parts read 2.4 MB by itself and took over 100 us.)
// The other CTAs (only with weights) do weights_out[j] = weights_in[j] + sum over the group's heads, ascending, of exp2(s_j - M) / L
// for kWeightRows rows of a unit; they join (M, L) of a cut unit for themselves.
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
constexpr int kWeightRows = kJoinThreads * 4;

// M and L of heads head0 .. head0 + heads - 1 over slots k (+ 1 of the first) .. last, to s_m and s_l; whole CTA
__device__ __forceinline__ void join_stats(const Partials& part, uint32_t k, uint32_t last, uint32_t head0, uint32_t heads, float (*s_part)[16], float* s_m,
                                           float* s_l) {
    uint32_t wide = 1;                                     // threads are dealt to the heads in turn
    while (wide < heads) wide *= 2;
    const uint32_t head = threadIdx.x % wide, step = kJoinThreads / wide, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool mine = head < heads;
    float m = -INFINITY, l = 0.0f;
    if (mine)
#pragma unroll 4
        for (uint32_t s = k + threadIdx.x / wide; s <= last; s += step) m = fmaxf(m, part.ml[(s * 2 + (s == k)) * 16 + head0 + head].x);
    for (uint32_t off = wide; off < 32; off *= 2) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, off));
    if (lane < wide) s_part[warp][lane] = m;
    __syncthreads();
    for (int w = 0; w < kJoinWarps; ++w) m = fmaxf(m, s_part[w][head]);
    __syncthreads();
    if (mine)
#pragma unroll 4
        for (uint32_t s = k + threadIdx.x / wide; s <= last; s += step) {
            const float2 ml = part.ml[(s * 2 + (s == k)) * 16 + head0 + head];
            l = __fmaf_rn(ml.y, ml.x == m ? 1.0f : ex2(__fsub_rn(ml.x, m)), l);
        }
    for (uint32_t off = wide; off < 32; off *= 2) l = __fadd_rn(l, __shfl_xor_sync(0xFFFFFFFFu, l, off));
    if (lane < wide) s_part[warp][lane] = l;
    __syncthreads();
    if (threadIdx.x < wide) {
        l = s_part[0][head];
        for (int w = 1; w < kJoinWarps; ++w) l = __fadd_rn(l, s_part[w][head]);
        s_m[head] = m;
        s_l[head] = l;
    }
    __syncthreads();
}

template <int D>
__global__ void __launch_bounds__(kJoinThreads) attn_decode_paged_join_kernel(View c, __nv_bfloat16* __restrict__ o, uint32_t hq, uint32_t ranges, uint32_t heads_each,
                                                                              Partials part, const float* weights_in, float* weights_out) {
    __shared__ float s_part[kJoinWarps][16], s_m[16], s_l[16];
    __shared__ float4 s_o[kJoinThreads];
    pdl_trigger();
    pdl_wait();
    const uint32_t tid = threadIdx.x, group = hq / c.hkv;
    const uint32_t slices = (group + heads_each - 1) / heads_each;
    if (blockIdx.x < ranges * slices) {
        const uint32_t k = blockIdx.x / slices, head0 = (blockIdx.x - k * slices) * heads_each, heads = min(heads_each, group - head0);
        const uint2 f = part.first[k];
        if (f.x == 0) return;
        const uint32_t last = f.x, b = f.y / c.hkv, h = f.y % c.hkv;
        join_stats(part, k, last, head0, heads, s_part, s_m, s_l);
        // a thread has four elements of a head; where the group has few heads, several threads share the parts of one
        const uint32_t items = heads * (D / 4), team = items < kJoinThreads ? kJoinThreads / items : 1;
        for (uint32_t i0 = 0; i0 < items; i0 += kJoinThreads) {
            const uint32_t item = i0 + tid % min(items, (uint32_t)kJoinThreads), member = tid / min(items, (uint32_t)kJoinThreads);
            const uint32_t head = item / (D / 4), d4 = item % (D / 4);
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (member < team && item < items) {
                const float M = s_m[head];
#pragma unroll 4
                for (uint32_t s = k + member; s <= last; s += team) {
                    const uint32_t slot = s * 2 + (s == k);
                    const float m = part.ml[slot * 16 + head0 + head].x, w = m == M ? 1.0f : ex2(__fsub_rn(m, M));
                    const float4 v = reinterpret_cast<const float4*>(part.o)[(slot * group + head0 + head) * (D / 4) + d4];
                    sum.x = __fmaf_rn(v.x, w, sum.x);
                    sum.y = __fmaf_rn(v.y, w, sum.y);
                    sum.z = __fmaf_rn(v.z, w, sum.z);
                    sum.w = __fmaf_rn(v.w, w, sum.w);
                }
            }
            __syncthreads();
            s_o[tid] = sum;
            __syncthreads();
            if (member == 0 && item < items) {
                for (uint32_t j = 1; j < team; ++j) {
                    const float4 v = s_o[j * items + tid];
                    sum.x = __fadd_rn(sum.x, v.x);
                    sum.y = __fadd_rn(sum.y, v.y);
                    sum.z = __fadd_rn(sum.z, v.z);
                    sum.w = __fadd_rn(sum.w, v.w);
                }
                store_o(o + ((size_t)b * hq + h * group + head0 + head) * D + d4 * 4, sum, s_l[head]);
            }
        }
        return;
    }
    const uint32_t blocks = (c.cap() + kWeightRows - 1) / kWeightRows, at = blockIdx.x - ranges * slices;
    const uint32_t unit = at / blocks, j0 = at % blocks * kWeightRows, b = unit / c.hkv;
    const uint2 cut = part.split[unit];                    // of a unit without rows: whatever was there
    const uint32_t n = c.length(b), j = j0 + tid * 4;
    if (j0 >= n) return;
    // four heads' scores are on their way while (M, L) are joined
    constexpr uint32_t kAhead = 4;
    const float* sc = part.scores + (size_t)unit * group * part.pitch + j;       // the pitch is a multiple of 4
    auto scores_of = [&](uint32_t i) { return *reinterpret_cast<const float4*>(sc + (size_t)i * part.pitch); };
    float4 ahead[kAhead];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
        if (i < group && j < n) ahead[i] = scores_of(i);
    if (cut.x <= cut.y) {
        join_stats(part, cut.x, cut.y, 0, group, s_part, s_m, s_l);
    } else if (tid < group) {
        const float2 ml = part.stats[(size_t)unit * group + tid];
        s_m[tid] = ml.x;
        s_l[tid] = ml.y;
    }
    __syncthreads();
    if (j >= n) return;
    float4 w = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](uint32_t i, const float4& s) {
        const float m = s_m[i] == -INFINITY ? 0.0f : s_m[i], r = s_l[i] == 0.0f ? 0.0f : __frcp_rn(s_l[i]);
        w.x = __fmaf_rn(ex2(__fsub_rn(s.x, m)), r, w.x);
        w.y = __fmaf_rn(ex2(__fsub_rn(s.y, m)), r, w.y);
        w.z = __fmaf_rn(ex2(__fsub_rn(s.z, m)), r, w.z);
        w.w = __fmaf_rn(ex2(__fsub_rn(s.w, m)), r, w.w);
    };
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
        if (i < group) add(i, ahead[i]);
#pragma unroll 4
    for (uint32_t i = kAhead; i < group; ++i) add(i, scores_of(i));
    const float ws[4] = {w.x, w.y, w.z, w.w};
    const size_t to = (size_t)unit * c.cap() + j;
#pragma unroll
    for (uint32_t e = 0; e < 4; ++e)
        if (j + e < n) weights_out[to + e] = weights_in ? __fadd_rn(weights_in[to + e], ws[e]) : ws[e];
}

// ---------------------------------------------------------------- host side
struct Plan {
    uint32_t ranges, pitch;
    uint64_t first, ml, o, split, stats, scores, bytes;       // byte offsets into the workspace
};
static Plan plan_for(const View& c, uint64_t d, uint64_t hq, bool weights) {
    Plan p = {};
    const uint64_t sms = tls().sm_count > 0 ? tls().sm_count : 148;
    const uint64_t tile = d == 128 ? Shape<128>::kTile : Shape<64>::kTile;
    const uint64_t most = (uint64_t)c.n_seqs * c.hkv * ceil_div_u64(c.cap(), tile);      // tiles when every sequence is full
    const uint64_t group = hq / c.hkv, resident = sms * ctas_per_sm(group > 8 ? 2 : 1);
    p.ranges = (uint32_t)(most < resident ? most : resident);
    const uint64_t ranges = p.ranges, units = (uint64_t)c.n_seqs * c.hkv;
    auto take = [&](uint64_t bytes) { const uint64_t at = p.bytes; p.bytes += (bytes + 255) & ~255ull; return at; };
    p.first = take(ranges * sizeof(uint2));
    p.ml = take(ranges * 2 * 16 * sizeof(float2));
    p.o = take(ranges * 2 * group * d * sizeof(float));
    if (weights) {
        p.pitch = (c.cap() + 3) & ~3u;
        p.split = take(units * sizeof(uint2));
        p.stats = take((uint64_t)c.n_seqs * hq * sizeof(float2));
        p.scores = take((uint64_t)c.n_seqs * hq * p.pitch * sizeof(float));
    }
    return p;
}
static catena_status_t check_heads(const View& c, uint64_t hq, bool weights) {
    if (hq == 0 || hq % c.hkv || hq / c.hkv > 16) return fail(CATENA_E_UNSUPPORTED, "attn_decode_paged: heads must be a multiple (<= 16) of kv heads");
    // tiles of the whole call, and CTAs of the second launch, are counted in 32 bits
    const uint64_t units = (uint64_t)c.n_seqs * c.hkv;
    if (units > 0x7FFFFFFFull || units * (c.cap() / 64 + 1) > 0xFFFFFFFFull || (weights && units * ceil_div_u64(c.cap(), kWeightRows) > 0x7FFF0000ull))
        return fail(CATENA_E_TOO_LARGE, "attn_decode_paged: more rows or (sequence, kv head) pairs than the kernels index");
    return CATENA_OK;
}

template <int D, int NT, bool WEIGHTS>
static catena_status_t launch_attention(const View& c, const Plan& p, const void* q, void* o, uint64_t hq, float scale, const float* weights_in,
                                        float* weights_out, uint8_t* ws) {
    auto kernel = attn_decode_paged_kernel<D, NT, WEIGHTS>;
    static thread_local uint32_t told = 0;
    CATENA_TRY(allow_smem(kernel, Shape<D>::kSmem, &told));
    Partials part = {(uint2*)(ws + p.first), (float2*)(ws + p.ml), (float*)(ws + p.o), nullptr, nullptr, nullptr, p.pitch};
    // eight parts per unit or more: a CTA per head
    const uint32_t group = (uint32_t)hq / c.hkv, heads_each = (uint64_t)c.n_seqs * c.hkv * 8 < p.ranges ? 1 : group;
    uint64_t ctas = p.ranges;
    if (WEIGHTS) {
        part.split = (uint2*)(ws + p.split);
        part.stats = (float2*)(ws + p.stats);
        part.scores = (float*)(ws + p.scores);
    }
    // Not before the launch ahead of it is done: CTAs that start early go to whichever SM has room, some get four and some two, and the
    // call takes as long as the SMs with four (133 against 92 us for 64 x 2048 rows on average).
    How how;
    how.early = false;
    CATENA_TRY(launch_as(how, "attn_decode_paged_kernel", kernel, dim3((unsigned)ctas), dim3(kThreads), Shape<D>::kSmem, c, (const __nv_bfloat16*)q,
                      (__nv_bfloat16*)o, (uint32_t)hq, scale * 1.44269504088896340736f, part));
    ctas *= (group + heads_each - 1) / heads_each;
    if (WEIGHTS) ctas += (uint64_t)c.n_seqs * c.hkv * ceil_div_u64(c.cap(), kWeightRows);
    return launch("attn_decode_paged_join_kernel", attn_decode_paged_join_kernel<D>, dim3((unsigned)ctas), dim3(kJoinThreads), 0, c, (__nv_bfloat16*)o,
                  (uint32_t)hq, p.ranges, heads_each, part, weights_in, weights_out);
}

}  // namespace paged

using namespace paged;

extern "C" {

uint64_t catena_b200_attn_decode_paged_workspace_bytes(const catena_paged_cache_t* cache, uint64_t n_heads, int weights) {
    View c;
    if (check_cache(cache, "attn_decode_paged: null cache", &c) != CATENA_OK || check_heads(c, n_heads, weights != 0) != CATENA_OK) return 0;
    return plan_for(c, cache->head_dim, n_heads, weights != 0).bytes;
}

catena_status_t catena_b200_attn_decode_paged_bf16_into(const catena_paged_cache_t* cache, const void* q, void* o, uint64_t n_heads, float scale,
                                                        const float* weights_in, float* weights_out, void* workspace, uint64_t workspace_bytes) {
    View c;
    CATENA_TRY(check_cache(cache, "attn_decode_paged: null cache", &c));
    CATENA_TRY(check_heads(c, n_heads, weights_out != nullptr));
    if (!c.n_seqs) return CATENA_OK;
    if (!q || !o || !workspace || (weights_in && !weights_out)) return fail(CATENA_E_BAD_ARG, "attn_decode_paged: null argument");
    if (q == o) return fail(CATENA_E_BAD_ARG, "attn_decode_paged: o must be another buffer than q");
    if (!aligned16(q) || !aligned16(o) || !aligned4(weights_in) || !aligned4(weights_out) || ((uintptr_t)workspace & 255))
        return fail(CATENA_E_BAD_ARG, "attn_decode_paged: q and o must be 16-byte aligned, the workspace 256-byte");
    if (!(fabsf(scale) < 1e30f)) return fail(CATENA_E_BAD_ARG, "attn_decode_paged: scale must be finite (below 1e30)");
    CATENA_TRY(begin(&c.err));
    const Plan p = plan_for(c, cache->head_dim, n_heads, weights_out != nullptr);
    if (workspace_bytes < p.bytes) return fail(CATENA_E_BAD_ARG, "attn_decode_paged: workspace too small");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const bool wide = n_heads / c.hkv > 8, w = weights_out != nullptr;
    using Fn = catena_status_t (*)(const View&, const Plan&, const void*, void*, uint64_t, float, const float*, float*, uint8_t*);
    static const Fn table[2][2][2] = {{{launch_attention<64, 1, false>, launch_attention<64, 1, true>}, {launch_attention<64, 2, false>, launch_attention<64, 2, true>}},
                                      {{launch_attention<128, 1, false>, launch_attention<128, 1, true>}, {launch_attention<128, 2, false>, launch_attention<128, 2, true>}}};
    CATENA_TRY(table[cache->head_dim == 128][wide][w](c, p, q, o, n_heads, scale, weights_in, weights_out, ws));
    return end();
}

}  // extern "C"

}  // namespace catena
