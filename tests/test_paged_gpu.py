"""Paged key/value cache and beam search against plain implementations in f64 (what is only moved: bit for bit)."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import catena_lang_b200 as cb

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def device():
    L = cb.lib()
    cb.check(L.catena_b200_init(0))
    cb.check(L.catena_b200_set_stream(None))
    L.catena_b200_set_blocking(1)
    yield
    cb.check(L.catena_b200_set_stream(None))
    L.catena_b200_set_blocking(1)
    L.catena_b200_check_device_errors()


def ptr(t):
    return None if t is None else t.data_ptr()


class Cache:
    """Pools full of NaN, every sequence's rows random in pages of its own; `spare` more pages."""

    def __init__(self, seed, lengths, hkv, d, page, max_pages=None, spare=0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.n, self.hkv, self.d, self.page = len(lengths), hkv, d, page
        self.max_pages = max_pages or max(1, -(-max(lengths) // page))
        used = [-(-n // page) for n in lengths]
        order = torch.randperm(sum(used) + spare, generator=g, device="cuda").int().cpu()
        self.table = torch.full((self.n, self.max_pages), -1, dtype=torch.int32)
        at = 0
        self.k = torch.full((max(1, len(order)), hkv, page, d), math.nan, device="cuda", dtype=torch.bfloat16)
        self.v = self.k.clone()
        for b, u in enumerate(used):
            self.table[b, :u] = order[at:at + u]
            for i in range(u):
                rows = min(page, lengths[b] - i * page)
                for pool in (self.k, self.v):
                    pool[order[at + i], :, :rows] = torch.randn(hkv, rows, d, generator=g, device="cuda", dtype=torch.bfloat16)
            at += u
        self.spare = order[at:]
        self.table = self.table.cuda()
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        self.gen = g

    @property
    def cap(self):
        return self.max_pages * self.page

    def struct(self):
        return cb.PagedCacheStruct(ptr(self.k), ptr(self.v), ptr(self.table), ptr(self.lengths), self.k.shape[0], self.page, self.table.shape[0],
                                   self.max_pages, self.hkv, self.d)

    def rows(self, pool, b, n, table=None):
        """[hkv, n, d] of sequence b in f64"""
        t = (self.table if table is None else table)[b].cpu().tolist()
        idx = torch.arange(n, device="cuda")
        pages = torch.tensor(t, device="cuda")[idx // self.page]
        return pool[pages, :, idx % self.page].transpose(0, 1)


def attend(c, q, scale, w_in=None, w_out=None, out=None, ws=None):
    L = cb.lib()
    s = c.struct()
    hq = q.shape[1]
    need = L.catena_b200_attn_decode_paged_workspace_bytes(C.byref(s), hq, int(w_out is not None))
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda") if ws is None else ws       # NaNs: nothing of it may be read unwritten
    out = torch.full_like(q, math.nan) if out is None else out
    status = L.catena_b200_attn_decode_paged_bf16_into(C.byref(s), ptr(q), ptr(out), hq, scale, ptr(w_in), ptr(w_out), ptr(ws), ws.numel())
    return status, out


def attention_reference(c, q, scale, b, n):
    """o, p summed per kv head, and bounds on what f32 sums may be off by, in f64."""
    hq = q.shape[1]
    group = hq // c.hkv
    k, v = c.rows(c.k, b, n).double(), c.rows(c.v, b, n).double()
    qq = q[b].double().view(c.hkv, group, c.d)
    s = scale * qq @ k.transpose(1, 2)                                   # [hkv, group, n]
    # a score: d products exact in f32, d additions and the scaling, each off by 2^-23 at most (the tensor core truncates)
    ds = ((c.d + 3) * 2.0 ** -23 * abs(scale) * (qq.abs() @ k.abs().transpose(1, 2))).amax(-1, keepdim=True)
    p = torch.softmax(s, -1)
    # exp2 of a difference of magnitude up to |s| log2 e, twice (running and joined maximum): 2^-22 each, its argument's rounding
    rel = torch.exp(2 * ds) - 1 + 4 * 2.0 ** -22 + 4 * s.abs().amax(-1, keepdim=True) * 1.5 * 2.0 ** -23 + (n / 16 + 80) * 2.0 ** -23
    # p as a bf16 pair: what is left after two roundings
    o = (p @ v).reshape(hq, c.d)
    o_off = ((rel + 2.0 ** -16) * (p @ v.abs())).reshape(hq, c.d)
    return o, o_off, p.sum(1), (rel * p).sum(1)


SHAPES = [  # lengths, hq, hkv, d, page
    ([1], 1, 1, 128, 16), ([5, 0, 64, 65], 4, 2, 128, 16), ([63, 200, 17], 8, 1, 128, 8), ([300], 16, 16, 128, 16), ([1000, 1, 0, 333, 128], 12, 3, 128, 24),
    ([129, 127, 2], 16, 1, 64, 16), ([500, 0], 6, 2, 64, 1), ([31, 4096, 700], 10, 2, 64, 64), ([2500, 90, 90, 1300], 32, 2, 128, 48), ([40] * 70, 2, 1, 128, 7),
    ([20000], 8, 8, 128, 128), ([9999], 9, 1, 64, 1000), ([0, 0, 0], 4, 4, 128, 16), ([128] * 300, 16, 8, 64, 32),
    ([0] * 150 + [1] + [0] * 40 + [70] + [0] * 33, 2, 2, 128, 16), (([0, 3] + [0] * 31) * 60, 4, 4, 64, 8),
]


@pytest.mark.parametrize("lengths,hq,hkv,d,page", SHAPES)
@pytest.mark.parametrize("weights", [False, True])
def test_attention(lengths, hq, hkv, d, page, weights):
    c = Cache(1, lengths, hkv, d, page, max_pages=max(1, -(-max(lengths) // page)) + 2)
    q = (torch.randn(c.n, hq, d, generator=c.gen, device="cuda") * torch.linspace(0.3, 3, hq, device="cuda")[:, None]).bfloat16()
    w_in = torch.rand(c.n, hkv, c.cap, generator=c.gen, device="cuda") if weights else None
    w_out = torch.full_like(w_in, 7.0) if weights else None
    scale = 1 / math.sqrt(d)
    status, got = attend(c, q, scale, w_in, w_out)
    cb.check(status)
    for b, n in enumerate(lengths):
        if n == 0:
            assert torch.equal(got[b], torch.zeros_like(got[b]))
        else:
            o, off, p, p_off = attention_reference(c, q, scale, b, n)
            assert ((got[b].double() - o).abs() <= 2.0 ** -8 * o.abs() + off * (1 + 2.0 ** -8) + 1e-38).all(), b
            if weights:
                want = w_in[b, :, :n].double() + p
                assert ((w_out[b, :, :n].double() - want).abs() <= p_off + 2.0 ** -23 * want).all(), b
        if weights:
            assert (w_out[b, :, n:] == 7.0).all()
    status, again = attend(c, q, scale, w_in, torch.full_like(w_in, 7.0) if weights else None)
    cb.check(status)
    assert torch.equal(got, again)


def test_attention_weights_in_place_and_from_nothing():
    c = Cache(2, [70, 0, 9], 2, 128, 16)
    q = torch.randn(3, 4, 128, generator=c.gen, device="cuda").bfloat16()
    w = torch.rand(3, 2, c.cap, generator=c.gen, device="cuda")
    apart, alone, place = torch.zeros_like(w), torch.zeros_like(w), w.clone()
    for w_in, w_out in ((w, apart), (None, alone), (place, place)):
        cb.check(attend(c, q, 0.1, w_in, w_out)[0])
    assert torch.equal(place[0, :, :70], apart[0, :, :70]) and torch.equal(place[1], w[1])
    # one rounding of the sum: half a step of a value below 8
    assert ((alone + w)[0, :, :70] - apart[0, :, :70]).abs().max() <= 2.0 ** -21
    assert torch.allclose(alone.sum(-1)[0], torch.full((2,), 2.0, device="cuda"), atol=1e-5)     # two query heads, each 1


def test_attention_of_extreme_scores():
    """Scores far apart, -inf and NaN: the running maximum rises late, falls never, and one head's NaN stays its own."""
    c = Cache(3, [400, 200, 90], 1, 128, 16)
    q = torch.zeros(3, 4, 128, device="cuda", dtype=torch.bfloat16)
    q[:, :, 0] = torch.tensor([1.0, -1.0, 0.0, 30.0])
    idx = torch.arange(400, device="cuda")
    for b, n in enumerate((400, 200, 90)):
        pages = c.table[b].long()[idx[:n] // 16]
        c.k[pages, 0, idx[:n] % 16, 0] = (idx[:n].float() - n / 2).bfloat16() * 4          # rises with the row: hundreds of octaves
    status, got = attend(c, q, 1.0)
    cb.check(status)
    for b, n in enumerate((400, 200, 90)):
        o, off, _, _ = attention_reference(c, q, 1.0, b, n)
        # rows of scores in the thousands: a score's own rounding (2^-24 of it) is what counts, and lies in `off`
        assert ((got[b].double() - o).abs() <= 2.0 ** -8 * o.abs() + off + 1e-30).all(), b
    c.k[c.table[0, 3].long(), 0, 2, 0] = -math.inf          # one key of sequence 0: head 0 sees -inf, head 1 +inf, head 2 0 * inf = NaN
    status, got = attend(c, q, 1.0)
    cb.check(status)
    assert got[0, 0].isfinite().all() and got[0, 3].isfinite().all() and got[0, 1].isnan().all() and got[0, 2].isnan().all()
    assert got[1:].isfinite().all()
    for b in (1, 2):
        c.k[c.table[b, : -(-(400, 200, 90)[b] // 16)].long(), 0, :, 0] = -math.inf
    status, got = attend(c, q, 1.0)
    cb.check(status)
    assert (got[1:, 0] == 0).all() and got[1:, 1].isnan().all()      # nothing but -inf: zeros


def test_attention_behind_32_bit_offsets():
    """Pages that start beyond 2^32 bytes and 2^31 elements of the pool."""
    page, hkv, d = 64, 2, 128
    n_pages = (1 << 33) // (page * hkv * d * 2) + 40
    k = torch.empty(n_pages, hkv, page, d, device="cuda", dtype=torch.bfloat16)
    v = torch.empty_like(k)
    c = Cache(4, [150, 64], hkv, d, page, spare=0)
    far = torch.tensor([[n_pages - 1, n_pages // 2 + 1, n_pages - 9], [n_pages - 2, 0, 0]], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, d, generator=c.gen, device="cuda").bfloat16()
    _, want = attend(c, q, 0.1)
    for b, u in ((0, 3), (1, 1)):
        k[far[b, :u].long()] = c.k[c.table[b, :u].long()]
        v[far[b, :u].long()] = c.v[c.table[b, :u].long()]
    c.k, c.v, c.table = k, v, far
    status, got = attend(c, q, 0.1)
    cb.check(status)
    assert torch.equal(got, want)


@pytest.mark.parametrize("bad", ["page", "negative", "length", "negative length"])
def test_bad_tables_are_reported_and_touch_nothing(bad):
    """Every access is behind the kernels' own checks; the other sequences are served."""
    c = Cache(5, [100, 50, 80], 2, 128, 16, spare=20)
    q = torch.randn(3, 4, 128, generator=c.gen, device="cuda").bfloat16()
    _, want = attend(c, q, 0.1)
    if bad == "page":
        c.table[1, 2] = c.k.shape[0]
    elif bad == "negative":
        c.table[1, 0] = -5
    else:
        c.lengths[1] = c.cap + 1 if bad == "length" else -1
    status, got = attend(c, q, 0.1)
    assert status == cb.E_ASSERT
    # the split moves with the lengths: the last bit of the others may, too
    for b in (0, 2):
        assert ((got[b].double() - want[b].double()).abs() <= 2.0 ** -7 * want[b].double().abs() + 1e-3).all()
    before = c.k.clone()
    qkv = torch.randn(3, 8 * 128, device="cuda").bfloat16()
    angles = torch.ones(200, 64, 2, device="cuda")
    s = c.struct()
    if "length" in bad:
        assert cb.lib().catena_b200_rope_append_paged_bf16_into(C.byref(s), ptr(qkv), 8 * 128, None, 3, None, ptr(angles), 200, 4, ptr(torch.zeros_like(q))) == cb.E_ASSERT
        changed = (c.k.view(torch.int16) != before.view(torch.int16)).flatten(1).any(1).nonzero().flatten().tolist()
        assert sorted(changed) == sorted([int(c.table[0, 6]), int(c.table[2, 4])])
    w = torch.rand(3, 2, c.cap, device="cuda")
    w_out, l_out = torch.zeros(3, 2, 48, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    t_out = c.spare[:9].cuda().view(3, 3).contiguous()
    ws = torch.zeros(3 * 2 * 40 * 4, dtype=torch.uint8, device="cuda")
    # ten of fifty rows go, so some of the bad page's sixteen stay
    assert cb.lib().catena_b200_kv_evict_paged_bf16_into(C.byref(s), ptr(w), 40, 0, ptr(t_out), 3, ptr(l_out), ptr(w_out), None, ptr(ws),
                                                         ws.numel()) == cb.E_ASSERT
    assert cb.lib().catena_b200_check_device_errors() == cb.OK       # reported once


# ---------------------------------------------------------------------------------------------------------------- append
def bf16(x):
    return torch.tensor(np.asarray(x, np.float32)).bfloat16()


@pytest.mark.parametrize("d,hq,hkv,page", [(128, 4, 2, 16), (64, 3, 3, 24), (128, 8, 1, 1), (64, 16, 4, 64)])
@pytest.mark.parametrize("ragged", [True, False])
def test_append(d, hq, hkv, page, ragged):
    lengths = [40, 1, 0, 130, 17, 64] if ragged else [40, 1, 3, 130, 17, 64]
    fresh = [5, 1, 0, 130, 2, 0] if ragged else [1] * 6
    pad = (2, 3) if ragged else (0, 0)                                  # tokens before the first and behind the last sequence
    c = Cache(6, lengths, hkv, d, page, spare=3)
    tokens = sum(fresh) + sum(pad)
    wide = torch.randn(tokens, (hq + 2 * hkv) * d + 8, generator=c.gen, device="cuda").bfloat16()     # rows with a pitch
    start = torch.tensor([pad[0] + sum(fresh[:b]) for b in range(7)], dtype=torch.int32, device="cuda") if ragged else None
    first = [3, 50, 9, 0, 1000, 7]
    positions = torch.tensor(first, dtype=torch.int32, device="cuda")
    angles = torch.randn(1100, d // 2, 2, generator=c.gen, device="cuda")
    q_out = torch.full((tokens, hq, d), 5.0, device="cuda", dtype=torch.bfloat16)
    k0, v0 = c.k.clone(), c.v.clone()
    s = c.struct()
    cb.check(cb.lib().catena_b200_rope_append_paged_bf16_into(C.byref(s), ptr(wide), wide.stride(0), ptr(start), tokens, ptr(positions), ptr(angles),
                                                              1100, hq, ptr(q_out)))
    x = wide.float().cpu().numpy()[:, : (hq + 2 * hkv) * d].reshape(tokens, hq + 2 * hkv, d)
    a = angles.cpu().numpy()
    q_want = np.full((tokens, hq, d), 5.0, np.float32)
    for b in range(6):
        for i in range(fresh[b]):
            t = pad[0] + sum(fresh[:b]) + i
            cs, sn = a[first[b] + i, :, 0], a[first[b] + i, :, 1]
            lo, hi = x[t, :, : d // 2], x[t, :, d // 2:]
            y = np.concatenate([lo * cs - hi * sn, hi * cs + lo * sn], -1)         # f32, products and sum rounded separately
            q_want[t] = y[:hq]
            row = lengths[b] - fresh[b] + i
            at = int(c.table[b, row // page])
            k0[at, :, row % page] = bf16(y[hq: hq + hkv]).cuda()
            v0[at, :, row % page] = bf16(x[t, hq + hkv:]).cuda()
    assert torch.equal(q_out.cpu(), bf16(q_want))
    assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16)) and torch.equal(c.v.view(torch.int16), v0.view(torch.int16))


def test_append_with_the_librarys_angles_is_the_contiguous_append(orc):
    """Same (cos, sin), same rotation: rows and queries have the bits of rope_append_bf16 at the same positions."""
    B, S, hq, hkv, pos0, page = 2, 5, 4, 2, 3, 4
    rng = np.random.default_rng(2)
    qkv = orc.f32_to_bf16_bits(rng.standard_normal((B * S, (hq + 2 * hkv) * 128)).astype(np.float32)).reshape(B * S, -1)
    kc = np.zeros((B, hkv, 16, 128), np.uint16)
    vc = kc.copy()
    q_o = orc.rope_append_bf16(qkv, kc, vc, S, pos0, hq, hkv, 10000.0)
    angles = torch.zeros(32, 64, 2, device="cuda")
    cb.check(cb.lib().catena_b200_rope_angles_f32_into(10000.0, 0, 32, 128, ptr(angles)))
    c = Cache(7, [pos0 + S] * B, hkv, 128, page)
    x = torch.from_numpy(qkv.view(np.int16)).cuda()
    q_out = torch.zeros(B * S, hq, 128, dtype=torch.int16, device="cuda")
    start = torch.tensor([0, S, 2 * S], dtype=torch.int32, device="cuda")
    s = c.struct()
    cb.check(cb.lib().catena_b200_rope_append_paged_bf16_into(C.byref(s), ptr(x), x.shape[1], ptr(start), B * S, None, ptr(angles), 32, hq, ptr(q_out)))
    assert np.array_equal(q_out.cpu().numpy().view(np.uint16).reshape(q_o.shape), q_o)
    for b in range(B):
        for pool, want in ((c.k, kc), (c.v, vc)):
            got = c.rows(pool, b, pos0 + S)[:, pos0:].contiguous().view(torch.int16).cpu().numpy().view(np.uint16)
            assert np.array_equal(got, want[b, :, pos0: pos0 + S])
    part = torch.zeros(4, 64, 2, device="cuda")
    cb.check(cb.lib().catena_b200_rope_angles_f32_into(10000.0, 9, 4, 128, ptr(part)))
    assert torch.equal(part, angles[9:13])


def test_append_reports_positions_and_counts_out_of_range():
    c = Cache(8, [10, 20], 1, 128, 16)
    k0 = c.k.clone()
    x = torch.randn(2, 3 * 128, device="cuda").bfloat16()
    angles, q_out, s = torch.ones(30, 64, 2, device="cuda"), torch.zeros(2, 1, 128, device="cuda", dtype=torch.bfloat16), c.struct()
    call = cb.lib().catena_b200_rope_append_paged_bf16_into
    for pos in ([-1, 30], [30, 2 ** 31 - 1]):
        p = torch.tensor(pos, dtype=torch.int32, device="cuda")
        assert call(C.byref(s), ptr(x), 384, None, 2, ptr(p), ptr(angles), 30, 1, ptr(q_out)) == cb.E_ASSERT
        assert torch.equal(k0.view(torch.int16), c.k.view(torch.int16)) and (q_out == 0).all()
    many = torch.tensor([-20, 1, 2], dtype=torch.int32, device="cuda")           # 21 new tokens of a sequence of 10 rows
    assert call(C.byref(s), ptr(x), 384, ptr(many), 1, None, ptr(angles), 30, 1, ptr(q_out)) == cb.E_ASSERT
    back = torch.tensor([0, 2, 1], dtype=torch.int32, device="cuda")             # boundaries that fall
    assert call(C.byref(s), ptr(x), 384, ptr(back), 2, None, ptr(angles), 30, 1, ptr(q_out)) in (cb.OK, cb.E_ASSERT)
    cb.lib().catena_b200_check_device_errors()


# ---------------------------------------------------------------------------------------------------------------- eviction
def kept_rows(w, n, budget, recent):
    if n <= budget:
        return list(range(n))
    m = n - recent
    w = [(-math.inf if math.isnan(x) else x) for x in w[:m]]
    best = sorted(range(m), key=lambda i: (-w[i], i))[: budget - recent]
    return sorted(best) + list(range(m, n))


@pytest.mark.parametrize("lengths,hkv,d,page,budget,recent,kind", [
    ([100, 30, 0, 31, 1], 2, 128, 16, 30, 10, "random"), ([64, 65], 1, 64, 16, 64, 64, "random"), ([50], 3, 128, 24, 20, 0, "ties"),
    ([3000, 1025, 1024], 2, 64, 64, 1024, 1, "random"), ([200] * 9, 2, 128, 7, 1, 0, "ties"), ([200], 2, 128, 16, 1, 1, "zeros"),
    ([700, 699], 1, 128, 16, 90, 30, "specials"), ([5000], 1, 64, 16, 2500, 100, "two values")])
@pytest.mark.parametrize("with_kept", [True, False])
def test_evict(lengths, hkv, d, page, budget, recent, kind, with_kept):
    check_evict(lengths, hkv, d, page, budget, recent, kind, with_kept, None)


@pytest.mark.parametrize("lengths,hkv,page,max_pages,kind", [([700, 100, 2000] + [40] * 77, 1, 64, 800, "random"), ([5000], 1, 4096, 100, "two values"),
                                                             ([5000, 9000], 2, 4096, 100, "random"), ([300] * 70, 2, 16, 20, "ties")])
def test_evict_from_tables_of_any_width(lengths, hkv, page, max_pages, kind):
    """The selection's launch goes by what the table could hold: more rows than a CTA keeps in shared memory, alone and in a cluster, and more
    heads than there are SMs."""
    check_evict(lengths, hkv, 64, page, 64, 10, kind, True, max_pages)


def check_evict(lengths, hkv, d, page, budget, recent, kind, with_kept, max_pages):
    pages_out = -(-budget // page) + 1
    c = Cache(9, lengths, hkv, d, page, max_pages=max_pages, spare=pages_out * len(lengths))
    w = torch.rand(c.n, hkv, c.cap, generator=c.gen, device="cuda")
    if kind == "ties":
        w = (w * 5).floor()
    elif kind == "zeros":
        w = torch.where(w < 0.5, 0.0, -0.0)
    elif kind == "two values":
        w = torch.where(w < 0.7, 1.0, 1.0000001)
    elif kind == "specials":
        w = torch.where(w < 0.3, math.nan, torch.where(w < 0.5, -math.inf, torch.where(w < 0.52, math.inf, w - 0.7)))
    t_out = c.spare.cuda().view(c.n, pages_out).contiguous()
    kept = torch.full((c.n, hkv, budget), -3, dtype=torch.int32, device="cuda") if with_kept else None
    w_out = torch.full((c.n, hkv, pages_out * page), 9.0, device="cuda")
    l_out = torch.full((c.n,), -3, dtype=torch.int32, device="cuda")
    k0, v0 = c.k.clone(), c.v.clone()
    s = c.struct()
    need = cb.lib().catena_b200_kv_evict_paged_workspace_bytes(C.byref(s), budget)
    ws = torch.full((max(16, need),), 0xFF, dtype=torch.uint8, device="cuda")
    cb.check(cb.lib().catena_b200_kv_evict_paged_bf16_into(C.byref(s), ptr(w), budget, recent, ptr(t_out), pages_out, ptr(l_out), ptr(w_out), ptr(kept),
                                                           ptr(ws), ws.numel()))
    wn = w.cpu().numpy()
    for b, n in enumerate(lengths):
        new = min(n, budget)
        assert int(l_out[b]) == new
        for h in range(hkv):
            rows = kept_rows(wn[b, h].tolist(), n, budget, recent)
            assert len(rows) == new
            if with_kept:
                assert kept[b, h].tolist() == rows + [-3] * (budget - new)
            src, dst = torch.tensor(rows, dtype=torch.long, device="cuda"), torch.arange(new, device="cuda")
            for pool in (k0, v0):
                pool[t_out[b].long()[dst // page], h, dst % page] = pool[c.table[b].long()[src // page], h, src % page]
            want = np.zeros(pages_out * page, np.float32)
            want[:new] = wn[b, h][rows]
            assert np.array_equal(w_out[b, h].cpu().numpy().view(np.uint32), want.view(np.uint32))
    assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16)) and torch.equal(c.v.view(torch.int16), v0.view(torch.int16))


# ---------------------------------------------------------------------------------------------------------------- beams
def select(logits, scores, batch, beams, k):
    rows, vocab = logits.shape
    L = cb.lib()
    need = L.catena_b200_beam_select_workspace_bytes(batch, beams, vocab, k)
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
    out = (torch.full((batch, k), math.nan, device="cuda"), torch.full((batch, k), -9, dtype=torch.int32, device="cuda"),
           torch.full((batch, k), -9, dtype=torch.int32, device="cuda"))
    fn = L.catena_b200_beam_select_f32_into if logits.dtype == torch.float32 else L.catena_b200_beam_select_bf16_into
    cb.check(fn(ptr(logits), logits.stride(0), ptr(scores), batch, beams, vocab, k, *map(ptr, out), ptr(ws), ws.numel()))
    return out


def select_reference(logits, scores, batch, beams, k):
    """By total, then beam, then logit, then token."""
    vocab = logits.shape[1]
    x = logits.double().nan_to_num(-math.inf, math.inf, -math.inf).clamp(max=torch.finfo(torch.float32).max)
    x, token = x.sort(dim=-1, descending=True, stable=True)
    t = x - x[:, :1]
    t = scores.double()[:, None] + (t - t.exp().sum(-1, keepdim=True).log())
    t = torch.where(x == -math.inf, -math.inf, t).nan_to_num(-math.inf, math.inf, -math.inf).view(batch, beams * vocab)
    value, index = t.sort(dim=-1, descending=True, stable=True)
    index = index[:, :k]
    return value[:, :k], index // vocab, token.view(batch, beams * vocab).gather(1, index)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,beams,vocab,k", [(1, 1, 1, 1), (2, 4, 100, 8), (3, 1, 7, 7), (1, 4, 32000, 8), (2, 5, 50257, 10), (2, 64, 4100, 64), (1, 2, 4096, 64),
                                                 (5, 3, 33, 64), (1, 1, 300000, 33), (40, 2, 9000, 4), (3, 16, 200, 32), (2, 12, 64, 24), (1, 2, 300, 64)])
@pytest.mark.parametrize("pad", [0, 3, 8])
def test_select(dtype, batch, beams, vocab, k, pad):
    g = torch.Generator("cuda").manual_seed(beams * 1000 + vocab)
    logits = (torch.randn(batch * beams, vocab + pad, generator=g, device="cuda") * 3).to(dtype)
    logits[:, vocab:] = math.nan                                           # the pitch's filling is not read
    logits = logits[:, :vocab]
    scores = -8 * torch.rand(batch * beams, generator=g, device="cuda")
    got = select(logits, scores, batch, beams, k)
    value, parent, token = select_reference(logits, scores, batch, beams, k)
    assert torch.equal(got[1].long(), parent) and torch.equal(got[2].long(), token)
    # rounding to f32, and a sum of n exponentials, each off by 2^-22 and its argument's rounding (|x - max| < 40): n-fold cancels in the mean
    assert ((got[0].double() - value).abs() <= 2.0 ** -24 * value.abs() + 2.0 ** -22 + 40 * 1.5 * 2.0 ** -23 + 64 * 2.0 ** -24).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_select_of_rows_that_start_anywhere(dtype):
    """Every start within a 16-byte piece, the best logits at the rows' ends; what lies around the rows is NaN."""
    n = 16 // torch.finfo(dtype).bits * 8
    for vocab in (1, 5, 127, 1024, 4093):
        for off in range(n):
            flat = torch.full((64 + 3 * (vocab + 5),), math.nan, device="cuda", dtype=dtype)
            logits = flat[16 + off:].as_strided((3, vocab), (vocab + 5, 1))
            logits.copy_(torch.randn(3, vocab, generator=torch.Generator("cuda").manual_seed(off), device="cuda"))
            logits[:, 0], logits[:, -1] = 20.0, 30.0
            k = min(4, 3 * vocab)
            got = select(logits, torch.zeros(3, device="cuda"), 1, 3, k)
            value, _, _ = select_reference(logits, torch.zeros(3, device="cuda"), 1, 3, k)
            # The rows' best totals are alike to 1e-10, and a row's sum of exponentials is f32: each term off by 2^-22 (ex2.approx) and
            # 2^-24 (its argument, near 0 where the term counts), 22 additions deep by 2^-24 each, below 2^-19 together.  So beams may
            # change places where totals are closer than 2^-18, and what was chosen has to be as good as the best to that.
            total = torch.log_softmax(logits.double(), -1)
            chosen = total[got[1][0].long(), got[2][0].long()]
            assert ((chosen - value[0]).abs() <= 2.0 ** -18).all() and len({*zip(got[1][0].tolist(), got[2][0].tolist())}) == k
            assert ((got[0].double() - value).abs() <= 1e-5).all()


def test_select_ties_go_to_the_lowest_beam_and_token():
    logits = torch.zeros(2 * 4, 5000, device="cuda")
    got = select(logits, torch.zeros(8, device="cuda"), 2, 4, 6)
    assert got[1].tolist() == [[0] * 6] * 2 and got[2].tolist() == [list(range(6))] * 2
    logits[:, 4998:] = 1.0                                                 # two of every beam, equal over the beams
    got = select(logits.bfloat16(), torch.zeros(8, device="cuda"), 2, 4, 7)
    assert got[1].tolist() == [[0, 0, 1, 1, 2, 2, 3]] * 2 and got[2].tolist() == [[4998, 4999] * 3 + [4998]] * 2
    ordered = torch.arange(5000, device="cuda").float().repeat(8, 1) * 0.01     # the best all in one chunk, in ascending order
    got = select(ordered, torch.tensor([0.0, -100, -100, -100] * 2, device="cuda"), 2, 4, 64)
    assert got[2].tolist() == [list(range(4999, 4999 - 64, -1))] * 2 and (got[1] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,beams,vocab,k", [(2, 4, 32000, 8), (3, 16, 200, 32), (2, 8, 5000, 64)])
def test_select_of_beams_of_very_different_merit(dtype, batch, beams, vocab, k):
    """The first step of a search marks all beams but one by a large negative score; later one beam leads by far."""
    g = torch.Generator("cuda").manual_seed(3)
    logits = (torch.randn(batch * beams, vocab, generator=g, device="cuda") * 3).to(dtype)
    for others in (-1e9, -math.inf, -40.0):
        scores = torch.full((batch, beams), others, device="cuda")
        scores[:, 1] = 0.0
        got = select(logits, scores.view(-1), batch, beams, k)
        value, parent, token = select_reference(logits, scores.view(-1), batch, beams, k)
        assert torch.equal(got[1].long(), parent) and torch.equal(got[2].long(), token)
        assert (parent == 1).all() or vocab < k


def test_select_of_masks_and_dead_beams():
    inf, low = math.inf, torch.finfo(torch.float32).min
    g = torch.Generator("cuda").manual_seed(5)
    logits = torch.randn(4, 9000, generator=g, device="cuda")
    logits[0] = -inf                                     # a beam that may go nowhere
    logits[1, 5:] = -inf                                 # five ways left
    logits[2, :] = low                                   # masked with the lowest value throughout: uniform
    logits[3, 7] = math.nan
    scores = torch.tensor([0.0, -1.0, -2.0, -inf], device="cuda")
    got = select(logits, scores, 1, 4, 12)
    value, parent, token = select_reference(logits, scores, 1, 4, 12)
    assert torch.equal(got[1].long(), parent) and torch.equal(got[2].long(), token)
    assert ((got[0].double() - value).abs() <= 1e-5).all()
    got = select(logits[:2, :4], torch.tensor([0.0, -inf], device="cuda"), 1, 2, 8)      # nothing is left: -inf, in order
    by_logit = logits[1, :4].sort(descending=True).indices.tolist()
    assert (got[0] == -inf).all() and got[1].tolist() == [[0] * 4 + [1] * 4] and got[2].tolist() == [[0, 1, 2, 3] + by_logit]
    holes = torch.randn(2, 5000, generator=g, device="cuda")
    holes[:, ::2] = math.nan                             # half of everything
    got = select(holes, torch.zeros(2, device="cuda"), 1, 2, 6)
    value, parent, token = select_reference(holes, torch.zeros(2, device="cuda"), 1, 2, 6)
    assert torch.equal(got[1].long(), parent) and torch.equal(got[2].long(), token)
    assert ((got[0].double() - value).abs() <= 1e-5).all()
    big = torch.zeros(1, 10, device="cuda")
    big[0, 3] = inf
    got = select(big, torch.zeros(1, device="cuda"), 1, 1, 2)
    assert got[2][0, 0] == 3 and got[0][0, 0] == 0.0
    got = select(torch.zeros(2, 10, device="cuda"), torch.tensor([math.nan, 1.0], device="cuda"), 1, 2, 3)
    assert (got[1] == 1).all()


@pytest.mark.parametrize("batch,beams,hkv,d,page,lengths", [(1, 4, 2, 128, 16, [37]), (3, 2, 1, 64, 24, [48, 0, 5]), (2, 3, 4, 128, 1, [3, 8]), (4, 1, 2, 64, 16, [1, 16, 17, 90])])
@pytest.mark.parametrize("weights", [False, True])
def test_reorder(batch, beams, hkv, d, page, lengths, weights):
    full = [n for n in lengths for _ in range(beams)]
    c = Cache(11, full, hkv, d, page, max_pages=-(-max(lengths) // page) + 1, spare=len(full))
    parents = torch.randint(0, beams, (batch, beams), generator=c.gen, device="cuda", dtype=torch.int32)
    fresh = c.spare.cuda()
    t_out, l_out = torch.full_like(c.table, -7), torch.full_like(c.lengths, -7)
    w = torch.rand(len(full), hkv, c.cap, generator=c.gen, device="cuda") if weights else None
    w_out = torch.full_like(w, 9.0) if weights else None
    k0, v0 = c.k.clone(), c.v.clone()
    s = c.struct()
    cb.check(cb.lib().catena_b200_beam_reorder_paged_bf16_into(C.byref(s), ptr(parents), beams, ptr(fresh), ptr(t_out), ptr(l_out), ptr(w), ptr(w_out)))
    for i in range(len(full)):
        p = i // beams * beams + int(parents.view(-1)[i])
        n, whole, rest = full[p], full[p] // page, full[p] % page
        want = c.table[p, :whole].tolist() + ([int(fresh[i])] if rest else [])
        assert t_out[i].tolist() == want + [-7] * (c.max_pages - len(want)) and int(l_out[i]) == n
        for pool, old in ((c.k, k0), (c.v, v0)):
            if rest:
                old[int(fresh[i]), :, :rest] = old[int(c.table[p, whole]), :, :rest]
        if weights:
            assert torch.equal(w_out[i, :, :n], w[p, :, :n]) and (w_out[i, :, n:] == 0).all()
    assert torch.equal(c.k.view(torch.int16), k0.view(torch.int16)) and torch.equal(c.v.view(torch.int16), v0.view(torch.int16))
    parents.view(-1)[0] = beams
    assert cb.lib().catena_b200_beam_reorder_paged_bf16_into(C.byref(s), ptr(parents), beams, ptr(fresh), ptr(t_out), ptr(l_out), None, None) == cb.E_ASSERT


# ---------------------------------------------------------------------------------------------------------------- together
def test_a_captured_step_replays_on_new_lengths_and_two_streams_do_not_meet():
    """append + attention captured once, replayed as the sequences grow, against eager calls; the capture on another stream."""
    L = cb.lib()
    c = Cache(12, [30, 5, 64], 2, 128, 16, max_pages=8, spare=24)
    spare = c.spare.cuda()
    for b in range(3):                                                   # pages for the growth, beforehand
        u = -(-int(c.lengths[b]) // 16)
        c.table[b, u:u + 3] = spare[b * 3: b * 3 + 3]
    qkv = torch.zeros(3, 8 * 128, device="cuda", dtype=torch.bfloat16)
    angles = torch.zeros(200, 64, 2, device="cuda")
    cb.check(L.catena_b200_rope_angles_f32_into(10000.0, 0, 200, 128, ptr(angles)))
    q, o = (torch.zeros(3, 4, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    s = c.struct()
    ws = torch.empty(L.catena_b200_attn_decode_paged_workspace_bytes(C.byref(s), 4, 0), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()

    def step():
        cb.check(L.catena_b200_rope_append_paged_bf16_into(C.byref(s), ptr(qkv), 1024, None, 3, None, ptr(angles), 200, 4, ptr(q)))
        cb.check(L.catena_b200_attn_decode_paged_bf16_into(C.byref(s), ptr(q), ptr(o), 4, 0.09, None, None, ptr(ws), ws.numel()))
    cb.check(L.catena_b200_set_stream(stream.cuda_stream))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        # blocking mode: refused, and the capture survives
        assert L.catena_b200_attn_decode_paged_bf16_into(C.byref(s), ptr(q), ptr(o), 4, 0.09, None, None, ptr(ws), ws.numel()) == cb.E_BAD_ARG
        L.catena_b200_set_blocking(0)
        step()
        graph.capture_end()
    k0, v0, len0 = c.k.clone(), c.v.clone(), c.lengths.clone()
    outs = []
    for mode in ("graph", "eager"):
        c.k.copy_(k0), c.v.copy_(v0), c.lengths.copy_(len0)
        got = []
        for i in range(20):
            c.lengths += 1
            qkv.copy_(torch.randn(3, 1024, generator=torch.Generator("cuda").manual_seed(i), device="cuda"))
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay() if mode == "graph" else step()
            torch.cuda.synchronize()
            got.append(o.clone())
        outs.append(torch.stack(got))
    assert torch.equal(outs[0], outs[1]) and outs[0].isfinite().all()
    o_ref, off, _, _ = attention_reference(c, q, 0.09, 1, int(c.lengths[1]))
    assert ((o[1].double() - o_ref).abs() <= 2.0 ** -8 * o_ref.abs() + off * (1 + 2.0 ** -8)).all()
    cb.check(L.catena_b200_check_device_errors())


def test_what_a_non_blocking_call_met_is_reported_by_the_check():
    L = cb.lib()
    c = Cache(30, [20, 40], 1, 128, 16)
    q = torch.randn(2, 2, 128, generator=c.gen, device="cuda").bfloat16()
    c.table[1, 1] = 1 << 20
    L.catena_b200_set_blocking(0)
    assert attend(c, q, 0.1)[0] == cb.OK
    assert L.catena_b200_check_device_errors() == cb.E_ASSERT and L.catena_b200_check_device_errors() == cb.OK


def test_a_threads_first_call_is_refused_inside_a_capture():
    """It would allocate the thread's error word; the capture survives the refusal, and after a call outside it is accepted."""
    import threading
    L = cb.lib()
    c = Cache(33, [20], 1, 128, 16)
    q = torch.randn(1, 2, 128, generator=c.gen, device="cuda").bfloat16()
    o, s = torch.zeros_like(q), c.struct()
    ws = torch.empty(L.catena_b200_attn_decode_paged_workspace_bytes(C.byref(s), 2, 0), dtype=torch.uint8, device="cuda")
    seen = []

    def work():
        def call():
            return L.catena_b200_attn_decode_paged_bf16_into(C.byref(s), ptr(q), ptr(o), 2, 0.1, None, None, ptr(ws), ws.numel())
        seen.append(L.catena_b200_init(0))
        L.catena_b200_set_blocking(0)
        stream = torch.cuda.Stream()
        seen.append(L.catena_b200_set_stream(stream.cuda_stream))
        torch.cuda.synchronize()
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.stream(stream):
                graph.capture_begin()
                seen.append(call())
                graph.capture_end()
            seen.append(call())
            stream.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        seen.append(L.catena_b200_check_device_errors())
    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    assert seen == [cb.OK, cb.OK, cb.E_UNSUPPORTED, cb.OK, cb.OK, cb.OK, cb.OK]


def test_sequences_that_share_pages():
    """Two sequences that name the same pages, and one that names a page twice, are read like any others; evicting them moves copies."""
    c = Cache(31, [48, 40, 37], 2, 64, 16, spare=6)
    c.table[1] = c.table[0]
    c.table[2, 2] = c.table[2, 0]
    q = torch.randn(3, 4, 64, generator=c.gen, device="cuda").bfloat16()
    status, got = attend(c, q, 0.125)
    cb.check(status)
    for b, n in enumerate((48, 40, 37)):
        o, off, _, _ = attention_reference(c, q, 0.125, b, n)
        assert ((got[b].double() - o).abs() <= 2.0 ** -8 * o.abs() + off * (1 + 2.0 ** -8)).all()
    w = torch.rand(3, 2, c.cap, generator=c.gen, device="cuda")
    t_out = c.spare.cuda().view(3, 2).contiguous()
    l_out, w_out = torch.zeros_like(c.lengths), torch.zeros(3, 2, 32, device="cuda")
    kept = torch.zeros(3, 2, 25, dtype=torch.int32, device="cuda")
    ws = torch.empty(3 * 2 * 25 * 4, dtype=torch.uint8, device="cuda")
    s = c.struct()
    cb.check(cb.lib().catena_b200_kv_evict_paged_bf16_into(C.byref(s), ptr(w), 25, 9, ptr(t_out), 2, ptr(l_out), ptr(w_out), ptr(kept), ptr(ws), ws.numel()))
    for b, n in enumerate((48, 40, 37)):
        old, new = c.rows(c.k, b, n), c.rows(c.k, b, 25, t_out)
        for h in range(2):
            rows = kept_rows(w[b, h].tolist(), n, 25, 9)
            assert kept[b, h].tolist() == rows and torch.equal(new[h], old[h][rows])


def test_captured_eviction_and_search_replay_on_new_inputs():
    """Launches in clusters, and copies that begin beside the selection: a replayed graph gives what the calls give."""
    L = cb.lib()
    c = Cache(32, [3000] * 4, 2, 128, 16, spare=4 * 20 + 4)          # pages for every length below
    spare = c.spare.cuda()
    t_out, fresh = spare[:80].view(4, 20).contiguous(), spare[80:].contiguous()
    w = torch.rand(4, 2, c.cap, generator=c.gen, device="cuda")
    l_out, w_out = torch.zeros_like(c.lengths), torch.zeros(4, 2, 320, device="cuda")
    kept = torch.zeros(4, 2, 300, dtype=torch.int32, device="cuda")
    logits, scores = torch.zeros(4, 20000, device="cuda"), torch.zeros(4, device="cuda")
    picked = torch.zeros(2, 2, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    t2, l2 = torch.zeros_like(c.table), torch.zeros_like(c.lengths)
    s = c.struct()
    ws = torch.empty(L.catena_b200_kv_evict_paged_workspace_bytes(C.byref(s), 300), dtype=torch.uint8, device="cuda")
    ws2 = torch.empty(L.catena_b200_beam_select_workspace_bytes(2, 2, 20000, 2), dtype=torch.uint8, device="cuda")
    cb.check(L.catena_b200_rope_angles_f32_into(10000.0, 0, 1, 128, ptr(torch.zeros(64, 2, device="cuda"))))     # the thread's first call

    def calls():
        cb.check(L.catena_b200_kv_evict_paged_bf16_into(C.byref(s), ptr(w), 300, 100, ptr(t_out), 20, ptr(l_out), ptr(w_out), ptr(kept), ptr(ws), ws.numel()))
        cb.check(L.catena_b200_beam_select_f32_into(ptr(logits), 20000, ptr(scores), 2, 2, 20000, 2, *map(ptr, picked), ptr(ws2), ws2.numel()))
        cb.check(L.catena_b200_beam_reorder_paged_bf16_into(C.byref(s), ptr(picked[1]), 2, ptr(fresh), ptr(t2), ptr(l2), None, None))
    stream = torch.cuda.Stream()
    cb.check(L.catena_b200_set_stream(stream.cuda_stream))
    L.catena_b200_set_blocking(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        calls()
        graph.capture_end()
    results = {"graph": [], "eager": []}
    for i in range(4):
        g = torch.Generator("cuda").manual_seed(i)
        w.copy_(torch.rand(w.shape, generator=g, device="cuda"))
        logits.copy_(torch.randn(logits.shape, generator=g, device="cuda"))
        c.lengths.copy_(torch.tensor([[3000, 100, 2500, 64], [2999, 299, 300, 301], [310, 0, 1, 3000], [5, 6, 700, 800]][i], dtype=torch.int32))
        k0, v0 = c.k.clone(), c.v.clone()
        for mode in results:
            c.k.copy_(k0), c.v.copy_(v0)
            for t in (l_out, w_out, kept, t2, l2, *picked):
                t.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay() if mode == "graph" else calls()
            torch.cuda.synchronize()
            results[mode].append([x.clone() for x in (c.k.view(torch.int16), c.v.view(torch.int16), l_out, w_out, kept, t2, l2, *picked)])
        n = c.lengths.tolist()
        for b in range(4):
            rows = kept_rows(w[b, 1].tolist(), n[b], 300, 100)
            assert int(l_out[b]) == len(rows) and kept[b, 1, : len(rows)].tolist() == rows
    for a, b in zip(results["graph"], results["eager"]):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    cb.check(L.catena_b200_check_device_errors())


def test_two_host_threads_on_streams_of_their_own():
    """Library state belongs to the thread: calls that overlap on the device, each with its own workspace, give the bits of calls alone."""
    import threading
    L = cb.lib()
    caches = [Cache(20 + i, [700, 3, 0, 1500, 64], 4, 128, 16, spare=40) for i in range(2)]
    qs = [torch.randn(5, 8, 128, generator=c.gen, device="cuda").bfloat16() for c in caches]
    want = [attend(c, q, 0.1)[1] for c, q in zip(caches, qs)]
    logits = [torch.randn(8, 20000, generator=c.gen, device="cuda") for c in caches]
    picked = [select(x, torch.zeros(8, device="cuda"), 2, 4, 8) for x in logits]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            cb.check(L.catena_b200_init(0))
            stream = torch.cuda.Stream()
            cb.check(L.catena_b200_set_stream(stream.cuda_stream))
            L.catena_b200_set_blocking(0)
            with torch.cuda.stream(stream):
                for _ in range(50):
                    status, got = attend(caches[i], qs[i], 0.1)
                    cb.check(status)
                    again = select(logits[i], torch.zeros(8, device="cuda"), 2, 4, 8)
                    stream.synchronize()
                    if not torch.equal(got, want[i]) or not all(torch.equal(a, b) for a, b in zip(again, picked[i])):
                        wrong.append(i)
            cb.check(L.catena_b200_check_device_errors())
        except Exception as exc:          # noqa: BLE001 - reported below
            wrong.append(repr(exc))
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_serving_run():
    """A prompt appended, steps with running weights, an eviction, beams branching off and going on: each stage against a dense model
    of the same rows in f64."""
    L = cb.lib()
    hq, hkv, d, page, beams = 4, 2, 128, 8, 3
    g = torch.Generator("cuda").manual_seed(1)
    pool = 200
    k = torch.full((pool, hkv, page, d), math.nan, device="cuda", dtype=torch.bfloat16)
    v = k.clone()
    angles = torch.zeros(200, d // 2, 2, device="cuda")
    cb.check(L.catena_b200_rope_angles_f32_into(10000.0, 0, 200, d, ptr(angles)))
    free = list(range(pool))
    n, cap_pages = beams, 10
    table = torch.tensor([[free.pop() for _ in range(cap_pages)] for _ in range(n)], dtype=torch.int32, device="cuda")
    lengths = torch.zeros(n, dtype=torch.int32, device="cuda")
    positions = torch.zeros(n, dtype=torch.int32, device="cuda")
    weights = torch.zeros(n, hkv, cap_pages * page, device="cuda")
    model_k = [[[] for _ in range(hkv)] for _ in range(n)]
    model_v = [[[] for _ in range(hkv)] for _ in range(n)]
    model_w = [[[] for _ in range(hkv)] for _ in range(n)]

    def struct():
        return cb.PagedCacheStruct(ptr(k), ptr(v), ptr(table), ptr(lengths), pool, page, n, cap_pages, hkv, d)

    def append(counts):
        tokens = sum(counts)
        qkv = torch.randn(tokens, (hq + 2 * hkv) * d, generator=g, device="cuda").bfloat16()
        start = torch.tensor([sum(counts[:b]) for b in range(n + 1)], dtype=torch.int32, device="cuda")
        lengths.add_(torch.tensor(counts, dtype=torch.int32, device="cuda"))
        q = torch.zeros(tokens, hq, d, device="cuda", dtype=torch.bfloat16)
        s = struct()
        cb.check(L.catena_b200_rope_append_paged_bf16_into(C.byref(s), ptr(qkv), qkv.shape[1], ptr(start), tokens, ptr(positions), ptr(angles), 200, hq, ptr(q)))
        x = qkv.float().view(tokens, hq + 2 * hkv, d)
        t = 0
        for b in range(n):
            for i in range(counts[b]):
                a = angles[int(positions[b]) + i]
                lo, hi = x[t, : hq + hkv, : d // 2], x[t, : hq + hkv, d // 2:]
                y = torch.cat([lo * a[:, 0] - hi * a[:, 1], hi * a[:, 0] + lo * a[:, 1]], -1).bfloat16()
                assert torch.equal(y[:hq], q[t])
                for h in range(hkv):
                    model_k[b][h].append(y[hq + h].double()), model_v[b][h].append(x[t, hq + hkv + h].double()), model_w[b][h].append(0.0)
                t += 1
        positions.add_(torch.tensor(counts, dtype=torch.int32, device="cuda"))
        return q

    def step():
        q = append([1] * n)
        o = torch.zeros_like(q)
        s = struct()
        ws = torch.empty(L.catena_b200_attn_decode_paged_workspace_bytes(C.byref(s), hq, 1), dtype=torch.uint8, device="cuda")
        cb.check(L.catena_b200_attn_decode_paged_bf16_into(C.byref(s), ptr(q), ptr(o), hq, 0.088, ptr(weights), ptr(weights), ptr(ws), ws.numel()))
        for b in range(n):
            for h in range(hkv):
                kk, vv = torch.stack(model_k[b][h]), torch.stack(model_v[b][h])
                p = torch.softmax(0.088 * q[b, h * 2: h * 2 + 2].double() @ kk.T, -1)
                want = p @ vv
                # scores up to about 5: their f32 sums and the probabilities are off by less than 2^-15 of the rows' mean magnitude
                assert ((o[b, h * 2: h * 2 + 2].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -14 * (p @ vv.abs())).all()
                model_w[b][h] = [x + float(y) for x, y in zip(model_w[b][h], p.sum(0))]
                got = weights[b, h, : len(model_w[b][h])].double().cpu()
                assert (got - torch.tensor(model_w[b][h])).abs().max() < 1e-4
                model_w[b][h] = got.tolist()                    # the eviction decides by the f32 sums
        return o

    append([11, 0, 30])
    for _ in range(4):
        step()
    budget, recent = 12, 4
    t_out = torch.tensor([[free.pop() for _ in range(cap_pages)] for _ in range(n)], dtype=torch.int32, device="cuda")
    l_out, w_out = torch.zeros_like(lengths), torch.zeros_like(weights)
    kept = torch.zeros(n, hkv, budget, dtype=torch.int32, device="cuda")
    s = struct()
    ws = torch.empty(L.catena_b200_kv_evict_paged_workspace_bytes(C.byref(s), budget), dtype=torch.uint8, device="cuda")
    cb.check(L.catena_b200_kv_evict_paged_bf16_into(C.byref(s), ptr(weights), budget, recent, ptr(t_out), cap_pages, ptr(l_out), ptr(w_out), ptr(kept), ptr(ws), ws.numel()))
    for b in range(n):
        for h in range(hkv):
            rows = kept_rows(model_w[b][h], int(lengths[b]), budget, recent)
            assert kept[b, h, : len(rows)].tolist() == rows
            for m in (model_k, model_v, model_w):
                m[b][h] = [m[b][h][r] for r in rows]
    k[table.long().flatten()] = math.nan                       # the old pages are free
    v[table.long().flatten()] = math.nan
    table, lengths, weights = t_out, l_out, w_out
    for _ in range(3):
        step()
    # all three are beams of one request from here on: cut to one length, the first one's state for all
    for m in (model_k, model_v, model_w):
        for b in range(n):
            m[b] = [list(x) for x in m[0]]
    first = torch.tensor([0, 0, 0], dtype=torch.int32, device="cuda")
    for parents in (first, torch.tensor([2, 0, 0], dtype=torch.int32, device="cuda"), torch.tensor([1, 1, 2], dtype=torch.int32, device="cuda")):
        logits = torch.randn(beams, 1000, generator=g, device="cuda")
        picked = select(logits, torch.zeros(beams, device="cuda"), 1, beams, beams)
        value, parent, token = select_reference(logits, torch.zeros(beams, device="cuda"), 1, beams, beams)
        assert torch.equal(picked[1].long(), parent) and torch.equal(picked[2].long(), token)
        fresh = torch.tensor([free.pop() for _ in range(n)], dtype=torch.int32, device="cuda")
        t_out = torch.tensor([[free.pop() for _ in range(cap_pages)] for _ in range(n)], dtype=torch.int32, device="cuda")   # pages to come
        l_out, w_out = torch.zeros_like(lengths), torch.zeros_like(weights)
        s = struct()
        cb.check(L.catena_b200_beam_reorder_paged_bf16_into(C.byref(s), ptr(parents), beams, ptr(fresh), ptr(t_out), ptr(l_out), ptr(weights), ptr(w_out)))
        for m in (model_k, model_v, model_w):
            m[:] = [[list(x) for x in m[int(p)]] for p in parents]
        positions = positions[parents.long()].contiguous()
        table, lengths, weights = t_out, l_out, w_out
        for _ in range(2):
            step()
