"""What is timed of the paged key/value cache and of the beam search: the cases, their inputs, the calls a user makes of the
library (`own`), the same operators in elementary torch operations, and their definitions in 64 bits.

A paged cache: k_pages / v_pages [n_pages, n_kv_heads, page_size, head_dim] bf16, `table` [n_seqs, max_pages] int32 (row r of
sequence b lies in page table[b, r // page_size], row r % page_size of it), `lengths` [n_seqs] int32.

  append   tokens of ragged sequences: rotates queries and keys by given (cos, sin) pairs, stores keys and values in their pages
  attend   one new token per sequence over its pages; optionally adds every row's attention weight to a running total
  evict    keeps the `recent` last rows of a sequence and the rows of greatest running weight, in their order, in other pages
  select   beam search: the k best of beams x vocabulary by score + log softmax(logits)
  reorder  beam search: every beam takes over its parent's pages, with a copy of the page that is still being filled
"""
import ctypes
import math

import torch

own = False

# ---------------------------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one user's chat at the start of an answer: latency counts
        dict(name="attend_one_short", op="attend", n_seqs=1, hq=16, hkv=16, d=128, page=16, longest=300, ragged=False, weights=False),
        # a server's batch of conversations of every length, grouped heads
        dict(name="attend_batch_ragged", op="attend", n_seqs=64, hq=32, hkv=8, d=128, page=16, longest=4096, ragged=True, weights=False),
        # a few very long documents
        dict(name="attend_long", op="attend", n_seqs=4, hq=64, hkv=8, d=128, page=64, longest=131072, ragged=False, weights=False),
        # narrow heads, an odd group, pages that are no power of two, running weights kept for a later eviction
        dict(name="attend_weights", op="attend", n_seqs=24, hq=12, hkv=4, d=64, page=24, longest=6000, ragged=True, weights=True),
        # one decode step's new keys and values
        dict(name="append_step", op="append", n_seqs=64, hq=32, hkv=8, d=128, page=16, longest=512, fresh=1, pad=0),
        # prompts of different lengths packed one behind the other, the batch padded at its end
        dict(name="append_prompts", op="append", n_seqs=12, hq=16, hkv=16, d=128, page=16, longest=2048, fresh=2048, pad=77),
        # a chat's cache cut to a quarter
        dict(name="evict_chat", op="evict", n_seqs=4, hkv=8, d=128, page=16, longest=2048, budget=512, recent=128),
        # long contexts cut to a budget that some of them have not reached
        dict(name="evict_long", op="evict", n_seqs=4, hkv=8, d=128, page=64, longest=16384, budget=4096, recent=1000),
        # one request, four beams, two candidates a beam
        dict(name="select_one", op="select", batch=1, beams=4, vocab=32000, k=8, dtype="bf16"),
        # a batch of requests over a large vocabulary, logits in f32
        dict(name="select_batch", op="select", batch=32, beams=8, vocab=128000, k=16, dtype="f32"),
        # one request's beams
        dict(name="reorder_one", op="reorder", batch=1, beams=4, hkv=16, d=128, page=16, longest=300, weights=False),
        # a batch of requests, running weights carried along
        dict(name="reorder_batch", op="reorder", batch=32, beams=8, hkv=4, d=128, page=32, longest=2048, weights=True),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "evict", "select", "reorder"])
    page = rng.choice([8, 16, 16, 24, 32, 48, 64, 128])
    d = rng.choice([64, 128, 128])
    hkv = rng.choice([1, 2, 3, 4, 8, 8, 16])
    if op == "attend":
        group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 8, 12, 16])
        n_seqs = _spread(rng, 1, 256)
        longest = _spread(rng, 1, max(1, min(131072, 4 * 131072 * 8 // (n_seqs * hkv))))
        return dict(op=op, n_seqs=n_seqs, hq=group * hkv, hkv=hkv, d=d, page=page, longest=longest, ragged=rng.random() < 0.7,
                    weights=n_seqs * hkv * group * longest <= 1 << 24 and rng.random() < 0.4)
    if op == "append":
        n_seqs = _spread(rng, 1, 128)
        longest = _spread(rng, 1, max(1, 12 * 2048 * 16 // (n_seqs * hkv)))
        return dict(op=op, n_seqs=n_seqs, hq=rng.choice([1, 2, 4, 8]) * hkv, hkv=hkv, d=d, page=page, longest=longest,
                    fresh=1 if rng.random() < 0.5 else min(longest, _spread(rng, 1, 2048)), pad=rng.choice([0, 0, 1, 30]))
    if op == "evict":
        n_seqs = _spread(rng, 1, 32)
        longest = _spread(rng, 2, max(2, min(65536, 4 * 16384 * 8 // (n_seqs * hkv))))
        budget = _spread(rng, 1, longest)
        return dict(op=op, n_seqs=n_seqs, hkv=hkv, d=d, page=page, longest=longest, budget=budget, recent=rng.randint(0, budget))
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        vocab = _spread(rng, 64, 200000)
        batch = _spread(rng, 1, max(1, min(64, 32 * 8 * 128000 // (beams * vocab))))
        return dict(op=op, batch=batch, beams=beams, vocab=vocab, k=rng.choice([1, beams, 2 * beams, 2 * beams]), dtype=rng.choice(["bf16", "f32"]))
    beams = rng.choice([1, 2, 3, 4, 5, 8])
    batch = _spread(rng, 1, 64)
    longest = _spread(rng, 1, max(1, min(8192, 32 * 2048 * 4 // (batch * hkv))))
    return dict(op=op, batch=batch, beams=beams, hkv=hkv, d=d, page=page, longest=longest, weights=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------------------- inputs

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _lengths(gen, n, longest, ragged=True):
    """Rows of each sequence: all alike, or evenly spread over 0 .. longest, in an order of the seed's."""
    if not ragged or n == 1:
        return torch.full((n,), longest, dtype=torch.int32, device="cuda")
    even = torch.arange(n, device="cuda", dtype=torch.int64) * longest // (n - 1)
    return even[torch.randperm(n, generator=gen, device="cuda")].int()


def _pages(gen, n_pages, hkv, page, d):
    k = torch.randn(n_pages, hkv, page, d, generator=gen, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(n_pages, hkv, page, d, generator=gen, device="cuda", dtype=torch.bfloat16)
    return k, v


def _angles(count, d):
    """(cos, sin) of every position, as a program makes them once for its model."""
    freq = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = torch.arange(count, device="cuda", dtype=torch.float64)[:, None] * freq
    return torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()


def _inputs(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = dict(case)
    op, page, d = case["op"], case.get("page"), case.get("d")
    if op == "select":
        rows = case["batch"] * case["beams"]
        logits = torch.randn(rows, case["vocab"], generator=gen, device="cuda") * 3
        s["logits"] = logits.to(_DTYPES[case["dtype"]])
        s["scores"] = -10 * torch.rand(rows, generator=gen, device="cuda")
        n = case["batch"] * case["k"]
        s["out_scores"] = torch.zeros(case["batch"], case["k"], device="cuda")
        s["parents"] = torch.zeros(case["batch"], case["k"], dtype=torch.int32, device="cuda")
        s["tokens"] = torch.zeros(case["batch"], case["k"], dtype=torch.int32, device="cuda")
        return s
    longest = case["longest"]
    max_pages = -(-longest // page)
    if op == "reorder":
        batch, beams = case["batch"], case["beams"]
        n_seqs = batch * beams
        # beams of one request share the pages of its prompt (most of it) and have written the rest themselves
        lengths = _lengths(gen, batch, longest).clamp(min=1)
        shared = (lengths * 7 // 8 // page)[:, None, None]
        column = torch.arange(max_pages, device="cuda")
        cell = torch.arange(n_seqs * max_pages, device="cuda").view(batch, beams, max_pages)
        cell = torch.where(column < shared, cell[:, :1], cell)
        live = (column < (-(-lengths // page))[:, None, None]).expand_as(cell)
        used, page_of = torch.unique(cell[live], return_inverse=True)
        order = torch.randperm(used.numel() + n_seqs, generator=gen, device="cuda", dtype=torch.int32)
        table = torch.full_like(cell, -1, dtype=torch.int32)
        table[live] = order[page_of]
        s["table"] = table.view(n_seqs, max_pages).contiguous()
        s["lengths"] = lengths.repeat_interleave(beams).contiguous()
        s["fresh_pages"] = order[used.numel():].contiguous()
        s["parents"] = torch.randint(0, beams, (batch, beams), generator=gen, device="cuda", dtype=torch.int32)
        s["table_out"] = torch.full_like(s["table"], -1)
        s["lengths_out"] = torch.zeros_like(s["lengths"])
        s["k_pages"], s["v_pages"] = _pages(gen, order.numel(), case["hkv"], page, d)
        s["weights_in"] = s["weights_out"] = None
        if case["weights"]:
            s["weights_in"] = torch.rand(n_seqs, case["hkv"], max_pages * page, generator=gen, device="cuda")
            s["weights_out"] = torch.zeros_like(s["weights_in"])
        return s
    n_seqs = case["n_seqs"]
    lengths = _lengths(gen, n_seqs, longest, case.get("ragged", True))
    pages_out = -(-case["budget"] // page) if op == "evict" else 0
    order = torch.randperm(n_seqs * (max_pages + pages_out), generator=gen, device="cuda", dtype=torch.int32)
    s["table"] = order[: n_seqs * max_pages].view(n_seqs, max_pages).contiguous()
    s["lengths"] = lengths
    s["k_pages"], s["v_pages"] = _pages(gen, order.numel(), case["hkv"], page, d)
    cap = max_pages * page
    if op == "attend":
        # heads that look at everything and heads that look at little
        sharp = torch.linspace(0.5, 3.0, case["hq"], device="cuda")[:, None]
        s["q"] = (torch.randn(n_seqs, case["hq"], d, generator=gen, device="cuda") * sharp).to(torch.bfloat16)
        s["o"] = torch.zeros_like(s["q"])
        s["weights_in"] = s["weights_out"] = None
        if case["weights"]:
            s["weights_in"] = torch.rand(n_seqs, case["hkv"], cap, generator=gen, device="cuda")
            s["weights_out"] = torch.zeros_like(s["weights_in"])
    elif op == "append":
        # each sequence's new tokens: up to `fresh`, at most three quarters of its rows
        fresh = (lengths - lengths // 4).clamp(max=case["fresh"])
        s["token_start"] = torch.cat([fresh.new_zeros(1), fresh.cumsum(0, dtype=torch.int32)]).contiguous()
        tokens = int(s["token_start"][-1]) + case["pad"]
        s["tokens_in"] = tokens
        width = (case["hq"] + 2 * case["hkv"]) * d
        s["qkv"] = torch.randn(tokens, width, generator=gen, device="cuda", dtype=torch.bfloat16)
        s["q_out"] = torch.zeros(tokens, case["hq"], d, device="cuda", dtype=torch.bfloat16)
        # positions count the tokens seen, rows evicted since included
        s["positions"] = lengths - fresh + torch.randint(0, 100, (n_seqs,), generator=gen, device="cuda", dtype=torch.int32)
        s["angles"] = _angles(longest + 100, d)
    else:
        s["table_out"] = order[n_seqs * max_pages:].view(n_seqs, pages_out).contiguous()
        # a few rows hold most of the weight
        s["weights_in"] = torch.rand(n_seqs, case["hkv"], cap, generator=gen, device="cuda").log().neg_().pow_(3)
        s["weights_out"] = torch.zeros(n_seqs, case["hkv"], pages_out * page, device="cuda")
        s["lengths_out"] = torch.zeros_like(lengths)
        s["kept"] = torch.full((n_seqs, case["hkv"], case["budget"]), -1, dtype=torch.int32, device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    import catena_lang_b200 as cb
    lib = cb.lib()
    cb.check(lib.catena_b200_init(torch.cuda.current_device()))
    lib.catena_b200_set_blocking(0)
    s["cb"], s["lib"] = cb, lib
    if case["op"] == "select":
        need = lib.catena_b200_beam_select_workspace_bytes(case["batch"], case["beams"], case["vocab"], case["k"])
    else:
        s["cache"] = cb.PagedCacheStruct(s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), s["table"].data_ptr(), s["lengths"].data_ptr(),
                                         s["k_pages"].shape[0], case["page"], s["table"].shape[0], s["table"].shape[1], case["hkv"], case["d"])
        s["cache_ref"] = ctypes.byref(s["cache"])
        if case["op"] == "attend":
            need = lib.catena_b200_attn_decode_paged_workspace_bytes(s["cache_ref"], case["hq"], int(case["weights"]))
        elif case["op"] == "evict":
            need = lib.catena_b200_kv_evict_paged_workspace_bytes(s["cache_ref"], case["budget"])
        else:
            need = 0
    s["workspace"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------------------- passes


def _ptr(t):
    return None if t is None else t.data_ptr()


def run(s):
    op = s["op"]
    if not own:
        return _PLAIN[op](s)
    lib, check = s["lib"], s["cb"].check
    check(lib.catena_b200_set_stream(torch.cuda.current_stream().cuda_stream))
    ws, ws_bytes = s["workspace"].data_ptr(), s["workspace"].numel()
    if op == "attend":
        check(lib.catena_b200_attn_decode_paged_bf16_into(s["cache_ref"], _ptr(s["q"]), _ptr(s["o"]), s["hq"], 1 / math.sqrt(s["d"]),
                                                          _ptr(s["weights_in"]), _ptr(s["weights_out"]), ws, ws_bytes))
    elif op == "append":
        check(lib.catena_b200_rope_append_paged_bf16_into(s["cache_ref"], _ptr(s["qkv"]), s["qkv"].stride(0), _ptr(s["token_start"]), s["tokens_in"],
                                                          _ptr(s["positions"]), _ptr(s["angles"]), s["angles"].shape[0], s["hq"], _ptr(s["q_out"])))
    elif op == "evict":
        check(lib.catena_b200_kv_evict_paged_bf16_into(s["cache_ref"], _ptr(s["weights_in"]), s["budget"], s["recent"], _ptr(s["table_out"]),
                                                       s["table_out"].shape[1], _ptr(s["lengths_out"]), _ptr(s["weights_out"]), _ptr(s["kept"]),
                                                       ws, ws_bytes))
    elif op == "select":
        call = lib.catena_b200_beam_select_bf16_into if s["dtype"] == "bf16" else lib.catena_b200_beam_select_f32_into
        check(call(_ptr(s["logits"]), s["logits"].stride(0), _ptr(s["scores"]), s["batch"], s["beams"], s["vocab"], s["k"], _ptr(s["out_scores"]),
                   _ptr(s["parents"]), _ptr(s["tokens"]), ws, ws_bytes))
    else:
        check(lib.catena_b200_beam_reorder_paged_bf16_into(s["cache_ref"], _ptr(s["parents"]), s["beams"], _ptr(s["fresh_pages"]),
                                                           _ptr(s["table_out"]), _ptr(s["lengths_out"]), _ptr(s["weights_in"]),
                                                           _ptr(s["weights_out"])))
    return _outputs(s)


def _bits(pages):
    """Rows that are only copied are compared as whole numbers."""
    return pages.view(torch.int16)


def _outputs(s):
    op = s["op"]
    if op == "attend":
        return {"o": s["o"], "weights": s["weights_out"]} if s["weights"] else {"o": s["o"]}
    if op == "append":
        return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": _bits(s["v_pages"])}
    if op == "evict":
        return {"k_pages": _bits(s["k_pages"]), "v_pages": _bits(s["v_pages"]), "weights": s["weights_out"].view(torch.int32),
                "lengths": s["lengths_out"], "kept": s["kept"]}
    if op == "select":
        return {"scores": s["out_scores"], "parents": s["parents"], "tokens": s["tokens"]}
    out = {"k_pages": _bits(s["k_pages"]), "v_pages": _bits(s["v_pages"]), "table": s["table_out"], "lengths": s["lengths_out"]}
    if s["weights"]:
        out["weights"] = s["weights_out"].view(torch.int32)
    return out


def _plain_attend(s):
    n_seqs, hq, d = s["q"].shape
    hkv, page, longest = s["hkv"], s["page"], s["longest"]
    rows = torch.arange(longest, device="cuda")
    live = rows < s["lengths"][:, None]                                            # [n_seqs, longest]
    at = s["table"].long()[:, rows // page]
    mask = live[:, :, None, None]
    k = torch.where(mask, s["k_pages"][at, :, rows % page], 0).float()             # [n_seqs, longest, hkv, d]
    q = s["q"].float().view(n_seqs, hkv, hq // hkv, d)
    score = torch.einsum("bhgd,bnhd->bhgn", q, k) * (1 / math.sqrt(d))
    del k
    score = score.masked_fill(~live[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1, total)
    v = torch.where(mask, s["v_pages"][at, :, rows % page], 0).float()
    s["o"].copy_(torch.einsum("bhgn,bnhd->bhgd", p, v).reshape(n_seqs, hq, d))
    if s["weights"]:
        seen = s["weights_in"][:, :, :longest]
        s["weights_out"][:, :, :longest] = torch.where(live[:, None], seen + p.sum(2), s["weights_out"][:, :, :longest])
    return _outputs(s)


def _plain_append(s):
    hq, hkv, d, page = s["hq"], s["hkv"], s["d"], s["page"]
    start = s["token_start"].long()
    real = torch.arange(s["tokens_in"], device="cuda")
    seq = torch.searchsorted(start, real, right=True) - 1
    real = real[seq < s["n_seqs"]]
    seq = seq[seq < s["n_seqs"]]
    nth = real - start[seq]
    row = s["lengths"].long()[seq] - (start[seq + 1] - start[seq]) + nth
    turn = s["angles"][s["positions"].long()[seq] + nth][:, None]                  # [tokens, 1, d / 2, 2]
    qkv = s["qkv"][real].view(-1, hq + 2 * hkv, d)
    x = qkv[:, : hq + hkv].float()
    lo, hi = x[..., : d // 2], x[..., d // 2:]
    x = torch.cat([lo * turn[..., 0] - hi * turn[..., 1], hi * turn[..., 0] + lo * turn[..., 1]], -1).to(torch.bfloat16)
    s["q_out"][real] = x[:, :hq]
    at = s["table"].long()[seq, row // page]
    s["k_pages"][at, :, row % page] = x[:, hq:]
    s["v_pages"][at, :, row % page] = qkv[:, hq + hkv:]
    return _outputs(s)


def _plain_evict(s):
    n_seqs, hkv, cap = s["weights_in"].shape
    page, budget, recent = s["page"], s["budget"], s["recent"]
    lengths = s["lengths"].long()
    rows = torch.arange(cap, device="cuda")
    weight = torch.where(rows < (lengths - recent)[:, None, None], s["weights_in"].nan_to_num(-math.inf, math.inf, -math.inf), -math.inf)
    order = weight.sort(dim=-1, descending=True, stable=True).indices
    chosen = torch.zeros_like(weight, dtype=torch.bool).scatter_(-1, order[..., : budget - recent], True)
    length = lengths[:, None, None]
    keep = torch.where(length > budget, (chosen & (rows < length - recent)) | ((rows >= length - recent) & (rows < length)), rows < length)
    seq, head, src = keep.nonzero(as_tuple=True)
    dst = (keep.cumsum(-1) - 1)[seq, head, src]
    s["kept"][seq, head, dst] = src.int()
    s["lengths_out"].copy_(lengths.clamp(max=budget))
    s["weights_out"].zero_()
    s["weights_out"][seq, head, dst] = s["weights_in"][seq, head, src]
    old, new = s["table"].long()[seq, src // page], s["table_out"].long()[seq, dst // page]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[new, head, dst % page] = pages[old, head, src % page]
    return _outputs(s)


def _plain_select(s):
    batch, beams, vocab, k = s["batch"], s["beams"], s["vocab"], s["k"]
    x = s["logits"].double()                                     # candidates lie close together: 64 bits tell them apart
    total = (x - x.amax(-1, keepdim=True)).exp().sum(-1, keepdim=True).log() + x.amax(-1, keepdim=True)
    total = (s["scores"].double()[:, None] + (x - total)).view(batch, beams * vocab)
    best = total.topk(k).values[:, -1:]                          # everything at least as good as the k-th, then in order
    item, index = (total >= best).nonzero(as_tuple=True)
    value = total[item, index]
    order = torch.argsort(value, descending=True, stable=True)
    order = order[torch.argsort(item[order], stable=True)]
    first = torch.searchsorted(item[order].contiguous(), torch.arange(batch, device="cuda"))
    take = order[(first[:, None] + torch.arange(k, device="cuda"))]
    s["out_scores"].copy_(value[take])
    s["parents"].copy_(index[take] // vocab)
    s["tokens"].copy_(index[take] % vocab)
    return _outputs(s)


def _plain_reorder(s):
    beams, page = s["beams"], s["page"]
    n_seqs, max_pages = s["table"].shape
    source = torch.arange(n_seqs, device="cuda") // beams * beams + s["parents"].view(-1)
    length = s["lengths"].long()[source]
    s["lengths_out"].copy_(length)
    full, rest = length // page, length % page
    column = torch.arange(max_pages, device="cuda")
    table = torch.where(column < full[:, None], s["table"][source], s["table_out"])
    s["table_out"].copy_(torch.where((column == full[:, None]) & (rest > 0)[:, None], s["fresh_pages"][:, None], table))
    seq, row = (torch.arange(page, device="cuda") < rest[:, None]).nonzero(as_tuple=True)
    old = s["table"].long()[source[seq], full[seq]]
    new = s["fresh_pages"].long()[seq]
    for pages in (s["k_pages"], s["v_pages"]):
        pages[new, :, row] = pages[old, :, row]
    if s["weights"]:
        rows = torch.arange(s["weights_in"].shape[2], device="cuda")
        s["weights_out"].copy_(torch.where(rows < length[:, None, None], s["weights_in"][source], 0))
    return _outputs(s)


_PLAIN = {"attend": _plain_attend, "append": _plain_append, "evict": _plain_evict, "select": _plain_select, "reorder": _plain_reorder}


# ---------------------------------------------------------------------------------------------------------------- work


def work(case):
    """Every live row once, every output once; lengths at their mean where they are spread."""
    op = case["op"]
    if op == "select":
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + case["batch"] * case["k"] * 12, "flops": 4 * n}
    row = 2 * case["d"] * 2                                      # bytes of a row's key and value
    if op == "reorder":
        n_seqs = case["batch"] * case["beams"]
        tables = n_seqs * (case["longest"] // 2 // case["page"] + 1) * 8
        rest = min(case["page"], case["longest"]) // 2
        weights = n_seqs * case["hkv"] * case["longest"] // 2 * 8 if case["weights"] else 0
        return {"bytes": n_seqs * case["hkv"] * rest * row * 2 + tables + weights, "flops": 0}
    n_seqs, hkv = case["n_seqs"], case["hkv"]
    mean = case["longest"] / 2 if case.get("ragged", True) else case["longest"]
    if op == "attend":
        live = n_seqs * mean
        weights = live * hkv * 8 if case["weights"] else 0
        return {"bytes": int(live * hkv * row + weights + live / case["page"] * 4 + n_seqs * case["hq"] * case["d"] * 4),
                "flops": int(4 * live * case["hq"] * case["d"])}
    if op == "append":
        rows = [case["longest"] * i // max(1, n_seqs - 1) for i in range(n_seqs)] if n_seqs > 1 else [case["longest"]]
        tokens = sum(min(case["fresh"], n - n // 4) for n in rows)
        return {"bytes": int(tokens * ((case["hq"] + 2 * hkv) * case["d"] * 2 * 2 + case["d"] * 4)), "flops": int(tokens * (case["hq"] + hkv) * case["d"] * 3)}
    over = max(0.0, 1 - case["budget"] / case["longest"])        # sequences that are longer than the budget
    kept = n_seqs * (over * case["budget"] + (1 - over) * case["budget"] / 2)
    return {"bytes": int(kept * hkv * (row * 2 + 8) + n_seqs * mean * hkv * 4), "flops": 0}


# ---------------------------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    """The definitions, sequence by sequence in f64; what is only copied has no value of its own."""
    s = _inputs(case, seed)
    op, page = case["op"], case.get("page")
    if op == "select":
        return _exact_select(s)
    if op == "attend":
        if case["n_seqs"] * case["hkv"] * case["longest"] > 1 << 23:
            return None
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        weights = s["weights_out"].double() if case["weights"] else None
        group = case["hq"] // case["hkv"]
        for b, n in enumerate(s["lengths"].tolist()):
            if n == 0:
                continue
            used = s["table"][b, : -(-n // page)].long()
            for h in range(case["hkv"]):
                k = s["k_pages"][used, h].reshape(-1, case["d"])[:n].double()
                v = s["v_pages"][used, h].reshape(-1, case["d"])[:n].double()
                p = torch.softmax(s["q"][b, h * group:(h + 1) * group].double() @ k.T / math.sqrt(case["d"]), -1)
                out[b, h * group:(h + 1) * group] = p @ v
                if weights is not None:
                    weights[b, h, :n] = s["weights_in"][b, h, :n].double() + p.sum(0)
        return {"o": out, "weights": weights} if case["weights"] else {"o": out}
    if op == "append":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        q, k_pages = s["q_out"].double(), s["k_pages"].double()
        qkv = s["qkv"].double().view(-1, hq + 2 * hkv, d)
        start, lengths, positions, table = (s[n].tolist() for n in ("token_start", "lengths", "positions", "table"))
        for b in range(case["n_seqs"]):
            t0, t1 = start[b], start[b + 1]
            if t0 == t1:
                continue
            turn = torch.complex(*s["angles"][positions[b]: positions[b] + t1 - t0].double().unbind(-1))[:, None]
            z = torch.complex(qkv[t0:t1, : hq + hkv, : d // 2], qkv[t0:t1, : hq + hkv, d // 2:]) * turn
            x = torch.cat([z.real, z.imag], -1)
            q[t0:t1] = x[:, :hq]
            r0 = lengths[b] - (t1 - t0)
            for i in range(r0 // page, -(-lengths[b] // page)):
                lo, hi = max(r0, i * page), min(lengths[b], (i + 1) * page)
                k_pages[table[b][i], :, lo - i * page: hi - i * page] = x[lo - r0: hi - r0, hq:].transpose(0, 1)
        return {"q": q, "k_pages": k_pages, "v_pages": None}
    return None


def _exact_select(s):
    batch, beams, vocab, k = s["batch"], s["beams"], s["vocab"], s["k"]
    scores = torch.empty(batch, k, dtype=torch.float64, device="cuda")
    parents, tokens = torch.empty_like(s["parents"]), torch.empty_like(s["tokens"])
    for i in range(batch):
        rows = slice(i * beams, (i + 1) * beams)
        total = torch.log_softmax(s["logits"][rows].double(), -1) + s["scores"][rows].double()[:, None]
        value, index = total.view(-1).sort(dim=-1, descending=True, stable=True)
        scores[i], parents[i], tokens[i] = value[:k], index[:k] // vocab, index[:k] % vocab
    return {"scores": scores, "parents": parents, "tokens": tokens}
