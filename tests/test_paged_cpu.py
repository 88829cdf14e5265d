"""What the paged cache and the beam search refuse before anything is launched: no GPU is touched (on a machine without one a call
that is NOT refused ends in E_NO_DEVICE)."""
import ctypes as C

import pytest

import catena_lang_b200 as cb

A = 1 << 20                      # an aligned address that nothing reads


def cache(**kw):
    f = dict(k_pages=A, v_pages=A, table=A, lengths=A, n_pages=8, page_size=16, n_seqs=2, max_pages=4, n_kv_heads=2, head_dim=128)
    f.update(kw)
    return cb.PagedCacheStruct(*[f[n] for n, _ in cb.PagedCacheStruct._fields_])


def attend(c=None, q=A, o=2 * A, heads=4, scale=0.1, w_in=None, w_out=None, ws=A, ws_bytes=1 << 40):
    c = c or cache()
    return cb.lib().catena_b200_attn_decode_paged_bf16_into(C.byref(c), q, o, heads, scale, w_in, w_out, ws, ws_bytes)


def append(c=None, qkv=A, pitch=(4 + 4) * 128, start=A, tokens=3, positions=A, angles=A, n_angles=100, heads=4, q_out=A):
    c = c or cache()
    return cb.lib().catena_b200_rope_append_paged_bf16_into(C.byref(c), qkv, pitch, start, tokens, positions, angles, n_angles, heads, q_out)


def evict(c=None, w=A, budget=20, recent=5, table=2 * A, pages=2, lengths=2 * A, w_out=2 * A, kept=None, ws=A, ws_bytes=1 << 40):
    c = c or cache()
    return cb.lib().catena_b200_kv_evict_paged_bf16_into(C.byref(c), w, budget, recent, table, pages, lengths, w_out, kept, ws, ws_bytes)


def reorder(c=None, parents=A, beams=2, fresh=A, table=2 * A, lengths=2 * A, w=None, w_out=None):
    c = c or cache()
    return cb.lib().catena_b200_beam_reorder_paged_bf16_into(C.byref(c), parents, beams, fresh, table, lengths, w, w_out)


def select(kind="f32", logits=A, pitch=100, scores=A, batch=2, beams=4, vocab=100, k=8, os=A, op=A, ot=A, ws=A, ws_bytes=1 << 40):
    fn = getattr(cb.lib(), f"catena_b200_beam_select_{kind}_into")
    return fn(logits, pitch, scores, batch, beams, vocab, k, os, op, ot, ws, ws_bytes)


BAD_CACHES = [(dict(k_pages=None), cb.E_BAD_ARG), (dict(v_pages=None), cb.E_BAD_ARG), (dict(table=None), cb.E_BAD_ARG), (dict(lengths=None), cb.E_BAD_ARG),
              (dict(k_pages=A + 8), cb.E_BAD_ARG), (dict(v_pages=A + 2), cb.E_BAD_ARG), (dict(table=A + 2), cb.E_BAD_ARG), (dict(lengths=A + 1), cb.E_BAD_ARG),
              (dict(n_pages=0), cb.E_BAD_ARG), (dict(page_size=0), cb.E_BAD_ARG), (dict(max_pages=0), cb.E_BAD_ARG), (dict(n_kv_heads=0), cb.E_BAD_ARG),
              (dict(head_dim=96), cb.E_UNSUPPORTED), (dict(head_dim=256), cb.E_UNSUPPORTED),
              (dict(n_pages=1 << 31), cb.E_TOO_LARGE), (dict(n_pages=1 << 28, page_size=16), cb.E_TOO_LARGE), (dict(max_pages=1 << 28), cb.E_TOO_LARGE),
              (dict(page_size=1 << 40), cb.E_TOO_LARGE), (dict(n_seqs=1 << 21), cb.E_TOO_LARGE), (dict(n_kv_heads=1 << 20), cb.E_TOO_LARGE)]


@pytest.mark.parametrize("change,status", BAD_CACHES)
def test_bad_caches(change, status):
    c = cache(**change)
    for call in (attend, append, evict, reorder):
        assert call(c) == status
    assert cb.lib().catena_b200_attn_decode_paged_workspace_bytes(C.byref(c), 4, 0) == 0
    assert cb.lib().catena_b200_kv_evict_paged_workspace_bytes(C.byref(c), 16) == 0


def test_null_cache():
    L = cb.lib()
    assert L.catena_b200_attn_decode_paged_bf16_into(None, A, A, 4, 0.1, None, None, A, 1 << 40) == cb.E_BAD_ARG
    assert L.catena_b200_rope_append_paged_bf16_into(None, A, 1024, A, 3, A, A, 100, 4, A) == cb.E_BAD_ARG
    assert L.catena_b200_kv_evict_paged_bf16_into(None, A, 20, 5, A, 2, A, A, None, A, 1 << 40) == cb.E_BAD_ARG
    assert L.catena_b200_beam_reorder_paged_bf16_into(None, A, 2, A, A, A, None, None) == cb.E_BAD_ARG


@pytest.mark.parametrize("change,status", [
    (dict(q=None), cb.E_BAD_ARG), (dict(o=None), cb.E_BAD_ARG), (dict(o=A), cb.E_BAD_ARG), (dict(ws=None), cb.E_BAD_ARG), (dict(q=A + 8), cb.E_BAD_ARG), (dict(o=A + 2), cb.E_BAD_ARG),
    (dict(ws=A + 16), cb.E_BAD_ARG), (dict(heads=3), cb.E_UNSUPPORTED), (dict(heads=0), cb.E_UNSUPPORTED), (dict(heads=34), cb.E_UNSUPPORTED),
    (dict(scale=float("nan")), cb.E_BAD_ARG), (dict(scale=float("inf")), cb.E_BAD_ARG), (dict(scale=-3e38), cb.E_BAD_ARG), (dict(w_in=A), cb.E_BAD_ARG), (dict(w_out=A + 1), cb.E_BAD_ARG)])
def test_attention_refusals(change, status):
    assert attend(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(qkv=None), cb.E_BAD_ARG), (dict(q_out=None), cb.E_BAD_ARG), (dict(angles=None), cb.E_BAD_ARG), (dict(qkv=A + 2), cb.E_BAD_ARG),
    (dict(pitch=1023), cb.E_BAD_ARG), (dict(pitch=1016), cb.E_BAD_ARG), (dict(start=None), cb.E_BAD_ARG), (dict(start=A + 2), cb.E_BAD_ARG),
    (dict(positions=A + 1), cb.E_BAD_ARG), (dict(angles=A + 8), cb.E_BAD_ARG), (dict(tokens=1 << 31), cb.E_TOO_LARGE), (dict(heads=1 << 16), cb.E_TOO_LARGE)])
def test_append_refusals(change, status):
    assert append(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(w=None), cb.E_BAD_ARG), (dict(table=None), cb.E_BAD_ARG), (dict(lengths=None), cb.E_BAD_ARG), (dict(w_out=None), cb.E_BAD_ARG),
    (dict(ws=None), cb.E_BAD_ARG), (dict(budget=0, recent=0), cb.E_BAD_ARG), (dict(recent=21), cb.E_BAD_ARG), (dict(budget=33), cb.E_BAD_ARG),
    (dict(table=A), cb.E_BAD_ARG), (dict(lengths=A), cb.E_BAD_ARG), (dict(w_out=A), cb.E_BAD_ARG), (dict(pages=0), cb.E_TOO_LARGE),
    (dict(pages=1 << 28), cb.E_TOO_LARGE), (dict(ws_bytes=16), cb.E_BAD_ARG), (dict(kept=A + 2), cb.E_BAD_ARG)])
def test_evict_refusals(change, status):
    assert evict(**change) == status


@pytest.mark.parametrize("change,status", [
    (dict(parents=None), cb.E_BAD_ARG), (dict(fresh=None), cb.E_BAD_ARG), (dict(table=None), cb.E_BAD_ARG), (dict(lengths=None), cb.E_BAD_ARG),
    (dict(beams=0), cb.E_BAD_ARG), (dict(beams=3), cb.E_BAD_ARG), (dict(beams=4), cb.E_BAD_ARG), (dict(table=A), cb.E_BAD_ARG), (dict(lengths=A), cb.E_BAD_ARG),
    (dict(w=A), cb.E_BAD_ARG), (dict(w_out=A), cb.E_BAD_ARG), (dict(w=A, w_out=A), cb.E_BAD_ARG), (dict(parents=A + 2), cb.E_BAD_ARG)])
def test_reorder_refusals(change, status):
    assert reorder(**change) == status


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("change,status", [
    (dict(logits=None), cb.E_BAD_ARG), (dict(scores=None), cb.E_BAD_ARG), (dict(os=None), cb.E_BAD_ARG), (dict(op=None), cb.E_BAD_ARG),
    (dict(ot=None), cb.E_BAD_ARG), (dict(ws=None), cb.E_BAD_ARG), (dict(pitch=99), cb.E_BAD_ARG), (dict(logits=A + 1), cb.E_BAD_ARG),
    (dict(ws=A + 16), cb.E_BAD_ARG), (dict(beams=0), cb.E_BAD_ARG), (dict(vocab=0), cb.E_BAD_ARG), (dict(k=0), cb.E_BAD_ARG),
    (dict(beams=65), cb.E_UNSUPPORTED), (dict(k=65), cb.E_UNSUPPORTED), (dict(beams=1, vocab=7, k=8), cb.E_BAD_ARG),
    (dict(vocab=1 << 31, pitch=1 << 31), cb.E_TOO_LARGE), (dict(batch=1 << 16), cb.E_TOO_LARGE)])
def test_select_refusals(kind, change, status):
    assert select(kind, **change) == status


def test_angles_refusals():
    fn = cb.lib().catena_b200_rope_angles_f32_into
    assert fn(10000.0, 0, 4, 96, A) == cb.E_UNSUPPORTED
    for base in (0.0, -1.0, float("inf"), float("nan")):
        assert fn(base, 0, 4, 128, A) == cb.E_BAD_ARG
    assert fn(10000.0, 0, 4, 128, None) == cb.E_BAD_ARG and fn(10000.0, 0, 4, 128, A + 8) == cb.E_BAD_ARG
    assert fn(10000.0, 1 << 31, 4, 128, A) == cb.E_TOO_LARGE and fn(10000.0, 0, 1 << 31, 128, A) == cb.E_TOO_LARGE


def test_calls_without_work_are_answered_at_once():
    none = cache(n_seqs=0)
    for call in (attend, append, evict, reorder):
        assert call(none) == cb.OK
    assert append(tokens=0) == cb.OK and select(batch=0) == cb.OK
    assert cb.lib().catena_b200_rope_angles_f32_into(10000.0, 0, 0, 128, None) == cb.OK


def test_sizes_whose_products_pass_64_bits_are_refused():
    L = cb.lib()
    c = cache(n_seqs=1 << 20, n_kv_heads=1 << 15, max_pages=1 << 20, page_size=1 << 10, n_pages=1, head_dim=64)
    for weights in (0, 1):
        assert L.catena_b200_attn_decode_paged_workspace_bytes(C.byref(c), 1 << 19, weights) == 0
    assert attend(c, heads=1 << 19, w_out=A) == cb.E_TOO_LARGE and attend(c, heads=1 << 19) == cb.E_TOO_LARGE
    assert L.catena_b200_kv_evict_paged_workspace_bytes(C.byref(c), 1 << 30) == 0
    assert evict(c, budget=1 << 20, pages=1 << 11) == cb.E_TOO_LARGE
    assert append(c, pitch=1 << 62, heads=1 << 16) == cb.E_TOO_LARGE
    wide = cache(n_seqs=64, n_kv_heads=1 << 14, max_pages=1 << 21, page_size=1 << 10, n_pages=1)
    assert attend(wide, heads=1 << 14, w_out=A) == cb.E_TOO_LARGE


def test_workspaces_cover_what_they_must():
    L = cb.lib()
    c = cache(n_seqs=3, max_pages=40)
    plain = L.catena_b200_attn_decode_paged_workspace_bytes(C.byref(c), 8, 0)
    with_weights = L.catena_b200_attn_decode_paged_workspace_bytes(C.byref(c), 8, 1)
    assert 0 < plain and with_weights >= plain + 3 * 8 * 640 * 4
    assert L.catena_b200_kv_evict_paged_workspace_bytes(C.byref(c), 100) >= 3 * 2 * 100 * 4
    assert L.catena_b200_beam_select_workspace_bytes(2, 4, 32000, 8) >= 2 * 4 * 8 * 8
    assert L.catena_b200_attn_decode_paged_workspace_bytes(C.byref(c), 3, 0) == 0
    assert L.catena_b200_beam_select_workspace_bytes(2, 4, 1, 8) == 0


@pytest.mark.skipif(cb.lib().catena_b200_device_count() > 0, reason="a GPU is present")
def test_no_device_fails_loudly():
    assert attend() == cb.E_NO_DEVICE and append() == cb.E_NO_DEVICE and evict() == cb.E_NO_DEVICE
    assert reorder() == cb.E_NO_DEVICE and select() == cb.E_NO_DEVICE and select("bf16") == cb.E_NO_DEVICE
