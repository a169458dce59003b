"""The serving operators without a GPU: descriptors and arguments that the entry points refuse
before they touch a device, with the reason in turt_last_error(); and arguments that pass every
check up to the missing context."""
import ctypes as C

import pytest

from turt_b200._lib import ERR_INVALID, last_error, lib
from turt_b200.runtime import make_logit_rules, make_paged_kv

P = 1 << 20  # an aligned address that no call reaches


def _kv(**kw):
    d = dict(k=P, v=P, page_table=P, lens=P, dtype="bf16", n_pages=10, page_size=16, n_kv_head=2, head_dim=64, batch=3,
             max_pages=4)
    d.update(kw)
    return make_paged_kv(**d)


def _append(kv, k=P, ks=128, v=P, vs=128, q=P, qs=256, qo=P + 4096, qos=256, heads=4, start=None, rows=3, rot=64,
            base=1e4):
    return lib().turt_paged_append(None, C.byref(kv) if kv else None, k, ks, v, vs, q, qs, qo, qos, heads, start, rows,
                                   rot, base)


def _attend(kv, q=P, qs=256, out=P, os=256, lse=None, heads=4, scale=0.125, window=0, ws=P, wsb=1 << 30):
    return lib().turt_paged_attention(None, C.byref(kv) if kv else None, q, qs, out, os, lse, heads, scale, window, ws,
                                      wsb)


BAD_CACHES = [
    (dict(n_pages=0), "must be positive"), (dict(page_size=0), "must be positive"),
    (dict(page_size=-1), "must be positive"), (dict(n_kv_head=0), "must be positive"),
    (dict(max_pages=0), "must be positive"), (dict(head_dim=0), "head_dim"), (dict(head_dim=63), "head_dim"),
    (dict(head_dim=258), "head_dim"), (dict(batch=-1), "batch"),
    (dict(max_pages=1 << 20, page_size=1 << 12), "2^31"), (dict(k=None), "null"), (dict(v=None), "null"),
    (dict(page_table=None), "null"), (dict(lens=None), "null"), (dict(k=P + 1), "misaligned"),
    (dict(lens=P + 2), "misaligned"), (dict(slot_stride=63, head_stride=1024, page_stride=2048), "overlap"),
    (dict(slot_stride=64, head_stride=0, page_stride=2048), "overlap"),
    (dict(slot_stride=64, head_stride=1024, page_stride=(1 << 40) + 1), "too large"),
]


@pytest.mark.parametrize("bad,why", BAD_CACHES)
def test_bad_descriptors(bad, why):
    kv = _kv(**bad)
    n = C.c_size_t()
    for rc in (_append(kv), _attend(kv), lib().turt_paged_attention_workspace(C.byref(kv), 4, C.byref(n))):
        assert rc == ERR_INVALID and why in last_error()


def test_bad_type_and_null_descriptor():
    kv = _kv()
    kv.dtype = 3
    assert _append(kv) == ERR_INVALID and "type" in last_error()
    assert _append(None) == ERR_INVALID and "null descriptor" in last_error()
    assert _attend(None) == ERR_INVALID and "null descriptor" in last_error()
    with pytest.raises(ValueError):
        _kv(dtype="f64")


@pytest.mark.parametrize("bad,why", [
    (dict(rows=-1), "negative rows"), (dict(rows=2), "one row per sequence"), (dict(rot=63), "rot_dim"),
    (dict(rot=66), "rot_dim"), (dict(rot=-2), "rot_dim"), (dict(base=0.0), "base"), (dict(base=float("nan")), "base"),
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(ks=127), "row strides"), (dict(vs=0), "row strides"),
    (dict(heads=0), "heads"), (dict(qo=None), "output"), (dict(qs=255), "query strides"), (dict(qos=1), "query strides"),
    (dict(qo=P, qos=512), "in place"), (dict(k=P + 2), "misaligned"), (dict(start=P + 1), "misaligned")])
def test_append_refuses(bad, why):
    assert _append(_kv(), **bad) == ERR_INVALID and why in last_error()


@pytest.mark.parametrize("bad,why", [
    (dict(heads=3), "multiple"), (dict(heads=0), "multiple"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(qs=255), "row strides"), (dict(os=0), "row strides"), (dict(window=-1), "window"),
    (dict(scale=float("inf")), "scale"), (dict(ws=None), "workspace"), (dict(ws=P + 8), "workspace"),
    (dict(wsb=0), "workspace"), (dict(lse=P + 1), "misaligned")])
def test_attention_refuses(bad, why):
    assert _attend(_kv(), **bad) == ERR_INVALID and why in last_error()


def test_workspace_size():
    n = C.c_size_t()
    assert lib().turt_paged_attention_workspace(C.byref(_kv()), 4, C.byref(n)) == 0 and n.value > 0
    assert _attend(_kv(), wsb=n.value) == ERR_INVALID and "null context" in last_error()
    assert _attend(_kv(), wsb=n.value - 1) == ERR_INVALID and "workspace" in last_error()
    assert lib().turt_paged_attention_workspace(C.byref(_kv()), 4, None) == ERR_INVALID
    assert lib().turt_paged_attention_workspace(C.byref(_kv()), 5, C.byref(n)) == ERR_INVALID


def test_good_arguments_reach_the_context():
    for rc in (_append(_kv()), _append(_kv(), start=P, rows=7), _append(_kv(), q=None, qo=None, heads=0),
               _append(_kv(), rot=0, base=0.0), _append(_kv(), qo=P), _append(_kv(batch=0), rows=0),
               _attend(_kv()), _attend(_kv(), lse=P, window=5), _attend(_kv(dtype="f32", head_dim=2), qs=8, os=8),
               _attend(_kv(page_size=1, max_pages=4))):
        assert rc == ERR_INVALID and "null context" in last_error()


def _rules(rows=4, vocab=100, x=P, ld=100, out=P + 4096, old=100, **kw):
    return lib().turt_logit_rules_apply(None, x, ld, out, old, rows, vocab, C.byref(make_logit_rules(**kw)))


@pytest.mark.parametrize("bad,why", [
    (dict(rows=-1), "size"), (dict(vocab=-1), "size"), (dict(rows=65536), "65535"), (dict(tokens=P), "token_start"),
    (dict(repetition=P), "need tokens"), (dict(presence=P), "need tokens"), (dict(frequency=P), "need tokens"),
    (dict(bias_ids=P, bias=P), "bias_start"), (dict(bias_ids=P, bias_start=P), "bias"), (dict(mask=P), "n_masks"),
    (dict(mask=P, n_masks=3), "per row"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(ld=99), "pitch"),
    (dict(old=99), "pitch"), (dict(out=P, old=104), "in place"), (dict(x=P + 2), "misaligned"),
    (dict(tokens=P + 1, token_start=P), "misaligned"), (dict(bias_ids=P, bias=P + 2, bias_start=P), "misaligned"),
    (dict(mask=P + 3, n_masks=9), "misaligned")])
def test_rules_refuse(bad, why):
    assert _rules(**bad) == ERR_INVALID and why in last_error()


def test_good_rules_reach_the_context():
    for rc in (_rules(), _rules(tokens=P, token_start=P), _rules(out=P), _rules(rows=1, ld=0, old=0),
               _rules(mask=P, n_masks=1, mask_row=P), _rules(rows=0), _rules(bias_ids=P, bias=P, bias_start=P)):
        assert rc == ERR_INVALID and "null context" in last_error()
    assert lib().turt_logit_rules_apply(None, P, 100, P, 100, 4, 100, None) == ERR_INVALID
