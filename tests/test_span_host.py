"""Host side of the ops over spans of a cache: refusals before a launch, workspace sizes, Meta shapes, and the 64-bit definitions that the
GPU tests compare with.  (No address here is ever touched.)"""

import math

import pytest
import torch

import alloy_b200  # noqa: F401
from alloy_b200 import _lib
from tests import _span_ref as R

OK = 1 << 20
E_SHAPE, E_ALIGN, E_DTYPE, E_NULL, E_WORKSPACE, E_LIMIT = -1, -2, -3, -4, -6, -8

LONG = dict(s=1 << 20, w=1 << 19)      # sizes that need a workspace


def window(q=OK, qd=_lib.F16, k=OK, v=OK, nk=OK, nv=OK, ns=64, pos=OK, pos_n=1, out=OK, b=2, h=4, kv=2, d=64, n=1, s=128, w=8, sinks=0, ws=OK,
           ws_bytes=1 << 40):
    return _lib.load().alloyb_attn_window(q, 64, 64, 64, qd, k, v, nk, nv, ns, ns, ns, pos, pos_n, out, b, h, kv, d, n, s, w, sinks, -1.0, ws, ws_bytes,
                                          None)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), E_NULL), (dict(k=None), E_NULL), (dict(nk=None), E_NULL), (dict(pos=None), E_NULL), (dict(out=None), E_NULL), (dict(ws=None, **LONG), E_NULL),
    (dict(b=0), E_SHAPE), (dict(h=5), E_SHAPE), (dict(kv=0), E_SHAPE), (dict(d=96), E_SHAPE), (dict(n=129), E_SHAPE), (dict(n=-1), E_SHAPE),
    (dict(s=0), E_SHAPE), (dict(w=0), E_SHAPE), (dict(sinks=-1), E_SHAPE), (dict(pos_n=3), E_SHAPE), (dict(qd=_lib.F32), E_DTYPE),
    (dict(k=OK + 8), E_ALIGN), (dict(v=OK + 2), E_ALIGN), (dict(nk=OK + 8), E_ALIGN), (dict(ns=60), E_ALIGN), (dict(out=OK + 2), E_ALIGN),
    (dict(ws=OK + 16, **LONG), E_ALIGN), (dict(ws_bytes=0, **LONG), E_WORKSPACE), (dict(b=1025, pos_n=1), E_LIMIT), (dict(b=1000, kv=66, h=66), E_LIMIT),
])
def test_window_refusals(change, code):
    assert window(**change) == code


def test_no_tokens_is_no_launch():
    assert window(n=0) == 0


def test_prefix_scored_and_evict_refusals():
    lib = _lib.load()

    def prefix(pk=OK, phs=1024, p=16):
        return lib.alloyb_attn_shared_prefix(OK, 64, 64, 64, _lib.F16, pk, OK, phs, p, OK, OK, None, None, 0, 0, 0, OK, 1, OK, 2, 4, 2, 64, 0, 128, -1.0, OK,
                                             1 << 40, None)
    assert prefix() == 0 and prefix(None, p=0) == 0
    assert prefix(None) == E_NULL and prefix(OK + 8) == E_ALIGN and prefix(phs=1028) == E_ALIGN and prefix(phs=1016) == E_SHAPE and prefix(p=-1) == E_SHAPE

    def scored(w):
        return lib.alloyb_attn_scored(OK, 64, 64, 64, _lib.F16, OK, OK, None, None, 0, 0, 0, OK, 1, w, OK, 2, 4, 2, 64, 0, 128, -1.0, OK, 1 << 40, None)
    assert scored(OK) == 0 and scored(None) == E_NULL and scored(OK + 2) == E_ALIGN

    mb = 1 << 20
    # (addresses a megabyte apart; a cache here is 2 * 2 * 100 * 64 * 2 = 51200 bytes)

    def evict(k=mb, ko=4 * mb, wo=6 * mb, b=2, d=64, s=100, s_out=50, keep=50, sinks=0, recent=0, count=2):
        return lib.alloyb_kv_evict(k, 2 * mb, 3 * mb, OK, count, ko, 5 * mb, wo, 7 * mb, 8 * mb, b, 2, d, s, s_out, keep, sinks, recent, None)
    assert evict(k=None) == E_NULL
    for bad in (dict(b=0), dict(d=96), dict(keep=51), dict(keep=0), dict(sinks=-1), dict(sinks=30, recent=21), dict(count=3), dict(ko=mb),
                dict(ko=mb + 16), dict(ko=2 * mb), dict(ko=mb + 51200 - 16), dict(wo=2 * mb)):
        assert evict(**bad) == E_SHAPE, bad
    assert evict(ko=mb + 512, s_out=100) == E_SHAPE
    assert evict(ko=4 * mb + 8) == E_ALIGN
    assert evict(b=40000, count=1) == E_LIMIT


def test_workspace_is_arithmetic_and_covers_what_the_calls_ask():
    size = _lib.load().alloyb_attn_span_workspace_bytes
    assert size(0, 4, 2, 64, 1, 128, 8, 0, 0, 0) == 0 and size(1, 4, 2, 64, 1, 128, -1, 0, 0, 0) == 0
    long = (2, 8, 2, 128, 1, 1 << 17)
    plain, with_prefix, with_scores = size(*long, 0, 0, 0, 0), size(*long, 0, 0, 999, 0), size(*long, 0, 0, 0, 1)
    assert 0 < plain and plain % 256 == 0 and with_prefix > plain and with_scores >= plain + 2 * 8 * (1 << 17) * 4
    assert size(1, 8, 2, 128, 1, 128, 64, 4, 0, 0) == 0                         # few keys: one launch that needs none
    assert size(64, 64, 8, 128, 1, 1 << 20, 4096, 4, 0, 0) < 64 << 20           # a window's does not grow with the cache
    for n in (1, 40):
        assert window(n=n, ws_bytes=size(2, 4, 2, 64, n, LONG["s"], LONG["w"], 0, 0, 0) - 1, **LONG) == E_WORKSPACE


def test_meta_shapes():
    ops = torch.ops.alloy
    q = torch.empty(2, 8, 3, 64, dtype=torch.bfloat16, device="meta")
    kv, c = torch.empty(2, 2, 3, 64, dtype=torch.float16, device="meta"), torch.empty(2, 2, 50, 64, dtype=torch.float16, device="meta")
    w, pos = torch.empty(2, 2, 50, device="meta"), torch.empty(2, dtype=torch.int32, device="meta")
    for out in (ops.attention_cache_window(q, kv, kv, pos, c, c, 8, 2), ops.attention_shared_prefix(q, kv, kv, pos, kv[0], kv[0], c, c),
                ops.attention_cache_scored(q, kv, kv, pos, c, c, w)):
        assert out.shape == q.shape and out.dtype == q.dtype and out.stride() == (3 * 8 * 64, 64, 8 * 64, 1)
    kept, n = ops.kv_evict(c, c, w, pos, c, c, w, 20, 2, 3)
    assert kept.shape == (2, 2, 20) and kept.dtype == torch.int32 and n.shape == (2,)
    with pytest.raises(NotImplementedError):
        ops.attention_cache_window(torch.zeros(1, 2, 1, 64), torch.zeros(1, 2, 1, 64), torch.zeros(1, 2, 1, 64), torch.zeros(1), torch.zeros(1, 2, 8, 64),
                                   torch.zeros(1, 2, 8, 64), 4)


def test_the_definitions_themselves():
    """A window as long as the context is plain attention; a cache cut at P is a prefix and the rest; weights sum to rows x tokens."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, x, y, 16, generator=g, dtype=torch.float64) for x, y in ((4, 2), (2, 20), (2, 20)))
    full, w, _, _ = R.attention(q, k, v, [15])
    s = (q[0, 3, 1] @ k[0, 1, :17].T / 4).softmax(0) @ v[0, 1, :17]
    assert torch.allclose(full[0, 3, 1], s)
    assert torch.allclose(full, R.attention(q, k, v, [15], window=17)[0]) and not torch.allclose(full, R.attention(q, k, v, [15], window=15)[0])
    assert torch.allclose(full, R.attention(q, k, v, [15], window=3, sinks=15)[0])
    cut = R.attention(q, k[:, :, 9:], v[:, :, 9:], [6], prefix=(k[0, :, :9], v[0, :, :9]))[0]
    assert torch.allclose(full, cut)
    assert math.isclose(float(w.sum()), 4 * 2)
    for kw in (dict(), dict(window=3, sinks=2), dict(prefix=(k[0, :, :9], v[0, :, :9]))):
        grown = torch.zeros(1, 2, 20, dtype=torch.float64)
        a, b = R.attention(q, k, v, [15], **kw), R.attention_wide(q, k, v, [15], weights=None if "prefix" in kw else grown, **kw)
        assert torch.allclose(a[0], b[0]) and torch.allclose(a[2], b[1]) and torch.allclose(a[1], grown)
    assert R.evict([5, 1, 3, 3, 2, 9, 0, 0], 8, 5, 1, 1) == [0, 2, 3, 5, 7]
    assert R.evict([1.0, float("nan"), 0.0, 1.0], 4, 3, 0, 0) == [0, 2, 3]


@pytest.mark.parametrize("change", [
    dict(new=3), dict(new=3, new_off=4), dict(new=0), dict(new=2), dict(new=4), dict(new=7), dict(kept=3), dict(kept=1), dict(kept=6), dict(kept=6, kept_off=96),
    dict(ko=5, ko_off=512), dict(vo=4, vo_off=16), dict(wo=4), dict(wo=5, wo_off=1024),
])
def test_evict_outputs_lie_apart(change):
    """The sequence's CTAs read its length while one of them writes the new one, and copies know no order among outputs."""
    mb = 1 << 20
    # places 0 .. 8, megabytes apart: k, v, weights, lengths, k_out, v_out, weights_out, kept, new_lengths

    def evict(ko=4, vo=5, wo=6, kept=7, new=8, ko_off=0, vo_off=0, wo_off=0, kept_off=0, new_off=0, b=2):
        at = lambda i, off=0: (i + 1) * mb + off  # noqa: E731
        return _lib.load().alloyb_kv_evict(at(0), at(1), at(2), at(3), 2, at(ko, ko_off), at(vo, vo_off), at(wo, wo_off), at(kept, kept_off), at(new, new_off), b, 2,
                                           64, 100, 50, 50, 0, 0, None)
    assert evict(b=3) == E_SHAPE                                               # (two lengths for three sequences: the call is refused before a launch)
    assert evict(**change) == E_SHAPE


def test_scored_workspace_is_bounded():
    """A prompt-sized scored call asks for no more than its parts of 1 GiB of scores (and what is joined), one token for what one token needs."""
    size = _lib.load().alloyb_attn_span_workspace_bytes
    gib = 1 << 30
    for n in (64, 2048, 4096, 32768):
        assert size(1, 32, 8, 128, n, 131072, 0, 0, 0, 1) < 1.5 * gib
    assert size(1, 32, 8, 128, 32, 1 << 18, 0, 0, 0, 1) >= gib                 # 32 MiB a token: a call of 32 is one part
    token = size(16, 64, 8, 64, 1, 1 << 20, 0, 0, 0, 1)
    assert token >= 4 * gib and size(16, 64, 8, 64, 5, 1 << 20, 0, 0, 0, 1) < token + gib // 4
    for n in (1, 33, 4096):
        need = size(1, 32, 8, 128, n, 131072, 0, 0, 0, 1)
        assert _lib.load().alloyb_attn_scored(OK, 64, 64, 64, _lib.F16, OK, OK, None, None, 0, 0, 0, OK, 1, OK, OK, 1, 32, 8, 128, n, 131072, -1.0, OK,
                                              need - 1, None) == E_WORKSPACE
