"""Attention over a window with sinks, behind a shared prefix and with its weights kept, and eviction by those weights, against their
definitions in 64 bits."""

import threading

import pytest
import torch

import alloy_b200  # noqa: F401
from alloy_b200 import _lib, ops
from tests import _span_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
OPS = torch.ops.alloy
BAD = float("nan")


class Case:
    """Inputs of one call.  Rows that no token sees hold NaN."""

    def __init__(self, b, h, kv_h, d, n, s, pos, dtype=torch.float16, seed=0, layout="model", prefix=0, q_scale=1.5):
        g = torch.Generator().manual_seed(seed * 7919 + b * 31 + h * 7 + d + n * 1009 + s)

        def rows(*shape, scale=1.0):
            return (torch.randn(*shape, generator=g) * scale)

        self.b, self.h, self.kv_h, self.d, self.n, self.s, self.pos, self.dtype = b, h, kv_h, d, n, s, list(pos), dtype
        q = rows(b, n, h, d, scale=q_scale).to(dtype)
        nk, nv = rows(b, n, kv_h, d).half(), rows(b, n, kv_h, d).half()
        if layout == "model":                      # (B, n, heads, D) seen as (B, heads, n, D)
            self.q, self.nk, self.nv = (x.to(DEV).transpose(1, 2) for x in (q, nk, nv))
        elif layout == "packed":                   # slices of one q|k|v buffer that begins off a 16-byte boundary
            buf = torch.zeros(b, n, (h + 2 * kv_h) * d + 3, dtype=dtype, device=DEV)
            self.q = buf[..., 1:1 + h * d].unflatten(-1, (h, d)).transpose(1, 2)
            self.q.copy_(q.to(DEV).transpose(1, 2))
            odd = torch.zeros(b, n, 2 * kv_h * d + 5, dtype=torch.float16, device=DEV)
            self.nk = odd[..., 1:1 + kv_h * d].unflatten(-1, (kv_h, d)).transpose(1, 2)
            self.nv = odd[..., 1 + kv_h * d:1 + 2 * kv_h * d].unflatten(-1, (kv_h, d)).transpose(1, 2)
            self.nk.copy_(nk.to(DEV).transpose(1, 2))
            self.nv.copy_(nv.to(DEV).transpose(1, 2))
        else:                                      # dense (B, heads, n, D)
            self.q, self.nk, self.nv = (x.to(DEV).transpose(1, 2).contiguous() for x in (q, nk, nv))
        self.k, self.v = rows(b, kv_h, s, d).half(), rows(b, kv_h, s, d).half()
        self.q64, self.nk64, self.nv64 = (x.transpose(1, 2).double() for x in (q, nk, nv))
        if prefix:
            self.pk, self.pv = (rows(kv_h, prefix, d).half() for _ in range(2))

    def place(self, i):
        p = self.pos[i if len(self.pos) > 1 else 0]
        return p if 0 <= p and p + self.n <= self.s else None

    def caches(self, write, window=0, sinks=0):
        """Device caches (the tokens' rows in them unless the call writes them), and both in 64 bits with the rows in place."""
        k, v = self.k.clone(), self.v.clone()
        full_k, full_v = k.double(), v.double()
        for i in range(self.b):
            p = self.place(i)
            if p is None:
                k[i], v[i] = BAD, BAD
                continue
            full_k[i, :, p:p + self.n], full_v[i, :, p:p + self.n] = self.nk64[i], self.nv64[i]
            k[i, :, p:], v[i, :, p:] = BAD, BAD
            if not write:
                k[i, :, p:p + self.n], v[i, :, p:p + self.n] = self.nk64[i].half(), self.nv64[i].half()
            if window:
                lo = max(0, p - window + 1)
                k[i, :, min(sinks, lo):lo], v[i, :, min(sinks, lo):lo] = BAD, BAD
        return k.to(DEV), v.to(DEV), full_k, full_v

    def pos_t(self, dtype=torch.int32):
        return torch.tensor(self.pos, dtype=dtype, device=DEV)

    def check_written(self, before, after, rows64, write):
        want = before.clone()
        if write:
            for i in range(self.b):
                p = self.place(i)
                if p is not None:
                    want[i, :, p:p + self.n] = rows64[i].half().to(DEV)
        assert torch.equal(after.view(torch.int16), want.view(torch.int16))


def check(out, ref, mag, dtype, what=""):
    got = out.double().cpu()
    assert _lib.load().alloyb_device_error(1) == 0
    over = (got - ref).abs() - R.out_bound(ref, mag, dtype)
    assert torch.isfinite(got).all() and float(over.max()) <= 0, f"{what}: {float((got - ref).abs().max()):.3e} off, {float(over.max()):.3e} over"


SHAPES = [
    # b, h, kv_h, d, n, s, pos, window, sinks, dtype, layout, write
    (1, 8, 2, 128, 1, 300, [299], 64, 4, torch.float16, "model", True),            # last row of the cache
    (1, 8, 2, 128, 1, 300, [0], 64, 4, torch.float16, "model", True),              # one row in it
    (3, 8, 8, 64, 1, 200, [0, 199, 77], 1, 0, torch.float16, "dense", True),       # a window of the token itself
    (4, 4, 4, 64, 1, 150, [-1, 149, 3, 64], 33, 37, torch.bfloat16, "model", True),  # an idle sequence, sinks past the window
    (2, 14, 2, 128, 1, 260, [130], 100, 1, torch.bfloat16, "packed", True),        # shared position, groups of seven, odd strides
    (2, 32, 2, 128, 1, 500, [499, 20], 200, 16, torch.float16, "model", False),    # sixteen heads a group
    (2, 64, 2, 64, 1, 500, [480, 20], 200, 16, torch.float16, "model", True),      # thirty-two: the row-tile kernel
    (1, 8, 1, 256, 1, 700, [650], 300, 100, torch.float16, "model", True),
    (1, 4, 2, 256, 3, 300, [200], 64, 2, torch.bfloat16, "packed", True),
    (2, 8, 2, 128, 4, 300, [10, 290], 7, 3, torch.float16, "model", True),         # a window shorter than two chunks
    (1, 8, 2, 128, 130, 400, [201], 90, 5, torch.float16, "model", True),          # chunk longer than the window
    (3, 14, 2, 64, 77, 700, [-1, 600, 0], 333, 5, torch.bfloat16, "packed", True),
    (1, 12, 4, 256, 70, 300, [100], 64, 70, torch.float16, "dense", False),
    (2, 8, 8, 128, 65, 900, [830, 400], 4000, 0, torch.float16, "model", True),    # a window past the cache: plain causal attention
    (1, 40, 2, 128, 9, 333, [300], 50, 20, torch.float16, "model", True),          # twenty heads a group
    (2, 8, 1, 128, 33, 3000, [2900, 1300], 2000, 129, torch.bfloat16, "packed", True),
    (1, 24, 1, 64, 300, 900, [599], 128, 1, torch.float16, "dense", True),
    (2, 4, 1, 128, 200, 400, [0, 200], 1, 0, torch.float16, "model", False),
]


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,window,sinks,dtype,layout,write", SHAPES)
def test_window(b, h, kv_h, d, n, s, pos, window, sinks, dtype, layout, write):
    c = Case(b, h, kv_h, d, n, s, pos, dtype, layout=layout)
    k, v, k64, v64 = c.caches(write, window, sinks)
    k0, v0 = k.clone(), v.clone()
    out = OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(), k, v, window, sinks, -1.0, write)
    ref, _, mag, _ = R.attention(c.q64, k64, v64, pos, window=window, sinks=sinks)
    assert out.shape == c.q.shape and out.dtype == dtype
    check(out, ref, mag, dtype)
    c.check_written(k0, k, c.nk64, write)
    c.check_written(v0, v, c.nv64, write)
    assert ops.span_status() == 0


@pytest.mark.parametrize("n", [1, 3, 40])
def test_positions_that_do_not_fit(n):
    """pos + n > S: flagged, output zeros, cache untouched; the neighbours are served."""
    s = 128
    c = Case(3, 8, 2, 128, n, s, [s - n + 1, s - n, 5])
    k, v, k64, v64 = c.caches(True, 50, 3)
    k0 = k.clone()
    assert ops.span_status() == 0
    out = OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(torch.int64), k, v, 50, 3)
    assert ops.span_status() == 1 and ops.span_status() == 0
    ref, _, mag, _ = R.attention(c.q64, k64, v64, c.pos, window=50, sinks=3)
    check(out, ref, mag, torch.float16)
    assert not out[0].any()
    c.check_written(k0, k, c.nk64, True)


@pytest.mark.parametrize("scale", [0.3, 1.0])
def test_window_scale_and_wide_scores(scale):
    """Scores up to +-200: the running maximum moves many times, most probabilities vanish."""
    c = Case(2, 8, 2, 64, 2, 300, [290, 100], q_scale=6.0)
    k, v, k64, v64 = c.caches(True, 120, 4)
    out = OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(), k, v, 120, 4, scale)
    ref, _, mag, big = R.attention(c.q64, k64, v64, c.pos, window=120, sinks=4, scale=scale)
    got = out.double().cpu()
    # the scores' own 32 bits count here: D roundings of sum |q k|, twice
    assert ((got - ref).abs() <= R.out_bound(ref, mag, torch.float16) + 2 * 64 * 2.0 ** -24 * big * mag).all()


def test_bf16_queries_beyond_fp16():
    """bf16 queries of 2^20 and of 2^-30: fp16 holds neither as it stands."""
    for factor, scale in ((2.0 ** 20, 2.0 ** -23), (2.0 ** -30, 2.0 ** 27)):
        c = Case(1, 8, 2, 128, 1, 200, [180], torch.bfloat16)
        c.q, c.q64 = c.q * factor, c.q64 * factor
        k, v, k64, v64 = c.caches(True, 100, 4)
        out = OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(), k, v, 100, 4, scale)
        ref, _, mag, _ = R.attention(c.q64, k64, v64, c.pos, window=100, sinks=4, scale=scale)
        check(out, ref, mag, torch.bfloat16)


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,p,dtype,layout,write", [
    (1, 8, 2, 128, 1, 64, [0], 1, torch.float16, "model", True),                   # one prefix row
    (3, 8, 2, 128, 1, 64, [0, 63, 20], 200, torch.float16, "model", True),
    (3, 8, 2, 128, 1, 64, [0, 63, 20], 0, torch.float16, "model", True),           # no prefix
    (4, 12, 4, 64, 3, 90, [-1, 80, 0, 33], 531, torch.bfloat16, "packed", True),   # an idle sequence
    (20, 8, 2, 128, 1, 40, list(range(20)), 129, torch.float16, "dense", False),   # two row tiles
    (2, 16, 2, 256, 1, 300, [250, 3], 77, torch.float16, "model", True),
    (2, 8, 1, 256, 5, 64, [50, 3], 700, torch.bfloat16, "model", True),            # 40 rows of a sequence
    (5, 14, 2, 64, 11, 64, [50, 3, 0, -1, 53], 64, torch.float16, "model", True),
    (70, 8, 2, 128, 1, 32, [i % 32 for i in range(70)], 300, torch.float16, "model", True),      # 280 rows a KV head: tensor memory
    (33, 16, 2, 64, 2, 24, [i % 23 - 1 for i in range(33)], 1025, torch.bfloat16, "packed", True),
    (24, 8, 1, 128, 1, 16, [3], 1, torch.float16, "model", True),
    (2, 8, 1, 128, 60, 80, [20, -1], 130, torch.float16, "model", True),                         # the own keys there too
])
def test_shared_prefix(b, h, kv_h, d, n, s, pos, p, dtype, layout, write):
    c = Case(b, h, kv_h, d, n, s, pos, dtype, layout=layout, prefix=max(p, 1))
    k, v, k64, v64 = c.caches(write)
    k0, v0 = k.clone(), v.clone()
    store = [torch.full((kv_h, p + 9, d), BAD, dtype=torch.float16, device=DEV) for _ in range(2)]
    for t, src in zip(store, (c.pk, c.pv)):
        t[:, :p] = src[:, :p].to(DEV)
    out = OPS.attention_shared_prefix(c.q, c.nk, c.nv, c.pos_t(), store[0][:, :p], store[1][:, :p], k, v, -1.0, write)
    ref, _, mag, _ = R.attention(c.q64, k64, v64, pos, prefix=(c.pk[:, :p].double(), c.pv[:, :p].double()))
    check(out, ref, mag, dtype)
    c.check_written(k0, k, c.nk64, write)
    c.check_written(v0, v, c.nv64, write)


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,dtype,layout,write", [
    (1, 8, 2, 128, 1, 301, [300], torch.float16, "model", True),
    (1, 8, 2, 128, 1, 301, [0], torch.float16, "model", True),
    (4, 14, 2, 64, 1, 1111, [-1, 1110, 5, 640], torch.bfloat16, "packed", True),
    (2, 32, 2, 128, 1, 700, [699, 20], torch.float16, "dense", False),
    (2, 8, 1, 256, 2, 90, [80, 3], torch.float16, "model", True),
    (2, 8, 2, 128, 13, 700, [687, 5], torch.float16, "model", True),               # 52 rows
    (1, 16, 1, 64, 20, 1300, [1200], torch.float16, "model", True),                # 320 rows
    (1, 12, 4, 256, 30, 130, [77], torch.bfloat16, "packed", False),
])
def test_scored(b, h, kv_h, d, n, s, pos, dtype, layout, write):
    c = Case(b, h, kv_h, d, n, s, pos, dtype, layout=layout)
    k, v, k64, v64 = c.caches(write)
    w0 = torch.rand(b, kv_h, s, generator=torch.Generator().manual_seed(1)) * 3
    for i in range(b):
        if c.place(i) is not None:
            w0[i, :, c.place(i):c.place(i) + n] = BAD                              # rows of tokens long gone
    w = w0.to(DEV)
    k0 = k.clone()
    out = OPS.attention_cache_scored(c.q, c.nk, c.nv, c.pos_t(), k, v, w, -1.0, write)
    ref, add, mag, big = R.attention(c.q64, k64, v64, pos)
    check(out, ref, mag, dtype)
    c.check_written(k0, k, c.nk64, write)
    got = w.cpu()
    for i in range(b):
        p = c.place(i)
        if p is None:
            assert torch.equal(got[i], w0[i])
            continue
        assert torch.equal(got[i, :, p + n:], w0[i, :, p + n:])
        want = add[i].clone()
        want[:, :p] += w0[i, :, :p].double()
        off = (got[i, :, :p + n].double() - want[:, :p + n]).abs()
        # one rounding of the sum on top of the probabilities' errors
        assert (off <= R.weight_bound(add[i][:, :p + n], big, d) + want[:, :p + n] * 2.0 ** -23).all()


# calls large enough for the 5th-generation tensor cores (192 rows of a KV head, 4e9 operations)
@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,window,sinks,dtype,layout,write", [
    (1, 8, 1, 128, 700, 6000, [5100], 4000, 129, torch.float16, "model", True),
    (1, 8, 1, 128, 700, 6000, [5300], 4000, 0, torch.float16, "model", False),     # to the cache's last row
    (4, 24, 2, 64, 500, 5000, [4000, -1, 0, 777], 3500, 5, torch.bfloat16, "packed", True),
    (2, 14, 2, 128, 1111, 1500, [389, 3], 9999, 7, torch.float16, "dense", True),   # causal, odd rows
    (2, 32, 2, 64, 777, 4000, [3000, 100], 2000, 3000, torch.float16, "model", True),   # more sinks than window
    (1, 64, 8, 128, 30, 20000, [19000], 16000, 64, torch.bfloat16, "model", True),  # few tiles: the keys are split
])
def test_window_long(b, h, kv_h, d, n, s, pos, window, sinks, dtype, layout, write):
    c = Case(b, h, kv_h, d, n, s, pos, dtype, layout=layout)
    k, v, k64, v64 = c.caches(write, window, sinks)
    k0, v0 = k.clone(), v.clone()
    out = OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(), k, v, window, sinks, -1.0, write)
    ref, mag = R.attention_wide(c.q64.to(DEV), k64.to(DEV), v64.to(DEV), pos, window=window, sinks=sinks)
    check(out, ref.cpu(), mag.cpu(), dtype)
    c.check_written(k0, k, c.nk64, write)
    c.check_written(v0, v, c.nv64, write)


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,p,dtype", [
    (70, 8, 2, 128, 1, 32, [i % 32 for i in range(70)], 14001, torch.float16),
    (33, 32, 2, 64, 2, 24, [i % 23 - 1 for i in range(33)], 8100, torch.bfloat16),
    (40, 64, 8, 128, 1, 3000, [i * 75 for i in range(40)], 3333, torch.float16),
    (2, 32, 1, 128, 100, 900, [800, -1], 5000, torch.float16),                     # a chunk each, few sequences
    (3, 64, 2, 64, 60, 9000, [8940, 10, 5000], 7000, torch.float16),               # the own keys too
])
def test_shared_prefix_long(b, h, kv_h, d, n, s, pos, p, dtype):
    c = Case(b, h, kv_h, d, n, s, pos, dtype, prefix=p)
    k, v, k64, v64 = c.caches(True)
    k0 = k.clone()
    store = [torch.full((kv_h, p + 8, d), BAD, dtype=torch.float16, device=DEV) for _ in range(2)]
    for t, src in zip(store, (c.pk, c.pv)):
        t[:, :p] = src.to(DEV)
    out = OPS.attention_shared_prefix(c.q, c.nk, c.nv, c.pos_t(), store[0][:, :p], store[1][:, :p], k, v)
    ref, mag = R.attention_wide(c.q64.to(DEV), k64.to(DEV), v64.to(DEV), pos, prefix=(c.pk.double().to(DEV), c.pv.double().to(DEV)))
    check(out, ref.cpu(), mag.cpu(), dtype)
    c.check_written(k0, k, c.nk64, True)


# calls past what clusters take: more (sequence, KV head)s than CTAs run at once, or long sequences
STREAMED = [
    # b, h, kv_h, d, n, s, pos, window, sinks, dtype, layout, write
    (40, 16, 8, 128, 1, 300, [(i * 37) % 300 if i % 9 else -1 for i in range(40)], 100, 4, torch.float16, "model", True),
    (60, 16, 8, 64, 2, 200, [(i * 31) % 199 if i % 7 else -1 for i in range(60)], 70, 20, torch.bfloat16, "packed", True),
    (20, 24, 8, 256, 1, 150, [(i * 17) % 150 for i in range(20)], 64, 1, torch.float16, "dense", False),
    (40, 8, 8, 128, 5, 128, [123 - i for i in range(40)], 300, 0, torch.float16, "model", True),
    (300, 2, 1, 64, 1, 40, [i % 41 - 1 for i in range(300)], 11, 2, torch.float16, "model", True),
    (1, 8, 2, 128, 1, 20000, [19999], 12000, 70, torch.float16, "model", True),
    (2, 14, 2, 64, 2, 33000, [32998, 5], 32000, 0, torch.bfloat16, "packed", True),
    (1, 16, 1, 256, 1, 9000, [8800], 8700, 3, torch.float16, "model", False),
    (3, 3, 3, 128, 1, 30000, [29990, 0, 17], 40000, 0, torch.float16, "model", True),
]


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,window,sinks,dtype,layout,write", STREAMED)
def test_window_streamed(b, h, kv_h, d, n, s, pos, window, sinks, dtype, layout, write):
    c = Case(b, h, kv_h, d, n, s, pos, dtype, layout=layout)
    k, v, k64, v64 = c.caches(write, window, sinks)
    k0, v0 = k.clone(), v.clone()
    out = OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(), k, v, window, sinks, -1.0, write)
    ref, mag = R.attention_wide(c.q64.to(DEV), k64.to(DEV), v64.to(DEV), pos, window=window, sinks=sinks)
    check(out, ref.cpu(), mag.cpu(), dtype)
    c.check_written(k0, k, c.nk64, write)
    c.check_written(v0, v, c.nv64, write)
    assert ops.span_status() == 0


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,window,sinks,dtype,layout,write", STREAMED)
def test_scored_streamed(b, h, kv_h, d, n, s, pos, window, sinks, dtype, layout, write):
    c = Case(b, h, kv_h, d, n, s, pos, dtype, layout=layout)
    k, v, k64, v64 = c.caches(write)
    w = torch.rand(b, kv_h, s, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = w.double()
    for i in range(b):
        if c.place(i) is not None:
            w[i, :, c.place(i):c.place(i) + n] = BAD
            want[i, :, c.place(i):c.place(i) + n] = 0.0
    before, add = want.clone(), torch.zeros_like(want)
    out = OPS.attention_cache_scored(c.q, c.nk, c.nv, c.pos_t(), k, v, w, -1.0, write)
    ref, mag = R.attention_wide(c.q64.to(DEV), k64.to(DEV), v64.to(DEV), pos, weights=add)
    check(out, ref.cpu(), mag.cpu(), dtype)
    big = float((c.q64.abs().amax() * c.k.abs().amax()) * d ** 0.5)            # above every scale * sum |q k|
    off = (w.double() - before - add).abs()
    assert (off <= R.weight_bound(add, big, d) + (before + add) * 2.0 ** -23).all()


def evict_case(b, kv_h, s, s_out, d, lengths, kind="random", seed=0):
    g = torch.Generator().manual_seed(seed + s)
    k, v = torch.randn(b, kv_h, s, d, generator=g).half(), torch.randn(b, kv_h, s, d, generator=g).half()
    w = torch.randn(b, kv_h, s, generator=g).mul(2).exp()
    if kind == "ties":
        w = torch.randint(0, 3, (b, kv_h, s), generator=g).float()
    elif kind == "equal":
        w = torch.full((b, kv_h, s), 0.25)
    elif kind == "odd":
        w = torch.randn(b, kv_h, s, generator=g)
        pick = torch.randint(0, 8, (b, kv_h, s), generator=g)
        for code, x in enumerate((0.0, -0.0, float("inf"), float("-inf"), BAD)):
            w[pick == code] = x
    for i, n in enumerate(lengths):
        k[i, :, n:], v[i, :, n:], w[i, :, n:] = BAD, BAD, 1e30       # what lies behind a sequence decides nothing
    return k, v, w


def evict_against_definition(b, kv_h, s, d, lengths, keep, sinks, recent, kind, in_place):
    k, v, w = evict_case(b, kv_h, s, keep, d, lengths, kind)
    kd, vd, wd = k.to(DEV), v.to(DEV), w.to(DEV)
    if in_place:
        ko, vo, wo = kd, vd, wd
    else:
        room = keep + 3
        ko, vo = (torch.full((b, kv_h, room, d), 7.0, dtype=torch.float16, device=DEV) for _ in range(2))
        wo = torch.full((b, kv_h, room), 7.0, device=DEV)
    sent, lengths = lengths, [n if 0 <= n <= s else 0 for n in lengths]                # out of range counts as 0, and is told
    before = [t.cpu().clone() for t in (ko, vo, wo)]
    kept, new = OPS.kv_evict(kd, vd, wd, torch.tensor(sent, dtype=torch.int32, device=DEV), ko, vo, wo, keep, sinks, recent)
    assert new.tolist() == [min(n, keep) for n in lengths]
    kept = kept.cpu()
    for i in range(b):
        for h in range(kv_h):
            rows = R.evict(w[i, h].tolist(), lengths[i], keep, sinks, recent)
            assert kept[i, h].tolist() == rows + [-1] * (keep - len(rows))
            for src, was in zip((k, v, w), before):
                was[i, h, :len(rows)] = src[i, h, rows]
    for t, want in zip((ko, vo, wo), before):
        ints = torch.int16 if t.dtype == torch.float16 else torch.int32
        assert torch.equal(t.cpu().view(ints), want.view(ints))
    if not in_place:
        assert torch.equal(kd.cpu().view(torch.int16), k.view(torch.int16))
    assert ops.span_status() == (0 if sent == lengths else 2)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("b,kv_h,s,d,lengths,keep,sinks,recent,kind", [
    (1, 2, 300, 128, [300], 100, 4, 20, "random"),
    (3, 2, 300, 64, [0, 99, 100], 100, 4, 20, "random"),               # nothing to evict
    (3, 1, 2000, 64, [101, 1999, 1], 100, 0, 0, "random"),
    (2, 2, 5000, 128, [4999, 2500], 2100, 4, 1000, "random"),
    (2, 2, 700, 256, [700, 650], 64, 64, 0, "random"),                 # sinks alone
    (2, 2, 700, 64, [700, 650], 64, 10, 54, "random"),                 # nothing is decided by weight
    (2, 3, 1500, 64, [1500, 1490], 777, 3, 5, "ties"),
    (1, 2, 1500, 64, [1400], 333, 1, 1, "equal"),
    (2, 2, 1500, 128, [1500, 1200], 600, 2, 3, "odd"),
    (1, 1, 1, 64, [1], 1, 0, 0, "random"),
    (1, 2, 12000, 64, [11999], 5000, 3, 700, "random"),
    (2, 1, 30000, 64, [30000, 29000], 7001, 4, 100, "odd"),
    (1, 1, 32768, 64, [32768], 32767, 0, 0, "equal"),
    (1, 1, 40000, 64, [40000], 39999, 0, 0, "ties"),
    (1, 1, 70000, 64, [69999], 100, 10, 20, "odd"),
])
def test_evict(b, kv_h, s, d, lengths, keep, sinks, recent, kind, in_place):
    evict_against_definition(b, kv_h, s, d, lengths, keep, sinks, recent, kind, in_place)


@pytest.mark.parametrize("b,kv_h,s,d,lengths,keep,sinks,recent", [
    (2, 2, 900, 128, [900, 640], 640, 0, 640),                         # nothing is decided by weight, all of it recent
    (2, 2, 900, 128, [900, 650], 641, 1, 640),
    (3, 2, 900, 128, [900, 300, 0], 512, 130, 320),                    # sinks past a CTA's rows; nothing to evict; no rows
    (2, 1, 1100, 64, [1100, 701], 700, 5, 300),
    (2, 1, 500, 256, [500, 431], 430, 33, 97),
    (5, 4, 3000, 128, [3000, 2048, 2049, 1, 2700], 2048, 4, 1500),
])
def test_evict_many_recent_rows(b, kv_h, s, d, lengths, keep, sinks, recent):
    evict_against_definition(b, kv_h, s, d, lengths, keep, sinks, recent, "random", False)
    evict_against_definition(b, kv_h, s, d, lengths, keep, sinks, recent, "ties", False)


@pytest.mark.parametrize("b,kv_h,s,d,lengths,keep,sinks,recent,kind", [
    (10, 8, 900, 128, [900 - 7 * i for i in range(10)], 640, 1, 320, "random"),        # more items than half the SMs: two launches
    (80, 1, 700, 64, [9 * i for i in range(80)], 300, 140, 150, "ties"),
    (19, 4, 400, 256, [400 - i for i in range(19)], 200, 0, 200, "odd"),
    (37, 2, 600, 128, [600] * 36 + [0], 130, 3, 0, "odd"),                             # half of them: two CTAs an item
    (1, 75, 9000, 64, [8999], 700, 5, 129, "equal"),
    (1, 1, 20000, 128, [19999], 147, 4, 30, "random"),                                 # a row a CTA, and none for the last
    (3, 1, 500, 256, [500, 3, 40], 2, 1, 1, "random"),
])
def test_evict_by_items(b, kv_h, s, d, lengths, keep, sinks, recent, kind):
    evict_against_definition(b, kv_h, s, d, lengths, keep, sinks, recent, kind, False)
    evict_against_definition(b, kv_h, s, d, lengths, keep, sinks, recent, kind, True)


def test_evict_length_out_of_range():
    k, v, w = (t.to(DEV) for t in evict_case(2, 1, 50, 20, 64, [50, 50]))
    k0 = k.clone()
    for bad in (51, -3):
        kept, new = OPS.kv_evict(k, v, w, torch.tensor([bad, 20], device=DEV), k, v, w, 20)
        assert ops.span_status() == 2 and new.tolist() == [0, 20] and (kept[0] == -1).all() and torch.equal(k, k0)


def test_weights_decide_what_stays_and_decoding_goes_on():
    """A prompt in two chunks under a window, its last tokens' weights, eviction, and decode steps over what is left: each step against the
    definition over the rows that stayed."""
    b, h, kv_h, d, s, room = 2, 8, 2, 128, 400, 160
    g = torch.Generator().manual_seed(5)
    q, nk, nv = (torch.randn(b, 330, x, d, generator=g).half().to(DEV).transpose(1, 2) for x in (h, kv_h, kv_h))
    k, v = (torch.zeros(b, kv_h, s, d, dtype=torch.float16, device=DEV) for _ in range(2))
    w = torch.zeros(b, kv_h, s, device=DEV)
    pos = lambda *p: torch.tensor(p, dtype=torch.int32, device=DEV)  # noqa: E731
    for a, z in ((0, 200), (200, 280)):
        out = OPS.attention_cache_window(q[:, :, a:z], nk[:, :, a:z], nv[:, :, a:z], pos(a), k, v, 90, 4)
        ref, _, mag, _ = R.attention(q[:, :, a:z].double().cpu(), nk.double().cpu(), nv.double().cpu(), [a], window=90, sinks=4)
        check(out, ref, mag, torch.float16, f"chunk {a}")
    OPS.attention_cache_scored(q[:, :, 280:300], nk[:, :, 280:300], nv[:, :, 280:300], pos(280), k, v, w)
    k2, v2 = (torch.zeros(b, kv_h, room, d, dtype=torch.float16, device=DEV) for _ in range(2))
    w2 = torch.zeros(b, kv_h, room, device=DEV)
    kept, length = OPS.kv_evict(k, v, w, pos(300, 300), k2, v2, w2, 120, 4, 30)
    rows = torch.gather(nk[:, :, :300], 2, kept.long()[..., None].expand(-1, -1, -1, d))
    assert torch.equal(k2[:, :, :120], rows) and torch.equal(w2[:, :, :120], torch.gather(w, 2, kept.long()))
    for step in range(3):
        a = 300 + step
        out = OPS.attention_cache_scored(q[:, :, a:a + 1], nk[:, :, a:a + 1], nv[:, :, a:a + 1], length, k2, v2, w2)
        ref, _, mag, _ = R.attention(q[:, :, a:a + 1].double().cpu(), k2.double().cpu(), v2.double().cpu(), length.tolist())
        check(out, ref, mag, torch.float16, f"step {step}")
        length = length + 1
    # the prompt's rows as a prefix of two new answers
    k3, v3 = (torch.zeros(b, kv_h, 32, d, dtype=torch.float16, device=DEV) for _ in range(2))
    for step in range(2):
        a = 310 + step
        out = OPS.attention_shared_prefix(q[:, :, a:a + 1], nk[:, :, a:a + 1], nv[:, :, a:a + 1], pos(step), k[0, :, :280], v[0, :, :280], k3, v3)
        ref, _, mag, _ = R.attention(q[:, :, a:a + 1].double().cpu(), k3.double().cpu(), v3.double().cpu(), [step],
                                     prefix=(k[0, :, :280].double().cpu(), v[0, :, :280].double().cpu()))
        check(out, ref, mag, torch.float16, f"answer {step}")


def test_captured_and_replayed_with_moving_positions():
    """One graph of all four ops; positions move between replays; a second graph of the same shapes replays on another stream meanwhile."""
    b, h, kv_h, d, s = 2, 8, 2, 128, 256

    def build(seed):
        c = Case(b, h, kv_h, d, 1, s, [100, 60], seed=seed, prefix=70)
        st = {"c": c, "pos": c.pos_t(), "w": torch.zeros(b, kv_h, s, device=DEV), "pk": c.pk.to(DEV), "pv": c.pv.to(DEV),
              "k": c.k.to(DEV), "v": c.v.to(DEV), "wo": torch.zeros(b, kv_h, 64, device=DEV)}
        st["ko"], st["vo"] = (torch.zeros(b, kv_h, 64, d, dtype=torch.float16, device=DEV) for _ in range(2))

        def step():
            a = OPS.attention_cache_window(c.q, c.nk, c.nv, st["pos"], st["k"], st["v"], 50, 4)
            p = OPS.attention_shared_prefix(c.q, c.nk, c.nv, st["pos"], st["pk"], st["pv"], st["k"], st["v"])
            o = OPS.attention_cache_scored(c.q, c.nk, c.nv, st["pos"], st["k"], st["v"], st["w"])
            e = OPS.kv_evict(st["k"], st["v"], st["w"], st["pos"], st["ko"], st["vo"], st["wo"], 64, 4, 8)
            return (a, p, o, *e, st["ko"], st["vo"], st["wo"])
        return st, step

    graphs = []
    for seed in (1, 2):
        st, step = build(seed)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((st, step, graph, outs, torch.cuda.Stream()))
    for pos in ([100, 60], [-1, 255], [0, 254], [200, 201]):
        for st, *_ in graphs:
            st["pos"].copy_(torch.tensor(pos, dtype=torch.int32))
            st["w"].zero_()
        torch.cuda.synchronize()
        for _, _, graph, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in outs] for _, _, _, outs, _ in graphs]
        for (st, step, *_), mine in zip(graphs, got):
            st["w"].zero_()
            want = step()
            for x, y in zip(mine, want):
                assert torch.equal(x, y)
        assert ops.span_status() == (2 if -1 in pos else 0)          # (-1 is an idle sequence's position, but no length)


def test_calls_in_a_row():
    """Launches begin under the ones before them: calls whose workspaces, caches and outputs follow one another without a pause give the
    bits that each gives alone."""
    p = 14001
    prefix = [Case(70, 8, 2, 128, 1, 32, [(i * 5 + j) % 32 for i in range(70)], prefix=p, seed=j) for j in range(2)]
    shared = [[t.to(DEV) for t in (c.pk, c.pv)] for c in prefix]
    chunk = Case(1, 8, 1, 128, 700, 6000, [5100])
    step = Case(40, 16, 8, 128, 1, 300, [(i * 37) % 300 for i in range(40)])
    weights = torch.rand(40, 8, 300, generator=torch.Generator().manual_seed(3)).to(DEV)
    lengths = torch.tensor([260 + i for i in range(40)], dtype=torch.int32, device=DEV)

    def behind(j):
        k, v, _, _ = prefix[j].caches(True)
        c = prefix[j]
        return lambda: (OPS.attention_shared_prefix(c.q, c.nk, c.nv, pos[j], *shared[j], kc := k.clone(), vc := v.clone()), kc, vc)

    def window():
        k, v, _, _ = chunk.caches(True)
        at = chunk.pos_t()
        return lambda: (OPS.attention_cache_window(chunk.q, chunk.nk, chunk.nv, at, kc := k.clone(), vc := v.clone(), 4000, 129), kc, vc)

    def scored_and_evicted():
        k, v = (x.to(DEV) for x in (step.k, step.v))
        at = step.pos_t()

        def run():
            kc, vc, w = k.clone(), v.clone(), weights.clone()
            out = OPS.attention_cache_scored(step.q, step.nk, step.nv, at, kc, vc, w)
            ko, vo, wo = (torch.zeros_like(x[:, :, :200]) for x in (kc, vc, w))
            return out, w, ko, vo, wo, *OPS.kv_evict(kc, vc, w, lengths, ko, vo, wo, 200, 4, 150)
        return run

    pos = [c.pos_t() for c in prefix]
    calls = [behind(0), window(), behind(1), scored_and_evicted()]
    alone = []
    for f in calls:
        torch.cuda.synchronize()
        alone.append([t.clone() for t in f()])
        torch.cuda.synchronize()
    rounds = [[f() for f in calls] for _ in range(4)]
    torch.cuda.synchronize()
    for got in rounds:
        for a, z in zip(alone, got):
            for x, y in zip(a, z):
                bits = torch.int16 if x.element_size() == 2 else torch.int32
                assert torch.equal(x.view(bits), y.view(bits))


def test_two_threads_on_one_stream():
    """Launches of two threads' calls may alternate on the stream that they share; each call still gives its own bits."""
    p = 14001
    behind = Case(70, 8, 2, 128, 1, 32, [(i * 5) % 32 for i in range(70)], prefix=p)
    pk, pv = behind.pk.to(DEV), behind.pv.to(DEV)
    step = Case(40, 16, 8, 128, 1, 300, [(i * 37) % 300 for i in range(40)])
    chunk = Case(2, 32, 8, 64, 12, 900, [700, 880])
    weights = {c: torch.rand(c.b, c.kv_h, c.s, generator=torch.Generator().manual_seed(3)).to(DEV) for c in (step, chunk)}
    caches = {c: [x.to(DEV) for x in (c.k, c.v)] for c in (behind, step, chunk)}
    pos = {c: c.pos_t() for c in caches}
    threads, rounds = 2, 60

    def prefix():
        return (OPS.attention_shared_prefix(behind.q, behind.nk, behind.nv, pos[behind], pk, pv, *caches[behind], -1.0, False),)

    def scored(c):
        w = weights[c].clone()
        return OPS.attention_cache_scored(c.q, c.nk, c.nv, pos[c], *caches[c], w, -1.0, False), w

    calls = [prefix, lambda: scored(step), lambda: scored(chunk)]
    alone = []
    for f in calls:
        torch.cuda.synchronize()
        alone.append([t.clone() for t in f()])
        torch.cuda.synchronize()
    got, failed, start = [[] for _ in range(threads)], [], threading.Barrier(threads)

    def work(i):
        try:
            start.wait()
            for n in range(rounds):
                k = (n + i) % len(calls)
                got[i].append((k, calls[k]()))
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    pool = [threading.Thread(target=work, args=(i,)) for i in range(threads)]
    for t in pool:
        t.start()
    for t in pool:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for k, results in (x for g in got for x in g):
        for x, y in zip(alone[k], results):
            bits = torch.int16 if x.element_size() == 2 else torch.int32
            assert torch.equal(x.view(bits), y.view(bits))


def test_same_bits_again_and_on_another_stream():
    c = Case(3, 32, 8, 128, 1, 3000, [2999, 1500, 7])
    k, v, _, _ = c.caches(True)
    w = torch.zeros(3, 8, 3000, device=DEV)
    first = OPS.attention_cache_scored(c.q, c.nk, c.nv, c.pos_t(), k, v, w)
    torch.cuda.synchronize()
    for _ in range(3):
        w2 = torch.zeros_like(w)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = OPS.attention_cache_scored(c.q, c.nk, c.nv, c.pos_t(), k, v, w2)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(first, again) and torch.equal(w, w2)


def test_prefix_layouts():
    """One head's rows for all KV heads (a stride of zero), rows with gaps, K and V of different strides: as the dense prefix."""
    c = Case(3, 8, 2, 128, 1, 64, [5, 20, 63], prefix=90)
    one_k, one_v = c.pk[:1].to(DEV), c.pv[:1].to(DEV)
    gaps = torch.zeros(2, 180, 128, dtype=torch.float16, device=DEV)[:, ::2]
    gaps.copy_(one_v.expand(2, -1, -1))
    outs = []
    for pk, pv in ((one_k.repeat(2, 1, 1), one_v.repeat(2, 1, 1)), (one_k.expand(2, -1, -1), one_v.expand(2, -1, -1)), (one_k.repeat(2, 1, 1), gaps)):
        k, v, _, _ = c.caches(True)
        outs.append(OPS.attention_shared_prefix(c.q, c.nk, c.nv, c.pos_t(), pk, pv, k, v))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_nothing_to_do():
    c = Case(2, 8, 2, 64, 1, 64, [10])
    k, v, _, _ = c.caches(True)
    empty = OPS.attention_cache_window(c.q[:, :, :0], c.nk[:, :, :0], c.nv[:, :, :0], c.pos_t(), k, v, 8)
    assert empty.shape == (2, 8, 0, 64)
    none = OPS.attention_cache_window(c.q[:0], c.nk[:0], c.nv[:0], c.pos_t(), k, v, 8)
    assert none.shape == (0, 8, 1, 64)


def test_refusals():
    c = Case(2, 8, 2, 64, 1, 64, [10, 11])
    k, v, _, _ = c.caches(True)
    w, pos = torch.zeros(2, 2, 64, device=DEV), c.pos_t()
    pk = torch.zeros(2, 16, 64, dtype=torch.float16, device=DEV)
    call = OPS.attention_cache_window
    with pytest.raises(ValueError, match="window"):
        call(c.q, c.nk, c.nv, pos, k, v, 0)
    with pytest.raises(ValueError, match="sinks"):
        call(c.q, c.nk, c.nv, pos, k, v, 4, -1)
    with pytest.raises(TypeError, match="q must be"):
        call(c.q.float(), c.nk, c.nv, pos, k, v, 4)
    with pytest.raises(TypeError, match="new_k"):
        call(c.q, c.nk.float(), c.nv, pos, k, v, 4)
    with pytest.raises(ValueError, match="cache"):
        call(c.q, c.nk, c.nv, pos, k[:, :, ::2], v[:, :, ::2], 4)
    with pytest.raises(ValueError, match="cache"):
        call(c.q, c.nk, c.nv, pos, k[:1], v[:1], 4)
    with pytest.raises(ValueError, match="positions"):
        call(c.q, c.nk, c.nv, torch.zeros(3, dtype=torch.int32, device=DEV), k, v, 4)
    with pytest.raises(ValueError, match="tensors must be on"):
        call(c.q, c.nk, c.nv, pos.cpu(), k, v, 4)
    with pytest.raises(ValueError, match="group"):
        call(c.q[:, :7], c.nk, c.nv, pos, k, v, 4)
    with pytest.raises(NotImplementedError, match="head_dim"):
        call(c.q[..., :32], c.nk[..., :32], c.nv[..., :32], pos, k[..., :32], v[..., :32], 4)
    with pytest.raises(ValueError, match="prefix_k"):
        OPS.attention_shared_prefix(c.q, c.nk, c.nv, pos, pk[:1], pk[:1], k, v)
    with pytest.raises(ValueError, match="weights"):
        OPS.attention_cache_scored(c.q, c.nk, c.nv, pos, k, v, w[:, :, :60])
    with pytest.raises(TypeError, match="weights"):
        OPS.attention_cache_scored(c.q, c.nk, c.nv, pos, k, v, w.half())
    with pytest.raises(ValueError, match="keep"):
        OPS.kv_evict(k, v, w, pos, k, v, w, 65)
    with pytest.raises(ValueError, match="keep"):
        OPS.kv_evict(k, v, w, pos, k, v, w, 8, 5, 4)
    with pytest.raises(alloy_b200._lib.AlloyB200Error):                       # an output over another input
        OPS.kv_evict(k, v, w, pos, v, k, w, 8)


def test_offsets_beyond_32_bits():
    """A cache of more than 2^32 bytes per tensor: the last sequences' rows lie behind offset 2^31 elements."""
    b, h, kv_h, d, s = 3, 4, 1, 256, 1 << 22
    k, v = (torch.zeros(b, kv_h, s, d, dtype=torch.float16, device=DEV) for _ in range(2))
    c = Case(b, h, kv_h, d, 1, 64, [63, 63, 63])
    pos = [s - 1, s - 1, s - 1]
    for t, src in ((k, c.k), (v, c.v)):
        t[:, :, s - 64:] = src.to(DEV)
    out = OPS.attention_cache_window(c.q, c.nk, c.nv, torch.tensor(pos, dtype=torch.int32, device=DEV), k, v, 64)
    _, _, k64, v64 = c.caches(True)
    ref, _, mag, _ = R.attention(c.q64, k64, v64, c.pos)
    check(out, ref, mag, torch.float16)
    w = torch.zeros(b, kv_h, s, device=DEV)
    w[:, :, s - 100:s - 60] = 1.0
    ko, vo, wo = (torch.zeros(b, kv_h, 64, *x, dtype=t, device=DEV) for x, t in (((d,), torch.float16), ((d,), torch.float16), ((), torch.float32)))
    kept, _ = OPS.kv_evict(k, v, w, torch.tensor([s], dtype=torch.int32, device=DEV), ko, vo, wo, 64, 0, 60)
    assert kept[2, 0].tolist() == list(range(s - 100, s - 96)) + list(range(s - 60, s))
    assert torch.equal(ko, k[:, :, kept[0, 0].long()])
