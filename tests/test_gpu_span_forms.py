"""The forms of the attention ops over spans of an fp16 cache give the same accuracy: each against the definition in 64 bits."""

import pytest
import torch

import alloy_b200  # noqa: F401
from alloy_b200 import _lib, ops
from tests import _span_ref as R
from tests.test_gpu_span import DEV, OPS, Case

pytestmark = pytest.mark.gpu


def work(c, keys):
    """Operations of a call's products, by its sizes."""
    return 4 * c.d * c.h * c.n * c.b * keys


class Cancelling(Case):
    """Scores are single products, exact in fp32 but for the scale's rounding.  Keys come in pairs of nearly equal scores and opposite values, so that
    the outputs are small beside what is added up and show each probability's own rounding."""

    def __init__(self, *args, spread=4.0, **kw):
        super().__init__(*args, **kw)
        g = torch.Generator().manual_seed(self.s * 31 + self.n)

        def pairs(x, step):
            x = x.clone()
            rows = x.shape[-2] // 2 * 2
            first = (torch.rand(x.shape[0], x.shape[1], rows // 2, generator=g) * 2 - 1) * spread
            x[..., :] = 0.0
            x[:, :, 0:rows:2, 0] = first.half()
            x[:, :, 1:rows:2, 0] = x[:, :, 0:rows:2, 0] + step
            return x

        def opposite(x):
            rows = x.shape[-2] // 2 * 2
            x[:, :, 1:rows:2] = -x[:, :, 0:rows:2]
            return x

        q = torch.zeros(self.q64.shape)
        q[..., 0] = 1.0 + torch.rand(q.shape[:-1], generator=g).bfloat16().float() / 2
        q = q.to(self.dtype)
        self.q.copy_(q.to(DEV))
        self.q64 = q.double()
        self.k, self.v = pairs(self.k, 2.0 ** -6).half(), opposite(self.v)
        nk, nv = pairs(self.nk64, 2.0 ** -6).half(), opposite(self.nv64.half())
        self.nk.copy_(nk.to(DEV))
        self.nv.copy_(nv.to(DEV))
        self.nk64, self.nv64 = nk.double(), nv.double()
        if hasattr(self, "pk"):
            self.pk, self.pv = pairs(self.pk[None], 2.0 ** -6)[0].half(), opposite(self.pv[None])[0]


def check_fine(out, ref, mag, dtype):
    """A probability in two fp16 halves is off by 2^-22 of it, the exponential by 2^-22, a score of up to 2^5 in the log2 frame by 2^-19 x ln 2
    (its product with the scale and the maximum's subtraction, half a step of 2^-24 x 2^5 each), the sums by a few 2^-24: below 2^-18 in all.  The
    output is rounded once, in fp16 by half of 2^-24 at least.  Probabilities of 11 bits are off by up to 2^-12 each, and by 2^-14 x mag and more in the mean."""
    got = out.double().cpu()
    assert _lib.load().alloyb_device_error(1) == 0 and torch.isfinite(got).all()
    over = (got - ref).abs() - (2.0 ** -18 * mag + torch.finfo(dtype).eps / 2 * ref.abs() * (1 + 2.0 ** -8) + 2.0 ** -25)
    assert float(over.max()) <= 0, f"{float((got - ref).abs().max()):.3e} off, {float(over.max()):.3e} over"


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,window,sinks,dtype", [
    (1, 8, 2, 128, 1, 90, [80], 60, 4, torch.float16),                             # few rows
    (40, 16, 8, 128, 1, 300, [(i * 37) % 300 for i in range(40)], 100, 4, torch.float16),
    (2, 64, 2, 64, 1, 90, [80, 20], 70, 6, torch.float16),                         # row tiles
    (2, 8, 2, 128, 20, 90, [60, 10], 70, 6, torch.float16),
    (1, 8, 2, 128, 77, 200, [101], 64, 0, torch.bfloat16),
    (2, 8, 1, 256, 33, 90, [50, 3], 70, 2, torch.float16),
])
def test_window_keeps_the_probabilities(b, h, kv_h, d, n, s, pos, window, sinks, dtype):
    c = Cancelling(b, h, kv_h, d, n, s, pos, dtype)
    k, v, k64, v64 = c.caches(True)
    out = OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(), k, v, window, sinks, 1.0)
    ref, _, mag, _ = R.attention(c.q64, k64, v64, pos, window=window, sinks=sinks, scale=1.0)
    check_fine(out, ref, mag, dtype)


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,p,dtype", [
    (3, 8, 2, 128, 1, 64, [0, 62, 20], 60, torch.float16),
    (4, 12, 4, 64, 3, 90, [-1, 30, 0, 33], 51, torch.bfloat16),
    (2, 8, 2, 256, 7, 64, [50, 3], 40, torch.float16),
    (3, 16, 2, 64, 6, 64, [50, 3, 8], 70, torch.float16),
])
def test_prefix_keeps_the_probabilities(b, h, kv_h, d, n, s, pos, p, dtype):
    c = Cancelling(b, h, kv_h, d, n, s, pos, dtype, prefix=p)
    k, v, k64, v64 = c.caches(True)
    out = OPS.attention_shared_prefix(c.q, c.nk, c.nv, c.pos_t(), c.pk.to(DEV), c.pv.to(DEV), k, v, 1.0)
    ref, _, mag, _ = R.attention(c.q64, k64, v64, pos, prefix=(c.pk.double(), c.pv.double()), scale=1.0)
    check_fine(out, ref, mag, dtype)


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,dtype", [
    (2, 8, 2, 128, 1, 90, [80, 3], torch.float16),
    (2, 8, 2, 128, 13, 90, [70, 5], torch.float16),
    (1, 16, 1, 64, 20, 100, [60], torch.bfloat16),
    (1, 12, 4, 256, 30, 100, [66], torch.float16),
])
def test_scored_keeps_the_probabilities(b, h, kv_h, d, n, s, pos, dtype):
    c = Cancelling(b, h, kv_h, d, n, s, pos, dtype)
    k, v, k64, v64 = c.caches(True)
    w = torch.zeros(b, kv_h, s, device=DEV)
    out = OPS.attention_cache_scored(c.q, c.nk, c.nv, c.pos_t(), k, v, w, 1.0)
    ref, _, mag, _ = R.attention(c.q64, k64, v64, pos, scale=1.0)
    check_fine(out, ref, mag, dtype)


# from 5e9 operations of more than 16 rows a KV head on: the 5th-generation tensor cores, with head_dim 64 and 128
@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,window,sinks,dtype", [
    (1, 8, 1, 128, 700, 6000, [5100], 4000, 129, torch.float16),
    (4, 24, 2, 64, 500, 5000, [4000, -1, 0, 777], 3500, 5, torch.bfloat16),
    (1, 64, 8, 128, 30, 20000, [19000], 16000, 64, torch.float16),                 # few tiles: the keys are split
])
def test_long_window_keeps_the_probabilities(b, h, kv_h, d, n, s, pos, window, sinks, dtype):
    c = Cancelling(b, h, kv_h, d, n, s, pos, dtype, spread=8.0)
    assert work(c, min(s, window + sinks + n)) >= 5e9
    k, v, k64, v64 = c.caches(True)
    out = OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(), k, v, window, sinks, 1.0)
    ref, mag = R.attention_wide(c.q64.to(DEV) * d ** 0.5, k64.to(DEV), v64.to(DEV), pos, window=window, sinks=sinks)
    check_fine(out, ref.cpu(), mag.cpu(), dtype)


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,p,dtype", [
    (70, 8, 2, 128, 1, 32, [i % 32 for i in range(70)], 14001, torch.float16),
    (33, 32, 2, 64, 2, 24, [i % 23 - 1 for i in range(33)], 8100, torch.bfloat16),
    (2, 32, 1, 128, 100, 900, [800, -1], 5000, torch.float16),
])
def test_long_prefix_keeps_the_probabilities(b, h, kv_h, d, n, s, pos, p, dtype):
    c = Cancelling(b, h, kv_h, d, n, s, pos, dtype, prefix=p, spread=8.0)
    assert work(c, p) >= 1.5e9
    k, v, k64, v64 = c.caches(True)
    out = OPS.attention_shared_prefix(c.q, c.nk, c.nv, c.pos_t(), c.pk.to(DEV), c.pv.to(DEV), k, v, 1.0)
    ref, mag = R.attention_wide(c.q64.to(DEV) * d ** 0.5, k64.to(DEV), v64.to(DEV), pos, prefix=(c.pk.double().to(DEV), c.pv.double().to(DEV)))
    check_fine(out, ref.cpu(), mag.cpu(), dtype)
