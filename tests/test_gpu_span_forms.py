"""The forms of the attention ops over spans of an fp16 cache give the same accuracy: each against the definition in 64 bits."""

import threading

import pytest
import torch

import alloy_b200  # noqa: F401
from alloy_b200 import _lib, ops
from tests import _span_ref as R
from tests.test_gpu_span import DEV, OPS, Case

pytestmark = pytest.mark.gpu


def tensor_cores(c, keys, prefix=False):
    """Whether a call's sizes send its own keys, or the prefix's, to the 5th-generation tensor cores."""
    rows, pairs = c.n * c.h // c.kv_h, c.h * c.n * c.b * keys
    if prefix and rows <= 16:
        return c.d <= 128 and rows * c.b >= 32 and pairs >= 1.3e7
    return c.d <= 128 and (rows > 16 or prefix and rows * c.b >= 32) and 4 * c.d * pairs >= 2e9


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


# from 2e9 operations of more than 16 rows a KV head on (a prefix with fewer each: 1.3e7 pairs of a row and a key): the 5th-generation tensor cores, with
# head_dim 64 and 128
@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,window,sinks,dtype", [
    (1, 8, 1, 128, 700, 6000, [5100], 4000, 129, torch.float16),
    (4, 24, 2, 64, 500, 5000, [4000, -1, 0, 777], 3500, 5, torch.bfloat16),
    (1, 64, 8, 128, 30, 20000, [19000], 16000, 64, torch.float16),                 # few tiles: the keys are split
])
def test_long_window_keeps_the_probabilities(b, h, kv_h, d, n, s, pos, window, sinks, dtype):
    c = Cancelling(b, h, kv_h, d, n, s, pos, dtype, spread=8.0)
    assert tensor_cores(c, min(s, window + sinks + n))
    k, v, k64, v64 = c.caches(True)
    out = OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(), k, v, window, sinks, 1.0)
    ref, mag = R.attention_wide(c.q64.to(DEV) * d ** 0.5, k64.to(DEV), v64.to(DEV), pos, window=window, sinks=sinks)
    check_fine(out, ref.cpu(), mag.cpu(), dtype)


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,p,dtype", [
    (70, 8, 2, 128, 1, 32, [i % 32 for i in range(70)], 24001, torch.float16),
    (33, 32, 2, 64, 2, 24, [i % 23 - 1 for i in range(33)], 8100, torch.bfloat16),
    (2, 32, 1, 128, 100, 900, [800, -1], 5000, torch.float16),
])
def test_long_prefix_keeps_the_probabilities(b, h, kv_h, d, n, s, pos, p, dtype):
    c = Cancelling(b, h, kv_h, d, n, s, pos, dtype, prefix=p, spread=8.0)
    assert tensor_cores(c, p, True)
    k, v, k64, v64 = c.caches(True)
    out = OPS.attention_shared_prefix(c.q, c.nk, c.nv, c.pos_t(), c.pk.to(DEV), c.pv.to(DEV), k, v, 1.0)
    ref, mag = R.attention_wide(c.q64.to(DEV) * d ** 0.5, k64.to(DEV), v64.to(DEV), pos, prefix=(c.pk.double().to(DEV), c.pv.double().to(DEV)))
    check_fine(out, ref.cpu(), mag.cpu(), dtype)


def replayed(*ways):
    """Each way: a change of the inputs and a call.  Captured once, replayed with other data each time, against the same call made directly; two graphs take turns."""
    graphs = []
    for change, call in ways:
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for turn in range(4):
        for change, _ in ways:
            change(turn)
        for graph, _ in graphs + graphs[:1]:                          # (the first once more: a replay right behind another's launches)
            graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in out] for _, out in graphs]
        for (_, call), mine in zip(ways, got):
            torch.cuda.synchronize()
            for x, y in zip(mine, call()):
                bits = torch.int16 if x.element_size() == 2 else torch.int32
                assert torch.equal(x.view(bits), y.view(bits)), turn
    assert _lib.load().alloyb_device_error(1) == 0 and ops.span_status() == 0


def moving(c, seed):
    """A change of q, of the new rows and of the positions in place."""
    at = c.pos_t()

    def change(turn):
        g = torch.Generator().manual_seed(seed * 100 + turn)
        c.q.copy_(torch.randn(c.q.shape, generator=g))
        c.nk.copy_(torch.randn(c.nk.shape, generator=g))
        c.nv.copy_(torch.randn(c.nv.shape, generator=g))
        new = torch.randint(-1, c.s - c.n + 1, (c.b,), generator=g)
        at.copy_(new.int() if turn else torch.tensor(c.pos, dtype=torch.int32).expand(c.b))
    return at, change


def scored_way(c, seed):
    at, change = moving(c, seed)
    k, v = c.k.to(DEV), c.v.to(DEV)
    w0 = torch.rand(c.b, c.kv_h, c.s, generator=torch.Generator().manual_seed(seed)).to(DEV)

    def call():
        w = w0.clone()
        return OPS.attention_cache_scored(c.q, c.nk, c.nv, at, k, v, w), w, k, v
    return change, call


def test_replays_of_launches_that_begin_beside_one_another():
    """Large prefixes with few own keys, and scored calls: launches that skip their wait when the one ahead has told that it may, in graphs."""
    c = Case(70, 8, 2, 128, 1, 32, [i % 32 for i in range(70)], prefix=24001)
    assert tensor_cores(c, 24001, True)
    pk, pv, k, v = (t.to(DEV) for t in (c.pk, c.pv, c.k, c.v))
    at, change = moving(c, 1)
    behind = change, lambda: (OPS.attention_shared_prefix(c.q, c.nk, c.nv, at, pk, pv, k, v), k, v)
    replayed(behind, scored_way(Case(40, 16, 8, 128, 1, 300, [(i * 37) % 300 for i in range(40)]), 2))
    replayed(scored_way(Case(2, 32, 8, 64, 12, 900, [700, 880]), 3), scored_way(Case(1, 16, 2, 128, 5, 9000, [8000]), 4))


def test_replays_of_large_chunks():
    """Tensor maps are made when a call is captured; what they lead to changes from replay to replay."""
    ways = []
    for seed, (b, h, kv_h, d, n, s, pos) in enumerate([(1, 8, 1, 128, 700, 6000, [5100]), (4, 24, 2, 64, 500, 5000, [4000, -1, 0, 777])]):
        c = Case(b, h, kv_h, d, n, s, pos)
        assert tensor_cores(c, min(s, 4000 + 129 + n))
        at, change = moving(c, seed + 9)
        k, v = c.k.to(DEV), c.v.to(DEV)
        ways.append((change, lambda c=c, at=at, k=k, v=v: (OPS.attention_cache_window(c.q, c.nk, c.nv, at, k, v, 4000, 129), k, v)))
    replayed(*ways)


# calls whose scores take more than 1 GiB, which run in parts
@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos,dtype,write", [
    (2, 64, 4, 128, 301, 8192, [7000, 0], torch.float16, True),                    # 4 MiB a token: parts of 151 and 150
    (2, 128, 1, 64, 5, 262143, [262138, 100], torch.bfloat16, False),              # 256 MiB a token: parts of 3 and 2
    (5, 64, 1, 64, 7, 200000, [199993, -1, 199994, 3, 70000], torch.float16, True),    # an idle sequence, one whose last token does not fit
])
def test_scored_in_parts(b, h, kv_h, d, n, s, pos, dtype, write):
    parts = -(-b * h * n * s * 4 // (1 << 30))
    assert parts > 1 and _lib.load().alloyb_attn_span_workspace_bytes(b, h, kv_h, d, n, s, 0, 0, 0, 1) < 3 << 29
    c = Case(b, h, kv_h, d, n, s, pos, dtype)
    k, v, k64, v64 = c.caches(write)
    k0 = k.clone()
    w = torch.rand(b, kv_h, s, generator=torch.Generator().manual_seed(1)).to(DEV)
    before, add = w.double(), torch.zeros(b, kv_h, s, dtype=torch.float64, device=DEV)
    for i in range(b):
        if c.place(i) is not None:
            w[i, :, c.place(i):c.place(i) + n] = float("nan")
            before[i, :, c.place(i):c.place(i) + n] = 0.0
    out = OPS.attention_cache_scored(c.q, c.nk, c.nv, c.pos_t(), k, v, w, -1.0, write)
    ref, mag = R.attention_wide(c.q64.to(DEV), k64.to(DEV), v64.to(DEV), pos, weights=add)
    got = out.double()
    assert ((got - ref).abs() <= R.out_bound(ref, mag, dtype)).all()
    big = float((c.q64.abs().amax() * c.k.abs().amax()) * d ** 0.5)
    # a rounding of the sum a part on top of the probabilities' errors
    assert ((w.double() - before - add).abs() <= R.weight_bound(add, big, d) + (before + add) * parts * 2.0 ** -23).all()
    c.check_written(k0, k, c.nk64, write)
    assert ops.span_status() == (1 if any(p + n > s for p in pos) else 0)


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos", [
    (2, 8, 2, 128, 1, 300, [290, 100]),                                            # clusters
    (40, 16, 8, 128, 1, 300, [299 - i for i in range(40)]),                        # streamed
    (1, 8, 1, 128, 1, 33000, [32000]),
    (1, 16, 2, 128, 5, 9000, [8000]),                                              # row tiles, several parts
    (2, 8, 2, 64, 40, 300, [200, 7]),
])
@pytest.mark.parametrize("at", [0, 5])
def test_scored_of_rows_that_are_not_numbers(b, h, kv_h, d, n, s, pos, at):
    """A NaN in a key makes every weight of the rows that see it a NaN, wherever among the keys it lies; sequence 0's first KV head has one."""
    c = Case(b, h, kv_h, d, n, s, pos)
    c.k[0, 0, at, 3] = float("nan")
    k, v, _, _ = c.caches(True)
    w = torch.zeros(b, kv_h, s, device=DEV)
    out = OPS.attention_cache_scored(c.q, c.nk, c.nv, c.pos_t(), k, v, w)
    assert out[0, :h // kv_h].isnan().all() and w[0, 0, :pos[0] + n].isnan().all() and not w[0, 0, pos[0] + n:].any()
    assert not out[0, h // kv_h:].isnan().any() and not w[0, 1:].isnan().any() and not w[1:].isnan().any() and not out[1:].isnan().any()


@pytest.mark.parametrize("b,h,kv_h,d,n,s,pos", [
    (2, 8, 2, 128, 1, 300, [290, 0]),
    (40, 16, 8, 128, 1, 300, [299 - i for i in range(40)]),
    (1, 8, 1, 128, 1, 33000, [32000]),
    (1, 16, 2, 128, 5, 9000, [8000]),
    (2, 8, 2, 64, 40, 300, [200, 7]),
])
def test_scored_of_rows_that_see_nothing(b, h, kv_h, d, n, s, pos):
    """Every score of sequence 0's first KV head is -inf: nothing is attended to, the outputs are zeros and the weights do not grow."""
    c = Case(b, h, kv_h, d, n, s, pos)
    c.k[0, 0, :, 0] = float("-inf")
    c.nk64[0, 0, :, 0] = float("-inf")
    c.nk[0, 0, :, 0] = float("-inf")
    c.q[0, :h // kv_h, :, 0] = 1.0
    k, v, _, _ = c.caches(True)
    w = torch.rand(b, kv_h, s, generator=torch.Generator().manual_seed(1)).to(DEV)
    want = w[0, 0].clone()
    want[pos[0]:pos[0] + n] = 0.0
    out = OPS.attention_cache_scored(c.q, c.nk, c.nv, c.pos_t(), k, v, w)
    assert not out[0, :h // kv_h].any() and torch.equal(w[0, 0], want)
    assert not w.isnan().any() and not out.isnan().any() and (kv_h == 1 or out[0, h // kv_h:].any())


def check_wide(c, out, k64, v64, pos, dtype, **kw):
    ref, mag = R.attention_wide(c.q64.to(DEV), k64.to(DEV), v64.to(DEV), pos, **kw)
    over = (out.double() - ref).abs() - R.out_bound(ref, mag, dtype)
    assert _lib.load().alloyb_device_error(1) == 0 and torch.isfinite(out).all() and float(over.max()) <= 0, float(over.max())


# the fewest rows that go to tiles of 128: one tile, mostly or nearly empty, full, and one row more
@pytest.mark.parametrize("b,h,kv_h,d,n,s,window,sinks,dtype,write", [
    (16, 68, 4, 128, 1, 3700, 9999, 0, torch.float16, True),                       # 17 rows
    (32, 32, 8, 128, 5, 820, 700, 100, torch.bfloat16, False),                     # 20
    (24, 12, 4, 64, 11, 2600, 2500, 70, torch.float16, True),                      # 33
    (6, 8, 8, 128, 127, 800, 600, 3, torch.float16, True),                         # 127
    (8, 32, 4, 64, 16, 2000, 1990, 0, torch.bfloat16, False),                      # 128
    (8, 6, 2, 128, 43, 2000, 1900, 65, torch.float16, True),                       # 129
])
def test_window_of_few_rows_on_tensor_cores(b, h, kv_h, d, n, s, window, sinks, dtype, write):
    pos = [(i * 977) % (s - n + 1) if i % 5 != 3 else -1 for i in range(b - 1)] + [s - n]
    c = Case(b, h, kv_h, d, n, s, pos, dtype)
    assert tensor_cores(c, min(s, window + sinks + n))
    k, v, k64, v64 = c.caches(write, window, sinks)
    k0, v0 = k.clone(), v.clone()
    out = OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(), k, v, window, sinks, -1.0, write)
    check_wide(c, out, k64, v64, pos, dtype, window=window, sinks=sinks)
    c.check_written(k0, k, c.nk64, write)
    c.check_written(v0, v, c.nv64, write)


@pytest.mark.parametrize("b,h,kv_h,d,n,p,dtype,write", [
    (8, 32, 8, 128, 1, 51001, torch.float16, True),                                # 32 rows in all
    (11, 12, 4, 64, 1, 99000, torch.bfloat16, False),                              # 33
    (127, 8, 8, 128, 1, 12801, torch.float16, True),                               # 127
    (32, 8, 2, 64, 1, 50790, torch.float16, False),                                # 128
    (43, 6, 2, 128, 1, 50400, torch.bfloat16, True),                               # 129
    (1, 36, 2, 128, 2, 55000, torch.float16, True),                                # 36 rows of one sequence
    (70, 8, 2, 128, 1, 24001, torch.float16, True),                                # 280
    (40, 64, 8, 128, 1, 5123, torch.float16, True),                                # 320
])
def test_prefix_of_few_rows_on_tensor_cores(b, h, kv_h, d, n, p, dtype, write):
    s = 150
    pos = [(i * 37) % (s - n + 1) if i % 6 != 4 else -1 for i in range(b)]
    c = Case(b, h, kv_h, d, n, s, pos, dtype, prefix=p)
    assert tensor_cores(c, p, True)
    k, v, k64, v64 = c.caches(write)
    k0 = k.clone()
    store = [torch.full((kv_h, p + 8, d), float("nan"), dtype=torch.float16, device=DEV) for _ in range(2)]
    for t, src in zip(store, (c.pk, c.pv)):
        t[:, :p] = src.to(DEV)
    out = OPS.attention_shared_prefix(c.q, c.nk, c.nv, c.pos_t(), store[0][:, :p], store[1][:, :p], k, v, -1.0, write)
    check_wide(c, out, k64, v64, pos, dtype, prefix=(c.pk.double().to(DEV), c.pv.double().to(DEV)))
    c.check_written(k0, k, c.nk64, write)


def prefix_and_scored():
    """Calls whose second launch may begin beside the first, and what each gives alone."""
    p = 24001
    c = Case(70, 8, 2, 128, 1, 32, [(i * 5) % 32 for i in range(70)], prefix=p)
    assert tensor_cores(c, p, True)
    step, chunk = Case(40, 16, 8, 128, 1, 300, [(i * 37) % 300 for i in range(40)]), Case(2, 32, 8, 64, 12, 900, [700, 880])
    data = {x: (x.pos_t(), x.k.to(DEV), x.v.to(DEV)) for x in (c, step, chunk)}
    pk, pv = c.pk.to(DEV), c.pv.to(DEV)

    def prefix():
        at, k, v = data[c]
        return OPS.attention_shared_prefix(c.q, c.nk, c.nv, at, pk, pv, kc := k.clone(), vc := v.clone()), kc, vc

    def scored(x):
        at, k, v = data[x]
        w = torch.ones(x.b, x.kv_h, x.s, device=DEV)
        return OPS.attention_cache_scored(x.q, x.nk, x.nv, at, kc := k.clone(), vc := v.clone(), w), kc, vc, w

    calls = [prefix, lambda: scored(step), prefix, lambda: scored(chunk)]
    alone = []
    for f in calls:
        torch.cuda.synchronize()
        alone.append([t.clone() for t in f()])
        torch.cuda.synchronize()
    return calls, alone


def same_bits(alone, got):
    for x, y in zip(alone, got):
        bits = torch.int16 if x.element_size() == 2 else torch.int32
        assert torch.equal(x.view(bits), y.view(bits))


def test_large_prefixes_in_a_row():
    calls, alone = prefix_and_scored()
    rounds = [[f() for f in calls] for _ in range(4)]
    torch.cuda.synchronize()
    for got in rounds:
        for a, z in zip(alone, got):
            same_bits(a, z)


def test_large_prefixes_of_two_threads_on_one_stream():
    calls, alone = prefix_and_scored()
    got, failed, start = [[], []], [], threading.Barrier(2)

    def turns(i):
        try:
            start.wait()
            for n in range(60):
                got[i].append(((n + i) % len(calls), calls[(n + i) % len(calls)]()))
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    pool = [threading.Thread(target=turns, args=(i,)) for i in range(2)]
    for t in pool:
        t.start()
    for t in pool:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for n, results in got[0] + got[1]:
        same_bits(alone[n], results)


def test_conversation_in_a_bounded_cache():
    """Steps and evictions in place, sequences that sit calls out among them: every new row is among the next eviction's, the last ones stay, and an
    idle sequence keeps its rows."""
    b, h, kv_h, d, s, keep, sinks, recent = 3, 8, 2, 64, 64, 40, 4, 8
    g = torch.Generator().manual_seed(11)
    k, v = (torch.zeros(b, kv_h, s, d, dtype=torch.float16, device=DEV) for _ in range(2))
    w = torch.zeros(b, kv_h, s, device=DEV)
    held = torch.zeros(b, dtype=torch.int32, device=DEV)
    for step, n in enumerate([30, 20, 1, 1, 17, 1]):
        idle = torch.tensor([step % 3 == 1, False, step == 2], device=DEV)
        q, nk, nv = (torch.randn(b, n, x, d, generator=g).half().to(DEV).transpose(1, 2) for x in (h, kv_h, kv_h))
        pos = torch.where(idle, -1, held)
        out = OPS.attention_cache_scored(q, nk, nv, pos, k, v, w)
        ref, _, mag, _ = R.attention(q.double().cpu(), k.double().cpu(), v.double().cpu(), pos.tolist())
        assert ((out.double().cpu() - ref).abs() <= R.out_bound(ref, mag, torch.float16)).all()
        before = k.clone()
        held = torch.where(idle, held, held + n)
        kept, left = OPS.kv_evict(k, v, w, held, k, v, w, keep, sinks, recent)
        for i in range(b):
            rows, new = held[i].item(), left[i].item()
            assert new == min(rows, keep)
            if idle[i]:
                assert kept[i, :, :new].tolist() == [list(range(new))] * kv_h
            else:
                last = min(n, recent, rows)
                assert kept[i, :, new - last:new].tolist() == [list(range(rows - last, rows))] * kv_h
                assert torch.equal(k[i, :, new - last:new], nk[i, :, n - last:])
            assert torch.equal(k[i, :, :new], torch.gather(before[i], 1, kept[i, :, :new].long()[..., None].expand(-1, -1, d)))
        held = left
    assert ops.span_status() == 0


@pytest.mark.parametrize("n", [1, 9, 40])
def test_caches_of_more_sequences_than_the_call(n):
    """The call has the cache's first sequences; the others' rows and weights are left alone."""
    b, h, kv_h, d, s, p = 2, 8, 2, 128, 200, 70
    c = Case(b, h, kv_h, d, n, s, [150, 3], prefix=p)
    wide = [torch.full((b + 2, kv_h, s, d), float("nan"), dtype=torch.float16, device=DEV) for _ in range(2)]
    w = torch.full((b + 2, kv_h, s), 7.0, device=DEV)
    k, v, k64, v64 = c.caches(True)
    for call, kw in (
        (lambda kk, vv: OPS.attention_cache_window(c.q, c.nk, c.nv, c.pos_t(), kk, vv, 50, 3), dict(window=50, sinks=3)),
        (lambda kk, vv: OPS.attention_shared_prefix(c.q, c.nk, c.nv, c.pos_t(), c.pk.to(DEV), c.pv.to(DEV), kk, vv), dict(prefix=(c.pk.double(), c.pv.double()))),
        (lambda kk, vv: OPS.attention_cache_scored(c.q, c.nk, c.nv, c.pos_t(), kk, vv, w), dict()),
    ):
        for t, src in zip(wide, (k, v)):
            t[:b] = src
        out = call(*wide)
        ref, _, mag, _ = R.attention(c.q64, k64, v64, c.pos, **kw)
        assert ((out.double().cpu() - ref).abs() <= R.out_bound(ref, mag, torch.float16)).all()
        c.check_written(k, wide[0][:b], c.nk64, True)
        assert wide[0][b:].isnan().all() and wide[1][b:].isnan().all()
    assert (w[b:] == 7.0).all() and not (w[:b] == 7.0).all()


def test_eviction_in_place_replayed():
    """A graph of an eviction in place gives what the call gives, on other weights and lengths each time."""
    b, kv_h, s, d, keep = 3, 2, 900, 64, 200
    g = torch.Generator().manual_seed(2)
    k, v = (torch.zeros(b, kv_h, s, d, dtype=torch.float16, device=DEV) for _ in range(2))
    w, lengths = torch.zeros(b, kv_h, s, device=DEV), torch.full((b,), s, dtype=torch.int32, device=DEV)

    def call():
        return OPS.kv_evict(k, v, w, lengths, k, v, w, keep, 4, 50)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept, new = call()
    for turn in range(3):
        data = [torch.randn(b, kv_h, s, d, generator=g).half(), torch.randn(b, kv_h, s, d, generator=g).half(), torch.rand(b, kv_h, s, generator=g)]
        lengths.copy_(torch.randint(0, s + 1, (b,), generator=g).int())
        got = []
        for run in (lambda: (graph.replay(), (kept, new))[1], call):
            for t, x in zip((k, v, w), data):
                t.copy_(x)
            out = run()
            torch.cuda.synchronize()
            got.append([t.clone() for t in (*out, k, v, w)])
        for x, y in zip(*got):
            assert torch.equal(x, y)
        for i in range(b):
            rows = R.evict(data[2][i, 0].tolist(), lengths[i].item(), keep, 4, 50)
            assert got[0][0][i, 0].tolist() == rows + [-1] * (keep - len(rows)) and torch.equal(got[0][2][i, 0, :len(rows)].cpu(), data[0][i, 0, rows])
    assert ops.span_status() == 0
