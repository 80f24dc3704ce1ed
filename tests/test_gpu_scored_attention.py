"""Decode attention over 8-bit caches and with capped, distance-biased or
windowed scores, against the 64-bit oracle."""

import pytest
import torch

from cscr import _lib
from cscr import attention as A
from oracle import quant_oracle as Q

pytestmark = pytest.mark.gpu

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def short(p):
    return str(p).replace("torch.", "") if isinstance(p, torch.dtype) else None


@pytest.fixture(autouse=True)
def _clean(built_lib):
    torch.cuda.set_device(0)
    _lib.device_status()
    yield
    torch.cuda.synchronize()


class Case:
    """A decode batch in a paged cache; blocks that no sequence owns, and rows
    past each sequence's end, hold NaN (bytes of all ones in the 8-bit types)."""

    def __init__(self, lens, h, kvh, d, bs, dtype, kind, seed=0, slack=3, spread=0.7):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens_list = lens
        counts = [max(0, -(-n // bs)) for n in lens]
        used = sum(counts)
        nb = used + slack
        self.scale = d ** -0.5
        self.q = torch.randn(len(lens), h, d, generator=g, device="cuda").to(dtype)
        width = max([1] + counts) + 1
        perm = torch.randperm(nb, generator=g, device="cuda").to(torch.int32)
        self.tables = torch.full((len(lens), width), nb + 7, dtype=torch.int32, device="cuda")
        live = torch.zeros(nb, bs, dtype=torch.bool, device="cuda")
        at = 0
        for i, (n, c) in enumerate(zip(lens, counts)):
            self.tables[i, :c] = perm[at:at + c]
            for j in range(c):
                live[perm[at + j].long(), :min(bs, n - j * bs)] = True
            at += c
        self.ks = self.vs = None
        made = []
        for row_spread in (0.7, spread):  # of the keys, of the values
            x = torch.randn(nb, kvh, bs, d, generator=g, device="cuda")
            x = x * torch.exp(row_spread * torch.randn(nb, kvh, bs, 1, generator=g, device="cuda"))
            x = x.to(dtype)
            dead = ~live[:, None, :]
            if kind in Q.QMAX:
                c, s = Q.quantize(x, kind)
                dead = dead.expand(nb, kvh, bs)
                c.view(torch.uint8)[dead] = 0xFF
                s.view(torch.uint8)[dead] = 0xFF
                made.append((c, s))
            else:
                x.masked_fill_(dead[..., None], float("nan"))
                made.append((x, None))
        (self.k, self.ks), (self.v, self.vs) = made
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def run(self, **kw):
        if self.ks is not None:
            return A.paged_attention_quantized(self.q, self.k, self.v, self.ks, self.vs,
                                               self.tables, self.lens, self.scale, **kw)
        return A.paged_attention_biased(self.q, self.k, self.v, self.tables, self.lens, self.scale,
                                        **kw)

    def check(self, out, plain=False, **kw):
        ref = Q.attention(self.q, self.k, self.v, self.ks, self.vs, self.tables, self.lens,
                          self.scale, **kw)
        Q.assert_within(out, ref[0], Q.attention_bound(*ref, self.q.dtype, self.k.dtype, plain))


def slopes(h):
    return torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h).float()


LENS = [0, 1, 31, 32, 33, 16, 17, 500, 1023, 64, 0, 2, 129, 7]
PAIRS = [(BF16, E4M3), (BF16, INT8), (F16, E4M3), (F16, INT8), (BF16, BF16), (F16, F16)]


@pytest.mark.parametrize("dtype,kind", PAIRS, ids=short)
@pytest.mark.parametrize("h,kvh,d,bs", [(16, 2, 128, 16), (14, 2, 64, 32), (4, 4, 128, 8),
                                        (24, 1, 64, 16), (16, 1, 128, 64), (5, 1, 64, 12),
                                        (35, 1, 128, 4), (1, 1, 64, 16)])
def test_head_layouts_and_lengths(h, kvh, d, bs, dtype, kind):
    c = Case(LENS, h, kvh, d, bs, dtype, kind)
    out = c.run()
    assert bool((out[0] == 0).all()) and bool((out[10] == 0).all())
    c.check(out)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype,kind", PAIRS + [(F32, E4M3), (F32, INT8), (F32, F32)], ids=short)
@pytest.mark.parametrize("mods", ["cap", "alibi", "window", "window1", "all"])
def test_score_modifiers(mods, dtype, kind):
    h = 12
    kw = {"cap": dict(softcap=3.0), "alibi": dict(alibi_slopes=slopes(h)),
          "window": dict(window=77), "window1": dict(window=1),
          "all": dict(softcap=20.0, alibi_slopes=slopes(h), window=130)}[mods]
    c = Case(LENS, h, 3, 64, 16, dtype, kind, seed=2)
    c.check(c.run(**kw), **kw)
    c128 = Case(LENS, h, 2, 128, 16, dtype, kind, seed=3)
    c128.check(c128.run(**kw), **kw)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("kind", [E4M3, F16], ids=short)
@pytest.mark.parametrize("cap", [1e-30, 1e-3, 1e4, 1e30])
def test_caps_far_from_the_scores(cap, kind):
    """A tiny cap makes all scores alike, a huge one leaves them as they are."""
    c = Case([300, 40], 8, 2, 64, 16, F16, kind, seed=18)
    c.check(c.run(softcap=cap), softcap=cap)


@pytest.mark.parametrize("dtype,kind", [(BF16, E4M3), (F16, INT8), (BF16, BF16), (F32, INT8)],
                         ids=short)
@pytest.mark.parametrize("h,kvh,d,bs", [(6, 2, 80, 16), (4, 1, 96, 16), (2, 2, 37, 8),
                                        (3, 1, 300, 16), (16, 2, 128, 5), (16, 2, 64, 1)])
def test_other_shapes(h, kvh, d, bs, dtype, kind):
    """Head dims and block sizes outside the tensor-core kernel."""
    c = Case([0, 1, 5, 66, 131], h, kvh, d, bs, dtype, kind, seed=4)
    kw = dict(softcap=9.0, alibi_slopes=slopes(h), window=60)
    c.check(c.run())
    c.check(c.run(**kw), **kw)


@pytest.mark.parametrize("dtype,kind", PAIRS, ids=short)
@pytest.mark.parametrize("lens", [[1], [40000], [9000, 3, 20000], [2] * 700, [33] * 300 + [5000],
                                  list(range(200, 0, -1))],
                         ids=["one", "long", "mixed", "short700", "tail", "ramp"])
def test_splits(lens, dtype, kind):
    """Units cut over warps and CTAs, many units per warp, more sequences than
    threads."""
    c = Case(lens, 8, 1, 64, 16, dtype, kind, seed=5)
    c.check(c.run())
    w = dict(window=301, softcap=30.0)
    c.check(c.run(**w), **w)


def test_one_long_sequence_many_heads():
    c = Case([33333], 32, 2, 128, 32, BF16, E4M3, seed=6)
    c.check(c.run())


@pytest.mark.parametrize("dtype,kind", [(BF16, E4M3), (F16, F16)], ids=short)
def test_holes_and_bad_ids(dtype, kind):
    """Negative block ids are skipped, ids past the pool are skipped and flagged,
    and a sequence that loses every block yields zeros."""
    c = Case([100, 48, 300, 64], 8, 2, 64, 16, dtype, kind, seed=7)
    c.tables[0, 1] = -1
    c.tables[1, :] = -5
    c.tables[2, 0:3] = -1
    c.check(c.run())
    assert _lib.device_status() == 0
    c.tables[3, 2] = c.k.shape[0]
    out = c.run()
    c.check(out)
    assert bool((out[1] == 0).all())
    assert _lib.device_status() == 0x1
    # a bad id outside the window is not read and not flagged
    out = c.run(window=16)
    c.check(out, window=16)
    assert _lib.device_status() == 0


def test_sequences_longer_than_their_table():
    c = Case([64, 10], 8, 2, 128, 16, BF16, INT8, seed=8)
    c.tables = c.tables[:, :4].contiguous()
    c.tables[1] = c.tables[0]
    c.lens = torch.tensor([1000, 64], dtype=torch.int32, device="cuda")
    out = c.run()
    assert torch.isfinite(out).all()
    ref = Q.attention(c.q, c.k, c.v, c.ks, c.vs, c.tables, torch.tensor([64, 64]), c.scale)
    Q.assert_within(out, ref[0], Q.attention_bound(*ref, BF16, INT8))
    assert _lib.device_status() == 0x2


@pytest.mark.parametrize("dtype", [BF16, F16], ids=short)
@pytest.mark.parametrize("kind", [E4M3, INT8], ids=short)
def test_rows_of_very_different_scales(dtype, kind):
    """Value rows some 2^+-12 apart, zero rows, and scores that rise by hundreds
    along the context, so that the references move often."""
    c = Case([700, 90], 8, 2, 128, 16, dtype, kind, seed=9, spread=3.0)
    c.v.view(torch.uint8)[::3, :, ::5] = 0
    c.q *= 0.02
    kw = dict(alibi_slopes=torch.full((8,), 0.5, device="cuda"))
    c.check(c.run(**kw), **kw)
    c.check(c.run())


def test_strided_query_rows():
    c = Case([77, 300, 5], 16, 2, 128, 16, BF16, E4M3, seed=10)
    wide = torch.zeros(3, 20 * 128, dtype=BF16, device="cuda")
    wide[:, :2048] = c.q.view(3, -1)
    want = c.run()
    c.q = wide[:, :2048].view(3, 16, 128)
    assert torch.equal(c.run(), want)
    odd = torch.zeros(3, 20 * 128 + 1, dtype=BF16, device="cuda")  # rows off 16 bytes
    odd[:, :2048] = wide[:, :2048]
    c.q = odd[:, :2048].view(3, 16, 128)
    c.check(c.run())
    with pytest.raises(RuntimeError, match="heads contiguously"):
        c.q = wide.view(3, 20, 128)[:, ::2][:, :16].transpose(0, 1).contiguous().transpose(0, 1)
        c.run()


def test_plain_scores_agree_with_paged_attention():
    """Without modifiers the biased op computes what paged_attention does."""
    c = Case([64, 1, 900, 33], 16, 2, 128, 16, F16, F16, seed=11)
    out = A.paged_attention(c.q, c.k, c.v, c.tables, c.lens, c.scale)
    c.check(out, plain=True)
    c.check(c.run())


def test_same_bits_every_run_and_on_another_stream():
    c = Case([9000, 3, 512, 70, 4000], 16, 2, 128, 16, BF16, E4M3, seed=12)
    first = c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(3):
        outs.append(c.run())
        with torch.cuda.stream(side):
            outs.append(c.run())
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, first)


def test_two_captured_graphs_run_at_once():
    """Graphs captured on one stream and replayed together share no scratch, and
    see lengths that changed since the capture."""
    cases = [Case([5000, 40], 16, 2, 128, 16, BF16, E4M3, seed=13),
             Case([700, 6000], 16, 2, 128, 16, BF16, E4M3, seed=14)]
    for c in cases:
        c.run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(c.run(softcap=30.0))
        graphs.append(gr)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(3):
        for c in cases:
            c.lens.sub_(step * 7)
        torch.cuda.synchronize()
        for _ in range(4):
            for gr, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    gr.replay()
        torch.cuda.synchronize()
        for c, o in zip(cases, outs):
            assert torch.equal(o, c.run(softcap=30.0))
    cases[0].lens.fill_(0)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert bool((outs[0] == 0).all())


@pytest.mark.parametrize("limit", [0, 1, 8])
@pytest.mark.parametrize("kind", [E4M3, BF16], ids=short)
def test_a_wait_that_gives_up_is_reported(kind, limit):
    """With no probes allowed every tile wait gives up (with few, some may): the
    kernel ends, the status says so, and the next call is whole."""
    c = Case([3000, 40, 700], 16, 2, 128, 16, BF16, kind, seed=16)
    want = c.run()
    torch.cuda.synchronize()
    try:
        _lib.set_wait_limit(limit)
        c.run()
        torch.cuda.synchronize()
    finally:
        _lib.set_wait_limit(_lib.WAIT_LIMIT_DEFAULT)
    assert _lib.device_status() in ((0x10,) if limit == 0 else (0, 0x10))
    assert torch.equal(c.run(), want)
    assert _lib.device_status() == 0


def test_refusals():
    c = Case([10], 4, 2, 64, 16, F16, INT8)
    with pytest.raises(RuntimeError, match="alibi_slopes"):
        c.run(alibi_slopes=torch.ones(3, device="cuda"))
    with pytest.raises(RuntimeError, match="alibi_slopes"):
        c.run(alibi_slopes=torch.ones(4))
    with pytest.raises(RuntimeError, match="softcap"):
        c.run(softcap=float("inf"))
    with pytest.raises(RuntimeError, match="window"):
        c.run(window=-1)
    with pytest.raises(RuntimeError, match="int32"):
        A.paged_attention_quantized(c.q, c.k, c.v, c.ks, c.vs, c.tables.long(), c.lens, 0.1)
    with pytest.raises(RuntimeError, match="divisible"):
        A.paged_attention_quantized(c.q[:, :3].contiguous(), c.k, c.v, c.ks, c.vs, c.tables, c.lens,
                                    0.1)
    with pytest.raises(RuntimeError, match="same CUDA device"):
        A.paged_attention_quantized(c.q, c.k, c.v, c.ks, c.vs, c.tables.cpu(), c.lens, 0.1)
    none = c.k[:0]
    out = A.paged_attention_quantized(c.q, none, none, c.ks[:0], c.vs[:0], c.tables, c.lens, 0.1)
    assert bool((out == 0).all())


def test_pool_past_32_bit_byte_offsets():
    nb, kvh, bs, d = 1_100_000, 2, 16, 128  # 4.5 GB per cache
    small = Case([200], 16, kvh, d, bs, BF16, E4M3, seed=15, slack=0)
    k = torch.empty(nb, kvh, bs, d, dtype=torch.uint8, device="cuda")
    v = torch.empty_like(k)
    ks = torch.empty(nb, kvh, bs, dtype=torch.uint8, device="cuda")
    vs = torch.empty_like(ks)
    n = small.k.shape[0]
    for big, src in ((k, small.k), (v, small.v), (ks, small.ks), (vs, small.vs)):
        big[-n:] = src.view(torch.uint8)
    tables = torch.where(small.tables < n, small.tables + (nb - n), 0).to(torch.int32)
    out = A.paged_attention_quantized(small.q, k.view(E4M3), v.view(E4M3),
                                      ks.view(torch.float8_e8m0fnu),
                                      vs.view(torch.float8_e8m0fnu), tables, small.lens,
                                      small.scale)
    assert torch.equal(out, small.run())


@pytest.mark.parametrize("dtype,kind", PAIRS, ids=short)
@pytest.mark.parametrize("d,h,kvh", [(64, 16, 2), (128, 16, 2), (128, 24, 2)])
def test_few_short_units(d, h, kvh, dtype, kind):
    """Batches whose units are taken whole by a CTA, and the first ones that are
    not (the longest is one tile past the limit for its width)."""
    for longest in (1, 95, 192, 193, 384, 385, 768, 769, 1536, 1537):
        c = Case([longest, 0, 1, longest // 2, 17], h, kvh, d, 8, dtype, kind, seed=17)
        c.tables = c.tables[:, :-1].contiguous()  # no spare column: the limit is exact
        c.check(c.run())
