"""Logits processing (csrc/logits_process.hip) against the 64-bit form of oracle/serving_oracle.py.

Tolerance: each of the at most five fp32 operations of a value (division or product, presence, frequency * c and its
subtraction, bias) is off by u = 2^-24 of its result, which is at most M = |x| max(r, 1 / r) + presence + frequency c + |bias|
(the scalars' own rounding to fp32 adds one u of each term): 8 u M; then half a step of out's type.  The
log-sum-exp: the values' error, (V / 64 + 64) u of the sum relative (online fp32 sums, at most V / threads terms a
thread, then the joins), the exponentials' few ulp (2^-21) and the final rounding."""
import math

import pytest
import torch

from conftest import PKG
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
lg = PKG.models.modules.logits
U = 2.0 ** -24


def make(n, vocab, hist, seed, dtype=torch.float32, bias=None, allowed=None, states=None, ties=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, vocab, generator=g) * 3
    if ties:
        x = (x * 2).round() / 2
    d = dict(logits=x.to(dtype))
    if hist is not None:
        t = torch.randint(-2, vocab + 2, (n, hist), generator=g)
        t = torch.where(torch.rand(n, hist, generator=g) < 0.5, t % max(1, vocab // 9 + 1), t)
        d["tokens"] = t.to(torch.int32)
        d["token_lens"] = torch.randint(0, hist + 1, (n,), generator=g).to(torch.int32)
        if n > 1:
            d["token_lens"][0], d["token_lens"][1] = hist, 0
    if bias == "shared":
        d["bias"] = torch.randn(vocab, generator=g)
    elif bias == "rows":
        d["bias"] = torch.randn(n, vocab, generator=g)
    if allowed:
        rows = {"one": 1, "rows": n, "states": 3}[allowed.split("-")[0]]
        ok = torch.rand(rows, vocab, generator=g) < 0.6
        if allowed.endswith("bits"):
            w = (vocab + 31) // 32
            p = torch.zeros(rows, w * 32, dtype=torch.int64)
            p[:, :vocab] = ok
            words = (p.view(rows, w, 32) << torch.arange(32)).sum(-1)
            ok = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
        d["allowed"] = ok if rows > 1 or allowed.startswith("rows") else ok[0]
        if allowed.startswith("states"):
            d["states"] = torch.randint(-1, 4, (n,), generator=g).to(torch.int32)
    return d


def up(d, dev):
    return {k: (t.to(dev) if isinstance(t, torch.Tensor) else t) for k, t in d.items()}


def bound(d):
    r = d.get("repetition", 1.0)
    col = lambda v: v[:, None].double() if isinstance(v, torch.Tensor) else v  # noqa: E731
    r = col(r)
    big = torch.maximum(torch.as_tensor(r, dtype=torch.float64), 1 / torch.as_tensor(r, dtype=torch.float64))
    m = d["logits"].double().abs() * big
    if d.get("tokens") is not None:
        m = m + abs(col(d.get("presence", 0.0))) + abs(col(d.get("frequency", 0.0))) * d["tokens"].shape[1]
    if d.get("bias") is not None:
        m = m + d["bias"].double().abs()
    return 8 * U * m


def check(d, dev, out_dtype=None):
    ref, best, lse = O.process_logits(**d)
    g = up(d, dev)
    out = None if out_dtype is None else torch.empty(ref.shape, dtype=out_dtype, device=dev)
    x, b, l = lg.process_logits(**g, out=out, stats=True)
    assert x.dtype == (out_dtype or torch.float32) and b.dtype == torch.int64
    tol = bound(d)
    u = 0.0 if out_dtype in (None, torch.float32) else torch.finfo(out_dtype).eps / 2
    x, b, l = x.double().cpu(), b.cpu(), l.double().cpu()
    same_inf = torch.isinf(ref)
    assert torch.equal(x[same_inf], ref[same_inf])
    fin = ~same_inf
    assert bool(((x - ref).abs() <= tol * (1 + u) + u * ref.abs())[fin].all())
    # the pick: the 64-bit best unless its lead is within the values' error
    vals = torch.where(same_inf, -math.inf, ref)
    for i in range(ref.shape[0]):
        if int(best[i]) < 0:
            assert int(b[i]) == -1
        else:
            assert float(vals[i, b[i]]) >= float(vals[i, best[i]]) - 2 * float(tol[i].max())
    V = ref.shape[1]
    ok = torch.isfinite(lse)
    ltol = tol.amax(1) + (V / 64 + 64) * U + 2.0 ** -21 + 2 * U * lse.abs()
    assert torch.equal(l[~ok], lse[~ok]) and bool(((l - lse).abs() <= ltol)[ok].all())
    token, logp = lg.pick_tokens(**g)
    assert torch.equal(token.cpu(), b)
    for i in range(ref.shape[0]):
        if int(b[i]) < 0:
            assert float(logp[i]) == -math.inf
        elif bool(ok[i]):
            assert abs(float(logp[i]) - float(vals[i, b[i]] - lse[i])) <= float(ltol[i] + tol[i].max() + 4 * U * abs(lse[i]))


PEN = dict(repetition=1.3, presence=0.4, frequency=0.15)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("n, vocab, hist", [(1, 1, 1), (3, 7, 5), (2, 40, 0), (5, 1000, 33), (3, 8191, 700), (2, 8192, 9),
                                            (2, 8193, 300), (4, 50021, 5000), (130, 999, 17)])
def test_penalties(dev, n, vocab, hist, dtype):
    check({**make(n, vocab, hist, n + vocab, dtype), **PEN}, dev)
    check({**make(n, vocab, hist, n + vocab + 1, dtype, bias="rows"), **PEN}, dev, out_dtype=dtype)


@pytest.mark.parametrize("n, vocab, hist", [(2, 20001, 2048), (2, 20001, 2049), (513, 2500, 5), (257, 9000, 20)])
def test_ways_to_cut_a_row(dev, n, vocab, hist):
    """Small and large tiles for histories of each side, rows in one tile and in several."""
    check({**make(n, vocab, hist, n + hist), **PEN}, dev)


@pytest.mark.parametrize("allowed", ["one", "rows", "states", "one-bits", "rows-bits", "states-bits"])
@pytest.mark.parametrize("vocab", [31, 1000, 8200, 20001])
def test_masks(dev, vocab, allowed):
    check(make(4, vocab, None, vocab, torch.bfloat16, bias="shared", allowed=allowed), dev)
    check({**make(4, vocab, 50, vocab, allowed=allowed), **PEN}, dev)


def test_per_row_penalties(dev):
    d = make(4, 500, 60, 1)
    d.update(repetition=torch.tensor([1.0, 0.5, 2.0, 1.7]), presence=torch.tensor([0.0, 1.0, -1.0, 0.3]),
             frequency=torch.tensor([0.2, 0.0, -0.1, 5.0]))
    check(d, dev)


def test_counts_every_occurrence(dev):
    """One token 5,000 times, and numbers outside the vocabulary."""
    d = dict(logits=torch.zeros(1, 100), tokens=torch.full((1, 5002), 42, dtype=torch.int32), frequency=0.001)
    d["tokens"][0, 0], d["tokens"][0, 1] = -1, 100
    x = lg.process_logits(**up(d, dev)).cpu()
    assert abs(float(x[0, 42]) + 5.0) <= 4 * U * 5 and float(x.abs().sum() - x[0, 42].abs()) == 0.0


@pytest.mark.parametrize("vocab", [40, 20001])
def test_ties_nan_and_nothing_left(dev, vocab):
    d = make(6, vocab, None, 3, ties=True)
    d["logits"][0] = 2.0
    d["logits"][1] = -math.inf
    d["logits"][2, vocab // 2] = math.nan
    d["logits"][2, vocab - 1] = math.nan
    d["logits"][3, vocab - 2] = math.inf
    d["logits"][4] = 0.0
    d["logits"][4, 5] = -0.0
    d["logits"][4, 3] = -0.0
    d["logits"][4, :3] = -1.0
    x, b, l = lg.process_logits(d["logits"].to(dev), stats=True)
    ref, best, lse = O.process_logits(d["logits"])
    assert b.tolist() == best.tolist() and b[0] == 0 and b[1] == -1 and b[2] == vocab // 2 and b[4] == 3
    assert torch.equal(x.cpu().nan_to_num(9.0), d["logits"].nan_to_num(9.0))
    assert l[1] == -math.inf and bool(l[2].isnan()) and l[3] == math.inf
    t, lp = lg.pick_tokens(d["logits"].to(dev))
    assert t.tolist() == best.tolist() and lp[1] == -math.inf and bool(lp[2].isnan())
    # masked: NaN and infinities in masked places are gone, and so is everything
    ok = torch.zeros(6, vocab, dtype=torch.bool)
    ok[2, 1] = ok[3, 2] = True
    x, b, l = lg.process_logits(d["logits"].to(dev), allowed=ok.to(dev), stats=True)
    assert b.tolist() == [-1, -1, 1, 2, -1, -1]
    assert bool((x.cpu()[~ok] == -math.inf).all())
    assert float(l[2]) == float(d["logits"][2, 1]) and float(l[0]) == -math.inf
    # the lowest number of each type
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        low = torch.full((1, vocab), torch.finfo(dt).min, dtype=dt, device=dev)
        t, lp = lg.pick_tokens(low)
        assert int(t) == 0 and abs(float(lp) + math.log(vocab)) <= 2 * U * abs(torch.finfo(dt).min)


def test_in_place_strides_and_types(dev):
    d = make(3, 77, 9, 4, torch.bfloat16, bias="rows", allowed="one")
    g = {**up(d, dev), **PEN}
    want = lg.process_logits(**g)
    wide = torch.zeros(3, 200, dtype=torch.bfloat16, device=dev)
    view = wide[:, 5:82]
    view.copy_(g["logits"])
    got = lg.process_logits(view, **{k: v for k, v in g.items() if k != "logits"}, out=view)
    assert got is view and torch.equal(view, want.to(torch.bfloat16))
    assert bool((wide[:, :5] == 0).all()) and bool((wide[:, 82:] == 0).all())
    t = dict(g, logits=g["logits"].t().contiguous().t(), tokens=g["tokens"].t().contiguous().t(),
             bias=g["bias"].t().contiguous().t())
    assert torch.equal(lg.process_logits(**t), want)
    h = torch.empty(3, 77, dtype=torch.float16, device=dev)
    lg.process_logits(**g, out=h)
    assert torch.equal(h, want.to(torch.float16))
    assert lg.process_logits(g["logits"][:0]).shape == (0, 77)


def test_stream_and_graph(dev):
    d = {**up(make(5, 20001, 300, 5, torch.bfloat16, bias="shared", allowed="states-bits"), dev), **PEN}
    want = lg.process_logits(**d, stats=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = lg.process_logits(**d, stats=True)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = lg.process_logits(**d, stats=True)
        pick = lg.pick_tokens(**d)
    for it in range(3):
        d["logits"].copy_(up(make(5, 20001, 300, 30 + it, torch.bfloat16), dev)["logits"])
        eager = lg.process_logits(**d, stats=True)
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a, b)
        assert torch.equal(pick[0], eager[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("vocab", [40, 8192, 20001])
def test_log_probability_of_large_logits(dev, vocab, dtype):
    """Rows of equal logits have -log V whatever their size, and rows of nearly equal large ones the log-probability of
    their differences, which fp32 holds exactly.

    Tolerance: the exponentials (differences of at most 2^6, times log2 e: 2^7 u; few ulp: 2^-21) and their sum
    ((V / 64 + 64) u) relative, so absolute in the logarithm; the logarithm's own 2 u of its value.  Equal logits: the sum
    is a whole number, exact."""
    top = torch.finfo(dtype).max
    for x in (0.0, 1e4, -3e4, top, -top):
        token, logp = lg.pick_tokens(torch.full((2, vocab), x, dtype=dtype, device=dev))
        assert token.tolist() == [0, 0]
        assert bool(((logp.double() + math.log(vocab)).abs() <= 4 * U * math.log(vocab)).all())
    g = torch.Generator().manual_seed(vocab)
    for base in (1e2, 1e4, -1e4, 6e4):
        step = max(2.0 ** -7, torch.finfo(dtype).eps * abs(base))
        x = (base - step * torch.randint(0, 9, (3, vocab), generator=g)).to(dtype)
        d = x.double() - x.double().amax(1, keepdim=True)
        keep = d > -64.0
        x = torch.where(keep, x, -math.inf)
        ref = -torch.where(keep, d, -math.inf).exp().sum(1).log()
        token, logp = lg.pick_tokens(x.to(dev))
        assert token.tolist() == x.double().argmax(1).tolist()
        tol = 2 ** 7 * U + 2.0 ** -21 + (vocab / 64 + 64) * U + 4 * U * ref.abs()
        assert bool(((logp.double().cpu() - ref).abs() <= tol).all())


def test_log_probability_without_a_finite_best(dev):
    x = torch.zeros(4, 20001, device=dev)
    x[0, 7] = math.inf
    x[1, 9] = math.nan
    x[2] = -math.inf
    x[3] = -math.inf
    x[3, 20000] = -5.0
    token, logp = lg.pick_tokens(x)
    assert token.tolist() == [7, 9, -1, 20000]
    assert bool(logp[:2].isnan().all()) and float(logp[2]) == -math.inf and float(logp[3]) == 0.0
