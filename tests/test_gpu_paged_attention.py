"""Paged attention (csrc/paged_attention.hip) against the 64-bit form of oracle/serving_oracle.py.

Tolerance, elementwise, with u = eps / 2 of the type (a rounding is off by at most half a step) and, over the row's visible
keys, A = sum_j p_j |v_j|, S = max_j scale sum_d |q_d k_jd|:
  u |out|                       the output's rounding
  u A                           the weights' rounding to the values' type before the matrix product (16-bit types)
  2 w A, w = (D + 8) 2^-24 S + 2^-20   the weights' relative error, in numerator and denominator: fp32 dot products of D
                                terms, the scaled difference and the exponential (2^-20 covers its few ulp and
                                the rescales)
  2 K 2^-24 A                   fp32 sums over K keys
  2^-25 sum_j |v_j|             fp16 only: weights below its smallest normal number, rounded to its steps of 2^-24
                                (the largest weight is 1, so the denominator is at least 1)
"""
import math

import pytest
import torch

from conftest import PKG
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
pc = PKG.models.modules.paged_cache
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def tolerance(ref, aux, dtype, dim, keys):
    u = torch.finfo(dtype).eps / 2
    A, V, S = aux
    w = (dim + 8) * 2.0 ** -24 * S[..., None] + 2.0 ** -20
    tol = u * ref.abs() + (u if dtype != F32 else 0.0) * A + 2 * w * A + 2 * keys * 2.0 ** -24 * A
    if dtype == FP:
        tol = tol + 2.0 ** -25 * V
    return tol + 1e-30


def make(n, rows, heads, kvh, dim, ps, kv, dtype, seed, packed=None, write=False, starts=None, spare=2):
    """CPU inputs: shuffled pages, NaN in every cell that belongs to no sequence's visible tokens."""
    g = torch.Generator().manual_seed(seed)
    need = [(max(v, 0) + ps - 1) // ps for v in kv]
    width = max(need + [1]) + 1
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((n, width), -1, dtype=torch.int32)
    live = torch.zeros(pages, ps, dtype=torch.bool)
    at = 0
    for s, m in enumerate(need):
        for c in range(m):
            table[s, c] = order[at]
            live[order[at], :max(0, min(ps, kv[s] - c * ps))] = True
            at += 1
    kp = torch.randn(pages, kvh, ps, dim, generator=g).to(dtype)
    vp = torch.randn(pages, kvh, ps, dim, generator=g).to(dtype)
    dead = ~live[:, None, :, None].expand_as(kp)
    kp[dead] = float("nan")
    vp[dead] = float("nan")
    lead = (n, rows) if packed is None else (packed[-1] + 3,)
    q = (torch.randn(*lead, heads, dim, generator=g) * 1.5).to(dtype)
    k = torch.randn(*lead, kvh, dim, generator=g).to(dtype) if write else None
    v = torch.randn(*lead, kvh, dim, generator=g).to(dtype) if write else None
    i32 = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return dict(q=q, k_pages=kp, v_pages=vp, table=table, kv_lens=i32(kv), k=k, v=v, starts=i32(starts),
                offsets=i32(packed))


def up(d, dev):
    return {k: (t.to(dev) if isinstance(t, torch.Tensor) else t) for k, t in d.items()}


def call(d, **kw):
    d = dict(d)
    return pc.paged_attention(d.pop("q"), d.pop("k_pages"), d.pop("v_pages"), d.pop("table"), d.pop("kv_lens"), **d, **kw)


def check(out, d, kp=None, vp=None, **kw):
    ref, aux, rk, rv = O.paged_attention(**d, **kw)
    tol = tolerance(ref, aux, d["q"].dtype, d["q"].shape[-1], int(d["kv_lens"].max()))
    err = (out.double().cpu() - ref).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((err / tol)[bad].max()), bad.nonzero()[:4].tolist())
    if kp is not None:  # the pages, cell for cell (NaN where nothing is)
        assert torch.equal(kp.cpu().nan_to_num(7.25), rk.nan_to_num(7.25))
        assert torch.equal(vp.cpu().nan_to_num(7.25), rv.nan_to_num(7.25))


CASES = [
    # n, rows, heads, kv_heads, dim, page, kv
    (3, 1, 4, 4, 64, 16, [1, 17, 0]),              # single tokens, an empty sequence
    (4, 2, 8, 8, 64, 16, [2, 19, 31, 33]),         # token + probe
    (2, 1, 8, 1, 128, 8, [300, 1]),                # eight heads of one key head, split along the keys
    (2, 3, 12, 4, 32, 1, [40, 5]),                 # one-token pages
    (2, 5, 6, 2, 96, 64, [200, 64]),               # dim between tiles
    (1, 20, 12, 12, 40, 32, [45]),                 # dim 40, one row tile per head
    (2, 70, 4, 2, 64, 16, [70, 131]),              # many rows: the shared-tile kernel
    (1, 150, 8, 1, 128, 128, [1000]),
    (2, 90, 3, 3, 8, 4, [95, 90]),                 # dim 8
    (1, 33, 8, 8, 128, 16, [2049]),                # two row tiles, key ranges
]


@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"r{c[1]}_h{c[2]}x{c[3]}_d{c[4]}_p{c[5]}")
def test_matches_64_bit(dev, case, dtype):
    n, rows, heads, kvh, dim, ps, kv = case
    d = make(n, rows, heads, kvh, dim, ps, kv, dtype, seed=rows * 7 + dim)
    g = up(d, dev)
    check(call(g), d)
    check(call(g, max_kv=max(kv)), d)
    check(call(g, causal=False, scale=0.3), d, causal=False, scale=0.3)


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"r{c[1]}_h{c[2]}x{c[3]}_d{c[4]}_p{c[5]}")
def test_writes_the_chunk(dev, case, dtype):
    """The chunk's own rows are written (also those the pages hold NaN for), read, and nothing else is touched."""
    n, rows, heads, kvh, dim, ps, kv = case
    d = make(n, rows, heads, kvh, dim, ps, kv, dtype, seed=rows * 11 + dim, write=True)
    g = up(d, dev)
    check(call(g), d, g["k_pages"], g["v_pages"])


@pytest.mark.parametrize("write", [False, True])
@pytest.mark.parametrize("max_rows", [None, 40])
def test_packed_rows(dev, write, max_rows):
    """Packed chunks of 0, 1, 33 and 40 rows; the rows behind the last sequence are 0, or left as they were."""
    packed = [0, 0, 1, 34, 74]
    d = make(4, 0, 8, 2, 64, 16, [9, 50, 33, 301], BF, 5, packed=packed, write=write)
    g = up(d, dev)
    out = call(g, max_rows=max_rows)
    check(out, d, g["k_pages"], g["v_pages"])
    assert bool((out[74:] == 0).all())
    mine = torch.full_like(out, 3.0)
    call(g, max_rows=max_rows, out=mine)
    assert torch.equal(mine[:74], out[:74]) and bool((mine[74:] == 3).all())


def test_packed_offsets_out_of_range_are_clamped(dev):
    d = make(2, 0, 4, 4, 64, 16, [30, 30], BF, 6, packed=[0, 5, 11])
    d["offsets"] = torch.tensor([0, 5, 1000], dtype=torch.int32)  # q has 14 rows
    g = up(d, dev)
    out = call(g)
    d["offsets"] = torch.tensor([0, 5, 14], dtype=torch.int32)
    d["starts"] = torch.tensor([25, 30 - 9], dtype=torch.int32)
    check(out, d)


@pytest.mark.parametrize("rows, dtype", [(2, BF), (2, F32), (80, BF), (80, F32)])
def test_starts(dev, rows, dtype):
    """Rows before the first key, a probe behind the last, far positions, a chunk inside the cache."""
    kv = [40, 41, 42, 150, 40]
    starts = [-3, 41 - 1, 2 ** 31 - 5, 20, -2 ** 31]
    d = make(5, rows, 4, 2, 64, 16, kv, dtype, 8, write=True, starts=starts)
    g = up(d, dev)
    out = call(g)
    check(out, d, g["k_pages"], g["v_pages"])
    assert bool((out[0, :3] == 0).all()) and bool((out[4] == 0).all())


@pytest.mark.parametrize("rows", [1, 80])
def test_bad_pages_and_lens_are_not_read(dev, rows):
    """Page numbers outside the pool hide their keys; lengths beyond the table are cut to it."""
    d = make(3, rows, 4, 2, 64, 16, [100, 90, 85], BF, 9, write=True)
    d["table"][0, 2] = -1
    d["table"][1, 0] = 10 ** 9
    d["table"][2, :] = -7
    d["kv_lens"][1] = 2 ** 30
    d["starts"] = torch.tensor([100 - rows, 90 - rows, 85 - rows], dtype=torch.int32)
    g = up(d, dev)
    d["k_pages"], d["v_pages"] = d["k_pages"].nan_to_num(0.5), d["v_pages"].nan_to_num(0.5)
    g["k_pages"], g["v_pages"] = d["k_pages"].to(dev), d["v_pages"].to(dev)
    out = call(g)
    check(out, d, g["k_pages"], g["v_pages"])
    assert bool((out[2] == 0).all())


@pytest.mark.parametrize("rows", [2, 70])
def test_strided_and_misaligned_inputs(dev, rows):
    d = make(2, rows, 4, 2, 64, 16, [80, 75], BF, 10, write=True)
    g = up(d, dev)
    want = call({**g, "k_pages": g["k_pages"].clone(), "v_pages": g["v_pages"].clone()})
    t = dict(g)
    for nm in ("q", "k", "v"):
        x = g[nm]
        t[nm] = x.transpose(1, 2).contiguous().transpose(1, 2)       # head-major storage
        assert not t[nm].is_contiguous()
    assert torch.equal(call({**t, "k_pages": g["k_pages"].clone(), "v_pages": g["v_pages"].clone()}), want)
    for nm in ("q", "k", "v"):
        x = torch.empty(g[nm].numel() + 3, dtype=BF, device=dev)[3:].view(g[nm].shape)  # 6 bytes off
        x.copy_(g[nm])
        t[nm] = x
    assert torch.equal(call({**t, "k_pages": g["k_pages"].clone(), "v_pages": g["v_pages"].clone()}), want)


def test_non_finite_values(dev):
    """A NaN query spoils its own row; NaN or infinite keys and values behind a sequence's length nothing."""
    d = make(2, 2, 4, 4, 64, 16, [20, 9], BF, 11)
    g = up(d, dev)
    clean = call(g)
    dead = g["k_pages"].isnan()
    for bad in (float("inf"), float("-inf")):
        h = dict(g)
        h["k_pages"], h["v_pages"] = g["k_pages"].clone(), g["v_pages"].clone()
        h["k_pages"][dead], h["v_pages"][dead] = bad, bad
        assert torch.equal(call(h), clean)
    h = dict(g, q=g["q"].clone())
    h["q"][0, 1, 2] = float("nan")
    out = call(h)
    assert bool(out[0, 1, 2].isnan().all())
    keep = torch.ones(out.shape[:-1], dtype=torch.bool, device=dev)
    keep[0, 1, 2] = False
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_infinite_value_of_a_later_token_stays_out_of_earlier_rows(dev, dtype):
    """A chunk's token with an infinite value reaches the rows that see it, and no row before it."""
    for rows in (3, 80):
        d = make(1, rows, 4, 2, 64, 16, [rows + 6], dtype, 12, write=True)
        g = up(d, dev)
        clean = call({**g, "k_pages": g["k_pages"].clone(), "v_pages": g["v_pages"].clone()})
        at = rows // 2
        v = g["v"].clone()
        v[0, at, 0, 5] = float("inf")
        out = call({**g, "v": v, "k_pages": g["k_pages"].clone(), "v_pages": g["v_pages"].clone()})
        assert torch.equal(out[0, :at], clean[0, :at])
        assert bool(torch.isinf(out[0, at:, 0, 5]).all()) and bool(torch.isinf(out[0, at:, 1, 5]).all())


def test_offsets_past_32_bits(dev):
    """Pages whose byte offsets pass 2^32 and element offsets 2^31."""
    kvh, ps, dim = 8, 64, 128
    pages = 2 ** 31 // (kvh * ps * dim) + 40
    kp = torch.empty(pages, kvh, ps, dim, dtype=BF, device=dev)
    vp = torch.empty(pages, kvh, ps, dim, dtype=BF, device=dev)
    d = make(2, 1, 16, 8, 128, 64, [200, 70], BF, 13, write=True)
    g = up(d, dev)
    far = torch.arange(pages - d["k_pages"].shape[0], pages, device=dev)
    kp[far], vp[far] = g["k_pages"], g["v_pages"]
    table = torch.where(g["table"] >= 0, g["table"] + int(far[0]), g["table"])
    out = call({**g, "k_pages": kp, "v_pages": vp, "table": table.to(torch.int32)})
    check(out, d, kp[far], vp[far])


def test_long_cache_split(dev):
    """One row over 30,001 keys: many key ranges joined; and the same through a wrong (small) max_kv."""
    d = make(1, 1, 4, 1, 64, 32, [30001], BF, 14)
    g = up(d, dev)
    check(call(g), d)
    check(call(g, max_kv=16), d)


def test_other_stream_and_graph(dev):
    d = make(3, 2, 8, 2, 128, 16, [900, 1200, 3], BF, 15, write=True)
    g = up(d, dev)
    want = call(g)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call(g)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):  # two graphs: their workspaces are their own
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = call(g)
        graphs.append((gr, out))
    for it in range(3):
        g["q"].copy_(up(make(3, 2, 8, 2, 128, 16, [900, 1200, 3], BF, 20 + it, write=True), dev)["q"])
        eager = call(g)
        for gr, out in graphs:
            out.zero_()
            gr.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, eager)


def test_empty_calls(dev):
    d = up(make(2, 1, 4, 2, 64, 16, [5, 6], BF, 16), dev)
    assert call({**d, "q": d["q"][:, :0]}).shape == (2, 0, 4, 64)
    z = {**d, "q": d["q"][:0], "table": d["table"][:0], "kv_lens": d["kv_lens"][:0]}
    assert call(z).shape == (0, 1, 4, 64)
    one = torch.ones(3, 4, 64, dtype=BF, device=dev)  # no sequence at all: every packed row is behind the last
    off = torch.zeros(1, dtype=torch.int32, device=dev)
    out = call({**z, "q": one, "offsets": off})
    assert bool((out == 0).all())
    assert bool((call({**d, "kv_lens": torch.zeros_like(d["kv_lens"])}) == 0).all())


def test_no_table_and_no_pages(dev):
    """A table without columns and a pool without pages: nothing is visible, nothing is written."""
    d = up(make(2, 2, 4, 2, 64, 16, [5, 6], BF, 17, write=True), dev)
    assert bool((call({**d, "table": d["table"][:, :0]}) == 0).all())
    none = d["k_pages"][:0]
    assert bool((call({**d, "k_pages": none, "v_pages": none}) == 0).all())


@pytest.mark.parametrize("n", [65, 130])
def test_packed_many_sequences(dev, n):
    """More sequences than a wave has lanes, empty ones among them, rows before the first sequence."""
    lens = [(i * 7) % 5 for i in range(n)]
    packed = [2]
    for x in lens:
        packed.append(packed[-1] + x)
    kv = [x + (i * 13) % 40 for i, x in enumerate(lens)]
    for heads, kvh in ((4, 2), (32, 1)):
        d = make(n, 0, heads, kvh, 64, 16, kv, BF, n, packed=packed, write=True)
        g = up(d, dev)
        out = call(g, max_rows=4)
        check(out, d, g["k_pages"], g["v_pages"])
        assert bool((out[:2] == 0).all()) and bool((out[packed[-1]:] == 0).all())


def test_expanded_and_single_row_strides(dev):
    """A query shared by all sequences (stride 0), and dimensions of one with arbitrary strides."""
    d = make(3, 1, 4, 2, 64, 16, [9, 30, 17], BF, 18)
    d["q"] = d["q"][:1].expand(3, -1, -1, -1)
    check(call(up(d, dev)), d)
    g = up(make(1, 1, 4, 2, 64, 16, [30], BF, 19), dev)
    want = call(g)
    odd = torch.as_strided(g["q"].contiguous(), (1, 1, 4, 64), (3, 5, 64, 1))
    assert torch.equal(call({**g, "q": odd}), want)


def test_sharers_of_one_page_read_the_same_keys(dev):
    """Two sequences over the same pages, at different lengths."""
    d = make(2, 1, 4, 4, 64, 16, [40, 40], FP, 20)
    d["table"][1] = d["table"][0]
    d["kv_lens"][1] = 35
    check(call(up(d, dev)), d)


@pytest.mark.parametrize("dtype, dim", [(BF, 64), (F32, 40), (FP, 128)], ids=["bf16", "fp32", "fp16"])
@pytest.mark.parametrize("write", [False, True])
def test_packed_rows_over_key_ranges(dev, dtype, dim, write):
    """Packed chunks over caches of 0 to 3,000 keys: some sequences in several key ranges, some in one, rows beyond
    max_rows, rows before the first sequence and behind the last, an empty sequence — for both kernels."""
    packed = [3, 8, 8, 48, 49, 60]
    kv = [3000, 40, 1500, 700, 11]
    for heads, kvh in ((4, 2), (2, 2)):
        d = make(5, 0, heads, kvh, dim, 32, kv, dtype, dim + heads, packed=packed, write=write)
        g = up(d, dev)
        mine = torch.full_like(g["q"], 3.0)
        out = call({**g, "k_pages": g["k_pages"].clone(), "v_pages": g["v_pages"].clone()}, max_rows=35, max_kv=3000,
                   out=mine)
        lim = dict(max_rows=35)
        ref, aux, _, _ = O.paged_attention(**d, **lim)
        tol = tolerance(ref, aux, dtype, dim, 3000)
        seen = torch.zeros(63, dtype=torch.bool)
        for s in range(5):
            seen[packed[s]:min(packed[s + 1], packed[s] + 35)] = True
        err = (out.double().cpu() - ref).abs()
        assert bool((err <= tol)[seen].all())
        assert bool((out.cpu()[~seen] == 3).all())
        full = call(g, max_kv=3000)
        check(full, d, g["k_pages"], g["v_pages"])
        assert bool((full[:3] == 0).all()) and bool((full[60:] == 0).all())


def test_many_rows_of_many_ranges(dev):
    """320 rows of up to 20 ranges each, joined by a workgroup a row; and 16 rows by a larger one."""
    for n in (40, 2):
        kv = [5000 - 120 * (i % 40) for i in range(n)]
        kv[-1] = 30
        d = make(n, 1, 8, 1, 32, 64, kv, BF, n)
        check(call(up(d, dev), max_kv=5000), d)


def test_chunk_over_key_ranges(dev):
    """A chunk of 100 rows whose own keys lie in the last of several ranges."""
    for dtype in (BF, F32):
        d = make(2, 100, 2, 1, 64, 16, [2100, 900], dtype, 31, write=True)
        g = up(d, dev)
        check(call(g, max_kv=2100), d, g["k_pages"], g["v_pages"])


@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("n, heads, kvh, dim, rows, kv", [
    (64, 8, 8, 32, 1, [1 + 699 * i // 63 for i in range(64)]),  # two waves of some hundred keys each
    (3, 64, 64, 16, 1, [6000, 1, 513]),                         # more ranges than run at once
    (1, 2, 2, 128, 2, [400]),                                   # ranges of 64 keys
    (1, 8, 1, 64, 5, [1500]),                                   # 40 rows of one key head: a tile of 128
], ids=["two-waves", "rounds", "short", "rows"])
def test_ways_to_cut_the_keys(dev, n, heads, kvh, dim, rows, kv, dtype):
    d = make(n, rows, heads, kvh, dim, 16, kv, dtype, seed=heads + dim)
    check(call(up(d, dev), max_kv=max(kv)), d)


@pytest.mark.parametrize("dtype", [FP, BF, F32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("bits", [24.5, 25.2, 30.0])
def test_many_small_weights_beside_a_large_one(dev, rows, bits, dtype):
    """One key of weight 1 and value 0 beside 32,000 keys of weight 2^-bits and value 1, in one range: the small ones
    are all that the row's answer is, N w / (1 + N w).

    Tolerance, relative, with u = eps / 2: the output's rounding u; the small weights' rounding u in a 16-bit type (fp16:
    half a step of its subnormal numbers, 2^-25, of weights computed at 2^7 of their size, 2^(7 - bits): 2^(bits - 32)
    of each where that is more); 2 w with w = (D + 8) 2^-24 S + 2^-20, S = bits ln 2; 2 K 2^-24 for the sums over K keys."""
    keys, dim, ps = 32001, 64, 64
    pages = (keys + ps - 1) // ps
    k = torch.zeros(pages, 1, ps, dim, dtype=dtype, device=dev)
    v = torch.ones_like(k)
    q = torch.zeros(1, rows, 1, dim, dtype=dtype, device=dev)
    q[..., 0] = 1.0
    k[0, 0, 0, 0] = 16.0
    v[0, 0, 0] = 0.0
    s = bits * math.log(2.0)
    out = pc.paged_attention(q, k, v, torch.arange(pages, dtype=torch.int32, device=dev)[None],
                             torch.tensor([keys], dtype=torch.int32, device=dev), scale=s / 16.0, causal=False, max_kv=64)
    u = torch.finfo(dtype).eps / 2
    weight = math.exp(-s)
    want = (keys - 1) * weight / (1.0 + (keys - 1) * weight)
    rel = u + 2 * ((dim + 8) * 2.0 ** -24 * s + 2.0 ** -20) + 2 * keys * 2.0 ** -24
    if dtype != F32:
        rel += max(u, 2.0 ** (bits - 32)) if dtype == FP else u
    # (an output below fp16's normal numbers is rounded to its steps of 2^-24)
    assert bool(((out.double() - want).abs() <= rel * want + (2.0 ** -25 if dtype == FP else 0.0)).all())


@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n, rows, heads, kvh, dim, kv", [
    (112, 2, 8, 8, 64, [1 + i % 19 for i in range(112)]),  # a wave each
    (3, 1, 8, 2, 128, [4000, 17, 900]),                    # key ranges and their join
    (2, 70, 4, 2, 64, [1500, 80]),                         # tiles of 128 rows
], ids=["words", "ranges", "rows"])
@pytest.mark.parametrize("write", [False, True])
def test_repeats_itself_exactly(dev, n, rows, heads, kvh, dim, kv, dtype, write):
    """The same call again, over pages that already hold the chunk and over fresh ones: bit for bit the same."""
    kv = [max(x, rows) for x in kv]
    d = make(n, rows, heads, kvh, dim, 16, kv, dtype, seed=n + dim, write=write)
    g = up(d, dev)
    first = call(g, max_kv=max(kv))
    pages = g["k_pages"].clone(), g["v_pages"].clone()
    for _ in range(5):
        h = up(d, dev)
        assert torch.equal(call(h, max_kv=max(kv)), first) and torch.equal(call(g, max_kv=max(kv)), first)
        for a, b in ((h["k_pages"], pages[0]), (h["v_pages"], pages[1]), (g["k_pages"], pages[0])):
            assert torch.equal(a.nan_to_num(7.25), b.nan_to_num(7.25))
