"""``generate`` of the caption decoders (paged cache, page updates, logits processing together) against a beam search
that re-runs the whole decoder in float64 on the host for every word, as the reference's greedy loop does
(models/deformable/unimodal_deformable_dvc.py:304-363).

The heads' weights are scaled up so that the choices are not near ties; scores are compared at 1e-3 of a sum of
at most 9 log-probabilities of magnitude up to ~50, computed by a float32 decoder of two layers (each logit off by some
1e-6 of its size, sums and a log-sum-exp over 40 words of them)."""
import copy
import math

import pytest
import torch

from conftest import PKG
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
M = PKG.models
BOS, EOS, PAD = 2, 3, 1
V, D, N, L, K = 40, 32, 4, 9, 15


def build(kind, seed=5):
    torch.manual_seed(seed)
    cls = (M.unimodal_caption_decoder.UnimodalCaptionDecoder if kind == "unimodal"
           else M.multimodal_caption_decoder.MultimodalCaptionDecoder)
    dec = cls(V, d_model=D, depth=2, num_heads=4, pre_norm=False, return_intermediate=True).double().eval()
    with torch.no_grad():
        dec.head.weight.mul_(8.0)
        dec.head.bias[EOS] += 4.0
    mem = torch.randn(N, K, D, dtype=torch.float64)
    mem2 = torch.randn(N, K + 3, D, dtype=torch.float64)
    kmask = torch.zeros(N, K, dtype=torch.bool)
    kmask[1, 9:] = True
    kmask2 = torch.zeros(N, K + 3, dtype=torch.bool)
    kmask2[2, :4] = True
    return dec, (mem, kmask) if kind == "unimodal" else (mem, kmask, mem2, kmask2)


def rows_fn(kind, dec, mems):
    """(sequence i, its captions (B, L)) -> logits (B, L, V) of the whole decoder."""
    logits = []
    handle = dec.head.register_forward_hook(lambda m, a, out: logits.append(out))

    def f(i, caps):
        look = torch.ones(L, L, dtype=torch.bool).triu(1)
        rep = [t[i:i + 1].expand(caps.shape[0], *t.shape[1:]) for t in mems]
        logits.clear()
        with torch.no_grad():
            if kind == "unimodal":
                pm = (caps == PAD)
                dec(caps, rep[0], tgt_mask=look, memory_mask=rep[1][:, None, None, :], tgt_padding_mask=pm)
            else:
                dec(caps, rep[0], rep[2], tgt_mask=look, tgt_padding_mask=caps == PAD, video_memory_padding_mask=rep[1],
                    audio_memory_padding_mask=rep[3])
        return logits[0][-1]
    return f, handle


def naive(kind, dec, mems, beams, prompt=None, prompt_lens=None, allowed=None, transitions=None, length_penalty=0.0,
          **pen):
    f, handle = rows_fn(kind, dec, mems)
    caps_out, scores_out = [], []
    for i in range(N):
        words = [] if prompt is None else prompt[i][:prompt.shape[1] if prompt_lens is None else prompt_lens[i]].tolist()
        state = 0
        if transitions is not None:
            for w in words:
                state = int(transitions[state, w])
        hyps = [(0.0, [BOS] + words, len(words) + 1 >= L, state)]
        while not all(h[2] for h in hyps):
            cand = []
            for score, toks, done, st in hyps:
                if done:
                    cand.append((score, toks, True, st))
                    continue
                c = torch.full((1, L), PAD, dtype=torch.int32)
                c[0, :len(toks)] = torch.tensor(toks, dtype=torch.int32)
                x = f(i, c)[0, len(toks)][None]
                hist = torch.tensor([toks[1:]], dtype=torch.int32).view(1, -1)
                x, _, lse = O.process_logits(x, hist, None, allowed=None if allowed is None else allowed.view(-1, V)[st:st + 1],
                                             **pen)
                for w in range(V):
                    lp = float(x[0, w] - lse[0])
                    if lp > -math.inf:
                        cand.append((score + lp, toks + [w], w == EOS or len(toks) + 1 >= L,
                                     st if transitions is None else int(transitions[st, w])))
            cand.sort(key=lambda h: -h[0])
            hyps = cand[:beams]
        fin = [(h[0] / (len(h[1]) ** length_penalty if length_penalty else 1.0), h[1]) for h in hyps]
        best = max(fin, key=lambda h: h[0])
        caps_out.append(best[1] + [PAD] * (L - len(best[1])))
        scores_out.append(best[0])
    handle.remove()
    return torch.tensor(caps_out, dtype=torch.int32), torch.tensor(scores_out)


def run(dec, mems, dev, beams, **kw):
    g = copy.deepcopy(dec).float().to(dev)
    args = [t.to(dev, torch.float32) if t.is_floating_point() else t.to(dev) for t in mems]
    kw = {k: (v.to(dev) if isinstance(v, torch.Tensor) else v) for k, v in kw.items()}
    caps, scores = g.generate(*args, BOS, EOS, PAD, L, beams=beams, **kw)
    return caps.cpu(), scores.double().cpu()


@pytest.mark.parametrize("kind", ["unimodal", "multimodal"])
@pytest.mark.parametrize("beams", [1, 3])
def test_equals_full_redecode(dev, kind, beams):
    dec, mems = build(kind)
    caps, scores = run(dec, mems, dev, beams)
    ref, rs = naive(kind, dec, mems, beams)
    assert torch.equal(caps, ref) and bool(((scores - rs).abs() <= 1e-3).all())


@pytest.mark.parametrize("kind", ["unimodal", "multimodal"])
def test_one_beam_is_the_greedy_decode(dev, kind):
    dec, mems = build(kind, seed=6)
    caps, _ = run(dec, mems, dev, 1)
    g = copy.deepcopy(dec).float().to(dev)
    args = [t.to(dev, torch.float32) if t.is_floating_point() else t.to(dev) for t in mems]
    greedy, _ = g.greedy_decode(*args, BOS, EOS, PAD, L)
    assert torch.equal(caps, greedy.cpu())


@pytest.mark.parametrize("beams", [1, 4])
def test_prompts_and_penalties(dev, beams):
    dec, mems = build("unimodal", seed=7)
    prompt = torch.tensor([[5, 6, 7], [8, 9, 1], [10, 1, 1], [1, 1, 1]], dtype=torch.int32)
    lens = torch.tensor([3, 2, 1, 0], dtype=torch.int32)
    pen = dict(repetition=1.4, presence=0.5, frequency=0.25)
    bias = torch.linspace(-1, 1, V)
    caps, scores = run(dec, mems, dev, beams, prompt=prompt, prompt_lens=lens, bias=bias, length_penalty=0.7, **pen)
    ref, rs = naive("unimodal", dec, mems, beams, prompt=prompt, prompt_lens=lens, bias=bias, length_penalty=0.7, **pen)
    assert torch.equal(caps, ref) and bool(((scores - rs).abs() <= 1e-3).all())
    same, _ = run(dec, mems, dev, beams, prompt=prompt[:1].expand(N, -1))
    ref, _ = naive("unimodal", dec, mems, beams, prompt=prompt[:1].expand(N, -1))
    assert torch.equal(same, ref)


@pytest.mark.parametrize("beams", [1, 3])
def test_grammar(dev, beams):
    """Words alternate between two classes, and a third word has to be <eos>."""
    dec, mems = build("unimodal", seed=8)
    allowed = torch.zeros(5, V, dtype=torch.bool)
    allowed[0, 4:20] = allowed[1, 20:] = allowed[2, 4:20] = True
    allowed[3, EOS] = allowed[4, EOS] = True
    trans = torch.tensor([1, 2, 3, 4, 4], dtype=torch.int32)[:, None].expand(5, V).contiguous()
    caps, scores = run(dec, mems, dev, beams, allowed=allowed, transitions=trans)
    ref, rs = naive("unimodal", dec, mems, beams, allowed=allowed, transitions=trans)
    assert torch.equal(caps, ref) and bool(((scores - rs).abs() <= 1e-3).all())
    assert bool((caps[:, 4] == EOS).all()) and bool((caps[:, 5:] == PAD).all())
    none = torch.zeros(V, dtype=torch.bool)  # nothing allowed: the captions end at once
    caps, _ = run(dec, mems, dev, beams, allowed=none)
    assert bool((caps[:, 1] == EOS).all()) and bool((caps[:, 2:] == PAD).all())


@pytest.mark.parametrize("beams", [1, 3])
@pytest.mark.parametrize("outside", [-1, 1, 1 << 30])
def test_leaving_the_grammar(dev, beams, outside):
    """A transition to a state that the grammar does not have: everything is allowed from then on."""
    dec, mems = build("unimodal", seed=8)
    allowed = torch.zeros(2, V, dtype=torch.bool)
    allowed[0, 4:20] = allowed[1] = True
    ones = torch.ones(2, V, dtype=torch.int32)
    prompt = torch.full((N, 1), 5, dtype=torch.int32)
    for kw in ({}, {"prompt": prompt}):
        want = run(dec, mems, dev, beams, allowed=allowed, transitions=ones, **kw)
        got = run(dec, mems, dev, beams, allowed=allowed[:1], transitions=torch.full_like(ones[:1], outside), **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_prompt_that_fills_the_caption(dev):
    dec, mems = build("unimodal", seed=9)
    prompt = torch.randint(4, V, (N, L - 1), dtype=torch.int32)
    caps, scores = run(dec, mems, dev, 2, prompt=prompt)
    assert torch.equal(caps[:, 1:], prompt) and bool((scores == 0).all())
    lens = torch.tensor([L - 1, 0, L - 2, 3], dtype=torch.int32)
    caps, scores = run(dec, mems, dev, 2, prompt=prompt, prompt_lens=lens)
    ref, rs = naive("unimodal", dec, mems, 2, prompt=prompt, prompt_lens=lens)
    assert torch.equal(caps, ref) and bool(((scores - rs).abs() <= 1e-3).all())


def test_under_autocast_and_refusals(dev):
    dec, mems = build("unimodal", seed=10)
    g = copy.deepcopy(dec).float().to(dev)
    args = [t.to(dev, torch.float32) if t.is_floating_point() else t.to(dev) for t in mems]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        caps, scores = g.generate(*args, BOS, EOS, PAD, L, beams=3)
    assert caps.shape == (N, L) and bool(torch.isfinite(scores).all()) and bool((caps[:, 0] == BOS).all())
    for kw in (dict(beams=0), dict(beams=V + 1), dict(prompt=torch.zeros(N, L, dtype=torch.int32)),
               dict(prompt_lens=torch.zeros(N, dtype=torch.int32)), dict(allowed=torch.ones(2, V, dtype=torch.bool)),
               dict(transitions=torch.zeros(1, V, dtype=torch.int32)), dict(beams=2, repetition=torch.ones(2 * N)),
               dict(beams=2, bias=torch.zeros(2 * N, V)), dict(allowed=torch.ones(V + 1, dtype=torch.bool))):
        with pytest.raises(ValueError):
            g.generate(*args, BOS, EOS, PAD, L, **kw)
    g.train()
    with pytest.raises(RuntimeError):
        g.generate(*args, BOS, EOS, PAD, L)


def test_dvc_inference_with_beams(dev):
    """The DVC wrapper's inference decodes by ``generate`` when its options ask for it; without them as before."""
    torch.manual_seed(0)
    model = PKG.dvc_core.build_dvc(d_model=128, num_queries=10, num_classes=5, T=64, enc_layers=1, dec_layers=2,
                                   caption_depth=2, vocab_size=120, seq_len=12, ff_dim=256).to(dev).eval()
    batch = PKG.dvc_core.synthetic_dvc_batch(2, T=64, feature_dim=128, vocab_size=120, seq_len=12, device=dev)
    with torch.no_grad():
        a = model(batch, is_training=False)
        model.caption_options = dict(beams=1)
        b = model(batch, is_training=False)
        model.caption_options = dict(beams=4, repetition=1.2)
        c = model(batch, is_training=False)
    assert torch.equal(a[1], b[1])
    assert c[1].shape == a[1].shape and c[0]['pred_captions'].shape == a[0]['pred_captions'].shape
    assert bool(torch.isfinite(c[0]['pred_captions']).all())


@pytest.mark.parametrize("kind", ["sparse", "multimodal"])
def test_the_other_wrappers_with_beams(dev, golden, kind):
    import test_dvc as T
    g = golden("sparse_dvc_f64" if kind == "sparse" else "mm_dvc_f64")
    model = T._load(T.build_sparse_dvc("cpu") if kind == "sparse" else T.build_mm_dvc("cpu"), g["state_dict"])
    model = model.float().to(dev).eval()

    def single(x):
        if isinstance(x, torch.Tensor):
            return x.to(dev).float() if x.is_floating_point() else x.to(dev)
        if isinstance(x, dict):
            return {k: single(v) for k, v in x.items()}
        return [single(v) for v in x] if isinstance(x, list) else x

    obj = single(dict(g["obj"]))
    kw = dict(is_training=False, val_mode="one_by_one") if kind == "sparse" else dict(is_training=False)
    with torch.no_grad():
        a = model(obj, **kw)
        model.caption_options = dict(beams=1)
        b = model(obj, **kw)
        model.caption_options = dict(beams=3, length_penalty=1.0)
        c = model(obj, **kw)
    assert torch.equal(a[1], b[1])
    assert c[1].shape == a[1].shape and bool(torch.isfinite(c[0]['pred_captions']).all())


def test_what_stands_behind_a_prompt_does_not_count(dev):
    """Numbers that are no words behind prompt_lens; words that are none within them are refused before they are looked up."""
    dec, mems = build("unimodal", seed=7)
    lens = torch.tensor([3, 2, 1, 0], dtype=torch.int32)
    prompt = torch.tensor([[5, 6, 7], [8, 9, -1], [10, V, 1 << 20], [-5, 99, V]])
    clean = torch.tensor([[5, 6, 7], [8, 9, PAD], [10, PAD, PAD], [PAD, PAD, PAD]])
    for beams in (1, 2):
        got, want = (run(dec, mems, dev, beams, prompt=p, prompt_lens=lens) for p in (prompt, clean))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        with pytest.raises(ValueError):
            run(dec, mems, dev, beams, prompt=prompt, prompt_lens=lens + 1)


@pytest.mark.parametrize("beams", [1, 3])
def test_captured_and_replayed(dev, beams):
    """The whole search as one graph, a prompt included, replayed over other memories."""
    dec, mems = build("unimodal", seed=7)
    g = copy.deepcopy(dec).float().to(dev)
    mem, mask = mems[0].to(dev, torch.float32), mems[1].to(dev)
    prompt = torch.full((N, 2), 5, dtype=torch.int32, device=dev)
    call = lambda: g.generate(mem, mask, BOS, EOS, PAD, L, beams=beams, prompt=prompt)  # noqa: E731
    call()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = call()
    for it in range(3):
        mem.copy_(torch.randn(mem.shape, generator=torch.Generator().manual_seed(it)))
        want = call()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("outside", [2 ** 32, -2 ** 32, 2 ** 63 - 1, -2 ** 63])
def test_transitions_of_64_bits_leave_the_grammar(dev, outside):
    """States that 32 bits would wrap into the grammar."""
    dec, mems = build("unimodal", seed=8)
    allowed = torch.zeros(1, V, dtype=torch.bool)
    allowed[0, 4:20] = True
    for beams in (1, 3):
        want = run(dec, mems, dev, beams, allowed=allowed, transitions=torch.full((1, V), -1))
        got = run(dec, mems, dev, beams, allowed=allowed, transitions=torch.full((1, V), outside))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    stays = run(dec, mems, dev, 1, allowed=allowed, transitions=torch.zeros(1, V, dtype=torch.int64))
    assert not torch.equal(stays[0], got[0])  # (leaving the grammar makes a difference here)


@pytest.mark.parametrize("kind", ["unimodal", "multimodal"])
@pytest.mark.parametrize("length", [1, 2, L])
def test_wrappers_get_the_greedy_outputs_with_one_beam(dev, kind, length):
    """What the DVC wrappers take from an inference pass, with caption_options and without: the captions, and the
    decoder's input that pred_captions is computed from."""
    dec, mems = build(kind, seed=6)
    g = copy.deepcopy(dec).float().to(dev)
    args = [t.to(dev, torch.float32) if t.is_floating_point() else t.to(dev) for t in mems]

    vocab = {"<bos>": BOS, "<eos>": EOS, "<pad>": PAD}
    a = M.dvc_common.decode_captions(g, args, vocab, length, False, None)
    b = M.dvc_common.decode_captions(g, args, vocab, length, False, dict(beams=1))
    assert torch.equal(a[0], b[0])
    assert (a[1] is None) == (b[1] is None) == (length == 1)
    if length > 1:
        assert a[1].dtype == b[1].dtype and torch.equal(a[1], b[1])


@pytest.mark.parametrize("amp", [False, True])
def test_captured_over_a_large_vocabulary(dev, amp):
    """A vocabulary over which the library's choice of the beams takes several workgroups a row, with penalties, a bias and
    a grammar of one state; every replay over other memories, eager calls between."""
    torch.manual_seed(3)
    vocab, n, length = 10000, 6, 8
    dec = M.unimodal_caption_decoder.UnimodalCaptionDecoder(vocab, d_model=64, depth=2, num_heads=2).eval().to(dev)
    with torch.no_grad():
        dec.head.weight.mul_(20.0)
    mem = torch.randn(n, 15, 64, device=dev)
    allowed = torch.rand(vocab, device=dev) < 0.8
    bias = torch.randn(vocab, device=dev)
    kw = dict(beams=4, repetition=1.3, presence=0.2, bias=bias, allowed=allowed, length_penalty=0.5)

    def call():
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=amp, cache_enabled=False):
            return dec.generate(mem, None, BOS, EOS, PAD, length, **kw)

    call()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = call()
    for it in range(4):
        mem.copy_(torch.randn(mem.shape, generator=torch.Generator().manual_seed(it)))
        want = call()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), it
