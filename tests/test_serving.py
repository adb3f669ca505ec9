"""Caption serving without a GPU: the headers against the binding, and the refusals of the entry points (in
Python before anything touches a device, in the C-ABI before a launch)."""
import ctypes
import os
import re

import pytest
import torch

from conftest import PKG, ROOT

nat = PKG._native
pc = PKG.models.modules.paged_cache
lg = PKG.models.modules.logits


def test_header_symbols_match_binding_and_library():
    names = set()
    for h in ("paged_cache.h", "logits_process.h"):
        text = open(os.path.join(ROOT, "include", h)).read()
        names |= set(re.findall(r"^(?:const\s+)?[a-z_0-9]+\s*\*?\s*(mfl_\w+)\s*\(", text, re.M))
    assert sorted(names) == sorted(nat.SERVING_SYMBOLS)
    lib = ctypes.CDLL(nat.LIB_PATH)
    for name in names:
        assert hasattr(lib, name), name


# --- paged attention --------------------------------------------------------------------------------

def _att(**kw):
    a = dict(q=torch.zeros(2, 3, 4, 64), k_pages=torch.zeros(5, 2, 16, 64), v_pages=torch.zeros(5, 2, 16, 64),
             table=torch.zeros(2, 2, dtype=torch.int32), kv_lens=torch.zeros(2, dtype=torch.int32))
    a.update(kw)
    return pc.paged_attention(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), a.pop("table"), a.pop("kv_lens"), **a)


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


@pytest.mark.parametrize("err, kw", [
    (TypeError, dict(q=torch.zeros(2, 3, 4, 64, dtype=torch.float64))),
    (TypeError, dict(k_pages=torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16))),
    (TypeError, dict(table=torch.zeros(2, 2, dtype=torch.int64))),
    (TypeError, dict(kv_lens=torch.zeros(2, dtype=torch.int64))),
    (TypeError, dict(starts=torch.zeros(2))),
    (ValueError, dict(q=torch.zeros(2, 3, 4, 32))),
    (ValueError, dict(q=torch.zeros(2, 3, 3, 64))),
    (ValueError, dict(q=torch.zeros(6, 4, 64))),
    (ValueError, dict(q=torch.zeros(3, 3, 4, 64))),
    (ValueError, dict(v_pages=torch.zeros(4, 2, 16, 64))),
    (ValueError, dict(k_pages=torch.zeros(5, 16, 2, 64).transpose(1, 2))),
    (ValueError, dict(k=torch.zeros(2, 3, 2, 64))),
    (ValueError, dict(k=torch.zeros(2, 3, 4, 64), v=torch.zeros(2, 3, 4, 64))),
    (ValueError, dict(kv_lens=_i(3))),
    (ValueError, dict(table=_i(2))),
    (ValueError, dict(offsets=_i(3))),
    (ValueError, dict(q=torch.zeros(6, 4, 64), offsets=_i(2))),
    (ValueError, dict(q=torch.zeros(6, 4, 64), offsets=_i(3), max_rows=-1)),
    (ValueError, dict(out=torch.zeros(2, 3, 4, 32))),
    (RuntimeError, dict(q=torch.zeros(2, 3, 4, 64, requires_grad=True))),
    (RuntimeError, dict()),  # host tensors: there is no CPU implementation
])
def test_attention_refuses(err, kw):
    with pytest.raises(err):
        _att(**kw)


def _att_args(**kw):
    f = dict(q=16, kn=0, vn=0, kp=16, vp=16, out=16, ws=16, table=16, kv_lens=16, starts=0, offsets=0, n=2, rows=3,
             total=0, heads=4, kv_heads=2, dim=64, pages=5, page_size=16, width=2, max_kv=32, q_seq=768, q_row=256,
             q_head=64, k_seq=0, k_row=0, k_head=0, v_seq=0, v_row=0, v_head=0, dtype=2, causal=1, zero_tail=0,
             scale=0.125)
    f.update(kw)
    return pc._ARGS.pack(*f.values())


@pytest.mark.parametrize("kw", [
    dict(dtype=1), dict(dtype=9), dict(n=-1), dict(rows=-1), dict(heads=3), dict(kv_heads=0), dict(dim=0), dict(dim=136),
    dict(dim=4), dict(dim=60), dict(page_size=0), dict(page_size=24), dict(page_size=2048), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(kn=16), dict(q_row=3), dict(q=8),
    dict(kp=24), dict(width=1 << 27), dict(rows=1 << 31), dict(q=0), dict(table=0), dict(kv_lens=0),
    dict(n=1 << 30, rows=1 << 20), dict(ws=0, max_kv=1 << 20, width=1 << 16, rows=1), dict(pages=1 << 31)])
def test_attention_c_abi_refuses(kw):
    lib = nat.load_library()
    assert lib.mfl_paged_attention(_att_args(**kw), None) == 1
    assert b"mfl_paged_attention" in lib.mfl_paged_last_error()


def test_attention_c_abi_empty_calls_and_workspace():
    lib = nat.load_library()
    assert lib.mfl_paged_attention(_att_args(n=0), None) == 0
    assert lib.mfl_paged_attention(_att_args(rows=0), None) == 0
    assert lib.mfl_paged_attention(None, None) == 1
    assert lib.mfl_paged_attention_workspace_bytes(_att_args(dim=60)) == -1
    assert lib.mfl_paged_attention_workspace_bytes(_att_args()) == 0
    assert lib.mfl_paged_attention_workspace_bytes(_att_args(rows=1, width=1 << 16, max_kv=1 << 20)) > 0


def test_attention_c_abi_refuses_a_join_past_the_launch_limit():
    """Packed rows behind max_rows are joined too (marked as not computed): as many as one launch takes."""
    lib = nat.load_library()
    kw = dict(offsets=16, n=1, rows=1, heads=8, kv_heads=8, dim=128, width=1 << 16, max_kv=1 << 20)
    assert lib.mfl_paged_attention_workspace_bytes(_att_args(total=1 << 20, **kw)) > 0
    assert lib.mfl_paged_attention_workspace_bytes(_att_args(total=1 << 24, **kw)) == -1
    assert lib.mfl_paged_attention(_att_args(total=1 << 24, **kw), None) == 1
    assert b"one launch" in lib.mfl_paged_last_error()


# --- pages -------------------------------------------------------------------------------------------

def _upd(**kw):
    a = dict(data=torch.zeros(1, 2, 6, 2, 16, 8), table=_i(3, 2), lens=_i(3), refs=_i(6))
    a.update(kw)
    return pc.pages_update(a.pop("data"), a.pop("table"), a.pop("lens"), a.pop("refs"), **a)


@pytest.mark.parametrize("err, kw", [
    (TypeError, dict(table=torch.zeros(3, 2))), (TypeError, dict(lens=torch.zeros(3, dtype=torch.int64))),
    (TypeError, dict(parents=torch.zeros(3, dtype=torch.int64))), (ValueError, dict(table=_i(3))),
    (ValueError, dict(lens=_i(2))), (ValueError, dict(refs=_i(5))), (ValueError, dict(refs=_i(6, 1))),
    (ValueError, dict(new_lens=_i(4))), (ValueError, dict(data=torch.zeros(2, 6, 2, 16, 8))),
    (ValueError, dict(data=torch.zeros(1, 2, 6, 2, 16, 3))), (ValueError, dict(page_size=8)),
    (ValueError, dict(data=None)), (RuntimeError, dict())])
def test_update_refuses(err, kw):
    with pytest.raises(err):
        _upd(**kw)


@pytest.mark.parametrize("err, kw", [
    (TypeError, dict(refs=torch.zeros(6))), (TypeError, dict(table=torch.zeros(3, 2))),
    (ValueError, dict(refs=_i(5))), (ValueError, dict(refs=_i(2, 3))), (RuntimeError, dict())])
def test_compact_refuses(err, kw):
    a = dict(data=torch.zeros(1, 2, 6, 2, 16, 8), table=_i(3, 2), refs=_i(6))
    a.update(kw)
    with pytest.raises(err):
        pc.pages_compact(a["data"], a["table"], a["refs"])


@pytest.mark.parametrize("err, kw", [
    (TypeError, dict(src=torch.zeros(2))), (ValueError, dict(dst=_i(3))), (ValueError, dict(src=_i(2, 1))),
    (ValueError, dict(data=None)), (RuntimeError, dict())])
def test_copy_refuses(err, kw):
    a = dict(data=torch.zeros(1, 2, 6, 2, 16, 8), src=_i(2), dst=_i(2))
    a.update(kw)
    with pytest.raises(err):
        pc.pages_copy(a["data"], a["src"], a["dst"])


def test_pages_c_abi_refuses():
    lib = nat.load_library()
    p = ctypes.c_void_p(16)  # never dereferenced
    good = [p, p, p, None, None, 3, 2, 6, 16, p, 2, 2, 64, p, p, p, p, p, None]
    for at, val in [(5, -1), (5, 1 << 21), (6, -1), (7, -1), (7, 1 << 31), (8, 0), (8, 24), (8, 2048), (10, 0), (11, 0),
                    (12, 8), (12, 24), (9, ctypes.c_void_p(24)), (0, None), (1, None), (2, None), (13, None), (14, None),
                    (15, None), (16, None), (17, None), (6, 1 << 28)]:
        a = list(good)
        a[at] = val
        assert lib.mfl_pages_update(*a) == 1, (at, val)
        assert b"mfl_pages_update" in lib.mfl_paged_last_error()
    good = [p, 6, p, 6, p, 2, 1024, p, p, p, p, p, None]
    for at, val in [(0, None), (1, -1), (2, None), (3, -1), (5, 0), (6, 8), (6, 0), (7, None), (8, None), (9, None),
                    (10, None), (11, None)]:
        a = list(good)
        a[at] = val
        assert lib.mfl_pages_compact(*a) == 1, (at, val)
    good = [p, p, 2, p, 2, 6, 1024, None]
    for at, val in [(0, None), (1, None), (2, -1), (3, None), (4, 0), (5, -1), (6, 24)]:
        a = list(good)
        a[at] = val
        assert lib.mfl_pages_copy(*a) == 1, (at, val)
    assert lib.mfl_pages_copy(p, p, 0, p, 2, 6, 1024, None) == 0
    assert lib.mfl_pages_update_workspace_bytes(-1, 4) == -1 and lib.mfl_pages_compact_workspace_bytes(-1) == -1


def test_cache_refuses_page_size():
    with pytest.raises(ValueError):
        pc.PagedKVCache(1, 2, 20, 2, 64, page_size=12, device="cpu")


@pytest.mark.parametrize("page_size", [0, -16, 2048, 1 << 20])
def test_cache_refuses_page_sizes_that_its_functions_refuse(page_size):
    with pytest.raises(ValueError, match="page_size"):
        pc.PagedKVCache(1, 2, 20, 2, 64, page_size=page_size, device="cpu")
    for good in (1, 1024):
        assert pc.PagedKVCache(1, 2, 20, 2, 64, page_size=good, device="cpu").data.shape[4] == good


# --- logits ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("err, kw", [
    (TypeError, dict(logits=torch.zeros(2, 40, dtype=torch.float64))), (ValueError, dict(logits=torch.zeros(40))),
    (ValueError, dict(logits=torch.zeros(2, 0))), (TypeError, dict(tokens=torch.zeros(2, 3, dtype=torch.int64))),
    (ValueError, dict(tokens=_i(3, 3))), (ValueError, dict(token_lens=_i(2))),
    (ValueError, dict(tokens=_i(2, 3), token_lens=_i(3))), (ValueError, dict(repetition=0.0)),
    (ValueError, dict(repetition=float("nan"))), (ValueError, dict(repetition=torch.ones(3))),
    (ValueError, dict(presence=torch.ones(2, dtype=torch.float64))), (TypeError, dict(bias=torch.zeros(40).bfloat16())),
    (ValueError, dict(bias=torch.zeros(41))), (TypeError, dict(allowed=torch.zeros(40))),
    (ValueError, dict(allowed=torch.ones(41, dtype=torch.bool))), (ValueError, dict(allowed=_i(3))),
    (ValueError, dict(allowed=torch.ones(3, 40, dtype=torch.bool))), (ValueError, dict(states=_i(2))),
    (ValueError, dict(allowed=_i(3, 2), states=_i(3))), (ValueError, dict(out=torch.zeros(2, 41))),
    (RuntimeError, dict(logits=torch.zeros(2, 40, requires_grad=True))), (RuntimeError, dict())])
def test_logits_refuse(err, kw):
    kw = dict(kw)
    x = kw.pop("logits", torch.zeros(2, 40))
    with pytest.raises(err):
        lg.process_logits(x, **kw)
    if "out" not in kw:
        with pytest.raises(err):
            lg.pick_tokens(x, **kw)


def _lg_args(**kw):
    f = dict(logits=16, out=32, best=16, lse=16, logprob=0, tokens=16, token_lens=0, rep=0, pres=0, freq=0, bias=0,
             allowed=0, states=0, ws=16, n=2, vocab=40, dtype=0, out_dtype=0, logits_row=40, out_row=40, hist=3,
             tokens_row=3, bias_row=0, kind=0, allowed_row=0, allowed_rows=0, repetition=1.0, presence=0.0, frequency=0.0)
    f.update(kw)
    return lg._ARGS.pack(*f.values())


@pytest.mark.parametrize("kw", [
    dict(n=-1), dict(vocab=-1), dict(vocab=0), dict(hist=-1), dict(dtype=1), dict(out_dtype=1), dict(kind=3),
    dict(kind=1, allowed=16, allowed_rows=0), dict(kind=1, allowed=16, allowed_rows=3, allowed_row=39),
    dict(kind=1, allowed=0, allowed_rows=1), dict(repetition=0.0), dict(out=16, out_dtype=2), dict(logits=0),
    dict(tokens=0), dict(out_row=39), dict(vocab=100000, out_row=100000, ws=0), dict(n=1 << 23, vocab=1 << 30)])
def test_logits_c_abi_refuses(kw):
    lib = nat.load_library()
    assert lib.mfl_logits_process(_lg_args(**kw), None) == 1
    assert b"mfl_logits_process" in lib.mfl_logits_last_error()
    assert lib.mfl_logits_process(None, None) == 1


# --- generate ----------------------------------------------------------------------------------------

def _decoder(vocab=12, d=16):
    return PKG.models.unimodal_caption_decoder.UnimodalCaptionDecoder(vocab, d_model=d, depth=1, num_heads=2).eval()


@pytest.mark.parametrize("beams", [1, 2])
@pytest.mark.parametrize("length_penalty", [0.0, 0.7])
def test_generate_without_a_word_to_pick(beams, length_penalty):
    """Captions of <bos> alone, and prompts that fill them: no decoder pass runs, so the host does."""
    dec, mem = _decoder(), torch.zeros(3, 5, 16)
    none = torch.zeros(3, 0, dtype=torch.int32)
    for kw in (dict(), dict(prompt=none), dict(prompt=none, prompt_lens=_i(3))):
        caps, scores = dec.generate(mem, None, 2, 3, 1, 1, beams=beams, length_penalty=length_penalty, **kw)
        assert caps.tolist() == [[2]] * 3 and scores.tolist() == [0.0] * 3
    caps, scores = dec.generate(mem, None, 2, 3, 1, 3, beams=beams, length_penalty=length_penalty,
                                prompt=torch.full((3, 2), 5, dtype=torch.int32))
    assert caps.tolist() == [[2, 5, 5]] * 3 and scores.tolist() == [0.0] * 3
    caps, scores = dec.generate(mem[:0], None, 2, 3, 1, 4, beams=beams, length_penalty=length_penalty)
    assert caps.shape == (0, 4) and scores.shape == (0,)


def test_generate_refuses_captions_past_the_position_table():
    dec, mem = _decoder(), torch.zeros(3, 5, 16)
    places = dec.positional_encoding.pos_embedding.shape[1]
    prompt = torch.full((3, places - 1), 5, dtype=torch.int32)
    caps, _ = dec.generate(mem, None, 2, 3, 1, places, prompt=prompt)  # (filled by the prompt: nothing runs)
    assert caps.shape == (3, places)
    for kw in (dict(), dict(beams=2), dict(prompt=prompt)):
        with pytest.raises(ValueError, match="positions"):
            dec.generate(mem, None, 2, 3, 1, places + 1, **kw)


@pytest.mark.parametrize("kw", [
    dict(bos=-1), dict(bos=12), dict(eos=-1), dict(eos=12), dict(pad=-1), dict(pad=12),
    dict(prompt=torch.tensor([[4, 5], [6, 12], [4, 4]])), dict(prompt=torch.tensor([[4, -1], [6, 7], [4, 4]])),
    dict(prompt=torch.tensor([[4, 5], [6, 7], [4, 2 ** 32 + 4]])), dict(prompt=torch.full((3, 2), 4.0)),
    dict(prompt=torch.tensor([[4, 99], [6, 7], [4, 4]]), prompt_lens=_i(3) + 2),
    dict(prompt=torch.full((3, 2), 4), prompt_lens=_i(3, 1)), dict(prompt=torch.full((3, 2), 4), prompt_lens=_i(2))])
def test_generate_refuses_words_that_are_none(kw):
    a = dict(bos=2, eos=3, pad=1)
    a.update(kw)
    bos, eos, pad = a.pop("bos"), a.pop("eos"), a.pop("pad")
    for beams in (1, 2):
        with pytest.raises(ValueError):
            _decoder().generate(torch.zeros(3, 5, 16), None, bos, eos, pad, 6, beams=beams, **a)


def test_words_behind_a_prompt_are_not_looked_at():
    """A prompt of length 0 whose tensor holds anything, in a caption that it fills."""
    caps, _ = _decoder().generate(torch.zeros(3, 5, 16), None, 2, 3, 1, 1, prompt=torch.zeros(3, 0, dtype=torch.int64),
                                  prompt_lens=_i(3))
    assert caps.tolist() == [[2]] * 3
    gen = PKG.models.caption_generate
    words = torch.tensor([[4, -7], [99, 99]])
    gen._words_known(words.masked_fill(torch.tensor([[False, True], [True, True]]), 1), 12)
    with pytest.raises(ValueError):
        gen._words_known(words, 12)


@pytest.mark.parametrize("rep", [1e-50, 1e39, float("inf"), -1.0])
def test_logits_refuse_a_repetition_that_float32_does_not_hold(rep):
    for f in (lg.process_logits, lg.pick_tokens):
        with pytest.raises(ValueError):
            f(torch.zeros(2, 40), tokens=_i(2, 3), repetition=rep)
    lib = nat.load_library()
    assert lib.mfl_logits_process(_lg_args(repetition=rep), None) == 1
    assert b"repetition" in lib.mfl_logits_last_error()
    for good in (1e-40, 0.5, 1.0, 3e38):
        with pytest.raises(RuntimeError):  # (host tensors)
            lg.process_logits(torch.zeros(2, 40), tokens=_i(2, 3), repetition=good)
        assert lib.mfl_logits_workspace_bytes(_lg_args(repetition=good)) >= 0


# --- gradients ---------------------------------------------------------------------------------------

def _calls():
    """Every entry point with each of its tensors that could want a gradient."""
    f = torch.zeros
    yield lambda x: _att(q=x), f(2, 3, 4, 64)
    yield lambda x: _att(k_pages=x), f(5, 2, 16, 64)
    yield lambda x: _att(v_pages=x), f(5, 2, 16, 64)
    yield lambda x: _att(k=x, v=f(2, 3, 2, 64)), f(2, 3, 2, 64)
    yield lambda x: _att(k=f(2, 3, 2, 64), v=x), f(2, 3, 2, 64)
    yield lambda x: _att(out=x), f(2, 3, 4, 64)
    yield lambda x: _upd(data=x), f(1, 2, 6, 2, 16, 8)
    yield lambda x: pc.pages_compact(x, _i(3, 2), _i(6)), f(1, 2, 6, 2, 16, 8)
    yield lambda x: pc.pages_copy(x, _i(2), _i(2)), f(1, 2, 6, 2, 16, 8)
    for call in (lg.process_logits, lg.pick_tokens):
        yield call, f(2, 40)
        yield lambda x, call=call: call(f(2, 40), bias=x), f(40)
        for name in ("repetition", "presence", "frequency"):
            yield lambda x, call=call, name=name: call(f(2, 40), tokens=_i(2, 3), **{name: x}), torch.ones(2)
    yield lambda x: lg.process_logits(f(2, 40), out=x), f(2, 40)


@pytest.mark.parametrize("at", range(20))
def test_no_gradient_is_lost_without_a_word(at):
    call, x = list(_calls())[at]
    with pytest.raises(RuntimeError, match="inference only"):
        call(x.clone().requires_grad_())
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU implementation"):
        call(x.clone().requires_grad_())
    ad = torch.autograd.forward_ad
    with ad.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="inference only"):
                call(ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call(x)


def test_every_tensor_is_asked_for_its_gradient():
    assert len(list(_calls())) == 20
