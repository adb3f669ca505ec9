"""Penalties for repeated tokens, biases and masks of allowed tokens on the caption decoders' logits as one HIP
kernel (csrc/logits_process.hip, include/logits_process.h), with each row's best token and log-sum-exp.

The reference takes the argmax of the softmax as it is (models/deformable/unimodal_deformable_dvc.py:334-338).
Inference only, no CPU implementation; on the current stream, no call waits for the host.
"""
import struct

import torch

from ... import _native

__all__ = ["process_logits", "pick_tokens"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 2, torch.float16: 3}
_ARGS = struct.Struct("=14Q12q3d")  # mfl_logits_args
# a repetition penalty is divided by in float32, where it must be neither zero nor infinite
_MIN_REP, _MAX_REP = 2.0 ** -149, torch.finfo(torch.float32).max


def _penalty(who, name, x, n, default):
    """(per-row tensor or None, scalar)"""
    if x is None:
        return None, default
    if isinstance(x, torch.Tensor):
        if x.dtype != torch.float32 or tuple(x.shape) != (n,):
            raise ValueError(f"{who}: {name} must be a number or ({n},) float32; got {tuple(x.shape)} {x.dtype}")
        return x.contiguous(), default
    x = float(x)
    if x != x or (name == "repetition" and not _MIN_REP <= x <= _MAX_REP):
        raise ValueError(f"{who}: {name} {x}")
    return None, x


def _rows_i32(who, name, t, n):
    if t.dtype != torch.int32 or t.shape != (n,):
        raise ValueError(f"{who}: {name} must be ({n},) int32")
    return t if t.is_contiguous() else t.contiguous()


def _mask(who, allowed, states, n, vocab):
    """(mask, kind, mask rows, elements a row)"""
    if allowed.dtype in (torch.bool, torch.uint8):
        kind, cols = 1, vocab
    elif allowed.dtype == torch.int32:
        kind, cols = 2, (vocab + 31) // 32
    else:
        raise TypeError(f"{who}: allowed must be bool (a token an element) or int32 (32 tokens an element), got "
                        f"{allowed.dtype}")
    if allowed.dim() not in (1, 2) or allowed.shape[-1] != cols:
        raise ValueError(f"{who}: allowed must be ({cols},) or (rows, {cols}); got {tuple(allowed.shape)}")
    rows = 1 if allowed.dim() == 1 else allowed.shape[0]
    if rows < 1 or (states is None and rows not in (1, n)):
        raise ValueError(f"{who}: {rows} mask rows for {n} rows of logits without states")
    return allowed if allowed.is_contiguous() else allowed.contiguous(), kind, rows, cols


def _run(who, logits, tokens, token_lens, repetition, presence, frequency, bias, allowed, states, out, write, stats):
    tag = _DTYPES.get(logits.dtype)
    if tag is None:
        raise TypeError(f"{who}: unsupported dtype {logits.dtype}")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"{who}: logits must be (n, vocab); got {tuple(logits.shape)}")
    n, vocab = logits.shape
    hist = tokens_row = 0
    if tokens is not None:
        if tokens.dim() != 2 or tokens.shape[0] != n:
            raise ValueError(f"{who}: tokens must be ({n}, length); got {tuple(tokens.shape)}")
        if tokens.dtype != torch.int32:
            raise TypeError(f"{who}: tokens must be int32, got {tokens.dtype}")
        hist = tokens.shape[1]
        if hist:
            tokens_row, step = tokens.stride()
            if step != 1:
                tokens = tokens.contiguous()
                tokens_row = hist
        if token_lens is not None:
            token_lens = _rows_i32(who, "token_lens", token_lens, n)
    elif token_lens is not None:
        raise ValueError(f"{who}: token_lens without tokens")
    rep_t, rep = _penalty(who, "repetition", repetition, n, 1.0)
    pres_t, pres = _penalty(who, "presence", presence, n, 0.0)
    freq_t, freq = _penalty(who, "frequency", frequency, n, 0.0)
    _native.inference_only(who, logits, bias, rep_t, pres_t, freq_t, out)
    bias_row = 0
    if bias is not None:
        if bias.dtype != torch.float32:
            raise TypeError(f"{who}: bias must be float32, got {bias.dtype}")
        if bias.shape != (vocab,) and bias.shape != (n, vocab):
            raise ValueError(f"{who}: bias must be ({vocab},) or ({n}, {vocab}); got {tuple(bias.shape)}")
        if bias.stride(-1) != 1 and vocab > 1:
            bias = bias.contiguous()
        bias_row = bias.stride(0) if bias.dim() == 2 else 0
    kind = mask_rows = mask_row = 0
    if allowed is not None:
        allowed, kind, mask_rows, mask_row = _mask(who, allowed, states, n, vocab)
        if states is not None:
            states = _rows_i32(who, "states", states, n)
    elif states is not None:
        raise ValueError(f"{who}: states without allowed")
    if out is not None and (out.shape != (n, vocab) or out.dtype not in _DTYPES or (vocab > 1 and out.stride(1) != 1)):
        raise ValueError(f"{who}: out must be ({n}, {vocab}) with contiguous rows, float32, bfloat16 or float16")
    dev = _native.device_index(who, (("logits", logits), ("tokens", tokens), ("token_lens", token_lens),
                                     ("repetition", rep_t), ("presence", pres_t), ("frequency", freq_t), ("bias", bias),
                                     ("allowed", allowed), ("states", states), ("out", out)))
    if out is not logits and vocab > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    lib = _native.load_library()
    with _native.on_device(dev):
        device = logits.device
        if write and out is None:
            out = torch.empty(n, vocab, dtype=torch.float32, device=device)
        best = rest = None
        bp = rp = 0
        if stats:
            best = torch.empty(n, dtype=torch.int64, device=device)
            rest = torch.empty(n, dtype=torch.float32, device=device)
            bp, rp = best.data_ptr(), rest.data_ptr()
        head = (logits.data_ptr(), 0 if out is None else out.data_ptr(), bp, rp if write else 0, 0 if write else rp,
                tokens.data_ptr() if hist else 0, 0 if token_lens is None else token_lens.data_ptr(),
                0 if rep_t is None else rep_t.data_ptr(), 0 if pres_t is None else pres_t.data_ptr(),
                0 if freq_t is None else freq_t.data_ptr(), 0 if bias is None else bias.data_ptr(),
                0 if allowed is None else allowed.data_ptr(), 0 if states is None else states.data_ptr())
        tail = (n, vocab, tag, 0 if out is None else _DTYPES[out.dtype], logits.stride(0),
                0 if out is None else out.stride(0), hist, tokens_row, bias_row, kind, mask_row, mask_rows, rep, pres, freq)
        args = _ARGS.pack(*head, 0, *tail)
        need = lib.mfl_logits_workspace_bytes(args)
        if need > 0:
            ws = torch.empty(need, dtype=torch.uint8, device=device)
            args = _ARGS.pack(*head, ws.data_ptr(), *tail)
        if need < 0 or lib.mfl_logits_process(args, _native.raw_stream(dev)) != 0:
            raise RuntimeError(f"{who}: " + lib.mfl_logits_last_error().decode(errors="replace"))
    return out, best, rest


def process_logits(logits, *, tokens=None, token_lens=None, repetition=None, presence=None, frequency=None, bias=None,
                   allowed=None, states=None, out=None, stats=False):
    """Penalised, biased and masked logits.

    logits (n, vocab) float32, bfloat16 or float16.  With c the number of times token v occurs in
    tokens[i, :token_lens[i]] (int32; numbers outside the vocabulary count nothing), in float32:
      c > 0:  x = x / repetition if x > 0 else x * repetition;  x -= presence;  x -= frequency * c
      x += bias[v] (float32, (vocab,) or (n, vocab));  x = -inf where the token is not allowed
    ``repetition`` (positive and finite), ``presence``, ``frequency``: numbers or (n,) float32.  ``allowed``: bool, one element a
    token, or int32, 32 tokens an element (token v is bit v % 32 of element v // 32); one mask row for all, one
    for each row, or any number with ``states`` (n,) int32 choosing row i's (outside the mask rows: everything
    is allowed).

    Returns ``out`` (n, vocab), float32 unless one is given (``out=logits`` works in place; other memory must be apart
    from the logits'); with ``stats``
    (out, best, lse): the best token (n,) int64 — the lowest of equals, NaN above all, -1 when nothing is
    left — and the log-sum-exp (n,) float32 of the values before they are rounded to out's type."""
    res = _run("process_logits", logits, tokens, token_lens, repetition, presence, frequency, bias, allowed, states, out,
               True, stats)
    return res if stats else res[0]


def pick_tokens(logits, *, tokens=None, token_lens=None, repetition=None, presence=None, frequency=None, bias=None,
                allowed=None, states=None):
    """(token (n,) int64, its log-probability (n,) float32) of the logits as ``process_logits`` would leave them,
    without writing them: the greedy choice (-1 and -inf where nothing is allowed).  The log-probability is summed
    against the token's own logit, so it keeps its bits however large the logits are."""
    return _run("pick_tokens", logits, tokens, token_lens, repetition, presence, frequency, bias, allowed, states, None,
                False, True)[1:]
