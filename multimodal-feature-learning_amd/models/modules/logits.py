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


def _penalty(who, name, x, n, default):
    """(per-row tensor or None, scalar)"""
    if x is None:
        return None, default
    if isinstance(x, torch.Tensor):
        if x.dtype != torch.float32 or tuple(x.shape) != (n,):
            raise ValueError(f"{who}: {name} must be a number or ({n},) float32; got {tuple(x.shape)} {x.dtype}")
        return x.contiguous(), default
    x = float(x)
    if x != x or (name == "repetition" and not x > 0.0):
        raise ValueError(f"{who}: {name} {x}")
    return None, x


def _run(who, logits, tokens, token_lens, repetition, presence, frequency, bias, allowed, states, out, write, stats):
    tag = _DTYPES.get(logits.dtype)
    if tag is None:
        raise TypeError(f"{who}: unsupported dtype {logits.dtype}")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"{who}: logits must be (n, vocab); got {tuple(logits.shape)}")
    n, vocab = logits.shape
    if torch.is_grad_enabled() and (logits.requires_grad or (bias is not None and bias.requires_grad)):
        raise RuntimeError(f"{who}: inference only (no gradient); call it under torch.no_grad()")
    hist = 0
    if tokens is not None:
        if tokens.dim() != 2 or tokens.shape[0] != n:
            raise ValueError(f"{who}: tokens must be ({n}, length); got {tuple(tokens.shape)}")
        if tokens.dtype != torch.int32:
            raise TypeError(f"{who}: tokens must be int32, got {tokens.dtype}")
        hist = tokens.shape[1]
        if hist and tokens.stride(1) != 1:
            tokens = tokens.contiguous()
    if token_lens is not None:
        if tokens is None:
            raise ValueError(f"{who}: token_lens without tokens")
        if token_lens.dtype != torch.int32 or tuple(token_lens.shape) != (n,):
            raise ValueError(f"{who}: token_lens must be ({n},) int32")
        token_lens = token_lens.contiguous()
    rep_t, rep = _penalty(who, "repetition", repetition, n, 1.0)
    pres_t, pres = _penalty(who, "presence", presence, n, 0.0)
    freq_t, freq = _penalty(who, "frequency", frequency, n, 0.0)
    bias_row = 0
    if bias is not None:
        if bias.dtype != torch.float32:
            raise TypeError(f"{who}: bias must be float32, got {bias.dtype}")
        if tuple(bias.shape) not in ((vocab,), (n, vocab)):
            raise ValueError(f"{who}: bias must be ({vocab},) or ({n}, {vocab}); got {tuple(bias.shape)}")
        if bias.stride(-1) != 1 and vocab > 1:
            bias = bias.contiguous()
        bias_row = bias.stride(0) if bias.dim() == 2 else 0
    kind = mask_rows = mask_row = 0
    if allowed is not None:
        if allowed.dtype in (torch.bool, torch.uint8):
            kind, cols = 1, vocab
        elif allowed.dtype == torch.int32:
            kind, cols = 2, (vocab + 31) // 32
        else:
            raise TypeError(f"{who}: allowed must be bool (a token an element) or int32 (32 tokens an element), got "
                            f"{allowed.dtype}")
        if allowed.dim() not in (1, 2) or allowed.shape[-1] != cols:
            raise ValueError(f"{who}: allowed must be ({cols},) or (rows, {cols}); got {tuple(allowed.shape)}")
        allowed = allowed.view(1, cols) if allowed.dim() == 1 else allowed
        mask_rows = allowed.shape[0]
        if mask_rows < 1 or (states is None and mask_rows not in (1, n)):
            raise ValueError(f"{who}: {mask_rows} mask rows for {n} rows of logits without states")
        allowed = allowed.contiguous()
        mask_row = cols
    if states is not None:
        if allowed is None:
            raise ValueError(f"{who}: states without allowed")
        if states.dtype != torch.int32 or tuple(states.shape) != (n,):
            raise ValueError(f"{who}: states must be ({n},) int32")
        states = states.contiguous()
    if out is not None and (tuple(out.shape) != (n, vocab) or out.dtype not in _DTYPES or
                            (vocab > 1 and out.stride(1) != 1)):
        raise ValueError(f"{who}: out must be ({n}, {vocab}) with contiguous rows, float32, bfloat16 or float16")
    dev = _native.device_index(who, (("logits", logits), ("tokens", tokens), ("token_lens", token_lens),
                                     ("repetition", rep_t), ("presence", pres_t), ("frequency", freq_t), ("bias", bias),
                                     ("allowed", allowed), ("states", states), ("out", out)))
    if out is not logits and vocab > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    lib = _native.load_library()
    with _native.on_device(dev):
        if write and out is None:
            out = torch.empty(n, vocab, dtype=torch.float32, device=logits.device)
        best = torch.empty(n, dtype=torch.int64, device=logits.device) if stats else None
        rest = torch.empty(n, dtype=torch.float32, device=logits.device) if stats else None

        def ptr(t):
            return 0 if t is None else t.data_ptr()

        head = (logits.data_ptr(), ptr(out), ptr(best), ptr(rest) if write else 0, 0 if write else ptr(rest),
                ptr(tokens) if hist else 0, ptr(token_lens), ptr(rep_t), ptr(pres_t), ptr(freq_t), ptr(bias), ptr(allowed),
                ptr(states))
        tail = (n, vocab, tag, _DTYPES[out.dtype] if out is not None else 0, logits.stride(0),
                out.stride(0) if out is not None else 0, hist, tokens.stride(0) if hist else 0, bias_row, kind, mask_row,
                mask_rows, rep, pres, freq)
        args = _ARGS.pack(*head, 0, *tail)
        need = lib.mfl_logits_workspace_bytes(args)
        if need > 0:
            ws = torch.empty(need, dtype=torch.uint8, device=logits.device)
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
    ``repetition`` (positive), ``presence``, ``frequency``: numbers or (n,) float32.  ``allowed``: bool, one element a
    token, or int32, 32 tokens an element (token v is bit v % 32 of element v // 32); one mask row for all, one
    for each row, or any number with ``states`` (n,) int32 choosing row i's (outside the mask rows: everything
    is allowed).

    Returns ``out`` (n, vocab), float32 unless one is given (``out=logits`` works in place); with ``stats``
    (out, best, lse): the best token (n,) int64 — the lowest of equals, NaN above all, -1 when nothing is
    left — and the log-sum-exp (n,) float32 of the values before they are rounded to out's type."""
    res = _run("process_logits", logits, tokens, token_lens, repetition, presence, frequency, bias, allowed, states, out,
               True, stats)
    return res if stats else res[0]


def pick_tokens(logits, *, tokens=None, token_lens=None, repetition=None, presence=None, frequency=None, bias=None,
                allowed=None, states=None):
    """(token (n,) int64, its log-probability (n,) float32) of the logits as ``process_logits`` would leave them,
    without writing them: the greedy choice (-1 and -inf where nothing is allowed)."""
    return _run("pick_tokens", logits, tokens, token_lens, repetition, presence, frequency, bias, allowed, states, None,
                False, True)[1:]
