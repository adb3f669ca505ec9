"""Beam search and constrained decoding of both caption decoders from a paged cache (``generate``).

The reference decodes greedily, re-running the decoder over the whole prefix for every word
(models/deformable/unimodal_deformable_dvc.py:318-354); ``greedy_decode`` (unimodal_caption_decoder.py) does that
with dense cached rows.  ``generate`` adds prompts, beams, penalties, biases and grammars.  The arithmetic of a
word is the same — its probabilities are the output row of a <pad> probe at its position, over the keys of the
committed words that are not <pad> — but the words' keys and values live in pages (modules/paged_cache.py): a
prompt enters as one chunk, beams share the pages of their common beginning, and a beam that dies frees its
own.  With one beam and no options it picks greedy_decode's words.  No host synchronisation inside the loop; a
prompt's words are checked before it."""
import torch

from .modules.layers import PagedCaptionCache
from .modules.logits import pick_tokens, process_logits

__all__ = ["generate"]


def _grammar(allowed, transitions, vocab, device):
    if allowed is None:
        if transitions is not None:
            raise ValueError("generate: transitions without allowed")
        return None
    if allowed.dim() not in (1, 2) or allowed.shape[-1] != vocab or allowed.dtype != torch.bool:
        raise ValueError(f"generate: allowed must be ({vocab},) or (states, {vocab}) bool; got {tuple(allowed.shape)} "
                         f"{allowed.dtype}")
    allowed = allowed.reshape(-1, vocab)
    if transitions is None:
        if allowed.shape[0] != 1:
            raise ValueError("generate: several states need transitions")
    elif transitions.shape != allowed.shape or transitions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"generate: transitions must be {tuple(allowed.shape)} int32; got {tuple(transitions.shape)} "
                         f"{transitions.dtype}")
    return allowed.to(device)


def _words_known(prompt, vocab):
    """Refuses words outside the vocabulary (on the device an embedding's assertion, which ends the process).  The only
    wait for the host in ``generate``; a captured call goes without."""
    if prompt.numel() and not (prompt.is_cuda and torch.cuda.is_current_stream_capturing()):
        low, high = torch.stack(prompt.aminmax()).tolist()
        if low < 0 or high >= vocab:
            raise ValueError(f"generate: prompt words {low} .. {high} of a vocabulary of {vocab}")


def _next_state(transitions, state, word):
    """A state outside the grammar (everything is allowed there) is not left again."""
    s, last = state.long(), transitions.shape[0] - 1
    return torch.where((s >= 0) & (s <= last), transitions[s.clamp(0, last), word], state)


@torch.no_grad()
def generate(decoder, prime, step, n, bos, eos, pad, length, device, beams=1, prompt=None, prompt_lens=None,
             repetition=None, presence=None, frequency=None, bias=None, allowed=None, transitions=None,
             length_penalty=0.0, page_size=16):
    """Shared loop of both decoders' ``generate``.  ``prime(cache)`` projects the memories; ``step(x, cache)`` runs the
    layers on rows x (rows, R, d).  See ``UnimodalCaptionDecoder.generate``."""
    if beams < 1 or length < 1:
        raise ValueError(f"generate: beams {beams}, length {length}")
    places = decoder.positional_encoding.pos_embedding.shape[1]
    if length > places:  # (on the device a position behind the table is an assertion, which ends the process)
        raise ValueError(f"generate: length {length}, the decoder has {places} positions")
    if decoder.training:
        raise RuntimeError("generate: the decoder is in training mode (its dropout would be applied); call eval()")
    vocab = decoder.vocab_size
    if not all(0 <= w < vocab for w in (bos, eos, pad)):
        raise ValueError(f"generate: <bos> {bos}, <eos> {eos} and <pad> {pad} must be among the {vocab} words")
    if beams > vocab:
        raise ValueError(f"generate: {beams} beams over {vocab} words")
    if beams > 1 and (any(isinstance(x, torch.Tensor) for x in (repetition, presence, frequency))
                      or (bias is not None and bias.dim() > 1)):
        raise ValueError("generate: penalties and biases of single rows need beams = 1")
    allowed = _grammar(allowed, transitions, vocab, device)
    m = 1
    if prompt is not None:
        if prompt.dim() != 2 or prompt.shape[0] != n or 1 + prompt.shape[1] > length:
            raise ValueError(f"generate: prompt must be ({n}, at most {length - 1}); got {tuple(prompt.shape)}")
        if prompt.is_floating_point() or prompt.is_complex():
            raise ValueError(f"generate: prompt must hold whole numbers; got {prompt.dtype}")
        if prompt_lens is not None and prompt_lens.shape != (n,):
            raise ValueError(f"generate: prompt_lens must be ({n},); got {tuple(prompt_lens.shape)}")
        m += prompt.shape[1]
    elif prompt_lens is not None:
        raise ValueError("generate: prompt_lens without prompt")
    rows = n * beams
    captions = torch.full((n, length), pad, dtype=torch.int32, device=device)
    captions[:, 0] = bos
    at = torch.full((n,), m, dtype=torch.int32, device=device)  # the next word's position
    if prompt is not None:
        prompt = prompt.to(device)
        if prompt_lens is not None:
            at = 1 + prompt_lens.to(device=device, dtype=torch.int32).clamp(0, m - 1)
            prompt = prompt.masked_fill(torch.arange(1, m, device=device) >= at[:, None], pad)
        _words_known(prompt, vocab)
        captions[:, 1:m] = prompt
    if n == 0 or length == 1 or m == length and prompt_lens is None:  # no word to pick
        return captions, torch.zeros(n, dtype=torch.float32, device=device)
    cache = PagedCaptionCache(rows, length, page_size, device)
    prime(cache)

    def logits_of(tokens, positions, probe):
        """The vocabulary logits of row ``probe`` of each sequence's chunk."""
        x = decoder.positional_encoding(decoder.target_embedding(tokens.long()), positions=positions)
        x = step(x, cache)
        return decoder.head(x[torch.arange(x.shape[0], device=device), probe])

    # the prompt (or <bos> alone) and its probe as one chunk, on the first row of each sequence's beams
    first = torch.arange(n, device=device) * beams
    lens = torch.zeros(rows, dtype=torch.int32, device=device)
    lens[first] = at
    cache.advance(None, lens, select=beams)
    width = min(m + 1, length)
    pos = torch.arange(width, device=device).expand(n, -1)
    # (a prompt that fills the caption leaves no position for a probe: that row's logits are not used)
    logits = logits_of(captions[:, :width], pos, at.long().clamp(max=width - 1))
    scores = torch.zeros(n, beams, device=device)
    done = at >= length
    state = torch.zeros(n, dtype=torch.int32, device=device) if allowed is not None else None
    if transitions is not None:
        # (cut before they are made 32 bits: 2^32 is no state, and must not become 0)
        transitions = transitions.to(device).clamp(-1, allowed.shape[0]).to(torch.int32)
        for c in range(1, m):  # the prompt's words move the grammar too
            word = captions[:, c].long()
            state = torch.where(c < at, _next_state(transitions, state, word), state)
    opts = dict(repetition=repetition, presence=presence, frequency=frequency, bias=bias, allowed=allowed)
    live = 1  # beams that hold something
    ends = at.clone()  # length of each caption: <bos>, the prompt and the closing <eos> included
    picks = length - (m if prompt_lens is None else 1)  # of the shortest prompt
    for left in range(picks - 1, -1, -1):
        if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            logits = logits.float()
        kw = dict(opts, states=state, tokens=captions[:, 1:], token_lens=at - 1)
        if beams == 1:
            parent = None
            word, logp = pick_tokens(logits, **kw)
            word = torch.where(word < 0, eos, word)  # (nothing allowed: the caption ends)
            scores = scores + torch.where(done, 0.0, logp.clamp(min=-1e30))[:, None]
        else:
            out, _, lse = process_logits(logits, stats=True, **kw)
            # (a row without an allowed word: every difference is -inf - -inf; it ends with <eos> at a price)
            stuck = torch.isneginf(lse)
            logp = torch.where(stuck[:, None], -float("inf"), out - lse[:, None])
            logp[:, eos] = torch.where(stuck, -1e30, logp[:, eos])
            logp.masked_fill_(done[:, None], -float("inf"))
            logp[:, pad] = torch.where(done, 0.0, logp[:, pad])  # a finished caption stays as it is
            cand = (scores[:, :live, None] + logp.view(n, live, vocab)).view(n, live * vocab)
            scores, pick = cand.topk(beams, dim=1)
            parent = (torch.arange(n, device=device)[:, None] * live + pick // vocab).view(rows)
            word = (pick % vocab).view(rows)
            captions, at, done, ends = captions[parent], at[parent], done[parent], ends[parent]
            if state is not None:
                state = state[parent]
        went = ~done  # (a caption that the prompt fills, or that has ended, stays as it is)
        idx = at.long().clamp(max=length - 1)[:, None]
        old = captions.gather(1, idx)
        captions.scatter_(1, idx, torch.where(went[:, None], word[:, None].to(torch.int32), old))
        if transitions is not None:
            state = torch.where(went, _next_state(transitions, state, word), state)
        grow = went & (word != pad)
        at = at + went.to(torch.int32)
        ends = torch.where(went, at, ends)
        done = done | (word == eos) | (at >= length)
        if not left:
            break
        # the chosen word and the probe behind it; a finished caption's rows are computed and dropped
        if parent is not None and live == 1:
            parent = parent * beams  # (the prompt's rows)
        cache.advance(parent, grow)
        live = beams
        tokens = torch.stack([word.to(torch.int32), torch.full_like(at, pad)], 1)
        pos = (at - 1)[:, None].long() + torch.arange(2, device=device)
        logits = logits_of(tokens, pos.clamp(max=length - 1), torch.ones_like(word))
    scores = scores / ends.view(n, beams).float().pow(length_penalty) if length_penalty else scores
    best = scores.argmax(1)
    pick = torch.arange(n, device=device) * beams + best
    return captions[pick], scores.gather(1, best[:, None])[:, 0]
