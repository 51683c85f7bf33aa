"""Drafted tokens: trees of them, and which of them the target model keeps.

A pass that checks drafted tokens brings each slot n rows: row 0 is its last token, whose K and V are not in the cache yet, the
others are drafted ones, row i following row parents[i] < i.  ``draft_tree`` makes the masks and depths that
PagedKV4.append_rope and .attend_tree take in every layer, ``verify_draft`` takes the logits of the rows and says what is kept
and which token follows, PagedKV4.keep drops the rest from the cache (e2e_decoder.PagedDecoder.verify runs all of
it).  The kernels are those of include/sx8_draft.h; no call waits for the device.  The reference decodes
one token a step (scripts/infer_sx8.py:109-173).
"""
from __future__ import annotations

import torch

import _sx8lib as _L
from sx8_paged_kv import _ints

_TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def draft_tree(parents, cu, words=1):
    """Masks (rows, words) int64 and depths (rows,) int32 of the slots' trees: parents (rows,) int32 is the row number in the slot of
    what a row follows (outside 0 .. row - 1: nothing), slot s has the rows cu[s] .. cu[s + 1] - 1 (int32).  Bit
    j % 64 of a mask's word j // 64 is set where row j is the row itself or above it; depth counts the rows above it.  words (1 to
    4) are for slots of up to 64 words rows: later rows get mask 0 and a depth far below zero, so that append_rope and
    attend_tree leave them out.  Rows of no slot: unset."""
    got = _L.py().draft_tree(parents, cu, words)
    if got is not None:
        return got
    if not isinstance(parents, torch.Tensor) or parents.device.type != "cuda":
        raise RuntimeError("parents must be an int32 vector on the GPU")
    device = parents.device
    with torch.cuda.device(device):
        _ints("parents", parents, None, device)
        _ints("cu", cu, None, device)
        mask = torch.empty(parents.numel(), int(words), dtype=torch.int64, device=device)
        depth = torch.empty(parents.numel(), dtype=torch.int32, device=device)
        _L.call("sx8_draft_tree", parents.data_ptr(), cu.data_ptr(), cu.numel() - 1, parents.numel(), int(words), mask.data_ptr(),
                depth.data_ptr(), _L.stream(device))
    return mask, depth


def _matrix(name, t, rows, vocab, device):
    """(rows, vocab) values whose rows the kernels read in place, or a contiguous copy."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or t.dtype not in _TYPES or t.device != device \
            or t.shape[0] != rows or (vocab is not None and t.shape[1] != vocab):
        want = f"({rows}, {'tokens' if vocab is None else vocab})"
        raise RuntimeError(f"{name} must be a {want} float16, bfloat16 or float32 tensor on {device}")
    t = t.resolve_neg()
    # (a row's stride is checked even where there is one row)
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.clone(memory_format=torch.contiguous_format)


def verify_draft(logits, tokens, parents, cu, uniforms=None, temperature=0.0, draft_probs=None, depth=None):
    """Which drafted tokens the target keeps.  logits (rows, vocabulary), fp16, bf16 or float32, are the target's behind each
    row; tokens (rows,) int64; parents and cu as draft_tree takes them; uniforms (rows,) float32 random numbers in [0, 1): a drafted row's
    decides on it, row 0's draws the token that follows; temperature a number or a (slots,) float32 vector.

    Where the temperature is above zero the kept tokens and the one that follows are distributed as if they were drawn
    from softmax(logits / temperature) one after another: a child of the current row is kept if its uniform lies below the
    token's probability; otherwise the token is taken out of the distribution and the next child tried.  Those drafts were
    chosen, not drawn.  With draft_probs (rows, vocabulary), row r the distribution that the children of row r were drawn
    from, child i is kept if uniform * draft_probs(token) < probability, otherwise the distribution becomes
    max(p - draft_probs, 0), scaled.  Where it is not above zero, tokens are kept while they are the first of the largest
    logits (uniforms may be None if that goes for all slots: a number as temperature).  NaN logits count as
    -infinity; a row of -infinities gives no token.  Sums are held in 64 bits.  Every case is written down in include/sx8_draft.h.
    depth (rows,) int32, as draft_tree gives it: a row whose depth is below zero (those past its words) is in no cache and was
    attended by none, so it is never kept, and a slot whose row 0 is one keeps none (counts 0, no token).  A pass over a cache gives it.

    Returns path (rows,) int32: the rows that slot s keeps, in path[cu[s]] .. (row 0 first, then -1); counts (slots,) int32: how
    many; and the tokens that follow, (slots,) int64 (-1: none).  PagedKV4.keep takes path and counts.  Outputs have no gradient."""
    if not isinstance(temperature, torch.Tensor):
        temperature = float(temperature)
    got = _L.py().draft_verify(logits, tokens, parents, cu, uniforms, temperature, draft_probs, depth)
    if got is not None:
        return got
    if not isinstance(logits, torch.Tensor) or logits.device.type != "cuda" or logits.dim() != 2:
        raise RuntimeError("logits must be a (rows, tokens) tensor on the GPU")
    device = logits.device
    with torch.cuda.device(device):
        rows, vocab = logits.shape
        logits = _matrix("logits", logits.detach(), rows, None, device)
        _ints("cu", cu, None, device)
        _ints("parents", parents, rows, device)
        if not isinstance(tokens, torch.Tensor) or tokens.dtype != torch.int64 or tokens.shape != (rows,) \
                or tokens.device != device or not tokens.is_contiguous() or tokens.is_neg():
            raise RuntimeError(f"tokens must be a contiguous int64 vector of {rows} on {device}")
        if depth is not None:
            _ints("depth", depth, rows, device)
        slots = cu.numel() - 1
        temp, number = None, 0.0
        if isinstance(temperature, torch.Tensor):
            temp = _floats("temperature", temperature, slots, device)
        else:
            number = float(temperature)
        if uniforms is not None:
            uniforms = _floats("uniforms", uniforms, rows, device)
        if draft_probs is not None:
            draft_probs = _matrix("draft_probs", draft_probs.detach(), rows, vocab, device)
        path = torch.empty(rows, dtype=torch.int32, device=device)
        counts = torch.empty(slots, dtype=torch.int32, device=device)
        following = torch.empty(slots, dtype=torch.int64, device=device)
        nb = int(_L.lib().sx8_draft_verify_workspace_bytes(slots, rows, vocab))
        ws = torch.empty(max(nb, 0), dtype=torch.uint8, device=device)
        _L.call("sx8_draft_verify_within", logits.data_ptr(), logits.stride(0), _TYPES[logits.dtype], tokens.data_ptr(),
                parents.data_ptr(), _ptr(depth), cu.data_ptr(), slots, rows, vocab, _ptr(uniforms), _ptr(temp), number, _ptr(draft_probs),
                0 if draft_probs is None else draft_probs.stride(0), 0 if draft_probs is None else _TYPES[draft_probs.dtype],
                path.data_ptr(), counts.data_ptr(), following.data_ptr(), ws.data_ptr(), nb, _L.stream(device))
    return path, counts, following


def _ptr(t):
    return None if t is None else t.data_ptr()


def _floats(name, t, n, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.shape != (n,) or t.device != device:
        raise RuntimeError(f"{name} must be a float32 vector of {n} on {device}")
    t = t.detach().resolve_neg()
    return t if t.is_contiguous() else t.contiguous()
