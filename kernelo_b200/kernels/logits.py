"""What a request asks of its logits before they are sampled: penalties for
repeated tokens, biases of single ones and a grammar's mask, in one pass.

:func:`adjust_logits` takes the logits of a step, one row per request, and what
each request holds on the device: its history of tokens, its factors, its
biases, the mask that its grammar allows now. ``softmax`` (``kernels/softmax.py``)
makes probabilities of the result.
"""

from __future__ import annotations

import torch

from kernelo_b200.kernels.attention import _check_output, _empty_like
from kernelo_b200.runtime import native

MAX_BIASES = 16384


def _check_rows(name: str, t: torch.Tensor, logits: torch.Tensor, dtype: torch.dtype, ndim: int, rows: int | None) -> None:
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.get_device() != logits.get_device():
        raise ValueError(f"{name} must be on {logits.device}, got {t.device}")
    if t.ndim != ndim or (rows is not None and t.shape[0] != rows):
        want = "rows" if rows is None else rows
        raise ValueError(f"{name} must have shape ({want}{', ' + 'columns' if ndim == 2 else ''}), got {tuple(t.shape)}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} must have contiguous {'rows' if ndim == 2 else 'elements'}")


def _check_logits(logits: torch.Tensor) -> None:
    if logits.ndim != 2:
        raise ValueError(f"expected logits (rows, vocabulary), got shape {tuple(logits.shape)}")
    if not logits.is_cuda:
        raise ValueError(f"logits must be a CUDA tensor, got {logits.device}")
    if logits.stride(1) != 1 and logits.shape[1] > 1:
        raise ValueError("logits must have contiguous rows. Pass logits.contiguous() explicitly.")


def _ints(t: torch.Tensor | None, device: int, shape: tuple, dtype: torch.dtype = torch.int32) -> bool:
    """Whether an optional operand of one dimension is right."""
    return t is None or (t.dtype is dtype and t.get_device() == device and t.shape == shape and t.is_contiguous())


def _history(tokens, token_lens, prompt_lens, repetition, frequency, presence, device: int, row: tuple) -> bool:
    if tokens is None:
        return token_lens is None and prompt_lens is None and repetition is None and frequency is None and presence is None
    return (token_lens is not None and tokens.dtype is torch.int32 and tokens.get_device() == device and tokens.ndim == 2
            and tokens.shape[0] == row[0] and tokens.stride(1) == 1 and _ints(token_lens, device, row)
            and _ints(prompt_lens, device, row) and _ints(repetition, device, row, torch.float32)
            and _ints(frequency, device, row, torch.float32) and _ints(presence, device, row, torch.float32))


def _lists(tokens, values, device: int, rows: int) -> bool:
    if tokens is None or values is None:
        return tokens is values
    return (tokens.dtype is torch.int32 and values.dtype is torch.float32 and tokens.get_device() == device
            and values.get_device() == device and tokens.ndim == 2 and tokens.shape == values.shape
            and tokens.shape[0] == rows and tokens.shape[1] <= MAX_BIASES and tokens.stride(1) == 1 == values.stride(1))


def _masks(allowed, allowed_rows, device: int, row: tuple, vocab: int) -> bool:
    if allowed is None:
        return allowed_rows is None
    return (allowed.dtype is torch.int32 and allowed.get_device() == device and allowed.ndim == 2 and allowed.stride(1) == 1
            and allowed.shape[1] * 32 >= vocab and (allowed_rows is not None or allowed.shape[0] == row[0])
            and _ints(allowed_rows, device, row))


def _check_all(logits, tokens, token_lens, prompt_lens, repetition, frequency, presence, bias_tokens, bias_values, allowed,
               allowed_rows) -> None:
    _check_logits(logits)
    rows, vocab = logits.shape
    if (tokens is None) != (token_lens is None):
        raise ValueError("tokens and token_lens go together")
    if tokens is not None:
        _check_rows("tokens", tokens, logits, torch.int32, 2, rows)
        _check_rows("token_lens", token_lens, logits, torch.int32, 1, rows)
        if prompt_lens is not None:
            _check_rows("prompt_lens", prompt_lens, logits, torch.int32, 1, rows)
        if repetition is not None:
            _check_rows("repetition", repetition, logits, torch.float32, 1, rows)
        if frequency is not None:
            _check_rows("frequency", frequency, logits, torch.float32, 1, rows)
        if presence is not None:
            _check_rows("presence", presence, logits, torch.float32, 1, rows)
    elif not (prompt_lens is None and repetition is None and frequency is None and presence is None):
        raise ValueError("penalties need tokens and token_lens")
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values go together")
    if bias_tokens is not None:
        _check_rows("bias_tokens", bias_tokens, logits, torch.int32, 2, rows)
        _check_rows("bias_values", bias_values, logits, torch.float32, 2, rows)
        if bias_tokens.shape != bias_values.shape:
            raise ValueError(f"bias_tokens and bias_values must have one shape, got {tuple(bias_tokens.shape)} and "
                             f"{tuple(bias_values.shape)}")
        if bias_tokens.shape[1] > MAX_BIASES:
            raise ValueError(f"a row may have {MAX_BIASES} biases at most, got {bias_tokens.shape[1]}")
    if allowed is not None:
        _check_rows("allowed", allowed, logits, torch.int32, 2, rows if allowed_rows is None else None)
        if allowed.shape[1] * 32 < vocab:
            raise ValueError(f"allowed has {allowed.shape[1]} words for {vocab} tokens")
        if allowed_rows is not None:
            _check_rows("allowed_rows", allowed_rows, logits, torch.int32, 1, rows)
    elif allowed_rows is not None:
        raise ValueError("allowed_rows needs allowed")


def adjust_logits(
    logits: torch.Tensor,
    *,
    tokens: torch.Tensor | None = None,
    token_lens: torch.Tensor | None = None,
    prompt_lens: torch.Tensor | None = None,
    repetition: torch.Tensor | None = None,
    frequency: torch.Tensor | None = None,
    presence: torch.Tensor | None = None,
    bias_tokens: torch.Tensor | None = None,
    bias_values: torch.Tensor | None = None,
    allowed: torch.Tensor | None = None,
    allowed_rows: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Logits ``(rows, vocabulary)`` after penalties, biases and masks, in that order, in fp32 and rounded once.

    * ``tokens`` (int32 ``(rows, columns)``) begins with each row's history of
      ``token_lens[r]`` (int32) tokens; the first ``prompt_lens[r]`` of them (none
      by default) are its prompt. ``repetition`` (fp32 ``(rows,)``, positive normal numbers)
      divides the positive logits of all tokens of the history and multiplies the
      others. A token that stands ``n`` times behind the prompt loses
      ``frequency[r] * n + presence[r]`` (fp32 ``(rows,)``).
    * ``bias_values[r, i]`` (fp32 ``(rows, biases)``, 16384 at most) is added to the logit of token
      ``bias_tokens[r, i]`` (int32, negative: none). A token that is listed twice
      gets the last value.
    * ``allowed`` (int32 ``(masks, words)``): where bit ``v % 32`` of word ``v //
      32`` is 0, token ``v`` becomes ``-inf``. Row ``r`` has mask
      ``allowed_rows[r]`` (int32; ``r`` by default); where that is negative or past
      the masks, every token is allowed.

    Token ids outside the vocabulary are ignored, also in a history. ``out`` may
    be ``logits`` itself, and shares no operand's memory otherwise. A row whose mask
    allows nothing is all ``-inf``.
    """
    rows, vocab = logits.shape if logits.ndim == 2 else (0, 0)
    # one expression for what is right, and the reasons only where it is not
    device, row = logits.get_device(), (rows,)
    if not (logits.ndim == 2 and logits.is_cuda and logits.stride(1) == 1 and _history(
            tokens, token_lens, prompt_lens, repetition, frequency, presence, device, row)
            and _lists(bias_tokens, bias_values, device, rows) and _masks(allowed, allowed_rows, device, row, vocab)):
        _check_all(logits, tokens, token_lens, prompt_lens, repetition, frequency, presence, bias_tokens, bias_values, allowed,
                   allowed_rows)
    if out is None:
        out = _empty_like(logits)
    else:
        if out.shape != logits.shape or out.dtype is not logits.dtype or out.get_device() != logits.get_device():
            raise ValueError(f"out must be {logits.dtype} {tuple(logits.shape)} on {logits.device}, got {out.dtype} "
                             f"{tuple(out.shape)} on {out.device}")
        if out.stride(1) != 1 and vocab > 1:
            raise ValueError("out must have contiguous rows")
        same = out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride()
        _check_output("out", out, {} if same else {"logits": logits})
    if logits.numel():
        native.adjust_logits(logits, out, tokens, token_lens, prompt_lens, repetition, frequency, presence, bias_tokens,
                             bias_values, allowed, allowed_rows)
    return out
