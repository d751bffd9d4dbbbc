"""Sampling of the next tokens on the device: temperature, top-k, top-p and min-p per row, then a
draw by given uniform numbers (so a run is reproduced by its random numbers).  One call of
libb200paged.so; raises if a tensor is not on a CUDA device."""
from __future__ import annotations

import numbers
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _native as N
from .paged_ops import _DTYPES, _on, _one_device, _ptr, _raw_stream, _status_ptr


@dataclass
class SamplingParams:
    """How a request's tokens are drawn.  ``temperature`` 0: the most likely token.  ``top_k`` 0
    or less: no limit.  ``seed`` starts the request's own sequence of random numbers (None:
    the engine gives each request one).  The temperature has to be finite in fp32, in which it is
    used."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: Optional[int] = None

    def __post_init__(self) -> None:
        for name in ("temperature", "top_p", "min_p"):
            if not isinstance(getattr(self, name), numbers.Real):
                raise ValueError(f"{name} must be a number, got {getattr(self, name)!r}")
            try:
                setattr(self, name, float(getattr(self, name)))
            except OverflowError:
                raise ValueError(f"{name} is beyond a float's range") from None
        for name in ("top_k", "seed"):
            if name == "seed" and self.seed is None:
                continue
            if not isinstance(getattr(self, name), numbers.Integral):
                raise ValueError(f"{name} must be a whole number, got {getattr(self, name)!r}")
            setattr(self, name, int(getattr(self, name)))
        # numbers from half a step above the largest fp32 number on become infinite
        if not 0.0 <= self.temperature < 2.0 ** 128 - 2.0 ** 103:
            raise ValueError(f"temperature must be finite in fp32 and at least 0, got {self.temperature}")
        if not 0.0 < self.top_p <= 1.0:
            raise ValueError(f"top_p must be in (0, 1], got {self.top_p}")
        if not 0.0 <= self.min_p <= 1.0:
            raise ValueError(f"min_p must be in [0, 1], got {self.min_p}")


def _check_row(t: Optional[torch.Tensor], dtype: torch.dtype, rows: int, name: str) -> None:
    if t is not None and (t.dtype != dtype or t.shape != (rows,) or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous {dtype} vector of one entry per row")


def sample(logits: torch.Tensor, uniform: torch.Tensor,
           temperature: Optional[torch.Tensor] = None, top_k: Optional[torch.Tensor] = None,
           top_p: Optional[torch.Tensor] = None, min_p: Optional[torch.Tensor] = None
           ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Draw one token per row of ``logits`` (rows, vocab; fp32, bf16 or f16; rows may be strided).

    Tokens are ordered by decreasing logit, ties by index.  top-k (int32, <= 0: off) keeps the
    first k; top-p keeps of those the shortest run from the top that holds top_p of their
    probability; min-p keeps tokens at least min_p times as likely as the most likely one.  The
    token is the first, in index order, whose cumulative probability among the kept ones exceeds
    ``uniform`` (fp32, in [0, 1)).  temperature 0 takes the most likely token.  Parameters are
    per-row device vectors; None leaves a step out.  NaN logits count as masked (-inf).

    Returns (tokens int64, log-probabilities fp32): the latter of the whole vocabulary's softmax
    at the row's temperature (at 1 for temperature 0), before the filters.  A row in which no
    token can be drawn (every logit masked, a parameter that is NaN, a uniform number outside [0, 1),
    a temperature that is negative or infinite) gives token -1, NaN and the status bit
    DEVICE_BAD_SAMPLE.  top_p and min_p outside [0, 1] act as the nearer end."""
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be (rows, vocab) with unit stride along a row")
    if logits.dtype not in _DTYPES:
        raise ValueError(f"unsupported logits dtype {logits.dtype}")
    rows, vocab = logits.shape
    if vocab == 0:
        raise ValueError("logits must have at least one column")
    if uniform is None:
        raise ValueError("uniform random numbers must be given")
    _check_row(uniform, torch.float32, rows, "uniform")
    _check_row(temperature, torch.float32, rows, "temperature")
    _check_row(top_k, torch.int32, rows, "top_k")
    _check_row(top_p, torch.float32, rows, "top_p")
    _check_row(min_p, torch.float32, rows, "min_p")
    dev = _one_device(logits, uniform, temperature, top_k, top_p, min_p)
    tokens = torch.empty(rows, dtype=torch.int64, device=dev)
    logprobs = torch.empty(rows, dtype=torch.float32, device=dev)
    with _on(dev):
        N.check(N.lib().b200_sample(
            logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0), rows, vocab,
            uniform.data_ptr(), _ptr(temperature), _ptr(top_k), _ptr(top_p), _ptr(min_p),
            tokens.data_ptr(), logprobs.data_ptr(), _status_ptr(dev), _raw_stream(dev)))
    return tokens, logprobs
