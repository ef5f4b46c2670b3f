"""Drawing an answer from scores: temperature, top-k, top-p, min-p, from given random numbers.

Where the top-K merge (``topk_merge``) ranks, this draws: one index per row of a score matrix
(``score_gemm``, ``mx_score``), so a serving job can explore in proportion to its model's
belief, and logs the probability each answer was drawn with.  The random numbers are the
caller's (one uniform per row), so an answer can be repeated.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import _native as N
from . import reference as R
from .mx import _INT_MAX, _TYPE, _launch, _same_device

Setting = Union[float, int, torch.Tensor]
_SHORT_ROW = 16384  # rows up to this are one workgroup's, without a workspace (the kernel library's own border)


def _setting(name: str, v: Setting, B: int, S: torch.Tensor, dtype, lo: float, hi: float):
    """``(per-row tensor or None, scalar)`` of one setting."""
    if isinstance(v, torch.Tensor):
        if v.dtype != dtype or tuple(v.shape) != (B,) or not v.is_contiguous():
            raise ValueError(f"sample_scores: {name} per row must be contiguous {dtype} [{B}], got {v.dtype} "
                             f"{tuple(v.shape)}")
        _same_device("sample_scores", S, v)
        return v, 0
    v = float(v) if dtype == torch.float32 else int(v)
    if not (lo <= v <= hi) or math.isinf(v):
        raise ValueError(f"sample_scores: {name} = {v} outside [{lo}, {hi}]")
    return None, v


def sample_scores(S: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0,
                  top_p: Setting = 1.0, min_p: Setting = 0.0, with_prob: bool = False
                  ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """One index per row of ``S [B, N]`` (fp32 / bf16 / fp16; rows may be strided), int32 ``[B]``.

    With ``w_i = exp((S_i - max S) / temperature)``, in this order:

    * ``top_k`` > 0 keeps the ``top_k`` largest scores (equal scores: lowest index first);
    * ``top_p`` < 1 keeps of those, best first, the ones before which less than ``top_p`` of their
      total weight lies (always the best one);
    * ``min_p`` > 0 keeps of those the ones with ``w_i >= min_p`` (the best one has ``w = 1``).

    The answer is the first index ``i`` at which the running weight of the kept scores, in index
    order, exceeds ``u`` times their total; ``u`` fp32 ``[B]`` in [0, 1) (below: the first kept index,
    above or NaN: the last).  ``temperature = 0`` takes the largest score, lowest index.  A score of
    -inf or NaN is masked; a row with nothing left answers -1.  If a row holds +inf, only its +inf
    scores have weight.  Weights and sums are held in 64 bits: where ``u`` times the total (or ``top_p`` times it) falls
    within about 1e-12 of the total from a step, either side may be taken.

    Every setting is a number or a per-row tensor (fp32 ``[B]``; ``top_k`` int32 ``[B]``).  Per-row
    values are not checked: a temperature that is not above 0 is greedy, a ``top_k`` <= 0, a ``top_p``
    >= 1 or NaN and a ``min_p`` <= 0 or NaN are off, a ``min_p`` above 1 counts as 1.
    ``with_prob``: also fp32 ``[B]``, the probability the index was drawn with (0 for -1)."""
    if S.dim() != 2 or S.dtype not in _TYPE:
        raise ValueError(f"sample_scores: scores must be fp32 / bf16 / fp16 [B, N], got {S.dtype} {tuple(S.shape)}")
    B, n = S.shape
    if S.numel() and (n > 1 and S.stride(1) != 1 or B > 1 and S.stride(0) < n):
        raise ValueError(f"sample_scores: score rows must be contiguous and apart, got strides {S.stride()}")
    if u.dtype != torch.float32 or tuple(u.shape) != (B,) or not u.is_contiguous():
        raise ValueError(f"sample_scores: u must be contiguous fp32 [{B}], got {u.dtype} {tuple(u.shape)}")
    _same_device("sample_scores", S, u)
    if n > _INT_MAX or B > _INT_MAX or (B > 65535 and n > _SHORT_ROW):
        raise ValueError(f"sample_scores: {B} rows of {n} scores: up to 2^31 - 1 of each, at most 65535 rows longer than "
                         f"{_SHORT_ROW}")
    t, t0 = _setting("temperature", temperature, B, S, torch.float32, 0.0, math.inf)
    k, k0 = _setting("top_k", top_k, B, S, torch.int32, 0, 2**62)
    p, p0 = _setting("top_p", top_p, B, S, torch.float32, 0.0, 1.0)
    m, m0 = _setting("min_p", min_p, B, S, torch.float32, 0.0, 1.0)
    out = torch.empty(B, dtype=torch.int32, device=S.device)
    prob: Optional[torch.Tensor] = torch.empty(B, dtype=torch.float32, device=S.device) if with_prob else None
    if n == 0:
        out.fill_(-1)
        if with_prob:
            prob.zero_()
    elif B and not S.is_cuda:
        i, q = R.sample_scores(S.detach(), u, t0 if t is None else t, k0 if k is None else k, p0 if p is None else p,
                               m0 if m is None else m)
        out.copy_(i)
        if with_prob:
            prob.copy_(q)
    elif B:
        settings = (N.ptr(t), t0, N.ptr(k), k0, N.ptr(p), p0, N.ptr(m), m0)
        ws = None
        if n > _SHORT_ROW:
            size = N.require().fps_sample_scores_ws_bytes(B, n, *settings)
            ws = torch.empty(size, dtype=torch.uint8, device=S.device)
        _launch("sample_scores", S.get_device(), S.data_ptr(), _TYPE[S.dtype], B, n, S.stride(0) if B > 1 else n,
                u.data_ptr(), *settings, out.data_ptr(), N.ptr(prob), N.ptr(ws))
    return (out, prob) if with_prob else out
