"""Verification of drafted tokens against the target model's probabilities (speculative sampling)."""
import torch

from . import dense_serving as dense
from .cache import _hip, _refuse_grad, pick_impl


def verify_drafts(target, draft, tokens, accept_u, sample_u, impl=None):
    """(accepted (B,) int64, out (B, N + 1) int64) of N drafted tokens (B, N) int64 for B sequences.

    target (B, N + 1, V) holds the target model's probabilities at the positions of the drafts and behind them, draft
    (B, N, V) those that the drafts were drawn from, or None if they were not drawn (they then count as certain); both
    fp32 or both fp16.  accept_u (B, N) and sample_u (B,) are float32 uniforms in [0, 1).

    Draft i is accepted while accept_u_i * draft_i(x_i) < target_i(x_i).  Behind the accepted ones out holds one more
    token, the lowest v whose running sum of weights passes sample_u times their sum: the weights are
    max(target - draft, 0) at the rejected position (the target's row if they are all zero) and the target's row where
    all drafts are accepted; then -1.  The outcome is distributed as the target's own samples.  A token outside
    0 .. V - 1, say -1 behind a sequence's last draft, ends its drafts.  A row with no positive finite sum gives -1.
    Comparisons and sums are in float64.
    """
    if target.dim() != 3 or tokens.dim() != 2 or target.shape[:2] != (tokens.shape[0], tokens.shape[1] + 1):
        raise ValueError("target must be (B, N + 1, V) and tokens (B, N)")
    B, N = tokens.shape
    V = target.shape[2]
    if B < 1 or V < 1:
        raise ValueError("target must hold at least one sequence and one token")
    if target.dtype not in (torch.float16, torch.float32):
        raise ValueError("target must be fp16 or fp32")
    if draft is not None and (draft.shape != (B, N, V) or draft.dtype != target.dtype):
        raise ValueError("draft must be (B, N, V) of target's type, or None")
    if tokens.dtype != torch.int64:
        raise ValueError("tokens must be int64")
    if accept_u.shape != (B, N) or sample_u.shape != (B,) or accept_u.dtype != torch.float32 or sample_u.dtype != torch.float32:
        raise ValueError("accept_u must be (B, N) and sample_u (B,), float32")
    dev = target.device
    if tokens.device != dev or accept_u.device != dev or sample_u.device != dev or (draft is not None and draft.device != dev):
        raise ValueError(f"draft, tokens, accept_u and sample_u must be on target's device, {dev}")
    _refuse_grad(target)
    if draft is not None:
        _refuse_grad(draft)
    if pick_impl(impl, target) == "reference":
        return dense.verify(target, draft, tokens, accept_u, sample_u)
    return _hip().verify(target, draft, tokens, accept_u, sample_u)
