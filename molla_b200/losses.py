"""What is trained on sampled tokens, over the C ABI: logprobs of given tokens with their gradient, the clipped policy
loss and the preference loss (`molla_sample_token_logprobs` and below in include/molla_sample.h, which has the formulas).

They start where the sampling calls stop. A rollout's tokens and old logprobs:

    out = sampler.sample_batch(logits, params, want_logprob=True)
    old = losses.token_logprobs(logits, out["tokens"], temperature=params["temperature"])["logprob"]

(`chosen_logprob` is of the logits as the model gave them; rows drawn at a temperature have the logprobs of that
temperature.) A training step, for logits that an autograd graph made:

    got = losses.policy_loss(logits.detach(), tokens, old, advantage, weight=mask, scale=1 / n_tokens)
    logits.backward(got["grad_logits"])

Loss and gradient come from one call; nothing here takes part in autograd. Calls are asynchronous on the
current stream of the logits' device, allocate their outputs from PyTorch and keep nothing, so they can be captured in a graph.
Rows that cannot be answered say so in `row_status` (capi.ROW_*) and turn the loss to NaN.
"""
from __future__ import annotations

import torch

from . import capi
from .sampler import _ptr, _stream_ptr

_TYPES = {torch.float32: capi.LOGITS_FP32, torch.bfloat16: capi.LOGITS_BF16, torch.float16: capi.LOGITS_FP16}


def _block(logits: torch.Tensor, tokens: torch.Tensor):
    if logits.dim() != 2 or logits.dtype not in _TYPES or not logits.is_cuda:
        raise ValueError("logits must be a 2-D fp32, bf16 or fp16 CUDA tensor")
    B, V = logits.shape
    if V == 0:
        raise ValueError("logits need a vocabulary")
    if B and (logits.stride(1) != 1 and V > 1 or logits.stride(0) < V and B > 1):
        raise ValueError("logit rows must be contiguous and must not overlap")
    _per_row("tokens", tokens, logits, B, torch.int32)
    return B, V, max(logits.stride(0), V)


def _per_row(name: str, t, logits: torch.Tensor, n: int, dtype=torch.float32, what: str = "row"):
    if t is None:
        return
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.shape != (n,) or t.device != logits.device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} tensor of one value a {what} ({n}) on the logits' device")


def _gradient(logits: torch.Tensor, stride: int, out):
    """The gradient's tensor: the caller's, or a new one laid out like the logits."""
    if out is None:
        return torch.empty_strided(logits.shape, (stride, 1), dtype=logits.dtype, device=logits.device)
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or not out.is_cuda:
        raise ValueError("the gradient must have the logits' shape, type and device")
    if out.numel() and (out.stride(1) != 1 and out.shape[1] > 1 or out.stride(0) < out.shape[1] and out.shape[0] > 1):
        raise ValueError("gradient rows must be contiguous and must not overlap")
    return out


def _call(fn, logits: torch.Tensor, *args):
    """A call of the library with the logits' device current."""
    if logits.device.index == torch.cuda.current_device():
        rc = fn(*args)
    else:
        with torch.cuda.device(logits.device):
            rc = fn(*args)
    capi.check(rc)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, temperature: torch.Tensor | None = None,
                   want_entropy: bool = False) -> dict:
    """Logprobs (and entropies) of one given token a row; token -1 is no token. `stats` is what
    `token_logprobs_backward` wants."""
    B, V, stride = _block(logits, tokens)
    _per_row("temperature", temperature, logits, B)
    new = lambda *shape, dt=torch.float32: torch.empty(shape, dtype=dt, device=logits.device)
    out = dict(logprob=new(B), entropy=new(B) if want_entropy else None, stats=new(B, 2), row_status=new(B, dt=torch.int32))
    if B:
        _call(capi.lib().molla_sample_token_logprobs, logits, _ptr(logits), _TYPES[logits.dtype], stride, B, V, _ptr(tokens),
              _ptr(temperature), _stream_ptr(logits.device), _ptr(out["logprob"]), _ptr(out["entropy"]), _ptr(out["stats"]),
              _ptr(out["row_status"]))
    return out


def token_logprobs_backward(logits: torch.Tensor, tokens: torch.Tensor, scored: dict, grad_logprob: torch.Tensor,
                            grad_entropy: torch.Tensor | None = None, temperature: torch.Tensor | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """The logits' gradient of a loss with these derivatives by the rows' logprobs and entropies. `scored` is
    what `token_logprobs` returned for the same logits, tokens and temperatures. `out` may be the logits themselves."""
    B, V, stride = _block(logits, tokens)
    for name, t in (("temperature", temperature), ("grad_logprob", grad_logprob), ("grad_entropy", grad_entropy)):
        _per_row(name, t, logits, B)
    if grad_logprob is None:
        raise ValueError("grad_logprob is required")
    stats, entropy = scored["stats"], scored["entropy"] if grad_entropy is not None else None
    if grad_entropy is not None and entropy is None:
        raise ValueError("derivatives by the entropies need the entropies (want_entropy=True)")
    if stats.shape != (B, 2) or stats.device != logits.device:
        raise ValueError("the stats are of another block of logits")
    _per_row("entropy", entropy, logits, B)
    out = _gradient(logits, stride, out)
    if B:
        _call(capi.lib().molla_sample_token_logprobs_backward, logits, _ptr(logits), _TYPES[logits.dtype], stride, B, V,
              _ptr(tokens), _ptr(temperature), _ptr(stats), _ptr(entropy), _ptr(grad_logprob), _ptr(grad_entropy),
              _stream_ptr(logits.device), _ptr(out), max(out.stride(0), V))
    return out


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logprob: torch.Tensor, advantage: torch.Tensor,
                weight: torch.Tensor | None = None, ref_logprob: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0,
                temperature: torch.Tensor | None = None, scale: float = 1.0, grad_scale: float = 1.0,
                want_grad: bool = True, want_entropy: bool = False, out: torch.Tensor | None = None) -> dict:
    """The clipped policy loss with a KL term and an entropy bonus, and the logits' gradient. Rows of weight 0 (prompts,
    padding) and of token -1 are not read. `out` (the gradient's place) may be the logits themselves."""
    B, V, stride = _block(logits, tokens)
    for name, t in (("old_logprob", old_logprob), ("advantage", advantage), ("weight", weight), ("ref_logprob", ref_logprob),
                    ("temperature", temperature)):
        _per_row(name, t, logits, B)
    if old_logprob is None or advantage is None:
        raise ValueError("old logprobs and advantages are required")
    grad = _gradient(logits, stride, out) if want_grad else None
    new = lambda *shape, dt=torch.float32: torch.empty(shape, dtype=dt, device=logits.device)
    got = dict(loss=new(), row_loss=new(B), logprob=new(B), entropy=new(B) if want_entropy or entropy_coef != 0 else None,
               kl=new(B) if ref_logprob is not None else None, clipped=new(B, dt=torch.bool), row_status=new(B, dt=torch.int32),
               grad_logits=grad)
    if B == 0:
        got["loss"].zero_()
        return got
    _call(capi.lib().molla_sample_policy_loss, logits, _ptr(logits), _TYPES[logits.dtype], stride, B, V, _ptr(tokens), _ptr(temperature),
          _ptr(old_logprob), _ptr(advantage), _ptr(weight), _ptr(ref_logprob), clip_low, clip_high, kl_coef, entropy_coef, scale,
          grad_scale, _stream_ptr(logits.device), _ptr(got["loss"]), _ptr(got["row_loss"]), _ptr(got["logprob"]),
          _ptr(got["entropy"]), _ptr(got["kl"]), _ptr(got["clipped"]), _ptr(grad), max(grad.stride(0), V) if want_grad else 0,
          _ptr(got["row_status"]))
    return got


def preference_loss(logits: torch.Tensor, tokens: torch.Tensor, seq_off: torch.Tensor, ref_logprob: torch.Tensor | None = None,
                    pair_weight: torch.Tensor | None = None, beta: float = 0.1, label_smoothing: float = 0.0,
                    temperature: torch.Tensor | None = None, scale: float = 1.0, grad_scale: float = 1.0,
                    want_grad: bool = True, out: torch.Tensor | None = None) -> dict:
    """The preference loss over pairs of sequences, and the logits' gradient. `seq_off` (int32, 2 x pairs + 1, on the
    device) has the rows where the sequences begin and end, each pair's chosen one before its rejected one. `out` (the gradient's
    place) may be the logits themselves."""
    B, V, stride = _block(logits, tokens)
    if not isinstance(seq_off, torch.Tensor) or seq_off.dim() != 1 or seq_off.numel() % 2 != 1:
        raise ValueError("seq_off must hold two sequences a pair and where the last one ends")
    pairs = seq_off.numel() // 2
    _per_row("seq_off", seq_off, logits, 2 * pairs + 1, torch.int32, "sequence")
    _per_row("pair_weight", pair_weight, logits, pairs, what="pair")
    for name, t in (("ref_logprob", ref_logprob), ("temperature", temperature)):
        _per_row(name, t, logits, B)
    grad = _gradient(logits, stride, out) if want_grad else None
    new = lambda *shape, dt=torch.float32: torch.empty(shape, dtype=dt, device=logits.device)
    got = dict(loss=new(), pair_loss=new(pairs), margin=new(pairs), seq_logratio=new(2 * pairs), logprob=new(B),
               row_status=new(B, dt=torch.int32), pair_status=new(pairs, dt=torch.int32), grad_logits=grad)
    if B == 0:   # (the C entry point would be handed null pointers)
        if pairs:
            raise ValueError("pairs of sequences need rows")
        got["loss"].zero_()
        return got
    ws = capi.lib().molla_sample_preference_workspace_bytes(B)
    buf = torch.empty(ws, dtype=torch.uint8, device=logits.device)
    _call(capi.lib().molla_sample_preference_loss, logits, _ptr(logits), _TYPES[logits.dtype], stride, B, V, _ptr(tokens), _ptr(temperature),
          _ptr(seq_off), pairs, _ptr(ref_logprob), _ptr(pair_weight), beta, label_smoothing, scale, grad_scale, _ptr(buf), ws,
          _stream_ptr(logits.device), _ptr(got["loss"]), _ptr(got["pair_loss"]), _ptr(got["margin"]), _ptr(got["seq_logratio"]),
          _ptr(got["logprob"]), _ptr(grad), max(grad.stride(0), V) if want_grad else 0, _ptr(got["row_status"]),
          _ptr(got["pair_status"]))
    return got
