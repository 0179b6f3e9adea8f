"""What is trained on sampled tokens, over the C ABI: logprobs of given tokens with their gradient, the clipped policy
loss and the preference loss (`molla_sample_token_logprobs` and below in include/molla_sample.h, which has the formulas).

They start where the sampling calls stop. A rollout's tokens and old logprobs:

    out = sampler.sample_batch(logits, params, want_logprob=True)
    old = losses.token_logprobs(logits, out["tokens"], temperature=params["temperature"])["logprob"]

(`chosen_logprob` is of the logits as the model gave them; rows drawn at a temperature have the logprobs of that
temperature; greedy rows, of temperature 0, have none and are scored at one above it. These are of the whole distribution: where top-k, top-p,
min-p, penalties or biases took part in the draw, the token was drawn from what they left. A final softcap is applied before
the logits come here: a decode step does so itself (`final_softcap`), nothing here does.) A training step, for logits that an autograd graph made:

    got = losses.policy_loss(logits.detach(), tokens, old, advantage, weight=mask, temperature=temperature, scale=1 / n_tokens)
    logits.backward(got["grad_logits"])

Loss and gradient come from one call; nothing here takes part in autograd. Calls are asynchronous on the
current stream of the logits' device, allocate their outputs from PyTorch and keep nothing, so they can be captured in a graph.
`out=logits.detach()` spares the gradient's memory where the logits' graph does not need their values (a linear head does not; one that
ends in a tanh does, and its backward pass then raises, as after any operation in place).
Rows that cannot be answered say so in `row_status` (capi.ROW_*) and turn the loss to NaN.
"""
from __future__ import annotations

import torch

from . import capi
from .sampler import _ptr

_TYPES = {torch.float32: capi.LOGITS_FP32, torch.bfloat16: capi.LOGITS_BF16, torch.float16: capi.LOGITS_FP16}
_F32, _I32 = torch.float32, torch.int32


def _block(logits: torch.Tensor, tokens: torch.Tensor):
    """(rows, vocabulary, row stride, type, pointers of logits and tokens, device index) of a block that can be read."""
    kind = _TYPES.get(logits.dtype)
    dev = logits.get_device()
    if kind is None or dev < 0 or logits.dim() != 2:
        raise ValueError("logits must be a 2-D fp32, bf16 or fp16 CUDA tensor")
    (B, V), (stride, step) = logits.shape, logits.stride()
    if V == 0:
        raise ValueError("logits need a vocabulary")
    if B and (step != 1 and V > 1 or stride < V and B > 1):
        raise ValueError("logit rows must be contiguous and must not overlap")
    return B, V, stride if stride > V else V, kind, logits.data_ptr(), _values("tokens", tokens, dev, B, _I32), dev


def _values(name: str, t, dev: int, n: int, dtype=_F32, what: str = "row"):
    """The pointer of a value a row, or None."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != (n,) or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} tensor of one value a {what} ({n}) on the logits' device")
    return t.data_ptr()


def _gradient(logits: torch.Tensor, stride: int, out):
    """The gradient's tensor (the caller's, or a new one laid out like the logits) and its row stride."""
    if out is None:
        if logits.is_contiguous():
            return torch.empty_like(logits), stride
        return torch.empty_strided(logits.shape, (stride, 1), dtype=logits.dtype, device=logits.device), stride
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("the gradient must have the logits' shape, type and device")
    if out.numel() and (out.stride(1) != 1 and out.shape[1] > 1 or out.stride(0) < out.shape[1] and out.shape[0] > 1):
        raise ValueError("gradient rows must be contiguous and must not overlap")
    torch.autograd.graph.increment_version(out)   # a graph that kept these values for its own backward pass has to know
    return out, max(out.stride(0), out.shape[1])


def _call(fn, dev: int, *args):
    """A call of the library with the logits' device current."""
    if dev == torch.cuda.current_device():
        rc = fn(*args)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args)
    if rc:
        capi.check(rc)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, temperature: torch.Tensor | None = None,
                   want_entropy: bool = False) -> dict:
    """Logprobs (and entropies) of one given token a row; token -1 is no token. `stats`, and `depth` where entropies are
    wanted, are what `token_logprobs_backward` wants."""
    B, V, stride, kind, x, tok, dev = _block(logits, tokens)
    temp = _values("temperature", temperature, dev, B)
    status = torch.empty_like(tokens)
    stats = tokens.new_empty((B, 2), dtype=_F32)
    logprob, entropy, depth = stats.new_empty((3, B)).unbind(0) if want_entropy else (stats.new_empty(B), None, None)
    if B:
        _call(capi.lib().molla_sample_token_logprobs_with_depth, dev, x, kind, stride, B, V, tok, temp, torch._C._cuda_getCurrentRawStream(dev),
              logprob.data_ptr(), _ptr(entropy), _ptr(depth), stats.data_ptr(), status.data_ptr())
    return dict(logprob=logprob, entropy=entropy, depth=depth, stats=stats, row_status=status)


def token_logprobs_backward(logits: torch.Tensor, tokens: torch.Tensor, scored: dict, grad_logprob: torch.Tensor,
                            grad_entropy: torch.Tensor | None = None, temperature: torch.Tensor | None = None,
                            out: torch.Tensor | None = None) -> torch.Tensor:
    """The logits' gradient of a loss with these derivatives by the rows' logprobs and entropies. `scored` is
    what `token_logprobs` returned for the same logits, tokens and temperatures (without its `depth` the entropies' own rounding
    is in their part of the gradient). `out` may be the logits themselves."""
    B, V, stride, kind, x, tok, dev = _block(logits, tokens)
    temp = _values("temperature", temperature, dev, B)
    g, h = _values("grad_logprob", grad_logprob, dev, B), _values("grad_entropy", grad_entropy, dev, B)
    if grad_logprob is None:
        raise ValueError("grad_logprob is required")
    stats, depth = scored["stats"], scored.get("depth") if h is not None else None
    entropy = scored["entropy"] if h is not None and depth is None else None
    if h is not None and entropy is None and depth is None:
        raise ValueError("derivatives by the entropies need the entropies (want_entropy=True)")
    if stats.shape != (B, 2) or stats.get_device() != dev or stats.dtype != _F32 or not stats.is_contiguous():
        raise ValueError("the stats are of another block of logits")
    of_entropy = _values("entropy", entropy, dev, B) if depth is None else _values("depth", depth, dev, B)
    out, grad_stride = _gradient(logits, stride, out)
    if B:
        L = capi.lib()
        _call(L.molla_sample_token_logprobs_backward if depth is None else L.molla_sample_token_logprobs_backward_with_depth, dev, x, kind, stride,
              B, V, tok, temp, stats.data_ptr(), of_entropy, g, h, torch._C._cuda_getCurrentRawStream(dev), out.data_ptr(), grad_stride)
    return out


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logprob: torch.Tensor, advantage: torch.Tensor,
                weight: torch.Tensor | None = None, ref_logprob: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, entropy_coef: float = 0.0,
                temperature: torch.Tensor | None = None, scale: float = 1.0, grad_scale: float = 1.0,
                want_grad: bool = True, want_entropy: bool = False, out: torch.Tensor | None = None) -> dict:
    """The clipped policy loss with a KL term and an entropy bonus, and the logits' gradient. Rows of weight 0 (prompts,
    padding) and of token -1 are not read. `out` (the gradient's place) may be the logits themselves."""
    B, V, stride, kind, x, tok, dev = _block(logits, tokens)
    if old_logprob is None or advantage is None:
        raise ValueError("old logprobs and advantages are required")
    old, adv = _values("old_logprob", old_logprob, dev, B), _values("advantage", advantage, dev, B)
    w, ref = _values("weight", weight, dev, B), _values("ref_logprob", ref_logprob, dev, B)
    temp = _values("temperature", temperature, dev, B)
    grad, grad_stride = _gradient(logits, stride, out) if want_grad else (None, 0)
    new = torch.empty_like   # (of the allocations PyTorch has the cheapest)
    got = dict(loss=old_logprob.new_empty(()), row_loss=new(old_logprob), logprob=new(old_logprob),
               entropy=new(old_logprob) if want_entropy or entropy_coef else None, kl=new(old_logprob) if ref is not None else None,
               clipped=new(old_logprob, dtype=torch.bool), row_status=new(tokens), grad_logits=grad)
    if B == 0:
        got["loss"].zero_()
        return got
    _call(capi.lib().molla_sample_policy_loss, dev, x, kind, stride, B, V, tok, temp, old, adv, w, ref, clip_low, clip_high, kl_coef,
          entropy_coef, scale, grad_scale, torch._C._cuda_getCurrentRawStream(dev), got["loss"].data_ptr(), got["row_loss"].data_ptr(),
          got["logprob"].data_ptr(), _ptr(got["entropy"]), _ptr(got["kl"]), got["clipped"].data_ptr(), _ptr(grad), grad_stride,
          got["row_status"].data_ptr())
    return got


def preference_loss(logits: torch.Tensor, tokens: torch.Tensor, seq_off: torch.Tensor, ref_logprob: torch.Tensor | None = None,
                    pair_weight: torch.Tensor | None = None, beta: float = 0.1, label_smoothing: float = 0.0,
                    temperature: torch.Tensor | None = None, scale: float = 1.0, grad_scale: float = 1.0,
                    want_grad: bool = True, out: torch.Tensor | None = None) -> dict:
    """The preference loss over pairs of sequences, and the logits' gradient. `seq_off` (int32, 2 x pairs + 1, on the
    device) has the rows where the sequences begin and end, each pair's chosen one before its rejected one. `out` (the gradient's
    place) may be the logits themselves."""
    B, V, stride, kind, x, tok, dev = _block(logits, tokens)
    if not isinstance(seq_off, torch.Tensor) or seq_off.dim() != 1 or len(seq_off) % 2 != 1:
        raise ValueError("seq_off must hold two sequences a pair and where the last one ends")
    pairs = len(seq_off) // 2
    off = _values("seq_off", seq_off, dev, 2 * pairs + 1, _I32, "sequence")
    w, ref = _values("pair_weight", pair_weight, dev, pairs, what="pair"), _values("ref_logprob", ref_logprob, dev, B)
    temp = _values("temperature", temperature, dev, B)
    grad, grad_stride = _gradient(logits, stride, out) if want_grad else (None, 0)
    new = tokens.new_empty
    got = dict(loss=new((), dtype=_F32), pair_loss=new(pairs, dtype=_F32), margin=new(pairs, dtype=_F32), seq_logratio=new(2 * pairs, dtype=_F32),
               logprob=new(B, dtype=_F32), row_status=new(B), pair_status=new(pairs), grad_logits=grad)
    if B == 0:   # (the C entry point would be handed null pointers)
        if pairs:
            raise ValueError("pairs of sequences need rows")
        got["loss"].zero_()
        return got
    ws = capi.lib().molla_sample_preference_workspace_bytes(B)
    buf = new(ws // 4)
    _call(capi.lib().molla_sample_preference_loss, dev, x, kind, stride, B, V, tok, temp, off, pairs, ref, w, beta, label_smoothing, scale,
          grad_scale, buf.data_ptr(), ws, torch._C._cuda_getCurrentRawStream(dev), got["loss"].data_ptr(), got["pair_loss"].data_ptr(),
          got["margin"].data_ptr(), got["seq_logratio"].data_ptr(), got["logprob"].data_ptr(), _ptr(grad), grad_stride, got["row_status"].data_ptr(), got["pair_status"].data_ptr())
    return got
