"""What a classifier answers and learns from (csrc/gf_output.hip, autograd nodes in csrc/gf_torch.cpp), over rows of logits:

    logp, entropy, top_logp, top_tokens = token_log_probs(logits, tokens, top=K)
    loss = distill_top(logits, indices, values)

The reference feeds its readouts to torch losses and reduces them to an error rate (examples/sourceLocGNN.py:167,
alegnn/modules/evaluation.py:58-71); here an answer is a probability with its alternatives, and those alternatives are what a second network
can be trained on."""
from __future__ import annotations

import torch

from . import _lib
from .functional_seq import _FLOATS, _no_tangent, _require_cuda, _same_device

TOP_MAX = 64
_I64 = (torch.int64,)


def _explain_logits(who, logits, dim, temperature):
    """(V, leading shape) of logits that are fine; raises otherwise."""
    assert logits.dim() >= 1 and -logits.dim() <= dim < logits.dim(), f"{who}: dim {dim} of logits with shape {tuple(logits.shape)}"
    _require_cuda(who, "logits", logits, _FLOATS)
    shape = list(logits.shape)
    V = shape.pop(dim)
    assert V > 0, f"{who}: logits have shape {tuple(logits.shape)}: no outputs to choose from"
    assert V < 2 ** 31 - 2 ** 16, f"{who}: {V} outputs (fewer than 2^31 - 2^16 are supported)"
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"alegnn_amd.{who}: temperature {temperature} (want a number between 1e-30 and 1e30)")
    return V, tuple(shape)


def _explain_tokens(logits, tokens, top, temperature, dim):
    who = "token_log_probs"
    _no_tangent(who, logits=logits)
    V, lead = _explain_logits(who, logits, dim, temperature)
    assert 0 <= top <= min(V, TOP_MAX), f"{who}: top={top} for {V} outputs (want 0..min(V, {TOP_MAX}))"
    assert tuple(tokens.shape) == lead, f"{who}: tokens have shape {tuple(tokens.shape)}, logits {tuple(logits.shape)} with the classes along {dim}"
    _require_cuda(who, "tokens", tokens, _I64)
    _same_device(who, "tokens", tokens, logits)
    raise RuntimeError(f"{who}: refused")


def _explain_distill(logits, indices, values, temperature, dim):
    who = "distill_top"
    _no_tangent(who, logits=logits, values=values)
    _, lead = _explain_logits(who, logits, dim, temperature)
    K = indices.shape[-1] if indices.dim() else 0
    assert 1 <= K <= TOP_MAX, f"{who}: indices have shape {tuple(indices.shape)} (want [..., K] with 1 <= K <= {TOP_MAX})"
    assert tuple(indices.shape) == (*lead, K) and values.shape == indices.shape, (
        f"{who}: indices {tuple(indices.shape)} and values {tuple(values.shape)} for logits {tuple(logits.shape)} with the classes along {dim}")
    _require_cuda(who, "indices", indices, _I64)
    _require_cuda(who, "values", values, _FLOATS)
    _same_device(who, "indices", indices, logits)
    _same_device(who, "values", values, logits)
    if values.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("distill_top: values.requires_grad is not supported (the teacher's outputs are constants); detach them")
    raise RuntimeError(f"{who}: refused")


def token_log_probs(logits, tokens, top=0, temperature=1.0, ignore_index=-100, entropy=True, dim=-1):
    """Log probabilities of the given outputs under softmax(logits / temperature), with the entropy and the `top` best alternatives.

    logits [..., V] in float32, bfloat16 or float16 (the classes along `dim`: 1 for a LocalGNN's B x C x N; another axis than the last
    is copied); tokens [...] int64: the given output of each row.  Returns (logp, entropy, top_logp, top_tokens): float32 [...], float32 [...]
    (None with entropy=False), float32 [..., top] and int64 [..., top] (None with top=0), alternatives in descending order, equal logits
    in ascending index order.
    A row whose token is `ignore_index` has logp 0 (its entropy and alternatives are answered all the same); any other token outside [0, V)
    gives NaN.  -inf marks an output that is ruled out; a row of nothing else has logp -inf, entropy 0 and gradient 0.  A NaN or +inf logit
    makes its row's values NaN.  0 <= top <= min(V, 64).  Differentiable (once, in reverse mode) in logits through logp, entropy and top_logp."""
    host = _lib.host()
    top, temperature = int(top), float(temperature)
    try:
        return host.token_log_probs(logits, tokens, top, temperature, int(ignore_index), bool(entropy), dim)
    except host.Refused:
        pass
    _explain_tokens(logits, tokens, top, temperature, dim)


def distill_top(logits, indices, values, temperature=1.0, tail=False, dim=-1):
    """Distillation loss of every row of logits against a teacher's K best outputs, with q = softmax(logits / temperature).

    logits [..., V] in float32, bfloat16 or float16 (classes along `dim`, as in token_log_probs); indices [..., K] int64 and values [..., K]
    floating point: the teacher's outputs, 1 <= K <= 64.  An index outside [0, V) (say -1) is padding.  Returns the loss [...] in float32.
      tail=False: values are logits (or log probabilities), p = softmax(values / temperature) over the row's entries;
                  loss = sum_k p_k (log p_k - log q[i_k]).
      tail=True:  values are log probabilities (at this temperature), p_k = exp(values_k), and what is left to one is one more outcome:
                  loss = sum_k p_k (log p_k - log q[i_k]) + p_r (log p_r - log q_r), q_r = the mass of the outputs that are not named.
                  (With every output named there are none, and the loss is inf if the values leave any mass, be it by rounding: then take
                  tail=False with values * temperature, which scales them to one.)
    A row without entries (tail=False: without mass) has loss 0 and gradient 0; an index that is named twice counts as two entries.  No factor
    temperature^2 is applied.  Differentiable (once, in reverse mode) in logits; the teacher's values are constants."""
    host = _lib.host()
    temperature = float(temperature)
    try:
        return host.distill_top(logits, indices, values, temperature, bool(tail), dim)
    except host.Refused:
        pass
    _explain_distill(logits, indices, values, temperature, dim)
