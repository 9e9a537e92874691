"""Hot-path operators.

Every function here has two bodies: the sm_100a CUDA kernels in
``rwkv7m_b200.ops.cuda`` (used for every CUDA tensor) and the plain PyTorch
statement in ``rwkv7m_b200.ops.reference`` (used on CPU, and as the oracle the
kernels are tested against).  A CUDA tensor never silently falls back: if the
compiled extension is missing the call raises.  ``reference_mode()`` forces the
PyTorch bodies on any device and exists for the numerics tests.
"""

from __future__ import annotations

import contextlib
from typing import NamedTuple

import torch

from . import reference

_FORCE_REFERENCE = False


@contextlib.contextmanager
def reference_mode(enabled: bool = True):
    """Run every op through its PyTorch statement (numerics oracle)."""
    global _FORCE_REFERENCE
    previous = _FORCE_REFERENCE
    _FORCE_REFERENCE = enabled
    try:
        yield
    finally:
        _FORCE_REFERENCE = previous


def use_cuda(t: torch.Tensor) -> bool:
    return t.is_cuda and not _FORCE_REFERENCE


def _cuda():
    from . import cuda  # noqa: WPS433 (deferred: loads the compiled extension)

    return cuda


def embedding(ids, weight, dtype):
    """Row gather from the embedding table, cast to the compute dtype."""
    if use_cuda(weight):
        return _cuda().embedding(ids, weight, dtype)
    return torch.nn.functional.embedding(ids.long(), weight).to(dtype)


def layer_norm(x, weight, bias, eps=1e-5):
    if use_cuda(x):
        return _cuda().layer_norm(x, weight, bias, eps)
    return reference.layer_norm(x, weight, bias, eps)


def layer_norm_residual(x, weight, bias, eps=1e-5):
    """(LayerNorm(x), x); on CUDA the gradient of the returned x is added inside the LayerNorm backward kernel."""
    if use_cuda(x):
        return _cuda().layer_norm_residual(x, weight, bias, eps)
    return reference.layer_norm(x, weight, bias, eps), x


def shift_mix(x, prev, mix):
    if use_cuda(x):
        return _cuda().shift_mix(x, prev, mix)
    return reference.shift_mix(x, prev, mix)


def linear(x, weight):
    if use_cuda(x):
        return _cuda().linear(x, weight)
    return reference.linear(x, weight)


def linear_relu_sq(x, weight):
    """relu(x @ W.T)**2 (the GEMM epilogue applies the activation on CUDA)."""
    if use_cuda(x):
        return _cuda().linear_relu_sq(x, weight)
    return reference.relu_sq(reference.linear(x, weight))


def linear_add(residual, x, weight):
    """residual + x @ W.T (the GEMM epilogue adds the residual on CUDA)."""
    if use_cuda(x):
        return _cuda().linear_add(residual, x, weight)
    return residual + reference.linear(x, weight)


def ffn(x, w_key, w_value, residual=None):
    """Channel mix: [residual +] relu(x @ Wk.T)**2 @ Wv.T as one autograd node on CUDA."""
    if use_cuda(x):
        return _cuda().ffn(x, w_key, w_value, residual)
    out = reference.linear(reference.relu_sq(reference.linear(x, w_key)), w_value)
    return out if residual is None else residual + out


def lora(x, down, up, mid="none"):
    """Low-rank path act(x @ down.T) @ up.T with weights stored [out,in]; no bias."""
    if use_cuda(x):
        return _cuda().lora(x, down, up, mid)
    return reference.lora(x, down, up, None, mid=mid)


def lora_group(items):
    """Several low-rank paths on inputs of one shape: ``items`` are ``(x, down, up, mid)`` tuples, the result is the list of
    outputs.  On the GPU the down-projections and the up-projections can each run as one grouped launch."""
    if items and use_cuda(items[0][0]):
        return _cuda().lora_group(items)
    return [reference.lora(x, d, u, None, mid=mid) for x, d, u, mid in items]


def tmix_pre(k, v, w_lora, a_lora, vg_lora, v_first, w0, a0, v0, k_k, k_a, n_heads):
    """Everything between the projections and the recurrence, in one pass:

    w = -softplus(-(w0 + w_lora)) - 0.5;  a = sigmoid(a0 + a_lora);
    v = v + (v_first - v) * sigmoid(v0 + vg_lora)   (skipped when ``vg_lora`` is None: layer 0);
    kk = normalize_per_head(k * k_k);  k_mod = k * (1 + (a - 1) * k_a).
    Returns (w, k_mod, v, -kk, kk * a).
    """
    if use_cuda(k):
        return _cuda().tmix_pre(k, v, w_lora, a_lora, vg_lora, v_first, w0, a0, v0, k_k, k_a, n_heads)
    return reference.tmix_pre(k, v, w_lora, a_lora, vg_lora, v_first, w0, a0, v0, k_k, k_a, n_heads)


class inplace_wkv_state:
    """Context: inference calls of the T = 1 recurrence on CUDA update their state argument in place (no-op on CPU)."""

    def __enter__(self):
        self.inner = _cuda().inplace_wkv_state() if torch.cuda.is_available() else None
        if self.inner is not None:
            self.inner.__enter__()

    def __exit__(self, *exc):
        if self.inner is not None:
            self.inner.__exit__(*exc)


def inplace_state_active() -> bool:
    import sys

    mod = sys.modules.get(__name__ + ".cuda")
    return bool(mod is not None and mod.WKV_INPLACE_STATE)


def last_token_state(x, prev):
    """fp32 copy of the last position of x [B, T, C] (the token-shift state of the next call).  Inside
    ``inplace_wkv_state()`` the previous state tensor is overwritten and returned, one kernel instead of a conversion
    plus a copy back into a static buffer; the caller must have consumed ``prev`` already."""
    if inplace_state_active() and prev is not None and prev.dtype == torch.float32 and prev.shape == x[:, -1].shape \
            and not torch.is_grad_enabled():
        prev.copy_(x[:, -1])
        return prev
    return x[:, -1].float()


def flush_deferred():
    """Issue any weight-gradient GEMM that the CUDA path held back during backward (no-op otherwise)."""
    import sys

    mod = sys.modules.get(__name__ + ".cuda")
    if mod is not None:
        mod.flush_deferred()


def _check_wkv_inputs(r, w, k, v, a, b, state0):
    """Shape and dtype contract of the recurrence (reference: src/rwkv7m/kernels/wkv.py validates the same way)."""
    if r.dim() != 4:
        raise ValueError(f"wkv7 vectors must be [B, T, H, N], got {tuple(r.shape)}")
    for name, t in (("w", w), ("k", k), ("v", v), ("a", a), ("b", b)):
        if t.shape != r.shape:
            raise ValueError(f"wkv7: {name} has shape {tuple(t.shape)}, r has {tuple(r.shape)}")
        if t.dtype != r.dtype:
            raise TypeError(f"wkv7: {name} is {t.dtype}, r is {r.dtype}")
    if not r.is_floating_point():
        raise TypeError(f"wkv7 needs floating-point vectors, got {r.dtype}")
    B, _, H, N = r.shape
    if tuple(state0.shape) != (B, H, N, N):
        raise ValueError(f"wkv7: initial state must be [B, H, N, N] = {(B, H, N, N)}, got {tuple(state0.shape)}")


def wkv7(r, w, k, v, a, b, state0):
    """WKV7 recurrence on [B,T,H,N] vectors with an fp32 [B,H,N,N] initial state.  The kernels implement reverse-mode
    differentiation only (a hand-written backward, as the reference's custom VJP, src/rwkv7m/model/wkv.py); forward-mode
    differentiation through a CUDA call raises in autograd, the PyTorch statement on CPU supports both."""
    _check_wkv_inputs(r, w, k, v, a, b, state0)
    from . import backends

    choice = backends.explicit_wkv_backend()      # None: automatic (kernels on CUDA tensors, PyTorch statement on CPU)
    if choice == "ffi" and not _FORCE_REFERENCE:
        return backends.external_wkv7(r, w, k, v, a, b, state0)
    if use_cuda(r) and choice != "reference":
        return _cuda().wkv7(r, w, k, v, a, b, state0, impl=choice)
    if choice == "chunked" and not r.is_cuda and not _FORCE_REFERENCE:
        # the matrix formulation in float64: the same numbers as the step recurrence without a Python loop over the steps
        return reference.wkv7_chunked(r, w, k, v, a, b, state0)
    return reference.wkv7(r, w, k, v, a, b, state0)


def wkv7_sharded(r, w, k, v, neg_kk, kka, initial_state, *, mesh=None, data_axis: str = "data", model_axis: str = "model"):
    """WKV7 on this process's shard of a ``data x model`` layout.  The recurrence never mixes heads or batch rows, so
    with one process per GPU the tensors a rank holds (its batch rows and its heads) are a complete problem: the call is
    the local recurrence, and the mesh arguments only document the partition (the reference needs an explicit shard-map
    boundary here, src/rwkv7m/model/wkv.py:82-130)."""
    del mesh, data_axis, model_axis
    return wkv7(r, w, k, v, neg_kk, kka, initial_state)


def wkv7_gn(r, w, k, v, a, b, state0, g, ln_w, ln_b, r_k, n_heads, eps=64e-5):
    """WKV7 followed by GroupNorm + bonus + gate: ``(out [B,T,C], final_state)``.  On the GPU the two are one autograd
    node, so the gradients that r, k and v receive from both halves are summed inside the WKV7 backward kernel."""
    from . import backends

    choice = backends.explicit_wkv_backend()
    if use_cuda(r) and choice not in ("ffi", "reference"):
        return _cuda().wkv7_gn(r, w, k, v, a, b, state0, g, ln_w, ln_b, r_k, n_heads, eps, impl=choice)
    B, T, H, N = r.shape
    y, sT = wkv7(r, w, k, v, a, b, state0)      # the PyTorch statement, or the backend chosen for the process
    C = H * N
    out = gn_bonus_gate(y.reshape(B, T, C), r.reshape(B, T, C), k.reshape(B, T, C), v.reshape(B, T, C), g,
                        ln_w, ln_b, r_k, n_heads, eps)
    return out, sT


def gn_bonus_gate(y, r, k, v, g, ln_w, ln_b, r_k, n_heads, eps=64e-5):
    if use_cuda(y):
        return _cuda().gn_bonus_gate(y, r, k, v, g, ln_w, ln_b, r_k, n_heads, eps)
    return reference.gn_bonus_gate(y, r, k, v, g, ln_w, ln_b, r_k, n_heads, eps)


def head_loss(hidden, ln_w, ln_b, head_w, targets, mask, chunk=None, eps=1e-5):
    """final LN -> LM head -> (ce_total, ce_count, l2_total, l2_count).

    The [tokens, V] logits are produced chunk by chunk over tokens so the full
    matrix never exists (reference: head chunks, src/rwkv7m/train/nnx_train.py:278-332).
    """
    if use_cuda(hidden):
        return _cuda().head_loss(hidden, ln_w, ln_b, head_w, targets, mask, chunk, eps)
    B, T, C = hidden.shape
    chunk = chunk or T
    totals = None
    for start in range(0, T, chunk):
        h = reference.layer_norm(hidden[:, start : start + chunk], ln_w, ln_b, eps)
        logits = reference.linear(h, head_w)
        part = reference.cross_entropy_l2wrap(
            logits, targets[:, start : start + chunk], None if mask is None else mask[:, start : start + chunk]
        )
        totals = part if totals is None else tuple(a + b for a, b in zip(totals, part))
    return totals


class TokenLogprobs(NamedTuple):
    """Scores of the distribution over the vocabulary, one entry per position: log-probability of the given token, entropy
    in nats, and (with ``top_k > 0``) the most likely ids with their log-probabilities, [..., top_k]."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: torch.Tensor | None = None
    top_logprobs: torch.Tensor | None = None

    @classmethod
    def join(cls, parts, dim=1):
        """The scores of consecutive slices (of time, by default) as one."""
        if len(parts) == 1:
            return parts[0]
        return cls(*(None if field[0] is None else torch.cat(field, dim=dim) for field in zip(*parts)))


TOP_K_MAX = 64            # alternatives of token_logprobs
TEACHER_K_MAX = 256       # alternatives a teacher may give per position


def _check_temperature(temperature):
    t = float(temperature)
    if not 1e-4 <= t <= 1e4:
        raise ValueError(f"temperature must lie between 1e-4 and 1e4, got {temperature}")
    return t


def _check_vocab_input(name, x, what):
    if not torch.is_tensor(x) or not x.is_floating_point():
        raise TypeError(f"{name}: {what} must be a floating-point tensor")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{name}: {what} need a last dimension of at least one, got {tuple(x.shape)}")
    if use_cuda(x) and x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{name}: {what} on a GPU are bfloat16 or float32, got {x.dtype}")


def _check_ids(name, ids, shape, device, what="ids"):
    if not torch.is_tensor(ids) or ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name}: {what} must be an int32 or int64 tensor")
    if tuple(ids.shape) != tuple(shape):
        raise ValueError(f"{name}: {what} have shape {tuple(ids.shape)}, expected {tuple(shape)}")
    if ids.device != device:
        raise ValueError(f"{name}: {what} are on {ids.device}, expected {device}")


def _check_teacher(name, rows_shape, device, teacher_ids, teacher_logits):
    if not torch.is_tensor(teacher_logits) or not teacher_logits.is_floating_point():
        raise TypeError(f"{name}: teacher_logits must be a floating-point tensor")
    if teacher_logits.dim() != len(rows_shape) + 1 or tuple(teacher_logits.shape[:-1]) != tuple(rows_shape):
        raise ValueError(f"{name}: teacher_logits have shape {tuple(teacher_logits.shape)}, expected {tuple(rows_shape)} "
                         "and a dimension of alternatives")
    if not 1 <= teacher_logits.shape[-1] <= TEACHER_K_MAX:
        raise ValueError(f"{name}: a teacher gives between 1 and {TEACHER_K_MAX} alternatives, got {teacher_logits.shape[-1]}")
    if teacher_logits.device != device:
        raise ValueError(f"{name}: teacher_logits are on {teacher_logits.device}, expected {device}")
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: the teacher is not differentiated, detach teacher_logits")
    _check_ids(name, teacher_ids, teacher_logits.shape, device, "teacher_ids")


def _check_mask(name, mask, shape, device):
    if mask is None:
        return
    if not torch.is_tensor(mask) or tuple(mask.shape) != tuple(shape):
        raise ValueError(f"{name}: mask must be a tensor of shape {tuple(shape)}")
    if mask.device != device:
        raise ValueError(f"{name}: mask is on {mask.device}, expected {device}")
    if mask.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: the mask is not differentiated, detach it")


def token_logprobs(logits, ids, *, top_k=0, temperature=1.0) -> TokenLogprobs:
    """Log-probability of ``ids`` [...] under softmax(``logits`` [..., V] / temperature), its entropy, and the ``top_k`` (at
    most 64) most likely ids with their log-probabilities, equal logits in the order of their index.

    fp32 results from bf16 or fp32 logits of any row stride.  An id outside the vocabulary (-1 for padding) is no token:
    log-probability 0, no gradient.  Columns at -inf have probability 0; a row with a NaN or without a finite logit has NaN
    for every result (ids of alternatives are then unspecified, -1 where there is none).  Differentiable in ``logits``
    through ``logprob``, ``entropy`` and ``top_logprobs``; on a GPU a row that no gradient reaches gets zeros whatever it
    holds."""
    _check_vocab_input("token_logprobs", logits, "logits")
    _check_ids("token_logprobs", ids, logits.shape[:-1], logits.device)
    temperature = _check_temperature(temperature)
    if not isinstance(top_k, int) or not 0 <= top_k <= min(TOP_K_MAX, logits.shape[-1]):
        raise ValueError(f"token_logprobs: top_k must be an integer between 0 and {min(TOP_K_MAX, logits.shape[-1])}, got {top_k}")
    if use_cuda(logits):
        return TokenLogprobs(*_cuda().token_logprobs(logits, ids, top_k, temperature))
    return TokenLogprobs(*reference.token_logprobs(logits, ids, top_k, temperature))


def distill_loss(logits, teacher_ids, teacher_logits, mask=None, *, temperature=1.0):
    """Distillation from a teacher's top logits: ``(kd_total, kd_count)``, the sum over positions of
    mask temperature^2 KL(p || softmax(``logits`` [..., V] / temperature)) and the sum of the mask, fp32 scalars.

    p is the softmax of ``teacher_logits`` [..., K] / temperature over the alternatives ``teacher_ids`` [..., K] (1 <= K <=
    256; log-probabilities serve as well as logits, p does not change with a constant).  An id outside the vocabulary or a
    logit of -inf marks an absent alternative; an id that occurs twice counts with both.  A position whose mask is 0 or
    whose teacher is empty adds nothing to ``kd_total`` and gets a zero gradient, whatever its logits hold.  Differentiable
    in ``logits``."""
    _check_vocab_input("distill_loss", logits, "logits")
    _check_teacher("distill_loss", logits.shape[:-1], logits.device, teacher_ids, teacher_logits)
    _check_mask("distill_loss", mask, logits.shape[:-1], logits.device)
    temperature = _check_temperature(temperature)
    if use_cuda(logits):
        return tuple(_cuda().distill_loss(logits, teacher_ids, teacher_logits, mask, temperature))
    return reference.distill_loss(logits, teacher_ids, teacher_logits, mask, temperature)


def _check_head(name, hidden, head_w):
    _check_vocab_input(name, hidden, "hidden states")
    if not torch.is_tensor(head_w) or not head_w.is_floating_point():
        raise TypeError(f"{name}: the head's weight must be a floating-point tensor")
    if head_w.dim() != 2 or head_w.shape[0] < 1 or head_w.shape[1] != hidden.shape[-1]:
        raise ValueError(f"{name}: the head's weight must be [V, {hidden.shape[-1]}], got {tuple(head_w.shape)}")
    if head_w.device != hidden.device:
        raise ValueError(f"{name}: the head's weight is on {head_w.device}, the hidden states are on {hidden.device}")
    if use_cuda(hidden) and head_w.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"{name}: the head's weight on a GPU is bfloat16 or float32, got {head_w.dtype}")


def head_token_logprobs(hidden, head_w, ids, *, temperature=1.0):
    """``(logprob, entropy)`` of :func:`token_logprobs` for the logits ``hidden`` [..., C] @ ``head_w`` [V, C].T, which are not
    returned: forward reduces them where the product leaves them, in fp32.  ``hidden`` is what the head reads (behind the
    final layer norm) and has to be finite at every position, scored or not.  Differentiable in both; for the backward pass
    the GPU keeps the logits in 16 bits up to ``RWKV7M_B200_HEAD_KEEP_BYTES`` (4 GiB) and computes larger ones again."""
    name = "head_token_logprobs"
    _check_head(name, hidden, head_w)
    _check_ids(name, ids, hidden.shape[:-1], hidden.device)
    temperature = _check_temperature(temperature)
    if use_cuda(hidden):
        return _cuda().head_token_logprobs(hidden, head_w, ids, temperature)
    return reference.token_logprobs(reference.linear(hidden, head_w), ids, 0, temperature)[:2]


def head_distill_loss(hidden, head_w, targets, mask, teacher_ids, teacher_logits, *, temperature=1.0):
    """The loss pieces of :func:`head_loss` and of :func:`distill_loss` in one pass over the head: ``(ce_total, ce_count,
    l2_total, l2_count, kd_total, kd_count)`` for the logits ``hidden`` [..., C] @ ``head_w`` [V, C].T, which are not returned
    (and kept for the backward pass as in :func:`head_token_logprobs`).

    Cross-entropy (at temperature 1) runs over positions with mask != 0 and a target inside the vocabulary, L2Wrap over
    every position, distillation (at ``temperature``) over positions with mask != 0 and a teacher that is not empty;
    ``kd_count`` is the sum of the mask.  ``hidden`` is what the head reads (behind the final layer norm) and has to be finite
    at every position, counted or not.  Differentiable in ``hidden`` and ``head_w``."""
    name = "head_distill_loss"
    _check_head(name, hidden, head_w)
    lead = hidden.shape[:-1]
    _check_ids(name, targets, lead, hidden.device, "targets")
    _check_mask(name, mask, lead, hidden.device)
    _check_teacher(name, lead, hidden.device, teacher_ids, teacher_logits)
    temperature = _check_temperature(temperature)
    if use_cuda(hidden):
        return _cuda().head_distill_loss(hidden, head_w, targets, mask, teacher_ids, teacher_logits, temperature)
    return reference.distill_components(reference.linear(hidden, head_w), targets, mask, teacher_ids, teacher_logits, temperature)


def screening_scan(mod, q_r, q_w, gate, delta_xh, delta_slot, h_base, state, **scalars):
    """Slot-dependent part of the screening memory, sequential over time."""
    if use_cuda(h_base):
        return _cuda().screening_scan(mod, q_r, q_w, gate, delta_xh, delta_slot, h_base, state, **scalars)
    from ..models.screening import screening_scan_reference

    return screening_scan_reference(mod, q_r, q_w, gate, delta_xh, delta_slot, h_base, state, **scalars)


from .backends import (WKVBackend, WKVFFIBackend, WKVGPUConfig, available_wkv_backends, register_wkv_ffi_backend,  # noqa: E402
                       resolve_wkv_backend, set_wkv_backend, unregister_wkv_ffi_backend)

__all__ = [
    "WKVBackend", "WKVFFIBackend", "WKVGPUConfig", "available_wkv_backends", "register_wkv_ffi_backend", "resolve_wkv_backend",
    "set_wkv_backend", "unregister_wkv_ffi_backend", "wkv7_sharded",
    "screening_scan",
    "embedding",
    "wkv7_gn",
    "reference",
    "reference_mode",
    "use_cuda",
    "layer_norm",
    "shift_mix",
    "linear",
    "linear_relu_sq",
    "lora",
    "lora_group",
    "tmix_pre",
    "wkv7",
    "gn_bonus_gate",
    "head_loss",
    "token_logprobs",
    "distill_loss",
    "TokenLogprobs",
    "head_token_logprobs",
    "head_distill_loss",
]
