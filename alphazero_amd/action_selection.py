"""Action selection functions (mirrors mctx_dist/_src/action_selection.py).

The four selection rules run inside the HIP search kernels.  As in the
reference, `search()` receives them as ``functools.partial`` objects binding
their keyword options; here the functions are markers that identify the rule
and carry those options to the kernels.

`sample_actions` selects without a search: a draw from (truncated) policy logits.
"""
import ctypes as C
import dataclasses
import math
from typing import Any

import torch

from . import _native as nat
from . import layers
from . import qtransforms as qt

_MSG = ("action selection runs inside the search kernels; pass this function (or a "
        "functools.partial of it) to search()")


def muzero_action_selection(rng_key=None, tree=None, node_index=None, depth=None, *,
                            pb_c_init=1.25, pb_c_base=19652.0,
                            qtransform=qt.qtransform_by_parent_and_siblings):
    """mctx_dist/_src/action_selection.py:48-90 (PUCT on softmax(prior logits))."""
    raise NotImplementedError(_MSG)


def sampled_muzero_action_selection(rng_key=None, tree=None, node_index=None, depth=None, *,
                                    pb_c_init=1.25, pb_c_base=19652.0,
                                    qtransform=qt.qtransform_by_parent_and_siblings):
    """mctx_dist/_src/action_selection.py:93-135 (PUCT on stored sample-based probabilities)."""
    raise NotImplementedError(_MSG)


def gumbel_muzero_root_action_selection(rng_key=None, tree=None, node_index=None, *,
                                        num_simulations=None, max_num_considered_actions=None,
                                        qtransform=qt.qtransform_completed_by_mix_value):
    """mctx_dist/_src/action_selection.py:148-200 (Sequential Halving with Gumbel)."""
    raise NotImplementedError(_MSG)


def gumbel_muzero_interior_action_selection(rng_key=None, tree=None, node_index=None, depth=None,
                                            *, qtransform=qt.qtransform_completed_by_mix_value):
    """mctx_dist/_src/action_selection.py:203-240 (deterministic interior selection)."""
    raise NotImplementedError(_MSG)


def stochastic_muzero_action_selection(rng_key=None, tree=None, node_index=None, depth=None, *,
                                       decision_node_selection_fn=None, num_actions=None):
    """mctx_dist/_src/policies.py:676-708 (_make_stochastic_action_selection_fn): decision nodes
    select with `decision_node_selection_fn` (a muzero_action_selection partial) over the first
    `num_actions` columns, chance nodes with argmax(softmax(chance logits) / (visits + 1))."""
    raise NotImplementedError(_MSG)


@dataclasses.dataclass(frozen=True)
class GumbelMuZeroExtraData:
    """mctx_dist/_src/action_selection.py:138-141"""
    root_gumbel: Any


def resolve(root_fn, interior_fn, desc, num_simulations):
    """Fills the native SearchDesc from the (root, interior) selection functions."""
    rf, rkw = qt.unwrap_partial(root_fn)
    inf, ikw = qt.unwrap_partial(interior_fn)
    rkw = dict(rkw)
    rkw.pop("depth", None)  # policies.py:98-100 binds depth=0 into the root function
    if rf is gumbel_muzero_root_action_selection and inf is gumbel_muzero_interior_action_selection:
        desc.variant = nat.VARIANT_GUMBEL
        m = rkw.get("max_num_considered_actions")
        if m is None:
            raise TypeError("gumbel_muzero_root_action_selection needs max_num_considered_actions")
        ns = rkw.get("num_simulations", num_simulations)
        if ns != num_simulations:
            raise ValueError("num_simulations bound into the root selection differs from search()'s")
        desc.max_num_considered = int(m)
        q_root = rkw.get("qtransform", qt.qtransform_completed_by_mix_value)
        q_int = ikw.get("qtransform", qt.qtransform_completed_by_mix_value)
    elif rf is inf and rf is stochastic_muzero_action_selection:
        dec, dkw = qt.unwrap_partial(ikw.get("decision_node_selection_fn"))
        if dec is not muzero_action_selection or rkw != ikw:
            raise NotImplementedError("stochastic selection: decision nodes select with a "
                                      "muzero_action_selection partial, the same at the root")
        desc.variant = nat.VARIANT_STOCHASTIC
        desc.num_decision_actions = int(ikw["num_actions"])
        desc.pb_c_init = float(dkw.get("pb_c_init", 1.25))
        desc.pb_c_base = float(dkw.get("pb_c_base", 19652.0))
        q_root = q_int = dkw.get("qtransform", qt.qtransform_by_parent_and_siblings)
    elif rf is inf and rf in (muzero_action_selection, sampled_muzero_action_selection):
        desc.variant = (nat.VARIANT_MUZERO if rf is muzero_action_selection
                        else nat.VARIANT_SAMPLED)
        for k in ("pb_c_init", "pb_c_base"):
            if rkw.get(k, None) != ikw.get(k, None):
                raise NotImplementedError("root and interior selection must share " + k)
        desc.pb_c_init = float(ikw.get("pb_c_init", 1.25))
        desc.pb_c_base = float(ikw.get("pb_c_base", 19652.0))
        q_root = rkw.get("qtransform", qt.qtransform_by_parent_and_siblings)
        q_int = ikw.get("qtransform", qt.qtransform_by_parent_and_siblings)
    else:
        raise NotImplementedError(
            "the search kernels implement the (muzero, muzero), (sampled, sampled) and "
            "(gumbel root, gumbel interior) selection pairs of the reference; got "
            f"{root_fn!r} / {interior_fn!r}")
    a, b = nat.SearchDesc(), nat.SearchDesc()
    qt.apply_to_desc(q_root, a)
    qt.apply_to_desc(q_int, b)
    if bytes(a) != bytes(b):
        raise NotImplementedError("root and interior selection must use the same qtransform")
    qt.apply_to_desc(q_int, desc)
    return desc


def sample_actions(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, invalid_actions=None):
    """Draws one action a row from truncated policy logits: (action int32 [B], log_prob float32 [B]).

    logits [B, A] float32 / bfloat16 / float16; uniform [B] float32, the row's random number in [0, 1);
    invalid_actions [B, A], nonzero where an action is illegal.  Of the legal actions in descending order of their
    logits (equal ones by index) the first `top_k` are kept (0: all), of these the fewest that hold
    `top_p` of their probability, of these the ones with at least `min_p` of the largest one's probability (and
    never one with less than 2^-40 of it).  The action is the first, in index order, whose cumulative
    probability among the kept ones exceeds `uniform`; log_prob is its log probability among them.  temperature
    divides the logits; 0 takes the largest one.  The four parameters are numbers or [B] tensors (in which a
    negative or NaN temperature counts as 0, top_k <= 0 as all, and top_p, min_p beyond [0, 1] as the nearer end).
    -inf and NaN logits are illegal; a row without a legal action gives action 0 and log_prob -inf.  Neither output
    carries a derivative.
    """
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"sample_actions: logits {tuple(logits.shape)} must be [B, A] with A >= 1")
    B, A = logits.shape
    if B > layers.MAX_ROWS or A > layers.MAX_ROWS:
        raise NotImplementedError(f"sample_actions: logits {tuple(logits.shape)}")
    code = layers.DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"sample_actions: float32, bfloat16 or float16 logits, got {logits.dtype}")
    if uniform.shape != (B,) or uniform.dtype != torch.float32:
        raise ValueError(f"sample_actions: uniform must be float32 [{B}], got {uniform.dtype} {tuple(uniform.shape)}")
    if invalid_actions is not None and invalid_actions.shape != (B, A):
        raise ValueError(f"sample_actions: invalid_actions {tuple(invalid_actions.shape)} must be {(B, A)}")
    d = nat.SampleDesc(code, B, A)
    keep = []
    values = (temperature, top_k, top_p, min_p)
    if any(isinstance(v, torch.Tensor) for v in values):
        values = list(values)
        for i, (name, dtype) in enumerate((("temperature", torch.float32), ("top_k", torch.int32),
                                           ("top_p", torch.float32), ("min_p", torch.float32))):
            value = values[i]
            if not isinstance(value, torch.Tensor) or value.dim() == 0:
                continue
            if value.shape != (B,):
                raise ValueError(f"sample_actions: {name} {tuple(value.shape)} must be a number or [{B}]")
            if value.device != logits.device:
                raise ValueError(f"sample_actions: {name} is on {value.device}, logits on {logits.device}")
            if name == "top_k":
                if value.is_floating_point() or value.is_complex():
                    raise TypeError(f"sample_actions: top_k must hold integers, got {value.dtype}")
                if value.dtype != dtype:   # (counts beyond 32 bits do not wrap)
                    value = value.long().clamp(0, A)
            keep.append(value.to(dtype).contiguous())
            setattr(d, name + "_rows", keep[-1].data_ptr())
            values[i] = 0
    temperature, top_k, top_p, min_p = values
    if not (0.0 <= temperature < math.inf and 0.0 <= top_p <= 1.0 and 0.0 <= min_p <= 1.0 and
            0 <= top_k < 2 ** 31 and top_k == int(top_k)):
        raise ValueError(f"sample_actions: temperature={temperature} top_k={top_k} top_p={top_p} min_p={min_p}")
    d.temperature, d.top_k, d.top_p, d.min_p = temperature, int(top_k), top_p, min_p
    layers._checked("sample_actions", logits, (("uniform", uniform), ("invalid_actions", invalid_actions)))
    logits, uniform = logits.detach().contiguous(), uniform.contiguous()
    d.logits, d.uniform = logits.data_ptr(), uniform.data_ptr()
    if invalid_actions is not None:
        if invalid_actions.dtype not in (torch.bool, torch.uint8, torch.int8):
            invalid_actions = invalid_actions != 0
        keep.append(invalid_actions.contiguous())
        d.invalid = keep[-1].data_ptr()
    action = torch.empty((B,), dtype=torch.int32, device=logits.device)
    log_prob = torch.empty((B,), dtype=torch.float32, device=logits.device)
    layers._native(logits.device, nat.lib().az_sample_actions, C.byref(d), action, log_prob)
    return action, log_prob
