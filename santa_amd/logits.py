"""Rules on a model's logits before a token is chosen: penalties for tokens that a
sequence holds already, biases and grammar masks, for single tokens and for the
nodes of drafted trees.

The reference takes the argmax of the logits as they are
(tutorial_code/runtime_common.py:574-675).  Which tokens a row of logits has seen is
said by the plan that its attention ran with (``santa_amd.paged.PagedPlan``): those
that the row's token attends to, a drafted token's own path included.

    plan = cache.plan(seqs, heads, new_tokens=[len(t) for t in trees], parents=trees)
    logits = model.extend(drafts, cache, seqs, ..., parents=trees)
    chosen = adjust_logits(logits, tokens, plan, prompts=prompts, repetition=1.1, allowed=bits, greedy=True)

On a GPU one pass over the logits does all of it (santa_logits.hip); torch
expressions are the CPU path and that of calls under autograd.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from .paged import _KINDS, PagedPlan, _elsewhere, _launch, _PlanInfo
from .runtime import _FusedOps, _plain

__all__ = ["adjust_logits"]

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float


class _Rules(ctypes.Structure):
    _fields_ = [("tokens", _P), ("tokens_wide", _I), ("tokens_rows", _I), ("tokens_len", _I), ("tokens_stride", _L),
                ("prompts", _P), ("repetition", _P), ("frequency", _P), ("presence", _P), ("repetition_all", _F),
                ("frequency_all", _F), ("presence_all", _F), ("bias_ids", _P), ("bias", _P), ("biases", _I),
                ("bias_stride", _L), ("allowed", _P), ("allowed_stride", _L), ("sequences", _I)]


_lib_ready = None


def _lib():
    global _lib_ready
    if _lib_ready is None:
        L = _FusedOps.lib()
        L.santa_adjust_logits_workspace_size.argtypes = [_I, _I, _I]
        L.santa_adjust_logits_workspace_size.restype = ctypes.c_size_t
        L.santa_adjust_logits.argtypes = [_P, _I, _L, _I, _I, ctypes.POINTER(_Rules), ctypes.POINTER(_PlanInfo), _P, _P, _P,
                                          _P, ctypes.c_size_t, _P]
        _lib_ready = L
    return _lib_ready


def _penalty(value, what: str, seqs: int, index: int, positive: bool) -> Union[float, torch.Tensor]:
    if isinstance(value, torch.Tensor):
        shape = value.shape
        if len(shape) != 1 or value.dtype != torch.float32 or value.get_device() != index or shape[0] < seqs:
            raise ValueError(f"{what} must be a number or float32 [sequences] on the logits' device, {seqs} or more")
        return value if value.is_contiguous() else value.contiguous()
    value = float(value)
    if not math.isfinite(value) or (positive and value <= 0.0):
        raise ValueError(f"{what} must be {'positive and ' if positive else ''}finite; got {value}")
    return value


def _rows(t: torch.Tensor, count: int, what: str) -> Tuple[torch.Tensor, int]:
    """t [1 or at least count, n] with contiguous rows, and its row stride (0: one row for all)."""
    shape = t.shape
    if len(shape) != 2 or (shape[0] != 1 and shape[0] < count):
        raise ValueError(f"{what} must have one row, or {count}; got {tuple(shape)}")
    if shape[1] > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0) if shape[0] > 1 else 0


def _bare(*ts: Optional[torch.Tensor]) -> bool:
    """Tensors with memory of their own: no subclasses, none under functorch transforms."""
    for t in ts:
        if t is not None and (type(t) is not torch.Tensor or torch._C._functorch.is_functorch_wrapped_tensor(t)):
            return False
    return True


def adjust_logits(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None,
                  plan: Union[None, PagedPlan, Sequence[int]] = None, *, prompts: Optional[torch.Tensor] = None,
                  repetition: Union[float, torch.Tensor] = 1.0, frequency: Union[float, torch.Tensor] = 0.0,
                  presence: Union[float, torch.Tensor] = 0.0,
                  bias: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, allowed: Optional[torch.Tensor] = None,
                  greedy: bool = False) -> torch.Tensor:
    """Logits [N, V] with rules applied, as float32 [N, V]; or, greedy, the token of
    each row's maximum, int64 [N] (as torch.argmax: NaN above any number, the first
    of equal values; the adjusted logits are not written).

    plan: the PagedPlan whose tokens the rows are, or the lengths of the
    sequences, each with one row; without one, row n is all there is of sequence n.
    tokens: [sequences, places] of int32 or int64, row plan.rows[b] holding the
    tokens of sequence b, place by place as the cache does (a drafted tree's one
    after the other).  A row has seen the tokens that its token of the plan attends
    to.  prompts: int32 [sequences], how many of a sequence's first tokens are its
    prompt's; the others, and drafted tokens of a tree, are its answer's.

    In this order: the logit of a token that the row has seen is divided by
    `repetition` where it is positive, and multiplied by it elsewhere; one that is in
    the answer c > 0 times loses c * frequency, and presence once; bias = (ids,
    values), int32 and float32 [1 or sequences, K], K at most 2046, is added (ids
    outside of the vocabulary, -1 for one, fill rows up; of a token named twice the last
    one counts); and a token that may not come is -inf: allowed, int32 [1 or N,
    ceil(V / 32)], has bit v % 32 of entry v // 32 set where token v may.  Penalties: a
    number, or float32 [sequences] on the device.  Tensors by sequence are read at the
    sequence's row of the block table, like tokens.  Tokens outside of the vocabulary
    are in no row's way.  At most 2^19 - 1 tokens are counted."""
    if logits.dim() != 2 or not logits.dtype.is_floating_point or logits.shape[1] == 0:
        raise ValueError(f"logits must be [rows, vocabulary] of a floating point dtype; got {tuple(logits.shape)}")
    N, V = logits.shape
    device, index = logits.device, logits.get_device()
    if tokens is not None and plan is None:
        raise ValueError("a plan, or the sequences' lengths, says which tokens a row has seen")
    if plan is not None and not isinstance(plan, PagedPlan):
        plan = PagedPlan(plan, heads=1, kv_heads=1, device=device)
    if plan is not None and (plan.tokens != N or plan.device != device):
        raise ValueError(f"the plan is for {plan.tokens} tokens on {plan.device}; got {N} rows on {device}")
    if index < 0:  # CPU and meta tensors have one number
        for name, t in (("tokens", tokens), ("prompts", prompts), ("repetition", repetition), ("frequency", frequency),
                        ("presence", presence), ("bias", None if bias is None else bias[0]),
                        ("bias", None if bias is None else bias[1]), ("allowed", allowed)):
            if isinstance(t, torch.Tensor) and _elsewhere(logits, t):
                raise ValueError(f"{name} must be on the logits' device; got {t.device}")
    seqs = N if plan is None else plan._info.max_row + 1
    if tokens is not None:
        if tokens.dim() != 2 or tokens.dtype not in (torch.int32, torch.int64) or tokens.get_device() != index:
            raise ValueError("tokens must be [sequences, places] of int32 or int64 on the logits' device")
        if tokens.shape[0] < seqs or tokens.shape[1] < plan._info.max_len:
            raise ValueError(f"tokens must hold {seqs} sequences of {plan._info.max_len} tokens; got {tuple(tokens.shape)}")
        if tokens.shape[1] > 1 and tokens.stride(1) != 1:
            tokens = tokens.contiguous()
    if prompts is not None and (prompts.dim() != 1 or prompts.dtype != torch.int32 or prompts.get_device() != index
                                or prompts.shape[0] < seqs):
        raise ValueError(f"prompts must be int32 [sequences] on the logits' device, {seqs} or more")
    penalties = [_penalty(x, name, seqs, index, name == "repetition")
                 for x, name in ((repetition, "repetition"), (frequency, "frequency"), (presence, "presence"))]
    ids = values = None
    if bias is not None:
        ids, values = bias
        if ids.shape != values.shape or ids.dtype != torch.int32 or values.dtype != torch.float32 or \
                ids.get_device() != index or values.get_device() != index:
            raise ValueError("bias must be (int32 ids, float32 values) of one shape on the logits' device")
        if ids.dim() == 2 and ids.shape[1] > 2046:
            raise ValueError(f"a row has at most 2046 biases; got {ids.shape[1]}")
        (ids, bias_stride), (values, value_stride) = _rows(ids, seqs, "bias"), _rows(values, seqs, "bias")
        if bias_stride != value_stride:
            ids, values = ids.contiguous(), values.contiguous()
            bias_stride = ids.stride(0) if ids.shape[0] > 1 else 0
    if allowed is not None:
        if allowed.dtype != torch.int32 or allowed.get_device() != index or allowed.dim() != 2 or \
                allowed.shape[1] != -(-V // 32):
            raise ValueError(f"allowed must be int32 [1 or {N}, {-(-V // 32)}] on the logits' device")
        allowed, allowed_stride = _rows(allowed, N, "allowed")
    if plan is not None and tokens is not None and plan._info.max_len >= 1 << 19:
        raise ValueError(f"at most {(1 << 19) - 1} tokens are counted; got {plan._info.max_len}")
    if tokens is None and plan is None and (prompts is not None or any(
            isinstance(p, torch.Tensor) or p != none for p, none in zip(penalties, (1.0, 0.0, 0.0)))):
        raise ValueError("penalties and prompts are for tokens that a row has seen: without tokens there are none")
    kind = _KINDS.get(logits.dtype)
    given = [t for t in (*penalties, values) if isinstance(t, torch.Tensor)]
    if not (device.type == "cuda" and kind is not None and _plain(logits, *given)
            and _bare(tokens, prompts, ids, allowed)):
        out = _expressions(logits, tokens, plan, prompts, penalties, ids, values, allowed)
        if plan is not None:
            plan._captured(0, False)
        return out.argmax(-1) if greedy else out
    if N > 0 and (V > 1 and logits.stride(1) != 1 or N > 1 and logits.stride(0) < V):
        logits = logits.contiguous()
    out = torch.empty((N,) if greedy else (N, V), dtype=torch.int64 if greedy else torch.float32, device=device)
    if N == 0:
        return out
    rules = _Rules()
    if tokens is not None:
        rules.tokens, rules.tokens_wide = tokens.data_ptr(), int(tokens.dtype == torch.int64)
        rules.tokens_rows, rules.tokens_len = tokens.shape
        rules.tokens_stride = tokens.stride(0)
    if prompts is not None:
        prompts = prompts.contiguous()
        rules.prompts = prompts.data_ptr()
    for name, x in zip(("repetition", "frequency", "presence"), penalties):
        if isinstance(x, torch.Tensor):
            setattr(rules, name, x.data_ptr())
        else:
            setattr(rules, name + "_all", x)
    if ids is not None:
        rules.bias_ids, rules.bias, rules.biases = ids.data_ptr(), values.data_ptr(), ids.shape[1]
        rules.bias_stride = bias_stride
    if allowed is not None:
        rules.allowed, rules.allowed_stride = allowed.data_ptr(), allowed_stride
    if plan is not None:
        rules.sequences = len(plan.seq_lens)
    lib = _lib()
    workspace = torch.empty(lib.santa_adjust_logits_workspace_size(N, V, rules.sequences) if greedy else 0, dtype=torch.uint8,
                            device=device)
    info, data = (None, None) if plan is None else (ctypes.byref(plan._info), plan._data.data_ptr())
    if plan is not None:
        plan._used()
    _launch(device, lib.santa_adjust_logits, logits.data_ptr(), kind, logits.stride(0) if N > 1 else V, N, V,
            ctypes.byref(rules), info, data, None if greedy else out.data_ptr(), out.data_ptr() if greedy else None,
            workspace.data_ptr(), workspace.numel())
    if plan is not None:
        plan._captured(1 << 30 if tokens is None else min(tokens.shape[1], (1 << 19) - 1), True)
    return out


def _expressions(logits, tokens, plan, prompts, penalties, ids, values, allowed) -> torch.Tensor:
    """adjust_logits in torch operations, float32 (float64 for float64)."""
    N, V = logits.shape
    device = logits.device
    x = logits.to(torch.float64 if logits.dtype == torch.float64 else torch.float32)
    rows = list(range(N)) if plan is None else [row for row, t in zip(plan.rows, plan.new_tokens) for _ in range(t)]
    at = torch.tensor(rows, dtype=torch.int64, device=device)
    repetition, frequency, presence = (p[at][:, None].to(x.dtype) if isinstance(p, torch.Tensor) else p for p in penalties)
    if tokens is not None and N > 0:
        none = torch.zeros(V + 1, dtype=torch.int64, device=device)  # the last one: no token of the vocabulary
        all_seen, counts = [], []
        for b, (row, n, t) in enumerate(zip(plan.rows, plan.seq_lens, plan.new_tokens)):
            ids_b = tokens[row, :n].long()
            ids_b = torch.where((ids_b >= 0) & (ids_b < V), ids_b, V)
            answer = (torch.arange(n, device=device) >= (0 if prompts is None else prompts[row])).long()
            tree = plan.parents is not None and plan.parents[b] is not None
            if tree:
                sees = plan._sees(b)
                answer = torch.cat([answer[:max(0, n - t)], answer.new_ones(min(n, t))])  # a tree's are the answer's
            used = set(plan._in_use(b))
            for i in range(t):
                if i not in used:
                    all_seen.append(none > 0), counts.append(none)
                    continue
                places = torch.arange(n - t + i + 1, device=device)
                if tree:
                    places = torch.cat([places[:n - t], n - t + sees[i].nonzero()[:, 0].to(device)])
                here = ids_b[places]
                all_seen.append(none.scatter_add(0, here, torch.ones_like(here)) > 0)
                counts.append(none.scatter_add(0, here, answer[places]))
        seen, count = torch.stack(all_seen)[:, :V], torch.stack(counts)[:, :V]
        x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
        x = torch.where(count > 0, x - frequency * count.to(x.dtype) - presence, x)
    if ids is not None and ids.shape[1]:
        each = torch.arange(ids.shape[1], device=device).expand(ids.shape)
        inside = (ids >= 0) & (ids < V)
        last = torch.full((len(ids), V + 1), -1, dtype=torch.int64, device=device)
        last = last.scatter_reduce(1, torch.where(inside, ids, V).long(), torch.where(inside, each, -1), "amax")
        last = last[:, :V].expand(N, V) if len(ids) == 1 else last[at, :V]
        row_values = values.expand(N, -1) if len(values) == 1 else values[at]
        x = torch.where(last >= 0, x + row_values.gather(1, last.clamp(min=0)).to(x.dtype), x)
    if allowed is not None:
        v = torch.arange(V, device=device)
        x = torch.where((allowed[:N, v >> 5] >> (v & 31)) & 1 > 0, x, -math.inf)
    return x
