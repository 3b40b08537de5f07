"""Routing of tokens to experts, and back.

`route` chooses each token's experts and their weights from its logits,
`dispatch` sorts the choices by expert (the `Plan` that mx.linear takes), and
`combine` sums the experts' outputs into the tokens'. `route_backward` and
`combine_backward` are the gradients. Every call launches on the current
stream, allocates only the outputs that it is not given, and raises ValueError
for tensors that do not fit it.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native
from .mx import allocate, check_output, check_tensor, dtype_code, launch_stream, library, strided_rows

SCORES = {"softmax": 0, "sigmoid": 1}


class Plan(NamedTuple):
    """Choices sorted by expert (int32): expert e's are order[offsets[e] .. offsets[e + 1] - 1], each the number of an
    entry of the [tokens][top] choices; slots [tokens][top] is an entry's place in order. -1 where an entry has no
    expert, and in order past the last entry that has one."""

    offsets: object
    order: object
    slots: object
    workspace: object = None


def _score_code(scores: str) -> int:
    if scores not in SCORES:
        raise ValueError(f"scores must be one of {', '.join(SCORES)}, not {scores!r}")
    return SCORES[scores]


def route(logits, top: int, bias=None, scores: str = "softmax", groups: int = 1, top_groups: int = 1,
          renormalize: bool = True, scale: float = 1.0, experts=None, weights=None, stream=None):
    """(experts, weights), int32 and float32 [tokens][top], of logits [tokens][experts].

    s = softmax or sigmoid of the logits; c = s + bias decides: of `groups` equal groups the `top_groups` with the
    largest sum of their two largest c stay, then the `top` largest c, in falling order and of equal ones the lower
    index. A logit of -inf masks its expert; -1, with weight 0, stands where none is left. The weights are s, divided
    by their sum if `renormalize`, times `scale`.
    """
    code = dtype_code(logits, "logits")
    tokens, count, stride, span = strided_rows(logits, "logits")
    experts = check_output(experts, "experts", (tokens, top), torch.int32, logits, stream)
    weights = check_output(weights, "weights", (tokens, top), torch.float32, logits, stream)
    if bias is None:
        handle = launch_stream(stream, logits, experts, weights)
    else:
        check_tensor(bias, "bias", (count,), torch.float32)
        handle = launch_stream(stream, logits, experts, weights, bias)
    entries = 4 * tokens * top
    status = library().mb_route(code, logits.data_ptr(), span * (2 if code else 4), tokens, count, stride,
                                None if bias is None else bias.data_ptr(), 4 * count, top, _score_code(scores), groups,
                                top_groups, int(renormalize), scale, experts.data_ptr(), entries, weights.data_ptr(),
                                entries, handle)
    if status:
        _native.check(status)
    return experts, weights


def route_backward(logits, experts, d_weights, scores: str = "softmax", renormalize: bool = True, scale: float = 1.0,
                   d_logits=None, stream=None):
    """d_logits, in the logits' type, for the gradient d_weights of route's weights and the experts it chose."""
    code = dtype_code(logits, "logits")
    tokens, count, stride, span = strided_rows(logits, "logits")
    if experts.dim() != 2 or experts.shape[0] != tokens:
        raise ValueError(f"experts must be [{tokens}][top], not {tuple(experts.shape)}")
    top = experts.shape[1]
    check_tensor(experts, "experts", (tokens, top), torch.int32)
    check_tensor(d_weights, "d_weights", (tokens, top), torch.float32)
    d_logits = check_output(d_logits, "d_logits", (tokens, count), logits.dtype, logits, stream)
    handle = launch_stream(stream, logits, experts, d_weights, d_logits)
    item, entries = 2 if code else 4, 4 * tokens * top
    status = library().mb_route_backward(code, logits.data_ptr(), span * item, tokens, count, stride,
                                         experts.data_ptr(), entries, d_weights.data_ptr(), entries, top,
                                         _score_code(scores), int(renormalize), scale, d_logits.data_ptr(),
                                         tokens * count * item, handle)
    if status:
        _native.check(status)
    return d_logits


def empty_plan(tokens: int, top: int, experts: int, device="cuda", stream=None) -> Plan:
    """A plan's buffers and workspace, for `dispatch` to fill."""
    needed = library().mb_dispatch_workspace(tokens * top, experts)
    return Plan(allocate(experts + 1, torch.int32, device, stream), allocate(tokens * top, torch.int32, device, stream),
                allocate((tokens, top), torch.int32, device, stream), allocate(needed, torch.uint8, device, stream))


def dispatch(experts, count: int, plan: Plan | None = None, stream=None) -> Plan:
    """The plan of the choices `experts` [tokens][top] (int32; outside 0 .. count - 1: none) of `count` experts."""
    if experts.dim() != 2:
        raise ValueError(f"experts must be [tokens][top], not {tuple(experts.shape)}")
    tokens, top = experts.shape
    entries = tokens * top
    check_tensor(experts, "experts", (tokens, top), torch.int32)
    if plan is None:
        plan = empty_plan(tokens, top, count, experts.device, stream)
    offsets, order, slots, workspace = plan
    check_tensor(offsets, "plan.offsets", (count + 1,), torch.int32)
    check_tensor(order, "plan.order", (entries,), torch.int32)
    check_tensor(slots, "plan.slots", (tokens, top), torch.int32)
    if workspace is None:
        handle, space = launch_stream(stream, experts, offsets, order, slots), (None, 0)
    else:
        handle = launch_stream(stream, experts, offsets, order, slots, workspace)
        space = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    status = library().mb_dispatch(experts.data_ptr(), 4 * entries, entries, count, offsets.data_ptr(), 4 * count + 4,
                                   order.data_ptr(), 4 * entries, slots.data_ptr(), 4 * entries, *space, handle)
    if status:
        _native.check(status)
    return plan


def _combine_sizes(y, slots, weights):
    if y.dim() != 2 or slots.dim() != 2 or not y.is_contiguous():
        raise ValueError(f"y must be contiguous [rows][n] and slots [tokens][top], not {tuple(y.shape)} and "
                         f"{tuple(slots.shape)}")
    shape = slots.shape
    check_tensor(slots, "slots", shape, torch.int32)
    check_tensor(weights, "weights", shape, torch.float32)
    return dtype_code(y, "y"), *y.shape, *shape


def combine(y, slots, weights, out=None, stream=None):
    """out[t] = the sum over j of weights[t][j] * y[slots[t][j]], in y's type; slots of -1 are left out."""
    code, rows, n, tokens, top = _combine_sizes(y, slots, weights)
    out = check_output(out, "out", (tokens, n), y.dtype, y, stream)
    handle = launch_stream(stream, y, slots, weights, out)
    item, entries = 2 if code else 4, 4 * tokens * top
    status = library().mb_combine(code, y.data_ptr(), rows * n * item, rows, slots.data_ptr(), entries,
                                  weights.data_ptr(), entries, out.data_ptr(), tokens * n * item, tokens, top, n,
                                  handle)
    if status:
        _native.check(status)
    return out


def combine_backward(d_out, y, slots, weights, d_y=None, d_weights=None, stream=None):
    """(d_y, d_weights) of combine for the gradient d_out; rows of a given d_y that no slot names stay as they are."""
    code, rows, n, tokens, top = _combine_sizes(y, slots, weights)
    check_tensor(d_out, "d_out", (tokens, n), y.dtype)
    if d_y is None:
        with torch.cuda.stream(stream):  # cleared in the order of the call's work
            d_y = torch.zeros_like(y)
    check_tensor(d_y, "d_y", (rows, n), y.dtype)
    d_weights = check_output(d_weights, "d_weights", (tokens, top), torch.float32, y, stream)
    handle = launch_stream(stream, y, slots, weights, d_out, d_y, d_weights)
    item, entries = 2 if code else 4, 4 * tokens * top
    status = library().mb_combine_backward(code, d_out.data_ptr(), tokens * n * item, y.data_ptr(), rows * n * item,
                                           rows, slots.data_ptr(), entries, weights.data_ptr(), entries,
                                           d_y.data_ptr(), rows * n * item, d_weights.data_ptr(), entries, tokens, top,
                                           n, handle)
    if status:
        _native.check(status)
    return d_y, d_weights
