"""What the row operators (embedding, dropout) share: argument checks and the C structs they fill."""
from __future__ import annotations

import threading
from typing import Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _C

#: a seed by value, or one int64 element of GPU memory that the kernels read
Seed = Union[int, Tensor]


def gpu_index(**tensors: Optional[Tensor]) -> int:
    """The GPU that all of the tensors (those that are not None) are on."""
    if forward_ad._current_level >= 0:
        refuse_tangents(**tensors)
    index = None
    for name, t in tensors.items():
        if t is None:
            continue
        at = t.get_device()
        if index is None:
            index = at
        if at < 0 or at != index:
            raise ValueError(f"{name} must be a tensor on the GPU" + (f" {index}" if index >= 0 and at >= 0 else ""))
    return index


def refuse_tangents(**tensors: Optional[Tensor]) -> None:
    """The operators have no forward-mode derivative: the kernels see no tangent, and the result would have none."""
    for name, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{name} has a forward-mode derivative, which this operator does not carry on")


def enqueue(name: str, fn, index: int, *args) -> None:
    """Calls the C entry ``fn`` with torch's current stream of GPU ``index`` as its last argument, that
    GPU being the current one."""
    if index == torch.cuda.current_device():
        rc = fn(*args, _C.current_stream_ptr(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _C.current_stream_ptr(index))
    if rc:
        _C.check(name, rc)


def written(t: Tensor) -> Tensor:
    """Tells autograd that a kernel has written into ``t``: a backward pass that needs its old values then raises."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)
    return t


def refuse_leaves(name: str, *tensors: Optional[Tensor]) -> None:
    """What is written outside autograd must not be part of a graph."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{name}: not for tensors that require gradients")


def row_stride(name: str, t: Tensor, cols: int) -> int:
    """Distance of the rows of ``t`` (its last dimension) in elements: the elements of a row must lie
    together and the rows at one common distance."""
    if t.is_contiguous():
        return cols
    if t.dim() > 0 and (cols == 1 or t.stride(-1) == 1):
        stride, extent = None, 1  # over the leading dimensions, the innermost first
        for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if stride is None:
                stride, extent = step, size
            elif step == stride * extent:
                extent *= size
            else:
                break
        else:
            return cols if stride is None else stride
    raise ValueError(f"{name}: the elements of a row must lie together and its rows at one distance (shape {tuple(t.shape)}, "
                     f"strides {tuple(t.stride())})")


def with_even_rows(t: Tensor) -> Tensor:
    """``t``, or a contiguous copy where its rows do not lie at one distance (gradients that arrive
    from a broadcast or a transposition)."""
    try:
        row_stride("gradient", t, t.shape[-1] if t.dim() else 1)
        return t
    except ValueError:
        return t.contiguous()


def dropout_record(index: int, p: float, seed: Seed, substream: int, first_index: int) -> "_C.Dropout":
    if not 0 <= substream < 1 << 32:
        raise ValueError("substream must be a 32-bit number")
    if not 0 <= first_index < 1 << 62:
        raise ValueError("first_index must be a number of 62 bits")
    if isinstance(seed, Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError("a seed in GPU memory is one int64 element")
        if seed.get_device() != index:
            raise ValueError(f"seed must be a tensor on the GPU {index}")
        return _C.Dropout(p, 0, seed.data_ptr(), first_index, substream, 0)
    if not 0 <= seed < 1 << 64:
        raise ValueError("seed must be a 64-bit number")
    return _C.Dropout(p, seed, None, first_index, substream, 0)


def token_record(tokens: Tensor, first_row: int, padding: Optional[int]) -> Tuple["_C.Tokens", int]:
    """The C record of ``tokens`` and how many they are."""
    if tokens.dtype == torch.int64:
        size = 8
    elif tokens.dtype == torch.int32:
        size = 4
    else:
        raise ValueError(f"tokens must be int64 or int32, not {tokens.dtype}")
    if not 0 <= first_row < 1 << 62:
        raise ValueError("first_row must not be negative")
    n = tokens.numel()
    if tokens.is_contiguous():
        outer, inner, outer_stride, inner_stride = 1, n, 0, 1
    elif tokens.dim() == 1:
        outer, inner, outer_stride, inner_stride = 1, n, 0, tokens.stride(0)
    elif tokens.dim() == 2:
        (outer, inner), (outer_stride, inner_stride) = tokens.shape, tokens.stride()
    else:
        raise ValueError("tokens of more than two dimensions must be contiguous")
    if padding is None:
        padding = _C.NO_PADDING
    elif not -(1 << 63) < padding < 1 << 63:
        raise ValueError("padding_token must be a 64-bit number")
    return _C.Tokens(tokens.data_ptr(), outer, inner, outer_stride, inner_stride, first_row, padding, size, 0), n


class StreamOrder:
    """``with order:`` around what one pass enqueues on the current stream: passes that change the same memory then run
    one behind the other, whatever streams they are on. On the default stream alone there is nothing to do.

    Recorded passes are ordered among those of the same recording; how replays lie to other work is up to the
    program that replays."""

    def __init__(self, index: int):
        self._index = index
        self._lock = threading.Lock()
        self._on_default = False                        # the last pass that was not recorded: on the default stream,
        self._event: Optional[torch.cuda.Event] = None  # or with this event behind it on another one
        self._last_recorded: Optional[torch.cuda.Stream] = None

    def __enter__(self) -> None:
        self._lock.acquire()
        try:
            self.wait()
        except BaseException:
            self._lock.release()
            raise

    def __exit__(self, *exc) -> None:
        try:
            self.mark()
        finally:
            self._lock.release()

    def wait(self) -> None:
        """The current stream waits for the last pass."""
        if self._event is None and _C.current_stream_ptr(self._index) == 0:
            return  # the default stream behind itself
        now = torch.cuda.current_stream(self._index)
        if torch.cuda.is_current_stream_capturing():
            last = self._last_recorded
            if last is not None and last != now and _is_recorded(last):
                now.wait_stream(last)
        elif self._event is not None:
            now.wait_event(self._event)
        elif self._on_default:
            now.wait_stream(torch.cuda.default_stream(self._index))

    def mark(self) -> None:
        """What has been enqueued on the current stream is the last pass."""
        if _C.current_stream_ptr(self._index) == 0:  # always there to be waited for, and never recorded
            self._event, self._on_default = None, True
            return
        now = torch.cuda.current_stream(self._index)
        if torch.cuda.is_current_stream_capturing():
            self._last_recorded = now
            return
        if self._event is None:
            self._event = torch.cuda.Event()
        self._event.record(now)  # now: a stream of the program's own may be gone by the next pass


def _is_recorded(stream: torch.cuda.Stream) -> bool:
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


def order_of(t: Tensor) -> StreamOrder:
    """The order of the passes that add into the memory of ``t``. It lives in that memory's own record and goes with it."""
    kept = t.untyped_storage().__dict__
    order = kept.get("_flextrain_order")
    return kept.setdefault("_flextrain_order", StreamOrder(t.get_device())) if order is None else order
