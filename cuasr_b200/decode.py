"""Operators of a decoding step, over the C entry points of include/cuasr_b200_decode.h.

`Q4Product` is the plus-times product of a few rows with weights held in 4 bits, `BeamStep` the max-plus step that keeps
the best continuations of a beam search with back-pointers, and `ReorderStates` moves the states of the prefixes after
those back-pointers.  They are used like `Srgemm`: the types are constructor arguments, buffers are device addresses or
torch CUDA tensors with their leading dimensions, `initialize(args)` checks and keeps a call and `run()` enqueues it;
calling the operator does both.  Buffers belong to the caller and stay alive until the work on the stream is done.
"""
from __future__ import annotations

import ctypes
import dataclasses
import struct
from typing import Any, Optional, Sequence, Tuple

from . import _lib
from .semiring import DType, Status
from .srgemm import _STATUS, _ptr, _stream_handle

_REAL = (DType.F32, DType.F16, DType.BF16)


def _real(dtype) -> DType:
    dtype = DType(dtype)
    if dtype not in _REAL:
        raise ValueError(f"the decoding operators take F32, F16 and BF16, not {dtype!r}")
    return dtype


def _device(buffers) -> Optional[int]:
    """The `device` field of a call on these buffers: d + 1 for tensors of CUDA device d, 0 (the current device) where all
    are addresses; None for tensors that are not on one CUDA device."""
    found = 0
    for x in buffers:
        device = getattr(x, "device", None)
        if device is None:
            continue
        if device.type != "cuda" or found not in (0, device.index + 1):
            return None
        found = device.index + 1
    return found


# the C arguments' layouts: a number that its field does not hold is an error here, where ctypes would cut it off
_PACK = {kind: struct.Struct(layout).pack for kind, layout in (
    (_lib.Q4Args, "8i" + 5 * "Qq" + "Q"), (_lib.BeamArgs, "8iQqq" + 5 * "Qq" + "QNQ"), (_lib.State, "QQ8qq4i"), (_lib.ReorderArgs, "4iQqQQ2iQ"))}


_NAMES = {DType.F32: ("float32",), DType.F16: ("float16",), DType.BF16: ("bfloat16",)}
_BYTES, _FLAGS, _INDEX = ("uint8",), ("uint8", "bool"), ("int32",)


def _typed(*buffers) -> bool:
    """Whether every tensor has one of the element types named beside it; addresses have none."""
    return all(str(x.dtype).rsplit(".", 1)[-1] in names for x, names in buffers if hasattr(x, "dtype"))


@dataclasses.dataclass
class Q4Arguments:
    """Y = X W^T: ref_X and ref_Y are row-major m x k and m x n, ref_W holds n rows of bytes (two weights each, the even k
    in the low half), ref_scales and ref_zeros n x ceil(k / group)."""
    problem_size: Tuple[int, int, int]      # (m, n, k)
    ref_X: Tuple[Any, int]                  # (pointer or tensor, leading dimension in elements)
    ref_W: Tuple[Any, int]                  # (pointer or tensor, bytes per row)
    ref_scales: Tuple[Any, int]
    ref_Y: Tuple[Any, int]
    ref_zeros: Tuple[Any, int] = (None, 0)  # without zero points, 8 stands for zero


@dataclasses.dataclass
class BeamArguments:
    """One step of `batch` searches.  ref_logits: (pointer or tensor, batch stride, beam stride) in elements, the vocabulary
    contiguous; the others are (pointer or tensor, leading dimension)."""
    problem_size: Tuple[int, int, int, int]  # (batch, beams, vocab, keep)
    ref_logits: Tuple[Any, int, int]
    ref_scores: Tuple[Any, int]              # float32, batch x beams
    ref_out_scores: Tuple[Any, int]          # float32, batch x keep; may be ref_scores
    ref_parents: Tuple[Any, int]             # int32, batch x keep
    ref_tokens: Tuple[Any, int]              # int32, batch x keep
    ref_finished: Tuple[Any, int] = (None, 0)  # uint8, batch x beams
    end_token: int = 0


@dataclasses.dataclass
class StateView:
    """cuasr_b200_state_t: one state tensor as batch x beams x segments x positions x bytes, strides in bytes."""
    src: Any
    dst: Any
    src_strides: Tuple[int, int, int, int]   # batch, beam, segment, position
    dst_strides: Tuple[int, int, int, int]
    bytes: int
    segments: int = 1
    positions: int = 1
    ragged: bool = False


def _empty(x) -> bool:
    """Whether x is a tensor without elements."""
    return hasattr(x, "numel") and x.numel() == 0


def state_view(src, dst=None, position_dim: Optional[int] = None) -> StateView:
    """StateView of a torch tensor whose first two dimensions are batch and beams (dst: the same tensor where it is left
    out).  Without position_dim a row is moved whole; with it, dimension position_dim counts positions and only the
    first lengths[s] of them are moved where the call has lengths.  At most one dimension (or several that lie one behind the
    other) in front of the positions and contiguous ones behind them can be described; other views raise ValueError.  A tensor
    without elements (a cache without positions yet) is a state of which a call moves nothing."""
    dst = src if dst is None else dst
    if src.dim() < 2 or src.dtype != dst.dtype or src.shape[0] != dst.shape[0] or src.shape[2:] != dst.shape[2:]:
        raise ValueError("src and dst are batch x beams x ... of one type and, but for the beams, one shape")
    if position_dim is not None and not 2 <= position_dim < src.dim():
        raise ValueError("position_dim comes after batch and beams")
    if _empty(src) and _empty(dst):
        return StateView(src, dst, (0, 0, 0, 0), (0, 0, 0, 0), 0, 0, 0, position_dim is not None)
    es = src.element_size()
    shape, sides = list(src.shape[2:]), [list(t.stride()[2:]) for t in (src, dst)]

    def folded(dims):
        """The dimensions as one: (extent, stride on either side); None where they do not lie one behind the other."""
        extent, strides = 1, None
        for d in reversed(dims):
            if shape[d] == 1:
                continue
            if strides is None:
                strides = [side[d] for side in sides]
            elif [side[d] for side in sides] != [extent * st for st in strides]:
                return None
            extent *= shape[d]
        return extent, strides if strides is not None else [1, 1]

    if position_dim is None:
        # as many of the last dimensions as are contiguous on both sides; the rest in front of them
        split = len(shape)
        while split > 0 and (inner := folded(range(split - 1, len(shape)))) is not None and inner[1] == [1, 1]:
            split -= 1
        inner, positions, position_strides, outer = folded(range(split, len(shape))), 1, [0, 0], folded(range(split))
    else:
        p = position_dim - 2
        inner, positions, position_strides, outer = folded(range(p + 1, len(shape))), shape[p], [side[p] for side in sides], folded(range(p))
    if inner is None or outer is None or inner[1] != [1, 1]:
        raise ValueError("this view needs more strides than a StateView has")
    strides = [tuple(es * n for n in (t.stride(0), t.stride(1), outer[1][i], position_strides[i])) for i, t in enumerate((src, dst))]
    return StateView(src, dst, strides[0], strides[1], inner[0] * es, outer[0], positions, position_dim is not None)


@dataclasses.dataclass
class ReorderArguments:
    """states[i].dst[s, j] = states[i].src[s, parents[s, j]] for the keep rows j of each search s."""
    problem_size: Tuple[int, int, int]      # (batch, beams, keep)
    ref_parents: Tuple[Any, int]            # int32, batch x keep
    states: Sequence[StateView]
    lengths: Any = None                     # int32, batch: positions in use; None: all of them


class _DecodeOperator:
    _name = ""

    def __init__(self):
        self._lib = _lib.load()
        self._can = getattr(self._lib, self._name + "_can_implement")
        self._run = getattr(self._lib, self._name)
        self._args = None
        self._args_ref = None
        self._keepalive = None

    def _pack(self, args, workspace, stream):
        try:
            return self._packed(args, workspace, stream)
        except struct.error:
            return None

    def _packed(self, args, workspace, stream):
        """The C arguments, or None for buffers that are not on one CUDA device; struct.error for numbers that the C fields
        do not hold."""
        raise NotImplementedError

    def _required_workspace(self, packed) -> int:
        return 0

    def _types_match(self, args) -> bool:
        raise NotImplementedError

    def can_implement(self, args) -> Status:
        return self._check(args, self._pack(args, None, None))

    def _check(self, args, packed) -> Status:
        if packed is None:
            return Status.kErrorInvalidProblem
        return _STATUS[self._can(ctypes.byref(packed))] if self._types_match(args) else Status.kErrorInvalidDataType

    def _check_workspace(self, packed) -> Status:
        """What the library's call would say to the workspace."""
        need = self._required_workspace(packed)
        if need == 0:
            return Status.kSuccess
        if not packed.workspace:
            return Status.kErrorWorkspaceNull
        if packed.workspace_bytes < need:
            return Status.kErrorInvalidProblem
        return Status.kSuccess if packed.workspace % 16 == 0 else Status.kErrorMisalignedOperand

    def initialize(self, args, workspace=None, stream=None) -> Status:
        """Checks the call and keeps it for run().  The operator keeps the buffers named in `args` alive."""
        packed = self._pack(args, workspace, stream)
        status = self._check(args, packed)
        if status is Status.kSuccess:
            status = self._check_workspace(packed)
        if status is Status.kSuccess:
            self._args, self._args_ref, self._keepalive = packed, ctypes.byref(packed), (args, workspace)
        return status

    def run(self, stream=None) -> Status:
        """Enqueues the initialised call on the stream of initialize(), or on another from now on."""
        if self._args is None:
            return Status.kErrorInternal
        if stream is not None:
            self._args.stream = _stream_handle(stream)
        return _STATUS[self._run(self._args_ref)]

    def __call__(self, args=None, workspace=None, stream=None) -> Status:
        if args is not None:
            status = self.initialize(args, workspace, stream)
            if status is not Status.kSuccess:
                return status
        return self.run(stream)


class Q4Product(_DecodeOperator):
    """cuasr_b200_q4_product."""
    _name = "cuasr_b200_q4_product"

    def __init__(self, dtype_x: DType = DType.BF16, dtype_y: Optional[DType] = None, dtype_scale: Optional[DType] = None,
                 group: int = 128):
        super().__init__()
        self.dtype_x = _real(dtype_x)
        self.dtype_y = self.dtype_x if dtype_y is None else _real(dtype_y)
        self.dtype_scale = self.dtype_x if dtype_scale is None else _real(dtype_scale)
        self.group = int(group)

    def _types_match(self, args: Q4Arguments) -> bool:
        return _typed((args.ref_X[0], _NAMES[self.dtype_x]), (args.ref_W[0], _BYTES), (args.ref_scales[0], _NAMES[self.dtype_scale]),
                      (args.ref_zeros[0], _BYTES), (args.ref_Y[0], _NAMES[self.dtype_y]))

    def _packed(self, args: Q4Arguments, workspace, stream):
        m, n, k = args.problem_size
        refs = (args.ref_X, args.ref_W, args.ref_scales, args.ref_zeros, args.ref_Y)
        device = _device(ref[0] for ref in refs)
        if device is None:
            return None
        return _lib.Q4Args.from_buffer_copy(_PACK[_lib.Q4Args](
            self.dtype_x, self.dtype_y, self.dtype_scale, self.group, m, n, k, device,
            *(field for ref in refs for field in (_ptr(ref[0]), ref[1])), _stream_handle(stream)))


class BeamStep(_DecodeOperator):
    """cuasr_b200_beam_step."""
    _name = "cuasr_b200_beam_step"

    def __init__(self, dtype: DType = DType.F32, normalise: bool = True):
        super().__init__()
        self.dtype, self.normalise = _real(dtype), bool(normalise)

    def _types_match(self, args: BeamArguments) -> bool:
        return _typed((args.ref_logits[0], _NAMES[self.dtype]), (args.ref_scores[0], _NAMES[DType.F32]), (args.ref_finished[0], _FLAGS),
                      (args.ref_out_scores[0], _NAMES[DType.F32]), (args.ref_parents[0], _INDEX), (args.ref_tokens[0], _INDEX))

    def _packed(self, args: BeamArguments, workspace, stream):
        refs = (args.ref_scores, args.ref_finished, args.ref_out_scores, args.ref_parents, args.ref_tokens)
        device = _device((args.ref_logits[0], workspace, *(ref[0] for ref in refs)))
        if device is None:
            return None
        size = workspace.numel() * workspace.element_size() if hasattr(workspace, "numel") else 0
        packed = _lib.BeamArgs.from_buffer_copy(_PACK[_lib.BeamArgs](
            self.dtype, self.normalise, *args.problem_size, args.end_token, device, _ptr(args.ref_logits[0]), *args.ref_logits[1:],
            *(field for ref in refs for field in (_ptr(ref[0]), ref[1])), _ptr(workspace), size, _stream_handle(stream)))
        if workspace is not None and not hasattr(workspace, "numel"):       # an address: as large as was asked for
            packed.workspace_bytes = self._required_workspace(packed)
        return packed

    def _required_workspace(self, packed) -> int:
        return int(self._lib.cuasr_b200_beam_step_workspace_size(ctypes.byref(packed)))

    def get_workspace_size(self, args: BeamArguments) -> int:
        packed = self._pack(args, None, None)
        return 0 if packed is None else self._required_workspace(packed)


class ReorderStates(_DecodeOperator):
    """cuasr_b200_reorder_states."""
    _name = "cuasr_b200_reorder_states"

    def _types_match(self, args: ReorderArguments) -> bool:
        return _typed((args.ref_parents[0], _INDEX), (args.lengths, _INDEX))

    def _packed(self, args: ReorderArguments, workspace, stream):
        device = _device((args.ref_parents[0], args.lengths, *(x for s in args.states for x in (s.src, s.dst))))
        if device is None:
            return None
        pack, some = _PACK[_lib.State], args.lengths is not None
        moved = [pack(_ptr(s.src), _ptr(s.dst), *s.src_strides, *s.dst_strides, s.bytes, s.segments, s.positions, bool(s.ragged and some), 0)
                 for s in args.states if not (_empty(s.src) and _empty(s.dst))]
        states = (_lib.State * max(1, len(moved))).from_buffer_copy(b"".join(moved) or bytes(ctypes.sizeof(_lib.State)))
        packed = _lib.ReorderArgs.from_buffer_copy(_PACK[_lib.ReorderArgs](
            *args.problem_size, len(moved), _ptr(args.ref_parents[0]), args.ref_parents[1], _ptr(args.lengths), ctypes.addressof(states), device, 0,
            _stream_handle(stream)))
        packed.kept = states         # as long as the pointer to them
        return packed
