"""The decoding operators without a device: layouts of the C structs, refusals, views of state tensors."""
import ctypes
import os
import subprocess

import pytest
import torch

from cuasr_b200 import (BeamArguments, BeamStep, DType, Q4Arguments, Q4Product, ReorderArguments, ReorderStates, Srgemm, Op,
                        StateView, Status, _lib, state_view)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = {"cuasr_b200_q4_args_t": _lib.Q4Args, "cuasr_b200_beam_args_t": _lib.BeamArgs, "cuasr_b200_state_t": _lib.State,
           "cuasr_b200_reorder_args_t": _lib.ReorderArgs}
P = 1 << 20                   # an address that is never followed


def test_structs_match_the_header(tmp_path):
    lines = [f'printf("%zu", sizeof({name}));' + "".join(f'printf(" %zu", offsetof({name}, {field[0]}));' for field in struct._fields_)
             + 'printf("\\n");' for name, struct in STRUCTS.items()]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "cuasr_b200_decode.h"\nint main(void) {' + "\n".join(lines) + "return 0; }\n")
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "sizes"), str(src)],
                   check=True)
    out = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, struct in zip(out, STRUCTS.values()):
        want = [ctypes.sizeof(struct)] + [getattr(struct, field[0]).offset for field in struct._fields_]
        assert [int(v) for v in line.split()] == want, struct


def q4_args(m=2, n=8, k=64, ldx=64, ldw=32, lds=2, ldy=8, x=P, w=P, s=P, y=P, z=(None, 0)):
    return Q4Arguments((m, n, k), (x, ldx), (w, ldw), (s, lds), (y, ldy), z)


@pytest.mark.parametrize("change,status", [
    ({}, Status.kSuccess),
    ({"m": 0}, Status.kErrorInvalidProblem), ({"n": 0}, Status.kErrorInvalidProblem), ({"k": 0}, Status.kErrorInvalidProblem),
    ({"m": -1}, Status.kErrorInvalidProblem),
    ({"ldx": 63}, Status.kErrorInvalidProblem), ({"ldw": 31}, Status.kErrorInvalidProblem),
    ({"k": 63, "ldw": 31}, Status.kErrorInvalidProblem), ({"lds": 1}, Status.kErrorInvalidProblem),
    ({"ldy": 7}, Status.kErrorInvalidProblem), ({"z": (P, 1)}, Status.kErrorInvalidProblem), ({"z": (P + 1, 2)}, Status.kSuccess),
    ({"x": None}, Status.kErrorInvalidProblem), ({"w": None}, Status.kErrorInvalidProblem),
    ({"s": None}, Status.kErrorInvalidProblem), ({"y": None}, Status.kErrorInvalidProblem),
    ({"x": P + 1}, Status.kErrorMisalignedOperand), ({"y": P + 1}, Status.kErrorMisalignedOperand),
    ({"s": P + 1}, Status.kErrorMisalignedOperand), ({"w": P + 1}, Status.kSuccess),
])
def test_q4_refusals(change, status):
    op = Q4Product(DType.F16, group=32)
    assert op.can_implement(q4_args(**change)) == status
    assert op.initialize(q4_args(**change)) == status
    if status != Status.kSuccess:
        assert op(q4_args(**change)) == status
        assert Q4Product(DType.F16, group=32).run() == Status.kErrorInternal      # nothing initialised


def test_q4_types_and_groups():
    for group in (0, -32, 1, 48):
        assert Q4Product(DType.F16, group=group).can_implement(q4_args()) == Status.kErrorNotSupported
    assert Q4Product(DType.F16, group=1024).can_implement(q4_args()) == Status.kSuccess
    for bad in (DType.F64, DType.S32):
        with pytest.raises(ValueError):
            Q4Product(bad)
        packed = Q4Product(DType.F16, group=32)._pack(q4_args(), None, None)
        packed.dtype_y = int(bad)
        assert _lib.load().cuasr_b200_q4_product(ctypes.byref(packed)) == Status.kErrorInvalidDataType
    assert _lib.load().cuasr_b200_q4_product(None) == Status.kErrorInvalidProblem


@pytest.mark.parametrize("change,status", [
    ({"n": 2 ** 31 - 2 ** 17, "ldy": 2 ** 31}, Status.kSuccess), ({"n": 2 ** 31 - 1, "ldy": 2 ** 31}, Status.kErrorNotSupported),
    ({"k": 2 ** 31 - 2 ** 17, "ldx": 2 ** 31, "ldw": 2 ** 30, "lds": 2 ** 26}, Status.kSuccess),
    ({"k": 2 ** 31 - 1, "ldx": 2 ** 31, "ldw": 2 ** 30, "lds": 2 ** 26}, Status.kErrorNotSupported),
    ({"m": 32 * 65535}, Status.kSuccess), ({"m": 32 * 65535 + 1}, Status.kErrorNotSupported),
    ({"lds": 2 ** 40, "z": (P, 2 ** 40)}, Status.kSuccess),
])
def test_q4_limits(change, status):
    assert Q4Product(DType.F16, group=32).can_implement(q4_args(**change)) == status


def test_semiring_products_take_no_16_bit_types():
    for dtype in (DType.F16, DType.BF16):
        with pytest.raises(ValueError):
            Srgemm(Op.PLUS, Op.MULTIPLIES, dtype)
    desc, args = _lib.Desc(0, 1, int(DType.BF16), 0, 0, 0, 0, 0), _lib.Args()
    assert _lib.load().cuasr_b200_srgemm(ctypes.byref(desc), ctypes.byref(args)) == Status.kErrorInvalidDataType


def beam_args(batch=2, beams=3, vocab=10, keep=4, logits=(P, 30, 10), scores=(P, 3), out=(P, 4), parents=(P, 4), tokens=(P, 4),
              finished=(None, 0)):
    return BeamArguments((batch, beams, vocab, keep), logits, scores, out if out[0] != P else (P + 4096, out[1]), parents, tokens, finished)


@pytest.mark.parametrize("change,status", [
    ({}, Status.kSuccess), ({"finished": (P + 1, 3)}, Status.kSuccess), ({"logits": (P, 0, 0)}, Status.kSuccess),
    ({"batch": 0}, Status.kErrorInvalidProblem), ({"beams": 0}, Status.kErrorInvalidProblem),
    ({"vocab": 0}, Status.kErrorInvalidProblem), ({"keep": 0}, Status.kErrorInvalidProblem),
    ({"keep": 65, "out": (P, 65), "parents": (P, 65), "tokens": (P, 65)}, Status.kErrorNotSupported),
    ({"beams": 1025, "scores": (P, 1025)}, Status.kErrorNotSupported),
    ({"logits": (P, -1, 10)}, Status.kErrorInvalidProblem), ({"logits": (P, 30, -1)}, Status.kErrorInvalidProblem),
    ({"logits": (None, 30, 10)}, Status.kErrorInvalidProblem), ({"scores": (None, 3)}, Status.kErrorInvalidProblem),
    ({"scores": (P, 2)}, Status.kErrorInvalidProblem), ({"finished": (P, 2)}, Status.kErrorInvalidProblem),
    ({"out": (P, 3)}, Status.kErrorInvalidProblem), ({"parents": (P, 3)}, Status.kErrorInvalidProblem),
    ({"tokens": (P, 3)}, Status.kErrorInvalidProblem), ({"tokens": (None, 4)}, Status.kErrorInvalidProblem),
    ({"logits": (P + 2, 30, 10)}, Status.kErrorMisalignedOperand), ({"scores": (P + 2, 3)}, Status.kErrorMisalignedOperand),
    ({"out": (P + 2, 4)}, Status.kErrorMisalignedOperand), ({"parents": (P + 1, 4)}, Status.kErrorMisalignedOperand),
])
def test_beam_refusals(change, status):
    op = BeamStep(DType.F32)
    assert op.can_implement(beam_args(**change)) == status
    assert op.initialize(beam_args(**change), P) == status


def test_beam_scores_in_place_need_one_leading_dimension():
    args = beam_args(beams=3, keep=3)
    args.ref_out_scores = (P, 3)
    assert BeamStep().can_implement(args) == Status.kSuccess
    args.ref_out_scores = (P, 4)
    assert BeamStep().can_implement(args) == Status.kErrorInvalidProblem


def test_beam_workspace():
    op = BeamStep(DType.F32)
    need = op.get_workspace_size(beam_args())
    assert need > 0 and op.get_workspace_size(beam_args(keep=0)) == 0
    assert op.initialize(beam_args()) == Status.kErrorWorkspaceNull
    assert op(beam_args()) == Status.kErrorWorkspaceNull
    packed = op._pack(beam_args(), P, None)
    assert packed.workspace_bytes == need
    packed.workspace_bytes = need - 1
    assert _lib.load().cuasr_b200_beam_step(ctypes.byref(packed)) == Status.kErrorInvalidProblem
    packed.workspace_bytes, packed.workspace = need, P + 8
    assert _lib.load().cuasr_b200_beam_step(ctypes.byref(packed)) == Status.kErrorMisalignedOperand
    with pytest.raises(ValueError):
        BeamStep(DType.F64)


WRAP = 2 ** 32                # added to a size, 32 bits do not show it


def test_numbers_that_the_fields_do_not_hold_are_refused():
    bad = Status.kErrorInvalidProblem
    for change in ({"m": WRAP + 2}, {"n": WRAP + 8}, {"k": WRAP + 64}, {"ldx": 2 ** 64 + 64}, {"ldw": 2 ** 63}, {"z": (P, 2 ** 64 + 2)}):
        op = Q4Product(DType.F16, group=32)
        assert op.can_implement(q4_args(**change)) == bad and op.initialize(q4_args(**change)) == bad and op(q4_args(**change)) == bad
    assert Q4Product(DType.F16, group=WRAP + 32).can_implement(q4_args()) == bad
    for change in ({"batch": WRAP + 2}, {"beams": WRAP + 3}, {"vocab": WRAP + 10}, {"keep": WRAP + 4}, {"logits": (P, 2 ** 64 + 30, 10)},
                   {"out": (P, 2 ** 64 + 4)}):
        op = BeamStep(DType.F32)
        assert op.can_implement(beam_args(**change)) == bad and op(beam_args(**change), P) == bad and op.get_workspace_size(beam_args(**change)) == 0
    args = beam_args()
    args.end_token = WRAP + 2
    assert BeamStep(DType.F32).can_implement(args) == bad
    for states, change in (([view()], {"batch": WRAP + 2}), ([view()], {"keep": WRAP + 4}), ([view(positions=WRAP + 2)], {}), ([view(segments=WRAP + 2)], {}),
                           ([view(nbytes=2 ** 64 + 4)], {}), ([view(strides=(64, 16, 2 ** 64 + 8, 4))], {}), ([view()], {"parents": (P, 2 ** 64 + 4)})):
        assert ReorderStates().can_implement(reorder_args(states, **change)) == bad


class Room:
    """A workspace of so many bytes at an address."""
    def __init__(self, size, at=P):
        self.size, self.at = size, at

    def numel(self):
        return self.size

    def element_size(self):
        return 1

    def data_ptr(self):
        return self.at


def test_beam_initialize_checks_the_workspace():
    op = BeamStep(DType.F32)
    need = op.get_workspace_size(beam_args())
    for room, status in ((Room(need), Status.kSuccess), (Room(need + 1), Status.kSuccess), (Room(need - 1), Status.kErrorInvalidProblem),
                         (Room(0), Status.kErrorInvalidProblem), (Room(need, P + 8), Status.kErrorMisalignedOperand), (P + 8, Status.kErrorMisalignedOperand),
                         (Room(need - 1, P + 8), Status.kErrorInvalidProblem), (None, Status.kErrorWorkspaceNull)):
        fresh = BeamStep(DType.F32)
        assert fresh.initialize(beam_args(), room) == status
        if status != Status.kSuccess:
            assert fresh.run() == Status.kErrorInternal                   # nothing initialised
            packed = op._pack(beam_args(), room, None)                    # the library says the same
            assert _lib.load().cuasr_b200_beam_step(ctypes.byref(packed)) == status


def reorder_args(states, batch=2, beams=4, keep=4, parents=(P, 4), lengths=None):
    return ReorderArguments((batch, beams, keep), parents, states, lengths)


def view(src=P, dst=None, strides=(64, 16, 8, 4), dst_strides=None, nbytes=4, segments=2, positions=2, ragged=False):
    return StateView(src, src if dst is None else dst, strides, strides if dst_strides is None else dst_strides, nbytes, segments,
                     positions, ragged)


FAR = P + (1 << 30)


@pytest.mark.parametrize("states,change,status", [
    ([view()], {}, Status.kSuccess),
    ([], {}, Status.kSuccess),
    ([view()], {"batch": 0}, Status.kErrorInvalidProblem), ([view()], {"beams": 0}, Status.kErrorInvalidProblem),
    ([view()], {"keep": 0}, Status.kErrorInvalidProblem),
    ([view()], {"parents": (None, 4)}, Status.kErrorInvalidProblem), ([view()], {"parents": (P, 3)}, Status.kErrorInvalidProblem),
    ([view()], {"parents": (P + 2, 4)}, Status.kErrorMisalignedOperand),
    ([view(ragged=True)], {}, Status.kSuccess),                                            # no lengths: all positions
    ([view(ragged=True)], {"lengths": P + 2}, Status.kErrorMisalignedOperand),
    ([view(src=None)], {}, Status.kErrorInvalidProblem), ([view(nbytes=0)], {}, Status.kErrorInvalidProblem),
    ([view(segments=0)], {}, Status.kErrorInvalidProblem), ([view(positions=0)], {}, Status.kErrorInvalidProblem),
    ([view(strides=(64, -16, 8, 4))], {}, Status.kErrorInvalidProblem),
    # rows, segments or positions of a destination that share bytes
    ([view(strides=(64, 8, 8, 4))], {}, Status.kErrorInvalidProblem), ([view(strides=(0, 16, 8, 4))], {}, Status.kErrorInvalidProblem),
    ([view(strides=(64, 16, 8, 3))], {}, Status.kErrorInvalidProblem),
    ([view(dst=FAR, strides=(0, 16, 8, 4), dst_strides=(64, 16, 8, 4))], {}, Status.kSuccess),      # a source that is broadcast
    # in place
    ([view()], {"keep": 5, "parents": (P, 5)}, Status.kErrorInvalidProblem),
    ([view()], {"keep": 3}, Status.kSuccess),
    ([view(strides=(4096, 16, 8, 4))], {"beams": 40, "keep": 32, "parents": (P, 32)}, Status.kSuccess),
    ([view(strides=(4096, 16, 8, 4))], {"beams": 40, "keep": 33, "parents": (P, 33)}, Status.kErrorNotSupported),
    ([view(dst=FAR, strides=(4096, 16, 8, 4))], {"beams": 40, "keep": 33, "parents": (P, 33)}, Status.kSuccess),
    # source and destination that overlap otherwise
    ([view(dst=P + 16)], {}, Status.kErrorInvalidProblem), ([view(dst_strides=(128, 16, 8, 4))], {}, Status.kErrorInvalidProblem),
    ([view(dst=P + 128)], {}, Status.kSuccess),
    # the same tensor twice
    ([view(), view()], {}, Status.kErrorInvalidProblem), ([view(), view(src=FAR, dst=P)], {}, Status.kErrorInvalidProblem),
    ([view(dst=FAR), view(src=FAR, dst=2 * FAR)], {}, Status.kErrorInvalidProblem),
    ([view(src=P, dst=FAR), view(src=P, dst=2 * FAR)], {}, Status.kSuccess),
    ([view(src=P + 128 * i) for i in range(256)], {}, Status.kSuccess),
    ([view(src=P + 128 * i) for i in range(257)], {}, Status.kErrorNotSupported),
    ([view(strides=(1 << 62, 16, 8, 4))], {}, Status.kErrorInvalidProblem),
    # in place, the rows of one search that are only read are those of another that are written
    ([view(strides=(32, 16, 8, 4))], {"keep": 2}, Status.kErrorInvalidProblem),
    ([view(dst=FAR, strides=(32, 16, 8, 4), dst_strides=(32, 16, 8, 4))], {"keep": 2}, Status.kSuccess),
    # more columns than a grid has blocks for
    ([view(src=P + 1, strides=(1 << 42, 1 << 40, 1 << 40, 1), nbytes=1 << 40, segments=1, positions=1)], {}, Status.kErrorNotSupported),
    ([view(src=P, strides=(1 << 42, 1 << 40, 1 << 40, 1), nbytes=1 << 40, segments=1, positions=1)], {"batch": 1}, Status.kSuccess),
])
def test_reorder_refusals(states, change, status):
    op = ReorderStates()
    assert op.can_implement(reorder_args(states, **change)) == status
    if status != Status.kSuccess:
        assert op(reorder_args(states, **change)) == status


def test_nothing_to_reorder_needs_no_device():
    assert ReorderStates()(reorder_args([])) == Status.kSuccess


def test_states_without_elements_are_left_out():
    none = Room(0, 0)
    op = ReorderStates()
    assert op(reorder_args([view(src=none, strides=(0, 0, 0, 0), nbytes=0, segments=0, positions=0)] * 2)) == Status.kSuccess
    packed = op._pack(reorder_args([view(src=none, nbytes=0), view(), view(src=none, positions=0)]), None, None)
    assert packed.n_states == 1 and packed.states[0].src == P
    # a side with elements is not nothing, and what is wrong with the call is still wrong
    assert op.can_implement(reorder_args([view(src=none, dst=P)])) == Status.kErrorInvalidProblem
    assert op.can_implement(reorder_args([view(src=none)], keep=0)) == Status.kErrorInvalidProblem


@pytest.mark.parametrize("shape,position_dim", [((2, 3, 4, 0, 8), 3), ((2, 3, 4, 0, 8), None), ((2, 3, 4, 0, 10, 8), 4), ((2, 3, 0), None), ((2, 3, 0, 4), 2)])
def test_views_of_states_without_elements(shape, position_dim):
    x = torch.zeros(shape)
    v = state_view(x, position_dim=position_dim)
    assert v.src is x and v.dst is x and v.ragged == (position_dim is not None)
    with pytest.raises(ValueError):
        state_view(x, torch.zeros(*shape[:-1], shape[-1] + 1), position_dim)


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(64, dtype=torch.float16)
    assert Q4Product(DType.F16, group=32).can_implement(q4_args(x=x)) == Status.kErrorInvalidProblem
    assert BeamStep().can_implement(beam_args(scores=(x, 3))) == Status.kErrorInvalidProblem
    assert BeamStep().get_workspace_size(beam_args(scores=(x, 3))) == 0
    assert ReorderStates().initialize(reorder_args([view(src=x)])) == Status.kErrorInvalidProblem


class Typed:
    """An address with an element type."""
    def __init__(self, dtype):
        self.dtype = dtype

    def data_ptr(self):
        return P


def test_tensors_of_another_type_are_refused():
    half, single, wide, flag = (Typed(t) for t in (torch.float16, torch.float32, torch.int64, torch.bool))
    bad = Status.kErrorInvalidDataType
    for change in ({"x": single}, {"w": half}, {"w": wide}, {"s": single}, {"y": single}, {"z": (half, 2)}):
        op = Q4Product(DType.F16, group=32)
        assert op.can_implement(q4_args(**change)) == bad and op.initialize(q4_args(**change)) == bad
    for change in ({"logits": (half, 30, 10)}, {"scores": (half, 3)}, {"out": (half, 4)}, {"parents": (wide, 4)}, {"tokens": (single, 4)},
                   {"finished": (wide, 3)}):
        assert BeamStep().can_implement(beam_args(**change)) == bad and BeamStep().initialize(beam_args(**change), P) == bad
    assert BeamStep().can_implement(beam_args(finished=(flag, 3), scores=(single, 3))) == Status.kSuccess
    assert Q4Product(DType.F16, group=32).can_implement(q4_args(x=half, w=Typed(torch.uint8), y=half)) == Status.kSuccess
    for change in ({"parents": (wide, 4)}, {"lengths": wide}):
        assert ReorderStates().can_implement(reorder_args([view()], **change)) == bad


def test_a_device_that_is_not_there_is_refused():
    packed = Q4Product(DType.F16, group=32)._pack(q4_args(), None, None)
    packed.device = 1000
    assert _lib.load().cuasr_b200_q4_product(ctypes.byref(packed)) == Status.kErrorInvalidProblem
    packed.device = -1
    assert _lib.load().cuasr_b200_q4_product(ctypes.byref(packed)) == Status.kErrorInvalidProblem


def test_state_views():
    cache = torch.zeros(2, 3, 4, 10, 8, dtype=torch.bfloat16)              # heads before positions
    v = state_view(cache, position_dim=3)
    assert (v.src_strides, v.bytes, v.segments, v.positions, v.ragged) == ((1920, 640, 160, 16), 16, 4, 10, True)
    assert v.src_strides == tuple(v.dst_strides)
    v = state_view(cache[:, :, :, :7], position_dim=3)                     # the first seven positions
    assert (v.src_strides, v.bytes, v.segments, v.positions) == ((1920, 640, 160, 16), 16, 4, 7)
    v = state_view(cache[:, :, :, :7])                                     # the same, whole
    assert (v.src_strides, v.bytes, v.segments, v.positions, v.ragged) == ((1920, 640, 160, 0), 112, 4, 1, False)
    v = state_view(cache)
    assert (v.bytes, v.segments, v.positions) == (640, 1, 1)
    v = state_view(torch.zeros(2, 3, 10, 4, 8), position_dim=2)            # positions before heads
    assert (v.src_strides, v.bytes, v.segments, v.positions) == ((3840, 1280, 4, 128), 128, 1, 10)
    v = state_view(torch.zeros(10, 2, 3, 8).permute(1, 2, 0, 3), position_dim=2)      # positions outermost
    assert (v.src_strides, v.bytes, v.segments, v.positions) == ((96, 32, 4, 192), 32, 1, 10)
    v = state_view(torch.zeros(2, 3, 4, 5, 10, 8)[:, :, :, :, :6], position_dim=4)    # two dimensions in front that fold
    assert (v.segments, v.positions, v.bytes, v.src_strides[2]) == (20, 6, 32, 320)
    v = state_view(torch.zeros(2, 3))
    assert (v.bytes, v.segments, v.positions, v.src_strides) == (4, 1, 1, (12, 4, 4, 0))
    src, dst = torch.zeros(2, 3, 4, 8), torch.zeros(2, 5, 4, 16)[..., :8]  # other strides on the other side
    v = state_view(src, dst)
    assert (v.src_strides, v.dst_strides, v.bytes, v.segments) == ((384, 128, 32, 0), (1280, 256, 64, 0), 32, 4)


@pytest.mark.parametrize("make", [
    lambda: state_view(torch.zeros(3)), lambda: state_view(torch.zeros(2, 3, 4), torch.zeros(2, 3, 5)),
    lambda: state_view(torch.zeros(2, 3, 4), torch.zeros(2, 3, 4, dtype=torch.int32)),
    lambda: state_view(torch.zeros(2, 3, 4), torch.zeros(4, 3, 4)),
    lambda: state_view(torch.zeros(2, 3, 4), position_dim=1), lambda: state_view(torch.zeros(2, 3, 4), position_dim=3),
    lambda: state_view(torch.zeros(2, 3, 4, 8)[..., ::2], position_dim=2),            # gaps inside a position
    lambda: state_view(torch.zeros(2, 3, 4, 6, 10, 8)[:, :, :, :4], position_dim=4),  # two strides in front of the positions
])
def test_state_views_that_cannot_be_described(make):
    with pytest.raises(ValueError):
        make()


def test_the_header_is_plain_c(tmp_path):
    src = tmp_path / "decode.c"
    src.write_text('#include "cuasr_b200_decode.h"\nint main(void) { return 0; }\n')
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(src)], check=True)
