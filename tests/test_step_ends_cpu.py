"""Refusals of the operators around a model's layers, and their plain forms, without a GPU."""
import math
from array import array

import numpy as np
import pytest
import torch

import plain_step_ends as plain
from kv_cache_optimization_for_llm_amd.ops import kernels as K
from kv_cache_optimization_for_llm_amd.ops.library import KernelError, check, hip_lib, launches


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def f32(*shape):
    return torch.zeros(shape)


def marks(*shape):
    return torch.zeros(shape, dtype=torch.uint8)


@pytest.mark.parametrize("bad", [
    dict(out=f32(3, 40)),
    dict(logits=f32(40)),
    dict(logits=f32(2, 80)[:, ::2]),
    dict(logits=f32(1, 40).expand(2, 40)),
    dict(row_seat=i32(2)),
    dict(marks=marks(4, 40)),
    dict(marks=marks(4, 41), row_seat=i32(2)),
    dict(counts=i32(4, 40)),
    dict(repetition=f32(2)),
    dict(marks=marks(4, 40), row_seat=i32(2), presence=f32(2)),
    dict(marks=marks(4, 40), row_seat=i32(2), counts=i32(3, 40)),
    dict(allowed=i32(1, 2)),
    dict(allowed=i32(1, 1), allowed_row=i32(2)),
    dict(allowed=i32(0, 2), allowed_row=i32(2)),
    dict(bias=(i32(2), i32(5), f32(5))),
    dict(bias=(i32(3), i32(5), f32(4))),
    dict(bias=(i32(3), i32(5))),
    dict(),                                 # all of it fits, but it is not on a GPU
])
def test_adjust_logits_refuses(bad):
    args = dict(logits=f32(2, 40), out=f32(2, 40))
    args.update(bad)
    with pytest.raises(KernelError):
        K.adjust_logits(args.pop("logits"), args.pop("out"), **args)


@pytest.mark.parametrize("bad", [
    dict(inv_temperature=None),
    dict(uniform=None),
    dict(rng_key=i32(2)),
    dict(rng_key=i32(2), rng_step=i32(2)),
    dict(inv_temperature=f32(3)),
    dict(top_k=i32(1)),
    dict(top_k=f32(2)),
    dict(top_p=f32(2, 1)),
    dict(kept=i32(3)),
    dict(logprob=f32(1)),
    dict(host_tokens=i32(2)),               # not pinned
    dict(),
])
def test_sample_truncated_refuses(bad):
    args = dict(inv_temperature=f32(2), uniform=f32(2))
    args.update(bad)
    with pytest.raises(KernelError):
        K.sample_truncated(f32(2, 40), i32(2), **args)


def test_tables_and_rows_refuse():
    with pytest.raises(KernelError):
        K.grow_tables(i32(4, 8), i32(3), i32(2), i32(3), 16, i32(9))
    with pytest.raises(KernelError):
        K.grow_tables(i32(4), i32(3), i32(3), i32(3), 16, i32(9))
    with pytest.raises(KernelError):
        K.grow_tables(i32(4, 8), i32(3), i32(3), i32(3), 16, i32(9), i32(3))
    with pytest.raises(KernelError):
        K.grow_tables(i32(4, 8), i32(3), i32(3), i32(3), 16, i32(9))
    with pytest.raises(KernelError):
        K.step_rows(i32(3), i32(3), i32(3), [i32(4, 8)], 16, i32(3), i32(5), i32(5), [i32(5)])
    with pytest.raises(KernelError):
        K.step_rows(i32(3), i32(3), i32(3), [i32(4, 8)], 16, i32(4), i32(5), i32(5), [i32(6)])
    with pytest.raises(KernelError):
        K.step_rows(i32(3), i32(3), i32(3), [i32(4, 8)], 16, i32(4), i32(5), i32(5), [])
    with pytest.raises(KernelError):
        K.step_rows(i32(3), i32(3), i32(3), [i32(8)], 16, i32(4), i32(5), i32(5), [i32(5)])
    with pytest.raises(KernelError):
        K.step_rows(i32(3), i32(3), i32(3), [i32(4, 8)], 16, i32(4), i32(5), i32(5), [i32(5)])
    with pytest.raises(KernelError):
        K.count_tokens(marks(2, 9), i32(2, 8), i32(3), i32(3))
    with pytest.raises(KernelError):
        K.count_tokens(marks(2, 9), None, i32(3), i32(2))
    with pytest.raises(KernelError):
        K.count_tokens(marks(2, 9), i32(2, 9), i32(3), i32(3))


def test_plain_truncated_by_hand():
    x = [0.0, math.log(4.0), math.log(3.0), math.log(2.0), -math.inf, math.nan]
    # weights 1, 4, 3, 2 of 10
    assert plain.truncated(x, 1.0, u=0.0)[:2] == (0, 4)
    assert plain.truncated(x, 1.0, u=0.11)[:2] == (1, 4)
    assert plain.truncated(x, 1.0, top_k=2, u=0.6)[:2] == (2, 2)
    assert plain.truncated(x, 1.0, top_p=0.75, u=0.99)[:2] == (3, 3)         # 4 + 3 < 7.5
    assert plain.truncated(x, 1.0, top_p=0.65, u=0.99)[:2] == (2, 2)
    assert plain.truncated(x, 1.0, top_k=2, top_p=0.5, u=0.99)[:2] == (1, 1)  # 4 of 7
    assert plain.truncated(x, 1.0, min_p=0.6, u=0.99)[:2] == (2, 2)
    token, kept, lp = plain.truncated(x, 1.0, top_k=2, u=0.6)
    assert abs(lp - math.log(3 / 7)) < 1e-14
    assert plain.truncated(x, 0.0)[:2] == (1, 1)
    assert plain.truncated([math.nan, -math.inf], 1.0)[:2] == (-1, 0)
    assert plain.truncated([0.0, math.inf], 1.0)[:2] == (-1, 0)


def test_plain_tables_by_hand():
    table, offsets = plain.grow_tables(np.full((3, 4), -1), [2, 0], [1, 0], [33, 16], 16, [7, 8, 9, 10])
    assert offsets.tolist() == [0, 2, 3]
    assert table.tolist() == [[9, -1, -1, -1], [-1] * 4, [-1, 7, 8, -1]]
    q, pos, seat, slots = plain.step_rows([2, 0, 1], [15, 3, 0], [2, 1, 0], [table], 16)
    assert q == [0, 2, 2, 3] and pos == [15, 16, 0] and seat == [2, 2, 0] and slots == [[-1, 112, 144]]


@pytest.mark.parametrize("message, call", [
    (r"row_seat is \(3,\), expected \(2,\)", lambda: K.adjust_logits(f32(2, 40), f32(2, 40), row_seat=i32(3), marks=marks(4, 40))),
    (r"marks is \(4, 41\), expected \(4, 40\)", lambda: K.adjust_logits(f32(2, 40), f32(2, 40), row_seat=i32(2), marks=marks(4, 41))),
    (r"marks is torch.int32", lambda: K.adjust_logits(f32(2, 40), f32(2, 40), row_seat=i32(2), marks=i32(4, 40))),
    (r"counts must be contiguous", lambda: K.adjust_logits(f32(2, 40), f32(2, 40), row_seat=i32(2), marks=marks(4, 40), counts=i32(40, 4).t())),
    (r"allowed is \(1, 1\), expected \(1, 2\)", lambda: K.adjust_logits(f32(2, 40), f32(2, 40), allowed=i32(1, 1), allowed_row=i32(2))),
    (r"bias_start is \(2,\), expected \(3,\)", lambda: K.adjust_logits(f32(2, 40), f32(2, 40), bias=(i32(2), i32(5), f32(5)))),
    (r"bias_value is \(4,\), expected \(5,\)", lambda: K.adjust_logits(f32(2, 40), f32(2, 40), bias=(i32(3), i32(5), f32(4)))),
    (r"bias is \(start, token, value\)", lambda: K.adjust_logits(f32(2, 40), f32(2, 40), bias=(None, i32(5), f32(5)))),
    (r"bias is \(start, token, value\)", lambda: K.adjust_logits(f32(2, 40), f32(2, 40), bias=(i32(3), i32(5), None))),
    (r"out .* is not float32", lambda: K.adjust_logits(f32(2, 40), f32(2, 40).bfloat16())),
    (r"repetition: expected a tensor", lambda: K.adjust_logits(f32(2, 40), f32(2, 40), row_seat=i32(2), marks=marks(4, 40), repetition=1.5)),
    (r"not on a GPU", lambda: K.adjust_logits(f32(2, 40), f32(2, 40))),
    (r"inv_temperature is \(3,\)", lambda: K.sample_truncated(f32(2, 40), i32(2), inv_temperature=f32(3), uniform=f32(2))),
    (r"out_tokens is \(3,\)", lambda: K.sample_truncated(f32(2, 40), i32(3), inv_temperature=f32(2), uniform=f32(2))),
    (r"logits are torch.bfloat16", lambda: K.sample_truncated(f32(2, 40).bfloat16(), i32(2), inv_temperature=f32(2), uniform=f32(2))),
    (r"top_k is torch.float32", lambda: K.sample_truncated(f32(2, 40), i32(2), inv_temperature=f32(2), uniform=f32(2), top_k=f32(2))),
    (r"not on a GPU", lambda: K.sample_truncated(f32(2, 40), i32(2), inv_temperature=f32(2), uniform=f32(2))),
    (r"held is \(2,\)", lambda: K.grow_tables(i32(4, 8), i32(3), i32(2), i32(3), 16, i32(9))),
    (r"offsets is \(3,\)", lambda: K.grow_tables(i32(4, 8), i32(3), i32(3), i32(3), 16, i32(9), i32(3))),
    (r"table must be contiguous", lambda: K.grow_tables(i32(8, 4).t(), i32(3), i32(3), i32(3), 16, i32(9))),
    (r"not on a GPU", lambda: K.grow_tables(i32(4, 8), i32(3), i32(3), i32(3), 16, i32(9))),
    (r"q_start is \(3,\)", lambda: K.step_rows(i32(3), i32(3), i32(3), [i32(4, 8)], 16, i32(3), i32(5), i32(5), [i32(5)])),
    (r"slots is \(6,\)", lambda: K.step_rows(i32(3), i32(3), i32(3), [i32(4, 8)], 16, i32(4), i32(5), i32(5), [i32(6)])),
    (r"not on a GPU", lambda: K.step_rows(i32(3), i32(3), i32(3), [i32(4, 8)], 16, i32(4), i32(5), i32(5), [i32(5)])),
    (r"counts is \(2, 8\)", lambda: K.count_tokens(marks(2, 9), i32(2, 8), i32(3), i32(3))),
    (r"not on a GPU", lambda: K.count_tokens(marks(2, 9), i32(2, 9), i32(3), i32(3)))])
def test_refusals_say_why(message, call):
    with pytest.raises(KernelError, match=message):
        call()


def test_native_launches_take_gpu_tensors_only():
    """Whatever they do not take goes to the checks in Python: too few arguments, wrong objects, tensors of the host."""
    native = launches()
    assert native is not None, "torch's headers are here: it has to build"
    calls = dict(adjust_logits=[f32(2, 40), f32(2, 40), i32(2), marks(3, 40), i32(3, 40), f32(2), f32(2), f32(2), (i32(3), i32(5), f32(5)), i32(2), i32(1, 2)],
                 count_tokens=[marks(3, 40), i32(3, 40), i32(5), i32(5)],
                 sample_truncated=[f32(2, 40), i32(2), f32(2), i32(2), f32(2), f32(2), f32(2), None, None, i32(2), f32(2), None, 0],
                 grow_tables=[i32(3, 4), i32(2), i32(2), i32(2), i32(9), i32(3), 16],
                 step_rows=[i32(2), i32(2), i32(2), [i32(3, 4)], 16, i32(3), i32(5), i32(5), [i32(5)]])
    for name, args in calls.items():
        call = getattr(native, name)
        assert call(*args, 0, 0) is None and call(*args, -1, 0) is None and call(*args) is None and call() is None
        for i in range(len(args)):
            for other in (None, 5, "a", 1 << 80, [], (1, 2), object()):
                assert call(*args[:i], other, *args[i + 1:], 0, 0) is None, (name, i)
    with pytest.raises(TypeError):
        native.bind(1, 2)


def test_a_launch_needs_its_tensors():
    """What the C entries refuse before any launch: addresses that are not there."""
    lib = hip_lib()
    none, one = array("q", [0] * 16), array("q", [4, 4])
    at, size = none.buffer_info()[0], one.buffer_info()[0]
    for call in (lambda: lib.kva_grow_tables(at, 4, 4, 2, 16, 3, 0), lambda: lib.kva_step_rows(at, size, 2, 1, 16, 2, 0),
                 lambda: lib.kva_count_tokens(0, 0, 2, 9, 0, 0, 3, 0), lambda: lib.kva_adjust_logits(at, 64, 40, 64, 0, 40, 2, 40, 0, 3, 0, 0),
                 lambda: lib.kva_sample_truncated(at, 64, 40, 2, 40, 0, 0, 0, 0)):
        with pytest.raises(KernelError):
            check(call(), "a launch")


def meta(*shape, dtype=torch.int32):
    return torch.empty(shape, dtype=dtype, device="meta")


MANY = (1 << 32) + 3            # 3, to who looks at 32 bits of it


@pytest.mark.parametrize("call", [
    lambda: K.adjust_logits(meta(MANY, 1, dtype=torch.float32), meta(MANY, 1, dtype=torch.float32)),
    lambda: K.adjust_logits(meta(2, MANY, dtype=torch.float32), meta(2, MANY, dtype=torch.float32)),
    lambda: K.adjust_logits(f32(2, 40), f32(2, 40), bias=(i32(3), meta(MANY), meta(MANY, dtype=torch.float32))),
    lambda: K.adjust_logits(meta(2, 40, dtype=torch.float32), meta(2, 40, dtype=torch.float32), row_seat=meta(2),
                            marks=meta(MANY, 40, dtype=torch.uint8)),
    lambda: K.sample_truncated(meta(MANY, 1, dtype=torch.float32), meta(MANY), inv_temperature=meta(MANY, dtype=torch.float32),
                               uniform=meta(MANY, dtype=torch.float32)),
    lambda: K.count_tokens(meta(MANY, 9, dtype=torch.uint8), None, meta(3), meta(3)),
    lambda: K.count_tokens(meta(3, 9, dtype=torch.uint8), None, meta(MANY), meta(MANY)),
    lambda: K.grow_tables(meta(MANY, 8), meta(3), meta(3), meta(3), 16, meta(9)),
    lambda: K.grow_tables(meta(4, 8), meta(3), meta(3), meta(3), 16, meta(MANY)),
    lambda: K.grow_tables(meta(4, 8), meta(3), meta(3), meta(3), MANY, meta(9)),
    lambda: K.grow_tables(meta(4, 8), meta(3), meta(3), meta(3), 2.5, meta(9)),
    lambda: K.step_rows(meta(3), meta(3), meta(3), [meta(4, 8)], -MANY, meta(4), meta(5), meta(5), [meta(5)]),
    lambda: K.step_rows(meta(3), meta(3), meta(3), [meta(4, 8)], "16", meta(4), meta(5), meta(5), [meta(5)]),
    lambda: K.step_rows(meta(3), meta(3), meta(3), [meta(MANY, 8)], 16, meta(4), meta(5), meta(5), [meta(5)]),
    lambda: K.step_rows(meta(3), meta(3), meta(3), [meta(4, 8)], 16, meta(4), meta(MANY), meta(MANY), [meta(MANY)])])
def test_sizes_that_32_bits_do_not_hold_are_refused(call):
    with pytest.raises(KernelError, match="32 bits"):
        call()


def test_sizes_that_a_launch_cannot_count_are_refused():
    lib = hip_lib()
    for call in (lambda: lib.kva_count_tokens(64, 0, 2, 9, 64, 64, (1 << 31) - 255, 0),
                 lambda: lib.kva_adjust_logits(array("q", [64] * 11).buffer_info()[0], 64, 40, 64, 0, 40, 2, 40, 2, (1 << 31) - 1, 1, 0)):
        with pytest.raises(KernelError, match="bad sizes|biases"):
            check(call(), "a launch")
