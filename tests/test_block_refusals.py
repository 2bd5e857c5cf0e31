"""What the operators around the experts refuse, without a GPU.

The Python checks see CPU tensors (never a launch); the C entry points are called
with addresses that are never read, because the arguments are refused first.
"""

import sys

import pytest
import torch

from calibration_free_moe.reader import _ext
from calibration_free_moe.reader.adapters import _overlap, apply_adapters
from calibration_free_moe.reader.dispatch import (ExpertOrder, combine_rows, gather_rows,
                                                  sort_by_expert)
from calibration_free_moe.reader.norms import join_block, norm_rows

AT = 0x10000
INT32_MAX = 2 ** 31 - 1


def refused(status, words):
    assert status == _ext.EINVAL
    assert words in _ext.library().cfmoe_last_error().decode()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    ids = torch.zeros(2, 1, dtype=torch.int32)
    order = ExpertOrder(torch.zeros(3, dtype=torch.int32), ids, ids.flatten())
    with pytest.raises(ValueError, match="CUDA"):
        sort_by_expert(ids, 2)
    with pytest.raises(ValueError, match="CUDA"):
        gather_rows(x, order)
    with pytest.raises(ValueError, match="CUDA"):
        combine_rows(x, order)
    with pytest.raises(ValueError, match="CUDA"):
        norm_rows(x, torch.ones(256, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA"):
        join_block(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        apply_adapters(x, x, torch.zeros(1, 8, 256, dtype=torch.bfloat16),
                       torch.zeros(1, 256, 8, dtype=torch.bfloat16), ids.flatten())


def call_sort(experts=8, top_k=2, ids=AT, offsets=AT, places=AT, pairs=AT, scratch=AT, tokens=1):
    return _ext.library().cfmoe_sort_by_expert(experts, top_k, 0, ids, None, offsets, places, pairs,
                                               scratch, tokens, None)


@pytest.mark.parametrize("arguments,words", [
    (dict(experts=0), "1 to 4096"), (dict(experts=4097), "1 to 4096"), (dict(top_k=0), "1 to 64"),
    (dict(top_k=65), "1 to 64"), (dict(tokens=-1), "2^30"), (dict(tokens=INT32_MAX), "2^30"),
    (dict(tokens=(1 << 29) + 1), "2^30"), (dict(ids=None), "NULL"), (dict(offsets=None), "NULL"),
    (dict(places=None), "NULL"), (dict(pairs=None), "NULL"),
    (dict(tokens=100000, scratch=None), "NULL"),
])
def test_sort_refuses(arguments, words):
    refused(call_sort(**arguments), words)


def call_rows(which, hidden=64, top_k=2, tokens=1, rows=AT, places=AT, out=AT):
    lib = _ext.library()
    if which == "gather":
        return lib.cfmoe_gather_rows(hidden, top_k, 0, rows, places, out, tokens, None)
    if which == "combine":
        return lib.cfmoe_combine_rows(hidden, top_k, 0, rows, places, None, out, tokens, None)
    return lib.cfmoe_combine_rows_backward(hidden, top_k, 0, rows, AT, places, None, AT, out, tokens,
                                           None)


@pytest.mark.parametrize("which", ["gather", "combine", "backward"])
@pytest.mark.parametrize("arguments,words", [
    (dict(hidden=0), "2^20"), (dict(hidden=(1 << 20) + 1), "2^20"), (dict(top_k=0), "1 to 64"),
    (dict(top_k=65), "1 to 64"), (dict(tokens=-1), "2^30"), (dict(tokens=INT32_MAX), "2^30"),
    (dict(rows=None), "NULL"), (dict(places=None), "NULL"),
])
def test_rows_refuse(which, arguments, words):
    refused(call_rows(which, **arguments), words)


def test_rows_refuse_no_output():
    refused(call_rows("gather", out=None), "NULL")
    refused(call_rows("combine", out=None), "NULL")
    lib = _ext.library()
    refused(lib.cfmoe_combine_rows_backward(64, 2, 0, AT, None, AT, None, AT, AT, 1, None), "NULL")
    # nothing asked for is no work
    assert lib.cfmoe_combine_rows_backward(64, 2, 0, AT, AT, AT, None, None, None, 1, None) == 0


def call_join(hidden_size=64, flags=0, hidden=AT, block=AT, post=None, gate=None, next_weight=None,
              epsilon=1e-6, joined=AT, out=AT, tokens=1):
    return _ext.library().cfmoe_join_block(hidden_size, flags, hidden, block, post, gate, 1.0,
                                           next_weight, epsilon, joined, out, None, tokens, None)


@pytest.mark.parametrize("arguments,words", [
    (dict(hidden_size=0), "1 to 8192"), (dict(hidden_size=8193), "1 to 8192"),
    (dict(tokens=-1), "zero or more"), (dict(epsilon=0.0), "epsilon"),
    (dict(epsilon=-1.0), "epsilon"), (dict(epsilon=float("nan")), "epsilon"),
    (dict(epsilon=float("inf")), "epsilon"), (dict(hidden=None), "NULL"),
    (dict(joined=None), "NULL"), (dict(next_weight=AT, out=None), "NULL"),
    (dict(block=None), "NULL"), (dict(flags=_ext.GATE_ROW), "NULL"),
    (dict(block=None, post=AT, next_weight=AT), "with a block"),
    (dict(block=None, gate=AT, flags=_ext.GATE_ROW, next_weight=AT), "with a block"),
    (dict(gate=AT, flags=_ext.GATE_FULL | _ext.GATE_FP32), "rows' type"),
])
def test_join_refuses(arguments, words):
    refused(call_join(**arguments), words)


def call_back(hidden_size=64, flags=0, hidden=AT, block=AT, post=None, gate=None, next_weight=None,
              statistics=AT, grad_joined=AT, grad_next=None, to=(AT, AT, None, None, None),
              scratch=AT, tokens=1):
    return _ext.library().cfmoe_join_block_backward(
        hidden_size, flags, hidden, block, post, gate, 1.0, next_weight, statistics, grad_joined,
        grad_next, *to, scratch, tokens, None)


@pytest.mark.parametrize("arguments,words", [
    (dict(hidden_size=8200), "1 to 8192"), (dict(tokens=-5), "zero or more"),
    (dict(hidden=None), "NULL"), (dict(grad_next=AT), "NULL"),
    (dict(post=AT, statistics=None), "NULL"),
    (dict(next_weight=AT, to=(AT, AT, None, None, AT)), "NULL"),
    (dict(to=(AT, AT, AT, None, None)), "NULL"), (dict(to=(AT, AT, None, AT, None)), "NULL"),
    (dict(post=AT, to=(AT, AT, AT, None, None), scratch=None), "NULL"),
    (dict(gate=None, flags=_ext.GATE_CHANNEL), "NULL"),
    (dict(block=None), "with a block"),
    (dict(gate=AT, flags=_ext.GATE_FULL | _ext.GATE_FP32), "rows' type"),
])
def test_join_backward_refuses(arguments, words):
    refused(call_back(**arguments), words)


def call_adapters(hidden=64, outputs=64, rank=8, adapters=2, base=AT, x=AT, encoder=AT, decoder=AT,
                  slots=AT, out=AT, scratch=AT, strides=(64, 64, 64), tokens=1):
    return _ext.library().cfmoe_apply_adapters(
        hidden, outputs, rank, adapters, 0, base, strides[0], x, strides[1], encoder, decoder, slots,
        None, out, strides[2], scratch, tokens, None)


@pytest.mark.parametrize("arguments,words", [
    (dict(hidden=60), "multiples of 8"), (dict(hidden=0), "multiples of 8"),
    (dict(hidden=65544), "65536"), (dict(outputs=4), "multiples of 8"),
    (dict(outputs=65544), "65536"), (dict(rank=12), "rank"), (dict(rank=0), "rank"),
    (dict(rank=264), "rank"), (dict(adapters=0), "4096"), (dict(adapters=4097), "4096"),
    (dict(tokens=-1), "2^24"), (dict(tokens=(1 << 24) + 1), "2^24"),
    (dict(base=None), "NULL"), (dict(x=None), "NULL"), (dict(encoder=None), "NULL"),
    (dict(decoder=None), "NULL"), (dict(slots=None), "NULL"), (dict(out=None), "NULL"),
    (dict(scratch=None), "NULL"), (dict(x=AT + 2), "16-byte"),
    (dict(base=AT + 8), "16-byte"), (dict(scratch=AT + 8), "16-byte"), (dict(out=AT + 4), "16-byte"), (dict(decoder=AT + 8), "16-byte"),
    (dict(strides=(60, 64, 64)), "strides"), (dict(strides=(64, 68, 64)), "strides"),
    (dict(strides=(64, 64, 56)), "strides"), (dict(strides=(-64, 64, 64)), "strides"),
])
def test_adapters_refuse(arguments, words):
    refused(call_adapters(**arguments), words)


def test_no_tokens_are_no_work():
    for which in ("gather", "combine", "backward"):
        assert call_rows(which, tokens=0) == 0
    assert call_join(tokens=0) == 0
    assert call_adapters(tokens=0) == 0
    assert call_back(tokens=0, hidden=None) == 0


def test_scratch_sizes():
    lib = _ext.library()
    assert lib.cfmoe_sort_by_expert_scratch_bytes(16, 8, 4096) == 0
    assert lib.cfmoe_sort_by_expert_scratch_bytes(100000, 8, 128) >= 129 * 4
    assert lib.cfmoe_sort_by_expert_scratch_bytes(1, 65, 8) == -_ext.EINVAL
    assert lib.cfmoe_join_block_backward_scratch_bytes(100, 2, 5) == 5 * 2 * 100 * 4
    assert lib.cfmoe_join_block_backward_scratch_bytes(9000, 2, 5) == -_ext.EINVAL
    adapters = lib.cfmoe_apply_adapters_scratch_bytes
    assert adapters(64, 64, 40, 4, 3, 0) >= 3 * 40 * 4
    assert adapters(2048, 64, 40, 4, 3, 0) >= 8 * 3 * 40 * 4
    assert adapters(64, 64, 16, 4, 5000, 0) >= 5000 * (16 * 4 + 8) + 5 * 4
    assert adapters(64, 64, 16, 4, 1 << 24, 0) >= (1 << 24) * 16 * 4
    assert adapters(64, 64, 16, 4, 3, 0) == 0  # one launch, unless out is what others still read
    assert adapters(64, 64, 16, 4, 3, 1) >= 3 * 16 * 4
    assert adapters(64, 64, 15, 4, 3, 0) == -_ext.EINVAL
    assert adapters(60, 64, 16, 4, 3, 0) == -_ext.EINVAL
    assert adapters(64, 60, 16, 4, 3, 0) == -_ext.EINVAL


def test_overlaps_of_out():
    wide = torch.zeros(6, 64, dtype=torch.bfloat16)
    out = wide[:, 16:32]
    assert not _overlap(out, wide[:, 16:32])            # the same rows
    assert not _overlap(out, wide[:, 32:48])            # columns behind
    assert not _overlap(out, wide[:, :16])              # columns before
    assert _overlap(out, wide[:, 24:40])
    assert _overlap(out, wide[:, 8:24])
    assert _overlap(out, wide[:, 16:40])
    assert _overlap(wide[:4, :16], wide[1:5, :16])      # the same columns, other rows
    assert _overlap(out, wide[1:2, 16:32].expand(6, 16))
    assert not _overlap(out, torch.zeros(6, 16, dtype=torch.bfloat16))
    assert _overlap(wide[:1, :16], wide[:1, 8:24])
    assert not _overlap(wide[:1, :16], wide[:1, 16:32])


def test_operators_module_is_of_this_library(monkeypatch):
    module = _ext.operators()
    assert module.ABI_VERSION == _ext.ABI_VERSION
    _ext.operators.cache_clear()
    with monkeypatch.context() as patch:
        patch.setattr(module, "ABI_VERSION", _ext.ABI_VERSION - 1)
        with pytest.raises(RuntimeError, match="ABI mismatch"):
            _ext.operators()
    with monkeypatch.context() as patch:
        patch.setitem(sys.modules, "calibration_free_moe.reader._torch", None)
        patch.delattr("calibration_free_moe.reader._torch")
        with pytest.raises(RuntimeError, match="_torch.so is missing"):
            _ext.operators()
    assert _ext.operators() is module
