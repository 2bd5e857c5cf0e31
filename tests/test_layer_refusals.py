"""What route, routed_experts and the 4-bit conversions refuse, without a GPU.

The Python checks see CPU tensors (never a launch); the C entry points are called
with addresses that are never read, because the arguments are refused first.
"""

import ctypes

import pytest
import torch

from calibration_free_moe.reader import _ext
from calibration_free_moe.reader.experts import routed_experts
from calibration_free_moe.reader.microscale import Fp4Weights, dequantise_fp4, quantise_fp4
from calibration_free_moe.reader.router import route

AT = 0x10000


def refused(status, words):
    assert status == _ext.EINVAL
    assert words in _ext.library().cfmoe_last_error().decode()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        route(x, torch.zeros(8, 256, dtype=torch.bfloat16), 2)
    ids = torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        routed_experts(x, torch.zeros(1, 64, 256, dtype=torch.bfloat16),
                       torch.zeros(1, 32, 256, dtype=torch.bfloat16).transpose(1, 2), ids,
                       torch.ones(2, 1))
    with pytest.raises(ValueError, match="CUDA"):
        quantise_fp4(torch.zeros(64))
    with pytest.raises(ValueError, match="CUDA"):
        dequantise_fp4(Fp4Weights(torch.zeros(16, dtype=torch.uint8),
                                  torch.zeros(1, dtype=torch.uint8)))


def test_one_of_the_weights_in_4_bits_is_refused():
    x = torch.zeros(2, 256, dtype=torch.bfloat16)
    fp4 = Fp4Weights(torch.zeros(1, 64, 128, dtype=torch.uint8),
                     torch.zeros(1, 64, 8, dtype=torch.uint8))
    with pytest.raises(ValueError, match="both"):
        routed_experts(x, fp4, torch.zeros(1, 256, 32, dtype=torch.bfloat16),
                       torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, 1))


def test_shape_of_4_bit_weights():
    weights = Fp4Weights(torch.zeros(3, 5, 48, dtype=torch.uint8),
                         torch.zeros(3, 5, 3, dtype=torch.uint8))
    assert weights.shape == (3, 5, 96) and not weights.valid()


def call_route(hidden=256, experts=8, top_k=2, x=AT, router=AT, ids=AT, scratch=AT, tokens=1):
    return _ext.library().cfmoe_route(hidden, experts, top_k, 0, x, router, None, ids, AT, scratch,
                                      tokens, None)


@pytest.mark.parametrize("arguments,words", [
    (dict(hidden=200), "multiple of 128"), (dict(hidden=0), "multiple of 128"),
    (dict(hidden=65664), "at most 65536"), (dict(experts=0), "1 to 1024"), (dict(experts=1025), "1 to 1024"),
    (dict(top_k=0), "1 to 64"), (dict(top_k=9), "no more than there are"),
    (dict(experts=100, top_k=65), "1 to 64"), (dict(tokens=-1), "zero or more"),
    (dict(x=None), "NULL"), (dict(router=None), "NULL"), (dict(ids=None), "NULL"),
    (dict(scratch=None), "NULL"), (dict(x=AT + 2), "16-byte"), (dict(router=AT + 8), "16-byte"),
    (dict(scratch=AT + 4), "16-byte"), (dict(tokens=2_000_000_000), "too many tokens"),
])
def test_route_refuses(arguments, words):
    refused(call_route(**arguments), words)


def test_no_tokens_are_no_work():
    assert call_route(tokens=0) == 0
    assert call_experts(tokens=0) == 0
    lib = _ext.library()
    assert lib.cfmoe_quantise_fp4(0, 0, None, None, None, None) == 0
    assert lib.cfmoe_dequantise_fp4(0, None, None, None, None) == 0
    assert lib.cfmoe_route_scratch_bytes(0, 8) == 0
    assert lib.cfmoe_routed_experts_scratch_bytes(256, 64, 8, 2, 0, 0) == 0


def call_experts(hidden=256, width=64, experts=8, top_k=2, flags=0, gate_up=AT, gate_up_scales=None,
                 down=AT, down_scales=None, x=AT, out=AT, scratch=AT, tokens=1):
    return _ext.library().cfmoe_routed_experts(
        hidden, width, experts, top_k, flags, gate_up, gate_up_scales, down, down_scales, x, AT, AT,
        None, out, scratch, tokens, None)


@pytest.mark.parametrize("arguments,words", [
    (dict(hidden=192), "multiple of 128"), (dict(hidden=4224), "at most 4096"),
    (dict(width=8), "multiple of 16"), (dict(width=0), "multiple of 16"),
    (dict(width=48, flags=_ext.FP4), "of 32"), (dict(width=4112), "at most 4096"),
    (dict(experts=0), "4096"), (dict(experts=4097), "4096"), (dict(top_k=65), "1 to 64"),
    (dict(tokens=4097), "8192"), (dict(tokens=-1), "8192"), (dict(tokens=2_000_000_000), "8192"),
    (dict(gate_up=None), "NULL"), (dict(down=None), "NULL"), (dict(x=None), "NULL"),
    (dict(out=None), "NULL"), (dict(scratch=None), "NULL"),
    (dict(flags=_ext.FP4), "NULL"), (dict(flags=_ext.FP4, gate_up_scales=AT), "NULL"),
    (dict(x=AT + 8), "16-byte"), (dict(down=AT + 2), "16-byte"), (dict(out=AT + 4), "16-byte"),
    (dict(flags=_ext.FP4, gate_up_scales=AT + 4, down_scales=AT), "16-byte"),
])
def test_routed_experts_refuses(arguments, words):
    refused(call_experts(**arguments), words)


def test_scratch_sizes():
    lib = _ext.library()
    # activations [pairs, 2, I] BF16 and one FP32 partial row per pair at least
    for flags in (0, _ext.FP4):
        for tokens in (1, 7, 500):
            size = lib.cfmoe_routed_experts_scratch_bytes(2048, 768, 128, 8, flags, tokens)
            assert size >= tokens * 8 * (4 * 768 + 4 * 2048)
    assert lib.cfmoe_routed_experts_scratch_bytes(100, 64, 8, 2, 0, 1) == -_ext.EINVAL
    assert lib.cfmoe_route_scratch_bytes(3, 2000) == -_ext.EINVAL


def test_conversions_refuse():
    lib = _ext.library()
    refused(lib.cfmoe_quantise_fp4(-1, 0, AT, AT, AT, None), "blocks")
    refused(lib.cfmoe_quantise_fp4(1, 0, None, AT, AT, None), "NULL")
    refused(lib.cfmoe_quantise_fp4(1, 0, AT + 2, AT, AT, None), "16-byte")
    refused(lib.cfmoe_quantise_fp4(1, 0, AT, AT + 2, AT, None), "4-byte")
    refused(lib.cfmoe_dequantise_fp4(1, AT, None, AT, None), "NULL")
    refused(lib.cfmoe_dequantise_fp4(1, AT, AT, AT + 8, None), "16-byte")
    refused(lib.cfmoe_dequantise_fp4((1 << 40) + 1, AT, AT, AT, None), "blocks")
