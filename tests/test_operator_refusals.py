"""CPU tier: the C entry points of the gate and MXFP4 operators refuse bad arguments before any device
work, and their Python calls refuse host tensors."""
import ctypes

import pytest
import torch

from ferry_amd import expert_ops as ops
from ferry_amd._lib import last_error, lib


def route(tokens=4, experts=64, topk=6, groups=1, topk_groups=1, dtype=1, top2=0):
    return lib().ferry_route_experts(None, dtype, tokens, experts, topk, 0, None, groups, topk_groups, top2, 1,
                                     1.0, None, None, None)


@pytest.mark.parametrize('bad,word', [
    (dict(tokens=-1), 'sizes'), (dict(experts=0), 'experts'), (dict(experts=513), 'experts'),
    (dict(topk=0), 'topk'), (dict(topk=33), 'topk'), (dict(experts=4, topk=5), 'topk'),
    (dict(groups=0), 'groups'), (dict(groups=5), 'groups'), (dict(groups=8, topk_groups=0), 'topk_groups'),
    (dict(groups=8, topk_groups=9), 'topk_groups'), (dict(groups=32, topk_groups=2), 'topk'),
    (dict(dtype=3), 'dtype'), (dict(groups=64, topk_groups=64, top2=1), 'two experts'), (dict(), 'null')])
def test_route_experts_arguments(bad, word):
    assert route(**bad) != 0
    assert word in last_error()


def test_route_experts_without_tokens():
    assert route(tokens=0) == 0


@pytest.mark.parametrize('args,word', [
    ((9, 2, 64, 64, 32, 2), 'dtype'), ((0, -1, 64, 64, 32, 2), 'sizes'), ((0, 2, -1, 64, 32, 2), 'sizes'),
    ((0, 2, 64, 63, 32, 2), 'stride'), ((0, 2, 64, 64, 28, 2), 'stride'), ((0, 2, 64, 64, 32, 1), 'stride'),
    ((0, 2, 64, 64, 33, 2), 'multiple of 4'), ((0, 2, 1 << 33, 1 << 33, 1 << 32, 1 << 28), '2^33'),
    ((0, 1 << 47, 64, 64, 32, 2), '2^48'), ((0, 2, 64, 64, 32, 2), 'null')])
def test_mxfp4_arguments(args, word):
    dtype, rows, cols, stride, ldc, lds = args
    assert lib().ferry_mxfp4_quantize(None, dtype, rows, cols, stride, None, ldc, None, lds, None) != 0
    assert word in last_error()
    assert lib().ferry_mxfp4_dequantize(None, ldc, None, lds, rows, cols, None, dtype, stride, None) != 0
    assert word in last_error()


def test_mxfp4_without_elements():
    assert lib().ferry_mxfp4_quantize(None, 0, 0, 64, 64, None, 32, None, 2, None) == 0
    assert lib().ferry_mxfp4_dequantize(None, 32, None, 2, 5, 0, None, 0, 64, None) == 0


def test_mxfp4_expert_ffn_of_more_pairs_than_rows():
    """list_rows of more than rows * topk pairs, an expert that is listed twice counted once."""
    ints = lambda *v: (ctypes.c_int32 * len(v))(*v)
    place = ctypes.create_string_buffer(64)           # no address is followed before the refusal
    at = (ctypes.addressof(place) + 15) // 16 * 16

    def call(experts, counts, rows=4, topk=2):
        return lib().ferry_mxfp4_expert_ffn(at, 2, 256, 128, at, None, rows, topk, at, at, at, at, ints(*experts),
                                            len(experts), ints(0, 1, 0, 1), 4, -1, 0, ints(*counts), at, at, 0, 3, 0, None)
    for experts, counts in (([0], [9]), ([0, 1, 2], [4, 4, 1]), ([0, 1, 0, 2], [4, 4, 4, 1])):
        assert call(experts, counts) != 0
        assert 'pairs' in last_error()


def test_host_tensors_are_refused():
    x = torch.zeros((4, 64))
    u = torch.zeros((4, 32), dtype=torch.uint8)
    for call in (lambda: ops.route_experts(x, 6), lambda: ops.mxfp4_quantize(x),
                 lambda: ops.mxfp4_dequantize(u, u[:, :2].contiguous()),
                 lambda: ops.mxfp4_expert_rows(torch.zeros((4, 128)))):
        with pytest.raises(RuntimeError, match='CUDA'):
            call()
