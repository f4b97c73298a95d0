"""CPU tier: the linear products refuse bad arguments before any device work."""
import ctypes

import pytest
import torch

from ferry_amd import expert_ops as ops
from ferry_amd._lib import last_error, lib

PLACE = ctypes.create_string_buffer(256)
AT = (ctypes.addressof(PLACE) + 15) // 16 * 16   # no address is followed before a refusal


def product(dtype=0, x_rows=4, k=64, xs=64, rows=None, pairs=4, starts=AT, groups=3, x=AT, w=AT, n=32, ws=64, wg=2048,
            bias_stride=32, act=0, residual=None, rs=0, out=AT, os=32):
    return lib().ferry_expert_linear(x, dtype, x_rows, k, xs, rows, pairs, starts, groups, w, n, ws, wg, None, bias_stride,
                                     act, residual, rs, None, out, os, 0, None, 0, None)


@pytest.mark.parametrize('bad,word', [
    (dict(dtype=1), 'bf16 or fp16'), (dict(dtype=7), 'bf16 or fp16'), (dict(pairs=-1), 'sizes'), (dict(n=0), 'sizes'),
    (dict(k=0), 'sizes'), (dict(pairs=1 << 30), 'sizes'), (dict(n=1 << 30), 'sizes'), (dict(groups=0), 'groups'),
    (dict(groups=513), 'groups'), (dict(starts=None), 'starts'), (dict(x_rows=3), 'row for every'),
    (dict(xs=63), 'strides'), (dict(ws=63), 'strides'), (dict(os=31), 'strides'), (dict(wg=-1), 'strides'),
    (dict(bias_stride=-1), 'strides'), (dict(residual=AT, rs=-1), 'strides'), (dict(act=5), 'activation'),
    (dict(act=-1), 'activation'), (dict(x=None), 'null'), (dict(w=None), 'null'), (dict(out=None), 'null')])
def test_expert_linear_arguments(bad, word):
    assert product(**bad) != 0
    assert word in last_error()


def test_without_rows():
    assert product(pairs=0) == 0
    assert lib().ferry_expert_linear_grad_x(AT, 0, 0, 32, 32, AT, 3, AT, 64, 64, 2048, AT, 0, None, 0, None) == 0
    assert lib().ferry_sum_pairs(AT, 0, 4, 8, AT, 0, 2, AT, None) == 0


def test_gradients_arguments():
    L = lib()
    assert L.ferry_expert_linear_grad_x(AT, 1, 4, 32, 32, AT, 3, AT, 64, 64, 2048, AT, 0, None, 0, None) != 0
    assert 'bf16 or fp16' in last_error()
    assert L.ferry_expert_linear_grad_x(AT, 0, 4, 32, 31, AT, 3, AT, 64, 64, 2048, AT, 0, None, 0, None) != 0
    assert 'strides' in last_error()
    assert L.ferry_expert_linear_grad_w(AT, 0, 4, 32, 32, AT, 3, 64, 64, None, AT, 3, AT, None, 0, None) != 0
    assert 'row for every' in last_error()
    assert L.ferry_expert_linear_grad_w(AT, 0, 4, 32, 32, AT, 4, 64, 64, None, AT, 3, None, None, 0, None) != 0
    assert 'null' in last_error()
    assert L.ferry_linear_grad_z(AT, 0, 4, 32, 32, None, 2, None, 1, AT, AT, None, 0, None) != 0
    assert 'pre and dz' in last_error()
    assert L.ferry_linear_grad_z(AT, 0, 4, 32, 32, AT, 2, AT, 3, AT, AT, None, 0, None) != 0
    assert 'no activation' in last_error()
    assert L.ferry_sum_pairs(AT, 1, 4, 8, AT, 2, 2, AT, None) != 0
    assert L.ferry_sum_pairs(AT, 0, 4, 0, AT, 2, 2, AT, None) != 0
    assert 'sizes' in last_error()


def test_workspaces_are_checked():
    """A contraction that is cut into parts needs its scratch memory: without it the call is refused."""
    L = lib()
    size = L.ferry_linear_workspace_bytes(2, 65536, 64, 64, 1)
    assert size > 0
    assert L.ferry_expert_linear_grad_w(AT, 0, 65536, 64, 64, AT, 65536, 64, 64, None, None, 1, AT, None, 0, None) != 0
    assert 'workspace too small' in last_error()
    assert L.ferry_expert_linear_grad_w(AT, 0, 65536, 64, 64, AT, 65536, 64, 64, None, None, 1, AT, AT, size - 1, None) != 0
    assert 'workspace too small' in last_error()
    assert L.ferry_expert_linear_grad_w(AT, 0, 65536, 64, 64, AT, 65536, 64, 64, None, None, 1, AT, AT + 4, size, None) != 0
    assert 'aligned' in last_error()
    for bad in ((4, 1, 1, 1, 1), (-1, 1, 1, 1, 1), (0, -1, 1, 1, 1), (0, 1, 0, 1, 1), (0, 1, 1, 1, 513)):
        assert L.ferry_linear_workspace_bytes(*bad) == -1


def test_host_tensors_are_refused():
    x, w = torch.zeros((4, 8), dtype=torch.bfloat16), torch.zeros((2, 8), dtype=torch.bfloat16)
    starts = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.linear(x, w), lambda: ops.linear_grad(x, x, w), lambda: ops.expert_linear(x, w[None], starts),
                 lambda: ops.expert_linear_grad(x, x, w[None], starts),
                 lambda: ops.sum_pairs(x, starts.int(), 1)):
        with pytest.raises(RuntimeError, match='CUDA'):
            call()


def test_names_of_activations():
    with pytest.raises(ValueError, match='activation'):
        ops.linear(torch.zeros((4, 8)), torch.zeros((2, 8)), activation='tanh')


@pytest.mark.parametrize('what', ['linear', 'expert_linear', 'linear_grad', 'expert_linear_grad', 'sum_pairs'])
def test_traces_are_refused(what):
    """torch.jit.trace would record the allocation of the result and no launch."""
    x, w = torch.zeros((4, 8), dtype=torch.bfloat16), torch.zeros((2, 8), dtype=torch.bfloat16)
    starts = torch.zeros(2, dtype=torch.int64)
    calls = dict(linear=lambda x: ops.linear(x, w), expert_linear=lambda x: ops.expert_linear(x, w[None], starts),
                 linear_grad=lambda x: ops.linear_grad(x[:, :2], x, w),
                 expert_linear_grad=lambda x: ops.expert_linear_grad(x[:, :2], x, w[None], starts),
                 sum_pairs=lambda x: ops.sum_pairs(x, starts.int(), 2))
    with pytest.raises(RuntimeError, match='cannot be traced'):
        torch.jit.trace(calls[what], x)


@pytest.mark.parametrize('leaf', [True, False])
def test_an_out_that_carries_gradients_is_refused(leaf, monkeypatch):
    """Its new values would keep the old ones' gradient."""
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    x, w = torch.zeros((4, 8), dtype=torch.bfloat16), torch.zeros((2, 8), dtype=torch.bfloat16)
    out = torch.zeros((4, 2), dtype=torch.bfloat16, requires_grad=True)
    out = out if leaf else out * 2
    starts = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.linear(x, w, out=out), lambda: ops.expert_linear(x, w[None], starts, out=out)):
        with pytest.raises(RuntimeError, match='no gradients'):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match='CUDA'):   # as any other out
            call()
