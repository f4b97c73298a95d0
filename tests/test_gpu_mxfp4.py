"""MXFP4 rows: codes and scales exactly as the definition in 64 bits, for every input type and layout."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

VALUES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def quantize_ref(x):
    """(codes, scales) of a float64 numpy matrix, by distance to the eight magnitudes."""
    n, cols = x.shape
    blocks = -(-cols // 32)
    v = np.zeros((n, blocks * 32))
    v[:, :cols] = x
    v = v.reshape(n, blocks, 32)
    amax = np.abs(v).max(-1)
    bad = ~np.isfinite(amax)
    with np.errstate(all='ignore'):
        e = np.where((amax > 0) & ~bad, np.frexp(np.where(bad, 1.0, amax))[1] - 3, -127)
    e = np.clip(e, -127, 127)
    a = np.abs(np.where(bad[..., None], 0.0, v)) / np.exp2(e)[..., None]
    a = np.minimum(a, 6.0)
    dist = np.abs(a[..., None] - VALUES)
    near = dist.min(-1, keepdims=True)
    # of two equally near ones the even code
    cand = np.where(dist == near, np.arange(8) + 10 * (np.arange(8) % 2), 100)
    code = cand.min(-1) % 10
    code = code | (np.signbit(np.where(bad[..., None], 0.0, v)).astype(np.int64) << 3)
    codes = (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8).reshape(n, blocks * 16)
    return codes, np.where(bad, 255, e + 127).astype(np.uint8)


def values_ref(codes, scales):
    n, blocks = scales.shape
    c = codes.reshape(n, blocks, 16)
    nib = np.stack([c & 15, c >> 4], -1).reshape(n, blocks, 32)
    v = np.where(nib >= 8, -1.0, 1.0) * VALUES[nib & 7]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * s[..., None]).reshape(n, -1)


def rows(n, cols, dtype, seed, spread=20):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, cols), generator=g) * torch.exp2(
        torch.randint(-spread, spread, (n, 1), generator=g).float())
    return x.to(dtype)


def check(x):
    from ferry_amd import expert_ops as ops
    codes, scales = ops.mxfp4_quantize(x.cuda())
    want_c, want_s = quantize_ref(x.double().numpy())
    np.testing.assert_array_equal(scales.cpu().numpy(), want_s)
    np.testing.assert_array_equal(codes.cpu().numpy(), want_c)
    v = values_ref(want_c, want_s)[:, :x.shape[1]]
    for dtype in (torch.bfloat16, torch.float32, torch.float16):
        got = ops.mxfp4_dequantize(codes, scales, columns=x.shape[1], dtype=dtype)
        assert got.shape == x.shape and got.dtype == dtype
        want = torch.from_numpy(v).to(torch.float32).to(dtype)   # exact in fp32 up to 6 * 2^125
        assert torch.equal(torch.nan_to_num(got.cpu(), nan=77.0), torch.nan_to_num(want, nan=77.0))
    return codes, scales


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('n,cols', [(1, 1), (3, 7), (1, 32), (5, 33), (17, 2048), (70, 31), (2, 4099), (259, 96),
                                    (1000, 1), (3, 100001)])
def test_rows(device, n, cols, dtype):
    check(rows(n, cols, dtype, n + cols, spread=8 if dtype == torch.float16 else 40))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
def test_borders_between_values(device, dtype):
    # a block's largest element 4 .. 7.99 fixes the scale; the others lie on and next to the midpoints
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0])
    out = []
    for top in (4.0, 6.0, 7.75):
        for e in (-10, 0, 7):
            m = mids.to(dtype)
            up, down = torch.nextafter(m, m + 100), torch.nextafter(m, m - 100)
            block = torch.cat([m, up, down, -m[:7], torch.tensor([top]).to(dtype)])
            block = torch.where(block.abs() > top, torch.zeros_like(block), block)
            out.append((block.float() * 2.0 ** e).to(dtype))
    check(torch.stack(out))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
def test_zeros_extremes_and_non_finite_blocks(device, dtype):
    f = torch.finfo(dtype)
    x = torch.zeros((9, 64), dtype=dtype)
    x[1, 0] = -0.0
    x[2, 5] = f.max
    x[3, 40] = f.smallest_normal
    x[4, 40] = f.smallest_normal / 4      # subnormal
    x[5] = rows(1, 64, dtype, 3, spread=1)[0]
    x[5, 33] = math.inf
    x[6] = rows(1, 64, dtype, 4, spread=1)[0]
    x[6, 0] = math.nan
    x[7] = -f.max
    x[8, ::2] = f.max
    x[8, 1::2] = f.smallest_normal
    check(x)


def test_layouts(device):
    from ferry_amd import expert_ops as ops
    base = rows(12, 160, torch.bfloat16, 5).cuda()
    want = ops.mxfp4_quantize(base[:, 3:99].contiguous())
    got = ops.mxfp4_quantize(base[:, 3:99])        # row stride, rows at odd addresses
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = ops.mxfp4_quantize(base[::3])
    want = ops.mxfp4_quantize(base[::3].contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    c3, s3 = ops.mxfp4_quantize(base.view(3, 4, 160))
    c2, s2 = ops.mxfp4_quantize(base)
    assert c3.shape == (3, 4, 80) and s3.shape == (3, 4, 5)
    assert torch.equal(c3.view(12, 80), c2) and torch.equal(s3.view(12, 5), s2)
    c1, s1 = ops.mxfp4_quantize(base[2])
    assert torch.equal(c1, c2[2]) and torch.equal(s1, s2[2])
    # the two parts of expert rows, in place in a larger buffer whose other rows stay
    x = base[:, :128].contiguous()
    buf = torch.full((14, 68), 9, dtype=torch.uint8, device='cuda')
    packed = ops.mxfp4_expert_rows(x, out=buf[1:13])
    assert packed.data_ptr() == buf[1].data_ptr() and (buf[0] == 9).all() and (buf[13] == 9).all()
    c, s = ops.mxfp4_quantize(x)
    assert torch.equal(packed[:, :64], c) and torch.equal(packed[:, 64:], s)
    assert torch.equal(ops.mxfp4_dequantize(packed[:, :64], packed[:, 64:]), ops.mxfp4_dequantize(c, s))


def test_empty_rows(device):
    from ferry_amd import expert_ops as ops
    for shape in ((0, 64), (4, 0), (0,)):
        c, s = ops.mxfp4_quantize(torch.empty(shape, device='cuda'))
        blocks = -(-shape[-1] // 32)
        assert c.shape == (*shape[:-1], 16 * blocks) and s.shape == (*shape[:-1], blocks)
        assert ops.mxfp4_dequantize(c, s, columns=shape[-1]).shape == shape


def test_long_row_and_many_rows(device):
    """Sizes that take more than one pass of the grid, against parts of the same call."""
    from ferry_amd import expert_ops as ops
    g = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randn((3, 1 << 24), generator=g, device='cuda', dtype=torch.bfloat16)
    c, s = ops.mxfp4_quantize(x)
    for r, lo in ((0, 0), (1, (1 << 23) - 64), (2, (1 << 24) - 4096)):
        part = x[r, lo:lo + 4096]
        want = quantize_ref(part.double().cpu().numpy()[None])
        n = part.numel()
        np.testing.assert_array_equal(c[r, lo // 2:lo // 2 + n // 2].cpu().numpy(), want[0][0])
        np.testing.assert_array_equal(s[r, lo // 32:lo // 32 + n // 32].cpu().numpy(), want[1][0])
    y = ops.mxfp4_dequantize(c, s)
    c2, s2 = ops.mxfp4_quantize(y)          # a fixed point: the values' own form is themselves
    assert torch.equal(ops.mxfp4_dequantize(c2, s2), y)
    tall = torch.randn((3000001, 5), generator=g, device='cuda')
    c, s = ops.mxfp4_quantize(tall)
    for r in (0, 1234567, 3000000):
        want = quantize_ref(tall[r:r + 1].double().cpu().numpy())
        np.testing.assert_array_equal(c[r:r + 1].cpu().numpy(), want[0])
        np.testing.assert_array_equal(s[r:r + 1].cpu().numpy(), want[1])


@pytest.mark.parametrize('rows,cols', [(70001, 65536), (140001, 65536), (70001, 65530)])
def test_more_than_2_32_elements(device, rows, cols):
    """One row in every 10,000 and the last ones are not zero; 2^33 elements are past a flattened row."""
    from ferry_amd import expert_ops as ops
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device='cuda')
    at = torch.cat([torch.arange(0, rows - 3, 10000), torch.arange(rows - 3, rows)]).cuda()
    some = torch.randn((len(at), cols), generator=torch.Generator(device='cuda').manual_seed(1), device='cuda').bfloat16()
    x[at] = some
    codes, scales = ops.mxfp4_quantize(x)
    want = ops.mxfp4_quantize(some)
    assert torch.equal(codes[at], want[0]) and torch.equal(scales[at], want[1])
    assert int((scales != 0).any(1).sum()) == len(at)
    back = ops.mxfp4_dequantize(codes, scales, columns=cols)
    assert torch.equal(back[at], ops.mxfp4_dequantize(*want, columns=cols))
    assert int((back != 0).any(1).sum()) == len(at)


def test_refusals(device):
    from ferry_amd import expert_ops as ops
    x = torch.zeros((4, 64), device='cuda')
    for bad in (x.double(), x.t(), x.int(), x.cpu(), x[:, ::2], x[:1].expand(4, 64), torch.tensor(1.0).cuda()):
        with pytest.raises(RuntimeError):
            ops.mxfp4_quantize(bad)
    c, s = ops.mxfp4_quantize(x)
    for bad in ((c, s, 65), (c, s, 32), (c[:, :16], s, 64), (c.int(), s, 64), (c, s.cpu(), 64), (c[:3], s, 64)):
        with pytest.raises(RuntimeError):
            ops.mxfp4_dequantize(*bad)
    with pytest.raises(RuntimeError):
        ops.mxfp4_dequantize(c, s, dtype=torch.float64)
    for bad in (x, x[0], torch.zeros((4, 128), device='cuda').double()):
        with pytest.raises(RuntimeError):
            ops.mxfp4_expert_rows(bad)
    with pytest.raises(RuntimeError):
        ops.mxfp4_expert_rows(torch.zeros((4, 128), device='cuda'),
                              out=torch.zeros((4, 67), dtype=torch.uint8, device='cuda'))
