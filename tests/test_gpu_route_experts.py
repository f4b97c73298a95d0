"""route_experts against its formulas in 64 bits: selections exactly, weights to one bf16 rounding."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def route_ref(logits, k, scoring, bias, groups, topk_groups, group_score, renorm, scale):
    """(weights float64 [T, k], ids) of the documented selection, row by row on the CPU."""
    x = logits.detach().cpu().double().numpy()
    b = np.zeros(x.shape[1]) if bias is None else bias.cpu().double().numpy()
    T, E = x.shape
    size = E // groups
    ws, ids = np.zeros((T, k)), np.zeros((T, k), np.int64)
    with np.errstate(all='ignore'):
        for t in range(T):
            row = x[t]
            if scoring == 'sigmoid':
                s = np.array([1 / (1 + np.exp(-v)) for v in row])
            else:
                top = np.fmax.reduce(row)
                s = np.where(row == -np.inf, 0.0, np.exp(row - top))
                total = s.sum()
                s = np.full(E, np.nan) if math.isnan(total) else (s / total if total > 0 else s * 0)
            c = s + b
            c = np.where((row == -np.inf) | np.isnan(c), -np.inf, c)
            open_ = np.ones(E, bool)
            if groups > 1:
                g = np.sort(c.reshape(groups, size), 1)
                score = g[:, -1] if group_score == 'max' else g[:, -1] + g[:, -2]
                score = np.where(np.isnan(score), -np.inf, score)
                best = sorted(range(groups), key=lambda i: (-score[i], i))[:topk_groups]
                open_ = np.isin(np.arange(E) // size, best)
            order = sorted((e for e in range(E) if open_[e]), key=lambda e: (-c[e], e))[:k]
            w = s[order]
            if renorm:
                w = w / w.sum() if not w.sum() <= 0 else w * 0
            ws[t], ids[t] = w * np.float64(np.float32(scale)), order
    return ws, ids


def check(logits, k, scoring='softmax', bias=None, groups=1, topk_groups=None, group_score='max',
          renorm=True, scale=1.0):
    from ferry_amd import expert_ops as ops
    w, ids = ops.route_experts(logits, k, scoring=scoring, bias=bias, groups=groups,
                               topk_groups=topk_groups, group_score=group_score, renorm=renorm, scale=scale)
    assert w.dtype == torch.bfloat16 and ids.dtype == torch.int64 and w.shape == ids.shape
    ws, want = route_ref(logits, k, scoring, bias, groups, topk_groups or groups, group_score, renorm, scale)
    np.testing.assert_array_equal(ids.cpu().numpy(), want)
    got = w.double().cpu().numpy()
    # one rounding to bf16 (half a step: 2^-9 of the next power of two, 2^-8 relative at most) of a value
    # that is 64-bit but for a rounding to fp32 before it (2^-24); below the least normal 2^-126 the steps are
    # 2^-133 and 2^-149, whatever the value
    np.testing.assert_array_equal(np.isnan(got), np.isnan(ws))
    fine = ~np.isnan(ws)
    assert (np.abs(got - ws)[fine] <= (2 ** -8 + 2 ** -23) * np.abs(ws[fine]) + 2.0 ** -134 + 2.0 ** -150).all()
    return w, ids


def randn(shape, seed, dtype=torch.float32, scale=1.5):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device='cuda') * scale).to(dtype)


GATES = [
    # experts, topk, groups, topk_groups
    (1, 1, 1, 1), (2, 2, 1, 1), (6, 3, 3, 2), (64, 6, 1, 1), (65, 8, 5, 2), (128, 8, 1, 1), (160, 6, 8, 3),
    (256, 8, 8, 4), (252, 7, 4, 4), (256, 32, 16, 2), (500, 16, 10, 3), (512, 8, 256, 40), (512, 32, 512, 32),
    (511, 5, 1, 1), (129, 4, 3, 1),
]


@pytest.mark.parametrize('E,k,G,TG', GATES)
@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_gates(device, E, k, G, TG, scoring, dtype):
    for T, seed in ((1, 1), (37, 2)):
        logits = randn((T, E), seed, dtype)
        bias = randn((E,), seed + 10, scale=0.2)
        score = 'top2' if E // G >= 2 else 'max'
        check(logits, k, scoring, bias, G, TG, score, True, 2.5)
        check(logits, k, scoring, None, G, TG, 'max', False, 16.0)


@pytest.mark.parametrize('E,k,G,TG', [(64, 6, 1, 1), (256, 8, 8, 4), (160, 6, 8, 3)])
@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
def test_ties_go_to_the_lowest_index(device, E, k, G, TG, scoring):
    # whole numbers: most experts and groups tie with others
    logits = randn((200, E), 3).round()
    check(logits, k, scoring, None, G, TG, 'max')
    check(logits, k, scoring, None, G, TG, 'top2')
    check(torch.zeros((4, E), device='cuda'), k, scoring, None, G, TG, 'top2')


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
def test_scores_that_differ_below_fp32(device, scoring):
    # neighbouring fp32 logits around 10: the sigmoid's values round to the same fp32 number
    x = torch.full((8, 64), 10.0, device='cuda')
    order = torch.from_numpy(np.stack([np.random.default_rng(i).permutation(64) for i in range(8)])).cuda()
    x += order.float() * 2.0 ** -20
    w, ids = check(x, 8, scoring)
    assert (ids == order.argsort(1, descending=True)[:, :8]).all()


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('groups', [1, 4])
def test_masked_and_special_logits(device, scoring, groups):
    E, k = 64, 8
    tg = max(1, groups // 2)
    inf, nan = math.inf, math.nan
    x = randn((12, E), 5)
    x[0] = -inf                               # nothing left
    x[1, 3:] = -inf                           # fewer than k left
    x[2, ::2] = -inf
    x[3, 5] = nan
    x[4] = nan
    x[5, 7] = inf
    x[6] = torch.finfo(torch.float32).min     # masks of the type's lowest value
    x[7, 10:] = torch.finfo(torch.float32).min
    x[8, :32] = -inf                          # whole groups masked
    x[9] = 0.0
    x[10] = -800.0                            # e^-800 is 0 in fp32, not in 64 bits
    x[10, 40] = -799.0
    x[11] = 90.0
    bias = randn((E,), 6, scale=0.3)
    bias[2], bias[9] = -inf, inf
    for b in (None, bias):
        w, ids = check(x, k, scoring, b, groups, tg, 'top2' if groups > 1 else 'max')
        assert all(len(set(r)) == k for r in ids.tolist()) and (ids >= 0).all() and (ids < E).all()
    w, _ = check(x[:1], k, scoring, None, groups, tg)
    assert (w == 0).all()


# more tokens than the library gives a wavefront each: four to a wavefront, fp32 scores where they decide
BATCH_GATES = [(1, 1, 1, 1), (6, 3, 3, 2), (64, 6, 1, 1), (65, 8, 5, 2), (128, 8, 1, 1), (160, 6, 8, 3),
               (256, 8, 8, 4), (252, 7, 4, 4), (256, 16, 128, 9), (129, 4, 3, 1), (256, 17, 1, 1)]


@pytest.mark.parametrize('E,k,G,TG', BATCH_GATES)
@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gates_on_batches(device, E, k, G, TG, scoring, dtype):
    logits = randn((2051, E), 5, dtype)
    logits[100:200] = logits[100:200].round()   # ties
    logits[200:210] = 0.5                       # nothing but ties
    bias = randn((E,), 6, scale=0.2)
    score = 'top2' if E // G >= 2 else 'max'
    check(logits, k, scoring, bias, G, TG, score, True, 2.5)
    check(logits, k, scoring, None, G, TG, 'max', False, 16.0)


@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('E,k,G,TG', [(64, 6, 1, 1), (256, 8, 8, 4)])
def test_special_batches(device, E, k, G, TG, scoring):
    logits = randn((2400, E), 7)
    inf, nan = float('inf'), float('nan')
    logits[0:50, 3:] = -inf            # three experts left, then none
    logits[50:60] = -inf
    logits[60:100, ::5] = -inf
    logits[100:120, 7] = nan
    logits[120:140, 9] = inf
    logits[140:160, 2] = nan
    logits[140:160, 40:] = -inf
    logits[160:400] *= 40              # scores from next to 1 down to 2^-250
    logits[400:600] -= 80
    logits[600:800] *= 2.0 ** -18      # scores that fp32 cannot tell apart, in part
    logits[800:1000] = 10 + logits[800:1000] * 2.0 ** -16
    check(logits, k, scoring, None, G, TG, 'max')
    check(logits, k, scoring, None, G, TG, 'top2', False)
    bias = randn((E,), 8, scale=0.01)
    check(logits, k, scoring, bias, G, TG, 'top2')
    # choice scores far below the scores' own size, or far above it
    check(logits, k, scoring, -torch.ones(E, device='cuda'), G, TG, 'top2')
    bias[::2] += 1000
    bias[1::4] -= 1000
    check(logits, k, scoring, bias, G, TG, 'top2')
    bias[5], bias[6], bias[7] = inf, -inf, nan
    check(logits, k, scoring, bias, G, TG, 'top2')
    check(logits, k, scoring, bias, G, TG, 'max')


def test_empty_and_large_batches(device):
    from ferry_amd import expert_ops as ops
    w, ids = ops.route_experts(torch.empty((0, 64), device='cuda'), 6)
    assert w.shape == (0, 6) and ids.shape == (0, 6)
    logits = randn((20011, 256), 8)
    bias = randn((256,), 9, scale=0.2)
    w, ids = ops.route_experts(logits, 8, scoring='sigmoid', bias=bias, groups=8, topk_groups=4,
                               group_score='top2')
    pick = torch.randperm(20011, generator=torch.Generator().manual_seed(0))[:300]
    pick[:2] = torch.tensor([0, 20010])
    w2, ids2 = check(logits[pick.cuda()], 8, 'sigmoid', bias, 8, 4, 'top2')
    assert torch.equal(ids[pick.cuda()], ids2) and torch.equal(w[pick.cuda()], w2)


def test_more_tokens_than_a_launch_takes(device):
    from ferry_amd import expert_ops as ops
    T = 2 ** 24 + 2500
    logits = randn((T, 4), 12, torch.bfloat16)
    w, ids = ops.route_experts(logits, 2, scoring='sigmoid')
    pick = torch.cat([torch.arange(50), torch.arange(2 ** 24 - 50, 2 ** 24 + 50), torch.arange(T - 50, T)]).cuda()
    w2, ids2 = check(logits[pick], 2, 'sigmoid')
    assert torch.equal(ids[pick], ids2) and torch.equal(w[pick], w2)
    assert bool((ids[:, 0] != ids[:, 1]).all()) and int(ids.min()) == 0 and int(ids.max()) == 3


def test_graph_replays_and_streams(device):
    from ferry_amd import expert_ops as ops
    logits = randn((50, 256), 11)

    def call():
        return ops.route_experts(logits, 8, scoring='sigmoid', groups=8, topk_groups=4, group_score='top2')
    want = call()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = call()
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        w, ids = call()
    for seed in (12, 13, 14):
        logits.copy_(randn((50, 256), seed))
        want = call()
        w.zero_(), ids.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, want[0]) and torch.equal(ids, want[1])


def test_refusals(device):
    from ferry_amd import expert_ops as ops
    x = randn((4, 64), 1)
    for bad in (dict(topk=0), dict(topk=33), dict(topk=65), dict(topk=6, groups=5), dict(topk=6, groups=0),
                dict(topk=6, groups=8, topk_groups=9), dict(topk=6, groups=8, topk_groups=0),
                dict(topk=9, groups=8, topk_groups=1), dict(topk=2, groups=64, group_score='top2'),
                dict(topk=6, bias=torch.zeros(63, device='cuda')),
                dict(topk=6, bias=torch.zeros(64, device='cuda', dtype=torch.bfloat16)),
                dict(topk=6, bias=torch.zeros(64))):
        with pytest.raises(RuntimeError):
            ops.route_experts(x, **bad)
    for bad in (dict(scoring='tanh'), dict(group_score='mean')):
        with pytest.raises(ValueError):
            ops.route_experts(x, 6, **bad)
    for bad in (x.double(), x[0], x.t(), torch.zeros((2, 513), device='cuda')):
        with pytest.raises(RuntimeError):
            ops.route_experts(bad, 2)


# further batches: logits in fp16, more experts and more of them chosen than 16 lanes hold
MORE_BATCH_GATES = [(512, 8, 8, 4), (511, 5, 1, 1), (500, 16, 10, 3), (512, 32, 256, 40), (257, 6, 1, 1), (256, 32, 16, 2),
                    (64, 17, 1, 1)]


@pytest.mark.parametrize('E,k,G,TG', BATCH_GATES + MORE_BATCH_GATES)
@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
def test_gates_on_fp16_batches(device, E, k, G, TG, scoring):
    test_gates_on_batches(device, E, k, G, TG, scoring, torch.float16)


@pytest.mark.parametrize('E,k,G,TG', MORE_BATCH_GATES)
@pytest.mark.parametrize('scoring', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_large_gates_on_batches(device, E, k, G, TG, scoring, dtype):
    test_gates_on_batches(device, E, k, G, TG, scoring, dtype)
