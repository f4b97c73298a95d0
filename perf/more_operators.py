"""Matrix products grouped by expert and dense products with an epilogue: what is timed, and their plain forms.

Kinds (`case["kind"]`):
  linear        linear: activation(x W^T + bias) + residual
  linear_train  the same, keeping what the backward pass needs, then linear_grad: the gradients of x, W and bias
  expert        expert_linear: row p of the grouped order times its expert's matrix, plus the expert's bias
  expert_train  expert_linear, then expert_linear_grad: the gradients of x, W and bias

Shapes are those of the two models this package evaluates (Qwen3-30B-A3B: hidden 2048, 128 experts of
intermediate 768, top 8, dense layers of 6144, 32 heads of 128; DeepSeek-V2-Lite: hidden 2048, 64 experts of
intermediate 1408, top 6, two shared ones) and generic ones.  Expert popularity is Zipf over a seeded
permutation: in a prefill the largest expert gets thousands of rows, some get none.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}


def _linear(name, kind, rows, k, n, bias=False, act='', residual=False, dtype='bf16'):
    return dict(name=name, kind=kind, rows=rows, k=k, n=n, bias=bias, act=act, residual=residual, dtype=dtype)


def _expert(name, kind, tokens, experts, topk, zipf, k, n, gather, bias=False, dtype='bf16'):
    return dict(name=name, kind=kind, tokens=tokens, experts=experts, topk=topk, zipf=zipf, k=k, n=n,
                gather=gather, bias=bias, dtype=dtype)


def listed():
    return [
        # one decoded token through a dense layer's up projection: the weight is read, little else
        _linear('linear_t1', 'linear', 1, 2048, 6144, act='silu'),
        # the attention's output projection of a decode step of 16 requests, added to the hidden rows
        _linear('linear_t16', 'linear', 16, 4096, 2048, residual=True),
        # a ragged prompt through a layer whose every size is odd: rows that start at any element
        _linear('linear_odd', 'linear', 777, 1001, 2047, bias=True, act='gelu', residual=True, dtype='fp16'),
        # a prefill batch through a dense layer's up projection
        _linear('linear_t8192', 'linear', 8192, 2048, 6144, bias=True, act='gelu_tanh'),
        # a short training batch of the two shared experts' gate projection
        _linear('linear_train_t300', 'linear_train', 300, 2048, 2816, bias=True, act='silu', dtype='fp16'),
        # a training batch of a dense layer
        _linear('linear_train_t8192', 'linear_train', 8192, 2048, 6144, bias=True, act='silu', residual=True),
        # one request's decode step, gate and up: 8 experts of one row
        _expert('expert_t1', 'expert', 1, 128, 8, 1.1, 2048, 1536, True),
        # a decode step of 16 requests: some 40 experts of a few rows
        _expert('expert_t16', 'expert', 16, 128, 8, 1.1, 2048, 1536, True),
        # one prompt of ordinary, ragged length, experts with biases
        _expert('expert_t777', 'expert', 777, 64, 6, 0.9, 2048, 2816, True, bias=True, dtype='fp16'),
        # the prefill batch, gate and up of every expert
        _expert('expert_t8192', 'expert', 8192, 128, 8, 1.1, 2048, 1536, True),
        # a short training batch through the experts' down projection: rows already grouped
        _expert('expert_train_t500', 'expert_train', 500, 64, 6, 0.9, 1408, 2048, False, bias=True),
        # a training batch through gate and up, rows gathered from the tokens
        _expert('expert_train_t8192', 'expert_train', 8192, 128, 8, 1.1, 2048, 1536, True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A row length: mostly a multiple of 64 or 8, now and then any number."""
    n = _log_uniform(rng, lo, hi)
    step = rng.choice([64, 64, 64, 8, 8, 1])
    return max(step, n // step * step)


def draw(rng):
    kind = rng.choice(['linear', 'linear', 'linear_train', 'expert', 'expert', 'expert_train'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16'])
    passes = 3 if kind.endswith('_train') else 1
    while True:
        k, n = _size(rng, 8, 8192), _size(rng, 8, 8192)
        if kind.startswith('linear'):
            rows = _log_uniform(rng, 1, 16384)
            if rows * k * n <= 8192 * 2048 * 6144 and 3 * rows * k * n * passes >= 1e6:
                return dict(kind=kind, rows=rows, k=k, n=n, bias=rng.random() < 0.5,
                            act=rng.choice(['', 'relu', 'silu', 'gelu', 'gelu_tanh']),
                            residual=rng.random() < 0.5, dtype=dtype)
            continue
        experts = _log_uniform(rng, 2, 256)
        topk = rng.randint(1, min(8, experts))
        tokens = _log_uniform(rng, 1, 8192)
        if (tokens * topk * k * n <= 8192 * 8 * 2048 * 1536 and experts * k * n <= 128 * 2048 * 1536
                and tokens * topk * (k + n) <= 8192 * 8 * 3584):
            return dict(kind=kind, tokens=tokens, experts=experts, topk=topk, zipf=round(rng.uniform(0.0, 1.2), 2),
                        k=k, n=n, gather=rng.random() < 0.5, bias=rng.random() < 0.4, dtype=dtype)


# -- inputs -------------------------------------------------------------------------------------

def _routing(case, seed):
    """Distinct experts of every token, ascending, int64 [tokens, topk]: the top-k of N(0, 1) plus the
    experts' log popularity."""
    rng = np.random.default_rng(seed)
    T, E, k = case['tokens'], case['experts'], case['topk']
    pop = -case['zipf'] * np.log(1.0 + rng.permutation(E))
    z = rng.standard_normal((T, E), dtype=np.float32) + pop.astype(np.float32)
    return np.sort(np.argpartition(-z, k - 1, axis=1)[:, :k], axis=1).astype(np.int64)


def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    dtype = DTYPES[case['dtype']]

    def normal(*shape, scale=1.0):
        out = torch.empty(shape, dtype=dtype, device='cuda')
        flat = out.view(-1)
        for lo in range(0, flat.numel(), 1 << 28):   # a part at a time, to bound the memory
            part = flat[lo:lo + (1 << 28)]
            part.copy_(torch.randn(part.shape, generator=g, device='cuda') * scale)
        return out

    K, N, train = case['k'], case['n'], case['kind'].endswith('_train')
    scale = 1.0 / math.sqrt(K)
    if case['kind'].startswith('linear'):
        M = case['rows']
        return dict(case=case, x=normal(M, K), w=normal(N, K, scale=scale),
                    bias=normal(N, scale=0.1) if case['bias'] else None,
                    residual=normal(M, N) if case['residual'] else None,
                    dy=normal(M, N) if train else None)
    T, E, k = case['tokens'], case['experts'], case['topk']
    ids = _routing(case, seed).reshape(-1)
    order = np.argsort(ids, kind='stable')
    inverse = np.empty(T * k, np.int32)
    inverse[order] = np.arange(T * k, dtype=np.int32)
    counts = np.bincount(ids, minlength=E)
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)
    gather = case['gather']
    return dict(case=case, x=normal(T if gather else T * k, K), w=normal(E, N, K, scale=scale),
                bias=normal(E, N, scale=0.1) if case['bias'] else None,
                dy=normal(T * k, N) if train else None, counts=counts,
                starts=torch.from_numpy(starts).cuda(),
                rows=torch.from_numpy(order // k).cuda() if gather else None,
                pair_pos=torch.from_numpy(inverse.reshape(T, k)).cuda() if gather else None)


# -- one pass -----------------------------------------------------------------------------------

def _plain_act(z, act):
    """(activation, its derivative) of z."""
    if act == '':
        return z, torch.ones_like(z)
    if act == 'relu':
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
    if act == 'silu':
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if act == 'gelu':
        p = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    c = math.sqrt(2 / math.pi)
    t = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    c, dtype = s['case'], s['x'].dtype
    x, w = s['x'].float(), s['w'].float()
    z = x @ w.t()
    if c['bias']:
        z = z + s['bias'].float()
    y, slope = _plain_act(z, c['act'])
    if c['residual']:
        y = y + s['residual'].float()
    y = y.to(dtype)
    if c['kind'] == 'linear':
        return y
    dz = s['dy'].float() * slope
    return dict(y=y, dx=(dz @ w).to(dtype), dw=(dz.t() @ x).to(dtype),
                db=dz.sum(0).to(dtype) if c['bias'] else None)


def _plain_expert(s):
    c, dtype, rows = s['case'], s['x'].dtype, s['rows']
    starts = np.concatenate([[0], np.cumsum(s['counts'])])
    P, N, K = int(starts[-1]), c['n'], c['k']
    train = c['kind'] == 'expert_train'
    y = torch.empty((P, N), dtype=dtype, device='cuda')
    if train:
        dxp = torch.empty((P, K), dtype=torch.float32, device='cuda')
        dw, db = torch.zeros_like(s['w']), torch.zeros_like(s['bias']) if c['bias'] else None
    # one product per expert: their row counts differ
    for e in np.flatnonzero(s['counts']):
        lo, hi = int(starts[e]), int(starts[e + 1])
        x = (s['x'][lo:hi] if rows is None else s['x'][rows[lo:hi]]).float()
        w = s['w'][e].float()
        z = x @ w.t()
        if c['bias']:
            z = z + s['bias'][e].float()
        y[lo:hi] = z.to(dtype)
        if train:
            dy = s['dy'][lo:hi].float()
            dxp[lo:hi] = dy @ w
            dw[e] = (dy.t() @ x).to(dtype)
            if c['bias']:
                db[e] = dy.sum(0).to(dtype)
    if not train:
        return y
    dx = dxp if rows is None else dxp[s['pair_pos'].long()].sum(1)
    return dict(y=y, dx=dx.to(dtype), dw=dw, db=db)


def run(s):
    c = s['case']
    if not own:
        return _plain_linear(s) if c['kind'].startswith('linear') else _plain_expert(s)
    from ferry_amd import expert_ops as ops
    if c['kind'] == 'linear':
        return ops.linear(s['x'], s['w'], bias=s['bias'], activation=c['act'] or None, residual=s['residual'])
    if c['kind'] == 'linear_train':
        y, pre = ops.linear(s['x'], s['w'], bias=s['bias'], activation=c['act'] or None,
                            residual=s['residual'], return_pre=True)
        dx, dw, db = ops.linear_grad(s['dy'], s['x'], s['w'], pre=pre, activation=c['act'] or None,
                                     need_bias=c['bias'])
        return dict(y=y, dx=dx, dw=dw, db=db)
    y = ops.expert_linear(s['x'], s['w'], s['starts'], bias=s['bias'], rows=s['rows'])
    if c['kind'] == 'expert':
        return y
    dx, dw, db = ops.expert_linear_grad(s['dy'], s['x'], s['w'], s['starts'], rows=s['rows'],
                                        pair_pos=s['pair_pos'], need_bias=c['bias'])
    return dict(y=y, dx=dx, dw=dw, db=db)


# -- the definitions in 64 bits -------------------------------------------------------------------

def _exact_act(z, act):
    if act == 'relu':
        return z.clamp(min=0)
    if act == 'silu':
        return z * torch.sigmoid(z)
    if act == 'gelu':
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if act == 'gelu_tanh':
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def exact(case, seed):
    """float64 outputs; the gradients are those of sum(y * dy), by automatic differentiation."""
    s = prepare(case, seed)
    train = case['kind'].endswith('_train')

    def leaf(t):
        return None if t is None else t.double().requires_grad_(train)

    if case['kind'].startswith('linear'):
        x, w, b = leaf(s['x']), leaf(s['w']), leaf(s['bias'])
        z = x.mm(w.t())
        y = _exact_act(z if b is None else z + b, case['act'])
        if s['residual'] is not None:
            y = y + s['residual'].double()
        if not train:
            return y
        got = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], s['dy'].double())
        return dict(y=y.detach(), dx=got[0], dw=got[1], db=got[2] if b is not None else None)
    E, N, K = s['w'].shape
    ends = s['starts'].tolist()
    P = ends[-1]
    token = torch.arange(P, device='cuda') if s['rows'] is None else s['rows']
    y = torch.zeros((P, N), dtype=torch.float64, device='cuda')
    dx = torch.zeros(s['x'].shape, dtype=torch.float64, device='cuda')
    dw = torch.zeros((E, N, K), dtype=torch.float64, device='cuda') if train else None
    db = torch.zeros((E, N), dtype=torch.float64, device='cuda') if train and case['bias'] else None
    for e in range(E):
        if ends[e] == ends[e + 1]:
            continue
        at = slice(ends[e], ends[e + 1])
        x, w = leaf(s['x'][token[at]]), leaf(s['w'][e])
        b = leaf(s['bias'][e]) if case['bias'] else None
        out = x.mm(w.t()) if b is None else torch.addmm(b, x, w.t())
        y[at] = out.detach()
        if train:
            got = torch.autograd.grad(out, [t for t in (x, w, b) if t is not None], s['dy'][at].double())
            dx.index_add_(0, token[at], got[0])
            dw[e] = got[1]
            if b is not None:
                db[e] = got[2]
    return dict(y=y, dx=dx, dw=dw, db=db) if train else y


# -- work -----------------------------------------------------------------------------------------

def work(case):
    K, N, train = case['k'], case['n'], case['kind'].endswith('_train')
    if case['kind'].startswith('linear'):
        M = case['rows']
        values = M * K + N * K + M * N * (2 if case['residual'] else 1) + (N if case['bias'] else 0)
        if train:   # dy in; dx, dw and db out
            values += M * N + M * K + N * K + (N if case['bias'] else 0)
        return dict(bytes=2 * values, flops=2 * M * N * K * (3 if train else 1))
    T, E, k = case['tokens'], case['experts'], case['topk']
    P, active = T * k, len(np.unique(_routing(case, 0)))
    rows = T if case['gather'] else P
    values = rows * K + active * N * K + P * N + (active * N if case['bias'] else 0)
    index = 8 * (E + 1) + (8 * P if case['gather'] else 0)
    if train:
        values += P * N + rows * K + E * N * K + (E * N if case['bias'] else 0)
        index += 4 * P if case['gather'] else 0
    return dict(bytes=2 * values + index, flops=2 * P * N * K * (3 if train else 1))
