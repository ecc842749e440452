"""Routing to experts and low-rank adapters: what stands beside a served model's
projections and experts, as a serving program calls it.

* ``route`` - the experts of each row of a gate's logits, and their weights:
  softmax or sigmoid scores, a selection bias, groups, top-k, renormalised and
  scaled (``native.route_experts``).
* ``adapter`` - a shared projection's rows plus what each row's own low-rank
  adapter adds, the adapters of many requests in one call
  (``native.adapter_out``).

The plain forms are the definitions in elementary torch operations.
"""
import functools
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def _route(name, rows, experts, top, score='softmax', bias=False, groups=1, kept=1, group_top=1, renormalize=True,
           scale=1.0, dtype='fp32', pad=0):
    case = dict(kind='route', rows=rows, experts=experts, top=top, score=score, bias=bias, groups=groups, kept=kept,
                group_top=group_top, renormalize=renormalize, scale=scale, dtype=dtype, pad=pad)
    return dict(name=name, **case) if name else case


def _adapter(name, rows, requests, slots, rank, n, k, parts=1, dtype='bf16', out='bf16', pad=0):
    case = dict(kind='adapter', rows=rows, requests=requests, slots=slots, rank=rank, n=n, k=k, parts=parts, dtype=dtype,
                out=out, pad=pad)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # one user's next token, the contract of the routed banks: softmax, the 8 best of 256, on the gate's
        # logits, which share their buffer with the shared expert's
        _route('route_softmax_1', 1, 256, 8, pad=1),
        # a decode batch of a model that balances by a bias and picks groups first
        _route('route_groups_32', 32, 256, 8, 'sigmoid', True, 8, 4, 2, scale=2.5),
        # the same model's prompts
        _route('route_groups_8192', 8192, 256, 8, 'sigmoid', True, 8, 4, 2, scale=2.5),
        # more and smaller experts, 16-bit logits with their many ties
        _route('route_wide_2000', 2000, 512, 10, dtype='bf16'),
        # few experts, weights as they are, an odd number of rows and of columns
        _route('route_few_1121', 1121, 60, 4, renormalize=False, dtype='fp16', pad=3),
        # one user with an adapter on a layer's largest projection: latency
        _adapter('adapter_1', 1, 1, 4, 16, 6144, 2048),
        # a decode batch, each row a request with an adapter of its own
        _adapter('adapter_32', 32, 32, 16, 16, 6144, 2048),
        # a full batch on a merged pair of projections, each with its own adapter, of a higher rank
        _adapter('adapter_pair_64', 64, 64, 16, 64, 1024, 2048, parts=2),
        # sizes off every tile: fp32 results, rows inside a wider buffer
        _adapter('adapter_odd_77', 77, 50, 6, 24, 5003, 2120, dtype='fp16', out='fp32', pad=5),
        # decode rows of many requests back into the hidden size
        _adapter('adapter_down_256', 256, 256, 32, 16, 2048, 4096),
        # prompts of a few requests in one batch
        _adapter('adapter_1120', 1120, 4, 8, 32, 6144, 2048),
        # the largest batch: prompts beside decode rows
        _adapter('adapter_8192', 8192, 40, 16, 16, 6144, 2048),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    if rng.random() < 0.45:
        groups = rng.choice((1, 1, 1, 2, 4, 8, 8, 16))
        size = _spread(rng, max(2, 8 // groups), 512 // groups)
        kept = rng.randint(1, groups)
        experts = groups * size
        top = min(rng.choice((1, 2, 4, 6, 8, 8, 10, 16)), kept * size)
        score = rng.choice(('softmax', 'sigmoid'))
        return _route(None, _spread(rng, 1, 8192 * 256 // max(experts, 256)), experts, top, score,
                      rng.random() < 0.5, groups, kept, rng.choice((1, 2)), rng.random() < 0.75,
                      rng.choice((1.0, 1.0, 2.5)), rng.choice(('bf16', 'fp16', 'fp32')), rng.choice((0, 0, 1, 7)))
    k = 8 * _spread(rng, 32, 1024)
    parts = rng.choice((1, 1, 2, 3))
    n = parts * _spread(rng, 64, 8192 // parts)
    rows = _spread(rng, 1, min(8192, 8192 * 6144 // n, 8192 * 2048 // k))
    rank = rng.choice((8, 16, 16, 32, 64, 24))
    slots = _spread(rng, 1, max(1, min(64, 2 ** 24 // (rows * parts * rank), 2 ** 25 // (rank * (n + parts * k)))))
    requests = rows if rng.random() < 0.4 else _spread(rng, 1, rows)
    dtype = rng.choice(('bf16', 'bf16', 'fp16'))
    return _adapter(None, rows, requests, slots, rank, n, k, parts, dtype,
                    rng.choice((dtype, dtype, 'fp32')) if 2 * rows * n <= 8192 * 6144 else dtype, rng.choice((0, 0, 5, 8)))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed, part):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed * 1000 + part)
    return gen


@functools.cache
def _library():
    """The package, found once, as a program imports it."""
    path = str(ROOT / 'ornith-ciru-halo-agent_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    from ornith_g256 import native
    return native


def _wide(value, pad, dtype):
    wide = torch.zeros((value.shape[0], value.shape[1] + pad), dtype=dtype, device='cuda')
    wide[:, :value.shape[1]] = value
    return wide[:, :value.shape[1]]


def _route_inputs(case, seed):
    """Gate logits: some experts are popular, and each row has its own taste.
    The bias works against popularity, as balancing leaves it."""
    rows, experts, gen = case['rows'], case['experts'], _gen(seed, 1)
    popular = 0.7 * torch.randn(experts, generator=gen, device='cuda')
    z = popular + 1.3 * torch.randn((rows, experts), generator=gen, device='cuda')
    bias = None
    if case['bias']:
        bias = 0.02 * torch.randn(experts, generator=gen, device='cuda') - 0.1 * popular
        if case['score'] == 'softmax':
            bias = bias / experts
    return dict(case=case, logits=_wide(z, case['pad'], DTYPES[case['dtype']]), bias=bias)


def _adapter_inputs(case, seed):
    """Rows in runs, one a request; a request in eight has no adapter."""
    rows, n, k, rank, slots, parts = (case[f] for f in ('rows', 'n', 'k', 'rank', 'slots', 'parts'))
    gen, dtype = _gen(seed, 1), DTYPES[case['dtype']]
    x = torch.randn((rows, k), generator=gen, device='cuda').to(dtype)
    a = (torch.randn((slots, parts * rank, k), generator=gen, device='cuda') / math.sqrt(k)).to(dtype)
    b = (torch.randn((slots, n, rank), generator=gen, device='cuda') / math.sqrt(rank)).to(dtype)
    scales = 0.25 + 0.5 * torch.rand(slots, generator=gen, device='cuda')
    base = torch.randn((rows, n), generator=gen, device='cuda')
    starts = torch.zeros(rows, dtype=torch.int64, device='cuda')
    if case['requests'] < rows:
        places = torch.randperm(rows - 1, generator=gen, device='cuda')[:case['requests'] - 1] + 1
        starts[places] = 1
    else:
        starts[1:] = 1
    of = starts.cumsum(0)
    slot = torch.randint(slots, (case['requests'],), generator=gen, device='cuda')
    none = torch.rand(case['requests'], generator=gen, device='cuda') < 0.125
    none[0] = False
    ids = torch.where(none, -1, slot)[of].int()
    return dict(case=case, x=x, a=a, b=b, scales=scales, base=_wide(base, case['pad'], DTYPES[case['out']]), ids=ids)


def prepare(case, seed):
    state = (_route_inputs if case['kind'] == 'route' else _adapter_inputs)(case, seed)
    if not own:
        return state
    # what the program allocates once
    native, rows = _library(), case['rows']
    state['flags'] = torch.zeros(1, dtype=torch.int32, device='cuda')
    if case['kind'] == 'route':
        state['weights'] = torch.empty((rows, case['top']), dtype=torch.float32, device='cuda')
        state['ids'] = torch.empty((rows, case['top']), dtype=torch.int32, device='cuda')
    else:
        state['workspace'] = torch.empty(native.adapter_bytes(rows, case['parts'] * case['rank']), dtype=torch.uint8,
                                         device='cuda')
        state['out'] = torch.empty_strided(state['base'].shape, state['base'].stride(), dtype=DTYPES[case['out']],
                                           device='cuda')
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    if state['case']['kind'] == 'route':
        return _route_own(state) if own else _route_plain(state)
    return _adapter_own(state) if own else _adapter_plain(state)


def _route_own(state):
    case = state['case']
    _library().route_experts(state['logits'], state['weights'], state['ids'], state['flags'], score=case['score'],
                             bias=state['bias'], groups=case['groups'], kept_groups=case['kept'],
                             group_top=case['group_top'], renormalize=case['renormalize'], scale=case['scale'])
    return dict(weights=state['weights'], ids=state['ids'])


def _adapter_own(state):
    case = state['case']
    _library().adapter_out(state['x'], state['a'], state['b'], state['scales'], state['ids'], state['base'], state['out'],
                           state['workspace'], state['flags'], slices=_slices(case))
    return state['out']


def _slices(case):
    return (case['n'] // case['parts'],) * case['parts']


def _route_plain(state):
    """In 64 bits: scores and sums of scores decide which of two experts is picked."""
    case, z = state['case'], state['logits'].double()
    rows, experts = z.shape
    groups, top = case['groups'], case['top']
    if case['score'] == 'softmax':
        e = torch.exp(z - z.max(1, keepdim=True).values)
        s = e / e.sum(1, keepdim=True)
    else:
        s = 1 / (1 + torch.exp(-z))
    c = s if state['bias'] is None else s + state['bias'].double()
    if case['kept'] < groups:
        best = torch.sort(c.view(rows, groups, -1), dim=2, descending=True).values[:, :, :case['group_top']].sum(2)
        order = torch.sort(best, dim=1, descending=True, stable=True).indices[:, :case['kept']]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter(1, order, True)
        c = torch.where(keep.repeat_interleave(experts // groups, 1), c, -math.inf)
    ids = torch.sort(c, dim=1, descending=True, stable=True).indices[:, :top]
    w = s.gather(1, ids)
    if case['renormalize']:
        w = w / w.sum(1, keepdim=True)
    return dict(weights=(w * case['scale']).float(), ids=ids.int())


def _adapter_plain(state):
    """Every row against every slot's A, the other slots' results cleared, then
    against every slot's B."""
    case, ids = state['case'], state['ids']
    rows, k = state['x'].shape
    slots, rank, parts = case['slots'], case['rank'], case['parts']
    of = ids.unsqueeze(1) == torch.arange(slots, device=ids.device)
    v = (state['x'].float() @ state['a'].float().view(-1, k).t()).view(rows, slots, parts, rank)
    v = v * (of * state['scales']).view(rows, slots, 1, 1)
    b = state['b'].float().view(slots, parts, -1, rank)
    delta = torch.cat([v[:, :, p].reshape(rows, -1) @ b[:, p].permute(0, 2, 1).reshape(slots * rank, -1)
                       for p in range(parts)], 1)
    return torch.where(ids.unsqueeze(1) < 0, state['base'], (state['base'].float() + delta).to(state['base'].dtype))


# ---------------------------------------------------------------------------
# What it takes, and the results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    rows, size = case['rows'], 4 if case['dtype'] == 'fp32' else 2
    if case['kind'] == 'route':
        # per logit: a difference, an exponential, a sum or a division, a bias and a comparison
        return dict(bytes=rows * (case['experts'] * size + case['top'] * 8) + (case['experts'] * 4 if case['bias'] else 0),
                    flops=5 * rows * case['experts'])
    n, k, rank, parts = case['n'], case['k'], case['rank'], case['parts']
    adapted = rows * (1 + 0.875 * (case['requests'] - 1)) / case['requests']
    used = case['slots'] * (1 - (1 - 1 / case['slots']) ** (1 + 0.875 * (case['requests'] - 1)))
    out = 4 if case['out'] == 'fp32' else 2
    return dict(bytes=adapted * k * 2 + used * rank * (parts * k + n) * 2 + rows * (2 * n * out + 4),
                flops=2 * adapted * rank * (parts * k + n))


def exact(case, seed):
    return _route_exact(_route_inputs(case, seed)) if case['kind'] == 'route' else _adapter_exact(_adapter_inputs(case, seed))


def _route_exact(state):
    """On the host: ranks by (value, -id), whole groups struck out."""
    case = state['case']
    z = state['logits'].float().cpu().numpy().astype(np.float64)
    rows, experts = z.shape
    if case['score'] == 'softmax':
        s = np.exp(z - np.logaddexp.reduce(z, axis=1)[:, None])
    else:
        s = np.exp(-np.logaddexp(0.0, -z))
    # without a bias the order of the scores is that of the logits
    c = z if state['bias'] is None else s + state['bias'].cpu().numpy().astype(np.float64)
    names = np.broadcast_to(np.arange(experts), z.shape)
    size = experts // case['groups']
    if case['kept'] < case['groups']:
        by = c if case['group_top'] == 1 or state['bias'] is not None else s
        score = np.partition(by.reshape(rows, -1, size), size - case['group_top'], axis=2)[:, :, -case['group_top']:].sum(2)
        worst = np.lexsort((np.broadcast_to(np.arange(case['groups']), score.shape), -score), axis=1)[:, case['kept']:]
        gone = np.zeros_like(score, dtype=bool)
        np.put_along_axis(gone, worst, True, axis=1)
        c = np.where(np.repeat(gone, size, axis=1), -np.inf, c)
    ids = np.lexsort((names, -c), axis=1)[:, :case['top']]
    w = np.take_along_axis(s, ids, axis=1)
    if case['renormalize']:
        w = w / w.sum(1, keepdims=True)
    return dict(weights=torch.from_numpy(w * case['scale']), ids=torch.from_numpy(ids.astype(np.int32)))


def _adapter_exact(state):
    case, ids = state['case'], state['ids'].cpu().tolist()
    rank, parts, width = case['rank'], case['parts'], case['n'] // case['parts']
    out = state['base'].double().clone()
    for slot in sorted(set(ids) - {-1}):
        at = torch.tensor([t for t, i in enumerate(ids) if i == slot], device='cuda')
        v = state['x'][at].double() @ state['a'][slot].double().t()
        for p in range(parts):
            cols = slice(p * width, (p + 1) * width)
            out[at, cols] += state['scales'][slot].double() * (v[:, p * rank:(p + 1) * rank]
                                                               @ state['b'][slot, cols].double().t())
    return out
