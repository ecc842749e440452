"""Sampling and plain 4-bit linears: the end of a decode step and the products
before it, as a serving program calls them.

* ``sample`` - one token a row from a head's logits: temperature, top-k, top-p
  and min-p per row and one given uniform number per row
  (``native.logits_sample``).
* ``w4`` - a linear or a head whose 4-bit weights carry a scale, and perhaps a
  zero point, per group of 32 to 256 inputs (``native.w4_out`` on the banks of
  ``storage.pack_w4``).

The plain forms are the definitions in elementary torch operations.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

ROOT = Path(__file__).resolve().parent.parent
DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
W8_VOCAB, G256_VOCAB = 248320, 151936


def listed():
    return [
        # one user's next token with the usual chat settings, after the W8 head
        dict(name='sample_chat_1', kind='sample', rows=1, n=W8_VOCAB, pad=0, dtype='bf16', mix='chat'),
        # a few users, nucleus only, on the fp32 logits of the G256 head
        dict(name='sample_nucleus_8', kind='sample', rows=8, n=G256_VOCAB, pad=0, dtype='fp32', mix='nucleus'),
        # a full batch where every request has settings of its own (greedy, grammar masks and all)
        dict(name='sample_mixed_64', kind='sample', rows=64, n=W8_VOCAB, pad=0, dtype='bf16', mix='mixed'),
        # a full batch drawn from the whole distribution (rollouts)
        dict(name='sample_whole_64', kind='sample', rows=64, n=W8_VOCAB, pad=0, dtype='bf16', mix='whole'),
        # draft positions over a shortened vocabulary, odd sizes, rows inside a wider buffer
        dict(name='sample_odd_33', kind='sample', rows=33, n=50001, pad=7, dtype='fp16', mix='mixed'),
        # many short rows: a shortlist re-scored per position
        dict(name='sample_short_256', kind='sample', rows=256, n=4096, pad=0, dtype='bf16', mix='mixed'),
        # the smallest linear of a layer, one user: latency
        dict(name='w4_1_small', kind='w4', rows=1, n=2048, k=512, group=128, zeros=False, dtype='bf16', out='bf16'),
        # a decode step's projections: one user, a few, and a full batch
        dict(name='w4_1', kind='w4', rows=1, n=6144, k=2048, group=128, zeros=False, dtype='bf16', out='bf16'),
        dict(name='w4_8_g32', kind='w4', rows=8, n=12288, k=2048, group=32, zeros=False, dtype='bf16', out='bf16'),
        dict(name='w4_64', kind='w4', rows=64, n=2048, k=4096, group=128, zeros=True, dtype='fp16', out='fp16'),
        # sizes off every tile: a pruned layer whose last group is short
        dict(name='w4_5_odd', kind='w4', rows=5, n=5003, k=2120, group=64, zeros=True, dtype='fp16', out='fp16'),
        # a 4-bit head: fp32 logits for the sampler
        dict(name='w4_head_32', kind='w4', rows=32, n=G256_VOCAB, k=2048, group=128, zeros=True, dtype='bf16', out='fp32'),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    if rng.random() < 0.5:
        n = _spread(rng, 256, W8_VOCAB)
        rows = _spread(rng, 1, max(1, min(512, 64 * W8_VOCAB // n)))
        dtype = rng.choice(('bf16', 'fp16', 'fp32'))
        return dict(kind='sample', rows=rows if dtype != 'fp32' else (rows + 1) // 2, n=n,
                    pad=rng.choice((0, 0, rng.randint(1, 100))), dtype=dtype,
                    mix=rng.choice(('chat', 'nucleus', 'mixed', 'mixed', 'whole')))
    k = 8 * _spread(rng, 8, 1024)
    n = _spread(rng, 64, min(G256_VOCAB, G256_VOCAB * 2048 // k))
    dtype = rng.choice(('bf16', 'fp16'))
    rows = _spread(rng, 1, 64 if 64 * n * k <= 32 * G256_VOCAB * 2048 else 32)
    return dict(kind='w4', rows=rows, n=n, k=k, group=rng.choice((32, 64, 128, 128, 256)),
                zeros=rng.random() < 0.5, dtype=dtype, out=rng.choice((dtype, dtype, 'fp32')))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _gen(seed, part):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed * 1000 + part)
    return gen


def _library():
    path = str(ROOT / 'ornith-ciru-halo-agent_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    from ornith_g256 import native, storage
    return native, storage


def _logits(case, seed):
    """Head logits: a broad body and, row by row, a tail that ranges from none
    (an unsure model) to a few dominant tokens."""
    rows, n, gen = case['rows'], case['n'], _gen(seed, 1)
    z = torch.randn((rows, n), generator=gen, device='cuda')
    spread = 1.5 + 1.5 * torch.rand((rows, 1), generator=gen, device='cuda')
    tail = 0.12 * torch.rand((rows, 1), generator=gen, device='cuda') ** 2
    z = spread * z * (1 + tail * z.clamp_min(0) ** 2)
    if case['mix'] == 'mixed':
        # one request in four is bound to a grammar: most columns are masked
        bound = torch.rand((rows, 1), generator=gen, device='cuda') < 0.25
        allowed = torch.rand((rows, n), generator=gen, device='cuda') < 0.02
        allowed[:, n // 2] = True
        z = torch.where(bound & ~allowed, -math.inf, z)
    wide = torch.zeros((rows, n + case['pad']), dtype=DTYPES[case['dtype']], device='cuda')
    wide[:, :n] = z
    return wide[:, :n]


def _settings(case, seed):
    rows, mix, gen = case['rows'], case['mix'], _gen(seed, 2)

    def pick(*values):
        of = torch.tensor(values, device='cuda')
        return of[torch.randint(len(values), (rows,), generator=gen, device='cuda')]

    s = dict(temperature=pick(0.6, 0.7, 0.8, 1.0), top_k=None, top_p=None, min_p=None)
    if mix == 'chat':
        s |= dict(top_k=pick(20, 40, 50).int(), top_p=pick(0.9, 0.95))
    elif mix == 'nucleus':
        s |= dict(top_p=pick(0.8, 0.9, 0.95))
    elif mix == 'mixed':
        s |= dict(temperature=pick(0.0, 0.3, 0.7, 1.0, 1.0, 1.3), top_k=pick(0, 0, 1, 20, 50, 200).int(),
                  top_p=pick(1.0, 1.0, 0.95, 0.9, 0.5), min_p=pick(0.0, 0.0, 0.02, 0.1))
    return s


def _sample_inputs(case, seed):
    uniform = torch.rand((case['rows'],), generator=_gen(seed, 3), device='cuda')
    return dict(case=case, logits=_logits(case, seed), settings=_settings(case, seed), uniform=uniform)


def _w4_inputs(case, seed):
    n, k, gen = case['n'], case['k'], _gen(seed, 1)
    groups = -(-k // case['group'])
    x = torch.randn((case['rows'], k), generator=gen, device='cuda').to(DTYPES[case['dtype']])
    codes = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), generator=gen, dtype=torch.int64, device='cuda').int()
    scales = (0.005 + 0.015 * torch.rand((n, groups), generator=gen, device='cuda')).to(DTYPES[case['dtype']])
    zeros = None
    if case['zeros']:
        zeros = (8 + 1.5 * torch.randn((n, groups), generator=gen, device='cuda')).round().clamp(0, 15).to(torch.uint8)
    return dict(case=case, x=x, codes=codes, scales=scales, zeros=zeros)


def prepare(case, seed):
    state = (_sample_inputs if case['kind'] == 'sample' else _w4_inputs)(case, seed)
    if not own:
        return state
    # what the program allocates once, and the weights in the library's layout
    native, storage = _library()
    rows, n = case['rows'], case['n']
    state['flags'] = torch.zeros(1, dtype=torch.int32, device='cuda')
    if case['kind'] == 'sample':
        state['workspace'] = torch.empty(native.logits_sample_bytes(rows, n), dtype=torch.uint8, device='cuda')
        state['token'] = torch.empty(rows, dtype=torch.int64, device='cuda')
        state['logprob'] = torch.empty(rows, dtype=torch.float32, device='cuda')
    else:
        state['codes'], state['meta'] = storage.pack_w4(state['codes'], state.pop('scales'), state.pop('zeros'),
                                                        case['group'])
        state['out'] = torch.empty((rows, n), dtype=DTYPES[case['out']], device='cuda')
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    if state['case']['kind'] == 'sample':
        return _sample_own(state) if own else _sample_plain(state)
    return _w4_own(state) if own else _w4_plain(state)


def _sample_own(state):
    native, _ = _library()
    native.logits_sample(state['logits'], state['uniform'], state['workspace'], state['token'], state['flags'],
                         logprob=state['logprob'], **state['settings'])
    return dict(token=state['token'], logprob=state['logprob'])


def _w4_own(state):
    native, _ = _library()
    case = state['case']
    native.w4_out(state['x'], state['codes'], state['meta'], state['out'], state['flags'], case['n'], case['k'],
                  case['group'])
    return state['out']


def _sample_plain(state):
    """In 64 bits: a cumulative sum over a vocabulary of small masses, read
    next to a border."""
    s, u = state['settings'], state['uniform'].double().unsqueeze(1)
    x = state['logits'].double()
    rows, n = x.shape
    rank = torch.arange(n, device=x.device)
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.max(1, keepdim=True).values
    t = s['temperature'].double().unsqueeze(1)
    e = torch.exp((x - top) / torch.where(t > 0, t, 1.0))
    e = torch.where(x == top, 1.0, e)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ordered = e.gather(1, order)
    keep = torch.ones_like(ordered, dtype=torch.bool)
    if s['top_k'] is not None:
        k = s['top_k'].unsqueeze(1)
        keep = (rank < k) | (k <= 0)
    if s['top_p'] is not None:
        p = s['top_p'].double().unsqueeze(1)
        left = ordered * keep
        running = left.cumsum(1)
        keep = keep & ((running - left < p * left.sum(1, keepdim=True)) | (p >= 1))
    if s['min_p'] is not None:
        keep = keep & (ordered >= s['min_p'].double().unsqueeze(1))
    keep = torch.where(t > 0, keep, rank == 0)
    kept = torch.zeros_like(e).scatter(1, order, ordered * keep)
    running = kept.cumsum(1)
    total = running[:, -1:]
    token = (running > u * total).int().argmax(1)
    logprob = torch.log(kept.gather(1, token.unsqueeze(1)) / total)
    return dict(token=token, logprob=logprob.squeeze(1).float())


def _w4_plain(state):
    case, codes = state['case'], state['codes']
    n, k, group = case['n'], case['k'], case['group']
    shifts = torch.arange(0, 32, 4, dtype=torch.int32, device=codes.device)
    q = ((codes.unsqueeze(2) >> shifts) & 15).view(n, k).float()
    of = torch.arange(k, device=codes.device) // group
    zero = 8.0 if state['zeros'] is None else state['zeros'].float()[:, of]
    w = (q - zero) * state['scales'].float()[:, of]
    return (state['x'].float() @ w.t()).to(DTYPES[case['out']])


# ---------------------------------------------------------------------------
# What it takes, and the results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    size = 4 if case.get('dtype') == 'fp32' else 2
    rows, n = case['rows'], case['n']
    if case['kind'] == 'sample':
        settings = {'chat': 12, 'nucleus': 8, 'mixed': 16, 'whole': 4}[case['mix']]
        # per logit: a difference, a product, an exponential and a sum
        return dict(bytes=rows * (n * size + settings + 4 + 12), flops=4 * rows * n)
    k = case['k']
    groups = -(-k // case['group'])
    return dict(bytes=n * k // 2 + n * groups * 2 + (n * groups // 2 if case['zeros'] else 0) + rows * k * 2
                + rows * n * (4 if case['out'] == 'fp32' else 2), flops=2 * rows * n * k)


def exact(case, seed):
    return _sample_exact(_sample_inputs(case, seed)) if case['kind'] == 'sample' else _w4_exact(_w4_inputs(case, seed))


def _sample_exact(state):
    """Row by row on the host: sort, cut, walk."""
    host = {k: None if v is None else v.cpu().numpy() for k, v in state['settings'].items()}
    logits, uniform = state['logits'].float().cpu().numpy().astype(np.float64), state['uniform'].cpu().numpy()
    tokens, logprobs = [], []
    for m, row in enumerate(logits):
        live = np.flatnonzero(row > -np.inf)
        ids = live[np.argsort(-row[live], kind='stable')]
        temperature = float(host['temperature'][m])
        if temperature == 0:
            tokens.append(int(ids[0]))
            logprobs.append(0.0)
            continue
        mass = np.exp((row[ids] - row[ids[0]]) / temperature)
        count = len(ids)
        if host['top_k'] is not None and 0 < host['top_k'][m] < count:
            count = int(host['top_k'][m])
        if host['top_p'] is not None and host['top_p'][m] < 1:
            total = np.cumsum(mass[:count])
            count = min(count, int(np.searchsorted(total, float(host['top_p'][m]) * total[-1])) + 1)
        if host['min_p'] is not None:
            count = min(count, int((mass >= float(host['min_p'][m])).sum()))
        kept = np.sort(ids[:count])
        weight = np.exp((row[kept] - row[ids[0]]) / temperature)
        total = np.cumsum(weight)
        at = int(np.searchsorted(total, float(uniform[m]) * total[-1], side='right'))
        tokens.append(int(kept[at]))
        logprobs.append(math.log(weight[at] / total[-1]))
    return dict(token=torch.tensor(tokens), logprob=torch.tensor(logprobs, dtype=torch.float64))


def _w4_exact(state):
    case = state['case']
    x, codes, scales = state['x'].double(), state['codes'], state['scales'].double()
    zeros = torch.full_like(scales, 8.0) if state['zeros'] is None else state['zeros'].double()
    columns = torch.arange(case['k'], device=x.device)
    out = torch.empty((case['rows'], case['n']), dtype=torch.float64, device=x.device)
    for a in range(0, case['n'], 16384):
        word = codes[a:a + 16384].long() & 0xffffffff
        code = (word[:, columns // 8] >> (4 * (columns % 8))) & 15
        at = columns // case['group']
        out[:, a:a + 16384] = x @ ((code.double() - zeros[a:a + 16384][:, at]) * scales[a:a + 16384][:, at]).t()
    return out
