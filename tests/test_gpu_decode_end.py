"""The end of a decode step as a server runs it: a plain 4-bit head, then the
sampler on its fp32 logits; captured and replayed, on several streams, with a
shared workspace, through the layer methods, and at addresses past 32 bits."""
import numpy as np
import pytest

from oracle import sampling as S
from oracle import w4 as W

pytestmark = pytest.mark.gpu

N, K, GROUP, ROWS = 20011, 512, 64, 6


def _head(rng, device, n=N, k=K, group=GROUP):
    import torch
    from ornith_g256 import storage
    words = rng.integers(0, 2 ** 32, (n, k // 8), dtype=np.uint32)
    scales = torch.from_numpy(rng.uniform(0.002, 0.01, (n, k // group))).to(torch.bfloat16).to(device)
    zeros = torch.from_numpy(rng.integers(6, 11, (n, k // group)).astype(np.uint8)).to(device)
    banks = storage.pack_w4(torch.from_numpy(words.view(np.int32)).to(device), scales, zeros, group)
    weights = W.weights(words, scales.double().cpu().numpy(), zeros.cpu().numpy(), group)
    return banks, weights


class Step:
    """Buffers of one decode step and its two calls."""

    def __init__(self, banks, device, rows=ROWS, workspace=None):
        import torch
        from ornith_g256 import native
        self.native, self.banks = native, banks
        self.x = torch.zeros((rows, K), dtype=torch.bfloat16, device=device)
        self.logits = torch.empty((rows, N), dtype=torch.float32, device=device)
        self.token = torch.empty(rows, dtype=torch.int64, device=device)
        self.logprob = torch.empty(rows, dtype=torch.float32, device=device)
        self.uniform = torch.zeros(rows, device=device)
        self.settings = dict(temperature=torch.ones(rows, device=device),
                             top_k=torch.zeros(rows, dtype=torch.int32, device=device),
                             top_p=torch.ones(rows, device=device), min_p=torch.zeros(rows, device=device))
        self.flags = torch.zeros(1, dtype=torch.int32, device=device)
        self.workspace = workspace if workspace is not None else torch.empty(
            native.logits_sample_bytes(rows, N), dtype=torch.uint8, device=device)

    def fill(self, rng):
        import torch
        rows = self.x.shape[0]
        self.x.copy_(torch.from_numpy(rng.standard_normal(self.x.shape).astype(np.float32)))
        self.uniform.copy_(torch.from_numpy(rng.random(rows).astype(np.float32)))
        for name, values in (('temperature', [0.0, 0.7, 1.0, 1.3]), ('top_k', [0, 1, 20, 3000]),
                             ('top_p', [1.0, 0.9, 0.5]), ('min_p', [0.0, 0.0, 0.05])):
            self.settings[name].copy_(torch.from_numpy(rng.choice(values, rows)))

    def run(self):
        self.native.w4_out(self.x, *self.banks, self.logits, self.flags, N, K, GROUP)
        self.native.logits_sample(self.logits, self.uniform, self.workspace, self.token, self.flags,
                                  logprob=self.logprob, **self.settings)

    def results(self):
        return [t.cpu().clone() for t in (self.logits, self.token, self.logprob)]


def _same(a, b):
    import torch
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def test_step_against_the_definitions(device):
    import torch
    rng = np.random.default_rng(1)
    banks, weights = _head(rng, device)
    step = Step(banks, device)
    step.fill(rng)
    step.run()
    torch.cuda.synchronize()
    logits, token, logprob = step.results()
    x = step.x.double().cpu().numpy()
    want = x @ weights.T
    # fp32 sums: 128 + K / 128 + 8 additions of at most 32 |s x| a term, and half a step of fp32
    scale = 32 * np.abs(x).sum(1, keepdims=True) * 0.01
    assert (np.abs(logits.double().numpy() - want) <= (140 * 2.0 ** -23) * scale).all()
    for m in range(ROWS):
        s = {k: float(v[m]) for k, v in step.settings.items()}
        args = (s['temperature'], int(s['top_k']), s['top_p'], s['min_p'])
        row = logits[m].double().numpy()                # the sampler's own input
        t, lp = S.sample(row, *args, float(step.uniform[m]))
        if args[0] > 0:
            # decided by arithmetic: u's distance to the ends of the token's interval
            mid, width = S.uniform_for(row, *args, t)
            assert abs(float(step.uniform[m]) - mid) < width / 2 - 2.0 ** -30
        assert int(token[m]) == t and abs(float(logprob[m]) - lp) <= 2.0 ** -24 * abs(lp) + 2.0 ** -21
    assert int(step.flags.item()) == 0


@pytest.mark.parametrize('rows', [1, 6, 130])
def test_captured_step_replays(device, rows):
    """Replays with new inputs each time, eager work and waits between them."""
    import torch
    rng = np.random.default_rng(2)
    banks, _ = _head(rng, device)
    step, eager = Step(banks, device, rows), Step(banks, device, rows)
    stream = torch.cuda.Stream()
    step.fill(rng)
    with torch.cuda.stream(stream):
        step.run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step.run()
    for r in range(5):
        seed = np.random.default_rng(100 + r)
        step.fill(seed)
        eager.fill(np.random.default_rng(100 + r))
        eager.run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert _same(step.results(), eager.results()), r
    assert int(step.flags.item()) == int(eager.flags.item()) == 0


def test_two_graphs_share_a_workspace(device):
    import torch
    rng = np.random.default_rng(3)
    banks, _ = _head(rng, device)
    first = Step(banks, device, 40)
    second = Step(banks, device, 3, workspace=first.workspace)
    stream = torch.cuda.Stream()
    graphs = []
    for step in (first, second):
        step.fill(rng)
        with torch.cuda.stream(stream):
            step.run()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                step.run()
        graphs.append(g)
    want = []
    for step in (first, second):
        alone = Step(banks, device, step.x.shape[0])
        for name in ('x', 'uniform'):
            getattr(alone, name).copy_(getattr(step, name))
        for k in alone.settings:
            alone.settings[k].copy_(step.settings[k])
        alone.run()
        torch.cuda.synchronize()
        want.append(alone.results())
    for _ in range(3):
        with torch.cuda.stream(stream):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        assert _same(first.results(), want[0]) and _same(second.results(), want[1])


def test_streams_with_workspaces_of_their_own(device):
    import torch
    rng = np.random.default_rng(4)
    banks, _ = _head(rng, device)
    steps = [Step(banks, device, r) for r in (1, 5, 12, 70)]
    for step in steps:
        step.fill(rng)
        step.run()
    torch.cuda.synchronize()
    want = [s.results() for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(4):
        for step in steps:
            step.token.fill_(-5)
            step.logprob.zero_()
        torch.cuda.synchronize()
        for step, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                step.run()
        torch.cuda.synchronize()
        assert all(_same(s.results(), w) for s, w in zip(steps, want))


def test_layer_methods(device):
    """A W4 linear and the W8 head on one runtime; the head's sampler."""
    import torch
    from ornith_g256 import methods, native

    class Layer(torch.nn.Module):
        def __init__(self, method):
            super().__init__()
            self.quant_method = method
            method.create_weights(self)

    rng = np.random.default_rng(5)
    n, k = 700, 2048
    lin = Layer(methods.W4LinearMethod('lin', n, k, group=32, zeros=True, scale_dtype=torch.float16)).to(device)
    words = rng.integers(0, 2 ** 32, (n, k // 8), dtype=np.uint32)
    scales = torch.from_numpy(2.0 ** rng.integers(-6, -3, (n, k // 32))).half()
    zeros = torch.from_numpy(rng.integers(0, 16, (n, k // 32)).astype(np.uint8))
    lin.load_packed('w4_codes', torch.from_numpy(words))
    lin.load_packed('w4_scales', scales)
    lin.load_packed('w4_zeros', zeros)
    lin.quant_method.process_weights_after_loading(lin)
    assert not hasattr(lin, 'w4_codes') and lin.w4_bank.is_cuda
    head = Layer(methods.W8HeadMethod('head')).to(device)
    codes = torch.from_numpy(rng.integers(0, 2 ** 32, (native.HEAD_VOCAB // 16, 128, 4, 16), dtype=np.uint32))
    head.load_packed('head_tilebank_codes', codes)
    head.load_packed('head_scales', torch.from_numpy(rng.uniform(1e-4, 3e-4, (native.HEAD_VOCAB, 16))).half())
    head.quant_method.process_weights_after_loading(head)
    model = torch.nn.ModuleDict(dict(lin=lin, head=head))
    native.reset_binding()
    rt = methods.Runtime(model, {}, 128, device)
    try:
        x = torch.from_numpy(rng.integers(-3, 4, (5, 3, k)).astype(np.float32)).to(torch.bfloat16).to(device)
        out = lin.quant_method.apply(lin, x)
        want = x.double().cpu().numpy() @ W.weights(words, scales.double().numpy(), zeros.numpy(), 32).T
        assert out.shape == (5, 3, n)
        assert torch.equal(out.cpu(), torch.from_numpy(want).to(torch.bfloat16))
        h = torch.randn((70, 2048), device=device).to(torch.bfloat16)
        logits = head.quant_method.apply(head, h)
        uniform = torch.rand(70, device=device)
        top_k = torch.randint(1, 30, (70,), dtype=torch.int32, device=device)
        token, logprob = head.quant_method.sample(head, h, uniform, top_k=top_k)
        kth = torch.sort(logits.float(), dim=1, descending=True).values.gather(1, top_k.long().unsqueeze(1) - 1)
        picked = logits.float().gather(1, token.unsqueeze(1))
        assert bool((picked >= kth).all()) and bool((logprob <= 0).all())
        greedy, _ = head.quant_method.sample(head, h, uniform, temperature=torch.zeros(70, device=device))
        best = torch.empty(70, dtype=torch.int64, device=device)
        native.logits_argmax(logits, best)
        assert torch.equal(greedy, best)
        rt.check_error_flags()
    finally:
        native.reset_binding()


@pytest.mark.parametrize('bad', ['nan', 'inf', 'zero'])
def test_pack_admission(device, bad):
    import torch
    from ornith_g256 import storage
    codes = torch.zeros((33, 8), dtype=torch.int32, device=device)
    scales = torch.ones((33, 2), dtype=torch.float16, device=device)
    zeros = torch.full((33, 2), 15, dtype=torch.uint8, device=device)
    storage.pack_w4(codes, scales, zeros, 32)
    if bad == 'zero':
        zeros[32, 1] = 16
    else:
        scales[7, 0] = float(bad)
    with pytest.raises(storage.AdmissionError):
        storage.pack_w4(codes, scales, zeros, 32)


def test_logits_past_32_bits(device):
    """Rows 2.4 GB apart."""
    import torch
    from ornith_g256 import native
    rng = np.random.default_rng(6)
    M, n, ld = 4, 20000, 1_200_000_000
    buf = torch.zeros(3 * ld + n, dtype=torch.bfloat16, device=device)
    logits = buf.as_strided((M, n), (ld, 1))
    near = torch.from_numpy(rng.standard_normal((M, n)).astype(np.float32) * 2).to(torch.bfloat16).to(device)
    logits.copy_(near)
    uniform = torch.rand(M, device=device)
    top_p = torch.tensor([0.9, 1.0, 0.5, 0.7], device=device)
    got = []
    for l in (logits, near):
        ws = torch.empty(native.logits_sample_bytes(M, n), dtype=torch.uint8, device=device)
        token, logprob = torch.empty(M, dtype=torch.int64, device=device), torch.empty(M, device=device)
        flags = torch.zeros(1, dtype=torch.int32, device=device)
        native.logits_sample(l, uniform, ws, token, flags, top_p=top_p, logprob=logprob)
        got.append((token.cpu(), logprob.cpu()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_bank_and_output_past_32_bits(device):
    """A bank of 4.3 GB whose last columns are known, and output rows 3.2 GB apart."""
    import torch
    from ornith_g256 import native, storage
    rng = np.random.default_rng(7)
    n, k, group, M = 1 << 20, 8192, 256, 20
    codes = torch.zeros((n, k // 8), dtype=torch.int32, device=device)
    words = rng.integers(0, 2 ** 32, (40, k // 8), dtype=np.uint32)
    codes[-40:] = torch.from_numpy(words.view(np.int32)).to(device)
    scales = torch.full((n, k // group), 0.0625, dtype=torch.bfloat16, device=device)
    banks = storage.pack_w4(codes, scales, None, group)
    del codes
    x = torch.from_numpy(rng.integers(-2, 3, (M, k)).astype(np.float32)).to(torch.bfloat16).to(device)
    flags = torch.zeros(1, dtype=torch.int32, device=device)
    want = x.double().cpu().numpy() @ W.weights(words, np.full((40, k // group), 0.0625), None, group).T
    for rows, ld in ((M, n), (3, 800_000_000)):
        buf = torch.empty((rows - 1) * ld + n, dtype=torch.float32, device=device)
        out = buf.as_strided((rows, n), (ld, 1))
        native.w4_out(x[:rows], *banks, out, flags, n, k, group)
        assert (out[:, -40:].double().cpu().numpy() == want[:rows]).all()
        # zero codes: -8 times the row's sum
        first = -8 * 0.0625 * x[:rows].double().sum(1).cpu().numpy()
        assert (out[:, :100].double().cpu().numpy() == first[:, None]).all()
        del buf, out
    assert int(flags.item()) == 0


def test_rows_past_one_grid(device):
    """More rows than a grid of 1024 threads a row can hold."""
    import torch
    from ornith_g256 import native
    rng = np.random.default_rng(8)
    n, some, M = 8, 1024, (1 << 22) + 1024
    near = torch.from_numpy(rng.standard_normal((some, n)).astype(np.float32)).to(torch.bfloat16).to(device)
    uniform, top_p = torch.rand(some, device=device), torch.full((some,), 0.8, device=device)
    got = []
    for times in (1, M // some):
        token = torch.full((times * some,), -7, dtype=torch.int64, device=device)
        flags = torch.zeros(1, dtype=torch.int32, device=device)
        native.logits_sample(near.repeat(times, 1), uniform.repeat(times), torch.empty(0, dtype=torch.uint8, device=device),
                             token, flags, top_p=top_p.repeat(times))
        assert int(flags) == 0
        got.append(token)
    assert torch.equal(got[1].view(-1, some), got[0].expand(M // some, some))


def test_pack_past_one_grid(device):
    """A bank of more 32-bit words than a grid has threads; its first and last columns are known."""
    import torch
    from ornith_g256 import native, storage
    rng = np.random.default_rng(9)
    n, k, group = 1 << 20, 32776, 256
    codes = torch.zeros((n, k // 8), dtype=torch.int32, device=device)
    words = rng.integers(0, 2 ** 32, (24, k // 8), dtype=np.uint32)
    codes[:24] = torch.from_numpy(words.view(np.int32)).to(device)
    codes[-24:] = codes[:24]
    groups = (k + group - 1) // group
    banks = storage.pack_w4(codes, torch.full((n, groups), 0.0625, dtype=torch.bfloat16, device=device), None, group)
    del codes
    x = torch.from_numpy(rng.integers(-2, 3, (1, k)).astype(np.float32)).to(torch.bfloat16).to(device)
    flags = torch.zeros(1, dtype=torch.int32, device=device)
    out = torch.empty((1, n), dtype=torch.float32, device=device)
    native.w4_out(x, *banks, out, flags, n, k, group)
    want = x.double().cpu().numpy() @ W.weights(words, np.full((24, groups), 0.0625), None, group).T
    got = out.double().cpu().numpy()
    assert (got[:, :24] == want).all() and (got[:, -24:] == want).all()
    assert (got[:, 24:-24] == -8 * 0.0625 * x.double().sum().item()).all()
