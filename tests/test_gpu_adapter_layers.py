"""Adapters and expert routing as a server runs them: beside the layers'
projections and before the routed experts; captured and replayed with other
requests, compiled, on several streams, with a shared workspace, at addresses
past 32 bits and with more rows than one pass takes."""
import numpy as np
import pytest

import test_gpu_adapter as A
from oracle import route as R

pytestmark = pytest.mark.gpu

CAP, SLOTS, RANK = 512, 5, 16


def _w4_layer(rng, device, n, k, prefix):
    import torch
    from ornith_g256 import methods
    layer = torch.nn.Module()
    layer.quant_method = methods.W4LinearMethod(prefix, n, k, group=64)
    layer.quant_method.create_weights(layer)
    layer.to(device)
    layer.load_packed('w4_codes', torch.from_numpy(rng.integers(0, 2 ** 32, (n, k // 8), dtype=np.uint32)))
    layer.load_packed('w4_scales', torch.from_numpy(rng.uniform(0.002, 0.006, (n, k // 64)).astype(np.float32)).to(torch.bfloat16))
    layer.quant_method.process_weights_after_loading(layer)
    return layer


def _meta(rng, shape):
    scale = rng.uniform(0.005, 0.02, shape).astype(np.float16)
    offset = (np.float32(-8) * scale.astype(np.float32)).astype(np.float16)
    return scale.view(np.uint16).astype(np.uint32) | offset.view(np.uint16).astype(np.uint32) << 16


def _g256_layer(rng, device, n, k, prefix):
    import torch
    from ornith_g256 import methods
    layer = torch.nn.Module()
    layer.quant_method = methods.G256LinearMethod(prefix, n, k)
    layer.quant_method.create_weights(layer)
    layer.load_packed('g256_codes', torch.from_numpy(rng.integers(0, 2 ** 32, (n // 16, k // 256, 32, 16), dtype=np.uint32)))
    layer.load_packed('g256_metadata', torch.from_numpy(_meta(rng, (n // 16, k // 256, 16))))
    layer.quant_method.process_weights_after_loading(layer)
    return layer.to(device)


def _experts(rng, device, routing):
    import torch
    from ornith_g256 import methods
    layer = torch.nn.Module()
    layer.quant_method = methods.G256MoEMethod('experts', routing)
    layer.quant_method.create_weights(layer)
    for proj, n, k in (('w13', 1024, 2048), ('w2', 2048, 512)):
        codes = rng.integers(0, 2 ** 32, (1, n // 16, k // 256, 32, 16), dtype=np.uint32)
        # (experts differ by their scales)
        layer.load_packed(f'{proj}_tilebank_codes', torch.from_numpy(np.broadcast_to(codes, (256, *codes.shape[1:])).copy()))
        layer.load_packed(f'{proj}_tilebank_metadata', torch.from_numpy(_meta(rng, (256, n // 16, k // 256, 16))))
    layer.quant_method.process_weights_after_loading(layer)
    return layer.to(device)


@pytest.fixture(scope='module')
def block(device):
    """x -> plain 4-bit projection -> G256 projection (two slices) -> gate -> routing -> experts."""
    import torch
    from ornith_g256 import methods, native
    rng = np.random.default_rng(1)
    model = torch.nn.Module()
    model.first = _w4_layer(rng, device, 2048, 1024, 'first')
    model.second = _g256_layer(rng, device, 2048, 2048, 'second')
    bias = torch.from_numpy((rng.standard_normal(256) * 0.05).astype(np.float32)).to(device)
    model.experts = _experts(rng, device, methods.ExpertRouting(8, 'sigmoid', 8, 4, 2, True, 2.5, bias))
    model.gate = torch.nn.Module()
    model.gate.weight = torch.nn.Parameter(torch.from_numpy((rng.standard_normal((256, 2048)) * 0.02).astype(np.float32))
                                           .to(torch.bfloat16).to(device), requires_grad=False)
    model.gate.quant_method = methods.RouterGateMethod('gate')
    for layer, slices in ((model.first, None), (model.second, (1500, 548))):
        ad = methods.attach_adapters(layer, SLOTS, RANK, slices)
        for slot in range(SLOTS - 1):                  # (the last slot is empty)
            r = (8, 16, 4, 16)[slot]
            a = [torch.from_numpy((rng.standard_normal((r, ad.k)) / np.sqrt(ad.k)).astype(np.float32)).to(torch.bfloat16)
                 for _ in ad.slices]
            ad.load(slot, a, torch.from_numpy((rng.standard_normal((ad.n, r)) * 0.3).astype(np.float32)).to(torch.bfloat16), 0.5 + slot)
    native.reset_binding()
    model.rt = methods.Runtime(model, {'routed_library': str(native.library_path(16))}, CAP, device)
    yield model
    native.reset_binding()


def _step(block, x):
    h = block.first.quant_method.apply(block.first, x)
    h = block.second.quant_method.apply(block.second, h)
    logits = block.gate.quant_method.apply(block.gate, h)
    return h, logits, block.experts.quant_method.apply_logits(block.experts, h, logits)


def _delta_case(layer, x, base, ids):
    ad = layer.adapters
    return dict(x=x, a=ad.a, b=ad.b, scales=ad.scales, ids=ids, base=base, slices=ad.slices, rank=ad.rank, dtype='bf16', out_type='bf16')


@pytest.mark.parametrize('rows', [1, 7, 40, 300])
def test_block(block, device, rows):
    import torch
    from ornith_g256 import native
    gen = torch.Generator(device=device).manual_seed(rows)
    x = torch.randn((rows, 1024), generator=gen, device=device).to(torch.bfloat16)
    ids = torch.randint(-1, SLOTS, (rows,), generator=gen, device=device).int()
    # each projection: its shared results, then the definition on them
    block.rt.set_adapter_ids(torch.full((rows,), -1, dtype=torch.int32, device=device))
    base = block.first.quant_method.apply(block.first, x)
    block.rt.set_adapter_ids(ids)
    h = block.first.quant_method.apply(block.first, x)
    A._check(_delta_case(block.first, x, base, ids), (h, 0))
    block.rt.set_adapter_ids(torch.full((rows,), -1, dtype=torch.int32, device=device))
    base = block.second.quant_method.apply(block.second, h)
    block.rt.set_adapter_ids(ids)
    h2 = block.second.quant_method.apply(block.second, h)
    A._check(_delta_case(block.second, h, base, ids), (h2, 0))
    got, logits, y = _step(block, x)
    assert torch.equal(got, h2)
    # the experts and their weights, and the routed kernels on them
    w, picked = block.experts.quant_method.routing.apply(logits, block.rt.slots[block.experts.quant_method.slot])
    bias = block.experts.quant_method.routing.bias.double().cpu().numpy()
    for m in range(rows):
        ww, wi, clear = R.route(logits[m].double().cpu().numpy(), 8, 'sigmoid', bias, 8, 4, 2, True, 2.5)
        if clear > 2.0 ** -38:
            assert picked[m].tolist() == wi.tolist()
            assert (np.abs(w[m].double().cpu().numpy() - ww) <= ww * (2.0 ** -24 + 2.0 ** -40)).all()
    assert torch.equal(block.experts.quant_method.apply(block.experts, h2, w, picked), y)
    assert block.rt.check_error_flags() == [0] * len(block.rt.slots)


@pytest.mark.parametrize('rows', [1, 33, 260])
def test_captured_block_replays_with_other_requests(block, device, rows):
    import torch
    x = torch.zeros((rows, 1024), dtype=torch.bfloat16, device=device)
    stream = torch.cuda.Stream()
    block.rt.set_adapter_ids(torch.zeros(rows, dtype=torch.int32, device=device))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        _step(block, x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = _step(block, x)
    for r in range(4):
        gen = torch.Generator(device=device).manual_seed(100 + r)
        x.copy_(torch.randn((rows, 1024), generator=gen, device=device))
        block.rt.set_adapter_ids(torch.randint(-1, SLOTS, (rows,), generator=gen, device=device).int())
        want = [t.clone() for t in _step(block, x)]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), r
    assert block.rt.check_error_flags() == [0] * len(block.rt.slots)


def _buffers(c):
    import torch
    from ornith_g256 import native
    M = c['base'].shape[0]
    return dict(out=torch.empty_like(c['base']), flags=torch.zeros(1, dtype=torch.int32, device=c['x'].device),
                workspace=torch.empty(native.adapter_bytes(M, c['a'].shape[1]), dtype=torch.uint8, device=c['x'].device))


def _call(c, b):
    from ornith_g256 import native
    native.adapter_out(c['x'], c['a'], c['b'], c['scales'], c['ids'], c['base'], b['out'], b['workspace'], b['flags'],
                       slices=c['slices'])


def test_streams_with_workspaces_of_their_own(device):
    import torch
    rng = np.random.default_rng(2)
    cases = [A._case(rng, M, 700, 512, R, 4, 1, 'bf16', 'bf16', device, False) for M, R in ((1, 16), (40, 64), (300, 16), (3000, 128))]
    buffers = [_buffers(c) for c in cases]
    for c, b in zip(cases, buffers):
        _call(c, b)
    torch.cuda.synchronize()
    want = [b['out'].clone() for b in buffers]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for b in buffers:
            b['out'].fill_(-1)
        torch.cuda.synchronize()
        for c, b, s in zip(cases, buffers, streams):
            with torch.cuda.stream(s):
                _call(c, b)
        torch.cuda.synchronize()
        assert all(torch.equal(b['out'], w) for b, w in zip(buffers, want))


def test_two_graphs_share_a_workspace(device):
    import torch
    rng = np.random.default_rng(3)
    cases = [A._case(rng, M, 300, 256, R, 6, 1, 'bf16', 'fp32', device, False) for M, R in ((500, 16), (90, 128))]
    buffers = [_buffers(c) for c in cases]
    buffers[1]['workspace'] = buffers[0]['workspace'] = torch.empty(
        max(b['workspace'].numel() for b in buffers), dtype=torch.uint8, device=device)
    want, graphs, stream = [], [], torch.cuda.Stream()
    for c, b in zip(cases, buffers):
        with torch.cuda.stream(stream):
            _call(c, b)
            torch.cuda.synchronize()
            want.append(b['out'].clone())
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=stream):
                _call(c, b)
            graphs.append(g)
    for _ in range(4):
        for b in buffers:
            b['out'].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(b['out'], w) for b, w in zip(buffers, want))


@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
def test_compiled(device, backend):
    import torch
    from ornith_g256 import native
    rng = np.random.default_rng(4)
    c = A._case(rng, 20, 260, 256, 16, 3, 2, 'bf16', 'fp32', device, False)
    b = _buffers(c)
    _call(c, b)
    want = b['out'].clone()
    weights, ids = torch.empty((20, 6), device=device), torch.empty((20, 6), dtype=torch.int32, device=device)
    native.route_experts(want, weights, ids, b['flags'], groups=4, kept_groups=2)

    def run(x, base, workspace, flags):
        out = base + 0
        native.adapter_out(x, c['a'], c['b'], c['scales'], c['ids'], None, out, workspace, flags, slices=c['slices'])
        w, i = torch.empty((20, 6), device=x.device), torch.empty((20, 6), dtype=torch.int32, device=x.device)
        native.route_experts(out, w, i, flags, groups=4, kept_groups=2)
        return out, w * 1, i
    torch._dynamo.reset()
    compiled = torch.compile(run, fullgraph=True, backend=backend, dynamic=False)
    off = torch.empty(3 + 20 * 256, dtype=torch.bfloat16, device=device)[3:].view(20, 256)      # (copied by the op)
    off.copy_(c['x'])
    for x in (c['x'], off):
        out, w, i = compiled(x, c['base'], b['workspace'], b['flags'])
        assert torch.equal(out, want) and torch.equal(w, weights) and torch.equal(i, ids)
    assert int(b['flags']) == 0


def test_rows_and_slots_past_32_bits(device):
    """base and out rows 2.4 GB apart, slots of A 3 GB and of B 2.6 GB apart."""
    import torch
    rng = np.random.default_rng(5)
    near = A._case(rng, 4, 200, 128, 16, 3, 1, 'bf16', 'bf16', device, True, ids=[2, 1, -1, 2])
    far = dict(near)
    for name, stride in (('a', 1_500_000_000), ('b', 1_300_000_000)):
        t = near[name]
        buf = torch.zeros(2 * stride + t[0].numel(), dtype=t.dtype, device=device)
        far[name] = buf.as_strided(t.shape, (stride, t.shape[2], 1))
        far[name].copy_(t)
    ld = 1_200_000_000
    for name in ('base', 'out'):
        buf = torch.zeros(3 * ld + 200, dtype=torch.bfloat16, device=device)
        far[name] = buf.as_strided((4, 200), (ld, 1))
    far['base'].copy_(near['base'])
    b = _buffers(near)
    _call(near, b)
    A._check(near, (b['out'], int(b['flags'])), exact=True)
    want = b['out']
    _call(far, b | dict(out=far['out']))
    assert torch.equal(far['out'], want) and int(b['flags']) == 0


@pytest.mark.parametrize('in_place', [False, True])
def test_more_rows_than_one_pass(device, in_place):
    import torch
    rng = np.random.default_rng(6)
    M, some = (1 << 20) + 1500, 500
    near = A._case(rng, some, 24, 16, 8, 3, 1, 'bf16', 'bf16', device, True)
    want, _ = A._run(near)
    times = -(-M // some)
    c = near | {n: near[n].repeat(times, 1)[:M] for n in ('x', 'base')} | dict(ids=near['ids'].repeat(times)[:M])
    out, flags = A._run(c, in_place=in_place)
    assert flags == 0 and torch.equal(out, want.repeat(times, 1)[:M])


def test_every_slot_of_the_largest_bank(device):
    rng = np.random.default_rng(7)
    for M in (200, 5000):
        ids = rng.permutation(4096)[np.arange(M) % 4096]
        c = A._case(rng, M, 40, 16, 8, 4096, 1, 'fp16', 'fp32', device, True, ids=ids)
        A._check(c, A._run(c), exact=True)
        A._check(c, A._run(c, in_place=True), exact=True)


def test_routing_rows_past_one_grid(device):
    """More rows than a grid of 64 threads a row can hold."""
    import torch
    from ornith_g256 import native
    M, some = (1 << 24) + 300, 1000
    near = torch.randn((some, 8), generator=torch.Generator(device=device).manual_seed(8), device=device)
    got = []
    for rows in (some, M):
        w, i = torch.empty((rows, 2), device=device), torch.empty((rows, 2), dtype=torch.int32, device=device)
        flags = torch.zeros(1, dtype=torch.int32, device=device)
        native.route_experts(near.repeat(-(-rows // some), 1)[:rows], w, i, flags)
        assert int(flags) == 0
        got.append((w, i))
    times = -(-M // some)
    assert all(torch.equal(b, a.repeat(times, 1)[:M]) for a, b in zip(*got))


def test_routing_rows_past_32_bits(device):
    import torch
    from ornith_g256 import native
    E, ld = 256, 1_500_000_000
    near = torch.randn((3, E), generator=torch.Generator(device=device).manual_seed(9), device=device).to(torch.bfloat16)
    far = torch.zeros(2 * ld + E, dtype=torch.bfloat16, device=device).as_strided((3, E), (ld, 1))
    far.copy_(near)
    got = []
    for z in (near, far):
        w, i = torch.empty((3, 8), device=device), torch.empty((3, 8), dtype=torch.int32, device=device)
        native.route_experts(z, w, i, torch.zeros(1, dtype=torch.int32, device=device), 'sigmoid', None, 8, 3, 2)
        got.append((w, i))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_routing_captured_and_streamed(device):
    import torch
    from ornith_g256 import native
    gen = torch.Generator(device=device).manual_seed(10)
    z = torch.randn((500, 257), generator=gen, device=device)[:, :256]
    w, i = torch.empty((500, 8), device=device), torch.empty((500, 8), dtype=torch.int32, device=device)
    flags, stream = torch.zeros(1, dtype=torch.int32, device=device), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        native.route_experts(z, w, i, flags)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            native.route_experts(z, w, i, flags, groups=8, kept_groups=4, group_top=2)
    for _ in range(3):
        z.copy_(torch.randn((500, 256), generator=gen, device=device))
        w2, i2 = torch.empty_like(w), torch.empty_like(i)
        native.route_experts(z, w2, i2, flags, groups=8, kept_groups=4, group_top=2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(w, w2) and torch.equal(i, i2)
