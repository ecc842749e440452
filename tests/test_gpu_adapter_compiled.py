"""Layers with adapters inside a compiled function, against the same layers outside."""
import numpy as np
import pytest

import test_gpu_adapter_layers as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
def test_compiled_layers(device, backend):
    import torch
    from ornith_g256 import methods, native
    rng = np.random.default_rng(11)
    model = torch.nn.Module()
    model.first = L._w4_layer(rng, device, 2048, 1024, 'first')
    model.second = L._g256_layer(rng, device, 2048, 2048, 'second')
    model.head = L._w4_layer(rng, device, 700, 2048, 'head')
    model.head.quant_method.out_dtype = torch.float32
    for layer, slices in ((model.first, None), (model.second, (1500, 548)), (model.head, None)):
        ad = methods.attach_adapters(layer, 4, 16, slices)
        for slot in range(3):
            a = [torch.from_numpy((rng.standard_normal((16, ad.k)) / np.sqrt(ad.k)).astype(np.float32)).to(torch.bfloat16)
                 for _ in ad.slices]
            ad.load(slot, a, torch.from_numpy((rng.standard_normal((ad.n, 16)) * 0.3).astype(np.float32)).to(torch.bfloat16), 0.5 + slot)
    native.reset_binding()
    try:
        rt = methods.Runtime(model, {}, 512, device)

        def step(x, last):
            h = model.first.quant_method.apply(model.first, x)
            h = model.second.quant_method.apply(model.second, h)
            return h * 1, model.head.quant_method.apply(model.head, h[last], adapter_ids=rt.adapter_ids[last])
        torch._dynamo.reset()
        compiled = torch.compile(step, fullgraph=True, backend=backend, dynamic=False)
        for rows in (1, 24, 300):
            x = torch.randn((rows, 1024), device=device).to(torch.bfloat16)
            last = torch.arange(0, rows, 3, device=device)
            for r in range(2):
                ids = torch.from_numpy(rng.integers(-1, 4, rows).astype(np.int32)).to(device)
                rt.set_adapter_ids(ids)
                want = step(x, last)
                got = compiled(x, last)
                assert all(torch.equal(g, w) for g, w in zip(got, want)), (rows, r)
        assert rt.check_error_flags() == [0, 0, 0]
    finally:
        native.reset_binding()
