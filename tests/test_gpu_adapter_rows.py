"""A plain 4-bit head with adapters on gathered rows of a step, each with the slot
of its own row, captured and replayed with other rows and requests."""
import numpy as np
import pytest

import test_gpu_adapter as A
import test_gpu_adapter_layers as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('rows,gathered', [(40, 7), (9, 9), (300, 60)])
def test_a_head_on_gathered_rows(device, rows, gathered):
    import torch
    from ornith_g256 import methods, native
    rng = np.random.default_rng(rows)
    model = torch.nn.Module()
    model.head = L._w4_layer(rng, device, 1000, 512, 'head')
    model.head.quant_method.out_dtype = torch.float32
    ad = methods.attach_adapters(model.head, 4, 8)
    for slot in range(4):
        ad.load(slot, torch.from_numpy((rng.standard_normal((8, 512)) / 16).astype(np.float32)).to(torch.bfloat16),
                torch.from_numpy(rng.standard_normal((1000, 8)).astype(np.float32)).to(torch.bfloat16), 0.5 + slot)
    native.reset_binding()
    try:
        rt = methods.Runtime(model, {}, 512, device)
        x = torch.randn((rows, 512), device=device).to(torch.bfloat16)
        at = torch.zeros(gathered, dtype=torch.int64, device=device)

        def step():
            return model.head.quant_method.apply(model.head, x[at], adapter_ids=rt.adapter_ids[at])
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            step()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = step()
        for r in range(3):
            ids = torch.from_numpy(rng.integers(-1, 4, rows).astype(np.int32)).to(device)
            rt.set_adapter_ids(ids)
            at.copy_(torch.from_numpy(np.sort(rng.choice(rows, gathered, replace=False))))
            with pytest.raises(ValueError, match='adapter_ids'):
                model.head.quant_method.apply(model.head, x[at])
            none = torch.full((gathered,), -1, dtype=torch.int32, device=device)
            base = model.head.quant_method.apply(model.head, x[at], adapter_ids=none)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            c = dict(x=x[at], a=ad.a, b=ad.b, scales=ad.scales, ids=ids[at], base=base, slices=ad.slices, rank=8, dtype='bf16',
                     out_type='fp32')
            A._check(c, (out, 0))
        assert rt.check_error_flags() == [0]
    finally:
        native.reset_binding()
