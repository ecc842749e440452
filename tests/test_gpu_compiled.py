"""Plain 4-bit linears and sampling inside a compiled function: the bits of the
plain calls."""
import numpy as np
import pytest

import test_gpu_decode_end as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('backend', ['eager', 'aot_eager'])
def test_compiled_step(device, backend):
    import torch
    from ornith_g256 import native
    rng = np.random.default_rng(1)
    banks, _ = D._head(rng, device)
    step = D.Step(banks, device)
    step.fill(rng)
    step.run()
    want = step.results()
    torch._dynamo.reset()

    def run(x, uniform, workspace, flags, settings):
        logits = torch.empty((x.shape[0], D.N), dtype=torch.float32, device=x.device)
        native.w4_out(x, *banks, logits, flags, D.N, D.K, D.GROUP)
        token = torch.empty(x.shape[0], dtype=torch.int64, device=x.device)
        logprob = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
        native.logits_sample(logits, uniform, workspace, token, flags, logprob=logprob, **settings)
        return logits, token, logprob
    compiled = torch.compile(run, fullgraph=True, backend=backend, dynamic=False)
    for lead in (0, 3):                                # (rows off the 16-byte grid: copied by the op)
        buf = torch.empty(lead + step.x.numel(), dtype=torch.bfloat16, device=device)
        x = buf[lead:].view(step.x.shape)
        x.copy_(step.x)
        got = [t.cpu() for t in compiled(x, step.uniform, step.workspace, step.flags, step.settings)]
        assert D._same(got, want)
    # settings that are off
    got = compiled(step.x, step.uniform, step.workspace, step.flags, dict(top_k=step.settings['top_k']))
    native.logits_sample(step.logits, step.uniform, step.workspace, step.token, step.flags, top_k=step.settings['top_k'],
                         logprob=step.logprob)
    assert D._same([t.cpu() for t in got[1:]], step.results()[1:]) and int(step.flags) == 0


def test_compiled_layer(device):
    import torch
    from ornith_g256 import methods
    import test_w4_layer_cpu as L
    rng = np.random.default_rng(2)
    layer = L._Layer(n=300, k=512, group=32).to(device)
    layer.load_packed('w4_codes', torch.from_numpy(rng.integers(0, 2 ** 32, (300, 64), dtype=np.uint32)))
    layer.load_packed('w4_scales', torch.from_numpy(rng.uniform(0.01, 0.02, (300, 16))).to(torch.bfloat16))
    layer.quant_method.process_weights_after_loading(layer)
    layer.quant_method.runtime = type('Runtime', (), dict(slots=(torch.zeros(1, dtype=torch.int32, device=device),)))
    layer.quant_method.slot = 0
    torch._dynamo.reset()
    compiled = torch.compile(lambda x: torch.relu(layer.quant_method.apply(layer, x)), fullgraph=True, backend='aot_eager')
    for shape in ((1, 512), (4, 7, 512)):
        x = torch.randn(shape, device=device).to(torch.bfloat16)
        assert torch.equal(compiled(x), torch.relu(layer.quant_method.apply(layer, x)))
    off = torch.randn(1 + 3 * 512, device=device).to(torch.bfloat16)[1:].view(3, 512)
    assert off.data_ptr() % 16 != 0
    want = layer.quant_method.apply(layer, off.clone())
    assert torch.equal(layer.quant_method.apply(layer, off), want) and torch.equal(compiled(off), torch.relu(want))


def test_compiled_without_optional_results(device):
    """No logprob and no settings: nothing optional among what the op writes."""
    import torch
    from ornith_g256 import native
    rng = np.random.default_rng(3)
    logits = torch.from_numpy(rng.standard_normal((3, 9000)).astype(np.float32)).to(device)
    uniform = torch.rand(3, device=device)
    flags = torch.zeros(1, dtype=torch.int32, device=device)
    workspace = torch.empty(native.logits_sample_bytes(3, 9000), dtype=torch.uint8, device=device)

    def run(logits, uniform, workspace, flags):
        token = torch.empty(logits.shape[0], dtype=torch.int64, device=logits.device)
        native.logits_sample(logits * 2, uniform, workspace, token, flags)
        return token + 1
    torch._dynamo.reset()
    for backend in ('eager', 'aot_eager'):
        compiled = torch.compile(run, fullgraph=True, backend=backend)
        assert torch.equal(compiled(logits, uniform, workspace, flags), run(logits, uniform, workspace, flags))
    assert int(flags) == 0
