"""Optimizers of several threads, whose steps are the same kernels with other amounts of shared memory (block sizes, window lengths): each steps as it does alone."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

# elements, m, quant_block_size, d_block_size, k_init
SETTINGS = [(400_000, 10, 64, None, 0.01), (30_000, 3, 64, 4096, 0.01), (90_000, 7, 128, 1024, 0.05), (200_001, 20, 64, 8192, 0.02)]


def _run(setting, dtype, use_fused, steps=12):
    from ista_daslab_optimizers_b200 import MicroAdam
    d, m, qbs, dbs, k = setting
    g = torch.Generator('cuda').manual_seed(d)
    p = torch.nn.Parameter(torch.randn(d, generator=g, device='cuda').to(dtype))
    opt = MicroAdam([p], m=m, lr=1e-2, quant_block_size=qbs, k_init=k, d_block_size=dbs, use_fused=use_fused)
    for _ in range(steps):
        p.grad = torch.randn(d, generator=g, device='cuda').to(dtype)
        opt.step()
    return p.detach().clone()


@pytest.mark.parametrize('use_fused', [True, False])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_steps_of_several_threads(dtype, use_fused):
    from ista_daslab_optimizers_b200 import _native as N
    want = [_run(s, dtype, use_fused) for s in SETTINGS]
    torch.cuda.synchronize()
    errors, got, start = [], {}, threading.Barrier(len(SETTINGS))

    def work(n):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(5):
                    got[n] = _run(SETTINGS[n], dtype, use_fused)
                torch.cuda.current_stream().synchronize()
        except Exception as e:                           # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in range(len(SETTINGS))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors[0]
    for n, w in enumerate(want):
        assert torch.equal(got[n], w)
    assert N.device_error() == 0
