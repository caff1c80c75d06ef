"""The serving example end to end against the resident batch-one engine.

Logits: the example rounds each GEMM's input and output to BF16 (relative error at most
2^-8, 2^-8 / sqrt(3) root mean square), the engine keeps FP32. A layer has six such places
one after another, and two layers with the head 13: independent errors come to
sqrt(13 * 2) * 2^-8 / sqrt(3) = 1.2 % of the logits' size in root mean square; four times
that is the bound. Of 151,936 logits the largest error is below 6 of its deviations."""
import importlib.util
import os
import sys

import pytest
import torch

import megakernel_b200 as mk

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
RMS = 4 * (26 / 3) ** 0.5 / 256


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_serving", os.path.join(ROOT, "examples", "paged_serving.py"))
    mod = importlib.util.module_from_spec(spec)
    sys.modules["paged_serving"] = mod  # (its dataclass looks its module up)
    spec.loader.exec_module(mod)
    return mod


def test_server_agrees_with_the_batch_one_engine(example, cuda_device):
    weights = example.random_weights(2, cuda_device)
    server = example.Server(*weights, pages=100, max_len=512, chunk=96)
    pool = sorted(server.free)
    g = torch.Generator().manual_seed(5)
    lengths = [1, 17, 64, 250, 33]  # the fourth comes in chunks, next to the others' decode
    requests = [server.add(torch.randint(0, example.VOCAB, (n,), generator=g).tolist(), 6) for n in lengths[:3]]
    steps = 0
    while server.step():
        steps += 1
        if steps == 2:
            requests += [server.add(torch.randint(0, example.VOCAB, (n,), generator=g).tolist(), 6) for n in lengths[3:]]
    assert [len(r.out) for r in requests] == [6] * 5 and sorted(server.free) == pool

    k = torch.zeros((2, 8, 512, 128), dtype=torch.bfloat16, device=cuda_device)
    eng = mk.DecodeEngine(*weights, k, torch.zeros_like(k))
    for r in requests:
        probe = example.Server(*weights, pages=100, max_len=512)
        again = probe.add(r.prompt, 1)
        probe.step()
        first = eng.prefill(torch.tensor(r.prompt, dtype=torch.int32, device=cuda_device))
        want, got = eng.logits.double().flatten(), probe.last_logits[0].double()
        size = want.pow(2).mean().sqrt()
        err = got - want
        assert float(err.pow(2).mean().sqrt()) <= RMS * float(size)
        assert float(err.abs().max()) <= 6 * RMS * float(size)
        assert again.out[0] == first or again.margins[0] <= 12 * RMS * float(size)
    eng.close()
    example.compare(weights, requests, 512, 12 * RMS * float(size))
