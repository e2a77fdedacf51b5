"""The serving operators together, as examples/serve_decode.py uses them."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ex():
    spec = importlib.util.spec_from_file_location("serve_decode", os.path.join(ROOT, "examples", "serve_decode.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def small(ex):
    return ex.Decoder(ex.Config(layers=2, width=512, q_heads=8, heads=2, head_dim=64, inner=1024, vocab=300, block=16))


@pytest.mark.parametrize("kv", [0, 1])
def test_chunks_and_steps_give_the_logits_of_one_pass(qg, cuda, ex, kv):
    """One request fed whole, in chunks and token by token: the last logits agree
    to the cache's precision (a block's scale may grow in other steps, so codes
    can differ by a rounding; E4M3's step is 2^-4 of a value, INT8's 2^-7 of the
    largest) and the plans' lengths and blocks are the same."""
    model = small(ex)
    tokens = torch.randint(0, 300, (150,), generator=torch.Generator().manual_seed(3)).tolist()
    got = []
    for sizes in ([150], [70, 64, 16], [100] + [1] * 50):
        server = ex.Server(model, 3, 200, 40, kv)
        at = 0
        for n in sizes:
            plan, logits = server.step({1: tokens[at:at + n]})
            at += n
        assert plan.lens.tolist() == [0, 150, 0] and int(plan.counts[0]) == 40 - 10 and int(plan.counts[3]) == 0
        got.append(logits[-1].float())
    for other in got[1:]:
        assert float((other - got[0]).norm() / got[0].norm()) < 0.1


def test_requests_come_and_go(qg, cuda, ex):
    """More requests than places, and blocks that are reused: every request gets the
    tokens it gets alone."""
    model = small(ex)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 300, (n,), generator=g).tolist() for n in (5, 40, 17, 90, 33, 1)]
    together = ex.serve(model, prompts, 6, qg.KV_E4M3, places=3, chunk=32)
    assert [len(t) for t in together] == [6] * 6
    alone = [ex.serve(model, [p], 6, qg.KV_E4M3, places=1, chunk=32)[0] for p in prompts]
    # the products' kernels depend on the rows of a step, so a near tie may fall either way
    assert sum(a == b for a, b in zip(together, alone)) >= 4
