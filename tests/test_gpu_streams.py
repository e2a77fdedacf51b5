"""Calls on a stream that is not the current one: what a call allocates or copies for
itself is that stream's."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def given_out(n):
    """Where the current stream's next allocation of n bytes lies."""
    return torch.empty(n, dtype=torch.uint8, device="cuda").data_ptr()


def test_workspaces_and_outputs_are_the_streams(qg, cuda):
    W = torch.randn((256, 512), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    X = torch.randn((40, 512), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(torch.bfloat16)
    p = qg.pack_mxfp4(W)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()

    def made(stream):
        yield qg.make_workspace(p, 40, stream=stream)
        yield qg.make_workspace(p, 40, stream)
        yield qg.make_grouped_workspace([p, p], 40, stream=stream)
        yield qg.make_tp_workspace(p, 40, stream=stream)
        yield qg.gemm_w4a16(p, X, stream=stream)
        yield qg.grouped_gemm_w4a16([p, p], X, [30, 10], stream=stream)
        yield qg.dequant(p, stream=stream)
        yield qg.pack_int4(W, 64, stream).data

    for t in made(s):
        at, n = t.data_ptr(), t.nbytes
        del t
        here = given_out(n)
        with torch.cuda.stream(s):
            there = given_out(n)
        assert there == at and here != at
        s.synchronize()


@pytest.mark.parametrize("M", [1, 40])
def test_a_call_on_another_stream_gives_the_same(qg, cuda, M):
    """Rows that need a copy first, no workspace, and the current stream taking memory of
    the workspace's size as soon as the call returns."""
    W = torch.randn((512, 1024), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    wide = torch.randn((M, 2048), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda").to(torch.bfloat16)
    p = qg.pack_nvfp4(W)
    want = qg.gemm_w4a16(p, wide[:, :1024])
    size = max(qg.workspace_size(p, M), 256)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert qg.nvfp4_tensor_scale(W, s) == p.tensor_scale
    for _ in range(20):
        got = qg.gemm_w4a16(p, wide[:, :1024], stream=s)
        taken = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(3)]
        s.synchronize()
        assert torch.equal(got, want)
        del taken
