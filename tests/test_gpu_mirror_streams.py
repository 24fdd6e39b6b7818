"""Calls of the Python mirror that are given a stream other than the current one: their results come from that stream's
memory, and are those of the same call on the current stream."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def calls(xm):
    g = torch.Generator().manual_seed(1)
    r = lambda *n: torch.randn(*n, generator=g).to(DEV)   # noqa: E731
    x, res, w = r(300, 512), r(300, 512), r(512)
    parts, weights = r(600, 512), torch.rand(300, 2, generator=g).to(DEV)
    q, s = xm.w8a8_quantize(x)
    m, ms = xm.w8a8_quantize(r(640, 512))
    cfg = xm.block_join_cfg(next_w=w)
    return {"norm": lambda st: xm.block_norm(x, w, quant=True, stream=st),
            "join": lambda st: xm.block_join(x, res, cfg, next_type=torch.bfloat16, quant=True, stream=st),
            "combine": lambda st: xm.moe_combine_join(parts, weights, res, cfg, next_type=torch.float32, stream=st)[:2],
            "quantize": lambda st: xm.w8a8_quantize(x, stream=st), "gemm": lambda st: (xm.w8a8_gemm(q, s, m, ms, stream=st),),
            "swiglu": lambda st: (xm.w8a8_swiglu(q, s, m, ms, m, ms, stream=st),),
            "q8_1": lambda st: (xm.quantize_q8_1_rows(x, stream=st),), "router": lambda st: xm.router_top10(x, 8, stream=st),
            "mmq": lambda st: (xm.iq_mmq_quantize(x, None, 512, 512, 300, False, stream=st),)}


@pytest.mark.parametrize("name", ["norm", "join", "combine", "quantize", "gemm", "swiglu", "q8_1", "router", "mmq"])
@pytest.mark.parametrize("raw", [False, True])
def test_results_on_another_stream(xm, name, raw):
    call = calls(xm)[name]
    want = [t.clone() for t in call(None)]
    side = torch.cuda.Stream()
    st = side.cuda_stream if raw else side
    busy = torch.randn(4096, 4096, device=DEV)
    torch.cuda.synchronize()
    # blocks of the results' sizes, dropped with writes to them still to come on the current stream
    for _ in range(4):
        busy = busy @ busy * 1e-2
    for t in want:
        torch.empty_like(t).fill_(3)
    got = call(st)
    at = [t.data_ptr() for t in got]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    sizes = [(t.shape, t.dtype) for t in got]
    del got, t, a
    # dropped, they are the side stream's to give again, not the current one's
    new = [torch.empty(s, dtype=d, device=DEV) for s, d in sizes]
    assert not {t.data_ptr() for t in new} & set(at)
    torch.cuda.synchronize()


def test_the_null_stream(xm):
    """The raw handle 0 on a side stream: the call runs on the default stream and has ended when it returns."""
    call = calls(xm)["join"]
    want = [t.clone() for t in call(None)]
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = call(0)
        host = [t.cpu() for t in got]
    for a, b in zip(host, want):
        assert torch.equal(a, b.cpu())
