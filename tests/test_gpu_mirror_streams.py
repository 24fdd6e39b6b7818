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


def test_threads_share_a_configuration(xm):
    """Four threads, each on a stream of its own, with one configuration and rows of their own."""
    import threading
    w = torch.rand(512, device=DEV)
    cfg = xm.block_join_cfg(norm=True, norm_w=w, gate=w, gate_kind="channel", next_w=w)
    sets = [(torch.randn(T, 512, device=DEV), torch.randn(T, 512, device=DEV)) for T in (1, 40, 300, 700)]
    want = [xm.block_join(y, r, cfg, next_type=torch.float32, quant=True) for y, r in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        for n in range(20):
            got = xm.block_join(*sets[i], cfg, next_type=torch.float32, quant=True, stream=stream if n % 2 else stream.cuda_stream)
            stream.synchronize()
            bad.extend(i for a, b in zip(got, want[i]) if not torch.equal(a, b))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("given", ["none", "side", "default"])
def test_no_rows(xm, given):
    st = {"none": None, "side": torch.cuda.Stream(), "default": torch.cuda.default_stream()}[given]
    x, w = torch.empty(0, 64, device=DEV), torch.rand(64, device=DEV)
    for gate, kind in ((None, "none"), (torch.empty(0, device=DEV), "token"), (w, "channel"), (x, "value")):
        cfg = xm.block_join_cfg(norm=True, norm_w=w, gate=gate, gate_kind=kind, next_w=w)
        for r in (xm.block_join(x, x, cfg, next_type=torch.float32, quant=True, stream=st),
                  xm.moe_combine_join(x, torch.empty(0, 8, device=DEV), x, cfg, next_type=torch.float32, quant=True, stream=st)):
            assert [list(t.shape) for t in r] == [[0, 64], [0, 64], [0, 64], [0]]
    y, q, s = xm.block_norm(x, w, quant=True, stream=st)
    assert y.shape == q.shape == x.shape and s.shape == (0,)
    q, s = xm.w8a8_quantize(x, stream=st)
    m, ms = xm.w8a8_quantize(torch.rand(24, 64, device=DEV))
    assert xm.w8a8_gemm(q, s, m, ms, stream=st).shape == (0, 24)
    assert xm.w8a8_swiglu(q, s, m, ms, m, ms, stream=st).shape == (0, 24)


def test_a_configuration_made_in_a_graph(xm):
    """A token gate computed in the captured work, its configuration made there: each replay takes that replay's gate."""
    T, n = 9, 512
    y, r, w, z = torch.randn(T, n, device=DEV), torch.randn(T, n, device=DEV), torch.rand(n, device=DEV), torch.randn(T, device=DEV)

    def step():
        cfg = xm.block_join_cfg(gate=z * 2, gate_kind="token", next_w=w)
        return xm.block_join(y, r, cfg, next_type=torch.float32, quant=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        z.copy_(torch.randn(T, generator=torch.Generator().manual_seed(i)))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
