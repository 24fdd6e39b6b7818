"""A join's configuration whose tensors are given other memory, sizes or types after it was made: the calls take them as they
then are, or refuse them (no GPU: the library is stood in for, and shows the configuration that it was handed)."""
import ctypes

import pytest
import torch
from torch.overrides import TorchFunctionMode

import xsmoe


class OnDevice(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        if getattr(func, "__name__", "") == "get_device":
            return 0
        return func(*args, **(kwargs or {}))


@pytest.fixture
def handed(monkeypatch):
    """The configuration that the last call handed to the library: [norm_w, gate, ld_gate, next_w, scales ...]."""
    got = []

    class Lib:
        def xs_block_join(self, j, *a):
            c = xsmoe.BlockJoinCfg.from_address(j)
            got[:] = [getattr(c, n) for n, _ in c._fields_]
            return 0

        def xs_block_norm(self, *a):
            return 0

        def xs_moe_combine_join(self, j, parts, weights, k, *a):
            got[:] = [weights, k]
            return 0

    monkeypatch.setattr(xsmoe, "lib", lambda: Lib())
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    with OnDevice():
        yield got


T, N = 3, 64


def case(gate_kind="token"):
    gate = {"token": torch.ones(T), "channel": torch.ones(N), "value": torch.ones(T, 2 * N)[:, :N]}[gate_kind]
    v = dict(norm=True, norm_w=torch.ones(N), norm_eps=1e-5, gate=gate, gate_kind=gate_kind, branch_scale=0.5,
             residual_scale=0.25, next_w=torch.ones(N), next_eps=1e-4)
    return v, xsmoe.block_join_cfg(**v)


def join(cfg):
    return xsmoe.block_join(torch.ones(T, N), torch.ones(T, N), cfg, quant=True)


def fields(v):
    c = xsmoe.block_join_cfg(**v)
    return [getattr(c, n) for n, _ in c._fields_]


@pytest.mark.parametrize("which", ["norm_w", "gate", "next_w"])
@pytest.mark.parametrize("gate_kind", ["token", "channel", "value"])
def test_other_memory_is_taken(handed, gate_kind, which):
    v, cfg = case(gate_kind)
    join(cfg)
    assert handed == fields(v)
    was = list(handed)
    t, old = v[which], v[which].data      # (the old memory is kept: an address of it would be told)
    t.data = torch.full(t.shape, 2.0)     # the value gate's rows closer together, too
    join(cfg)
    assert handed == fields(v) and handed != was
    t.data = old
    join(cfg)
    assert handed == was


@pytest.mark.parametrize("which", ["norm_w", "gate", "next_w"])
@pytest.mark.parametrize("gate_kind", ["token", "channel", "value"])
def test_what_no_longer_fits_is_refused(handed, gate_kind, which):
    for spoil in (lambda t: torch.ones([n - 1 for n in t.shape]), lambda t: torch.ones(t.shape, dtype=torch.float16),
                  lambda t: torch.ones([2 * n for n in t.shape])[tuple(slice(None, None, 2) for _ in t.shape)]):
        v, cfg = case(gate_kind)
        v[which].data = spoil(v[which])
        with pytest.raises(xsmoe.XsError, match=which):
            join(cfg)
    if gate_kind == "value" and which == "gate":
        return
    v, cfg = case(gate_kind)
    v[which].resize_(v[which].numel() - 1)                # the same address
    with pytest.raises(xsmoe.XsError, match=which):
        join(cfg)
    v, cfg = case(gate_kind)
    v[which].untyped_storage().resize_(0)                 # an address of NULL would mean no weights
    assert "freed" in message(lambda: join(cfg))


def message(call):
    """What the call raises, in words (a failing test's report would read its freed tensors)."""
    try:
        call()
    except Exception as e:
        return str(e)
    return "nothing"


def test_freed_weights_are_refused(handed):
    w = torch.ones(N)
    w.untyped_storage().resize_(0)
    assert "w's memory has been freed" in message(lambda: xsmoe.block_norm(torch.ones(T, N), w))


def test_one_row_of_a_wider_buffers_weights(handed):
    """The stride of one row says nothing; that of two has to be k."""
    buffer, cfg = torch.ones(4, 6), xsmoe.block_join_cfg()
    for row in (0, 3):
        w = buffer[row:row + 1, 2:5]
        xsmoe.moe_combine_join(torch.ones(3, N), w, torch.ones(1, N), cfg)
        assert handed == [w.data_ptr(), 3]
    with pytest.raises(xsmoe.XsError, match="6 values apart"):
        xsmoe.moe_combine_join(torch.ones(6, N), buffer[:2, :3], torch.ones(2, N), cfg)


def test_one_tensor_in_two_places(handed):
    """Each place asks for its own size, whichever tensor stands there."""
    g = torch.ones(T)
    for v in (dict(gate=g, gate_kind="token", next_w=g), dict(gate=g, gate_kind="token", norm=True, norm_w=g)):
        with pytest.raises(xsmoe.XsError, match="_w is not 64"):
            join(xsmoe.block_join_cfg(**v))
    rows = torch.ones(T, N)
    with pytest.raises(xsmoe.XsError, match="next_w is not 64"):
        join(xsmoe.block_join_cfg(gate=rows, gate_kind="value", next_w=rows))
    w = torch.ones(N)
    join(xsmoe.block_join_cfg(gate=w, gate_kind="channel", next_w=w, norm=True, norm_w=w))
