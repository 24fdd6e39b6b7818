"""Where the Python mirror's new tensors are made when a call is given a stream (no GPU: the library, torch's streams and
the device are stood in for)."""
import contextlib
import inspect

import pytest
import torch
from torch.overrides import TorchFunctionMode

import xsmoe


class Side:
    """A torch stream that is not the current one."""
    cuda_stream, device_index = 4096, 0


class Factories(TorchFunctionMode):
    """Notes of each tensor that is made which stream was current; every tensor says that it is on device 0."""

    def __init__(self):
        super().__init__()
        self.current, self.made = None, []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        name = getattr(func, "__name__", "")
        if name == "get_device":
            return 0
        out = func(*args, **(kwargs or {}))
        if name in ("empty", "zeros", "new_empty", "new_zeros", "empty_strided"):
            self.made.append(self.current)
        return out


class Lib:
    """A library whose every call succeeds and is asked for 64 bytes of workspace."""

    def __getattr__(self, name):
        return lambda *a: 64 if name.endswith("bytes") else 0


f32, i8, i32 = (lambda *n: torch.ones(n)), (lambda *n: torch.ones(n, dtype=torch.int8)), (lambda *n: torch.ones(n, dtype=torch.int32))
LAYOUT = xsmoe.Layout(n_embd=32, n_ff=32)
CALLS = {   # every call that takes a stream and makes tensors: its arguments
    "quantize_rows": lambda: (xsmoe.Q8_0, f32(32)), "iq_dequant_f32": lambda: (xsmoe.Q8_0, i8(34), 32),
    "iq_dequant_bf16": lambda: (xsmoe.Q8_0, i8(34), 32), "iq_dequant_f16": lambda: (xsmoe.Q8_0, i8(34), 32),
    "quantize_q8_1_rows": lambda: (f32(2, 32),), "router_top10": lambda: (f32(2, 8), 2),
    "router_grouped_sigmoid": lambda: (f32(2, 8), None, 2, 1, 2, 1.0), "router_logits_f32": lambda: (f32(2, 8), f32(4, 8)),
    "prefill_route": lambda: (i32(4), 2, 8, None, 0, True), "f32_gemv_fp32_mmvf_multi": lambda: (f32(2, 8), f32(4, 8)),
    "f32_gemm_rows": lambda: (f32(2, 8), f32(4, 8)), "f32_to_bf16_bulk": lambda: (f32(8),),
    "bf16_gemv": lambda: (i32(8), i32(4, 8)), "project_bf16": lambda: (f32(8), i32(4, 8)),
    "iq_mmq_quantize": lambda: (f32(2, 32), None, 32, 32, 2, False),
    "iq_mmq_quantize_scatter": lambda: (f32(2, 32), i32(4), 32, 32, 2, 2, False),
    "mmq_swiglu": lambda: (f32(2, 8), 2, 4, True), "mmq_iota": lambda: (4, None, "cpu"),
    "shared_expert_decode": lambda: (LAYOUT, i8(64), f32(2, 32), f32(32)),
    "block_norm": lambda: (f32(2, 24), None, 1e-6, torch.float32, True),
    "block_join": lambda: (f32(2, 24), f32(2, 24), xsmoe.block_join_cfg(), None, torch.float32, True),
    "moe_combine_join": lambda: (f32(4, 24), f32(2, 2), f32(2, 40)[:, :24], xsmoe.block_join_cfg(), None, None, None,
                                 torch.float32, True),
    "w8a8_quantize": lambda: (f32(2, 24),), "w8a8_gemm": lambda: (i8(2, 32), f32(2), i8(4, 32), f32(4)),
    "w8a8_swiglu": lambda: (i8(2, 32), f32(2), i8(4, 32), f32(4), i8(4, 32), f32(4)),
}
NOTHING_MADE = {"resident_plan", "native_expert_grouped", "native_expert_gate_up", "native_expert_down", "moe_prefill_experts",
                "iq_mmq_grouped", "native_moe_combine_multi", "native_moe_combine_multi_hits", "moe_combine_residual",
                "moe_layer_decode_noalloc", "noalloc_status_check", "wait_flag_ge", "copy_i32_from_mapped",
                "copy_rows_from_mapped", "fetch_blobs", "rebase_ptrs", "moe_hit_add"}


def test_every_call_with_a_stream_is_listed():
    takes = {n for n, f in vars(xsmoe).items() if inspect.isfunction(f) and not n.startswith("_") and
             "stream" in inspect.signature(f).parameters}
    assert takes == set(CALLS) | NOTHING_MADE


@pytest.mark.parametrize("stream", [Side(), 4096, 0, xsmoe.STREAM_LEGACY, None], ids=["torch", "raw", "null", "legacy", "none"])
@pytest.mark.parametrize("name", CALLS)
def test_new_tensors_are_made_on_the_calls_stream(monkeypatch, name, stream):
    args = CALLS[name]()
    mode = Factories()

    @contextlib.contextmanager
    def made_current(s):
        before, mode.current = mode.current, s
        yield
        mode.current = before

    monkeypatch.setattr(torch.cuda, "stream", made_current)
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda h, device=None: ("raw", h))
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: "default")
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    monkeypatch.setattr(xsmoe, "lib", lambda: Lib())
    with mode:
        getattr(xsmoe, name)(*args, stream=stream)
    want = {4096: ("raw", 4096), 0: "default", 1: "default"}.get(stream, stream) if not isinstance(stream, Side) else stream
    assert mode.made and all(m == want for m in mode.made), mode.made


def test_a_stream_of_another_device_is_refused(monkeypatch):
    class Other(Side):
        device_index = 1

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    with pytest.raises(xsmoe.XsError, match="a stream of cuda:1 for tensors on cuda:0"):
        xsmoe._launch(lambda *a: 0, 0, Other(), ())
