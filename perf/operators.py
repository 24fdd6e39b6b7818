"""What stands around and beside the MoE layer, as timed cases: the norm before a block, the join after one (with its
gate, its scales and the next block's norm), the same join over the MoE layer's parts, the 8-bit product with a scale a
token and a scale an output, and the gated pair of such products.

  do        what
  norm      x [tokens, hidden] -> RMS norm times its weights, as rows of `y` and, with quant, as int8 codes a token's scale
  join      a block's output y and the residual -> the new residual, and the next block's norm of it
  combine   the same, the block's output being the weighted sum of a token's k expert rows and a shared row
  product   rows of x (float rows quantized in the call, or int8 codes) times int8 weights [n_out, n_in]
  gated     SwiGLU of two such products over int8 codes

Hidden sizes and expert widths are those of perf/cases.py's layers, or generic.  run() gives the operators' plain form in
torch or, where `own` is true, the library's calls.  int8 codes are returned as the values they stand for.
"""
import math
import pathlib
import sys

import torch

own = False

DEV = "cuda"
FLOAT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "none": 0}
EPS = 1e-6
TINY = 2.0 ** -126   # the smallest scale: codes of smaller rows count in it


# ---------------------------------------------------------------------------------------------------- the cases

def _norm(name, tokens, hidden, x="f32", y="none", quant=True):
    return dict(name=name, do="norm", tokens=tokens, hidden=hidden, x=x, y=y, quant=quant)


def _join(name, tokens, hidden, y="f32", r="f32", norm=False, gate="none", next="none", quant=False, k=0, shared="none"):
    """norm: the block's output is normed first.  gate: none, token (a sigmoid), channel or value (multipliers).  next: the
    type of the next block's normed rows, quant: that norm as int8 codes too.  k: of so many expert rows a token, with a
    shared row (none, plain or gated)."""
    return dict(name=name, do="combine" if k else "join", tokens=tokens, hidden=hidden, y=y, r=r, norm=norm, gate=gate,
                next=next, quant=quant, k=k, shared=shared)


def _product(name, tokens, n_in, n_out, x="q8", y="f32"):
    return dict(name=name, do="product", tokens=tokens, n_in=n_in, n_out=n_out, x=x, y=y)


def _gated(name, tokens, n_in, n_ff, y="bf16"):
    return dict(name=name, do="gated", tokens=tokens, n_in=n_in, n_ff=n_ff, y=y)


def listed():
    return [
        # generating one sequence: the norm before a block, straight to the codes its products read; launch latency
        _norm("norm_2048_1", 1, 2048),
        # a long prompt chunk: the residual's rows normed for 16-bit products; bandwidth
        _norm("norm_7168_4096", 4096, 7168, y="bf16", quant=False),
        # checking a few draft tokens: a normed and gated block joins, the next block's codes come with it
        _join("join_4096_7", 7, 4096, norm=True, gate="token", quant=True),
        # a prompt of odd length, 16-bit residual, a multiplier a channel, the next block's rows
        _join("join_5120_1531", 1531, 5120, y="bf16", r="bf16", norm=True, gate="channel", next="bf16"),
        # a few tokens after the MoE layer: parts and a gated shared row to the next block's codes
        _join("combine_2048_5", 5, 2048, quant=True, k=8, shared="gated"),
        # a prompt chunk after the widest MoE layer
        _join("combine_7168_1024", 1024, 7168, norm=True, next="bf16", k=8, shared="plain"),
        # one token through a dense projection: the weights out of memory
        _product("product_4096_1", 1, 4096, 4096),
        # a small batch, odd sizes, quantized in the call
        _product("product_7168_37", 37, 7168, 2050, x="bf16", y="bf16"),
        # a long prompt chunk through a wide projection: the matrix cores
        _product("product_7168_4096", 4096, 7168, 8192, x="f32", y="bf16"),
        # one token through a dense block's gate and up rows
        _gated("gated_4096_1", 1, 4096, 8192, y="f32"),
        # a serving batch through a shared expert's gate and up rows
        _gated("gated_2048_77", 77, 2048, 1536),
        # a prompt chunk through the widest dense block: the largest
        _gated("gated_7168_2048", 2048, 7168, 16384),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A size of the range: most are whole numbers of 128s, as models have them, the others anything."""
    n = _log_int(rng, lo, hi)
    return max(128, n // 128 * 128) if rng.random() < 0.6 else n


def draw(rng):
    do = rng.choice(("norm", "join", "combine", "product", "product", "gated"))
    real = ("f32", "bf16", "f16")
    if do in ("norm", "join", "combine"):
        hidden = _width(rng, 128, 8192)
        tokens = _log_int(rng, 1, 4096 if do != "combine" else 1024)
        nxt, quant = rng.choice((("none", True), ("f32", False), ("bf16", False), ("bf16", True), ("none", False)))
        if do == "norm":
            case = _norm("", tokens, hidden, rng.choice(real), nxt, quant or nxt == "none")
        else:
            case = _join("", tokens, hidden, "f32" if do == "combine" else rng.choice(real), rng.choice(real),
                         rng.random() < 0.5, rng.choice(("none", "token", "channel", "value")), nxt, quant,
                         rng.randint(1, 8) if do == "combine" else 0,
                         rng.choice(("none", "plain", "gated")) if do == "combine" else "none")
    else:
        n_in, n_out = _width(rng, 256, 8192), _width(rng, 256, 8192)
        tokens = _log_int(rng, 1, 4096 if do == "product" else 3500)
        y = rng.choice(real)
        case = _product("", tokens, n_in, n_out, rng.choice(("q8",) + real), y) if do == "product" else \
            _gated("", tokens, n_in, n_out, y)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------- inputs

class State:
    """What the caller holds before the call."""


def _rows(g, rows, cols, std=1.0):
    """Activations: normal values on channels of unequal size, a few of them ten times the rest."""
    size = torch.exp(0.5 * torch.randn(cols, generator=g, device=DEV))
    size = torch.where(torch.rand(cols, generator=g, device=DEV) < 0.003, 10 * size, size)
    return torch.randn(rows, cols, generator=g, device=DEV) * (size * std)


def _codes(x):
    """Rows -> int8 codes in rows of a whole number of 16 bytes (a view of the first columns), and their scales."""
    rows, cols = x.shape
    scale = (x.abs().amax(1) / 127).clamp_min(TINY)
    q = torch.zeros(rows, (cols + 15) // 16 * 16, dtype=torch.int8, device=x.device)
    q[:, :cols] = (x.double() / scale.double()[:, None]).round().to(torch.int8)
    return q[:, :cols], scale


def _weights(g, rows, cols):
    return _codes(torch.randn(rows, cols, generator=g, device=DEV) / math.sqrt(cols))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = State()
    s.case = case
    T = case["tokens"]
    if case["do"] in ("product", "gated"):
        x = _rows(g, T, case["n_in"])
        if case["do"] == "gated" or case["x"] == "q8":
            s.q, s.scale = _codes(x)
        else:
            s.x = x.to(FLOAT[case["x"]])
        if case["do"] == "product":
            s.w, s.w_scale = _weights(g, case["n_out"], case["n_in"])
        else:
            s.gate, s.gate_scale = _weights(g, case["n_ff"], case["n_in"])
            s.up, s.up_scale = _weights(g, case["n_ff"], case["n_in"])
        return s
    H = case["hidden"]
    if case["do"] == "norm":
        s.x = _rows(g, T, H).to(FLOAT[case["x"]])
        s.w = 1 + 0.2 * torch.randn(H, generator=g, device=DEV)
        return s
    s.residual = _rows(g, T, H, 4.0).to(FLOAT[case["r"]])
    s.norm_w = 1 + 0.2 * torch.randn(H, generator=g, device=DEV) if case["norm"] else None
    s.next_w = 1 + 0.2 * torch.randn(H, generator=g, device=DEV) if case["next"] != "none" or case["quant"] else None
    shape = dict(none=None, token=(T,), channel=(H,), value=(T, H))[case["gate"]]
    s.gate = torch.randn(shape, generator=g, device=DEV) if shape else None
    s.branch_scale, s.residual_scale = 0.75, 0.9375
    s.shared = s.shared_gate = None
    if case["do"] == "join":
        s.y = _rows(g, T, H).to(FLOAT[case["y"]])
    else:
        s.parts = _rows(g, T * case["k"], H)
        s.weights = torch.rand(T, case["k"], generator=g, device=DEV) + 0.1
        s.weights = s.weights / s.weights.sum(1, keepdim=True)
        if case["shared"] != "none":
            s.shared = _rows(g, T, H)
        if case["shared"] == "gated":
            s.shared_gate = torch.randn(T, generator=g, device=DEV)
    # a token's or a value's gate is computed for the call, its configuration made with it; what holds only weights is kept
    s.join = _join_cfg(s) if own and case["gate"] in ("none", "channel") else None
    return s


def _join_cfg(s):
    c = s.case
    return _library().block_join_cfg(norm=c["norm"], norm_w=s.norm_w, norm_eps=EPS, gate=s.gate, gate_kind=c["gate"],
                                     branch_scale=s.branch_scale, residual_scale=s.residual_scale, next_w=s.next_w,
                                     next_eps=EPS)


def _library():
    """The library's Python mirror, imported once."""
    if "xsmoe" not in sys.modules:
        sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent / "xestrata-win_amd"))
        import xsmoe  # noqa: F401
    return sys.modules["xsmoe"]


# ---------------------------------------------------------------------------------------------------- one pass

def _out(**v):
    return {k: x for k, x in v.items() if x is not None}


def _values(q, scale):
    return None if q is None else q * scale[:, None]


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    xm, c = _library(), s.case
    if c["do"] == "norm":
        y, q, scale = xm.block_norm(s.x, s.w, EPS, out_type=FLOAT.get(c["y"]), quant=c["quant"])
        return _out(y=y, values=_values(q, scale), scale=scale)
    if c["do"] in ("join", "combine"):
        want = dict(next_type=FLOAT.get(c["next"]), quant=c["quant"])
        cfg = s.join or _join_cfg(s)
        if c["do"] == "join":
            out, nxt, q, scale = xm.block_join(s.y, s.residual, cfg, **want)
        else:
            out, nxt, q, scale = xm.moe_combine_join(s.parts, s.weights, s.residual, cfg, shared=s.shared,
                                                     shared_gate=s.shared_gate, **want)
        return _out(out=out, next=nxt, values=_values(q, scale), scale=scale)
    if c["do"] == "product":
        q, scale = (s.q, s.scale) if c["x"] == "q8" else xm.w8a8_quantize(s.x)
        return dict(y=xm.w8a8_gemm(q, scale, s.w, s.w_scale, out_type=FLOAT[c["y"]]))
    return dict(h=xm.w8a8_swiglu(s.q, s.scale, s.gate, s.gate_scale, s.up, s.up_scale, out_type=FLOAT[c["y"]]))


def _plain_norm(x, w):
    """x in fp32.  The squares' sum in 64 bits, the factor rounded once, the two products in fp32."""
    ss = x.double().square().sum(1, keepdim=True)
    r = (1 / (ss / x.shape[1] + EPS).sqrt()).float()
    return x * r * w


def _plain_quantize(x):
    scale = (x.abs().amax(1) / 127).clamp_min(TINY)
    return (x.double() / scale.double()[:, None]).round().to(torch.int8), scale   # (64 bits: values next to a border)


def _sigmoid(z):
    return (1 / (1 + (-z.double()).exp())).float()


def _plain_product(q, scale, w, w_scale):
    return (q.float() @ w.float().T) * scale[:, None] * w_scale


def _run_plain(s):
    c = s.case
    if c["do"] == "norm":
        y = _plain_norm(s.x.float(), s.w)
        q, scale = _plain_quantize(y) if c["quant"] else (None, None)
        return _out(y=y.to(FLOAT[c["y"]]) if c["y"] != "none" else None, values=_values(q, scale), scale=scale)
    if c["do"] in ("join", "combine"):
        if c["do"] == "join":
            b = s.y.float()
        else:
            T, k = s.weights.shape
            p = s.parts.view(T, k, -1) * s.weights[:, :, None]
            b = p[:, 0]
            for j in range(1, k):   # in rank order
                b = b + p[:, j]
            if s.shared is not None:
                b = b + (s.shared * _sigmoid(s.shared_gate)[:, None] if s.shared_gate is not None else s.shared)
        if c["norm"]:
            b = _plain_norm(b, s.norm_w)
        if c["gate"] != "none":
            b = b * (_sigmoid(s.gate)[:, None] if c["gate"] == "token" else s.gate)
        out = (s.residual.float() * s.residual_scale + b * s.branch_scale).to(FLOAT[c["r"]])
        nxt = q = scale = None
        if s.next_w is not None:
            y = _plain_norm(out.float(), s.next_w)
            nxt = y.to(FLOAT[c["next"]]) if c["next"] != "none" else None
            q, scale = _plain_quantize(y) if c["quant"] else (None, None)
        return _out(out=out, next=nxt, values=_values(q, scale), scale=scale)
    if c["do"] == "product":
        q, scale = (s.q, s.scale) if c["x"] == "q8" else _plain_quantize(s.x.float())
        return dict(y=_plain_product(q, scale, s.w, s.w_scale).to(FLOAT[c["y"]]))
    g = _plain_product(s.q, s.scale, s.gate, s.gate_scale)
    u = _plain_product(s.q, s.scale, s.up, s.up_scale)
    return dict(h=(g / (1 + (-g).exp()) * u).to(FLOAT[c["y"]]))


# ---------------------------------------------------------------------------------------------------- accounting

def work(case):
    T = case["tokens"]
    if case["do"] in ("product", "gated"):
        K = case["n_in"]
        N, rows = (case["n_out"], case["n_out"]) if case["do"] == "product" else (case["n_ff"], 2 * case["n_ff"])
        x = SIZE[case["x"]] if case.get("x", "q8") != "q8" else 1
        return dict(bytes=float(T * K * x + rows * K + 4 * rows + T * N * SIZE[case["y"]]), flops=2.0 * T * rows * K)
    H = case["hidden"]
    if case["do"] == "norm":
        return dict(bytes=float(T * H * (SIZE[case["x"]] + SIZE[case["y"]] + case["quant"]) + 4 * H), flops=4.0 * T * H)
    value = 2 * SIZE[case["r"]] + SIZE[case["next"]] + case["quant"] + 4 * (case["gate"] == "value")
    value += SIZE[case["y"]] if case["do"] == "join" else 4 * case["k"] + 4 * (case["shared"] != "none")
    return dict(bytes=float(T * H * value), flops=T * H * (10.0 + 2 * case["k"]))


# ---------------------------------------------------------------------------------------------------- in 64 bits

def _f32(v):
    """One of the roundings to fp32 that the definition names, kept in 64 bits."""
    return v.to(torch.float32).to(torch.float64)


def _norm64(x, w):
    factor = _f32((x.pow(2).mean(dim=-1) + EPS).rsqrt())
    return _f32(_f32(x * factor.unsqueeze(-1)) * w.to(torch.float64))


def _quant64(y):
    """(the codes' values, their scales)"""
    step = torch.maximum(_f32(y.abs().max(dim=-1).values / 127.0), torch.full((), TINY, dtype=torch.float64, device=DEV))
    return torch.round(y / step.unsqueeze(-1)) * step.unsqueeze(-1), step


def exact(case, seed):
    s = prepare(case, seed)
    if case["do"] == "norm":
        y = _norm64(s.x.to(torch.float64), s.w)
        values, step = _quant64(y) if case["quant"] else (None, None)
        return _out(y=y if case["y"] != "none" else None, values=values, scale=step)
    if case["do"] in ("join", "combine"):
        if case["do"] == "join":
            block = s.y.to(torch.float64)
        else:
            T, k = s.weights.shape
            parts = s.parts.to(torch.float64).reshape(T, k, -1)
            block = torch.zeros_like(parts[:, 0])
            for j in range(k):
                block = _f32(block + _f32(parts[:, j] * s.weights[:, j:j + 1].to(torch.float64)))
            if s.shared is not None:
                row = s.shared.to(torch.float64)
                if s.shared_gate is not None:
                    row = _f32(row * _f32(torch.sigmoid(s.shared_gate.to(torch.float64))).unsqueeze(1))
                block = _f32(block + row)
        if case["norm"]:
            block = _norm64(block, s.norm_w)
        if case["gate"] != "none":
            gate = s.gate.to(torch.float64)
            block = _f32(block * (_f32(torch.sigmoid(gate)).unsqueeze(1) if case["gate"] == "token" else gate))
        total = _f32(_f32(s.residual.to(torch.float64) * s.residual_scale) + _f32(block * s.branch_scale))
        y = values = step = None
        if s.next_w is not None:
            y = _norm64(total.to(FLOAT[case["r"]]).to(torch.float64), s.next_w)   # of the residual as it is stored
            values, step = _quant64(y) if case["quant"] else (None, None)
        return _out(out=total, next=y if case["next"] != "none" else None, values=values, scale=step)
    if case["do"] == "product":
        if case["x"] == "q8":
            x = s.q.to(torch.float64) * s.scale.to(torch.float64).unsqueeze(1)
        else:
            x, _ = _quant64(s.x.to(torch.float64))
        return dict(y=x @ (s.w.to(torch.float64) * s.w_scale.to(torch.float64).unsqueeze(1)).T)
    x = s.q.to(torch.float64) * s.scale.to(torch.float64).unsqueeze(1)
    gate = x @ (s.gate.to(torch.float64) * s.gate_scale.to(torch.float64).unsqueeze(1)).T
    up = x @ (s.up.to(torch.float64) * s.up_scale.to(torch.float64).unsqueeze(1)).T
    return dict(h=torch.nn.functional.silu(gate) * up)
