"""The operators of a linear layer in 8-bit floating point, as cases that can be timed and compared.

  norm      root-mean-square norm of x (+ residual), result in the input's type or in e4m3 with a scale for each 128 columns
  gated     act(gate) * up on the two halves of one matrix, result as above
  quantize  a matrix to e4m3 with a scale for each row's 128 columns (activations) or each 128 x 128 block (weights)
  matmul    C = A * B^T on e4m3 operands with those scales, optional bias and ReLU

A block of 8-bit values: s = max(largest finite |y|, 2^-100) / 448, q = y / s rounded to e4m3; what is not finite becomes NaN.

`own` false: the operators from elementary torch operations in 32 bits.  `own` true: the library's entry points.
"""
import math

import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
CODE = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 3}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
ACT = {"none": 0, "relu": 1, "hard_sigmoid": 2, "hard_swish": 3, "sigmoid": 4, "silu": 5}
BLOCK, TOP, LEAST, EPS = 128, 448.0, 2.0 ** -100, 1e-6


# --------------------------------------------------------------------------------------------------------------------
# the cases
# --------------------------------------------------------------------------------------------------------------------
def _norm(m, k, dtype, out, residual, pad=0, name=None):
    """pad: elements between the rows of x beyond K (a slice of a wider matrix)."""
    return _named(dict(op="norm", m=m, k=k, dtype=dtype, out=out, residual=residual, pad=pad), name)


def _gated(m, k, dtype, out, act, name=None):
    return _named(dict(op="gated", m=m, k=k, dtype=dtype, out=out, act=act), name)


def _quantize(m, k, dtype, rows, name=None):
    return _named(dict(op="quantize", m=m, k=k, dtype=dtype, rows=rows), name)


def _matmul(m, n, k, c, epilogue=False, name=None):
    return _named(dict(op="matmul", m=m, n=n, k=k, c=c, epilogue=epilogue), name)


def _named(case, name):
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token of a decoder: a single row, where the call's latency is all there is
        _norm(1, 4096, "f16", "f16", True, name="norm f16 1x4096 residual"),
        # the tokens of a long prompt or a batch of image patches, ready for the 8-bit product
        _norm(4096, 4096, "bf16", "e4m3", True, name="norm bf16 4096x4096 to e4m3"),
        # fp32 features whose width is no multiple of a block, cut from a wider matrix
        _norm(777, 1000, "f32", "e4m3", False, pad=24, name="norm f32 777x1000 to e4m3"),
        # gate and up projections of a long prompt
        _gated(2048, 8192, "bf16", "e4m3", "silu", name="gated bf16 2048x8192 to e4m3"),
        # the same layer for a few sequences that are decoded together, result in 16 bits
        _gated(16, 2048, "f16", "f16", "silu", name="gated f16 16x2048"),
        # activations that come from an operator without an 8-bit output
        _quantize(8192, 2048, "bf16", 1, name="quantize bf16 8192x2048 rows"),
        # a layer's fp32 weights, once at load
        _quantize(4096, 4096, "f32", 128, name="quantize f32 4096x4096 blocks"),
        # one token through a square layer: reading the weights is the work
        _matmul(1, 4096, 4096, "bf16", name="matmul 1x4096x4096 bf16"),
        # sixteen sequences decoded together, through the wide projection of a smaller network
        _matmul(16, 8192, 2048, "f16", name="matmul 16x8192x2048 f16"),
        # a classifier head on a ragged batch: logits in fp32 with bias
        _matmul(100, 1000, 2048, "f32", epilogue=True, name="matmul 100x1000x2048 f32 bias"),
        # the square size of the matmul sweep
        _matmul(4096, 4096, 4096, "bf16", name="matmul 4096 bf16"),
        # a long prompt through a large layer: the largest call
        _matmul(8192, 8192, 4096, "bf16", name="matmul 8192x8192x4096 bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choices(("matmul", "norm", "gated", "quantize"), (5, 2, 1.5, 1.5))[0]
    if op == "matmul":
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 16, 8192), 16 * _log(rng, 1, 512)
            if rng.random() < 0.6:
                n = max(16, n // 8 * 8)
            if m * n * k <= 8192 * 8192 * 4096:
                return _matmul(m, n, k, rng.choice(("f32", "f16", "bf16")), rng.random() < 0.4)
    m, k, dtype = _log(rng, 1, 8192), _log(rng, 64, 8192), rng.choice(("bf16", "bf16", "f16", "f16", "f32"))
    if rng.random() < 0.75:
        k = max(64, k // 16 * 16)
    if m * k > 4096 * 4096:
        m = 4096 * 4096 // k
    if op == "norm":
        return _norm(m, k, dtype, rng.choice(("e4m3", dtype)), rng.random() < 0.6, rng.choice((0, 0, 8, 40)))
    if op == "gated":
        return _gated(m, k, dtype, rng.choice(("e4m3", dtype)), rng.choice(("silu", "silu", "silu", "hard_swish", "sigmoid")))
    return _quantize(m, k, dtype, rng.choice((1, 1, 128)))


# --------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# --------------------------------------------------------------------------------------------------------------------
def _blocks(k):
    return -(-k // BLOCK)


def _activations(g, m, k, dtype):
    """Normal values with a few columns that are much larger, as hidden states have them."""
    x = torch.randn((m, k), generator=g, device="cuda")
    loud = torch.rand(k, generator=g, device="cuda") < 0.01
    return (x * torch.where(loud, 20.0, 1.0)).to(DT[dtype])


def _operand(x, rows):
    """An fp32 matrix in e4m3 with its scales (one for `rows` x 128 values)."""
    m, k = x.shape
    mb, kb = -(-m // rows), _blocks(k)
    p = torch.nn.functional.pad(x, (0, kb * BLOCK - k, 0, mb * rows - m)).view(mb, rows, kb, BLOCK)
    s = p.abs().amax(dim=(1, 3)).clamp_min(LEAST) / TOP
    q = (p / s[:, None, :, None]).view(mb * rows, kb * BLOCK)[:m, :k].to(torch.float8_e4m3fn)
    return q.contiguous(), s.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    op, s = case["op"], dict(case)
    if op == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["sa"] = _operand(_activations(g, m, k, "f32"), 1)
        s["b"], s["sb"] = _operand(torch.randn((n, k), generator=g, device="cuda") / math.sqrt(k), BLOCK)
        s["bias"] = torch.randn(n, generator=g, device="cuda") if case["epilogue"] else None
        s["c_out"] = torch.empty((m, n), device="cuda", dtype=DT[case["c"]])
        return s
    m, k, dtype = case["m"], case["k"], case["dtype"]
    out = case.get("out", "e4m3")
    rows = case.get("rows", 1)
    s["y"] = torch.empty((m, k), device="cuda", dtype=DT[out])
    s["s"] = torch.empty((-(-m // rows), _blocks(k)), device="cuda") if out == "e4m3" else None
    if op == "norm":
        s["x"] = _activations(g, m, k + case["pad"], dtype)[:, :k]
        s["res"] = _activations(g, m, k, dtype) if case["residual"] else None
        s["w"] = 1.0 + 0.1 * torch.randn(k, generator=g, device="cuda")
        s["sum"] = torch.empty((m, k), device="cuda", dtype=DT[dtype]) if case["residual"] else None
    elif op == "gated":
        s["x"] = torch.randn((m, 2 * k), generator=g, device="cuda").mul_(2.0).to(DT[dtype])   # gate | up
    elif rows == 1:
        s["x"] = _activations(g, m, k, dtype)
    else:
        s["x"] = (torch.randn((m, k), generator=g, device="cuda") / math.sqrt(k)).to(DT[dtype])
    return s


# --------------------------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------------------------
def _round(y, dtype):
    """To the type of the result; fp16 keeps finite values finite, as the library's other kernels do."""
    if dtype == "f16":
        top = 65504.0
        y = torch.where(y.isfinite(), y.clamp(-top, top), y)
    return y.to(DT[dtype])


def _to_blocks(y, rows):
    """y in e4m3 with a scale for each block of `rows` x 128."""
    m, k = y.shape
    mb, kb = -(-m // rows), _blocks(k)
    p = torch.nn.functional.pad(y, (0, kb * BLOCK - k, 0, mb * rows - m)).view(mb, rows, kb, BLOCK)
    s = torch.where(p.isfinite(), p.abs(), 0.0).amax(dim=(1, 3)).clamp_min(LEAST) / TOP
    q = p / s[:, None, :, None]
    q = torch.where(q.isfinite(), q.clamp(-TOP, TOP), float("nan")).to(torch.float8_e4m3fn)
    return q.view(mb * rows, kb * BLOCK)[:m, :k].contiguous(), s


def _act(x, act):
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-x))
    if act == "hard_swish":
        return x * ((x + 3.0) / 6.0).clamp(0.0, 1.0)
    return x


def _plain(s):
    op = s["op"]
    if op == "matmul":
        m, n, k = s["m"], s["n"], s["k"]
        a = s["a"].float() * s["sa"].repeat_interleave(BLOCK, 1)[:, :k]
        b = s["b"].float() * s["sb"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
        c = a @ b.T
        if s["bias"] is not None:
            c = (c + s["bias"]).clamp_min(0.0)
        return [_round(c, s["c"])]
    out = s.get("out", "e4m3")
    if op == "norm":
        h = s["x"].float()
        if s["res"] is not None:
            h = h + s["res"].float()
        y = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * s["w"]
        got = [_round(h, s["dtype"])] if s["res"] is not None else []
    elif op == "gated":
        k, got = s["k"], []
        y = _act(s["x"][:, :k].float(), s["act"]) * s["x"][:, k:].float()
    else:
        y, got = s["x"].float(), []
    if out == "e4m3":
        return got + list(_to_blocks(y, s.get("rows", 1)))
    return got + [_round(y, out)]


def _p(t):
    return None if t is None else t.data_ptr()


_library = None


def _own(s):
    global _library
    if _library is None:
        from nncv_b200 import _lib
        _library = _lib.lib(), _lib.check
    (L, check), op = _library, s["op"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "matmul":
        check(L.nncv_b200_matmul_e4m3(_p(s["a"]), _p(s["sa"]), _p(s["b"]), _p(s["sb"]), _p(s["c_out"]), s["m"], s["n"], s["k"], CODE[s["c"]],
                                      _p(s["bias"]), int(s["bias"] is not None), stream))
        return [s["c_out"]]
    m, k, dtype, x = s["m"], s["k"], CODE[s["dtype"]], s["x"]
    if op == "norm":
        check(L.nncv_b200_rmsnorm(_p(x), x.stride(0), _p(s["res"]), _p(s["w"]), EPS, _p(s["sum"]), _p(s["y"]), CODE[s["out"]], _p(s["s"]), dtype,
                                  m, k, stream))
        return [t for t in (s["sum"], s["y"], s["s"]) if t is not None]
    if op == "gated":
        check(L.nncv_b200_gated_activation(_p(x), _p(x[:, k:]), 2 * k, _p(s["y"]), CODE[s["out"]], _p(s["s"]), dtype, m, k, ACT[s["act"]], stream))
        return [t for t in (s["y"], s["s"]) if t is not None]
    check(L.nncv_b200_quantize_e4m3(_p(x), k, dtype, _p(s["y"]), _p(s["s"]), m, k, s["rows"], stream))
    return [s["y"], s["s"]]


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    op, m, k = case["op"], case["m"], case["k"]
    if op == "matmul":
        n = case["n"]
        scales = 4 * _blocks(k) * (m + _blocks(n))
        return {"bytes": m * k + n * k + m * n * SIZE[case["c"]] + scales + (4 * n if case["epilogue"] else 0), "flops": 2 * m * n * k}
    e, out = SIZE[case["dtype"]], case.get("out", "e4m3")
    rows = case.get("rows", 1)
    scales = 4 * -(-m // rows) * _blocks(k) if out == "e4m3" else 0
    if op == "norm":
        return {"bytes": m * k * (e + (2 * e if case["residual"] else 0) + SIZE[out]) + 4 * k + scales, "flops": 6 * m * k}
    if op == "gated":
        return {"bytes": m * k * (2 * e + SIZE[out]) + scales, "flops": 8 * m * k}
    return {"bytes": m * k * (e + 1) + scales, "flops": 3 * m * k}


# --------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits (values that leave in 8 or 16 bits as they are before that rounding)
# --------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op, m, k = case["op"], case["m"], case["k"]
    if op == "matmul":
        n, total = case["n"], 0
        total = torch.zeros((m, n), device="cuda", dtype=torch.float64)
        for b in range(_blocks(k)):
            cols = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            wide = s["sb"][:, b].double()[torch.arange(n, device="cuda") // BLOCK]
            total += (s["a"][:, cols].double() * s["sa"][:, b, None].double()) @ (s["b"][:, cols].double() * wide[:, None]).T
        if s["bias"] is not None:
            total = torch.relu(total + s["bias"].double())
        return [total]
    first = []
    x = s["x"].double()
    if op == "norm":
        if case["residual"]:
            x = x + s["res"].double()
            first = [x]
        y = x * torch.rsqrt(x.square().sum(1, keepdim=True) / k + EPS) * s["w"].double()
    elif op == "gated":
        gate, up = x.split(k, 1)
        if case["act"] == "silu":
            y = gate * torch.sigmoid(gate) * up
        elif case["act"] == "sigmoid":
            y = torch.sigmoid(gate) * up
        else:
            y = gate * torch.minimum(torch.maximum(gate + 3, torch.zeros_like(gate)) / 6, torch.ones_like(gate)) * up
    else:
        y = x
    if case.get("out", "e4m3") != "e4m3":
        return first + [y]
    rows, kb = case.get("rows", 1), _blocks(k)
    scale = torch.zeros((-(-m // rows), kb), device="cuda", dtype=torch.float64)
    q = torch.empty_like(y)
    if rows == 1:
        for b in range(kb):
            part = y[:, b * BLOCK:(b + 1) * BLOCK]
            scale[:, b] = part.abs().amax(1).clamp(min=LEAST) / 448
            q[:, b * BLOCK:(b + 1) * BLOCK] = part / scale[:, b, None]
    else:
        for r in range(scale.shape[0]):
            for b in range(kb):
                part = y[r * rows:(r + 1) * rows, b * BLOCK:(b + 1) * BLOCK]
                scale[r, b] = part.abs().max().clamp(min=LEAST) / 448
                q[r * rows:(r + 1) * rows, b * BLOCK:(b + 1) * BLOCK] = part / scale[r, b]
    return first + [q, scale]
