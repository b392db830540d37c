"""The 8-bit linear layer in 64 bits, from its definition, and how far fp32 arithmetic may be from it."""
import numpy as np
import torch

U = 2.0 ** -24                     # half a step of fp32, relative
HALF = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}   # half a step among the subnormals


def blocks(k):
    return -(-k // 128)


def dequantize(q, s, rows):
    """fp64 values of an e4m3 matrix with a scale for rows x 128 values."""
    m, k = q.shape
    return q.double() * s.double().repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]


def operand(g, m, k, rows, spread=1.0):
    """Random e4m3 values that use the whole range, and scales that differ by orders of magnitude."""
    q = (torch.randn((m, k), generator=g, device="cuda") * 60).clamp(-448, 448).to(torch.float8_e4m3fn)
    s = torch.exp(torch.randn((-(-m // rows), blocks(k)), generator=g, device="cuda") * spread) / 60
    return q, s


def matmul(a, sa, b, sb, bias, relu):
    """The product, and the sum of its terms' absolute values."""
    x, y = dequantize(a, sa, 1), dequantize(b, sb, 128)
    c, size = x @ y.T, x.abs() @ y.abs().T
    if bias is not None:
        c, size = c + bias.double(), size + bias.double().abs()
    return (c.relu() if relu else c), size


def matmul_bound(c, size, k, dtype):
    """A block's 128 terms are exact in fp32 and are added one after the other in the worst case, by an adder that may cut instead of
    round (2^-23 each); then a product of scales, a fused multiply-add a block, partial sums of up to eight groups and the bias."""
    return (128 * 2 + blocks(k) + 10) * U * size + HALF[dtype] * (c.abs() * 1.001) + TINY[dtype]


def scales_of(y, rows):
    m, k = y.shape
    kb, mb = blocks(k), -(-m // rows)
    p = torch.zeros((mb * rows, kb * 128), dtype=torch.float64, device=y.device)
    p[:m, :k] = torch.where(y.isfinite(), y.abs(), 0.0)
    return p.view(mb, rows, kb, 128).amax(dim=(1, 3)).clamp_min(2.0 ** -100) / 448


def half_step(v):
    """Half of e4m3's step at |v|."""
    e = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6)))
    return torch.exp2(e - 4)


def check_e4m3(q, s, y, rows, rel):
    """q, s against y in 64 bits, where fp32 may have y wrong by `rel` of itself."""
    want = scales_of(y, rows)
    assert torch.isfinite(s).all() and (s > 0).all()
    # the constant 1 / 448, its product, and what y itself is off
    assert ((s.double() - want).abs() <= (rel + 3 * U) * want).all()
    v = y / want.repeat_interleave(rows, 0)[: y.shape[0]].repeat_interleave(128, 1)[:, : y.shape[1]]
    fin = y.isfinite()
    got = q.float().double()
    assert torch.isnan(got[~fin]).all()
    v, got = v[fin], got[fin]
    # to the nearest: off by half a step, and by what y, the scale, its reciprocal and the product are off
    assert ((got - v).abs() <= half_step(v) + (2 * rel + 6 * U) * v.abs()).all()
    assert got.abs().max().item() <= 448 if got.numel() else True


def act(x, name):
    x = x.double()
    if name == "none":
        return x
    if name == "relu":
        return torch.where(x <= 0, 0.0, x)
    if name == "hard_sigmoid":
        return ((x + 3) / 6).clamp(0, 1)
    if name == "hard_swish":
        return x * ((x + 3) / 6).clamp(0, 1)
    s = 1 / (1 + torch.exp(-x))
    return s if name == "sigmoid" else x * s


def act_bound(x, y, name, fast):
    """How far fp32 may have the activation from y, absolutely.  The exponential of t is off by 2 ulp and by what rounding t * log2(e) makes of it
    (|t| * 2^-23 at most, with the multiplication's own step as much again); its sum with 1 and the reciprocal another few steps.  hard_sigmoid is
    off by a few steps of a value of at most (|x| + 3) / 6."""
    x = x.double()
    if name in ("none", "relu"):
        return torch.zeros_like(y)
    if name in ("sigmoid", "silu"):
        return (2 * x.abs() + 12) * 2 * U * y.abs() + 2.0 ** -125 * (x.abs() + 1)
    h = ((x.abs() + 3) / 6) * 4 * U
    return h if name == "hard_sigmoid" else h * x.abs() + U * y.abs()


def exactly(a, b):
    return np.array_equal(a.cpu().view(torch.uint8).numpy(), b.cpu().view(torch.uint8).numpy())
