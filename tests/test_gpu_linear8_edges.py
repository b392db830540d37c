"""The 8-bit linear layer where a definition is easily missed: quotients at ties, gates far below zero, infinities, weights far from one,
empty tensors, calls of several sizes in one graph."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import linear8_ref as R  # noqa: E402
from nncv_b200._lib import BF16, E4M3, F16, F32, check, lib  # noqa: E402
from test_gpu_linear8 import ACT, DT, gen, guarded, p, run_gated, run_matmul, run_norm, status, stream  # noqa: E402

U = R.U
INF, NAN = float("inf"), float("nan")


# ---------------------------------------------------------------------------------------------------------------- e4m3 of a quotient
def quotients(x, rows):
    """q and scales of finite fp32 values as the definition has them, each operation in fp32 and correctly rounded (on the CPU)."""
    x = x.float().cpu()
    m, k = x.shape
    mb, kb = -(-m // rows), R.blocks(k)
    pad = torch.zeros((mb * rows, kb * 128))
    pad[:m, :k] = x
    amax = pad.view(mb, rows, kb, 128).abs().amax(dim=(1, 3)).clamp_min(2.0 ** -100)
    s = amax * (torch.tensor(1.0) / torch.tensor(448.0))
    return (x / s.repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]).clamp(-448, 448).to(torch.float8_e4m3fn), s


def run_quantize(x, dt, rows):
    m, k = x.shape
    q, free = guarded(m, k, torch.float8_e4m3fn)
    s, free_s = guarded(-(-m // rows), R.blocks(k), torch.float32)
    check(lib().nncv_b200_quantize_e4m3(p(x), x.stride(0), dt, p(q), p(s), m, k, rows, stream()))
    status()
    free()
    free_s()
    return q, s


def at_ties(m, k, seed):
    """Values that lie half way between two e4m3 values times the scale of their block, to the bit where the scale comes out as it was meant: it has 15
    bits, so that its products with 448 and with a midpoint (5 bits) are exact in fp32."""
    g = torch.Generator().manual_seed(seed)
    s = (torch.randint(2 ** 14, 2 ** 15, (m, R.blocks(k)), generator=g) | 1).float() * 2.0 ** -20
    e = torch.randint(0, 14, (m, k), generator=g) - 6
    half = (torch.randint(8, 16, (m, k), generator=g).float() + 0.5) / 8 * torch.exp2(e.float())
    half = half.clamp_max(432.0) * (torch.randint(0, 2, (m, k), generator=g) * 2 - 1)
    half[:, ::128] = 448.0
    return half * s.repeat_interleave(128, 1)[:, :k]


@pytest.mark.parametrize("m,k", [(300, 1024), (7, 1000), (64, 77)])
def test_quantize_rows_at_ties(m, k):
    x = at_ties(m, k, m + k)
    want, s = quotients(x, 1)
    q, got_s = run_quantize(x.cuda(), F32, 1)
    assert torch.equal(got_s.cpu(), s)
    assert R.exactly(q, want), (q.cpu().view(torch.uint8) != want.view(torch.uint8)).float().mean().item()


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("m,k,size", [(600, 2048, 1.0), (129, 1000, 1e-3), (600, 2048, 30.0)])
def test_quantize_is_the_quotient(dt, rows, m, k, size):
    x = (torch.randn((m, k), generator=gen(m, k, dt, rows), device="cuda") * size).to(DT[dt])
    want, s = quotients(x, rows)
    q, got_s = run_quantize(x, dt, rows)
    assert torch.equal(got_s.cpu(), s)
    assert R.exactly(q, want), (q.cpu().view(torch.uint8) != want.view(torch.uint8)).float().mean().item()


@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("size", [3e38, 1e30, 1e-20, 1e-28, 1e-30, 3e-31, 1e-35, 1e-40])
def test_quantize_is_the_quotient_at_both_ends_of_fp32(rows, size):
    x = torch.rand((256, 512), generator=gen(rows), device="cuda").mul_(2).sub_(1).mul_(size)
    want, s = quotients(x, rows)
    q, got_s = run_quantize(x, F32, rows)
    assert torch.equal(got_s.cpu(), s) and R.exactly(q, want)


@pytest.mark.parametrize("with_up", [True, False])
def test_gated_to_e4m3_is_the_quotient(with_up):
    """Without an activation the product is one rounding, so that every bit is known."""
    g = gen(71, with_up)
    gate, up = (torch.randn((300, 1024), generator=g, device="cuda").bfloat16() for _ in range(2))
    out, s = run_gated(gate, up if with_up else None, "none", BF16, True)
    want, want_s = quotients(gate.float() * up.float() if with_up else gate.float(), 1)
    assert torch.equal(s.cpu(), want_s) and R.exactly(out, want)


# ---------------------------------------------------------------------------------------------------------------- gates far below zero
def far_gates(dt):
    x = torch.linspace(-120.0, -70.0, 2048, dtype=torch.float64)
    return torch.cat([x, -x[:512], torch.linspace(-3.0, 3.0, 512, dtype=torch.float64)]).to(DT[dt]).cuda().view(3, 1024)


@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("size", [1.0, 1e30, 1e38])
@pytest.mark.parametrize("pad", [0, 5])
def test_gates_far_below_zero(dt, act, size, pad):
    """act(gate) is a small number there and no zero, and a large `up` makes an ordinary value of it.  In fp32 with an exponential of 2 ulp: ten
    steps in all where the activation is a normal number, half a step of the subnormals (times up) below."""
    gate = torch.zeros((3, 1024 + pad), device="cuda", dtype=DT[dt])
    gate[:, :1024] = far_gates(dt)
    up = torch.full_like(gate, size)
    gate, up = gate[:, :1024], up[:, :1024]
    a = R.act(gate, act)
    y = a * up.double()
    y = torch.where(y.abs() > torch.finfo(DT[dt]).max, torch.copysign(torch.full_like(y, INF), y), y)
    out, _ = run_gated(gate, up, act, dt, False)
    off = 12 * U * y.abs() + 2 * 2.0 ** -149 * up.double().abs()
    fin = y.isfinite()
    assert torch.equal(out.double()[~fin], y[~fin])
    assert ((out.double() - y).abs()[fin] <= (off + R.HALF[DT[dt]] * 1.001 * (y.abs() + off) + R.TINY[DT[dt]])[fin]).all()


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("k", [512, 515])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("with_up", [True, False])
@pytest.mark.parametrize("e4m3", [True, False])
def test_a_far_gate_leaves_the_rest_as_it_is(dt, k, act, with_up, e4m3):
    g = gen(72, dt, k)
    gate, up = (torch.randn((40, k), generator=g, device="cuda").to(DT[dt]) for _ in range(2))
    gate[:, ::128] = 3.0
    up[:, ::128] = 50.0                          # with up the largest value of every block
    want = run_gated(gate, up if with_up else None, act, dt, e4m3)
    far = torch.rand((40, k), generator=g, device="cuda") < 0.01
    far[:, ::128] = False
    other = gate.clone()
    other[far] = -95.0
    # without up a gate beyond 3 may be a block's largest value; where that becomes a far one, the block has another scale
    y = R.act(gate, act) * (up.double() if with_up else 1)
    same = R.scales_of(y, 1) == R.scales_of(torch.where(far, 0.0, y), 1)
    assert same.float().mean() > 0.95 and (same.all() or not with_up)
    rest = ~far & (same.repeat_interleave(128, 1)[:, :k] if e4m3 else True)
    for place in ("apart", "gate", "up"):
        if place == "apart" or e4m3 or (place == "up" and not with_up):
            got = run_gated(other, up if with_up else None, act, dt, e4m3)
        else:
            a, b = other.clone(), up.clone()
            o = {"gate": a, "up": b}[place]
            check(lib().nncv_b200_gated_activation(p(a), p(b) if with_up else None, 0, p(o), dt, None, dt, 40, k, ACT[act], stream()))
            status()
            got = (o, None)
        assert torch.equal(got[0].float()[rest], want[0].float()[rest])
        assert (got[0].float()[far].abs() <= 1e-30).all()
        assert not e4m3 or torch.equal(got[1][same], want[1][same])


# ---------------------------------------------------------------------------------------------------------------- infinities in 16 bits
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("k", [512, 515, 16400, 16403])
def test_norm_keeps_infinities(dt, k):
    """The sum with the residual is itself infinite, not the type's largest value; the row's norm is 1 / inf."""
    g = gen(81, dt, k)
    x, r = (torch.randn((6, k), generator=g, device="cuda").to(DT[dt]) for _ in range(2))
    x[0, 3], x[1, k - 1], r[2, 200], x[3, 7], x[4, 9], r[4, 9] = INF, -INF, INF, NAN, INF, -INF
    want = x.double() + r.double()
    for e4m3 in (False, True):
        out, sums, s = run_norm(x, r, None, 1e-6, dt, e4m3, True)
        assert torch.equal(sums.double().isnan(), want.isnan())
        bad = want.isinf()
        assert bad.sum() == 3 and torch.equal(sums.double()[bad], want[bad])
        v = out.float()
        assert torch.isnan(v[3]).all() and torch.isnan(v[4]).all() and torch.isfinite(v[5]).all()
        for row in range(3):
            assert torch.isnan(v[row][bad[row]]).all() and (v[row][~bad[row]] == 0).all()
    big = torch.full((1, k), 60000.0 if dt == F16 else 1.0, device="cuda").to(DT[dt])
    _, sums, _ = run_norm(big, big, None, 1e-6, dt, False, True)
    assert (sums == (65504 if dt == F16 else 2)).all()      # what is finite stays finite


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("k", [512, 515])
@pytest.mark.parametrize("act", ["none", "silu", "hard_swish"])
@pytest.mark.parametrize("with_up", [True, False])
def test_gated_keeps_infinities(dt, k, act, with_up):
    g = gen(82, dt, k)
    gate, up = (torch.randn((6, k), generator=g, device="cuda").to(DT[dt]) for _ in range(2))
    up = up.abs() + 0.25
    gate[0, 3], gate[1, k - 1], gate[2, 130] = INF, NAN, 200.0
    up[2, 130], up[3, 5], up[4, 6] = (65504.0 if dt == F16 else 2.0), NAN, INF
    gate[4, 6] = 2.0
    out, _ = run_gated(gate, up if with_up else None, act, dt, False)
    assert out[0, 3] == INF and torch.isnan(out[1, k - 1])
    assert out[2, 130] == ((65504 if dt == F16 else 400) if with_up else 200)
    bad = [(0, 3), (1, k - 1)]
    if with_up:
        assert torch.isnan(out[3, 5]) and out[4, 6] == INF
        bad += [(3, 5), (4, 6)]
    q, s = run_gated(gate, up if with_up else None, act, dt, True)
    v = R.dequantize(q, s, 1)
    for t in (out, v):
        fin = torch.ones_like(t, dtype=torch.bool)
        for at in bad:
            fin[at] = False
        assert torch.isfinite(t[fin]).all()
    assert all(torch.isnan(v[at]) for at in bad) and torch.isfinite(s).all()


@pytest.mark.parametrize("m,n,k", [(3, 64, 2048), (40, 264, 256), (40, 261, 256), (776, 5000, 640), (2304, 2304, 1152), (1600, 1999, 2000)])
@pytest.mark.parametrize("cdt", [F32, F16, BF16])
@pytest.mark.parametrize("epilogue", [False, True])
def test_matmul_keeps_infinities(m, n, k, cdt, epilogue):
    """An infinite scale makes its row infinite in every type; what is finite but beyond fp16 becomes its largest value."""
    g = gen(83, m, n, k)
    a, sa = R.operand(g, m, k, 1)
    b, sb = R.operand(g, n, k, 128)
    a.view(torch.uint8).bitwise_and_(0x7F)   # no negative values, so that no row adds infinities of both signs
    b.view(torch.uint8).bitwise_and_(0x7F)
    sa[1, 0] = INF
    sa[2] *= 1e7
    bias = torch.randn(n, generator=g, device="cuda") if epilogue else None
    c = run_matmul(a, sa, b, sb, cdt, bias, epilogue)
    assert (c[1] == INF).all()
    assert (c[2] == 65504).all() if cdt == F16 else torch.isfinite(c[2]).all()
    rest = [i for i in range(m) if i not in (1, 2)]
    assert torch.isfinite(c[rest]).all()


# ---------------------------------------------------------------------------------------------------------------- weights far from one
@pytest.mark.parametrize("k", [512, 9000, 16400])
@pytest.mark.parametrize("size,weight", [(1e16, 1e-25), (1e-16, 1e24), (1e15, 1e-30)])
def test_norm_with_weights_far_from_one(k, size, weight):
    """The row is brought to size one before the weight comes: neither passes fp32's range."""
    x = torch.randn((3, k), generator=gen(91, k), device="cuda") * size
    w = (torch.randn(k, generator=gen(92, k), device="cuda") + 2) * weight
    out, _, _ = run_norm(x, None, w, 0.0, F32, False, False)
    h = x.double()
    y = h / torch.sqrt((h * h).mean(1, keepdim=True)) * w.double()
    assert ((out.double() - y).abs() <= 50 * U * y.abs()).all()


# ---------------------------------------------------------------------------------------------------------------- empty tensors
def test_empty_tensors_are_calls_that_do_nothing():
    """A tensor without rows has no memory: its address is null."""
    L, n0 = lib(), lib().nncv_b200_launch_count()
    x = torch.empty((0, 256), device="cuda", dtype=torch.bfloat16)
    q, s = torch.empty((0, 256), device="cuda", dtype=torch.float8_e4m3fn), torch.empty((0, 2), device="cuda")
    b, sb = R.operand(gen(6), 64, 256, 128)
    c = torch.empty((0, 64), device="cuda")
    assert p(x) == p(q) == p(s) == p(c) == 0
    check(L.nncv_b200_rmsnorm(p(x), 0, p(x), None, 1e-6, p(x), p(x), BF16, None, BF16, 0, 256, stream()))
    check(L.nncv_b200_rmsnorm(p(x), 0, p(x), None, 1e-6, p(x), p(q), E4M3, p(s), BF16, 0, 256, stream()))
    check(L.nncv_b200_gated_activation(p(x), p(x), 0, p(x), BF16, None, BF16, 0, 256, ACT["silu"], stream()))
    check(L.nncv_b200_gated_activation(p(x), p(x), 0, p(q), E4M3, p(s), BF16, 0, 256, ACT["silu"], stream()))
    for rows in (1, 128):
        check(L.nncv_b200_quantize_e4m3(p(x), 0, BF16, p(q), p(s), 0, 256, rows, stream()))
    check(L.nncv_b200_matmul_e4m3(p(q), p(s), p(b), p(sb), p(c), 0, 64, 256, F32, None, 0, stream()))
    status()
    assert L.nncv_b200_launch_count() == n0


# ---------------------------------------------------------------------------------------------------------------- several sizes in one graph
def test_products_of_several_heights_in_one_graph():
    """Fewer rows take less shared memory: neither a later node of the graph nor a call between its capture and its replay takes
    away what an earlier node needs."""
    g = gen(95)
    b, sb = R.operand(g, 512, 1024, 128)
    ops = [R.operand(g, m, 1024, 1) for m in (128, 100, 64, 40, 17, 8, 1)]
    outs = [torch.empty((a.shape[0], 512), device="cuda") for a, _ in ops]

    def all_of(which):
        for i in which:
            (a, sa), c = ops[i], outs[i]
            check(lib().nncv_b200_matmul_e4m3(p(a), p(sa), p(b), p(sb), p(c), a.shape[0], 512, 1024, F32, None, 0, stream()))
    all_of(range(len(ops)))
    status()
    want = [c.clone() for c in outs]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        all_of(range(len(ops)))
    for last in (len(ops) - 1, 0):
        all_of([last])
        status()
        for c in outs:
            c.fill_(NAN)
        gr.replay()
        status()
        assert all(torch.equal(c, w) for c, w in zip(outs, want))


# ---------------------------------------------------------------------------------------------------------------- the same bits
@pytest.mark.parametrize("e4m3", [True, False])
def test_every_call_gives_the_same_bits(e4m3):
    g = gen(96)
    t = torch.randn((512, 8192), generator=g, device="cuda").bfloat16()
    w = torch.randn(4096, generator=g, device="cuda")
    first = None
    for _ in range(4):
        got = [o for o in run_gated(t[:, :4096], t[:, 4096:], "silu", BF16, e4m3) + run_norm(t[:, :4096], t[:, 4096:].contiguous(), w, 1e-6, BF16, e4m3, True)
               if o is not None]
        first = first or got
        assert all(R.exactly(a, b) for a, b in zip(got, first))
