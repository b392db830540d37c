"""The 8-bit linear layer (norm, gated activation, quantisation, block-scaled matmul) against 64 bits, through the C ABI.
Tolerances are derived in linear8_ref.py."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import linear8_ref as R  # noqa: E402
from nncv_b200._lib import BF16, E4M3, F16, F32, check, lib  # noqa: E402

DT = {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}
ACT = {"none": 0, "relu": 1, "hard_sigmoid": 2, "hard_swish": 3, "sigmoid": 4, "silu": 5}
U = R.U


def gen(*seed):
    return torch.Generator(device="cuda").manual_seed(sum((i + 1) * 7919 * int(s) for i, s in enumerate(seed)))


def p(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def status():
    torch.cuda.synchronize()
    assert lib().nncv_b200_device_status() == 0


def guarded(m, k, dtype, offset=0):
    """An [m,k] tensor `offset` elements into its memory, with what lies around it; and a check that this is still as it was."""
    edge = 512
    flat = torch.empty(edge + offset + m * k + edge, device="cuda", dtype=torch.uint8 if dtype == torch.float8_e4m3fn else dtype)
    flat.view(torch.uint8).fill_(0xA5)
    lo = edge + offset
    t = flat[lo:lo + m * k].view(m, k)
    before = flat.clone()

    def untouched():
        a, b = flat.view(torch.uint8), before.view(torch.uint8)
        e = flat.element_size()
        assert torch.equal(a[:lo * e], b[:lo * e]) and torch.equal(a[(lo + m * k) * e:], b[(lo + m * k) * e:])

    return (t.view(torch.float8_e4m3fn) if dtype == torch.float8_e4m3fn else t), untouched


# ---------------------------------------------------------------------------------------------------------------- matmul
def run_matmul(a, sa, b, sb, cdt, bias=None, relu=False, offset=0):
    m, k = a.shape
    n = b.shape[0]
    c, untouched = guarded(m, n, DT[cdt], offset)
    check(lib().nncv_b200_matmul_e4m3(p(a), p(sa), p(b), p(sb), p(c), m, n, k, cdt, p(bias), int(relu), stream()))
    status()
    untouched()
    return c


def check_matmul(m, n, k, cdt, epilogue, offset=0, spread=1.0):
    g = gen(m, n, k, cdt)
    a, sa = R.operand(g, m, k, 1, spread)
    b, sb = R.operand(g, n, k, 128, spread)
    bias = torch.randn(n, generator=g, device="cuda") * 10 if epilogue else None
    c = run_matmul(a, sa, b, sb, cdt, bias, epilogue, offset)
    ref, size = R.matmul(a, sa, b, sb, bias, epilogue)
    if cdt == F16:
        ref = ref.clamp(-65504, 65504)
    far = (c.double() - ref).abs()
    bound = R.matmul_bound(ref, size, k, DT[cdt])
    assert torch.isfinite(c.float()).all()
    assert (far <= bound).all(), (far / bound).max().item()
    return c


@pytest.mark.parametrize("m,n,k", [
    (1, 16, 16), (1, 128, 128), (1, 1, 16), (2, 3, 48), (1, 4096, 4096), (5, 200, 144), (16, 1024, 512), (33, 65, 1040), (64, 512, 272),
    (100, 1000, 2048), (127, 129, 128), (128, 128, 256), (129, 257, 384), (130, 1000, 112), (256, 2048, 1024), (300, 640, 4000), (1000, 1111, 640),
    (513, 4096, 256), (2048, 1024, 512), (4096, 512, 144), (1, 8192, 16), (8192, 16, 64), (1500, 2056, 528), (2304, 2304, 1152)])
@pytest.mark.parametrize("cdt,epilogue", [(F32, False), (F16, True), (BF16, False), (F32, True)])
def test_matmul(m, n, k, cdt, epilogue):
    check_matmul(m, n, k, cdt, epilogue)


@pytest.mark.parametrize("m,n,k", [
    (2304, 2307, 1152), (2300, 2304, 1152),          # 256 x 128 on pairs
    (1600, 1999, 2000), (1500, 2056, 2064),          # 256 x 256 on pairs
    (777, 5000, 640), (776, 5001, 656),              # 128 x 128
    (1, 5876, 2080), (9, 2999, 4096), (9, 3000, 4096), (1, 999, 2720),     # 128 x 128, two, four and eight CTAs a tile
    (3, 4607, 2752), (40, 2050, 8192), (200, 129, 8192), (200, 128, 8192)])   # 128 x 64, likewise
@pytest.mark.parametrize("cdt,epilogue", [(F32, True), (F16, False), (BF16, True), (F32, False)])
def test_matmul_every_tile(m, n, k, cdt, epilogue):
    """The sizes that the model gives to each tile and each number of CTAs, with and without rows on 16-byte boundaries."""
    check_matmul(m, n, k, cdt, epilogue)


@pytest.mark.parametrize("m,n,k,cdt,offset", [(1600, 2000, 2000, BF16, 1), (1600, 2000, 2000, F32, 2), (3, 64, 128, F32, 1), (40, 264, 256, BF16, 1), (40, 264, 256, BF16, 2), (200, 1024, 256, F16, 4), (1, 2048, 512, BF16, 8)])
def test_matmul_into_any_address(m, n, k, cdt, offset):
    check_matmul(m, n, k, cdt, False, offset)


def test_matmul_scales_far_apart():
    check_matmul(150, 300, 1024, F32, False, spread=8.0)


def test_matmul_an_absurd_value_stays_in_its_row_and_column():
    g = gen(3)
    a, sa = R.operand(g, 200, 512, 1)
    b, sb = R.operand(g, 300, 512, 128)
    want = run_matmul(a, sa, b, sb, F32)
    a2, sa2, b2 = a.clone(), sa.clone(), b.clone()
    a2.view(torch.uint8)[7, 300] = 0x7F        # NaN
    sa2[150, 1] = float("inf")
    b2.view(torch.uint8)[299, 5] = 0xFF        # NaN
    got = run_matmul(a2, sa2, b2, sb, F32)
    assert torch.isnan(got[7]).all() and torch.isnan(got[:, 299]).all()
    assert not torch.isfinite(got[150]).any()
    keep = torch.ones_like(got, dtype=torch.bool)
    keep[7] = keep[150] = False
    keep[:, 299] = False
    assert torch.equal(got[keep], want[keep])


def test_matmul_nan_passes_relu_and_zeros_stay():
    g = gen(4)
    a, sa = R.operand(g, 130, 256, 1)
    b, sb = R.operand(g, 64, 256, 128)
    a.view(torch.uint8)[0, 0] = 0x7F
    a.view(torch.uint8)[1] = 0
    c = run_matmul(a, sa, b, sb, BF16, None, True)
    assert torch.isnan(c[0]).all() and (c[1] == 0).all() and (c[2:] >= 0).all()


def test_matmul_fp16_saturates():
    a = torch.full((2, 256), 448.0, device="cuda").to(torch.float8_e4m3fn)
    b = torch.full((32, 256), 448.0, device="cuda").to(torch.float8_e4m3fn)
    c = run_matmul(a, torch.ones(2, 2, device="cuda"), b, torch.ones(1, 2, device="cuda"), F16)
    assert (c == 65504).all()


def test_matmul_same_bits_every_time_and_for_any_batch():
    """A row's result does not change from call to call."""
    g = gen(5)
    a, sa = R.operand(g, 96, 4096, 1)
    b, sb = R.operand(g, 640, 4096, 128)
    want = run_matmul(a, sa, b, sb, F32)
    for _ in range(3):
        assert torch.equal(run_matmul(a, sa, b, sb, F32), want)


def test_matmul_no_rows_is_a_call_that_does_nothing():
    c = torch.full((4,), 7.0, device="cuda")
    b, sb = R.operand(gen(6), 64, 128, 128)
    n0 = lib().nncv_b200_launch_count()
    check(lib().nncv_b200_matmul_e4m3(p(b), p(sb), p(b), p(sb), p(c), 0, 64, 128, F32, None, 0, stream()))
    status()
    assert (c == 7).all() and lib().nncv_b200_launch_count() == n0


def test_matmul_result_past_2_31_elements():
    m, n, k = 66000, 33000, 64
    g = gen(7)
    a, sa = R.operand(g, m, k, 1)
    b, sb = R.operand(g, n, k, 128)
    c = torch.empty((m, n), device="cuda", dtype=torch.bfloat16)
    check(lib().nncv_b200_matmul_e4m3(p(a), p(sa), p(b), p(sb), p(c), m, n, k, BF16, None, 0, stream()))
    status()
    for lo in (0, m // 2, m - 64):
        ref, size = R.matmul(a[lo:lo + 64], sa[lo:lo + 64], b, sb, None, False)
        assert ((c[lo:lo + 64].double() - ref).abs() <= R.matmul_bound(ref, size, k, torch.bfloat16)).all()


# ---------------------------------------------------------------------------------------------------------------- norm
# Relative error of a norm in fp32: the sum of squares adds 64 and 10 + 5 terms one after the other (74 steps, halved by the root), each
# square twice the error of h (1 step); quotient, eps, root, reciprocal and two products 6 more.
NORM_REL = 48 * U


def norm_inputs(g, m, k, dt, pad, offset, residual, weight, big):
    def make(rows, cols):
        flat = torch.randn(offset + rows * cols, generator=g, device="cuda").mul_(big).to(DT[dt])
        return flat[offset:].view(rows, cols)
    x = make(m, k + pad)[:, :k]
    r = make(m, k) if residual else None
    w = (torch.randn(offset + k, generator=g, device="cuda") + 1)[offset:] if weight else None
    return x, r, w


def run_norm(x, r, w, eps, dt, e4m3, keep_sum, offset=0):
    m, k = x.shape
    out, free_out = guarded(m, k, torch.float8_e4m3fn if e4m3 else DT[dt], offset)
    sums, free_sum = guarded(m, k, DT[dt], offset) if keep_sum else (None, None)
    scale, free_scale = guarded(m, R.blocks(k), torch.float32) if e4m3 else (None, None)
    check(lib().nncv_b200_rmsnorm(p(x), x.stride(0), p(r), p(w), eps, p(sums), p(out), E4M3 if e4m3 else dt, p(scale), dt, m, k, stream()))
    status()
    for f in (free_out, free_sum, free_scale):
        if f:
            f()
    return out, sums, scale


def check_norm(m, k, dt, e4m3, residual=True, weight=True, pad=0, offset=0, big=1.0, eps=1e-6):
    g = gen(m, k, dt, e4m3, pad)
    x, r, w = norm_inputs(g, m, k, dt, pad, offset, residual, weight, big)
    out, sums, scale = run_norm(x, r, w, eps, dt, e4m3, residual, offset)
    h = x.double() + (r.double() if residual else 0)
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    y = y * w.double() if weight else y
    if residual:
        assert ((sums.double() - h).abs() <= (R.HALF[DT[dt]] * 1.001 + U) * h.abs() + R.TINY[DT[dt]]).all()
    # h is off by a step of itself where two terms cancel, and of the others' size in the sum of squares
    if e4m3:
        R.check_e4m3(out, scale, y, 1, NORM_REL)
    else:
        assert ((out.double() - y).abs() <= (R.HALF[DT[dt]] * 1.001 + NORM_REL) * y.abs() + R.TINY[DT[dt]]).all()


@pytest.mark.parametrize("m,k", [(1, 1), (1, 8), (2, 7), (1, 4096), (3, 128), (5, 129), (7, 1000), (64, 1024), (33, 2047), (9, 5120), (4, 8192),
                                 (2, 8200), (3, 16384), (2, 16392), (2, 32768), (1, 32767), (3, 40000), (300, 6144), (450, 12000), (700, 512), (1025, 200)])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("e4m3", [True, False])
def test_norm(m, k, dt, e4m3):
    check_norm(m, k, dt, e4m3)


@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("residual,weight,pad,offset", [(False, True, 0, 0), (True, False, 0, 0), (False, False, 24, 0), (True, True, 8, 0), (True, True, 3, 0),
                                                        (True, True, 0, 1), (False, True, 0, 3)])
def test_norm_forms(e4m3, residual, weight, pad, offset):
    for dt in (F32, F16, BF16):
        check_norm(37, 768, dt, e4m3, residual, weight, pad, offset)


def test_norm_sizes_of_values():
    check_norm(16, 512, F32, True, big=1e15)
    check_norm(16, 512, F32, False, big=1e-15, eps=0.0)
    check_norm(16, 512, BF16, True, big=1e-10)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("k", [768, 771, 9000, 16400, 16403])
def test_norm_in_place(dt, k):
    g = gen(11, dt, k)
    x, r, w = norm_inputs(g, 50, k, dt, 0, 0, True, True, 1.0)
    out, sums, _ = run_norm(x, r, w, 1e-5, dt, False, True)
    q, _, scale = run_norm(x, r, w, 1e-5, dt, True, True)
    for sum_at, out_at in (("r", "x"), ("x", "r"), ("r", None), ("x", None)):
        x2, r2 = x.clone(), r.clone()
        at = {"x": x2, "r": r2}
        o = at[out_at] if out_at else torch.empty_like(x)
        check(lib().nncv_b200_rmsnorm(p(x2), 0, p(r2), p(w), 1e-5, p(at[sum_at]), p(o), dt, None, dt, 50, k, stream()))
        status()
        assert torch.equal(at[sum_at], sums) and torch.equal(o, out)
    q2, s2 = torch.empty((50, k), device="cuda", dtype=torch.float8_e4m3fn), torch.empty_like(scale)
    check(lib().nncv_b200_rmsnorm(p(x), 0, p(r), p(w), 1e-5, p(r), p(q2), E4M3, p(s2), dt, 50, k, stream()))
    status()
    assert R.exactly(q2, q) and torch.equal(s2, scale) and torch.equal(r, sums)


def test_norm_of_zeros_and_of_what_is_not_finite():
    x = torch.randn((4, 512), generator=gen(12), device="cuda")
    x[0] = 0
    x[1, 300] = float("nan")
    x[2, 5] = float("inf")
    q, _, s = run_norm(x, None, None, 1e-6, F32, True, False)
    v = R.dequantize(q, s, 1)
    assert (v[0] == 0).all() and torch.isnan(v[1]).all() and torch.isfinite(s).all() and (s > 0).all()
    assert torch.isnan(v[2, 5]) and (v[2, 6:] == 0).all()      # 1 / inf for the others, inf * 0 for itself
    R.check_e4m3(q[3:], s[3:], x[3:].double() / torch.sqrt(x[3:].double().square().mean() + 1e-6), 1, NORM_REL)


# ---------------------------------------------------------------------------------------------------------------- gated activation, quantisation
def run_gated(gate, up, act, dt, e4m3, offset=0):
    m, k = gate.shape
    out, free = guarded(m, k, torch.float8_e4m3fn if e4m3 else DT[dt], offset)
    scale, free_scale = guarded(m, R.blocks(k), torch.float32) if e4m3 else (None, None)
    check(lib().nncv_b200_gated_activation(p(gate), p(up), gate.stride(0), p(out), E4M3 if e4m3 else dt, p(scale), dt, m, k, ACT[act], stream()))
    status()
    free()
    if e4m3:
        free_scale()
    return out, scale


def check_gated(m, k, dt, act, e4m3, with_up=True, pad=0, offset=0):
    g = gen(m, k, dt, ACT[act], pad)
    t = torch.randn(offset + m * (2 * k + pad), generator=g, device="cuda").mul_(3).to(DT[dt])[offset:].view(m, 2 * k + pad)
    gate, up = t[:, :k], t[:, k:2 * k] if with_up else None
    out, scale = run_gated(gate, up, act, dt, e4m3, offset)
    a = R.act(gate, act)
    u = up.double() if with_up else torch.ones_like(a)
    y = a * u
    off = R.act_bound(gate, a, act, dt != F32) * u.abs() + U * y.abs()
    if e4m3:
        s = scale.double().repeat_interleave(128, 1)[:, :k]
        want = R.scales_of(y, 1)
        most = R.scales_of(off, 1)
        assert ((scale.double() - want).abs() <= most + 3 * U * want).all()
        assert ((out.float().double() * s - y).abs() <= R.half_step(y / s) * s * 1.0001 + off + 6 * U * y.abs()).all()
    else:
        assert ((out.double() - y).abs() <= off + R.HALF[DT[dt]] * 1.001 * (y.abs() + off) + R.TINY[DT[dt]]).all()


@pytest.mark.parametrize("m,k", [(1, 1), (1, 8), (1, 2048), (16, 2048), (3, 130), (7, 1000), (129, 768), (1000, 264), (5, 11008), (2, 77), (4097, 128)])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("e4m3", [True, False])
def test_gated_silu(m, k, dt, e4m3):
    check_gated(m, k, dt, "silu", e4m3)


@pytest.mark.parametrize("act", ["none", "relu", "hard_sigmoid", "hard_swish", "sigmoid", "silu"])
@pytest.mark.parametrize("e4m3", [True, False])
@pytest.mark.parametrize("with_up,pad,offset", [(True, 0, 0), (False, 0, 0), (True, 16, 0), (True, 5, 0), (True, 0, 1)])
def test_gated_forms(act, e4m3, with_up, pad, offset):
    for dt in (F32, F16, BF16):
        check_gated(21, 392, dt, act, e4m3, with_up, pad, offset)


@pytest.mark.parametrize("dt", [F32, F16, BF16])
def test_gated_in_place(dt):
    g = gen(21, dt)
    gate, up = (torch.randn((40, 520), generator=g, device="cuda").to(DT[dt]) for _ in range(2))
    want, _ = run_gated(gate, up, "silu", dt, False)
    for place in (0, 1):
        a, b = gate.clone(), up.clone()
        o = (a, b)[place]
        check(lib().nncv_b200_gated_activation(p(a), p(b), 0, p(o), dt, None, dt, 40, 520, ACT["silu"], stream()))
        status()
        assert torch.equal(o, want)


@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 129), (128, 128), (129, 256), (200, 1000), (1000, 77), (640, 4096), (4096, 72), (127, 2048)])
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("rows", [1, 128])
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 0), (1, 1)])
def test_quantize(m, k, dt, rows, pad, offset):
    g = gen(m, k, dt, rows)
    x = (torch.randn(offset + m * (k + pad), generator=g, device="cuda") * torch.exp(torch.randn((), generator=g, device="cuda") * 3)).to(DT[dt])
    x = x[offset:].view(m, k + pad)[:, :k]
    q, free = guarded(m, k, torch.float8_e4m3fn, offset)
    s, free_s = guarded(-(-m // rows), R.blocks(k), torch.float32)
    check(lib().nncv_b200_quantize_e4m3(p(x), x.stride(0), dt, p(q), p(s), m, k, rows, stream()))
    status()
    free()
    free_s()
    R.check_e4m3(q, s, x.double(), rows, 0.0)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_what_is_not_finite_and_blocks_of_nothing(rows):
    x = torch.randn((256, 384), generator=gen(31), device="cuda")
    x[0:128, 0:128] = 0
    x[5, 200], x[6, 201], x[7, 202] = float("nan"), float("inf"), float("-inf")
    x[128:, 256:] = float("nan")
    x[130, 0:128] = 1e-40
    x[131, 0:128] = 3e38
    q, s = torch.empty_like(x, dtype=torch.float8_e4m3fn), torch.empty((256 // rows, 3), device="cuda")
    check(lib().nncv_b200_quantize_e4m3(p(x), 0, F32, p(q), p(s), 256, 384, rows, stream()))
    status()
    R.check_e4m3(q, s, x.double(), rows, 0.0)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_past_2_31_elements(rows):
    m, k = 131200, 16400
    x = torch.empty((m, k), device="cuda", dtype=torch.bfloat16)
    x.normal_(generator=gen(32))
    q = torch.empty((m, k), device="cuda", dtype=torch.float8_e4m3fn)
    s = torch.empty((-(-m // rows), R.blocks(k)), device="cuda")
    check(lib().nncv_b200_quantize_e4m3(p(x), 0, BF16, p(q), p(s), m, k, rows, stream()))
    status()
    for lo in (0, 130944, m - 128):
        lo = lo // 128 * 128
        R.check_e4m3(q[lo:lo + 128], s[lo // rows:lo // rows + 128 // rows], x[lo:lo + 128].double(), rows, 0.0)


# ---------------------------------------------------------------------------------------------------------------- together
class Block:
    """norm -> gate and up -> gated activation -> down, as a decoder's or a vision transformer's block has them."""

    def __init__(self, m, width, inner, dt, seed):
        g = gen(seed)
        self.m, self.width, self.inner, self.dt = m, width, inner, dt
        self.x = torch.randn((m, width), generator=g, device="cuda").to(DT[dt])
        self.res = torch.randn((m, width), generator=g, device="cuda").to(DT[dt])
        self.w = 1 + 0.1 * torch.randn(width, generator=g, device="cuda")
        self.w1 = torch.randn((2 * inner, width), generator=g, device="cuda") / width ** 0.5
        self.w2 = torch.randn((width, inner), generator=g, device="cuda") / inner ** 0.5
        e4, f = torch.float8_e4m3fn, torch.float32
        def new(r, c, t):
            return torch.empty((r, c), device="cuda", dtype=t)
        kb, ib = R.blocks(width), R.blocks(inner)
        self.q1, self.s1 = new(2 * inner, width, e4), new(R.blocks(2 * inner), kb, f)
        self.q2, self.s2 = new(width, inner, e4), new(R.blocks(width), ib, f)
        self.h, self.hs = new(m, width, e4), new(m, kb, f)
        self.g, self.a, self.as_ = new(m, 2 * inner, DT[dt]), new(m, inner, e4), new(m, ib, f)
        self.sum, self.out = new(m, width, DT[dt]), new(m, width, DT[dt])

    def weights(self):
        L = lib()
        check(L.nncv_b200_quantize_e4m3(p(self.w1), 0, F32, p(self.q1), p(self.s1), 2 * self.inner, self.width, 128, stream()))
        check(L.nncv_b200_quantize_e4m3(p(self.w2), 0, F32, p(self.q2), p(self.s2), self.width, self.inner, 128, stream()))

    def forward(self):
        L, m, w, n, dt = lib(), self.m, self.width, self.inner, self.dt
        check(L.nncv_b200_rmsnorm(p(self.x), 0, p(self.res), p(self.w), 1e-6, p(self.sum), p(self.h), E4M3, p(self.hs), dt, m, w, stream()))
        check(L.nncv_b200_matmul_e4m3(p(self.h), p(self.hs), p(self.q1), p(self.s1), p(self.g), m, 2 * n, w, dt, None, 0, stream()))
        check(L.nncv_b200_gated_activation(p(self.g), self.g.data_ptr() + n * self.g.element_size(), 2 * n, p(self.a), E4M3, p(self.as_), dt, m, n,
                                           ACT["silu"], stream()))
        check(L.nncv_b200_matmul_e4m3(p(self.a), p(self.as_), p(self.q2), p(self.s2), p(self.out), m, w, n, dt, None, 0, stream()))

    def verify(self):
        h = self.x.double() + self.res.double()
        R.check_e4m3(self.h, self.hs, h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * self.w.double(), 1, NORM_REL)
        t = DT[self.dt]
        for got, a, sa, b, sb, k in ((self.g, self.h, self.hs, self.q1, self.s1, self.width), (self.out, self.a, self.as_, self.q2, self.s2, self.inner)):
            ref, size = R.matmul(a, sa, b, sb, None, False)
            assert ((got.double() - ref).abs() <= R.matmul_bound(ref, size, k, t)).all()
        gate, up = self.g[:, :self.inner], self.g[:, self.inner:]
        act = R.act(gate, "silu")
        y = act * up.double()
        off = R.act_bound(gate, act, "silu", True) * up.double().abs() + U * y.abs()
        s = self.as_.double().repeat_interleave(128, 1)[:, :self.inner]
        assert ((self.a.float().double() * s - y).abs() <= R.half_step(y / s) * s * 1.0001 + off + 6 * U * y.abs()).all()
        # against the layer on unrounded operands: three roundings to e4m3 (weights, activations, gated) of half a step of 2^-3 at most each,
        # independent, so that the norm of the error stays well below their sum
        full = (R.act((h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * self.w.double()) @ self.w1.double().T[:, :self.inner], "silu")
                * ((h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6) * self.w.double()) @ self.w1.double().T[:, self.inner:])) @ self.w2.double().T
        assert ((self.out.double() - full).norm() / full.norm()).item() <= 5 * 2.0 ** -4


@pytest.mark.parametrize("m,width,inner", [(1, 512, 1024), (77, 768, 2048), (300, 1024, 1040)])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_a_block_in_a_row_of_calls(m, width, inner, dt):
    b = Block(m, width, inner, dt, m + width)
    b.weights()
    b.forward()
    status()
    b.verify()


def test_blocks_on_two_streams_at_once():
    here = torch.cuda.current_stream()
    blocks = [Block(64 + i, 512, 768, BF16, 40 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in blocks]
    for s in streams:
        s.wait_stream(here)
    for _ in range(3):
        for b, s in zip(blocks, streams):
            with torch.cuda.stream(s):
                b.weights()
                b.forward()
    status()
    for b in blocks:
        b.verify()


def test_two_captured_blocks_replayed_with_new_inputs():
    blocks = [Block(24, 512, 640, F16, 50 + i) for i in range(2)]
    graphs = []
    for b in blocks:
        b.weights()
        b.forward()
        status()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            b.forward()
        graphs.append(gr)
    other = torch.cuda.Stream()
    for k in range(2):
        for i, b in enumerate(blocks):
            b.x.copy_(torch.randn(b.x.shape, generator=gen(60 + k, i), device="cuda"))
            b.out.fill_(float("nan"))
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        status()
        for b in blocks:
            b.verify()


FIRST_CALLS_IN_A_CAPTURE = """
import torch
from nncv_b200._lib import F32, check, lib
L = lib()
x = torch.randn(256, 512, device="cuda")
e4, p = torch.float8_e4m3fn, lambda t: t.data_ptr()
q, s = torch.empty(256, 512, device="cuda", dtype=e4), torch.empty(256, 4, device="cuda")
wq, ws = torch.empty(256, 512, device="cuda", dtype=e4), torch.empty(2, 4, device="cuda")
c, y = torch.empty(256, 256, device="cuda"), torch.empty_like(x)
check(L.nncv_b200_device_status())   # sets the library up on this device
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    st = torch.cuda.current_stream().cuda_stream
    check(L.nncv_b200_quantize_e4m3(p(x), 0, F32, p(q), p(s), 256, 512, 1, st))
    check(L.nncv_b200_quantize_e4m3(p(x), 0, F32, p(wq), p(ws), 256, 512, 128, st))
    check(L.nncv_b200_matmul_e4m3(p(q), p(s), p(wq), p(ws), p(c), 256, 256, 512, F32, None, 0, st))
    check(L.nncv_b200_rmsnorm(p(x), 0, None, None, 1e-6, None, p(y), F32, None, F32, 256, 512, st))
    check(L.nncv_b200_gated_activation(p(y), None, 0, p(y), F32, None, F32, 256, 512, 0, st))
x.mul_(2.0)
g.replay()
torch.cuda.synchronize()
# two roundings to e4m3 of half a step of 2^-3 at most, independent: the norm of the error is well below their sum
ref = x.double() @ x.double().T
assert ((c.double() - ref).norm() / ref.norm()).item() <= 2 * 2.0 ** -4
assert (y.double() - x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + 1e-6)).abs().max().item() <= 6 * 48 * 2.0 ** -24
check(L.nncv_b200_device_status())
print("captured")
"""


def test_first_calls_of_a_process_in_a_capture():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS_IN_A_CAPTURE], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stdout[-500:] + done.stderr[-2000:]
