"""The 8-bit product with every tile and every number of CTAs that share one, asked for by name; which one ran is checked.  Rows of a small batch and
of a large one, scales at the ends of fp32.  Tolerances are derived in linear8_ref.py."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import linear8_ref as R  # noqa: E402
from nncv_b200._lib import BF16, F16, F32, lib  # noqa: E402
from test_gpu_linear8 import DT, check_matmul, gen, run_matmul  # noqa: E402

EVERY = [(0, 1), (0, 2), (0, 4), (0, 8), (1, 1), (1, 2), (1, 4), (1, 8), (2, 1), (3, 1)]


@pytest.fixture
def force():
    def ask(tile, ctas):
        lib().nncv_b200_matmul_e4m3_tile(tile, ctas)
    yield ask
    ask(-1, 0)


def took():
    return divmod(lib().nncv_b200_matmul_e4m3_tile(-2, 0), 16)


# few rows and columns, ragged ones, whole ones, one block of K for each of eight CTAs, a last block of 16 values; at most 9 x 2 tiles, so that as many clusters fit
SHAPES = [(1, 1, 1024), (1, 16, 2064), (3, 100, 1040), (40, 264, 2048), (65, 129, 1936), (127, 128, 1024), (128, 200, 4096), (129, 257, 1056), (200, 127, 8192),
          (256, 256, 1024), (257, 130, 1168), (300, 251, 2576)]


@pytest.mark.parametrize("tile,ctas", EVERY)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_every_tile_on_every_shape(force, tile, ctas, m, n, k):
    for cdt, epilogue in ((F32, False), (F16, True), (BF16, False), (BF16, True)):
        force(tile, ctas)
        check_matmul(m, n, k, cdt, epilogue)
        assert took() == (tile, ctas)


@pytest.mark.parametrize("tile", range(4))
@pytest.mark.parametrize("m,n,k", [(2304, 2307, 144), (1600, 2000, 400), (4100, 129, 272), (70, 8000, 640), (1, 20000, 256)])
def test_every_tile_in_several_rounds(force, tile, m, n, k):
    """More tiles than CTAs: the accumulators, the ring and the slots of the scales go from one tile to the next."""
    force(tile, 1)
    for cdt in (F32, BF16):
        check_matmul(m, n, k, cdt, False)
        assert took() == (tile, 1)


def test_what_does_not_fit_is_chosen_as_without(force):
    for tile, ctas, m, n, k in ((0, 2, 64, 64, 128), (0, 8, 64, 64, 896), (1, 8, 4096, 4096, 1024), (2, 2, 512, 512, 512), (4, 1, 64, 64, 128), (0, 3, 64, 64, 512)):
        force(-1, 0)
        check_matmul(m, n, k, F32, False)
        want = took()
        force(tile, ctas)
        check_matmul(m, n, k, F32, False)
        assert took() == want != (tile, ctas)


@pytest.mark.parametrize("tile,ctas", EVERY)
def test_infinities_in_every_tile(force, tile, ctas):
    force(tile, ctas)
    g = gen(17, tile, ctas)
    for n in (136, 131):
        a, sa = R.operand(g, 130, 1024, 1)
        b, sb = R.operand(g, n, 1024, 128)
        a.view(torch.uint8).bitwise_and_(0x7F)
        b.view(torch.uint8).bitwise_and_(0x7F)
        sa[5, 3], sa[129] = float("inf"), sa[129] * 1e8
        for cdt in (F32, F16, BF16):
            c = run_matmul(a, sa, b, sb, cdt)
            assert took() == (tile, ctas)
            assert (c[5] == float("inf")).all() and torch.isfinite(torch.cat([c[:5], c[6:]])).all()
            assert cdt != F16 or (c[129] == 65504).all()


def test_the_same_bits_from_the_same_tile(force):
    g = gen(18)
    a, sa = R.operand(g, 300, 2048, 1)
    b, sb = R.operand(g, 250, 2048, 128)
    for tile, ctas in EVERY:
        force(tile, ctas)
        first = run_matmul(a, sa, b, sb, F32).clone()
        for _ in range(3):
            assert torch.equal(run_matmul(a, sa, b, sb, F32), first)


@pytest.mark.parametrize("cdt", [F32, F16, BF16])
def test_rows_of_a_small_batch_and_of_a_large_one(cdt):
    """The tile depends on the batch, and with it the order of a row's sum: the rows agree as far as either agrees with 64 bits."""
    g = gen(19)
    a, sa = R.operand(g, 2000, 2064, 1)
    b, sb = R.operand(g, 1111, 2064, 128)
    ref, size = R.matmul(a, sa, b, sb, None, False)
    bound = R.matmul_bound(ref, size, 2064, DT[cdt])
    whole = run_matmul(a, sa, b, sb, cdt).double()
    tiles = {took()}
    for m in (1, 7, 16, 100, 300, 1000):
        part = run_matmul(a[:m], sa[:m], b, sb, cdt).double()
        tiles.add(took())
        assert ((part - whole[:m]).abs() <= 2 * bound[:m]).all()
    assert len(tiles) > 2


def powers(rows, k, e, spread):
    """Scales 2^e times a power of two between 1 and 2^spread, by block."""
    i = torch.arange(rows * R.blocks(k), device="cuda") % (spread + 1)
    return torch.exp2((e + i).float()).view(rows, R.blocks(k))


@pytest.mark.parametrize("ea,eb", [(-60, -66), (-108, -18), (-1, -125), (40, 50), (99, 0), (-100, 200 - 100)])
@pytest.mark.parametrize("m,n,k", [(5, 40, 1040), (300, 264, 512)])
def test_scales_whose_product_is_normal(ea, eb, m, n, k):
    """From 2^-126 to where the result leaves fp32."""
    g = gen(20, m, n)
    a, _ = R.operand(g, m, k, 1)
    b, _ = R.operand(g, n, k, 128)
    sa, sb = powers(m, k, ea, 2), powers(R.blocks(n), k, eb, 1)
    c = run_matmul(a, sa, b, sb, F32)
    ref, size = R.matmul(a, sa, b, sb, None, False)
    assert torch.isfinite(c).all() and c.abs().max() > 0
    assert ((c.double() - ref).abs() <= R.matmul_bound(ref, size, k, torch.float32)).all()


def test_scales_whose_product_is_the_largest():
    """One product of ones, times 2^127."""
    a = torch.zeros((3, 256), device="cuda")
    b = torch.zeros((16, 256), device="cuda")
    a[0, 3] = b[2, 3] = 1.0
    c = run_matmul(a.to(torch.float8_e4m3fn), torch.full((3, 2), 2.0 ** 100, device="cuda"), b.to(torch.float8_e4m3fn), torch.full((1, 2), 2.0 ** 27, device="cuda"), F32)
    assert c[0, 2] == 2.0 ** 127 and c.count_nonzero() == 1


@pytest.mark.parametrize("ea,eb", [(-70, -70), (-108, -30), (-100, -60)])
def test_scales_whose_product_is_below_normal(ea, eb):
    """The product of scales is off by 2^-150 at most, a block's sum is below 448^2 * 128 < 2^24.7, and adding rounds once a block."""
    g = gen(21, ea)
    m, n, k = 70, 130, 1024
    a, _ = R.operand(g, m, k, 1)
    b, _ = R.operand(g, n, k, 128)
    sa, sb = powers(m, k, ea, 2) * 1.3, powers(R.blocks(n), k, eb, 1) * 1.7
    c = run_matmul(a, sa, b, sb, F32)
    ref, size = R.matmul(a, sa, b, sb, None, False)
    assert ((c.double() - ref).abs() <= R.matmul_bound(ref, size, k, torch.float32) + R.blocks(k) * 2.0 ** -125).all()


def test_scales_whose_product_is_beyond_fp32():
    a = torch.full((2, 128), 2.0, device="cuda")
    a[1] = 0
    b = torch.full((16, 128), 1.0, device="cuda").to(torch.float8_e4m3fn)
    c = run_matmul(a.to(torch.float8_e4m3fn), torch.full((2, 1), 2.0 ** 100, device="cuda"), b, torch.full((1, 1), 2.0 ** 28, device="cuda"), F32)
    assert (c[0] == float("inf")).all() and torch.isnan(c[1]).all()
