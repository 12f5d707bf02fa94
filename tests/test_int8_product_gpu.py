"""Rows and matrices held in 8-bit codes, and their products."""
import pytest
import torch

import int8_plain as plain

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float32]


def coded(w):
    """A matrix's codes in rows of whole 16 bytes, and its scales, made on the GPU."""
    from nnis_b200.csrc import ops
    codes = torch.full((w.shape[0], ops.int8_width(w.shape[1])), 55, dtype=torch.int8, device="cuda")
    scales = torch.empty(w.shape[0], device="cuda")
    ops.quantize_rows(w.cuda(), codes, scales)
    return codes, scales


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 15), (5, 16), (7, 17), (2, 511), (4, 576), (3, 2048), (2, 8192), (1, 20001), (300, 40)])
def test_rows_become_codes(dtype, rows, k):
    """To the last bit, zeros behind each row; rows further apart than they are long too."""
    x = torch.randn((rows, k), generator=torch.Generator().manual_seed(k)).to(dtype)
    if rows > 2:
        x[1] = 0
        x[2, k // 2] = float("nan")
    for view in (x.cuda(), torch.cat((x, x), 1).cuda()[:, :k]):
        codes, scales = coded(view)
        want, want_scales = plain.codes_of(x)
        assert torch.equal(codes[:, :k].cpu(), want) and (codes[:, k:] == 0).all()
        assert torch.equal(torch.nan_to_num(scales.cpu(), nan=-9.0), torch.nan_to_num(want_scales, nan=-9.0))


def check(dtype, m, n, k, mode, bias=False, seed=0, stride=0):
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    gen = torch.Generator().manual_seed(seed + m + n + k)
    rows = 2 * n if mode == ops.GEMM_GATED else n
    x = (torch.randn((m, k), generator=gen) * (0.1 + 2 * torch.rand((m, 1), generator=gen))).to(dtype)
    w, w_scales = coded(torch.randn((rows, k), generator=gen) * k ** -0.5)
    b = torch.randn(rows, generator=gen) if bias else None
    want, bound = plain.product(x, w.cpu(), k, w_scales.cpu(), b, mode == ops.GEMM_GATED)
    kept = dtype if mode in (ops.STORE, ops.GEMM_GATED) else torch.float32
    out = torch.randn((m, n), generator=gen).to(kept).cuda()
    before = out.cpu().double()
    given = torch.full((m, k + stride), float("nan"), dtype=dtype, device="cuda")
    given[:, :k] = x.cuda()
    ops.linear_int8(given[:, :k], w, w_scales, b.cuda() if bias else None, out, mode, Workspace(torch.device("cuda")))
    if mode == ops.ADD_F32:
        want = want + before
        bound = bound + 2.0 ** -24 * want.abs()
    got = out.cpu().double()
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


SIZES = [(1, 960, 576), (2, 130, 64), (3, 1, 16), (8, 512, 2048), (9, 577, 300), (16, 64, 8192), (17, 96, 33), (33, 200, 1000), (64, 640, 576),
         (65, 129, 17), (128, 256, 256), (130, 257, 515), (1, 1, 1), (5, 8192, 128), (300, 72, 4104), (257, 1000, 576)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("mode", [0, 1, 2, 3])
def test_products(dtype, m, n, k, mode):
    check(dtype, m, n, k, mode)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 960, 576), (7, 65, 40), (40, 130, 700), (200, 384, 512)])
@pytest.mark.parametrize("mode", [0, 1, 2, 3])
def test_products_with_a_bias_and_rows_further_apart(dtype, m, n, k, mode):
    check(dtype, m, n, k, mode, bias=True, seed=1, stride=3)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_large_product(dtype):
    check(dtype, 1500, 1100, 2056, 0)


@pytest.mark.parametrize("m", [1, 20, 200])
@pytest.mark.parametrize("k", [8192, 133136])
def test_the_largest_sums(m, k):
    """All codes at their ends: the sum is the largest that k allows, exact to its last bit."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    x = torch.full((m, k), -1.0, dtype=torch.bfloat16, device="cuda")
    w, w_scales = coded(torch.full((70, k), 1.0))
    out = torch.empty((m, 70), device="cuda")
    ops.linear_int8(x, w, w_scales, None, out, ops.STORE_F32, Workspace(torch.device("cuda")))
    one = torch.tensor(1.0) / torch.tensor(127.0)
    want = torch.tensor(float(-127 * 127 * k)) * one * one
    assert (out.cpu() == want).all()


@pytest.mark.parametrize("m", [1, 40, 300])
def test_tokens_that_are_no_numbers_stay_alone(m):
    """An infinity or a NaN in a token, or in a row of the matrix, makes NaN of that row or column of the output, of no others."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    gen = torch.Generator().manual_seed(3)
    x, w = torch.randn((m, 64), generator=gen).to(torch.bfloat16), torch.randn((96, 64), generator=gen)
    if m > 1:
        x[m // 2, 3] = float("inf")
    w[17, 5] = float("nan")
    codes, scales = coded(w)
    out = torch.empty((m, 96), dtype=torch.bfloat16, device="cuda")
    ops.linear_int8(x.cuda(), codes, scales, None, out, ops.STORE, Workspace(torch.device("cuda")))
    want = torch.zeros((m, 96), dtype=torch.bool)
    want[:, 17] = True
    if m > 1:
        want[m // 2] = True
    assert torch.equal(torch.isnan(out).cpu(), want)


def test_products_on_a_stream_and_in_a_graph():
    """Two products that share a workspace, one after the other, captured and replayed with other rows."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    gen = torch.Generator().manual_seed(4)
    w1, s1 = coded(torch.randn((2 * 256, 128), generator=gen))
    w2, s2 = coded(torch.randn((128, 256), generator=gen))
    x = torch.randn((24, 128), generator=gen).to(torch.bfloat16).cuda()
    act, out, ws = torch.empty((24, 256), dtype=torch.bfloat16, device="cuda"), torch.zeros((24, 128), device="cuda"), Workspace(torch.device("cuda"))

    def step():
        ops.linear_int8(x, w1, s1, None, act, ops.GEMM_GATED, ws)
        ops.linear_int8(act, w2, s2, None, out, ops.STORE_F32, ws)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(2):
        x.copy_(torch.randn((24, 128), generator=gen).to(torch.bfloat16))
        graph.replay()
        first = out.clone()
        step()
        assert torch.equal(first, out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,width", [(1, 4), (3, 20), (7, 576), (40, 2048), (2, 8192), (5, 1028), (300, 64)])
def test_a_norm_and_codes_in_one(dtype, n, width):
    """The codes of the norm's rows: a value may fall to the neighbouring code where the norm's sums, in another order, end an ulp apart."""
    from nnis_b200.csrc import ops
    gen = torch.Generator().manual_seed(width)
    x, w = torch.randn((n, width), generator=gen).cuda(), (1 + 0.1 * torch.randn(width, generator=gen)).cuda()
    normed = torch.empty((n, width), dtype=dtype, device="cuda")
    ops.rmsnorm(x, w, 1e-5, normed)
    codes, scales = coded(normed)
    got, got_scales = torch.full_like(codes, 77), torch.empty_like(scales)
    ops.rmsnorm_int8(x, w, 1e-5, got, got_scales, dtype)
    # sums of `width` squares in two orders differ by up to width roundings of 2^-24 each, their roots by half of that; a few roundings
    # follow, then one of `dtype` that may fall otherwise, in a value or in its row's largest
    step = torch.finfo(dtype).eps + (width + 8) * 2.0 ** -24
    assert ((got_scales - scales).abs() <= 1.01 * step * scales).all() and (got[:, width:] == 0).all()
    assert (got.int() - codes.int()).abs().max() <= 1 + int(2 * 127 * step)
    out, want = torch.empty((n, 24), device="cuda"), torch.empty((n, 24), device="cuda")
    m, s = coded(torch.randn((24, width), generator=gen))
    ops.linear_int8_coded(codes, scales, width, m, s, None, out, ops.STORE)
    from nnis_b200.engine.workspace import Workspace
    ops.linear_int8(normed, m, s, None, want, ops.STORE_F32, Workspace(torch.device("cuda")))
    assert torch.equal(out, want)


@pytest.mark.parametrize("m,n,k,is_coded", [(1, 512, 16384, False), (2, 960, 8192, False), (1, 576, 960, False), (8, 512, 20000, True), (64, 512, 20000, True),
                                           (512, 4096, 2048, True)])
def test_a_matrix_that_was_just_put_into_codes(m, n, k, is_coded):
    """The product right behind the kernel that makes its matrix, in a graph, reads the new codes: products ask for their matrix ahead of
    their wait."""
    from nnis_b200.csrc import ops
    from nnis_b200.engine.workspace import Workspace
    ws, gen = Workspace(torch.device("cuda")), torch.Generator("cuda").manual_seed(n + k)
    x, w = (torch.randn((rows, k), generator=gen, device="cuda").bfloat16() for rows in (m, n))
    (codes, scales), (x_codes, x_scales) = coded(w), coded(x)
    out = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")

    def product():
        if is_coded:
            ops.linear_int8_coded(x_codes, x_scales, k, codes, scales, None, out, ops.STORE)
        else:
            ops.linear_int8(x, codes, scales, None, out, ops.STORE, ws)
    product()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.quantize_rows(w, codes, scales)
        product()
    for _ in range(5):
        w.copy_(torch.randn((n, k), generator=gen, device="cuda").bfloat16())
        torch.cuda.synchronize()
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        product()
        assert torch.equal(got, out)
    del graph


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(300, 997, 64), (131, 65, 100), (1999, 1537, 64), (2050, 1543, 33)])
@pytest.mark.parametrize("mode", [0, 1, 2, 3])
def test_outputs_whose_rows_are_no_multiple_of_16_bytes(dtype, m, n, k, mode):
    """Tiles of one CTA and of pairs, whole and cut off at both ends, that no bulk copy can write."""
    check(dtype, m, n, k, mode, bias=n % 2 == 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(70, 4609, 2050), (129, 2305, 2100), (66, 1000, 1300), (40, 50, 1537), (128, 129, 1200)])
@pytest.mark.parametrize("mode", [0, 1, 2, 3])
def test_tiles_whose_k_several_ctas_share(dtype, m, n, k, mode):
    """In two, three, five and six parts, the last shorter than the others."""
    check(dtype, m, n, k, mode, bias=m % 2 == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,width", [(1, 4), (3, 20), (7, 576), (40, 2048), (2, 8192), (5, 1028), (300, 64)])
def test_a_norm_s_codes_are_the_nearest(dtype, n, width):
    """Every code of a norm's row is the nearest whole number to what the row allows, and the product of these codes is theirs.

    A thread adds width / 256 squares, 13 additions join the threads' sums, and the root halves that error; the mean, the epsilon, the root,
    its inverse, and two products are seven roundings more: less than width / 256 + 24 of 2^-24.  So a value lies between the roundings to
    `dtype` of two numbers that far apart, its quotient by the largest between two quotients, and its code within half a step of those (the
    two roundings of the product with 127 / top: 2^-22 of at most 127)."""
    from nnis_b200.csrc import ops
    gen = torch.Generator().manual_seed(width + n)
    x, w = 3.0 * torch.randn((n, width), generator=gen), 1 + 0.1 * torch.randn(width, generator=gen)
    codes, scales = torch.full((n, ops.int8_width(width)), 77, dtype=torch.int8, device="cuda"), torch.empty(n, device="cuda")
    ops.rmsnorm_int8(x.cuda(), w.cuda(), 1e-5, codes, scales, dtype)
    got, got_scales = codes.cpu()[:, :width].double(), scales.cpu().double()[:, None]
    assert (codes.cpu()[:, width:] == 0).all()
    y = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + 1e-5) * w.double()
    off = (width / 256 + 24) * 2.0 ** -24
    # (rounded from 64 bits at once: through float32 first, a value could fall on the wrong side of a tie)
    ends = [y.abs() * (1 + side * off) for side in (-1, 1)]
    low, high = (round_to(e, dtype) for e in ends)
    top_low, top_high = low.amax(1, keepdim=True), high.amax(1, keepdim=True)
    assert (got_scales >= top_low / 127 * (1 - 2.0 ** -23)).all() and (got_scales <= top_high / 127 * (1 + 2.0 ** -23)).all()
    least, most = 127 * low / top_high - 0.5 - 127 * 2.0 ** -22, 127 * high / top_low + 0.5 + 127 * 2.0 ** -22
    assert (got.abs() >= least).all() and (got.abs() <= most).all() and (torch.sign(got) * torch.sign(y) >= 0).all()
    assert ((most - least) < 1.01 + 254 * off).double().mean() > 0.9  # (few values may fall either way)
    m, s = coded(torch.randn((24, width), generator=gen))
    out = torch.empty((n, 24), device="cuda")
    ops.linear_int8_coded(codes, scales, width, m, s, None, out, ops.STORE)
    want = (got @ m.cpu()[:, :width].double().T) * got_scales * s.cpu().double()
    # (the sum as float32, two products)
    assert ((out.cpu().double() - want).abs() <= 3.01 * 2.0 ** -24 * want.abs() + 1e-37).all()


def round_to(x, dtype):
    """float64 to the nearest number of `dtype` (24 or 8 bits, ties to even), exactly."""
    mantissa, exponent = torch.frexp(x)
    bits = 24 if dtype == torch.float32 else 8
    return torch.ldexp(torch.round(torch.ldexp(mantissa, torch.tensor(bits))), exponent - bits)
