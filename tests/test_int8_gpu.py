"""The 8-bit operators on a B200 against their definitions in 64 bits.

q is compared for equality (its definition has no rounding but the last one); a product differs from its definition by three
fp32 roundings (of the sum, and one for each scale), one more where a bias is added, and half a step of the output's type."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import warpc_public_release_b200 as w  # noqa: E402
from warpc_public_release_b200 import _lib  # noqa: E402
from warpc_public_release_b200._lib import WG_E_ARG, WG_E_VARIANT, WarpcError  # noqa: E402

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U32 = 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def up16(k):
    return -(-k // 16) * 16


# ---------------------------------------------------------------- the product
def operands(m, n, k, seed=0, lda=None, ldb=None, low=-128):
    g = gen(seed)
    a = torch.randint(low, 128, (m, lda or up16(k)), generator=g, device="cuda").to(torch.int8)
    b = torch.randint(low, 128, (n, ldb or up16(k)), generator=g, device="cuda").to(torch.int8)
    sa = torch.exp(torch.randn(m, generator=g, device="cuda")) * 0.02
    sb = torch.exp(torch.randn(n, generator=g, device="cuda")) * 0.002
    return a, b, sa, sb, torch.randn(n, generator=g, device="cuda")


def product64(a, b, sa, sb, k):
    return (a[:, :k].double() @ b[:, :k].double().t()) * sa.double()[:, None] * sb.double()


def check_product(got, a, b, sa, sb, k, out, bias=None):
    ref = product64(a, b, sa, sb, k)
    tol = 3 * U32 * ref.abs()
    if bias is not None:
        ref = ref + bias.double()
        tol = tol + U32 * ref.abs()
    eps = torch.finfo(TYPES[out])
    # half a step of the output's type, of the value before it (itself `tol` off); below the smallest normal, half the smallest step
    tol = tol * 1.001 + eps.eps / 2 * (ref.abs() + tol) + eps.smallest_normal * eps.eps / 2
    over = ref.abs() + tol >= eps.max
    off = (got.double() - ref).abs()
    assert bool(((off <= tol) | over).all()), "largest %g of what is allowed" % float((off / tol)[~over].max())


def run_product(m, n, k, out="bf16", bias=False, program=None, seed=0, ldc=None, shift=0, lda=None, ldb=None):
    a, b, sa, sb, add = operands(m, n, k, seed, lda, ldb)
    ldc = ldc or n
    store = torch.full((m + 2, ldc + 8), -7.0, dtype=TYPES[out], device="cuda")  # what the launch may not write
    flat = store.view(-1)
    plan = w.Int8Plan(n, k, b.data_ptr(), sb.data_ptr(), dBias=add.data_ptr() if bias else None, out=out, ldb=b.shape[1])
    if program:
        plan.set_program(*program)
    plan.set_timeout_ms(1000)
    size = store.element_size()
    plan.launch(m, a.data_ptr(), sa.data_ptr(), store.data_ptr() + shift * size, lda=a.shape[1], ldc=ldc)
    plan.status()
    plan.close()
    got = torch.as_strided(flat, (m, n), (ldc, 1), shift)
    check_product(got, a, b, sa, sb, k, out, add if bias else None)
    got.fill_(-7.0)
    assert bool((store == -7.0).all()), "written outside the output"


PROGRAMS = [("gemv", t, 0, s) for t in (1, 2, 4, 8) for s in (1, 8)] + [("few", t, 128, s) for t in (32, 64) for s in (1, 2, 4, 8)] + \
           [("tile", 256, 256, 1), ("tile", 256, 128, 1), ("tile", 128, 128, 1), ("tile", 128, 64, 1)]


@pytest.mark.parametrize("program", PROGRAMS, ids=lambda p: "-".join(map(str, p)))
@pytest.mark.parametrize("shape", [(1, 1, 1), (5, 37, 130), (77, 300, 1111), (200, 515, 1024), (300, 260, 2049)], ids=lambda s: "x".join(map(str, s)))
def test_every_program_at_ragged_sizes(program, shape):
    m, n, k = shape
    kernel, tile_m, _, split = program
    if kernel == "gemv":
        m = min(m, tile_m)
    if kernel == "few" and split > -(-k // 128):
        pytest.skip("no k-step for every CTA")
    out = ("bf16", "fp16", "fp32")[(m + n + split) % 3]
    run_product(m, n, k, out, bias=bool(n & 1), program=program)


@pytest.mark.parametrize("out", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("program", [("gemv", 2, 0, 2), ("few", 32, 128, 4), ("tile", 256, 256, 1), ("tile", 256, 128, 1), ("tile", 128, 128, 1), ("tile", 128, 64, 1)],
                         ids=lambda p: "-".join(map(str, p)))
@pytest.mark.parametrize("layout", ["aligned", "wide", "stride of 8 bytes", "stride of 4 bytes", "odd stride", "odd start", "odd length"])
def test_output_types_and_layouts(out, program, layout):
    m, n, k = (2 if program[0] == "gemv" else 290), 328, 640
    step = 1 if out == "fp32" else 2
    n = n - 3 if layout == "odd length" else n  # rows in pieces of 8 bytes, the last piece cut
    ldc, shift = {"aligned": (n, 0), "wide": (n + 24, 0), "stride of 8 bytes": (n + 2 * step, 0), "stride of 4 bytes": (n + step, 0), "odd stride": (n + 1, 0),
                  "odd start": (n, 1), "odd length": (n + 3 + 2 * step, 2 * step)}[layout]
    run_product(m, n, k, out, bias=True, program=program, ldc=ldc, shift=shift, lda=k + 48, ldb=k + 16)


@pytest.mark.parametrize("shape", [(1, 4096, 4096), (2, 100, 5000), (3, 4097, 512), (4, 64, 16384), (5, 4096, 4096), (8, 1000, 1000), (9, 2048, 300),
                                   (32, 1024, 4096), (64, 515, 1500), (100, 4096, 1024), (128, 130, 131), (129, 1030, 700), (512, 2048, 1024),
                                   (1000, 1000, 1000), (1024, 1024, 1024), (2300, 1800, 512), (4096, 4096, 256), (70000, 72, 64), (60, 40000, 128)],
                         ids=lambda s: "x".join(map(str, s)))
def test_the_rules_programs(shape):
    run_product(*shape, out=("bf16", "fp32", "fp16")[shape[0] % 3], bias=bool(shape[1] & 2))


@pytest.mark.parametrize("program", [("gemv", 4, 0, 8), ("few", 32, 128, 8), ("tile", 256, 256, 1), ("tile", 128, 64, 1)], ids=lambda p: "-".join(map(str, p)))
@pytest.mark.parametrize("sign", [1, -1])
def test_the_largest_sums_are_exact(program, sign):
    """131071 products of 128 * 128 (and of 127 * -128): the sum stays inside 32 bits and comes out unharmed."""
    m, n, k = 3, 70, 131071
    a = torch.full((m, 131072), -128, dtype=torch.int8, device="cuda")
    b = torch.full((n, 131072), -128 if sign > 0 else 127, dtype=torch.int8, device="cuda")
    one_m, one_n = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    c = torch.zeros(m, n, device="cuda")
    plan = w.Int8Plan(n, k, b.data_ptr(), one_n.data_ptr(), out="fp32", ldb=131072)
    plan.set_program(*program)
    plan.launch(m, a.data_ptr(), one_m.data_ptr(), c.data_ptr(), lda=131072)
    plan.status()
    want = float(np.float32(sign * 128 * (128 if sign > 0 else 127) * k))
    assert bool((c == want).all())


def test_the_same_bits_from_every_program():
    m, n, k = 4, 200, 3000
    a, b, sa, sb, bias = operands(m, n, k)
    plan = w.Int8Plan(n, k, b.data_ptr(), sb.data_ptr(), dBias=bias.data_ptr(), out="fp32", ldb=b.shape[1])
    first = None
    for program in PROGRAMS:
        if program[0] == "gemv" and program[1] < m:
            continue
        plan.set_program(*program)
        for _ in range(2):
            c = torch.full((m, n), float("nan"), device="cuda")
            plan.launch(m, a.data_ptr(), sa.data_ptr(), c.data_ptr(), lda=a.shape[1])
            plan.status()
            first = c if first is None else first
            assert bool((c == first).all()), program


def test_scales_of_zero_infinity_and_nan():
    m, n, k = 140, 70, 256
    for program in (("few", 64, 128, 2), ("tile", 256, 256, 1), ("tile", 128, 64, 1)):
        a, b, sa, sb, _ = operands(m, n, k)
        sa[3], sa[5], sb[7] = 0.0, float("nan"), float("inf")
        c = torch.zeros(m, n, device="cuda")
        plan = w.Int8Plan(n, k, b.data_ptr(), sb.data_ptr(), out="fp32", ldb=b.shape[1])
        plan.set_program(*program)
        plan.launch(m, a.data_ptr(), sa.data_ptr(), c.data_ptr(), lda=a.shape[1])
        plan.status()
        ref = product64(a, b, sa, sb, k)
        assert torch.equal(torch.isnan(c), torch.isnan(ref)) and torch.equal(torch.isinf(c), torch.isinf(ref))
        fine = torch.isfinite(ref)
        assert bool(((c.double() - ref).abs()[fine] <= 4 * U32 * ref.abs()[fine]).all())


def test_a_long_output_passes_32_bit_offsets():
    """Rows of C more than 2^31 elements apart from the first: every program that can write there."""
    n, k, ldc = 64, 64, 1 << 25
    for m, program in ((130, ("tile", 128, 64, 1)), (130, ("tile", 256, 128, 1)), (130, ("few", 64, 128, 1)), (8, ("gemv", 8, 0, 1))):
        ld = ldc if m == 130 else 1 << 29
        a, b, sa, sb, _ = operands(m, n, k)
        c = torch.zeros((m - 1) * ld + n, dtype=torch.bfloat16, device="cuda")
        plan = w.Int8Plan(n, k, b.data_ptr(), sb.data_ptr(), ldb=b.shape[1])
        plan.set_program(*program)
        plan.launch(m, a.data_ptr(), sa.data_ptr(), c.data_ptr(), lda=a.shape[1], ldc=ld)
        plan.status()
        check_product(torch.as_strided(c, (m, n), (ld, 1)), a, b, sa, sb, k, "bf16")
        del c


def test_launches_on_streams_and_in_graphs():
    """One plan on two streams at once, and two captured graphs replayed side by side: nothing is shared between launches."""
    n, k = 1030, 2000
    sets = []
    b, sb = operands(1, n, k)[1], operands(1, n, k)[3]
    plan = w.Int8Plan(n, k, b.data_ptr(), sb.data_ptr(), out="fp32", ldb=b.shape[1])
    for i, m in enumerate((1, 3, 20, 100, 700)):
        a, _, sa, _, _ = operands(m, n, k, seed=i)
        sets.append((m, a, sa, torch.zeros(m, n, device="cuda")))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def go(s, stream):
        m, a, sa, c = s
        plan.launch(m, a.data_ptr(), sa.data_ptr(), c.data_ptr(), lda=a.shape[1], stream=stream.cuda_stream)

    for _ in range(3):
        for i, s in enumerate(sets):
            go(s, streams[i % 2])
    torch.cuda.synchronize()
    for m, a, sa, c in sets:
        check_product(c, a, b, sa, sb, k, "fp32")
        c.zero_()
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(s, torch.cuda.current_stream())
        graphs.append(g)
    for i, g in enumerate(graphs):
        with torch.cuda.stream(streams[i % 2]):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    plan.status()
    for m, a, sa, c in sets:
        check_product(c, a, b, sa, sb, k, "fp32")


def test_launch_refusals_and_no_tokens():
    a, b, sa, sb, _ = operands(4, 64, 64)
    c = torch.full((4, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    plan = w.Int8Plan(64, 64, b.data_ptr(), sb.data_ptr())
    ok = dict(m=4, dA=a.data_ptr(), dScaleA=sa.data_ptr(), dC=c.data_ptr())
    for change in (dict(m=-1), dict(dA=None), dict(dScaleA=None), dict(dC=None), dict(dA=a.data_ptr() + 1), dict(dScaleA=sa.data_ptr() + 2),
                   dict(dC=c.data_ptr() + 1), dict(lda=48), dict(lda=72), dict(ldc=63)):
        with pytest.raises(WarpcError) as e:
            plan.launch(**{**ok, **change})
        assert e.value.code == WG_E_ARG
    plan.launch(0, None, None, None)
    plan.status()
    assert bool((c == 5.0).all())
    for bad in (("gemv", 3, 0, 1), ("gemv", 1, 0, 3), ("few", 32, 64, 1), ("few", 128, 128, 1), ("few", 32, 128, 3), ("few", 32, 128, 2), ("tile", 256, 64, 1), ("tile", 128, 128, 2)):
        with pytest.raises(WarpcError) as e:  # (64 values of K are one k-step: nothing to share)
            plan.set_program(*bad)
        assert e.value.code == WG_E_VARIANT
    plan.set_program("gemv", 2, 0, 1)
    with pytest.raises(WarpcError) as e:
        plan.launch(**ok)
    assert e.value.code == WG_E_VARIANT
    plan.set_program()
    plan.launch(**ok)
    plan.status()
    check_product(c, a, b, sa, sb, 64, "bf16")


# ---------------------------------------------------------------- rows
def rows_of(m, k, dtype, seed, ld=None, shift=0):
    """m rows of k values, `ld` apart, the first `shift` values into its memory: normal, rows of all magnitudes, a few large columns."""
    g = gen(seed)
    ld = ld or k
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp(2 * torch.randn(m, 1, generator=g, device="cuda"))
    x[:, :: max(1, k // 3)] *= 10
    store = torch.full((m * ld + shift + 16,), 3.0, dtype=TYPES[dtype], device="cuda")
    view = torch.as_strided(store, (m, k), (ld, 1), shift)
    view.copy_(x)
    return view


def q_of(t):
    """The definition in 64 bits, of t exact in 64 bits -> (q, max) with rows that cannot be divided as zeros."""
    a = t.abs().amax(1)
    bad = ~torch.isfinite(t).all(1) | (a == 0)
    q = torch.round(t * 127 / a[:, None])
    q[bad] = 0
    return q.to(torch.int8), a


def scale_of(a):
    """a / 127 rounded once to 32 bits.  (A quotient of 24 bits by 7 lies no nearer a border of 32 bits than 2^-32 of it, so the way
    through 64 bits rounds alike; torch's 32-bit division by a number multiplies by 1 / 127 on the GPU, which does not.)"""
    return (a / 127).float()


def run_quantise(x, dtype, ldq=None, qshift=0):
    m, k = x.shape
    ldq = ldq or up16(k)
    store = torch.full((m * ldq + qshift + 32,), 99, dtype=torch.int8, device="cuda")
    scale = torch.full((m + 1,), -1.0, device="cuda")
    w.quantise_rows(m, k, x.data_ptr(), store.data_ptr() + qshift, scale.data_ptr(), dtype=dtype, ldx=x.stride(0), ldq=ldq)
    torch.cuda.synchronize()
    q = torch.as_strided(store, (m, k), (ldq, 1), qshift)
    got = q.clone()
    q.fill_(99)
    assert bool((store == 99).all()) and scale[m] == -1.0, "written outside the output"
    return got, scale[:m]


LENGTHS = [1, 2, 7, 8, 31, 64, 100, 255, 256, 257, 512, 513, 1000, 1111, 2048, 4096, 4100, 8192, 9000, 16384, 16392, 32768, 32769, 70001]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("k", LENGTHS)
def test_quantise_lengths(dtype, k):
    for m in (1, 3, 700):
        if m * k > 30e6:
            continue
        x = rows_of(m, k, dtype, k + m)
        q, scale = run_quantise(x, dtype)
        want, a = q_of(x.double())
        assert torch.equal(q, want)
        assert torch.equal(scale, scale_of(a))  # one division of exact numbers: the same bits


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("ld,shift,ldq,qshift", [(1111, 0, 1120, 0), (1112, 0, 1111, 3), (1200, 8, 1112, 0), (1200, 1, 1112, 8), (1201, 0, 1136, 4), (1204, 0, 1112, 0), (1204, 4, 1120, 4),
                                                  (1202, 2, 1116, 2), (1104, 0, 1104, 0)])
def test_quantise_strides_and_alignment(dtype, ld, shift, ldq, qshift):
    x = rows_of(40, 1104 if ld == 1104 else 1111, dtype, 5, ld, shift)
    q, scale = run_quantise(x, dtype, ldq, qshift)
    want, a = q_of(x.double())
    assert torch.equal(q, want) and torch.equal(scale, scale_of(a))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("k", [5, 200, 1111, 5000])
def test_quantise_special_rows(dtype, k):
    t = torch.finfo(TYPES[dtype])
    x = rows_of(12, k, dtype, 1)
    x[0] = 0
    x[1, k // 2] = float("nan")
    x[2, k - 1] = float("inf")
    x[3, 0] = -float("inf")
    x[4] = t.max
    x[5] = 0
    x[5, k // 3] = t.smallest_normal * t.eps  # the smallest number there is
    x[6] = x[6] * 0 + torch.arange(k, device="cuda").remainder(7).to(x.dtype) * (t.smallest_normal * t.eps)
    x[7] = t.smallest_normal
    x[8] = -x[8].abs()
    x[9] = 0
    x[9, : k // 2] = float("nan")
    q, scale = run_quantise(x, dtype)
    want, a = q_of(x.double())
    assert torch.equal(q, want)
    bad = [1, 2, 3, 9]
    assert bool(torch.isnan(scale[bad]).all()) and scale[0] == 0
    good = [i for i in range(12) if i not in bad]
    assert torch.equal(scale[good], scale_of(a)[good])


def test_quantise_ties_and_neighbours_of_ties():
    """Quotients that are exactly half way between two integers go to the even one; the next numbers either side do not."""
    half = torch.arange(-254, 255, device="cuda", dtype=torch.float32)  # max 254: q = x / 2
    for dtype in ("bf16", "fp16", "fp32"):
        x = half.to(TYPES[dtype]).repeat(3, 1)
        q, _ = run_quantise(x, dtype)
        assert torch.equal(q, torch.round(half.double() / 2).to(torch.int8).repeat(3, 1))
    g = gen(3)
    a = torch.exp(3 * torch.randn(400, 1, generator=g, device="cuda"))
    x = ((torch.arange(-127, 127, device="cuda") + 0.5).double() * a.double() / 127).float()  # as near to half way as 32 bits get
    x = torch.cat([x, torch.nextafter(x, torch.full_like(x, 1e30)), torch.nextafter(x, torch.full_like(x, -1e30)), a], 1).contiguous()
    q, _ = run_quantise(x, "fp32")
    assert torch.equal(q, q_of(x.double())[0])
    y = x.to(torch.bfloat16)
    assert torch.equal(run_quantise(y, "bf16")[0], q_of(y.double())[0])


def norm64(x, r, wt, eps):
    """-> q, scale in 64 bits, h as stored.  The sum is rounded to fp32 and then to the rows' type, the product to fp32: the definition."""
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    t = (h.float() * wt.float()).double()
    q, a = q_of(t)
    return q, a / 127 / torch.sqrt((h.double() ** 2).mean(1) + eps), h


def run_norm(x, r, wt, dtype, eps=1e-6, h=None):
    m, k = x.shape
    ldq = up16(k)
    q = torch.full((m, ldq), 99, dtype=torch.int8, device="cuda")
    scale = torch.empty(m, device="cuda")
    more = {}
    if r is not None:
        h = torch.empty(m, k, dtype=x.dtype, device="cuda") if h is None else h
        more = dict(dR=r.data_ptr(), ldr=r.stride(0), dH=h.data_ptr(), ldh=h.stride(0))
    w.norm_quantise_rows(m, k, x.data_ptr(), wt.data_ptr(), eps, q.data_ptr(), scale.data_ptr(), dtype=dtype, ldx=x.stride(0), ldq=ldq, **more)
    torch.cuda.synchronize()
    assert bool((q[:, k:] == 99).all())
    return q[:, :k], scale, h


def scale_tolerance(k):
    """Of the sum of squares: one rounding per value that a thread adds (at least 64 values or k / 512, and the square's own), ten
    for the lanes and warps; half of that after the root, and six more for the root, the divisions and the mean."""
    return ((max(64, k / 512 + 64) + 10) / 2 + 6) * U32


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("k", LENGTHS)
def test_norm_lengths(dtype, residual, k):
    for m in (1, 3, 700):
        if m * k > 30e6:
            continue
        x = rows_of(m, k, dtype, k + m)
        r = rows_of(m, k, dtype, k + m + 1) if residual else None
        wt = (1 + 0.3 * torch.randn(k, generator=gen(9), device="cuda")).to(TYPES[dtype])
        q, scale, h = run_norm(x, r, wt, dtype)
        want, s, h64 = norm64(x, r, wt, 1e-6)
        if residual:
            assert torch.equal(h, h64)
        assert torch.equal(q, want)
        assert bool(((scale.double() - s).abs() <= scale_tolerance(k) * s).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("ld,shift", [(1111, 0), (1200, 0), (1200, 1), (1201, 8), (1204, 0), (1202, 2)])
def test_norm_strides_and_in_place(dtype, ld, shift):
    """Any stride and start; the sum in its own memory, in the residual's, in x's."""
    k = 1111
    wt = (1 + 0.3 * torch.randn(k + 1, generator=gen(9), device="cuda")).to(TYPES[dtype])[shift % 2: k + shift % 2]
    for where in ("own", "x", "r"):
        x, r = rows_of(50, k, dtype, 1, ld, shift), rows_of(50, k, dtype, 2, ld + 8, shift)
        want, s, h64 = norm64(x, r, wt, 1e-6)
        q, scale, h = run_norm(x, r, wt, dtype, h={"own": None, "x": x, "r": r}[where])
        assert torch.equal(q, want) and torch.equal(h, h64)
        assert bool(((scale.double() - s).abs() <= scale_tolerance(k) * s).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("k", [70, 500, 1029, 2500, 4100, 6003, 8204, 12001, 16390, 33001])
def test_norm_rows_of_every_alignment(dtype, k):
    """Every width of access with every way a row is spread over threads: rows 16, 8, 4 and 2 bytes apart from a boundary."""
    wt = (1 + 0.3 * torch.randn(k, generator=gen(9), device="cuda")).to(TYPES[dtype])
    for m in (5, 400):
        for extra in (0, 1, 2, 4, 8):
            ld = -(-k // 8) * 8 + extra
            x, r = rows_of(m, k, dtype, 1, ld), rows_of(m, k, dtype, 2, ld)
            h = torch.empty(m, ld, dtype=TYPES[dtype], device="cuda")[:, :k]
            for residual in (None, r):
                want, s, h64 = norm64(x, residual, wt, 1e-6)
                q, scale, got = run_norm(x, residual, wt, dtype, h=h if residual is not None else None)
                assert torch.equal(q, want) and (residual is None or torch.equal(got, h64))
                assert bool(((scale.double() - s).abs() <= scale_tolerance(k) * s).all())


@pytest.mark.parametrize("k", [40, 1111, 5000, 40000])
def test_norm_in_place_over_many_rows(k):
    """More rows than blocks: a block's next row is fetched before this one is written."""
    m = 3000 if k < 40000 else 500
    x, r = rows_of(m, k, "bf16", 1), rows_of(m, k, "bf16", 2)
    wt = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    want, s, h64 = norm64(x, r, wt, 1e-5)
    q, scale, h = run_norm(x, r, wt, "bf16", 1e-5, h=r)
    assert torch.equal(q, want) and torch.equal(h, h64)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("k", [6, 1111, 5000, 40000])
def test_norm_special_rows(dtype, k):
    t = torch.finfo(TYPES[dtype])
    x = rows_of(14, k, dtype, 1)
    wt = (1 + 0.3 * torch.randn(k, generator=gen(9), device="cuda")).to(TYPES[dtype])
    wt[k // 2] = 0
    x[0] = 0
    x[1, k // 3] = float("nan")
    x[2, k - 1] = float("inf")
    x[3, k // 2] = -float("inf")       # times a weight of zero: NaN
    x[4] = t.max / 4                    # squares that 32 bits cannot hold (but for fp16)
    x[5] = t.smallest_normal * 4        # squares that 32 bits lose (but for fp16)
    x[6] = 0
    x[6, k // 2] = 5.0                  # all there is is multiplied by zero
    x[7] = 0
    x[7, 0] = 1.0
    q, scale, _ = run_norm(x, None, wt, dtype)
    want, s, _ = norm64(x, None, wt, 1e-6)
    assert torch.equal(q, want)
    assert bool(torch.isnan(scale[[1, 2, 3]]).all()) and scale[0] == 0 and scale[6] == 0
    good = [4, 5, 7, 8, 9, 10, 11, 12, 13]
    assert bool(((scale.double() - s).abs()[good] <= scale_tolerance(k) * s[good]).all())
    q, scale, _ = run_norm(x[4:6].contiguous(), None, wt, dtype, eps=0.0)
    want, s, _ = norm64(x[4:6], None, wt, 0.0)
    assert torch.equal(q, want) and bool(((scale.double() - s).abs() <= scale_tolerance(k) * s).all())


def test_norm_sum_that_leaves_the_type():
    """x + r beyond fp16: an infinity in the stream, so the row has no scale."""
    x = torch.ones(2, 100, dtype=torch.float16, device="cuda")
    x[0, 5] = 60000
    q, scale, h = run_norm(x, x.clone(), torch.ones(100, dtype=torch.float16, device="cuda"), "fp16")
    assert torch.isnan(scale[0]) and bool((q[0] == 0).all()) and torch.isinf(h[0, 5]) and bool(torch.isfinite(scale[1]))


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("tokens", [1, 3, 40, 333])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_a_block_in_8_bits(tokens, dtype):
    """As a model runs them, captured into one graph: norm with the residual, a projection, and (in 8 bits again) the projection back,
    each step against its definition on what the step before wrote, and the whole against the block in 64 bits."""
    d, inner = 712, 1500
    g = gen(tokens)
    kind = TYPES[dtype]
    x, r = (torch.randn(tokens, d, generator=g, device="cuda").to(kind) for _ in range(2))
    wt = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(kind)
    w1 = (torch.randn(inner, d, generator=g, device="cuda") / math.sqrt(d)).to(kind)
    w2 = (torch.randn(d, inner, generator=g, device="cuda") / math.sqrt(inner)).to(kind)

    def eight(m, k):
        return torch.zeros(m, up16(k), dtype=torch.int8, device="cuda"), torch.empty(m, device="cuda")

    q1, s1 = eight(inner, d)
    q2, s2 = eight(d, inner)
    w.quantise_rows(inner, d, w1.data_ptr(), q1.data_ptr(), s1.data_ptr(), dtype=dtype, ldq=up16(d))
    w.quantise_rows(d, inner, w2.data_ptr(), q2.data_ptr(), s2.data_ptr(), dtype=dtype, ldq=up16(inner))
    p1 = w.Int8Plan(inner, d, q1.data_ptr(), s1.data_ptr(), out=dtype, ldb=up16(d))
    p2 = w.Int8Plan(d, inner, q2.data_ptr(), s2.data_ptr(), out=dtype, ldb=up16(inner))
    qa, sa = eight(tokens, d)
    qb, sb = eight(tokens, inner)
    h, y, z = (torch.empty(tokens, c, dtype=kind, device="cuda") for c in (d, inner, d))

    def block():
        s = torch.cuda.current_stream().cuda_stream
        w.norm_quantise_rows(tokens, d, x.data_ptr(), wt.data_ptr(), 1e-5, qa.data_ptr(), sa.data_ptr(), dR=r.data_ptr(), dH=h.data_ptr(), dtype=dtype,
                             ldq=up16(d), stream=s)
        p1.launch(tokens, qa.data_ptr(), sa.data_ptr(), y.data_ptr(), lda=up16(d), stream=s)
        w.quantise_rows(tokens, inner, y.data_ptr(), qb.data_ptr(), sb.data_ptr(), dtype=dtype, ldq=up16(inner), stream=s)
        p2.launch(tokens, qb.data_ptr(), sb.data_ptr(), z.data_ptr(), lda=up16(inner), stream=s)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block()
    graph.replay()
    torch.cuda.synchronize()
    p1.status(), p2.status()
    want, s, h64 = norm64(x, r, wt, 1e-5)
    assert torch.equal(qa[:, :d], want) and torch.equal(h, h64)
    check_product(y, qa, q1, sa, s1, d, dtype)
    assert torch.equal(qb[:, :inner], q_of(y.double())[0])
    check_product(z, qb, q2, sb, s2, inner, dtype)
    # the block without 8 bits: three quantisations of operands (half a step of 127 at the largest value, in both operands of each product) --
    # a value's error is below max / 254, so relative to the root mean square of normal values (max < 5 of them) below 2 % an operand
    n = h64.double()
    n = n / torch.sqrt((n ** 2).mean(1, keepdim=True) + 1e-5) * wt.double()
    full = (n @ w1.double().t()) @ w2.double().t()
    assert float((z.double() - full).norm() / full.norm()) < 4 * 0.02 + 2 * torch.finfo(kind).eps
    first = z.clone()
    block()
    torch.cuda.synchronize()
    assert torch.equal(z, first)


def test_order_of_launches_in_a_stream():
    """Launches may be set up while the one before them ends: each step's buffers are rewritten by the next step without a
    synchronisation between them, weights just before the product that reads them, and every step's result is kept."""
    n, k, steps = 300, 700, 40
    ld = up16(k)
    g = gen(11)
    for m in (1, 20, 90, 300):
        xs = torch.randn(steps, m, k, generator=g, device="cuda").to(torch.bfloat16)
        ws = torch.randn(steps, n, k, generator=g, device="cuda").to(torch.bfloat16)
        wt = torch.ones(k, dtype=torch.bfloat16, device="cuda")
        x, r, qa, sa = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(m, k, dtype=torch.bfloat16, device="cuda"), \
            torch.zeros(m, ld, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda")
        b, qb, sb = torch.zeros(n, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, ld, dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
        y = torch.zeros(m, n, device="cuda")
        plan = w.Int8Plan(n, k, qb.data_ptr(), sb.data_ptr(), out="fp32", ldb=ld)

        def run(wait):
            kept = []
            r.zero_()
            for i in range(steps):
                x.copy_(xs[i])
                b.copy_(ws[i])
                w.quantise_rows(n, k, b.data_ptr(), qb.data_ptr(), sb.data_ptr(), ldq=ld)
                wait()
                w.norm_quantise_rows(m, k, x.data_ptr(), wt.data_ptr(), 1e-6, qa.data_ptr(), sa.data_ptr(), dR=r.data_ptr(), dH=r.data_ptr(), ldq=ld)
                wait()
                plan.launch(m, qa.data_ptr(), sa.data_ptr(), y.data_ptr(), lda=ld)
                wait()
                kept.append(y.clone())
                plan.launch(m, qa.data_ptr(), sa.data_ptr(), y.data_ptr(), lda=ld)  # over what the copy reads
            torch.cuda.synchronize()
            return torch.stack(kept)

        apart = run(torch.cuda.synchronize)
        assert torch.equal(run(lambda: None), apart)
        plan.status()


def test_first_calls_of_a_process_inside_a_capture():
    """A process whose first launches are captured: nothing has to have run before (limits raised and code loaded in the capture)."""
    import os
    import subprocess
    import sys
    code = """
import torch, warpc_public_release_b200 as w
m, k, n = 400, 8192, 256
x = torch.randn(m, k, device="cuda").bfloat16(); f = torch.randn(m, k, device="cuda"); wt = torch.ones(k, device="cuda").bfloat16()
q, q2, s = torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.zeros(m, device="cuda")
s2, b, sb = torch.zeros(m, device="cuda"), torch.ones(n, k, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda")
y, y1 = torch.zeros(m, n, device="cuda"), torch.zeros(3, n, device="cuda")
plan = w.Int8Plan(n, k, b.data_ptr(), sb.data_ptr(), out="fp32")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    st = torch.cuda.current_stream().cuda_stream
    w.norm_quantise_rows(m, k, x.data_ptr(), wt.data_ptr(), 1e-6, q.data_ptr(), s.data_ptr(), stream=st)
    w.quantise_rows(m, k, f.data_ptr(), q2.data_ptr(), s2.data_ptr(), dtype="fp32", stream=st)
    plan.launch(m, q.data_ptr(), s.data_ptr(), y.data_ptr(), stream=st)
    plan.launch(3, q2.data_ptr(), s2.data_ptr(), y1.data_ptr(), stream=st)
g.replay(); torch.cuda.synchronize(); plan.status()
assert torch.allclose(y, (q.double().sum(1) * s.double()).float()[:, None].expand(m, n), rtol=1e-6)
assert torch.allclose(y1, (q2[:3].double().sum(1) * s2[:3].double()).float()[:, None].expand(3, n), rtol=1e-6)
plan.reset()
print("captured")
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=200)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("args", [["1", "300", "1111"], ["70", "260", "500", "2", "--norm"], ["300", "512", "640", "3", "--norm", "--out", "fp32"],
                                  ["5", "64", "64", "1", "--out", "fp16"]], ids=" ".join)
def test_the_command(args, capsys):
    from warpc_public_release_b200 import run_int8
    assert run_int8.main(args) == 0
    assert " MATCH bad=0/" in capsys.readouterr().out
