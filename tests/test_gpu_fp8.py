"""Block quantisation to 8-bit floating point and the GEMM of such operands on the GPU, against their formulas in 64 bits.

Quantisation: the scale is a power of two, so the value is rounded once: results are equal, not near.
GEMM: with S = sum over blocks of |sa sb| sum |a b|, a block's 128 products are exact in fp32 and each addition is off by at
most one fp32 step (2^-23: a tensor core may cut instead of rounding), the two products with scales by half a step each, the sum over nb
blocks by nb half steps: (128 + nb + 2) 2^-23 S in all; alpha, beta and bias by half a step of what they give; the
result by half a step of its type.
"""
import numpy as np
import pytest

from accera_b200 import runtime as rt

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FORMAT = {"e4m3": (3, -6, 448.0), "e5m2": (2, -14, 57344.0)}


def _up(a, b):
    return -(-a // b)


def _quantize_want(x, kind, block):
    """(q, s) in float64 from the definition; x float64 on the CPU"""
    bits, low, top = FORMAT[kind]
    m, k = x.shape
    q, s = np.zeros((m, k)), np.zeros((_up(m, block), _up(k, 128)))
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            g = x[i * block:(i + 1) * block, j * 128:(j + 1) * 128]
            amax = np.abs(g[np.isfinite(g)]).max(initial=0.0)
            e = -200
            while amax > top * 2.0 ** e:
                e += 1
            s[i, j] = 2.0 ** min(max(e, -126), 127) if amax > 0 else 1.0
            y = g / s[i, j]
            with np.errstate(invalid="ignore"):
                step = 2.0 ** (np.maximum(np.frexp(y)[1] - 1, low) - bits)
                r = np.round(y / step) * step
            q[i * block:(i + 1) * block, j * 128:(j + 1) * 128] = np.where(np.isfinite(g), r, np.nan)
    return q, s


def _same(a, b):
    return np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.nan_to_num(a), np.nan_to_num(b))


def _values(m, k, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(3 * torch.randn(m, 1, generator=g)) * torch.exp(3 * torch.randn(1, k, generator=g))
    return x.clamp(-60000, 60000)


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("to", ["e4m3", "e5m2"])
@pytest.mark.parametrize("m,k", [(1, 128), (1, 1), (3, 127), (129, 129), (128, 256), (40, 1000), (260, 392), (1, 5000)])
def test_quantisation_equals_the_formula(block, src, to, m, k):
    x = _values(m, k, m * 1000 + k).to(TYPES[src])
    want = _quantize_want(x.double().numpy(), to, block)
    for across in (False, True):
        xd = x.t().contiguous().cuda().t() if across else x.cuda()
        q = torch.zeros(m, k, dtype=TYPES[to], device="cuda")
        s = torch.zeros(_up(m, block), _up(k, 128), device="cuda")
        rt.quantize_fp8(xd, q, s)
        rt.synchronize()
        assert _same(s.cpu().double().numpy(), want[1]), (across, "scales")
        assert _same(q.cpu().double().numpy(), want[0]), (across, "values")


def test_quantisation_borders_and_special_values():
    top = 448.0
    rows = [
        [top, 1.0], [np.nextafter(np.float32(top), np.float32(1e9)), 1.0], [0.0, -0.0], [np.inf, 3.0], [-np.inf, np.nan],
        [2.0 ** -140, 2.0 ** -149], [3.4e38, -3.4e38], [2.0 ** -126, 2.0 ** -133], [17.0, 19.0], [1.0625, 1.1875], [-0.0, 2.0 ** -9],
    ]
    x = torch.zeros(len(rows), 130)
    for i, r in enumerate(rows):
        x[i, :2] = torch.tensor(r, dtype=torch.float64).float()
        x[i, 2] = float(r[0]) / 16 + float(r[0]) / 256 if np.isfinite(r[0]) else 0.0            # halfway values
    want = _quantize_want(x.double().numpy(), "e4m3", 1)
    q = torch.empty(len(rows), 130, dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty(len(rows), 2, device="cuda")
    rt.quantize_fp8(x.cuda(), q, s)
    rt.synchronize()
    assert _same(s.cpu().double().numpy(), want[1]) and _same(q.cpu().double().numpy(), want[0])
    assert torch.equal(torch.signbit(q.cpu().float()[2, :2]), torch.tensor([False, True]))


@pytest.mark.parametrize("across", [False, True])
def test_quantisation_strides_leave_the_rest_alone(across):
    m, k = 70, 300
    x = _values(k if across else m, (m if across else k) + 9, 1).to(torch.bfloat16).cuda()
    x = x[:, 3:-6].t() if across else x[:, 3:-6]                     # unaligned rows, a pitch that is no multiple of 16 bytes
    want = _quantize_want(x.cpu().double().numpy(), "e5m2", 1)
    q = torch.full((m, 333), 2.0, device="cuda").to(torch.float8_e5m2)
    s = torch.full((3, 75), 9.0, device="cuda")
    rt.quantize_fp8(x, q[:, 1:301], s[:, :70].t())
    rt.synchronize()
    assert _same(q[:, 1:301].cpu().double().numpy(), want[0]) and _same(s[:, :70].t().cpu().double().numpy(), want[1])
    rest = torch.cat([q[:, :1], q[:, 301:]], 1).float()
    assert (rest == 2).all() and (s[:, 70:] == 9).all()
    every_second = torch.randn(40, 512, device="cuda")[:, ::2]         # no contiguous direction
    want = _quantize_want(every_second.cpu().double().numpy(), "e4m3", 128)
    q, s = torch.empty(40, 256, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(1, 2, device="cuda")
    rt.quantize_fp8(every_second, q, s)
    rt.synchronize()
    assert _same(q.cpu().double().numpy(), want[0]) and _same(s.cpu().double().numpy(), want[1])


def _operands(m, n, k, a, b, ga, gb, seed):
    """A [m, k], sa, B [n, k], sb with arbitrary fp32 scales, on the CPU"""
    g = torch.Generator().manual_seed(seed)
    A = (torch.randn(m, k, generator=g) * 40).to(TYPES[a])
    B = (torch.randn(n, k, generator=g) * 40).to(TYPES[b])
    sa = torch.exp(2 * torch.randn(_up(m, ga), _up(k, 128), generator=g))
    sb = torch.exp(2 * torch.randn(_up(n, gb), _up(k, 128), generator=g)) * 0.01
    return A, sa, B, sb


def _gemm_want(A, sa, B, sb, ga, gb, old=None, alpha=1.0, beta=0.0, bias=None, relu=False):
    """-> exact result, error bound of the fp32 arithmetic"""
    m, k = A.shape
    n = B.shape[0]
    c, size = torch.zeros(m, n, dtype=torch.float64), torch.zeros(m, n, dtype=torch.float64)
    nb = _up(k, 128)
    for j in range(nb):
        x, y = A[:, j * 128:(j + 1) * 128].double(), B[:, j * 128:(j + 1) * 128].double()
        f = sa[:, j].double().repeat_interleave(ga)[:m, None] * sb[:, j].double().repeat_interleave(gb)[None, :n]
        c += f * (x @ y.t())
        size += f.abs() * (x.abs() @ y.abs().t())
    err = abs(alpha) * (128 + nb + 2) * 2.0 ** -23 * size
    c = alpha * c
    steps = c.abs()
    if beta:
        c = c + beta * old.double()
        steps = steps + beta * old.double().abs() + c.abs()
    if bias is not None:
        c = c + bias.double()
        steps = steps + c.abs()
    err = err + 2.0 ** -24 * steps * 1.001
    return (torch.relu(c) if relu else c), err


def _check(got, want, err, what):
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    off = (got.double() - want).abs()
    bad = ~(off <= err * (1 + half) + half * want.abs() + tiny)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, rows {bad.any(1).nonzero().flatten()[:8].tolist()}, columns "
                           f"{bad.any(0).nonzero().flatten()[:8].tolist()}: got {got[bad][0]}, want {want[bad][0]}, bound {err[bad][0]}")


def _run(A, sa, B, sb, ga, gb, c_type, layout="tn", compute="auto", **kw):
    """layout: contiguous direction of A and of B, 't' = along K, 'n' = along M / N"""
    Ad = A.cuda() if layout[0] == "t" else A.t().contiguous().cuda().t()
    Bd = B.cuda().t() if layout[1] == "n" else B.t().contiguous().cuda()
    old = kw.pop("old", None)
    C = old.clone().cuda() if old is not None else torch.full((A.shape[0], B.shape[0]), float("nan"), dtype=TYPES[c_type], device="cuda")
    bias = kw.pop("bias", None)
    rt.gemm_fp8(Ad, Bd, C, sa.cuda(), sb.cuda().t(), beta=kw.pop("beta", 0.0), bias=None if bias is None else bias.cuda(), compute=compute, **kw)
    rt.synchronize()
    return C.cpu()


# tokens from one to a few tiles, sides around tile borders, K around block borders, K that TMA cannot take directly
SHAPES = [(1, 128, 128), (1, 1, 1), (2, 130, 300), (7, 264, 512), (16, 200, 129), (17, 512, 1024), (33, 96, 127), (64, 640, 2048),
          (65, 129, 48), (100, 256, 1000), (127, 1000, 16), (128, 128, 256), (129, 255, 384), (200, 300, 640), (256, 256, 1152), (300, 520, 4096)]


# every kernel takes every shape: which one runs is a matter of speed alone
PATHS = {"auto": {}, "simt": {}, "pair": {"gemm_fp8.kernel": 1, "gemm_fp8.slices": 1}, "pair4": {"gemm_fp8.kernel": 1, "gemm_fp8.slices": 4}, "tile": {"gemm_fp8.kernel": 2, "gemm_fp8.slices": 1},
         "tile2": {"gemm_fp8.kernel": 2, "gemm_fp8.slices": 2}, "tile8": {"gemm_fp8.kernel": 2, "gemm_fp8.slices": 8}}


@pytest.mark.parametrize("path", list(PATHS))
@pytest.mark.parametrize("ga,gb", [(1, 128), (1, 1), (128, 128), (128, 1)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm_equals_the_formula(path, ga, gb, m, n, k):
    A, sa, B, sb = _operands(m, n, k, "e4m3", "e4m3", ga, gb, m + n + k)
    want, err = _gemm_want(A, sa, B, sb, ga, gb)
    with rt.options(**PATHS[path]):
        got = _run(A, sa, B, sb, ga, gb, "f32", compute="simt" if path == "simt" else "tensor" if path != "auto" else "auto")
    _check(got, want, err, (path, ga, gb))


@pytest.mark.parametrize("a,b", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("c", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["tn", "tt", "nn", "nt"])
@pytest.mark.parametrize("path,m,n,k", [("tile", 9, 144, 272), ("tile8", 144, 272, 1040), ("pair", 272, 400, 528), ("pair4", 272, 400, 1040)])
def test_gemm_types_and_layouts(a, b, c, layout, path, m, n, k):
    A, sa, B, sb = _operands(m, n, k, a, b, 1, 128, 3)
    sb *= 0.001                                                        # inside fp16's range
    want, err = _gemm_want(A, sa, B, sb, 1, 128)
    assert want.abs().max() < 60000
    with rt.options(**PATHS[path]):
        got = _run(A, sa, B, sb, 1, 128, c, layout, compute="tensor")
    _check(got, want, err, (a, b, c, layout))


@pytest.mark.parametrize("alpha,beta,relu,use_bias", [(1.0, 1.0, False, False), (0.5, 0.0, True, True), (-2.0, 0.25, False, True), (1.0, 1.0, True, True)])
@pytest.mark.parametrize("c", ["f32", "bf16"])
@pytest.mark.parametrize("path", ["pair", "pair4", "tile", "tile8", "simt"])
@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (40, 203, 300), (200, 264, 768), (520, 512, 256)])
def test_gemm_epilogue(alpha, beta, relu, use_bias, c, path, m, n, k):
    A, sa, B, sb = _operands(m, n, k, "e4m3", "e4m3", 1, 128, 4)
    old = (torch.randn(m, n) * 100).to(TYPES[c])
    bias = torch.randn(n) * 100 if use_bias else None
    want, err = _gemm_want(A, sa, B, sb, 1, 128, old, alpha, beta, bias, relu)
    with rt.options(**PATHS[path]):
        got = _run(A, sa, B, sb, 1, 128, c, old=old, alpha=alpha, beta=beta, relu=relu, bias=bias, compute="simt" if path == "simt" else "auto")
    _check(got, want, err, "epilogue")


@pytest.mark.parametrize("path,m,n,k", [("tile", 3, 130, 256), ("tile2", 200, 300, 384), ("pair", 200, 300, 384), ("pair4", 200, 300, 512)])
def test_gemm_result_strides_leave_the_rest_alone(path, m, n, k):
    A, sa, B, sb = _operands(m, n, k, "e4m3", "e4m3", 1, 128, 5)
    want, err = _gemm_want(A, sa, B, sb, 1, 128)
    for make in (lambda: torch.full((m, n + 5), 7.0, device="cuda")[:, 2:n + 2], lambda: torch.full((n + 3, m + 1), 7.0, device="cuda")[1:n + 1, :m].t(),
                 lambda: torch.full((m, 2 * n), 7.0, device="cuda")[:, ::2]):
        C = make()
        base = C._base if C._base is not None else C
        with rt.options(**PATHS[path]):
            rt.gemm_fp8(A.cuda(), B.cuda().t(), C, sa.cuda(), sb.cuda().t(), beta=0.0)
        rt.synchronize()
        _check(C.cpu(), want, err, tuple(C.stride()))
        left = base.clone()
        left.as_strided(C.shape, C.stride(), C.storage_offset()).fill_(7.0)
        assert (left == 7).all()


def test_gemm_operands_without_aligned_rows_and_views():
    m, n, k = 70, 200, 515
    A, sa, B, sb = _operands(m, n, k + 20, "e4m3", "e5m2", 1, 1, 6)
    Av, Bv = A.cuda()[:, 5:5 + k], B.cuda()[:, 3:3 + k]               # pitch 535, odd offsets
    want, err = _gemm_want(A[:, 5:5 + k], sa[:, :5], B[:, 3:3 + k], sb[:, :5], 1, 1)
    C = torch.empty(m, n, device="cuda")
    rt.gemm_fp8(Av, Bv.t(), C, sa.cuda()[:, :5], sb.cuda()[:, :5].t(), beta=0.0)
    rt.synchronize()
    _check(C.cpu(), want, err, "views")
    Ax = torch.zeros(m, 2 * k).to(torch.float8_e4m3fn).cuda()[:, ::2]  # no contiguous direction: the CUDA-core kernel
    Ax.copy_(Av)
    rt.gemm_fp8(Ax, Bv.t(), C, sa.cuda()[:, :5], sb.cuda()[:, :5].t(), beta=0.0)
    rt.synchronize()
    _check(C.cpu(), want, err, "strided")
    with pytest.raises(rt.AccbError):
        rt.gemm_fp8(Ax, Bv.t(), C, sa.cuda()[:, :5], sb.cuda()[:, :5].t(), beta=0.0, compute="tensor")


def test_gemm_empty_k_and_special_scales():
    old = torch.randn(5, 300, device="cuda").to(torch.bfloat16)
    want = torch.relu(old.double() * 0.5 + 1.0)
    C = old.clone()
    e = torch.zeros(5, 0, device="cuda").to(torch.float8_e4m3fn)
    f = torch.zeros(0, 300, device="cuda").to(torch.float8_e4m3fn)
    z = torch.zeros(5, 0, device="cuda")
    rt.gemm_fp8(e, f, C, z, torch.zeros(0, 3, device="cuda"), alpha=2.0, beta=0.5, bias=torch.ones(300, device="cuda"), relu=True)
    rt.synchronize()
    assert torch.equal(C, want.to(torch.bfloat16))
    rt.gemm_fp8(e[:0], f, C[:0], z[:0], torch.zeros(0, 3, device="cuda"))
    # NaN and infinities stay in their row or column; rows behind the matrix edge bring nothing in
    m, n, k = 150, 300, 260
    A, sa, B, sb = _operands(m, n, k, "e4m3", "e4m3", 1, 1, 7)
    A[3, 5] = float("nan")
    sa[9, 1] = float("inf")
    sa[20, 0] = 0.0
    sb[17, 2] = float("nan")
    for path in PATHS:
        with rt.options(**PATHS[path]):
            got = _run(A, sa, B, sb, 1, 1, "f32", compute="simt" if path == "simt" else "auto")
        _check_broken(got, m, n)


def _check_broken(got, m, n):
    broken = torch.zeros(m, n, dtype=torch.bool)
    broken[3] = broken[9] = True
    broken[:, 17] = True
    assert torch.equal(got.isfinite(), ~broken)


@pytest.mark.parametrize("m,n,k", [(4, 512, 1024), (600, 512, 1024)])
def test_gemm_streams_graphs_and_equal_bits(m, n, k):
    A, sa, B, sb = [t.cuda() for t in _operands(m, n, k, "e4m3", "e4m3", 1, 128, 8)]
    want = torch.empty(m, n, device="cuda")
    rt.gemm_fp8(A, B.t(), want, sa, sb.t(), beta=0.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [torch.empty(m, n, device="cuda") for _ in range(2)]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                rt.gemm_fp8(A, B.t(), got[i], sa, sb.t(), beta=0.0)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], want)
    graphs = []
    for i in range(2):
        got[i].fill_(1.0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            rt.gemm_fp8(A, B.t(), got[i], sa, sb.t(), beta=0.0)
        graphs.append(g)
    for i in (0, 1, 0):
        with torch.cuda.stream(streams[i]):
            graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], want)


@pytest.mark.parametrize("path", ["pair", "tile", "tile2"])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(path):
    A, sa, B, sb = _operands(150, 300, 512, "e4m3", "e4m3", 1, 1, 10)
    want, err = _gemm_want(A, sa, B, sb, 1, 1)
    rt.synchronize()
    with rt.options(**PATHS[path], **{"gemm.test_drop_commit": 1, "gemm.wait_limit_us": 20000}):
        C = torch.zeros(150, 300, device="cuda")
        rt.gemm_fp8(A.cuda(), B.cuda().t(), C, sa.cuda(), sb.cuda().t(), beta=0.0)
        with pytest.raises(rt.AccbError) as e:
            rt.synchronize()
        assert e.value.code == rt.ERR_TIMEOUT and "epilogue waiting" in str(e.value)
    with rt.options(**PATHS[path]):
        _check(_run(A, sa, B, sb, 1, 1, "f32"), want, err, path)


@pytest.mark.parametrize("max_ctas", [1, 2, 7, 1000])
def test_gemm_on_a_bounded_grid(max_ctas):
    A, sa, B, sb = _operands(700, 600, 640, "e4m3", "e4m3", 1, 128, 11)
    want, err = _gemm_want(A, sa, B, sb, 1, 128)
    _check(_run(A, sa, B, sb, 1, 128, "bf16", max_ctas=max_ctas), want, err, max_ctas)


def test_scales_in_any_layout():
    # four blocks' scales of a row side by side and aligned, the same unaligned, block-major, and every second value
    m, n, k = 300, 520, 2048
    A, sa, B, sb = _operands(m, n, k, "e4m3", "e4m3", 1, 1, 12)
    want, err = _gemm_want(A, sa, B, sb, 1, 1)
    Ad, Bd = A.cuda(), B.cuda().t()
    for make in (lambda s: s.cuda(), lambda s: torch.zeros(s.shape[0], s.shape[1] + 3, device="cuda")[:, 1:17].copy_(s), lambda s: s.t().contiguous().cuda().t(),
                 lambda s: torch.zeros(s.shape[0], 2 * s.shape[1], device="cuda")[:, ::2].copy_(s)):
        for path in ("pair", "pair4", "tile", "simt"):
            C = torch.zeros(m, n, device="cuda")
            with rt.options(**PATHS[path]):
                rt.gemm_fp8(Ad, Bd, C, make(sa), make(sb).t(), beta=0.0, compute="simt" if path == "simt" else "auto")
            rt.synchronize()
            _check(C.cpu(), want, err, (path, make(sa).stride()))


def test_host_arrays():
    rng = np.random.default_rng(2)
    x = rng.standard_normal((33, 300), dtype=np.float32)
    w = rng.standard_normal((70, 300), dtype=np.float32)
    qx, sx = np.zeros((33, 300), np.uint8), np.zeros((33, 3), np.float32)
    qw, sw = np.zeros((70, 300), np.uint8), np.zeros((1, 3), np.float32)
    rt.quantize_fp8(x, qx, sx, q_kind="float8_e4m3")
    rt.quantize_fp8(w, qw, sw, q_kind="float8_e4m3")
    want, s = _quantize_want(x.astype(np.float64), "e4m3", 1)
    as_values = lambda q: torch.from_numpy(q).view(torch.float8_e4m3fn)
    assert _same(as_values(qx).double().numpy(), want) and _same(sx.astype(np.float64), s)
    c = np.zeros((33, 70), np.float32)
    rt.gemm_fp8(qx, qw.T, c, sx, sw.T, beta=0.0, a_kind="float8_e4m3", b_kind="float8_e4m3")
    want, err = _gemm_want(as_values(qx), torch.from_numpy(sx), as_values(qw), torch.from_numpy(sw), 1, 128)
    _check(torch.from_numpy(c), want, err, "host")


def test_a_tied_table_trained_one_step():
    """Lookup, head product in 8 bits, both gradients of the head's product, and the table's gradient from both uses, each held
    to the formula on the inputs that it got."""
    vocab, dim, tokens = 520, 256, 200
    g = torch.Generator().manual_seed(9)
    table = torch.randn(vocab, dim, generator=g)
    ids = torch.randint(0, vocab, (tokens,), generator=g)
    dy = torch.randn(tokens, vocab, generator=g).to(torch.bfloat16)
    td, idd, dyd = table.cuda(), ids.cuda(), dy.cuda()
    f8 = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.float8_e4m3fn)
    f32 = lambda *s: torch.zeros(*s, device="cuda")
    x = torch.empty(tokens, dim, device="cuda", dtype=torch.bfloat16)
    rt.embedding(td, idd, x, scale=dim ** 0.5)
    qx, sx, qw, sw = f8(tokens, dim), f32(tokens, 2), f8(vocab, dim), f32(_up(vocab, 128), 2)
    rt.quantize_fp8(x, qx, sx)
    rt.quantize_fp8(td, qw, sw)
    logits = f32(tokens, vocab)
    rt.gemm_fp8(qx, qw.t(), logits, sx, sw.t(), beta=0.0)
    # gradient of the head's input: contraction over the vocabulary, the weights read along their other direction
    qdy, sdy = torch.zeros(tokens, vocab, device="cuda", dtype=torch.float8_e5m2), f32(tokens, 5)
    rt.quantize_fp8(dyd, qdy, sdy)
    dx = torch.empty(tokens, dim, device="cuda", dtype=torch.bfloat16)
    rt.gemm_fp8(qdy, qw, dx, sdy, sw, beta=0.0)
    # gradient of the table as head weights (contraction over the tokens), then as lookup table, added
    qdyt, sdyt = torch.zeros(vocab, tokens, device="cuda", dtype=torch.float8_e5m2), f32(vocab, 2)
    qxt, sxt = f8(dim, tokens), f32(dim, 2)
    rt.quantize_fp8(dyd.t(), qdyt, sdyt)
    rt.quantize_fp8(x.t(), qxt, sxt)
    dw = f32(vocab, dim)
    rt.gemm_fp8(qdyt, qxt.t(), dw, sdyt, sxt.t(), beta=0.0)
    head = dw.cpu()
    rt.embedding_grad(dx, idd, dw, scale=dim ** 0.5, beta=1.0)
    rt.synchronize()
    assert torch.equal(x.cpu(), (table[ids] * dim ** 0.5).to(torch.bfloat16))
    cpu = lambda *t: [v.cpu() for v in t]
    _check(logits.cpu(), *_gemm_want(*cpu(qx, sx, qw, sw), 1, 128), "logits")
    qwt, swt = qw.t().contiguous(), sw.t().contiguous()
    want = torch.zeros(tokens, dim, dtype=torch.float64)
    size = torch.zeros(tokens, dim, dtype=torch.float64)
    for j in range(5):
        rows = slice(j * 128, (j + 1) * 128)
        f = sdy[:, j].cpu().double()[:, None] * sw[j].cpu().double().repeat_interleave(128)[None, :dim]
        want += f * (qdy[:, rows].cpu().double() @ qw[rows].cpu().double())
        size += f * (qdy[:, rows].cpu().double().abs() @ qw[rows].cpu().double().abs())
    _check(dx.cpu(), want, (128 + 5 + 2) * 2.0 ** -23 * size, "input gradient")
    _check(head, *_gemm_want(*cpu(qdyt, sdyt, qxt, sxt), 1, 1), "weight gradient")
    both = head.double().index_add(0, ids, dx.cpu().double() * dim ** 0.5)
    size = head.double().abs().index_add(0, ids, dx.cpu().double().abs() * dim ** 0.5)
    assert ((dw.cpu().double() - both).abs() <= tokens * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("ga,gb", [(1, 128), (1, 1)])
@pytest.mark.parametrize("path,k,dropped", [("pair", 1152, "scales"), ("pair", 512, "scales"), ("pair4", 4096, "scales"), ("tile", 1152, "scales"),
                                            ("tile8", 4096, "scales"), ("pair4", 4096, "commit"), ("tile8", 4096, "commit")])
def test_scales_and_slices_that_never_arrive_are_reported(path, k, dropped, ga, gb):
    # 9 blocks of K (8 a slice with four slices): the last slot of scales begins behind blocks whose sums are on their way
    m, n = 300, 520
    A, sa, B, sb = _operands(m, n, k, "e4m3", "e4m3", ga, gb, 13)
    want, err = _gemm_want(A, sa, B, sb, ga, gb)
    rt.synchronize()
    drop = {"scales": "gemm_fp8.test_drop_scales", "commit": "gemm.test_drop_commit"}[dropped]
    with rt.options(**PATHS[path], **{drop: 1, "gemm.wait_limit_us": 20000}):
        C = torch.zeros(m, n, device="cuda")
        rt.gemm_fp8(A.cuda(), B.cuda().t(), C, sa.cuda(), sb.cuda().t(), beta=0.0)
        with pytest.raises(rt.AccbError) as e:
            rt.synchronize()
        # (behind scales that never come the MMA's wait for a free accumulator may run out first)
        assert e.value.code == rt.ERR_TIMEOUT and (dropped == "scales" or "waiting for the accumulator" in str(e.value))
    with rt.options(**PATHS[path]):
        _check(_run(A, sa, B, sb, ga, gb, "f32"), want, err, path)


@pytest.mark.parametrize("path", ["pair", "pair4", "tile", "auto"])
@pytest.mark.parametrize("step", [16, 48, 1, 7])
def test_gemm_operands_whose_rows_overlap(path, step):
    # windows of a longer signal: rows of A 16, 48, 1 or 7 bytes apart; the same for the columns of B
    m, n, k = 90, 150, 520
    g = torch.Generator().manual_seed(14)
    signal = [(torch.randn(max(m, n) * step + k, generator=g) * 40).to(torch.float8_e4m3fn).cuda() for _ in range(2)]
    A, B = signal[0].as_strided((m, k), (step, 1)), signal[1].as_strided((n, k), (step, 1))
    _, sa, _, sb = _operands(m, n, k, "e4m3", "e4m3", 1, 128, 15)
    Ac, Bc = A.cpu().contiguous(), B.cpu().contiguous()
    want, err = _gemm_want(Ac, sa, Bc, sb, 1, 128)
    C = torch.full((m, n), float("nan"), device="cuda")
    with rt.options(**PATHS[path]):
        rt.gemm_fp8(A, B.t(), C, sa.cuda(), sb.cuda().t(), beta=0.0)
    rt.synchronize()
    _check(C.cpu(), want, err, (path, step))


def test_aligned_copies_count_as_launches():
    m, n, k = 40, 512, 1000                                           # rows of 1000 bytes: both operands are copied
    A, sa, B, sb = [t.cuda() for t in _operands(m, n, k, "e4m3", "e4m3", 1, 128, 23)]
    C = torch.empty(m, n, device="cuda")
    for path, launches in (("tile2", 3), ("pair", 3), ("pair4", 4)):
        with rt.options(**PATHS[path]):
            before = rt.launch_count()
            rt.gemm_fp8(A, B.t(), C, sa, sb.t(), beta=0.0)
            assert rt.launch_count() - before == launches, path
    rt.synchronize()


def _check_16(got, want, err, what):
    """_check, for results some of which fp16 cannot hold: from 65520 (its largest value and half a step) on they round to infinity;
    within the bound of that border either answer is right."""
    if got.dtype != torch.float16:
        return _check(got, want, err, what)
    over = want.abs() - err >= 65520
    near = ~over & (want.abs() + err >= 65520)
    assert torch.equal(got[over].double(), torch.sign(want[over]) * float("inf")), what
    _check(torch.where(over | near, torch.zeros_like(got), got), torch.where(over | near, torch.zeros_like(want), want), err, what)


# (200, 264): rows of C that are whole vectors in every type; (130, 203): not; (512, 512): whole tiles, stored without an epilogue's branches
@pytest.mark.parametrize("alpha,beta,relu,use_bias", [(1.0, 0.0, False, False), (0.5, 0.0, True, True), (-2.0, 0.25, False, True), (1.0, 1.0, True, True)])
@pytest.mark.parametrize("c", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ga,gb", [(1, 1), (128, 1), (128, 128), (1, 128)])
@pytest.mark.parametrize("path", ["pair", "pair4", "tile2"])
@pytest.mark.parametrize("m,n,k", [(200, 264, 768), (130, 203, 700), (512, 512, 640)])
def test_gemm_epilogue_with_every_scale_layout(alpha, beta, relu, use_bias, c, ga, gb, path, m, n, k):
    A, sa, B, sb = _operands(m, n, k, "e4m3", "e4m3", ga, gb, 16)
    g = torch.Generator().manual_seed(17)
    sb *= 0.0005                                                       # nearly all inside fp16's range
    old = (torch.randn(m, n, generator=g) * 100).to(TYPES[c])
    bias = torch.randn(n, generator=g) * 100 if use_bias else None
    want, err = _gemm_want(A, sa, B, sb, ga, gb, old, alpha, beta, bias, relu)
    with rt.options(**PATHS[path]):
        got = _run(A, sa, B, sb, ga, gb, c, old=old, alpha=alpha, beta=beta, relu=relu, bias=bias)
    _check_16(got, want, err, "epilogue")


@pytest.mark.parametrize("a,b", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2")])
@pytest.mark.parametrize("c", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["tn", "tt", "nn", "nt"])
@pytest.mark.parametrize("ga,gb", [(1, 1), (128, 1)])
@pytest.mark.parametrize("path,m,n,k", [("pair", 272, 400, 528), ("pair4", 272, 400, 1040), ("tile", 40, 272, 528)])
def test_gemm_types_and_layouts_with_a_scale_per_column(a, b, c, layout, ga, gb, path, m, n, k):
    A, sa, B, sb = _operands(m, n, k, a, b, ga, gb, 18)
    sb *= 0.0005
    want, err = _gemm_want(A, sa, B, sb, ga, gb)
    with rt.options(**PATHS[path]):
        got = _run(A, sa, B, sb, ga, gb, c, layout, compute="tensor")
    _check_16(got, want, err, (a, b, c, layout))


@pytest.mark.parametrize("c", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("beta", [0.0, 1.0])
@pytest.mark.parametrize("gb", [1, 128])
@pytest.mark.parametrize("path,m,n,k", [("pair", 200, 300, 384), ("pair4", 200, 300, 512), ("pair", 33, 257, 130), ("tile2", 33, 257, 300)])
def test_gemm_result_strides_of_every_type_leave_the_rest_alone(c, beta, gb, path, m, n, k):
    A, sa, B, sb = _operands(m, n, k, "e4m3", "e4m3", 1, gb, 19)
    sb *= 0.0005
    old = torch.full((m, n), 7.0).to(TYPES[c])
    want, err = _gemm_want(A, sa, B, sb, 1, gb, old, 1.0, beta)
    full = lambda *shape: torch.full(shape, 7.0, device="cuda", dtype=TYPES[c])
    for make in (lambda: full(m, n + 5)[:, 2:n + 2], lambda: full(n + 3, m + 1)[1:n + 1, :m].t(), lambda: full(m, 2 * n)[:, ::2], lambda: full(m, n + 16 - n % 8)[:, 8:n + 8]):
        C = make()
        base = C._base
        with rt.options(**PATHS[path]):
            rt.gemm_fp8(A.cuda(), B.cuda().t(), C, sa.cuda(), sb.cuda().t(), beta=beta)
        rt.synchronize()
        _check_16(C.cpu(), want, err, tuple(C.stride()))
        left = base.clone()
        left.as_strided(C.shape, C.stride(), C.storage_offset()).fill_(7.0)
        assert (left == 7).all()


@pytest.mark.parametrize("c", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("ga,gb", [(1, 1), (128, 128)])
@pytest.mark.parametrize("max_ctas", [0, 2, 7])
def test_gemm_over_several_groups_of_row_tiles(c, ga, gb, max_ctas):
    # 11 row tiles of 256: a whole group of eight and a part of one; with two or six CTAs every pair takes many tiles, the ring
    # of scales and both accumulators running on from one to the next
    m, n, k = 2700, 600, 1152
    A, sa, B, sb = _operands(m, n, k, "e4m3", "e4m3", ga, gb, 20)
    sb *= 0.0005
    want, err = _gemm_want(A, sa, B, sb, ga, gb)
    with rt.options(**PATHS["pair"]):
        got = _run(A, sa, B, sb, ga, gb, c, max_ctas=max_ctas)
    _check_16(got, want, err, (ga, gb, max_ctas))


def _with_temporaries(kind):
    """-> (options, m, n, k, offset of A's rows): calls that take aligned copies, sums of K slices, or both from the library's pool"""
    return {"copy": (PATHS["pair"], 300, 512, 1000, 3), "slices": (PATHS["pair4"], 300, 512, 2048, 0), "both": (PATHS["pair4"], 300, 512, 2000, 3),
            "copy, tile": (PATHS["tile2"], 40, 512, 1000, 3)}[kind]


@pytest.mark.parametrize("kind", ["copy", "slices", "both", "copy, tile"])
@pytest.mark.parametrize("gb", [1, 128])
def test_gemm_temporaries_are_not_shared_by_streams_and_graphs(kind, gb):
    path, m, n, k, lead = _with_temporaries(kind)
    data, want = [], []
    for seed in (21, 22):                                              # different inputs: a shared temporary would show
        A, sa, B, sb = _operands(m, n, k, "e4m3", "e4m3", 1, gb, seed)
        wide = torch.zeros(m, k + 7).to(torch.float8_e4m3fn)
        wide[:, lead:lead + k] = A
        data.append([wide.cuda()[:, lead:lead + k] if lead else A.cuda(), B.cuda().t(), sa.cuda(), sb.cuda().t()])
        want.append(_gemm_want(A, sa, B, sb, 1, gb))

    def call(i, C):
        A, B, sa, sb = data[i]
        rt.gemm_fp8(A, B, C, sa, sb, beta=0.0)

    with rt.options(**path):
        first = [torch.empty(m, n, device="cuda") for _ in range(2)]
        for i in range(2):
            call(i, first[i])
        rt.synchronize()
        for i in range(2):
            _check_16(first[i].cpu(), *want[i], kind)
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = [torch.empty(m, n, device="cuda") for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(30):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    call(i, got[i])
        torch.cuda.synchronize()
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
        graphs = []
        for i in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                for _ in range(2):                                     # twice: a freed temporary used again inside the graph
                    call(i, got[i])
            graphs.append(graph)
        other = [torch.empty(m, n, device="cuda") for _ in range(2)]
        for g in got:
            g.fill_(5.0)
        torch.cuda.synchronize()
        for _ in range(3):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
                call(i, other[i])                                      # and eager calls beside the replays, on a third stream
        torch.cuda.synchronize()
        rt.synchronize()
        for i in range(2):
            assert torch.equal(got[i], first[i]) and torch.equal(other[i], first[i])


@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("across", [False, True])
@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("to", ["e4m3", "e5m2"])
@pytest.mark.parametrize("m,k", [(264, 392), (131, 259), (2, 128)])
def test_quantisation_of_infinities_nan_and_subnormals(block, across, src, to, m, k):
    x = _values(m, k, m + k).to(TYPES[src])
    inf, nan = float("inf"), float("nan")
    for i, v in enumerate([inf, -inf, nan, -nan]):                     # in every word, half and lane; whole vectors of them; a group's largest
        x[(7 * i) % m, (11 * i) % k] = v
        x[(7 * i + 1) % m, (11 * i + 1) % k] = v
        x[m - 1, (k - 1 - 3 * i) % k] = v
    if m > 64:
        x[40, 32:64] = inf
        x[50, :128] = nan                                              # a group of nothing finite
        x[51, :] = 0.0
        x[52, :] = torch.finfo(TYPES[src]).smallest_normal * torch.finfo(TYPES[src]).eps * 3     # subnormal
        x[53, 5] = torch.finfo(TYPES[src]).max
        x[64:96, 130] = nan
    if m > 256:
        x[128:256, 128:256] = torch.tensor([inf, nan]).repeat(128, 64).to(TYPES[src])            # a tile of nothing finite
    want = _quantize_want(x.double().numpy(), to, block)
    xd = x.t().contiguous().cuda().t() if across else x.cuda()
    q = torch.zeros(m, k, dtype=TYPES[to], device="cuda")
    s = torch.zeros(_up(m, block), _up(k, 128), device="cuda")
    rt.quantize_fp8(xd, q, s)
    rt.synchronize()
    assert _same(s.cpu().double().numpy(), want[1])
    assert _same(q.cpu().double().numpy(), want[0])


@pytest.mark.parametrize("compute", ["auto", "simt", "tensor"])
def test_gemm_without_products_applies_the_epilogue_in_every_mode(compute):
    f8 = lambda *shape: torch.zeros(*shape, device="cuda", dtype=torch.float8_e4m3fn)
    old = torch.randn(6, 40, device="cuda")
    C = old.clone()
    rt.gemm_fp8(f8(6, 0), f8(0, 40), C, torch.zeros(6, 0, device="cuda"), torch.zeros(0, 1, device="cuda"), beta=-1.0, relu=True, compute=compute)
    rt.synchronize()
    assert torch.equal(C, torch.relu(-old))
