"""Token table lookup and its gradient on the GPU, against the formulas in 64 bits.

Lookup: one fp32 product and one rounding to the result's type, so results equal torch's (x.float() * scale).to(type) bit for bit.
Gradient of a word with L tokens: an fp32 sum of L terms in any order is off by at most (L - 1) 2^-24 sum|g|, the product with scale
and the addition of beta * old by 2^-24 each of what they give, the result by half a step of its type.
"""
import ctypes

import numpy as np
import pytest

from accera_b200 import runtime as rt

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _ids(kind, n, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "uniform":
        return torch.randint(0, vocab, (n,), generator=g)
    if kind == "one":
        return torch.full((n,), vocab - 1)
    if kind == "two":                                    # two words that alternate: long and interleaved
        return torch.arange(n) % 2 * (vocab - 1)
    if kind == "runs":                                   # every length around a chunk border
        return (torch.repeat_interleave(torch.arange(n), torch.arange(n) % 70 + 1)[:n] * 7919) % vocab
    u = torch.rand(n, generator=g, dtype=torch.float64)
    return (float(vocab) ** u - 1).long().clamp(0, vocab - 1)


def _grad_want(g, ids, old, scale, beta, padding=None, vocab=None):
    ids = ids.clone()
    keep = (ids >= 0) & (ids < vocab)
    if padding is not None:
        keep &= ids != padding
    g64, i = g.double()[keep], ids[keep]
    total = torch.zeros(vocab, g.shape[1], dtype=torch.float64).index_add_(0, i, g64)
    size = torch.zeros(vocab, g.shape[1], dtype=torch.float64).index_add_(0, i, g64.abs())
    count = torch.zeros(vocab, dtype=torch.float64).index_add_(0, i, torch.ones(len(i), dtype=torch.float64))
    want = scale * total + (beta * old.double() if beta else 0.0)
    err32 = 2.0 ** -24 * ((count[:, None] + 2) * abs(scale) * size + (abs(beta) * old.double().abs() * 2 if beta else 0.0))
    return want, err32


def _check_grad(got, want, err32, what):
    half_step = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2      # half a subnormal step
    err = (got.double() - want).abs()
    tol = err32 * (1 + half_step) + half_step * want.abs() + tiny
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: got {got[bad][0]} want {want[bad][0]}"


@pytest.mark.parametrize("tokens,dim", [(1, 4096), (8, 8), (33, 1), (257, 100), (1000, 129), (3, 20000), (19, 1023), (10, 1025), (7, 3283), (2, 20001)])
@pytest.mark.parametrize("tt,tr", [("bf16", "bf16"), ("f32", "bf16"), ("f16", "f32"), ("f32", "f32")])
def test_lookup_equals_the_formula(tokens, dim, tt, tr):
    g = torch.Generator().manual_seed(tokens + dim)
    table = torch.randn(777, dim, generator=g).to(TYPES[tt])
    ids = torch.randint(0, 777, (tokens,), generator=g)
    out = torch.full((tokens, dim), float("nan"), dtype=TYPES[tr], device="cuda")
    rt.embedding(table.cuda(), ids.cuda(), out, scale=11.3125)
    rt.synchronize()
    assert torch.equal(out.cpu(), (table[ids].float() * 11.3125).to(TYPES[tr]))
    rt.embedding(table.cuda(), ids.int().cuda(), out)
    rt.synchronize()
    assert torch.equal(out.cpu(), table[ids].to(TYPES[tr]))


def test_lookup_strides_shapes_and_special_values():
    table = torch.randn(50, 96, device="cuda").to(torch.bfloat16)
    table[3] = float("inf"); table[4] = float("nan"); table[5, 0] = -0.0
    ids = torch.tensor([[3, 4, 5], [0, 49, 3]], device="cuda")
    wide = torch.full((2, 3, 200), 7.0, device="cuda", dtype=torch.bfloat16)
    rt.embedding(table[:, 8:73], ids, wide[:, :, 5:70])                   # unaligned views: pitch 96 and 200, offsets 8 and 5
    rt.synchronize()
    want = table[:, 8:73][ids]
    assert torch.equal(wide[:, :, 5:70].nan_to_num(3.5), want.nan_to_num(3.5)) and torch.equal(wide[:, :, 5:70].isnan(), want.isnan())
    assert (wide[:, :, :5] == 7).all() and (wide[:, :, 70:] == 7).all()   # the bytes between rows stay
    sparse = table[::2]                                                   # every second row
    out = torch.empty(2, 96, device="cuda", dtype=torch.bfloat16)
    rt.embedding(sparse, torch.tensor([24, 1], device="cuda"), out, scale=2.0)
    rt.synchronize()
    assert torch.equal(out.nan_to_num(1.0), (sparse[[24, 1]].float() * 2).to(torch.bfloat16).nan_to_num(1.0))


def test_bad_ids_give_zero_rows_and_are_reported_once():
    table = torch.ones(10, 64, device="cuda")
    out = torch.full((5, 64), 9.0, device="cuda")
    rt.synchronize()
    rt.embedding(table, torch.tensor([0, -1, 9, 10, 1 << 40], device="cuda"), out)
    with pytest.raises(rt.AccbError, match=r"embedding: 3 token id"):
        rt.synchronize()
    rt.synchronize()
    assert out[:, 0].tolist() == [1, 0, 1, 0, 0]
    got = torch.full((10, 64), 9.0, device="cuda")
    rt.embedding_grad(torch.ones(4, 64, device="cuda"), torch.tensor([2, 10, -7, 2], device="cuda"), got)
    with pytest.raises(rt.AccbError, match=r"embedding: 2 token id"):
        rt.synchronize()
    assert got[2].eq(2).all() and got.sum() == 128
    many = torch.full((3000,), 7, device="cuda")
    many[5], many[1700], many[2999] = 10, -1, 1 << 33
    rt.embedding_grad(torch.ones(3000, 64, device="cuda"), many, got)
    with pytest.raises(rt.AccbError, match=r"embedding: 3 token id"):
        rt.synchronize()
    assert got[7].eq(2997).all() and got.sum() == 2997 * 64
    with pytest.raises(rt.AccbError) as e:                                # host arrays: from the call itself
        rt.embedding(np.ones((4, 8), np.float32), np.array([4]), np.zeros((1, 8), np.float32))
    assert e.value.code == rt.ERR_INDEX
    rt.synchronize()


@pytest.mark.parametrize("kind", ["uniform", "one", "two", "runs", "zipf"])
@pytest.mark.parametrize("tokens,vocab,dim", [(1, 5, 8), (31, 1, 7), (32, 2, 8), (33, 511, 257), (64, 512, 1), (65, 40000, 8), (1000, 3000, 64),
                                              (2049, 300000, 8), (5000, 100, 33), (20001, 262143, 16)])
def test_gradient_equals_the_formula(kind, tokens, vocab, dim):
    ids = _ids(kind, tokens, vocab, tokens)
    g = torch.randn(tokens, dim, generator=torch.Generator().manual_seed(vocab)).to(torch.bfloat16)
    want, err = _grad_want(g, ids, None, 3.0, 0.0, vocab=vocab)
    got = torch.full((vocab, dim), float("nan"), device="cuda")
    rt.embedding_grad(g.cuda(), ids.cuda(), got, scale=3.0)
    rt.synchronize()
    _check_grad(got.cpu(), want, err, kind)
    again = torch.full((vocab, dim), 5.0, device="cuda")
    rt.embedding_grad(g.cuda(), ids.int().cuda(), again, scale=3.0)       # same bits on every run, whatever the table held
    rt.synchronize()
    assert torch.equal(got, again)


@pytest.mark.parametrize("tg,tt", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("beta,padding", [(0.0, None), (1.0, 2), (-0.5, 0), (1.0, None)])
@pytest.mark.parametrize("tokens", [300, 700, 1500, 2500])                # few tokens by 512, 1024 and 2048, and sorted tokens
def test_gradient_types_beta_padding_and_strides(tokens, tg, tt, beta, padding):
    ids = _ids("zipf", tokens, 90, 5)
    ids[::50] = 2
    g = torch.randn(tokens, 80).to(TYPES[tg])
    old = torch.randn(90, 80).to(TYPES[tt])
    want, err = _grad_want(g, ids, old, 0.75, beta, padding, 90)
    for pad_cols, lead in ((0, 0), (16, 8), (3, 1)):                      # dense, aligned pitch, unaligned pitch and base
        table = torch.full((90, 80 + pad_cols), 4.0, dtype=TYPES[tt], device="cuda")
        rows = torch.zeros(tokens, 80 + pad_cols, dtype=TYPES[tg], device="cuda")
        lead = min(lead, pad_cols)
        table[:, lead:lead + 80] = old.cuda()
        rows[:, lead:lead + 80] = g.cuda()
        rt.embedding_grad(rows[:, lead:lead + 80], ids.cuda(), table[:, lead:lead + 80], scale=0.75, beta=beta, padding_id=padding)
        rt.synchronize()
        _check_grad(table[:, lead:lead + 80].cpu(), want, err, (tg, tt, beta, padding, pad_cols))
        assert (table[:, :lead] == 4).all() and (table[:, lead + 80:] == 4).all()


@pytest.mark.parametrize("tokens", [1, 511, 512, 513, 1024, 1025, 2047, 2048, 2049, 6000])
@pytest.mark.parametrize("vocab,dim", [(33, 40), (1000, 20), (4097, 1), (300, 5000), (70, 20000)])
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_words_without_a_token_between_frequent_ones(tokens, vocab, dim, beta):
    if tokens * dim > 2 ** 24:
        tokens = 2049 if tokens > 2048 else 600                           # (small tables of long rows: enough with these)
    ids = torch.arange(tokens) % 3 * 11 + torch.arange(tokens) % 7 // 6   # words 0, 1, 11, 12, 22, 23, often; the rest never but for the last
    ids[-1] = vocab - 1
    g = torch.randint(-3, 4, (tokens, dim)).to(torch.bfloat16)
    old = torch.randint(-8, 9, (vocab, dim)).float()
    want = torch.zeros(vocab, dim, dtype=torch.float64).index_add_(0, ids, g.double()) + beta * old.double()
    got = old.cuda()
    rt.embedding_grad(g.cuda(), ids.cuda(), got, beta=beta)
    rt.synchronize()
    assert torch.equal(got.cpu().double(), want)                          # sums of small whole numbers: exact


def test_words_without_a_token_keep_their_bytes_with_beta_one():
    table = torch.full((1000, 40), float("nan"), device="cuda")
    table[7] = 1.0
    rt.embedding_grad(torch.ones(3, 40, device="cuda"), torch.tensor([7, 7, 7], device="cuda"), table, beta=1.0)
    rt.synchronize()
    assert (table[7] == 4).all() and table.isnan().sum() == 999 * 40
    rt.embedding_grad(torch.ones(0, 40, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), table, beta=1.0)
    rt.embedding_grad(torch.ones(0, 40, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), table)
    rt.synchronize()
    assert (table == 0).all()                                             # no tokens, beta = 0: all zero, NaN not read


def test_infinities_stay_with_their_word_and_column():
    ids = _ids("zipf", 3000, 40, 1)
    g = torch.randn(3000, 24)
    g[100, 3] = float("inf"); g[200, 5] = float("nan")
    got = torch.empty(40, 24, device="cuda")
    rt.embedding_grad(g.cuda(), ids.cuda(), got)
    rt.synchronize()
    want = torch.zeros(40, 24, dtype=torch.float64).index_add_(0, ids, g.double())
    assert torch.equal(got.cpu().isinf(), want.isinf()) and torch.equal(got.cpu().isnan(), want.isnan())


def test_gradient_against_differences():
    # d/d table of sum(w * embedding(table)) by central differences of the lookup itself: the lookup is linear, so a step of 1 is exact
    table = torch.randint(-8, 9, (6, 8)).float().cuda()
    ids = torch.tensor([1, 4, 1, 1, 0], device="cuda")
    w = torch.randint(-4, 5, (5, 8)).float().cuda()
    got = torch.empty(6, 8, device="cuda")
    rt.embedding_grad(w, ids, got, scale=0.5)
    out = torch.empty(5, 8, device="cuda")

    def loss(t):
        rt.embedding(t, ids, out, scale=0.5)
        return float((out.double() * w.double()).sum())

    for v in range(6):
        for c in range(0, 8, 3):
            up, down = table.clone(), table.clone()
            up[v, c] += 1
            down[v, c] -= 1
            assert (loss(up) - loss(down)) / 2 == float(got[v, c])


def test_streams_graphs_and_two_captured_graphs():
    n, vocab, dim = 3000, 500, 64
    ids = [_ids("zipf", n, vocab, s).cuda() for s in (1, 2)]
    g = [torch.randn(n, dim, device="cuda").to(torch.bfloat16) for _ in range(2)]
    want = []
    for i in range(2):
        t = torch.empty(vocab, dim, device="cuda")
        rt.embedding_grad(g[i], ids[i], t)
        want.append(t)
    torch.cuda.synchronize()
    got = [torch.empty(vocab, dim, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):                                                   # two streams at once: no shared workspace
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                rt.embedding_grad(g[i], ids[i], got[i])
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for i in range(2):
        got[i].fill_(3.0)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            rt.embedding_grad(g[i], ids[i], got[i])
        graphs.append(graph)
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ids[0].copy_(ids[1])                                                  # a replay reads the ids of now
    g[0].copy_(g[1])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[1])


def test_host_arrays():
    rng = np.random.default_rng(3)
    table = rng.standard_normal((30, 20), dtype=np.float32)
    ids = rng.integers(0, 30, (4, 5))
    out = np.zeros((4, 5, 20), np.float32)
    rt.embedding(table, ids, out, scale=4.0)
    assert np.array_equal(out, table[ids] * 4)
    padded = np.full((30, 25), 6, np.float32)
    padded[:, :20] = table
    rt.embedding_grad(out, ids.astype(np.int32), padded[:, :20], beta=1.0)
    want = table.astype(np.float64)
    np.add.at(want, ids.reshape(-1), out.reshape(-1, 20).astype(np.float64))
    np.testing.assert_allclose(padded[:, :20], want, rtol=0, atol=22 * 2.0 ** -24 * 20 * np.abs(out).max())
    assert (padded[:, 20:] == 6).all()


def test_offsets_beyond_32_bits():
    # 2^20 + 8 rows of 4096 bf16 values: 8.6 GB, element offsets beyond 2^32
    vocab, dim = (1 << 20) + 8, 4096
    table = torch.zeros(vocab, dim, device="cuda", dtype=torch.bfloat16)
    table[vocab - 1] = 3.0
    ids = torch.tensor([vocab - 1, 0, vocab - 1], device="cuda")
    out = torch.empty(3, dim, device="cuda", dtype=torch.bfloat16)
    rt.embedding(table, ids, out)
    rt.embedding_grad(out, ids, table, beta=1.0)
    rt.synchronize()
    assert (out[0] == 3).all() and (out[1] == 0).all() and (table[vocab - 1] == 9).all() and (table[0] == 0).all()
    assert (table[vocab - 2] == 0).all()


@pytest.mark.parametrize("tokens", [4, 3000])                             # few tokens, and sorted
@pytest.mark.parametrize("padding", [None, 3])
def test_every_negative_id_is_reported(tokens, padding):
    ids = torch.full((tokens,), 2)
    ids[0], ids[1], ids[2] = -2 ** 63, -1, 3
    got = torch.empty(10, 8, device="cuda")
    rt.synchronize()
    rt.embedding_grad(torch.ones(tokens, 8, device="cuda"), ids.cuda(), got, padding_id=padding)
    with pytest.raises(rt.AccbError, match=r"embedding: 2 token id"):
        rt.synchronize()
    assert (got[2] == tokens - 3).all() and (got[3] == (0 if padding else 1)).all() and got.sum() == 8 * (tokens - (3 if padding else 2))


@pytest.mark.parametrize("tg,tt", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("tokens,vocab,dim", [(4000, 70, 1001), (30000, 900, 33), (29000, 5000, 136), (10000, 300, 2056), (3000, 300, 2056)])
@pytest.mark.parametrize("kind", ["runs", "zipf"])
def test_sorted_gradients_of_many_blocks(kind, tokens, vocab, dim, tg, tt):
    # blocks of 32 tokens and a slab of columns, beyond six an SM but for the last size: rows of whole vectors and others, long and
    # short words
    ids = _ids(kind, tokens, vocab, 8)
    g = torch.randn(tokens, dim, generator=torch.Generator().manual_seed(dim)).to(TYPES[tg])
    old = torch.randn(vocab, dim, generator=torch.Generator().manual_seed(9)).to(TYPES[tt])
    want, err = _grad_want(g, ids, old, 0.5, 1.0, 1, vocab)
    got = old.cuda()
    rt.embedding_grad(g.cuda(), ids.cuda(), got, scale=0.5, beta=1.0, padding_id=1)
    rt.synchronize()
    _check_grad(got.cpu(), want, err, (kind, tg, tt))
    want, err = _grad_want(g, ids, None, 0.5, 0.0, None, vocab)
    got = torch.full((vocab, dim), float("nan"), device="cuda", dtype=TYPES[tt])
    again = torch.full((vocab, dim), 3.0, device="cuda", dtype=TYPES[tt])
    rt.embedding_grad(g.cuda(), ids.cuda(), got, scale=0.5)
    rt.embedding_grad(g.cuda(), ids.int().cuda(), again, scale=0.5)
    rt.synchronize()
    _check_grad(got.cpu(), want, err, (kind, tg, tt))
    assert torch.equal(got, again)
