"""The operators on learned tables against plain forms in 64 bits: lookup, its gradient by sorted
tokens, and the AdamW step with moments in 32 and in 8 bits.

Tolerances: a rounding is off by at most half a step, eps / 2 of the type, relative to the value;
a float32 sum of n terms by n * 2^-24 times the sum of their magnitudes."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
arb = pytest.importorskip("arboretum_b200")
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24  # half a step of float32


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _rng(*key):
    return torch.Generator().manual_seed(sum((i + 1) * 7919 * k for i, k in enumerate(key)) % (1 << 31))


def _near(got, want, magnitude, terms, dtype):
    """|got - want| within float32 sums of `terms` terms of that total magnitude, rounded to dtype."""
    got, want, magnitude = got.double().cpu(), want.double(), magnitude.double()
    limit = (terms + 2) * U * magnitude
    limit = limit + (want.abs() + limit) * (0 if dtype == F32 else _half_step(dtype)) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert got.shape == want.shape
    worst = ((got - want).abs() - limit).max() if got.numel() else torch.tensor(-1.0)
    assert worst <= 0, float(worst)


def _tokens(bags, per_bag, rows, index, gen, empty=0.2):
    tok = torch.randint(0, max(1, rows), (bags, per_bag), generator=gen)
    out = torch.rand((bags, per_bag), generator=gen) < empty
    wrong = torch.tensor([-1, rows, rows + 5, -2 ** 31, 2 ** 31 - 1])
    if index == torch.int64:  # their low 32 bits would be rows of the table
        wrong = torch.cat([wrong, torch.tensor([2 ** 32, -2 ** 63, 2 ** 40 + 1])])
    tok[out] = wrong[torch.randint(0, len(wrong), (int(out.sum()),), generator=gen)]
    if rows == 0:
        tok[:] = -1
    return tok.to(index)


def _plain_lookup(tok, table, scale):
    ok = (tok >= 0) & (tok < table.shape[0])
    t = torch.cat([table.double().cpu(), torch.zeros(1, table.shape[1], dtype=torch.float64)])
    each = t[torch.where(ok, tok.long(), table.shape[0])]
    return each.sum(1) * scale, each.abs().sum(1) * abs(scale)


def _plain_grad(grad, tok, rows, scale):
    """(gradient, sum of magnitudes, tokens a row) in 64 bits"""
    g = grad.double().cpu()[:, None].expand(tok.shape + (grad.shape[-1],)).reshape(tok.numel(), grad.shape[-1])
    flat = tok.long().reshape(-1)
    flat = torch.where((flat >= 0) & (flat < rows), flat, rows)
    z = lambda d: torch.zeros(rows + 1, d, dtype=torch.float64)  # noqa: E731
    total, size = z(g.shape[1]).index_add(0, flat, g)[:rows], z(g.shape[1]).index_add(0, flat, g.abs())[:rows]
    count = z(1).index_add(0, flat, torch.ones(len(flat), 1, dtype=torch.float64))[:rows]
    return total * scale, size * abs(scale), count


SHAPES = [  # bags, tokens a bag, rows, columns
    (0, 1, 5, 8), (1, 1, 1, 1), (1, 1, 9, 4096), (7, 1, 0, 3), (33, 1, 100, 8), (5, 0, 10, 4), (1000, 1, 257, 33),
    (63, 5, 40, 100), (1, 700, 3000, 1), (2, 513, 3000, 770), (257, 100, 6400, 1), (129, 17, 300, 2), (40, 3, 50, 1030),
    (5000, 1, 70000, 16), (12, 1, 3, 0), (300, 1, 2, 257), (4097, 3, 1, 5),
]
TYPES = [(F32, F32), (BF16, BF16), (BF16, F32), (F16, F16), (F16, F32)]


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("shape", SHAPES)
def test_lookup(shape, index):
    bags, per_bag, rows, dim = shape
    gen = _rng(bags, per_bag, rows, dim)
    tok = _tokens(bags, per_bag, rows, index, gen)
    for dtype, out_dtype in TYPES:
        table = torch.randn(rows, dim, generator=gen).to(dtype)
        want, size = _plain_lookup(tok, table, 1.7)
        got = arb.embedding(tok.cuda(), table.cuda(), scale=1.7, pooled=True, out_dtype=out_dtype)
        assert got.dtype == out_dtype
        _near(got, want, size, per_bag, out_dtype)
        if per_bag == 1:
            flat = arb.embedding(tok.cuda()[:, 0], table.cuda(), scale=1.7, out_dtype=out_dtype)
            assert torch.equal(flat, got)


def test_lookup_shapes_and_plain_copies():
    table = torch.randn(50, 24, generator=_rng(1)).cuda()
    tok = torch.randint(0, 50, (3, 4, 5), generator=_rng(2)).cuda()
    assert torch.equal(arb.embedding(tok, table), table[tok])
    assert torch.equal(arb.embedding(tok[1, 2, 3], table), table[tok[1, 2, 3]])
    assert torch.equal(arb.embedding(tok.transpose(0, 2), table), table[tok.transpose(0, 2)])
    assert torch.equal(arb.embedding(tok[0, :, 2], table.half()), table.half()[tok[0, :, 2]])
    out = torch.full((3, 4, 5, 24), 7.0, device="cuda")
    assert arb.embedding(tok, table, out=out) is out and torch.equal(out, table[tok])


@pytest.mark.parametrize("offset", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("dim,pad", [(8, 0), (8, 1), (32, 8), (33, 2), (260, 4), (301, 0), (512, 1), (777, 2), (1030, 3)])
def test_lookup_and_gradient_of_strided_and_offset_memory(dim, pad, offset):
    """Rows and starts of every alignment; what lies between the rows stays as it was."""
    gen = _rng(dim, pad, offset)
    bags, rows = 70, 90
    for dtype in (F32, BF16):
        store = torch.randn(offset + rows * (dim + pad), generator=gen).to(dtype).cuda()
        table = store[offset:].view(rows, dim + pad)[:, :dim]
        tok = _tokens(bags, 1, rows, torch.int32, gen)
        wide = torch.full((offset + bags * (dim + pad),), 5.0, dtype=dtype, device="cuda")
        out = wide[offset:].view(bags, dim + pad)[:, :dim]
        arb.embedding(tok.cuda()[:, 0], table, scale=0.5, out=out)
        want, size = _plain_lookup(tok, table.cpu(), 0.5)
        _near(out, want, size, 1, dtype)
        assert (wide[offset:].view(bags, dim + pad)[:, dim:] == 5).all() and (wide[:offset] == 5).all()
        # and the way back
        gstore = torch.randn(offset + bags * (dim + pad), generator=gen).to(dtype).cuda()
        grad = gstore[offset:].view(bags, dim + pad)[:, :dim]
        gwide = torch.full((offset + rows * (dim + pad),), 5.0, dtype=dtype, device="cuda")
        gout = gwide[offset:].view(rows, dim + pad)[:, :dim]
        arb.embedding_grad(grad, tok.cuda()[:, 0], rows, scale=0.5, out=gout)
        want, size, count = _plain_grad(grad, tok, rows, 0.5)
        _near(gout, want, size, count, dtype)
        assert (gwide[offset:].view(rows, dim + pad)[:, dim:] == 5).all() and (gwide[:offset] == 5).all()


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("shape", SHAPES)
def test_gradient(shape, index):
    bags, per_bag, rows, dim = shape
    gen = _rng(bags, per_bag, rows, dim, 3)
    tok = _tokens(bags, per_bag, rows, index, gen)
    order = arb.token_order(tok.cuda(), rows, pooled=True)
    for dtype, out_dtype in TYPES:
        grad = torch.randn(bags, dim, generator=gen).to(dtype)
        want, size, count = _plain_grad(grad, tok, rows, -0.6)
        got = arb.embedding_grad(grad.cuda(), tok.cuda(), rows, scale=-0.6, pooled=True, out_dtype=out_dtype)
        assert got.dtype == out_dtype
        _near(got, want, size, count, out_dtype)
        again = arb.embedding_grad(grad.cuda(), order, rows, scale=-0.6, out_dtype=out_dtype)
        assert torch.equal(got, again)
        if per_bag == 1:
            assert torch.equal(got, arb.embedding_grad(grad.cuda(), tok.cuda()[:, 0], rows, scale=-0.6, out_dtype=out_dtype))
        before = torch.randn(rows, dim, generator=gen).to(out_dtype)
        out = before.cuda()
        assert arb.embedding_grad(grad.cuda(), order, rows, scale=-0.6, out=out, accumulate=True) is out
        untouched = (count == 0).expand(rows, dim)
        assert torch.equal(out.cpu()[untouched], before[untouched])
        _near(out, want + before.double(), size + before.double().abs(), count + 1, out_dtype)


@pytest.mark.parametrize("bags,rows,dim,kind", [
    (20000, 4, 3, "same"), (20000, 50, 64, "zipf"), (9000, 3000, 257, "zipf"), (70000, 70000, 1, "zipf"),
    (3000, 17, 1030, "same"), (100000, 300, 2, "zipf"), (16385, 1 << 19, 4, "zipf"), (300000, 5, 1, "even")])
def test_gradient_of_frequent_tokens(bags, rows, dim, kind):
    gen = _rng(bags, rows, dim)
    u = torch.rand(bags, 1, generator=gen, dtype=torch.float64)
    tok = {"same": torch.full((bags, 1), rows - 1), "even": (u * rows).long(),
           "zipf": ((rows + 1.0) ** u - 1).long().clamp(0, rows - 1)}[kind]
    for dtype in (F32, BF16):
        grad = torch.randn(bags, dim, generator=gen).to(dtype)
        want, size, count = _plain_grad(grad, tok, rows, 1.0)
        got = arb.embedding_grad(grad.cuda(), tok.cuda()[:, 0], rows)
        _near(got, want, size, count, dtype)
        assert torch.equal(got, arb.embedding_grad(grad.cuda(), tok.cuda()[:, 0], rows))  # no order of arrival in it


@pytest.mark.parametrize("count", [1, 31, 512, 513, 2049, 16384, 16385, 32768, 32769, 1 << 20, (1 << 20) + 77])
@pytest.mark.parametrize("rows", [1, 700, 1 << 18, (1 << 18) + 1])
def test_every_sort_and_cut(count, rows):
    """Numbers of tokens around the limits of the sorts, rows around that of the marks they clear, rows
    cut into pieces at every place; integers, so that sums in any order are exact."""
    gen = _rng(count, rows)
    u = torch.rand(count, generator=gen, dtype=torch.float64)
    for tok in (((rows + 1.0) ** u - 1).long().clamp(0, rows - 1) * 7919 % rows,  # few frequent ones
                (torch.arange(count) // 45) % rows):                              # runs of 45
        tok[torch.rand(count, generator=gen) < 0.05] = -1
        grad = torch.randint(-8, 9, (count, 2), generator=gen).float()
        want, _, _ = _plain_grad(grad, tok[:, None], rows, 1.0)
        assert want.abs().max() < 2 ** 24
        got = arb.embedding_grad(grad.cuda(), tok.cuda(), rows)
        assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("bags,per_bag,leaves,dim", [(1, 3, 8, 1), (1000, 50, 16, 1), (30011, 20, 256, 1), (513, 7, 64, 3), (100003, 3, 2, 2)])
def test_forest_layout(bags, per_bag, leaves, dim):
    """Tokens tree after tree, every tree with rows of its own: lookup and gradient through the strides."""
    gen = _rng(bags, per_bag, leaves)
    rows = per_bag * leaves
    tok = torch.randint(0, leaves, (per_bag, bags), generator=gen, dtype=torch.int32) + torch.arange(per_bag, dtype=torch.int32)[:, None] * leaves
    table = torch.randn(rows, dim, generator=gen)
    want, size = _plain_lookup(tok.t(), table, 0.1)
    _near(arb.embedding(tok.cuda().t(), table.cuda(), scale=0.1, pooled=True), want, size, per_bag, F32)
    grad = torch.randn(bags, dim, generator=gen)
    want, size, count = _plain_grad(grad, tok.t(), rows, 0.1)
    order = arb.token_order(tok.cuda().t(), rows, pooled=True)
    _near(arb.embedding_grad(grad.cuda(), order, rows, scale=0.1), want, size, count, F32)


@pytest.mark.parametrize("bags,per_bag,rows,dim", [
    (40001, 9, 90, 1), (40000, 9, 90, 3), (16384 * 2 + 1, 17, 33, 2), (70001, 5, 7, 5), (50000, 6, 20, 64), (33000, 8, 3, 1),
    (20000, 40, 500, 2), (65536, 4, 2, 8), (300007, 2, 600, 33)])
def test_many_bags_over_few_rows(bags, per_bag, rows, dim):
    """Where the lookup holds the table in shared memory and the order is kept by runs of bags."""
    gen = _rng(bags, per_bag, rows, dim)
    for index, by_slot in ((torch.int32, True), (torch.int64, False), (torch.int64, True)):
        tok = _tokens(bags, per_bag, rows, index, gen, empty=0.1)
        tok[:, 0] = rows - 1  # a row that every bag names
        tok = tok.t().contiguous().t() if by_slot else tok
        dev = tok.cuda().t().contiguous().t() if by_slot else tok.cuda()
        for dtype, out_dtype in ((F32, F32), (BF16, F32), (F16, F16)):
            table = torch.randn(rows, dim, generator=gen).to(dtype)
            want, size = _plain_lookup(tok, table, 0.3)
            _near(arb.embedding(dev, table.cuda(), scale=0.3, pooled=True, out_dtype=out_dtype), want, size, per_bag, out_dtype)
            grad = (torch.randn(bags, dim, generator=gen) * 0.01).to(dtype)
            want, size, count = _plain_grad(grad, tok, rows, 0.3)
            got = arb.embedding_grad(grad.cuda(), dev, rows, scale=0.3, pooled=True, out_dtype=out_dtype)
            _near(got, want, size, count, out_dtype)
            assert torch.equal(got, arb.embedding_grad(grad.cuda(), arb.token_order(dev, rows, pooled=True), rows, scale=0.3, out_dtype=out_dtype))
            before = torch.randn(rows, dim, generator=gen).to(out_dtype)
            out = before.cuda()
            arb.embedding_grad(grad.cuda(), dev, rows, scale=0.3, pooled=True, out=out, accumulate=True)
            assert torch.equal(out.cpu()[(count == 0).expand(rows, dim)], before[(count == 0).expand(rows, dim)])
            _near(out, want + before.double(), size + before.double().abs(), count + 1, out_dtype)


@pytest.mark.parametrize("rows", [32769 * 16, 32769 * 16 + 1, 15])
def test_rows_without_a_bag_of_orders_one_after_the_other(rows):
    """Orders in memory that others left behind: rows that no bag names get zeros all the same."""
    gen = _rng(rows)
    for i in range(3):
        tok = torch.randint(0, rows // 3, (32769,), generator=gen) * 3 + i  # rows other than the last order's
        got = arb.embedding_grad(torch.ones((), device="cuda").expand(32769, 3), tok.cuda(), rows)
        assert torch.equal(got, torch.bincount(tok, minlength=rows).float().cuda()[:, None].expand(rows, 3))


def test_gradient_of_broadcast_inputs():
    tok = torch.randint(0, 30, (6, 50), generator=_rng(5))
    row = torch.randn(40, generator=_rng(6)).cuda()
    full = arb.embedding_grad(row.expand(6, 50, 40).contiguous(), tok.cuda(), 30)
    assert torch.equal(arb.embedding_grad(row.expand(6, 50, 40), tok.cuda(), 30), full)
    assert torch.equal(arb.embedding_grad(row.expand(300, 40), tok.cuda().view(-1), 30), full)
    one = torch.ones((), device="cuda")
    assert torch.equal(arb.embedding_grad(one.expand(300, 40), tok.cuda().view(-1), 30),
                       torch.bincount(tok.view(-1), minlength=30).float().cuda()[:, None].expand(30, 40))
    # the order of an expanded index: every bag names the same tokens
    same = tok[0].cuda().expand(6, 50)
    g = torch.randn(6, 40, generator=_rng(7)).cuda()
    want, size, count = _plain_grad(g, same.cpu(), 30, 1.0)
    _near(arb.embedding_grad(g, same, 30, pooled=True), want, size, count, F32)


def test_gradient_against_differences():
    """The lookup is linear: the difference of two lookups is the gradient's inner product."""
    gen = _rng(11)
    tok = _tokens(400, 6, 150, torch.int64, gen).cuda()
    a, d = torch.randn(150, 48, generator=gen).cuda(), torch.randn(150, 48, generator=gen).cuda()
    g = torch.randn(400, 48, generator=gen).cuda()
    f = lambda t: arb.embedding(tok, t, scale=0.3, pooled=True).double()  # noqa: E731
    lhs = ((f(a + d) - f(a - d)) / 2 * g.double()).sum()
    rhs = (arb.embedding_grad(g, tok, 150, scale=0.3, pooled=True).double() * d.double()).sum()
    # every product of the two sums is off by a few float32 roundings of terms of these magnitudes
    size = (arb.embedding(tok, a.abs() + d.abs(), scale=0.3, pooled=True).double() * g.abs().double()).sum()
    assert abs(lhs - rhs) <= 20 * U * size


def test_infinities_and_nan_stay_in_their_rows():
    table = torch.randn(20, 16, generator=_rng(12))
    table[3], table[4], table[5, 0] = float("nan"), float("inf"), -float("inf")
    tok = torch.tensor([[0, -1, 2], [4, -1, -1], [-1, -1, -1], [1, 1, 3], [4, 5, -1]])
    got = arb.embedding(tok.cuda(), table.cuda(), pooled=True).cpu()
    assert torch.isfinite(got[0]).all() and torch.isposinf(got[1]).all() and (got[2] == 0).all()
    assert torch.isnan(got[3]).all() and torch.isnan(got[4, 0]) and torch.isposinf(got[4, 1:]).all()
    grad = torch.ones(4, 16)
    grad[1], grad[2] = float("nan"), float("inf")
    got = arb.embedding_grad(grad.cuda(), torch.tensor([0, -1, 2, 0], device="cuda"), 5).cpu()
    assert (got[0] == 2).all() and (got[1] == 0).all() and torch.isposinf(got[2]).all() and (got[3:] == 0).all()


def test_rows_beyond_32_bit_offsets():
    rows, dim = 70000, 65536  # 4.6 G elements of bf16
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    table = torch.zeros(rows, dim, dtype=BF16, device="cuda")
    table[-1] = 3.0
    tok = torch.tensor([rows - 1, 0, rows - 1], device="cuda")
    got = arb.embedding(tok, table, scale=2.0)
    assert (got[0] == 6).all() and (got[1] == 0).all() and (got[2] == 6).all()
    arb.embedding_grad(got, tok, rows, out=table)
    assert (table[-1] == 12).all() and not table[:-1].any()


def test_accumulation_of_frequent_rows_and_gradients_of_one_tensor():
    """The same index many times, added to what is there; the output of one call as the input of the next."""
    gen = _rng(77)
    tok = torch.randint(0, 3, (5000,), generator=gen).cuda()
    g = torch.randint(-4, 5, (5000, 37), generator=gen).float().cuda()
    total = torch.zeros(4, 37, device="cuda")
    for _ in range(3):
        arb.embedding_grad(g, tok, 4, out=total, accumulate=True)
    want = torch.zeros(4, 37, device="cuda").index_add(0, tok, g) * 3  # integers: exact in any order
    assert torch.equal(total, want)
    again = arb.embedding(tok, total)
    assert torch.equal(again, total[tok])
    # a table of one row, a bag that names it in every slot
    assert torch.equal(arb.embedding(torch.zeros(2, 700, dtype=torch.int32, device="cuda"), total[:1], pooled=True), (total[:1] * 700).expand(2, 37))


def test_refusals_on_the_device():
    t, i = torch.zeros(5, 4, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        arb.embedding(i, t, out=t[:3])
    with pytest.raises(ValueError, match="shares memory"):
        arb.embedding_grad(t[:3], i, 5, out=t)
    with pytest.raises(ValueError, match="out must have shape"):
        arb.embedding(i, t, out=torch.zeros(4, 4, device="cuda"))
    with pytest.raises(TypeError, match="out must be"):
        arb.embedding(i, t, out=torch.zeros(3, 4, device="cuda", dtype=BF16))
    with pytest.raises(ValueError, match="contiguous"):
        arb.embedding(i, t, out=torch.zeros(4, 3, device="cuda").t())
    with pytest.raises(arb.ArboretumError, match="overlap"):
        arb.embedding(i, t, out=torch.zeros(1, 4, device="cuda").expand(3, 4))
    with pytest.raises(ValueError, match="on cpu"):
        arb.embedding(i.cpu(), t)
    with pytest.raises(ValueError, match="order was made"):
        arb.embedding_grad(t[:3], arb.token_order(i, 6), 5)
    o = arb.AdamW([t])
    for bad in ([], [None, None], [torch.zeros(4, 5, device="cuda").t()], [torch.zeros(5, 4)], [t[:4]]):
        with pytest.raises(ValueError):
            o.step(bad)
    with pytest.raises(TypeError):
        o.step([t.half()])
    with pytest.raises(ValueError, match="no gradients"):
        o.step()
    with pytest.raises(arb.ArboretumError, match="finite"):
        o.step([t.clone()], lr=float("nan"))
    with pytest.raises(ValueError):
        o.load_state_dict({"step": 1})
    assert o.steps == 0


# ---- AdamW -----------------------------------------------------------------------------------
def _hash(index, step, seed):
    m = np.uint64(0xFFFFFFFF)
    i = index.astype(np.uint64)
    x = (i & m) ^ ((i >> np.uint64(32)) * np.uint64(0x9E3779B1) & m) ^ np.uint64(step * 0x85EBCA6B & 0xFFFFFFFF) ^ np.uint64(seed * 0xC2B2AE35 & 0xFFFFFFFF)
    x = (x ^ (x >> np.uint64(16))) * np.uint64(0x7FEB352D) & m
    x = (x ^ (x >> np.uint64(15))) * np.uint64(0x846CA68B) & m
    return x ^ (x >> np.uint64(16))


def _decode(code, scale):
    """e4m3 codes times their block's scale, in float32"""
    c = code.astype(np.int64)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * 2.0 ** (e - 7.0)) * np.where(c & 128, -1, 1)
    return (v.astype(np.float32) * np.repeat(scale, 128)[:len(v)]).astype(np.float32)


def _encode(x, index, step, seed, shift, positive):
    """Codes and scales of a float32 slot of whole blocks: the format's definition, from the real
    numbers: floor(x / step + u) with u the middle of one of 65536 equal parts of [0, 1)."""
    blocks = np.abs(x.reshape(-1, 128)).max(1).astype(np.float64)
    part, power = np.frexp(blocks)
    scale = np.maximum(np.ldexp(1.0, np.where(part > 0.875, power - 8, power - 9)), 2.0 ** -126)
    scale[blocks == 0] = 2.0 ** -126
    y = np.abs(x).astype(np.float64) / np.repeat(scale, 128)
    y = np.where(y < 2.0 ** -6, np.rint(y * 2.0 ** 29) * 2.0 ** -29, y)  # the kernel's smallest exponent ends there
    e = np.maximum(np.frexp(y)[1] - 1, -6)
    u = ((_hash(index, step, seed) >> np.uint64(shift)) & np.uint64(0xFFFF)).astype(np.float64)
    q = np.floor(y / 2.0 ** (e - 3) + (u + 0.5) / 65536)  # steps of 2^(e-3)
    value = np.minimum(q * 2.0 ** (e - 3), 448.0)
    if positive:
        value = np.where((x > 0) & (value == 0), 2.0 ** -9, value)
    fe = np.maximum(np.frexp(value)[1] - 1, -6)
    f = np.round(value / 2.0 ** (fe - 3)).astype(np.int64)  # 8 .. 15, or below 8 at the smallest exponent
    code = np.where(f >= 8, (fe + 7) * 8 + (f - 8), f)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8), scale.astype(np.float32)


class Plain:
    """The step in float32, operation by operation, and beside it in 64 bits from the same state."""

    def __init__(self, sizes, lr, b1, b2, eps, wd, bits, seed):
        self.h = (lr, b1, b2, eps, wd)
        self.bits, self.seed, self.t = bits, seed, 0
        self.slots, end = [], 0
        for n in sizes:
            self.slots.append(end)
            end += (n + 127) // 128 * 128
        self.kept = np.zeros(end, bool)
        for at, n in zip(self.slots, sizes):
            self.kept[at:at + n] = True
        self.m, self.v = np.zeros(end, np.float32), np.zeros(end, np.float32)
        if bits == 8:
            self.c1, self.c2 = np.zeros(end, np.uint8), np.zeros(end, np.uint8)
            self.s1, self.s2 = np.zeros(end // 128, np.float32), np.zeros(end // 128, np.float32)

    def step(self, p, g):
        """p, g: flat float32 in the slots' layout -> (float32 p, 64-bit p, limit of their difference)"""
        lr, b1, b2, eps, wd = self.h
        self.t += 1
        f = np.float32
        if self.bits == 8:
            m, r = _decode(self.c1, self.s1), _decode(self.c2, self.s2)
            v = r * r
        else:
            m, v = self.m, self.v
        g8, m8, v8, p8 = (x.astype(np.float64) for x in (g, m, v, p))
        m8, size = b1 * m8 + (1 - b1) * g8, b1 * abs(m8) + (1 - b1) * abs(g8)
        v8 = b2 * v8 + (1 - b2) * g8 * g8
        below = np.sqrt(v8) / np.sqrt(1 - b2 ** self.t) + eps
        rate = lr / (1 - b1 ** self.t)
        want = p8 * (1 - lr * wd) - rate * m8 / below
        # roundings: m 4 of its parts' magnitude (2 constants, 2 products, 1 sum); the root's chain 8
        # relative (constants, products and sum of v half of theirs, root, constant, product, sum);
        # division, rate and product 3; p's constant, product and difference 3
        limit = U * (4 * abs(p8) + rate * (5 * size + 12 * abs(m8)) / below)
        m = m * f(b1) + g * f(1 - b1)
        v = v * f(b2) + (g * g) * f(1 - b2)
        r = np.sqrt(v)
        p = p * f(1 - lr * wd) - (m / (r * f(1 / np.sqrt(1 - b2 ** self.t)) + f(eps))) * f(rate)
        if self.bits == 8:
            i = np.arange(len(m))
            self.c1, self.s1 = _encode(m, i, self.t, self.seed, 0, False)
            self.c2, self.s2 = _encode(r, i, self.t, self.seed, 16, True)
        self.m, self.v = m, v
        return p, want, limit


SIZES = [[1], [128], [127, 129], [4096], [4097, 5, 1, 8191, 128], [30000, 3, 0, 77], [64] * 50]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("sizes", SIZES)
def test_adamw(sizes, bits):
    lr, b1, b2, eps, wd = 3e-3, 0.9, 0.98, 1e-8, 0.1
    for dtype, grad_dtype, master in [(F32, F32, False), (F32, F32, True), (BF16, BF16, False), (BF16, F32, True), (F16, F16, True), (F16, F32, False)]:
        gen = _rng(len(sizes), sizes[0], bits)
        start = [torch.randn(n, generator=gen).to(dtype) for n in sizes]
        params = [p.cuda() for p in start]
        o = arb.AdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, state_bits=bits, master=master, seed=5)
        ref = Plain(sizes, lr, b1, b2, eps, wd, bits, 5)
        assert o.slots == ref.slots
        flat = lambda xs: np.concatenate([np.pad(x.float().cpu().numpy(), (0, -len(x) % 128)) for x in xs])  # noqa: E731
        p = flat(start)
        for step in range(3):
            # gradients of very different magnitudes inside a block, zeros among them
            grads = [(torch.randn(n, generator=gen) * 10 ** (6 * torch.rand(n, generator=gen) - 5) * (torch.rand(n, generator=gen) < 0.9)).to(grad_dtype) for n in sizes]
            o.step([g.cuda() for g in grads])
            p32, want, limit = ref.step(p, flat(grads))
            # the moments are float32 arithmetic and nothing else: equal bits
            if bits == 8:
                assert np.array_equal(o.moment1.view(torch.uint8).cpu().numpy(), ref.c1)
                assert np.array_equal(o.moment2.view(torch.uint8).cpu().numpy(), ref.c2)
                assert np.array_equal(o.scale1.cpu().numpy(), ref.s1) and np.array_equal(o.scale2.cpu().numpy(), ref.s2)
                assert (ref.c2[(p32 == p32) & (ref.v > 0)] > 0).all()
            else:
                assert np.array_equal(o.moment1.cpu().numpy(), ref.m) and np.array_equal(o.moment2.cpu().numpy(), ref.v)
            got = o.master.cpu().numpy() if master else flat(params)
            off = limit if master or dtype == F32 else limit + (np.abs(want) + limit) * _half_step(dtype) + 2.0 ** -25
            assert (np.abs(got.astype(np.float64) - want) <= off)[ref.kept].all()
            if master:  # the parameters are the copy, rounded
                for x, at in zip(params, o.slots):
                    assert torch.equal(x, o.master[at:at + x.numel()].to(dtype))
            p = got.astype(np.float32)
        assert o.steps == 3
        for k, x in enumerate(params):
            m, v = o.moments(k)
            assert m.shape == x.shape and v.shape == x.shape and (v >= 0).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,grad_dtype", [(F32, F32), (BF16, BF16), (F16, F32)])
def test_adamw_at_every_alignment(bits, dtype, grad_dtype):
    """Parameters and gradients that begin anywhere give the bits of aligned ones; what lies around them stays."""
    n = 1000
    gen = _rng(n, bits)
    start = torch.randn(n, generator=gen).to(dtype).cuda()
    grad = torch.randn(n, generator=gen).to(grad_dtype).cuda()
    want = start.clone()
    first = arb.AdamW([want], lr=0.1, state_bits=bits)
    for _ in range(2):
        first.step([grad])
    for shift in range(1, 9):
        store = torch.full((n + 16,), 3.0, dtype=dtype, device="cuda")
        p = store[shift:shift + n]
        p.copy_(start)
        g = torch.zeros(n + 16, dtype=grad_dtype, device="cuda")[16 - shift:][:n]
        g.copy_(grad)
        o = arb.AdamW([p], lr=0.1, state_bits=bits)
        for _ in range(2):
            o.step([g])
        assert torch.equal(p, want) and torch.equal(o.moment1.view(torch.uint8), first.moment1.view(torch.uint8))
        assert (store[:shift] == 3).all() and (store[shift + n:] == 3).all()


def test_adamw_dither_keeps_the_mean():
    """A moment whose change is far below half an e4m3 step still follows it on average."""
    n = 1 << 16
    p = torch.zeros(n, device="cuda")
    o = arb.AdamW([p], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8)
    g = torch.full((n,), 1.0, device="cuda")
    for _ in range(40):
        o.step([g])
    m, v = o.moments(0)
    want_m, want_v = 1 - 0.9 ** 40, 1 - 0.999 ** 40
    # one element's m jumps by at most an eighth of itself, and jumps made k steps ago have decayed by
    # 0.9^k: its spread is below 0.125 / 2 / sqrt(1 - 0.81); the mean's is that over sqrt(n); six of them
    assert abs(m.double().mean() - want_m) < 6 * 0.0625 / np.sqrt(1 - 0.81) / np.sqrt(n)
    # the root's steps do not decay in 40 steps: below 0.0625 sqrt(40) of it for one element; v is the
    # square, whose mean is above the root's squared mean by the spread's square
    root = np.sqrt(want_v)
    spread = 0.0625 * np.sqrt(40) * root
    assert abs(v.double().sqrt().mean() - root) < 6 * spread / np.sqrt(n) + 0.5 * 0.0625 ** 2 * root * 40


def test_adamw_not_finite():
    for bits in (32, 8):
        p = torch.ones(300, device="cuda")
        o = arb.AdamW([p], state_bits=bits)
        g = torch.ones(300)
        g[5], g[200] = float("nan"), float("inf")
        o.step([g.cuda()])
        assert torch.isnan(p[5]) and torch.isnan(p[200])
        rest = torch.ones(300, dtype=torch.bool)
        rest[5] = rest[200] = False
        assert torch.isfinite(p.cpu()[rest]).all()
        m, v = (x.cpu() for x in o.moments(0))
        if bits == 8:  # the two blocks that hold them, and no other
            assert torch.isnan(m[:256]).all() and torch.isnan(v[:256]).all() and torch.isfinite(m[256:]).all()
        else:
            assert torch.isnan(m[5]) and torch.isinf(m[200]) and torch.isfinite(m[rest]).all()


def test_adamw_left_out_scaled_and_bound():
    gen = _rng(21)
    make = lambda: [torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda() for n in (300, 40, 5000)]  # noqa: E731
    grads = [torch.randn(n, generator=gen).cuda() for n in (300, 40, 5000)]
    for bits in (32, 8):
        a, b, c = make(), make(), make()
        oa, ob = arb.AdamW(a, lr=0.01, state_bits=bits), arb.AdamW(b, lr=1.0, state_bits=bits, grads=grads)
        oc = arb.AdamW(c, lr=torch.tensor([0.01], device="cuda"), state_bits=bits)
        oa.step([grads[0], None, grads[2]])
        assert torch.equal(a[1], make()[1]) and not oa.moments(1)[0].any() and oa.moments(0)[0].any()
        oa.step(grads, lr=0.02)
        half = [g * 0.5 for g in grads]
        ob.step([grads[0], None, grads[2]], lr=torch.tensor(0.01, device="cuda"))
        ob.step(lr=0.02)
        oc.step([half[0], None, half[2]], grad_scale=torch.tensor(2.0, device="cuda"))
        oc.step(half, lr=0.02, grad_scale=torch.tensor([2.0], device="cuda"))
        for x, y, z in zip(a, b, c):
            assert torch.equal(x, y)
            # lr passes through float32 in one of them: the rate of one step is off by half a step of
            # float32, and the parameters by that of a change of 0.02 and by their own rounding
            assert (x - z).abs().max() <= 4 * U * 6
        assert oa.steps == ob.steps == oc.steps == 2


def test_adamw_state_moves_to_another_optimizer():
    gen = _rng(22)
    grads = [torch.randn(1000, generator=gen).cuda() for _ in range(4)]
    for bits in (32, 8):
        for master in (False, True):
            a = torch.ones(1000, device="cuda", dtype=BF16)
            oa = arb.AdamW([a], state_bits=bits, master=master)
            for g in grads[:2]:
                oa.step([g])
            b = a.clone()
            ob = arb.AdamW([b], state_bits=bits, master=master)
            ob.load_state_dict({k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in oa.state_dict().items()})
            for g in grads[2:]:
                oa.step([g])
                ob.step([g])
            assert torch.equal(a, b) and torch.equal(oa.moment1.view(torch.uint8), ob.moment1.view(torch.uint8)) and ob.steps == 4


def test_adamw_many_tensors():
    """More tensors than one launch takes; every one of them moves once."""
    store = torch.ones(5000, 3, device="cuda")
    params = [store[i] for i in range(5000)]
    o = arb.AdamW(params, lr=0.5, weight_decay=0.0, eps=0.0)
    o.step([torch.ones(3, device="cuda")] * 5000)
    # m / sqrt(v) is 1 up to the roundings of its chain: 0.5 = 1 - 0.5 within 16 half steps
    assert (store - 0.5).abs().max() <= 16 * U and o.steps == 1
    assert len(torch.unique(store)) == 1


def test_autograd_sees_the_step():
    p = torch.ones(10, device="cuda", requires_grad=True)
    y = (p * p).sum()
    o = arb.AdamW([p])
    o.step([torch.ones(10, device="cuda")])
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_a_parameter_or_gradient_that_moved_is_refused():
    p, g, e = torch.ones(10, device="cuda"), torch.ones(10, device="cuda"), torch.zeros(0, device="cuda")
    o = arb.AdamW([p, e], grads=[g, None])
    o.step()
    g.data = torch.ones(10, device="cuda")
    with pytest.raises(ValueError, match="gradient's memory has moved"):
        o.step()
    o.step([g, e.clone()])
    p.data = torch.ones(10, device="cuda")
    with pytest.raises(ValueError, match="parameter's memory has moved"):
        o.step([g, None])
    assert o.steps == 2 and (p == 1).all()


# ---- together --------------------------------------------------------------------------------
def _train(steps, bits, side_stream, capture):
    """A table learned through the lookup: squared error of pooled rows against targets."""
    gen = torch.Generator().manual_seed(3)
    bags, per_bag, rows, dim = 700, 5, 90, 12
    tok = _tokens(bags, per_bag, rows, torch.int32, gen).cuda()
    target = torch.randn(bags, dim, generator=gen).cuda()
    table = torch.zeros(rows, dim, device="cuda")
    grad = torch.zeros(rows, dim, device="cuda")
    o = arb.AdamW([table], lr=0.05, weight_decay=0.0, state_bits=bits, grads=[grad])

    def step():
        e = (arb.embedding(tok, table, scale=0.5, pooled=True) - target) * (2.0 / bags)
        arb.embedding_grad(e, tok, rows, scale=0.5, pooled=True, out=grad)
        o.step()
    stream = torch.cuda.Stream() if side_stream else torch.cuda.current_stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        if capture:
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                step()
            for _ in range(steps - 1):
                graph.replay()
        else:
            for _ in range(steps):
                step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    assert o.steps == steps
    return table, tok, target


@pytest.mark.parametrize("bits", [32, 8])
def test_training_step_on_streams_and_in_a_graph(bits):
    table, tok, target = _train(6, bits, False, False)
    for side_stream, capture in ((True, False), (True, True)):
        other, _, _ = _train(6, bits, side_stream, capture)
        assert torch.equal(table, other)
    if bits == 32:  # the same steps in 64 bits
        t = torch.zeros(table.shape, dtype=torch.float64)
        m, v = torch.zeros_like(t), torch.zeros_like(t)
        for k in range(1, 7):
            e = (_plain_lookup(tok.cpu(), t, 0.5)[0] - target.double().cpu()) * (2.0 / len(target))
            g = _plain_grad(e, tok.cpu(), len(t), 0.5)[0]
            m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
            t = t - 0.05 / (1 - 0.9 ** k) * m / ((v / (1 - 0.999 ** k)).sqrt() + 1e-8)
        # a step is at most 0.05 times a ratio near 1; the ratio's relative error is that of the
        # gradient sums, whose cancellation is at most a few hundred fold here: 6 * 0.05 * 500 * 64 U
        assert (table.double().cpu() - t).abs().max() <= 6 * 0.05 * 500 * 64 * U


def test_two_graphs_and_two_streams_at_once():
    """Two captured calls replayed on two streams together with an eager one: none shares scratch."""
    gen = _rng(31)
    rows, dim, bags = 3000, 64, 20000
    cases = []
    for k in range(3):
        tok = torch.randint(0, rows, (bags,), generator=gen).cuda()
        g = torch.randn(bags, dim, generator=gen).cuda()
        cases.append((tok, g, arb.embedding_grad(g, tok, rows).clone()))
    graphs, outs = [], []
    for tok, g, _ in cases[:2]:
        arb.embedding_grad(g, tok, rows)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(arb.embedding_grad(g, tok, rows))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            third = arb.embedding_grad(cases[2][1], cases[2][0], rows)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], cases[0][2]) and torch.equal(outs[1], cases[1][2]) and torch.equal(third, cases[2][2])


def test_a_device_that_is_not_there():
    """The C entry points take a device ordinal that exists, or say so."""
    t = torch.zeros(4, 4, device="cuda")
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    o = torch.zeros(2, 4, device="cuda")
    e = arb.lib().AEmbedding(t.data_ptr(), 0, 4, 4, 4, i.data_ptr(), 4, 2, 1, 1, 0, 1.0, o.data_ptr(), 0, 4, 4095, None)
    assert e is not None and b"CUDA error" in e
    assert torch.equal(arb.embedding(i, t), o)  # and the context is as it was


# ---- a forest's leaf values ------------------------------------------------------------------
def _grown(objective, rounds=5, rows=300, depth=4, classes=3):
    rng = np.random.default_rng(objective + 7)
    X = rng.normal(size=(rows, 6)).astype(np.float32)
    X[::17, 2] = np.nan
    score = X[:, 0] - 0.5 * np.nan_to_num(X[:, 2]) + rng.normal(size=rows) * 0.3
    cfg = {"objective": objective, "method": 1, "internals": {"hist_size": 63, "seed": 0},
           "verbose": {"gpu": False, "booster": False, "data": False},
           "tree": {"eta": 0.2, "max_depth": depth, "lambda": 1.0, "min_child_weight": 1.0, "initial_y": 0.4}}
    target = {"y": score.astype(np.float32)}
    if objective == 1:
        target = {"y": (score > 0).astype(np.float32)}
    if objective == 3:
        cfg["tree"]["labels_count"] = classes
        target = {"labels": np.digitize(score, [-0.5, 0.5]).astype(np.uint8)}
    data = arb.DMatrix(X, **target)
    return arb.train(cfg, data, rounds), data, X, target


def _weights(model):
    import json
    return np.array([t["weights"] for t in json.loads(model.dump())["model"]])


def _link(objective, yhat):
    if objective == 1:
        return 1 / (1 + np.exp(-yhat))
    if objective == 3:
        e = np.exp(yhat - yhat.max(1, keepdims=True))
        return e / e.sum(1, keepdims=True)
    return yhat


@pytest.mark.parametrize("objective", [0, 1, 3])
def test_refined_leaves_follow_the_formula(objective):
    """Tokens, lookup, gradient by token and AdamW step together, against the same steps in 64 bits."""
    model, data, X, target = _grown(objective)
    K = 3 if objective == 3 else 1
    n = len(X)
    tok = model.leaf_tokens(data)
    w = _weights(model).astype(np.float64)
    T, leaves = w.shape
    assert tok.shape == (n, T) and tok.dtype == np.int32
    leaf = tok - np.arange(T) * leaves
    assert (leaf >= 0).all() and (leaf < leaves).all()
    out = torch.empty(T, n, dtype=torch.int32, device="cuda")
    assert np.array_equal(model.leaf_tokens(data, out=out).cpu().numpy(), tok)
    assert np.array_equal(model.leaf_tokens(data, n_rounds=2), tok[:, :2])
    start = 0.4 if objective != 1 else np.log(0.4 / 0.6)

    def yhat(w):
        each = w[np.arange(T), leaf]
        return np.stack([each[:, k::K].sum(1) for k in range(K)], 1)
    # a prediction: a float32 sum of T leaf values and the start
    off = (T + 2) * U * (np.abs(w[np.arange(T), leaf]).sum(1).max() + abs(start))
    got = model.predict(data).reshape(n, K)
    assert np.abs(got - _link(objective, yhat(w) + start)).max() <= off + 4 * U
    lr, b1, b2, eps, wd, steps = 0.05, 0.9, 0.99, 1e-2, 0.02, 4
    m, v = np.zeros_like(w), np.zeros_like(w)
    largest = 0.0
    for s in range(1, steps + 1):
        p = _link(objective, yhat(w) + start)
        r = p - (np.eye(K)[target["labels"]] if objective == 3 else target["y"].astype(np.float64)[:, None])
        largest = max(largest, np.abs(r).max())
        g = np.zeros_like(w)
        for t in range(T):
            g[t] = np.bincount(leaf[:, t], weights=r[:, t % K] / n, minlength=leaves)
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        w = w * (1 - lr * wd) - lr / (1 - b1 ** s) * m / (np.sqrt(v / (1 - b2 ** s)) + eps)
    model.refine_leaves(data, steps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd)
    # a gradient is a float32 sum of at most n residuals, each off by a few roundings; a step passes its
    # error on with a slope of at most lr / eps (twice: once through m, once through the root), and the
    # moved values change the next residuals by no more than that again
    slack = (n + 8) * U * largest * lr / eps * 2 * steps * 2
    assert np.abs(_weights(model) - w).max() <= slack + 16 * U * np.abs(w).max()
    got = model.predict(data).reshape(n, K)
    assert np.abs(got - _link(objective, yhat(_weights(model)) + start)).max() <= off * 2 + 8 * U
    again = arb.load(model.dump())
    again.labels_count = K
    assert np.array_equal(again.predict(data).reshape(n, K), got)
    # training goes on from the moved values
    model.grow_tree()
    grown = _weights(model)
    assert np.array_equal(grown[:T].astype(np.float32), _weights(again).astype(np.float32)) and len(grown) == T + K
    internal = model.train_yhat().T
    assert np.abs(_link(objective, internal.astype(np.float64)) - model.predict(data).reshape(n, K)).max() <= 2 * off + 8 * U


def test_refinement_in_8_bits_and_without_steps():
    model, data, X, target = _grown(0)
    before = _weights(model)
    model.refine_leaves(data, 0)
    assert np.array_equal(_weights(model), before)
    # each step moves a value by lr times a ratio of at most sqrt(1 / (1 - 0.999)) or so; here by less than 2 lr
    model.refine_leaves(data, 10, lr=1e-3, state_bits=8)
    after = _weights(model)
    assert np.isfinite(after).all() and not np.array_equal(after, before) and np.abs(after - before).max() < 10 * 2e-3
    loaded = arb.load(model.dump())
    other = arb.DMatrix(X, **target)
    loaded.refine_leaves(other, 3)  # a loaded model, another matrix
    assert not np.array_equal(_weights(loaded), after)


def test_refinement_refuses():
    model, data, X, _ = _grown(0, rounds=1)
    with pytest.raises(arb.ArboretumError, match="no targets"):
        model.refine_leaves(arb.DMatrix(X), 1)
    with pytest.raises(arb.ArboretumError, match="betas"):
        model.refine_leaves(data, 1, betas=(1.0, 0.9))
    with pytest.raises(arb.ArboretumError, match="feature"):
        model.refine_leaves(arb.DMatrix(X[:, :1], y=X[:, 0]), 1)
    with pytest.raises(ValueError, match="out must be"):
        model.leaf_tokens(data, out=torch.empty(2, 300, dtype=torch.int32, device="cuda"))


def test_refinement_of_many_rows():
    """The order kept by runs of bags, and the table in shared memory: the same operators at a size
    where the library chooses them, against the lookups of the public functions."""
    rng = np.random.default_rng(3)
    rows = 120000
    X = rng.normal(size=(rows, 5)).astype(np.float32)
    y = (X[:, 0] * 2 + rng.normal(size=rows) * 0.1).astype(np.float32)
    cfg = {"objective": 0, "method": 1, "internals": {"hist_size": 63, "seed": 0},
           "verbose": {"gpu": False, "booster": False, "data": False}, "tree": {"eta": 0.1, "max_depth": 3, "initial_y": 0.0}}
    data = arb.DMatrix(X, y=y)
    model = arb.train(cfg, data, 8)
    T, leaves = _weights(model).shape
    tok = model.leaf_tokens(data, out=torch.empty(T, rows, dtype=torch.int32, device="cuda"))
    table = torch.tensor(_weights(model), dtype=F32, device="cuda").view(-1, 1)
    target = torch.tensor(y, device="cuda")[:, None]
    grad = torch.zeros_like(table)
    o = arb.AdamW(list(table.view(T, leaves)), lr=0.01, eps=1e-8, weight_decay=0.0,
                  grads=list(grad.view(T, leaves)))
    order = arb.token_order(tok, T * leaves, pooled=True)
    for _ in range(3):
        r = (arb.embedding(tok, table, pooled=True) + 0.0 - target) * np.float32(1.0 / rows)
        arb.embedding_grad(r, order, T * leaves, out=grad)
        o.step()
    model.refine_leaves(data, 3, lr=0.01)
    assert np.array_equal(_weights(model).astype(np.float32), table.view(T, leaves).cpu().numpy())


@pytest.mark.parametrize("objective", [0, 3])
def test_accumulated_predictions_follow_refined_leaves(objective):
    """A matrix that rounds were added to gives the refined values' predictions, in the bits of predict."""
    grown, data, X, target = _grown(objective)
    some = lambda n: arb.DMatrix(X[:n], **{k: v[:n] for k, v in target.items()})  # noqa: E731
    models = []
    for _ in range(2):
        models.append(arb.Garden(grown.config, data))
        models[-1].labels_count = grown.labels_count
    model, other = models
    kept, shared = some(200), some(150)
    for _ in range(3):
        model.grow_tree()
        model.append_last_tree(kept)
    assert np.array_equal(model.get_y(kept), model.predict(kept))
    before = model.get_y(kept)
    model.refine_leaves(data, 3, lr=0.05)
    assert np.array_equal(model.get_y(kept), model.predict(kept)) and not np.array_equal(model.get_y(kept), before)
    model.grow_tree()
    model.append_last_tree(kept)
    model.refine_leaves(data, 2, lr=0.05)
    model.grow_tree()
    model.append_last_tree(kept)  # the rounds before follow here too
    assert np.array_equal(model.get_y(kept), model.predict(kept))
    # two models added to one matrix: what cannot follow says so, the other model's call goes on
    other.grow_tree()
    model.append_last_tree(shared)
    other.append_last_tree(shared)
    mixed = model.get_y(shared)
    assert np.array_equal(other.get_y(shared), mixed)
    model.refine_leaves(data, 1)
    with pytest.raises(arb.ArboretumError, match="another model"):
        model.get_y(shared)
    with pytest.raises(arb.ArboretumError, match="another model"):
        model.append_last_tree(shared)
    assert np.array_equal(other.get_y(shared), mixed)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_smallest_eps_without_gradients(bits):
    """0 / (0 + eps) is 0 for the smallest eps there is."""
    p = torch.ones(300, device="cuda")
    o = arb.AdamW([p], eps=2.0 ** -126, weight_decay=0.0, state_bits=bits)
    o.step([torch.zeros(300, device="cuda")])
    assert (p == 1).all()
    with pytest.raises(arb.ArboretumError, match="2.-126"):
        arb.AdamW([p], eps=1e-40)


@pytest.mark.parametrize("empty", [0, 1, 2])
def test_adamw_bound_gradients_with_an_empty_parameter(empty):
    """Tensors of no elements take part wherever they stand, with gradients given once or every time."""
    sizes = [300, 41]
    sizes.insert(empty, 0)
    make = lambda: [torch.ones(n, device="cuda") for n in sizes]  # noqa: E731
    a, b, grads = make(), make(), make()
    bound, given = arb.AdamW(a, grads=grads), arb.AdamW(b)
    left_out = arb.AdamW(make(), grads=[g if len(g) != 41 else None for g in grads])
    for _ in range(2):
        bound.step()
        given.step(grads)
        left_out.step()
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and (a[sizes.index(41)] < 1).all()
    assert bound.steps == given.steps == left_out.steps == 2
    assert (left_out.params[sizes.index(41)] == 1).all() and torch.equal(left_out.params[sizes.index(300)], a[sizes.index(300)])
    grads[sizes.index(41)].data = torch.ones(41, device="cuda")
    with pytest.raises(ValueError, match="gradient's memory has moved"):
        bound.step()
    left_out.step()


def test_gradients_and_outputs_whose_memory_is_gone_are_refused():
    p = torch.ones(10, device="cuda")
    o = arb.AdamW([p])
    whole = torch.ones(20, device="cuda")
    parts = whole[:10], whole[10:]
    o.step([parts[1]])
    whole.untyped_storage().resize_(0)
    for g in parts:
        with pytest.raises(ValueError, match="memory"):
            o.step([g])
        with pytest.raises(ValueError, match="memory"):
            arb.AdamW([torch.ones(10, device="cuda")], grads=[g])
    assert o.steps == 1
    out, table = torch.zeros(24, device="cuda")[12:].view(3, 4), torch.ones(3, 4, device="cuda")
    out.untyped_storage().resize_(0)
    i = torch.zeros(3, dtype=torch.int64, device="cuda")
    for call in (lambda: arb.embedding(i, table, out=out), lambda: arb.embedding_grad(table, i, 3, out=out)):
        with pytest.raises(ValueError, match="memory"):
            call()


def test_autograd_sees_every_tensor_written_in_place():
    """A backward pass that needs what a call has overwritten says so, whatever way the tensor went in."""
    gen = _rng(5)
    w = torch.ones(3, 4, device="cuda", requires_grad=True)
    tok, table = torch.tensor([1, 0, 2], device="cuda"), torch.randn(3, 4, generator=gen).cuda()
    order = arb.token_order(tok, 3)
    for write in (lambda x: arb.embedding(tok, table, out=x), lambda x: arb.embedding(tok.view(1, 3).t(), table, pooled=True, out=x),
                  lambda x: arb.embedding_grad(table, tok, 3, out=x), lambda x: arb.embedding_grad(table, order, 3, out=x, accumulate=True),
                  lambda x: arb.AdamW([x]).step([table]), lambda x: arb.AdamW([x.detach()]).step([table]),
                  lambda x: arb.AdamW([x.view(12)]).step([table.view(12)])):
        x = torch.randn(3, 4, generator=gen).cuda()
        y = (x * w).sum()
        write(x)
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
    # what a call has only read, or left as it was, stays usable
    x = torch.randn(3, 4, generator=gen).cuda()
    y = (x * w).sum()
    arb.embedding(tok, x)
    arb.embedding_grad(x, tok, 3)
    arb.AdamW([x, torch.ones(4, device="cuda")]).step([None, table[0].contiguous()])
    y.backward()
    assert torch.equal(w.grad, x)


def test_leaf_tokens_written_in_place_are_seen():
    model, data, X, _ = _grown(0)
    out = torch.zeros(5, len(X), dtype=torch.int32, device="cuda")
    values = torch.ones(5 * 8, 2, device="cuda", requires_grad=True)
    y = torch.nn.functional.embedding(out, values).sum()
    model.leaf_tokens(data, out=out)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_inference_tensors():
    """They have no version to count, with and without a gradient asked for."""
    with torch.inference_mode():
        p, q = torch.ones(10, device="cuda"), torch.ones(10, device="cuda").requires_grad_()
        out, tok, table = torch.zeros(3, 4, device="cuda"), torch.tensor([1, 0, 2], device="cuda"), torch.ones(3, 4, device="cuda")
        o = arb.AdamW([p, q])
        o.step([torch.ones(10, device="cuda")] * 2)
    o.step([torch.ones(10, device="cuda")] * 2)
    arb.embedding(tok, table, out=out)
    arb.embedding_grad(table, tok, 3, out=out, accumulate=True)
    assert torch.equal(p, q) and (p < 1).all() and o.steps == 2 and (out == 2).all()
    with torch.inference_mode():
        arb.embedding(tok, table, out=out)
        assert (out == 1).all()


def test_tangents_are_refused():
    from torch.autograd import forward_ad
    i, t = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.ones(3, 4, device="cuda")
    o = arb.AdamW([t.clone()])
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, torch.ones_like(t))
        for call in (lambda: arb.embedding(i, dual), lambda: arb.embedding(i, t, out=dual.clone()), lambda: arb.embedding_grad(dual, i, 3),
                     lambda: arb.AdamW([dual]), lambda: o.step([dual]), lambda: arb.AdamW([t], grads=[dual]),
                     lambda: o.step([t], grad_scale=dual[0, :1])):
            with pytest.raises(ValueError, match="tangent"):
                call()
    for call in (lambda x: arb.embedding(i, x), lambda x: arb.embedding_grad(x, i, 3)):
        for transform in (lambda f: torch.func.jvp(f, (t,), (t,)), lambda f: torch.vmap(f)(t[None]), lambda f: torch.func.vjp(f, t)):
            with pytest.raises((ValueError, RuntimeError)):
                transform(call)
    assert o.steps == 0


def test_views_to_be_negated_are_refused():
    i, t = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.ones(3, 4, device="cuda")
    turned = torch._neg_view(torch.ones(3, 4, device="cuda"))
    o = arb.AdamW([t])
    for call in (lambda: arb.embedding(i, t, out=turned), lambda: arb.embedding_grad(t, i, 3, out=turned), lambda: o.step([turned]),
                 lambda: arb.AdamW([turned]), lambda: arb.AdamW([t], grads=[turned]), lambda: o.step([t], lr=turned[0, :1]),
                 lambda: o.step([t], grad_scale=turned[0, :1])):
        with pytest.raises(ValueError, match="negated"):
            call()
    assert torch.equal(arb.embedding(i, turned.resolve_neg()), -t) and o.steps == 0


def test_leaf_tokens_on_the_models_device():
    import ctypes
    model, data, X, _ = _grown(0)
    device = ctypes.c_int(-1)
    assert arb.lib().AModelDevice(model.handle, ctypes.byref(device)) is None and device.value == torch.cuda.current_device()
    want = model.leaf_tokens(data)
    out = torch.empty(5, len(X), dtype=torch.int32, device=torch.device("cuda", device.value))
    assert np.array_equal(model.leaf_tokens(data, out=out).cpu().numpy(), want)
    if torch.cuda.device_count() > 1:
        with pytest.raises(ValueError, match="the model works on"):
            model.leaf_tokens(data, out=out.to("cuda:%d" % (1 - device.value)))


@pytest.mark.parametrize("bags,per_bag,rows,dim", [(200000, 2, 3, 8), (100003, 3, 1, 40), (300007, 2, 600, 256), (70001, 5, 2, 7),
                                                   (70001, 5, 2, 1), (65536, 4, 2, 3)])
def test_sums_of_equal_values_do_not_drift(bags, per_bag, rows, dim):
    """Sums of one sign over an order kept by runs, where every rounding can go the same way: the limit
    follows from the longest chain of additions, not from the number of terms."""
    gen = _rng(bags, rows)
    tok = torch.randint(0, rows, (bags, per_bag), generator=gen)
    tok[:, 0] = 0  # a row that every bag names
    count = torch.bincount(tok.view(-1), minlength=rows).double()[:, None]
    if dim > 3:
        # eight bags: seven additions; sums of eights in 64 bits, rounded a share; their join in 64 bits, rounded, times scale
        chain = 7 + 1 + 2
    else:
        # eight bags: seven; a warp's 32 vectors: five; what the 32 before them carry on: one for every 256
        # bags of a row in a run of 16383 bags; the join as above
        chain = 7 + 5 + -(-16383 * per_bag // 256) + 1 + 2
    for dtype in (F32, BF16):
        value = torch.tensor(0.1).to(dtype)
        got = arb.embedding_grad(value.expand(bags, dim).contiguous().cuda(), tok.cuda(), rows, scale=0.3, pooled=True, out_dtype=F32)
        want = count * value.double() * float(np.float32(0.3))
        assert ((got.double().cpu() - want).abs() <= (chain + 1) * U * want).all(), float(((got.double().cpu() - want) / want).abs().max() / U)


@pytest.mark.parametrize("bags,per_bag,dim", [(1, 1 << 20, 1), (1, 1 << 20, 64), (3, 300000, 257), (300, 65536, 1), (2000, 4097, 2), (2000, 4096, 2),
                                              (2, 1025, 1030), (64, 2500, 2048)])
def test_long_bags_do_not_drift(bags, per_bag, dim):
    """Equal values, where every rounding can go the same way: at most 4096 rows are added in one chain, and
    the sums of 1024 rows after one another; a whole CTA's lanes may share a bag."""
    chain = max(4096, 1024 + per_bag // 1024 + 1) + 8 + 1
    for dtype in (F32, F16):
        table = torch.full((3, dim), 0.1, dtype=dtype, device="cuda")
        want = per_bag * table[0, 0].double().cpu() * float(np.float32(0.3))
        rows = torch.randint(0, 3, (per_bag, bags), generator=_rng(bags, per_bag), dtype=torch.int32).cuda()
        for tok in (rows.t(), rows.t().contiguous()):
            got = arb.embedding(tok, table, scale=0.3, pooled=True, out_dtype=F32)
            assert got.shape == (bags, dim) and ((got.double().cpu() - want).abs() <= chain * U * want).all()
    # and the sums themselves: integers, exact in any order
    table = torch.randint(-3, 4, (500, dim), generator=_rng(dim)).float()
    tok = torch.randint(-1, 500, (per_bag, bags), generator=_rng(per_bag), dtype=torch.int32)
    total = torch.zeros(bags, dim, dtype=torch.float64)
    for b in range(min(bags, 8)):
        n = torch.bincount(tok[:, b].long() + 1, minlength=501)[1:].double()
        total[b] = n @ table.double()
    for view in (tok.cuda().t(), tok.cuda().t().contiguous()):
        assert torch.equal(arb.embedding(view, table.cuda(), pooled=True).cpu().double()[:8], total[:8])


@pytest.mark.parametrize("bags,per_bag,rows,dim", [(40000, 1, 3000, 24), (33000, 1, 40000 * 17, 3), (40000, 5, 90, 2), (40000, 5, 90, 7), (1000, 3, 50, 70),
                                                   (9, 1, 300000, 5), (0, 2, 40, 4)])
def test_orders_in_graphs_and_on_other_streams(bags, per_bag, rows, dim):
    """Every sort captured and replayed on new tokens; an order made on one stream and used on another
    after its owner let it go."""
    gen = _rng(bags, rows, dim)
    make = lambda: (_tokens(bags, per_bag, rows, torch.int32, gen).cuda(), torch.randn(bags, dim, generator=gen).cuda())  # noqa: E731
    tok, g = make()
    want = arb.embedding_grad(g, tok, rows, pooled=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = arb.embedding_grad(g, tok, rows, pooled=True)
        order = arb.token_order(tok, rows, pooled=True)
        kept = arb.embedding_grad(g, order, rows)
        bags_out = arb.embedding(tok, kept, pooled=True)
    for _ in range(3):
        out.fill_(7)
        kept.fill_(7)
        graph.replay()
        assert torch.equal(out, want) and torch.equal(kept, want) and torch.equal(bags_out, arb.embedding(tok, want, pooled=True))
        new = make()
        tok.copy_(new[0])
        g.copy_(new[1])
        want = arb.embedding_grad(g, tok, rows, pooled=True)
    side = torch.cuda.Stream()
    order = arb.token_order(tok, rows, pooled=True)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = arb.embedding_grad(g, order, rows)
    size = order._order[0].numel()
    del order
    torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # would take the order's memory, were it free already
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


@pytest.mark.parametrize("rows,trees", [(1, 1), (33, 3), (20011, 70)])
def test_leaf_tokens_of_other_sizes(rows, trees):
    """Against a walk of the dumped trees."""
    import json
    model, data, X, _ = _grown(0, rounds=trees)
    rng = np.random.default_rng(rows)
    Z = rng.normal(size=(rows, 6)).astype(np.float32)
    Z[rng.random(Z.shape) < 0.05] = np.nan
    tok = model.leaf_tokens(arb.DMatrix(Z))
    dumped = json.loads(model.dump())["model"]
    leaves = len(dumped[0]["weights"])
    assert tok.shape == (rows, trees)
    for t, tree in enumerate(dumped):
        nodes = {n["id"]: n for n in tree["nodes"]}
        at = np.zeros(rows, int)
        for _ in range(tree["depth"] - 1):
            fid = np.array([nodes[i]["fid"] for i in range(leaves - 1)])
            thr = np.array([np.inf if nodes[i]["threshold"] is None else nodes[i]["threshold"] for i in range(leaves - 1)], np.float32)
            left = Z[np.arange(rows), fid[at]] < thr[at]  # NaN goes right
            at = 2 * at + np.where(left, 1, 2)
        assert np.array_equal(tok[:, t], t * leaves + at - (leaves - 1))


def test_a_state_that_is_refused_changes_nothing():
    p = torch.ones(200, device="cuda")
    o = arb.AdamW([p])
    o.step([torch.ones(200, device="cuda")])
    kept = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in o.state_dict().items()}
    zeros = torch.zeros(256, device="cuda")
    for bad in (dict(step=-1), dict(step="x"), dict(step=None), dict(moment1=zeros[:200]), dict(moment2=zeros.half())):
        state = dict(step=5, moment1=zeros, moment2=zeros)
        state.update(bad)
        with pytest.raises((ValueError, TypeError, arb.ArboretumError)):
            o.load_state_dict(state)
        assert o.steps == 1 and torch.equal(o.moment1, kept["moment1"]) and torch.equal(o.moment2, kept["moment2"])
