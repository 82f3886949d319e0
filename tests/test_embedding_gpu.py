"""Embedding lookup, grouping of ids and embedding gradient (loops_amd/embedding.py) against plain fp64 arithmetic on the host.

Tolerances.  u = finfo(type).eps / 2 is the largest relative rounding of a store, e = 2^-24 that of a float32 operation.
Lookup: one float product (e) and one store (u): |error| <= (u + e)(1 + e) |scale * w|, taken as (u + 2e) |scale * w| (float32: 2e).
Gradient: a row of m tokens is m float additions in some order (each rounds the partial sum by at most e, partial sums are at most
the sum of magnitudes A), joined from parts (additions as well), then one product or fused multiply-add (e) and one store (u):
|error| <= |scale| A m e (1 + e)^m + (u + e) (|result| + ...), taken as 1.01 |scale| A (m + 2) e + (u + e) |result| (adding: the old value
counts in the result and, through the fused multiply-add, adds no rounding of its own).  f16: results below its smallest normal number round
by half a spacing, 2^-25."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2 if dtype is not torch.float32 else E


def _tiny(dtype):
    return 2.0 ** -25 if dtype is torch.float16 else 0.0


def _check(got, want, bound):
    got = got.detach().cpu().double().numpy()
    assert got.shape == want.shape
    worst = np.abs(got - want) - bound
    assert not np.isnan(got).any() and (worst <= 0).all(), (np.unravel_index(np.argmax(worst), worst.shape), worst.max())


def _ids(rng, n, rows, kind):
    if kind == "uniform":
        return rng.integers(0, rows, n)
    if kind == "zipf":
        return np.minimum((np.exp(rng.random(n) * np.log(rows + 1.0)) - 1).astype(np.int64), rows - 1)
    if kind == "one":
        return np.full(n, rows // 2)
    if kind == "ends":
        return rng.choice([0, rows - 1], n)
    if kind == "outside":
        return rng.choice([-1, -5, rows, rows + 7, 2 ** 31 - 1, -2 ** 31], n)
    assert kind == "mixed"
    ids = rng.integers(-rows // 2, rows + rows // 2 + 1, n)
    ids[::3] = rows // 3
    return ids


def _matrix(rng, rows, cols, dtype, pitch=None):
    """[rows, cols] of the type on the GPU, `pitch` elements between rows, and the same in float64."""
    m = torch.from_numpy(rng.standard_normal((rows, pitch or cols)).astype(np.float32)).to(dtype)
    return m.cuda()[:, :cols], m[:, :cols].double().numpy()


# ---- lookup -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("dim,pitch", [(1, None), (3, 4), (7, None), (8, None), (9, None), (64, None), (100, 104), (513, None), (1001, 1024), (4096, None)])
def test_lookup(dtype, id_type, dim, pitch):
    from loops_amd import embedding
    rng = np.random.default_rng(dim * 7 + (pitch or 0))
    rows = 211
    table, wide = _matrix(rng, rows, dim, dtype, pitch)
    for n, kind, first, scale in [(1, "uniform", 0, 1.0), (2, "outside", 0, 3.0), (65, "mixed", 0, -0.37), (257, "zipf", 40, dim ** 0.5)]:
        ids = _ids(rng, n, rows, kind)
        out = torch.full((n, dim), 7.0, dtype=dtype, device="cuda")
        got = embedding.lookup(table, torch.from_numpy(ids).to(id_type).cuda(), scale=scale, first_id=first, out=out)
        assert got is out
        at = torch.from_numpy(ids).to(id_type).long().numpy() - first
        inside = (at >= 0) & (at < rows)
        want = np.where(inside[:, None], wide[np.where(inside, at, 0)], 0.0) * np.float32(scale).astype(np.float64)
        _check(got, want, (_half_step(dtype) + 2 * E) * np.abs(want) + _tiny(dtype))
        assert (got.cpu().numpy()[~inside] == 0).all() if dtype is not torch.bfloat16 else (got.cpu().float().numpy()[~inside] == 0).all()


def test_lookup_into_padded_rows_leaves_the_padding():
    from loops_amd import embedding
    rng = np.random.default_rng(5)
    for dtype in TYPES:
        for dim, pitch in [(5, 6), (77, 80), (520, 523)]:
            table, wide = _matrix(rng, 50, dim, dtype)
            buffer = torch.full((33, pitch), 9.0, dtype=dtype, device="cuda")
            ids = torch.from_numpy(rng.integers(0, 50, 33)).cuda()
            embedding.lookup(table, ids, out=buffer[:, :dim])
            assert torch.equal(buffer[:, :dim], table[ids])
            assert (buffer[:, dim:] == 9.0).all()


def test_lookup_many_packets_and_shapes():
    """More packets than the small launch takes; tokens of two dimensions; values that are not finite stay in their places."""
    from loops_amd import embedding
    rng = np.random.default_rng(6)
    table, wide = _matrix(rng, 1000, 2056, torch.bfloat16)
    table[7, 5], table[7, 6], table[8, 2055] = float("inf"), float("-inf"), float("nan")
    tokens = torch.from_numpy(rng.integers(0, 1000, (16, 515))).cuda()
    tokens[3, 4], tokens[3, 5] = 7, 8
    got = embedding.lookup(table, tokens)
    assert got.shape == (16, 515, 2056) and got.dtype is torch.bfloat16
    assert torch.equal(got.isnan(), table[tokens].isnan())
    assert torch.equal(got.nan_to_num(), table[tokens].nan_to_num())
    assert embedding.lookup(table, tokens[:0]).shape == (0, 515, 2056)
    assert (embedding.lookup(table[:0], tokens) == 0).all()


# ---- grouping -----------------------------------------------------------------------------------------------------------------
def _groups(ids, rows, first=0, drop=-1):
    ids = ids.astype(np.int64)
    key = np.where((ids >= first) & (ids < first + rows) & (ids != drop), ids - first, rows)
    order = np.argsort(key, kind="stable")
    return key[order].astype(np.int32), order.astype(np.int32)


@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 1000, 1024, 1025, 4096, 4097, 8192, 8193, 20000, 70001])
@pytest.mark.parametrize("rows", [1, 2, 511, 512, 1023, 1024, 50021, 131072, 2 ** 20, 2 ** 30])
def test_group_tokens(n, rows):
    from loops_amd import embedding
    rng = np.random.default_rng(n * 31 + rows % 1000)
    for kind, id_type in [("uniform", torch.int64), ("zipf", torch.int32), ("one", torch.int32), ("ends", torch.int64), ("outside", torch.int64), ("mixed", torch.int32)]:
        ids = _ids(rng, n, rows, kind)
        ids = torch.from_numpy(ids).to(id_type)
        got = embedding.group_tokens(ids.cuda(), rows)
        key, order = _groups(ids.numpy(), rows)
        assert got.rows == rows and got.ids.dtype is torch.int32 and got.positions.dtype is torch.int32
        assert np.array_equal(got.ids.cpu().numpy(), key), kind
        assert np.array_equal(got.positions.cpu().numpy(), order), kind


def test_group_tokens_first_and_dropped_ids():
    from loops_amd import embedding
    rng = np.random.default_rng(3)
    for n in (300, 9001):
        ids = rng.integers(0, 4000, n)
        got = embedding.group_tokens(torch.from_numpy(ids).cuda(), 1000, first_id=1500, drop_id=1777)
        key, order = _groups(ids, 1000, 1500, 1777)
        assert np.array_equal(got.ids.cpu().numpy(), key) and np.array_equal(got.positions.cpu().numpy(), order)
    big = torch.from_numpy(rng.integers(0, 1000, 500) + 2 ** 40).cuda()  # ids past 32 bits
    got = embedding.group_tokens(big, 1000, first_id=2 ** 40)
    key, order = _groups(big.cpu().numpy(), 1000, 2 ** 40)
    assert np.array_equal(got.ids.cpu().numpy(), key) and np.array_equal(got.positions.cpu().numpy(), order)


def test_group_tokens_many_spans():
    """More than 256 times 4 096 positions: longer spans; expert choices of two dimensions."""
    from loops_amd import embedding
    rng = np.random.default_rng(4)
    for rows in (256, 131072):
        ids = rng.integers(-1, rows, (150001, 8)).astype(np.int32)
        got = embedding.group_tokens(torch.from_numpy(ids).cuda(), rows)
        key, order = _groups(ids.reshape(-1), rows)
        assert np.array_equal(got.ids.cpu().numpy(), key) and np.array_equal(got.positions.cpu().numpy(), order)


# ---- gradient -----------------------------------------------------------------------------------------------------------------
def _gradient(ids, grad, rows, scale, old=None):
    """(result, bound without the store's rounding) in float64."""
    keep = (ids >= 0) & (ids < rows)
    total, size, many = np.zeros((rows, grad.shape[1])), np.zeros((rows, grad.shape[1])), np.zeros(rows)
    np.add.at(total, ids[keep], grad[keep])
    np.add.at(size, ids[keep], np.abs(grad[keep]))
    np.add.at(many, ids[keep], 1)
    scale = float(np.float32(scale))
    want = total * scale + (0 if old is None else old)
    return want, 1.01 * abs(scale) * size * (many + 2)[:, None] * E, many


@pytest.mark.parametrize("dtype,out_type", [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32),
                                            (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("dim", [1, 5, 8, 64, 67, 513, 1001, 1024])
def test_gradient(dtype, out_type, dim):
    from loops_amd import embedding
    rng = np.random.default_rng(dim)
    for n, rows, kind in [(0, 9, "uniform"), (1, 1, "uniform"), (1, 300, "uniform"), (70, 1, "one"), (129, 40, "mixed"), (1000, 500, "zipf"), (700, 33, "ends"),
                          (3000, 77, "one"), (64, 64, "outside"), (2500, 3000, "zipf")]:
        ids = _ids(rng, n, rows, kind)
        grad, wide = _matrix(rng, n, dim, dtype)
        groups = embedding.group_tokens(torch.from_numpy(ids).cuda(), rows)
        for scale, add in [(1.0, False), (-0.3, False), (dim ** 0.5 / 8, True)]:
            old, old_wide = _matrix(rng, rows, dim, out_type)
            before = old.clone()
            want, bound, many = _gradient(ids, wide, rows, scale, old_wide if add else None)
            if add:
                got = embedding.gradient(groups, grad, scale=scale, out=old, accumulate=True)
                assert got is old
                untouched = torch.from_numpy(many == 0).cuda()
                assert torch.equal(got[untouched], before[untouched])
                bound, want = bound[many > 0], want[many > 0]
                _check(got[~untouched], want, bound + (_half_step(out_type) + E) * np.abs(want) * 1.001 + _half_step(out_type) * bound + _tiny(out_type))
            else:
                got = embedding.gradient(groups, grad, scale=scale, dtype=out_type)
                assert got.dtype is out_type
                _check(got, want, bound + (_half_step(out_type) + E) * np.abs(want) * 1.001 + _half_step(out_type) * bound + _tiny(out_type))
                assert (got[torch.from_numpy(many == 0).cuda()] == 0).all()


@pytest.mark.parametrize("add", [False, True])
def test_gradient_long_rows_over_many_tiles(add):
    """One id holds most of 30 000 tokens: its sum is joined from hundreds of tiles; two runs give the same bits."""
    from loops_amd import embedding
    rng = np.random.default_rng(8)
    n, rows, dim = 30000, 700, 72
    ids = _ids(rng, n, rows, "zipf")
    ids[rng.random(n) < 0.7] = 350
    grad, wide = _matrix(rng, n, dim, torch.bfloat16)
    groups = embedding.group_tokens(torch.from_numpy(ids).cuda(), rows)
    old, old_wide = _matrix(rng, rows, dim, torch.float32)
    outs = [embedding.gradient(groups, grad, out=old.clone(), accumulate=add) for _ in range(2)]
    assert torch.equal(*outs)
    want, bound, _ = _gradient(ids, wide, rows, 1.0, old_wide if add else None)
    _check(outs[0], want, bound + 2 * E * np.abs(want))


def test_gradient_is_the_derivative_of_the_lookup():
    """<G, lookup(W + h D)> - <G, lookup(W - h D)> = 2 h <gradient(G), D>: the lookup is linear, so differences are exact but for
    rounding: integers, and a scale that is a power of two, leave none."""
    from loops_amd import embedding
    rng = np.random.default_rng(9)
    rows, dim, n = 60, 33, 500
    whole = lambda *shape: torch.from_numpy(rng.integers(-4, 5, shape).astype(np.float32)).cuda()  # noqa: E731
    w, d, g = whole(rows, dim), whole(rows, dim), whole(n, dim)
    tokens = torch.from_numpy(_ids(rng, n, rows, "mixed")).cuda()
    up, down = embedding.lookup(w + d, tokens, scale=0.5), embedding.lookup(w - d, tokens, scale=0.5)
    left = ((up.double() - down.double()) * g.double()).sum() / 2
    right = (embedding.gradient(embedding.group_tokens(tokens, rows), g, scale=0.5).double() * d.double()).sum()
    assert left.item() == right.item() and right.item() != 0


def test_gradient_strides_and_shapes():
    from loops_amd import embedding
    rng = np.random.default_rng(10)
    rows, dim = 90, 75
    tokens = torch.from_numpy(rng.integers(0, rows, (6, 50))).cuda()
    groups = embedding.group_tokens(tokens, rows)
    for dtype in TYPES:
        grad, wide = _matrix(rng, 300, dim, dtype, 81)
        want, bound, _ = _gradient(tokens.cpu().numpy().reshape(-1), wide, rows, 1.0)
        buffer = torch.full((rows, 83), 5.0, dtype=dtype, device="cuda")
        embedding.gradient(groups, grad, out=buffer[:, :dim])
        _check(buffer[:, :dim], want, bound * 1.01 + (_half_step(dtype) + E) * np.abs(want) * 1.001 + _tiny(dtype))
        assert (buffer[:, dim:] == 5.0).all()
        assert torch.equal(embedding.gradient(groups, grad.contiguous().view(6, 50, dim)), buffer[:, :dim])


def test_gradient_keeps_dropped_tokens_out():
    """Gradient rows of tokens without a row of the table may hold anything."""
    from loops_amd import embedding
    rng = np.random.default_rng(11)
    rows, dim, n = 40, 24, 200
    ids = rng.integers(0, rows, n)
    ids[::4] = -1
    ids[1::4] = 17
    grad, _ = _matrix(rng, n, dim, torch.float32)
    groups = embedding.group_tokens(torch.from_numpy(ids).cuda(), rows, drop_id=17)
    clean = grad.clone()
    clean[(torch.from_numpy((ids < 0) | (ids == 17))).cuda()] = 0
    dirty = grad.clone()
    dirty[(torch.from_numpy((ids < 0) | (ids == 17))).cuda()] = float("nan")
    assert torch.equal(embedding.gradient(groups, dirty), embedding.gradient(groups, clean))
    assert (embedding.gradient(groups, dirty)[17] == 0).all()
