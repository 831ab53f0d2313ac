"""The minibatch operators on the GPU against their formulas in 64 bits.

Tolerances count roundings (half a step each: u = 2^-24 in fp32, h = eps / 2 of the output's type) and are worked out from
the formulas, element by element, from the absolute values that are summed."""
import math

import pytest
import torch

import recommender_amd as ra

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 1e-30
F32, BF16 = torch.float32, torch.bfloat16


def half(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def ids_of(g, n, rows, dtype=torch.int32):
    return torch.randint(0, max(rows, 1), (n,), device="cuda", generator=g).to(dtype)


def close(got, want, tol):
    got = got.double()
    assert got.shape == want.shape
    assert bool(torch.isfinite(got).all())
    over = ((got - want).abs() - tol).max().item() if got.numel() else -1.0
    assert over <= 0, f"off by {((got - want).abs() / (tol + TINY)).max().item():.3g} times the tolerance"


# ------------------------------------------------------------------ lookup
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, rows, d, pad", [(1, 1, 1, 0), (7, 5, 3, 0), (33, 100, 40, 24), (1000, 37, 100, 0), (257, 1000, 128, 0),
                                             (64, 20, 129, 1), (5000, 3000, 256, 0), (3, 10, 1000, 6),
                                             (500, 60, 4, 0), (500, 60, 5, 2), (500, 60, 7, 1), (501, 60, 8, 3), (501, 60, 9, 0),
                                             (333, 60, 127, 0), (333, 60, 130, 1), (12, 60, 1031, 0), (300000, 60, 131, 0)])
def test_embedding(dtype, n, rows, d, pad):
    g = gen(n + d)
    table = normal(g, rows, d + pad, dtype=dtype)[:, :d]
    ids = ids_of(g, n, rows)
    ids[n // 2] = -1
    if n > 4:
        ids[1], ids[2] = rows, 2 ** 31 - 1
    out = ra.embedding(table, ids, scale=1.7)
    inside = (ids >= 0) & (ids < rows)
    want = table.double()[ids.long().clamp(0, rows - 1)] * 1.7
    close(out[inside], want[inside], (half(dtype) + 2 * U) * want[inside].abs())      # 1.7 in fp32, the product, the store
    assert bool((out[ids < 0] == 0).all()) and bool(torch.isnan(out[ids >= rows].float()).all())


def test_embedding_shapes_and_alignment():
    g = gen(1)
    base = normal(g, 1 + 50 * 16, dtype=BF16)
    table = base[1:].view(50, 16)                     # rows that start 2 bytes behind a multiple of 16
    ids = ids_of(g, 24, 50).view(2, 3, 4)
    assert torch.equal(ra.embedding(table, ids), table[ids.long()])
    assert torch.equal(ra.embedding(table.t().contiguous().t(), ids), table[ids.long()])       # columns contiguous
    assert torch.equal(ra.embedding(table[:1].expand(9, 16), ids % 9), table[:1].expand(2, 3, 4, 16))
    assert ra.embedding(table, ids[:0]).shape == (0, 3, 4, 16)
    none = ra.embedding(table[:0], torch.tensor([-1, 0], dtype=torch.int32, device="cuda")).float()
    assert float(none[0].abs().sum()) == 0 and bool(torch.isnan(none[1]).all())
    assert torch.equal(ra.embedding(table, ids.transpose(0, 2)), table[ids.transpose(0, 2).long()])


def test_embedding_far_rows():
    """A table of more than 2^32 bytes and 2^31 elements: offsets in 64 bits."""
    rows, d = (1 << 23) + 5, 260
    table = torch.zeros(rows, d, dtype=BF16, device="cuda")
    ids = torch.tensor([0, 1 << 22, rows - 1, rows - 2], dtype=torch.int32, device="cuda")
    for k, i in enumerate(ids.tolist()):
        table[i] = k + 1.0
    assert torch.equal(ra.embedding(table, ids)[:, 259].float().cpu(), torch.arange(1.0, 5.0))
    grad = torch.ones(4, d, dtype=BF16, device="cuda")
    ra.embedding_grad(grad, ids, rows, out=table, accumulate=True)
    assert torch.equal(table[ids.long(), 259].float().cpu(), torch.arange(2.0, 6.0)) and float(table[5].abs().sum()) == 0


def test_embedding_many_rows():
    """More pieces than a dimension of a grid has threads: 2^34 elements come out, the same rows again and again."""
    d, period = 33, 1 << 10
    n = (1 << 34) // d + period
    table = normal(gen(3), 100, d, dtype=BF16)
    ids = ids_of(gen(4), period, 100).repeat(n // period + 1)[:n]
    out = ra.embedding(table, ids)
    whole = n // period * period
    assert torch.equal(out[:period], table[ids[:period].long()])
    for a in range(period, whole, 1 << 24):
        part = out[a:min(a + (1 << 24), whole)].view(-1, period, d)
        assert bool((part == out[:period]).all())
    assert torch.equal(out[whole:], out[:n - whole])


# ------------------------------------------------------------------ its gradient
def grad_want(grad, ids, rows, scale):
    inside = (ids >= 0) & (ids < rows)
    at = ids[inside].long()
    want = torch.zeros(rows, grad.shape[1], dtype=torch.float64, device="cuda")
    mass = want.clone()
    want.index_put_((at,), grad.double()[inside] * scale, accumulate=True)
    mass.index_put_((at,), grad.double()[inside].abs() * abs(scale), accumulate=True)
    count = torch.bincount(at, minlength=rows).double()[:, None]
    return want, mass, count


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, rows, d, kind", [
    (0, 5, 8, "even"), (1, 1, 1, "even"), (1, 7, 40, "even"), (63, 1000, 3, "even"), (64, 10, 100, "even"), (257, 1, 33, "even"),
    (300, 50, 128, "one"), (1000, 1682, 32, "popular"), (4095, 600, 129, "popular"), (4096, 1024, 64, "one"),
    (4097, 1023, 64, "popular"), (8192, 1024, 17, "one"), (20000, 17770, 128, "popular"), (30011, 59047, 200, "popular"),
    (50000, 3, 256, "even"), (5000, 2000003, 4, "even"), (6000, 100, 520, "popular"),
    # a row of many stretches: joined by one workgroup, then in two steps; rows that begin and end inside stretches
    (131072, 9, 520, "one"), (20001, 70, 700, "popular"), (131073, 9, 40, "one"), (140003, 50, 36, "popular"), (300001, 1000, 33, "popular"),
    (270000, 40000, 16, "popular"),
    # widths that no piece of 16 bytes divides; a row's last piece alone in its round
    (900, 300, 515, "popular"), (900, 300, 258, "popular"), (6000, 3, 515, "one"), (6000, 4, 259, "even"), (5000, 3, 9, "popular"),
    (3000, 700, 127, "popular"), (9000, 5, 5, "popular"), (700, 90, 7, "even")])
def test_embedding_grad(dtype, n, rows, d, kind):
    g = gen(n + rows + d)
    grad = normal(g, n, d, dtype=dtype)
    if kind == "one":
        ids = torch.full((n,), rows // 2, dtype=torch.int32, device="cuda")
    else:
        u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
        ids = ((u ** 4 if kind == "popular" else u) * rows).clamp(max=rows - 1).int()
    if n > 10:
        ids[3], ids[7], ids[9] = -1, rows, 2 ** 31 - 1
    want, mass, count = grad_want(grad, ids, rows, -0.75)
    out = ra.embedding_grad(grad, ids, rows, scale=-0.75)
    tol = (count + 1) * U * mass * 1.01 + half(dtype) * want.abs()
    close(out, want, tol)
    assert bool((out[(count == 0)[:, 0]] == 0).all())
    assert torch.equal(out, ra.embedding_grad(grad, ids, rows, scale=-0.75))          # the same bits
    # added to a padded table of its own
    base = normal(g, rows, d + 5, dtype=dtype)
    before = base.clone()
    got = ra.embedding_grad(grad, ids, rows, scale=-0.75, out=base[:, :d], accumulate=True)
    assert got.data_ptr() == base.data_ptr()
    full = want + before[:, :d].double()
    close(got, full, (count + 1) * U * 1.01 * mass + U * full.abs() + half(dtype) * full.abs() + TINY)
    assert torch.equal(base[:, d:], before[:, d:])                                    # what lies between the rows
    assert torch.equal(base[(count == 0)[:, 0]], before[(count == 0)[:, 0]])


@pytest.mark.parametrize("n, rows, d", [(900, 70, 8), (7000, 600, 33), (20000, 2000, 64)])
def test_embedding_grad_order_of_few_tokens(n, rows, d):
    """Rows of up to 16 tokens: the bits of the sum in the order of ids, whatever else is in the batch."""
    g = gen(n)
    ids = torch.arange(n, device="cuda", dtype=torch.int32) % rows
    ids = ids[torch.randperm(n, device="cuda", generator=g)]
    grad = normal(g, n, d)
    by_id, place = torch.sort(ids.long(), stable=True)
    first = torch.searchsorted(by_id, torch.arange(rows + 1, device="cuda"))
    count = first[1:] - first[:-1]
    assert int(count.max()) <= 16
    want = torch.zeros(rows, d, device="cuda")
    for k in range(16):                                           # every row's k-th token
        here = torch.nonzero(k < count)[:, 0]
        want[here] += grad[place[first[here] + k]]
    assert torch.equal(ra.embedding_grad(grad, ids, rows), want)
    more = torch.cat([ids, torch.full((100,), rows, dtype=torch.int32, device="cuda")])        # another row's tokens behind them
    assert torch.equal(ra.embedding_grad(torch.cat([grad, grad[:100]]), more, rows + 1)[:rows], want)


def test_embedding_grad_many_table_rows():
    """More lanes for the table's rows than a dimension of a grid has threads."""
    rows, d = (1 << 28) + 7, 33
    ids = torch.tensor([0, rows - 1, 1 << 27, rows - 1, -1, rows - 8], dtype=torch.int32, device="cuda")
    grad = torch.arange(1.0, 7.0, device="cuda")[:, None].expand(6, d).to(BF16).contiguous()
    out = ra.embedding_grad(grad, ids, rows)
    assert out[[0, rows - 1, 1 << 27, rows - 8], d - 1].tolist() == [1.0, 6.0, 3.0, 6.0]
    assert sum(int((out[a:a + (1 << 24)] != 0).sum()) for a in range(0, rows, 1 << 24)) == 4 * d


def test_embedding_grad_is_the_lookups():
    """<dY, lookup(T + e D) - lookup(T - e D)> / 2e = <gradient, D>: the lookup is linear, so the difference has no remainder."""
    g = gen(3)
    table, way, grad = normal(g, 90, 24), normal(g, 90, 24), normal(g, 500, 24)
    ids = ids_of(g, 500, 90)
    ids[5] = -1
    up, down = ra.embedding(table + way, ids, 1.5), ra.embedding(table - way, ids, 1.5)
    left = (grad.double() * (up.double() - down.double())).sum() / 2
    right = (ra.embedding_grad(grad, ids, 90, 1.5).double() * way.double()).sum()
    size = (grad.double().abs() * (up.double().abs() + down.double().abs())).sum()
    assert abs(left - right) <= 40 * U * size


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("n, rows, d", [(40, 100, 8), (9000, 20000, 33)])
def test_embedding_scale_that_is_no_number(dtype, scale, n, rows, d):
    """Rows of no id and padding are zero whatever the scale is, and the others show it."""
    ids = ids_of(gen(n), n, rows)
    ids[3] = -1
    ones = torch.ones(n, d, dtype=dtype, device="cuda")
    named = torch.zeros(rows, dtype=torch.bool, device="cuda")
    named[ids[ids >= 0].long()] = True
    grad = ra.embedding_grad(ones, ids, rows, scale=scale)
    assert float(grad[~named].abs().sum()) == 0 and not bool(torch.isfinite(grad[named]).any())
    out = ra.embedding(torch.ones(rows, d, dtype=dtype, device="cuda"), ids, scale=scale)
    assert float(out[3].abs().sum()) == 0 and not bool(torch.isfinite(out[ids >= 0]).any())


# ------------------------------------------------------------------ loss
def loss_case(g, n, items, d, dtype, bias, spread=2.0):
    x = normal(g, n, d, dtype=dtype)
    w = normal(g, items, d, dtype=dtype, std=spread / math.sqrt(d))
    b = normal(g, items) if bias else None
    return x, w, ids_of(g, n, items), b


def loss_want(x, w, t, b, scale, weights=None):
    """(loss, lse, dx, dw, db) and the same of absolute values, in 64 bits; rows without a target have no part in it"""
    n, items = x.shape[0], w.shape[0]
    x, w = x.double(), w.double()
    live = (t >= 0) & (t < items)
    x = torch.where(live[:, None], x, torch.zeros_like(x))
    z = scale * x @ w.T
    size = scale * x.abs() @ w.abs().T
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    lse = torch.logsumexp(z, 1)
    at = t.long().clamp(0, items - 1)[:, None]
    hit = torch.zeros_like(z).scatter_(1, at, 1.0)
    p = torch.exp(z - lse[:, None])
    others = (p * (1 - hit)).sum(1, keepdim=True)
    share = (torch.ones(n, device="cuda", dtype=torch.float64) if weights is None else weights.double().expand(n)) * live
    gr = torch.where(hit > 0, -others, p) * share[:, None]
    out = [torch.where(live, lse - z.gather(1, at)[:, 0], 0.0), torch.where(live, lse, 0.0), scale * gr @ w, scale * gr.T @ x, gr.sum(0)]
    big = gr.abs()
    return out, [size.where(torch.isfinite(size), torch.zeros_like(size)).amax(1), scale * big @ w.abs(), scale * big.T @ x.abs(), big.sum(0)]


def loss_tolerances(out, mass, n, items, d, dtype):
    """A logit: d products and sums (three bf16 parts leave 3 u of a product) and the steps to and from log2 units, on values
    up to `size`; a lane's running sum of up to items / 32 terms of which each exponential is off by its argument's error."""
    size = mass[0]
    logit = (d + 16) * U * size
    lse = 2 * logit + (items / 32 + 64) * U + 4 * U * out[1].abs() + 2 * U
    rel = (2 * lse + logit).max()
    held = 2.0 ** -8 if dtype == BF16 else 4 * U                # the exponentials as operands of the second product
    grad = lambda k, terms: (rel + held + (terms + 64) * U) * mass[k - 1] + half(dtype) * out[k].abs() + TINY    # noqa: E731
    return [2 * lse, 2 * lse, grad(2, items), grad(3, n), (rel + (n + 64) * U) * mass[3] + TINY]


LOSS_CASES = [(1, 1, 1), (1, 5, 8), (3, 31, 40), (33, 64, 16), (40, 33, 32), (64, 1000, 64), (129, 257, 100), (200, 700, 128),
              (31, 2000, 129), (65, 300, 192), (130, 500, 193), (300, 129, 256), (1000, 40, 24),
              # more rows than convert the other side on the way: the planes' kernels, of every width
              (700, 900, 32), (600, 1100, 64), (513, 257, 65), (530, 2100, 128), (1025, 333, 192), (520, 1500, 256), (1999, 77, 250)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, items, d", LOSS_CASES)
def test_softmax_loss_and_gradients(dtype, n, items, d):
    g = gen(n * items + d)
    bias, scale = (n + d) % 2 == 0, 0.8
    x, w, t, b = loss_case(g, n, items, d, dtype, bias)
    if n > 3:
        t[1], t[n - 1] = -1, -100
    each = normal(g, n) if n % 2 else None                       # weights of either sign
    out, mass = loss_want(x, w, t, b, torch.tensor(scale, dtype=F32).double().item(), each)
    tol = loss_tolerances(out, mass, n, items, d, dtype)
    loss, lse = ra.softmax_loss(x, w, t, bias=b, scale=scale)
    close(loss, out[0], tol[0])
    close(lse, out[1], tol[1])
    got = ra.softmax_loss_grads(x, w, t, bias=b, scale=scale, weights=1.0 if each is None else each)
    for k in range(4 if b is None else 5):
        close(got[k], out[k], tol[k])
    assert (got[4] is None) == (b is None) and got[2].dtype == dtype and got[3].dtype == dtype
    again = ra.softmax_loss_grads(x, w, t, bias=b, scale=scale, weights=1.0 if each is None else each)
    assert all(a is None or torch.equal(a, c) for a, c in zip(got, again))           # the same bits
    if n > 3:
        assert float(loss[1]) == 0 and float(lse[1]) == 0 and float(got[2][1].abs().sum()) == 0


def test_softmax_loss_many_items_and_rows():
    """Several parts of either axis, joined."""
    for n, items, d, dtype in ((70, 60000, 64, BF16), (5000, 300, 128, BF16), (2, 100000, 128, F32), (4100, 4099, 40, F32)):
        x, w, t, b = loss_case(gen(items), n, items, d, dtype, True)
        out, mass = loss_want(x, w, t, b, 1.0, torch.tensor(1.0 / n, dtype=F32).cuda())
        tol = loss_tolerances(out, mass, n, items, d, dtype)
        got = ra.softmax_loss_grads(x, w, t, bias=b, weights=1.0 / n)
        for k in range(5):
            close(got[k], out[k], tol[k])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, d", [(70, 48), (620, 128), (600, 250)])
def test_softmax_loss_masks(dtype, n, d):
    g = gen(8)
    items = 300
    x, w, t, b = loss_case(g, n, items, d, dtype, True)
    out_of = torch.rand(items, device="cuda", generator=g) < 0.4
    out_of[64:128] = True                                         # a whole tile
    b[out_of] = -math.inf
    out_of[7], b[7] = True, torch.finfo(F32).min                  # the type's lowest value
    w[20], w[64:128] = math.nan, math.inf                          # whatever the rows of items that are out hold
    b[20], out_of[20] = -math.inf, True
    kept = torch.nonzero(~out_of)[:, 0]
    t = kept[t.long() % len(kept)].int()
    t[5] = -1
    x[5] = math.nan                                               # padding is not looked at
    want_b = torch.where(out_of, torch.full_like(b, -math.inf), b)
    clean = torch.where(out_of[:, None], torch.zeros_like(w), w)
    out, mass = loss_want(x, clean, t, want_b, 1.0)
    tol = loss_tolerances(out, mass, n, items, d, dtype)
    got = ra.softmax_loss_grads(x, w, t, bias=b)
    for k in range(5):
        close(got[k], out[k], tol[k])
    assert float(got[3][out_of].abs().sum()) == 0 and float(got[4][out_of].abs().sum()) == 0
    assert torch.equal(ra.softmax_loss(x, w, t, bias=b)[0], got[0])
    # a target that is out of the catalogue, one behind the table
    t2 = t.clone()
    t2[0], t2[1] = 20, items
    loss, lse, dx, dw, db = ra.softmax_loss_grads(x, w, t2, bias=b)
    assert math.isinf(float(loss[0])) and float(loss[0]) > 0 and math.isfinite(float(lse[0]))
    assert math.isnan(float(loss[1])) and float(dx[:2].abs().sum()) == 0
    assert bool(torch.isfinite(dx).all()) and bool(torch.isfinite(dw).all()) and bool(torch.isfinite(db).all())
    assert float(db[20]) == 0
    # nothing in the catalogue
    loss, lse, dx, dw, db = ra.softmax_loss_grads(x, w, t, bias=torch.full_like(b, -math.inf))
    live = t >= 0
    assert bool((loss[live] == math.inf).all()) and bool((lse[live] == -math.inf).all())
    assert float(dx.abs().sum()) == 0 and float(dw.abs().sum()) == 0 and float(db.abs().sum()) == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [40, 700])
@pytest.mark.parametrize("weight", [math.inf, math.nan])
def test_softmax_loss_no_gradient_whatever_the_weight(dtype, n, weight):
    """Padding and a row whose target is out of the catalogue have no gradient, and their weights are not looked at."""
    g = gen(83)
    x, w, t, b = loss_case(g, n, 300, 64, dtype, True)
    b[20] = -math.inf
    t[t == 20] = 21
    t[0], t[1] = 20, -1
    each = torch.rand(n, device="cuda", generator=g)
    each[:2] = 0.0
    want = ra.softmax_loss_grads(x, w, t, bias=b, weights=each)
    each[:2] = weight
    got = ra.softmax_loss_grads(x, w, t, bias=b, weights=each)
    assert all(bool(torch.isfinite(v).all()) for v in got[2:]) and all(torch.equal(a, c) for a, c in zip(got, want))


def test_softmax_loss_first_items_masked():
    """No item of the catalogue among the first ones: the sums' reference is set late, and far from the masked zeros."""
    n, items, d = 40, 400, 32
    g = gen(81)
    for shift in (-300.0, 300.0):                                 # e^z is far outside fp32
        x, w, t, b = loss_case(g, n, items, d, F32, True)
        b += shift
        b[:200] = -math.inf
        t = 200 + t % 200
        out, mass = loss_want(x, w, t, b, 1.0)
        tol = loss_tolerances(out, mass, n, items, d, F32)
        got = ra.softmax_loss_grads(x, w, t, bias=b)
        for k in range(5):
            close(got[k], out[k], tol[k])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_softmax_loss_targets_keep_their_digits(dtype):
    """Weights that are no powers of two: the target's -g (1 - p) outweighs all else in an item's gradient.  In bf16 it enters in
    fp32, the other items' g p rounded to 8 bits, so a row of dW is off by its own rounding and by those of the others' only."""
    g = gen(82)
    for n, items, d in ((37, 500, 40), (600, 2000, 128)):
        x, w, t, b = loss_case(g, n, items, d, dtype, True)
        each = torch.rand(n, device="cuda", generator=g) + 0.1
        out, _ = loss_want(x, w, t, b, 1.0, each)
        z = torch.softmax(x.double() @ w.double().T + b.double(), 1)
        others = (z * (torch.arange(items, device="cuda")[None, :] != t[:, None].long()) * each.double()[:, None]).T @ x.double().abs()
        _, _, _, dw, _ = ra.softmax_loss_grads(x, w, t, bias=b, weights=each)
        held = 2.0 ** -8 if dtype == BF16 else 4 * U
        # the logits' errors move all of a row's terms: 30 is above every |z|, |x| |w| sum and term count in use here
        room = (d + items / 32 + n + 200) * U * 30 * (each.double()[None, :] @ x.double().abs())
        close(dw, out[3], half(dtype) * out[3].abs() + held * others + room + TINY)


def test_softmax_loss_many_wide_items():
    """A table of more than 2^32 bytes and 2^31 elements: every item but three is zero, so the sums are known."""
    items, d = (1 << 23) + 77, 256
    table = torch.zeros(items, d, dtype=BF16, device="cuda")
    for k, v in enumerate((5, items - 1, items - 70)):
        table[v, k] = 4.0
    x = torch.zeros(3, d, dtype=BF16, device="cuda")
    x[0, 0], x[1, 1], x[2, 2] = 1.0, 2.0, 4.0                     # logits 4, 8 and 16 on an item each
    t = torch.tensor([5, items - 1, 9], dtype=torch.int32, device="cuda")
    loss, lse, dx, dw, _ = ra.softmax_loss_grads(x, table, t)
    top = torch.tensor([4.0, 8.0, 16.0], dtype=torch.float64)
    want = torch.log(items - 1 + torch.exp(top))
    # a lane adds some 10^6 ones and half a chip's lanes join: 2^-24 of the sum a step, far from its own share of them
    assert (lse.double().cpu() - want).abs().max() < 1e-3
    assert (loss.double().cpu() - (want - torch.tensor([4.0, 8.0, 0.0], dtype=torch.float64))).abs().max() < 1e-3
    p = torch.exp(top - want)
    assert abs(float(dx[0, 0]) - 4 * (float(p[0]) - 1)) < 0.02 and abs(float(dx[2, 2]) - 4 * float(p[2])) < 0.02
    assert abs(float(dw[items - 1, 1]) - 2 * (float(p[1]) - 1)) < 0.02 and abs(float(dw[items - 70, 2]) - 4 * float(p[2])) < 0.02
    assert abs(float(dw[9, 2]) + 4) < 0.02 and float(dw[items - 2].abs().sum()) < 1e-4


def test_softmax_loss_many_rows():
    """More rows than a dimension of a grid has waves."""
    n = (1 << 26) + 300
    x, w, t, b = loss_case(gen(84), n, 3, 1, BF16, True)
    got = ra.softmax_loss(x, w, t, bias=b)
    for a, z in ((0, 1000), ((1 << 26) - 500, n)):
        out, mass = loss_want(x[a:z], w, t[a:z], b, 1.0)
        tol = loss_tolerances(out, mass, z - a, 3, 1, BF16)
        close(got[0][a:z], out[0], tol[0])
        close(got[1][a:z], out[1], tol[1])


def test_softmax_loss_not_a_number_shows():
    x, w, t, b = loss_case(gen(9), 40, 100, 32, F32, True)
    x[3, 4] = math.nan
    loss, lse = ra.softmax_loss(x, w, t, bias=b)
    assert bool(torch.isnan(loss[3])) and bool(torch.isnan(lse[3]))
    others = torch.arange(40, device="cuda") != 3
    assert bool(torch.isfinite(loss[others]).all())
    w[50, 2] = math.inf
    assert not bool(torch.isfinite(ra.softmax_loss(x, w, t, bias=b)[0]).any())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_softmax_loss_learnt_rows(dtype):
    """Targets that hold nearly the whole probability: loss and gradient keep their digits."""
    n, items, d = 64, 200, 64
    g = gen(10)
    t = ids_of(g, n, items)
    w = normal(g, items, d, dtype=dtype)
    x = (w[t.long()].float() * 0.35).to(dtype)                    # the target's logit lies about 0.35 d = 22 above the others
    out, mass = loss_want(x, w, t, None, 1.0)
    tol = loss_tolerances(out, mass, n, items, d, dtype)
    got = ra.softmax_loss_grads(x, w, t)
    # here the loss itself is small, and its error relative to it: the others' share times the error of their logits
    rel = 4 * (d + 16) * U * mass[0].max() + (items / 32 + 64) * U
    close(got[0], out[0], rel * out[0] + TINY)
    close(got[2], out[2], tol[2])
    close(got[3], out[3], tol[3])


def test_softmax_loss_large_logits():
    """Logits of some thousand, rising along the items: the running maximum moves all the time."""
    n, items, d = 33, 900, 32
    x = torch.ones(n, d, device="cuda")
    w = torch.arange(items, device="cuda", dtype=F32)[:, None].expand(items, d) / 8
    w = w.contiguous()
    t = torch.arange(n, device="cuda", dtype=torch.int32) * 27
    for way in (w, w.flip(0).contiguous()):
        out, mass = loss_want(x, way, t, None, 1.0)
        tol = loss_tolerances(out, mass, n, items, d, F32)
        got = ra.softmax_loss_grads(x, way, t)
        for k in range(4):
            close(got[k], out[k], tol[k])


def far_below_case(n, items, d, dtype, wide, high):
    """Logits of nearly nothing but the bias: 0, 40 on the items `high` (e^40 is below 2^58), -44 on the targets, last items."""
    g = gen(items + d)
    x, w = normal(g, n, d, dtype=dtype, std=1e-4), normal(g, items, d, dtype=dtype, std=wide)
    b = torch.zeros(items, device="cuda")
    b[high] = 40.0
    t = (items - 1 - torch.arange(n, device="cuda") % 3).int()
    b[items - 3:] = -44.0
    return x, w, t, b, torch.rand(n, device="cuda", generator=g) + 0.5


def far_below_holds(x, w, t, b, each, scale=1.0):
    n, (items, d) = x.shape[0], w.shape
    out, mass = loss_want(x, w, t, b, torch.tensor(scale, dtype=F32).double().item(), each)
    assert float(out[0].min()) > 80
    tol = loss_tolerances(out, mass, n, items, d, x.dtype)
    loss, lse = ra.softmax_loss(x, w, t, bias=b, scale=scale)
    close(loss, out[0], tol[0])
    close(lse, out[1], tol[1])
    got = ra.softmax_loss_grads(x, w, t, bias=b, scale=scale, weights=each)
    for k in range(5):
        close(got[k], out[k], tol[k])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, d, wide", [(5, 8, 400.0), (5, 8, 1.0), (3, 128, 30.0), (140, 40, 400.0)])
def test_softmax_loss_target_far_below(dtype, n, d, wide):
    """The first items set a low reference, the sum stands 2^58 above it and the target 2^63 below: fp32 has to hold what the
    join makes of them, times the items' elements."""
    far_below_holds(*far_below_case(n, 64, d, dtype, wide, [50]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, items, d", [(5, 64, 8), (140, 700, 40), (600, 300, 128)])
def test_softmax_loss_largest_elements(dtype, n, items, d):
    """Elements up to 1e20, the smallest scale, and sums 2^58 above their references: all within fp32."""
    x, w, t, b, each = far_below_case(n, items, d, dtype, 3e19, [50])
    x = normal(gen(d), n, d, dtype=dtype, std=1e-2)
    far_below_holds(x, w.clamp(-9.9e19, 9.9e19), t, b, each, scale=1e-20)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, items, d", [(1, 17770, 128), (40, 9000, 40), (700, 9000, 64)])
def test_softmax_loss_target_far_below_many_parts(dtype, n, items, d):
    """... and the sums of many parts of the items, of which each starts at a multiple of 32 or 64 items and is as far above its
    first ones: whatever the number of parts is, one of these inputs has the high items behind the start of all of them."""
    for tile in (32, 64):
        tiles = (items + tile - 1) // tile
        for parts in (8, 16, 24, 32, 48, 64, 96, 128, 192, 256):
            starts = {tiles * k // parts for k in range(parts)}
            high = [k * tile + tile // 2 + 3 if tile == 64 else (k + 1) * tile + 3 for k in starts]
            high = [i for i in high if i < items - 3 and (tile == 64 or i // tile not in starts)]
            far_below_holds(*far_below_case(n, items, d, dtype, 1.0, high))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, items, d", [(1, 3, 8), (40, 100, 32), (3, 5000, 128), (700, 300, 64)])
@pytest.mark.parametrize("how", ["row", "bias", "product"])
def test_softmax_loss_infinite_target_shows(dtype, n, items, d, how):
    """The target's logit is +inf: lse - z is not a number, and the row is not a perfectly learnt one."""
    for at in {2, min(items - 1, 50), items - 1}:
        x, w, t, b = loss_case(gen(at), n, items, d, dtype, True)
        t[:] = (at + 1) % items
        t[0], x[0, 2] = at, 1.5
        if how == "row":
            w[at, 2] = math.inf
        elif how == "bias":
            b[at] = math.inf
        else:
            x[0, 2], w[at, 2] = 1e30, 1e30
        loss, lse = ra.softmax_loss(x, w, t, bias=b)
        assert math.isnan(float(loss[0])) and not math.isfinite(float(lse[0])), at
        loss, lse, dx, _, _ = ra.softmax_loss_grads(x, w, t, bias=b)
        assert math.isnan(float(loss[0])) and not math.isfinite(float(lse[0])) and bool(torch.isnan(dx[0]).all()), at


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, items, d", [(1, 3, 8), (40, 100, 32), (3, 5000, 128), (700, 300, 64)])
def test_softmax_loss_target_without_probability(dtype, n, items, d):
    """A target of the catalogue whose logit is -inf: an infinite loss, and the gradient of probability 0, not none.  An fp32
    element is the sum of three bf16 ones, and -inf less its first part is not a number: there it may show as that instead."""
    for at in {2, min(items - 1, 50), items - 1}:
        x, w, t, b = loss_case(gen(at), n, items, d, dtype, True)
        t[:], x[:, 2], w[at, 2] = at, 1.5, -math.inf
        loss, lse = ra.softmax_loss(x, w, t, bias=b)
        got, _, dx, dw, db = ra.softmax_loss_grads(x, w, t, bias=b, weights=0.5)
        assert not bool(torch.isfinite(torch.cat([loss, got, dx[:, 2]])).any()), at
        if dtype == F32:
            assert not bool(torch.isfinite(dw[at]).any()) or float(dw[at].abs().sum()) > 0
            continue
        assert bool((loss == math.inf).all()) and bool((got == math.inf).all()) and bool(torch.isfinite(lse).all()), at
        want = -0.5 * x.double().sum(0)
        close(dw[at], want, half(dtype) * want.abs() + (n + 8) * U * 0.5 * x.double().abs().sum(0))
        assert abs(float(db[at]) + 0.5 * n) <= n * n * U


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n, items, d", [(1, 3, 8), (40, 100, 32), (3, 5000, 128), (700, 300, 64)])
def test_softmax_loss_infinite_item_shows(dtype, n, items, d):
    """An item's logit of +inf that is no row's target."""
    for at in {2, min(items - 1, 50), items - 1}:
        x, w, t, b = loss_case(gen(at), n, items, d, dtype, True)
        t[:], x[:, 2], w[at, 2] = (at + 1) % items, 1.5, math.inf
        for loss, lse, *_ in (ra.softmax_loss(x, w, t, bias=b), ra.softmax_loss_grads(x, w, t, bias=b)):
            assert bool(torch.isnan(loss).all()) and bool(torch.isnan(lse).all()), at


def test_softmax_loss_strides():
    g = gen(11)
    n, items, d = 37, 90, 64
    wide = normal(g, items, 96, dtype=BF16)
    xs = normal(g, n, 70, dtype=BF16)
    t = ids_of(g, n, items)
    want = ra.softmax_loss_grads(xs[:, :d].contiguous(), wide[:, :d].contiguous(), t)
    got = ra.softmax_loss_grads(xs[:, :d], wide[:, :d], t)
    assert all(torch.equal(a, b) for a, b in zip(got[:4], want[:4]))
    odd = normal(g, 1 + items * d, dtype=BF16)[1:].view(items, d).copy_(wide[:, :d])       # not at a multiple of 16 bytes
    got = ra.softmax_loss_grads(xs[:, :d].t().contiguous().t(), odd, t)
    assert all(torch.equal(a, b) for a, b in zip(got[:4], want[:4]))
    none = ra.softmax_loss_grads(xs[:0, :d], wide[:, :d], t[:0])
    assert none[0].shape == (0,) and none[2].shape == (0, d) and float(none[3].abs().sum()) == 0


def test_softmax_loss_workspace_holds_no_copy_of_the_table():
    """A bf16 table of the operand's width is read where it is; one of another address is copied; the results are the same."""
    n, items, d = 700, 40000, 128
    x, w, t, b = loss_case(gen(13), n, items, d, BF16, True)
    odd = torch.zeros(1 + items * d, dtype=BF16, device="cuda")[1:].view(items, d).copy_(w)

    def call(table):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        loss = ra.softmax_loss(x, table, t, bias=b)
        return loss, torch.cuda.max_memory_allocated() - before
    (one, small), (two, large) = call(w), call(odd)
    assert all(torch.equal(a, c) for a, c in zip(one, two))
    assert small < w.numel() < large                     # half the table's bytes: the parts' sums are far fewer
    got, want = ra.softmax_loss_grads(x, w, t, bias=b), ra.softmax_loss_grads(x, odd, t, bias=b)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_softmax_gradients_against_differences():
    """d/de of the 64-bit loss at x + e u, w + e v, b + e c, by central differences, is <dx, u> + <dw, v> + <db, c>."""
    g = gen(12)
    n, items, d = 50, 170, 40
    x, w, t, b = loss_case(g, n, items, d, F32, True, spread=1.0)
    t[4] = -1
    each = normal(g, n)
    _, _, dx, dw, db = ra.softmax_loss_grads(x, w, t, bias=b, weights=each)
    u, v, c = normal(g, n, d), normal(g, items, d), normal(g, items)

    def total(e):
        out, _ = loss_want(x.double() + e * u.double(), w.double() + e * v.double(), t, b.double() + e * c.double(), 1.0)
        return float((out[0] * each.double()).sum())
    e = 1e-4
    slope = (total(e) - total(-e)) / (2 * e)
    wider = (total(2 * e) - total(-2 * e)) / (4 * e)
    said = sum(float((a.double() * k.double()).sum()) for a, k in ((dx, u), (dw, v), (db, c)))
    out, mass = loss_want(x, w, t, b, 1.0, each)
    tol = loss_tolerances(out, mass, n, items, d, F32)
    room = sum(float((tol[k] * y.abs()).sum()) for k, y in ((2, u), (3, v), (4, c)))
    assert abs(said - slope) <= room + abs(wider - slope)         # the remainder is a third of what doubling e changes


# ------------------------------------------------------------------ norm and clipping
SETS = [[(1,)], [(5,), (0,), (3, 7)], [(4096,), (4097,), (12289,)], [(6040, 64), (3706, 64), (6040,), (3706,)],
        [(i % 7,) for i in range(300)], [(3000, 1000), (11,)]]


@pytest.mark.parametrize("shapes", SETS, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("kind", ["f32", "bf16", "mixed"])
def test_clip(shapes, kind):
    g = gen(len(shapes))
    types = {"f32": [F32], "bf16": [BF16], "mixed": [F32, BF16]}[kind]
    grads = [normal(g, *s, dtype=types[i % len(types)]) for i, s in enumerate(shapes)]
    norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in grads))
    assert abs(float(ra.grad_norm(grads)) - norm) <= 4 * U * norm               # float64 sums, rounded once
    for top in (0.25 * norm, 4 * norm):
        want = [t.double() * min(1.0, top / norm) for t in grads]
        out = [torch.full_like(t, math.nan) for t in grads]
        keep = [t.clone() for t in grads]
        assert abs(float(ra.clip_grads(grads, top, out=out)) - norm) <= 4 * U * norm
        for t, k, o, x in zip(grads, keep, out, want):
            assert torch.equal(t, k)
            if t.numel():
                close(o, x, (half(t.dtype) + 8 * U) * x.abs())
        place = [t.clone() for t in grads]
        ra.clip_grads(place, top)
        assert all(torch.equal(a, b) for a, b in zip(place, out))


def test_clip_views_and_odd_addresses():
    g = gen(20)
    base = normal(g, 40000)
    parts = [base[1:10001], base[10003:20000].view(13, 769), base[20001:20002], base[30000:39999:1].view(99, 101).t()]
    before = base.clone()
    norm = math.sqrt(sum(float((p.double() ** 2).sum()) for p in parts))
    ra.clip_grads(parts, norm / 2)
    moved = torch.zeros(40000, dtype=torch.bool, device="cuda")
    for a, z in ((1, 10001), (10003, 20000), (20001, 20002), (30000, 39999)):
        moved[a:z] = True
    assert torch.equal(base[~moved], before[~moved])
    close(base[moved], before[moved].double() / 2, 10 * U * before[moved].double().abs())


def test_clip_extremes():
    for value in (1e30, 1e-30):                                  # squares that fp32 cannot hold
        t = torch.full((1000,), value, device="cuda")
        norm = value * math.sqrt(1000)
        assert abs(float(ra.grad_norm([t])) / norm - 1) < 1e-5
        ra.clip_grads([t], norm / 10)
        assert abs(float(t[7]) / value * 10 - 1) < 1e-5
    t = torch.zeros(10, device="cuda")
    assert float(ra.clip_grads([t], 1.0)) == 0 and float(t.abs().sum()) == 0
    t = torch.ones(10, device="cuda")
    t[3] = math.inf
    assert math.isinf(float(ra.clip_grads([t], 1.0))) and float(t[0]) == 0 and math.isnan(float(t[3]))
    t = torch.ones(10, device="cuda")
    t[3] = math.nan
    assert math.isnan(float(ra.clip_grads([t], 1.0))) and bool(torch.isnan(t).all())
    assert float(ra.grad_norm([torch.empty(0, device="cuda")])) == 0
    t = torch.ones(8, device="cuda")
    with pytest.raises(Exception, match="shares memory"):
        ra.clip_grads([t, t[4:]], 1.0)


# ------------------------------------------------------------------ together
def step_want(users, items, P, Q, b, lr, top, scale):
    n = len(users)
    P, Q, b = P.double(), Q.double(), b.double()
    out, _ = loss_want(P[users.long()], Q, items, b, scale, torch.tensor(1.0 / n).cuda())
    dP = torch.zeros_like(P).index_add_(0, users.long(), out[2])
    norm = math.sqrt(sum(float((t ** 2).sum()) for t in (dP, out[3], out[4])))
    f = lr * min(1.0, top / norm)
    return out[0], norm, P - f * dP, Q - f * out[3], b - f * out[4]


def batch(seed, n=600, users=90, items=700, d=40):
    g = gen(seed)
    P, Q, b = normal(g, users, d), normal(g, items, d), normal(g, items)
    u, i = ids_of(g, n, users), ids_of(g, n, items)
    i[3] = -1
    return u, i, P, Q, b


def test_ranking_step():
    u, i, P, Q, b = batch(30)
    want = step_want(u, i, P, Q, b, 0.5, 0.05, 0.3)
    loss, norm = ra.ExplicitMF.ranking_step(u, i, P, Q, b, lr=0.5, max_norm=0.05, scale=0.3)
    # fp32 throughout: gradients to 1e-5 of the largest (some hundred roundings), the step is lr times them
    assert abs(float(norm) / want[1] - 1) < 1e-5
    close(loss, want[0], 1e-5 + torch.zeros_like(want[0]))
    for got, x in ((P, want[2]), (Q, want[3]), (b, want[4])):
        close(got, x, 2 * U * x.abs() + 0.5 * 0.05 * 1e-5)


def test_ranking_step_bf16_without_bias_or_clipping():
    g = gen(38)
    P, Q = normal(g, 50, 64, dtype=BF16), normal(g, 300, 64, dtype=BF16)
    u, i = ids_of(g, 200, 50), ids_of(g, 200, 300)
    u[7], i[7] = -1, -1                                           # a padding row
    before = [P.clone(), Q.clone()]
    x = ra.embedding(P, u)
    loss, _, dx, dq, _ = ra.softmax_loss_grads(x, Q, i, scale=0.2, weights=1.0 / 200)
    dp = ra.embedding_grad(dx, u, 50)
    got, norm = ra.ExplicitMF.ranking_step(u, i, P, Q, lr=3.0, scale=0.2)
    assert torch.equal(got, loss) and torch.equal(norm, ra.grad_norm([dp, dq]))
    for t, b, d in ((P, before[0], dp), (Q, before[1], dq)):
        assert torch.equal(t, b.sub(d, alpha=3.0))


def test_ranking_step_users_out_of_range():
    """A user that is no row of the table has no part in the step: padding, or a loss that is not a number."""
    u, i, P, Q, b = batch(31)
    far, away = u.clone(), i.clone()
    far[10], far[11], away[10], away[11] = -1, 90, -1, -1
    one, two = [t.clone() for t in (P, Q, b)], [P, Q, b]
    loss, norm = ra.ExplicitMF.ranking_step(far, i, *one, lr=0.5, max_norm=0.05, scale=0.3)
    want, length = ra.ExplicitMF.ranking_step(u, away, *two, lr=0.5, max_norm=0.05, scale=0.3)
    assert float(loss[10]) == 0 and math.isnan(float(loss[11])) and torch.equal(norm, length)
    loss[11] = 0
    assert torch.equal(loss, want) and all(torch.equal(x, y) for x, y in zip(one, two))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_ranking_step_one_table(dtype):
    """Users and items are rows of one table: one gradient, by which the step is clipped too."""
    g = gen(39)
    n, rows, d = 300, 400, 40
    T, b = normal(g, rows, d, dtype=dtype), normal(g, rows)
    u, i = ids_of(g, n, rows), ids_of(g, n, rows)
    out, _ = loss_want(T.double()[u.long()], T, i, b, 0.3, torch.tensor(1.0 / n).cuda())
    grad = out[3].index_add(0, u.long(), out[2])
    norm = math.sqrt(float((grad ** 2).sum() + (out[4] ** 2).sum()))
    want = T.double() - 0.5 * min(1.0, 0.02 / norm) * grad
    loss, length = ra.ExplicitMF.ranking_step(u, i, T, T, b, lr=0.5, max_norm=0.02, scale=0.3)
    # bf16: dx, dtable, their sum and the clipped gradient are rounded, half a step each of no more than the largest gradient row
    rough = 1e-5 if dtype == F32 else 4 * half(BF16)
    assert abs(float(length) / norm - 1) < rough
    close(T, want, half(dtype) * want.abs() + 2 * U * want.abs() + 0.5 * 0.02 * rough)
    close(loss, out[0], 1e-5 + torch.zeros_like(out[0]))


def test_ranking_step_columns_of_one_buffer():
    """Factors and biases as columns of one wider table: the same step as on tables of their own."""
    u, i, P, Q, b = batch(40, users=700)
    wide = torch.cat([P, Q, b[:, None]], 1)
    loss, norm = ra.ExplicitMF.ranking_step(u, i, wide[:, :40], wide[:, 40:80], wide[:, 80], max_norm=0.05)
    want, length = ra.ExplicitMF.ranking_step(u, i, P, Q, b, max_norm=0.05)
    assert torch.equal(loss, want) and torch.equal(norm, length) and torch.equal(wide, torch.cat([P, Q, b[:, None]], 1))


def test_ranking_step_tables_that_require_gradients():
    """All of them or one: the same step, and none of it recorded."""
    for which in ((0, 1, 2), (1,), (2,)):
        u, i, *tables = batch(37)
        plain = [t.clone() for t in tables]
        for k in which:
            tables[k].requires_grad_()
        loss, norm = ra.ExplicitMF.ranking_step(u, i, *tables, max_norm=0.05)
        want, length = ra.ExplicitMF.ranking_step(u, i, *plain, max_norm=0.05)
        assert torch.equal(loss, want) and torch.equal(norm, length) and not loss.requires_grad
        assert all(torch.equal(a, b) and a.grad_fn is None for a, b in zip(tables, plain))


def test_captured_step_replays():
    """The whole step in a graph, replayed on new inputs with eager work of the same kind in between."""
    u, i, P, Q, b = batch(31, n=5000)
    keep = [t.clone() for t in (P, Q, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ra.ExplicitMF.ranking_step(u, i, P, Q, b, max_norm=0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, norm = ra.ExplicitMF.ranking_step(u, i, P, Q, b, max_norm=0.1)
    for seed in (32, 33, 34, 35):
        u2, i2, *_ = batch(seed, n=5000)
        u.copy_(u2)
        i.copy_(i2)
        for t, k in zip((P, Q, b), keep):
            t.copy_(k)
        graph.replay()
        mine = [k.clone() for k in keep]
        loss2, norm2 = ra.ExplicitMF.ranking_step(u2, i2, *mine, max_norm=0.1)
        torch.cuda.synchronize()
        assert torch.equal(loss, loss2) and torch.equal(norm, norm2)
        assert all(torch.equal(a, c) for a, c in zip((P, Q, b), mine))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_wide_and_large_calls(dtype):
    """The widest rows (more than 64 KB of LDS a workgroup) and a batch whose popular rows are joined in two steps, in one graph,
    replayed with other inputs and eager calls in between."""
    def inputs(seed):
        g = gen(seed)
        x, w, t, b = loss_case(g, 600, 3000, 256, dtype, True)
        ids = torch.where(torch.rand(300000, device="cuda", generator=g) < 0.5, 7, ids_of(g, 300000, 3000)).int()
        return [x, w, t, b, normal(g, 300000, 40, dtype=dtype), ids]

    def step(x, w, t, b, grad, ids):
        loss, lse, dx, dw, db = ra.softmax_loss_grads(x, w, t, bias=b, weights=1.0 / 600)
        de = ra.embedding_grad(grad, ids, 3000)
        norm = ra.clip_grads([dx, dw, db, de], 0.5)
        return [loss, lse, dx, dw, db, de, norm, ra.embedding(de, ids), *ra.softmax_loss(x, w, t, bias=b)]
    held = inputs(50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*held)
    for seed in (51, 52, 53, 54):
        new = inputs(seed)
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        want = step(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once():
    """Calls on two streams have a workspace each."""
    g = gen(36)
    sets = [loss_case(g, 300, 5000, 64, BF16, True) for _ in range(2)]
    grads = [(normal(g, 20000, 32), ids_of(g, 20000, 500)) for _ in range(2)]
    want = [(ra.softmax_loss_grads(x, w, t, bias=b), ra.embedding_grad(*e, 500)) for (x, w, t, b), e in zip(sets, grads)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for s, (x, w, t, b), e in zip(streams, sets, grads):
            with torch.cuda.stream(s):
                got.append((ra.softmax_loss_grads(x, w, t, bias=b), ra.embedding_grad(*e, 500)))
        torch.cuda.synchronize()
        for (a, e), (c, f) in zip(got, want):
            assert all(torch.equal(y, z) for y, z in zip(a, c)) and torch.equal(e, f)


def test_one_device():
    with pytest.raises(ValueError, match="one ROCm device"):
        ra.embedding(torch.zeros(3, 4, device="cuda"), torch.zeros(2, dtype=torch.int32))
