"""Layer norm, embedding, gate and 8-bit product (csrc/layer_norm.hip, embedding.hip, row_sort.hip, gate.hip, int8_product.hip) against
plain formulas in 64 bits on the CPU.

Tolerances count roundings.  U = 2^-24 is half a step of fp32; HALF[type] half a step of the output's type, relative to the value.  A sum of
terms t_i along a chain of at most d additions is off by at most d U sum |t_i|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}       # half a step of the smallest numbers
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def within(got, ref, tol, half_of=None):
    """|got - ref| <= tol (+ the rounding to ``half_of``) everywhere; NaNs and infinities in the same places."""
    got, ref = got.detach().cpu().double(), ref.double()
    assert got.shape == ref.shape, (got.shape, ref.shape)
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    assert torch.equal(got[~fine & ~torch.isnan(ref)], ref[~fine & ~torch.isnan(ref)])
    if half_of is not None:
        tol = tol + (ref.abs() + tol) * HALF[half_of] + TINY[half_of]
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(ref)
    over = (got - ref).abs() - tol
    over[~fine] = -1
    assert not over.numel() or float(over.max()) <= 0, (float(over.max()), int(over.argmax()), float((got - ref).abs()[fine].max()))


# ---- layer norm ------------------------------------------------------------------------------------------------------------------

def norm_oracle(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    h = (x - mean) * rstd
    y = h
    if w is not None:
        y = y * w.double()
    if b is not None:
        y = y + b.double()
    return y, mean, rstd, h


def norm_chain(C):
    """Additions in a row's sum: up to 32 in a lane (wide rows: C / 256), 6 across lanes, 4 across waves."""
    return 48 + C // 256


def check_norm(x, w, b, dy, eps=1e-5):
    from mega_nerf.layer_norm import layer_norm_backward, layer_norm_forward
    dev = lambda t: None if t is None else t.to(DEV)      # noqa: E731
    C = x.shape[-1]
    d = norm_chain(C)
    y64, mean, rstd, h = norm_oracle(x, w, b, eps)
    y, m, r = layer_norm_forward(dev(x), dev(w), dev(b), eps)
    wa = torch.ones(C, dtype=torch.float64) if w is None else w.double().abs()
    ba = torch.zeros(C, dtype=torch.float64) if b is None else b.double().abs()
    # h: the difference to the corrected mean is off by 3 U |h| + d U mean|h| (mean|h| <= 1), rstd by (d + 6) U of itself
    tol_h = U * ((d + 9) * h.abs() + d)
    within(y, y64, wa * tol_h + 3 * U * (wa * h.abs() + ba), x.dtype)
    assert y.dtype == x.dtype and y.shape == x.shape
    dx, dw, db = layer_norm_backward(dev(dy), dev(x), dev(w), m, r)
    g = dy.double() * (1 if w is None else w.double())
    s1, s2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx64 = rstd * (g - s1 - h * s2)
    # the kept mean is rounded: h moves by a = 2 U |mean| rstd besides its own roundings
    a = 2 * U * mean.abs() * rstd + U * d
    tol_h = a + U * (d + 9) * h.abs()
    mg, mgh = g.abs().mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
    tol_s2 = (g.abs() * tol_h).mean(-1, keepdim=True) + U * (d + 4) * mgh
    tol = rstd * (U * 4 * g.abs() + U * (d + 4) * mg + h.abs() * tol_s2 + tol_h * s2.abs() + 4 * U * (h * s2).abs() + 4 * U * s1.abs())
    tol = tol + U * (d + 8) * dx64.abs()
    within(dx, dx64, tol, x.dtype)
    rows = x.numel() // C
    if rows:
        D = 128 + rows // 1000                               # 8 rows or rows / 1024 a group, 32 groups, 1024 / 32 + 32 partial sums
        dyf, hf = dy.double().reshape(rows, C), h.reshape(rows, C)
        within(dw, (dyf * hf).sum(0), U * D * (dyf * hf).abs().sum(0) + (dyf.abs() * tol_h.reshape(rows, C)).sum(0), dw.dtype)
        within(db, dyf.sum(0), U * D * dyf.abs().sum(0), db.dtype)
    else:
        assert float(dw.abs().sum()) == 0 and float(db.abs().sum()) == 0
    return y, dx, dw, db


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,C', [(1, 1), (3, 2), (5, 31), (33, 48), (17, 63), (9, 64), (70, 65), (5, 127), (130, 256), (7, 319), (64, 512), (3, 513),
                                    (2, 1024), (9, 1025), (3, 2048), (4, 2049), (5, 4096), (3, 5001), (2, 8192), (2, 8193), (1, 20001), (0, 64),
                                    (4099, 75)])
def test_layer_norm_against_64_bits(rows, C, dtype):
    g = gen(rows * 7919 + C)
    x = (torch.randn(rows, C, generator=g) * 1.7 + 0.4).to(dtype)
    dy = torch.randn(rows, C, generator=g).to(dtype)
    check_norm(x, 1 + 0.2 * torch.randn(C, generator=g), 0.1 * torch.randn(C, generator=g), dy)


@pytest.mark.parametrize('rows,C,dtype', [(130, 4100, torch.float32), (4099, 4100, torch.float32), (2500, 8192, torch.float32), (2100, 8200, torch.bfloat16),
                                          (2500, 2052, torch.float32), (6000, 1100, torch.float32), (2100, 4100, torch.bfloat16), (4700, 2056, torch.float16)])
def test_layer_norm_many_wide_rows(rows, C, dtype):
    """Rows that a workgroup shares (1025 to 4096 columns of fp32, 2049 to 8192 of 16 bits) or reads over and over (wider ones), in more
    rows than workgroups: several turns of the row loops, several strips of rows whose column sums are joined, a ragged last strip."""
    g = gen(rows + C)
    x = (torch.randn(rows, C, generator=g) * 1.7 + 0.4).to(dtype)
    dy = torch.randn(rows, C, generator=g).to(dtype)
    check_norm(x, 1 + 0.2 * torch.randn(C, generator=g), 0.1 * torch.randn(C, generator=g), dy)


@pytest.mark.parametrize('wdtype', TYPES + [None])
def test_layer_norm_weight_types_and_none(wdtype):
    g = gen(5)
    x, dy = torch.randn(37, 203, generator=g).to(torch.bfloat16), torch.randn(37, 203, generator=g).to(torch.bfloat16)
    w = None if wdtype is None else (1 + 0.2 * torch.randn(203, generator=g)).to(wdtype)
    b = None if wdtype is None else (0.2 * torch.randn(203, generator=g)).to(wdtype)
    _, _, dw, db = check_norm(x, w, b, dy)
    assert dw.dtype == (wdtype or torch.float32) and db.dtype == dw.dtype


def test_layer_norm_far_from_zero_constant_rows_and_nan():
    from mega_nerf.layer_norm import layer_norm_forward
    g = gen(6)
    x = torch.randn(21, 300, generator=g) + 10000.0          # a spread of 1 on a mean of 10^4: the mean's rounding must not show in y
    check_norm(x, None, None, torch.randn(21, 300, generator=g))
    flat = torch.full((4, 100), 3.3)
    y, _, r = layer_norm_forward(flat.to(DEV), None, None, 1e-5)
    assert float(y.abs().max()) <= 1e-3 and abs(float(r[0]) - 1e-5 ** -0.5) < 1e-2
    x = torch.randn(5, 77, generator=g)
    x[1, 3], x[2, 76] = math.nan, math.inf
    y, _, _ = layer_norm_forward(x.to(DEV))
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 3, 4]]).all()


def test_wide_layer_norm_far_from_zero():
    """Rows wider than a workgroup's registers keep their precision on a mean of 10^4 as narrow ones do: with the corrected mean rounded
    to fp32 (half a step of 10^4 is 4.9e-4, in units of the spread of 1) y was off by 4e-4; the bound below is 4e-6 at h = 0."""
    for rows, C in ((21, 4100), (3, 20001)):
        g = gen(C)
        x = torch.randn(rows, C, generator=g) + 10000.0
        check_norm(x, None, None, torch.randn(rows, C, generator=g))


def test_layer_norm_strided_rows_and_offsets():
    from mega_nerf.layer_norm import layer_norm_backward, layer_norm_forward
    g = gen(7)
    big = torch.randn(40, 200, generator=g).to(DEV, torch.bfloat16)
    dyb = torch.randn(40, 333, generator=g).to(DEV, torch.bfloat16)
    w, b = torch.randn(101, generator=g).to(DEV), torch.randn(101, generator=g).to(DEV)
    x, dy = big[3:, 55:156], dyb[3:, 7:108]                                    # odd starts, pitches 200 and 333
    y, m, r = layer_norm_forward(x, w, b)
    y2, m2, r2 = layer_norm_forward(x.contiguous(), w, b)
    assert torch.equal(y, y2) and torch.equal(m, m2)
    for a, c in zip(layer_norm_backward(dy, x, w, m, r), layer_norm_backward(dy.contiguous(), x.contiguous(), w, m2, r2)):
        assert torch.equal(a, c)
    xt = torch.randn(64, 40, generator=g).to(DEV).t()                          # not a row pitch: copied
    assert torch.equal(layer_norm_forward(xt)[0], layer_norm_forward(xt.contiguous())[0])
    x3 = torch.randn(2, 3, 64, generator=g).to(DEV)
    assert torch.equal(layer_norm_forward(x3)[0].view(6, 64), layer_norm_forward(x3.view(6, 64))[0])
    spread = torch.randn(64, 2, generator=g).to(DEV)[:, 0]
    assert torch.equal(layer_norm_forward(x3, spread)[0], layer_norm_forward(x3, spread.contiguous())[0])


def test_layer_norm_gradient_against_differences_and_autograd():
    from mega_nerf.layer_norm import layer_norm
    g = gen(8)
    x, w, b = torch.randn(4, 23, generator=g), 1 + 0.3 * torch.randn(23, generator=g), torch.randn(23, generator=g)
    c = torch.randn(4, 23, generator=g)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    (layer_norm(*leaves) * c.to(DEV)).sum().backward()
    f = lambda x, w, b: float((norm_oracle(x, w, b, 1e-5)[0] * c.double()).sum())          # noqa: E731
    for which, leaf in enumerate(leaves):
        args = [t.double() for t in (x, w, b)]
        flat = args[which].reshape(-1)
        for i in range(0, flat.numel(), 5):
            at, step = float(flat[i]), 1e-5
            flat[i] = at + step
            hi = f(*args)
            flat[i] = at - step
            lo = f(*args)
            flat[i] = at
            want = (hi - lo) / (2 * step)                    # differences: step^2 f''' / 6 and 2^-52 f / step, under 1e-8 here
            assert abs(float(leaf.grad.view(-1)[i]) - want) <= 2e-5 * max(1.0, abs(want))
    # only some gradients wanted; weight and bias absent
    xs = x.to(DEV).requires_grad_()
    layer_norm(xs).sum().backward()
    assert xs.grad is not None
    ws = w.to(DEV).requires_grad_()
    layer_norm(x.to(DEV), ws, b.to(DEV)).sum().backward()
    assert ws.grad is not None


def test_layer_norm_many_rows_same_bits_twice():
    from mega_nerf.layer_norm import layer_norm_backward, layer_norm_forward
    x = torch.randn(50000, 200, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    dy = torch.randn(50000, 200, device=DEV, generator=torch.Generator(DEV).manual_seed(2))
    w = torch.ones(200, device=DEV)
    y, m, r = layer_norm_forward(x, w)
    one = layer_norm_backward(dy, x, w, m, r)
    two = layer_norm_backward(dy, x, w, m, r)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    check_norm(x[:30000].cpu(), None, None, dy[:30000].cpu())


# ---- embedding -------------------------------------------------------------------------------------------------------------------

def check_embedding(idx, table, dy, scale, pad=None, dtype=None):
    from mega_nerf.embedding import embedding_backward, embedding_forward
    count, width = table.shape
    k = idx.long().clamp(0, count - 1)
    out = embedding_forward(idx.to(DEV), table.to(DEV), scale)
    assert torch.equal(out.cpu(), (table[k].float() * torch.tensor(scale, dtype=torch.float32)).to(table.dtype))
    grad = embedding_backward(dy.to(DEV), idx.to(DEV), count, scale, pad, dtype)
    flat, rows = k.reshape(-1), dy.reshape(-1, width).double()
    s = torch.zeros(count, width, dtype=torch.float64).index_add_(0, flat, rows)
    sa = torch.zeros(count, width, dtype=torch.float64).index_add_(0, flat, rows.abs())
    n = torch.zeros(count, dtype=torch.float64).index_add_(0, flat, torch.ones(flat.numel(), dtype=torch.float64))
    if pad is not None:
        s[pad], sa[pad] = 0, 0
    f = torch.tensor(scale, dtype=torch.float32).double()
    within(grad, s * f, (n[:, None].clamp(max=200) + 2) * U * sa * f.abs(), grad.dtype)        # 32 in a tile, tiles / 4 or / 32 and 32 to join
    assert float(grad.cpu().double()[n == 0].abs().sum()) == 0
    assert torch.equal(grad, embedding_backward(dy.to(DEV), idx.to(DEV), count, scale, pad, dtype))
    return grad


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('n,count,width', [(1, 1, 1), (1, 10, 48), (7, 3, 5), (64, 2, 48), (333, 40, 63), (1000, 1, 75), (4096, 300, 17), (4097, 300, 17),
                                           (5000, 70001, 33), (9000, 1920, 48), (700, 19, 1030), (2049, 257, 129)])
def test_embedding_against_64_bits(n, count, width, dtype):
    g = gen(n + count + width)
    idx = torch.randint(count, (n,), generator=g)
    check_embedding(idx, torch.randn(count, width, generator=g).to(dtype), torch.randn(n, width, generator=g).to(dtype), 1.0)


@pytest.mark.parametrize('order', ['one', 'runs', 'sorted', 'skewed'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_embedding_long_runs(order, dtype):
    g = gen(11)
    n, count, width = 20011, 50, 40
    idx = {'one': torch.full((n,), 7), 'runs': torch.randint(count, (n // 192 + 1,), generator=g).repeat_interleave(192)[:n],
           'sorted': torch.randint(count, (n,), generator=g).sort().values, 'skewed': (count * torch.rand(n, generator=g) ** 6).long()}[order]
    check_embedding(idx, torch.randn(count, width, generator=g).to(dtype), torch.randn(n, width, generator=g).to(dtype), 4.5)


def test_embedding_runs_over_many_tiles():
    """Runs of thousands of tiles (their ends are searched for), beside short ones, in narrow and wide tables."""
    g = gen(13)
    for n, width, share in ((200003, 5, 0.9), (70001, 140, 0.5), (30000, 600, 0.7)):
        idx = torch.where(torch.rand(n, generator=g) < share, torch.randint(1, 4, (n,), generator=g) * 7, torch.randint(300, (n,), generator=g))
        check_long(idx, torch.randn(n, width, generator=g), 300)


def check_long(idx, dy, count):
    """Sums of up to 10^5 rows: 16 in a tile, then tiles / 32 in a phase, 32 phases."""
    from mega_nerf.embedding import embedding_backward
    grad = embedding_backward(dy.to(DEV), idx.to(DEV), count)
    s = torch.zeros(count, dy.shape[1], dtype=torch.float64).index_add_(0, idx, dy.double())
    sa = torch.zeros(count, dy.shape[1], dtype=torch.float64).index_add_(0, idx, dy.double().abs())
    within(grad, s, (16 + len(idx) / 512 + 40) * U * sa)


def test_embedding_index_types_padding_and_clamping():
    from mega_nerf.embedding import embedding, embedding_backward, embedding_forward
    g = gen(12)
    table, dy = torch.randn(9, 20, generator=g), torch.randn(6, 4, 20, generator=g)
    idx = torch.randint(9, (6, 4), generator=g)
    for t in (torch.int32, torch.int64, torch.float32):
        check_embedding(idx.to(t), table, dy, 0.5, pad=3)
    check_embedding(idx, table.to(torch.bfloat16), dy.to(torch.bfloat16), 1.0, dtype=torch.float32)
    wild = torch.tensor([-5, 0, 8, 9, 100, 2 ** 40, -2 ** 40])
    check_embedding(wild, table, torch.randn(7, 20, generator=g), 1.0)
    f = torch.tensor([math.nan, -0.5, 3.9, 1e30, -math.inf])
    assert torch.equal(embedding_forward(f.to(DEV), table.to(DEV)).cpu(), table[[0, 0, 3, 8, 0]])
    empty = torch.empty(0, dtype=torch.int64, device=DEV)
    assert embedding_forward(empty, table.to(DEV)).shape == (0, 20)
    assert float(embedding_backward(torch.empty(0, 20, device=DEV), empty, 9).abs().sum()) == 0
    # strided table, gradient rows and indices
    big, dyb = torch.randn(9, 50, generator=g).to(DEV), torch.randn(30, 33, generator=g).to(DEV)
    rays = torch.randint(9, (30, 2), generator=g).to(DEV)
    assert torch.equal(embedding_forward(rays[:, 1], big[:, 3:24]), big[:, 3:24][rays[:, 1]])
    assert torch.equal(embedding_backward(dyb[:, 5:26], rays[:, 1], 9), embedding_backward(dyb[:, 5:26].contiguous(), rays[:, 1].contiguous(), 9))
    # autograd
    leaf = table.to(DEV).requires_grad_()
    (embedding(idx.to(DEV), leaf, 2.0, padding_idx=0) * dy.to(DEV)).sum().backward()
    assert torch.equal(leaf.grad, embedding_backward(dy.to(DEV), idx.to(DEV), 9, 2.0, 0))
    # differences: linear in the table, so one unit step is exact up to roundings
    unit = torch.zeros_like(table)
    unit[int(idx[0, 0]), 4] = 1
    want = float((table * 0 + unit)[idx].double().mul(dy.double()).sum()) * 2
    if int(idx[0, 0]) != 0:
        assert abs(float(leaf.grad[int(idx[0, 0]), 4]) - want) < 1e-5


# ---- gate ------------------------------------------------------------------------------------------------------------------------

def gate_oracle(x, k, score, bias=None, mask=None, n_groups=1, k_groups=1, group_top=1, renormalise=True, scale=1.0):
    """(weights, cells, scores) by sorting Python lists of float64 values."""
    x = x.double()
    rows, n = x.shape
    open_ = (x > -math.inf) | torch.isnan(x)
    if mask is not None:
        open_ = open_ & mask
    x = torch.where(open_, x, torch.full_like(x, -math.inf))
    if score == 'softmax':
        high = x.max(1, keepdim=True).values
        e = torch.exp(x - torch.where(high > -math.inf, high, torch.zeros_like(high)))
        s = e / e.sum(1, keepdim=True)
        s[~open_] = 0
    else:
        s = torch.sigmoid(x)
    by = s if bias is None else s + bias.double()
    value = x if bias is None else by
    weights, cells = torch.zeros(rows, k, dtype=torch.float64), torch.full((rows, k), -1, dtype=torch.int64)
    m = n // n_groups
    for r in range(rows):
        ok = [bool(o) for o in open_[r]]
        bad = any(ok[e] and (math.isnan(float(x[r, e])) or (score == 'softmax' and float(x[r, e]) == math.inf)) for e in range(n))
        if bad:
            weights[r] = math.nan
            continue
        if n_groups > 1:
            totals = []
            for q in range(n_groups):
                got = sorted((float((by if group_top > 1 else value)[r, e]) for e in range(q * m, q * m + m) if ok[e]), reverse=True)[:group_top]
                if got:
                    totals.append((-sum(got), q))
            keep = {q for _, q in sorted(totals)[:k_groups]}
            ok = [ok[e] and e // m in keep for e in range(n)]
        best = sorted((-float(value[r, e]), e) for e in range(n) if ok[e])[:k]
        for j, (_, e) in enumerate(best):
            cells[r, j], weights[r, j] = e, s[r, e]
    if renormalise:
        lw = torch.where(cells >= 0, (x if score == 'softmax' else torch.nn.functional.logsigmoid(x)).gather(1, cells.clamp(min=0)), torch.tensor(-math.inf).double())
        lw = torch.softmax(lw, 1)                            # of the chosen alone: the same quotients without underflow
        weights = torch.where(torch.isnan(weights), weights, torch.where(cells >= 0, lw, torch.zeros_like(lw)))
    return weights * scale, cells, s


def check_gate(x, k, dw=None, **how):
    from mega_nerf.gating import route_topk_backward, route_topk_forward
    dev = lambda t: t.to(DEV) if isinstance(t, torch.Tensor) else t      # noqa: E731
    w64, cells64, s = gate_oracle(x, k, **how)
    w, cells = route_topk_forward(dev(x), k, **{a: dev(b) for a, b in how.items()})
    assert torch.equal(cells.cpu().long(), cells64)
    # exp(x - base): the difference rounds by U |x - base|, expf and the sums by less than 64 U
    spread = 64 + 2 * x.double()[torch.isfinite(x)].abs().max().item() if torch.isfinite(x).any() else 64
    scale = how.get('scale', 1.0)
    within(w, w64, U * spread * w64.abs().nan_to_num() + 1e-37)
    if dw is None:
        return w, cells
    back = {a: dev(how[a]) for a in ('score', 'mask', 'renormalise', 'scale') if a in how}
    dx = route_topk_backward(dev(dw), dev(x), cells, **back)
    g = torch.where(cells64 >= 0, dw.double(), torch.zeros((), dtype=torch.float64)) * scale
    at, has = cells64.clamp(min=0), (cells64 >= 0).any(1, keepdim=True)
    p = torch.where(cells64 >= 0, w64 / scale, torch.zeros((), dtype=torch.float64))
    ref = torch.zeros(x.shape, dtype=torch.float64)
    size = torch.zeros(x.shape, dtype=torch.float64)          # what the roundings are relative to
    total = (p * g).sum(1, keepdim=True)
    if how['score'] == 'softmax' and not how.get('renormalise', True):
        ref.scatter_add_(1, at, p * g)
        ref -= s * total
        size.scatter_add_(1, at, (p * g).abs())
        size += s * (p * g).abs().sum(1, keepdim=True)
    else:
        renorm = how.get('renormalise', True)
        off = 1.0
        if how['score'] == 'sigmoid':
            off = torch.sigmoid(-x.double()).gather(1, at).masked_fill(cells64 < 0, 0)
        ref.scatter_add_(1, at, p * off * (g - total if renorm else g))
        size.scatter_add_(1, at, p * (g.abs() + ((p * g).abs().sum(1, keepdim=True) if renorm else 0)))
    ref, size = ref.masked_fill(~has, 0), size.masked_fill(~has, 0)
    within(dx, ref, U * 4 * spread * size + 1e-37, x.dtype)
    return w, cells


def gate_inputs(rows, n, k, dtype, seed):
    g = gen(seed)
    return (1.5 * torch.randn(rows, n, generator=g)).to(dtype), 0.2 * torch.randn(n, generator=g), torch.randn(rows, k, generator=g), \
        torch.rand(rows, n, generator=g) < 0.5


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('renormalise', [True, False])
@pytest.mark.parametrize('rows,n,k', [(1, 1, 1), (1, 8, 2), (5, 2, 2), (33, 7, 3), (70, 16, 4), (41, 25, 2), (9, 25, 25), (37, 33, 5), (20, 64, 8), (11, 100, 7),
                                      (6, 129, 32), (10, 256, 8), (5, 300, 9), (3, 513, 32), (2, 1024, 32)])
def test_gate_against_64_bits(rows, n, k, score, renormalise):
    for dtype in TYPES:
        x, bias, dw, mask = gate_inputs(rows, n, k, dtype, rows + n + k)
        check_gate(x, k, dw, score=score, renormalise=renormalise, scale=2.5)
        check_gate(x, k, dw, score=score, renormalise=renormalise, bias=bias, mask=mask)


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('n,groups,k_groups,k', [(8, 4, 1, 2), (25, 5, 2, 3), (94, 2, 1, 4), (64, 8, 4, 6), (256, 8, 4, 8), (256, 128, 7, 8), (60, 60, 9, 8), (1024, 8, 3, 32)])
def test_gate_groups(n, groups, k_groups, k, score):
    for top in (1, 2):
        x, bias, dw, mask = gate_inputs(13, n, k, torch.float32, n + top)
        for how in (dict(), dict(bias=bias), dict(bias=bias, mask=mask), dict(mask=mask)):
            check_gate(x, k, dw, score=score, n_groups=groups, k_groups=k_groups, group_top=top, scale=1.5, **how)


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('n,groups,k_groups,k', [(1024, 2, 1, 8), (512, 2, 1, 8), (512, 4, 3, 8), (32, 2, 1, 3)])
def test_gate_groups_of_many_lanes(n, groups, k_groups, k, score):
    """Groups of 1, 8, 16 and 32 whole lanes."""
    for top in (1, 2):
        x, bias, dw, mask = gate_inputs(13, n, k, torch.float32, n + top)
        for how in (dict(), dict(bias=bias), dict(bias=bias, mask=mask), dict(mask=mask)):
            check_gate(x, k, dw, score=score, n_groups=groups, k_groups=k_groups, group_top=top, scale=1.5, **how)


@pytest.mark.parametrize('score', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('n,groups,k_groups,k', [(256, 8, 4, 8), (256, 1, 1, 8), (8, 1, 1, 2), (25, 5, 2, 3)])
def test_gate_with_a_bias_of_zeros(n, groups, k_groups, k, score):
    """A balance bias as training starts with it: scores tie wherever 16-bit logits do, in every row where all logits are alike."""
    g = gen(n + groups)
    fine = (1.5 * torch.randn(150, n, generator=g)).to(torch.bfloat16)
    coarse = torch.randn(150, n, generator=g).mul(4).round().div(4)
    for x in (fine, coarse.to(torch.bfloat16), coarse.to(torch.float16), torch.zeros(70, n), torch.full((70, n), -2.5).to(torch.bfloat16)):
        for top in (1, 2):
            for bias in (torch.zeros(n), torch.full((n,), 0.25)):
                check_gate(x, k, torch.randn(len(x), k, generator=g), score=score, bias=bias, n_groups=groups, k_groups=k_groups, group_top=top)


@pytest.mark.parametrize('n,groups', [(256, 8), (300, 1), (25, 1)])
def test_gate_more_rows_than_workgroups(n, groups):
    from mega_nerf.gating import route_topk_backward, route_topk_forward
    g = torch.Generator(DEV).manual_seed(n)
    rows = 140000 if n > 32 else 2200000
    x, bias = torch.randn(rows, n, device=DEV, generator=g).to(torch.bfloat16), 0.2 * torch.randn(n, device=DEV, generator=g)
    how = dict(score='sigmoid', bias=bias, n_groups=groups, k_groups=max(1, groups // 2), group_top=2)
    w, c = route_topk_forward(x, 3, **how)
    dw = torch.randn(rows, 3, device=DEV, generator=g)
    dx = route_topk_backward(dw, x, c, score='sigmoid')
    for part in (slice(0, 50), slice(rows // 2, rows // 2 + 50), slice(rows - 37, rows)):
        w2, c2 = route_topk_forward(x[part].clone(), 3, **how)
        assert torch.equal(w[part], w2) and torch.equal(c[part], c2)
        assert torch.equal(dx[part], route_topk_backward(dw[part].clone(), x[part].clone(), c2, score='sigmoid'))


def test_gate_ties_go_to_the_lowest_cell():
    x = torch.tensor([[1.0, 2.0, 2.0, 2.0, 0.0], [0.0, -0.0, 0.0, -0.0, 0.0], [50.0, 60.0, 70.0, 60.0, 80.0]])
    for how in (dict(), dict(bias=torch.zeros(5)), dict(bias=torch.full((5,), 0.25))):
        for dtype in TYPES:
            check_gate(x.to(dtype), 3, torch.ones(3, 3), score='softmax', **how)
            check_gate(x[:2].to(dtype), 3, torch.ones(2, 3), score='sigmoid', **how)
    from mega_nerf.gating import route_topk_forward
    _, cells = route_topk_forward(x.to(DEV), 3, score='sigmoid')             # scores of 1.0 all, but the logits differ
    assert cells[2].tolist() == [4, 2, 1]
    coarse = torch.randn(200, 40, generator=gen(3)).to(torch.bfloat16).mul(4).round().div(4)
    check_gate(coarse, 8, score='softmax')
    check_gate(coarse, 8, score='sigmoid', bias=torch.randint(3, (40,), generator=gen(4)) / 4)


def test_gate_near_ties_are_decided_in_64_bits():
    # scores whose order fp32 cannot see: logits one fp32 step apart where the sigmoid is flat
    base = torch.full((64, 12), 9.0)
    step = torch.randperm(12, generator=gen(5)).float()
    x = base + step * 2.0 ** -20
    check_gate(x, 5, score='sigmoid', bias=torch.zeros(12))
    check_gate(x, 5, score='softmax', bias=torch.zeros(12))
    check_gate(x, 5, score='sigmoid', bias=torch.full((12,), 1000.0))


def test_gate_empty_rows_infinities_and_nan():
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf] * 4, [1.0, -inf, -inf, -inf], [nan, 1.0, 2.0, 3.0], [inf, 1.0, 2.0, 3.0], [nan, inf, 0.5, 0.25], [-3e38, -3.4e38, 3.4e38, 0.0]])
    mask = torch.ones(6, 4, dtype=torch.bool)
    mask[4, :2] = False                                      # what the mask hides may hold anything
    dw = torch.ones(6, 3)
    for score in ('softmax', 'sigmoid'):
        for renormalise in (True, False):
            w, cells = check_gate(x, 3, dw, score=score, renormalise=renormalise, mask=mask)
            assert cells[0].tolist() == [-1, -1, -1] and w[0].tolist() == [0, 0, 0]
            assert cells[1].tolist() == [0, -1, -1] and cells[4].tolist() == [2, 3, -1] and cells[2].tolist() == [-1, -1, -1]
    low = torch.full((3, 9), torch.finfo(torch.float32).min)
    check_gate(low, 2, torch.ones(3, 2), score='softmax')
    check_gate(low, 2, torch.ones(3, 2), score='sigmoid')
    deep = torch.tensor([[-200.0, -201.0, 5.0]])             # renormalised over scores that underflow
    check_gate(deep, 2, torch.ones(1, 2), score='softmax', bias=torch.tensor([1.0, 1.0, -9.0]))
    check_gate(deep, 2, torch.ones(1, 2), score='sigmoid', bias=torch.tensor([1.0, 1.0, -9.0]))
    one = torch.zeros(5, 6, dtype=torch.bool)
    one[:, 2] = True
    check_gate(torch.randn(5, 6, generator=gen(1)), 2, torch.ones(5, 2), score='softmax', mask=one[0])
    check_gate(torch.randn(5, 6, generator=gen(1)), 2, torch.ones(5, 2), score='softmax', mask=torch.zeros(6, dtype=torch.bool))


def test_gate_gradient_against_differences():
    from mega_nerf.gating import route_topk
    x, bias, dw, _ = gate_inputs(3, 11, 4, torch.float32, 77)
    for score in ('softmax', 'sigmoid'):
        for renormalise in (True, False):
            leaf = x.to(DEV).requires_grad_()
            w, cells = route_topk(leaf, 4, score=score, bias=bias.to(DEV), renormalise=renormalise, scale=1.5)
            (w * dw.to(DEV)).sum().backward()
            for r in range(3):
                for e in range(11):
                    vals = []
                    for sign in (1, -1):
                        y = x.double().clone()
                        y[r, e] += sign * 1e-6
                        y = torch.softmax(y, 1) if score == 'softmax' else torch.sigmoid(y)
                        p = y.gather(1, cells.cpu().long())
                        vals.append(float((dw.double() * 1.5 * (p / p.sum(1, keepdim=True) if renormalise else p)).sum()))
                    want = (vals[0] - vals[1]) / 2e-6
                    assert abs(float(leaf.grad[r, e]) - want) <= 1e-5 * max(1.0, abs(want))


def test_gate_strides_and_shapes():
    from mega_nerf.gating import route_topk_backward, route_topk_forward
    g = gen(9)
    big, mb = torch.randn(40, 50, generator=g).to(DEV), (torch.rand(40, 77, generator=g) < 0.6).to(DEV)
    x, m = big[1:, 3:24], mb[1:, 9:30]
    a = route_topk_forward(x, 3, mask=m)
    b = route_topk_forward(x.contiguous(), 3, mask=m.contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    dwb = torch.randn(39, 7, generator=g).to(DEV)
    kw = dict(mask=m, renormalise=False)
    assert torch.equal(route_topk_backward(dwb[:, 2:5], x, a[1], **kw), route_topk_backward(dwb[:, 2:5].contiguous(), x.contiguous(), a[1], **kw))
    w, c = route_topk_forward(torch.randn(4, 5, 12, generator=g).to(DEV), 2)
    assert w.shape == (4, 5, 2) and c.shape == (4, 5, 2)
    w, c = route_topk_forward(torch.empty(0, 12, device=DEV), 2)
    assert w.shape == (0, 2) and c.shape == (0, 2)
    assert route_topk_backward(w, torch.empty(0, 12, device=DEV), c).shape == (0, 12)


@pytest.mark.parametrize('n_cells', [1, 2, 25, 255, 256, 257, 70000])
@pytest.mark.parametrize('slots', [0, 1, 63, 64, 65, 511, 4095, 4096, 4097, 12289, 300001])
def test_dispatch_is_the_stable_order(slots, n_cells):
    from mega_nerf.gating import dispatch
    g = gen(slots + n_cells)
    cells = torch.randint(-1, n_cells, (slots,), generator=g, dtype=torch.int32)
    cells[torch.rand(slots, generator=g) < 0.01] = n_cells + 5                  # outside: as -1
    order, offsets = dispatch(cells.to(DEV), n_cells)
    key = torch.where((cells < 0) | (cells >= n_cells), n_cells, cells.long())
    assert torch.equal(order.cpu().long(), torch.sort(key, stable=True).indices)
    assert torch.equal(offsets.cpu().long(), torch.searchsorted(key.sort().values, torch.arange(n_cells + 1)))


@pytest.mark.parametrize('slots', [1100003, 2100001])
def test_orders_of_more_rows_than_two_to_the_20(slots):
    """2048 and 4096 rows a workgroup of the sort, in one pass and in two, under the dispatch and under the table's gradient."""
    from mega_nerf.embedding import embedding_backward
    from mega_nerf.gating import dispatch
    g = gen(slots)
    for n_cells in (25, 70000):
        cells = torch.randint(-1, n_cells, (slots,), generator=g, dtype=torch.int32)
        order, offsets = dispatch(cells.to(DEV), n_cells)
        key = torch.where(cells < 0, n_cells, cells.long())
        ordered, want = torch.sort(key, stable=True)
        assert torch.equal(order.cpu().long(), want)
        assert torch.equal(offsets.cpu().long(), torch.searchsorted(ordered, torch.arange(n_cells + 1)))
        idx, dy = torch.randint(n_cells, (slots,), generator=g), torch.randn(slots, 3, generator=g)
        grad = embedding_backward(dy.to(DEV), idx.to(DEV), n_cells)
        sums = torch.zeros(n_cells, 3, dtype=torch.float64).index_add_(0, idx, dy.double())
        sizes = torch.zeros(n_cells, 3, dtype=torch.float64).index_add_(0, idx, dy.double().abs())
        run = torch.bincount(idx, minlength=n_cells).double()[:, None]
        # 15 additions in a tile of 16 rows, its tiles in 32 phases, the phases: 2100001 rows over 25 cells are runs of 84000, 164 a phase
        within(grad, sums, (16 + run / 512 + 34) * U * sizes)


def test_dispatch_one_cell_and_none():
    from mega_nerf.gating import dispatch
    for fill in (-1, 0, 3, 6):
        order, offsets = dispatch(torch.full((5000, 2), fill, dtype=torch.int32, device=DEV), 7)
        assert torch.equal(order.cpu(), torch.arange(10000, dtype=torch.int32))
        assert offsets.tolist() == [0 if fill < 0 or c <= fill else 10000 for c in range(8)]


# ---- 8-bit product ---------------------------------------------------------------------------------------------------------------

def quantize_oracle(x):
    x = x.double()
    high = x.abs().amax(1)
    q = torch.round(x * 127 / torch.where(high > 0, high, torch.ones_like(high))[:, None])
    return q, high / 127


def check_quantize(x):
    from mega_nerf.quantized import quantize_rows
    q = quantize_rows(x.to(DEV))
    v, s = quantize_oracle(x)
    assert torch.equal(q.values.cpu().double(), v)
    within(q.scale, s, s * U + 2.0 ** -149)
    pitch = q.values.stride(0) if q.values.shape[0] > 1 else q.values.shape[1]
    assert pitch % 16 == 0 or q.values.shape[0] <= 1
    return q


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,cols', [(1, 1), (3, 15), (5, 16), (7, 63), (65, 64), (9, 319), (33, 512), (3, 1000), (2, 1024), (5, 2048), (3, 4100), (2, 9001)])
def test_quantize_rows(rows, cols, dtype):
    check_quantize(torch.randn(rows, cols, generator=gen(rows + cols)).to(dtype))


def test_quantize_rows_halves_zeros_and_infinities():
    from mega_nerf.quantized import quantize_rows
    x = torch.zeros(6, 300)
    x[0, :255] = (torch.arange(255) - 127) / 2 + 0.0         # multiples of a half up to 63.5 with the maximum at 127: ties
    x[0, 255] = 127.0
    x[1, :3] = torch.tensor([1.0, 0.5, -0.5])                # 63.5 -> 64, by the even rule
    x[3] = torch.randn(300, generator=gen(1)) * 1e-38
    x[4] = torch.randn(300, generator=gen(2)) * 1e37
    x[5] = 2.0 ** -149
    check_quantize(x)
    big = torch.randn(4000, 200, generator=gen(3))           # values within fp32's doubt of a half
    big[:, 0] = 10
    big[:, 1:] = (torch.randint(-127, 127, (4000, 199), generator=gen(4)) + 0.5) * (10 / 127)
    check_quantize(big)
    x = torch.randn(3, 40, generator=gen(5))
    x[0, 3], x[1, 39] = math.nan, -math.inf
    q = quantize_rows(x.to(DEV))
    assert torch.isnan(q.scale[:2]).all() and torch.isfinite(q.scale[2]) and float(q.values[:2].abs().sum()) == 0
    assert quantize_rows(torch.empty(0, 20, device=DEV)).values.shape == (0, 20)
    wide = torch.randn(20, 90, generator=gen(6)).to(DEV)[:, 3:70]
    assert torch.equal(quantize_rows(wide).values, quantize_rows(wide.contiguous()).values)


def check_product(m, n, k, dtype, bias, relu, seed, a=None, b=None):
    from mega_nerf.quantized import QuantizedRows, int8_product
    g = gen(seed)
    a = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8) if a is None else a
    b = torch.randint(-128, 128, (n, k), generator=g, dtype=torch.int8) if b is None else b
    sa, sb = torch.rand(m, generator=g) * 0.01, torch.rand(n, generator=g) * 0.01
    bv = torch.randn(n, generator=g) if bias else None
    y = int8_product(QuantizedRows(a.to(DEV), sa.to(DEV)), QuantizedRows(b.to(DEV), sb.to(DEV)), None if bv is None else bv.to(DEV), relu, dtype)
    p = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()
    ref = p + (0 if bv is None else bv.double())
    tol = U * (3 * p.abs() + ref.abs())                       # int to float, two scales, the bias
    if relu:
        ref = ref.clamp(min=0)
    assert y.dtype == dtype
    within(y, ref, tol, dtype)


@pytest.mark.parametrize('m,n,k', [(1, 1, 1), (1, 2048, 2048), (1, 17, 100), (2, 300, 320), (3, 5, 7), (16, 256, 319), (17, 129, 64), (33, 64, 2000), (63, 70, 75),
                                   (64, 64, 64), (65, 257, 130), (100, 128, 1040), (129, 127, 65), (200, 300, 16), (256, 256, 256), (257, 511, 513),
                                   (515, 260, 640), (1000, 256, 319), (700, 1025, 1)])
def test_product_against_64_bits(m, n, k):
    for i, dtype in enumerate(TYPES):
        check_product(m, n, k, dtype, bias=i != 1, relu=i == 2, seed=m + n + k)


@pytest.mark.parametrize('m,n,k', [(12289, 1100, 200), (12300, 1030, 64), (49200, 250, 33), (2000, 1000, 333), (1500, 1100, 1), (3000, 800, 512)])
def test_product_many_tiles(m, n, k):
    """Enough tiles for the 256 x 256 and the 128 x 128 kernels, whole and ragged, from one step of K to an odd number of them."""
    for i, dtype in enumerate(TYPES):
        check_product(m, n, k, dtype, bias=i != 1, relu=i == 2, seed=m + n + k)


@pytest.mark.parametrize('m,n,k', [(4352, 4096, 64), (4400, 4300, 100), (4352, 4097, 1), (8300, 4700, 333),
                                   (38400, 250, 333), (24000, 500, 64), (38000, 256, 1)])
def test_product_more_tiles_than_workgroups(m, n, k):
    """Workgroups that take a second and a third tile: 272, 306, 289 and 627 tiles of 256 x 256 on 256 workgroups, 600, 752 and 594 tiles
    of 128 x 128 on 512, whole and ragged, K of one step, with a tail and of an uneven number of steps."""
    for i, dtype in enumerate(TYPES):
        check_product(m, n, k, dtype, bias=i != 1, relu=i == 2, seed=m + n + k)


def test_product_extremes_and_long_sums():
    full = lambda r, c, v: torch.full((r, c), v, dtype=torch.int8)      # noqa: E731
    check_product(3, 70, 131071, torch.float32, False, False, 1, full(3, 131071, -128), full(70, 131071, -128))     # 2^31 - 2^14: the largest sum
    check_product(130, 70, 131071, torch.float32, False, False, 1, full(130, 131071, -128), full(70, 131071, 127))
    check_product(20, 40, 40000, torch.float32, True, True, 2)


def test_product_layouts():
    """Operands as a user may hold them: odd pitches and starts, a tail of rubbish, transposed storage."""
    from mega_nerf.quantized import QuantizedRows, int8_product
    g = gen(3)
    for k in (64, 100, 319):
        m, n = 70, 150
        a, b = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8), torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
        sa, sb = torch.rand(m, generator=g).to(DEV), torch.rand(n, generator=g).to(DEV)
        want = (a.double() @ b.double().t()) * sa.cpu().double()[:, None] * sb.cpu().double()

        def held(t, pitch, start):
            big = torch.randint(-127, 128, (t.shape[0] * pitch + start + 64,), generator=g, dtype=torch.int8).to(DEV)
            v = big[start:start + t.shape[0] * pitch].view(t.shape[0], pitch)
            v[:, :t.shape[1]] = t.to(DEV)
            return v[:, :t.shape[1]]

        for pitch, start in ((k, 0), (k + 1, 0), (512, 0), (512, 16), (512, 5), (336 if k < 337 else 512, 48)):
            y = int8_product(QuantizedRows(held(a, pitch, start), sa), QuantizedRows(held(b, pitch, start), sb))
            within(y, want, U * 4 * want.abs())
        y = int8_product(QuantizedRows(a.t().contiguous().t().to(DEV), sa), QuantizedRows(b.to(DEV).t().contiguous().t(), sb))
        within(y, want, U * 4 * want.abs())


def test_int8_linear_of_a_layer():
    from mega_nerf.quantized import int8_linear, quantize_rows
    g = gen(4)
    for dtype in TYPES:
        x, w, b = torch.randn(3, 50, 319, generator=g).to(dtype), torch.randn(256, 319, generator=g) / 18, torch.randn(256, generator=g)
        wq = quantize_rows(w.to(DEV))
        y = int8_linear(x.to(DEV), wq, b.to(DEV), relu=True)
        assert y.shape == (3, 50, 256) and y.dtype == dtype
        q, s = quantize_oracle(x.reshape(150, 319))
        qw, sw = quantize_oracle(w)
        p = (q @ qw.t()) * s[:, None] * sw
        ref = p + b.double()
        within(y.view(150, 256), ref.clamp(min=0), U * (6 * p.abs() + ref.abs()), dtype)
        # and near the layer it stands for: half a step of 1 / 127 on each side of 319 products
        full = torch.relu(x.reshape(150, 319).double() @ w.double().t() + b.double())
        assert float((y.view(150, 256).cpu().double() - full).abs().max()) < 0.2
    assert int8_linear(torch.empty(0, 319, device=DEV), wq).shape == (0, 256)
    assert int8_linear(torch.zeros(2, 319, device=DEV), wq).abs().sum() == 0
    assert int8_linear(torch.ones(2, 319, device=DEV), wq, out_dtype=torch.float16).dtype == torch.float16


# ---- the four together, streams, graphs ------------------------------------------------------------------------------------------

def gate_network(idx, feats, table, w, b, wg, k, P):
    """Appearance vectors beside the features, a norm, a dense layer of scores and the gate over the cells."""
    x = torch.cat([feats, P['embedding'](idx, table, 2.0)], 1)
    h = P['norm'](x, w, b)
    return P['gate'](h @ wg, k)


def test_a_gate_trained_end_to_end():
    from mega_nerf.embedding import embedding
    from mega_nerf.gating import dispatch, route_topk
    from mega_nerf.layer_norm import layer_norm
    g = gen(20)
    rows, n = 700, 25
    idx, feats = torch.randint(40, (rows,), generator=g), torch.randn(rows, 63, generator=g)
    params = [torch.randn(40, 48, generator=g) * 0.1, 1 + 0.1 * torch.randn(111, generator=g), 0.1 * torch.randn(111, generator=g),
              torch.randn(111, n, generator=g) / 10]
    mine = [p.to(DEV).requires_grad_() for p in params]
    P = dict(embedding=embedding, norm=layer_norm, gate=route_topk)
    w, cells = gate_network(idx.to(DEV), feats.to(DEV), *mine[:3], mine[3], 2, P)
    target = torch.randn(rows, 2, generator=g)
    ((w * target.to(DEV)) ** 2).sum().backward()
    ref = [p.double().requires_grad_() for p in params]

    def gate64(x, k):
        p = torch.softmax(x, 1).gather(1, cells.cpu().long())
        return p / p.sum(1, keepdim=True)
    w64 = gate_network(idx, feats.double(), *ref[:3], ref[3], 2, dict(
        embedding=lambda i, t, s: t[i] * s, norm=lambda x, a, c: norm_oracle(x, None, None, 1e-5)[0] * a + c, gate=gate64))
    ((w64 * target.double()) ** 2).sum().backward()
    # the fp32 product of 111 terms rounds by 111 U of its terms' sizes (about 3 U 111): scores off by 4e-5 at most, so gradients by 1e-4
    within(w, w64.detach(), 1e-4)
    for a, r in zip(mine, ref):
        within(a.grad, r.grad, 1e-4 * float(r.grad.abs().max()))
    order, offsets = dispatch(cells, n)
    flat = cells.view(-1)[order.long()]
    assert torch.equal(flat, flat.sort().values) and int(offsets[-1]) == rows * 2


def test_the_gate_served_in_8_bits_and_the_cells_blended():
    """embedding -> norm -> 8-bit scores -> gate -> the rows of every cell -> blended outputs by mnr_route_accumulate."""
    from mega_nerf import _native as N
    from mega_nerf.embedding import embedding_forward
    from mega_nerf.gating import dispatch, route_topk_forward
    from mega_nerf.layer_norm import layer_norm_forward
    from mega_nerf.quantized import int8_linear, quantize_rows
    g = gen(21)
    for rows in (1, 333):
        n, k = 8, 2
        idx, table = torch.randint(30, (rows,), generator=g).to(DEV), torch.randn(30, 64, generator=g).to(DEV)
        wg = quantize_rows(torch.randn(n, 64, generator=g).to(DEV))
        h = layer_norm_forward(embedding_forward(idx, table))[0]
        weights, cells = route_topk_forward(int8_linear(h, wg), k)
        order, offsets = dispatch(cells, n)
        out = torch.zeros(rows, 4, device=DEV)
        want = torch.zeros(rows, 4, dtype=torch.float64)
        ends = offsets.tolist()
        for c in range(n):
            slots = order[ends[c]:ends[c + 1]]
            if not len(slots):
                continue
            rows_of = (slots // k).to(torch.int32).contiguous()
            sub = torch.randn(len(rows_of), 4, generator=g).to(DEV)
            per_row = torch.zeros(rows, device=DEV)
            per_row[rows_of.long()] = weights.view(-1)[slots.long()]
            count = torch.tensor([len(rows_of)], dtype=torch.int32, device=DEV)
            N.check(N.lib().mnr_route_accumulate(out.data_ptr(), 4, sub.data_ptr(), 4, 4, rows_of.data_ptr(), count.data_ptr(), rows, per_row.data_ptr(),
                                                 0, N.stream_ptr()))
            for i, r in enumerate(rows_of.tolist()):
                want[r] += sub[i].cpu().double() * float(per_row[r])
        within(out, want, 1e-6 * 8)
        assert abs(float(weights.sum()) - rows) < 1e-4 * rows


def passes():
    """(name, call) of every explicit pass on fixed inputs, for streams and graphs."""
    from mega_nerf.embedding import embedding_backward, embedding_forward
    from mega_nerf.gating import dispatch, route_topk_backward, route_topk_forward
    from mega_nerf.layer_norm import layer_norm_backward, layer_norm_forward
    from mega_nerf.quantized import int8_linear, quantize_rows
    g = gen(30)
    x, dy, w = (torch.randn(6000, 96, generator=g).to(DEV) for _ in range(3))
    w = w[0].contiguous()
    idx = torch.randint(50, (6000,), generator=g).to(DEV)
    table = torch.randn(50, 96, generator=g).to(DEV)
    dw = torch.randn(6000, 3, generator=g).to(DEV)
    wq = quantize_rows(torch.randn(200, 96, generator=g).to(DEV))
    _, m, r = layer_norm_forward(x, w)
    _, c = route_topk_forward(x, 3)
    torch.cuda.synchronize()
    return [('norm', lambda: layer_norm_forward(x, w)), ('norm backward', lambda: layer_norm_backward(dy, x, w, m, r)),
            ('embedding', lambda: (embedding_forward(idx, table),)), ('embedding backward', lambda: (embedding_backward(dy, idx, 50),)),
            ('gate', lambda: route_topk_forward(x, 3)), ('gate backward', lambda: (route_topk_backward(dw, x, c),)), ('dispatch', lambda: dispatch(c, 96)),
            ('product', lambda: (int8_linear(x, wq),)), ('product one row', lambda: (int8_linear(x[:1], wq),))]


def test_one_dimensional_inputs_and_expanded_gradients():
    """One row without a row dimension, and the gradient of a sum: one value for all elements, no pitch at all."""
    from mega_nerf.embedding import embedding, embedding_forward
    from mega_nerf.gating import dispatch, route_topk, route_topk_forward
    from mega_nerf.layer_norm import layer_norm, layer_norm_forward
    from mega_nerf.quantized import int8_linear, quantize_rows
    g = gen(40)
    x, table = torch.randn(5, 40, generator=g).to(DEV), torch.randn(9, 40, generator=g).to(DEV)
    wq = quantize_rows(torch.randn(24, 40, generator=g).to(DEV))
    col = x.t().contiguous().t()[2]                          # a row whose elements lie five apart
    for row in (x[2], col):
        assert torch.equal(layer_norm_forward(row)[0], layer_norm_forward(x)[0][2])
        w, c = route_topk_forward(row, 3)
        w2, c2 = route_topk_forward(x, 3)
        assert torch.equal(w, w2[2]) and torch.equal(c, c2[2])
        assert torch.equal(int8_linear(row, wq), int8_linear(x, wq)[2])
    assert torch.equal(dispatch(c, 40)[0].cpu().long(), torch.sort(c.cpu(), stable=True).indices)
    assert torch.equal(embedding_forward(torch.tensor(4, device=DEV), table, 2.0), table[4] * 2)
    for shape in ((5, 40), (40,), (2, 3, 40)):
        leaves = [torch.randn(shape, generator=gen(41)).to(DEV).requires_grad_() for _ in range(2)]
        for leaf, full in zip(leaves, (False, True)):
            y = torch.cat([layer_norm(leaf), route_topk(leaf, 32, renormalise=False)[0]], -1)
            if full:
                y.backward(torch.ones_like(y))
            else:
                y.sum().backward()
        assert torch.equal(leaves[0].grad, leaves[1].grad)
    t1, t2 = table.clone().requires_grad_(), table.clone().requires_grad_()
    idx = torch.randint(9, (4, 6), generator=g).to(DEV)
    embedding(idx, t1).sum().backward()
    y = embedding(idx, t2)
    y.backward(torch.ones_like(y))
    assert torch.equal(t1.grad, t2.grad) and float((t1.grad.sum(1).cpu() - 40 * torch.bincount(idx.cpu().view(-1), minlength=9)).abs().max()) == 0


class Guarded:
    """A buffer [rows, pitch] inside a larger one, filled with a byte pattern: what a call may write is ``cols`` of each row."""

    def __init__(self, rows, cols, pitch, dtype, lead=1):
        self.rows, self.cols, self.pitch = rows, cols, pitch
        self.raw = torch.full(((rows + 2) * pitch + lead,), 0, dtype=dtype, device=DEV)
        self.raw.view(torch.uint8).fill_(0xa5)
        self.body = self.raw[pitch + lead:pitch + lead + rows * pitch].view(rows, pitch)
        self.before = self.raw.clone()

    def ptr(self):
        return self.body.data_ptr()

    def result(self):
        """The rows, after a check that nothing else has changed."""
        out = self.body[:, :self.cols].clone()
        self.body[:, :self.cols] = self.before[:1]
        assert torch.equal(self.raw.view(torch.uint8), self.before.view(torch.uint8))
        self.body[:, :self.cols] = out
        return out


def same_bits(a, b):
    return a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize('dtype', TYPES)
def test_entries_write_their_rows_and_their_workspace_alone(dtype):
    """The C entries with pitches wider than their rows, rows that start at any element and workspaces of exactly the bytes they ask for:
    the results of the tight calls, and not a byte changed behind a row, before the first, behind the last or behind the workspace."""
    from mega_nerf import _native as N
    from mega_nerf import embedding as E, gating as G, layer_norm as L, quantized as Q
    lib, code, g = N.lib(), N.ELEMENT_TYPES[dtype], gen(50)

    def call(fn, *args):
        N.launch(torch.empty(0, device=DEV), fn, *args)

    def space(size):
        return Guarded(1, size, size + 256, torch.uint8, lead=(-(size + 256)) % 256)

    for rows, C in ((1, 7), (21, 63), (70, 64), (333, 129), (1000, 319), (5, 4100), (3, 8200)):
        x, dy = (torch.randn(rows, C, generator=g).to(DEV, dtype) for _ in range(2))
        w, b = torch.randn(C, generator=g).to(DEV), torch.randn(C, generator=g).to(DEV)
        y, m, r = L.layer_norm_forward(x, w, b)
        out = Guarded(rows, C, C + 5, dtype)
        call(lib.mnr_layer_norm_forward, out.ptr(), C + 5, None, None, x.data_ptr(), C, w.data_ptr(), b.data_ptr(), rows, C, 1e-5, code, 0)
        assert same_bits(out.result(), y)
        size = lib.mnr_layer_norm_backward_workspace_bytes(rows, C, code)
        dx, ws = Guarded(rows, C, C + 3, dtype), space(size)
        dw, db = Guarded(1, C, C, torch.float32), Guarded(1, C, C, torch.float32)
        call(lib.mnr_layer_norm_backward, dx.ptr(), C + 3, dw.ptr(), db.ptr(), dy.data_ptr(), C, x.data_ptr(), C, w.data_ptr(), m.data_ptr(), r.data_ptr(), rows, C,
             code, 0, ws.ptr(), size)
        ws.result()
        for a, c in zip((dx, dw, db), L.layer_norm_backward(dy, x, w, m, r)):
            assert same_bits(a.result().view(c.shape), c)
    for rows, count, width in ((1, 1, 1), (50, 7, 33), (4096, 90, 17), (5000, 3, 40), (9000, 5001, 20), (70000, 257, 5)):
        idx = torch.randint(count, (rows,), generator=g).to(DEV)
        table, dy = torch.randn(count, width, generator=g).to(DEV, dtype), torch.randn(rows, width, generator=g).to(DEV, dtype)
        out = Guarded(rows, width, width + 3, dtype)
        call(lib.mnr_embedding_forward, out.ptr(), width + 3, table.data_ptr(), width, count, width, idx.data_ptr(), 4, 2.0, rows, code)
        assert same_bits(out.result(), E.embedding_forward(idx, table, 2.0))
        size = lib.mnr_embedding_backward_workspace_bytes(rows, count, width)
        ws, grad = space(size), Guarded(1, count * width, count * width + (count * width) % 2, dtype, lead=0)
        call(lib.mnr_embedding_backward, grad.ptr(), code, dy.data_ptr(), width, idx.data_ptr(), 4, rows, count, width, -1, 2.0, code, ws.ptr(), size)
        ws.result()
        assert same_bits(grad.result().view(count, width), E.embedding_backward(dy, idx, count, 2.0))
    for rows, n, k in ((1, 8, 2), (70, 25, 3), (33, 100, 8), (9, 300, 5), (3, 1000, 32)):
        x, bias, dwt = torch.randn(rows, n, generator=g).to(DEV, dtype), torch.randn(n, generator=g).to(DEV), torch.randn(rows, k, generator=g).to(DEV)
        for b in (None, bias):
            wt, ce = Guarded(1, rows * k, rows * k, torch.float32), Guarded(1, rows * k, rows * k, torch.int32)
            call(lib.mnr_gate_forward, wt.ptr(), ce.ptr(), x.data_ptr(), n, N.ptr(b), None, 0, rows, n, k, 0, 1, 1, 1, 0, 1.5, code)
            w2, c2 = G.route_topk_forward(x, k, bias=b, renormalise=False, scale=1.5)
            assert same_bits(wt.result().view(rows, k), w2) and same_bits(ce.result().view(rows, k), c2)
        dx = Guarded(rows, n, n + 7, dtype)
        call(lib.mnr_gate_backward, dx.ptr(), n + 7, dwt.data_ptr(), k, x.data_ptr(), n, c2.data_ptr(), None, 0, rows, n, k, 0, 0, 1.5, code)
        assert same_bits(dx.result(), G.route_topk_backward(dwt, x, c2, renormalise=False, scale=1.5))
    for slots, n in ((1, 1), (4096, 300), (4097, 25), (70001, 5000)):
        cells = torch.randint(-1, n, (slots,), generator=g, dtype=torch.int32).to(DEV)
        size = lib.mnr_gate_dispatch_workspace_bytes(slots, n)
        ws, order, offsets = space(size), Guarded(1, slots, slots, torch.int32), Guarded(1, n + 1, n + 1, torch.int32)
        call(lib.mnr_gate_dispatch, order.ptr(), offsets.ptr(), cells.data_ptr(), slots, n, ws.ptr(), size)
        ws.result()
        for a, c in zip((order, offsets), G.dispatch(cells, n)):
            assert same_bits(a.result().view(-1), c)
    for m, n, k in ((1, 33, 100), (40, 70, 319), (300, 129, 64), (2000, 1001, 80), (4200, 3300, 48)):
        x, w = torch.randn(m, k, generator=g).to(DEV, dtype), Q.quantize_rows(torch.randn(n, k, generator=g).to(DEV))
        pitch = (k + 15) // 16 * 16
        values, scale = Guarded(m, pitch, pitch, torch.int8, lead=(-pitch) % 256), Guarded(1, m, m, torch.float32)
        call(lib.mnr_quantize_rows, values.ptr(), pitch, scale.ptr(), x.data_ptr(), k, m, k, code)
        q = Q.quantize_rows(x)
        held = values.result()
        assert same_bits(held[:, :k], q.values) and float(held[:, k:].abs().sum()) == 0 and same_bits(scale.result().view(-1), q.scale)
        size, ldb = lib.mnr_int8_linear_workspace_bytes(m, k), w.values.stride(0)
        y, ws = Guarded(m, n, n + 5, dtype), space(size)
        call(lib.mnr_int8_linear, y.ptr(), n + 5, x.data_ptr(), k, code, w.values.data_ptr(), ldb, w.scale.data_ptr(), None, m, n, k, 1, code, ws.ptr(), size)
        ws.result()
        want = Q.int8_linear(x, w, relu=True)
        assert same_bits(y.result(), want)
        y = Guarded(m, n, n + 2, dtype)
        call(lib.mnr_int8_product, y.ptr(), n + 2, held.data_ptr(), pitch, q.scale.data_ptr(), w.values.data_ptr(), ldb, w.scale.data_ptr(), None, m, n, k, 1, code)
        assert same_bits(y.result(), want)


def test_every_pass_in_a_graph_replayed():
    todo = passes()
    eager = [[t.clone() for t in f()] for _, f in todo]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _, f in todo:
            f()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [f() for _, f in todo]
    for again in range(4):
        for ts in out:
            for t in ts:
                t.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        for (name, f), got, want in zip(todo, out, eager):
            for a, b in zip(got, want):
                assert torch.equal(a, b), (name, again)
            for a, b in zip(f(), want):                       # the program's own work between the replays
                assert torch.equal(a, b), (name, again)


def test_a_graph_replayed_on_new_inputs():
    """One recording, other values in the same buffers for each replay: indices in short and in long runs, ties that send rows of the gate to
    64 bits, cells of which a row has none.  Nothing of the recording's values is kept."""
    from mega_nerf.embedding import embedding_backward, embedding_forward
    from mega_nerf.gating import dispatch, route_topk_backward, route_topk_forward
    from mega_nerf.layer_norm import layer_norm_backward, layer_norm_forward
    from mega_nerf.quantized import int8_linear, quantize_rows
    g = gen(60)
    rows, C, count = 6000, 64, 50
    x, dy = torch.randn(rows, C, generator=g).to(DEV), torch.randn(rows, C, generator=g).to(DEV)
    w, table, bias = torch.randn(C, generator=g).to(DEV), torch.randn(count, C, generator=g).to(DEV), torch.randn(C, generator=g).to(DEV)
    idx, mask = torch.zeros(rows, dtype=torch.int64, device=DEV), torch.ones(rows, C, dtype=torch.bool, device=DEV)
    wq = quantize_rows(torch.randn(130, C, generator=g).to(DEV))

    def step():
        e = embedding_forward(idx, table, 0.5)
        h, m, r = layer_norm_forward(x, w)
        weights, cells = route_topk_forward(h, 3, score='sigmoid', bias=bias, mask=mask, n_groups=4, k_groups=2, group_top=2)
        dh = route_topk_backward(weights, h, cells, score='sigmoid', mask=mask)
        return (e, h, weights, cells, dh) + tuple(layer_norm_backward(dh, x, w, m, r)) + tuple(dispatch(cells, C)) + (embedding_backward(dy, idx, count),
                                                                                                                  int8_linear(h, wq))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for again in range(6):
        x.copy_(torch.randn(rows, C, generator=g) * (0.0 if again == 2 else 1.0))
        if again == 3:
            x.copy_(x.mul(2).round().div(2))
        bias.copy_(torch.randn(C, generator=g) * (again % 2))
        dy.copy_(torch.randn(rows, C, generator=g))
        idx.copy_(torch.randint(count, (rows,), generator=g) if again < 2 else torch.full((rows,), 7) if again == 2 else
                  torch.randint(count, (rows // 500 + 1,), generator=g).repeat_interleave(500)[:rows])
        mask.copy_(torch.rand(rows, C, generator=g) < (0.02 if again == 4 else 0.7))
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(out, step())):
            assert same_bits(a, b), (again, i)


def test_two_streams_at_once_and_two_graphs():
    todo = passes()
    eager = [[t.clone() for t in f()] for _, f in todo]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = [f() for _, f in todo]
    torch.cuda.synchronize()
    for i in range(2):
        for (name, _), a, b in zip(todo, got[i], eager):
            assert all(torch.equal(p, q) for p, q in zip(a, b)), name
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([f() for _, f in todo])
        graphs.append(graph)
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            for (name, _), a, b in zip(todo, o, eager):
                assert all(torch.equal(p, q) for p, q in zip(a, b)), name


def test_captured_autograd_backward_is_refused():
    """... while an eager graph of the same leaf is alive; the explicit pass is captured instead."""
    from mega_nerf import _native as N
    from mega_nerf.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward
    leaf = torch.randn(64, 32, device=DEV, requires_grad=True)
    dy = torch.randn(64, 32, device=DEV)
    y = layer_norm(leaf)                                     # alive throughout
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(N.NativeError, match='layer_norm_backward'):
            torch.autograd.grad(layer_norm(leaf), leaf, dy)
        _, m, r = layer_norm_forward(leaf)
        dx, _, _ = layer_norm_backward(dy, leaf, None, m, r)
    graph.replay()
    torch.cuda.synchronize()
    y.backward(dy)
    assert torch.equal(leaf.grad, dx)


def test_large_offsets():
    """Element offsets past 2^31: rows at the far end of a buffer of more than 2^31 elements."""
    from mega_nerf.embedding import embedding_backward, embedding_forward
    from mega_nerf.layer_norm import layer_norm_forward
    from mega_nerf.quantized import quantize_rows
    big = torch.zeros(4_300_000, 512, dtype=torch.bfloat16, device=DEV)          # 2.2e9 elements, 4.4 GB
    big[-3:] = torch.randn(3, 512, device=DEV).to(torch.bfloat16)
    y, _, _ = layer_norm_forward(big)
    assert torch.equal(y[-3:], layer_norm_forward(big[-3:].clone())[0]) and float(y[:5].abs().sum()) == 0
    idx = torch.tensor([4_299_999, 0, 4_299_998, 4_299_999], device=DEV)
    assert torch.equal(embedding_forward(idx, big), big[idx])
    del y
    q = quantize_rows(big)
    assert torch.equal(q.values[-3:], quantize_rows(big[-3:].clone()).values)
    del q
    dy = torch.randn(4, 512, device=DEV).to(torch.bfloat16)
    grad = embedding_backward(dy, idx, 4_300_000)
    assert torch.equal(grad[-1], (dy[0].float() + dy[3].float()).to(torch.bfloat16)) and torch.equal(grad[-2], dy[2])
    assert int((grad != 0).any(1).sum()) == 3
