"""The row operators (esgd.ops) on the GPU against their formulas in 64 bits.

Tolerances are bounds, derived here and not fitted.  With u = 2^-24 (fp32's half step) and h the
result type's half step (2^-24, bf16 2^-8, fp16 2^-11, with half its smallest subnormal below):
  * a product rounded once to fp32 and once to the result: (u + h) |x|, doubled for their product
  * a sum of m fp32 terms in any order: (m + 2) u sum|terms|, then h |result|
  * distillation: d = z - m is rounded once, its scaling by log2(e) / temperature three times (the
    constant, its quotient, the product) and 2^x is off by one step, so a share has the relative error
    (4 T + 2) u with T the row's largest |d| / temperature; the sum of V shares adds V' u with V'
    the longest chain of additions and rescalings, at most V / 64 + 128 in any of the kernels
"""
import ctypes as C
import math

import pytest
import torch

from esgd import _lib, ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=F32):
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def close(got, want, bound):
    """|got - want| <= bound everywhere, want and bound in float64."""
    assert got.shape == want.shape
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    if bad.any():
        at = tuple(int(x) for x in torch.nonzero(bad)[0])
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off, first at {at}: {float(got[at])} for "
                             f"{float(want[at])}, {float(d[at])} off, {float(bound[at])} allowed")


def rounded(want, dtype, exact_bound):
    """The bound of a result in `dtype` whose fp32 value is within exact_bound of `want`."""
    return exact_bound * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * want.abs() + TINY[dtype]


# ---- embedding -----------------------------------------------------------------------------

def lookup_want(w, t, scale):
    ok = (t >= 0) & (t < w.shape[0])
    rows = w.double()[t.long().clamp(0, max(0, w.shape[0] - 1))] * scale
    return torch.where(ok[..., None], rows, torch.zeros_like(rows))


@pytest.mark.parametrize("wdt,odt", [(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)])
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 7, 3), (5, 100, 64), (63, 33, 31), (257, 1001, 513), (1000, 50, 1024),
                                   (33, 64, 2051)])
def test_embedding(wdt, odt, n, v, d):
    g = gen(n + v + d)
    w = normal(g, v, d, dtype=wdt)
    t = torch.randint(-1, v + 1, (n,), device=DEV, generator=g)   # -1 and v: outside
    for tokens in (t, t.int()):
        for scale in (1.0, 0.3):
            out = ops.embedding(w, tokens, scale, dtype=odt)
            s32 = float(torch.tensor(scale, dtype=F32))
            want = lookup_want(w, tokens, s32)
            close(out, want, rounded(want, odt, U * want.abs()))


def grad_want(grad, t, v, scale, skip=None):
    ok = (t >= 0) & (t < v)
    if skip is not None:
        ok &= t != skip
    g = torch.where(ok[:, None], grad.double(), torch.zeros((), dtype=torch.float64, device=DEV))
    at = t.long().clamp(0, v - 1)
    total = torch.zeros(v, grad.shape[1], dtype=torch.float64, device=DEV).index_add_(0, at, g) * scale
    size = torch.zeros_like(total).index_add_(0, at, g.abs()) * abs(scale)
    m = torch.zeros(v, dtype=torch.float64, device=DEV).index_add_(0, at, ok.double())
    return total, size * (m[:, None] + 3) * U


# tokens: all the same, all different, few distinct ones, a random mixture, nothing inside the table
TOKENS = {
    "same": lambda g, n, v: torch.full((n,), v - 1, device=DEV),
    "different": lambda g, n, v: torch.randperm(max(n, v), device=DEV, generator=g)[:n],
    "few": lambda g, n, v: torch.randint(0, min(3, v), (n,), device=DEV, generator=g) * max(1, (v - 1) // 2),
    "mixed": lambda g, n, v: torch.randint(-2, v + 2, (n,), device=DEV, generator=g),
    "none": lambda g, n, v: torch.full((n,), -1, device=DEV),
}


@pytest.mark.parametrize("kind", list(TOKENS))
@pytest.mark.parametrize("n,v,d", [(1, 1, 1), (1, 300, 5), (8, 3, 130), (9, 511, 33), (64, 512, 7), (65, 513, 257), (1000, 40, 64),
                                   (4095, 1023, 65), (4096, 1024, 36), (4097, 1025, 33), (9000, 70000, 19),
                                   (70001, 2000, 17)])
def test_embedding_grad(kind, n, v, d):
    g = gen(n * 7 + v + d)
    grad = normal(g, n, d)
    t = TOKENS[kind](g, n, v)
    want, bound = grad_want(grad, t, v, 0.5)
    got = ops.embedding_grad(grad, t, v, 0.5)
    close(got, want, rounded(want, F32, bound))
    again = ops.embedding_grad(grad, t.int(), v, 0.5)
    assert torch.equal(got, again)   # the same bits, whatever the tokens' type


@pytest.mark.parametrize("gdt,wdt", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("n,v,d", [(7, 5, 3), (300, 64, 1000), (5000, 999, 1023)])
def test_embedding_grad_types(gdt, wdt, n, v, d):
    g = gen(n + d)
    grad = normal(g, n, d, dtype=gdt)
    t = torch.randint(0, v, (n,), device=DEV, generator=g)
    want, bound = grad_want(grad, t, v, 2.0, skip=2)
    got = ops.embedding_grad(grad, t, v, 2.0, padding_index=2, dtype=wdt)
    assert got.dtype == wdt
    close(got, want, rounded(want, wdt, bound))
    assert not got[2].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [0, 1, 50, 6000])
def test_embedding_grad_accumulates_into_the_rows_named(dtype, n):
    v, d = 3001, 129
    g = gen(n + 1)
    grad, old = normal(g, n, d, dtype=dtype), normal(g, v, d, dtype=dtype)
    t = torch.randint(0, v // 4, (n,), device=DEV, generator=g) * 3
    out = old.clone()
    out[1] = float("nan")   # a row that no token names: neither read nor written
    assert ops.embedding_grad(grad, t, v, 0.25, out=out, accumulate=True) is out
    total, bound = grad_want(grad, t, v, 0.25)
    assert out[1].isnan().all()
    out[1] = old[1]
    want = old.double() + total
    named = torch.zeros(v, dtype=torch.bool, device=DEV)
    named[t] = True
    assert torch.equal(out[~named], old[~named])
    close(out, want, rounded(want, dtype, bound + U * want.abs()))


def test_embedding_grad_into_out_writes_every_row():
    g = gen(3)
    for n in (0, 10, 5000):
        out = torch.full((2000, 77), float("nan"), device=DEV)
        grad = normal(g, n, 77)
        t = torch.randint(0, 2000, (n,), device=DEV, generator=g)
        ops.embedding_grad(grad, t, 2000, out=out)
        want, bound = grad_want(grad, t, 2000, 1.0)
        close(out, want, rounded(want, F32, bound))


def test_embedding_grad_into_out_counts_as_written():
    # a tensor that autograd has saved and that a gradient was then added to is not used as it was
    g = gen(8)
    t = torch.randint(0, 5, (9,), device=DEV, generator=g)
    out, x = normal(g, 5, 4), normal(g, 5, 4).requires_grad_()
    y = (out * x).sum()
    ops.embedding_grad(normal(g, 9, 4), t, 5, out=out, accumulate=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_embedding_grad_leaves_its_neighbours_alone():
    # out in the middle of a buffer, off every alignment but the element's
    for dtype, off in ((F32, 1), (F32, 3), (BF16, 1), (BF16, 5)):
        for n in (100, 5000):
            v, d = 500, 31
            buf = torch.full((off + v * d + 64,), 7.0, device=DEV, dtype=dtype)
            out = buf[off:off + v * d].view(v, d)
            g = gen(off)
            grad, t = normal(g, n, d, dtype=dtype), torch.randint(0, v, (n,), device=DEV, generator=g)
            ops.embedding_grad(grad, t, v, out=out)
            want, bound = grad_want(grad, t, v, 1.0)
            close(out, want, rounded(want, dtype, bound))
            assert (buf[:off] == 7).all() and (buf[off + v * d:] == 7).all()


def test_embedding_strided_and_many_dimensions():
    g = gen(5)
    big = normal(g, 90, 200)
    t = torch.randint(0, 90, (3, 5, 7), device=DEV, generator=g)
    for w in (big[:, 3:102], big[:, ::2], big.t().contiguous().t(), big[::2]):
        tt = t % w.shape[0]
        out = ops.embedding(w, tt)
        assert out.shape == (3, 5, 7, w.shape[1]) and torch.equal(out, w[tt])
    grad = normal(g, 3, 5, 7, 200)
    for gr in (grad[..., 1:100], grad[..., ::3], torch.ones((), device=DEV).expand(3, 5, 7, 40),
               grad[:, :, :, :64].transpose(0, 1).contiguous().transpose(0, 1)):
        want, bound = grad_want(gr.reshape(-1, gr.shape[-1]), t.reshape(-1), 90, 1.0)
        close(ops.embedding_grad(gr, t, 90), want, rounded(want, F32, bound))
    assert ops.embedding(big, t[:0]).shape == (0, 5, 7, 200)
    assert ops.embedding(big[:0], t).abs().sum() == 0
    assert ops.embedding(big, t.transpose(0, 2)).shape == (7, 5, 3, 200)


def test_embedding_nonfinite_rows_stay_in_their_tokens():
    g = gen(6)
    grad = normal(g, 5000, 40)
    t = torch.randint(0, 300, (5000,), device=DEV, generator=g)
    t[17], t[18], t[19] = -1, 5, 9
    grad[17], grad[18], grad[19] = float("nan"), float("inf"), float("nan")
    got = ops.embedding_grad(grad, t, 300)
    assert torch.isposinf(got[5]).all() and got[9].isnan().all()
    rest = torch.ones(300, dtype=torch.bool, device=DEV)
    rest[5] = rest[9] = False
    assert got[rest].isfinite().all()


def test_embedding_autograd():
    g = gen(8)
    w = normal(g, 301, 65).requires_grad_()
    t = torch.randint(-1, 301, (40, 11), device=DEV, generator=g)
    up = normal(g, 40, 11, 65, dtype=BF16)
    out = ops.embedding(w, t, 3.0, dtype=BF16, padding_index=7)
    assert out.dtype == BF16 and torch.equal(out, ops.embedding(w.detach(), t, 3.0, dtype=BF16))
    out.backward(up)
    want, bound = grad_want(up.reshape(-1, 65), t.reshape(-1), 301, 3.0, skip=7)
    close(w.grad, want, rounded(want, F32, bound))
    # against differences: the operator is linear, so a step of any length gives the slope
    d = normal(g, 301, 65)
    d[7] = 0
    with torch.no_grad():
        w64 = w.double()
        up_slope = ((lookup_want(w64 + d.double(), t, 3.0) - lookup_want(w64 - d.double(), t, 3.0)) / 2 * up.double()).sum()
    slope = (w.grad.double() * d.double()).sum()
    assert abs(float(slope - up_slope)) <= float((bound * d.double().abs()).sum() + U * (want * d.double()).abs().sum())
    # no gradient asked for: none made
    with torch.no_grad():
        assert not ops.embedding(w, t).requires_grad


# ---- tokens by expert ------------------------------------------------------------------------

def order_want(pick, e):
    flat = pick.reshape(-1).long()
    dropped = (flat < 0) | (flat >= e)
    key = torch.where(dropped, torch.full_like(flat, e), flat)
    by = torch.sort(key, stable=True).indices
    place = torch.empty_like(by)
    place[by] = torch.arange(by.numel(), device=DEV)
    slots = torch.where(dropped, -1 - place, place).reshape(pick.shape).int()
    offsets = torch.searchsorted(key[by].contiguous(), torch.arange(e + 1, device=DEV)).int()
    return offsets, slots


@pytest.mark.parametrize("e", [1, 2, 7, 64, 511, 512, 1000, 1023, 1024, 5000])
@pytest.mark.parametrize("n,k", [(0, 2), (1, 1), (3, 5), (64, 1), (341, 3), (4096, 1), (4097, 1), (8192, 8), (21846, 3),
                                 (70000, 4)])
def test_expert_sort(e, n, k):
    g = gen(e + n)
    pick = torch.randint(0, e, (n, k), device=DEV, generator=g)
    mixed = torch.where(torch.rand(n, k, device=DEV, generator=g) < 0.2, torch.full_like(pick, -1), pick)
    for p in (pick, mixed.int(), torch.full_like(pick, e - 1), torch.full_like(pick, e), (mixed // 3).int()):
        order = ops.expert_sort(p, e)
        offsets, slots = order_want(p, e)
        assert order.offsets.dtype == order.slots.dtype == torch.int32
        assert torch.equal(order.offsets, offsets)
        assert torch.equal(order.slots, slots)


@pytest.mark.parametrize("e", [3, 300, 1024, 100000])
@pytest.mark.parametrize("n", [262143, 262144, 262145, 1048576, 1048577, 3000001])
def test_expert_sort_many(e, n):
    # where tiles become larger, and where their counts are summed by a kernel of its own
    g = gen(e + n)
    pick = (torch.rand(n, 1, device=DEV, generator=g).pow(2) * (e + 2)).int() - 1
    order = ops.expert_sort(pick, e)
    offsets, slots = order_want(pick, e)
    assert torch.equal(order.offsets, offsets) and torch.equal(order.slots, slots)


@pytest.mark.parametrize("e", [1, 61, 511, 1022, 1023, 1024, 40000])
@pytest.mark.parametrize("n", [1023, 1024, 1025, 2049, 4095, 4096, 16384, 16385, 32768, 32769, 65536, 65537, 262144, 262145])
def test_expert_sort_borders(e, n):
    # where the sort goes from one workgroup to tiles, to larger tiles and to counts summed apart
    g = gen(e * 3 + n)
    pick = (torch.rand(n, 1, device=DEV, generator=g).pow(3) * (e + 2)).long() - 1
    for p in (pick, torch.full_like(pick, e // 2)):
        order = ops.expert_sort(p, e)
        offsets, slots = order_want(p, e)
        assert torch.equal(order.offsets, offsets) and torch.equal(order.slots, slots)


def test_expert_sort_strided_and_flat():
    g = gen(4)
    pick = torch.randint(-1, 9, (100, 6), device=DEV, generator=g)
    for p in (pick[:, ::2], pick.t().contiguous().t(), pick[::3]):
        offsets, slots = order_want(p, 9)
        order = ops.expert_sort(p, 9)
        assert torch.equal(order.offsets, offsets) and torch.equal(order.slots, slots)
    order = ops.expert_sort(pick[:, 0], 9)
    assert order.slots.shape == (100, 1) and torch.equal(order.slots, order_want(pick[:, :1], 9)[1])


def kept_place(order):
    kept = order.slots >= 0
    return kept, torch.where(kept, order.slots, -1 - order.slots).long()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,k,e,d", [(1, 1, 1, 1), (1, 4, 3, 7), (5, 2, 4, 8), (63, 3, 9, 33), (64, 1, 2, 257), (300, 5, 16, 130),
                                     (1025, 2, 61, 769), (50, 8, 128, 2055), (2000, 9, 40, 24)])
def test_experts(dtype, n, k, e, d):
    g = gen(n + k + e + d)
    pick = torch.randint(-1, e, (n, k), device=DEV, generator=g)
    order = ops.expert_sort(pick, e)
    kept, place = kept_place(order)
    x, y = normal(g, n, d, dtype=dtype), normal(g, n * k, d, dtype=dtype)
    w = torch.rand(n, k, device=DEV, generator=g)
    y[place[~kept]] = float("nan")   # dropped rows and weights take no part
    w[~kept] = float("nan")
    rows = ops.expert_dispatch(x, order)
    want = torch.zeros(n * k, d, device=DEV, dtype=dtype)
    want[place[kept]] = x[:, None].expand(n, k, d)[kept]
    assert torch.equal(rows, want)

    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    w64 = torch.where(kept, w.double(), zero)
    y64 = torch.where(kept[..., None], y.double()[place], zero)
    out = ops.expert_combine(y, w, order)
    terms = w64[..., None] * y64
    close(out, terms.sum(1), rounded(terms.sum(1), dtype, (k + 2) * U * terms.abs().sum(1)))

    grad = normal(g, n, d, dtype=dtype)
    gy, gw = ops.expert_combine_grad(grad, y, w, order)
    want = torch.zeros(n * k, d, dtype=torch.float64, device=DEV)
    want[place.reshape(-1)] = (w64[..., None] * grad.double()[:, None]).reshape(n * k, d)
    close(gy, want, rounded(want, dtype, U * want.abs()))
    terms = y64 * grad.double()[:, None]
    assert gw.dtype == F32
    close(gw, terms.sum(-1), (d + 3) * U * terms.abs().sum(-1))

    gr = normal(g, n * k, d, dtype=dtype)
    gr[place[~kept]] = float("nan")
    gx = ops.expert_dispatch_grad(gr, order)
    terms = torch.where(kept[..., None], gr.double()[place], zero)
    close(gx, terms.sum(1), rounded(terms.sum(1), dtype, (k + 2) * U * terms.abs().sum(1)))


def test_experts_all_dropped_none_and_strided():
    g = gen(9)
    order = ops.expert_sort(torch.full((6, 2), -1, device=DEV), 4)
    assert not order.offsets.any()
    x, y, w = normal(g, 6, 10), normal(g, 12, 10), torch.rand(6, 2, device=DEV, generator=g)
    assert not ops.expert_dispatch(x, order).any() and not ops.expert_combine(y, w, order).any()
    gy, gw = ops.expert_combine_grad(x, y, w, order)
    assert not gy.any() and not gw.any() and not ops.expert_dispatch_grad(y, order).any()
    empty = ops.expert_sort(torch.zeros(0, 2, device=DEV, dtype=torch.int32), 4)
    assert not empty.offsets.any() and ops.expert_dispatch(x[:0], empty).shape == (0, 10)
    assert ops.expert_combine(y[:0], w[:0], empty).shape == (0, 10)
    order = ops.expert_sort(torch.randint(0, 4, (6, 2), device=DEV, generator=g), 4)
    big, tall = normal(g, 6, 64), normal(g, 12, 64)
    for cut in (lambda a: a[:, 5:38], lambda a: a[:, ::2], lambda a: a[:1].expand(a.shape)):
        assert torch.equal(ops.expert_dispatch(cut(big), order), ops.expert_dispatch(cut(big).contiguous(), order))
        assert torch.equal(ops.expert_combine(cut(tall), w, order), ops.expert_combine(cut(tall).contiguous(), w, order))
        a = ops.expert_combine_grad(cut(big), cut(tall), w, order)
        b = ops.expert_combine_grad(cut(big).contiguous(), cut(tall).contiguous(), w, order)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        assert torch.equal(ops.expert_dispatch_grad(cut(tall), order), ops.expert_dispatch_grad(cut(tall).contiguous(), order))


@pytest.mark.parametrize("wdt", [F32, BF16])
def test_experts_autograd(wdt):
    g = gen(10)
    n, k, e, d = 57, 3, 5, 40
    pick = torch.randint(-1, e, (n, k), device=DEV, generator=g)
    order = ops.expert_sort(pick, e)
    x = normal(g, n, d).requires_grad_()
    w = torch.rand(n, k, device=DEV, generator=g).to(wdt).requires_grad_()
    up = normal(g, n, d)
    out = ops.expert_combine(ops.expert_dispatch(x, order) * 2.0, w, order)
    out.backward(up)
    # dispatch then combine: out[t] = 2 (sum of kept weights) x[t]
    kept, _ = kept_place(order)
    total = torch.where(kept, w.detach().double(), 0.0).sum(1, keepdim=True)
    want = 2 * total * x.detach().double()
    close(out.detach(), want, (k + 3) * U * want.abs() + TINY[F32])
    want = 2 * total * up.double()
    close(x.grad, want, (k + 4) * U * want.abs() + TINY[F32])
    dots = (2 * x.detach().double() * up.double())
    want = torch.where(kept, dots.sum(1, keepdim=True), 0.0)
    assert w.grad.dtype == wdt
    close(w.grad, want, rounded(want, wdt, (d + 4) * U * dots.abs().sum(1, keepdim=True).expand(n, k)))
    # against differences (out is linear in x and in w)
    dx = normal(g, n, d)
    slope = ((ops.expert_combine(ops.expert_dispatch(x.detach() + dx, order) * 2.0, w.detach(), order).double()
              - ops.expert_combine(ops.expert_dispatch(x.detach() - dx, order) * 2.0, w.detach(), order).double())
             / 2 * up.double()).sum()
    size = float((2 * total * (x.detach().double().abs() + dx.double().abs()) * up.double().abs()).sum())
    assert abs(float((x.grad.double() * dx.double()).sum() - slope)) <= (2 * k + 10) * U * size


# ---- distillation ----------------------------------------------------------------------------

def distill_want(z, t, index, tau):
    """(loss, gradient of each row's loss, the loss's bound, the gradient's before rounding)."""
    n, v = z.shape
    known = (index >= 0) & (index < v)
    z64 = z.double()
    said = torch.where(known, t.double() / tau, torch.full((), -math.inf, dtype=torch.float64, device=DEV))
    some = (said > -math.inf).any(1)
    log_p = torch.where(some[:, None], torch.log_softmax(torch.where(some[:, None], said, 0.0), 1), 0.0)
    p = torch.where(some[:, None], log_p.exp(), 0.0) * (said > -math.inf)
    z64 = torch.where(some[:, None], z64, 0.0)   # a row without a teacher: its logits do not count
    log_q = torch.log_softmax(z64 / tau, 1)
    at = index.long().clamp(0, v - 1)
    lq = log_q.gather(1, at)
    terms = torch.where(p > 0, p * (log_p - lq), 0.0)
    loss = terms.sum(1) * tau ** 2
    q = log_q.exp()
    taken = torch.zeros_like(q).scatter_add_(1, at, p)
    grad = torch.where(some[:, None], (q - taken) * tau, 0.0)
    finite = torch.where(z64 > -1e30, z64, z64.max(1, keepdim=True).values)
    span = (finite.max(1).values - finite.min(1).values).clamp(0, 200 * tau) / tau   # shares below 2^-149 are 0
    span = span + torch.where(known & (said > -1e30), said.abs(), 0.0).max(1).values * 2 if index.shape[1] else span
    eps = (4 * span + 2 + v / 64 + 128 + index.shape[1]) * U
    size = torch.where((p > 0) & lq.isfinite(), p * (log_p.abs() + lq.abs() + 4), 0.0).sum(1)
    loss_bound = tau ** 2 * eps * (size + 1)
    grad_bound = eps[:, None] * (q + taken) * tau + 1e-37
    return loss, grad, loss_bound, grad_bound


def distill_case(g, n, v, k, dtype, index_dtype=torch.int64):
    z = (torch.randn(n, v, device=DEV, generator=g) * 2).to(dtype)
    index = torch.randint(-1, v + 1, (n, k), device=DEV, generator=g).to(index_dtype)   # some outside, some twice
    t = (torch.rand(n, k, device=DEV, generator=g) * 6).to(dtype)
    return z, t, index


def check_distill(z, t, index, tau, g):
    n = z.shape[0]
    up = torch.rand(n, device=DEV, generator=g) + 0.5
    want, grad, loss_bound, grad_bound = distill_want(z, t, index, tau)
    loss, got = ops.distill_loss_grad(z, t, index, up, tau)
    fine = want.isfinite()
    assert torch.equal(loss.isinf(), ~fine)
    close(loss[fine], want[fine], loss_bound[fine])
    grad, grad_bound = grad * up[:, None].double(), grad_bound * up[:, None].double()
    close(got, grad, rounded(grad, z.dtype, grad_bound + 3 * U * grad.abs()))
    alone = ops.distill_loss(z, t, index, tau)
    assert torch.equal(alone, loss)
    zz = z.detach().clone().requires_grad_()
    (ops.distill_loss(zz, t, index, tau) * up).sum().backward()
    close(zz.grad, grad, rounded(grad, z.dtype, grad_bound + 3 * U * grad.abs()))
    return loss, got


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,v,k,tau", [(1, 1, 1, 1.0), (1, 2, 3, 2.0), (3, 17, 5, 1.0), (5, 63, 64, 4.0), (64, 1001, 10, 4.0),
                                       (9, 2049, 100, 0.5), (130, 8191, 33, 1.0), (2, 8193, 1, 1.0), (7, 40000, 130, 2.0),
                                       (200, 16385, 7, 1.0), (1, 100003, 1024, 1.0), (127, 9001, 64, 1.5), (128, 9001, 64, 1.5)])
def test_distill(dtype, n, v, k, tau):
    g = gen(n + v + k)
    z, t, index = distill_case(g, n, v, k, dtype)
    check_distill(z, t, index, tau, g)


def test_distill_types_of_teacher_and_index():
    g = gen(1)
    for tdt in (F32, BF16, F16):
        z, t, index = distill_case(g, 6, 333, 9, BF16, torch.int32)
        check_distill(z, t.to(tdt), index, 2.0, g)


@pytest.mark.parametrize("n,v", [(6, 500), (6, 30000), (150, 20000)])
def test_distill_rows_without_teacher(n, v):
    # no entry inside the vocabulary, only entries of -inf, or none at all: loss and gradient
    # are 0 whatever the logits hold
    g = gen(2)
    z, t, index = distill_case(g, n, v, 8, F32)
    index = index.clamp(0, v - 1)
    index[1] = -1
    index[2] = v
    t[3] = -math.inf
    t[4, :5] = -math.inf
    index[5, 1:] = index[5, 0]
    z[1:4] = float("nan")
    loss, grad = check_distill(z, t, index, 1.0, g)
    assert not loss[1:4].any() and not grad[1:4].any() and loss[[0, 4, 5]].all()
    loss, grad = ops.distill_loss_grad(z, t[:, :0], index[:, :0], torch.ones(n, device=DEV))
    assert not loss.any() and not grad.any() and grad.shape == z.shape


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", [(5, 700), (5, 20000)])
def test_distill_masked_logits(dtype, n, v):
    g = gen(3)
    z, t, index = distill_case(g, n, v, 6, dtype)
    index = index.clamp(0, v // 2 - 1)
    low = torch.finfo(dtype).min
    z[0, v // 2:] = -math.inf       # a padded vocabulary
    z[1, v // 2:] = low
    z[2] = low                      # all equal: uniform
    z[3] = -math.inf
    z[3, index[3, 0].item()] = 1.0
    index[3] = index[3, 0].item()   # the only one left: q = 1 there
    index[4, 0] = v - 1
    z[4, v - 1] = -math.inf         # the teacher wants what the student rules out
    loss, grad = ops.distill_loss_grad(z, t, index, torch.ones(n, device=DEV))
    want, gw, loss_bound, grad_bound = distill_want(z, t, index, 1.0)
    assert torch.isposinf(loss[4]) and loss[:4].isfinite().all()
    close(loss[:4], want[:4], loss_bound[:4])
    close(grad, gw, rounded(gw, dtype, grad_bound + 3 * U * gw.abs()))
    p = torch.softmax(t[3].double(), 0)   # six times the same index and q = 1: sum p log p is left
    assert abs(float(loss[3].double() - (p * p.log()).sum())) <= float(loss_bound[3])


@pytest.mark.parametrize("n,v", [(3, 900), (3, 20000)])
def test_distill_nonfinite_logits_stay_in_their_rows(n, v):
    g = gen(4)
    z, t, index = distill_case(g, n, v, 6, F32)
    index = index.clamp(0, v - 1)
    for bad in (float("nan"), float("inf")):
        z[1, v - 1] = bad
        loss, grad = ops.distill_loss_grad(z, t, index, torch.ones(n, device=DEV))
        assert loss[1].isnan() and grad[1].isnan().all()
        assert loss[[0, 2]].isfinite().all() and grad[[0, 2]].isfinite().all()
    z[1] = -math.inf   # nothing left for the student
    loss, grad = ops.distill_loss_grad(z, t, index, torch.ones(n, device=DEV))
    assert loss[1].isnan() and grad[1].isnan().all() and loss[[0, 2]].isfinite().all()


def test_distill_strided_and_many_dimensions():
    g = gen(5)
    for v, pitch in ((333, 400), (20000, 20001)):
        buf = torch.full((10, pitch), float("nan"), device=DEV, dtype=BF16)
        z, t, index = distill_case(g, 10, v, 12, BF16)
        buf[:, :v] = z
        up = torch.rand(10, device=DEV, generator=g)
        a = ops.distill_loss_grad(z, t, index, up)
        b = ops.distill_loss_grad(buf[:, :v], t, index, up)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        z3 = z.view(2, 5, v)
        loss, grad = ops.distill_loss_grad(z3, t.view(2, 5, 12), index.view(2, 5, 12), up.view(2, 5))
        assert loss.shape == (2, 5) and torch.equal(loss.view(-1), a[0]) and torch.equal(grad.view(10, v), a[1])
        one = ops.distill_loss(z[0], t[0], index[0])
        assert one.shape == () and torch.equal(one, a[0][0])
        same = torch.full((), 0.25, device=DEV).expand(10)
        assert torch.equal(ops.distill_loss_grad(z, t, index, same)[1],
                           ops.distill_loss_grad(z, t, index, same.contiguous())[1])
        zz = z.clone().requires_grad_()
        ops.distill_loss(zz, t, index).sum().backward()   # an expanded upstream gradient
        ones = torch.ones(10, device=DEV)
        close(zz.grad, ops.distill_loss_grad(z, t, index, ones)[1].double(),
              2 * HALF_STEP[BF16] * zz.grad.double().abs() + TINY[BF16])
    assert ops.distill_loss(z[:0], t[:0], index[:0]).shape == (0,)


def test_distill_gradient_against_differences():
    # loss((z + h d)) - loss(z - h d) over 2 h.  The third derivative of a row's loss along d is
    # tau^2 times that of log sum exp(z / tau), at most 2 max|d|^3 / tau^3 * tau^2, so the
    # difference is off by h^2 / 3 max|d|^3 / tau and by the losses' own errors over h
    g = gen(6)
    n, v, k, tau, h = 8, 1001, 12, 2.0, 0.02
    z, t, index = distill_case(g, n, v, k, F32)
    z.requires_grad_()
    ops.distill_loss(z, t, index, tau).sum().backward()
    d = (torch.rand(n, v, device=DEV, generator=g) - 0.5) * 2
    zp, zm = z.detach() + h * d, z.detach() - h * d
    slope = (ops.distill_loss(zp, t, index, tau).double() - ops.distill_loss(zm, t, index, tau).double()) / (2 * h)
    bound = h * h / 3 / tau + (distill_want(zp, t, index, tau)[2] + distill_want(zm, t, index, tau)[2]) / (2 * h)
    close(slope, (z.grad.double() * d.double()).sum(1), bound + 1e-6)


# ---- how they are called -----------------------------------------------------------------------

def passes(n=300, v=700, d=96, k=3, e=9, vocab=9000, long_tokens=5000):
    """Every operator once, both directions, as a list of tensors (fixed inputs)."""
    g = gen(77)
    w = normal(g, v, d)
    t = torch.randint(-1, v, (n,), device=DEV, generator=g)
    many = torch.randint(-1, v, (long_tokens,), device=DEV, generator=g)
    up, up_many = normal(g, n, d), normal(g, long_tokens, d)
    pick, pick_many = (torch.randint(-1, e, (m, k), device=DEV, generator=g) for m in (n, long_tokens))
    y, wt = normal(g, n * k, d), torch.rand(n, k, device=DEV, generator=g)
    zs = [distill_case(g, rows, vocab, 17, BF16) for rows in (4, 140)]
    ones = [torch.ones(z.shape[0], device=DEV) for z, _, _ in zs]

    def call():
        order, big = ops.expert_sort(pick, e), ops.expert_sort(pick_many, e)
        got = [ops.embedding(w, t, 2.0), ops.embedding_grad(up, t, v, 2.0), ops.embedding_grad(up_many, many, v),
               order.offsets, order.slots, big.offsets, big.slots, ops.expert_dispatch(up, order),
               ops.expert_combine(y, wt, order), *ops.expert_combine_grad(up, y, wt, order),
               ops.expert_dispatch_grad(y, order)]
        for (z, top, index), g1 in zip(zs, ones):
            got += [ops.distill_loss(z, top, index, 2.0), *ops.distill_loss_grad(z, top, index, g1, 2.0)]
        return got
    return call


def same(a, b):
    assert len(a) == len(b)
    for i, (x, y) in enumerate(zip(a, b)):
        assert torch.equal(x, y), i


def test_same_bits_at_every_call_and_on_another_stream():
    call = passes()
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [call() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for got in other + [call()]:
        same(got, first)


def test_work_goes_to_the_current_stream():
    # inputs made on a side stream behind a long kernel queue there, used at once on that stream
    side = torch.cuda.Stream()
    w = torch.zeros(2000, 512, device=DEV)
    t = torch.arange(2000, device=DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(50):
            w += 1
        out = ops.embedding(w, t)
        grad = ops.embedding_grad(out, t, 2000)
    side.synchronize()
    assert (out == 50).all() and (grad == 50).all()


def test_graph_capture_and_replay():
    call = passes()
    eager = call()
    graphs = []
    for _ in range(2):   # two graphs, each with its own work memory
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = call()
        graphs.append((graph, outs))
    for turn in range(4):
        for graph, outs in graphs:
            for o in outs:
                o.zero_()
            graph.replay()
            if turn % 2:
                call()   # eager work between replays
        torch.cuda.synchronize()
        for graph, outs in graphs:
            same(outs, eager)


def test_graph_of_a_training_step():
    # forward and backward captured together, replayed on new inputs
    g = gen(12)
    w = normal(g, 400, 64).requires_grad_()
    t = torch.randint(0, 400, (6, 50), device=DEV, generator=g)
    index = torch.randint(0, 400, (6, 50, 8), device=DEV, generator=g)
    top = torch.rand(6, 50, 8, device=DEV, generator=g)

    def step():
        h = ops.embedding(w, t, 2.0)
        logits = h @ w.detach().t()
        grad, = torch.autograd.grad(ops.distill_loss(logits, top, index).mean(), w)
        return grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        t.copy_(torch.randint(0, 400, (6, 50), device=DEV, generator=gen(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        close(got, step().double(), 64 * U * got.double().abs() + 1e-7)


def test_offsets_beyond_32_bits():
    # 2^31 elements and more in the table's gradient, the rows and the logits
    g = gen(13)
    v, d = 70001, 32768                       # 2.29e9 bf16 elements
    t = torch.tensor([0, v - 1, 40000, v - 1, -1], device=DEV)
    grad = normal(g, 5, d, dtype=BF16)
    table = ops.embedding_grad(grad, t, v)
    want, bound = grad_want(grad, torch.tensor([0, 1, 2, 1, -1], device=DEV), 3, 1.0)
    close(table[[0, v - 1, 40000]], want, rounded(want, BF16, bound))
    assert int((table != 0).any(1).sum()) == 3
    assert torch.equal(ops.embedding(table, t)[:4], table[t[:4]])
    del table
    n, vocab = 16500, 131072                  # 2.16e9
    z = torch.zeros(n, vocab, device=DEV, dtype=BF16)
    z[-1, -1] = 5.0
    index = torch.full((n, 1), vocab - 1, device=DEV)
    loss, gz = ops.distill_loss_grad(z, torch.ones(n, 1, device=DEV), index, torch.ones(n, device=DEV))
    lse = math.log(vocab - 1 + math.exp(5.0))
    assert abs(float(loss[0]) - math.log(vocab)) < 1e-4 and abs(float(loss[-1]) - (lse - 5.0)) < 1e-4
    assert abs(float(gz[-1, -1]) - (math.exp(5.0 - lse) - 1)) < 2 ** -8 and float(gz[0, -1]) == -1.0
    assert abs(float(gz[-2, 7]) * vocab - 1) < 2 ** -7


def test_a_step_of_a_language_model():
    # tokens -> embedding -> experts -> head -> distillation, and back to every parameter, against
    # the same step in 64 bits.  The values are fp32; each stage's relative error is some tens of
    # u and the chain's stays below 4096 u of the largest gradient.
    g = gen(14)
    n, v, d, k, e = 512, 1001, 64, 2, 4
    table = normal(g, v, d).requires_grad_()
    experts = [(normal(g, d, d) / 8).requires_grad_() for _ in range(e)]
    head = (normal(g, d, v) / 8).requires_grad_()
    gate = normal(g, n, e).requires_grad_()
    tokens = torch.randint(-1, v, (n,), device=DEV, generator=g)
    top, pick = torch.topk(gate.detach(), k, dim=1)
    pick = torch.where(torch.rand(n, k, device=DEV, generator=g) < 0.1, torch.full_like(pick, -1), pick)
    t_top, t_index = torch.topk(normal(g, n, v), 16, dim=1)

    def step(p, plain):
        table, head, gate, experts = p
        weights = torch.softmax(gate, 1).gather(1, pick.clamp(min=0))
        if plain:
            x = lookup_want(table, tokens, 2.0)
            out = 0
            for j in range(k):
                for i, m in enumerate(experts):
                    out = out + (pick[:, j] == i)[:, None] * weights[:, j:j + 1] * (x @ m)
            log_p = torch.log_softmax(t_top.double() / 2, 1)
            log_q = torch.log_softmax((x + out) @ head / 2, 1).gather(1, t_index)
            return (log_p.exp() * (log_p - log_q)).sum(1).mean() * 4
        x = ops.embedding(table, tokens, 2.0)
        order = ops.expert_sort(pick, e)
        rows = ops.expert_dispatch(x, order)
        at = order.offsets.tolist() + [n * k]
        y = torch.cat([rows[at[i]:at[i + 1]] @ m for i, m in enumerate(experts)] + [rows[at[e]:]])
        return ops.distill_loss((x + ops.expert_combine(y, weights, order)) @ head, t_top, t_index, 2.0).mean()

    p = [table, head, gate, experts]
    step(p, False).backward()
    q = [a.detach().double().requires_grad_() for a in (table, head, gate)] + [
        [m.detach().double().requires_grad_() for m in experts]]
    step(q, True).backward()
    for a, b in zip([table, head, gate, *experts], [*q[:3], *q[3]]):
        close(a.grad, b.grad, torch.full_like(b.grad, 4096 * U * float(b.grad.abs().max())))


@pytest.mark.parametrize("dtype,vocab", [(BF16, 65537), (BF16, 131072), (BF16, 131073), (F32, 32769), (F32, 65537), (F16, 300001)])
@pytest.mark.parametrize("n", [1, 63, 64, 65, 127, 128, 300])
def test_distill_long_rows(dtype, vocab, n):
    # the borders between rows held by one workgroup, rows read twice and rows in parts
    g = gen(n + vocab)
    z, t, index = distill_case(g, n, vocab, 20, dtype)
    index[n // 2] = -1
    check_distill(z, t, index, 1.0, g)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_distill_rows_just_long_enough_for_parts(dtype):
    # where few rows begin to be split, with entries on both sides of every cut
    g = gen(33)
    for vocab in (45055, 45056, 45057, 49153, 65536):
        for n in (1, 8, 64, 65):
            z, t, index = distill_case(g, n, vocab, 30, dtype)
            cuts = torch.arange(1, 13, device=DEV) * 4096
            index[0, :12] = cuts.clamp(max=vocab - 1)
            index[0, 12:24] = cuts.clamp(max=vocab - 1) - 1
            check_distill(z, t, index, 1.0, g)


@pytest.mark.parametrize("dtype,E", [(F32, 4), (BF16, 8)])
def test_distill_borders_of_the_layers(dtype, E):
    # rows that fill whole layers of vectors, and those an element or a vector shorter and longer
    g = gen(31)
    for vectors in (1, 2, 255, 256, 257, 512, 1024, 1025, 4095, 4096, 4097, 8191, 8192, 8193, 16384):
        for more in (-1, 0, 1):
            vocab = vectors * E + more
            z, t, index = distill_case(g, 3, vocab, 5, dtype)
            index[0, 0], index[0, 1] = vocab - 1, 0
            check_distill(z, t, index, 1.0, g)


@pytest.mark.parametrize("vocab", [1001, 60000])
def test_distill_more_rows_than_workgroups(vocab):
    # every workgroup goes through several rows, with and without a teacher in turn
    g = gen(32)
    n = 5003 if vocab < 2000 else 1300
    z, t, index = distill_case(g, n, vocab, 6, BF16)
    index[::3] = -1
    index[1::7] = 5
    loss, grad = check_distill(z, t, index, 1.0, g)
    none = ~((index >= 0) & (index < vocab)).any(1)   # (some of every third row have got a 5 again)
    assert none.sum() > n // 4 and not loss[none].any() and not grad[none].any()


@pytest.mark.parametrize("d", [1, 2, 3, 4, 5, 8, 9, 31, 33, 64, 65, 128, 129, 255, 257])
@pytest.mark.parametrize("gdt,wdt", [(F32, F32), (BF16, F32), (F16, F16)])
def test_embedding_grad_of_narrow_rows(gdt, wdt, d):
    # runs through many tiles where a row does not fill a wave
    g = gen(d)
    v, n = 50, 4111
    for t in (torch.full((n,), 7, device=DEV), torch.randint(0, 3, (n,), device=DEV, generator=g),
              (torch.rand(n, device=DEV, generator=g).pow(4) * (v + 2)).long() - 1):
        grad = normal(g, n, d, dtype=gdt)
        want, bound = grad_want(grad, t, v, 0.5)
        close(ops.embedding_grad(grad, t, v, 0.5, dtype=wdt), want, rounded(want, wdt, bound))
        had = normal(g, v, d, dtype=wdt)
        out = had.clone()
        ops.embedding_grad(grad, t, v, 0.5, out=out, accumulate=True)
        total = want + had.double()
        close(out, total, rounded(total, wdt, bound + 2 * U * total.abs()))


@pytest.mark.parametrize("kind", ["different", "few", "mixed", "none"])
@pytest.mark.parametrize("gdt,wdt", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("n,v,d", [(5000, 3001, 1001), (4500, 40009, 1023), (9000, 1100000, 129), (20000, 20011, 2047)])
def test_embedding_grad_of_large_tables(kind, gdt, wdt, n, v, d):
    # tables whose rows without a token are zeroed one by one while the sort runs, off alignment
    if gdt == F32 and v == 1100000:
        d = 257
    g = gen(n + v)
    grad = normal(g, n, d, dtype=gdt)
    t = TOKENS[kind](g, n, v)[:n]
    buf = torch.full((v * d + 3,), float("nan"), device=DEV, dtype=wdt)
    out = buf[1:1 + v * d].view(v, d)
    ops.embedding_grad(grad, t, v, 0.5, out=out)
    assert buf[0].isnan() and buf[-2:].isnan().all()
    named = torch.zeros(v, dtype=torch.bool, device=DEV)
    named[t[(t >= 0) & (t < v)].long()] = True
    assert not out[~named].any()   # NaN counts as any
    rows = torch.nonzero(named)[:, 0]
    if len(rows):
        place = torch.full((v,), -1, device=DEV)
        place[rows] = torch.arange(len(rows), device=DEV)
        small = torch.where((t >= 0) & (t < v), place[t.clamp(0, v - 1).long()], -1)
        want, bound = grad_want(grad, small, len(rows), 0.5)
        close(out[rows], want, rounded(want, wdt, bound))


@pytest.mark.parametrize("dtype,n,vocab", [(BF16, 5, 140001), (BF16, 150, 140001), (F32, 5, 70001), (F32, 5, 40001), (F32, 150, 70001)])
def test_distill_odd_values_in_long_rows(dtype, n, vocab):
    # what the shorter rows are tested with, where a row is split, read twice or held by one workgroup
    g = gen(40)
    z, t, index = distill_case(g, n, vocab, 6, dtype)
    index = index.clamp(0, vocab // 2 - 1)
    one = torch.ones(n, device=DEV)
    index[1] = -1
    z[1] = float("nan")                             # no teacher: whatever the logits are
    z[2, vocab // 2:] = -math.inf                   # a padded vocabulary
    z[3] = torch.finfo(dtype).min                   # all equal
    loss, grad = check_distill(z, t, index, 1.0, g)
    assert not loss[1] and not grad[1].any() and not grad[2, vocab // 2:].any()
    for bad in (float("nan"), float("inf")):
        z[4, vocab - 1] = bad
        loss, grad = ops.distill_loss_grad(z, t, index, one)
        assert loss[4].isnan() and grad[4].isnan().all()
        assert loss[:4].isfinite().all() and grad[:4].isfinite().all()
    z[4] = -math.inf
    loss, grad = ops.distill_loss_grad(z, t, index, one)
    assert loss[4].isnan() and grad[4].isnan().all() and grad[:4].isfinite().all()


@pytest.mark.parametrize("n,vocab", [(3, 500), (3, 9000), (2, 140001), (150, 140001)])
def test_distill_odd_values_of_the_teacher(n, vocab):
    # its lowest value is a value, +inf and NaN make the row's results NaN and no other's
    g = gen(41)
    z, t, index = distill_case(g, n, vocab, 5, F32)
    index = index.clamp(0, vocab - 1)
    one = torch.ones(n, device=DEV)
    t[0, 2] = torch.finfo(F32).min
    t[1, :] = torch.finfo(F32).min                  # all the lowest: equal shares
    want, gw, loss_bound, grad_bound = distill_want(z[:2], t[:2], index[:2], 1.0)
    loss, grad = ops.distill_loss_grad(z, t, index, one)
    close(loss[:2], want, loss_bound)
    close(grad[:2], gw, grad_bound + 4 * U * gw.abs() + TINY[F32])
    for bad in (float("nan"), float("inf")):
        t[0, 1] = bad
        loss, grad = ops.distill_loss_grad(z, t, index, one)
        assert loss[0].isnan() and grad[0, index[0]].isnan().any()
        assert loss[1:].isfinite().all() and grad[1:].isfinite().all()


def test_calls_of_two_threads_at_once():
    import threading
    call = passes(n=200, long_tokens=4500)
    want = call()
    torch.cuda.synchronize()
    got, errors = {}, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                got[i] = [call() for _ in range(4)]
            stream.synchronize()
        except Exception as e:   # noqa: BLE001 -- told below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for runs in got.values():
        for r in runs:
            same(r, want)


def test_first_calls_of_a_process_inside_a_capture():
    # a fresh process whose very first call of every operator is captured
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = f"""
import sys
sys.path[:0] = [{here!r}, {os.path.dirname(here)!r}, {os.path.join(os.path.dirname(here), "eager-sgd_amd")!r}]
import torch
import test_ops_gpu as t
call = t.passes()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = call()
graph.replay()
torch.cuda.synchronize()
t.same(outs, call())
print("captured first")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "captured first" in r.stdout, r.stderr[-2000:]


def test_distill_gradient_of_very_many_rows():
    # more rows than a launch has workgroups: every row as it comes in a call of a few
    g = gen(71)
    few, v, n = 1021, 5, (1 << 24) + 3
    z, t, index = distill_case(g, few, v, 2, BF16, torch.int32)
    t[7] = -float("inf")   # and rows without a teacher among them

    def grad_of(z, t, index):
        z = z.clone().requires_grad_()
        ops.distill_loss(z, t, index, 2.0).sum().backward()
        return z.grad

    want = grad_of(z, t, index)
    times = n // few + 1
    got = grad_of(*(x.repeat(times, 1)[:n] for x in (z, t, index)))
    assert torch.equal(got[:n // few * few].view(-1, few, v), want.expand(n // few, few, v))
    assert torch.equal(got[n // few * few:], want[:n % few])


@pytest.mark.parametrize("gdt,wdt", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("n,d", [(1, 5), (4095, 1000), (4096, 512), (16384, 256), (16385, 257), (32769, 1024), (65536, 513), (65537, 512)])
def test_embedding_grad_stays_in_its_work_memory(gdt, wdt, n, d):
    # exactly what it asks for, with marked bytes behind; half the rows are one token's, so that
    # every tile leaves partial sums
    h, size, v = _lib.lib(), C.c_size_t(), 301
    _lib.check(h.esgd_embedding_grad_work(n, v, d, C.byref(size)))
    work = torch.full((size.value + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
    g = gen(n + d)
    grad, out = normal(g, n, d, dtype=gdt), torch.empty(v, d, dtype=wdt, device=DEV)
    t = torch.randint(0, v, (n,), device=DEV, generator=g)
    t[::2] = 7
    code = {F32: _lib.FLOAT, BF16: _lib.BF16, F16: ops.HALF}
    ptr = [C.c_void_p(x.data_ptr()) for x in (grad, t, out, work)]
    _lib.check(h.esgd_embedding_grad(code[gdt], ptr[0], d, n, d, 64, ptr[1], -1, 0.5, code[wdt], ptr[2], v, 0, ptr[3],
                                     size.value, C.c_void_p(torch.cuda.current_stream().cuda_stream or 1)))
    assert (work[size.value:] == 0xA5).all()
    want, bound = grad_want(grad, t, v, 0.5)
    close(out, want, rounded(want, wdt, bound))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_embedding_grad_into_the_gap_between_the_rows_it_reads(dtype):
    # out may lie between rows that stand apart, as close as can be; nothing else is written
    g = gen(21)
    n, d, pitch = 300, 12, 100
    buf = normal(g, n, pitch, dtype=dtype)
    grad, before = buf[:, 5:5 + d], buf.clone()
    t = torch.randint(0, 7, (n,), device=DEV, generator=g)
    want, bound = grad_want(grad, t, 7, 0.5)
    start = 17 * pitch + 5 + d
    out = buf.view(-1)[start:start + 7 * d].view(7, d)   # 84 of the 88 elements between rows 17 and 18
    ops.embedding_grad(grad, t, 7, 0.5, out=out)
    close(out, want, rounded(want, dtype, bound))
    before.view(-1)[start:start + 7 * d] = out.reshape(-1)
    assert torch.equal(buf, before)
    for at in (start - 1, start + 5):   # one element into the row before, one into the row behind
        with pytest.raises(ValueError, match="shares memory with grad"):
            ops.embedding_grad(grad, t, 7, 0.5, out=buf.view(-1)[at:at + 7 * d].view(7, d))
