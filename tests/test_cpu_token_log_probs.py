"""Log probabilities of given tokens, entropies, alternatives (`ops.token_log_probs`) and the logits' gradient, against their
definition in 64 bits, on the host.  The GPU runs the same checks (`test_gpu_token_log_probs.py`)."""
import math

import pytest
import torch

import bagua_core_b200.ops as ops

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # half a step of fp32
INF = float("inf")


def plain(x, targets, top, ignored, a=None, b=None):
    """(log probs, entropies, values, ids, gradient) in 64 bits of rows [n, vocab]."""
    x = x.detach().cpu().double()
    t = targets.cpu()
    n, vocab = x.shape
    scored = t != ignored
    none = (x == -INF).all(1)
    lost = (x.isnan() | (x == INF)).any(1)
    d = x - torch.where(none | lost, 0.0, x.amax(1))[:, None]  # differences first: values may be as large as fp32's
    lp_all = torch.where(x == -INF, -INF, d - d.exp().sum(1).log()[:, None])
    lp_all[lost] = math.nan
    p = torch.where(none[:, None], 0.0, lp_all.exp())
    plogp = torch.where(p > 0, p * lp_all, 0.0)
    plogp[lost] = math.nan
    entropy = torch.where(none, 0.0, -plogp.sum(1))
    hit = torch.zeros_like(x).scatter_(1, t.clamp(0, vocab - 1)[:, None], 1.0)
    lp = lp_all.gather(1, t.clamp(0, vocab - 1)[:, None])[:, 0]
    order = torch.sort(torch.where(x.isnan(), -INF, x), dim=1, descending=True, stable=True)
    values, ids = lp_all.gather(1, order.indices)[:, :top], order.indices[:, :top].clone()
    ids[lost] = -1
    values[~scored], ids[~scored] = -INF, -1
    grad = None
    if a is not None:
        a, b = a.cpu().double(), b.cpu().double()
        grad = a[:, None] * (hit - p) - b[:, None] * (plogp + p * entropy[:, None])
        grad[~scored | none] = 0
    return torch.where(scored, lp, 0.0), torch.where(scored, entropy, 0.0), values, ids, grad


def close(got, want, bound):
    got = got.detach().cpu().double()
    same = (got == want) | (got.isnan() & want.isnan())
    assert (same | ((got - want).abs() <= bound)).all(), float(((got - want).abs() - bound).masked_fill(same, -1).max())


def logits(n, vocab, dtype, seed=0, size=3.0, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, vocab, generator=g) * size * torch.rand(n, 1, generator=g)
    if masked:
        x[torch.rand(n, vocab, generator=g) < masked] = -INF
    return x.to(dtype), torch.randint(0, vocab, (n,), generator=g)


def check(x, targets, top=0, ignored=-100, backward=True, make=lambda x: x):
    """`make`: the tensor of the same values that the operator is given."""
    n, vocab = x.shape
    y = make(x.detach()).requires_grad_(backward)
    r = ops.token_log_probs(y, targets.to(y.device), top, ignored)
    g = torch.Generator().manual_seed(5)
    a, b = torch.randn(n, generator=g), torch.randn(n, generator=g)
    lp, entropy, values, ids, grad = plain(x, targets, top, ignored, a, b)
    # each exponential 2^-22, its argument two half steps of its size (below 2^7 where it counts), a sum of up to vocab / 256 + 64 terms in a
    # row; then logarithm, difference and product
    off = 2.0 ** -22 + (vocab / 256 + 64 + 2 ** 8) * U
    size = x.detach().cpu().double().nan_to_num(0, 0, 0).abs().clamp(max=1e30)
    m = torch.where(size.isinf(), 0, size).amax(1)
    close(r.log_probs, lp, off + 4 * U * (lp.abs().nan_to_num(0, 0, 0) + m))
    close(r.entropy, entropy, 2 * off * (1 + entropy.abs().nan_to_num(0, 0, 0) + 4))
    if top:
        assert r.top_ids.shape == (n, top) and torch.equal(r.top_ids.cpu(), ids)
        close(r.top_log_probs, values, off + 4 * U * (values.abs().nan_to_num(0, 0, 0) + m[:, None]))
        assert not r.top_log_probs.requires_grad
    else:
        assert r.top_ids is None and r.top_log_probs is None
    if backward:
        (d,) = torch.autograd.grad((r.log_probs, r.entropy), y, (a.to(y.device), b.to(y.device)))
        assert d.shape == y.shape and d.dtype == y.dtype
        half = torch.finfo(x.dtype).eps / 2
        lpa = torch.log_softmax(x.detach().cpu().double().clamp(min=-1e30), 1).nan_to_num(0, 0, 0).abs().clamp(max=100)
        p = torch.exp(-lpa)
        entropy = entropy.abs().nan_to_num(0, 0, 0)
        # (where p is below 2^-100 nothing is left of it)
        parts = p * (a.abs()[:, None] + b.abs()[:, None] * (lpa + entropy[:, None] + 4).double()) + a.abs()[:, None] * 0
        close(d, grad, 4 * off * parts + half * grad.abs().nan_to_num(0, 0, 0) + U * a.abs()[:, None] * 2 + torch.finfo(x.dtype).smallest_normal * half + 2.0 ** -100)
    return r


SIZES = [(1, 1), (3, 2), (4, 7), (5, 33), (9, 255), (3, 1000)]


@pytest.mark.parametrize("dtype", TYPES.values())
@pytest.mark.parametrize("n,vocab", SIZES)
def test_against_the_definition(n, vocab, dtype):
    x, t = logits(n, vocab, dtype)
    check(x, t, min(vocab, 5))
    x, t = logits(n, vocab, dtype, masked=0.5)
    check(x, t, min(vocab, 32))


def check_special(device):
    for dtype in TYPES.values():
        low = torch.finfo(dtype).min
        for vocab in (40, 3000):
            x, t = logits(12, vocab, dtype)
            x[0] = -INF                  # no token left
            x[1] = low                   # all equal, at the type's lowest value
            x[2, 1:] = low               # one left by a mask of that value
            x[3, 1:] = -INF              # one left
            x[4, 7] = math.nan
            x[5, 3] = INF
            x[6] = torch.finfo(dtype).max
            x[7, ::2] = low
            x[8] = x[8, 0]               # all equal
            x[9, 5] = x[9].max() + 1
            x[9, 20] = x[9, 5]           # two equal at the top
            t[10] = -100
            x[11] = -INF
            t[11] = -100
            t[2], t[3], t[9] = 0, 0, 20
            check(x.to(device), t, 6)
            check(x.to(device), t, 32)
            x[10] = math.nan             # a row that is not looked at
            r = check(x.to(device), t, 1)
            assert r.log_probs[10] == 0 and r.entropy[10] == 0
            # another mark, which may be a token
            check(x.to(device), t.masked_fill(t == -100, 4), 2, ignored=4)


def test_special_rows():
    check_special("cpu")


def check_ends_of_the_range(device):
    """Rows with logits at the ends of the type's range have the values that their formula says, whatever the size of their logits."""
    g = torch.Generator().manual_seed(11)
    for dtype in TYPES.values():
        low, top = torch.finfo(dtype).min, torch.finfo(dtype).max
        for vocab in (40, 1000, 3000):
            x = torch.zeros(8, vocab)
            x[0] = low                                # all equal
            x[1] = top
            x[2] = low                                # one left
            x[2, 9] = 0.25
            x[3], x[3, 9] = low, low / 2              # one left among large ones
            x[4, ::2], x[4, 1::2] = low, 0.0          # a half, all alike
            x[5, :10], x[5, 10:] = top, low           # ten
            x[6], x[6, :vocab // 2] = low, -INF       # half of nothing but the lowest
            x[7], x[7, 9] = 1.0, top                  # one far above
            n = torch.tensor([vocab, vocab, 1, 1, vocab // 2, 10, vocab - vocab // 2, 1.0])
            t = torch.tensor([1, 1, 9, 9, 1, 0, vocab - 1, 9])
            b = torch.randn(8, generator=g)
            y = x.to(dtype).to(device).requires_grad_()
            r = ops.token_log_probs(y, t.to(device), 3)
            (d,) = torch.autograd.grad((r.log_probs, r.entropy), y, (torch.ones(8, device=device), b.to(device)))
            # logarithms below 2^3.1 in base 2: sums of up to 3000 exact ones, log2 and its product, within 2^-20
            close(r.log_probs, -n.double().log(), 2.0 ** -20)
            # each p log p: p is off by half a step of its logarithm (up to 8, so 2^-22), by exp's step and a half, and by the product's half:
            # 2^-21 of it at most, and the whole, up to 8, by that and half a step for each of the levels of its sum
            close(r.entropy, n.double().log(), 2.0 ** -17)
            assert torch.equal(r.top_ids[:, 0].cpu(), torch.tensor([0, 0, 9, 9, 1, 0, vocab // 2, 9]))
            close(r.top_log_probs[:, 0], -n.double().log(), 2.0 ** -20)
            # all that are left are alike: no gradient of the entropy, and 1 / n of the log probability's
            left = (x.to(dtype) == x.to(dtype).amax(1, keepdim=True)).double()
            want = torch.zeros(8, vocab, dtype=torch.float64).scatter_(1, t[:, None], 1.0) - left / n.double()[:, None]
            close(d, want, (torch.finfo(dtype).eps / 2 + 2.0 ** -20) * want.abs() + 2.0 ** -20 * (1 + b.abs()[:, None]) * left)


def test_ends_of_the_range():
    check_ends_of_the_range("cpu")


def check_layouts(device):
    x, t = logits(24, 37, torch.bfloat16)
    x, t = x.to(device), t.to(device)
    want = ops.token_log_probs(x, t, 3)

    # The order of a row's sum follows its alignment: two orders differ by at most what each may be off (37 terms, sums and
    # values below 2^5), gradients by that relative to 1 and then by a step of bf16.
    off = 2 * (2.0 ** -22 + (37 + 64) * U) * 8

    def alike(d, first):
        return ((d.double() - first.double()).abs() <= 2 * off + 2.0 ** -7 * first.double().abs()).all()

    def same(y, shape, u=t):
        y = y.requires_grad_()
        r = ops.token_log_probs(y, u.view(shape), 3)
        assert r.log_probs.shape == shape and torch.equal(r.top_ids.reshape(24, 3), want.top_ids) and r.top_ids.shape == (*shape, 3)
        assert all(((p.reshape(q.shape) - q).abs() <= off).all() for p, q in zip(r[:3], want[:3]))
        (d,) = torch.autograd.grad((r.log_probs.sum(), r.entropy.sum()), y)
        assert d.shape == y.shape
        return d.reshape(24, 37)

    first = same(x.clone(), (24,))
    assert alike(same(x.clone().view(2, 3, 4, 37), (2, 3, 4)), first)
    for pad in (1, 3, 11):  # a vocabulary padded to a multiple: rows that start anywhere
        wide = torch.full((24, 37 + pad), 9.0, dtype=x.dtype, device=device)
        wide[:, :37] = x
        assert alike(same(wide[:, :37], (24,)), first)
        wide[:, pad:] = x
        assert alike(same(wide[:, pad:].unflatten(0, (4, 6)), (4, 6)), first)
    assert alike(same(x.t().contiguous().t(), (24,)), first)
    half = torch.zeros(48, 37, dtype=x.dtype, device=device)
    half[::2] = x
    assert alike(same(half[::2], (24,)), first)
    swapped = x.view(4, 6, 37).transpose(0, 1).contiguous().transpose(0, 1)  # rows in another order
    assert alike(same(swapped, (4, 6)), first)
    one = ops.token_log_probs(x[5], t[5], 2)
    assert one.log_probs.shape == () and (one.log_probs - want.log_probs[5]).abs() <= off and torch.equal(one.top_ids, want.top_ids[5, :2])
    # one row for many targets: the gradients of a broadcast row are summed
    row = x[:1].float().requires_grad_()
    u = torch.arange(37, device=device)
    lp = ops.token_log_probs(row.expand(37, 37), u).log_probs
    (d,) = torch.autograd.grad(lp.sum(), row)
    p = torch.softmax(row.detach().double(), 1)
    assert (d.double() - (1 - 37 * p)).abs().max() <= 37 * 40 * U
    # no rows
    for shape in ((0, 5), (2, 0, 5)):
        e = torch.zeros(shape, device=device, requires_grad=True)
        r = ops.token_log_probs(e, torch.zeros(shape[:-1], dtype=torch.int64, device=device), 2)
        assert r.log_probs.shape == shape[:-1] and r.top_ids.shape == (*shape[:-1], 2)
        r.log_probs.sum().backward()
        assert e.grad.shape == shape


def test_layouts():
    check_layouts("cpu")


def check_partial_gradients(device):
    x, t = logits(6, 50, torch.float32)
    for k in range(2):
        y = x.to(device).requires_grad_()
        r = ops.token_log_probs(y, t.to(device))
        (d,) = torch.autograd.grad(r[k].sum(), y)
        a, b = torch.full((6,), float(k == 0)), torch.full((6,), float(k == 1))
        want = plain(x, t, 0, -100, a, b)[4]
        assert (d.cpu().double() - want).abs().max() <= 400 * U
    # against differences in 64 bits of the definition
    eps = 1e-5
    y = x.to(device).requires_grad_()
    r = ops.token_log_probs(y, t.to(device))
    (d,) = torch.autograd.grad((2.0 * r.log_probs - 0.5 * r.entropy).sum(), y)
    for i, j in ((0, 0), (2, 49), (5, int(t[5]))):
        ends = []
        for s in (1, -1):
            z = x.double().clone()
            z[i, j] += s * eps
            lp, h, *_ = plain(z, t, 0, -100)
            ends.append(float((2.0 * lp - 0.5 * h).sum()))
        assert abs((ends[0] - ends[1]) / (2 * eps) - float(d[i, j])) < 1e-5


def test_one_gradient_of_two():
    check_partial_gradients("cpu")


def check_second_order(device):
    x, t = logits(3, 6, torch.float32)
    x[0, 2] = -INF
    t[2] = -100
    f = lambda y: (lambda r: (r.log_probs * torch.tensor([1.0, -2.0, 3.0], device=device)).sum() + r.entropy.sum())(ops.token_log_probs(y, t.to(device)))  # noqa: E731

    def g(y):
        r = torch.log_softmax(y, 1)
        p = r.exp()
        lp = r.gather(1, t.to(device)[:, None].clamp(min=0))[:, 0]
        h = -(p * r.clamp(min=-1e30)).sum(1)
        return lp[0] - 2 * lp[1] + h[0] + h[1]

    ys = [x.to(device).requires_grad_() for _ in range(2)]
    v = torch.randn(3, 6, generator=torch.Generator().manual_seed(2)).to(device)
    v[0, 2] = 0
    got = []
    for fn, y in zip((f, g), ys):
        (d,) = torch.autograd.grad(fn(y), y, create_graph=True)
        got.append((d.detach(), torch.autograd.grad((d * v).sum(), y)[0]))
    assert torch.allclose(got[0][0], got[1][0], atol=1e-6) and torch.allclose(got[0][1], got[1][1], atol=1e-6)


def test_second_order():
    check_second_order("cpu")


def check_scaled_entropy_gradients(device):
    """Entropy's gradient under factors as loss scales bring them, where masks leave one token, few, or half of them."""
    for dtype in TYPES.values():
        half = torch.finfo(dtype).eps / 2
        for vocab in (40, 3000):
            for low in (-INF, torch.finfo(dtype).min):
                x, t = logits(6, vocab, dtype, seed=vocab)
                x[0, 1:] = low
                x[1, :vocab - 1] = low
                x[2, 3:] = low
                x[3, vocab // 2:] = low
                x[4, ::2] = low
                t = torch.zeros_like(t)
                for size in (1e-3, 5.0, 1e4 if dtype == torch.float16 else 1e5) + (() if dtype == torch.float16 else (1e20,)):
                    b = size * torch.tensor([1.0, -1.0, 1.0, -1.0, 1.0, -1.0])
                    _, entropy, _, _, want = plain(x, t, 0, -100, torch.zeros(6), b)
                    y = x.to(device).requires_grad_()
                    (d,) = torch.autograd.grad(ops.token_log_probs(y, t.to(device)).entropy, y, b.to(device))
                    assert d.isfinite().all() and not d.cpu()[x == low].any()
                    # as in check(): a probability is off by `off` relative to itself, its logarithm and the entropy by that relative to 1
                    # and their size; what is below 2^-126 is lost
                    off = 2.0 ** -22 + (vocab / 256 + 64 + 2 ** 8) * U
                    lp = torch.log_softmax(x.double().clamp(min=-1e30), 1).clamp(min=-100)
                    parts = lp.exp() * b.abs()[:, None] * (lp.abs() + entropy[:, None] + 4)
                    close(d, want, 4 * off * parts + half * want.abs() + torch.finfo(dtype).smallest_normal * half + size * 2.0 ** -110)


def test_scaled_entropy_gradients():
    check_scaled_entropy_gradients("cpu")


def check_large_alternatives(device):
    """Alternatives' values do not lose the row's sum beside large logits."""
    for dtype, sizes in ((torch.float32, (1e3, 3e4, 1e10, 1e30, 3e38)), (torch.bfloat16, (1e3, 1e10, 3e38)), (torch.float16, (1e3, 3e4, 65504.0))):
        for size in sizes:
            for sign in (1, -1):
                x = torch.full((3, 50), sign * size).to(dtype)
                x[1, 7] = 0.5 * size
                x[2, 25:] = -INF
                r = ops.token_log_probs(x.to(device), torch.zeros(3, dtype=torch.int64, device=device), 2)
                want = torch.tensor([[math.log(1 / 50)] * 2, [math.log(1 / 49)] * 2, [math.log(1 / 25)] * 2], dtype=torch.float64)
                if sign < 0:
                    want[1] = torch.tensor([0.0, float(x[1, 0].double() - x[1, 7].double())])
                close(r.top_log_probs, want, 2.0 ** -22 + 2 ** 5 * U * 4 + 2 * U * want.abs())


def test_large_alternatives():
    check_large_alternatives("cpu")


def check_kept_graphs(device, unknown=False):
    """The gradient does not depend on whether it will be differentiated, and its own is that of the formula: for targets that a mask
    forbids, rows that it leaves nothing of, and unknown targets."""
    x, t = logits(5, 9, torch.float32)
    x[0, 2:5], t[0] = -INF, 3
    x[1], t[1] = -INF, 0
    x[2, :8], t[2] = -INF, 8
    t[3] = -100
    ok = t.to(device)
    if unknown:
        t = t.clone()
        t[4] = 9
    dropped = torch.tensor([False, True, False, True, unknown])
    g = torch.Generator().manual_seed(3)
    a, b, v = torch.randn(5, generator=g), torch.randn(5, generator=g), torch.randn(5, 9, generator=g)

    def formula(y, a, b):
        ls = torch.log_softmax(torch.where(dropped[:, None], 0.0, y), 1)
        p = ls.exp()
        h = -(p * ls.clamp(min=-200)).sum(1, keepdim=True)
        hit = torch.zeros_like(p).scatter_(1, t.clamp(0, 8)[:, None], 1.0)
        d = a[:, None] * (hit - p) - b[:, None] * p * (ls.clamp(min=-200) + h)
        return torch.where(dropped[:, None], 0.0, d)

    ins = [z.double().requires_grad_() for z in (x, a, b)]
    want = formula(*ins)
    seconds = torch.autograd.grad((want * v).sum(), ins)
    for both in (0, 1, 2):  # gradients of both, of the log probabilities, of the entropies
        got = []
        for keep in (False, True):
            y, c, e = (z.to(device).requires_grad_() for z in (x, a, b))
            r = ops.token_log_probs(y, t.to(device))
            if unknown:
                torch.cuda.synchronize()
                with pytest.raises(RuntimeError, match="not in the vocabulary"):
                    ops.token_log_probs(y, ok)
            outs, ups = ((r.log_probs, r.entropy), (c, e)) if both == 0 else ((r[both - 1],), ((c, e)[both - 1],))
            (d,) = torch.autograd.grad(outs, y, ups, create_graph=keep)
            got.append(d.detach().cpu().double())
        # values of some units, sums of 9 terms, a hundred roundings at most
        assert (got[0] - got[1]).abs().max() <= 400 * U
        if both == 0:
            assert (got[1] - want.detach()).abs().max() <= 400 * U
            for z, w in zip(torch.autograd.grad((d * v.to(device)).sum(), (y, c, e)), seconds):
                assert (z.cpu().double() - w).abs().max() <= 1000 * U


def test_kept_graphs():
    check_kept_graphs("cpu")


def large_rows(vocab, dtype, size, g):
    """Rows whose logits are near `size` in different ways, and tokens to ask for."""
    x = torch.randn(6, vocab, generator=g)
    x[0] = size                                          # all equal
    x[1] = size                                          # one that is not
    x[1, vocab // 2] = 0.5 * size
    x[2, vocab // 3] = size                              # one among ordinary ones
    x[3, :vocab // 2] = size                             # a half
    x[4, torch.rand(vocab, generator=g) < 0.5] = size    # every other one
    # neighbours of `size`, some steps of fp32 or of the type apart
    step = max(abs(size) * 2.0 ** -23, 2.0 ** -3 if abs(size) >= 2 ** 20 else 0, abs(size) * torch.finfo(dtype).eps)
    x[5] = size + step * torch.randint(-40, 41, (vocab,), generator=g).double()
    return x.clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).to(dtype), torch.tensor([3, vocab // 2, vocab // 3, vocab - 1, 0, 1])


def check_large_logits(device, vocabs, rows):
    """Against 64 bits, with a tolerance that does not grow with the logits: a log probability is a difference of logits, each exact."""
    g = torch.Generator().manual_seed(7)
    for dtype in TYPES.values():
        half = torch.finfo(dtype).eps / 2
        sizes = [100.0, 3e4, 59968.0, 6e4, 65000.0] if dtype == torch.float16 else [
            1e5, 2.0 ** 20 - 1, 2.0 ** 20, 2.0 ** 20 + 1, 3e6, 1e9, 6e9, 1e10, 1e12, 1e20, 1e30, 9e36, 3e37, 9.9e37, 1.1e38, 3e38]
        for vocab in vocabs:
            off = 2.0 ** -22 + (vocab / 256 + 64 + 2 ** 8) * U
            for size in sizes:
                for sign in (1, -1):
                    x, t = large_rows(vocab, dtype, sign * size, g)
                    for lo in range(0, len(x), rows):
                        u, v = x[lo:lo + rows], t[lo:lo + rows]
                        a, b = torch.randn(len(u), generator=g), torch.randn(len(u), generator=g)
                        lp, entropy, values, ids, want = plain(u, v, 7, -100, a, b)
                        y = u.to(device).requires_grad_()
                        r = ops.token_log_probs(y, v.to(device), 7)
                        (d,) = torch.autograd.grad((r.log_probs, r.entropy), y, (a.to(device), b.to(device)))
                        # log sum: a relative error `off` of the sum, and half a step of its logarithm, below 2^5; difference and product
                        # three half steps of the result
                        close(r.log_probs, lp, off + 2 ** 5 * U + 4 * U * lp.abs())
                        close(r.top_log_probs, values, off + 2 ** 5 * U + 4 * U * values.abs())
                        assert torch.equal(r.top_ids.cpu(), ids)
                        close(r.entropy, entropy, 2 * off * (1 + entropy.abs() + 4))
                        w = u.double() - u.double().amax(1)[:, None]
                        la = torch.log_softmax(w, 1).clamp(min=-100)
                        parts = la.exp() * (a.abs()[:, None] + b.abs()[:, None] * (la.abs() + entropy.abs()[:, None] + 4))
                        close(d, want, 4 * off * parts + (half + 2 * U) * (want.abs() + a.abs()[:, None]) + torch.finfo(dtype).smallest_normal + 2.0 ** -100)


def test_large_logits():
    check_large_logits("cpu", (40, 3000), 6)


def check_refusals(device):
    x, t = torch.zeros(3, 5, device=device), torch.zeros(3, dtype=torch.int64, device=device)
    for args in ((x.double(), t), (x.long(), t), (x, t.int()), (x, t[:2]), (x, t.view(3, 1)), (x, t, 6), (x, t, -1), (x[:, :0], t),
                 (torch.zeros((), device=device), t), (torch.zeros(3, 50, device=device), t, 33), (x.to_sparse(), t)):
        with pytest.raises(RuntimeError):
            ops.token_log_probs(*args)


def test_refusals():
    check_refusals("cpu")
    x = torch.zeros(3, 5)
    for bad in (-1, 5):
        with pytest.raises(RuntimeError, match="not in the vocabulary"):
            ops.token_log_probs(x, torch.tensor([0, bad, -100]))
