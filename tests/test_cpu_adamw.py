"""AdamW steps over lists of tensors (`ops.adamw_step`), moments in fp32 and in 8 bits, and the flat optimizer on them: on the
host, against the definition in 64 bits.  The GPU runs the same checks (`test_gpu_adamw.py`)."""
import copy

import pytest
import torch

import adamw_plain as plain
import bagua_core_b200.ops as ops
import bagua_core_b200.parallel as P

TYPES = [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.float32, torch.float16),
         (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32)]
SIZES = [1, 3, 255, 256, 257, 1024, 5000]
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
U = 2.0 ** -24  # half a step of fp32


def tensors(sizes, dtypes, device, seed=0):
    """Parameters, gradients and moments whose sizes differ from block to block by orders of magnitude."""
    g = torch.Generator().manual_seed(seed)
    ps, gs, ms, vs = [], [], [], []
    for n in sizes:
        scale = torch.exp(2 * torch.randn((n + 255) // 256, generator=g) - 6).repeat_interleave(256)[:n]
        ps.append(torch.randn(n, generator=g).to(dtypes[0]))
        gs.append((torch.randn(n, generator=g) * scale).to(dtypes[1]))
        ms.append(torch.randn(n, generator=g) * scale * 0.3)
        vs.append((torch.randn(n, generator=g) * scale).square() + 0.1 * scale * scale)
    return [[t.to(device) for t in x] for x in (ps, gs, ms, vs)]


def close_param(got, want, old, dtype, lr):
    """p is rounded to its type once; before that: three fp32 roundings of p's size, and of the update (at most 10 lr here, since the
    moments of a test fit each other to within that) its division, its factors and both moments, 16 roundings at most."""
    half = torch.finfo(dtype).eps / 2
    bound = want.abs() * half + torch.finfo(dtype).smallest_normal * half + 3 * U * (old.double().abs() + want.abs()) + 10 * lr * 16 * U
    assert ((got.cpu().double() - want).abs() <= bound).all()


def check_step32(device, dtypes, t, copies=True, sizes=SIZES, hyper=HYPER):
    ps, gs, ms, vs = tensors(sizes, dtypes, device)
    old = [[t.cpu().clone() for t in x] for x in (ps, gs, ms, vs)]
    cs = [torch.zeros_like(p, dtype=torch.bfloat16) for p in ps] if copies else None
    ops.adamw_step(ps, gs, ms, vs, step=t, copies=cs, **hyper)
    b1, b2 = hyper["betas"]
    for k in range(len(sizes)):
        p, g, m, v = (x[k] for x in old)
        want = plain.step(p, g, m, v, t, hyper["lr"], b1, b2, hyper["eps"], hyper["weight_decay"])
        close_param(ps[k], want[0], p, dtypes[0], hyper["lr"])
        # a product, a multiply-add and two constants rounded: two half steps of each term and one of the sum
        assert ((ms[k].cpu().double() - want[1]).abs() <= 3 * U * ((b1 * m).abs() + ((1 - b1) * g.double()).abs()) + 1e-45).all()
        assert ((vs[k].cpu().double() - want[2]).abs() <= 4 * U * (b2 * v + (1 - b2) * g.double().square()) + 1e-45).all()
        assert torch.equal(gs[k].cpu(), g)
        if copies and dtypes[0] == torch.float32:
            assert torch.equal(cs[k], ps[k].bfloat16())


def check_step8(device, dtypes, t, sizes=SIZES, seed=7, first_index=2, offset=0):
    """One step from moments that were written by earlier steps; `offset`: where the tensors start in their memory."""
    ps, gs, _, _ = tensors(sizes, dtypes, device)
    if offset:
        move = lambda xs: [torch.zeros(x.numel() + offset, dtype=x.dtype, device=device)[offset:].copy_(x) for x in xs]  # noqa: E731
        ps, gs = move(ps), move(gs)
    state = [ops.adamw_state8(p) for p in ps]
    if offset:
        state = [(move([a])[0], move([b])[0], s) for a, b, s in state]
    ms, vs, ss = ([s[i] for s in state] for i in range(3))
    b1, b2 = HYPER["betas"]
    for j in range(1, 3):
        ops.adamw_step(ps, gs, ms, vs, step=j, scales=ss, seed=seed, **HYPER)
        gs = [g * 0.7 + g.roll(1) * 0.5 if g.numel() > 1 else g for g in gs]
    old = [[t.cpu().clone() for t in x] for x in (ps, gs, ms, vs, ss)]
    ops.adamw_step(ps, gs, ms, vs, step=t, scales=ss, seed=seed, first_index=first_index, **HYPER)
    for k, n in enumerate(sizes):
        m0, v0 = plain.read(old[2][k], old[3][k], old[4][k])
        want, m, v = plain.step(old[0][k], old[1][k], m0, v0, t, HYPER["lr"], b1, b2, HYPER["eps"], HYPER["weight_decay"])
        close_param(ps[k], want, old[0][k], dtypes[0], HYPER["lr"])
        random = plain.random_bits(seed, t, first_index + k, n)
        # the moments (4 half steps), the scale (their largest, divided: 5), its reciprocal and the product (2)
        slack = 12 * U
        for x, row, largest, table, u, code in ((m, 0, 480, plain.FIRST, random & 0xFFFF, ms[k]), (v, 1, 496, plain.SECOND, random >> 16, vs[k])):
            scale = ss[k][row].cpu().double()
            assert ((scale - plain.tops(x) / largest).abs() <= 6 * U * scale + 2.0 ** -126).all()
            lo, hi = plain.codes(x, plain.spread(ss[k][row].cpu(), n), table, (u.double() + 0.5) / 65536, slack)
            c = code.cpu().long().flatten()
            if row == 0:
                # the first moment is a difference where its two terms cancel: allow what they leave
                terms = (b1 * m0.abs() + (1 - b1) * old[1][k].double().abs()) * 4 * U / plain.spread(ss[k][0].cpu(), n).clamp(min=1e-300)
                lo2, _ = plain.codes((x.abs() / plain.spread(ss[k][0].cpu(), n) - terms).clamp(min=0), torch.ones(n, dtype=torch.float64), table,
                                     (u.double() + 0.5) / 65536, slack)
                _, hi2 = plain.codes(x.abs() / plain.spread(ss[k][0].cpu(), n) + terms, torch.ones(n, dtype=torch.float64), table,
                                     (u.double() + 0.5) / 65536, slack)
                lo, hi = torch.minimum(lo, lo2), torch.maximum(hi, hi2)
                assert ((c & 127 >= lo) & (c & 127 <= hi)).all()
                assert (((c > 127) == (x < 0)) | (c & 127 == 0)).all()
            else:
                assert ((c >= lo.clamp(min=1)) & (c <= hi.clamp(min=1)) | (x == 0) & (c == 0)).all()
    outs = [[torch.empty_like(p, dtype=d) for p in ms] for d in (torch.float32, torch.float32)]
    ops.adamw_read8(ms, vs, ss, *outs)
    for k, n in enumerate(sizes):
        m, v = plain.read(ms[k], vs[k], ss[k])
        assert ((outs[0][k].cpu().double() - m).abs() <= U * m.abs() + 1e-45).all()
        assert ((outs[1][k].cpu().double() - v).abs() <= U * v.abs() + 1e-45).all()


@pytest.mark.parametrize("dtypes", TYPES)
@pytest.mark.parametrize("t", [1, 1000])
def test_step_with_fp32_moments(dtypes, t):
    check_step32("cpu", dtypes, t)


@pytest.mark.parametrize("dtypes", TYPES)
def test_step_with_8_bit_moments(dtypes):
    check_step8("cpu", dtypes, 3)


def check_mean(device):
    """Moments that a step changes by less than a code's distance follow their mean: a constant gradient after another one."""
    n = 1 << 14
    p, g = torch.zeros(n, device=device), torch.full((n,), 1e-3, device=device)
    g[::256] = 4e-3  # the largest of each block
    m, v, s = ops.adamw_state8(p)
    for t in range(1, 2001):
        if t == 1001:
            g *= 0.5
        ops.adamw_step([p], [g], [m], [v], step=t, lr=0.0, weight_decay=0.0, scales=[s], seed=3)
    mean_m, mean_v, ref = torch.zeros(1, device=device), torch.zeros(1, device=device), 0.0
    out = torch.empty_like(p), torch.empty_like(p)
    ops.adamw_read8([m], [v], [s], [out[0]], [out[1]])
    keep = torch.arange(n, device=device) % 256 != 0
    mean_m, mean_v = out[0][keep].double().mean().item(), out[1][keep].double().mean().item()
    for t in range(1, 2001):
        ref = 0.999 * ref + 0.001 * ((1e-3 if t <= 1000 else 5e-4) ** 2)
    # standard error of the mean over 16320 elements: a code's rounding varies by at most 1/64 of its square (v: an element in
    # between two codes a sixteenth apart), summed over 500 steps' memory: 35 % of an element, 0.3 % of the mean; five of them
    assert abs(mean_v / ref - 1) < 0.015
    assert abs(mean_m / 5e-4 - 1) < 0.005


def test_8_bit_moments_follow_their_mean():
    check_mean("cpu")


def check_special(device):
    z = lambda *v: torch.tensor(v, dtype=torch.float32, device=device)  # noqa: E731
    # no gradient ever: nothing moves but by the weight decay
    p, g = z(1.0, -2.0), z(0.0, 0.0)
    m, v, s = ops.adamw_state8(p)
    ops.adamw_step([p], [g], [m], [v], step=1, lr=0.1, weight_decay=0.5, scales=[s])
    assert torch.equal(p.cpu(), torch.tensor([0.95, -1.9])) and not m.any() and not v.any() and not s.any()
    # gradients at the ends of fp32's range, and one that is not finite: that block, and no other, is lost
    p = torch.zeros(512, device=device)
    g = torch.full((512,), 1e-20, device=device)
    g[300] = float("inf")
    m, v, s = ops.adamw_state8(p)
    ops.adamw_step([p], [g], [m], [v], step=1, lr=0.1, scales=[s])
    assert torch.isfinite(p[:256]).all() and torch.isfinite(s[:, 0]).all() and s[:, 1].isnan().all()
    out = torch.empty_like(p), torch.empty_like(p)
    ops.adamw_read8([m], [v], [s], [out[0]], [out[1]])
    assert out[0][256:].isnan().all() and torch.isfinite(out[0][:256]).all()
    # moments below the smallest normal number: held or lost, never infinite
    for size in (1e-36, 1e-38, 1e-42, 1e-45):
        p, g = torch.zeros(300, device=device), torch.full((300,), size, device=device)
        m, v, s = ops.adamw_state8(p)
        for t in range(1, 4):
            ops.adamw_step([p], [g], [m], [v], step=t, lr=0.1, scales=[s])
        assert torch.isfinite(p).all() and torch.isfinite(s).all()
    # empty lists and empty tensors
    assert ops.adamw_step([], [], [], [], step=1, lr=0.1) == 0
    e = torch.empty(0, device=device)
    ops.adamw_step([e], [e.clone()], [e.clone()], [e.clone()], step=1, lr=0.1)
    # matrices whose elements lie in another order than their rows
    p = torch.randn(30, 20, device=device).t()
    g, m, v = (torch.rand(30, 20, device=device).t() for _ in range(3))
    want = plain.step(p.cpu(), g.cpu(), m.cpu(), v.cpu(), 5, 0.1, 0.9, 0.999, 1e-8, 0.01)
    ops.adamw_step([p], [g], [m], [v], step=5, lr=0.1)
    close_param(p, want[0], torch.ones(20, 30) * 4, torch.float32, 0.1)


def test_special_values():
    check_special("cpu")


def check_refusals(device):
    t = lambda n=8, d=torch.float32: torch.zeros(n, dtype=d, device=device)  # noqa: E731
    good = dict(step=1, lr=0.1)
    s8 = ops.adamw_state8(t())
    both = t(12)
    for args, more in [
        (([t()], [t()], [t()], []), good),                                               # lists of different lengths
        (([t()], [t(9)], [t()], [t()]), good),                                           # sizes
        (([t(8, torch.float64)], [t(8, torch.float64)], [t()], [t()]), good),            # types
        (([t(8, torch.bfloat16)], [t(8, torch.float16)], [t()], [t()]), good),
        (([t()], [t()], [t(8, torch.bfloat16)], [t(8, torch.bfloat16)]), good),
        (([t()], [t()], [s8[0]], [s8[1]]), good),                                        # codes without scales
        (([t()], [t()], [t()], [t()]), dict(good, scales=[s8[2]])),                      # scales without codes
        (([t()], [t()], [s8[0]], [s8[1]]), dict(good, scales=[torch.zeros(2, 2, device=device)])),
        (([t()], [t()], [t()], [t()]), dict(good, copies=[t()])),                        # a copy that is not bf16
        (([t(), t(8, torch.bfloat16)], [t(), t(8, torch.bfloat16)], [t(), t()], [t(), t()]), good),  # two kinds
        (([t(16)[::2]], [t()], [t()], [t()]), good),                                     # gaps
        (([both[:8]], [both[4:]], [t()], [t()]), good),                                  # a gradient inside its parameter
        (([both[:8], both[4:]], [t(), t()], [t(), t()], [t(), t()]), good),              # parameters that overlap
        (([t()], [t()], [t()], [t()]), dict(good, step=0)),
        (([t()], [t()], [t()], [t()]), dict(good, step=torch.tensor([1, 2], device=device))),
        (([t()], [t()], [t()], [t()]), dict(good, step=torch.tensor(1.0, device=device))),
        (([t()], [t()], [t()], [t()]), dict(good, lr=-1.0)),
        (([t()], [t()], [t()], [t()]), dict(good, lr=float("nan"))),
        (([t()], [t()], [t()], [t()]), dict(good, betas=(0.9, 1.0))),
        (([t()], [t()], [t()], [t()]), dict(good, eps=-1e-8)),
        (([t().to_sparse()], [t()], [t()], [t()]), good),
    ]:
        with pytest.raises(RuntimeError):
            ops.adamw_step(*args, **more)
    one = t()
    with pytest.raises(RuntimeError):  # the same tensor twice
        ops.adamw_step([one, one], [t(), t()], [t(), t()], [t(), t()], **good)
    with pytest.raises(RuntimeError):
        ops.adamw_read8([s8[0]], [s8[1]], [s8[2]], [t()], [t(8, torch.bfloat16)])
    with pytest.raises(RuntimeError):
        ops.adamw_read8([s8[0]], [s8[1]], [s8[2]], [t(9)], [t(9)])
    with pytest.raises(RuntimeError):
        ops.adamw_read8([s8[0]], [s8[1]], [s8[2]], [one], [one])


def test_refusals():
    check_refusals("cpu")


def check_unaligned32(device):
    """fp32 moments in tensors that start anywhere: all alike, so that whole vectors are found further on, and each elsewhere."""
    for offsets in ((1, 1, 1, 1, 1), (3, 3, 3, 3, 3), (2, 2, 2, 2, 0), (1, 2, 3, 0, 1)):
        for n in (1, 2, 3, 4, 5, 1023, 1024, 1025, 1027, 5000):
            ps, gs, ms, vs = tensors([n], (torch.float32, torch.float32), "cpu", seed=n)
            want = [x[0].clone().to(device) for x in (ps, gs, ms, vs)]
            got = [torch.full((n + 8,), 9.0, device=device)[o:o + n].copy_(x[0]) for o, x in zip(offsets, (ps, gs, ms, vs))]
            copies = [torch.zeros(n + 8, dtype=torch.bfloat16, device=device)[offsets[4]:offsets[4] + n], torch.zeros(n, dtype=torch.bfloat16, device=device)]
            for (p, g, m, v), c in ((got, copies[0]), (want, copies[1])):
                ops.adamw_step([p], [g], [m], [v], step=3, copies=[c], **HYPER)
            assert all(torch.equal(a, b) for a, b in zip(got + copies[:1], want + copies[1:]))
            for t, o in zip(got, offsets):  # what lies around them is as it was
                whole = torch.as_strided(t, (n + 8,), (1,), 0)
                assert (whole[:o] == 9).all() and (whole[o + n:] == 9).all()


def test_fp32_moments_that_start_anywhere():
    check_unaligned32("cpu")


def check_weight_decay(device):
    """A decay of a few steps of fp32 and less is taken as it is: the new parameter is off by its own rounding and the update's, no more."""
    n = 20000
    for lr, wd in ((1e-2, 0.1), (5e-5, 1e-2), (2e-5, 1e-2), (1e-6, 1e-2), (1e-3, 0.0)):
        for bits in (32, 8):
            g = torch.Generator().manual_seed(3)
            p, grad = torch.randn(n, generator=g), torch.randn(n, generator=g)
            if bits == 8:
                m, v, scales = ops.adamw_state8(p)
            else:
                m, v, scales = torch.zeros(n), torch.zeros(n), None
            want, _, _ = plain.step(p, grad, torch.zeros(n), torch.zeros(n), 1, lr, 0.9, 0.999, 1e-8, wd)
            q, m, v = (x.clone().to(device) for x in (p, m, v))
            ops.adamw_step([q], [grad.to(device)], [m], [v], step=1, lr=lr, weight_decay=wd, scales=None if scales is None else [scales.to(device)])
            step = 2.0 ** (want.abs().log2().floor() - 23)
            # the first step's update is lr: its factors, moments, root, division and sum, 16 roundings at most, or 2^-21 with the GPU's
            # approximate root and reciprocal; the decay's own factor and product
            assert ((q.cpu().double() - want).abs() <= step / 2 * (1 + 2.0 ** -10) + 2.0 ** -20 * lr + 4 * U * lr * wd * want.abs()).all()
            # infinite ones stay, next to others that are as they were
            inf = p.clone()
            inf[5::300], inf[7::300], inf[-1] = -float("inf"), float("inf"), -float("inf")
            r = inf.to(device)
            if bits == 8:
                m, v, scales = (x.to(device) for x in ops.adamw_state8(p))
            else:
                m, v = torch.zeros_like(r), torch.zeros_like(r)
            ops.adamw_step([r], [grad.to(device)], [m], [v], step=1, lr=lr, weight_decay=wd, scales=None if scales is None else [scales])
            assert torch.equal(r, torch.where(inf.isinf().to(device), inf.to(device), q))


def test_weight_decay_is_taken_as_it_is():
    check_weight_decay("cpu")


def check_versions(device):
    """A graph whose values a step has changed since is noticed."""
    p = torch.ones(4, device=device, requires_grad=True)
    y = (p * p).sum()
    m, v = torch.zeros(4, device=device), torch.zeros(4, device=device)
    ops.adamw_step([p], [torch.ones(4, device=device)], [m], [v], step=1, lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_graphs_notice_a_step():
    check_versions("cpu")


def check_versions_of_all_written(device):
    """Copies, which forward passes read and graphs keep, scales, and moments that are read back."""
    p = torch.randn(300, device=device).view(20, 15)
    m, v, scales = ops.adamw_state8(p)
    h = p.bfloat16()
    x = torch.randn(4, 15, device=device).bfloat16().requires_grad_()
    y = torch.nn.functional.linear(x, h)
    z = [torch.ones(2, 2, device=device, requires_grad=True) * s for s in (scales, scales[:, :1])]  # also through a view
    ops.adamw_step([p], [torch.ones_like(p)], [m], [v], scales=[scales], copies=[h], step=1, lr=0.1)
    outs = [torch.zeros_like(p) for _ in range(2)]
    w = [x.float().sum() * o for o in outs]
    ops.adamw_read8([m], [v], [scales], *([o] for o in outs))
    for used in (y, *z, *w):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            used.sum().backward()
    torch.nn.functional.linear(x, h).sum().backward()  # the next forward pass


def test_graphs_notice_all_that_is_written():
    check_versions_of_all_written("cpu")


def check_step_on_device(device):
    """A step's number in a tensor gives what the same number of the host gives, to the bit."""
    for bits in (32, 8):
        got = []
        for number in (17, torch.tensor([17], device=device)):
            ps, gs, ms, vs = tensors([300, 77], (torch.float32, torch.float32), device)
            more = {}
            if bits == 8:
                state = [ops.adamw_state8(p) for p in ps]
                ms, vs, ss = ([s[i] for s in state] for i in range(3))
                more = dict(scales=ss, seed=5)
            ops.adamw_step(ps, gs, ms, vs, step=number, **HYPER, **more)
            got.append(ps + ms + vs)
        assert all(torch.equal(a, b) for a, b in zip(*got))


def test_step_number_in_a_tensor():
    check_step_on_device("cpu")


# ---- the optimizer -------------------------------------------------------------------------------
def nets(device, steps=5, bits=32, cls=None, **more):
    """The same small network trained by torch's AdamW and by FlatAdamW, on parameters of their own."""
    torch.manual_seed(1)
    a = torch.nn.Sequential(torch.nn.Linear(9, 33), torch.nn.Tanh(), torch.nn.Linear(33, 3)).to(device)
    b = copy.deepcopy(a)
    groups = lambda m: [{"params": [m[0].weight, m[2].weight], "weight_decay": 0.1}, {"params": [m[0].bias, m[2].bias], "weight_decay": 0.0, "lr": 2e-2}]  # noqa: E731
    return a, torch.optim.AdamW(groups(a), lr=1e-2), b, P.FlatAdamW(groups(b), lr=1e-2, state_bits=bits, **more)


def train(model, opt, steps, seed=0, zero=True):
    g = torch.Generator().manual_seed(seed)
    dev = next(model.parameters()).device
    for s in range(steps):
        x, y = torch.randn(16, 9, generator=g).to(dev), torch.randn(16, 3, generator=g).to(dev)
        opt.zero_grad()
        torch.nn.functional.mse_loss(model(x), y).backward()
        opt.step()


def near(a, b, lr=2e-2, steps=5):
    """fp32 steps in another order of operations: each adds at most 16 half steps of an update of at most 10 lr, and one of the parameter; what
    that does to the next gradients is of the same size, here for a few steps."""
    for p, q in zip(a.parameters(), b.parameters()):
        assert ((p - q).abs() <= steps * steps * (10 * lr * 16 * U + 2 * U * p.abs())).all()


def test_flat_adamw_is_adamw():
    a, oa, b, ob = nets("cpu")
    train(a, oa, 5), train(b, ob, 5)
    near(a, b)
    m, v = ob.moments(b[0].weight)
    assert torch.allclose(m, oa.state[a[0].weight]["exp_avg"], rtol=1e-4, atol=1e-7)
    assert torch.allclose(v, oa.state[a[0].weight]["exp_avg_sq"], rtol=1e-4, atol=1e-9)


def test_each_parameter_counts_its_own_steps():
    p, q = (torch.nn.Parameter(torch.ones(4)) for _ in range(2))
    opt = P.FlatAdamW([p, q], lr=0.1, weight_decay=0.0)
    p.grad = torch.full((4,), 0.5)
    for _ in range(3):
        opt.step()
    q.grad = torch.full((4,), 2.0)  # takes part from the fourth step on: its first step is one of lr
    opt.step()
    assert opt.state[p]["step"] == 4 and opt.state[q]["step"] == 1
    assert torch.allclose(q, torch.full((4,), 0.9), atol=1e-6)


@pytest.mark.parametrize("bits", [32, 8])
def test_state_goes_through_a_checkpoint(bits):
    _, _, a, oa = nets("cpu", bits=bits, seed=9)
    train(a, oa, 3)
    saved_model, saved = copy.deepcopy(a.state_dict()), copy.deepcopy(oa.state_dict())
    train(a, oa, 3, seed=1)
    _, _, b, ob = nets("cpu", bits=bits, seed=9)
    b.load_state_dict(saved_model), ob.load_state_dict(saved)
    train(b, ob, 3, seed=1)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)
        assert all(torch.equal(x, y) for x, y in zip(oa.moments(p), ob.moments(q)))
    other = P.FlatAdamW([{"params": g["params"]} for g in ob.param_groups], state_bits=40 - bits)
    with pytest.raises(ValueError):
        other.load_state_dict(saved)


def test_gradients_and_parameters_of_any_layout():
    base = torch.randn(4, 6, 8)
    p = torch.nn.Parameter(base[:, ::2, :])  # gaps
    q = torch.nn.Parameter(torch.randn(6, 4).t())
    pc, qc = torch.nn.Parameter(p.detach().clone()), torch.nn.Parameter(q.detach().clone())
    flat, ref = P.FlatAdamW([p, q], lr=0.1), torch.optim.AdamW([pc, qc], lr=0.1)
    for _ in range(3):
        g, h = torch.randn(4, 3, 8), torch.randn(4, 6)
        p.grad, q.grad, pc.grad, qc.grad = g, h, g.clone(), h.clone()
        flat.step(), ref.step()
    assert torch.allclose(p, pc, atol=3e-6) and torch.allclose(q, qc, atol=3e-6)
    assert torch.equal(base[:, 1::2, :], base.clone()[:, 1::2, :])


def test_optimizer_refusals():
    p = [torch.nn.Parameter(torch.ones(3))]
    with pytest.raises(KeyError):
        P.FlatAdamW(p).moments(p[0])
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=16), dict(seed=-1)):
        with pytest.raises(ValueError):
            P.FlatAdamW(p, **bad)


def _wrapped(rank, world, bits, shadow):
    import bagua_core_b200.parallel as P
    from bagua_core_b200.models import MLP

    torch.manual_seed(7)
    model = MLP(16, 33, 5, depth=3)
    P.init_process_group(torch.device("cpu"))
    decay = [p for n, p in model.named_parameters() if not n.endswith("bias")]
    plain_ = [p for n, p in model.named_parameters() if n.endswith("bias")]
    opt = P.FlatAdamW([{"params": decay, "weight_decay": 0.1}, {"params": plain_, "weight_decay": 0.0, "lr": 2e-2}], lr=1e-2,
                      state_bits=bits, bf16_shadow=shadow)
    bm = P.with_bagua(model, [opt], P.GradientAllReduceAlgorithm(), bucket_bytes=4096)
    xs, ys = _batches(world)
    bs = xs.shape[1] // world
    states = []
    for s in range(6):
        if s == 2:
            opt.param_groups[0]["lr"] = 5e-3
        if s == 3:
            bm._reset()  # buckets are laid out again: the moments go along
        opt.zero_grad()
        torch.nn.functional.mse_loss(bm(xs[s, rank * bs:(rank + 1) * bs]), ys[s, rank * bs:(rank + 1) * bs]).backward()
        opt.step()
    states = opt.state_dict()
    flat = torch.cat([p.detach().reshape(-1) for p in model.parameters()])
    copies = [bool(torch.equal(p._bagua_bf16.view, p.detach().bfloat16())) for p in model.parameters()] if shadow else []
    steps = sorted({s["step"] for s in states["state"].values()})
    kinds = sorted({str(s["exp_avg"].dtype) for s in states["state"].values()})
    P.destroy_process_group()
    return flat, copies, steps, kinds


def _resumed(rank, world, bits):
    import bagua_core_b200.parallel as P
    from bagua_core_b200.models import MLP

    def make():
        torch.manual_seed(7)
        model = MLP(16, 33, 5, depth=3)
        return model, P.FlatAdamW(model.parameters(), lr=1e-2, state_bits=bits, seed=3)

    def wrap(model, opt):
        return P.with_bagua(model, [opt], P.GradientAllReduceAlgorithm(), bucket_bytes=4096)

    def run(bm, opt, steps):
        for s in steps:
            opt.zero_grad()
            torch.nn.functional.mse_loss(bm(xs[s, rank * bs:(rank + 1) * bs]), ys[s, rank * bs:(rank + 1) * bs]).backward()
            opt.step()

    P.init_process_group(torch.device("cpu"))
    xs, ys = _batches(world)
    bs = xs.shape[1] // world
    model, opt = make()
    bm = wrap(model, opt)
    run(bm, opt, range(3))
    saved = copy.deepcopy(model.state_dict()), copy.deepcopy(opt.state_dict())
    run(bm, opt, range(3, 6))
    out = []
    for m, o in ((model, opt), make(), make()):
        if m is not model:
            first = not out[1:]  # the state is loaded before the buckets are laid out, and after
            w = None if first else wrap(m, o)
            m.load_state_dict(saved[0])
            o.load_state_dict(saved[1])
            run(w or wrap(m, o), o, range(3, 6))
        out.append([p.detach().clone() for p in m.parameters()] + [x for p in m.parameters() for x in o.moments(p)])
    P.destroy_process_group()
    return out


@pytest.mark.parametrize("bits", [32, 8])
def test_training_goes_on_from_a_checkpoint(bits):
    from mp_util import run_ranks

    for a, b, c in run_ranks(_resumed, 2, args=(bits,)):
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and all(torch.equal(x, y) for x, y in zip(a, c))


def near_moments8(opt, p, m, v, decay=(1.0, 1.0), steps=1):
    """The moments of `p` are m and v, each rounded to the nearest code of its block, then `steps - 1` times to a neighbouring one: a code's
    distance is an eighth (first moment) or a sixteenth of its value, and 2^-9 or 2^-10 of the scale for the smallest."""
    state = opt.state[p]
    flat = lambda t: torch.empty_like(state["exp_avg"], dtype=torch.float64).copy_(t).as_strided((t.numel(),), (1,))  # noqa: E731
    for row, (got, old, part, least) in enumerate(zip(opt.moments(p), (m, v), (2.0 ** -3, 2.0 ** -4), (2.0 ** -9, 2.0 ** -10))):
        got, old = flat(got), flat(old)
        scale = plain.spread(state["scales"][row].cpu(), p.numel()).to(got.device)
        want = old * decay[row]
        bound = (steps - 0.5) * (1 + 1e-3) * torch.maximum(torch.maximum(old.abs(), want.abs()) * part * 1.2, scale * least)
        if row:
            bound = torch.maximum(bound, scale * least)  # held above zero
            assert (got > 0)[old > 0].all()
        assert ((got - want).abs() <= bound).all(), (row, float(((got - want).abs() / bound).max()))


def in_another_order(device):
    """A parameter with 8-bit moments of a few steps, and its values with the channels last: blocks of other elements, of other sizes."""
    torch.manual_seed(0)
    p = torch.nn.Parameter(torch.randn(40, 24, 3, 3, device=device))
    opt = P.FlatAdamW([p], state_bits=8)
    for _ in range(3):
        p.grad = torch.randn_like(p) * torch.rand(40, 1, 1, 1, device=device).mul(6).exp()
        opt.step()
    return p, opt, p.detach().clone().contiguous(memory_format=torch.channels_last)


def check_other_orders(device):
    p, opt, last = in_another_order(device)
    m, v = opt.moments(p)
    # a checkpoint of one order in a model of another, and back
    q = torch.nn.Parameter(last)
    other = P.FlatAdamW([q], state_bits=8)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert other.state[q]["exp_avg"].stride() == q.stride()
    near_moments8(other, q, m, v)
    m2, v2 = other.moments(q)
    opt.load_state_dict(other.state_dict())
    near_moments8(opt, p, m2, v2)
    # laid out anew between two steps
    m, v = opt.moments(p)
    p.data = last
    p.grad = torch.zeros_like(p)
    opt.step()
    near_moments8(opt, p, m, v, (0.9, 0.999), steps=2)
    # codes that say nothing of their order
    bad = copy.deepcopy(opt.state_dict())
    bad["state"][0]["exp_avg"] = torch.zeros(40, 24, 3, 6, dtype=torch.uint8, device=device)[..., ::2]
    with pytest.raises(ValueError, match="gaps"):
        opt.load_state_dict(bad)


def test_8_bit_moments_in_another_order():
    check_other_orders("cpu")


def _other_order_in_a_bucket(rank, world):
    import bagua_core_b200.parallel as P

    P.init_process_group(torch.device("cpu"))
    p, opt, last = in_another_order("cpu")
    m, v = opt.moments(p)
    model = torch.nn.Conv2d(24, 40, 3, bias=False)
    p.data, p.grad = last, None  # (a gradient has the parameter's layout)
    model.weight = p
    P.with_bagua(model, [opt], P.GradientAllReduceAlgorithm())
    attached = id(p) in opt._attached_ids and p.stride() == last.stride()
    near_moments8(opt, p, m, v)
    P.destroy_process_group()
    return attached


def test_8_bit_moments_in_another_order_go_into_a_bucket():
    from mp_util import run_ranks

    assert run_ranks(_other_order_in_a_bucket, 1)[0]


def _refused(rank, world):
    import bagua_core_b200.parallel as P
    from bagua_core_b200.models import MLP

    P.init_process_group(torch.device("cpu"))
    out = []
    for bits in (8, 32):
        torch.manual_seed(7)
        model, loose = MLP(16, 33, 5, depth=2), torch.nn.Parameter(torch.randn(300))
        opt = P.FlatAdamW([*model.parameters(), loose], lr=1e-2, state_bits=bits)
        bm = P.with_bagua(model, [opt], P.GradientAllReduceAlgorithm(), bucket_bytes=4096)

        def run(steps):
            for s in range(steps):
                opt.zero_grad()
                torch.nn.functional.mse_loss(bm(torch.randn(4, 16)), torch.randn(4, 5)).backward()
                loose.grad = torch.randn(300)
                opt.step()

        run(3)
        good = copy.deepcopy(opt.state_dict())
        run(2)
        now = copy.deepcopy(opt.state_dict())
        wrong = []
        for _ in range(7):
            w = copy.deepcopy(good)
            w["param_groups"][0]["lr"] = 7.0
            wrong.append(w)
        last = max(good["state"])  # the loose one; the flat ones in front of it fit
        other = {"step": 1, "exp_avg": torch.zeros(300), "exp_avg_sq": torch.zeros(300)}
        wrong[0]["state"][last] = other if bits == 8 else {**other, "scales": torch.zeros(2, 2)}
        wrong[1]["state"][last]["exp_avg"] = wrong[1]["state"][last]["exp_avg"][:-1]
        wrong[2]["state"][last]["exp_avg_sq"] = wrong[2]["state"][last]["exp_avg_sq"].double()
        wrong[3]["state"][last]["step"] = -1
        del wrong[4]["state"][0]["exp_avg"]
        wrong[5]["param_groups"].append(wrong[5]["param_groups"][0])
        del wrong[6]["state"]
        for w in wrong:
            with pytest.raises((ValueError, KeyError)):
                opt.load_state_dict(w)
            got = opt.state_dict()
            same = got["param_groups"] == now["param_groups"] and got["state"].keys() == now["state"].keys()
            for k, st in got["state"].items():
                same = same and all(torch.equal(torch.as_tensor(x), torch.as_tensor(now["state"][k][n])) for n, x in st.items())
            out.append(same)
        # hooks see, and may adapt, what is loaded
        seen = []
        hooks = [opt.register_load_state_dict_pre_hook(lambda o, d: {**d, "state": {k: dict(v, step=v["step"] + 10) for k, v in d["state"].items()}}),
                 opt.register_load_state_dict_post_hook(lambda o: seen.append(sorted(s["step"] for s in o.state.values())))]
        opt.load_state_dict(good)
        out.append(seen[0] == [13] * len(good["state"]) and sorted(s["step"] for s in opt.state_dict()["state"].values()) == seen[0])
        for h in hooks:
            h.remove()
        run(1)
        out.append(sorted({s["step"] for s in opt.state_dict()["state"].values()}) == [14])
    P.destroy_process_group()
    return out


def test_a_refused_checkpoint_changes_nothing():
    from mp_util import run_ranks

    assert all(run_ranks(_refused, 1)[0])


def _decentralized(rank, world):
    import bagua_core_b200.parallel as P
    from bagua_core_b200.models import MLP

    torch.manual_seed(7)
    model = MLP(16, 33, 5, depth=3)
    P.init_process_group(torch.device("cpu"))
    opt = P.FlatAdamW(model.parameters(), lr=1e-2, state_bits=8)
    bm = P.with_bagua(model, [opt], P.DecentralizedAlgorithm(peer_selection_mode="all"), bucket_bytes=4096)
    xs, ys = _batches(world)
    bs = xs.shape[1] // world
    before = torch.cat([p.detach().reshape(-1) for p in model.parameters()])
    for s in range(3):
        opt.zero_grad()
        torch.nn.functional.mse_loss(bm(xs[s, rank * bs:(rank + 1) * bs]), ys[s, rank * bs:(rank + 1) * bs]).backward()
        opt.step()
    after = torch.cat([p.detach().reshape(-1) for p in model.parameters()])
    P.destroy_process_group()
    return before, after, len(opt._flat)


def test_flat_adamw_on_buckets_of_weights():
    from mp_util import run_ranks

    for before, after, flat in run_ranks(_decentralized, 2):
        assert flat > 1 and torch.isfinite(after).all()
        # three steps of about lr each, none of more than ten times that
        assert 1e-3 < (after - before).abs().max() <= 3 * 10 * 1e-2


def _batches(world):
    g = torch.Generator().manual_seed(5)
    return torch.randn(6, 4 * world, 16, generator=g), torch.randn(6, 4 * world, 5, generator=g)


@pytest.mark.parametrize("bits,shadow", [(32, True), (8, False)])
def test_flat_adamw_on_buckets(bits, shadow):
    from bagua_core_b200.models import MLP
    from mp_util import run_ranks

    res = run_ranks(_wrapped, 2, args=(bits, shadow))
    assert torch.equal(res[0][0], res[1][0])
    assert all(res[0][1]) and res[0][2] == [6] and res[0][3] == ["torch.float32" if bits == 32 else "torch.uint8"]
    torch.manual_seed(7)
    model = MLP(16, 33, 5, depth=3)
    decay = [p for n, p in model.named_parameters() if not n.endswith("bias")]
    plain_ = [p for n, p in model.named_parameters() if n.endswith("bias")]
    opt = torch.optim.AdamW([{"params": decay, "weight_decay": 0.1}, {"params": plain_, "weight_decay": 0.0, "lr": 2e-2}], lr=1e-2)
    xs, ys = _batches(2)
    for s in range(6):
        if s == 2:
            opt.param_groups[0]["lr"] = 5e-3
        opt.zero_grad()
        torch.nn.functional.mse_loss(model(xs[s]), ys[s]).backward()
        opt.step()
    want = torch.cat([p.detach().reshape(-1) for p in model.parameters()])
    if bits == 32:
        assert torch.allclose(res[0][0], want, atol=2e-5)  # 6 steps of at most 2e-2, gradients averaged in another order
    else:
        # rounded moments: an update is off by less than an eighth and a thirty-second of itself at each of 6 steps of about lr
        assert ((res[0][0] - want).abs() <= 6 * 2e-2).all() and (res[0][0] - want).abs().mean() <= 6 * 1e-2 * (1 / 8 + 1 / 32)


def _device_counted(rank, world, bits):
    import bagua_core_b200.parallel as P
    from bagua_core_b200.models import MLP

    P.init_process_group(torch.device("cpu"))
    xs, ys = _batches(world)
    bs = xs.shape[1] // world
    out = []
    for capturable in (False, True):
        torch.manual_seed(7)
        model = MLP(16, 33, 5, depth=3)
        opt = P.FlatAdamW(model.parameters(), lr=1e-2, state_bits=bits, seed=3, capturable=capturable)
        bm = P.with_bagua(model, [opt], P.GradientAllReduceAlgorithm(), bucket_bytes=4096)
        for s in range(5):
            if s == 2:
                bm._reset()
            if s == 3:  # parameters that differ in their numbers of steps
                state = copy.deepcopy(opt.state_dict())
                state["state"][0]["step"] = 1
                opt.load_state_dict(state)
            opt.zero_grad()
            torch.nn.functional.mse_loss(bm(xs[s, rank * bs:(rank + 1) * bs]), ys[s, rank * bs:(rank + 1) * bs]).backward()
            opt.step()
        steps = [s["step"] for s in opt.state_dict()["state"].values()]
        out.append([p.detach().clone() for p in model.parameters()] + [x for p in model.parameters() for x in opt.moments(p)] + [torch.tensor(steps)])
    P.destroy_process_group()
    return out


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_counted_on_the_device(bits):
    """Counting them there changes nothing, also behind a new layout and a loaded state."""
    from mp_util import run_ranks

    for a, b in run_ranks(_device_counted, 2, args=(bits,)):
        assert a[-1].tolist() == [3] + [5] * (len(a[-1]) - 1)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("which", range(4))
def test_negated_views_are_refused(which):
    """The memory of a lazily negated view holds the opposites of its values."""
    parts = [[torch._neg_view(torch.ones(8)) if k == which else torch.ones(8)] for k in range(4)]
    assert parts[which][0].is_neg()
    with pytest.raises(RuntimeError, match="negated views"):
        ops.adamw_step(*parts, step=1, lr=0.1)


def check_codes(device, dtypes, n):
    """Two steps give, to the bit, the codes and scales that the definition in 64 bits gives.  fp32 alone would round one code in some
    800,000 the other way (100 of 80 million, counted).  Left out are first moments that are the difference of larger terms: what fp32 leaves of those is not bounded."""
    (p,), (g,), _, _ = tensors([n], dtypes, "cpu", seed=1)
    b1, b2 = HYPER["betas"]
    p, g = p.to(device), g.to(device)
    m, v, s = ops.adamw_state8(p)
    exact = []
    for t in (1, 2):
        m0, v0 = plain.read(m, v, s)
        _, first, second = plain.step(p.cpu(), g.cpu(), m0, v0, t, HYPER["lr"], b1, b2, HYPER["eps"], HYPER["weight_decay"])
        ops.adamw_step([p], [g], [m], [v], step=t, scales=[s], seed=9, **HYPER)
        random = plain.random_bits(9, t, 0, n)
        for x, row, largest, table, u, code in ((first, 0, 480, plain.FIRST, random & 0xFFFF, m), (second, 1, 496, plain.SECOND, random >> 16, v)):
            scale = plain.tops(x).float() * torch.tensor(1 / largest)  # in fp32 (and of normal size here)
            assert ((s[row].cpu() - scale).abs() <= 6 * U * scale).all()
            want, same = plain.codes(x, plain.spread(scale, n), table, (u.double() + 0.5) / 65536, 0)
            assert torch.equal(want, same)
            got = code.cpu().long() & (127 if row == 0 else 255)
            # (a second moment above zero has a code above zero)
            wrong = got != (want if row == 0 else want.clamp(min=1))
            if row == 0:
                wrong &= (b1 * m0).abs() + (1 - b1) * g.cpu().double().abs() <= 1.001 * x.abs()
            exact.append(int(wrong.sum()))
        g = g * 0.75 + g.roll(1) * 0.5
    assert exact == [0, 0, 0, 0]


@pytest.mark.parametrize("dtypes", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)])
def test_codes_are_those_of_64_bits(dtypes):
    check_codes("cpu", dtypes, 3_000_001)
