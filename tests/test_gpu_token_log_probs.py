"""The log-probability kernels (`csrc/kernels/token_log_probs.cu`) against the definition in 64 bits."""
import math

import pytest
import torch

import bagua_core_b200.ops as ops
import test_cpu_token_log_probs as host

pytestmark = pytest.mark.gpu
INF = float("inf")


def check(n, vocab, dtype, top=0, masked=0.0, ignored=0.0, seed=0, **more):
    x, t = host.logits(n, vocab, dtype, seed, masked=masked)
    if ignored:
        t[torch.rand(n, generator=torch.Generator().manual_seed(seed)) < ignored] = -100
    return host.check(x.cuda(), t, top, **more)


# around a vector, a warp's and a block's share, where a warp ends and a block begins, and where rows are split
@pytest.mark.parametrize("vocab", [1, 2, 5, 7, 8, 9, 31, 32, 33, 255, 256, 257, 1000, 1023, 1024, 1025, 1031, 2048, 2049, 4099, 8192, 30522])
@pytest.mark.parametrize("dtype", host.TYPES.values())
def test_vocabularies(vocab, dtype):
    check(5, vocab, dtype, top=min(vocab, 5))
    check(13, vocab, dtype, top=min(vocab, 32), masked=0.4, ignored=0.2)


@pytest.mark.parametrize("n", [1, 2, 36, 37, 38, 74, 147, 148, 149, 296, 300, 1000])
@pytest.mark.parametrize("vocab", [5001, 16384])
def test_rows(n, vocab):
    check(n, vocab, torch.bfloat16, top=4)
    check(n, vocab, torch.float32)


@pytest.mark.parametrize("n", [1, 3, 200])
def test_wide_vocabulary(n):
    check(n, 131075, torch.bfloat16, top=20)
    check(n, 200000, torch.float16, top=1)


@pytest.mark.parametrize("top", [1, 2, 31, 32])
def test_alternatives_in_every_order(top):
    """Values that rise, fall or are all equal along the row, in steps that types share: ties go to the lowest id."""
    n = 70000
    ramp = (torch.arange(n) // 64).float()
    rows = torch.stack([ramp, -ramp, torch.zeros(n), (torch.arange(n) * 7919 % 1009).float(), torch.where(torch.arange(n) % 5 == 0, -INF, 1.0),
                        torch.where(torch.arange(n) < 3, 1.0, -INF)])
    for dtype in host.TYPES.values():
        for width in (n, 1000):
            x = rows[:, :width].clamp(-1000, 1000).to(dtype).cuda()
            host.check(x, torch.tensor([0, 1, 2, 3, 4, 0]), top, backward=False)


@pytest.mark.parametrize("vocab", [5000, 30522, 131072])
@pytest.mark.parametrize("left", [1, 19, 300, 1200])
def test_alternatives_of_few_neighbouring_tokens(vocab, left):
    """Rows of which a mask leaves tokens that are neighbours: the threads of a few warps hold them all."""
    g = torch.Generator().manual_seed(left)
    for n in (1, 3, 700 if vocab < 10000 else 40):
        x = torch.full((n, vocab), -INF)
        first = torch.randint(0, vocab - left, (n,), generator=g)
        for i in range(n):
            x[i, first[i]:first[i] + left] = torch.randn(left, generator=g)
        host.check(x.bfloat16().cuda(), first + left // 2, 20, backward=False)


def test_special_rows():
    host.check_special("cuda")


def test_ends_of_the_range():
    host.check_ends_of_the_range("cuda")


def test_layouts():
    host.check_layouts("cuda")


@pytest.mark.parametrize("lead", range(1, 8))
def test_rows_that_start_anywhere(lead):
    for dtype in host.TYPES.values():
        for vocab in (200, 5000):
            x, t = host.logits(9, vocab, dtype)
            host.check(x.cuda(), t, 3, make=lambda x: torch.zeros(9 * (vocab + lead) + lead, dtype=dtype, device="cuda")[lead:].view(9, -1)[:, :vocab].copy_(x))


def test_gradients_and_refusals():
    host.check_partial_gradients("cuda")
    host.check_second_order("cuda")
    host.check_refusals("cuda")


def test_scaled_entropy_gradients():
    host.check_scaled_entropy_gradients("cuda")


@pytest.mark.parametrize("vocab,rows", [(40, 6), (1000, 6), (3000, 6), (9001, 1), (30522, 6)])
def test_large_logits(vocab, rows):
    host.check_large_logits("cuda", (vocab,), rows)


def test_large_alternatives():
    host.check_large_alternatives("cuda")


@pytest.mark.parametrize("unknown", [False, True])
def test_kept_graphs(unknown):
    host.check_kept_graphs("cuda", unknown)


def test_targets_outside_the_vocabulary():
    x = torch.randn(4, 3000, device="cuda", requires_grad=True)
    t = torch.tensor([5, -1, 3000, 7], device="cuda")
    r = ops.token_log_probs(x, t, 2)
    torch.cuda.synchronize()
    assert r.log_probs[1:3].isnan().all() and torch.isfinite(r.log_probs[[0, 3]]).all() and torch.isfinite(r.entropy).all()
    with pytest.raises(RuntimeError, match="not in the vocabulary"):
        ops.token_log_probs(x, t.clamp(0, 2999))
    (d,) = torch.autograd.grad(r.log_probs[[0, 3]].sum(), x)
    assert not d[1:3].any() and d[0].any()
    ops.token_log_probs(x, t.clamp(0, 2999))


def test_gradients_that_are_not_contiguous():
    x, t = host.logits(64, 5000, torch.bfloat16)
    y = x.cuda().requires_grad_()
    u = t.cuda()
    (want,) = torch.autograd.grad(ops.token_log_probs(y, u).log_probs, y, torch.arange(64.0, device="cuda"))
    (got,) = torch.autograd.grad(ops.token_log_probs(y, u).log_probs, y, torch.arange(128.0, device="cuda").view(64, 2)[:, 0] / 2)
    assert torch.equal(got, want)
    (a,) = torch.autograd.grad(ops.token_log_probs(y, u).log_probs, y, torch.ones((), device="cuda").expand(64))
    (b,) = torch.autograd.grad(ops.token_log_probs(y, u).log_probs, y, torch.ones(64, device="cuda"))
    assert torch.equal(a, b)
    z = x.cuda().view(8, 8, 5000).requires_grad_()
    (c,) = torch.autograd.grad(ops.token_log_probs(z, u.view(8, 8)).log_probs, z, torch.arange(64.0, device="cuda").view(8, 8).t().contiguous().t())
    assert torch.equal(c.view(64, 5000), want)


def test_contexts_of_few_sms():
    """Green contexts may run smaller clusters: a row is split over fewer blocks."""
    green = pytest.importorskip("torch.cuda.green_contexts")
    torch.cuda.synchronize()
    try:
        contexts = [green.GreenContext.create(sms, 0) for sms in (8, 16)]
    except RuntimeError as e:
        pytest.skip(str(e))
    for context in contexts:
        context.set_context()
        try:
            for n in (1, 40):
                check(n, 30522, torch.bfloat16, top=9)
                check(n, 131072, torch.float32, top=32)
            torch.cuda.synchronize()
        finally:
            context.pop_context()


def test_changed_logits_are_noticed():
    x = torch.randn(3, 5000, device="cuda", requires_grad=True)
    y = x * 2
    r = ops.token_log_probs(y[:, :4999], torch.zeros(3, dtype=torch.int64, device="cuda"))
    y.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.log_probs.sum().backward()


def test_captured_and_replayed_beside_another_stream():
    cases = []
    for n in (3, 400):
        x = torch.randn(n, 9000, device="cuda").bfloat16().requires_grad_()
        t = torch.randint(0, 9000, (n,), device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(ops.token_log_probs(x, t, 5).log_probs.sum(), x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            r = ops.token_log_probs(x, t, 5)
            (d,) = torch.autograd.grad(r.log_probs.sum() + r.entropy.sum(), x)
        cases.append((x, t, graph, r, d, side))
    for _ in range(3):
        for x, t, *_ in cases:
            with torch.no_grad():
                x.copy_(torch.randn_like(x))
            t.copy_(torch.randint_like(t, 0, 9000))
        torch.cuda.synchronize()
        for x, t, graph, r, d, side in cases:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for x, t, graph, r, d, side in cases:
            want = ops.token_log_probs(x, t, 5)
            (e,) = torch.autograd.grad(want.log_probs.sum() + want.entropy.sum(), x)
            assert all(torch.equal(p, q) for p, q in zip(r, want)) and torch.equal(d, e)


def test_offsets_beyond_32_bits():
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    n, vocab = 33000, 131072  # 4.3e9 logits
    x = torch.zeros(n, vocab, dtype=torch.bfloat16, device="cuda")
    x[-2:] = torch.randn(2, vocab, device="cuda") * 3
    t = torch.full((n,), -100, device="cuda")
    t[-2:] = torch.tensor([5, vocab - 1], device="cuda")
    t[0] = 9
    y = x.requires_grad_()
    r = ops.token_log_probs(y, t, 3)
    want = ops.token_log_probs(x[-2:].detach().clone(), t[-2:], 3)
    # two rows are split over blocks and sum in another order: each is off by at most (check())
    off = 2 * (2.0 ** -22 + (vocab / 256 + 64 + 2 ** 8) * host.U) * 16
    assert all(((p[-2:] - q).abs() <= off).all() for p, q in zip(r[:3], want[:3])) and torch.equal(r.top_ids[-2:], want.top_ids)
    assert abs(float(r.log_probs[0].detach()) + math.log(vocab)) < 1e-5
    (d,) = torch.autograd.grad(r.log_probs.sum(), y)
    z = x[-2:].detach().clone().requires_grad_()
    (e,) = torch.autograd.grad(ops.token_log_probs(z, t[-2:]).log_probs.sum(), z)
    assert ((d[-2:].double() - e.double()).abs() <= off + 2.0 ** -7 * e.double().abs()).all() and not d[1:-2].any() and d[0, 9] > 0.9


def test_negated_views():
    """Lazily negated views, as the imaginary part of a conjugate is one, are the values that they stand for."""
    g = torch.Generator().manual_seed(0)
    z = torch.randn(5, 333, dtype=torch.complex64, generator=g).cuda()
    d = torch.randn(5, dtype=torch.complex64, generator=g).cuda()
    t = torch.randint(0, 333, (5,), generator=g).cuda()
    x, d = z.conj().imag, d.conj().imag
    assert x.is_neg() and d.is_neg()
    got = []
    for logits, dy in ((x, d), (x.resolve_neg(), d.resolve_neg())):
        logits = logits.detach().requires_grad_()
        r = ops.token_log_probs(logits, t, top=3)
        r[0].backward(dy)
        got.append([*r, logits.grad])
    assert all(torch.equal(a, b) for a, b in zip(*got))
