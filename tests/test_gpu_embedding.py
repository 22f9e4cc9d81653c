"""The lookup and gradient kernels (`csrc/kernels/embedding.cu`) against the definition in 64 bits."""
import pytest
import torch

import bagua_core_b200.ops as ops
import test_cpu_embedding as host
from bagua_core_b200 import _native
from bagua_core_b200.ops import wgrad

pytestmark = pytest.mark.gpu
TYPES = host.TYPES


@pytest.fixture(autouse=True)
def in_place_off():
    before, wgrad.enabled = wgrad.enabled, False
    yield
    wgrad.enabled = before


@pytest.mark.parametrize("table_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H", [8, 13, 256])
def test_types(table_type, out_type, H):
    host.check("cuda", 700, 90, H, TYPES[table_type], TYPES[out_type])


# rows around the ends of a digit, tokens around those of a tile, a chunk and a block
@pytest.mark.parametrize("n,rows", [(1, 1), (1, 300), (31, 7), (32, 255), (33, 256), (1023, 257), (1024, 65535), (1025, 65536), (2048, 65537),
                                    (2049, 3), (8192, 1), (8193, 1000), (12288, 30522), (65536, 5000), (65537, 511), (131072, 4001), (131073, 70000), (150001, 20000)])
@pytest.mark.parametrize("how", ["any", "few", "one", "ordered"])
def test_tokens_and_rows(n, rows, how):
    host.check("cuda", n, rows, 16, how=how)


@pytest.mark.parametrize("H", [1, 7, 8, 63, 64, 65, 72, 128, 129, 136, 255, 264, 1024, 2056, 5000])
@pytest.mark.parametrize("out_type", ["f32", "bf16"])
def test_widths(H, out_type):
    host.check("cuda", 3001, 77, H, TYPES["f32"], TYPES[out_type], how="few")


def test_more_rows_than_two_digits_count():
    host.check("cuda", 5000, 1 << 24, 1, TYPES["bf16"])
    host.check("cuda", 70000, 70000 * 3, 8, TYPES["bf16"])


@pytest.mark.parametrize("n", [500, 9000, 70000])
def test_padding_and_narrow_ids(n):
    host.check("cuda", n, 40, 16, padding=20, how="one")     # nothing but padding
    host.check("cuda", n, 40, 16, padding=0, how="few", ids_type=torch.int32)
    host.check("cuda", n, 40, 16, padding=-1)


def test_tables_of_any_stride_and_alignment():
    host.check("cuda", 500, 30, 16, make=lambda w: torch.zeros(30, 40, device="cuda")[:, 3:19].copy_(w))
    host.check("cuda", 500, 30, 16, make=lambda w: torch.zeros(481, device="cuda")[1:].view(30, 16).copy_(w))
    host.check("cuda", 500, 30, 16, make=lambda w: torch.zeros(16, 30, device="cuda").t().copy_(w))
    host.check_shapes("cuda")


def test_same_bits_every_time():
    a = host.check("cuda", 40001, 259, 333, TYPES["f16"], how="few")
    b = host.check("cuda", 40001, 259, 333, TYPES["f16"], how="few")
    assert torch.equal(a, b)


def test_refusals_orders_and_module():
    host.check_refusals("cuda")
    host.check_second_order("cuda")
    host.check_module("cuda")


@pytest.mark.parametrize("n", [100, 10000, 70000])
def test_ids_outside_the_table(n):
    w = torch.randn(50, 16, device="cuda", requires_grad=True)
    ids = torch.randint(0, 50, (n,), device="cuda")
    bad = ids.clone()
    bad[3], bad[n // 2], bad[n - 1] = -1, 50, 1 << 40
    y = ops.embedding(bad, w)
    torch.cuda.synchronize()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[[3, n // 2, n - 1]] = False
    assert y[~keep].isnan().all() and torch.equal(y[keep], w[ids[keep]])
    with pytest.raises(RuntimeError, match="not in the table"):
        ops.embedding(ids, w)
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))  # the error was told: the gradient goes without them
    assert torch.equal(g, torch.bincount(ids[keep], minlength=50)[:, None].float().expand(50, 16))
    torch.cuda.synchronize()
    ops.embedding(ids, w)


@pytest.mark.parametrize("n", [300, 20000, 140000])
def test_added_to_the_gradient_in_place(n):
    """With `wgrad.enabled` the rows that occur are added to `.grad`; the others are not touched."""
    wgrad.enabled = True
    w = torch.nn.Parameter(torch.randn(1000, 24, device="cuda"))
    w.grad = torch.randn(1000, 24, device="cuda")
    before, grad = w.grad.clone(), w.grad
    ids = host.tokens(n, 500, "few").cuda()
    dout = torch.randn(n, 24, device="cuda").bfloat16()
    ops.embedding(ids, w, scale=2.0, padding_idx=1, dtype=torch.bfloat16).backward(dout)
    assert w.grad is grad
    sums, size = (torch.zeros(1000, 24, dtype=torch.float64, device="cuda").index_add_(0, ids, 2 * x) for x in (dout.double(), dout.double().abs()))
    count = torch.bincount(ids, minlength=1000)[:, None]
    sums[1] = size[1] = 0
    assert ((grad.double() - before.double() - sums).abs() <= host.U * ((count + 2) * size + 2 * (before.abs() + sums.abs()))).all()
    untouched = count[:, 0] == 0
    assert torch.equal(grad[untouched], before[untouched]) and torch.equal(grad[1], before[1])
    # a second use of the table in the graph: autograd adds the two first
    w.grad = None
    (ops.embedding(ids, w).sum() + ops.embedding(ids, w).sum()).backward()
    assert torch.equal(w.grad, 2 * count.float().expand(1000, 24))


def test_contexts_of_few_sms():
    """Green contexts run smaller clusters, or none of this size: fewer blocks sort, or the tokens go through memory."""
    green = pytest.importorskip("torch.cuda.green_contexts")
    torch.cuda.synchronize()
    try:
        contexts = [green.GreenContext.create(sms, 0) for sms in (8, 16, 32)]
    except RuntimeError as e:
        pytest.skip(str(e))
    for context in contexts:
        context.set_context()
        try:
            for n in (100, 5000, 40000, 70000, 131072):
                host.check("cuda", n, 3000, 16, how="few")
            torch.cuda.synchronize()
        finally:
            context.pop_context()
    host.check("cuda", 40000, 3000, 16, how="few")


def test_captured_and_replayed_beside_another_stream():
    """Two captured passes hold scratch of their own; replays on two streams at once give what eager calls give."""
    cases = []
    for k in range(2):
        w = torch.randn(3000, 64, device="cuda", requires_grad=True)
        ids = torch.randint(0, 3000, (20000,), device="cuda")
        dout = torch.randn(20000, 64, device="cuda")
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(ops.embedding(ids, w), w, dout)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y = ops.embedding(ids, w)
            (g,) = torch.autograd.grad(y, w, dout)
        cases.append((w, ids, dout, graph, y, g, side))
    for _ in range(3):
        for w, ids, dout, graph, y, g, side in cases:
            ids.copy_(torch.randint(0, 3000, (20000,), device="cuda"))
        torch.cuda.synchronize()
        for *_, graph, y, g, side in cases:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for w, ids, dout, graph, y, g, side in cases:
            want = ops.embedding(ids, w)
            assert torch.equal(y, want) and torch.equal(g, torch.autograd.grad(want, w, dout)[0])


def test_offsets_beyond_32_bits():
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    rows, H = (1 << 21) + 3, 1032  # the last rows start behind element 2^31
    w = torch.zeros(rows, H, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    with torch.no_grad():
        w[-2:] = torch.randn(2, H, device="cuda")
    ids = torch.tensor([rows - 1, rows - 2, 0, rows - 1], device="cuda")
    y = ops.embedding(ids, w)
    assert torch.equal(y, w.detach()[ids])
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert g[-1].eq(2).all() and g[-2].eq(1).all() and g[0].eq(1).all() and not g[1:-2].any()
    del g, w, y
    n = (1 << 21) + 5  # and outputs
    w = torch.randn(100, H, device="cuda").bfloat16().requires_grad_()
    ids = torch.arange(n, device="cuda") % 100
    y = ops.embedding(ids, w)
    assert torch.equal(y[-300:], w.detach()[ids[-300:]])
    (g,) = torch.autograd.grad(y, w, torch.ones_like(y))
    assert torch.equal(g, torch.bincount(ids, minlength=100)[:, None].float().expand(100, H).bfloat16())


def test_negated_views():
    """Lazily negated views, as the imaginary part of a conjugate is one: the table, and the gradient that comes back."""
    g = torch.Generator().manual_seed(0)
    z = torch.randn(9, 40, dtype=torch.complex64, generator=g).cuda()
    table, ids = z.conj().imag, torch.tensor([3, 0, 3, 8], device="cuda")
    assert table.is_neg()
    assert torch.equal(ops.embedding(ids, table), -z.imag[ids])
    w = torch.randn(9, 40, generator=g).cuda().requires_grad_()
    d = torch.randn(4, 40, dtype=torch.complex64, generator=g).cuda()
    ops.embedding(ids, w).backward(d.conj().imag)
    want = torch.zeros(9, 40, device="cuda", dtype=torch.float64).index_add_(0, ids, -d.imag.double())
    assert torch.equal(w.grad, want.float())  # sums of two values at most, rounded once
