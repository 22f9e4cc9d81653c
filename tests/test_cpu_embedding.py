"""Rows looked up by token (`ops.embedding`, `ops.ScaledEmbedding`) and the table's gradient, against their definition in 64 bits, on
the host.  The GPU runs the same checks (`test_gpu_embedding.py`)."""
import pytest
import torch

import bagua_core_b200.ops as ops

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # half a step of fp32


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tokens(n, rows, how, seed=0):
    g = torch.Generator().manual_seed(seed)
    if how == "one":  # all the same
        return torch.full((n,), rows // 2, dtype=torch.int64)
    if how == "few":  # some very often
        return (torch.rand(n, generator=g) ** 6 * rows).long().clamp_(max=rows - 1)
    if how == "ordered":
        return (torch.arange(n) * rows // max(n, 1)).clamp_(max=rows - 1)
    return torch.randint(0, rows, (n,), generator=g)


def check(device, n, rows, H, table_type=torch.float32, out_type=None, scale=0.75, padding=None, how="any", ids_type=torch.int64, make=None,
          seed=0):
    g = torch.Generator().manual_seed(seed + 1)
    ids = tokens(n, rows, how, seed).to(ids_type)
    table = torch.randn(rows, H, generator=g).to(table_type)
    w = table.to(device)
    if make is not None:
        w = make(w)
    w.requires_grad_()
    y = ops.embedding(ids.to(device), w, scale=scale, padding_idx=padding, dtype=out_type)
    out_type = out_type or table_type
    assert y.shape == (n, H) and y.dtype == out_type
    want = table[ids.long()].double() * scale
    assert ((y.detach().cpu().double() - want).abs() <= (half(out_type) + U) * want.abs() + torch.finfo(out_type).smallest_normal * half(out_type)).all()
    dout = torch.randn(n, H, generator=g).to(out_type)
    (got,) = torch.autograd.grad(y, w, dout.to(device))
    assert got.shape == (rows, H) and got.dtype == table_type
    sums, size = (torch.zeros(rows, H, dtype=torch.float64).index_add_(0, ids.long(), x) for x in (dout.double(), dout.double().abs()))
    count = torch.bincount(ids.long(), minlength=rows)[:, None]
    if padding is not None:
        sums[padding] = 0
        size[padding] = 0
    sums, size = sums * scale, size * abs(scale)
    # a sum of k terms in any order: at most k - 1 roundings of partial sums; the scale, its product, the rounding to the table's type
    bound = (count + 2) * U * size + half(table_type) * (sums.abs() + (count + 2) * U * size) + torch.finfo(table_type).smallest_normal * half(table_type)
    assert ((got.cpu().double() - sums).abs() <= bound).all()
    absent = count[:, 0] == 0
    assert not got.cpu()[absent].any()
    return got


@pytest.mark.parametrize("table_type,out_type", [("f32", None), ("f32", "bf16"), ("bf16", None), ("f16", "f32"), ("f16", None)])
def test_lookup_and_gradient(table_type, out_type):
    check("cpu", 200, 50, 24, TYPES[table_type], TYPES[out_type] if out_type else None)


def test_padding_and_id_types():
    check("cpu", 100, 20, 8, padding=3)
    check("cpu", 100, 20, 8, padding=-1, ids_type=torch.int32)
    check("cpu", 1, 1, 1)


def check_shapes(device):
    w = torch.randn(7, 4, device=device, requires_grad=True)
    for shape in ((), (0,), (3, 0, 2), (2, 3), (1, 2, 1)):
        ids = torch.ones(shape, dtype=torch.int64, device=device)
        y = ops.embedding(ids, w)
        assert y.shape == (*shape, 4)
        (g,) = torch.autograd.grad(y.sum(), w)
        assert g.shape == w.shape and float(g.sum()) == 4 * ids.numel()
    # ids and tables that are not contiguous
    ids = torch.arange(12, device=device).view(3, 4).t() % 7
    assert torch.equal(ops.embedding(ids, w), w[ids])
    wide = torch.randn(7, 24, device=device)
    assert torch.equal(ops.embedding(ids, wide[:, 8:16]), wide[:, 8:16][ids])
    assert torch.equal(ops.embedding(ids, wide.t()[:, :5]), wide.t()[:, :5][ids])
    assert torch.equal(ops.embedding(ids, wide[:, ::3]), wide[:, ::3][ids])
    # a gradient that is not contiguous: broadcast along the columns
    y = ops.embedding(ids, w, scale=0.5)
    (g,) = torch.autograd.grad(y, w, torch.ones(4, 3, 1, device=device).expand(4, 3, 4))
    assert torch.equal(g, torch.bincount(ids.reshape(-1), minlength=7)[:, None].expand(7, 4) * 0.5)


def test_shapes():
    check_shapes("cpu")


def check_refusals(device):
    w, ids = torch.zeros(4, 3, device=device), torch.zeros(2, dtype=torch.int64, device=device)
    for args, more in [((ids.float(), w), {}), ((ids, w[0]), {}), ((ids, w.double()), {}), ((ids, w), dict(dtype=torch.float64)),
                       ((ids, w), dict(scale=float("nan"))), ((ids, w.to_sparse()), {})]:
        with pytest.raises((RuntimeError, TypeError)):
            ops.embedding(*args, **more)
    for padding in (4, -5):
        with pytest.raises(ValueError):
            ops.embedding(ids, w, padding_idx=padding)


def test_refusals():
    check_refusals("cpu")
    w = torch.zeros(4, 3)
    for bad in (-1, 4):
        with pytest.raises(RuntimeError, match="not in the table"):
            ops.embedding(torch.tensor([0, bad]), w)


def check_second_order(device):
    """Gradients of gradients go through the plain composition: linear in the table, so that they vanish, and in the gradient that comes in."""
    w = torch.randn(5, 8, device=device, requires_grad=True)
    ids = torch.tensor([1, 3, 1], device=device)
    v = torch.randn(3, 8, device=device, requires_grad=True)
    y = ops.embedding(ids, w, scale=2.0, padding_idx=3)
    (g,) = torch.autograd.grad(y, w, v, create_graph=True)
    (gv,) = torch.autograd.grad((g * w.detach()).sum(), v)
    want = 2.0 * w.detach()[ids]
    want[1] = 0
    assert torch.allclose(gv, want, atol=1e-6)


def test_second_order():
    check_second_order("cpu")


def test_module_of_a_given_table():
    table = torch.randn(10, 8)
    m = ops.ScaledEmbedding.from_pretrained(table, padding_idx=-1, scale=2.0)
    ids = torch.tensor([3, 9])
    assert m.weight.data_ptr() == table.data_ptr() and not m.weight.requires_grad and m.padding_idx == 9
    assert (m.num_embeddings, m.embedding_dim) == (10, 8) and torch.equal(m(ids), 2.0 * table[ids])
    m = ops.ScaledEmbedding.from_pretrained(table, freeze=False, dtype_out=torch.bfloat16)
    m(ids).sum().backward()
    assert m(ids).dtype == torch.bfloat16 and m.weight.grad.sum() == 16
    with pytest.raises(ValueError):
        ops.ScaledEmbedding.from_pretrained(table[0])


def check_module(device):
    m = ops.ScaledEmbedding(10, 8, scale=3.0, padding_idx=2).to(device)
    ids = torch.tensor([[0, 2], [9, 9]], device=device)
    assert torch.equal(m(ids), m.weight[ids] * 3.0)
    with torch.autocast(device, dtype=torch.bfloat16):
        y = m(ids)
    assert y.dtype == torch.bfloat16 and torch.equal(y, (m.weight[ids] * 3.0).bfloat16())
    y.float().sum().backward()
    want = torch.zeros(10, 1, device=device)
    want[0], want[9] = 3, 6
    assert torch.equal(m.weight.grad, want.expand(10, 8))


def test_module():
    check_module("cpu")
