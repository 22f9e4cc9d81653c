"""The token operators together, as a training step uses them; BERT with more tokens than its own embedding kernel takes."""
import os

import pytest
import torch

import bagua_core_b200.ops as ops
import bagua_core_b200.parallel as P
import test_cpu_token_step as host
import token_model as tm
from bagua_core_b200 import models
from bagua_core_b200.ops import wgrad

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def settings():
    before, tf32 = wgrad.enabled, torch.backends.cuda.matmul.allow_tf32
    wgrad.enabled, torch.backends.cuda.matmul.allow_tf32 = False, False
    yield
    wgrad.enabled, torch.backends.cuda.matmul.allow_tf32 = before, tf32


@pytest.mark.parametrize("bits", [32, 8])
def test_training_step(bits):
    host.check_step("cuda", bits)


@pytest.mark.parametrize("bits,in_place", [(32, True), (8, True), (8, False)])
def test_wrapped_training_steps_in_bf16(bits, in_place):
    """Through `with_bagua`, under bf16 autocast, with bf16 copies and gradients added in place: gradients against 64 bits, and steps that
    a second run repeats bit for bit."""
    wgrad.enabled = in_place
    os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
    os.environ.setdefault("MASTER_PORT", "29561")
    dev, runs = torch.device("cuda", 0), []
    for _ in range(2):
        torch.manual_seed(2)
        model = tm.Model().to(dev)
        P.init_process_group(dev)
        opt = P.FlatAdamW(model.parameters(), lr=1e-3, state_bits=bits, bf16_shadow=True, seed=4)
        bm = P.with_bagua(model, [opt], P.GradientAllReduceAlgorithm(), bucket_bytes=100 << 10)
        assert len(bm.bagua_buckets) > 1
        for step in range(3):
            ids, targets = tm.batch(dev, step)
            opt.zero_grad()
            with torch.autocast("cuda", dtype=torch.bfloat16):
                logits = bm(ids)
            assert logits.dtype == torch.bfloat16
            loss, r = tm.loss_of(logits, targets)
            loss.backward()
            want, picked = tm.plain_gradients(model, ids, targets)
            # bf16 activations, weights and logits: half a step each of values below 8; gradients a few of them relative to their tensor's norm
            assert (r.log_probs.detach().cpu().double() - picked).abs().max() <= 8 * 8 * 2.0 ** -8
            for n, p in model.named_parameters():
                assert (p.grad.cpu().double() - want[n]).norm() <= 8 * 2.0 ** -8 * want[n].norm(), n
            opt.step()
            assert all(torch.equal(p._bagua_bf16.view, p.detach().bfloat16()) for p in model.parameters())
        assert opt.kernel_launches == 3
        runs.append([p.detach().clone() for p in model.parameters()] + [x for p in model.parameters() for x in opt.moments(p)])
        P.destroy_process_group()
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("in_place", [False, True])
def test_bert_with_many_tokens_looks_them_up_by_sorting(in_place):
    """More tokens than the encoder's embedding kernel takes: the same output as the framework's lookup, the same gradients but for the
    order of their sums."""
    wgrad.enabled = in_place
    config = models.BertConfig.tiny()
    config.dropout = 0.0
    torch.manual_seed(0)
    model = models.BertForQuestionAnswering(config).cuda()
    batch, seq = 72, 128
    assert batch * seq > ops._C.max_embedding_tokens
    ids = (torch.rand(batch, seq, device="cuda") ** 4 * config.vocab_size).long()
    spans = torch.randint(0, seq, (2, batch), device="cuda")
    got = []
    for own in (True, False):
        for p in model.parameters():
            p.grad = torch.zeros_like(p)
        # a hook on the table's module: it is called, not replaced
        handle = None if own else model.tok.register_forward_hook(lambda *a: None)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            loss = model(ids, spans[0], spans[1])
        before = ops._C.op_stats()["launches"]
        loss.backward()
        got.append((loss.detach().clone(), model.tok.weight.grad.clone(), model.pos.weight.grad.clone(), ops._C.op_stats()["launches"] - before))
        if handle:
            handle.remove()
    assert torch.equal(got[0][0], got[1][0]) and got[0][3] > got[1][3]
    # sums of up to 3,000 rows in two orders: a few roundings of the largest sums
    want = got[1][1].double()
    assert (got[0][1].double() - want).abs().max() <= 64 * 2.0 ** -24 * want.abs().max() + 2.0 ** -24 * want.norm()
    assert (got[0][1].double() - want).norm() <= 2.0 ** -20 * want.norm()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_optimizer_steps(bits):
    """With `capturable=True` a captured step of the flat buffers, replayed, does what as many calls do, also behind a loaded state;
    without it, it is refused."""
    os.environ.setdefault("MASTER_ADDR", "127.0.0.1")
    os.environ.setdefault("MASTER_PORT", "29563")
    dev = torch.device("cuda", 0)
    g = torch.Generator().manual_seed(3)
    P.init_process_group(dev)

    def make(capturable):
        torch.manual_seed(2)
        model = tm.Model().to(dev)
        biases = [p for n, p in model.named_parameters() if n.endswith("bias")]
        weights = [p for n, p in model.named_parameters() if not n.endswith("bias")]
        opt = P.FlatAdamW([{"params": weights}, {"params": biases, "weight_decay": 0.0}], lr=1e-2, state_bits=bits, capturable=capturable)
        return model, opt, P.with_bagua(model, [opt], P.GradientAllReduceAlgorithm(), bucket_bytes=100 << 10)

    eager, captured = make(False), make(True)
    grads = [torch.randn(p.shape, generator=g).to(dev) for p in eager[0].parameters()]
    for model, *_ in (eager, captured):
        for p, x in zip(model.parameters(), grads):
            p.grad.copy_(x)
    graph = torch.cuda.CUDAGraph()
    eager[1].step(), captured[1].step()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured[1].step()
    for _ in range(3):
        eager[1].step(), graph.replay()

    def same():
        torch.cuda.synchronize()
        a, b = (o.state_dict()["state"] for o in (eager[1], captured[1]))
        assert all(x["step"] == y["step"] for x, y in zip(a.values(), b.values()))
        assert all(torch.equal(p, q) for p, q in zip(eager[0].parameters(), captured[0].parameters()))
        assert all(torch.equal(x, y) for p, q in zip(eager[0].parameters(), captured[0].parameters())
                   for x, y in zip(eager[1].moments(p), captured[1].moments(q)))
        return {k: {n: v.clone() if isinstance(v, torch.Tensor) else v for n, v in x.items()} for k, x in a.items()}

    saved = same()
    assert {x["step"] for x in saved.values()} == {4}
    eager[1].step(), graph.replay()
    for _, opt, _ in (eager, captured):
        opt.load_state_dict({"state": saved, "param_groups": opt.state_dict()["param_groups"]})
    eager[1].step(), graph.replay()
    assert {x["step"] for x in same().values()} == {5}
    refused = torch.cuda.CUDAGraph()
    x = torch.zeros(1, device=dev)
    with torch.cuda.graph(refused):
        x.add_(1)
        with pytest.raises(RuntimeError, match="captured"):
            eager[1].step()
    P.destroy_process_group()
