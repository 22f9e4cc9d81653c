"""The token operators together, as a training step uses them, on the host (`test_gpu_token_step.py` has the GPU's)."""
import pytest
import torch

import adamw_plain
import bagua_core_b200.parallel as P
import token_model as tm

U = 2.0 ** -24


def check_step(device, bits):
    torch.manual_seed(2)
    model = tm.Model().to(device)
    opt = P.FlatAdamW(model.parameters(), lr=1e-2, state_bits=bits, seed=4)
    for step in range(1, 4):
        ids, targets = tm.batch(device, step)
        before = {n: p.detach().cpu().clone() for n, p in model.named_parameters()}
        held = {n: (torch.zeros_like(before[n]),) * 2 if step == 1 else tuple(x.cpu() for x in opt.moments(p)) for n, p in model.named_parameters()}
        opt.zero_grad()
        loss, r = tm.loss_of(model(ids), targets)
        loss.backward()
        want, picked = tm.plain_gradients(model, ids, targets)
        # fp32: products of 64 terms in two layers and sums over 150 tokens; a few hundred roundings of values of the tensors' sizes
        assert (r.log_probs.detach().cpu().double() - picked).abs().max() <= 400 * U * 16
        assert not r.log_probs[1, 30:].any() and (r.top_ids[1, 30:] == -1).all()
        for n, p in model.named_parameters():
            assert (p.grad.cpu().double() - want[n]).abs().max() <= 1000 * U * want[n].abs().max(), n
        assert not model.tok.weight.grad[tm.PAD].any()
        opt.step()
        for n, p in model.named_parameters():
            q, m, v = adamw_plain.step(before[n], p.grad.cpu(), *held[n], step, 1e-2, 0.9, 0.999, 1e-8, 1e-2)
            assert ((p.detach().cpu().double() - q).abs() <= 3 * U * (before[n].abs() + q.abs()) + 10 * 1e-2 * 16 * U).all(), n
            got = opt.moments(p)
            if bits == 32:
                assert (got[0].cpu().double() - m).abs().max() <= 4 * U * m.abs().max()
            else:  # an eighth of a value, or the smallest code's distance, 2^-9 / 480 of a block's largest
                assert ((got[0].flatten().cpu().double() - m.flatten()).abs() <= 1.01 * (m.flatten().abs() / 8 + m.abs().max() * 2.0 ** -9 / 480)).all(), n


@pytest.mark.parametrize("bits", [32, 8])
def test_training_step(bits):
    check_step("cpu", bits)
