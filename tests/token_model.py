"""A small language model that goes through the token operators as a training step meets them: scaled lookup, a layer, logits from the same
table, log probabilities with an entropy bonus, AdamW; and the same in plain torch in 64 bits."""
import torch
import torch.nn as nn
import torch.nn.functional as F

import bagua_core_b200.ops as ops
from bagua_core_b200.ops.fused_linear import ShadowLinear

VOCAB, HIDDEN, BATCH, SEQ, PAD = 1031, 64, 3, 50, 7


class Model(nn.Module):
    def __init__(self):
        super().__init__()
        self.tok = ops.ScaledEmbedding(VOCAB, HIDDEN, scale=HIDDEN ** 0.5, padding_idx=PAD)
        self.fc = ShadowLinear(HIDDEN, HIDDEN)
        self.out = nn.Linear(HIDDEN, VOCAB)
        nn.init.normal_(self.tok.weight, 0.0, 0.05)

    def forward(self, ids):
        x = self.tok(ids)
        return self.out(x + self.fc(x, "gelu"))


def loss_of(logits, targets):
    r = ops.token_log_probs(logits, targets, top=4)
    count = (targets != -100).sum()
    return -(r.log_probs.sum() + 0.01 * r.entropy.sum()) / count, r


def plain_gradients(model, ids, targets):
    """Gradients of the loss in 64 bits, by parameter name, and the log probabilities."""
    p = {n: q.detach().double().cpu().requires_grad_() for n, q in model.named_parameters()}
    i, t = ids.cpu(), targets.cpu()
    x = F.embedding(i, p["tok.weight"], padding_idx=PAD) * HIDDEN ** 0.5
    y = x + F.gelu(F.linear(x, p["fc.weight"], p["fc.bias"]))
    lp = torch.log_softmax(F.linear(y, p["out.weight"], p["out.bias"]), -1)
    scored = t != -100
    picked = lp.gather(-1, t.clamp(min=0)[..., None])[..., 0]
    entropy = -(lp.exp() * lp).sum(-1)
    loss = -((picked + 0.01 * entropy) * scored).sum() / scored.sum()
    names = list(p)
    return dict(zip(names, torch.autograd.grad(loss, [p[n] for n in names]))), (picked * scored).detach()


def batch(device, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, VOCAB, (BATCH, SEQ), generator=g)
    ids[1, 30:] = PAD
    targets = torch.randint(0, VOCAB, (BATCH, SEQ), generator=g)
    targets[1, 30:] = -100
    return ids.to(device), targets.to(device)
