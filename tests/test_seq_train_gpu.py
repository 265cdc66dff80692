"""The sequence-model operators together, as a program uses them: a small recurrent language model
scores its answers, takes clipped policy steps with AdamW, and then generates token by token."""
import pytest
import torch
import torch.nn.functional as F

import seq_oracle as so

pytestmark = pytest.mark.gpu
V, D = 61, 24


class Model(torch.nn.Module):
    """Embedding -> (candidates, gates) -> recurrence -> head; `scan` is the recurrence."""

    def __init__(self, scan):
        super().__init__()
        g = torch.Generator().manual_seed(0)
        self.emb = torch.nn.Parameter(torch.randn(V, D, generator=g))
        self.w = torch.nn.Parameter(torch.randn(2 * D, D, generator=g) * D ** -0.5)
        self.head = torch.nn.Parameter(torch.randn(V, D, generator=g) * D ** -0.5)
        self.scan = scan

    def gates(self, ids):
        return F.linear(F.embedding(ids, self.emb), self.w).chunk(2, -1)

    def forward(self, ids, lengths):
        z, f = self.gates(ids)
        y, h = self.scan(z, f + 1, lengths)
        return F.linear(y, self.head), h


def _plain_scan(z, f, lengths):
    h, out = torch.zeros_like(z[:, 0]), []
    a = torch.sigmoid(f)
    for t in range(z.shape[1]):
        on = (t < lengths)[:, None]
        h = torch.where(on, a[:, t] * h + (1 - a[:, t]) * z[:, t], h)
        out.append(torch.where(on, h, 0.0))
    return torch.stack(out, 1), h


def _plain_loss(logits, tokens, old, adv, ref, mask):
    lp = torch.log_softmax(logits, -1).gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
    rho = torch.exp(lp - old)
    k = torch.exp(ref - lp) - (ref - lp) - 1
    term = -torch.minimum(rho * adv, rho.clamp(0.8, 1.2) * adv) + 0.05 * k
    return torch.where(mask, term, 0.0).sum() / mask.sum()


@pytest.mark.parametrize("bits", [32, 8])
def test_policy_steps_of_a_recurrent_model(bits):
    from language_interpolation_amd import functional as PF
    from language_interpolation_amd.train import AdamW
    gen = torch.Generator().manual_seed(1)
    b, t = 6, 40
    ids = torch.randint(0, V, (b, t + 1), generator=gen)
    lengths = torch.tensor([40, 33, 0, 1, 17, 40], dtype=torch.int32)
    mask = (torch.arange(t) < lengths[:, None]) & (torch.arange(t) >= 3)
    tokens = torch.where(mask, ids[:, 1:], -100)
    adv = torch.randn(b, generator=gen)
    model = Model(lambda z, f, n: PF.gated_recurrence(z, f, lengths=n)).cuda()
    exact = Model(_plain_scan).double()
    dev = [x.cuda() for x in (ids[:, :-1], lengths, tokens, mask, adv)]
    with torch.no_grad():
        logits, _ = model(dev[0], dev[1])
        old = PF.token_log_probs(logits, dev[2], dev[3])
        ref = PF.token_log_probs(logits * 0.9, dev[2], dev[3])
    opt = AdamW(model.parameters(), lr=2e-2, moment_bits=bits, seed=3)
    opt.MIN_8BIT = 512
    for step in range(4):
        opt.zero_grad(set_to_none=True)
        logits, _ = model(dev[0], dev[1])
        loss, kl, cut = PF.clipped_policy_loss(logits, dev[2], old, dev[4], ref, dev[3], kl_coef=0.05)
        loss.backward()
        # the same weights in 64 bits: loss and every gradient
        with torch.no_grad():
            for q, p in zip(exact.parameters(), model.parameters()):
                q.copy_(p)
        exact.zero_grad()
        x, _ = exact(ids[:, :-1], lengths)
        want = _plain_loss(x, tokens, old.cpu().double(), adv[:, None].double(), ref.cpu().double(), mask)
        want.backward()
        assert abs(float(loss.detach()) - float(want.detach())) < 1e-5
        for q, p in zip(exact.parameters(), model.parameters()):
            # sums of some hundred fp32 products, each off by a few 2^-24 of terms of the sum's size
            assert float((p.grad.cpu().double() - q.grad).norm()) < 1e-5 * float(q.grad.norm())
        before = [(p.detach().cpu().numpy().ravel(), p.grad.cpu().numpy().ravel(), dict(opt.state[p])) for p in model.parameters()]
        kept = [{k: (v.cpu().numpy().ravel() if torch.is_tensor(v) else v) for k, v in s.items()} for _, _, s in before]
        opt.step()
        if bits == 32:
            for (w, g, _), s, p in zip(before, kept, model.parameters()):
                m, v = (s.get(k, 0 * w) for k in ("exp_avg", "exp_avg_sq"))
                assert (so.adamw(w, g, m, v, step + 1, 2e-2, (0.9, 0.999), 1e-8, 1e-2)[0]
                        == p.detach().cpu().numpy().ravel()).all()
        else:
            assert opt.state[model.emb]["exp_avg"].dtype == torch.uint8
    assert 0 <= float(cut) <= 1 and float(kl) >= 0
    # generation: the prompt at once, then token by token, is the whole at once
    with torch.no_grad():
        full, _ = model(dev[0], torch.full_like(dev[1], t))
        z, f = model.gates(dev[0])
        y, h = PF.gated_recurrence(z[:, :25], f[:, :25] + 1)
        rows = [y]
        for i in range(25, t):
            rows.append(PF.gated_recurrence_step(z[:, i], f[:, i] + 1, h)[:, None])
        pieces = F.linear(torch.cat(rows, 1), model.head)
        assert float((pieces - full).abs().max()) < 1e-5 * float(full.abs().max())


@pytest.mark.parametrize("name", ["adamw", "adamw_8bit"])
def test_the_configured_optimizers_train(name):
    """optimizer=adamw / adamw_8bit of the training command, eager and from a captured graph: the same
    weights after the same batches."""
    import os

    from language_interpolation_amd import train as T
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "configs",
                        "high_order_interpolation.yaml")
    cfg = T.load_config(root, [f"optimizer={name}", "optimizer.lr=1e-3", "batch_size=64"])
    text = T.synthetic_text(5000)
    nets = []
    for graph in (False, True):
        torch.manual_seed(0)
        net = T.prediction_net(cfg, device="cuda")
        T.fit(net, T.make_data(cfg, text), 5, 64, graph=graph)
        nets.append(net)
    for p, q in zip(*(n.parameters() for n in nets)):
        assert bool(torch.isfinite(p).all())
        # float atomics in the small layers' weight gradients: the last bits differ, and an entry whose
        # gradient is nothing but those may step either way, 5 steps of lr
        assert float((p - q).detach().abs().max()) <= 5 * 2.2e-3


def test_second_derivatives_are_refused():
    """A graph of the gradient may be asked for (another term of the loss may need it); using it is an error."""
    from language_interpolation_amd import functional as PF
    z, f = (torch.randn(2, 20, 8, device="cuda", requires_grad=True) for _ in range(2))
    x = torch.randn(2, 5, 30, device="cuda", requires_grad=True)
    tok = torch.randint(0, 30, (2, 5), device="cuda")
    old, adv = torch.full((2, 5), -3.0, device="cuda"), torch.ones(2, device="cuda")
    calls = [(lambda: PF.gated_recurrence(z, f)[0].square().sum(), z), (lambda: PF.token_log_probs(x, tok).square().sum(), x),
             (lambda: PF.clipped_policy_loss(x, tok, old, adv)[0].square(), x)]
    for call, leaf in calls:
        (plain,) = torch.autograd.grad(call(), leaf)
        (g,) = torch.autograd.grad(call(), leaf, create_graph=True)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError, match="twice"):
            g.sum().backward()
