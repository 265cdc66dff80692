"""Which checkpoints train.AdamW goes on from, and which it refuses before it has touched anything."""
import copy

import pytest
import torch

from language_interpolation_amd.train import AdamW, Lion


def _params(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).requires_grad_() for s in ((6, 5), (7,))]


def _checkpoint(kind, steps=2, **kw):
    ps = _params()
    opt = kind(ps, **kw)
    for step in range(steps):
        for p in ps:
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(step))
        opt.step()
    return opt.state_dict()


def _refused(state, match):
    ps = _params()
    opt = AdamW(ps, lr=0.5, seed=9)
    opt.state[ps[0]]["kept"] = 1
    groups, saved = copy.deepcopy([{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups]), copy.deepcopy(state)
    with pytest.raises(ValueError, match=match):
        opt.load_state_dict(state)
    assert [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups] == groups
    assert opt.state[ps[0]] == {"kept": 1}
    assert str(state) == str(saved)


def test_another_rule_is_refused():
    adam, adamw = torch.optim.Adam, torch.optim.AdamW
    _refused(_checkpoint(adamw, maximize=True), "maximize")
    _refused(_checkpoint(adamw, amsgrad=True), "amsgrad")
    _refused(_checkpoint(adam, amsgrad=True), "amsgrad")
    _refused(_checkpoint(adam, weight_decay=0.1), "coupled")
    _refused(_checkpoint(torch.optim.RAdam), "Adam")
    _refused(_checkpoint(torch.optim.NAdam), "Adam")
    _refused(Lion(_params()).state_dict(), "Adam")
    # a checkpoint from before torch noted the rule: whose it is has to be said
    old = _checkpoint(adamw, weight_decay=0.1)
    del old["param_groups"][0]["decoupled_weight_decay"]
    _refused(old, "coupled")
    # in the second group only
    two = _checkpoint(adamw)
    both = AdamW([{"params": [p]} for p in _params()])
    state = both.state_dict()
    state["param_groups"][1]["maximize"] = True
    with pytest.raises(ValueError, match="maximize"):
        both.load_state_dict(state)
    assert "maximize" not in both.param_groups[1] and len(two["param_groups"]) == 1


def test_the_same_rule_is_loaded():
    for state in (_checkpoint(torch.optim.AdamW, weight_decay=0.1), _checkpoint(torch.optim.Adam),
                  _checkpoint(torch.optim.Adam, weight_decay=0.1, decoupled_weight_decay=True)):
        ps = _params()
        opt = AdamW(ps, lr=0.5, seed=9)
        opt.load_state_dict(state)
        group = opt.param_groups[0]
        assert group["lr"] == 1e-3 and group["seed"] == 9 and group["moment_bits"] == 32
        for i, p in enumerate(ps):
            assert opt.state[p]["step"] == 2
            assert torch.equal(opt.state[p]["exp_avg"], state["state"][i]["exp_avg"])
            assert torch.equal(opt.state[p]["exp_avg_sq"], state["state"][i]["exp_avg_sq"])
        again = AdamW(_params())
        again.load_state_dict(opt.state_dict())
        assert again.param_groups[0]["seed"] == 9


def test_moments_of_another_shape_are_refused():
    """A moment that could be spread over the weight is not, and the optimizer keeps what it had."""
    for name in ("exp_avg", "exp_avg_sq"):
        for shape in ((1, 5), (), (5, 6), (30,)):
            state = _checkpoint(torch.optim.AdamW)
            state["state"][0][name] = torch.ones(shape)
            _refused(state, "shape")


def test_codes_that_do_not_fit_are_refused():
    ps = [torch.zeros(100, 50).requires_grad_()]

    def state(p, shape=(100, 50), blocks=20, **kw):
        entry = {"step": 3}
        for name in ("exp_avg", "exp_avg_sq"):
            entry[name] = torch.zeros(shape, dtype=torch.uint8)
            entry[name + "_exponent"] = torch.zeros(blocks, dtype=torch.uint8)
        entry.update(kw)
        return {"state": {0: entry}, "param_groups": AdamW([p], moment_bits=8).state_dict()["param_groups"]}
    for kw, match in ((dict(shape=(100, 1)), "shape"), (dict(blocks=19), "exponents"), (dict(blocks=1), "exponents"),
                      (dict(exp_avg=torch.zeros(50, 100, dtype=torch.uint8).t()), "order"),
                      (dict(exp_avg_exponent=torch.zeros(20)), "exponents")):
        opt = AdamW(ps, lr=0.25)
        with pytest.raises(ValueError, match=match):
            opt.load_state_dict(state(ps[0], **kw))
        assert not opt.state and opt.param_groups[0]["lr"] == 0.25
    half = [torch.zeros(100, 50, dtype=torch.bfloat16).requires_grad_()]
    opt = AdamW(half)
    with pytest.raises(ValueError, match="shape"):
        opt.load_state_dict(state(half[0], master=torch.zeros(50)))
    opt.load_state_dict(state(half[0], master=torch.ones(100, 50)))
    assert float(opt.state[half[0]]["master"].sum()) == 5000
    assert opt.state[half[0]]["exp_avg"].dtype == torch.uint8
