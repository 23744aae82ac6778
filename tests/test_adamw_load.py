"""CPU: what AdamW checks before it changes anything."""
import copy

import pytest
import torch

from haste_amd.optim_adamw import AdamW


def saved_state(bits, n=200):
    w = torch.nn.Parameter(torch.ones(n))
    opt = AdamW([w], state_bits=bits, lr=0.5)
    opt._new_state(w, bits)
    return w, opt, opt.state_dict()


def snapshot(opt):
    return copy.deepcopy(opt.state_dict())


def same(a, b):
    assert a["param_groups"] == b["param_groups"] and a["state"].keys() == b["state"].keys()
    for k, s in a["state"].items():
        assert s.keys() == b["state"][k].keys()
        for name, v in s.items():
            w = b["state"][k][name]
            if isinstance(v, torch.Tensor):
                assert v.dtype == w.dtype and torch.equal(v.view(torch.uint8), w.view(torch.uint8))
            else:
                assert v == w


@pytest.mark.parametrize("spoil,word", [
    (lambda s: s["param_groups"][0].update(state_bits=32), "does not fit"),
    (lambda s: s["state"][0].update(exp_avg=torch.zeros(3)), "does not fit"),
    (lambda s: s["state"][0].pop("rms"), "does not fit"),
    (lambda s: s["state"][0].pop("step"), "step"),
    (lambda s: s["param_groups"][0].pop("state_bits"), "state_bits"),
    (lambda s: s["param_groups"][0].update(state_bits=16), "state_bits")])
def test_a_state_that_is_refused_replaces_nothing(spoil, word):
    _, opt, _ = saved_state(8)
    before = snapshot(opt)
    _, other, state = saved_state(8)
    other.param_groups[0]["lr"] = 0.25
    state = snapshot(other)
    spoil(state)
    with pytest.raises(ValueError, match=word):
        opt.load_state_dict(state)
    same(snapshot(opt), before)


def test_a_saved_state_of_torchs_own_adamw_is_refused_whole():
    w = torch.nn.Parameter(torch.ones(200))
    theirs = torch.optim.AdamW([w])
    w.grad = torch.ones(200)
    theirs.step()
    _, opt, _ = saved_state(32)
    before = snapshot(opt)
    with pytest.raises(ValueError, match="state_bits"):
        opt.load_state_dict(theirs.state_dict())
    same(snapshot(opt), before)


def test_hooks_may_change_the_state_that_is_loaded():
    w, opt, state = saved_state(32)
    state = copy.deepcopy(state)

    def hook(optimizer, s):
        s = copy.deepcopy(s)
        s["state"][0]["exp_avg"] += 2
        s["state"][0]["step"] = 7
        return s
    opt.register_load_state_dict_pre_hook(hook)
    opt.load_state_dict(state)
    assert (opt.state[w]["exp_avg"] == 2).all() and opt.state[w]["step"] == 7
    opt.load_state_dict(state)          # (as often as it is called)
    assert (opt.state[w]["exp_avg"] == 2).all()


@pytest.mark.parametrize("later", [False, True])
def test_state_bits_of_one_group_are_checked(later):
    a, b = (torch.nn.Parameter(torch.ones(4)) for _ in range(2))
    with pytest.raises(ValueError, match="state_bits"):
        if later:
            AdamW([a]).add_param_group(dict(params=[b], state_bits=16))
        else:
            AdamW([dict(params=[a]), dict(params=[b], state_bits=16)])
