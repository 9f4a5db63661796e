"""What the dense layer and the optimiser ask of their callers, without a GPU."""
import pytest
import torch

from compressgnn_b200 import _lib, optim


@pytest.mark.parametrize("dtype, packed", [(0, 6), (2, 2), (3, 2)])
def test_a_weight_gradient_of_one_split_has_no_copy_in_the_scratch(dtype, packed):
    """There are more tiles than multiprocessors: a split writes the gradient itself, and the scratch holds the weight's image (six bytes
    an element in fp32) and a sum for each column."""
    room = _lib.lib().cgnn_linear_backward_scratch_bytes(dtype, 4000, 4096, 4096)
    assert packed * 4096 * 4096 <= room <= packed * 4096 * 4096 + (1 << 16)


# ---------------------------------------------------------------------------------------------
# what the groups of an optimiser have in common
# ---------------------------------------------------------------------------------------------
def parameter():
    return torch.nn.Parameter(torch.zeros(3))


@pytest.mark.parametrize("name, value", [("max_norm", 0.1), ("seed", 5)])
def test_a_group_has_no_norm_and_no_seed_of_its_own(name, value):
    with pytest.raises(ValueError, match=name):
        optim.AdamW([dict(params=[parameter()]), dict(params=[parameter()], **{name: value})])
    with pytest.raises(ValueError, match=name):
        optim.AdamW([dict(params=[parameter()], **{name: value})])
    opt = optim.AdamW([dict(params=[parameter()], **{name: value})], **{name: value})
    with pytest.raises(ValueError, match=name):
        opt.add_param_group(dict(params=[parameter()], **{name: value + 1}))
    assert len(opt.param_groups) == 1
    # one that is added later takes what the others have by then
    opt.param_groups[0][name] = value + 1
    opt.add_param_group(dict(params=[parameter()]))
    assert opt.param_groups[1][name] == value + 1
    opt.step()
    opt.param_groups[0][name] = value
    with pytest.raises(RuntimeError, match="common to all groups"):
        opt.step()


def test_a_loaded_state_brings_its_norm_and_seed(monkeypatch):
    seen = []
    monkeypatch.setattr(optim._native, "adamw_step", lambda *args: seen.append((args[9], args[12])))
    p = parameter()
    saved = optim.AdamW([p], max_norm=0.25, seed=9).state_dict()
    opt = optim.AdamW([p], max_norm=1.0)
    opt.load_state_dict(saved)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    p.grad = torch.ones(3)
    opt.step()
    opt.param_groups[0]["max_norm"] = 0.5
    opt.step()
    assert seen == [(0.25, 9), (0.5, 9)]


def test_a_state_of_another_optimiser_is_refused():
    p = parameter()
    p.grad = torch.ones(3)
    theirs = torch.optim.AdamW([p])
    opt = optim.AdamW([p], lr=0.5)
    with pytest.raises(ValueError, match="another optimiser"):
        opt.load_state_dict(theirs.state_dict())  # before its first step: the groups
    theirs.step()
    state = theirs.state_dict()
    state["param_groups"] = opt.state_dict()["param_groups"]
    with pytest.raises(ValueError, match="another optimiser"):
        opt.load_state_dict(state)
    assert not opt.state and opt.param_groups[0]["lr"] == 0.5
