"""The copies of the expert weights that ``PermutedSparseMoE`` keeps (4-bit bank, transposed
down weights) follow every write to the weights; no GPU is needed: the quantisation is
replaced by a plain copy of what it is given."""

import pytest
import torch

from moe_inference_verify_microbench_b200 import PermutedSparseMoE, W4Experts, ops


class Copied:
    def __init__(self, weights):
        self.weights = [w.clone() for w in weights]


@pytest.fixture
def module(monkeypatch):
    made, made_into = [], []

    def quantize(cls, w_gate, w_up, w_down, group_size=128, symmetric=True, into=None):
        made.append(Copied((w_gate, w_up, w_down)))
        made_into.append(into)
        return made[-1]

    monkeypatch.setattr(W4Experts, "quantize", classmethod(quantize))
    monkeypatch.setattr(ops, "transpose_down_weights", lambda w: w.transpose(1, 2).contiguous())
    mod = PermutedSparseMoE(64, 64, 4, 2, expert_weights="w4", group_size=64)
    mod.made, mod.made_into = made, made_into
    return mod


def is_current(mod):
    want = [torch.stack([getattr(e, n).weight.detach() for e in mod.experts])
            for n in ("gate_proj", "up_proj", "down_proj")]
    return (all(torch.equal(a, b) for a, b in zip(mod.experts_4bit().weights, want))
            and torch.equal(mod.down_weights_transposed(), want[2].transpose(1, 2)))


def other_state(mod):
    return {n: torch.randn_like(t) for n, t in mod.state_dict().items()}


def test_load_state_dict_after_a_forward(module):
    assert is_current(module)
    module.load_state_dict(other_state(module))
    assert is_current(module)
    module.load_state_dict(other_state(module), assign=True)
    assert is_current(module)


def test_load_of_one_expert(module):
    assert is_current(module)
    module.experts[2].load_state_dict(other_state(module.experts[2]))
    assert is_current(module)


@pytest.mark.parametrize("name", ["gate_proj", "up_proj", "down_proj"])
@pytest.mark.parametrize("expert", [0, 1, 3])
def test_write_through_one_parameter(module, name, expert):
    assert is_current(module)
    with torch.no_grad():
        getattr(module.experts[expert], name).weight.mul_(0.5)
    assert is_current(module)


def test_optimizer_step(module):
    assert is_current(module)
    opt = torch.optim.SGD(module.experts.parameters(), lr=0.1)
    for p in module.experts.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    assert is_current(module)


def test_write_through_the_stack(module):
    assert is_current(module)
    module.pack()[1].add_(1.0)
    assert is_current(module)


def test_copies_are_kept_while_nothing_is_written(module):
    assert is_current(module)
    bank, down = module.experts_4bit(), module.down_weights_transposed()
    module.state_dict()
    assert module.experts_4bit() is bank and module.down_weights_transposed() is down
    assert len(module.made) == 1
    assert module.experts_4bit(refresh=True) is not bank


def test_another_stack_in_the_same_place(module):
    """A stack that is bound later may lie where an earlier one lay and have been written as
    often: neither its address nor its version tells them apart."""
    assert is_current(module)
    bank = module.experts_4bit()
    old = module.pack()
    with torch.no_grad():
        module._bank.w_gate, module._bank.w_up, module._bank.w_down = (t.view_as(t) for t in old)
        assert [t.data_ptr() for t in module.pack()] == [t.data_ptr() for t in old]
        assert [t._version for t in module.pack()] == [t._version for t in old]
        assert module.experts_4bit() is not bank


def test_writes_under_inference_mode(module):
    with torch.inference_mode():
        assert is_current(module)
        module.experts[1].up_proj.weight.mul_(2.0)
        assert is_current(module)
        module.load_state_dict(other_state(module))
        assert is_current(module)


def test_module_made_and_bound_under_inference_mode(module):
    """The stacks and the parameters that are bound to them count their writes, whatever
    mode the module was made and first run in."""
    with torch.inference_mode():
        made = PermutedSparseMoE(64, 64, 4, 2, expert_weights="w4", group_size=64)
        assert is_current(made)
        made.experts[2].gate_proj.weight.add_(1.0)
        assert is_current(made)
    with torch.no_grad():
        made.experts[0].down_proj.weight.add_(1.0)
    assert is_current(made)
    assert not any(t.is_inference() for t in (*made.pack(), *made.experts.parameters()))


def test_a_copy_is_made_again_in_its_place(module):
    """What a captured forward reads stays where it is."""
    assert is_current(module)
    down = module.down_weights_transposed()
    bank = module.experts_4bit()
    module.load_state_dict(other_state(module))
    with torch.inference_mode():
        assert is_current(module)
    assert module.down_weights_transposed().data_ptr() == down.data_ptr()
    assert module.made_into[-1] is bank and module.made_into[0] is None
    module.load_state_dict(other_state(module))
    assert is_current(module)
    module.double()  # moved or cast: in memory of its own
    assert module.down_weights_transposed().dtype is torch.float64
    module.experts_4bit()
    assert module.made_into[-1] is None


@pytest.mark.parametrize("expert", [0, 2, 3])
def test_pack_after_a_parameter_was_replaced(module, expert):
    """``pack()`` (or a refresh) binds any expert's new ``Parameter`` object."""
    assert is_current(module)
    new = torch.randn(64, 64)
    module.experts[expert].up_proj.weight = torch.nn.Parameter(new.clone())
    assert torch.equal(module.pack()[1][expert], new)
    assert is_current(module)
    module.experts[expert].load_state_dict(other_state(module.experts[expert]), assign=True)
    module.experts_4bit(refresh=True)
    assert is_current(module)
    with torch.no_grad():
        module.experts[expert].up_proj.weight.zero_()
    assert is_current(module) and not bool(module.pack()[1][expert].any())
