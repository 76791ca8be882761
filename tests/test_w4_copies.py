"""A packed bank, and a module that holds one, can be copied, pickled and saved; no GPU is
needed: the packed tensors are plain bytes here."""

import copy
import io
import pickle

import pytest
import torch

from moe_inference_verify_microbench_b200 import PermutedSparseMoE, W4Experts, _native, ops


def bank(seed=0, E=2, H=64, I=64, group=64, zeros=True):
    gen = torch.Generator().manual_seed(seed)

    def packed(rows, cols):
        q = torch.randint(0, 256, (E * rows * cols // 2,), generator=gen, dtype=torch.uint8)
        return q, torch.randn(E * rows * (cols // group) * (2 if zeros else 1), generator=gen).bfloat16()

    return W4Experts(packed(2 * I, H), packed(H, I), E, H, I, group, zeros)


def struct_of(b):
    return _native.W4BankStruct.from_address(b.native)


def saved(value):
    buf = io.BytesIO()
    torch.save(value, buf)
    buf.seek(0)
    return torch.load(buf, weights_only=False)


COPIES = [copy.copy, copy.deepcopy, lambda b: pickle.loads(pickle.dumps(b)), saved]


@pytest.mark.parametrize("make", COPIES)
def test_bank(make):
    b = bank()
    c = make(b)
    for name in ("num_experts", "hidden", "intermediate", "group_size", "has_zeros", "device"):
        assert getattr(c, name) == getattr(b, name)
    assert c.nbytes() == b.nbytes()
    for s, t in zip((*b.w13, *b.w2), (*c.w13, *c.w2)):
        assert torch.equal(s, t) and (make is copy.copy) == (s.data_ptr() == t.data_ptr())
    # the struct that the kernels are given holds the copy's own addresses
    assert c.native != b.native
    st = struct_of(c)
    assert [st.w13_q, st.w13_s, st.w2_q, st.w2_s] == [t.data_ptr() for t in (*c.w13, *c.w2)]
    assert (st.E, st.H, st.I, st.group, st.has_zeros) == (2, 64, 64, 64, 1)
    del b  # nothing of the copy hangs on the original
    assert struct_of(c).w13_q == c.w13[0].data_ptr()


@pytest.fixture
def module(monkeypatch):
    made = []
    monkeypatch.setattr(W4Experts, "quantize",
                        classmethod(lambda cls, *a, **k: made.append(bank(len(made))) or made[-1]))
    monkeypatch.setattr(ops, "transpose_down_weights", lambda w: w.transpose(1, 2).contiguous())
    mod = PermutedSparseMoE(64, 64, 2, 1, expert_weights="w4", group_size=64)
    mod.experts_4bit()
    mod.down_weights_transposed()
    made.clear()
    return mod, made


@pytest.mark.parametrize("make", COPIES[1:])
def test_module_that_has_run(module, make):
    mod, made = module
    own = mod.experts_4bit()
    c = make(mod)
    for (n, s), (m, t) in zip(mod.named_parameters(), c.named_parameters()):
        assert n == m and torch.equal(s, t) and s.data_ptr() != t.data_ptr()
    assert not made and mod.experts_4bit() is own, "the original keeps its bank"
    assert c.experts_4bit() is not own and len(made) == 1, "the copy makes one of its weights"
    with torch.no_grad():
        c.experts[1].down_proj.weight.fill_(3.0)
    assert bool((c.down_weights_transposed()[1] == 3.0).all())
    assert not bool((mod.down_weights_transposed()[1] == 3.0).any())
    assert mod.experts_4bit() is own
