"""Which changes of the expert weights a quantised module sees; no GPU needed.

The packed weights stand in as strings: what is tested comes before any kernel.
"""
import copy
import importlib
import io

import pytest
import torch

from _helpers import package


@pytest.fixture(scope="module")
def layers():
    package()
    return importlib.import_module("hrm-moe_b200.layers")


def _quantised(experts):
    experts._mxfp4 = ("gate_up", "down", experts._weights_state(),
                      (experts.gate_up_weight, experts.down_weight))
    return experts


@pytest.fixture
def experts(layers):
    m = layers.SparseMoESwiGLU(32, 16, 4, 2, True, dtype=torch.bfloat16)
    return _quantised(m.experts)


@torch.no_grad()
def _optimizer_step(m):
    for w in m.parameters():
        w.grad = torch.ones_like(w)
    torch.optim.SGD(m.parameters(), lr=0.1).step()


def _in_inference_mode(write):
    def run(m):
        with torch.inference_mode():
            write(m)
    return run


def _swap_and_back(m):
    w = m.down_weight
    kept = torch.Tensor.data.__get__(w)
    w.data = torch.zeros_like(kept)
    kept.mul_(2)
    w.data = kept


WRITES = {
    "data.mul_": lambda m: m.down_weight.data.mul_(2),
    "data.copy_": lambda m: m.gate_up_weight.data.copy_(torch.zeros_like(m.gate_up_weight)),
    "view of data": lambda m: m.down_weight.data[1].view(-1)[3:].fill_(1),
    "indexed data": lambda m: m.gate_up_weight.data.__setitem__((0, 0, 0), 1.0),
    "foreach on data": lambda m: torch._foreach_mul_([w.data for w in m.parameters()], 2.0),
    "data in inference mode": _in_inference_mode(lambda m: m.down_weight.data.mul_(2)),
    "in place in inference mode": _in_inference_mode(lambda m: m.down_weight.mul_(2)),
    "in place": torch.no_grad()(lambda m: m.down_weight.mul_(2)),
    "detach": lambda m: m.down_weight.detach().mul_(2),
    "new data": lambda m: setattr(m.down_weight, "data", m.down_weight.data.clone()),
    "new data and back": _swap_and_back,
    "transposed data": lambda m: setattr(m.down_weight, "data", m.down_weight.data.mT),
    "another parameter": lambda m: setattr(m, "down_weight", torch.nn.Parameter(m.down_weight.detach())),
    "optimizer step": _optimizer_step,
    "load_state_dict": lambda m: m.load_state_dict({k: v + 1 for k, v in m.state_dict().items()}),
    "assigning load_state_dict": lambda m: m.load_state_dict(
        {k: v + 1 for k, v in m.state_dict().items()}, assign=True),
    "vector_to_parameters": lambda m: torch.nn.utils.vector_to_parameters(
        torch.zeros(sum(w.numel() for w in m.parameters())), m.parameters()),
    "another type": lambda m: m.to(torch.float32),
    "init": lambda m: torch.nn.init.zeros_(m.down_weight),
}


@pytest.mark.parametrize("write", WRITES)
def test_a_write_is_seen(experts, write):
    assert experts.quantized() == ("gate_up", "down")
    WRITES[write](experts)
    with pytest.raises(RuntimeError, match="changed"):
        experts.quantized()
    assert _quantised(experts).quantized() == ("gate_up", "down")


READS = {
    "data": lambda m: m.down_weight.data.sum() + m.gate_up_weight.data[0, 0, 0],
    "state_dict": lambda m: [v.sum() for v in m.state_dict().values()],
    "save": lambda m: torch.save(m, io.BytesIO()),
    "deepcopy": copy.deepcopy,
    "the same device and type": lambda m: m.to("cpu", torch.bfloat16),
    "the same data": lambda m: setattr(m.down_weight, "data", m.down_weight.data),
    "eval": lambda m: m.eval().requires_grad_(False),
    "parameters_to_vector": lambda m: torch.nn.utils.parameters_to_vector(m.parameters()),
    "zero_grad": lambda m: m.zero_grad(),
}


@pytest.mark.parametrize("read", READS)
def test_reading_is_no_change(experts, read):
    READS[read](experts)
    assert experts.quantized() == ("gate_up", "down")
    assert isinstance(experts.down_weight, torch.nn.Parameter)


def test_copies_are_stale_and_plain(experts):
    f = io.BytesIO()
    torch.save(experts, f)
    f.seek(0)
    for other in (copy.deepcopy(experts), torch.load(f, weights_only=False)):
        for name, w in other.named_parameters():
            assert type(w) is torch.nn.Parameter and not hasattr(w, "_alias"), name
            assert torch.equal(w, getattr(experts, name))
        with pytest.raises(RuntimeError, match="changed"):
            other.quantized()
        other.down_weight.data.zero_()
        other.drop_quantized_experts()
        assert other.quantized() is None
    assert experts.quantized() == ("gate_up", "down")


def test_dropping_gives_the_parameters_back(experts):
    w = experts.down_weight
    version = w._version
    experts.drop_quantized_experts()
    assert type(w) is torch.nn.Parameter and experts.down_weight is w
    assert not hasattr(w, "_alias") and w._version == version
    w.data.mul_(2)
    w.data = w.data.clone()
    assert experts.quantized() is None


def test_a_parameter_of_two_modules(layers):
    a, b = (layers.SparseMoESwiGLU(32, 16, 4, 2, True, dtype=torch.bfloat16).experts for _ in range(2))
    b.down_weight = a.down_weight
    _quantised(a), _quantised(b)
    assert a.quantized() and b.quantized()
    b.drop_quantized_experts()       # ends the watch: a cannot know any more
    a.down_weight.data.mul_(2)
    _quantised(b)
    with pytest.raises(RuntimeError, match="changed"):
        a.quantized()
    assert b.quantized()
    a.down_weight.data.mul_(2)
    with pytest.raises(RuntimeError, match="changed"):
        b.quantized()


def test_parameters_without_a_record_of_writes_are_refused(layers):
    with torch.inference_mode():
        m = layers.SparseMoESwiGLU(32, 16, 4, 2, True, dtype=torch.bfloat16)
        with pytest.raises(RuntimeError, match="inference mode"):
            m.quantize_experts()
        with pytest.raises(RuntimeError, match="changed"):
            _quantised(m.experts).quantized()
    m = layers.SparseMoESwiGLU(32, 16, 4, 2, True, dtype=torch.bfloat16)

    class Other(torch.nn.Parameter):
        pass

    m.experts.down_weight = Other(m.experts.down_weight.detach())
    with pytest.raises(TypeError, match="plain parameters"):
        m.quantize_experts()


def test_a_module_pickled_without_packed_weights_loads(layers):
    m = layers.SparseMoESwiGLU(32, 16, 4, 2, True, dtype=torch.bfloat16)
    m.experts.__dict__.pop("_mxfp4", None)  # as pickled before the attribute existed
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    old = torch.load(f, weights_only=False)
    assert old.experts.quantized() is None
    old.drop_quantized_experts()
    assert _quantised(old.experts).quantized() == ("gate_up", "down")
    old.drop_quantized_experts()
    assert old.experts.quantized() is None and m.experts.quantized() is None
