"""What experts.backward refuses before its first call (CPU): tensors that are not the forward's, whose
rows an index out of range would read as zeros."""
import pytest
import torch

from moonshine_amd import experts, fp8, grouped
from moonshine_amd.synth import ACT_SWIGLU
from test_training_refusals import Called, bf, ints, stopped  # noqa: F401

E, H, F, T, k = 3, 16, 24, 4, 2


def backward(**change):
    a = dict(doutput=bf(T, H), gate_up=bf(E, 2 * F, H), down=bf(E, H, F))
    a.update(change)
    plan = grouped.RoutePlan(ints(T, k), E, ints(E), ints(E + 1), ints(T * k), ints(T * k))
    saved = experts.Saved(plan, bf(T, H), torch.ones(T, k), bf(T * k, 2 * F), bf(T * k, F), ACT_SWIGLU, 4.0, 25.0)
    return experts.backward(saved=saved, **a)


def test_a_backward_in_order_passes(stopped):  # noqa: F811
    with pytest.raises(Called):
        backward()


@pytest.mark.parametrize("change", [
    dict(doutput=bf(T - 1, H)), dict(doutput=bf(T + 1, H)), dict(doutput=bf(T, H + 8)), dict(gate_up=bf(E, 2 * F, H + 8)),
    dict(gate_up=bf(E + 1, 2 * F, H)), dict(gate_up=bf(E, 2 * F + 8, H)), dict(down=bf(E, H, F + 8)),
    dict(down=bf(E - 1, H, F))])
def test_backward_refuses_what_is_not_the_forwards(stopped, change):  # noqa: F811
    with pytest.raises(ValueError):
        backward(**change)


@pytest.mark.parametrize("change", [
    dict(dgate_up=torch.zeros(E, 2 * F, H + 8)), dict(dgate_up=bf(E, 2 * F, H)), dict(dgate_up=torch.zeros(2 * F, H)),
    dict(dgate_up=torch.zeros(E, H, 2 * F).transpose(1, 2)), dict(ddown=torch.zeros(E, F, H)), dict(ddown=bf(E, H, F)),
    dict(dgate_up=torch.zeros(2 * E * F * H + 1)[1:].view(E, 2 * F, H)),
    dict(gate_up=bf(2 * E * F * H + 1)[1:].view(E, 2 * F, H))])
def test_backward_refuses_a_gradient_before_it_adds_to_the_other(stopped, monkeypatch, change):  # noqa: F811
    def layout(t, name, dtypes, dim, device=None):
        if t.dtype not in dtypes or t.dim() != dim or not t.is_contiguous():
            raise ValueError(name)
        return t.data_ptr()

    monkeypatch.setattr(fp8, "_layout", layout)
    a = dict(dgate_up=torch.zeros(E, 2 * F, H), ddown=torch.zeros(E, H, F))
    with pytest.raises(Called):
        backward(**a)
    with pytest.raises(ValueError):
        backward(**dict(a, **change))
