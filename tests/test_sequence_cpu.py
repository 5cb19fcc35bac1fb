"""Host side of the sequence operators without a GPU: the facade's checks (mobileposer_amd/sequence.py) in front of a stand-in
library that must not be reached, and the C entries' workspace sizes and NULL handles."""
import pytest
import torch

from mobileposer_amd import _lib
from mobileposer_amd.sequence import SequenceOps


class NotReached:
    def __getattr__(self, name):
        raise AssertionError("%s was called" % name)


class Ops(SequenceOps):
    def __init__(self):
        self.device, self._device_index, self._lib = torch.device("cpu"), -1, NotReached()

    def _require_weights(self):
        pass


def delta(B=2, T=5, Hk=2, Hv=4, dk=16, dv=8):
    z = torch.zeros
    return {"q": z(B, T, Hk, dk), "k": z(B, T, Hk, dk), "v": z(B, T, Hv, dv), "g": z(B, T, Hv), "beta": z(B, T, Hv)}


@pytest.mark.parametrize("change", [
    {"k": torch.zeros(2, 5, 2, 16, dtype=torch.bfloat16)}, {"k": torch.zeros(2, 4, 2, 16)}, {"v": torch.zeros(2, 5, 3, 8)}, {"v": torch.zeros(2, 5, 4, 0)},
    {"g": torch.zeros(2, 5, 3)}, {"g": torch.zeros(2, 5, 4, dtype=torch.float64)}, {"beta": torch.zeros(2, 5, 4, dtype=torch.bfloat16)},
    {"input_lengths": [5]}, {"input_lengths": [5, 6]}, {"input_lengths": [-1, 5]}, {"state": torch.zeros(2, 4, 8, 16)},
    {"state": torch.zeros(2, 4, 16, 8, dtype=torch.bfloat16)}, {"q": torch.zeros(2, 5, 2, 16, requires_grad=True)},
    {n: torch.zeros(2, 5, 2, 16, dtype=torch.float16) for n in "qk"}, {n: torch.zeros(2, 5, 2, 257) for n in "qk"}, {n: torch.zeros(2, 5, 0, 16) for n in "qk"},
    {n: torch.zeros(5, 2, 16) for n in "qk"}], ids=lambda c: " ".join(c))
def test_delta_rule_refuses(change):
    with pytest.raises(RuntimeError):
        Ops().delta_rule(**{**delta(), **change})


@pytest.mark.parametrize("change", [
    {"state": torch.zeros(1, 4, 16, 8)}, {"state": torch.zeros(2, 4, 8, 16).transpose(2, 3)}, {"state": torch.zeros(2, 4, 16, 9)}, {"slots": [0, 2]},
    {"slots": [0]}, {"state": torch.zeros(2, 4, 16, 8, dtype=torch.bfloat16)}, {"q": torch.zeros(3, 2, 16)}], ids=lambda c: " ".join(c))
def test_delta_rule_online_refuses(change):
    args = {n: t[:, 0] for n, t in delta().items()}
    with pytest.raises(RuntimeError):
        Ops().delta_rule_online(**{**args, "state": torch.zeros(2, 4, 16, 8), **change})


@pytest.mark.parametrize("change", [
    {"weight": torch.zeros(24, 15)}, {"weight": torch.zeros(24, 16, dtype=torch.bfloat16)}, {"bias": torch.zeros(23)}, {"up": torch.zeros(2, 24, 3)},
    {"up": torch.zeros(2, 23, 4)}, {"down": torch.zeros(2, 129, 16), "up": torch.zeros(2, 24, 129)}, {"down": torch.zeros(0, 4, 16), "up": torch.zeros(0, 24, 4)},
    {"scale": torch.zeros(3)}, {"scale": torch.zeros(2, dtype=torch.bfloat16)}, {"ids": [0]}, {"ids": [0, 2]}, {"x": torch.zeros(16)},
    {"x": torch.zeros(2, 3, 16, requires_grad=True)}], ids=lambda c: " ".join(c))
def test_linear_adapted_refuses(change):
    args = {"x": torch.zeros(2, 3, 16), "weight": torch.zeros(24, 16), "bias": torch.zeros(24), "down": torch.zeros(2, 4, 16), "up": torch.zeros(2, 24, 4),
            "scale": torch.zeros(2), "ids": [0, 1]}
    with pytest.raises(RuntimeError):
        Ops().linear_adapted(**{**args, **change})


def test_entries_without_a_handle_and_workspace_sizes():
    lib = _lib.load()
    assert lib.mp_delta_rule(None, 0, *[None] * 7, 1, 1, 1, 1, 1, 1, 1.0, *[None] * 4, 0, None) == _lib.MP_ERR_INVALID
    assert lib.mp_delta_rule_online(None, 0, *[None] * 7, 1, 1, 1, 1, 1, 1, 1.0, *[None] * 3) == _lib.MP_ERR_INVALID
    assert lib.mp_linear_adapted(None, 0, *[None] * 8, 1, 1, 1, 1, 1, 1, 0, None, None, 0, None) == _lib.MP_ERR_INVALID
    for f in (lambda B, T, Hv: lib.mp_delta_rule_workspace(B, T, Hv, 64, 64), lib.mp_linear_adapted_workspace):
        assert f(0, 1, 1) == f(1, 0, 1) == f(1, 1, 0) == 0
        assert 0 < f(1, 1, 1) <= f(2, 1, 1) <= f(2, 33, 1) <= f(2, 33, 3)
        assert f(4096, 65536, 64) > 2 ** 32                # sizes pass 32 bits


def block(**change):
    z = torch.zeros
    layers = {"linear1": (z(2, 4, 60), z(2, 256, 4), z(2)), "linear2": (z(2, 8, 512), z(2, 72, 8), None)}
    return Ops()._block_adapters({**layers, **change}, [0, -1], 2, {"linear1": (60, 256), "linear2": (512, 72)})


@pytest.mark.parametrize("change", [
    {"linear0": None}, {"linear1": (torch.zeros(2, 4, 61), torch.zeros(2, 256, 4), None)}, {"linear1": (torch.zeros(2, 4, 60), torch.zeros(2, 255, 4), None)},
    {"linear1": (torch.zeros(3, 4, 60), torch.zeros(3, 256, 4), None)}, {"linear2": (torch.zeros(2, 129, 512), torch.zeros(2, 72, 129), None)},
    {"linear2": (torch.zeros(2, 8, 512), torch.zeros(2, 72, 8), torch.zeros(3))}, {"linear2": (torch.zeros(2, 8, 512).double(), torch.zeros(2, 72, 8).double(), None)},
    {"linear2": (torch.zeros(2, 8, 512).bfloat16(), torch.zeros(2, 72, 8).bfloat16(), None)}, {"linear2": (torch.zeros(2, 8, 512, requires_grad=True), torch.zeros(2, 72, 8), None)},
], ids=lambda c: next(iter(c)))
def test_block_adapters_refuses(change):
    with pytest.raises(RuntimeError):
        block(**change)
    with pytest.raises(RuntimeError):
        Ops()._block_adapters({}, [0, 1], 2, {"linear1": (60, 256), "linear2": (512, 72)})
    lib = _lib.load()
    assert lib.mp_rnn_forward_adapted(None, 0, None, None, 1, 1, *[None] * 6, 1, *[None] * 3, 1, None, 1, None, 0, None) == _lib.MP_ERR_INVALID


def linear():
    z = torch.zeros
    return {"x": z(2, 3, 16), "weight": z(24, 16), "bias": z(24), "down": z(2, 4, 16), "up": z(2, 24, 4), "scale": z(2), "ids": [0, 1]}


@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta", "state"])
def test_delta_rule_refuses_a_tangent(name):
    from torch.autograd import forward_ad
    args = {**delta(), "state": torch.zeros(2, 4, 16, 8)}
    with forward_ad.dual_level():
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="tangent"):
            Ops().delta_rule(**args)
        with pytest.raises(RuntimeError, match="tangent"):
            Ops().delta_rule_online(**{n: t if n == "state" else t[:, 0] for n, t in args.items()})


@pytest.mark.parametrize("name", ["x", "weight", "bias", "down", "up", "scale"])
def test_linear_adapted_refuses_a_tangent(name):
    from torch.autograd import forward_ad
    args = linear()
    with forward_ad.dual_level():
        args[name] = forward_ad.make_dual(args[name], torch.ones_like(args[name]))
        with pytest.raises(RuntimeError, match="tangent"):
            Ops().linear_adapted(**args)
        if name in ("down", "up", "scale"):
            layer = {n: forward_ad.make_dual(t, t) if n == name else t for n, t in (("down", torch.zeros(2, 4, 60)), ("up", torch.zeros(2, 256, 4)), ("scale", torch.zeros(2)))}
            with pytest.raises(RuntimeError, match="tangent"):
                block(linear1=tuple(layer.values()))
