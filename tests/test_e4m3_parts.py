"""Feed-forwards in 8 bits beside parts from elsewhere, without a GPU: who is handed rows in 8 bits, and what is said of a part that stays in
bfloat16."""
import types

import pytest
import torch

import harness as H  # noqa: F401  (path setup)
from lastengine_b200.engine.workspace import Workspace
from lastengine_b200.ops import kernels as K
from lastengine_b200.parts import base, block, ffn, norm

CPU = torch.device("cpu")


@pytest.fixture
def launched(monkeypatch):
    """The names of the norms launched, in the place of the kernels."""
    got = []
    monkeypatch.setattr(K, "rmsnorm_e4m3", lambda *a, **k: got.append("8 bits"))
    monkeypatch.setattr(K, "rmsnorm", lambda *a, **k: got.append("plain"))
    monkeypatch.setattr(K, "quantize_e4m3", lambda *a, **k: None)
    return got


def env():
    return base.BuildEnv(device=CPU, dtype=torch.bfloat16, workspace=Workspace(CPU), ffn_e4m3=True)


def loaded(part, e):
    part.load({n: torch.zeros(s.concrete_shape()) for n, s in part.tensors().items()}, e)
    return part


class Subclass(ffn.SwiGLU):
    def forward(self, h, out, accumulate, batch, env):
        assert isinstance(h, torch.Tensor) and h.shape == out.shape


class SaysSo(ffn.SwiGLU):
    reads_e4m3 = True

    def forward(self, h, out, accumulate, batch, env):
        assert isinstance(h, ffn.EightBitRows)


class WrappedNorm(norm.RMSNorm):
    def forward(self, out, x, rows=None, add=False):
        K.rmsnorm(out, x, self.weight, self.eps)


def handed(reader, n, e):
    """What a block hands `reader` behind the norm `n`."""
    b = block.PreNormResidualBlock(None, reader, None, n)
    return b._normed(n, torch.zeros(3, 64), None, e, reader)


def test_the_librarys_own_parts_are_handed_8_bits(launched):
    e = env()
    n = norm.RMSNorm(64, 1e-5)
    for part in (ffn.SwiGLU(64, 96), ffn.DenseFeedForward(64, 96)):
        assert isinstance(handed(loaded(part, e), n, e), ffn.EightBitRows)
    assert launched == ["8 bits", "8 bits"]
    assert isinstance(handed(loaded(ffn.SigmoidTopKMoE(64, 4, 2, 32), e), n, e), torch.Tensor)


def wrapped_on_the_object(part, monkeypatch):
    own = part.forward
    part.forward = lambda h, *a: own(h, *a)
    return part


def wrapped_on_the_class(part, monkeypatch):
    own = type(part).forward
    monkeypatch.setattr(type(part), "forward", lambda self, h, *a: own(self, h, *a))
    return part


def another_class(part, monkeypatch):
    part.__class__ = type("Elsewhere", (type(part),), {"forward": Subclass.forward})
    return part


@pytest.mark.parametrize("change", [wrapped_on_the_object, wrapped_on_the_class, another_class])
def test_what_is_wrapped_gets_tensors(change, launched, monkeypatch):
    e = env()
    n = norm.RMSNorm(64, 1e-5)
    part = change(loaded(ffn.SwiGLU(64, 96), e), monkeypatch)
    h = handed(part, n, e)
    assert isinstance(h, torch.Tensor) and h.dtype is torch.bfloat16 and launched == ["plain"]


def test_classes_from_elsewhere(launched):
    e = env()
    n = norm.RMSNorm(64, 1e-5)
    h = handed(loaded(Subclass(64, 96), e), n, e)
    assert isinstance(h, torch.Tensor)
    Subclass.forward(None, h, torch.zeros(3, 64), False, None, e)
    assert isinstance(handed(loaded(SaysSo(64, 96), e), n, e), ffn.EightBitRows)
    assert launched == ["plain", "8 bits"]


def test_a_norm_from_elsewhere_is_called(launched):
    e = env()
    part = loaded(ffn.SwiGLU(64, 96), e)
    assert isinstance(handed(part, WrappedNorm(64, 1e-5), e), torch.Tensor)
    n = norm.RMSNorm(64, 1e-5)
    own, seen = n.forward, []
    n.forward = lambda *a, **k: (seen.append(1), own(*a, **k))
    assert isinstance(handed(part, n, e), torch.Tensor)
    assert launched == ["plain", "plain"] and seen == [1]


def test_a_part_without_the_attribute(launched):
    """A feed-forward that is no subclass of the library's is called with tensors."""
    e = env()
    part = types.SimpleNamespace(forward=lambda *a: None)
    assert isinstance(handed(part, norm.RMSNorm(64, 1e-5), e), torch.Tensor)


def model(e, kind):
    """A model of four layers whose second feed-forward is `kind`, on the host."""
    import dataclasses
    from lastengine_b200 import registry
    from lastengine_b200.engine.model import Model
    from tiny_configs import TINY_A
    plan = registry.plan_from_config(TINY_A)
    ls = plan.layers[1]
    plan.layers[1] = dataclasses.replace(ls, ffn=dataclasses.replace(ls.ffn, kind=kind))
    m = Model(plan, e)
    m.load({n: torch.zeros(s.concrete_shape()) for n, s in m.tensor_specs().items()})
    return m


class StaysInBfloat16(ffn.SwiGLU):
    def load(self, tensors, env):
        self.w13, self.w2 = ffn.fuse_gate_up(tensors[self.n_gate], tensors[self.n_up], False), tensors[self.n_down]


@pytest.fixture
def registered():
    from lastengine_b200.registry import FEED_FORWARDS
    FEED_FORWARDS.register("stays_in_bfloat16", replace=True)(StaysInBfloat16)
    yield "stays_in_bfloat16"
    FEED_FORWARDS.unregister("stays_in_bfloat16")


def test_a_part_that_stays_in_bfloat16_is_named(launched, registered):
    with pytest.warns(UserWarning, match="StaysInBfloat16 did not bring its matrices"):
        m = model(env(), registered)
    assert [b.ffn.in_e4m3 for b in m.blocks] == [True, False, True, True]


@pytest.mark.parametrize("asked", [True, False])
def test_nothing_is_said_where_there_is_nothing_to_say(asked, launched, registered, recwarn):
    e = env()
    e.ffn_e4m3 = asked
    m = model(e, "swiglu" if asked else registered)
    assert not recwarn.list and [b.ffn.in_e4m3 for b in m.blocks] == [asked] * 4
