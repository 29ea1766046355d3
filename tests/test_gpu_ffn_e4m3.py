"""Feed-forwards and experts with their matrices in 8 bits: each part against itself in bfloat16, and engines that run them."""
import pytest
import torch

import harness as H
from lenesun_configs import L_A
from tiny_configs import TINY_A, TINY_B, TINY_C

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def parts():
    from lastengine_b200.parts import ffn
    return ffn


def env_of(eight):
    from lastengine_b200.engine.workspace import Workspace
    from lastengine_b200.parts.base import BuildEnv
    return BuildEnv(device=DEV, dtype=BF16, workspace=Workspace(DEV), ffn_e4m3=eight)


MAKE = {
    "swiglu": lambda f: f.SwiGLU(128, 320),
    "gelu": lambda f: f.SwiGLU(128, 320, "gelu_tanh"),
    "clamped": lambda f: f.SwiGLU(128, 320, "clamped_sigmoid", limit=7.0, alpha=1.702),
    "clamped, a slope of its own": lambda f: f.SwiGLU(128, 320, "clamped_sigmoid", limit=7.0, alpha=1.5),
    "odd sizes": lambda f: f.SwiGLU(104, 150),
    "dense": lambda f: f.DenseFeedForward(128, 300),
    "dense, squared relu": lambda f: f.DenseFeedForward(100, 256, "relu_squared"),
    "experts": lambda f: f.SigmoidTopKMoE(128, 12, 3, 96),
    "experts, weighted rows": lambda f: f.SigmoidTopKMoE(128, 12, 3, 96, weight_input=True),
    "experts, softmax, odd": lambda f: f.SigmoidTopKMoE(104, 8, 2, 50, router="softmax_chosen", activation="clamped_sigmoid", limit=7.0, alpha=1.702),
    "experts and a shared one": lambda f: f.SigmoidTopKMoE(128, 8, 4, 64, router="softmax_grouped", groups=(4, 2), shared_size=160),
    "experts without gates": lambda f: f.SigmoidTopKMoE(128, 8, 2, 96, router="sigmoid_grouped", groups=(2, 1), activation="relu_squared", gated=False),
}


@pytest.mark.parametrize("name", MAKE)
def test_a_part_in_8_bits(name):
    """Four roundings to 8 bits stand between the two: of the input, the first matrix, the activation's result and the last matrix.  Each is
    off by half a step of 2^-4 at most, and some 2.6% over many numbers; the products are linear, the gated activations' slopes up to
    1.13 for either factor (a square's is 2).  Wrong rows, scales or experts would be off by about as much as the result is large."""
    f = parts()
    g = torch.Generator(device=DEV).manual_seed(3)
    one = MAKE[name](f)
    tensors = {}
    for n, spec in one.tensors().items():
        t = torch.randn(spec.shape, generator=g, device=DEV) * (0.1 if len(spec.shape) == 1 else spec.shape[-1] ** -0.5)
        tensors[n] = t if spec.role in ("vector", "bias") else t.to(BF16)
    envs = {eight: env_of(eight) for eight in (False, True)}
    made = {}
    for eight, env in envs.items():
        made[eight] = MAKE[name](f)
        made[eight].load({k: v.clone() for k, v in tensors.items()}, env)
    for M in (1, 3, 40, 300):
        h = torch.randn(M, one.D, generator=g, device=DEV).to(BF16)
        out = {}
        for eight, part in made.items():
            for accumulate in (False, True):
                o = torch.full((M, one.D), 0.5, device=DEV)
                part.forward(h, o, accumulate, None, envs[eight])
                out[eight, accumulate] = o
        # (one float addition each: what is added differs from what is stored by its roundings)
        assert float((out[True, True] - 0.5 - out[True, False]).abs().max()) <= 2.0 ** -22 * (1 + float(out[True, False].abs().max()))
        far = float((out[True, False] - out[False, False]).norm() / out[False, False].norm())
        assert far < 4 * 2.0 ** -4, (name, M, far)
        assert far > 1e-3                                    # it did run in 8 bits
    if getattr(made[True], "reads_e4m3", False):             # rows that a norm has brought to 8 bits are taken as they are
        from lastengine_b200.ops import kernels
        q, s = kernels.e4m3_rows(300, one.D, device=DEV), torch.empty(300, device=DEV)
        kernels.quantize_e4m3(q, s, h)
        o = torch.empty(300, one.D, device=DEV)
        made[True].forward(f.EightBitRows(q, s), o, False, None, envs[True])
        assert torch.equal(o, out[True, False])
    assert made[True].w13.dtype is E4M3 if hasattr(made[True], "w13") else made[True].w1.dtype is E4M3


@pytest.mark.parametrize("cfg", [TINY_A, TINY_B, TINY_C, L_A], ids=["A", "B", "C", "lenesun"])
def test_an_engine_in_8_bits(cfg):
    """The same requests give the same tokens with and without captured steps, whole and cut; the weights take less room."""
    from lastengine_b200 import Engine, SamplingParams
    eng = Engine.from_config(cfg, seed=5, ffn_dtype="e4m3", max_tokens=2048)
    base = Engine.from_config(cfg, seed=5, max_tokens=2048)
    assert eng.weight_bytes() < base.weight_bytes()
    prompts = [[3, 1, 4, 1, 5, 9, 2, 6], [2, 7, 1], [8] * 30]
    greedy = SamplingParams(temperature=0.0)
    with_graphs = eng.generate(prompts, greedy, max_new_tokens=12, use_graphs=True).tokens
    without = eng.generate(prompts, greedy, max_new_tokens=12, use_graphs=False).tokens
    assert with_graphs == without and all(len(t) == 12 for t in with_graphs)
    # a prompt as one step against a prompt row by row: the norm and the activations are rounded per row, so only the sums' order differs,
    # which may move a number to the next one of 8 bits (2^-4 apart, half a step of the sums' own roundings in bfloat16)
    s, t = eng.new_sequence(), base.new_sequence()
    whole, plain = eng.step([s], [prompts[2]], want=[list(range(len(prompts[2])))]).clone(), base.step([t], [prompts[2]], want=[list(range(len(prompts[2])))]).clone()
    assert bool(whole.isfinite().all()) and not torch.equal(whole, plain)
    if any(type(b.ffn).__name__ == "SigmoidTopKMoE" for b in eng.model.blocks):
        return                                               # (a router's near-tie may choose another expert)
    u = eng.new_sequence()
    rows = torch.cat([eng.step([u], [[p]], want="last").clone() for p in prompts[2]])
    assert float((rows - whole).norm() / whole.norm()) < 2.0 ** -4


def test_the_norm_in_8_bits_gives_what_the_norm_and_its_rounding_give():
    """A dense layer whose norm leaves its rows in 8 bits against one whose feed-forward brings them there: the latter's rows are rounded
    to bfloat16 first, 2^-8 at most, which moves some of them by one step of 2^-4 at the feed-forward's input."""
    from lastengine_b200 import Engine
    eng = Engine.from_config(TINY_A, seed=5, ffn_dtype="e4m3", max_tokens=1024)
    tokens = [[5, 4, 3, 2, 1] * 8]
    s = eng.new_sequence()
    fused = eng.step([s], tokens, want=[list(range(40))]).clone()
    dense = [b.ffn for b in eng.model.blocks if getattr(b.ffn, "reads_e4m3", False)]
    assert dense
    for f in dense:
        f.reads_e4m3 = False
    t = eng.new_sequence()
    apart = eng.step([t], tokens, want=[list(range(40))]).clone()
    assert not torch.equal(fused, apart)
    assert float((fused - apart).norm() / fused.norm()) < len(dense) * 2.0 ** -4


def test_options_that_do_not_go_together():
    from lastengine_b200 import Engine
    with pytest.raises(ValueError, match="bfloat16"):
        Engine.from_config(TINY_A, seed=0, dtype="float32", ffn_dtype="e4m3")
    with pytest.raises(ValueError, match="e5m2"):
        Engine.from_config(TINY_A, seed=0, ffn_dtype="e5m2")


def test_generate_from_the_command_line(tmp_path, capsys):
    import json
    from lastengine_b200.cli import main
    p = tmp_path / "config.json"
    p.write_text(json.dumps(TINY_A))
    assert main(["generate", "--config", str(p), "--prompt-ids", "1,2,3", "--max-new-tokens", "4", "--temperature", "0", "--ffn-dtype", "e4m3"]) == 0
    assert len(json.loads(capsys.readouterr().out.splitlines()[0])["tokens"]) <= 4
