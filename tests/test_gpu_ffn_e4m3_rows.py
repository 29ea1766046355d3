"""Feed-forwards and experts in 8 bits, number by number and row by row: every stage of a part against the definition on what the stage before left,
and whole models of every architecture against their own 32-bit path, a row at a time."""
import pytest
import torch

import harness as H  # noqa: F401  (path setup)
import plain_e4m3 as P
from test_gpu_e4m3 import check_rows
from test_gpu_ffn_e4m3 import DEV, MAKE, env_of, parts
from test_product_chain import CONFIGS

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def numbers(rows):
    """(the 8-bit numbers, the scales) as the definitions take them."""
    return rows[0].float().cpu().double(), rows[1].cpu()


def product(x, w, expert=None):
    """The scaled product in double and how far float sums of its terms may be off (a tensor core cuts, so a step of 2^-23 a term); rows of expert
    expert[m] each, or all of the one matrix."""
    (q, s), (qw, sw) = x, w
    if expert is None:
        z, size = P.product(q, s, qw, sw)
    else:
        z, size = (torch.empty(q.shape[0], qw.shape[1], dtype=torch.float64) for _ in range(2))
        for e in expert.unique().tolist():
            z[expert == e], size[expert == e] = P.product(q[expert == e], s[expert == e], qw[e], sw[e])
    return z, (q.shape[1] + 4) * 2.0 ** -23 * size


def halves(z, interleaved):
    """(gate, up) columns."""
    if interleaved:
        b = z.reshape(z.shape[0], -1, 2, 16)
        return b[:, :, 0].reshape(z.shape[0], -1), b[:, :, 1].reshape(z.shape[0], -1)
    return z.chunk(2, 1)


def check_activated(part, a, z, dz):
    """`a` (bfloat16) is the activation of z, which the kernels have within dz.  The activations' slopes are at most 1.2 in either factor (a
    square's is 2 z); half a step of bfloat16; the float arithmetic of the activation itself 2^-19, and where tanh comes from the special
    function unit (gelu for bfloat16) 2^-10."""
    names = {v: k for k, v in parts()._ACTIVATIONS.items()} if getattr(part, "gated", True) else {}
    got = a.cpu().double()
    if getattr(part, "gated", True) and part.__class__.__name__ != "DenseFeedForward":
        (g, u), (dg, du) = halves(z, part.fused), halves(dz, part.fused)
        act = names[part.act]
        if act == "clamped_sigmoid":
            gc, uc = g.clamp(max=part.limit), u.clamp(-part.limit, part.limit)
            want = gc * torch.sigmoid(part.alpha * gc) * (uc + 1)
        else:
            want = (g * torch.sigmoid(g) if act == "silu" else P.gelu_tanh(g)) * u
        unit = 2.0 ** -10 if act == "gelu_tanh" else 2.0 ** -19
        far = 1.2 * (dg * (u.abs() + 1 + du) + g.abs() * du) + unit * g.abs() * (u.abs() + 1)
    else:
        from lastengine_b200.ops import kernels
        act = {v: k for k, v in kernels.PLAIN_ACTIVATIONS.items()}[part.act]
        want = P.PLAIN[act](z)
        far = (2 * z.abs() + dz) * dz + 2.0 ** -19 * want.abs() if act == "relu_squared" else 1.2 * dz + 2.0 ** -19 * z.abs()
    assert bool(((got - want).abs() <= 2.0 ** -8 * 1.01 * want.abs() + far + 1e-30).all()), act


def stored(part, tensors):
    """The part's matrices as they were given, rows in the order in which they are kept, and what is kept."""
    def first(gate, up):
        if gate is None:
            return up
        if not part.fused:
            return torch.cat([gate, up])
        return torch.stack([gate.reshape(-1, 16, gate.shape[1]), up.reshape(-1, 16, up.shape[1])], 1).reshape(-1, gate.shape[1])
    kind = type(part).__name__
    if kind == "SwiGLU":
        return (first(tensors[part.n_gate], tensors[part.n_up]), (part.w13, part.s13)), (tensors[part.n_down], (part.w2, part.s2))
    if kind == "DenseFeedForward":
        return (tensors[part.n_up], (part.w1, part.s1)), (tensors[part.n_down], (part.w2, part.s2))
    n = part.n
    one = torch.cat([first(tensors[n["gate"].format(e=e)] if part.gated else None, tensors[n["up"].format(e=e)]) for e in range(part.E)])
    return (one, (part.w13, part.s13)), (torch.cat([tensors[n["down"].format(e=e)] for e in range(part.E)]), (part.w2, part.s2))


def check_dense(part, h, ws, out, before=None, before_far=0.0):
    """A dense feed-forward's stages for rows h; `before`: what was in `out` already, and how far it may be off."""
    f = parts()
    M = h.shape[0]
    x, a = f.eight_bit_room(ws, "ffn.h8", M, part.D), ws.get("ffn.a", (M, part.F), BF16)
    a8 = f.eight_bit_room(ws, "ffn.a8", M, part.F)
    check_rows(x.values, x.scale, h.float().cpu())
    w1, w2 = ((part.w13, part.s13) if hasattr(part, "w13") else (part.w1, part.s1)), (part.w2, part.s2)
    check_activated(part, a, *product(numbers(x), numbers(w1)))
    check_rows(a8.values, a8.scale, a.float().cpu())
    z, dz = product(numbers(a8), numbers(w2))
    if before is not None:
        z = z + before
        dz = dz + before_far
    assert bool(((out.cpu().double() - z).abs() <= dz + 2.0 ** -23 * z.abs()).all())


@pytest.mark.parametrize("M", [1, 3, 40, 300, 1100])
@pytest.mark.parametrize("name", MAKE)
def test_every_stage_of_a_part(name, M):
    f = parts()
    g = torch.Generator(device=DEV).manual_seed(3)
    part = MAKE[name](f)
    tensors = {}
    for n, spec in part.tensors().items():
        t = torch.randn(spec.shape, generator=g, device=DEV) * (0.1 if len(spec.shape) == 1 else spec.shape[-1] ** -0.5)
        tensors[n] = t if spec.role in ("vector", "bias") else t.to(BF16)
    env = env_of(True)
    part.load({k: v.clone() for k, v in tensors.items()}, env)
    for given, (q, s) in stored(part, tensors):
        check_rows(q.float().cpu().reshape(given.shape), s.cpu().reshape(-1), given.float().cpu())
    h = torch.randn(M, part.D, generator=g, device=DEV).to(BF16)
    out = torch.full((M, part.D), 0.5, device=DEV)
    part.forward(h, out, False, None, env)
    ws = env.workspace
    if type(part).__name__ != "SigmoidTopKMoE":
        check_dense(part, h, ws, out)
        return
    Pn = M * part.k
    ids, wts = ws.get("moe.ids", (M, part.k), torch.int32).cpu(), ws.get("moe.w", (M, part.k), F32).cpu().double()
    offsets, order = ws.get("moe.offsets", (part.E + 1,), torch.int32).cpu(), ws.get("moe.sorted", (Pn,), torch.int32).cpu().long()
    assert torch.equal(order.sort().values, torch.arange(Pn)) and int(offsets[0]) == 0 and int(offsets[-1]) == Pn
    expert = ids.reshape(-1)[order].long()
    assert torch.equal(expert, torch.repeat_interleave(torch.arange(part.E), offsets.long().diff()))
    x, a, a8 = f.eight_bit_room(ws, "moe.x8", Pn, part.D), ws.get("moe.a", (Pn, part.Fe), BF16), f.eight_bit_room(ws, "moe.a8", Pn, part.Fe)
    check_rows(x.values, x.scale, h.float().cpu()[order // part.k], wts.reshape(-1)[order] if part.weight_input else None)
    check_activated(part, a, *product(numbers(x), numbers((part.w13, part.s13)), expert))
    check_rows(a8.values, a8.scale, a.float().cpu())
    z, dz = product(numbers(a8), numbers((part.w2, part.s2)), expert)
    weight = torch.ones(Pn, dtype=torch.float64) if part.weight_input else wts.reshape(-1)[order]
    want, far, size = (torch.zeros(M, part.D, dtype=torch.float64) for _ in range(3))
    want.index_add_(0, order // part.k, z * weight[:, None])
    far.index_add_(0, order // part.k, dz * weight.abs()[:, None])
    size.index_add_(0, order // part.k, z.abs() * weight.abs()[:, None])
    far += (part.k + 1) * 2.0 ** -23 * size                     # the weighted sum's own roundings
    if part.shared is not None:
        check_dense(part.shared, h, ws, out, want, far)
    else:
        assert bool(((out.cpu().double() - want).abs() <= far + 1e-30).all())


# ---- whole models ----------------------------------------------------------------------------------------------------
def chosen(eng, seen):
    """Notes the experts that every layer chooses, sorted (other code around a part: it gets tensors)."""
    for b in eng.model.blocks:
        part = getattr(b, "ffn", None)
        if type(part).__name__ == "SigmoidTopKMoE":
            def spy(h, out, accumulate, batch, env, part=part, own=part.forward):
                own(h, out, accumulate, batch, env)
                seen.append(env.workspace.get("moe.ids", (h.shape[0], part.k), torch.int32).sort(1).values.clone())
            part.forward = spy


# A number rounded to 8 bits is off by half a step at most, even over +- 2^-4 / m of its size for a fraction m from 1 to 2: a root mean square of
# 2^-4 / sqrt(3) (3 / (8 ln 2))^(1/2) = 2.65%.  Rows and weights together put a product off by sqrt(2) times that, 3.75% of its typical size; a gated
# activation has two such factors with slopes of up to 1.13 (6%), a square has the slope 2 (10% of a square's typical size); the last product adds
# 3.75%.  So a feed-forward's result is off by 7 to 11% of its own size, in independent directions, and the median row of logits, which the
# streams' other parts make smaller and later layers about as large again, by 1/8 at most.
TYPICAL, NOISE = 1 / 8, 0.11
# What that is in one row's logits depends on the row: some streams cancel, and what is left of them shows the same error larger.  It is measured
# in 32 bits, by independent normal errors of that size on every feed-forward's result, 16 times.  To first order a row's error is a sum of
# many independent parts with the same covariance, so that it is beyond 5 times its root mean square in less than one of a million
# rows; a root mean square of 16 draws is itself off by a factor of 6/5 at most, but for one in some hundred.
TIMES, DRAWS = 6.0, 16


def disturbed(eng, gen):
    """Puts such errors on what the feed-forwards of `eng` give, from now on."""
    for b in eng.model.blocks:
        part = getattr(b, "ffn", None)
        if part is not None:
            def noisy(h, out, accumulate, batch, env, own=part.forward):
                t = torch.zeros_like(out)
                own(h, t, False, batch, env)
                t += NOISE * t.square().mean(1, keepdim=True).sqrt() * torch.randn(t.shape, generator=gen, device=t.device)
                out.copy_(out + t if accumulate else t)
            part.forward = noisy


def check_logits(name, eight, exact, far_of, same=None):
    """The rows' distances to the 32-bit path against what such errors make of them there."""
    far = (eight - exact).norm(dim=1) / exact.norm(dim=1)
    rms = torch.stack([((z - exact).norm(dim=1) / exact.norm(dim=1)).square() for z in far_of]).mean(0).sqrt()
    same = torch.ones_like(far, dtype=torch.bool) if same is None else same
    print(name, "rows", int(same.sum()), "median", float(far[same].median()), "most", float(far[same].max()), "against errors in 32 bits", float((far / rms)[same].max()))
    assert float(far[same].median()) < TYPICAL
    assert bool((far <= TIMES * rms)[same].all())


def folder(cfg, path):
    """Random weights; those of the feed-forwards are brought to the size that keeps a row's, so that they make up most of the stream."""
    from lastengine_b200.engine.model import Model
    from lastengine_b200.engine.workspace import Workspace
    from lastengine_b200.parts.base import MATRIX, BuildEnv, FeedForward
    from lastengine_b200.registry import plan_from_config
    from lastengine_b200.weights import write_model_dir
    from lastengine_b200.weights.safetensors_io import SafetensorsFile, save_file
    write_model_dir(cfg, path, seed=4, dtype="bfloat16", norm_init="random")
    sf = SafetensorsFile(path + "/model.safetensors")
    t = {n: sf.tensor(n).clone() for n in sf.names()}
    m = Model(plan_from_config(cfg), BuildEnv(device=torch.device("cpu"), dtype=BF16, workspace=Workspace(torch.device("cpu"))))
    scaled = 0
    for prefix, part in m.named_parts():
        for rel, spec in part.tensors().items() if isinstance(part, FeedForward) else ():
            n = m._name(prefix, rel, spec)
            n = n if n in t else f"model.{n}"                   # (as one architecture's folders name them)
            if spec.role == MATRIX and n in t:
                t[n] = (t[n].float() * (t[n].shape[-1] ** -0.5 / t[n].float().std())).to(t[n].dtype)
                scaled += 1
    del sf
    save_file(t, path + "/model.safetensors")
    return scaled


@pytest.mark.parametrize("name", sorted(CONFIGS))
def test_a_models_logits_row_by_row(name, tmp_path):
    """The same weights in 8 bits and in 32, every architecture: one token each of 100 sequences (a row depends on nothing but itself; rows for
    which some layer chose other experts are left out), and without experts a prompt as well."""
    from lastengine_b200 import Engine
    d = str(tmp_path / "m")
    if not folder(CONFIGS[name], d):
        pytest.skip("a model without feed-forwards")
    eight, exact = Engine.from_pretrained(d, ffn_dtype="e4m3", max_tokens=8192), Engine.from_pretrained(d, dtype="float32", max_tokens=8192)
    layers = [b.ffn for b in eight.model.blocks if getattr(b, "ffn", None) is not None]
    assert layers and all(f.in_e4m3 for f in layers)
    experts = any(type(f).__name__ == "SigmoidTopKMoE" for f in layers)
    tokens = [[(7 * i + 3) % eight.vocab_size] for i in range(100)]
    prompt = [(11 * i + 5) % eight.vocab_size for i in range(50)]
    ids: dict = {eight: [], exact: []}

    def ones(eng):
        seqs = [eng.new_sequence() for _ in tokens]
        z = eng.step(seqs, tokens, "last", check=True).clone().double()
        eng.release(seqs)
        return z

    def rows(eng):
        seq = eng.new_sequence()
        z = eng.step([seq], [prompt], want=[list(range(50))], check=True).clone().double()
        eng.release(seq)
        return z
    if not experts:
        prompts = rows(eight), rows(exact)
    for eng in (eight, exact):
        chosen(eng, ids[eng])
    got, want = ones(eight), ones(exact)
    same = torch.ones(100, dtype=torch.bool, device=DEV)
    for a, b in zip(ids[eight], ids[exact], strict=True):
        same &= (a == b).all(1)
    assert int(same.sum()) >= 10
    disturbed(exact, torch.Generator(device=DEV).manual_seed(1))
    check_logits(name, got, want, [ones(exact) for _ in range(DRAWS)], same)
    if not experts:
        check_logits(name + ", a prompt", *prompts, [rows(exact) for _ in range(DRAWS)])
