"""The paged serving example: requests that come and go through few rows, against the decoder's formulas over the
whole sequence so far, and its pages all back at the end. The formulas are computed in 64 bits and rounded to bf16
where the kernels store (the norms behind the mixer and the MLP blow up the roundings of small projections, so a
reference without them is several percent away).

Tolerance: about 25 bf16 roundings lie on the way to a logit of the two-layer model (a dozen a layer), each 2^-9 / sqrt 3
of its value in the mean: sqrt(25) * 1.1e-3 = 0.6% of the logits' size, allowed eight times for what the norms add. A
wrong page, position or mask is of the logits' own size."""
import importlib.util
import sys

import numpy as np
import pytest

from conftest import REPO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def serving():
    torch = pytest.importorskip("torch")
    if not torch.cuda.is_available():
        pytest.skip("CUDA device required")
    spec = importlib.util.spec_from_file_location("paged_serving", REPO / "examples" / "paged_serving.py")
    sys.modules["paged_serving"] = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(sys.modules["paged_serving"])
    return sys.modules["paged_serving"]


def reference_logits(torch, engine, ids, freq):
    """The last position's logits of the decoder over `ids`, in 64 bits, rounded where the kernels store."""
    c, w = engine.cfg, {k: v.double() for k, v in engine.weights.items()}
    n, heads, kv, dim = len(ids), c.num_attention_heads, c.num_key_value_heads, c.head_dim
    bf = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
    unit = lambda x: x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    norm = lambda x, g, off: bf(bf(unit(x)) * bf(g + off))  # noqa: E731
    x = w["model.embed_tokens.weight"][torch.tensor(ids, device="cuda")]
    pos = torch.arange(n, device="cuda", dtype=torch.float64)
    for i in range(c.num_hidden_layers):
        layer = lambda name: w[f"model.layers.layers.{i}.{name}.weight"]  # noqa: E731,B023
        full = c.is_global(i)
        angle = pos[:, None] * torch.tensor(freq["full" if full else "local"], device="cuda", dtype=torch.float64)
        scale = 1.5545177444479562 if full else 1.0
        cos, sin = bf(angle.cos() * scale)[:, None], bf(angle.sin() * scale)[:, None]
        h = bf(norm(x, layer("pre_mixer_norm"), 1.0) @ layer("mixer.qkv_proj").T).view(n, heads + 2 * kv, dim)
        q, k, v = h[:, :heads], h[:, heads:heads + kv], h[:, heads + kv:]

        def turn(t, g):
            t = unit(t) * (g + 1.0)
            a, b = t[..., :dim // 2], t[..., dim // 2:]
            return bf(torch.cat([a * cos - b * sin, b * cos + a * sin], -1))  # noqa: B023

        q, k = turn(q, layer("mixer.q_norm")), turn(k, layer("mixer.k_norm"))
        k, v = (t.repeat_interleave(heads // kv, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * dim ** -0.5
        back = pos[:, None] - pos[None]
        seen = (back >= 0) & (back < (n + 1 if full else c.window_size))
        o = bf(torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(~seen, -torch.inf), -1), v).reshape(n, -1))
        x = bf(x + norm(bf(o @ layer("mixer.o_proj").T), layer("post_mixer_norm"), 0.2))
        g, u = bf(norm(x, layer("pre_mlp_norm"), 1.0) @ layer("mlp.gate_up_proj").T).chunk(2, -1)
        act = bf(bf(torch.nn.functional.silu(g)) * u)
        x = bf(x + norm(bf(act @ layer("mlp.down_proj").T), layer("post_mlp_norm"), 5.0 ** -1.5))
    return bf(norm(x[-1], w["model.norm.weight"], 1.0) @ w["lm_head.weight"].T)


def test_requests_come_and_go(serving, micro_dir, pkg):
    import json

    import torch
    engine = serving.Engine(micro_dir, rows=3, pages=40, page_size=8, context=160, tokens=128)
    freq = json.loads((micro_dir / "config-mlx.json").read_text())["plamo_rope_inv_freq"]
    prompts = [pkg.synthetic.seeded_tokens(n, engine.cfg.vocab_size, seed=n) for n in (1, 40, 7, 16, 90, 23)]
    answers, checked = [list() for _ in prompts], 0

    def check(eng, running):
        nonlocal checked
        ids = eng.ids.tolist()
        for r, i in enumerate(running):
            if i is None:
                continue
            want = reference_logits(torch, eng, prompts[i] + answers[i], freq)
            got = eng.logits[r].double()
            err, size = float((got - want).square().mean().sqrt()), float(want.square().mean().sqrt())
            assert err <= 0.05 * size, (i, len(answers[i]), err / size)
            assert ids[r] == int(eng.logits[r].float().argmax())  # greedy: no temperature given below
            answers[i].append(ids[r])
            checked += 1

    controls = [(0.0, 0, 1.0, 0.0)] * len(prompts)
    got = serving.serve(engine, prompts, 30, controls, check)
    assert got == answers and all(len(a) == 30 for a in got) and checked == 30 * len(prompts)
    engine.plan([-1] * engine.rows)  # the last requests' pages
    assert int(engine.counts[0][0]) == engine.pages
    assert sorted(engine.free_list.tolist()) == list(range(engine.pages))


def test_sampled_ids_follow_their_controls(serving, micro_dir, pkg):
    import torch
    engine = serving.Engine(micro_dir, rows=4, pages=64, page_size=16, context=128, tokens=256)
    prompts = [pkg.synthetic.seeded_tokens(20, engine.cfg.vocab_size, seed=9)] * 8
    torch.manual_seed(3)
    ranks = []

    def look(eng, running):
        for r, i in enumerate(running):
            if i is not None:
                order = eng.logits[r].float().argsort(descending=True, stable=True)
                ranks.append(int((order == eng.ids[r]).nonzero()))

    answers = serving.serve(engine, prompts, 12, [(1.0, 5, 1.0, 0.0)] * 8, look)
    assert len(ranks) == 96 and max(ranks) < 5 and len(set(ranks)) > 2
    assert len({tuple(a) for a in answers}) > 1  # the same prompt, other uniform numbers


def test_too_few_pages_are_reported(serving, micro_dir, pkg):
    engine = serving.Engine(micro_dir, rows=2, pages=3, page_size=8, context=64, tokens=64)
    with pytest.raises(RuntimeError, match="got no pages"):
        serving.serve(engine, [list(range(30))], 4)
    assert np.array_equal(engine.lens[0].cpu().numpy(), [0, 0])
