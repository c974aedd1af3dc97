"""Serving a changing set of requests from one paged key-value cache, with sampled ids.

    python examples/paged_serving.py [--model DIR] [--requests 12] [--rows 4] [--new-tokens 32]

A step takes the next tokens of every running request (a whole prompt, or the id it got last) through the decoder
with the kernel-level entry points (include/plamo_kernels.h): one plan gives the tokens their pages and slots,
every layer appends its keys and values to its own cache by the same slots and attends over the pages, and the last
hidden row of every request becomes an id by its own controls. Requests come and go between steps; the pages of an
ended one return to the free list in the plan of the step after. Only the ids and the number of refused requests
leave the device.

Without --model, a small synthetic model is written to a temporary directory.
"""
from __future__ import annotations

import argparse
import importlib.util
import json
import struct
import sys
import tempfile
import time
from pathlib import Path

import numpy as np
import torch

PKG = Path(__file__).resolve().parents[1] / "plamo3-0.8b-runtime_b200"
ROPE_SCALE = 1.5545177444479562  # of the full-history layers' cosines and sines (rope_scaling_factor 256)
POST_MIXER, POST_MLP = 0.2, 5.0 ** -1.5  # weight offsets of the norms behind the mixer and the MLP


def package():
    if "plamo_b200" not in sys.modules:
        spec = importlib.util.spec_from_file_location("plamo_b200", PKG / "__init__.py", submodule_search_locations=[str(PKG)])
        sys.modules["plamo_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["plamo_b200"])
    return sys.modules["plamo_b200"]


def load_weights(directory) -> dict:
    """The bf16 tensors of model.safetensors on the device."""
    path = Path(directory) / "model.safetensors"
    with open(path, "rb") as f:
        size = struct.unpack("<Q", f.read(8))[0]
        header = json.loads(f.read(size))
    data = np.memmap(path, dtype=np.uint8, mode="r", offset=8 + size)
    out = {}
    for name, info in header.items():
        if name != "__metadata__":
            begin, end = info["data_offsets"]
            bits = torch.from_numpy(np.array(data[begin:end]).view(np.int16))
            out[name] = bits.view(torch.bfloat16).reshape(info["shape"]).cuda()
    return out


def rope_table(inv_freq, rows, scale=1.0):
    """bf16 cosine and sine of every position and frequency in one word: cos | sin << 16."""
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * torch.tensor(inv_freq, dtype=torch.float64)
    bits = [(t * scale).to(torch.bfloat16).view(torch.int16).to(torch.int32) & 0xFFFF for t in (angle.cos(), angle.sin())]
    return (bits[0] | (bits[1] << 16)).cuda()


class Engine:
    """A decoder over a paged cache for up to `rows` requests at a time."""

    def __init__(self, directory, rows=4, pages=256, page_size=16, context=1024, tokens=512):
        self.rt, synthetic = package().runtime, package().synthetic
        self.cfg = c = synthetic.read_config(directory)
        self.weights = load_weights(directory)
        freq = json.loads((Path(directory) / "config-mlx.json").read_text())["plamo_rope_inv_freq"]
        self.ropes = (rope_table(freq["local"], context), rope_table(freq["full"], context, ROPE_SCALE))
        self.rows, self.pages, self.page_size, self.context, self.tokens = rows, pages, page_size, context, tokens
        self.width = -(-context // page_size)
        ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device="cuda")  # noqa: E731
        half = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        kv, dim = c.num_key_value_heads, c.head_dim
        self.caches = []
        for _ in range(c.num_hidden_layers):
            keys, values = (half(pages, page_size, kv, dim) for _ in range(2))
            self.caches.append((keys, values, self.rt.PagedCache(keys.data_ptr(), values.data_ptr(), 0, pages, page_size, kv, dim,
                                                                 page_size * kv * dim, kv * dim, dim)))
        self.table, self.free_list = ints(rows, self.width) - 1, torch.arange(pages, dtype=torch.int32, device="cuda")
        # a step reads one set of lengths and counts and writes the other
        self.lens, self.counts = [ints(rows), ints(rows)], [ints(4) + pages, ints(4)]
        self.row_start, self.slots, self.positions = ints(rows + 1), ints(tokens), ints(tokens)
        self.workspace = torch.empty(self.rt.paged_attention_workspace(), dtype=torch.uint8, device="cuda")
        self.ids, self.kept = ints(rows), ints(rows)
        self.logprobs = torch.zeros(rows, device="cuda")
        self.logits = half(rows, c.vocab_size)
        d, f = c.hidden_size, c.intermediate_size
        self.h, self.proj, self.act = half(tokens, d), half(tokens, d), half(tokens, f)
        self.qkv, self.q, self.att = half(tokens, c.qkv_rows), half(tokens, c.q_dim), half(tokens, c.q_dim)

    def plan(self, append):
        """Pages and slots for append[r] tokens of every request (-1: it has ended)."""
        t_append = torch.tensor(append, dtype=torch.int32, device="cuda")
        old, new = self.lens
        self.rt.k_paged_plan(old.data_ptr(), t_append.data_ptr(), self.rows, self.page_size, self.pages, self.table.data_ptr(),
                             self.width, self.free_list.data_ptr(), self.counts[0].data_ptr(), new.data_ptr(),
                             self.row_start.data_ptr(), self.slots.data_ptr(), self.positions.data_ptr(), self.tokens,
                             self.counts[1].data_ptr())
        self.lens.reverse()
        self.counts.reverse()

    def step(self, append, ids, temperature=None, top_k=None, top_p=None, min_p=None, u=None):
        """One step: append[r] next tokens of every request, packed in `ids`. The next id of every request (those
        without tokens keep their last). Controls are device tensors with a value a request, or None."""
        rt, c, w = self.rt, self.cfg, self.weights
        p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        n = len(ids)
        if n != sum(max(0, a) for a in append) or n > self.tokens:
            raise ValueError(f"{n} ids for {append}, at most {self.tokens} a step")
        self.plan(append)
        if n == 0:
            return self.ids
        lens, row_start, table = self.lens[0], self.row_start, self.table
        rows, q_rows = self.rows, n
        if max(append) > 1:
            # prompts: every token is a request of its own that sees the keys up to its own
            owner = torch.tensor([r for r, a in enumerate(append) for _ in range(max(0, a))], device="cuda")
            lens, table, row_start, rows = self.positions[:n] + 1, self.table[owner].contiguous(), None, n
        kv, heads, dim, d, f = c.num_key_value_heads, c.num_attention_heads, c.head_dim, c.hidden_size, c.intermediate_size
        x = w["model.embed_tokens.weight"][torch.tensor(ids, device="cuda")].contiguous()
        rt.k_norm(p(w["model.layers.layers.0.pre_mixer_norm.weight"]), p(x), p(self.h), n, d, 1.0, 0)
        for i, (_, _, cache) in enumerate(self.caches):
            layer = lambda name: p(w[f"model.layers.layers.{i}.{name}.weight"])  # noqa: E731,B023
            full = c.is_global(i)
            rt.k_linear(layer("mixer.qkv_proj"), 0, p(self.h), n, d, c.qkv_rows, 0, p(self.qkv))
            rt.k_paged_qkv(cache, p(self.qkv), c.qkv_rows, n, heads, layer("mixer.q_norm"), layer("mixer.k_norm"), 1e-6,
                           p(self.ropes[full]), self.context, p(self.positions), p(self.slots), p(self.q), c.q_dim)
            rt.k_paged_attention(cache, p(self.q), c.q_dim, q_rows, heads, p(table), self.width, p(lens), rows, p(row_start),
                                 self.context, 0 if full else c.window_size, dim ** -0.5, p(self.att), c.q_dim, 0,
                                 p(self.workspace), self.workspace.numel())
            rt.k_linear(layer("mixer.o_proj"), 0, p(self.att), n, c.q_dim, d, 0, p(self.proj))
            rt.k_norm(layer("post_mixer_norm"), p(self.proj), p(x), n, d, POST_MIXER, 1, layer("pre_mlp_norm"), p(self.h))
            rt.k_linear(layer("mlp.gate_up_proj"), 0, p(self.h), n, d, 2 * f, 1, p(self.act))
            rt.k_linear(layer("mlp.down_proj"), 0, p(self.act), n, f, d, 0, p(self.proj))
            last = i + 1 == c.num_hidden_layers
            after = 0 if last else p(w[f"model.layers.layers.{i + 1}.pre_mixer_norm.weight"])
            rt.k_norm(layer("post_mlp_norm"), p(self.proj), p(x), n, d, POST_MLP, 1, after, 0 if last else p(self.h))
        # the last row of every request; one without tokens repeats a row, and its id is put back
        idle = torch.tensor([a <= 0 for a in append], device="cuda")
        hidden = x[(self.row_start[1:].long() - 1).clamp(min=0)].contiguous()
        rt.k_norm(p(w["model.norm.weight"]), p(hidden), p(self.h), self.rows, d, 1.0, 0)
        rt.k_linear(p(w["lm_head.weight"]), 0, p(self.h), self.rows, d, c.vocab_size, 0, p(self.logits))
        before = self.ids.clone()
        u = torch.rand(self.rows, device="cuda") if u is None else u
        rt.k_sample(p(self.logits), 0, self.rows, c.vocab_size, c.vocab_size, p(temperature), p(top_k), p(top_p), p(min_p), p(u),
                    p(self.ids), p(self.logprobs), p(self.kept))
        self.ids = torch.where(idle, before, self.ids)
        return self.ids


def serve(engine, prompts, new_tokens, controls=None, on_step=None):
    """Runs every prompt to new_tokens ids, as many at a time as the engine has rows. Returns the ids by prompt.
    controls: (temperature, top_k, top_p, min_p) by prompt. on_step(engine, running): called after every step.
    ValueError for a prompt that no step could take: an empty one, one longer than a step has room for beside a token
    of every other row, one that outgrows the context."""
    room = engine.tokens - engine.rows
    if new_tokens < 1:
        raise ValueError(f"new_tokens is {new_tokens}, at least 1 is needed")
    for i, prompt in enumerate(prompts):
        if not len(prompt):
            raise ValueError(f"prompt {i} is empty")
        if len(prompt) > room:
            raise ValueError(f"prompt {i} has {len(prompt)} ids, a step takes at most {room}")
        if len(prompt) + new_tokens - 1 > engine.context:
            raise ValueError(f"prompt {i} with {new_tokens} new ids outgrows the context of {engine.context}")
    waiting, running, answers = list(range(len(prompts))), [None] * engine.rows, [[] for _ in prompts]
    ended = [False] * engine.rows
    while waiting or any(r is not None for r in running):
        append, ids, budget = [0] * engine.rows, [], engine.tokens
        for r in range(engine.rows):
            if running[r] is not None and answers[running[r]]:
                append[r], chunk = 1, [answers[running[r]][-1]]
            elif ended[r]:  # its pages return in this step's plan; the row is free from the next on
                append[r], ended[r], chunk = -1, False, []
            elif running[r] is None and waiting and len(prompts[waiting[0]]) <= budget - engine.rows:
                running[r] = waiting.pop(0)
                chunk = prompts[running[r]]
                append[r] = len(chunk)
            else:
                continue
            ids += chunk
            budget -= len(chunk)
        values = [None] * 4
        if controls:
            by_row = [controls[i] if i is not None else (0.0, 0, 1.0, 0.0) for i in running]
            types = (torch.float32, torch.int32, torch.float32, torch.float32)
            values = [torch.tensor(list(v), dtype=t, device="cuda") for v, t in zip(zip(*by_row), types)]
        out = engine.step(append, ids, *values)
        refused = int(engine.counts[0][3])
        if refused:
            raise RuntimeError(f"{refused} requests got no pages")
        for r, token in enumerate(out.tolist()):
            if running[r] is not None and append[r] > 0:
                answers[running[r]].append(token)
        if on_step:
            on_step(engine, [i if a > 0 else None for i, a in zip(running, append)])
        for r in range(engine.rows):
            if running[r] is not None and len(answers[running[r]]) >= new_tokens:
                running[r], ended[r] = None, True
    engine.plan([-1 if e else 0 for e in ended])
    return answers


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--model", help="a model directory (default: a small synthetic one)")
    ap.add_argument("--requests", type=int, default=12)
    ap.add_argument("--rows", type=int, default=4)
    ap.add_argument("--new-tokens", type=int, default=32)
    a = ap.parse_args()
    with tempfile.TemporaryDirectory() as tmp:
        directory = a.model or package().synthetic.write_model(Path(tmp) / "model", package().synthetic.TINY)
        engine = Engine(directory, rows=a.rows)
        vocab = engine.cfg.vocab_size
        prompts = [package().synthetic.seeded_tokens(5 + 17 * i % 90, vocab, seed=i) for i in range(a.requests)]
        controls = [(0.0, 0, 1.0, 0.0) if i % 3 == 0 else (0.8, 50, 0.95, 0.02) for i in range(a.requests)]
        began = time.perf_counter()
        answers = serve(engine, prompts, a.new_tokens, controls)
        torch.cuda.synchronize()
        spent = time.perf_counter() - began
    for i, ids in enumerate(answers):
        print(f"request {i}: {len(prompts[i])} prompt ids -> {ids[:10]} ...")
    total = sum(len(v) for v in answers)
    print(f"{total} ids in {spent:.2f} s; free pages at the end: {int(engine.counts[0][0])} of {engine.pages}")


if __name__ == "__main__":
    main()
