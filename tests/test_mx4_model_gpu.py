"""Models whose matrices are kept in microscaled 4-bit numbers: the engine against the plain implementation with the same definition in its
products, however requests are cut into steps; the captured decode step; experts of few and of many tokens; the command line."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import plain_mx4
import plain_qwen2
from nodutar_tiny import ND_A, write_nodutar
from replays import batch_steps, plain_logits, requests_for, run_steps, tail_steps, whole_steps
from test_mx4_gpu import experts_plain, within
from tiny import TINIES, write_tiny

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"

# A run in bfloat16 gives a product other rows than the plain implementation does: a little other by its roundings in front of E2M3, and more behind
# the first product.  What E2M3 makes of two values that differ by d differs by d and by the two roundings, each at most half a step: 2^-4 of a
# value (at the lower end of a binade; less elsewhere), evenly spread in that, so 2^-4 / sqrt(3) rms and both together 2^-4 sqrt(2 / 3) = 5.1 %.
# (That d itself makes few values cross a border holds for the first product alone: at 1.3 % of a value, of which a border is never
# further than 2^-4, most of the second product's values already may.)  Four products a layer add theirs up, independent of each other:
# 5.1 % sqrt(4 layers) rms of the logits' standard deviation, and six times that for the largest of a row.
ROUNDING = 2.0 ** -4 * (2.0 / 3.0) ** 0.5


class PlainMX4(plain_qwen2.PlainQwen2):
    """The plain model whose products (all but the head's) are those of the definition."""

    def forward(self, tokens):
        plain, vocab = plain_qwen2.linear, self.config_vocab

        def linear(x, w, b=None):
            if w.shape[0] == vocab:
                return plain(x, w, b)
            w4 = plain_mx4.values(*plain_mx4.nearest(torch.from_numpy(w), plain_mx4.E2M1), plain_mx4.E2M1, w.shape[1]).numpy()
            return plain(plain_mx4.rows6(torch.from_numpy(x)).numpy(), w4, b)
        plain_qwen2.linear = linear
        try:
            return super().forward(tokens)
        finally:
            plain_qwen2.linear = plain


def plain_of(folder, name):
    model = PlainMX4.from_folder(folder)
    model.config_vocab = TINIES[name]["vocab_size"]
    return model


@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_engine_against_plain(tmp_path, name):
    from minfer_amd import Engine
    from minfer_amd.engine import load_model
    folder = write_tiny(tmp_path, name)
    engine = Engine(load_model(folder, weights="mx4"), max_tokens=2048, max_seqs=4)
    requests = requests_for(TINIES[name]["vocab_size"], (1, 23, 70, 150))
    ref = plain_logits(plain_of(folder, name), requests)
    bound = ROUNDING * (4 * TINIES[name]["num_hidden_layers"]) ** 0.5
    for steps in (whole_steps(requests), tail_steps(requests), batch_steps(requests, [list(requests)[:2], list(requests)[2:]])):
        for (rid, p), got in run_steps(engine, steps).items():
            want = ref[rid][p]
            off = got.astype(np.float64) - want
            assert np.isfinite(got).all()
            assert np.sqrt(np.mean(off * off)) <= bound * want.std(), (name, rid, p, np.sqrt(np.mean(off * off)) / want.std())
            assert np.abs(off).max() <= 6 * bound * want.std(), (name, rid, p)


@pytest.mark.parametrize("name", ["A", "C"])
def test_captured_decode_is_the_eager_one(tmp_path, name):
    from minfer_amd import LLM
    llm = LLM(write_tiny(tmp_path, name), weights="mx4", n_ctx=200, n_slots=3)
    prompts = [[5, 6, 7], [9] * 40, [1, 2]]
    runs = [llm.generate(prompts, max_new=24, temp=0.0, repeat_penalty=1.0, stop_tokens=[], use_graph=g).tokens for g in (True, False, True)]
    assert runs[0] == runs[1] == runs[2] and all(len(t) == 24 for t in runs[0])


def test_layers_made_again_from_a_record(tmp_path):
    """Layers alike are launched from the record of the first one: as if each had run by itself."""
    from minfer_amd import Engine
    from minfer_amd.engine import alike, load_model
    engine = Engine(load_model(write_tiny(tmp_path, "B"), weights="mx4"), max_tokens=1024, max_seqs=2)
    requests = requests_for(TINIES["B"]["vocab_size"], (90, 33))
    with_record = run_steps(engine, whole_steps(requests))
    most, alike.MOST_VALUES = alike.MOST_VALUES, -1
    try:
        import minfer_amd.engine.model as model
        kept, model.MOST_VALUES = model.MOST_VALUES, -1
        without = run_steps(engine, whole_steps(requests))
        model.MOST_VALUES = kept
    finally:
        alike.MOST_VALUES = most
    assert all(np.array_equal(with_record[k], without[k]) for k in with_record)


def experts_part(hidden, ff, n, top, act, limit, seed):
    from minfer_amd.parts.base import FEED_FORWARDS, Runtime, make_part
    from minfer_amd.parts.spec import PartSpec
    params = dict(hidden_size=hidden, intermediate_size=ff, n_experts=n, top=top, act=act, expert="e{}", router="r")
    if act == "clamped_swish":
        params["limit"] = limit
    part = make_part(FEED_FORWARDS, PartSpec("grouped_moe", params), Runtime(torch.bfloat16, torch.device(DEV), mx4=True), "feed-forward")
    gen = torch.Generator().manual_seed(seed)
    tensors = {name: (torch.randn(spec.shape, generator=gen) * 0.08).to(torch.bfloat16).to(DEV) for name, spec in part.tensor_specs().items()}
    part.load(tensors.__getitem__)
    stack = lambda end: torch.stack([plain_mx4.values(*plain_mx4.nearest(tensors[f"e{i}{end}"], plain_mx4.E2M1), plain_mx4.E2M1,   # noqa: E731
                                                      tensors[f"e{i}{end}"].shape[1]) for i in range(n)])
    return part, [stack(end) for end in (".gate", ".up", ".down")]


@pytest.mark.parametrize("act,limit,kind", [("silu", 0.0, 1), ("clamped_swish", 0.7, 0)])
@pytest.mark.parametrize("tokens", [1, 16, 40, 150])
def test_experts_of_few_and_many_tokens(tokens, act, limit, kind):
    class Ctx:
        all_decode, token_ids, kept_rows = False, None, None
        host_tokens = host_rows = None
    ctx = Ctx()
    ctx._memo = {"route_log": []}
    part, held = experts_part(96, 80, 5, 2, act, limit, tokens)
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((tokens, 96), generator=gen).to(torch.bfloat16).to(DEV)
    h = torch.randn((tokens, 96), generator=gen).to(DEV)
    out = h.clone()
    part.forward(x, out, ctx)
    chosen = ctx._memo["route_log"][0]
    weights = torch.empty(chosen.shape, device=DEV)
    part.choose(x, ctx, torch.empty_like(chosen), weights)
    want, bound = experts_plain(x, held, chosen, weights, limit, kind)
    within(out, want + h.double(), bound + 2.0 ** -22 * (want.abs() + h.double().abs() + bound))


def test_a_model_with_experts(tmp_path):
    from minfer_amd import LLM
    folder = str(tmp_path / "nd")
    write_nodutar(folder, ND_A, 1)
    llm = LLM(folder, weights="mx4", n_ctx=128, n_slots=2)
    runs = [llm.generate([[3, 4, 5], [7] * 30], max_new=12, temp=0.0, repeat_penalty=1.0, stop_tokens=[], use_graph=g).tokens for g in (True, False)]
    assert runs[0] == runs[1] and all(len(t) == 12 for t in runs[0])


def test_command_line_generates(tmp_path):
    config = tmp_path / "config.json"
    config.write_text(json.dumps(TINIES["A"]))
    cmd = [sys.executable, os.path.join(ROOT, "bin", "minfer"), "--config", str(config), "--random-weights", "--prompt-tokens", "1,2,3", "--greedy",
           "-n", "5", "--weights", "mx4"]
    done = subprocess.run(cmd, capture_output=True, text=True, timeout=100)
    assert done.returncode == 0, done.stderr[-1000:]
