"""A model served from an 8-bit cache, against the plain model whose keys and values pass through the same
8 bits (in 64 bits).

Tolerance of the logits.  Engine and plain model quantise keys and values that differ in their last 32-bit
(bfloat16: 8-bit) digits, so now and then a code falls on the other side of a rounding; that moves one channel
of one row by a step, 1/127 (int8) or at most 1/14 (e4m3: 2^-3 of a value, of which the largest are 448/448) of
the row's largest element.  Allowed: one such step at the logits' scale in 32-bit (2^-7, 2^-4) and twice that
in bfloat16, whose own rounding of q, k and v moves more codes."""
import numpy as np
import pytest
import torch

import plain_qwen2 as plain
import replay
from tiny import CONFIGS, make_folder, prompt

pytestmark = pytest.mark.gpu
LIMIT = {"int8": 127.0, "fp8": 448.0}


def kept(x, kind):
    """Rows [T, heads, hd] (64 bits) as the cache gives them back."""
    unit = (x.abs().amax(-1, keepdim=True) / LIMIT[kind]).clamp(min=2.0 ** -126)
    y = x / unit
    if kind == "int8":
        return torch.round(y) * unit
    grid = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / grid) * grid * unit


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("kept")
    return {(n, dt): make_folder(root, n, seed=8, storage=dt, sharp=False)
            for n in ("B", "E", "F") for dt in ("float32", "bfloat16")}


def plain_logits(monkeypatch, folder, toks, kind, dtype):
    inner = plain.gqa_attention
    monkeypatch.setattr(plain, "gqa_attention",
                        lambda q, k, v, *a, **kw: inner(q, kept(k, kind), kept(v, kind), *a, **kw))
    cfg, w = plain.read_model_folder(folder)
    if dtype == "bfloat16":
        plain.Stored.bf16()
    try:
        return plain.forward(w, cfg, toks).numpy()
    finally:
        plain.Stored.exact()
        monkeypatch.setattr(plain, "gqa_attention", inner)


def runner_of(folder, dtype, kind, **kw):
    from ginfer_b200.engine import ModelRunner
    from ginfer_b200.engine.loading import load_model
    model, _ = load_model(folder, dtype)
    args = dict(page_size=16, max_num_seqs=8, max_seq_len=512, num_pages=80, kv_cache_dtype=kind)
    return ModelRunner(model, **dict(args, **kw))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("name,page", [("E", 16), ("F", 16), ("B", 8), ("E", 24)])
def test_logits(folders, monkeypatch, name, page, kind, dtype):
    """Whole prompts, portions, portions beside single tokens, tokens one by one: the same logits, the plain model's."""
    folder, vocab = folders[name, dtype], CONFIGS[name]["vocab_size"]
    reqs = {"a": prompt(200, vocab, seed=1), "b": prompt(91, vocab, seed=2), "c": prompt(37, vocab, seed=3)}
    want = {r: plain_logits(monkeypatch, folder, t, kind, dtype) for r, t in reqs.items()}
    scale = max(float(np.abs(v).max()) for v in want.values())
    lim = (2.0 ** -7 if kind == "int8" else 2.0 ** -4) * scale * (1 if dtype == "float32" else 2)
    for steps in (replay.cut_whole(reqs), replay.cut_portions(reqs, sizes=(70, 3, 1, 66, 2, 17)),
                  replay.cut_mixed(reqs, max_live=3, seed=1)[0], replay.cut_tail_decode(reqs)):
        rows = replay.run_in_process(runner_of(folder, dtype, kind, page_size=page), steps)
        assert len(rows) == sum(map(len, reqs.values()))
        worst = max(float(np.abs(row - want[r][p]).max()) for (r, p), row in rows.items())
        assert worst <= lim, (worst, lim, scale)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_generation(folders, monkeypatch, kind, dtype):
    """Decode steps and portions replayed from graphs, few pages with preemption, eagerly: every token is the plain
    model's choice along the engine's own continuation, or as good within the logits' tolerance."""
    from ginfer_b200.engine.llm import Engine
    from ginfer_b200.sampling import SamplingParams
    folder, vocab = folders["E", dtype], CONFIGS["E"]["vocab_size"]
    prompts = [prompt(n, vocab, seed=n) for n in (5, 70, 131, 44)]
    for kw in (dict(), dict(enforce_eager=True, max_num_batched_tokens=48), dict(num_kvcache_blocks=14),
               dict(capture_graphs=True, kvcache_block_size=8)):
        args = dict(max_num_seqs=4, max_num_batched_tokens=256, max_seq_len=256, num_kvcache_blocks=64,
                    kvcache_block_size=16, kv_cache_dtype=kind)
        eng = Engine(model_path=folder, dtype=dtype, **dict(args, **kw))
        outs = eng.generate(prompts, SamplingParams(max_tokens=10, ignore_eos=True))
        for p, o in zip(prompts, outs):
            assert len(o) == 10
            logits = plain_logits(monkeypatch, folder, list(p) + o[:-1], kind, dtype)
            for i, tok in enumerate(o):
                row = logits[len(p) - 1 + i]
                lim = (2.0 ** -7 if kind == "int8" else 2.0 ** -4) * np.abs(row).max() * (1 if dtype == "float32" else 2)
                assert row[tok] >= row.max() - 2 * lim, (kw, i, tok, int(row.argmax()))


def test_long_prompts_in_graph_replayed_portions(folders, monkeypatch):
    """Portions of whole budgets, replayed from a graph at other starts than it was captured at."""
    folder, vocab = folders["E", "bfloat16"], CONFIGS["E"]["vocab_size"]
    from ginfer_b200.engine import StepEntry
    run = runner_of(folder, "bfloat16", "int8", max_seq_len=1024, num_pages=80, enforce_eager=False)
    toks = prompt(900, vocab, seed=4)
    want = plain_logits(monkeypatch, folder, toks, "int8", "bfloat16")
    lim = 2.0 ** -6 * float(np.abs(want).max())
    at = 0
    for n in (260, 260, 260, 120):
        got = run.step([StepEntry("r", toks[at:at + n], [n - 1])]).cpu().numpy()[0]
        at += n
        assert np.abs(got - want[at - 1]).max() <= lim
    assert any(k[0] == "portions" for k in run._graphs)
