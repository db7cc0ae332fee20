"""The engine over pages held in 8 bits (``cache_dtype="e4m3"``): every layer of mixed steps against attention in 64 bits over what its pages hold, the same tokens
whichever way a step is run, and what is refused."""

from __future__ import annotations

import json
import subprocess
import sys

import pytest
import torch

import plain_qwen3 as plain
import replay_util as ru
from conftest import ROOT, TINY_INIT

pytestmark = pytest.mark.gpu

HALF_E4M3, HALF_F32 = 2.0 ** -4, 2.0 ** -24


def held(cache, layer, seq):
    """(keys, values, unit of each) of a request, as values [tokens, heads, d]."""
    kv = cache.layer_pools(layer)
    spec = next(g.spec for g in cache.layout.groups if layer in g.layers)
    n = cache.manager.tokens(seq)
    table = torch.tensor(cache.manager.table(seq), device="cuda:0")
    at = torch.arange(n, device="cuda:0")
    page = table[at // cache.block_size]
    out = []
    for pool, power in zip(kv, cache._powers[layer]):
        unit = torch.exp2(power.view(torch.uint8).double()[page] - 127).unsqueeze(-1)
        out.append(pool.double().view(-1, spec.kv_heads, spec.head_dim)[page * cache.block_size + at % cache.block_size] * unit)
        out.append(unit)
    return out[0].cpu(), out[2].cpu(), out[1].cpu(), out[3].cpu()


@pytest.mark.parametrize("name,pad", [("A", None), ("A", 64), ("C", None), ("C", 64)])
def test_every_layer_of_mixed_steps(model_dirs, name, pad):
    """32-bit steps with named activations: what attention gives is its rows over what the pages hold, and the pages hold the rows' keys and values."""
    from paged_llm_rs_amd.cache import PagedCache
    from paged_llm_rs_amd.engine.batch import StepEntry
    from paged_llm_rs_amd.engine.step import commit_step, run_step
    from paged_llm_rs_amd.parts.model import load_model

    cfg = TINY_INIT[name]["config"]
    nq, nkv, d = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"]
    group, theta = nq // nkv, plain.config_rope_theta(cfg)
    _, model = load_model(model_dirs(name, "float32"), "float32", "cuda:0")
    cache = PagedCache(model.cache_layout, 8, 64, torch.float32, "cuda:0", max_seqs=4, eight_bit=True)
    prompts = ru.make_prompts(cfg["vocab_size"], [5, 30, 17], seed=3)
    tokens = [list(p) for p in prompts.values()]
    for s in range(3):
        cache.manager.add_sequence(s)
    done = [0, 0, 0]
    # prompts whole and in portions, single tokens beside them
    for brings in ([5, 11, 9], [1, 12, 8], [1, 7, 1], [1, 1, 1]):
        entries = []
        for s, count in enumerate(brings):
            while len(tokens[s]) < done[s] + count:
                tokens[s].append((7 * len(tokens[s]) + s) % cfg["vocab_size"])
            assert cache.manager.reserve(s, count)
            entries.append(StepEntry(s, tokens[s][done[s]:done[s] + count], done[s], want=[count - 1]))
        trace = {}
        logits = run_step(model, cache, entries, pad_to=pad, trace=trace)
        commit_step(cache, entries)
        assert bool(logits.isfinite().all()) and logits.shape == (3, cfg["vocab_size"])
        for layer in range(cfg["num_hidden_layers"]):
            get = lambda what: trace[f"model.layers.{layer}.self_attn.{what}"].double().cpu()  # noqa: E731
            at = 0
            for s, count in enumerate(brings):
                rows, positions = slice(at, at + count), torch.arange(done[s], done[s] + count)
                at += count
                q = plain.apply_rope(get("q_norm.out")[rows].reshape(count, nq, d), positions, theta)
                k = plain.apply_rope(get("k_norm.out")[rows].reshape(count, nkv, d), positions, theta)
                keys, values, k_unit, v_unit = held(cache, layer, s)
                # one rounding to e4m3 of the rows that this step wrote (half a step: 2^-4 of a value, 2^-10 units of the smallest), after 32-bit norms and rotations
                for have, want, unit in ((keys, k, k_unit), (values, get("v_proj.out")[rows].reshape(count, nkv, d), v_unit)):
                    off = (have[done[s]:] - want).abs()
                    assert bool((off <= torch.maximum(HALF_E4M3 * want.abs(), 2.0 ** -10 * unit[done[s]:]) + 1e-5 * want.abs().amax(-1, keepdim=True)).all()), (layer, s)
                seen = torch.arange(done[s] + count).view(1, -1) <= positions.view(-1, 1)
                out = get("o_proj.in")[rows].reshape(count, nkv, group, d)
                for h in range(nkv):
                    x = q.view(count, nkv, group, d)[:, h].reshape(count * group, d)
                    score = (x @ keys[:, h].T / d ** 0.5).view(count, group, -1).masked_fill(~seen.unsqueeze(1), -torch.inf)
                    size = (x.abs() @ keys[:, h].abs().T / d ** 0.5).view(count, group, -1).amax(-1, keepdim=True)
                    p = torch.softmax(score, -1)
                    want, most = p @ values[:, h], p @ values[:, h].abs()
                    # the recorded q is rounded to 32 bits before the rotation and norms take a dozen roundings: 32 halves of a last place of a score beside its own d + 16 sums of three products
                    allowed = most * (2 * size * (3 * (d + 16) + 32) * HALF_F32 + 64 * HALF_F32) + HALF_F32 * want.abs()
                    assert bool(((out[:, h] - want).abs() <= allowed).all()), (layer, s, h, float(((out[:, h] - want).abs() / allowed).max()))
        done = [x + y for x, y in zip(done, brings)]


@pytest.mark.parametrize("name,dtype", [("A", "f32"), ("A", "bf16"), ("D", "bf16")])
def test_the_same_tokens_whichever_way_steps_are_run(model_dirs, name, dtype):
    """Captured and launched kernel by kernel, a step ahead or not, and again on the same engine (whose pages then hold what others left)."""
    from paged_llm_rs_amd import Engine

    cfg = TINY_INIT[name]["config"]
    path = model_dirs(name, "float32" if dtype == "f32" else "bfloat16")
    prompts = list(ru.make_prompts(cfg["vocab_size"], [5, 17, 40, 1, 90], seed=5).values())
    results = []
    for options in (dict(), dict(graphs=False), dict(ahead=False), dict(graphs=False, ahead=False)):
        engine = Engine(path, dtype=dtype, block_size=16, num_blocks=64, max_batch=4, chunk=32, prefix_cache=False, cache_dtype="e4m3", **options)
        for _ in range(2):
            out = engine.generate(prompts, max_tokens=40, temperature=0.0, stop_tokens=[])
            results.append([r["tokens"] for r in out])
            assert all(len(r["tokens"]) == 40 and r["finish"] == "length" for r in out)
        assert "in e4m3" in engine.describe()
    assert all(r == results[0] for r in results)


def test_twice_the_tokens_in_the_same_bytes_and_pages_that_run_out(model_dirs):
    from paged_llm_rs_amd import Engine

    path = model_dirs("A", "bfloat16")
    cfg = TINY_INIT["A"]["config"]
    wide = Engine(path, dtype="bf16", block_size=16, cache_mib=8)
    small = Engine(path, dtype="bf16", block_size=16, cache_mib=8, cache_dtype="e4m3")
    per_page = 16 * small.bytes_per_token
    beside = cfg["num_hidden_layers"] * 2 * cfg["num_key_value_heads"]
    assert small.bytes_per_token * 2 == wide.bytes_per_token and small.num_blocks == (8 << 20) // (per_page + beside)
    assert small.cache.bytes == small.num_blocks * (per_page + beside) <= 8 << 20
    # (requests that are thrown out and begin again, prefixes that are shared)
    engine = Engine(path, dtype="bf16", block_size=8, num_blocks=16, max_batch=4, chunk=16, cache_dtype="e4m3")
    prompts = [[1 + i % 50 for i in range(24)] + [60 + j] for j in range(5)]
    out = engine.generate(prompts, max_tokens=30, temperature=0.0, stop_tokens=[])
    assert all(len(r["tokens"]) == 30 for r in out)
    assert engine.metrics()["available"] == engine.metrics()["total"]


def test_refusals(model_dirs, tmp_path):
    from paged_llm_rs_amd import Engine, kernels
    from paged_llm_rs_amd.errors import ConfigError, TensorError

    path = model_dirs("A", "float32")
    with pytest.raises(ConfigError):
        Engine(path, dtype="f32", cache_dtype="e5m2", num_blocks=8)
    engine = Engine(path, dtype="f32", cache_dtype="e4m3", num_blocks=8, graphs=False)
    kernels.set_attention("tensor")
    try:
        with pytest.raises(TensorError):
            engine.generate([[1, 2, 3]], max_tokens=2)
    finally:
        kernels.set_attention("kernel")
    import lefavik_util

    other = lefavik_util.write_model(tmp_path / "lefavik", lefavik_util.ODD)
    with pytest.raises(ConfigError):
        Engine(other, dtype="f32", cache_dtype="e4m3", num_blocks=8)


def test_the_command_line_takes_it(model_dirs):
    path = model_dirs("A", "bfloat16")
    run = subprocess.run([sys.executable, str(ROOT / "bin" / "pagedllm"), "--model", str(path), "--prompt-ids", "1,2,3", "--max-tokens", "5", "--temperature", "0", "--stop-ids", "250",
                          "--cache-dtype", "e4m3"], capture_output=True, text=True, timeout=100)
    assert run.returncode == 0, run.stderr
    assert "in e4m3" in run.stderr and len(json.loads(run.stdout.strip().splitlines()[-1])["tokens"]) == 5
