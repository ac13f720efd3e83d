"""Models over an 8-bit cache, through the engine's own entry points: the step function's logits against the plain model in 64
bits that reads the very keys and values the cache holds, which kernels run, captured and eager steps, pages used again, and
generation, replay and the command line."""

import json
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from acorninfer_b200.config.model_config import Qwen3Config
from tests.plain import f8_cache as f8
from tests.plain import model as plain
from tests.tiny import TINY_A, TINY_C, TINY_D, make_model_dir, random_tokens, read_weights, sizes_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# head size 64, eight query heads to a kv head
TINY_E = dict(cfg=Qwen3Config(num_hidden_layers=3, hidden_size=128, num_attention_heads=8, num_key_value_heads=1, head_dim=64,
                              intermediate_size=256, rms_norm_eps=1e-6, rope_theta=1e6, vocab_size=300, tie_word_embeddings=True,
                              bos_token_id=None, eos_token_id=()), sigma=0.05, sigma_norm=0.1, seed=505, page_size=32)
TINIES = {"a": TINY_A, "c": TINY_C, "d": TINY_D, "e": TINY_E}
TOL = 6e-2        # of logits of the bfloat16 engine against 64 bits at these sizes: as for the bfloat16 cache (test_replay_gpu.py)


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    return {k: make_model_dir(tmp_path_factory.mktemp("f8") / k, t) for k, t in TINIES.items()}


def runner_of(folder, tiny, **kw):
    from acorninfer_b200.engine.runner import ModelRunner
    kw = {"num_blocks": 96, "page_size": tiny["page_size"], "max_requests": 6, "kv_dtype": "float8", **kw}
    return ModelRunner.from_model_dir(folder, dtype="bfloat16", **kw)


def counts_of(fn):
    from acorninfer_b200.kernels import ops
    before = dict(ops.COUNTS)
    fn()
    return {k: v - before.get(k, 0) for k, v in ops.COUNTS.items() if v - before.get(k, 0)}


def cached(runner, rc, entry, length):
    """Keys and values of a request as its pages hold them, in 64 bits: [nkv, length, d] each."""
    k, v = runner.manager.kv_pages(entry)
    s = runner.manager.kv_scales(entry).view(torch.uint8).cpu()
    P = runner.manager.page_size
    gi = runner.manager.group_of(entry)
    pages = torch.tensor([rc.tables[gi][p // P - rc.page_base[gi]] for p in range(length)])
    slots = torch.arange(length) % P
    out = []
    for which, t in enumerate((k, v)):
        codes = t.view(torch.uint8).cpu()[pages, :, slots].view(torch.float8_e4m3fn)
        out.append(f8.dequantise(codes, s[pages, :, slots, which]).transpose(0, 1))
    return out


def plain_over_cache(tiny, w, ids, caches):
    """The plain model on ``ids`` with every layer's keys and values as given; the layers' own come back beside the logits."""
    sizes = sizes_of(tiny["cfg"])
    w = {k: t.double() for k, t in w.items()}
    positions = torch.arange(len(ids))
    x, own = w["model.embed_tokens.weight"][torch.as_tensor(ids)], []
    for i, kv in enumerate(caches):
        p = f"model.layers.{i}."
        h = plain.rms_norm(x, w[p + "input_layernorm.weight"], sizes["rms_norm_eps"])
        own.append(plain.attention_keys_values(h, w, p + "self_attn.", sizes, positions))
        x, _ = plain.decoder_layer(x, w, i, sizes, positions, None, kv)
    x = plain.rms_norm(x, w["model.norm.weight"], sizes["rms_norm_eps"])
    head = w["lm_head.weight"] if not tiny["cfg"].tie_word_embeddings else w["model.embed_tokens.weight"]
    return x @ head.T, own


@pytest.mark.parametrize("which", list(TINIES))
@pytest.mark.parametrize("graph", [False, True])
def test_steps_match_the_plain_model_over_the_same_cache(folders, which, graph):
    """Prompts whole and in portions, short portions, decoded tokens, all beside one another."""
    from acorninfer_b200.engine.batch import StepEntry
    tiny = TINIES[which]
    V, L = tiny["cfg"].vocab_size, tiny["cfg"].num_hidden_layers
    runner = runner_of(folders[which], tiny, decode_graph=graph)
    reqs = {"x": random_tokens(150, V, 1), "y": random_tokens(60, V, 2), "z": random_tokens(9, V, 3)}
    rcs = {r: runner.open(r) for r in reqs}
    at = dict.fromkeys(reqs, 0)
    got = {r: {} for r in reqs}
    cuts = [{"x": 130}, {"y": 40, "x": 1}, {"z": 1, "x": 3, "y": 1}, {"z": 5, "y": 17}] + [{"x": 1}] * 4 + [{"x": 1, "y": 1, "z": 1}] * 2
    for cut in cuts:
        entries, wanted = [], []
        for r, n in cut.items():
            want = sorted({0, n // 2, n - 1})
            entries.append(StepEntry(rcs[r], reqs[r][at[r]:at[r] + n], want))
            wanted += [(r, at[r] + j) for j in want]
            at[r] += n
        logits = runner.step(entries).double().cpu()
        for (r, pos), row in zip(wanted, logits):
            got[r][pos] = row
    assert graph is False or runner.graph_replays >= 2
    w = read_weights(folders[which])
    for r in reqs:
        n = at[r]
        caches = [cached(runner, rcs[r], e, n) for e in range(L)]
        want, own = plain_over_cache(tiny, w, reqs[r][:n], caches)
        for pos, row in got[r].items():
            assert float((row - want[pos]).abs().max()) < TOL, (r, pos)
        # what the cache holds is what the model computes, to half a code (2^-4) and the activations' rounding (3e-2 of a row)
        for (k, v), (pk, pv) in zip(caches, own):
            for have, should in ((k, pk), (v, pv)):
                far = (have - should).norm(dim=-1) / should.norm(dim=-1)
                assert float(far.max()) < 2.0 ** -4 + 3e-2
    for rc in rcs.values():
        runner.close(rc)
    runner.manager.assert_balanced()


def test_which_kernels_run(folders):
    from acorninfer_b200.engine.batch import StepEntry
    tiny = TINY_D
    V, L = tiny["cfg"].vocab_size, tiny["cfg"].num_hidden_layers
    runner = runner_of(folders["d"], tiny, decode_graph=False)
    a, b, c = runner.open("a"), runner.open("b"), runner.open("c")
    n = counts_of(lambda: runner.step([StepEntry(a, random_tokens(40, V, 1), [39]), StepEntry(b, random_tokens(5, V, 2), [4])]))
    assert n["qk_rope_kv_f8"] == n["attention_prefill_f8"] == n["attention_decode_f8"] == L
    # two decoded tokens: norm, rotation and the cache write ride on the q/k/v product
    n = counts_of(lambda: runner.step([StepEntry(a, [3], [0]), StepEntry(b, [4], [0])]))
    assert n["gemm_tc_qkv_rope"] == n["attention_decode_f8"] == L and "attention_prefill_f8" not in n and "qk_rope_kv_f8" not in n
    n = counts_of(lambda: runner.step([StepEntry(a, [3], [0]), StepEntry(b, [4, 5], [1]), StepEntry(c, random_tokens(33, V, 3), [])]))
    assert n["attention_decode_f8"] == 2 * L and n["attention_prefill_f8"] == L
    assert not any(k.startswith("attention_") and not k.endswith("_f8") for k in n) and "gemm_tc_qkv_rope" not in n
    other = runner_of(folders["c"], TINY_C, decode_graph=False)                 # head size 48
    d = other.open("d")
    n = counts_of(lambda: other.step([StepEntry(d, random_tokens(40, 300, 1), [39])]))
    assert n["attention_f8_plain"] == TINY_C["cfg"].num_hidden_layers


def test_half_the_bytes(folders):
    wide, narrow = runner_of(folders["d"], TINY_D, kv_dtype=None), runner_of(folders["d"], TINY_D)
    assert narrow.manager.bytes_per_token() == wide.manager.bytes_per_token() // 2 + TINY_D["cfg"].num_hidden_layers * 2 * 2


def test_captured_steps_are_the_eager_ones(folders):
    from acorninfer_b200.engine.batch import StepEntry
    tiny = TINY_D
    prompt, tail = random_tokens(90, tiny["cfg"].vocab_size, 5), random_tokens(12, tiny["cfg"].vocab_size, 6)
    rows = []
    for graph in (False, True):
        runner = runner_of(folders["d"], tiny)
        # the prompt eagerly in both: a captured portion is padded to its bucket, 30 tokens to 32, which go to another kernel
        runner.decode_graph = False
        rc = runner.open("a")
        runner.step([StepEntry(rc, prompt[:60], [])])
        runner.step([StepEntry(rc, prompt[60:], [29])])
        runner.decode_graph = graph
        rows.append(torch.stack([runner.step([StepEntry(rc, [t], [0])])[0].clone() for t in tail]))
    assert runner.graph_replays >= 8 and torch.equal(rows[0], rows[1])


def test_pages_used_again_leave_no_trace(folders):
    from acorninfer_b200.engine.batch import StepEntry
    tiny = TINY_E
    V = tiny["cfg"].vocab_size

    def run(runner, name, seed):
        rc = runner.open(name)
        out = [runner.step([StepEntry(rc, random_tokens(70, V, seed), [69])]).clone()]
        out += [runner.step([StepEntry(rc, [t], [0])]).clone() for t in random_tokens(5, V, seed + 1)]
        runner.close(rc)
        return torch.cat(out)

    used = runner_of(folders["e"], tiny, num_blocks=4, decode_graph=False)
    for seed in (1, 11, 21):
        run(used, f"before{seed}", seed)
    fresh = runner_of(folders["e"], tiny, num_blocks=4, decode_graph=False)
    assert torch.equal(run(used, "again", 31), run(fresh, "first", 31))


def test_generate_and_engine(folders):
    from acorninfer_b200 import generate
    from acorninfer_b200.engine.batch import StepEntry
    tiny = TINY_D
    V = tiny["cfg"].vocab_size
    prompts = [random_tokens(n, V, 40 + n) for n in (5, 33, 70, 1)]
    got = generate(folders["d"], prompts, max_new_tokens=12, num_blocks=64, page_size=16, eos_ids=(), kv_dtype="float8")
    assert [len(g) for g in got] == [len(p) + 12 for p in prompts] and all(g[:len(p)] == p for g, p in zip(got, prompts))
    # one request alone: the tokens of the step function fed by hand
    alone = generate(folders["d"], [prompts[1]], max_new_tokens=12, num_blocks=64, page_size=16, eos_ids=(), kv_dtype="float8")[0]
    runner = runner_of(folders["d"], tiny)
    rc = runner.open("a")
    ids, new = list(prompts[1]), prompts[1]
    for _ in range(12):
        new = [int(runner.step([StepEntry(rc, new, [len(new) - 1])])[0].argmax())]
        ids += new
    assert ids == alone
    # a pool so small that requests are preempted and recomputed
    few = generate(folders["d"], prompts, max_new_tokens=12, num_blocks=10, page_size=16, watermark_blocks=1, eos_ids=(), kv_dtype="float8")
    assert [len(g) for g in few] == [len(g) for g in got]


def test_replay_and_command_line(folders, tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    steps = [{"step": 0, "entries": [{"id": "a", "tokens": random_tokens(40, 500, 1), "want": [39]}]},
             {"step": 1, "entries": [{"id": "a", "tokens": [7], "want": [0]}], "end": ["a"]}]
    env = dict(os.environ, PYTHONPATH=root)
    cmd = [sys.executable, "-m", "acorninfer_b200.replay", "--model", str(folders["d"]), "--dtype", "bfloat16", "--kv-dtype", "float8", "--out",
           str(tmp_path), "--max-tokens", "64"]
    done = subprocess.run(cmd, input="\n".join(json.dumps(s) for s in steps), text=True, capture_output=True, env=env, timeout=300)
    assert done.returncode == 0 and done.stdout.split("\n")[:2] == ["done 0", "done 1"], done.stderr[-500:]
    assert np.isfinite(np.fromfile(tmp_path / "1.f32", "<f4")).all()
    cmd = [sys.executable, "-m", "acorninfer_b200", "generate", "--model-dir", str(folders["d"]), "--prompt-ids", "5,6,7", "--max-new-tokens", "4",
           "--kv-dtype", "float8"]
    done = subprocess.run(cmd, text=True, capture_output=True, env=env, timeout=300)
    assert done.returncode == 0 and done.stdout.strip().startswith("5,6,7,") and len(done.stdout.strip().split(",")) == 7, done.stderr[-500:]
