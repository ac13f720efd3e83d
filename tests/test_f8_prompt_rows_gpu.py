"""Prompts beside rows that only decode, over an 8-bit cache: which rows' keys the prompt kernel makes into bfloat16 rows, the
room it takes for them, and the same results as without the list of rows."""

import pytest
import torch

from tests.test_f8_cache_gpu import attend, check_attention, ops, raises, random_cache
from tests.test_f8_engine_gpu import TOL, cached, plain_over_cache, runner_of
from tests.tiny import TINY_D, make_model_dir, random_tokens, read_weights

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
P, FILL = 16, 0x4b4b          # what fresh scratch holds here: a row of it in bfloat16 is no key's


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def tiles_of_rows(rows, qlens):
    return i32([(r, q0) for r in rows for q0 in range(0, qlens[r], 128)]).view(-1, 2)


def scratch_of(monkeypatch, fn):
    """The call's result, and the scratch [2, kv heads, keys, d] of its bfloat16 keys and values, filled with FILL before."""
    real, kept = torch.empty, []

    def empty(*size, **kw):
        t = real(*size, **kw)
        if kw.get("dtype") == torch.bfloat16:
            t.view(torch.int16).fill_(FILL)
            kept.append(t)
        return t

    with monkeypatch.context() as m:
        m.setattr(torch, "empty", empty)
        out = fn()
    torch.cuda.synchronize()
    return out, kept


def written_keys(scratch):
    """Key rows that the call wrote, per kv head."""
    flat = scratch.view(torch.int16).view(2, -1, scratch.shape[-1])
    k = (flat[0] != FILL).any(-1)
    assert torch.equal(k, (flat[1] != FILL).any(-1))
    return int(k.sum())


BEFORES, PROMPTS = [700, 0, 1500, 300, 40, 2000, 999], [1, 3]


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("first,splits", [(300, 3), (700, 1)])
def test_only_rows_with_tiles_are_read(monkeypatch, listed, d, first, splits):
    """Tiles of two rows among seven: five tiles, fewer than rows, and eight."""
    nq, nkv, QLENS = 4, 2, [1, first, 1, 140, 1, 3, 1]
    lay, cache, keys, values = random_cache(BEFORES, QLENS, nkv, d, P, 51)
    q = torch.randn(lay["num_tokens"], nq * d, generator=torch.Generator().manual_seed(52)).to(torch.bfloat16).to(DEV)
    out = torch.full((lay["num_tokens"], nq * d), 7.0, dtype=torch.bfloat16, device=DEV)
    kw = dict(prompt_rows=i32(PROMPTS), prompt_keys=[BEFORES[r] + QLENS[r] for r in PROMPTS]) if listed else {}
    tiles = tiles_of_rows(PROMPTS, QLENS)
    assert (tiles.shape[0] >= len(QLENS)) == (first == 700)
    got, scratch = scratch_of(monkeypatch, lambda: attend("prefill", q, cache, lay, QLENS, nq, nkv, d, d ** -0.5, tiles=tiles, out=out,
                                                          num_splits=splits, **kw))
    assert len(scratch) == 1
    blocks = [-(-(BEFORES[r] + QLENS[r]) // 128) for r in PROMPTS]
    assert written_keys(scratch[0]) == nkv * 128 * sum(blocks)
    if listed:
        assert scratch[0].shape[:2] == (2, nkv) and scratch[0].shape[2] <= 128 * (sum(blocks) + len(blocks))
    at = [sum(QLENS[:r]) for r in range(len(QLENS) + 1)]
    for r in range(len(QLENS)):
        rows = slice(at[r], at[r + 1])
        if r in PROMPTS:
            check_attention(got[rows], q[rows], keys[r:r + 1], values[r:r + 1], BEFORES[r:r + 1], QLENS[r:r + 1], nq, d, d ** -0.5)
        else:
            assert bool((got[rows] == 7).all())


@pytest.mark.parametrize("mask", [dict(), dict(window=200), dict(window=130, keep_first=70), dict(chunk=256)])
@pytest.mark.parametrize("heads_at_once", [1, 4])
def test_the_list_changes_nothing_but_the_room(monkeypatch, mask, heads_at_once):
    """Forty prompts among sixty rows, in any order, a few heads at a time: the bits of a call without the list."""
    nq, nkv, d = 8, 4, 64
    g = torch.Generator().manual_seed(3)
    befores = torch.randint(0, 500, (60,), generator=g).tolist()
    qlens = [1 if r % 3 == 0 else 33 + 5 * (r % 29) for r in range(60)]
    lay, cache, _, _ = random_cache(befores, qlens, nkv, d, P, 53)
    q = torch.randn(lay["num_tokens"], nq * d, generator=g).to(torch.bfloat16).to(DEV)
    rows = [r for r in range(60) if r % 3]
    tiles = tiles_of_rows(rows, qlens)
    call = lambda **kw: attend("prefill", q, cache, lay, qlens, nq, nkv, d, 0.1, tiles=tiles, num_splits=2, **mask, **kw)     # noqa: E731
    want = call()
    order = torch.randperm(40, generator=g).tolist()
    listed = dict(prompt_rows=i32([rows[k] for k in order]), prompt_keys=[befores[rows[k]] + qlens[rows[k]] for k in order])
    room = sum(-(-k // 128) + 1 for k in listed["prompt_keys"]) * 128
    monkeypatch.setattr(ops(), "F8_PREFILL_SCRATCH", heads_at_once * room * d * 4)
    at = torch.cat([torch.arange(a, a + qlens[r]) for r, a in ((r, sum(qlens[:r])) for r in rows)]).to(DEV)
    assert torch.equal(call(**listed)[at], want[at])


def test_windowed_rows_that_gave_pages_back():
    nq, nkv, d, window = 4, 2, 128, 100
    befores, qlens = [900, 333, 50, 640], [200, 1, 130, 64]
    lay, cache, keys, values = random_cache(befores, qlens, nkv, d, P, 54)
    table, base = torch.zeros_like(lay["block_table"]), [max(0, b - window + 1) // P for b in befores]
    for r, b in enumerate(base):
        kept = lay["tables"][r][b:]
        table[r, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
    lay["block_table"], lay["page_base"] = table, i32(base)
    q = torch.randn(lay["num_tokens"], nq * d, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)
    rows = [3, 0, 2]
    got = attend("prefill", q, cache, lay, qlens, nq, nkv, d, 0.1, tiles=tiles_of_rows([0, 2, 3], qlens), window=window,
                 prompt_rows=i32(rows), prompt_keys=[befores[r] + qlens[r] - base[r] * P for r in rows])
    for r in rows:
        part = slice(sum(qlens[:r]), sum(qlens[:r + 1]))
        check_attention(got[part], q[part], keys[r:r + 1], values[r:r + 1], befores[r:r + 1], qlens[r:r + 1], nq, d, 0.1, window=window)


def test_scratch_is_for_the_prompts_and_not_for_the_widest_row(monkeypatch):
    """Sixteen short prompts beside a row whose table names 131,072 keys: one pass over the heads, a few MB."""
    nq, nkv, d = 8, 8, 64
    befores, qlens = [0] * 16 + [30], [40] * 16 + [1]
    lay, cache, keys, values = random_cache(befores, qlens, nkv, d, P, 55)
    wide = torch.zeros(17, 131072 // P, dtype=torch.int32, device=DEV)
    wide[:, :lay["block_table"].shape[1]] = lay["block_table"]
    lay["block_table"] = wide
    q = torch.randn(lay["num_tokens"], nq * d, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16).to(DEV)
    got, scratch = scratch_of(monkeypatch, lambda: attend("prefill", q, cache, lay, qlens, nq, nkv, d, 0.1, tiles=tiles_of_rows(range(16), qlens),
                                                          prompt_rows=i32(list(range(16))), prompt_keys=[40] * 16))
    assert [t.numel() * 2 for t in scratch] == [2 * nkv * 16 * 256 * d * 2]
    check_attention(got[:640], q[:640], keys[:16], values[:16], befores[:16], qlens[:16], nq, d, 0.1)


def test_lists_that_do_not_fit_are_refused_or_flagged():
    nq, nkv, d = 4, 2, 64
    lay, cache, _, _ = random_cache([20, 300], [130, 40], nkv, d, P, 56)
    q = torch.randn(170, nq * d).to(torch.bfloat16).to(DEV)
    call = lambda rows, keys: attend("prefill", q, cache, lay, [130, 40], nq, nkv, d, 0.1, prompt_rows=rows, prompt_keys=keys)      # noqa: E731
    call(i32([0, 1]), [150, 340])
    for rows, keys in ((i32([0, 1]), None), (None, [150, 340]), (i32([0, 1]), [150]), (i32([0, 1]).long(), [150, 340]), (i32([[0, 1]]), [150, 340]),
                       (i32([0, 1]).cpu(), [150, 340]), (i32([0, 1, 0]), [150, 340, 150]), (i32([]), []), (i32([0, 1]), [150, 0])):
        with raises():
            call(rows, keys)
    o = ops()
    torch.cuda.synchronize()
    o.raise_on_kernel_error()
    for rows, keys in ((i32([0, 1]), [1, 1]), (i32([1]), [340])):             # lengths below the rows'; a tile's row not listed
        call(rows, keys)
        torch.cuda.synchronize()
        with raises("attention_prefill_f8"):
            o.raise_on_kernel_error()
    call(i32([0, 1]), [150, 340])
    torch.cuda.synchronize()
    o.raise_on_kernel_error()


def test_captured_portions_replayed_for_longer_rows(tmp_path):
    """A portion of a prompt alone in its step, captured once and replayed for rows that hold more: the plain model's logits."""
    from acorninfer_b200.engine.batch import StepEntry
    tiny = {**TINY_D, "page_size": 16}
    folder = make_model_dir(tmp_path / "m", tiny)
    V, L, w = tiny["cfg"].vocab_size, tiny["cfg"].num_hidden_layers, read_weights(folder)
    runner = runner_of(folder, tiny, num_blocks=64)
    for r in range(5):
        rc, ids, got = runner.open(f"r{r}"), random_tokens(36 * 7, V, 70 + r), {}
        for at in range(0, len(ids), 36):                     # buckets of 64; tables of 8 pages, then of 16
            got[at + 35] = runner.step([StepEntry(rc, ids[at:at + 36], [35])])[0].double().cpu()
        want, _ = plain_over_cache(tiny, w, ids, [cached(runner, rc, e, len(ids)) for e in range(L)])
        for pos, row in got.items():
            assert float((row - want[pos]).abs().max()) < TOL, (r, pos)
        runner.close(rc)
    assert runner.graph_replays >= 15
