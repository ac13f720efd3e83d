"""The 8-bit cache without a device: its format in the plain implementation, the manager's storage, what engines and layers
refuse, and the lists of tiles a step brings."""

import numpy as np
import pytest
import torch

from acorninfer_b200.cache.manager import CacheManager
from acorninfer_b200.config.engine_config import EngineConfig
from acorninfer_b200.engine.batch import StepEntry, pad_decode_plan, plan_step
from acorninfer_b200.kernels import attention as attn
from acorninfer_b200.kernels import ops
from acorninfer_b200.models.decoder import Decoder
from acorninfer_b200.parts.attention import Attention
from acorninfer_b200.parts.base import BuildContext, KVNeeds
from acorninfer_b200.registry import spec_for
from tests.plain import f8_cache as f8
from tests.tiny import TINIES, TINY_A

F8 = torch.float8_e4m3fn


def test_the_plain_format_agrees_with_the_type():
    table = f8.e4m3_numbers()
    assert torch.equal(table.float(), torch.arange(127, dtype=torch.uint8).view(F8).float())
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.randn(20000) * 0.01, table.float(), (table[1:] + table[:-1]).float() / 2])
    assert torch.equal(f8.nearest_e4m3(x).float(), x.to(F8).float())


@pytest.mark.parametrize("most,e", [(0.0, -120), (2.0 ** -149, -120), (448.0, 0), (448.0001, 1), (449.0, 1), (224.0, -1), (1.0, -8), (1.75, -8),
                                    (1.7500001, -7), (1e-36, -120), (3.3e38, 120), (1.75 * 2.0 ** 127, 119)])
def test_row_exponents(most, e):
    row = torch.tensor([[0.0, -most, most / 2]], dtype=torch.float64)
    assert int(f8.row_exponents(row)) == e
    codes, got = f8.quantise(row)
    assert int(got) == e and bool((codes.abs() <= 448).all())
    back = f8.dequantise(codes, got + 127)
    assert bool(torch.isfinite(back.float()).all()) and torch.equal(back.to(torch.bfloat16).double(), back)


def test_the_manager_keeps_codes_and_scales():
    needs = {0: KVNeeds(2, 64, dtype=F8), 1: KVNeeds(2, 64, dtype=F8), 2: KVNeeds(2, 64)}
    m = CacheManager(needs, {}, num_pages=5, page_size=16, num_slots=2, dtype=torch.bfloat16, device="cpu")
    assert len(m.groups) == 2                                  # 8-bit layers are a group of their own
    k, v = m.kv_pages(1)
    s = m.kv_scales(1)
    assert k.dtype == F8 and k.shape == v.shape == (6, 2, 16, 64) and s.shape == (6, 2, 16, 2) and s.dtype == torch.float8_e8m0fnu
    assert k.is_contiguous() and s.is_contiguous() and m.kv_scales(2) is None and m.kv_pages(2)[0].dtype == torch.bfloat16
    assert m.bytes_per_token() == 2 * 2 * (2 * 64 + 2) + 2 * 2 * 64 * 2
    assert float(k.float().abs().sum()) == 0
    dry = CacheManager(needs, {}, num_pages=5, page_size=16, num_slots=2, allocate=False)
    assert dry.bytes_per_token() == m.bytes_per_token()
    with pytest.raises(ValueError, match="one width"):
        CacheManager({0: KVNeeds(2, 64, dtype=F8, value_dim=32)}, {}, num_pages=5, page_size=16, num_slots=2, device="cpu")


def test_engine_options():
    assert EngineConfig(kv_dtype="float8").kv_dtype == "float8" and EngineConfig().kv_dtype is None
    with pytest.raises(ValueError, match="kv_dtype"):
        EngineConfig(kv_dtype="int8")
    with pytest.raises(ValueError, match="bfloat16"):
        EngineConfig(kv_dtype="float8", dtype="float32")


def test_runner_options():
    from acorninfer_b200.engine.runner import _dtypes
    assert _dtypes({"kv_dtype": "float8"}) == (torch.bfloat16, F8) and _dtypes({"dtype": "float32"}) == (torch.float32, None)
    with pytest.raises(ValueError, match="kv_dtype"):
        _dtypes({"kv_dtype": "fp8"})
    with pytest.raises(ValueError, match="bfloat16"):
        _dtypes({"kv_dtype": "float8", "dtype": "float32"})


def test_what_attention_layers_refuse():
    ctx = BuildContext(torch.bfloat16, torch.device("cpu"), 16, kv_dtype=F8)
    make = lambda d=64, **kw: Attention(ctx, 128, 4, 2, d, None, 0.125, **kw)           # noqa: E731
    assert make().cache_needs().kv.dtype == F8 and make(window=9, keep_first=2, sink=True, bias=True).eight_bit
    for kw, word in ((dict(value_dim=32), "another width"), (dict(values_from_keys=True), "taken from the keys"), (dict(conv_taps=3), "convolution"),
                     (dict(slope_exponent=8.0), "distance"), (dict(softcap=20.0), "capped"), (dict(q_temp=(0.1, 10)), "temperature"),
                     (dict(qk_norm_rows=True, qk_norm_eps=1e-6), "whole rows"), (dict(d=60), "60 entries"), (dict(d=264), "264 entries"),
                     (dict(qk_norm_eps=1e-6, norm_after_rotation=True, qk_norm_weights=False), "after the rotation")):
        with pytest.raises(ValueError, match=word):
            make(**kw)
    plain = Attention(BuildContext(torch.bfloat16, torch.device("cpu"), 16), 128, 4, 2, 60, None, 0.125, softcap=20.0)
    assert not plain.eight_bit and plain.cache_needs().kv.dtype is None


@pytest.mark.parametrize("name", ["kogonex", "vagulorn", "tedenex", "zigolix", "zusolix", "badepel"])
def test_models_whose_layers_keep_something_else_are_refused(name):
    import importlib
    tiny = importlib.import_module(f"tests.{name}_tiny")
    cfg = next(v["cfg"] if isinstance(v, dict) and "cfg" in v else v for k, v in vars(tiny).items()
               if (isinstance(v, dict) and "cfg" in v) or hasattr(v, "num_hidden_layers"))
    with pytest.raises(ValueError, match="8-bit|no form"):
        Decoder(spec_for(cfg), torch.bfloat16, "cpu", 16, F8).cache_needs()


def test_a_model_of_attention_layers_takes_it():
    for tiny in TINIES.values():
        kv, state = Decoder(spec_for(tiny["cfg"]), torch.bfloat16, "cpu", 16, F8).cache_needs()
        assert not state and all(n.dtype == F8 for n in kv.values())


def plan_of(lens, held, arrays):
    m = CacheManager({0: KVNeeds(2, 64, dtype=F8)}, {}, num_pages=400, page_size=16, num_slots=len(lens) + 1, allocate=False)
    entries = []
    for i, (n, h) in enumerate(zip(lens, held)):
        rc = m.open(i)
        m.extend(rc, h + n)
        m.commit(rc, h)
        entries.append(StepEntry(rc, [1] * n, [n - 1]))
    return plan_step(entries, m, arrays), m


def test_step_arrays_hold_every_token_once():
    arrays = attn.f8_step_arrays(8, 2)                          # four query heads a kv head: four tokens a tile
    lens, held = [1, 130, 7, 1, 31, 32, 300, 2], [40, 0, 100, 0, 9, 1000, 17, 3]
    plan, _ = plan_of(lens, held, arrays)
    seen = [np.zeros(n, int) for n in lens]
    for name, step in (("attention.f8_single", 1), ("attention.f8_short4", 4), ("attention.f8_large", 128)):
        assert plan.extra[name].dtype == np.int32 and plan.extra[name].shape[1] == 2
        for r, q0 in plan.extra[name]:
            seen[r][q0:q0 + step] += 1
    assert all((s == 1).all() for s in seen)
    big = plan.extra["attention.f8_large"]
    keys = [held[r] + min(q0 + 128, lens[r]) for r, q0 in big]
    assert keys == sorted(keys, reverse=True) and {r for r, _ in big} == {1, 5, 6}
    assert [r for r, _ in plan.extra["attention.f8_single"]] == [0, 3]


def test_decode_steps_of_a_bucket_have_arrays_of_one_shape():
    arrays = attn.f8_step_arrays(8, 2)
    shapes = set()
    for n in (9, 10):
        plan, m = plan_of([1] * n, [5 * i for i in range(n)], arrays)
        padded = pad_decode_plan(plan, m.pad_pages, m.pad_slot, arrays)
        shapes.add(tuple((k, padded.extra[k].shape) for k in sorted(padded.extra)))
        assert padded.extra["attention.f8_single"].shape[0] == padded.num_rows == 10
    assert len(shapes) == 1


@pytest.mark.parametrize("nq,nkv,tokens", [(8, 8, 16), (8, 2, 4), (10, 2, 3), (24, 2, 1), (40, 1, 1), (9, 1, 1), (16, 2, 2)])
def test_tokens_a_tile(nq, nkv, tokens):
    assert ops.f8_tile_tokens(nq, nkv) == tokens


def test_splits_are_within_the_kernels_limits():
    for tiles in (1, 2, 7, 41, 148, 500):
        for bound in (16, 300, 1000, 4096, 40000, 1 << 20):
            for shares in (0, 444):
                s = ops.decode_f8_splits(tiles, 8, bound, 128, shares)
                assert s in ops.F8_SPLITS and (shares or s)             # without CTAs to share there are no shares
            assert 1 <= ops.prefill_f8_splits(tiles * 16, -(-bound // 128)) <= min(ops.F8_MAX_SPLITS, -(-bound // 128))
    assert ops.decode_f8_splits(1, 8, 16, 128, 444) == 1 and ops.prefill_f8_splits(2000, 64) == 1
    assert ops.decode_f8_splits(64, 8, 4096, 128, 444) == 0


def test_generation_and_command_line_take_the_option():
    import inspect

    from acorninfer_b200 import generation, replay
    assert "kv_dtype" in inspect.signature(generation.build_engine).parameters
    args = replay.parse_args(["--model", "m", "--dtype", "bfloat16", "--out", "o", "--max-tokens", "64", "--kv-dtype", "float8"])
    assert args.kv_dtype == "float8" and TINY_A["cfg"].head_dim == 16
