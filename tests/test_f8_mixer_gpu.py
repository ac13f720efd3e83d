"""The attention mixer over an 8-bit cache with each of its options, through steps as an engine lays them out, against the formulas in
64 bits over the very keys and values the cache holds; and what the cache holds against the formulas.

Tolerances.  A projected row is rounded to bfloat16 and so is a finished query: where a float32 sum falls to the other side of a tie, an entry of
the query is off by up to 2^-7 of itself, a score by 2^-7 of the sum of its products' magnitudes (``size``), a weight by that in the exponent,
in the numerator and the denominator.  The result is rounded to bfloat16, and again where it is gated or scaled; a gate's own rounding moves its
sigmoid by 2^-8 of the gate.  Weights as in ``test_f8_cache_gpu.py``.  Keys and values: half a code's spacing and 2^-7 of an entry, a rotation
adding two of them (2^-6 of the row's largest)."""

import math

import pytest
import torch

from tests.plain import f8_cache as f8
from tests.test_f8_cache_gpu import write_wanted

pytestmark = pytest.mark.gpu
DEV, HIDDEN, EPS = "cuda:0", 256, 1e-6
BF16 = torch.bfloat16


class Layer:
    """An attention mixer with weights of its own, its cache and requests."""

    def __init__(self, nq, nkv, d, P=16, pages=64, position=("rope", {"theta": 1e4}), norm=True, hidden=HIDDEN, eye=False, seed=1, **options):
        from acorninfer_b200.cache.manager import CacheManager
        from acorninfer_b200.engine.batch import StepWorkspace
        from acorninfer_b200.kernels import ops
        from acorninfer_b200.models.decoder import EntryCache
        from acorninfer_b200.parts.base import MIXERS, POSITION_ENCODINGS, BuildContext, PartSpec, build_part
        import acorninfer_b200.parts.attention  # noqa: F401
        import acorninfer_b200.parts.rope  # noqa: F401
        ctx = BuildContext(dtype=BF16, device=torch.device(DEV), page_size=P, kv_dtype=ops.F8)
        if position is not None:
            ctx.positions["rope"] = build_part(POSITION_ENCODINGS, PartSpec(position[0], {"head_dim": d, **position[1]}), ctx)
        self.nq, self.nkv, self.d, self.options, self.position = nq, nkv, d, options, ctx.positions.get("rope")
        self.mixer = build_part(MIXERS, PartSpec("attention", dict(
            hidden_size=hidden, num_heads=nq, num_kv_heads=nkv, head_dim=d, position="rope" if position else None, scale=d ** -0.5,
            qk_norm_eps=EPS if norm else None, **options)), ctx)
        g = torch.Generator().manual_seed(seed)
        self.tensors = {}
        for name, spec in self.mixer.tensor_specs().items():
            t = torch.randn(spec.shape, generator=g)
            t = 1 + 0.2 * t if "norm" in name else t / math.sqrt(spec.shape[-1]) if len(spec.shape) == 2 else 0.5 * t
            self.tensors[name] = t.to(BF16).to(DEV)
        if eye:                                               # the projected row is the input's
            at = 0
            for name in ("q_proj.weight", "k_proj.weight", "v_proj.weight"):
                n = self.tensors[name].shape[0]
                self.tensors[name] = torch.eye(hidden)[at:at + n].to(BF16).to(DEV)
                at += n
        self.mixer.bind(self.tensors)
        self.manager = CacheManager({0: self.mixer.cache_needs().kv}, {}, pages, P, 8, dtype=BF16, device=DEV)
        k, v = self.manager.kv_pages(0)
        self.cache = EntryCache(0, 0, k, v, True, None, self.manager.kv_scales(0))
        self.workspace = StepWorkspace(DEV, 1 << 16)

    def inputs(self, lens):
        """A step that brings ``lens`` = {request: tokens}, its pages taken."""
        from acorninfer_b200.engine.batch import StepEntry, plan_step
        for rc, n in lens.items():
            self.manager.extend(rc, rc.length + n)
        return self.workspace.upload(plan_step([StepEntry(rc, [0] * n, []) for rc, n in lens.items()], self.manager, self.mixer.step_arrays()))

    def commit(self, lens):
        for rc, n in lens.items():
            self.manager.commit(rc, rc.length + n)

    def projected(self, x):
        """(rows [T, (nq + 2 nkv) d], gates [T, nq] or None) as bfloat16 numbers in 64 bits, before any bias."""
        t = self.tensors
        of = lambda n: (x.double() @ t[n].double().T).to(BF16).double()                         # noqa: E731
        gate = of("g_proj.weight").cpu() if "g_proj.weight" in t else None
        return torch.cat([of("q_proj.weight"), of("k_proj.weight"), of("v_proj.weight")], 1), gate

    def finished(self, x, positions):
        """Queries, keys and values in 64 bits, and the gates."""
        t, pos = self.tensors, self.position
        rows, gate = self.projected(x)
        b = torch.cat([t[n + "_proj.bias"] for n in "qkv"]) if "q_proj.bias" in t else None
        inv, rot = (pos.inv_freq, pos.rotary_dim) if pos else (torch.zeros(0), 0)
        w = [t.get("q_norm.weight"), t.get("k_norm.weight")]
        return (*write_wanted(rows, w, b, inv, torch.as_tensor(positions), self.nq, self.nkv, self.d, rot, bool(pos and pos.interleaved), EPS,
                              pos.magnitude if pos else 1.0), gate)

    def held(self, rc, lo, hi):
        """Keys and values of a request's tokens lo .. hi - 1 as its pages hold them: [n, nkv, d] each."""
        P = self.manager.page_size
        s = self.cache.scales.view(torch.uint8).cpu()
        pages = torch.tensor([rc.tables[0][p // P - rc.page_base[0]] for p in range(lo, hi)])
        slots = torch.arange(lo, hi) % P
        return [f8.dequantise(t.view(torch.uint8).cpu()[pages, :, slots].view(torch.float8_e4m3fn), s[pages, :, slots, which])
                for which, t in enumerate((self.cache.k_pages, self.cache.v_pages))]

    def mask(self):
        return {k: self.options[k] for k in ("window", "chunk", "keep_first") if k in self.options}

    def sink(self):
        return self.tensors["sink"].double().cpu() if self.options.get("sink") else torch.zeros(self.nq).double() if self.options.get("unit_sink") else None


def check_step(layer, got, x, lens, kept, scale=1.0, queries_of=None):
    """``got``: the step's heads; ``kept``: {request: [keys, values]} that grow by what the step wrote; ``queries_of``: the layer whose
    queries read ``layer``'s cache."""
    at, reader = 0, queries_of or layer
    for rc, n in lens.items():
        held = rc.length
        q, _, _, gate = reader.finished(x[at:at + n], range(held, held + n))
        if queries_of is None:
            _, k, v, _ = layer.finished(x[at:at + n], range(held, held + n))
            for new, should in zip(layer.held(rc, held, held + n), (k, v)):
                most = should.abs().amax(-1, keepdim=True)
                assert bool(((new - should).abs() <= should.abs() * 2.0 ** -4 + most * (2.0 ** -10 + 2.0 ** -6)).all())
        old = kept.setdefault(rc.request_id, [torch.zeros(0, layer.nkv, layer.d, dtype=torch.float64)] * 2)
        if old[0].shape[0] < held + n:
            kept[rc.request_id] = old = [torch.cat([a, b]) for a, b in zip(old, layer.held(rc, held, held + n))]
        q = q.to(BF16).double()
        want, spread, size = f8.attention(q, *old, reader.d ** -0.5, held, sink=reader.sink(), **reader.mask())
        g = (torch.sigmoid(gate[:, :, None]) if gate is not None else 1.0) * scale
        off = (got[at:at + n].double().cpu().view(n, reader.nq, reader.d) - want * g).abs()
        share = 2.0 ** -8 + 2 * torch.expm1(2.0 ** -7 * size)[..., None]
        moved = 3 * 2.0 ** -8 + (gate.abs()[:, :, None] * 2.0 ** -8 if gate is not None else 0.0)
        assert bool((off <= (moved * want.abs() + share * spread) * g).all()), (rc.request_id, float((off / (spread * g)).max()))
        at += n


CUTS = [{"a": 130}, {"b": 40, "a": 1}, {"a": 3, "b": 1}, {"c": 33, "a": 17, "b": 5}, {"a": 1, "b": 1, "c": 1}, {"b": 1}]
SIZES = [(8, 2, 128), (6, 3, 48), (8, 1, 64)]
OPTIONS = [dict(), dict(bias=True), dict(head_gate=True), dict(window=40, keep_first=5), dict(window=70), dict(chunk=48), dict(sink=True),
           dict(unit_sink=True, window=33), dict(bias=True, head_gate=True, sink=True, window=60, keep_first=20)]
POSITIONS = [("rope", {"theta": 1e4}), None, ("rope", {"theta": 1e4, "rotary_dim": 16, "pairing": "interleaved"}),
             ("scaled_rope", {"theta": 1e4, "factor": 4.0, "original": 64, "fast": 32.0, "slow": 1.0, "pairing": "half"})]


def rows(n, seed, hidden=HIDDEN):
    return torch.randn(n, hidden, generator=torch.Generator().manual_seed(seed)).to(BF16).to(DEV)


def run_steps(layer, check, cuts=CUTS):
    rcs = {r: layer.manager.open(r) for r in "abc"}
    for i, cut in enumerate(cuts):
        lens = {rcs[r]: n for r, n in cut.items()}
        x = rows(sum(cut.values()), 100 + i)
        check(x, layer.inputs(lens), lens)
        layer.commit(lens)
    from acorninfer_b200.kernels import ops
    torch.cuda.synchronize()
    ops.raise_on_kernel_error()


@pytest.mark.parametrize("nq,nkv,d", SIZES)
@pytest.mark.parametrize("options", OPTIONS, ids=lambda o: "-".join(o) or "plain")
def test_options(nq, nkv, d, options):
    layer, kept = Layer(nq, nkv, d, **options), {}
    run_steps(layer, lambda x, inputs, lens: check_step(layer, layer.mixer.inner(x, inputs, layer.cache), x, lens, kept))


@pytest.mark.parametrize("nq,nkv,d", SIZES)
@pytest.mark.parametrize("position", POSITIONS, ids=["half", "none", "interleaved", "scaled"])
@pytest.mark.parametrize("norm", [True, False])
def test_positions(nq, nkv, d, position, norm):
    layer, kept = Layer(nq, nkv, d, position=position, norm=norm), {}
    run_steps(layer, lambda x, inputs, lens: check_step(layer, layer.mixer.inner(x, inputs, layer.cache), x, lens, kept))


@pytest.mark.parametrize("nq,nkv,d", SIZES)
@pytest.mark.parametrize("gate", [False, True])
def test_scaled_results_in_rows_of_a_wider_buffer(nq, nkv, d, gate):
    layer, kept = Layer(nq, nkv, d, head_gate=gate), {}

    def check(x, inputs, lens):
        wide = torch.full((x.shape[0], nq * d + 16), 7.0, dtype=BF16, device=DEV)
        got = layer.mixer.inner(x, inputs, layer.cache, out_scale=0.375, out=wide[:, 8:8 + nq * d])
        assert got.data_ptr() == wide[:, 8:].data_ptr() and bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + nq * d:] == 7).all())
        check_step(layer, got, x, lens, kept, scale=0.375)

    run_steps(layer, check)


@pytest.mark.parametrize("nq,nkv,d", SIZES)
def test_a_layer_that_reads_another_ones_cache(nq, nkv, d):
    """Its queries over the other layer's keys and values, which stay as they are; fewer of them under a window of its own."""
    from dataclasses import replace
    first, kept = Layer(nq, nkv, d), {}
    second = Layer(nq, nkv, d, seed=2, window=50)

    def check(x, inputs, lens):
        check_step(first, first.mixer.inner(x, inputs, first.cache), x, lens, kept)
        before = [t.view(torch.uint8).clone() for t in (first.cache.k_pages, first.cache.v_pages, first.cache.scales)]
        y = rows(x.shape[0], 900 + x.shape[0])
        check_step(first, second.mixer.inner(y, inputs, replace(first.cache, write=False)), y, lens, kept, queries_of=second)
        assert all(torch.equal(a, t.view(torch.uint8)) for a, t in zip(before, (first.cache.k_pages, first.cache.v_pages, first.cache.scales)))

    run_steps(first, check)
    with pytest.raises(ValueError, match="cache of the run's own"):
        biased, rc = Layer(nq, nkv, d, bias=True), first.manager.open("z")
        biased.mixer.inner(rows(1, 1), first.inputs({rc: 1}), replace(first.cache, write=False))


@pytest.mark.parametrize("nq,nkv,d", [(2, 1, 128), (3, 1, 64), (2, 2, 48)])
@pytest.mark.parametrize("tokens", [1, 5, 60])
@pytest.mark.parametrize("write", [True, False])
def test_angles_of_far_positions(monkeypatch, nq, nkv, d, tokens, write):
    """The finished queries of tokens after 131,000: right to their rounding (2^-8) and 2^-19 of the largest, whoever writes the cache; the
    projection hands its input on, so that nothing else is rounded."""
    from acorninfer_b200.parts import attention as part
    from dataclasses import replace
    hidden = (nq + 2 * nkv) * d
    layer = Layer(nq, nkv, d, pages=8300, eye=True, hidden=hidden, norm=False)
    rc = layer.manager.open("far")
    layer.manager.extend(rc, 131000)
    layer.manager.commit(rc, 131000)
    taken = []
    monkeypatch.setattr(part.attn_kernels, "paged_attention_f8", lambda q, *a, **kw: taken.append(q) or q[:, :nq * d].contiguous())
    x = rows(tokens, 3, hidden)
    layer.mixer.inner(x, layer.inputs({rc: tokens}), replace(layer.cache, write=write))
    want, k, v, _ = layer.finished(x, range(131000, 131000 + tokens))
    off = (taken[0][:, :nq * d].double().cpu().view(tokens, nq, d) - want).abs()
    assert bool((off <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * want.abs().amax(-1, keepdim=True)).all()), float(off.max())
    if write:
        for new, should in zip(layer.held(rc, 131000, 131000 + tokens), (k, v)):
            most = should.abs().amax(-1, keepdim=True)
            assert bool(((new - should).abs() <= should.abs() * 2.0 ** -4 + most * 2.0 ** -10).all())
