"""The write into an 8-bit cache where the norm's sum of squares leaves float32, and its two writers (the kernel of its own, and the
epilogue of the q/k/v product of few rows) on the same rows.  Tolerances: those of ``test_f8_cache_gpu.py``."""

import pytest
import torch

from tests.plain import f8_cache as f8
from tests.test_f8_cache_gpu import check_rows, empty_cache, ops, rows_of, write_inputs, write_wanted

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("nq,nkv,d,rot,inter", [(4, 2, 64, 64, False), (3, 1, 128, 128, False), (6, 3, 96, 48, False), (2, 1, 256, 256, True), (1, 1, 8, 8, True)])
@pytest.mark.parametrize("power", [61, 64, 90, 122])
def test_norms_of_large_rows(nq, nkv, d, rot, inter, power):
    """Rows of entries about 2^power, beside rows of ordinary ones; an infinity still spoils its own row only."""
    P, T, eps = 16, 7, 1e-6
    qkv, w, _, inv = write_inputs(T, nq, nkv, d, rot, True, False, 61)
    qkv = qkv.clamp(-32, 32)
    qkv[::2] *= 2.0 ** power
    positions = torch.arange(T, dtype=torch.int32, device=DEV) * 1000
    cache = empty_cache(T * 1000 // P + 1, nkv, P, d)
    table = torch.arange(cache[0].shape[0], dtype=torch.int32, device=DEV)[None]
    call = lambda x, c: ops().qk_rope_kv_f8(x, w[0], w[1], inv, positions, i32([0] * T), table, i32([0]), *c, nq, nkv, d, rot, inter, eps)    # noqa: E731
    q = call(qkv, cache)
    wq, wk, wv = write_wanted(qkv, w, None, inv, positions, nq, nkv, d, rot, inter, eps, 1.0)
    off = (q.double().cpu().view(T, nq, d) - wq).abs()
    assert bool((off <= 2.0 ** -8 * wq.abs() + 2.0 ** -19 * wq.abs().amax(-1, keepdim=True)).all())
    kc, vc, kb, vb = rows_of(cache, table[0].tolist(), (T - 1) * 1000 + 1, P)
    check_rows(kc[::1000], kb[::1000], wk)
    check_rows(vc[::1000], vb[::1000], wv)
    bad, spoilt = qkv.clone(), empty_cache(cache[0].shape[0], nkv, P, d)
    bad[2, nq * d] = float("inf")                            # a key of token 2
    q2 = call(bad, spoilt)
    assert torch.equal(q2, q)
    _, _, kb2, vb2 = rows_of(spoilt, table[0].tolist(), (T - 1) * 1000 + 1, P)
    assert int(kb2[2000, 0]) == 255
    kb2[2000, 0] = kb[2000, 0]
    assert torch.equal(kb2, kb) and torch.equal(vb2, vb)


@pytest.mark.parametrize("power", [0, 66, 100])
def test_norms_of_large_rows_in_the_epilogue(power):
    """x of about 2^power: q and k as from the product in 64 bits, to the sums' error."""
    o, nq, nkv, d, K, T, P = ops(), 4, 2, 128, 512, 5, 16
    g = torch.Generator().manual_seed(62)
    x = (torch.randn(T, K, generator=g) * 2.0 ** power).to(torch.bfloat16).to(DEV)
    w = (torch.randn((nq + 2 * nkv) * d, K, generator=g) / K ** 0.5).to(torch.bfloat16).to(DEV)
    norms = [(1 + 0.2 * torch.randn(d, generator=g)).to(DEV) for _ in range(2)]
    inv = (1.0 / (1e6 ** (torch.arange(0, d, 2, dtype=torch.float32) / d))).to(DEV)
    pos, cache = torch.arange(T, dtype=torch.int32, device=DEV), empty_cache(1, nkv, P, d)
    out = o.gemm_tc_qkv_rope(x, w, o.RopeKvEpilogue(pos, i32([0] * T), i32([[0]]), i32([0]), cache[0], cache[1], norms[0], norms[1], inv, nq, nkv,
                                                    1e-6, scales=cache[2]))
    assert o.gemm_tc_error() == 0
    proj = x.double() @ w.double().T
    wq, wk, wv = write_wanted(proj, norms, None, inv, pos, nq, nkv, d, d, False, 1e-6, 1.0)
    off = float((x.double().abs() @ w.double().abs().T).amax() * K * 2.0 ** -24)             # of an entry of the product
    size = proj.view(T, -1, d).square().mean(-1).sqrt().cpu()
    move = 1.6 * 2 * off / size                              # as in test_write_as_the_epilogue_of_the_projection
    got = out[:, :nq * d].double().cpu().view(T, nq, d)
    assert bool(((got - wq).abs() <= 2.0 ** -8 * wq.abs() + move[:, :nq, None] + 2.0 ** -19 * wq.abs().amax(-1, keepdim=True)).all())
    kc, vc, kb, vb = rows_of(cache, [0], T, P)
    for codes, byte, want, slack in ((kc, kb, wk, move[:, nq:nq + nkv]), (vc, vb, wv, torch.full((T, nkv), off))):
        e = byte.double() - 127
        spacing = torch.exp2(torch.floor(torch.log2((want.abs() * torch.exp2(-e)[..., None]).clamp(min=2.0 ** -6))) - 3 + e[..., None])
        assert bool(((f8.dequantise(codes, byte) - want).abs() <= spacing / 2 + 2 * slack[..., None]).all())


@pytest.mark.parametrize("nq,nkv,d,rot,inter", [(4, 2, 64, 64, False), (3, 1, 128, 128, False), (6, 3, 96, 48, False), (2, 1, 256, 256, True), (20, 1, 8, 6, True)])
@pytest.mark.parametrize("norm,bias", [(True, False), (False, True)])
def test_queries_alone(nq, nkv, d, rot, inter, norm, bias):
    """Without pages: the bits of the queries of a call that writes, at near and far positions."""
    P, T = 16, 300
    qkv, w, b, inv = write_inputs(T, nq, nkv, d, rot, norm, bias, 63, extra=8)
    positions = torch.arange(T, dtype=torch.int32, device=DEV) * 449
    pages = 300 * 449 // P + 1
    cache, table = empty_cache(pages, nkv, P, d), torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    call = lambda *c, **kw: ops().qk_rope_kv_f8(qkv, w[0], w[1], inv, positions, i32([0] * T), table, i32([0]), *c, nq, nkv, d, rot, inter, 1e-6,     # noqa: E731
                                                bias32=b, magnitude=1.25, **kw)
    want = call(*cache)
    before = qkv.clone()
    assert torch.equal(call(None, None, None), want) and torch.equal(qkv, before)
    out = torch.full((T, nq * d + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    call(None, None, None, out=out)
    assert torch.equal(out[:, :nq * d], want) and bool((out[:, nq * d:] == 7).all())
    for pages_given in ((cache[0], None, None), (None, cache[1], cache[2]), (cache[0], cache[1], None)):
        with pytest.raises(ops().KernelError, match="go together"):
            call(*pages_given)


def test_queries_alone_in_the_epilogue():
    o, nq, nkv, d, K, T, P = ops(), 4, 2, 128, 512, 11, 16
    g = torch.Generator().manual_seed(64)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16).to(DEV)
    w = (torch.randn((nq + 2 * nkv) * d, K, generator=g) / K ** 0.5).to(torch.bfloat16).to(DEV)
    norms = [(1 + 0.2 * torch.randn(d, generator=g)).to(DEV) for _ in range(2)]
    inv = (1.0 / (1e6 ** (torch.arange(0, d, 2, dtype=torch.float32) / d))).to(DEV)
    pos = torch.arange(T, dtype=torch.int32, device=DEV) * 13001
    pages = T * 13001 // P + 1
    cache, table = empty_cache(pages, nkv, P, d), torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    ep = lambda k, v, s, **kw: o.RopeKvEpilogue(pos, i32([0] * T), table, i32([0]), k, v, norms[0], norms[1], inv, nq, nkv, 1e-6, scales=s, **kw)     # noqa: E731
    want = o.gemm_tc_qkv_rope(x, w, ep(*cache))[:, :nq * d]
    assert torch.equal(o.gemm_tc_qkv_rope(x, w, ep(None, None, None, eight_bit=True))[:, :nq * d], want)
    for bad in (ep(cache[0], cache[1], None, eight_bit=True), ep(None, None, cache[2])):
        with pytest.raises(o.KernelError):
            o.gemm_tc_qkv_rope(x, w, bad)


@pytest.mark.parametrize("T", [1, 9, 40])
def test_both_writers_on_the_same_rows(T):
    """A projection that hands its input on (so that both have the same rows): each right to half a spacing and 2^-19, at far positions too."""
    o, nq, nkv, d, P, eps = ops(), 2, 2, 128, 16, 1e-6
    x, wn, _, inv = write_inputs(T, nq, nkv, d, d, True, False, 65)
    pos = 131071 - 7 * torch.arange(T, dtype=torch.int32, device=DEV)
    pages = 131072 // P
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    wq, wk, wv = write_wanted(x, wn, None, inv, pos, nq, nkv, d, d, False, eps, 1.0)
    eye, a, b = torch.eye(x.shape[1]).to(torch.bfloat16).to(DEV), empty_cache(pages, nkv, P, d), empty_cache(pages, nkv, P, d)
    q1 = o.qk_rope_kv_f8(x, wn[0], wn[1], inv, pos, i32([0] * T), table, i32([0]), *a, nq, nkv, d, d, False, eps)
    q2 = o.gemm_tc_qkv_rope(x, eye, o.RopeKvEpilogue(pos, i32([0] * T), table, i32([0]), b[0], b[1], wn[0], wn[1], inv, nq, nkv, eps, scales=b[2]))
    for q, cache in ((q1, a), (q2[:, :nq * d], b)):
        off = (q.double().cpu().view(T, nq, d) - wq).abs()
        assert bool((off <= 2.0 ** -8 * wq.abs() + 2.0 ** -19 * wq.abs().amax(-1, keepdim=True)).all())
        kc, vc, kb, vb = rows_of(cache, table[0].tolist(), 131072, P)
        check_rows(kc[pos.cpu().long()], kb[pos.cpu().long()], wk)
        check_rows(vc[pos.cpu().long()], vb[pos.cpu().long()], wv)
