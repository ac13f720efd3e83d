"""The 8-bit cache's kernels against its definition in 64 bits: the write with norm and rotation, attention of few tokens and
of prompts over its pages, and the calls they refuse.

Tolerances.  The write: a query is rounded once to bfloat16 (2^-8 of it); before that come float32 sums and products of at most
256 terms and an angle right to 2^-22, which move an entry by less than 2^-19 of its row's largest.  A code is the nearest number, so
half a spacing off, plus the same 2^-19.  Attention: the result is rounded to bfloat16 (2^-8 of it); the weights, which meet
exact values, are rounded to 16 bits (2^-8 of each, so at most 2^-8 of the sum of weights times |v|); a score is a float32 sum of d
products (d 2^-24 of the sum of their magnitudes, which is the same share of its weight, once in the numerator and once in the
denominator), its exponential right to 2^-18 of itself."""

import pytest
import torch

from tests.paged import rows_layout
from tests.plain import f8_cache as f8

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def ops():
    from acorninfer_b200.kernels import ops as o
    return o


def raises(match=None):
    return pytest.raises(ops().KernelError, match=match)


def empty_cache(pages, nkv, P, d, byte=127):
    k = torch.zeros(pages, nkv, P, d, dtype=torch.uint8, device=DEV).view(E4M3)
    return k, torch.zeros_like(k.view(torch.uint8)).view(E4M3), torch.full((pages, nkv, P, 2), byte, dtype=torch.uint8, device=DEV).view(E8M0)


def rows_of(cache, table, length, P):
    """(codes, bytes) of keys and of values of a row's first tokens: [length, nkv, d], [length, nkv]."""
    k, v, s = (t.view(torch.uint8).cpu() for t in cache)
    pages = torch.tensor([table[p // P] for p in range(length)])
    slots = torch.arange(length) % P
    kc, vc, sc = k[pages, :, slots], v[pages, :, slots], s[pages, :, slots]
    return kc.view(E4M3), vc.view(E4M3), sc[..., 0], sc[..., 1]


# ------------------------------------------------------------------ the write


def write_inputs(T, nq, nkv, d, rot, norm, bias, seed, extra=0):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, (nq + 2 * nkv) * d + extra, generator=g) * torch.exp(torch.randn(T, 1, generator=g))
    w = [(1 + 0.2 * torch.randn(d, generator=g)).to(DEV) if norm else None for _ in range(2)]
    b = torch.randn((nq + 2 * nkv) * d, generator=g).to(DEV) if bias else None
    inv = 1.0 / (5e5 ** (torch.arange(0, rot, 2, dtype=torch.float32) / max(rot, 1)))
    return qkv.to(torch.bfloat16).to(DEV), w, b, inv.to(DEV)


def write_wanted(qkv, w, b, inv, positions, nq, nkv, d, rot, inter, eps, magnitude):
    x = qkv.double().cpu()[:, :(nq + 2 * nkv) * d]
    if b is not None:
        x = x + b.double().cpu()
    x = x.view(-1, nq + 2 * nkv, d)
    heads = []
    for part, weight in ((x[:, :nq], w[0]), (x[:, nq:nq + nkv], w[1])):
        if weight is not None:
            part = part / torch.sqrt(part.square().mean(-1, keepdim=True) + eps) * weight.double().cpu()
        ang = positions.cpu().double()[:, None, None] * inv.cpu().double()
        c, s = ang.cos() * magnitude, ang.sin() * magnitude
        out = part.clone()
        a_at, b_at = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
        out[..., a_at] = part[..., a_at] * c - part[..., b_at] * s
        out[..., b_at] = part[..., b_at] * c + part[..., a_at] * s
        heads.append(out)
    return heads[0], heads[1], x[:, nq + nkv:]


def check_rows(codes, byte, want):
    """Codes and exponents of rows against the exact rows, to half a spacing and 2^-19 of the row's largest entry."""
    most = want.abs().amax(-1)
    slack = 2.0 ** -19
    e = byte.double() - 127
    assert bool((448 * torch.exp2(e) >= most * (1 - slack)).all())
    assert bool(((448 * torch.exp2(e - 1) < most * (1 + slack)) | (byte == 7)).all())
    spacing = torch.exp2(torch.floor(torch.log2((want.abs() * torch.exp2(-e)[..., None]).clamp(min=2.0 ** -6))) - 3 + e[..., None])
    off = (f8.dequantise(codes, byte) - want).abs()
    assert bool((off <= spacing / 2 + slack * most[..., None]).all())


WRITES = [(4, 2, 64, 64, False, True, False, 16, 1.0), (10, 2, 128, 128, False, True, False, 8, 1.0), (3, 1, 128, 32, True, True, True, 32, 1.3),
          (6, 3, 96, 48, False, False, True, 1, 1.0), (5, 5, 8, 8, True, True, False, 4, 0.7), (2, 1, 256, 256, False, True, False, 16, 1.0),
          (32, 8, 128, 128, False, True, False, 16, 1.0), (1, 1, 16, 0, False, False, False, 2, 1.0), (7, 1, 40, 6, True, True, True, 64, 1.0)]


@pytest.mark.parametrize("nq,nkv,d,rot,inter,norm,bias,P,magnitude", WRITES)
@pytest.mark.parametrize("qlens", [[21, 1, 2, 17], [1], [400, 1, 2, 17]])
def test_write(nq, nkv, d, rot, inter, norm, bias, P, magnitude, qlens):
    befores, eps = [0, 37, 131071, 15][:len(qlens)], 2e-6
    pages = sum(-(-(b + n) // P) for b, n in zip(befores, qlens)) + 5
    lay = rows_layout(befores, qlens, P, pages, seed=1)
    T = lay["num_tokens"]
    qkv, w, b, inv = write_inputs(T, nq, nkv, d, rot, norm, bias, 7, extra=8)
    cache = empty_cache(pages, nkv, P, d, byte=99)
    before = qkv.clone()
    q = ops().qk_rope_kv_f8(qkv, w[0], w[1], inv, lay["positions"], lay["token_row"], lay["block_table"], lay["page_base"], *cache,
                            nq, nkv, d, rot, inter, eps, bias32=b, magnitude=magnitude)
    assert torch.equal(qkv, before) and q.shape == (T, nq * d)
    wq, wk, wv = write_wanted(qkv, w, b, inv, lay["positions"], nq, nkv, d, rot, inter, eps, magnitude)
    off = (q.double().cpu().view(T, nq, d) - wq).abs()
    assert bool((off <= 2.0 ** -8 * wq.abs() + 2.0 ** -19 * wq.abs().amax(-1, keepdim=True)).all())
    at, used = 0, torch.zeros(pages, P, dtype=torch.bool)
    for r, (held, n) in enumerate(zip(befores, qlens)):
        kc, vc, kb, vb = rows_of(cache, lay["tables"][r], held + n, P)
        check_rows(kc[held:], kb[held:], wk[at:at + n])
        if b is None:                                        # values as projected: the definition to the bit
            codes, e = f8.quantise(wv[at:at + n])
            held_codes, byte = f8.to_tensors(codes, e)
            assert torch.equal(vc[held:].view(torch.uint8), held_codes.view(torch.uint8)) and torch.equal(vb[held:], byte)
        else:
            check_rows(vc[held:], vb[held:], wv[at:at + n])
        for p in range(held, held + n):
            used[lay["tables"][r][p // P], p % P] = True
        at += n
    # slots of no token of the step stay as they were
    for t in cache[:2]:
        assert int(t.view(torch.uint8).cpu().transpose(1, 2)[~used].sum()) == 0
    assert bool((cache[2].view(torch.uint8).cpu().transpose(1, 2)[~used] == 99).all())


def test_write_rows_of_every_size():
    """Value rows over the whole range of bfloat16: zeros, subnormal numbers, the largest, ties, numbers that are none."""
    nkv, d, P = 1, 64, 16
    top = torch.finfo(torch.bfloat16).max
    rows = [torch.zeros(d), torch.full((d,), 2.0 ** -133), torch.linspace(-448, 448, d), torch.linspace(-449, 449, d),
            torch.linspace(-1, 1, d) * top, torch.full((d,), 1.75 * 2.0 ** 127), torch.full((d,), -top),
            torch.tensor([448.0] + [17 + 2.0 * i for i in range(d - 1)]),                # ties between neighbours of spacing 2
            torch.tensor([448.0] + [2.0 ** -10 * (2 * i + 1) for i in range(d - 1)]),     # ties among the subnormal codes
            torch.linspace(-1, 1, d) * 2.0 ** -111, torch.linspace(-1, 1, d) * 2.0 ** -113, torch.linspace(1, 2, d) * 2.0 ** -126]
    rows += [r.clone() for r in (rows[2], rows[2], rows[2], rows[2])]
    rows[-4][5], rows[-3][0], rows[-2][63], rows[-1][7] = float("nan"), float("inf"), float("-inf"), -0.0
    T = len(rows)
    v = torch.stack(rows).to(torch.bfloat16)
    qkv = torch.cat([torch.ones(T, 2 * d, dtype=torch.bfloat16), v], 1).to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    cache = empty_cache(2, nkv, P, d)
    ops().qk_rope_kv_f8(qkv, None, None, torch.zeros(0, device=DEV), torch.arange(T, **i32), torch.zeros(T, **i32),
                        torch.tensor([[1, 0]], **i32), torch.zeros(1, **i32), *cache, 1, nkv, d, 0, False, 0.0)
    _, vc, _, vb = rows_of(cache, [1, 0], T, P)
    codes, e = f8.quantise(v.double()[:, None])
    held, byte = f8.to_tensors(codes, e)
    assert torch.equal(vc.float(), held.float()) and torch.equal(vb, byte)
    assert bool(torch.isfinite(f8.dequantise(vc, vb).float()[:-4]).all())
    back = f8.dequantise(vc, vb)[torch.isfinite(v).all(-1)]
    assert torch.equal(back.to(torch.bfloat16).double(), back)              # every row is one of bfloat16 numbers


def test_write_numbers_that_are_none_stay_in_their_rows():
    nq, nkv, d, P, T = 2, 2, 128, 16, 5
    qkv, w, _, inv = write_inputs(T, nq, nkv, d, d, True, False, 3)
    clean = empty_cache(1, nkv, P, d), empty_cache(1, nkv, P, d)
    i32 = dict(dtype=torch.int32, device=DEV)
    args = (w[0], w[1], inv, torch.arange(T, **i32), torch.zeros(T, **i32), torch.zeros(1, 1, **i32), torch.zeros(1, **i32))
    q0 = ops().qk_rope_kv_f8(qkv, *args, *clean[0], nq, nkv, d, d, False, 1e-6)
    bad = qkv.clone()
    bad[1, nq * d + 3] = float("inf")                        # token 1: key head 0
    bad[3, (nq + 2 * nkv - 1) * d] = float("nan")            # token 3: value head 1
    q1 = ops().qk_rope_kv_f8(bad, *args, *clean[1], nq, nkv, d, d, False, 1e-6)
    assert torch.equal(q0, q1)
    k0, v0, a0, b0 = rows_of(clean[0], [0], T, P)
    k1, v1, a1, b1 = rows_of(clean[1], [0], T, P)
    assert int(a1[1, 0]) == 255 and int(b1[3, 1]) == 255 and float(k1[1, 0].float().abs().sum()) == 0
    a1[1, 0], b1[3, 1] = a0[1, 0], b0[3, 1]
    k1.view(torch.uint8)[1, 0], v1.view(torch.uint8)[3, 1] = k0.view(torch.uint8)[1, 0], v0.view(torch.uint8)[3, 1]
    assert torch.equal(a0, a1) and torch.equal(b0, b1)
    assert torch.equal(k0.view(torch.uint8), k1.view(torch.uint8)) and torch.equal(v0.view(torch.uint8), v1.view(torch.uint8))


def test_write_refusals():
    nq, nkv, d, P, T = 4, 2, 64, 16, 3
    qkv, w, b, inv = write_inputs(T, nq, nkv, d, d, True, True, 3)
    i32 = dict(dtype=torch.int32, device=DEV)
    pos, row, table, base = torch.arange(T, **i32), torch.zeros(T, **i32), torch.zeros(1, 1, **i32), torch.zeros(1, **i32)
    k, v, s = empty_cache(2, nkv, P, d)
    call = lambda qkv=qkv, qw=w[0], inv=inv, pos=pos, table=table, k=k, v=v, s=s, nq=nq, nkv=nkv, d=d, rot=d, **kw: \
        ops().qk_rope_kv_f8(qkv, qw, w[1], inv, pos, row, table, base, k, v, s, nq, nkv, d, rot, False, 1e-6, **kw)   # noqa: E731
    call()
    for bad in (dict(qkv=qkv.float()), dict(qkv=qkv[:, 8:]), dict(qkv=qkv.cpu()), dict(qw=w[0][:32].contiguous()), dict(qw=w[0].half()),
                dict(inv=inv[:-1].contiguous()), dict(pos=pos.long()), dict(pos=pos[:2].contiguous()), dict(table=table[0]),
                dict(k=k.view(torch.uint8)), dict(v=v[:1]), dict(s=s.view(torch.uint8)), dict(s=s[:, :, :, :1].contiguous()),
                dict(nq=5), dict(nkv=1), dict(d=32), dict(rot=8), dict(rot=d + 16), dict(bias32=b[:-1].contiguous()),
                dict(out=torch.empty(T, nq * d, device=DEV)), dict(out=torch.empty(T - 1, nq * d, device=DEV, dtype=torch.bfloat16)),
                dict(k=k.transpose(1, 2), v=v.transpose(1, 2))):
        with raises():
            call(**bad)
    three = empty_cache(2, nkv, 3, d)
    with raises("power of two"):
        call(k=three[0], v=three[1], s=three[2])
    assert call(qkv=qkv[:0], pos=pos[:0]).shape == (0, nq * d)               # no tokens: nothing to do


# ------------------------------------------------------------------ attention


def random_cache(befores, qlens, nkv, d, P, seed, spoil=()):
    """A cache whose pages no token owns, and whose slots beyond a row's end, hold codes and exponents of any kind; the
    rows' keys and values in 64 bits.  ``spoil``: (row, token, kv head, 0 key / 1 value) to be stored as no number."""
    g = torch.Generator().manual_seed(seed)
    pages = sum(-(-(b + n) // P) for b, n in zip(befores, qlens)) + 7
    lay = rows_layout(befores, qlens, P, pages, seed=seed)
    junk = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8)                              # noqa: E731
    k, v, s = junk(pages, nkv, P, d), junk(pages, nkv, P, d), junk(pages, nkv, P, 2)
    keys, values = [], []
    for r, (held, n) in enumerate(zip(befores, qlens)):
        L = held + n
        at = torch.tensor([lay["tables"][r][p // P] for p in range(L)]), torch.arange(L) % P
        for which, (pages_of, kept) in enumerate(((k, keys), (v, values))):
            x = torch.randn(L, nkv, d, generator=g) * torch.exp((0.3, 1.5)[which] * torch.randn(L, nkv, 1, generator=g))
            codes, e = f8.quantise(x)
            held_codes, byte = f8.to_tensors(codes, e)
            for row, token, head, kind in spoil:
                if row == r and kind == which:
                    held_codes.view(torch.uint8)[token, head], byte[token, head] = 0, 255
            pages_of[at[0], :, at[1]] = held_codes.view(torch.uint8)
            s[at[0], :, at[1], which] = byte
            kept.append(f8.dequantise(held_codes, byte))
    lay["row_start"] = torch.tensor([sum(qlens[:r]) for r in range(len(qlens) + 1)], dtype=torch.int32, device=DEV)
    lay["row_pos"] = torch.tensor(befores, dtype=torch.int32, device=DEV)
    return lay, (k.to(DEV).view(E4M3), v.to(DEV).view(E4M3), s.to(DEV).view(E8M0)), keys, values


def tiles_of(qlens, step):
    return torch.tensor([(r, q0) for r, n in enumerate(qlens) for q0 in range(0, n, step)], dtype=torch.int32, device=DEV).view(-1, 2)


def attend(which, q, cache, lay, qlens, nq, nkv, d, scale, stride=None, **kw):
    o = ops()
    step = o.f8_tile_tokens(nq, nkv) if which == "decode" else o.F8_PREFILL_TILE
    fn = o.attention_decode_f8 if which == "decode" else o.attention_prefill_f8
    tiles = kw.pop("tiles", None)
    window = kw.pop("window", None)
    return fn(q, stride or q.stride(0), *cache, lay["block_table"], lay["page_base"], lay["row_start"], lay["row_pos"],
              tiles_of(qlens, step) if tiles is None else tiles, lay["num_tokens"], nq, nkv, d, scale, window, **kw)


def check_attention(got, q, keys, values, befores, qlens, nq, d, scale, weights_off=2.0 ** -8, **mask):
    at = 0
    sink = mask.pop("sink32", None)
    for r, (held, n) in enumerate(zip(befores, qlens)):
        want, spread, size = f8.attention(q[at:at + n].double().cpu().view(n, nq, d), keys[r], values[r], scale, held,
                                          sink=None if sink is None else sink.cpu(), **mask)
        have = got[at:at + n].double().cpu().view(n, nq, d)
        assert torch.equal(torch.isnan(have), torch.isnan(want))
        share = weights_off + 2 * (2.0 ** -18 + d * 2.0 ** -24 * size)[..., None]
        off = torch.nan_to_num(have - want).abs()
        assert bool((off <= 2.0 ** -8 * torch.nan_to_num(want).abs() + share * spread).all()), (r, float((off / (spread + 1e-30)).max()))
        at += n


# around the kernels' tiles and blocks (16, 32, 64 and 128 keys; 16 rows and 128 queries), one token to many
BEFORES = [0, 300, 129, 16, 0, 1100, 63, 127, 64, 2047]
QLENS = [150, 1, 2, 1, 1, 3, 1, 130, 5, 1]
SIZES = [(32, 8, 128, 16), (8, 8, 128, 8), (12, 2, 64, 16), (4, 4, 64, 32), (16, 1, 128, 64), (10, 2, 128, 128), (5, 1, 64, 256),
         (6, 3, 128, 16), (16, 8, 64, 8), (3, 1, 40, 4), (20, 1, 64, 16), (4, 2, 256, 16), (34, 2, 128, 16), (4, 2, 128, 2)]


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("nq,nkv,d,P", SIZES)
def test_attention(which, nq, nkv, d, P):
    lay, cache, keys, values = random_cache(BEFORES, QLENS, nkv, d, P, 2)
    T, scale = lay["num_tokens"], d ** -0.5
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(T, nq * d + 64, generator=g).to(torch.bfloat16).to(DEV)         # queries at the head of wider rows
    got = attend(which, wide, cache, lay, QLENS, nq, nkv, d, scale)
    assert got.shape == (T, nq * d) and got.dtype == torch.bfloat16
    check_attention(got, wide[:, :nq * d], keys, values, BEFORES, QLENS, nq, d, scale)
    # the same rows from a buffer of their own width: the same bits
    assert torch.equal(got, attend(which, wide[:, :nq * d].contiguous(), cache, lay, QLENS, nq, nkv, d, scale))


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("mask", [dict(window=1), dict(window=33), dict(window=700), dict(chunk=48), dict(chunk=256, window=100),
                                  dict(window=70, keep_first=5), dict(window=130, keep_first=200), dict(keep_first=3, chunk=64),
                                  dict(sink32=True), dict(window=40, keep_first=2, sink32=True), dict(window=5000)])
@pytest.mark.parametrize("nq,nkv,d,P", [(8, 2, 128, 16), (6, 1, 64, 8), (2, 1, 24, 16)])
def test_attention_masks(which, mask, nq, nkv, d, P):
    lay, cache, keys, values = random_cache(BEFORES, QLENS, nkv, d, P, 3)
    scale = d ** -0.5
    mask = dict(mask)
    g = torch.Generator().manual_seed(6)
    if mask.get("sink32"):
        mask["sink32"] = (3 * torch.randn(nq, generator=g)).to(DEV)
    q = torch.randn(lay["num_tokens"], nq * d, generator=g).to(torch.bfloat16).to(DEV)
    got = attend(which, q, cache, lay, QLENS, nq, nkv, d, scale, **mask)
    check_attention(got, q, keys, values, BEFORES, QLENS, nq, d, scale, **mask)


@pytest.mark.parametrize("which", ["decode", "prefill"])
def test_attention_of_a_windowed_row_that_gave_pages_back(which):
    """The table starts at the first page that the window still reads; the pages before are another's."""
    nq, nkv, d, P, window = 8, 2, 128, 16, 100
    befores, qlens = [900, 333], [3, 200]
    lay, cache, keys, values = random_cache(befores, qlens, nkv, d, P, 4)
    table = torch.zeros_like(lay["block_table"])
    base = [(b - window + 1) // P for b in befores]
    for r, b in enumerate(base):
        kept = lay["tables"][r][b:]
        table[r, :len(kept)] = torch.tensor(kept, dtype=torch.int32)
    lay["block_table"], lay["page_base"] = table, torch.tensor(base, dtype=torch.int32, device=DEV)
    q = torch.randn(lay["num_tokens"], nq * d).to(torch.bfloat16).to(DEV)
    got = attend(which, q, cache, lay, qlens, nq, nkv, d, 0.1, window=window)
    check_attention(got, q, keys, values, befores, qlens, nq, d, 0.1, window=window)


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("d", [64, 128, 48])
def test_attention_of_rows_that_differ_in_size(which, d):
    """Values of tokens from 2^-40 to 2^40, the largest where the weights are smallest; keys one of which decides all."""
    nq, nkv, P, L = 4, 2, 16, 300
    befores, qlens = [L - 4], [4]
    lay, cache, keys, values = random_cache(befores, qlens, nkv, d, P, 8)
    g = torch.Generator().manual_seed(1)
    for spread in (0, 20, 40):
        size = torch.linspace(-spread, spread, L)[torch.randperm(L, generator=g)]
        x = torch.randn(L, nkv, d, generator=g) * torch.exp2(size)[:, None, None]
        y = torch.randn(L, nkv, d, generator=g) * 0.05
        y[:, :, 0] = -size[:, None] * 0.69                     # a weight times its value's size is about 1
        q = 0.02 * torch.randn(4, nq * d, generator=g)
        q.view(4, nq, d)[..., 0] = 1
        q = q.to(torch.bfloat16).to(DEV)
        at = torch.tensor([lay["tables"][0][p // P] for p in range(L)], device=DEV), torch.arange(L, device=DEV) % P
        for which_, (pages, rows) in enumerate(((cache[0], y), (cache[1], x))):
            codes, byte = f8.to_tensors(*f8.quantise(rows))
            pages.view(torch.uint8)[at[0], :, at[1]] = codes.view(torch.uint8).to(DEV)
            cache[2].view(torch.uint8)[at[0], :, at[1], which_] = byte.to(DEV)
            (keys, values)[which_][0] = f8.dequantise(codes, byte)
        got = attend(which, q, cache, lay, qlens, nq, nkv, d, 1.0)
        check_attention(got, q, keys, values, befores, qlens, nq, d, 1.0)


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("nq,nkv,d,P", [(8, 2, 128, 16), (8, 4, 64, 16), (4, 2, 32, 8)])
def test_attention_numbers_that_are_none_reach_the_queries_that_read_them(which, nq, nkv, d, P):
    befores, qlens = [0, 290, 140], [150, 1, 5]
    # row 0: key of token 70 (head 0) and value of token 149 (head 1); row 1: a value outside the window; row 2: its newest key
    spoil = [(0, 70, 0, 0), (0, 149, 1, 1), (1, 3, 0, 1), (2, 144, 1, 0)]
    lay, cache, keys, values = random_cache(befores, qlens, nkv, d, P, 9, spoil)
    q = torch.randn(lay["num_tokens"], nq * d).to(torch.bfloat16).to(DEV)
    for mask in (dict(window=200), dict(window=40)):
        got = attend(which, q, cache, lay, qlens, nq, nkv, d, 0.11, **mask)
        check_attention(got, q, keys, values, befores, qlens, nq, d, 0.11, **mask)
    # a query that is no number spoils its own head only
    for bad in (float("nan"), float("inf"), float("-inf")):
        q2 = q.clone()
        q2[151, d + 1] = bad                                   # row 2's first query, head 1
        new = attend(which, q2, cache, lay, qlens, nq, nkv, d, 0.11, window=40)
        assert bool(torch.isnan(new[151].view(nq, d)[1]).all())
        same = torch.ones(got.shape[0], nq, dtype=torch.bool)
        same[151, 1] = False
        a, b = new.view(-1, nq, d).cpu()[same], got.view(-1, nq, d).cpu()[same]
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.nan_to_num(a), torch.nan_to_num(b))


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("d", [128, 64, 16])
def test_attention_of_large_and_small_queries(which, d):
    """Queries over bfloat16's range: tiny ones weigh all keys alike, huge ones choose one key."""
    nq, nkv, P = 4, 2, 16
    befores, qlens = [77], [4]
    lay, cache, keys, values = random_cache(befores, qlens, nkv, d, P, 11)
    q = torch.randn(4, nq * d)
    q *= torch.tensor([2.0 ** -100, 2.0 ** 60, 2.0 ** 10, 1.0])[:, None]
    q[2, 1::2] *= 2.0 ** -60
    q = q.to(torch.bfloat16).to(DEV)
    got = attend(which, q, cache, lay, qlens, nq, nkv, d, d ** -0.5)
    # where scores are huge one key takes all: the yardstick of a score's error no longer says anything
    rows = [0, 3]
    for i in range(4):
        want, spread, size = f8.attention(q[i:i + 1].double().cpu().view(1, nq, d), keys[0], values[0], d ** -0.5, 77 + i)
        have = got[i:i + 1].double().cpu().view(1, nq, d)
        if i in rows:
            share = 2.0 ** -8 + 2 * (2.0 ** -18 + d * 2.0 ** -24 * size)[..., None]
            assert bool(((have - want).abs() <= 2.0 ** -8 * want.abs() + share * spread).all())
        else:
            assert bool(((have - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -7 * spread).all())


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("d", [128, 64, 24])
def test_attention_leaves_other_rows_and_reads_listed_tiles(which, d):
    nq, nkv, P = 8, 2, 16
    befores, qlens = [40, 0, 200], [1, 7, 2]
    lay, cache, keys, values = random_cache(befores, qlens, nkv, d, P, 12)
    q = torch.randn(lay["num_tokens"], nq * d).to(torch.bfloat16).to(DEV)
    out = torch.full((lay["num_tokens"] + 3, nq * d), 7.0, dtype=torch.bfloat16, device=DEV)
    tiles = tiles_of([0, 0, 2], 4)
    whole = attend(which, q, cache, lay, qlens, nq, nkv, d, 0.2)
    assert attend(which, q, cache, lay, qlens, nq, nkv, d, 0.2, out=out, tiles=tiles) is out
    assert bool((out[:8] == 7).all()) and bool((out[10:] == 7).all()) and torch.equal(out[8:10], whole[8:10])
    # no tiles: nothing is launched, nothing written
    attend(which, q, cache, lay, qlens, nq, nkv, d, 0.2, out=out, tiles=tiles[:0])
    assert bool((out[:8] == 7).all())


@pytest.mark.parametrize("which", ["decode", "prefill"])
def test_attention_on_two_streams_and_replayed(which):
    """Two calls at once on streams of their own, each captured into a graph; replays read what the buffers hold then."""
    nq, nkv, d, P = 8, 2, 128, 16
    befores, qlens = [500, 900], [1, 3]
    made = [random_cache(befores, qlens, nkv, d, P, 20 + i) for i in range(2)]
    qs = [torch.randn(4, nq * d).to(torch.bfloat16).to(DEV) for _ in range(2)]
    tiles = tiles_of(qlens, ops().f8_tile_tokens(nq, nkv) if which == "decode" else 128)
    call = lambda i, out=None: attend(which, qs[i], made[i][1], made[i][0], qlens, nq, nkv, d, 0.1, tiles=tiles, out=out)    # noqa: E731
    call(0)
    want = [call(0), call(1)]
    graphs, outs, streams = [], [torch.empty_like(w) for w in want], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[i]):
            call(i, outs[i])
        graphs.append(graph)
    for _ in range(5):
        for i in range(2):
            outs[i].zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    qs[0].copy_(qs[1])
    graphs[0].replay()
    torch.cuda.synchronize()
    new = call(0)
    assert torch.equal(outs[0], new) and not torch.equal(new, want[0])


@pytest.mark.parametrize("which", ["decode", "prefill"])
def test_attention_refusals(which):
    nq, nkv, d, P = 4, 2, 64, 16
    lay, (k, v, s), _, _ = random_cache([20, 5], [3, 1], nkv, d, P, 1)
    q = torch.randn(4, nq * d).to(torch.bfloat16).to(DEV)
    tiles = tiles_of([3, 1], 4)
    fn = ops().attention_decode_f8 if which == "decode" else ops().attention_prefill_f8

    def call(q=q, stride=nq * d, k=k, v=v, s=s, table=lay["block_table"], base=lay["page_base"], start=lay["row_start"],
             pos=lay["row_pos"], tiles=tiles, T=4, nq=nq, nkv=nkv, d=d, window=None, **kw):
        return fn(q, stride, k, v, s, table, base, start, pos, tiles, T, nq, nkv, d, 0.1, window, **kw)

    call()
    for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q.t()), dict(stride=nq * d - 8), dict(stride=nq * d + 4), dict(stride=nq * d + 8),
                dict(T=5), dict(k=k.view(torch.uint8)), dict(v=v[1:]), dict(s=s.view(torch.uint8)), dict(s=s[..., :1].contiguous()),
                dict(table=lay["block_table"].long()), dict(base=lay["page_base"][:1]), dict(start=lay["row_start"][:2]),
                dict(pos=lay["row_pos"].cpu()), dict(tiles=tiles.view(-1)), dict(tiles=torch.cat([tiles, tiles], 1)), dict(nq=5), dict(nkv=4),
                dict(d=32), dict(window=-1), dict(chunk=-2), dict(keep_first=-1), dict(sink32=torch.zeros(3, device=DEV)),
                dict(out=torch.empty(3, nq * d, dtype=torch.bfloat16, device=DEV)), dict(out=torch.empty(4, nq * d, device=DEV))):
        with raises():
            call(**bad)
    for size in ((1, 1, 16, 12), (1, 1, 16, 264), (1, 1, 12, 64)):           # head sizes 12 and 264, 12 tokens a page
        pages, heads, P_, d_ = size
        kk, vv, ss = empty_cache(pages, heads, P_, d_)
        with raises():
            call(q=torch.zeros(4, d_ + (-d_) % 8, dtype=torch.bfloat16, device=DEV), stride=d_ + (-d_) % 8, k=kk, v=vv, s=ss, nq=1, nkv=1, d=d_)


def test_written_then_read():
    """The pieces as a layer uses them: rows written in portions, each followed by its attention, a decoded token last; the
    attention of what was written is that of the rows in 64 bits, to the codes' half spacing."""
    nq, nkv, d, P = 8, 2, 128, 16
    portions = [130, 1, 3, 40, 1]
    o, i32 = ops(), dict(dtype=torch.int32, device=DEV)
    cache = empty_cache(20, nkv, P, d)
    table = torch.randperm(20, generator=torch.Generator().manual_seed(0)).to(torch.int32).to(DEV)[None]
    base, held = torch.zeros(1, **i32), 0
    for n in portions:
        qkv, w, _, inv = write_inputs(n, nq, nkv, d, d, True, False, 50 + held)
        pos = torch.arange(held, held + n, **i32)
        q = o.qk_rope_kv_f8(qkv, w[0], w[1], inv, pos, torch.zeros(n, **i32), table, base, *cache, nq, nkv, d, d, False, 1e-6)
        lay = {"block_table": table, "page_base": base, "row_start": torch.tensor([0, n], **i32),
               "row_pos": torch.tensor([held], **i32), "num_tokens": n}
        held += n
        kc, vc, kb, vb = rows_of(cache, table[0].tolist(), held, P)
        keys, values = [f8.dequantise(kc, kb)], [f8.dequantise(vc, vb)]
        both = [attend(which, q, cache, lay, [n], nq, nkv, d, d ** -0.5) for which in ("decode", "prefill")]
        for got in both:
            check_attention(got, q, keys, values, [held - n], [n], nq, d, d ** -0.5)


@pytest.mark.parametrize("which,nq,nkv,d", [("decode", 8, 2, 128), ("prefill", 4, 2, 64)])
def test_attention_does_not_depend_on_the_other_rows(which, nq, nkv, d):
    """A row alone and the same row among others: the same bits (one split of its keys in both)."""
    befores, qlens = [100, 37, 220], [2, 1, 4]
    lay, cache, _, _ = random_cache(befores, qlens, nkv, d, 16, 13)
    q = torch.randn(7, nq * d).to(torch.bfloat16).to(DEV)
    kw = dict(num_splits=1) if which == "decode" else {}
    whole = attend(which, q, cache, lay, qlens, nq, nkv, d, 0.1, **kw)
    for r, (a, b) in enumerate(((0, 2), (2, 3), (3, 7))):
        alone = {"block_table": lay["block_table"][r:r + 1].contiguous(), "page_base": lay["page_base"][:1],
                 "row_start": torch.tensor([0, b - a], dtype=torch.int32, device=DEV), "row_pos": lay["row_pos"][r:r + 1],
                 "num_tokens": b - a}
        assert torch.equal(attend(which, q[a:b].contiguous(), cache, alone, [b - a], nq, nkv, d, 0.1, **kw), whole[a:b])


@pytest.mark.parametrize("nq,nkv,K,qlens,norm,P", [(4, 2, 256, [7, 1, 5], True, 16), (6, 1, 520, [1, 1, 1, 1], False, 8), (2, 2, 2048, [30], True, 32),
                                                   (8, 4, 1024, [3, 20], True, 16), (4, 2, 1024, [41, 1], True, 16), (1, 1, 64, [1], True, 1)])
def test_write_as_the_epilogue_of_the_projection(nq, nkv, K, qlens, norm, P):
    """The q/k/v product of few rows that norms, rotates, quantises and writes.  Its sums of K float32 terms are off by less than
    K 2^-24 of the sum of their magnitudes; a key's norm divides by the row's own size, so that share of a row stays."""
    o, d, eps = ops(), 128, 3e-6
    befores = [0, 37, 131000, 15][:len(qlens)]
    pages = sum(-(-(b + n) // P) for b, n in zip(befores, qlens)) + 5
    lay = rows_layout(befores, qlens, P, pages, seed=2)
    T = lay["num_tokens"]
    g = torch.Generator().manual_seed(K)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16).to(DEV)
    w = (torch.randn((nq + 2 * nkv) * d, K, generator=g) / K ** 0.5).to(torch.bfloat16).to(DEV)
    norms = [(1 + 0.2 * torch.randn(d, generator=g)).to(DEV) if norm else None for _ in range(2)]
    inv = (1.0 / (1e6 ** (torch.arange(0, d, 2, dtype=torch.float32) / d))).to(DEV)
    cache = empty_cache(pages, nkv, P, d, byte=99)
    out = o.gemm_tc_qkv_rope(x, w, o.RopeKvEpilogue(lay["positions"], lay["token_row"], lay["block_table"], lay["page_base"], cache[0], cache[1],
                                                    norms[0], norms[1], inv, nq, nkv, eps, scales=cache[2]))
    assert o.gemm_tc_error() == 0
    proj = x.double() @ w.double().T
    off = float((x.double().abs() @ w.double().abs().T).amax() * K * 2.0 ** -24)            # of an entry of the product
    wq, wk, wv = write_wanted(proj, norms, None, inv, lay["positions"], nq, nkv, d, d, False, eps, 1.0)
    # 1.6: the largest norm weight; a rotation adds two entries; a norm divides by the row's root mean square
    size = proj.view(T, -1, d).square().mean(-1).sqrt().cpu()
    move = 1.6 * 2 * off / (size if norm else torch.ones_like(size))
    got = out[:, :nq * d].double().cpu().view(T, nq, d)
    assert bool(((got - wq).abs() <= 2.0 ** -8 * wq.abs() + move[:, :nq, None] + 2.0 ** -19 * wq.abs().amax(-1, keepdim=True)).all())
    at, used = 0, torch.zeros(pages, P, dtype=torch.bool)
    for r, (held, n) in enumerate(zip(befores, qlens)):
        kc, vc, kb, vb = rows_of(cache, lay["tables"][r], held + n, P)
        for codes, byte, want, slack in ((kc, kb, wk, move[:, nq:nq + nkv]), (vc, vb, wv, torch.full((T, nkv), off))):
            want, slack = want[at:at + n], slack[at:at + n]
            codes, byte = codes[held:], byte[held:]
            e, most = byte.double() - 127, want.abs().amax(-1)
            assert bool((448 * torch.exp2(e) >= most - slack).all()) and bool((448 * torch.exp2(e - 1) < most + slack).all())
            spacing = torch.exp2(torch.floor(torch.log2((want.abs() * torch.exp2(-e)[..., None]).clamp(min=2.0 ** -6))) - 3 + e[..., None])
            assert bool(((f8.dequantise(codes, byte) - want).abs() <= spacing / 2 + 2 * slack[..., None]).all())
        for p in range(held, held + n):
            used[lay["tables"][r][p // P], p % P] = True
        at += n
    for t in cache[:2]:
        assert int(t.view(torch.uint8).cpu().transpose(1, 2)[~used].sum()) == 0
    assert bool((cache[2].view(torch.uint8).cpu().transpose(1, 2)[~used] == 99).all())


def test_the_epilogue_writes_rows_that_are_no_numbers_as_such():
    o, nq, nkv, d, K, T, P = ops(), 2, 2, 128, 256, 4, 16
    x = torch.randn(T, K).to(torch.bfloat16).to(DEV)
    w = (torch.randn((nq + 2 * nkv) * d, K) / 16).to(torch.bfloat16).to(DEV)
    inv = (1.0 / (1e6 ** (torch.arange(0, d, 2, dtype=torch.float32) / d))).to(DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    x[2, 5] = float("inf")
    cache = empty_cache(1, nkv, P, d)
    o.gemm_tc_qkv_rope(x, w, o.RopeKvEpilogue(torch.arange(T, **i32), torch.zeros(T, **i32), torch.zeros(1, 1, **i32), torch.zeros(1, **i32), cache[0],
                                              cache[1], None, None, inv, nq, nkv, 0.0, scales=cache[2]))
    s = cache[2].view(torch.uint8)[0, :, :T].cpu()
    assert bool((s[:, 2] == 255).all()) and bool((s[:, [0, 1, 3]] < 255).all())
    assert int(cache[0].view(torch.uint8)[0, :, 2].sum()) == int(cache[1].view(torch.uint8)[0, :, 2].sum()) == 0
    with raises("8-bit"):                                                   # more rows than the kernel of few rows takes
        many = torch.zeros(64, K, dtype=torch.bfloat16, device=DEV)
        o.gemm_tc_qkv_rope(many, w, o.RopeKvEpilogue(torch.arange(64, **i32), torch.zeros(64, **i32), torch.zeros(1, 4, **i32), torch.zeros(1, **i32),
                                                     cache[0], cache[1], None, None, inv, nq, nkv, 0.0, scales=cache[2]))
    with raises():                                                          # bfloat16 pages with scales
        o.gemm_tc_qkv_rope(x, w, o.RopeKvEpilogue(torch.arange(T, **i32), torch.zeros(T, **i32), torch.zeros(1, 1, **i32), torch.zeros(1, **i32),
                                                  cache[0].bfloat16(), cache[1].bfloat16(), None, None, inv, nq, nkv, 0.0, scales=cache[2]))


@pytest.mark.parametrize("which", ["decode", "prefill"])
@pytest.mark.parametrize("d", [128, 64, 32])
def test_attention_wherever_the_pages_lie(which, d):
    """Value pages before the key pages in memory, far from them, and the key pages themselves as values."""
    nq, nkv, P = 8, 2, 16
    befores, qlens = [77, 500], [3, 40]
    lay, (k, v, s), keys, values = random_cache(befores, qlens, nkv, d, P, 14)
    q = torch.randn(43, nq * d).to(torch.bfloat16).to(DEV)
    n = k.numel()
    room = torch.zeros(3 * n, dtype=torch.uint8, device=DEV)
    lower, upper = (room[i * n:(i + 1) * n].view(E4M3).view(k.shape) for i in (0, 2))
    want = attend(which, q, (k, v, s), lay, qlens, nq, nkv, d, 0.1)
    for kk, vv in ((lower, upper), (upper, lower)):
        kk.view(torch.uint8).copy_(k.view(torch.uint8))
        vv.view(torch.uint8).copy_(v.view(torch.uint8))
        assert torch.equal(attend(which, q, (kk, vv, s), lay, qlens, nq, nkv, d, 0.1), want)
    same = s.view(torch.uint8).clone()
    same[..., 1] = same[..., 0]
    got = attend(which, q, (k, k, same.view(E8M0)), lay, qlens, nq, nkv, d, 0.1)
    check_attention(got, q, keys, keys, befores, qlens, nq, d, 0.1)


def test_pools_beyond_4_gib():
    """Rows whose bytes lie beyond 2^32 of their tensor: written, read by every kernel."""
    nq, nkv, d, P = 4, 2, 128, 16
    pages = (1 << 32) // (nkv * P * d) + 40
    k = torch.empty((pages, nkv, P, d), dtype=torch.uint8, device=DEV).view(E4M3)
    v = torch.empty((pages, nkv, P, d), dtype=torch.uint8, device=DEV).view(E4M3)
    s = torch.empty((pages, nkv, P, 2), dtype=torch.uint8, device=DEV).view(E8M0)
    i32 = dict(dtype=torch.int32, device=DEV)
    T = 200
    table = torch.arange(pages - 1, pages - 15, -1, **i32)[None]
    qkv, w, _, inv = write_inputs(T, nq, nkv, d, d, True, False, 5)
    pos, row, base = torch.arange(T, **i32), torch.zeros(T, **i32), torch.zeros(1, **i32)
    q = ops().qk_rope_kv_f8(qkv, w[0], w[1], inv, pos, row, table, base, k, v, s, nq, nkv, d, d, False, 1e-6)
    small = empty_cache(14, nkv, P, d)
    near = torch.arange(13, -1, -1, **i32)[None]
    q2 = ops().qk_rope_kv_f8(qkv, w[0], w[1], inv, pos, row, near, base, *small, nq, nkv, d, d, False, 1e-6)
    assert torch.equal(q, q2)
    for far, close in zip((k, v, s), small):
        assert torch.equal(far.view(torch.uint8)[pages - 12:, :, :8], close.view(torch.uint8)[2:, :, :8])
    lay = {"page_base": base, "row_start": torch.tensor([0, T], **i32), "row_pos": torch.zeros(1, **i32), "num_tokens": T}
    for which in ("decode", "prefill"):
        far = attend(which, q, (k, v, s), {**lay, "block_table": table}, [T], nq, nkv, d, 0.1)
        assert torch.equal(far, attend(which, q, small, {**lay, "block_table": near}, [T], nq, nkv, d, 0.1))
    narrow = [t.view(torch.uint8).view(pages, nkv, 2 * P, -1) for t in (k, v)]                  # the same bytes as heads of 64 on the way to the
    far32 = ops().attention_decode_f8(q[:, :nq * 64].contiguous(), nq * 64, *(t.view(E4M3) for t in narrow),      # general kernel: pages of 32
                                      torch.full((pages, nkv, 2 * P, 2), 127, dtype=torch.uint8, device=DEV).view(E8M0), table, base,
                                      lay["row_start"], lay["row_pos"], tiles_of([4], 4), T, nq, nkv, 64, 0.1, None)
    assert bool(torch.isfinite(far32[:4]).all())
    del k, v, s, narrow
    torch.cuda.empty_cache()


@pytest.mark.parametrize("which,splits", [("decode", s) for s in (0, 1, 2, 3, 5, 7, 8, 16)] + [("prefill", s) for s in (1, 2, 3, 7, 16)])
@pytest.mark.parametrize("nq,nkv,d,P", [(8, 2, 128, 16), (8, 1, 64, 8), (3, 1, 128, 32)])
def test_attention_in_parts(which, splits, nq, nkv, d, P):
    """Keys cut into more and fewer parts than there are blocks, parts that a mask leaves empty, rows that are no number."""
    spoil = [(0, 70, 0, 0), (1, 3, 0, 1), (5, 1100, 0, 0)]
    lay, cache, keys, values = random_cache(BEFORES, QLENS, nkv, d, P, 31, spoil)
    g = torch.Generator().manual_seed(32)
    q = torch.randn(lay["num_tokens"], nq * d, generator=g).to(torch.bfloat16).to(DEV)
    sink = (3 * torch.randn(nq, generator=g)).to(DEV)
    for mask in (dict(), dict(window=1), dict(window=70, keep_first=5, sink32=sink), dict(chunk=256)):
        got = attend(which, q, cache, lay, QLENS, nq, nkv, d, d ** -0.5, num_splits=splits, **mask)
        check_attention(got, q, keys, values, BEFORES, QLENS, nq, d, d ** -0.5, **mask)


@pytest.mark.parametrize("heads_at_once", [1, 2])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("d", [64, 128])
def test_prompts_whose_keys_are_made_a_few_heads_at_a_time(monkeypatch, heads_at_once, splits, d):
    """Scratch for one kv head, and for two of three: the same bits as from all heads at once."""
    nq, nkv, P = 6, 3, 16
    lay, cache, keys, values = random_cache(BEFORES, QLENS, nkv, d, P, 33)
    g = torch.Generator().manual_seed(34)
    q = torch.randn(lay["num_tokens"], nq * d, generator=g).to(torch.bfloat16).to(DEV)
    mask = dict(window=300, keep_first=4, sink32=torch.randn(nq, generator=g).to(DEV))
    whole = attend("prefill", q, cache, lay, QLENS, nq, nkv, d, d ** -0.5, num_splits=splits, **mask)
    cap = (-(-lay["block_table"].shape[1] * P // 128) + 1) * 128
    monkeypatch.setattr(ops(), "F8_PREFILL_SCRATCH", heads_at_once * min(len(QLENS), len(tiles_of(QLENS, 128))) * cap * d * 4)
    got = attend("prefill", q, cache, lay, QLENS, nq, nkv, d, d ** -0.5, num_splits=splits, **mask)
    assert torch.equal(got, whole)
    check_attention(got, q, keys, values, BEFORES, QLENS, nq, d, d ** -0.5, **mask)


@pytest.mark.parametrize("d", [64, 128])
def test_single_tokens_of_more_rows_than_are_shared_out(d):
    nq, nkv, P, rows = 4, 2, 16, 300
    befores, qlens = [(7 * r) % 150 for r in range(rows)], [1] * rows
    lay, cache, keys, values = random_cache(befores, qlens, nkv, d, P, 35)
    q = torch.randn(rows, nq * d, generator=torch.Generator().manual_seed(36)).to(torch.bfloat16).to(DEV)
    got = attend("decode", q, cache, lay, qlens, nq, nkv, d, d ** -0.5, tiles=tiles_of(qlens, 1))
    check_attention(got, q, keys, values, befores, qlens, nq, d, d ** -0.5)
    with raises("num_splits"):
        attend("decode", q, cache, lay, qlens, nq, nkv, d, d ** -0.5, tiles=tiles_of(qlens, 1), num_splits=0)


@pytest.mark.parametrize("which,splits", [("decode", 0), ("decode", 1), ("decode", 3), ("prefill", 1), ("prefill", 3), ("plain", None)])
def test_sinks_far_above_and_below_the_scores(which, splits):
    """A sink of exp(200) leaves next to nothing of the keys, one of exp(-200) all of it, however the keys are cut.  Sizes below
    2^-126 (float32's smallest normal number) may become zero."""
    nq, nkv, P, d = 6, 2, 16, 128 if which != "plain" else 48
    befores, qlens = [300, 0], [3, 130]
    lay, cache, keys, values = random_cache(befores, qlens, nkv, d, P, 41)
    q = torch.randn(lay["num_tokens"], nq * d, generator=torch.Generator().manual_seed(42)).to(torch.bfloat16).to(DEV)
    sink = torch.tensor([200.0, 60.0, 0.0, -200.0, 100.0, 5.0], device=DEV)
    kw = {} if splits is None else dict(num_splits=splits)
    got = attend("prefill" if which == "plain" else which, q, cache, lay, qlens, nq, nkv, d, d ** -0.5, sink32=sink, **kw).double().cpu()
    at = 0
    for r, (held, n) in enumerate(zip(befores, qlens)):
        want, spread, size = f8.attention(q[at:at + n].double().cpu().view(n, nq, d), keys[r], values[r], d ** -0.5, held, sink=sink.cpu())
        off = (got[at:at + n].view(n, nq, d) - want).abs()
        share = 2.0 ** -8 + 2 * (2.0 ** -18 + d * 2.0 ** -24 * size)[..., None]
        most = torch.tensor([float(values[r].abs().max())]).double()
        assert bool((off <= 2.0 ** -8 * want.abs() + share * spread + 2.0 ** -126 * (1 + most)).all())
        at += n
