"""The operators of the 8-bit key/value cache: what is measured of them, in plain torch and through the kernels.

The cache holds every key row and value row (one token, one kv head, ``d`` entries) as e4m3 numbers and one power of two:
``row = code * 2^e`` with ``e`` the smallest integer in -120..120 for which ``448 * 2^e`` is not below the row's largest
magnitude, and every code the nearest e4m3 number (ties to even).  Codes lie in pages ``[pages, kv heads, page, d]``, the
exponents of a token's key and value side by side in ``[pages, kv heads, page, 2]``, one byte each (2^(byte - 127)).

Three operators:

``write``    norm and rotation of the query and key heads of projected rows ``[q | k | v]``, the keys and values
             quantised and written into their pages: what a layer does before its attention;
``decode``   attention of one new token a request (or of a few) over its pages;
``prefill``  causal attention of prompts, or portions of them, packed one behind the other, over their pages, which
             already hold their keys and values.

Keys of a case: ``rows`` requests that hold ``context`` tokens and bring ``new`` ones (``ragged``: 35 to 100 % of each),
``nq`` query heads over ``nkv`` kv heads of ``d`` entries, ``page`` tokens a page, ``window`` (0: none).  Of a write:
``rot`` rotated entries a head, ``interleaved`` pairs, ``norm`` or not.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False
DEVICE = "cuda:0"
E4M3, E8M0, BF16 = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.bfloat16
EPS = 1e-6


# ------------------------------------------------------------------ the cases


def _case(name, op, *, rows=1, context=0, new=1, ragged=False, nq=32, nkv=8, d=128, page=16, window=0, rot=None,
          interleaved=False, norm=True):
    c = {"name": name, "op": op, "rows": rows, "context": context, "new": new, "ragged": ragged, "nq": nq, "nkv": nkv, "d": d,
         "page": page}
    if op == "write":
        c.update(rot=d if rot is None else rot, interleaved=interleaved, norm=norm)
    else:
        c.update(window=window)
    return c


def listed():
    return [
        # the decode step of eight users (32 query heads over 8): hardly any bytes, a launch
        _case("write-decode-8", "write", rows=8, context=4000),
        # a prompt's rows on their way into the cache
        _case("write-prompt-2048", "write", new=2048),
        # packed prompts of different odd lengths, small heads, half of a head rotated in neighbouring pairs, no norm
        _case("write-packed-d64", "write", rows=5, context=77, new=1723, ragged=True, nq=32, nkv=4, d=64, page=32, rot=32,
              interleaved=True, norm=False),
        # one user of a small model early in an answer
        _case("decode-1-ctx300", "decode", context=300, nq=16),
        # the benchmark's headline: eight users late in their answers
        _case("decode-8-ctx4000", "decode", rows=8, context=4000),
        # a server's steady state: answers of many lengths
        _case("decode-41-ragged", "decode", rows=41, context=1700, ragged=True),
        # one long document: a row's keys split over the whole device (64 query heads over 8)
        _case("decode-1-ctx131071", "decode", context=131071, nq=64),
        # drafted tokens, three a request, checked at once over a window; small heads, eight to a kv head
        _case("decode-24-new3-window-d64", "decode", rows=24, context=2501, new=3, ragged=True, nq=32, nkv=4, d=64, page=32,
              window=1024),
        # three short prompts at once, small heads
        _case("prefill-3x601-d64", "prefill", rows=3, new=601, ragged=True, nq=16, nkv=8, d=64),
        # a prompt to its first token
        _case("prefill-2048", "prefill", new=2048),
        # the next portion of a long prompt that is fed in pieces
        _case("prefill-512-after-16001", "prefill", context=16001, new=512),
        # a long prompt whole
        _case("prefill-8192", "prefill", new=8192),
    ]


HEADS = [(16, 8, 128), (32, 8, 128), (64, 8, 128), (8, 8, 128), (40, 8, 128), (24, 8, 64), (32, 4, 64), (16, 16, 64), (12, 2, 64)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["write", "decode", "decode", "prefill", "prefill"])
    nq, nkv, d = rng.choice(HEADS)
    c = dict(nq=nq, nkv=nkv, d=d, page=rng.choice([8, 16, 16, 32, 64]), ragged=rng.random() < 0.6)
    if op == "write":
        new = _log(rng, 1, 2048)
        rot = rng.choice([d, d, d // 2])
        c.update(rows=_log(rng, 1, max(1, min(64, 8192 // new))), context=_log(rng, 1, 30000) - 1, new=new, rot=rot,
                 interleaved=rng.random() < 0.3, norm=rng.random() < 0.7)
    elif op == "decode":
        rows = _log(rng, 1, 64)
        c.update(rows=rows, context=_log(rng, 1, min(32768, 131072 // rows)) - 1, new=rng.choice([1, 1, 1, 1, 2, 4, 7]),
                 window=rng.choice([0, 0, 0, 512, 1000]))
    else:
        new = _log(rng, 2, 4096)
        # the queries of all rows times their keys stay below those of the largest listed case
        pairs = 8192 * 8192 // 2 * 32 * 128 // (nq * d)
        context = max(0, min(rng.choice([0, 0, _log(rng, 1, 16384)]), pairs // new - new // 2 - 1))
        most = pairs // (new * (context + new // 2 + 1))
        c.update(rows=_log(rng, 1, max(1, min(6, most, 8192 // new))), context=context, new=new,
                 window=rng.choice([0, 0, 0, 512, 1000]))
    c = _case("", op, **c)
    c.pop("name")
    return c


def _lens(case):
    """(tokens held, tokens brought) of every row; the first row has them whole."""
    part = [1.0] + [0.35 + 0.65 * (i * 0.6180339887 % 1.0) for i in range(1, case["rows"])]
    if not case["ragged"]:
        part = [1.0] * case["rows"]
    return [(int(case["context"] * f), max(1, int(case["new"] * (f if case["op"] != "decode" else 1.0)))) for f in part]


def _pairs(case):
    """Query-key pairs that the masks leave, and keys that are read at all, summed over the rows."""
    w, pairs, keys = case["window"], 0, 0
    for held, new in _lens(case):
        if not w or held + new <= w:
            pairs += new * held + new * (new + 1) // 2
            keys += held + new
        else:
            pairs += sum(min(w, p + 1) for p in range(held, held + new))
            keys += held + new - max(0, held - w + 1)
    return pairs, keys


def work(case):
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    tokens = sum(n for _, n in _lens(case))
    if case["op"] == "write":
        return {"bytes": tokens * ((2 * nq + 2 * nkv) * d * 2 + nkv * (2 * d + 2)), "flops": tokens * (nq + nkv) * d * 8}
    pairs, keys = _pairs(case)
    return {"bytes": tokens * nq * d * 4 + keys * nkv * (2 * d + 2), "flops": 4 * nq * d * pairs}


# ------------------------------------------------------------------ inputs


def _quantise(x):
    """(codes in e4m3, exponents as bytes) of rows of 32-bit numbers."""
    mantissa, exponent = torch.frexp(x.abs().amax(dim=-1))
    e = torch.where(mantissa == 0, -120, exponent - 9 + (mantissa > 0.875).to(exponent.dtype)).clamp(-120, 120)
    codes = torch.ldexp(x, -e[..., None]).clamp(-448, 448).to(E4M3)
    return codes, (e + 127).to(torch.uint8)


def _power(byte):
    return torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte.to(torch.int32) - 127)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    nq, nkv, d, P = case["nq"], case["nkv"], case["d"], case["page"]
    lens = _lens(case)
    R = len(lens)
    s = SimpleNamespace(case=case, nq=nq, nkv=nkv, d=d, P=P, scale=d ** -0.5)
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEVICE)                              # noqa: E731
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEVICE)                                 # noqa: E731
    # pages in no order; a write holds the pages that it touches, a windowed row has given the pages before its window back
    first = []
    for held, _ in lens:
        if case["op"] == "write":
            first.append(held // P)
        else:
            first.append(max(0, held - case["window"] + 1) // P if case["window"] else 0)
    counts = [-(-(held + new) // P) - b for (held, new), b in zip(lens, first)]
    total = sum(counts)
    pages = torch.randperm(total, generator=g, device=DEVICE).to(torch.int32)
    s.block_table = torch.zeros((R, max(counts)), dtype=torch.int32, device=DEVICE)
    at = torch.arange(max(counts), device=DEVICE)[None, :] < ints(counts)[:, None]
    s.block_table[at] = pages
    s.page_base, s.row_pos = ints(first), ints([held for held, _ in lens])
    s.row_start = ints([sum(n for _, n in lens[:i]) for i in range(R + 1)])
    s.token_row = torch.repeat_interleave(torch.arange(R, device=DEVICE), ints([n for _, n in lens])).to(torch.int32)
    T = s.token_row.numel()
    s.positions = (torch.arange(T, device=DEVICE) - s.row_start[s.token_row.long()] + s.row_pos[s.token_row.long()]).to(torch.int32)
    s.T, s.R, s.newest, s.keys = T, R, max(n for _, n in lens), max(a + n for a, n in lens)
    # channels of keys differ, a few stand out; tokens differ in size, values more than keys
    channel = 0.5 + torch.rand((nkv, 1, d), generator=g, device=DEVICE)
    channel[:, :, :: max(1, d // 3)] *= 5
    if case["op"] == "write":
        s.k_pages = torch.zeros((total, nkv, P, d), dtype=E4M3, device=DEVICE)
        s.v_pages = torch.zeros_like(s.k_pages)
        s.scales = torch.full((total, nkv, P, 2), 127, dtype=torch.uint8, device=DEVICE).view(E8M0)
        rows = randn(T, nq + 2 * nkv, d)
        rows[:, nq:nq + nkv] *= channel[:, 0]
        rows[:, nq + nkv:] *= torch.exp(0.5 * randn(T, nkv, 1))
        s.qkv = rows.view(T, -1).to(BF16)
        s.q_norm = 1 + 0.2 * randn(d) if case["norm"] else None
        s.k_norm = 1 + 0.2 * randn(d) if case["norm"] else None
        half = case["rot"] // 2
        s.inv_freq = (1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)).to(torch.float32)
        return s
    s.k_pages, kb = _quantise(randn(total, nkv, P, d) * channel * torch.exp(0.2 * randn(total, nkv, P, 1)))
    s.v_pages, vb = _quantise(randn(total, nkv, P, d) * torch.exp(0.5 * randn(total, nkv, P, 1)))
    s.scales = torch.stack([kb, vb], dim=-1).view(E8M0)
    s.q = (1.2 * randn(T, nq * d)).to(BF16)
    # query tiles (row, first token within the row): 128 queries, the ones with the most keys first, for prompts; for few
    # tokens as many as 16 rows of (token, head of a group) hold
    step = 128 if case["op"] == "prefill" else 16 // (nq // nkv)
    tiles = [(r, q0) for r, (_, n) in enumerate(lens) for q0 in range(0, n, step)]
    if case["op"] == "prefill":
        tiles.sort(key=lambda t: -(lens[t[0]][0] + min(t[1] + 128, lens[t[0]][1])))
    s.tiles = ints(tiles).view(-1, 2)
    return s


# ------------------------------------------------------------------ one pass


def run(s):
    op = s.case["op"]
    if own:
        from acorninfer_b200.kernels import ops
        if op == "write":
            q = ops.qk_rope_kv_f8(s.qkv, s.q_norm, s.k_norm, s.inv_freq, s.positions, s.token_row, s.block_table, s.page_base,
                                  s.k_pages, s.v_pages, s.scales, s.nq, s.nkv, s.d, s.case["rot"], s.case["interleaved"], EPS)
            return {"q": q, "k": s.k_pages, "v": s.v_pages, "scales": s.scales}
        attention = ops.attention_decode_f8 if op == "decode" else ops.attention_prefill_f8
        return attention(s.q, s.q.stride(0), s.k_pages, s.v_pages, s.scales, s.block_table, s.page_base, s.row_start, s.row_pos,
                         s.tiles, s.T, s.nq, s.nkv, s.d, s.scale, s.case["window"] or None)
    return _plain_write(s) if op == "write" else _plain_attention(s)


def _plain_write(s):
    nq, nkv, d, rot = s.nq, s.nkv, s.d, s.case["rot"]
    x = s.qkv.view(s.T, nq + 2 * nkv, d).float()
    heads, v = x[:, :nq + nkv], x[:, nq + nkv:]
    if s.q_norm is not None:
        w = torch.cat([s.q_norm.expand(nq, d), s.k_norm.expand(nkv, d)])
        heads = heads * torch.rsqrt(heads.square().mean(dim=-1, keepdim=True) + EPS) * w
    angle = s.positions.double()[:, None] * s.inv_freq.double()           # far positions need more than 24 bits
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    turned = heads.clone()
    if s.case["interleaved"]:
        a, b = heads[..., 0:rot:2], heads[..., 1:rot:2]
        turned[..., 0:rot:2], turned[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = heads[..., :rot // 2], heads[..., rot // 2:rot]
        turned[..., :rot // 2], turned[..., rot // 2:rot] = a * cos - b * sin, b * cos + a * sin
    r = s.token_row.long()
    page = s.block_table[r, s.positions.long() // s.P - s.page_base[r].long()].long()
    slot = s.positions.long() % s.P
    k_codes, kb = _quantise(turned[:, nq:])
    v_codes, vb = _quantise(v)
    s.k_pages.view(torch.uint8)[page, :, slot] = k_codes.view(torch.uint8)
    s.v_pages.view(torch.uint8)[page, :, slot] = v_codes.view(torch.uint8)
    s.scales.view(torch.uint8)[page, :, slot] = torch.stack([kb, vb], dim=-1)
    return {"q": turned[:, :nq].reshape(s.T, nq * d).to(BF16), "k": s.k_pages, "v": s.v_pages, "scales": s.scales}


def _plain_attention(s):
    nq, nkv, d, P, R, L, N = s.nq, s.nkv, s.d, s.P, s.R, s.keys, s.newest
    # every row's keys and values side by side, padded to the longest row
    key = torch.arange(L, device=DEVICE)[None, :]
    col = (key // P - s.page_base[:, None]).clamp(0, s.block_table.shape[1] - 1)
    page = s.block_table.gather(1, col).long()
    slot = (key % P).expand(R, L)
    power = _power(s.scales.view(torch.uint8)[page, :, slot])                              # [R, L, nkv, 2]
    k = s.k_pages.view(torch.uint8)[page, :, slot].view(E4M3).float() * power[..., :1]
    v = s.v_pages.view(torch.uint8)[page, :, slot].view(E4M3).float() * power[..., 1:]
    # queries likewise
    n = s.row_start[1:] - s.row_start[:-1]
    j = torch.arange(N, device=DEVICE)[None, :]
    token = (s.row_start[:-1, None] + torch.minimum(j, n[:, None] - 1)).long()
    q = s.q.view(s.T, nkv, nq // nkv, d)[token].float() * s.scale                           # [R, N, nkv, rep, d]
    position = s.row_pos[:, None] + j
    sees = key[:, None, :] <= position[:, :, None]                                          # [R, N, L]
    if s.case["window"]:
        sees &= key[:, None, :] > position[:, :, None] - s.case["window"]
    score = q.permute(0, 2, 3, 1, 4).reshape(R, nkv, -1, d) @ k.permute(0, 2, 3, 1)         # [R, nkv, rep N, L]
    del q, k
    score = score.view(R, nkv, nq // nkv, N, L).masked_fill_(~sees[:, None, None], -math.inf)
    score -= score.amax(dim=-1, keepdim=True)
    score.exp_()
    total = score.sum(dim=-1, keepdim=True)
    out = (score.view(R, nkv, -1, L) @ v.permute(0, 2, 1, 3)).view(R, nkv, nq // nkv, N, d) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(R, N, nq * d)
    return out[j < n[:, None]].to(BF16)


# ------------------------------------------------------------------ the definition, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_write(s) if case["op"] == "write" else _exact_attention(s)


def _e4m3(x):
    """The nearest e4m3 number of every entry (|x| <= 448), ties to even, by the spacing of its binade."""
    spacing = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / spacing) * spacing


def _exact_rows(x):
    """(codes, powers of two) of rows of 64-bit numbers: the exponent by search over its range."""
    most = x.abs().amax(dim=-1, keepdim=True)
    power = torch.exp2(torch.arange(-120, 121, dtype=torch.float64, device=x.device))
    e = torch.searchsorted(448 * power, most.contiguous()).clamp(max=240)
    return _e4m3(x / power[e]), power[e][..., 0]


def _exact_write(s):
    nq, nkv, d, rot, P = s.nq, s.nkv, s.d, s.case["rot"], s.P
    x = s.qkv.double().view(s.T, -1, d)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]

    def turn(h, w):
        if w is not None:
            h = h / torch.sqrt((h * h).sum(-1, keepdim=True) / d + EPS) * w.double()
        pairs = h[..., :rot].unflatten(-1, (rot // 2, 2) if s.case["interleaved"] else (2, rot // 2))
        pairs = pairs if s.case["interleaved"] else pairs.transpose(-1, -2)
        z = torch.view_as_complex(pairs.contiguous())
        angle = s.positions.double()[:, None, None] * s.inv_freq.double()
        z = torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle))
        z = z if s.case["interleaved"] else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), h[..., rot:]], dim=-1)

    kc, kp = _exact_rows(turn(k, s.k_norm))
    vc, vp = _exact_rows(v)
    pages = s.k_pages.shape[0]
    row = s.token_row.long()
    where = s.block_table[row, (s.positions // P).long() - s.page_base[row].long()].long() * P + (s.positions % P).long()
    flat = lambda *tail: torch.zeros((pages * P, nkv, *tail), dtype=torch.float64, device=x.device)    # noqa: E731
    back = lambda t: t.view(pages, P, *t.shape[1:]).transpose(1, 2).contiguous()                       # noqa: E731
    kf, vf, sf = flat(d), flat(d), flat(2) + 1
    kf[where], vf[where], sf[where] = kc, vc, torch.stack([kp, vp], dim=-1)
    return {"q": turn(q, s.q_norm).reshape(s.T, nq * d), "k": back(kf), "v": back(vf), "scales": back(sf)}


def _exact_attention(s):
    nq, nkv, d, P, window = s.nq, s.nkv, s.d, s.P, s.case["window"]
    rep = nq // nkv
    out = torch.empty((s.T, nq, d), dtype=torch.float64, device=DEVICE)
    start, held, base = s.row_start.tolist(), s.row_pos.tolist(), s.page_base.tolist()
    for r in range(s.R):
        a, b = start[r], start[r + 1]
        end = held[r] + b - a
        pages = s.block_table[r, :-(-end // P) - base[r]].long()
        low = base[r] * P
        for h in range(nkv):
            power = torch.exp2(s.scales.view(torch.uint8)[pages, h].double().reshape(-1, 2)[:end - low] - 127)
            k, v = (t.view(torch.uint8)[pages, h].view(E4M3).double().reshape(-1, d)[:end - low] for t in (s.k_pages, s.v_pages))
            k, v = k * power[:, :1], v * power[:, 1:]
            at = torch.arange(low, end, device=DEVICE)
            for a0 in range(a, b, 1024):
                b0 = min(b, a0 + 1024)
                pos = torch.arange(held[r] + a0 - a, held[r] + b0 - a, device=DEVICE)[:, None, None]
                hidden = at > pos
                if window:
                    hidden = hidden | (at <= pos - window)
                q = s.q[a0:b0].double().view(-1, nq, d)[:, h * rep:(h + 1) * rep]
                score = torch.where(hidden, -math.inf, q @ k.T * s.scale)
                out[a0:b0, h * rep:(h + 1) * rep] = torch.softmax(score, dim=-1) @ v
    return out.view(s.T, nq * d)
