"""Attention over an 8-bit cache whose value rows lie at the ends of the format, or are zero: a row of zeros has the smallest
exponent there is, -120, and every weight is held against values of any size.

Tolerances: those of ``test_f8_cache_gpu.py`` (``check_attention``), relative to the result and to the sum of weights times |v|.
What is below 2^-126 in float32, or comes from values that are all zero, is compared as it is: zero."""

import pytest
import torch

from tests.plain import f8_cache as f8
from tests.test_f8_cache_gpu import attend, check_attention, random_cache

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
P = 16
SPLITS = [None, 0, 1, 3, 6, 8, 16]
HEADS = [(8, 2, 128), (8, 1, 128), (8, 2, 64), (8, 1, 64)]          # four and eight query heads to a kv head: one and two times eight rows


def cache_with(values_of, held, qlens, nkv, d, seed):
    """A cache of one row a query length whose value rows are ``values_of(random normal rows [length, nkv, d])``."""
    befores = [held] * len(qlens)
    lay, cache, keys, values = random_cache(befores, qlens, nkv, d, P, seed)
    g = torch.Generator().manual_seed(seed + 1)
    for r, n in enumerate(qlens):
        L = held + n
        codes, byte = f8.to_tensors(*f8.quantise(values_of(torch.randn(L, nkv, d, generator=g, dtype=torch.float64))))
        at = torch.tensor([lay["tables"][r][p // P] for p in range(L)], device=DEV), torch.arange(L, device=DEV) % P
        cache[1].view(torch.uint8)[at[0], :, at[1]] = codes.view(torch.uint8).to(DEV)
        cache[2].view(torch.uint8)[at[0], :, at[1], 1] = byte.to(DEV)
        values[r] = f8.dequantise(codes, byte)
    return lay, cache, keys, values, befores


def queries(T, nq, d, size, seed=3):
    return (size * torch.randn(T, nq * d, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16).to(DEV)


def zeros_in_head_0(v):
    v[:, 0] = 0
    return v


@pytest.mark.parametrize("splits", SPLITS)
@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("size", [0.0, 1.0, 3.0])
def test_a_head_whose_values_are_zero(splits, nq, nkv, d, size):
    """Equal scores and scattered ones over 4,000 keys: zeros, and the other head as ever."""
    qlens = [1, 2]
    lay, cache, keys, values, befores = cache_with(zeros_in_head_0, 4000, qlens, nkv, d, 5)
    q = queries(3, nq, d, size)
    got = attend("decode", q, cache, lay, qlens, nq, nkv, d, d ** -0.5, num_splits=splits)
    assert int(got.view(3, nkv, -1)[:, 0].count_nonzero()) == 0
    check_attention(got, q, keys, values, befores, qlens, nq, d, d ** -0.5)


@pytest.mark.parametrize("splits", SPLITS)
@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("zeros,size", [(64, 1.0), (300, 3.0), (9000, 0.0), (9000, 2.0)])
def test_values_that_begin_with_zeros(splits, nq, nkv, d, zeros, size):
    def values_of(v):
        v[:zeros] = 0
        return v

    qlens = [2]
    lay, cache, keys, values, befores = cache_with(values_of, zeros + 70, qlens, nkv, d, 7)
    q = queries(2, nq, d, size)
    got = attend("decode", q, cache, lay, qlens, nq, nkv, d, d ** -0.5, num_splits=splits)
    check_attention(got, q, keys, values, befores, qlens, nq, d, d ** -0.5)


@pytest.mark.parametrize("splits", SPLITS)
@pytest.mark.parametrize("nq,nkv,d", HEADS)
@pytest.mark.parametrize("power", [-115, -90, 90, 110])
@pytest.mark.parametrize("sink", [False, True])
def test_values_at_the_ends_of_the_format(splits, nq, nkv, d, power, sink):
    qlens = [1, 2]
    lay, cache, keys, values, befores = cache_with(lambda v: v * 2.0 ** power, 2500, qlens, nkv, d, 9)
    q = queries(3, nq, d, 3.0)
    kw = dict(sink32=torch.linspace(-6, 9, nq, device=DEV)) if sink else {}
    got = attend("decode", q, cache, lay, qlens, nq, nkv, d, d ** -0.5, num_splits=splits, **kw)
    check_attention(got, q, keys, values, befores, qlens, nq, d, d ** -0.5, **kw)


@pytest.mark.parametrize("splits", SPLITS)
@pytest.mark.parametrize("nq,nkv,d", HEADS)
def test_values_of_every_size_beside_zeros(splits, nq, nkv, d):
    """Rows from 2^-118 to 2^0 with zeros among them, windows that leave only some, a row that is no number."""
    def values_of(v):
        v *= torch.exp2(torch.linspace(-118, 0, v.shape[0], dtype=torch.float64))[torch.randperm(v.shape[0], generator=torch.Generator().manual_seed(2)), None, None]
        v[::5] = 0
        v[100, 0, 3] = float("nan")
        return v

    qlens = [1, 3]
    lay, cache, keys, values, befores = cache_with(values_of, 1300, qlens, nkv, d, 11)
    q = queries(4, nq, d, 2.0)
    for mask in (dict(), dict(window=700), dict(window=90, keep_first=30)):
        got = attend("decode", q, cache, lay, qlens, nq, nkv, d, d ** -0.5, num_splits=splits, **mask)
        check_attention(got, q, keys, values, befores, qlens, nq, d, d ** -0.5, **mask)


@pytest.mark.parametrize("d,splits", [(128, 1), (128, 3), (64, 1), (64, 3), (48, None)])
@pytest.mark.parametrize("power", [None, -115, 60])
def test_prompts_over_such_values(d, splits, power):
    """The prompt kernel, and at head size 48 the general one: zeros in one head and before the rows, and values far from one."""
    def values_of(v):
        if power is not None:
            return v * 2.0 ** power
        v[:700] = 0
        return zeros_in_head_0(v)

    nq, nkv, qlens = 4, 2, [130]
    lay, cache, keys, values, befores = cache_with(values_of, 900, qlens, nkv, d, 13)
    q = queries(130, nq, d, 2.0)
    got = attend("prefill", q, cache, lay, qlens, nq, nkv, d, d ** -0.5, num_splits=splits)
    check_attention(got, q, keys, values, befores, qlens, nq, d, d ** -0.5)


@pytest.mark.parametrize("nkv,d", [(8, 128), (8, 64)])
def test_a_step_of_rows_with_such_a_head(nkv, d):
    """Eight rows of 4,000 keys under the default rule."""
    nq, qlens = 4 * nkv, [1] * 8
    lay, cache, keys, values, befores = cache_with(zeros_in_head_0, 3999, qlens, nkv, d, 15)
    q = queries(8, nq, d, 1.0)
    got = attend("decode", q, cache, lay, qlens, nq, nkv, d, d ** -0.5)
    check_attention(got, q, keys, values, befores, qlens, nq, d, d ** -0.5)
