"""Prompt attention over a cache of 4 bits where keys or values of very different sizes lie side by side: a result is as exact as what its query
attends makes it, whatever else the tile's other queries, or keys of no weight, bring.

The bound.  With h = 2^-11, a number of a key or a value is off by 2 h of its row's largest (of float16 operands under a power of two that leaves them 11 bits:
zeros and steps have eight, so they are exact but below 2^-17, where 15 steps are off by 2^-21, h of a largest of 2^-10 or more; the number is rounded once).
That moves the score of key j by e_j = 2 h · scale · Σ|q| · |k_j|max, its weight by a factor within exp(±(e_j + e)), e the mean of the e_j under the weights,
and a result by Σ_j p_j |v_j|max (expm1(e_j + e) + 3 h) with the rounding of the weight itself.

A weight times the power w_j that its value lies divided by is held to 2^-25 where the largest such product has 2^4 or more; so the part of key k is off by
2^-29 (|v_k|max / w_k) max_j p_j w_j, and never by more than itself.  w_j is between |v_j|max / 2^15 and 2^10 |v_j|max, and the same for tokens of like size.
`least` is 2^-29 times the most that (w_j / |v_j|max) (|v_k|max / w_k) is among the tokens that a query sees; tokens that were not resized differ by less than 2^5.

Sums in float32 add (n + 32) units of 2^-24, and the result is rounded once to bfloat16."""
import math

import pytest
import torch

import plain_packed as plain

pytestmark = pytest.mark.gpu
U, HALF_STEP, H = 2.0 ** -24, 2.0 ** -8, 2.0 ** -11


def resized(pages, name, tokens, size):
    for t in tokens:
        block = int(pages.table[0, t // 64])
        pages.host[name][block, :, t % 64] = (pages.host[name][block, :, t % 64].float() * size).bfloat16()


def check(pages, qkv, out, heads, dim, scale, window, past, rows, least):
    k, v = pages.context(0)
    for t in rows:
        q = qkv[t, :heads * dim].double().view(heads, dim)
        pos = past + t
        first = max(0, pos - window + 1) if window else 0
        want = plain.attend(q, k, v, scale, window, pos)
        for h in range(heads):
            kk, vv = k[first:pos + 1, h], v[first:pos + 1, h]
            p = torch.softmax(scale * (kk @ q[h]), 0)
            e = (2 * H + (dim + 16) * U) * scale * kk.abs().amax(1) * float(q[h].abs().sum())
            e = (e + float((p * e).sum())).clamp(max=50.0)
            at_most = p * vv.abs().amax(1)
            n = pos + 1 - first
            tol = float((at_most * (torch.expm1(e) * (1 + 3 * H) + 3 * H + (n + 32) * U)).sum() + at_most.clamp(max=least(first) * float(at_most.max())).sum())
            tol = tol + HALF_STEP * (want[h].abs() + tol)
            off = (out[t].double().cpu().view(heads, dim)[h] - want[h]).abs()
            assert bool((off <= tol).all()), (t, h, float((off / tol).max()))


def attend(pages, new, heads, dim, window, groups, n_parts, qkv, scale):
    from test_packed_kv_kernels import DEV, err_word, prefill
    out = torch.zeros((new, heads * dim), dtype=torch.bfloat16, device=DEV)
    e = err_word()
    for name in ("k", "k_pairs", "v", "v_pairs"):
        getattr(pages.cache, name).copy_(pages.host[name])
    prefill(pages, [new], heads, heads, dim, window, groups, n_parts)(qkv.to(DEV), 0, pages.table.to(DEV), None, None, out, scale, e)
    assert int(e.item()) == 0
    return out


ROWS = (0, 3, 9, 63, 64, 65, 100, 127, 128, 129, 190, 191, 192, 255, 256, 257, 299)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("groups,n_parts", [(1, 1), (2, 1), (2, 3)])
@pytest.mark.parametrize("which", ["k_pairs", "v_pairs", "both"])
@pytest.mark.parametrize("size", [2.0 ** -18, 2.0 ** -9, 2.0 ** 12, 2.0 ** 18, 2.0 ** 30, 2.0 ** 60])
@pytest.mark.parametrize("past", [0, 30])
def test_a_block_that_later_queries_do_not_see_takes_nothing_from_them(dim, groups, n_parts, which, size, past):
    """A window of 64, and the first 64 tokens' keys or values `size` times the others'."""
    from test_packed_kv_kernels import Pages
    heads, new = 2, 300
    pages = Pages([past + new], heads, dim, seed=6)
    for name in ["k_pairs", "v_pairs"] if which == "both" else [which]:
        resized(pages, name, range(64), size)
    qkv = (torch.randn((new, 3 * heads * dim), generator=torch.Generator().manual_seed(9)) * 1.2).bfloat16()
    scale = 1.0 / math.sqrt(dim)
    out = attend(pages, new, heads, dim, 64, groups, n_parts, qkv, scale)
    # (of keys that large the bound says nothing.)  Rows that see tokens of both sizes: large ones divided by the small ones' power, up to 2^15; else those that
    # just keep their block's power, 2^-10 of it, beside those that have their own
    rows = [t for t in ROWS if which == "v_pairs" or past + t >= 128 or size <= 1]
    check(pages, qkv, out, heads, dim, scale, 64, past, rows, lambda first: 2.0 ** -14 if size < 1 and first < 64 else 2.0 ** -18)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("groups,n_parts", [(1, 1), (2, 1), (1, 4)])
@pytest.mark.parametrize("size", [2.0 ** 18, 2.0 ** 30, 2.0 ** 60])
def test_large_values_of_no_weight(dim, groups, n_parts, size):
    """The first block's values are large, and its keys' scores so low that the values others have are the result."""
    from test_packed_kv_kernels import Pages
    heads, new = 2, 300
    pages = Pages([new], heads, dim, seed=7)
    resized(pages, "v_pairs", range(64), size)
    block = int(pages.table[0, 0])
    pages.host["k_pairs"][block, :, :, :, 1] -= 16.0
    qkv = (torch.randn((new, 3 * heads * dim), generator=torch.Generator().manual_seed(9)) * 0.5 + 1.0).bfloat16()
    scale = 1.0 / math.sqrt(dim)
    out = attend(pages, new, heads, dim, 0, groups, n_parts, qkv, scale)
    check(pages, qkv, out, heads, dim, scale, 0, 0, ROWS, lambda first: 2.0 ** -24)           # (every token a power of its own, or the first block's its own)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("groups,n_parts", [(1, 1), (2, 1), (2, 3)])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("size", [2.0 ** -9, 2.0 ** -12, 2.0 ** -20, 2.0 ** -40, 0.0])
def test_small_tokens_among_others(dim, groups, n_parts, window, size):
    """Single tokens, half a block and whole blocks whose values are small, or zeros, behind a block of ordinary ones; keys too."""
    from test_packed_kv_kernels import Pages
    heads, new = 2, 300
    pages = Pages([new], heads, dim, seed=8)
    resized(pages, "v_pairs", [70, 100, 101] + list(range(140, 172)) + list(range(192, 299)), size)
    resized(pages, "k_pairs", [71, 100] + list(range(150, 180)), size)
    qkv = (torch.randn((new, 3 * heads * dim), generator=torch.Generator().manual_seed(9)) * 1.2).bfloat16()
    scale = 1.0 / math.sqrt(dim)
    out = attend(pages, new, heads, dim, window, groups, n_parts, qkv, scale)
    check(pages, qkv, out, heads, dim, scale, window, 0, ROWS + (200, 235, 250, 290, 298), lambda first: 2.0 ** (-14 if size > 2.0 ** -18 else -22))
