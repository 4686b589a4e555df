"""The kernels over a paged cache of keys and values in 4 bits against exact rational arithmetic and float64.

Tolerances, from the arithmetic.  Codes, steps and zeros: none, every rounding is that of an exact quotient.  Numbers read back: none, zero +
step · code is one rounding.  Attention: a result is a mean of values with weights softmax(s).  With u = 2^-24, a score is a sum of
dim products in float32, off by at most e_s = (dim + 16) u · scale · Σ |q| (|zero| + 15 step); weights are then off by a factor of at most
exp(2 e_s), their exponentials and sums by (keys + 32) u.  bfloat16 has eight significant bits: numbers of the binade from 1 on are 2^-7 apart, so
a rounding to it is off by at most 2^-8 of the number.  On the tensor cores a weight times a step is rounded to it, which moves a result by
at most 2^-8 · 15 step of the values' groups; and a bfloat16 result is rounded once."""
import math

import pytest
import torch

import plain_packed as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U, HALF_STEP = 2.0 ** -24, 2.0 ** -8


def err_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


class Pages:
    """Sequences of given lengths in shuffled blocks of a cache full of another owner's leftovers (NaN among them)."""

    def __init__(self, lengths, kv_heads, dim, seed=0, spare=3):
        from vlrf_b200.csrc import ops
        gen = torch.Generator().manual_seed(seed)
        need = [-(-n // 64) for n in lengths]
        self.n_blocks = sum(need) + spare
        order = torch.randperm(self.n_blocks, generator=gen)
        self.table = torch.full((len(lengths), max(need + [1]) + 1), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n].int()
            at += n
        groups = dim // plain.group_of(dim)
        shape = (self.n_blocks, kv_heads, 64)
        self.host = {}
        for name, size in (("k", 1.3), ("v", 0.7)):
            self.host[name] = torch.randint(0, 256, shape + (dim // 2,), generator=gen, dtype=torch.uint8)
            step = torch.rand(shape + (groups,), generator=gen) * 0.3 * size + 0.01
            zero = -7.5 * step + torch.randn(shape + (groups,), generator=gen) * 0.4
            self.host[name + "_pairs"] = torch.stack([step, zero], -1).bfloat16()
        # what lies behind a sequence's last token, and in blocks of nobody: not a number
        owned = torch.zeros(shape[:1] + (64,), dtype=torch.bool)
        for i, n in enumerate(lengths):
            for p in range(n):
                owned[self.table[i, p // 64], p % 64] = True
        for name in ("k_pairs", "v_pairs"):
            self.host[name][~owned[:, None, :].expand(shape)] = float("nan")
        self.cache = ops.PackedKV(*[self.host[n].to(DEV) for n in ("k", "k_pairs", "v", "v_pairs")])
        self.lengths = lengths

    def context(self, i):
        n = self.lengths[i]
        place = torch.arange(n)
        blocks = self.table[i].long()[place // 64]
        return [plain.unpacked(self.host[name], self.host[name + "_pairs"])[blocks, :, place % 64] for name in ("k", "v")]

    def reach(self, i, name):
        """|zero| + 15 step of sequence i's tokens, per entry, and 15 step alone."""
        n = self.lengths[i]
        place = torch.arange(n)
        blocks = self.table[i].long()[place // 64]
        pairs = self.host[name + "_pairs"][blocks, :, place % 64].double()
        return (pairs[..., 1].abs() + 15 * pairs[..., 0]), 15 * pairs[..., 0]


def bound(pages, i, pos, first, q, scale, want, dtype, tensor_cores):
    """The derivation above, for one token: [heads, 1]."""
    share = q.shape[0] // pages.context(i)[0].shape[1]
    rk, _ = pages.reach(i, "k")
    rv, sv = pages.reach(i, "v")
    dim = q.shape[1]
    group = dim // rk.shape[-1]
    out = []
    for h in range(q.shape[0]):
        k_reach = rk[first:pos + 1, h // share].repeat_interleave(group, -1)
        e_s = (dim + 16) * U * scale * float((k_reach * q[h].abs()).sum(-1).max())
        v_max, s_max = float(rv[first:pos + 1, h // share].max()), float(sv[first:pos + 1, h // share].max())
        rel = math.expm1(2 * e_s) + (pos + 1 - first + 32) * U
        out.append(2 * rel * v_max + (HALF_STEP * s_max if tensor_cores else 0.0))
    tol = torch.tensor(out, dtype=torch.float64)[:, None].expand_as(want)
    if dtype == torch.bfloat16:
        tol = tol + HALF_STEP * (want.abs() + tol)
    return tol


# ---- append and read ---------------------------------------------------------------------------------------------------

def rows_of(T, width, dtype, seed, kind="plain"):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((T, width), generator=gen) * 1.5 + torch.randn((1, width), generator=gen)
    if kind == "grid":                         # quotients on the borders: ties
        x = torch.randint(-31, 32, (T, width), generator=gen).float() * 0.25
    if kind == "wild":                         # many sizes in one row, down to subnormal
        x = x * torch.exp2(torch.randint(-130, 60, (T, 1), generator=gen).float())
    if kind == "flat":
        x = torch.full((T, width), 1.0) * torch.randn((T, 1), generator=gen)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["plain", "grid", "wild", "flat"])
@pytest.mark.parametrize("heads,kv_heads,dim,new,past", [
    (12, 12, 64, [1], [515]), (4, 2, 128, [3, 1, 70], [0, 63, 60]), (3, 3, 32, [5, 66], [62, 0]), (5, 5, 16, [9], [0]), (2, 1, 80, [65], [1]),
    (3, 1, 256, [2], [64]), (2, 2, 192, [4], [0]), (6, 3, 96, [7, 1], [128, 0])])
def test_append_holds_the_exact_codes_and_reads_back(dtype, kind, heads, kv_heads, dim, new, past):
    from vlrf_b200.csrc import ops
    T, width = sum(new), (heads + 2 * kv_heads) * dim
    pages = Pages([a + b for a, b in zip(new, past)], kv_heads, dim, seed=dim)
    rows = rows_of(T, width, dtype, seed=T + dim, kind=kind)
    slot = torch.tensor([i for i, a in enumerate(new) for _ in range(a)], dtype=torch.int32)
    pos = torch.tensor([b + j for a, b in zip(new, past) for j in range(a)], dtype=torch.int32)
    k_off, v_off = heads * dim, (heads + kv_heads) * dim
    e = err_word()
    ops.kv_append_packed(rows.to(DEV), k_off, v_off, pages.cache, pages.table.to(DEV), slot.to(DEV), pos.to(DEV), T, kv_heads, dim, e)
    assert int(e.item()) == 0
    want = {name: plain.quantise(rows[:, at:at + kv_heads * dim], dim) for name, at in (("k", k_off), ("v", v_off))}
    got = {n: getattr(pages.cache, n).cpu() for n in ("k", "k_pairs", "v", "v_pairs")}
    touched = torch.zeros((pages.n_blocks, 64), dtype=torch.bool)
    for t in range(T):
        blk, at = int(pages.table[slot[t], pos[t] // 64]), int(pos[t] % 64)
        touched[blk, at] = True
        for name in ("k", "v"):
            codes = torch.stack([got[name][blk, :, at] & 15, got[name][blk, :, at] >> 4], -1).flatten(-2)
            pairs = got[name + "_pairs"][blk, :, at]
            assert torch.equal(pairs.double(), want[name][1][t]), (name, t)
            assert torch.equal(codes.long(), want[name][0][t]), (name, t)
    for name in got:                           # everything else is as it was
        same = ~touched[:, None, :].expand(got[name].shape[:3])
        assert torch.equal(got[name][same].view(torch.uint8), pages.host[name][same].view(torch.uint8))
    for out_dtype in (torch.float32, torch.bfloat16):
        out = [torch.full((T, kv_heads * dim), 7.0, dtype=out_dtype, device=DEV) for _ in range(2)]
        ops.kv_read_packed(pages.cache, pages.table.to(DEV), slot.to(DEV), pos.to(DEV), out[0], out[1], T, e)
        for o, name in zip(out, ("k", "v")):
            assert torch.equal(o.cpu(), plain.values(*want[name]).reshape(T, -1).float().to(out_dtype))
    assert int(e.item()) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_group_that_is_not_finite_reads_back_as_nan_and_no_other(dtype):
    from vlrf_b200.csrc import ops
    pages = Pages([8], 2, 128)
    rows = rows_of(8, 3 * 256, dtype, seed=1)
    rows[2, 256 + 70] = float("nan")           # keys, head 0, second group
    rows[3, 512 + 128] = float("inf")          # values, head 1, first group
    rows[4, 256] = -float("inf")
    rows[5, 256:320] = torch.tensor([-3.0e38, 3.0e38] * 32).to(dtype)      # finite numbers, a range that is not
    slot, pos = torch.zeros(8, dtype=torch.int32, device=DEV), torch.arange(8, dtype=torch.int32, device=DEV)
    e = err_word()
    ops.kv_append_packed(rows.to(DEV), 256, 512, pages.cache, pages.table.to(DEV), slot, pos, 8, 2, 128, e)
    out = [torch.empty(8, 256, device=DEV) for _ in range(2)]
    ops.kv_read_packed(pages.cache, pages.table.to(DEV), slot, pos, out[0], out[1], 8, e)
    nan = [torch.zeros(8, 256, dtype=torch.bool) for _ in range(2)]
    nan[0][2, 64:128] = nan[0][4, :64] = nan[0][5, :64] = nan[1][3, 128:192] = True
    for o, n in zip(out, nan):
        assert torch.equal(torch.isnan(o.cpu()), n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_append_and_read_with_strides_and_odd_alignment(dtype, shift):
    """Columns that begin anywhere in wider rows, in and out."""
    from vlrf_b200.csrc import ops
    T, kv_heads, dim = 37, 3, 64
    pages = Pages([T], kv_heads, dim)
    wide = torch.full((T, 700), float("nan"), dtype=dtype)
    rows = rows_of(T, 2 * 192, dtype, seed=5)
    wide[:, shift:shift + 384] = rows
    dev = wide.to(DEV)
    slot, pos = torch.zeros(T, dtype=torch.int32, device=DEV), torch.arange(T, dtype=torch.int32, device=DEV)
    e = err_word()
    ops.kv_append_packed(dev[:, shift:shift + 384], 0, 192, pages.cache, pages.table.to(DEV), slot, pos, T, kv_heads, dim, e)
    out = torch.full((T, 700), 9.0, dtype=dtype, device=DEV)
    ops.kv_read_packed(pages.cache, pages.table.to(DEV), slot, pos, out[:, shift:shift + 192], out[:, 300 + shift:492 + shift], T, e)
    want = [plain.values(*plain.quantise(rows[:, at:at + 192], dim)).reshape(T, -1).float().to(dtype) for at in (0, 192)]
    got = out.cpu()
    assert torch.equal(got[:, shift:shift + 192], want[0]) and torch.equal(got[:, 300 + shift:492 + shift], want[1])
    got[:, shift:shift + 192] = got[:, 300 + shift:492 + shift] = 9.0
    assert bool((got == 9.0).all()) and int(e.item()) == 0


def test_padding_rows_and_blocks_that_are_not_mapped():
    from vlrf_b200.csrc import ops
    pages = Pages([70, 5], 2, 64)
    before = {n: getattr(pages.cache, n).clone() for n in ("k", "k_pairs", "v", "v_pairs")}
    rows = rows_of(4, 3 * 128, torch.bfloat16, seed=2).to(DEV)
    table = pages.table.to(DEV)
    slot = torch.tensor([-1, -1, -1, -1], dtype=torch.int32, device=DEV)
    pos = torch.tensor([3, 900, 0, 12], dtype=torch.int32, device=DEV)
    e = err_word()
    ops.kv_append_packed(rows, 128, 256, pages.cache, table, slot, pos, 4, 2, 64, e)
    assert all(torch.equal(getattr(pages.cache, n).view(torch.uint8), before[n].view(torch.uint8)) for n in before) and int(e.item()) == 0
    out = [torch.full((4, 128), 5.0, device=DEV) for _ in range(2)]
    ops.kv_read_packed(pages.cache, table, slot, pos, out[0], out[1], 4, e)
    assert all(bool((o == 0).all()) for o in out) and int(e.item()) == 0
    # positions without a block, beyond the table, negative; block numbers outside the cache: an error bit, nothing written
    bad = pages.table.clone()
    bad[0, 0] = pages.n_blocks
    for where, at in ((pages.table, 130), (pages.table, 10_000), (pages.table, -1), (bad, 3)):
        e = err_word()
        slot = torch.zeros(1, dtype=torch.int32, device=DEV)
        pos = torch.tensor([at], dtype=torch.int32, device=DEV)
        ops.kv_append_packed(rows, 128, 256, pages.cache, where.to(DEV), slot, pos, 1, 2, 64, e)
        assert int(e.item()) == 4
        e = err_word()
        ops.kv_read_packed(pages.cache, where.to(DEV), slot, pos, out[0], out[1], 1, e)
        assert int(e.item()) == 4 and bool((out[0][0] == 0).all())
        assert all(torch.equal(getattr(pages.cache, n).view(torch.uint8), before[n].view(torch.uint8)) for n in before)


# ---- attention ----------------------------------------------------------------------------------------------------------

def run_tokens(fn, pages, new, heads, kv_heads, dim, dtype, window, scale=None, seed=3, sharp=1.5, tensor_cores=False, check=True):
    """Sequence i's last new[i] tokens attend; `fn(qkv, q_off, table, slot, pos, out, scale, dev_err)`."""
    gen = torch.Generator().manual_seed(seed)
    T = sum(new)
    scale = 1 / math.sqrt(dim) if scale is None else scale
    qkv = (torch.randn((T, (heads + 2 * kv_heads) * dim), generator=gen) * sharp).to(dtype)
    slot = torch.tensor([i for i, a in enumerate(new) for _ in range(a)], dtype=torch.int32)
    pos = torch.tensor([n - a + j for a, n in zip(new, pages.lengths) for j in range(a)], dtype=torch.int32)
    out = torch.full((T, heads * dim), 3.0, dtype=dtype, device=DEV)
    e = err_word()
    fn(qkv.to(DEV), 0, pages.table.to(DEV), slot.to(DEV), pos.to(DEV), out, scale, e)
    assert int(e.item()) == 0
    if not check:
        return out
    contexts = [pages.context(i) for i in range(len(new))]
    worst = 0.0
    for t in range(T):
        i, p = int(slot[t]), int(pos[t])
        q = qkv[t, :heads * dim].double().view(heads, dim)
        want = plain.attend(q, contexts[i][0], contexts[i][1], scale, window, p)
        tol = bound(pages, i, p, max(0, p - window + 1) if window else 0, q, scale, want, dtype, tensor_cores)
        off = (out[t].double().cpu().view(heads, dim) - want).abs()
        assert bool((off <= tol).all()), (t, i, p, float(off.max()), float(tol.max()))
        worst = max(worst, float((off / tol).max()))
    return out, worst


SHAPES = [(3, 3, 64), (8, 2, 128), (4, 1, 32), (5, 5, 16), (2, 2, 80), (6, 3, 96), (2, 1, 256), (2, 2, 192), (12, 1, 64), (24, 1, 128)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("window", [0, 1, 37])
def test_general_attention(dtype, heads, kv_heads, dim, window):
    from vlrf_b200.csrc import ops
    pages = Pages([1, 64, 65, 200], kv_heads, dim, seed=heads)
    run_tokens(lambda qkv, q_off, table, slot, pos, out, scale, e: ops.attention_packed(
        qkv, q_off, pages.cache, table, slot, pos, out, slot.numel(), heads, kv_heads, dim, scale, window, e),
        pages, [1, 1, 2, 5], heads, kv_heads, dim, dtype, window)


def test_general_attention_skips_padding_and_reports_missing_blocks():
    from vlrf_b200.csrc import ops
    pages = Pages([100], 2, 64)
    qkv = torch.randn(3, 6 * 64, device=DEV)
    out = torch.full((3, 128), 8.0, device=DEV)
    slot, pos = torch.tensor([-1, 0, -1], dtype=torch.int32, device=DEV), torch.tensor([5, 99, 0], dtype=torch.int32, device=DEV)
    e = err_word()
    ops.attention_packed(qkv, 0, pages.cache, pages.table.to(DEV), slot, pos, out, 3, 2, 2, 64, 0.125, 0, e)
    assert bool((out[0] == 8).all()) and bool((out[2] == 8).all()) and not bool((out[1] == 8).all()) and int(e.item()) == 0
    pos[1] = 200                              # beyond the sequence's blocks
    ops.attention_packed(qkv, 0, pages.cache, pages.table.to(DEV), slot, pos, out, 3, 2, 2, 64, 0.125, 0, e)
    assert int(e.item()) == 4


def scratch(rows, heads, kv_heads, dim, n_split):
    from vlrf_b200.csrc import ops
    floats, ints = ops.packed_decode_scratch(rows, heads, kv_heads, dim, n_split)
    return torch.full((floats,), float("nan"), device=DEV), torch.zeros(ints, dtype=torch.int32, device=DEV)


@pytest.fixture(params=[1, 0], ids=["a CTA an SM", "several"])
def few(request):
    return request.param


DECODE_SHAPES = [(3, 3, 64), (8, 2, 128), (6, 2, 64), (4, 2, 128), (4, 4, 128), (2, 1, 256), (2, 2, 192), (12, 1, 64), (24, 1, 128), (40, 2, 64), (10, 1, 256)]


@pytest.mark.parametrize("heads,kv_heads,dim", DECODE_SHAPES)
@pytest.mark.parametrize("window", [0, 1, 70])
@pytest.mark.parametrize("n_split,part_tiles", [(1, 32), (3, 11), (37, 1), (2, 1)])
def test_decode_attention_on_the_tensor_cores(heads, kv_heads, dim, window, n_split, part_tiles, few):
    """Contexts of one token, of whole blocks, of a token more, longer than all stages of a warp's ring; more parts than tiles."""
    from vlrf_b200.csrc import ops
    pages = Pages([1, 64, 65, 130, 2000, 7], kv_heads, dim, seed=heads)
    run_tokens(lambda qkv, q_off, table, slot, pos, out, scale, e: ops.attention_decode_packed(
        qkv, q_off, pages.cache, table, slot, pos, out, slot.numel(), heads, kv_heads, dim, scale, window, (few, n_split, part_tiles), e,
        *scratch(6, heads, kv_heads, dim, n_split)),
        pages, [1] * 6, heads, kv_heads, dim, torch.bfloat16, window, tensor_cores=True)


@pytest.mark.parametrize("scale,sharp", [(1.0, 4.0), (1e-4, 1.0), (0.125, 1e-20), (0.125, 1e4)])
def test_decode_attention_with_sharp_and_flat_scores(scale, sharp, few):
    """Scores of many sizes: one key takes all, all alike; queries near the ends of what they may be."""
    from vlrf_b200.csrc import ops
    pages = Pages([300, 900], 2, 64, seed=4)
    run_tokens(lambda qkv, q_off, table, slot, pos, out, scale, e: ops.attention_decode_packed(
        qkv, q_off, pages.cache, table, slot, pos, out, 2, 4, 2, 64, scale, 0, (few, 2, 8), e, *scratch(2, 4, 2, 64, 2)),
        pages, [1, 1], 4, 2, 64, torch.bfloat16, 0, scale=scale, sharp=sharp, tensor_cores=True)


def test_decode_attention_skips_padding_reports_missing_blocks_and_repeats_itself(few):
    from vlrf_b200.csrc import ops
    pages = Pages([500, 40, 1300], 3, 64)
    qkv = torch.randn(5, 9 * 64, device=DEV).bfloat16()
    slot = torch.tensor([-1, 2, 0, -1, 1], dtype=torch.int32, device=DEV)
    pos = torch.tensor([5, 1299, 499, 0, 39], dtype=torch.int32, device=DEV)
    table, e = pages.table.to(DEV), err_word()
    outs, room = [], scratch(5, 3, 3, 64, 4)
    for n_split in (1, 4, 4):
        out = torch.full((5, 192), 8.0, device=DEV, dtype=torch.bfloat16)
        ops.attention_decode_packed(qkv, 0, pages.cache, table, slot, pos, out, 5, 3, 3, 64, 0.125, 0, (few, n_split, 6), e, *room)
        assert int(room[1].abs().sum()) == 0
        assert bool((out[0] == 8).all()) and bool((out[3] == 8).all()) and int(e.item()) == 0
        outs.append(out)
    assert torch.equal(outs[1], outs[2])
    bad = table.clone()
    bad[2, 7], bad[0, 1] = -1, pages.n_blocks        # a page in the middle that is not mapped, one outside the cache
    ops.attention_decode_packed(qkv, 0, pages.cache, bad, slot, pos, outs[1], 5, 3, 3, 64, 0.125, 0, (few, 4, 6), e, *room)
    assert int(e.item()) == 4 and torch.equal(outs[1][4], outs[2][4])
    pos[1] = 100_000
    e.zero_()
    ops.attention_decode_packed(qkv, 0, pages.cache, table, slot, pos, outs[1], 5, 3, 3, 64, 0.125, 0, (few, 4, 6), e, *room)
    assert int(e.item()) == 4


def prefill(pages, new, heads, kv_heads, dim, window, groups, n_parts, scratch=None):
    """For `run_tokens`: the prompt kernel over sequences that bring new[i] tokens each."""
    from vlrf_b200.csrc import ops
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)   # noqa: E731
    start = [0]
    for a in new:
        start.append(start[-1] + a)
    floats, counts = ops.packed_prefill_scratch(len(new), max(new), heads, dim, groups, n_parts)
    partials, counters = torch.full((floats,), float("nan"), device=DEV), torch.zeros(counts, dtype=torch.int32, device=DEV)

    def fn(qkv, q_off, table, slot, pos, out, scale, e):
        ops.attention_prefill_packed(qkv, q_off, pages.cache, table, ints(list(range(len(new)))), ints(start), ints([n - a for a, n in zip(new, pages.lengths)]),
                                     out, sum(new), len(new), max(new), heads, kv_heads, dim, scale, window, e, groups, n_parts, 2, partials, counters)
        assert int(counters.abs().sum()) == 0
    return fn


PROMPTS = [([1], [0]), ([5], [64]), ([128], [0]), ([129, 2], [0, 127]), ([300, 1, 64], [77, 700, 0]), ([260], [500])]


@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 3, 64), (4, 1, 64), (2, 2, 128), (6, 2, 128)])
@pytest.mark.parametrize("new,past", PROMPTS)
@pytest.mark.parametrize("window", [0, 1, 100])
@pytest.mark.parametrize("groups,n_parts", [(1, 1), (2, 1), (1, 3), (2, 16)])
def test_prompt_attention_on_the_tensor_cores(heads, kv_heads, dim, new, past, window, groups, n_parts):
    """The bound counts three roundings here: a weight, a key and a value as float16."""
    pages = Pages([a + b for a, b in zip(new, past)], kv_heads, dim, seed=heads + sum(new))
    check_prompt(prefill(pages, new, heads, kv_heads, dim, window, groups, n_parts), pages, new, heads, kv_heads, dim, window)


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 64), (2, 2, 128)])
@pytest.mark.parametrize("new,past", [([1, 1, 1, 300, 1, 2, 1, 1, 1], [5, 70, 0, 100, 64, 3, 200, 63, 9]), ([1] * 33 + [270, 3, 130] + [1] * 4, list(range(40))),
                                      ([0, 400, 0, 0, 0, 1, 0, 0, 0], [3, 0, 1, 64, 0, 127, 0, 5, 0])])
@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("groups,n_parts", [(1, 1), (2, 1), (2, 3)])
def test_prompt_attention_of_one_long_sequence_among_single_tokens(heads, kv_heads, dim, new, past, window, groups, n_parts):
    """More sequences than tiles of the longest: the grid has a place a tile."""
    pages = Pages([a + b for a, b in zip(new, past)], kv_heads, dim, seed=heads + len(new))
    check_prompt(prefill(pages, new, heads, kv_heads, dim, window, groups, n_parts), pages, new, heads, kv_heads, dim, window)


def check_prompt(fn, pages, new, heads, kv_heads, dim, window):
    """A sample of the tokens against float64.  A number of a key or a value is off by h = 2^-11 of itself, and, where it lies below float16's normal range (2^-14
    of its first block's, or 2^-28 of its own row's largest), by less than that of the largest; so by 2 h of the largest at the very most.  That moves a score by
    e_k ≤ 2 h · scale · Σ |q| · |k|max, the weights by a factor of exp(2 e_k) together, and the result by 2 h |v|max.  A weight is off by h of itself, and below
    float16's range by 2^-25 where the row's reference point has 2^4: h + n 2^-29 of |v|max."""
    T, scale = sum(new), 1 / math.sqrt(dim)
    qkv = (torch.randn((T, (heads + 2 * kv_heads) * dim), generator=torch.Generator().manual_seed(9)) * 1.2).bfloat16()
    slot = [i for i, a in enumerate(new) for _ in range(a)]
    pos = [n - a + j for a, n in zip(new, pages.lengths) for j in range(a)]
    out = torch.full((T, heads * dim), 3.0, dtype=torch.bfloat16, device=DEV)
    e = err_word()
    fn(qkv.to(DEV), 0, pages.table.to(DEV), None, None, out, scale, e)
    assert int(e.item()) == 0
    got, share = out.double().cpu(), heads // kv_heads
    contexts = [pages.context(i) for i in range(len(new))]
    edges = {0, T - 1}
    for i, a in enumerate(new):
        s = sum(new[:i])
        edges |= {s, s + a - 1} | {s + x for x in (1, 63, 64, 127, 128, 129, 255, 256) if x < a}
    for t in sorted((edges | set(range(0, T, 37))) & set(range(T))):        # (a sequence that brings nothing has no rows)
        i, p = slot[t], pos[t]
        k, v = contexts[i]
        first = max(0, p - window + 1) if window else 0
        q = qkv[t, :heads * dim].double().view(heads, dim)
        want = plain.attend(q, k, v, scale, window, p)
        for h in range(heads):
            kk, vv = k[first:p + 1, h // share], v[first:p + 1, h // share]
            e_k = (2.0 ** -10 + (dim + 16) * U) * scale * float(kk.abs().max() * q[h].abs().sum())
            tol = float(vv.abs().max()) * (math.expm1(2 * e_k) + 3 * 2.0 ** -11 + (p + 1 - first) * 2.0 ** -29 + (p + 1 - first + 32) * U)
            tol = tol + HALF_STEP * (want[h].abs() + tol)
            off = (got[t].view(heads, dim)[h] - want[h]).abs()
            assert bool((off <= tol).all()), (t, i, p, h, float(off.max()), float(tol.max()))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("groups,n_parts", [(1, 1), (2, 1), (1, 4)])
def test_prompt_attention_is_as_good_as_its_roundings_are_random(dim, groups, n_parts):
    """The bound above takes every rounding at its worst; over many numbers they cancel, and what is left beside the result's own rounding is little.  The
    mean square error of 400 tokens is held to that of the same roundings done in float64 on the host, plus a quarter."""
    heads, new = 2, [400]
    pages = Pages([700], heads, dim, seed=2)
    qkv = (torch.randn((400, 3 * heads * dim), generator=torch.Generator().manual_seed(9)) * 1.2).bfloat16()
    out = torch.empty((400, heads * dim), dtype=torch.bfloat16, device=DEV)
    e = err_word()
    prefill(pages, new, heads, heads, dim, 0, groups, n_parts)(qkv.to(DEV), 0, pages.table.to(DEV), None, None, out, 1 / math.sqrt(dim), e)
    k, v = pages.context(0)
    r = lambda x: x.float().bfloat16().double()   # noqa: E731
    err = ref = 0.0
    for h in range(heads):
        q = qkv[:, h * dim:(h + 1) * dim].double()
        mask = torch.arange(700)[None] <= torch.arange(300, 700)[:, None]
        want = torch.softmax(((q @ k[:, h].T) / math.sqrt(dim)).masked_fill(~mask, -math.inf), 1) @ v[:, h]
        s = ((q @ k[:, h].half().double().T) / math.sqrt(dim)).masked_fill(~mask, -math.inf)
        w = torch.exp(s - s[:, :64].amax(1, keepdim=True))
        rounded = r((w.half().double() @ v[:, h].half().double()) / w.sum(1, keepdim=True))
        err += float(((out.double().cpu()[:, h * dim:(h + 1) * dim] - want) ** 2).mean())
        ref += float(((rounded - want) ** 2).mean())
    assert int(e.item()) == 0 and err <= 1.25 * ref, (err, ref)


def test_prompt_attention_skips_padding_reports_missing_blocks_and_leaves_rows_behind():
    from vlrf_b200.csrc import ops
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)   # noqa: E731
    pages = Pages([200, 150], 2, 64)
    qkv = torch.randn(120, 6 * 64, device=DEV).bfloat16()
    table = pages.table.to(DEV)
    outs = []
    for slots in ([0, -1], [0, 1]):
        out = torch.full((120, 128), 8.0, device=DEV, dtype=torch.bfloat16)
        e = err_word()
        ops.attention_prefill_packed(qkv, 0, pages.cache, table, ints(slots), ints([0, 50, 100]), ints([150, 100]), out, 100, 2, 50, 2, 2, 64, 0.125, 0, e)
        assert int(e.item()) == 0 and bool((out[100:] == 8).all()) and bool((out[50:100] == 8).all()) == (slots[1] < 0)
        outs.append(out)
    assert torch.equal(outs[0][:50], outs[1][:50])
    for value in (-1, pages.n_blocks):
        bad = table.clone()
        bad[1, 0] = value
        e = err_word()
        ops.attention_prefill_packed(qkv, 0, pages.cache, bad, ints([0, 1]), ints([0, 50, 100]), ints([150, 100]), out, 100, 2, 50, 2, 2, 64, 0.125, 0, e)
        assert int(e.item()) == 4 and torch.equal(out[:50], outs[1][:50])
        e = err_word()                         # a block that lies wholly before the window is not asked for
        ops.attention_prefill_packed(qkv, 0, pages.cache, bad, ints([0, 1]), ints([0, 50, 100]), ints([150, 100]), out, 100, 2, 50, 2, 2, 64, 0.125, 37, e)
        assert int(e.item()) == 0 and not bool(torch.isnan(out[:100]).any())


@pytest.mark.parametrize("dim", [64, 128])
def test_prompt_rows_that_do_not_see_a_number_that_is_not_finite_stay_finite(dim):
    pages = Pages([200], 2, dim)
    for name, p, head in (("k_pairs", 90, 0), ("v_pairs", 130, 1)):
        getattr(pages.cache, name)[int(pages.table[0, p // 64]), head, p % 64, -1] = float("nan")
    qkv = torch.randn(150, 6 * dim, device=DEV).bfloat16()
    for window in (0, 20):
        for groups, n_parts in ((1, 1), (2, 1), (1, 3)):
            out = torch.zeros(150, 2 * dim, device=DEV, dtype=torch.bfloat16)
            e = err_word()
            prefill(pages, [150], 2, 2, dim, window, groups, n_parts)(qkv, 0, pages.table.to(DEV), None, None, out, 0.1, e)
            pos = torch.arange(50, 200)
            for head, p in ((0, 90), (1, 130)):
                sees = (pos >= p) & ((pos < p + window) if window else torch.ones_like(pos, dtype=torch.bool))
                nan = torch.isnan(out.cpu()[:, head * dim:(head + 1) * dim])
                assert torch.equal(nan.any(1), sees) and torch.equal(nan.all(1), sees), (window, groups, n_parts, head)


def test_numbers_that_are_not_finite_show_in_their_rows_only(few):
    """A visible key or value that is not a number makes its sequence's head NaN; hidden ones nothing (the pages' leftovers are NaN everywhere)."""
    from vlrf_b200.csrc import ops
    pages = Pages([200, 200], 2, 64)
    blk = int(pages.table[0, 1])
    pages.cache.k_pairs[blk, 0, 5] = float("nan")
    blk = int(pages.table[1, 0])
    pages.cache.v_pairs[blk, 1, 60] = float("nan")
    qkv = torch.randn(2, 6 * 64, device=DEV).bfloat16()
    slot, pos = torch.arange(2, dtype=torch.int32, device=DEV), torch.full((2,), 199, dtype=torch.int32, device=DEV)
    for n_split, window in ((1, 0), (3, 0), (1, 50), (2, 140)):
        out, general = [torch.zeros(2, 128, device=DEV, dtype=torch.bfloat16) for _ in range(2)]
        ops.attention_decode_packed(qkv, 0, pages.cache, pages.table.to(DEV), slot, pos, out, 2, 2, 2, 64, 0.125, window, (few, n_split, 2), err_word(),
                                    *scratch(2, 2, 2, 64, n_split))
        ops.attention_packed(qkv, 0, pages.cache, pages.table.to(DEV), slot, pos, general, 2, 2, 2, 64, 0.125, window, err_word())
        nan = torch.zeros(2, 128, dtype=torch.bool)
        nan[0, :64] = window == 0 or window == 140   # position 69
        nan[1, 64:] = window in (0, 140)             # position 60
        assert torch.equal(torch.isnan(out.cpu()), nan) and torch.equal(torch.isnan(general.cpu()), nan), (n_split, window)


def test_refusals():
    from vlrf_b200.csrc import KernelError, ops
    pages = Pages([70], 2, 64)
    rows, table = torch.randn(4, 6 * 64, device=DEV), pages.table.to(DEV)
    slot, pos, e = torch.zeros(4, dtype=torch.int32, device=DEV), torch.arange(4, dtype=torch.int32, device=DEV), err_word()
    out = torch.empty(4, 128, device=DEV)

    def append(**kw):
        a = dict(qkv=rows, k_off=128, v_off=256, cache=pages.cache, block_table=table, tok_slot=slot, tok_pos=pos, n_tokens=4, n_kv_heads=2,
                 head_dim=64, dev_err=e)
        ops.kv_append_packed(**dict(a, **kw))

    def attend(**kw):
        a = dict(qkv=rows, q_off=0, cache=pages.cache, block_table=table, tok_slot=slot, tok_pos=pos, out=out, n_tokens=4, n_heads=2, n_kv_heads=2,
                 head_dim=64, scale=0.125, window=0, dev_err=e)
        ops.attention_packed(**dict(a, **kw))

    append(); attend()
    c = pages.cache
    for call, kw in [(append, dict(qkv=rows.half())), (append, dict(qkv=rows.cpu())), (append, dict(k_off=-1)), (append, dict(v_off=257)),
                     (append, dict(n_tokens=5)), (append, dict(head_dim=32)), (append, dict(head_dim=72)), (append, dict(n_kv_heads=1)),
                     (append, dict(cache=None)), (append, dict(tok_pos=pos.long())),
                     (append, dict(block_table=table[0])), (append, dict(qkv=rows.t())),
                     (attend, dict(out=out.bfloat16())), (attend, dict(n_heads=3)), (attend, dict(q_off=400)), (attend, dict(window=-1)),
                     (attend, dict(out=out[:3])), (attend, dict(qkv=rows[:2]))]:
        with pytest.raises(KernelError):
            call(**kw)
    with pytest.raises(KernelError):
        ops.kv_read_packed(c, table, slot, pos, out[:, :64], out, 4, e)
    for tensors in [(c.k, c.k_pairs.float(), c.v, c.v_pairs), (c.k, c.k_pairs, c.v[:1], c.v_pairs), (c.k.cpu(), c.k_pairs, c.v, c.v_pairs),
                    (c.k, c.k_pairs, c.v, c.v_pairs[..., :1]), (c.k.char(), c.k_pairs, c.v, c.v_pairs)]:
        with pytest.raises(KernelError):
            ops.PackedKV(*tensors)
    with pytest.raises(KernelError):
        ops.PackedKV.zeros(3, 2, 64, 24, DEV)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sharp,size", [(1e4, 1.0), (1e-6, 1.0), (1.0, 1e5), (1.0, 1e-6), (1e3, 1e-3), (0.0, 1.0), (1.0, 1e-30), (1e-30, 1.0), (1e12, 1e20)])
def test_prompt_attention_with_queries_and_keys_of_many_sizes(dim, sharp, size):
    """Queries and keys that float16 does not hold as they are."""
    heads, new = 2, [140]
    pages = Pages([200], heads, dim, seed=5)
    pages.host["k_pairs"] = (pages.host["k_pairs"].float() * size).bfloat16()
    pages.cache.k_pairs.copy_(pages.host["k_pairs"])
    qkv = (torch.randn((140, 3 * heads * dim), generator=torch.Generator().manual_seed(9)) * sharp).bfloat16()
    scale = 1.0 / (math.sqrt(dim) * max(sharp, 1e-9) * size)
    out = torch.zeros((140, heads * dim), dtype=torch.bfloat16, device=DEV)
    e = err_word()
    prefill(pages, new, heads, heads, dim, 0, 2, 1)(qkv.to(DEV), 0, pages.table.to(DEV), None, None, out, scale, e)
    assert int(e.item()) == 0
    k, v = pages.context(0)
    for t in (0, 1, 70, 139):
        q = qkv[t, :heads * dim].double().view(heads, dim)
        want = plain.attend(q, k, v, scale, 0, 60 + t)
        for h in range(heads):
            kk, vv = k[:61 + t, h], v[:61 + t, h]
            e_k = (2.0 ** -10 + (dim + 16) * U) * scale * float(kk.abs().max() * q[h].abs().sum())
            tol = float(vv.abs().max()) * (math.expm1(2 * e_k) + 3 * 2.0 ** -11 + 400 * U)
            tol = tol + HALF_STEP * (want[h].abs() + tol)
            assert bool(((out[t].double().cpu().view(heads, dim)[h] - want[h]).abs() <= tol).all()), (t, h)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("groups,n_parts", [(1, 1), (2, 1), (2, 3)])
@pytest.mark.parametrize("which", ["k_pairs", "v_pairs", "both"])
@pytest.mark.parametrize("far,size", [((70, 100, 101, 190), 2.0 ** 20), ((3, 150), 2.0 ** 40), (tuple(range(64)), 2.0 ** 18), ((66, 130), 2.0 ** 15),
                                      (tuple(range(64, 128)), 2.0 ** 60), (tuple(range(0, 200, 2)), 2.0 ** 17)])
def test_prompt_attention_with_tokens_of_many_sizes(dim, groups, n_parts, which, far, size):
    """Tokens whose keys or values lie far above those of the others; a row that does not see them has nothing of it."""
    heads, new, past = 2, [140], 60
    pages = Pages([200], heads, dim, seed=6)
    parts = ["k_pairs", "v_pairs"] if which == "both" else [which]
    for name in parts:
        for t in far:
            block = int(pages.table[0, t // 64])
            pages.host[name][block, :, t % 64] = (pages.host[name][block, :, t % 64].float() * size).bfloat16()
        getattr(pages.cache, name).copy_(pages.host[name])
    qkv = (torch.randn((140, 3 * heads * dim), generator=torch.Generator().manual_seed(9)) * 1.2).bfloat16()
    scale = 1.0 / (math.sqrt(dim) * (size if "k_pairs" in parts else 1.0))
    out = torch.zeros((140, heads * dim), dtype=torch.bfloat16, device=DEV)
    e = err_word()
    prefill(pages, new, heads, heads, dim, 0, groups, n_parts)(qkv.to(DEV), 0, pages.table.to(DEV), None, None, out, scale, e)
    assert int(e.item()) == 0
    k, v = pages.context(0)
    for t in (0, 3, 9, 10, 40, 41, 70, 89, 90, 139):
        q = qkv[t, :heads * dim].double().view(heads, dim)
        want = plain.attend(q, k, v, scale, 0, past + t)
        for h in range(heads):
            kk, vv = k[:past + 1 + t, h], v[:past + 1 + t, h]
            e_k = (2.0 ** -10 + (dim + 16) * U) * scale * float(kk.abs().max() * q[h].abs().sum())
            tol = float(vv.abs().max()) * (math.expm1(2 * e_k) + 3 * 2.0 ** -11 + 400 * U)
            tol = tol + HALF_STEP * (want[h].abs() + tol)
            assert bool(((out[t].double().cpu().view(heads, dim)[h] - want[h]).abs() <= tol).all()), (t, h)


def test_a_query_that_is_not_finite_leaves_the_other_rows_alone():
    pages = Pages([150], 2, 64)
    qkv = torch.randn(150, 6 * 64).bfloat16()
    outs = []
    for bad in (None, float("inf"), float("nan")):
        x = qkv.clone()
        if bad is not None:
            x[77, 3] = bad                     # head 0
        out = torch.zeros(150, 128, device=DEV, dtype=torch.bfloat16)
        e = err_word()
        prefill(pages, [150], 2, 2, 64, 0, 2, 1)(x.to(DEV), 0, pages.table.to(DEV), None, None, out, 0.125, e)
        outs.append(out.cpu())
    for o in outs[1:]:
        assert bool(torch.isnan(o[77, :64]).any())
        o[77, :64] = outs[0][77, :64]
        assert torch.equal(o, outs[0])
