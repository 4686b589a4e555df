"""The cache in 4 bits the way programs use it: append, attend and read in one run, on another stream, captured and replayed, in caches whose
offsets pass 32 bits, in steps that bring nothing, and from the command line.  The kernels' numbers are held elsewhere; here results are
compared bit by bit with those of the same calls made plainly, or with float64 within the bound of bfloat16 results."""
import math

import pytest
import torch

import plain_packed as plain
from vlrf_b200.cli import main
from vlrf_b200.parts.context import StepContext, Workspace

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF_STEP = 2.0 ** -8


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def step_of(new, past, ws=None, slots=None):
    start = [0]
    for a in new:
        start.append(start[-1] + a)
    slots = list(range(len(new))) if slots is None else slots
    tok_slot = ints([s for s, a in zip(slots, new) for _ in range(a)])
    tok_pos = ints([b + j for a, b in zip(new, past) for j in range(a)])
    return StepContext(n_tokens=sum(new), tokens=tok_slot, tok_slot=tok_slot, tok_pos=tok_pos, n_seqs=len(new), seq_slot=ints(slots), seq_start=ints(start),
                       seq_pos0=ints(past), max_new=max(new), max_context=max(a + b for a, b in zip(new, past)), logit_rows=tok_slot, n_logit_rows=0,
                       act_dtype=torch.bfloat16, dev_err=ints([0]), ws=ws or Workspace(DEV), host_seq_slots=slots, host_seq_lens=list(new),
                       host_seq_pos0=list(past), min_new=min(new))


def run_step(cache, table, rows, out, ctx, H, G, d, scale=None, window=0):
    from vlrf_b200.csrc import ops
    ops.kv_append_packed(rows, H * d, (H + G) * d, cache, table, ctx.tok_slot, ctx.tok_pos, ctx.n_tokens, G, d, ctx.dev_err)
    ops.attention_packed_step(rows, 0, cache, table, out, ctx, H, G, d, 1 / math.sqrt(d) if scale is None else scale, window)


def check_against_float64(all_rows, got, at, H, G, d, scale, window=0, held=None):
    """got[i] is the attention of the row at position at[i] over all rows up to it; bounds as for bfloat16 weights times steps and a bfloat16 result, scores
    in float32 or of float16 operands (off by 2^-10 of Σ |q| |k|max at most).  held: what the cache holds, where it is known (else the rows, quantised)."""
    k, v = held or [plain.values(*plain.quantise(all_rows[:, c:c + G * d], d)) for c in (H * d, (H + G) * d)]
    for i, p in enumerate(at):
        q = all_rows[p, :H * d].double().view(H, d)
        want = plain.attend(q, k, v, scale, window, p)
        for h in range(H):
            kk, vv = k[:p + 1, h // (H // G)], v[:p + 1, h // (H // G)]
            e_k = 2.0 ** -10 * abs(scale) * float(kk.abs().max() * q[h].abs().sum())
            tol = float(vv.abs().max()) * (math.expm1(2 * e_k) + 2 * HALF_STEP)     # (15 step of a group is twice its largest number at most)
            tol = tol + HALF_STEP * (want[h].abs() + tol)
            assert bool(((got[i].double().cpu().view(H, d)[h] - want[h]).abs() <= tol).all()), (p, h)


def cache_for(n_tokens, G, d, n_seqs=1, spare=2):
    from vlrf_b200.csrc import ops
    per = -(-n_tokens // 64)
    cache = ops.PackedKV.zeros(per * n_seqs + spare, G, 64, d, DEV)
    cache.k_pairs.fill_(float("nan")); cache.v_pairs.fill_(float("nan"))
    order = torch.randperm(per * n_seqs + spare, generator=torch.Generator().manual_seed(1))[:per * n_seqs]
    return cache, order.int().view(n_seqs, per).to(DEV)


def qkv_rows(T, H, G, d, seed=0):
    return (torch.randn((T, (H + 2 * G) * d), generator=torch.Generator().manual_seed(seed)) * 1.2).bfloat16()


@pytest.mark.parametrize("H,G,d", [(4, 4, 64), (8, 2, 128), (3, 1, 256), (2, 2, 80)])
@pytest.mark.parametrize("window", [0, 50])
def test_a_prompt_its_pieces_single_tokens_and_reading_back(H, G, d, window):
    from vlrf_b200.csrc import ops
    pieces = [130, 1, 64, 7, 1, 1, 200, 1]
    T, scale = sum(pieces), 1 / math.sqrt(d)
    cache, table = cache_for(T, G, d)
    rows = qkv_rows(T, H, G, d)
    got, at, ws = torch.full((T, H * d), 3.0, dtype=torch.bfloat16, device=DEV), 0, Workspace(DEV)
    for n in pieces:
        ctx = step_of([n], [at], ws)
        run_step(cache, table, rows[at:at + n].to(DEV), got[at:at + n], ctx, H, G, d, window=window)
        assert int(ctx.dev_err.item()) == 0
        at += n
    check = [0, 1, 63, 64, 129, 130, 131, 194, 195, 201, 202, 203, 204, 300, T - 2, T - 1]
    check_against_float64(rows, got[check], check, H, G, d, scale, window)
    back = [torch.empty((T, G * d), device=DEV) for _ in range(2)]
    e = ints([0])
    ops.kv_read_packed(cache, table, ints([0] * T), ints(list(range(T))), back[0], back[1], T, e)
    for x, c in zip(back, (H * d, (H + G) * d)):
        assert torch.equal(x.cpu().double(), plain.values(*plain.quantise(rows[:, c:c + G * d], d)).flatten(1).float().double())


@pytest.mark.parametrize("n_new", [1, 70])
def test_offsets_past_32_bits(n_new):
    """A cache of 140,000 blocks of 8 heads of 64: its codes alone are 2 · 4.3 GiB, and the sequence lies in the last blocks."""
    from vlrf_b200.csrc import ops
    H, G, d, n_blocks, past = 8, 8, 64, 140_000, 100
    cache = ops.PackedKV.zeros(n_blocks, G, 64, d, DEV)
    assert cache.k.numel() > 2 ** 31
    table = ints([[n_blocks - 1, 5, n_blocks - 2]])
    rows = qkv_rows(past + n_new, H, G, d)
    out = torch.zeros((past + n_new, H * d), dtype=torch.bfloat16, device=DEV)
    first, then = step_of([past], [0]), step_of([n_new], [past])
    run_step(cache, table, rows[:past].to(DEV), out[:past], first, H, G, d)
    run_step(cache, table, rows[past:].to(DEV), out[past:], then, H, G, d)
    assert int(first.dev_err.item()) == 0 and int(then.dev_err.item()) == 0
    check = [0, 64, past - 1, past, past + n_new - 1]
    check_against_float64(rows, out[check], check, H, G, d, 1 / math.sqrt(d))
    assert int(cache.k[n_blocks - 1].any()) and not int(cache.k[6:n_blocks - 2].any())


@pytest.mark.parametrize("H,G,d", [(25, 25, 64), (32, 4, 128)])
@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("new", [[1] * 9 + [150], [70, 1, 0, 1, 1, 130, 1, 1, 1, 1], [3, 1, 1, 1, 1, 1, 1, 1]])
def test_single_tokens_among_prompts_go_to_the_decode_kernel(H, G, d, window, new, monkeypatch):
    """Many single tokens with long contexts: two kernels share the step, no row is left out or written by the wrong one."""
    from vlrf_b200.csrc import ops
    past = [(97 * i + 460) % 900 for i in range(len(new))]
    seen = []
    for name in ("attention_decode_packed", "attention_prefill_packed"):
        inner = getattr(ops, name)
        monkeypatch.setattr(ops, name, lambda *a, inner=inner, name=name, **kw: (seen.append(name), inner(*a, **kw)) and None)
    cache, table = cache_for(1100, G, d, len(new))
    whole, ws = [], Workspace(DEV)
    for i, (a, b) in enumerate(zip(new, past)):            # the contexts, sequence by sequence
        whole.append(qkv_rows(a + b, H, G, d, seed=i))
        if b:
            ctx = step_of([b], [0], slots=[i])
            ops.kv_append_packed(whole[i][:b].to(DEV), H * d, (H + G) * d, cache, table, ctx.tok_slot, ctx.tok_pos, b, G, d, ctx.dev_err)
    out = torch.full((sum(new) + 2, H * d), 3.0, dtype=torch.bfloat16, device=DEV)
    ctx = step_of(new, past, ws)
    run_step(cache, table, torch.cat([w[b:] for w, b in zip(whole, past)]).to(DEV), out[:sum(new)], ctx, H, G, d, window=window)
    assert int(ctx.dev_err.item()) == 0 and bool((out[sum(new):] == 3).all()) and seen == ["attention_prefill_packed", "attention_decode_packed"]
    at, host, blocks = 0, {n: getattr(cache, n).cpu() for n in ("k", "k_pairs", "v", "v_pairs")}, table.cpu().long()
    for i, (w, a, b) in enumerate(zip(whole, new, past)):
        if a:
            place = torch.arange(a + b)
            held = [plain.unpacked(host[n][blocks[i, place // 64], :, place % 64], host[n + "_pairs"][blocks[i, place // 64], :, place % 64]) for n in ("k", "v")]
            check_against_float64(w, out[[at, at + a - 1]], [b, b + a - 1], H, G, d, 1 / math.sqrt(d), window, held)
        at += a
    # the same step in one kernel is no further off than the two may be from one another
    monkeypatch.setattr(ops, "PACKED_SINGLES_APART", 10 ** 9)
    alone = torch.zeros_like(out)
    run_step(cache, table, torch.cat([w[b:] for w, b in zip(whole, past)]).to(DEV), alone[:sum(new)], step_of(new, past), H, G, d, window=window)
    at = 0
    for a in new:
        if a != 1:
            assert torch.equal(alone[at:at + a], out[at:at + a]) or float((alone[at:at + a] - out[at:at + a]).abs().max()) <= 2 * HALF_STEP * float(out.abs().max())
        at += a


def test_rows_of_entries_are_checked():
    from vlrf_b200.csrc import KernelError, ops
    cache, table = cache_for(64, 2, 64)
    rows, out = qkv_rows(3, 2, 2, 64).to(DEV), torch.zeros((3, 128), dtype=torch.bfloat16, device=DEV)
    for row_of in (ints([0, 1, 2]), torch.tensor([0, 1, 2, 3], device=DEV)):            # too few; int64
        with pytest.raises(KernelError):
            ops.attention_decode_packed(rows, 0, cache, table, ints([0, 0, 0]), ints([0, 1, 2]), out, 3, 2, 2, 64, 0.125, 0, (False, 1, 1), ints([0]), row_of=row_of)


@pytest.mark.parametrize("new,past", [([1, 1, 1], [700, 3, 300]), ([90, 1, 300], [700, 64, 0])])
def test_another_stream(new, past):
    H, G, d = 4, 2, 128
    outs = []
    for side in (False, True):
        cache, table = cache_for(1100, G, d, len(new))
        cache.k_pairs.fill_(0.5); cache.v_pairs.fill_(0.25)
        rows, out, ctx = qkv_rows(sum(new), H, G, d).to(DEV), torch.zeros((sum(new), H * d), dtype=torch.bfloat16, device=DEV), step_of(new, past)
        stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            run_step(cache, table, rows, out, ctx, H, G, d)
        stream.synchronize()
        assert int(ctx.dev_err.item()) == 0
        outs.append(out)
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("new,past", [([1] * 3, [2000, 3, 300]), ([90, 1, 300], [900, 64, 0])])
def test_captured_and_replayed_with_other_numbers(new, past):
    """Two graphs of the same workspace, replayed in turn with other rows in place."""
    H, G, d = 4, 2, 64
    T = sum(new)
    caches = [cache_for(2100, G, d, len(new)) for _ in range(4)]
    for c, _ in caches:
        c.k_pairs.fill_(0.5); c.v_pairs.fill_(0.25)
    ws, graphs, bufs = Workspace(DEV), [], []
    for i in range(2):
        cache, table = caches[i]
        rows, out, ctx = qkv_rows(T, H, G, d, 50 + i).to(DEV), torch.zeros((T, H * d), dtype=torch.bfloat16, device=DEV), step_of(new, past, ws)
        run_step(cache, table, rows, out, ctx, H, G, d)                           # (makes the workspaces)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run_step(cache, table, rows, out, ctx, H, G, d)
        graphs.append(g); bufs.append((rows, out, ctx))
    for turn in range(3):
        for i in range(2):
            x = qkv_rows(T, H, G, d, 10 * turn + i).to(DEV)
            bufs[i][0].copy_(x)
            graphs[i].replay()
            torch.cuda.synchronize()
            want, ctx = torch.zeros_like(bufs[i][1]), step_of(new, past)
            run_step(*caches[2 + i], x, want, ctx, H, G, d)
            assert torch.equal(bufs[i][1], want) and int(bufs[i][2].dev_err.item()) == 0
            assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in
                       zip((caches[i][0].k, caches[i][0].k_pairs, caches[i][0].v, caches[i][0].v_pairs),
                           (caches[2 + i][0].k, caches[2 + i][0].k_pairs, caches[2 + i][0].v, caches[2 + i][0].v_pairs)))


@pytest.mark.parametrize("scale", [-0.125, 0.0])
@pytest.mark.parametrize("n_new", [1, 80])
def test_scales_of_zero_and_below(scale, n_new):
    H, G, d = 2, 1, 64
    T = 150
    cache, table = cache_for(T, G, d)
    rows = qkv_rows(T, H, G, d)
    out = torch.zeros((T, H * d), dtype=torch.bfloat16, device=DEV)
    for a, b in ((0, T - n_new), (T - n_new, T)):
        ctx = step_of([b - a], [a])
        run_step(cache, table, rows[a:b].to(DEV), out[a:b], ctx, H, G, d, scale=scale)
        assert int(ctx.dev_err.item()) == 0
    check = [0, 1, 69, 70, T - 1]
    check_against_float64(rows, out[check], check, H, G, d, scale)


@pytest.mark.parametrize("d", [64, 80])
def test_steps_that_bring_nothing_and_sequences_that_do(d):
    from vlrf_b200.csrc import ops
    H, G = 2, 2
    cache, table = cache_for(200, G, d, 3)
    before = [t.clone() for t in (cache.k, cache.k_pairs.view(torch.int16), cache.v, cache.v_pairs.view(torch.int16))]
    out = torch.full((4, H * d), 7.0, dtype=torch.bfloat16, device=DEV)
    rows, e, none = qkv_rows(4, H, G, d).to(DEV), ints([0]), ints([0, 0, 0, 0])
    ops.kv_append_packed(rows, H * d, 2 * H * d, cache, table, none, none, 0, G, d, e)
    ops.attention_packed(rows, 0, cache, table, none, none, out, 0, H, G, d, 0.1, 0, e)
    if d == 64:
        ops.attention_decode_packed(rows, 0, cache, table, none, none, out, 0, H, G, d, 0.1, 0, (False, 1, 1), e)
        ops.attention_prefill_packed(rows, 0, cache, table, none, none, none, out, 0, 3, 0, H, G, d, 0.1, 0, e)
    assert bool((out == 7).all()) and int(e.item()) == 0
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.k_pairs.view(torch.int16), cache.v, cache.v_pairs.view(torch.int16))))
    # the middle sequence brings nothing; the others' rows are what they are without it
    outs = []
    for new, past, slots in (([3, 0, 70], [0, 50, 0], [0, 1, 2]), ([3, 70], [0, 0], [0, 2])):
        ctx = step_of(new, past, slots=slots)
        outs.append(torch.zeros((73, H * d), dtype=torch.bfloat16, device=DEV))
        run_step(cache, table, qkv_rows(73, H, G, d).to(DEV), outs[-1], ctx, H, G, d)
        assert int(ctx.dev_err.item()) == 0
    assert torch.equal(outs[0], outs[1]) and bool(torch.isfinite(outs[0]).all())


def test_the_command_line(model_dirs, tmp_path, capsys):
    f = tmp_path / "prompts.txt"
    f.write_text("5 17 3 900 44\n7\n")
    texts = []
    for extra in (["--kv-cache", "int4"], ["--kv-cache", "model"]):
        assert main(["run", "--model", str(model_dirs["tiny_b"]), "--prompts-file", str(f), "--tokens", "6", "--greedy", "--stop-id", "999",
                     "--dtype", "float32"] + extra) in (0, None)
        texts.append(capsys.readouterr().out)
        assert "12 generated" in texts[-1]
