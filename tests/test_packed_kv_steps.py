"""Steps over a cache of 4 bits as a whole: the scratch they take, and lengths that the host does not know.  On the CPU the kernels' launches are the test's stand-ins; the plans and the scratch are
the library's own."""
import random

import pytest
import torch

from vlrf_b200.parts.context import StepContext, Workspace


@pytest.fixture
def launches(monkeypatch):
    """What a step launches, as (name, positional arguments, others), on a device of 148 SMs."""
    from vlrf_b200.csrc import ops
    seen = []
    monkeypatch.setattr(ops, "_SM_COUNT", 148)
    ops._packed_decode_shape.cache_clear(); ops._packed_prefill_shape.cache_clear()
    for name in ("attention_packed", "attention_decode_packed", "attention_prefill_packed"):
        monkeypatch.setattr(ops, name, lambda *a, name=name, **kw: seen.append((name, a, kw)))
    yield seen
    ops._packed_decode_shape.cache_clear(); ops._packed_prefill_shape.cache_clear()


def step(new, past, H, G, d, window=0, ws=None, lists=True, scale=0.125, dtype=torch.bfloat16):
    from vlrf_b200.csrc import ops
    T, B = sum(new), len(new)
    t = torch.zeros(B + 1, dtype=torch.int32)
    ws = ws or Workspace("cpu")
    ctx = StepContext(n_tokens=T, tokens=t, tok_slot=t, tok_pos=t, n_seqs=B, seq_slot=t, seq_start=t, seq_pos0=t, max_new=max(new),
                      max_context=max(a + b for a, b in zip(new, past)), logit_rows=t, n_logit_rows=0, act_dtype=dtype, dev_err=t, ws=ws,
                      host_seq_slots=list(range(B)), min_new=min(new))
    if lists:
        ctx.host_seq_lens, ctx.host_seq_pos0 = list(new), list(past)
    rows = torch.empty((T, (H + 2 * G) * d), dtype=dtype)
    out = torch.empty((T, H * d), dtype=dtype)
    ops.attention_packed_step(rows, 0, ops.PackedKV.zeros(1, G, 64, d, "cpu"), t.view(1, -1), out, ctx, H, G, d, scale, window)
    return ws


@pytest.mark.parametrize("new,past,H,G,d,window", [([1000] + [1] * 60, [0] + [400] * 60, 25, 25, 64, 0), ([700] + [1] * 30, [0] + [2000] * 30, 32, 8, 128, 0),
                                                    ([512] + [1] * 63, [7500] + [1000] * 63, 32, 8, 128, 0), ([1000] + [1] * 255, [4000] + [500] * 255, 12, 12, 64, 0),
                                                    ([1000] + [30] * 60, [0] * 61, 25, 25, 64, 0), ([1] * 30 + [512, 2, 2], [900] * 30 + [6000, 10, 10], 32, 8, 128, 3000)])
def test_scratch_of_a_step_is_what_its_tiles_fill(launches, new, past, H, G, d, window):
    """One long prompt among many sequences: parts of a tile meet in scratch, and only tiles that are dealt to several CTAs have any."""
    ws = step(new, past, H, G, d, window)
    assert any(name == "attention_prefill_packed" for name, _, _ in launches)
    assert ws.bytes() <= 30e6


@pytest.mark.parametrize("new,past,H,G,d", [([70, 3], [0, 10], 4, 4, 64), ([512], [7500], 32, 8, 128), ([300] + [1] * 40, [100] + [900] * 40, 25, 25, 64), ([2, 1], [0, 0], 2, 2, 96)])
def test_a_step_whose_lengths_the_host_does_not_know(launches, new, past, H, G, d):
    """The lists are there for plans; without them a step runs all the same, planned from what its context says."""
    step(new, past, H, G, d, lists=False)
    assert launches and launches[0][0] == ("attention_prefill_packed" if d in (64, 128) else "attention_packed")


@pytest.mark.parametrize("dim", [16, 64, 80, 128, 192, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale", [0.125, -1.0])
def test_the_kernels_that_a_layer_names_are_those_that_its_steps_launch(launches, dim, dtype, scale):
    from vlrf_b200.csrc import ops
    from vlrf_b200.engine.model import DecoderModel
    from vlrf_b200.parts.mixer import CausalSelfAttention
    H, G = 6, 3
    mixer = CausalSelfAttention(torch.zeros((H + 2 * G) * dim, 1), None, torch.zeros(1, H * dim), None, n_heads=H, n_kv_heads=G, head_dim=dim, scale=scale)
    model = object.__new__(DecoderModel)
    model.act_dtype, model.layers = dtype, [type("Layer", (), dict(mixer=mixer))(), object()]
    (layer, name, kinds), = model.describe_kernels(kv_bits=4)
    assert (layer, name) == (0, "CausalSelfAttention")
    for kind, new, past in (("prompt", [70, 3], [0, 10]), ("decode", [1, 1], [9, 700])):
        launches.clear()
        step(new, past, H, G, dim, scale=scale, dtype=dtype)
        assert [n for n, _, _ in launches] == [{"tcgen05": "attention_prefill_packed", "mma.sync": "attention_decode_packed", "CUDA cores": "attention_packed"}[kinds[kind]]]


def test_a_layer_off_the_tensor_cores_is_said_of_the_cache_that_it_has(capsys, monkeypatch):
    """Heads of 192: decode over 4 bits is on the tensor cores, prompts are not; the plain cache's kernels are not spoken of."""
    from vlrf_b200 import log
    from vlrf_b200.engine.loading import say_kernels
    from vlrf_b200.engine.model import DecoderModel
    from vlrf_b200.parts.mixer import CausalSelfAttention
    monkeypatch.setattr(log, "_level", log.LEVELS["warn"])
    model = object.__new__(DecoderModel)
    model.act_dtype = torch.bfloat16
    model.layers = [type("Layer", (), dict(mixer=CausalSelfAttention(torch.zeros(3 * 192, 1), None, torch.zeros(1, 192), None, n_heads=1, n_kv_heads=1, head_dim=192,
                                                                     scale=0.1)))() for _ in range(2)]
    say_kernels(model, 4)
    said = capsys.readouterr().err
    assert "layers 0…1 (CausalSelfAttention): prompt attention on CUDA cores, decode attention on mma.sync, keys and values in 4 bits" in said


@pytest.mark.parametrize("lists", [True, False])
@pytest.mark.parametrize("new", [[0, 0], [0]])
def test_a_step_that_brings_nothing(launches, new, lists):
    step(new, [5] * len(new), 4, 2, 64, lists=lists)
    assert [name for name, _, _ in launches] in ([], ["attention_packed"])


def test_scratch_for_a_number_of_tiles_that_is_none():
    import ctypes
    from vlrf_b200.csrc import library
    lib = library()
    p = [ctypes.c_void_p(4096)] * 4
    for groups, n_parts, places in ((1, 1, -1), (2, 2, -5), (0, 1, 0), (3, 1, 0)):
        assert lib.vlrf_attn_packed_prefill_places(p[0], 512, 0, *p, 10, p[0], 4, *p, 256, 210, 3, 70, 4, 2, 64, 64, 0.125, 0, 1, groups, n_parts, 1, places, p[0], p[0],
                                                   p[0], None) != 0
        assert b"attn_packed_prefill" in lib.vlrf_last_error()


@pytest.mark.parametrize("heads,tokens", [(0, 64), (2, 0)])
def test_a_cache_without_heads_or_tokens_is_refused(heads, tokens):
    from vlrf_b200.csrc import KernelError, ops
    with pytest.raises(KernelError):
        ops.PackedKV.zeros(3, heads, tokens, 64, "cpu")


@pytest.mark.parametrize("entry", [1, 2, 3, -1, 99, (2, 1), (7, 0)])
def test_reading_back_an_entry_that_is_not_there(entry):
    from vlrf_b200.cache import KVNeed, SequenceCache, StateNeed
    from vlrf_b200.engine.step import Engine, StepError
    eng = object.__new__(Engine)
    eng.cache = SequenceCache([KVNeed(3, 64), None, (KVNeed(2, 32), StateNeed((4,)))], max_tokens=128, max_seq_len=128, dtype=torch.bfloat16, device="cpu", kv_bits=4)
    slot = eng.start_sequence()
    with pytest.raises(StepError, match="cache entry"):
        eng.keys_values(slot, entry)


def test_every_tile_that_parts_share_has_a_place():
    """Against the tiles one by one: those that reach more than part_blocks blocks are dealt; without a window nothing else has a place."""
    from vlrf_b200.csrc import ops
    rng = random.Random(5)
    for _ in range(400):
        n = rng.randint(1, 6)
        new, past = [rng.choice([0, 1, 2, rng.randint(1, 700)]) for _ in range(n)], [rng.choice([0, rng.randint(0, 3000)]) for _ in range(n)]
        groups, each, window = rng.choice([1, 2]), rng.randint(1, 30), rng.choice([0, 0, rng.randint(1, 2500)])
        dealt, rows = 0, 128 * groups
        for a, b in zip(new, past):
            for t in range(0, a, rows):
                first = max(0, b + t - window + 1) if window > 0 else 0
                dealt += (b + min(t + rows, a) - 1) // 64 - first // 64 + 1 > each
        places = ops.packed_prefill_places(new, past, groups, 2, each, window)
        assert places == dealt if window == 0 else places >= dealt
        assert ops.packed_prefill_places(new, past, groups, 1, each, window) == 0


#: us of the prompt kernel, measured on 148 SMs: new tokens, those before them, heads, head size, window, {(groups, parts, blocks a part): time}
MEASURED = [
    ([1024, 1024], [0, 0], 12, 64, 0, {(1, 1, 16): 28.4, (1, 2, 8): 27.3, (1, 2, 12): 28.5, (1, 3, 6): 35.9, (2, 1, 16): 26.1, (2, 2, 8): 22.1, (2, 2, 12): 22.1, (2, 3, 6): 34.4}),
    ([512], [7500], 32, 128, 0, {(2, 1, 126): 204.8, (2, 2, 63): 119.7, (2, 2, 95): 119.5, (2, 3, 42): 163.8, (2, 4, 32): 135.9, (2, 8, 16): 166.3, (2, 16, 8): 226.4}),
    ([1, 17, 300, 640, 1], [900, 0, 129, 384, 77], 25, 64, 256, {(1, 1, 7): 24.0, (2, 1, 8): 33.4, (2, 2, 6): 39.8}),
    ([200], [0], 12, 64, 0, {(1, 1, 4): 10.9, (2, 1, 4): 11.5}),
    ([1000], [0], 25, 64, 0, {(1, 1, 16): 28.8, (1, 2, 8): 29.1, (1, 2, 12): 28.1, (1, 3, 6): 36.0, (2, 1, 16): 25.8, (2, 2, 8): 29.5, (2, 2, 12): 22.0, (2, 3, 6): 34.1}),
    ([1000] * 4, [0] * 4, 25, 64, 0, {(1, 1, 16): 66.4, (1, 2, 8): 93.6, (1, 2, 12): 84.1, (1, 3, 6): 103.7, (2, 1, 16): 59.8, (2, 2, 8): 84.6, (2, 2, 12): 72.7, (2, 3, 6): 97.4}),
    ([1000] * 4, [4000] * 4, 12, 64, 0, {(1, 1, 79): 243.7, (1, 2, 40): 212.7, (1, 2, 60): 212.8, (1, 3, 27): 214.0, (1, 4, 20): 227.9, (1, 8, 10): 275.5, (2, 1, 79): 182.3, (2, 2, 40): 166.5, (2, 2, 60): 166.5, (2, 3, 27): 167.6, (2, 4, 20): 189.9, (2, 8, 10): 244.4}),
    ([1000] * 4, [0] * 4, 32, 128, 0, {(2, 1, 16): 106.2, (2, 2, 8): 151.2, (2, 2, 12): 128.2, (2, 3, 6): 178.1}),
    ([17], [6000], 12, 64, 0, {(1, 1, 95): 122.1, (1, 2, 48): 70.1, (1, 2, 72): 69.9, (1, 3, 32): 51.4, (1, 4, 24): 41.1, (1, 8, 12): 29.2, (1, 16, 6): 30.4, (2, 1, 95): 92.8, (2, 2, 48): 54.9, (2, 2, 72): 55.2, (2, 3, 32): 41.9, (2, 4, 24): 34.5, (2, 8, 12): 26.3, (2, 12, 8): 26.5, (2, 16, 6): 37.7}),
    ([400, 30, 90], [1000, 3000, 0], 28, 128, 0, {(2, 1, 48): 74.8, (2, 2, 24): 55.3, (2, 2, 36): 55.2, (2, 3, 16): 72.1, (2, 4, 12): 71.8, (2, 8, 6): 97.9}),
    ([1000, 600], [5000, 300], 12, 64, 300, {(1, 1, 8): 26.0, (1, 2, 6): 30.9, (2, 1, 10): 23.9, (2, 2, 8): 34.6}),
    ([2, 2], [50, 900], 8, 128, 0, {(2, 1, 15): 28.6, (2, 2, 8): 25.7, (2, 2, 12): 25.7}),
    ([256], [640], 12, 64, 0, {(1, 1, 14): 23.8, (1, 2, 7): 18.8, (1, 2, 11): 18.9, (2, 1, 14): 23.2, (2, 2, 7): 20.3, (2, 2, 11): 20.4}),
    ([64], [2000], 32, 128, 0, {(2, 1, 33): 53.6, (2, 2, 17): 38.1, (2, 2, 25): 37.9, (2, 3, 11): 32.5, (2, 4, 9): 31.1}),
    ([2000], [0], 8, 128, 0, {(2, 1, 32): 59.2, (2, 2, 16): 42.0, (2, 2, 24): 47.7, (2, 3, 11): 36.7, (2, 4, 8): 51.3}),
    ([700], [100], 32, 128, 0, {(2, 1, 13): 31.4, (2, 2, 7): 44.8, (2, 2, 10): 30.1}),
    ([100] * 8, [0, 50, 100, 150, 200, 250, 300, 350], 12, 64, 0, {(1, 1, 8): 15.7, (1, 2, 6): 20.0, (2, 1, 8): 14.3, (2, 2, 6): 17.8}),
]


@pytest.mark.parametrize("lens,pos0,heads,dim,window,times", MEASURED)
def test_the_shape_of_a_prompt_step_is_the_fastest_or_within_a_tenth_of_it(monkeypatch, lens, pos0, heads, dim, window, times):
    from vlrf_b200.csrc import ops
    monkeypatch.setattr(ops, "_SM_COUNT", 148)
    ops._packed_prefill_shape.cache_clear()
    shape = ops.packed_prefill_shape(lens, pos0, heads, dim, window)
    ops._packed_prefill_shape.cache_clear()
    assert times[shape] <= 1.1 * min(times.values())


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 3, 64), (4, 2, 128)])
@pytest.mark.parametrize("new,past", [([300, 1, 64], [77, 700, 0]), ([1] * 33 + [270, 3, 130] + [1] * 4, list(range(40))), ([2, 0, 513], [900, 50, 200]),
                                      ([1, 400, 90] * 12, [7, 300, 0] * 12)])
@pytest.mark.parametrize("window", [0, 90, 400])
@pytest.mark.parametrize("groups,n_parts,part_blocks,short", [(1, 3, 2, 0), (1, 3, 2, 1), (2, 16, 1, 0), (2, 2, 5, 0), (2, 2, 5, 100)])
def test_prompt_attention_with_scratch_for_the_tiles_that_are_dealt(heads, kv_heads, dim, new, past, window, groups, n_parts, part_blocks, short):
    """Scratch of exactly the size, and of less: tiles without a place are not dealt, and nothing lies outside it."""
    from test_packed_kv_kernels import DEV, Pages, check_prompt
    from vlrf_b200.csrc import ops
    pages = Pages([a + b for a, b in zip(new, past)], kv_heads, dim, seed=heads + sum(new))
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)   # noqa: E731
    start = [sum(new[:i]) for i in range(len(new) + 1)]
    places = max(0, ops.packed_prefill_places(new, past, groups, n_parts, part_blocks, window) - short)
    floats, counts = ops.packed_prefill_scratch(len(new), max(new), heads, dim, groups, n_parts, places)
    partials, counters = torch.full((floats + 1024,), 77.0, device=DEV), torch.full((counts + 64,), 5, dtype=torch.int32, device=DEV)
    counters[:counts] = 0

    def fn(qkv, q_off, table, slot, pos, out, scale, e):
        ops.attention_prefill_packed(qkv, q_off, pages.cache, table, ints(list(range(len(new)))), ints(start), ints(past), out, sum(new), len(new), max(new), heads,
                                     kv_heads, dim, scale, window, e, groups, n_parts, part_blocks, partials, counters, n_places=places)
        assert not bool(counters[:counts].any()) and bool((counters[counts:] == 5).all()) and bool((partials[floats:] == 77).all())
        if places and window == 0 and not short:
            assert bool((partials[:floats] != 77).any())
    check_prompt(fn, pages, new, heads, kv_heads, dim, window)


@pytest.mark.gpu
@pytest.mark.parametrize("new,past,H,G,d", [([70, 3], [0, 10], 4, 4, 64), ([300, 1, 9], [1500, 900, 0], 8, 2, 128), ([1, 1, 1], [5, 700, 64], 4, 2, 128), ([40] + [1] * 30, [0] + [900] * 30, 25, 25, 64)])
def test_lengths_that_the_host_does_not_know_change_the_plan_alone(new, past, H, G, d):
    """Two plans of a step are apart by their roundings.  The decode kernel's weights times steps: 2^-8 of 15 steps, twice the values' largest at most; the prompt
    kernel's operands: less; every result: 2^-8 of the largest.  So by 6 times 2^-8 of it (scores in float32, or of float16 operands, move weights by less)."""
    from test_packed_kv_uses import DEV, HALF_STEP, cache_for, qkv_rows, run_step, step_of
    from vlrf_b200.csrc import ops
    cache, table = cache_for(2000, G, d, len(new))
    whole = [qkv_rows(a + b, H, G, d, seed=i) for i, (a, b) in enumerate(zip(new, past))]
    for i, b in enumerate(past):
        if b:
            ctx = step_of([b], [0], slots=[i])
            ops.kv_append_packed(whole[i][:b].to(DEV), H * d, (H + G) * d, cache, table, ctx.tok_slot, ctx.tok_pos, b, G, d, ctx.dev_err)
    rows = torch.cat([w[b:] for w, b in zip(whole, past)]).to(DEV)
    outs = []
    for known in (True, False):
        ctx = step_of(new, past)
        if not known:
            ctx.host_seq_lens, ctx.host_seq_pos0 = [], []
        outs.append(torch.full((sum(new), H * d), 3.0, dtype=torch.bfloat16, device=DEV))
        run_step(cache, table, rows, outs[-1], ctx, H, G, d)
        assert int(ctx.dev_err.item()) == 0
    largest = max(float(w[:, (H + G) * d:].abs().max()) for w in whole)
    assert float((outs[0].float() - outs[1].float()).abs().max()) <= 6 * HALF_STEP * largest


@pytest.mark.gpu
def test_steps_of_one_size_behind_short_and_long_contexts_captured_and_replayed(tmp_path):
    """256 tokens behind 256 (tiles taken whole) and behind 640 (dealt to parts that meet in scratch), 40 beside single tokens of short and long contexts, each
    several times in an engine that replays what it has seen: the same bits as without replaying, and the counters of the parts are left zero."""
    from conftest import random_ids
    from test_engine import GPT2_WIDE
    from vlrf_b200.engine import Engine, StepEntry, load_model
    from vlrf_b200.weights import write_random_model
    d = write_random_model(dict(GPT2_WIDE, vocab_size=1003, bos_token_id=1, eos_token_id=2), 79, tmp_path / "small")
    ids, runs = [random_ids(1003, 1024, 600 + i) for i in range(9)], []
    for capture in (True, False):
        eng = Engine(load_model(d, "bfloat16"), max_tokens=9 * 1024, kv_cache="int4")
        eng.capture_repeated_steps = capture
        logits = []
        for past in (256, 256, 640, 256, 640, 640, 256, 700, 300):
            slot = eng.start_sequence()
            eng.step([StepEntry(slot, ids[0][:past], [])])
            logits.append(eng.step([StepEntry(slot, ids[0][past:past + 256], [0, 200, 255])]).clone())
            eng.end_sequence(slot)
        for past in (9, 9, 900, 9, 900, 900, 9):
            slots = [eng.start_sequence() for _ in ids]
            eng.step([StepEntry(s, x[:past], []) for s, x in zip(slots[1:], ids[1:])])
            logits.append(eng.step([StepEntry(slots[0], ids[0][:40], [0, 39])] + [StepEntry(s, x[past:past + 1], [0]) for s, x in zip(slots[1:], ids[1:])]).clone())
            for s in slots:
                eng.end_sequence(s)
        eng.check_device_errors()
        assert not bool(eng.ws._bufs["packed_counters"].any())
        assert (len(eng._graphs) >= 4) == capture
        runs.append(logits)
    assert all(torch.equal(a, b) for a, b in zip(*runs))
