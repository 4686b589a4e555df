"""GPT-2 with its keys and values held in 4 bits: what every layer writes and attends, held against the plain implementation on the
layer's own inputs; pieces of prompts; replayed steps; pages that come and go."""
import math

import pytest
import torch

import plain_packed as plain
from conftest import random_ids
from vlrf_b200.engine.step import StepEntry

pytestmark = pytest.mark.gpu
U, HALF_STEP = 2.0 ** -24, 2.0 ** -8


def make(model_dirs, name, dtype, max_tokens, **kw):
    from vlrf_b200.engine import Engine, load_model
    eng = Engine(load_model(model_dirs[name], dtype), max_tokens=max_tokens, kv_cache="int4", **kw)
    for g in eng.cache._groups:                # whatever is read without having been written shows
        for p in g.packed:
            p.k_pairs.fill_(float("nan")); p.v_pairs.fill_(float("nan"))
    return eng


class Watch:
    """Checks every attention of an engine's steps on its own inputs: the cache holds exactly the quantised keys and values of the step's tokens, and
    the result is attention over what the cache stands for."""

    def __init__(self, monkeypatch, eng):
        from vlrf_b200.parts.mixer import CausalSelfAttention
        self.calls, self.eng = 0, eng
        eng.capture_repeated_steps = False
        inner = CausalSelfAttention._attend

        def attend(mixer, qkv, view, merged, ctx):
            inner(mixer, qkv, view, merged, ctx)
            self.check(mixer, qkv, view, merged, ctx)
        monkeypatch.setattr(CausalSelfAttention, "_attend", attend)

    def check(self, mixer, qkv, view, merged, ctx):
        self.calls += 1
        H, G, d = mixer.n_heads, mixer.n_kv_heads, mixer.head_dim
        rows, got = qkv[:ctx.n_tokens].cpu(), merged[:ctx.n_tokens].double().cpu()
        host = {n: getattr(view.packed, n).cpu() for n in ("k", "k_pairs", "v", "v_pairs")}
        table, t = view.block_table.cpu(), 0
        for slot, a, b in zip(ctx.host_seq_slots, ctx.host_seq_lens, ctx.host_seq_pos0):
            place = torch.arange(a + b)
            blocks = table[slot].long()[place // 64]
            k, v = [plain.unpacked(host[n], host[n + "_pairs"])[blocks, :, place % 64] for n in ("k", "v")]
            for n, at in (("k", mixer.k_off), ("v", mixer.v_off)):
                codes, pairs = plain.quantise(rows[t:t + a, at:at + G * d], d)
                held = host[n][blocks[b:], :, place[b:] % 64]
                assert torch.equal(torch.stack([held & 15, held >> 4], -1).flatten(-2).long(), codes)
                assert torch.equal(host[n + "_pairs"][blocks[b:], :, place[b:] % 64].double(), pairs)
            for j in sorted({0, a - 1} | set(range(0, a, 23))):
                q, p = rows[t + j, :H * d].double().view(H, d), b + j
                want = plain.attend(q, k, v, mixer.scale, mixer.window, p)
                for h in range(H):
                    kk, vv = k[:p + 1, h // (H // G)], v[:p + 1, h // (H // G)]
                    half = HALF_STEP if rows.dtype == torch.bfloat16 else 0.0       # (as in the kernels' tests)
                    # on the tensor cores a decode step's scores are sums of products scaled one by one: Σ |q| (|zero| + 15 step) ≤ 31 Σ |q| max |k|
                    e_k = (half + (d + 16) * U * 31) * mixer.scale * float((kk.abs().amax(0) * q[h].abs()).sum())
                    tol = float(vv.abs().max()) * (math.expm1(2 * e_k) + 2 * half + (p + 33) * U * 31)
                    tol = tol + half * (want[h].abs() + tol)
                    assert bool(((got[t + j].view(H, d)[h] - want[h]).abs() <= tol).all()), (slot, p, h)
            t += a


MODELS = [("tiny_a", [21, 70, 3]), ("tiny_b", [40, 1, 130]), ("tiny_c", [65, 250, 1]), ("tiny_sharp", [130, 64, 2]), ("tiny_d", [33, 100])]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name,lens", MODELS)
def test_every_layer_writes_and_attends_what_it_should(model_dirs, plain_models, monkeypatch, name, lens, dtype):
    """Prompts of unequal lengths in one step, the next tokens one by one, a second piece of a prompt beside single tokens."""
    eng = make(model_dirs, name, dtype, 640)
    vocab, layers = plain_models[name][0]["vocab_size"], plain_models[name][0]["n_layer"]
    watch = Watch(monkeypatch, eng)
    slots = [eng.start_sequence() for _ in lens]
    ids = [random_ids(vocab, n + 20, 3 + i) for i, n in enumerate(lens)]
    at = list(lens)
    eng.step([StepEntry(s, x[:n], [n - 1]) for s, x, n in zip(slots, ids, lens)])
    for _ in range(2):
        eng.step([StepEntry(s, x[n:n + 1], [0]) for s, x, n in zip(slots, ids, at)])
        at = [n + 1 for n in at]
    eng.step([StepEntry(s, x[n:n + (7 if i == 0 else 1)], []) for i, (s, x, n) in enumerate(zip(slots, ids, at))])
    eng.check_device_errors()
    assert watch.calls == 4 * layers
    eng.end_sequence(slots[0])                 # its blocks go to the next one
    slot = eng.start_sequence()
    eng.step([StepEntry(slot, random_ids(vocab, 66, 9), [65])])
    eng.check_device_errors()
    eng.cache.check()


def test_keys_and_values_are_read_back(model_dirs, plain_models):
    from vlrf_b200.engine.step import StepError
    eng = make(model_dirs, "tiny_c", "bfloat16", 320)
    other, slot = eng.start_sequence(), eng.start_sequence()
    eng.step([StepEntry(other, [5] * 70, []), StepEntry(slot, random_ids(777, 100, 1), [])])
    view, place = eng.cache.view(1), torch.arange(30, 100)
    blocks = view.block_table[slot].long().cpu()[place // 64]
    for dtype in (torch.float32, torch.bfloat16, None):
        got = eng.keys_values(slot, 1, 30, 100, dtype)
        for g, n in zip(got, ("k", "v")):
            want = plain.unpacked(getattr(view.packed, n).cpu(), getattr(view.packed, n + "_pairs").cpu())[blocks, :, place % 64].reshape(70, -1)
            assert g.dtype == (dtype or torch.bfloat16) and torch.equal(g.cpu(), want.float().to(g.dtype))
    assert eng.keys_values(slot, 0)[0].shape == (100, 192) and eng.keys_values(slot, 0, 7, 7)[1].shape == (0, 192)
    for bad in ((slot, 0, 5, 101), (slot, 0, -1, 5), (slot, 0, 9, 3), (17, 0, 0, 1)):
        with pytest.raises(StepError):
            eng.keys_values(*bad)
    eng.check_device_errors()


@pytest.mark.parametrize("name", ["tiny_b", "tiny_c"])
def test_replayed_steps_answer_like_plain_ones(model_dirs, plain_models, name):
    """Generation through captured decode steps and prompt steps, twice, against the same without graphs: token for token."""
    from vlrf_b200 import Model, SamplingParams
    vocab = plain_models[name][0]["vocab_size"]
    prompts = [random_ids(vocab, n, n) for n in (40, 3, 70, 12)]
    params = SamplingParams(max_new_tokens=24, do_sample=False)
    answers = []
    for use_graph in (True, False):
        model = Model.load(model_dirs[name], "bfloat16", max_tokens=1024, kv_cache="int4")
        model.backend.use_graph = use_graph
        model.engine.capture_repeated_steps = use_graph
        answers += [[r.new_tokens for r in model.generate_ids(prompts, params)] for _ in range(3)]
        assert model.engine.cache.slots.n_held == 0
    assert all(a == answers[0] for a in answers)


def test_a_prompt_may_come_in_pieces(model_dirs, plain_models):
    """The same tokens whole, in portions and one by one, in 32 bits: the cache holds the same codes but for numbers beside a border, so the logits agree
    as far as a few codes that differ by one let them: within the error that 4 bits make against a cache in 32 bits."""
    from engine_drives import drive_portions, drive_tail_one_by_one, drive_whole
    from vlrf_b200.engine import Engine, load_model
    reqs = [random_ids(777, 150, 4)]
    whole32 = drive_whole(Engine(load_model(model_dirs["tiny_c"], "float32"), max_tokens=320), reqs)[0]
    runs = [drive(make(model_dirs, "tiny_c", "float32", 320), reqs, *a)[0] for drive, a in ((drive_whole, ()), (drive_portions, (41,)), (drive_tail_one_by_one, (32,)))]
    made = float((runs[0] - whole32).abs().max())
    assert 0 < made < 0.25 * float(whole32.abs().max())
    for other in runs[1:]:
        assert float((runs[0] - other).abs().max()) <= made


def test_the_cache_is_smaller_and_models_that_do_not_take_it_are_refused(model_dirs):
    from vlrf_b200 import Model
    from vlrf_b200.config import load_preset
    from vlrf_b200.engine.step import StepError
    plain_model = Model.load(model_dirs["tiny_c"], max_tokens=256)
    model = Model.load(model_dirs["tiny_c"], max_tokens=256, kv_cache="int4")
    assert model.kv_cache_bytes() * 32 == plain_model.kv_cache_bytes() * 9        # 4.5 bits of 16
    logits = model.get_logits([1, 2, 3], all_positions=True)
    assert bool(torch.isfinite(logits).all())
    with pytest.raises(StepError):
        Model.load(model_dirs["tiny_c"], max_tokens=256, kv_cache="q3")
    with pytest.raises(ValueError, match="4 bits"):
        Model.init_random(load_preset("suposun-tiny"), max_tokens=256, kv_cache="int4")
