"""A cache in 4 bits, what needs no GPU: the plain implementation, and the refusals of the kernel library's entries (all sizes are checked
before anything is launched)."""
import ctypes
from fractions import Fraction

import pytest
import torch

import plain_packed as plain


def test_plain_quantisation_of_known_numbers():
    assert plain.quantise_group([0.0, 15.0, 7.4, 7.5, 8.5, 1.0]) == (1.0, 0.0, [0, 15, 7, 8, 8, 1])          # ties to even
    assert plain.quantise_group([2.0] * 4) == (0.0, 2.0, [0] * 4)
    step, zero, codes = plain.quantise_group([1.0, 1.001953125])       # the least number, and a range below bfloat16's spacing at 1
    assert zero == 1.0 and codes == [0, 15] and step == float(plain._bfloat16(Fraction(1.001953125 - 1.0) / 15))
    assert plain._bfloat16(Fraction(257)) == 256 and plain._bfloat16(Fraction(259)) == 260
    assert all(v != v for v in plain.quantise_group([1.0, float("inf")])[:2])


def test_a_number_read_back_is_within_half_a_step():
    x = torch.randn(20, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    codes, pairs = plain.quantise(x, 64)
    off = (plain.values(codes, pairs).view(20, 2, 64) - x.double().view(20, 2, 64)).abs()
    step = pairs[..., 0].view(20, 2, 1)
    # half a step, and where the step was rounded down, by at most 2^-8 of itself, the last code may lie 15 · 2^-8 of a step further off
    assert bool((off <= step * (0.5 + 15 * 2.0 ** -8)).all())


@pytest.mark.parametrize("dim,group", [(16, 16), (32, 32), (48, 16), (64, 64), (80, 16), (96, 32), (128, 64), (192, 64), (256, 64), (24, 0), (0, 0),
                                       (-64, 0), (272, 0)])
def test_groups(dim, group):
    from vlrf_b200.csrc import library, ops
    assert ops.packed_group(dim) == group and library().vlrf_packed_group(dim) == group
    if group:
        assert plain.group_of(dim) == group


def pointers(n):
    return [ctypes.c_void_p(4096)] * n


@pytest.mark.parametrize("change", [dict(dh=24), dict(dh=512), dict(T=-1), dict(Hkv=0), dict(BT=0), dict(max_blocks=0), dict(dtype=2), dict(dev_err=None),
                                    dict(T=2 ** 30, Hkv=64)])
def test_append_and_read_refuse(change):
    from vlrf_b200.csrc import library
    lib = library()
    a = dict(dict(dtype=0, T=3, Hkv=2, dh=64, BT=64, max_blocks=4, dev_err=ctypes.c_void_p(4096)), **change)
    assert lib.vlrf_packed_append(*pointers(1), a["dtype"], 384, 128, 256, *pointers(4), 10, *pointers(1), a["max_blocks"], *pointers(2), a["T"], a["Hkv"],
                                  a["dh"], a["BT"], a["dev_err"], None) != 0
    assert b"packed_append" in lib.vlrf_last_error()
    assert lib.vlrf_packed_read(*pointers(4), 10, *pointers(1), a["max_blocks"], *pointers(3), 128, *pointers(1), 128, a["dtype"], a["T"], a["Hkv"], a["dh"],
                                a["BT"], a["dev_err"], None) != 0
    assert b"packed_read" in lib.vlrf_last_error()


@pytest.mark.parametrize("change", [dict(dh=24), dict(dh=512), dict(T=-1), dict(H=3), dict(H=0), dict(BT=48), dict(BT=0), dict(max_blocks=0), dict(dtype=2),
                                    dict(window=-1), dict(dev_err=None)])
def test_attention_refuses(change):
    from vlrf_b200.csrc import library
    lib = library()
    a = dict(dict(dtype=0, T=3, H=4, Hkv=2, dh=64, BT=64, max_blocks=4, window=0, dev_err=ctypes.c_void_p(4096)), **change)
    assert lib.vlrf_attn_packed(*pointers(1), a["dtype"], 384, 0, *pointers(4), 10, *pointers(1), a["max_blocks"], *pointers(3), 256, a["T"], a["H"], a["Hkv"],
                                a["dh"], a["BT"], 0.125, a["window"], a["dev_err"], None) != 0
    assert b"attn_packed" in lib.vlrf_last_error()


@pytest.mark.parametrize("change", [dict(dh=32), dict(dh=320), dict(rows=-1), dict(rows=70000), dict(H=3), dict(BT=32), dict(max_blocks=0), dict(window=-1),
                                    dict(dev_err=None), dict(n_split=0), dict(n_split=65), dict(n_split=2), dict(part_tiles=0), dict(ld=385), dict(q_off=4), dict(ld_out=130), dict(qkv=4100)])
def test_decode_attention_refuses(change):
    from vlrf_b200.csrc import library
    lib = library()
    a = dict(dict(rows=3, H=4, Hkv=2, dh=64, BT=64, max_blocks=4, window=0, n_split=1, part_tiles=1, ld=512, q_off=0, ld_out=256, qkv=4096,
                  dev_err=ctypes.c_void_p(4096)), **change)
    assert lib.vlrf_attn_packed_decode(ctypes.c_void_p(a["qkv"]), a["ld"], a["q_off"], *pointers(4), 10, *pointers(1), a["max_blocks"], *pointers(2), None, *pointers(1),
                                       a["ld_out"], a["rows"], a["H"], a["Hkv"], a["dh"], a["BT"], 0.125, a["window"], 0, a["n_split"], a["part_tiles"], None, None, a["dev_err"],
                                       None) != 0
    assert b"attn_packed_decode" in lib.vlrf_last_error()


@pytest.mark.parametrize("change", [dict(dh=32), dict(dh=192), dict(n_seqs=-1), dict(n_seqs=70000), dict(max_new=-1), dict(H=3), dict(BT=32), dict(n_tokens=-1), dict(least_new=0),
                                    dict(max_blocks=0), dict(window=-1), dict(dev_err=None), dict(n_parts=0), dict(n_parts=17), dict(n_parts=2),
                                    dict(groups=0), dict(groups=3), dict(part_blocks=0), dict(scale=-1.0), dict(ld=385), dict(q_off=4), dict(ld_out=130), dict(qkv=4100),
                                    dict(max_new=2 ** 24)])
def test_prompt_attention_refuses(change):
    from vlrf_b200.csrc import library
    lib = library()
    a = dict(dict(n_seqs=3, max_new=70, H=4, Hkv=2, dh=64, BT=64, max_blocks=4, window=0, groups=1, n_parts=1, part_blocks=1, scale=0.125, ld=512, q_off=0, ld_out=256, qkv=4096,
                  dev_err=ctypes.c_void_p(4096)), **change)
    assert lib.vlrf_attn_packed_prefill(ctypes.c_void_p(a["qkv"]), a["ld"], a["q_off"], *pointers(4), 10, *pointers(1), a["max_blocks"], *pointers(4),
                                        a["ld_out"], a.get("n_tokens", abs(a["n_seqs"] * a["max_new"]) % 2 ** 31), a["n_seqs"], a["max_new"], a["H"], a["Hkv"], a["dh"], a["BT"],
                                        a["scale"], a["window"], a.get("least_new", 1), a["groups"],
                                        a["n_parts"], a["part_blocks"], None, None, a["dev_err"], None) != 0
    assert b"attn_packed_prefill" in lib.vlrf_last_error()


def test_no_cpu_path():
    from vlrf_b200.csrc import KernelError, ops
    cache = ops.PackedKV.zeros(3, 2, 64, 64, "cpu")
    assert cache.bytes() == 3 * 2 * 64 * (64 + 8)
    t = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(KernelError):
        ops.kv_append_packed(torch.zeros(4, 384), 128, 256, cache, t.view(1, 4), t, t, 4, 2, 64, t)
    with pytest.raises(KernelError):
        ops.kv_read_packed(cache, t.view(1, 4), t, t, torch.zeros(4, 128), torch.zeros(4, 128), 4, t)
    with pytest.raises(KernelError):
        ops.attention_packed(torch.zeros(4, 384), 0, cache, t.view(1, 4), t, t, torch.zeros(4, 128), 4, 2, 2, 64, 0.125, 0, t)


def test_cache_books_in_4_bits():
    from vlrf_b200.cache import CacheError, KVNeed, LatentNeed, SequenceCache, StateNeed
    c = SequenceCache([KVNeed(3, 64), KVNeed(3, 64), LatentNeed(48), (KVNeed(2, 32, "window", 100), StateNeed((4,))), None], max_tokens=256, max_seq_len=256,
                      dtype=torch.bfloat16, device="cpu", kv_bits=4)
    view = c.view(1)
    assert view.k is None and view.packed.k.shape == (4, 3, 64, 32) and view.packed.k_pairs.shape == (4, 3, 64, 1, 2)
    assert c.view(0).packed.k.data_ptr() != view.packed.k.data_ptr() and c.view(2).rows.dtype == torch.bfloat16
    assert c.view(3).parts[0].packed.head_dim == 32 and c.view(3).parts[1].state.shape == (c.n_slots, 4)
    slot = c.acquire()
    c.reserve(slot, 70)
    c.advance(slot, 70)
    assert c.live_kv_bytes([slot]) == 70 * (2 * 3 * 2 * 36 + 48 * 2 + 2 * 2 * 20)
    assert c.bytes() == 256 * (2 * 3 * 2 * 36 + 48 * 2 + 2 * 2 * 20) + c.n_slots * 4 * 4
    c.release(slot)
    c.check()
    for need, bits in ((KVNeed(3, 64), 8), (KVNeed(3, 24), 4), (KVNeed(3, 64, v_dim=32), 4), (KVNeed(1, 512), 4)):
        with pytest.raises(CacheError):
            SequenceCache([need], max_tokens=64, max_seq_len=64, dtype=torch.bfloat16, device="cpu", kv_bits=bits)


def test_models_say_whether_they_take_4_bits():
    from vlrf_b200.cache import KVNeed
    from vlrf_b200.engine.model import DecoderModel
    from vlrf_b200.parts.mixer import CausalSelfAttention

    class Mixer:
        takes_packed_kv = True

    class Layer:
        def __init__(self, need, mixer):
            self.need, self.mixer = need, mixer

        def cache_need(self):
            return self.need
    model = object.__new__(DecoderModel)
    model.layers = [Layer(KVNeed(1, 64), Mixer()), Layer(None, object())]
    model.check_packed_kv()
    for need in (KVNeed(1, 64), (None, KVNeed(1, 64))):
        model.layers = [Layer(need, object())]
        with pytest.raises(ValueError, match="4 bits"):
            model.check_packed_kv()
    assert CausalSelfAttention.takes_packed_kv


def test_scratch_sizes_are_the_library_s():
    from vlrf_b200.csrc import library, ops
    lib = library()
    floats, ints = ctypes.c_longlong(0), ctypes.c_longlong(0)
    for rows, heads, kv_heads, dim, parts in ((1, 12, 12, 64, 1), (7, 25, 25, 64, 3), (2, 32, 8, 128, 64), (3, 28, 4, 128, 5), (1, 80, 2, 256, 2), (4, 6, 3, 192, 9), (5, 24, 1, 64, 2)):
        assert lib.vlrf_attn_packed_decode_scratch(rows, heads, kv_heads, dim, parts, ctypes.byref(floats), ctypes.byref(ints)) == 0
        assert ops.packed_decode_scratch(rows, heads, kv_heads, dim, parts) == (floats.value, ints.value)
    for seqs, new, heads, dim, groups, parts in ((1, 1, 12, 64, 1, 1), (3, 300, 25, 64, 2, 4), (2, 128, 8, 128, 1, 16), (1, 257, 4, 128, 2, 2)):
        assert lib.vlrf_attn_packed_prefill_scratch(seqs, new, heads, dim, groups, parts, ctypes.byref(floats), ctypes.byref(ints)) == 0
        assert ops.packed_prefill_scratch(seqs, new, heads, dim, groups, parts) == (floats.value, ints.value)
    assert lib.vlrf_attn_packed_decode_scratch(1, 3, 2, 64, 1, ctypes.byref(floats), ctypes.byref(ints)) != 0
    assert lib.vlrf_attn_packed_prefill_scratch(1, 3, 2, 96, 1, 1, ctypes.byref(floats), ctypes.byref(ints)) != 0


def test_shapes_of_steps(monkeypatch):
    """Shapes hold the longest context, are within what the kernels take, and are the measured best (or within a tenth of it) where several were
    measured on 148 SMs."""
    from vlrf_b200.csrc import ops
    monkeypatch.setattr(ops, "_SM_COUNT", 148)
    ops._packed_decode_shape.cache_clear(); ops._packed_prefill_shape.cache_clear()
    for rows in (1, 2, 7, 32, 200, 5000):
        for heads, kv_heads in ((12, 12), (32, 8), (7, 1), (48, 1)):
            for dim in (64, 128, 192, 256):
                for context in (0, 1, 64, 65, 1000, 8192, 200_000):
                    few, parts, each = ops.packed_decode_shape(rows, heads, kv_heads, dim, context)
                    assert few in (0, 1) and 1 <= parts <= 64 and each >= 1 and parts * each * 64 >= context
    assert ops.packed_decode_shape(1, 12, 12, 64, 701)[1] == 1                        # one row of 700 tokens: not cut
    assert ops.packed_decode_shape(32, 25, 25, 64, 1014)[:2] == (0, 1)                # the places are full
    assert ops.packed_decode_shape(1, 32, 8, 128, 131_071)[1] >= 18                   # one long row: cut to fill the GPU
    assert ops.packed_prefill_shape([512], [7500], 32, 128)[:2] == (2, 2)
    assert ops.packed_prefill_shape([200], [0], 12, 64) == (1, 1, 4)
    for lens, pos0, window in (([1], [0], 0), ([1, 5000], [100_000, 0], 0), ([300], [90_000], 100), ([2] * 40, list(range(40)), 1)):
        groups, parts, each = ops.packed_prefill_shape(lens, pos0, 8, 128, window)
        assert groups in (1, 2) and 1 <= parts <= 16 and each >= 1
    ops._packed_decode_shape.cache_clear(); ops._packed_prefill_shape.cache_clear()
