"""The operators over a paged cache of keys and values in 4 bits, and what they are measured on.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) the tensors that a user's program has in hand before the call
    run(state)          one pass through an operator: its plain form, or (`own`) the framework's kernels
    work(case)          the bytes and operations that a pass cannot do without
    exact(case, seed)   what `run` returns, from the definition in 64 bits

A row of keys (or values) of one token and head is cut into groups of 64 entries.  A group is held as
    zero = its least entry, rounded to bfloat16
    step = (its largest entry − zero) / 15, rounded to bfloat16
    code = (entry − zero) / step, rounded to a whole number from 0 to 15 (0 where step = 0)
and an entry read back is zero + step · code.  The codes of entries 2c and 2c + 1 are the low and the high half of byte c.  A cache
is paged: blocks of 64 tokens, [block][head][token], found through a table [slot][block index].

A case has a `kind`:

  append   the keys and values of a step's new tokens are quantised into the cache, and read back from it
  read     tokens' keys and values as plain rows
  decode   attention of one query a sequence over its whole context
  prompt   causal attention of every sequence's new tokens over its context, themselves included
"""
from __future__ import annotations

import math

import torch

own = False                    # set from outside: the framework's kernels instead of the plain forms
DEVICE = "cuda"
BLOCK, GROUP = 64, 64


# ---- the cases --------------------------------------------------------------------------------------------------------

def listed() -> list:
    return [
        # one token of GPT-2 small's heads: the smallest call, all latency
        dict(name="append one token", kind="append", dtype="bfloat16", heads=12, kv_heads=12, dim=64, new="1", past="515"),
        # prompts of unequal lengths on GPT-2 XL's heads, some continuing inside a block
        dict(name="append prompts", kind="append", dtype="bfloat16", heads=25, kv_heads=25, dim=64, new="1024,1013,517,64,1",
             past="0,0,333,64,1000"),
        # 32-bit activations, shared heads of 128
        dict(name="append float32", kind="append", dtype="float32", heads=32, kv_heads=8, dim=128, new="777,400", past="0,31"),
        # a long history, handed over as bfloat16
        dict(name="read a history", kind="read", dtype="bfloat16", heads=32, kv_heads=8, dim=128, new="8191", past="0"),
        # a few sequences of odd lengths in 32 bits
        dict(name="read float32", kind="read", dtype="float32", heads=12, kv_heads=12, dim=64, new="700,311,65,1,129,1000",
             past="0,5,64,0,63,17"),
        # one user answering: launches and latencies
        dict(name="decode one row", kind="decode", dtype="bfloat16", heads=12, kv_heads=12, dim=64, past="700", window=0),
        # a full server of GPT-2 XL: the cache is the traffic
        dict(name="decode 32 rows", kind="decode", dtype="bfloat16", heads=25, kv_heads=25, dim=64,
             past=",".join(str(300 + 23 * i) for i in range(32)), window=0),
        # shared heads of 128, contexts of thousands
        dict(name="decode shared heads", kind="decode", dtype="bfloat16", heads=32, kv_heads=8, dim=128,
             past=",".join(str(1 + 541 * i) for i in range(16)), window=0),
        # one very long context: the work has to be split
        dict(name="decode one long row", kind="decode", dtype="bfloat16", heads=32, kv_heads=8, dim=128, past="131070", window=0),
        # two whole prompts of the longest length GPT-2 takes
        dict(name="prompt two", kind="prompt", dtype="bfloat16", heads=12, kv_heads=12, dim=64, new="1024,1024", past="0,0", window=0),
        # a piece of a long prompt on shared heads of 128
        dict(name="prompt piece", kind="prompt", dtype="bfloat16", heads=32, kv_heads=8, dim=128, new="512", past="7500", window=0),
        # prompts that join sequences in the middle of their answers, with a window
        dict(name="prompt mixed", kind="prompt", dtype="bfloat16", heads=25, kv_heads=25, dim=64, new="1,17,300,640,1",
             past="900,0,129,384,77", window=256),
    ]


def _spread(rng, low: int, high: int) -> int:
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng) -> dict:
    kind = rng.choice(["append", "read", "decode", "decode", "prompt", "prompt"])
    dim = rng.choice([64, 64, 128])
    kv_heads = rng.choice([1, 4, 8, 12, 20, 25]) if dim == 64 else rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 7])
    case = dict(kind=kind, dtype="bfloat16", heads=heads, kv_heads=kv_heads, dim=dim)
    text = lambda values: ",".join(str(v) for v in values)   # noqa: E731
    if kind in ("append", "read"):
        n = rng.randint(1, 6)
        most = max(1, 2_500_000 // (kv_heads * dim * n))
        case.update(dtype=rng.choice(["bfloat16", "float32"]), new=text(_spread(rng, 1, most) for _ in range(n)),
                    past=text(rng.choice([0, _spread(rng, 1, 1000)]) for _ in range(n)))
    elif kind == "decode":
        rows = _spread(rng, 1, 64)
        most = max(2, min(100_000, 60_000_000 // (kv_heads * dim * rows)))
        longest = _spread(rng, 2, most)
        case.update(past=text(rng.randint(longest // 3, longest - 1) for _ in range(rows)), window=rng.choice([0, 0, 0, _spread(rng, 1, 2000)]))
    else:
        n = rng.randint(1, 4)
        new = [_spread(rng, 1, 1000) for _ in range(n)]
        past = [rng.choice([0, _spread(rng, 1, 6000)]) for _ in range(n)]
        new[0] = max(new[0], 2)
        while sum(a * (a + b) for a, b in zip(new, past)) * heads * dim > 8_000_000_000:
            new, past = [max(2, a // 2) for a in new], [b // 2 for b in past]
        case.update(new=text(new), past=text(past), window=rng.choice([0, 0, 0, _spread(rng, 1, 1500)]))
    return case


def _numbers(text: str) -> list:
    return [int(v) for v in text.split(",")]


def _lengths(case) -> tuple:
    """(new tokens, tokens before them) of every sequence."""
    past = _numbers(case["past"])
    return (_numbers(case["new"]) if "new" in case else [1] * len(past)), past


def _pairs(new: list, past: list, window: int) -> int:
    """How many (query, visible key) pairs a step has."""
    total = 0
    for a, b in zip(new, past):
        if window <= 0 or b + a <= window:
            total += a * b + a * (a + 1) // 2
        else:
            total += sum(min(b + i + 1, window) for i in range(a))
    return total


def work(case) -> dict:
    new, past = _lengths(case)
    T, H, G, d = sum(new), case["heads"], case["kv_heads"], case["dim"]
    size = 4 if case["dtype"] == "float32" else 2
    held = G * (d + 8 * (d // GROUP))                            # bytes of a token's keys and values in the cache
    if case["kind"] == "append":
        return {"bytes": T * (2 * G * d * size + held + 2 * G * d * 4), "flops": T * 2 * G * d * 6}
    if case["kind"] == "read":
        return {"bytes": T * (held + 2 * G * d * size), "flops": T * 2 * G * d * 2}
    window = case["window"]
    seen = sum(min(a + b, a + window - 1) if window > 0 else a + b for a, b in zip(new, past))
    return {"bytes": seen * held + 2 * T * H * d * size, "flops": 4 * H * d * _pairs(new, past, window)}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _inputs(case, seed: int) -> dict:
    """Everything that the seed decides, plain tensors on the GPU."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    new, past = _lengths(case)
    H, G, d = case["heads"], case["kv_heads"], case["dim"]
    dtype = getattr(torch, case["dtype"])
    T, B = sum(new), len(new)
    need = [-(-(a + b) // BLOCK) for a, b in zip(new, past)]
    n_blocks = sum(need) + 3
    order = torch.randperm(n_blocks, generator=gen, device=DEVICE)
    table = torch.full((B, max(need)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n].int()
        at += n
    # keys have channels with offsets of their own and a few large ones, as caches have
    offset = torch.randn((G, 1, d), generator=gen, device=DEVICE) * 0.7
    spread = 1.0 + 3.0 * (torch.rand((G, 1, d), generator=gen, device=DEVICE) < 0.03)
    state = dict(new=new, past=past, table=table, n_blocks=n_blocks)
    if case["kind"] == "append":
        q = torch.randn((T, H * d), generator=gen, device=DEVICE)
        k = (torch.randn((T, G, d), generator=gen, device=DEVICE) * spread[:, 0] + offset[:, 0]).reshape(T, G * d)
        v = torch.randn((T, G * d), generator=gen, device=DEVICE) * 0.6
        state["rows"] = torch.cat([q, k, v], dim=1).to(dtype)
        return state
    for name, scale, shift in (("k", spread, offset), ("v", 0.6, 0.0)):
        x = torch.randn((n_blocks, G, BLOCK, d), generator=gen, device=DEVICE) * scale + shift
        lo, hi = [f(x.view(n_blocks, G, BLOCK, d // GROUP, GROUP), -1) for f in (torch.amin, torch.amax)]
        zero = lo.bfloat16()
        step = ((hi - zero.float()) / 15.0).bfloat16()
        code = ((x.view(n_blocks, G, BLOCK, d // GROUP, GROUP) - zero.float()[..., None]) / step.float()[..., None]).round_().clamp_(0, 15)
        code = code.to(torch.uint8).view(n_blocks, G, BLOCK, d // 2, 2)
        state[name] = code[..., 0] | (code[..., 1] << 4)
        state[name + "_pairs"] = torch.stack([step, zero], dim=-1)
        del x, code
    if case["kind"] != "read":
        state["rows"] = (torch.randn((T, (H + 2 * G) * d), generator=gen, device=DEVICE) * 1.6).to(dtype)
    return state


def prepare(case, seed: int) -> dict:
    state = dict(_inputs(case, seed), case=case)
    if not own:
        return state
    from vlrf_b200.csrc import ops
    from vlrf_b200.parts.context import StepContext, Workspace
    new, past, H, G, d = state["new"], state["past"], case["heads"], case["kv_heads"], case["dim"]
    dtype = getattr(torch, case["dtype"])
    T, B = sum(new), len(new)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device=DEVICE)   # noqa: E731
    start = [0]
    for a in new:
        start.append(start[-1] + a)
    tok_slot = ints([i for i, a in enumerate(new) for _ in range(a)])
    tok_pos = ints([b + j for a, b in zip(new, past) for j in range(a)])
    dev_err = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    if case["kind"] == "append":
        state["cache"] = ops.PackedKV.zeros(state["n_blocks"], G, BLOCK, d, DEVICE)
    else:
        state["cache"] = ops.PackedKV(state["k"], state["k_pairs"], state["v"], state["v_pairs"])
    if case["kind"] in ("append", "read"):
        out_dtype = torch.float32 if case["kind"] == "append" else dtype
        state["out"] = [torch.empty((T, G * d), dtype=out_dtype, device=DEVICE) for _ in range(2)]
    else:
        state["out"] = torch.empty((T, H * d), dtype=dtype, device=DEVICE)
    state["ctx"] = StepContext(n_tokens=T, tokens=tok_slot, tok_slot=tok_slot, tok_pos=tok_pos, n_seqs=B, seq_slot=ints(list(range(B))),
                               seq_start=ints(start), seq_pos0=ints(past), max_new=max(new), max_context=max(a + b for a, b in zip(new, past)),
                               logit_rows=tok_slot, n_logit_rows=0, act_dtype=dtype, dev_err=dev_err, ws=Workspace(DEVICE),
                               host_seq_slots=list(range(B)), host_seq_lens=new, host_seq_pos0=past, min_new=min(new))
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    from vlrf_b200.csrc import ops
    case, ctx, cache = state["case"], state["ctx"], state["cache"]
    H, G, d, out = case["heads"], case["kv_heads"], case["dim"], state["out"]
    if case["kind"] == "append":
        ops.kv_append_packed(state["rows"], H * d, (H + G) * d, cache, state["table"], ctx.tok_slot, ctx.tok_pos, ctx.n_tokens, G, d, ctx.dev_err)
    if case["kind"] in ("append", "read"):
        ops.kv_read_packed(cache, state["table"], ctx.tok_slot, ctx.tok_pos, out[0], out[1], ctx.n_tokens, ctx.dev_err)
        return out
    ops.attention_packed_step(state["rows"], 0, cache, state["table"], out, ctx, H, G, d, 1.0 / math.sqrt(d), case["window"])
    return out


def _to_bfloat16(x):
    """float64 numbers rounded once to bfloat16's eight bits (a cast goes through float32 and may round twice)."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 256.0), e - 8)


def _quantised(x):
    """What a cache in 4 bits stands for in place of the rows x [T, heads · dim] (float64 from the borders on)."""
    g = x.double().view(x.shape[0], -1, GROUP)
    zero = _to_bfloat16(g.amin(-1, keepdim=True))
    step = _to_bfloat16((g.amax(-1, keepdim=True) - zero) / 15.0)
    code = torch.where(step > 0, (g - zero) / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(g)).round().clamp(0, 15)
    return (zero + step * code).view(x.shape)


def _values(codes, pairs):
    """float32 [..., dim] from codes [..., dim / 2] and (step, zero) [..., dim / 64, 2]."""
    code = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).float()
    code = code.view(*code.shape[:-1], -1, GROUP)
    pairs = pairs.float()
    return (pairs[..., 1:] + pairs[..., :1] * code).flatten(-2)


def _context(state, name: str, i: int, first: int, last: int):
    """The values of sequence i's tokens first … last − 1: float32 [heads, tokens, dim]."""
    b0, b1 = first // BLOCK, -(-last // BLOCK)
    blocks = state["table"][i, b0:b1].long()
    x = _values(state[name][blocks], state[name + "_pairs"][blocks])
    return x.transpose(0, 1).flatten(1, 2)[:, first - b0 * BLOCK:last - b0 * BLOCK]


def _run_plain(state):
    case, new, past = state["case"], state["new"], state["past"]
    H, G, d = case["heads"], case["kv_heads"], case["dim"]
    dtype = getattr(torch, case["dtype"])
    if case["kind"] == "append":
        rows = state["rows"]
        return [_quantised(rows[:, at:at + G * d]).float() for at in (H * d, (H + G) * d)]
    if case["kind"] == "read":
        return [torch.cat([_context(state, name, i, b, b + a).transpose(0, 1).reshape(a, G * d) for i, (a, b) in enumerate(zip(new, past))]).to(dtype)
                for name in ("k", "v")]
    out, at, window = [], 0, case["window"]
    for i, (a, b) in enumerate(zip(new, past)):
        first = max(0, b - window + 1) if window > 0 else 0
        k, v = _context(state, "k", i, first, a + b), _context(state, "v", i, first, a + b)
        q = state["rows"][at:at + a, :H * d].float().view(a, G, H // G, d).permute(1, 2, 0, 3).reshape(G, -1, d)
        s = torch.matmul(q, k.transpose(1, 2)).view(G, H // G, a, -1) / math.sqrt(d)
        if a > 1:
            age = torch.arange(b, a + b, device=DEVICE)[:, None] - torch.arange(first, a + b, device=DEVICE)[None, :]
            s = s.masked_fill((age < 0) | (age >= window if window > 0 else age < 0), float("-inf"))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(p.view(G, -1, p.shape[-1]), v).view(G, H // G, a, d) / p.sum(-1, keepdim=True)
        out.append(o.permute(2, 0, 1, 3).reshape(a, H * d).to(dtype))
        at += a
    return torch.cat(out)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed: int):
    inputs = _inputs(case, seed)
    H, G, d = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        rows = inputs["rows"].double()
        return [_nearest_values(rows[:, at:at + G * d]) for at in (H * d, (H + G) * d)]
    new, past = inputs["new"], inputs["past"]
    held = {}
    for name in ("k", "v"):
        raw = inputs[name].to(torch.int16)
        code = torch.empty(raw.shape[:-1] + (d,), dtype=torch.float64, device=DEVICE)
        code[..., 0::2] = (raw % 16).double()
        code[..., 1::2] = (raw // 16).double()
        step, zero = inputs[name + "_pairs"].double().unbind(-1)
        held[name] = code * step.repeat_interleave(GROUP, -1) + zero.repeat_interleave(GROUP, -1)      # [block, head, token, dim]
    outputs = ([], []) if case["kind"] == "read" else []
    at = 0
    for i, (a, b) in enumerate(zip(new, past)):
        place = torch.arange(0, a + b, device=DEVICE)
        blocks = inputs["table"][i].long()[place // BLOCK]
        k, v = [held[name][blocks, :, place % BLOCK] for name in ("k", "v")]                           # [tokens, head, dim]
        if case["kind"] == "read":
            outputs[0].append(k[b:].reshape(a, G * d))
            outputs[1].append(v[b:].reshape(a, G * d))
            continue
        q = inputs["rows"][at:at + a, :H * d].double().view(a, H, d)
        result = torch.empty((a, H, d), dtype=torch.float64, device=DEVICE)
        here = torch.arange(b, a + b, device=DEVICE)
        seen = place[None, :] <= here[:, None]
        if case["window"] > 0:
            seen &= place[None, :] > here[:, None] - case["window"]
        for h in range(H):
            logit = (q[:, h] @ k[:, h // (H // G)].T) * d ** -0.5
            weight = torch.softmax(logit.masked_fill(~seen, -math.inf), dim=1)
            result[:, h] = weight @ v[:, h // (H // G)]
        outputs.append(result.view(a, H * d))
        at += a
    if case["kind"] == "read":
        return [torch.cat(part) for part in outputs]
    return torch.cat(outputs)


def _nearest_eight_bits(x, numerator, divisor: float):
    """The number of eight significant bits nearest numerator / divisor, found from x, an approximation of it, by comparing exact
    products (ties to the even one)."""
    _, e = torch.frexp(x)
    unit = torch.ldexp(torch.ones_like(x), e - 8)
    low = torch.floor(x / unit)
    rest = numerator - divisor * low * unit                     # (products of few bits: exact)
    up = 2.0 * rest - divisor * unit
    return torch.where((up > 0) | ((up == 0) & (low % 2 == 1)), low + 1, low) * unit


def _nearest_values(x):
    T, width = x.shape
    g = x.reshape(T, width // GROUP, GROUP)
    least, most = g.min(-1).values, g.max(-1).values
    zero = _nearest_eight_bits(least, least, 1.0)
    step = _nearest_eight_bits((most - zero) / 15, most - zero, 15.0)
    zero, step = zero[..., None], step[..., None]
    rest = g - zero
    low = torch.floor(rest / step).nan_to_num(0.0, 0.0, 0.0).clamp(0, 15)
    twice = 2.0 * (rest - low * step) - step
    code = torch.where((twice > 0) | ((twice == 0) & (low % 2 == 1)), low + 1, low).clamp(0, 15)
    return (zero + step * code).reshape(T, width)
