"""Operators around an 8-bit paged KV cache, as cases to time and compare.

  write      K/V rows are quantised to e4m3 / e5m2 as they go into the paged cache (reshape_and_cache_flash)
  read       sequences are read back from the paged cache as packed rows of 16 or 32 bits (gather_cache_flash)
  attention  flash_attn_varlen_func over a paged cache that is 8-bit, or that is attended with a sliding window and a few
             first tokens that stay visible, or both: single tokens, a few tokens, chunks of new tokens

`run` computes them from elementary torch operations in 32 bits, or through this package where `own` is set.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_FORMATS = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_PAIRS = [(32, 8), (8, 8), (32, 4), (16, 2), (8, 1), (6, 2), (40, 8), (4, 4)]


# ---- cases ---------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decoding step of a batch of sequences: one token each
        dict(name="write a decoding step", op="write", tokens=64, heads=8, dim=128, page=16, dtype="bf16", fmt="e4m3", scales="one"),
        # a batch of prompts, the size of the benchmark's cache writes, a scale for each head
        dict(name="write prompts", op="write", tokens=16384, heads=32, dim=128, page=16, dtype="bf16", fmt="e4m3", scales="head"),
        # the cached part of a few short prompts, for a consumer that wants 16 bits
        dict(name="read short prompts", op="read", batch=3, keys=1000, ragged=7, heads=8, dim=128, page=16, dtype="f16", fmt="e5m2", scales="one"),
        # long cached contexts read back in one piece
        dict(name="read long contexts", op="read", batch=16, keys=8192, ragged=5, heads=8, dim=128, page=32, dtype="bf16", fmt="e4m3", scales="head"),
        # one user, one token, a short context: latency
        dict(name="one token, short", op="attention", batch=1, new=1, keys=513, ragged=0, hq=32, hk=8, dim=128, page=16, dtype="bf16",
             fmt="e4m3", scales="one", window=-1, sinks=0),
        # a decoding step of the benchmark's batch
        dict(name="tokens of a batch", op="attention", batch=64, new=1, keys=4096, ragged=0, hq=32, hk=8, dim=128, page=16, dtype="bf16",
             fmt="e4m3", scales="one", window=-1, sinks=0),
        # few sequences with very long, uneven contexts
        dict(name="tokens, long contexts", op="attention", batch=3, new=1, keys=131072, ragged=11, hq=32, hk=8, dim=128, page=64, dtype="bf16",
             fmt="e4m3", scales="seq", window=-1, sinks=0),
        # a few proposed tokens a sequence are checked at once
        dict(name="a few tokens each", op="attention", batch=16, new=5, keys=2047, ragged=3, hq=16, hk=4, dim=64, page=16, dtype="f16",
             fmt="e5m2", scales="head", window=-1, sinks=0),
        # chunks of long prompts over what is cached of them
        dict(name="chunks over a cache", op="attention", batch=4, new=1024, keys=8192, ragged=9, hq=32, hk=8, dim=128, page=16, dtype="bf16",
             fmt="e4m3", scales="one", window=-1, sinks=0),
        # streaming generation: 16-bit cache, a window and four first tokens
        dict(name="sinks, tokens", op="attention", batch=32, new=1, keys=32768, ragged=13, hq=32, hk=8, dim=128, page=16, dtype="bf16",
             fmt="same", scales="one", window=4095, sinks=4),
        # a prompt under the same mask
        dict(name="sinks, a prompt", op="attention", batch=1, new=8192, keys=8192, ragged=0, hq=32, hk=8, dim=128, page=16, dtype="bf16",
             fmt="same", scales="one", window=1023, sinks=4),
        # the same mask over an 8-bit cache, odd lengths
        dict(name="sinks, chunks, 8 bits", op="attention", batch=5, new=333, keys=5001, ragged=17, hq=8, hk=2, dim=64, page=32, dtype="f16",
             fmt="e4m3", scales="head", window=700, sinks=5),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of these ranges, at most as costly as the largest listed ones."""
    op = rng.choice(["write", "read", "attention", "attention", "attention", "attention"])
    c = dict(op=op, dim=rng.choice([64, 128, 128, 80, 96, 256]), page=rng.choice([16, 16, 32, 64, 48, 256]), dtype=rng.choice(["bf16", "bf16", "f16"]),
             fmt=rng.choice(["e4m3", "e4m3", "e5m2"]), scales=rng.choice(["one", "head"]))
    if op == "write":
        return dict(c, tokens=_log_int(rng, 1, 16384), heads=rng.choice([1, 2, 3, 4, 8, 16, 32]) * 128 // max(c["dim"], 128),
                    dtype=rng.choice(["bf16", "f16", "f32"])) if c["dim"] <= 128 else dict(c, tokens=_log_int(rng, 1, 8000), heads=rng.choice([1, 2, 4, 8]))
    if op == "read":
        return dict(c, batch=_log_int(rng, 1, 16), keys=_log_int(rng, 1, 8192), ragged=rng.randint(1, 1 << 20), heads=rng.choice([1, 2, 4, 8]),
                    dim=min(c["dim"], 128), fmt=rng.choice(["e4m3", "e5m2", "same"]))
    c["hq"], c["hk"] = rng.choice(_PAIRS)
    kind = rng.choice(["token", "token", "few", "chunk"])
    c.update(batch=_log_int(rng, 1, 64), keys=_log_int(rng, 1, 32768), new=1 if kind == "token" else rng.randint(2, 9) if kind == "few" else _log_int(rng, 10, 2048),
             ragged=rng.randint(1, 1 << 20), scales=rng.choice(["one", "head", "seq"]), window=-1, sinks=0)
    if rng.random() < 0.5:
        c.update(window=_log_int(rng, 1, 5000), sinks=rng.choice([1, 2, 4, 4, 7, 64]), fmt=rng.choice(["same", c["fmt"]]))
    c["keys"] = max(c["keys"], c["new"])
    limit = 4 * 1024 * 8192 * 32 * 128  # (new token, key, head, element) products of the largest listed chunks
    while c["batch"] > 1 and (c["batch"] * c["new"] * c["keys"] * c["hq"] * c["dim"] > limit or c["batch"] * c["keys"] * c["hk"] * c["dim"] > 64 * 4096 * 8 * 128):
        c["batch"] -= 1
    while c["new"] * c["keys"] * c["hq"] * c["dim"] > limit or c["keys"] * c["hk"] * c["dim"] > 64 * 4096 * 8 * 128:
        c["keys"], c["new"] = max(1, c["keys"] * 3 // 4), max(1, min(c["new"], c["keys"] * 3 // 4))
    return c


def _lengths(case):
    """[(new tokens, keys)] of the sequences: all alike, or spread below the largest."""
    new, keys = case.get("new", 1), case["keys"]
    if not case["ragged"]:
        return [(new, keys)] * case["batch"]
    rng, got = random.Random(case["ragged"]), [(new, keys)]
    for _ in range(case["batch"] - 1):
        k = rng.randint(max(1, keys // 8), keys)
        got.append((rng.randint(1, min(new, k)), k))
    return got


def _visible(case):
    """(visible (token, key) pairs, keys that some token sees), over all sequences."""
    pairs = seen = 0
    for q, k in _lengths(case):
        if case["window"] < 0:
            pairs += q * k - q * (q - 1) // 2
            seen += k
            continue
        for t in range(k - q, k):
            low = max(0, t - case["window"])
            pairs += t + 1 - low + min(low, case["sinks"])
        low = max(0, k - q - case["window"])
        seen += k - low + min(low, case["sinks"])
    return pairs, seen


def work(case):
    wide = _DTYPES[case["dtype"]].itemsize
    narrow = wide if case["fmt"] == "same" else 1
    if case["op"] == "write":
        n = 2 * case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": n * (wide + narrow) + 8 * case["tokens"], "flops": n}
    if case["op"] == "read":
        rows = sum(k for _, k in _lengths(case))
        n = 2 * rows * case["heads"] * case["dim"]
        return {"bytes": n * (wide + narrow) + 4 * (rows // case["page"] + 1), "flops": n}
    pairs, seen = _visible(case)
    rows = sum(q for q, _ in _lengths(case))
    return {"bytes": rows * case["hq"] * (2 * case["dim"] * wide + 4) + 2 * seen * case["hk"] * case["dim"] * narrow + 4 * (seen // case["page"] + 1),
            "flops": 4 * pairs * case["hq"] * case["dim"]}


# ---- what a program has in hand ------------------------------------------------------------------------------------------

def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _scales(case, g, heads):
    """Scales of the kind a calibration leaves: the largest value seen over the format's, for the tensor, a head, or a
    sequence's heads.  (Three standard deviations of the inputs here go to an eighth of the format's largest value.)"""
    if case["fmt"] == "same":
        return None, None
    base = 3.0 * 8 / torch.finfo(_FORMATS[case["fmt"]]).max
    shape = {"one": (1,), "head": (heads,), "seq": (case.get("batch", 1), heads)}[case["scales"]]
    spread = torch.rand(2, *shape, generator=g, device="cuda") + 0.75
    return base * spread[0], base * spread[1]


def _stored(case, x, scale):
    return x.to(_DTYPES[case["dtype"]]) if case["fmt"] == "same" else (x / (3.0 * 8 / torch.finfo(_FORMATS[case["fmt"]]).max)).to(_FORMATS[case["fmt"]])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, page, dim = _DTYPES[case["dtype"]], case["page"], case["dim"]
    heads = case["hk"] if case["op"] == "attention" else case["heads"]
    k_scale, v_scale = _scales(case, g, heads)
    s = dict(case=case, k_scale=k_scale, v_scale=v_scale)
    if case["op"] == "write":
        n = case["tokens"]
        pages = 2 * (n // page + 1)
        s["key"], s["value"] = (_normal(g, n, heads, dim).to(dt) for _ in range(2))
        s["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:n]
        if n > 8:
            s["slots"][n // 2] = -1  # a padding token
        s["key_cache"], s["value_cache"] = (torch.zeros(pages, page, heads, dim, dtype=_FORMATS[case["fmt"]], device="cuda") for _ in range(2))
        return s
    lens = _lengths(case)
    table_len = max(-(-k // page) for _, k in lens)
    pages = sum(-(-k // page) for _, k in lens) + 8
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(len(lens), table_len, dtype=torch.int32, device="cuda")
    at = 0
    for b, (_, k) in enumerate(lens):
        n = -(-k // page)
        table[b, :n] = order[at:at + n]
        at += n
    s["table"] = table
    s["key_cache"], s["value_cache"] = (_stored(case, _normal(g, pages, page, heads, dim), None) for _ in range(2))
    s["keys"] = torch.tensor([k for _, k in lens], dtype=torch.int32, device="cuda")
    if case["op"] == "read":
        s["starts"] = torch.tensor([0] + [k for _, k in lens], dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
        s["rows"] = sum(k for _, k in lens)
        return s
    s["starts"] = torch.tensor([0] + [q for q, _ in lens], dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
    s["max_new"], s["max_keys"] = max(q for q, _ in lens), max(k for _, k in lens)
    s["q"] = (1.5 * _normal(g, sum(q for q, _ in lens), case["hq"], dim)).to(dt)
    return s


# ---- the operators ---------------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        return _own(s)
    return {"write": _write, "read": _read, "attention": _attention}[case["op"]](s)


def _own(s):
    import flag_gems

    case = s["case"]
    if case["op"] == "write":
        flag_gems.reshape_and_cache_flash(s["key"], s["value"], s["key_cache"], s["value_cache"], s["slots"], "fp8_" + case["fmt"], s["k_scale"], s["v_scale"])
        return s["key_cache"], s["value_cache"]
    if case["op"] == "read":
        return flag_gems.gather_cache_flash(s["key_cache"], s["value_cache"], s["table"], s["starts"], s["rows"], k_scale=s["k_scale"], v_scale=s["v_scale"],
                                            dtype=_DTYPES[case["dtype"]])
    return flag_gems.flash_attn_varlen_func(
        s["q"], s["key_cache"], s["value_cache"], s["max_new"], s["starts"], s["max_keys"], seqused_k=s["keys"], causal=True, block_table=s["table"],
        window_size=(case["window"], 0), num_sink_tokens=case["sinks"], k_descale=s["k_scale"], v_descale=s["v_scale"], return_softmax_lse=True)


def _write(s):
    fmt = s["key_cache"].dtype
    top, page = torch.finfo(fmt).max, s["case"]["page"]
    live = s["slots"] >= 0
    slots = s["slots"][live]
    for x, cache, scale in ((s["key"], s["key_cache"], s["k_scale"]), (s["value"], s["value_cache"], s["v_scale"])):
        q = (x[live].float() / scale[:, None]).clamp(-top, top).to(fmt)
        cache.view(torch.uint8)[slots // page, slots % page] = q.view(torch.uint8)
    return s["key_cache"], s["value_cache"]


def _read(s):
    page = s["case"]["page"]
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    pos = row - s["starts"].long()[seq]
    block = s["table"][seq, pos // page].long()
    out = []
    for cache, scale in ((s["key_cache"], s["k_scale"]), (s["value_cache"], s["v_scale"])):
        x = _rows(cache, block, pos % page)
        out.append(x if scale is None else (x.float() * scale[:, None]).to(_DTYPES[s["case"]["dtype"]]))
    return tuple(out)


def _rows(cache, block, slot):
    """cache[block, slot], for 8-bit floats too."""
    return cache.view(torch.uint8)[block, slot].view(cache.dtype)


def _attention(s):
    case = s["case"]
    q, table, keys, starts = s["q"], s["table"].long(), s["keys"].long(), s["starts"].long()
    batch, hq, hk, dim, page = table.shape[0], case["hq"], case["hk"], case["dim"], case["page"]
    new = starts[1:] - starts[:-1]
    first = keys - new                                        # position of a sequence's first new token
    # the positions of the keys that some new token may see: all, or the first ones and the window
    if case["window"] < 0:
        pos = torch.arange(s["max_keys"], device="cuda").expand(batch, -1)
        use = pos < keys[:, None]
    else:
        low = (first - case["window"]).clamp(min=0)
        near = low[:, None] + torch.arange(min(s["max_keys"], case["window"] + s["max_new"]), device="cuda")
        sink = torch.arange(case["sinks"], device="cuda").expand(batch, -1)
        pos = torch.cat([sink, near], 1)
        use = torch.cat([sink < low[:, None], near < keys[:, None]], 1)
    at = pos.clamp(max=s["max_keys"] - 1)
    block = table.gather(1, at // page)
    k, v = (_rows(c, block, at % page).float() for c in (s["key_cache"], s["value_cache"]))     # [batch, n, hk, dim]
    if s["k_scale"] is not None:
        k, v = (x * scale.reshape((-1, 1, scale.shape[-1], 1) if scale.dim() == 2 else (1, 1, -1, 1)) for x, scale in ((k, s["k_scale"]), (v, s["v_scale"])))
    v = torch.where(use[:, :, None, None], v, 0.0)
    # queries, padded to the largest number of new tokens: [batch, hk, group * new, dim]
    tok = torch.arange(s["max_new"], device="cuda")
    row = (starts[:-1, None] + tok).clamp(max=q.shape[0] - 1)
    x = q[row].float().view(batch, s["max_new"], hk, hq // hk, dim).permute(0, 2, 3, 1, 4).reshape(batch, hk, -1, dim)
    score = torch.matmul(x, k.permute(0, 2, 3, 1)).mul_(dim ** -0.5).view(batch, hk, hq // hk, s["max_new"], -1)
    mine = (first[:, None] + tok)[:, :, None]                 # [batch, new, 1]
    seen = use[:, None, :] & (pos[:, None, :] <= mine)
    if case["window"] >= 0:
        seen = seen & ((pos[:, None, :] >= mine - case["window"]) | (pos[:, None, :] < case["sinks"]))
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(batch, hk, -1, score.shape[-1]), v.permute(0, 2, 1, 3)).view(batch, hk, hq // hk, s["max_new"], dim)
    o = o / total.clamp(min=1e-30)
    lse = (total.log() + top).squeeze(-1)
    live = tok < new[:, None]
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, s["max_new"], hq, dim)[live]
    lse = lse.permute(0, 3, 1, 2).reshape(batch, s["max_new"], hq)[live].t()
    return o.to(q.dtype), lse.contiguous()


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------------

def _nearest(x, fmt):
    """x rounded to the nearest value of an 8-bit format, ties to the even one, values beyond the largest cut to it."""
    bits, low = (3, -6) if fmt == "e4m3" else (2, -14)
    top = float(torch.finfo(_FORMATS[fmt]).max)
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -60))).clamp(min=low)
    step = torch.exp2(e - bits)
    return (torch.round(x / step) * step).clamp(-top, top)


def exact(case, seed):
    s = prepare(case, seed)
    wide = lambda x: x.float().double()  # noqa: E731
    of = lambda scale, b, h: 1.0 if scale is None else scale.double().expand(case.get("batch", 1), heads)[b, h]  # noqa: E731
    if case["op"] == "write":
        out = []
        for x, cache, scale in ((s["key"], s["key_cache"], s["k_scale"]), (s["value"], s["value_cache"], s["v_scale"])):
            held = wide(cache).view(-1, case["heads"], case["dim"])
            live = s["slots"] >= 0
            held[s["slots"][live]] = _nearest(wide(x[live]) / scale.double()[:, None], case["fmt"])
            out.append(held.view(cache.shape))
        return tuple(out)
    heads = case["hk"] if case["op"] == "attention" else case["heads"]
    out, lses, table, page = [], [], s["table"].long().cpu(), case["page"]
    starts = s["starts"].tolist()
    for b, (n, length) in enumerate(_lengths(case)):
        blocks = table[b, :-(-length // page)].cuda()
        k, v = (wide(c.view(torch.uint8)[blocks].view(c.dtype)).flatten(0, 1)[:length] for c in (s["key_cache"], s["value_cache"]))
        if case["op"] == "read":
            out.append([x if z is None else x * z.double().view(1, -1, 1) for x, z in ((k, s["k_scale"]), (v, s["v_scale"]))])
            continue
        q = wide(s["q"][starts[b]:starts[b] + n])
        i = torch.arange(length - n, length, device="cuda")[:, None]
        j = torch.arange(length, device="cuda")[None, :]
        gone = j > i
        if case["window"] >= 0:
            gone |= (j < i - case["window"]) & (j >= case["sinks"])
        o, l = torch.empty_like(q), torch.empty(case["hq"], n, dtype=torch.float64, device="cuda")
        for h in range(case["hq"]):
            kv = h * heads // case["hq"]
            z = (q[:, h] @ k[:, kv].t()) * (of(s["k_scale"], b, kv) / math.sqrt(case["dim"]))
            z[gone] = -math.inf
            l[h] = torch.logsumexp(z, 1)
            o[:, h] = torch.softmax(z, 1) @ v[:, kv] * of(s["v_scale"], b, kv)
        out.append(o)
        lses.append(l)
    if case["op"] == "read":
        return tuple(torch.cat(x) for x in zip(*out))
    return torch.cat(out), torch.cat(lses, 1)
