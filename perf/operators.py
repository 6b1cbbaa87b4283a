"""The work of a decode or prefill step between the projections: rotary positions, the paged key-value cache and the attention that
reads it, through machx_inference_engine_amd.ops.  One pass of

  kind "rope"    rotates the query and key heads of T tokens (they lie side by side in a row of the fused projection)
  kind "fill"    a prompt's chunk: queries and keys rotated, keys and values written to their slots of the paged cache (as fp16 or as
                 Q8_0: int8 with an fp16 scale for each 32), then every sequence's keys and values read back as fp16 rows, as
                 a prompt's attention wants them
  kind "step"    a decode step: one new token a sequence rotated and written, then attention over the cache
  kind "decode"  the attention alone: one query a sequence over the cache, each group of query heads sharing a key-value head; with a
                 sliding window and a learned extra logit for each head ("sink") where the model has them

Q8_0 follows the weight format of that name: d = amax / 127 kept as fp16, q = round-half-away(x * (127 / amax)), and what is quantised
are the fp16 values that the fp16 cache would hold.  Scores, softmax and sums are fp32.
"""
import math

import torch

own = False
DEV = "cuda"


def listed():
    return [
        # one token of a Llama-3-8B layer: the smallest call, launches and host work count
        {"name": "rope_T1", "kind": "rope", "T": 1, "Hq": 32, "Hkv": 8, "D": 128, "n_rot": 128, "inter": True, "yarn": False, "far": 8192},
        # a long prompt of a gpt-oss layer, positions up to 128 k with the frequencies stretched for them
        {"name": "rope_T8192_yarn", "kind": "rope", "T": 8192, "Hq": 64, "Hkv": 8, "D": 64, "n_rot": 64, "inter": False, "yarn": True, "far": 131072},
        # a ragged prompt with a quarter of each wide head rotated
        {"name": "rope_T333_part", "kind": "rope", "T": 333, "Hq": 16, "Hkv": 2, "D": 256, "n_rot": 64, "inter": False, "yarn": False, "far": 32768},
        # the prompt's last chunk of a few Llama-3-8B sequences; the whole prompts are read back
        {"name": "fill_f16_B4", "kind": "fill", "fmt": "f16", "B": 4, "ctx": 4096, "new": 512, "ragged": True, "ps": 16, "Hq": 32, "Hkv": 8, "D": 128,
         "n_rot": 128, "inter": True, "yarn": False},
        # a long Qwen3-30B-A3B prompt in one sequence, quantised
        {"name": "fill_q8_0_B1", "kind": "fill", "fmt": "q8_0", "B": 1, "ctx": 30001, "new": 2047, "ragged": False, "ps": 64, "Hq": 32, "Hkv": 4, "D": 128,
         "n_rot": 128, "inter": False, "yarn": False},
        # one sequence, early in its answer: latency
        {"name": "step_f16_B1", "kind": "step", "fmt": "f16", "B": 1, "ctx": 500, "ragged": False, "pad": 0, "ps": 16, "Hq": 32, "Hkv": 8, "D": 128,
         "n_rot": 128, "inter": True, "yarn": False, "window": 0, "sinks": False},
        # a batch of Qwen3-30B-A3B sequences over a quantised cache, some places of the batch empty
        {"name": "step_q8_0_B48", "kind": "step", "fmt": "q8_0", "B": 48, "ctx": 4000, "ragged": True, "pad": 5, "ps": 64, "Hq": 32, "Hkv": 4, "D": 128,
         "n_rot": 128, "inter": False, "yarn": False, "window": 0, "sinks": False},
        # a gpt-oss layer with its window of 128 tokens
        {"name": "decode_f16_window", "kind": "decode", "fmt": "f16", "B": 32, "ctx": 8000, "ragged": True, "pad": 0, "ps": 16, "Hq": 64, "Hkv": 8, "D": 64,
         "window": 128, "sinks": True},
        # its layer without one, a ragged batch
        {"name": "decode_q8_0_sinks_B17", "kind": "decode", "fmt": "q8_0", "B": 17, "ctx": 6001, "ragged": True, "pad": 0, "ps": 32, "Hq": 64, "Hkv": 8, "D": 64,
         "window": 0, "sinks": True},
        # one very long sequence: nothing but its length to divide among the compute units
        {"name": "decode_q8_0_B1_long", "kind": "decode", "fmt": "q8_0", "B": 1, "ctx": 131071, "ragged": False, "pad": 0, "ps": 256, "Hq": 32, "Hkv": 8, "D": 128,
         "window": 0, "sinks": False},
        # wide heads, few of them for keys
        {"name": "decode_f16_D256", "kind": "decode", "fmt": "f16", "B": 5, "ctx": 16384, "ragged": True, "pad": 0, "ps": 16, "Hq": 16, "Hkv": 2, "D": 256,
         "window": 0, "sinks": False},
        # the largest: a full batch of long sequences
        {"name": "decode_f16_B64", "kind": "decode", "fmt": "f16", "B": 64, "ctx": 8192, "ragged": False, "pad": 0, "ps": 16, "Hq": 32, "Hkv": 8, "D": 128,
         "window": 0, "sinks": False},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], uniform in the logarithm."""
    return min(hi // step * step, max(-(-lo // step) * step, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def _heads(rng, fmt):
    Hkv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8, 16])
    if Hkv * group > 64:
        group = 64 // Hkv
    return {"Hq": Hkv * group, "Hkv": Hkv, "D": rng.choice([64, 96, 128, 128, 256] + ([80, 112] if fmt == "f16" else []))}


def _rotation(rng, D):
    inter = rng.random() < 0.4
    return {"n_rot": D if rng.random() < 0.7 else max(16, D // rng.choice([2, 4]) // 16 * 16), "inter": inter, "yarn": rng.random() < 0.3}


def draw(rng):
    kind = rng.choice(["rope", "fill", "fill", "step", "step", "decode", "decode", "decode"])
    fmt = rng.choice(["f16", "q8_0"])
    h = _heads(rng, fmt if kind != "rope" else "f16")
    if kind == "rope":
        return {"kind": kind, "T": _log(rng, 1, 8192), **h, **_rotation(rng, h["D"]), "far": _log(rng, 9000, 131072)}
    ps = rng.choice([16, 16, 32, 48, 64, 128, 256])
    room = 2 ** 29  # values of keys and values together, as in the largest listed case
    if kind == "fill":
        B = _log(rng, 1, 16)
        most = max(64, min(32768, room // 8 // (B * h["Hkv"] * h["D"] * 2)))
        return {"kind": kind, "fmt": fmt, "B": B, "ctx": _log(rng, 1, most), "new": _log(rng, 1, min(2048, most)), "ragged": rng.random() < 0.7, "ps": ps, **h,
                **_rotation(rng, h["D"])}
    B = _log(rng, 1, 128)
    most = max(256, min(131072, room // (B * h["Hkv"] * h["D"] * 2)))
    c = {"kind": kind, "fmt": fmt, "B": B, "ctx": _log(rng, 1, most), "ragged": rng.random() < 0.6, "pad": rng.choice([0, 0, 1]) * (B // 8), "ps": ps, **h}
    if kind == "step":
        c.update(_rotation(rng, h["D"]))
    c.update({"window": rng.choice([0, 0, 0, 128, 1000]), "sinks": rng.random() < 0.3})
    return c


# ------------------------------------------------------------------------------------------------------------------- inputs
def _part(b, ragged):
    """A share in (0, 1] for sequence b; sequence 0 is the longest."""
    return 1.0 - (b * 0.6180339887498949) % 1.0 * 0.95 if ragged else 1.0


def _lengths(case):
    """(tokens in the cache before the pass, tokens that the pass writes) of every sequence."""
    old, new = [], []
    live = case["B"] - case.get("pad", 0)
    for b in range(case["B"]):
        s = _part(b, case["ragged"])
        old.append(max(1, int(case["ctx"] * s)) if b < live else 0)
        new.append(0 if case["kind"] == "decode" or b >= live else 1 if case["kind"] == "step" else max(1, int(case["new"] * _part(b + 1, case["ragged"]))))
    return old, new


def _freqs(n_rot, yarn):
    """Radians a position for every pair, in 64 bits, and the factor on the rotated values.  yarn: a context of 4096 stretched 32 times; pairs
    that turn often within it keep their frequency, those that do not turn once are slowed down, those between are mixed."""
    base, i = (150000.0 if yarn else 500000.0), torch.arange(n_rot // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / n_rot)
    if not yarn:
        return f.to(DEV), 1.0
    scale, ctx, fast, slow = 1.0 / 32.0, 4096.0, 32.0, 1.0
    dim = lambda turns: n_rot * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(0.0, math.floor(dim(fast))), min(n_rot - 1.0, math.ceil(dim(slow)))
    keep = 1.0 - ((i - low) / max(0.001, high - low)).clamp(0.0, 1.0)
    return (f * scale * (1 - keep) + f * keep).to(DEV), 1.0 + 0.1 * math.log(1.0 / scale)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, dtype=torch.float16, device=DEV, generator=g)  # noqa: E731
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    s = {"case": case}
    # keys have a few channels that are much larger than the others
    loud = torch.exp(0.6 * torch.randn(D, device=DEV, generator=g)).half()
    if "n_rot" in case:
        s["freqs"], s["mscale"] = _freqs(case["n_rot"], case["yarn"])
    if case["kind"] == "rope":
        s["x"] = rand(case["T"], Hq + Hkv, D)
        start = int(torch.randint(0, case["far"] - case["T"] + 1, (1,), device=DEV, generator=g))
        s["pos"] = torch.arange(start, start + case["T"], dtype=torch.int32, device=DEV)
        return s
    old, new = _lengths(case)
    B, ps = case["B"], case["ps"]
    lens = [a + b for a, b in zip(old, new)]
    pages = [-(-n // ps) for n in lens]
    n_pages, wide = sum(pages) + 3, max(pages)
    order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    first = [sum(pages[:b]) for b in range(B)]
    at, pages_d = torch.arange(wide, dtype=torch.int32, device=DEV)[None], _i32(pages)[:, None]
    s["table"] = torch.where(at < pages_d, order[(_i32(first)[:, None] + at).clamp(max=n_pages - 1).long()], 0).to(torch.int32).contiguous()
    s["lens"], s["max_len"] = _i32(lens), max(lens)
    shape = (n_pages, Hkv, ps, D)
    if case["fmt"] == "f16":
        s["cache"] = (rand(*shape).mul_(loud), rand(*shape))
    else:
        q8 = lambda: (torch.randn(shape, dtype=torch.float16, device=DEV, generator=g) * 40).clamp_(-127, 127).round_().to(torch.int8)  # noqa: E731
        d = lambda: (torch.rand(shape[:3] + (D // 32,), device=DEV, generator=g) * 0.02 + 0.012).half()  # noqa: E731
        s["cache"] = (q8(), d(), q8(), d())
    if case["kind"] in ("fill", "step"):
        T = sum(new)
        qkv = rand(T, (Hq + 2 * Hkv) * D)
        s["q"], s["k"], s["v"] = (t.view(T, -1, D) for t in qkv.split((Hq * D, Hkv * D, Hkv * D), 1))
        s["k"] *= loud
        seq = torch.repeat_interleave(torch.arange(B, device=DEV), torch.tensor(new, device=DEV))
        cum = torch.tensor([sum(new[:b]) for b in range(B)], device=DEV)
        pos = torch.arange(T, device=DEV) - cum[seq] + torch.tensor(old, device=DEV)[seq]
        s["pos"] = pos.to(torch.int32)
        s["slots"] = (s["table"].long()[seq, pos // ps] * ps + pos % ps).to(torch.int32)
    if case["kind"] == "fill":
        s["total"] = sum(lens)
        s["rows"] = _i32([sum(lens[:b]) for b in range(B + 1)])
    if case["kind"] == "step":  # a row of the batch for every sequence; the empty ones at its end have no token
        s["live"] = B - case["pad"]
        s["q_rows"] = torch.zeros(B, Hq, D, dtype=torch.float16, device=DEV)
    if case["kind"] == "decode":
        s["q"] = rand(B, Hq, D)
    if case["kind"] != "fill":
        s["window"], s["sinks"] = case["window"], torch.randn(Hq, device=DEV, generator=g) if case["sinks"] else None
    return s


# ------------------------------------------------------------------------------------------------------------------- plain forms
def _rope(x, pos, freqs, inter, mscale):
    """Pair (x0, x1) turned by pos * freq: angles in 64 bits, products in 32; interleaved pairs are (2i, 2i + 1), others (i, i + n_rot / 2)."""
    n = 2 * freqs.numel()
    a = pos.double()[:, None] * freqs
    c, s = (a.cos() * mscale).float()[:, None], (a.sin() * mscale).float()[:, None]
    r = x[..., :n].float()
    x0, x1 = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., : n // 2], r[..., n // 2:])
    y0, y1 = x0 * c - x1 * s, x0 * s + x1 * c
    y = torch.stack((y0, y1), -1).flatten(-2) if inter else torch.cat((y0, y1), -1)
    return torch.cat((y.half(), x[..., n:]), -1)


def _q8_0(x):
    b = x.float().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    y = b * torch.where(amax > 0, 127.0 / amax, 0.0)
    return ((y.abs() + 0.5).floor() * y.sign()).to(torch.int8).flatten(-2), (amax / 127.0).squeeze(-1).half()


def _write(x, planes, slots, ps):
    page, at = (slots // ps).long(), (slots % ps).long()
    if len(planes) == 1:
        planes[0][page, :, at] = x
    else:
        planes[0][page, :, at], planes[1][page, :, at] = _q8_0(x)


def _split(cache):
    return (cache[:1], cache[1:]) if len(cache) == 2 else (cache[:2], cache[2:])


def _gather(planes, table):
    """[B, Hkv, tokens of the widest row of the table, D] in 32 bits."""
    p = [t[table.long()].transpose(1, 2).flatten(2, 3) for t in planes]
    if len(p) == 1:
        return p[0].float()
    return (p[0].unflatten(-1, (-1, 32)).float() * p[1].float()[..., None]).flatten(-2)


def _attention(q, cache, table, lens, window, sinks):
    K, V = (_gather(p, table) for p in _split(cache))
    B, Hkv, L, D = K.shape
    x = torch.matmul(q.float().view(B, Hkv, -1, D), K.transpose(2, 3)) * D ** -0.5
    t = torch.arange(L, device=DEV)[None]
    live = t < lens[:, None] if not window else (t < lens[:, None]) & (t >= lens[:, None] - window)
    x = x.masked_fill(~live[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    if sinks is not None:
        m = torch.maximum(m, sinks.view(1, Hkv, -1, 1))
    p = torch.where(live[:, None, None], torch.exp(x - m), 0.0)
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sinks.view(1, Hkv, -1, 1) - m)
    o = torch.matmul(p, V) / total
    return torch.where(lens[:, None, None, None] > 0, o, 0.0).half().view(B, -1, D)


def run(s):
    c = s["case"]
    if own:
        from machx_inference_engine_amd import ops
        if c["kind"] == "rope":
            return ops.rope(s["x"], s["pos"], s["freqs"], interleaved=c["inter"], mscale=s["mscale"])
        q = s["q"]
        if c["kind"] == "fill":
            q = ops.rope_kv_write(q, s["k"], s["v"], s["pos"], s["slots"], s["cache"], s["freqs"], interleaved=c["inter"], mscale=s["mscale"])
            return q, *ops.kv_read(s["cache"], s["table"], s["rows"], s["total"])
        if c["kind"] == "step":
            q = s["q_rows"]
            ops.rope_kv_write(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["cache"], s["freqs"], interleaved=c["inter"], mscale=s["mscale"], q_out=q[: s["live"]])
        y = ops.attn_decode(q, s["cache"], s["table"], s["lens"], window=s["window"], sinks=s["sinks"], max_len=s["max_len"])
        return (q, y) if c["kind"] == "step" else y
    if c["kind"] == "rope":
        return _rope(s["x"], s["pos"], s["freqs"], c["inter"], s["mscale"])
    q = s["q"]
    if c["kind"] in ("fill", "step"):
        q = _rope(q, s["pos"], s["freqs"], c["inter"], s["mscale"])
        kp, vp = _split(s["cache"])
        _write(_rope(s["k"], s["pos"], s["freqs"], c["inter"], s["mscale"]), kp, s["slots"], c["ps"])
        _write(s["v"], vp, s["slots"], c["ps"])
    if c["kind"] == "fill":
        live = torch.arange(s["table"].shape[1] * c["ps"], device=DEV)[None] < s["lens"][:, None]
        return q, *(_gather(p, s["table"]).transpose(1, 2)[live].half() for p in _split(s["cache"]))
    if c["kind"] == "step":
        s["q_rows"][: s["live"]] = q
        q = s["q_rows"]
    y = _attention(q, s["cache"], s["table"], s["lens"], s["window"], s["sinks"])
    return (q, y) if c["kind"] == "step" else y


# ------------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_rope(x, pos, freqs, inter, mscale):
    """The pairs as complex numbers, times mscale * exp(i * angle)."""
    n, x = 2 * freqs.numel(), x.double()
    turn = torch.polar(torch.full_like(freqs, mscale)[None].expand(pos.numel(), -1), pos.double()[:, None] * freqs)[:, None]
    y = x.clone()
    if inter:
        z = torch.complex(x[..., 0:n:2].contiguous(), x[..., 1:n:2].contiguous()) * turn
        y[..., 0:n:2], y[..., 1:n:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., : n // 2].contiguous(), x[..., n // 2: n].contiguous()) * turn
        y[..., : n // 2], y[..., n // 2: n] = z.real, z.imag
    return y


def _exact_stored(x, fmt):
    """What a cache of the format holds of these values, which reach it as fp16."""
    x = x.half().double()
    if fmt == "f16":
        return x
    b = x.reshape(x.shape[:-1] + (-1, 32))
    top = b.abs().max(-1, keepdim=True).values
    y = b * 127 / top.clamp(min=1e-300)
    return (torch.trunc(y + 0.5 * torch.sign(y)) * (top / 127).half().double()).reshape(x.shape)


def _exact_rows(s, b, n):
    """Sequence b's n keys and values as they stand in the cache before the pass: [n, Hkv, D] each."""
    c = s["case"]
    t = torch.arange(n, device=DEV)
    page, at = s["table"][b].long()[t // c["ps"]], t % c["ps"]
    pick = [p[page, :, at].double() for p in s["cache"]]
    if c["fmt"] == "q8_0":
        pick = [pick[0] * pick[1].repeat_interleave(32, -1), pick[2] * pick[3].repeat_interleave(32, -1)]
    return pick


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(s["x"], s["pos"], s["freqs"], case["inter"], s["mscale"])
    old, new = _lengths(case)
    q = s["q"].double()
    if case["kind"] != "decode":
        q, k = (_exact_rope(s[n], s["pos"], s["freqs"], case["inter"], s["mscale"]) for n in ("q", "k"))
        k, v = _exact_stored(k, case["fmt"]), _exact_stored(s["v"], case["fmt"])
    keys, values, outs, first = [], [], [], 0
    for b in range(case["B"]):
        n = old[b] + new[b]
        K, V = _exact_rows(s, b, n)
        if new[b]:
            K[old[b]:], V[old[b]:] = k[first: first + new[b]], v[first: first + new[b]]
            first += new[b]
        if case["kind"] == "fill":
            keys.append(K)
            values.append(V)
            continue
        if n == 0:
            outs.append(torch.zeros(case["Hq"], case["D"], dtype=torch.float64, device=DEV))
            continue
        lo = max(0, n - case["window"]) if case["window"] else 0
        qb = q[b].half().double().reshape(case["Hkv"], -1, case["D"])
        x = torch.stack([qb[h] @ K[lo:, h].T for h in range(case["Hkv"])]) / math.sqrt(case["D"])
        if s["sinks"] is not None:
            x = torch.cat((x, s["sinks"].double().reshape(case["Hkv"], -1, 1)), -1)
        p = torch.softmax(x, -1)[..., : n - lo]
        outs.append(torch.stack([p[h] @ V[lo:, h] for h in range(case["Hkv"])]).reshape(case["Hq"], case["D"]))
    if case["kind"] == "fill":
        return q, torch.cat(keys), torch.cat(values)
    y = torch.stack(outs)
    if case["kind"] == "step":
        rows = torch.zeros(s["q_rows"].shape, dtype=torch.float64, device=DEV)
        rows[: s["live"]] = q
        return rows, y
    return y


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Bytes: q, k and v read and the rotated queries written, the new rows of the cache written, the rows that are used of it read
    once, outputs written.  Operations: three a rotated value; two for every product of a score and of the sum of values."""
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if case["kind"] == "rope":
        return {"bytes": case["T"] * ((Hq + Hkv) * D * 4 + 4) + case["n_rot"] * 4, "flops": 3 * case["T"] * (Hq + Hkv) * case["n_rot"]}
    old, new = _lengths(case)
    row = Hkv * 2 * (2 * D if case["fmt"] == "f16" else D + D // 16)  # one token's keys and values in the cache
    T, total, flops = sum(new), 0, 3 * sum(new) * (Hq + Hkv) * case.get("n_rot", 0)
    total += T * ((2 * Hq + 2 * Hkv) * D * 2 + row + 8)
    lens = [a + b for a, b in zip(old, new)]
    if case["kind"] == "fill":
        return {"bytes": total + sum(old) * row + sum(lens) * Hkv * D * 4, "flops": flops}
    if case["window"]:
        lens = [min(n, case["window"]) for n in lens]
    used = sum(lens) * row - T * row  # the rows that this pass wrote need not be read again
    return {"bytes": total + used + case["B"] * Hq * D * (2 if case["kind"] == "step" else 4), "flops": flops + 4 * sum(lens) * Hq * D}
