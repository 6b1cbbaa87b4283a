"""More of what a layer does between its projections, through machx_inference_engine_amd.ops: a key-value cache held in 4 bits with the attention that reads
it, the residual's addition with the norm behind it, and the routing to experts by sigmoid or softmax scores, a bias and groups.  One pass of

  kind "norm"    a layer's output added to the residual stream (fp16), the sum normalised (fp32 weights), and the normalised rows as fp16 and as the 8-bit stream that
                 the int-dot products take; "halves": the stream with a sum for each half of a block, as the expert products of a prompt take it
  kind "route"   from router logits to expert ids (ascending) and their weights: scores are softmax or sigmoid; score + bias is what is compared; of the groups of experts
                 the best by their largest, or by the sum of their two largest, are kept, and of their experts the best k; the weights are the scores without the bias,
                 over their sum, times a factor.  Equal ones: the lowest id first
  kind "fill"    a prompt's chunk: queries and keys rotated, keys and values written to their slots of the paged cache as Q4_0 (4-bit codes with an fp16 scale for
                 each 32), then every sequence's keys and values read back as fp16 rows
  kind "step"    a decode step: one new token a sequence rotated and written, then attention over the cache
  kind "decode"  the attention alone: one query a sequence, groups of query heads sharing a key-value head, with a sliding window and a learned extra logit for each
                 head ("sink") where the model has them

Q4_0 follows the weight format of that name: d = (the value of largest magnitude, the first of equal ones) / -8 kept as fp16, code = min(15, floor(x / d + 8.5)) with the
unrounded d and without rounding in between, value = d * (code - 8); byte j of a block's 16 holds elements j (low) and j + 16 (high).  What is quantised are the fp16
values that an fp16 cache would hold.  Scores, softmax and sums of attention and norm are fp32; what decides between two codes or two experts is 64 bits.
"""
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-5


def listed():
    return [
        # one token of a Llama-3-8B layer: the smallest call, launches and host work count
        {"name": "norm_T1", "kind": "norm", "T": 1, "H": 4096, "halves": False},
        # a ragged gpt-oss prompt, the stream for its experts
        {"name": "norm_T333_halves", "kind": "norm", "T": 333, "H": 2880, "halves": True},
        # a long Llama-3-8B prompt: memory alone
        {"name": "norm_T8192", "kind": "norm", "T": 8192, "H": 4096, "halves": False},
        # one token of a Qwen3-30B-A3B layer: latency
        {"name": "route_T1", "kind": "route", "T": 1, "E": 128, "k": 8, "score": "softmax", "bias": False, "groups": 1, "kept": 1, "two": False, "renorm": True, "scale": 1.0, "f32": False},
        # a prompt over many experts in groups, balanced by a bias
        {"name": "route_T4096_groups", "kind": "route", "T": 4096, "E": 256, "k": 8, "score": "sigmoid", "bias": True, "groups": 8, "kept": 4, "two": True, "renorm": True, "scale": 2.5,
         "f32": True},
        # the prompts' last chunk of a few Llama-3-8B sequences; the whole prompts are read back
        {"name": "fill_B4", "kind": "fill", "B": 4, "ctx": 4096, "new": 512, "ragged": True, "ps": 16, "Hq": 32, "Hkv": 8, "D": 128, "n_rot": 128, "inter": True},
        # a long Qwen3-30B-A3B prompt in one sequence
        {"name": "fill_B1", "kind": "fill", "B": 1, "ctx": 30001, "new": 2047, "ragged": False, "ps": 64, "Hq": 32, "Hkv": 4, "D": 128, "n_rot": 128, "inter": False},
        # one sequence, early in its answer: latency
        {"name": "step_B1", "kind": "step", "B": 1, "ctx": 500, "ragged": False, "pad": 0, "ps": 16, "Hq": 32, "Hkv": 8, "D": 128, "n_rot": 128, "inter": True, "window": 0, "sinks": False},
        # a batch of Qwen3-30B-A3B sequences, some places of the batch empty
        {"name": "step_B48", "kind": "step", "B": 48, "ctx": 4000, "ragged": True, "pad": 5, "ps": 64, "Hq": 32, "Hkv": 4, "D": 128, "n_rot": 128, "inter": False, "window": 0,
         "sinks": False},
        # a ragged batch of gpt-oss sequences: narrow heads, sinks
        {"name": "decode_sinks_B17", "kind": "decode", "B": 17, "ctx": 6001, "ragged": True, "pad": 0, "ps": 32, "Hq": 64, "Hkv": 8, "D": 64, "window": 0, "sinks": True},
        # one very long sequence: nothing but its length to divide among the compute units
        {"name": "decode_B1_long", "kind": "decode", "B": 1, "ctx": 131071, "ragged": False, "pad": 0, "ps": 256, "Hq": 32, "Hkv": 8, "D": 128, "window": 0, "sinks": False},
        # the largest: a full batch of long sequences, whose fp16 cache would be four times the size
        {"name": "decode_B64", "kind": "decode", "B": 64, "ctx": 8192, "ragged": False, "pad": 0, "ps": 16, "Hq": 32, "Hkv": 8, "D": 128, "window": 0, "sinks": False},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], uniform in the logarithm."""
    return min(hi // step * step, max(-(-lo // step) * step, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def _draw_route(rng):
    groups, size = rng.choice([1, 1, 2, 3, 4, 8, 16]), rng.choice([4, 5, 8, 12, 20, 32, 64])
    if groups == 1:
        size = rng.choice([8, 17, 32, 60, 64, 100, 128, 160, 256, 384, 512])
    kept = rng.randint(1, groups)
    score = rng.choice(["softmax", "sigmoid"])
    return {"kind": "route", "T": _log(rng, 1, min(8192, (1 << 20) // (groups * size))), "E": groups * size, "k": rng.randint(1, min(16, kept * size)), "score": score,
            "bias": rng.random() < (0.7 if score == "sigmoid" else 0.3), "groups": groups, "kept": kept, "two": rng.random() < 0.5, "renorm": rng.random() < 0.8,
            "scale": rng.choice([1.0, 1.0, 2.5]), "f32": rng.random() < 0.5}


def draw(rng):
    kind = rng.choice(["norm", "norm", "route", "route", "fill", "fill", "step", "step", "decode", "decode", "decode"])
    if kind == "route":
        return _draw_route(rng)
    if kind == "norm":
        H = _log(rng, 64, 16384, 32)
        return {"kind": kind, "T": _log(rng, 1, max(1, (1 << 25) // H)), "H": H, "halves": rng.random() < 0.4}
    Hkv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 4, 5, 7, 8, 16])
    if Hkv * group > 64:
        group = 64 // Hkv
    D = rng.choice([32, 64, 64, 96, 128, 128, 128, 160, 256])
    h = {"Hq": Hkv * group, "Hkv": Hkv, "D": D}
    turn = {"n_rot": D if rng.random() < 0.7 else max(16, D // rng.choice([2, 4]) // 16 * 16), "inter": rng.random() < 0.4}
    ps = rng.choice([16, 16, 32, 48, 64, 128, 256])
    room = 2 ** 29  # values of keys and values together
    if kind == "fill":
        B = _log(rng, 1, 16)
        most = max(64, min(32768, room // 8 // (B * Hkv * D * 2)))
        return {"kind": kind, "B": B, "ctx": _log(rng, 1, most), "new": _log(rng, 1, min(2048, most)), "ragged": rng.random() < 0.7, "ps": ps, **h, **turn}
    B = _log(rng, 1, 128)
    most = max(256, min(131072, room // (B * Hkv * D * 2)))
    c = {"kind": kind, "B": B, "ctx": _log(rng, 1, most), "ragged": rng.random() < 0.6, "pad": rng.choice([0, 0, 1]) * (B // 8), "ps": ps, **h}
    if kind == "step":
        c.update(turn)
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


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, dtype=torch.float16, device=DEV, generator=g)  # noqa: E731
    s = {"case": case}
    if case["kind"] == "norm":
        # a residual stream has a few channels that are much larger than the others
        loud = torch.exp(1.2 * torch.randn(case["H"], device=DEV, generator=g)).half()
        s["res"], s["x"] = rand(case["T"], case["H"]) * loud, rand(case["T"], case["H"])
        s["w"] = 1.0 + 0.3 * torch.randn(case["H"], device=DEV, generator=g)
        return s
    if case["kind"] == "route":
        logits = torch.randn((case["T"], case["E"]), device=DEV, generator=g) * 2.0
        s["logits"] = logits if case["f32"] else logits.half()
        s["bias"] = 0.1 * torch.randn(case["E"], device=DEV, generator=g) if case["bias"] else None
        return s
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    loud = torch.exp(0.6 * torch.randn(D, device=DEV, generator=g)).half()
    if "n_rot" in case:
        s["freqs"] = 500000.0 ** (-2.0 * torch.arange(case["n_rot"] // 2, dtype=torch.float64, device=DEV) / case["n_rot"])
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
    shape = (n_pages, Hkv, ps)
    codes = lambda: torch.randint(0, 256, shape + (D // 2,), dtype=torch.uint8, device=DEV, generator=g)  # noqa: E731
    # scales of either sign, those of the keys as loud as their blocks' channels
    d = lambda: ((torch.rand(shape + (D // 32,), device=DEV, generator=g) * 0.2 + 0.15) * (torch.randint(0, 2, shape + (D // 32,), device=DEV, generator=g) * 2 - 1)).half()  # noqa: E731
    s["cache"] = (codes(), d() * loud.view(-1, 32).amax(1), codes(), d())
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
def _norm(x, res, w):
    """(sum, normalised rows, what their 8-bit stream stands for): blocks of 32 with d = amax / 127, q = round-half-away(y * (127 / amax))."""
    h = (x.float() + res.float()).half()
    f = h.float()
    y = (f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * w).half()
    b = y.float().unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    t = b * torch.where(amax > 0, 127.0 / amax, 0.0)
    return h, y, ((t.abs() + 0.5).floor() * t.sign() * (amax / 127.0)).half().flatten(-2)


def _stream_values(stream, T, H, size):
    """The values of a stream of 8-bit blocks (fp32 d at its start, 32 codes at its end), in one product."""
    b = stream.view(T, H // 32, size)
    return torch.mul(b[..., size - 32:].view(torch.int8), b[..., :4].view(torch.float32), out=torch.empty(T, H // 32, 32, dtype=torch.float16, device=stream.device)).view(T, H)


def _best(score, n):
    """Where the n largest of the last axis are, the first of equal ones, in ascending order."""
    return torch.sort(torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :n], dim=-1).values


def _route(logits, bias, c):
    x = logits.double()
    if c["score"] == "softmax":
        e = torch.exp(x - x.amax(-1, keepdim=True))
        score = e / e.sum(-1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    choice = score if bias is None else score + bias.double()
    if c["groups"] > 1:
        by = choice.unflatten(-1, (c["groups"], -1))
        group = torch.sort(by, dim=-1, descending=True).values[..., :2].sum(-1) if c["two"] else by.amax(-1)
        kept = torch.zeros_like(group, dtype=torch.bool).scatter(-1, _best(group, c["kept"]), True)
        choice = torch.where(kept[..., None], by, -math.inf).flatten(-2)
    idx = _best(choice, c["k"])
    w = score.gather(-1, idx)
    if c["renorm"]:
        w = w / (w.sum(-1, keepdim=True) + 1e-20)
    return idx.to(torch.int32), (w * c["scale"]).half()


def _rope(x, pos, freqs, inter):
    """Pair (x0, x1) turned by pos * freq: angles in 64 bits, sines and the second product in 32, the first product and the sum rounded together, as a multiply-add does: a
    key next to a border between two codes, and so its code, goes by that rounding.  Interleaved pairs are (2i, 2i + 1), others (i, i + n_rot / 2)."""
    n = 2 * freqs.numel()
    a = pos.double()[:, None] * freqs
    c, s = a.cos().float()[:, None], a.sin().float()[:, None]
    r = x[..., :n].float()
    x0, x1 = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., : n // 2], r[..., n // 2:])
    y0, y1 = x0.double() * c - (x1 * s).double(), x0.double() * s + (x1 * c).double()
    y = torch.stack((y0, y1), -1).flatten(-2) if inter else torch.cat((y0, y1), -1)
    return torch.cat((y.float().half(), x[..., n:]), -1)


def _q4_0(x):
    b = x.unflatten(-1, (-1, 32))
    top = b.gather(-1, _best(b.abs(), 1)).double()
    code = torch.where(top != 0, b.double() * -8.0 / top + 8.5, 8.0).floor().clamp(max=15.0).to(torch.uint8)
    return (code[..., :16] | code[..., 16:] << 4).flatten(-2), (top / -8.0).squeeze(-1).half()


def _write(x, planes, slots, ps):
    page, at = (slots // ps).long(), (slots % ps).long()
    planes[0][page, :, at], planes[1][page, :, at] = _q4_0(x)


def _gather(planes, table):
    """[B, Hkv, tokens of the widest row of the table, D] in 32 bits."""
    codes, d = (t[table.long()].transpose(1, 2).flatten(2, 3) for t in planes)
    b = codes.unflatten(-1, (-1, 16))
    return ((torch.cat((b & 15, b >> 4), -1).float() - 8.0) * d.float()[..., None]).flatten(-2)


def _attention(q, cache, table, lens, window, sinks):
    K, V = _gather(cache[:2], table), _gather(cache[2:], table)
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
        if c["kind"] == "norm":
            h, y, stream = ops.add_rms_norm_f32w_q8(s["x"], s["res"], s["w"], EPS, halves=c["halves"])
            return h, y, _stream_values(stream, c["T"], c["H"], 48 if c["halves"] else 40)
        if c["kind"] == "route":
            return ops.moe_route(s["logits"], c["k"], score=c["score"], bias=s["bias"], n_groups=c["groups"], topk_groups=c["kept"], group_score="top2" if c["two"] else "max",
                                 renormalize=c["renorm"], scale=c["scale"])
        q = s["q"]
        if c["kind"] == "fill":
            q = ops.rope_kv_write(q, s["k"], s["v"], s["pos"], s["slots"], s["cache"], s["freqs"], interleaved=c["inter"])
            return q, *ops.kv_read(s["cache"], s["table"], s["rows"], s["total"])
        if c["kind"] == "step":
            q = s["q_rows"]
            ops.rope_kv_write(s["q"], s["k"], s["v"], s["pos"], s["slots"], s["cache"], s["freqs"], interleaved=c["inter"], q_out=q[: s["live"]])
        y = ops.attn_decode(q, s["cache"], s["table"], s["lens"], window=s["window"], sinks=s["sinks"], max_len=s["max_len"])
        return (q, y) if c["kind"] == "step" else y
    if c["kind"] == "norm":
        return _norm(s["x"], s["res"], s["w"])
    if c["kind"] == "route":
        return _route(s["logits"], s["bias"], c)
    q = s["q"]
    if c["kind"] in ("fill", "step"):
        q = _rope(q, s["pos"], s["freqs"], c["inter"])
        _write(_rope(s["k"], s["pos"], s["freqs"], c["inter"]), s["cache"][:2], s["slots"], c["ps"])
        _write(s["v"], s["cache"][2:], s["slots"], c["ps"])
    if c["kind"] == "fill":
        live = torch.arange(s["table"].shape[1] * c["ps"], device=DEV)[None] < s["lens"][:, None]
        return q, *(_gather(p, s["table"]).transpose(1, 2)[live].half() for p in (s["cache"][:2], s["cache"][2:]))
    if c["kind"] == "step":
        s["q_rows"][: s["live"]] = q
        q = s["q_rows"]
    y = _attention(q, s["cache"], s["table"], s["lens"], s["window"], s["sinks"])
    return (q, y) if c["kind"] == "step" else y


# ------------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_norm(s):
    """The sum and the normalised rows are fp16 values on the way, as the operator has them: the rows are those of the rounded sum, the stream that of the rounded rows."""
    total = s["x"].double() + s["res"].double()
    h = total.half().double()
    y = h / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt() * s["w"].double()
    b = y.half().double().reshape(y.shape[0], -1, 32)
    step = b.abs().max(2, keepdim=True).values.clamp(min=1e-300) / 127
    n = b / step
    return total, y, (torch.trunc(n + 0.5 * torch.sign(n)) * step).reshape(y.shape)


def _exact_route(s, c):
    """Experts are struck one after another: groups first, then those chosen.  The ids are whole numbers: the weights alone have a value in 64 bits."""
    x = s["logits"].double()
    p = torch.softmax(x, 1) if c["score"] == "softmax" else torch.sigmoid(x)
    key = p.clone() if s["bias"] is None else p + s["bias"].double()
    T, E = x.shape
    size, rows = E // c["groups"], torch.arange(T, device=x.device)
    if c["groups"] > 1:
        worth = key.view(T, c["groups"], size).topk(min(2, size), 2).values
        worth = worth.sum(2) if c["two"] else worth[:, :, 0]
        struck = torch.ones(T, c["groups"], dtype=torch.bool, device=x.device)
        for _ in range(c["kept"]):
            first = (worth == worth.max(1, keepdim=True).values).to(torch.uint8).argmax(1)
            struck[rows, first] = False
            worth[rows, first] = -math.inf
        key[struck.repeat_interleave(size, 1)] = -math.inf
    picked = torch.zeros(T, E, dtype=torch.bool, device=x.device)
    for _ in range(c["k"]):
        first = (key == key.max(1, keepdim=True).values).to(torch.uint8).argmax(1)
        picked[rows, first] = True
        key[rows, first] = -math.inf
    w = p[picked].view(T, c["k"])
    return None, c["scale"] * (w / (w.sum(1, keepdim=True) + 1e-20) if c["renorm"] else w)


def _exact_rope(x, pos, freqs, inter):
    """The pairs as complex numbers, times exp(i * angle)."""
    n, x = 2 * freqs.numel(), x.double()
    turn = torch.polar(torch.ones_like(freqs)[None].expand(pos.numel(), -1), pos.double()[:, None] * freqs)[:, None]
    y = x.clone()
    if inter:
        z = torch.complex(x[..., 0:n:2].contiguous(), x[..., 1:n:2].contiguous()) * turn
        y[..., 0:n:2], y[..., 1:n:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., : n // 2].contiguous(), x[..., n // 2: n].contiguous()) * turn
        y[..., : n // 2], y[..., n // 2: n] = z.real, z.imag
    return y


def _exact_stored(x):
    """What a Q4_0 cache holds of these values, which reach it as fp16."""
    x = x.half().double()
    b = x.reshape(x.shape[:-1] + (-1, 32))
    up, down = b.max(-1, keepdim=True), b.min(-1, keepdim=True)
    first_up, first_down = ((b == t.values).to(torch.uint8).argmax(-1, keepdim=True) for t in (up, down))
    positive = (up.values > -down.values) | ((up.values == -down.values) & (first_up < first_down))
    step = torch.where(positive, up.values, down.values) / -8
    code = torch.floor(b / torch.where(step == 0, 1.0, step) + 8.5).clamp(max=15)
    return ((code - 8) * step.half().double()).reshape(x.shape)


def _exact_rows(s, b, n):
    """Sequence b's n keys and values as they stand in the cache before the pass: [n, Hkv, D] each."""
    c = s["case"]
    t = torch.arange(n, device=DEV)
    page, at = s["table"][b].long()[t // c["ps"]], t % c["ps"]
    rows = []
    for codes, d in (s["cache"][:2], s["cache"][2:]):
        byte = codes[page, :, at].to(torch.int64).reshape(n, c["Hkv"], c["D"] // 32, 16)
        value = torch.stack((byte % 16, byte // 16), -2).reshape(n, c["Hkv"], c["D"]) - 8
        rows.append(value.double() * d[page, :, at].double().repeat_interleave(32, -1))
    return rows


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "norm":
        return _exact_norm(s)
    if case["kind"] == "route":
        return _exact_route(s, case)
    old, new = _lengths(case)
    q = s["q"].double()
    if case["kind"] != "decode":
        q, k = (_exact_rope(s[n], s["pos"], s["freqs"], case["inter"]) for n in ("q", "k"))
        k, v = _exact_stored(k), _exact_stored(s["v"])
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
    """Bytes: rows, logits, weights and the new tokens' q, k and v read, results written, the new rows of the cache written, the rows that are used of it read once.
    Operations: ten a normalised element (sum, square, three products, the block's largest, product, rounding, product back, sum), about eight a score (exponential, sum,
    quotient, comparisons), three a rotated value, two for every product of an attention score and of the sum of values."""
    if case["kind"] == "norm":
        n = case["T"] * case["H"]
        return {"bytes": 8 * n + n // 32 * (48 if case["halves"] else 40) + 4 * case["H"], "flops": 10 * n}
    if case["kind"] == "route":
        n = case["T"] * case["E"]
        return {"bytes": n * (4 if case["f32"] else 2) + 6 * case["T"] * case["k"] + (4 * case["E"] if case["bias"] else 0), "flops": 8 * n}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    old, new = _lengths(case)
    row = Hkv * 2 * (D // 2 + D // 16)  # one token's keys and values in the cache
    T, total, flops = sum(new), 0, 3 * sum(new) * (Hq + Hkv) * case.get("n_rot", 0)
    total += T * ((2 * Hq + 2 * Hkv) * D * 2 + row + 8)
    lens = [a + b for a, b in zip(old, new)]
    if case["kind"] == "fill":
        return {"bytes": total + sum(old) * row + sum(lens) * Hkv * D * 4, "flops": flops}
    if case["window"]:
        lens = [min(n, case["window"]) for n in lens]
    used = sum(lens) * row - T * row  # the rows that this pass wrote need not be read again
    return {"bytes": total + used + case["B"] * Hq * D * (2 if case["kind"] == "step" else 4), "flops": flops + 4 * sum(lens) * Hq * D}
