"""The operators of decoder-only language models next to the attention path, as work to be timed and compared: attention
with a sliding window and visible first keys (forward, training step, one decoding step over a cache), rotary positions
(whole prompts, and new rows rotated into a cache), and log probabilities of given tokens with entropy and the best
alternatives (forward, and with the gradient of the logits).

`run` computes an operator in elementary torch operations, or, where `own` is set, with this package's calls."""
import math

import torch

own = False

_ctx = None


def _context():
    """The one context a program keeps for its lifetime."""
    global _ctx
    if _ctx is None:
        from dl4s_amd import lib
        _ctx = lib.Context(torch.cuda.current_device())
    return _ctx


# ---------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one short sequence through one layer: every pass is a handful of launches
        dict(name="window forward, 128 tokens", op="window", train=False, B=1, H=8, Hkv=8, Lq=128, Lk=128, d=64, window=32,
             sinks=4, ragged=False, token_major=False),
        # a batch of prompts, one key head per query head
        dict(name="window forward, 8 x 2048", op="window", train=False, B=8, H=16, Hkv=16, Lq=2048, Lk=2048, d=64, window=512,
             sinks=4, ragged=False, token_major=False),
        # one long document, four query heads on a key head, operands as the projections leave them
        dict(name="window forward, 8192 tokens", op="window", train=False, B=1, H=16, Hkv=4, Lq=8192, Lk=8192, d=128,
             window=1024, sinks=16, ragged=False, token_major=True),
        # a small training step on a padded batch (the last rows of the shorter sequences see no key)
        dict(name="window training, 4 x 512", op="window", train=True, B=4, H=8, Hkv=8, Lq=512, Lk=512, d=64, window=128,
             sinks=0, ragged=True, token_major=False),
        # a large training step: shared key heads, a head dim between two tile widths, an odd window
        dict(name="window training, 2 x 4096", op="window", train=True, B=2, H=16, Hkv=4, Lq=4096, Lk=4096, d=96, window=777,
             sinks=5, ragged=False, token_major=True),
        # serving: a batch of sequences of different lengths, one token each
        dict(name="window decode, 16 x 4096", op="decode", B=16, H=16, Hkv=16, T=4096, Tcap=4160, d=64, window=1024, sinks=4),
        # serving far into long caches (an element offset past 2^31), grouped heads
        dict(name="window decode, 32 x 30001", op="decode", B=32, H=32, Hkv=8, T=30001, Tcap=32768, d=128, window=4096,
             sinks=4),
        # one new token per sequence: its query rotated, its key and value written to the cache
        dict(name="rotary append, 16 x 1", op="append", B=16, L=1, H=16, Hkv=16, Tcap=4160, d=64, rot=64, interleaved=False,
             token_major=True, scale=1.0),
        # queries and keys of long prompts, half of the head turned, frequencies stretched for a longer context
        dict(name="rotary, 2 x 8192", op="rotary", B=2, L=8192, H=32, Hkv=8, d=128, rot=64, interleaved=True,
             token_major=True, inverse=False, far=100000, scale=4.0),
        # one decoding step's logits: the chosen tokens' log probabilities and a few alternatives
        dict(name="log probabilities, 8 x 32000", op="logprobs", train=False, rows=8, n=32000, stride=32000, top=8, temp=0.7),
        # scoring whole documents
        dict(name="log probabilities, 4096 x 100000", op="logprobs", train=False, rows=4096, n=100000, stride=100000, top=20,
             temp=1.0),
        # a loss over a vocabulary of odd size in padded rows, with an entropy term
        dict(name="log probability loss, 2048 x 50257", op="logprobs", train=True, rows=2048, n=50257, stride=50304, top=0,
             temp=1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["window", "window", "training", "decode", "append", "rotary", "logprobs", "loss"])
    if op in ("window", "training"):
        d = rng.choice([32, 40, 64, 64, 80, 96, 128, 128, rng.randint(1, 128)])
        Hkv = rng.choice([1, 2, 4, 8])
        H = Hkv * rng.choice([1, 1, 2, 3, 4])
        Lk = _log_int(rng, 8 if op == "training" else 1, 4096)
        Lq = Lk if op == "training" or rng.random() < 0.6 else _log_int(rng, 1, Lk)     # a later piece of a prompt
        B = max(1, min(8, _log_int(rng, 1, 8), (1 << 28) // (H * Lq * Lk)))
        return dict(op="window", train=op == "training", B=B, H=H, Hkv=Hkv, Lq=Lq, Lk=Lk, d=d,
                    window=_log_int(rng, 2 if op == "training" else 1, 2048),   # (one visible key: the gradient is all rounding)
                    sinks=rng.choice([0, 0, 1, 4, 7, 64]), ragged=rng.random() < 0.4, token_major=rng.random() < 0.5)
    if op == "decode":
        Hkv = rng.choice([1, 2, 4, 8, 16])
        T = _log_int(rng, 1, 20000)
        return dict(op="decode", B=_log_int(rng, 1, 32), H=Hkv * rng.choice([1, 1, 2, 3, 4, 8]), Hkv=Hkv, T=T,
                    Tcap=T + rng.randint(0, 100), d=rng.choice([32, 64, 64, 80, 128, 128, rng.randint(1, 128)]),
                    window=_log_int(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 4, 33]))
    if op in ("append", "rotary"):
        d = rng.choice([32, 64, 64, 80, 96, 128, 128, 256, 2 * rng.randint(1, 128)])
        Hkv = rng.choice([1, 2, 4, 8, 16])
        c = dict(op=op, B=_log_int(rng, 1, 16), H=Hkv * rng.choice([1, 1, 2, 3, 4]), Hkv=Hkv, d=d,
                 rot=d if rng.random() < 0.6 else 2 * rng.randint(1, d // 2), interleaved=rng.random() < 0.5,
                 token_major=rng.random() < 0.5, scale=rng.choice([1.0, 1.0, 4.0, 8.0]))
        if op == "append":
            return dict(c, L=_log_int(rng, 1, 512) if rng.random() < 0.4 else 1, Tcap=_log_int(rng, 600, 8192))
        return dict(c, L=_log_int(rng, 1, 4096), inverse=rng.random() < 0.4, far=_log_int(rng, 1, 1000000))
    n = _log_int(rng, 2, 150000)
    rows = max(1, min(_log_int(rng, 1, 4096), (1 << 28) // n))
    train = op == "loss"
    return dict(op="logprobs", train=train, rows=rows, n=n, stride=n + rng.choice([0, 0, 0, rng.randint(1, 64)]),
                top=0 if train else min(n, rng.choice([0, 1, 5, 20, 64])), temp=rng.choice([1.0, 1.0, 0.6, 1.3]))


# --------------------------------------------------------------------------------------------------------- the inputs

def _lengths(B, L, ragged):
    """Valid keys of each batch element: from L down to a little over half of it."""
    return [L - (b * L) // (2 * B) if ragged else L for b in range(B)]


def _turns(rot, scale):
    """Turns per position of each pair, in 64 bits: 10000^(-2i / rot) radians, and for a context stretched `scale` times the
    slow pairs (less than one turn over 4096 positions) slowed by that factor, the fast ones (over four) left, a ramp between."""
    f = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / rot) / (2 * math.pi)
    keep = ((4096 * f - 1) / 3).clamp(0, 1)
    return f * (keep + (1 - keep) / scale)


def _amplitude(scale):
    """The factor on the turned columns that goes with a stretched context."""
    return 1.0 if scale == 1.0 else float(torch.tensor(0.1 * math.log(scale) + 1))


def _heads(c, L, H):
    return (c["B"], L, H, c["d"]) if c["token_major"] else (c["B"], H, L, c["d"])


def prepare(case, seed):
    c, g = case, torch.Generator("cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    like = lambda *shape: torch.empty(*shape, device="cuda")  # noqa: E731
    s = {"case": c}
    if c["op"] == "window":
        s.update(q=rand(*_heads(c, c["Lq"], c["H"])) * 1.5, k=rand(*_heads(c, c["Lk"], c["Hkv"])), v=rand(*_heads(c, c["Lk"], c["Hkv"])),
                 lengths=torch.tensor(_lengths(c["B"], c["Lk"], True), dtype=torch.int32, device="cuda") if c["ragged"] else None)
        s.update(out=torch.empty_like(s["q"]))
        if c["train"]:
            s.update(dout=rand(*s["q"].shape), stats=like(c["B"], c["H"], c["Lq"], 2), dq=torch.empty_like(s["q"]),
                     dk=torch.empty_like(s["k"]), dv=torch.empty_like(s["v"]))
    elif c["op"] == "decode":
        s.update(q=rand(c["B"], c["H"], 1, c["d"]) * 1.5, kcache=rand(c["B"], c["Hkv"], c["Tcap"], c["d"]),
                 vcache=rand(c["B"], c["Hkv"], c["Tcap"], c["d"]),
                 lengths=torch.tensor(_lengths(c["B"], c["T"], True), dtype=torch.int32, device="cuda"))
        s.update(out=torch.empty_like(s["q"]))
    elif c["op"] == "append":
        s.update(q=rand(*_heads(c, c["L"], c["H"])), k=rand(*_heads(c, c["L"], c["Hkv"])), v=rand(*_heads(c, c["L"], c["Hkv"])),
                 kcache=rand(c["B"], c["Hkv"], c["Tcap"], c["d"]), vcache=rand(c["B"], c["Hkv"], c["Tcap"], c["d"]),
                 starts=torch.randint(0, c["Tcap"] - c["L"] + 1, (c["B"],), device="cuda", generator=g, dtype=torch.int32),
                 turns=_turns(c["rot"], c["scale"]), amplitude=_amplitude(c["scale"]))
        s.update(q_out=torch.empty_like(s["q"]))
    elif c["op"] == "rotary":
        start = torch.randint(0, c["far"], (c["B"], 1), device="cuda", generator=g, dtype=torch.int32)
        s.update(q=rand(*_heads(c, c["L"], c["H"])), k=rand(*_heads(c, c["L"], c["Hkv"])),
                 positions=(start + torch.arange(c["L"], device="cuda", dtype=torch.int32)).contiguous(),
                 turns=_turns(c["rot"], c["scale"]), amplitude=_amplitude(c["scale"]))
        s.update(q_out=torch.empty_like(s["q"]), k_out=torch.empty_like(s["k"]))
    else:
        rows, n = c["rows"], c["n"]
        logits = rand(rows, c["stride"]) * 2.5
        targets = torch.randint(0, n, (rows,), device="cuda", generator=g, dtype=torch.int32)
        targets[::7] = -1                                       # padding: takes no part
        s.update(logits=logits, targets=targets, logprobs=like(rows), entropy=like(rows))
        if c["top"]:
            s.update(top_logprobs=like(rows, c["top"]), top_tokens=torch.empty(rows, c["top"], dtype=torch.int32, device="cuda"))
        if c["train"]:
            s.update(stats=like(rows, 3), dlogprobs=rand(rows) / rows, dentropy=rand(rows) / rows,
                     dlogits=torch.zeros(rows, c["stride"], device="cuda"))
    return s


# ------------------------------------------------------------------------------------------------------ the plain forms

def _visible(Lq, Lk, window, sinks, lengths):
    """[B or 1, 1, 1, Lq, Lk]: whether query i, at position Lk - Lq + i, sees key j."""
    p = torch.arange(Lq, device="cuda")[:, None] + (Lk - Lq)
    j = torch.arange(Lk, device="cuda")[None, :]
    see = ((j <= p) & ((j > p - window) | (j < sinks)))[None, None, None]
    return see if lengths is None else see & (j < lengths[:, None, None])[:, None, None]


def _softmax(s, see):
    """Weights over the last axis where `see`; a row that sees nothing has none."""
    s = torch.where(see, s, -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _grouped(x, c, groups):
    """[B, Hkv, groups, L, d] view of a tensor in either layout."""
    x = x.transpose(1, 2) if c["token_major"] else x
    return x.reshape(x.shape[0], c["Hkv"], groups, x.shape[2], x.shape[3])


def _laid_out(x, c):
    """Back from [B, Hkv, groups, L, d] to the layout of the inputs."""
    x = x.reshape(x.shape[0], x.shape[1] * x.shape[2], x.shape[3], x.shape[4])
    return x.transpose(1, 2).contiguous() if c["token_major"] else x


def _window_plain(s, c):
    G, t = c["H"] // c["Hkv"], c["d"] ** -0.5
    q, k, v = _grouped(s["q"], c, G) * t, _grouped(s["k"], c, 1), _grouped(s["v"], c, 1)
    w = _softmax(q @ k.transpose(-1, -2), _visible(c["Lq"], c["Lk"], c["window"], c["sinks"], s["lengths"]))
    out = w @ v
    if not c["train"]:
        return {"out": _laid_out(out, c)}
    dout = _grouped(s["dout"], c, G)
    dw = dout @ v.transpose(-1, -2)
    ds = w * (dw - (dout * out).sum(-1, keepdim=True))
    return {"out": _laid_out(out, c), "dq": _laid_out((ds @ k) * t, c),
            "dk": _laid_out((ds.transpose(-1, -2) @ q).sum(2, keepdim=True), c),
            "dv": _laid_out((w.transpose(-1, -2) @ dout).sum(2, keepdim=True), c)}


def _decode_plain(s, c):
    B, H, Hkv, d = c["B"], c["H"], c["Hkv"], c["d"]
    n = s["lengths"][:, None].long()
    near = n - c["window"] + torch.arange(c["window"], device="cuda")           # the window's rows, the first key's side first
    first = torch.arange(c["sinks"], device="cuda").expand(B, -1)
    rows = torch.cat([first, near], 1)
    see = torch.cat([(first < n) & (first < n - c["window"]), near >= 0], 1)
    at = rows.clamp(0, c["Tcap"] - 1)
    b = torch.arange(B, device="cuda")[:, None]
    k, v = s["kcache"][b, :, at].transpose(1, 2), s["vcache"][b, :, at].transpose(1, 2)
    q = s["q"].reshape(B, Hkv, H // Hkv, d) * d ** -0.5
    w = _softmax(q @ k.transpose(-1, -2), see[:, None, None])
    return {"out": (w @ v).reshape(B, H, 1, d)}


def _turned(x, c, angle, amplitude, inverse=False):
    """x with its first `rot` columns turned by `angle` (turns, 64 bits, [B, L, rot / 2])."""
    angle = (angle - angle.floor()) * (2 * math.pi)
    cos, sin = (torch.cos(angle) * amplitude).float(), (torch.sin(angle) * amplitude).float()
    if inverse:
        sin = -sin
    cos, sin = (t.unsqueeze(2 if c["token_major"] else 1) for t in (cos, sin))
    h = c["rot"] // 2
    a, b = (x[..., 0:c["rot"]:2], x[..., 1:c["rot"]:2]) if c["interleaved"] else (x[..., :h], x[..., h:c["rot"]])
    y, z = a * cos - b * sin, a * sin + b * cos
    front = torch.stack([y, z], -1).flatten(-2) if c["interleaved"] else torch.cat([y, z], -1)
    return torch.cat([front, x[..., c["rot"]:]], -1)


def _append_plain(s, c):
    rows = s["starts"][:, None].long() + torch.arange(c["L"], device="cuda")
    angle = rows[..., None].double() * s["turns"]
    k, v = _turned(s["k"], c, angle, s["amplitude"]), s["v"]
    if not c["token_major"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    b = torch.arange(c["B"], device="cuda")[:, None]
    s["kcache"][b, :, rows] = k
    s["vcache"][b, :, rows] = v
    return {"q": _turned(s["q"], c, angle, s["amplitude"]), "kcache": s["kcache"], "vcache": s["vcache"]}


def _rotary_plain(s, c):
    angle = s["positions"][..., None].double() * s["turns"]
    return {x: _turned(s[x], c, angle, s["amplitude"], c["inverse"]) for x in ("q", "k")}


def _logprobs_plain(s, c):
    n, t = c["n"], s["targets"].long()
    scaled = s["logits"][:, :n] * (1 / c["temp"]) + 0.0         # + 0: the two zeros are one value
    z = scaled - scaled.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    p, log_total = e / total, torch.log(total)
    given = (t >= 0)
    at = torch.where(given, t, 0)[:, None]
    entropy = log_total[:, 0] - torch.where(p > 0, p * z, 0.0).sum(-1)
    r = {"logprobs": torch.where(given, (z.gather(1, at) - log_total)[:, 0], 0.0), "entropy": entropy}
    if c["top"]:
        bits = scaled.contiguous().view(torch.int32).long()      # whole numbers in the order of the scaled logits, ...
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        order = (order << 32) - torch.arange(n, device="cuda")   # ... of equal ones the first token before the others
        top = torch.topk(order, c["top"], dim=1)[1]
        r.update(top_logprobs=z.gather(1, top) - log_total, top_tokens=top.int())
    if c["train"]:
        log_p = z - log_total
        g = torch.where(given, s["dlogprobs"], 0.0)[:, None]
        d = -p * (g + s["dentropy"][:, None] * (log_p + entropy[:, None]))
        d = d.scatter_add(1, at, g) * (1 / c["temp"])
        r["dlogits"] = torch.cat([d, torch.zeros(c["rows"], c["stride"] - n, device="cuda")], 1)
    return r


_plain = {"window": _window_plain, "decode": _decode_plain, "append": _append_plain, "rotary": _rotary_plain,
          "logprobs": _logprobs_plain}


# ------------------------------------------------------------------------------------------------------ the package's calls

def _address(t):
    return None if t is None else t.data_ptr()


def _window_own(s, c, ctx, lib):
    a = {x: _address(t) for x, t in s.items() if isinstance(t, torch.Tensor)}
    desc = ctx.window_desc(c["window"], sinks=c["sinks"], q_offset=c["Lk"] - c["Lq"], lengths=a.get("lengths"))
    flags = lib.SDPA_TOKEN_MAJOR if c["token_major"] else 0
    shape = (c["B"], c["H"], c["Hkv"], c["Lq"], c["Lk"], c["d"], c["d"] ** -0.5, desc, flags)
    ctx.sdpa_window_fwd(a["q"], a["k"], a["v"], a["out"], a.get("stats"), *shape)
    if not c["train"]:
        return {"out": s["out"]}
    ctx.sdpa_window_bwd(a["q"], a["k"], a["v"], a["out"], a["stats"], a["dout"], a["dq"], a["dk"], a["dv"], *shape)
    return {x: s[x] for x in ("out", "dq", "dk", "dv")}


def _decode_own(s, c, ctx, lib):
    ctx.sdpa_window_decode(_address(s["q"]), _address(s["kcache"]), _address(s["vcache"]), _address(s["out"]), c["B"], c["H"],
                           c["Hkv"], c["T"], c["Tcap"], c["d"], c["d"] ** -0.5, c["window"], c["sinks"], _address(s["lengths"]))
    return {"out": s["out"]}


def _rotary_flags(c, lib):
    return ((lib.ROTARY_INTERLEAVED if c["interleaved"] else 0) | (lib.ROTARY_TOKEN_MAJOR if c["token_major"] else 0)
            | (lib.ROTARY_INVERSE if c.get("inverse") else 0))


def _append_own(s, c, ctx, lib):
    a = {x: _address(t) for x, t in s.items() if isinstance(t, torch.Tensor)}
    ctx.rotary_append(a["q"], a["k"], a["v"], a["q_out"], a["kcache"], a["vcache"], c["B"], c["L"], c["H"], c["Hkv"], c["Tcap"],
                      c["d"], c["rot"], a["turns"], a["starts"], amplitude=s["amplitude"], flags=_rotary_flags(c, lib))
    return {"q": s["q_out"], "kcache": s["kcache"], "vcache": s["vcache"]}


def _rotary_own(s, c, ctx, lib):
    a = {x: _address(t) for x, t in s.items() if isinstance(t, torch.Tensor)}
    ctx.rotary(a["q"], a["q_out"], a["k"], a["k_out"], c["B"], c["L"], c["H"], c["Hkv"], c["d"], c["rot"], a["turns"],
               positions=a["positions"], amplitude=s["amplitude"], flags=_rotary_flags(c, lib))
    return {"q": s["q_out"], "k": s["k_out"]}


def _logprobs_own(s, c, ctx, lib):
    a = {x: _address(t) for x, t in s.items() if isinstance(t, torch.Tensor)}
    shape = (c["rows"], c["n"], c["stride"])
    ctx.token_logprobs(a["logits"], *shape, a["targets"], a["logprobs"], entropy=a["entropy"], stats=a.get("stats"),
                       inv_temperature=1 / c["temp"], ignore_index=-1, top_k=c["top"], top_logprobs=a.get("top_logprobs"),
                       top_tokens=a.get("top_tokens"))
    if c["train"]:
        ctx.token_logprobs_bwd(a["logits"], *shape, a["targets"], a["stats"], a["dlogits"], dlogprobs=a["dlogprobs"],
                               dentropy=a["dentropy"], inv_temperature=1 / c["temp"], ignore_index=-1)
    return {x: s[x] for x in ("logprobs", "entropy", "top_logprobs", "top_tokens", "dlogits") if x in s}


_own = {"window": _window_own, "decode": _decode_own, "append": _append_own, "rotary": _rotary_own, "logprobs": _logprobs_own}


def run(state):
    c = state["case"]
    if own:
        from dl4s_amd import lib
        return _own[c["op"]](state, c, _context(), lib)
    return _plain[c["op"]](state, c)


# ------------------------------------------------------------------------------------------------------ what a pass costs

def _pairs(c):
    """Visible (query, key) pairs of one head, over the batch."""
    total = 0
    for n in _lengths(c["B"], c["Lk"], c["ragged"]):
        for p in range(c["Lk"] - c["Lq"], c["Lk"]):
            low = max(0, p - c["window"] + 1)
            total += max(0, min(p + 1, n) - low) + min(c["sinks"], low, n)
    return total


def work(case):
    c = case
    if c["op"] == "window":
        q, kv = c["B"] * c["H"] * c["Lq"] * c["d"], c["B"] * c["Hkv"] * c["Lk"] * c["d"]
        flops = 2 * (7 if c["train"] else 2) * c["d"] * c["H"] * _pairs(c)
        return {"bytes": 4 * ((4 * q + 4 * kv) if c["train"] else (2 * q + 2 * kv)), "flops": flops}
    if c["op"] == "decode":
        seen = sum(min(n, c["window"]) + max(0, min(c["sinks"], n - c["window"])) for n in _lengths(c["B"], c["T"], True))
        return {"bytes": 8 * c["d"] * (c["Hkv"] * seen + c["B"] * c["H"]), "flops": 4 * c["d"] * c["H"] * seen}
    if c["op"] in ("append", "rotary"):
        tokens = c["B"] * c["L"]
        moved = c["H"] + c["Hkv"] * (2 if c["op"] == "append" else 1)
        return {"bytes": 8 * tokens * moved * c["d"], "flops": 3 * tokens * (c["H"] + c["Hkv"]) * c["rot"]}
    values = c["rows"] * c["n"]
    return {"bytes": 4 * values * (2 if c["train"] else 1) + 8 * c["rows"] * (1 + c["top"]), "flops": (9 if c["train"] else 5) * values}


# ------------------------------------------------------------------------------------------------------ 64 bits

def _exact_window(s, c):
    B, H, Hkv, G = c["B"], c["H"], c["Hkv"], c["H"] // c["Hkv"]
    per_head = lambda x: (x.permute(0, 2, 1, 3) if c["token_major"] else x).double()  # noqa: E731
    q, k, v = (per_head(s[x]).requires_grad_(c["train"]) for x in ("q", "k", "v"))
    pos = torch.arange(c["Lk"] - c["Lq"], c["Lk"], device="cuda").reshape(-1, 1)
    key = torch.arange(c["Lk"], device="cuda").reshape(1, -1)
    r = {x: torch.empty(s[y].shape, dtype=torch.float64, device="cuda") for x, y in
         (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v")) if c["train"] or x == "out"}
    view = {x: r[x].permute(0, 2, 1, 3) if c["token_major"] else r[x] for x in r}
    for b, n in enumerate(_lengths(B, c["Lk"], c["ragged"])):
        hidden = (key > pos) | ((key <= pos - c["window"]) & (key >= c["sinks"])) | (key >= n)
        empty = hidden.all(1)
        hidden_or_empty = hidden & ~empty[:, None]              # a softmax over nothing is replaced by zeros below
        for h in range(Hkv):
            kk, vv = k[b, h].detach().requires_grad_(c["train"]), v[b, h].detach().requires_grad_(c["train"])
            dk = dv = 0
            for i in range(h * G, (h + 1) * G):
                qq = q[b, i].detach().requires_grad_(c["train"])
                scores = (torch.matmul(qq, kk.t()) / math.sqrt(c["d"])).masked_fill(hidden_or_empty, -math.inf)
                o = torch.matmul(torch.softmax(scores, 1), vv).masked_fill(empty[:, None], 0.0)
                view["out"][b, i] = o.detach()
                if c["train"]:
                    up = (s["dout"][b, :, i] if c["token_major"] else s["dout"][b, i]).double()
                    gq, gk, gv = torch.autograd.grad(o, (qq, kk, vv), up)
                    view["dq"][b, i], dk, dv = gq, dk + gk, dv + gv
            if c["train"]:
                view["dk"][b, h], view["dv"][b, h] = dk, dv
    return r


def _exact_decode(s, c):
    G = c["H"] // c["Hkv"]
    out = torch.empty(c["B"], c["H"], 1, c["d"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(c["B"], c["T"], True)):
        low = max(0, n - c["window"])
        keep = list(range(min(c["sinks"], low))) + list(range(low, n))
        keep = torch.tensor(keep, device="cuda")
        k, v = s["kcache"][b].index_select(1, keep).double(), s["vcache"][b].index_select(1, keep).double()
        for h in range(c["H"]):
            weights = torch.softmax(k[h // G] @ s["q"][b, h, 0].double() / math.sqrt(c["d"]), 0)
            out[b, h, 0] = weights @ v[h // G]
    return {"out": out}


def _exact_turn(x, c, positions, turns, amplitude, sign):
    """The turned columns as complex numbers times exp(i angle); x [B, L, heads, d] in 64 bits, positions [B, L]."""
    rot = c["rot"]
    front = x[..., :rot]
    pairs = front.reshape(*front.shape[:-1], rot // 2, 2) if c["interleaved"] else front.reshape(*front.shape[:-1], 2, rot // 2).transpose(-1, -2)
    number = torch.view_as_complex(pairs.contiguous())
    angle = 2 * math.pi * torch.remainder(positions.double()[..., None] * turns, 1.0)
    number = number * torch.polar(torch.full_like(angle, amplitude), sign * angle)[:, :, None]
    pairs = torch.view_as_real(number)
    front = pairs.reshape(*front.shape) if c["interleaved"] else pairs.transpose(-1, -2).reshape(*front.shape)
    return torch.cat([front, x[..., rot:]], -1)


def _exact_rotary(s, c):
    tokens_first = lambda x: x.double() if c["token_major"] else x.double().transpose(1, 2)  # noqa: E731
    back = lambda x: x if c["token_major"] else x.transpose(1, 2).contiguous()  # noqa: E731
    if c["op"] == "rotary":
        sign = -1 if c["inverse"] else 1
        return {x: back(_exact_turn(tokens_first(s[x]), c, s["positions"], s["turns"], s["amplitude"], sign)) for x in ("q", "k")}
    positions = s["starts"].long()[:, None] + torch.arange(c["L"], device="cuda")[None]
    q, k = (_exact_turn(tokens_first(s[x]), c, positions, s["turns"], s["amplitude"], 1) for x in ("q", "k"))
    kcache, vcache, v = s["kcache"].double(), s["vcache"].double(), tokens_first(s["v"])
    for b, start in enumerate(s["starts"].tolist()):
        kcache[b, :, start:start + c["L"]] = k[b].transpose(0, 1)
        vcache[b, :, start:start + c["L"]] = v[b].transpose(0, 1)
    return {"q": back(q), "kcache": kcache, "vcache": vcache}


def _exact_logprobs(s, c):
    z = (s["logits"][:, :c["n"]].double() / c["temp"])
    log_p = torch.log_softmax(z, 1)
    p = torch.exp(log_p)
    given = s["targets"] >= 0
    at = s["targets"].long().clamp(min=0)
    entropy = -(p * log_p).sum(1)
    r = {"logprobs": log_p[torch.arange(c["rows"], device="cuda"), at] * given, "entropy": entropy}
    if c["top"]:
        r.update(top_logprobs=torch.topk(log_p, c["top"], dim=1)[0], top_tokens=None)
    if c["train"]:
        g, e = (s["dlogprobs"].double() * given)[:, None], s["dentropy"].double()[:, None]
        d = torch.zeros(c["rows"], c["stride"], dtype=torch.float64, device="cuda")
        d[:, :c["n"]] = -(p * g) - e * p * (log_p + entropy[:, None])
        d[torch.arange(c["rows"], device="cuda"), at] += g[:, 0]
        r["dlogits"] = d / c["temp"]
    return r


def exact(case, seed):
    s = prepare(case, seed)
    return {"window": _exact_window, "decode": _exact_decode, "append": _exact_rotary, "rotary": _exact_rotary,
            "logprobs": _exact_logprobs}[case["op"]](s, case)
