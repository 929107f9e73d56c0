"""The 8-bit paged KV-cache operators as they are measured: slot planning, rotary positions, quantised append, and
attention over the 8-bit cache, each in its plain form (elementary torch operations) and as a user calls it.

Layouts (those of the engine's bf16 cache, one byte per value): pages [page][K|V][kv head][16][head_dim] e4m3 codes,
scales [page][K|V][kv head] powers of two in fp32, block tables [request][width] int32, slots page * 16 + offset.
"""
import math
import zlib

import torch

own = False

PAGE = 16
E4M3_MAX = 448.0


# ---- cases -------------------------------------------------------------------------------

def listed():
    return [
        # one serving step of the 64-sequence batch: every request gets one token; pure latency
        {"name": "plan-decode-64", "op": "plan", "n": 64, "ctx_lo": 32000, "ctx_hi": 32768, "new_lo": 1, "new_hi": 1,
         "release": 0.0, "pad": 0},
        # admission of many prompts at once while finished requests return their pages
        {"name": "plan-admit-512", "op": "plan", "n": 512, "ctx_lo": 0, "ctx_hi": 3000, "new_lo": 0, "new_hi": 1000,
         "release": 0.1, "pad": 777},
        # one decode step's queries and keys at the engine's shape (a quarter of the head rotates)
        {"name": "rope-decode-64", "op": "rope", "tokens": 64, "hq": 16, "hk": 2, "d": 256, "rot": 64, "dtype": "f32",
         "layout": "half", "scaling": "none", "factor": 1.0, "theta": 1e7, "max_pos": 32768},
        # a long prompt with whole-head interleaved positions stretched past the trained context
        {"name": "rope-prefill-32771", "op": "rope", "tokens": 32771, "hq": 32, "hk": 8, "d": 128, "rot": 128,
         "dtype": "bf16", "layout": "interleaved", "scaling": "yarn", "factor": 8.0, "theta": 1e6, "max_pos": 262144},
        # one decode step of 64 sequences into pages in every state of filling
        {"name": "append-decode-64", "op": "append", "n": 64, "ctx_lo": 0, "ctx_hi": 2000, "new_lo": 1, "new_hi": 1,
         "hk": 2, "d": 256, "dtype": "bf16"},
        # ragged prompts at the engine's shape
        {"name": "append-prefill-7", "op": "append", "n": 7, "ctx_lo": 0, "ctx_hi": 500, "new_lo": 1500,
         "new_hi": 3500, "hk": 2, "d": 256, "dtype": "bf16"},
        # many short prompts of a small model in fp32
        {"name": "append-f32-300", "op": "append", "n": 300, "ctx_lo": 0, "ctx_hi": 40, "new_lo": 0, "new_hi": 90,
         "hk": 4, "d": 64, "dtype": "f32"},
        # one sequence, one token: the single-sequence decode step
        {"name": "decode-1x4096", "op": "attn", "n": 1, "len_lo": 4096, "len_hi": 4096, "q_lo": 1, "q_hi": 1,
         "hk": 2, "group": 8, "d": 256, "dtype": "f32"},
        # the batched decode step at its benchmark shape
        {"name": "decode-64x32768", "op": "attn", "n": 64, "len_lo": 32768, "len_hi": 32768, "q_lo": 1, "q_hi": 1,
         "hk": 2, "group": 8, "d": 256, "dtype": "bf16"},
        # ragged decode of a small model, empty requests among them
        {"name": "decode-ragged-48", "op": "attn", "n": 48, "len_lo": 0, "len_hi": 6000, "q_lo": 1, "q_hi": 1,
         "hk": 1, "group": 4, "d": 64, "dtype": "bf16"},
        # prompts of the prefill benchmark's length
        {"name": "prefill-4x8192", "op": "attn", "n": 4, "len_lo": 8192, "len_hi": 8192, "q_lo": 8192, "q_hi": 8192,
         "hk": 2, "group": 8, "d": 256, "dtype": "bf16"},
        # chunks of new tokens on cached contexts, fp32 activations
        {"name": "extend-ragged-5", "op": "attn", "n": 5, "len_lo": 700, "len_hi": 5000, "q_lo": 1, "q_hi": 300,
         "hk": 8, "group": 4, "d": 128, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "append", "attn", "attn"])
    if op == "plan":
        decode = rng.random() < 0.5
        n = _log(rng, 1, 2000) if decode else _log(rng, 1, 600)
        ctx = _log(rng, 1, 20000) if decode else _log(rng, 1, 4000)
        return {"op": "plan", "n": n, "ctx_lo": 0, "ctx_hi": ctx, "new_lo": 1 if decode else 0,
                "new_hi": 1 if decode else _log(rng, 2, 1000), "release": rng.choice([0.0, 0.05, 0.3]),
                "pad": rng.choice([0, 1, 100])}
    if op == "rope":
        d = rng.choice([64, 128, 256])
        hk = rng.choice([1, 2, 4, 8])
        tokens = _log(rng, 1, max(2, min(32000, 32771 * 40 * 128 // (hk * 5 * d))))
        return {"op": "rope", "tokens": tokens, "hq": hk * rng.choice([1, 3, 4]), "hk": hk, "d": d,
                "rot": rng.choice([d, d // 2, d // 4]), "dtype": rng.choice(["bf16", "f32"]),
                "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(["none", "linear", "yarn"]),
                "factor": rng.choice([2.0, 4.0, 8.0]), "theta": rng.choice([1e4, 1e6, 1e7]),
                "max_pos": _log(rng, 512, 1000000)}
    d = rng.choice([64, 128, 256])
    hk = rng.choice([1, 2, 4, 8])
    dtype = rng.choice(["bf16", "f32"])
    if op == "append":
        new_hi = rng.choice([1, _log(rng, 2, 2000)])
        n = _log(rng, 1, max(2, min(500, 24000 * 512 // (hk * d * new_hi))))
        return {"op": "append", "n": n, "ctx_lo": 0, "ctx_hi": _log(rng, 1, 2000), "new_lo": rng.choice([0, 1]),
                "new_hi": new_hi, "hk": hk, "d": d, "dtype": dtype}
    group = rng.choice([1, 2, 3, 4, 6, 8, 16])
    if rng.random() < 0.6:  # decode: at most half a GB of cache
        most = 500_000_000 // (2 * hk * d)
        len_hi = _log(rng, 1, 40000)
        n = _log(rng, 1, max(2, min(300, most // len_hi)))
        return {"op": "attn", "n": n, "len_lo": rng.choice([0, len_hi // 2, len_hi]), "len_hi": len_hi, "q_lo": 1,
                "q_hi": 1, "hk": hk, "group": group, "d": d, "dtype": dtype}
    q_hi = _log(rng, 2, 1500)
    len_hi = q_hi + rng.choice([0, _log(rng, 1, 4000)])
    n = _log(rng, 1, 8)
    return {"op": "attn", "n": n, "len_lo": q_hi, "len_hi": len_hi, "q_lo": rng.choice([0, 1, q_hi]), "q_hi": q_hi,
            "hk": hk, "group": group, "d": d, "dtype": dtype}


# ---- inputs ------------------------------------------------------------------------------

def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _ints(case, seed):
    """The request lengths of a case: the case's own mix, in the order that the seed gives."""
    g = torch.Generator().manual_seed(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))
    n = case["n"]

    def between(lo, hi):
        return torch.randint(lo, hi + 1, (n,), generator=g)

    if case["op"] == "attn":
        a, b = between(case["len_lo"], case["len_hi"]), between(case["q_lo"], case["q_hi"])
        a[0] = max(1, a[0])
    else:
        a, b = between(case["ctx_lo"], case["ctx_hi"]), between(case["new_lo"], case["new_hi"])
        if case["op"] == "plan":
            b[torch.rand(n, generator=g) < case["release"]] = -1
    if case["op"] != "plan":
        b[0] = max(1, b[0])  # never without a token
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed))
    return a[order], b[order]


def _codes(shape, gen):
    """e4m3 codes as a cache holds them: each block's largest value near the top of the range."""
    n = math.prod(shape)
    out = torch.empty(n, dtype=torch.uint8, device="cuda")
    step = 1 << 27
    for a in range(0, n, step):
        b = min(n, a + step)
        x = torch.randn(b - a, generator=gen, device="cuda").mul_(100.0).clamp_(-E4M3_MAX, E4M3_MAX)
        out[a:b] = x.to(torch.float8_e4m3fn).view(torch.uint8)
    return out.view(shape)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    s = {"case": case}
    if case["op"] == "rope":
        t, dt = case["tokens"], _dtype(case)
        s["q"] = torch.randn(t, case["hq"], case["d"], generator=gen, device=dev).to(dt)
        s["k"] = torch.randn(t, case["hk"], case["d"], generator=gen, device=dev).to(dt)
        s["positions"] = torch.randint(0, case["max_pos"], (t,), generator=gen, device=dev, dtype=torch.int32)
        s["freq"], s["mscale"] = _frequencies(case)
        s["freq"] = s["freq"].to(dev)
        if own:
            from disk_streaming_moe_engine_b200 import kv8
            s["plan"] = kv8.RopePlan(case["d"], case["rot"], theta=case["theta"], layout=case["layout"],
                                     scaling=case["scaling"], factor=case["factor"], original_context=32768)
        return s
    if case["op"] == "plan":
        ctx, new = _ints(case, seed)
        have = (ctx + PAGE - 1) // PAGE
        width = int(((ctx + new.clamp(min=0) + PAGE - 1) // PAGE).max()) + 1
        grow = int(((ctx + new.clamp(min=0) + PAGE - 1) // PAGE - have).sum())
        pages = int(have.sum()) + grow + 64
        perm = torch.randperm(pages, generator=gen, device=dev, dtype=torch.int32)
        used = torch.arange(width)[None, :] < have[:, None]
        table = torch.full((case["n"], width), -1, dtype=torch.int32, device=dev)
        table[used.to(dev)] = perm[:int(have.sum())]
        count = pages - int(have.sum())
        free = torch.full((pages,), -1, dtype=torch.int32, device=dev)
        free[:count] = perm[int(have.sum()):]
        s.update(free=free, table=table, ctx=ctx.to(dev, torch.int32), new=new.to(dev, torch.int32),
                 state=torch.tensor([count, 0], dtype=torch.int32, device=dev),
                 state_out=torch.zeros(2, dtype=torch.int32, device=dev),
                 max_tokens=max(1, int(new.clamp(min=0).sum()) + case["pad"]))
        return s
    hk, d = case["hk"], case["d"]
    a, b = _ints(case, seed)
    if case["op"] == "append":
        total = a + b
        t = int(b.sum())
        s["k"] = torch.randn(t, hk, d, generator=gen, device=dev).mul_(1.5).to(_dtype(case))
        s["v"] = torch.randn(t, hk, d, generator=gen, device=dev).mul_(0.7).to(_dtype(case))
    else:
        total = a
        t = int(b.sum())
        s["q"] = torch.randn(t, hk * case["group"], d, generator=gen, device=dev).to(_dtype(case))
        s["lens"], s["rows"] = a.tolist(), b.tolist()
        s["seq_lens"] = a.to(dev, torch.int32)
        s["cu_q"] = torch.cat([torch.zeros(1, dtype=torch.long), b.cumsum(0)]).to(dev, torch.int32)
        s["max_q"] = int(b.max())
        s["sm_scale"] = 1.0 / math.sqrt(d)
    have = (total + PAGE - 1) // PAGE
    pages = max(1, int(have.sum()))
    width = max(1, int(have.max()))
    perm = torch.randperm(pages, generator=gen, device=dev, dtype=torch.int32)
    used = torch.arange(width)[None, :] < have[:, None]
    table = torch.zeros((case["n"], width), dtype=torch.int32, device=dev)
    table[used.to(dev)] = perm[:int(have.sum())]
    s["table"] = table
    s["pages"] = _codes((pages, 2, hk, PAGE, d), gen)
    s["scales"] = torch.exp2(torch.randint(-9, -6, (pages, 2, hk), generator=gen, device=dev).float())
    if case["op"] == "append":
        req = torch.repeat_interleave(torch.arange(case["n"]), b)
        start = torch.cat([torch.zeros(1, dtype=torch.long), b.cumsum(0)])[:-1]
        pos = torch.arange(t) - start[req] + a[req]
        req, pos = req.to(dev), pos.to(dev)
        s["slots"] = (table[req, pos // PAGE] * PAGE + (pos % PAGE)).to(torch.int32)
    if own:
        from disk_streaming_moe_engine_b200 import kv8
        s["cache"] = kv8.Kv8Cache(s["pages"], s["scales"])
        if case["op"] == "attn":
            s["workspace"] = kv8.attention_workspace(s["cache"])
    return s


# ---- the operators -----------------------------------------------------------------------

def run(state):
    case = state["case"]
    return {"plan": _plan, "rope": _rope, "append": _append, "attn": _attn}[case["op"]](state, case)


def _plan(s, case):
    if own:
        from disk_streaming_moe_engine_b200 import kv8
        p = kv8.plan_slots(s["free"], s["state"], s["table"], s["ctx"], s["new"], s["max_tokens"],
                           state_out=s["state_out"])
        return {"seq_lens": p.seq_lens, "cu_new": p.cu_new, "slots": p.slots, "positions": p.positions,
                "requests": p.requests, "table": s["table"], "free": s["free"], "count": s["state_out"][:1]}
    ctx, new, table, free, count = s["ctx"].long(), s["new"].long(), s["table"], s["free"], s["state"][0].long()
    n, width = table.shape
    rel = new < 0
    add_tok = new.clamp(min=0)
    have = (ctx + PAGE - 1) // PAGE
    need = (ctx + add_tok + PAGE - 1) // PAGE
    add = torch.where(rel, 0, need - have)
    back = torch.where(rel, have, 0)
    cu_new = torch.cat([add_tok.new_zeros(1), add_tok.cumsum(0)])
    add0, back0 = add.cumsum(0) - add, back.cumsum(0) - back
    r, m = back.sum(), add.sum()
    p = torch.arange(width, device=ctx.device)[None, :]
    stack = torch.cat([free, free.new_zeros(1)])
    dest = torch.where(rel[:, None] & (p < have[:, None]), count + back0[:, None] + p, free.numel())
    stack.scatter_(0, dest.reshape(-1), table.reshape(-1))
    fresh = (p >= have[:, None]) & (p < need[:, None]) & ~rel[:, None]
    pop = (count + r - 1 - (add0[:, None] + p - have[:, None])).clamp(0, free.numel())
    table = torch.where(fresh, stack[pop], table)
    t = torch.arange(s["max_tokens"], device=ctx.device)
    live = t < cu_new[-1]
    req = torch.searchsorted(cu_new[1:].contiguous(), t, right=True).clamp(max=n - 1)
    pos = ctx[req] + t - cu_new[req]
    page = table[req, (pos // PAGE).clamp(0, width - 1)].long()
    i = torch.arange(free.numel(), device=ctx.device)
    left = torch.where((i >= count) & (i < count + r - m), stack[:-1], free)
    as32 = lambda x: torch.where(live, x, -1).to(torch.int32)
    return {"seq_lens": torch.where(rel, 0, ctx + add_tok).to(torch.int32), "cu_new": cu_new.to(torch.int32),
            "slots": as32(page * PAGE + pos % PAGE), "positions": as32(pos), "requests": as32(req), "table": table,
            "free": left, "count": (count + r - m).to(torch.int32).reshape(1)}


def _frequencies(case):
    """Angles per position of the rotating pairs (64 bits), and the factor on the rotated values."""
    rot, theta, f = case["rot"], case["theta"], case["factor"]
    i = torch.arange(rot // 2, dtype=torch.float64)
    freq = theta ** (-2.0 * i / rot)
    if case["scaling"] == "linear":
        return freq / f, 1.0
    if case["scaling"] == "yarn":  # pairs that turn often keep their angle, pairs that hardly turn are stretched
        def pair(turns):
            return rot * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(theta))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return freq * (1 - ramp) + freq / f * ramp, 0.1 * math.log(f) + 1.0
    return freq, 1.0


def _rotate(x, cos, sin, rot, layout):
    x1, x2 = (x[..., :rot // 2], x[..., rot // 2:rot]) if layout == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    y = torch.cat([y1, y2], -1) if layout == "half" else torch.stack([y1, y2], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _rope(s, case):
    if own:
        from disk_streaming_moe_engine_b200 import kv8
        q, k = kv8.rope(s["plan"], s["q"], s["k"], s["positions"])
        return {"q": q, "k": k}
    angle = (s["positions"].double()[:, None] * s["freq"])[:, None, :]
    cos, sin = (torch.cos(angle) * s["mscale"]).float(), (torch.sin(angle) * s["mscale"]).float()
    return {n: _rotate(s[n].float(), cos, sin, case["rot"], case["layout"]).to(s[n].dtype) for n in ("q", "k")}


def _append(s, case):
    if own:
        from disk_streaming_moe_engine_b200 import kv8
        kv8.append(s["cache"], s["k"], s["v"], s["slots"])
        return {"pages": s["pages"].view(torch.float8_e4m3fn), "scales": s["scales"]}
    pages, scales, slots = s["pages"], s["scales"], s["slots"].long()
    if slots.numel():
        x = torch.stack([s["k"], s["v"]], 1).float()  # [t][K|V][head][d]
        page, off = slots // PAGE, slots % PAGE
        lead = torch.cat([torch.ones_like(page[:1], dtype=torch.bool), page[1:] != page[:-1]])
        run = lead.cumsum(0) - 1
        t = torch.arange(slots.numel(), device=slots.device)
        # per run of tokens in one page: its page, the offset of its first token, its largest value
        first = torch.zeros_like(page).scatter_add_(0, run, torch.where(lead, off, 0))
        where = torch.zeros_like(page).scatter_add_(0, run, torch.where(lead, page, 0))
        each = run[:, None, None].expand(-1, *x.shape[1:3])
        amax = torch.zeros(each.shape, device=x.device).scatter_reduce_(0, each, x.abs().amax(-1), "amax")
        m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
        want = torch.where(amax > 0, torch.ldexp(torch.ones_like(m), (e - 9 + (m > 0.875)).clamp(-100, 100)), 2.0 ** -100)
        old = scales[where]
        scale = torch.where((first > 0)[:, None, None], torch.maximum(want, old), want)
        # tokens that the pages held before the run, rounded again where the scale grew
        keep = torch.arange(PAGE, device=x.device)[None, :] < first[:, None]
        held = pages[where].view(torch.float8_e4m3fn).float() * (old / scale)[..., None, None]
        live = t <= run[-1]
        rows = torch.where(keep[:, None, None, :, None], held.to(torch.float8_e4m3fn).view(torch.uint8), pages[where])
        # runs behind the last one repeat the last one's row
        at = torch.where(live, t, run[-1])
        pages[where[at]] = rows[at]
        scales[where[at]] = scale[at]
        codes = (x / scale[run][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
        pages[page, :, :, off] = codes
    return {"pages": pages.view(torch.float8_e4m3fn), "scales": scales}


def _visible(m, length, rows, device):
    """Query j of the request's `rows` sees the keys before length - rows + j + 1."""
    return torch.arange(length, device=device)[None, :] <= torch.arange(m[0], m[1], device=device)[:, None] + (length - rows)


def _attn(s, case):
    if own:
        from disk_streaming_moe_engine_b200 import kv8
        return kv8.attention(s["cache"], s["q"], s["table"], s["seq_lens"], cu_q=s["cu_q"], max_q_len=s["max_q"],
                             sm_scale=s["sm_scale"], workspace=s["workspace"])
    return _attend(s, case, torch.float32).to(s["q"].dtype)


def _attend(s, case, dt):
    q, hk, grp, d = s["q"], case["hk"], case["group"], case["d"]
    out = torch.zeros(q.shape, dtype=dt, device=q.device)
    at = 0
    for i, (length, rows) in enumerate(zip(s["lens"], s["rows"])):
        if rows and length:
            ids = s["table"][i, :(length + PAGE - 1) // PAGE].long()
            kv = s["pages"][ids].view(torch.float8_e4m3fn).to(dt) * s["scales"][ids].to(dt)[..., None, None]
            kv = kv.permute(1, 2, 0, 3, 4).reshape(2, hk, -1, d)[:, :, :length]  # [K|V][head][token][d]
            step = max(1, min(rows, (1 << 28) // (length * grp)))
            for a in range(0, rows, step):
                b = min(rows, a + step)
                end = min(length, max(1, length - rows + b))  # keys behind the last of these queries count for none
                see = _visible((a, b), length, rows, q.device)[:, :end]
                for h in range(hk):
                    x = q[at + a:at + b, h * grp:(h + 1) * grp].to(dt).reshape(-1, d)
                    sc = (x @ kv[0, h, :end].T).mul_(s["sm_scale"]).view(b - a, grp, end)
                    sc.masked_fill_(~see[:, None, :], -math.inf)
                    sc.sub_(sc.amax(-1, keepdim=True).clamp(min=torch.finfo(dt).min)).exp_()
                    total = sc.sum(-1, keepdim=True)
                    y = (sc.view(-1, end) @ kv[1, h, :end]).view(b - a, grp, d)
                    out[at + a:at + b, h * grp:(h + 1) * grp] = y / total.clamp(min=torch.finfo(dt).tiny)
        at += rows
    return out


# ---- the definitions in 64 bits ------------------------------------------------------------

def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(s, case)
    if case["op"] == "append":
        return _exact_append(s, case)
    return _exact_attn(s, case)


def _exact_rope(s, case):
    """Pairs as complex numbers times e^{i angle}."""
    turn = torch.polar(torch.full_like(s["freq"], s["mscale"])[None, :].expand(case["tokens"], -1).contiguous(),
                       s["positions"].double()[:, None] * s["freq"][None, :])[:, None, :]
    out = {}
    for n in ("q", "k"):
        x = s[n].double()
        part = x[..., :case["rot"]]
        if case["layout"] == "half":
            a, b = part.chunk(2, -1)
        else:
            a, b = part.unflatten(-1, (-1, 2)).unbind(-1)
        z = torch.complex(a.contiguous(), b.contiguous()) * turn
        y = x.clone()
        if case["layout"] == "half":
            y[..., :case["rot"] // 2], y[..., case["rot"] // 2:case["rot"]] = z.real, z.imag
        else:
            y[..., 0:case["rot"]:2], y[..., 1:case["rot"]:2] = z.real, z.imag
        out[n] = y
    return out


def _to_e4m3(x):
    """Nearest value with 3 mantissa bits and exponents from -6 (ties to even), in 64 bits."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def _exact_append(s, case):
    pages = s["pages"].view(torch.float8_e4m3fn).double()
    scales = s["scales"].double()
    x = torch.stack([s["k"], s["v"]], 1).double()
    slots = s["slots"].tolist()
    a = 0
    while a < len(slots):
        page, off = divmod(slots[a], PAGE)
        b = a
        while b < len(slots) and slots[b] // PAGE == page:
            b += 1
        new = x[a:b].permute(1, 2, 0, 3)  # [K|V][head][token][d]
        amax = new.abs().amax((-1, -2))
        half, e = torch.frexp((amax / E4M3_MAX).clamp(min=2.0 ** -100))
        want = torch.ldexp(torch.ones_like(half), e - (half == 0.5).to(e.dtype))  # the power of two at or above it
        if off:
            scale = torch.maximum(scales[page], want)
            pages[page, :, :, :off] = _to_e4m3(pages[page, :, :, :off] * (scales[page] / scale)[..., None, None])
        else:
            scale = want
        scales[page] = scale
        pages[page, :, :, off:off + b - a] = _to_e4m3(new / scale[..., None, None])
        a = b
    return {"pages": pages, "scales": scales}


def _exact_attn(s, case):
    hk, grp, d = case["hk"], case["group"], case["d"]
    if sum(m * n for m, n in zip(s["lens"], s["rows"])) * hk * grp * d * 4 > 6e12:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    cu = s["cu_q"].tolist()
    for i, length in enumerate(s["lens"]):
        rows = cu[i + 1] - cu[i]
        if rows == 0 or length == 0:
            continue
        k = torch.empty(length, hk, d, dtype=torch.float64, device="cuda")
        v = torch.empty_like(k)
        pos = torch.arange(length, device="cuda")
        ids, off = s["table"][i].long()[pos // PAGE], pos % PAGE
        for c, dst in ((0, k), (1, v)):
            dst.copy_(s["pages"].view(torch.float8_e4m3fn)[ids, c, :, off].double() * s["scales"][ids, c].double()[..., None])
        step = max(1, (1 << 26) // (length * grp))
        for a in range(0, rows, step):
            q = s["q"][cu[i] + a:min(cu[i + 1], cu[i] + a + step)].double().unflatten(1, (hk, grp))
            w = torch.einsum("thgd,khd->htgk", q, k) * s["sm_scale"]
            last = length - rows + a + torch.arange(q.shape[0], device="cuda")
            w = w.masked_fill((pos[None, :] > last[:, None])[None, :, None, :], -math.inf)
            w = torch.softmax(w, -1).nan_to_num(0.0)
            out[cu[i] + a:cu[i] + a + q.shape[0]] = torch.einsum("htgk,khd->thgd", w, v).flatten(1, 2)
    return out


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "rope":
        values = case["tokens"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * size * values + 4 * case["tokens"],
                "flops": 3 * case["tokens"] * (case["hq"] + case["hk"]) * case["rot"]}
    n = case["n"]
    if case["op"] == "attn":
        mid, rows = (case["len_lo"] + case["len_hi"]) / 2, (case["q_lo"] + case["q_hi"]) / 2
        hq = case["hk"] * case["group"]
        pairs = rows * (mid - (rows - 1) / 2) if mid >= rows else rows * mid
        cache = n * 2 * case["hk"] * (mid * case["d"] + 4 * math.ceil(mid / PAGE))
        return {"bytes": int(cache + 2 * n * rows * hq * case["d"] * size + 4 * n * math.ceil(mid / PAGE)),
                "flops": int(4 * n * hq * case["d"] * pairs)}
    tokens = n * (max(case["new_lo"], 0) + case["new_hi"]) / 2
    if case["op"] == "append":
        touched = max(1, tokens / PAGE + n / 2)
        return {"bytes": int(tokens * 2 * case["hk"] * case["d"] * (size + 1) + 4 * tokens + touched * 2 * case["hk"] * 8),
                "flops": int(tokens * 2 * case["hk"] * case["d"] * 2)}
    return {"bytes": int(8 * n + 8 * n + 12 * (tokens + case["pad"]) + 8 * tokens / PAGE + 8),
            "flops": int(4 * (tokens + n))}
