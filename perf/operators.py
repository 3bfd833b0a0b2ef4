"""Going on with cached sequences by a chunk of new tokens: rotary positions, the append to the paged cache, and the attention over it.

The cases are steps of a decoder with 28 query heads on 4 key/value heads of 128 (and of one with heads of 64): single tokens, a few
drafted tokens, portions of prompts behind a cached context, long contexts. The cache is [pages, 2 (keys, values), key/value heads, rows
of a page, head] with a table of pages per sequence."""
import math

import torch

own = False

DEVICE = "cuda"


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the newest token of one sequence: latency only
        dict(name="rotate one token", op="rotary", T=1, heads=32, head=128, rot=128, halves=True, back=False, dtype="bf16", first=4093, scaling="none"),
        # fp32 rows of heads of 64 of which half is rotated, pairs side by side, rotated back (keys that move, or a gradient)
        dict(name="rotate back 777 fp32 pairs", op="rotary", T=777, heads=17, head=64, rot=32, halves=False, back=True, dtype="fp32", first=0, scaling="linear"),
        # a long portion at far positions of a context that was stretched
        dict(name="rotate 32768 stretched", op="rotary", T=32768, heads=32, head=128, rot=128, halves=True, back=False, dtype="bf16", first=98304, scaling="yarn"),
        # a step of 32 sequences, a token each
        dict(name="append 32 tokens", op="append", seqs=32, new=1, behind=1024, ragged=True, hq=28, hkv=4, head=128, rot=128, halves=True, page=64, scaling="none"),
        # portions of five prompts, pairs, part of the head, small pages
        dict(name="append 5 portions pairs", op="append", seqs=5, new=411, behind=2000, ragged=True, hq=16, hkv=16, head=64, rot=48, halves=False, page=16, scaling="linear"),
        # long portions of four prompts
        dict(name="append 4 x 4096", op="append", seqs=4, new=4096, behind=4096, ragged=False, hq=28, hkv=4, head=128, rot=128, halves=True, page=64, scaling="yarn"),
        # one token behind a prompt with an image
        dict(name="attend 1 x 1 behind 1087", op="attend", seqs=1, new=1, behind=1087, ragged=False, hq=28, hkv=4, head=128, page=64),
        # a batched step of single tokens over contexts of many lengths
        dict(name="attend 32 x 1 behind 4096", op="attend", seqs=32, new=1, behind=4096, ragged=True, hq=28, hkv=4, head=128, page=64),
        # a few drafted tokens per sequence to be looked through, heads of 64, odd lengths and small pages
        dict(name="attend 8 x 5 behind 1531", op="attend", seqs=8, new=5, behind=1531, ragged=True, hq=14, hkv=2, head=64, page=16),
        # the next portion of one prompt
        dict(name="attend 512 behind 4096", op="attend", seqs=1, new=512, behind=4096, ragged=False, hq=28, hkv=4, head=128, page=64),
        # portions of several prompts
        dict(name="attend 4 x 2048 behind 2048", op="attend", seqs=4, new=2048, behind=2048, ragged=True, hq=28, hkv=4, head=128, page=64),
        # the last portion of a long prompt
        dict(name="attend 2048 behind 28672", op="attend", seqs=1, new=2048, behind=28672, ragged=False, hq=28, hkv=4, head=128, page=64),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend"])
    head = rng.choice([64, 128, 128])
    if op == "rotary":
        return dict(op=op, T=_log(rng, 1, 32768), heads=rng.randint(1, 32), head=head, rot=rng.choice([head, head // 2, 24]), halves=rng.random() < 0.5,
                    back=rng.random() < 0.3, dtype=rng.choice(["bf16", "fp32"]), first=_log(rng, 1, 400000), scaling=rng.choice(["none", "linear", "yarn"]))
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 4, 7, 8])
    page = rng.choice([16, 24, 64, 64, 128])
    seqs = _log(rng, 1, 32)
    if op == "append":
        new = _log(rng, 1, max(1, 16384 // seqs))
        return dict(op=op, seqs=seqs, new=new, behind=_log(rng, 1, 4096), ragged=rng.random() < 0.7, hq=hq, hkv=hkv, head=head, rot=rng.choice([head, head // 2]),
                    halves=rng.random() < 0.5, page=page, scaling=rng.choice(["none", "linear", "yarn"]))
    new = 1 if rng.random() < 0.3 else _log(rng, 1, max(1, 4096 // seqs))
    behind = _log(rng, 1, 8192 if seqs <= 8 else 4096)
    while seqs * new * hq * (new + behind) * head > 28 * 2048 * 30000 * 128 // 2:
        new = max(1, new // 2)
    return dict(op=op, seqs=seqs, new=new, behind=behind, ragged=rng.random() < 0.7, hq=hq, hkv=hkv, head=head, page=page)


def _lengths(case):
    """New tokens and whole contexts of every sequence: with `ragged` from about a third of the case's numbers up to them, by a fixed rule of the case."""
    new, ctx = [], []
    for s in range(case["seqs"]):
        part = 1.0 if not case["ragged"] or s == 0 else 0.3 + 0.7 * ((s * 61 + case["behind"]) % 97) / 97
        n = max(1, int(case["new"] * part))
        new.append(n)
        ctx.append(n + int(case["behind"] * (1.0 if not case["ragged"] or s == 0 else 0.3 + 0.7 * ((s * 37 + 11) % 89) / 89)))
    return new, ctx


def _turns(rot, scaling):
    """Frequencies in turns per position (float64), and the factor on cosine and sine."""
    theta, span = 1e6, 32768.0
    inv = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    m = 1.0
    if scaling == "linear":
        inv = [f / 4.0 for f in inv]
    elif scaling == "yarn":
        # slow frequencies (less than one turn over the trained span) by a factor of four, fast ones (over 32 turns) as they are, a ramp between
        at = lambda turns: rot * math.log(span / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(0, math.floor(at(32.0))), min(rot - 1, math.ceil(at(1.0)))
        ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 1e-3))) for i in range(rot // 2)]
        inv = [f / 4.0 * r + f * (1 - r) for f, r in zip(inv, ramp)]
        m = 0.1 * math.log(4.0) + 1.0
    return torch.tensor([f / (2 * math.pi) for f in inv], dtype=torch.float64), m


# ---------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, device=DEVICE, generator=g)  # noqa: E731
    if case["op"] == "rotary":
        dtype = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
        turns, m = _turns(case["rot"], case["scaling"])
        return dict(case=case, x=normal(case["T"], case["heads"] * case["head"]).to(dtype),
                    pos=(torch.arange(case["T"], device=DEVICE) + case["first"] + seed % 7).to(torch.int32), turns=turns.to(DEVICE), m=m)
    new, ctx = _lengths(case)
    hq, hkv, d, page, T = case["hq"], case["hkv"], case["head"], case["page"], sum(new)
    max_pages = (max(ctx) + page - 1) // page
    pages = case["seqs"] * max_pages
    order = torch.randperm(pages, device=DEVICE, generator=g)
    state = dict(case=case, table=order.to(torch.int32).view(case["seqs"], max_pages), max_new=max(new), max_ctx=max(ctx))
    # channels of queries and keys are of different size, as a trained projection leaves them
    size = torch.exp(0.5 * normal(d))
    qkv = normal(T, hq + 2 * hkv, d)
    qkv[:, : hq + hkv] *= size
    state["qkv"] = qkv.view(T, -1).to(torch.bfloat16)
    pool = torch.empty(pages, 2, hkv, page, d, device=DEVICE, dtype=torch.bfloat16)
    pool[:, 0] = (normal(pages, hkv, page, d) * size).to(torch.bfloat16)
    pool[:, 1] = normal(pages, hkv, page, d).to(torch.bfloat16)
    state["pool"] = pool
    if case["op"] == "append":
        state["pos"] = torch.cat([torch.arange(c - n, c) for n, c in zip(new, ctx)]).to(torch.int32).to(DEVICE)
        state["seq"] = torch.cat([torch.full((n,), s) for s, n in enumerate(new)]).to(torch.int32).to(DEVICE)
        turns, state["m"] = _turns(case["rot"], case["scaling"])
        state["turns"] = turns.to(DEVICE)
    else:
        state["cu"] = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).to(DEVICE)
        state["ctx"] = torch.tensor(ctx, dtype=torch.int32).to(DEVICE)
        state["scale"] = d ** -0.5
    return state


# ---------------------------------------------------------------------------------------------------------------- one pass
def _rotate(x, pos, turns, m, rot, halves, back):
    """x fp32 [T, heads, head]."""
    a = pos.double()[:, None] * turns
    a = (a - a.round()) * (2 * math.pi)
    c, s = (m * a.cos()).float()[:, None], (m * a.sin()).float()[:, None]
    if back:
        s = -s
    y = x.clone()
    u, v = (x[..., : rot // 2], x[..., rot // 2 : rot]) if halves else (x[..., 0:rot:2], x[..., 1:rot:2])
    if halves:
        y[..., : rot // 2], y[..., rot // 2 : rot] = u * c - v * s, v * c + u * s
    else:
        y[..., 0:rot:2], y[..., 1:rot:2] = u * c - v * s, v * c + u * s
    return y


def _plain_rotary(st):
    case = st["case"]
    x = st["x"]
    y = _rotate(x.float().view(case["T"], case["heads"], case["head"]), st["pos"], st["turns"], st["m"], case["rot"], case["halves"], case["back"])
    return y.view(x.shape).to(x.dtype)


def _plain_append(st):
    case = st["case"]
    hq, hkv, d, page = case["hq"], case["hkv"], case["head"], case["page"]
    qkv = st["qkv"].view(-1, hq + 2 * hkv, d)
    y = _rotate(qkv[:, : hq + hkv].float(), st["pos"], st["turns"], st["m"], case["rot"], case["halves"], False).to(torch.bfloat16)
    pos, seq = st["pos"].long(), st["seq"].long()
    at, row = st["table"][seq, pos // page].long(), pos % page
    st["pool"][at, 0, :, row] = y[:, hq:]
    st["pool"][at, 1, :, row] = qkv[:, hq + hkv :]
    return {"q": y[:, :hq].reshape(-1, hq * d), "pool": st["pool"]}


def _plain_attend(st):
    case = st["case"]
    hq, hkv, d, page = case["hq"], case["hkv"], case["head"], case["page"]
    q = st["qkv"][:, : hq * d].float().view(-1, hkv, hq // hkv, d)
    n, c = st["cu"].diff().long(), st["ctx"].long()
    t, j = torch.arange(st["max_new"], device=q.device), torch.arange(st["max_ctx"], device=q.device)
    row = (st["cu"][:-1].long()[:, None] + t).clamp(max=q.shape[0] - 1)                                     # [seqs, new]
    at = st["table"][:, j // page].long()                                                                   # [seqs, ctx]
    k, v = (st["pool"][at, i, :, (j % page).expand_as(at)].float().transpose(1, 2) for i in (0, 1))         # [seqs, hkv, ctx, d]
    seen = (j < (c - n)[:, None, None] + t[:, None] + 1) & (t < n[:, None])[..., None]                      # [seqs, new, ctx]
    x = q[row].permute(0, 2, 3, 1, 4).reshape(len(c), hkv, -1, d)                                           # [seqs, hkv, rep * new, d]
    s = (x @ k.transpose(-1, -2)).view(len(c), hkv, hq // hkv, len(t), len(j)).mul_(st["scale"])
    s.masked_fill_(~seen[:, None, None], -math.inf)
    s.sub_(s.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    total = s.sum(-1, keepdim=True)
    o = (s.view(len(c), hkv, -1, len(j)) @ v).view(len(c), hkv, hq // hkv, len(t), d) / total.clamp_(min=1e-30)
    live = t < n[:, None]
    out = torch.empty(q.shape[0], hq * d, device=q.device, dtype=torch.bfloat16)
    out[row[live]] = o.permute(0, 3, 1, 2, 4).reshape(len(c), len(t), hq * d)[live].to(torch.bfloat16)
    return out


def run(state):
    st, case = state, state["case"]
    if not own:
        return {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}[case["op"]](st)
    from omchat_b200 import lib
    if case["op"] == "rotary":
        return lib.rotary(st["x"], st["pos"], st["turns"], case["heads"], case["head"], halves=case["halves"], back=case["back"], mscale=st["m"])
    if case["op"] == "append":
        q = lib.rotary_kv_append(st["qkv"], st["pos"], st["seq"], st["turns"], case["hq"], st["pool"], st["table"], halves=case["halves"], mscale=st["m"])
        return {"q": q, "pool": st["pool"]}
    q = st["qkv"][:, : case["hq"] * case["head"]]
    return lib.paged_attention(q, st["pool"], st["table"], st["cu"], st["ctx"], st["max_new"], st["max_ctx"], case["hq"], st["scale"])


# ---------------------------------------------------------------------------------------------------------------- work and exact values
def work(case):
    if case["op"] == "rotary":
        n = case["T"] * case["heads"] * case["head"]
        return {"bytes": 2 * n * (2 if case["dtype"] == "bf16" else 4) + 4 * case["T"], "flops": 3 * n}
    new, ctx = _lengths(case)
    hq, hkv, d, T = case["hq"], case["hkv"], case["head"], sum(new)
    if case["op"] == "append":
        return {"bytes": 2 * (2 * T * (hq + 2 * hkv) * d) + 8 * T, "flops": 3 * T * (hq + hkv) * d}
    pairs = sum(n * c - n * (n - 1) // 2 for n, c in zip(new, ctx))
    return {"bytes": 2 * 2 * T * hq * d + 2 * 2 * sum(ctx) * hkv * d, "flops": 4 * d * hq * pairs}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "attend":
        new, ctx = _lengths(case)
        hq, hkv, d = case["hq"], case["hkv"], case["head"]
        out = torch.zeros(sum(new), hq, d, device=DEVICE, dtype=torch.float64)
        first = 0
        for s, (n, c) in enumerate(zip(new, ctx)):
            rows = st["pool"][st["table"][s].long()].double().permute(1, 2, 0, 3, 4).reshape(2, hkv, -1, d)[:, :, :c]
            hidden = torch.ones(n, c, device=DEVICE, dtype=torch.bool).triu_(c - n + 1)
            for h in range(hq):
                q = st["qkv"][first : first + n, h * d : (h + 1) * d].double()
                score = torch.einsum("td,jd->tj", q, rows[0, h * hkv // hq]) / math.sqrt(d)
                out[first : first + n, h] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=1) @ rows[1, h * hkv // hq]
            first += n
        return out.view(-1, hq * d)
    rot, pos = case["rot"], st["pos"].double()
    wave = st["m"] * torch.exp(2j * math.pi * (pos[:, None] * st["turns"]).frac())[:, None]              # [T, 1, rot / 2], complex
    if case["op"] == "rotary" and case["back"]:
        wave = wave.conj()
    rows = (st["x"] if case["op"] == "rotary" else st["qkv"]).double().view(len(pos), -1, case["head"])
    turned = rows.clone()
    which = rows.shape[1] if case["op"] == "rotary" else case["hq"] + case["hkv"]
    part = rows[:, :which, :rot]
    if case["halves"]:
        z = torch.complex(part[..., : rot // 2], part[..., rot // 2 :]) * wave
        turned[:, :which, :rot] = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.view_as_complex(part.reshape(len(pos), which, rot // 2, 2)) * wave
        turned[:, :which, :rot] = torch.view_as_real(z).flatten(-2)
    if case["op"] == "rotary":
        return turned.view(len(pos), -1)
    hq, hkv, page = case["hq"], case["hkv"], case["page"]
    pool = st["pool"].double()
    at = st["table"].long()[st["seq"].long(), torch.div(st["pos"], page, rounding_mode="floor").long()]
    place = (at[:, None] * 2 + torch.arange(2, device=DEVICE)) * hkv                                       # [T, 2]
    place = (place[..., None] + torch.arange(hkv, device=DEVICE)) * page + (st["pos"].long() % page)[:, None, None]
    pool.view(-1, case["head"])[place.reshape(-1)] = turned[:, hq:].reshape(-1, case["head"])
    return {"q": turned[:, :hq].reshape(len(pos), -1), "pool": pool}
