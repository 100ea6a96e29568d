"""Performance cases of the operators that serve drafted and portioned tokens over a paged cache.

A case is a dict of plain values.  Kinds:

  append     `ops.qkv_axes_rope_append`: fused query / key / value rows turned by their positions on several axes (time, height, width), keys and
             values into the pages of their sequences
  attention  `ops.paged_attention`: the new tokens of every sequence (one, a few drafted ones, a portion of a prompt) over its pages
  verify     `ops.verify_drafts`: drafted tokens against the target's probabilities, from given random numbers

`run` computes them in elementary torch operations, or with `own` set through the framework's entry points.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token of one user: latency counts
        dict(name="append_one_token", kind="append", dtype="bf16", seqs=1, new=1, ctx=700, mix="equal", shape=1, heads=32, kv_heads=8, dim=128,
             rot=128, halves=True, spread=False, far=0, page=16, order="rows"),
        # 32 users with drafted tokens, half of each head turned in adjacent pairs, positions far out, pages with the heads outside
        dict(name="append_drafts_far", kind="append", dtype="f16", seqs=32, new=5, ctx=3000, mix="ragged", shape=2, heads=32, kv_heads=8, dim=64,
             rot=32, halves=False, spread=False, far=900000, page=32, order="heads"),
        # portions of prompts with pictures, frequencies of the axes in turn
        dict(name="append_prompt", kind="append", dtype="bf16", seqs=3, new=2048, ctx=1500, mix="ragged", shape=3, heads=32, kv_heads=8, dim=128,
             rot=128, halves=True, spread=True, far=0, page=64, order="rows"),
        # one user, one token behind a page or two
        dict(name="attn_one_token", kind="attention", dtype="bf16", seqs=1, new=1, ctx=600, mix="equal", shape=4, heads=32, kv_heads=8, dim=128,
             window=0, page=16, order="rows"),
        # 32 users decoding over caches of different lengths, some without a token in this step
        dict(name="attn_decode_batch", kind="attention", dtype="f16", seqs=32, new=1, ctx=4096, mix="ragged", shape=5, heads=32, kv_heads=8, dim=128,
             window=0, page=64, order="rows"),
        # drafted tokens of 16 users, up to five and the one before them
        dict(name="attn_drafts", kind="attention", dtype="bf16", seqs=16, new=6, ctx=6000, mix="ragged", shape=6, heads=64, kv_heads=8, dim=128,
             window=0, page=16, order="heads"),
        # one long document, one token
        dict(name="attn_long", kind="attention", dtype="bf16", seqs=1, new=1, ctx=131072, mix="equal", shape=7, heads=32, kv_heads=8, dim=128,
             window=0, page=128, order="rows"),
        # continuous batching: most users decode, some bring a portion of a prompt; heads of 64 in a sliding window
        dict(name="attn_mixed_window", kind="attention", dtype="f16", seqs=24, new=500, ctx=2500, mix="mixed", shape=8, heads=32, kv_heads=8, dim=64,
             window=1024, page=32, order="rows"),
        # a long portion of a long prompt
        dict(name="attn_prompt", kind="attention", dtype="bf16", seqs=1, new=4096, ctx=4096, mix="equal", shape=9, heads=32, kv_heads=8, dim=128,
             window=0, page=64, order="rows"),
        # three drafted tokens of one user, a small vocabulary
        dict(name="verify_one", kind="verify", seqs=1, drafts=3, vocab=32000, given=True, ragged=False),
        # 64 users, a large vocabulary, some with fewer drafts
        dict(name="verify_batch", kind="verify", seqs=64, drafts=5, vocab=128256, given=True, ragged=True),
        # drafts looked up in the prompt: no draft probabilities, a vocabulary of odd size
        dict(name="verify_lookup", kind="verify", seqs=13, drafts=8, vocab=50257, given=False, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "verify"])
    if kind == "verify":
        vocab = _log(rng, 1000, 152000)
        seqs, drafts = _log(rng, 1, 64), rng.randint(1, 8)
        while seqs * (drafts + 1) * vocab > 64 * 6 * 128256:
            seqs = (seqs + 1) // 2
        return dict(kind=kind, seqs=seqs, drafts=drafts, vocab=vocab, given=rng.random() < 0.7, ragged=rng.random() < 0.5)
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 64), (16, 16, 64), (8, 1, 128), (64, 8, 128), (28, 4, 128), (24, 8, 64)])
    case = dict(kind=kind, dtype=rng.choice(["bf16", "f16"]), shape=rng.randrange(1 << 20), heads=heads, kv_heads=kv_heads, dim=dim,
                page=rng.choice([1, 8, 16, 20, 32, 64, 128, 256]), order=rng.choice(["rows", "heads"]))
    if kind == "append":
        case.update(seqs=_log(rng, 1, 32), new=_log(rng, 1, 2048), ctx=_log(rng, 1, 4000), mix=rng.choice(["equal", "ragged", "mixed"]),
                    rot=rng.choice([dim, dim // 2, 6 * (dim // 8)]), halves=rng.random() < 0.6, spread=rng.random() < 0.5,
                    far=rng.choice([0, 0, _log(rng, 1000, 4000000)]))
        while case["seqs"] * case["new"] > 6000:
            case["seqs"] = (case["seqs"] + 1) // 2
        return case
    form = rng.choice(["decode", "drafts", "mixed", "prompt"])
    if form == "decode":
        seqs = _log(rng, 1, 64)
        case.update(seqs=seqs, new=1, ctx=_log(rng, 1, 131072 // seqs), mix=rng.choice(["equal", "ragged"]))
    elif form == "drafts":
        seqs = _log(rng, 1, 32)
        case.update(seqs=seqs, new=rng.randint(2, 9), ctx=_log(rng, 1, 65536 // seqs), mix=rng.choice(["equal", "ragged"]))
    elif form == "mixed":
        case.update(seqs=_log(rng, 2, 24), new=_log(rng, 10, 600), ctx=_log(rng, 1, 2500), mix="mixed")
    else:
        case.update(seqs=1, new=_log(rng, 16, 3500), ctx=_log(rng, 1, 4500), mix="equal")
        if rng.random() < 0.4:
            case.update(seqs=rng.randint(2, 4), new=_log(rng, 16, 1500), ctx=_log(rng, 1, 2500), mix="ragged")
    case["window"] = rng.choice([0, 0, 0, _log(rng, 1, 2000)])
    while work(case)["flops"] > 4.1e11:
        case["new"] = case["new"] * 2 // 3
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _lens(case):
    """[(cached, new)] of the sequences, from the case alone.  equal: all the same; ragged: anything up to the bounds, and in places no new token;
    mixed: one in six a portion of a prompt, the others one token."""
    rng, out = random.Random(case["shape"]), []
    for i in range(case["seqs"]):
        if case["mix"] == "equal" or i == 0:
            out.append((case["ctx"], case["new"]))
        elif case["mix"] == "ragged":
            out.append((_log(rng, 1, case["ctx"] + 1) - 1 if i % 3 == 0 else rng.randint(0, case["ctx"]), 0 if i % 7 == 6 else rng.randint(1, case["new"])))
        else:
            out.append((rng.randint(0, case["ctx"]), rng.randint(1, case["new"]) if i % 6 == 0 else 1))
    return out


def _paged(case, g):
    """Caches of random rows, pages in no order, and the tables that a scheduler keeps beside them."""
    lens, page, hk, d = _lens(case), case["page"], case["kv_heads"], case["dim"]
    need = [-(-(c + n) // page) for c, n in lens]
    pages, dtype = sum(need) + 3, TYPES[case["dtype"]]
    ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(need) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = ids[at:at + m]
        at += m
    shape = (pages, page, hk, d) if case["order"] == "rows" else (pages, hk, page, d)
    k, v = _randn(g, *shape, dtype=dtype), _randn(g, *shape, dtype=dtype)
    if case["order"] == "heads":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    new = torch.tensor([n for _, n in lens], device="cuda")
    total = torch.tensor([c + n for c, n in lens], dtype=torch.int32, device="cuda")
    starts = torch.zeros(len(lens) + 1, dtype=torch.int32, device="cuda")
    starts[1:] = new.cumsum(0)
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), new)
    index = torch.arange(seq.numel(), device="cuda") - starts[seq]
    return {"k": k, "v": v, "table": table, "lens": total, "starts": starts, "seq": seq.to(torch.int32), "index": index.to(torch.int32),
            "place": (total[seq] - new[seq] + index).to(torch.int32), "max_new": max(n for _, n in lens)}


def _axes(case):
    """Which axis turns each frequency: a quarter of them by time, the others by height and width, in one piece each or in turn."""
    half = case["rot"] // 2
    a, b = half // 4, half // 4 + (half - half // 4 + 1) // 2
    if case["spread"]:
        return [(i % 3) if i < 3 * a else 1 + (i - 3 * a) % 2 for i in range(half)]
    return [0 if i < a else 1 if i < b else 2 for i in range(half)]


def _append_tensors(case, g):
    s = _paged(case, g)
    t, width = s["seq"].numel(), (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
    place = s["place"].to(torch.int64) + case["far"]
    grid = s["index"].to(torch.int64)
    picture = (grid // 100) % 2 == 1                                 # text and pictures of ten by ten patches in turn
    rows = torch.where(picture, place - grid % 100, place)
    pos = torch.stack([rows, rows + torch.where(picture, grid % 100 // 10, 0), rows + torch.where(picture, grid % 10, 0)]).to(torch.int32)
    half = case["rot"] // 2
    s.update(qkv=_randn(g, t, width, dtype=TYPES[case["dtype"]]), pos=pos.contiguous(), axis=torch.tensor(_axes(case), dtype=torch.int32, device="cuda"),
             freq=1000000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half))
    return s


def _attention_tensors(case, g):
    s = _paged(case, g)
    s["q"] = _randn(g, s["seq"].numel(), case["heads"] * case["dim"], dtype=TYPES[case["dtype"]], scale=1.5)
    return s


def _verify_tensors(case, g):
    """Probabilities as a model leaves them: a few likely words and a long tail; the drafting model is near the target."""
    b, k, v = case["seqs"], case["drafts"], case["vocab"]
    z = _randn(g, b, k + 1, v, scale=2.0)
    z.scatter_add_(2, torch.randint(0, v, (b, k + 1, 4), generator=g, device="cuda"), _randn(g, b, k + 1, 4, scale=3.0).abs() + 6.0)
    target = torch.softmax(z, -1)
    draft = torch.softmax(z[:, :k] + _randn(g, b, k, v, scale=0.5), -1)
    drafted = torch.multinomial(draft.reshape(b * k, v), 1, generator=g).reshape(b, k).to(torch.int32)
    count = torch.randint(0, k + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
    return {"target": target, "draft": draft if case["given"] else None, "drafted": drafted, "count": count,
            "accept": torch.rand(b, k, generator=g, device="cuda"), "sample": torch.rand(b, generator=g, device="cuda")}


def prepare(case, seed):
    s = {"append": _append_tensors, "attention": _attention_tensors, "verify": _verify_tensors}[case["kind"]](case, _gen(seed))
    s["kind"] = case["kind"]
    if case["kind"] != "verify":
        s.update(heads=case["heads"], kv_heads=case["kv_heads"], dim=case["dim"], scale=case["dim"] ** -0.5, window=case.get("window", 0),
                 halves=case.get("halves", True), page=case["page"])
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------------------
def _turn(x, c, s, halves):
    """x (T, heads, dim) fp32, its first 2 * half columns turned by the angles of c and s (T, 1, half)."""
    half = c.shape[-1]
    if halves:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([y, x[..., 2 * half:]], -1)


def _append(s):
    h, hk, d, qkv = s["heads"], s["kv_heads"], s["dim"], s["qkv"]
    t = qkv.shape[0]
    angle = s["pos"][s["axis"].long()].T.double() * s["freq"]
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x = qkv.view(t, h + 2 * hk, d).float()
    q = _turn(x[:, :h], c, n, s["halves"]).to(qkv.dtype).view(t, h * d)
    place = s["place"].long()
    page, row = s["table"][s["seq"].long(), place // s["page"]].long(), place % s["page"]
    s["k"][page, row] = _turn(x[:, h:h + hk], c, n, s["halves"]).to(qkv.dtype)
    s["v"][page, row] = qkv.view(t, h + 2 * hk, d)[:, h + hk:]
    return q, s["k"], s["v"]


def _attend(s):
    h, hk, d, q = s["heads"], s["kv_heads"], s["dim"], s["q"]
    seq, index, lens, starts = s["seq"].long(), s["index"].long(), s["lens"].long(), s["starts"].long()
    b, m = lens.numel(), s["max_new"]
    rows = torch.zeros(b, m, hk, h // hk, d, device=q.device)
    rows[seq, index] = q.view(-1, hk, h // hk, d).float()
    pages = s["table"].clamp(min=0).long()
    k = s["k"][pages].reshape(b, -1, hk, d).float()
    v = s["v"][pages].reshape(b, -1, hk, d).float()
    at = torch.arange(k.shape[1], device=q.device)
    own_place = (lens - (starts[1:] - starts[:-1]))[:, None] + torch.arange(m, device=q.device)
    seen = (at <= own_place[..., None]) & (at < lens[:, None, None])
    if s["window"]:
        seen &= at > own_place[..., None] - s["window"]
    x = torch.einsum("bnhgd,bkhd->bhgnk", rows, k).mul_(s["scale"])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    o = torch.einsum("bhgnk,bkhd->bnhgd", x, v)
    total = x.sum(-1).permute(0, 3, 1, 2)[..., None]
    return torch.where(total > 0, o / total, 0.0)[seq, index].reshape(q.shape).to(q.dtype)


def _verify(s):
    target, draft, drafted = s["target"].double(), s["draft"], s["drafted"].long()
    b, k = drafted.shape
    count = s["count"].long() if s["count"] is not None else torch.full((b,), k, device=target.device)
    p = target[:, :k].gather(2, drafted[..., None])[..., 0]
    q = draft.gather(2, drafted[..., None])[..., 0].double() if draft is not None else torch.ones_like(p)
    step = torch.arange(k, device=target.device)
    taken = (s["accept"].double() * q < p) & (step < count[:, None])
    accepted = taken.long().cumprod(1).sum(1)
    each = torch.arange(b, device=target.device)
    row, last = target[each, accepted], accepted.clamp(max=k - 1)
    if draft is not None:
        less = draft[each, last].double()
    else:
        less = torch.zeros_like(row).scatter_(1, drafted[each, last][:, None], 1.0)
    rest = torch.where((accepted < count)[:, None], (row - less).clamp(min=0.0), row)
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, row)
    total = rest.cumsum(1)
    word = torch.searchsorted(total, (s["sample"].double() * total[:, -1])[:, None], right=True)[:, 0]
    tokens = torch.where(torch.arange(k + 1, device=target.device) < accepted[:, None], torch.nn.functional.pad(drafted, (0, 1)), -1)
    tokens[each, accepted] = torch.minimum(word, (rest > 0).long().cumsum(1).argmax(1))
    return accepted.to(torch.int32), tokens.to(torch.int32)


def run(s):
    if own:
        from zhilight_b200 import ops
        if s["kind"] == "append":
            q = ops.qkv_axes_rope_append(s["qkv"], s["pos"], s["freq"], s["axis"], s["seq"], s["place"], s["table"], s["k"], s["v"], s["heads"],
                                         layout=ops.ROT_HALVES if s["halves"] else ops.ROT_ADJACENT)
            return q, s["k"], s["v"]
        if s["kind"] == "attention":
            return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"], s["scale"], window=s["window"], max_new=s["max_new"])
        return ops.verify_drafts(s["target"], s["draft"], s["drafted"], s["accept"], s["sample"], s["count"])
    return {"append": _append, "attention": _attend, "verify": _verify}[s["kind"]](s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "verify":                                     # a row of the target and one of the draft decide a sequence's last token
        rows = 2 if case["given"] else 1
        return {"bytes": case["seqs"] * (rows * 4 * case["vocab"] + 24 * case["drafts"] + 12), "flops": case["seqs"] * 3 * case["vocab"]}
    h, hk, d, lens = case["heads"], case["kv_heads"], case["dim"], _lens(case)
    t = sum(n for _, n in lens)
    if case["kind"] == "append":
        return {"bytes": t * ((h + 2 * hk) * d * 4 + 20), "flops": t * (h + hk) * case["rot"] * 3}
    w, pairs, rows = case["window"], 0, 0
    for c, n in lens:
        rows += (min(c + n, n + w - 1) if w else c + n) if n else 0
        full = n * c + n * (n + 1) // 2                              # all that the rows see without a window
        if w:
            hidden = max(0, c + n - w)                               # of the last row; of those before it one less each
            less = min(n, hidden)
            full -= less * hidden - less * (less - 1) // 2
        pairs += full
    return {"bytes": rows * hk * d * 4 + t * h * d * 4 + 4 * (rows // case["page"] + 3 * case["seqs"]), "flops": 4 * pairs * h * d}


# ---- the same in 64 bits -------------------------------------------------------------------------------------------------------
def _exact_append(case, s):
    """Rows as complex numbers, times e^(i angle)."""
    h, hk, d, half = case["heads"], case["kv_heads"], case["dim"], case["rot"] // 2
    x = s["qkv"].double().view(-1, h + 2 * hk, d)
    at = torch.stack([s["pos"][a] for a in _axes(case)], 1).double() * s["freq"]
    turn = torch.polar(torch.ones_like(at), at)[:, None]
    re, im = (slice(0, half), slice(half, 2 * half)) if case["halves"] else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    z = torch.complex(x[:, :h + hk, re].contiguous(), x[:, :h + hk, im].contiguous()) * turn
    y = x.clone()
    y[:, :h + hk, re], y[:, :h + hk, im] = z.real, z.imag
    k, v = s["k"].double(), s["v"].double()
    seq, place, table = s["seq"].tolist(), s["place"].tolist(), s["table"].tolist()
    pages = torch.tensor([table[b][p // case["page"]] for b, p in zip(seq, place)], device="cuda")
    rows = torch.tensor([p % case["page"] for p in place], device="cuda")
    k.index_put_((pages, rows), y[:, h:h + hk])
    v.index_put_((pages, rows), y[:, h + hk:])
    return y[:, :h].reshape(-1, h * d), k, v


def _exact_attention(case, s):
    """One sequence, one key head and a thousand rows at a time."""
    h, hk, d, page, w = case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
    g, out, at = h // hk, torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    q = s["q"].double().view(-1, h, d)
    for b, (c, n) in enumerate(_lens(case)):
        ids = s["table"][b, :-(-(c + n) // page)].long()
        for j in range(hk if n else 0):
            k = s["k"][ids, :, j].reshape(-1, d)[:c + n].double()
            v = s["v"][ids, :, j].reshape(-1, d)[:c + n].double()
            for r in range(0, n, 1024):
                m = min(1024, n - r)
                sees = torch.arange(c + r, c + r + m, device="cuda")[:, None] - torch.arange(c + n, device="cuda")[None]
                hide = (sees < 0) | (sees >= w) if w else sees < 0
                x = (q[at + r:at + r + m, j * g:(j + 1) * g].transpose(0, 1) @ k.T) * d ** -0.5
                o = torch.softmax(x.masked_fill(hide, -math.inf), -1) @ v
                out[at + r:at + r + m].view(m, h, d)[:, j * g:(j + 1) * g] = o.transpose(0, 1)
        at += n
    return out


def _exact_verify(case, s):
    """A sequence at a time, its sums added up in order on the host."""
    k, accepted, tokens = case["drafts"], [], []
    draft = s["draft"].cpu() if case["given"] else None
    counts = s["count"].tolist() if s["count"] is not None else [k] * case["seqs"]
    for b, m in enumerate(counts):
        target, words, lucky = s["target"][b].cpu().double(), s["drafted"][b].tolist(), s["accept"][b].double().tolist()
        n = 0
        while n < m and lucky[n] * (float(draft[b, n, words[n]]) if case["given"] else 1.0) < float(target[n, words[n]]):
            n += 1
        rest = target[n].clone()
        if n < m:
            if case["given"]:
                rest = torch.relu(rest - draft[b, n].double())
            else:
                rest[words[n]] = 0.0
        if not bool((rest > 0).any()):
            rest = target[n].clone()
        total = torch.cumsum(rest, 0)
        beyond = (total > float(s["sample"][b]) * float(total[-1])).nonzero()
        word = int(beyond[0]) if len(beyond) else int((rest > 0).nonzero()[-1])
        accepted.append(n)
        tokens.append(words[:n] + [word] + [-1] * (k - n))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "verify": _exact_verify}[case["kind"]](case, s)
