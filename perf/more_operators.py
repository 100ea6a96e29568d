"""Performance cases of the operators of a serving step over a paged cache that is held in 4 bits.

A case is a dict of plain values.  Kinds:

  append     `ops.qkv_axes_rope_append_int4`: fused query / key / value rows turned by their positions on several axes (time, height, width), keys and
             values into the pages of their sequences as 4-bit codes; then `ops.int4_cache_values`, what the caches stand for
  attention  `ops.paged_attention_int4`: the new tokens of every sequence (one, a few drafted ones, a portion of a prompt) over its pages
  logits     `ops.adjust_logits`: penalties for repeated words, biases, temperature and grammar masks on the rows that words are drawn from

A row of a head in the cache: the codes, then (step, low) of every 32 columns in the rows' type.  A code c stands for low + step * c, rounded to that type.

`run` computes them in elementary torch operations, or with `own` set through the framework's entry points.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
GROUP = 32                                                            # columns that share a step and a lowest value
NIBBLE = (0, 2, 4, 6, 1, 3, 5, 7)                                     # column of each nibble of 32 bits, the lowest first


def listed():
    return [
        # one token of one user: latency counts
        dict(name="append4_one_token", kind="append", dtype="bf16", seqs=1, new=1, ctx=700, mix="equal", shape=1, heads=32, kv_heads=8, dim=128,
             rot=128, halves=True, spread=False, far=0, page=16, order="rows"),
        # 32 users with drafted tokens, half of each head turned in adjacent pairs, positions far out, pages with the heads outside
        dict(name="append4_drafts_far", kind="append", dtype="f16", seqs=32, new=5, ctx=3000, mix="ragged", shape=2, heads=32, kv_heads=8, dim=64,
             rot=32, halves=False, spread=False, far=900000, page=32, order="heads"),
        # portions of prompts with pictures, frequencies of the axes in turn
        dict(name="append4_prompt", kind="append", dtype="bf16", seqs=3, new=2048, ctx=1500, mix="ragged", shape=3, heads=32, kv_heads=8, dim=128,
             rot=128, halves=True, spread=True, far=0, page=64, order="rows"),
        # one user, one token behind a page or two
        dict(name="attn4_one_token", kind="attention", dtype="bf16", seqs=1, new=1, ctx=600, mix="equal", shape=4, heads=32, kv_heads=8, dim=128,
             window=0, page=16, order="rows"),
        # 32 users decoding over caches of different lengths, some without a token in this step
        dict(name="attn4_decode_batch", kind="attention", dtype="f16", seqs=32, new=1, ctx=4096, mix="ragged", shape=5, heads=32, kv_heads=8, dim=128,
             window=0, page=64, order="rows"),
        # drafted tokens of 16 users, up to five and the one before them
        dict(name="attn4_drafts", kind="attention", dtype="bf16", seqs=16, new=6, ctx=6000, mix="ragged", shape=6, heads=64, kv_heads=8, dim=128,
             window=0, page=16, order="heads"),
        # one long document, one token: what 4 bits are for
        dict(name="attn4_long", kind="attention", dtype="bf16", seqs=1, new=1, ctx=131072, mix="equal", shape=7, heads=32, kv_heads=8, dim=128,
             window=0, page=128, order="heads"),
        # continuous batching: most users decode, some bring a portion of a prompt; heads of 64 in a sliding window
        dict(name="attn4_mixed_window", kind="attention", dtype="f16", seqs=24, new=500, ctx=2500, mix="mixed", shape=8, heads=32, kv_heads=8, dim=64,
             window=1024, page=32, order="rows"),
        # a long portion of a long prompt
        dict(name="attn4_prompt", kind="attention", dtype="bf16", seqs=1, new=2048, ctx=6000, mix="equal", shape=9, heads=32, kv_heads=8, dim=128,
             window=0, page=64, order="rows"),
        # one user's next word
        dict(name="logits_one", kind="logits", dtype="bf16", wide=False, seqs=1, drafts=0, vocab=32000, hist=700, bias=4, masks=0, shape=10),
        # 64 users, a large vocabulary, answers of every length, two in three under one of a few grammars
        dict(name="logits_batch", kind="logits", dtype="bf16", wide=True, seqs=64, drafts=0, vocab=128256, hist=4000, bias=16, masks=5, shape=11),
        # rows behind drafted words: each of them repeats what the drafts before it have brought; a vocabulary of odd size
        dict(name="logits_drafts", kind="logits", dtype="f32", wide=False, seqs=13, drafts=8, vocab=50257, hist=9000, bias=300, masks=13, shape=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "logits"])
    if kind == "logits":
        seqs, drafts, vocab = _log(rng, 1, 128), rng.choice([0, 0, rng.randint(1, 8)]), _log(rng, 1000, 152000)
        while seqs * (drafts + 1) * vocab > 128 * 128256:
            seqs = (seqs + 1) // 2
        return dict(kind=kind, dtype=rng.choice(["bf16", "f16", "f32"]), wide=rng.random() < 0.5, seqs=seqs, drafts=drafts, vocab=vocab, hist=_log(rng, 1, 16000),
                    bias=rng.choice([0, _log(rng, 1, 500)]), masks=rng.choice([0, 1, rng.randint(2, 20)]), shape=rng.randrange(1 << 20))
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (32, 8, 64), (16, 16, 64), (8, 1, 128), (64, 8, 128), (28, 4, 128), (24, 8, 64)])
    case = dict(kind=kind, dtype=rng.choice(["bf16", "f16"]), shape=rng.randrange(1 << 20), heads=heads, kv_heads=kv_heads, dim=dim,
                page=rng.choice([1, 8, 16, 20, 32, 64, 128, 256]), order=rng.choice(["rows", "heads"]))
    if kind == "append":
        case.update(seqs=_log(rng, 1, 32), new=_log(rng, 1, 2048), ctx=_log(rng, 1, 4000), mix=rng.choice(["equal", "ragged", "mixed"]),
                    rot=rng.choice([dim, dim // 2, 6 * (dim // 8)]), halves=rng.random() < 0.6, spread=rng.random() < 0.5,
                    far=rng.choice([0, 0, _log(rng, 1000, 4000000)]))
        while case["seqs"] * case["new"] > 5000:
            case["new"] = case["new"] * 2 // 3
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
        case.update(seqs=1, new=_log(rng, 16, 2500), ctx=_log(rng, 1, 6000), mix="equal")
        if rng.random() < 0.4:
            case.update(seqs=rng.randint(2, 4), new=_log(rng, 16, 1000), ctx=_log(rng, 1, 2500), mix="ragged")
    case["window"] = rng.choice([0, 0, 0, _log(rng, 1, 2000)])
    while work(case)["flops"] > 2.3e11:
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


def _pack(x):
    """Rows (..., dim) in 16 bits -> (..., dim / 2 + dim / 8) bytes: 4-bit codes, then step and lowest value of every 32 columns in the rows' type.
    The step is a 15th of the range, rounded down: no code stands for more than the highest; a code is the nearest whole number of steps, at most 15."""
    v = x.float().unflatten(-1, (-1, GROUP))
    low, high = v.amin(-1, keepdim=True), v.amax(-1, keepdim=True)
    part = (high * 0.5 - low * 0.5) / 7.5                             # halves: a range may be beyond the largest number
    step = part.to(x.dtype)
    step = (step.view(torch.int16) - (step.float() > part).to(torch.int16)).view(x.dtype)
    s = step.float()
    code = torch.where(s >= 2.0 ** -126, ((v * 0.5 - low * 0.5) / torch.where(s > 0, s, 1.0) * 2.0).round().clamp(0, 15), 0.0).to(torch.uint8).flatten(-2)
    code = code.unflatten(-1, (-1, 8))[..., NIBBLE].flatten(-2)
    meta = torch.cat([step, low.to(x.dtype)], -1).flatten(-2).contiguous().view(torch.uint8)
    return torch.cat([code[..., 0::2] | code[..., 1::2] << 4, meta], -1)


def _unpack(rows, dtype):
    """What rows of a cache stand for, in the type that they were written from."""
    n = rows.shape[-1] // 5 * 4
    code = torch.stack([rows[..., :n] & 15, rows[..., :n] >> 4], -1).flatten(-2).unflatten(-1, (-1, 8))
    code = code[..., [NIBBLE.index(i) for i in range(8)]].flatten(-2)
    meta = rows[..., n:].contiguous().view(dtype).float().unflatten(-1, (-1, 2))
    return (meta[..., 1:] + meta[..., :1] * code.float().unflatten(-1, (-1, GROUP))).flatten(-2).to(dtype)


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
    # keys have columns that lie far from zero, as a turned key's slow columns do
    middle = _randn(g, hk, 1, d, scale=1.5) if case["order"] == "heads" else _randn(g, hk, d, scale=1.5)
    k, v = _pack((_randn(g, *shape) + middle).to(dtype)), _pack(_randn(g, *shape, dtype=dtype))
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
    s["q"] = _randn(g, s["seq"].numel(), case["heads"] * case["dim"], dtype=TYPES[case["dtype"]], scale=0.8)
    return s


def _histories(case):
    """[(words of the prompt, words in all)] of the sequences, from the case alone."""
    rng = random.Random(case["shape"])
    lens = [case["hist"]] + [rng.randint(0, case["hist"]) for _ in range(case["seqs"] - 1)]
    return [(rng.randint(0, n), n) for n in lens]


def _bias_counts(case):
    rng = random.Random(case["shape"] + 1)
    return [rng.randint(0, case["bias"]) for _ in range(case["seqs"] * (case["drafts"] + 1))]


def _mask_rows(case):
    """The grammar of every row, -1: none."""
    rng = random.Random(case["shape"] + 2)
    return [rng.randrange(case["masks"]) if case["masks"] and rng.random() < 0.7 else -1 for _ in range(case["seqs"] * (case["drafts"] + 1))]


def _logits_tensors(case, g):
    """Logits as a model leaves them, histories in which few words are frequent, settings that differ from user to user, neutral ones among them."""
    b, k, v, hist = case["seqs"], case["drafts"] + 1, case["vocab"], _histories(case)
    r, dev = b * k, torch.device("cuda")
    words = (v * torch.rand(b, case["hist"] + k, generator=g, device=dev) ** 4).to(torch.int32).clamp(max=v - 1)
    seq = torch.arange(b, device=dev).repeat_interleave(k)
    lens = torch.tensor([n + i for _, n in hist for i in range(k)], dtype=torch.int32, device=dev)
    each = torch.rand(4, b, generator=g, device=dev)

    def setting(i, lo, hi, plain):
        return torch.where(each[i] < 0.25, plain, lo + (hi - lo) * each[i])[seq].contiguous()

    counts = torch.tensor(_bias_counts(case), device=dev)
    starts = torch.zeros(r + 1, dtype=torch.int32, device=dev)
    starts[1:] = counts.cumsum(0)
    n = sum(_bias_counts(case))
    heavy = torch.rand(n, generator=g, device=dev) < 0.2
    bias = torch.where(heavy, -100.0, _randn(g, n, scale=4.0))
    mask = None
    if case["masks"]:                                                # a grammar allows anything from nearly all words to a few
        share = torch.rand(case["masks"], 1, generator=g, device=dev) ** 3
        bits = (torch.rand(case["masks"], -(-v // 32) * 32, generator=g, device=dev) < share).unflatten(1, (-1, 32)).to(torch.int64)
        mask = (bits << torch.arange(32, device=dev)).sum(-1)
        mask = torch.where(mask >= 2 ** 31, mask - 2 ** 32, mask).to(torch.int32)
    return {"logits": _randn(g, r, v, dtype=TYPES[case["dtype"]], scale=4.0), "words": words, "seq": seq.to(torch.int32), "lens": lens,
            "prompt": torch.tensor([p for p, _ in hist], dtype=torch.int32, device=dev)[seq].contiguous(),
            "repetition": setting(0, 0.9, 1.4, 1.0), "frequency": setting(1, -0.1, 0.6, 0.0), "presence": setting(2, -0.2, 1.0, 0.0),
            "temperature": setting(3, 0.2, 1.4, 0.0), "bias_starts": starts, "bias_row": torch.arange(r, device=dev).repeat_interleave(counts),
            "bias_words": torch.randint(0, v, (n,), generator=g, device=dev, dtype=torch.int32), "bias": bias, "mask": mask,
            "mask_row": torch.tensor(_mask_rows(case), dtype=torch.int32, device=dev), "out_dtype": torch.float32 if case["wide"] else TYPES[case["dtype"]]}


def prepare(case, seed):
    s = {"append": _append_tensors, "attention": _attention_tensors, "logits": _logits_tensors}[case["kind"]](case, _gen(seed))
    s["kind"] = case["kind"]
    if case["kind"] != "logits":
        s.update(heads=case["heads"], kv_heads=case["kv_heads"], dim=case["dim"], scale=case["dim"] ** -0.5, window=case.get("window", 0),
                 halves=case.get("halves", True), page=case["page"], dtype=TYPES[case["dtype"]])
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
    c, n = angle.cos()[:, None], angle.sin()[:, None]                # keys in 64 bits: the codes are whole numbers
    x = qkv.view(t, h + 2 * hk, d)
    q = _turn(x[:, :h].float(), c.float(), n.float(), s["halves"]).to(qkv.dtype).view(t, h * d)
    place = s["place"].long()
    page, row = s["table"][s["seq"].long(), place // s["page"]].long(), place % s["page"]
    s["k"][page, row] = _pack(_turn(x[:, h:h + hk].double(), c, n, s["halves"]).to(qkv.dtype))
    s["v"][page, row] = _pack(x[:, h + hk:])
    return q, _unpack(s["k"], qkv.dtype), _unpack(s["v"], qkv.dtype)


def _attend(s):
    h, hk, d, q = s["heads"], s["kv_heads"], s["dim"], s["q"]
    seq, index, lens, starts = s["seq"].long(), s["index"].long(), s["lens"].long(), s["starts"].long()
    b, m = lens.numel(), s["max_new"]
    rows = torch.zeros(b, m, hk, h // hk, d, device=q.device)
    rows[seq, index] = q.view(-1, hk, h // hk, d).float()
    pages = s["table"].clamp(min=0).long()
    k = _unpack(s["k"][pages].reshape(b, -1, hk, d // 8 * 5), q.dtype).float()
    v = _unpack(s["v"][pages].reshape(b, -1, hk, d // 8 * 5), q.dtype).float()
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


def _adjust(s):
    z, words, mask = s["logits"].float(), s["words"][s["seq"].long()].long(), s["mask"]
    place = torch.arange(words.shape[1], device=z.device)
    there = place < s["lens"][:, None]
    seen = torch.zeros_like(z).scatter_add_(1, words, there.float())
    count = torch.zeros_like(z).scatter_add_(1, words, (there & (place >= s["prompt"][:, None])).float())
    r = s["repetition"][:, None]
    z = torch.where(seen > 0, torch.where(z > 0, z / r, z * r), z)
    z = z - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    z = z.index_put((s["bias_row"], s["bias_words"].long()), s["bias"], accumulate=True)
    heat = s["temperature"][:, None]
    z = torch.where(heat > 0, z / heat, z)
    if mask is not None:
        word = torch.arange(z.shape[1], device=z.device)
        allowed = (mask[s["mask_row"].clamp(min=0).long()][:, word >> 5] >> (word & 31) & 1 == 1) | (s["mask_row"] < 0)[:, None]
        z = torch.where(allowed, z, -math.inf)
    return z.to(s["out_dtype"])


def run(s):
    if own:
        from zhilight_b200 import ops
        if s["kind"] == "append":
            q = ops.qkv_axes_rope_append_int4(s["qkv"], s["pos"], s["freq"], s["axis"], s["seq"], s["place"], s["table"], s["k"], s["v"], s["heads"],
                                              layout=ops.ROT_HALVES if s["halves"] else ops.ROT_ADJACENT)
            k, v = ops.int4_cache_values(s["k"], s["v"], s["dtype"])
            return q, k, v
        if s["kind"] == "attention":
            return ops.paged_attention_int4(s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"], s["scale"], window=s["window"], max_new=s["max_new"])
        return ops.adjust_logits(s["logits"], tokens=s["words"], token_seq=s["seq"], token_lens=s["lens"], prompt_lens=s["prompt"],
                                 repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"], bias_starts=s["bias_starts"],
                                 bias_words=s["bias_words"], bias=s["bias"], temperature=s["temperature"], mask=s["mask"],
                                 mask_row=s["mask_row"] if s["mask"] is not None else None, out_dtype=s["out_dtype"])
    return {"append": _append, "attention": _attend, "logits": _adjust}[s["kind"]](s)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] == "logits":
        r, v, size = case["seqs"] * (case["drafts"] + 1), case["vocab"], 2 if case["dtype"] != "f32" else 4
        once = sum(n + case["drafts"] for _, n in _histories(case))
        grammars = len(set(_mask_rows(case)) - {-1})
        return {"bytes": r * v * (size + (4 if case["wide"] else size)) + 4 * once + 8 * sum(_bias_counts(case)) + grammars * 4 * -(-v // 32) + 36 * r, "flops": 2 * r * v}
    h, hk, d, lens = case["heads"], case["kv_heads"], case["dim"], _lens(case)
    t, row = sum(n for _, n in lens), case["dim"] // 8 * 5
    if case["kind"] == "append":
        pool = (sum(-(-(c + n) // case["page"]) for c, n in lens) + 3) * case["page"] * hk
        return {"bytes": t * ((h + 2 * hk) * d * 2 + h * d * 2 + 2 * hk * row + 20) + 2 * pool * (row + 2 * d),
                "flops": t * (h + hk) * case["rot"] * 3 + t * 2 * hk * d * 4 + 4 * pool * d}
    w, pairs, rows = case["window"], 0, 0
    for c, n in lens:
        rows += (min(c + n, n + w - 1) if w else c + n) if n else 0
        full = n * c + n * (n + 1) // 2                              # all that the rows see without a window
        if w:
            hidden = max(0, c + n - w)                               # of the last row; of those before it one less each
            less = min(n, hidden)
            full -= less * hidden - less * (less - 1) // 2
        pairs += full
    return {"bytes": 2 * rows * hk * row + t * h * d * 4 + 4 * (rows // case["page"] + 3 * case["seqs"]), "flops": 4 * pairs * h * d}


# ---- the same in 64 bits -------------------------------------------------------------------------------------------------------
def _values64(rows, dtype):
    """Of whole rows of a cache: nibble by nibble."""
    d = rows.shape[-1] * 8 // 5
    meta = rows[..., d // 2:].contiguous().view(dtype).double()
    out = torch.empty(*rows.shape[:-1], d, dtype=torch.float64, device=rows.device)
    for i in range(d):
        at = NIBBLE.index(i % 8)
        code = rows[..., i // 8 * 4 + at // 2] >> (4 * (at % 2)) & 15
        out[..., i] = meta[..., i // GROUP * 2 + 1] + meta[..., i // GROUP * 2] * code
    return out.to(dtype).double()


def _stored64(x, dtype):
    """What rows (T, heads, dim) stand for once they have been written: columns of a group between its ends in 15 equal steps."""
    out, bits = torch.empty(x.shape, dtype=torch.float64, device=x.device), 8 if dtype == torch.bfloat16 else 11
    x = x.to(dtype).double()
    for i in range(0, x.shape[-1], GROUP):
        part = x[..., i:i + GROUP]
        low = part.min(-1, keepdim=True).values
        mantissa, power = torch.frexp((part.max(-1, keepdim=True).values - low) / 15)
        step = torch.floor(mantissa * 2.0 ** bits) * torch.exp2((power - bits).double())
        out[..., i:i + GROUP] = low + step * torch.where(step > 0, torch.round((part - low) / step), 0.0).clamp(max=15)
    return out.to(dtype).double()


def _exact_append(case, s):
    """Rows as complex numbers, times e^(i angle)."""
    h, hk, d, half, dtype = case["heads"], case["kv_heads"], case["dim"], case["rot"] // 2, TYPES[case["dtype"]]
    x = s["qkv"].double().view(-1, h + 2 * hk, d)
    at = torch.stack([s["pos"][a] for a in _axes(case)], 1).double() * s["freq"]
    turn = torch.polar(torch.ones_like(at), at)[:, None]
    re, im = (slice(0, half), slice(half, 2 * half)) if case["halves"] else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    z = torch.complex(x[:, :h + hk, re].contiguous(), x[:, :h + hk, im].contiguous()) * turn
    y = x.clone()
    y[:, :h + hk, re], y[:, :h + hk, im] = z.real, z.imag
    k, v = _values64(s["k"], dtype), _values64(s["v"], dtype)
    seq, place, table = s["seq"].tolist(), s["place"].tolist(), s["table"].tolist()
    pages = torch.tensor([table[b][p // case["page"]] for b, p in zip(seq, place)], device="cuda")
    rows = torch.tensor([p % case["page"] for p in place], device="cuda")
    k.index_put_((pages, rows), _stored64(y[:, h:h + hk], dtype))
    v.index_put_((pages, rows), _stored64(y[:, h + hk:], dtype))
    return y[:, :h].reshape(-1, h * d), k, v


def _exact_attention(case, s):
    """One sequence, one key head and a thousand rows at a time."""
    h, hk, d, page, w = case["heads"], case["kv_heads"], case["dim"], case["page"], case["window"]
    g, out, at = h // hk, torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    q = s["q"].double().view(-1, h, d)
    for b, (c, n) in enumerate(_lens(case)):
        ids = s["table"][b, :-(-(c + n) // page)].long()
        for j in range(hk if n else 0):
            k, v = (_values64(x[ids, :, j].reshape(-1, d // 8 * 5)[:c + n], q_type) for x, q_type in ((s["k"], s["q"].dtype), (s["v"], s["q"].dtype)))
            for r in range(0, n, 1024):
                m = min(1024, n - r)
                sees = torch.arange(c + r, c + r + m, device="cuda")[:, None] - torch.arange(c + n, device="cuda")[None]
                hide = (sees < 0) | (sees >= w) if w else sees < 0
                x = (q[at + r:at + r + m, j * g:(j + 1) * g].transpose(0, 1) @ k.T) * d ** -0.5
                o = torch.softmax(x.masked_fill(hide, -math.inf), -1) @ v
                out[at + r:at + r + m].view(m, h, d)[:, j * g:(j + 1) * g] = o.transpose(0, 1)
        at += n
    return out


def _exact_logits(case, s):
    """A row at a time."""
    v, k, out, at = case["vocab"], case["drafts"] + 1, [], 0
    counts, grammars = _bias_counts(case), _mask_rows(case)
    settings = [s[n].double().tolist() for n in ("repetition", "frequency", "presence", "temperature")]
    bits = None
    if s["mask"] is not None:
        bits = torch.stack([s["mask"] >> i & 1 for i in range(32)], -1).flatten(1)[:, :v].bool()
    for r, (b, i) in enumerate((b, i) for b in range(case["seqs"]) for i in range(k)):
        prompt, n = _histories(case)[b] if i == 0 else (prompt, n)
        words, z = s["words"][b].long(), s["logits"][r].double()
        rep, freq, pres, heat = (x[r] for x in settings)
        z = torch.where(torch.isin(torch.arange(v, device="cuda"), words[:n + i]), torch.minimum(z * rep, z / rep) if rep >= 1 else torch.maximum(z * rep, z / rep), z)
        times = torch.bincount(words[min(prompt, n + i):n + i], minlength=v).double()
        z = z - freq * times - pres * times.clamp(max=1.0)
        z.index_put_((s["bias_words"][at:at + counts[r]].long(),), s["bias"][at:at + counts[r]].double(), accumulate=True)
        at += counts[r]
        z = z / heat if heat > 0 else z
        out.append(z.masked_fill(~bits[grammars[r]], -math.inf) if grammars[r] >= 0 else z)
    return torch.stack(out)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logits": _exact_logits}[case["kind"]](case, s)
