"""Operators of a decode step of many completions of one prompt, as cases that can be timed and checked.

``attn`` - attention of a batch whose sequences share a long prefix in the paged cache: single new tokens, or several a
sequence (drafts, questions behind a system prompt), a bf16 cache or fp8 rows.  ``logits`` - penalties for tokens that were
there before, biases and grammar masks on the logits in front of the sampler.  ``logprobs`` - the log-probability and the
rank of the sampled tokens, and the likeliest tokens with theirs.

A case's lengths follow from the case; the seed gives their order and all values.
"""
import math

import torch

own = False

BLOCK = 16  # cache positions a page, the engine's default
TAIL = 16  # bytes behind the numbers of an fp8 cache row, the first four its scale
F32, F64 = torch.float32, torch.float64

# query heads, kv heads and head width of the repository's own configurations
HEADS = [(25, 25, 64), (12, 12, 64), (16, 16, 64), (32, 32, 128), (40, 40, 128), (64, 8, 128), (48, 1, 128), (16, 16, 256), (8, 1, 128)]
VOCABS = [32000, 49152, 50257, 50400, 131071]


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # four answers to one question on a small model: latency
        dict(name="attn_4x509", op="attn", nh=25, nkv=25, dim=64, rows=4, prefix=509, own_max=40, q_max=1, idle=0, fp8=False),
        # the benchmark's 64 sequences behind a system prompt
        dict(name="attn_64x2048", op="attn", nh=32, nkv=32, dim=128, rows=64, prefix=2048, own_max=192, q_max=1, idle=2, fp8=False),
        # grouped heads, a document as the prefix, 128 conversations about it: the products count
        dict(name="attn_grouped_128x16381", op="attn", nh=64, nkv=8, dim=128, rows=128, prefix=16381, own_max=500, q_max=1,
             idle=3, fp8=False),
        # a longer document in a quantised cache, fewer readers with longer answers
        dict(name="attn_fp8_23x30011", op="attn", nh=64, nkv=8, dim=128, rows=23, prefix=30011, own_max=1000, q_max=1, idle=0,
             fp8=True),
        # one kv head for all query heads
        dict(name="attn_mqa_33x7990", op="attn", nh=48, nkv=1, dim=128, rows=33, prefix=7990, own_max=200, q_max=1, idle=1, fp8=False),
        # questions of up to 150 tokens behind the same instructions, wide heads
        dict(name="attn_questions_24x1777", op="attn", nh=16, nkv=16, dim=256, rows=24, prefix=1777, own_max=170, q_max=150, idle=1,
             fp8=False),
        # one conversation with a repetition penalty
        dict(name="logits_1x32000", op="logits", rows=1, vocab=32000, fp32=True, known=130, penalties=True, biases=0, masks=0),
        # the benchmark's 64 sequences on an odd vocabulary, each under its own state of a grammar
        dict(name="logits_64x50257", op="logits", rows=64, vocab=50257, fp32=False, known=1000, penalties=True, biases=8, masks=64),
        # a large batch and vocabulary, long contexts, biases of users, few grammars
        dict(name="logits_256x131071", op="logits", rows=256, vocab=131071, fp32=True, known=8000, penalties=True, biases=300, masks=20),
        # one answer with its five likeliest tokens
        dict(name="logprobs_1x32000", op="logprobs", rows=1, vocab=32000, fp32=False, top=5),
        # the benchmark's batch, ranks for best-of-n
        dict(name="logprobs_64x50257", op="logprobs", rows=64, vocab=50257, fp32=False, top=1),
        # a large batch and vocabulary with the twenty likeliest
        dict(name="logprobs_256x131071", op="logprobs", rows=256, vocab=131071, fp32=True, top=20),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _scores(c):
    """Scores that a form with a rectangle a sequence holds: rows x longest portion x heads x keys."""
    return c["rows"] * c["q_max"] * c["nh"] * (c["prefix"] + c["own_max"])


def draw(rng):
    op = rng.choice(["attn", "attn", "logits", "logprobs"])
    if op == "attn":
        nh, nkv, dim = rng.choice(HEADS)
        c = dict(op=op, nh=nh, nkv=nkv, dim=dim, rows=_log(rng, 1, 128), prefix=_log(rng, 40, 32000),
                 q_max=1 if rng.random() < 0.65 else _log(rng, 2, 200), idle=0, fp8=rng.random() < 0.35)
        c["own_max"] = c["q_max"] - 1 + _log(rng, 1, 1000)
        c["idle"] = rng.randint(0, c["rows"] // 8)
        most = listed()[2]
        while _scores(c) > _scores(most) or work(c)["bytes"] > work(most)["bytes"]:
            if c["rows"] == 1:
                c["prefix"], c["q_max"] = c["prefix"] * 2 // 3, max(1, c["q_max"] // 2)
            c["rows"], c["idle"] = max(1, c["rows"] * 2 // 3), 0
        return c
    c = dict(op=op, rows=_log(rng, 1, 256), vocab=rng.choice(VOCABS) if rng.random() < 0.7 else _log(rng, 1000, 131071),
             fp32=rng.random() < 0.5)
    if op == "logprobs":
        c["top"] = rng.choice([1, 1, 5, 20, 64])
        return c
    c.update(known=_log(rng, 4, 8000), penalties=rng.random() < 0.8, biases=rng.choice([0, 0, _log(rng, 1, 300)]),
             masks=rng.choice([0, rng.randint(1, c["rows"])]))
    return c


# ---------------------------------------------------------------------------------------------------------- lengths
def _portions(c):
    """New tokens of each sequence: 1, or evenly from 1 to q_max."""
    n, m = c["rows"], c["q_max"]
    return [1 + (m - 1) * i // max(1, n - 1) if n > 1 else m for i in range(n)]


def _contexts(c):
    """(new tokens, context) of each sequence before its place in the batch is drawn: positions behind the prefix evenly up to
    own_max, at least the new ones; the first of several has its new tokens alone there. Idle rows have a context of 0."""
    got = []
    for i, q in enumerate(_portions(c)):
        mine = q + (c["own_max"] - q) * i // (c["rows"] - 1) if c["rows"] > 1 else c["own_max"]
        got.append([q, 0 if i < c["idle"] else c["prefix"] + mine])
    return got


def _known(c):
    """Known tokens of each row and how many of them are its prompt."""
    n = c["rows"]
    lens = [max(1, c["known"] * (i + 1) // n) for i in range(n)]
    return lens, [k * 3 // 4 for k in lens]


# ----------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 13)


def _order(n, seed):
    return torch.randperm(n, generator=torch.Generator().manual_seed(int(seed) + 5)).tolist()


def _fp8_rows(x):
    """Cache rows of e4m3 numbers with one scale a row."""
    top = x.abs().amax(-1, keepdim=True)
    scale = torch.where(top > 0, top / 448.0, torch.ones_like(top))
    rows = torch.zeros(*x.shape[:-1], x.shape[-1] + TAIL, dtype=torch.uint8, device=x.device)
    rows[..., :x.shape[-1]] = (x / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    rows[..., x.shape[-1]:x.shape[-1] + 4] = scale.contiguous().view(torch.uint8)
    return rows


def prepare(case, seed):
    """What a serving process has in hand: the projections' rows, the cache and its tables; or the step's logits with what is
    known of each row."""
    c, g = case, _gen(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if c["op"] == "attn":
        nh, nkv, dim = c["nh"], c["nkv"], c["dim"]
        seqs = _contexts(c)
        seqs = [seqs[i] for i in _order(len(seqs), seed)]
        pages_p = -(-c["prefix"] // BLOCK)
        width = -(-c["own_max"] // BLOCK)
        pages = pages_p + len(seqs) * width
        ids = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        T = sum(q for q, _ in seqs)
        shape = (pages, nkv, BLOCK, dim)
        k, v = randn(*shape), randn(*shape)
        # keys share a direction and queries lean on it, as in trained heads: some positions weigh far more than others
        lean = randn(1, nkv, 1, dim)
        k = k + lean * randn(pages, nkv, BLOCK, 1) * 0.5
        qkv = randn(T, (nh + 2 * nkv) * dim)
        qkv[:, :nh * dim] += (lean.view(nkv, 1, dim).expand(nkv, nh // nkv, dim).reshape(1, -1)) * 0.5
        caches = (_fp8_rows(k), _fp8_rows(v)) if c["fp8"] else (k.to(torch.bfloat16), v.to(torch.bfloat16))
        cu = [0]
        for q, _ in seqs:
            cu.append(cu[-1] + q)
        i32 = dict(dtype=torch.int32, device="cuda")
        return dict(case=c, qkv=qkv.to(torch.bfloat16), k=caches[0], v=caches[1], prefix_table=ids[:pages_p].contiguous(),
                    tables=ids[pages_p:].view(len(seqs), width).contiguous(), ctx=torch.tensor([n for _, n in seqs], **i32),
                    cu=torch.tensor(cu, **i32), scale=1.0 / math.sqrt(dim))
    V, n = c["vocab"], c["rows"]
    wide = -(-V // 64) * 64  # the head's columns, padded
    x = randn(n, wide) * 2.5 + randn(1, wide) * 1.5
    logits = x if c["fp32"] else x.to(torch.bfloat16)
    if c["op"] == "logprobs":
        # mostly likely tokens, now and then any
        likely = (logits[:, :V].float() + 3 * randn(n, V)).argmax(-1)
        other = torch.randint(0, V, (n,), generator=g, device="cuda")
        return dict(case=c, logits=logits, tokens=torch.where(randn(n) > 1.2, other, likely))
    lens, prompts = _known(c)
    order = _order(n, seed)
    lens, prompts = [lens[i] for i in order], [prompts[i] for i in order]
    # few tokens come again and again, most once or never
    u = torch.rand(n, c["known"], generator=g, device="cuda")
    known = (torch.exp(u * math.log(V)) - 1).long().clamp(0, V - 1)
    shuffle = torch.randperm(V, generator=g, device="cuda")
    known = shuffle[known]
    i32 = dict(dtype=torch.int32, device="cuda")
    s = dict(case=c, logits=logits, ids=known, lens=torch.tensor(lens, **i32), prompts=torch.tensor(prompts, **i32),
             repetition=None, presence=None, frequency=None, bias_ids=None, bias=None, mask=None, mask_rows=None)
    if c["penalties"]:
        s["repetition"] = 1 + 0.5 * torch.rand(n, generator=g, device="cuda")
        s["presence"] = torch.rand(n, generator=g, device="cuda") * 1.5
        s["frequency"] = torch.rand(n, generator=g, device="cuda") * 0.5
    if c["biases"]:
        at = torch.randint(0, V, (n, c["biases"]), generator=g, device="cuda", dtype=torch.int32)
        last = torch.arange(c["biases"], device="cuda")[None, :] >= c["biases"] - torch.arange(n, device="cuda")[:, None] % c["biases"]
        s["bias_ids"] = torch.where(last, -1, at).to(torch.int32)  # rows with fewer biases than the widest
        s["bias"] = randn(n, c["biases"]) * 5
    if c["masks"]:
        words = -(-V // 32)
        bits = torch.randint(-2 ** 31, 2 ** 31, (c["masks"], words), generator=g, device="cuda")
        thin = torch.randint(-2 ** 31, 2 ** 31, (4, c["masks"], words), generator=g, device="cuda")
        # a state allows half of the words' tokens, or few of them; the last state of several allows none
        few = (torch.arange(c["masks"], device="cuda") % 2 == 0)[:, None]
        bits = torch.where(few, bits & thin[0] & thin[1] & thin[2] & thin[3], bits)
        if c["masks"] > 2:
            bits[-1] = 0
        s["mask"] = bits.to(torch.int32)
        rows = torch.randint(-1, c["masks"], (n,), generator=g, device="cuda", dtype=torch.int32)
        s["mask_rows"] = rows
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
def _values(cache, pages, dim):
    """Rows of the pages as 32-bit numbers [.., kv heads, positions of a page, dim]."""
    rows = cache[pages.long()]
    if rows.dtype == torch.uint8:
        scale = rows[..., dim:dim + 4].contiguous().view(F32)
        return rows[..., :dim].contiguous().view(torch.float8_e4m3fn).to(F32) * scale
    return rows.to(F32)


def _attn_plain(s):
    c = s["case"]
    nh, nkv, dim, P, Q = c["nh"], c["nkv"], c["dim"], c["prefix"], c["q_max"]
    G, T, n = nh // nkv, s["qkv"].shape[0], s["ctx"].shape[0]
    dev = s["qkv"].device
    cu, ctx = s["cu"].long(), s["ctx"].long()
    qlen = cu[1:] - cu[:-1]
    i = torch.arange(Q, device=dev)
    token = (cu[:-1, None] + i).clamp(max=T - 1)  # [n, Q], a sequence's tokens from the left
    there = i[None, :] < qlen[:, None]
    seen = torch.where(there, ctx[:, None] - qlen[:, None] + i + 1, 0).clamp(min=0)  # positions that a token sees
    q = s["qkv"][:, :nh * dim].to(F32)[token].view(n, Q, nkv, G, dim).permute(2, 0, 3, 1, 4)  # [nkv, n, G, Q, dim]
    kp, vp = (_values(s[w], s["prefix_table"], dim).permute(1, 0, 2, 3).reshape(nkv, -1, dim)[:, :P] for w in ("k", "v"))
    ko, vo = (_values(s[w], s["tables"], dim).permute(2, 0, 1, 3, 4).reshape(nkv, n, -1, dim) for w in ("k", "v"))
    S = ko.shape[2]
    sp = torch.matmul(q.reshape(nkv, n * G * Q, dim), kp.transpose(1, 2).contiguous()).view(nkv, n, G, Q, P) * s["scale"]
    so = torch.matmul(q.reshape(nkv, n, G * Q, dim), ko.transpose(2, 3).contiguous()).view(nkv, n, G, Q, S) * s["scale"]
    none = torch.tensor(float("-inf"), device=dev)
    sp = torch.where((torch.arange(P, device=dev) < seen[..., None])[None, :, None], sp, none)
    so = torch.where((P + torch.arange(S, device=dev) < seen[..., None])[None, :, None], so, none)
    top = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    top = torch.where(top == none, torch.zeros_like(top), top)
    sp, so = torch.exp(sp - top), torch.exp(so - top)
    total = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
    vo = torch.where((P + torch.arange(S, device=dev) < ctx[:, None])[None, :, :, None], vo, torch.zeros((), device=dev))
    o = torch.matmul(sp.reshape(nkv, n * G * Q, P), vp).view(nkv, n, G, Q, dim)
    o = o + torch.matmul(so.reshape(nkv, n, G * Q, S), vo).view(nkv, n, G, Q, dim)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(1, 3, 0, 2, 4).reshape(n, Q, nh * dim)
    return o[there].to(torch.bfloat16)  # sequence by sequence, as the tokens lie


def _logits_plain(s):
    c = s["case"]
    n, V = c["rows"], c["vocab"]
    dev = s["logits"].device
    y = s["logits"][:, :V].to(F32)
    place = torch.arange(s["ids"].shape[1], device=dev)[None, :]
    known = place < s["lens"][:, None]
    said = known & (place >= s["prompts"][:, None])
    seen = torch.zeros(n, V, device=dev).scatter_add_(1, s["ids"], known.to(F32)) > 0
    count = torch.zeros(n, V, device=dev).scatter_add_(1, s["ids"], said.to(F32))
    if s["repetition"] is not None:
        r = s["repetition"][:, None]
        y = torch.where(seen, torch.where(y > 0, y / r, y * r), y)
        y = y - count * s["frequency"][:, None]
        y = torch.where(count > 0, y - s["presence"][:, None], y)
    if s["bias"] is not None:
        used = s["bias_ids"] >= 0
        y = y + torch.zeros(n, V, device=dev).scatter_add_(1, s["bias_ids"].clamp(min=0).long(), torch.where(used, s["bias"], 0.0))
    if s["mask"] is not None:
        t = torch.arange(V, device=dev)
        bits = (s["mask"][:, t >> 5] >> (t & 31)) & 1
        open_ = (bits[s["mask_rows"].clamp(min=0).long()] != 0) | (s["mask_rows"] < 0)[:, None]
        y = torch.where(open_, y, torch.tensor(float("-inf"), device=dev))
    return y.to(s["logits"].dtype)


def _logprobs_plain(s):
    c = s["case"]
    x = s["logits"][:, :c["vocab"]].to(F32)
    top = x.amax(-1, keepdim=True)
    total = torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    mine = torch.gather(x, 1, s["tokens"][:, None])
    rank = (x > mine).sum(-1) + 1
    value, at = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lowest index first
    return [((mine - top) - total)[:, 0], rank, at[:, :c["top"]].contiguous(), (value[:, :c["top"]] - top) - total]


# -------------------------------------------------------------------------------------------------------------- run
def run(state):
    s, c = state, state["case"]
    if own:
        from llmss_amd import ops

        if c["op"] == "attn":
            several = c["q_max"] > 1
            return ops.attn_shared(s["qkv"], s["k"], s["v"], s["prefix_table"], c["prefix"], s["tables"], s["ctx"], c["nh"],
                                   c["nkv"], c["dim"], s["scale"], cu_q=s["cu"] if several else None, max_qlen=c["q_max"],
                                   max_own=c["own_max"])
        if c["op"] == "logits":
            return ops.adjust_logits(s["logits"], s["ids"], s["lens"], s["prompts"], repetition=s["repetition"],
                                     presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"], bias=s["bias"],
                                     mask=s["mask"], mask_rows=s["mask_rows"], vocab=c["vocab"])
        return list(ops.token_logprobs(s["logits"], s["tokens"], c["top"], vocab=c["vocab"]))
    return {"attn": _attn_plain, "logits": _logits_plain, "logprobs": _logprobs_plain}[c["op"]](s)


def work(case):
    c = case
    if c["op"] == "attn":
        nh, nkv, dim, P = c["nh"], c["nkv"], c["dim"], c["prefix"]
        row = dim + 4 if c["fp8"] else 2 * dim
        T = keys = mine = 0
        for q, ctx in _contexts(c):
            T += q
            if ctx:
                mine += ctx - P
                keys += q * ctx - q * (q - 1) // 2
        return {"bytes": 2 * nkv * row * (P + mine) + 4 * T * nh * dim, "flops": 4 * nh * dim * keys}
    n, V = c["rows"], c["vocab"]
    size = 4 if c["fp32"] else 2
    if c["op"] == "logprobs":
        return {"bytes": n * V * size + n * (8 + 4 + 8 + 12 * c["top"]), "flops": 3 * n * V}
    lens, _ = _known(c)
    known = 8 * sum(lens) if c["penalties"] else 0
    return {"bytes": 2 * n * V * size + known + 8 * n * c["biases"] + c["masks"] * -(-V // 32) * 4, "flops": 2 * n * V}


# ------------------------------------------------------------------------------------------ the definitions in 64 bits
def _row64(cache, page, at, dim):
    """Positions `at` of the pages `page`, all kv heads: [positions, kv heads, dim]."""
    r = cache[page, :, at]
    if r.dtype == torch.uint8:
        return r[..., :dim].contiguous().view(torch.float8_e4m3fn).to(F64) * r[..., dim:dim + 4].contiguous().view(F32).to(F64)
    return r.to(F64)


def _attn_exact(c, s):
    nh, nkv, dim, P = c["nh"], c["nkv"], c["dim"], c["prefix"]
    G = nh // nkv
    out = torch.zeros(s["qkv"].shape[0], nh, dim, dtype=F64, device="cuda")
    j = torch.arange(P, device="cuda")
    page, at = s["prefix_table"].long()[j // BLOCK], j % BLOCK
    kp, vp = _row64(s["k"], page, at, dim), _row64(s["v"], page, at, dim)
    cu, ctx = s["cu"].tolist(), s["ctx"].tolist()
    for b in range(len(ctx)):
        a, e = cu[b], cu[b + 1]
        if not ctx[b]:
            continue
        j = torch.arange(max(0, ctx[b] - P), device="cuda")
        page, at = s["tables"][b].long()[j // BLOCK], j % BLOCK
        q = s["qkv"][a:e, :nh * dim].to(F64).view(e - a, nkv, G, dim)
        last = torch.arange(ctx[b] - (e - a), ctx[b], device="cuda")
        hidden = torch.arange(ctx[b], device="cuda")[None, :] > last[:, None]
        k, v = torch.cat([kp[:ctx[b]], _row64(s["k"], page, at, dim)]), torch.cat([vp[:ctx[b]], _row64(s["v"], page, at, dim)])
        for h in range(nkv):
            w = torch.mm(q[:, h].reshape(-1, dim), k[:, h].t().contiguous()).view(e - a, G, -1) * s["scale"]
            w = torch.softmax(w.masked_fill(hidden[:, None, :], float("-inf")), -1)
            out[a:e, h * G:(h + 1) * G] = torch.mm(w.view((e - a) * G, -1), v[:, h].contiguous()).view(e - a, G, dim)
    return out.view(-1, nh * dim)


def _logits_exact(c, s):
    V = c["vocab"]
    y = s["logits"][:, :V].to(F64)
    lens, prompts = s["lens"].tolist(), s["prompts"].tolist()
    for b in range(c["rows"]):
        row = y[b]
        if s["repetition"] is not None:
            every = torch.unique(s["ids"][b, :lens[b]])
            x = row[every]
            row[every] = torch.where(x > 0, x / s["repetition"][b].double(), x * s["repetition"][b].double())
            said, times = torch.unique(s["ids"][b, prompts[b]:lens[b]], return_counts=True)
            row[said] -= times * s["frequency"][b].double() + s["presence"][b].double()
        if s["bias"] is not None:
            use = s["bias_ids"][b] >= 0
            row.index_put_((s["bias_ids"][b][use].long(),), s["bias"][b][use].double(), accumulate=True)
        if s["mask"] is not None and int(s["mask_rows"][b]) >= 0:
            word = s["mask"][int(s["mask_rows"][b])].long() & 0xFFFFFFFF
            bits = (word[:, None] >> torch.arange(32, device="cuda")) & 1
            row[bits.view(-1)[:V] == 0] = float("-inf")
    return y


def _logprobs_exact(c, s):
    x = s["logits"][:, :c["vocab"]].to(F64)
    lp = torch.log_softmax(x, -1)
    mine = lp[torch.arange(c["rows"], device="cuda"), s["tokens"]]
    rank = 1 + (x > x[torch.arange(c["rows"], device="cuda"), s["tokens"]][:, None]).sum(-1)
    at = torch.argsort(-x, dim=-1, stable=True)[:, :c["top"]]
    return [mine, rank, at, torch.gather(lp, 1, at)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _attn_exact, "logits": _logits_exact, "logprobs": _logprobs_exact}[case["op"]](case, s)
