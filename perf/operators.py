"""The serving operators' cases, their plain forms and their definitions in 64 bits.

Three operators of one serving step: ``append`` (new tokens into the latent cache, with the latent's
norm and the position rotation), ``prefix`` (decode attention of a batch that shares prefixes) and
``lora`` (a shared projection with the requests' low-rank adapters beside it)."""

import math
import os
import random
import sys

import torch

own = False

DC, DR = 512, 64                       # latent and rope widths of a cache row
WIDTH = DC + DR
SCALE = 1.0 / math.sqrt(128 + DR)      # 1 / sqrt(qk_nope_head_dim + qk_rope_head_dim)
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # one chat request's next token, with the 16 heads of one GPU of eight
        dict(name="append token", op="append", dtype="bf16", batch=1, tokens=1, start=1000, heads=16, page=64,
             norm=True, lens=1),
        # a decode step of a full batch, all 128 heads' queries rotated with it
        dict(name="append batch", op="append", dtype="bf16", batch=256, tokens=1, start=4096, heads=128, page=64,
             norm=True, lens=2),
        # prompts of many lengths arriving at once, into contiguous sequences
        dict(name="append prompts", op="append", dtype="fp16", batch=12, tokens=4099, start=0, heads=16, page=0,
             norm=False, lens=3),
        # four requests behind a short system prompt: latency
        dict(name="prefix small", op="prefix", dtype="bf16", batch=4, heads=16, groups=1, prefix=1000, suffix=33,
             page=64, lens=4),
        # a batch behind one long system prompt, heads split over eight GPUs
        dict(name="prefix h16", op="prefix", dtype="bf16", batch=64, heads=16, groups=1, prefix=8192, suffix=1024,
             page=64, lens=5),
        # several tenants, each with a prompt of its own
        dict(name="prefix groups", op="prefix", dtype="fp16", batch=96, heads=32, groups=8, prefix=16384, suffix=700,
             page=128, lens=6),
        # all 128 heads on one GPU
        dict(name="prefix h128", op="prefix", dtype="bf16", batch=64, heads=128, groups=1, prefix=8192, suffix=512,
             page=64, lens=7),
        # questions about one very long document
        dict(name="prefix document", op="prefix", dtype="bf16", batch=32, heads=16, groups=1, prefix=131072,
             suffix=300, page=0, lens=8),
        # one token through the rope-query projection
        dict(name="lora token", op="lora", dtype="bf16", tokens=1, n=8192, k=5120, rank=16, adapters=4, lens=9),
        # a batch through the output projection, with a dozen fine-tunes loaded
        dict(name="lora batch", op="lora", dtype="bf16", tokens=67, n=7168, k=16384, rank=16, adapters=12, lens=10),
        # a full batch through the absorbed query projection, with many adapters of a high rank
        dict(name="lora wide", op="lora", dtype="bf16", tokens=256, n=65536, k=7168, rank=64, adapters=32, lens=11),
        # a prompt chunk of several requests
        dict(name="lora prompt", op="lora", dtype="fp16", tokens=2051, n=5120, k=16384, rank=32, adapters=4, lens=12),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n + 1 if n == 3072 else n))


def draw(rng):
    op = rng.choice(["append", "prefix", "prefix", "lora"])
    c = dict(op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), lens=rng.randrange(1 << 20))
    if op == "append":
        heads = rng.choice([1, 5, 16, 32, 128])
        batch = _log(rng, 1, 256)
        tokens = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(8192, 700000 // (batch * (heads + 18)))))
        c.update(batch=batch, tokens=tokens, start=_log(rng, 1, 100000 // batch) - 1, heads=heads,
                 page=rng.choice([0, 64, 128, 256]), norm=rng.random() < 0.6)
    elif op == "prefix":
        heads = rng.choice([1, 5, 8, 16, 24, 32, 64, 128])
        batch = _log(rng, 1, 256)
        groups = rng.choice([1, 1, 2, 5, 8])
        groups = min(groups, batch)
        suffix = _log(rng, 1, max(1, min(4096, 200000 // batch)))
        most = int(1.3e11 / (batch * heads * 2 * (DC + WIDTH))) - suffix
        prefix = _log(rng, 1, max(1, min(131072, 300000 // groups, most)))
        c.update(batch=batch, heads=heads, groups=groups, prefix=prefix, suffix=suffix, page=rng.choice([0, 64, 128]))
    else:
        tokens = _log(rng, 1, 2051)
        k = 8 * _log(rng, 16, 2048)
        n = _log(rng, 64, max(64, min(65536, int(3.0e11 / (2.0 * tokens * k)))))
        c.update(tokens=tokens, n=n, k=k + 8 if k == 3072 else k, rank=rng.choice([8, 16, 16, 32, 64]),
                 adapters=_log(rng, 1, 32))
    return c


def _append_counts(c):
    """New tokens and length before of each sequence: whole batches of single tokens, or ragged prompts
    (some sequences bring none)."""
    r = random.Random(c["lens"])
    counts = [c["tokens"] if c["tokens"] == 1 else max(0, r.randint(-c["tokens"] // 8, c["tokens"]))
              for _ in range(c["batch"])]
    counts[0] = c["tokens"]
    return counts, [r.randint(c["start"] // 2, c["start"]) for _ in range(c["batch"])]


def _prefix_lens(c):
    """Requests of each group, prefix length of each group, own length of each request (some have none)."""
    r = random.Random(c["lens"])
    b, g = c["batch"], c["groups"]
    sizes = [(i + 1) * b // g - i * b // g for i in range(g)]
    for i in range(g - 1):                       # uneven groups: a request or so to the next one
        if sizes[i] > 1 and r.random() < 0.5:
            sizes[i] -= 1
            sizes[i + 1] += 1
    prefix = [c["prefix"] if i == 0 else r.randint(c["prefix"] // 8, c["prefix"]) for i in range(g)]
    suffix = [r.randint(0, c["suffix"]) for _ in range(b)]
    suffix[-1] = c["suffix"]
    return sizes, prefix, suffix


def _lora_ids(c):
    """Adapter of each token: requests of one token (small batches) or runs of tokens; one in eight has none."""
    r = random.Random(c["lens"])
    run = 1 if c["tokens"] <= 256 else 97
    ids = []
    while len(ids) < c["tokens"]:
        ids += [-1 if r.random() < 0.125 else r.randrange(c["adapters"])] * run
    ids[0] = 0
    return ids[: c["tokens"]]


def work(c):
    if c["op"] == "append":
        t = sum(_append_counts(c)[0])
        el = DC + DR + c["heads"] * DR
        return {"bytes": t * (4 * el + 4 * DR), "flops": t * (3.0 * (DR + c["heads"] * DR) + (4.0 * DC if c["norm"] else 0))}
    if c["op"] == "prefix":
        sizes, prefix, suffix = _prefix_lens(c)
        pairs = sum(n * p for n, p in zip(sizes, prefix)) + sum(suffix)
        return {"bytes": 2.0 * WIDTH * (sum(prefix) + sum(suffix)) + 2.0 * c["batch"] * c["heads"] * (WIDTH + DC),
                "flops": 2.0 * (WIDTH + DC) * c["heads"] * pairs}
    m, n, k, r = c["tokens"], c["n"], c["k"], c["rank"]
    ids = _lora_ids(c)
    act, with_one = len(set(ids) - {-1}), sum(i >= 0 for i in ids)
    return {"bytes": 2.0 * (n * k + m * k + m * n + act * r * (k + n)),
            "flops": 2.0 * m * n * k + 2.0 * with_one * r * (k + n)}


# ---------------------------------------------------------------------------------------------- inputs

def _pages(counts, page, g, dev, spare):
    """A table of shuffled page ids for sequences of `counts` rows: (len, most pages), and the pool's pages."""
    need = [-(-n // page) for n in counts]
    pool = sum(need) + spare
    ids = torch.randperm(pool, generator=g, device=dev, dtype=torch.int64).to(torch.int32)
    width = max(1, max(need))
    slot = torch.arange(width, device=dev)[None, :]
    n = torch.tensor(need, device=dev)[:, None]
    first = torch.tensor([sum(need[:i]) for i in range(len(need))], device=dev)[:, None]
    table = torch.where(slot < n, ids[(first + slot).clamp(max=pool - 1)], -1).to(torch.int32)
    return table.contiguous(), pool


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dt)

    def ints(v, t=torch.int32):
        return torch.tensor(v, dtype=t, device=dev)

    if c["op"] == "append":
        counts, before = _append_counts(c)
        t, cap = sum(counts), max(a + b for a, b in zip(counts, before))
        s = dict(case=c, c_kv=normal(t, DC, std=2.0), k_rope=normal(t, DR), q_rope=normal(t, c["heads"], DR),
                 cu_tokens=ints([sum(counts[:i]) for i in range(len(counts) + 1)]), seq_lens=ints(before), cap=cap)
        s["weight"] = (1.0 + 0.1 * torch.randn(DC, generator=g, device=dev)).to(dt) if c["norm"] else None
        pos = torch.arange(cap, dtype=torch.float32, device=dev)
        ang = pos[:, None] / 10000.0 ** (torch.arange(0, DR, 2, dtype=torch.float32, device=dev) / DR)[None, :]
        s["cos"], s["sin"] = ang.cos().contiguous(), ang.sin().contiguous()
        if c["page"]:
            s["table"], pool = _pages([a + b for a, b in zip(counts, before)], c["page"], g, dev, 3)
            rows = pool * c["page"]
        else:
            s["offsets"] = ints([i * cap for i in range(len(counts))], torch.int64)
            rows = len(counts) * cap
        s["kv"] = torch.zeros(rows, WIDTH, dtype=dt, device=dev)
        s["q_out"], s["new_lens"] = torch.empty_like(s["q_rope"]), torch.empty_like(s["seq_lens"])
        return s
    if c["op"] == "prefix":
        sizes, prefix, suffix = _prefix_lens(c)
        b, h = c["batch"], c["heads"]
        s = dict(case=c, q_absorbed=normal(b, h, DC, std=0.5), q_rope=normal(b, h, DR),
                 group_starts=ints([sum(sizes[:i]) for i in range(len(sizes) + 1)]), prefix_lens=ints(prefix),
                 seq_lens=ints(suffix), most=max(sizes))
        if c["page"]:
            table, pool = _pages(prefix + suffix, c["page"], g, dev, 2)
            s["prefix_table"], s["table"] = table[: len(prefix)].contiguous(), table[len(prefix):].contiguous()
            s["table"] = s["table"][:, : max(1, -(-c["suffix"] // c["page"]))].contiguous()
            rows = pool * c["page"]
        else:
            at = [0]
            for n in prefix + suffix:
                at.append(at[-1] + n)
            s["prefix_offsets"] = ints(at[: len(prefix)], torch.int64)
            s["offsets"] = ints(at[len(prefix): -1], torch.int64)
            rows = at[-1]
        s["kv"] = normal(rows, WIDTH)
        return s
    m, n, k, r = c["tokens"], c["n"], c["k"], c["rank"]
    return dict(case=c, x=normal(m, k), W=normal(n, k, std=k ** -0.5), A=normal(c["adapters"], r, k, std=k ** -0.5),
                B=normal(c["adapters"], n, r, std=r ** -0.5), ids=ints(_lora_ids(c)),
                scales=0.25 + torch.rand(c["adapters"], generator=g, device=dev))


# ---------------------------------------------------------------------------------------------- one pass

_modules = None


def _framework():
    global _modules
    if _modules is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "latent-attn_b200"))
        from latent_attn import MLAConfig, functional
        _modules = functional, MLAConfig
    return _modules


def run(s):
    c = s["case"]
    if own:
        F, Config = _framework()
        if c["op"] == "append":
            F.mla_cache_append_rope(s["kv"], s["c_kv"], s["k_rope"], s["cu_tokens"], s["seq_lens"], s["cap"],
                                    Config(0, DC, 128, DR, c["heads"], 128), rope_cos=s["cos"], rope_sin=s["sin"],
                                    norm_weight=s["weight"], norm_eps=EPS, kv_offsets=s.get("offsets"),
                                    page_table=s.get("table"), page_rows=c["page"], q_rope=s["q_rope"],
                                    q_out=s["q_out"], new_lens=s["new_lens"])
            return {"cache": s["kv"], "q": s["q_out"], "lens": s["new_lens"]}
        if c["op"] == "prefix":
            return F.mla_prefix_decode(s["kv"], s["q_absorbed"], s["q_rope"], Config(0, DC, 128, DR, c["heads"], 128),
                                       group_starts=s["group_starts"], prefix_lens=s["prefix_lens"],
                                       max_prefix_len=c["prefix"], seq_lens=s["seq_lens"], max_seq_len=c["suffix"],
                                       prefix_offsets=s.get("prefix_offsets"), kv_offsets=s.get("offsets"),
                                       prefix_table=s.get("prefix_table"), page_table=s.get("table"),
                                       page_rows=c["page"])
        return F.linear_lora(s["x"], s["W"], s["A"], s["B"], s["ids"], scales=s["scales"])
    return {"append": _append, "prefix": _prefix, "lora": _lora}[c["op"]](s)


def _row_of(pos, offsets, table, page):
    """Cache rows of positions `pos` (sequences, positions); positions past a table's pages read row 0."""
    if table is None:
        return offsets[:, None] + pos
    ids = table.long().gather(1, (pos // page).clamp(max=table.shape[1] - 1)).clamp(min=0)
    return ids * page + pos % page


def _append(s):
    c = s["case"]
    cu, before = s["cu_tokens"].long(), s["seq_lens"].long()
    t = torch.arange(s["c_kv"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = before[b] + t - cu[b]
    if c["page"]:
        row = s["table"].long()[b, pos // c["page"]] * c["page"] + pos % c["page"]
    else:
        row = s["offsets"][b] + pos
    x = s["c_kv"].float()
    if s["weight"] is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    cos, sin = s["cos"][pos], s["sin"][pos]

    def rotate(v, co, si):
        lo, hi = v[..., : DR // 2], v[..., DR // 2:]
        return torch.cat([lo * co - hi * si, lo * si + hi * co], -1)

    s["kv"][row] = torch.cat([x, rotate(s["k_rope"].float(), cos, sin)], -1).to(s["kv"].dtype)
    s["q_out"].copy_(rotate(s["q_rope"].float(), cos[:, None], sin[:, None]))
    s["new_lens"].copy_(s["seq_lens"] + cu.diff())
    return {"cache": s["kv"], "q": s["q_out"], "lens": s["new_lens"]}


def _prefix(s):
    c, dev = s["case"], s["kv"].device
    q = torch.cat([s["q_absorbed"], s["q_rope"]], -1).float() * SCALE
    bsz, h = q.shape[:2]
    starts, plen, slen = s["group_starts"].long(), s["prefix_lens"].long(), s["seq_lens"].long()
    gid = torch.searchsorted(starts, torch.arange(bsz, device=dev), right=True) - 1
    at = torch.arange(bsz, device=dev) - starts[gid]                     # place within the group
    # the prefixes: all the query rows of a group at once
    pos = torch.arange(c["prefix"], device=dev)[None, :].expand(len(plen), -1)
    rows = _row_of(torch.minimum(pos, (plen[:, None] - 1).clamp(min=0)), s.get("prefix_offsets"), s.get("prefix_table"),
                   c["page"])
    keys = s["kv"][rows.clamp(0, s["kv"].shape[0] - 1)].float()
    qg = torch.zeros(len(plen), s["most"], h, WIDTH, device=dev)
    qg[gid, at] = q
    s1 = torch.matmul(qg.flatten(1, 2), keys.transpose(1, 2))             # (groups, most * h, prefix)
    s1 = torch.where((pos < plen[:, None])[:, None, :], s1, -math.inf)
    # each request's own rows
    pos2 = torch.arange(c["suffix"], device=dev)[None, :].expand(bsz, -1)
    rows2 = _row_of(torch.minimum(pos2, (slen[:, None] - 1).clamp(min=0)), s.get("offsets"), s.get("table"), c["page"])
    keys2 = s["kv"][rows2.clamp(0, s["kv"].shape[0] - 1)].float()
    s2 = torch.matmul(q, keys2.transpose(1, 2))                           # (requests, h, suffix)
    s2 = torch.where((pos2 < slen[:, None])[:, None, :], s2, -math.inf)
    top = torch.maximum(s1.amax(-1).view(len(plen), s["most"], h)[gid, at], s2.amax(-1))
    top = torch.where(top == -math.inf, 0.0, top)
    topg = torch.zeros(len(plen), s["most"], h, device=dev)
    topg[gid, at] = top
    e1 = torch.exp(s1 - topg.flatten(1, 2)[..., None])
    e2 = torch.exp(s2 - top[..., None])
    total = e1.sum(-1).view(len(plen), s["most"], h)[gid, at] + e2.sum(-1)
    o = torch.matmul(e1, keys[..., :DC]).view(len(plen), s["most"], h, DC)[gid, at] + torch.matmul(e2, keys2[..., :DC])
    return torch.where(total[..., None] > 0, o / total[..., None], 0.0).to(s["q_absorbed"].dtype)


def _lora(s):
    x, ids = s["x"].float(), s["ids"].long()
    n_ad, r = s["A"].shape[:2]
    mine = (ids[:, None] == torch.arange(n_ad, device=x.device)[None, :]).float() * s["scales"][None, :]
    u = (x @ s["A"].float().flatten(0, 1).T).view(-1, n_ad, r) * mine[..., None]
    delta = u.flatten(1, 2) @ s["B"].float().transpose(1, 2).flatten(0, 1)
    return (x @ s["W"].float().T + delta).to(s["x"].dtype)


# ---------------------------------------------------------------------------------------------- 64 bits

def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "append":
        counts, before = _append_counts(c)
        kv, q = s["kv"].double(), s["q_out"].double()
        freq_cos, freq_sin = s["cos"].double(), s["sin"].double()
        t = 0
        for b, n in enumerate(counts):
            if not n:
                continue
            p = torch.arange(before[b], before[b] + n, device=kv.device)
            at = s["table"][b].long()[p // c["page"]] * c["page"] + p % c["page"] if c["page"] else s["offsets"][b] + p
            lat = s["c_kv"][t:t + n].double()
            if c["norm"]:
                lat = lat / torch.sqrt(lat.pow(2).sum(-1, keepdim=True) / DC + EPS) * s["weight"].double()
            # the pair (i, i + DR/2) as a complex number, turned by the position's angle
            turn = torch.complex(freq_cos[p], freq_sin[p])
            kr = s["k_rope"][t:t + n].double()
            kc = torch.complex(kr[:, : DR // 2].contiguous(), kr[:, DR // 2:].contiguous()) * turn
            kv[at] = torch.cat([lat, kc.real, kc.imag], 1)
            qr = s["q_rope"][t:t + n].double()
            qc = torch.complex(qr[..., : DR // 2].contiguous(), qr[..., DR // 2:].contiguous()) * turn[:, None, :]
            q[t:t + n] = torch.cat([qc.real, qc.imag], 2)
            t += n
        return {"cache": kv, "q": q, "lens": None}
    if c["op"] == "prefix":
        sizes, prefix, suffix = _prefix_lens(c)
        kv = s["kv"]

        def rows(kind, i, n):
            p = torch.arange(n, device=kv.device)
            if c["page"]:
                return s[("prefix_" if kind else "") + "table"][i].long()[p // c["page"]] * c["page"] + p % c["page"]
            return s[("prefix_" if kind else "") + "offsets"][i] + p

        out, b = [], 0
        for g, n in enumerate(sizes):
            shared = kv[rows(True, g, prefix[g])].double()
            for _ in range(n):
                qa, qr = s["q_absorbed"][b].double(), s["q_rope"][b].double()
                mine = kv[rows(False, b, suffix[b])].double()
                score = torch.cat([qa @ k[:, :DC].T + qr @ k[:, DC:].T for k in (shared, mine)], 1) * SCALE
                if score.shape[1]:
                    p = torch.softmax(score, 1)
                    out.append(p[:, : prefix[g]] @ shared[:, :DC] + p[:, prefix[g]:] @ mine[:, :DC])
                else:
                    out.append(torch.zeros(c["heads"], DC, dtype=torch.float64, device=kv.device))
                b += 1
        return torch.stack(out)
    x, y = s["x"].double(), []
    ids = s["ids"].long()
    for n0 in range(0, c["n"], 8192):
        y.append(x @ s["W"][n0:n0 + 8192].double().T)
    y = torch.cat(y, 1)
    for a in range(c["adapters"]):
        at = (ids == a).nonzero()[:, 0]
        if len(at):
            y[at] += s["scales"][a].double() * ((x[at] @ s["A"][a].double().T) @ s["B"][a].double().T)
    return y
