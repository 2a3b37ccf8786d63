"""Cases for the serving operators around the cache: what a server runs next to compression.

Five calls of ``nexusquant_b200.kernels`` in four operators:

  rope     norm_rope_qk: RMS norm of every query and key head (optional), split-half position
           rotation, and the store of the rotated keys and the values into cache pages.
  prompt   attend_prompt: causal attention of packed sequences of different lengths, grouped
           heads; the keys of a sequence may start before its queries (a later chunk).
  decode   attend_pages: one query token per sequence against a prefix that the whole batch
           shares (read once for all) followed by each sequence's own pages.
  pages    copy_pages (a fork copies the partly filled last pages) and compact_pages (the kept
           tokens of an eviction move to the front of fresh pages).

Pages are [n_pages, heads, page, head_dim] per layer.  Keys have four outlier channels scaled by
8, as in nexusquant_b200.synthetic.  ``run`` computes the plain form in torch (fp32, rounded
once) or, with ``own``, calls the framework.  Rotation angles are position * inverse frequency
with both in fp32: that rounding is part of the operator (models are trained with it).
"""
import math
import random

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_EB = {"fp16": 2, "bf16": 2, "fp32": 4}
_BASE = 10000.0
_EPS = 1e-6


def listed():
    return [
        # one decoding step of eight requests: the keys of the new tokens are normed, rotated and stored
        dict(name="rope_step", op="rope", n=8, hq=32, h=8, d=128, dt="bf16", norm=True, fused=True, page=16),
        # a 16384-token prompt batch at 64 query heads, 8 KV heads, out of one fused projection
        dict(name="rope_prompt", op="rope", n=16384, hq=64, h=8, d=128, dt="fp16", norm=True, fused=True, page=64),
        # three chat turns arriving together: latency counts
        dict(name="prompt_short", op="prompt", seqs=3, n=203, past=0, hq=16, h=2, d=64, dt="bf16", fused=False, cut=11),
        # twelve prompts of different lengths packed to one batch, heads read from a fused projection
        dict(name="prompt_packed", op="prompt", seqs=12, n=8191, past=0, hq=32, h=8, d=128, dt="fp16", fused=True,
             cut=12),
        # one long document
        dict(name="prompt_long", op="prompt", seqs=1, n=16384, past=0, hq=32, h=8, d=128, dt="bf16", fused=False,
             cut=13),
        # the next chunk of two long prompts whose first 15000 tokens are already cached (32 KV heads of 96)
        dict(name="prompt_chunk", op="prompt", seqs=2, n=1000, past=15000, hq=32, h=32, d=96, dt="fp16", fused=False,
             cut=14),
        # three requests with one system prompt, just begun
        dict(name="decode_small", op="decode", b=3, prefix=700, own_len=60, hq=32, h=8, d=128, dt="fp16", page=16,
             cut=21),
        # 64 samples of one 32768-token context
        dict(name="decode_shared", op="decode", b=64, prefix=32768, own_len=500, hq=32, h=8, d=128, dt="bf16",
             page=64, cut=22),
        # sixteen requests with nothing in common, long contexts of their own
        dict(name="decode_own", op="decode", b=16, prefix=0, own_len=9000, hq=64, h=8, d=128, dt="fp16", page=16,
             cut=23),
        # 24 forks: the partly filled last page of each, in all 32 layers
        dict(name="fork_copy", op="copy", layers=32, pages=24, h=8, d=128, dt="fp16", page=16, cut=31),
        # two short requests after eviction, four layers
        dict(name="compact_short", op="compact", layers=4, b=2, n=900, keep=0.65, h=32, d=96, dt="fp16", page=16,
             cut=32),
        # a 32768-token context, 60 % evicted, four layers of 8 heads
        dict(name="compact_long", op="compact", layers=4, b=1, n=32768, keep=0.4, h=8, d=128, dt="fp16", page=64,
             cut=33),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "prompt", "prompt", "decode", "decode", "copy", "compact"])
    h, g = rng.choice([(2, 8), (8, 1), (8, 4), (8, 8), (4, 3), (32, 1), (4, 7), (1, 16)])
    c = dict(op=op, h=h, d=rng.choice([64, 96, 128, 128]), dt=rng.choice(["fp16", "bf16"]),
             page=rng.choice([16, 32, 64, 128]))
    cut = rng.randrange(1 << 30)
    if op == "rope":
        c.update(n=_log(rng, 1, 16384), hq=h * g, norm=rng.random() < 0.6, fused=rng.random() < 0.5)
    elif op == "prompt":
        c.pop("page")
        past = rng.choice([0, 0, 0, _log(rng, 1, 12000)])
        n = _log(rng, 1, 12000 if past == 0 else 1500)
        c.update(hq=h * g, n=n, past=past, seqs=min(n, rng.choice([1, 2, 3, 5, 9, 20])), fused=rng.random() < 0.3,
                 cut=cut)
        most = 8e9 / max(1, h * g) / max(1, c["seqs"])  # logits of the padded batch, in elements
        while _longest(c) * (_longest(c) + past) > most:
            c["n"] = max(c["seqs"], c["n"] * 3 // 4)
            c["past"] = past = past * 3 // 4
    elif op == "decode":
        c.update(hq=h * g, b=_log(rng, 1, 96), prefix=rng.choice([0, _log(rng, 1, 32768), _log(rng, 64, 32768)]),
                 own_len=_log(rng, 1, 4000), cut=cut)
        while c["b"] * c["own_len"] * h > 1_000_000:
            c["own_len"] = c["own_len"] * 3 // 4
    elif op == "copy":
        c.update(layers=_log(rng, 1, 32), pages=_log(rng, 1, 64), cut=cut)
        while c["layers"] * c["pages"] * c["page"] * h > 1_000_000:
            c["pages"] = max(1, c["pages"] // 2)
            c["layers"] = max(1, c["layers"] // 2)
    else:
        c.update(layers=_log(rng, 1, 8), b=rng.choice([1, 1, 2, 5]), n=_log(rng, 1, 20000),
                 keep=rng.choice([0.2, 0.4, 0.65, 1.0]), cut=cut)
        while c["layers"] * c["b"] * c["n"] * h > 1_000_000:
            c["n"] = max(1, c["n"] // 2)
    return c


# ------------------------------------------------------------------------------------ sizes of a case
def _cut(total, parts, seed):
    """``total`` tokens in ``parts`` sequences of one or more, unequal."""
    rng = random.Random(seed)
    w = [rng.uniform(0.2, 2.0) for _ in range(parts)]
    lens = [max(1, int(total * x / sum(w))) for x in w]
    lens[lens.index(max(lens))] += total - sum(lens)
    return lens


def _longest(c):
    return max(_cut(c["n"], c["seqs"], c["cut"]))


def _past(c):
    """Cached tokens before each sequence's queries: about ``past``."""
    rng = random.Random(c["cut"] + 1)
    return [int(c["past"] * rng.uniform(0.6, 1.0)) for _ in range(c["seqs"])]


def _own_lens(c):
    rng = random.Random(c["cut"])
    lens = [rng.randint(1, c["own_len"]) for _ in range(c["b"])]
    lens[0] = c["own_len"]
    if c["prefix"] and c["b"] > 1:
        lens[-1] = 0  # forked this very step: nothing of its own yet
    return lens


def _kept_counts(c):
    rng = random.Random(c["cut"])
    return [max(1, min(c["n"], int(c["n"] * c["keep"] * rng.uniform(0.8, 1.0)))) for _ in range(c["b"])]


def _ceil(a, b):
    return -(-a // b)


# ------------------------------------------------------------------------------------ inputs
def _keys(shape, d, dt, g):
    """N(0, 1) with four outlier channels scaled by 8."""
    k = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    ch = torch.randperm(d, generator=g, device="cuda")[:4]
    k[..., ch] *= 8.0
    return k.to(dt)


def _normal(shape, dt, g):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, h, d, op = _DT[case["dt"]], case["h"], case["d"], case["op"]
    s = {"case": dict(case)}
    if op in ("rope", "prompt"):
        hq, n = case["hq"], case["n"]
        nk = n if op == "rope" else n + sum(_past(case))
        if case["fused"] and nk == n:
            x = _normal((n, hq + 2 * h, d), dt, g)
            x[:, hq:hq + h] = _keys((n, h, d), d, dt, g)
            s["q"], s["k"], s["v"] = x[:, :hq], x[:, hq:hq + h], x[:, hq + h:]
        else:
            s["q"], s["k"], s["v"] = _normal((n, hq, d), dt, g), _keys((nk, h, d), d, dt, g), _normal((nk, h, d), dt, g)
    if op == "rope":
        page = case["page"]
        n_pages = _ceil(n, page) + 2
        # a decoding step is somewhere in a long context; a prompt starts at 0
        first = int(torch.randint(0, 30000, (1,), generator=g, device="cuda")) if n < 64 else 0
        s["positions"] = torch.arange(first, first + n, device="cuda", dtype=torch.int32)
        s["rows"] = first + n
        order = torch.randperm(n_pages, generator=g, device="cuda")
        t = torch.arange(n, device="cuda")
        s["slots"] = (order[t // page] * page + t % page).to(torch.int32)
        s["k_pages"] = torch.zeros((n_pages, h, page, d), dtype=dt, device="cuda")
        s["v_pages"] = torch.zeros_like(s["k_pages"])
        s["wq"] = s["wk"] = None
        if case["norm"]:
            s["wq"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
            s["wk"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
    elif op == "prompt":
        lens = _cut(n, case["seqs"], case["cut"])
        klens = [a + b for a, b in zip(lens, _past(case))]
        s["longest"], s["longest_k"] = max(lens), max(klens)
        at, atk = [0], [0]
        for a, b in zip(lens, klens):
            at.append(at[-1] + a)
            atk.append(atk[-1] + b)
        s["starts"], s["k_starts"] = _ints(at), _ints(atk)
    elif op == "decode":
        page, lens = case["page"], _own_lens(case)
        pre, width = _ceil(case["prefix"], page), _ceil(max(lens), page)
        n_pages = pre + case["b"] * width + 1
        s["q"] = _normal((case["b"], case["hq"], d), dt, g)
        s["k_pages"], s["v_pages"] = _keys((n_pages, h, page, d), d, dt, g), _normal((n_pages, h, page, d), dt, g)
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        s["prefix_table"], s["tables"] = order[:pre].clone(), order[pre:pre + case["b"] * width].view(case["b"], width)
        s["lens"], s["max_len"] = _ints(lens), max(lens)
    elif op == "copy":
        n_pages = 2 * case["pages"] + 3
        shape = (case["layers"], n_pages, h, case["page"], d)
        s["k_pages"], s["v_pages"] = _normal(shape, dt, g), _normal(shape, dt, g)
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        s["src"], s["dst"] = order[:case["pages"]].clone(), order[case["pages"]:2 * case["pages"]].clone()
    else:
        page, b, n, counts = case["page"], case["b"], case["n"], _kept_counts(case)
        width, to = _ceil(n, page), _ceil(max(counts), page)
        n_pages = b * (width + to)
        shape = (case["layers"], n_pages, h, page, d)
        s["k_pages"], s["v_pages"] = _normal(shape, dt, g), _normal(shape, dt, g)
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        s["tables"], s["dst_tables"] = order[:b * width].view(b, width), order[b * width:].view(b, to)
        # the shape of an importance ranking's keep set: the first token, the newest, and a scattered rest
        score = torch.rand((b, n), generator=g, device="cuda")
        score[:, 0] = 3.0
        score[:, max(0, n - 32):] += 2.0
        rank = score.argsort(dim=1, descending=True)
        idx = torch.full((b, n), n, dtype=torch.int64, device="cuda")
        for i, m in enumerate(counts):
            idx[i, :m] = rank[i, :m].sort().values
        s["kept_idx"], s["kept_count"], s["max_kept"] = idx.to(torch.int32), _ints(counts), max(counts)
    return s


# ------------------------------------------------------------------------------------ one pass
def run(state):
    return (_run_own if own else _run_plain)(state["case"]["op"], state)


def _run_own(op, s):
    from nexusquant_b200 import kernels as K
    if op == "rope":
        q, _ = K.norm_rope_qk(s["q"], s["k"], s["positions"], q_weight=s["wq"], k_weight=s["wk"], eps=_EPS, v=s["v"],
                              k_pages=s["k_pages"], v_pages=s["v_pages"], slots=s["slots"], rope_base=_BASE,
                              rope_rows=s["rows"])
        return q, s["k_pages"], s["v_pages"]
    if op == "prompt":
        return K.attend_prompt(s["q"], s["k"], s["v"], s["starts"], k_starts=s["k_starts"])
    if op == "decode":
        return K.attend_pages(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lens"],
                              prefix_table=s["prefix_table"], prefix_len=s["case"]["prefix"], max_len=s["max_len"])
    if op == "copy":
        K.copy_pages(s["k_pages"], s["v_pages"], s["src"], s["dst"])
    else:
        K.compact_pages(s["k_pages"], s["v_pages"], s["tables"], s["kept_idx"], s["kept_count"], s["dst_tables"],
                        max_kept=s["max_kept"])
    return s["k_pages"], s["v_pages"]


def _run_plain(op, s):
    return {"rope": _rope, "prompt": _prompt, "decode": _decode, "copy": _copy, "compact": _compact}[op](s)


def _rotated(x, w, cos, sin):
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _rope(s):
    d, page = s["case"]["d"], s["case"]["page"]
    inv = _inv_freq(d).cuda()
    angle = s["positions"].float()[:, None] * inv
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    q = _rotated(s["q"], s["wq"], cos, sin).to(s["q"].dtype)
    k = _rotated(s["k"], s["wk"], cos, sin).to(s["k"].dtype)
    slot = s["slots"].long()
    s["k_pages"][slot // page, :, slot % page] = k
    s["v_pages"][slot // page, :, slot % page] = s["v"]
    return q, s["k_pages"], s["v_pages"]


def _inv_freq(d):
    return 1.0 / (_BASE ** (torch.arange(0, d, 2, dtype=torch.float32) / d))


def _padded(starts, longest, x):
    """Rows of the packed x [n, heads, d] as [seqs, heads, longest, d] and each row's index."""
    row = starts[:-1, None].long() + torch.arange(longest, device=x.device)
    row = row.clamp(max=x.shape[0] - 1)
    return x[row].transpose(1, 2).float(), row


def _prompt(s):
    c = s["case"]
    h, d, gq, lq, lk = c["h"], c["d"], c["hq"] // c["h"], s["longest"], s["longest_k"]
    q, row = _padded(s["starts"], lq, s["q"])
    k, _ = _padded(s["k_starts"], lk, s["k"])
    v, _ = _padded(s["k_starts"], lk, s["v"])
    n_seq = q.shape[0]
    nq, nk = (s["starts"][1:] - s["starts"][:-1]).long(), (s["k_starts"][1:] - s["k_starts"][:-1]).long()
    i, j = torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda")
    # query i stands at key position nk - nq + i
    hidden = j[None, None, :] > (nk - nq)[:, None, None] + i[None, :, None]
    x = (q.reshape(n_seq, h, gq * lq, d) * d ** -0.5) @ k.transpose(2, 3)
    x = x.view(n_seq, h, gq, lq, lk).masked_fill_(hidden[:, None, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    y = (x.view(n_seq, h, gq * lq, lk) @ v).view(n_seq, h, gq, lq, d) / total
    y = y.reshape(n_seq, c["hq"], lq, d).transpose(1, 2).to(s["q"].dtype)
    return y[i[None, :] < nq[:, None]]


def _decode(s):
    c = s["case"]
    b, h, d, gq, page, pre = c["b"], c["h"], c["d"], c["hq"] // c["h"], c["page"], c["prefix"]
    q = s["q"].float().view(b, h, gq, d) * d ** -0.5
    own_k, own_v = (_pages(p, s["tables"]) for p in (s["k_pages"], s["v_pages"]))
    x = q @ own_k.transpose(2, 3)
    j = torch.arange(x.shape[-1], device="cuda")
    x = x.masked_fill_((j >= s["lens"][:, None])[:, None, None], -math.inf)
    if pre:
        pk, pv = (_pages(p, s["prefix_table"][None])[0, :, :pre] for p in (s["k_pages"], s["v_pages"]))
        x = torch.cat([torch.einsum("bhgd,hjd->bhgj", q, pk), x], dim=-1)
    x = (x - x.amax(-1, keepdim=True)).exp()
    total = x.sum(-1, keepdim=True)
    y = x[..., pre:] @ own_v
    if pre:
        y = y + torch.einsum("bhgj,hjd->bhgd", x[..., :pre], pv)
    return (y / total).reshape(b, c["hq"], d).to(s["q"].dtype)


def _pages(p, tables):
    """[b, heads, tokens, d] of page tables [b, width], fp32."""
    x = p[tables.long()]
    return x.transpose(1, 2).reshape(x.shape[0], x.shape[2], -1, x.shape[4]).float()


def _copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k_pages"][:, dst] = s["k_pages"][:, src]
    s["v_pages"][:, dst] = s["v_pages"][:, src]
    return s["k_pages"], s["v_pages"]


def _compact(s):
    page, n = s["case"]["page"], s["max_kept"]
    j = torch.arange(n, device="cuda")
    valid = j[None, :] < s["kept_count"][:, None]
    idx = s["kept_idx"][:, :n].long().clamp(max=s["case"]["n"] - 1)
    src_page = s["tables"].long().gather(1, idx // page)[valid]
    src_off = (idx % page)[valid]
    dst_page = s["dst_tables"].long()[:, j // page][valid]
    dst_off = (j % page).expand_as(idx)[valid]
    s["k_pages"][:, dst_page, :, dst_off] = s["k_pages"][:, src_page, :, src_off]
    s["v_pages"][:, dst_page, :, dst_off] = s["v_pages"][:, src_page, :, src_off]
    return s["k_pages"], s["v_pages"]


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("copy", "compact"):
        return _moved(s, "k_pages"), _moved(s, "v_pages")  # copies: the values themselves
    if op == "rope":
        pos = s["positions"].cpu().float()
        ang = torch.outer(pos, _inv_freq(case["d"])).double().cuda()
        turn = torch.polar(torch.ones_like(ang), ang)[:, None, :]

        def one(x, w):
            x = x.double()
            if w is not None:
                x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / case["d"] + _EPS) * w.double()
            half = case["d"] // 2
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
            return torch.cat([z.real, z.imag], -1)

        pool = s["k_pages"].double()
        flat = pool.transpose(1, 2).reshape(-1, case["h"], case["d"])
        flat[s["slots"].long()] = one(s["k"], s["wk"])
        pool = flat.view(-1, case["page"], case["h"], case["d"]).transpose(1, 2)
        return one(s["q"], s["wq"]), pool, None
    g = case["hq"] // case["h"]
    scale = 1.0 / math.sqrt(case["d"])
    if op == "prompt":
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        st, kst = s["starts"].tolist(), s["k_starts"].tolist()
        for a, b, ka, kb in zip(st, st[1:], kst, kst[1:]):
            i = torch.arange(b - a, device="cuda") + (kb - ka) - (b - a)
            seen = torch.arange(kb - ka, device="cuda")[None, :] <= i[:, None]
            for head in range(case["hq"]):
                x = s["q"][a:b, head].double() @ s["k"][ka:kb, head // g].double().T * scale
                p = torch.softmax(torch.where(seen, x, -math.inf), dim=-1)
                out[a:b, head] = p @ s["v"][ka:kb, head // g].double()
        return out
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    flat_k, flat_v = (s[n].transpose(0, 1).reshape(case["h"], -1, case["d"]) for n in ("k_pages", "v_pages"))
    t = torch.arange(case["page"], device="cuda")

    def tokens(table, n):
        return (table.long()[:, None] * case["page"] + t).reshape(-1)[:n]

    pre = tokens(s["prefix_table"], case["prefix"])
    for b, n in enumerate(s["lens"].tolist()):
        at = torch.cat([pre, tokens(s["tables"][b], n)])
        k, v = flat_k[:, at].double(), flat_v[:, at].double()
        q = s["q"][b].double().view(case["h"], g, -1)
        out[b] = torch.bmm(torch.softmax(torch.bmm(q, k.transpose(1, 2)) * scale, -1), v).view(case["hq"], -1)
    return out


def _moved(s, name):
    c, pool = s["case"], s[name].double()
    if c["op"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pool[:, b] = pool[:, a]
        return pool
    for i, m in enumerate(s["kept_count"].tolist()):
        rows = pool[:, s["tables"][i].long()].transpose(1, 2).flatten(2, 3)  # [layers, heads, tokens, d]
        rows = rows[:, :, s["kept_idx"][i, :m].long()]
        for p, page in enumerate(s["dst_tables"][i].tolist()):
            part = rows[:, :, p * c["page"]:(p + 1) * c["page"]]
            pool[:, page, :, :part.shape[2]] = part
    return pool


# ------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    eb, h, d, op = _EB[case["dt"]], case["h"], case["d"], case["op"]
    if op == "rope":
        n, hq = case["n"], case["hq"]
        # q, k, v read once and written once; positions, slots and the rotation rows read once
        return {"bytes": 2 * n * (hq + 2 * h) * d * eb + n * 8 + n * d * 4, "flops": n * (hq + h) * d * (7 if case["norm"] else 3)}
    if op == "prompt":
        lens, past = _cut(case["n"], case["seqs"], case["cut"]), _past(case)
        pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(lens, past))
        return {"bytes": (2 * case["n"] * case["hq"] + 2 * (case["n"] + sum(past)) * h) * d * eb,
                "flops": 4 * pairs * case["hq"] * d}
    if op == "decode":
        lens = _own_lens(case)
        return {"bytes": (2 * (case["prefix"] + sum(lens)) * h + 2 * case["b"] * case["hq"]) * d * eb,
                "flops": 4 * (case["b"] * case["prefix"] + sum(lens)) * case["hq"] * d}
    if op == "copy":
        return {"bytes": 4 * case["layers"] * case["pages"] * h * case["page"] * d * eb, "flops": 0}
    return {"bytes": 4 * case["layers"] * sum(_kept_counts(case)) * h * d * eb + 4 * sum(_kept_counts(case)), "flops": 0}
