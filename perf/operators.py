"""What is measured of the paged K/V cache operators: appending rotated keys and values,
attention of new tokens over the cached pages, copying pages, and committing the accepted
tokens of a draft.

`own` False computes the plain form (elementary torch operations in fp32, rounded once);
True calls kernrelay_b200's operators on the same inputs."""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# query heads, KV heads, head_dim of the repository's configurations and tests
_HEADS = [(14, 2, 64), (28, 4, 128), (32, 8, 128), (8, 2, 128), (4, 2, 64), (2, 1, 128),
          (4, 4, 128), (4, 1, 128)]


def listed():
    return [
        # 8 sequences decode one token each: the append before every attention of a small batch
        dict(name="append_decode", op="append", n=8, hq=28, hkv=4, d=128, page=16, norm=False,
             dtype="bf16", layout="hnd"),
        # 203 drafted tokens of a batch, cache with the head axis inside the slot axis
        dict(name="append_draft", op="append", n=203, hq=14, hkv=2, d=64, page=32, norm=False,
             dtype="bf16", layout="nhd"),
        # the prompts of a full prefill step, with per-head norms
        dict(name="append_prompt", op="append", n=8192, hq=32, hkv=8, d=128, page=64, norm=True,
             dtype="fp16", layout="hnd"),
        # one user decoding behind a short prompt: pure latency
        dict(name="decode_one", op="attention", b=1, t=1, lo=317, hi=317, hq=14, hkv=2, d=64,
             page=16, tree=False, dtype="bf16", layout="hnd"),
        # a serving batch decoding, ragged lengths
        dict(name="decode_batch", op="attention", b=64, t=1, lo=1999, hi=8050, hq=28, hkv=4, d=128,
             page=16, tree=False, dtype="bf16", layout="hnd"),
        # two users with very long contexts: few rows, work split over the keys
        dict(name="decode_long", op="attention", b=2, t=1, lo=98303, hi=131071, hq=28, hkv=4, d=128,
             page=64, tree=False, dtype="bf16", layout="hnd"),
        # verification of 8-token drafts, batch 16
        dict(name="tree_small", op="attention", b=16, t=8, lo=1001, hi=4040, hq=32, hkv=8, d=128,
             page=32, tree=True, dtype="fp16", layout="nhd"),
        # verification of wide 64-token trees, batch 8
        dict(name="tree_wide", op="attention", b=8, t=64, lo=2011, hi=7920, hq=28, hkv=4, d=128,
             page=16, tree=True, dtype="bf16", layout="hnd"),
        # two prompt chunks of about a thousand tokens over cached prefixes
        dict(name="chunk", op="attention", b=2, t=1024, lo=999, hi=8190, hq=28, hkv=4, d=128,
             page=64, tree=False, dtype="bf16", layout="hnd"),
        # 256 pages of every layer: a batch of forks whose last pages are duplicated, and pages
        # moved together after sequences ended
        dict(name="copy_many", op="copy", pairs=256, pages=640, layers=28, hkv=4, d=128, page=16,
             dtype="bf16", layout="hnd"),
        # one accepted path of a single user's draft
        dict(name="commit_one", op="commit", b=1, t=8, keep=4, layers=24, hkv=2, d=64, page=16,
             dtype="bf16", layout="hnd", ctx=411),
        # the accepted paths of a batch of wide drafts
        dict(name="commit_batch", op="commit", b=64, t=64, keep=9, layers=28, hkv=4, d=128, page=16,
             dtype="bf16", layout="hnd", ctx=190),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "copy", "commit"])
    hq, hkv, d = rng.choice(_HEADS)
    c = dict(op=op, hkv=hkv, d=d, page=rng.choice([8, 16, 32, 64, 128]),
             dtype=rng.choice(["bf16", "fp16"]), layout=rng.choice(["hnd", "nhd"]))
    if op == "append":
        n = _log(rng, 1, 8192)
        c.update(n=max(1, n * 4096 // max(4096, (hq + 2 * hkv) * d)), hq=hq,
                 norm=rng.random() < 0.5)
    elif op == "attention":
        t = rng.choice([1, 1, rng.randint(2, 16), rng.randint(17, 128), _log(rng, 129, 1024)])
        hi = _log(rng, 16, 32768)
        # at most the listed chunk's products and the listed batch's cached tokens
        pairs = 2 * 1024 * 8192 * 28 * 128 // (t * hq * d)
        hi = max(1, min(hi, pairs - t))
        tokens = min(300000 * 512 // (hkv * d), pairs) // (hi + t)
        b = _log(rng, 1, max(1, min(64, tokens)))
        c.update(b=b, t=t, lo=rng.randint(0, hi), hi=hi, hq=hq, tree=1 < t <= 128)
    elif op == "copy":
        layers = rng.randint(1, 28)
        most = 256 * 28 * 16 * 512 // (layers * c["page"] * hkv * d)
        pairs = _log(rng, 1, max(1, min(256, most)))
        c.update(pairs=pairs, pages=2 * pairs + rng.randint(0, 31), layers=layers)
    else:
        t = rng.randint(2, 64)
        layers, b = rng.randint(1, 28), _log(rng, 1, 64)
        c.update(b=b, t=t, keep=rng.randint(1, min(t, 9)), layers=layers, ctx=rng.randint(0, 200))
    return c


def _spans(c):
    """Per sequence: cached tokens before the step, new tokens.  Fixed by the case."""
    b, lo, hi = c["b"], c["lo"], c["hi"]
    ctx = [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]
    new = [max(1, c["t"] - (i % 3) * (c["t"] // 16)) for i in range(b)]
    return ctx, new


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _cache(g, c, layers, pages):
    """K and V [layers, pages, heads, page, d]; "nhd" stores the slot axis outside the heads'."""
    hkv, page, d, dt = c["hkv"], c["page"], c["d"], _TYPES[c["dtype"]]
    shape = (layers, pages, hkv, page, d) if c["layout"] == "hnd" else (layers, pages, page, hkv, d)
    kv = [torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g) for _ in range(2)]
    return [x if c["layout"] == "hnd" else x.transpose(2, 3) for x in kv]


def _table(g, lens, page, pages):
    """Random distinct pages for sequences of these lengths: int32 [b, most], unused entries 0."""
    most = max(1, max(-(-n // page) for n in lens))
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), most), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(lens):
        k = -(-n // page)
        table[i, :k] = perm[at:at + k]
        at += k
    return table


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tree_bits(seed, new, words):
    """Masks of random trees: bit j of row i says that token i sees token j of its sequence (its
    ancestors and itself)."""
    r = random.Random(seed)
    rows = []
    for t in new:
        sees = []
        for i in range(t):
            sees.append((1 << i) | (sees[r.randint(max(0, i - 8), i - 1)] if i else 0))
        rows += sees
    words_of = [[(x >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for x in rows]
    return torch.tensor(words_of, dtype=torch.int64).to(torch.int32).cuda()


def _rope_tables(max_pos, d):
    inv = 1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    a = torch.outer(torch.arange(max_pos, dtype=torch.float64, device="cuda"), inv)
    a = torch.cat([a, a], -1)
    return a.cos().to(torch.bfloat16), a.sin().to(torch.bfloat16)


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = _TYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "append":
        n, hq, hkv, d = c["n"], c["hq"], c["hkv"], c["d"]
        pages = -(-n // c["page"]) + 7
        s["k"], s["v"] = _cache(g, c, 1, pages)
        s["qkv"] = _normal(g, (n, (hq + 2 * hkv) * d), dt, 1.5)
        s["cos"], s["sin"] = _rope_tables(4096, d)
        s["positions"] = torch.randint(0, 4096, (n,), generator=g, device="cuda")
        s["slots"] = torch.randperm(pages * c["page"], generator=g, device="cuda")[:n].clone()
        w = 1 + 0.1 * torch.randn((2, d), generator=g, device="cuda")
        s["q_norm"], s["k_norm"] = w.to(torch.bfloat16) if c["norm"] else (None, None)
    elif c["op"] == "attention":
        ctx, new = _spans(c)
        lens = [a + b for a, b in zip(ctx, new)]
        pages = sum(-(-n // c["page"]) for n in lens) + 3
        s["k"], s["v"] = _cache(g, c, 1, pages)
        s["table"] = _table(g, lens, c["page"], pages)
        s["kv_lens"] = _ints(lens)
        s["q_starts"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        s["max_q"] = max(new)
        # twice unit normal: scores of standard deviation 2, as peaked as trained heads are
        s["q"] = _normal(g, (sum(new), c["hq"] * c["d"]), dt, 2.0)
        s["scale"] = 1.0 / math.sqrt(c["d"])
        s["mask"] = _tree_bits(seed, new, -(-max(new) // 32)) if c["tree"] else None
    elif c["op"] == "copy":
        s["k"], s["v"] = _cache(g, c, c["layers"], c["pages"])
        order = torch.randperm(c["pages"], generator=torch.Generator().manual_seed(seed)).tolist()
        s["src"], s["dst"] = order[:c["pairs"]], order[c["pairs"]:2 * c["pairs"]]
    else:
        lens = [c["ctx"] + i + c["t"] for i in range(c["b"])]
        pages = sum(-(-n // c["page"]) for n in lens) + 3
        s["k"], s["v"] = _cache(g, c, c["layers"], pages)
        s["table"] = _table(g, lens, c["page"], pages)
        s["bases"] = _ints([c["ctx"] + i for i in range(c["b"])])
        rest = torch.rand((c["b"], c["t"] - 1), generator=g, device="cuda").argsort(-1) + 1
        path = torch.cat([torch.zeros_like(rest[:, :1]), rest], 1)[:, :c["keep"]]
        s["accepted"] = path.sort(-1).values.to(torch.int32).contiguous()
        s["counts"] = _ints([max(1, c["keep"] - i % 2) for i in range(c["b"])])
    return s


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return x * cos[:, None, :] + torch.cat([-b, a], -1) * sin[:, None, :]


def _plain_append(s):
    c = s["case"]
    n, hq, hkv, d, page = c["n"], c["hq"], c["hkv"], c["d"], c["page"]
    x = s["qkv"].view(n, hq + 2 * hkv, d)
    q, k = x[:, :hq].float(), x[:, hq:hq + hkv].float()
    if s["q_norm"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + 1e-6) * s["q_norm"].float()
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + 1e-6) * s["k_norm"].float()
    cos, sin = s["cos"][s["positions"]].float(), s["sin"][s["positions"]].float()
    p, o = s["slots"] // page, s["slots"] % page
    s["k"][0][p, :, o] = _rotate(k, cos, sin).to(x.dtype)
    s["v"][0][p, :, o] = x[:, hq + hkv:]
    return _rotate(q, cos, sin).to(x.dtype).view(n, hq * d)


def _plain_attention(s):
    c = s["case"]
    b, hq, hkv, d = c["b"], c["hq"], c["hkv"], c["d"]
    g, t, dev = hq // hkv, s["max_q"], s["q"].device
    n = s["q"].shape[0]
    at = torch.arange(n, dtype=torch.int32, device=dev)
    seq = torch.bucketize(at, s["q_starts"][1:], right=True)
    row = at - s["q_starts"][seq]
    q = torch.zeros((b, t, hkv, g, d), device=dev)
    q[seq, row] = s["q"].view(n, hkv, g, d).float()
    k, v = (x[0][s["table"]].transpose(1, 2).reshape(b, hkv, -1, d).float()
            for x in (s["k"], s["v"]))
    keys = torch.arange(k.shape[2], device=dev)
    j = keys[None, :] - (s["kv_lens"] - s["q_starts"].diff())[:, None]  # drafted index of a key
    if s["mask"] is None:
        sees = j[:, None, :] <= torch.arange(t, device=dev)[None, :, None]
    else:
        bits = torch.zeros((b, t, s["mask"].shape[1]), dtype=torch.int32, device=dev)
        bits[seq, row] = s["mask"]
        jj = j.clamp(0, 32 * bits.shape[2] - 1)
        word = bits.gather(2, (jj // 32)[:, None, :].expand(b, t, -1))
        sees = (j < 0)[:, None, :] | ((word >> (jj % 32)[:, None, :]) & 1).bool()
    live = keys[None, :] < s["kv_lens"][:, None]
    sees = sees & live[:, None, :]
    v = torch.where(live[:, None, :, None], v, 0.0)
    x = q.permute(0, 2, 3, 1, 4).reshape(b, hkv, g * t, d) @ k.transpose(2, 3)
    x = x.view(b, hkv, g, t, -1).mul_(s["scale"])
    x = x.masked_fill_(~sees[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = e.sum(-1, keepdim=True)
    o = (e.view(b, hkv, g * t, -1) @ v).view(b, hkv, g, t, d)
    o = o / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, t, hq * d)
    return o[seq, row].to(s["q"].dtype)


def _plain_copy(s):
    src, dst = (torch.tensor(x, device="cuda") for x in (s["src"], s["dst"]))
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]


def _plain_commit(s):
    page = s["case"]["page"]
    a = s["accepted"].shape[1]
    i = torch.arange(a, device="cuda")[None, :]
    kept = i < s["counts"][:, None]
    to = s["bases"][:, None] + i
    # a place that is not kept copies its own row
    at = s["bases"][:, None] + torch.where(kept, s["accepted"], i)
    pt, pa = (s["table"].gather(1, x // page) for x in (to, at))
    ot, oa = to % page, at % page
    s["k"][:, pt, :, ot] = s["k"][:, pa, :, oa]
    s["v"][:, pt, :, ot] = s["v"][:, pa, :, oa]


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from kernrelay_b200 import _lib as krb
        if "cache" not in s:  # the handle that a program makes once for its cache
            s["cache"] = krb.KVCache(s["k"], s["v"])
        if op == "append":
            q = krb.qk_norm_rope_paged(s["qkv"], s["cache"], s["positions"], s["slots"],
                                       s["case"]["hq"], s["cos"], s["sin"], s["q_norm"],
                                       s["k_norm"], eps=1e-6)
        elif op == "attention":
            return krb.attention_paged(s["q"], s["cache"], s["table"], s["kv_lens"],
                                       s["q_starts"], s["max_q"], s["scale"], mask=s["mask"])
        elif op == "copy":
            krb.kv_copy_pages(s["cache"], s["src"], s["dst"])
        else:
            krb.kv_commit(s["cache"], s["table"], s["bases"], s["accepted"], s["counts"])
    elif op == "append":
        q = _plain_append(s)
    elif op == "attention":
        return _plain_attention(s)
    elif op == "copy":
        _plain_copy(s)
    else:
        _plain_commit(s)
    if op == "append":
        return {"q": q, "k": s["k"], "v": s["v"].view(torch.int16)}
    # moved rows are the same bits
    return {"k": s["k"].view(torch.int16), "v": s["v"].view(torch.int16)}


def work(case):
    c = case
    if c["op"] == "append":
        row = (c["hq"] + 2 * c["hkv"]) * c["d"] * 2
        tables = min(c["n"], 4096) * c["d"] * 2 * 2
        rotated = c["n"] * (c["hq"] + c["hkv"]) * c["d"]
        return {"bytes": 2 * c["n"] * row + tables + 16 * c["n"], "flops": 8 * rotated}
    if c["op"] == "attention":
        ctx, new = _spans(c)
        cached = sum(a + b for a, b in zip(ctx, new)) * c["hkv"] * c["d"] * 2 * 2
        pairs = sum(a * t + t * (t + 1) // 2 for a, t in zip(ctx, new))
        return {"bytes": cached + 2 * sum(new) * c["hq"] * c["d"] * 2,
                "flops": 4 * pairs * c["hq"] * c["d"]}
    if c["op"] == "copy":
        page = c["layers"] * c["hkv"] * c["page"] * c["d"] * 2 * 2
        return {"bytes": 2 * c["pairs"] * page, "flops": 0}
    rows = sum(max(1, c["keep"] - i % 2) - 1 for i in range(c["b"]))
    row = c["layers"] * c["hkv"] * c["d"] * 2 * 2
    return {"bytes": 2 * rows * row + 4 * c["b"] * (c["keep"] + 2), "flops": 0}


def exact(case, seed):
    """The definition in 64 bits, sequence by sequence and token by token."""
    c, s = case, prepare(case, seed)
    if c["op"] == "append":
        hq, hkv, d = c["hq"], c["hkv"], c["d"]
        x = s["qkv"].double().view(c["n"], -1, d)
        half = d // 2
        angle_cos, angle_sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
        out = []
        for heads, w in ((x[:, :hq], s["q_norm"]), (x[:, hq:hq + hkv], s["k_norm"])):
            if w is not None:
                heads = heads / (heads.pow(2).sum(-1, keepdim=True) / d + 1e-6).sqrt() * w.double()
            y = torch.empty_like(heads)
            for lo, hi, sign, other in ((0, half, -1, half), (half, d, 1, 0)):
                y[..., lo:hi] = (heads[..., lo:hi] * angle_cos[:, None, lo:hi]
                                 + sign * heads[..., other:other + half]
                                 * angle_sin[:, None, lo:hi])
            out.append(y)
        k = s["k"].double()
        flat = k[0].transpose(1, 2).reshape(-1, hkv, d)  # by slot
        flat[s["slots"]] = out[1]
        k = flat.view(1, -1, c["page"], hkv, d).transpose(2, 3)
        return {"q": out[0].reshape(c["n"], -1), "k": k, "v": None}
    if c["op"] == "attention":
        ctx, new = _spans(c)
        hq, hkv, d = c["hq"], c["hkv"], c["d"]
        out, at = [], 0
        for i, (a, t) in enumerate(zip(ctx, new)):
            slots = torch.arange(a + t, device="cuda")
            pages = s["table"][i].long()[slots // c["page"]]
            sees = torch.ones((t, a + t), dtype=torch.bool, device="cuda")
            if s["mask"] is None:
                sees[:, a:] = torch.ones((t, t), device="cuda").tril().bool()
            else:
                bit = torch.arange(t, device="cuda")
                words = s["mask"][at:at + t].long()
                sees[:, a:] = ((words[:, bit // 32] >> (bit % 32)) & 1).bool()
            rows = s["q"][at:at + t].double().view(t, hkv, hq // hkv, d)
            heads = []
            for h in range(hkv):
                key = s["k"][0, :, h][pages, slots % c["page"]].double()
                value = s["v"][0, :, h][pages, slots % c["page"]].double()
                x = torch.einsum("tgd,sd->tgs", rows[:, h], key) * s["scale"]
                x = x.masked_fill(~sees[:, None, :], -math.inf)
                heads.append(torch.softmax(x, -1).nan_to_num(0.0) @ value)
            out.append(torch.stack(heads, 1).reshape(t, hq * d))
            at += t
        return torch.cat(out)
    return None  # rows and pages are moved, nothing is computed
