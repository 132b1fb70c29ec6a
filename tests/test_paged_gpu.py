"""The paged K/V cache operators against their definitions in 64 bits.

Tolerances (u = half a step of the 2-byte type, eps / 2):
* append: one rounding, u |y|, and the fp32 arithmetic before it, at most 16 operations of 2^-24
  relative to |x_lo cos| + |x_hi sin| (the norm's factor included: its terms are squares, so the
  sum's relative error is below D * 2^-24 and halves under the root).
* attention, with A = sum_j p_j |v_j|: the output's rounding u |o|, the probabilities' u A (the row
  sum takes them unrounded), and the scores' fp32 error: D + 4 roundings of 2^-24 of
  S = scale * sum_d |q_d k_d| change a probability by twice that, relative; the sums over n keys
  n 2^-24 (of fp32 products, whose order is free), exp2 2^-21.  fp16 probabilities below 2^-14
  have an absolute error, 2^-25, where the row's largest is at least 1: 2^-25 sum_j |v_j|; so does
  an fp16 output below 2^-14 (its neighbours are 2^-24 apart): 2^-25.
* copies and commits: the same bits."""
import math
import random

import pytest

pytestmark = pytest.mark.gpu


def _dt(name):
    import torch
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[name]


def _gen(seed):
    import torch
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache_tensors(layers, pages, heads, page, D, dtype, layout, fill=None, g=None):
    """K and V views [layers, pages, heads, page, D] of several memory orders."""
    import torch
    kw = dict(dtype=dtype, device="cuda")
    if layout == "hnd":
        kv = [torch.empty(layers, pages, heads, page, D, **kw) for _ in range(2)]
    elif layout == "nhd":
        kv = [torch.empty(layers, pages, page, heads, D, **kw).transpose(2, 3) for _ in range(2)]
    elif layout == "paired":  # K and V of a page side by side, pages outermost
        both = torch.empty(pages, layers, 2, heads, page, D, **kw)
        kv = [both[:, :, i].transpose(0, 1) for i in range(2)]
    else:  # "padded": every axis with room between its rows
        kv = [torch.empty(layers, pages, heads + 1, page + 8, D + 8, **kw)[:, :, :heads, :page, :D]
              for _ in range(2)]
    for x in kv:
        if fill is None:
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        else:
            x.fill_(fill)
    return kv


def _rope_tables(n, D):
    import torch
    inv = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    a = torch.outer(torch.arange(n, dtype=torch.float64, device="cuda"), inv)
    a = torch.cat([a, a], -1)
    return a.cos().to(torch.bfloat16), a.sin().to(torch.bfloat16)


# ---------------------------------------------------------------- append
def _append_ref(x, w, cos, sin):
    """x [n, h, D] double -> (y, |x_lo cos| + |x_hi sin|)"""
    import torch
    D = x.shape[-1]
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    a, b = x[..., :D // 2], x[..., D // 2:]
    c, s = cos.double()[:, None], sin.double()[:, None]
    rot = torch.cat([-b, a], -1)
    return x * c + rot * s, (x * c).abs() + (rot * s).abs()


@pytest.mark.parametrize("n,HQ,HKV,D,page,norm,dtype,layout", [
    (1, 14, 2, 64, 16, False, "bf16", "hnd"),
    (1, 2, 1, 128, 8, True, "fp16", "nhd"),
    (7, 28, 4, 128, 16, False, "bf16", "paired"),
    (203, 32, 8, 128, 64, True, "bf16", "nhd"),
    (130, 4, 4, 64, 32, True, "fp16", "padded"),
    (1025, 14, 2, 64, 128, True, "bf16", "hnd"),
    (64, 4, 1, 128, 1024, False, "fp16", "hnd"),
    (6001, 32, 8, 128, 64, True, "bf16", "hnd"),  # 74 MB: stored past L2
])
@pytest.mark.parametrize("in_place", [False, True])
def test_append(cuda, krlib, n, HQ, HKV, D, page, norm, dtype, layout, in_place):
    import torch
    dt, g = _dt(dtype), _gen(n + D)
    u = torch.finfo(dt).eps / 2
    pages, layers, layer = -(-n // page) + 2, 2, 1
    k, v = _cache_tensors(layers, pages, HKV, page, D, dt, layout, g=g)
    k0, v0 = k.clone(), v.clone()
    wide = torch.randn(n, (HQ + 2 * HKV) * D + 24, generator=g, device="cuda").to(dt)
    qkv = wide[:, 8:-16]
    before = qkv.clone()
    cos, sin = _rope_tables(500, D)
    pos = torch.randint(0, 500, (n,), generator=g, device="cuda")
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:n].contiguous()
    if n > 1:
        slots[n // 2] = -1
    qn, kn = [(1 + 0.1 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16)
              if norm else None for _ in range(2)]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = krlib.KVCache(k, v)
    out = qkv[:, :HQ * D] if in_place else None
    q = krlib.qk_norm_rope_paged(qkv, cache, pos, slots, HQ, cos, sin, qn, kn, layer=layer, out=out,
                                 status=status)
    torch.cuda.synchronize()
    assert status.item() == 0
    x = before.double().view(n, HQ + 2 * HKV, D)
    for got, heads, w in ((q.view(n, HQ, D), x[:, :HQ], qn), (None, x[:, HQ:HQ + HKV], kn)):
        ref, mag = _append_ref(heads, w, cos[pos], sin[pos])
        bound = u * ref.abs() + (16 + D / 2) * 2.0 ** -24 * mag * (1 + u) + 2.0 ** -25 * (dtype == "fp16")
        if got is None:
            keep = slots >= 0
            got = k[layer].transpose(1, 2).reshape(-1, HKV, D)[slots[keep]]
            ref, bound = ref[keep], bound[keep]
        assert ((got.double() - ref).abs() <= bound).all()
    keep = slots >= 0
    want = v0.clone()
    flat = want[layer].transpose(1, 2).reshape(-1, HKV, D).clone()
    flat[slots[keep]] = before.view(n, -1, D)[keep, HQ + HKV:]
    want[layer] = flat.view(pages, page, HKV, D).transpose(1, 2)
    assert torch.equal(v, want)
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots[keep]] = False
    assert torch.equal(k[0], k0[0])  # the other layer, and slots that no row names
    after, first = (x[layer].transpose(1, 2).reshape(-1, HKV, D)[rest] for x in (k, k0))
    assert torch.equal(after, first)
    if not in_place:
        assert torch.equal(qkv, before)


def test_append_bad_indices(cuda, krlib):
    """A position or slot outside its range is reported, and its row is not written."""
    import torch
    g = _gen(3)
    HQ, HKV, D, page, n = 4, 2, 64, 16, 9
    k, v = _cache_tensors(1, 3, HKV, page, D, torch.bfloat16, "hnd", fill=7.0)
    cos, sin = _rope_tables(32, D)
    qkv = torch.randn(n, (HQ + 2 * HKV) * D, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.tensor([0, 31, 32, -1, 5, 6, 7, 2 ** 40, 8], device="cuda")
    slots = torch.tensor([0, 1, 2, 3, 48, -2, -1, 4, 2 ** 40], device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = krlib.qk_norm_rope_paged(qkv, krlib.KVCache(k, v), pos, slots, HQ, cos, sin, status=status)
    torch.cuda.synchronize()
    assert status.item() == 1 << 8
    for i in (2, 3, 7):
        assert q[i].abs().max().item() == 0
    for i in (0, 1, 4, 5, 6, 8):
        assert q[i].abs().max().item() > 0
    for t in (k, v):
        rows = t[0].transpose(1, 2).reshape(-1, HKV * D)
        written = (rows != 7.0).any(-1).nonzero().flatten().tolist()
        assert written == [0, 1]


def test_append_no_rows(cuda, krlib):
    import torch
    k, v = _cache_tensors(1, 2, 2, 16, 64, torch.bfloat16, "hnd", fill=1.0)
    cos, sin = _rope_tables(8, 64)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    q = krlib.qk_norm_rope_paged(torch.empty(0, 8 * 64, dtype=torch.bfloat16, device="cuda"),
                                 krlib.KVCache(k, v), none, none, 4, cos, sin)
    assert q.shape == (0, 4 * 64)


# ---------------------------------------------------------------- attention
def _tree(rng, t, words, empty=()):
    """[t, words] int32 mask rows of a random tree, and the boolean [t, t] they stand for."""
    import torch
    sees = []
    for i in range(t):
        x = (1 << i) | (sees[rng.randint(max(0, i - 6), i - 1)] if i else 0)
        sees.append(x)
    sees = [0 if i in empty else x for i, x in enumerate(sees)]
    seen = torch.tensor([[(x >> j) & 1 for j in range(t)] for x in sees], dtype=torch.bool)
    # bits behind the last token are the caller's: set them
    sees = [x | (((1 << (32 * words - t)) - 1) << t) for x in sees]
    rows = [[(x >> (32 * w)) & 0xFFFFFFFF for w in range(words)] for x in sees]
    return torch.tensor(rows, dtype=torch.int64).to(torch.int32).view(t, words), seen.view(t, t)


class Batch:
    """Random sequences over a paged cache whose unused slots hold NaN."""

    def __init__(self, seqs, HQ, HKV, D, page, dtype="bf16", layout="hnd", masked=False, seed=0,
                 empty=(), layers=1, q_std=2.0, spare_rows=3):
        import torch
        self.g, rng = _gen(seed), random.Random(seed)
        self.seqs, self.HQ, self.HKV, self.D, self.page = seqs, HQ, HKV, D, page
        dt = self.dt = _dt(dtype)
        lens = [c + t for c, t in seqs]
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + 3
        self.layer = layers - 1
        k, v = _cache_tensors(layers, self.pages, HKV, page, D, dt, layout, fill=float("nan"))
        order = list(range(self.pages))
        rng.shuffle(order)
        most = max(need + [1]) + 2
        table = torch.full((len(seqs), most + 3), 10 ** 9, dtype=torch.int32)  # never to be read
        self.K, self.V, at = [], [], 0
        for b, n in enumerate(lens):
            ids = order[at:at + need[b]]
            at += need[b]
            table[b, :need[b]] = torch.tensor(ids, dtype=torch.int32)
            kb, vb = (torch.randn(n, HKV, D, generator=self.g, device="cuda").to(dt) for _ in range(2))
            p = torch.arange(n, device="cuda")
            idx = torch.tensor(ids, device="cuda", dtype=torch.long)[p // page]
            k[self.layer][idx, :, p % page] = kb
            v[self.layer][idx, :, p % page] = vb
            self.K.append(kb)
            self.V.append(vb)
        self.k, self.v = k, v
        self.table = table.cuda()[:, :most]
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        starts = [0]
        for _, t in seqs:
            starts.append(starts[-1] + t)
        self.starts_host = starts
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.N = starts[-1] + spare_rows
        wide = torch.randn(self.N, HQ * D + 16, generator=self.g, device="cuda") * q_std
        self.q = wide.to(dt)[:, 8:-8]
        self.max_q = max([t for _, t in seqs] + [1])
        self.scale = 1 / math.sqrt(D)
        self.mask, self.sees = None, []
        words = -(-self.max_q // 32)
        rows = torch.full((self.N, words + 1), -1, dtype=torch.int32)
        for b, (c, t) in enumerate(seqs):
            if masked:
                m, s = _tree(rng, t, words, empty)
                rows[starts[b]:starts[b + 1], :words] = m
            else:
                s = torch.ones(t, t, dtype=torch.bool).tril()
            self.sees.append(s.cuda())
        if masked:
            self.mask = rows.cuda()[:, :words]

    def run(self, krlib, out=None, **kw):
        import torch
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")
        if out is None:
            out = torch.full((self.N, self.HQ * self.D), 5.0, dtype=self.dt, device="cuda")
        return krlib.attention_paged(self.q, krlib.KVCache(self.k, self.v), self.table, self.lens,
                                     self.starts, kw.pop("max_q", self.max_q), self.scale,
                                     mask=self.mask, layer=self.layer, out=out, status=self.status, **kw)

    def check(self, out, only=None):
        import torch
        u = torch.finfo(self.dt).eps / 2
        G, D = self.HQ // self.HKV, self.D
        for b, (c, t) in enumerate(self.seqs):
            if t == 0 or (only is not None and b not in only):
                continue
            rows = slice(self.starts_host[b], self.starts_host[b + 1])
            q = self.q[rows].double().view(t, self.HKV, G, D)
            K, V = self.K[b].double(), self.V[b].double()
            n = c + t
            sees = torch.cat([torch.ones(t, c, dtype=torch.bool, device="cuda"), self.sees[b]], 1)
            s = torch.einsum("thgd,nhd->thgn", q, K) * self.scale
            p = torch.softmax(s.masked_fill(~sees[:, None, None], -math.inf), -1).nan_to_num(0.0)
            ref = torch.einsum("thgn,nhd->thgd", p, V)
            A = torch.einsum("thgn,nhd->thgd", p, V.abs())
            S = (torch.einsum("thgd,nhd->thgn", q.abs(), K.abs()) * self.scale).amax(-1, keepdim=True)
            rel = 2 * (D + 4) * 2.0 ** -24 * S + n * 2.0 ** -24 + 2.0 ** -20
            bound = u * ref.abs() + (u + rel) * A * (1 + 2 * u)
            if self.dt == torch.float16:
                bound = bound + 2.0 ** -25 * (1 + V.abs().sum(0)[None, :, None])
            got = out[rows].double().view(t, self.HKV, G, D)
            bad = ~((got - ref).abs() <= bound)
            assert not bad.any(), (b, bad.sum().item(), (got - ref).abs().max().item(),
                                   bad.nonzero()[:4].tolist())
            none = ~sees.any(1)
            assert (got[none] == 0).all()


HEADS = [(14, 2, 64), (28, 4, 128), (32, 8, 128), (4, 4, 128), (2, 1, 128), (4, 1, 64)]


@pytest.mark.parametrize("HQ,HKV,D", HEADS)
@pytest.mark.parametrize("page,dtype,layout", [(16, "bf16", "hnd"), (8, "fp16", "nhd"),
                                               (64, "bf16", "paired"), (256, "fp16", "padded")])
def test_decode(cuda, krlib, HQ, HKV, D, page, dtype, layout):
    import torch
    b = Batch([(0, 1), (1, 1), (62, 1), (63, 1), (64, 1), (65, 1), (700, 1), (0, 0), (1500, 1), (15, 1)],
              HQ, HKV, D, page, dtype, layout, seed=page + D, layers=2)
    out = b.run(krlib)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    b.check(out)
    assert (out[b.starts_host[-1]:] == 5.0).all()


@pytest.mark.parametrize("ctx", [0, 1, 40, 4000, 70001])
@pytest.mark.parametrize("HQ,HKV,D", [(28, 4, 128), (14, 2, 64)])
def test_decode_one_sequence(cuda, krlib, ctx, HQ, HKV, D):
    """One sequence over all SMs: every unit is split, down to one block per CTA."""
    import torch
    b = Batch([(ctx, 1)], HQ, HKV, D, 16, seed=ctx + 1)
    out = b.run(krlib)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    b.check(out)


@pytest.mark.parametrize("T", [2, 3, 4, 5, 8, 9, 16, 17, 31, 32, 33, 64, 65, 100])
@pytest.mark.parametrize("HQ,HKV,D,dtype", [(28, 4, 128, "bf16"), (14, 2, 64, "fp16"),
                                            (4, 4, 128, "fp16"), (32, 8, 128, "bf16")])
def test_tree(cuda, krlib, T, HQ, HKV, D, dtype):
    """Trees of drafted tokens at every offset of the draft inside a block and a mask word."""
    import torch
    seqs = [(0, T), (5, T), (64 - T % 64, T), (127, T), (77, 0), (333, max(1, T - 1)), (1, 1), (990, T)]
    b = Batch(seqs, HQ, HKV, D, 16, dtype, "nhd", masked=True, seed=T, empty={0, T // 2})
    out = b.run(krlib)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    b.check(out)
    assert (out[b.starts_host[-1]:] == 5.0).all()


@pytest.mark.parametrize("T,ctxs", [(2, (0, 61)), (7, (3, 120)), (40, (0, 24)), (130, (0, 1, 500)),
                                    (257, (77,)), (700, (0, 129))])
@pytest.mark.parametrize("HQ,HKV,D,page,dtype", [(28, 4, 128, 16, "bf16"), (14, 2, 64, 32, "fp16"),
                                                 (4, 1, 128, 64, "fp16")])
def test_chunk(cuda, krlib, T, ctxs, HQ, HKV, D, page, dtype):
    """Causal chunks of a prompt over a cached prefix, mixed with decoding sequences."""
    import torch
    b = Batch([(c, T - i) for i, c in enumerate(ctxs)] + [(450, 1), (0, 2)], HQ, HKV, D, page,
              dtype, seed=T)
    out = b.run(krlib)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    b.check(out)


@pytest.mark.parametrize("HQ,HKV,D,T", [(64, 1, 64, 1), (64, 1, 128, 3), (40, 2, 128, 1), (9, 3, 64, 6),
                                        (17, 1, 128, 2), (33, 1, 64, 1)])
def test_groups(cuda, krlib, HQ, HKV, D, T):
    """Group sizes that do not divide a tile, up to the largest."""
    import torch
    b = Batch([(200, T), (63, T), (0, T)], HQ, HKV, D, 16, seed=HQ)
    out = b.run(krlib)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    b.check(out)


@pytest.mark.parametrize("T", [1, 3, 30, 200])
@pytest.mark.parametrize("HQ,HKV,D", [(28, 4, 128), (14, 2, 64)])
def test_output_rows_16_byte_aligned(cuda, krlib, T, HQ, HKV, D):
    """Output rows at every multiple of 16 bytes, whole units and split ones; what lies between
    them stays."""
    import torch
    b = Batch([(300, T), (0, T), (1000, 1)], HQ, HKV, D, 16, "fp16", seed=T)
    for lead, tail in ((8, 0), (8, 8), (24, 16)):
        wide = torch.full((b.N, lead + HQ * D + tail + 8), 5.0, dtype=b.dt, device="cuda")
        out = wide[:, lead:lead + HQ * D]
        b.run(krlib, out=out)
        torch.cuda.synchronize()
        assert b.status.item() == 0
        b.check(out)
        assert (wide[:, :lead] == 5.0).all() and (wide[:, lead + HQ * D:] == 5.0).all()


@pytest.mark.parametrize("T,HQ,HKV,D", [(200, 14, 2, 64), (130, 4, 4, 128), (300, 8, 1, 128)])
def test_wide_tree(cuda, krlib, T, HQ, HKV, D):
    """Masks of many words, over several units of a sequence."""
    import torch
    b = Batch([(70, T), (0, T), (500, 3)], HQ, HKV, D, 32, "bf16", masked=True, seed=T, empty={1})
    out = b.run(krlib)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    b.check(out)


def test_many_sequences(cuda, krlib):
    """More sequences than a warp's lanes, and than CTAs; several without new tokens."""
    import torch
    rng = random.Random(5)
    seqs = [(rng.choice([0, 3, 64, 100, 200]), rng.choice([0, 1, 1, 1, 2])) for _ in range(389)]
    b = Batch(seqs, 4, 2, 64, 16, seed=5)
    out = b.run(krlib)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    b.check(out)


def test_peaked_scores(cuda, krlib):
    """Scores far apart: the running maximum moves by more than an fp16 exponent's range."""
    import torch
    for T in (1, 3, 40):
        b = Batch([(700, T), (129, T)], 8, 2, 128, 16, seed=T, q_std=60.0)
        out = b.run(krlib)
        torch.cuda.synchronize()
        b.check(out)


def test_infinite_keys_hidden(cuda, krlib):
    """Keys that a row does not see may hold anything: infinities and NaN do not reach it."""
    import torch
    for T in (4, 40):
        b = Batch([(100, T)], 8, 2, 128, 16, seed=T, masked=True)
        seen = b.sees[0]
        j = T - 1  # the last drafted token: only its own row sees it
        seen[:, j] = False
        seen[j, j] = True
        b.mask[:T] = 0
        for w in range(b.mask.shape[1]):
            bits = seen[:, 32 * w:32 * w + 32].long()
            word = (bits << torch.arange(bits.shape[1], device="cuda")).sum(1)
            b.mask[:T, w] = word.to(torch.int32)
        slot = 100 + j
        page = b.table[0, slot // 16].long()
        for bad in (float("inf"), float("nan")):
            b.k[0][page, :, slot % 16] = bad
            out = b.run(krlib)
            torch.cuda.synchronize()
            q = out[:T - 1].clone()
            assert torch.isfinite(q).all()
            b2 = Batch([(100, T)], 8, 2, 128, 16, seed=T, masked=True)
            b2.mask = b.mask
            ref = b2.run(krlib)
            assert torch.equal(q, ref[:T - 1])


def test_refused_sequences(cuda, krlib):
    """Impossible lengths are reported, their rows left, and the others computed."""
    import torch
    seqs = [(100, 1), (64, 2), (10, 1), (300, 2), (0, 1)]
    b = Batch(seqs, 28, 4, 128, 16, seed=1)
    good = b.run(krlib).clone()
    for lens, bad in (({1: 1}, {1}), ({0: -5}, {0}), ({3: 10 ** 9}, {3}), ({4: 0, 2: 2 ** 31 - 1}, {2, 4})):
        saved = b.lens.clone()
        for i, n in lens.items():
            b.lens[i] = n
        out = b.run(krlib)
        torch.cuda.synchronize()
        assert b.status.item() == 1 << 7
        b.lens.copy_(saved)
        for i in range(len(seqs)):
            rows = slice(b.starts_host[i], b.starts_host[i + 1])
            if i in bad:
                assert (out[rows] == 5.0).all()
        b.check(out, only=set(range(len(seqs))) - bad)
    # more new tokens than max_q, rows outside q, descending starts
    out = b.run(krlib, max_q=1)
    torch.cuda.synchronize()
    assert b.status.item() == 1 << 7
    b.check(out, only={0, 2, 4})
    for i, x in ((5, b.N + 1), (0, -1), (2, 99)):
        saved = b.starts.clone()
        b.starts[i] = x
        out = b.run(krlib)
        torch.cuda.synchronize()
        assert b.status.item() == 1 << 7
        b.starts.copy_(saved)
        assert torch.isfinite(out).all()
    assert torch.equal(b.run(krlib), good)


def test_bad_pages(cuda, krlib):
    """Pages outside the cache are reported and not followed."""
    import torch
    b = Batch([(200, 1), (100, 1)], 28, 4, 128, 16, seed=2)
    for bad in (b.pages, -1, 2 ** 31 - 1):
        b.table[0, 3] = bad
        out = b.run(krlib)
        torch.cuda.synchronize()
        assert b.status.item() == 1 << 8
        b.check(out, only={1})


def test_streams_and_workspace(cuda, krlib):
    """Two calls at once on two streams, each with a workspace of its own, dirty from before."""
    import torch
    bs = [Batch([(3000 + 500 * i, 1 + i)], 28, 4, 128, 16, seed=i) for i in range(2)]
    want = [b.run(krlib).clone() for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for b, s, o in zip(bs, streams, outs):
            with torch.cuda.stream(s):
                o.append(b.run(krlib))
    for b, s, o in zip(bs, streams, outs):
        ws = torch.full((krlib.KVCache(b.k, b.v).attention_workspace(28, b.max_q),), 255,
                        dtype=torch.uint8, device="cuda")
        out = torch.full((b.N, b.HQ * b.D), 5.0, dtype=b.dt, device="cuda")
        torch.cuda.synchronize()
        o.append(b.run(krlib, stream=s, workspace=ws, out=out))
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        for x in o:
            assert torch.equal(x, w)


@pytest.mark.parametrize("T", [1, 40])
def test_order_across_streams(cuda, krlib, T):
    """Each operator starts behind the work before it on its stream, and behind what that stream was
    told to wait for, although its launch is set up early: producers kept busy on either."""
    import torch
    HQ, HKV, D, page, n = 8, 2, 128, 16, 512
    g, dt = _gen(T), torch.bfloat16
    k, v = _cache_tensors(1, 2 * n // page + 2, HKV, page, D, dt, "hnd", fill=0.0)
    cache = krlib.KVCache(k, v)
    cos, sin = _rope_tables(n + 1, D)
    table = torch.arange(k.shape[1], dtype=torch.int32, device="cuda")[None]
    pos = torch.arange(n, device="cuda")
    lens, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([n], [0, T]))
    busy = torch.randn(4096, 4096, generator=g, device="cuda")
    rows = torch.randn(6, n, (HQ + 2 * HKV) * D, generator=g, device="cuda").to(dt)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    src = torch.empty_like(rows[0])
    scale = 1 / math.sqrt(D)

    def step(x, s1, s2):
        with torch.cuda.stream(s1):
            (busy @ busy).sum()
            src.copy_(x)
            q = krlib.qk_norm_rope_paged(src, cache, pos, pos, HQ, cos, sin)
            (busy @ busy).sum()
            krlib.kv_copy_pages(cache, [0, 1], [n // page + 1, n // page])
            done = torch.cuda.Event()
            done.record()
        with torch.cuda.stream(s2):
            s2.wait_event(done)
            out = krlib.attention_paged(q[n - T:], cache, table, lens, starts, T, scale)
            held = torch.stack([k[0, n // page + 1], k[0, n // page]])
            back = torch.cuda.Event()
            back.record()
        q.record_stream(s2)
        s1.wait_event(back)
        return out, held

    torch.cuda.synchronize()
    want = [step(x, a, a) for x in rows]
    torch.cuda.synchronize()
    got = [step(x, a, b) for x in rows]
    torch.cuda.synchronize()
    for i, ((o1, h1), (o2, h2)) in enumerate(zip(want, got)):
        assert torch.equal(o1, o2) and torch.equal(h1, h2), i
    for (o1, _), (o2, _) in zip(want, want[1:]):
        assert not torch.equal(o1, o2)


def test_graph_follows_lengths(cuda, krlib):
    """A captured call reads lengths and pages when it is replayed."""
    import torch
    b = Batch([(900, 1), (333, 1), (64, 1)], 28, 4, 128, 16, seed=9)
    out = torch.full((b.N, b.HQ * b.D), 5.0, dtype=b.dt, device="cuda")
    b.run(krlib, out=out)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = krlib.KVCache(b.k, b.v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        krlib.attention_paged(b.q, cache, b.table, b.lens, b.starts, 1, b.scale, out=out, status=status)
    for cut in (0, 17, 63):
        b.lens.copy_(torch.tensor([901 - cut, 334 - cut, 65 - cut], dtype=torch.int32))
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert status.item() == 0
        short = Batch([(900, 1), (333, 1), (64, 1)], 28, 4, 128, 16, seed=9)
        short.seqs = [(900 - cut, 1), (333 - cut, 1), (64 - cut, 1)]
        short.K = [x[:c + 1] for x, (c, _) in zip(short.K, short.seqs)]
        short.V = [x[:c + 1] for x, (c, _) in zip(short.V, short.seqs)]
        short.check(out)


def test_two_graphs_at_once(cuda, krlib):
    """Two captured calls replayed on two streams at a time: neither uses the other's workspace."""
    import torch
    bs = [Batch([(2000 + 700 * i, 1 + 20 * i), (55, 1)], 28, 4, 128, 16, seed=20 + i) for i in range(2)]
    want = [b.run(krlib).clone() for b in bs]
    outs = [torch.empty_like(w) for w in want]
    caches = [krlib.KVCache(b.k, b.v) for b in bs]
    status = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in bs]
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in bs]
    for b, o, c, st in zip(bs, outs, caches, status):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            krlib.attention_paged(b.q, c, b.table, b.lens, b.starts, b.max_q, b.scale, out=o, status=st)
    for _ in range(10):
        for o in outs:
            o.fill_(5.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for w, o, b in zip(want, outs, bs):
            assert torch.equal(w[:b.starts_host[-1]], o[:b.starts_host[-1]])


def test_same_result_twice(cuda, krlib):
    import torch
    b = Batch([(5000, 1), (77, 1), (2500, 1)], 28, 4, 128, 16, seed=4)
    a = b.run(krlib)
    for _ in range(5):
        assert torch.equal(a, b.run(krlib))


# ---------------------------------------------------------------- page copies
@pytest.mark.parametrize("layout", ["hnd", "nhd", "paired", "padded"])
@pytest.mark.parametrize("layers,heads,page,D,pairs", [(1, 1, 8, 64, 1), (3, 4, 16, 128, 5),
                                                       (2, 2, 64, 64, 20), (28, 2, 8, 64, 500)])
def test_copy_pages(cuda, krlib, layout, layers, heads, page, D, pairs):
    import torch
    g = _gen(pairs)
    pages = 2 * pairs + 3
    k, v = _cache_tensors(layers, pages, heads, page, D, torch.bfloat16, layout, g=g)
    want = [k.clone(), v.clone()]
    rng = random.Random(pairs)
    order = list(range(pages))
    rng.shuffle(order)
    dst = order[:pairs]
    src = [rng.choice(order[pairs:]) for _ in dst]  # one page may be copied to several
    src[0], dst[0] = (dst[0], dst[0]) if pairs > 1 else (src[0], dst[0])
    for s, d in zip(src, dst):
        for w in want:
            w[:, d] = w[:, s]
    krlib.kv_copy_pages(krlib.KVCache(k, v), src, dst)
    torch.cuda.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_copy_pages_captured(cuda, krlib):
    """The page lists are read before the call returns: a replay copies the captured pages."""
    import torch
    g = _gen(0)
    k, v = _cache_tensors(2, 8, 2, 16, 64, torch.float16, "hnd", g=g)
    cache, src = krlib.KVCache(k, v), [0, 1]
    krlib.kv_copy_pages(cache, src, [2, 3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        krlib.kv_copy_pages(cache, src, [4, 5])
    src[0] = 7
    k.normal_(generator=g)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(k[:, 4], k[:, 0]) and torch.equal(k[:, 5], k[:, 1])
    assert torch.equal(v[:, 4], v[:, 0])


# ---------------------------------------------------------------- commit
@pytest.mark.parametrize("layout", ["hnd", "nhd", "paired", "padded"])
@pytest.mark.parametrize("layers,heads,page,D,T,dtype", [(1, 1, 8, 64, 4, "bf16"),
                                                         (3, 4, 16, 128, 33, "fp16"),
                                                         (24, 2, 32, 64, 64, "bf16")])
def test_commit(cuda, krlib, layout, layers, heads, page, D, T, dtype):
    import torch
    g, rng = _gen(T), random.Random(T)
    B = 7
    bases = [0, 1, page - 1, page, 3 * page + 2, 50, 20]
    need = [-(-(b + T) // page) for b in bases]
    pages = sum(need) + 1
    k, v = _cache_tensors(layers, pages, heads, page, D, _dt(dtype), layout, g=g)
    order = list(range(pages))
    rng.shuffle(order)
    table = torch.full((B, max(need)), -7, dtype=torch.int32)
    want, at = [k.clone(), v.clone()], 0
    accepted = torch.full((B, T + 2), -1, dtype=torch.int32)
    counts = []
    for b in range(B):
        ids = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = torch.tensor(ids, dtype=torch.int32)
        n = [0, T, 1, min(T, 9), T // 2, min(T, 17), 2][b]
        acc = sorted(rng.sample(range(T), n))
        accepted[b, :n] = torch.tensor(acc, dtype=torch.int32)
        counts.append(n)
        place = lambda p: (ids[p // page], p % page)  # noqa: E731
        for w in want:
            rows = [w[:, place(bases[b] + x)[0], :, place(bases[b] + x)[1]].clone() for x in acc]
            for i, row in enumerate(rows):
                p, o = place(bases[b] + i)
                w[:, p, :, o] = row
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    krlib.kv_commit(krlib.KVCache(k, v), table.cuda(), i32(bases), accepted.cuda()[:, :T],
                    i32(counts), status=status)
    torch.cuda.synchronize()
    assert status.item() == 0
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_commit_long_list(cuda, krlib):
    """More accepted tokens than a CTA keeps at a time (a prompt's rows closed up)."""
    import torch
    g, rng = _gen(9), random.Random(9)
    page, T, n = 16, 900, 700
    k, v = _cache_tensors(2, T // page + 2, 2, page, 64, torch.float16, "hnd", g=g)
    ids = list(range(k.shape[1]))
    rng.shuffle(ids)
    acc = sorted(rng.sample(range(T), n))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    want = []
    for t in (k, v):
        flat = t[:, ids].transpose(2, 3).reshape(2, -1, 2, 64).clone()  # by position
        flat[:, 3:3 + n] = flat[:, [3 + a for a in acc]]
        want.append(flat)
    krlib.kv_commit(krlib.KVCache(k, v), i32([ids]), i32([3]), i32([acc]), i32([n]))
    torch.cuda.synchronize()
    for t, w in zip((k, v), want):
        assert torch.equal(t[:, ids].transpose(2, 3).reshape(2, -1, 2, 64), w)


def test_commit_refuses_per_sequence(cuda, krlib):
    import torch
    g = _gen(1)
    page, T, B = 8, 6, 8
    k, v = _cache_tensors(2, 4 * B, 2, page, 64, torch.bfloat16, "hnd", g=g)
    k0 = k.clone()
    table = torch.arange(4 * B, dtype=torch.int32).view(B, 4)
    table[5, 1] = 4 * B
    accepted = torch.tensor([[0, 2, 5], [2, 2, 3], [1, 0, 2], [-1, 0, 1], [0, 1, 30], [0, 2, 5],
                             [0, 2, 5], [0, 2, 5]], dtype=torch.int32)
    bases = torch.tensor([5, 5, 5, 5, 5, 5, -1, 5], dtype=torch.int32)
    counts = torch.tensor([3, 3, 3, 3, 3, 3, 3, 4], dtype=torch.int32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    krlib.kv_commit(krlib.KVCache(k, v), table.cuda(), bases.cuda(), accepted.cuda(), counts.cuda(),
                    status=status)
    torch.cuda.synchronize()
    assert status.item() == 1 << 8
    assert torch.equal(k[:, 4:], k0[:, 4:])
    flat0, flat = (x[:, :4].transpose(2, 3).reshape(2, -1, 2, 64) for x in (k0, k))
    assert torch.equal(flat[:, 6], flat0[:, 7]) and torch.equal(flat[:, 7], flat0[:, 10])


# ---------------------------------------------------------------- large caches and batches
@pytest.mark.parametrize("T", [1, 9])
def test_past_32_bits(cuda, krlib, T):
    """A cache of more than 2^31 elements: every operator on its last pages does what it does in a
    small cache, bit for bit."""
    import torch
    HQ, HKV, D, page, n = 16, 8, 128, 64, 600
    dt, g = torch.bfloat16, _gen(T)
    most = 2 ** 31 // (HKV * page * D) + 1200
    cos, sin = _rope_tables(n, D)
    qkv = torch.randn(n, (HQ + 2 * HKV) * D, generator=g, device="cuda").to(dt)
    pos = torch.arange(n, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    need = -(-n // page)
    got = []
    for pages, ids in ((need + 1, list(range(need + 1))),
                       (most, [most - 1 - 7 * i for i in range(need - 1)] + [3, most - 3])):
        k, v = (torch.empty(pages, HKV, page, D, dtype=dt, device="cuda") for _ in range(2))
        cache = krlib.KVCache(k, v)
        slots = torch.tensor(ids, device="cuda")[pos // page] * page + pos % page
        q = krlib.qk_norm_rope_paged(qkv, cache, pos, slots, HQ, cos, sin)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        args = (i32([ids[:need]]), i32([n]), i32([0, T]), T, D ** -0.5)
        first = krlib.attention_paged(q[n - T:], cache, *args, status=status)
        krlib.kv_copy_pages(cache, [ids[0]], [ids[need]])
        krlib.kv_commit(cache, args[0], i32([n - 80]), i32([[1, 4, 70]]), i32([3]), status=status)
        last = krlib.attention_paged(q[n - T:], cache, *args, status=status)
        torch.cuda.synchronize()
        assert status.item() == 0
        got.append([q, first, last, k[ids[need]].clone(), v[ids[need]].clone(), k[ids[0]].clone()])
        del k, v, cache
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert not torch.equal(got[0][1], got[0][2])  # the commit moved rows that are attended to
    torch.cuda.empty_cache()


def test_thousands_of_sequences(cuda, krlib):
    import torch
    rng = random.Random(3)
    b = Batch([(rng.choice([0, 1, 7, 30]), rng.choice([0, 1, 1])) for _ in range(3001)], 4, 2, 64, 8, seed=3)
    out = b.run(krlib)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    b.check(out)


def test_long_chunk(cuda, krlib):
    """Thousands of new tokens in one sequence: hundreds of units of its own."""
    import torch
    b = Batch([(100, 5000), (9, 2)], 8, 2, 64, 64, "fp16", seed=8)
    out = b.run(krlib)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    b.check(out)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("HQ,HKV,D,dtype", [(14, 2, 64, "bf16"), (8, 2, 128, "fp16")])
def test_draft_verify_commit(cuda, krlib, HQ, HKV, D, dtype):
    """Two sequences, one forked from the other, grow by drafted trees of which a path is kept:
    each step's attention equals that of the tokens' plain history."""
    import torch
    dt, g, rng = _dt(dtype), _gen(7), random.Random(7)
    u = torch.finfo(dt).eps / 2
    page, T, pages, G = 16, 12, 64, HQ // HKV
    k, v = _cache_tensors(1, pages, HKV, page, D, dt, "hnd", fill=float("nan"))
    cache = krlib.KVCache(k, v)
    cos, sin = _rope_tables(256, D)
    free = list(range(pages))
    rng.shuffle(free)
    table = [[free.pop() for _ in range(8)] for _ in range(2)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def qkv(n):
        return torch.randn(n, (HQ + 2 * HKV) * D, generator=g, device="cuda").to(dt)

    def slots(b, positions):
        return [table[b][p // page] * page + p % page for p in positions]

    def rotated(x, pos):
        x = x.double().view(x.shape[0], -1, D)
        return _append_ref(x, None, cos[pos], sin[pos])[0]

    # the prompt of sequence 0; sequence 1 shares its full pages and gets its own last one
    L = 37
    x = qkv(L)
    pos = torch.arange(L, device="cuda")
    krlib.qk_norm_rope_paged(x, cache, pos, torch.tensor(slots(0, range(L)), device="cuda"), HQ, cos, sin)
    own = table[1][:]
    table[1] = table[0][:L // page] + own[L // page:]
    krlib.kv_copy_pages(cache, [table[0][L // page]], [table[1][L // page]])
    hist = [[(rotated(x, pos)[i, HQ:HQ + HKV], x.double().view(L, -1, D)[i, HQ + HKV:]) for i in range(L)]
            for _ in range(2)]
    lens = [L, L]
    for step in range(4):
        xs, positions, all_slots, masks, paths, sees = [], [], [], [], [], []
        for b in range(2):
            parent = [-1] + [rng.randint(0, i - 1) for i in range(1, T)]
            up = [{i} for i in range(T)]
            for i in range(1, T):
                up[i] |= up[parent[i]]
            depth = [len(s) - 1 for s in up]
            xs.append(qkv(T))
            positions += [lens[b] + d for d in depth]
            all_slots += slots(b, range(lens[b], lens[b] + T))
            masks += [[sum(1 << j for j in s)] for s in up]
            sees.append(up)
            paths.append(sorted(up[rng.randrange(T)]))
        x = torch.cat(xs)
        pos = torch.tensor(positions, device="cuda")
        q = krlib.qk_norm_rope_paged(x, cache, pos, torch.tensor(all_slots, device="cuda"), HQ, cos, sin)
        out = krlib.attention_paged(q, cache, i32(table), i32([n + T for n in lens]), i32([0, T, 2 * T]),
                                    T, 1 / math.sqrt(D), mask=i32(masks))
        torch.cuda.synchronize()
        rot = rotated(x, pos)
        for b in range(2):
            for i in range(T):
                r = b * T + i
                ks = [h[0] for h in hist[b]] + [rot[b * T + j, HQ:HQ + HKV] for j in sorted(sees[b][i])]
                vs = [h[1] for h in hist[b]] + [x.double().view(2 * T, -1, D)[b * T + j, HQ + HKV:]
                                                for j in sorted(sees[b][i])]
                K, V = torch.stack(ks), torch.stack(vs)
                s = torch.einsum("hgd,nhd->hgn", rot[r, :HQ].view(HKV, G, D), K) / math.sqrt(D)
                p = torch.softmax(s, -1)
                ref = torch.einsum("hgn,nhd->hgd", p, V).reshape(-1)
                A = torch.einsum("hgn,nhd->hgd", p, V.abs()).reshape(-1)
                # q and k are stored rounded: scores move by up to 2u S, probabilities by 4u S
                S = (torch.einsum("hgd,nhd->hgn", rot[r, :HQ].view(HKV, G, D).abs(), K.abs())
                     / math.sqrt(D)).max()
                assert ((out[r].double() - ref).abs() <= u * ref.abs() + (u + 4.5 * u * S + 1e-4) * A).all()
        acc = torch.full((2, T), -1, dtype=torch.int32)
        for b in range(2):
            acc[b, :len(paths[b])] = torch.tensor(paths[b], dtype=torch.int32)
            hist[b] += [(rot[b * T + j, HQ:HQ + HKV], x.double().view(2 * T, -1, D)[b * T + j, HQ + HKV:])
                        for j in paths[b]]
        krlib.kv_commit(cache, i32(table), i32(lens), acc.cuda(), i32([len(p) for p in paths]))
        lens = [n + len(p) for n, p in zip(lens, paths)]


# ---------------------------------------------------------------- small probabilities
@pytest.mark.parametrize("T", [1, 8, 40])
@pytest.mark.parametrize("HQ,HKV,D", [(28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("fall", [(15.0, 15.0), (24.875, 24.875), (25.125, 25.125), (14.0, 30.0)])
def test_small_probabilities_count_in_fp16(cuda, krlib, T, HQ, HKV, D, fall):
    """One key far above all others, whose value is zero: the output is what the thousands of small
    probabilities add up to, 2^-14 to 2^-30 of the largest each (below fp16's normal numbers).  Bound:
    that of the attention tests with a probability's absolute error 2^-25 relative to the largest
    one's power of two, which is 2^15 or, behind an offset that lags by up to 8, 2^7."""
    import torch
    B, n, page = 128, 16384, 64  # units enough that most lie whole in a CTA, the largest key with them
    u = 2.0 ** -11
    g = _gen(T)
    x = torch.linspace(*fall, n, device="cuda")  # log2 of how far a key is below the first
    x[0] = 0
    k = torch.zeros(1, n // page, HKV, page, D, dtype=torch.float16, device="cuda")
    v = torch.rand(k.shape, generator=g, device="cuda").add_(0.5).half()
    k[0, ..., 0] = (-x / 8).half().view(n // page, 1, page)
    v[0, 0, :, 0] = 0
    q = torch.zeros(B * T, HQ, D, dtype=torch.float16, device="cuda")
    q[..., 0] = 8
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").repeat(B, 1)
    mask = torch.full((B * T, 2), -1, dtype=torch.int32, device="cuda")  # every row sees every key
    out = krlib.attention_paged(q.view(B * T, -1), krlib.KVCache(k, v), table, i32([n] * B),
                                i32([T * i for i in range(B + 1)]), T, math.log(2), mask=mask)
    torch.cuda.synchronize()
    K, V = (t[0].transpose(1, 2).reshape(n, HKV, D).double() for t in (k, v))
    p = torch.softmax(K[:, 0, 0] * 8 * math.log(2), 0)
    ref = torch.einsum("n,nhd->hd", p, V)
    S = fall[1] * math.log(2)
    rel = 2 * (D + 4) * 2.0 ** -24 * S + n * 2.0 ** -24 + 2.0 ** -20
    bound = u * ref + (u + rel) * ref * (1 + 2 * u) + 2.0 ** -32 * V.sum(0) + 2.0 ** -25
    got = out.double().view(B * T, HKV, HQ // HKV, D)
    bad = ~((got - ref[None, :, None]).abs() <= bound[None, :, None])
    assert not bad.any(), ((got - ref[None, :, None]) / ref[None, :, None]).abs().max().item()


# ---------------------------------------------------------------- outputs beside inputs
@pytest.mark.parametrize("T", [1, 40])
def test_outputs_between_input_rows(cuda, krlib, T):
    """q, qkv and outputs as columns of one buffer, of equal and of different pitches, overlap in no
    element: they are taken, and give what apart from each other they give."""
    import torch
    b = Batch([(70, T), (9, T)], 8, 2, 64, 16, seed=T)
    want = b.run(krlib)
    N, w = b.q.shape
    for lda, at, ldo in ((3 * w, w, 3 * w), (4 * w, w, 2 * w), (2 * w + 8, w + 8, 2 * w + 8)):
        flat = torch.full((N * 4 * w,), 5.0, dtype=b.dt, device="cuda")
        q = flat.as_strided((N, w), (lda, 1))
        q.copy_(b.q)
        out = flat.as_strided((N, w), (ldo, 1), at)
        out.fill_(5.0)
        keep, b.q = b.q, q
        got = b.run(krlib, out=out)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(q, keep)
        b.q = keep
    HQ, HKV, D = 8, 2, 64
    wide = torch.randn(N, 2 * (HQ + 2 * HKV) * D, generator=b.g, device="cuda").to(b.dt)
    qkv, out = wide[:, :(HQ + 2 * HKV) * D], wide[:, (HQ + 2 * HKV) * D:][:, :HQ * D]
    cos, sin = _rope_tables(64, D)
    pos = torch.arange(N, device="cuda") % 64
    slots = torch.full((N,), -1, device="cuda")
    cache = krlib.KVCache(b.k, b.v)
    want = krlib.qk_norm_rope_paged(qkv, cache, pos, slots, HQ, cos, sin)
    got = krlib.qk_norm_rope_paged(qkv, cache, pos, slots, HQ, cos, sin, out=out)
    assert torch.equal(got, want)
    assert torch.equal(krlib.qk_norm_rope_paged(qkv, cache, pos, slots, HQ, cos, sin, out=qkv[:, :HQ * D]),
                       want)  # in place
    with pytest.raises(krlib.KrbError, match="overlaps qkv"):
        krlib.qk_norm_rope_paged(qkv, cache, pos, slots, HQ, cos, sin, out=qkv[:, D:HQ * D + D])
    with pytest.raises(krlib.KrbError, match="overlaps q"):
        b.run(krlib, out=b.q)


# ---------------------------------------------------------------- steps without tokens
@pytest.mark.parametrize("max_q", [0, 1, 40])
def test_attention_without_tokens(cuda, krlib, max_q):
    import torch
    k, v = _cache_tensors(1, 2, 2, 16, 64, torch.bfloat16, "hnd", fill=1.0)
    cache = krlib.KVCache(k, v)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.empty(0, 8 * 64, dtype=torch.bfloat16, device="cuda")
    assert krlib.attention_paged(q, cache, i32(3, 2), i32(3), i32(4), max_q, 0.1).shape == q.shape
    assert krlib.attention_paged(q, cache, i32(0, 2), i32(0), i32(1), max_q, 0.1).shape == q.shape
    out = torch.full((5, 8 * 64), 5.0, dtype=torch.bfloat16, device="cuda")
    got = krlib.attention_paged(torch.ones_like(out), cache, i32(0, 2), i32(0), i32(1), max_q, 0.1, out=out)
    torch.cuda.synchronize()
    assert (got == 5.0).all()  # rows of no sequence
    assert cache.attention_workspace(8, 0) == cache.attention_workspace(8, 1) > 0


# ---------------------------------------------------------------- refusals in every kernel
# 28 heads over 4: rows of 1 token are 7 (mma.sync), of 8 tokens 56 (tcgen05, one tile), of 40 two tiles
TOKENS = [1, 8, 40]


def _left(b, out, refused):
    """Rows of refused sequences, and rows of none, are as they were."""
    for i in refused:
        assert (out[b.starts_host[i]:b.starts_host[i + 1]] == 5.0).all(), i
    assert (out[b.starts_host[-1]:] == 5.0).all()


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("masked", [False, True])
def test_refused_lengths_leave_rows(cuda, krlib, T, masked):
    import torch
    seqs = [(100, T), (64, T), (10, max(1, T - 1)), (300, T), (0, T)]
    b = Batch(seqs, 28, 4, 128, 16, seed=T, masked=masked)
    for lens, bad in (({1: T - 1}, {1}), ({0: -5}, {0}), ({3: 10 ** 9}, {3}), ({4: 0, 2: 2 ** 31 - 1}, {2, 4}),
                      ({0: -2 ** 31, 1: -1, 2: 0, 3: 0, 4: -1}, {0, 1, 2, 3, 4})):
        saved = b.lens.clone()
        for i, n in lens.items():
            b.lens[i] = n
        out = b.run(krlib)
        torch.cuda.synchronize()
        assert b.status.item() == 1 << 7
        b.lens.copy_(saved)
        _left(b, out, bad)
        b.check(out, only=set(range(5)) - bad)
    if T > 1:  # more new tokens than max_q
        out = b.run(krlib, max_q=T - 1)
        torch.cuda.synchronize()
        assert b.status.item() == 1 << 7
        _left(b, out, {0, 1, 3, 4})
        b.check(out, only={2})


@pytest.mark.parametrize("T", TOKENS)
def test_refused_starts_leave_rows(cuda, krlib, T):
    import torch
    seqs = [(100, T), (64, T), (10, T), (300, T), (0, T)]
    b = Batch(seqs, 28, 4, 128, 16, seed=T)
    want = b.run(krlib).clone()
    for i, x, bad in ((5, b.N + 1, {4}), (0, -1, {0}), (2, b.N + 7, {1, 2}), (3, 2 * T - 1, {2, 3}),
                      (5, -2 ** 31, {4}), (1, 2 ** 31 - 1, {0, 1})):
        saved = b.starts.clone()
        b.starts[i] = x
        out = b.run(krlib)
        torch.cuda.synchronize()
        assert b.status.item() == 1 << 7
        b.starts.copy_(saved)
        _left(b, out, bad)
        for j in set(range(5)) - bad:
            rows = slice(T * j, T * j + T)
            b.check(out, only={j})
            assert torch.isfinite(out[rows]).all()
    assert torch.equal(b.run(krlib), want)


@pytest.mark.parametrize("T", TOKENS)
def test_bad_pages_read_as_page_0(cuda, krlib, T):
    import torch
    b = Batch([(200, T), (100, T)], 28, 4, 128, 16, seed=2)
    saved = b.table.clone()
    b.table[0, 3] = 0
    want = b.run(krlib).clone()
    for bad in (b.pages, -1, 2 ** 31 - 1, -2 ** 31):
        b.table[0, 3] = bad
        out = b.run(krlib)
        torch.cuda.synchronize()
        assert b.status.item() == 1 << 8
        b.check(out, only={1})
        assert torch.equal(out.view(torch.int16), want.view(torch.int16))
        _left(b, out, set())
    b.table.copy_(saved)
    out = b.run(krlib)
    torch.cuda.synchronize()
    assert b.status.item() == 0
    b.check(out)


@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("heads,B", [(8, 2), (4, 33)])
def test_refused_calls(cuda, krlib, T, heads, B):
    """More than 2^26 blocks of 64 keys in a sequence, or 2^31 in the batch: the whole call is refused
    before a key is read (2^30 positions are 2^24 blocks a head)."""
    import torch
    page, D = 1024, 64
    k, v = _cache_tensors(1, 2, heads, page, D, torch.bfloat16, "hnd", fill=1.0)
    table = torch.zeros(B, 2 ** 30 // page, dtype=torch.int32, device="cuda")
    lens = torch.full((B,), 2 ** 30, dtype=torch.int32, device="cuda")
    if heads == 8:
        lens[0] = 100
    starts = torch.arange(B + 1, dtype=torch.int32, device="cuda") * T
    q = torch.ones(B * T, heads * D, dtype=torch.bfloat16, device="cuda")
    out = torch.full_like(q, 5.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    krlib.attention_paged(q, krlib.KVCache(k, v), table, lens, starts, T, 0.1, out=out, status=status)
    torch.cuda.synchronize()
    assert status.item() == 1 << 7
    assert (out == 5.0).all()
    lens.fill_(T + 100)  # the same arrays, lengths that are taken
    status.zero_()
    krlib.attention_paged(q, krlib.KVCache(k, v), table, lens, starts, T, 0.1, out=out, status=status)
    torch.cuda.synchronize()
    assert status.item() == 0
    assert (out == 1.0).all()


@pytest.mark.parametrize("T", TOKENS)
def test_graph_follows_lengths_and_starts(cuda, krlib, T):
    import torch
    seqs = [(900, T), (333, T), (64, T)]
    b = Batch(seqs, 28, 4, 128, 16, seed=9)
    b.run(krlib)
    out = torch.full((b.N, b.HQ * b.D), 5.0, dtype=b.dt, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache = krlib.KVCache(b.k, b.v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        krlib.attention_paged(b.q, cache, b.table, b.lens, b.starts, T, b.scale, out=out, status=status)
    for cut, new in ((0, (T, T, T)), (17, (T, 0, T)), (63, (max(1, T - 3), T, 1)), (5, (0, 0, 0)),
                     (1, (T, T, T))):
        lens = [c - cut + t for (c, _), t in zip(seqs, new)]
        starts = [sum(new[:i]) for i in range(4)]
        b.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        b.starts.copy_(torch.tensor(starts, dtype=torch.int32))
        out.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        assert status.item() == 0
        now = Batch(seqs, 28, 4, 128, 16, seed=9)
        now.seqs, now.starts_host = [(c - cut, t) for (c, _), t in zip(seqs, new)], starts
        now.sees = [torch.ones(t, t, dtype=torch.bool, device="cuda").tril() for t in new]
        now.K, now.V = ([x[:n] for x, n in zip(xs, lens)] for xs in (now.K, now.V))
        now.check(out)
        assert (out[starts[-1]:] == 5.0).all()


@pytest.mark.parametrize("T", [8, 40])
@pytest.mark.parametrize("masked", [False, True])
def test_same_result_twice_many_rows(cuda, krlib, T, masked):
    import torch
    b = Batch([(5000, T), (77, T), (2500, T)], 28, 4, 128, 16, seed=4, masked=masked)
    a = b.run(krlib)
    for _ in range(5):
        assert torch.equal(a, b.run(krlib))


@pytest.mark.parametrize("B,n", [(1, 63), (1, 64), (3, 65), (1, 1999), (70, 1999), (1, 8191), (50, 4097)])
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("HQ,HKV,D,dtype", [(28, 4, 128, "bf16"), (14, 2, 64, "fp16")])
def test_every_key_counts_once(cuda, krlib, B, n, T, HQ, HKV, D, dtype):
    """Scores of 0, and values of one in column j % D for key j: a column is its number of keys over n, so
    one key lost or taken twice moves it by D / n, far more than the roundings (of 1 / n, of the product
    and the output's: the sums are whole numbers)."""
    import torch
    dt, page, g = _dt(dtype), 16, _gen(n)
    need = -(-n // page)
    v = torch.eye(D, device="cuda")[torch.arange(need * page, device="cuda") % D].to(dt)
    v = v.view(1, need, page, 1, D).expand(1, need, page, HKV, D).transpose(2, 3).contiguous()
    k = torch.randn(v.shape, generator=g, device="cuda").to(dt)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(need, dtype=torch.int32, device="cuda").repeat(B, 1)
    mask = torch.full((B * T, 2), -1, dtype=torch.int32, device="cuda")
    q = torch.zeros(B * T, HQ * D, dtype=dt, device="cuda")
    out = krlib.attention_paged(q, krlib.KVCache(k, v), table, i32([n] * B),
                                i32([T * i for i in range(B + 1)]), T, 0.1, mask=mask)
    torch.cuda.synchronize()
    count = torch.bincount(torch.arange(n, device="cuda") % D, minlength=D).double()
    ref = count / n
    bound = (torch.finfo(dt).eps / 2 + 2.0 ** -22) * ref + 2.0 ** -25 * (dt == torch.float16)
    assert D / n > 2 * bound.max() / ref.max() or n < D
    assert ((out.double().view(B * T, HQ, D) - ref).abs() <= bound).all()


# ---------------------------------------------------------------- streams
def test_stream_argument(cuda, krlib):
    """append, page copies and commits on the stream that they are given, behind its work and not behind
    (or in) the current one's."""
    import torch
    HQ, HKV, D, page, n = 8, 2, 128, 16, 256
    g, dt = _gen(1), torch.bfloat16
    cos, sin = _rope_tables(n, D)
    pos = torch.arange(n, device="cuda")
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    table, bases, accepted, counts = i32([list(range(n // page))]), i32([100]), i32([[1, 5, 9]]), i32([3])
    busy = torch.randn(4096, 4096, generator=g, device="cuda")
    x = torch.randn(n, (HQ + 2 * HKV) * D, generator=g, device="cuda").to(dt)

    def step(**kw):
        k, v = _cache_tensors(1, n // page + 1, HKV, page, D, dt, "hnd", fill=0.0)
        cache, src = krlib.KVCache(k, v), torch.zeros_like(x)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.stream(kw.get("stream") or torch.cuda.current_stream()):
            for _ in range(3):
                (busy @ busy).sum()
            src.copy_(x)
        q = krlib.qk_norm_rope_paged(src, cache, pos, pos, HQ, cos, sin, status=status, **kw)
        krlib.kv_copy_pages(cache, [3], [n // page], **kw)
        krlib.kv_commit(cache, table, bases, accepted, counts, status=status, **kw)
        torch.cuda.synchronize()
        assert status.item() == 0
        return q, k, v

    want, got = step(), step(stream=torch.cuda.Stream())
    for a, b in zip(want, got):
        assert torch.equal(a, b) and a.abs().max() > 0
    assert torch.equal(want[1][0, n // page], want[1][0, 3])


# ---------------------------------------------------------------- a whole step captured
@pytest.mark.parametrize("T", TOKENS)
def test_step_captured(cuda, krlib, T):
    """Append, attention, page copy and commit in one graph: a replay on new rows, slots, lengths, masks
    and lists does what the calls do."""
    import torch
    HQ, HKV, D, page, B, L = 28, 4, 128, 16, 3, 2
    dt, g, need = torch.bfloat16, _gen(T), 12
    pages = B * need + 1
    cos, sin = _rope_tables(need * page, D)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    words = -(-T // 32)

    def inputs(seed):
        r = random.Random(seed)
        ids = list(range(pages - 1))
        r.shuffle(ids)
        rows = [ids[b * need:(b + 1) * need] for b in range(B)]
        ctx = [r.randint(0, need * page - T) for _ in range(B)]
        at = [(b, c + t) for b, c in enumerate(ctx) for t in range(T)]
        acc = [sorted(r.sample(range(T), min(T, 2))) + [-1] * (2 - min(T, 2)) for _ in range(B)]
        masks = torch.cat([_tree(r, T, words)[0] for _ in range(B)])
        return dict(qkv=torch.randn(B * T, (HQ + 2 * HKV) * D, generator=_gen(seed), device="cuda").to(dt),
                    pos=torch.tensor([p for _, p in at], device="cuda"),
                    slots=torch.tensor([rows[b][p // page] * page + p % page for b, p in at], device="cuda"),
                    table=i32(rows), lens=i32([c + T for c in ctx]), bases=i32(ctx), acc=i32(acc),
                    counts=i32([r.randint(0, min(T, 2)) for _ in range(B)]), mask=masks.cuda())

    starts = i32([T * i for i in range(B + 1)])
    k0, v0 = _cache_tensors(L, pages, HKV, page, D, dt, "nhd", g=g)

    def step(s, cache, status):
        outs = []
        for layer in range(L):
            q = krlib.qk_norm_rope_paged(s["qkv"], cache, s["pos"], s["slots"], HQ, cos, sin, layer=layer,
                                         status=status)
            outs.append(krlib.attention_paged(q, cache, s["table"], s["lens"], starts, T, D ** -0.5,
                                              mask=s["mask"], layer=layer, status=status))
        krlib.kv_copy_pages(cache, [3], [pages - 1])
        krlib.kv_commit(cache, s["table"], s["bases"], s["acc"], s["counts"], status=status)
        return outs

    held, status = inputs(0), torch.zeros(1, dtype=torch.int32, device="cuda")
    k, v = k0.clone(), v0.clone()
    cache = krlib.KVCache(k, v)
    step(held, cache, status)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(held, cache, status)
    for seed in (1, 2, 3):
        new = inputs(seed)
        for name, x in new.items():
            held[name].copy_(x)
        k.copy_(k0)
        v.copy_(v0)
        graph.replay()
        torch.cuda.synchronize()
        k1, v1 = k0.clone(), v0.clone()
        want = step(new, krlib.KVCache(k1, v1), status)
        torch.cuda.synchronize()
        assert status.item() == 0
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        assert torch.equal(k, k1) and torch.equal(v, v1)
        assert not torch.equal(outs[0], outs[1]) and not torch.equal(k, k0)


# ---------------------------------------------------------------- very large scores
@pytest.mark.parametrize("T", TOKENS)
@pytest.mark.parametrize("HQ,HKV,D", [(28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("sign", [1, -1])
def test_very_large_scores(cuda, krlib, T, HQ, HKV, D, dtype, sign):
    """Scores up to 2^27 (in log2 units), where neighbouring fp32 numbers are 8 apart and a maximum's
    product with the scale is off by as much: one key far above the others is the output, whatever
    those roundings.  Its probability is rounded once (u), the output once more (u)."""
    import torch
    dt, B, n, page, g = _dt(dtype), 40, 700, 16, _gen(T)
    u = torch.finfo(dt).eps / 2
    need = -(-n // page)
    k = torch.empty(1, need, HKV, page, D, dtype=dt, device="cuda").fill_(992 if sign > 0 else 1024)
    k[0, 30, :, 5] = 1000
    if sign < 0:
        k[0, 30, :, 5] = 1000  # the least negative of them
    v = torch.randn(k.shape, generator=g, device="cuda").to(dt)
    top = 2.0 ** torch.linspace(18, 27, B * T, device="cuda")
    scale = D ** -0.5
    q = (sign * top / (1000 * D * scale * math.log2(math.e)))[:, None, None].expand(B * T, HQ, D).to(dt)
    assert torch.isfinite(q).all()
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    table = torch.arange(need, dtype=torch.int32, device="cuda").repeat(B, 1)
    mask = torch.full((B * T, 2), -1, dtype=torch.int32, device="cuda")
    out = krlib.attention_paged(q.reshape(B * T, -1), krlib.KVCache(k, v), table, i32([n] * B),
                                i32([T * i for i in range(B + 1)]), T, scale, mask=mask)
    torch.cuda.synchronize()
    ref = v[0, 30, :, 5].double()[None, :, None]
    got = out.double().view(B * T, HKV, HQ // HKV, D)
    bad = ~((got - ref).abs() <= (2 * u + u * u + 2.0 ** -20) * ref.abs() + 2.0 ** -25)
    assert not bad.any(), bad.view(B * T, -1).any(1).nonzero().flatten().tolist()[:9]
