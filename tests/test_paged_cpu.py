"""Refusals of the paged K/V cache operators, none of which reaches a GPU: through the C ABI with
addresses that are never followed, and through the Python wrappers with CPU tensors."""
import ctypes

import pytest


def _desc(krlib, **over):
    d = krlib.KVCacheDesc(4096, 8192, 0, 2, 10, 4, 16, 128,
                          (ctypes.c_int64 * 4)(81920, 8192, 2048, 128),
                          (ctypes.c_int64 * 4)(81920, 8192, 2048, 128))
    for key, x in over.items():
        setattr(d, key, (ctypes.c_int64 * 4)(*x) if key.endswith("stride") else x)
    return d


def _message(krlib):
    return krlib.lib().krb_last_error().decode()


BAD_CACHES = [
    (dict(k=0), "without K or V"), (dict(v=0), "without K or V"), (dict(k=4104), "aligned"),
    (dict(v=4096), "same array"),
    (dict(dtype=2), "dtype"), (dict(layers=0), "layers"), (dict(pages=-1), "pages"),
    (dict(heads=0), "heads"), (dict(head_dim=96), "head_dim"), (dict(page_size=24), "power of two"),
    (dict(page_size=4), "power of two"),
    (dict(k_stride=(81920, 8192, 2048, 120)), "overlap"),
    (dict(v_stride=(81920, 8192, 2044, 128)), "multiples of 8"),
    (dict(k_stride=(0, 8192, 2048, 128)), "overlap"),
    (dict(v_stride=(81920, -8192, 2048, 128)), "overlap"),
    (dict(k_stride=(40960, 8192, 2048, 128)), "overlap"),
]


@pytest.mark.parametrize("over,what", BAD_CACHES)
def test_bad_caches(krlib, over, what):
    L = krlib.lib()
    ref = ctypes.addressof(d := _desc(krlib, **over))
    one = (ctypes.c_int * 1)(1)
    assert L.krb_kv_copy_pages(ref, one, one, 1, None) == 1 and what in _message(krlib)
    assert L.krb_qk_norm_rope_paged(ref, 0, 16, 4096, 16, 4096, 16, 16, 1, 28, 16, 16, 8, None, None,
                                    1e-6, None, None) == 1 and what in _message(krlib)
    assert L.krb_attention_paged(ref, 0, 16, 3584, 16, 3584, 1, 28, 16, 8, 8, 16, 16, 1, 1, None, 0, 0,
                                 0.1, 16, 1 << 30, None, None) == 1 and what in _message(krlib)
    assert L.krb_kv_commit(ref, 16, 8, 8, 16, 16, 4, 4, 16, 1, None, None) == 1 and what in _message(krlib)
    assert L.krb_attention_paged_workspace(ref, 28, 1) == 0 and what in _message(krlib)
    del d
    assert L.krb_kv_copy_pages(None, one, one, 1, None) == 1 and "no cache" in _message(krlib)


def test_legal_cache_layouts(krlib):
    """Axis orders and lengths of one that check_cache takes: the next refusal is reached."""
    L = krlib.lib()
    bad = (ctypes.c_int * 1)(99)
    for over in (dict(), dict(k_stride=(81920, 8192, 128, 512), v_stride=(81920, 8192, 128, 512)),
                 dict(k_stride=(8192 * 2, 8192 * 4, 2048, 128)),
                 dict(layers=1, k_stride=(0, 8192, 2048, 128)),
                 dict(heads=1, k_stride=(81920, 8192, 3, 128))):
        d = _desc(krlib, **over)
        assert L.krb_kv_copy_pages(ctypes.addressof(d), bad, bad, 1, None) == 1
        assert "no page 99" in _message(krlib)


@pytest.mark.parametrize("src,dst,what", [
    ([0], [10], "no page 10"), ([-1], [2], "no page -1"), ([0, 1], [2, 2], "page 2 is written twice"),
    ([0, 1], [1, 2], "page 1 is read and written"), ([1, 0], [2, 1], "page 1 is read and written"),
])
def test_copy_refusals(krlib, src, dst, what):
    d = _desc(krlib)
    a, b = ((ctypes.c_int * len(x))(*x) for x in (src, dst))
    L = krlib.lib()
    assert L.krb_kv_copy_pages(ctypes.addressof(d), a, b, len(src), None) == 1
    assert what in _message(krlib)
    assert L.krb_kv_copy_pages(ctypes.addressof(d), None, b, 1, None) == 1
    assert "null" in _message(krlib)
    assert L.krb_kv_copy_pages(ctypes.addressof(d), a, b, -1, None) == 1
    assert L.krb_kv_copy_pages(ctypes.addressof(d), a, b, 0, None) == 0
    same = (ctypes.c_int * 2)(3, 4)  # pages onto themselves: nothing to launch
    assert L.krb_kv_copy_pages(ctypes.addressof(d), same, same, 2, None) == 0


APPEND = dict(layer=0, qkv=16, ldqkv=36 * 128, q=16, ldq=28 * 128, pos=16, slots=16, N=3, HQ=28, cos=16,
              sin=16, max_pos=8, qn=None, kn=None)


@pytest.mark.parametrize("over,what", [
    (dict(layer=2), "layer"), (dict(layer=-1), "layer"), (dict(N=-1), "bad N"), (dict(HQ=0), "bad N"),
    (dict(qkv=None), "null"), (dict(pos=None), "null"), (dict(slots=None), "null"), (dict(cos=None), "null"),
    (dict(qn=16), "neither"), (dict(max_pos=0), "empty"), (dict(ldqkv=36 * 128 - 8), "pitch"),
    (dict(ldq=28 * 128 + 4), "pitch"), (dict(qkv=8), "aligned"), (dict(q=24), "aligned"),
    (dict(qn=16, kn=18), "aligned"),
])
def test_append_refusals(krlib, over, what):
    d, a = _desc(krlib), {**APPEND, **over}
    rc = krlib.lib().krb_qk_norm_rope_paged(
        ctypes.addressof(d), a["layer"], a["qkv"], a["ldqkv"], a["q"], a["ldq"], a["pos"], a["slots"],
        a["N"], a["HQ"], a["cos"], a["sin"], a["max_pos"], a["qn"], a["kn"], 1e-6, None, None)
    assert rc == 1 and what in _message(krlib)


ATTN = dict(layer=0, q=16, ldq=28 * 128, out=16, ldo=28 * 128, N=3, HQ=28, table=16, ldp=8, P=8, lens=16,
            starts=16, B=2, max_q=1, mask=None, ldm=0, words=0, scale=0.1, ws=16)


@pytest.mark.parametrize("over,what", [
    (dict(layer=2), "layer"), (dict(HQ=27), "multiple"), (dict(HQ=0), "multiple"),
    (dict(HQ=4 * 65, ldq=65 * 512, ldo=65 * 512), "64 query heads"), (dict(max_q=0), "max_q"),
    (dict(N=-1), "negative"), (dict(B=-1), "negative"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(table=None), "null"), (dict(lens=None), "null"), (dict(starts=None), "null"),
    (dict(ldq=28 * 128 - 8), "pitch"), (dict(ldo=28 * 128 + 1), "pitch"), (dict(q=2), "aligned"),
    (dict(out=8), "aligned"), (dict(ws=8), "aligned"), (dict(P=0), "page table"), (dict(ldp=7), "page table"),
    (dict(P=1 << 27, ldp=1 << 27), "2^30"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(mask=16, words=0, ldm=4), "mask"), (dict(mask=16, words=1, ldm=1, max_q=33), "mask"),
    (dict(mask=16, words=2, ldm=1), "mask"),
])
def test_attention_refusals(krlib, over, what):
    d, a = _desc(krlib), {**ATTN, **over}
    rc = krlib.lib().krb_attention_paged(
        ctypes.addressof(d), a["layer"], a["q"], a["ldq"], a["out"], a["ldo"], a["N"], a["HQ"],
        a["table"], a["ldp"], a["P"], a["lens"], a["starts"], a["B"], a["max_q"], a["mask"], a["ldm"],
        a["words"], a["scale"], a["ws"], 1 << 40, None, None)
    assert rc == 1 and what in _message(krlib)


@pytest.mark.parametrize("over,what", [
    (dict(table=None), "null"), (dict(bases=None), "null"), (dict(acc=None), "null"),
    (dict(counts=None), "null"), (dict(P=0), "page table"), (dict(ldp=7), "page table"),
    (dict(lda=3), "accepted"), (dict(B=-1), "negative"), (dict(A=-1), "negative"),
    (dict(P=1 << 27, ldp=1 << 27), "2^30"),
])
def test_commit_refusals(krlib, over, what):
    a = {**dict(table=16, ldp=8, P=8, bases=16, acc=16, lda=4, A=4, counts=16, B=2), **over}
    d = _desc(krlib)
    rc = krlib.lib().krb_kv_commit(ctypes.addressof(d), a["table"], a["ldp"], a["P"], a["bases"],
                                   a["acc"], a["lda"], a["A"], a["counts"], a["B"], None, None)
    assert rc == 1 and what in _message(krlib)


def test_empty_calls_do_nothing(krlib):
    d = ctypes.addressof(keep := _desc(krlib))
    L = krlib.lib()
    assert L.krb_qk_norm_rope_paged(d, 0, None, 0, None, 0, None, None, 0, 28, None, None, 0, None, None,
                                    1e-6, None, None) == 0
    for N, B in ((0, 2), (3, 0)):
        assert L.krb_attention_paged(d, 0, None, 0, None, 0, N, 28, None, 0, 0, None, None, B, 1, None, 0,
                                     0, 0.1, None, 0, None, None) == 0
    for A, B in ((0, 2), (3, 0)):
        assert L.krb_kv_commit(d, None, 0, 0, None, None, 0, A, None, B, None, None) == 0
    del keep


# ---------------------------------------------------------------- the wrappers
def _cpu_cache(krlib, **kw):
    import torch
    k = torch.zeros(2, 6, 2, 16, 64, dtype=kw.get("dtype", torch.bfloat16))
    return krlib.KVCache(k, torch.zeros_like(k))


def test_cache_handle_refusals(krlib):
    import torch
    k = torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16)
    c = krlib.KVCache(k, k.clone())
    assert (c.layers, c.pages, c.heads, c.page_size, c.head_dim) == (1, 6, 2, 16, 64)
    for a, b, what in ((k, k[:5], "must be"), (k[0], k[0], "must be"), (k.float(), k.float(), "bf16"),
                       (k, k.half(), "bf16"), (k.transpose(2, 3), k.transpose(2, 3), "contiguous")):
        with pytest.raises(krlib.KrbError, match=what):
            krlib.KVCache(a, b)


def test_wrapper_refusals(krlib):
    import torch
    c = _cpu_cache(krlib)
    bf = torch.bfloat16
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    qkv, pos = torch.zeros(3, 8 * 64, dtype=bf), torch.zeros(3, dtype=torch.int64)
    tab = torch.zeros(9, 64, dtype=bf)
    good = dict(qkv=qkv, positions=pos, slots=pos, HQ=4, cos=tab, sin=tab)
    for over, what in ((dict(qkv=qkv.half()), "qkv"), (dict(qkv=qkv[:, :-64]), "HKV"),
                       (dict(positions=pos.int()), "positions"), (dict(slots=pos[:2]), "slots"),
                       (dict(cos=tab.float()), "cos"), (dict(sin=tab[:5]), "cos and sin"),
                       (dict(cos=tab[:, :32], sin=tab[:, :32]), "cos and sin"),
                       (dict(q_norm=tab[0][:32]), "q_norm"), (dict(out=qkv[:, :64]), "out"),
                       (dict(status=pos), "status")):
        with pytest.raises(krlib.KrbError, match=what):
            krlib.qk_norm_rope_paged(**{**good, "cache": c, **over})
    q = torch.zeros(3, 4 * 64, dtype=bf)
    c._workspaces[4, 1] = 64  # asked of the device elsewhere
    good = dict(q=q, page_table=i32(2, 4), kv_lens=i32(2), q_starts=i32(3), max_q=1, scale=0.1)
    for over, what in ((dict(q=q.half()), "q must"), (dict(q=q[:, :-1]), "head_dim"),
                       (dict(page_table=i32(2, 4).long()), "page_table"), (dict(q_starts=i32(2)), "batch"),
                       (dict(page_table=i32(1, 4)), "batch"), (dict(mask=i32(2, 1)), "mask"),
                       (dict(mask=i32(3, 1).long()), "mask"), (dict(out=q[:2]), "out"),
                       (dict(workspace=i32(9)), "workspace")):
        with pytest.raises(krlib.KrbError, match=what):
            krlib.attention_paged(**{**good, "cache": c, **over})
    good = dict(page_table=i32(2, 4), bases=i32(2), accepted=i32(2, 3), counts=i32(2))
    for over, what in ((dict(bases=i32(3)), "batch"), (dict(counts=i32(2).long()), "counts"),
                       (dict(accepted=i32(3, 3)), "batch"), (dict(page_table=i32(4)), "page_table")):
        with pytest.raises(krlib.KrbError, match=what):
            krlib.kv_commit(c, **{**good, **over})
    with pytest.raises(krlib.KrbError, match="length"):
        krlib.kv_copy_pages(c, [1, 2], [3])
    for bad in (1.5, 2 ** 32 + 1, "1", None):
        with pytest.raises(krlib.KrbError, match="host integers"):
            krlib.kv_copy_pages(c, [bad], [3])
    with pytest.raises(krlib.KrbError, match="not on a GPU"):
        krlib.kv_copy_pages(c, [1], [3])


@pytest.fixture
def copied(krlib, monkeypatch):
    """What kv_copy_pages hands to the library: (src, dst), n entries of each."""
    calls = []

    class Fake:
        def krb_kv_copy_pages(self, cache, src, dst, n, stream):
            calls.append(tuple(list((ctypes.c_int * n).from_address(x)) if n else [] for x in (src, dst)))
            return 0

    monkeypatch.setattr(krlib, "_enter", lambda cache: None)
    monkeypatch.setattr(krlib, "_raw_stream", lambda stream, index: None)
    monkeypatch.setattr(krlib, "lib", lambda: Fake())
    return calls


def test_copy_page_lists_of_every_kind(krlib, copied):
    """Every host sequence of integers means its elements: bytes are page numbers up to 255, not memory
    of four-byte entries."""
    from array import array

    import numpy as np
    import torch
    c = _cpu_cache(krlib)
    kinds = [bytes, bytearray, memoryview, list, tuple, np.array, torch.tensor,
             lambda x: array("q", x), lambda x: array("B", x), lambda x: np.array(x, dtype=np.uint8),
             lambda x: range(x[0], x[-1] + 1)]
    for kind in kinds:
        values = [5, 6, 7, 8] if kind is kinds[-1] else [5, 0, 0, 1]
        held = bytes(values) if kind is memoryview else values
        copied.clear()
        krlib.kv_copy_pages(c, kind(held), kind(held))
        assert copied == [(values, values)], kind
    copied.clear()
    krlib.kv_copy_pages(c, b"\x05\x01\x02", (1, 2, 3))  # no multiple of four long
    assert copied == [([5, 1, 2], [1, 2, 3])]


def test_copy_page_lists_whose_length_lies(krlib, copied):
    class Short(list):
        def __len__(self):
            return 9

    class Long:
        def __len__(self):
            return 1

        def tolist(self):
            return [1, 2, 3]

    c = _cpu_cache(krlib)
    for x in (Short([1, 2]), Long()):
        with pytest.raises(krlib.KrbError, match="flat sequences"):
            krlib.kv_copy_pages(c, x, x)
    assert copied == []


# ---------------------------------------------------------------- the kernels' error paths
def _blocks(text, head):
    """Spans of the brace blocks that `head` opens."""
    at = 0
    while (at := text.find(head, at)) >= 0:
        depth, end = 1, at + len(head)
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield at, end
        at += 1


def bare_waits(text):
    """Calls of mbar_wait whose outcome steers code that a whole warp runs."""
    import re
    text = re.sub(r"//[^\n]*", "", text)
    single = list(_blocks(text, "if (lane == 0) {"))
    found = []
    for m in re.finditer(r"\bmbar_wait\(", text):
        used = re.search(r"(return|[=(!&|,])\s*$", text[:m.start()])
        if used and not any(a < m.start() < b for a, b in single):
            found.append(text[m.start():text.index(";", m.start())])
    return found


def test_a_warp_leaves_its_waits_together():
    """A wait that runs out does so lane by lane.  Where a warp goes on to votes, barriers or
    tensor-memory accesses, its lanes decide together (mbar_wait_warp): one that left alone would
    leave the others waiting for good.  (A wait cannot be made to run out on a GPU without a kernel
    that is broken for it; the sources are what can be checked.)"""
    from pathlib import Path
    csrc = Path(__file__).resolve().parents[1] / "kernrelay_b200" / "csrc"
    assert bare_waits("ok = mbar_wait(&a[b], 1, n);  // x\nif (ok) {}") == ["mbar_wait(&a[b], 1, n)"]
    assert not bare_waits("if (lane == 0) { ok = mbar_wait(a, 1, n); }  for (;;) mbar_wait(a, 1, n);")
    for name in ("attention_paged.cu", "attention_paged_tc.cu"):
        text = (csrc / name).read_text()
        assert bare_waits(text) == [], name
        for a, b in _blocks(text, "if (lane == 0) {"):
            assert "mbar_wait_warp" not in text[a:b]
    head = (csrc / "attention_paged.cuh").read_text()
    assert "return __all_sync(0xffffffffu, mbar_wait(bar, parity, kMbarLimitNs));" in head
    assert len(bare_waits(head)) == 1


# ---------------------------------------------------------------- outputs over inputs
W, W3 = 28 * 128, 36 * 128  # q's columns, and qkv's, of the calls above


@pytest.mark.parametrize("at,ldo,N,free", [
    (0, W, 3, False), (0, W, 1, False), (8, W, 1, False), (W - 8, W, 1, False), (W, W, 1, True),
    (2 * W, W, 3, False), (3 * W, W, 3, True), (-3 * W, W, 3, True), (-3 * W + 8, W, 3, False),
    (-W, W, 1, True), (W, 3 * W, 3, False), (2 * W, 2 * W + 8, 3, False), (-W, W + 8, 2, False),
])
def test_attention_output_over_q(krlib, at, ldo, N, free):
    """Rows of q (dense, at 1 << 30) and out at every way of touching.  No workspace is given, so that
    what is not refused for its overlap is refused behind it."""
    d, base = _desc(krlib), 1 << 30
    rc = krlib.lib().krb_attention_paged(
        ctypes.addressof(d), 0, base, W, base + 2 * at, ldo, N, 28, 16, 8, 8, 16, 16, 2, 1, None, 0, 0,
        0.1, None, 0, None, None)
    assert rc == 1
    assert ("out overlaps q" in _message(krlib)) == (not free)


@pytest.mark.parametrize("at,lda,ldo,free", [
    (W, 2 * W, 2 * W, True), (W - 8, 2 * W, 2 * W, False), (W + 8, 2 * W, 2 * W, False),
    (W + 8, 2 * W + 8, 2 * W + 8, True), (-W, 2 * W, 2 * W, True), (W, 4 * W, 2 * W, True),
    (W, 4 * W, 2 * W + 8, False), (3 * W, 4 * W, 4 * W, True), (3 * W + 8, 4 * W, 4 * W, False),
])
def test_attention_output_beside_q(krlib, at, lda, ldo, free):
    """Columns of one buffer: rows that lie between each other without sharing an element are taken."""
    d, base = _desc(krlib), 1 << 30
    rc = krlib.lib().krb_attention_paged(
        ctypes.addressof(d), 0, base, lda, base + 2 * at, ldo, 50, 28, 16, 8, 8, 16, 16, 2, 1, None, 0, 0,
        0.1, None, 0, None, None)
    assert rc == 1
    assert ("out overlaps q" in _message(krlib)) == (not free)
    brute = any(abs(at + j * ldo - i * lda) < W for i in range(50) for j in range(50))
    assert brute == (not free)


@pytest.mark.parametrize("at,ldq,N", [(8, W3, 3), (0, W, 3), (W, W3, 3), (8 * 128, W, 2), (W3 - 8, W, 1),
                                      (-8, W, 1), (-3 * W + 8, W, 3)])
def test_append_output_over_qkv(krlib, at, ldq, N):
    d, base = _desc(krlib), 1 << 30
    rc = krlib.lib().krb_qk_norm_rope_paged(
        ctypes.addressof(d), 0, base, W3, base + 2 * at, ldq, 16, 16, N, 28, 16, 16, 8, None, None, 1e-6,
        None, None)
    assert rc == 1 and "overlaps qkv" in _message(krlib)


def test_attention_of_a_step_without_tokens(krlib):
    """No rows or no sequences: nothing is done, and max_q, a bound of nothing, may be 0."""
    d = ctypes.addressof(keep := _desc(krlib))
    L = krlib.lib()
    for N, B in ((0, 2), (3, 0), (0, 0)):
        assert L.krb_attention_paged(d, 0, None, 0, None, 0, N, 28, None, 0, 0, None, None, B, 0, None, 0,
                                     0, 0.1, None, 0, None, None) == 0
        assert L.krb_attention_paged(d, 0, None, 0, None, 0, N, 28, None, 0, 0, None, None, B, -1, None, 0,
                                     0, 0.1, None, 0, None, None) == 1 and "max_q" in _message(krlib)
    del keep


def test_masks_and_status_without_elements(krlib):
    """A mask of no words is no mask's absence, and a status of no entries reports nothing: refused."""
    import torch
    c = _cpu_cache(krlib)
    c._workspaces[4, 1] = 64
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    q, pos = torch.zeros(3, 4 * 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    good = dict(q=q, cache=c, page_table=i32(2, 4), kv_lens=i32(2), q_starts=i32(3), max_q=1, scale=0.1)
    with pytest.raises(krlib.KrbError, match="mask must have words"):
        krlib.attention_paged(**good, mask=i32(3, 0))
    tab = torch.zeros(9, 64, dtype=torch.bfloat16)
    for call in (lambda **kw: krlib.attention_paged(**good, **kw),
                 lambda **kw: krlib.qk_norm_rope_paged(torch.zeros(3, 8 * 64, dtype=q.dtype), c, pos, pos, 4,
                                                       tab, tab, **kw),
                 lambda **kw: krlib.kv_commit(c, i32(2, 4), i32(2), i32(2, 3), i32(2), **kw)):
        with pytest.raises(krlib.KrbError, match="status"):
            call(status=i32(0))
        with pytest.raises(krlib.KrbError, match="not on a GPU"):
            call(status=i32(1))


def test_index_arrays_between_their_elements(krlib):
    """Addresses that an index array cannot have: refused, where the kernels would fault on them."""
    L, d = krlib.lib(), ctypes.addressof(keep := _desc(krlib))
    base = 1 << 30

    def append(pos=64, slots=64, status=None):
        return L.krb_qk_norm_rope_paged(d, 0, base, W3, 16, W, pos, slots, 3, 28, 16, 16, 8, None, None, 1e-6,
                                        status, None)

    def attention(table=64, lens=64, starts=64, mask=None, status=None):
        return L.krb_attention_paged(d, 0, base, W, 16, W, 3, 28, table, 8, 8, lens, starts, 2, 1, mask, 1, 1,
                                     0.1, None, 0, status, None)

    def commit(table=64, bases=64, acc=64, counts=64, status=None):
        return L.krb_kv_commit(d, table, 8, 8, bases, acc, 4, 4, counts, 2, status, None)

    for call, size, names in ((append, 8, ("pos", "slots")), (append, 4, ("status",)),
                              (attention, 4, ("table", "lens", "starts", "mask", "status")),
                              (commit, 4, ("table", "bases", "acc", "counts", "status"))):
        for name in names:
            for off in (1, 2, size - 1, size // 2):
                assert call(**{name: 64 + off}) == 1, name
                assert f"{size}-byte aligned" in _message(krlib), name
    del keep


@pytest.mark.parametrize("layer", [-1, 2, 2 ** 32, 2 ** 32 + 1, -2 ** 32])
def test_layers_outside_the_cache(krlib, layer):
    """Refused as they are, not modulo 2^32."""
    import torch
    c = _cpu_cache(krlib)
    c._workspaces[4, 1] = 64
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    q, pos = torch.zeros(3, 4 * 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    tab = torch.zeros(9, 64, dtype=torch.bfloat16)
    with pytest.raises(krlib.KrbError, match="no such layer"):
        krlib.attention_paged(q, c, i32(2, 4), i32(2), i32(3), 1, 0.1, layer=layer)
    with pytest.raises(krlib.KrbError, match="no such layer"):
        krlib.qk_norm_rope_paged(torch.zeros(3, 8 * 64, dtype=q.dtype), c, pos, pos, 4, tab, tab, layer=layer)


@pytest.mark.parametrize("max_q", [-1, 2 ** 31, 2 ** 32 + 1, 2 ** 32])
def test_max_q_outside_an_int(krlib, max_q):
    with pytest.raises(krlib.KrbError, match="max_q"):
        _cpu_cache(krlib).attention_workspace(4, max_q)
