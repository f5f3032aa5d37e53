"""Attention behind a shared prefix (csrc/attention_shared.hip), rules on logits (csrc/logits.hip) and log-probabilities of tokens
(csrc/logprobs.hip): the CPU definitions and the GPU kernels against plain forms in 64 bits, their refusals, and a decode step of several
completions of one prompt that runs them together.

Tolerances count roundings. Attention: each weight is rounded to bf16 once (at most 2^-8 of it) where it meets its value and once in
the sum, and the result once; with A = sum_j p_j |v_j| that is at most 2^-8 (2 A + |o|) <= 3 * 2^-8 A, and 2^-10 A are left for the
fp32 products of scores (128 products of numbers around 1 and their sum: 2^-24 * 128 * 4 in a score, far below). fp32 results:
each operation 2^-24 of its terms."""
import math
import pathlib
import re

import pytest
import torch

from llmss_amd import ops
from llmss_amd.ops import reference as ref

F64 = torch.float64
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


# ------------------------------------------------------------------------------------------------------------- attention
def _case(dev, nh, nkv, D, prefix, owns, qlens=None, bs=16, fp8=False, seed=0, spare=3, own_cols=None, poison=True):
    """Caches whose unused places hold NaN, tables with -1 behind a row's pages, sequences of ``owns`` positions behind the prefix
    (negative: the context ends inside the prefix; None: idle)."""
    g = torch.Generator().manual_seed(seed)
    B = len(owns)
    qlens = qlens or [1] * B
    pp = -(-prefix // bs)
    op = [-(-max(o or 0, 0) // bs) for o in owns]
    cols = own_cols or max(1, max(op))
    nb = pp + sum(op) + spare
    k = torch.full((nb, nkv, bs, D), float("nan") if poison else 0.0)
    v = torch.full((nb, nkv, bs, D), float("nan") if poison else 0.0)
    perm = torch.randperm(nb, generator=g).to(torch.int32)
    ptab, at = perm[:pp].clone(), pp
    bt = torch.full((B, cols), -1, dtype=torch.int32)
    fill = [(ptab, prefix)]
    for b in range(B):
        bt[b, :op[b]] = perm[at:at + op[b]]
        at += op[b]
        fill.append((bt[b], max(owns[b] or 0, 0)))
    for tab, n in fill:
        for j in range(n):
            k[tab[j // bs], :, j % bs] = torch.randn(nkv, D, generator=g)
            v[tab[j // bs], :, j % bs] = torch.randn(nkv, D, generator=g)
    if fp8:
        bad = k.isnan()
        kc, vc = ref.kv_rows_quant(torch.nan_to_num(k)), ref.kv_rows_quant(torch.nan_to_num(v))
        if poison:
            kc[bad[..., 0]] = 0xFF  # e4m3 and fp32 NaN
            vc[bad[..., 0]] = 0xFF
    else:
        kc, vc = k.bfloat16(), v.bfloat16()
    T = sum(qlens)
    q = (torch.randn(T, (nh + 2 * nkv) * D, generator=g) * 1.5).bfloat16()
    ctx = torch.tensor([0 if o is None else prefix + o for o in owns], dtype=torch.int32)
    cu = torch.tensor([0] + torch.tensor(qlens).cumsum(0).tolist(), dtype=torch.int32)
    return dict(q=q.to(dev), k=kc.to(dev), v=vc.to(dev), ptab=ptab.to(dev), prefix=prefix, bt=bt.to(dev), ctx=ctx.to(dev),
                cu=cu.to(dev), qlens=qlens, nh=nh, nkv=nkv, D=D, bs=bs, scale=1 / math.sqrt(D))


def _run(c, **kw):
    several = max(c["qlens"]) > 1
    kw.setdefault("cu_q", c["cu"] if several else None)
    kw.setdefault("max_qlen", max(c["qlens"]))
    return ops.attn_shared(c["q"], c["k"], c["v"], c["ptab"], c["prefix"], c["bt"], c["ctx"], c["nh"], c["nkv"], c["D"], c["scale"], **kw)


def _plain(c, dev="cpu"):
    """In 64 bits, a row at a time: (result, A = sum p |v|)."""
    c = {n: x.to(dev if n in "qkv" else "cpu") if torch.is_tensor(x) else x for n, x in c.items()}
    nh, nkv, D, bs, P = c["nh"], c["nkv"], c["D"], c["bs"], c["prefix"]
    T = c["q"].shape[0]
    out, A = torch.zeros(T, nh, D, dtype=F64, device=dev), torch.zeros(T, nh, D, dtype=F64, device=dev)
    t = 0
    for b, n in enumerate(c["qlens"]):
        for i in range(n):
            see = min(max(int(c["ctx"][b]) - n + i + 1, 0), P + c["bt"].shape[1] * bs)
            page = [int(c["ptab"][j // bs]) if j < P else int(c["bt"][b, (j - P) // bs]) for j in range(see)]
            at = [j % bs if j < P else (j - P) % bs for j in range(see)]
            if see:
                kk, vv = c["k"][page, :, at], c["v"][page, :, at]
                if c["k"].dtype == torch.uint8:
                    kk, vv = (x[..., :D].contiguous().view(torch.float8_e4m3fn).to(F64)
                              * x[..., D:D + 4].contiguous().view(torch.float32).to(F64) for x in (kk, vv))
                kk, vv = (x.to(F64).repeat_interleave(nh // nkv, 1) for x in (kk, vv))
                w = torch.softmax((c["q"][t, :nh * D].view(nh, D).to(F64)[None] * kk).sum(-1) * c["scale"], 0)
                out[t] = (w[..., None] * vv).sum(0)
                A[t] = (w[..., None] * vv.abs()).sum(0)
            t += 1
    return out.view(T, -1).cpu(), A.view(T, -1).cpu()


def _near(got, c, rows=None, dev="cpu"):
    want, A = _plain(c, dev)
    got = got.cpu().to(F64)
    if rows is not None:
        got, want, A = got[rows], want[rows], A[rows]
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / (A * (3 * 2.0 ** -8 + 2.0 ** -10) + 1e-30)).max()
    assert worst <= 1, f"{float(worst)} of what the roundings allow"


HEADS = [(4, 4, 64), (8, 2, 128), (3, 1, 128), (2, 2, 256), (20, 1, 64), (6, 2, 256), (48, 1, 128)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("nh,nkv,D", HEADS)
def test_attention_of_single_tokens(dev, nh, nkv, D, fp8):
    # an own part of its new token alone, one that fills pages, one that ends inside; an idle row; a prefix that ends inside a page
    c = _case(dev, nh, nkv, D, 101, [1, 32, 45, None, 17, 130], fp8=fp8)
    _near(_run(c), c)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("nh,nkv,D", HEADS)
def test_attention_of_several_tokens(dev, nh, nkv, D, fp8):
    c = _case(dev, nh, nkv, D, 77, [5, 40, 33, 70], qlens=[5, 1, 3, 70], fp8=fp8, seed=1)
    _near(_run(c), c)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 64, 65, 127, 129, 700])
@pytest.mark.parametrize("rows", [1, 2, 17])
def test_attention_lengths(dev, prefix, rows):
    c = _case(dev, 4, 2, 64, prefix, [1 + (7 * i) % 50 for i in range(rows)], seed=prefix)
    _near(_run(c), c)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("bs", [1, 5, 8, 32, 48])
def test_attention_page_sizes(dev, bs):
    for fp8 in (False, True):
        c = _case(dev, 4, 2, 128, 150, [1, 20, 37], bs=bs, fp8=fp8, seed=bs)
        _near(_run(c), c)
        c = _case(dev, 4, 2, 128, 90, [21, 20, 37], qlens=[21, 4, 30], bs=bs, fp8=fp8, seed=bs)
        _near(_run(c), c)


@pytest.mark.parametrize("dev", DEVICES)
def test_contexts_that_end_inside_the_prefix(dev):
    c = _case(dev, 8, 2, 64, 90, [-30, 4, -90, -89, 0, -1], seed=3)
    got = _run(c)
    _near(got, c)
    assert (got[2] == 0).all()
    c = _case(dev, 8, 2, 64, 90, [-30, 4, -85, 12], qlens=[7, 9, 9, 12], seed=4)  # (the third has rows before the first position)
    got = _run(c)
    _near(got, c)
    assert (got[16:20] == 0).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see_may_be_anything(dev, fp8, value):
    """A later position of the same portion, or of the prefix, holds keys and values that are not finite: the rows that do not see it
    keep their results, the others get what the formula gives."""
    if fp8 and math.isinf(value):
        pytest.skip("e4m3 has no infinities")
    c = _case(dev, 4, 2, 128, 70, [20, -10, 3], qlens=[20, 2, 3], fp8=fp8, seed=5)
    want = _run(c)
    bs = c["bs"]
    for tab, j in ((c["bt"][0], 12), (c["ptab"], 65)):
        for cache in (c["k"], c["v"]):
            if cache is c["k"] and not math.isnan(value):
                continue
            if fp8:
                cache[tab[j // bs], :, j % bs, 5] = 0x7F
            else:
                cache[tab[j // bs], :, j % bs, 5] = value
    got = _run(c)
    # rows 0 .. 19 see prefix position 65: poisoned in the prefix. The second sequence's context ends at 60
    assert torch.equal(got[20:22], want[20:22])
    c = _case(dev, 4, 2, 128, 70, [20, -10, 3], qlens=[20, 2, 3], fp8=fp8, seed=5)
    for cache in (c["v"],):
        cache[c["bt"][0][0], :, 12, 5] = 0x7F if fp8 else value
    got = _run(c).view(25, 4, 128)
    want = want.view(25, 4, 128)
    assert torch.equal(got[:12], want[:12]) and torch.equal(got[20:], want[20:])
    seen = got[12:20, :, 5].float()
    assert seen.isnan().all() if math.isnan(value) else (seen == value).all()
    rest = torch.ones(128, dtype=torch.bool)
    rest[5] = False
    assert torch.isfinite(got[12:20][..., rest.to(got.device)].float()).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_of_no_sequence_stay(dev):
    c = _case(dev, 4, 2, 64, 40, [3, 30, 1], qlens=[3, 2, 1], seed=6)
    q = torch.cat([c["q"], torch.full_like(c["q"][:5], float("nan"))])
    out = torch.full((q.shape[0] + 2, 4 * 64 + 8), 7.0, dtype=torch.bfloat16, device=dev)
    c2 = dict(c, q=q)
    got = _run(c2, out=out)
    _near(got[:6, :256], c)
    assert (out[6:] == 7).all() and (out[:, 256:] == 7).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_empty_portions_and_hints_that_are_too_small(dev):
    c = _case(dev, 4, 1, 64, 50, [30, 0, 200, 9], qlens=[30, 0, 140, 9], seed=7)
    _near(_run(c), c)
    _near(_run(c, max_qlen=1, max_own=1), c)
    c = _case(dev, 4, 1, 64, 50, [30, 1, 400, 9], seed=8)
    _near(_run(c, max_own=0), c)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("G", [1, 20])
def test_rows_in_front_of_the_first_sequence_stay_and_contexts_end_with_the_table(dev, G):
    c = _case(dev, 2 * G, 2, 64, 40, [3, 30, 48], qlens=[3, 2, 1], seed=18)
    want = _run(c)
    q = torch.cat([torch.full_like(c["q"][:2], float("nan")), c["q"]])
    out = torch.full((8, 2 * G * 64), 7.0, dtype=torch.bfloat16, device=dev)
    ctx = c["ctx"].clone()
    ctx[2] += 1000  # (its table holds 48 positions; the others' rows must not move)
    _run(dict(c, q=q, ctx=ctx), cu_q=c["cu"] + 2, out=out)
    assert (out[:2] == 7).all()
    _near(out[2:7], dict(c, q=q[2:7], qlens=[3, 2]))
    assert torch.equal(out[7], want[5])


@pytest.mark.parametrize("dev", DEVICES)
def test_strided_operands(dev):
    c = _case(dev, 4, 2, 64, 33, [3, 30, 18], seed=9)
    want = _run(c)
    wide = torch.zeros(3, 2 * c["q"].shape[1], dtype=torch.bfloat16, device=dev)
    wide[:, 64:64 + c["q"].shape[1]] = c["q"]
    tables = torch.zeros(3, 9, dtype=torch.int32, device=dev)
    tables[:, 4:4 + c["bt"].shape[1]] = c["bt"]
    got = _run(dict(c, q=wide[:, 64:], bt=tables[:, 4:4 + c["bt"].shape[1]]))
    assert torch.equal(got, want)


def test_loads_into_lds_by_assembly_say_what_they_change():
    """The compiler sees into no string: a statement that writes m0 names it as changed, and a memory instruction in it takes its scalar
    address from a move of the same statement (the compiler keeps the distance from a vector write of it for its own instructions only)."""
    csrc = pathlib.Path(ops.__file__).parents[1] / "csrc"
    found = 0
    for f in sorted(csrc.glob("*.hip")) + sorted(csrc.glob("*.h")):
        for code, rest in re.findall(r'asm volatile\(("(?:[^"\\]|\\.)*")\s*:(.*?)\);', f.read_text(), re.S):
            if "global_load_lds" in code:
                found += 1
                outputs = len(re.findall(r'"[=+]', rest))
                base = re.search(r"global_load_lds\w+ %\d, (?:%(\d)|off)", code)
                assert base, code
                assert base[1] is None or int(base[1]) < outputs, f"{f.name}: {code}"
            assert not re.search(r"\w m0,", code) or '"m0"' in rest, f"{f.name}: {code}"
    assert found >= 2


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nh,nkv,owns,qlens", [
    (8, 2, [40, 30], [1, 1]), (8, 2, [40, 30, 9], [9, 30, 1]), (8, 8, [1 + i % 40 for i in range(70)], [1] * 70),
    (24, 8, [9 + i % 40 for i in range(70)], [1 + i % 5 for i in range(70)])])
def test_attention_in_place_and_beside_its_queries(dev, nh, nkv, owns, qlens):
    c = _case(dev, nh, nkv, 128, 300, owns, qlens=qlens, seed=27, own_cols=9)
    want = _run(c)
    q = c["q"].clone()
    assert torch.equal(_run(c, out=c["q"])[:, :nh * 128], want) and torch.equal(c["q"][:, nh * 128:], q[:, nh * 128:])
    c["q"].copy_(q)
    beside = torch.zeros(q.shape[0], 2 * nh * 128, dtype=torch.bfloat16, device=dev)
    beside[:, nh * 128:] = q[:, :nh * 128]
    assert torch.equal(_run(dict(c, q=beside[:, nh * 128:]), out=beside[:, :nh * 128]), want)
    assert torch.equal(beside[:, nh * 128:], q[:, :nh * 128])


@pytest.mark.parametrize("dev", DEVICES)
def test_attention_refuses_a_result_that_overlaps_its_queries_otherwise(dev):
    c = _case(dev, 4, 2, 64, 33, [3, 30, 18])
    wide = c["q"].shape[1]
    flat = torch.zeros(8 * wide, dtype=torch.bfloat16, device=dev)
    for q, out in ((flat[:3 * wide].view(3, wide), flat[8:8 + 3 * wide].view(3, wide)),
                   (flat.view(8, wide)[:3], flat.view(8, wide)[1:4]),
                   (flat.view(8, wide)[:3], flat[:3 * 256].view(3, 256)),
                   (flat.view(8, wide)[:3, 248:], flat.view(8, wide)[:3])):
        with pytest.raises(ValueError, match="out"):
            _run(dict(c, q=q), out=out)


def _many(B, several):
    """Own parts and portions of B sequences: idle ones, contexts that end in the prefix, one token to some pages."""
    owns = [(1, 20, 37, None, -30, 90, 64, 16, 33, 5)[i % 10] for i in range(B)]
    qlens = [1] * B if not several else [min(1 + i % several, max(1, o or 0)) for i, o in enumerate(owns)]
    return owns, qlens


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("nh,several,bs", [(8, 0, 16), (16, 0, 5), (24, 3, 16), (16, 7, 48)])
def test_many_sequences_of_several_key_heads(fp8, nh, several, bs):
    """640 (sequence, key head) pairs: own parts in a launch that joins the prefix's results."""
    owns, qlens = _many(80, several)
    c = _case("cuda", nh, 8, 128, 200, owns, qlens=qlens, bs=bs, fp8=fp8, seed=19)
    _near(_run(c), c, dev="cuda")
    if several:
        _near(_run(c, max_qlen=1), c, dev="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,D,several,parts", [(256, 32, 128, 0, 3), (256, 32, 128, 4, 3), (256, 32, 64, 0, 2)])
def test_many_rows_of_many_heads(nh, nkv, D, several, parts):
    """Enough rows that each wave takes two groups of them (heads of 128; single tokens: the prefix in two runs, own parts in one)."""
    from llmss_amd.ops import hip

    owns, qlens = _many(100, several)
    c = _case("cuda", nh, nkv, D, 2400, owns, qlens=qlens, seed=20)
    q = c["q"].shape[0]
    assert several or hip.lib().attn_shared_parts(q, 100, nh, nkv, D, 2400, 1, c["bt"].shape[1] * 16, False) == parts
    _near(_run(c), c, dev="cuda")


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("qlens", [[1, 1, 1], [3, 1, 5]])
def test_tables_without_pages(dev, qlens):
    """Every context lies within the prefix (tables of no columns), or nothing is shared (a prefix of no pages)."""
    for nh, D in ((4, 64), (2, 256), (32, 128)):
        c = _case(dev, nh, 2, D, 90, [0, -5, -60], qlens=qlens, seed=12)
        c["bt"] = c["bt"][:, :0]
        _near(_run(c), c)
        _near(_run(c, max_own=0), c)
        c = _case(dev, nh, 2, D, 0, [9, 70, 33], qlens=qlens, seed=13)
        assert c["ptab"].numel() == 0
        _near(_run(c), c)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nh,nkv,D,fp8", [(2, 1, 128, False), (16, 1, 64, True), (2, 2, 256, False)])
def test_long_contexts_of_few_rows(dev, nh, nkv, D, fp8):
    """Many partial results a row: a prefix of a few thousand positions, and own parts as long."""
    for owns, qlens in (([1], [1]), ([2900, 40], [1, 1]), ([2300], [20])):
        c = _case(dev, nh, nkv, D, 3500, owns, qlens=qlens, fp8=fp8, seed=14)
        _near(_run(c), c)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(dev, sign):
    """Products of +-2^112 beside each other: all keys are the same, so every weight is, and the result is the mean of the values."""
    for qlens in ([1, 1], [1, 30]):
        c = _case(dev, 8, 2, 64, 50, [20, 30], qlens=qlens, seed=15)
        c["q"][:] = sign * 2.0 ** 53
        c["k"][:] = 2.0 ** 53
        _near(_run(c), c)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("size", [20, 24, 32, 40, 60, 100])
@pytest.mark.parametrize("nh,nkv,D,owns,qlens", [
    (8, 2, 128, [40, 30], [1, 1]),            # the whole batch by keys, two parts
    (8, 2, 128, [40, 30, 9], [9, 30, 1]),     # by rows
    (48, 1, 128, [40, 30, 70], [1, 1, 1]),
    (4, 4, 64, [40, 30, 70], [9, 30, 1]),
    (2, 2, 256, [40, 30, 70], [9, 30, 1]),
    (8, 8, 128, [1 + i % 40 for i in range(70)], [1] * 70),  # the prefix by rows, own parts by keys
])
def test_large_scores_that_differ(dev, fp8, size, nh, nkv, D, owns, qlens):
    """Scores of some 2^(size + 3) that are no powers of two and lie far apart: the largest takes all, whatever the rounding of its
    exponent is by itself. With these seeds the largest is ahead by 2^-15.3 of sum |q k| and more (heads of 256 2^-13.3), and two sums
    of D products in 32 bits are off by 2 D 2^-24 of it at most (2^-16, 2^-15): what is left, at a sum of 2^27 from the smallest size on,
    is an exponent of 100."""
    c = _case(dev, nh, nkv, D, 600, owns, qlens=qlens, fp8=fp8, seed=23 if fp8 else 22)
    c["q"] = (c["q"].float() * 2.0 ** size).bfloat16()
    want, A = _plain(c)  # (one key's value, as it is)
    assert ((want.abs() - A).abs() <= 2.0 ** -30 * A).all()
    _near(_run(c), c)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [24, 40])
def test_large_scores_of_many_rows_of_many_heads(size):
    """The same where a wave takes two groups of rows: a key head's queries are one direction times powers of two, so that its keys are in one
    order. The largest is ahead by 2^-9.9 of sum |q k| with this seed (the sums are off by 2^-16 of it)."""
    owns, qlens = _many(100, 0)
    c = _case("cuda", 256, 32, 128, 2400, owns, qlens=qlens, seed=24)
    g = torch.Generator().manual_seed(24)
    lean = torch.randn(1, 32, 1, 128, generator=g) * 1.5
    c["q"] = (lean * 2.0 ** (size + torch.randint(0, 4, (100, 32, 8, 1), generator=g))).reshape(100, -1).bfloat16().cuda()
    want, A = _plain(c, "cuda")
    assert ((want.abs() - A).abs() <= 2.0 ** -30 * A).all()
    _near(_run(c), c, dev="cuda")


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("nh,nkv,D,owns,qlens", [
    (8, 2, 128, [40, 30], [1, 1]), (8, 2, 128, [40, 30, 9], [9, 30, 1]), (2, 2, 256, [40, 30, 9], [9, 30, 1]),
    (48, 1, 64, [400, 30, -20], [1, 1, 1]), (8, 8, 128, [1 + i % 40 for i in range(70)], [1] * 70)])
def test_keys_of_minus_infinity(dev, nh, nkv, D, owns, qlens):
    """Keys whose scores are -infinity weigh nothing; a row that sees no others has no softmax, and NaN in its result, not the zeros of
    a row that sees nothing."""
    c = _case(dev, nh, nkv, D, 600, owns, qlens=qlens, seed=26)
    c["q"][:, 3].abs_().clamp_(min=1.0)
    for h in range(nh):
        c["q"][:, h * D + 3] = c["q"][:, 3]
    j = torch.arange(600)
    c["k"][c["ptab"].long()[j // 16], :, (j % 16).to(dev), 3] = torch.where(j % 3 > 0, float("-inf"), 1.0).bfloat16().to(dev)[:, None]
    _near(_run(c), c)
    c["k"][..., 3] = float("-inf")
    assert _run(c).isnan().all()
    c["ctx"][1] = 0
    at = sum(qlens[:1])
    got = _run(c)
    assert (got[at:at + qlens[1]] == 0).all() and got[:at].isnan().all() and got[at + qlens[1]:].isnan().all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("qlens", [[1, 1, 1], [3, 20, 5]])
def test_fp8_rows_of_zeros_and_of_any_scale(dev, qlens):
    """A row whose scale is 0 has its weight all the same; scales from 1e-20 to 1e20 beside each other."""
    c = _case(dev, 8, 2, 128, 70, [5, 30, 40], qlens=qlens, fp8=True, seed=21, poison=False)
    for j, scale in ((3, 0.0), (40, 0.0), (50, 1e-20), (60, 1e20), (66, 1e-37)):
        row = c["v"][c["ptab"][j // 16], :, j % 16]
        if scale == 0:
            row[:, :128] = 0
        row[:, 128:132] = torch.tensor([scale]).view(torch.uint8).to(dev)
    _near(_run(c), c)


@pytest.mark.gpu
@pytest.mark.parametrize("qlens", [[1, 1, 1], [4, 20, 3]])
def test_a_cache_of_more_than_four_gigabytes(qlens):
    """Pages at both ends of a cache whose rows lie more than 2^32 bytes apart give what the same rows give in a small one."""
    c = _case("cuda", 8, 2, 128, 100, [4, 50, 33], qlens=qlens, seed=16)
    want = _run(c)
    small = c["k"].shape[0]
    nb = 540000  # of 8 KiB each
    k, v = (torch.empty(nb, 2, 16, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    to = torch.arange(small, device="cuda")
    to[1::2] = nb - 1 - to[1::2]
    k[to], v[to] = c["k"], c["v"]
    far = lambda t: torch.where(t >= 0, to[t.clamp(min=0).long()], t.long()).int()  # noqa: E731
    assert torch.equal(_run(dict(c, k=k, v=v, ptab=far(c["ptab"]), bt=far(c["bt"]))), want)


@pytest.mark.gpu
def test_rows_of_logits_past_32_bits():
    """The last rows of logits that lie 2^32 bytes and more behind the first, and the same mask row for all."""
    B, V = 40, 50000
    buf = torch.empty(B, 1 << 25, dtype=torch.float32, device="cuda")
    x = buf[:, :V]
    x.copy_(torch.randn(B, V, generator=torch.Generator().manual_seed(3)))
    mask = torch.full((1, (V + 31) // 32), 0x55555555, dtype=torch.int32, device="cuda")
    rows = torch.zeros(B, dtype=torch.int32, device="cuda")
    ids = torch.full((B, 2), V - 1, device="cuda")
    n = torch.full((B,), 2, dtype=torch.int32, device="cuda")
    p = torch.ones(B, device="cuda")
    for got in (ops.adjust_logits(x, ids, n, presence=p, mask=mask, mask_rows=rows),
                ops.adjust_logits(x, ids, n, presence=p, mask=mask, mask_rows=rows, out=torch.empty_like(buf)[:, :V])):
        assert torch.equal(got[:, ::2], x[:, ::2]) and (got[:, 1::2] == float("-inf")).all()
    tok = torch.full((B,), 7, device="cuda")
    for a, b in zip(ops.token_logprobs(x, tok, 5), ops.token_logprobs(x.contiguous(), tok, 5)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dev", DEVICES)
def test_attention_refuses_what_passes_32_bits(dev):
    """Places in a cache, rows and positions that the kernels' numbers do not hold: ValueError, as for everything that is not taken,
    before anything is allocated. Hints may be of any size."""
    i32 = dict(dtype=torch.int32, device=dev)
    q = torch.randn(1, 192, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    k = torch.randn(3, 1, 2048, 64, generator=torch.Generator().manual_seed(2)).bfloat16().to(dev)
    far = torch.zeros(1 << 20, **i32)  # (2^31 positions of one page)
    near = torch.tensor([[1]], **i32)
    ctx = torch.tensor([3000], **i32)
    cu = torch.tensor([0, 1], **i32)

    def call(q=q, k=k, ptab=near[0], prefix=2048, bt=near, **kw):
        return ops.attn_shared(q, k, k, ptab, prefix, bt, ctx, 1, 1, 64, 0.1, **kw)

    def no(match, **kw):
        with pytest.raises(ValueError, match=match):
            call(**kw)

    no("pages", k=torch.empty(1, 1, 1 << 24, 64, dtype=torch.bfloat16, device=dev))
    no("rows", q=q.expand(1 << 30, 192), cu_q=cu)
    no("prefix_len", ptab=far, prefix=1 << 31)
    no("prefix_len", ptab=far, prefix=1 << 30)
    for got in (call(), call(bt=torch.cat([near, far[None, 1:]], 1)), call(bt=torch.cat([near, far[None, 1:]], 1), max_own=(1 << 31) - 1),
                call(cu_q=cu, max_qlen=1 << 40), call(cu_q=cu, max_qlen=1 << 30)):
        _near(got, dict(q=q, k=k, v=k, ptab=near[0], prefix=2048, bt=near, ctx=ctx, qlens=[1], nh=1, nkv=1, D=64, bs=2048, scale=0.1))


def test_more_workgroups_than_a_launch_takes_are_refused():
    """At the native entry, which looks at them before it touches anything."""
    from llmss_amd import _native

    C = _native()
    T = 1 << 26  # (four rows a workgroup of the joining launch: 2^32 threads)
    parts = C.attn_shared_parts(T, 1, 1, 1, 256, 0, 1, 1, False)
    with pytest.raises(ValueError, match="too many rows"):
        C.attn_shared(0, 256, 0, 0, 1, 0, 0, 0, 1, 1, 0, 0, 0, 256, 0, parts, T, 1, 1, 1, 256, 16, 1, 1, 0.1, False, 0)


def test_attention_refusals():
    c = _case("cpu", 4, 2, 64, 33, [3, 30, 18])

    def no(match, **kw):
        args = dict(q=c["q"], k=c["k"], v=c["v"], ptab=c["ptab"], prefix=c["prefix"], bt=c["bt"], ctx=c["ctx"], nh=4, nkv=2, D=64,
                    scale=0.1, cu_q=None, max_qlen=1, max_own=None, out=None)
        args.update(kw)
        a = [args.pop(n) for n in ("q", "k", "v", "ptab", "prefix", "bt", "ctx", "nh", "nkv", "D", "scale")]
        with pytest.raises(ValueError, match=match):
            ops.attn_shared(*a, **args)

    no("nh must", nh=3)
    no("head_dim", D=32)
    no("q bf16", q=c["q"].float())
    no("q bf16", q=c["q"][:, :100])
    no("k_cache", k=c["k"].float())
    no("k_cache", nkv=4)
    no("v_cache", v=c["v"][:-1])
    no("prefix_table", ptab=c["ptab"].long())
    no("prefix_len", prefix=49)
    no("prefix_len", prefix=-1)
    no("block_tables", bt=c["bt"][0])
    no("ctx_lens", ctx=c["ctx"][:2])
    no("cu_q", max_qlen=2)
    no("cu_q", cu_q=c["cu"].long())
    no("max_own", max_own=1000)
    no("out", out=torch.zeros(2, 256, dtype=torch.bfloat16))
    no("out", out=torch.zeros(1, 256, dtype=torch.bfloat16).expand(3, 256))
    no("scale", scale=0.0)


# ---------------------------------------------------------------------------------------------------------------- logits
def _rules_plain(x, ids, lens, prompts, r, p, f, bids, bias, mask, rows, V):
    """In 64 bits, token by token: (result, sum of the magnitudes that enter it)."""
    y, mag = x[:, :V].to(F64).clone(), x[:, :V].to(F64).abs()
    for b in range(x.shape[0]):
        n = int(lens[b]) if lens is not None else 0
        seen, count = set(), {}
        for i in range(min(max(n, 0), ids.shape[1]) if lens is not None else 0):
            t = int(ids[b, i])
            if 0 <= t < V:
                seen.add(t)
                if i >= (int(prompts[b]) if prompts is not None else 0):
                    count[t] = count.get(t, 0) + 1
        if r is not None:
            for t in seen:
                y[b, t] = y[b, t] / float(r[b]) if y[b, t] > 0 else y[b, t] * float(r[b])
                mag[b, t] = y[b, t].abs()
        for t, k in count.items():
            if f is not None:
                y[b, t] -= k * float(f[b])
                mag[b, t] += abs(k * float(f[b]))
            if p is not None:
                y[b, t] -= float(p[b])
                mag[b, t] += abs(float(p[b]))
        if bids is not None:
            for t, v in zip(bids[b].tolist(), bias[b].tolist()):
                if 0 <= t < V:
                    y[b, t] += v
                    mag[b, t] += abs(v)
        if mask is not None:
            m = int(rows[b]) if rows is not None else b
            if 0 <= m < mask.shape[0]:
                for t in range(V):
                    if not (int(mask[m, t // 32]) >> (t % 32)) & 1:
                        y[b, t] = float("-inf")
    return y, mag


def _rules_case(B, V, wide, dtype, known, biases, masks, seed=0, ids=torch.int64):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(B, wide, generator=g) * 3).to(dtype)
    hist = torch.randint(-2, min(V + 3, 40), (B, known), generator=g).to(ids)  # (outside the vocabulary too, many of them twice)
    hist[:, ::3] = torch.randint(0, V, hist[:, ::3].shape, generator=g).to(ids)
    lens = torch.randint(0, known + 2, (B,), generator=g, dtype=torch.int32)
    prompts = (lens // 2).int()
    r, p, f = 0.6 + torch.rand(B, generator=g), torch.rand(B, generator=g) * 2 - 1, torch.rand(B, generator=g)
    bids = bias = mask = rows = None
    if biases:
        bids = torch.randint(-1, V + 1, (B, biases), generator=g, dtype=torch.int32)
        bids[:, -1] = bids[:, 0]
        bias = torch.randn(B, biases, generator=g) * 4
    if masks:
        mask = torch.randint(-2 ** 31, 2 ** 31, (masks, -(-V // 32)), generator=g).to(torch.int32)
        mask[-1] = 0
        rows = torch.randint(-1, masks + 1, (B,), generator=g, dtype=torch.int32)
    return x, hist, lens, prompts, r, p, f, bids, bias, mask, rows


def _adjust(dev, c, V, **kw):
    x, ids, lens, prompts, r, p, f, bids, bias, mask, rows = (t.to(dev) if t is not None else None for t in c)
    return ops.adjust_logits(x, ids, lens, prompts, repetition=r, presence=p, frequency=f, bias_ids=bids, bias=bias, mask=mask,
                             mask_rows=rows, vocab=V, **kw)


def _rules_near(got, c, V, dtype):
    want, mag = _rules_plain(*c, V)
    got = got.cpu()
    assert got.shape == want.shape and got.dtype == dtype
    shut = want == float("-inf")
    assert torch.equal(got == float("-inf"), shut)
    # a division or product, count times frequency, two differences, up to a few sums: 8 roundings of what enters, and the result's own
    step = 8 * 2.0 ** -24 * mag + (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0)
    assert ((got.to(F64) - want).abs()[~shut] <= step[~shut] + 1e-30).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V,wide,known,biases,masks", [
    (1, 1, 1, 1, 0, 0), (3, 33, 40, 5, 2, 1), (2, 1000, 1000, 60, 9, 3), (5, 2049, 2056, 300, 64, 2), (4, 1025, 1031, 37, 1024, 5),
    (2, 5003, 5003, 700, 0, 2), (300, 70, 72, 20, 3, 0)])
def test_rules_on_logits(dev, dtype, B, V, wide, known, biases, masks):
    c = _rules_case(B, V, wide, dtype, known, biases, masks, seed=V)
    _rules_near(_adjust(dev, c, V), c, V, dtype)
    if dtype == torch.bfloat16:
        out = torch.full((B + 1, V + 2), 7.0, device=dev)
        got = _adjust(dev, c, V, out=out)
        _rules_near(got, c, V, torch.float32)
        assert got.data_ptr() == out.data_ptr() and (out[B:] == 7).all() and (out[:, V:] == 7).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_rules_in_place_and_each_alone(dev):
    c = list(_rules_case(4, 700, 704, torch.float32, 50, 6, 2, seed=1, ids=torch.int32))
    x = c[0].to(dev)
    for keep in ((4,), (5,), (6,), (7, 8), (9, 10), ()):
        one = [t if i < 4 or i in keep else None for i, t in enumerate(c)]
        if not set(keep) & {4, 5, 6}:
            one[1] = one[2] = None
        mine = x.clone()
        got = ops.adjust_logits(mine, *(t.to(dev) if t is not None else None for t in one[1:4]),
                                **{n: t.to(dev) if t is not None else None for n, t in zip(
                                    ("repetition", "presence", "frequency", "bias_ids", "bias", "mask", "mask_rows"), one[4:])},
                                vocab=700, out=mine)
        assert got.data_ptr() == mine.data_ptr() and torch.equal(mine[:, 700:], x[:, 700:])
        _rules_near(got, one, 700, torch.float32)
        if not keep:
            assert torch.equal(got, x[:, :700])


@pytest.mark.parametrize("dev", DEVICES)
def test_rules_pass_on_what_is_not_finite(dev):
    x = torch.tensor([[float("nan"), float("inf"), float("-inf"), -0.0, 3.0, float("nan"), float("inf"), 1.0]] * 2).to(dev)
    mask = torch.tensor([[0x1F]], dtype=torch.int32, device=dev)
    ids = torch.tensor([[1, 2, 4]] * 2, device=dev)
    n = torch.tensor([3, 0], dtype=torch.int32, device=dev)
    got = ops.adjust_logits(x, ids, n, repetition=torch.tensor([2.0, 2.0], device=dev), mask=mask,
                            mask_rows=torch.zeros(2, dtype=torch.int32, device=dev)).cpu()
    for row, last in zip(got, (1.5, 3.0)):
        assert row[0].isnan() and row[1] == float("inf") and row[2] == float("-inf") and row[3] == 0 and row[4] == last
        assert (row[5:] == float("-inf")).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_rules_pass_over_what_is_out_of_range(dev):
    lo64, hi64, lo32, hi32 = -2 ** 63, 2 ** 63 - 1, -2 ** 31, 2 ** 31 - 1
    V = 3000
    x = torch.randn(4, V, generator=torch.Generator().manual_seed(4)).to(dev)
    ids = torch.tensor([[lo64, hi64, V, -1, 2500, lo32, hi32, 7]] * 4).to(dev)
    lens = torch.tensor([8, hi32, -5, 5], dtype=torch.int32, device=dev)
    prompts = torch.tensor([lo32, 5, 3, hi32], dtype=torch.int32, device=dev)
    bids = torch.tensor([[lo32, hi32, V, 2999]] * 4, dtype=torch.int32, device=dev)
    mask = torch.zeros(1, 94, dtype=torch.int32, device=dev)
    got = ops.adjust_logits(x, ids, lens, prompts, presence=torch.full((4,), 0.5, device=dev), bias_ids=bids,
                            bias=torch.ones(4, 4, device=dev), mask=mask,
                            mask_rows=torch.tensor([lo32, hi32, 1, -1], dtype=torch.int32, device=dev))
    want = x.clone()
    want[:, 2999] += 1
    want[0, [2500, 7]] -= 0.5  # all behind the prompt; of the second row 7 alone, of the others none
    want[1, 7] -= 0.5
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_rules_of_long_histories():
    """Counters of 16 bits up to 32767 known tokens, of 32 beyond; one token that was said each time."""
    for known in (16383, 16384, 32767, 32768, 40000):
        x = torch.randn(2, 3000, device="cuda")
        ids = torch.randint(0, 3000, (2, known), device="cuda")
        ids[1] = 17
        n = torch.tensor([known, known], dtype=torch.int32, device="cuda")
        f = torch.tensor([0.01, 0.01], device="cuda")
        got = ops.adjust_logits(x, ids, n, frequency=f).cpu().double()
        want = x.cpu().double()
        for b in range(2):
            want[b] -= torch.bincount(ids[b].cpu(), minlength=3000).double() * float(f[b])
        assert ((got - want).abs() <= 4 * 2.0 ** -24 * (x.cpu().abs().double() + (want - x.cpu().double()).abs()) + 1e-30).all()


@pytest.mark.gpu
def test_biases_of_one_token_are_summed_in_order():
    g = torch.Generator().manual_seed(2)
    ids = torch.full((3, 500), 77, dtype=torch.int32)
    ids[1, ::2] = 5
    bias = torch.randn(3, 500, generator=g) * 1e3
    x = torch.zeros(3, 100)
    want = ops.adjust_logits(x, bias_ids=ids, bias=bias)
    for _ in range(5):
        got = ops.adjust_logits(x.cuda(), bias_ids=ids.cuda(), bias=bias.cuda())
        assert torch.equal(got.cpu(), want)


def test_rules_refusals():
    x = torch.zeros(2, 64)
    i = torch.zeros(2, 3, dtype=torch.int64)
    n = torch.zeros(2, dtype=torch.int32)
    f = torch.zeros(2)
    no = lambda match, *a, **kw: pytest.raises(ValueError, ops.adjust_logits, *a, **kw).match(match)  # noqa: E731
    no("logits", x.half())
    no("logits", x[0])
    no("vocab", x, vocab=65)
    no("vocab", x, vocab=0)
    no("ids and lens", x, i)
    no("penalties", x, repetition=f)
    no("ids", x, i.float(), n, repetition=f)
    no("lens", x, i, n.long(), repetition=f)
    no("prompt_lens", x, i, n, n.long())
    no("repetition", x, i, n, repetition=f.double())
    no("presence", x, i, n, presence=f[:1])
    no("bias", x, bias=f)
    no("bias_ids", x, bias_ids=i, bias=i.float())
    no("1024", x, bias_ids=torch.zeros(2, 1025, dtype=torch.int32), bias=torch.zeros(2, 1025))
    no("mask_rows", x, mask_rows=n)
    no("mask", x, mask=torch.zeros(2, 1, dtype=torch.int32))
    no("mask", x, mask=torch.zeros(1, 2, dtype=torch.int32))
    no("out", x, out=torch.zeros(2, 63))
    no("out", x, out=x.bfloat16())
    no("out", x, out=x[:1].expand(2, 64))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rules_in_place_on_rows_that_are_not_aligned(dev, dtype):
    c = list(_rules_case(5, 2049, 2051, dtype, 60, 64, 2))
    x = torch.zeros(5 * 2051 + 8, device=dev).to(dtype)[1:1 + 5 * 2051].view(5, 2051)
    x.copy_(c[0])
    got = _adjust(dev, [x, *c[1:]], 2049, out=x)
    assert got.data_ptr() == x.data_ptr() and torch.equal(x[:, 2049:].cpu(), c[0][:, 2049:])
    _rules_near(got, c, 2049, dtype)


@pytest.mark.parametrize("dev", DEVICES)
def test_rules_refuse_a_result_that_overlaps_the_logits_otherwise(dev):
    """A result that lies over other logits than its own: some would be overwritten before they are read."""
    buf = torch.zeros(8, 128, device=dev)
    flat = buf.view(-1)
    no = lambda x, **kw: pytest.raises(ValueError, ops.adjust_logits, x, **kw).match("out")  # noqa: E731
    no(flat[:192].view(3, 64), out=flat[8:200].view(3, 64))
    no(flat[8:200].view(3, 64), out=flat[:192].view(3, 64))
    no(buf[:4], out=buf[1:5])
    no(buf[:2, :64], out=flat[:256].view(4, 64)[:2])  # (the same first row, the second over the first's)
    no(buf[:, 8:72], out=buf[:, 71:])
    no(buf[:, 8:72], vocab=57, out=buf[:, 64:])
    half = flat.view(torch.bfloat16)[:256].view(2, 128)
    no(half, out=flat[:256].view(2, 128))
    no(half[:1], out=flat[:128].view(1, 128))
    # beside them, between them, of a row that only one of them has: as good as anywhere
    buf.copy_(torch.arange(8 * 128).view(8, 128))
    want = buf.clone()
    for x, out, kw in ((buf[:, :64], buf[:, 64:], {}), (buf[::2], buf[1::2], {}), (buf[:, 8:72], buf[:, 64:], dict(vocab=56)),
                       (buf[:3], buf[3:], {}), (buf[:3], buf[:3], {}), (buf[:1], buf[:2], {}), (buf[1:3, :64], buf[:2, 64:], {})):
        buf.copy_(want)
        V = kw.get("vocab", x.shape[1])
        old = x.clone()
        got = ops.adjust_logits(x, out=out, **kw)
        assert torch.equal(got, old[:, :V]) and got.data_ptr() == out.data_ptr()


# -------------------------------------------------------------------------------------------------------------- logprobs
def _lp_near(got, want):
    """64 bits' log-softmax: the maximum's difference, an exponential and a logarithm round, and a sum of up to 2^17 terms in
    partial sums of at most 32 + 14 additions: 64 roundings of 2^-24 of 1 + |lp|."""
    got, want = got.cpu().double(), want.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine) and torch.equal(got[~fine], want[~fine])
    assert ((got - want).abs()[fine] <= 64 * 2.0 ** -24 * (1 + want[fine].abs())).all()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V,wide,n", [(1, 1, 1, 1), (2, 5, 8, 5), (3, 64, 64, 64), (4, 2049, 2056, 20), (2, 8193, 8193, 1), (1, 9001, 9008, 0),
                                        (70, 333, 336, 33), (2, 30000, 30000, 64)])
def test_log_probabilities(dev, dtype, B, V, wide, n):
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(B, wide, generator=g) * 4).to(dtype)
    x[:, V // 2] = x[:, 0]  # (equal logits: the lower token first)
    tok = torch.randint(0, V, (B,), generator=g)
    tok[-1] = x[-1, :V].float().argmax()
    lp, rank, ids, top = ops.token_logprobs(x.to(dev), tok.to(dev), n, vocab=V)
    x64 = x[:, :V].to(F64)
    want = torch.log_softmax(x64, -1)
    at = torch.arange(B)
    _lp_near(lp, want[at, tok])
    assert torch.equal(rank.cpu(), 1 + (x64 > x64[at, tok][:, None]).sum(-1))
    order = torch.sort(x64, dim=-1, descending=True, stable=True)[1][:, :n]
    assert torch.equal(ids.cpu(), order) and ids.shape == (B, n)
    _lp_near(top, want.gather(1, order))


@pytest.mark.parametrize("dev", DEVICES)
def test_log_probabilities_of_rows_out_of_the_ordinary(dev):
    V = 5000
    x = torch.randn(6, V)
    x[0] = float("-inf")
    x[1, 1:] = float("-inf")
    x[2, 7] = float("nan")
    x[3] = 2.0  # all equal
    x[4, :] = float("nan")
    x[4, 3] = float("-inf")
    x[5, 10], x[5, 4000] = -0.0, 0.0
    x[5, x[5] > 0] *= -1
    tok = torch.tensor([5, 0, 3, 4, -1, V], dtype=torch.int64)
    lp, rank, ids, top = (t.cpu() for t in ops.token_logprobs(x.to(dev), tok.to(dev), 4))
    inf = float("-inf")
    assert lp[0] == inf and ids[0].tolist() == [0, 1, 2, 3] and (top[0] == inf).all() and rank[0] == 1
    assert lp[1] == 0 and ids[1].tolist() == [0, 1, 2, 3] and top[1].tolist() == [0, inf, inf, inf]
    assert lp[2].isnan() and 7 not in ids[2].tolist() and top[2].isnan().all()
    assert ids[3].tolist() == [0, 1, 2, 3] and abs(float(lp[3]) + math.log(V)) < 1e-5 and rank[3] == 1
    assert lp[4] == 0 and rank[4] == 0 and ids[4].tolist() == [3, -1, -1, -1]
    assert lp[5] == 0 and rank[5] == 0 and ids[5][:2].tolist() == [10, 4000]


@pytest.mark.gpu
def test_log_probabilities_do_not_depend_on_the_batch():
    """The same rows alone and among as many as take the other cut, over vocabularies on both sides of each cut."""
    for V in (16384, 16385, 32768, 32769, 50257, 65536, 65537):
        for dtype in (torch.float32, torch.bfloat16):
            x = (torch.randn(600, V, generator=torch.Generator(device="cuda").manual_seed(V), device="cuda") * 4).to(dtype)
            tok = torch.randint(0, V, (600,), device="cuda")
            many = ops.token_logprobs(x, tok, 5)
            few = ops.token_logprobs(x[:9], tok[:9], 5)
            assert torch.equal(many[1][:9], few[1]) and torch.equal(many[2][:9], few[2])
            want = torch.log_softmax(x[:9].cpu().double(), -1)
            for lp, _, ids, top in (many, few):
                _lp_near(lp[:9], want.gather(1, tok[:9, None].cpu())[:, 0])
                _lp_near(top[:9], want.gather(1, ids[:9].cpu()))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [300, 20000, 70000])
def test_log_probabilities_of_logits_masked_with_the_lowest_value(dev, dtype, V):
    low = torch.finfo(dtype).min
    x = torch.full((3, V), low).to(dtype)
    x[0, 5], x[0, V - 1] = 2.0, 1.0
    x[1, V // 2:V // 2 + 9] = torch.arange(9).to(dtype)
    tok = torch.tensor([V - 1, 0, 3])
    lp, rank, ids, top = (t.cpu() for t in ops.token_logprobs(x.to(dev), tok.to(dev), 4))
    want = torch.log_softmax(x.double(), -1)
    for got, w in ((lp, want[torch.arange(3), tok]), (top, want.gather(1, ids))):
        ok = w > low / 2  # (the others are the lowest value or below it)
        _lp_near(got[ok], w[ok])
        assert (got[~ok] <= low * 0.99).all() and not got.isnan().any()
    assert rank.tolist() == [2, 10, 1] and ids[0].tolist() == [5, V - 1, 0, 1] and ids[2].tolist() == [0, 1, 2, 3]
    assert ids[1].tolist() == [V // 2 + 8 - i for i in range(4)]


@pytest.mark.gpu
def test_the_likeliest_of_sorted_rows():
    """Rising and falling rows put the likeliest into few threads' tokens; rows of two values are all ties."""
    V = 40001
    up = torch.arange(V, dtype=torch.float32) * 1e-3
    x = torch.stack([up, up.flip(0), (torch.arange(V) % 2).float(), torch.zeros(V)]).cuda()
    for n in (1, 4, 5, 20, 32, 33, 64):
        _, _, ids, _ = ops.token_logprobs(x, None, n)
        assert torch.equal(ids, torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :n])


def _unusual_rows(V, dtype):
    """Rows that strain the search for the likeliest, for cuts of some thousand tokens: (rows, tokens)."""
    g = torch.Generator().manual_seed(V)
    nan, inf = float("nan"), float("inf")
    run = V // 16
    x = torch.randn(14, V, generator=g) * 3
    up = torch.arange(V, dtype=torch.float32) * 1e-3
    x[0], x[1], x[2], x[3], x[4] = up, up.flip(0), (torch.arange(V) % 2).float(), 2.0, -inf
    few = torch.randperm(V, generator=g)
    x[5, few[3:]] = nan  # three numbers among NaN, and forty
    x[6, few[40:]] = nan
    x[7, 2 * run:5 * run] = nan  # whole runs of NaN, of -inf, all but one of -inf
    x[8, 2 * run:5 * run] = -inf
    x[9, :9 * run] = -inf
    x[9, 11 * run:] = -inf
    x[10] = nan
    x[11] = torch.finfo(dtype).min
    x[11, few[:5]] = torch.arange(5).float()
    x[12, V // 2] = inf
    x[13] = torch.where(x[13] > 0, 0.0, -0.0)
    tok = torch.randint(0, V, (14,), generator=g)
    tok[5], tok[9], tok[11], tok[12] = few[1], 10 * run, few[2], V // 2
    return x.to(dtype), tok


def _likeliest_plain(x, n):
    """The n likeliest of each row: falling values, the lower token first, no NaN; -1 where there are fewer."""
    ids = torch.full((x.shape[0], n), -1, dtype=torch.int64)
    for b in range(x.shape[0]):
        at = torch.nonzero(~x[b].isnan())[:, 0]
        order = at[torch.sort(x[b][at].double(), descending=True, stable=True)[1]][:n]
        ids[b, :order.numel()] = order
    return ids


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("wide", [0, 1])  # (odd strides: rows that are not aligned)
@pytest.mark.parametrize("B,V", [(14, 65537), (14, 131071), (300, 50257)])
def test_log_probabilities_in_two_launches(B, V, wide, dtype):
    """Vocabularies and batches whose rows are several workgroups', with up to 64 likeliest: ordinary rows and unusual ones."""
    from llmss_amd.ops import hip

    assert hip.lib().logprobs_runs(B, V) > 1
    odd, tok = _unusual_rows(V, dtype)
    cols = V + wide if wide else (V + 7) // 8 * 8
    x = torch.zeros(B, cols, dtype=dtype, device="cuda")[:, :V]
    x[:14] = odd.cuda()
    if B > 14:
        x[14:] = (torch.randn(B - 14, V, generator=torch.Generator(device="cuda").manual_seed(B), device="cuda") * 4).to(dtype)
        tok = torch.cat([tok, torch.randint(0, V, (B - 14,), generator=torch.Generator().manual_seed(B))])
    at = torch.arange(B)
    want = torch.log_softmax(x.double(), -1).cpu()
    want[4] = float("-inf")
    rank = 1 + (x.double() > x.double()[at, tok.cuda()][:, None]).sum(-1).cpu()
    every = _likeliest_plain(x.cpu(), 64)
    for n in (0, 1, 20, 33, 64):
        lp, r, ids, top = (t.cpu() for t in ops.token_logprobs(x, tok.cuda(), n))
        assert torch.equal(ids, every[:, :n]) and torch.equal(r, rank) and top.shape == (B, n)
        for got, w in ((lp, want[at, tok]), (top, torch.where(ids < 0, float("nan"), want.gather(1, ids.clamp(min=0))))):
            assert torch.equal(got.isnan(), w.isnan())
            _lp_near(got[~got.isnan()], w[~w.isnan()])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("V", [300, 9001, 20001, 65536])
def test_log_probabilities_of_unusual_rows(dev, V):
    """The same rows where each is one workgroup's, and by the definition."""
    for dtype in (torch.float32, torch.bfloat16):
        x, tok = _unusual_rows(V, dtype)
        want = torch.log_softmax(x.double(), -1)
        want[4] = float("-inf")
        for n in (0, 1, 20, 33, 64):
            lp, r, ids, top = (t.cpu() for t in ops.token_logprobs(x.to(dev), tok.to(dev), n))
            assert torch.equal(ids, _likeliest_plain(x, n))
            assert torch.equal(r, 1 + (x.double() > x.double()[torch.arange(14), tok][:, None]).sum(-1))
            for got, w in ((lp, want[torch.arange(14), tok]), (top, torch.where(ids < 0, float("nan"), want.gather(1, ids.clamp(min=0))))):
                assert torch.equal(got.isnan(), w.isnan())
                _lp_near(got[~got.isnan()], w[~w.isnan()])


def test_log_probabilities_refusals():
    x = torch.zeros(2, 64)
    t = torch.zeros(2, dtype=torch.int64)
    no = lambda match, *a, **kw: pytest.raises(ValueError, ops.token_logprobs, *a, **kw).match(match)  # noqa: E731
    no("logits", x.half(), t)
    no("tokens", x, t.int())
    no("tokens", x, t[:1])
    no("top_n", x, t, 65)
    no("top_n", x, t, 10, vocab=5)
    no("top_n", x, t, -1)
    no("vocab", x, t, vocab=65)


# --------------------------------------------------------------------------------------------------------------- together
def _step_state(dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    nh, nkv, D, V, B, P, bs = 4, 2, 64, 500, 6, 45, 16
    c = _case(dev, nh, nkv, D, P, [1] * B, seed=seed, spare=B + 3, own_cols=2, poison=False)
    head = (torch.randn(V + 4, nh * D, generator=g) * 0.6).bfloat16().to(dev)  # (padded, as the projection wants it)
    qkv = (torch.randn(4, B, (nh + 2 * nkv) * D, generator=g) * 1.5).bfloat16().to(dev)
    mask = torch.full((2, -(-V // 32)), -1, dtype=torch.int32)
    mask[1] = 0x0F0F0F0F
    return dict(c=c, head=head, qkv=qkv, V=V, B=B, P=P, bs=bs, nkv=nkv, D=D, mask=mask.to(dev),
                rows=torch.tensor([-1, 0, 1, 1, 0, -1], dtype=torch.int32, device=dev),
                temp=torch.tensor([0.0, 0.8, 0.0, 0.9, 1.0, 0.7], device=dev), topk=torch.full((B,), 40, dtype=torch.int32, device=dev),
                topp=torch.full((B,), 0.95, device=dev), ids=torch.zeros(B, 8, dtype=torch.int64, device=dev),
                rep=torch.full((B,), 1.3, device=dev), pres=torch.full((B,), 0.4, device=dev), freq=torch.full((B,), 0.2, device=dev))


def _step(s, i):
    """Token i of six completions of one prompt: cache rows, attention, head, rules, sampler, log-probabilities."""
    c = s["c"]
    qkv, B = s["qkv"][i], s["B"]
    nh, nkv, D = c["nh"], s["nkv"], s["D"]
    k, v = qkv[:, nh * D:(nh + nkv) * D].view(B, nkv, D), qkv[:, (nh + nkv) * D:].view(B, nkv, D)
    page = c["bt"][:, i // s["bs"]].long()
    c["k"][page, :, i % s["bs"]] = k
    c["v"][page, :, i % s["bs"]] = v
    dev = qkv.device
    ctx = torch.full((B,), s["P"] + i + 1, dtype=torch.int32, device=dev)
    o = ops.attn_shared(qkv, c["k"], c["v"], c["ptab"], s["P"], c["bt"], ctx, nh, nkv, D, c["scale"])
    logits = ops.linear(o, s["head"])
    n = torch.full((B,), i, dtype=torch.int32, device=dev)
    x = ops.adjust_logits(logits, s["ids"], n, repetition=s["rep"], presence=s["pres"], frequency=s["freq"], mask=s["mask"],
                          mask_rows=s["rows"], vocab=s["V"], out=torch.empty(B, s["V"], device=dev))
    tok = ops.sample(x, s["temp"], s["topk"], s["topp"], torch.arange(B, device=dev) + 100 * i)
    s["ids"][:, i] = tok
    return o, x, tok, ops.token_logprobs(x, tok, 3)


@pytest.mark.parametrize("dev", DEVICES)
def test_a_decode_step_of_completions_of_one_prompt(dev):
    s = _step_state(dev)
    for i in range(4):
        before = s["ids"].clone()
        o, x, tok, (lp, rank, ids, top) = _step(s, i)
        _near(o, dict(s["c"], q=s["qkv"][i], ctx=torch.full((6,), s["P"] + i + 1), qlens=[1] * 6))
        assert torch.equal(x.cpu()[[2, 3]][:, 4:8], torch.full((2, 4), float("-inf")))  # (bits 4 .. 7 of the second mask are clear)
        assert all((int(s["mask"][1, int(t) // 32]) >> (int(t) % 32)) & 1 for t in tok[2:4])
        want = torch.log_softmax(x.double().cpu(), -1)
        _lp_near(lp, want[torch.arange(6), tok.cpu()])
        assert torch.equal(tok[[0, 2]], ids[[0, 2], 0]) and (rank[[0, 2]] == 1).all()  # greedy rows took the likeliest
        assert torch.equal(before[:, :i], s["ids"][:, :i])


@pytest.mark.gpu
def test_a_captured_step_replays_with_new_inputs():
    """Two captured steps of different sizes, replayed in turn with eager calls between them."""
    s, e = _step_state("cuda"), _step_state("cuda")
    other = _case("cuda", 8, 2, 128, 300, [4, 60, 33], seed=2)
    want_other = _run(other)
    _step(s, 0)
    torch.cuda.synchronize()
    s = _step_state("cuda")
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        got = _step(s, 0)
    with torch.cuda.graph(g2):
        got_other = _run(other)
    for seed in range(4):
        new = torch.randn(6, s["qkv"].shape[2], generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
        s["qkv"][0].copy_(new)
        e["qkv"][0].copy_(new)
        g1.replay()
        _run(_case("cuda", 4, 4, 64, 40, [3] * 30, seed=seed))
        g2.replay()
        want = _step(e, 0)
        torch.cuda.synchronize()
        assert torch.equal(got_other, want_other)
        for a, b in zip((got[0], got[1], got[2], *got[3]), (want[0], want[1], want[2], *want[3])):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_calls_on_several_streams():
    cases = [_case("cuda", 4, 2, 128, 200 + 50 * i, [1 + i, 20, 40], seed=i) for i in range(4)]
    want = [_run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_run(cases[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for xs, w in zip(got, want) for x in xs)


@pytest.mark.gpu
def test_shared_attention_agrees_with_decode_attention():
    """The same pages through attn_decode's tables, where the prefix is whole pages."""
    c = _case("cuda", 8, 2, 128, 320, [1, 50, 17, 200], seed=11)
    tables = torch.cat([c["ptab"][None].expand(4, -1), c["bt"].clamp(min=0)], 1).contiguous()
    want = ops.attn_decode(c["q"], c["k"], c["v"], tables, c["ctx"], 8, 2, 128, c["scale"], tables.shape[1] * 16)
    got = _run(c)
    _, A = _plain(c)
    # each is within 3 * 2^-8 A of the exact result
    assert ((got.cpu().double() - want.cpu().double()).abs() <= 6 * 2.0 ** -8 * A + 2.0 ** -9 * A).all()


@pytest.mark.gpu
def test_operands_of_another_place_are_refused():
    c = _case("cuda", 4, 2, 64, 33, [3, 30, 18])
    with pytest.raises(ValueError, match="current device"):
        _run(dict(c, ctx=c["ctx"].cpu()))
    with pytest.raises(ValueError, match="current device"):
        ops.adjust_logits(torch.zeros(2, 64, device="cuda"), mask=torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="current device"):
        ops.token_logprobs(torch.zeros(2, 64, device="cuda"), torch.zeros(2, dtype=torch.int64))
    q = torch.zeros(3, c["q"].shape[1] + 4, dtype=torch.bfloat16, device="cuda")[:, 4:]
    with pytest.raises(ValueError, match="aligned"):
        _run(dict(c, q=q))
    k = torch.zeros(c["k"].numel() + 8, dtype=torch.bfloat16, device="cuda")[4:-4].view(c["k"].shape)
    with pytest.raises(ValueError, match="aligned"):
        _run(dict(c, k=k))


@pytest.mark.parametrize("dev", DEVICES)
def test_empty_batches(dev):
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    c = _case(dev, 4, 2, 64, 33, [3], seed=17)
    assert _run(dict(c, q=c["q"][:0], bt=c["bt"][:0], ctx=none)).shape == (0, 256)
    assert ops.adjust_logits(torch.zeros(0, 8, device=dev)).shape == (0, 8)
    lp, rank, ids, top = ops.token_logprobs(torch.zeros(0, 8, device=dev), None, 3)
    assert lp.shape == rank.shape == (0,) and ids.shape == top.shape == (0, 3)
