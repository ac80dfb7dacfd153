"""The speculative decoding operators (include/kvbp.h, speculative.py) against plain 64-bit
statements of the same formulas (tests/spec_ref.py), at the sizes and masks where they can go
wrong.  Tolerances count roundings and are derived beside each check."""

import math
from decimal import Decimal, getcontext

import numpy as np
import pytest
import torch

import spec_ref as ref
from kvcacheboundaryprotection_b200 import build, capi, speculative as sp

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _lib():
    build.build()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------ tree attention
def _attn_case(B, T, hq, hkv, S, seed, mask="slots", lens=None, kind="tree", loud=1.5):
    g, rng = _gen(seed), np.random.default_rng(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    c = {"q": (loud * r(B, T, hq, 128)).to(BF), "k": r(B, hkv, S, 128).to(BF), "v": r(B, hkv, S, 128).to(BF),
         "kd": r(B, hkv, T, 128).to(BF), "vd": r(B, hkv, T, 128).to(BF),
         "parents": torch.tensor([ref.random_tree(rng, T, kind, (b * 7) % (T // 3 + 1)) for b in range(B)],
                                 dtype=torch.int32),
         "slot_pos": None, "lens": None}
    if mask == "slots":
        c["slot_pos"] = torch.where(torch.rand(B, S, generator=g) < 0.2, -1, torch.arange(S)).to(torch.int32)
    elif mask == "none":
        c["slot_pos"] = torch.full((B, S), -1, dtype=torch.int32)
    if lens is not None:
        c["lens"] = torch.tensor([lens[b % len(lens)] for b in range(B)], dtype=torch.int32)
    return c


def _gpu(c):
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in c.items()}


def _run(c, score=None, **kw):
    d = _gpu(c)
    return sp.tree_attend(d["q"], d["k"], d["v"], d["kd"], d["vd"], d["parents"], slot_pos=d["slot_pos"],
                          lens=d["lens"], node_score=score, **kw)


def _check_attn(c, out, score=None, before=None, scale=None):
    want, top, mag, spread = ref.attend(c["q"], c["k"], c["v"], c["kd"], c["vd"], c["parents"], c["slot_pos"],
                                        c["lens"], scale)
    # a logit: 128 products and their sum in fp32, each step off by 2^-24 of sum |q k|, scaled and
    # carried in the exponent (a few roundings of the largest logit); p is off by as much, relatively
    logit = 140 * 2.0 ** -24 * spread[..., None].double() + 2.0 ** -21
    # out: half a step of bf16 (2^-8), each weight half a step of bf16 in the sum and in its total
    tol = 2.0 ** -8 * want.abs() + (2 * 2.0 ** -8 + 2 * logit) * mag * 1.01 + 1e-30
    err = (out.double().cpu() - want).abs()
    assert torch.isfinite(out).all() and (err <= tol).all(), (err / tol).max().item()
    if score is not None:
        # p: the logit's error twice (its own and the sum's), fp32 sums of up to S terms in steps of a
        # tile, 2^x and the division
        n = c["k"].shape[2] + c["q"].shape[1]
        rel = 2 * logit.amax((2, 3))[..., None] + (256 + n / 128 + 16) * 2.0 ** -24
        want_s = torch.maximum(top, before.double()) if before is not None else top
        e = (score.double().cpu() - want_s).abs()
        assert (e <= rel * top + 1e-37).all(), (e / (rel * top + 1e-37)).max().item()


SHAPES = [  # B, T, Hq, Hkv, S
    (1, 1, 8, 1, 1), (2, 1, 7, 1, 129), (1, 8, 16, 2, 256), (3, 5, 28, 4, 127), (2, 16, 28, 4, 128), (1, 17, 7, 1, 300),
    (2, 33, 8, 8, 64), (1, 64, 32, 8, 515), (1, 128, 8, 2, 200), (2, 128, 16, 2, 131), (1, 37, 14, 2, 1032), (4, 2, 2, 2, 15),
    (1, 3, 40, 1, 260), (1, 9, 128, 1, 140), (5, 19, 6, 2, 33),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kind", ["tree", "chain", "star"])
def test_attention_with_free_slots_and_score(shape, kind):
    B, T, hq, hkv, S = shape
    c = _attn_case(B, T, hq, hkv, S, 11 * T + S, kind=kind)
    score = torch.zeros(B, T, S + T, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = _run(c, score, dev_err=err)
    _check_attn(c, out, score)
    assert err.item() == 0


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_without_masks(shape):
    c = _attn_case(*shape, seed=5, mask=None)
    _check_attn(c, _run(c))


@pytest.mark.parametrize("shape", [(4, 6, 8, 2, 400), (7, 33, 28, 4, 260), (3, 128, 8, 1, 129)], ids=str)
def test_attention_of_ragged_lengths(shape):
    B, T, _, _, S = shape
    c = _attn_case(*shape, seed=3, mask="slots", lens=[S, 0, 1, 128, 127, 129, 64])
    score = torch.zeros(B, T, S + T, device="cuda")
    _check_attn(c, _run(c, score), score)
    c["slot_pos"] = None
    _check_attn(c, _run(c))


@pytest.mark.parametrize("T,hq,hkv", [(4, 8, 2), (64, 8, 2), (128, 8, 1)])
def test_attention_over_the_tree_alone(T, hq, hkv):
    """No cache at all, an empty one and one whose slots are all free."""
    for S, mask in ((0, None), (140, "none")):
        c = _attn_case(2, T, hq, hkv, S, 9, mask=mask)
        score = torch.zeros(2, T, S + T, device="cuda")
        _check_attn(c, _run(c, score), score)
    c["lens"] = torch.zeros(2, dtype=torch.int32)
    _check_attn(c, _run(c))


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -3e38])
@pytest.mark.parametrize("shape", [(2, 6, 8, 2, 300), (1, 40, 28, 4, 140)], ids=str)
def test_what_a_row_does_not_see_never_reaches_it(shape, bad):
    """Free slots, slots past the length, unused nodes and other branches hold NaN or infinities."""
    B, T, hq, hkv, S = shape
    c = _attn_case(*shape, seed=21, mask="slots", lens=[S - 9], kind="star")
    c["parents"][:, 1:] = torch.arange(T - 1).clamp(max=T // 2) * (torch.arange(T - 1) % 2)  # some branches
    c["parents"][0, 3] = 0
    c["parents"][:, T - 1] = -2
    clean, clean_top, _, _ = ref.attend(c["q"], c["k"], c["v"], c["kd"], c["vd"], c["parents"], c["slot_pos"], c["lens"])
    hidden = torch.ones(B, S, dtype=torch.bool)
    for b in range(B):
        hidden[b, : S - 9] = c["slot_pos"][b, : S - 9] < 0
    for x in ("k", "v"):
        c[x] = torch.where(hidden[:, None, :, None], torch.tensor(bad).to(BF), c[x])
    node = 2  # a branch: only what descends from it may see it
    for x in ("kd", "vd"):
        c[x][:, :, T - 1] = bad
        c[x][:, :, node, ::3] = bad
    score = torch.zeros(B, T, S + T, device="cuda")
    out = _run(c, score).double().cpu()
    for b in range(B):
        for t, seen in enumerate(ref.sees(c["parents"][b].tolist())):
            if seen is None:
                assert (out[b, t] == 0).all() and (score[b, t] == 0).all()
            elif node not in seen:
                assert (out[b, t] - clean[b, t]).abs().max() < 0.05, (b, t)  # 3 * 2^-8 of |v| <= 4
                assert (score[b, t].double().cpu() - clean_top[b, t]).abs().max() < 1e-4, (b, t)


@pytest.mark.parametrize("T", [4, 20, 40, 100])
@pytest.mark.parametrize("B,S,lens", [(1, 900, None), (2, 1200, [1200, 3]), (64, 130, None), (300, 300, None)])
def test_rows_whose_logits_are_all_minus_infinity(T, B, S, lens):
    """softmax gives 0 / 0 there: NaN in such rows and only there, however the units are cut and joined; unused nodes
    stay 0."""
    c = _attn_case(B, T, 8, 2, S, 4, mask="slots" if S < 1000 else None, lens=lens)
    c["k"][:, 1], c["kd"][:, 1] = -float("inf"), -float("inf")
    c["q"][:, 1:, 4:] = c["q"][:, 1:, 4:].abs() + 0.01  # kv head 1's rows but for the root's
    c["q"][:, 0, 4:] = -0.5
    c["parents"][:, T - 1] = -2
    out = _run(c).float().cpu()
    used = torch.tensor([[s is not None for s in ref.sees(p)] for p in c["parents"].tolist()])
    assert (out[~used] == 0).all() and torch.isfinite(out[:, :, :4]).all()
    assert torch.isnan(out[:, :, 4:][used]).all()  # (the root's: +inf logits)


@pytest.mark.parametrize("T,hq,hkv,S", [(6, 8, 2, 200), (40, 16, 2, 300), (128, 4, 4, 70), (3, 60, 1, 500)])
def test_nan_weights_reach_the_scores(T, hq, hkv, S):
    """A NaN in a node's query (one head of it): its scores are NaN for all that it sees, and only there; the error
    word says so, and so does the commit that reads them."""
    c = _attn_case(2, T, hq, hkv, S, 4, mask="slots", kind="star")
    c["parents"][1, T - 1] = -2
    c["q"][0, 2, hq // 2, 7] = float("nan")
    c["q"][1, T - 1] = float("nan")  # an unused node's
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    score = torch.zeros(2, T, S + T, device="cuda")
    _run(c, score, dev_err=err)
    assert err.item() == 2
    live = c["slot_pos"][0] >= 0
    want = torch.zeros(2, T, S + T, dtype=torch.bool)
    want[0, 2, :S] = live
    want[0, 2, S], want[0, 2, S + 2] = True, True
    assert torch.equal(torch.isnan(score).cpu(), want)
    c["q"] = torch.nan_to_num(c["q"])
    clean = torch.zeros_like(score)
    err.zero_()
    _run(c, clean, dev_err=err)
    assert err.item() == 0 and torch.equal(torch.where(want.cuda(), 0, clean), torch.where(want.cuda(), 0, score))


def test_a_value_that_is_seen_counts():
    """Infinities and NaN of a seen node's V reach the rows that see it, in their dims only."""
    c = _attn_case(1, 6, 8, 2, 200, 4, mask=None, kind="star")
    c["parents"][0] = torch.tensor([-1, 0, 1, 0, 3, 0])
    c["vd"][0, :, 1, 5] = float("inf")
    c["vd"][0, :, 1, 77] = float("nan")
    out = _run(c)[0].float().cpu()
    for t in range(6):
        sees = t in (1, 2)
        assert torch.isposinf(out[t, :, 5]).all() if sees else torch.isfinite(out[t]).all()
        assert torch.isnan(out[t, :, 77]).all() == sees
        keep = [d for d in range(128) if d not in (5, 77)]
        assert torch.isfinite(out[t][:, keep]).all()


def test_scores_accumulate_and_unused_columns_stay():
    c = _attn_case(2, 10, 8, 2, 260, 6, mask="slots")
    before = torch.rand(2, 10, 270, generator=_gen(2)) * 0.02
    score = before.cuda()
    out = _run(c, score)
    _check_attn(c, out, score, before)
    again = score.clone()
    _run(c, again)
    assert torch.equal(again, score)


def test_extreme_logits_and_scale():
    c = _attn_case(1, 12, 8, 2, 300, 8, mask="slots", loud=200.0)  # one key takes all, or a few share it
    score = torch.zeros(1, 12, 312, device="cuda")
    _check_attn(c, _run(c, score), score)
    c = _attn_case(1, 12, 8, 2, 300, 8, mask="slots")
    score.zero_()
    _check_attn(c, _run(c, score, scale=0.0), score, scale=0.0)
    score.zero_()
    _check_attn(c, _run(c, score, scale=-0.3), score, scale=-0.3)


@pytest.mark.parametrize("with_score", [False, True])
@pytest.mark.parametrize("T,hq,hkv,S", [(9, 8, 2, 1500), (5, 8, 2, 3000), (13, 8, 2, 3000), (29, 8, 2, 3000),
                                        (40, 8, 2, 2600), (64, 4, 1, 5000)])
def test_growing_logits(T, hq, hkv, S, with_score):
    """The running maximum rises in every tile: few and many rows, one and two row tiles, several
    tiles a CTA (two sequences of which one is empty: ranges over all SMs)."""
    c = _attn_case(2, T, hq, hkv, S, 8, mask=None, lens=[S, 0])
    c["q"] = c["q"].abs()
    c["k"] = (c["k"].abs() * torch.linspace(0.01, 6, S)[:, None]).to(BF)
    score = torch.zeros(2, T, S + T, device="cuda") if with_score else None
    _check_attn(c, _run(c, score), score)
    c = {k: v[:1] if torch.is_tensor(v) else v for k, v in c.items()}
    c["lens"] = None
    many = {k: v.repeat(*([40] + [1] * (v.dim() - 1))) if torch.is_tensor(v) else v for k, v in c.items()}
    out = _run(many)  # forty copies, cut in different places
    for i in (0, 7, 18, 39):
        _check_attn(c, out[i:i + 1])
    assert torch.equal(_run(many), out)


@pytest.mark.parametrize("T,hq,hkv,S", [(40, 8, 2, 140), (33, 28, 4, 70), (128, 8, 1, 300)])
def test_many_units_of_two_row_tiles_a_cta(T, hq, hkv, S):
    """Several hundred units over the SMs, so that every CTA goes from unit to unit, maxima that rise and fall
    with them: the rows' statistics of one unit are not those of the next.  The same bits in every run."""
    B = 900 // hkv // (2 if T == 128 else 1)
    c = _attn_case(4, T, hq, hkv, S, 3, mask="slots", kind="chain")
    c["k"] = (c["k"] * torch.linspace(0.05, 5, S)[:, None]).to(BF)
    c["k"][1::2] = c["k"][1::2].flip(2)
    c["q"] = (c["q"] * torch.tensor([0.1, 3.0, 1.0, 6.0])[:, None, None, None]).to(BF)
    many = {k: v.repeat(*([B // 4 + 1] + [1] * (v.dim() - 1)))[:B].cuda() if torch.is_tensor(v) else v for k, v in c.items()}
    out = _run(many)
    for i in (0, 4 * (B // 8), B // 4 * 4 - 4):
        _check_attn(c, out[i:i + 4])
    score = torch.zeros(B, T, S + T, device="cuda")
    assert torch.equal(_run(many, score), out)
    _check_attn(c, out[:4], score[:4])
    for _ in range(20):
        assert torch.equal(_run(many), out)


def test_bad_parents_and_lengths_are_flagged():
    c = _attn_case(2, 6, 8, 2, 70, 8, mask=None)
    c["parents"][0] = torch.tensor([-1, 0, 4, 2, 7, 1])  # 2 and 4 name later nodes; 3 hangs on 2
    c["lens"] = torch.tensor([99, -5], dtype=torch.int32)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = _run(c, dev_err=err)
    assert err.item() == 4
    _check_attn(c, out)
    assert (out[0, 2:5] == 0).all()


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements: the last kv head's slots lie past them."""
    hkv, S, T = 2, 9_000_000, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.empty(1, hkv, S, 128, dtype=BF, device="cuda")
    v = torch.empty_like(k)
    for h in range(hkv):
        k[0, h].normal_(generator=g)
        v[0, h].normal_(generator=g)
    q = torch.randn(1, T, 2, 128, generator=g, device="cuda").to(BF) * 2
    kd, vd = (torch.randn(1, hkv, T, 128, generator=g, device="cuda").to(BF) for _ in range(2))
    par = torch.tensor([[-1, 0, 1]], dtype=torch.int32, device="cuda")
    out = sp.tree_attend(q, k, v, kd, vd, par).double()
    for h in range(2):
        for t in range(T):
            lg = torch.cat([torch.mv(k[0, h].float(), q[0, t, h].float()), kd[0, h, :t + 1].float() @ q[0, t, h].float()])
            p = torch.softmax(lg.double() / math.sqrt(128), 0)
            want = torch.zeros(128, dtype=torch.float64, device="cuda")
            mag = torch.zeros_like(want)
            for i in range(0, S, 1 << 20):
                want += p[i:min(S, i + (1 << 20))] @ v[0, h, i:i + (1 << 20)].double()
                mag += p[i:min(S, i + (1 << 20))] @ v[0, h, i:i + (1 << 20)].double().abs()
            want += p[S:] @ vd[0, h, :t + 1].double()
            # as _check_attn; sums of 9 million weights in fp32, tile by tile
            tol = 2.0 ** -8 * want.abs() + (2 * 2.0 ** -8 + 1e-3) * mag
            assert ((out[0, t, h] - want).abs() <= tol).all()


def test_attention_in_a_graph_and_on_two_streams():
    cs = [_attn_case(2, 12, 28, 4, 700, s, mask="slots") for s in (1, 2)]
    ds = [_gpu(c) for c in cs]
    scores = [torch.zeros(2, 12, 712, device="cuda") for _ in cs]

    def call(d, s, out=None):
        return sp.tree_attend(d["q"], d["k"], d["v"], d["kd"], d["vd"], d["parents"], slot_pos=d["slot_pos"],
                              node_score=s, out=out)

    plain = [call(d, s) for d, s in zip(ds, scores)]
    want = [s.clone() for s in scores]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    outs = [None, None]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i] = call(ds[i], scores[i])
    torch.cuda.synchronize()
    for o, p, s, w in zip(outs, plain, scores, want):
        assert torch.equal(o, p) and torch.equal(s, w)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(plain[0])
    with torch.cuda.graph(graph):
        call(ds[0], scores[0], out)
    ds[0]["q"].copy_(ds[1]["q"])
    scores[0].zero_()
    graph.replay()
    torch.cuda.synchronize()
    c = dict(cs[0], q=cs[1]["q"])
    _check_attn(c, out, scores[0])


# -------------------------------------------------------------------------------- verification
def _verify_case(B, T, V, seed, kind="tree", f32=False, draft=False, temp=None, pad=0):
    g, rng = _gen(seed), np.random.default_rng(seed)
    x = torch.randn(B, T, V, generator=g) * 2
    x.scatter_(2, torch.randint(0, V, (B, T, min(V, 5)), generator=g), math.log(V) + 2)
    t = torch.zeros(B, T, V + pad, dtype=torch.float32 if f32 else BF)
    t[..., :V] = x.to(t.dtype)
    t[..., V:] = 1000.0  # padding is never read
    par = torch.tensor([ref.random_tree(rng, T, kind, (b * 5) % (T // 3 + 1)) for b in range(B)], dtype=torch.int32)
    temps = None if temp is None else torch.tensor([temp[b % len(temp)] for b in range(B)], dtype=torch.float32)
    q = None
    if draft:
        q = torch.softmax(t[..., :V].float() + torch.randn(B, T, V, generator=g) * 0.5, -1)
    tokens = torch.zeros(B, T, dtype=torch.int32)
    for b in range(B):
        for n in range(1, T):
            p = max(0, int(par[b, n]))
            if draft:
                tokens[b, n] = int(torch.multinomial(q[b, p].double(), 1, generator=g))
            else:
                rank = int((par[b, :n] == par[b, n]).sum()) % min(V, 5)
                tokens[b, n] = int(torch.topk(t[b, p, :V].float(), min(V, 5))[1][rank])
    return {"target": t, "V": V, "tokens": tokens, "parents": par, "u": torch.rand(B, T, generator=g),
            "s": torch.rand(B, generator=g), "temp": temps, "draft": q}


def _run_verify(c, **kw):
    d = _gpu(c)
    return sp.verify_tree(d["target"][..., : c["V"]], d["tokens"], d["parents"], d["u"], d["s"], temperature=d["temp"],
                          draft_probs=d["draft"], **kw)


def _check_verify(c, got):
    path, n, token = (x.cpu() for x in got)
    for b in range(path.shape[0]):
        way, tok = ref.verify(c["target"][b, :, : c["V"]].double().numpy(), c["tokens"][b].tolist(),
                              c["parents"][b].tolist(), c["u"][b].tolist(), c["s"][b].item(),
                              None if c["temp"] is None else c["temp"][b].item(),
                              None if c["draft"] is None else c["draft"][b].numpy())
        assert n[b].item() == len(way) and path[b].tolist() == way + [-1] * (path.shape[1] - len(way)), b
        assert token[b].item() == tok, (b, way)


@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (3, 2, 2), (8, 6, 31), (5, 16, 1000), (16, 33, 4097), (2, 128, 3001),
                                   (3, 9, 50257), (2, 5, 152064), (1, 3, 260001)])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_verification(B, T, V, draft, f32):
    for kind, temp in (("tree", None), ("chain", [0.7, 0.0, 1.3]), ("star", [1.0, 0.4])):
        c = _verify_case(B, T, V, 7 * T + V, kind, f32, draft, temp)
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        _check_verify(c, _run_verify(c, dev_err=err))
        assert err.item() == 0


@pytest.mark.parametrize("V,pad", [(1000, 24), (1003, 5), (50257, 47), (152064, 1)])
def test_verification_of_padded_rows(V, pad):
    for f32 in (False, True):
        c = _verify_case(3, 7, V, 3, "tree", f32, False, [0.9], pad)
        _check_verify(c, _run_verify(c))


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("B,T,V", [(3, 9, 1000), (16, 33, 4097), (2, 6, 50257)])
def test_verification_where_fp32_decides_nothing(B, T, V, draft):
    """Logits far from zero: the fp32 sums' error bound grows with the maximum, so that every test and
    draw is made again in double."""
    for kind, temp in (("star", [1.0]), ("chain", [0.7, 0.0, 1.3])):
        c = _verify_case(B, T, V, 5 * T + V, kind, True, draft, temp)
        c["target"] += 2.0 ** 18
        _check_verify(c, _run_verify(c))


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("temp", [1e-3, 1e-5, 1e-6, 1e-7, 1e-9, 1e-20, 1e-30, 1e-38, 1e-42])
def test_verification_at_very_low_temperatures(temp, draft, f32):
    """The logit over the temperature is so large that fp32 does not hold the differences between logits: ties of
    the largest logits share the weight, what lies below has what is left of it."""
    c = _verify_case(32, 6, 3001, 17, "star", f32, draft, [temp])
    top = 20 + 44 * torch.rand(32, 6, generator=_gen(4))
    for i, at in enumerate((40, 41, 1500, 2900)):
        c["target"][:, :, at] = (top * (1 if i != 2 else 1 + 2.0 ** -20)).to(c["target"].dtype)
    if draft:
        c["draft"] = 0.5 * c["draft"]
        c["draft"][:, :, [40, 41, 1500, 2900]] += 0.125
    c["tokens"][:, 1:] = torch.tensor([40, 2900, 1500, 41, 7], dtype=torch.int32)
    for seed in range(4):
        c["u"], c["s"] = torch.rand(32, 6, generator=_gen(seed)), torch.rand(32, generator=_gen(seed + 9))
        _check_verify(c, _run_verify(c))


def test_verification_at_an_infinite_temperature():
    """Every finite logit has the same weight, filtered tokens none."""
    c = _verify_case(4, 4, 1000, 3, "star", True, False, [float("inf")])
    c["target"][2:, :, ::2] = -float("inf")
    c["parents"][:] = torch.tensor([-1, 0, 0, 0])
    c["tokens"][:, 1:] = torch.tensor([11, 12, 13], dtype=torch.int32)
    c["u"][:] = torch.tensor([0.0, 0.01, 0.0, 0.0])  # 0.01 * 1000 and 0.01 * 500 are above 1
    c["s"] = torch.tensor([0.25, 0.999, 0.25, 0.999])
    path, n, token = _run_verify(c)
    assert path[:, :2].tolist() == [[0, 2], [0, 2], [0, 3], [0, 3]] and n.tolist() == [2] * 4
    assert token.tolist() == [250, 999, 251, 999]


def test_verification_of_greedy_ties_and_equal_tokens():
    c = _verify_case(4, 8, 300, 3, "star", temp=[0.0, 1.0])
    c["target"][:, :, 17] = c["target"][:, :, 211] = 50.0  # a tie: the first one
    c["tokens"][:, 1:] = torch.tensor([211, 17, 17, 211, 17, 5, 5], dtype=torch.int32)
    _check_verify(c, _run_verify(c))
    path, n, token = _run_verify(c)
    assert path[0, 1].item() == 2 and token[0].item() == 17


def test_verification_of_odd_logits():
    """-inf (filtered tokens), +inf, NaN, rows with a single finite value, whole rows of -inf."""
    inf = float("inf")
    c = _verify_case(6, 5, 500, 13, "star", f32=True, temp=[1.0, 0.8, 0.0])
    c["target"][:, :, ::2] = -inf
    c["target"][1] = -inf
    c["target"][1, :, 3] = -700.0
    c["target"][2, 0, 44] = float("nan")
    c["target"][3, 0, [9, 99]] = inf
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    _check_verify(c, _run_verify(c, dev_err=err))
    assert err.item() == 2
    c["target"][4] = -inf
    c["target"][5] = float("nan")
    path, n, token = _run_verify(c, dev_err=err)
    assert n[4].item() >= 1 and 0 <= token[4].item() < 500  # all the same weight
    assert token[5].item() in range(-1, 500)


@pytest.mark.parametrize("temp", [0.0, 0.7])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("what", [-float("inf"), float("nan")])
def test_verification_flags_rows_without_any_weight(what, f32, temp):
    """All tokens of such a row have the same weight (greedy: the first one is its maximum), and the error word
    says so; only where the walk comes by."""
    c = _verify_case(2, 3, 700, 4, "chain", f32, temp=[temp])
    c["parents"][:] = torch.tensor([-1, 0, 1])
    c["tokens"][:, 1] = torch.argmax(c["target"][:, 0].float(), -1).to(torch.int32)
    c["u"][:] = torch.tensor([0.0, 0.0, 0.5])
    c["s"] = torch.tensor([0.5, 0.0])
    c["target"][:, 2] = what  # never reached: node 2 is rejected
    c["tokens"][:, 2] = 699
    c["target"][:, 1, 699] = -float("inf")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    _check_verify(c, _run_verify(c, dev_err=err))
    assert err.item() == 0
    c["target"][:, 1] = what
    path, n, token = _run_verify(c, dev_err=err)
    _check_verify(c, (path, n, token))
    assert err.item() == 2 and n.tolist() == [2, 2]
    # node 2's token is rejected there (0.5 * 700 >= 1): of 699 weights the 350th is the first past 349.5
    assert token.tolist() == ([0, 0] if temp == 0 else [349, 0])


def test_verification_of_bad_tokens_and_unused_roots():
    c = _verify_case(3, 4, 100, 2, "star")
    c["tokens"][0, 1:] = torch.tensor([-1, 100, 2 ** 31 - 1], dtype=torch.int32)
    c["parents"][1] = -2
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = _run_verify(c, dev_err=err)
    _check_verify(c, got)
    assert err.item() == 4 and got[1][1].item() == 0 and got[2][1].item() == -1 and got[1][0].item() == 1


@pytest.mark.parametrize("b,node,parent", [(0, 0, 0), (1, 0, 3), (2, 3, 3), (2, 2, 4), (1, 4, 2 ** 31 - 1)])
def test_verification_flags_parents_that_are_no_earlier_node(b, node, parent):
    """Such a node counts as unused, a root of the kind leaves its sequence without a tree."""
    c = _verify_case(3, 5, 300, 6, "tree")
    c["parents"][:] = torch.tensor([-1, 0, 0, 1, 2])
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    _check_verify(c, _run_verify(c, dev_err=err))
    assert err.item() == 0
    c["parents"][b, node] = parent
    got = _run_verify(c, dev_err=err)
    _check_verify(c, got)
    assert err.item() == 4 and (got[1][b].item() == 0) == (node == 0)


def test_verification_at_the_ends_of_the_random_numbers():
    c = _verify_case(6, 6, 999, 4, "tree", draft=True)
    c["u"][:3] = 0.0  # accepted wherever the target has any weight
    c["u"][3:] = 1 - 2.0 ** -24
    c["s"] = torch.tensor([0.0, 1 - 2.0 ** -24, 0.5, 0.0, 1 - 2.0 ** -24, 0.5])
    _check_verify(c, _run_verify(c))
    c["u"][:] = float("nan")
    c["s"][:] = 2.0  # outside the range: still a token of the vocabulary
    _, n, token = _run_verify(c)
    assert (n == 1).all() and ((token >= 0) & (token < 999)).all()


def test_the_double_weights_bits():
    """e^-d of the double path to 6e-14.  Token 0 has the logit -d, token 1 the logit 0; a draft that is the target's
    distribution but for its last fp32 digits leaves p - q of about 2^-24 p after a rejection, and the
    draw between the two tokens changes where u passes r0 / (r0 + r1), which an error of w in p moves by at most
    2^24 of it (q is at least a step below p, and r1 moves less): 1e-6 on either side holds 6e-14."""
    getcontext().prec = 60
    n = 512
    d = (torch.rand(n, generator=_gen(3)).double() * 80).float()
    d[:8] = torch.tensor([2.0 ** -20, 1e-3, 0.0108, 0.0109, 0.3465, 0.3466, 0.6931, 0.6932])
    q = torch.zeros(n, 2, 3)
    u = torch.zeros(2, n)
    below = lambda p, steps: np.float32(p) * np.float32(1 - steps * 2.0 ** -23)  # noqa: E731
    for i in range(n):
        w = (-Decimal(d[i].item())).exp()
        p0, p1 = w / (1 + w), 1 / (1 + w)
        q[i, 0] = torch.tensor([below(p0, 2), below(p1, 2), 0.25])
        r0, r1 = p0 - Decimal(q[i, 0, 0].item()), p1 - Decimal(q[i, 0, 1].item())
        assert r0 > p0 * Decimal(2) ** -24 and r1 > p1 * Decimal(2) ** -24
        border = r0 / (r0 + r1)
        u[0, i], u[1, i] = float(border * (1 - Decimal("1e-6"))), float(border * (1 + Decimal("1e-6")))
    target = torch.zeros(n, 2, 3)
    target[:, :, 0] = -d[:, None]
    target[:, :, 2] = -1000.0
    par = torch.tensor([[-1, 0]] * n, dtype=torch.int32).cuda()
    tokens = torch.full((n, 2), 2, dtype=torch.int32).cuda()  # no weight left: rejected
    for side in range(2):
        _, count, token = sp.verify_tree(target.cuda(), tokens, par, torch.full((n, 2), 0.5).cuda(), u[side].cuda(),
                                         draft_probs=q.cuda())
        assert (count == 1).all() and (token == side).all(), (token != side).nonzero().flatten().tolist()


@pytest.mark.parametrize("draft", [False, True])
def test_verified_tokens_follow_the_target(draft):
    """60000 draws of the first new token over a small vocabulary: Pearson's statistic against the
    target's distribution stays below the 1 - 1e-6 quantile of chi-square with 11 degrees (49.9)."""
    V, T, n = 12, 4, 60000
    g = _gen(8)
    row = torch.randn(V, generator=g) * 1.5
    q = torch.softmax(row + torch.randn(V, generator=g), 0)
    par = torch.tensor([-1, 0, 0, 0], dtype=torch.int32)
    tokens = torch.zeros(n, T, dtype=torch.int32)
    if draft:
        tokens[:, 1:] = torch.multinomial(q.double(), n * 3, replacement=True, generator=g).view(n, 3).to(torch.int32)
    else:
        tokens[:, 1:] = torch.topk(q, 3)[1].to(torch.int32)
    target = row.expand(n, T, V).contiguous().cuda()
    path, count, token = sp.verify_tree(
        target, tokens.cuda(), par.expand(n, T).contiguous().cuda(), torch.rand(n, T, generator=g).cuda(),
        torch.rand(n, generator=g).cuda(), draft_probs=q.expand(n, T, V).contiguous().cuda() if draft else None)
    first = torch.where(count.cpu() > 1, tokens[torch.arange(n), path.cpu()[:, 1].clamp(min=0).long()], token.cpu())
    want = torch.softmax(row.double(), 0) * n
    seen = torch.bincount(first.long(), minlength=V).double()
    assert ((seen - want) ** 2 / want).sum().item() < 49.9


def test_verification_in_a_graph():
    c = _verify_case(4, 9, 5001, 5, "tree", temp=[0.9, 0.0])
    d = _gpu(c)
    call = lambda: sp.verify_tree(d["target"], d["tokens"], d["parents"], d["u"], d["s"], temperature=d["temp"])  # noqa: E731
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    other = _verify_case(4, 9, 5001, 6, "tree", temp=[0.9, 0.0])
    for k in ("target", "tokens", "parents", "u", "s"):
        d[k].copy_(other[k])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    _check_verify(other, got)


# --------------------------------------------------------------------------------------- commit
SLOT = ("slot_pos", "insert_step", "last_access", "access_count", "attn", "max_attn", "cumul", "prefill")
KINDS = dict(zip(SLOT, (np.int32,) * 4 + (np.float32,) * 2 + (np.float64, np.float32)))


def _commit_case(B, T, L, hkv, S, live, seed, W=None, score=True, longest=None, far=None):
    rng = np.random.default_rng(seed)
    far = far or 4 * S + 50
    st = {k: np.zeros((B, S), KINDS[k]) for k in SLOT}
    st["slot_pos"][:] = -1
    W = W or (far + T) // 32 + 2
    bits = np.zeros((B, W * 32), bool)
    step = rng.integers(5, 200, B).astype(np.int32)
    path, n = np.full((B, T), -1, np.int32), np.zeros(B, np.int32)
    for b in range(B):
        at, pos = rng.permutation(S)[:live], rng.permutation(far)[:live]
        st["slot_pos"][b, at] = pos
        bits[b, pos] = True
        st["insert_step"][b, at] = rng.integers(0, step[b], live)
        st["last_access"][b, at] = np.maximum(st["insert_step"][b, at], rng.integers(0, step[b] + 1, live))
        st["access_count"][b, at] = rng.integers(1, 9, live)
        for k in ("attn", "max_attn", "prefill"):
            st[k][b, at] = rng.random(live) ** 3
        st["cumul"][b, at] = np.round(rng.random(live) * 4) / 4  # ties
        n[b] = rng.integers(0 if b else 1, min(T, longest or T) + 1)
        path[b, : n[b]] = np.sort(np.concatenate([[0], 1 + rng.permutation(T - 1)])[: n[b]])
    words = (bits.reshape(B, W, 32).astype(np.uint64) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)
    state = {k: torch.from_numpy(v) for k, v in st.items()}
    state.update(posmap=torch.from_numpy(words.view(np.int32)), seq_step=torch.from_numpy(step),
                 next_pos=torch.full((B,), far, dtype=torch.int32), evlog=torch.full((B, 4 * S), -9, dtype=torch.int32),
                 evcount=torch.full((B,), 3, dtype=torch.int32))
    g = _gen(seed)
    rows = lambda r: torch.randn(L, B, hkv, r, 128, generator=g).to(BF)  # noqa: E731
    return {"state": state, "path": torch.from_numpy(path), "n": torch.from_numpy(n), "kd": rows(T), "vd": rows(T),
            "k": rows(S), "v": rows(S), "score": torch.rand(B, T, S + T, generator=g) ** 4 if score else None}


def _run_commit(c, evict=None, out=None, **kw):
    d = {k: v.cuda() for k, v in c.items() if torch.is_tensor(v)}
    st = sp.SlotState(**{k: v.cuda() for k, v in c["state"].items()})
    new = st.like() if out else None
    write = sp.commit_tree(st, d["path"], d["n"], d["kd"], d["vd"], d["k"], d["v"], node_score=d.get("score"),
                           evict=evict, out=new, **kw)
    return st, new if out else st, write, d["k"], d["v"]


def _check_commit(c, new, write, k, v, evict=None):
    spec = None if evict is None else (evict.policy, evict.capacity, evict.evict_every, evict.protect,
                                       evict.prefix_frac, evict.suffix_frac)
    if spec and evict.regime == "prefill":
        spec = None
    kw, vw = c["k"].clone(), c["v"].clone()
    got = {f: getattr(new, f).cpu().numpy() for f in c["state"]}
    for b in range(c["path"].shape[0]):
        st = {f: c["state"][f][b].numpy().copy() for f in SLOT}
        st.update(seq_step=int(c["state"]["seq_step"][b]), next_pos=int(c["state"]["next_pos"][b]), log=[])
        n, path = int(c["n"][b]), c["path"][b].tolist()
        slots = ref.commit(st, path, n, None if c["score"] is None else c["score"][b].numpy(), spec)
        assert write[b].tolist() == slots + [-1] * (len(path) - n), b
        for f in SLOT:
            assert np.array_equal(got[f][b], st[f]), (b, f)
        assert got["seq_step"][b] == st["seq_step"] and got["next_pos"][b] == st["next_pos"]
        assert got["evcount"][b] == 3 + len(st["log"])
        assert got["evlog"][b, 3:3 + len(st["log"])].tolist() == st["log"]
        held = sorted(int(p) for p in st["slot_pos"] if p >= 0)
        bits = np.unpackbits(got["posmap"][b].view(np.uint8), bitorder="little")
        assert np.flatnonzero(bits).tolist() == held
        for i, s in enumerate(slots):
            if s >= 0:
                kw[:, b, :, s], vw[:, b, :, s] = c["kd"][:, b, :, path[i]], c["vd"][:, b, :, path[i]]
    assert torch.equal(k.cpu(), kw) and torch.equal(v.cpu(), vw)


@pytest.mark.parametrize("B,T,L,hkv,S,live", [(1, 1, 1, 1, 4, 2), (3, 8, 2, 2, 70, 60), (2, 128, 1, 1, 700, 500), (5, 16, 3, 4, 1100, 1037),
                                              (4, 24, 28, 1, 40, 3), (2, 9, 2, 8, 513, 0), (2, 5, 1, 2, 5000, 4990)])
@pytest.mark.parametrize("score", [True, False])
@pytest.mark.parametrize("out", [True, False])
def test_commit_without_eviction(B, T, L, hkv, S, live, score, out):
    c = _commit_case(B, T, L, hkv, S, live, S + T, score=score, longest=S - live)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    old, new, write, k, v = _run_commit(c, out=out, dev_err=err)
    _check_commit(c, new, write, k, v)
    assert err.item() == 0
    if out:
        for f, t in c["state"].items():
            assert torch.equal(getattr(old, f).cpu(), t), f


@pytest.mark.parametrize("policy", ["lru", "h2o_faithful", "h2o", "snapkv", "snapkv_faithful", "adakv", "quest",
                                    "streamingllm"])
@pytest.mark.parametrize("protect,cap,every", [(True, 60, 8), (False, 60, 4), (True, 6, 2), (True, 64, 1)])
def test_commit_with_eviction(policy, protect, cap, every):
    evict = sp.EvictionSpec(policy=policy, capacity=cap, evict_every=every, protect=protect)
    for seed in range(3):
        c = _commit_case(4, 12, 2, 2, cap + 20, cap + 2, seed, longest=12)
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        _, new, write, k, v = _run_commit(c, evict, out=seed == 1, dev_err=err)
        _check_commit(c, new, write, k, v, evict)
        assert err.item() == 0


def test_commit_with_eviction_of_many_slots():
    evict = sp.EvictionSpec(policy="h2o_faithful", capacity=16000, evict_every=4)
    c = _commit_case(2, 6, 1, 1, 16384, 16010, 5)
    c["n"][:] = 6
    c["path"][:] = torch.arange(6)
    _, new, write, k, v = _run_commit(c, evict)
    _check_commit(c, new, write, k, v, evict)


def test_commit_in_the_prefill_regime_never_evicts():
    evict = sp.EvictionSpec(policy="lru", capacity=4, evict_every=1, regime="prefill")
    c = _commit_case(3, 6, 1, 1, 60, 30, 2)
    _, new, write, k, v = _run_commit(c, evict)
    _check_commit(c, new, write, k, v, evict)


def test_commit_equals_single_steps():
    """The same positions and scores appended one at a time by the single-step kernels."""
    c = _commit_case(3, 7, 1, 2, 90, 70, 4)
    c["n"][:] = torch.tensor([7, 3, 5], dtype=torch.int32)
    c["path"][:] = torch.arange(7)
    _, new, write, _, _ = _run_commit(c)
    L, st = capi.lib(), torch.cuda.current_stream().cuda_stream
    for b in range(3):
        one = {k: v[b:b + 1].cuda() for k, v in c["state"].items()}
        s = capi.State(1, 90, one["posmap"].shape[1], *[one[k].data_ptr() for k in SLOT + ("posmap",)])
        cfg = capi.EvictCfg(90, 8, 0, 0, 0, 0, 0)
        cur, ws = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        where = []
        for i in range(int(c["n"][b])):
            capi.check(L.kvbp_append_evict(st, capi.C.byref(s), capi.C.byref(cfg), one["seq_step"].data_ptr(),
                                           one["next_pos"].data_ptr(), cur.data_ptr(), ws.data_ptr(), None, None, 0,
                                           one["evlog"].data_ptr(), one["evcount"].data_ptr(), 360, None, None), "append")
            where.append(ws.item())
            step = c["score"][b, i, :90].clone()
            for j, slot in enumerate(where):
                step[slot] = c["score"][b, i, 90 + j]
            step = step.cuda().view(1, 90).contiguous()
            capi.check(L.kvbp_score_update(st, capi.C.byref(s), one["seq_step"].data_ptr(), step.data_ptr(), None), "update")
        assert write[b, : len(where)].tolist() == where
        for k in one:
            assert torch.equal(getattr(new, k)[b:b + 1], one[k]), k


def test_commit_of_bad_paths_and_a_full_cache():
    c = _commit_case(4, 6, 1, 1, 30, 27, 3)
    c["n"][:] = torch.tensor([6, 9, -2, 4], dtype=torch.int32)
    c["path"][:] = torch.arange(6)
    c["path"][1, 2] = 6  # ends there
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    _, new, write, k, v = _run_commit(c, dev_err=err)
    assert err.item() == (1 | 4)  # three slots for six nodes; bad counts and nodes
    c["n"][:] = torch.tensor([6, 2, 0, 4], dtype=torch.int32)
    _check_commit(c, new, write, k, v)
    # positions past the bitmap
    c = _commit_case(1, 3, 1, 1, 30, 20, 3, far=100, W=4)
    c["state"]["next_pos"][:] = 127
    c["n"][:] = 3
    c["path"][:] = torch.arange(3)
    err.zero_()
    evict = sp.EvictionSpec(policy="lru", capacity=18, evict_every=1, protect=False)
    _, new, write, _, _ = _run_commit(c, evict, dev_err=err)
    assert err.item() == 4 and (new.slot_pos >= 0).sum().item() == 18


def test_commit_flags_nan_scores():
    c = _commit_case(1, 3, 1, 1, 30, 20, 3)
    c["n"][:] = 2
    c["path"][0, :2] = torch.tensor([0, 1], dtype=torch.int32)
    c["score"][0, 1, 32] = float("nan")  # node 2 is not on the path
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    c["score"][0, 0, int((c["state"]["slot_pos"][0] >= 0).nonzero()[0])] = float("nan")
    _run_commit(c, dev_err=err)
    assert err.item() == 2


def test_commit_in_a_graph():
    """Two states in turn: each replay takes the step from one to the other, and back."""
    c = _commit_case(3, 8, 2, 2, 80, 64, 7)
    evict = sp.EvictionSpec(policy="h2o_faithful", capacity=60, evict_every=4)
    d = {k: v.cuda() for k, v in c.items() if torch.is_tensor(v)}
    st = sp.SlotState(**{k: v.cuda() for k, v in c["state"].items()})
    new = st.like()
    call = lambda: sp.commit_tree(st, d["path"], d["n"], d["kd"], d["vd"], d["k"], d["v"], node_score=d["score"],  # noqa: E731
                                  evict=evict, out=new)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        write = call()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    _check_commit(c, new, write, d["k"], d["v"], evict)
