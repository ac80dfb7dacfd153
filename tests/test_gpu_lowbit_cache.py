"""The 4-bit cache under the framework's other kernels: eviction over its slots, and prefill
attention over rows read back from it."""

import math

import pytest
import torch

import lowbit_ref as ref
from kvcacheboundaryprotection_b200 import build, capi, lowbit
from test_gpu_evict import Driver
from test_gpu_lowbit_values import _bound
from test_gpu_prefill import _run, torch_reference

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HQ, HKV = 8, 2


@pytest.fixture(scope="module", autouse=True)
def _lib():
    build.build()


def _slots_of(gather_src, P):
    """gather_src [B, S] (prompt position per slot) the other way round: slot per position, -1
    where the position was evicted, as kv4_append takes it."""
    slots = torch.full((gather_src.shape[0], P), -1, dtype=torch.int32, device=gather_src.device)
    b, s = (gather_src >= 0).nonzero(as_tuple=True)
    slots[b, gather_src[b, s].long()] = s.to(torch.int32)
    return slots


def _rows_at(pool, table, b, slots):
    """The 144 bytes of each slot and head as (codes, scales) of K and V, flat."""
    page = pool.shape[2] * 16
    pg, at = table[b][slots // page].long(), slots % page
    return torch.cat([torch.cat([c[pg, :, at].double(), s[pg, :, at]], -1) for c, s in ref.decode(pool)], -1)


@pytest.mark.parametrize("policy", ["h2o_faithful", "snapkv", "lru"])
@pytest.mark.parametrize("evict_every,protect", [(1, True), (4, False)])
def test_eviction_over_the_slots_of_a_4_bit_cache(policy, evict_every, protect):
    """Prompt, step-0 eviction and compaction, then decode steps with eviction: slot_pos, write_slot
    and step_score mean the same with pages underneath.  Every step's output and scores are the
    64-bit ones of the live slots, and each live slot holds the row of the position it names."""
    B, P, cap, steps, page = 3, 90, 48, 24, 16
    n_pre, n_suf = capi.protection_sizes(cap, 0.1, 0.2) if protect else (0, 0)
    cfg = capi.EvictCfg(cap, evict_every, capi.policy_id(policy), int(protect), n_pre, n_suf, 1)
    S = cap + evict_every + 3
    D = Driver(B, S, (P + steps + 2 + 31) // 32, P + steps + 2, steps, cfg)
    g = torch.Generator().manual_seed(5)
    width = (S + page - 1) // page
    table = torch.randperm(B * width, generator=g).to(torch.int32).view(B, width).cuda()
    pool = lowbit.kv4_pool(B * width, HKV, page)
    freq = (1e6 ** (-torch.arange(64) / 64.0)).float().cuda()
    qkv = torch.randn(B, P + steps, (HQ + 2 * HKV) * 128, generator=g).to(BF).cuda()
    # every position's row, as stored in a cache that evicts nothing
    whole_w = (P + steps + page - 1) // page
    whole_t = torch.arange(B * whole_w, dtype=torch.int32).view(B, whole_w).cuda()
    whole = lowbit.kv4_pool(B * whole_w, HKV, page)
    every = torch.arange(P + steps, dtype=torch.int32).repeat(B).cuda()
    lowbit.kv4_append(whole, whole_t, qkv.flatten(0, 1), every, n_heads=HQ, positions=every, inv_freq=freq)

    src = D.prefill(P, None if policy == "lru" else torch.rand(B, P, generator=g))
    slots = _slots_of(src, P)
    pos = torch.arange(P, dtype=torch.int32).repeat(B).cuda()
    lowbit.kv4_append(pool, table, qkv[:, :P].reshape(B * P, -1), slots.view(-1), n_heads=HQ, positions=pos, inv_freq=freq,
                      dev_err=D.err)
    lens = torch.full((B,), S, dtype=torch.int32).cuda()
    for t in range(steps):
        D.append_evict()
        new = qkv[torch.arange(B), P + t]
        assert (D.cur_pos == P + t).all()
        q = lowbit.kv4_append(pool, table, new, D.write_slot, n_heads=HQ, positions=D.cur_pos, inv_freq=freq, dev_err=D.err)
        out = lowbit.kv4_attend(pool, table, lens, q, slot_pos=D.slot_pos, step_score=D.step_score, dev_err=D.err)
        want, score, bound, drel, _ = _bound(pool.cpu(), table, lens, q, D.slot_pos, 1 / math.sqrt(128))
        assert ((out.cpu().double() - want).abs() <= bound).all()
        got = D.step_score.cpu().double()
        assert ((got - score[:, :S]).abs() <= (drel[:, None] + 2.0 ** -20) * score[:, :S] + 2.0 ** -60).all()
        assert (got[D.slot_pos.cpu() < 0] == 0).all()
        D.score_update()
        assert not D.step_score.any() and int((D.slot_pos >= 0).sum(1).max()) <= cap + evict_every
    assert int(D.err) == 0, capi.decode_dev_errors(int(D.err))
    assert int(D.evcount.min()) >= P - cap + steps - evict_every
    host, host_whole = pool.cpu(), whole.cpu()
    for b in range(B):
        live = (D.slot_pos[b].cpu() >= 0).nonzero()[:, 0]
        a = _rows_at(host, table.cpu(), b, live)
        w = _rows_at(host_whole, whole_t.cpu(), b, D.slot_pos[b].cpu()[live].long())
        assert torch.equal(a, w)


@pytest.mark.parametrize("P,hq,hkv,page", [(1, 4, 2, 16), (129, 8, 2, 48), (700, 28, 4, 64)])
def test_prefill_attention_over_rows_read_back(P, hq, hkv, page):
    """kv4_gather(heads_first=True) is the layout that the prefill attention reads: a prompt kept in
    4 bits, attended as bf16."""
    g = torch.Generator().manual_seed(P)
    qkv = torch.randn(P, (hq + 2 * hkv) * 128, generator=g).to(BF).cuda()
    width = (P + page - 1) // page
    table = torch.randperm(width + 3, generator=g)[:width].to(torch.int32)[None].cuda()
    pool = lowbit.kv4_pool(width + 3, hkv, page)
    pos = torch.arange(P, dtype=torch.int32).cuda()
    q = lowbit.kv4_append(pool, table, qkv, pos, n_heads=hq, positions=pos,
                          inv_freq=(1e6 ** (-torch.arange(64) / 64.0)).float().cuda())
    k, v = lowbit.kv4_gather(pool, table, pos, heads_first=True)
    assert k.shape == (hkv, P, 128) and k.is_contiguous() and v.is_contiguous()
    for got, rows in zip((k, v), ref.values(pool.cpu())):
        want = rows[table[0].cpu().long()].transpose(0, 1).reshape(hkv, -1, 128)[:, :P]
        assert torch.equal(got.cpu(), want.float().to(BF))
    colmax = torch.zeros(P, device="cuda")
    out = _run(q, k, v, colmax)
    want, want_col = torch_reference(q, k, v)
    d = (out.float() - want).abs()
    assert d.max().item() <= 1.6e-2 and (out.float() == want).float().mean().item() >= 0.97
    rel = (colmax - want_col).abs() / want_col.clamp_min(1e-30)
    assert (rel <= 1e-5).float().mean().item() >= 0.97 and rel.max().item() <= 2e-2


@pytest.mark.parametrize("pages", [0, 150])
def test_decode_steps_with_eviction_as_a_graph(pages):
    """One captured step (bookkeeping, append, attention with the score, score update), replayed:
    the eager run's outputs, slots, scores and cache, in the short and the streaming form."""
    B, P, cap, steps, page = 4, 40, 32, 20, 16
    cfg = capi.EvictCfg(cap, 2, capi.policy_id("h2o_faithful"), 0, 0, 0, 1)
    width = (cap + 5 + page - 1) // page
    S = cap + 5 if not pages else pages * page  # more slots than the one-launch form takes
    g = torch.Generator().manual_seed(9)
    table = torch.full((B, max(width, pages)), -1, dtype=torch.int32)
    table[:, :width] = torch.randperm(B * width, generator=g).view(B, width)
    table = table.cuda()
    qkv = torch.randn(P + steps, B, (HQ + 2 * HKV) * 128, generator=g).to(BF).cuda()
    freq = (1e6 ** (-torch.arange(64) / 64.0)).float().cuda()
    scores = torch.rand(B, P, generator=g)
    lens = torch.full((B,), cap + 5, dtype=torch.int32).cuda()

    def start():
        D = Driver(B, S, (P + steps + 2 + 31) // 32, P + steps + 2, steps, cfg)
        pool = lowbit.kv4_pool(B * width, HKV, page)
        slots = _slots_of(D.prefill(P, scores), P)
        pos = torch.arange(P, dtype=torch.int32).repeat(B).cuda()
        lowbit.kv4_append(pool, table, qkv[:P].transpose(0, 1).reshape(B * P, -1), slots.view(-1), n_heads=HQ,
                          positions=pos, inv_freq=freq, dev_err=D.err)
        return D, pool

    def step(D, pool, row):
        D.append_evict()
        q = lowbit.kv4_append(pool, table, row, D.write_slot, n_heads=HQ, positions=D.cur_pos, inv_freq=freq, dev_err=D.err)
        out = lowbit.kv4_attend(pool, table, lens, q, slot_pos=D.slot_pos, step_score=D.step_score, dev_err=D.err)
        D.score_update()
        return out

    D, pool = start()
    outs = [step(D, pool, qkv[P + t]) for t in range(steps)]
    G, gpool = start()
    row = qkv[P].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(G, gpool, row)
    for t in range(steps):
        row.copy_(qkv[P + t])
        graph.replay()
        assert torch.equal(out, outs[t]), t
    assert torch.equal(pool, gpool) and int(D.err) == 0 and int(G.err) == 0
    assert all(torch.equal(a, b) for a, b in zip(D.metadata(), G.metadata()))
