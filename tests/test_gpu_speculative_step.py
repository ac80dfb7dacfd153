"""The speculative decoding operators together, as a decoder uses them: tree forward over the engine's
slots (its weights, projections, RoPE and norms), verification, commit; against the engine's own steps."""

import numpy as np
import pytest
import torch

import spec_ref as ref
from kvcacheboundaryprotection_b200 import build, capi, speculative as sp
from kvcacheboundaryprotection_b200.config import get_config
from kvcacheboundaryprotection_b200.engine import CappedKVEngine, EvictionSpec
from kvcacheboundaryprotection_b200.weights import init_weights

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _lib():
    build.build()


def _tree_forward(eng, tokens, parents, depth, kd, vd, node_score):
    """Logits [B, T, vocab] of every node; each layer's drafted K and V to kd / vd [L, B, Hkv, T, 128]."""
    c, L, st, err = eng.cfg, capi.lib(), eng.stream, eng.dev_err.data_ptr()
    B, T = tokens.shape
    R, H, D = B * T, c.hidden, c.head_dim
    e = lambda *s: torch.empty(*s, dtype=BF, device="cuda")  # noqa: E731

    def gemm(epi, N, K, w, x, out):
        capi.check(L.kvbp_prefill_gemm(st, epi, R, N, K, w.data_ptr(), x.data_ptr(), x.stride(0), out.data_ptr(),
                                       out.stride(0), err), "prefill_gemm")

    def norm(delta, w):
        capi.check(L.kvbp_add_rmsnorm(st, R, H, h.data_ptr(), None if delta is None else delta.data_ptr(), w.data_ptr(),
                                      x.data_ptr(), c.eps), "rmsnorm")

    h, x, qkv, q = e(R, H), e(R, H), e(R, c.qkv_dim), e(B, T, c.n_heads, D)
    o, act, down, logits = e(R, H), e(R, c.ffn), e(R, H), e(R, c.vocab)
    pos = (eng.next_pos[:, None] + depth).to(torch.int32).reshape(-1).contiguous()
    node = torch.arange(T, dtype=torch.int32, device="cuda").repeat(B)
    capi.check(L.kvbp_embed(st, R, c.vocab, H, eng.embed_w.data_ptr(), tokens.data_ptr(), h.data_ptr(), err), "embed")
    delta = None
    for li, w in enumerate(eng.layers):
        norm(delta, w["in_norm"])
        gemm(0, c.qkv_dim, H, w["w_qkv"], x, qkv)
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        capi.check(L.kvbp_qkv_rope_scatter(st, R, T, c.n_heads, c.n_kv_heads, D, T, qkv.data_ptr(), c.qkv_dim,
                                           ptr(w["b_qkv"]), ptr(w["q_norm"]), ptr(w["k_norm"]), c.eps,
                                           eng.inv_freq.data_ptr(), pos.data_ptr(), node.data_ptr(), q.data_ptr(),
                                           kd[li].data_ptr(), vd[li].data_ptr(), err), "scatter")
        att = sp.tree_attend(q, eng.kc[li], eng.vc[li], kd[li], vd[li], parents, slot_pos=eng.slot_pos,
                             node_score=node_score, dev_err=eng.dev_err)
        gemm(0, H, c.n_heads * D, w["w_o"], att.view(R, -1), o)
        norm(o, w["post_norm"])
        gemm(2, 2 * c.ffn, H, w["w_gu"], x, act)
        gemm(0, H, c.ffn, w["w_down"], act, down)
        delta = down
    norm(delta, eng.final_norm)
    gemm(0, c.vocab, H, eng.lm_w, x, logits)
    return logits.view(B, T, c.vocab)


def _engines(every, B=3, P=70, cap=48, steps=24):
    cfg = get_config("parity-qwen2")
    w = init_weights(cfg, seed=1)
    prompts = torch.from_numpy(np.random.default_rng(2).integers(0, cfg.vocab, (B, P)).astype(np.int32))
    out = []
    for _ in range(2):
        eng = CappedKVEngine(cfg, w, batch=B, evict=EvictionSpec("h2o_faithful", cap, every, True), max_prompt_len=P,
                             max_new_tokens=steps)
        eng.prefill(prompts)
        out.append(eng)
    return out


def _close(got, want):
    """Two layers' bf16 activations, each rounded at some seven places on the way (half a step is 2^-8):
    14 * 2^-8 of the whole, in the 2-norm."""
    got, want = got.double(), want.double()
    assert (got - want).norm() <= 14 * 2.0 ** -8 * want.norm(), ((got - want).norm() / want.norm()).item()


def test_speculative_steps_equal_the_engines_single_steps():
    """Drafts that hold the engine's own next tokens beside others, accepted by the random numbers: after
    every commit the slots are those of the single steps, with the same rows, scores and logits."""
    one, spec = _engines(every=64)
    B, T = one.B, 6
    parents = torch.tensor([[-1, 0, 0, 1, 1, 4]] * B, dtype=torch.int32, device="cuda")
    depth = torch.tensor([0, 1, 1, 2, 2, 3], device="cuda")
    state = sp.SlotState.of(spec)
    kd = torch.empty(one.cfg.n_layers, B, one.cfg.n_kv_heads, T, 128, dtype=BF, device="cuda")
    vd = torch.empty_like(kd)
    score = torch.empty(B, T, spec.S + T, device="cuda")
    for it in range(4):
        # the engine's three or four next tokens: the root is forwarded first
        n_new = 4 if it % 2 == 0 else 2
        toks, logits = [], []
        for _ in range(n_new):
            toks.append(one.tokens.clone())
            one.run_step(use_graph=False)
            logits.append(one.logits.clone())
        nxt = one.tokens.clone()
        other = (toks[0] + 1) % one.cfg.vocab
        fill = lambda i: toks[i] if i < n_new else nxt  # noqa: E731
        # the path 0 - 1 - 4 - 5 holds the engine's tokens; 2 and 3 are decoys
        tokens = torch.stack([toks[0], fill(1), other, other, fill(2), fill(3)], 1).contiguous()
        u = torch.tensor([0, 0, 1 - 2.0 ** -24, 1 - 2.0 ** -24, 0, 0], device="cuda").repeat(B, 1)
        if n_new == 2:
            u[:, 4:] = 1 - 2.0 ** -24  # only node 1 passes
        score.zero_()
        got = _tree_forward(spec, tokens, parents, depth, kd, vd, score)
        path, n, _ = sp.verify_tree(got, tokens, parents, u, torch.full((B,), 0.5, device="cuda"))
        way = [0, 1, 4, 5][:n_new]
        assert n.tolist() == [n_new] * B and path[:, :n_new].tolist() == [way] * B
        write = sp.commit_tree(state, path, n, kd, vd, spec.kc, spec.vc, node_score=score,
                               evict=EvictionSpec("h2o_faithful", 48, 64, True), dev_err=spec.dev_err)
        one.apply_pending_scores()
        for name in ("slot_pos", "insert_step", "posmap", "seq_step", "next_pos", "evcount"):
            assert torch.equal(getattr(one, name), getattr(spec, name)), (it, name)
        assert (write[:, :n_new] >= 0).all()
        for i, node in enumerate(way):
            _close(got[:, node], logits[i])
        live = one.slot_pos >= 0
        for name in ("attn_s", "max_attn", "cumul"):
            _close(getattr(spec, name)[live], getattr(one, name)[live])
        where = live[:, None, :, None]
        for li in range(one.cfg.n_layers):
            _close(spec.kc[li] * where, one.kc[li] * where)
            _close(spec.vc[li] * where, one.vc[li] * where)
    one.check_device_errors()
    spec.check_device_errors()


def test_speculative_steps_with_eviction_in_a_graph():
    """Greedy steps with eviction, one captured graph replayed: the capacity holds, positions go on without
    a gap, and every chosen token is the logits' first maximum."""
    _, eng = _engines(every=4, steps=60)
    B, T, cap = eng.B, 5, 48
    c = eng.cfg
    parents = torch.tensor([[-1, 0, 0, 1, 2]] * B, dtype=torch.int32, device="cuda")
    depth = torch.tensor([0, 1, 1, 2, 2], device="cuda")
    kd = torch.empty(c.n_layers, B, c.n_kv_heads, T, 128, dtype=BF, device="cuda")
    vd = torch.empty_like(kd)
    score = torch.empty(B, T, eng.S + T, device="cuda")
    state = sp.SlotState.of(eng)
    tokens = torch.zeros(B, T, dtype=torch.int32, device="cuda")
    u = torch.rand(B, T, device="cuda")
    spec = EvictionSpec("h2o_faithful", cap, 1, True)  # every commit
    cold = torch.zeros(B, device="cuda")

    def step():
        score.zero_()
        tokens[:, 0] = eng.tokens
        logits = _tree_forward(eng, tokens, parents, depth, kd, vd, score)
        path, n, nxt = sp.verify_tree(logits, tokens, parents, u, cold, temperature=cold, dev_err=eng.dev_err)
        sp.commit_tree(state, path, n, kd, vd, eng.kc, eng.vc, node_score=score, evict=spec, dev_err=eng.dev_err)
        eng.tokens.copy_(nxt)
        return logits, path, n, nxt

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits, path, n, nxt = step()
    for i in range(8):
        before = eng.next_pos.clone()
        tokens[:, 1:] = torch.randint(0, c.vocab, (B, T - 1), dtype=torch.int32, device="cuda")
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(eng.next_pos, before + n)
        held = (eng.slot_pos >= 0).sum(1)
        assert (held == cap).all()
        last = path[torch.arange(B), n.long() - 1].long()
        assert torch.equal(nxt.long(), logits[torch.arange(B), last].float().argmax(-1))
    eng.check_device_errors()


SLOT = {"slot_pos": "slot_pos", "insert_step": "insert_step", "last_access": "last_access", "access_count": "access_count",
        "attn": "attn_s", "max_attn": "max_attn", "cumul": "cumul", "prefill": "prefill_s"}


def _snapshot(eng, b):
    """Sequence b of an engine as ``ref.commit`` takes it."""
    st = {k: getattr(eng, v)[b].cpu().numpy().copy() for k, v in SLOT.items()}
    st.update(seq_step=int(eng.seq_step[b]), next_pos=int(eng.next_pos[b]), log=[])
    return st


def _equal(eng, b, st, logged):
    for k, v in SLOT.items():
        assert np.array_equal(getattr(eng, v)[b].cpu().numpy(), st[k]), (b, k)
    assert int(eng.seq_step[b]) == st["seq_step"] and int(eng.next_pos[b]) == st["next_pos"]
    assert eng.evlog[b, logged: int(eng.evcount[b])].tolist() == st["log"]


def _commits(eng, state, T, steps, seed, kd, vd, longest):
    """``steps`` commits of random paths with random scores, each checked against ``ref.commit``."""
    g, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    ev = eng.ev
    spec = (ev.policy, ev.capacity, ev.evict_every, ev.protect, ev.prefix_frac, ev.suffix_frac)
    lost = 0
    for it in range(steps):
        n = torch.tensor([longest if it % 3 else 1 + int(rng.integers(longest)) for _ in range(eng.B)], dtype=torch.int32)
        path = torch.full((eng.B, T), -1, dtype=torch.int32)
        for b in range(eng.B):
            path[b, : n[b]] = torch.from_numpy(np.sort(np.concatenate([[0], 1 + rng.permutation(T - 1)])[: n[b]]))
        score = torch.rand(eng.B, T, eng.S + T, generator=g) ** 4
        before = [_snapshot(eng, b) for b in range(eng.B)]
        logged = eng.evcount.tolist()
        write = sp.commit_tree(state, path.cuda(), n.cuda(), kd, vd, eng.kc, eng.vc, node_score=score.cuda(), evict=ev)
        for b in range(eng.B):
            slots = ref.commit(before[b], path[b].tolist(), int(n[b]), score[b].numpy(), spec)
            assert write[b].tolist() == slots + [-1] * (T - int(n[b])), (it, b)
            _equal(eng, b, before[b], logged[b])
            for i, s in enumerate(slots):
                lost += s < 0
                if s >= 0:
                    assert torch.equal(eng.kc[:, b, :, s], kd[:, b, :, path[b, i]])
                    assert torch.equal(eng.vc[:, b, :, s], vd[:, b, :, path[b, i]])
    return lost


@pytest.mark.parametrize("policy,every,longest", [("h2o_faithful", 8, 3), ("lru", 4, 5), ("streamingllm", 1, 2)])
def test_commits_at_the_engines_own_cadence(policy, every, longest):
    """Steps of several tokens over many evictions of one cadence: an engine with slots for the longest path
    loses none (without them the step before an eviction finds no free slot)."""
    B, T, cap = 3, 6, 48
    cfg = get_config("parity-qwen2")
    w = init_weights(cfg, seed=1)
    kd = torch.randn(cfg.n_layers, B, cfg.n_kv_heads, T, 128, device="cuda").to(BF)
    vd = torch.randn_like(kd)
    for extra in (longest - 1, 0):
        eng = CappedKVEngine(cfg, w, batch=B, evict=EvictionSpec(policy, cap, every, True), max_prompt_len=70,
                             max_new_tokens=80, extra_slots=extra)
        assert eng.S == cap + every + extra
        eng.synthetic_prefill(70, seed=3)
        lost = _commits(eng, sp.SlotState.of(eng), T, 14, 5, kd, vd, longest)
        if extra:
            # a victim may be among the newest, but no entry goes without a slot
            eng.check_device_errors()
        else:
            assert lost
            with pytest.raises(capi.KVBPError, match="slot"):
                eng.check_device_errors()


def _arrays(eng):
    return [getattr(eng, n).clone() for n in (*SLOT.values(), "posmap", "seq_step", "next_pos", "evcount", "evlog",
                                              "upd_pending", "step_score", "tokens", "kc", "vc")]


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("graph_steps", [False, True])
def test_commits_between_the_engines_own_steps(captured, graph_steps):
    """run_step leaves its scores pending: a commit (eager, or captured and replayed) applies them first, once,
    and the next run_step starts from the committed state.  Against the plain sequence with the scores applied
    by hand and the commit by ``ref.commit``."""
    B, T, n = 3, 5, 3
    cfg = get_config("parity-qwen2")
    w = init_weights(cfg, seed=1)
    engs = []
    for _ in range(2):
        eng = CappedKVEngine(cfg, w, batch=B, evict=EvictionSpec("h2o_faithful", 48, 4, True), max_prompt_len=70,
                             max_new_tokens=60, extra_slots=n - 1)
        eng.synthetic_prefill(70, seed=3)
        if graph_steps:
            eng.capture()
        engs.append(eng)
    one, plain = engs
    ev = one.ev
    spec = (ev.policy, ev.capacity, ev.evict_every, ev.protect, ev.prefix_frac, ev.suffix_frac)
    kd = torch.randn(cfg.n_layers, B, cfg.n_kv_heads, T, 128, device="cuda").to(BF)
    vd = torch.randn_like(kd)
    path = torch.tensor([[0, 2, 3, -1, -1]] * B, dtype=torch.int32, device="cuda")
    count = torch.full((B,), n, dtype=torch.int32, device="cuda")
    score = torch.zeros(B, T, one.S + T, device="cuda")
    state = sp.SlotState.of(one)
    call = lambda: sp.commit_tree(state, path, count, kd, vd, one.kc, one.vc, node_score=score, evict=ev)  # noqa: E731
    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            write = call()
    for it in range(7):
        for eng in engs:
            for _ in range(it % 3):  # none, one or two steps between commits
                eng.run_step(use_graph=graph_steps)
        score.copy_(torch.rand(B, T, one.S + T, generator=torch.Generator().manual_seed(it)) ** 4)
        if captured:
            graph.replay()
        else:
            write = call()
        if it % 3:  # the plain sequence
            capi.check(capi.lib().kvbp_score_update(plain.stream, capi.C.byref(plain._state), plain.seq_step.data_ptr(),
                                                    plain.step_score.data_ptr(), plain.dev_err.data_ptr()), "score_update")
            plain.upd_pending.zero_()
            plain._forwarded = False
        for b in range(B):
            st = _snapshot(plain, b)
            logged = int(plain.evcount[b])
            slots = ref.commit(st, path[b].tolist(), n, score[b].cpu().numpy(), spec)
            assert write[b].tolist() == slots + [-1] * (T - n), (it, b)
            _equal(one, b, st, logged)
        sp.commit_tree(sp.SlotState.of(plain), path, count, kd, vd, plain.kc, plain.vc, node_score=score, evict=ev)
        for x, y in zip(_arrays(one), _arrays(plain)):
            assert torch.equal(x, y), it
        assert int(one.upd_pending.sum()) == 0 and float(one.step_score.abs().sum()) == 0
    for eng in engs:
        eng.run_step(use_graph=graph_steps)
        eng.check_device_errors()
    for x, y in zip(_arrays(one), _arrays(plain)):
        assert torch.equal(x, y)


def test_an_engine_refuses_a_negative_number_of_slots():
    cfg = get_config("parity-qwen2")
    with pytest.raises(ValueError, match="extra_slots"):
        CappedKVEngine(cfg, {}, batch=1, evict=EvictionSpec("lru", 8, 4), max_prompt_len=8, max_new_tokens=4, extra_slots=-1)
