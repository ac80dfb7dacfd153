"""Cases for the operators of speculative decoding over the capped cache: attention of a tree of
drafted tokens over the slots, verification of the drafted tokens against the target's
probabilities, and the commit of the accepted path into the slots.

``run`` computes a case either in its plain form (elementary torch operations) or, where ``own``
is true, through the framework's public calls.

A tree is ``parents`` [sequences, nodes]: node 0 is the root (parent -1), every other node's
parent is an earlier node; a parent below -1 marks an unused node.

Attention.  Node t of a sequence sees the live slots of its cache (s < lens, slot_pos >= 0) and, of
the drafted keys, its ancestors and itself; the eviction score of (node, key) is the largest
probability over the heads, max-accumulated.

Verification.  The nodes are walked in order; a node whose parent is the last accepted one is
tested: its token x is accepted when u * q(x) * R < r(x), where r starts as the target's
distribution at that parent (R its sum) and q is the distribution that x was drawn from (1 at x
where the draft is not random).  A rejection leaves r <- max(r / R - q, 0).  At the end one token
is drawn from r of the last accepted node: the first x whose running sum exceeds u * R.
Temperature 0: x is accepted when it is the row's first largest, and that token ends the path.

Commit.  The path's nodes are appended in order, each into the lowest free slot, with the score
update of its step; where the step counter passes a multiple of ``evict_every`` the policy's
victims are freed down to the capacity; K and V of what stays are copied from the drafts.
"""

import math

import numpy as np
import torch

own = False

DIM = 128
DEV = "cuda"


# ---------------------------------------------------------------------------- the cases
def listed():
    return [
        # one sequence, a short cache and a small tree: the smallest attention call
        {"name": "attend_1x8x256", "op": "attend", "batch": 1, "nodes": 8, "heads": 16, "kv_heads": 2, "slots": 256,
         "tree": "tree", "lens": "full", "masked": True, "score": True},
        # sixteen capped sequences with freed slots and the eviction score of every node
        {"name": "attend_16x16x1032", "op": "attend", "batch": 16, "nodes": 16, "heads": 28, "kv_heads": 4,
         "slots": 1032, "tree": "tree", "lens": "full", "masked": True, "score": True},
        # a large batch with short drafted chains: streaming the cache is all there is
        {"name": "attend_64x5x4104", "op": "attend", "batch": 64, "nodes": 5, "heads": 32, "kv_heads": 8,
         "slots": 4104, "tree": "chain", "lens": "full", "masked": True, "score": False},
        # sequences of very different lengths (an empty one among them), an odd number of nodes
        {"name": "attend_ragged_12x33", "op": "attend", "batch": 12, "nodes": 33, "heads": 28, "kv_heads": 4,
         "slots": 32701, "tree": "tree", "lens": "ragged", "masked": False, "score": False},
        # one long sequence and a large tree: as much arithmetic as memory
        {"name": "attend_1x64x131071", "op": "attend", "batch": 1, "nodes": 64, "heads": 32, "kv_heads": 8,
         "slots": 131071, "tree": "tree", "lens": "full", "masked": False, "score": False},
        # one sequence's drafted chain, sampled: the latency of a few rows of the vocabulary
        {"name": "verify_1x6x151936", "op": "verify", "batch": 1, "nodes": 6, "vocab": 151936, "tree": "chain",
         "temperature": 1.0, "draft": True, "f32": False},
        # greedy decoding of sixteen sequences
        {"name": "verify_greedy_16x16x152064", "op": "verify", "batch": 16, "nodes": 16, "vocab": 152064,
         "tree": "tree", "temperature": 0.0, "draft": False, "f32": False},
        # the most likely tokens as candidates, an odd vocabulary, 32-bit logits
        {"name": "verify_24x20x50257", "op": "verify", "batch": 24, "nodes": 20, "vocab": 50257, "tree": "tree",
         "temperature": 0.7, "draft": False, "f32": True},
        # a large batch of trees drawn from a draft model's distributions
        {"name": "verify_64x32x152064", "op": "verify", "batch": 64, "nodes": 32, "vocab": 152064, "tree": "tree",
         "temperature": 0.8, "draft": True, "f32": False},
        # one sequence's accepted chain into 36 layers: latency
        {"name": "commit_1x8x256", "op": "commit", "batch": 1, "nodes": 8, "layers": 36, "kv_heads": 2,
         "capacity": 256, "every": 8, "policy": "h2o_faithful", "score": True},
        # sixteen capped sequences
        {"name": "commit_16x16x1024", "op": "commit", "batch": 16, "nodes": 16, "layers": 28, "kv_heads": 4,
         "capacity": 1024, "every": 8, "policy": "h2o_faithful", "score": True},
        # a large batch without scores
        {"name": "commit_64x24x1000", "op": "commit", "batch": 64, "nodes": 24, "layers": 28, "kv_heads": 4,
         "capacity": 1000, "every": 16, "policy": "lru", "score": False},
    ]


HEADS = [(28, 4), (16, 2), (32, 8), (8, 2), (7, 1), (8, 8), (24, 4), (8, 1)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "verify", "verify", "commit"])
    heads, kv = rng.choice(HEADS)
    tree = rng.choice(["tree", "tree", "chain"])
    if op == "attend":
        batch, nodes = _log(rng, 1, 100), _log(rng, 1, 128)
        most = min(131072, 2000000 // (batch * kv), 260000000 // (batch * nodes * heads))
        slots = _log(rng, 1, max(2, most))
        masked = rng.random() < 0.5
        return {"op": op, "batch": batch, "nodes": nodes, "heads": heads, "kv_heads": kv, "slots": slots, "tree": tree,
                "lens": rng.choice(["full", "ragged"]), "masked": masked, "score": masked and rng.random() < 0.6}
    if op == "verify":
        batch, vocab = _log(rng, 1, 64), _log(rng, 500, 260000)
        nodes = _log(rng, 1, max(2, min(128, 300000000 // (batch * vocab))))
        return {"op": op, "batch": batch, "nodes": nodes, "vocab": vocab, "tree": tree,
                "temperature": rng.choice([0.0, 0.5, 0.8, 1.0, 1.3]), "draft": rng.random() < 0.5,
                "f32": rng.random() < 0.4}
    batch, nodes, layers = _log(rng, 1, 64), _log(rng, 1, 64), _log(rng, 1, 36)
    cap = _log(rng, 40, max(64, min(4096, 7000000 // (batch * layers * kv))))
    return {"op": op, "batch": batch, "nodes": nodes, "layers": layers, "kv_heads": kv, "capacity": cap,
            "every": rng.choice([4, 8, 16]), "policy": rng.choice(["h2o_faithful", "lru"]), "score": rng.random() < 0.7}


# --------------------------------------------------------------------------- the inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _parents(kind, batch, nodes, seed):
    """Parents [batch, nodes] (numpy int32): chains, or trees whose nodes mostly hang on recent
    levels, those of every other sequence with up to a third of the nodes unused."""
    rng = np.random.RandomState(seed % (1 << 31))
    par = np.full((batch, nodes), -1, np.int32)
    t = np.arange(1, nodes)
    if kind == "chain":
        par[:, 1:] = t - 1
    else:
        # three children a node in the mean: a parent about a third of the way down
        lo, hi = np.maximum(0, t // 3 - 2), np.minimum(t - 1, t // 3 + 1)
        par[:, 1:] = lo + (rng.rand(batch, nodes - 1) * (hi - lo + 1)).astype(np.int32)
        used = nodes - rng.randint(0, nodes // 3 + 1, batch)
        used[::2] = nodes
        par[np.arange(nodes)[None, :] >= used[:, None]] = -2
    return par


def prepare(case, seed):
    return {"attend": _prepare_attend, "verify": _prepare_verify, "commit": _prepare_commit}[case["op"]](case, seed)


def _prepare_attend(c, seed):
    g = _gen(seed)
    B, T, hq, hkv, S = c["batch"], c["nodes"], c["heads"], c["kv_heads"], c["slots"]
    loud = 1 + 3 * (torch.rand(hkv, 1, DIM, generator=g, device=DEV) < 0.03).to(torch.float32)
    k = torch.empty(B, hkv, S, DIM, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    for b in range(B):
        k[b] = (_randn(g, hkv, S, DIM) * loud).to(torch.bfloat16)
        v[b] = _randn(g, hkv, S, DIM).to(torch.bfloat16)
    s = {"case": c, "k": k, "v": v, "q": (1.5 * _randn(g, B, T, hq, DIM)).to(torch.bfloat16),
         "k_draft": (_randn(g, B, hkv, T, DIM) * loud).to(torch.bfloat16),
         "v_draft": _randn(g, B, hkv, T, DIM).to(torch.bfloat16),
         "parents": torch.from_numpy(_parents(c["tree"], B, T, seed)).to(DEV),
         "lens": None, "slot_pos": None, "score": None}
    if c["lens"] == "ragged":  # lengths over the whole range, with an empty one in a batch
        lens = torch.exp(torch.rand(B, generator=g, device=DEV) * math.log(S + 1)).to(torch.int32).clamp(1, S)
        lens[0] = S
        if B > 2:
            lens[B // 2] = 0
        s["lens"] = lens
    if c["masked"]:  # a twentieth of the slots are free
        pos = torch.arange(S, device=DEV, dtype=torch.int32).repeat(B, 1)
        free = torch.rand(B, S, generator=g, device=DEV) < 0.05
        s["slot_pos"] = torch.where(free, torch.full_like(pos, -1), pos)
    if c["score"]:
        s["score"] = torch.zeros(B, T, S + T, dtype=torch.float32, device=DEV)
    return s


def _prepare_verify(c, seed):
    """Target rows with a handful of likely tokens over a long tail; a draft that knows them
    approximately."""
    g = _gen(seed)
    B, T, V = c["batch"], c["nodes"], c["vocab"]
    par = torch.from_numpy(_parents(c["tree"], B, T, seed)).to(DEV)
    up, seqs = par.clamp(min=0).long(), torch.arange(B, device=DEV)
    target = torch.empty(B, T, V, dtype=torch.float32 if c["f32"] else torch.bfloat16, device=DEV)
    draft = torch.empty(B, T, V, dtype=torch.float32, device=DEV) if c["draft"] else None
    temp = c["temperature"] if c["temperature"] > 0 else 1.0
    few = min(8, V)
    hunch = 0.7 * _randn(g, V)  # what the draft gets wrong about each token
    for t in range(T):
        row = 2 * _randn(g, B, V)
        top = torch.randint(0, V, (B, few), generator=g, device=DEV)
        row.scatter_(1, top, math.log(V) + 3 + 2 * _randn(g, B, few))
        target[:, t] = row.to(target.dtype)
        if draft is not None:
            draft[:, t] = torch.softmax((target[:, t].to(torch.float32) + hunch) / temp, -1)
    tokens = torch.zeros(B, T, dtype=torch.int32, device=DEV)
    for t in range(1, T):
        if draft is not None:  # a draw from the parent's draft distribution
            x = torch.rand(B, V, generator=g, device=DEV).clamp(min=1e-30)
            tokens[:, t] = torch.argmax(draft[seqs, up[:, t]] / -torch.log(x), -1).to(torch.int32)
        else:  # the parent's next most likely token, as the draft sees it
            rank = ((par[:, :t] == par[:, t:t + 1]).sum(1)).clamp(max=few - 1)
            best = torch.topk(target[seqs, up[:, t]].to(torch.float32) + hunch, few, -1)[1]
            tokens[:, t] = best[seqs, rank].to(torch.int32)
    return {"case": c, "target": target, "draft": draft, "tokens": tokens, "parents": par,
            "accept_u": torch.rand(B, T, generator=g, device=DEV), "sample_u": torch.rand(B, generator=g, device=DEV),
            "temperature": torch.full((B,), c["temperature"], device=DEV)}


STATE = {"slot_pos": torch.int32, "insert_step": torch.int32, "last_access": torch.int32, "access_count": torch.int32,
         "attn": torch.float32, "max_attn": torch.float32, "cumul": torch.float64, "prefill": torch.float32}


def _prepare_commit(c, seed):
    """Sequences some way into decoding: capacity + a few slots in use at scattered positions,
    and a path of one to a quarter of the nodes (eight at most) accepted."""
    g = _gen(seed)
    rng = np.random.RandomState((seed + 1) % (1 << 31))
    B, T, L, hkv, C, E = c["batch"], c["nodes"], c["layers"], c["kv_heads"], c["capacity"], c["every"]
    S, far, W, evcap = C + E + T, 6 * C + 64, (6 * C + 64 + 2 * T + 31) // 32 + 1, 8 * C + 512
    st = {k: np.zeros((B, S), {torch.int32: np.int32, torch.float32: np.float32, torch.float64: np.float64}[d])
          for k, d in STATE.items()}
    st["slot_pos"][:] = -1
    posmap = np.zeros((B, W * 32), bool)
    step = rng.randint(1, 5 * C, B).astype(np.int32)
    path = np.full((B, T), -1, np.int32)
    count = np.zeros(B, np.int32)
    for b in range(B):
        live = C + int(step[b] % E)
        at = rng.permutation(S)[:live]
        pos = rng.permutation(far)[:live]
        st["slot_pos"][b, at] = pos
        posmap[b, pos] = True
        st["insert_step"][b, at] = rng.randint(0, step[b], live)
        st["last_access"][b, at] = np.maximum(st["insert_step"][b, at], rng.randint(0, step[b] + 1, live))
        st["access_count"][b, at] = rng.randint(1, 50, live)
        st["attn"][b, at] = rng.rand(live) ** 4
        st["max_attn"][b, at] = np.maximum(st["attn"][b, at], rng.rand(live) ** 3)
        st["cumul"][b, at] = st["max_attn"][b, at].astype(np.float64) * rng.randint(1, 40, live)
        count[b] = rng.randint(1, max(2, min(8, T // 4 + 1) + 1))
        count[b] = min(count[b], T)
        if B > 2 and b == B // 2:
            count[b] = 0  # a sequence that sits this step out
        path[b, :count[b]] = np.sort(np.concatenate([[0], 1 + rng.permutation(T - 1)]).astype(np.int32)[:count[b]])
    bits = posmap.reshape(B, W, 32).astype(np.uint64) << np.arange(32, dtype=np.uint64)
    state = {k: torch.from_numpy(a).to(DEV) for k, a in st.items()}
    state["posmap"] = torch.from_numpy(bits.sum(-1).astype(np.uint32).view(np.int32)).to(DEV)
    state["seq_step"] = torch.from_numpy(step).to(DEV)
    state["next_pos"] = torch.full((B,), far, dtype=torch.int32, device=DEV)
    state["evlog"] = torch.zeros(B, evcap, dtype=torch.int32, device=DEV)
    state["evcount"] = torch.full((B,), 17, dtype=torch.int32, device=DEV)
    after = {k: torch.zeros_like(t) for k, t in state.items()}
    after["evlog"] = state["evlog"]  # a log is appended to in place
    s = {"case": c, "state": state, "after": after, "path": torch.from_numpy(path).to(DEV),
         "n_path": torch.from_numpy(count).to(DEV), "score": None}
    for name, rows in (("k", S), ("v", S), ("k_draft", T), ("v_draft", T)):
        s[name] = torch.empty(L, B, hkv, rows, DIM, dtype=torch.bfloat16, device=DEV)
        for i in range(L):
            s[name][i].normal_(generator=g)
    if c["score"]:
        s["score"] = torch.rand(B, T, S + T, generator=g, device=DEV) ** 6
    if own:
        from kvcacheboundaryprotection_b200 import speculative

        s["states"] = [speculative.SlotState(**x) for x in (state, after)]
        s["evict"] = speculative.EvictionSpec(policy=c["policy"], capacity=C, evict_every=E, protect=True)
    return s


# ------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        from kvcacheboundaryprotection_b200 import speculative

        if op == "attend":
            out = speculative.tree_attend(s["q"], s["k"], s["v"], s["k_draft"], s["v_draft"], s["parents"],
                                          slot_pos=s["slot_pos"], lens=s["lens"], node_score=s["score"])
            return {"out": out} if s["score"] is None else {"out": out, "score": s["score"]}
        if op == "verify":
            path, n, token = speculative.verify_tree(s["target"], s["tokens"], s["parents"], s["accept_u"],
                                                     s["sample_u"], temperature=s["temperature"],
                                                     draft_probs=s["draft"])
            return {"path": path, "n_path": n, "next_token": token}
        write = speculative.commit_tree(s["states"][0], s["path"], s["n_path"], s["k_draft"], s["v_draft"], s["k"],
                                        s["v"], node_score=s["score"], evict=s["evict"], out=s["states"][1])
        return {"write_slot": write, "k": s["k"], "v": s["v"], **s["after"]}
    return {"attend": _plain_attend, "verify": _plain_verify, "commit": _plain_commit}[op](s)


def _ancestors(par):
    """Truth [B, T, T]: node j is an ancestor of node i, or i itself; rows of unused nodes are empty."""
    B, T = par.shape
    anc = torch.zeros(B, T, T, dtype=torch.bool, device=par.device)
    seqs = torch.arange(B, device=par.device)
    for t in range(T):
        used = par[:, t] >= -1
        if t:
            used = used & ((par[:, t] == -1) | anc[seqs, par[:, t].clamp(min=0).long()].any(-1))
            anc[:, t] = anc[seqs, par[:, t].clamp(min=0).long()] & (par[:, t] >= 0)[:, None] & used[:, None]
        anc[:, t, t] = used
    return anc


def _plain_attend(s):
    """softmax(q . k / sqrt(128)) v over the live slots and the ancestors in 32 bits, and each key's
    largest probability over the heads."""
    c = s["case"]
    B, T, hq, hkv, S = c["batch"], c["nodes"], c["heads"], c["kv_heads"], c["slots"]
    G = hq // hkv
    live = torch.ones(B, S, dtype=torch.bool, device=DEV)
    if s["lens"] is not None:
        live = live & (torch.arange(S, device=DEV) < s["lens"][:, None])
    if s["slot_pos"] is not None:
        live = live & (s["slot_pos"] >= 0)
    anc = _ancestors(s["parents"])
    live = torch.cat([live[:, None, :] & anc.any(-1)[:, :, None], anc], -1)              # [B, T, S + T]
    k = torch.cat([s["k"], s["k_draft"]], 2).to(torch.float32)                           # [B, hkv, S + T, 128]
    q = s["q"].to(torch.float32).reshape(B, T, hkv, G, DIM).permute(0, 2, 1, 3, 4).reshape(B, hkv, T * G, DIM)
    l = (torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(DIM))).reshape(B, hkv, T, G, S + T)
    del k
    live = live[:, None, :, None, :]
    l = torch.where(live, l, torch.full((), -math.inf, device=DEV))
    top = l.amax(-1, keepdim=True)
    l = torch.exp(l - torch.where(top > -math.inf, top, torch.zeros_like(top)))          # 0 where masked
    total = l.sum(-1, keepdim=True)
    p = l / torch.where(total > 0, total, torch.ones_like(total))
    del l
    v = torch.cat([s["v"], s["v_draft"]], 2).to(torch.float32)
    out = torch.matmul(p.reshape(B, hkv, T * G, S + T), v).reshape(B, hkv, T, G, DIM)
    out = {"out": out.permute(0, 2, 1, 3, 4).reshape(B, T, hq, DIM).to(torch.bfloat16)}
    if s["score"] is not None:
        s["score"].copy_(torch.maximum(s["score"], p.amax((1, 3))))
        out["score"] = s["score"]
    return out


def _plain_verify(s):
    """The walk over the nodes for all sequences at once.  The weights and their sums are in 64 bits:
    a token is chosen where a running sum of a hundred thousand terms passes a border."""
    c = s["case"]
    B, T = c["batch"], c["nodes"]
    seqs = torch.arange(B, device=DEV)
    par, greedy = s["parents"], s["temperature"] <= 0
    temp = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).to(torch.float64)[:, None]

    def weights(node):
        x = s["target"][seqs, node].to(torch.float64)
        top, at = x.max(-1, keepdim=True)
        first = torch.argmax((x == top).to(torch.int8), -1, keepdim=True)  # the lowest index of a tie
        one = torch.zeros_like(x).scatter_(1, first, 1.0)
        return torch.where(greedy[:, None], one, torch.exp((x - top) / temp))

    cur = torch.zeros(B, dtype=torch.long, device=DEV)
    r = weights(cur)
    path = torch.full((B, T), -1, dtype=torch.int32, device=DEV)
    path[:, 0] = 0
    n = torch.ones(B, dtype=torch.int32, device=DEV)
    for t in range(1, T):
        mine = par[:, t] == cur
        x = s["tokens"][:, t].long()
        R = r.sum(-1)
        rx = r[seqs, x]
        if s["draft"] is not None:
            q = s["draft"][seqs, cur].to(torch.float64)
            qx = q[seqs, x]
        else:
            q, qx = None, torch.ones_like(R)
        qx = torch.where(greedy, torch.ones_like(qx), qx)
        yes = mine & (s["accept_u"][:, t].to(torch.float64) * qx * R < rx)
        no = mine & ~yes
        left = r.clone()
        left[seqs, x] = 0
        if q is not None:
            left = torch.where(greedy[:, None], left, (r / R[:, None] - q).clamp(min=0))
        cur = torch.where(yes, torch.full_like(cur, t), cur)
        r = torch.where(yes[:, None], weights(cur), torch.where(no[:, None], left, r))
        path[seqs, torch.where(yes, n, torch.zeros_like(n)).long()] = torch.where(
            yes, torch.full_like(n, t), torch.zeros_like(n))
        n = n + yes.to(torch.int32)
    total = torch.cumsum(r, -1)
    want = s["sample_u"].to(torch.float64) * total[:, -1]
    token = torch.argmax((total > want[:, None]).to(torch.int8), -1)
    return {"path": path, "n_path": n, "next_token": token.to(torch.int32)}


def _spelled(pos):
    """Numbers in the order of the strings of pos: a shorter one sorts before what it begins."""
    p = pos.to(torch.int64).clamp(min=0)
    digits = torch.ones_like(p)
    for i in range(1, 10):
        digits = digits + (p >= 10 ** i)
    return p * torch.pow(torch.full_like(p, 10), 10 - digits) * 16 + digits


def _rank_by(keys, able):
    """Slots [B, S] in the order of the keys (the first decides), those that are not ``able`` last."""
    order = torch.arange(able.shape[1], device=DEV).repeat(able.shape[0], 1)
    for key in list(keys)[::-1] + [~able]:
        order = torch.gather(order, 1, torch.argsort(torch.gather(key, 1, order), dim=1, stable=True))
    return order


def _plain_commit(s):
    """Appends and score updates node by node for all sequences at once, then the eviction."""
    c = s["case"]
    B, T, L, C, E = c["batch"], c["nodes"], c["layers"], c["capacity"], c["every"]
    a, before = s["after"], s["state"]
    for name, t in before.items():
        if name != "evlog":
            a[name].copy_(t)
    S, W = a["slot_pos"].shape[1], a["posmap"].shape[1]
    seqs = torch.arange(B, device=DEV)
    write = torch.full((B, T), -1, dtype=torch.int32, device=DEV)
    where = torch.arange(S, device=DEV)
    bit = torch.ones((), dtype=torch.int32, device=DEV)
    for i in range(min(T, 9)):
        on = i < s["n_path"]
        node = s["path"][:, i].clamp(min=0).long()
        a["seq_step"] += on.to(torch.int32)
        step, pos = a["seq_step"], a["next_pos"].clone()
        slot = torch.argmax((a["slot_pos"] < 0).to(torch.int8), -1)
        new = on[:, None] & (where == slot[:, None])
        for name, value in (("slot_pos", pos), ("insert_step", step), ("last_access", step)):
            a[name].copy_(torch.where(new, value[:, None], a[name]))
        a["access_count"].copy_(torch.where(new, torch.ones_like(a["access_count"]), a["access_count"]))
        for name in ("attn", "max_attn", "cumul", "prefill"):
            a[name].copy_(torch.where(new, torch.zeros_like(a[name]), a[name]))
        word = (pos >> 5).clamp(max=W - 1).long()
        a["posmap"][seqs, word] |= torch.where(on, bit << (pos & 31), torch.zeros_like(pos))
        a["next_pos"] += on.to(torch.int32)
        write[:, i] = torch.where(on, slot.to(torch.int32), write[:, i])
        if s["score"] is None:
            continue
        row = s["score"][seqs, node]
        x = row[:, :S].clone()
        for j in range(i + 1):  # what the path's own nodes got
            at, from_ = write[:, j].clamp(min=0).long(), s["path"][:, j].clamp(min=0).long()
            x[seqs, at] = torch.where(on, row[seqs, S + from_], x[seqs, at])
        live = on[:, None] & (a["slot_pos"] >= 0)
        x = torch.where(live, x, torch.zeros_like(x))
        used = live & (x > (0.05 * x.amax(1, keepdim=True).to(torch.float64)).to(torch.float32))
        a["attn"].copy_(torch.where(live, x, a["attn"]))
        a["max_attn"].copy_(torch.where(live, torch.maximum(x, a["max_attn"]), a["max_attn"]))
        a["cumul"].copy_(torch.where(live, a["cumul"] + x.to(torch.float64), a["cumul"]))
        a["last_access"].copy_(torch.where(used, step[:, None], a["last_access"]))
        a["access_count"] += used.to(torch.int32)
    # the eviction: capacity // 10 positions at either end are protected
    due = (a["seq_step"] // E) > (before["seq_step"] // E)
    edge = max(4, int(C * 0.10))
    live = a["slot_pos"] >= 0
    R = live.sum(1)
    nth = torch.empty_like(a["slot_pos"], dtype=torch.int64)
    nth.scatter_(1, _rank_by([a["slot_pos"]], live), where.repeat(B, 1))
    able = live & (nth >= edge) & (nth < (R - edge)[:, None]) & (due & (R > C) & (R > edge))[:, None]
    k = torch.minimum((R - C).clamp(min=0), able.sum(1))
    lead = [a["cumul"]] if c["policy"] == "h2o_faithful" else []
    _free(a, _rank_by(lead + [a["last_access"], a["insert_step"], _spelled(a["slot_pos"])], able), k)
    live = a["slot_pos"] >= 0
    over = torch.where(due, (live.sum(1) - C).clamp(min=0), torch.zeros_like(R))
    _free(a, _rank_by([a["last_access"], a["insert_step"], a["slot_pos"]], live), over)
    for i in range(min(T, 9)):
        at = write[:, i].clamp(min=0).long()
        kept = (write[:, i] >= 0) & (a["slot_pos"][seqs, at] == before["next_pos"] + i)
        write[:, i] = torch.where(kept, write[:, i], torch.full_like(write[:, i], -1))
        node = s["path"][:, i].clamp(min=0).long()
        for cache, draft in ((s["k"], s["k_draft"]), (s["v"], s["v_draft"])):
            cache[:, seqs, :, at] = torch.where(kept[:, None, None, None], draft[:, seqs, :, node],
                                                cache[:, seqs, :, at])
    return {"write_slot": write, "k": s["k"], "v": s["v"], **a}


def _free(a, order, count):
    """Frees the first ``count`` [B] slots of ``order`` and logs their positions."""
    B, S = order.shape
    n = torch.arange(S, device=DEV)
    out = n < count[:, None]
    pos = torch.gather(a["slot_pos"], 1, order)
    at = (a["evcount"].long()[:, None] + n).clamp(max=a["evlog"].shape[1] - 1)
    a["evlog"].scatter_(1, at, torch.where(out, pos, torch.gather(a["evlog"], 1, at)))
    gone = torch.zeros_like(a["posmap"])
    bit = torch.ones((), dtype=torch.int32, device=DEV)
    word = (pos >> 5).clamp(0, gone.shape[1] - 1).long()
    gone.scatter_add_(1, word, torch.where(out, bit << (pos & 31), torch.zeros_like(pos)))  # distinct bits: a sum is an or
    a["posmap"] &= ~gone
    a["slot_pos"].scatter_(1, order, torch.where(out, torch.full_like(pos, -1), pos))
    a["evcount"] += count.to(torch.int32)


# -------------------------------------------------------------------------- the work done
def _slots_in_use(c):
    """Slots that a pass reads: of a ragged batch the lengths' mean (they are drawn)."""
    if c["lens"] == "full":
        return c["batch"] * c["slots"] * (0.95 if c["masked"] else 1)
    S, n = c["slots"], max(0, c["batch"] - (2 if c["batch"] > 2 else 1))
    return S + n * max(1.0, S / math.log(S + 1))


def work(case):
    c = case
    if c["op"] == "attend":
        B, T, n = c["batch"], c["nodes"], _slots_in_use(c) + c["batch"] * c["nodes"]
        extra = (4 * n if c["masked"] else 0) + (8 * n * T if c["score"] else 0)
        return {"bytes": n * c["kv_heads"] * 512 + extra + 512 * B * T * c["heads"] + 4 * B * T,
                "flops": 4 * n * c["heads"] * T * DIM}
    if c["op"] == "verify":
        # rows on the accepted path: the root's, and a few levels of the tree (as the inputs are drawn,
        # about two thirds of the levels' candidates pass)
        depth = c["nodes"] - 1 if c["tree"] == "chain" else math.log(max(1, 2 * c["nodes"] / 3 + 1), 3)
        rows = c["batch"] * (1 + min(2.0, 0.6 * depth))
        one = (4 if c["f32"] else 2) + (2 if c["draft"] and c["temperature"] > 0 else 0)
        return {"bytes": rows * c["vocab"] * one + 24 * c["batch"] * c["nodes"], "flops": 4 * rows * c["vocab"]}
    B, T, S = c["batch"], c["nodes"], c["capacity"] + c["every"] + c["nodes"]
    m = (1 + max(1, min(8, T // 4 + 1))) / 2
    score = 4 * B * m * (S + m) if c["score"] else 0
    return {"bytes": 2 * B * S * 36 + score + 4 * m * B * c["layers"] * c["kv_heads"] * DIM * 2, "flops": B * S * (m + 8)}


# ---------------------------------------------------------------------- 64-bit definition
def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "verify": _exact_verify, "commit": _exact_commit}[case["op"]](case, s)


def _above(par):
    """For each node the nodes it sees, itself last; None for an unused one."""
    sees = []
    for t, p in enumerate(par):
        sees.append([t] if p == -1 else sees[p] + [t] if 0 <= p < t and sees[p] is not None else None)
    return sees


def _exact_attend(c, s):
    B, T, hq, hkv, S = c["batch"], c["nodes"], c["heads"], c["kv_heads"], c["slots"]
    G = hq // hkv
    out = torch.zeros(B, T, hq, DIM, dtype=torch.float64, device=DEV)
    score = None if s["score"] is None else s["score"].double()
    for b in range(B):
        at = torch.arange(S if s["lens"] is None else int(s["lens"][b]), device=DEV)
        if s["slot_pos"] is not None:
            at = at[s["slot_pos"][b, at] >= 0]
        sees = _above(s["parents"][b].tolist())
        hidden = torch.ones(T, T, dtype=torch.bool, device=DEV)
        for t in range(T):
            if sees[t] is not None:
                hidden[t, sees[t]] = False
        used = [t for t in range(T) if sees[t] is not None]
        if not used:
            continue
        for h in range(hkv):
            k = torch.cat([s["k"][b, h, at], s["k_draft"][b, h]]).double()
            v = torch.cat([s["v"][b, h, at], s["v_draft"][b, h]]).double()
            q = s["q"][b, used, h * G:(h + 1) * G].double()
            z = torch.einsum("tgd,nd->tgn", q, k) / math.sqrt(DIM)
            z[..., len(at):].masked_fill_(hidden[used][:, None], -math.inf)
            p = torch.softmax(z, -1)
            out[b, used, h * G:(h + 1) * G] = torch.einsum("tgn,nd->tgd", p, v)
            if score is not None:
                cols = torch.cat([at, torch.arange(S, S + T, device=DEV)])
                for j, t in enumerate(used):
                    score[b, t, cols] = torch.maximum(score[b, t, cols], p[j].amax(0))
    return {"out": out} if score is None else {"out": out, "score": score}


def _exact_verify(c, s):
    path, count, token = [], [], []
    for b in range(c["batch"]):
        par, toks, us = (s[n][b].tolist() for n in ("parents", "tokens", "accept_u"))
        heat, way = float(s["temperature"][b]), [0]

        def law(node):
            x = s["target"][b, node].double()
            if heat <= 0:
                one = torch.zeros_like(x)
                one[int((x == x.max()).nonzero()[0])] = 1
                return one
            return torch.softmax(x / heat, -1)

        p = law(0)
        for t in range(1, c["nodes"]):
            if par[t] != way[-1]:
                continue
            x = toks[t]
            q = torch.zeros_like(p)
            q[x] = 1
            if s["draft"] is not None and heat > 0:
                q = s["draft"][b, way[-1]].double()
            if us[t] * float(q[x]) < float(p[x]):
                way.append(t)
                p = law(t)
            else:
                p = torch.clamp(p - q, min=0)
                p = p / p.sum()
        run_ = torch.cumsum(p, 0)
        token.append(int((run_ > float(s["sample_u"][b]) * float(run_[-1])).nonzero()[0]))
        path.append(way + [-1] * (c["nodes"] - len(way)))
        count.append(len(way))
    whole = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return {"path": whole(path), "n_path": whole(count), "next_token": whole(token)}


def _exact_commit(c, s):
    B, T, C, E = c["batch"], c["nodes"], c["capacity"], c["every"]
    st = {k: v.cpu().numpy().copy() for k, v in s["state"].items()}
    score = None if s["score"] is None else s["score"].cpu().numpy()
    path, count = s["path"].tolist(), s["n_path"].tolist()
    S, W = st["slot_pos"].shape[1], st["posmap"].shape[1]
    write = np.full((B, T), -1, np.int32)
    edge = max(4, int(C * 0.10))
    for b in range(B):
        r = {k: st[k][b] for k in STATE}
        was = int(st["seq_step"][b])
        held = {int(p): i for i, p in enumerate(r["slot_pos"]) if p >= 0}
        slots = []
        for i, node in enumerate(path[b][:count[b]]):
            st["seq_step"][b] += 1
            now, pos = int(st["seq_step"][b]), int(st["next_pos"][b])
            st["next_pos"][b] += 1
            slot = int(np.flatnonzero(r["slot_pos"] < 0)[0])
            for name, value in (("slot_pos", pos), ("insert_step", now), ("last_access", now), ("access_count", 1),
                                ("attn", 0), ("max_attn", 0), ("cumul", 0), ("prefill", 0)):
                r[name][slot] = value
            held[pos] = slot
            slots.append((slot, pos))
            if score is None:
                continue
            got = score[b, node, :S].copy()
            for (at, _), other in zip(slots, path[b]):
                got[at] = score[b, node, S + other]
            at = np.array(sorted(held.values()))
            floor = np.float32(0.05 * float(got[at].max()))
            r["attn"][at] = got[at]
            r["max_attn"][at] = np.maximum(r["max_attn"][at], got[at])
            r["cumul"][at] += got[at].astype(np.float64)
            hot = at[got[at] > floor]
            r["last_access"][hot] = now
            r["access_count"][hot] += 1
        if int(st["seq_step"][b]) // E > was // E:
            log = []
            there = sorted(held)
            want = max(0, len(there) - C)
            inner = there[edge:len(there) - edge] if want and edge < len(there) else []

            def order(p):
                i = held[p]
                last = (int(r["last_access"][i]), int(r["insert_step"][i]), str(p))
                return (float(r["cumul"][i]),) + last if c["policy"] == "h2o_faithful" else last

            log += sorted(inner, key=order)[:want]
            rest = [p for p in there if p not in set(log)]
            rest.sort(key=lambda p: (int(r["last_access"][held[p]]), int(r["insert_step"][held[p]]), p))
            log += rest[:max(0, len(rest) - C)]
            for p in log:
                r["slot_pos"][held.pop(p)] = -1
                st["evlog"][b, st["evcount"][b]] = p
                st["evcount"][b] += 1
        bits = np.zeros(W * 32, np.uint64)
        bits[list(held)] = 1
        st["posmap"][b] = (bits.reshape(W, 32) << np.arange(32, dtype=np.uint64)).sum(1).astype(np.uint32).view(np.int32)
        for i, (slot, pos) in enumerate(slots):
            if held.get(pos) == slot:
                write[b, i] = slot
                for name in ("k", "v"):
                    s[name][:, b, :, slot] = s[name + "_draft"][:, b, :, path[b][i]]
    return {"write_slot": torch.from_numpy(write).to(DEV), "k": s["k"], "v": s["v"],
            **{k: torch.from_numpy(v).to(DEV) for k, v in st.items()}}
