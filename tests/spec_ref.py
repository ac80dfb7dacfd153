"""Plain statements of the speculative decoding operators in 64 bits: tree attention, verification
of drafted tokens, commit of the accepted path (victims by the oracle's policies)."""

import math

import numpy as np
import torch

from oracle.policies import Meta, PolicySpec, hard_cap


def sees(parents):
    """For each node the list of the nodes that it sees (ancestors, itself last); None: unused."""
    out = []
    for t, p in enumerate(parents):
        if p == -1:
            out.append([t])
        elif 0 <= p < t and out[p] is not None:
            out.append(out[p] + [t])
        else:
            out.append(None)
    return out


def random_tree(rng, T, kind="tree", unused=0):
    """parents of T nodes, the last ``unused`` of them unused."""
    par = [-1]
    for t in range(1, T):
        par.append(t - 1 if kind == "chain" else 0 if kind == "star" else int(rng.integers(max(0, t // 3 - 2), t)))
    for t in range(T - unused, T):
        par[t] = -2
    return par


def attend(q, k, v, kd, vd, parents, slot_pos=None, lens=None, scale=None):
    """(out [B, T, Hq, 128], p [B, T, S + T] the largest probability over the heads, mag [B, T, Hq, 128]
    the sum of p |v|, spread [B, T, Hq] the largest sum of |q k scale|) in 64 bits, on the CPU."""
    B, T, hq, D = q.shape
    hkv, S = k.shape[1], k.shape[2]
    G = hq // hkv
    scale = 1 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, T, hq, D, dtype=torch.float64)
    mag, top, spread = torch.zeros_like(out), torch.zeros(B, T, S + T, dtype=torch.float64), torch.zeros(B, T, hq)
    for b in range(B):
        n = S if lens is None else min(max(int(lens[b]), 0), S)
        at = torch.arange(n)
        if slot_pos is not None:
            at = at[slot_pos[b, :n].cpu() >= 0]
        for t, seen in enumerate(sees(parents[b].tolist())):
            if seen is None:
                continue
            cols = torch.cat([at, S + torch.tensor(seen)])
            for h in range(hq):
                kk = torch.cat([k[b, h // G, at], kd[b, h // G, seen]]).double()
                vv = torch.cat([v[b, h // G, at], vd[b, h // G, seen]]).double()
                qq = q[b, t, h].double()
                p = torch.softmax(kk @ qq * scale, 0)
                out[b, t, h] = p @ vv
                mag[b, t, h] = p @ vv.abs()
                spread[b, t, h] = (kk.abs() @ qq.abs()).max() * abs(scale)
                top[b, t, cols] = torch.maximum(top[b, t, cols], p)
    return out, top, mag, spread


def verify(target, tokens, parents, accept_u, sample_u, temperature=None, draft=None):
    """(path, next token) of one sequence: target [T, V] 64-bit numpy, draft [T, V] or None."""
    T, V = target.shape
    if parents[0] != -1:
        return [], -1
    heat = 1.0 if temperature is None else float(temperature)
    greedy = not heat > 0

    def law(n):
        x = np.where(np.isnan(target[n]), -np.inf, target[n])
        if greedy:
            w = np.zeros(V)
            w[int(np.argmax(x))] = 1
            return w
        with np.errstate(invalid="ignore"):
            return np.where(x == x.max(), 1.0, np.exp((x - x.max()) / heat))

    way, r = [0], law(0)
    r0 = r
    for t in range(1, T):
        if parents[t] != way[-1] or not 0 <= tokens[t] < V:
            continue
        x = int(tokens[t])
        if draft is not None and not greedy:
            q = draft[way[-1]].astype(np.float64)
        else:
            q = np.zeros(V)
            q[x] = 1
        if float(accept_u[t]) * q[x] * r.sum() < r[x]:
            way.append(t)
            r = r0 = law(t)
        elif draft is not None and not greedy:
            r = np.maximum(r / r.sum() - q, 0)
        else:
            r = r.copy()
            r[x] = 0
    if not r.sum() > 0:
        r = r0
    run = np.cumsum(r)
    over = np.flatnonzero((run > float(sample_u) * run[-1]) & (r > 0))
    return way, int(over[0]) if len(over) else int(np.flatnonzero(r > 0)[-1])


def commit(st, path, n, score, evict=None):
    """The state (dict of numpy arrays of one sequence, changed in place; scalars seq_step, next_pos;
    list log) after the commit of ``path[:n]``; returns the slot of each entry (-1: none).  evict:
    (policy, capacity, every, protect, prefix_frac, suffix_frac)."""
    S = len(st["slot_pos"])
    was, slots = st["seq_step"], []
    for i in range(n):
        st["seq_step"] += 1
        now, pos = st["seq_step"], st["next_pos"]
        st["next_pos"] += 1
        free = np.flatnonzero(st["slot_pos"] < 0)
        slot = int(free[0]) if len(free) else -1
        slots.append((slot, pos))
        if slot >= 0:
            for name, val in (("slot_pos", pos), ("insert_step", now), ("last_access", now), ("access_count", 1),
                              ("attn", 0), ("max_attn", 0), ("cumul", 0), ("prefill", 0)):
                st[name][slot] = val
        if score is None:
            continue
        got = score[path[i], :S].copy()
        for (s, _), node in zip(slots, path):
            if s >= 0:
                got[s] = score[path[i], S + node]
        at = np.flatnonzero(st["slot_pos"] >= 0)
        floor = np.float32(0.05 * float(max(np.float32(0), got[at].max()))) if len(at) else 0
        st["attn"][at] = got[at]
        st["max_attn"][at] = np.maximum(st["max_attn"][at], got[at])
        st["cumul"][at] += got[at].astype(np.float64)
        hot = at[got[at] > floor]
        st["last_access"][hot] = now
        st["access_count"][hot] += 1
    if evict is not None and st["seq_step"] // evict[2] > was // evict[2]:
        name, cap, _, protect, pf, sf = evict
        held = {int(p): s for s, p in enumerate(st["slot_pos"]) if p >= 0}
        m = Meta.zeros(max(held) + 1)
        for p, s in held.items():
            for a, b in (("insert_step", "insert_step"), ("last_access", "last_access"), ("attn", "attn"),
                         ("max_attn", "max_attn"), ("cumul", "cumul"), ("prefill", "prefill")):
                getattr(m, a)[p] = st[b][s]
        there = sorted(held)
        spec = PolicySpec(name, cap, protect=protect, prefix_frac=pf, suffix_frac=sf)
        vict = spec.select(there, m, max(0, len(there) - cap), st["seq_step"]) if len(there) > cap else []
        rest = [p for p in there if p not in set(vict)]
        vict = list(vict) + hard_cap(rest, m, len(rest) - cap)
        for p in vict:
            st["slot_pos"][held[p]] = -1
        st["log"] += vict
    return [s if s >= 0 and st["slot_pos"][s] == p else -1 for s, p in slots]
