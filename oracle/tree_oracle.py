"""Plain NumPy forms, in 64 bits, of the operators of a step with several drafted tokens (include/msaq_b200.h: msaq_kv_write_qkv,
msaq_kv_tree_attention, msaq_verify_tree, msaq_kv_keep).  Test infrastructure only; loops, one sequence and one node at a time."""

import numpy as np

from . import msaq_oracle as orc


def tree_mask(parents):
    """parents [T] -> list of sets: the nodes each node attends."""
    seen = []
    for i, p in enumerate(parents):
        if i == 0:
            seen.append({0})
        else:
            seen.append(seen[p] | {i} if p >= 0 and seen[p] else set())
    return seen


def mask_words(seen):
    """Sets of nodes -> int64 mask words."""
    return np.array([sum(1 << j for j in s) for s in seen], dtype=np.uint64).view(np.int64)


def norm_heads(x, gain, eps):
    """x [..., D] (values of bf16) -> (x r) g with r rounded to fp32 and every product too."""
    if gain is None:
        return np.asarray(x, np.float32)
    x64 = np.asarray(x, np.float64)
    r = (1.0 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + eps)).astype(np.float32)
    return (np.asarray(x, np.float32) * r) * np.asarray(gain, np.float32)


def write_qkv(qkv, planes_k, planes_v, Hq, Hkv, D, u, gs, start, tables, q_gain, k_gain, eps, pos, counts, rotate):
    """qkv [B,T,(Hq+2Hkv)*D] float32 values of bf16; planes (scale, upper, shared) NumPy, written in place -> q [B,T,Hq,D]."""
    B, T, _ = qkv.shape
    heads = qkv.reshape(B, T, Hq + 2 * Hkv, D)
    Lcap = planes_k[0].shape[3]
    q = np.zeros((B, T, Hq, D), np.float32)
    for b in range(B):
        for t in range(T):
            if counts is not None and t >= counts[b]:
                continue
            slot = start[b] + t
            p = slot if pos is None else pos[b, t]
            qr, kr = norm_heads(heads[b, t, :Hq], q_gain, eps), norm_heads(heads[b, t, Hq:Hq + Hkv], k_gain, eps)
            ok = True
            if tables is not None:
                rows = len(tables[0])
                at = 0 if rows == 1 else min(max(p, 0), rows - 1)
                ok = rows == 1 or at == p
                qr, kr = orc.rope(qr, tables[0][at], tables[1][at]), orc.rope(kr, tables[0][at], tables[1][at])
            qr, kr = orc.to_bf16(qr), orc.to_bf16(kr)
            q[b, t] = qr
            if not ok or slot < 0 or slot >= Lcap:
                continue
            pk = (orc.pack_kv_rotated if rotate else orc.pack_kv)(kr[:, None, :], u, gs)
            pv = orc.pack_kv(heads[b, t, Hq + Hkv:][:, None, :], u, gs)
            for planes, pack in ((planes_k, pk), (planes_v, pv)):
                for plane, key in zip(planes, ("scale_exp", "upper", "shared")):
                    plane[b, :, :, slot] = pack[key][:, :, 0]
    return q


def tree_attention(q, planes_k, planes_v, u, gs, lens, seen, rotate):
    """q [B,T,Hq,D]; seen[b][i]: nodes that node i attends -> (out, mag, big, all) in 64 bits: the result, the same
    average of |v|, per (b, i, head) the largest sum |q_d k_d| / sqrt(D) over the attended keys, and the plain sum of |v| over them."""
    B, T, Hq, D = q.shape
    Hkv = planes_k[0].shape[1]
    G = Hq // Hkv
    out, mag, big, all_v = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:3]), np.zeros(q.shape)
    for b in range(B):
        need = lens[b] + T
        K = orc.dequant_kv_planes(*[p[b][:, :, :need] for p in planes_k], u, gs).astype(np.float64)
        V = orc.dequant_kv_planes(*[p[b][:, :, :need] for p in planes_v], u, gs).astype(np.float64)
        for i in range(T):
            keys = list(range(lens[b])) + [lens[b] + j for j in sorted(seen[b][i]) if j < T]
            if not keys:
                continue
            qi = orc.rotate_f32(q[b, i]).astype(np.float64) if rotate else q[b, i].astype(np.float64)
            for h in range(Hq):
                k, v = K[h // G][keys], V[h // G][keys]
                s = k @ qi[h] / np.sqrt(D)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, i, h], mag[b, i, h] = p @ v, p @ np.abs(v)
                all_v[b, i, h] = np.abs(v).sum(0)
                big[b, i, h] = (np.abs(k) @ np.abs(qi[h])).max() / np.sqrt(D)
    return out, mag, big, all_v


def _clean(p):
    p = np.asarray(p, np.float64)
    return np.where((p > 0) & np.isfinite(p), p, 0.0)


def verify_tree(target, tokens, parents, u, draft=None):
    """One sequence: target [T,V], tokens [T], parents [T], u [T], draft [T,V] or None -> (path, token)."""
    T, V = target.shape
    cur, path = 0, [0]
    r, Z = _clean(target[0]), 1.0
    for j in range(1, T):
        x = int(tokens[j])
        if parents[j] != cur or not 0 <= x < V:
            continue
        q = None if draft is None else _clean(draft[cur])
        if float(u[j]) * (1.0 if q is None else q[x]) * Z < r[x]:
            cur = j
            path.append(j)
            r, Z = _clean(target[j]), 1.0
        elif q is None:
            Z -= r[x]
            r[x] = 0.0
        else:
            r = np.maximum(r - Z * q, 0.0)
            Z = r.sum()
    if r.sum() <= 0:
        r = _clean(target[cur])
    if r.sum() <= 0:
        return path, -1
    above = np.nonzero(np.cumsum(r) > float(u[0]) * r.sum())[0]
    return path, int(above[0]) if len(above) else int(np.nonzero(r)[0][-1])


def keep(planes, start, path, count):
    """The planes after the move, new arrays."""
    out = [p.copy() for p in planes]
    for new, old in zip(out, planes):
        for b in range(len(path)):
            for k in range(count[b]):
                new[b, :, :, start[b] + k] = old[b, :, :, start[b] + path[b][k]]
    return out
